// Attention of new tokens over a paged e4m3 cache with a sliding window and sink tokens.
//
// A query at position p (its context is p + 1) sees key j iff j <= p and (W = 0 or j > p - W or
// j < S): the last W positions, its own among them, and the first S tokens of the sequence.
//   o = softmax(q K^T * scale) V, then o * sigmoid(gate) where a gate is given, rounded to bf16 once.
// Queries keep their bf16 value and probabilities about that of bf16 (the kernels of attention_tc.cu
// round both to one e4m3 number). A row that sees no key is zero. Keys outside the visible range are
// never used, whatever their pages hold.
//
// KV cache layout: [pages][kv_heads][64][head_dim] e4m3 for K and V separately.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <climits>
#include "common.cuh"

namespace r9k {

namespace wa {
constexpr int PAGE = 64;

struct Args {
  const __nv_bfloat16* q;  // [T, Hq, D], token stride ld_q
  int64_t ld_q;
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* table;  // [S, width]
  const int32_t* seq_start;
  const int32_t* seq_len;
  const int32_t* tok_ctx;
  const __nv_bfloat16* gate;  // [T, Hq * D], token stride ld_gate, or null
  __nv_bfloat16* out;         // [T, Hq * D], token stride ld_out
  int64_t ld_gate, ld_out;
  int T, S, Hq, Hkv, G, width, pages, window, sinks, max_new;
  float scale;    // sm_scale * k_scale
  float v_scale;
  int* status;
};
}  // namespace wa

// One warp a (token, query head) row; a lane holds D / 32 of its dims; running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) window_attn_simple_kernel(const wa::Args a) {
  using namespace wa;
  pdl_wait();
  pdl_trigger();
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int seq = blockIdx.z, j = blockIdx.x;
  if (h >= a.Hq) return;
  const int t0 = a.seq_start[seq], len = a.seq_len[seq];
  if (len > a.max_new && j == 0 && h == 0 && lane == 0) report_error(a.status, kErrConfig, 300, len);
  if (j >= len) return;
  if (t0 < 0 || t0 + len > a.T) {
    if (lane == 0) report_error(a.status, kErrBounds, 300, t0);
    return;
  }
  const int t = t0 + j;
  int ctx = a.tok_ctx[t];
  if (ctx > a.width * PAGE) {
    if (lane == 0) report_error(a.status, kErrBounds, 301, ctx);
    ctx = a.width * PAGE;
  }
  const int lo = a.window > 0 ? max(0, ctx - a.window) : 0;
  const int ns = min(a.sinks, lo);
  float qv[PER], acc[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    qv[i] = __bfloat162float(a.q[(int64_t)t * a.ld_q + h * D + lane + 32 * i]) * a.scale;
    acc[i] = 0.f;
  }
  const int kvh = h / a.G;
  for (int i = 0; i < ns + ctx - lo; ++i) {
    const int key = i < ns ? i : lo + i - ns;
    const int page = a.table[(int64_t)seq * a.width + key / PAGE];
    if ((unsigned)page >= (unsigned)a.pages) {
      if (lane == 0) report_error(a.status, kErrBounds, 302, page);
      continue;
    }
    const int64_t base = (((int64_t)page * a.Hkv + kvh) * PAGE + key % PAGE) * D + lane;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < PER; ++c) s += qv[c] * e4m3_to_f32(a.k[base + 32 * c]);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, s);
    if (mn == -INFINITY) continue;  // no weight yet, and none in this key
    const float corr = __expf(m - mn), pw = __expf(s - mn);
    l = l * corr + pw;
#pragma unroll
    for (int c = 0; c < PER; ++c) acc[c] = acc[c] * corr + pw * e4m3_to_f32(a.v[base + 32 * c]);
    m = mn;
  }
  const float inv = l > 0.f || l != l ? a.v_scale / l : 0.f;
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int d = h * D + lane + 32 * c;
    float o = acc[c] * inv;
    if (a.gate != nullptr) o *= sigmoid_f(__bfloat162float(a.gate[(int64_t)t * a.ld_gate + d]));
    a.out[(int64_t)t * a.ld_out + d] = __float2bfloat16(o);
  }
}

void window_attention(torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor block_table,
                      torch::Tensor seq_start, torch::Tensor seq_len, torch::Tensor tok_ctx, double sm_scale,
                      double k_scale, double v_scale, int64_t window, int64_t sinks, c10::optional<torch::Tensor> gate,
                      torch::Tensor out, int64_t max_new, int64_t max_ctx, torch::Tensor status) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.dtype() == torch::kBFloat16, "window_attention: q bf16 [tokens, heads, head_dim]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), S = seq_start.numel();
  TORCH_CHECK(D == 128 || D == 256, "window_attention: head_dim must be 128 or 256");
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) == D, "window_attention: a token's heads must be contiguous");
  for (const torch::Tensor* c : {&k_cache, &v_cache})
    TORCH_CHECK(c->device() == q.device() && c->dtype() == torch::kUInt8 && c->dim() == 4 && c->is_contiguous() &&
                    c->sizes() == k_cache.sizes() && c->size(2) == wa::PAGE && c->size(3) == D,
                "window_attention: caches uint8 (e4m3) [pages, kv_heads, 64, head_dim], contiguous");
  const int64_t Hkv = k_cache.size(1);
  TORCH_CHECK(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 128, "window_attention: query heads a multiple (<= 128) of kv heads");
  auto ints = [&](const torch::Tensor& t, int64_t n, const char* what) {
    TORCH_CHECK(t.device() == q.device() && t.dtype() == torch::kInt32 && t.is_contiguous() && t.dim() == 1 && t.size(0) == n,
                "window_attention: ", what, " int32 [", n, "]");
  };
  ints(seq_start, S, "seq_start");
  ints(seq_len, S, "seq_len");
  TORCH_CHECK(tok_ctx.dim() == 1 && tok_ctx.size(0) >= T, "window_attention: tok_ctx for every token");
  ints(tok_ctx, tok_ctx.size(0), "tok_ctx");
  TORCH_CHECK(block_table.device() == q.device() && block_table.dtype() == torch::kInt32 && block_table.dim() == 2 &&
                  block_table.size(0) == S && block_table.size(1) >= 1 && block_table.is_contiguous(),
              "window_attention: block_table int32 [sequences, pages]");
  auto rows = [&](const torch::Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == q.device() && t.dtype() == torch::kBFloat16 && t.dim() == 2 && t.size(0) == T &&
                    t.size(1) == Hq * D && t.stride(1) == 1, "window_attention: ", what, " bf16 [tokens, heads * head_dim]");
  };
  rows(out, "out");
  if (gate.has_value()) rows(*gate, "gate");
  for (int64_t b : {(int64_t)(uintptr_t)q.data_ptr(), q.stride(0) * 2, (int64_t)(uintptr_t)out.data_ptr(), out.stride(0) * 2,
                    gate.has_value() ? (int64_t)(uintptr_t)gate->data_ptr() : 0, gate.has_value() ? gate->stride(0) * 2 : 0,
                    (int64_t)(uintptr_t)k_cache.data_ptr(), (int64_t)(uintptr_t)v_cache.data_ptr()})
    TORCH_CHECK(b % 16 == 0, "window_attention: rows and caches must start on 16-byte boundaries");
  TORCH_CHECK(window >= 0 && sinks >= 0 && window <= INT_MAX / 2 && sinks <= INT_MAX / 2, "window_attention: window and sinks are >= 0");
  TORCH_CHECK(max_new >= 1 && max_ctx >= 1, "window_attention: max_new and max_ctx are >= 1");
  TORCH_CHECK(status.device() == q.device() && status.dtype() == torch::kInt32 && status.numel() >= 4, "window_attention: status");
  TORCH_CHECK(T * Hq * D <= ((int64_t)1 << 40) && T <= INT_MAX && S <= 65535 && max_new <= INT_MAX && Hq <= 65535 &&
                  block_table.size(1) <= (1 << 24) && k_cache.size(0) * Hkv * wa::PAGE <= INT_MAX,
              "window_attention: sizes out of range");
  if (T == 0 || S == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  wa::Args a = {};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.ld_q = q.stride(0);
  a.k = k_cache.data_ptr<uint8_t>();
  a.v = v_cache.data_ptr<uint8_t>();
  a.table = block_table.data_ptr<int32_t>();
  a.seq_start = seq_start.data_ptr<int32_t>();
  a.seq_len = seq_len.data_ptr<int32_t>();
  a.tok_ctx = tok_ctx.data_ptr<int32_t>();
  if (gate.has_value()) {
    a.gate = reinterpret_cast<const __nv_bfloat16*>(gate->data_ptr());
    a.ld_gate = gate->stride(0);
  }
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.ld_out = out.stride(0);
  a.T = (int)T;
  a.S = (int)S;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.width = (int)block_table.size(1);
  a.pages = (int)k_cache.size(0);
  a.window = (int)window;
  a.sinks = window > 0 ? (int)sinks : 0;
  a.max_new = (int)std::min(max_new, T);
  a.scale = (float)(sm_scale * k_scale);
  a.v_scale = (float)v_scale;
  a.status = status.data_ptr<int>();
  const dim3 grid((unsigned)a.max_new, (unsigned)((Hq + 3) / 4), (unsigned)S);
  TORCH_CHECK(launch_pdl(D == 128 ? window_attn_simple_kernel<128> : window_attn_simple_kernel<256>, grid, dim3(128), 0, st,
                         a) == cudaSuccess, "window_attention launch");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace r9k
