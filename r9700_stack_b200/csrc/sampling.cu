// Token sampling from logits rows and one given uniform number a row: temperature, top-k, top-p, min-p.
//
// For a row x [V] (NaN counts as -inf) with maximum m and temperature T > 0:
//   weight  w_i = floor(2^31 exp((x_i - m) / T)), 2^31 where x_i = m, 0 where x_i = -inf;
//   order   by (x descending, index ascending), B_i = the weights before i in that order;
//   top-k   keeps the first k; P = the kept weights' sum; top-p keeps i = first or B_i < p P;
//   min-p   keeps exp((x_i - m) / T) >= min_p;
//   token   the first index (in index order) whose running sum of kept weights exceeds u * (their sum).
// T <= 0 takes the lowest index of the maximum. The weights are whole numbers of 2^-31 of the largest
// one (finer than the 2^-24 steps of the uniform number itself), so every sum is exact: the token
// depends on the row and its number alone, not on the order of additions, the batch or the launch.
//
// A row belongs to a cluster of CTAs. Each holds a slice of it in shared memory, so the logits are
// read from memory once; the CTAs exchange a few numbers a round through distributed shared memory.
// Both cuts are of the form "the smallest key B with F(keys <= B) >= target", F = count or weight.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.cuh"

namespace r9k {

namespace sm {
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 16;
constexpr float ONE = 2147483648.f;  // 2^31

struct Args {
  const void* logits;
  int64_t ld;
  int V, slice;
  const float* u;
  const float* temperature;
  const int32_t* top_k;  // or null
  const float* top_p;    // or null
  const float* min_p;    // or null
  int64_t* tokens;
  float* logprobs;
};

// one number of each CTA of the cluster, two rounds deep (a round's slots are written again two
// rounds later, when every CTA has passed the barrier after its reads)
struct Shared {
  unsigned long long slot[2];
  unsigned long long warp[WARPS];
  unsigned long long result[2];
};

R9K_DEVINL unsigned long long ld_dsmem_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

R9K_DEVINL float load_logit(const Args& a, int64_t i, float) { return reinterpret_cast<const float*>(a.logits)[i]; }
R9K_DEVINL float load_logit(const Args& a, int64_t i, __nv_bfloat16) {
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.logits)[i]);
}

// larger x -> smaller key (x is not NaN, and -0 counts as 0)
R9K_DEVINL uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}

struct Row {
  float m, inv_t, min_p;
  R9K_DEVINL float e(float x) const {
    if (x == m) return 1.f;
    if (!(x > -INFINITY)) return 0.f;
    return expf((x - m) * inv_t);
  }
  R9K_DEVINL uint32_t w(float x) const { return (uint32_t)(e(x) * ONE); }
};

enum Op { SUM, MAX };

R9K_DEVINL unsigned long long join(unsigned long long a, unsigned long long b, Op op) {
  return op == SUM ? a + b : (a > b ? a : b);
}

// The cluster's sum or maximum of v, in every thread; own: this CTA's; before: of the CTAs before it
R9K_DEVINL unsigned long long cluster_join(unsigned long long v, Op op, Shared* s, int& round, unsigned long long* before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), op);
  if (lane == 0) s->warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    unsigned long long t = lane < WARPS ? s->warp[lane] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = join(t, __shfl_xor_sync(0xffffffffu, t, o), op);
    if (lane == 0) s->slot[round & 1] = t;
  }
  cluster_sync();
  if (warp == 0) {
    const int n = (int)cluster_nctarank(), me = (int)cluster_ctarank();
    unsigned long long t = lane < n ? ld_dsmem_u64(mapa_shared(smem_u32(&s->slot[round & 1]), (uint32_t)lane)) : 0ull;
    unsigned long long b = lane < me ? t : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t = join(t, __shfl_xor_sync(0xffffffffu, t, o), op);
      b = join(b, __shfl_xor_sync(0xffffffffu, b, o), op);
    }
    if (lane == 0) { s->result[0] = t; s->result[1] = b; }
  }
  __syncthreads();
  ++round;
  const unsigned long long r = s->result[0];
  if (before != nullptr) *before = s->result[1];
  __syncthreads();
  return r;
}
}  // namespace sm

template <typename T>
__global__ void __launch_bounds__(sm::THREADS) sample_kernel(const sm::Args a) {
  using namespace sm;
  pdl_wait();
  pdl_trigger();
  extern __shared__ float xs[];  // this CTA's slice of the row
  __shared__ Shared sh;
  const int n_cta = (int)cluster_nctarank(), me = (int)cluster_ctarank();
  const int row = blockIdx.x / n_cta;
  const int tid = threadIdx.x;
  const int i0 = me * a.slice;
  const int n = max(0, min(a.V - i0, a.slice));
  int round = 0;

  // the row's maximum and its lowest index
  unsigned long long best = 0;
  for (int i = tid; i < n; i += THREADS) {
    float x = load_logit(a, (int64_t)row * a.ld + i0 + i, T());
    if (x != x) x = -INFINITY;
    xs[i] = x;
    const unsigned long long k = ((unsigned long long)~order_key(x) << 32) | (uint32_t)~(i0 + i);
    best = best > k ? best : k;
  }
  best = cluster_join(best, MAX, &sh, round, nullptr);  // its barriers make the slice visible too
  const int arg = (int)~(uint32_t)best;
  const uint32_t kmax = ~(uint32_t)(best >> 32);
  Row r;
  r.m = __uint_as_float((kmax & 0x80000000u) ? kmax : ~kmax & 0x7fffffffu);
  const float t = a.temperature[row];
  if (!(t > 0.f) || r.m == -INFINITY) {  // greedy; a row with nothing to draw from has no token
    if (me == 0 && tid == 0) {
      a.tokens[row] = r.m == -INFINITY ? -1 : arg;
      a.logprobs[row] = r.m == -INFINITY ? -INFINITY : 0.f;
    }
    cluster_sync();
    return;
  }
  r.inv_t = 1.f / t;
  r.min_p = a.min_p ? fminf(fmaxf(a.min_p[row], 0.f), 1.f) : 0.f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f;

  // last kept key of the order, as (key, index); all bits set: everything
  unsigned long long last = ~0ull;
  for (int cut = 0; cut < 2; ++cut) {
    if (cut == 0 ? !(k > 0 && k < a.V) : !(p < 1.f)) continue;
    unsigned long long target = (unsigned long long)k;
    if (cut == 1) {
      unsigned long long sum = 0;
      for (int i = tid; i < n; i += THREADS) {
        const unsigned long long key = ((unsigned long long)order_key(xs[i]) << 32) | (uint32_t)(i0 + i);
        if (key <= last) sum += r.w(xs[i]);
      }
      sum = cluster_join(sum, SUM, &sh, round, nullptr);
      // B_i < p P of whole numbers: the cut is the first key whose running sum reaches ceil(p P)
      target = (unsigned long long)max(1ll, (long long)ceil((double)p * (double)sum));
    }
    unsigned long long lo = 0;  // F(keys < lo) < target
    for (int bit = 63; bit >= 0; --bit) {
      if (bit < 32 && (1ll << bit) >= 2ll * a.V) continue;  // no index has this bit
      const unsigned long long trial = lo | (1ull << bit);
      unsigned long long f = 0;
      for (int i = tid; i < n; i += THREADS) {
        const unsigned long long key = ((unsigned long long)order_key(xs[i]) << 32) | (uint32_t)(i0 + i);
        if (key < trial && key <= last) f += cut == 0 ? 1u : r.w(xs[i]);
      }
      f = cluster_join(f, SUM, &sh, round, nullptr);
      if (f < target) lo = trial;
    }
    last = lo;
  }

  // weights of the kept tokens; the draw in index order
  unsigned long long sum = 0;
  for (int i = tid; i < n; i += THREADS) {
    const float x = xs[i];
    const unsigned long long key = ((unsigned long long)order_key(x) << 32) | (uint32_t)(i0 + i);
    if (key <= last && r.e(x) >= r.min_p) sum += r.w(x);
  }
  unsigned long long before;
  const unsigned long long total = cluster_join(sum, SUM, &sh, round, &before);
  const double at = floor((double)a.u[row] * (double)total);
  unsigned long long target = at > 0. ? (unsigned long long)at : 0ull;  // a NaN draws the first
  if (target > total - 1) target = total - 1;
  // running sums of 512 indexes at a time
  unsigned long long base = before;
  for (int c = 0; c < n; c += THREADS) {
    const int i = c + tid;
    uint32_t w = 0;
    if (i < n) {
      const float x = xs[i];
      const unsigned long long key = ((unsigned long long)order_key(x) << 32) | (uint32_t)(i0 + i);
      if (key <= last && r.e(x) >= r.min_p) w = r.w(x);
    }
    const int lane = tid & 31, warp = tid >> 5;
    unsigned long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sh.warp[warp] = inc;
    __syncthreads();
    unsigned long long pre = base, all = 0;
    for (int j = 0; j < WARPS; ++j) {
      if (j < warp) pre += sh.warp[j];
      all += sh.warp[j];
    }
    if (w > 0 && pre + inc - w <= target && target < pre + inc) {
      a.tokens[row] = i0 + i;
      a.logprobs[row] = (float)log((double)w / (double)total);
    }
    base += all;
    __syncthreads();
    if (base > target) break;
  }
  cluster_sync();  // peers may still read this CTA's slots
}

void sample_logits(torch::Tensor logits, torch::Tensor u, torch::Tensor temperature, c10::optional<torch::Tensor> top_k,
                   c10::optional<torch::Tensor> top_p, c10::optional<torch::Tensor> min_p, torch::Tensor tokens,
                   torch::Tensor logprobs) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1 && logits.stride(1) == 1,
              "sample_logits: logits [rows, vocabulary] on a GPU, a row's entries next to each other");
  TORCH_CHECK(logits.dtype() == torch::kFloat32 || logits.dtype() == torch::kBFloat16, "sample_logits: fp32 or bf16 logits");
  const int64_t R = logits.size(0), V = logits.size(1);
  auto chk = [&](const torch::Tensor& t, torch::ScalarType ty, const char* what) {
    TORCH_CHECK(t.device() == logits.device() && t.dtype() == ty && t.dim() == 1 && t.size(0) == R && t.is_contiguous(),
                "sample_logits: ", what, " must hold one ", ty, " a row on the logits' device");
  };
  chk(u, torch::kFloat32, "u");
  chk(temperature, torch::kFloat32, "temperature");
  if (top_k.has_value()) chk(*top_k, torch::kInt32, "top_k");
  if (top_p.has_value()) chk(*top_p, torch::kFloat32, "top_p");
  if (min_p.has_value()) chk(*min_p, torch::kFloat32, "min_p");
  chk(tokens, torch::kInt64, "tokens");
  chk(logprobs, torch::kFloat32, "logprobs");
  constexpr int MAX_SLICE = 55 * 1024;  // floats of shared memory
  TORCH_CHECK(V <= (int64_t)sm::MAX_CLUSTER * MAX_SLICE, "sample_logits: vocabulary too large");
  if (R == 0) return;
  const at::cuda::CUDAGuard guard(logits.device());
  int C = 1;
  while (C < sm::MAX_CLUSTER && (V + C - 1) / C > 16384) C *= 2;
  TORCH_CHECK(R * C <= INT_MAX, "sample_logits: too many rows");
  sm::Args a{logits.data_ptr(), logits.stride(0), (int)V, (int)((V + C - 1) / C), u.data_ptr<float>(),
             temperature.data_ptr<float>(), top_k.has_value() ? top_k->data_ptr<int32_t>() : nullptr,
             top_p.has_value() ? top_p->data_ptr<float>() : nullptr,
             min_p.has_value() ? min_p->data_ptr<float>() : nullptr, tokens.data_ptr<int64_t>(),
             logprobs.data_ptr<float>()};
  auto kern = logits.dtype() == torch::kFloat32 ? sample_kernel<float> : sample_kernel<__nv_bfloat16>;
  TORCH_CHECK(ensure_smem_attr((const void*)kern, MAX_SLICE * 4) == cudaSuccess, "sample_logits: shared memory attribute");
  TORCH_CHECK(cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess,
              "sample_logits: cluster attribute");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * C));
  cfg.blockDim = dim3(sm::THREADS);
  cfg.dynamicSmemBytes = (size_t)a.slice * 4;
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)C, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TORCH_CHECK(cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess, "sample_logits launch");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace r9k
