// The plan of a serving step, made on the device from request lengths (no host round trip).
//
// Inputs: tokens to run now for every request (new_len [S]) and the state of the paged cache:
//   state = {ring head, free pages, cached tokens [S], first live page [S]}, the page tables
//   block_table [S, width] and a ring of free page numbers. A page holds 64 tokens.
// With c = cached tokens and n = new tokens of request r, in request order:
//   fits:    n > 0, c + n <= 64 * width, and the tokens of all fitting requests up to r are <= cap;
//   need:    ceil((c + n) / 64) - ceil(c / 64) pages, taken from the ring's head;
//   served:  fits, and need = 0 or the needs of all fitting requests up to r are <= the free pages;
//   back:    with a window W, pages of a served request in [max(first live, ceil(sinks / 64)),
//            floor((c - W + 1) / 64)): the oldest new token (position c) sees keys > c - W only, so
//            nothing will read them again. They go to the ring's tail, for the steps after this one.
// Outputs per token slot (cap of them; the unused ones are padding): position, KV slot (-1), request,
// context (position + 1; 0); per request: first token, tokens; and the state after the step.
//
// The step is a transaction: block_table and ring are only written where the old state does not look
// (pages past the cached ones, ring entries past the tail), with values that depend on the inputs
// alone, and the new state goes to the outputs. Planning again from the same state gives the same
// step; the caller commits it by taking the new state.
//
// Every quantity is a prefix sum over the requests. Each block makes them for itself (a few hundred
// integers, cheaper than a second launch), then the blocks share the tokens and the pages that move,
// one item a thread, each found by bisecting the sums in shared memory. What bounds it is latency:
// launch, one dependent read (lengths), the sums, one more dependent read (table or ring entry). On the
// device 2.9 us for one request, 4.7 us for 256 requests, 5.1 us for 8192 tokens; a call from Python 10 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <climits>
#include "common.cuh"

namespace r9k {

namespace sp {
constexpr int PAGE = 64;
constexpr int MAX_SEQS = 4096;
constexpr int MAX_TOKENS = 1 << 18;
constexpr int MAX_WIDTH = 1 << 18;

struct Args {
  const int32_t* new_len;
  const int32_t* state;
  int32_t* table;
  int32_t* ring;
  int32_t* out;
  int S, width, ring_len, cap, window, sinks;
};

// exclusive sums of three values over the block; tot: the block's totals
R9K_DEVINL void block_scan3(int (&v)[3], int (&tot)[3], int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int in[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) in[k] = v[k];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int x = __shfl_up_sync(0xffffffffu, in[k], o);
      if (lane >= o) in[k] += x;
    }
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < 3; ++k) scratch[k * 32 + warp] = in[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int s = lane < warps ? scratch[k * 32 + lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += x;
    }
    tot[k] = __shfl_sync(0xffffffffu, s, 31);
    const int before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
    v[k] = in[k] - v[k] + (warp > 0 ? before : 0);
  }
  __syncthreads();  // scratch is free again
}

// the request whose [first[r], first[r + 1]) holds i; first[S] > i
R9K_DEVINL int holder(const int32_t* first, int S, int i) {
  int lo = 0, hi = S;  // first[lo] <= i < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

R9K_DEVINL int pages_of(int tokens) { return (tokens + PAGE - 1) / PAGE; }
}  // namespace sp

__global__ void step_plan_kernel(const sp::Args a) {
  using namespace sp;
  pdl_wait();
  pdl_trigger();
  extern __shared__ int32_t smem[];
  const int S = a.S;
  int32_t* tok0 = smem;             // [S + 1] first token of each request (sums of served tokens)
  int32_t* need0 = tok0 + S + 1;    // [S + 1] sums of served needs
  int32_t* back0 = need0 + S + 1;   // [S + 1] sums of pages given back
  int32_t* ctx = back0 + S + 1;     // [S]
  int32_t* from = ctx + S;          // [S] first page to give back
  int32_t* ok = from + S;           // [S] served
  int32_t* scratch = ok + S;        // [96]
  const int tid = threadIdx.x, nt = blockDim.x;
  const int N = a.ring_len;
  int head = a.state[0] % N;
  if (head < 0) head += N;
  const int avail = min(max(a.state[1], 0), N);
  const int low = pages_of(a.sinks);

  // One pass gives all sums when every request that fits its table also fits the step; where tokens
  // or pages run out, two more passes narrow the served requests down (fits, then served) first.
  for (int pass = 0; pass < 4; ++pass) {
    int carry[3] = {0, 0, 0};
    for (int base = 0; base < S; base += nt) {
      const int r = base + tid;
      int v[3] = {0, 0, 0}, tot[3];
      int mine = 0, c = 0, f = 0;
      if (r < S) {
        c = a.state[2 + r];
        const int n = a.new_len[r];
        if (pass == 0) mine = n > 0 && c >= 0 && (int64_t)c + n <= (int64_t)a.width * PAGE;
        else mine = ok[r];
        if (mine) {
          f = max(max(a.state[2 + S + r], 0), low);
          const int to = a.window > 0 ? max(0, c - a.window + 1) / PAGE : 0;
          v[0] = min(n, a.cap + 1);  // a request over the budget stops the line, and the sum stays small
          v[1] = pages_of(c + n) - pages_of(c);
          v[2] = max(0, to - f);
        }
      }
      const int n1 = v[0], p1 = v[1];
      block_scan3(v, tot, scratch);
      if (r < S) {
        if (pass == 0) { ctx[r] = c; from[r] = f; ok[r] = mine; }
        if (pass == 1) ok[r] = mine && carry[0] + v[0] + n1 <= a.cap;
        if (pass == 2) ok[r] = mine && (p1 == 0 || carry[1] + v[1] + p1 <= avail);
        tok0[r] = carry[0] + v[0];
        need0[r] = carry[1] + v[1];
        back0[r] = carry[2] + v[2];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) carry[k] += tot[k];
    }
    if (tid == 0) { tok0[S] = carry[0]; need0[S] = carry[1]; back0[S] = carry[2]; }
    __syncthreads();
    if (pass == 0 && carry[0] <= a.cap && carry[1] <= avail) break;
  }

  const int total = tok0[S], taken = need0[S], back = back0[S];
  const int cap = a.cap;
  int32_t* positions = a.out;
  int32_t* slots = positions + cap;
  int32_t* tok_seq = slots + cap;
  int32_t* tok_ctx = tok_seq + cap;
  int32_t* seq_start = tok_ctx + cap;
  int32_t* seq_len = seq_start + S;
  int32_t* state = seq_len + S;
  const int gtid = blockIdx.x * nt + tid, gnt = gridDim.x * nt;

  for (int t = gtid; t < cap; t += gnt) {
    int pos = 0, slot = -1, r = 0, c1 = 0;
    if (t < total) {
      r = holder(tok0, S, t);
      const int c = ctx[r];
      pos = c + t - tok0[r];
      const int p = pos / PAGE, have = pages_of(c);
      int page;
      if (p < have) page = a.table[(int64_t)r * a.width + p];
      else page = a.ring[(head + need0[r] + p - have) % N];
      slot = page * PAGE + pos % PAGE;
      c1 = pos + 1;
    }
    positions[t] = pos;
    slots[t] = slot;
    tok_seq[t] = r;
    tok_ctx[t] = c1;
  }
  for (int i = gtid; i < taken; i += gnt) {
    const int r = holder(need0, S, i);
    a.table[(int64_t)r * a.width + pages_of(ctx[r]) + i - need0[r]] = a.ring[(head + i) % N];
  }
  for (int i = gtid; i < back; i += gnt) {
    const int r = holder(back0, S, i);
    a.ring[(int)(((int64_t)head + avail + i) % N)] = a.table[(int64_t)r * a.width + from[r] + i - back0[r]];
  }
  for (int r = gtid; r < S; r += gnt) {
    const int n = tok0[r + 1] - tok0[r];
    const int to = n > 0 && a.window > 0 ? max(0, ctx[r] - a.window + 1) / PAGE : 0;
    seq_start[r] = tok0[r];
    seq_len[r] = n;
    state[2 + r] = ctx[r] + n;
    state[2 + S + r] = max(a.state[2 + S + r], to);
  }
  if (gtid == 0) {
    state[0] = (head + taken) % N;
    state[1] = avail - taken + back;
  }
}

void plan_step(torch::Tensor new_len, torch::Tensor state, torch::Tensor block_table, torch::Tensor ring, int64_t cap,
               int64_t window, int64_t sinks, torch::Tensor out) {
  const int64_t S = new_len.numel();
  for (const torch::Tensor* t : {&new_len, &state, &block_table, &ring, &out})
    TORCH_CHECK(t->is_cuda() && t->device() == new_len.device() && t->dtype() == torch::kInt32 && t->is_contiguous(),
                "plan_step: contiguous int32 tensors on one device");
  TORCH_CHECK(new_len.dim() == 1 && S >= 1 && S <= sp::MAX_SEQS, "plan_step: new_len [1..", sp::MAX_SEQS, "]");
  TORCH_CHECK(state.numel() == 2 + 2 * S, "plan_step: state holds 2 + 2 * requests numbers");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == S && block_table.size(1) >= 1 &&
                  block_table.size(1) <= sp::MAX_WIDTH, "plan_step: block_table [requests, pages]");
  TORCH_CHECK(ring.numel() >= 1 && ring.numel() <= (1 << 25), "plan_step: ring of 1..2^25 pages");  // slots fit int32
  TORCH_CHECK(cap >= 1 && cap <= sp::MAX_TOKENS, "plan_step: token capacity 1..", sp::MAX_TOKENS);
  TORCH_CHECK(window >= 0 && window <= INT_MAX && sinks >= 0 && sinks <= INT_MAX - 64, "plan_step: window and sinks are >= 0");
  TORCH_CHECK(out.numel() == 4 * cap + 4 * S + 2, "plan_step: out holds 4 * cap + 4 * requests + 2 numbers");
  TORCH_CHECK(state.data_ptr<int32_t>() + state.numel() <= out.data_ptr<int32_t>() ||
                  out.data_ptr<int32_t>() + out.numel() <= state.data_ptr<int32_t>(), "plan_step: out overlaps state");
  const at::cuda::CUDAGuard guard(new_len.device());
  const int smem = (int)(6 * S + 3 + 96) * 4;
  TORCH_CHECK(ensure_smem_attr((const void*)step_plan_kernel, (6 * sp::MAX_SEQS + 99) * 4) == cudaSuccess,
              "plan_step: shared memory attribute");
  const int64_t items = std::max(S, cap);
  const int threads = (int)std::min<int64_t>(1024, (items + 31) / 32 * 32);
  const int blocks = (int)std::min<int64_t>(64, (cap + threads - 1) / threads);
  sp::Args a{new_len.data_ptr<int32_t>(), state.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(),
             ring.data_ptr<int32_t>(), out.data_ptr<int32_t>(), (int)S, (int)block_table.size(1), (int)ring.numel(),
             (int)cap, (int)window, (int)sinks};
  TORCH_CHECK(launch_pdl(step_plan_kernel, dim3(blocks), dim3(threads), (size_t)smem, at::cuda::getCurrentCUDAStream(),
                         a) == cudaSuccess, "plan_step launch");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace r9k
