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
// A row belongs to a cluster of CTAs; each has a slice of it, held in shared memory or read again from L2. Both
// cuts look for "the smallest key B with F(keys <= B) >= target", F = count or weight, keys ordered as above:
//   * a histogram of (m - x) / T over 1024 bins a CTA (shared-memory atomics on whole numbers), summed by
//     the cluster's first CTA, gives the bin in which F crosses the target. Top-k first tries the
//     threads' maxima alone: at least k keys lie at or before the k-th of them, and hardly more than k
//     where k is well below the number of threads, so one atomic a thread does instead of one a key;
//   * if all keys up to that bin are few (top-k and most nuclei), they go to the first CTA, which sorts
//     them, applies all three filters and draws; the other CTAs are done;
//   * else the crossing bin's keys are sorted there (after a second, 1024 times finer histogram if they
//     are many; bit by bit over the cluster if thousands tie), and the cut key goes back to all CTAs,
//     which sum and draw over their slices.
//
// What bounds it: for few rows the chain of exchanges (a cluster barrier and a remote read are about 1 us
// each; one row of 248320 fp32: 13.8 us, of which 3 us load it); for many rows the second read and the
// exchanges of rows that share an SM (256 rows: 120 us, the first read alone 39 us at copy bandwidth); for
// wide nuclei the histogram's three atomics a key (64 x 100003 bf16: 52 us). Rows whose cut falls on more than
// CAP equal logits pay for the search bit by bit: rows of one value, top-p 0.9, take 300 us (one of 248320 fp32; 49 with
// normal logits), 740 us (16; 90) and 4.3 ms (256; 460).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <climits>
#include <type_traits>
#include "common.cuh"

namespace r9k {

namespace sm {
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 16;
constexpr int BINS = 2 * THREADS;
constexpr int CAP = 2 * THREADS;         // keys that one CTA sorts: two a thread
constexpr float ONE = 2147483648.f;      // 2^31
constexpr float REACH = 21.6f;           // exp(-z) 2^31 < 1 beyond: no weight
constexpr int WORK_BYTES = 3 * BINS * 4;  // histograms (count, low and high half of the weights), or the list
static_assert(CAP * 8 <= WORK_BYTES, "the list lies over the histograms");

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

using u64 = unsigned long long;

enum Op { SUM, MAX };
enum Action { DONE, FINISH, CUT, REFINE, BITS, KEYS };

struct Verdict {  // of the first CTA, sent to all
  u64 target, before;
  int action, bin;
};

struct Shared {
  u64 slot[2][MAX_CLUSTER];  // one number of each CTA, two rounds deep
  u64 warp[WARPS];
  u64 warp2[WARPS];
  u64 last;
  Verdict verdict;
  uint32_t listed;
};

R9K_DEVINL void st_dsmem(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
R9K_DEVINL uint2 ld_dsmem_u2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
R9K_DEVINL uint32_t ld_dsmem_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
R9K_DEVINL uint32_t add_dsmem(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}
R9K_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
R9K_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// larger x -> smaller key (x is not NaN, and -0 counts as 0)
R9K_DEVINL uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}
R9K_DEVINL float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu); }
R9K_DEVINL u64 full_key(float x, int i) { return ((u64)order_key(x) << 32) | (uint32_t)i; }

struct Row {
  float m, inv_t, min_p, p, bins;  // bins: histogram bins of one unit of (m - x) / T
  int k;
  R9K_DEVINL float e(float x) const {
    if (x == m) return 1.f;
    if (!(x > -INFINITY)) return 0.f;
    return expf((x - m) * inv_t);
  }
  R9K_DEVINL uint32_t w(float x) const { return (uint32_t)(e(x) * ONE); }
  // place in the histogram, ascending in the order of keys; >= BINS: no weight (NaN does not compare).
  // Every use has to round alike, so the products are not to be fused with what follows.
  R9K_DEVINL float place(float x) const { return x == m ? 0.f : __fmul_rn(__fmul_rn(m - x, inv_t), bins); }
};

R9K_DEVINL u64 join(u64 a, u64 b, Op op) { return op == SUM ? a + b : (a > b ? a : b); }

// The cluster's sum or maximum of v, in every thread; before: the sum over the CTAs before this one.
// Every CTA writes its number to all others; a round's slots are written again two rounds later, after
// a barrier that comes after everybody's reads.
R9K_DEVINL u64 cluster_join(u64 v, Op op, Shared* s, int& round, u64* before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = (int)cluster_nctarank(), me = (int)cluster_ctarank();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), op);
  if (lane == 0) s->warp[warp] = v;
  __syncthreads();
  u64* slot = s->slot[round & 1];
  if (warp == 0) {
    u64 t = lane < WARPS ? s->warp[lane] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = join(t, __shfl_xor_sync(0xffffffffu, t, o), op);
    if (lane < n) st_dsmem(mapa_shared(smem_u32(&slot[me]), (uint32_t)lane), t);
  }
  cluster_sync();
  u64 t = 0, b = 0;
  for (int i = 0; i < n; ++i) {
    if (i == me) b = t;
    t = join(t, slot[i], op);
  }
  ++round;
  if (before != nullptr) *before = b;
  return t;
}

// the cluster's maxima of two 32-bit numbers at once
R9K_DEVINL uint2 cluster_max2(uint32_t x, uint32_t y, Shared* s, int& round) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = (int)cluster_nctarank(), me = (int)cluster_ctarank();
  x = __reduce_max_sync(0xffffffffu, x);
  y = __reduce_max_sync(0xffffffffu, y);
  if (lane == 0) s->warp[warp] = ((u64)x << 32) | y;
  __syncthreads();
  u64* slot = s->slot[round & 1];
  if (warp == 0) {
    const u64 t = lane < WARPS ? s->warp[lane] : 0ull;
    x = __reduce_max_sync(0xffffffffu, (uint32_t)(t >> 32));
    y = __reduce_max_sync(0xffffffffu, (uint32_t)t);
    if (lane < n) st_dsmem(mapa_shared(smem_u32(&slot[me]), (uint32_t)lane), ((u64)x << 32) | y);
  }
  cluster_sync();
  const u64 t = lane < n ? slot[lane] : 0ull;
  ++round;
  return make_uint2(__reduce_max_sync(0xffffffffu, (uint32_t)(t >> 32)), __reduce_max_sync(0xffffffffu, (uint32_t)t));
}

// inclusive sums over the block; total: of all threads
R9K_DEVINL u64 block_scan(u64 v, u64* scratch, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  u64 t = lane < WARPS ? scratch[lane] : 0ull;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += x;
  }
  *total = __shfl_sync(0xffffffffu, t, 31);
  const u64 pre = __shfl_sync(0xffffffffu, t, (warp + 31) & 31);
  __syncthreads();
  return v + (warp > 0 ? pre : 0ull);
}

// Ascending sort of two numbers a thread (places t and t + THREADS) of which the first n matter; the
// others are ~0. Neighbours nearer than a warp exchange by shuffles, further ones through buf [CAP].
R9K_DEVINL void block_sort(u64 (&v)[2], int n, u64* buf) {
  const int t = threadIdx.x;
  const bool two = n > THREADS;
  for (int size = 2; size < 2 * n; size <<= 1) {
    for (int j = size >> 1; j > 0; j >>= 1) {
      if (j == THREADS) {
        const u64 a = v[0], b = v[1];
        v[0] = a < b ? a : b;
        v[1] = a < b ? b : a;
        continue;
      }
      u64 o[2] = {~0ull, ~0ull};
      if (j >= 32) {
        buf[t] = v[0];
        if (two) buf[t + THREADS] = v[1];
        __syncthreads();
        o[0] = buf[t ^ j];
        if (two) o[1] = buf[(t ^ j) + THREADS];
        __syncthreads();
      } else {
        o[0] = __shfl_xor_sync(0xffffffffu, v[0], j);
        if (two) o[1] = __shfl_xor_sync(0xffffffffu, v[1], j);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = t + i * THREADS;
        const bool low = ((at & j) == 0) == ((at & size) == 0);
        v[i] = low == (v[i] < o[i]) ? v[i] : o[i];
      }
    }
  }
}

template <typename T>
R9K_DEVINL float as_logit(T v);
template <>
R9K_DEVINL float as_logit(float v) { return v != v ? -INFINITY : v; }
template <>
R9K_DEVINL float as_logit(__nv_bfloat16 v) { return as_logit(__bfloat162float(v)); }

// entries before the first 16-byte boundary of a slice
template <typename T>
R9K_DEVINL int lead(const T* src) { return (int)(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T)); }

// The part of a slice's 16-byte loads that a warp takes: neighbouring ones, so that the warps' sums are in
// index order (the entries before the first boundary go to the first warp, those after the last to the last).
struct Share {
  int lo, hi;
  R9K_DEVINL Share(int vecs, int warp) {
    const int per = (vecs + WARPS - 1) / WARPS;
    lo = min(vecs, warp * per);
    hi = min(vecs, lo + per);
  }
};

// Every logit i < n of a slice in global or shared memory, a thread each: four(x, i) for four at a time
// from the first 16-byte boundary on (four loads in flight), one(x, i) for those around them.
template <typename T, typename F1, typename F4>
R9K_DEVINL void scan(const T* src, int n, F1 one, F4 four) {
  constexpr int VEC = 16 / sizeof(T);
  const int head = min(n, lead(src));
  const int vecs = (n - head) / VEC, rest = head + vecs * VEC;
  const uint4* body = reinterpret_cast<const uint4*>(src + head);
  auto each = [&](uint4 raw, int v) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float x[4] = {as_logit(e[i]), as_logit(e[i + 1]), as_logit(e[i + 2]), as_logit(e[i + 3])};
      four(x, head + v * VEC + i);
    }
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Share mine(vecs, warp);
  int v = mine.lo + lane;
  for (; v + 96 < mine.hi; v += 128) {
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = body[v + 32 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j) each(raw[j], v + 32 * j);
  }
  for (; v < mine.hi; v += 32) each(body[v], v);
  if (warp == 0 && lane < head) one(as_logit(src[lane]), lane);
  if (warp == WARPS - 1 && lane < n - rest) one(as_logit(src[rest + lane]), rest + lane);
}
template <typename T, typename F>
R9K_DEVINL void scan(const T* src, int n, F f) {
  scan(src, n, f, [&](const float (&x)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f(x[j], i + j);
  });
}

// Ascending sort of 32 * E numbers of one warp, number i of lane l at place i * 32 + l.
template <int E>
R9K_DEVINL void warp_sort(u64 (&v)[E]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32 * E; size <<= 1) {
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) {
      if (j >= 32) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int o = i ^ (j >> 5);
          if (o > i) {
            const bool up = ((i * 32) & size) == 0;
            const u64 x = v[i], y = v[o];
            const bool swap = (x > y) == up;
            v[i] = swap ? y : x;
            v[o] = swap ? x : y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const u64 o = __shfl_xor_sync(0xffffffffu, v[i], j);
          const bool low = ((lane & j) == 0) == (((i * 32 + lane) & size) == 0);
          v[i] = low == (v[i] < o) ? v[i] : o;
        }
      }
    }
  }
}
template <int E>
R9K_DEVINL u64 warp_scan(const u64 (&w)[E], u64 (&upto)[E]) {  // inclusive; returns the total
  const int lane = threadIdx.x & 31;
  u64 total = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    u64 v = w[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    upto[i] = total + v;
    total += __shfl_sync(0xffffffffu, v, 31);
  }
  return total;
}

// finish_list() for up to 32 * E keys by one warp, without a barrier
template <int E>
R9K_DEVINL void finish_short(const Args& a, const Row& r, int row, int n, u64 all, const u64* list) {
  const int lane = threadIdx.x & 31;
  u64 v[E], w[E], upto[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = i * 32 + lane < n ? list[i * 32 + lane] : ~0ull;
  warp_sort<E>(v);
  const int k = r.k > 0 ? min(r.k, n) : n;
#pragma unroll
  for (int i = 0; i < E; ++i) w[i] = i * 32 + lane < k ? r.w(key_value((uint32_t)(v[i] >> 32))) : 0ull;
  u64 total = warp_scan<E>(w, upto);
  if (all == 0) all = total;
  const double enough = (double)r.p * (double)all;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int at = i * 32 + lane;
    const bool keep = at < k && (at == 0 || !(r.p < 1.f) || (double)(upto[i] - w[i]) < enough) &&
                      r.e(key_value((uint32_t)(v[i] >> 32))) >= r.min_p;
    v[i] = keep ? (v[i] << 32) | w[i] : ~0ull;  // now by index
  }
  warp_sort<E>(v);
#pragma unroll
  for (int i = 0; i < E; ++i) w[i] = v[i] == ~0ull ? 0ull : (uint32_t)v[i];
  total = warp_scan<E>(w, upto);
  const double at = floor((double)a.u[row] * (double)total);
  u64 target = at > 0. ? (u64)at : 0ull;
  if (target > total - 1) target = total - 1;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (upto[i] - w[i] <= target && target < upto[i]) {
      a.tokens[row] = (int64_t)(v[i] >> 32);
      a.logprobs[row] = (float)log((double)w[i] / (double)total);
    }
}

// The first CTA's last step: the keys up to the cut, sorted; all filters; the draw in index order.
// all: the weight that top-p is a share of (0: that of the first k keys).
R9K_DEVINL void finish_list(const Args& a, const Row& r, int row, int n, u64 all, u64* list, Shared* s) {
  const int t = threadIdx.x;
  u64 v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = t + i * THREADS < n ? list[t + i * THREADS] : ~0ull;
  __syncthreads();
  block_sort(v, n, list);
  const int k = r.k > 0 ? min(r.k, n) : n;
  u64 w[2], upto[2], total = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = t + i * THREADS < k ? r.w(key_value((uint32_t)(v[i] >> 32))) : 0ull;
    u64 part;
    upto[i] = total + block_scan(w[i], s->warp, &part);
    total += part;
  }
  if (all == 0) all = total;
  const double enough = (double)r.p * (double)all;
  int kept = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = t + i * THREADS;
    const bool keep = at < k && (at == 0 || !(r.p < 1.f) || (double)(upto[i] - w[i]) < enough) &&
                      r.e(key_value((uint32_t)(v[i] >> 32))) >= r.min_p;
    kept += keep;
    v[i] = keep ? (v[i] << 32) | w[i] : ~0ull;  // now by index
  }
  // the kept keys are the first ones: how many
  u64 count;
  block_scan((u64)kept, s->warp, &count);
  block_sort(v, (int)count, list);
  total = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = v[i] == ~0ull ? 0ull : (uint32_t)v[i];
    u64 part;
    upto[i] = total + block_scan(w[i], s->warp, &part);
    total += part;
  }
  const double at = floor((double)a.u[row] * (double)total);
  u64 target = at > 0. ? (u64)at : 0ull;  // a NaN draws the first
  if (target > total - 1) target = total - 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (upto[i] - w[i] <= target && target < upto[i]) {
      a.tokens[row] = (int64_t)(v[i] >> 32);
      a.logprobs[row] = (float)log((double)w[i] / (double)total);
    }
}
}  // namespace sm

// HELD: the slice is kept in shared memory as fp32; else it is read again (from L2) by each pass
template <typename T, bool HELD>
__global__ void __launch_bounds__(sm::THREADS, 2) sample_kernel(const sm::Args a) {
  using namespace sm;
  using U = std::conditional_t<HELD, float, T>;
  pdl_wait();
  pdl_trigger();
  cluster_arrive();  // every CTA runs before its shared memory is written to (waited for below)
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  uint32_t* count = reinterpret_cast<uint32_t*>(smem);  // histograms
  uint32_t* wlow = count + BINS;
  uint32_t* whigh = wlow + BINS;
  u64* list = reinterpret_cast<u64*>(smem);  // the first CTA's, after the histograms
  const int n_cta = (int)cluster_nctarank(), me = (int)cluster_ctarank();
  const int row = blockIdx.x / n_cta;
  const int tid = threadIdx.x;
  const int i0 = me * a.slice;
  const int n = max(0, min(a.V - i0, a.slice));
  int round = 0;
  const float t = a.temperature[row];
  const float min_p = a.min_p ? a.min_p[row] : 0.f, top_p = a.top_p ? a.top_p[row] : 1.f;
  const int top_k = a.top_k ? a.top_k[row] : 0;

  float hi = -INFINITY, lo = INFINITY;
  auto see = [&](float x) {
    hi = fmaxf(hi, x);
    if (x > -INFINITY) lo = fminf(lo, x);
  };
  const T* src = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ld + i0;
  const U* xs;
  if constexpr (HELD) {
    // shifted so that the slice's 16-byte boundaries stay such
    float* buf = reinterpret_cast<float*>(smem + WORK_BYTES) + ((4 - (lead(src) & 3)) & 3);
    scan(src, n,
         [&](float x, int i) {
           see(x);
           buf[i] = x;
         },
         [&](const float (&x)[4], int i) {
#pragma unroll
           for (int j = 0; j < 4; ++j) see(x[j]);
           *reinterpret_cast<float4*>(buf + i) = make_float4(x[0], x[1], x[2], x[3]);
         });
    xs = buf;
  } else {
    scan(src, n, [&](float x, int) { see(x); });
    xs = src;
  }
  cluster_wait();
  // ~key ascends with the value, a key descends: the largest and the smallest value
  const uint2 ends = cluster_max2(~order_key(hi), lo < INFINITY ? order_key(lo) : 0u, &sh, round);
  Row r;
  r.m = key_value(~ends.x);
  if (r.m == -INFINITY) {  // nothing to draw from
    if (me == 0 && tid == 0) {
      a.tokens[row] = -1;
      a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (!(t > 0.f)) {
    uint32_t best = 0;  // ~index
    scan(xs, n, [&](float x, int i) {
      if (x == r.m) best = max(best, ~(uint32_t)(i0 + i));
    });
    const u64 first = cluster_join((u64)best, MAX, &sh, round, nullptr);
    if (me == 0 && tid == 0) {
      a.tokens[row] = (int64_t)(uint32_t)~(uint32_t)first;
      a.logprobs[row] = 0.f;
    }
    return;
  }
  r.inv_t = 1.f / t;
  r.min_p = fminf(fmaxf(min_p, 0.f), 1.f);
  r.k = top_k > 0 && top_k < a.V ? top_k : 0;
  r.p = top_p < 1.f ? top_p : 1.f;
  const bool cuts[2] = {r.k > 0, r.p < 1.f};

  u64 last = ~0ull;  // last kept key
  if (cuts[0] || cuts[1]) {
    // bins over what the row spans, where that is less than the weights' reach (high temperatures)
    const float span = fminf(REACH, (r.m - key_value(ends.y)) * r.inv_t * 1.001f);
    r.bins = span > 1e-6f ? (float)BINS / span : (float)BINS * 1e6f;  // infinities: span = REACH
  }
  for (int cut = 0; cut < 2; ++cut) {
    if (!cuts[cut]) continue;
    float cell = 0.f, fine = 1.f;  // the histogram covers places [cell, cell + BINS / fine)
    u64 target = (u64)r.k, before = 0;
    bool maxima = cut == 0 && r.k <= THREADS * n_cta / 4;  // 1.15 k keys expected at most
    for (int level = 0;; ++level) {
      for (int i = tid; i < (cut == 0 ? BINS : 3 * BINS); i += THREADS) count[i] = 0;
      if (tid == 0) sh.listed = 0;
      __syncthreads();
      if (maxima) {
        const float at = r.place(hi);
        if (at < (float)BINS) atomicAdd(&count[(int)at], 1u);
      }
      else
        scan(xs, n, [&](float x, int i) {
          const float at = (r.place(x) - cell) * fine;
          if (at >= 0.f && at < (float)BINS && full_key(x, i0 + i) <= last) {
            const int bin = (int)at;
            atomicAdd(&count[bin], 1u);
            if (cut == 1) {  // 2^31 a weight, fewer than 2^16 weights a CTA: the halves' sums fit 32 bits
              const uint32_t w = r.w(x);
              if (w & 0xffffu) atomicAdd(&wlow[bin], w & 0xffffu);
              if (w >> 16) atomicAdd(&whigh[bin], w >> 16);
            }
          }
        });
      cluster_sync();
      if (me == 0) {
        u64 c[2] = {0, 0}, f[2] = {0, 0};  // this thread's two bins
#pragma unroll 4
        for (int i = 0; i < n_cta; ++i) {
          const uint32_t at = mapa_shared(smem_u32(&count[2 * tid]), (uint32_t)i);
          const uint2 v = ld_dsmem_u2(at);
          c[0] += v.x;
          c[1] += v.y;
          if (cut == 1) {
            const uint2 l = ld_dsmem_u2(at + BINS * 4), h = ld_dsmem_u2(at + 2 * BINS * 4);
            f[0] += ((u64)h.x << 16) + l.x;
            f[1] += ((u64)h.y << 16) + l.y;
          }
        }
        if (cut == 0) {
          f[0] = c[0];
          f[1] = c[1];
        }
        u64 all, keys;
        const u64 upto = block_scan(f[0] + f[1], sh.warp, &all);
        const u64 cupto = block_scan(c[0] + c[1], sh.warp2, &keys);
        if (level == 0 && cut == 1) target = (u64)max(1ll, (long long)ceil((double)r.p * (double)all));
        // no crossing: fewer than k keys have weight (or fewer than k maxima)
        if (tid == 0) sh.verdict = Verdict{target, 0, maxima ? KEYS : keys <= CAP ? FINISH : DONE, BINS - 1};
        __syncthreads();
        const u64 want = target - before;
        const u64 b0 = upto - f[0] - f[1], b1 = upto - f[1];
        const int hit = b0 < want && want <= b1 ? 0 : b1 < want && want <= upto ? 1 : -1;
        if (hit >= 0) {
          const u64 through = cupto - (hit == 0 ? c[1] : 0ull);  // keys up to and with the bin
          Verdict v{target, before + (hit == 0 ? b0 : b1), BITS, 2 * tid + hit};
          if (level == 0 && through <= CAP) v.action = FINISH;
          else if (maxima) v.action = KEYS;
          else if (c[hit] <= CAP) v.action = CUT;
          else if (level == 0) v.action = REFINE;
          sh.verdict = v;
        }
        __syncthreads();
        if (tid == 0 && level == 0 && cut == 1) sh.last = all;
        if (tid > 0 && tid < n_cta) {
          const u64* from = reinterpret_cast<const u64*>(&sh.verdict);
#pragma unroll
          for (int i = 0; i < (int)(sizeof(Verdict) / 8); ++i)
            st_dsmem(mapa_shared(smem_u32(&sh.verdict), (uint32_t)tid) + 8 * i, from[i]);
        }
      }
      cluster_sync();
      const Verdict v = sh.verdict;
      target = v.target;
      before = v.before;
      if (v.action == DONE) break;
      if (v.action == KEYS) {
        maxima = false;
        before = 0;
        --level;
        continue;
      }
      if (v.action == REFINE) {
        cell = (float)v.bin;
        fine = (float)BINS;
        continue;
      }
      // the crossing bin in places: [from, to)
      const float from = cell + (float)v.bin / fine, to = cell + (float)(v.bin + 1) / fine;
      if (v.action == BITS) {
        u64 low = 0;  // F(keys < low) < target
        for (int bit = 63; bit >= 0; --bit) {
          if (bit < 32 && (1ll << bit) >= 2ll * a.V) continue;  // no index has this bit
          const u64 trial = low | (1ull << bit);
          u64 f = 0;
          scan(xs, n, [&](float x, int i) {
            const float at = r.place(x);
            const u64 key = full_key(x, i0 + i);
            if (at >= from && at < to && key < trial && key <= last) f += cut == 0 ? 1u : r.w(x);
          });
          f = cluster_join(f, SUM, &sh, round, nullptr);
          if (before + f < target) low = trial;
        }
        last = low;
        break;
      }
      // FINISH: every key up to the bin; CUT: the bin's
      const bool finish = v.action == FINISH;
      const uint32_t counter = mapa_shared(smem_u32(&sh.listed), 0u), dst = mapa_shared(smem_u32(list), 0u);
      scan(xs, n, [&](float x, int i) {
        const float at = r.place(x);
        if (at < to && (finish || at >= from)) {
          const u64 key = full_key(x, i0 + i);
          if (key <= last) {
            const uint32_t slot = add_dsmem(counter, 1u);
            if (slot < CAP) st_dsmem(dst + slot * 8, key);
          }
        }
      });
      cluster_sync();
      if (maxima) {  // the maxima did not say how many keys there are
        const bool over = ld_dsmem_u32(counter) > CAP;
        cluster_arrive();  // the first CTA outlives this read
        if (me == 0 || over) cluster_wait();
        if (over) {
          maxima = false;
          before = 0;
          --level;
          continue;
        }
      }
      if (finish) {
        if (me != 0) return;
        const int m = min((int)sh.listed, CAP);
        const u64 all = cut == 1 ? sh.last : 0ull;
        if (m > 128) finish_list(a, r, row, m, all, list, &sh);
        else if (tid < 32 && m > 64) finish_short<4>(a, r, row, m, all, list);
        else if (tid < 32) finish_short<2>(a, r, row, m, all, list);
        return;
      }
      if (me == 0) {
        const int m = min((int)sh.listed, CAP);
        u64 k2[2], total = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) k2[i] = tid + i * THREADS < m ? list[tid + i * THREADS] : ~0ull;
        __syncthreads();
        block_sort(k2, m, list);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const u64 w = tid + i * THREADS >= m ? 0ull : cut == 0 ? 1ull : r.w(key_value((uint32_t)(k2[i] >> 32)));
          u64 part;
          const u64 upto = before + total + block_scan(w, sh.warp, &part);
          total += part;
          if (upto - w < target && target <= upto) sh.last = k2[i];
        }
        __syncthreads();
        if (tid > 0 && tid < n_cta) st_dsmem(mapa_shared(smem_u32(&sh.last), (uint32_t)tid), sh.last);
      }
      cluster_sync();
      last = sh.last;
      break;
    }
  }

  // weights of the kept tokens, a slice a CTA and a part of it a warp; the draw in index order
  u64 sum = 0;
  scan(xs, n, [&](float x, int i) {
    if (full_key(x, i0 + i) <= last && r.e(x) >= r.min_p) sum += r.w(x);
  });
  u64 part = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if ((tid & 31) == 0) sh.warp2[tid >> 5] = part;
  u64 base;
  const u64 total = cluster_join(sum, SUM, &sh, round, &base);
  const double at = floor((double)a.u[row] * (double)total);
  u64 target = at > 0. ? (u64)at : 0ull;  // a NaN draws the first
  if (target > total - 1) target = total - 1;
  if (target < base) return;
  int w0 = 0;
  while (w0 < WARPS && base + sh.warp2[w0] <= target) base += sh.warp2[w0++];
  if (w0 == WARPS) return;  // a later CTA's
  constexpr int VEC = 16 / sizeof(U);
  const int head = min(n, lead(xs)), vecs = (n - head) / VEC;
  const Share share(vecs, w0);
  const int end = w0 == WARPS - 1 ? n : head + share.hi * VEC;
  for (int c = w0 == 0 ? 0 : head + share.lo * VEC; c < end && base <= target; c += THREADS) {  // 512 indexes at a time
    const int i = c + tid;
    u64 w = 0;
    if (i < end) {
      const float x = as_logit(xs[i]);
      if (full_key(x, i0 + i) <= last && r.e(x) >= r.min_p) w = r.w(x);
    }
    u64 all;
    const u64 upto = base + block_scan(w, sh.warp, &all);
    if (upto - w <= target && target < upto) {
      a.tokens[row] = i0 + i;
      a.logprobs[row] = (float)log((double)w / (double)total);
    }
    base += all;
  }
}

// Clusters of 16 have to be asked for, once a kernel and device.
static cudaError_t allow_wide_clusters(const void* kern) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  if (done.count({kern, dev})) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.insert({kern, dev});
  return e;
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
  constexpr int HELD_SLICE = 25600;  // two CTAs an SM
  constexpr int MAX_SLICE = 65532;  // a histogram's halves of weights sum to 32 bits
  TORCH_CHECK(V <= (int64_t)sm::MAX_CLUSTER * MAX_SLICE, "sample_logits: vocabulary too large");
  if (R == 0) return;
  const at::cuda::CUDAGuard guard(logits.device());
  // The most CTAs a row that still let all rows run in one wave (two CTAs an SM, of which clusters leave an
  // eighth, those of 16 a quarter unused), a slice of at least 4096; where no count does, the fewest. Measured,
  // CTAs a row x 16 / 8 / 4: 256 rows x 248320 fp32, top-k, 250 / 158 / 120 us; 64 rows 84 / 61 / -; 16 rows
  // 35 / 28 / -; 64 rows x 100003 bf16, top-p, 86 / 59 / 54 us.
  const int64_t sms = device_sm_count();
  auto slice_of = [&](int c) { return ((V + c - 1) / c + 3) / 4 * 4; };
  auto wave = [&](int c) { return c == 16 ? sms * 3 / 2 : sms * 7 / 4; };
  int least = 1;
  while (slice_of(least) > MAX_SLICE) least *= 2;
  int C = sm::MAX_CLUSTER;
  while (C > least && (slice_of(C) < 4096 || R * C > wave(C))) C /= 2;
  // Slices held in shared memory are read once; as long as two of them fit an SM and one wave takes all rows
  // (64 x 100003 bf16, 4 CTAs a row: 54 us held, 68 not; one row, 16 CTAs: 13.7 held, 15.4 not).
  const bool held = slice_of(C) <= HELD_SLICE && R * C <= wave(C);
  TORCH_CHECK(R * C <= INT_MAX, "sample_logits: too many rows");
  sm::Args a{logits.data_ptr(), logits.stride(0), (int)V, (int)slice_of(C), u.data_ptr<float>(),
             temperature.data_ptr<float>(), top_k.has_value() ? top_k->data_ptr<int32_t>() : nullptr,
             top_p.has_value() ? top_p->data_ptr<float>() : nullptr,
             min_p.has_value() ? min_p->data_ptr<float>() : nullptr, tokens.data_ptr<int64_t>(),
             logprobs.data_ptr<float>()};
  const bool f32 = logits.dtype() == torch::kFloat32;
  auto kern = held ? (f32 ? sample_kernel<float, true> : sample_kernel<__nv_bfloat16, true>)
                   : (f32 ? sample_kernel<float, false> : sample_kernel<__nv_bfloat16, false>);
  TORCH_CHECK(ensure_smem_attr((const void*)kern, sm::WORK_BYTES + (held ? HELD_SLICE * 4 + 16 : 0)) == cudaSuccess &&
                  allow_wide_clusters((const void*)kern) == cudaSuccess, "sample_logits: kernel attributes");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * C));
  cfg.blockDim = dim3(sm::THREADS);
  cfg.dynamicSmemBytes = (size_t)sm::WORK_BYTES + (held ? (size_t)a.slice * 4 + 16 : 0);
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
