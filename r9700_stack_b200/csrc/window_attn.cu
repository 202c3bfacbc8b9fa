// Attention of new tokens over a paged e4m3 cache with a sliding window and sink tokens.
//
// A query at position p (its context is p + 1) sees key j iff j <= p and (W = 0 or j > p - W or
// j < S): the last W positions, its own among them, and the first S tokens of the sequence.
//   o = softmax(q K^T * scale) V, then o * sigmoid(gate) where a gate is given, rounded to bf16 once.
// A row that sees no key is zero. Keys outside the visible range are never used, whatever their pages
// hold.
//
// Precision. The cache stays e4m3 in shared memory, where the MMA reads it; the other operand of each
// product is the sum of two 8-bit numbers, both multiplied into fp32 accumulators: a query q as two e4m3
// numbers after a power-of-two scaling of its row (exact for |q| >= amax / 1792, else within 2^-17 amax),
// a probability p as an e4m3 number and what that leaves, within 2^-7 of itself (rms 2^-10) or 2^-19 of the
// row's largest. The rest has a wider range than the first number: e5m2 where both share an accumulator,
// e4m3 of 16 times itself where each has its own. A first token that takes most of the weight (a sink)
// leaves the others weights of 2^-14, of which an e4m3 rest would keep two bits. Two 8-bit products cost
// what one bf16 product does, and no key or value has to be widened on the way.
//
// KV cache layout: [pages][kv_heads][64][head_dim] e4m3 for K and V separately.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <climits>
#include "common.cuh"
#include "tmap.h"

namespace r9k {

namespace wa {
constexpr int PAGE = 64;
constexpr int KT = 128;  // keys of a tile: the MMA's M (single tokens) or N (chunks)

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
  float scale_log2;  // sm_scale * k_scale, for powers of two
  float v_scale;
  int* status;
  uint64_t timeout_ns;
};

// The keys that a group of rows can see, as a list of pages: those of the sinks first, then the window's
// from a page boundary on. A tile is two neighbours of the list.
constexpr int NO_KEY = INT_MAX / 2;
struct Span {
  int base, n_sink, pages, n;  // first window page, pages of the sinks, pages, tiles
  R9K_DEVINL int key(int i) const {  // first key of page i of the list; NO_KEY past its end
    return i < n_sink ? i * PAGE : i < pages ? (base + i - n_sink) * PAGE : NO_KEY;
  }
};

// ctx_min, ctx_max: smallest and largest context of the rows that see anything (0, 0: none does)
R9K_DEVINL Span make_span(const Args& a, int ctx_min, int ctx_max) {
  Span s;
  s.base = (a.window > 0 ? max(0, ctx_min - a.window) : 0) / PAGE;
  s.n_sink = min((a.sinks + PAGE - 1) / PAGE, s.base);
  s.pages = s.n_sink + max(0, (ctx_max + PAGE - 1) / PAGE - s.base);
  s.n = (s.pages + 1) / 2;
  return s;
}

// whether every row that sees anything (contexts in [ctx_min, ctx_max]) sees the whole page at key
R9K_DEVINL bool whole_page(const Args& a, int key, int ctx_min, int ctx_max) {
  return key + PAGE <= ctx_min && (a.window == 0 || key >= ctx_max - a.window || key + PAGE <= a.sinks);
}

R9K_DEVINL bool visible(const Args& a, int key, int ctx) {
  return key < ctx && (a.window == 0 || key >= ctx - a.window || key < a.sinks);
}

// a token's context, cut to what its table row can hold
R9K_DEVINL int context(const Args& a, int tok) {
  const int c = a.tok_ctx[tok];
  if (c > a.width * PAGE) {
    report_error(a.status, kErrBounds, 301, c);
    return a.width * PAGE;
  }
  return max(c, 0);
}

// smallest (of the positive ones) and largest context of n tokens from tok0 on; one warp
R9K_DEVINL void context_range(const Args& a, int tok0, int n, int& lo, int& hi) {
  lo = INT_MAX;
  hi = 0;
  for (int i = lane_id(); i < n; i += 32) {
    const int c = context(a, tok0 + i);
    if (c > 0) lo = min(lo, c);
    hi = max(hi, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (hi == 0) lo = 0;
}

R9K_DEVINL int page_of(const Args& a, int seq, int key) {
  const int p = a.table[(int64_t)seq * a.width + key / PAGE];
  if ((unsigned)p >= (unsigned)a.pages) {
    report_error(a.status, kErrBounds, 302, p);
    return 0;
  }
  return p;
}

// The loading warp's view of the page list: 32 page numbers at a time, a lane each, so that the table's
// latency is paid once in 16 tiles and not once a tile.
struct Pages {
  int first = -1, mine = 0;  // list index of lane 0's page
  R9K_DEVINL int get(const Args& a, const Span& sp, int seq, int i, int origin) {
    const int f = origin + (i - origin) / 32 * 32;
    if (f != first) {
      first = f;
      const int key = sp.key(f + (int)lane_id());
      mine = key != NO_KEY ? page_of(a, seq, key) : 0;  // page 0 stands in past the list's end (masked)
    }
    return __shfl_sync(0xffffffffu, mine, i - f);
  }
};

// K or V tile j -> shared memory: two pages, D / 128 column halves, 128-byte swizzled rows. A whole warp;
// `go` is true in the lane that issues.
template <int D>
R9K_DEVINL void load_tile(const Args& a, const CUtensorMap* map, uint8_t* dst, uint64_t* bar, const Span& sp, Pages& pages, int j,
                          int origin, int seq, int kvh, bool go) {
  int page[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) page[p] = pages.get(a, sp, seq, 2 * j + p, 2 * origin);
  if (go) {
    mbar_arrive_expect_tx(bar, KT * D);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int h = 0; h < D / 128; ++h)
        tma_load_2d(dst + h * (KT * 128) + p * (PAGE * 128), map, bar, h * 128, (page[p] * a.Hkv + kvh) * PAGE);
  }
}

// The MMA warp runs as a whole, so that addresses stay in uniform registers (a lone thread pays dozens of
// cycles an MMA to move them there), and one elected lane issues: `go` is that lane's predicate.
R9K_DEVINL void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accum, bool go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accum), "r"((uint32_t)go)
      : "memory");
}
// A from TMEM: 4 e4m3 numbers of a row in a 32-bit column
R9K_DEVINL void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accum, bool go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"((uint32_t)accum), "r"((uint32_t)go)
      : "memory");
}
R9K_DEVINL void commit(uint64_t* bar, bool go) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"((uint32_t)go)
      : "memory");
}
R9K_DEVINL bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t timeout_ns) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, timeout_ns));
}

// operand descriptor, MN-major 128-byte swizzle (values: head dims contiguous, keys along K)
R9K_DEVINL uint64_t sdesc_mn(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((KT * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

R9K_DEVINL float ld_dsmem(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

R9K_DEVINL uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
R9K_DEVINL float2 f32x2(uint32_t e) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)e, __NV_E4M3);
  return __half22float2(__half2(h));
}
// (hi, lo) e4m3 pairs of two numbers: x ~ hi + lo
R9K_DEVINL void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = e4m3x2(x, y);
  const float2 b = f32x2(hi);
  lo = e4m3x2(x - b.x, y - b.y);
}

// The same for probabilities (0..448): by way of f16, whose conversions are cheaper and whose 2^-12 (2^-25
// below 2^-14) is far below the rest's. E5M2: the rest as e5m2; else as e4m3 of 16 times itself.
template <bool E5M2>
R9K_DEVINL void split2p(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 p = __floats2half2_rn(x, y);
  hi = (uint32_t)__nv_cvt_halfraw2_to_fp8x2(__half2_raw(p), __NV_SATFINITE, __NV_E4M3);
  __half2 rest = __hsub2(p, __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)hi, __NV_E4M3)));
  if (!E5M2) rest = __hmul2(rest, __float2half2_rn(16.f));
  lo = (uint32_t)__nv_cvt_halfraw2_to_fp8x2(__half2_raw(rest), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}
R9K_DEVINL float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bf16 of a row -> 16 bytes hi and lo, scaled
R9K_DEVINL void split16(const uint4 (&r)[2], float inv, uint4& hi, uint4& lo) {
  const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(r);
  uint32_t* ph = reinterpret_cast<uint32_t*>(&hi);
  uint32_t* pl = reinterpret_cast<uint32_t*>(&lo);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h0, l0, h1, l1;
    split2(__bfloat162float(e[4 * i]) * inv, __bfloat162float(e[4 * i + 1]) * inv, h0, l0);
    split2(__bfloat162float(e[4 * i + 2]) * inv, __bfloat162float(e[4 * i + 3]) * inv, h1, l1);
    ph[i] = h0 | (h1 << 16);
    pl[i] = l0 | (l1 << 16);
  }
}
R9K_DEVINL float amax16(const uint4 (&r)[2]) {
  const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(r);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(__bfloat162float(e[i])));
  return m;
}

// Probabilities are exp2(s - m_ref + P_SHIFT): m_ref follows the running maximum once that has grown by
// P_LAG (O is rescaled then), so the largest lies in [2^6, 2^8.75], below e4m3's 448. Below 2^-6 the
// first number has steps of 2^-9; the rest, 2^-10 at most, is held to 2^-13 (e5m2) or 2^-14, which is
// 2^-19 of the largest or less.
constexpr float P_SHIFT = 6.f, P_LAG = 2.75f;

// One value row (key r of a tile, column halves [H0, H1)) whose key some of the rows do not see. A NaN code
// in it would reach those rows too (0 * NaN), so such a row of values is cleared, and the rows that do
// see its key are marked: they become NaN as a whole. Values of keys that no row sees are stale bytes.
template <int H0, int H1, typename P>
R9K_DEVINL void clean_value_row(const Args& a, uint8_t* tile, int r, int key, int tok0, int ntok, P* poison) {
  uint32_t nan = 0;
#pragma unroll
  for (int h = H0; h < H1; ++h)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint4 v = *reinterpret_cast<const uint4*>(tile + h * (KT * 128) + r * 128 + ((c ^ (r & 7)) << 4));
      nan |= ((v.x & 0x7f7f7f7fu) + 0x01010101u) | ((v.y & 0x7f7f7f7fu) + 0x01010101u) |
             ((v.z & 0x7f7f7f7fu) + 0x01010101u) | ((v.w & 0x7f7f7f7fu) + 0x01010101u);
    }
  if ((nan & 0x80808080u) == 0) return;
  for (int i = 0; i < ntok; ++i)
    if (visible(a, key, context(a, tok0 + i))) poison[i] = 1;
#pragma unroll
  for (int h = H0; h < H1; ++h)
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<uint4*>(tile + h * (KT * 128) + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
}
}  // namespace wa

// ------------------------------------------------------------------------------------------------
// Single tokens and a few drafts: up to 16 rows (tokens x heads of one kv head's group) of a sequence.
//
// The 128 keys of a tile are the MMA's M rows and the query rows its N = 16 columns, so no product is
// spent on padding rows: S^T = K Q^T [keys x rows], O^T += V^T P^T [dims x rows], both in TMEM. K and V
// tiles share one ring of shared-memory slots in the order in which the MMAs use them (K0 K1 V0 K2 V1
// ...). Warp 0 loads (TMA), warp 1 issues MMAs, warps 2-5 hold one key a thread: they mask, find the
// column maxima together, and write the probabilities as two e4m3 planes.
// The CTAs of a cluster take neighbouring shares of the tiles; at the end each of them sums a share of
// the dims over the others' partial results in distributed shared memory, and writes the output.
//
// hi and lo planes are columns of one product (N = 2 x 8 or 2 x 16), not two products: small MMAs cost
// about 40 cycles of issue each, whatever N. What bounds it: for a batch the cache's bytes (64 sequences x
// window 4096, 4 x 256 kv heads, 520 MB: 88 us, 0.92 of copy bandwidth); for one sequence latency (14.9 us:
// launch, three dependent reads before the first tile, 5 key tiles of 1.1 us on each of 8 CTAs, the join).
// Key shares for 1 / 2 / 4 / 8 CTAs: 64 sequences 89 / 92 / 110 / 144 us, one sequence 43 / 27 / 18 / 15 us.
// ------------------------------------------------------------------------------------------------
namespace wd {
using namespace wa;
constexpr int ROWS = 16;  // most query rows
constexpr int THREADS = 192;
template <int D, int NC>
struct Cfg {
  static constexpr int N = 2 * NC;  // columns: the rows' hi planes, then their lo planes
  static constexpr int HALVES = D / 128;
  static constexpr int UNIT = KT * D;                 // one K or V tile
  static constexpr int SLOTS = D == 256 ? 3 : 6;      // two CTAs on an SM
  static constexpr int Q_BYTES = HALVES * N * 128;    // a swizzled tile a column half
  static constexpr int P_BYTES = N * 128;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = OFF_Q + Q_BYTES;
  static constexpr int OFF_P = OFF_RING + SLOTS * UNIT;     // [parity]
  static constexpr int OFF_RED = OFF_P + 2 * P_BYTES;       // float maxima [parity][NC][4 warps]; at the end sums
  static constexpr int OFF_COL = OFF_RED + 2 * 4 * NC * 4;  // scale, ctx, poison (by token), m, l [ROWS]
  static constexpr int OFF_W = OFF_COL + 5 * ROWS * 4;      // weights of the cluster's partial results [ROWS][8]
  static constexpr int OFF_BAR = OFF_W + ROWS * 8 * 4;
  static constexpr int NBAR = 1 + 2 * SLOTS + 8;  // q_full, full[], empty[], s_full[2], s_free[2], p_full[2], pv_done[2]
  static constexpr int OFF_TMEM = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;
  static constexpr int TMEM_COLS = 4 * N;
  static constexpr int S_COL = 0, O_COL = 2 * N;  // two S buffers, O^T halves
};
}  // namespace wd

R9K_DEVINL void wd_bar() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int D, int NC>
__global__ void __launch_bounds__(wd::THREADS, 2)
    window_attn_dec_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const wa::Args a) {
  using namespace wd;
  using C = Cfg<D, NC>;
  constexpr int N = C::N, S_COL = C::S_COL, O_COL = C::O_COL;
  pdl_wait();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;
  uint64_t* empty = full + C::SLOTS;
  uint64_t* s_full = empty + C::SLOTS;
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* pv_done = p_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_TMEM);
  float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
  float* col_scale = reinterpret_cast<float*>(smem + C::OFF_COL);
  int* col_ctx = reinterpret_cast<int*>(col_scale + ROWS);
  int* poison = col_ctx + ROWS;  // by token
  float* col_m = reinterpret_cast<float*>(poison + ROWS);
  float* col_l = col_m + ROWS;
  float* weight = reinterpret_cast<float*>(smem + C::OFF_W);

  const int warp = warp_id(), lane = lane_id();
  const int seq = blockIdx.x, kvh = blockIdx.y;
  const int nsplit = gridDim.z, split = blockIdx.z;
  const int tok0 = a.seq_start[seq], ntok = a.seq_len[seq];
  // the same decision in every CTA of the cluster: nobody is left at its barrier
  if (ntok <= 0) return;
  if (ntok > a.max_new || tok0 < 0 || tok0 > a.T - ntok) {
    if (threadIdx.x == 0) report_error(a.status, ntok > a.max_new ? kErrConfig : kErrBounds, 310, ntok);
    return;
  }
  int ctx_min, ctx_max;
  context_range(a, tok0, ntok, ctx_min, ctx_max);
  const Span sp = make_span(a, ctx_min, ctx_max);
  const int share = (sp.n + nsplit - 1) / nsplit;
  const int j0 = min(sp.n, split * share), n = min(sp.n, j0 + share) - j0;
  const int NQ = ntok * a.G;  // <= NC

  if (threadIdx.x == 0) {
    mbar_init(q_full, 128);
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 128);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1);
    }
    fence_mbar_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (threadIdx.x < ROWS) poison[threadIdx.x] = 0;
  if (warp == 1) {
    tmem_alloc(tmem_holder, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now: a dependent kernel that takes TMEM ahead of its own wait must not come between a CTA of this
  // grid and its columns.
  pdl_trigger();
  const uint32_t tbase = *tmem_holder;
  // the order of use: K0, then K(j + 1) (if there is one) and V(j)
  auto unit_v = [&](int j) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; };

  if (warp == 0) {
    const bool go = elect_one();
    Pages pages;
    for (int u = 0; u < 2 * n; ++u) {
        const bool is_k = u == 0 || ((u & 1) && u < 2 * n - 1);
        const int j = is_k ? (u + 1) / 2 : (u == 2 * n - 1 ? n - 1 : u / 2 - 1);
        const int s = u % C::SLOTS;
        if (!warp_wait(&empty[s], (uint32_t)(((u / C::SLOTS) & 1) ^ 1), a.timeout_ns)) {
          if (go) report_error(a.status, kErrMbarTimeout, 311, u);
          break;
        }
        load_tile<D>(a, is_k ? &tmK : &tmV, smem + C::OFF_RING + s * C::UNIT, &full[s], sp, pages, j0 + j, j0, seq, kvh, go);
      }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      constexpr uint32_t idesc_s = idesc_dense(kFmtE4M3, kFmtE4M3, KT, N);
      constexpr uint32_t idesc_o = idesc_dense(kFmtE4M3, kFmtE4M3, 128, N) | (1u << 15);  // A (V^T) MN-major
      const bool go = elect_one();
      const uint64_t q_desc = sdesc_k_sw128(smem_u32(smem + C::OFF_Q));
      const uint64_t k_desc = sdesc_k_sw128(smem_u32(smem + C::OFF_RING));
      const uint64_t v_desc = sdesc_mn(smem_u32(smem + C::OFF_RING));
      const uint64_t p_desc = sdesc_k_sw128(smem_u32(smem + C::OFF_P));
      bool ok = warp_wait(q_full, 0, a.timeout_ns);
      auto wait_unit = [&](int u) { return warp_wait(&full[u % C::SLOTS], (uint32_t)((u / C::SLOTS) & 1), a.timeout_ns); };
      auto issue_s = [&](int j) -> bool {
        const int s = j & 1, u = j == 0 ? 0 : 2 * j - 1;
        if (!wait_unit(u)) return false;
        if (!warp_wait(&s_free[s], (uint32_t)(((j >> 1) & 1) ^ 1), a.timeout_ns)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)((u % C::SLOTS) * (C::UNIT >> 4));
#pragma unroll
        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ss(tbase + S_COL + s * N, kd + ((h * (KT * 128) + 32 * k) >> 4), q_desc + ((h * (N * 128) + 32 * k) >> 4),
                   idesc_s, h > 0 || k > 0, go);
        commit(&s_full[s], go);
        commit(&empty[u % C::SLOTS], go);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; ok && j < n; ++j) {
        if (j + 1 < n && !issue_s(j + 1)) { ok = false; break; }
        const int pb = j & 1, u = unit_v(j);
        if (!warp_wait(&p_full[pb], (uint32_t)((j >> 1) & 1), a.timeout_ns)) { ok = false; break; }
        if (!wait_unit(u)) { ok = false; break; }
        tc_fence_after();
        const uint64_t vd = v_desc + (uint64_t)((u % C::SLOTS) * (C::UNIT >> 4));
        const uint64_t pd = p_desc + (uint64_t)(pb * C::P_BYTES >> 4);
#pragma unroll
        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ss(tbase + O_COL + h * N, vd + ((h * (KT * 128) + k * 4096) >> 4), pd + (32 * k >> 4), idesc_o, j > 0 || k > 0,
                   go);
        commit(&pv_done[pb], go);
        commit(&empty[u % C::SLOTS], go);
      }
      if (!ok && lane == 0) report_error(a.status, kErrMbarTimeout, 312, 0);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int r = q * 32 + lane;      // TMEM lane: key of the tile, then dim of the output
    const int tr = threadIdx.x - 64;  // 0..127
    // columns past NQ: a zero query and context 0, which gives them no weight at the end; eight threads a query row
    {
      const int row = tr >> 3, part = tr & 7;
      const bool valid = row < NQ;
      const int tok = tok0 + (valid ? row / a.G : 0), head = kvh * a.G + row % a.G;
      constexpr int CH = D / 128;  // 16-element chunks a thread
      uint4 raw[CH][2];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int e0 = (c * 8 + part) * 16;
        if (valid) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.ld_q + head * D + e0);
          raw[c][0] = src[0];
          raw[c][1] = src[1];
        } else {
          raw[c][0] = raw[c][1] = make_uint4(0, 0, 0, 0);
        }
        amax = fmaxf(amax, amax16(raw[c]));
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int e = mx_exponent(amax, 448.f);
      if (row < NC) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          uint4 hi, lo;
          split16(raw[c], exp2i(-e), hi, lo);
          uint8_t* dst = smem + C::OFF_Q + c * (N * 128) + row * 128 + ((part ^ (row & 7)) << 4);  // NC % 8 == 0: lo alike
          *reinterpret_cast<uint4*>(dst) = hi;
          *reinterpret_cast<uint4*>(dst + NC * 128) = lo;
        }
        if (part == 0) {
          col_scale[row] = a.scale_log2 * exp2i(max(e, -126));
          col_ctx[row] = valid ? context(a, tok) : 0;
        }
      }
      fence_proxy_async();
      mbar_arrive(q_full);
    }
    wd_bar();
    float mref[NC], lsum[NC], csc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      mref[c] = -INFINITY;
      lsum[c] = 0.f;
      csc[c] = col_scale[c];
    }
    // A wait that runs out is told to the other warps (a NaN in place of a maximum, which never is one):
    // all four leave at the same exchange, so none is left at their barrier.
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int s = j & 1, pb = j & 1;
      ok &= warp_wait(&s_full[s], (uint32_t)((j >> 1) & 1), a.timeout_ns);
      tc_fence_after();
      float sv[N];
#pragma unroll
      for (int c = 0; c < N; c += 16) tmem_ld16(tbase + ((uint32_t)(q * 32) << 16) + S_COL + s * N + c, sv + c);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(&s_free[s]);
      const int key0 = sp.key(2 * (j0 + j) + (q >> 1));  // of this warp's page
      const int key = key0 + (r & (PAGE - 1));
      const bool whole = whole_page(a, key0, ctx_min, ctx_max);
      float* rmax = red + pb * 4 * NC;
      float mx[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        sv[c] = (sv[c] + sv[NC + c]) * csc[c];
        if (!whole && !visible(a, key, col_ctx[c])) sv[c] = -INFINITY;
        mx[c] = fmaxf(sv[c], -INFINITY);  // not a NaN
      }
      // the warp's maxima: each step halves the columns a lane answers for, so NC / 2 + NC / 4 ... exchanges
      // do where a butterfly of every column takes 5 NC
#pragma unroll
      for (int w = NC / 2, o = 16; w > 0; w >>= 1, o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int c = 0; c < NC / 2; ++c)
          if (c < w) {
            const float keep = up ? mx[c + w] : mx[c], give = up ? mx[c] : mx[c + w];
            mx[c] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, o));
          }
      }
#pragma unroll
      for (int o = 16 / NC; o > 0; o >>= 1) mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
      // lane's column: its top bits, the highest first
      if ((lane & (32 / NC - 1)) == 0) rmax[(lane / (32 / NC)) * 4 + q] = ok ? mx[0] : __int_as_float(0x7fffffff);
      if (!whole) {
        const int u = unit_v(j);
        ok &= warp_wait(&full[u % C::SLOTS], (uint32_t)((u / C::SLOTS) & 1), a.timeout_ns);
        clean_value_row<0, C::HALVES>(a, smem + C::OFF_RING + (u % C::SLOTS) * C::UNIT, r, key, tok0, ntok, poison);
      }
      // P buffer pb is free once the PV of tile j - 2 is done
      if (j >= 2) ok &= warp_wait(&pv_done[pb], (uint32_t)(((j - 2) >> 1) & 1), a.timeout_ns);
      wd_bar();
      float t[NC];
      bool any = false, fail = false;  // by what was exchanged alone; a later failure is told with the next tile
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float4 m4 = *reinterpret_cast<const float4*>(rmax + c * 4);
        if (c == 0) fail = m4.x != m4.x || m4.y != m4.y || m4.z != m4.z || m4.w != m4.w;
        t[c] = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
        any |= t[c] > mref[c] + P_LAG;  // the first key seen among them
      }
      if (fail) {  // known to all: rmax of this tile is not written again before they have read it
        ok = false;
        break;
      }
      if (any) {
        float fac[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const bool need = t[c] > mref[c] + P_LAG;
          fac[c] = need ? ex2(mref[c] - t[c]) : 1.f;  // 0 for the first
          if (need) mref[c] = t[c];
          lsum[c] *= fac[c];
        }
        if (j >= 1) {
          // O is complete before it is rescaled
          ok &= warp_wait(&pv_done[(j - 1) & 1], (uint32_t)(((j - 1) >> 1) & 1), a.timeout_ns);
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
            for (int c0 = 0; c0 < N; c0 += 16) {
              const uint32_t orow = tbase + ((uint32_t)(q * 32) << 16) + O_COL + h * N + c0;
              float o[16];
              tmem_ld16(orow, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= fac[(c0 + i) % NC];
              tmem_st16(orow, o);
            }
          tmem_st_wait();
        }
      }
      uint8_t* prow = smem + C::OFF_P + pb * C::P_BYTES;
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        float p[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[i] = sv[c + i] == -INFINITY ? 0.f : ex2(sv[c + i] - mref[c + i] + P_SHIFT);
          lsum[c + i] += p[i];  // of this thread's keys; they are added up at the end
        }
        uint32_t hi, lo;
        split2p<false>(p[0], p[1], hi, lo);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint8_t* dst = prow + (c + i) * 128 + ((((r >> 4) ^ ((c + i) & 7)) << 4) | (r & 15));
          dst[0] = (uint8_t)(hi >> (8 * i));
          dst[NC * 128] = (uint8_t)(lo >> (8 * i));
        }
      }
      fence_proxy_async();
      tc_fence_before();
      mbar_arrive(&p_full[pb]);
    }
    if (ok && n > 0) {
      // the products of the last two tiles: their barriers are separate
      ok = warp_wait(&pv_done[(n - 1) & 1], (uint32_t)(((n - 1) >> 1) & 1), a.timeout_ns);
      tc_fence_after();
    }
    if (!ok) report_error(a.status, kErrMbarTimeout, 313, r);
    wd_bar();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lsum[c] += __shfl_xor_sync(0xffffffffu, lsum[c], o);
      if (lane == 0) red[c * 4 + q] = lsum[c];
    }
    // this CTA's partial results [row][dim], over the ring (all its tiles have been used)
    if (n > 0 && ok) {
      float* part = reinterpret_cast<float*>(smem + C::OFF_RING);
#pragma unroll
      for (int h = 0; h < C::HALVES; ++h) {
        float o[N];
#pragma unroll
        for (int c0 = 0; c0 < N; c0 += 16) tmem_ld16(tbase + ((uint32_t)(q * 32) << 16) + O_COL + h * N + c0, o + c0);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < NC; ++c) part[c * D + h * 128 + r] = o[c] + o[NC + c] * 0.0625f;
      }
    }
    wd_bar();
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (tr == c) {
        const float4 l4 = *reinterpret_cast<const float4*>(red + c * 4);
        col_m[c] = n > 0 && ok ? mref[c] : -INFINITY;
        col_l[c] = n > 0 && ok ? (l4.x + l4.y) + (l4.z + l4.w) : 0.f;
        if (c < NQ && poison[c / a.G]) col_l[c] = __int_as_float(0x7fffffff);
        if (col_ctx[c] == 0) col_l[c] = 0.f;  // sees nothing (its scores of whole pages were not masked)
      }
  }
  __syncwarp();  // the cluster's barrier wants whole warps
  tc_fence_before();
  if (nsplit > 1) cluster_sync();
  else __syncthreads();

  // each CTA of the cluster joins a share of the dims of every row: the partial results' weights first
  {
    const uint32_t part = smem_u32(smem + C::OFF_RING), ml = smem_u32(col_m);
    if (threadIdx.x < NQ) {
      const int row = threadIdx.x;
      float m[8], l[8], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < nsplit) {
          const uint32_t b = mapa_shared(ml, (uint32_t)s);
          m[s] = ld_dsmem(b + row * 4);
          l[s] = ld_dsmem(b + (ROWS + row) * 4);
          if (l[s] != 0.f) M = fmaxf(M, m[s]);
        }
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < nsplit) {
          m[s] = l[s] == 0.f ? 0.f : m[s] == -INFINITY ? 1.f : ex2(m[s] - M);
          if (l[s] != 0.f) L += m[s] * l[s];
        }
      const float inv = L != 0.f ? a.v_scale / L : 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < nsplit) weight[row * 8 + s] = m[s] * inv;
    }
    __syncthreads();
    const int dn = D / 4 / nsplit;  // four dims an item
    for (int i = threadIdx.x; i < NQ * dn; i += THREADS) {
      const int row = i / dn, d = 4 * (split * dn + i % dn);
      const int tok = tok0 + row / a.G, col = (kvh * a.G + row % a.G) * D + d;
      uint2 g = make_uint2(0, 0);
      if (a.gate != nullptr) g = *reinterpret_cast<const uint2*>(a.gate + (int64_t)tok * a.ld_gate + col);
      float o[4] = {0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < nsplit; ++s) {
        const float w = weight[row * 8 + s];
        if (w == 0.f) continue;  // nothing was seen there: nothing was written either
        const float4 v = ld_dsmem_f4(mapa_shared(part, (uint32_t)s) + (row * D + d) * 4);
        o[0] += w * v.x;
        o[1] += w * v.y;
        o[2] += w * v.z;
        o[3] += w * v.w;
      }
      const __nv_bfloat16* ge = reinterpret_cast<const __nv_bfloat16*>(&g);
      uint2 w2;
      __nv_bfloat16* we = reinterpret_cast<__nv_bfloat16*>(&w2);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (a.gate != nullptr) o[c] *= sigmoid_f(__bfloat162float(ge[c]));
        we[c] = __float2bfloat16(o[c]);
      }
      *reinterpret_cast<uint2*>(a.out + (int64_t)tok * a.ld_out + col) = w2;
    }
  }
  if (nsplit > 1) cluster_sync();  // peers read this CTA's shared memory until here
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------
// Chunks: a tile of up to 128 rows (128 / G tokens x the G heads of one kv head's group), rows on the
// MMA's M side.
//
// S = Q K^T [rows x keys] with two S buffers in TMEM, so the next tile's product runs during this
// tile's softmax; O += P V with V read as it lies (MN-major B operand), O in TMEM. Two threads a row, in two
// warpgroups, take 64 keys each: scores from TMEM, the row's running maximum (exchanged through shared
// memory, one barrier of the two warps a tile), their part of the sum, and the probabilities as two planes,
// written over the scores in TMEM: as the A operand of PV they cost no shared memory bandwidth, which is
// what two products on one K or V tile run into (both planes' MMAs read it). MMAs run in order, so S(j + 2)
// does not overtake PV(j) on the buffer they share, and only a rescale of O has to wait for PV(j - 1).
// One CTA an SM. Two of them with one S buffer each, for which heads of 128 leave room, took 160 us where
// this takes 146 (3850 ragged tokens, 32 / 8 heads, window 1024): their registers held half the scores, so
// every score was read and masked twice.
// K and V tiles share a ring of slots in the order of use, as above. Few tiles: a cluster of CTAs
// shares the keys of a tile and joins the partial results through distributed shared memory.
//
// What bounds it: 8192 tokens, 24 / 4 heads of 256, window 4096: 890 to 975 us with the card's clocks, 850 to
// 930 TFLOP/s of useful products, 0.51 to 0.55 of the bf16 rate (the tensor pipe is busy 0.46 of the time at the
// 8-bit rate, on two planes). Stamps of all 1568 CTAs at 1.8 GHz: 141000 cycles a CTA. Its start (page
// and length reads, queries) takes 14700, 33 key tiles 100000 and its end (last product, gate, output) 25700;
// nothing covers a start or an end, as one CTA fills an SM. A tile takes 3020 on average: 2510 where O stays as
// it is, 3000 where some row's is rescaled (three in four), 3500 at the masked edges (two a CTA). 2050 of them are
// MMA at the least, beside a softmax chain of about 2200 (1024 the exponential unit's 16 a cycle), 2600 with its
// wait for the scores.
// Ragged prompts, 3850 tokens, 32 / 8 heads of 128, window 1024: 148 us. A CTA of nine tiles takes 40000 cycles:
// 27700 in the tiles, 3080 each, 7500 before them and 2800 after.
// Shares of 1 / 2 / 4 / 8 CTAs for 16 sequences x 1..8 drafts, 16 / 2 heads: 34 / 27 / 21 / 44 us.
// ------------------------------------------------------------------------------------------------
namespace wc {
using namespace wa;
constexpr int ROWS = 128;
constexpr int THREADS = 320;   // TMA, MMA, two softmax warpgroups
constexpr int SOFT = 256;
template <int D>
struct Cfg {
  static constexpr int HALVES = D / 128;
  static constexpr int UNIT = KT * D;
  static constexpr int SLOTS = D == 256 ? 5 : 8;
  static constexpr int PLANE_Q = ROWS * D;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_RING = OFF_Q + 2 * PLANE_Q;
  static constexpr int OFF_RED = OFF_RING + SLOTS * UNIT;  // maxima [parity][half][ROWS]; at the end l[half][ROWS], m[ROWS]
  static constexpr int OFF_POISON = OFF_RED + 4 * ROWS * 4;  // bytes by token
  static constexpr int OFF_BAR = OFF_POISON + ROWS;
  static constexpr int NBAR = 1 + 2 * SLOTS + 6;  // q_full, full[], empty[], s_full[2], p_full[2], pv_done[2]
  static constexpr int OFF_TMEM = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_TMEM + 16;
  static constexpr int TMEM_COLS = 512;
  static constexpr int O_COL = 0, S_COL = D;  // S buffers of 128 columns; P planes at columns 0 and 32 of them
  static_assert(D + 2 * KT <= TMEM_COLS && SMEM <= 232448, "TMEM and shared memory");
  static_assert(SLOTS * UNIT >= ROWS * D * 4, "the ring holds the partial results");
};
}  // namespace wc

template <int D>
__global__ void __launch_bounds__(wc::THREADS, 1)
    window_attn_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const wa::Args a) {
  using namespace wc;
  using C = Cfg<D>;
  constexpr int O_COL = C::O_COL, S_COL = C::S_COL;
  pdl_wait();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;
  uint64_t* empty = full + C::SLOTS;
  uint64_t* s_full = empty + C::SLOTS;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_TMEM);
  float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
  float* row_l = red;             // [half][ROWS]
  float* row_m = red + 2 * ROWS;  // [ROWS]
  uint8_t* poison = smem + C::OFF_POISON;

  const int warp = warp_id(), lane = lane_id();
  const int kvh = blockIdx.y;
  const int nsplit = gridDim.z, split = blockIdx.z;
  const int per = ROWS / a.G;  // tokens of a tile

  // the sequence and the tokens of this tile: tiles are numbered through the sequences
  int seq = -1, tok0 = 0, ntok = 0, len_seq = 0, start = 0;
  {
    int before = 0;
    for (int s0 = 0; s0 < a.S && seq < 0; s0 += 32) {
      const int len = s0 + lane < a.S ? max(a.seq_len[s0 + lane], 0) : 0;
      const int st = s0 + lane < a.S ? a.seq_start[s0 + lane] : 0;
      const int tiles = len > a.max_new ? 0 : (len + per - 1) / per;
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, (int)blockIdx.x < before + inc);
      if (hit != 0) {
        const int src = __ffs((int)hit) - 1;
        const int first = (int)blockIdx.x - before - (__shfl_sync(0xffffffffu, inc - tiles, src));
        seq = s0 + src;
        tok0 = first * per;
        len_seq = __shfl_sync(0xffffffffu, len, src);
        start = __shfl_sync(0xffffffffu, st, src);
        ntok = min(per, len_seq - tok0);
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && split == 0 && warp == 0) {
    // One warp of the grid looks at every sequence (the search above ends at the block's own). The grid holds the
    // tiles of T tokens: sequences that share tokens would need more.
    int all = 0;
    for (int i = lane; i < a.S; i += 32) {
      const int len = a.seq_len[i];
      if (len > a.max_new) report_error(a.status, kErrConfig, 320, len);
      else if (len > 0) all += (len + per - 1) / per;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    if (all > (int)gridDim.x && lane == 0) report_error(a.status, kErrBounds, 326, all);
  }
  if (seq < 0) return;  // the grid is a bound: the same in the whole cluster
  if (smem_u32(smem) & 1023) {  // the swizzled tiles need it
    if (threadIdx.x == 0) report_error(a.status, kErrConfig, 325, (int)smem_u32(smem));
    return;
  }
  if (start < 0 || start > a.T - len_seq) {
    if (threadIdx.x == 0) report_error(a.status, kErrBounds, 321, start);
    return;
  }
  tok0 += start;
  const int nrows = ntok * a.G;
  // softmax warps: this thread's half of its query row, on its way while the CTA is set up
  constexpr int QC = D / 32;  // 16-element pieces of half a row
  const int r = (warp & 3) * 32 + lane, half = warp >= 2 ? (warp - 2) >> 2 : 0;
  const bool valid = warp >= 2 && r < nrows;
  const int rt = valid ? r / a.G : 0, rg = r % a.G;
  const int tok = tok0 + rt, head = kvh * a.G + rg;
  uint4 qraw[QC][2];
#pragma unroll
  for (int c = 0; c < QC; ++c) {
    qraw[c][0] = qraw[c][1] = make_uint4(0, 0, 0, 0);
    if (valid) {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.ld_q + head * D) + 2 * (half * QC + c);
      qraw[c][0] = src[0];
      qraw[c][1] = src[1];
    }
  }
  if (valid && a.gate != nullptr && nsplit == 1) {  // wanted at the end: from DRAM to L2 meanwhile
    const char* g = reinterpret_cast<const char*>(a.gate + (int64_t)tok * a.ld_gate + head * D + half * (D / 2));
#pragma unroll
    for (int i = 0; i < D; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(g + i));
  }
  const int ctx = valid ? context(a, tok) : 0;
  int ctx_min, ctx_max;
  context_range(a, tok0, ntok, ctx_min, ctx_max);
  const Span sp = make_span(a, ctx_min, ctx_max);
  const int share = (sp.n + nsplit - 1) / nsplit;
  const int j0 = min(sp.n, split * share), n = min(sp.n, j0 + share) - j0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, SOFT);
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], SOFT);
      mbar_init(&pv_done[s], 1);
    }
    fence_mbar_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (threadIdx.x < ROWS) poison[threadIdx.x] = 0;
  if (warp == 1) {
    tmem_alloc(tmem_holder, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now: a dependent kernel that takes TMEM ahead of its own wait must not come between a CTA of this
  // grid and its columns.
  pdl_trigger();
  const uint32_t tbase = *tmem_holder;
  // the order of use: K0 K1 V0 K2 V1 ...
  auto unit_k = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto unit_v = [&](int j) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; };

  if (warp == 0) {
    const bool go = elect_one();
    Pages pages;
    for (int u = 0; u < 2 * n; ++u) {
        const bool is_k = u == 0 || ((u & 1) && u < 2 * n - 1);
        const int j = is_k ? (u + 1) / 2 : u == 2 * n - 1 ? n - 1 : u / 2 - 1;
        const int s = u % C::SLOTS;
        if (!warp_wait(&empty[s], (uint32_t)(((u / C::SLOTS) & 1) ^ 1), a.timeout_ns)) {
          if (go) report_error(a.status, kErrMbarTimeout, 322, u);
          break;
        }
        load_tile<D>(a, is_k ? &tmK : &tmV, smem + C::OFF_RING + s * C::UNIT, &full[s], sp, pages, j0 + j, j0, seq, kvh, go);
      }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      constexpr uint32_t idesc_s = idesc_dense(kFmtE4M3, kFmtE4M3, ROWS, KT);
      // B (V) MN-major; A is P's e4m3 plane, then its e5m2 plane
      constexpr uint32_t idesc_o[2] = {idesc_dense(kFmtE4M3, kFmtE4M3, ROWS, D) | (1u << 16),
                                       idesc_dense(kFmtE5M2, kFmtE4M3, ROWS, D) | (1u << 16)};
      const bool go = elect_one();
      const uint64_t q_desc = sdesc_k_sw128(smem_u32(smem + C::OFF_Q));
      const uint64_t k_desc = sdesc_k_sw128(smem_u32(smem + C::OFF_RING));
      const uint64_t v_desc = sdesc_mn(smem_u32(smem + C::OFF_RING));
      bool ok = warp_wait(q_full, 0, a.timeout_ns);
      auto wait_unit = [&](int u) { return warp_wait(&full[u % C::SLOTS], (uint32_t)((u / C::SLOTS) & 1), a.timeout_ns); };
      auto issue_s = [&](int j) -> bool {
        const int u = unit_k(j);
        if (!wait_unit(u)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)((u % C::SLOTS) * (C::UNIT >> 4));
        const uint32_t d = tbase + S_COL + (j & 1) * KT;
#pragma unroll
        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int pl = 0; pl < 2; ++pl)
              mma_ss(d, q_desc + ((pl * C::PLANE_Q + h * (ROWS * 128) + 32 * k) >> 4), kd + ((h * (KT * 128) + 32 * k) >> 4),
                     idesc_s, h > 0 || k > 0 || pl > 0, go);
        commit(&s_full[j & 1], go);
        commit(&empty[u % C::SLOTS], go);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int j = 0; ok && j < n; ++j) {
        if (j + 1 < n && !issue_s(j + 1)) { ok = false; break; }
        const int u = unit_v(j);
        if (!warp_wait(&p_full[j & 1], (uint32_t)((j >> 1) & 1), a.timeout_ns)) { ok = false; break; }
        if (!wait_unit(u)) { ok = false; break; }
        tc_fence_after();
        const uint64_t vd = v_desc + (uint64_t)((u % C::SLOTS) * (C::UNIT >> 4));
        const uint32_t p = tbase + S_COL + (j & 1) * KT;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int pl = 0; pl < 2; ++pl)
            mma_ts(tbase + O_COL, p + pl * 32 + 8 * k, vd + (k * 4096 >> 4), pl == 0 ? idesc_o[0] : idesc_o[1], j > 0 || k > 0 || pl > 0, go);
        commit(&pv_done[j & 1], go);
        commit(&empty[u % C::SLOTS], go);
      }
      if (!ok && lane == 0) report_error(a.status, kErrMbarTimeout, 323, 0);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;  // r is the TMEM lane and the tile's row
    const int seen = a.window > 0 ? ctx - a.window : 0;  // keys from here on are in the window
    auto pair_bar = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory"); };  // the two warps of these rows
    float sl2;
    {
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < QC; ++c) amax = fmaxf(amax, amax16(qraw[c]));
      red[half * ROWS + r] = amax;
      pair_bar();
      amax = fmaxf(amax, red[(half ^ 1) * ROWS + r]);
      pair_bar();  // red is used again
      const int e = amax > 0.f ? mx_exponent(amax, 448.f) : 0;
      sl2 = fmaxf(fabsf(a.scale_log2) * exp2i(max(e, -126)), 1.17549435e-38f);
      const float inv = copysignf(exp2i(-e), a.scale_log2);  // scores come out with the scale's sign
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const int pc = half * QC + c;  // 16-byte piece of the row
        uint4 hi, lo;
        split16(qraw[c], inv, hi, lo);
        uint8_t* dst = smem + C::OFF_Q + (pc / 8) * (ROWS * 128) + r * 128 + (((pc % 8) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = hi;
        *reinterpret_cast<uint4*>(dst + C::PLANE_Q) = lo;
      }
      fence_proxy_async();
      mbar_arrive(q_full);
    }
    float m_ref = -INFINITY, l = 0.f;
    const uint32_t trow = tbase + ((uint32_t)(q * 32) << 16);
    constexpr int HK = KT / 2;  // keys of this thread's half
    bool ok = true;
    // A wait that runs out is told to the other warp of the pair (a NaN in place of the maximum, which
    // never is one): both leave at the next exchange, so neither is left at their barrier.
    for (int j = 0; j < n; ++j) {
      const int s = j & 1;
      ok &= warp_wait(&s_full[s], (uint32_t)((j >> 1) & 1), a.timeout_ns);
      tc_fence_after();
      const uint32_t scol = trow + S_COL + s * KT + half * HK;
      const int key0 = sp.key(2 * (j0 + j) + half);  // of this thread's page
      const bool whole = whole_page(a, key0, ctx_min, ctx_max);
      // columns that this row sees: [first, first + count), and those before sink
      const int first = max(seen - key0, 0), sink = min(a.sinks, ctx) - key0;
      const uint32_t count = (uint32_t)max(min(ctx - key0, HK) - first, 0);
      float sv[HK];
#pragma unroll
      for (int c = 0; c < HK; c += 16) tmem_ld16(scol + c, sv + c);
      tmem_ld_wait();
      if (!whole) {
#pragma unroll
        for (int c = 0; c < HK; ++c)
          if ((uint32_t)(c - first) >= count && c >= sink) sv[c] = -INFINITY;
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < HK; ++c) m4[c & 3] = fmaxf(m4[c & 3], sv[c]);
      float tmax = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      // value rows of pages that some row does not see whole: a thread a row and column half
      const int vkey = sp.key(2 * (j0 + j) + (q >> 1));
      if (half < C::HALVES && !whole_page(a, vkey, ctx_min, ctx_max)) {
        const int u = unit_v(j);
        ok &= warp_wait(&full[u % C::SLOTS], (uint32_t)((u / C::SLOTS) & 1), a.timeout_ns);
        uint8_t* tile = smem + C::OFF_RING + (u % C::SLOTS) * C::UNIT;
        const int key = vkey + (r & (PAGE - 1));
        if (half == 0) clean_value_row<0, 1>(a, tile, r, key, tok0, ntok, poison);
        else clean_value_row<C::HALVES - 1, C::HALVES>(a, tile, r, key, tok0, ntok, poison);
        fence_proxy_async();  // the product reads the cleared rows
      }
      red[((j & 1) * 2 + half) * ROWS + r] = ok ? tmax : __int_as_float(0x7fffffff);
      pair_bar();
      const float theirs = red[((j & 1) * 2 + (half ^ 1)) * ROWS + r];
      if (!ok || theirs != theirs) {
        ok = false;
        break;
      }
      tmax = fmaxf(tmax, theirs);
      if (tmax != -INFINITY) tmax *= sl2;
      const bool need = m_ref != -INFINITY && tmax > m_ref + P_LAG;
      const float f = need ? ex2(m_ref - tmax) : 1.f;
      if (need || m_ref == -INFINITY) m_ref = tmax;
      const float off = m_ref == -INFINITY ? 0.f : P_SHIFT - m_ref;  // a row that has seen no key: exp2(-inf) = 0
      float ls[2] = {0.f, 0.f};
      float ph[HK / 4], pl[HK / 4];  // four 8-bit numbers each
#pragma unroll
      for (int c = 0; c < HK; c += 4) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = ex2(fmaf(sv[c + k], sl2, off));
        ls[0] += p[0] + p[1];
        ls[1] += p[2] + p[3];
        uint32_t h0, l0, h1, l1;
        split2p<true>(p[0], p[1], h0, l0);
        split2p<true>(p[2], p[3], h1, l1);
        ph[c / 4] = __uint_as_float(h0 | (h1 << 16));
        pl[c / 4] = __uint_as_float(l0 | (l1 << 16));
      }
      l = l * f + (ls[0] + ls[1]);
      // both threads of the row have read their scores (the exchange came after)
      const uint32_t pcol = trow + S_COL + s * KT + half * (HK / 4);
      tmem_st16(pcol, ph);
      tmem_st16(pcol + 32, pl);
      // A parity tells neighbouring phases apart only, so every phase of a barrier is looked at, here or in the
      // MMA warp, before the next but one can complete. PV(j - 2) is done (S(j) came after it): this never waits long.
      if (j >= 2) ok &= warp_wait(&pv_done[s], (uint32_t)(((j - 2) >> 1) & 1), a.timeout_ns);
      if (__any_sync(0xffffffffu, need)) {
        if (j > 0) ok &= warp_wait(&pv_done[(j - 1) & 1], (uint32_t)(((j - 1) >> 1) & 1), a.timeout_ns);
        tc_fence_after();
#pragma unroll 2
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
          float o[32];
          tmem_ld16(trow + O_COL + c, o);
          tmem_ld16(trow + O_COL + c + 16, o + 16);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= f;
          tmem_st16(trow + O_COL + c, o);
          tmem_st16(trow + O_COL + c + 16, o + 16);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }
    uint4 graw[QC][2] = {};  // the gate of this thread's half of the output, on its way during the last product
    if (nsplit == 1 && valid && a.gate != nullptr) {
      const uint4* g = reinterpret_cast<const uint4*>(a.gate + (int64_t)tok * a.ld_gate + head * D + half * (D / 2));
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        graw[c][0] = g[2 * c];
        graw[c][1] = g[2 * c + 1];
      }
    }
    if (n > 0 && ok) ok = warp_wait(&pv_done[(n - 1) & 1], (uint32_t)(((n - 1) >> 1) & 1), a.timeout_ns);
    tc_fence_after();
    if (!ok) report_error(a.status, kErrMbarTimeout, 324, r);
    const bool have = n > 0 && ok;
    asm volatile("bar.sync 5, 256;" ::: "memory");  // maxima read, poison marks written
    if (valid && poison[rt]) l = __int_as_float(0x7fffffff);
    if (ctx == 0) l = 0.f;  // sees nothing (its scores of whole tiles were not masked)
    row_l[half * ROWS + r] = have ? l : 0.f;
    if (half == 0) row_m[r] = have ? m_ref : -INFINITY;
    if (nsplit == 1) {
      pair_bar();
      l += row_l[(half ^ 1) * ROWS + r];
      const float inv = have && l != 0.f ? a.v_scale / l : 0.f;
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const int col = half * (D / 2) + 16 * c;
        float o[16];
        if (have) {
          tmem_ld16(trow + O_COL + col, o);
          tmem_ld_wait();
        }
        const __nv_bfloat16* ge = reinterpret_cast<const __nv_bfloat16*>(graw[c]);
        uint4 w[2];
        __nv_bfloat16* we = reinterpret_cast<__nv_bfloat16*>(w);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v = inv != 0.f ? o[i] * inv : 0.f;  // O of a row without weights was never written
          if (a.gate != nullptr) v *= sigmoid_f(__bfloat162float(ge[i]));
          we[i] = __float2bfloat16(v);
        }
        if (valid) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + (int64_t)tok * a.ld_out + head * D + col);
          dst[0] = w[0];
          dst[1] = w[1];
        }
      }
    } else {
      // partial results over the ring: row r's 16-byte pieces at c ^ (r & 31), so that a warp's
      // stores spread over the banks
      float* part = reinterpret_cast<float*>(smem + C::OFF_RING) + r * D;
#pragma unroll 1
      for (int c = half * (D / 2); c < (half + 1) * (D / 2) && have; c += 16) {
        float o[16];
        tmem_ld16(trow + O_COL + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(part + (((c / 4 + i) ^ (r & 31)) << 2)) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
    }
  }
  __syncwarp();  // the cluster's barrier wants whole warps
  tc_fence_before();
  if (nsplit > 1) {
    cluster_sync();
    // rows r = split, split + nsplit, ...: a warp a row, a lane four dims at a time
    const uint32_t part = smem_u32(smem + C::OFF_RING), ml = smem_u32(row_m), ll = smem_u32(row_l);
    for (int r = split + nsplit * warp; r < nrows; r += nsplit * (THREADS / 32)) {
      const float m_l = lane < nsplit ? ld_dsmem(mapa_shared(ml, (uint32_t)lane) + r * 4) : -INFINITY;
      const uint32_t lat = mapa_shared(ll, (uint32_t)(lane < nsplit ? lane : 0));
      const float l_l = lane < nsplit ? ld_dsmem(lat + r * 4) + ld_dsmem(lat + (ROWS + r) * 4) : 0.f;
      float M = l_l != 0.f ? m_l : -INFINITY;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      const float w_l = l_l == 0.f ? 0.f : m_l == -INFINITY ? 1.f : exp2f(m_l - M);
      float L = l_l == 0.f ? 0.f : w_l * l_l;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      const float inv = L != 0.f ? a.v_scale / L : 0.f;
      const int tok = tok0 + r / a.G, head = kvh * a.G + r % a.G;
      for (int c = lane; c < D / 4; c += 32) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < nsplit; ++s) {
          const float w = __shfl_sync(0xffffffffu, w_l, s);
          const float4 v = ld_dsmem_f4(mapa_shared(part, (uint32_t)s) + (r * D + ((c ^ (r & 31)) << 2)) * 4);
          if (w != 0.f) {
            acc.x += w * v.x;
            acc.y += w * v.y;
            acc.z += w * v.z;
            acc.w += w * v.w;
          }
        }
        float o[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
        const int64_t col = (int64_t)head * D + 4 * c;
        uint2 w2;
        __nv_bfloat16* we = reinterpret_cast<__nv_bfloat16*>(&w2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (a.gate != nullptr) o[i] *= sigmoid_f(__bfloat162float(a.gate[(int64_t)tok * a.ld_gate + col + i]));
          we[i] = __float2bfloat16(o[i]);
        }
        *reinterpret_cast<uint2*>(a.out + (int64_t)tok * a.ld_out + col) = w2;
      }
    }
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, C::TMEM_COLS);
  }
}

template <typename K>
static void launch_cluster(K kern, int smem, dim3 grid, int threads, const CUtensorMap& tk, const CUtensorMap& tv, const wa::Args& a) {
  TORCH_CHECK(ensure_smem_attr((const void*)kern, smem) == cudaSuccess, "window_attention: shared memory attribute");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {1, 1, grid.z};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TORCH_CHECK(cudaLaunchKernelEx(&cfg, kern, tk, tv, a) == cudaSuccess, "window_attention launch");
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
                  block_table.size(1) <= (1 << 23) && k_cache.size(0) * Hkv * wa::PAGE <= INT_MAX,
              "window_attention: sizes out of range");
  if (T == 0 || S == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
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
  a.v_scale = (float)v_scale;
  a.status = status.data_ptr<int>();
  a.scale_log2 = (float)(sm_scale * k_scale * 1.4426950408889634);
  a.timeout_ns = 1000000000ull;
  const CUtensorMap tk = tmap_u8_kmajor(k_cache.data_ptr(), k_cache.size(0) * Hkv * wa::PAGE, D, wa::PAGE);
  const CUtensorMap tv = tmap_u8_kmajor(v_cache.data_ptr(), v_cache.size(0) * Hkv * wa::PAGE, D, wa::PAGE);
  // tiles of keys that one group of rows can see at most
  const int64_t span = window > 0 ? std::min(max_ctx, window + sinks + a.max_new + 2 * wa::PAGE) : max_ctx;
  const int64_t tiles = (span + wa::KT - 1) / wa::KT;
  const int64_t sms = device_sm_count();
  const int64_t nq = (int64_t)a.max_new * a.G;  // rows of the longest sequence and one kv head
  const bool dec = nq <= wd::ROWS;
  const int64_t per = wc::ROWS / a.G;
  const int64_t groups = dec ? S : std::min(T / per + S, S * ((a.max_new + per - 1) / per));
  // CTAs of a cluster share a group's keys while all groups run at once and each CTA has a tile (the figures
  // of both sides stand at the kernels)
  int64_t nsplit = 1;
  while (nsplit < 8 && groups * Hkv * nsplit * 2 <= sms * (dec ? 2 : 1) && nsplit * 2 <= tiles) nsplit *= 2;
  const dim3 grid((unsigned)groups, (unsigned)Hkv, (unsigned)nsplit);
  TORCH_CHECK(groups <= INT_MAX, "window_attention: too many rows");
  if (dec) {
    if (D == 128) {
      if (nq <= 8) launch_cluster(window_attn_dec_kernel<128, 8>, wd::Cfg<128, 8>::SMEM, grid, wd::THREADS, tk, tv, a);
      else launch_cluster(window_attn_dec_kernel<128, 16>, wd::Cfg<128, 16>::SMEM, grid, wd::THREADS, tk, tv, a);
    } else {
      if (nq <= 8) launch_cluster(window_attn_dec_kernel<256, 8>, wd::Cfg<256, 8>::SMEM, grid, wd::THREADS, tk, tv, a);
      else launch_cluster(window_attn_dec_kernel<256, 16>, wd::Cfg<256, 16>::SMEM, grid, wd::THREADS, tk, tv, a);
    }
  } else if (D == 128) {
    launch_cluster(window_attn_chunk_kernel<128>, wc::Cfg<128>::SMEM, grid, wc::THREADS, tk, tv, a);
  } else {
    launch_cluster(window_attn_chunk_kernel<256>, wc::Cfg<256>::SMEM, grid, wc::THREADS, tk, tv, a);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace r9k
