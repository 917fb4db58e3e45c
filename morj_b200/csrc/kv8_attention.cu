// Tree attention over the 8-bit K/V cache (kv8.cuh): the mask rules of tree_attention_kernel, K and V read as e4m3
// codes and scaled per (block of 64 slots, head).
//
//   s_ij = sm_scale * (q_i . code_k[j]) * scale_k[block(j)],  p = softmax over the visible j,
//   o_i  = sum_j p_ij * scale_v[block(j)] * code_v[j],        a row that sees nothing is 0.
//
// A segment's rows are its (query, head of the group) pairs of one KV head. The host sends segments of few rows to
// rows_kernel, which converts codes where it uses them, and the others in tiles of 128 to tile_kernel, for which
// expand_kernel converts the listed pages once. It cuts the keys of a tile into parts until the SMs are filled once; parts
// leave (maximum, sum, O) in a workspace and combine_kernel joins them in a fixed order.
//
// rows_kernel: codes become FP16 by one conversion for two of them (exact), so both products run as FP16 x FP16 with FP32
// sums and the scales stay out of the operands: K's multiplies the scores, V's the probabilities (relative to the
// largest V scale met so far, so the products stay inside FP16 and O is kept in units of that scale). A query row is
// brought to [1, 2) by a power of two before it is rounded to FP16, which keeps every bit of a BF16 row that matters at
// 2^-25 of its largest element. tile_kernel: K as BF16 (exact) against the queries as they are, P and V as FP16, V's scales
// in V or, where a head's lie far apart, in P.
#include <algorithm>
#include <climits>
#include <unordered_map>
#include <vector>

#include "kv8.cuh"

namespace morj {
namespace kv8 {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int UNIT = 16;             // rows of a partial unit in the workspace
constexpr int WARPS = 4;
constexpr int STEP = 32;             // keys a warp of rows_kernel takes at a time
constexpr int T_ROWS = 128;           // rows of a tile_kernel tile
constexpr int BN = 64;                // keys it takes at a time
// Segments of at most this many rows go to rows_kernel, which reads a segment's codes once per 16 rows; the others to
// tile_kernel, behind the expansion. Both ways, 16 heads of 128, us (rows, tiles): one segment of 18 rows over 4,096 /
// 16,384 / 65,536 keys 18, 27 / 40, 72 / 123, 270, of 64 rows 26, 29 / 72, 73 / 247, 267, of 126 rows 41, 29 / 131, 74 / 482,
// 266; eight segments of 18 rows over 16,384 keys each 359, 637, over the same 16,384 keys 355, 265, of 126 rows 879, 599 and
// 872, 210. So 17 to about 64 rows over keys of their own would be better off here, and are not sent: the rule goes by rows
// alone, and over shared keys the tiles win from two 16-row tiles on.
constexpr int FEW_ROWS = 16;
// ... and all segments of a call, 16 rows at a time, whose 16-row tiles see at most this many keys together (times the KV
// heads) in at most one CTA per resident place: one launch in place of two and no expansion. 1 to 8 segments of 32 to
// 2,048 rows, heads of 64 and 128, both ways: 6 to 16 us against 9 to 22 up to it, level on the whole at twice as many,
// up to 27 against 21 at four times.
constexpr long long FEW_KEYS = 65536;
constexpr int T_CTAS = 2, T_MIN_KEYS = 256;  // resident CTAs per SM, and the fewest keys of a part: tiles
constexpr int R_CTAS = 3, R_MIN_KEYS = 256;  // ... few rows
constexpr float P_SCALE = 1024.0f;   // probabilities are rounded to FP16 as 1024 p: 2^-34 is their smallest step

// What a CTA needs to know, in one load: which rows and keys of which segment.
struct __align__(16) Item {
  int seg, r0;         // segment, its first row (row = query * G + head of the group)
  int t0, t1;          // keys [t0, t1) of the segment's list
  int unit;            // first partial unit, -1: the only part, straight to `out`
  int parts, stride;   // joins: parts, and units between them
  int tile;            // rows of the tile
  int q_start, q_len;  // the segment's queries
  int kv_base, kv_len; // its first list entry and its keys
};

// Quotients by a number the host knows, from a 32-bit reciprocal (exact for 0 <= t < 2^31): the GPU has no division, and
// some 30 instructions for one in every loader's and store loop cost up to a third of a call.
struct Quotient {
  int d, shift;
  unsigned magic;  // t / d = umulhi(t, magic) >> shift for d > 1
  // with l = ceil(log2 d): floor(t / d) = t * (floor(2^(31 + l) / d) + 1) >> (31 + l) for 0 <= t < 2^31, 2 <= d < 2^31
  explicit Quotient(int d_) : d(d_), shift(0), magic(0) {
    int l = 0;
    while (l < 31 && (1u << l) < (unsigned)d) ++l;
    if (d > 1) magic = (unsigned)((1ull << (31 + l)) / d + 1), shift = l - 1;
  }
  MORJ_DEV int of(int t) const { return d == 1 ? t : (int)(__umulhi((unsigned)t, magic) >> shift); }
};

struct Args {
  const __nv_bfloat16* q;
  const uint8_t* k;
  const float* ks;
  const uint8_t* v;
  const float* vs;
  __nv_bfloat16* out;
  const int* kv_indices;
  int n_bidir, hq, hk, window, pool_slots;
  Quotient page, group;  // by the page size, by hq / hk
  float scale_log2;
  float* ws;
};

// keys [lo, hi] query j of a segment sees (hi < lo: none)
__host__ __device__ inline void visible(int q_len, int kv_len, bool bidir, int window, int j, int* lo, int* hi) {
  const int diag = kv_len - q_len;
  if (bidir) {
    *hi = kv_len - 1;
    *lo = window > 0 ? diag + (j - (window - 1) < 0 ? j - (window - 1) : 0) : 0;
  } else {
    *hi = diag + j;
    *lo = window > 0 ? *hi - (window - 1) : 0;
  }
  if (*lo < 0) *lo = 0;
}

// slot of key t in the page with list entry `entry`
MORJ_DEV long long slot_of(const Args& a, int entry, int t) {
  return (long long)entry * a.page.d + (t - a.page.of(t) * a.page.d);
}
// where row `row` of an item's segment (query * G + head of the group) lies in q and out: its (token, head) index
MORJ_DEV size_t row_index(const Args& a, const Item& it, int h, int row) {
  const int query = a.group.of(row);
  return (size_t)(it.q_start + query) * a.hq + h * a.group.d + (row - query * a.group.d);
}

MORJ_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit elements, lane 4 i + j with elements (i, 2 j) and (i, 2 j + 1), transposed
MORJ_DEV uint32_t transposed(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
MORJ_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
MORJ_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// The power of two 2^x with |amax| / 2^x in [1, 2) (2^-126 for subnormals and 0; 1 when amax is not finite).
MORJ_DEV float row_scale(float amax) {
  const uint32_t e = __float_as_uint(amax) & 0x7f800000u;
  return e == 0x7f800000u ? 1.f : __uint_as_float(e == 0 ? 0x00800000u : e);
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows per segment (at most 16; the single-token form): the codes' bytes bound the call, so each of an SM's twelve
// warps has a group of 32 keys (8 KB) on its way while it works on another. Groups are taken in turn by the four warps of
// a CTA; keys are one lane each for their page entry (two groups ahead) and scales. A group whose slots follow one
// another comes by two TMA boxes, others are gathered by cp.async; either way the rows of K and V lie as they come,
// 16-byte units XOR-swizzled by the key, so both products read their fragments without bank conflicts: mma.m16n8k16
// leaves the order of the head dimension (q . k) and of the output columns (P V) free, and each lane takes 32 (16)
// consecutive codes of a K row and 16 (8) of a V row for D = 128 (64).
// Measured: 64 single queries over 1 to 8,048 keys of 16 heads of 128, 786 MB, 122 us back to back = 6.4 TB/s (0.98 of the
// measured copy), 143 with cold caches; 9 readout rows of 1,560 keys 16 us back to back, 22 alone (latency: page entry ->
// codes -> five groups a warp -> join). Not kept: the
// codes of K straight into an e4m3 mma against queries split in two codes (167 against 148 us at the time).
// ---------------------------------------------------------------------------------------------------------------
constexpr int R_STAGES = 2;

template <int D>
struct RSmem {
  static constexpr int SIDE = STEP * D;                     // codes of one group, K or V
  static constexpr int STAGE = 2 * SIDE;
  static constexpr int SCALE_OFF = WARPS * R_STAGES * STAGE;           // [warp][stage] K scales, V scales
  static constexpr int BAR_OFF = SCALE_OFF + WARPS * R_STAGES * 2 * STEP * 4;  // [warp][stage], then the abort flag
  static constexpr int TOTAL = BAR_OFF + WARPS * R_STAGES * 8 + 16;
  static_assert(SCALE_OFF >= WARPS * 16 * (D + 2) * 4 || D == 64, "the warps' results are joined in the rings");
  static_assert(SCALE_OFF + WARPS * R_STAGES * 2 * STEP * 4 >= WARPS * 16 * (D + 2) * 4, "... or in them and the scales");
};

MORJ_DEV void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// one arrival of this thread on `bar` once its cp.asyncs so far have landed
MORJ_DEV void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
MORJ_DEV void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A whole warp waits for a barrier's phase. Every lane polls (one broadcast read) and the warp goes on when all have seen
// it: a lane polling for the others costs the shuffle that tells them as well.
MORJ_DEV bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  unsigned long long t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (__all_sync(0xffffffffu, mbar_test_suspend(bar, parity, 20000))) return true;
    if ((i & 63) == 0) {
      const unsigned long long now = global_ns();
      if (t0 == 0) t0 = now;
      const bool late = now - t0 > kWaitLimitNs;
      if (late) *abort = 1, report(kErrTimeoutAttention);
      if (__any_sync(0xffffffffu, late || *abort)) return false;
    }
  }
}
MORJ_DEV void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
MORJ_DEV uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
MORJ_DEV uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
MORJ_DEV float lds4(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// byte offset of 16-byte unit u of key k's row in a group (the 128-byte, for D = 64 the 64-byte swizzle of TMA)
template <int D>
MORJ_DEV uint32_t unit_at(int k, int u) {
  return D == 128 ? (uint32_t)(k * 128 + ((u ^ (k & 7)) << 4)) : (uint32_t)(k * 64 + ((u ^ ((k >> 1) & 3)) << 4));
}

// 16-byte unit u of row r's FP32 results: where eight lanes of two column runs and four rows write, eight bank groups
template <int D>
MORJ_DEV int spread(int r, int u) {
  const int x = (r >> 1) & 3;
  return u ^ (D == 128 ? x : (x & 1) * 4 + (x >> 1));
}

// ROWS = 8 or 16 rows per tile. Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: the MMA's 16 rows are
// keys and output columns, of which there are always enough, and its 8 columns the tile's rows (two MMAs for 16). With
// the rows on the 16 side half of every MMA and of its sums was empty for 8 of them: 148 us for 64 single queries.
template <int D, int ROWS>
__global__ void __launch_bounds__(WARPS * 32, 3)
    rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a,
                const Item* __restrict__ items) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  using L = RSmem<D>;
  constexpr int KS = D / 16;       // MMA depth steps of q . k
  constexpr int NT = D / 16;       // 16-column output tiles
  constexpr int HALVES = ROWS / 8;
  constexpr int KRUN = D / 4;      // consecutive codes of a key one lane reads of K
  constexpr int VRUN = D / 8;      // ... and of V
  constexpr int LPR = D / 16;      // 16-byte units of a row
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // the swizzle follows the address
    if (threadIdx.x == 0) report(kErrBadAlignment);
    return;
  }

  const Item it = items[blockIdx.x / a.hk];
  const int h = blockIdx.x % a.hk;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, c4 = lane % 4;
  const bool bidir = it.seg < a.n_bidir;
  const int G = a.hq / a.hk, n_rows = it.q_len * G;
  const int t_end = it.t1;

  // ---- the warp's groups: keys [it.t0 + 32 (warp + 4 i), + 32)
  const uint32_t ring = smem_u32(smem) + warp * R_STAGES * L::STAGE;
  const uint32_t scale_at = smem_u32(smem) + L::SCALE_OFF + warp * R_STAGES * (2 * STEP * 4);
  const uint32_t bars = smem_u32(smem) + L::BAR_OFF + warp * R_STAGES * 8;
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::BAR_OFF + WARPS * R_STAGES * 8);
  if (lane == 0) {
    for (int i = 0; i < R_STAGES; ++i) mbar_init(bars + 8 * i, 32);
    if (warp == 0) *abort = 0;
    fence_mbar_init();
    tma_prefetch(&k_map);
    tma_prefetch(&v_map);
  }
  __syncthreads();
  const int t_first = it.t0 + warp * STEP;
  const int groups = t_first < t_end ? (t_end - t_first + WARPS * STEP - 1) / (WARPS * STEP) : 0;
  const int* list = a.kv_indices + it.kv_base;
  const unsigned row_bytes = (unsigned)a.hk * D;
  auto key = [&](int i) { return t_first + i * (WARPS * STEP) + lane; };
  auto entry = [&](int i) { return i < groups ? __ldg(list + a.page.of(min(key(i), t_end - 1))) : 0; };
  auto issue = [&](int i, int e) {  // ask for group i; e: the lane's page entry
    if (i >= groups) return;
    const int place = i % R_STAGES;
    const uint32_t st = ring + place * L::STAGE, bar = bars + 8 * place;
    const int t = key(i);
    const long long at = slot_of(a, e, min(t, t_end - 1));
    const bool in_pool = at >= 0 && at < a.pool_slots;
    if (!in_pool) report(kErrBadIndex);
    const bool ok = t < t_end && in_pool;
    const unsigned slot = in_pool ? (unsigned)at : 0u;
    const size_t si = (size_t)(slot >> BLOCK_SHIFT) * a.hk + h;
    const uint32_t sc = scale_at + place * (2 * STEP * 4) + lane * 4;
    cp_async4(sc, a.ks + si, ok ? 4u : 0u);
    cp_async4(sc + STEP * 4, a.vs + si, ok ? 4u : 0u);
    const unsigned first = __shfl_sync(0xffffffffu, slot, 0);
    if (__all_sync(0xffffffffu, ok && slot == first + lane)) {
      if (lane == 0) {
        mbar_expect_tx(bar, L::STAGE);
        tma_load_3d(st, &k_map, bar, 0, h, (int)first);
        tma_load_3d(st + L::SIDE, &v_map, bar, 0, h, (int)first);
      }
    } else {
      const unsigned there = __ballot_sync(0xffffffffu, ok);
      const size_t unit = (size_t)h * D + (lane % LPR) * 16;
#pragma unroll 2
      for (int k = lane / LPR; k < STEP; k += 32 / LPR) {
        const unsigned long long off = (unsigned long long)__shfl_sync(0xffffffffu, slot, k) * row_bytes + unit;
        const uint32_t n = (there >> k) & 1 ? 16u : 0u;
        cp_async16(st + unit_at<D>(k, lane % LPR), a.k + off, n);
        cp_async16(st + L::SIDE + unit_at<D>(k, lane % LPR), a.v + off, n);
      }
    }
    cp_async_arrive(bar);
  };
  int e_next = entry(0);
#pragma unroll 1
  for (int i = 0; i < R_STAGES - 1; ++i) {
    const int e = e_next;
    e_next = entry(i + 1);
    issue(i, e);
  }

  // ---- Q^T fragments: rows r0 + g (+ 8), this lane's run of the head dimension
  uint32_t qf[HALVES][KS][2];
  float qs[HALVES];
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    const int r = it.r0 + g + 8 * b;
    uint4 raw[KRUN / 8];
#pragma unroll
    for (int i = 0; i < KRUN / 8; ++i) raw[i] = make_uint4(0, 0, 0, 0);
    if (r < n_rows) {
      const uint4* src = reinterpret_cast<const uint4*>(
          a.q + row_index(a, it, h, r) * D + c4 * KRUN);
#pragma unroll
      for (int i = 0; i < KRUN / 8; ++i) raw[i] = __ldg(src + i);
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < KRUN / 8; ++i) {
      float x[8];
      unpack8(raw[i], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    qs[b] = row_scale(amax);
    const float inv = 1.f / qs[b];
    qs[b] *= a.scale_log2;
#pragma unroll
    for (int i = 0; i < KRUN / 8; ++i) {
      float x[8];
      unpack8(raw[i], x);
      qf[b][2 * i][0] = pack_f16x2(x[0] * inv, x[1] * inv), qf[b][2 * i][1] = pack_f16x2(x[2] * inv, x[3] * inv);
      qf[b][2 * i + 1][0] = pack_f16x2(x[4] * inv, x[5] * inv), qf[b][2 * i + 1][1] = pack_f16x2(x[6] * inv, x[7] * inv);
    }
  }

  // ---- this lane's rows of the results: r0 + 2 c4, the next one (+ 8)
  float row_qs[HALVES][2];
  int lo[HALVES][2], hi[HALVES][2];
  float o[HALVES][NT][4];  // (column g VRUN + 2 tile, row 0), (.., row 1), (the next column, row 0), (.., row 1)
  float m[HALVES][2], l[HALVES][2];
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = it.r0 + 2 * c4 + e + 8 * b;
      row_qs[b][e] = __shfl_sync(0xffffffffu, qs[b], 4 * (2 * c4 + e));
      lo[b][e] = INT_MAX, hi[b][e] = -1;
      if (r < n_rows) {
        visible(it.q_len, it.kv_len, bidir, a.window, a.group.of(r), &lo[b][e], &hi[b][e]);
        hi[b][e] = min(hi[b][e], t_end - 1);
      }
      m[b][e] = -INFINITY, l[b][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) o[b][j][0] = o[b][j][1] = o[b][j][2] = o[b][j][3] = 0.f;
  }
  float vref = 0.f;  // the largest V scale met: O is in units of vref / P_SCALE

#pragma unroll 1
  for (int i = 0; i < groups; ++i) {
    __syncwarp();  // every lane is done with the group whose place is refilled now
    {
      const int e = e_next;
      e_next = entry(i + R_STAGES);
      issue(i + R_STAGES - 1, e);
    }
    const int place = i % R_STAGES;
    if (!warp_wait(bars + 8 * place, (i / R_STAGES) & 1, abort)) {
      // (given up, perhaps because another warp did: what this warp asked for, group i too, must land before the CTA
      // writes over the rings and leaves)
      for (int x = i; x < min(groups, i + R_STAGES); ++x)
        if (lane == 0) mbar_wait_landed(bars + 8 * (x % R_STAGES), (x / R_STAGES) & 1);
      break;
    }
    const uint32_t st = ring + place * L::STAGE;
    const uint32_t kf_at = scale_at + place * (2 * STEP * 4), vf_at = kf_at + STEP * 4;
    const int base = t_first + i * (WARPS * STEP);
    // V scales: O moves to the new unit when a larger one appears (as unsigned bits a NaN is the largest)
    const float vmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lds4(vf_at + lane * 4))));
    float unit = 1.f;  // old unit / new unit
    if (!(vmax <= vref)) {
      unit = vref / vmax;
      vref = vmax;
    }
    const float inv_v = vref != 0.f ? P_SCALE / vref : 0.f;
    // scores of keys base + 16 half + g (+ 8), this lane's rows
    float s[2][HALVES][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int b = 0; b < HALVES; ++b) s[half][b][0] = s[half][b][1] = s[half][b][2] = s[half][b][3] = 0.f;
      uint32_t w[2][KRUN / 4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int u = 0; u < KRUN / 16; ++u) {
          const uint4 x = lds16(st + unit_at<D>(half * 16 + e * 8 + g, c4 * (KRUN / 16) + u));
          w[e][4 * u] = x.x, w[e][4 * u + 1] = x.y, w[e][4 * u + 2] = x.z, w[e][4 * u + 3] = x.w;
        }
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const uint32_t a0 = codes2_f16(w[0][x]), a1 = codes2_f16(w[1][x]);
        const uint32_t a2 = codes2_f16(w[0][x] >> 16), a3 = codes2_f16(w[1][x] >> 16);
#pragma unroll
        for (int b = 0; b < HALVES; ++b) mma_f16(s[half][b], a0, a1, a2, a3, qf[b][x][0], qf[b][x][1]);
      }
    }
    float mx[HALVES][2];
#pragma unroll
    for (int b = 0; b < HALVES; ++b) mx[b][0] = mx[b][1] = -INFINITY;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int k8 = 0; k8 < 2; ++k8) {
        const int k = half * 16 + k8 * 8 + g, t = base + k;
        const float f = lds4(kf_at + k * 4);
#pragma unroll
        for (int b = 0; b < HALVES; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[half][b][2 * k8 + e];
            x = t >= lo[b][e] && t <= hi[b][e] ? x * (f * row_qs[b][e]) : -INFINITY;
            mx[b][e] = max_nan(mx[b][e], x);
          }
      }
    float alpha[HALVES][2];
    bool same = true;
#pragma unroll
    for (int b = 0; b < HALVES; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mx[b][e] = max_nan(mx[b][e], __shfl_xor_sync(0xffffffffu, mx[b][e], x));
        const float now = max_nan(m[b][e], mx[b][e]);
        alpha[b][e] = m[b][e] == -INFINITY ? 0.f : fast_exp2(m[b][e] - now);
        m[b][e] = now;
        l[b][e] *= alpha[b][e];
        alpha[b][e] *= unit;
        same = same && alpha[b][e] == 1.f;
      }
    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
      for (int b = 0; b < HALVES; ++b)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          o[b][j][0] *= alpha[b][0], o[b][j][1] *= alpha[b][1];
          o[b][j][2] *= alpha[b][0], o[b][j][3] *= alpha[b][1];
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t pf[HALVES][2];
#pragma unroll
      for (int k8 = 0; k8 < 2; ++k8) {
        const float f = lds4(vf_at + (half * 16 + k8 * 8 + g) * 4) * inv_v;
#pragma unroll
        for (int b = 0; b < HALVES; ++b) {
          float p[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            p[e] = fast_exp2(s[half][b][2 * k8 + e] - (m[b][e] == -INFINITY ? 0.f : m[b][e]));
            l[b][e] += p[e];
          }
          pf[b][k8] = transposed(pack_f16x2(p[0] * f, p[1] * f));
        }
      }
      // V of keys c4 * 2 + {0, 1, 8, 9}, output columns g * VRUN ..: four columns a word, paired per column
      uint32_t vw[4][VRUN / 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = half * 16 + (e >> 1) * 8 + c4 * 2 + (e & 1);
        if constexpr (VRUN == 16) {
          const uint4 x = lds16(st + L::SIDE + unit_at<D>(k, g));
          vw[e][0] = x.x, vw[e][1] = x.y, vw[e][2] = x.z, vw[e][3] = x.w;
        } else {
          const uint2 x = lds8(st + L::SIDE + unit_at<D>(k, g >> 1) + (g & 1) * 8);
          vw[e][0] = x.x, vw[e][1] = x.y;
        }
      }
#pragma unroll
      for (int w = 0; w < VRUN / 4; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t lo2 = prmt(vw[0][w], vw[1][w], e ? 0x7362 : 0x5140);
          const uint32_t hi2 = prmt(vw[2][w], vw[3][w], e ? 0x7362 : 0x5140);
          const uint32_t a0 = codes2_f16(lo2), a1 = codes2_f16(lo2 >> 16);
          const uint32_t a2 = codes2_f16(hi2), a3 = codes2_f16(hi2 >> 16);
#pragma unroll
          for (int b = 0; b < HALVES; ++b) mma_f16(o[b][2 * w + e], a0, a1, a2, a3, pf[b][0], pf[b][1]);
        }
    }
  }

  // the four warps' results, joined in the rings
  __syncthreads();
  float* sh_o = reinterpret_cast<float*>(smem);        // [warp][row][D]
  float* sh_m = sh_o + WARPS * ROWS * D;               // [warp][row]
  float* sh_l = sh_m + WARPS * ROWS;
  const float scale_o = vref / P_SCALE;
#pragma unroll
  for (int b = 0; b < HALVES; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], x);
      const int r = 2 * c4 + e + 8 * b;
      if (g == 0) sh_m[warp * ROWS + r] = m[b][e], sh_l[warp * ROWS + r] = l[b][e];
      const uint32_t row_at = smem_u32(sh_o) + (warp * ROWS + r) * (D * 4);
#pragma unroll
      for (int q = 0; q < VRUN / 4; ++q)
        sts16(row_at + spread<D>(r, g * (VRUN / 4) + q) * 16, __float_as_uint(o[b][2 * q][e] * scale_o),
              __float_as_uint(o[b][2 * q][2 + e] * scale_o), __float_as_uint(o[b][2 * q + 1][e] * scale_o),
              __float_as_uint(o[b][2 * q + 1][2 + e] * scale_o));
    }
  __syncthreads();
  float* part = it.unit < 0 ? nullptr : a.ws + ((size_t)it.unit * a.hk + h) * (UNIT * (D + 2));
#pragma unroll 1
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += WARPS * 32) {
    const int r = i / (D / 4), u = i % (D / 4);
    if (it.r0 + r >= n_rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, sh_m[w * ROWS + r]);
    float ll = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = sh_m[w * ROWS + r];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - mm);
      ll += f * sh_l[w * ROWS + r];
      const uint4 v = lds16(smem_u32(sh_o) + (w * ROWS + r) * (D * 4) + spread<D>(r, u) * 16);
      x[0] += f * __uint_as_float(v.x), x[1] += f * __uint_as_float(v.y);
      x[2] += f * __uint_as_float(v.z), x[3] += f * __uint_as_float(v.w);
    }
    if (part) {
      if (u == 0) part[r] = mm, part[UNIT + r] = ll;
      reinterpret_cast<float4*>(part + 2 * UNIT + r * D)[u] = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = ll == 0.f ? 0.f : x[e] / ll;
      *reinterpret_cast<uint2*>(a.out + row_index(a, it, h, it.r0 + r) * D + 4 * u) =
          make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Many rows per segment: the pages these segments list are expanded once to 16 bits, then attended to on tcgen05.
//
// expand_kernel: every distinct listed slot in the order the lists name them, K as BF16 (code * scale is exact there, and
// queries are BF16), V as FP16(code * scale / ref) with the head's largest scale among them, so that probabilities can be
// FP16 too (11 bits). That is exact while the head's scales lie within 2^15 of one another (the smallest code is 2^-9, the
// smallest FP16 2^-24). Where they do not, V is expanded as its codes, and tile_kernel takes each key's scale into its
// probability, relative to the largest one its tile has met, so that what other segments hold costs a segment no precision.
// A key is used by every 128-row tile that sees it:
// expanding costs 3 bytes of traffic per code once (35.7 M codes, the 8,704 tokens of a 16-head layer, K and V), where
// converting in the tile loaders (built and measured) cost each tile the conversion, the address arithmetic and the
// instruction cache: 130 us on the op-level tree (2048 + 8 x 64) against 73 now.
// ---------------------------------------------------------------------------------------------------------------
// A CTA takes 64 slots of a head's K or V. Three steps of loads that depend on one another (page, codes, convert), each
// asked for at once, and many CTAs an SM: one warp's share with the lookups inline took 27 us for those 35.7 M codes.
constexpr int E_THREADS = 128;
constexpr float EXACT_SPREAD = 32768.f;  // scales of a head within this factor: V relative to the largest is exact in FP16
constexpr float SCALES_APART = -1.f;     // a head's reference where they are not: V is its codes

template <int D>
__global__ void __launch_bounds__(E_THREADS, 12) expand_kernel(const Args a, const int2* __restrict__ pages,
                                                               int n_slots, const int* __restrict__ blocks,
                                                               int n_blocks, uint16_t* __restrict__ k_out,
                                                               uint16_t* __restrict__ v_out, float* __restrict__ refs) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  constexpr int LPR = D / 8;              // lanes per row: 8 codes in, 16 bytes out
  constexpr int ROWS = E_THREADS / LPR;   // rows per iteration of the CTA
  constexpr int N = BN / ROWS;
  __shared__ int slots[BN];               // of the pool; -1: nothing listed (zeros)
  __shared__ float factor[BN];
  __shared__ float red[E_THREADS / 32], low[E_THREADS / 32];
  const int h = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const bool is_v = blockIdx.z;
  const int t0 = blockIdx.x * BN, part = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const float* scales = (is_v ? a.vs : a.ks) + h;
  const unsigned row_bytes = (unsigned)a.hk * D;
  float sc = 0.f;
  if (threadIdx.x < BN) {
    const int t = t0 + threadIdx.x;
    int slot = -1;
    if (t < n_slots) {
      const int p = a.page.of(t), at = t - p * a.page.d;
      const int2 page = __ldg(pages + p);  // (page of the pool, its slots up to the last one seen: the rest is zeros)
      const long long s = (long long)page.x * a.page.d + at;
      if (at < page.y) {
        if (s < a.pool_slots)
          slot = (int)s;
        else
          report(kErrBadIndex);
      }
    }
    slots[threadIdx.x] = slot;
    if (slot >= 0) sc = __ldg(scales + (size_t)(slot >> BLOCK_SHIFT) * a.hk);
  }
  __syncthreads();
  const uint8_t* codes = (is_v ? a.v : a.k) + (size_t)h * D + part * 8;
  uint2 w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = slots[i * ROWS + r0];
    w[i] = make_uint2(0, 0);
    if (slot >= 0) w[i] = __ldg(reinterpret_cast<const uint2*>(codes + (size_t)slot * row_bytes));
  }
  float inv = 1.f;
  if (is_v) {  // V's largest scale of the head (every CTA of the head finds the same)
    float vr = 0.f, vm = INFINITY;  // ... and its smallest (0 and NaN mark blocks nothing was stored in)
    for (int i = threadIdx.x; i < n_blocks; i += E_THREADS) {
      const int b = __ldg(blocks + i);
      if (b >= 0 && (long long)b * BLOCK < a.pool_slots) {  // (else: reported)
        const float x = __ldg(a.vs + (size_t)b * a.hk + h);
        vr = fmaxf(vr, x);
        if (x > 0.f) vm = fminf(vm, x);
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
      vr = fmaxf(vr, __shfl_xor_sync(0xffffffffu, vr, x));
      vm = fminf(vm, __shfl_xor_sync(0xffffffffu, vm, x));
    }
    if (lane == 0) red[warp] = vr, low[warp] = vm;
    __syncthreads();
    vr = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    vm = fminf(fminf(low[0], low[1]), fminf(low[2], low[3]));
    const bool apart = vr > vm * EXACT_SPREAD;
    if (blockIdx.x == 0 && threadIdx.x == 0) refs[h] = apart ? SCALES_APART : vr;
    if (apart)
      sc = 1.f;
    else if (vr > 0.f)
      inv = 1.f / vr;
  }
  if (threadIdx.x < BN) factor[threadIdx.x] = sc * inv;
  __syncthreads();
  uint16_t* out = (is_v ? v_out : k_out) + (size_t)h * D + part * 8;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = i * ROWS + r0;
    if (t0 + r >= n_slots) break;
    const float f = factor[r];
    const float2 x0 = codes2_f32(w[i].x & 0xffffu), x1 = codes2_f32(w[i].x >> 16);
    const float2 x2 = codes2_f32(w[i].y & 0xffffu), x3 = codes2_f32(w[i].y >> 16);
    uint4 u;
    if (is_v)
      u = make_uint4(pack_f16x2(x0.x * f, x0.y * f), pack_f16x2(x1.x * f, x1.y * f), pack_f16x2(x2.x * f, x2.y * f),
                     pack_f16x2(x3.x * f, x3.y * f));
    else
      u = make_uint4(pack_bf16x2(x0.x * f, x0.y * f), pack_bf16x2(x1.x * f, x1.y * f), pack_bf16x2(x2.x * f, x2.y * f),
                     pack_bf16x2(x3.x * f, x3.y * f));
    *reinterpret_cast<uint4*>(out + (size_t)(t0 + r) * row_bytes) = u;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// tile_kernel: 128 rows of a segment and KV head against 64 keys at a time, on tcgen05 (BF16 scores, FP16 P V, FP32 in
// TMEM).
//   warps 0, 2  K and V loaders: a chunk whose 64 expanded slots are consecutive by TMA, others gathered by cp.async
//   warp 1      MMA issuer (one thread): S_c = Q K_c^T into TMEM buffer c % 2, O += P_c V_c with P read from TMEM
//   warp 3      Q rows by cp.async (any hq / hk)
//   warps 4-7   softmax (thread = row): mask, online maximum and sum, P as FP16 over its own scores in TMEM, the final
//               O / l or the part's (maximum, sum, O), staged through shared memory to store whole rows
// The pipeline is tree_attention_kernel's (S and P double-buffered in TMEM, a K buffer free once its S is complete, a V
// buffer once its P V is, two CTAs per SM); what it lacks there is the parts of a key range and rows that see nothing.
// Bound by the softmax of a chunk, which one warpgroup takes through its steps in turn while the chunk's MMAs wait for it.
// Clocks read in the softmax warps (which cost 5-8% themselves), 8 x 64 rows on 8,192 keys: 1,700 cycles a chunk, of which
// 820 for the exponentials with sum and packing, 260 for mask and maximum (460 at the ragged chunks of a window), 415 waiting
// for S, 115 for the rescale's vote and the rare rescale, 100 for TMEM loads and stores. Two CTAs share an SM, so one chunk
// every 850 cycles, where the MMAs need 640 (N = 64 reads shared memory for 48 of them per 16-deep step, not 32). On
// top come 10,000 cycles to a CTA's first S and 7,500 to store its O, of 128,000, and here only 256 CTAs for 296 places.
// 51.8 GFLOP (2048 + 8 x 64 rows, 32 heads of 128) in a call of 71 us back to back = 725 TFLOP/s with the expansion.
// Measured and not kept: the MMAs by a whole warp with one lane's predicate, or elected (30-60% slower), P handed over in
// halves (1-3% slower), keys cut further to even out the CTAs (5% slower, the joins cost more).
// ---------------------------------------------------------------------------------------------------------------
constexpr int T_THREADS = 256;
constexpr int T_TMEM_COLS = 256;        // S/P buffers at columns [0, 64) and [64, 128), O at [128, 128 + D)
constexpr float T_RESCALE_LOG2 = 8.0f;  // O is rescaled when a row's maximum grows by more than 2^8 (2^4: 3-4% slower),
constexpr float T_P_LOG2 = 7.0f;        // so that 2^7 p <= 2^15 stays inside FP16: p's smallest step is 2^-31

template <int D>
struct TSmem {
  static constexpr int Q_BYTES = T_ROWS * D * 2;
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int K_OFF = Q_BYTES;               // 2 buffers
  static constexpr int V_OFF = K_OFF + 2 * KV_BYTES;  // 2 buffers
  static constexpr int BAR_OFF = V_OFF + 2 * KV_BYTES;
  // barriers: q_full, k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], done; TMEM slot, abort flag
  static constexpr int TOTAL = BAR_OFF + 128;
};

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major = false) {
  return (1u << 4)  // D: FP32; A and B: FP16 (0)
         | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// One loader warp fills buffer `dst` with the expanded rows of keys [t0, t0 + BN) and completes `full`. s0, s1: the
// expanded slots of this lane's keys t0 + 2 lane and the next, -1 outside the part. Where the slots follow one another the
// box around them is loaded. Of K also where only those inside the part do: the box's other rows are keys the softmax
// masks, whatever they hold. Of V only when the whole chunk is inside: the product with a masked key's probability 0 is NaN
// where its value is, so the first and last chunk of a part are gathered, with zeros outside.
template <int D>
MORJ_DEV void load_chunk(uint32_t dst, uint32_t full, const CUtensorMap* map, const uint16_t* __restrict__ pool, bool whole,
                         int s0, int s1, int hk, int h, int lane) {
  const unsigned any = __ballot_sync(0xffffffffu, s0 >= 0 || s1 >= 0);
  const int mine = s0 >= 0 ? s0 - 2 * lane : s1 - 2 * lane - 1;  // slot of key t0 if the run holds
  const int first = __shfl_sync(0xffffffffu, mine, any ? __ffs(any) - 1 : 0);
  if (__all_sync(0xffffffffu, (s0 < 0 ? !whole : s0 == first + 2 * lane) && (s1 < 0 ? !whole : s1 == first + 2 * lane + 1))) {
    if (lane == 0) {
      mbar_arrive_expect_tx(full, BN * D * 2);
#pragma unroll
      for (int half = 0; half < D / 64; ++half) tma_load_3d(dst + half * (BN * 128), map, full, half * 64, h, first);
    }
    return;
  }
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) {
    const int k = 2 * lane + k2, slot = k2 ? s1 : s0;
    const uint16_t* src = pool + (slot >= 0 ? ((size_t)slot * hk + h) * D : 0);
#pragma unroll 4
    for (int u = 0; u < D / 8; ++u)
      cp_async16(dst + (uint32_t)((u >> 3) * (BN * 128)) + sw128_offset(k, u & 7), src + u * 8, slot >= 0 ? 16u : 0u);
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
}

// The softmax warps' walk over a part's chunks: a thread's row, its visible keys [lo, hi], running maximum m_used and sum
// l_run (in units of 2^-T_P_LOG2, as P and O). False when a wait ran out.
// APART: the V scales of the head lie far apart and V is its codes: each probability is multiplied by its key's V scale
// relative to `vr`, the largest one the part has met so far, in units of which O is.
struct ChunkSide {
  uint32_t t_lane, s_full, p_full, pv_done;
  int t_begin, t0, t_stop, n_chunks, lo, hi;
  float scale;  // scores times it are in the log2 domain (> 0)
  volatile int* abort;
};
template <int D, bool APART>
MORJ_DEV bool softmax_chunks(const Args& a, int h, const int2* pages, const int* places, int n_slots, const ChunkSide& x,
                             float& m_used, float& l_run, float& vr) {
  const int lane = threadIdx.x % 32;
  const float scale = x.scale;
  auto scale_of = [&](int t) {  // V's of key t, 0 outside the part
    if (t < x.t0 || t >= x.t_stop) return 0.f;
    const int place = __ldg(places + a.page.of(t));
    if ((long long)place * a.page.d >= n_slots) return 0.f;  // (reported by the loaders, as is a slot outside the pool)
    const long long s = slot_of(a, __ldg(pages + place).x, t);
    return s < a.pool_slots ? __ldg(a.vs + (size_t)(s >> BLOCK_SHIFT) * a.hk + h) : 0.f;
  };
  for (int c = 0; c < x.n_chunks; ++c) {
    const int b = c & 1;
    if (!warp_wait(x.s_full + 8 * b, (c >> 1) & 1, x.abort)) return false;
    tc_fence_after();
    uint32_t sr[2][32];
    tmem_ld32(x.t_lane + b * BN, sr[0]);
    tmem_ld32(x.t_lane + b * BN + 32, sr[1]);
    tmem_wait_ld();
    const int t0 = x.t_begin + c * BN;
    // (the maximum and the sum run over 8 independent partials: short dependency chains)
    float m8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m8[i] = -INFINITY;
    if (__all_sync(0xffffffffu, t0 >= x.lo && t0 + BN - 1 <= x.hi)) {
#pragma unroll
      for (int j = 0; j < BN; j += 2)
        m8[(j >> 1) & 7] = max3f(m8[(j >> 1) & 7], __uint_as_float(sr[j >> 5][j & 31]),
                                 __uint_as_float(sr[(j + 1) >> 5][(j + 1) & 31]));
    } else {
#pragma unroll
      for (int j = 0; j < BN; ++j) {
        const int t = t0 + j;
        const float v = (t >= x.lo && t <= x.hi) ? __uint_as_float(sr[j >> 5][j & 31]) : -INFINITY;
        sr[j >> 5][j & 31] = __float_as_uint(v);
        m8[j & 7] = fmaxf(m8[j & 7], v);
      }
    }
    const float mx = scale * fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                                   fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
    float alpha = 1.f;
    if (mx > m_used + T_RESCALE_LOG2 || m_used == -INFINITY) {
      if (m_used != -INFINITY) alpha = fast_exp2(m_used - mx);
      if (mx != -INFINITY) m_used = mx;
    }
    l_run *= alpha;
    float f0 = 1.f, f1 = 1.f;  // APART: V scales of keys t0 + lane and t0 + 32 + lane relative to vr
    if constexpr (APART) {
      f0 = scale_of(t0 + lane), f1 = scale_of(t0 + 32 + lane);
      // (as unsigned bits a NaN is the largest)
      const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, max(__float_as_uint(f0), __float_as_uint(f1))));
      if (!(most <= vr)) {
        alpha *= vr / most;  // (l_run is past it)
        vr = most;
      }
      const float inv = vr != 0.f ? 1.f / vr : 0.f;
      f0 *= inv, f1 *= inv;
    }
    // exp2(-inf) = 0 for masked keys; a row with no visible key yet keeps m_used = -inf and p = 0
    const float shift = m_used == -INFINITY ? 0.f : T_P_LOG2 - m_used;
    // scores in pairs: one packed FMA scales and shifts two of them, one packed add sums two probabilities
    const uint64_t scale2 = f2_pack(scale, scale), shift2 = f2_pack(shift, shift);
    uint64_t s4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s4[i] = f2_pack(0.f, 0.f);
    uint32_t pk[BN / 2];
    if constexpr (!APART) {
#pragma unroll
      for (int j = 0; j < BN; j += 2) {
        float y0, y1;
        f2_unpack(f2_fma(f2_bits(sr[j >> 5][j & 31], sr[(j + 1) >> 5][(j + 1) & 31]), scale2, shift2), y0, y1);
        const float p0 = fast_exp2(y0), p1 = fast_exp2(y1);
        s4[(j >> 1) & 3] = f2_add(s4[(j >> 1) & 3], f2_pack(p0, p1));
        pk[j / 2] = pack_f16x2(p0, p1);
      }
    } else {  // (the sum takes p, the product p times its key's scale)
#pragma unroll
      for (int j = 0; j < BN; j += 2) {
        const float p0 = fast_exp2(fmaf(__uint_as_float(sr[j >> 5][j & 31]), scale, shift));
        const float p1 = fast_exp2(fmaf(__uint_as_float(sr[(j + 1) >> 5][(j + 1) & 31]), scale, shift));
        s4[(j >> 1) & 3] = f2_add(s4[(j >> 1) & 3], f2_pack(p0, p1));
        const float f = j < 32 ? f0 : f1;
        pk[j / 2] = pack_f16x2(p0 * __shfl_sync(0xffffffffu, f, j & 31), p1 * __shfl_sync(0xffffffffu, f, (j + 1) & 31));
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float u, v;
      f2_unpack(s4[i], u, v);
      sum += u + v;
    }
    l_run += sum;
    // a rescale of O waits until the previous chunk's PV has completed (the next one needs this chunk's P)
    if (c >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
      if (!warp_wait(x.pv_done + 8 * (b ^ 1), ((c - 1) >> 1) & 1, x.abort)) return false;
      tc_fence_after();
#pragma unroll 1
      for (int col = 0; col < D; col += 32) {
        uint32_t o[32];
        tmem_ld32(x.t_lane + 128 + col, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st32(x.t_lane + 128 + col, o);
      }
    }
    tmem_st32(x.t_lane + b * BN, pk);  // P_c over the first 32 columns of S_c
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(x.p_full + 8 * b);
  }
  return true;
}
// (A call of its own costs the usual walk 0.7%; inlined, its code and registers cost it 3-6%. Static, so that it keeps to its
// callers' 128 registers.)
template <int D>
static __device__ __noinline__ bool softmax_chunks_apart(const Args& a, int h, const int2* pages, const int* places,
                                                         int n_slots, const ChunkSide& x, float& m_used, float& l_run,
                                                         float& vr) {
  return softmax_chunks<D, true>(a, h, pages, places, n_slots, x, m_used, l_run, vr);
}

template <int D>
__global__ void __launch_bounds__(T_THREADS, 2)
    tile_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                const __grid_constant__ Args a,
                const Item* __restrict__ items, const int2* __restrict__ pages, const int* __restrict__ list,
                const uint16_t* __restrict__ k_pool, const uint16_t* __restrict__ v_pool, int n_slots,
                const float* __restrict__ refs) {
  pdl_wait();  // the previous kernel on the stream has completed
  using L = TSmem<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  if (sbase & 1023) {  // the swizzled operand tiles need 1024-byte alignment
    if (threadIdx.x == 0) report(kErrBadAlignment);
    return;
  }
  const uint32_t bar0 = sbase + L::BAR_OFF;
  const uint32_t q_full = bar0, k_full = bar0 + 8, v_full = bar0 + 24;
  const uint32_t s_full = bar0 + 40, p_full = bar0 + 56, pv_done = bar0 + 72, done = bar0 + 88;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::BAR_OFF + 96);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::BAR_OFF + 100);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Item it = items[blockIdx.x / a.hk];
  const int h = blockIdx.x % a.hk;  // (the KV head is the fast index: every head of the longest item starts first)
  const int G = a.hq / a.hk, n_rows = it.q_len * G;
  const bool bidir = it.seg < a.n_bidir;
  const int t_begin = it.t0 - it.t0 % BN;  // chunks line up with 64-slot pages
  const int t_stop = it.t1;
  const int n_chunks = t_stop > it.t0 ? (t_stop - t_begin + BN - 1) / BN : 0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(k_full + 8 * b, 1);
      mbar_init(v_full + 8 * b, 1);
      mbar_init(s_full + 8 * b, 1);
      mbar_init(p_full + 8 * b, 4);  // one arrival per softmax warp
      mbar_init(pv_done + 8 * b, 1);
    }
    mbar_init(done, 1);
    *abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), T_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // (behind the allocation: no CTA of the next kernel may take the columns this one is waiting for)
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 || warp == 2) {
    const bool is_k = warp == 0;
    const CUtensorMap* map = is_k ? &k_map : &v_map;
    if (lane == 0) tma_prefetch(map);
    const uint32_t base = sbase + (is_k ? L::K_OFF : L::V_OFF);
    // a K buffer is free once the scores of the chunk two back are complete, a V buffer once its P V is
    const uint32_t full = is_k ? k_full : v_full, empty = is_k ? s_full : pv_done;
    const int* places = list + it.kv_base;
    auto slot = [&](int t) {  // expanded slot of key t, -1 outside the part
      if (t < it.t0 || t >= t_stop) return -1;
      const long long s = slot_of(a, __ldg(places + a.page.of(t)), t);
      if (s < 0 || s >= n_slots) {
        report(kErrBadIndex);
        return -1;
      }
      return (int)s;
    };
    int s0 = slot(t_begin + 2 * lane), s1 = slot(t_begin + 2 * lane + 1), c = 0;
    for (; c < n_chunks; ++c) {
      const int b = c & 1, next = t_begin + (c + 1) * BN + 2 * lane;
      const int n0 = slot(next), n1 = slot(next + 1);
      if (c >= 2 && !warp_wait(empty + 8 * b, ((c >> 1) - 1) & 1, abort)) break;
      load_chunk<D>(base + b * L::KV_BYTES, full + 8 * b, map, is_k ? k_pool : v_pool, !is_k, s0, s1, a.hk, h,
                    lane);
      s0 = n0, s1 = n1;
    }
    // no copy may still be in flight when the CTA exits (after a wait that ran out nobody else has seen the last ones land)
    if (lane == 0)
      for (int x = max(c - 2, 0); x < c; ++x) mbar_wait_landed(full + 8 * (x & 1), (x >> 1) & 1);
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t IDESC_S = idesc_bf16(T_ROWS, BN);
      constexpr uint32_t IDESC_O = idesc_f16(T_ROWS, D, /*b_mn_major=*/true);
      bool ok = n_chunks > 0 && mbar_wait(q_full, 0, abort, kErrTimeoutAttention);
      // operand descriptors: one per buffer, advanced per 16-deep K step by the byte offset (>> 4)
      const uint64_t q_desc = sw128_desc(sbase);
      const uint64_t k_desc0 = sw128_desc(sbase + L::K_OFF), v_desc0 = sw128_desc(sbase + L::V_OFF, BN * 128);
      constexpr uint64_t KV_STEP = L::KV_BYTES >> 4;
      auto k_landed = [&](int c) { return mbar_wait(k_full + 8 * (c & 1), (c >> 1) & 1, abort, kErrTimeoutAttention); };
      auto issue_qk = [&](int c) {
        const int b = c & 1;
        const uint64_t k_desc = k_desc0 + b * KV_STEP;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qa = ((kk >> 2) * (T_ROWS * 128) + (kk & 3) * 32) >> 4;
          const uint32_t kb = ((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4;
          umma_bf16(tmem + b * BN, q_desc + qa, k_desc + kb, IDESC_S, kk > 0);  // (kind::f16: the types are in IDESC)
        }
        umma_commit(s_full + 8 * b);
      };
      for (int c = 0; c < min(n_chunks, 2) && ok; ++c) {
        ok = k_landed(c);
        tc_fence_after();
        if (ok) issue_qk(c);
      }
      for (int c = 0; c < n_chunks && ok; ++c) {
        const int b = c & 1;
        // O += P_c V_c, P_c from TMEM buffer b (packed FP16 pairs, 8 columns per 16 keys). The copies are waited for
        // first: they have landed long before P_c comes, and a wait costs 100 cycles even then.
        ok = mbar_wait(v_full + 8 * b, (c >> 1) & 1, abort, kErrTimeoutAttention) &&
             (c + 2 >= n_chunks || k_landed(c + 2)) &&
             mbar_wait(p_full + 8 * b, (c >> 1) & 1, abort, kErrTimeoutAttention);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v_desc = v_desc0 + b * KV_STEP;
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          umma_bf16_tmem_a(tmem + 128, tmem + b * BN + kk * 8, v_desc + kk * (2048 >> 4), IDESC_O, (c | kk) != 0);
        umma_commit(pv_done + 8 * b);
        if (c + 2 < n_chunks) issue_qk(c + 2);  // in issue order after this PV, which reads P_c first
      }
      // TMEM is freed only after every MMA issued here has completed
      umma_commit(done);
      mbar_wait_landed(done, 0);
    }
  } else if (warp == 3) {
    // ---------------- Q rows into the swizzled tile: D / 8 lanes share a row ----------------
    constexpr int LPR = D / 8;
#pragma unroll 4
    for (int i = lane / LPR; i < T_ROWS; i += 32 / LPR) {
      const int x = it.r0 + i, u = lane % LPR;
      const bool ok = x < n_rows;
      const __nv_bfloat16* src = a.q + (ok ? row_index(a, it, h, x) * D + u * 8 : 0);
      cp_async16(sbase + (u >> 3) * (T_ROWS * 128) + sw128_offset(i, u & 7), src, ok ? 16u : 0u);
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
  } else {
    // ---------------- softmax warpgroup ----------------
    const int r = (warp & 3) * 32 + lane, row = it.r0 + r, qi = a.group.of(row);
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool row_ok = row < n_rows;
    float vr = refs ? __ldg(refs + h) : 0.f;
    const bool apart = vr == SCALES_APART;
    if (apart) vr = 0.f;  // the largest V scale met so far: O is in units of it
    int lo = 1, hi = 0;  // visible key positions [lo, hi] of this part
    if (row_ok) {
      visible(it.q_len, it.kv_len, bidir, a.window, qi, &lo, &hi);
      lo = max(lo, it.t0), hi = min(hi, t_stop - 1);
    }
    float m_used = -INFINITY, l_run = 0.f;
    bool ok;
    if (!apart) {
      const ChunkSide side{t_lane, s_full, p_full, pv_done, t_begin, it.t0, t_stop, n_chunks, lo, hi, a.scale_log2, abort};
      ok = softmax_chunks<D, false>(a, h, nullptr, nullptr, 0, side, m_used, l_run, vr);
    } else {  // (numbers of its own: those of the usual walk stay in registers)
      const ChunkSide side{t_lane, s_full, p_full, pv_done, t_begin, it.t0, t_stop, n_chunks, lo, hi, a.scale_log2, abort};
      float m = -INFINITY, l = 0.f, v = 0.f;
      ok = softmax_chunks_apart<D>(a, h, pages, list + it.kv_base, n_slots, side, m, l, v);
      m_used = m, l_run = l, vr = v;
    }
    if (ok && (n_chunks == 0 || warp_wait(pv_done + 8 * ((n_chunks - 1) & 1), ((n_chunks - 1) >> 1) & 1, abort))) {
      tc_fence_after();
      // A finished row: O / l times V's reference; a part: (maximum, sum, O in units of the values). The warp's 32 rows
      // go through its quarter of the K and V buffers, which nothing reads any more, and out as whole rows.
      const bool part_of = it.unit >= 0;
      const float unit = exp2_int(-(int)T_P_LOG2);
      const float back = l_run == 0.f ? 0.f : part_of ? vr * unit : vr / l_run;
      float* part = a.ws + ((size_t)(max(it.unit, 0) + r / UNIT) * a.hk + h) * (UNIT * (D + 2));
      if (part_of && row_ok) part[r % UNIT] = m_used, part[UNIT + r % UNIT] = l_run * unit;
      const uint32_t stage = sbase + L::K_OFF + (warp & 3) * (32 * D * 4);
#pragma unroll 1
      for (int col = 0; col < D; col += 32) {
        uint32_t o[32];
        if (n_chunks) {
          tmem_ld32(t_lane + 128 + col, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int v8 = 0; v8 < 4; ++v8) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = back == 0.f ? 0.f : __uint_as_float(o[v8 * 8 + e]) * back;
          const int c8 = col / 8 + v8;  // (16-byte units swizzled by the row: free of bank conflicts both ways)
          if (part_of) {
            sts16(stage + lane * (D * 4) + (((2 * c8) ^ (lane & 7)) << 4), __float_as_uint(x[0]), __float_as_uint(x[1]),
                  __float_as_uint(x[2]), __float_as_uint(x[3]));
            sts16(stage + lane * (D * 4) + (((2 * c8 + 1) ^ (lane & 7)) << 4), __float_as_uint(x[4]),
                  __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
          } else {
            sts16(stage + lane * (D * 2) + ((c8 ^ (lane & 7)) << 4), pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                  pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
          }
        }
      }
      __syncwarp();
      const int units = part_of ? D / 4 : D / 8;  // 16-byte units of a row, a power of two up to 32
      for (int i = lane / units; i < 32; i += 32 / units) {
        const int u = lane % units, x = (warp & 3) * 32 + i, rx = it.r0 + x;
        if (rx >= n_rows) break;
        const uint4 v = lds16(stage + i * (units * 16) + ((u ^ (i & 7)) << 4));
        if (part_of) {
          float* dst = a.ws + ((size_t)(it.unit + x / UNIT) * a.hk + h) * (UNIT * (D + 2)) + 2 * UNIT + (x % UNIT) * D;
          reinterpret_cast<uint4*>(dst)[u] = v;
        } else {
          __nv_bfloat16* dst = a.out + row_index(a, it, h, rx) * D;
          reinterpret_cast<uint4*>(dst)[u] = v;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, T_TMEM_COLS);
  }
}

// Joins the parts of one 16-row unit: o = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p. A warp per row, every part's
// numbers asked for before the first is used.
constexpr int C_WARPS = 8;
template <int D>
__global__ void __launch_bounds__(C_WARPS * 32) combine_kernel(const Args a, const Item* __restrict__ items) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  constexpr int V = D / 32;  // columns of a lane
  const Item it = items[blockIdx.x / a.hk];
  const int h = blockIdx.x % a.hk, lane = threadIdx.x % 32;
  const int r = blockIdx.y * C_WARPS + threadIdx.x / 32, row = it.r0 + r;
  const int G = a.hq / a.hk;
  if (r >= it.tile || row >= it.q_len * G) return;
  const size_t step = (size_t)it.stride * a.hk * (UNIT * (D + 2));
  const float* first = a.ws + ((size_t)it.unit * a.hk + h) * (UNIT * (D + 2));
  float mm = -INFINITY, ll = 0.f, o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.f;
  for (int p0 = 0; p0 < it.parts; p0 += 32) {  // (a lane's part: its maximum and sum)
    const int p = p0 + lane;
    const float m = p < it.parts ? __ldcg(first + p * step + r) : -INFINITY;
    const float l = p < it.parts ? __ldcg(first + p * step + UNIT + r) : 0.f;
    float now = max_nan(mm, m);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) now = max_nan(now, __shfl_xor_sync(0xffffffffu, now, x));
    const float back = mm == -INFINITY ? 0.f : exp2f(mm - now);
    const float f = m == -INFINITY ? 0.f : exp2f(m - now);
    float sum = f * l;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    ll = ll * back + sum;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] *= back;
    mm = now;
    const int n = min(32, it.parts - p0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      const float* src = first + (size_t)(p0 + i) * step + 2 * UNIT + r * D + lane * V;
      float x[V];
      if constexpr (V == 4) {
        const float4 u = __ldcg(reinterpret_cast<const float4*>(src));
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      } else {
        const float2 u = __ldcg(reinterpret_cast<const float2*>(src));
        x[0] = u.x, x[1] = u.y;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(w, x[e], o[e]);
    }
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  __nv_bfloat16* dst = a.out + row_index(a, it, h, row) * D + lane * V;
#pragma unroll
  for (int e = 0; e < V; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(ll == 0.f ? 0.f : o[e] * inv, ll == 0.f ? 0.f : o[e + 1] * inv);
}

// cudaFuncSetAttribute holds per device
template <int D>
static int configure() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
    const auto max_smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    e = cudaFuncSetAttribute(tile_kernel<D>, max_smem, TSmem<D>::TOTAL);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rows_kernel<D, 8>, max_smem, RSmem<D>::TOTAL);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rows_kernel<D, 16>, max_smem, RSmem<D>::TOTAL);
    if (e == cudaSuccess && dev < 64) done[dev] = true;
  }
  return e == cudaSuccess ? MORJ_OK : set_error(MORJ_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
}

// Offsets in the caller's workspace: the expanded K and V, V's reference scales, the parts.
struct Space {
  size_t k, v, refs, parts, bytes;
  Space(const int* counts, int hk, int d, int page_size) {
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t pool = up((size_t)counts[6] * page_size * hk * d * sizeof(uint16_t));
    k = 0, v = pool, refs = 2 * pool;
    parts = refs + (counts[6] ? up((size_t)hk * sizeof(float)) : 0);
    bytes = parts + (size_t)counts[2] * hk * UNIT * (d + 2) * sizeof(float);
  }
};

template <int D>
static int launch(Args a, const int* counts, const int* work, char* ws, cudaStream_t s) {
  const Space at(counts, a.hk, D, a.page.d);
  a.ws = reinterpret_cast<float*>(ws + at.parts);
  const int n_rows = counts[0], n_combine = counts[1], n_tiles = counts[5], n_pages = counts[6], n_blocks = counts[7];
  const Item* items = reinterpret_cast<const Item*>(work);
  int st = configure<D>();
  if (st) return st;
  if (n_tiles) {
    const int* pages = work + (size_t)(n_tiles + n_rows + n_combine) * (sizeof(Item) / sizeof(int));
    const int* blocks = pages + 2 * (size_t)n_pages;
    const int* list = blocks + n_blocks;
    const int n_slots = n_pages * a.page.d;
    uint16_t* kx = reinterpret_cast<uint16_t*>(ws + at.k);
    uint16_t* vx = reinterpret_cast<uint16_t*>(ws + at.v);
    float* refs = reinterpret_cast<float*>(ws + at.refs);
    CUtensorMap km, vm;
    // expanded pools [slots, hk, D]: box = 64 columns x 1 head x 64 slots (one slot and an unused map where none is seen)
    const unsigned long long dims[3] = {(unsigned long long)D, (unsigned long long)a.hk,
                                        (unsigned long long)(n_slots ? n_slots : 1)};
    const unsigned long long strides[2] = {(unsigned long long)D * 2, (unsigned long long)a.hk * D * 2};
    const unsigned box[3] = {64u, 1u, (unsigned)BN};
    void* kp = n_slots ? (void*)kx : const_cast<uint8_t*>(a.k);
    void* vp = n_slots ? (void*)vx : const_cast<uint8_t*>(a.v);
    if ((st = encode_tiled(&km, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, kp, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)))
      return st;
    if ((st = encode_tiled(&vm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, vp, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)))
      return st;
    if (n_slots)
      st = launch_pdl("expand_kernel", expand_kernel<D>, dim3((n_slots + BN - 1) / BN, a.hk, 2), dim3(E_THREADS), 0, s, a,
                      reinterpret_cast<const int2*>(pages), n_slots, blocks, n_blocks, kx, vx, refs);
    else
      refs = nullptr;
    if (st) return st;
    st = launch_pdl("tile_kernel", tile_kernel<D>, dim3((unsigned)n_tiles * a.hk), dim3(T_THREADS), TSmem<D>::TOTAL, s,
                    km, vm, a, items, reinterpret_cast<const int2*>(pages), list, (const uint16_t*)kx, (const uint16_t*)vx,
                    n_slots, (const float*)refs);
    if (st) return st;
    items += n_tiles;
  }
  if (n_rows) {
    CUtensorMap km, vm;  // code pools [slots, hk, D]: box = a row's codes x 1 head x 32 slots
    const unsigned long long dims[3] = {(unsigned long long)D, (unsigned long long)a.hk, (unsigned long long)a.pool_slots};
    const unsigned long long strides[2] = {(unsigned long long)D, (unsigned long long)a.hk * D};
    const unsigned box[3] = {(unsigned)D, 1u, (unsigned)STEP};
    const CUtensorMapSwizzle swizzle = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if ((st = encode_tiled(&km, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.k, dims, strides, box, swizzle))) return st;
    if ((st = encode_tiled(&vm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.v, dims, strides, box, swizzle))) return st;
    const dim3 grid((unsigned)n_rows * a.hk);
    st = counts[3] == 8 ? launch_pdl("rows_kernel", rows_kernel<D, 8>, grid, dim3(WARPS * 32), RSmem<D>::TOTAL, s, km,
                                     vm, a, items)
                        : launch_pdl("rows_kernel", rows_kernel<D, 16>, grid, dim3(WARPS * 32), RSmem<D>::TOTAL, s, km,
                                     vm, a, items);
    items += n_rows;
  }
  if (st == MORJ_OK && n_combine)
    st = launch_pdl("combine_kernel", combine_kernel<D>, dim3((unsigned)n_combine * a.hk, UNIT / C_WARPS),
                    dim3(C_WARPS * 32), 0, s, a, items);
  return st;
}

// The tiles' key ranges cut into parts so that together they fill `slots` resident CTAs once: a part holds an equal
// share of all keys, at least min_keys, and a tile is cut only into whole shares. (Cutting further to even out the lengths
// was measured slower: an SM's last CTAs run faster by themselves, 161 against 166-171 us for 64 single queries over 1 to
// 8,048 keys.) Parts write units of 16 rows to the workspace; `joins` gets one entry per 16 rows of a cut tile.
static std::vector<Item> cut(const std::vector<Item>& tiles, int hk, int slots, int min_keys, int& units,
                             std::vector<Item>& joins) {
  long long total = 0;
  for (const Item& it : tiles) total += it.t1 - it.t0;
  const long long share = std::max<long long>(min_keys, (total * hk + slots - 1) / slots);
  std::vector<Item> out;
  for (const Item& it : tiles) {
    const int keys = it.t1 - it.t0;
    const int parts = (int)std::max<long long>(1, keys / share);
    if (parts == 1) {
      out.push_back(it);
      continue;
    }
    // (whole 64-key chunks, counted from a 64-key boundary)
    const int first = it.t0 - it.t0 % BN, chunks = (it.t1 - first + BN - 1) / BN;
    const int step = (chunks + parts - 1) / parts * BN, per = (it.tile + UNIT - 1) / UNIT;
    Item join = it;
    join.parts = 0, join.stride = per;
    for (int t = first; t < it.t1; t += step) {
      Item part = it;
      part.t0 = std::max(it.t0, t), part.t1 = std::min(it.t1, t + step);
      part.unit = units + per * join.parts++;
      out.push_back(part);
    }
    for (int u = 0; u < per; ++u) {
      Item j = join;
      j.r0 += u * UNIT, j.unit = units + u, j.tile = std::min(UNIT, it.tile);
      joins.push_back(j);
    }
    units += per * join.parts;
  }
  // longest first: the last CTAs to start are the short ones
  std::stable_sort(out.begin(), out.end(), [](const Item& x, const Item& y) { return x.t1 - x.t0 > y.t1 - y.t0; });
  return out;
}

}  // namespace kv8
}  // namespace morj

extern "C" int morj_tree_attention_kv8_work(const int* qo_indptr_host, const int* kv_indptr_host,
                                            const int* kv_indices_host, const int* kv_last_page_len_host,
                                            int n_segments, int n_bidir, int hq, int hk, int page_size, int window,
                                            int* work_host, int cap, int* counts) {
  using namespace morj;
  using kv8::Item;
  if (!qo_indptr_host || !kv_indptr_host || !counts || n_segments < 0 || n_bidir < 0 || n_bidir > n_segments ||
      hk <= 0 || hq <= 0 || hq % hk || page_size <= 0 || cap < 0 || (cap && !work_host) ||
      (n_segments && kv_indptr_host[n_segments] > 0 && !kv_indices_host)) {
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: bad arguments");
  }
  const int G = hq / hk;
  try {
    for (int s = 0; s < n_segments; ++s) {
      const long long rows = ((long long)qo_indptr_host[s + 1] - qo_indptr_host[s]) * G;
      if (qo_indptr_host[s] < 0 || rows < 0 || rows > (1 << 30) || kv_indptr_host[s] < 0 || kv_indptr_host[s + 1] < kv_indptr_host[s])
        return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: segment %d's tables are out of order", s);
    }
    std::vector<Item> tiles, rows, joins;
    std::vector<int> kv_len(n_segments);
    // the keys that rows [r0, r0 + n) of a segment see: what its first query sees from, its last query to
    auto seen = [&](int s, int r0, int n, int* lo, int* hi) {
      const int q_len = qo_indptr_host[s + 1] - qo_indptr_host[s];
      int x;
      kv8::visible(q_len, kv_len[s], s < n_bidir, window, r0 / G, lo, &x);
      kv8::visible(q_len, kv_len[s], s < n_bidir, window, (std::min(r0 + n, q_len * G) - 1) / G, &x, hi);
    };
    const long long places = (long long)kv8::R_CTAS * num_sms();
    long long few_tiles = 0, few_keys = 0;  // if rows_kernel took every segment
    int most = 0, most_few = 0;             // the largest segment, and the largest that it takes anyhow
    for (int s = 0; s < n_segments; ++s) {
      const int n_pages = kv_indptr_host[s + 1] - kv_indptr_host[s];
      const int last = kv_last_page_len_host ? kv_last_page_len_host[s] : page_size;
      if (last < 0 || last > page_size)  // (more would be keys past the segment's list)
        return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: the last page of segment %d holds %d of %d slots", s,
                         last, page_size);
      const long long kv = n_pages == 0 ? 0 : (long long)(n_pages - 1) * page_size + last;
      if (kv > INT_MAX)
        return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: segment %d has %lld keys", s, kv);
      kv_len[s] = (int)kv;
      const int n = (qo_indptr_host[s + 1] - qo_indptr_host[s]) * G;
      most = std::max(most, n);
      if (n <= kv8::FEW_ROWS) most_few = std::max(most_few, n);
      for (int r0 = 0; r0 < n && few_tiles * hk <= places; r0 += kv8::FEW_ROWS) {
        int lo, hi;
        seen(s, r0, kv8::FEW_ROWS, &lo, &hi);
        ++few_tiles, few_keys += std::max(hi - lo + 1, 0);
      }
    }
    const bool all_few = few_tiles * hk <= places && few_keys * hk <= kv8::FEW_KEYS;
    const int few = (all_few ? most : most_few) <= 8 ? 8 : 16;
    // what the tiled segments see: the distinct pages in the order the lists name them, how many slots of each are
    // listed, and every list entry's place among them
    std::vector<int> near, pages, used, list;
    std::unordered_map<int, int> far;  // (pages past what a table should be made for)
    auto place = [&](int page) -> int& {  // the page's place, -1 before it has one
      if (page >= 1 << 24) return far.emplace(page, -1).first->second;
      if ((size_t)page >= near.size()) near.resize(std::max<size_t>(page + 1, 2 * near.size()), -1);
      return near[page];
    };
    for (int s = 0; s < n_segments; ++s) {
      const int q_len = qo_indptr_host[s + 1] - qo_indptr_host[s];
      const int kv = kv_len[s];
      const bool many = !all_few && q_len * G > kv8::FEW_ROWS;
      const int tile = many ? kv8::T_ROWS : few;
      int from = INT_MAX, to = -1;  // keys the segment's queries see
      for (int r0 = 0; r0 < q_len * G; r0 += tile) {
        int lo, hi;
        seen(s, r0, tile, &lo, &hi);
        Item it{s, r0, 0, 0, -1, 1, 1, tile, qo_indptr_host[s], q_len, kv_indptr_host[s], kv};
        if (hi >= lo) it.t0 = lo, it.t1 = hi + 1, from = std::min(from, lo), to = std::max(to, hi);
        (many ? tiles : rows).push_back(it);
      }
      if (q_len * G <= kv8::FEW_ROWS || to < from) continue;
      if (many && list.empty()) list.resize(kv_indptr_host[n_segments], 0);
      for (int p = from / page_size; p <= to / page_size; ++p) {
        const int at = kv_indptr_host[s] + p, page = kv_indices_host[at];
        if (page < 0) return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: page %d in segment %d's list", page, s);
        if (!many) continue;
        int& index = place(page);
        if (index < 0) {
          index = (int)pages.size();
          pages.push_back(page);
          used.push_back(0);
        }
        list[at] = index;
        const int n = p == to / page_size ? to % page_size + 1 : page_size;
        used[index] = std::max(used[index], n);
      }
    }
    if ((long long)pages.size() * page_size > INT_MAX - 64)
      return set_error(MORJ_ERR_UNSUPPORTED, "morj_tree_attention_kv8_work: %zu pages of %d slots to expand", pages.size(),
                       page_size);
    std::vector<int> blocks;  // 64-slot blocks that hold listed slots
    for (size_t i = 0; i < pages.size(); ++i) {
      const long long first = (long long)pages[i] * page_size;
      for (long long b = first / kv8::BLOCK; b <= (first + used[i] - 1) / kv8::BLOCK; ++b)
        blocks.push_back((int)std::min<long long>(b, INT_MAX));  // (past every pool: the kernel looks at none there)
    }
    std::sort(blocks.begin(), blocks.end());
    blocks.erase(std::unique(blocks.begin(), blocks.end()), blocks.end());
    int units = 0;
    const std::vector<Item> cut_tiles = kv8::cut(tiles, hk, num_sms() * kv8::T_CTAS, kv8::T_MIN_KEYS, units, joins);
    const std::vector<Item> cut_rows = kv8::cut(rows, hk, num_sms() * kv8::R_CTAS, kv8::R_MIN_KEYS, units, joins);
    const size_t ints = (cut_tiles.size() + cut_rows.size() + joins.size()) * (sizeof(Item) / sizeof(int)) +
                        2 * pages.size() + blocks.size() + list.size();
    if (ints > (size_t)INT_MAX)
      return set_error(MORJ_ERR_UNSUPPORTED, "morj_tree_attention_kv8_work: a work list of %zu ints", ints);
    const int got[10] = {(int)cut_rows.size(), (int)joins.size(), units, few, (int)ints, (int)cut_tiles.size(),
                        (int)pages.size(), (int)blocks.size(), (int)list.size(),
                         n_segments ? qo_indptr_host[n_segments] : 0};
    std::copy(got, got + 10, counts);
    if (counts[4] > cap) {
      if (cap == 0) return MORJ_OK;  // (a call that only asks for the counts)
      return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: %d ints exceed capacity %d", counts[4], cap);
    }
    Item* out = reinterpret_cast<Item*>(work_host);
    out = std::copy(cut_tiles.begin(), cut_tiles.end(), out);
    out = std::copy(cut_rows.begin(), cut_rows.end(), out);
    out = std::copy(joins.begin(), joins.end(), out);
    int* rest = reinterpret_cast<int*>(out);
    for (size_t i = 0; i < pages.size(); ++i) *rest++ = pages[i], *rest++ = used[i];
    rest = std::copy(blocks.begin(), blocks.end(), rest);
    std::copy(list.begin(), list.end(), rest);
    return MORJ_OK;
  } catch (...) {
    return set_error(MORJ_ERR_OOM, "morj_tree_attention_kv8_work: out of host memory");
  }
}

extern "C" int morj_tree_attention_kv8_workspace(const int* counts, int hk, int d, int page_size,
                                                 unsigned long long* bytes) {
  using namespace morj;
  if (!counts || !bytes || hk <= 0 || d <= 0 || page_size <= 0 || counts[2] < 0 || counts[6] < 0)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_workspace: bad arguments");
  *bytes = kv8::Space(counts, hk, d, page_size).bytes;
  return MORJ_OK;
}

extern "C" int morj_tree_attention_kv8(const void* q, int n_q, const void* k_codes, const float* k_scale,
                                       const void* v_codes, const float* v_scale, int pool_slots, void* out,
                                       const int* kv_indices, int n_bidir, int hq, int hk, int d, int page_size,
                                       int window, float sm_scale, const int* work, const int* counts,
                                       void* workspace, unsigned long long workspace_bytes, void* stream) {
  using namespace morj;
  if (!counts) return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: null counts");
  if (counts[0] == 0 && counts[5] == 0) return MORJ_OK;
  if (!q || !k_codes || !k_scale || !v_codes || !v_scale || !out || !kv_indices || !work ||
      n_q <= 0 || pool_slots <= 0 || counts[0] < 0 || counts[1] < 0 || counts[2] < 0 || counts[5] < 0 || counts[6] < 0 || counts[7] < 0)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: null pointer or bad size");
  if (hq <= 0 || hk <= 0 || hq % hk)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: hq=%d is not a multiple of hk=%d", hq, hk);
  if (!(sm_scale > 0.f))
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: sm_scale must be positive");
  if (n_q < counts[9])
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: %d queries, the work list has %d", n_q, counts[9]);
  if (page_size <= 0 || n_bidir < 0)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: bad page_size %d or n_bidir %d", page_size, n_bidir);
  if (d != 64 && d != 128)
    return set_error(MORJ_ERR_UNSUPPORTED, "morj_tree_attention_kv8: head_dim %d unsupported (64, 128)", d);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(workspace)) &
      15)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: q, codes, out, work and workspace must be 16-byte aligned");
  const unsigned long long need = kv8::Space(counts, hk, d, page_size).bytes;
  if (workspace_bytes < need || (need && !workspace))
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: a workspace of %llu bytes given, %llu needed",
                     workspace_bytes, need);
  const kv8::Args a{(const __nv_bfloat16*)q, (const uint8_t*)k_codes, k_scale, (const uint8_t*)v_codes, v_scale,
                    (__nv_bfloat16*)out, kv_indices, n_bidir, hq, hk, window, pool_slots, kv8::Quotient(page_size),
                    kv8::Quotient(hq / hk), sm_scale * kv8::LOG2E, nullptr};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return d == 128 ? kv8::launch<128>(a, counts, work, (char*)workspace, s)
                  : kv8::launch<64>(a, counts, work, (char*)workspace, s);
}
