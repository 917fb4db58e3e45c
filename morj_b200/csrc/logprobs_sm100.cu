// Log-probabilities of given tokens over the whole vocabulary, without the [rows, vocab] logits in memory.
//
//   l_iv = h_i . w_v,  z = c tanh(l / c) (c = 0: z = l),  lse_i = log sum_v exp z_iv,
//   logp_it = z_it - lse_i,  entropy_i = lse_i - sum_v p_iv z_iv,  top k by (l descending, id ascending).
//
// logits_kernel is a GEMM whose epilogue folds every accumulator row into three running numbers, with m the largest z
// so far: m, s = sum exp(z - m) and t = sum exp(z - m) (z - m), so that lse = m + log s and entropy = log s - t / s
// without cancellation. A CTA keeps them per row across the vocabulary tiles it computes. finish_kernel joins the CTAs'
// numbers of a row and adds the given tokens' logits as plain dot products.
//
// Top alternatives: the softcap is monotone, so candidates are compared by the raw logit. A logit is appended, unordered,
// to the CTA's list of the row when it reaches a bound that at least `top` logits of the row are known to reach: at first
// the top-th largest of the 32 group maxima of the CTA's first tile, then the largest such bound of any CTA. That leaves
// about ten candidates a row and CTA and no branch per logit; a list that fills up all the same (equal or rising logits)
// is cut to its top ones. (A sorted list per row in shared memory cost 1.0 ms of 2.1 on 540 rows with 5 alternatives: one
// of 32 rows inserting holds up the warp.)
//
// Bound by the tensor cores or, for few rows, by reading w (262,144 x 5,376). The SM clock, and with it the first two, depends
// on the box and on what ran before (the power cap): 2,040 rows (5.75 TFLOP) 4.45-4.9 ms = 1,170-1,290 TFLOP/s, 540 rows
// (five row blocks of 128, the last with 28) 1.30-1.55 ms = 980-1,170, 9 rows (2.82 GB) 0.457-0.469 ms = 6.0-6.2 TB/s back
// to back, 0.50 with cold caches. 1 row of 4,096 logits, 13 us back to back, 18 alone, is latency: three dependent steps in
// two launches.
//
// One CTA per SM: warp 0 TMA producer, warp 1 MMA issuer (tcgen05, M = 128, N = 256, two TMEM accumulators), warps 2-5
// epilogue (thread = row). Row blocks are the fast tile index: the CTAs in flight share a few vocabulary tiles, so w
// crosses HBM once per call of up to 2048 rows (larger calls go in chunks of 2048).
#include <algorithm>
#include <climits>

#include "common.cuh"

namespace morj {
namespace logprobs {

constexpr int BM = 128, BK = 64;
constexpr int BN_WIDE = 256, BN_NARROW = 64;  // vocabulary rows of a tile
constexpr int A_BYTES = BM * BK * 2;
constexpr int STAGES = 4;
constexpr int MAX_TOP = MORJ_MAX_TOP;
constexpr int CAND = 64;  // candidates a CTA's list of a row holds: top ones (32 at most) and one group of 32 more
static_assert(CAND >= MAX_TOP + 32, "a cut list takes a whole group of columns");
constexpr int smem_bytes(int bn) { return STAGES * (A_BYTES + bn * BK * 2) + 1024 /*align*/ + 256 /*barriers*/; }
static_assert(smem_bytes(BN_WIDE) <= 232448, "shared memory per CTA");
constexpr int THREADS = 192;
constexpr int CHUNK_ROWS = 2048;
constexpr float LOG2E = 1.4426950408889634f;

// What the CTAs know of the rows.
struct Scratch {
  float4* stats;    // [cta][row]: m, s, t, number of candidates
  float* own;       // [cta][row]: candidates must exceed it (the top-th of a cut list)
  uint2* lists;     // [cta][row block][CAND][128 rows]: candidates (logit, id)
  unsigned* bound;  // [row]: at least `top` logits reach it, as an ordered integer; 0: none known. Null: one tile per CTA
  int rows;         // rows of a chunk rounded up to whole row blocks
  int top;
};

// floats as unsigned integers of the same order (never 0 for a number; -0 as +0), and the next float below such a one
MORJ_DEV unsigned ordered(float f) {
  const unsigned b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
MORJ_DEV float below(unsigned o) {
  const unsigned p = o - (o == 0x80000000u ? 2u : 1u);  // (below +0 comes -0, which is not below it)
  return __uint_as_float(p & 0x80000000u ? p & 0x7fffffffu : ~p);
}

// z = c tanh(l / c). Near 0 tanh's series, a few 2^-24 of z; elsewhere 1 - 2 / (1 + e^2x), whose error (ex2.approx,
// rcp.approx, the rounded argument) is absolute, about 2^-22 c: a few parts in 2^22 of z right above c / 4.
MORJ_DEV float cap_near(float l, float c, float inv_c) {  // |l| <= c / 4
  const float x = l * inv_c, x2 = x * x;
  const float p = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  return __fmul_rn(l, p);  // (not joined with what is subtracted from it: one value whether or not others are far)
}
MORJ_DEV float cap_far(float l, float c, float inv_c) {
  float r;
  const float e = fast_exp2(l * (inv_c * 2.f * LOG2E));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return fmaf(-2.f * c, r, c);
}
MORJ_DEV float cap(float l, float c, float inv_c) {
  if (c == 0.f) return l;
  return fabsf(l) <= 0.25f * c ? cap_near(l, c, inv_c) : cap_far(l, c, inv_c);
}

// Running numbers of a row moved to a larger maximum.
MORJ_DEV void raise(float& m, float& s, float& t, float now) {
  if (m != -INFINITY) {
    const float f = fast_exp2((m - now) * LOG2E);
    t = f * (t + s * (m - now));
    s *= f;
  }
  m = now;
}

// 32 logits into a row's numbers. CAP: 0 no softcap, 1 every |l| of the warp's rows is at most c / 4, 2 any.
template <int CAP>
MORJ_DEV void fold(const uint32_t (&r)[32], int valid, float c, float inv_c, float& m, float& s, float& t, float mx) {
  const float zmx = CAP ? cap(mx, c, inv_c) : mx;
  if (zmx > m) raise(m, s, t, zmx);
  const float shift = m == -INFINITY ? 0.f : m;
  float s4[4] = {0.f, 0.f, 0.f, 0.f}, t4[4] = {0.f, 0.f, 0.f, 0.f};  // (short sums: the total rounds once per 32)
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float l = __uint_as_float(r[i]);
    float u = (CAP == 0 ? l : CAP == 1 ? cap_near(l, c, inv_c) : cap(l, c, inv_c)) - shift;
    if (CAP == 0) u = max_nan(u, -1e30f);  // (a logit of -infinity: exp 0, and 0 in t; a softcap leaves none)
    const float e = fast_exp2(u * LOG2E);
    if (i < valid) {
      s4[i & 3] += e;
      t4[i & 3] = fmaf(e, u, t4[i & 3]);
    }
  }
  s += (s4[0] + s4[1]) + (s4[2] + s4[3]);
  t += (t4[0] + t4[1]) + (t4[2] + t4[3]);
}

// (logit, id) order of candidates: larger logit first, then the lower id; id < 0: none
MORJ_DEV bool before(float v, int id, float w, int jd) { return id >= 0 && (jd < 0 || v > w || (v == w && id < jd)); }

// Cuts a row's list (entries 128 apart) to its `top` first ones, keeping their order of ids; returns the last one's logit.
__device__ __noinline__ float cut_list(uint2* list, int count, int top) {
  float v[CAND];
  int id[CAND];
  for (int i = 0; i < count; ++i) {
    const uint2 e = list[i * BM];
    v[i] = __uint_as_float(e.x), id[i] = (int)e.y;
  }
  float pv = INFINITY;
  int pid = -1;
  for (int k = 0; k < top; ++k) {  // the next one after (pv, pid)
    float bv = 0.f;
    int bid = -1;
    for (int i = 0; i < count; ++i)
      if ((k == 0 || before(pv, pid, v[i], id[i])) && before(v[i], id[i], bv, bid)) bv = v[i], bid = id[i];
    pv = bv, pid = bid;
  }
  int n = 0;
  for (int i = 0; i < count; ++i)
    if (!before(pv, pid, v[i], id[i])) list[n++ * BM] = make_uint2(__float_as_uint(v[i]), (unsigned)id[i]);
  return pv;
}

template <int BN>
__global__ void __launch_bounds__(THREADS, 1)
    logits_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, int M, int V,
                  int K, int a_bytes, float c, const Scratch sc) {
  constexpr int B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  constexpr uint32_t IDESC = idesc_bf16(BM, BN);
  constexpr int TMEM_COLS = 2 * BN;  // (two accumulators)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  // bars: full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const uint32_t accf0 = smem_u32(bars + 2 * STAGES), acce0 = smem_u32(bars + 2 * STAGES + 2);
  const uint32_t done0 = smem_u32(bars + 2 * STAGES + 4);
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, 128);
    }
    mbar_init(done0, 1);
    *abort = 0;
    fence_mbar_init();
    tma_prefetch(&map_h);
    tma_prefetch(&map_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();  // (set-up above touches no global memory) the previous kernel on the stream has completed
  pdl_trigger();

  const int num_m = (M + BM - 1) / BM, num_n = (V + BN - 1) / BN;
  const int tiles = num_m * num_n, kblocks = (K + BK - 1) / BK;
  const uint32_t smem_base = smem_u32(smem);

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_h = policy_evict_last();
      const uint64_t pol_w = num_m == 1 ? policy_evict_first() : policy_evict_normal();
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok && !*abort; t += gridDim.x) {
        const int m = t % num_m, n = t / num_m;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, abort, kErrTimeoutGemmProducer)) {
            ok = false;
            break;
          }
          const uint32_t sa = smem_base + stage * STAGE_BYTES;
          mbar_arrive_expect_tx(full0 + 8 * stage, a_bytes + B_BYTES);
          tma_load_2d(sa, &map_h, full0 + 8 * stage, kb * BK, m * BM, pol_h);
          tma_load_2d(sa + A_BYTES, &map_w, full0 + 8 * stage, kb * BK, n * BN, pol_w);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // no copy may still be in flight when the CTA exits: wait for the last fills to land
      const int pending = issued < STAGES ? issued : STAGES;
      for (int j = 1; j <= pending; ++j) {
        const int s = (stage - j + STAGES) % STAGES;
        const uint32_t ph = (stage - j >= 0) ? phase : (phase ^ 1);
        mbar_wait_landed(full0 + 8 * s, ph);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        if (!mbar_wait(acce0 + 8 * acc, acc_phase ^ 1, abort, kErrTimeoutGemmMma)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(full0 + 8 * stage, phase, abort, kErrTimeoutGemmMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_base + stage * STAGE_BYTES, sb = sa + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_bf16(d_tmem, sw128_desc(sa + 32 * k), sw128_desc(sb + 32 * k), IDESC, (kb | k) != 0);
          umma_commit(empty0 + 8 * stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        umma_commit(accf0 + 8 * acc);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // TMEM is freed below only after every MMA issued here has completed
      umma_commit(done0);
      mbar_wait_landed(done0, 0);
    }
  } else {
    const int quarter = warp & 3;
    const int r128 = quarter * 32 + lane;
    const int top = sc.top;
    const float inv_c = c > 0.f ? 1.f / c : 0.f;
    float4* stats = sc.stats + (size_t)blockIdx.x * sc.rows + r128;
    float* own_of = sc.own + (size_t)blockIdx.x * sc.rows + r128;
    uint2* lists = sc.lists + (size_t)blockIdx.x * sc.rows * CAND + r128;
    for (int m = 0; m < num_m; ++m) {  // (each thread's own entries: nobody else writes them)
      stats[m * BM] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      if (top) own_of[m * BM] = -INFINITY;
    }
    int acc = 0;
    uint32_t acc_phase = 0;
    int held = -1;  // the row block whose numbers are in registers
    float4 st = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    int count = 0;
    float own = -INFINITY;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int m = t % num_m, n = t / num_m;
      const bool row_ok = m * BM + r128 < M;
      if (m != held) {
        if (held >= 0) {
          st.w = __int_as_float(count);
          stats[held * BM] = st;
          if (top) own_of[held * BM] = own;
        }
        st = stats[m * BM];
        count = __float_as_int(st.w);
        own = top ? own_of[m * BM] : INFINITY;
        held = m;
      }
      uint2* list = lists + (size_t)m * CAND * BM;
      const unsigned known = sc.bound && row_ok ? __ldcg(sc.bound + m * BM + r128) : 0u;  // (arrives during the wait below)
      int ok = lane == 0 ? (int)mbar_wait(accf0 + 8 * acc, acc_phase, abort, kErrTimeoutGemmEpilogue) : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
      float tau = row_ok ? own : INFINITY;  // candidates must exceed it
      if (known) tau = fmaxf(tau, below(known));
      const bool fresh = top && st.x == -INFINITY && known == 0;
      if (__any_sync(0xffffffffu, fresh)) {  // (the TMEM loads are the whole warp's)
        // the rows' first tile: the top-th largest of its 32 groups of columns (columns past V are zeros: left out)
        constexpr int GROUP = BN / 32, PER = 32 / GROUP;
        float g[32];
#pragma unroll
        for (int col = 0; col < BN; col += 32) {
          uint32_t r[32];
          tmem_ld32(tacc + col, r);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < PER; ++q) {
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < GROUP; ++i)
              x = fmaxf(x, n * BN + col + q * GROUP + i < V ? __uint_as_float(r[q * GROUP + i]) : -INFINITY);
            g[col / GROUP + q] = x;
          }
        }
        float first = INFINITY;
        for (int k = 0; k < top; ++k) {
          first = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i) first = fmaxf(first, g[i]);
#pragma unroll
          for (int i = 0; i < 32; ++i) g[i] = g[i] == first ? -INFINITY : g[i];
        }
        if (fresh && row_ok && first > -INFINITY) {
          if (sc.bound) atomicMax(sc.bound + m * BM + r128, ordered(first));
          tau = fmaxf(tau, below(ordered(first)));
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int col = 0; col < BN; col += 32) {
        const int id0 = n * BN + col, valid = min(32, V - id0);
        if (valid <= 0) break;  // (warp-uniform)
        uint32_t r[32];
        tmem_ld32(tacc + col, r);
        tmem_wait_ld();
        float mx = -INFINITY, far = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          mx = fmaxf(mx, i < valid ? __uint_as_float(r[i]) : -INFINITY);
          far = fmaxf(far, fabsf(__uint_as_float(r[i])));
        }
        if (c == 0.f)
          fold<0>(r, valid, c, inv_c, st.x, st.y, st.z, mx);
        else if (__all_sync(0xffffffffu, far <= 0.25f * c || !row_ok))
          fold<1>(r, valid, c, inv_c, st.x, st.y, st.z, mx);
        else
          fold<2>(r, valid, c, inv_c, st.x, st.y, st.z, mx);
        if (__any_sync(0xffffffffu, mx > tau)) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = __uint_as_float(r[i]);
            if (i < valid && x > tau) list[count++ * BM] = make_uint2(r[i], (unsigned)(id0 + i));
          }
          if (count > CAND - 32) {
            own = cut_list(list, count, top);
            count = top;
            if (sc.bound) atomicMax(sc.bound + m * BM + r128, ordered(own));
            tau = fmaxf(tau, own);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      mbar_arrive(acce0 + 8 * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (held >= 0) {
      st.w = __int_as_float(count);
      stats[held * BM] = st;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---- finish: two CTAs per row, one for its numbers and top alternatives, one for the given tokens -------------------
constexpr int F_THREADS = 256;
constexpr int POOL = 1024;

struct Outputs {
  const int* targets;
  int n_targets;
  float* logprobs;
  float* lse;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
};

MORJ_DEV float cap_exact(float l, float c) { return c > 0.f ? c * tanhf(l / c) : l; }

__global__ void __launch_bounds__(F_THREADS)
    finish_kernel(const __nv_bfloat16* __restrict__ h, long long ld_h, const __nv_bfloat16* __restrict__ w,
                  long long ld_w, int V, int K, float c, int ctas, const Scratch sc, const Outputs o, int row0) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  __shared__ float red_s[F_THREADS / 32], red_t[F_THREADS / 32], red_v[2][F_THREADS / 32];
  __shared__ int red_i[2][F_THREADS / 32], red_c[2][F_THREADS / 32];
  const int local = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const size_t row = (size_t)row0 + local;
  // what does not depend on anything is asked for first
  float4 st = make_float4(-INFINITY, 0.f, 0.f, 0.f);
  if (threadIdx.x < ctas) st = sc.stats[(size_t)threadIdx.x * sc.rows + local];
  const uint2* list = sc.lists + ((size_t)threadIdx.x * sc.rows + (local / BM) * BM) * CAND + local % BM;
  constexpr int AHEAD = 16;
  uint2 head[AHEAD];  // the first entries of this thread's list (left over from another call past its count)
  unsigned known = 0;
  if (blockIdx.y == 0 && sc.top) {
    known = sc.bound ? sc.bound[local] : 0u;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) head[i] = threadIdx.x < ctas ? __ldcg(list + i * BM) : make_uint2(0, 0);
  }
  // the given tokens' logits: eight warps share a round of up to eight of them, each target's columns cut evenly
  __shared__ float dots[F_THREADS / 32];
  const int round = min(o.n_targets, F_THREADS / 32);
  const int per = round ? F_THREADS / 32 / round : 1;
  auto dot = [&](int j) {  // this warp's share of the target it has in the round from j on
    const int mine = j + warp / per;
    float acc = 0.f;
    if (warp / per < round && mine < o.n_targets) {
      const int id = o.targets[row * o.n_targets + mine];
      if (id >= 0 && id < V) {
        const __nv_bfloat16* hr = h + row * ld_h;
        const __nv_bfloat16* wr = w + (size_t)id * ld_w;
#pragma unroll 4
        for (int k = (warp % per * 32 + lane) * 8; k < K; k += per * 256) {
          float a[8], b[8];
          load8(hr + k, a);
          load8(wr + k, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc = fmaf(a[e], b[e], acc);
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, x);
    if (lane == 0) dots[warp] = acc;
  };
  if (blockIdx.y == 1) dot(0);
  float m = st.x;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  if (lane == 0) red_v[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < F_THREADS / 32; ++i) m = fmaxf(m, red_v[0][i]);
  float s = st.y, t = st.z;
  if (st.x != -INFINITY) raise(st.x, s, t, m);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, x);
    t += __shfl_xor_sync(0xffffffffu, t, x);
  }
  if (lane == 0) red_s[warp] = s, red_t[warp] = t;
  __syncthreads();
  s = t = 0.f;
#pragma unroll
  for (int i = 0; i < F_THREADS / 32; ++i) s += red_s[i], t += red_t[i];
  const float ls = logf(s), lse = (m == -INFINITY ? 0.f : m) + ls;

  if (blockIdx.y == 0) {
    if (threadIdx.x == 0) {
      if (o.lse) o.lse[row] = lse;
      if (o.entropy) o.entropy[row] = ls - t / s;
    }
    if (!sc.top) return;
    // Thread i has CTA i's list. The bound is raised once more: the largest candidates of the CTAs are different logits,
    // so at least `top` logits reach the top-th largest of them, and few others do. What reaches it goes to shared memory
    // in any order, and each one's place is the number of those before it. (Rounds that take one alternative each, over
    // the bound the CTAs had found, took 23 us for 9 rows of 262144 logits.)
    const int count = threadIdx.x < ctas ? __float_as_int(st.w) : 0;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < count) most = fmaxf(most, __uint_as_float(head[i].x));
#pragma unroll 8
    for (int i = AHEAD; i < count; ++i) most = fmaxf(most, __uint_as_float(__ldcg(list + i * BM).x));
    __shared__ float mosts[F_THREADS];
    __shared__ uint2 pool[POOL];
    __shared__ unsigned raised;
    __shared__ int kept;
    mosts[threadIdx.x] = most;
    if (threadIdx.x == 0) kept = 0, raised = known;
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < ctas; ++i) rank += mosts[i] > most || (mosts[i] == most && i < (int)threadIdx.x);
    if (count && rank == sc.top - 1) atomicMax(&raised, ordered(most));
    __syncthreads();
    const float least = raised ? below(raised) : -INFINITY;  // candidates exceed it
    auto keep = [&](const uint2& e) {
      if (__uint_as_float(e.x) > least) {
        const int at = atomicAdd(&kept, 1);
        if (at < POOL) pool[at] = e;
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < count) keep(head[i]);
    for (int i = AHEAD; i < count; ++i) keep(__ldcg(list + i * BM));
    __syncthreads();
    auto take = [&](int k, float v, int id) {  // id < 0: the row has fewer logits that can be compared
      o.top_ids[row * sc.top + k] = id;
      o.top_logprobs[row * sc.top + k] = id < 0 ? NAN : cap_exact(v, c) - lse;
    };
    const int n = kept;
    if (n <= POOL) {
      for (int i = threadIdx.x; i < n; i += F_THREADS) {
        const uint2 e = pool[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += before(__uint_as_float(pool[j].x), (int)pool[j].y, __uint_as_float(e.x), (int)e.y);
        if (place < sc.top) take(place, __uint_as_float(e.x), (int)e.y);
      }
      for (int k = n + threadIdx.x; k < sc.top; k += F_THREADS) take(k, 0.f, -1);
      return;
    }
    // Many equal logits: in each round a thread offers the first of its list that comes after the one taken last.
    float v = 0.f;
    int id = -1;
    auto next = [&](bool any, float pv, int pid) {  // this thread's first one after (pv, pid)
      float bv = 0.f;
      int bid = -1;
      for (int i = 0; i < count; ++i) {
        const uint2 e = __ldcg(list + i * BM);
        const float x = __uint_as_float(e.x);
        if ((any || before(pv, pid, x, (int)e.y)) && before(x, (int)e.y, bv, bid)) bv = x, bid = (int)e.y;
      }
      v = bv, id = bid;
    };
    next(true, 0.f, 0);
    for (int k = 0; k < sc.top; ++k) {
      float bv = v;
      int bi = id, bc = threadIdx.x;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, x);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, x), oc = __shfl_xor_sync(0xffffffffu, bc, x);
        if (before(ov, oi, bv, bi)) bv = ov, bi = oi, bc = oc;
      }
      const int b = k & 1;  // (two buffers: one barrier a round)
      if (lane == 0) red_v[b][warp] = bv, red_i[b][warp] = bi, red_c[b][warp] = bc;
      __syncthreads();
      bv = red_v[b][0], bi = red_i[b][0], bc = red_c[b][0];
#pragma unroll
      for (int i = 1; i < F_THREADS / 32; ++i)
        if (before(red_v[b][i], red_i[b][i], bv, bi)) bv = red_v[b][i], bi = red_i[b][i], bc = red_c[b][i];
      if (threadIdx.x == 0) take(k, bv, bi);
      if (bi >= 0 && bc == (int)threadIdx.x) next(false, bv, bi);
    }
    return;
  }
  for (int j = 0; j < o.n_targets; j += round) {
    if (j) dot(j);
    __syncthreads();
    const int mine = j + threadIdx.x;
    if (threadIdx.x < round && mine < o.n_targets) {
      const int id = o.targets[row * o.n_targets + mine];
      float l = 0.f;
      for (int i = 0; i < per; ++i) l += dots[threadIdx.x * per + i];
      float lp = cap_exact(l, c) - lse;
      if (id == -1) lp = 0.f;
      if (id < -1 || id >= V) {
        report(kErrBadIndex);
        lp = NAN;
      }
      o.logprobs[row * o.n_targets + mine] = lp;
    }
    __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
static int chunk_rows(int n) { return ((n < CHUNK_ROWS ? n : CHUNK_ROWS) + BM - 1) / BM * BM; }

// Offsets in the caller's workspace.
struct Space {
  size_t own, lists, bound, bytes;
  Space(int n, int top) {
    const size_t rows = chunk_rows(n), per_cta = rows * num_sms();
    own = per_cta * sizeof(float4);
    lists = own + (top ? per_cta * sizeof(float) : 0);
    bound = lists + (top ? per_cta * CAND * sizeof(uint2) : 0);
    bytes = bound + (top ? rows * sizeof(unsigned) : 0);
  }
};

static int make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
  const unsigned long long dims[2] = {(unsigned long long)cols, (unsigned long long)rows};
  const unsigned long long strides[1] = {(unsigned long long)(ld * 2)};
  const unsigned box[2] = {(unsigned)BK, (unsigned)box_rows};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// cudaFuncSetAttribute holds per device
static int configure() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
    e = cudaFuncSetAttribute(logits_kernel<BN_WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(BN_WIDE));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(logits_kernel<BN_NARROW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               smem_bytes(BN_NARROW));
    if (e == cudaSuccess && dev < 64) done[dev] = true;
  }
  return e == cudaSuccess ? MORJ_OK : set_error(MORJ_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
}

}  // namespace logprobs
}  // namespace morj

extern "C" int morj_token_logprobs_workspace(int n, int top, unsigned long long* bytes) {
  using namespace morj;
  if (!bytes || n < 0 || top < 0 || top > logprobs::MAX_TOP)
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs_workspace: bad arguments (n=%d top=%d)", n, top);
  *bytes = n ? logprobs::Space(n, top).bytes : 0;
  return MORJ_OK;
}

extern "C" int morj_token_logprobs(const void* h, long long ld_h, int n, const void* w, long long ld_w, int vocab,
                                   int H, float softcap, const int* targets, int n_targets, float* logprobs_out,
                                   float* lse, float* entropy, int top, int* top_ids, float* top_logprobs,
                                   void* workspace, unsigned long long workspace_bytes, void* stream) {
  using namespace morj;
  using namespace morj::logprobs;
  if (n == 0) return MORJ_OK;
  if (!h || !w || n < 0 || vocab <= 0 || vocab > INT_MAX - BN_WIDE || H <= 0 || n_targets < 0 ||
      (n_targets && (!targets || !logprobs_out)) || (top && (!top_ids || !top_logprobs)))
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: null pointer or bad size (n=%d vocab=%d H=%d)", n, vocab, H);
  if (top < 0 || top > MAX_TOP || top > vocab)
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: top %d must be in [0, %d] and at most vocab", top, MAX_TOP);
  if (!(softcap >= 0.f) || softcap > 1e30f || (softcap > 0.f && softcap < 1e-30f))
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: softcap must be 0 (none) or in [1e-30, 1e30]");
  if (H % 8 || ld_h % 8 || ld_w % 8 || ld_h < H || ld_w < H)
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: H and leading dimensions must be multiples of 8 (H=%d)", H);
  if ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: h, w and workspace must be 16-byte aligned");
  const Space at(n, top);
  const unsigned long long need = at.bytes;
  if (!workspace || workspace_bytes < need)
    return set_error(MORJ_ERR_ARG, "morj_token_logprobs: a workspace of %llu bytes given, %llu needed", workspace_bytes,
                     need);
  int st = configure();
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Scratch sc;
  sc.rows = chunk_rows(n), sc.top = top;
  char* ws = static_cast<char*>(workspace);
  sc.stats = reinterpret_cast<float4*>(ws);
  sc.own = reinterpret_cast<float*>(ws + at.own);
  sc.lists = reinterpret_cast<uint2*>(ws + at.lists);
  const Outputs o{targets, n_targets, logprobs_out, lse, entropy, top_ids, top_logprobs};
  for (int r0 = 0; r0 < n; r0 += CHUNK_ROWS) {
    const int rows = std::min(n - r0, CHUNK_ROWS);
    const int box = rows >= BM ? BM : (rows + 7) / 8 * 8;  // few rows: only those are loaded
    CUtensorMap mh;
    if ((st = make_map(&mh, static_cast<const __nv_bfloat16*>(h) + (size_t)r0 * ld_h, rows, H, ld_h, box))) return st;
    // Wide tiles where there are enough of them for most SMs, else four times as many narrow ones: the epilogue's passes
    // over a tile's columns are what a small call waits for (1 row, 4096 x 256, alone: 18 against 25 us).
    const int blocks = (rows + BM - 1) / BM, wide = (vocab + BN_WIDE - 1) / BN_WIDE;
    const int bn = (long long)blocks * wide * 2 > num_sms() ? BN_WIDE : BN_NARROW;
    const long long tiles = (long long)blocks * ((vocab + bn - 1) / bn);
    CUtensorMap mw;
    if ((st = make_map(&mw, w, vocab, H, ld_w, bn))) return st;
    const int ctas = (int)std::min<long long>(tiles, std::min(num_sms(), F_THREADS));
    // (CTAs with one tile each have no later tile to use a bound for: nothing to clear)
    sc.bound = top && tiles > ctas ? reinterpret_cast<unsigned*>(ws + at.bound) : nullptr;
    if (sc.bound) {
      const cudaError_t e = cudaMemsetAsync(sc.bound, 0, sc.rows * sizeof(unsigned), s);
      if (e != cudaSuccess) return set_error(MORJ_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
    }
    st = launch_pdl("logits_kernel", bn == BN_WIDE ? logits_kernel<BN_WIDE> : logits_kernel<BN_NARROW>, dim3(ctas),
                    dim3(THREADS), smem_bytes(bn), s, mh, mw, rows, vocab, H, box * BK * 2, softcap, sc);
    if (st) return st;
    st = launch_pdl("finish_kernel", finish_kernel, dim3(rows, n_targets ? 2 : 1), dim3(F_THREADS), 0, s,
                    (const __nv_bfloat16*)h, ld_h, (const __nv_bfloat16*)w, ld_w, vocab, H, softcap, ctas, sc, o, r0);
    if (st) return st;
  }
  return MORJ_OK;
}
