// Tree attention over the 8-bit K/V cache (kv8.cuh): the mask rules of tree_attention_kernel, K and V read as e4m3
// codes and scaled per (block of 64 slots, head).
//
//   s_ij = sm_scale * (q_i . code_k[j]) * scale_k[block(j)],  p = softmax over the visible j,
//   o_i  = sum_j p_ij * scale_v[block(j)] * code_v[j],        a row that sees nothing is 0.
//
// Codes become FP16 by one conversion for two of them (exact), so both products run as FP16 x FP16 with FP32 sums and
// the scales stay out of the operands: K's multiplies the scores, V's the probabilities (relative to the largest V
// scale met so far, so the products stay inside FP16 and O is kept in units of that scale). A query row is brought to
// [1, 2) by a power of two before it is rounded to FP16, which keeps every bit of a BF16 row that matters at 2^-25 of
// its largest element.
//
// rows_kernel: tiles of 8 or 16 rows (a segment's (query, head) pairs of one KV head), for the single-token form. Every
// warp walks its own groups of 32 keys with mma.m16n8k16, operands straight from global memory: the fragment layouts
// leave the order of the head dimension (QK) and of the output columns (PV) free, so each lane reads 16 or 32
// consecutive codes of a key. The host cuts the keys of a tile into parts until the SMs are filled; parts leave
// (maximum, sum, O) in a workspace and combine_kernel joins them.
#include <algorithm>
#include <climits>
#include <vector>

#include "kv8.cuh"

namespace morj {
namespace kv8 {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int UNIT = 16;             // rows of a partial unit in the workspace
constexpr int WARPS = 4;
constexpr int STEP = 32;             // keys a warp takes at a time
constexpr float P_SCALE = 1024.0f;   // probabilities are rounded to FP16 as 1024 p: 2^-34 is their smallest step

struct Item {
  int seg, r0;         // segment, its first row (row = query * G + head of the group)
  int t0, t1;          // keys [t0, t1) of the segment's list
  int unit;            // first partial unit, -1: the only part, straight to `out`
  int parts, stride;   // combine entries: parts, and units between them
  int tile;            // rows of the tile
};

struct Args {
  const __nv_bfloat16* q;
  const uint8_t* k;
  const float* ks;
  const uint8_t* v;
  const float* vs;
  __nv_bfloat16* out;
  const int* qo_indptr;
  const int* kv_indptr;
  const int* kv_indices;
  const int* kv_last_page_len;
  int n_bidir, hq, hk, page_size, window, pool_slots;
  float scale_log2;
  float* ws;
};

struct Seg {
  int q_start, q_len, kv_base, kv_len;
};
MORJ_DEV Seg load_segment(const Args& a, int seg) {
  Seg s;
  s.q_start = a.qo_indptr[seg];
  s.q_len = a.qo_indptr[seg + 1] - s.q_start;
  s.kv_base = a.kv_indptr[seg];
  const int pages = a.kv_indptr[seg + 1] - s.kv_base;
  s.kv_len = a.page_size == 1 ? pages
             : pages == 0     ? 0
                              : (pages - 1) * a.page_size + (a.kv_last_page_len ? a.kv_last_page_len[seg] : a.page_size);
  return s;
}

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

// pool slot of key t of a segment, -1 (device error recorded) outside the pool
MORJ_DEV int key_slot(const Args& a, int kv_base, int t) {
  const long long page = __ldg(a.kv_indices + kv_base + (a.page_size == 1 ? t : t / a.page_size));
  const long long slot = a.page_size == 1 ? page : page * a.page_size + t % a.page_size;
  if (slot < 0 || slot >= a.pool_slots) {
    report(kErrBadIndex);
    return -1;
  }
  return (int)slot;
}

MORJ_DEV void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with rows 8..15 of A zero: their sums are dropped
MORJ_DEV void mma_f16_top(float (&c)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  float x, y;
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"
               : "+f"(c[0]), "+f"(c[1]), "=f"(x), "=f"(y)
               : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}
// maximum that keeps a NaN
MORJ_DEV float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
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

// N consecutive codes of one head of a pool row
template <int N>
MORJ_DEV void load_codes(const uint8_t* p, bool ok, uint32_t (&w)[N / 4]) {
  if constexpr (N == 8) {
    const uint2 u = ok ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
    w[0] = u.x, w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 u = ok ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
      w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
    }
  }
}

// ROWS = 8 or 16 rows per tile. Rows 8..15 of the MMA's 16 are zeros when ROWS = 8 and cost no registers.
template <int D, int ROWS>
__global__ void __launch_bounds__(WARPS * 32) rows_kernel(const Args a, const Item* __restrict__ items) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  constexpr int KS = D / 16;       // MMA depth steps of q . k
  constexpr int NT = D / 8;        // 8-column output tiles
  constexpr int HALVES = ROWS / 8;
  constexpr int KRUN = D / 4;      // consecutive codes of a key one lane reads of K
  constexpr int VRUN = D / 8;      // ... and of V
  __shared__ float sh_o[WARPS][ROWS][D];
  __shared__ float sh_m[WARPS][ROWS], sh_l[WARPS][ROWS];

  const Item it = items[blockIdx.x / a.hk];
  const int h = blockIdx.x % a.hk;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, c4 = lane % 4;
  const Seg sg = load_segment(a, it.seg);
  const bool bidir = it.seg < a.n_bidir;
  const int G = a.hq / a.hk, n_rows = sg.q_len * G;
  const int t_end = min(it.t1, sg.kv_len);

  // this lane's rows: r0 + g and r0 + g + 8
  uint32_t qf[HALVES][KS][2];
  float qs[HALVES];
  int lo[HALVES], hi[HALVES];
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    const int r = it.r0 + g + 8 * b;
    lo[b] = INT_MAX, hi[b] = -1, qs[b] = 0.f;
    float v[KRUN];
#pragma unroll
    for (int i = 0; i < KRUN; ++i) v[i] = 0.f;
    if (r < n_rows) {
      visible(sg.q_len, sg.kv_len, bidir, a.window, r / G, &lo[b], &hi[b]);
      const __nv_bfloat16* src = a.q + ((size_t)(sg.q_start + r / G) * a.hq + h * G + r % G) * D + c4 * KRUN;
#pragma unroll
      for (int i = 0; i < KRUN; i += 8) {
        float x[8];
        load8(src + i, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i + e] = x[e];
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < KRUN; ++i) amax = fmaxf(amax, fabsf(v[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    qs[b] = row_scale(amax);
    const float inv = 1.f / qs[b];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[b][s][0] = pack_f16x2(v[4 * s] * inv, v[4 * s + 1] * inv);
      qf[b][s][1] = pack_f16x2(v[4 * s + 2] * inv, v[4 * s + 3] * inv);
    }
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[HALVES], l[HALVES];
#pragma unroll
  for (int b = 0; b < HALVES; ++b) m[b] = -INFINITY, l[b] = 0.f;
  float vref = 0.f;  // the largest V scale met: O is in units of vref / P_SCALE

  const size_t head_off = (size_t)h * D;
  const size_t row_codes = (size_t)a.hk * D;
  for (int base = it.t0 + warp * STEP; base < t_end; base += WARPS * STEP) {
    // lane = key: its pool row and scales
    int slot = -1;
    float kf = 0.f, vf = 0.f;
    if (base + lane < t_end) slot = key_slot(a, sg.kv_base, base + lane);
    if (slot >= 0) {
      const size_t si = (size_t)(slot >> BLOCK_SHIFT) * a.hk + h;
      kf = __ldg(a.ks + si) * a.scale_log2;
      vf = __ldg(a.vs + si);
    }
    uint32_t kw[4][KRUN / 4], vw[2][4][VRUN / 4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = __shfl_sync(0xffffffffu, slot, j * 8 + g);
      load_codes<KRUN>(a.k + (s < 0 ? 0 : (size_t)s * row_codes + head_off + c4 * KRUN), s >= 0, kw[j]);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = __shfl_sync(0xffffffffu, slot, kk * 16 + (e >> 1) * 8 + c4 * 2 + (e & 1));
        load_codes<VRUN>(a.v + (s < 0 ? 0 : (size_t)s * row_codes + head_off + g * VRUN), s >= 0, vw[kk][e]);
      }
    // V scales: O moves to the new unit when a larger one appears
    float vmax = vf;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, x));
    float unit = 1.f;  // old unit / new unit
    if (vmax > vref) {
      unit = vref / vmax;
      vref = vmax;
    }
    vf *= vref > 0.f ? P_SCALE / vref : 0.f;

    // scores of 8 keys per MMA column tile: rows g (and g + 8), keys c4 * 2 + {0, 1}
    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const uint32_t b0 = codes2_f16(kw[j][x] & 0xffffu), b1 = codes2_f16(kw[j][x] >> 16);
        if constexpr (HALVES == 2)
          mma_f16(s[j], qf[0][x][0], qf[1][x][0], qf[0][x][1], qf[1][x][1], b0, b1);
        else
          mma_f16_top(s[j], qf[0][x][0], qf[0][x][1], b0, b1);
      }
    }
    float mx[HALVES];
#pragma unroll
    for (int b = 0; b < HALVES; ++b) mx[b] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = j * 8 + c4 * 2 + e, t = base + key;
        const float f = __shfl_sync(0xffffffffu, kf, key);
#pragma unroll
        for (int b = 0; b < HALVES; ++b) {
          float& x = s[j][2 * b + e];
          x = (t >= lo[b] && t <= hi[b] && t < t_end) ? x * (f * qs[b]) : -INFINITY;
          mx[b] = max_nan(mx[b], x);
        }
      }
    float alpha[HALVES];
#pragma unroll
    for (int b = 0; b < HALVES; ++b) {
      mx[b] = max_nan(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 1));
      mx[b] = max_nan(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 2));
      const float now = max_nan(m[b], mx[b]);
      alpha[b] = m[b] == -INFINITY ? 0.f : exp2f(m[b] - now);
      m[b] = now;
      l[b] *= alpha[b];
      alpha[b] *= unit;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[HALVES - 1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int b = 0; b < HALVES; ++b) o[j][2 * b] *= alpha[b], o[j][2 * b + 1] *= alpha[b];
    }
    uint32_t pf[HALVES][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f0 = __shfl_sync(0xffffffffu, vf, j * 8 + c4 * 2), f1 = __shfl_sync(0xffffffffu, vf, j * 8 + c4 * 2 + 1);
#pragma unroll
      for (int b = 0; b < HALVES; ++b) {
        const float shift = m[b] == -INFINITY ? 0.f : m[b];
        const float p0 = exp2f(s[j][2 * b] - shift), p1 = exp2f(s[j][2 * b + 1] - shift);
        l[b] += p0 + p1;
        pf[b][j] = pack_f16x2(p0 * f0, p1 * f1);
      }
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int w = 0; w < VRUN / 4; ++w) {
        // four output columns: the codes of keys (0, 1) and (8, 9) of the 16-key step, paired per column
        const uint32_t a01 = prmt(vw[kk][0][w], vw[kk][1][w], 0x5140), a23 = prmt(vw[kk][0][w], vw[kk][1][w], 0x7362);
        const uint32_t b01 = prmt(vw[kk][2][w], vw[kk][3][w], 0x5140), b23 = prmt(vw[kk][2][w], vw[kk][3][w], 0x7362);
        const uint32_t av[4] = {a01 & 0xffffu, a01 >> 16, a23 & 0xffffu, a23 >> 16};
        const uint32_t bv[4] = {b01 & 0xffffu, b01 >> 16, b23 & 0xffffu, b23 >> 16};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b0 = codes2_f16(av[e]), b1 = codes2_f16(bv[e]);
          if constexpr (HALVES == 2)
            mma_f16(o[4 * w + e], pf[0][2 * kk], pf[1][2 * kk], pf[0][2 * kk + 1], pf[1][2 * kk + 1], b0, b1);
          else
            mma_f16_top(o[4 * w + e], pf[0][2 * kk], pf[0][2 * kk + 1], b0, b1);
        }
      }
  }

  // the four warps' results, joined
  const float scale_o = vref / P_SCALE;
#pragma unroll
  for (int b = 0; b < HALVES; ++b) {
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 1);
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 2);
    const int r = g + 8 * b;
    if (c4 == 0) sh_m[warp][r] = m[b], sh_l[warp][r] = l[b];
    // column tile j, column n of the MMA is output column n * VRUN + j
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sh_o[warp][r][(2 * c4) * VRUN + j] = o[j][2 * b] * scale_o;
      sh_o[warp][r][(2 * c4 + 1) * VRUN + j] = o[j][2 * b + 1] * scale_o;
    }
  }
  __syncthreads();
  float* part = it.unit < 0 ? nullptr : a.ws + ((size_t)it.unit * a.hk + h) * (UNIT * (D + 2));
  for (int i = threadIdx.x; i < ROWS * D; i += WARPS * 32) {
    const int r = i / D, d = i % D;
    if (it.r0 + r >= n_rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      mm = fmaxf(mm, sh_m[w][r]);
    }
    float ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = sh_m[w][r] == -INFINITY ? 0.f : exp2f(sh_m[w][r] - mm);
      ll += f * sh_l[w][r];
      oo += f * sh_o[w][r][d];
    }
    if (part) {
      if (d == 0) part[r] = mm, part[UNIT + r] = ll;
      part[2 * UNIT + r * D + d] = oo;
    } else {
      const int row = it.r0 + r;
      a.out[((size_t)(sg.q_start + row / G) * a.hq + h * G + row % G) * D + d] =
          __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
    }
  }
}

// Joins the parts of one 16-row unit: o = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p.
template <int D>
__global__ void __launch_bounds__(D) combine_kernel(const Args a, const Item* __restrict__ items) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  const Item it = items[blockIdx.x / a.hk];
  const int h = blockIdx.x % a.hk, d = threadIdx.x;
  const Seg sg = load_segment(a, it.seg);
  const int G = a.hq / a.hk, n_rows = sg.q_len * G;
  const size_t step = (size_t)it.stride * a.hk * (UNIT * (D + 2));
  const float* first = a.ws + ((size_t)it.unit * a.hk + h) * (UNIT * (D + 2));
  for (int r = blockIdx.y; r < UNIT && it.r0 + r < n_rows && r < it.tile; r += gridDim.y) {
    float mm = -INFINITY;
    for (int p = 0; p < it.parts; ++p) mm = fmaxf(mm, __ldcg(first + p * step + r));
    float ll = 0.f, oo = 0.f;
    for (int p = 0; p < it.parts; ++p) {
      const float* part = first + p * step;
      const float mp = __ldcg(part + r);
      const float f = mp == -INFINITY ? 0.f : exp2f(mp - mm);
      ll += f * __ldcg(part + UNIT + r);
      oo += f * __ldcg(part + 2 * UNIT + r * D + d);
    }
    const int row = it.r0 + r;
    a.out[((size_t)(sg.q_start + row / G) * a.hq + h * G + row % G) * D + d] =
        __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
  }
}

template <int D>
static int launch(const Args& a, const int* counts, const int* work, cudaStream_t s) {
  const Item* items = reinterpret_cast<const Item*>(work);
  const int n_rows = counts[0], n_combine = counts[1];
  int st = MORJ_OK;
  if (n_rows) {
    const dim3 grid((unsigned)n_rows * a.hk);
    st = counts[3] == 8
             ? launch_pdl("rows_kernel", rows_kernel<D, 8>, grid, dim3(WARPS * 32), 0, s, a, items)
             : launch_pdl("rows_kernel", rows_kernel<D, 16>, grid, dim3(WARPS * 32), 0, s, a, items);
  }
  if (st == MORJ_OK && n_combine)
    st = launch_pdl("combine_kernel", combine_kernel<D>, dim3((unsigned)n_combine * a.hk, 4), dim3(D), 0, s, a,
                    items + n_rows);
  return st;
}

}  // namespace kv8
}  // namespace morj

extern "C" int morj_tree_attention_kv8_work(const int* qo_indptr_host, const int* kv_indptr_host,
                                            const int* kv_last_page_len_host, int n_segments, int n_bidir, int hq,
                                            int hk, int page_size, int window, int* work_host, int cap, int* counts) {
  using namespace morj;
  using kv8::Item;
  if (!qo_indptr_host || !kv_indptr_host || !counts || n_segments < 0 || n_bidir < 0 || n_bidir > n_segments ||
      hk <= 0 || hq <= 0 || hq % hk || page_size <= 0 || cap < 0 || (cap && !work_host)) {
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: bad arguments");
  }
  const int G = hq / hk;
  try {
    std::vector<Item> items, joins;
    int rows_max = 0;
    long long total = 0;  // keys over all tiles
    for (int s = 0; s < n_segments; ++s) {
      const long long rows = (long long)(qo_indptr_host[s + 1] - qo_indptr_host[s]) * G;
      if (rows < 0 || rows > (1 << 30) || kv_indptr_host[s + 1] < kv_indptr_host[s])
        return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: segment %d's tables are out of order", s);
      rows_max = std::max(rows_max, (int)rows);
    }
    const int tile = rows_max <= 8 ? 8 : 16;
    for (int s = 0; s < n_segments; ++s) {
      const int q_len = qo_indptr_host[s + 1] - qo_indptr_host[s];
      const int pages = kv_indptr_host[s + 1] - kv_indptr_host[s];
      const long long kv =
          page_size == 1 || pages == 0
              ? pages
              : (long long)(pages - 1) * page_size + (kv_last_page_len_host ? kv_last_page_len_host[s] : page_size);
      if (kv < 0 || kv > INT_MAX)
        return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: segment %d has %lld keys", s, kv);
      for (int r0 = 0; r0 < q_len * G; r0 += tile) {
        int lo, hi, x;  // what the tile's first query sees from, its last query to
        kv8::visible(q_len, (int)kv, s < n_bidir, window, r0 / G, &lo, &x);
        kv8::visible(q_len, (int)kv, s < n_bidir, window, (std::min(r0 + tile, q_len * G) - 1) / G, &x, &hi);
        Item it{s, r0, 0, 0, -1, 1, 1, tile};
        if (hi >= lo) it.t0 = lo, it.t1 = hi + 1;
        total += it.t1 - it.t0;
        items.push_back(it);
      }
    }
    // parts: about four CTAs' worth of warps per SM, at least 256 keys each
    const long long slots = (long long)num_sms() * 4;
    long long len = (total * hk + slots - 1) / slots;
    len = std::max(256LL, (len + 127) / 128 * 128);
    std::vector<Item> cut;
    int units = 0;
    for (const Item& it : items) {
      const int keys = it.t1 - it.t0;
      const int parts = keys > len ? (int)((keys + len - 1) / len) : 1;
      if (parts == 1) {
        cut.push_back(it);
        continue;
      }
      const int step = ((keys + parts - 1) / parts + 127) / 128 * 128;
      Item join = it;
      join.unit = units, join.parts = 0;
      for (int t = it.t0; t < it.t1; t += step) {
        Item part = it;
        part.t0 = t, part.t1 = std::min(it.t1, t + step);
        part.unit = units++;
        ++join.parts;
        cut.push_back(part);
      }
      joins.push_back(join);
    }
    // longest first: the last CTAs to start are the short ones
    std::stable_sort(cut.begin(), cut.end(), [](const Item& x, const Item& y) { return x.t1 - x.t0 > y.t1 - y.t0; });
    counts[0] = (int)cut.size();
    counts[1] = (int)joins.size();
    counts[2] = units;
    counts[3] = tile;
    counts[4] = (int)((cut.size() + joins.size()) * (sizeof(Item) / sizeof(int)));
    const size_t need = (cut.size() + joins.size()) * (sizeof(Item) / sizeof(int));
    if (need > (size_t)cap) {
      if (cap == 0) return MORJ_OK;  // (a call that only asks for the counts)
      return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8_work: %zu ints exceed capacity %d", need, cap);
    }
    std::copy(cut.begin(), cut.end(), reinterpret_cast<Item*>(work_host));
    std::copy(joins.begin(), joins.end(), reinterpret_cast<Item*>(work_host) + cut.size());
    return MORJ_OK;
  } catch (...) {
    return set_error(MORJ_ERR_OOM, "morj_tree_attention_kv8_work: out of host memory");
  }
}

extern "C" int morj_tree_attention_kv8(const void* q, int n_q, const void* k_codes, const float* k_scale,
                                       const void* v_codes, const float* v_scale, int pool_slots, void* out,
                                       const int* qo_indptr, const int* kv_indptr, const int* kv_indices,
                                       const int* kv_last_page_len, int n_segments, int n_bidir, int hq, int hk, int d,
                                       int page_size, int window, float sm_scale, const int* work, const int* counts,
                                       void* workspace, unsigned long long workspace_bytes, void* stream) {
  using namespace morj;
  if (!counts) return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: null counts");
  if (counts[0] == 0 || n_segments == 0) return MORJ_OK;
  if (!q || !k_codes || !k_scale || !v_codes || !v_scale || !out || !qo_indptr || !kv_indptr || !kv_indices || !work ||
      n_q <= 0 || pool_slots <= 0 || counts[0] < 0 || counts[1] < 0 || counts[2] < 0)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: null pointer or bad size");
  if (hq <= 0 || hk <= 0 || hq % hk)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: hq=%d is not a multiple of hk=%d", hq, hk);
  if (page_size <= 0 || n_bidir < 0 || n_bidir > n_segments)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: bad page_size %d or n_bidir %d", page_size, n_bidir);
  if (d != 64 && d != 128)
    return set_error(MORJ_ERR_UNSUPPORTED, "morj_tree_attention_kv8: head_dim %d unsupported (64, 128)", d);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(workspace)) &
      15)
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: q, codes, out, work and workspace must be 16-byte aligned");
  const unsigned long long need = (unsigned long long)counts[2] * hk * kv8::UNIT * (d + 2) * sizeof(float);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(MORJ_ERR_ARG, "morj_tree_attention_kv8: a workspace of %llu bytes given, %llu needed",
                     workspace_bytes, need);
  const kv8::Args a{(const __nv_bfloat16*)q, (const uint8_t*)k_codes, k_scale, (const uint8_t*)v_codes, v_scale,
                    (__nv_bfloat16*)out, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, n_bidir, hq, hk, page_size,
                    window, pool_slots, sm_scale * kv8::LOG2E, (float*)workspace};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return d == 128 ? kv8::launch<128>(a, counts, work, s) : kv8::launch<64>(a, counts, work, s);
}
