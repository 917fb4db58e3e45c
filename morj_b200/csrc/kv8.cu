// Store into and rows out of the 8-bit K/V cache (layout in kv8.cuh).
//
// A block of 64 slots and one head share a scale, the smallest power of two that keeps the block's values within e4m3's
// range. e4m3 is a floating-point format, so a scale larger than a row needs costs no precision until values reach the
// subnormals (2^-15 below the largest); scales therefore only grow, and a growing one moves exponents: resident codes
// are rescaled exactly unless they become subnormal.
//
// One CTA owns one (block, head) of K or V: it reads the block's new rows once into registers (all loads issued up front,
// eight CTAs an SM), reduces their largest magnitude, moves the block's other codes if the scale grew, and writes the new
// codes. No second pass over memory; the result does not depend on the order of the rows.
// Bound by HBM: 8,704 rows of 16 heads of 128, K and V, 107 MB in 20 us back to back = 5.3 TB/s (0.81 of the measured copy),
// 25 alone, 29 with cold caches (four CTAs an SM with rows asked for one after another: 52 us). 64 rows scattered over 256
// blocks: 9 us alone, a launch and three loads in a row.
#include <algorithm>
#include <vector>

#include "kv8.cuh"

namespace morj {
namespace kv8 {

constexpr int THREADS = 128;
constexpr float kBf16Max = 3.3895313892515355e38f;  // the largest finite BF16

struct Side {  // K or V
  const __nv_bfloat16* rows;
  long long ld;
  uint8_t* codes;
  float* scale;
};

// The largest magnitude in 8 BF16 values as bits of a BF16 (0x7f80 and above: not finite), pairs at a time.
MORJ_DEV unsigned amax_bits(unsigned m, const uint4& u) {
  m = __vmaxu2(m, u.x & 0x7fff7fffu);
  m = __vmaxu2(m, u.y & 0x7fff7fffu);
  m = __vmaxu2(m, u.z & 0x7fff7fffu);
  return __vmaxu2(m, u.w & 0x7fff7fffu);
}
MORJ_DEV uint32_t finite2(uint32_t two) {  // infinities and NaN as 0
  if ((two & 0x7f80u) == 0x7f80u) two &= 0xffff0000u;
  if ((two & 0x7f800000u) == 0x7f800000u) two &= 0x0000ffffu;
  return two;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 8) store_kernel(const Side k, const Side v, int n, int hk,
                                                           const int* __restrict__ work, int n_blocks,
                                                           int pool_slots) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  constexpr int LPR = D / 8;                       // lanes per row, 8 values each
  constexpr int ROWS = THREADS / LPR;              // rows per iteration of the CTA
  constexpr int ITERS = BLOCK / ROWS;
  __shared__ int2 pair[BLOCK];                     // (slot, row) of the rows; slot -1: none
  __shared__ unsigned red[THREADS / 32];
  __shared__ unsigned written[2];                  // slots of the block this call writes
  const int entry = blockIdx.x, h = blockIdx.y;
  const Side a = blockIdx.z ? v : k;
  const int block = work[3 * entry], first = work[3 * entry + 1], count = work[3 * entry + 2];
  const int part = threadIdx.x % LPR, r0 = threadIdx.x / LPR, lane = threadIdx.x % 32;
  const __nv_bfloat16* src = a.rows + (size_t)h * D + part * 8;
  uint8_t* codes = a.codes + (size_t)h * D + part * 8;
  const size_t row_bytes = (size_t)hk * D;
  if ((unsigned)count > BLOCK || block < 0 || (long long)block * BLOCK >= pool_slots) {
    if (threadIdx.x == 0) report(kErrBadIndex);
    return;
  }
  float* scale = a.scale + (size_t)block * hk + h;
  const float stored = *scale;
  if (threadIdx.x < BLOCK) {
    int2 p = make_int2(-1, 0);
    if (threadIdx.x < count) {
      p = reinterpret_cast<const int2*>(work + 3 * n_blocks + (n_blocks & 1))[first + threadIdx.x];
      if ((p.x >> BLOCK_SHIFT) != block || p.x >= pool_slots || (unsigned)p.y >= (unsigned)n) {
        report(kErrBadIndex);
        p = make_int2(-1, 0);
      }
    }
    pair[threadIdx.x] = p;
  }
  if (threadIdx.x < 2) written[threadIdx.x] = 0;
  __syncthreads();

  uint4 raw[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int2 p = pair[i * ROWS + r0];
    raw[i] = make_uint4(0, 0, 0, 0);
    if (p.x >= 0) raw[i] = *reinterpret_cast<const uint4*>(src + (size_t)p.y * a.ld);
  }
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < ITERS; ++i) m = amax_bits(m, raw[i]);
  m = max(m & 0xffffu, m >> 16);
  const bool bad = m >= 0x7f80u;
  if (bad) {  // infinite or NaN: reported, and not counted
    report(kErrNotFinite);
    m = 0;
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
      m = amax_bits(m, make_uint4(finite2(raw[i].x), finite2(raw[i].y), finite2(raw[i].z), finite2(raw[i].w)));
    m = max(m & 0xffffu, m >> 16);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[threadIdx.x / 32] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  const float amax = __uint_as_float(m << 16);
  const float old = stored > 0.f ? stored : 0.f;  // (0 or NaN: no codes yet)
  const float now = fmaxf(old, scale_for(amax));
  if (threadIdx.x == 0 && now != stored) *scale = now;  // (every thread read `stored` before the barriers above)

  if (old > 0.f && now > old) {
    // the block's scale grew: the codes of the slots this call does not write move to it
    if (threadIdx.x < count && pair[threadIdx.x].x >= 0) {
      const int at = pair[threadIdx.x].x & (BLOCK - 1);
      atomicOr(&written[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    const float ratio = old / now;  // (powers of two: exact)
#pragma unroll 2
    for (int r = r0; r < BLOCK; r += ROWS) {
      const long long s = (long long)block * BLOCK + r;
      if (s >= pool_slots || ((written[r >> 5] >> (r & 31)) & 1)) continue;
      uint2* p = reinterpret_cast<uint2*>(codes + (size_t)s * row_bytes);
      const uint2 c = *p;
      const float2 x0 = codes2_f32(c.x & 0xffffu), x1 = codes2_f32(c.x >> 16);
      const float2 x2 = codes2_f32(c.y & 0xffffu), x3 = codes2_f32(c.y >> 16);
      *p = make_uint2(f32_codes2(x0.x * ratio, x0.y * ratio) | f32_codes2(x1.x * ratio, x1.y * ratio) << 16,
                      f32_codes2(x2.x * ratio, x2.y * ratio) | f32_codes2(x3.x * ratio, x3.y * ratio) << 16);
    }
  }

  const float inv = 1.0f / now;  // (a power of two)
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int slot = pair[i * ROWS + r0].x;
    if (slot < 0) continue;
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= inv;
    if (bad) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? x[e] : 0.f;  // NaN: 0; infinite: saturated by the conversion
    }
    *reinterpret_cast<uint2*>(codes + (size_t)slot * row_bytes) =
        make_uint2(f32_codes2(x[0], x[1]) | f32_codes2(x[2], x[3]) << 16,
                   f32_codes2(x[4], x[5]) | f32_codes2(x[6], x[7]) << 16);
  }
}

// out[i, h, :] = bf16(code * scale) of pool row slots[i]; one warp-wide strip of 8 values per thread
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t* __restrict__ codes,
                                                     const float* __restrict__ scale, int pool_slots,
                                                     const int* __restrict__ slots, int hk, int d,
                                                     __nv_bfloat16* __restrict__ out, long long ld_out) {
  pdl_wait();  // the previous kernel on the stream has completed
  pdl_trigger();
  const int slot = slots[blockIdx.x];
  if ((unsigned)slot >= (unsigned)pool_slots) {
    if (threadIdx.x == 0) report(kErrBadIndex);
    return;
  }
  const int width = hk * d;
  const uint8_t* src = codes + (size_t)slot * width;
  const float* sc = scale + (size_t)(slot >> BLOCK_SHIFT) * hk;
  __nv_bfloat16* dst = out + (size_t)blockIdx.x * ld_out;
  for (int c = threadIdx.x * 8; c < width; c += blockDim.x * 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(src + c);
    const float s = sc[c / d];
    const float2 x0 = codes2_f32(u.x & 0xffffu), x1 = codes2_f32(u.x >> 16);
    const float2 x2 = codes2_f32(u.y & 0xffffu), x3 = codes2_f32(u.y >> 16);
    float v[8] = {x0.x * s, x0.y * s, x1.x * s, x1.y * s, x2.x * s, x2.y * s, x3.x * s, x3.y * s};
    // (a value that BF16's largest rounded up to, 2^128, comes back as that largest value; a NaN code stays one)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (fabsf(v[e]) > kBf16Max) v[e] = copysignf(kBf16Max, v[e]);
    store8(dst + c, v);
  }
}

static int store(const Side& k, const Side& v, int n, int hk, int d, const int* work, int n_blocks, int pool_slots,
                 cudaStream_t s) {
  const dim3 grid(n_blocks, hk, 2);
  if (d == 128)
    return launch_pdl("store_kernel", store_kernel<128>, grid, dim3(THREADS), 0, s, k, v, n, hk, work, n_blocks,
                      pool_slots);
  return launch_pdl("store_kernel", store_kernel<64>, grid, dim3(THREADS), 0, s, k, v, n, hk, work, n_blocks, pool_slots);
}

}  // namespace kv8
}  // namespace morj

extern "C" int morj_kv8_store_work(const int* slots_host, int n, int pool_slots, int* work_host, int cap) {
  using namespace morj;
  if (n < 0 || pool_slots < 0 || cap < 0 || (n && (!slots_host || !work_host))) {
    set_error(MORJ_ERR_ARG, "morj_kv8_store_work: bad arguments (n=%d pool_slots=%d)", n, pool_slots);
    return -1;
  }
  try {
    std::vector<std::pair<int, int>> order(n);  // (slot, row)
    for (int i = 0; i < n; ++i) {
      if (slots_host[i] < 0 || slots_host[i] >= pool_slots) {
        set_error(MORJ_ERR_ARG, "morj_kv8_store_work: row %d's slot %d is outside the pool of %d", i, slots_host[i],
                  pool_slots);
        return -1;
      }
      order[i] = {slots_host[i], i};
    }
    std::sort(order.begin(), order.end());
    int blocks = 0;
    for (int i = 0; i < n; ++i) {
      if (i && order[i].first == order[i - 1].first) {
        set_error(MORJ_ERR_ARG, "morj_kv8_store_work: rows %d and %d have the same slot %d", order[i - 1].second,
                  order[i].second, order[i].first);
        return -1;
      }
      blocks += !i || order[i].first / kv8::BLOCK != order[i - 1].first / kv8::BLOCK;
    }
    if ((long long)3 * blocks + (blocks & 1) + (long long)2 * n > cap) {
      set_error(MORJ_ERR_ARG, "morj_kv8_store_work: %d blocks and %d rows exceed capacity %d", blocks, n, cap);
      return -1;
    }
    int* pairs = work_host + 3 * blocks + (blocks & 1);  // (8-byte aligned pairs)
    if (blocks & 1) pairs[-1] = 0;
    for (int i = 0, b = -1; i < n; ++i) {
      const int block = order[i].first / kv8::BLOCK;
      if (b < 0 || work_host[3 * b] != block) {
        ++b;
        work_host[3 * b] = block;
        work_host[3 * b + 1] = i;
        work_host[3 * b + 2] = 0;
      }
      ++work_host[3 * b + 2];
      pairs[2 * i] = order[i].first;
      pairs[2 * i + 1] = order[i].second;
    }
    return blocks;
  } catch (...) {
    set_error(MORJ_ERR_OOM, "morj_kv8_store_work: out of host memory");
    return -1;
  }
}

extern "C" int morj_kv8_store(const void* k, long long ld_k, const void* v, long long ld_v, int n, int hk, int d,
                              const int* work, int n_blocks, void* k_codes, float* k_scale, void* v_codes,
                              float* v_scale, int pool_slots, void* stream) {
  using namespace morj;
  if (n == 0 || n_blocks == 0) return MORJ_OK;
  if (!k || !v || !work || !k_codes || !k_scale || !v_codes || !v_scale || n < 0 || n_blocks < 0 || n_blocks > n ||
      pool_slots <= 0 || hk <= 0 || hk > 65535)
    return set_error(MORJ_ERR_ARG, "morj_kv8_store: null pointer or bad size (n=%d n_blocks=%d hk=%d pool_slots=%d)", n,
                     n_blocks, hk, pool_slots);
  if (d != 64 && d != 128) return set_error(MORJ_ERR_UNSUPPORTED, "morj_kv8_store: head_dim %d unsupported (64, 128)", d);
  if (ld_k % 8 || ld_v % 8 || ld_k < (long long)hk * d || ld_v < (long long)hk * d)
    return set_error(MORJ_ERR_ARG, "morj_kv8_store: leading dimensions %lld, %lld must be multiples of 8, at least %d",
                     ld_k, ld_v, hk * d);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_codes) |
       reinterpret_cast<uintptr_t>(v_codes)) & 15)
    return set_error(MORJ_ERR_ARG, "morj_kv8_store: rows and codes must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(work) & 7) || ((reinterpret_cast<uintptr_t>(k_scale) |
                                                   reinterpret_cast<uintptr_t>(v_scale)) & 3))
    return set_error(MORJ_ERR_ARG, "morj_kv8_store: work must be 8-byte, scales 4-byte aligned");
  const kv8::Side ks{(const __nv_bfloat16*)k, ld_k, (uint8_t*)k_codes, k_scale};
  const kv8::Side vs{(const __nv_bfloat16*)v, ld_v, (uint8_t*)v_codes, v_scale};
  return kv8::store(ks, vs, n, hk, d, work, n_blocks, pool_slots, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int morj_kv8_gather(const void* codes, const float* scale, int pool_slots, const int* slots, int n, int hk,
                               int d, void* out, long long ld_out, void* stream) {
  using namespace morj;
  if (n == 0) return MORJ_OK;
  if (!codes || !scale || !slots || !out || n < 0 || pool_slots <= 0 || hk <= 0 || d <= 0 || d % 8)
    return set_error(MORJ_ERR_ARG, "morj_kv8_gather: null pointer or bad size (n=%d hk=%d d=%d)", n, hk, d);
  if (ld_out % 8 || ld_out < (long long)hk * d)
    return set_error(MORJ_ERR_ARG, "morj_kv8_gather: leading dimension %lld must be a multiple of 8, at least %d",
                     ld_out, hk * d);
  if ((reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15))
    return set_error(MORJ_ERR_ARG, "morj_kv8_gather: codes and out must be 16-byte aligned");
  return launch_pdl("gather_kernel", kv8::gather_kernel, dim3(n), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream),
                    (const uint8_t*)codes, scale, pool_slots, slots, hk, d, (__nv_bfloat16*)out, ld_out);
}
