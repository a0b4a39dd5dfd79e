// Shared by the cache writers and the attention kernels over pages (sparse.hip, kv8.hip): page
// lookup, waits, lane swaps, and the norm and rotation of the rows that are written.
#pragma once
#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int PAGE = 16;
constexpr float kLog2e = 1.4426950408889634f;

inline hipStream_t S(void* s) { return (hipStream_t)s; }

// This wave of the workgroup, as a scalar: what depends on it alone is scalar work then.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// The block of request b's page, or -1 past the table's width or where the entry is no block.
__device__ __forceinline__ int page_block(const int32_t* __restrict__ table, int64_t stride, int b,
                                          int64_t page, int64_t blocks) {
  if (page < 0 || page >= stride) return -1;
  const int e = table[(int64_t)b * stride + page];
  return e >= 0 && e < blocks ? e : -1;
}

// s_waitcnt on the vector-memory counter only (gfx9 encoding: vmcnt in bits 3:0 and 15:14, no wait on
// the others).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// On the LDS counter only: this wave's LDS reads have ended.
__device__ __forceinline__ void wait_lgkmcnt0() {
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));
}

// Workgroup barrier without the wait of __syncthreads for every load in flight.
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The maximum over the four lanes of a column (lanes col, col + 16, ..), by row and half-wave swaps.
__device__ __forceinline__ float column_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// The same with NaN kept, and the sum, in a fixed order.
__device__ __forceinline__ float column_maximum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Inclusive prefix sums over the wave's lanes, by row shifts and broadcasts.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // lanes 1, 2, 4, 8 back in a row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // lane 15 to the next row
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // lane 31 to the upper half
  return v;
}

// op over W neighbouring lanes, in every one of them: lanes 32 apart, then 16, 8, 4, 2 and 1.
template <int W, typename Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op) {
  static_assert(W == 8 || W == 16 || W == 32 || W == 64, "neighbours that have a head's row or part of it");
  if constexpr (W == 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (W >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (W >= 16) {
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));   // 8 round a row of 16
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));   // 4: eighths are alike
  } else {
    const int up = __builtin_amdgcn_update_dpp((int)v, (int)v, 0x104, 0xf, 0x5, false);    // 4 on, lanes 0 .. 3 of 8
    v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(up, (int)v, 0x114, 0xf, 0xa, false));  // 4 back, lanes 4 .. 7
  }
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));
  return op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));
}

template <int W>
__device__ __forceinline__ float sum_over_lanes(float v) {
  return __uint_as_float(over_lanes<W>(__float_as_uint(v), [](uint32_t x, uint32_t y) {
    return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
  }));
}

// What the norm and rotation of elements 8 c .. 8 c + 7 take besides the row: gammas of these and of
// their partners, and angles, the sine with the sign of its term. Loaded once for a thread's heads.
struct Rotation {
  u32x4 gamma, other_gamma;
  float cosv[8], sinv[8];
  float eps;
  int partner;             // the thread of the rotation's other half
  bool norm, turn;
};

__device__ __forceinline__ Rotation load_rotation(int c, const uint16_t* gamma, float eps, const float* cr,
                                                  const float* sr, int half) {
  Rotation a;
  const int h8 = half / 8;
  a.eps = eps;
  a.partner = c < h8 ? c + h8 : c < 2 * h8 ? c - h8 : c;
  a.norm = gamma != nullptr;
  a.turn = c < 2 * h8;
  if (a.norm) {
    a.gamma = *(const u32x4*)(gamma + 8 * c);
    a.other_gamma = *(const u32x4*)(gamma + 8 * a.partner);
  }
  if (a.turn) {
    const int i0 = c < h8 ? 8 * c : 8 * (c - h8);
    const float sign = c < h8 ? -1.f : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a.cosv[e] = cr[i0 + e];
      a.sinv[e] = sign * sr[i0 + e];
    }
  }
  return a;
}

// Eight elements y of a head, d = 8 c .. 8 c + 7, normalised and rotated in fp32; the D / 8 threads of a
// head are neighbours in one wave. The rotation partner's raw words come from its thread.
template <int D>
__device__ __forceinline__ void rotate_norm_f32(float (&y)[8], u32x4 raw, const Rotation& a) {
  constexpr int W = D / 8;
  float inv = 1.f;
  if (a.norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = __uint_as_float(raw[i] << 16), hi = __uint_as_float(raw[i] & 0xffff0000u);
      ss = __builtin_fmaf(lo, lo, ss);
      ss = __builtin_fmaf(hi, hi, ss);
    }
    ss = sum_over_lanes<W>(ss);
    inv = __frsqrt_rn(ss / (float)D + a.eps);
  }
  u32x4 other;
#pragma unroll
  for (int i = 0; i < 4; ++i) other[i] = (uint32_t)__shfl((int)raw[i], a.partner, W);
  float z[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = __uint_as_float(raw[i] << 16) * inv;
    y[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u) * inv;
    z[2 * i] = __uint_as_float(other[i] << 16) * inv;
    z[2 * i + 1] = __uint_as_float(other[i] & 0xffff0000u) * inv;
  }
  if (a.norm) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] *= __uint_as_float(a.gamma[i] << 16);
      y[2 * i + 1] *= __uint_as_float(a.gamma[i] & 0xffff0000u);
      z[2 * i] *= __uint_as_float(a.other_gamma[i] << 16);
      z[2 * i + 1] *= __uint_as_float(a.other_gamma[i] & 0xffff0000u);
    }
  }
  if (a.turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(y[e], a.cosv[e], z[e] * a.sinv[e]);
  }
}

// The same, rounded once to bf16.
template <int D>
__device__ __forceinline__ u32x4 rotate_norm(u32x4 raw, const Rotation& a) {
  float y[8];
  rotate_norm_f32<D>(y, raw, a);
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
  return o;
}

// Query rows [batch, T] of a cache write: row m, head h at q + m * stride + h * D, to out [rows, Hq, D].
struct QueryRows {
  const uint16_t* q;       // null: no queries
  int64_t stride;
  const uint16_t* gamma;   // null: no norm
  const float* cosv;       // [rows, half], rows cs_stride apart
  const float* sinv;
  int64_t cs_stride;
  float eps;
  uint16_t* out;
  const int32_t* starts;   // [batch] position of a request's first row; negative: none of its rows
  const int32_t* counts;   // [batch] its rows
  int batch, T, Hq, half;
};

constexpr int Q_HEADS = 4;   // heads of a row that a thread rotates: their loads are in flight at once

// The queries of a cache write: D / 8 neighbouring threads take unit u, Q_HEADS heads of one row
// (ceil(heads / Q_HEADS) units a row), c of them this thread. PASS_BY: past the caches (queries_pass_by).
template <int D, bool PASS_BY>
__device__ __forceinline__ void rotate_queries(uint32_t u, int c, const QueryRows& a) {
  const uint32_t groups = (uint32_t)(a.Hq + Q_HEADS - 1) / Q_HEADS;
  const uint32_t m = u / groups;
  const int head = (int)(u % groups) * Q_HEADS;
  const uint32_t b = m / (uint32_t)a.T;
  const bool live = b < (uint32_t)a.batch && (int)(m % (uint32_t)a.T) < a.counts[b] && a.starts[b] >= 0;
  const int64_t mr = live ? m : 0;
  const int heads = live ? a.Hq - head < Q_HEADS ? a.Hq - head : Q_HEADS : 0;
  u32x4 raw[Q_HEADS];
#pragma unroll
  for (int i = 0; i < Q_HEADS; ++i) {
    raw[i] = u32x4{0u, 0u, 0u, 0u};
    const u32x4* p = (const u32x4*)(a.q + mr * a.stride + (int64_t)(head + i) * D + 8 * c);
    if (i < heads) raw[i] = PASS_BY ? __builtin_nontemporal_load(p) : *p;
  }
  const Rotation turn =
      load_rotation(c, a.gamma, a.eps, a.cosv + mr * a.cs_stride, a.sinv + mr * a.cs_stride, a.half);
#pragma unroll
  for (int i = 0; i < Q_HEADS; ++i) {
    const u32x4 o = rotate_norm<D>(raw[i], turn);
    u32x4* p = (u32x4*)(a.out + (mr * a.Hq + head + i) * D + 8 * c);
    if (i >= heads) continue;
    if (PASS_BY) __builtin_nontemporal_store(o, p);
    else *p = o;
  }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
constexpr int64_t MAX_BATCH_ROWS = 1 << 24;   // batch * tokens

// A launch holds fewer than 2^32 threads.
inline bool grid_ok(int64_t wgs, int64_t threads) { return wgs <= 0xffffffffll / threads; }

// Whether a cache write's queries go past the caches: from 40 MiB of them on, which go in and out beside the
// keys and values. Over three sets of buffers in turn, 34 MB of queries take 18.3 us and past the caches 20.3
// (17 MB 11.7 and 13.3, 1.2 MB 4.4 and 4.9), 50 MB 28.4 and 27.0, 134 MB 68 and 62.
inline bool queries_pass_by(int64_t rows, int64_t Hq, int64_t D) { return rows * Hq * D * 2 >= (40ll << 20); }

inline bool head_shape_ok(int64_t batch, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D) {
  return batch >= 0 && tokens >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq <= 4096 &&
         (D == 64 || D == 128 || D == 256) &&
         (tokens == 0 || batch <= MAX_BATCH_ROWS / tokens);
}

}  // namespace
