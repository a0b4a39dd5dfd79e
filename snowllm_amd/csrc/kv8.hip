// The paged KV cache in 8 bits, in four operators:
//
//   axes      cos and sin of rotary positions with several axes
//   append    the cache write of new rows: optional per-head RMSNorm, rotate-half RoPE, quantised
//   read      cached rows back in bf16
//   attend    softmax attention of new rows over the cache, causal or by ancestor masks
//
// The cache: codes of a (token, kv head)'s row x with one fp32 scale,
//   scale = max(max_d |x_d|, 2^-100) / 127,  code_d = rint(x_d / scale),  x_d ~ code_d * scale,
// in pages of 16 tokens: K [blocks, Hkv, 4, d/16, 4, 16] (token t is group t / 4, place t % 4), V
// [blocks, Hkv, d, 16], scales [blocks, Hkv, 16]. A row with an element that is not finite has a NaN
// scale and zero codes. The least scale keeps 127 / max finite and every scale a normal number; elements
// below half of it (2^-101 / 127) read back as zeros.
//
// The layouts are the operands of the attention's 64-key products (v_mfma_i32_16x16x64_i8): 16 bytes
// of K are 16 elements of a token, 16 bytes of V the 16 tokens of a page at one element, and a lane's
// scores are of one page, see attend.
#include "common.h"
#include "pages.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float LEAST = 0x1p-100f;

struct Cache {
  int8_t* k;
  int8_t* v;
  float* k_scale;
  float* v_scale;
};

// ---------------------------------------------------------------------------------------
// axes
// ---------------------------------------------------------------------------------------
constexpr int MAX_AXES = 4;

struct AxesArgs {
  const int64_t* pos;      // [axes, rows]
  const float* inv_freq;   // [half]
  float* cosv;             // [rows, half]
  float* sinv;
  int64_t rows;
  int half, axes, interleaved;
  int count[MAX_AXES];     // pairs of each axis
};

// cos and sin of 2 pi t for |t| <= 1/2: a quarter turn and what is left, |z| <= pi / 4, rounded to 32 bits
// once; its Taylor series to z^9 and z^8 leave less than 2^-24.
__device__ __forceinline__ void cos_sin_turns(double t, float& c, float& s) {
  const double quarter = rint(4. * t);
  const float z = (float)((t - 0.25 * quarter) * 6.28318530717958647693), y = z * z;
  float a = __builtin_fmaf(y, 1.f / 362880.f, -1.f / 5040.f);
  a = __builtin_fmaf(y, a, 1.f / 120.f);
  a = __builtin_fmaf(y, a, -1.f / 6.f);
  a = __builtin_fmaf(y * z, a, z);
  float b = __builtin_fmaf(y, 1.f / 40320.f, -1.f / 720.f);
  b = __builtin_fmaf(y, b, 1.f / 24.f);
  b = __builtin_fmaf(y, b, -0.5f);
  b = __builtin_fmaf(y, b, 1.f);
  const int q = (int)quarter;   // -2 .. 2
  const float x = q & 1 ? a : b, w = q & 1 ? b : a;
  c = __uint_as_float(__float_as_uint(x) ^ ((uint32_t)(q + 1) & 2u) << 30);
  s = __uint_as_float(__float_as_uint(w) ^ ((uint32_t)q & 2u) << 30);
}

// The angle in turns, pos * inv_freq / 2 pi, is taken in 64 bits and without its whole turns: a
// 32-bit product at position 220000 is off by up to 2^-7 of a radian. A thread takes V pairs of AXES_ROWS
// rows, whose frequencies it converts once; bound by its writes (262144 rows of 32 pairs: 73 MB in 15 us).
constexpr int AXES_ROWS = 4;

template <int V>
__global__ void __launch_bounds__(256) axes_kernel(AxesArgs a) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x, cols = (uint32_t)(a.half / V);
  const int64_t m0 = (int64_t)(idx / cols) * AXES_ROWS;
  const int i0 = (int)(idx % cols) * V;
  if (m0 >= a.rows) return;
  int axis[V];
  double freq[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = i0 + v;
    axis[v] = 0;
    if (a.interleaved) {
      const int x = i % a.axes;
#pragma unroll
      for (int k = 0; k < MAX_AXES; ++k)
        if (k == x && i / a.axes < a.count[k]) axis[v] = k;
    } else {
      int end = 0;
#pragma unroll
      for (int k = 0; k < MAX_AXES - 1; ++k) {
        end += a.count[k];
        if (k + 1 < a.axes && i >= end) axis[v] = k + 1;
      }
    }
    freq[v] = (double)a.inv_freq[i] * 0.15915494309189533577;
  }
#pragma unroll
  for (int r = 0; r < AXES_ROWS; ++r) {
    const int64_t m = m0 + r;
    if (m >= a.rows) return;
    float c[V], s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double turns = (double)a.pos[axis[v] * a.rows + m] * freq[v];
      cos_sin_turns(turns - rint(turns), c[v], s[v]);
    }
    float* cp = a.cosv + m * a.half + i0;
    float* sp = a.sinv + m * a.half + i0;
    if constexpr (V == 4) {
      *(floatx4*)cp = floatx4{c[0], c[1], c[2], c[3]};
      *(floatx4*)sp = floatx4{s[0], s[1], s[2], s[3]};
    } else {
      *cp = c[0];
      *sp = s[0];
    }
  }
}

// ---------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------
struct AppendArgs {
  QueryRows rows;          // the queries, rotated alongside
  const uint16_t* k;       // row m, head h at k + m * k_stride + h * D
  const uint16_t* v;
  int64_t k_stride, v_stride;
  const uint16_t* k_gamma; // null: no norm
  Cache cache;
  const int32_t* table;
  int64_t table_stride, blocks;
  int Hkv, pages;          // pages: most pages that T rows touch
  int64_t page_wgs;        // workgroups over (request, page, kv head); the rest rotate queries
};

// Eight codes of a row whose D / 8 threads are neighbours in a wave, and its scale. Magnitudes are
// compared as integers, in which infinities and NaN lie above all finite values.
template <int D>
__device__ __forceinline__ u32x2 quantise(const float (&y)[8], float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  top = over_lanes<D / 8>(top, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
  const bool fine = top < 0x7f800000u;
  const float most = fmaxf(__uint_as_float(top), LEAST);
  scale = fine ? __fdiv_rn(most, 127.f) : __uint_as_float(0x7fc00000u);
  const float inv = __fdiv_rn(127.f, most);
  u32x2 w = {0u, 0u};
  if (fine)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e >> 2] |= (uint32_t)((int)rintf(y[e] * inv) & 255) << (8 * (e & 3));
  return w;
}

// 2 D threads: sixteen rows of D / 8 threads each. A page workgroup owns one (request, page, kv head):
// its threads take a token's row each, and the codes go through LDS into the page's layout, so that every
// write is of 16 bytes but in pages that begin or end a request. Bound by bytes, most of them the
// queries' (8192 rows of 16 + 2 heads of 256: 145 MB in 31 us).
template <int D, bool PASS_BY>
__global__ void __launch_bounds__(2 * D) append_kernel(AppendArgs a) {
  constexpr int W = D / 8, VP = D + 8;   // VP: pitch of V's codes in LDS, by token
  __shared__ __attribute__((aligned(16))) uint8_t ks[PAGE * D];
  __shared__ __attribute__((aligned(16))) uint8_t vs[PAGE * VP];
  const int tid = threadIdx.x, r = tid / W, c = tid % W;
  int64_t wg = blockIdx.x;
  if (wg >= a.page_wgs) {
    rotate_queries<D, PASS_BY>((uint32_t)(wg - a.page_wgs) * 16 + r, c, a.rows);
    return;
  }
  const int h = (int)(wg % a.Hkv);
  wg /= a.Hkv;
  const int j = (int)(wg % a.pages), b = (int)(wg / a.pages);
  const int64_t start = a.rows.starts[b];
  int64_t count = a.rows.counts[b];
  count = count < a.rows.T ? count : a.rows.T;
  if (start < 0 || count <= 0) return;
  const int64_t page = start / PAGE + j, first = page * PAGE;
  const int64_t end = start + count;   // one past the last position
  if (first >= end) return;
  const int blk = page_block(a.table, a.table_stride, b, page, a.blocks);
  if (blk < 0) return;
  const int lo = start > first ? (int)(start - first) : 0;             // new tokens lo .. hi - 1
  const int hi = end - first < PAGE ? (int)(end - first) : PAGE;
  const int64_t at = (int64_t)blk * a.Hkv + h;
  {
    const bool live = r >= lo && r < hi;
    const int64_t m = (int64_t)b * a.rows.T + (live ? first + r - start : 0);
    u32x4 kraw = {0u, 0u, 0u, 0u}, vraw = {0u, 0u, 0u, 0u};
    if (live) {
      kraw = *(const u32x4*)(a.k + m * a.k_stride + (int64_t)h * D + 8 * c);
      vraw = *(const u32x4*)(a.v + m * a.v_stride + (int64_t)h * D + 8 * c);
    }
    float y[8], z[8], k_scale, v_scale;
    rotate_norm_f32<D>(y, kraw, load_rotation(c, a.k_gamma, a.rows.eps, a.rows.cosv + m * a.rows.cs_stride,
                                              a.rows.sinv + m * a.rows.cs_stride, a.rows.half));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[2 * i] = __uint_as_float(vraw[i] << 16);
      z[2 * i + 1] = __uint_as_float(vraw[i] & 0xffff0000u);
    }
    const u32x2 kc = quantise<D>(y, k_scale), vc = quantise<D>(z, v_scale);
    *(u32x2*)(ks + ((r / 4) * (D / 16) + c / 2) * 64 + (r % 4) * 16 + (c % 2) * 8) = kc;
    *(u32x2*)(vs + r * VP + 8 * c) = vc;
    if (live && c == 0) {
      a.cache.k_scale[at * PAGE + r] = k_scale;
      a.cache.v_scale[at * PAGE + r] = v_scale;
    }
  }
  __syncthreads();
  if (tid < D) {   // 16 bytes of K: token, sixteen elements
    const int tok = tid / (D / 4) * 4 + tid % 4;
    if (tok >= lo && tok < hi)
      *(u32x4*)(a.cache.k + at * PAGE * D + tid * 16) = *(const u32x4*)(ks + tid * 16);
  } else {         // an element of V: its tokens
    const int d = tid - D;
    int8_t* vp = a.cache.v + at * PAGE * D + d * 16;
    if (hi - lo == PAGE) {
      u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < PAGE; ++t) w[t >> 2] |= (uint32_t)vs[t * VP + d] << (8 * (t & 3));
      *(u32x4*)vp = w;
    } else {
      for (int t = lo; t < hi; ++t) vp[t] = (int8_t)vs[t * VP + d];
    }
  }
}

// ---------------------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------------------
struct ReadArgs {
  Cache cache;
  const int32_t* table;
  const int32_t* starts;
  const int32_t* counts;
  uint16_t* k;             // [rows, Hkv, D]
  uint16_t* v;
  int64_t table_stride, blocks;
  int T, Hkv, pages;
};

// Eight codes times their scale, rounded once to bf16.
__device__ __forceinline__ u32x4 values(u32x2 w, float scale) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = (int)w[i >> 1] >> (16 * (i & 1));
    o[i] = pack_bf16x2((float)(int8_t)(x & 255) * scale, (float)(int8_t)(x >> 8 & 255) * scale);
  }
  return o;
}

// 2 D threads take a (request, page, kv head): sixteen rows of D / 8 threads each; V goes through LDS. Bound
// by bytes (131071 rows of 2 heads of 256: 405 MB in 79 us).
template <int D>
__global__ void __launch_bounds__(2 * D) read_kernel(ReadArgs a) {
  constexpr int W = D / 8, VP = D + 8;
  __shared__ __attribute__((aligned(16))) uint8_t vs[PAGE * VP];
  const int tid = threadIdx.x, r = tid / W, c = tid % W;
  int64_t wg = blockIdx.x;
  const int h = (int)(wg % a.Hkv);
  wg /= a.Hkv;
  const int j = (int)(wg % a.pages), b = (int)(wg / a.pages);
  const int64_t start = a.starts[b];
  int64_t count = a.counts[b];
  count = count < a.T ? count : a.T;
  if (start < 0 || count <= 0) return;
  const int64_t page = start / PAGE + j, first = page * PAGE, end = start + count;
  if (first >= end) return;
  const int blk = page_block(a.table, a.table_stride, b, page, a.blocks);
  if (blk < 0) return;
  const int64_t at = (int64_t)blk * a.Hkv + h;
  const u32x2 kc = *(const u32x2*)(a.cache.k + at * PAGE * D + ((r / 4) * (D / 16) + c / 2) * 64 +
                                   (r % 4) * 16 + (c % 2) * 8);
  const float k_scale = a.cache.k_scale[at * PAGE + r], v_scale = a.cache.v_scale[at * PAGE + r];
  {   // half of an element's tokens, by token into LDS
    const int d = tid % D, t0 = tid / D * 8;
    const u32x2 w = *(const u32x2*)(a.cache.v + at * PAGE * D + d * 16 + t0);
#pragma unroll
    for (int t = 0; t < 8; ++t) vs[(t0 + t) * VP + d] = (uint8_t)(w[t >> 2] >> (8 * (t & 3)));
  }
  __syncthreads();
  const int64_t pos = first + r;
  if (pos < start || pos >= end) return;
  const int64_t o = (((int64_t)b * a.T + pos - start) * a.Hkv + h) * D + 8 * c;
  *(u32x4*)(a.k + o) = values(kc, k_scale);
  *(u32x4*)(a.v + o) = values(*(const u32x2*)(vs + r * VP + 8 * c), v_scale);
}

// ---------------------------------------------------------------------------------------
// attend
// ---------------------------------------------------------------------------------------
// The products run on the 8-bit matrix cores, exactly, with q and the weights as two 8-bit terms:
//   q_d = qs (256 h_d + l_d),   qs = max(max |q|, 2^-100) / 32512: off by at most 2^-16 of the row's largest
//   S_k = scale qs ks_k (256 K_k.h + K_k.l)
//   p_k = 2^(S_k log2 e - m),   l = sum p_k,   m from the row's maximum to 2^4 above it
//   p_k vs_k = g (256 a_k + b_k),  g = max(max_k (p_k vs_k) / 32512, 2^-126) over 64 or 128 keys
//   o_d += g (256 V_d.a + V_d.b),  sums of integers below 2^31, o and l in fp32
// h and l are signed bytes; a is in 0 .. 127, b signed. Because g follows the keys, one with a large
// weight costs only its neighbours' weights precision (2^-16 of it), not the whole context's.
//
// Rows of a kv head are ordered r = t * G + g, in tiles of 16 (columns of the products). For four
// pages, product n = 0 .. 3 takes row 4 q + i of its K operand from page q, token 4 n + i; then the
// lane (column, q) holds the scores of page q's sixteen tokens, in the order of the V operand's bytes
// (16 bytes: the page's tokens at one element), and the weights go from the scores' registers into the
// second product's operand without leaving the lane.
struct AttendArgs {
  const uint16_t* q;       // row m at q + m * q_stride
  int64_t q_stride;
  Cache cache;
  uint16_t* out;           // [rows, Hq, D]
  const int32_t* table;
  const int32_t* starts;
  const int32_t* counts;
  const uint64_t* tree;    // [rows] ancestor masks or null (causal)
  float* part_o;           // [Hkv, slots, tiles, 16, D]
  float* part_ml;          // [Hkv, slots, tiles, 16, 2]
  int64_t table_stride, blocks;
  int T, Hq, Hkv, G, tiles;
  int slots;               // workgroups of a kv head and tiles
  int splits;              // of every request, 0: by the requests' lengths, batch <= 64 and <= slots
  int batch;
  int unit, longer;        // a split's share of a request's steps; the first `longer` have one more
  uint32_t g_inv;          // floor(2^32 / G), at most 2^32 - 1
  float scale;
};

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float TERM = 32512.f;      // the largest value of two terms, 127 * 256
constexpr float MARGIN = 4.f;        // how far m is set above a row's maximum, as an exponent of 2

// One row of a lane's column: it sees the positions below `end`, and those from there on by its mask.
struct Row {
  int64_t m;               // its index, -1: no row
  int head, end;
  uint64_t mask;
};

template <int D>
struct RowState {
  float o[D / 4];          // elements 16 t + 4 quad + i at 4 t + i
  float m, l;
};

template <int D>
struct Query {
  i32x4 h[D / 64], l[D / 64];
  float s;                 // scores' factor, as an exponent of 2
};

// Row r of a kv head as (token, head of its group). r g_inv / 2^32 is below r / G by less than r / 2^32 + 1.
struct RowPlace {
  int t, g;
};
__device__ __forceinline__ RowPlace place(const AttendArgs& a, int r) {
  int t = (int)__umulhi((uint32_t)r, a.g_inv), g = r - t * a.G;
  if (g >= a.G) ++t, g -= a.G;
  return {t, g};
}

__device__ __forceinline__ int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

__device__ __forceinline__ Row find_row(const AttendArgs& a, int b, int h, int r, int64_t start, int count) {
  Row x{-1, 0, 0, 0};
  const RowPlace at = place(a, r);
  const int t = at.t;
  if (t >= count) return x;
  x.m = (int64_t)b * a.T + t;
  x.head = h * a.G + at.g;
  // nothing past the table
  const int64_t width = a.table_stride * PAGE;
  const int64_t end = a.tree ? start : start + t + 1;
  x.end = (int)(end < width ? end : width);
  if (a.tree) {
    const int64_t left = width - start, n = count < left ? count : left;
    x.mask = a.tree[x.m] & (n >= 64 ? ~0ull : n > 0 ? (1ull << n) - 1 : 0ull);
  }
  return x;
}

// Which of the sixteen positions from p on a row sees, by bits.
__device__ __forceinline__ uint32_t seen_from(const Row& x, int p) {
  const int n = x.end - p;
  if (n >= 16) return 0xffffu;
  const uint32_t below = n > 0 ? (1u << n) - 1 : 0u;
  const uint64_t own = n >= 0 ? x.mask << n : -n < 64 ? x.mask >> -n : 0ull;
  return below | ((uint32_t)own & 0xffffu);
}

// Four values as two terms each, in bytes: z = x + 2^23 (+ 2^22) + 128 has x + 128 in its low bits, of
// which the second byte is the larger term and the first, less 128, the smaller.
__device__ __forceinline__ void two_terms(const float (&z)[4], int& h, int& l) {
  const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(z[1]), __float_as_uint(z[0]), 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(z[3]), __float_as_uint(z[2]), 0x05010400u);
  l = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
  h = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
}

// A row as it is, fetched before its request's lengths are known (one past the last: the first one's).
template <int D>
struct RawQuery {
  u32x4 w[D / 64][2];
};

template <int D>
__device__ __forceinline__ void fetch_query(RawQuery<D>& raw, const AttendArgs& a, int b, int h, int r, int quad) {
  const RowPlace at = place(a, r);
  const uint16_t* p =
      a.q + ((int64_t)b * a.T + (at.t < a.T ? at.t : 0)) * a.q_stride + (int64_t)(h * a.G + at.g) * D + 16 * quad;
#pragma unroll
  for (int s = 0; s < D / 64; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i) raw.w[s][i] = *(const u32x4*)(p + 64 * s + 8 * i);
}

// A row that is not `there` (past the request's count) as zeros: whatever its memory holds would have a say in
// when the maxima of the tile's other rows move, and so in their bits. False where an element is not finite: such a
// row's scores are finite and mean nothing, so that its sum says whether it sees a key (see sum_of).
template <int D>
__device__ __forceinline__ bool quantise_query(Query<D>& q, const AttendArgs& a, const RawQuery<D>& raw, bool there) {
  float v[D / 64][16], top = 0.f;
#pragma unroll
  for (int s = 0; s < D / 64; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = there ? raw.w[s][i][e] : 0u;
        v[s][8 * i + 2 * e] = __uint_as_float(w << 16);
        v[s][8 * i + 2 * e + 1] = __uint_as_float(w & 0xffff0000u);
      }
#pragma unroll
  for (int s = 0; s < D / 64; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[s][e]));   // NaN stays
  top = column_maximum(top);
  // in units of 2^-100 / 32512 at least: elements below half of that count as zeros
  const float most = fmaxf(top, LEAST);
  const float f = a.scale < 0.f ? -TERM / most : TERM / most;
  // (never zero: a hidden key's -inf times it stays -inf)
  const bool fine = top < __builtin_huge_valf();
  q.s = fine ? fmaxf(most * (1.f / TERM) * __builtin_fabsf(a.scale) * kLog2e, 0x1p-126f) : 0x1p-126f;
#pragma unroll
  for (int s = 0; s < D / 64; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = __builtin_fmaf(v[s][4 * e + i], f, 12583040.f);
      int h, l;
      two_terms(z, h, l);
      q.h[s][e] = h;
      q.l[s][e] = l;
    }
  return fine;
}

// The sum l of a row's weights, NaN where its query is not finite and it sees a key.
__device__ __forceinline__ float sum_of(float l, bool fine) {
  return fine || l == 0.f ? l : __uint_as_float(0x7fc00000u);
}

// N times 64 keys (four pages): of the c-th, k(c, n, s) is the K operand of product n, elements 64 s ..,
// v(c, t) the V operand of elements 16 t .., ks(c, n) and vs(c, n) the scales of this lane's page, tokens
// 4 n ... Where !all, this lane's row sees the tokens of its pages whose bits `seen` has, sixteen a page.
// scored() is called when k, ks and vs are done with, feed(i) with i = 0, 1, .. once a stage of the
// products, 4 N + D / 16 times.
template <int D, int N, typename K, typename V, typename KS, typename VS, typename Scored, typename Feed>
__device__ __forceinline__ void attend_keys(RowState<D>& st, const Query<D>& q, K k, V v, KS ks, VS vs,
                                            Scored scored, Feed feed, bool all, uint32_t seen) {
  constexpr int NS = D / 64;
  float x[16 * N], p[16 * N];   // scores; scales of V, then weights times them
  // stage n loads what product n + 1 takes, issues product n and converts product n - 2, whose sums are
  // there by then
  {
    i32x4 w[2][NS], hi[3], lo[3];
    floatx4 f[3];
#pragma unroll
    for (int n = -1; n < 4 * N + 2; ++n) {
      if (n + 1 < 4 * N) {
#pragma unroll
        for (int s = 0; s < NS; ++s) w[(n + 1) & 1][s] = k((n + 1) / 4, (n + 1) % 4, s);
      }
      if (n >= 0 && n < 4 * N) {
        f[n % 3] = ks(n / 4, n % 4);
        hi[n % 3] = lo[n % 3] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          hi[n % 3] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[n & 1][s], q.h[s], hi[n % 3], 0, 0, 0);
          lo[n % 3] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[n & 1][s], q.l[s], lo[n % 3], 0, 0, 0);
        }
        feed(n);
      }
      if (n >= 2) {
        const int m = n - 2;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[4 * m + i] = (float)(int)(((uint32_t)hi[m % 3][i] << 8) + (uint32_t)lo[m % 3][i]) * f[m % 3][i];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int n = 0; n < 4 * N; ++n) {
    const floatx4 g = vs(n / 4, n % 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[4 * n + i] = g[i];
  }
  scored();
  if (!all) {
    asm volatile("" : "+v"(seen));   // stays a branch: most keys are seen by every row
#pragma unroll
    for (int j = 0; j < 16 * N; ++j) {   // the scales of a key that is not there may be anything
      const bool s = seen >> j & 1;
      x[j] = s ? x[j] : NEG_INF;
      p[j] = s ? p[j] : 0.f;
    }
  }
  float top = x[0];
#pragma unroll
  for (int j = 1; j < 16 * N; ++j) top = fmaxf(top, x[j]);
  top *= q.s;
  // m (the same in the four lanes of a row) moves only when a score is above it somewhere in the wave, and
  // then past it: weights are at most 1, so that with any V in bf16 their products are finite, and the
  // largest at least 2^-4, so that 2^15 units of them are with V's least scale too.
  if (__builtin_amdgcn_ballot_w64(top > st.m) != 0) {
    const float m = fmaxf(st.m, column_max(top) + MARGIN);
    const float f = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(st.m - m);
#pragma unroll
    for (int d = 0; d < D / 4; ++d) st.o[d] *= f;
    st.l *= f;
    st.m = m;
  }
  const float nm = st.m == NEG_INF ? 0.f : -st.m;
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 16 * N; ++j) {
    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], q.s, nm));
    st.l += e;
    p[j] *= e;
  }
#pragma unroll
  for (int j = 0; j < 16 * N; ++j) most = __builtin_elementwise_maximum(most, p[j]);   // NaN stays
  most = column_maximum(most);
  // g and its inverse are of one number that both can hold: products below 2^-111 get a unit of 2^-126, which
  // is 2^-19 of V's least scale
  const float g = __builtin_elementwise_maximum(most * (1.f / TERM), 0x1p-126f);   // NaN stays
  const float f = __builtin_amdgcn_rcpf(g);
  i32x4 pa[N], pb[N], w[2][N];
#pragma unroll
  for (int c = 0; c < N; ++c) w[0][c] = v(c, 0);
#pragma unroll
  for (int n = 0; n < 4 * N; ++n) {
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __builtin_fmaf(p[4 * n + i], f, 8388736.f);
    int h, l;
    two_terms(z, h, l);
    pa[n / 4][n % 4] = h;
    pb[n / 4][n % 4] = l;
  }
  __builtin_amdgcn_sched_barrier(0);
  constexpr int T = D / 16;
  i32x4 hi[3], lo[3];
#pragma unroll
  for (int t = 0; t < T + 2; ++t) {
    if (t + 1 < T) {
#pragma unroll
      for (int c = 0; c < N; ++c) w[(t + 1) & 1][c] = v(c, t + 1);
    }
    if (t < T) {
      hi[t % 3] = lo[t % 3] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < N; ++c) {
        hi[t % 3] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t & 1][c], pa[c], hi[t % 3], 0, 0, 0);
        lo[t % 3] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t & 1][c], pb[c], lo[t % 3], 0, 0, 0);
      }
      feed(4 * N + t);
    }
    if (t >= 2) {
      const int m = t - 2;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st.o[4 * m + i] = __builtin_fmaf((float)(int)(((uint32_t)hi[m % 3][i] << 8) + (uint32_t)lo[m % 3][i]), g,
                                         st.o[4 * m + i]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int D>
__device__ __forceinline__ void clear(RowState<D>& st) {
#pragma unroll
  for (int d = 0; d < D / 4; ++d) st.o[d] = 0.f;
  st.m = NEG_INF;
  st.l = 0.f;
}

template <int D>
__device__ __forceinline__ floatx4 elements(const RowState<D>& st, int t) {
  return floatx4{st.o[4 * t], st.o[4 * t + 1], st.o[4 * t + 2], st.o[4 * t + 3]};
}

__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }   // NaN stays

// A slot's part of a request, as far as the keys go: the splits of the request are the slots from `first`.
struct Slot {
  int b, first, splits, c0, c1;
};

// Steps of STEP chunks of 64 keys that request b's rows see (one where there are rows and no key).
template <int STEP>
__device__ __forceinline__ int request_steps(const AttendArgs& a, int b) {
  const int64_t start = a.starts[b];
  int64_t count = a.counts[b], end;
  count = count < a.T ? count : a.T;
  end = start + count < a.table_stride * PAGE ? start + count : a.table_stride * PAGE;
  if (start < 0 || count <= 0) return 0;
  return end > 0 ? (int)((end + 64 * STEP - 1) / (64 * STEP)) : 1;
}

// The slot `slot`, or the first one of request b (slot < 0). Where the lengths decide, every wave finds
// the least steps a slot, from the mean on, with which all requests' splits have slots: lane b has request
// b. (Sixteen blocks of 9 rows behind 4K to 8K tokens: 7 steps at most instead of 9.)
template <int STEP>
__device__ __forceinline__ Slot find_slot(const AttendArgs& a, int slot, int b) {
  if (a.splits) {
    if (slot >= 0) b = slot / a.splits;
    const int split = slot - b * a.splits;
    return {b, b * a.splits, a.splits, STEP * (split * a.unit + (split < a.longer ? split : a.longer)),
            STEP * ((split + 1) * a.unit + (split + 1 < a.longer ? split + 1 : a.longer))};
  }
  const int lane = threadIdx.x & 63;
  const int steps = lane < a.batch ? request_steps<STEP>(a, lane) : 0;
  const int total = __builtin_amdgcn_readlane(wave_scan(steps), 63);
  int share = (total + a.slots - 1) / a.slots, mine, upto;
  share = share > 0 ? share : 1;
  for (;;) {   // ends: with a share of the longest request, requests need no more slots than there are
    mine = (int)((unsigned)(steps + share - 1) / (unsigned)share);
    upto = wave_scan(mine);
    if (__builtin_amdgcn_readlane(upto, 63) <= a.slots) break;
    share += 1 + share / 16;
  }
  if (slot >= 0) {
    const uint64_t found = __builtin_amdgcn_ballot_w64(slot < upto);
    if (found == 0) return {-1, 0, 0, 0, 0};   // no part is left for it
    b = __builtin_ctzll(found);
  }
  const int splits = __builtin_amdgcn_readlane(mine, b), first = __builtin_amdgcn_readlane(upto, b) - splits;
  return {b, first, splits, STEP * share * (slot - first), STEP * share * (slot - first + 1)};
}

// The workgroup's kv head, group of tiles and slot. Workgroups go to the eight XCDs in turn: those that
// read the same keys, the groups of a (head, slot), are eight apart, so that their XCD's cache has the keys
// (9 rows of 16 heads behind 24000 tokens 20 us; 28 with the groups side by side).
struct Spot {
  int h, group, slot;
};

__device__ __forceinline__ Spot find_spot(int Hkv, int groups) {
  if (groups == 1) return {(int)blockIdx.x, 0, (int)blockIdx.y};   // heads side by side, as in memory
  const uint32_t n = (uint32_t)groups, pairs = (uint32_t)Hkv * gridDim.y, whole = pairs / 8 * 8;
  uint32_t at = blockIdx.y * gridDim.x + blockIdx.x, first = 0, wide = 8;
  if (at >= whole * n) {
    at -= whole * n;
    first = whole;
    wide = pairs - whole;
  }
  const uint32_t row = at / wide, pair = first + row / n * wide + (at - row * wide);
  return {(int)(pair % (uint32_t)Hkv), (int)(row % n), (int)(pair / (uint32_t)Hkv)};
}

// What a workgroup does: tiles of a (request, kv head) against the chunks c0 .. c1 - 1 of 64 keys.
struct Share {
  int64_t start;           // position of the request's first row
  int64_t end;             // one past the last position that the tiles see
  int count;               // the request's rows; 0: nothing to do
  int b, h, slot, c0, c1;
  bool single;             // no other split
};

// The first tile and how many: chunks up to the last position that one of their rows sees.
__device__ __forceinline__ Share find_share(const AttendArgs& a, int start, int count, const Slot& at, int slot, int h,
                                            int tile, int tiles) {
  Share w{start, 0, count, at.b, h, slot, at.c0, 0, at.splits == 1};
  w.count = w.count < a.T ? w.count : a.T;
  if (w.start < 0 || w.count <= 0 || (int64_t)tile * 16 >= (int64_t)w.count * a.G) {
    w.count = 0;
    return w;
  }
  int t_last = place(a, (tile + tiles) * 16 - 1).t;
  t_last = t_last < w.count ? t_last : w.count - 1;
  w.end = a.tree ? w.start + w.count : w.start + t_last + 1;
  w.end = w.end < a.table_stride * PAGE ? w.end : a.table_stride * PAGE;
  w.c1 = (int)min64((w.end + 63) / 64, at.c1);
  return w;
}

// Four elements of a row's result.
template <int D>
__device__ __forceinline__ void write_out(const AttendArgs& a, int64_t m, int head, int d, floatx4 o, float f) {
  *(u32x2*)(a.out + (m * a.Hq + head) * D + d) =
      u32x2{pack_bf16x2(o[0] * f, o[1] * f), pack_bf16x2(o[2] * f, o[3] * f)};
}

// A row's place among the splits' states.
__device__ __forceinline__ int64_t part_row(const AttendArgs& a, const Share& w, int r) {
  return (((int64_t)w.h * a.slots + w.slot) * a.tiles + r / 16) * 16 + r % 16;
}

__device__ __forceinline__ void write_sums(const AttendArgs& a, int64_t part, float m, float l) {
  a.part_ml[part * 2] = m;
  a.part_ml[part * 2 + 1] = l;
}

// The states of a tile's N waves joined through LDS (os: a pitch of D + 4 floats a row).
template <int D, int N>
__device__ __forceinline__ void join_waves(const AttendArgs& a, const Share& w, const RowState<D>& st, float* os,
                                           float (*ml)[16][2], int wave, int tile) {
  constexpr int P = D + 4;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const float l = column_sum(st.l);
#pragma unroll
  for (int t = 0; t < D / 16; ++t) *(floatx4*)(os + (wave * 16 + col) * P + t * 16 + 4 * quad) = elements(st, t);
  if (quad == 0) {
    ml[wave][col][0] = st.m;
    ml[wave][col][1] = l;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < 16 * (D / 4); u += 64 * N) {
    const int r = u / (D / 4), d = u % (D / 4) * 4, row = tile * 16 + r;
    const RowPlace at = place(a, row);
    if (at.t >= w.count) break;   // rows only grow
    float m = NEG_INF, sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) m = fmaxf(m, ml[n][r][0]);
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float f = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(ml[n][r][0] - m);
      sum += f * ml[n][r][1];
      o += f * *(const floatx4*)(os + (n * 16 + r) * P + d);
    }
    if (w.single) {
      write_out<D>(a, (int64_t)w.b * a.T + at.t, w.h * a.G + at.g, d, o, inverse_sum(sum));
    } else {
      const int64_t part = part_row(a, w, row);
      *(floatx4*)(a.part_o + part * D + d) = o;
      if (d == 0) write_sums(a, part, m, sum);
    }
  }
}

// A workgroup for each (request, kv head, tile, split); the waves take the split's chunks in turn and
// join their states at the end. Operands come straight from memory into registers, the next chunk's K as
// soon as the scores are done and its V after the products, so that a wave has 64 D .. 128 D bytes in
// flight all the time. Bound by bytes for single tokens (64 requests of 8192 tokens, 8 kv heads of 128: 836 MB
// in 154 us), by the chain of table, keys, join where there are few (one: 8 us and 3 for the join).
constexpr int WAVES = 4;

// The arguments that the first loads take come again in front, where they arrive in registers.
#define KV8_FRONT                                                                                             \
  const int32_t *__restrict__ h_table, const int32_t *__restrict__ h_starts, const int32_t *__restrict__ h_counts, \
      const uint16_t *__restrict__ h_q, int64_t h_table_stride, int h_splits, int h_unit, int h_longer,       \
      int h_tiles, int h_Hkv, uint32_t h_g_inv, AttendArgs a
#define KV8_TAKE_FRONT                                                                     \
  a.table = h_table, a.starts = h_starts, a.counts = h_counts, a.q = h_q;                  \
  a.table_stride = h_table_stride, a.splits = h_splits, a.unit = h_unit, a.longer = h_longer; \
  a.tiles = h_tiles, a.Hkv = h_Hkv, a.g_inv = h_g_inv

template <int D>
__global__ void __launch_bounds__(64 * WAVES) attend_kernel(KV8_FRONT) {
  KV8_TAKE_FRONT;
  constexpr int NS = D / 64, T = D / 16;
  __shared__ __attribute__((aligned(16))) float os[WAVES * 16 * (D + 4)];
  __shared__ float ml[WAVES][16][2];
  const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15, quad = lane >> 4;
  const Spot spot = find_spot(a.Hkv, a.tiles);
  const int h = spot.h, tile = spot.group;
  const Slot slot = find_slot<WAVES>(a, spot.slot, 0);
  const int b = slot.b;
  if (b < 0) return;
  const int start = a.starts[b], count = a.counts[b];
  const int64_t page_bytes = PAGE * D, block_bytes = page_bytes * a.Hkv;
  const int8_t* kh = a.cache.k + h * page_bytes + quad * 64 + (col & 3) * 16;
  const int8_t* vh = a.cache.v + h * page_bytes + col * 16;
  const int32_t* trow = a.table + (int64_t)b * a.table_stride;
  // the blocks of this lane's page of K and of V, -1: none
  struct Pages {
    int k, v;
  };
  auto look_up = [&](int c) {
    const int64_t pk = 4ll * c + (col >> 2), pv = 4ll * c + quad;
    const int64_t last = a.table_stride - 1;
    if (last < 0) return Pages{-1, -1};   // (uniform)
    Pages p{trow[pk < last ? pk : last], trow[pv < last ? pv : last]};
    p.v = pv <= last ? p.v : -1;   // (a K of another page is a V that is not there: hidden)
    return p;
  };
  auto valid = [&](int e) { return e >= 0 && e < a.blocks; };
  int c = slot.c0 + wave;
  Pages here = look_up(c), next = look_up(c + WAVES);
  RawQuery<D> raw;
  fetch_query(raw, a, b, h, tile * 16 + col, quad);
  const Share w = find_share(a, start, count, slot, spot.slot, h, tile, 1);
  if (w.count == 0) return;
  i32x4 kw[4][NS], vw[T];
  floatx4 kf[4], vf[4];
  auto load_k = [&](Pages p) {
    const int64_t bk = valid(p.k) ? p.k : 0, bv = valid(p.v) ? p.v : 0;
    const int8_t* kp = kh + bk * block_bytes;
    const int64_t at = (bv * a.Hkv + h) * PAGE;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int s = 0; s < NS; ++s) kw[n][s] = *(const i32x4*)(kp + n * 4 * D + s * 256);
      kf[n] = *(const floatx4*)(a.cache.k_scale + at + 4 * n);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) vf[n] = *(const floatx4*)(a.cache.v_scale + at + 4 * n);
  };
  auto load_v = [&](Pages p) {
    const int8_t* vp = vh + (int64_t)(valid(p.v) ? p.v : 0) * block_bytes;
#pragma unroll
    for (int t = 0; t < T; ++t) vw[t] = *(const i32x4*)(vp + t * 256);
  };
  if (c < w.c1) {
    load_k(here);
    load_v(here);
  }
  const Row x = find_row(a, b, h, tile * 16 + col, w.start, w.count);
  // every row of the tile sees the positions below
  const int common = (int)min64(w.end, a.tree ? w.start : w.start + place(a, tile * 16).t + 1);
  RowState<D> st;
  clear(st);
  Query<D> q;
  const bool fine = quantise_query(q, a, raw, x.m >= 0);
  for (; c < w.c1; c += WAVES) {
    const bool there = valid(here.v), more = c + WAVES < w.c1;
    const bool all = __builtin_amdgcn_ballot_w64(!there) == 0 && c * 64 + 64 <= common;
    attend_keys<D, 1>(
        st, q, [&](int, int n, int s) { return kw[n][s]; }, [&](int, int t) { return vw[t]; },
        [&](int, int n) { return kf[n]; }, [&](int, int n) { return vf[n]; },
        [&] {
          if (more) load_k(next);
        },
        [](int) {}, all, there ? seen_from(x, c * 64 + quad * 16) : 0u);
    if (more) {
      load_v(next);
      here = next;
      next = look_up(c + 2 * WAVES);
    }
  }
  st.l = sum_of(st.l, fine);
  join_waves<D, WAVES>(a, w, st, os, ml, wave, tile);
}

// Up to eight tiles: eight waves share the chunks of a split, two a step, through a ring in LDS. All eight load
// (each one plane, K or V, of one of a chunk's four pages, and its scales) straight into LDS, ahead of
// the products. Of n tiles the first 2 n - 8 have a wave each, which takes both chunks of a step at once
// (one conversion of the sums for 128 keys); the others two, a chunk each, so that the four SIMDs have
// about the same to do: six tiles 1.5 tiles a chunk and SIMD instead of 2. Bound by the products and the
// softmax beside them (1024 rows of 16 heads of 256 behind 16001 tokens: 277 GFLOP, twice that in 8 bits, in
// 288 us with the join); with few rows about as long for the loads (11 rows behind 220K tokens: 229 MB in
// 65 us, either alone 53).
constexpr int RING_WAVES = 8;

template <int D>
struct ChunkImage {
  // a page of K, padded: a read of 16 bytes a lane goes in quarters of lanes 0 .. 3, 12 .. 15, 20 .. 23 and
  // 24 .. 27 and the like, whose four pages are on different banks then
  static constexpr int KS = 16 * D + 128;
  static constexpr int VS = 16 * D;
  static constexpr int V = 4 * KS, SCALES = V + 4 * VS, BYTES = SCALES + 512;
  static constexpr int SLOTS = D == 256 ? 4 : 8;
};
typedef __attribute__((address_space(3))) void lds_void;

// 1 KiB (16 bytes a lane) from src, this lane's place, straight into LDS at dst, both `offset` bytes on.
// Written out because the compiler would wait for every such load before any LDS read; the ring's own
// waits say which have to be done. To the compiler they are clobbers of memory: its own waits stay good,
// since loads that it does not know of only make them longer. (m0 is used by nothing else in the kernel.)
__device__ __forceinline__ void load_to_lds(const void* src, uint32_t dst, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2" ::"s"(dst), "v"(src), "i"(offset)
               : "memory");
}

template <int D>
__global__ void __launch_bounds__(64 * RING_WAVES) attend_ring_kernel(KV8_FRONT) {
  KV8_TAKE_FRONT;
  using G = ChunkImage<D>;
  constexpr int STEPS = G::SLOTS / 2, LOADS = 2 * (D / 64 + 1);
  static_assert(RING_WAVES / 2 * 16 * D * 4 <= G::SLOTS * G::BYTES, "states are joined in the ring");
  __shared__ __attribute__((aligned(16))) uint8_t ring[G::SLOTS * G::BYTES];
  __shared__ float ml[RING_WAVES / 2][16][2];
  const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15, quad = lane >> 4;
  const Spot spot = find_spot(a.Hkv, (a.tiles + RING_WAVES - 1) / RING_WAVES);
  const int h = spot.h, tile0 = spot.group * RING_WAVES;
  const Slot at_slot = find_slot<2>(a, spot.slot, 0);
  const int b = at_slot.b;
  if (b < 0) return;
  const int start = a.starts[b], count = a.counts[b];
  const int tiles = a.tiles - tile0 < RING_WAVES ? a.tiles - tile0 : RING_WAVES;
  const int whole = 2 * tiles > RING_WAVES ? 2 * tiles - RING_WAVES : 0;   // tiles of one wave
  const bool pair = wave >= whole;
  const int tile = tile0 + (pair ? whole + (wave - whole) / 2 : wave), part = (wave - whole) & 1;
  const int32_t* trow = a.table + (int64_t)b * a.table_stride;
  const int c0 = at_slot.c0;
  // blocks of this wave's page in 64 chunks, one a lane
  auto look_up = [&](int first) {   // (past the table: its last page)
    const int64_t p = 4ll * (c0 + first + lane) + (wave & 3);
    return a.table_stride > 0 ? trow[p < a.table_stride ? p : a.table_stride - 1] : 0;
  };
  auto valid = [&](int e) { return e >= 0 && e < a.blocks; };
  int ids = look_up(0), ids_from = 0;
  RawQuery<D> raw;
  fetch_query(raw, a, b, h, tile * 16 + col, quad);
  const Share w = find_share(a, start, count, at_slot, spot.slot, h, tile0, tiles);
  if (w.count == 0) return;
  const int n_chunks = w.c1 - w.c0;
  // pages without a block are rare: whether there is one is found once, and each looked up only then
  const int64_t pages = (w.end + PAGE - 1) / PAGE;
  auto hole_in = [&](int first, int e) {
    return first + lane < n_chunks && 4ll * (c0 + first + lane) + (wave & 3) < pages && !valid(e);
  };
  bool hole = hole_in(0, ids);
  for (int i = 64; i < n_chunks; i += 64) hole |= hole_in(i, look_up(i));
  const bool holes = __syncthreads_or(hole);
  ids = valid(ids) ? ids : 0;
  // the query is waited for here: later a wait for it would be one for the loads behind it too
#pragma unroll
  for (int s = 0; s < D / 64; ++s) asm volatile("" ::"v"(raw.w[s][0]), "v"(raw.w[s][1]));
  const int64_t page_bytes = PAGE * D;
  const int8_t* plane = wave < 4 ? a.cache.k : a.cache.v;
  const float* scales = wave < 4 ? a.cache.k_scale : a.cache.v_scale;
  const uint32_t ring_at = (uint32_t)(uintptr_t)(lds_void*)ring;
  // the loads of a step: load i of LOADS, of chunk i / (LOADS / 2)
  const int8_t* src[2];
  const float* src_scale[2];
  uint32_t dst[2];
  auto aim = [&](int step) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      int i = step * 2 + n;
      i = i < n_chunks ? i : n_chunks - 1;
      if (i - ids_from >= 64) {   // (uniform)
        ids_from = i;
        ids = look_up(i);
        ids = valid(ids) ? ids : 0;
      }
      const int64_t at = (int64_t)__builtin_amdgcn_readlane(ids, i - ids_from) * a.Hkv + h;
      src[n] = plane + at * page_bytes + lane * 16;
      src_scale[n] = scales + at * PAGE + lane * 4;
      dst[n] = ring_at + (step % STEPS * 2 + n) * G::BYTES;
    }
  };
  auto load = [&](int i) {
    const int n = i / (LOADS / 2), j = i % (LOADS / 2);
    if (j < D / 64)
      load_to_lds(src[n], dst[n] + (wave < 4 ? wave * G::KS : G::V + (wave - 4) * G::VS), j * 1024);
    else if (lane < 4)
      load_to_lds(src_scale[n], dst[n] + G::SCALES + wave * 64, 0);
  };
  auto load_step = [&](int step) {
    aim(step);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(i);
  };
  const int steps = (n_chunks + 1) / 2;
#pragma unroll
  for (int s = 0; s < STEPS - 1; ++s)
    if (s < steps) load_step(s);
  const bool idle = tile >= tile0 + tiles || (int64_t)tile * 16 >= (int64_t)w.count * a.G;
  const Row x = idle ? Row{-1, 0, 0, 0} : find_row(a, b, h, tile * 16 + col, w.start, w.count);
  // every row of the tile sees the positions below `common`, none those from `until` on
  const int common = (int)min64(w.end, a.tree ? w.start : w.start + place(a, tile * 16).t + 1);
  int t_last = place(a, tile * 16 + 15).t;
  t_last = t_last < w.count ? t_last : w.count - 1;
  const int until = idle ? 0 : (int)min64(w.end, a.tree ? w.start + w.count : w.start + t_last + 1);
  RowState<D> st;
  clear(st);
  Query<D> q;
  const bool fine = quantise_query(q, a, raw, x.m >= 0);
  // a wave's steps: N = 2, both chunks of each, or 1, the part-th
  auto walk = [&](auto chunks) {
    constexpr int N = decltype(chunks)::value;
    for (int s = 0; s < steps; ++s) {
      // this wave's loads of the step have landed ..
      if (s + STEPS - 2 < steps) wait_vmcnt<(STEPS - 2) * LOADS>();
      else wait_vmcnt<0>();
      wait_lgkmcnt0();
      block_barrier();   // .. and every wave's; the step before is done with its slots
      const bool more = s + STEPS - 1 < steps;   // a step to load, between the products where there are any
      if (more) aim(s + STEPS - 1);
      const int o = N == 2 ? 0 : part, c = w.c0 + s * 2 + o;
      if (c >= w.c1 || c * 64 >= until) {   // (uniform over the wave)
        if (more)
#pragma unroll
          for (int i = 0; i < LOADS; ++i) load(i);
        continue;
      }
      uint32_t seen = 0, there = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        bool page = c + i < w.c1;
        if (holes && page) {
          const int64_t p = 4ll * (c + i) + quad;
          const int e = p < a.table_stride ? trow[p] : -1;
          page = e >= 0 && e < a.blocks;
        }
        there |= (uint32_t)page << i;
        if (page) seen |= seen_from(x, (c + i) * 64 + quad * 16) << (16 * i);
      }
      const bool all =
          c + N <= w.c1 && c * 64 + 64 * N <= common && (!holes || __builtin_amdgcn_ballot_w64(there != (1u << N) - 1) == 0);
      const uint8_t* slot = ring + (s % STEPS * 2 + o) * G::BYTES;
      const uint8_t* kp = slot + (col >> 2) * G::KS + quad * 64 + (col & 3) * 16;
      const uint8_t* vp = slot + G::V + quad * G::VS + col * 16;
      const uint8_t* sp = slot + G::SCALES + quad * 64;
      attend_keys<D, N>(
          st, q, [&](int i, int n, int t) { return *(const i32x4*)(kp + i * G::BYTES + n * 4 * D + t * 256); },
          [&](int i, int t) { return *(const i32x4*)(vp + i * G::BYTES + t * 256); },
          [&](int i, int n) { return *(const floatx4*)(sp + i * G::BYTES + 16 * n); },
          [&](int i, int n) { return *(const floatx4*)(sp + i * G::BYTES + 256 + 16 * n); }, [] {},
          [&](int i) {
            if (i < LOADS && more) load(i);
          },
          all, seen);
    }
  };
  if (pair) walk(std::integral_constant<int, 1>());
  else walk(std::integral_constant<int, 2>());
  wait_vmcnt<0>();   // no load may still go to LDS
  float l = column_sum(st.l);
  if (whole < tiles) {   // the second waves of the pairs pass their states on, in lanes' places
    floatx4(*os)[D / 16][64] = (floatx4(*)[D / 16][64])ring;
    const int i = (wave - whole) / 2;
    __syncthreads();   // the ring is free
    if (pair && part == 1) {
#pragma unroll
      for (int t = 0; t < D / 16; ++t) os[i][t][lane] = elements(st, t);
      if (quad == 0) {
        ml[i][col][0] = st.m;
        ml[i][col][1] = l;
      }
    }
    __syncthreads();
    if (pair && part == 1) return;
    if (pair) {
      const float m1 = ml[i][col][0], m = fmaxf(st.m, m1);
      const float f0 = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(st.m - m);
      const float f1 = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(m1 - m);
      st.m = m;
      l = f0 * l + f1 * ml[i][col][1];
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const floatx4 o = os[i][t][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[4 * t + e] = f0 * st.o[4 * t + e] + f1 * o[e];
      }
    }
  }
  if (x.m < 0) return;
  l = sum_of(l, fine);
  if (w.single) {
    const float f = inverse_sum(l);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) write_out<D>(a, x.m, x.head, t * 16 + 4 * quad, elements(st, t), f);
  } else {
    const int64_t part_at = part_row(a, w, tile * 16 + col);
    float* po = a.part_o + part_at * D + 4 * quad;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) *(floatx4*)(po + t * 16) = elements(st, t);
    if (quad == 0) write_sums(a, part_at, st.m, l);
  }
}

// The splits of a row joined: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s. The threads of COLS
// elements come GROUPS times, each with its splits, eight loads in flight: once for a few splits, else as
// often as a workgroup holds.
constexpr int JOIN = 512, AHEAD = 8;

template <int D, int STEP, int COLS, int GROUPS>
__global__ void __launch_bounds__(JOIN) join_kernel(AttendArgs a) {
  constexpr int W = COLS / 4, ROWS = JOIN / W / GROUPS;
  __shared__ floatx4 red[GROUPS > 1 ? GROUPS : 1][ROWS][W];
  const int c = threadIdx.x % W + blockIdx.x % (D / COLS) * W, g = threadIdx.x / W % GROUPS;
  const int i = threadIdx.x / W / GROUPS, r = blockIdx.x / (D / COLS) * ROWS + i, h = blockIdx.y, b = blockIdx.z;
  const RowPlace at = place(a, r);
  const Slot slot = find_slot<STEP>(a, -1, b);
  if (slot.splits <= 1) return;   // (uniform: written already)
  const int most = a.tiles * 16 - 1, rc = r < most ? r : most;
  const int64_t part = (((int64_t)h * a.slots + slot.first) * a.tiles + rc / 16) * 16 + rc % 16;
  const int64_t next = (int64_t)a.tiles * 16;   // the next split's
  const float2* ml = (const float2*)a.part_ml + part;
  const float* po = a.part_o + part * D + 4 * c;
  floatx4 x[AHEAD];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = s0 + k * GROUPS;
      if (s < slot.splits) x[k] = *(const floatx4*)(po + s * next * D);
    }
  };
  fetch(g);   // with the maxima, the sums and the request's lengths: one round trip
  int count = a.counts[b];
  count = count < a.T ? count : a.T;
  const bool live = a.starts[b] >= 0 && at.t < count;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.f;
  // a row's maximum and sum, by W threads or more
  constexpr int L = W < 64 ? W : 64;
  const int lane = threadIdx.x % L;
  for (int s = lane; s < slot.splits; s += L) m = fmaxf(m, ml[s * next].x);
  m = __uint_as_float(over_lanes<L>(__float_as_uint(m), [](uint32_t x, uint32_t y) {
    return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
  }));
  const float base = m == NEG_INF ? 0.f : m;
  for (int s = lane; s < slot.splits; s += L) {
    const float2 e = ml[s * next];
    l += __builtin_amdgcn_exp2f(e.x - base) * e.y;
  }
  l = sum_over_lanes<L>(l);
  for (int s0 = g; s0 < slot.splits; s0 += AHEAD * GROUPS) {
    if (s0 != g) fetch(s0);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = s0 + k * GROUPS;
      if (s < slot.splits) o += __builtin_amdgcn_exp2f(ml[s * next].x - base) * x[k];
    }
  }
  if constexpr (GROUPS > 1) {
    red[g][i][c % W] = o;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) o += red[k][i][c % W];
  }
  if (!live) return;
  write_out<D>(a, (int64_t)b * a.T + at.t, h * a.G + at.g, 4 * c, o, inverse_sum(l));
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
constexpr int64_t MAX_PAGES = 1 << 26;   // of a request: positions stay below 2^30

struct Plan {
  int64_t tiles, groups, slots, splits, units;
  bool ring;
};

// The form, and the split of the keys.
Plan attend_plan(int64_t batch, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D, int64_t width) {
  Plan p;
  p.tiles = (tokens * (Hq / Hkv) + 15) / 16;
  const int64_t chunks = (width + 3) / 4, heads = batch * Hkv;
  // In the ring's form a head's tiles share what is loaded, but a workgroup takes longer to start and its
  // 128 rows make more to join. It is taken from a megabyte of keys a CU on that the tiles would each load
  // (9 rows of 16 heads of 256 behind 220K tokens 78 us instead of 109; behind 24000 tokens 29 instead of
  // 20; of 32 heads of 128 behind 64000 tokens 44 instead of 48, behind 8192 17 instead of 14.4), and for
  // the tiles of many short prompts (8 of 128 rows, heads of 128: 11 us instead of 23).
  p.ring = p.tiles > 1 && (p.tiles * heads * chunks >= (1 << 21) / D ||
                           (p.tiles >= RING_WAVES && p.tiles * heads >= (1 << 18) / D));
  p.groups = p.ring ? (p.tiles + RING_WAVES - 1) / RING_WAVES : p.tiles;
  const int64_t step = p.ring ? 2 : WAVES;
  p.units = (chunks + step - 1) / step;
  // A workgroup for every CU, in the ring and with heads of 256, of which one has 128 KiB in flight (two
  // for every CU: 100K tokens 37 us instead of 29); two with the others (16 requests of 4K to 8K tokens,
  // heads of 128: 50 us instead of 55).
  const int64_t per_head = (p.ring || D == 256 ? 256 : 512) / (Hkv * p.groups);
  if (batch > 1 && batch <= 64 && batch < per_head && p.units > 2) {
    // several requests share them by their lengths (16 blocks of 9 rows behind 4K to 8K tokens: 44 us
    // instead of 47)
    p.splits = 0;
    p.slots = per_head < batch * p.units ? per_head : batch * p.units;
    return p;
  }
  // two steps stay together: joining them takes longer (400 tokens 12.2 us instead of 7.9)
  p.splits = p.units > 2 ? per_head / batch : 1;
  if (p.splits > 128) p.splits = 256 / (Hkv * p.groups * batch);   // (100K tokens, heads of 64: 17 us instead of 21)
  if (p.splits > p.units) p.splits = p.units;
  if (p.splits < 1) p.splits = 1;
  p.slots = batch * p.splits;
  return p;
}

int64_t attend_bytes(const Plan& p, int64_t Hkv, int64_t D) {
  return p.splits == 1 ? 0 : Hkv * p.slots * p.tiles * 16 * (D + 2) * 4;
}

template <int D, int STEP>
void launch_join(const AttendArgs& a, hipStream_t s) {
  constexpr int COLS = D < 128 ? D : 128, MOST = JOIN / (COLS / 4);
  const int splits = a.splits ? a.splits : a.slots / a.batch;   // (about: any count is right in any form)
  const int rows = a.T * a.G, groups = splits <= AHEAD ? 1 : splits <= 8 * AHEAD ? 8 : MOST;
  const int per = groups == MOST ? 1 : JOIN / (D / 4) / groups;
  const dim3 grid((unsigned)((rows + per - 1) / per * (groups == MOST ? D / COLS : 1)), (unsigned)a.Hkv,
                  (unsigned)a.batch);
  if (groups == 1) hipLaunchKernelGGL((join_kernel<D, STEP, D, 1>), grid, dim3(JOIN), 0, s, a);
  else if (groups == 8) hipLaunchKernelGGL((join_kernel<D, STEP, D, 8>), grid, dim3(JOIN), 0, s, a);
  else hipLaunchKernelGGL((join_kernel<D, STEP, COLS, MOST>), grid, dim3(JOIN), 0, s, a);
}

template <int D>
void launch_attend(const AttendArgs& a, const Plan& p, hipStream_t s) {
  // the heads of a page side by side: they lie behind one another in memory
  const dim3 grid((unsigned)(p.groups * a.Hkv), (unsigned)p.slots);
  hipLaunchKernelGGL(p.ring ? attend_ring_kernel<D> : attend_kernel<D>, grid, dim3(64 * (p.ring ? RING_WAVES : WAVES)),
                     0, s, a.table, a.starts, a.counts, a.q, a.table_stride, a.splits, a.unit, a.longer, a.tiles, a.Hkv,
                     a.g_inv, a);
  if (p.splits == 1 || hipPeekAtLastError() != hipSuccess) return;
  if (p.ring) launch_join<D, 2>(a, s);
  else launch_join<D, WAVES>(a, s);
}

}  // namespace

SV_API int snowverify_rope_axes(const int64_t* pos, const float* inv_freq, float* cosv, float* sinv,
                                int64_t rows, int64_t half, int64_t axes, const int64_t* sections,
                                int interleaved, void* stream) {
  if (rows < 0 || half <= 0 || half > 4096 || axes <= 0 || axes > MAX_AXES || !sections) return SV_EINVAL;
  AxesArgs a{pos, inv_freq, cosv, sinv, rows, (int)half, (int)axes, interleaved != 0, {}};
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > half) return SV_EINVAL;
    // the pairs in turn: an axis' last pair has to be there
    if (interleaved && i && sections[i] && i + axes * (sections[i] - 1) >= half) return SV_EINVAL;
    a.count[i] = (int)sections[i];
    sum += sections[i];
  }
  if (sum != half) return SV_EINVAL;
  if (rows == 0) return SV_OK;
  if (!pos || !inv_freq || !cosv || !sinv || rows > ((int64_t)1 << 33) / half) return SV_EINVAL;
  const bool four = half % 4 == 0 && (((uintptr_t)cosv | (uintptr_t)sinv) & 15) == 0;
  const int64_t threads = (rows + AXES_ROWS - 1) / AXES_ROWS * (four ? half / 4 : half);
  hipLaunchKernelGGL(four ? axes_kernel<4> : axes_kernel<1>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0,
                     S(stream), a);
  SV_CHECK_LAUNCH();
  return SV_OK;
}

SV_API int snowverify_kv8_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                 const void* q, int64_t q_stride, const float* cos_in,
                                 const float* sin_in, int64_t cs_stride, int64_t half,
                                 const void* q_gamma, const void* k_gamma, float eps, void* k_pool,
                                 void* v_pool, float* k_scale, float* v_scale, void* q_out,
                                 const int32_t* table, const int32_t* starts, const int32_t* counts,
                                 int64_t batch, int64_t tokens, int64_t num_heads,
                                 int64_t num_kv_heads, int64_t head_size, int64_t table_stride,
                                 int64_t blocks, void* stream) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || half < 0 || half % 8 ||
      2 * half > head_size || table_stride < 0 || blocks < 0 || k_stride % 8 || v_stride % 8 ||
      q_stride % 8 || (q && !q_out))
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  if (!k || !v || (blocks && (!k_pool || !v_pool || !k_scale || !v_scale)) ||
      (table_stride && !table) || !starts || !counts || (half && (!cos_in || !sin_in)))
    return SV_EINVAL;
  AppendArgs a{};
  a.rows = {(const uint16_t*)q, q_stride, (const uint16_t*)q_gamma, cos_in, sin_in, cs_stride, eps,
            (uint16_t*)q_out, starts, counts, (int)batch, (int)tokens, (int)num_heads, (int)half};
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.k_gamma = (const uint16_t*)k_gamma;
  a.cache = {(int8_t*)k_pool, (int8_t*)v_pool, k_scale, v_scale};
  a.table = table;
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.Hkv = (int)num_kv_heads;
  a.pages = (int)((tokens + PAGE - 2) / PAGE + 1);
  a.page_wgs = batch * a.pages * num_kv_heads;
  const int64_t groups = (num_heads + Q_HEADS - 1) / Q_HEADS;
  const int64_t grid = a.page_wgs + (q ? (batch * tokens * groups + 15) / 16 : 0);
  if (!grid_ok(grid, 2 * head_size)) return SV_EINVAL;
  const bool by = q && queries_pass_by(batch * tokens, num_heads, head_size);
  auto kern = head_size == 64    ? by ? append_kernel<64, true> : append_kernel<64, false>
              : head_size == 128 ? by ? append_kernel<128, true> : append_kernel<128, false>
              : by               ? append_kernel<256, true> : append_kernel<256, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3((unsigned)(2 * head_size)), 0, S(stream), a);
  SV_CHECK_LAUNCH();
  return SV_OK;
}

SV_API int snowverify_kv8_read(const void* k_pool, const void* v_pool, const float* k_scale,
                               const float* v_scale, const int32_t* table, const int32_t* starts,
                               const int32_t* counts, void* k, void* v, int64_t batch, int64_t tokens,
                               int64_t num_kv_heads, int64_t head_size, int64_t table_stride,
                               int64_t blocks, void* stream) {
  if (!head_shape_ok(batch, tokens, num_kv_heads, num_kv_heads, head_size) || table_stride < 0 || blocks < 0)
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  if ((blocks && (!k_pool || !v_pool || !k_scale || !v_scale)) || (table_stride && !table) || !starts ||
      !counts || !k || !v)
    return SV_EINVAL;
  ReadArgs a{{(int8_t*)k_pool, (int8_t*)v_pool, (float*)k_scale, (float*)v_scale}, table, starts, counts,
             (uint16_t*)k, (uint16_t*)v, table_stride, blocks, (int)tokens, (int)num_kv_heads,
             (int)((tokens + PAGE - 2) / PAGE + 1)};
  const int64_t grid = batch * a.pages * num_kv_heads;
  if (!grid_ok(grid, 2 * head_size)) return SV_EINVAL;
  auto kern = head_size == 64 ? read_kernel<64> : head_size == 128 ? read_kernel<128> : read_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3((unsigned)(2 * head_size)), 0, S(stream), a);
  SV_CHECK_LAUNCH();
  return SV_OK;
}

SV_API int64_t snowverify_kv8_attention_scratch_bytes(int64_t batch, int64_t tokens, int64_t num_heads,
                                                      int64_t num_kv_heads, int64_t head_size,
                                                      int64_t table_stride) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      table_stride > MAX_PAGES || batch * tokens == 0)
    return 0;
  const Plan p = attend_plan(batch, tokens, num_heads, num_kv_heads, head_size, table_stride);
  return attend_bytes(p, num_kv_heads, head_size);
}

SV_API int snowverify_kv8_attention_form(int64_t batch, int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                                         int64_t head_size, int64_t table_stride) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      table_stride > MAX_PAGES || batch * tokens == 0)
    return -1;
  return attend_plan(batch, tokens, num_heads, num_kv_heads, head_size, table_stride).ring;
}

SV_API int snowverify_kv8_attention(const void* q, int64_t q_stride, const void* k_pool,
                                    const void* v_pool, const float* k_scale, const float* v_scale,
                                    void* out, const int32_t* table, const int32_t* starts,
                                    const int32_t* counts, const uint64_t* tree, int64_t batch,
                                    int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                                    int64_t head_size, int64_t table_stride, int64_t blocks, float scale,
                                    void* scratch, int64_t scratch_bytes, void* stream) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      table_stride > MAX_PAGES || blocks < 0 || q_stride % 8 || !(scale - scale == 0.f) ||
      (tree && tokens > 64))
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  const int64_t need = snowverify_kv8_attention_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                              head_size, table_stride);
  if (!q || !out || out == q || (blocks && (!k_pool || !v_pool || !k_scale || !v_scale)) ||
      (table_stride && !table) || !starts || !counts || scratch_bytes < need || (need && !scratch))
    return SV_EINVAL;
  const Plan p = attend_plan(batch, tokens, num_heads, num_kv_heads, head_size, table_stride);
  if (batch > 65535 || !grid_ok(p.groups * num_kv_heads, 64 * RING_WAVES)) return SV_ENOTSUP;
  AttendArgs a{};
  a.q = (const uint16_t*)q;
  a.q_stride = q_stride;
  a.cache = {(int8_t*)k_pool, (int8_t*)v_pool, (float*)k_scale, (float*)v_scale};
  a.out = (uint16_t*)out;
  a.table = table;
  a.starts = starts;
  a.counts = counts;
  a.tree = tree;
  a.table_stride = blocks ? table_stride : 0;   // no block, no key
  a.blocks = blocks;
  a.T = (int)tokens;
  a.Hq = (int)num_heads;
  a.Hkv = (int)num_kv_heads;
  a.G = (int)(num_heads / num_kv_heads);
  a.tiles = (int)p.tiles;
  a.slots = (int)p.slots;
  a.splits = (int)p.splits;
  a.batch = (int)batch;
  a.unit = p.splits ? (int)(p.units / p.splits) : 0;
  a.longer = p.splits ? (int)(p.units % p.splits) : 0;
  a.g_inv = (uint32_t)std::min<uint64_t>((1ull << 32) / (uint64_t)a.G, 0xffffffffull);
  a.scale = scale;
  a.part_o = (float*)scratch;
  a.part_ml = (float*)scratch + num_kv_heads * p.slots * p.tiles * 16 * head_size;
  if (head_size == 64) launch_attend<64>(a, p, S(stream));
  else if (head_size == 128) launch_attend<128>(a, p, S(stream));
  else launch_attend<256>(a, p, S(stream));
  SV_CHECK_LAUNCH();
  return SV_OK;
}
