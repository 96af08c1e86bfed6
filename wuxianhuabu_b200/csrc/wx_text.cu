// wx_text.cu — the text side of the pipeline between its linears: rotary positions of a
// token stream, and the paged K/V cache that is quantised as it is written.
//
// Cache layout: k and v are [pages][kv_heads][page_size][head_dim] (bf16, int8 or e4m3),
// k_scale and v_scale [pages][kv_heads][page_size] fp32 (8-bit formats). A slot is
// page * page_size + offset; one (token, head) row of head_dim values has one scale.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "wx_internal.h"
#include "wx_text_dev.cuh"

namespace wx {

// ------------------------------------------------------------------ rope tables
struct RopeFreqs {
  double inv[kRopeMaxPairs];
};

// cos / sin of position * inv_freq: the product and the functions in 64 bits (at position
// 100,000 a 32-bit product would already be 0.004 rad off), one rounding to fp32
__global__ void rope_table_kernel(RopeFreqs f, int nf, int64_t positions, double magnitude, float* __restrict__ cos_t,
                                  float* __restrict__ sin_t) {
  const int64_t total = positions * nf;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    double sn, cs;
    sincos((double)(i / nf) * f.inv[i % nf], &sn, &cs);
    cos_t[i] = (float)(cs * magnitude);
    sin_t[i] = (float)(sn * magnitude);
  }
}

// --------------------------------------------------------------- rows of a token
// One launch serves rope alone, the cache write alone and both fused. A token's rows are its q
// heads, then k heads, then v heads. HD / (2 W) neighbouring lanes own a row; a lane holds two
// groups of W columns, placed so that both halves of each pair it turns are its own (W = 8: 16-byte
// accesses; W = 4 where rot is no multiple of 16).
//
// Bound by HBM: each value is read once and written once, the table row of a token (rot * 4 bytes)
// is shared by its heads. A warp issues the loads of all its rows (up to kRowGroups groups) before
// the first store: the outputs may alias the inputs, so the compiler could not.
// Measured: rope of 8,192 tokens, 32 + 8 heads of 128, 36 us after a flush that leaves L2 dirty, 31.7 us
// = 5.45 TB/s with clean lines (three or two groups in flight 43 and 67, five 38); 4,096 tokens
// with rope into an int8 cache and read back, 40 us for both (35.6). 300 tokens take 3 us on the
// device, a third of the call.
constexpr int kRowGroups = 4;

struct RowsParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int nq, nkv;                           // q rows, and k (= v) rows of a token (0 without a cache)
  int nv;                                // head_rows_kernel: v rows
  int64_t tokens;
  int rows_per_warp, chunks;             // a token's rows are dealt to `chunks` warps
  // rotation (rot = 0: none)
  const float *cos_t, *sin_t;
  const int32_t* pos;
  int64_t positions;
  int rot, interleaved;
  __nv_bfloat16* q_out;
  int64_t q_out_stride;
  // cache
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int64_t* slots;
  int64_t n_slots;
  int page_shift;
  int* err;
};

template <int W>
struct Cols {  // W bf16 columns in memory
  uint32_t w[W / 2];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    if constexpr (W == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x, w[1] = x.y;
    }
  }
  __device__ __forceinline__ void lds(uint32_t at) {
    if constexpr (W == 8) {
      const uint4 x = lds128(at);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = lds64(at);
      w[0] = x.x, w[1] = x.y;
    }
  }
  __device__ __forceinline__ void sts(uint32_t at) const {
    if constexpr (W == 8)
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    else asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(at), "r"(w[0]), "r"(w[1]) : "memory");
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const {
    if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
};

// N values of a row (its other values in the neighbouring kLanes lanes) -> the stored format,
// packed in words. The scale is amax / 127 or amax / 448 of the fp32 values; the value stored is
// value * (127 | 448) / amax rounded to nearest even. A row with infinity or NaN stores scale NaN
// and zeros, so that it reads back as NaN; a row below 2^-100 everywhere (127 / amax could
// overflow) stores zeros.
//
// This kernel is issue-bound before it is HBM-bound, hence: the magnitudes are compared as bits
// (NaN and infinity come out on top), int8 values are rounded by adding 1.5 * 2^23 (the low byte of
// the sum is the integer), products are packed in pairs.
template <int FMT, int N, int kLanes>
__device__ __forceinline__ float quantise(const float (&x)[N], uint32_t (&w)[N / 4]) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) bits = max(bits, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  constexpr float kMax = FMT == kKvInt8 ? 127.f : 448.f;
  const float amax = __uint_as_float(bits);
  const bool finite = bits < 0x7f800000u;
  const bool live = finite && amax >= 0x1p-100f;
  const float inv = live ? __fdiv_rn(kMax, amax) : 0.f;
  const float2 inv2 = make_float2(inv, inv);
#pragma unroll
  for (int h = 0; h < N / 4; ++h) {
    float2 lo = __fmul2_rn(make_float2(x[4 * h], x[4 * h + 1]), inv2);
    float2 hi = __fmul2_rn(make_float2(x[4 * h + 2], x[4 * h + 3]), inv2);
    if constexpr (FMT == kKvInt8) {
      // (single sums: a packed one would be fused with the product before it, into one rounding)
      auto byte = [](float y) { return __float_as_uint(__fadd_rn(y, 12582912.f)); };
      const uint32_t a = __byte_perm(byte(lo.x), byte(lo.y), 0x0040);
      const uint32_t b = __byte_perm(byte(hi.x), byte(hi.y), 0x0040);
      w[h] = __byte_perm(a, b, 0x5410);
    } else {
      const uint32_t a = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3);
      const uint32_t b = __nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3);
      w[h] = a | b << 16;
    }
    if (!live) w[h] = 0;
  }
  return finite ? (live ? __fdiv_rn(amax, kMax) : 0.f) : __int_as_float(0x7fc00000);
}

template <int FMT, int HD, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 3) text_rows_kernel(RowsParams p) {
  constexpr int kLanes = HD / (2 * W);  // lanes of a row
  constexpr int kRows = 32 / kLanes;    // rows of a warp at a time
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes;
  const int per_token = p.nq + 2 * p.nkv;
  // a block: eight tokens, the same chunk of each
  const unsigned blk = blockIdx.x / (unsigned)p.chunks;
  const int64_t t = (int64_t)blk * 8 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int r0 = (int)(blockIdx.x - blk * (unsigned)p.chunks) * p.rows_per_warp;
  const int r1 = min(per_token, r0 + p.rows_per_warp);

  const bool turn = j < p.rot / (2 * W);
  const bool apart = turn && !INTERLEAVED;  // pairs (i, i + rot / 2)
  const int c0 = apart ? W * j : 2 * W * j;
  const int c1 = apart ? p.rot / 2 + W * j : 2 * W * j + W;

  Cols<W> a[kRowGroups], b[kRowGroups];
#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    const int r = r0 + g * kRows + lane / kLanes;
    if (r >= r1) continue;
    const __nv_bfloat16* src = r < p.nq           ? p.q + t * p.q_stride + (int64_t)r * HD
                               : r < p.nq + p.nkv ? p.k + t * p.k_stride + (int64_t)(r - p.nq) * HD
                                                  : p.v + t * p.v_stride + (int64_t)(r - p.nq - p.nkv) * HD;
    a[g].load(src + c0);
    b[g].load(src + c1);
  }

  float cs[W], sn[W];
  if (p.rot) {
    const int64_t pos = p.pos[t];
    if (pos < 0 || pos >= p.positions) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
      return;
    }
    if (turn) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const float4 c = *reinterpret_cast<const float4*>(p.cos_t + pos * (p.rot / 2) + W * j + i);
        const float4 s = *reinterpret_cast<const float4*>(p.sin_t + pos * (p.rot / 2) + W * j + i);
        cs[i] = c.x, cs[i + 1] = c.y, cs[i + 2] = c.z, cs[i + 3] = c.w;
        sn[i] = s.x, sn[i + 1] = s.y, sn[i + 2] = s.z, sn[i + 3] = s.w;
      }
    }
  }
  int64_t slot = -1;
  if (p.nkv) {
    slot = p.slots[t];
    if (slot >= p.n_slots) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
      slot = -1;
    }
  }

#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    if (r0 + g * kRows >= r1) break;  // (the warp as a whole)
    const int r = r0 + g * kRows + lane / kLanes;
    const bool live = r < r1;
    const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv;
    const int h = is_q ? r : is_v ? r - p.nq - p.nkv : r - p.nq;
    float x[2 * W];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const uint32_t u = live ? a[g].w[i] : 0, v = live ? b[g].w[i] : 0;
      x[2 * i] = bf16_lo(u), x[2 * i + 1] = bf16_hi(u);
      x[W + 2 * i] = bf16_lo(v), x[W + 2 * i + 1] = bf16_hi(v);
    }
    if (turn && !is_v) {
      // (x1, x2) -> (x1 c - x2 s, x2 c + x1 s)
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        float &a0 = x[INTERLEAVED ? 2 * i : i], &a1 = x[INTERLEAVED ? 2 * i + 2 : i + 1];
        float &b0 = x[INTERLEAVED ? 2 * i + 1 : W + i], &b1 = x[INTERLEAVED ? 2 * i + 3 : W + i + 1];
        const float2 x1 = make_float2(a0, a1), x2 = make_float2(b0, b1);
        const float2 c = make_float2(cs[i], cs[i + 1]), s = make_float2(sn[i], sn[i + 1]);
        const float2 ns = make_float2(-sn[i], -sn[i + 1]);
        const float2 u = __ffma2_rn(x1, c, __fmul2_rn(x2, ns));
        const float2 v = __ffma2_rn(x2, c, __fmul2_rn(x1, s));
        a0 = u.x, a1 = u.y, b0 = v.x, b1 = v.y;
      }
    }
    uint32_t qv[W / 2] = {};
    float scale = 0.f;
    if constexpr (FMT != kKvBf16) scale = quantise<FMT, 2 * W, kLanes>(x, qv);  // (all lanes: it shuffles)
    if (!live) continue;
    const int64_t row = ((((slot >> p.page_shift) * p.nkv + h) << p.page_shift) | (slot & ((1 << p.page_shift) - 1)));
    if (!WX_IN_BOUNDS(p.err, is_q ? h >= 0 && h < p.nq : h >= 0 && h < p.nkv && (slot < 0 || row < p.n_slots * p.nkv)))
      continue;
    if (is_q || FMT == kKvBf16) {
      __nv_bfloat16* o = is_q ? p.q_out + t * p.q_out_stride + (int64_t)h * HD
                              : reinterpret_cast<__nv_bfloat16*>(is_v ? p.vc : p.kc) + row * HD;
      if (!is_q && slot < 0) continue;
      Cols<W> lo, hi;
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        lo.w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
        hi.w[i] = pack_bf16x2(x[W + 2 * i], x[W + 2 * i + 1]);
      }
      lo.store(o + c0);
      hi.store(o + c1);
    } else if (slot >= 0) {
      uint8_t* o = (is_v ? p.vc : p.kc) + row * HD;
      if constexpr (W == 8) {
        *reinterpret_cast<uint2*>(o + c0) = make_uint2(qv[0], qv[1]);
        *reinterpret_cast<uint2*>(o + c1) = make_uint2(qv[2], qv[3]);
      } else {
        *reinterpret_cast<uint32_t*>(o + c0) = qv[0];
        *reinterpret_cast<uint32_t*>(o + c1) = qv[1];
      }
      if (j == 0) (is_v ? p.vs : p.ks)[row] = scale;
    }
  }
}

// ---------------------------------------------------------------- head norms and position axes
// q and k rows normalised, y = x / sqrt(mean x^2 + eps) * w, and turned, each pair by the position of its own axis;
// k and v into a cache, or k beside q. All of it in fp32 until the one rounding (or quantisation) at the end.
//
// Lanes, columns and loads as above. There is more to do for the same bytes, and issue slots run out before HBM
// does (366 instructions for the four rows that a warp works on at a time: 43 us for a clip's 8,064 tokens, 32 + 8
// heads of 128; rope alone takes 162 and 28 us), hence:
// - a warp's rows are of one norm, q or k (and v), and the weight goes into the rotation's factors:
//   u = x1 (w1 c) - x2 (w2 s), v = x2 (w2 c) + x1 (w1 s). A warp makes them for its token, a lane a pair or two,
//   while its rows are on their way, and reads them from shared memory as it needs them (in registers
//   they would cost an SM a block of its three);
// - q rows lie side by side: one address and constant offsets. Squares, scaling, rotation in packed pairs.
// Measured with kernels as below, in us beside their rule (launch_heads).
struct HeadParams {
  RowsParams r;
  int nk;  // k rows (of a cache, or to k_out)
  const __nv_bfloat16 *q_norm, *k_norm;  // nullptr: not normalised
  float eps;
  uint64_t axis_of[2];  // two bits for each pair
  int64_t pos_stride;   // between the axes' positions
  __nv_bfloat16* k_out;
  int64_t k_out_stride;
  int q_chunks;  // of the `chunks` warps of a token
};

// W floats of shared memory as pairs
template <int W>
__device__ __forceinline__ void lds_pairs(uint32_t at, float2 (&f)[W / 2]) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const uint4 x = lds128(at + i * 4);
    f[i / 2] = make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
    f[i / 2 + 1] = make_float2(__uint_as_float(x.z), __uint_as_float(x.w));
  }
}

// a lane's first, second, third and fourth factors, and where it reads them
template <int W>
struct Factors {
  float2 a[W / 2], b[W / 2], c[W / 2], d[W / 2];
};
struct FactorsAt {
  uint32_t a, b, c, d;
  template <int W>
  __device__ __forceinline__ void load(Factors<W>& f) const {
    lds_pairs<W>(a, f.a);
    lds_pairs<W>(b, f.b);
    lds_pairs<W>(c, f.c);
    lds_pairs<W>(d, f.d);
  }
};
template <int HD, int W, bool INTERLEAVED>
__device__ __forceinline__ FactorsAt factors_at(const float* table, int j) {
  constexpr int kPairs = HD / 2;
  FactorsAt f;
  f.a = smem_u32(table) + (INTERLEAVED ? 2 : 1) * W * j * 4;
  f.b = f.a + (INTERLEAVED ? 2 : 1) * kPairs * 4;
  f.c = f.a + (INTERLEAVED ? W : 2 * kPairs) * 4;
  f.d = f.b + (INTERLEAVED ? W : 2 * kPairs) * 4;
  return f;
}
// one pair's factors, of columns cA and cB: w_A c, -w_B s, w_B c, w_A s (columns that do not turn: c 1, s 0). Half
// layout: an array of each; interleaved: the first and third side by side, then the others
template <int HD, int W, bool INTERLEAVED>
__device__ __forceinline__ void put_factors(float* f, int pair, float c, float s, float wa, float wb) {
  constexpr int kPairs = HD / 2;
  if constexpr (INTERLEAVED) {
    *reinterpret_cast<float2*>(f + 2 * pair) = make_float2(wa * c, wb * c);
    *reinterpret_cast<float2*>(f + 2 * kPairs + 2 * pair) = make_float2(-wb * s, wa * s);
  } else {
    f[pair] = wa * c;
    f[kPairs + pair] = -wb * s;
    f[2 * kPairs + pair] = wb * c;
    f[3 * kPairs + pair] = wa * s;
  }
}
template <int W, bool INTERLEAVED>
__device__ __forceinline__ int2 columns_of(int pair, int rot) {
  if (INTERLEAVED) return make_int2(2 * pair, 2 * pair + 1);
  if (pair < rot / 2) return make_int2(pair, rot / 2 + pair);
  return make_int2(2 * pair - pair % W, 2 * pair - pair % W + W);
}

// A lane's columns c0.. (x1) and c1.. (x2) of a row
template <int W>
__device__ __forceinline__ void unpack(const Cols<W>& lo, const Cols<W>& hi, float2 (&x1)[W / 2], float2 (&x2)[W / 2]) {
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    x1[i] = make_float2(bf16_lo(lo.w[i]), bf16_hi(lo.w[i]));
    x2[i] = make_float2(bf16_lo(hi.w[i]), bf16_hi(hi.w[i]));
  }
}
template <int W>
__device__ __forceinline__ float square_sum(const float2 (&x1)[W / 2], const float2 (&x2)[W / 2]) {
  float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    s1 = __ffma2_rn(x1[i], x1[i], s1);
    s2 = __ffma2_rn(x2[i], x2[i], s2);
  }
  return (s1.x + s1.y) + (s2.x + s2.y);
}
// scaled, weighted and turned
template <int W, bool INTERLEAVED>
__device__ __forceinline__ void turn_row(float2 (&x1)[W / 2], float2 (&x2)[W / 2], float rstd, bool turn, const Factors<W>& f) {
  const float2 rr = make_float2(rstd, rstd);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    x1[i] = __fmul2_rn(x1[i], rr);
    x2[i] = __fmul2_rn(x2[i], rr);
  }
  if (turn) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      if (INTERLEAVED) {  // a pair's columns times (w_A c, w_B c), their swap times (-w_B s, w_A s)
        x1[i] = __ffma2_rn(x1[i], f.a[i], __fmul2_rn(make_float2(x1[i].y, x1[i].x), f.b[i]));
        x2[i] = __ffma2_rn(x2[i], f.c[i], __fmul2_rn(make_float2(x2[i].y, x2[i].x), f.d[i]));
      } else {
        const float2 u = __ffma2_rn(x1[i], f.a[i], __fmul2_rn(x2[i], f.b[i]));
        x2[i] = __ffma2_rn(x2[i], f.c[i], __fmul2_rn(x1[i], f.d[i]));
        x1[i] = u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      x1[i] = __fmul2_rn(x1[i], f.a[i]);
      x2[i] = __fmul2_rn(x2[i], f.c[i]);
    }
  }
}
template <int W>
__device__ __forceinline__ void pack(const float2 (&x1)[W / 2], const float2 (&x2)[W / 2], Cols<W>& lo, Cols<W>& hi) {
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    lo.w[i] = pack_bf16x2(x1[i].x, x1[i].y);
    hi.w[i] = pack_bf16x2(x2[i].x, x2[i].y);
  }
}
// quantised to row `row` of the cache, head column c0.. and to_c1 behind it. All lanes of the warp call
template <int FMT, int HD, int W>
__device__ __forceinline__ void store_quantised(const RowsParams& p, const float2 (&x1)[W / 2], const float2 (&x2)[W / 2],
                                                bool write, bool is_v, int64_t row, int c0, int to_c1, bool first_lane) {
  float x[2 * W];
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    x[2 * i] = x1[i].x, x[2 * i + 1] = x1[i].y;
    x[W + 2 * i] = x2[i].x, x[W + 2 * i + 1] = x2[i].y;
  }
  uint32_t q[W / 2];
  const float scale = quantise<FMT, 2 * W, HD / (2 * W)>(x, q);
  if (!write) return;
  uint8_t* o = (is_v ? p.vc : p.kc) + row * HD + c0;
  if constexpr (W == 8) {
    *reinterpret_cast<uint2*>(o) = make_uint2(q[0], q[1]);
    *reinterpret_cast<uint2*>(o + to_c1) = make_uint2(q[2], q[3]);
  } else {
    *reinterpret_cast<uint32_t*>(o) = q[0];
    *reinterpret_cast<uint32_t*>(o + to_c1) = q[1];
  }
  if (first_lane) (is_v ? p.vs : p.ks)[row] = scale;
}

template <int FMT, int HD, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 3) head_rows_kernel(HeadParams hp) {
  const RowsParams& p = hp.r;
  constexpr int kLanes = HD / (2 * W);  // lanes of a row
  constexpr int kRows = 32 / kLanes;    // rows of a warp at a time
  constexpr int kPairs = HD / 2;
  // of the warp's token
  __shared__ __align__(16) float factors[8][4 * kPairs];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane % kLanes, sub = lane / kLanes;
  const unsigned blk = blockIdx.x / (unsigned)p.chunks;
  const int64_t t = (int64_t)blk * 8 + warp;
  if (t >= p.tokens) return;
  const int chunk = (int)(blockIdx.x - blk * (unsigned)p.chunks);
  const bool is_q = chunk < hp.q_chunks;
  // rows of this warp: r0.. of q, or of k and then v (from n0 on)
  const int r0 = (is_q ? chunk : chunk - hp.q_chunks) * p.rows_per_warp;
  const int n0 = is_q ? p.nq : hp.nk;
  const int r1 = min(is_q ? p.nq : hp.nk + p.nv, r0 + p.rows_per_warp);

  const bool turn = j < p.rot / (2 * W);
  const bool apart = turn && !INTERLEAVED;  // pairs (i, i + rot / 2)
  const int c0 = apart ? W * j : 2 * W * j;
  const int c1 = apart ? p.rot / 2 + W * j : 2 * W * j + W;

  // row 0's columns c0.. of q or k, and of v nk rows before its first
  const __nv_bfloat16* src0 = (is_q ? p.q + t * p.q_stride : p.k + t * p.k_stride) + c0;
  const __nv_bfloat16* src1 = is_q ? src0 : p.v + t * p.v_stride - (int64_t)hp.nk * HD + c0;
  const int to_c1 = c1 - c0;
  Cols<W> a[kRowGroups], b[kRowGroups];
  const __nv_bfloat16* q_from = src0 + (r0 + sub) * HD;
#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    const int r = r0 + g * kRows + sub;
    if (r < r1) {
      const __nv_bfloat16* src = is_q ? q_from + g * (kRows * HD) : (r < n0 ? src0 : src1) + r * HD;
      a[g].load(src);
      b[g].load(src + to_c1);
    } else {  // (its lanes are a row of their own)
      a[g].clear();
      b[g].clear();
    }
  }

  // ---- the factors, with the rows on their way
  const __nv_bfloat16* weight = is_q ? hp.q_norm : hp.k_norm;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPairs / 32; ++i) {
    const int pair = i * 32 + lane;
    const int2 cols = columns_of<W, INTERLEAVED>(pair, p.rot);
    float c = 1.f, s = 0.f;
    if (pair < p.rot / 2) {
      const int axis = (int)(hp.axis_of[i] >> (2 * lane)) & 3;
      const int64_t pos = p.pos[axis * hp.pos_stride + t];
      if (pos < 0 || pos >= p.positions) {
        bad = true;
      } else {
        const int64_t at = pos * (p.rot / 2) + pair;
        c = __ldg(p.cos_t + at);
        s = __ldg(p.sin_t + at);
      }
    }
    float wa = 1.f, wb = 1.f;
    if (weight) wa = __bfloat162float(weight[cols.x]), wb = __bfloat162float(weight[cols.y]);
    put_factors<HD, W, INTERLEAVED>(factors[warp], pair, c, s, wa, wb);
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0) set_dev_error(p.err, kDevBadArgs);
    return;
  }
  __syncwarp();
  const FactorsAt factor = factors_at<HD, W, INTERLEAVED>(factors[warp], j);

  // ---- where the rows go
  const bool cached = !is_q && !hp.k_out;
  // (rows of a bf16 cache and plain ones by address, those of an 8-bit cache by their number)
  __nv_bfloat16 *dst0 = is_q ? p.q_out + t * p.q_out_stride : hp.k_out + t * hp.k_out_stride, *dst1 = dst0;
  int64_t row0 = 0;  // cache row of head 0
  if (cached) {
    const int64_t slot = p.slots[t];
    if (slot >= p.n_slots && lane == 0) set_dev_error(p.err, kDevBadArgs);
    if (slot < 0 || slot >= p.n_slots) return;
    row0 = ((slot >> p.page_shift) * hp.nk << p.page_shift) | (slot & ((1 << p.page_shift) - 1));
    if (FMT == kKvBf16) {
      dst0 = reinterpret_cast<__nv_bfloat16*>(p.kc) + row0 * HD;
      dst1 = reinterpret_cast<__nv_bfloat16*>(p.vc) + row0 * HD - ((int64_t)hp.nk * HD << p.page_shift);
    }
  }
  dst0 += c0;
  dst1 += c0;
  const int64_t stride = cached ? (int64_t)HD << p.page_shift : HD;

  __nv_bfloat16* q_to = dst0 + (r0 + sub) * HD;
#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    if (r0 + g * kRows >= r1) break;  // (the warp as a whole)
    const int r = r0 + g * kRows + sub;
    const bool live = r < r1, is_v = r >= n0;
    float2 x1[W / 2], x2[W / 2];
    unpack<W>(a[g], b[g], x1, x2);
    float rstd = 1.f;
    if (weight) {  // (all lanes: it shuffles)
      float ss = square_sum<W>(x1, x2);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rstd = rsqrtf(ss * (1.f / HD) + hp.eps);
    }
    if (!is_v) {
      Factors<W> f;
      factor.load(f);
      turn_row<W, INTERLEAVED>(x1, x2, rstd, turn, f);
    }
    if (FMT == kKvBf16 || !cached) {
      if (!live) continue;
      if (!WX_IN_BOUNDS(p.err, r >= 0 && r < (is_q ? p.nq : hp.nk + p.nv) && (is_q || !is_v || cached))) continue;
      __nv_bfloat16* o = is_q ? q_to + g * (kRows * HD) : (is_v ? dst1 : dst0) + r * stride;
      Cols<W> lo, hi;
      pack<W>(x1, x2, lo, hi);
      lo.store(o);
      hi.store(o + to_c1);
    } else {
      const int64_t row = row0 + ((int64_t)(is_v ? r - hp.nk : r) << p.page_shift);
      const bool write = live && WX_IN_BOUNDS(p.err, row >= 0 && row < p.n_slots * hp.nk);
      store_quantised<FMT, HD, W>(p, x1, x2, write, is_v, row, c0, to_c1, j == 0);
    }
  }
}

// The same for many tokens: persistent warps, each with a ring of its own in shared memory, through which the
// rows of its tokens pass in chunks of 4 KB. Bulk copies bring them (a token's heads lie side by side) and
// take them away, so that loads stay in flight while the warp computes; in the kernel above a warp's life is a load,
// then its arithmetic, and neither keeps HBM busy. Positions run two tokens ahead, table rows one. A chunk's row
// groups are worked on side by side: one after the other (12 warps, 4 stages) their latency made it 42 us.
// Measured: q and k of 8,064 tokens, 32 + 8 heads of 128, three axes, 31.9 us = 5.3 TB/s (rows kernel 41); 4,277 tokens
// into an int8 cache 21 us (30). Issue slots 53 % busy, four warps to a scheduler.
constexpr int kStreamWarps = 16, kStreamStages = 3, kStreamChunk = 4096;
template <int HD>
struct StreamGeom {
  static constexpr int kRing = kStreamWarps * kStreamStages * kStreamChunk;
  static constexpr int kFactors = kStreamWarps * 2 * 2 * HD * 4;  // of q's and of k's norm
  static constexpr int kSmem = kRing + kFactors + kStreamWarps * kStreamStages * 8 + 16;
};

__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// waits until at most N of the thread's groups still read shared memory
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int FMT, int HD, int W, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kStreamWarps, 1) head_stream_kernel(HeadParams hp) {
  const RowsParams& p = hp.r;
  using G = StreamGeom<HD>;
  constexpr int kLanes = HD / (2 * W), kRows = 32 / kLanes, kPairs = HD / 2;
  constexpr int kChunkRows = kStreamChunk / (2 * HD), kGroups = kChunkRows / kRows;
  extern __shared__ uint4 smem_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane % kLanes, sub = lane / kLanes;
  uint8_t* smem = reinterpret_cast<uint8_t*>(smem_raw);
  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * kStreamStages * kStreamChunk);
  float* table_q = reinterpret_cast<float*>(smem + G::kRing) + warp * 2 * 4 * kPairs;
  float* table_k = table_q + 4 * kPairs;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kRing + G::kFactors) + warp * kStreamStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + G::kRing + G::kFactors + kStreamWarps * kStreamStages * 8);
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < kStreamStages; ++i) mbar_init(smem_u32(bars + i), 1);
    fence_mbar_init();
  }
  __syncthreads();

  const int q_chunks = (p.nq + kChunkRows - 1) / kChunkRows, chunks = q_chunks + (hp.nk + p.nv + kChunkRows - 1) / kChunkRows;
  const int64_t step = (int64_t)gridDim.x * kStreamWarps, first = (int64_t)warp * gridDim.x + blockIdx.x;

  // ---- loads, by lane 0: chunk after chunk of the warp's tokens
  int64_t load_t = first;
  int load_c = 0;
  auto issue = [&](uint32_t stage) {
    if (load_t >= p.tokens) return;
    const uint32_t dst = ring + stage * kStreamChunk, bar = smem_u32(bars + stage);
    if (load_c < q_chunks) {
      const int a = load_c * kChunkRows, n = min(p.nq - a, kChunkRows);
      mbar_arrive_expect_tx(bar, (uint32_t)(n * HD * 2));
      bulk_load(dst, p.q + load_t * p.q_stride + a * HD, (uint32_t)(n * HD * 2), bar);
    } else {
      const int a = (load_c - q_chunks) * kChunkRows, e = min(hp.nk + p.nv, a + kChunkRows);
      const int nk = max(0, min(e, hp.nk) - a), nv = e - a - nk;
      mbar_arrive_expect_tx(bar, (uint32_t)((nk + nv) * HD * 2));
      if (nk) bulk_load(dst, p.k + load_t * p.k_stride + a * HD, (uint32_t)(nk * HD * 2), bar);
      if (nv)
        bulk_load(dst + nk * HD * 2, p.v + load_t * p.v_stride + (a + nk - hp.nk) * HD, (uint32_t)(nv * HD * 2), bar);
    }
    if (++load_c == chunks) load_c = 0, load_t += step;
  };
  if (lane == 0)
    for (int i = 0; i < kStreamStages - 1; ++i) issue(i);

  // ---- positions and table rows, ahead of their tokens; a lane has pairs lane, lane + 32
  constexpr int kMine = kPairs / 32;
  int64_t pos[kMine];
  float cs[kMine], sn[kMine], qa[kMine], qb[kMine], ka[kMine], kb[kMine];
  bool bad = false;
  auto fetch_pos = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int axis = (int)(hp.axis_of[i] >> (2 * lane)) & 3;
      pos[i] = t < p.tokens && i * 32 + lane < p.rot / 2 ? p.pos[axis * hp.pos_stride + t] : -1;
    }
  };
  auto fetch_rows = [&](int64_t t) {
    bad = false;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      cs[i] = 1.f, sn[i] = 0.f;
      if (t >= p.tokens || i * 32 + lane >= p.rot / 2) continue;
      if (pos[i] < 0 || pos[i] >= p.positions) {
        bad = true;
        continue;
      }
      const int64_t at = pos[i] * (p.rot / 2) + i * 32 + lane;
      cs[i] = __ldg(p.cos_t + at);
      sn[i] = __ldg(p.sin_t + at);
    }
  };
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int2 c = columns_of<W, INTERLEAVED>(i * 32 + lane, p.rot);
    qa[i] = hp.q_norm ? __bfloat162float(hp.q_norm[c.x]) : 1.f;
    qb[i] = hp.q_norm ? __bfloat162float(hp.q_norm[c.y]) : 1.f;
    ka[i] = hp.k_norm ? __bfloat162float(hp.k_norm[c.x]) : 1.f;
    kb[i] = hp.k_norm ? __bfloat162float(hp.k_norm[c.y]) : 1.f;
  }
  const bool cached = !hp.k_out && hp.nk > 0;
  fetch_pos(first);
  int64_t slot = cached && first < p.tokens ? p.slots[first] : -1, next_slot = -1;
  fetch_rows(first);
  fetch_pos(first + step);

  const bool turn = j < p.rot / (2 * W);
  const bool apart = turn && !INTERLEAVED;  // pairs (i, i + rot / 2)
  const int c0 = apart ? W * j : 2 * W * j;
  const int to_c1 = apart ? p.rot / 2 : W;
  const FactorsAt fq = factors_at<HD, W, INTERLEAVED>(table_q, j), fk = factors_at<HD, W, INTERLEAVED>(table_k, j);

  uint32_t task = 0;
  bool ok = true;
  for (int64_t t = first; t < p.tokens && ok; t += step) {
    // ---- this token's factors; the next one's table row, the one's after it positions
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      put_factors<HD, W, INTERLEAVED>(table_q, i * 32 + lane, cs[i], sn[i], qa[i], qb[i]);
      put_factors<HD, W, INTERLEAVED>(table_k, i * 32 + lane, cs[i], sn[i], ka[i], kb[i]);
    }
    const bool skip = __any_sync(0xffffffffu, bad);
    if (skip && lane == 0) set_dev_error(p.err, kDevBadArgs);
    fetch_rows(t + step);
    fetch_pos(t + 2 * step);
    next_slot = cached && t + step < p.tokens ? p.slots[t + step] : -1;
    if (slot >= p.n_slots && cached) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
      slot = -1;
    }
    // cache row of head 0
    const int64_t row0 = ((slot >> p.page_shift) * hp.nk << p.page_shift) | (slot & ((1 << p.page_shift) - 1));
    __syncwarp();

    for (int c = 0; c < chunks; ++c, ++task) {
      const uint32_t stage = task % kStreamStages, at = ring + stage * kStreamChunk;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(bars + stage), (task / kStreamStages) & 1, p.err, kDevTimeoutFull,
                                             abort_flag))) {
        ok = false;
        break;
      }
      const bool is_q = c < q_chunks;
      const int r0 = (is_q ? c : c - q_chunks) * kChunkRows;
      const int n0 = is_q ? p.nq : hp.nk;
      const int r1 = min(is_q ? p.nq : hp.nk + p.nv, r0 + kChunkRows);
      const bool to_cache = !is_q && cached;
      const bool norm = (is_q ? hp.q_norm : hp.k_norm) != nullptr;
      if (!skip && !(to_cache && slot < 0)) {
        // (all groups' reads, sums and joins over the lanes together: one after the other, their latency was
        // most of a chunk's time)
        Cols<W> lo[kGroups], hi[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const uint32_t x_at = at + (uint32_t)((g * kRows + sub) * HD + c0) * 2;
          lo[g].lds(x_at);
          hi[g].lds(x_at + to_c1 * 2);
        }
        float rstd[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float2 x1[W / 2], x2[W / 2];
          unpack<W>(lo[g], hi[g], x1, x2);
          rstd[g] = norm ? square_sum<W>(x1, x2) : 1.f;
        }
        if (norm) {
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) rstd[g] += __shfl_xor_sync(0xffffffffu, rstd[g], o);
#pragma unroll
          for (int g = 0; g < kGroups; ++g) rstd[g] = rsqrtf(rstd[g] * (1.f / HD) + hp.eps);
        }
        Factors<W> f;
        (is_q ? fq : fk).load(f);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          if (r0 + g * kRows >= (FMT == kKvBf16 ? min(n0, r1) : r1)) break;  // (the warp as a whole; bf16 v goes as it came)
          const int r = r0 + g * kRows + sub;
          const bool live = r < r1, is_v = r >= n0;
          float2 x1[W / 2], x2[W / 2];
          unpack<W>(lo[g], hi[g], x1, x2);
          if (!is_v) turn_row<W, INTERLEAVED>(x1, x2, rstd[g], turn, f);
          if (FMT == kKvBf16 || !to_cache) {
            const uint32_t x_at = at + (uint32_t)((g * kRows + sub) * HD + c0) * 2;
            Cols<W> y, z;
            pack<W>(x1, x2, y, z);
            if (live && !is_v) {
              y.sts(x_at);
              z.sts(x_at + to_c1 * 2);
            }
          } else {
            const int64_t row = row0 + ((int64_t)(is_v ? r - hp.nk : r) << p.page_shift);
            const bool write = live && WX_IN_BOUNDS(p.err, row >= 0 && row < p.n_slots * hp.nk);
            store_quantised<FMT, HD, W>(p, x1, x2, write, is_v, row, c0, to_c1, j == 0);
          }
        }
        // ---- away with them: rows of one output as a whole, those of a cache one by one
        fence_proxy_async_smem();
        __syncwarp();
        if (!to_cache) {
          __nv_bfloat16* o = is_q ? p.q_out + t * p.q_out_stride : hp.k_out + t * hp.k_out_stride;
          if (lane == 0 && WX_IN_BOUNDS(p.err, r0 >= 0 && r1 <= n0)) bulk_store(o + r0 * HD, at, (uint32_t)((r1 - r0) * HD * 2));
        } else if (FMT == kKvBf16) {
          for (int r = r0 + lane; r < r1; r += 32) {
            const int64_t row = row0 + ((int64_t)(r >= n0 ? r - hp.nk : r) << p.page_shift);
            if (WX_IN_BOUNDS(p.err, row >= 0 && row < p.n_slots * hp.nk))
              bulk_store((r >= n0 ? p.vc : p.kc) + row * HD * 2, at + (uint32_t)((r - r0) * HD * 2), HD * 2);
          }
        }
      }
      bulk_commit();
      bulk_wait_read<1>();  // the chunk before this one has left its stage:
      __syncwarp();         // that is the one to fill next
      if (lane == 0) issue((task + kStreamStages - 1) % kStreamStages);
    }
    slot = next_slot;
  }
  bulk_wait_all();
  if (!ok) {  // copies still in flight must land before the CTA ends: the time of one more bounded wait
    const uint64_t from = globaltimer_ns();
    while (globaltimer_ns() - from < 2000000ull) {}
  }
}

// ------------------------------------------------------------------- reading back
// value * scale, one rounding to bf16; a slot < 0 reads zeros. A lane reads 16 values of a row,
// HD / 16 lanes a row; a warp has up to kRowGroups groups of rows in flight, as above.
struct ReadParams {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int64_t* slots;
  int64_t tokens, n_slots;
  int nkv, page_shift;
  int rows_per_warp, chunks;
  __nv_bfloat16 *k, *v;
  int64_t out_stride;
  int* err;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams p) {
  constexpr int kLanes = HD / 16, kRows = 32 / kLanes;
  constexpr int kVec = FMT == kKvBf16 ? 2 : 1;  // 16-byte units of 16 values
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes;
  const unsigned blk = blockIdx.x / (unsigned)p.chunks;  // (as above)
  const int64_t t = (int64_t)blk * 8 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int r0 = (int)(blockIdx.x - blk * (unsigned)p.chunks) * p.rows_per_warp;
  const int r1 = min(2 * p.nkv, r0 + p.rows_per_warp);
  int64_t slot = p.slots[t];
  if (slot >= p.n_slots) {
    if (lane == 0) set_dev_error(p.err, kDevBadArgs);
    slot = -1;
  }
  const int64_t page = slot >> p.page_shift, inside = slot & ((1 << p.page_shift) - 1);
  uint4 x[kRowGroups][kVec];
  float s[kRowGroups];
#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    const int r = r0 + g * kRows + lane / kLanes;
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[g][e] = make_uint4(0, 0, 0, 0);
    s[g] = 0.f;
    if (r >= r1 || slot < 0) continue;
    const bool is_v = r >= p.nkv;
    const int64_t row = ((page * p.nkv + (is_v ? r - p.nkv : r)) << p.page_shift) | inside;
    if (!WX_IN_BOUNDS(p.err, row >= 0 && row < p.n_slots * p.nkv)) continue;
    const uint4* src = reinterpret_cast<const uint4*>(is_v ? p.vc : p.kc) + (row * HD / 16 + j) * kVec;
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[g][e] = __ldg(src + e);
    if constexpr (FMT != kKvBf16) s[g] = __ldg((is_v ? p.vs : p.ks) + row);
  }
#pragma unroll
  for (int g = 0; g < kRowGroups; ++g) {
    const int r = r0 + g * kRows + lane / kLanes;
    if (r >= r1) continue;
    const bool is_v = r >= p.nkv;
    uint4* dst = reinterpret_cast<uint4*>((is_v ? p.v : p.k) + t * p.out_stride +
                                          (int64_t)(is_v ? r - p.nkv : r) * HD) + 2 * j;
    if constexpr (FMT == kKvBf16) {
      dst[0] = x[g][0];
      dst[1] = x[g][1];
    } else {
      const uint4 u = x[g][0];
      dst[0] = make_uint4(bytes_times<FMT>(u.x, 0, s[g]), bytes_times<FMT>(u.x, 1, s[g]),
                          bytes_times<FMT>(u.y, 0, s[g]), bytes_times<FMT>(u.y, 1, s[g]));
      dst[1] = make_uint4(bytes_times<FMT>(u.z, 0, s[g]), bytes_times<FMT>(u.z, 1, s[g]),
                          bytes_times<FMT>(u.w, 0, s[g]), bytes_times<FMT>(u.w, 1, s[g]));
    }
  }
}

// --------------------------------------------------------------------- host side
int check_kv_cache(wx_ctx* ctx, const wx_kv_cache* c) {
  WX_CHECK_ARG(ctx, c && c->k && c->v && c->pages > 0 && c->kv_heads > 0);
  if (c->head_dim != 128 && c->head_dim != 64)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "cache head_dim must be 128 or 64 (got %d)", c->head_dim);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return set_error(ctx, WX_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)", c->page_size);
  if (c->format != WX_KV_BF16 && c->format != WX_KV_INT8 && c->format != WX_KV_E4M3)
    return set_error(ctx, WX_ERR_INVALID, "unknown cache format %d", c->format);
  WX_CHECK_ARG(ctx, c->format == WX_KV_BF16 || (c->k_scale && c->v_scale));
  WX_CHECK_ARG(ctx, aligned16(c->k) && aligned16(c->v) && aligned16(c->k_scale) && aligned16(c->v_scale));
  // rows of the cache are indexed by 32-bit tile coordinates
  if (c->pages > INT32_MAX / c->page_size / c->kv_heads)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "pages * kv_heads * page_size must be below 2^31");
  return WX_OK;
}

static int check_rope(wx_ctx* ctx, const wx_rope* r, int head_dim, const int32_t* pos) {
  WX_CHECK_ARG(ctx, r && r->cos_t && r->sin_t && pos && r->positions > 0);
  WX_CHECK_ARG(ctx, r->rot > 0 && r->rot % 8 == 0 && r->rot <= head_dim);
  WX_CHECK_ARG(ctx, aligned16(r->cos_t) && aligned16(r->sin_t));
  return WX_OK;
}

// How a token's rows are dealt to warps: as many as a warp keeps in flight, fewer where there are
// too few tokens to give every SM 64 warps (a warp's rows follow one another).
static int64_t deal_rows(wx_ctx* ctx, int64_t tokens, int per_token, int rows_at_once, int* rows_per_warp, int* chunks) {
  *rows_per_warp = rows_at_once * kRowGroups;
  while (*rows_per_warp > rows_at_once &&
         tokens * ((per_token + *rows_per_warp - 1) / *rows_per_warp) < (int64_t)ctx->num_sms * 64)
    *rows_per_warp /= 2;
  *chunks = (per_token + *rows_per_warp - 1) / *rows_per_warp;
  return (tokens + 7) / 8 * *chunks;  // blocks of 8 warps
}

template <int FMT, int HD, int W>
static void start_rows(unsigned g, cudaStream_t s, const RowsParams& p) {
  if (p.interleaved) text_rows_kernel<FMT, HD, W, true><<<g, 256, 0, s>>>(p);
  else text_rows_kernel<FMT, HD, W, false><<<g, 256, 0, s>>>(p);
}

template <int HD, int W>
static void start_rows(int fmt, unsigned g, cudaStream_t s, const RowsParams& p) {
  if (fmt == kKvInt8) start_rows<kKvInt8, HD, W>(g, s, p);
  else if (fmt == kKvE4m3) start_rows<kKvE4m3, HD, W>(g, s, p);
  else start_rows<kKvBf16, HD, W>(g, s, p);
}

static int launch_rows(wx_ctx* ctx, RowsParams& p, int fmt, int head_dim) {
  if (p.tokens == 0) return WX_OK;
  const int W = p.rot % 16 == 0 ? 8 : 4;
  const int64_t blocks =
      deal_rows(ctx, p.tokens, p.nq + 2 * p.nkv, 32 / (head_dim / (2 * W)), &p.rows_per_warp, &p.chunks);
  if (blocks > INT32_MAX) return set_error(ctx, WX_ERR_UNSUPPORTED, "too many tokens in one call");
  p.err = ctx->dev_err;
  ProfScope prof(ctx, kProfRow);
  const unsigned g = (unsigned)blocks;
  if (head_dim == 128)
    W == 8 ? start_rows<128, 8>(fmt, g, ctx->stream, p) : start_rows<128, 4>(fmt, g, ctx->stream, p);
  else
    W == 8 ? start_rows<64, 8>(fmt, g, ctx->stream, p) : start_rows<64, 4>(fmt, g, ctx->stream, p);
  return launch_status(ctx, "text_rows");
}

static bool row_ok(const void* p, int64_t stride, int64_t heads, int hd) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= heads * hd;
}

static void set_rope(RowsParams& p, const wx_rope* r, const int32_t* pos) {
  p.cos_t = r->cos_t;
  p.sin_t = r->sin_t;
  p.positions = r->positions;
  p.rot = r->rot;
  p.interleaved = r->interleaved != 0;
  p.pos = pos;
}

static void set_cache(RowsParams& p, const wx_kv_cache* c, const int64_t* slots) {
  p.nkv = c->kv_heads;
  p.kc = static_cast<uint8_t*>(c->k);
  p.vc = static_cast<uint8_t*>(c->v);
  p.ks = c->k_scale;
  p.vs = c->v_scale;
  p.slots = slots;
  p.n_slots = c->pages * c->page_size;
  p.page_shift = __builtin_ctz((unsigned)c->page_size);
}

// head norms and position axes of a call
static int set_heads(wx_ctx* ctx, HeadParams& p, const wx_rope* rope, const wx_rope_axes* axes, const void* q_norm,
                     const void* k_norm, float eps) {
  WX_CHECK_ARG(ctx, aligned16(q_norm) && aligned16(k_norm));
  WX_CHECK_ARG(ctx, (!q_norm && !k_norm) || (eps > 0.f && eps < INFINITY));
  p.q_norm = static_cast<const __nv_bfloat16*>(q_norm);
  p.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  p.eps = eps;
  if (!axes) return WX_OK;
  WX_CHECK_ARG(ctx, axes->n_axes >= 1 && axes->n_axes <= 4);
  // (0: positions that all axes share, as text's are)
  WX_CHECK_ARG(ctx, axes->n_axes == 1 || axes->position_stride == 0 || axes->position_stride >= p.r.tokens);
  p.pos_stride = axes->position_stride;
  for (int i = 0; i < rope->rot / 2; ++i) {
    WX_CHECK_ARG(ctx, axes->axis_of_pair[i] < axes->n_axes);
    p.axis_of[i / 32] |= (uint64_t)axes->axis_of_pair[i] << (2 * (i % 32));
  }
  return WX_OK;
}

template <int FMT, int HD, int W, bool INTERLEAVED>
static int start_heads(wx_ctx* ctx, const HeadParams& p, unsigned grid, bool stream) {
  if (!stream) {
    head_rows_kernel<FMT, HD, W, INTERLEAVED><<<grid, 256, 0, ctx->stream>>>(p);
    return launch_status(ctx, "head_rows");
  }
  auto fn = head_stream_kernel<FMT, HD, W, INTERLEAVED>;
  const int st = ensure_smem_attr(ctx, (const void*)fn, StreamGeom<HD>::kSmem, "head_stream");
  if (st) return st;
  fn<<<grid, 32 * kStreamWarps, StreamGeom<HD>::kSmem, ctx->stream>>>(p);
  return launch_status(ctx, "head_stream");
}
template <int FMT, int HD>
static int start_heads(wx_ctx* ctx, const HeadParams& p, unsigned g, bool wide, bool stream) {
  if (wide)
    return p.r.interleaved ? start_heads<FMT, HD, 8, true>(ctx, p, g, stream) : start_heads<FMT, HD, 8, false>(ctx, p, g, stream);
  return p.r.interleaved ? start_heads<FMT, HD, 4, true>(ctx, p, g, stream) : start_heads<FMT, HD, 4, false>(ctx, p, g, stream);
}
template <int HD>
static int start_heads(wx_ctx* ctx, int fmt, const HeadParams& p, unsigned g, bool wide, bool stream) {
  if (fmt == kKvInt8) return start_heads<kKvInt8, HD>(ctx, p, g, wide, stream);
  if (fmt == kKvE4m3) return start_heads<kKvE4m3, HD>(ctx, p, g, wide, stream);
  return start_heads<kKvBf16, HD>(ctx, p, g, wide, stream);
}
static int launch_heads(wx_ctx* ctx, HeadParams& p, int fmt, int head_dim) {
  const bool wide = p.r.rot % 16 == 0;
  p.r.err = ctx->dev_err;
  ProfScope prof(ctx, kProfRow);
  // The persistent kernel takes chunks of 4 KB: it wants one and a half for each of its warps at least, and rows
  // that fill them. Rows kernel : persistent, us a call, 32 + 8 heads of 128 (48 rows in 3 chunks) 600 tokens
  // 12.3 : 12.3, 1,500 18.5 : 14.3, 8,000 45 : 39 (into int8 55 : 47); 8 + 1 heads (10 rows in 2 chunks)
  // 8,000 22.5 : 24.5; 16 + 16 heads of 64 (48 of 64 rows) 4,000 18.4 : 16.4, 8,000 into int8 31 : 35.
  const int per = kStreamChunk / (2 * head_dim), per_token = p.r.nq + p.nk + p.r.nv;
  const int64_t filled = (p.r.nq + per - 1) / per + (p.nk + p.r.nv + per - 1) / per;
  const bool stream = 2 * p.r.tokens * filled >= 3 * (int64_t)ctx->num_sms * kStreamWarps && 5 * per_token >= 3 * filled * per;
  unsigned grid;
  if (stream) {
    grid = (unsigned)ctx->num_sms;
  } else {
    // as deal_rows, but for q rows and k and v rows apart
    const int at_once = 32 / (head_dim / (wide ? 16 : 8));
    int rows = at_once * kRowGroups;
    auto chunks = [&] { return (p.r.nq + rows - 1) / rows + (p.nk + p.r.nv + rows - 1) / rows; };
    while (rows > at_once && p.r.tokens * chunks() < (int64_t)ctx->num_sms * 64) rows /= 2;
    p.r.rows_per_warp = rows;
    p.q_chunks = (p.r.nq + rows - 1) / rows;
    p.r.chunks = chunks();
    const int64_t blocks = (p.r.tokens + 7) / 8 * p.r.chunks;
    if (blocks > INT32_MAX) return set_error(ctx, WX_ERR_UNSUPPORTED, "too many tokens in one call");
    grid = (unsigned)blocks;
  }
  return head_dim == 128 ? start_heads<128>(ctx, fmt, p, grid, wide, stream)
                         : start_heads<64>(ctx, fmt, p, grid, wide, stream);
}

}  // namespace wx

using namespace wx;

extern "C" {

int wx_rope_inv_freq(int rot, double base, int scaling, double factor, double original_positions, double low,
                     double high, double* inv_freq) {
  if (!inv_freq || rot <= 0 || rot % 2 || rot > 2 * kRopeMaxPairs || !(base > 0.0)) return WX_ERR_INVALID;
  if (scaling != WX_ROPE_PLAIN && !(factor >= 1.0)) return WX_ERR_INVALID;
  if (scaling == WX_ROPE_BY_PARTS && (!(original_positions > 0.0) || !(high > low))) return WX_ERR_INVALID;
  for (int i = 0; i < rot / 2; ++i) {
    const double inv = pow(base, -2.0 * i / rot);
    double v = inv;
    if (scaling == WX_ROPE_LINEAR) {
      v = inv / factor;
    } else if (scaling == WX_ROPE_BY_PARTS) {
      // turns of this pair over the original length: few turns are interpolated, many kept
      const double turns = original_positions * inv / (2.0 * M_PI);
      const double w = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
      v = (1.0 - w) * inv / factor + w * inv;
    } else if (scaling != WX_ROPE_PLAIN) {
      return WX_ERR_INVALID;
    }
    inv_freq[i] = v;
  }
  return WX_OK;
}

int wx_rope_table(wx_ctx* ctx, const double* inv_freq, int nf, int64_t positions, double magnitude, float* cos_t,
                  float* sin_t) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && inv_freq && cos_t && sin_t && nf > 0 && nf <= kRopeMaxPairs && positions >= 0);
  WX_CHECK_ARG(ctx, positions < (int64_t)1 << 40);
  if (!positions) return WX_OK;
  RopeFreqs f{};
  for (int i = 0; i < nf; ++i) f.inv[i] = inv_freq[i];
  const unsigned grid = (unsigned)std::min<int64_t>((positions * nf + 255) / 256, (int64_t)ctx->num_sms * 16);
  rope_table_kernel<<<grid, 256, 0, ctx->stream>>>(f, nf, positions, magnitude, cos_t, sin_t);
  return launch_status(ctx, "rope_table");
}

int wx_rope_apply(wx_ctx* ctx, const wx_rope* rope, const int32_t* positions, const void* x, int64_t row_stride,
                  int64_t tokens, int heads, int head_dim, void* y, int64_t y_stride) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0 && heads > 0);
  if (head_dim != 128 && head_dim != 64)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "rope head_dim must be 128 or 64 (got %d)", head_dim);
  if (!tokens) return WX_OK;
  int st = check_rope(ctx, rope, head_dim, positions);
  if (st) return st;
  WX_CHECK_ARG(ctx, row_ok(x, row_stride, heads, head_dim) && row_ok(y, y_stride, heads, head_dim));
  RowsParams p{};
  set_rope(p, rope, positions);
  p.q = static_cast<const __nv_bfloat16*>(x);
  p.q_stride = row_stride;
  p.nq = heads;
  p.tokens = tokens;
  p.q_out = static_cast<__nv_bfloat16*>(y);
  p.q_out_stride = y_stride;
  return launch_rows(ctx, p, kKvBf16, head_dim);
}

int wx_kv_append(wx_ctx* ctx, const wx_kv_cache* cache, const void* k, int64_t k_stride, const void* v,
                 int64_t v_stride, int64_t tokens, const int64_t* slots) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0);
  int st = check_kv_cache(ctx, cache);
  if (st || !tokens) return st;
  WX_CHECK_ARG(ctx, slots && row_ok(k, k_stride, cache->kv_heads, cache->head_dim) &&
                        row_ok(v, v_stride, cache->kv_heads, cache->head_dim));
  RowsParams p{};
  set_cache(p, cache, slots);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.tokens = tokens;
  return launch_rows(ctx, p, cache->format, cache->head_dim);
}

int wx_rope_kv_append(wx_ctx* ctx, const wx_rope* rope, const int32_t* positions, const void* q, int64_t q_stride,
                      int q_heads, const wx_kv_cache* cache, const void* k, int64_t k_stride, const void* v,
                      int64_t v_stride, int64_t tokens, const int64_t* slots, void* q_out, int64_t q_out_stride) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0 && q_heads > 0);
  int st = check_kv_cache(ctx, cache);
  if (st || !tokens) return st;
  if ((st = check_rope(ctx, rope, cache->head_dim, positions))) return st;
  const int hd = cache->head_dim;
  WX_CHECK_ARG(ctx, slots && row_ok(q, q_stride, q_heads, hd) && row_ok(q_out, q_out_stride, q_heads, hd) &&
                        row_ok(k, k_stride, cache->kv_heads, hd) && row_ok(v, v_stride, cache->kv_heads, hd));
  RowsParams p{};
  set_rope(p, rope, positions);
  set_cache(p, cache, slots);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.nq = q_heads;
  p.tokens = tokens;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_out_stride = q_out_stride;
  return launch_rows(ctx, p, cache->format, hd);
}

int wx_norm_rope_apply(wx_ctx* ctx, const wx_rope* rope, const wx_rope_axes* axes, const int32_t* positions,
                       const void* q, int64_t q_stride, int q_heads, const void* q_norm, const void* k,
                       int64_t k_stride, int k_heads, const void* k_norm, float eps, int64_t tokens, int head_dim,
                       void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0 && q_heads > 0 && k_heads >= 0 && q_heads <= INT32_MAX - k_heads);
  if (head_dim != 128 && head_dim != 64)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "rope head_dim must be 128 or 64 (got %d)", head_dim);
  if (!tokens) return WX_OK;
  int st = check_rope(ctx, rope, head_dim, positions);
  if (st) return st;
  WX_CHECK_ARG(ctx, row_ok(q, q_stride, q_heads, head_dim) && row_ok(q_out, q_out_stride, q_heads, head_dim));
  WX_CHECK_ARG(ctx, k_heads == 0 ||
                        (row_ok(k, k_stride, k_heads, head_dim) && row_ok(k_out, k_out_stride, k_heads, head_dim)));
  HeadParams p{};
  set_rope(p.r, rope, positions);
  p.r.tokens = tokens;
  if ((st = set_heads(ctx, p, rope, axes, q_norm, k_norm, eps))) return st;
  p.r.q = static_cast<const __nv_bfloat16*>(q);
  p.r.k = static_cast<const __nv_bfloat16*>(k);
  p.r.q_stride = q_stride;
  p.r.k_stride = k_stride;
  p.r.nq = q_heads;
  p.nk = k_heads;
  p.r.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.r.q_out_stride = q_out_stride;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.k_out_stride = k_out_stride;
  return launch_heads(ctx, p, kKvBf16, head_dim);
}

int wx_norm_rope_kv_append(wx_ctx* ctx, const wx_rope* rope, const wx_rope_axes* axes, const int32_t* positions,
                           const void* q, int64_t q_stride, int q_heads, const void* q_norm, const void* k_norm,
                           float eps, const wx_kv_cache* cache, const void* k, int64_t k_stride, const void* v,
                           int64_t v_stride, int64_t tokens, const int64_t* slots, void* q_out,
                           int64_t q_out_stride) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0 && q_heads > 0);
  int st = check_kv_cache(ctx, cache);
  if (st || !tokens) return st;
  if ((st = check_rope(ctx, rope, cache->head_dim, positions))) return st;
  const int hd = cache->head_dim;
  WX_CHECK_ARG(ctx, slots && row_ok(q, q_stride, q_heads, hd) && row_ok(q_out, q_out_stride, q_heads, hd) &&
                        row_ok(k, k_stride, cache->kv_heads, hd) && row_ok(v, v_stride, cache->kv_heads, hd));
  HeadParams p{};
  set_rope(p.r, rope, positions);
  set_cache(p.r, cache, slots);
  p.r.tokens = tokens;
  if ((st = set_heads(ctx, p, rope, axes, q_norm, k_norm, eps))) return st;
  p.r.q = static_cast<const __nv_bfloat16*>(q);
  p.r.k = static_cast<const __nv_bfloat16*>(k);
  p.r.v = static_cast<const __nv_bfloat16*>(v);
  p.r.q_stride = q_stride;
  p.r.k_stride = k_stride;
  p.r.v_stride = v_stride;
  p.r.nq = q_heads;
  p.nk = p.r.nv = cache->kv_heads;
  p.r.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.r.q_out_stride = q_out_stride;
  return launch_heads(ctx, p, cache->format, hd);
}

int wx_kv_read(wx_ctx* ctx, const wx_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out,
               int64_t out_stride) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && tokens >= 0);
  int st = check_kv_cache(ctx, cache);
  if (st || !tokens) return st;
  WX_CHECK_ARG(ctx, slots && row_ok(k_out, out_stride, cache->kv_heads, cache->head_dim) &&
                        row_ok(v_out, out_stride, cache->kv_heads, cache->head_dim));
  ReadParams p{};
  p.kc = static_cast<const uint8_t*>(cache->k);
  p.vc = static_cast<const uint8_t*>(cache->v);
  p.ks = cache->k_scale;
  p.vs = cache->v_scale;
  p.slots = slots;
  p.tokens = tokens;
  p.n_slots = cache->pages * cache->page_size;
  p.nkv = cache->kv_heads;
  p.page_shift = __builtin_ctz((unsigned)cache->page_size);
  p.k = static_cast<__nv_bfloat16*>(k_out);
  p.v = static_cast<__nv_bfloat16*>(v_out);
  p.out_stride = out_stride;
  p.err = ctx->dev_err;
  const int64_t blocks =
      deal_rows(ctx, tokens, 2 * cache->kv_heads, 32 / (cache->head_dim / 16), &p.rows_per_warp, &p.chunks);
  if (blocks > INT32_MAX) return set_error(ctx, WX_ERR_UNSUPPORTED, "too many tokens in one call");
  ProfScope prof(ctx, kProfRow);
  const unsigned g = (unsigned)blocks;
  const bool big = cache->head_dim == 128;
  if (cache->format == WX_KV_INT8)
    big ? kv_read_kernel<kKvInt8, 128><<<g, 256, 0, ctx->stream>>>(p)
        : kv_read_kernel<kKvInt8, 64><<<g, 256, 0, ctx->stream>>>(p);
  else if (cache->format == WX_KV_E4M3)
    big ? kv_read_kernel<kKvE4m3, 128><<<g, 256, 0, ctx->stream>>>(p)
        : kv_read_kernel<kKvE4m3, 64><<<g, 256, 0, ctx->stream>>>(p);
  else
    big ? kv_read_kernel<kKvBf16, 128><<<g, 256, 0, ctx->stream>>>(p)
        : kv_read_kernel<kKvBf16, 64><<<g, 256, 0, ctx->stream>>>(p);
  return launch_status(ctx, "kv_read");
}

}  // extern "C"
