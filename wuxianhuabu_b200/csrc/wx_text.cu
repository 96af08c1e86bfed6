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
//
// With HEADS, q and k rows are normalised first, y = x / sqrt(mean x^2 + eps) * w, the squares summed over
// the row's lanes, and each pair may turn by a position of its own axis. All of it stays in fp32 until
// the one rounding (or quantisation) at the end.
constexpr int kRowGroups = 4;

struct RowsParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int nq, nkv, nv;                       // q, k and v rows of a token (no cache: v none)
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
  // HEADS: norm weights (nullptr: none), two bits for each pair's axis, where the axes' positions lie,
  // and k rows that go here instead of into a cache
  const __nv_bfloat16 *q_norm, *k_norm;
  float eps;
  int axes;
  uint64_t axis_of[2];
  int64_t pos_stride;
  __nv_bfloat16* k_out;
  int64_t k_out_stride;
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

template <int FMT, int HD, int W, bool INTERLEAVED, bool HEADS>
__global__ void __launch_bounds__(256, 3) text_rows_kernel(RowsParams p) {
  constexpr int kLanes = HD / (2 * W);  // lanes of a row
  constexpr int kRows = 32 / kLanes;    // rows of a warp at a time
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes;
  const int per_token = p.nq + p.nkv + p.nv;
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
    int64_t pos = p.pos[t];
    bool bad = pos < 0 || pos >= p.positions;
    int64_t pos_of[4] = {pos, pos, pos, pos};
    uint32_t codes = 0;  // axes of this lane's pairs, two bits each
    if constexpr (HEADS) {
      if (p.axes > 1) {
        bool same = true;
#pragma unroll
        for (int a = 1; a < 4; ++a) {
          if (a >= p.axes) break;
          pos_of[a] = p.pos[a * p.pos_stride + t];
          bad |= pos_of[a] < 0 || pos_of[a] >= p.positions;
          same &= pos_of[a] == pos;
        }
        // (text: the axes run together, and one row of the table serves all pairs)
        if (!same) codes = (uint32_t)(p.axis_of[j * W >= 32] >> (2 * (j * W & 31))) & ((1u << 2 * W) - 1u);
      }
    }
    if (bad) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
      return;
    }
    if (turn) {
      bool whole = true;
      if constexpr (HEADS) {
        whole = codes == (codes & 3u) * (0x5555u & ((1u << 2 * W) - 1u));
        if (whole) pos = (codes & 3u) == 0 ? pos_of[0] : (codes & 3u) == 1 ? pos_of[1] : (codes & 3u) == 2 ? pos_of[2] : pos_of[3];
      }
      if (whole) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const float4 c = *reinterpret_cast<const float4*>(p.cos_t + pos * (p.rot / 2) + W * j + i);
          const float4 s = *reinterpret_cast<const float4*>(p.sin_t + pos * (p.rot / 2) + W * j + i);
          cs[i] = c.x, cs[i + 1] = c.y, cs[i + 2] = c.z, cs[i + 3] = c.w;
          sn[i] = s.x, sn[i + 1] = s.y, sn[i + 2] = s.z, sn[i + 3] = s.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const uint32_t a = codes >> (2 * i) & 3u;
          const int64_t at = (a == 0 ? pos_of[0] : a == 1 ? pos_of[1] : a == 2 ? pos_of[2] : pos_of[3]) * (p.rot / 2) + W * j + i;
          cs[i] = p.cos_t[at];
          sn[i] = p.sin_t[at];
        }
      }
    }
  }
  int64_t slot = -1;
  if (HEADS ? p.slots != nullptr : p.nkv) {
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
    if constexpr (HEADS) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const __nv_bfloat16* weight = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
      if (weight) {
        const float rstd = rsqrtf(ss * (1.f / HD) + p.eps);
        Cols<W> lo, hi;
        lo.load(weight + c0);
        hi.load(weight + c1);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          x[2 * i] *= rstd * bf16_lo(lo.w[i]), x[2 * i + 1] *= rstd * bf16_hi(lo.w[i]);
          x[W + 2 * i] *= rstd * bf16_lo(hi.w[i]), x[W + 2 * i + 1] *= rstd * bf16_hi(hi.w[i]);
        }
      }
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
    const bool plain_k = HEADS && !is_q && p.k_out;
    if (is_q || FMT == kKvBf16) {
      __nv_bfloat16* o = is_q      ? p.q_out + t * p.q_out_stride + (int64_t)h * HD
                         : plain_k ? p.k_out + t * p.k_out_stride + (int64_t)h * HD
                                   : reinterpret_cast<__nv_bfloat16*>(is_v ? p.vc : p.kc) + row * HD;
      if (!is_q && !plain_k && slot < 0) continue;
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
static void start_rows(unsigned g, cudaStream_t s, const RowsParams& p, bool heads) {
  if (heads) {
    if (p.interleaved) text_rows_kernel<FMT, HD, W, true, true><<<g, 256, 0, s>>>(p);
    else text_rows_kernel<FMT, HD, W, false, true><<<g, 256, 0, s>>>(p);
  } else {
    if (p.interleaved) text_rows_kernel<FMT, HD, W, true, false><<<g, 256, 0, s>>>(p);
    else text_rows_kernel<FMT, HD, W, false, false><<<g, 256, 0, s>>>(p);
  }
}

template <int HD, int W>
static void start_rows(int fmt, unsigned g, cudaStream_t s, const RowsParams& p, bool heads) {
  if (fmt == kKvInt8) start_rows<kKvInt8, HD, W>(g, s, p, heads);
  else if (fmt == kKvE4m3) start_rows<kKvE4m3, HD, W>(g, s, p, heads);
  else start_rows<kKvBf16, HD, W>(g, s, p, heads);
}

static int launch_rows(wx_ctx* ctx, RowsParams& p, int fmt, int head_dim, bool heads = false) {
  if (p.tokens == 0) return WX_OK;
  const int W = p.rot % 16 == 0 ? 8 : 4;
  const int64_t blocks =
      deal_rows(ctx, p.tokens, p.nq + p.nkv + p.nv, 32 / (head_dim / (2 * W)), &p.rows_per_warp, &p.chunks);
  if (blocks > INT32_MAX) return set_error(ctx, WX_ERR_UNSUPPORTED, "too many tokens in one call");
  p.err = ctx->dev_err;
  ProfScope prof(ctx, kProfRow);
  const unsigned g = (unsigned)blocks;
  if (head_dim == 128)
    W == 8 ? start_rows<128, 8>(fmt, g, ctx->stream, p, heads) : start_rows<128, 4>(fmt, g, ctx->stream, p, heads);
  else
    W == 8 ? start_rows<64, 8>(fmt, g, ctx->stream, p, heads) : start_rows<64, 4>(fmt, g, ctx->stream, p, heads);
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
  p.nkv = p.nv = c->kv_heads;
  p.kc = static_cast<uint8_t*>(c->k);
  p.vc = static_cast<uint8_t*>(c->v);
  p.ks = c->k_scale;
  p.vs = c->v_scale;
  p.slots = slots;
  p.n_slots = c->pages * c->page_size;
  p.page_shift = __builtin_ctz((unsigned)c->page_size);
}

// head norms and position axes of a call
static int set_heads(wx_ctx* ctx, RowsParams& p, const wx_rope* rope, const wx_rope_axes* axes, const void* q_norm,
                     const void* k_norm, float eps) {
  WX_CHECK_ARG(ctx, aligned16(q_norm) && aligned16(k_norm));
  WX_CHECK_ARG(ctx, (!q_norm && !k_norm) || (eps > 0.f && eps < INFINITY));
  p.q_norm = static_cast<const __nv_bfloat16*>(q_norm);
  p.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  p.eps = eps;
  p.axes = 1;
  if (!axes) return WX_OK;
  WX_CHECK_ARG(ctx, axes->n_axes >= 1 && axes->n_axes <= 4);
  WX_CHECK_ARG(ctx, axes->n_axes == 1 || axes->position_stride >= p.tokens);
  p.axes = axes->n_axes;
  p.pos_stride = axes->position_stride;
  for (int i = 0; i < rope->rot / 2; ++i) {
    WX_CHECK_ARG(ctx, axes->axis_of_pair[i] < axes->n_axes);
    p.axis_of[i / 32] |= (uint64_t)axes->axis_of_pair[i] << (2 * (i % 32));
  }
  return WX_OK;
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
  RowsParams p{};
  set_rope(p, rope, positions);
  p.tokens = tokens;
  if ((st = set_heads(ctx, p, rope, axes, q_norm, k_norm, eps))) return st;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.nq = q_heads;
  p.nkv = k_heads;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_out_stride = q_out_stride;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.k_out_stride = k_out_stride;
  return launch_rows(ctx, p, kKvBf16, head_dim, true);
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
  RowsParams p{};
  set_rope(p, rope, positions);
  set_cache(p, cache, slots);
  p.tokens = tokens;
  if ((st = set_heads(ctx, p, rope, axes, q_norm, k_norm, eps))) return st;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.nq = q_heads;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.q_out_stride = q_out_stride;
  return launch_rows(ctx, p, cache->format, hd, true);
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
