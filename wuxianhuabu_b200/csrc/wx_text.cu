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
#include "wx_ptx.cuh"
#include "wx_text.h"

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
// One launch serves rope alone, the cache write alone and both fused. A token's rows are
// its q heads, then k heads, then v heads; HD/8 neighbouring lanes own a row, 8 values each.
struct RowsParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int nq, nkv;                           // q rows, and k (= v) rows of a token (0 without a cache)
  int64_t tokens;
  int rows_per_warp;
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

// 8 values of a row -> the stored format. The scale is amax / 127 or amax / 448 of the fp32
// values (amax reduced over the row's lanes); the value stored is value * (127 | 448) / amax
// rounded to nearest even. A row with infinity or NaN stores scale NaN and zeros, so that it
// reads back as NaN; a row below 2^-100 everywhere (127 / amax could overflow) stores zeros.
template <int FMT, int HD>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float* scale) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  bool bad = false;  // fmaxf drops NaN
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= !(fabsf(x[i]) <= 3.402823466e38f);
  if (bad) amax = INFINITY;
#pragma unroll
  for (int o = HD / 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  constexpr float kMax = FMT == kKvInt8 ? 127.f : 448.f;
  const bool finite = amax <= 3.402823466e38f;
  const bool live = finite && amax >= 0x1p-100f;
  const float inv = live ? __fdiv_rn(kMax, amax) : 0.f;
  *scale = finite ? (live ? __fdiv_rn(amax, kMax) : 0.f) : __int_as_float(0x7fc00000);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = live ? __fmul_rn(x[4 * h + i], inv) : 0.f;
    if constexpr (FMT == kKvInt8) {
      uint32_t b = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) b |= ((uint32_t)__float2int_rn(y[i]) & 0xffu) << (8 * i);
      w[h] = b;
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | hi << 16;
    }
  }
  return make_uint2(w[0], w[1]);
}

template <int FMT, int HD>
__global__ void __launch_bounds__(256) text_rows_kernel(RowsParams p) {
  constexpr int kLanes = HD / 8;         // lanes of a row
  constexpr int kRows = 32 / kLanes;     // rows of a warp at a time
  const int lane = threadIdx.x & 31;
  const int j = lane % kLanes;
  const int per_token = p.nq + 2 * p.nkv;
  const int chunks = (per_token + p.rows_per_warp - 1) / p.rows_per_warp;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t t = w / chunks;
  if (t >= p.tokens) return;
  const int r0 = (int)(w % chunks) * p.rows_per_warp;
  const int r1 = min(per_token, r0 + p.rows_per_warp);

  // columns of this lane: two groups of 4, so that both halves of a pair sit in one lane
  const bool turn = j < p.rot / 8;
  const int c0 = turn ? (p.interleaved ? 8 * j : 4 * j) : 8 * j;
  const int c1 = turn ? (p.interleaved ? 8 * j + 4 : p.rot / 2 + 4 * j) : 8 * j + 4;
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  bool pos_ok = true;
  if (p.rot) {
    const int64_t pos = p.pos[t];
    pos_ok = pos >= 0 && pos < p.positions;
    if (!pos_ok) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
    } else if (turn) {
      cs = *reinterpret_cast<const float4*>(p.cos_t + pos * (p.rot / 2) + 4 * j);
      sn = *reinterpret_cast<const float4*>(p.sin_t + pos * (p.rot / 2) + 4 * j);
    }
  }
  if (!pos_ok) return;
  int64_t slot = -1;
  if (p.nkv) {
    slot = p.slots[t];
    if (slot >= p.n_slots) {
      if (lane == 0) set_dev_error(p.err, kDevBadArgs);
      slot = -1;
    }
  }

#pragma unroll 4
  for (int rb = r0; rb < r1; rb += kRows) {
    const int r = rb + lane / kLanes;
    const bool live = r < r1;
    const bool is_q = r < p.nq, is_v = r >= p.nq + p.nkv;
    const int h = is_q ? r : is_v ? r - p.nq - p.nkv : r - p.nq;
    const __nv_bfloat16* src = is_q   ? p.q + t * p.q_stride + (int64_t)h * HD
                               : is_v ? p.v + t * p.v_stride + (int64_t)h * HD
                                      : p.k + t * p.k_stride + (int64_t)h * HD;
    uint2 a = make_uint2(0, 0), b = make_uint2(0, 0);
    if (live) {
      a = *reinterpret_cast<const uint2*>(src + c0);
      b = *reinterpret_cast<const uint2*>(src + c1);
    }
    float x[8] = {bf16_lo(a.x), bf16_hi(a.x), bf16_lo(a.y), bf16_hi(a.y),
                  bf16_lo(b.x), bf16_hi(b.x), bf16_lo(b.y), bf16_hi(b.y)};
    if (turn && !is_v) {
      // (x1, x2) -> (x1 c - x2 s, x2 c + x1 s), each product rounded by itself: the same
      // bits whichever path rotates (a contracted form would depend on the compiler)
      const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {sn.x, sn.y, sn.z, sn.w};
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x1 = p.interleaved ? x[2 * i] : x[i], x2 = p.interleaved ? x[2 * i + 1] : x[i + 4];
        y[i] = __fsub_rn(__fmul_rn(x1, c[i]), __fmul_rn(x2, s[i]));
        y[i + 4] = __fadd_rn(__fmul_rn(x2, c[i]), __fmul_rn(x1, s[i]));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p.interleaved ? y[(i >> 1) + 4 * (i & 1)] : y[i];
    }
    if (is_q || FMT == kKvBf16) {
      a = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
      b = make_uint2(pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    }
    const int64_t row = slot < 0 ? 0 : ((((slot >> p.page_shift) * p.nkv + h) << p.page_shift) |
                                        (slot & ((1 << p.page_shift) - 1)));
    uint2 qv = make_uint2(0, 0);
    float scale = 0.f;
    if constexpr (FMT != kKvBf16) qv = quantise8<FMT, HD>(x, &scale);  // (all lanes: it shuffles)
    if (!live) continue;
    if (is_q) {
      __nv_bfloat16* o = p.q_out + t * p.q_out_stride + (int64_t)h * HD;
      *reinterpret_cast<uint2*>(o + c0) = a;
      *reinterpret_cast<uint2*>(o + c1) = b;
    } else if (slot >= 0) {
      uint8_t* base = is_v ? p.vc : p.kc;
      if constexpr (FMT == kKvBf16) {
        __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(base) + row * HD;
        *reinterpret_cast<uint2*>(o + c0) = a;
        *reinterpret_cast<uint2*>(o + c1) = b;
      } else {
        *reinterpret_cast<uint32_t*>(base + row * HD + c0) = qv.x;
        *reinterpret_cast<uint32_t*>(base + row * HD + c1) = qv.y;
        if (j == 0) (is_v ? p.vs : p.ks)[row] = scale;
      }
    }
  }
}

// ------------------------------------------------------------------- reading back
// value * scale, one rounding to bf16; a slot < 0 reads zeros
struct ReadParams {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int64_t* slots;
  int64_t tokens, n_slots;
  int nkv, page_shift;
  __nv_bfloat16 *k, *v;
  int64_t out_stride;
  int* err;
};

__device__ __forceinline__ float int8_at(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }
__device__ __forceinline__ float2 e4m3x2(uint32_t w, int i) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
  return __half22float2(__half2(h));
}

template <int FMT, int HD>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams p) {
  constexpr int kLanes = HD / 8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int j = (int)(i % kLanes);
  const int64_t row_i = i / kLanes;
  const int h2 = (int)(row_i % (2 * p.nkv));
  const int64_t t = row_i / (2 * p.nkv);
  if (t >= p.tokens) return;
  const bool is_v = h2 >= p.nkv;
  const int h = is_v ? h2 - p.nkv : h2;
  int64_t slot = p.slots[t];
  if (slot >= p.n_slots) {
    if (j == 0) set_dev_error(p.err, kDevBadArgs);
    slot = -1;
  }
  uint4 o = make_uint4(0, 0, 0, 0);
  if (slot >= 0) {
    const int64_t row = (((slot >> p.page_shift) * p.nkv + h) << p.page_shift) | (slot & ((1 << p.page_shift) - 1));
    const uint8_t* base = is_v ? p.vc : p.kc;
    if constexpr (FMT == kKvBf16) {
      o = *reinterpret_cast<const uint4*>(base + (row * HD + 8 * j) * 2);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(base + row * HD + 8 * j);
      const float s = (is_v ? p.vs : p.ks)[row];
      float x[8];
      if constexpr (FMT == kKvInt8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = int8_at(e < 4 ? w.x : w.y, e & 3);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = e4m3x2(e < 2 ? w.x : w.y, e & 1);
          x[2 * e] = f.x;
          x[2 * e + 1] = f.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= s;
      o = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                     pack_bf16x2(x[6], x[7]));
    }
  }
  __nv_bfloat16* dst = (is_v ? p.v : p.k) + t * p.out_stride + (int64_t)h * HD + 8 * j;
  *reinterpret_cast<uint4*>(dst) = o;
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
  if (c->pages > INT32_MAX || c->pages * c->kv_heads * c->page_size > INT32_MAX)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "pages * kv_heads * page_size must be below 2^31");
  return WX_OK;
}

static int check_rope(wx_ctx* ctx, const wx_rope* r, int head_dim, const int32_t* pos) {
  WX_CHECK_ARG(ctx, r && r->cos_t && r->sin_t && pos && r->positions > 0);
  WX_CHECK_ARG(ctx, r->rot > 0 && r->rot % 8 == 0 && r->rot <= head_dim);
  WX_CHECK_ARG(ctx, aligned16(r->cos_t) && aligned16(r->sin_t));
  return WX_OK;
}

static int launch_rows(wx_ctx* ctx, RowsParams& p, int fmt, int head_dim) {
  if (p.tokens == 0) return WX_OK;
  const int per_token = p.nq + 2 * p.nkv;
  const int rows = 256 / head_dim;  // rows of a warp at a time
  // Eight rows a warp reuse the token's table row and keep 4 loads in flight per lane; with few
  // tokens fewer rows a warp fill the SMs instead (a warp's rows follow one another).
  p.rows_per_warp = 8;
  while (p.rows_per_warp > rows &&
         p.tokens * ((per_token + p.rows_per_warp - 1) / p.rows_per_warp) < (int64_t)ctx->num_sms * 32)
    p.rows_per_warp /= 2;
  const int64_t warps = p.tokens * ((per_token + p.rows_per_warp - 1) / p.rows_per_warp);
  const int64_t blocks = (warps + 7) / 8;
  if (blocks > INT32_MAX) return set_error(ctx, WX_ERR_UNSUPPORTED, "too many tokens in one call");
  p.err = ctx->dev_err;
  ProfScope prof(ctx, kProfRow);
  const unsigned g = (unsigned)blocks;
  if (head_dim == 128) {
    if (fmt == kKvInt8) text_rows_kernel<kKvInt8, 128><<<g, 256, 0, ctx->stream>>>(p);
    else if (fmt == kKvE4m3) text_rows_kernel<kKvE4m3, 128><<<g, 256, 0, ctx->stream>>>(p);
    else text_rows_kernel<kKvBf16, 128><<<g, 256, 0, ctx->stream>>>(p);
  } else {
    if (fmt == kKvInt8) text_rows_kernel<kKvInt8, 64><<<g, 256, 0, ctx->stream>>>(p);
    else if (fmt == kKvE4m3) text_rows_kernel<kKvE4m3, 64><<<g, 256, 0, ctx->stream>>>(p);
    else text_rows_kernel<kKvBf16, 64><<<g, 256, 0, ctx->stream>>>(p);
  }
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

int wx_kv_read(wx_ctx* ctx, const wx_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out,
               int64_t out_stride) {
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
  const int64_t threads = tokens * 2 * cache->kv_heads * (cache->head_dim / 8);
  const int64_t blocks = (threads + 255) / 256;
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
