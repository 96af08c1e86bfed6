// wx_text_dev.cuh — device pieces shared by the text side's attention kernels (wx_text_attn.cu,
// wx_text_flash.cu): launch parameters, a sequence's bounds, 8-bit -> bf16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "wx_ptx.cuh"
#include "wx_text.h"

namespace wx {

struct TextAttnParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  float* lse;
  const int32_t* cu_q;
  const int32_t* cu_k;      // contiguous K/V (block_table == nullptr)
  const int32_t* kv_lens;   // paged K/V
  const int32_t* block_table;
  int64_t blocks_per_seq;
  const float *ks, *vs;     // scales of an 8-bit cache
  int64_t pages;
  int page_shift;
  int batch, hq, hkv, group;
  int64_t total_q, total_k;
  int causal, window;
  float sl2;  // scale * log2(e): scores and maxima are kept in base 2
  float* part;              // split items: [2 * gridDim][16][hd] sums, then [..][16] maxima and denominators
  float* part_ml;
  int* counters;            // per item: pieces that have arrived (0 between launches)
  int64_t n_items;          // of them
  int* err;
};

// where K and V rows lie: `rows` rows of `cols` elements (strides in elements)
struct KvSource {
  const void *k, *v;
  uint64_t rows, cols, k_stride, v_stride;
  int format;
};

// attention for many query rows (wx_text_flash.cu)
int text_flash(wx_ctx* ctx, const TextAttnParams& p, int head_dim, const KvSource& kv);

// One sequence as the kernels see it; lengths and offsets from the device are clamped to the
// buffers, so that wrong ones give wrong rows and an error word but no access outside.
struct Seq {
  int64_t q0, k0;
  int lq, lk;
};

__device__ __forceinline__ Seq load_seq(const TextAttnParams& p, int b) {
  Seq s;
  const int64_t a = p.cu_q[b], e = p.cu_q[b + 1];
  s.q0 = min64(max64(a, 0), p.total_q);
  const int64_t q1 = min64(max64(e, s.q0), p.total_q);
  s.lq = (int)(q1 - s.q0);
  bool bad = s.q0 != a || q1 != e;
  if (p.block_table) {
    const int64_t n = p.kv_lens[b], cap = p.blocks_per_seq << p.page_shift;
    s.k0 = 0;
    s.lk = (int)min64(max64(n, 0), cap);
    bad |= s.lk != n;
  } else {
    const int64_t c = p.cu_k[b], d = p.cu_k[b + 1];
    s.k0 = min64(max64(c, 0), p.total_k);
    const int64_t k1 = min64(max64(d, s.k0), p.total_k);
    s.lk = (int)(k1 - s.k0);
    bad |= s.k0 != c || k1 != d;
  }
  if (bad) set_dev_error(p.err, kDevBadArgs);
  return s;
}

// Keys [lo, hi) that query token `tok` of a sequence sees. In 32 bits for every length and window:
// tok - lq is above -2^31 and below 0, and a window is taken off a number that is not below 0 (off a
// negative one, one near 2^31 would wrap to a bound beyond every key).
__device__ __forceinline__ int key_hi(const TextAttnParams& p, const Seq& s, int tok) {
  return p.causal ? max(0, min(s.lk, tok - s.lq + s.lk + 1)) : s.lk;
}
__device__ __forceinline__ int key_lo(const TextAttnParams& p, const Seq& s, int tok) {
  return p.window > 0 ? max(0, max(0, tok - s.lq + s.lk + 1) - p.window) : 0;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ 8-bit -> bf16
// Two stored bytes -> a bf16 pair, exactly, in units of kByteUnit. int8: byte + 128 as the bits of a
// bf16 is (byte + 128) * 2^-133 (subnormal or the first binade: one line), so one fused product with 2^120
// and sum gives byte * 2^-13. e4m3: through f16 and fp32 in four conversions a pair, which keep NaN; shifting
// the bits into a bf16 took five instructions and made numbers of the NaN codes (decoding over 65,537 keys,
// 64 / 8 heads of 128: 41 us against 45).
template <int FMT>
constexpr float kByteUnit = FMT == kKvInt8 ? 8192.f : 1.f;
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// byte `lo` of {b:a} to the low half, byte `hi` to the high half
template <int FMT>
__device__ __forceinline__ uint32_t bytes_to_bf16x2(uint32_t a, uint32_t b, int lo, int hi) {
  if constexpr (FMT == kKvInt8) {
    a ^= 0x80808080u;
    // (bytes of one word are put between zeros at once)
    const uint32_t w = hi < 4 ? __byte_perm(a, 0u, (uint32_t)(0x4040 | lo | hi << 8))
                              : __byte_perm(a, b ^ 0x80808080u, (uint32_t)(lo | hi << 8)) & 0x00ff00ffu;
    return fma_bf16x2(w, 0x7b807b80u, 0xbc80bc80u);  // * 2^120 - 2^-6
  } else {
    const uint32_t w = lo == 0 && hi == 1   ? a
                       : lo == 2 && hi == 3 ? a >> 16
                                            : __byte_perm(a, b, (uint32_t)(lo | hi << 4));
    const float2 x = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
    return pack_bf16x2(x.x, x.y);
  }
}

// NaN codes (0x7f, 0xff) of an e4m3 cache: kv_append writes none, a cache that was filled elsewhere may hold
// some. They expand to NaN, as they should, but for a value that only some of the rows at work see.
// Bit 7 of each byte that is one (the low seven bits of the others do not carry into it).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// the same as one bit for each of the four bytes
__device__ __forceinline__ uint32_t nan_code_mask(uint32_t w) {
  const uint32_t b = nan_codes(w) >> 7;
  return (b | b >> 7 | b >> 14 | b >> 21) & 15u;
}
// the word with zeros in their place
__device__ __forceinline__ uint32_t without_nan_codes(uint32_t w) { return w & ~((nan_codes(w) >> 7) * 255u); }

// stored bytes 2 h, 2 h + 1 of a word, times a scale, rounded to a bf16 pair
template <int FMT>
__device__ __forceinline__ uint32_t bytes_times(uint32_t w, int h, float scale) {
  float2 x;
  if constexpr (FMT == kKvInt8) {  // 2^23 + (byte + 128) is an fp32 number whose low byte is byte + 128
    w ^= 0x80808080u;
    x = make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, h ? 0x7442 : 0x7440)),
                    __uint_as_float(__byte_perm(w, 0x4b000000u, h ? 0x7443 : 0x7441)));
    x = __fadd2_rn(x, make_float2(-8388736.f, -8388736.f));
  } else {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
    x = __half22float2(__half2(r));
  }
  x = __fmul2_rn(x, make_float2(scale, scale));
  return pack_bf16x2(x.x, x.y);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

}  // namespace wx
