// wx_text_dev.cuh — device pieces shared by the text side's attention kernels (wx_text_attn.cu,
// wx_text_flash.cu): launch parameters, a sequence's bounds, 8-bit -> bf16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "wx_ptx.cuh"
#include "wx_text.h"

namespace wx {

// Which keys a row sees: those up to its place within the window (kPlainKeys), these and the
// sequence's first `sinks` (kSinkKeys), or a prefix common to all sequences and then its own
// sequence's up to its place (kPrefixKeys; kChunkKeys: the same in the rows kernel's form for short
// sequences). The attention kernels are compiled for each.
enum : int { kPlainKeys = 0, kSinkKeys = 1, kPrefixKeys = 2, kChunkKeys = 3 };

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
  int sinks;  // kSinkKeys: first keys that stay visible beside the window
  // kPrefixKeys
  int prefix;  // its keys,
  int front;   // in tiles of 128
  const int32_t* prefix_blocks;
  int64_t table_stride;
  int shared;  // text_flash: one walk over the prefix for the rows of all sequences (otherwise: each
               // sequence's items walk the prefix, then its own keys). Rows kernel: sequence 0 is that walk
  float* layer_o;     // sums of rows [layer][total_q * hq][hd], brought together by prefix_join_kernel
  int layers;
  float2* layer_ml;   // their maxima (base 2) and denominators
  int own_layer;      // rows kernel: of the sequences' own keys (kChunkKeys: of their first chunk)
  int chunk, chunks;  // kChunkKeys: keys of a unit, a layer each, at least, and units at most; 0: one layer
  int max_q;          // host: the caller's longest query length
  int ctas;           // kChunkKeys, host
  int after_walk;     // kChunkKeys, host: launched right behind the shared walk by text_flash
  size_t ws_reserved; // bytes of the workspace in use before the kernel's own
  float sl2;  // scale * log2(e): scores and maxima are kept in base 2
  float* part;              // split items: [2 * gridDim][16][hd] sums, then [..][16] maxima and denominators
  float* part_ml;
  int* counters;            // per item: pieces that have arrived (0 between launches)
  int64_t n_items;          // of them
  int* err;
};

// kChunkKeys: a sequence's keys go to `most` units at most, of whole steps of 16 and `chunk` keys at least.
__host__ __device__ inline int chunk_of(int chunk, int most, int lk) {
  const int even = (lk / most + 16) & ~15;  // (more than lk / most)
  return even > chunk ? even : chunk;
}
__host__ __device__ inline int chunks_of(int chunk, int most, int lk) {
  return lk > 0 ? (lk - 1) / chunk_of(chunk, most, lk) + 1 : 1;
}
// Layers that a walk over lk keys writes (chunk 0: a single one): what is joined is this many, no more. Room is made
// for those of every length up to `keys`: of some longer ones there are fewer, their chunks being rounded up to 16 keys.
__host__ __device__ inline int layers_of(int chunk, int most, int lk) { return chunk ? chunks_of(chunk, most, lk) : 1; }
__host__ __device__ inline int most_layers(int chunk, int most, int64_t keys) {
  return chunk && keys >= (int64_t)most * chunk ? most : layers_of(chunk, most, (int)keys);
}

// where K and V rows lie: `rows` rows of `cols` elements (strides in elements)
struct KvSource {
  const void *k, *v;
  uint64_t rows, cols, k_stride, v_stride;
  int format;
};

// attention for many query rows (wx_text_flash.cu)
int text_flash(wx_ctx* ctx, const TextAttnParams& p, int head_dim, const KvSource& kv, int keys = kPlainKeys);
// workspace that it takes beside layers, and the pieces (layers) of a shared walk over the prefix
size_t text_flash_ws(wx_ctx* ctx);
int text_flash_layers(wx_ctx* ctx, const TextAttnParams& p);
int64_t text_flash_walk_ctas(const TextAttnParams& p, int layers);

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

// whether a row with bounds [lo, hi) sees key j
// (kPrefixKeys: of its own sequence; a key of the prefix goes by -1)
template <int KEYS>
__device__ __forceinline__ bool key_seen(const TextAttnParams& p, int j, int lo, int hi) {
  if constexpr (KEYS >= kPrefixKeys) return j < hi;
  return j < hi && (j >= lo || (KEYS == kSinkKeys && j < p.sinks));
}
// Between the first keys and the window lie keys that no row of an item (of a call, in the rows kernel)
// sees. Kernels walk a sequence's keys without them: of `first` units before the first row's window,
// those that hold first keys stay, and unit u stands for u + gap from there on.
struct KeyGap {
  int first, gap;
  __device__ __forceinline__ int operator()(int u) const { return u < first ? u : u + gap; }
};
template <int KEYS>
__device__ __forceinline__ KeyGap key_gap(const TextAttnParams& p, int first, int unit) {
  if constexpr (KEYS != kSinkKeys) return KeyGap{0, 0};
  const int seen = (int)min64(first, ((int64_t)p.sinks + unit - 1) / unit);
  return KeyGap{seen, first - seen};
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
// Dependent launches: a kernel lets the next one on its stream begin (where that was launched for it), and
// waits for the one before to be complete and its memory visible.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// ------------------------------------------------------------------ partial sums of rows, joined
// Layer i of row r holds o = sum 2^(s - m) v at (i * rows + r), and (m, l) beside it (base 2; l 0: the layer's
// keys are not seen, its sums may be anything). A warp joins R neighbouring rows, in the order of the layers:
//   M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.
// Bound by the layers' bytes, if enough of them are in flight: eight rows' loads go out at once, of eight layers where
// rows are few (a row a warp), and of two layers where there are many: the rows of a warp belong to one token, so
// that what is found out about its sequence serves them all. Whole calls with a row : four rows a warp: 2,048 rows of
// up to 15 layers 41.4 : 43.5 us, 8,192 of up to 8 279 : 276, 33,852 of 3 236 : 221.
template <int HD, int R>
__device__ __forceinline__ void join_rows(const float* o_base, const float2* ml_base, int64_t rows, int64_t row0, int n,
                                          int layers, __nv_bfloat16* out, float* lse) {
  constexpr int kPer = HD / 32, kLayers = 8 / R;
  const int lane = threadIdx.x & 31, mine = lane % R;  // lane: layer c + lane / R of row row0 + mine
  auto ml_of = [&](int c) {
    const int i = c + lane / R;
    return i < layers && mine < n ? __ldcg(ml_base + i * rows + row0 + mine) : make_float2(-INFINITY, 0.f);
  };
  float M = -INFINITY, L = 0.f;
  for (int c = 0; c < layers; c += 32 / R) {
    const float2 ml = ml_of(c);
    M = fmaxf(M, ml.y != 0.f ? ml.x : -INFINITY);
  }
#pragma unroll
  for (int d = R; d < 32; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  float o[R][kPer] = {};
  for (int c = 0; c < layers; c += 32 / R) {
    const float2 ml = ml_of(c);
    const float f = ml.y != 0.f ? exp2_approx(ml.x - M) : 0.f;
    const uint32_t seen = __ballot_sync(0xffffffffu, ml.y != 0.f);
    if (ml.y != 0.f) L += ml.y * f;
#pragma unroll 1
    for (int i = 0; i < 32 / R && c + i < layers; i += kLayers) {
      float x[kLayers][R][kPer];
#pragma unroll
      for (int q = 0; q < kLayers; ++q)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float* src = o_base + (min(c + i + q, layers - 1) * rows + row0 + min(r, n - 1)) * HD + lane * kPer;
          if constexpr (kPer == 4) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(src));
            x[q][r][0] = y.x, x[q][r][1] = y.y, x[q][r][2] = y.z, x[q][r][3] = y.w;
          } else {
            const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
            x[q][r][0] = y.x, x[q][r][1] = y.y;
          }
        }
#pragma unroll
      for (int q = 0; q < kLayers; ++q)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int from = (i + q) * R + r;
          const float w = __shfl_sync(0xffffffffu, f, from);
          if (seen >> from & 1u)
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[r][e] += x[q][r][e] * w;
        }
    }
  }
#pragma unroll
  for (int d = R; d < 32; d <<= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float l = __shfl_sync(0xffffffffu, L, r);
    if (r >= n) break;
    const float inv = l == 0.f ? 0.f : __fdividef(1.0f, l);
    uint32_t* dst = reinterpret_cast<uint32_t*>(out + r * HD + lane * kPer);
    if constexpr (kPer == 4)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_bf16x2(o[r][0] * inv, o[r][1] * inv), pack_bf16x2(o[r][2] * inv, o[r][3] * inv));
    else dst[0] = pack_bf16x2(o[r][0] * inv, o[r][1] * inv);
  }
  if (lse && lane < n) lse[lane] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.69314718055994531f;
}
// the warp's token and first head: a token's heads in groups of R
template <int R>
__device__ __forceinline__ int64_t join_token(const TextAttnParams& p, int& head) {
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int groups = (p.hq + R - 1) / R;
  const int64_t token = at / groups;
  head = (int)(at - token * groups) * R;
  return token;
}
inline unsigned join_blocks(const TextAttnParams& p, int R) {
  return (unsigned)((p.total_q * ((p.hq + R - 1) / R) + 7) / 8);
}
// rows of a warp: four, where that leaves every SM twelve warps
inline bool join_by_fours(const wx_ctx* ctx, const TextAttnParams& p) { return p.total_q * p.hq >= (int64_t)ctx->num_sms * 48; }
// last sequence that begins at or before a token
__device__ __forceinline__ int seq_of_token(const TextAttnParams& p, int64_t token) {
  int b = 0;
  for (int n = p.batch; n > 1;) {
    const int half = n / 2;
    if (p.cu_q[b + half] <= token) b += half;
    n -= half;
  }
  return b;
}

}  // namespace wx
