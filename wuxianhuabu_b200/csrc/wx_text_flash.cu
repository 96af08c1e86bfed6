// wx_text_flash.cu — attention of the text side for many query rows: whole packed prompts, and
// chunks of new tokens over the paged cache.
//
// Mathematics: the query rows of one K/V head are flattened to r = token * G + g, so the rows of
// 2 * floor(128 / G) tokens share one walk over the keys they may see; each row keeps a running maximum
// and denominator, o = sum 2^(s - m) v is rescaled only when the maximum has grown by more than
// 2^8, and the weights are rounded to bf16 for the second product (the denominator is not).
//
// One persistent CTA per SM works on two slots of 128 rows at once, so that one slot's
// exponentials overlap the other's products. Per 128-key tile a slot needs S = Q K^T and
// O += P V: 2 x 128 x 128 x HD products; at HD 128 that is 1024 tensor cycles per slot, as many
// as its 128 x 128 exponentials take on the MUFU pipe.
//   TMEM (512 columns): S/P of slot A [0,128), of B [128,256), O of A from 256, of B from 384;
//   P overwrites the first half of its S as packed bf16.
//   Warp 0: TMA producer of K and V. Warps 1 / 2: MMA issuer of slot A / B. Warp 3: finds the
//   items and mends masked V tiles. Warps 4-7 / 8-11: softmax and epilogue of slot A / B (thread
//   r owns row r); one of their threads fetches the next item's Q as soon as the last S is done.
//   8-bit cache: warp 0 brings raw rows and scales, warps 12-15 turn them into bf16 tiles (exact:
//   the key's scale multiplies its scores, the value's scale its weights, both in fp32).
//
// Measured (caches flushed from L2): packed causal prompts of 9001 + 1 + 5003 + 2380 tokens, 32 / 8
// heads of 128: 785 us in single calls (1.17 PFLOP/s of useful work), 920 in a row under the power
// cap; 4096 + 1117 tokens, 16 heads of 64, window 1024: 64 us; 1024 + 300 tokens over 16,384 + 9,999
// cached keys, 32 / 8 heads of 128: 360 us at bf16, 550 at e4m3. Tensor pipe 51 % busy on a prompt
// of 4096 tokens, 28 % on an e4m3 cache. What bounds it is a slot's chain from one S to the next (S,
// its maxima, the exponentials in their turn, the issue of P V and S): some 3,700 cycles at bf16 against 2,048
// tensor cycles for both slots; on 8-bit caches 5,400, the four conversion warps being nearly as long.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "wx_text_dev.cuh"

namespace wx {

constexpr int kTfVStages = 2;
constexpr int kTfRaw = 3;       // 8-bit: raw half tiles (64 keys) in flight
constexpr int kTfScales = 4;    // 8-bit: tiles of scales kept
constexpr int kTfItems = 2;     // item slots: the one at work and the next
constexpr int kTfChunk = 128 * 128;  // one 64-column SW128 chunk of a 128-row tile
constexpr int kTfWaves = 3;          // pieces for each SM below which items are cut up
constexpr int kTfMinTiles = 8;       // tiles of a piece of an item: its start and end cost one or two
constexpr int64_t kTfL2 = int64_t(48) << 20;
// V rows with non-finite values remembered per item: every row of its masked tiles (an item's 256 tokens
// end, and where a window cuts begin, in up to three tiles each)
constexpr int kTfBadRows = 6 * 128;
constexpr int kTfBadWords = 9;       // key, columns with +infinity or NaN, columns with -infinity or NaN

template <int FMT, int HD>
struct TfGeom {
  static constexpr bool kWide = FMT != kKvBf16;
  static constexpr int kThreads = kWide ? 512 : 384;
  static constexpr int kKStages = kWide ? 2 : 3;
  // quarters of P that are handed over first, together; each hand-over waits for its stores, and a
  // tile's last products should be few (9001 + 5003 + 2380 tokens: 1: 808, 2: 795, 3: 800, 4: 840 us)
  static constexpr int kFirstP = kWide ? 1 : 2;
  // registers of the control (and conversion) warps and of the softmax warps after setmaxnreg
  static constexpr int kRegsLow = kWide ? 104 : 72, kRegsHigh = kWide ? 152 : 216;
  static constexpr int kRegsUsed = kRegsLow * (kThreads - 256) + kRegsHigh * 256;
  static_assert(kRegsUsed <= 65536 / kThreads / 8 * 8 * kThreads, "register split exceeds the launch");
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kChunks = HD / 64;
  static constexpr int kRawBytes = 64 * HD;
  static constexpr int kRawOff = (2 + kKStages + kTfVStages) * kTile;
  static constexpr int kScaleOff = kRawOff + (kWide ? kTfRaw * kRawBytes : 0);  // [tile][k, v][key]
  static constexpr int kBarOff = kScaleOff + (kWide ? kTfScales * 1024 : 0);
  static constexpr int kItemOff = kBarOff + 512;
  static constexpr int kSmem = kItemOff + kTfItems * 128 + 1024;
};

// One item: the query heads of one K/V head for 2 * TT tokens of one sequence
struct TfItem {
  int valid;
  int b, h, tok0;  // tok0: first token
  int lq, lk, q0, k0;
  int a0, a1, b0, b1;    // key tiles [a0, a1) of slot A, [b0, b1) of slot B
  int free_hi, free_lo;  // tiles inside [free_lo, free_hi) are unmasked for every row
  int bad;               // V rows with non-finite values (8-bit: NaN codes) found in masked tiles
  int piece, pieces;     // this part of the item's key tiles, and how many it was cut into
  __device__ int lo(int X) const { return X ? b0 : a0; }
  __device__ int hi(int X) const { return X ? b1 : a1; }
  __device__ int first() const { return a1 <= a0 ? b0 : b1 <= b0 ? a0 : min(a0, b0); }
  __device__ int last() const { return max(first(), max(a1 > a0 ? a1 : 0, b1 > b0 ? b1 : 0)); }
  __device__ bool masked(int t) const { return t * 128 + 128 > free_hi || t * 128 < free_lo; }
};

enum : int {
  kBTfItemFull = 0,                       // [items]
  kBTfItemEmpty = kBTfItemFull + kTfItems,  // [items] count 11 (8-bit: 15): every other warp is done with it
  kBTfQFull = kBTfItemEmpty + kTfItems,   // [2]
  kBTfKFull = kBTfQFull + 2,              // [3] (8-bit: count 4, the conversion warps)
  kBTfKEmpty = kBTfKFull + 3,             // [3] count 2: both slots
  kBTfVRaw = kBTfKEmpty + 3,              // [V stages] a masked tile has landed
  kBTfVFull = kBTfVRaw + kTfVStages,      // [V stages] count 2: landed, and mended where masked (8-bit: 4)
  kBTfVEmpty = kBTfVFull + kTfVStages,    // count 2
  kBTfSFull = kBTfVEmpty + kTfVStages,    // [2]
  kBTfPFull = kBTfSFull + 2,              // [2][4] count 4
  kBTfOFull = kBTfPFull + 8,              // [2]
  kBTfOEmpty = kBTfOFull + 2,             // [2] count 4: the epilogue has read O
  kBTfTurn = kBTfOEmpty + 2,              // [2] count 4: a slot's exponentials of a tile are issued
  kBTfDrain = kBTfTurn + 2,               // [2]
  kBTfRawFull = kBTfDrain + 2,            // [raw] 8-bit rows have landed
  kBTfRawEmpty = kBTfRawFull + kTfRaw,    // [raw] count 4
  kBTfScale = kBTfRawEmpty + kTfRaw,      // [scales] a tile's scales have landed
  kBTfCount = kBTfScale + kTfScales
};
static_assert(kBTfCount * 8 + 32 <= 512, "barriers overlap the items");

__device__ __forceinline__ float max3_f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// true in one lane of the (converged) warp, the same each time
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 32 lanes x 16 columns of 32-bit: thread i of the warp gets lane (base + i), 16 columns
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The shape of a matrix fragment, 16 lanes by 8 columns of 32 bits a repeat: thread (g, t) =
// (lane / 4, lane % 4) holds columns 2t and 2t + 1 of lane g (first two registers) and of lane g + 8.
__device__ __forceinline__ void tmem_ld_frag4(uint32_t taddr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_frag4(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
               : "memory");
}
// waits for the thread's loads, of which v is one: nothing that uses v moves before it
__device__ __forceinline__ void tmem_wait_ld32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])::"memory");
}
// 16 lanes by 4 columns a repeat: column t of lane g, then of lane g + 8
__device__ __forceinline__ void tmem_st_half4(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Zeroes the non-finite values of row r of a V tile and notes their columns and signs in `entry`.
template <int HD>
__device__ __noinline__ void remember_row(uint32_t row, int r, int key, uint32_t* entry) {
  uint32_t plus[4] = {0, 0, 0, 0}, minus[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int d = 0; d < HD; ++d) {
    const uint32_t at = row + (d >> 6) * kTfChunk + ((((d >> 3) & 7) ^ (r & 7)) << 4) + (d & 7) * 2;
    const uint32_t x = lds_u16(at);
    if ((x & 0x7f80u) != 0x7f80u) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t bit = (d >> 5) == e ? 1u << (d & 31) : 0u;
      if (x != 0xff80u) plus[e] |= bit;
      if (x != 0x7f80u) minus[e] |= bit;
    }
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)0) : "memory");
  }
  if (!entry) return;
  entry[0] = (uint32_t)key;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    entry[1 + e] = plus[e];
    entry[5 + e] = minus[e];
  }
}

// The same for the NaN codes of 64 raw e4m3 rows from `key0`, before 128 threads expand them: each thread
// looks at the 16 bytes that it will expand itself (HD / 16 lanes a row), zeroes the codes there, and
// their columns go to a new entry of the item's list, one a row. Behind the last key nobody sees them.
template <int HD>
__device__ __noinline__ void remember_codes(uint32_t raw, int tid, int key0, int lk, int& bad, uint32_t* list) {
  constexpr int kLanes = HD / 16;
  const int c = tid % kLanes;
#pragma unroll 1
  for (int u = tid; u < 64 * kLanes; u += 128) {
    const uint32_t at = raw + (uint32_t)u * 16;
    const uint4 w = lds128(at);
    const uint32_t bits =
        nan_code_mask(w.x) | nan_code_mask(w.y) << 4 | nan_code_mask(w.z) << 8 | nan_code_mask(w.w) << 12;
    if (!__any_sync(0xffffffffu, bits != 0)) continue;
    sts128(at, make_uint4(without_nan_codes(w.x), without_nan_codes(w.y), without_nan_codes(w.z),
                          without_nan_codes(w.w)));
    uint32_t mask[4], any = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mask[e] = (c >> 1) == e ? bits << (16 * (c & 1)) : 0u;
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) mask[e] |= __shfl_xor_sync(0xffffffffu, mask[e], o);
      any |= mask[e];
    }
    const int key = key0 + u / kLanes;
    if (c == 0 && any && key < lk) {
      const int slot = atomicAdd(&bad, 1);
      if (slot < kTfBadRows) {
        uint32_t* entry = list + slot * kTfBadWords;
        entry[0] = (uint32_t)key;
#pragma unroll
        for (int e = 0; e < 4; ++e) entry[1 + e] = entry[5 + e] = mask[e];
      }
      __threadfence_block();
    }
    __syncwarp();
    fence_proxy_async_smem();  // the rows that are copied here next come after these zeros
  }
}

__device__ __forceinline__ float2 lds_f2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}

struct TfParams {
  TextAttnParams a;
  int tt;              // tokens of a slot: floor(128 / G)
  int box;             // rows of a K/V box: 128, or a page where pages are smaller
  int* next;           // [2] items handed out, CTAs that have finished (0, 0 between launches)
  uint32_t* bad_rows;  // [CTA][kTfItems][kTfBadRows][kTfBadWords]
  const uint8_t *k8, *v8;  // rows of an 8-bit cache
  int splits;              // at most this many pieces of an item
  float* part;             // [splits][total_q * hq][HD] sums of the pieces' rows (items cut up only)
  float2* part_ml;         // [splits][total_q * hq] maximum (base 2) and denominator
};

// Key tiles that tokens [k0, k0 + tt) of a sequence see: [x.x, x.y)
__device__ __forceinline__ int2 slot_tiles(const TextAttnParams& p, const Seq& s, int k0, int tt) {
  const int k1 = min(s.lq, k0 + tt);
  if (k0 >= k1) return make_int2(0, 0);
  const int hi = key_hi(p, s, k1 - 1), lo = key_lo(p, s, k0);
  return hi > lo ? make_int2(lo >> 7, (hi + 127) >> 7) : make_int2(0, 0);
}
// The item's tiles [first, last) and the pieces that they are cut into, of at least kTfMinTiles
__device__ __forceinline__ void cut_item(int2 a, int2 b, int splits, int& first, int& last, int& pieces) {
  first = a.y <= a.x ? b.x : b.y <= b.x ? a.x : min(a.x, b.x);
  last = max(first, max(a.y > a.x ? a.y : 0, b.y > b.x ? b.y : 0));
  pieces = min(splits, max(1, (last - first) / kTfMinTiles));
}

template <int FMT, int HD>
__global__ void __launch_bounds__(TfGeom<FMT, HD>::kThreads, 1)
    text_flash_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, TfParams tp) {
  using G = TfGeom<FMT, HD>;
  constexpr bool kW = G::kWide;
  constexpr int kTile = G::kTile, kKStages = G::kKStages;
  const TextAttnParams& p = tp.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  auto sQ = [&](int X) { return sbase + (uint32_t)X * kTile; };
  auto sK = [&](int s) { return sbase + (uint32_t)(2 + s) * kTile; };
  auto sV = [&](int s) { return sbase + (uint32_t)(2 + kKStages + s) * kTile; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kBarOff);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBTfCount);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  TfItem* items = reinterpret_cast<TfItem*>(smem + G::kItemOff);
  static_assert(sizeof(TfItem) <= 128, "item slots");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kBTfCount; ++i) {
      uint32_t c = 1;
      if (i >= kBTfItemEmpty && i < kBTfItemEmpty + kTfItems) c = kW ? 15 : 11;
      if (i >= kBTfKFull && i < kBTfKEmpty && kW) c = 4;
      if (i >= kBTfKEmpty && i < kBTfVRaw) c = 2;
      if (i >= kBTfVFull && i < kBTfVEmpty) c = kW ? 4 : 2;
      if (i >= kBTfVEmpty && i < kBTfSFull) c = 2;
      if ((i >= kBTfPFull && i < kBTfOFull) || (i >= kBTfOEmpty && i < kBTfDrain)) c = 4;
      if (i >= kBTfRawEmpty && i < kBTfScale) c = 4;
      mbar_init(bar(i), c);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // item n, in shared memory until this warp drops it (nullptr: no more items, or a wait ran out)
  auto take_item = [&](int n) -> const TfItem* {
    if (!mbar_wait(bar(kBTfItemFull + n % kTfItems), (n / kTfItems) & 1, p.err, kDevTimeoutOther, abort_flag))
      return nullptr;
    const TfItem* it = items + n % kTfItems;
    return it->valid ? it : nullptr;
  };
  auto drop_item = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kBTfItemEmpty + n % kTfItems));
  };

  if (warp == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kRegsLow));
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    uint32_t nk = 0, nv = 0;  // tiles loaded
    const int boxes = 128 / tp.box;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const TfItem* at = take_item(n);
      if (!at) break;
      const TfItem& it = *at;
      const int t0 = it.first(), t1 = it.last();
      int ids = 0, ids_from = -1;  // block entries of 32 consecutive boxes, one per lane
      // block entry of box b of the sequence (b0: the tile's first box)
      auto page_of = [&](int b0, int bx) -> int {
        if (ids_from < 0 || b0 < ids_from || b0 + boxes > ids_from + 32) {
          ids_from = b0;
          const int64_t j = (int64_t)(b0 + lane) * tp.box;
          ids = 0;
          if (j < it.lk) {
            ids = p.block_table[it.b * p.blocks_per_seq + (j >> p.page_shift)];
            if (ids < 0 || ids >= p.pages) {
              set_dev_error(p.err, kDevBadArgs);
              ids = 0;
            }
          }
        }
        return __shfl_sync(0xffffffffu, ids, (b0 - ids_from + bx) & 31);
      };
      auto cache_row = [&](int page, int j) -> int64_t {
        return (((int64_t)page * p.hkv + it.h) << p.page_shift) | (j & ((1 << p.page_shift) - 1));
      };
      // 8-bit: a tile in two halves of 64 raw rows, its scales with the keys; rows past the
      // sequence's last key are not loaded (any byte expands to a finite value or, in K, NaN: masked)
      auto load_raw = [&](bool is_k, int t) -> bool {
        const int per_half = 64 / tp.box;
        const int page = page_of(t * boxes, lane % boxes);
        const int nb = min(boxes, (it.lk - t * 128 + tp.box - 1) / tp.box);
        int64_t row = cache_row(page, t * 128 + (lane % boxes) * tp.box);
        // (the copy's bytes are waited for: it reads the first rows instead)
        if (lane < nb && !WX_IN_BOUNDS(p.err, row >= 0 && row + tp.box <= (p.pages * p.hkv) << p.page_shift)) row = 0;
        if (is_k) {
          const uint32_t sc = nk % kTfScales, full = bar(kBTfScale + sc);
          const uint32_t dst = sbase + G::kScaleOff + sc * 1024 + (uint32_t)lane * tp.box * 4;
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(nb * tp.box * 8));
          __syncwarp();
          if (lane < nb) {
            bulk_load(dst, p.ks + row, (uint32_t)tp.box * 4, full);
            bulk_load(dst + 512, p.vs + row, (uint32_t)tp.box * 4, full);
          }
          ++nk;
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half, ++nv) {  // (nv counts raw halves here)
          const uint32_t s = nv % kTfRaw;
          if (!mbar_wait(bar(kBTfRawEmpty + s), ((nv / kTfRaw) & 1) ^ 1u, p.err, kDevTimeoutEmpty, abort_flag)) return false;
          const int n = max(0, min(per_half, nb - half * per_half)), bx = lane - half * per_half;
          if (lane == 0) mbar_arrive_expect_tx(bar(kBTfRawFull + s), (uint32_t)(n * tp.box * HD));
          __syncwarp();
          if (bx >= 0 && bx < n)
            bulk_load(sbase + G::kRawOff + s * G::kRawBytes + (uint32_t)(bx * tp.box * HD),
                      (is_k ? tp.k8 : tp.v8) + row * HD, (uint32_t)(tp.box * HD), bar(kBTfRawFull + s));
        }
        return true;
      };
      auto load = [&](bool is_k, int t) -> bool {
        if constexpr (kW) return load_raw(is_k, t);
        const uint32_t cnt = is_k ? nk : nv;
        const int ns = is_k ? kKStages : kTfVStages;
        const uint32_t s = cnt % ns, par = ((cnt / ns) & 1) ^ 1u;
        if (!mbar_wait(bar((is_k ? kBTfKEmpty : kBTfVEmpty) + s), par, p.err, kDevTimeoutEmpty, abort_flag)) return false;
        const bool mend = !is_k && it.masked(t);
        const uint32_t full = bar((is_k ? kBTfKFull : mend ? kBTfVRaw : kBTfVFull) + s);
        const uint32_t dst = is_k ? sK(s) : sV(s);
        const CUtensorMap* tm = is_k ? &tmK : &tmV;
        // boxes past the sequence's last key are not loaded (no page stands there)
        const int nb = p.block_table ? min(boxes, (it.lk - t * 128 + tp.box - 1) / tp.box) : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(full, (uint32_t)(nb * tp.box * HD * 2));
          if (!is_k) mbar_arrive(bar(kBTfVFull + s));
        }
        __syncwarp();
        if (!p.block_table) {
          if (lane < G::kChunks) tma_load_2d(dst + lane * kTfChunk, tm, full, it.h * HD + lane * 64, it.k0 + t * 128);
        } else {
          const int bx = lane / G::kChunks, ch = lane % G::kChunks;
          const int page = page_of(t * boxes, bx);
          if (bx < nb) {
            const int row = (int)cache_row(page, t * 128 + bx * tp.box);
            tma_load_2d(dst + ch * kTfChunk + bx * tp.box * 128, tm, full, ch * 64, row);
          }
        }
        if (is_k) ++nk; else ++nv;
        return true;
      };
      // K two tiles ahead of V: K0 K1 V0 K2 V1 ...
#pragma unroll 1
      for (int i = 0; i < 2 * (t1 - t0) && ok; ++i) {
        const int tiles = t1 - t0;
        const bool tail = i >= 2 * tiles - 1;  // (the last two are both V; a single tile is K0 V0)
        const bool is_k = i < 2 ? (i == 0 || tiles > 1) : !tail && (i & 1);
        ok = load(is_k, t0 + (is_k ? (i < 2 ? i : (i + 1) / 2) : tail ? tiles - 1 : (i - 1) / 2));
      }
      drop_item(n);
    }
    // Copies still in flight must land before the CTA ends. On the regular path every tile was
    // consumed; after a wait that ran out, give them the time of one more bounded wait.
    if (!ok || *abort_flag) {
      if (lane == 0) {
        const uint64_t from = globaltimer_ns();
        while (globaltimer_ns() - from < 2000000ull) {}
      }
    }
  } else if (warp == 1 || warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kRegsLow));
    // ------------------------------------------------------------ MMA issuer of slot X
    const int X = __shfl_sync(0xffffffffu, warp, 0) - 1;
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, false, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(128, HD, false, true);  // P from TMEM, V MN-major
    const uint32_t tS = tmem + (uint32_t)(X * 128);
    const uint32_t tO = tmem + 256 + (uint32_t)(X * 128);
    const uint64_t dq = smem_desc_sw128(sQ(X), 16, 1024);
    uint32_t kv = 0;    // tiles of all items before this one (K and V alike)
    uint32_t mine = 0;  // tiles of this slot so far
    uint32_t n_o = 0;   // items in which this slot had tiles
    bool ok = true, issued = false;
    // The whole warp walks the tiles, one elected lane issues, from descriptors in uniform registers
    // (long prompts 793 -> 784 us against lane 0 walking alone).
    auto wait = [&](int which, uint32_t parity, int code) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar(which), parity, p.err, code, abort_flag));
    };
    for (int n = 0; ok; ++n) {
      const TfItem* at = take_item(n);
      if (!__all_sync(0xffffffffu, at != nullptr)) break;
      const TfItem& it = *at;
      const int t0 = it.first(), t1 = it.last();
      const bool any = it.hi(X) > it.lo(X);
      const int a0 = any ? it.lo(X) : t1, a1 = any ? it.hi(X) : t1;
      if (any) ok = wait(kBTfQFull + X, n_o & 1, kDevTimeoutSoftmax);
      // step t: O += P(t) V(t), then S(t + 1); a tile that only the other slot works on is
      // just given back
#pragma unroll 1
      for (int t = t0 - 1; t < t1 && ok; ++t) {
        // V(t) and K(t+1) are waited for before P(t): PV(t) and S(t+1) then go out back to back
        const uint32_t cv = kv + (uint32_t)(t - t0), ck = cv + 1;
        const uint32_t sv = cv % kTfVStages, sk = ck % kKStages;
        if (t >= t0) ok = wait(kBTfVFull + sv, (cv / kTfVStages) & 1, kDevTimeoutFull);
        if (ok && t + 1 < t1) ok = wait(kBTfKFull + sk, (ck / kKStages) & 1, kDevTimeoutFull);
        // the first product of an item overwrites O: the last epilogue must have read it
        if (ok && t == a0 && n_o > 0) ok = wait(kBTfOEmpty + X, (n_o - 1) & 1, kDevTimeoutSoftmax);
        if (!ok) break;
        if (t >= a0 && t < a1) {
          const uint64_t dv = smem_desc_sw128(sV(sv), kTfChunk, 1024);
#pragma unroll
          for (int part = 0; part < 4; ++part) {  // (the first kFirstP quarters come together)
            const int full = part < G::kFirstP ? G::kFirstP - 1 : part;
            if ((part == 0 || part >= G::kFirstP) &&
                !wait(kBTfPFull + X * 4 + full, (mine + (uint32_t)(t - a0)) & 1, kDevTimeoutSoftmax)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k2 = 0; k2 < 2; ++k2) {
                const int kk = part * 2 + k2;
                umma_bf16_ts(tO, tS + kk * 8, dv + (uint64_t)(kk * (2048 >> 4)), idesc_o, (t > a0 || kk > 0) ? 1u : 0u);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (elect_one()) {
            umma_commit(bar(kBTfVEmpty + sv));
            if (t == a1 - 1) umma_commit(bar(kBTfOFull + X));
          }
          __syncwarp();
        } else if (t >= t0) {
          if (lane == 0) mbar_arrive(bar(kBTfVEmpty + sv));
        }
        if (t + 1 >= a0 && t + 1 < a1) {
          tc_fence_after();
          const uint64_t dk = smem_desc_sw128(sK(sk), 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * kTfChunk + (kk & 3) * 32) >> 4;
              umma_bf16(tS, dq + off, dk + off, idesc_s, kk > 0 ? 1u : 0u);
            }
            umma_commit(bar(kBTfSFull + X));
            umma_commit(bar(kBTfKEmpty + sk));
          }
          __syncwarp();
          issued = true;
        } else if (t + 1 < t1) {
          if (lane == 0) mbar_arrive(bar(kBTfKEmpty + sk));
        }
      }
      mine += (uint32_t)(a1 - a0);
      kv += (uint32_t)(t1 - t0);
      n_o += any ? 1 : 0;
      drop_item(n);
    }
    if (issued && elect_one()) {  // every MMA of this thread completes before TMEM is released
      umma_commit(bar(kBTfDrain + X));
      mbar_drain(bar(kBTfDrain + X), 0);
    }
    __syncwarp();
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kRegsLow));
    // ------------------------------------------------------------ items, and masked V tiles
    // Items in the order (sequence, chunk of K/V heads, rows from the last, head): the long causal
    // rows go first, so that the short ones level the CTAs out at the end, and a chunk holds as
    // many heads as keep their keys and values (kTfL2 bytes) in L2 together.
    auto seq_items = [&](int b) -> int {
      if (b >= p.batch) return 0;
      const Seq s = load_seq(p, b);
      return (int)((unsigned)(s.lq + 2 * tp.tt - 1) / (unsigned)(2 * tp.tt)) * p.hkv * tp.splits;
    };
    int wb = 0;
    int wi = 0;  // items of the sequences before wb
    // piece number `at` into its slot (every lane works it out, lane 0 writes); 0: no such piece, 2: an
    // item that has fewer
    auto find = [&](int at, TfItem* dst) -> int {
      while (wb < p.batch) {
        const int n = seq_items(wb + lane);
        int nc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, nc, o);
          if (lane >= o) nc += a;
        }
        const int all = __shfl_sync(0xffffffffu, nc, 31);
        if (at < wi + all) {
          const int src = __ffs(__ballot_sync(0xffffffffu, at < wi + nc)) - 1;
          const unsigned of_b = (unsigned)(at - wi - __shfl_sync(0xffffffffu, nc - n, src));
          const unsigned in_b = of_b / (unsigned)tp.splits;
          int found = 1;
          if (lane == 0) {
            const Seq s = load_seq(p, wb + src);
            const unsigned tiles = (unsigned)(s.lq + 2 * tp.tt - 1) / (unsigned)(2 * tp.tt);
            const unsigned fit = (unsigned)(kTfL2 / (HD * 4)) / (unsigned)max(1, s.lk);
            const unsigned heads = max(1u, min((unsigned)p.hkv, fit));
            const unsigned chunk = in_b / (tiles * heads), rest = in_b - chunk * tiles * heads;
            const unsigned mine = min(heads, p.hkv - chunk * heads);
            const int tok0 = (int)((tiles - 1 - rest / mine) * 2) * tp.tt;
            dst->valid = 1;
            dst->bad = 0;
            dst->b = wb + src;
            dst->h = (int)(chunk * heads + rest % mine);
            dst->tok0 = tok0;
            dst->lq = s.lq;
            dst->lk = s.lk;
            dst->q0 = (int)s.q0;
            dst->k0 = (int)s.k0;
            int2 a = slot_tiles(p, s, tok0, tp.tt), b = slot_tiles(p, s, tok0 + tp.tt, tp.tt);
            int first, last, pieces;
            cut_item(a, b, tp.splits, first, last, pieces);
            const int piece = (int)(of_b - in_b * (unsigned)tp.splits), per = (last - first + pieces - 1) / pieces;
            first += piece * per;
            last = min(last, first + per);
            a = make_int2(max(a.x, first), min(a.y, last));
            b = make_int2(max(b.x, first), min(b.y, last));
            dst->a0 = a.y > a.x ? a.x : 0;
            dst->a1 = a.y > a.x ? a.y : 0;
            dst->b0 = b.y > b.x ? b.x : 0;
            dst->b1 = b.y > b.x ? b.y : 0;
            dst->piece = piece;
            dst->pieces = pieces;
            if (piece >= pieces) found = 2;
            dst->free_hi = key_hi(p, s, tok0);
            dst->free_lo = key_lo(p, s, min(s.lq, tok0 + 2 * tp.tt) - 1);
          }
          return __shfl_sync(0xffffffffu, found, 0);
        }
        wi += all;
        wb += 32;
      }
      return 0;
    };
    uint32_t nv = 0;                 // V tiles of the items before
    uint32_t raw[kTfVStages] = {};   // masked tiles mended per stage
    // Items are handed out on demand: their costs differ by the length of their key range, and
    // dealt out in turn the CTA that gets a head's first item would get every head's first.
    auto hand_out = [&]() {
      int i = 0;
      if (lane == 0) i = atomicAdd(tp.next, 1);
      return __shfl_sync(0xffffffffu, i, 0);
    };
    bool ok = true;
    // finds the item that comes n-th on this CTA and announces it, once its slot is free
    auto announce = [&](int n) -> bool {
      int at = hand_out();
      if (n >= kTfItems && ok &&
          !mbar_wait(bar(kBTfItemEmpty + n % kTfItems), ((n / kTfItems) & 1) ^ 1u, p.err, kDevTimeoutOther, abort_flag))
        ok = false;
      int found = 0;
      while (ok && (found = find(at, items + n % kTfItems)) == 2) at = hand_out();
      const bool more = found != 0;
      if (!more && lane == 0) items[n % kTfItems].valid = 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kBTfItemFull + n % kTfItems));
      __syncwarp();
      return more;
    };
    // Item n is announced while item n - 1 is at work (as soon as the slot of the one before is
    // free), so that its loads and first products follow on without a gap; then the masked V
    // tiles of item n - 1 are mended as they land.
    bool more = true;
    for (int next = 0; more; ++next) {
      more = announce(next);
      const int n = next - 1;
      if (n < 0) continue;
      const TfItem& cur = items[n % kTfItems];
      uint32_t* list =
          tp.bad_rows + ((int64_t)blockIdx.x * kTfItems + n % kTfItems) * (int64_t)kTfBadRows * kTfBadWords;
      const int t0 = cur.first(), t1 = cur.last();
      int bad = 0;
      for (int t = t0; t < t1 && ok; ++t) {
        if (kW || !cur.masked(t)) continue;
        const uint32_t s = (nv + (uint32_t)(t - t0)) % kTfVStages;
        uint32_t& done = s == 0 ? raw[0] : raw[1];
        if (!mbar_wait(bar(kBTfVRaw + s), done & 1, p.err, kDevTimeoutFull, abort_flag)) {
          ok = false;
          break;
        }
        ++done;
        // A masked weight is 0, but 0 * NaN is not: keys past the end are zeroed, and non-finite
        // values elsewhere are zeroed and remembered for the rows that do see them.
#pragma unroll 1
        for (int r = lane; r < 128; r += 32) {
          const uint32_t row = sV(s) + (uint32_t)r * 128;
          const bool past = t * 128 + r >= cur.lk;
          __nv_bfloat162 probe = __floats2bfloat162_rn(0.f, 0.f);
          const __nv_bfloat162 zero = probe;
#pragma unroll 4
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 w = lds128(row + (c >> 3) * kTfChunk + (((c & 7) ^ (r & 7)) << 4));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) probe = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&ww[e]), zero, probe);
          }
          const bool odd = !past && (__hisnan(probe.x) || __hisnan(probe.y));
          if (past) {
#pragma unroll 1
            for (int c = 0; c < HD / 8; ++c) sts128(row + (c >> 3) * kTfChunk + (c << 4 & 127), make_uint4(0, 0, 0, 0));
          }
          const uint32_t who = __ballot_sync(0xffffffffu, odd);
          if (odd) {
            const int slot = bad + __popc(who & ((1u << lane) - 1u));
            remember_row<HD>(row, r, t * 128 + r, slot < kTfBadRows ? list + slot * kTfBadWords : nullptr);
          }
          bad += __popc(who);
          __syncwarp();
        }
        if (bad && lane == 0) items[n % kTfItems].bad = bad;
        __threadfence_block();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBTfVFull + s));
      }
      nv += (uint32_t)(t1 - t0);
    }
    if (lane == 0 && atomicAdd(tp.next + 1, 1) == (int)gridDim.x - 1) {
      tp.next[0] = 0;  // nobody asks any more: ready for the next launch
      tp.next[1] = 0;
      __threadfence();
    }
  } else if (kW && warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kRegsLow));
    // ------------------------------------------------ 8-bit rows -> bf16 tiles (128 threads)
    const int tid = (int)threadIdx.x - 384;
    uint32_t nk = 0, nv = 0, nr = 0;  // K tiles, V tiles, raw halves so far
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const TfItem* at = take_item(n);
      if (!at) break;
      const int t0 = at->first(), tiles = at->last() - t0;
      const uint32_t at_first = nk;  // (K and V tiles before this item: as many)
      uint32_t* list =
          tp.bad_rows + ((int64_t)blockIdx.x * kTfItems + n % kTfItems) * (int64_t)kTfBadRows * kTfBadWords;
#pragma unroll 1
      for (int i = 0; i < 2 * tiles && ok; ++i) {  // in the producer's order
        const bool tail = i >= 2 * tiles - 1;
        const bool is_k = i < 2 ? (i == 0 || tiles > 1) : !tail && (i & 1);
        const uint32_t cnt = is_k ? nk : nv;
        const uint32_t s = cnt % 2;
        static_assert(kTfVStages == 2, "two K and two V stages");
        if (!mbar_wait(bar((is_k ? kBTfKEmpty : kBTfVEmpty) + s), ((cnt / 2) & 1) ^ 1u, p.err, kDevTimeoutEmpty, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t dst = is_k ? sK(s) : sV(s);
        const int t = t0 + (int)(cnt - at_first);
        const bool masked = at->masked(t);
#pragma unroll 1
        for (int half = 0; half < 2; ++half, ++nr) {
          const uint32_t rs = nr % kTfRaw;
          if (ok && !mbar_wait(bar(kBTfRawFull + rs), (nr / kTfRaw) & 1, p.err, kDevTimeoutFull, abort_flag)) ok = false;
          if (!ok) break;
          const uint32_t raw = sbase + G::kRawOff + rs * G::kRawBytes;
          // (NaN codes do what they should in a key and in a value that every row sees)
          if (FMT == kKvE4m3 && !is_k && masked)
            remember_codes<HD>(raw, tid, t * 128 + half * 64, at->lk, items[n % kTfItems].bad, list);
#pragma unroll
          for (int j = 0; j < 64 * HD / 16 / 128; ++j) {
            const int u = j * 128 + tid, row = half * 64 + u / (HD / 16), c = u % (HD / 16);
            const uint4 w = lds128(raw + (uint32_t)u * 16);
            const uint4 x0 = make_uint4(bytes_to_bf16x2<FMT>(w.x, 0, 0, 1), bytes_to_bf16x2<FMT>(w.x, 0, 2, 3),
                                        bytes_to_bf16x2<FMT>(w.y, 0, 0, 1), bytes_to_bf16x2<FMT>(w.y, 0, 2, 3));
            const uint4 x1 = make_uint4(bytes_to_bf16x2<FMT>(w.z, 0, 0, 1), bytes_to_bf16x2<FMT>(w.z, 0, 2, 3),
                                        bytes_to_bf16x2<FMT>(w.w, 0, 0, 1), bytes_to_bf16x2<FMT>(w.w, 0, 2, 3));
            const uint32_t at_row = dst + (uint32_t)((c >> 2) * kTfChunk + row * 128);
            // (the upper half of a 128-byte row stores its second unit first: no bank conflicts)
            const int first = (c >> 2) & 1;
            sts128(at_row + (((((c & 3) << 1) + first) ^ (row & 7)) << 4), first ? x1 : x0);
            sts128(at_row + (((((c & 3) << 1) + (first ^ 1)) ^ (row & 7)) << 4), first ? x0 : x1);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBTfRawEmpty + rs));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(bar((is_k ? kBTfKFull : kBTfVFull) + s));
        if (is_k) ++nk; else ++nv;
      }
      drop_item(n);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kRegsHigh));
    // ------------------------------------------------ softmax + epilogue of slot X
    const int X = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_addr + (uint32_t)(X * 128);
    const uint32_t tO = tmem + lane_addr + 256 + (uint32_t)(X * 128);
    uint32_t mine = 0;   // tiles of this slot so far
    uint32_t both = 0;   // key tiles of all items before this one
    uint32_t n_o = 0;    // items in which this slot had tiles

    // The item's Q by TMA: G heads of TT tokens are the slot's rows in order (rows of other
    // sequences or past the end may come along: their results are not written).
    const uint32_t q_bytes = (uint32_t)(tp.tt * p.group * HD * 2);
    auto load_q = [&](const TfItem& c) {
      if (c.hi(X) <= c.lo(X) || quarter != 0 || lane != 0) return;
      mbar_arrive_expect_tx(bar(kBTfQFull + X), q_bytes);
#pragma unroll
      for (int ch = 0; ch < G::kChunks; ++ch)
        tma_load_3d(sQ(X) + ch * kTfChunk, &tmQ, bar(kBTfQFull + X), ch * 64, c.h * p.group, c.q0 + c.tok0 + X * tp.tt);
    };

    const int my_tok = r / p.group, my_g = r % p.group;  // (rows past TT * G are not live)
    // The exponentials of the two slots take turns, A before B in each tile: together they would
    // share the MUFU pipe while the tensor pipe idles. Every tile of an item counts for both
    // slots, so that neither is ever more than one turn ahead.
    auto my_turn = [&](uint32_t g) {
      if (X == 0)
        return g == 0 || mbar_wait(bar(kBTfTurn + 1), (g - 1) & 1, p.err, kDevTimeoutSoftmax, abort_flag);
      return mbar_wait(bar(kBTfTurn), g & 1, p.err, kDevTimeoutSoftmax, abort_flag);
    };
    auto pass_turn = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kBTfTurn + X));
    };
    // One tile of an 8-bit cache, in matrix fragments: a thread has 32 columns of the four rows
    // lane / 4 + 8 j instead of all columns of one, so that it reads 32 scales of each kind, not 128
    // (as broadcasts these took as long as the products). S is read twice, a quarter at a time, rather
    // than kept: unrolled over 128 registers the tile's code did not stay in the instruction cache
    // beside the conversion's. 1324 tokens over 26,383 cached e4m3 keys, 32 / 8 heads: 942 us with a
    // row per thread, 856 in fragments unrolled, 664 like this (bf16, a row per thread and unrolled:
    // 420, and rolled it loses a tenth).
    auto frag_tile = [&](uint32_t g, int t, int a0, bool masked, int hi, int lo, float (&m)[4], float (&l)[4]) -> bool {
      const int tq = lane & 3;
      const uint32_t scales = sbase + G::kScaleOff + (g % kTfScales) * 1024 + tq * 8;
      if (!mbar_wait(bar(kBTfScale + g % kTfScales), (g / kTfScales) & 1, p.err, kDevTimeoutFull, abort_flag)) return false;
      const float k_unit = p.sl2 * kByteUnit<FMT>;
      const float2 sl2x2 = make_float2(k_unit, k_unit);
      // bits of this thread's columns that row j sees
      uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
      if (masked) {
        auto below = [&](int limit) -> uint32_t {  // of its columns before `limit`
          const int x = max(0, limit - t * 128 - 2 * tq), n = 2 * (x >> 3) + min(2, x & 7);
          return n >= 32 ? ~0u : (1u << n) - 1u;
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int from = (lane >> 2) + 8 * j;
          keep[j] = below(__shfl_sync(0xffffffffu, hi, from)) & ~below(__shfl_sync(0xffffffffu, lo, from));
        }
      }
      // the row maxima, in base 2 and scaled
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      auto maxima = [&](auto mk) {
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          float v[2][16];  // [16 lanes][column / 8][row g, row g + 8][2]
          tmem_ld_frag4(tS + x * 32, v[0]);
          tmem_ld_frag4(tS + (1u << 20) + x * 32, v[1]);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __fmul2_rn(lds_f2(scales + x * 128 + k * 32), sl2x2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float* s = v[j >> 1] + k * 4 + (j & 1) * 2;
              float2 y = __fmul2_rn(make_float2(s[0], s[1]), f);
              if constexpr (decltype(mk)::value) {
                const uint32_t bits = keep[j] >> (8 * x + 2 * k);
                if (!(bits & 1u)) y.x = -INFINITY;
                if (!(bits & 2u)) y.y = -INFINITY;
              }
              mx[j] = max3_f(mx[j], y.x, y.y);
            }
          }
        }
      };
      if (masked) maxima(std::true_type{});
      else maxima(std::false_type{});
      bool grown = t == a0;
#pragma unroll
      for (int j = 0; j < 4; ++j) grown |= mx[j] - m[j] > 8.0f;
      // as for rows below; without growth by 2^8 the maxima need not even be gathered
      if (__any_sync(0xffffffffu, grown)) {
        float alpha[4];
        bool need = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
          alpha[j] = 1.f;
          if (t == a0) {
            m[j] = mx[j];
          } else if (mx[j] - m[j] > 8.0f) {
            alpha[j] = exp2_approx(m[j] - mx[j]);
            m[j] = mx[j];
            l[j] *= alpha[j];
            need = true;
          }
        }
        if (__any_sync(0xffffffffu, need)) {
          // PV(t-1) completed before S(t) (the tensor pipe runs in order): O is stable
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            const uint32_t at = tO + ((uint32_t)(c & 1) << 20) + (c >> 1) * 32;
            const float a = c & 1 ? alpha[2] : alpha[0], b = c & 1 ? alpha[3] : alpha[1];
            float o[16];
            tmem_ld_frag4(at, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= i & 2 ? b : a;
            tmem_st_frag4(at, o);
          }
        }
      }
      float2 rs[4];
      float nmu[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        rs[j] = make_float2(0.f, 0.f);
        nmu[j] = m[j] == -INFINITY ? 0.f : -m[j];
      }
      auto weights = [&](auto mk, int c, const float (&v)[32]) {  // columns 32 c .. 32 c + 31
        uint32_t pk[2][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 ks = __fmul2_rn(lds_f2(scales + (c * 4 + i) * 32), sl2x2);
          const float2 vs = lds_f2(scales + 512 + (c * 4 + i) * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float* s = v + (j >> 1) * 16 + i * 4 + (j & 1) * 2;
            const float2 a = __ffma2_rn(make_float2(s[0], s[1]), ks, make_float2(nmu[j], nmu[j]));
            float2 e = make_float2(exp2_approx(a.x), exp2_approx(a.y));
            float2 w = __fmul2_rn(e, vs);
            if constexpr (decltype(mk)::value) {  // an unseen key's scales may be anything: its weight is 0, not 0 * scale
              const uint32_t bits = keep[j] >> (8 * c + 2 * i);
              if (!(bits & 1u)) e.x = w.x = 0.f;
              if (!(bits & 2u)) e.y = w.y = 0.f;
            }
            rs[j] = __fadd2_rn(rs[j], e);
            pk[j >> 1][2 * i + (j & 1)] = pack_bf16x2(w.x, w.y);
          }
        }
        tmem_st_half4(tS + c * 16, pk[0]);
        tmem_st_half4(tS + (1u << 20) + c * 16, pk[1]);
      };
      auto load = [&](int c, float (&v)[32]) {
        tmem_ld_frag4(tS + c * 32, v);
        tmem_ld_frag4(tS + (1u << 20) + c * 32, v + 16);
      };
      auto publish = [&](int c) {
        tmem_wait_st();  // this quarter of P is in TMEM (over S that has been read): its products may start
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBTfPFull + X * 4 + c));
      };
      if (!my_turn(g)) return false;
      auto walk = [&](auto mk) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v0[32];
          load(c, v0);
          tmem_wait_ld32(v0);
          weights(mk, c, v0);
          if (c == 3) pass_turn();
          publish(c);
        }
      };
      if (masked) walk(std::true_type{});
      else walk(std::false_type{});
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] += rs[j].x + rs[j].y;
      return true;
    };
    bool ok = true;
    const TfItem* at = take_item(0);
    if (at) load_q(*at);
    for (int n = 0; at; ++n) {
      const TfItem& it = *at;
      const int t0 = it.first(), t1 = it.last();
      const bool any = it.hi(X) > it.lo(X);
      const int a0 = any ? it.lo(X) : t1, a1 = any ? it.hi(X) : t1;
      const int tok = it.tok0 + X * tp.tt + my_tok;
      const bool live = r < tp.tt * p.group && tok < it.lq;
      int hi = 0, lo = 0;
      if (live) {
        const Seq s{it.q0, it.k0, it.lq, it.lk};
        hi = key_hi(p, s, tok);
        lo = key_lo(p, s, tok);
      }
      bool q_sent = false;
      // (8-bit: of the four rows of the thread's fragments, l over the thread's columns)
      float m = -INFINITY, l = 0.f;
      float m4[4], l4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m4[j] = -INFINITY;
        l4[j] = 0.f;
      }
      for (int t = t0; t < t1; ++t) {
        if (t < a0 || t >= a1) {  // the other slot's alone
          if (!(ok = my_turn(both + (uint32_t)(t - t0)))) break;
          pass_turn();
          continue;
        }
        if (!mbar_wait(bar(kBTfSFull + X), (mine + (uint32_t)(t - a0)) & 1, p.err, kDevTimeoutSoftmax, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // the slot's last S is done: its Q may be replaced, if the next item is known yet
        if (t == a1 - 1 && quarter == 0 && mbar_try_wait(bar(kBTfItemFull + (n + 1) % kTfItems), ((n + 1) / kTfItems) & 1)) {
          const TfItem& c = items[(n + 1) % kTfItems];
          if (c.valid) load_q(c);
          q_sent = true;
        }
        const bool masked = it.masked(t);
        if constexpr (kW) {
          const uint32_t g = both + (uint32_t)(t - t0);
          if (!frag_tile(g, t, a0, masked, hi, lo, m4, l4)) {
            ok = false;
            break;
          }
          continue;
        }
        const int lim = hi - t * 128, from = lo - t * 128;
        // bits of the keys 32 c .. 32 c + 31 that this row sees
        auto keep_bits = [&](int c) -> uint32_t {
          const int a = min(32, max(0, lim - c * 32)), b = min(32, max(0, from - c * 32));
          return (a == 32 ? ~0u : (1u << a) - 1u) & ~(b == 32 ? ~0u : (1u << b) - 1u);
        };
        if (masked) {
          // a short loop over S in TMEM: few tiles are masked, and unrolled over 128 registers this
          // code left the instruction cache between two of them (2 to 4 us a tile instead of 0.5)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float x[32];
            tmem_ld32(tS + c * 32, x);
            const uint32_t keep = keep_bits(c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(keep >> i & 1u)) x[i] = -INFINITY;
            tmem_st32(tS + c * 32, x);
          }
          tmem_wait_st();
        }
        float v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, *reinterpret_cast<float(*)[32]>(v + c * 32));
        tmem_wait_ld();
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8) {
          mx[0] = max3_f(mx[0], v[i], v[i + 1]);
          mx[1] = max3_f(mx[1], v[i + 2], v[i + 3]);
          mx[2] = max3_f(mx[2], v[i + 4], v[i + 5]);
          mx[3] = max3_f(mx[3], v[i + 6], v[i + 7]);
        }
        const float m_new = fmaxf(m, max3_f(fmaxf(mx[0], mx[1]), mx[2], mx[3]));
        // the maximum is moved only when it has grown by 2^8: the weights stay below 2^8, far from
        // fp32's and bf16's range, and most tiles leave O alone
        const bool need = t > a0 && (m_new - m) * p.sl2 > 8.0f;
        float alpha = 1.0f;
        if (t == a0) m = m_new;
        if (need) {
          alpha = exp2_approx((m - m_new) * p.sl2);
          m = m_new;
        }
        if (__any_sync(0xffffffffu, need)) {
          // PV(t-1) completed before S(t) (the tensor pipe runs in order): O is stable
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(tO + c * 32, o);
          }
        }
        if (!my_turn(both + (uint32_t)(t - t0))) {
          ok = false;
          break;
        }
        const float mu = m == -INFINITY ? 0.f : m * p.sl2;
        const float2 sl2x2 = make_float2(p.sl2, p.sl2), nmu2 = make_float2(-mu, -mu);
        float2 rs[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) rs[q] = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 a = __ffma2_rn(make_float2(v[32 * c + 2 * i], v[32 * c + 2 * i + 1]), sl2x2, nmu2);
            const float2 e = make_float2(exp2_approx(a.x), exp2_approx(a.y));
            rs[i & 3] = __fadd2_rn(rs[i & 3], e);
            pk[i] = pack_bf16x2(e.x, e.y);
          }
          tmem_st16(tS + c * 16, pk);
          if (c == 3) pass_turn();
          if (c + 1 < G::kFirstP) continue;
          tmem_wait_st();  // this quarter of P is in TMEM: its products may start
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBTfPFull + X * 4 + c));
        }
        const float2 u = __fadd2_rn(__fadd2_rn(rs[0], rs[1]), __fadd2_rn(rs[2], rs[3]));
        l = l * alpha + (u.x + u.y);
      }
      mine += (uint32_t)(a1 - a0);
      both += (uint32_t)(t1 - t0);
      if constexpr (kW) {  // back to the thread's own row
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = l4[j];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          const float lj = __shfl_sync(0xffffffffu, x, (lane & 7) * 4);
          const float mj = __shfl_sync(0xffffffffu, m4[j], (lane & 7) * 4);
          if ((lane >> 3) == j) {
            l = lj;
            m = mj;
          }
        }
      }
      // the next item's Q goes in first: its products then run while this item's rows are written
      const TfItem* next = ok ? take_item(n + 1) : nullptr;
      if (next && !q_sent) load_q(*next);
      if (ok && any) ok = mbar_wait(bar(kBTfOFull + X), n_o & 1, p.err, kDevTimeoutSoftmax, abort_flag);
      n_o += any ? 1 : 0;
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : __fdividef(kByteUnit<FMT>, l);
      const int bad = any ? *reinterpret_cast<const volatile int*>(&it.bad) : 0;
      const bool cut = it.pieces > 1;
      const bool write = ok && live &&
                         WX_IN_BOUNDS(p.err, it.q0 >= 0 && it.q0 + tok < p.total_q && it.h * p.group + my_g < p.hq &&
                                                 it.piece >= 0 && it.piece < tp.splits);
      const int64_t at_row = ((int64_t)it.q0 + tok) * p.hq + it.h * p.group + my_g;
      const int64_t at_part = it.piece * (p.total_q * p.hq) + at_row;
      __nv_bfloat16* row = p.out + ((int64_t)it.q0 + tok) * p.out_stride + (int64_t)(it.h * p.group + my_g) * HD;
      if (!write || cut) row = nullptr;
      // 16-byte units are exchanged between two neighbouring lanes, so that a store covers 32
      // bytes (a whole sector) of each row: `even` is the row of the lower lane, `odd` the other's
      const auto other = reinterpret_cast<__nv_bfloat16*>(
          __shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), 1));
      __nv_bfloat16 *even = lane & 1 ? other : row, *odd = lane & 1 ? row : other;
#pragma unroll 1
      for (int c = 0; c < HD / 16; ++c) {
        float o[16];
        if (any) {
          tmem_ld16(tO + c * 16, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0.f;
        }
        if (bad) {  // non-finite values of V that this row does see: infinities add up, both signs to NaN
          const int col = c * 16;
          uint32_t plus = 0u, minus = 0u;
          const uint32_t* list =
              tp.bad_rows + ((int64_t)blockIdx.x * kTfItems + n % kTfItems) * (int64_t)kTfBadRows * kTfBadWords;
#pragma unroll 1
          for (int e = 0; e < min(bad, kTfBadRows); ++e) {
            const uint32_t* entry = list + e * kTfBadWords;
            const int key = (int)__ldcg(entry);
            if (key >= lo && key < hi) {
              plus |= __ldcg(entry + 1 + (col >> 5)) >> (col & 31);
              minus |= __ldcg(entry + 5 + (col >> 5)) >> (col & 31);
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (plus >> i & 1u) o[i] += INFINITY;
            if (minus >> i & 1u) o[i] -= INFINITY;
          }
        }
        if (cut) {
          if (write) {
            float* dst = tp.part + at_part * HD + c * 16;
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(dst + i) =
                  make_float4(o[i] * kByteUnit<FMT>, o[i + 1] * kByteUnit<FMT>, o[i + 2] * kByteUnit<FMT>, o[i + 3] * kByteUnit<FMT>);
          }
          continue;
        }
        uint4 w0 = make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                              pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
        uint4 w1 = make_uint4(pack_bf16x2(o[8] * inv, o[9] * inv), pack_bf16x2(o[10] * inv, o[11] * inv),
                              pack_bf16x2(o[12] * inv, o[13] * inv), pack_bf16x2(o[14] * inv, o[15] * inv));
        // lower lane: both first units, upper lane: both second units
        uint4 give = lane & 1 ? w0 : w1;
        give.x = __shfl_xor_sync(0xffffffffu, give.x, 1);
        give.y = __shfl_xor_sync(0xffffffffu, give.y, 1);
        give.z = __shfl_xor_sync(0xffffffffu, give.z, 1);
        give.w = __shfl_xor_sync(0xffffffffu, give.w, 1);
        if (lane & 1) w0 = give;
        else w1 = give;
        const int at_col = c * 16 + (lane & 1) * 8;
        if (even) *reinterpret_cast<uint4*>(even + at_col) = w0;
        if (odd) *reinterpret_cast<uint4*>(odd + at_col) = w1;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && any) mbar_arrive(bar(kBTfOEmpty + X));
      const float m2 = kW ? m : m * p.sl2;
      if (cut && write) tp.part_ml[at_part] = make_float2(m2, l);
      if (!cut && write && p.lse) p.lse[at_row] = l == 0.f ? -INFINITY : (m2 + __log2f(l)) * 0.69314718055994531f;
      drop_item(n);
      at = next;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Rows of items that were cut up: sums of the pieces, in order, brought to one maximum. A warp a row.
template <int HD>
__global__ void __launch_bounds__(256) text_flash_join_kernel(TfParams tp) {
  const TextAttnParams& p = tp.a;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = p.total_q * p.hq;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int64_t token = row / p.hq;
  int b = 0;  // last sequence that begins at or before the token
  for (int n = p.batch; n > 1;) {
    const int half = n / 2;
    if (p.cu_q[b + half] <= token) b += half;
    n -= half;
  }
  const Seq s = load_seq(p, b);
  const int64_t tok = token - s.q0;
  if (tok < 0 || tok >= s.lq) return;
  const int tok0 = (int)tok / (2 * tp.tt) * (2 * tp.tt);
  int first, last, pieces;
  cut_item(slot_tiles(p, s, tok0, tp.tt), slot_tiles(p, s, tok0 + tp.tt, tp.tt), tp.splits, first, last, pieces);
  if (pieces < 2) return;
  constexpr int kPer = HD / 32;
  float o[kPer] = {};
  float M = -INFINITY, L = 0.f;
  auto piece = [&](int i) { return i < pieces ? tp.part_ml[i * rows + row] : make_float2(-INFINITY, 0.f); };
  for (int c = 0; c < pieces; c += 32) {
    const float2 ml = piece(c + lane);
    float m = ml.y != 0.f ? ml.x : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    M = fmaxf(M, m);
  }
  for (int c = 0; c < pieces; c += 32) {
    const float2 ml = piece(c + lane);
    const float f = ml.y != 0.f ? exp2_approx(ml.x - M) : 0.f;
    const uint32_t seen = __ballot_sync(0xffffffffu, ml.y != 0.f);
    float l = ml.y != 0.f ? ml.y * f : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    L += l;
    const int n = min(32, pieces - c);
#pragma unroll 1
    for (int i = 0; i < n; i += 8) {  // eight pieces' rows in flight
      float x[8][kPer];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float* src = tp.part + (min(c + i + q, pieces - 1) * rows + row) * HD + lane * kPer;
        if constexpr (kPer == 4) {
          const float4 y = *reinterpret_cast<const float4*>(src);
          x[q][0] = y.x;
          x[q][1] = y.y;
          x[q][2] = y.z;
          x[q][3] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(src);
          x[q][0] = y.x;
          x[q][1] = y.y;
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float w = __shfl_sync(0xffffffffu, f, (i + q) & 31);
        if (i + q < n && (seen >> (i + q) & 1u))  // (nothing seen: its sums may be anything)
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[e] += x[q][e] * w;
      }
    }
  }
  const float inv = L == 0.f ? 0.f : __fdividef(1.0f, L);
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + token * p.out_stride + (row - token * p.hq) * HD + lane * kPer);
#pragma unroll
  for (int e = 0; e < kPer; e += 2) dst[e / 2] = pack_bf16x2(o[e] * inv, o[e + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.69314718055994531f;
}

template <int FMT, int HD>
static int launch_flash(wx_ctx* ctx, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, TfParams& tp) {
  using G = TfGeom<FMT, HD>;
  auto fn = text_flash_kernel<FMT, HD>;
  int st = ensure_smem_attr(ctx, (const void*)fn, G::kSmem, "text_flash");
  if (st) return st;
  // setmaxnreg moves registers within what the launch reserved
  static const bool regs_ok = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, (const void*)text_flash_kernel<FMT, HD>) == cudaSuccess &&
           fa.numRegs * G::kThreads >= G::kRegsUsed;
  }();
  if (!regs_ok) return set_error(ctx, WX_ERR_CUDA, "text_flash: register split does not fit");
  const TextAttnParams& p = tp.a;
  const int64_t items = (int64_t)p.hkv * (p.total_q / (2 * tp.tt) + p.batch);
  // Too few items to level the SMs out are cut into pieces of their keys, as many as give kTfWaves
  // to an SM and as the longest range that a row can see allows.
  int64_t keys = p.block_table ? p.blocks_per_seq << p.page_shift : p.total_k;
  if (p.window) keys = std::min<int64_t>(keys, (int64_t)p.window + 2 * tp.tt);
  tp.splits = (int)std::max<int64_t>(1, std::min((kTfWaves * ctx->num_sms + items - 1) / items, keys / (128 * kTfMinTiles)));
  const int grid = (int)std::min<int64_t>(ctx->num_sms, items * tp.splits);
  const int64_t rows = tp.splits > 1 ? p.total_q * p.hq * tp.splits : 0;
  Carve c;
  const size_t o_bad = c.take((size_t)ctx->num_sms * kTfItems * kTfBadRows * kTfBadWords * 4);
  const size_t o_part = c.take((size_t)rows * HD * 4), o_ml = c.take((size_t)rows * 8);
  uint8_t* ws = static_cast<uint8_t*>(workspace(ctx, c.off, &st));
  if (!ws) return st;
  tp.bad_rows = reinterpret_cast<uint32_t*>(ws + o_bad);
  tp.part = reinterpret_cast<float*>(ws + o_part);
  tp.part_ml = reinterpret_cast<float2*>(ws + o_ml);
  if (!(tp.next = arrival_counters(ctx, 2, &st))) return st;
  ProfScope prof(ctx, kProfAttn);
  fn<<<grid, G::kThreads, G::kSmem, ctx->stream>>>(tq, tk, tv, tp);
  if (tp.splits == 1) return launch_status(ctx, "text_flash");
  text_flash_join_kernel<HD><<<(unsigned)((p.total_q * p.hq + 7) / 8), 256, 0, ctx->stream>>>(tp);
  return launch_status(ctx, "text_flash", 2);
}

int text_flash(wx_ctx* ctx, const TextAttnParams& p, int head_dim, const KvSource& kv) {
  TfParams tp{};
  tp.a = p;
  tp.box = p.block_table ? std::min(128, 1 << p.page_shift) : 128;
  tp.tt = 128 / p.group;
  CUtensorMap tq, tk, tv;
  int st;
  const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)p.hq, (uint64_t)p.total_q};
  const uint64_t ld[2] = {(uint64_t)head_dim, (uint64_t)p.q_stride};
  const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)tp.tt};
  if ((st = make_tmap_bf16_3d(ctx, &tq, p.q, dims, ld, box))) return st;
  const bool big = head_dim == 128;
  if (kv.format != kKvBf16) {  // raw rows by untiled copies: the maps of K and V are not used
    tp.box = std::min(64, 1 << p.page_shift);
    tp.k8 = static_cast<const uint8_t*>(kv.k);
    tp.v8 = static_cast<const uint8_t*>(kv.v);
    if (kv.format == kKvInt8)
      return big ? launch_flash<kKvInt8, 128>(ctx, tq, tq, tq, tp) : launch_flash<kKvInt8, 64>(ctx, tq, tq, tq, tp);
    return big ? launch_flash<kKvE4m3, 128>(ctx, tq, tq, tq, tp) : launch_flash<kKvE4m3, 64>(ctx, tq, tq, tq, tp);
  }
  if ((st = make_tmap_bf16_2d(ctx, &tk, kv.k, kv.rows, kv.cols, kv.k_stride, 64, tp.box))) return st;
  if ((st = make_tmap_bf16_2d(ctx, &tv, kv.v, kv.rows, kv.cols, kv.v_stride, 64, tp.box))) return st;
  return big ? launch_flash<kKvBf16, 128>(ctx, tq, tk, tv, tp) : launch_flash<kKvBf16, 64>(ctx, tq, tk, tv, tp);
}

}  // namespace wx
