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
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "wx_text_dev.cuh"

namespace wx {

constexpr int kTfThreads = 384;
constexpr int kTfRegsLow = 72, kTfRegsHigh = 216;
static_assert(kTfRegsLow * 128 + kTfRegsHigh * 256 <= 168 * kTfThreads, "register split exceeds the launch");
constexpr int kTfKStages = 3, kTfVStages = 2;
constexpr int kTfItems = 2;     // item slots: the one at work and the next
constexpr int kTfChunk = 128 * 128;  // one 64-column SW128 chunk of a 128-row tile
constexpr int kTfBadRows = 1024;     // V rows with non-finite values remembered per item
constexpr int kTfBadWords = 5;       // key, 128-bit column mask

template <int HD>
struct TfGeom {
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kChunks = HD / 64;
  static constexpr int kBarOff = (2 + kTfKStages + kTfVStages) * kTile;
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
  int bad;               // V rows with non-finite values found in masked tiles
  __device__ int lo(int X) const { return X ? b0 : a0; }
  __device__ int hi(int X) const { return X ? b1 : a1; }
  __device__ int first() const { return a1 <= a0 ? b0 : b1 <= b0 ? a0 : min(a0, b0); }
  __device__ int last() const { return max(first(), max(a1 > a0 ? a1 : 0, b1 > b0 ? b1 : 0)); }
  __device__ bool masked(int t) const { return t * 128 + 128 > free_hi || t * 128 < free_lo; }
};

enum : int {
  kBTfItemFull = 0,                       // [items]
  kBTfItemEmpty = kBTfItemFull + kTfItems,  // [items] count 11: every other warp has read it
  kBTfQFull = kBTfItemEmpty + kTfItems,   // [2]
  kBTfKFull = kBTfQFull + 2,              // [K stages]
  kBTfKEmpty = kBTfKFull + kTfKStages,    // count 2: both slots
  kBTfVRaw = kBTfKEmpty + kTfKStages,     // [V stages] a masked tile has landed
  kBTfVFull = kBTfVRaw + kTfVStages,      // [V stages] count 2: landed, and mended where masked
  kBTfVEmpty = kBTfVFull + kTfVStages,    // count 2
  kBTfSFull = kBTfVEmpty + kTfVStages,    // [2]
  kBTfPFull = kBTfSFull + 2,              // [2][4] count 4
  kBTfOFull = kBTfPFull + 8,              // [2]
  kBTfOEmpty = kBTfOFull + 2,             // [2] count 4: the epilogue has read O
  kBTfDrain = kBTfOEmpty + 2,             // [2]
  kBTfCount = kBTfDrain + 2
};
static_assert(kBTfCount * 8 + 32 <= 512, "barriers overlap the items");

__device__ __forceinline__ float max3_f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// a value the compiler recomputes where it is used (keeps descriptors out of registers)
__device__ __forceinline__ uint64_t fresh64(uint64_t v) {
  uint64_t r;
  asm volatile("mov.b64 %0, %1;" : "=l"(r) : "l"(v));
  return r;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

struct TfParams {
  TextAttnParams a;
  int tt;              // tokens of a slot: floor(128 / G)
  int box;             // rows of a K/V box: 128, or a page where pages are smaller
  int* next;           // [2] items handed out, CTAs that have finished (0, 0 between launches)
  uint32_t* bad_rows;  // [CTA][kTfItems][kTfBadRows][kTfBadWords]
};

template <int HD>
__global__ void __launch_bounds__(kTfThreads, 1)
    text_flash_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, TfParams tp) {
  using G = TfGeom<HD>;
  constexpr int kTile = G::kTile;
  const TextAttnParams& p = tp.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  auto sQ = [&](int X) { return sbase + (uint32_t)X * kTile; };
  auto sK = [&](int s) { return sbase + (uint32_t)(2 + s) * kTile; };
  auto sV = [&](int s) { return sbase + (uint32_t)(2 + kTfKStages + s) * kTile; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kBarOff);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBTfCount);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* turns = reinterpret_cast<int*>(tmem_slot + 2);  // [2] warps x tiles whose exponentials are done
  TfItem* items = reinterpret_cast<TfItem*>(smem + G::kItemOff);
  static_assert(sizeof(TfItem) <= 128, "item slots");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kBTfCount; ++i) {
      uint32_t c = 1;
      if (i >= kBTfItemEmpty && i < kBTfItemEmpty + kTfItems) c = 11;
      if ((i >= kBTfKEmpty && i < kBTfKEmpty + kTfKStages) || (i >= kBTfVFull && i < kBTfVEmpty + kTfVStages)) c = 2;
      if ((i >= kBTfPFull && i < kBTfPFull + 8) ||
          (i >= kBTfOEmpty && i < kBTfOEmpty + 2))
        c = 4;
      mbar_init(bar(i), c);
    }
    *abort_flag = 0;
    turns[0] = turns[1] = 0;
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

  // item n as this warp sees it; its slot goes back when the warp is done with it
  auto take_item = [&](int n, TfItem& it) -> bool {
    if (!mbar_wait(bar(kBTfItemFull + n % kTfItems), (n / kTfItems) & 1, p.err, kDevTimeoutOther, abort_flag)) {
      it.valid = 0;
      return false;
    }
    it = items[n % kTfItems];
    return it.valid != 0;
  };
  auto drop_item = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kBTfItemEmpty + n % kTfItems));
  };

  if (warp == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTfRegsLow));
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    uint32_t nk = 0, nv = 0;  // tiles loaded
    const int boxes = 128 / tp.box;
    TfItem it;
    bool ok = true;
    for (int n = 0; ok && take_item(n, it); ++n) {
      const int t0 = it.first(), t1 = it.last();
      int ids = 0, ids_from = -1;  // block entries of 32 consecutive boxes, one per lane
      auto load = [&](bool is_k, int t) -> bool {
        const uint32_t cnt = is_k ? nk : nv;
        const int ns = is_k ? kTfKStages : kTfVStages;
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
          const int b0 = t * boxes;
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
          const int bx = lane / G::kChunks, ch = lane % G::kChunks;
          const int page = __shfl_sync(0xffffffffu, ids, (b0 - ids_from + bx) & 31);
          if (bx < nb) {
            const int j = t * 128 + bx * tp.box;
            const int row = (int)((((int64_t)page * p.hkv + it.h) << p.page_shift) | (j & ((1 << p.page_shift) - 1)));
            tma_load_2d(dst + ch * kTfChunk + bx * tp.box * 128, tm, full, ch * 64, row);
          }
        }
        if (is_k) ++nk; else ++nv;
        return true;
      };
      ok = t1 <= t0 || (load(true, t0) && (t0 + 1 >= t1 || load(true, t0 + 1)));
      for (int t = t0; t < t1 && ok; ++t) {
        ok = load(false, t);
        if (ok && t + 2 < t1) ok = load(true, t + 2);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTfRegsLow));
    // ------------------------------------------------------------ MMA issuer of slot X
    const int X = warp - 1;
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, false, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(128, HD, false, true);  // P from TMEM, V MN-major
    const uint32_t tS = tmem + (uint32_t)(X * 128);
    const uint32_t tO = tmem + 256 + (uint32_t)(X * 128);
    const uint64_t dq = fresh64(smem_desc_sw128(sQ(X), 16, 1024));
    uint32_t kv = 0;    // tiles of all items before this one (K and V alike)
    uint32_t mine = 0;  // tiles of this slot so far
    uint32_t n_o = 0;   // items in which this slot had tiles
    bool ok = true, issued = false;
    TfItem it;
    for (int n = 0; ok && take_item(n, it); ++n) {
      const int t0 = it.first(), t1 = it.last();
      const bool any = it.hi(X) > it.lo(X);
      const int a0 = any ? it.lo(X) : t1, a1 = any ? it.hi(X) : t1;
      if (lane == 0) {
        auto wait_k = [&](int t) {
          const uint32_t c = kv + (uint32_t)(t - t0);
          return mbar_wait(bar(kBTfKFull + c % kTfKStages), (c / kTfKStages) & 1, p.err, kDevTimeoutFull, abort_flag);
        };
        auto wait_v = [&](int t) {
          const uint32_t c = kv + (uint32_t)(t - t0);
          return mbar_wait(bar(kBTfVFull + c % kTfVStages), (c / kTfVStages) & 1, p.err, kDevTimeoutFull, abort_flag);
        };
        auto kbar = [&](int t) { return bar(kBTfKEmpty + (kv + (uint32_t)(t - t0)) % kTfKStages); };
        auto vbar = [&](int t) { return bar(kBTfVEmpty + (kv + (uint32_t)(t - t0)) % kTfVStages); };
        auto skip = [&](int t) {  // a tile only the other slot works on
          if (!wait_k(t)) return false;
          mbar_arrive(kbar(t));
          if (!wait_v(t)) return false;
          mbar_arrive(vbar(t));
          return true;
        };
        auto issue_s = [&](int t) {
          tc_fence_after();
          const uint64_t dk = fresh64(smem_desc_sw128(sK((kv + (uint32_t)(t - t0)) % kTfKStages), 16, 1024));
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kTfChunk + (kk & 3) * 32) >> 4;
            umma_bf16(tS, dq + off, dk + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          issued = true;
          umma_commit(bar(kBTfSFull + X));
          umma_commit(kbar(t));
        };
        if (any) ok = mbar_wait(bar(kBTfQFull + X), n_o & 1, p.err, kDevTimeoutSoftmax, abort_flag);
        for (int t = t0; ok && t < a0; ++t) ok = skip(t);
        if (ok && a0 < a1 && (ok = wait_k(a0))) issue_s(a0);
        for (int t = a0; ok && t < a1; ++t) {
          // V(t) and K(t+1) are waited for before P(t): PV(t) and S(t+1) then go out back to back
          ok = wait_v(t) && (t + 1 >= a1 || wait_k(t + 1));
          // the first product of an item overwrites O: the last epilogue must have read it
          if (ok && t == a0 && n_o > 0)
            ok = mbar_wait(bar(kBTfOEmpty + X), (n_o - 1) & 1, p.err, kDevTimeoutSoftmax, abort_flag);
          if (!ok) break;
          const uint64_t dv =
              fresh64(smem_desc_sw128(sV((kv + (uint32_t)(t - t0)) % kTfVStages), kTfChunk, 1024));
#pragma unroll
          for (int part = 0; part < 4 && ok; ++part) {
            if (!mbar_wait(bar(kBTfPFull + X * 4 + part), (mine + (uint32_t)(t - a0)) & 1, p.err, kDevTimeoutSoftmax,
                           abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
              const int kk = part * 2 + k2;
              umma_bf16_ts(tO, tS + kk * 8, dv + (uint64_t)(kk * (2048 >> 4)), idesc_o, (t > a0 || kk > 0) ? 1u : 0u);
            }
          }
          if (!ok) break;
          umma_commit(vbar(t));
          if (t + 1 < a1) issue_s(t + 1);
        }
        if (ok && a0 < a1) umma_commit(bar(kBTfOFull + X));
        for (int t = max(a1, t0); ok && t < t1; ++t) ok = skip(t);
        mine += (uint32_t)(a1 - a0);
        kv += (uint32_t)(t1 - t0);
        n_o += any ? 1 : 0;
      }
      drop_item(n);
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    if (lane == 0 && issued) {  // every MMA of this thread completes before TMEM is released
      umma_commit(bar(kBTfDrain + X));
      mbar_drain(bar(kBTfDrain + X), 0);
    }
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTfRegsLow));
    // ------------------------------------------------------------ items, and masked V tiles
    // Items in the order (sequence, K/V head, rows from the last): CTAs that run at the same
    // time share a head's keys in L2, and the long causal rows of a head go first.
    auto seq_items = [&](int b) -> int64_t {
      if (b >= p.batch) return 0;
      const Seq s = load_seq(p, b);
      return (int64_t)((s.lq + 2 * tp.tt - 1) / (2 * tp.tt)) * p.hkv;
    };
    int wb = 0;
    int64_t wi = 0;  // items of the sequences before wb
    auto find = [&](int64_t at, TfItem& c) {
      c.valid = 0;
      c.bad = 0;
      while (wb < p.batch) {
        const int64_t n = seq_items(wb + lane);
        int64_t nc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t a = __shfl_up_sync(0xffffffffu, nc, o);
          if (lane >= o) nc += a;
        }
        const int64_t all = __shfl_sync(0xffffffffu, nc, 31);
        if (at < wi + all) {
          const int src = __ffs(__ballot_sync(0xffffffffu, at < wi + nc)) - 1;
          const int in_b = (int)(at - wi - __shfl_sync(0xffffffffu, nc - n, src));
          const Seq s = load_seq(p, wb + src);
          const int tiles = (s.lq + 2 * tp.tt - 1) / (2 * tp.tt);
          c.valid = 1;
          c.b = wb + src;
          c.h = in_b / tiles;
          c.tok0 = (tiles - 1 - in_b % tiles) * 2 * tp.tt;
          c.lq = s.lq;
          c.lk = s.lk;
          c.q0 = (int)s.q0;
          c.k0 = (int)s.k0;
          auto tiles_of = [&](int k0, int& x0, int& x1) {
            const int k1 = min(s.lq, k0 + tp.tt);  // tokens [k0, k1)
            x0 = x1 = 0;
            if (k0 >= k1) return;
            const int hi = key_hi(p, s, k1 - 1), lo = key_lo(p, s, k0);
            if (hi <= lo) return;
            x0 = lo >> 7;
            x1 = (hi + 127) >> 7;
          };
          tiles_of(c.tok0, c.a0, c.a1);
          tiles_of(c.tok0 + tp.tt, c.b0, c.b1);
          c.free_hi = key_hi(p, s, c.tok0);
          c.free_lo = key_lo(p, s, min(s.lq, c.tok0 + 2 * tp.tt) - 1);
          return;
        }
        wi += all;
        wb += 32;
      }
    };
    uint32_t nv = 0;                 // V tiles of the items before
    uint32_t raw[kTfVStages] = {};   // masked tiles mended per stage
    // Items are handed out on demand: their costs differ by the length of their key range, and
    // dealt out in turn the CTA that gets a head's first item would get every head's first.
    auto hand_out = [&]() {
      int i = 0;
      if (lane == 0) i = atomicAdd(tp.next, 1);
      return (int64_t)__shfl_sync(0xffffffffu, i, 0);
    };
    bool ok = true;
    auto announce = [&](int n, TfItem& c) {
      if (n >= kTfItems && ok &&
          !mbar_wait(bar(kBTfItemEmpty + n % kTfItems), ((n / kTfItems) & 1) ^ 1u, p.err, kDevTimeoutOther, abort_flag))
        ok = false;
      if (!ok) c.valid = 0;
      if (lane == 0) {
        items[n % kTfItems] = c;
        mbar_arrive(bar(kBTfItemFull + n % kTfItems));
      }
      __syncwarp();
    };
    TfItem cur, next;
    find(hand_out(), next);
    announce(0, next);
    for (int n = 0; next.valid; ++n) {
      cur = next;
      // the next item is announced while this one is at work (as soon as the last one's slot is
      // free), so that its loads and first products follow on without a gap
      find(hand_out(), next);
      announce(n + 1, next);
      uint32_t* list =
          tp.bad_rows + ((int64_t)blockIdx.x * kTfItems + n % kTfItems) * (int64_t)kTfBadRows * kTfBadWords;
      const int t0 = cur.first(), t1 = cur.last();
      int bad = 0;
      for (int t = t0; t < t1 && ok; ++t) {
        if (!cur.masked(t)) continue;
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
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 w = lds128(row + (c >> 3) * kTfChunk + (((c & 7) ^ (r & 7)) << 4));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) probe = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&ww[e]), zero, probe);
          }
          const bool odd = !past && (__hisnan(probe.x) || __hisnan(probe.y));
          if (past) {
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) sts128(row + (c >> 3) * kTfChunk + (c << 4 & 127), make_uint4(0, 0, 0, 0));
          }
          const uint32_t who = __ballot_sync(0xffffffffu, odd);
          if (odd) {
            uint32_t mask[4] = {0, 0, 0, 0};
#pragma unroll 1
            for (int c = 0; c < HD / 8; ++c) {
              const uint32_t at = row + (c >> 3) * kTfChunk + (((c & 7) ^ (r & 7)) << 4);
#pragma unroll 1
              for (int e = 0; e < 8; ++e)
                if ((lds_u16(at + 2 * e) & 0x7f80u) == 0x7f80u) {
                  const int d = c * 8 + e;
                  mask[0] |= d < 32 ? 1u << (d & 31) : 0u;
                  mask[1] |= (d >> 5) == 1 ? 1u << (d & 31) : 0u;
                  mask[2] |= (d >> 5) == 2 ? 1u << (d & 31) : 0u;
                  mask[3] |= (d >> 5) == 3 ? 1u << (d & 31) : 0u;
                  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + 2 * e), "h"((uint16_t)0) : "memory");
                }
            }
            const int slot = bad + __popc(who & ((1u << lane) - 1u));
            if (slot < kTfBadRows) {
              list[slot * kTfBadWords] = (uint32_t)(t * 128 + r);
#pragma unroll
              for (int e = 0; e < 4; ++e) list[slot * kTfBadWords + 1 + e] = mask[e];
            }
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
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTfRegsHigh));
    // ------------------------------------------------ softmax + epilogue of slot X
    const int X = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_addr + (uint32_t)(X * 128);
    const uint32_t tO = tmem + lane_addr + 256 + (uint32_t)(X * 128);
    uint32_t base_a = 0, base_b = 0;  // tiles of slot A / B in the items before
    uint32_t n_o = 0;           // items of this slot that had tiles

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
    TfItem it, nx;
    bool ok = true;
    bool have = take_item(0, it);
    if (have) load_q(it);
    for (int n = 0; have; ++n) {
      const int a0 = it.lo(X), a1 = it.hi(X);
      const bool live = r < tp.tt * p.group && it.tok0 + X * tp.tt + my_tok < it.lq;
      const int tok = live ? it.tok0 + X * tp.tt + my_tok : 0;
      const int head = it.h * p.group + my_g;
      bool q_sent = false;
      const int hi = live ? (p.causal ? max(0, min(it.lk, tok + it.lk - it.lq + 1)) : it.lk) : 0;
      const int lo = p.window > 0 ? max(0, tok + it.lk - it.lq - p.window + 1) : 0;
      float m = -INFINITY, l = 0.f;
      for (int t = a0; t < a1; ++t) {
        if (!mbar_wait(bar(kBTfSFull + X), ((X ? base_b : base_a) + (uint32_t)(t - a0)) & 1, p.err, kDevTimeoutSoftmax, abort_flag)) {
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
        float v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, *reinterpret_cast<float(*)[32]>(v + c * 32));
        tmem_wait_ld();
        if (it.masked(t)) {
          const int lim = hi - t * 128, from = lo - t * 128;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= lim || i < from) v[i] = -INFINITY;
        }
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
        // The exponentials of the two slots take turns: together they would share the MUFU pipe
        // while the tensor pipe idles. A tile the other slot does not have is not waited for.
        // (Only a matter of speed: the wait is bounded and needs no order.)
        {
          const int to = X == 0 ? t - 1 : t;  // the other slot's tile that goes before
          if (to >= it.lo(X ^ 1) && to < it.hi(X ^ 1)) {
            const int want = 4 * ((int)(X ? base_a : base_b) + to - it.lo(X ^ 1) + 1);
            for (int i = 0; i < 512 && *reinterpret_cast<volatile int*>(turns + (X ^ 1)) - want < 0; ++i) {}
          }
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
          if (c == 3) {
            __syncwarp();
            if (lane == 0) atomicAdd(turns + X, 1);
          }
          tmem_wait_st();  // this quarter of P is in TMEM: its products may start
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBTfPFull + X * 4 + c));
        }
        const float2 u = __fadd2_rn(__fadd2_rn(rs[0], rs[1]), __fadd2_rn(rs[2], rs[3]));
        l = l * alpha + (u.x + u.y);
      }
      base_a += (uint32_t)max(0, it.a1 - it.a0);
      base_b += (uint32_t)max(0, it.b1 - it.b0);
      // the next item's Q goes in first: its products then run while this item's rows are written
      have = ok && take_item(n + 1, nx);
      if (have && !q_sent) load_q(nx);
      const bool any = a1 > a0;
      if (ok && any) ok = mbar_wait(bar(kBTfOFull + X), n_o & 1, p.err, kDevTimeoutSoftmax, abort_flag);
      n_o += any ? 1 : 0;
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const int bad = any ? *reinterpret_cast<volatile int*>(&items[n % kTfItems].bad) : 0;
      __nv_bfloat16* orow = p.out + ((int64_t)it.q0 + tok) * p.out_stride + (int64_t)head * HD;
      const uint32_t* list =
          tp.bad_rows + ((int64_t)blockIdx.x * kTfItems + n % kTfItems) * (int64_t)kTfBadRows * kTfBadWords;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float o[32];
        if (any) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (bad) {  // non-finite values of V that this row does see
          uint32_t hit = 0;
#pragma unroll 1
          for (int e = 0; e < min(bad, kTfBadRows); ++e) {
            const int key = (int)__ldcg(list + e * kTfBadWords);
            if (key >= lo && key < hi) hit |= __ldcg(list + e * kTfBadWords + 1 + c);
          }
          if (bad > kTfBadRows) hit = 0xffffffffu;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (hit >> i & 1u) o[i] = __int_as_float(0x7fc00000);
        }
        if (ok && live && WX_IN_BOUNDS(p.err, it.q0 + tok < p.total_q)) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            *reinterpret_cast<uint4*>(orow + c * 32 + i) =
                make_uint4(pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv),
                           pack_bf16x2(o[i + 4] * inv, o[i + 5] * inv), pack_bf16x2(o[i + 6] * inv, o[i + 7] * inv));
        }
      }
      if (ok && live && p.lse)
        p.lse[((int64_t)it.q0 + tok) * p.hq + head] =
            l == 0.f ? -INFINITY : (m * p.sl2 + log2f(l)) * 0.69314718055994531f;
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && any) mbar_arrive(bar(kBTfOEmpty + X));
      drop_item(n);
      it = nx;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
static int launch_flash(wx_ctx* ctx, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, TfParams& tp) {
  auto fn = text_flash_kernel<HD>;
  int st = ensure_smem_attr(ctx, (const void*)fn, TfGeom<HD>::kSmem, "text_flash");
  if (st) return st;
  // setmaxnreg moves registers within what the launch reserved
  static const bool regs_ok = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, (const void*)text_flash_kernel<HD>) == cudaSuccess &&
           fa.numRegs * kTfThreads >= kTfRegsLow * 128 + kTfRegsHigh * 256;
  }();
  if (!regs_ok) return set_error(ctx, WX_ERR_CUDA, "text_flash: register split does not fit");
  const TextAttnParams& p = tp.a;
  const int64_t items = (int64_t)p.hkv * (p.total_q / (2 * tp.tt) + p.batch);
  const int grid = (int)std::min<int64_t>(ctx->num_sms, items);
  void* ws = workspace(ctx, (size_t)ctx->num_sms * kTfItems * kTfBadRows * kTfBadWords * 4, &st);
  if (!ws) return st;
  tp.bad_rows = static_cast<uint32_t*>(ws);
  if (!(tp.next = arrival_counters(ctx, 2, &st))) return st;
  ProfScope prof(ctx, kProfAttn);
  fn<<<grid, kTfThreads, TfGeom<HD>::kSmem, ctx->stream>>>(tq, tk, tv, tp);
  return launch_status(ctx, "text_flash");
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
  if ((st = make_tmap_bf16_2d(ctx, &tk, kv.k, kv.rows, kv.cols, kv.k_stride, 64, tp.box))) return st;
  if ((st = make_tmap_bf16_2d(ctx, &tv, kv.v, kv.rows, kv.cols, kv.v_stride, 64, tp.box))) return st;
  return head_dim == 128 ? launch_flash<128>(ctx, tq, tk, tv, tp) : launch_flash<64>(ctx, tq, tk, tv, tp);
}

}  // namespace wx
