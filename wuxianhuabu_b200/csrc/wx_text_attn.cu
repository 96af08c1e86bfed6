// wx_text_attn.cu — attention of the text side: packed causal prompts with grouped heads, and
// new tokens over the paged (optionally 8-bit) K/V cache.
//
// The query rows of one K/V head of a sequence are flattened to rows r = token * G + g (G
// query heads share the K/V head), so a tile of rows shares every K/V byte it reads.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "wx_text_dev.cuh"

namespace wx {

// C[16 x 8] += A[16 x 16] B[16 x 8], bf16, fp32 accumulators. Lane (g, t) = (lane / 4, lane % 4)
// holds C rows g (c0, c1) and g + 8 (c2, c3), columns 2t and 2t + 1; A rows g (a0, a2) and g + 8
// (a1, a3), columns 2t.. (a0, a1) and 2t + 8.. (a2, a3); B column g, rows 2t.. (b0) and 2t + 8.. (b1).
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of bf16, lane (g, t) holding row g, columns 2t and 2t + 1, transposed
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 16 bytes (4: plain) from global to shared memory, in the thread's open group of copies
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most N of the thread's groups are open
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------- few query rows: text_rows_attn_kernel
// For decoding and for a few new tokens: 8 NT flattened query rows share a walk over the keys. So
// few rows against 128-wide heads are a few FLOP per K/V byte, far below the ridge: the walk is
// bound by the K/V bytes, and what has to be kept small beside them is the work per key. The
// products are therefore turned round, the 16 keys of a step being the tensor tile's rows and the
// query rows its columns (S^T = K Q^T, O^T += V^T P^T): no tile row is padding, a lane's K and V
// scales are two numbers, and sums take 32 NT / (128 / HD) registers instead of twice that.
//
// Each warp keeps several steps in flight in a ring of its own, filled by 16-byte copies whose lanes
// lie side by side in memory (copies of half lines, each lane its own operands, cost a third more
// at bf16); 8-bit values become bf16 in registers, exactly. The keys and head columns of a step are
// dealt to the fragments in the order in which they lie in memory: a dot product does not care for
// the order of its terms, so q and K (head columns) and P and V (keys) are permuted alike, and the
// head columns of O^T are put in order when they are written. (A ring of TMA boxes per warp spent a
// third of each step on issuing its copies; one ring for the CTA, and tcgen05 with the keys as 128
// rows, were slower still on 8-bit caches.)
//
// A CTA's warps take 16-key steps of its key range in turn, each with its own running maximum and
// denominator; they are joined once, at the end of the range. Work is split evenly: the (sequence,
// K/V head, row tile) items, each cut into units of 128 keys, form one line of units that is divided
// into equal runs, one per CTA. A CTA whose run covers part of an item leaves its partial sums; the
// last to arrive joins them in key order (so the result does not depend on who is last).
//
// kChunkKeys (own keys behind a shared prefix, many short sequences): units of `chunk` keys go to single
// warps, on demand, and each leaves its sums as a layer for prefix_join_kernel. No warp waits for another, where
// a piece per CTA costs its search, loads and join in turn: 64 sequences of 1 to 701 bf16 keys behind 8,011 that they
// share, 32 / 8 heads of 128, 77 us by pieces, 42 by chunks of 112 (64: 43, 128: 41, 256: 48).
//
// Measured, caches flushed from L2: 64 sequences, 32 / 8 heads of 128, 238,000 bf16 keys 191 us =
// 5.4 TB/s (6.2 TB/s a further key); one sequence, 64 / 8 heads, 65,537 int8 keys 42 us = 3.3 TB/s, e4m3
// 41 (the expansion's instructions are the bound: issue slots 53 % busy, DRAM 34 %; the start and the
// join are a third of it); a call with a few keys 11 us, of which 7 on the device.
constexpr int kUnit = 128;
constexpr uint64_t kMaxUnits = 0xf0000000u;  // of a line: its end and one CTA's run more are below 2^32

template <int FMT, int HD, int NT>
struct RowsGeom {
  static constexpr bool kWide = FMT != kKvBf16;  // 8-bit rows
  // as many warps as registers (8-bit: 12 against 16, 51 : 51 us) and ring stages (bf16: 10 against
  // 8, 191 : 196 us) allow; 16 rows take twice the registers
  static constexpr int kWarps = NT == 1 ? (kWide ? 12 : 10) : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRows = 8 * NT;
  static constexpr int kUnits16 = kWide ? HD / 64 : HD / 32;  // 16-byte units of a key that a lane reads
  static constexpr int kPitch = HD + 4;
  static constexpr int kJoin = kWarps * kRows * (kPitch + 2) * 4 + 64;
  // a step's keys, values (and scales), and as many steps in flight as shared memory holds, up to 6
  static constexpr int kKvBytes = 16 * HD * (kWide ? 1 : 2);
  static constexpr int kStep = 2 * kKvBytes + (kWide ? 128 : 0);
  static constexpr int kFit = (227 * 1024 - kJoin) / (kWarps * kStep);
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kSmem = kWarps * kStages * kStep + kJoin;
};

template <int FMT, int HD, int NT, int KEYS>
__global__ void __launch_bounds__(RowsGeom<FMT, HD, NT>::kThreads, 1)
    text_rows_attn_kernel(const uint8_t* __restrict__ k_base, const uint8_t* __restrict__ v_base, int64_t k_stride,
                          int64_t v_stride, TextAttnParams p, int min_units) {
  using G = RowsGeom<FMT, HD, NT>;
  constexpr bool kW = G::kWide;
  constexpr bool kSolo = KEYS == kChunkKeys;  // a unit is one warp's
  constexpr int kWarps = G::kWarps, kRows = G::kRows, kU = G::kUnits16;
  constexpr int kMT = HD / 16;                 // 16-column tiles of O^T
  constexpr int kRowBytes = kW ? HD : HD * 2;
  constexpr int kD = G::kStages;
  extern __shared__ uint4 smem_raw[];          // [warp][stage][step]
  // [warp][row][pitch], then [warp][row](maximum, denominator)
  float* join = reinterpret_cast<float*>(smem_raw) + kWarps * kD * G::kStep / 4;
  float* join_ml = join + kWarps * kRows * G::kPitch;
  int* last_flag = reinterpret_cast<int*>(join_ml + kWarps * kRows * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)(warp * kD * G::kStep);

  // behind a prefix: where it is shared, the rows of all sequences over its keys come first
  constexpr bool kBehind = KEYS >= kPrefixKeys;
  const int front = kBehind && p.shared ? 1 : 0;
  auto seq_of = [&](int b) -> Seq {
    if (kBehind && b < front) return Seq{0, 0, (int)p.total_q, p.prefix};
    return load_seq(p, kBehind ? b - front : b);
  };
  auto hi_of = [&](int b, const Seq& s, int tok) -> int { return kBehind && b < front ? s.lk : key_hi(p, s, tok); };
  auto blocks_of = [&](int b) -> const int32_t* {
    if constexpr (kBehind) return b < front ? p.prefix_blocks : p.block_table + (b - front) * p.table_stride;
    return p.block_table + b * p.blocks_per_seq;
  };

  // ---- the line of units, walked 32 sequences at a time by each warp for itself (32-bit
  // arithmetic: 64-bit divisions were most of a short call's start)
  // (k16: first key; with first keys that stay visible, the 16-key steps before the window)
  auto line_of = [&](int b, unsigned& items, unsigned& nu, int& k16) {
    items = nu = 0;
    k16 = 0;
    if (b >= p.batch) return;
    const Seq s = seq_of(b);
    k16 = key_lo(p, s, 0) & ~15;
    items = ((unsigned)(s.lq * p.group) + kRows - 1) / kRows * (unsigned)p.hkv;
    const int skip = KEYS == kSinkKeys ? key_gap<KEYS>(p, k16 >> 4, 16).gap << 4 : k16;
    nu = kSolo ? (unsigned)chunks_of(p.chunk, p.chunks, s.lk) : (unsigned)max(1, (s.lk - skip + kUnit - 1) / kUnit);
  };
  unsigned my_items = 0, my_nu = 0;  // of sequence loaded + lane
  int my_k16 = 0, loaded = -1;
  uint64_t mine = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    line_of(b0 + lane, my_items, my_nu, my_k16);
    loaded = b0;
    mine += (uint64_t)my_items * my_nu;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  // (a line beyond 32 bits takes sequences of many query rows, which this kernel is not chosen for unless
  // the caller's longest length was far too small: an error, not rows left out)
  unsigned total = (unsigned)mine;
  if (mine > kMaxUnits) {
    set_dev_error(p.err, kDevBadArgs);
    total = 0;
  }
  const unsigned per = max((unsigned)min_units, (total + gridDim.x - 1) / gridDim.x);
  // (kSolo: units are handed out on demand. Beside the shared walk CTAs begin late: nothing is set apart for them)
  const unsigned apart = kSolo && !p.after_walk ? gridDim.x * kWarps : 0;
  auto take_unit = [&]() -> unsigned { return lane == 0 ? apart + (unsigned)atomicAdd(p.counters, 1) : 0u; };
  unsigned u = !kSolo ? min(total, blockIdx.x * per)
               : apart ? blockIdx.x + gridDim.x * warp
                       : __shfl_sync(0xffffffffu, take_unit(), 0);
  const unsigned u_end = kSolo ? total : min(total, u + per);

  int wb = 0;               // sequences before wb hold
  unsigned wu = 0, wi = 0;  // this many units and items
  struct Piece {
    Seq s;
    int b, h, rt;
    unsigned item, item_u0, nu;  // the item, its first unit and its units
    unsigned u_in;               // its first unit of the item
    int k_lo, k_hi;              // keys of this piece (k_lo a multiple of 16), without those in the gap
    KeyGap at16;                 // of 16-key steps
    int steps;                   // 16-key steps of this piece for this warp
  };
  // the sequence found last: its first unit and item, the end of its units, its row tiles and first key
  unsigned b_u0 = 0, b_end = 0, b_i0 = 0, rts = 1;
  int k16 = 0;
  auto piece_at = [&](unsigned at, Piece& c) -> unsigned {
    while (at >= b_end) {
      if (loaded != wb) {
        line_of(wb + lane, my_items, my_nu, my_k16);
        loaded = wb;
      }
      const unsigned n = my_items * my_nu;
      unsigned nc = n, ic = my_items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned a = __shfl_up_sync(0xffffffffu, nc, o), e = __shfl_up_sync(0xffffffffu, ic, o);
        if (lane >= o) {
          nc += a;
          ic += e;
        }
      }
      const unsigned all = __shfl_sync(0xffffffffu, nc, 31);
      if (at < wu + all) {
        const int src = __ffs(__ballot_sync(0xffffffffu, at < wu + nc)) - 1;
        c.b = wb + src;
        b_u0 = wu + __shfl_sync(0xffffffffu, nc - n, src);
        b_end = wu + __shfl_sync(0xffffffffu, nc, src);
        b_i0 = wi + __shfl_sync(0xffffffffu, ic - my_items, src);
        c.s = seq_of(c.b);
        rts = __shfl_sync(0xffffffffu, my_items, src) / (unsigned)p.hkv;
        c.nu = __shfl_sync(0xffffffffu, my_nu, src);
        k16 = __shfl_sync(0xffffffffu, my_k16, src);
        break;
      }
      wu += all;
      wi += __shfl_sync(0xffffffffu, ic, 31);
      wb += 32;
    }
    const unsigned i = (at - b_u0) / c.nu, u_in = (at - b_u0) - i * c.nu;
    c.h = (int)(i / rts);
    c.rt = (int)(i % rts);
    c.item = b_i0 + i;
    c.item_u0 = b_u0 + i * c.nu;
    const unsigned units = kSolo ? 1 : min(c.nu - u_in, u_end - at);
    c.u_in = u_in;
    c.at16 = key_gap<KEYS>(p, k16 >> 4, 16);
    const int unit = kSolo ? chunk_of(p.chunk, p.chunks, c.s.lk) : kUnit;
    c.k_lo = (KEYS == kSinkKeys ? 0 : k16) + (int)u_in * unit;
    c.k_hi = min(c.s.lk - (c.at16.gap << 4), c.k_lo + (int)units * unit);
    const int n16 = max(0, (c.k_hi - c.k_lo + 15) / 16);
    c.steps = kSolo ? n16 : n16 > warp ? (n16 - warp + kWarps - 1) / kWarps : 0;
    return units;
  };

  // ---- loads: step i of this warp starts at key k_lo + (i * kWarps + warp) * 16; the pages of 32
  // consecutive steps are fetched at once, one per lane
  const bool paged = kW || p.block_table;
  [[maybe_unused]] const int64_t kv_rows = paged ? (p.pages * p.hkv) << p.page_shift : p.total_k;
  int page_of = 0;
  // (without a sign: steps that a piece near 2^31 keys does not have may lie beyond)
  auto step_key = [&](const Piece& c, int i) {
    return (int)((unsigned)c.k_lo + (unsigned)(kSolo ? i : i * kWarps + warp) * 16u);
  };
  auto first_key = [&](const Piece& c, int i) {
    const int j = step_key(c, i);
    return KEYS == kSinkKeys ? c.at16(j >> 4) << 4 : j;
  };
  // row of the step's first key: of the cache, or of the packed keys
  auto step_row = [&](const Piece& c, int i) -> int64_t {
    const int j0 = first_key(c, i);
    if (!paged) return c.s.k0 + j0;
    if ((i & 31) == 0) {
      const int jl = first_key(c, i + lane);
      page_of = 0;
      if ((unsigned)step_key(c, i + lane) < (unsigned)c.k_hi) {
        page_of = blocks_of(c.b)[jl >> p.page_shift];
        if (page_of < 0 || page_of >= p.pages) {
          set_dev_error(p.err, kDevBadArgs);
          page_of = 0;
        }
      }
    }
    const int page = __shfl_sync(0xffffffffu, page_of, i & 31);
    return (((int64_t)page * p.hkv + c.h) << p.page_shift) | (j0 & ((1 << p.page_shift) - 1));
  };
  // A step's rows are copied whole, 16 bytes a lane, the lanes of a copy side by side in memory. Their
  // 16-byte units are swizzled such that the eight lanes of a read's phase, two rows of K by four
  // units or four even rows of V by two, meet eight groups of banks. One group of copies per step; steps that a
  // piece does not have are empty groups. (packed keys: rows past the sequence's last are not read,
  // the last one stands in; a page is whole)
  constexpr int kRU = kRowBytes / 16;   // units of a row
  constexpr int kVN = kW ? 1 : HD / 64; // V units of a row that a lane reads
  auto k_swz = [](int row) { return kRU == 4 ? 0 : (row & 1) << 2; };
  auto v_swz = [](int row) { return kRU == 4 ? (row >> 1) & 3 : row & 6; };
  const float* scale_at = kW ? (lane < 16 ? p.ks : p.vs) + (lane & 15) : nullptr;
  auto load_step = [&](const Piece& c, int i, uint32_t stage) {
    const int left = paged || i >= c.steps ? 15 : c.s.lk - 1 - first_key(c, i);
    const int64_t row = i < c.steps ? step_row(c, i) : 0;
    if (i < c.steps && WX_IN_BOUNDS(p.err, row >= 0 && left >= 0 && row + min(left, 15) < kv_rows)) {
      // (an 8-bit cache is paged: its 16 rows lie together)
      const int64_t kst = kW ? kRowBytes : k_stride, vst = kW ? kRowBytes : v_stride;
      const int64_t col = (paged ? 0 : (int64_t)c.h * kRowBytes) + lane % kRU * 16;
      const uint8_t* kb = k_base + row * kst + col;
      const uint8_t* vb = v_base + row * vst + col;
#pragma unroll
      for (int x = 0; x < kRU / 2; ++x) {
        const int r = x * (32 / kRU) + lane / kRU;
        copy_async16(stage + (r * kRU + (lane % kRU ^ k_swz(r))) * 16, kb + (int64_t)(kW ? r : min(r, left)) * kst);
      }
#pragma unroll
      for (int x = 0; x < kRU / 2; ++x) {
        const int r = x * (32 / kRU) + lane / kRU;
        copy_async16(stage + G::kKvBytes + (r * kRU + (lane % kRU ^ v_swz(r))) * 16,
                     vb + (int64_t)(kW ? r : min(r, left)) * vst);
      }
      if constexpr (kW) copy_async4(stage + 2 * G::kKvBytes + lane * 4, scale_at + row);  // keys' scales, then values'
    }
    copy_async_commit();
  };
  struct Values {
    uint4 v[4][kVN];
  };
  auto word = [](const uint4& x, int i) -> uint32_t { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; };
  // bf16 pair (keys of rows ra and rb) of this lane's d-th head column
  auto value_pair = [&](const Values& f, int ra, int rb, int d) -> uint32_t {
    if constexpr (kW)
      return bytes_to_bf16x2<FMT>(word(f.v[ra][0], d >> 2), word(f.v[rb][0], d >> 2), d & 3, 4 + (d & 3));
    else
      return __byte_perm(word(f.v[ra][d >> 3], (d & 7) >> 1), word(f.v[rb][d >> 3], (d & 7) >> 1), d & 1 ? 0x7632 : 0x5410);
  };
  // head column of this lane's d-th: the units of lane group g
  auto column = [&](int d) { return kW ? g * (HD / 8) + d : (d >> 3) * 64 + g * 8 + (d & 7); };

  Piece cur;
  uint32_t at_stage = 0;  // stage of the next step to be worked on
  auto next_stage = [&](uint32_t x) { return x + 1 == (uint32_t)kD ? 0u : x + 1; };
  auto first_loads = [&](const Piece& c) {
    uint32_t to = at_stage;
#pragma unroll
    for (int i = 0; i < kD; ++i, to = next_stage(to)) load_step(c, i, ring + to * G::kStep);
  };
  bool have = u < u_end;
  unsigned units = 0;
  if (have) {
    units = piece_at(u, cur);
    first_loads(cur);
  }
  while (have) {
    [[maybe_unused]] const unsigned next_u = kSolo ? take_unit() : 0;
    const int n_rows = cur.s.lq * p.group;
    const int row0 = cur.rt * kRows;
    // ---- q fragments: row 8 n + g, columns in the order of the K reads; the limits of rows 2t, 2t+1
    uint32_t qf[NT][HD / 16][2];
    int lim_hi[NT][2], lim_lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const bool live = r < n_rows && WX_IN_BOUNDS(p.err, cur.s.q0 >= 0 && cur.s.q0 + r / p.group < p.total_q);
      const int tok = live ? (int)((unsigned)r / (unsigned)p.group) : 0;
      const __nv_bfloat16* src = p.q + (cur.s.q0 + tok) * p.q_stride +
                                 (int64_t)(cur.h * p.group + (live ? r - tok * p.group : 0)) * HD;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (live)
          w = __ldg(reinterpret_cast<const uint4*>(src + (kW ? (i >> 1) * 64 + t * 16 + (i & 1) * 8 : i * 32 + t * 8)));
        qf[n][2 * i][0] = w.x;
        qf[n][2 * i][1] = w.y;
        qf[n][2 * i + 1][0] = w.z;
        qf[n][2 * i + 1][1] = w.w;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = row0 + 8 * n + 2 * t + e;
        const bool here = rr < n_rows;
        const int tk = here ? (int)((unsigned)rr / (unsigned)p.group) : 0;
        lim_hi[n][e] = here ? hi_of(cur.b, cur.s, tk) : 0;
        lim_lo[n][e] = here ? key_lo(p, cur.s, tk) : 0;
      }
    }
    // a step between these sees no mask in any row of the tile
    const int last_tok = (int)((unsigned)(min(n_rows, row0 + kRows) - 1) / (unsigned)p.group);
    const int free_hi = hi_of(cur.b, cur.s, (int)((unsigned)row0 / (unsigned)p.group));
    const int free_lo = key_lo(p, cur.s, last_tok);

    float acc[NT][kMT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < kMT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][j][i] = 0.f;
    float m[NT][2], l[NT][2];  // of rows 8 n + 2t + e; l: this lane's keys only
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }

    for (int i = 0; i < cur.steps; ++i, at_stage = next_stage(at_stage)) {
      const uint32_t stage = ring + at_stage * G::kStep;
      copy_async_wait<kD - 1>();
      __syncwarp();
      const int j0 = first_key(cur, i);
      const bool masked = j0 + 16 > free_hi || (j0 < free_lo && (KEYS != kSinkKeys || j0 + 16 > p.sinks));
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
      for (int c = 0; c < kU; ++c) {
        const uint32_t at = stage + (g * kRU + (c * 4 + t ^ k_swz(g))) * 16;
        const uint4 kx = lds128(at), ky = lds128(at + 8 * kRowBytes);
        if constexpr (kW) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = word(kx, e), y = word(ky, e);
            const uint32_t a0 = bytes_to_bf16x2<FMT>(x, 0, 0, 1), a1 = bytes_to_bf16x2<FMT>(y, 0, 0, 1);
            const uint32_t a2 = bytes_to_bf16x2<FMT>(x, 0, 2, 3), a3 = bytes_to_bf16x2<FMT>(y, 0, 2, 3);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(sc[n], a0, a1, a2, a3, qf[n][4 * c + e][0], qf[n][4 * c + e][1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_bf16(sc[n], kx.x, ky.x, kx.y, ky.y, qf[n][2 * c][0], qf[n][2 * c][1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_bf16(sc[n], kx.z, ky.z, kx.w, ky.w, qf[n][2 * c + 1][0], qf[n][2 * c + 1][1]);
        }
      }
      const float k_unit = p.sl2 * kByteUnit<FMT>;
      float f[2] = {k_unit, k_unit}, vs[2] = {1.f, 1.f};  // of keys g and g + 8
      if constexpr (kW) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[e] *= lds_f32(stage + 2 * G::kKvBytes + (e * 8 + g) * 4);
          vs[e] = lds_f32(stage + 2 * G::kKvBytes + 64 + (e * 8 + g) * 4);
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sc[n][q] *= f[q >> 1];
        if (masked) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int j = j0 + g + 8 * (q >> 1);
            if (!key_seen<KEYS>(p, j, lim_lo[n][q & 1], lim_hi[n][q & 1])) sc[n][q] = -INFINITY;
          }
        }
        // The maximum is moved only when it has grown by 2^8: most steps leave O^T alone and take no
        // more than a vote, and the weights stay below 2^8, far from fp32's and bf16's range
        const float mx[2] = {fmaxf(sc[n][0], sc[n][2]), fmaxf(sc[n][1], sc[n][3])};
        auto grown = [&](int e) { return mx[e] > m[n][e] + 8.f || (m[n][e] == -INFINITY && mx[e] > -INFINITY); };
        if (__any_sync(0xffffffffu, grown(0) || grown(1))) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = mx[e];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            x = fmaxf(x, m[n][e]);
            alpha[e] = x == -INFINITY ? 1.f : exp2_approx(m[n][e] - x);
            m[n][e] = x;
            l[n][e] *= alpha[e];
          }
#pragma unroll
          for (int j = 0; j < kMT; ++j) {
            acc[n][j][0] *= alpha[0];
            acc[n][j][1] *= alpha[1];
            acc[n][j][2] *= alpha[0];
            acc[n][j][3] *= alpha[1];
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m[n][e] == -INFINITY ? 0.f : m[n][e];
          const float x0 = exp2_approx(sc[n][e] - mu), x1 = exp2_approx(sc[n][2 + e] - mu);
          l[n][e] += x0 + x1;
          float w0 = x0, w1 = x1;
          if constexpr (kW) {
            w0 *= vs[0];
            w1 *= vs[1];
            if (masked) {  // an unseen key's scale may be anything: its weight is 0, not 0 * scale
              if (sc[n][e] == -INFINITY) w0 = 0.f;
              if (sc[n][2 + e] == -INFINITY) w1 = 0.f;
            }
          }
          sc[n][e] = w0;
          sc[n][2 + e] = w1;
        }
        // P rounded to bf16 for the tensor product, which takes both operands in V's type (the denominator sums the
        // unrounded values): up to 2^-8 of each weight, which partly cancels over the keys. Relative to 64 bits a row is
        // off by 0.0019 to 0.0024, where weights kept in fp32 leave 0.0016, the output's own rounding.
        pb[n][0] = transpose_8x8(pack_bf16x2(sc[n][0], sc[n][1]));
        pb[n][1] = transpose_8x8(pack_bf16x2(sc[n][2], sc[n][3]));
      }
      Values vf;
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
#pragma unroll
        for (int e = 0; e < kVN; ++e) {
          const int r = 2 * t + (rr & 1) + (rr >> 1) * 8;
          const uint32_t at = stage + G::kKvBytes + r * kRowBytes;
          if constexpr (kRU > 4) {
            vf.v[rr][e] = lds128(at + ((e * 8 + g) ^ v_swz(r)) * 16);
          } else {
            const uint2 x = lds64(at + ((g >> 1) ^ v_swz(r)) * 16 + (g & 1) * 8);
            vf.v[rr][e] = make_uint4(x.x, x.y, 0, 0);
          }
        }
      bool slow = false;
      if constexpr (FMT == kKvE4m3) {
        if (masked) {
          // NaN codes of values that only some rows see: zero in the products, NaN in their columns of the
          // rows that do see them (int8 has none; a NaN scale is the weight's, and that is 0 where unseen)
          uint32_t codes[4], odd = 0;  // of this lane's keys, a bit a column
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            uint4& x = vf.v[rr][0];
            codes[rr] = nan_code_mask(x.x) | nan_code_mask(x.y) << 4;
            if constexpr (HD == 128) codes[rr] |= nan_code_mask(x.z) << 8 | nan_code_mask(x.w) << 12;
            odd |= codes[rr];
          }
          if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
            for (int rr = 0; rr < 4; ++rr) {
              uint4& x = vf.v[rr][0];
              x = make_uint4(without_nan_codes(x.x), without_nan_codes(x.y), without_nan_codes(x.z),
                             without_nan_codes(x.w));
            }
#pragma unroll 1
            for (int kk = 0; kk < 16; ++kk) {
              const int from = g * 4 + ((kk & 7) >> 1), rr = (kk & 1) + 2 * (kk >> 3), j = j0 + kk;
              const uint32_t mine = rr == 0 ? codes[0] : rr == 1 ? codes[1] : rr == 2 ? codes[2] : codes[3];
              const uint32_t x = __shfl_sync(0xffffffffu, mine, from);
#pragma unroll
              for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if ((x >> d & 1u) && key_seen<KEYS>(p, j, lim_lo[n][e], lim_hi[n][e]))
                      acc[n][d >> 1][2 * (d & 1) + e] = __int_as_float(0x7fc00000);
            }
          }
        }
      }
      if constexpr (!kW) {
        if (masked) {
          // 0 * NaN is NaN: keys past the end are zeroed; with a non-finite value at a key that only
          // some rows see, this step's products go by scalar sums
          bool odd = false;
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const bool past = j0 + 2 * t + (rr & 1) + (rr >> 1) * 8 >= cur.s.lk;
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
              if (past) vf.v[rr][e] = make_uint4(0, 0, 0, 0);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint32_t x = word(vf.v[rr][e], q);
                odd |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
              }
            }
          }
          slow = __any_sync(0xffffffffu, odd);
          if (slow) {
#pragma unroll 1
            for (int kk = 0; kk < 16; ++kk) {
              const int from = g * 4 + ((kk & 7) >> 1), rr = (kk & 1) + 2 * (kk >> 3);
              const int j = j0 + kk;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float w[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  w[e] = round_bf16(__shfl_sync(0xffffffffu, kk < 8 ? sc[n][e] : sc[n][2 + e], (kk & 7) * 4 + t));
#pragma unroll
                for (int d = 0; d < HD / 8; ++d) {
                  uint32_t mine = 0;
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    if (q == rr) mine = word(vf.v[q][d >> 3], (d & 7) >> 1);
                  // (every lane offers its row rr; the wanted key is that of lane `from`)
                  const uint32_t x = __shfl_sync(0xffffffffu, mine, from);
                  const float v = d & 1 ? bf16_hi(x) : bf16_lo(x);
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (key_seen<KEYS>(p, j, lim_lo[n][e], lim_hi[n][e])) acc[n][d >> 1][2 * (d & 1) + e] += w[e] * v;
                }
              }
            }
          }
        }
      }
      if (!slow) {
#pragma unroll
        for (int j = 0; j < kMT; ++j) {
          const uint32_t a0 = value_pair(vf, 0, 1, 2 * j), a1 = value_pair(vf, 0, 1, 2 * j + 1);
          const uint32_t a2 = value_pair(vf, 2, 3, 2 * j), a3 = value_pair(vf, 2, 3, 2 * j + 1);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_bf16(acc[n][j], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      }
      __syncwarp();  // the stage has been read
      load_step(cur, i + kD, stage);
    }

    // ---- the next piece's first loads go out before this one is joined
    const Piece done = cur;
    const unsigned u_done = u;
    u = kSolo ? __shfl_sync(0xffffffffu, next_u, 0) : u + units;
    have = u < u_end;
    if (have) {
      units = piece_at(u, cur);
      first_loads(cur);
    }

    if constexpr (kSolo) {
      const int64_t layer = (done.b < front ? 0 : p.own_layer) + (int64_t)done.u_in;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[n][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
          const int r = row0 + 8 * n + 2 * t + e;
          if (r >= n_rows) continue;
          const int tk = (int)((unsigned)r / (unsigned)p.group);
          const int64_t tok = done.s.q0 + tk;
          const int head = done.h * p.group + r - tk * p.group;
          if (!WX_IN_BOUNDS(p.err, tok >= 0 && tok < p.total_q && head >= 0 && head < p.hq && layer < p.layers)) continue;
          const int64_t at = layer * (p.total_q * p.hq) + tok * p.hq + head;
          if (g == 0) p.layer_ml[at] = make_float2(m[n][e], x);
          if (done.steps == 0) continue;  // (nothing seen: the sums are not looked at)
          float* dst = p.layer_o + at * HD;
          constexpr float kB = kByteUnit<FMT>;
#pragma unroll
          for (int d = 0; d < HD / 8; d += 4)
            *reinterpret_cast<float4*>(dst + column(d)) = make_float4(
                acc[n][d >> 1][e] * kB, acc[n][d >> 1][2 + e] * kB, acc[n][(d >> 1) + 1][e] * kB, acc[n][(d >> 1) + 1][2 + e] * kB);
        }
      continue;
    }
    // ---- join the warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        const int row = warp * kRows + 8 * n + 2 * t + e;
        if (g == 0) *reinterpret_cast<float2*>(join_ml + row * 2) = make_float2(m[n][e], x);
        if (done.steps > 0) {
          float* dst = join + row * G::kPitch;
#pragma unroll
          for (int d = 0; d < HD / 8; d += 4)
            *reinterpret_cast<float4*>(dst + column(d)) =
                make_float4(acc[n][d >> 1][e], acc[n][d >> 1][2 + e], acc[n][(d >> 1) + 1][e], acc[n][(d >> 1) + 1][2 + e]);
        }
      }
    __syncthreads();
    const bool whole = u_done <= done.item_u0 && u >= done.item_u0 + done.nu;
    const unsigned c0 = done.item_u0 / per, c1 = (done.item_u0 + done.nu - 1) / per;  // CTAs of this item
    constexpr int kPer = HD / 16;  // columns of a thread, 16 threads to a row
    constexpr int kGroups = 2 * kWarps / kRows;  // groups of threads that cover the rows
    const int jr = (threadIdx.x >> 4) % kRows, jg = (threadIdx.x >> 4) / kRows, jc = (threadIdx.x & 15) * kPer;
    float o[kPer] = {};
    float M = -INFINITY, L = 0.f;
    auto add = [&](const float4& x, int i, float f) {
      o[i] += x.x * f;
      o[i + 1] += x.y * f;
      o[i + 2] += x.z * f;
      o[i + 3] += x.w * f;
    };
    auto clear = [&]() {
      M = -INFINITY;
      L = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] = 0.f;
    };
    auto write = [&]() {
      const int r = done.rt * kRows + jr;
      if (r >= done.s.lq * p.group) return;
      const int tk = (int)((unsigned)r / (unsigned)p.group);
      const int64_t tok = done.s.q0 + tk;
      const int head = done.h * p.group + r - tk * p.group;
      if (!WX_IN_BOUNDS(p.err, tok >= 0 && tok < p.total_q && head >= 0 && head < p.hq)) return;
      if constexpr (kBehind) {
        const int64_t at = (done.b < front ? 0 : p.own_layer) * (p.total_q * p.hq) + tok * p.hq + head;
#pragma unroll
        for (int i = 0; i < kPer; i += 4)
          *reinterpret_cast<float4*>(p.layer_o + at * HD + jc + i) =
              make_float4(o[i] * kByteUnit<FMT>, o[i + 1] * kByteUnit<FMT>, o[i + 2] * kByteUnit<FMT>, o[i + 3] * kByteUnit<FMT>);
        if ((threadIdx.x & 15) == 0) p.layer_ml[at] = make_float2(M, L);
        return;
      }
      const float inv = L == 0.f ? 0.f : kByteUnit<FMT> / L;
      uint32_t w[kPer / 2];
#pragma unroll
      for (int i = 0; i < kPer; i += 2) w[i / 2] = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
      __nv_bfloat16* dst = p.out + tok * p.out_stride + (int64_t)head * HD + jc;
      if constexpr (kPer == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      if (p.lse && (threadIdx.x & 15) == 0)
        p.lse[tok * p.hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
    };
    // partial sums of CTA c for this item: slot 0 if the item began in an earlier CTA, 1 if there
    auto slot_row = [&](unsigned c, int row) -> int64_t {
      const int64_t at = (int64_t)(2 * c + (done.item_u0 >= c * per ? 1 : 0)) * kRows + row;
      return WX_IN_BOUNDS(p.err, at >= 0 && at < 2 * (int64_t)gridDim.x * kRows) ? at : 0;
    };
    if (jg == 0) {
      clear();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, join_ml[(w * kRows + jr) * 2]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = *reinterpret_cast<const float2*>(join_ml + (w * kRows + jr) * 2);
        if (ml.y == 0.f) continue;
        const float f = exp2_approx(ml.x - M);
        L += ml.y * f;
#pragma unroll
        for (int i = 0; i < kPer; i += 4)
          add(*reinterpret_cast<const float4*>(join + (w * kRows + jr) * G::kPitch + jc + i), i, f);
      }
      if (whole) {
        write();
      } else {
        const int64_t at = slot_row(blockIdx.x, jr);
#pragma unroll
        for (int i = 0; i < kPer; i += 4)
          *reinterpret_cast<float4*>(p.part + at * HD + jc + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        if ((threadIdx.x & 15) == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        // (sequences that overlap in cu_q could count more items than there are counters)
        const bool known = (int64_t)done.item < p.n_items;
        const int before = known ? atomicAdd(p.counters + done.item, 1) : -1;
        *last_flag = before == (int)(c1 - c0);
        if (*last_flag) p.counters[done.item] = 0;
        if (!known) set_dev_error(p.err, kDevBadArgs);
      }
      __syncthreads();
      if (*last_flag) {
        // All pieces' maxima and denominators at once, then the thread groups share the pieces, four
        // in flight each: one after the other, the latency of 20 pieces was 11 us of a call.
        __threadfence();
        const int n = (int)(c1 - c0) + 1;
        for (int i = threadIdx.x; i < n * kRows; i += G::kThreads)
          *reinterpret_cast<float2*>(join + 2 * i) =
              __ldcg(reinterpret_cast<const float2*>(p.part_ml + slot_row(c0 + i / kRows, i % kRows) * 2));
        __syncthreads();
        clear();
        for (int c = 0; c < n; ++c) M = fmaxf(M, join[2 * (c * kRows + jr)]);
        for (int c = jg < kGroups ? jg : n; c < n; c += 4 * kGroups) {
          float4 x[4][kPer / 4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* src = p.part + slot_row(c0 + min(c + q * kGroups, n - 1), jr) * HD + jc;
#pragma unroll
            for (int i = 0; i < kPer / 4; ++i) x[q][i] = __ldcg(reinterpret_cast<const float4*>(src) + i);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (c + q * kGroups >= n) continue;
            const float2 ml = *reinterpret_cast<const float2*>(join + 2 * ((c + q * kGroups) * kRows + jr));
            if (ml.y == 0.f) continue;
            const float f = exp2_approx(ml.x - M);
            L += ml.y * f;
#pragma unroll
            for (int i = 0; i < kPer; i += 4) add(x[q][i / 4], i, f);
          }
        }
        if constexpr (kGroups > 1) {
          __syncthreads();
          float* mine = join + ((jg * kRows + jr) * 16 + (threadIdx.x & 15)) * (kPer + 1);
          if (jg > 0 && jg < kGroups) {
            mine[kPer] = L;
#pragma unroll
            for (int i = 0; i < kPer; ++i) mine[i] = o[i];
          }
          __syncthreads();
          if (jg == 0) {
#pragma unroll
            for (int w = 1; w < kGroups; ++w) {
              const float* src = mine + w * kRows * 16 * (kPer + 1);
              L += src[kPer];
#pragma unroll
              for (int i = 0; i < kPer; ++i) o[i] += src[i];
            }
          }
        }
        if (jg == 0) write();
      }
    }
    __syncthreads();  // the join buffer is free again
  }
  if constexpr (kSolo) {
    let_next_begin();
    __syncwarp();
    if (lane == 0 && atomicAdd(p.counters + 1, 1) == (int)gridDim.x * kWarps - 1) {
      p.counters[0] = 0;  // nobody asks any more: ready for the next launch
      p.counters[1] = 0;
    }
    wait_for_last();  // (the join is told of this kernel's end alone, and needs the shared walk's too)
  }
}

// --------------------------------------------------------------------- host side
// a launch that may begin before the kernel before it has ended (as soon as that lets it)
template <class... P, class... A>
static int launch_dependent(wx_ctx* ctx, void (*fn)(P...), unsigned grid, unsigned threads, size_t smem, A... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  WX_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...));
  return WX_OK;
}

static int check_dims(wx_ctx* ctx, const wx_attn_dims* d, const void* q, int64_t q_stride, const void* out,
                      int64_t out_stride, const int32_t* cu_q) {
  WX_CHECK_ARG(ctx, ctx && d && d->total_q >= 0 && d->batch >= 0 && d->q_heads > 0 && d->kv_heads > 0);
  WX_CHECK_ARG(ctx, d->q_heads % d->kv_heads == 0 && d->max_q >= 0 && d->window >= 0);
  WX_CHECK_ARG(ctx, d->window == 0 || d->causal);
  WX_CHECK_ARG(ctx, d->scale > 0.f && d->scale < INFINITY);
  if (d->head_dim != 128 && d->head_dim != 64)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "attention head_dim must be 128 or 64 (got %d)", d->head_dim);
  if (d->q_heads / d->kv_heads > 128)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "at most 128 query heads per K/V head");
  // row tiles and items are counted in 32 bits
  if (d->total_q > INT32_MAX || d->total_q * d->q_heads > INT32_MAX)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "total_q * q_heads must be below 2^31");
  if (d->total_q == 0 || d->batch == 0) return WX_OK;
  WX_CHECK_ARG(ctx, q && out && cu_q && aligned16(q) && aligned16(out));
  WX_CHECK_ARG(ctx, q_stride % 8 == 0 && q_stride >= (int64_t)d->q_heads * d->head_dim);
  WX_CHECK_ARG(ctx, out_stride % 8 == 0 && out_stride >= (int64_t)d->q_heads * d->head_dim);
  return WX_OK;
}

static void fill_params(wx_ctx* ctx, const wx_attn_dims* d, const void* q, int64_t q_stride, const int32_t* cu_q,
                        void* out, int64_t out_stride, float* lse, TextAttnParams& p) {
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.lse = lse;
  p.cu_q = cu_q;
  p.batch = d->batch;
  p.hq = d->q_heads;
  p.hkv = d->kv_heads;
  p.group = d->q_heads / d->kv_heads;
  p.total_q = d->total_q;
  p.causal = d->causal != 0;
  p.window = d->window;
  p.sl2 = (float)((double)d->scale * 1.4426950408889634);
  p.max_q = d->max_q;
  p.err = ctx->dev_err;
}

template <int FMT, int HD, int NT, int KEYS>
static int launch_rows_attn(wx_ctx* ctx, TextAttnParams p, const KvSource& kv) {
  using G = RowsGeom<FMT, HD, NT>;
  constexpr bool kSolo = KEYS == kChunkKeys, kBehind = KEYS >= kPrefixKeys;
  // (an item's pieces: the join buffer)
  const int grid = kSolo ? p.ctas : std::min(ctx->num_sms, G::kWarps * (G::kPitch + 2) / 2);
  const int64_t walks = kBehind && p.shared ? 2 : 1;  // of each row
  const int64_t items = (int64_t)p.hkv * (walks * (p.total_q * p.group / G::kRows) + p.batch);
  // the line of units is counted in 32 bits (only block tables that repeat pages get near)
  const int64_t most_keys = std::max<int64_t>(p.blocks_per_seq << p.page_shift, kBehind ? p.prefix : 0);
  if (p.block_table && items > UINT32_MAX / (kSolo ? p.chunks : most_keys / kUnit + 1))
    return set_error(ctx, WX_ERR_UNSUPPORTED, "batch * kv_heads * blocks_per_seq too large (2^32 units of 128 keys)");
  int st;
  auto fn = text_rows_attn_kernel<FMT, HD, NT, KEYS>;
  const int64_t bytes = G::kWide ? 1 : 2;
  const auto *k = static_cast<const uint8_t*>(kv.k), *v = static_cast<const uint8_t*>(kv.v);
  if constexpr (kSolo) {
    // It may begin while the shared walk is at work, on the SMs that this leaves free: what it reads was there before.
    // (counters of its own, beside the walk's)
    if (!(p.counters = arrival_counters(ctx, 16, &st))) return st;
    p.counters += 8;
    constexpr int smem = G::kWarps * G::kStages * G::kStep;
    if ((st = ensure_smem_attr(ctx, (const void*)fn, smem, "text_rows_attn"))) return st;
    ProfScope prof(ctx, kProfAttn);
    const int64_t ks = (int64_t)kv.k_stride * bytes, vs = (int64_t)kv.v_stride * bytes;
    if (p.after_walk) st = launch_dependent(ctx, fn, grid, G::kThreads, smem, k, v, ks, vs, p, 1);
    else fn<<<grid, G::kThreads, smem, ctx->stream>>>(k, v, ks, vs, p, 1);
    return st ? st : launch_status(ctx, "text_rows_attn");
  }
  const size_t rows = (size_t)grid * 2 * G::kRows;
  Carve c{p.ws_reserved};
  const size_t o_part = c.take(rows * HD * 4), o_ml = c.take(rows * 8);
  uint8_t* ws = static_cast<uint8_t*>(workspace(ctx, c.off, &st));
  if (!ws) return st;
  p.part = reinterpret_cast<float*>(ws + o_part);
  p.part_ml = reinterpret_cast<float*>(ws + o_ml);
  p.n_items = items;
  if (!(p.counters = arrival_counters(ctx, items, &st))) return st;
  if ((st = ensure_smem_attr(ctx, (const void*)fn, G::kSmem, "text_rows_attn"))) return st;
  ProfScope prof(ctx, kProfAttn);
  fn<<<grid, G::kThreads, G::kSmem, ctx->stream>>>(k, v, (int64_t)kv.k_stride * bytes, (int64_t)kv.v_stride * bytes, p, 2);
  return launch_status(ctx, "text_rows_attn");
}

template <int FMT, int KEYS>
static int launch_rows_attn(wx_ctx* ctx, int head_dim, int64_t rows, const TextAttnParams& p, const KvSource& kv) {
  if (head_dim == 128)
    return rows <= 8 ? launch_rows_attn<FMT, 128, 1, KEYS>(ctx, p, kv) : launch_rows_attn<FMT, 128, 2, KEYS>(ctx, p, kv);
  return rows <= 8 ? launch_rows_attn<FMT, 64, 1, KEYS>(ctx, p, kv) : launch_rows_attn<FMT, 64, 2, KEYS>(ctx, p, kv);
}

template <int KEYS>
static int launch_rows_attn(wx_ctx* ctx, int head_dim, int64_t rows, const TextAttnParams& p, const KvSource& kv) {
  if (kv.format == kKvInt8) return launch_rows_attn<kKvInt8, KEYS>(ctx, head_dim, rows, p, kv);
  if (kv.format == kKvE4m3) return launch_rows_attn<kKvE4m3, KEYS>(ctx, head_dim, rows, p, kv);
  return launch_rows_attn<kKvBf16, KEYS>(ctx, head_dim, rows, p, kv);
}

// Few flattened rows a sequence (a decoding step, a few drafted tokens) go to the rows kernel, which
// walks the keys once per 16 rows, more to the tcgen05 kernel, which does so once per 256. Rows : tcgen05
// in us:                                                bf16        e4m3        int8
//   32 sequences of 4,000 keys, 32 / 8 x 128, 24 rows   172 : 150   150 : 216   135 : 210
//                                             40 rows   249 : 155   217 : 220   195 : 214
//                                             56 rows   315 : 157   281 : 222   250 : 220
//                               32 / 8 x 64,  24 rows   111 : 132   111 : 191   104 : 189
//                                             40 rows   162 : 134   160 : 194   150 : 193
//                                             56 rows   205 : 136   205 : 196   190 : 195
//   1 sequence of 30,000 keys,  32 / 8 x 128, 24 rows    55 : 56     50 : 77     45 : 75
//                                             40 rows    68 : 56     63 : 77     57 : 75
//   8 sequences of 500 keys,    32 / 8 x 128, 24 rows    16 : 21     16 : 29     14 : 27
//                                             56 rows    33 : 20     31 : 27     31 : 27
//   16 of 8,000, window 700,    8 / 1 x 64,   64 rows    16 : 25     16 : 35     14 : 35
// The bounds are set for many keys at head_dim 128. Where there is little work for the whole card (one
// K/V head, short or windowed keys) the rows kernel stays ahead beyond them, by up to 2.4 times; a rule on
// the amount of work, which is known on the device only, was not tried.
static int dispatch_attn(wx_ctx* ctx, const wx_attn_dims* d, const TextAttnParams& p, const KvSource& kv) {
  const int64_t rows = (int64_t)d->max_q * p.group;
  const int keys = p.window && p.sinks ? kSinkKeys : kPlainKeys;
  if (rows > (kv.format == kKvBf16 ? 16 : kv.format == kKvE4m3 ? 32 : 48)) return text_flash(ctx, p, d->head_dim, kv, keys);
  return keys == kSinkKeys ? launch_rows_attn<kSinkKeys>(ctx, d->head_dim, rows, p, kv)
                           : launch_rows_attn<kPlainKeys>(ctx, d->head_dim, rows, p, kv);
}

// ------------------------------------------------------------------ a prefix that all sequences share
// softmax over the prefix P and the row's own keys S: with o = sum 2^(s - m) v, m and l of each part,
//   M = max(m_P, m_S), out = (2^(m_P - M) o_P + 2^(m_S - M) o_S) / (2^(m_P - M) l_P + 2^(m_S - M) l_S).
// The rows of all sequences walk the prefix together, so that its bytes are read once for up to 256 rows and
// not once for each sequence; their own keys are walked as in any paged call. The parts' sums stay
// in fp32 and are joined here, in the order of the keys.
template <int HD, int R>
__global__ void __launch_bounds__(256) prefix_join_kernel(TextAttnParams p) {
  int head;
  const int64_t token = join_token<R>(p, head);
  const int b = seq_of_token(p, token);
  const bool live = token < p.total_q && token >= p.cu_q[b] && token < p.cu_q[b + 1];
  const int layers = p.own_layer + layers_of(p.chunk, p.chunks, load_seq(p, b).lk);
  wait_for_last();
  if (!live) return;
  const int64_t row0 = token * p.hq + head;
  join_rows<HD, R>(p.layer_o, p.layer_ml, p.total_q * p.hq, row0, min(R, p.hq - head), layers,
                   p.out + token * p.out_stride + (int64_t)head * HD, p.lse ? p.lse + row0 : nullptr);
}

// Few rows a sequence: the prefix is walked for all rows together, by the kernel for few rows where they are few
// in all or the prefix is short, else by the tcgen05 kernel (64 rows over 2,000 bf16 keys, 8 heads, 17.2 us against
// 20.7, over 20,000 80 against 45; 100 rows over 1,000 e4m3 keys, 16 heads of 64, 33 against 26). Many rows a sequence
// (new prompts) fill an item by themselves: each walks the prefix and its own keys in one go.
static int dispatch_prefix(wx_ctx* ctx, const wx_attn_dims* d, TextAttnParams& p, const KvSource& kv) {
  const int64_t few = kv.format == kKvBf16 ? 16 : kv.format == kKvE4m3 ? 32 : 48;
  const int64_t own = (int64_t)d->max_q * p.group, all = p.total_q * p.group;
  if (own > few) return text_flash(ctx, p, d->head_dim, kv, kPrefixKeys);
  const bool flash = p.prefix && all > few && (all + 15) / 16 * p.prefix * p.hkv > 65536;
  const bool both = p.prefix && !flash;  // the rows kernel walks the prefix too
  // Own keys in chunks for single warps, the longer the more items there are (keys a chunk: us in all. 3 sequences
  // behind 333 keys, 16 heads of 64, 64 items: 64: 9.4, 128: 10.8; 8 of 900 bf16 keys behind 4,000, 96 items: 64: 27, 96: 22,
  // 128: 24; 64 of 1 to 701 behind 8,011, 512 items: 64: 41, 128: 42, 256: 49). With many items the lengths decide, which
  // only the device knows: 128 : 256 : 384 keys a chunk, 32 / 8 heads, sequences of 1 to 700 keys behind 8,000, 640 items
  // at bf16 66 : 76 : 80, 1,024 items 82 : 86 : 100 and at e4m3 84 : 96 : 102; of 20 to 3,000, 640 items 137 : 135 : 133 and
  // 117 : 111 : 121, 1,024 items 182 : 182 : 182 and 148 : 141 : 143; 100 of 1,200 behind 5,000, 16 / 16 heads, 1,600 items
  // 250 : 229 : 234; 128 of 20 to 1,520 e4m3 keys behind 40,000, 64 / 8 heads, 1,024 items 303 : 293 : 287. Chunks are
  // longer where there would be more than so many of a sequence: each is a layer, for which room is set aside, and the
  // more items there are, the fewer chunks give each warp its share.
  // Items that are too few to give every warp a unit although their keys may be many, which the tables' width bounds,
  // are left to a piece per CTA, which divides them evenly. A piece per CTA : chunks of 64, us in tables of 131,072
  // keys, 32 / 8 heads: 1 x 30,000 own keys 47 : 66, 5 x 100,000 338 : 471, 6 of up to 300 behind 333 22.5 : 16.4, 5 of
  // 100 to 500 behind 8,000 45 : 35, the most that a wide table costs short sequences; 8 / 2 heads, 20 of which one has
  // 100,000, 66 : 180.
  const int64_t most = std::max<int64_t>(p.blocks_per_seq << p.page_shift, both ? p.prefix : 0);
  const int64_t items = (int64_t)p.hkv * (both ? p.batch * ((own + 7) / 8) + (all + 7) / 8 : p.batch * ((own + 7) / 8));
  p.chunk = items < 80 ? 64 : items < 256 ? 96 : items < 1024 ? 128 : 256;
  p.chunks = items < 1024 ? 32 : items < 4096 ? 16 : items < 16384 ? 8 : 4;
  if (items * p.chunks < 12 * (int64_t)ctx->num_sms && most > p.chunks * p.chunk) p.chunk = 0;
  // (the prefix's layers are all joined, so they are those that its walk writes; own lengths are known on the device)
  p.own_layer = flash ? text_flash_layers(ctx, p) : both ? layers_of(p.chunk, p.chunks, p.prefix) : 0;
  p.layers = p.own_layer + most_layers(p.chunk, p.chunks, p.blocks_per_seq << p.page_shift);
  const int64_t rows = p.total_q * p.hq;
  Carve c;
  const size_t o_o = c.take((size_t)(p.layers * rows) * d->head_dim * 4), o_ml = c.take((size_t)(p.layers * rows) * 8);
  p.ws_reserved = c.off;
  // what the kernels take for themselves is asked for now: a workspace that grew between them would lose the layers
  const size_t rows_ws = (size_t)ctx->num_sms * 2 * 16 * (d->head_dim * 4 + 8) + 512;
  int st;
  uint8_t* ws = static_cast<uint8_t*>(workspace(ctx, c.off + std::max(rows_ws, text_flash_ws(ctx)), &st));
  if (!ws) return st;
  p.layer_o = reinterpret_cast<float*>(ws + o_o);
  p.layer_ml = reinterpret_cast<float2*>(ws + o_ml);
  if (flash) {
    TextAttnParams f = p;
    f.shared = 1;
    f.batch = 1;
    if ((st = text_flash(ctx, f, d->head_dim, kv, kPrefixKeys))) return st;
  }
  TextAttnParams r = p;
  r.after_walk = flash;
  // Beside the shared walk there is a CTA for each SM that it leaves free, if those are a third: CTAs
  // that begin behind it would find the work done, and hold the join up by their own start (3 us)
  r.ctas = ctx->num_sms;
  if (flash) {
    const int64_t left = ctx->num_sms - text_flash_walk_ctas(p, p.own_layer);
    if (3 * left >= ctx->num_sms) r.ctas = (int)left;
  }
  if (both) {
    r.shared = 1;
    ++r.batch;
  }
  st = p.chunk ? launch_rows_attn<kChunkKeys>(ctx, d->head_dim, both ? all : own, r, kv)
               : launch_rows_attn<kPrefixKeys>(ctx, d->head_dim, both ? all : own, r, kv);
  if (st) return st;
  ProfScope prof(ctx, kProfAttn);
  if (join_by_fours(ctx, p))
    st = d->head_dim == 128 ? launch_dependent(ctx, prefix_join_kernel<128, 4>, join_blocks(p, 4), 256, 0, p)
                            : launch_dependent(ctx, prefix_join_kernel<64, 4>, join_blocks(p, 4), 256, 0, p);
  else
    st = d->head_dim == 128 ? launch_dependent(ctx, prefix_join_kernel<128, 1>, join_blocks(p, 1), 256, 0, p)
                            : launch_dependent(ctx, prefix_join_kernel<64, 1>, join_blocks(p, 1), 256, 0, p);
  return st ? st : launch_status(ctx, "prefix_join");
}

// checks of a call over the paged cache, and its parameters
static int paged_params(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride, const wx_kv_cache* cache,
                        const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table,
                        int64_t blocks_per_seq, void* out, int64_t out_stride, float* lse, TextAttnParams& p,
                        KvSource& kv, bool& empty) {
  empty = true;
  int st = check_dims(ctx, dims, q, q_stride, out, out_stride, cu_q);
  if (st) return st;
  if ((st = check_kv_cache(ctx, cache))) return st;
  WX_CHECK_ARG(ctx, cache->kv_heads == dims->kv_heads && cache->head_dim == dims->head_dim);
  WX_CHECK_ARG(ctx, cache->format != WX_KV_INT8 || dims->scale < 0x1p100f);  // (int8 scores are formed in units of 2^13)
  if (dims->total_q == 0 || dims->batch == 0) return WX_OK;
  WX_CHECK_ARG(ctx, kv_lens && block_table && blocks_per_seq > 0);
  WX_CHECK_ARG(ctx, blocks_per_seq <= INT32_MAX / cache->page_size);
  fill_params(ctx, dims, q, q_stride, cu_q, out, out_stride, lse, p);
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.blocks_per_seq = blocks_per_seq;
  p.ks = cache->k_scale;
  p.vs = cache->v_scale;
  p.pages = cache->pages;
  p.page_shift = __builtin_ctz((unsigned)cache->page_size);
  kv = KvSource{cache->k, cache->v, (uint64_t)cache->pages * cache->kv_heads * cache->page_size,
                (uint64_t)cache->head_dim, (uint64_t)cache->head_dim, (uint64_t)cache->head_dim, cache->format};
  empty = false;
  return WX_OK;
}

}  // namespace wx

using namespace wx;

extern "C" {

int wx_prompt_attention_sinks(wx_ctx* ctx, const wx_attn_dims* dims, int32_t sinks, const void* q, int64_t q_stride,
                              const void* k, int64_t k_stride, const void* v, int64_t v_stride, int64_t total_k,
                              const int32_t* cu_q, const int32_t* cu_k, void* out, int64_t out_stride, float* lse) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && sinks >= 0);
  int st = check_dims(ctx, dims, q, q_stride, out, out_stride, cu_q);
  if (st || dims->total_q == 0 || dims->batch == 0) return st;
  const int64_t cols = (int64_t)dims->kv_heads * dims->head_dim;
  WX_CHECK_ARG(ctx, total_k >= 0 && total_k <= INT32_MAX && (cu_k || total_k == dims->total_q));
  WX_CHECK_ARG(ctx, k_stride % 8 == 0 && v_stride % 8 == 0 && k_stride >= cols && v_stride >= cols);
  WX_CHECK_ARG(ctx, total_k == 0 || (k && v && aligned16(k) && aligned16(v)));
  TextAttnParams p{};
  fill_params(ctx, dims, q, q_stride, cu_q, out, out_stride, lse, p);
  p.sinks = sinks;
  p.cu_k = cu_k ? cu_k : cu_q;
  p.total_k = total_k;
  // (with no keys at all nothing is read: any valid address serves the tensor maps)
  const KvSource kv{total_k ? k : q, total_k ? v : q, (uint64_t)std::max<int64_t>(total_k, 1), (uint64_t)cols,
                    (uint64_t)k_stride, (uint64_t)v_stride, kKvBf16};
  return dispatch_attn(ctx, dims, p, kv);
}

int wx_prompt_attention(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride, const void* k,
                        int64_t k_stride, const void* v, int64_t v_stride, int64_t total_k, const int32_t* cu_q,
                        const int32_t* cu_k, void* out, int64_t out_stride, float* lse) {
  return wx_prompt_attention_sinks(ctx, dims, 0, q, q_stride, k, k_stride, v, v_stride, total_k, cu_q, cu_k, out,
                                   out_stride, lse);
}

int wx_paged_attention_sinks(wx_ctx* ctx, const wx_attn_dims* dims, int32_t sinks, const void* q, int64_t q_stride,
                             const wx_kv_cache* cache, const int32_t* cu_q, const int32_t* kv_lens,
                             const int32_t* block_table, int64_t blocks_per_seq, void* out, int64_t out_stride,
                             float* lse) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && sinks >= 0);
  TextAttnParams p{};
  KvSource kv;
  bool empty;
  const int st = paged_params(ctx, dims, q, q_stride, cache, cu_q, kv_lens, block_table, blocks_per_seq, out, out_stride,
                              lse, p, kv, empty);
  if (st || empty) return st;
  p.sinks = sinks;
  return dispatch_attn(ctx, dims, p, kv);
}

int wx_prefix_attention(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride,
                        const wx_kv_cache* cache, const int32_t* prefix_blocks, int64_t prefix_len,
                        const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table,
                        int64_t blocks_per_seq, int64_t table_stride, void* out, int64_t out_stride, float* lse) {
  DeviceScope on_device(ctx);
  TextAttnParams p{};
  KvSource kv;
  bool empty;
  WX_CHECK_ARG(ctx, ctx && dims && dims->window == 0);
  const int st = paged_params(ctx, dims, q, q_stride, cache, cu_q, kv_lens, block_table, blocks_per_seq, out, out_stride,
                              lse, p, kv, empty);
  if (st || empty) return st;
  WX_CHECK_ARG(ctx, prefix_len >= 0 && (prefix_len == 0 || prefix_blocks));
  if (prefix_len > INT32_MAX - 8192)  // (tiles and steps behind the last key are counted in 32 bits too)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "prefix_len must be below 2^31 - 8192");
  WX_CHECK_ARG(ctx, table_stride >= blocks_per_seq || table_stride == 0);
  p.prefix = (int)prefix_len;
  p.front = (int)((prefix_len + 127) / 128);
  p.prefix_blocks = prefix_blocks;
  p.table_stride = table_stride;
  return dispatch_prefix(ctx, dims, p, kv);
}

int wx_paged_attention(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride,
                       const wx_kv_cache* cache, const int32_t* cu_q, const int32_t* kv_lens,
                       const int32_t* block_table, int64_t blocks_per_seq, void* out, int64_t out_stride,
                       float* lse) {
  return wx_paged_attention_sinks(ctx, dims, 0, q, q_stride, cache, cu_q, kv_lens, block_table, blocks_per_seq, out,
                                  out_stride, lse);
}

}  // extern "C"
