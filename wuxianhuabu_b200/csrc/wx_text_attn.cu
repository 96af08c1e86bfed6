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

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------- few query rows: text_rows_attn_kernel
// For decoding and for a few new tokens: 16 flattened query rows share one walk over the keys.
// 16 rows against 128-wide heads are 32 FLOP per K/V byte at bf16, far below the ridge, so the
// walk is bound by the K/V bytes; the tensor work (mma.sync, M = 16) and the 8-bit expansion
// stay in registers below that bound.
//
// A CTA's eight warps take 16-key steps of its key range in turn, each with its own ring of
// TMA-filled stages (kStages deep, swizzled so that both fragment reads are conflict-free) and
// its own running maximum and denominator; they are joined once, at the end of the range. A
// step's keys and head columns are dealt to the fragments in the order that makes every
// shared-memory read a 16-byte one and the products need no transposition: a dot product does
// not care for the order of its terms, so q, K (head columns) and P, V (keys) are permuted alike.
//
// Work is split evenly: the (sequence, K/V head, row tile) items, each cut into units of 128
// keys, form one line of units that is divided into equal runs, one per CTA. A CTA whose run
// covers part of an item leaves its partial sums; the last to arrive joins them in key order
// (so the result does not depend on who is last).
template <int FMT, int HD>
struct RowsGeom {
  static constexpr bool kWide = FMT != kKvBf16;               // 8-bit rows
  static constexpr int kTiles = kWide ? 1 : HD / 64;          // boxes per 16-key K (or V) step
  static constexpr int kRowBytes = kWide ? HD : 128;          // bytes of a box row (swizzle span)
  static constexpr int kTileBytes = 16 * kRowBytes;
  static constexpr int kKvBytes = kTiles * kTileBytes;        // K (or V) of a step
  static constexpr int kStepBytes = 2 * kKvBytes;
  static constexpr int kStages = kWide ? 4 : (HD == 128 ? 2 : 4);
  static constexpr int kWarps = 8;
  static constexpr int kRing = kWarps * kStages * kStepBytes;
  static constexpr int kScales = kWide ? kWarps * kStages * 128 : 0;
  static constexpr int kPitch = HD + 4;
  static constexpr int kJoin = kWarps * 16 * (kPitch + 2) * 4;
  static constexpr int kBars = kWarps * kStages * 8 + 64;
  static constexpr int kSmem = kRing + kScales + kJoin + kBars + 1024;
};

constexpr int kUnit = 128;  // keys of a unit: one step of each warp

template <int FMT, int HD>
__global__ void __launch_bounds__(256, 1)
    text_rows_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                          TextAttnParams p, int min_units) {
  using G = RowsGeom<FMT, HD>;
  constexpr bool kW = G::kWide;
  constexpr int kD = G::kStages;
  constexpr int kNB = HD / 8;  // 8-column blocks of the output
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  float* join = reinterpret_cast<float*>(smem + G::kRing + G::kScales);
  float* join_ml = join + G::kWarps * 16 * G::kPitch;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kRing + G::kScales + G::kJoin);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + G::kWarps * kD);
  int* last_flag = const_cast<int*>(abort_flag) + 1;
  auto stage = [&](int s) { return sbase + (uint32_t)((warp * kD + s) * G::kStepBytes); };
  auto sscale = [&](int s) { return sbase + G::kRing + (uint32_t)((warp * kD + s) * 128); };
  auto bar = [&](int s) { return smem_u32(bars + warp * kD + s); };

  if (lane == 0)
    for (int s = 0; s < kD; ++s) mbar_init(bar(s), 1);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_mbar_init();
  fence_proxy_async_smem();
  __syncthreads();

  // ---- the line of units, walked 32 sequences at a time by each warp for itself
  auto seq_units = [&](int b, int& items) -> int64_t {
    items = 0;
    if (b >= p.batch) return 0;
    const Seq s = load_seq(p, b);
    const int rt = (int)(((int64_t)s.lq * p.group + 15) / 16);
    items = rt * p.hkv;
    const int k16 = key_lo(p, s, 0) & ~15;
    return (int64_t)items * max(1, (s.lk - k16 + kUnit - 1) / kUnit);
  };
  int64_t total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int it;
    int64_t n = seq_units(b0 + lane, it);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  const int64_t per = max64(min_units, (total + gridDim.x - 1) / gridDim.x);
  int64_t u = (int64_t)blockIdx.x * per;
  const int64_t u_end = min64(total, u + per);

  // sequence group being walked: units and items before it
  int wb = 0;
  int64_t wu = 0;
  int wi = 0;
  struct Piece {
    Seq s;
    int b, h, rt, item;
    int k_lo, k_hi;          // keys of this piece (k_lo a multiple of 16)
    int64_t item_u0;         // the item's first unit, and its units
    int nu;
    int steps;               // 16-key steps of this piece for this warp
  };
  auto piece_at = [&](int64_t at, Piece& c) {
    while (true) {
      int it;
      const int64_t n = seq_units(wb + lane, it);
      int64_t nc = n;
      int ic = it;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, nc, o);
        const int e = __shfl_up_sync(0xffffffffu, ic, o);
        if (lane >= o) {
          nc += a;
          ic += e;
        }
      }
      const int64_t group_units = __shfl_sync(0xffffffffu, nc, 31);
      if (at < wu + group_units) {
        const int src = __ffs(__ballot_sync(0xffffffffu, at < wu + nc)) - 1;
        c.b = wb + src;
        const int64_t b_u0 = wu + __shfl_sync(0xffffffffu, nc - n, src);
        const int b_i0 = wi + __shfl_sync(0xffffffffu, ic - it, src);
        c.s = load_seq(p, c.b);
        const int rts = (int)(((int64_t)c.s.lq * p.group + 15) / 16);
        const int k16 = key_lo(p, c.s, 0) & ~15;
        c.nu = max(1, (c.s.lk - k16 + kUnit - 1) / kUnit);
        const int64_t in_b = at - b_u0;
        const int i = (int)(in_b / c.nu);
        const int u_in = (int)(in_b % c.nu);
        c.h = i / rts;
        c.rt = i % rts;
        c.item = b_i0 + i;
        c.item_u0 = b_u0 + (int64_t)i * c.nu;
        const int u_stop = (int)min64(c.nu, u_in + (u_end - at));
        c.k_lo = k16 + u_in * kUnit;
        c.k_hi = min(c.s.lk, k16 + u_stop * kUnit);
        const int n16 = max(0, (c.k_hi - c.k_lo + 15) / 16);
        c.steps = n16 > warp ? (n16 - warp + 7) / 8 : 0;
        return u_stop - u_in;
      }
      wu += group_units;
      wi += __shfl_sync(0xffffffffu, ic, 31);
      wb += 32;
    }
  };

  // ---- loads: step i of this warp starts at key k_lo + (i * 8 + warp) * 16; the pages of 32
  // consecutive steps are fetched at once, one per lane
  uint32_t issued = 0, used = 0;  // steps loaded / consumed so far
  bool ok = true;
  int page_of = 0;
  auto load_step = [&](const Piece& c, int i) {
    const int j0 = c.k_lo + (i * 8 + warp) * 16;
    int row, x = 0;
    if (p.block_table) {
      if ((i & 31) == 0) {
        const int jl = c.k_lo + ((i + lane) * 8 + warp) * 16;
        page_of = 0;
        if (jl < c.k_hi) {
          page_of = p.block_table[c.b * p.blocks_per_seq + (jl >> p.page_shift)];
          if (page_of < 0 || page_of >= p.pages) {
            set_dev_error(p.err, kDevBadArgs);
            page_of = 0;
          }
        }
      }
      const int page = __shfl_sync(0xffffffffu, page_of, i & 31);
      row = (int)((((int64_t)page * p.hkv + c.h) << p.page_shift) | (j0 & ((1 << p.page_shift) - 1)));
    } else {
      row = (int)(c.s.k0 + j0);
      x = c.h * HD;
    }
    if (lane == 0) {
      const int s = issued % kD;
      mbar_arrive_expect_tx(bar(s), G::kStepBytes + (kW ? 128 : 0));
#pragma unroll
      for (int ch = 0; ch < G::kTiles; ++ch) {
        tma_load_2d(stage(s) + ch * G::kTileBytes, &tmK, bar(s), x + ch * 64, row);
        tma_load_2d(stage(s) + G::kKvBytes + ch * G::kTileBytes, &tmV, bar(s), x + ch * 64, row);
      }
      if constexpr (kW) {
        bulk_load(sscale(s), p.ks + row, 64, bar(s));
        bulk_load(sscale(s) + 64, p.vs + row, 64, bar(s));
      }
    }
    ++issued;
  };

  // dealing of keys to fragment columns and of 16-byte chunks to lane groups
  auto kp = [](int n) { return (kW && HD == 64) ? n : (n >> 1) | ((n & 1) << 2); };
  auto swz = [](int row, int chunk) {  // byte offset of a 16-byte chunk in a swizzled box
    return (kW && HD == 64) ? (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4))
                            : (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
  };
  // head column of output block j, fragment column n
  auto out_dim = [&](int j, int n) {
    if constexpr (!kW) return (j >> 3) * 64 + kp(n) * 8 + (j & 7);
    else if constexpr (HD == 128) return kp(n) * 16 + j;
    else return n * 8 + j;
  };

  Piece cur;
  bool have = u < u_end;
  int units = 0;
  if (have) {
    units = piece_at(u, cur);
    for (int i = 0; i < kD && i < cur.steps; ++i) load_step(cur, i);
  }
  while (have) {
    const int64_t n_rows = (int64_t)cur.s.lq * p.group;
    const int row0 = cur.rt * 16;
    // ---- q fragments: rows g and g + 8, columns in the order of the K reads
    uint32_t qf[HD / 16][4];
    int lim_hi[2], lim_lo[2];
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      const int r = row0 + g + 8 * hrow;
      const bool live = r < n_rows;
      const int tok = live ? r / p.group : 0;
      const int head = cur.h * p.group + (live ? r % p.group : 0);
      lim_hi[hrow] = live ? key_hi(p, cur.s, tok) : 0;
      lim_lo[hrow] = live ? key_lo(p, cur.s, tok) : 0;
      const __nv_bfloat16* src = p.q + (cur.s.q0 + tok) * p.q_stride + (int64_t)head * HD;
      if constexpr (!kW) {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (live) w = *reinterpret_cast<const uint4*>(src + (i >> 1) * 64 + ((i & 1) * 4 + t) * 8);
          qf[2 * i][hrow] = w.x;
          qf[2 * i][2 + hrow] = w.y;
          qf[2 * i + 1][hrow] = w.z;
          qf[2 * i + 1][2 + hrow] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (live) w = *reinterpret_cast<const uint4*>(src + i * 64 + t * 16 + e * 8);
            qf[4 * i + 2 * e][hrow] = w.x;
            qf[4 * i + 2 * e][2 + hrow] = w.y;
            qf[4 * i + 2 * e + 1][hrow] = w.z;
            qf[4 * i + 2 * e + 1][2 + hrow] = w.w;
          }
        }
      }
    }
    // a step between these sees no mask in any row of the tile
    const int last_tok = (int)(min64(n_rows - 1, row0 + 15) / p.group);
    const int free_hi = key_hi(p, cur.s, row0 / p.group);
    const int free_lo = key_lo(p, cur.s, last_tok);

    float acc[kNB][4];
#pragma unroll
    for (int j = 0; j < kNB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int i = 0; i < cur.steps; ++i) {
      const int s = used % kD;
      const int j0 = cur.k_lo + (i * 8 + warp) * 16;
      if (ok && !mbar_wait(bar(s), (used / kD) & 1, p.err, kDevTimeoutFull, abort_flag)) ok = false;
      if (!ok) break;
      const uint32_t sk = stage(s), sv = stage(s) + G::kKvBytes;
      float sc[2][4];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nb][e] = 0.f;
        const int row = nb * 8 + kp(g);
        if constexpr (!kW) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            const uint4 w = lds128(sk + (c >> 1) * G::kTileBytes + swz(row, (c & 1) * 4 + t));
            mma_bf16(sc[nb], qf[2 * c], w.x, w.y);
            mma_bf16(sc[nb], qf[2 * c + 1], w.z, w.w);
          }
        } else {
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            const uint4 w = lds128(sk + swz(row, c * 4 + t));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mma_bf16(sc[nb], qf[4 * c + e], bytes_to_bf16x2<FMT>(ww[e], 0, 0, 1),
                       bytes_to_bf16x2<FMT>(ww[e], 0, 2, 3));
          }
        }
      }
      // scores in base 2, scaled, masked; key of column e of block nb
      const bool masked = j0 + 16 > free_hi || j0 < free_lo;
      float vscale[2][2];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int kk = nb * 8 + kp(2 * t + e);
          float f = p.sl2;
          vscale[nb][e] = 1.f;
          if constexpr (kW) {
            f *= lds_f32(sscale(s) + kk * 4);
            vscale[nb][e] = lds_f32(sscale(s) + 64 + kk * 4);
          }
          sc[nb][e] *= f;
          sc[nb][2 + e] *= f;
          if (masked) {
            const int j = j0 + kk;
#pragma unroll
            for (int hrow = 0; hrow < 2; ++hrow)
              if (j >= lim_hi[hrow] || j < lim_lo[hrow]) sc[nb][2 * hrow + e] = -INFINITY;
          }
        }
      float alpha[2];
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow) {
        float mx = fmaxf(fmaxf(sc[0][2 * hrow], sc[0][2 * hrow + 1]), fmaxf(sc[1][2 * hrow], sc[1][2 * hrow + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[hrow], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        alpha[hrow] = exp2_approx(m[hrow] - mu);
        m[hrow] = mn;
        float sum = 0.f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[nb][2 * hrow + e];
            const bool off = x == -INFINITY;
            x = exp2_approx(x - mu);
            sum += x;
            // a masked key's scale may be anything: its weight is 0, not 0 * scale
            if constexpr (kW) x = off ? 0.f : x * vscale[nb][e];
          }
        l[hrow] = l[hrow] * alpha[hrow] + sum;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < kNB; ++j) {
          acc[j][0] *= alpha[0];
          acc[j][1] *= alpha[0];
          acc[j][2] *= alpha[1];
          acc[j][3] *= alpha[1];
        }
      }
      // P rounded to bf16 for the tensor product (the denominator sums the unrounded values)
      const uint32_t pf[4] = {pack_bf16x2(sc[0][0], sc[0][1]), pack_bf16x2(sc[0][2], sc[0][3]),
                              pack_bf16x2(sc[1][0], sc[1][1]), pack_bf16x2(sc[1][2], sc[1][3])};
      const int vr[4] = {kp(2 * t), kp(2 * t + 1), 8 + kp(2 * t), 8 + kp(2 * t + 1)};
      if constexpr (!kW) {
        bool slow = false;
#pragma unroll
        for (int c = 0; c < G::kTiles; ++c) {
          uint32_t w[4][4];
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const uint4 x = lds128(sv + c * G::kTileBytes + swz(vr[rr], kp(g)));
            w[rr][0] = x.x;
            w[rr][1] = x.y;
            w[rr][2] = x.z;
            w[rr][3] = x.w;
          }
          if (masked) {
            // keys past the end are another sequence's or nobody's: zero them (0 * NaN is NaN).
            // A non-finite value at a key that only some rows see: the whole step goes by
            // scalar sums below.
            bool odd = false;
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (j0 + vr[rr] >= cur.s.lk) w[rr][e] = 0;
                odd |= (w[rr][e] & 0x7f80u) == 0x7f80u || (w[rr][e] & 0x7f800000u) == 0x7f800000u;
              }
            if (c == 0) {
              // (both halves are checked before the first product)
              if constexpr (G::kTiles == 2) {
#pragma unroll
                for (int rr = 0; rr < 4; ++rr) {
                  const uint4 x = lds128(sv + G::kTileBytes + swz(vr[rr], kp(g)));
                  const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    odd |= j0 + vr[rr] < cur.s.lk &&
                           ((y[e] & 0x7f80u) == 0x7f80u || (y[e] & 0x7f800000u) == 0x7f800000u);
                }
              }
              slow = __any_sync(0xffffffffu, odd);
            }
            if (slow) break;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            mma_bf16(acc[c * 8 + 2 * e], pf, __byte_perm(w[0][e], w[1][e], 0x5410),
                     __byte_perm(w[2][e], w[3][e], 0x5410));
            mma_bf16(acc[c * 8 + 2 * e + 1], pf, __byte_perm(w[0][e], w[1][e], 0x7632),
                     __byte_perm(w[2][e], w[3][e], 0x7632));
          }
        }
        if (slow) {
#pragma unroll 1
          for (int kk = 0; kk < 16; ++kk) {
            const int n = ((kk & 3) << 1) | ((kk & 7) >> 2);  // fragment column that holds this key
            const int src = (lane & ~3) | (n >> 1);
            const float a0 = kk < 8 ? ((n & 1) ? sc[0][1] : sc[0][0]) : ((n & 1) ? sc[1][1] : sc[1][0]);
            const float a1 = kk < 8 ? ((n & 1) ? sc[0][3] : sc[0][2]) : ((n & 1) ? sc[1][3] : sc[1][2]);
            const float p0 = round_bf16(__shfl_sync(0xffffffffu, a0, src));
            const float p1 = round_bf16(__shfl_sync(0xffffffffu, a1, src));
            const int j = j0 + kk;
            const bool see0 = j < lim_hi[0] && j >= lim_lo[0], see1 = j < lim_hi[1] && j >= lim_lo[1];
#pragma unroll
            for (int jb = 0; jb < kNB; ++jb)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int chunk = kp(2 * t + e);
                const float v = __uint_as_float(
                    lds_u16(sv + (jb >> 3) * G::kTileBytes + swz(kk, chunk) + (uint32_t)(jb & 7) * 2) << 16);
                if (see0) acc[jb][e] += p0 * v;
                if (see1) acc[jb][2 + e] += p1 * v;
              }
          }
        }
      } else if constexpr (HD == 128) {
        uint32_t w[4][4];
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
          const uint4 x = lds128(sv + swz(vr[rr], kp(g)));
          w[rr][0] = x.x;
          w[rr][1] = x.y;
          w[rr][2] = x.z;
          w[rr][3] = x.w;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j)
          mma_bf16(acc[j], pf, bytes_to_bf16x2<FMT>(w[0][j >> 2], w[1][j >> 2], j & 3, 4 + (j & 3)),
                   bytes_to_bf16x2<FMT>(w[2][j >> 2], w[3][j >> 2], j & 3, 4 + (j & 3)));
      } else {
        uint32_t w[4][2];
#pragma unroll
        for (int rr = 0; rr < 4; ++rr) {
          const uint2 x = lds64(sv + swz(vr[rr], g >> 1) + (uint32_t)(g & 1) * 8);
          w[rr][0] = x.x;
          w[rr][1] = x.y;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mma_bf16(acc[j], pf, bytes_to_bf16x2<FMT>(w[0][j >> 2], w[1][j >> 2], j & 3, 4 + (j & 3)),
                   bytes_to_bf16x2<FMT>(w[2][j >> 2], w[3][j >> 2], j & 3, 4 + (j & 3)));
      }
      ++used;
      __syncwarp();  // every lane has read the stage
      if (i + kD < cur.steps) load_step(cur, i + kD);
    }

    // ---- the next piece's first loads go out before this one is joined
    const Piece done = cur;
    const int64_t u_done = u;
    u += units;
    have = u < u_end;
    if (have) {
      units = piece_at(u, cur);
      if (ok)
        for (int i = 0; i < kD && i < cur.steps; ++i) load_step(cur, i);
    }

    // ---- join the eight warps
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 1);
      l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 2);
      if (t == 0) {
        join_ml[(warp * 16 + g + 8 * hrow) * 2] = m[hrow];
        join_ml[(warp * 16 + g + 8 * hrow) * 2 + 1] = l[hrow];
      }
    }
    if (done.steps > 0) {
#pragma unroll
      for (int j = 0; j < kNB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          join[(warp * 16 + g + 8 * (e >> 1)) * G::kPitch + out_dim(j, 2 * t + (e & 1))] = acc[j][e];
    }
    __syncthreads();
    constexpr int kPer = HD / 16;  // columns of a thread
    const int jr = threadIdx.x >> 4, jc = (threadIdx.x & 15) * kPer;
    float M = -INFINITY, L = 0.f, o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) M = fmaxf(M, join_ml[(w * 16 + jr) * 2]);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float lw = join_ml[(w * 16 + jr) * 2 + 1];
      if (lw == 0.f) continue;
      const float f = exp2_approx(join_ml[(w * 16 + jr) * 2] - M);
      L += lw * f;
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(&join[(w * 16 + jr) * G::kPitch + jc + i]);
        o[i] += x.x * f;
        o[i + 1] += x.y * f;
        o[i + 2] += x.z * f;
        o[i + 3] += x.w * f;
      }
    }
    const bool whole = u_done <= done.item_u0 && u >= done.item_u0 + done.nu;
    bool write = whole;
    if (!whole) {
      // this CTA's piece of an item: slot 0 if the item began in an earlier CTA, 1 if it goes on
      const int slot = 2 * blockIdx.x + (done.item_u0 >= (int64_t)blockIdx.x * per ? 1 : 0);
      float* dst = p.part + ((int64_t)slot * 16 + jr) * HD + jc;
#pragma unroll
      for (int i = 0; i < kPer; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      if ((threadIdx.x & 15) == 0) {
        p.part_ml[((int64_t)slot * 16 + jr) * 2] = M;
        p.part_ml[((int64_t)slot * 16 + jr) * 2 + 1] = L;
      }
      __threadfence();
      __syncthreads();
      const int c0 = (int)(done.item_u0 / per), c1 = (int)((done.item_u0 + done.nu - 1) / per);
      if (threadIdx.x == 0) {
        // (sequences that overlap in cu_q could count more items than there are counters)
        const bool known = done.item < p.n_items;
        const int before = known ? atomicAdd(p.counters + done.item, 1) : -1;
        *last_flag = before == c1 - c0;
        if (before == c1 - c0) p.counters[done.item] = 0;
        if (!known) set_dev_error(p.err, kDevBadArgs);
      }
      __syncthreads();
      write = *last_flag != 0;
      if (write) {
        __threadfence();
        M = -INFINITY;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = 0.f;
        for (int c = c0; c <= c1; ++c) {
          const int sl = 2 * c + (done.item_u0 >= (int64_t)c * per ? 1 : 0);
          M = fmaxf(M, __ldcg(p.part_ml + ((int64_t)sl * 16 + jr) * 2));
        }
        for (int c = c0; c <= c1; ++c) {
          const int sl = 2 * c + (done.item_u0 >= (int64_t)c * per ? 1 : 0);
          const float lw = __ldcg(p.part_ml + ((int64_t)sl * 16 + jr) * 2 + 1);
          if (lw == 0.f) continue;
          const float f = exp2_approx(__ldcg(p.part_ml + ((int64_t)sl * 16 + jr) * 2) - M);
          L += lw * f;
#pragma unroll
          for (int i = 0; i < kPer; i += 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part + ((int64_t)sl * 16 + jr) * HD + jc + i));
            o[i] += x.x * f;
            o[i + 1] += x.y * f;
            o[i + 2] += x.z * f;
            o[i + 3] += x.w * f;
          }
        }
      }
    }
    const int r = done.rt * 16 + jr;
    if (write && r < (int64_t)done.s.lq * p.group) {
      const int64_t tok = done.s.q0 + r / p.group;
      const int head = done.h * p.group + r % p.group;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      uint32_t w[kPer / 2];
#pragma unroll
      for (int i = 0; i < kPer; i += 2) w[i / 2] = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
      __nv_bfloat16* dst = p.out + tok * p.out_stride + (int64_t)head * HD + jc;
      if constexpr (kPer == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      if (p.lse && (threadIdx.x & 15) == 0)
        p.lse[tok * p.hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
    }
    __syncthreads();  // the join buffer is free again
  }
  // after a wait that ran out: copies still in flight land before the CTA's memory goes away
  for (; used < issued; ++used) mbar_drain(bar(used % kD), (used / kD) & 1);
}

// --------------------------------------------------------------------- host side
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
  p.err = ctx->dev_err;
}

template <int FMT, int HD>
static int launch_rows_attn(wx_ctx* ctx, TextAttnParams p, const KvSource& kv) {
  using G = RowsGeom<FMT, HD>;
  const int grid = ctx->num_sms;
  const int64_t items = (int64_t)p.hkv * (p.total_q * p.group / 16 + p.batch);
  CUtensorMap tk, tv;
  int st;
  if (FMT == kKvBf16) {
    if ((st = make_tmap_bf16_2d(ctx, &tk, kv.k, kv.rows, kv.cols, kv.k_stride, 64, 16))) return st;
    if ((st = make_tmap_bf16_2d(ctx, &tv, kv.v, kv.rows, kv.cols, kv.v_stride, 64, 16))) return st;
  } else {
    if ((st = make_tmap_u8_rows(ctx, &tk, kv.k, kv.rows, (uint32_t)kv.cols, 16))) return st;
    if ((st = make_tmap_u8_rows(ctx, &tv, kv.v, kv.rows, (uint32_t)kv.cols, 16))) return st;
  }
  Carve c;
  const size_t o_part = c.take((size_t)grid * 2 * 16 * HD * 4), o_ml = c.take((size_t)grid * 2 * 16 * 8);
  uint8_t* ws = static_cast<uint8_t*>(workspace(ctx, c.off, &st));
  if (!ws) return st;
  p.part = reinterpret_cast<float*>(ws + o_part);
  p.part_ml = reinterpret_cast<float*>(ws + o_ml);
  p.n_items = items;
  if (!(p.counters = arrival_counters(ctx, items, &st))) return st;
  auto fn = text_rows_attn_kernel<FMT, HD>;
  if ((st = ensure_smem_attr(ctx, (const void*)fn, G::kSmem, "text_rows_attn"))) return st;
  ProfScope prof(ctx, kProfAttn);
  fn<<<grid, 256, G::kSmem, ctx->stream>>>(tk, tv, p, 2);
  return launch_status(ctx, "text_rows_attn");
}

// Up to 16 flattened rows a sequence (a decoding step, a few drafted tokens) fill one tile of the
// rows kernel, which is bound by the K/V bytes; more rows go to the tcgen05 kernel.
static int dispatch_attn(wx_ctx* ctx, const wx_attn_dims* d, const TextAttnParams& p, const KvSource& kv) {
  const bool big = d->head_dim == 128;
  if ((int64_t)d->max_q * p.group > 16) return text_flash(ctx, p, d->head_dim, kv);
  if (kv.format == kKvInt8)
    return big ? launch_rows_attn<kKvInt8, 128>(ctx, p, kv) : launch_rows_attn<kKvInt8, 64>(ctx, p, kv);
  if (kv.format == kKvE4m3)
    return big ? launch_rows_attn<kKvE4m3, 128>(ctx, p, kv) : launch_rows_attn<kKvE4m3, 64>(ctx, p, kv);
  return big ? launch_rows_attn<kKvBf16, 128>(ctx, p, kv) : launch_rows_attn<kKvBf16, 64>(ctx, p, kv);
}

}  // namespace wx

using namespace wx;

extern "C" {

int wx_prompt_attention(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride, const void* k,
                        int64_t k_stride, const void* v, int64_t v_stride, int64_t total_k, const int32_t* cu_q,
                        const int32_t* cu_k, void* out, int64_t out_stride, float* lse) {
  int st = check_dims(ctx, dims, q, q_stride, out, out_stride, cu_q);
  if (st || dims->total_q == 0 || dims->batch == 0) return st;
  const int64_t cols = (int64_t)dims->kv_heads * dims->head_dim;
  WX_CHECK_ARG(ctx, total_k >= 0 && total_k <= INT32_MAX && (cu_k || total_k == dims->total_q));
  WX_CHECK_ARG(ctx, k_stride % 8 == 0 && v_stride % 8 == 0 && k_stride >= cols && v_stride >= cols);
  WX_CHECK_ARG(ctx, total_k == 0 || (k && v && aligned16(k) && aligned16(v)));
  TextAttnParams p{};
  fill_params(ctx, dims, q, q_stride, cu_q, out, out_stride, lse, p);
  p.cu_k = cu_k ? cu_k : cu_q;
  p.total_k = total_k;
  // (with no keys at all nothing is read: any valid address serves the tensor maps)
  const KvSource kv{total_k ? k : q, total_k ? v : q, (uint64_t)std::max<int64_t>(total_k, 1), (uint64_t)cols,
                    (uint64_t)k_stride, (uint64_t)v_stride, kKvBf16};
  return dispatch_attn(ctx, dims, p, kv);
}

int wx_paged_attention(wx_ctx* ctx, const wx_attn_dims* dims, const void* q, int64_t q_stride,
                       const wx_kv_cache* cache, const int32_t* cu_q, const int32_t* kv_lens,
                       const int32_t* block_table, int64_t blocks_per_seq, void* out, int64_t out_stride,
                       float* lse) {
  int st = check_dims(ctx, dims, q, q_stride, out, out_stride, cu_q);
  if (st) return st;
  if ((st = check_kv_cache(ctx, cache))) return st;
  WX_CHECK_ARG(ctx, cache->kv_heads == dims->kv_heads && cache->head_dim == dims->head_dim);
  if (dims->total_q == 0 || dims->batch == 0) return WX_OK;
  WX_CHECK_ARG(ctx, kv_lens && block_table && blocks_per_seq > 0);
  WX_CHECK_ARG(ctx, blocks_per_seq <= INT32_MAX / cache->page_size);
  TextAttnParams p{};
  fill_params(ctx, dims, q, q_stride, cu_q, out, out_stride, lse, p);
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.blocks_per_seq = blocks_per_seq;
  p.ks = cache->k_scale;
  p.vs = cache->v_scale;
  p.pages = cache->pages;
  p.page_shift = __builtin_ctz((unsigned)cache->page_size);
  const KvSource kv{cache->k, cache->v, (uint64_t)cache->pages * cache->kv_heads * cache->page_size,
                    (uint64_t)cache->head_dim, (uint64_t)cache->head_dim, (uint64_t)cache->head_dim, cache->format};
  return dispatch_attn(ctx, dims, p, kv);
}

}  // extern "C"
