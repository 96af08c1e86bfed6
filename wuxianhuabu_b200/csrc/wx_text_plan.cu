// wx_text_plan.cu — the step of a paged batch made on the device: from the requests' lengths their
// pages, block tables, slots, positions and packed offsets.
//
// Sequence b has old[b] cached tokens in have = ceil(old / page) pages, keeps keep[b] of them and gets
// add[b] more: want = ceil((keep + add) / page) pages. The free list is a stack that grows downwards
// (its entries from `taken` on are free): the pages that sequences give back (have > want) are put
// on top of it in the order of the sequences, then those that others need are taken off it in that order.
//
// Offsets of tokens, taken and given pages are prefix sums over the batch. Every CTA makes them for itself
// (a few loads a thread), so that no CTA waits for another: a token's page, a page that is taken and
// one that is given back each follow from the offsets and from arrays that this launch does not write there. What
// the call may update in place (lengths and the stack's height) is written by the last CTA to finish.
//
// A few bytes a sequence and 12 a token: what bounds it is a launch and its chain of dependent loads
// (lengths, sums, search, table entry).
#include <cuda_runtime.h>

#include <algorithm>

#include "wx_ptx.cuh"
#include "wx_text.h"

namespace wx {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxBatch = 8192;  // five numbers a sequence in shared memory

struct PlanParams {
  const int32_t *old, *keep, *add;
  const int32_t* taken;
  int32_t *table, *free_pages;
  int64_t blocks, pages, tokens, first;
  int batch, page_shift;
  int32_t* positions;
  int64_t* slots;
  int32_t *cu, *lens, *taken_out;
  int* arrived;
  int* err;
};

// index of the last offset at or below x (off[0] = 0)
__device__ __forceinline__ int last_at(const int* off, int n, int x) {
  int b = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (off[b + half] <= x) b += half;
    n -= half;
  }
  return b;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PlanParams p) {
  extern __shared__ int sm[];
  int* tok = sm;                      // [batch + 1] first token
  int* take = tok + p.batch + 1;      // [batch + 1] first page taken
  int* give = take + p.batch + 1;     // [batch + 1] first page given back
  int* keeps = give + p.batch + 1;    // [batch]
  int* haves = keeps + p.batch;       // [batch] pages held before
  __shared__ int64_t warp_sum[kPlanThreads / 32][3];
  __shared__ int bad_any, last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << p.page_shift;
  if (tid == 0) bad_any = 0;
  const int taken = *p.taken;

  // ---- this thread's sequences, then sums over the block. In 64 bits: what does not fit is found here
  const int per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  int64_t sum[3] = {0, 0, 0};
  bool bad = taken < 0 || taken > p.pages;
  for (int b = b0; b < b1; ++b) {
    const int64_t old = p.old[b], add = p.add[b], keep = p.keep ? p.keep[b] : old;
    const int64_t have = (old + page - 1) >> p.page_shift, want = (keep + add + page - 1) >> p.page_shift;
    if (keep < 0 || add < 0 || keep > old || max(have, want) > p.blocks || keep + add + p.first > INT32_MAX) {
      bad = true;
      break;
    }
    keeps[b] = (int)keep;
    haves[b] = (int)have;
    tok[b] = (int)add;
    take[b] = (int)max((int64_t)0, want - have);
    give[b] = (int)max((int64_t)0, have - want);
    sum[0] += add;
    sum[1] += take[b];
    sum[2] += give[b];
  }
  int64_t at[3];  // before this thread
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int64_t x = sum[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    at[i] = x - sum[i];
    if (lane == 31) warp_sum[warp][i] = x;
  }
  __syncthreads();
  if (bad) bad_any = 1;
  int64_t all[3] = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (w < warp) at[i] += warp_sum[w][i];
      all[i] += warp_sum[w][i];
    }
  __syncthreads();
  const bool ok = !bad_any && all[0] <= p.tokens && all[2] <= taken && all[1] <= p.pages - taken + all[2];
  if (ok) {
    for (int b = b0; b < b1; ++b) {
      const int n[3] = {tok[b], take[b], give[b]};
      tok[b] = (int)at[0];
      take[b] = (int)at[1];
      give[b] = (int)at[2];
#pragma unroll
      for (int i = 0; i < 3; ++i) at[i] += n[i];
    }
    if (tid == 0) {
      tok[p.batch] = (int)all[0];
      take[p.batch] = (int)all[1];
      give[p.batch] = (int)all[2];
    }
  } else if (tid == 0) {
    set_dev_error(p.err, kDevBadArgs);
  }
  __syncthreads();
  const int total = ok ? (int)all[0] : 0, takes = ok ? (int)all[1] : 0, gives = ok ? (int)all[2] : 0;
  const int top = taken - gives;  // of the stack, once the pages are back on it

  auto want_of = [&](int b) { return (keeps[b] + (tok[b + 1] - tok[b]) + page - 1) >> p.page_shift; };
  auto entry = [&](int b, int j) -> int32_t& {
    const bool in = WX_IN_BOUNDS(p.err, b >= 0 && b < p.batch && j >= 0 && j < p.blocks);
    return p.table[in ? b * p.blocks + j : 0];
  };
  // k-th page given back (the giver's entries behind its last page are not written)
  auto given = [&](int k) -> int32_t {
    const int b = last_at(give, p.batch, k);
    return entry(b, want_of(b) + k - give[b]);
  };
  // k-th page taken: those given back come first
  auto fresh = [&](int k) -> int32_t {
    if (k < gives) return given(k);
    const bool in = WX_IN_BOUNDS(p.err, top + k >= 0 && top + k < p.pages);
    return p.free_pages[in ? top + k : 0];
  };

  const int64_t step = (int64_t)gridDim.x * kPlanThreads, from = (int64_t)blockIdx.x * kPlanThreads + tid;
  for (int64_t t = from; t < p.tokens; t += step) {
    int64_t slot = -1, pos = 0;
    if (t < total) {
      const int b = last_at(tok, p.batch, (int)t);
      const int i = keeps[b] + (int)t - tok[b], j = i >> p.page_shift;
      const int pg = j < haves[b] ? entry(b, j) : fresh(take[b] + j - haves[b]);
      pos = p.first + i;
      if (pg < 0 || pg >= p.pages) set_dev_error(p.err, kDevBadArgs);
      else slot = ((int64_t)pg << p.page_shift) | (i & (page - 1));
    }
    p.positions[t] = (int)pos;
    p.slots[t] = slot;
  }
  for (int64_t k = from; k < takes; k += step) {
    const int b = last_at(take, p.batch, (int)k);
    entry(b, haves[b] + (int)k - take[b]) = fresh((int)k);
  }
  for (int64_t k = from; k < gives; k += step) {
    const bool in = WX_IN_BOUNDS(p.err, top + k >= 0 && top + k < p.pages);
    if (in) p.free_pages[top + k] = given((int)k);
  }
  for (int64_t b = from; b <= p.batch; b += step) p.cu[b] = ok ? tok[b] : 0;

  // ---- the last CTA brings lengths and stack up to date: every other has read them
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    last = gridDim.x == 1 || atomicAdd(p.arrived, 1) == (int)gridDim.x - 1;
    if (last && gridDim.x > 1) *p.arrived = 0;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  for (int b = tid; b < p.batch; b += kPlanThreads) p.lens[b] = ok ? keeps[b] + tok[b + 1] - tok[b] : p.old[b];
  if (tid == 0) *p.taken_out = taken - gives + takes;
}

}  // namespace wx

using namespace wx;

extern "C" {

int wx_page_plan(wx_ctx* ctx, const wx_page_pool* pool, const int32_t* keep, const int32_t* add, int64_t tokens,
                 int64_t first_position, int32_t* positions, int64_t* slots, int32_t* cu, int32_t* kv_lens,
                 int32_t* taken_out) {
  DeviceScope on_device(ctx);
  WX_CHECK_ARG(ctx, ctx && pool && tokens >= 0 && tokens <= INT32_MAX);
  WX_CHECK_ARG(ctx, first_position >= 0 && first_position <= INT32_MAX);
  WX_CHECK_ARG(ctx, pool->batch >= 0 && pool->pages > 0 && pool->blocks_per_seq > 0);
  if (pool->page_size < 16 || pool->page_size > 256 || (pool->page_size & (pool->page_size - 1)))
    return set_error(ctx, WX_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)", pool->page_size);
  if (pool->batch > kPlanMaxBatch)
    return set_error(ctx, WX_ERR_UNSUPPORTED, "at most %d sequences in a plan (got %d)", kPlanMaxBatch, pool->batch);
  WX_CHECK_ARG(ctx, pool->pages <= INT32_MAX && pool->blocks_per_seq <= INT32_MAX / pool->page_size);
  WX_CHECK_ARG(ctx, pool->free_pages && pool->taken && cu && taken_out);
  WX_CHECK_ARG(ctx, pool->batch == 0 || (pool->lens && pool->table && add && kv_lens));
  WX_CHECK_ARG(ctx, tokens == 0 || (positions && slots));
  PlanParams p{};
  p.old = pool->lens;
  p.keep = keep;
  p.add = add;
  p.taken = pool->taken;
  p.table = pool->table;
  p.free_pages = pool->free_pages;
  p.blocks = pool->blocks_per_seq;
  p.pages = pool->pages;
  p.tokens = tokens;
  p.first = first_position;
  p.batch = pool->batch;
  p.page_shift = __builtin_ctz((unsigned)pool->page_size);
  p.positions = positions;
  p.slots = slots;
  p.cu = cu;
  p.lens = kv_lens;
  p.taken_out = taken_out;
  p.err = ctx->dev_err;
  const int smem = (5 * p.batch + 3) * 4;
  int st = WX_OK;
  if (smem > 32 * 1024 &&
      (st = ensure_smem_attr(ctx, (const void*)page_plan_kernel, (5 * kPlanMaxBatch + 3) * 4, "page_plan")))
    return st;
  // a CTA for 512 tokens: each makes the sums for itself, and the batch is at most 16 sequences a thread
  const int grid = (int)std::min<int64_t>(ctx->num_sms, std::max<int64_t>(1, (tokens + kPlanThreads - 1) / kPlanThreads));
  if (grid > 1) {
    if (!workspace(ctx, 256, &st)) return st;  // (finds out whether the stream is being captured)
    if (!(p.arrived = arrival_counters(ctx, 1, &st))) return st;
  }
  ProfScope prof(ctx, kProfOther);
  page_plan_kernel<<<grid, kPlanThreads, smem, ctx->stream>>>(p);
  return launch_status(ctx, "page_plan");
}

}  // extern "C"
