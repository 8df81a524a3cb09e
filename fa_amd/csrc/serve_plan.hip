// Block tables and slot maps from request lengths, in one launch.
//
// With n_b new tokens behind p_b stored ones and pages of P tokens, request b
// needs need_b = ceil((p_b + n_b) / P) - ceil(p_b / P) pages. Exclusive sums of
// n (starts) and need (first) over the requests give every token and every new
// page its request: token t belongs to the last b with starts[b] <= t, new page
// k to the last b with first[b] <= k. The work is two integers written a token
// and one a new page, so a launch is bound by its latency, not by bandwidth:
// every workgroup makes both sums over all requests for itself in LDS (two
// loads a request, in parallel) instead of waiting for a first kernel's, and
// finds a token's request by a binary search there. 48 requests of one token take
// 3.5 us, 300 requests with 90 prompts (54000 tokens, 450 KB) 4.8.

#include "serve_common.h"

namespace {

constexpr int PLAN_THREADS = 256;
constexpr int PLAN_BATCH = 4096;            // requests: three LDS words each
constexpr unsigned PLAN_GRID = 1024;

struct PlanArgs {
  const int *past, *fresh;
  int* table;
  const int *pages, *taken;
  int *starts, *lengths, *positions, *slots, *taken_out;
  int64_t table_stride;
  int batch, tokens, shift, max_pages, pages_count;
};

// The last b in [0, batch) with at[b] <= x (at[0] = 0 <= x).
__device__ __forceinline__ int owner(const int* at, int batch, int x) {
  int lo = 0, n = batch;
  while (n > 1) {
    const int half = n >> 1;
    if (at[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) fa_serve_plan_kernel(PlanArgs a) {
  extern __shared__ int lds[];
  int* starts = lds;                        // exclusive sums of the new tokens
  int* first = lds + a.batch;               // and of the new pages
  int* past = lds + 2 * a.batch;
  __shared__ uint64_t wave_sum[PLAN_THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t round = ((int64_t)1 << a.shift) - 1;
  const int taken = *a.taken;
  // Both sums at once, tokens in the upper and pages in the lower half of a
  // 64-bit word, 256 requests at a time.
  uint64_t carry = 0;
  for (int b0 = 0; b0 < a.batch; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    int64_t p = 0, n = 0;
    if (b < a.batch) {
      p = max(a.past[b], 0);
      n = max(a.fresh[b], 0);
    }
    const uint64_t mine = (uint64_t)n << 32 | (uint64_t)(((p + n + round) >> a.shift) - ((p + round) >> a.shift));
    uint64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t other = __shfl_up(sum, d);
      if (lane >= d) sum += other;
    }
    __syncthreads();                        // the last round's wave sums have been read
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    uint64_t before = carry;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; ++w) {
      if (w < wave) before += wave_sum[w];
      carry += wave_sum[w];
    }
    if (b < a.batch) {
      const uint64_t at = before + sum - mine;
      starts[b] = (int)(at >> 32);
      first[b] = (int)at;
      past[b] = (int)p;
      if (blockIdx.x == 0) {
        a.starts[b] = (int)(at >> 32);
        a.lengths[b] = (int)min(p + n, (int64_t)INT32_MAX);
      }
    }
  }
  const int total = (int)(carry >> 32), need = (int)carry;
  if (blockIdx.x == 0 && tid == 0) {
    a.starts[a.batch] = total;
    *a.taken_out = taken + need;
  }
  __syncthreads();
  // The page of column `column` of request b; -1 where there is none. Columns
  // that held pages before this call are read from the table, which gets
  // nothing but the others' here.
  auto held = [&](int b) { return (int)(((int64_t)past[b] + round) >> a.shift); };
  auto fresh_page = [&](int b, int column) {
    const int64_t i = (int64_t)taken + first[b] + column - held(b);
    return i >= 0 && i < a.pages_count ? a.pages[i] : -1;
  };
  const int step = gridDim.x * PLAN_THREADS;
  for (int64_t t = (int64_t)blockIdx.x * PLAN_THREADS + tid; t < a.tokens; t += step) {
    int position = 0, slot = -1;
    if (t < total) {
      const int b = owner(starts, a.batch, (int)t);
      position = past[b] + (int)t - starts[b];
      const int column = position >> a.shift;
      if ((unsigned)column < (unsigned)a.max_pages) {
        const int page = column < held(b) ? a.table[(int64_t)b * a.table_stride + column]
                                          : fresh_page(b, column);
        const int64_t s = ((int64_t)page << a.shift) + (position & round);
        slot = page >= 0 && s <= INT32_MAX ? (int)s : -1;
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  for (int64_t k = (int64_t)blockIdx.x * PLAN_THREADS + tid; k < need; k += step) {
    const int b = owner(first, a.batch, (int)k);
    const int column = held(b) + (int)k - first[b];
    if (column < a.max_pages) a.table[(int64_t)b * a.table_stride + column] = fresh_page(b, column);
  }
}

}  // namespace

extern "C" {

int fa_plan_pages(const fa_page_plan* p, const int32_t* past, const int32_t* fresh, int32_t* table,
                  const int32_t* pages, const int32_t* taken, int32_t* starts, int32_t* lengths,
                  int32_t* positions, int32_t* slots, int32_t* taken_out, void* stream) {
  if (!p) return FA_SERVE_ERR_NULL;
  const int64_t limit = (int64_t)1 << 30;
  if (p->batch < 1 || p->batch > PLAN_BATCH || p->tokens < 0 || p->tokens > limit || p->max_pages < 1 ||
      p->max_pages > limit || p->pages_count < 0 || p->pages_count > limit)
    return FA_SERVE_ERR_GEOMETRY;
  const int shift = page_shift(p->page_size);
  if (shift < 0) return FA_SERVE_ERR_PAGE;
  if (p->table_stride < p->max_pages || p->table_stride > limit) return FA_SERVE_ERR_STRIDE;
  if (!past || !fresh || !table || !taken || !starts || !lengths || !taken_out ||
      (p->pages_count && !pages) || (p->tokens && (!positions || !slots)))
    return FA_SERVE_ERR_NULL;
  for (const void* ptr : {(const void*)past, (const void*)fresh, (const void*)table, (const void*)pages,
                          (const void*)taken, (const void*)starts, (const void*)lengths,
                          (const void*)positions, (const void*)slots, (const void*)taken_out})
    if (!aligned(ptr, 4)) return FA_SERVE_ERR_ALIGN;
  const int rc = check_stream_device(stream);
  if (rc) return rc;
  PlanArgs a{past, fresh, table, pages, taken, starts, lengths, positions, slots, taken_out,
             p->table_stride, (int)p->batch, (int)p->tokens, shift, (int)p->max_pages,
             (int)p->pages_count};
  void* args[] = {&a};
  const int64_t wanted = (p->tokens + PLAN_THREADS - 1) / PLAN_THREADS;
  const unsigned grid = wanted < 1 ? 1 : wanted > PLAN_GRID ? PLAN_GRID : (unsigned)wanted;
  return enqueue(reinterpret_cast<const void*>(&fa_serve_plan_kernel), dim3(grid), dim3(PLAN_THREADS),
                 args, (unsigned)(3 * p->batch * sizeof(int)), stream);
}

}  // extern "C"
