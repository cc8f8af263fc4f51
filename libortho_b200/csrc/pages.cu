// Pages, slots and positions of a step's new tokens from the requests' lengths: running sums of two small quantities per request
// (tokens and new pages), then one independent lookup per page and per token.
//
//     c, f = cached, fresh;  have = min(ceil(c / P), W), want = min(ceil((c + f) / P), W)   (W: columns of the table)
//     starts = exclusive sums of f, first = exclusive sums of want - have
//     block_table[b][have + j] = free[n - 1 - (first[b] + j)], -1 where none is left;  slot of token t of b = page(c + t - starts[b]) * P + (c + t - starts[b]) % P
//
// 16 bytes per request and per token, 8 per page: bound by latency (a load of the lengths, the sums, a load of the page).  Every CTA forms
// the sums of all requests for itself, a chunk of them at a time in shared memory, and serves its share of the tokens and pages, so
// that one launch does and nothing passes between CTAs.  256 decoding requests 4.0 us, 61 requests with 28,479 new tokens 3.8 us of GPU time.
#include "launch.cuh"

namespace ob {

constexpr int kPageThreads = 512;

struct PageSums { unsigned long long tokens, pages; };

__device__ __forceinline__ PageSums operator+(PageSums a, PageSums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

// largest i in [0, n) with start[i] <= v; start[0] <= v
__device__ __forceinline__ int last_not_above(const unsigned long long *start, int n, unsigned long long v)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int32_t as_count(unsigned long long v) { return v > 0x7FFFFFFFull ? 0x7FFFFFFF : (int32_t)v; }

__global__ void __launch_bounds__(kPageThreads)
page_step_kernel(ortho_b200_page_step_desc d)
{
    __shared__ unsigned long long tokens_at[kPageThreads], pages_at[kPageThreads];
    __shared__ uint32_t cached_of[kPageThreads], have_of[kPageThreads];
    __shared__ PageSums warp_sum[kPageThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t P = (uint32_t)d.page_size, W = d.width < 0xFFFFFFFFll ? (uint32_t)d.width : 0xFFFFFFFFu;
    const unsigned long long share = ((unsigned long long)d.tokens + gridDim.x - 1) / gridDim.x;
    const unsigned long long t0 = share * blockIdx.x, t1 = t0 + share < (unsigned long long)d.tokens ? t0 + share : (unsigned long long)d.tokens;
    griddep_wait();
    griddep_launch();
    const int32_t n_raw = *d.available;
    const unsigned long long n = n_raw <= 0 ? 0 : n_raw < d.free_count ? (unsigned long long)n_raw : (unsigned long long)d.free_count;
    auto new_page = [&](unsigned long long i) { return i < n ? d.free_pages[n - 1 - i] : -1; };
    PageSums before = {0, 0};                    // of the chunks before this one
    for (int64_t b0 = 0; b0 < d.requests; b0 += kPageThreads) {
        const int64_t b = b0 + tid;
        const int in_chunk = d.requests - b0 < kPageThreads ? (int)(d.requests - b0) : kPageThreads;
        uint32_t c = 0, f = 0;
        if (b < d.requests) {
            c = (uint32_t)max(d.cached[b], 0);
            f = (uint32_t)max(d.fresh[b], 0);
        }
        // (only pages that the table has a column for: one without could not be given back)
        const uint32_t all = c + f, have = min(c / P + (c % P != 0), W), want = min(all / P + (all % P != 0), W);
        PageSums mine = {f, want - have}, sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const PageSums up = {__shfl_up_sync(0xffffffffu, sum.tokens, o), __shfl_up_sync(0xffffffffu, sum.pages, o)};
            if (lane >= o) sum = sum + up;
        }
        __syncthreads();                         // the chunk before has been served
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        PageSums total = before;
#pragma unroll
        for (int w = 0; w < kPageThreads / 32; w++) {
            if (w == warp) sum = sum + total;
            total = total + warp_sum[w];
        }
        const PageSums first = {sum.tokens - mine.tokens, sum.pages - mine.pages};
        tokens_at[tid] = first.tokens;
        pages_at[tid] = first.pages;
        cached_of[tid] = c;
        have_of[tid] = have;
        if (b < d.requests && blockIdx.x == (b0 / kPageThreads) % gridDim.x) {
            d.lengths[b] = as_count(all);
            d.starts[b] = as_count(first.tokens);
        }
        __syncthreads();
        // a column that gets no page says so: what it held may be another request's by now
        for (unsigned long long p = before.pages + (unsigned long long)blockIdx.x * kPageThreads + tid; p < total.pages;
             p += (unsigned long long)gridDim.x * kPageThreads) {
            const int i = last_not_above(pages_at, in_chunk, p);
            const unsigned long long col = have_of[i] + (p - pages_at[i]);
            d.block_table[(b0 + i) * d.table_stride + (int64_t)col] = max(new_page(p), -1);
        }
        const unsigned long long from = before.tokens > t0 ? before.tokens : t0, to = total.tokens < t1 ? total.tokens : t1;
        for (unsigned long long t = from + tid; t < to; t += kPageThreads) {
            const int i = last_not_above(tokens_at, in_chunk, t);
            const uint32_t pos = cached_of[i] + (uint32_t)(t - tokens_at[i]), col = pos / P;
            int32_t page = -1;
            if (col < W)
                page = col < have_of[i] ? d.block_table[(b0 + i) * d.table_stride + col] : new_page(pages_at[i] + (col - have_of[i]));
            d.slots[t] = page >= 0 ? (int64_t)page * P + pos % P : -1;
            d.positions[t] = (int32_t)min(pos, 0x7FFFFFFFu);
            d.request_of[t] = (int32_t)(b0 + i);
        }
        before = total;
    }
    for (unsigned long long t = (before.tokens > t0 ? before.tokens : t0) + tid; t < t1; t += kPageThreads) {
        d.slots[t] = -1;
        d.positions[t] = -1;
        d.request_of[t] = -1;
    }
    if (blockIdx.x == 0 && tid == 0) {
        d.starts[d.requests] = as_count(before.tokens);
        d.counts[0] = as_count(before.tokens);
        d.counts[1] = as_count(before.pages);
        d.counts[2] = as_count(before.pages < n ? n - before.pages : 0);
    }
}

}  // namespace ob

using namespace ob;

extern "C" int ortho_b200_page_step(const ortho_b200_page_step_desc *d, void *stream)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->requests < 0 || d->width < 0 || d->free_count < 0 || d->tokens < 0 || d->page_size < 1 || d->page_size > 0x7FFFFFFF
        || d->requests > 0x7FFFFFFF || d->tokens > 0x7FFFFFFF || d->free_count > 0x7FFFFFFF) return ORTHO_B200_ERR_SHAPE;
    if (!d->starts || !d->counts || !d->available) return ORTHO_B200_ERR_NULL;
    if (d->requests && (!d->cached || !d->fresh || !d->lengths || (d->width && !d->block_table))) return ORTHO_B200_ERR_NULL;
    if (d->free_count && !d->free_pages) return ORTHO_B200_ERR_NULL;
    if (d->tokens && (!d->slots || !d->positions || !d->request_of)) return ORTHO_B200_ERR_NULL;
    const int st = check_device();
    if (st) return st;
    // Where this step's lengths take the place of the last one's, or its counts those that `available` lies in, no CTA may write them while another
    // still reads: one CTA does it all then, whose threads read theirs first.
    auto meet = [](const int32_t *a, int64_t n, const int32_t *b, int64_t m) { return a < b + m && b < a + n; };
    const bool in_place = meet(d->lengths, d->requests, d->cached, d->requests) || meet(d->counts, 3, d->available, 1);
    const int64_t sms = in_place ? 1 : device_sm_count(current_device_index()), want = ceil_div(d->tokens, kPageThreads);
    return launch_dependent(page_step_kernel, dim3((unsigned)(want < 1 ? 1 : want < sms ? want : sms)), kPageThreads, 0, (cudaStream_t)stream, *d);
}
