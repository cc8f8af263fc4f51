// Attention of one new token per row over a paged key-value cache (one source for both 16-bit types):
//
//     s_j = scale q . k_j,   out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max),   lse = max + log sum_j exp(s_j - max)
//
// Keys and values are read once and dominate everything else: with G query heads per key-value head there are G multiplications a byte.
// So the cache streams through shared memory by asynchronous 16-byte copies, a ring of its own per warp (no barrier per tile), and all
// query heads of a key-value head meet every key as the 8-column operand of m16n8k16 products: S^T = K Q^T (16 keys x 8 queries), running
// maximum and sum per query in FP32, then O^T += V^T P^T (16 elements x 8 queries).  Queries are the narrow operand because there are few of
// them; P^T gets from accumulator to operand layout by an 8 x 8 transposition in registers.
//
// The work is cut evenly whatever the lengths are.  A unit is 64 keys of one request and key-value head (16 per warp); a request and head ("an
// item") costs its units and one more for its start and end.  These costs are numbered in a row over all requests, and CTA c takes
// [c per, (c + 1) per) of them: every CTA finds its place by summing the lengths itself.  An item that lies within one CTA is
// finished there; of one that is cut each CTA leaves its sums in the workspace, and join_kernel, launched behind as a programmatic
// dependent, adds them in order.  Few items (CLUSTER): a cluster of CTAs has an item and joins its sums through distributed shared memory.
// Neither uses atomics: the same bits every time.
// Measured (GPU time, us): 2 x 131072 keys of 8 heads of 128, 1.07 GB: 163 to 166 = 6.5 TB/s, 184 = 5.8 TB/s in long runs at the clock that the power cap leaves;
// 32 requests of up to 4096 keys, log-spread, 74 MB: 22.8, of which 2.6 pass before the first copy (lengths, place, pages, each from memory) and 4.2
// with join_kernel; 1 x 1000 keys of 32 heads, 16 MB: 6.2.  Joining cut items in this kernel, by the last CTA to count itself in, took 7 us more than
// join_kernel (fence, counter, two rounds of reads, one after the other in one CTA).
#pragma once

#include "launch.cuh"
#include "tma.cuh"

namespace ob {

struct AttentionArgs {
    ortho_b200_paged_attention_desc d;
    FastDiv by_page;
    float scale_log2;                            // scale log2 e: exponentials are powers of two
    int per_group, groups;                       // query heads of a key-value head in one unit, units' groups of them
    int ctas;
    int4 *cut;                                   // [ctas] of a CTA's last item: {row, head group, last CTA, 1} if it goes on, {.., 0} if not
    float2 *sums;                                // [2 ctas][rows] (max, sum) of cut items: continued from the CTA before, going on behind
    float *part;                                 // [2 ctas][rows][head_dim]
};

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps, kWarpKeys = 16, kUnitKeys = kWarpKeys * kAttnWarps;

// Probabilities are powers of two of s - reference + lift.  The reference is the running maximum, but it stays where it is until a score is kSlack above it:
// the search for the maximum over the lanes and the scaling of what has been summed are then left out in almost every tile, and the result does
// not depend on the reference.  In FP16 the largest probability is 2^15 and what is 2^-32 of the reference still has a value.
constexpr float kSlack = 7.f;
template <class T> struct AttnType;
template <> struct AttnType<__half> {
    static constexpr float lift = 8.f, below = 1.f - 1.f / 1024.f;
    static __device__ __forceinline__ uint32_t pack_rz(float lo, float hi)
    {
        uint32_t r;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct AttnType<__nv_bfloat16> {
    static constexpr float lift = 0.f, below = 1.f - 1.f / 128.f;
    static __device__ __forceinline__ uint32_t pack_rz(float lo, float hi)
    {
        uint32_t r;
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// Shared memory of one CTA.  Rows of DP elements: 16-byte chunks exchanged within groups of eight by the row's number where a row is a multiple of
// 128 bytes, 16 bytes of padding elsewhere; both put the eight rows that one ldmatrix phase reads into different banks.
template <int DP, int NT>
struct AttnShape {
    static constexpr bool kSwap = DP % 64 == 0;
    static constexpr int kPitch = DP * 2 + (kSwap ? 0 : 16), kChunks = DP / 8;
    static constexpr int kHalfTile = kWarpKeys * kPitch;                       // keys, then values
    static constexpr int kStage = 2 * kHalfTile;
    static constexpr int kQ = NT * 8 * kPitch;
    static constexpr int kFoldPitch = DP + 4;                                  // 8 queries of a warp in FP32, rows apart by 4 banks: in a stage that is done with
    static_assert(8 * kFoldPitch * 4 <= kStage, "room for 8 queries");
    static constexpr int bytes(int stages) { return stages * (kAttnWarps * kStage + kQ) + kAttnWarps * NT * 8 * 8 + kAttnWarps * stages * 4 + 64; }
    // Room of a CTA with three, two or one on an SM.  Three where registers and a ring of two stages allow it, up to 8 queries and head dims up to 112:
    // a CTA waits for its own chain of steps in every unit, which more warps fill (3 against 2, us: heads of 64, 200 requests of 1000 keys with 4 key-value
    // heads 46.7, 59.5; of 96 75, 79; of 112, 2 x 32768 keys with 8 heads 50, 62; of 128 53.7, 51.5: two).
    static constexpr int kThree = 73728, kTwo = 115712, kOne = 232448;
    static constexpr bool kTriple = NT == 1 && DP <= 112 && bytes(2) <= kThree;
    static constexpr int kRoom = kTriple ? kThree : bytes(2) <= kTwo ? kTwo : kOne;
    static constexpr int kStages = bytes(4) <= kRoom ? 4 : bytes(3) <= kRoom ? 3 : 2, kBytes = bytes(kStages), kPerSm = kTriple ? 3 : kBytes <= kTwo ? 2 : 1;
    static constexpr int kMostRanks = 8;                                       // of a cluster; what arrives from them: (max, sum) and a share of the sums
    static constexpr int kArrived = kMostRanks * NT * 8 * 8 + NT * 8 * DP * 4 + kMostRanks * 16, kClusterBytes = (kBytes + 15) / 16 * 16 + kArrived;
    static constexpr int kClusterPerSm = kTriple && kClusterBytes <= kThree + 2048 ? 3 : kClusterBytes <= kTwo ? 2 : kClusterBytes <= kOne ? 1 : 0;
    static constexpr bool kKeepQ = NT <= 2;                                    // query operands stay in registers
    static __device__ __forceinline__ uint32_t at(int row, int chunk) { return (uint32_t)(row * kPitch + ((kSwap ? chunk ^ (row & 7) : chunk) << 4)); }
};

// One request as the units of UNIT keys see it
struct Span { int from, n, units; int64_t row; };
template <int UNIT>
__device__ __forceinline__ Span span_of(const ortho_b200_paged_attention_desc &d, int64_t b)
{
    Span s;
    s.row = d.row_of ? (int64_t)d.row_of[b] : b;
    const int most = (int)(d.width * d.page_size);
    int n = s.row >= 0 && s.row < d.rows ? d.lengths[b] : 0;
    n = n < 0 ? 0 : n < most ? n : most;
    s.n = n;
    s.from = d.window > 0 && n > d.window ? n - (int)d.window : 0;
    s.units = (n - s.from + UNIT - 1) / UNIT;
    return s;
}

// Place in the row of all units: request, head group, UNIT keys.  `left`: costs up to the end of this CTA's share, the unit's own among them.  In a
// cluster a CTA has every `stride`-th unit of one item.
template <int UNIT>
struct Walk {
    int64_t b;
    int inner, unit;
    Span s;
    long long left;
    __device__ __forceinline__ bool last() const { return unit == s.units - 1; }
    template <bool CLUSTER> __device__ __forceinline__ bool more(int stride) const { return CLUSTER ? unit + stride < s.units : left > (last() ? 2 : 1); }
    template <bool CLUSTER> __device__ __forceinline__ void step(const ortho_b200_paged_attention_desc &d, int inners, int stride)
    {
        if constexpr (CLUSTER) {
            unit += stride;
        } else {
            left--;
            if (++unit < s.units) return;
            left--;
            unit = 0;
            if (++inner < inners) return;
            inner = 0;
            do b++, s = b < d.batch ? span_of<UNIT>(d, b) : Span{0, 0, 1, 0}; while (s.units == 0);
        }
    }
};

// A CTA's first unit, and how many costs it has.  per: costs of a CTA; item_at: number of the item's first cost.
template <int UNIT, bool CLUSTER>
__device__ __forceinline__ Walk<UNIT> first_unit(const ortho_b200_paged_attention_desc &d, int inners, int ctas, int rank, int ranks, long long &per, long long &item_at)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
    Walk<UNIT> now;
    now.left = 0;
    if constexpr (CLUSTER) {                     // every ranks-th unit of the cluster's item
        const int64_t item = cta / ranks;
        now.b = item / inners;
        now.inner = (int)(item - now.b * inners);
        now.unit = rank;
        now.s = span_of<UNIT>(d, now.b);
        now.left = rank < now.s.units;
    } else {
        __shared__ long long warp_cost[kAttnWarps], first_rest;
        __shared__ int first_b;
        // a thread's requests, one after the other; up to kAttnThreads requests each thread has one
        const int64_t chunk = (d.batch + kAttnThreads - 1) / kAttnThreads, b0 = tid * chunk, b1 = b0 + chunk < d.batch ? b0 + chunk : d.batch;
        long long mine = 0;
        for (int64_t b = b0; b < b1; b++) {
            const int units = span_of<UNIT>(d, b).units;
            mine += units + (units > 0);
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) warp_cost[warp] = upto;
        __syncthreads();
        long long total = 0;
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            if (w == warp) upto += total;
            total += warp_cost[w];
        }
        total *= inners;
        // (32 bits where they do: a division in 64 takes some 200 cycles)
        per = total < 0x7FFFFFFF ? ((uint32_t)total + ctas - 1) / (uint32_t)ctas : (total + ctas - 1) / ctas;
        const long long from = per * cta, to = from + per < total ? from + per : total;
        long long rest = from - (upto - mine) * inners;
        if (from < to && rest >= 0 && rest < mine * inners) {
            int64_t b = b0;
            for (; b + 1 < b1; b++) {
                const int units = span_of<UNIT>(d, b).units;
                const long long here = (long long)(units + (units > 0)) * inners;
                if (rest < here) break;
                rest -= here;
            }
            first_b = (int)b;
            first_rest = rest;
        }
        __syncthreads();
        if (from < to) {
            now.b = first_b;
            now.s = span_of<UNIT>(d, now.b);
            const long long rest = first_rest;
            now.inner = rest < 0x7FFFFFFF ? (int)((uint32_t)rest / (uint32_t)(now.s.units + 1)) : (int)(rest / (now.s.units + 1));
            const int at = (int)(rest - (long long)now.inner * (now.s.units + 1));                // 0: the cost of the item's start and end, then its units
            now.unit = at > 0 ? at - 1 : 0;
            now.left = to - from - (at == 0);
            item_at = from - at;
        }
    }
    return now;
}

template <class T>
__device__ __forceinline__ void store4(const ortho_b200_paged_attention_desc &d, int64_t b, int64_t head, int el, float4 x, float inverse)
{
    uint2 r;
    r.x = Half<T>::pack(x.x * inverse, x.y * inverse);
    r.y = Half<T>::pack(x.z * inverse, x.w * inverse);
    *reinterpret_cast<uint2 *>((T *)d.out + b * d.out_token_stride + head * d.out_head_stride + el) = r;
}
template <class T>
__device__ __forceinline__ float lse_of(float top, float sum)
{
    return sum == 0.f ? -INFINITY : (top - AttnType<T>::lift + __log2f(sum)) * 0.6931471805599453f;
}

// The four warps' sums over their keys of query t * 8 + (0 .. 7) of an item become one: to the output, to the workspace, or to the cluster's CTAs.
// folds: [warps][8 queries][elements], the warps WARP_FLOATS and the queries FOLD apart; sums: (maximum, sum) of [warps][NT * 8 queries].
template <class T, int DP, int NT, bool CLUSTER, int WARP_FLOATS, int FOLD>
__device__ __forceinline__ void add_warps(const AttentionArgs &a, const float *folds, const float2 *sums, int t, int64_t b, int64_t h0, int heads, bool whole, int64_t slot,
                      int rank, int ranks, float2 *arrived_sums, float4 *arrived)
{
    const auto &d = a.d;
    const int tid = threadIdx.x, D = (int)d.head_dim;
    // a thread has one query and every 16th quad of its elements
    const int fq = tid >> 4, row = t * 8 + fq;
    if (row < heads) {
        float m = -INFINITY, l = 0.f, factor[kAttnWarps];
        float2 x[kAttnWarps];
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            x[w] = sums[w * NT * 8 + row];
            m = fmaxf(m, x[w].x);
        }
#pragma unroll
        for (int w = 0; w < kAttnWarps; w++) {
            factor[w] = x[w].x == -INFINITY ? 0.f : exp2_approx(x[w].x - m);
            l += x[w].x == -INFINITY ? x[w].y : x[w].y * factor[w];               // (nothing, or NaN)
        }
        const float inverse = l == 0.f ? 0.f : 1.f / l;
        if constexpr (CLUSTER) {
            if ((tid & 15) < ranks) st_dsmem_v2(mapa_shared(shared_addr(arrived_sums + rank * NT * 8 + row), tid & 15), m, l);
        } else if ((tid & 15) == 0) {
            if (!whole) a.sums[slot * NT * 8 + row] = make_float2(m, l);
            else if (d.lse) d.lse[b * d.q_heads + h0 + row] = lse_of<T>(m, l);
        }
#pragma unroll
        for (int i = 0; i < (DP + 63) / 64; i++) {
            const int el = i * 64 + (tid & 15) * 4;
            if (el >= D) break;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kAttnWarps; w++) {
                const float4 z = *reinterpret_cast<const float4 *>(folds + w * WARP_FLOATS + fq * FOLD + el);
                y.x += factor[w] * z.x; y.y += factor[w] * z.y; y.z += factor[w] * z.z; y.w += factor[w] * z.w;
            }
            if constexpr (CLUSTER) {
                const int share = (heads * (D / 4) + ranks - 1) / ranks, at = row * (D / 4) + el / 4, to = at / share;
                st_dsmem_v4(mapa_shared(shared_addr(arrived + rank * share + (at - to * share)), to), y);
            } else if (whole) store4<T>(d, b, h0 + row, el, y, inverse);
            else *reinterpret_cast<float4 *>(a.part + (slot * NT * 8 + row) * D + el) = y;
        }
    }
}

// This CTA's share of an item's elements from what its cluster's CTAs have sent
template <class T, int NT, int MOST>
__device__ __forceinline__ void add_cluster(const AttentionArgs &a, int64_t b, int64_t h0, int heads, int rank, int ranks, const float2 *arrived_sums, const float4 *arrived)
{
    const auto &d = a.d;
    const int tid = threadIdx.x, D = (int)d.head_dim;
    const int quads = D / 4, share = (heads * quads + ranks - 1) / ranks;
    for (int i = tid; i < share; i += kAttnThreads) {
        const int at = rank * share + i, row = at / quads, el = (at - row * quads) * 4;
        if (row >= heads) break;
        float m = -INFINITY, l = 0.f;
        float2 x[MOST];
        float4 z[MOST], y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < MOST; r++) {
            x[r] = r < ranks ? arrived_sums[r * NT * 8 + row] : make_float2(-INFINITY, 0.f);
            // (nothing has arrived from a CTA without keys)
            z[r] = x[r].x == -INFINITY && x[r].y == 0.f ? y : arrived[r * share + i];
            m = fmaxf(m, x[r].x);
        }
#pragma unroll
        for (int r = 0; r < MOST; r++) {
            const float f = x[r].x == -INFINITY ? 0.f : exp2_approx(x[r].x - m);
            l += x[r].x == -INFINITY ? x[r].y : x[r].y * f;
            y.x += f * z[r].x; y.y += f * z[r].y; y.z += f * z[r].z; y.w += f * z[r].w;
        }
        store4<T>(d, b, h0 + row, el, y, l == 0.f ? 0.f : 1.f / l);
        if (d.lse && el == 0) d.lse[b * d.q_heads + h0 + row] = lse_of<T>(m, l);
    }
}

// Rows without keys
template <class T, int UNIT>
__device__ __forceinline__ void empty_rows(const ortho_b200_paged_attention_desc &d)
{
    const int tid = threadIdx.x, D = (int)d.head_dim;
    for (int64_t b = blockIdx.x; b < d.batch; b += gridDim.x) {
        if (span_of<UNIT>(d, b).units) continue;
        const int chunks = D / 8;
        for (int i = tid; i < (int)d.q_heads * chunks; i += kAttnThreads) {
            const int h = i / chunks, c = i - h * chunks;
            *reinterpret_cast<uint4 *>((T *)d.out + b * d.out_token_stride + h * d.out_head_stride + c * 8) = make_uint4(0, 0, 0, 0);
            if (d.lse && c == 0) d.lse[b * d.q_heads + h] = -INFINITY;
        }
    }
}

template <class T, int DP, int NT, bool CLUSTER>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<DP, NT>::kPerSm)
paged_attention_kernel(const __grid_constant__ AttentionArgs a)
{
    using Shape = AttnShape<DP, NT>;
    using Type = AttnType<T>;
    constexpr int S = Shape::kStages, KS = DP / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    const auto &d = a.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, D = (int)d.head_dim;
    unsigned char *const ring = smem + warp * (S * Shape::kStage);
    unsigned char *const q_ring = smem + kAttnWarps * S * Shape::kStage;
    float2 *const sums = reinterpret_cast<float2 *>(q_ring + S * Shape::kQ);
    uint32_t *const seen = reinterpret_cast<uint32_t *>(sums + kAttnWarps * NT * 8) + warp * S;
    const int inners = (int)d.kv_heads * a.groups, cta = blockIdx.x;
    float2 *const arrived_sums = reinterpret_cast<float2 *>(smem + (Shape::kBytes + 15) / 16 * 16);           // [ranks][rows]
    float4 *const arrived = reinterpret_cast<float4 *>(arrived_sums + Shape::kMostRanks * NT * 8);            // [ranks][this CTA's share]

    if constexpr (CLUSTER) cluster_arrive();
    auto others_started = [&]() { if constexpr (CLUSTER) { __syncwarp(); cluster_wait(); } };         // before anything is sent to them, once the first copies are under way
    griddep_wait();
    griddep_launch();

    // ---- this CTA's units -------------------------------------------------------------------------------------
    [[maybe_unused]] long long per = 0, item_at = 0;                           // costs of a CTA; cost number of the item's first cost
    [[maybe_unused]] const int rank = CLUSTER ? (int)cluster_ctarank() : 0, ranks = CLUSTER ? (int)cluster_nctarank() : 1;
    Walk<kUnitKeys> now = first_unit<kUnitKeys, CLUSTER>(d, inners, a.ctas, rank, ranks, per, item_at);       // the unit that is computed
    if (now.left <= 0) {                         // (a share of one cost may be that of an item's start alone)
        others_started();
        if (!CLUSTER && tid == 0) a.cut[cta] = make_int4(0, 0, 0, 0);
    } else {
        // What the copies of a unit need.  The page of a lane's key is looked up well ahead of its use, those of the first units together.
        struct Ticket { int64_t b; int inner, page, place; bool valid, queries; };
        Walk<kUnitKeys> ahead = now;                        // the unit of the next ticket
        bool more_tickets = true;
        auto ticket = [&]() {
            Ticket t;
            t.valid = more_tickets;
            t.b = ahead.b;
            t.inner = ahead.inner;
            t.queries = CLUSTER ? ahead.unit == rank : ahead.unit == 0 || (ahead.b == now.b && ahead.inner == now.inner && ahead.unit == now.unit);
            t.page = -1;
            t.place = 0;
            const int key = ahead.s.from + ahead.unit * kUnitKeys + warp * kWarpKeys + (lane & 15);
            if (more_tickets && key < ahead.s.n) {
                const int col = (int)a.by_page.quotient((uint32_t)key);
                t.place = key - col * (int)d.page_size;
                t.page = d.block_table[ahead.s.row * d.table_stride + col];
            }
            if (more_tickets) {
                more_tickets = ahead.more<CLUSTER>(ranks);
                if (more_tickets) ahead.step<CLUSTER>(d, inners, ranks);
            }
            return t;
        };
        int fresh_q = 0;                         // items issued so far: place in the ring of queries
        const bool alike = d.k_page_stride == d.v_page_stride && d.k_slot_stride == d.v_slot_stride;
        auto issue = [&](const Ticket &t, int stage) {
            if (t.valid) {
                const int head = t.inner / a.groups, group = t.inner - head * a.groups, place = t.place, page = t.page < d.pages ? t.page : -1;
                const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0) & 0xFFFFu;
                if (lane == 0) seen[stage] = ok;
                const uint32_t dst = shared_addr(ring + stage * Shape::kStage);
                const T *const k = (const T *)d.k_cache + head * d.k_head_stride, *const v = (const T *)d.v_cache + head * d.v_head_stride;
                // a lane's own key's place in the caches; the lanes that copy a row get it from there
                const int64_t k_mine = page >= 0 ? page * d.k_page_stride + place * d.k_slot_stride : 0;
                const int64_t v_mine = alike || page < 0 ? k_mine : page * d.v_page_stride + place * d.v_slot_stride;
#pragma unroll
                for (int i = 0; i < Shape::kChunks / 2; i++) {
                    const int at = i * 32 + lane, row = at / Shape::kChunks, chunk = at % Shape::kChunks;
                    const int64_t k_at = __shfl_sync(0xffffffffu, k_mine, row), v_at = alike ? k_at : __shfl_sync(0xffffffffu, v_mine, row);
                    const bool on = (ok >> row & 1) && chunk * 8 < D;          // (else zeros; the address is that of the first page)
                    const int e = chunk * 8 < D ? chunk * 8 : 0;
                    copy16_async(dst + Shape::at(row, chunk), k + k_at + e, on);
                    copy16_async(dst + Shape::kHalfTile + Shape::at(row, chunk), v + v_at + e, on);
                }
                if (t.queries) {                                               // its queries, a quarter per warp
                    const uint32_t qdst = shared_addr(q_ring + fresh_q * Shape::kQ);
                    const int h0 = head * (int)(d.q_heads / d.kv_heads) + group * a.per_group;
                    const int heads = min(a.per_group, (int)(d.q_heads / d.kv_heads) - group * a.per_group);
                    for (int at = tid; at < NT * 8 * Shape::kChunks; at += kAttnThreads) {
                        const int row = at / Shape::kChunks, chunk = at % Shape::kChunks;
                        const bool on = row < heads && chunk * 8 < D;
                        copy16_async(qdst + Shape::at(row, chunk),
                                     (const T *)d.q + t.b * d.q_token_stride + (on ? (h0 + row) * d.q_head_stride + chunk * 8 : 0), on);
                    }
                    if (++fresh_q == S) fresh_q = 0;
                }
            }
            copy_commit();
        };
        Ticket pending;
        {
            Ticket first[S - 1];
#pragma unroll
            for (int i = 0; i < S - 1; i++) first[i] = ticket();
            pending = ticket();
#pragma unroll
            for (int i = 0; i < S - 1; i++) issue(first[i], i);
        }
        others_started();

        uint32_t q[Shape::kKeepQ ? NT : 1][Shape::kKeepQ ? KS : 1][2];
        float o[KS][NT][4], top[NT][2], sum[NT][2];
        int stage = 0, q_at = -1;
        bool started_here = true;                // the request's first unit is this CTA's
        for (bool first_unit = true, more = true; more; first_unit = false) {
            copy_wait<S - 2>();
            __syncwarp();
            if (first_unit || (!CLUSTER && now.unit == 0)) {
                started_here = now.unit == 0;
                if (++q_at == S) q_at = 0;
                __syncthreads();                 // every warp's part of the queries is there, and the sums of the item before are read
                if constexpr (Shape::kKeepQ) {
                    const uint32_t src = shared_addr(q_ring + q_at * Shape::kQ);
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int ks = 0; ks < KS; ks++) ldmatrix2(q[t][ks][0], q[t][ks][1], src + Shape::at(t * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)));
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    top[t][0] = top[t][1] = -INFINITY;
                    sum[t][0] = sum[t][1] = 0.f;
#pragma unroll
                    for (int i = 0; i < KS; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[i][t][e] = 0.f;
                }
            }
            const uint32_t ok = seen[stage];
            const uint32_t keys = shared_addr(ring + stage * Shape::kStage), values = keys + Shape::kHalfTile;
            issue(pending, stage == 0 ? S - 1 : stage - 1);
            pending = ticket();
            if (ok) {
                float s[NT][4], odd[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++) s[t][0] = s[t][1] = s[t][2] = s[t][3] = odd[t][0] = odd[t][1] = odd[t][2] = odd[t][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t k[4];
                    ldmatrix4(k, keys + Shape::at((lane & 7) + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)));
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        uint32_t b0, b1;
                        if constexpr (Shape::kKeepQ) { b0 = q[t][ks][0]; b1 = q[t][ks][1]; }
                        else ldmatrix2(b0, b1, shared_addr(q_ring + q_at * Shape::kQ) + Shape::at(t * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)));
                        Half<T>::mma(NT <= 2 && (ks & 1) ? odd[t] : s[t], k, b0, b1);              // (two chains of products where there are few)
                    }
                }
                if constexpr (NT <= 2) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][e] += odd[t][e];
                }
                // rows (keys) lane / 4 and lane / 4 + 8, columns (queries) 2 (lane % 4) and the next
                const bool on0 = (ok >> (lane >> 2)) & 1, on1 = (ok >> ((lane >> 2) + 8)) & 1;
                bool grows = false;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        s[t][e] = on0 ? s[t][e] * a.scale_log2 : -INFINITY;
                        s[t][e + 2] = on1 ? s[t][e + 2] * a.scale_log2 : -INFINITY;
                        grows = grows || fmaxf(s[t][e], s[t][e + 2]) > top[t][e] + kSlack;
                    }
                if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float keep[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float m = fmaxf(s[t][e], s[t][e + 2]);
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                            m = fmaxf(m, top[t][e]);
                            keep[e] = m == -INFINITY ? 1.f : exp2_approx(top[t][e] - m);
                            top[t][e] = m;
                            sum[t][e] *= keep[e];
                        }
#pragma unroll
                        for (int i = 0; i < KS; i++) {
                            o[i][t][0] *= keep[0]; o[i][t][1] *= keep[1]; o[i][t][2] *= keep[0]; o[i][t][3] *= keep[1];
                        }
                    }
                }
                // Probabilities as two 16-bit parts: one alone would add an error as large as the output's own rounding.  The upper part is kept strictly
                // below the value and the lower above zero: an infinite value then meets two positive factors, as in the formula.  What the two
                // hold is off by up to 2^-14 of it in BF16 (2^-15.7 in the mean square) and 2^-20 in FP16, and the output by no more of sum p |v|; its own
                // rounding is up to 2^-8 and 2^-11.  Of BF16 outputs about one in a hundred comes out as the neighbouring value; the error against 64 bits
                // is that of an FP32 softmax to five digits (131072 keys: 1.64233e-3 and 1.64226e-3).
                uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float base = (top[t][e] == -INFINITY ? 0.f : top[t][e]) - Type::lift;
                        p[e] = exp2_approx(s[t][e] - base);
                        p[e + 2] = exp2_approx(s[t][e + 2] - base);
                        sum[t][e] += p[e] + p[e + 2];
                    }
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint32_t h = Type::pack_rz(p[2 * r] * Type::below, p[2 * r + 1] * Type::below);
                        const float2 f = Half<T>::unpack(h);
                        hi[t][r] = transpose8x8(h);
                        lo[t][r] = transpose8x8(Half<T>::pack(p[2 * r] - f.x, p[2 * r + 1] - f.y));
                    }
                }
#pragma unroll
                for (int i0 = 0; i0 < KS; i0 += 2) {
                    uint32_t v[2][4];
#pragma unroll
                    for (int i = 0; i < 2 && i0 + i < KS; i++)
                        ldmatrix4_trans(v[i], values + Shape::at((lane & 7) + (lane >> 4) * 8, (i0 + i) * 2 + ((lane >> 3) & 1)));
#pragma unroll
                    for (int part = 0; part < 2; part++)
#pragma unroll
                        for (int i = 0; i < 2 && i0 + i < KS; i++)
#pragma unroll
                            for (int t = 0; t < NT; t++)
                                Half<T>::mma(o[i0 + i][t], v[i], part ? lo[t][0] : hi[t][0], part ? lo[t][1] : hi[t][1]);
                }
            }
            const bool last = now.last();
            more = now.more<CLUSTER>(ranks);
            if (CLUSTER ? !more : last || !more) {
                // ---- the four warps' sums over their keys of this item become one.  They pass through the stage that was just used: its next copies are
                // issued behind the barrier above.
                const int head = now.inner / a.groups, group = now.inner - head * a.groups;
                const int64_t h0 = head * (d.q_heads / d.kv_heads) + group * a.per_group;
                const int heads = min(a.per_group, (int)(d.q_heads / d.kv_heads) - group * a.per_group);
                const bool whole = started_here && last;
                const int64_t slot = 2 * (int64_t)cta + (started_here ? 1 : 0);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float l = sum[t][e];
                        l += __shfl_xor_sync(0xffffffffu, l, 4);
                        l += __shfl_xor_sync(0xffffffffu, l, 8);
                        l += __shfl_xor_sync(0xffffffffu, l, 16);
                        if (lane < 4) sums[warp * NT * 8 + t * 8 + 2 * lane + e] = make_float2(top[t][e], l);
                    }
                float *const fold = reinterpret_cast<float *>(ring + stage * Shape::kStage) + 2 * (lane & 3) * Shape::kFoldPitch + (lane >> 2);
                const float *const folds = reinterpret_cast<const float *>(smem + stage * Shape::kStage);
                constexpr int WARP_FLOATS = S * Shape::kStage / 4;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    __syncwarp();                // the warp has read its values
                    if (t) __syncthreads();
#pragma unroll
                    for (int i = 0; i < KS; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) fold[(e & 1) * Shape::kFoldPitch + i * 16 + (e >> 1) * 8] = o[i][t][e];
                    __syncthreads();
                    add_warps<T, DP, NT, CLUSTER, WARP_FLOATS, Shape::kFoldPitch>(a, folds, sums, t, now.b, h0, heads, whole, slot, rank, ranks, arrived_sums, arrived);
                }
                if constexpr (!CLUSTER) {
                    if (!more && tid == 0) a.cut[cta] = make_int4((int)now.b, now.inner, (int)((item_at + now.s.units) / per), started_here && !last ? 1 : 0);
                    item_at += now.s.units + 1;
                }
            }
            if (++stage == S) stage = 0;
            if (more) now.step<CLUSTER>(d, inners, ranks);
        }
        copy_wait<0>();
    }
    if constexpr (CLUSTER) {
        // ---- the cluster's sums become one, a share of the elements in each CTA ----------------------------------------------
        const int head = now.inner / a.groups, group = now.inner - head * a.groups;
        const int64_t h0 = head * (d.q_heads / d.kv_heads) + group * a.per_group;
        const int heads = min(a.per_group, (int)(d.q_heads / d.kv_heads) - group * a.per_group);
        for (int i = tid; i < heads * ranks && now.left <= 0; i += kAttnThreads)                  // no unit: nothing is added
            st_dsmem_v2(mapa_shared(shared_addr(arrived_sums + rank * NT * 8 + i / ranks), i % ranks), -INFINITY, 0.f);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (now.s.units > 0) add_cluster<T, NT, Shape::kMostRanks>(a, now.b, h0, heads, rank, ranks, arrived_sums, arrived);
    }
    empty_rows<T, kUnitKeys>(d);
}

// Adds the parts of an item that was cut, in the order of its keys.  A CTA per CTA of the kernel above (the one where a cut item starts) and
// query head; its warps take every fourth part, a lane four elements (eight: head dims above 128).
template <class T>
__global__ void __launch_bounds__(128)
join_kernel(const __grid_constant__ AttentionArgs a, int rows)
{
    __shared__ float4 acc[3][64];
    const auto &d = a.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y, D = (int)d.head_dim;
    griddep_wait();
    griddep_launch();
    const int4 cut = a.cut[blockIdx.x];
    if (!cut.w) return;
    const int head = cut.y / a.groups, group = cut.y - head * a.groups, per_kv = (int)(d.q_heads / d.kv_heads);
    if (row >= min(a.per_group, per_kv - group * a.per_group)) return;
    const int first = blockIdx.x, parts = cut.z - first + 1;
    auto slot = [&](int i) { return ((int64_t)2 * (first + i) + (i == 0 ? 1 : 0)) * rows + row; };
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, a.sums[slot(i)].x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int i = lane; i < parts; i += 32) {
        const float2 s = a.sums[slot(i)];
        l += s.x == -INFINITY ? s.y : s.y * exp2_approx(s.x - m);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float4 x[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
    for (int i = warp; i < parts; i += 4) {
        const float top = a.sums[slot(i)].x, f = top == -INFINITY ? 0.f : exp2_approx(top - m);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int el = (h * 32 + lane) * 4;
            if (el < D) {
                const float4 y = *reinterpret_cast<const float4 *>(a.part + slot(i) * D + el);
                x[h].x += f * y.x; x[h].y += f * y.y; x[h].z += f * y.z; x[h].w += f * y.w;
            }
        }
    }
    if (warp) { acc[warp - 1][lane] = x[0]; acc[warp - 1][32 + lane] = x[1]; }
    __syncthreads();
    if (warp) return;
    const float inverse = l == 0.f ? 0.f : 1.f / l;
    const int64_t h0 = head * per_kv + group * a.per_group + row;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int el = (h * 32 + lane) * 4;
        if (el >= D) continue;
#pragma unroll
        for (int w = 0; w < 3; w++) { const float4 y = acc[w][h * 32 + lane]; x[h].x += y.x; x[h].y += y.y; x[h].z += y.z; x[h].w += y.w; }
        store4<T>(d, cut.x, h0, el, x[h], inverse);
    }
    if (d.lse && lane == 0) d.lse[cut.x * d.q_heads + h0] = lse_of<T>(m, l);
}

// ---- host: which variant, how much workspace -----------------------------------------------------------------
struct AttnPlan { int dp, nt, per_group, groups, ctas, cluster; int64_t bytes; };
AttnPlan plan_attention(const ortho_b200_paged_attention_desc &d);             // attention.cu
template <class T> int launch_attention(const AttentionArgs &a, const AttnPlan &p, cudaStream_t stream);

template <class T, int DP, int NT>
int launch_attention_as(const AttentionArgs &a, const AttnPlan &p, cudaStream_t stream)
{
    using Shape = AttnShape<DP, NT>;
    const int dev = current_device_index();
    if (dev < 0) return ORTHO_B200_ERR_CUDA;
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes));
        if constexpr (Shape::kClusterPerSm > 0)
            OB_CUDA(cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kClusterBytes));
        attr_set[dev] = true;
    }
    if constexpr (Shape::kClusterPerSm > 0) {
        if (p.cluster) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)a.ctas); cfg.blockDim = dim3(kAttnThreads); cfg.dynamicSmemBytes = Shape::kClusterBytes; cfg.stream = stream;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = (unsigned)p.cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
            cfg.attrs = attr; cfg.numAttrs = 2;
            OB_CUDA(cudaLaunchKernelEx(&cfg, paged_attention_kernel<T, DP, NT, true>, a));
            count_launch();
            return ORTHO_B200_OK;
        }
    }
    const int st = launch_dependent(paged_attention_kernel<T, DP, NT, false>, dim3((unsigned)a.ctas), kAttnThreads, Shape::kBytes, stream, a);
    if (st) return st;
    return launch_dependent(join_kernel<T>, dim3((unsigned)a.ctas, (unsigned)a.per_group), 128, 0, stream, a, NT * 8);
}

template <class T, int DP>
int launch_attention_dim(const AttentionArgs &a, const AttnPlan &p, cudaStream_t stream)
{
    if (p.nt == 1) return launch_attention_as<T, DP, 1>(a, p, stream);
    if (p.nt == 2) return launch_attention_as<T, DP, 2>(a, p, stream);
    if constexpr (DP <= 128) return launch_attention_as<T, DP, 4>(a, p, stream);
    return ORTHO_B200_ERR_SHAPE;
}

#define OB_ATTENTION_DIMS(X) X(64) X(80) X(96) X(112) X(128) X(192) X(256)

template <class T>
int launch_attention(const AttentionArgs &a, const AttnPlan &p, cudaStream_t stream)
{
#define OB_CASE(DP) if (p.dp == DP) return launch_attention_dim<T, DP>(a, p, stream);
    OB_ATTENTION_DIMS(OB_CASE)
#undef OB_CASE
    return ORTHO_B200_ERR_SHAPE;
}

}  // namespace ob
