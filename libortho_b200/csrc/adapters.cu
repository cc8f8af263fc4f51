// Low-rank adapters of many requests beside a shared projection:
//
//     v[t] = down_e x[t],   out[t] = y[t] + scale_e up_e v[t],   e = ids[t]
//
// Few tokens: bound by the weights of the adapters in use (2 rank (K + N) bytes each).  Many tokens: by the activations (2 (K + 2 N) bytes a
// token).  The operations are a few per byte either way, so both products run on m16n8k16 tensor-core instructions.
//
// Tokens are grouped first, so that an adapter's weights are read once for all its tokens: `order` lists them by adapter, a tile is up to
// 16 or 64 of them with one adapter.
//
// Up to kFewTokens tokens every CTA groups them for itself, and where there is little to do few_kernel does it all.  Else a kernel computes v
// (down_few_kernel or down_many_kernel; more tokens are grouped by a kernel in front) and up_kernel the outputs: it starts beside the kernel for v
// and fetches its first weights and rows of y meanwhile.
//
// Measured (GPU time, us): 1 token, 4096 -> 12288, rank 16: 4.7; 64 tokens over twenty adapters of rank 8 to 64, 8192 -> 10240, 26 MB: 18.9 (38 MB are read: a
// column's row of `up` has the highest rank's 128 bytes, of which an adapter of rank 8 uses 16 and memory delivers more); 4096 tokens,
// six adapters of rank 32, 4096 -> 12288, 241 MB: 65, of which grouping 5, v 9, outputs 49 (4.1 TB/s: no pipe is full, the chain of barrier, operands,
// products and results of 16 warps an SM).
#include "launch.cuh"
#include "tma.cuh"

#include <type_traits>

namespace ob {

constexpr int kFewTokens = 128, kFewRank = 64, kMostAdapters = 8192, kGroupThreads = 1024;       // kFewRank: few_kernel's highest

struct LowRankArgs {
    ortho_b200_low_rank_desc d;
    int *heads;                                  // {tiles with an adapter, all tiles}; these three: more than kFewTokens tokens
    int *order;                                  // [tokens] grouped by adapter, those without one last
    int4 *tiles;                                 // {adapter or -1, first place in order, tokens, rank}
    float *v;                                    // [tokens][rank], by place in order
    int rank_groups;                             // groups of ranks that the kernel for v computes apart
    int blocks, padded, up_groups;               // of up_kernel's columns; rank in whole 16; groups of 64 ranks
    bool vectors, copies;                        // rows of y and out in 16-byte pieces; out is not y
};

__device__ __forceinline__ int rank_of(const ortho_b200_low_rank_desc &d, int e)
{
    if (!d.ranks) return (int)d.rank;
    const int64_t r = ((int64_t)max(__ldcg(d.ranks + e), 0) + 7) / 8 * 8;
    return (int)(r < d.rank ? r : d.rank);
}
// the adapter of a token and its rank; d.adapters for none
__device__ __forceinline__ int adapter_of(const ortho_b200_low_rank_desc &d, int64_t t, int &rank)
{
    const int32_t e = __ldcg(d.ids + t);
    rank = e >= 0 && e < d.adapters ? rank_of(d, e) : 0;
    return rank > 0 ? e : (int)d.adapters;
}

// ---- grouping ----------------------------------------------------------------------------------------------------
struct FewTokens { int adapter[kFewTokens], order[kFewTokens]; int4 at[kFewTokens], tiles[kFewTokens]; int count[kFewTokens / 32]; };

// by a CTA of kFewTokens threads; returns (tiles with an adapter, all tiles)
template <int TILE>
__device__ __forceinline__ int2 group_few(FewTokens &g, const ortho_b200_low_rank_desc &d)
{
    const int t = threadIdx.x, T = (int)d.tokens, lane = t & 31, warp = t >> 5;
    int rank = 0;
    const int e = t < T ? adapter_of(d, t, rank) : 0x7FFFFFFF;
    g.adapter[t] = e;
    g.at[t] = make_int4(-2, 0, 0, 0);
    __syncthreads();
    int less = 0, before = 0, same = 0;
    for (int i = 0; i < T; i += 4) {
        const int4 o = *reinterpret_cast<const int4 *>(g.adapter + i);
        less += (o.x < e) + (o.y < e) + (o.z < e) + (o.w < e);
        same += (o.x == e) + (o.y == e) + (o.z == e) + (o.w == e);
        before += (o.x == e && i < t) + (o.y == e && i + 1 < t) + (o.z == e && i + 2 < t) + (o.w == e && i + 3 < t);
    }
    const int place = less + before;
    if (t < T) {
        g.order[place] = t;
        if (before % TILE == 0) g.at[place] = make_int4(e < d.adapters ? e : -1, place, min(TILE, same - before), rank);
    }
    __syncthreads();
    const int4 mine = g.at[t];
    const uint32_t leads = __ballot_sync(0xffffffffu, mine.x != -2);
    if (lane == 0) g.count[warp] = __popc(leads);
    const int real = __syncthreads_count(mine.x >= 0), all = __syncthreads_count(mine.x != -2);
    int at = __popc(leads & ((1u << lane) - 1));
    for (int w = 0; w < warp; w++) at += g.count[w];
    if (mine.x != -2) g.tiles[at] = mine;
    __syncthreads();
    return make_int2(real, all);
}

// any number of tokens, one CTA: counts per adapter, running sums, places.  Equal adapters within a warp are counted by one atomic.  The
// order of an adapter's tokens differs from run to run; no result depends on it.
template <int TILE>
__global__ void __launch_bounds__(kGroupThreads)
group_kernel(const __grid_constant__ LowRankArgs a)
{
    constexpr int AHEAD = 4;                     // tokens of a thread that are loaded together
    extern __shared__ int counts[];              // [adapters + 1]
    __shared__ int2 warp_sum[kGroupThreads / 32];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = (int)d.adapters + 1, T = (int)d.tokens;
    int *const first_tile = counts + E, *const start = first_tile + E;
    griddep_wait();
    griddep_launch();
    for (int e = tid; e < E; e += kGroupThreads) counts[e] = 0;
    __syncthreads();
    // AHEAD tokens of each thread: their adapters and ranks, and from the counters their numbers among their adapters' tokens
    int e[AHEAD], rank[AHEAD], among[AHEAD];
    auto number = [&](int t0) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int t = t0 + i * kGroupThreads + tid;
            rank[i] = 0;
            e[i] = t < T ? adapter_of(d, t, rank[i]) : -1;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (t0 + i * kGroupThreads >= T) break;
            const uint32_t peers = __match_any_sync(0xffffffffu, e[i]);
            const int leader = __ffs(peers) - 1;
            int base = 0;
            if (e[i] >= 0 && leader == lane) base = atomicAdd(counts + e[i], __popc(peers));
            among[i] = __shfl_sync(0xffffffffu, base, leader) + __popc(peers & ((1u << lane) - 1));
        }
    };
    for (int t0 = 0; t0 < T; t0 += AHEAD * kGroupThreads) number(t0);
    __syncthreads();
    int2 before = make_int2(0, 0);               // tokens and tiles of the adapters before
    for (int e0 = 0; e0 < E; e0 += kGroupThreads) {
        const int e = e0 + tid, n = e < E ? counts[e] : 0, tiles = (n + TILE - 1) / TILE;
        int2 sum = make_int2(n, tiles);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
            if (lane >= o) { sum.x += x; sum.y += y; }
        }
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        // every warp adds up the warps' sums for itself
        int2 w = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, w.x, o), y = __shfl_up_sync(0xffffffffu, w.y, o);
            if (lane >= o) { w.x += x; w.y += y; }
        }
        const int px = __shfl_sync(0xffffffffu, w.x, warp ? warp - 1 : 0), py = __shfl_sync(0xffffffffu, w.y, warp ? warp - 1 : 0);
        sum.x += before.x + (warp ? px : 0);
        sum.y += before.y + (warp ? py : 0);
        if (e < E) { start[e] = sum.x - n; first_tile[e] = sum.y - tiles; counts[e] = 0; }
        if (e == E - 1) { a.heads[0] = sum.y - tiles; a.heads[1] = sum.y; }
        before.x += __shfl_sync(0xffffffffu, w.x, 31);
        before.y += __shfl_sync(0xffffffffu, w.y, 31);
        __syncthreads();
    }
    for (int t0 = 0; t0 < T; t0 += AHEAD * kGroupThreads) {
        if (T > AHEAD * kGroupThreads) number(t0);                             // (else they are at hand)
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (e[i] < 0) continue;
            const int at = start[e[i]] + among[i];
            a.order[at] = t0 + i * kGroupThreads + tid;
            if (among[i] % TILE == 0) {
                const int end = e[i] + 1 < E ? start[e[i] + 1] : T;
                a.tiles[first_tile[e[i]] + among[i] / TILE] = make_int4(e[i] + 1 < E ? e[i] : -1, at, min(TILE, end - at), rank[i]);
            }
        }
    }
}

// ---- v = down x ------------------------------------------------------------------------------------------------------
constexpr int kFewTile = 16, kFewCtas = 8, kManyTile = 64, kManyCtas = 8, kDownStages = 4;

// Few tokens: MB blocks of 16 ranks (the 16-row operand) by 16 tokens, by a cluster of eight CTAs whose 32 warps have the K of usual layers in flight
// almost at once.
template <class T, int MB>
__global__ void __launch_bounds__(128, 2)
down_few_kernel(const __grid_constant__ LowRankArgs a)
{
    // a step is 32 k; CHUNKS steps of a warp are loaded together, 64 to 128 registers
    constexpr int NT = kFewTile / 8, CTAS = kFewCtas, WARPS = 4, TOKENS = NT * 8, RANKS = MB * 16, PITCH = RANKS + 4, CHUNKS = 4;
    constexpr int QUADS = TOKENS * RANKS / 4, SHARE = QUADS / CTAS, WARP_QUADS = TOKENS * PITCH / 4;
    static_assert(QUADS % CTAS == 0, "every CTA adds up the same share");
    __shared__ __align__(16) float sums[WARPS][TOKENS][PITCH];
    // this CTA's share of the results, from every CTA of the cluster, of two units
    __shared__ __align__(16) float4 arrived[2][CTAS][SHARE];
    __shared__ FewTokens few;
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = (int)cluster_ctarank();
    cluster_arrive();                            // (waited for before the first store into another CTA: it has started then)
    griddep_wait();
    griddep_launch();
    const int real = group_few<TOKENS>(few, d).x;
    const int *const order = few.order;
    const int4 *const tiles = few.tiles;
    const int K = (int)d.K, steps = (K + 31) / 32, clusters = gridDim.x / CTAS;
    const int quad = lane & 3, row = lane >> 2;
    int turn = 0;
    cluster_wait();
    for (int64_t unit = blockIdx.x / CTAS; unit < (int64_t)real * a.rank_groups; unit += clusters) {
        const int4 tile = tiles[unit / a.rank_groups];
        const int r0 = (int)(unit % a.rank_groups) * RANKS, rank = tile.w;
        if (r0 >= rank) continue;                // (the whole cluster)
        const T *x[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) x[j] = (const T *)d.x + (int64_t)order[tile.y + min(j * 8 + row, tile.z - 1)] * d.x_stride;
        const T *const w = (const T *)d.down + ((int64_t)tile.x * d.rank + r0 + row) * d.K;
        float acc[MB][NT][4];
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
        // 8 of a step's k (16 bytes of every row) a lane; steps are dealt to the cluster's warps in turn
        constexpr int STRIDE = CTAS * WARPS;
        for (int s0 = cta * WARPS + warp; s0 < steps; s0 += CHUNKS * STRIDE) {
            uint4 wv[CHUNKS][MB][2], xv[CHUNKS][NT];
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const int k = (s0 + c * STRIDE) * 32 + quad * 8;
                const bool on = k < K;
#pragma unroll
                for (int m = 0; m < MB; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        wv[c][m][h] = on && r0 + m * 16 + h * 8 + row < rank ? ldg_stream(w + (int64_t)(m * 16 + h * 8) * d.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NT; j++)
                    xv[c][j] = on && j * 8 < tile.z ? load16(x[j] + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        const uint4 w0 = wv[c][m][0], w1 = wv[c][m][1];
                        const uint32_t part[4] = {h ? w0.z : w0.x, h ? w1.z : w1.x, h ? w0.w : w0.y, h ? w1.w : w1.y};
#pragma unroll
                        for (int j = 0; j < NT; j++)
                            if (j * 8 < tile.z) Half<T>::mma(acc[m][j], part, h ? xv[c][j].z : xv[c][j].x, h ? xv[c][j].w : xv[c][j].y);
                    }
        }
        // The warps' sums are added in order and sent to the CTA that adds up the cluster's.  One barrier a unit: the results of the next one
        // arrive in the other half of `arrived`, and those of the one behind it only after a barrier that this CTA reaches when it has read these.
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) sums[warp][j * 8 + quad * 2 + (e & 1)][m * 16 + row + (e >> 1) * 8] = acc[m][j][e];
        __syncthreads();
        const float4 *const mine = reinterpret_cast<const float4 *>(&sums[0][0][0]);
        const uint32_t to = shared_addr(&arrived[turn][cta][0]);
        for (int i = tid; i < QUADS; i += (32 * WARPS)) {
            const int at = i / (RANKS / 4) * (PITCH / 4) + i % (RANKS / 4);
            float4 s = mine[at];
#pragma unroll
            for (int o = 1; o < WARPS; o++) {
                const float4 y = mine[o * WARP_QUADS + at];
                s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
            }
            st_dsmem_v4(mapa_shared(to + 16 * (i % SHARE), i / SHARE), s);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        for (int i = tid; i < SHARE; i += (32 * WARPS)) {
            const int token = (cta * SHARE + i) / (RANKS / 4), r = r0 + (cta * SHARE + i) % (RANKS / 4) * 4;
            if (token >= tile.z || r >= rank) continue;
            float4 s = arrived[turn][0][i];
#pragma unroll
            for (int o = 1; o < CTAS; o++) {
                const float4 y = arrived[turn][o][i];
                s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
            }
            *reinterpret_cast<float4 *>(a.v + (int64_t)(tile.y + token) * d.rank + r) = s;
        }
        turn ^= 1;
    }
}

// Many tokens: MB blocks of 16 ranks by 64 tokens, by a cluster of eight CTAs.  A CTA's share of K comes through a ring of four stages of 64 k; a warp
// has 16 tokens and all ranks.  Bound by reading x.
template <class T, int MB>
__global__ void __launch_bounds__(128, 4)
down_many_kernel(const __grid_constant__ LowRankArgs a)
{
    constexpr int S = kDownStages, RANKS = MB * 16, CTAS = kManyCtas, X_BYTES = kManyTile * 128, STAGE = X_BYTES + RANKS * 128, W_PIECES = RANKS * 8 / 128;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(16) float arrived[CTAS][kManyTile / CTAS][RANKS];     // sums of this CTA's share of the tokens, from every CTA of the cluster
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, row = lane >> 2, cta = (int)cluster_ctarank();
    cluster_arrive();                            // (waited for before the first store into another CTA: it has started then)
    griddep_wait();
    griddep_launch();
    const int real = a.heads[0], K = (int)d.K, blocks = (K + 63) / 64, first = blocks * cta / CTAS, count = blocks * (cta + 1) / CTAS - first;
    // rows of 128 bytes in 16-byte chunks, exchanged by the row's number against bank conflicts; a thread copies the same chunk of every 16th row
    auto at = [](int r, int chunk) { return (uint32_t)(r * 128 + ((chunk ^ (r & 7)) << 4)); };
    const int chunk = tid & 7;
    cluster_wait();
    for (int64_t unit = blockIdx.x / CTAS; unit < (int64_t)real * a.rank_groups; unit += gridDim.x / CTAS) {
        const int4 tile = a.tiles[unit / a.rank_groups];
        const int r0 = (int)(unit % a.rank_groups) * RANKS, rank = tile.w;
        if (r0 >= rank) continue;                // (the whole cluster)
        const T *x[kManyTile / 16], *w[W_PIECES];
#pragma unroll
        for (int u = 0; u < kManyTile / 16; u++) {
            const int t = u * 16 + (tid >> 3);
            x[u] = t < tile.z ? (const T *)d.x + (int64_t)a.order[tile.y + t] * d.x_stride + first * 64 + chunk * 8 : nullptr;
        }
#pragma unroll
        for (int u = 0; u < W_PIECES; u++) {
            const int r = u * 16 + (tid >> 3);
            w[u] = r0 + r < rank ? (const T *)d.down + ((int64_t)tile.x * d.rank + r0 + r) * d.K + first * 64 + chunk * 8 : nullptr;
        }
        int issued = 0;
        auto issue = [&](int stage) {
            if (issued < count) {
                const uint32_t to = shared_addr(smem + stage * STAGE);
                const bool in = (first + issued) * 64 + chunk * 8 < K;
#pragma unroll
                for (int u = 0; u < kManyTile / 16; u++) {
                    const bool on = in && x[u];
                    copy16_async(to + at(u * 16 + (tid >> 3), chunk), on ? x[u] + issued * 64 : d.x, on);
                }
#pragma unroll
                for (int u = 0; u < W_PIECES; u++) {
                    const bool on = in && w[u];
                    copy16_async(to + X_BYTES + at(u * 16 + (tid >> 3), chunk), on ? w[u] + issued * 64 : d.down, on);
                }
                issued++;
            }
            copy_commit();
        };
#pragma unroll
        for (int s = 0; s < S - 1; s++) issue(s);
        float acc[MB][2][4];
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
        for (int b = 0, stage = 0; b < count; b++) {
            copy_wait<S - 2>();
            __syncthreads();                     // the stage is there, and everybody is done with the one before it
            issue(stage == 0 ? S - 1 : stage - 1);
            const uint32_t xs = shared_addr(smem + stage * STAGE), ws = xs + X_BYTES;
            if (warp * 16 < tile.z) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t v[4], r[MB][4];
                    ldmatrix4(v, xs + at(warp * 16 + (lane & 7) + (lane >> 4) * 8, k * 2 + ((lane >> 3) & 1)));
#pragma unroll
                    for (int m = 0; m < MB; m++) ldmatrix4(r[m], ws + at(m * 16 + (lane & 15), k * 2 + (lane >> 4)));
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        Half<T>::mma(acc[m][0], r[m], v[0], v[1]);
                        Half<T>::mma(acc[m][1], r[m], v[2], v[3]);
                    }
                }
            }
            if (++stage == S) stage = 0;
        }
        copy_wait<0>();
        // every CTA sends its sums of eight tokens to the CTA that adds them up
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t to = mapa_shared(shared_addr(&arrived[cta][0][0]), warp * 2 + j);
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) st_dsmem(to + ((quad * 2 + (e & 1)) * RANKS + m * 16 + row + (e >> 1) * 8) * 4, acc[m][j][e]);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        for (int i = tid; i < kManyTile / CTAS * RANKS / 4; i += 128) {
            const int t = i / (RANKS / 4), r = i % (RANKS / 4) * 4, token = cta * (kManyTile / CTAS) + t;
            if (token >= tile.z || r0 + r >= rank) continue;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int o = 0; o < CTAS; o++) {
                const float4 y = *reinterpret_cast<const float4 *>(&arrived[o][t][r]);
                s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
            }
            *reinterpret_cast<float4 *>(a.v + (int64_t)(tile.y + token) * d.rank + r0 + r) = s;
        }
        if (unit + gridDim.x / CTAS < (int64_t)real * a.rank_groups) {         // the next unit's sums may arrive, and its copies, when these are read
            __syncwarp();
            cluster_arrive();
            cluster_wait();
        }
    }
}

// ---- out = y + scale up v -------------------------------------------------------------------------------------------
// The products run over v in two 16-bit parts, which hold a value to 2^-16 of it in BF16 and 2^-22 in FP16 (one part alone would add an error as large as
// the output's own rounding, up to 2^-8 and 2^-11).  In FP16 it is brought to the token's largest |v| in [2^13, 2^14) by a power of two first (else it
// could leave FP16's range, or lose its small values; what is left of these is off by 2^-38 of the largest): `down`, and `back` for the result.
struct PowerOfTwo { float down, back; };
template <class T>
__device__ __forceinline__ PowerOfTwo bring_near(float top)
{
    const uint32_t exponent = min(__float_as_uint(top) >> 23, 254u);           // top in [2^(exponent - 127), 2^(exponent - 126)), or infinite
    if (!std::is_same<T, __half>::value || exponent < 14) return {1.f, 1.f};   // (tiny as it is)
    return {__uint_as_float((267 - exponent) << 23), __uint_as_float((exponent - 13) << 23)};
}
template <class T>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t &hi, uint32_t &lo)
{
    hi = Half<T>::pack(a, b);
    const float2 f = Half<T>::unpack(hi);
    lo = Half<T>::pack(isinf(f.x) ? 0.f : a - f.x, isinf(f.y) ? 0.f : b - f.y);                    // (what is infinite stays so: no infinity minus another)
}
__device__ __forceinline__ float largest(float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }

constexpr int kUpThreads = 128, kUpStages = 3;                                // (stages: 2 pairs are under way while one is worked on)
static_assert(kFewTokens == kUpThreads && kGroupThreads == 32 * 32, "a thread per token, a lane per warp");

// Columns of a unit of work and the layout of a stage: rows of G ranks, 16 bytes of padding against bank conflicts, then every thread's own pieces of y.
// Column c of 8 in product tile j stands for output column 8 (c / 2) + 2 j + c % 2 of 32, so that a lane's results over four tiles are
// eight neighbours.
template <int MT, int G>
struct UpShape {
    static constexpr int kTokens = MT * 16, kColumns = MT == 1 ? 128 : 64, kPieces = G / 8, kPitch = G * 2 + 16, kWeights = kColumns * kPitch + 64;
    static constexpr int kTaken = MT == 1 ? 2 : 4;                             // 16-byte pieces of y that a thread needs for its results
    static constexpr int kStage = kWeights + kTaken * kUpThreads * 16;
    static __device__ __forceinline__ int at(int n) { return (n & ~31) + (n >> 1 & 3) * 8 + (n >> 3 & 3) * 2 + (n & 1); }      // row of a column in a stage
};

// A lane's place in its two tokens' rows of y and out
template <class T> struct Rows { const T *y[2]; T *out[2]; bool has[2]; };

// v as two 16-bit parts into shared memory, rows `pitch` bytes apart, and the factor of each token's result.  `from(t, r)`: four ranks of token t.
template <class T, int TOKENS, class F>
__device__ __forceinline__ void place_v(unsigned char *upper, unsigned char *lower, float *factor, int pitch, int padded, float scale, F &&from)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // lanes of a token: the power of two that holds a quarter of the rank, at most a warp (twice: above 128)
    const int width = padded <= 16 ? 4 : padded <= 32 ? 8 : padded <= 64 ? 16 : 32, rows = 32 / width, sub = lane & (width - 1);
#pragma unroll 4
    for (int i = 0; i < TOKENS / 4; i += rows) {
        const int t = warp * (TOKENS / 4) + i + lane / width;
        if (TOKENS / 4 < rows && t >= (warp + 1) * (TOKENS / 4)) break;        // (a warp has four tokens, lanes for eight)
        float4 x[2];
        float top = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            x[h] = from(t, (h * 32 + sub) * 4);
            top = fmaxf(top, largest(x[h]));
        }
        const uint32_t here = TOKENS / 4 < rows ? (1u << (TOKENS / 4 * width)) - 1 : 0xFFFFFFFFu;
        for (int o = width >> 1; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(here, top, o));
        const PowerOfTwo by = bring_near<T>(top);
        if (sub == 0) factor[t] = by.back * scale;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = (h * 32 + sub) * 4;
            if (r >= padded) continue;
            uint32_t hi[2], lo[2];
            two_parts<T>(x[h].x * by.down, x[h].y * by.down, hi[0], lo[0]);
            two_parts<T>(x[h].z * by.down, x[h].w * by.down, hi[1], lo[1]);
            *reinterpret_cast<uint2 *>(upper + t * pitch + r * 2) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2 *>(lower + t * pitch + r * 2) = make_uint2(lo[0], lo[1]);
        }
    }
}

// acc += v up over `steps` times 16 ranks of a stage, for 16 tokens and 4 J columns' tiles of 8.  v_at: this lane's row of v in the upper part, `apart` to the lower.
template <class T, int G, int J>
__device__ __forceinline__ void multiply_up(float (&acc)[J][4], uint32_t v_at, uint32_t apart, uint32_t weights, int steps)
{
    constexpr int PITCH = G * 2 + 16;
#pragma unroll
    for (int k = 0; k < G / 16; k += 2) {
        if (k >= steps) break;
        const bool both = G > 16 && k + 1 < steps;
        uint32_t hi[2][4], lo[2][4];
        ldmatrix4(hi[0], v_at + k * 32);
        ldmatrix4(lo[0], v_at + apart + k * 32);
        if (both) {
            ldmatrix4(hi[1], v_at + k * 32 + 32);
            ldmatrix4(lo[1], v_at + apart + k * 32 + 32);
        }
#pragma unroll
        for (int j0 = 0; j0 < J; j0 += 4) {
            uint32_t w[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) ldmatrix4(w[j], weights + (j0 + j) * 8 * PITCH + k * 32);          // (an odd number of steps: half of it)
#pragma unroll
            for (int j = 0; j < 4; j++) Half<T>::mma(acc[j0 + j], hi[0], w[j][0], w[j][1]);
#pragma unroll
            for (int j = 0; j < 4; j++) Half<T>::mma(acc[j0 + j], lo[0], w[j][0], w[j][1]);
            if (both) {
#pragma unroll
                for (int j = 0; j < 4; j++) Half<T>::mma(acc[j0 + j], hi[1], w[j][2], w[j][3]);
#pragma unroll
                for (int j = 0; j < 4; j++) Half<T>::mma(acc[j0 + j], lo[1], w[j][2], w[j][3]);
            }
        }
    }
}

// out = y + factor acc of a lane's two tokens.  whole: y has come to `staged` (pieces of a thread 16 kUpThreads bytes apart); else rows that are not aligned, or
// the last columns (`rest` of them from this lane's first one on), one by one.
template <class T, int Q>
__device__ __forceinline__ void write_out(const Rows<T> &now, const float (&acc)[Q * 4][4], const float *factor, int t, bool adds, bool whole, const unsigned char *staged, int rest)
{
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (!now.has[h]) continue;
        const float f = adds ? factor[t + h * 8] : 0.f;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            if (whole) {
                const uint4 y = *reinterpret_cast<const uint4 *>(staged + (h * Q + q) * (kUpThreads * 16));
                uint32_t p[4] = {y.x, y.y, y.z, y.w};
                if (adds) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 was = Half<T>::unpack(p[j]);
                        p[j] = Half<T>::pack(was.x + f * acc[q * 4 + j][2 * h], was.y + f * acc[q * 4 + j][2 * h + 1]);
                    }
                }
                *reinterpret_cast<uint4 *>(now.out[h] + q * 32) = make_uint4(p[0], p[1], p[2], p[3]);
            } else {
                T was[8];
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < rest - q * 32) was[i] = now.y[h][q * 32 + i];
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < rest - q * 32) now.out[h][q * 32 + i] = adds ? Half<T>::from_float(Half<T>::to_float(was[i]) + f * acc[q * 4 + (i >> 1)][2 * h + (i & 1)]) : was[i];
            }
        }
    }
}

// The (tile, columns) pairs are numbered in a row and dealt evenly, a run of them to each CTA, so that v comes into shared memory about once per CTA.
// Rows of `up` (up to 64 ranks) and y arrive in a ring of three stages, the first ones while the kernel for v still runs.  Tiles of 16 tokens (MT = 1):
// a warp has 32 of 128 columns, bound by the weights.  Of 64 (MT = 4): a warp has 16 tokens and 64 columns, bound by y and out.
template <class T, int MT, int G, bool FEW>
__global__ void __launch_bounds__(kUpThreads, 4)
up_kernel(const __grid_constant__ LowRankArgs a)
{
    using Shape = UpShape<MT, G>;
    constexpr int TOKENS = Shape::kTokens, COLUMNS = Shape::kColumns, Q = MT == 1 ? 1 : COLUMNS / 32, S = kUpStages, PIECES = Shape::kPieces, PITCH = Shape::kPitch;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float factor[TOKENS];
    __shared__ __align__(16) unsigned char few_smem[FEW ? sizeof(FewTokens) : 16];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, row = lane >> 2;
    const int padded = a.padded, groups = G < 64 ? 1 : a.up_groups, v_pitch = padded * 2 + 16, N = (int)d.N;
    const int t0 = MT == 1 ? 0 : warp * 16, c0 = MT == 1 ? warp * 32 : 0;      // this warp's first token of the tile and column of the pair
    unsigned char *const upper = smem + S * Shape::kStage, *const lower = upper + TOKENS * v_pitch;
    // What is read in front of the wait was complete before the kernel for v let this kernel start: it does so behind its own wait.  (From L2: this SM's L1 may
    // hold older values.)
    griddep_launch();
    FewTokens &few = *reinterpret_cast<FewTokens *>(few_smem);
    int all;
    if constexpr (FEW) {
        const int2 n = group_few<TOKENS>(few, d);
        all = a.copies ? n.y : n.x;
    } else {
        all = __ldcg(a.heads + (a.copies ? 1 : 0));
    }
    auto tile_at = [&](int i) { if constexpr (FEW) return few.tiles[i]; else return __ldcg(a.tiles + i); };
    const int64_t pairs = (int64_t)all * a.blocks, first = pairs * blockIdx.x / gridDim.x, end = pairs * (blockIdx.x + 1) / gridDim.x;
    int left = (int)(end - first), to_issue = left;
    auto rows_of = [&](const int4 &tile, int block) {
        Rows<T> r;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int t = t0 + h * 8 + row;
            r.has[h] = t < tile.z;
            const int64_t token = !r.has[h] ? 0 : FEW ? few.order[tile.y + t] : __ldcg(a.order + tile.y + t);
            r.y[h] = (const T *)d.y + token * d.y_stride + block * COLUMNS + c0 + quad * 8;
            r.out[h] = (T *)d.out + token * d.out_stride + block * COLUMNS + c0 + quad * 8;
        }
        return r;
    };
    // the copies of a step (pair, up to 64 ranks); each thread has some of the 16-byte pieces of `up` and its own of y, which come with the last ranks
    int next_group = 0, next_tile = left ? (int)(first / a.blocks) : 0, next_block = left ? (int)(first - (int64_t)next_tile * a.blocks) : 0;
    int4 ahead = make_int4(-1, 0, 0, 0);
    Rows<T> coming;
    if (left) {
        ahead = tile_at(next_tile);
        coming = rows_of(ahead, next_block);
    }
    const uint32_t mine = Shape::kWeights + tid * 16;
    auto issue = [&](int stage) {
        if (to_issue > 0) {
            const int r0 = next_group * G;
            if (next_group == groups - 1 && a.vectors && (next_block + 1) * COLUMNS <= N) {
                const uint32_t to = shared_addr(smem + stage * Shape::kStage) + mine;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int q = 0; q < Q; q++)
                        if (coming.has[h]) copy16_async(to + (h * Q + q) * (kUpThreads * 16), coming.y[h] + q * 32, true);
            }
            if (ahead.x >= 0 && r0 < ahead.w) {
                const uint32_t to = shared_addr(smem + stage * Shape::kStage);
                const T *const from = (const T *)d.up + ((int64_t)ahead.x * N + next_block * COLUMNS) * d.rank + r0;
                const int columns = N - next_block * COLUMNS, ranks = ahead.w - r0;
#pragma unroll
                for (int u = 0; u < COLUMNS * PIECES / kUpThreads; u++) {
                    const int i = u * kUpThreads + tid, n = i / PIECES, piece = i % PIECES;
                    const bool on = n < columns && piece * 8 < ranks;
                    copy16_async(to + Shape::at(n) * PITCH + piece * 16, on ? from + n * (int)d.rank + piece * 8 : from, on);
                }
            }
            if (++next_group == groups) {
                next_group = 0;
                to_issue--;
#pragma unroll
                for (int h = 0; h < 2; h++) coming.y[h] += COLUMNS;
                if (++next_block == a.blocks && to_issue > 0) {
                    next_block = 0;
                    ahead = tile_at(++next_tile);
                    coming = rows_of(ahead, 0);
                }
            }
        }
        copy_commit();
    };
#pragma unroll
    for (int s = 0; s < S - 1; s++) issue(s);
    griddep_wait();
    if (left == 0) return;

    int tile_number = (int)(first / a.blocks), block = (int)(first - (int64_t)tile_number * a.blocks), stage = 0;
    bool new_tile = true;
    int4 tile;
    Rows<T> now;
    for (int last = 0;;) {
        float acc[Q * 4][4];
#pragma unroll
        for (int j = 0; j < Q * 4; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        for (int group = 0; group < groups; group++) {
            copy_wait<S - 2>();
            __syncthreads();                     // the stage is there, and everybody is done with the one before it and with v
            issue(stage == 0 ? S - 1 : stage - 1);
            if (new_tile) {
                new_tile = false;
                tile = tile_at(tile_number);
                now = rows_of(tile, block);
                if (tile.x >= 0)
                    place_v<T, TOKENS>(upper, lower, factor, v_pitch, padded, d.scales ? __ldcg(d.scales + tile.x) : 1.f, [&](int t, int r) {
                        return t < tile.z && r < tile.w ? __ldcg(reinterpret_cast<const float4 *>(a.v + (int64_t)(tile.y + t) * d.rank + r)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    });
                __syncthreads();
            }
            const int ranks = tile.x < 0 ? 0 : min(tile.w - group * G, G), steps = (ranks + 15) / 16;             // of 16 ranks
            if (steps > 0 && t0 < tile.z)
                multiply_up<T, G, Q * 4>(acc, shared_addr(upper) + (uint32_t)((t0 + (lane & 15)) * v_pitch + group * (G * 2) + (lane >> 4) * 16), (uint32_t)(TOKENS * v_pitch),
                                         shared_addr(smem + stage * Shape::kStage) + (uint32_t)((c0 + (lane & 7)) * PITCH + (lane >> 3) * 16), steps);
            last = stage;
            if (++stage == S) stage = 0;
        }
        write_out<T, Q>(now, acc, factor, t0 + row, tile.x >= 0, a.vectors && (block + 1) * COLUMNS <= N, smem + last * Shape::kStage + mine, N - (block * COLUMNS + c0 + quad * 8));
        if (--left == 0) break;
        if (++block == a.blocks) {
            block = 0;
            tile_number++;
            new_tile = true;
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) { now.y[h] += COLUMNS; now.out[h] += COLUMNS; }
        }
    }
}

// ---- few tokens and columns: both products in one kernel ------------------------------------------------------------------------------
// A cluster of eight CTAs has a tile of up to 16 tokens and a share of the columns.  It computes v of the tile (again in every cluster that has some of its
// columns: the weights come from L2 then), K split over its 32 warps; every CTA sends its sums to all the others and adds up what
// arrives, in order.  Then every CTA has some blocks of 128 columns, a warp 32 of them.  The first rows of `up` and of y are under way from the
// start.  Bound by the weights, and at a token or two by the chain of loads: ids, weights and x, exchange, results.
template <int MB>
struct FewShape {
    static constexpr int kRanks = MB * 16, kCtas = 8, kPitch = kRanks + 4;
    using Up = UpShape<1, kRanks>;
    static constexpr int kSums = 4 * 16 * kPitch * 4, kArrived = 2 * kCtas * 16 * kRanks * 4;
    static int bytes(int padded) { return kUpStages * Up::kStage + kSums + kArrived + 2 * 16 * (padded * 2 + 16) + 16 * padded * 4; }
};

template <class T, int MB>
__global__ void __launch_bounds__(kUpThreads, 2)
few_kernel(const __grid_constant__ LowRankArgs a)
{
    using Shape = FewShape<MB>;
    using Up = typename Shape::Up;
    constexpr int S = kUpStages, CTAS = Shape::kCtas, RANKS = Shape::kRanks, PITCH = Shape::kPitch, CHUNKS = 4, STRIDE = CTAS * 4, COLUMNS = Up::kColumns, PIECES = Up::kPieces;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ FewTokens few;
    __shared__ float factor[16];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, row = lane >> 2, cta = (int)cluster_ctarank();
    const int padded = a.padded, v_pitch = padded * 2 + 16, K = (int)d.K, N = (int)d.N, steps_k = (K + 31) / 32;
    float *const sums = reinterpret_cast<float *>(smem + S * Up::kStage);      // [4 warps][16 tokens][PITCH]
    float4 *const arrived = reinterpret_cast<float4 *>(reinterpret_cast<unsigned char *>(sums) + Shape::kSums);           // [2][CTAS][16 tokens][RANKS]
    float *const v = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(arrived) + Shape::kArrived);             // [16][padded]
    unsigned char *const upper = reinterpret_cast<unsigned char *>(v + 16 * padded), *const lower = upper + 16 * v_pitch;
    cluster_arrive();                            // (waited for before the first store into another CTA: it has started then)
    griddep_wait();
    griddep_launch();
    const int2 count = group_few<16>(few, d);
    const int all = a.copies ? count.y : count.x, clusters = gridDim.x / CTAS;
    // clusters of a tile
    const int shares = all > 0 ? max(1, min(clusters / all, (a.blocks + CTAS - 1) / CTAS)) : 1;
    int turn = 0;
    cluster_wait();
    for (int unit = blockIdx.x / CTAS; unit < all * shares; unit += clusters) {
        const int4 tile = few.tiles[unit / shares];
        const int part = unit % shares * CTAS + cta, parts = shares * CTAS;
        int block = (int)((int64_t)a.blocks * part / parts);
        const int end = (int)((int64_t)a.blocks * (part + 1) / parts), rank = tile.x < 0 ? 0 : tile.w, groups = rank ? (rank + RANKS - 1) / RANKS : 1;
        const float scale = rank && d.scales ? __ldcg(d.scales + tile.x) : 1.f;
        Rows<T> now;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int t = h * 8 + row;
            now.has[h] = t < tile.z;
            const int64_t token = now.has[h] ? few.order[tile.y + t] : 0;
            now.y[h] = (const T *)d.y + token * d.y_stride + block * COLUMNS + warp * 32 + quad * 8;
            now.out[h] = (T *)d.out + token * d.out_stride + block * COLUMNS + warp * 32 + quad * 8;
        }
        // the copies of a step: up to RANKS ranks of a block of columns, y with the last of them
        int next_block = block, next_group = 0;
        const uint32_t mine = Up::kWeights + tid * 16;
        auto issue = [&](int stage) {
            if (next_block < end) {
                const uint32_t to = shared_addr(smem + stage * Up::kStage);
                if (next_group == groups - 1 && a.vectors && (next_block + 1) * COLUMNS <= N) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (now.has[h]) copy16_async(to + mine + h * (kUpThreads * 16), now.y[h] + (next_block - block) * COLUMNS, true);
                }
                if (rank) {
                    const int r0 = next_group * RANKS, columns = N - next_block * COLUMNS, ranks = rank - r0;
                    const T *const from = (const T *)d.up + ((int64_t)tile.x * N + next_block * COLUMNS) * d.rank + r0;
#pragma unroll
                    for (int u = 0; u < COLUMNS * PIECES / kUpThreads; u++) {
                        const int i = u * kUpThreads + tid, n = i / PIECES, piece = i % PIECES;
                        const bool on = n < columns && piece * 8 < ranks;
                        copy16_async(to + Up::at(n) * Up::kPitch + piece * 16, on ? from + n * (int)d.rank + piece * 8 : from, on);
                    }
                }
                if (++next_group == groups) {
                    next_group = 0;
                    next_block++;
                }
            }
            copy_commit();
        };
        __syncthreads();                         // the unit before is done with the stages and with v
#pragma unroll
        for (int s = 0; s < S - 1; s++) issue(s);

        // ---- v = down x: 32 k a step, 8 of them (16 bytes of every row) a lane, steps dealt to the cluster's warps in turn
        const T *x[2];
#pragma unroll
        for (int j = 0; j < 2; j++) x[j] = (const T *)d.x + (int64_t)few.order[tile.y + min(j * 8 + row, tile.z - 1)] * d.x_stride;
        for (int r0 = 0; r0 < rank; r0 += RANKS) {
            const T *const w = (const T *)d.down + ((int64_t)tile.x * d.rank + r0 + row) * d.K;
            float acc[MB][2][4];
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
            for (int s0 = cta * 4 + warp; s0 < steps_k; s0 += CHUNKS * STRIDE) {
                uint4 wv[CHUNKS][MB][2], xv[CHUNKS][2];
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    const int k = (s0 + c * STRIDE) * 32 + quad * 8;
                    const bool on = k < K;
#pragma unroll
                    for (int m = 0; m < MB; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            wv[c][m][h] = on && r0 + m * 16 + h * 8 + row < rank ? load16(w + (int64_t)(m * 16 + h * 8) * d.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 2; j++) xv[c][j] = on && j * 8 < tile.z ? load16(x[j] + k) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int m = 0; m < MB; m++) {
                            const uint4 w0 = wv[c][m][0], w1 = wv[c][m][1];
                            const uint32_t half[4] = {h ? w0.z : w0.x, h ? w1.z : w1.x, h ? w0.w : w0.y, h ? w1.w : w1.y};
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                if (j * 8 < tile.z) Half<T>::mma(acc[m][j], half, h ? xv[c][j].z : xv[c][j].x, h ? xv[c][j].w : xv[c][j].y);
                        }
            }
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sums[(warp * 16 + j * 8 + quad * 2 + (e & 1)) * PITCH + m * 16 + row + (e >> 1) * 8] = acc[m][j][e];
            __syncthreads();
            // The CTA's sums go to every CTA of the cluster.  One barrier: the next ones arrive in the other half of `arrived`, and those behind them only
            // after a barrier that this CTA reaches when it has read these.
            constexpr int QUADS = 16 * RANKS / 4;
            const uint32_t to = shared_addr(arrived + (turn * CTAS + cta) * QUADS);
            for (int i = tid; i < QUADS; i += kUpThreads) {
                const int t = i / (RANKS / 4), q = i % (RANKS / 4) * 4;
                if (t >= tile.z) break;
                float4 s = *reinterpret_cast<const float4 *>(sums + t * PITCH + q);
#pragma unroll
                for (int o = 1; o < 4; o++) {
                    const float4 y = *reinterpret_cast<const float4 *>(sums + (o * 16 + t) * PITCH + q);
                    s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
                }
#pragma unroll
                for (int o = 0; o < CTAS; o++) st_dsmem_v4(mapa_shared(to + 16 * i, o), s);
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            for (int i = tid; i < QUADS; i += kUpThreads) {
                const int t = i / (RANKS / 4), r = r0 + i % (RANKS / 4) * 4;
                if (t >= tile.z) break;
                if (r >= padded) continue;
                float4 s = arrived[turn * CTAS * QUADS + i];
#pragma unroll
                for (int o = 1; o < CTAS; o++) {
                    const float4 y = arrived[(turn * CTAS + o) * QUADS + i];
                    s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
                }
                *reinterpret_cast<float4 *>(v + t * padded + r) = r < rank ? s : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            turn ^= 1;
        }
        if (rank) {
            __syncthreads();
            place_v<T, 16>(upper, lower, factor, v_pitch, padded, scale, [&](int t, int r) {
                return t < tile.z && r < rank ? *reinterpret_cast<const float4 *>(v + t * padded + r) : make_float4(0.f, 0.f, 0.f, 0.f);
            });
        }

        // ---- out = y + scale up v (the barrier in the loop is also that of v)
        for (int stage = 0, last = 0; block < end; block++) {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            for (int group = 0; group < groups; group++) {
                copy_wait<S - 2>();
                __syncthreads();                 // the stage is there, and everybody is done with the one before it
                issue(stage == 0 ? S - 1 : stage - 1);
                const int ranks = min(rank - group * RANKS, RANKS);
                if (ranks > 0)
                    multiply_up<T, RANKS, 4>(acc, shared_addr(upper) + (uint32_t)((lane & 15) * v_pitch + group * (RANKS * 2) + (lane >> 4) * 16), (uint32_t)(16 * v_pitch),
                                             shared_addr(smem + stage * Up::kStage) + (uint32_t)((warp * 32 + (lane & 7)) * Up::kPitch + (lane >> 3) * 16), (ranks + 15) / 16);
                last = stage;
                if (++stage == S) stage = 0;
            }
            write_out<T, 1>(now, acc, factor, row, rank > 0, a.vectors && (block + 1) * COLUMNS <= N, smem + last * Up::kStage + mine, N - (block * COLUMNS + warp * 32 + quad * 8));
#pragma unroll
            for (int h = 0; h < 2; h++) { now.y[h] += COLUMNS; now.out[h] += COLUMNS; }
        }
        copy_wait<0>();
    }
}

static int check_low_rank(const ortho_b200_low_rank_desc *d)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->tokens < 0 || d->tokens > 0x7FFF0000 || d->K < 8 || d->K % 8 || d->K > 0x3FFFFFFF || d->N < 1 || d->N > 0x3FFFFFFF || d->adapters < 1 || d->adapters > kMostAdapters || d->rank < 8 || d->rank % 8 || d->rank > 256)
        return ORTHO_B200_ERR_SHAPE;
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->x || !d->y || !d->out || !d->down || !d->up || !d->ids) return ORTHO_B200_ERR_NULL;
    if ((((uintptr_t)d->x | (uintptr_t)d->down | (uintptr_t)d->up) & 15u) || d->x_stride % 8) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

// ---- host -------------------------------------------------------------------------------------------------------------
struct LowRankSpace { int64_t order, tiles, v, bytes; };

// the most tiles that these tokens can have: an adapter's last tile may hold fewer tokens
static int64_t most_tiles(const ortho_b200_low_rank_desc &d, int tile)
{
    const int64_t most = d.tokens / tile + d.adapters + 1;
    return most < d.tokens ? most : d.tokens;
}

// Up to kFewTokens tokens both products run in one kernel (one launch, no exchange through memory) where it is not the slower way.  A unit is a tile and eight blocks
// of columns, the work of a cluster, of which the GPU holds some 32 at once.  Every cluster computes v of its tile for itself, 32 ranks a round that ends with an
// exchange: several clusters of a tile (wide) do that over again, and two kernels split ranks and columns over the whole GPU.  Tiles are reckoned as one per
// adapter that can be in use.  Measured, one kernel / two, GPU us, first K = 4096 then 14336:
//   wide,   1 token, 12288 columns (12 units): rank 16 4.7 / 5.0, 7.2 / 7.4;  32 5.5 / 5.6, 9.0 / 8.7;  48 8.0 / 6.1;  256 23.4 / 9.8
//   wide,   24 units: rank 16 5.2 / 5.1, 8.0 / 7.6;  32 6.2 / 5.6, 10.7 / 9.0;  48 9.2 / 6.2.   32 units: rank 16 6.4 / 5.2;  32 8.7 / 5.8.   48: rank 16 9.9 / 5.6
//   narrow, 1 unit: rank 16 4.7 / 5.1;  32 5.5 / 5.7, 8.9 / 8.8;  48 7.9 / 6.3;  256 22.9 / 9.1.   16 units: rank 32 6.5 / 7.0;  48 9.4 / 7.9
//   narrow, 28 units: rank 16 5.8 / 7.0;  32 7.0 / 7.7;  48 10.0 / 12.2;  64 10.3 / 12.4;  128 17.8 / 17.8;  256 49.8 / 29.3.   36 units: rank 16 10.2 / 7.3
static bool in_one_kernel(const ortho_b200_low_rank_desc &d)
{
    // (a cluster reads x while another writes: not where out lies in x)
    const char *const x = static_cast<const char *>(d.x), *const out = static_cast<const char *>(d.out);
    if (out < x + 2 * ((d.tokens - 1) * d.x_stride + d.K) && x < out + 2 * ((d.tokens - 1) * d.out_stride + d.N)) return false;
    if (d.tokens > kFewTokens || d.rank > kFewRank) return false;
    const int64_t sms = device_sm_count(current_device_index()), clusters = ceil_div(ceil_div(d.N, UpShape<1, 16>::kColumns), FewShape<1>::kCtas);
    const int64_t in_use = d.tokens < d.adapters ? d.tokens : d.adapters, full = ceil_div(d.tokens, kFewTile), units = (in_use > full ? in_use : full) * clusters;
    if (clusters > 1) return units <= sms / (d.rank <= 16 ? 6 : 12) && d.rank <= 32;
    return units <= 2 * sms / 9 && (d.rank <= 32 || units >= sms / 6);
}

static LowRankSpace low_rank_space(const ortho_b200_low_rank_desc &d)
{
    auto room = [](int64_t b) { return (b + 255) / 256 * 256; };
    LowRankSpace s = {};
    if (in_one_kernel(d)) return s;
    if (d.tokens > kFewTokens) {
        s.order = 256;
        s.tiles = s.order + room(4 * d.tokens);
        s.v = s.tiles + room(16 * most_tiles(d, kManyTile));
    }
    s.bytes = s.v + room(4 * d.tokens * d.rank);
    return s;
}

// clusters of `ctas` CTAs, `count` of them, as a programmatic dependent
static int launch_clusters(void (*kernel)(LowRankArgs), int64_t count, int ctas, size_t smem, const LowRankArgs &a, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(count * ctas)); cfg.blockDim = dim3(128); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    OB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    count_launch();
    return ORTHO_B200_OK;
}
template <class T, int MB>
static int launch_few(LowRankArgs &a, int dev, cudaStream_t stream)
{
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(few_kernel<T, MB>, cudaFuncAttributeMaxDynamicSharedMemorySize, FewShape<MB>::bytes(kFewRank)));
        attr_set[dev] = true;
    }
    a.blocks = (int)ceil_div(a.d.N, UpShape<1, 16>::kColumns);
    const int64_t units = most_tiles(a.d, kFewTile) * ceil_div(a.blocks, FewShape<MB>::kCtas), room = 2 * (int64_t)device_sm_count(dev) / FewShape<MB>::kCtas;
    return launch_clusters(few_kernel<T, MB>, units < room ? units : room, FewShape<MB>::kCtas, (size_t)FewShape<MB>::bytes(a.padded), a, stream);
}

template <class T, int MB, bool FEW>
static int launch_down(LowRankArgs &a, int dev, cudaStream_t stream)
{
    a.rank_groups = (int)ceil_div(a.d.rank, MB * 16);
    const int64_t units = most_tiles(a.d, FEW ? kFewTile : kManyTile) * a.rank_groups, room = 4 * (int64_t)device_sm_count(dev) / kManyCtas;
    static_assert(kFewCtas == kManyCtas, "clusters of one size");
    if constexpr (FEW) {
        return launch_clusters(down_few_kernel<T, MB>, units < room ? units : room, kFewCtas, 0, a, stream);
    } else {
        constexpr int smem = kDownStages * (kManyTile + MB * 16) * 128;
        static bool attr_set[kMaxDevices] = {};
        if (!attr_set[dev]) {
            OB_CUDA(cudaFuncSetAttribute(down_many_kernel<T, MB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            attr_set[dev] = true;
        }
        return launch_clusters(down_many_kernel<T, MB>, units < room ? units : room, kManyCtas, smem, a, stream);
    }
}

template <class T, int G, bool FEW>
static int launch_up(LowRankArgs &a, int dev, cudaStream_t stream)
{
    constexpr int MT = FEW ? kFewTile / 16 : kManyTile / 16;
    using Shape = UpShape<MT, G>;
    auto bytes = [](int padded) { return kUpStages * Shape::kStage + 2 * Shape::kTokens * (padded * 2 + 16); };
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(up_kernel<T, MT, G, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(256)));
        attr_set[dev] = true;
    }
    a.blocks = (int)ceil_div(a.d.N, Shape::kColumns);
    const int smem = bytes(a.padded), fit = 227 * 1024 / (smem + (FEW ? 7 : 2) * 1024);
    const int64_t pairs = most_tiles(a.d, Shape::kTokens) * a.blocks, room = (fit < 4 ? fit : 4) * (int64_t)device_sm_count(dev);
    return launch_dependent(up_kernel<T, MT, G, FEW>, dim3((unsigned)(pairs < room ? pairs : room)), kUpThreads, (size_t)smem, stream, a);
}

template <class T, bool FEW>
static int launch_two(LowRankArgs &a, int dev, cudaStream_t stream)
{
    const int st = a.d.rank <= 16 ? launch_down<T, 1, FEW>(a, dev, stream) : launch_down<T, 2, FEW>(a, dev, stream);
    if (st) return st;
    return a.padded <= 16 ? launch_up<T, 16, FEW>(a, dev, stream) : a.padded <= 32 ? launch_up<T, 32, FEW>(a, dev, stream) : launch_up<T, 64, FEW>(a, dev, stream);
}

template <class T>
static int launch_low_rank(LowRankArgs &a, cudaStream_t stream)
{
    const auto &d = a.d;
    const int dev = current_device_index();
    if (dev < 0) return ORTHO_B200_ERR_CUDA;
    if (in_one_kernel(d)) return d.rank <= 16 ? launch_few<T, 1>(a, dev, stream) : launch_few<T, 2>(a, dev, stream);
    if (d.tokens <= kFewTokens) return launch_two<T, true>(a, dev, stream);
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(group_kernel<kManyTile>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * (kMostAdapters + 1)));
        attr_set[dev] = true;
    }
    const int st = launch_dependent(group_kernel<kManyTile>, dim3(1), kGroupThreads, (size_t)(3 * 4 * (d.adapters + 1)), stream, a);
    return st ? st : launch_two<T, false>(a, dev, stream);
}

}  // namespace ob

using namespace ob;

extern "C" int64_t ortho_b200_low_rank_add_workspace_bytes(const ortho_b200_low_rank_desc *d)
{
    if (check_low_rank(d) != ORTHO_B200_OK) return -1;
    return d->tokens ? low_rank_space(*d).bytes : 0;
}

extern "C" int ortho_b200_low_rank_add(const ortho_b200_low_rank_desc *d, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_low_rank(d);
    if (st || d->tokens == 0) return st;
    const LowRankSpace space = low_rank_space(*d);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes || ((uintptr_t)workspace & 255u))) return ORTHO_B200_ERR_WORKSPACE;
    st = check_device();
    if (st) return st;
    LowRankArgs a = {};
    a.d = *d;
    unsigned char *const w = static_cast<unsigned char *>(workspace);
    a.heads = reinterpret_cast<int *>(w);
    a.order = reinterpret_cast<int *>(w + space.order);
    a.tiles = reinterpret_cast<int4 *>(w + space.tiles);
    a.v = reinterpret_cast<float *>(w + space.v);
    a.padded = (int)((d->rank + 15) / 16 * 16);
    a.up_groups = (int)ceil_div(d->rank, 64);
    a.vectors = (((uintptr_t)d->y | (uintptr_t)d->out) & 15u) == 0 && d->y_stride % 8 == 0 && d->out_stride % 8 == 0;
    a.copies = d->out != d->y || d->out_stride != d->y_stride;
    return d->type == ORTHO_B200_TYPE_F16 ? launch_low_rank<__half>(a, (cudaStream_t)stream) : launch_low_rank<__nv_bfloat16>(a, (cudaStream_t)stream);
}
