// Low-rank adapters of many requests beside a shared projection:
//
//     v[t] = down_e x[t],   out[t] = y[t] + scale_e up_e v[t],   e = ids[t]
//
// Few tokens: bound by the weights of the adapters in use (2 rank (K + N) bytes each).  Many tokens: by the activations (2 (K + 2 N) bytes a
// token).  The operations are a few per byte either way, so both products run on m16n8k16 tensor-core instructions with operands loaded
// straight from global memory, 16 or 8 bytes a lane: the order of k (or of the rank) inside an instruction is free as long as both operands use
// the same one.
//
// Tokens are grouped first, so that an adapter's weights are read once for all its tokens: `order` lists them by adapter, a tile is up to
// kTile of them with one adapter.  Up to kFewTokens tokens every CTA groups them for itself; more are grouped by a kernel in front.
//
// down_kernel: a cluster of CTAs per tile and 16 to 64 ranks, K split over its warps, their sums joined through distributed shared memory in a fixed
// order.  up_kernel: a CTA per tile and some columns; it is launched as a programmatic dependent and loads its first weights (constants of
// the layer) while down_kernel still runs.
#include "launch.cuh"
#include "tma.cuh"

namespace ob {

constexpr int kFewTokens = 128, kMostAdapters = 8192, kGroupThreads = 1024;

struct LowRankArgs {
    ortho_b200_low_rank_desc d;
    int *heads;                                  // {tiles with an adapter, all tiles}; these three: more than kFewTokens tokens
    int *order;                                  // [tokens] grouped by adapter, those without one last
    int4 *tiles;                                 // {adapter or -1, first place in order, tokens, 0}
    float *v;                                    // [tokens][rank], by place in order
    int rank_groups;
    bool vectors, copies;                        // rows of y and out in 16-byte pieces; out is not y
};

__device__ __forceinline__ int rank_of(const ortho_b200_low_rank_desc &d, int e)
{
    if (!d.ranks) return (int)d.rank;
    const int64_t r = ((int64_t)max(__ldcg(d.ranks + e), 0) + 7) / 8 * 8;
    return (int)(r < d.rank ? r : d.rank);
}
// the adapter of a token, or d.adapters for none
__device__ __forceinline__ int adapter_of(const ortho_b200_low_rank_desc &d, int64_t t)
{
    const int32_t e = __ldcg(d.ids + t);
    return e >= 0 && e < d.adapters && rank_of(d, e) > 0 ? e : (int)d.adapters;
}

// ---- grouping ----------------------------------------------------------------------------------------------------
struct FewTokens { int adapter[kFewTokens], order[kFewTokens]; int4 at[kFewTokens], tiles[kFewTokens]; int count[kFewTokens / 32]; };

// by a CTA of kFewTokens threads; returns (tiles with an adapter, all tiles)
template <int TILE>
__device__ __forceinline__ int2 group_few(FewTokens &g, const ortho_b200_low_rank_desc &d)
{
    const int t = threadIdx.x, T = (int)d.tokens, lane = t & 31, warp = t >> 5;
    const int e = t < T ? adapter_of(d, t) : 0x7FFFFFFF;
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
        if (before % TILE == 0) g.at[place] = make_int4(e < d.adapters ? e : -1, place, min(TILE, same - before), 0);
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
    extern __shared__ int counts[];              // [adapters + 1], then the next free place of each
    __shared__ int2 warp_sum[kGroupThreads / 32];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = (int)d.adapters + 1, T = (int)d.tokens;
    int *const first_tile = counts + E, *const start = first_tile + E;
    griddep_wait();
    griddep_launch();
    for (int e = tid; e < E; e += kGroupThreads) counts[e] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < T; t0 += kGroupThreads) {
        const int t = t0 + tid, e = t < T ? adapter_of(d, t) : -1;
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && __ffs(peers) - 1 == lane) atomicAdd(counts + e, __popc(peers));
    }
    __syncthreads();
    int2 before = make_int2(0, 0);               // tokens and tiles of the adapters before
    int real = 0;
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
        int2 total = before;
        for (int w = 0; w < kGroupThreads / 32; w++) {
            if (w == warp) { sum.x += total.x; sum.y += total.y; }
            total.x += warp_sum[w].x;
            total.y += warp_sum[w].y;
        }
        if (e < E) { start[e] = sum.x - n; first_tile[e] = sum.y - tiles; }
        if (e == E - 1) real = sum.y - tiles;
        before = total;
        __syncthreads();
    }
    if ((E - 1) % kGroupThreads == tid) { a.heads[0] = real; a.heads[1] = before.y; }
    int *const place = counts;                   // how many of an adapter have their place
    // (the counts are needed for the tiles' sizes: the next adapter's start less one's own)
    for (int e = tid; e < E; e += kGroupThreads) place[e] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < T; t0 += kGroupThreads) {
        const int t = t0 + tid, e = t < T ? adapter_of(d, t) : -1;
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        const int leader = __ffs(peers) - 1;
        int base = 0;
        if (e >= 0 && leader == lane) base = atomicAdd(place + e, __popc(peers));
        base = __shfl_sync(0xffffffffu, base, leader);
        if (e >= 0) {
            const int among = base + __popc(peers & ((1u << lane) - 1)), at = start[e] + among;
            a.order[at] = t;
            if (among % TILE == 0) {
                const int end = e + 1 < E ? start[e + 1] : T;
                a.tiles[first_tile[e] + among / TILE] = make_int4(e + 1 < E ? e : -1, at, min(TILE, end - at), 0);
            }
        }
    }
}

// ---- v = down x ------------------------------------------------------------------------------------------------------
constexpr int kDownWarps = 4;

// MB blocks of 16 ranks (the 16-row operand) by NT of 8 tokens
template <class T, int MB, int NT, bool FEW>
__global__ void __launch_bounds__(32 * kDownWarps)
down_kernel(const __grid_constant__ LowRankArgs a)
{
    constexpr int TOKENS = NT * 8, RANKS = MB * 16, PITCH = RANKS + 4, CHUNKS = MB * NT >= 8 ? 2 : 4;
    __shared__ __align__(16) float sums[kDownWarps][TOKENS][PITCH];
    __shared__ __align__(16) unsigned char few_smem[FEW ? sizeof(FewTokens) : 16];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = (int)cluster_ctarank(), ctas = (int)cluster_nctarank();
    griddep_wait();
    griddep_launch();
    FewTokens &few = *reinterpret_cast<FewTokens *>(few_smem);
    const int *order;
    const int4 *tiles;
    int real;
    if constexpr (FEW) {
        real = group_few<TOKENS>(few, d).x;
        order = few.order;
        tiles = few.tiles;
    } else {
        real = a.heads[0];
        order = a.order;
        tiles = a.tiles;
    }
    const int K = (int)d.K, steps = (K + 31) / 32, clusters = gridDim.x / ctas;
    const int quad = lane & 3, row = lane >> 2;
    for (int64_t unit = blockIdx.x / ctas; unit < (int64_t)real * a.rank_groups; unit += clusters) {
        const int4 tile = tiles[unit / a.rank_groups];
        const int r0 = (int)(unit % a.rank_groups) * RANKS, rank = rank_of(d, tile.x);
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
        // 32 k a step, 8 of them (16 bytes of every row) a lane; steps are dealt to the cluster's warps in turn
        const int stride = ctas * kDownWarps;
        for (int s0 = cta * kDownWarps + warp; s0 < steps; s0 += CHUNKS * stride) {
            uint4 wv[CHUNKS][MB][2], xv[CHUNKS][NT];
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const int k = (s0 + c * stride) * 32 + quad * 8;
                const bool on = k < K;
#pragma unroll
                for (int m = 0; m < MB; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        wv[c][m][h] = on && r0 + m * 16 + h * 8 + row < rank ? ldg_stream(w + (int64_t)(m * 16 + h * 8) * d.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NT; j++)
                    xv[c][j] = on && j * 8 < tile.z ? *reinterpret_cast<const uint4 *>(x[j] + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if (j * 8 >= tile.z) continue;
#pragma unroll
                    for (int m = 0; m < MB; m++) {
                        const uint32_t lo[4] = {wv[c][m][0].x, wv[c][m][1].x, wv[c][m][0].y, wv[c][m][1].y};
                        const uint32_t hi[4] = {wv[c][m][0].z, wv[c][m][1].z, wv[c][m][0].w, wv[c][m][1].w};
                        Half<T>::mma(acc[m][j], lo, xv[c][j].x, xv[c][j].y);
                        Half<T>::mma(acc[m][j], hi, xv[c][j].z, xv[c][j].w);
                    }
                }
        }
#pragma unroll
        for (int m = 0; m < MB; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) sums[warp][j * 8 + quad * 2 + (e & 1)][m * 16 + row + (e >> 1) * 8] = acc[m][j][e];
        __syncthreads();
        // the warps' sums, then the cluster's, each in order
        float4 *const mine = reinterpret_cast<float4 *>(&sums[0][0][0]);
        constexpr int QUADS = RANKS / 4, WARP_QUADS = TOKENS * PITCH / 4;
        for (int i = tid; i < TOKENS * QUADS; i += 32 * kDownWarps) {
            const int at = i / QUADS * (PITCH / 4) + i % QUADS;
            float4 s = mine[at];
#pragma unroll
            for (int o = 1; o < kDownWarps; o++) {
                const float4 y = mine[o * WARP_QUADS + at];
                s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
            }
            mine[at] = s;
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        for (int i = cta * 32 * kDownWarps + tid; i < TOKENS * QUADS; i += ctas * 32 * kDownWarps) {
            const int token = i / QUADS, q = i % QUADS;
            if (token >= tile.z || r0 + q * 4 >= rank) continue;
            const uint32_t at = shared_addr(mine + token * (PITCH / 4) + q);
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int o = 0; o < ctas; o++) {
                const uint32_t from = mapa_shared(at, o);
                float4 y;
                asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(from));
                s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
            }
            *reinterpret_cast<float4 *>(a.v + (int64_t)(tile.y + token) * d.rank + r0 + q * 4) = s;
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

// ---- out = y + scale up v -------------------------------------------------------------------------------------------
static_assert(kFewTokens == 32 * kDownWarps, "a thread per token");
constexpr int kUpWarps = 4, kUpColumns = 32 * kUpWarps;

// One unit of 32 columns by 64 ranks: rows of `up` as the 8-column operand, 4 tiles of 8 by 4 steps of 16 ranks.  Column c of tile j stands for
// output column 8 (c / 2) + 2 j + c % 2, so that a lane's results over the four tiles are eight neighbours.
template <class T>
__device__ __forceinline__ void load_up(uint2 (&w)[4][4], const LowRankArgs &a, int e, int rank, int64_t n0, int r0, int lane)
{
    const int row = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t n = n0 + (row >> 1) * 8 + j * 2 + (row & 1);
        const T *const p = (const T *)a.d.up + ((int64_t)e * a.d.N + n) * a.d.rank + r0 + quad * 4;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            w[j][s] = make_uint2(0, 0);
            if (n < a.d.N && r0 + s * 16 + quad * 4 < rank)
                asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(w[j][s].x), "=r"(w[j][s].y) : "l"(p + s * 16));
        }
    }
}

// MT tiles of 16 tokens
template <class T, int MT, bool FEW>
__global__ void __launch_bounds__(32 * kUpWarps)
up_kernel(const __grid_constant__ LowRankArgs a)
{
    constexpr int TOKENS = MT * 16;
    constexpr bool NORMED = sizeof(T) == 2 && std::is_same<T, __half>::value;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float factor[TOKENS];
    __shared__ __align__(16) unsigned char few_smem[FEW ? sizeof(FewTokens) : 16];
    const auto &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, row = lane >> 2;
    const int padded = ((int)d.rank + 15) / 16 * 16, pitch = padded * 2 + 16;
    unsigned char *const upper = smem, *const lower = smem + TOKENS * pitch;
    // What is read in front of the wait was complete before down_kernel began (it lets this kernel start behind its own wait), or is
    // a constant of the layer.
    griddep_launch();
    FewTokens &few = *reinterpret_cast<FewTokens *>(few_smem);
    const int *order;
    const int4 *tiles;
    int all;
    if constexpr (FEW) {
        const int2 n = group_few<TOKENS>(few, d);
        all = a.copies ? n.y : n.x;
        order = few.order;
        tiles = few.tiles;
    } else {
        all = __ldcg(a.heads + (a.copies ? 1 : 0));
        order = a.order;
        tiles = a.tiles;
    }
    const int64_t blocks = (d.N + kUpColumns - 1) / kUpColumns;
    // blocks of columns per unit: several where there are units enough, so that v is brought into place less often
    int64_t span = all * blocks / ((int64_t)gridDim.x * 4);
    span = span < 1 ? 1 : span < 8 ? span : 8;
    const int64_t spans = (blocks + span - 1) / span, units = all * spans;
    bool waited = false;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        int4 tile;
        if constexpr (FEW) tile = tiles[unit / spans];
        else tile = __ldcg(tiles + unit / spans);
        const int64_t first = unit % spans * span * kUpColumns, end = min(first + span * kUpColumns, d.N);
        const int e = tile.x, rank = e < 0 ? 0 : rank_of(d, e);
        uint2 w[4][4];
        if (e >= 0) load_up<T>(w, a, e, rank, first + warp * 32, 0, lane);
        if (!waited) griddep_wait();
        waited = true;
        __syncthreads();                         // the unit before is done with v
        if (e >= 0) {
            // v as two 16-bit parts, ranks in the order of the loads above; FP16: relative to the token's largest, by a power of two
            for (int t = warp; t < TOKENS; t += kUpWarps) {
                float4 x[2];
                float top = 0.f;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int r = (h * 32 + lane) * 4;
                    x[h] = t < tile.z && r < rank ? __ldcg(reinterpret_cast<const float4 *>(a.v + (int64_t)(tile.y + t) * d.rank + r)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x[h].x), fabsf(x[h].y)), fmaxf(fabsf(x[h].z), fabsf(x[h].w))));
                }
                float back = 1.f;
                if (NORMED) {
#pragma unroll
                    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const int exponent = (int)(__float_as_uint(top) >> 23);                   // top in [2^(exponent - 127), 2^(exponent - 126))
                    if (exponent >= 14 && exponent <= 253) {                                  // (else: tiny, infinite or NaN as it is)
                        const float down = __uint_as_float((uint32_t)(min(127 + 140 - exponent, 254)) << 23);
                        back = __uint_as_float((uint32_t)(254 - min(127 + 140 - exponent, 254)) << 23);
#pragma unroll
                        for (int h = 0; h < 2; h++) { x[h].x *= down; x[h].y *= down; x[h].z *= down; x[h].w *= down; }
                    }
                }
                if (lane == 0) factor[t] = back * (d.scales ? __ldcg(d.scales + e) : 1.f);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int r = (h * 32 + lane) * 4;
                    if (r >= padded) continue;
                    const uint32_t u0 = Half<T>::pack(x[h].x, x[h].y), u1 = Half<T>::pack(x[h].z, x[h].w);
                    const float2 f0 = Half<T>::unpack(u0), f1 = Half<T>::unpack(u1);
                    const int at = t * pitch + (r >> 4) * 32 + (r & 15);                      // four ranks: two words, eight ranks apart
                    *reinterpret_cast<uint32_t *>(upper + at) = u0;
                    *reinterpret_cast<uint32_t *>(upper + at + 16) = u1;
                    *reinterpret_cast<uint32_t *>(lower + at) = Half<T>::pack(x[h].x - f0.x, x[h].y - f0.y);
                    *reinterpret_cast<uint32_t *>(lower + at + 16) = Half<T>::pack(x[h].z - f1.x, x[h].w - f1.y);
                }
            }
        }
        __syncthreads();
        for (int64_t n0 = first + warp * 32; n0 < end; n0 += kUpColumns) {
            const int64_t n = n0 + quad * 8;
            float acc[MT][4][4];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
            const bool whole = a.vectors && n + 8 <= d.N;
            for (int r0 = 0; r0 < rank; r0 += 64) {
                uint2 next[4][4];
                const bool more = r0 + 64 < rank || n0 + kUpColumns < end;
                if (more) load_up<T>(next, a, e, rank, r0 + 64 < rank ? n0 : n0 + kUpColumns, r0 + 64 < rank ? r0 + 64 : 0, lane);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (r0 + s * 16 >= rank) break;
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        if (m * 16 >= tile.z) break;
                        uint32_t v[4];
                        const int at = (m * 16 + (lane & 15)) * pitch + (r0 / 16 + s) * 32 + (lane >> 4) * 16;
                        ldmatrix4(v, shared_addr(upper + at));
#pragma unroll
                        for (int j = 0; j < 4; j++) Half<T>::mma(acc[m][j], v, w[j][s].x, w[j][s].y);
                        ldmatrix4(v, shared_addr(lower + at));
#pragma unroll
                        for (int j = 0; j < 4; j++) Half<T>::mma(acc[m][j], v, w[j][s].x, w[j][s].y);
                    }
                }
                if (more) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int s = 0; s < 4; s++) w[j][s] = next[j][s];
                }
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int t = m * 16 + h * 8 + row;
                    if (t >= tile.z || n >= d.N) continue;
                    const int64_t token = FEW ? order[tile.y + t] : __ldcg(order + tile.y + t);
                    const T *const y = (const T *)d.y + token * d.y_stride + n;
                    T *const out = (T *)d.out + token * d.out_stride + n;
                    const float f = e < 0 ? 0.f : factor[t];
                    if (whole) {
                        uint4 u = *reinterpret_cast<const uint4 *>(y);
                        if (e >= 0) {
                            uint32_t *const p = reinterpret_cast<uint32_t *>(&u);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const float2 was = Half<T>::unpack(p[j]);
                                p[j] = Half<T>::pack(was.x + f * acc[m][j][2 * h], was.y + f * acc[m][j][2 * h + 1]);
                            }
                        }
                        *reinterpret_cast<uint4 *>(out) = u;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (n + i < d.N) out[i] = e < 0 ? y[i] : Half<T>::from_float(Half<T>::to_float(y[i]) + f * acc[m][i >> 1][2 * h + (i & 1)]);
                    }
                }
        }
    }
    if (!waited) griddep_wait();
}

static int check_low_rank(const ortho_b200_low_rank_desc *d)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->tokens < 0 || d->tokens > 0x7FFFFFFF || d->K < 8 || d->K % 8 || d->K > 0x3FFFFFFF || d->N < 1 || d->N > 0x7FFFFFFF || d->adapters < 1 || d->adapters > kMostAdapters || d->rank < 8 || d->rank % 8 || d->rank > 256)
        return ORTHO_B200_ERR_SHAPE;
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->x || !d->y || !d->out || !d->down || !d->up || !d->ids) return ORTHO_B200_ERR_NULL;
    if ((((uintptr_t)d->x | (uintptr_t)d->down | (uintptr_t)d->up) & 15u) || d->x_stride % 8) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

// ---- host -------------------------------------------------------------------------------------------------------------
struct LowRankSpace { int64_t order, tiles, v, bytes; };
constexpr int kFewTile = 16, kManyTile = 64;

static LowRankSpace low_rank_space(const ortho_b200_low_rank_desc &d)
{
    auto room = [](int64_t b) { return (b + 255) / 256 * 256; };
    LowRankSpace s = {};
    if (d.tokens > kFewTokens) {
        s.order = 256;
        s.tiles = s.order + room(4 * d.tokens);
        const int64_t most = d.tokens / kManyTile + d.adapters + 1;             // an adapter's last tile may hold fewer tokens
        s.v = s.tiles + room(16 * (most < d.tokens ? most : d.tokens));
    }
    s.bytes = s.v + room(4 * d.tokens * d.rank);
    return s;
}

template <class T, int MB, int NT, bool FEW>
static int launch_down(LowRankArgs &a, int cluster, cudaStream_t stream)
{
    const auto &d = a.d;
    const int tile = NT * 8;
    a.rank_groups = (int)ceil_div(d.rank, MB * 16);
    const int64_t most = d.tokens / tile + d.adapters, units = (most < d.tokens ? most : d.tokens) * a.rank_groups;
    const int64_t room = 4 * (int64_t)device_sm_count(current_device_index()) / cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((units < room ? units : room) * cluster)); cfg.blockDim = dim3(32 * kDownWarps); cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    OB_CUDA(cudaLaunchKernelEx(&cfg, down_kernel<T, MB, NT, FEW>, a));
    count_launch();
    return ORTHO_B200_OK;
}

template <class T, int MT, bool FEW>
static int launch_up(const LowRankArgs &a, cudaStream_t stream)
{
    const auto &d = a.d;
    const int64_t pitch = (d.rank + 15) / 16 * 32 + 16, smem = 2 * MT * 16 * pitch;
    const int dev = current_device_index();
    if (dev < 0) return ORTHO_B200_ERR_CUDA;
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(up_kernel<T, MT, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * MT * 16 * (256 * 2 + 16)));
        attr_set[dev] = true;
    }
    const int64_t most = d.tokens / (MT * 16) + d.adapters + 1, units = (most < d.tokens ? most : d.tokens) * ceil_div(d.N, kUpColumns);
    const int64_t room = (int64_t)device_sm_count(dev) * (FEW ? 4 : 3);
    return launch_dependent(up_kernel<T, MT, FEW>, dim3((unsigned)(units < room ? units : room)), 32 * kUpWarps, (size_t)smem, stream, a);
}

template <class T>
static int launch_low_rank(LowRankArgs &a, cudaStream_t stream)
{
    const auto &d = a.d;
    int st;
    if (d.tokens <= kFewTokens) {
        st = d.rank <= 16 ? launch_down<T, 1, kFewTile / 8, true>(a, 8, stream)
           : d.rank <= 32 ? launch_down<T, 2, kFewTile / 8, true>(a, 8, stream) : launch_down<T, 4, kFewTile / 8, true>(a, 8, stream);
        return st ? st : launch_up<T, kFewTile / 16, true>(a, stream);
    }
    const int dev = current_device_index();
    if (dev < 0) return ORTHO_B200_ERR_CUDA;
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(group_kernel<kManyTile>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * (kMostAdapters + 1)));
        attr_set[dev] = true;
    }
    st = launch_dependent(group_kernel<kManyTile>, dim3(1), kGroupThreads, (size_t)(3 * 4 * (d.adapters + 1)), stream, a);
    if (st) return st;
    st = d.rank <= 16 ? launch_down<T, 1, kManyTile / 8, false>(a, 4, stream) : launch_down<T, 2, kManyTile / 8, false>(a, 4, stream);
    return st ? st : launch_up<T, kManyTile / 16, false>(a, stream);
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
    if (!workspace || workspace_bytes < space.bytes || ((uintptr_t)workspace & 255u)) return ORTHO_B200_ERR_WORKSPACE;
    st = check_device();
    if (st) return st;
    LowRankArgs a = {};
    a.d = *d;
    unsigned char *const w = static_cast<unsigned char *>(workspace);
    a.heads = reinterpret_cast<int *>(w);
    a.order = reinterpret_cast<int *>(w + space.order);
    a.tiles = reinterpret_cast<int4 *>(w + space.tiles);
    a.v = reinterpret_cast<float *>(w + space.v);
    a.vectors = (((uintptr_t)d->y | (uintptr_t)d->out) & 15u) == 0 && d->y_stride % 8 == 0 && d->out_stride % 8 == 0;
    a.copies = d->out != d->y || d->out_stride != d->y_stride;
    return d->type == ORTHO_B200_TYPE_F16 ? launch_low_rank<__half>(a, (cudaStream_t)stream) : launch_low_rank<__nv_bfloat16>(a, (cudaStream_t)stream);
}
