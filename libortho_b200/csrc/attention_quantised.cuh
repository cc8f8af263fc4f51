// Attention of one new token per row over a paged cache held in 4 bits (quantised.cuh; one source for both 16-bit types):
//
//     s_j = scale sum_g (ks_jg sum_i q_i (c_ji - 8) + (kz_jg + 8 ks_jg) sum_i q_i),
//     out_i = sum_j p_j (vs_jg (d_ji - 8) + vz_jg + 8 vs_jg) / sum_j p_j,     p_j = exp(s_j - max)
//
// with codes c and d of keys and values, scales and zeros of their groups g.  The division of the work and the joining are those of attention.cuh; a unit is 128 keys, 32 a
// warp.  The bytes are a quarter, so what bounds it is the warps' instructions (some 400 for 16 keys of 128 elements and up to 8 queries, 130 of them unpacking).
// Codes enter the products as whole numbers, and scales and zeros are applied to what a group's elements or 16 keys have in common:
//   * A code in the low bits of a 16-bit half is itself a subnormal FP16 number.  The tensor core aligns a product by its factors' exponents, which of a subnormal number is that of the
//     smallest normal one, 2^-14, and cuts what lies 2^-25 below the largest product or sum of a step, towards zero (measured with single products).  A code at bits 0 to 3 therefore
//     leaves a factor only 15 bits below the step's largest one.
//   * Keys: codes at bits 2 to 5 and 6 to 9, code 2^-22 and code 2^-18, a shift for two of them and a mask each; a query's small elements keep their digits, lse of a few keys
//     is off by 1.5e-7 (1.3e-6 at bits 0 to 3 and 4 to 7, with a shift less a word; 9e-8 as the values below, 3 us of 91 more).  Elements are taken in the order in which a word has them, the
//     queries likewise, and a sixteenth of those that meet codes 2^-18.  S^T = K Q^T starts from -8 sum q: codes around zero keep sums small.
//   * Values: codes less 8 as normal numbers, an FP16 multiply-add each.  Weights differ by orders of magnitude, and what small ones lost beside large ones as
//     subnormal factors had one sign: 1.1e-4 of an average over 131072 keys, 28 % of FP16 outputs rounded otherwise than those of an FP32 form (now 0.9 %; 90.7 us against 88.5).
//     Up to 8 queries: FP32 adds up sums of 32 keys.  More: they stay in the tensor core's, where every step of 16 keys may take 2^-23 off them.
//   * p vs enters as FP16, with its rest as a second part.  A power of two per query brings the largest of its item to 2^7 .. 2^15: one of the scales alone, or one
//     kept from item to item, would let a key that weighs nothing, or another request, push the others' into FP16's subnormal numbers.  p (vz + 8 vs) is summed in FP32 per query.
// FP16 serves BF16 models too: a query is multiplied by a power of two that brings its largest element to 2^14.
// Measured (GPU time, us): 2 x 131072 keys of 8 heads of 128, 285 MB: 91 = 3.1 TB/s (a 16-bit cache: 166); 32 requests of up to 4096 keys, log-spread: 21;
// 100 of up to 8000 with scales for every 64 elements: 54; 16 of up to 10000 with 16 queries and heads of 256: 25; 1 x 1000 keys of 32 heads: 7.7.  Warps wait for fixed latencies, 56 % of
// the issue slots in use; in short runs for instructions, because a unit's are more than the nearest cache holds (heads of 256: three of seven cycles).  Tried, against what the kernel took
// then: four CTAs an SM with 128 registers 93 (88), two 107 (99); a pair of lanes for the rows of a pair of keys, which saves exchanges of addresses but touches four times the lines a
// copy, 99 (91); tiles of 16 keys one by one 94 (91); values' codes as subnormal numbers at bits 2 to 5 and 6 to 9, their sums turned round every other time, 96 (91).
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "quantised.cuh"

namespace ob {

struct QuantisedAttentionArgs {
    AttentionArgs a;                             // (d.kv_heads, head_dim, pages, page_size are the cache's; the other fields of a cache are not read)
    ortho_b200_quantised_cache c;
    int wide;                                    // rows of the cache are whole 16-byte pieces, fewer than 2^32 of them; and strides in such pieces
    uint32_t k_page, k_slot, v_page, v_slot, ks_page, ks_slot, vs_page, vs_slot;
};

constexpr float kNone = -1e30f;
constexpr int kQWarpKeys = 32, kQUnitKeys = kQWarpKeys * kAttnWarps;

template <int DP, int NT, bool GROUPED>
struct QuantisedShape {
    static constexpr int kGroups = GROUPED ? DP / kQuantGroup : 1;
    // Rows are an odd number of 16-byte pieces, so that the words that a warp reads together (8 keys x 4 words; 4 pairs of keys x 8 words) lie in 32 banks
    static constexpr int kPitch = DP / 2 + (DP / 32 % 2 ? 0 : 16), kPieces = DP / 32;
    static constexpr int kCodes = kQWarpKeys * kPitch, kScales = kQWarpKeys * kGroups * 4;
    static constexpr int kStage = 2 * (kCodes + kScales);
    static constexpr int kQPitch = DP * 2 + 16, kQ = NT * 8 * kQPitch;
    static constexpr int kFoldPitch = DP + 4;
    static_assert(8 * kFoldPitch * 4 <= kStage, "room for 8 queries");
    static constexpr bool kKeepQ = NT * DP <= 256;                             // query operands stay in registers
    static constexpr int kOperands = kKeepQ ? 0 : NT * DP / 32 * 512;
    static constexpr int bytes(int stages) { return stages * (kAttnWarps * kStage + kQ) + kOperands + kAttnWarps * NT * 8 * 8; }
    static constexpr int kFour = 57088, kThree = 76458, kTwo = 115712, kOne = 232448;
    // CTAs an SM, by the registers that NT * DP sums and up to 16 queries' operands leave: four have 128 of them, three 168, two 255.  Measured, 60 requests of up to 8000 keys, log-spread, 8
    // key-value heads, us.  Four / three: heads of 64, 8 queries or fewer 25.9 / 25.8, 16 queries 51.5 / 38.7; of 96 32.4 / 29.5, of 128 37.0 / 33.4.  Three / two: of 192 46.2 / 46.9;
    // of 96, 16 queries 57.9 / 48.6; of 128, 12 queries 59.4 / 51.8, of 64, 24 queries 90.7 / 65.7.
    static constexpr int kWanted = NT * DP <= 64 ? 4 : NT * DP <= (NT == 1 ? 192 : 128) ? 3 : 2;
    static constexpr int kRoom = kWanted == 4 && bytes(2) <= kFour ? kFour : kWanted >= 3 && bytes(2) <= kThree ? kThree : kWanted >= 2 && bytes(2) <= kTwo ? kTwo : kOne;
    static constexpr int kStages = bytes(4) <= kRoom ? 4 : bytes(3) <= kRoom ? 3 : 2, kBytes = bytes(kStages);
    static constexpr int kPerSm = kRoom == kFour ? 4 : kRoom == kThree ? 3 : kRoom == kTwo ? 2 : 1;
    static constexpr int kMostRanks = 8;
    static constexpr int kArrived = kMostRanks * NT * 8 * 8 + NT * 8 * DP * 4 + kMostRanks * 16, kClusterBytes = (kBytes + 15) / 16 * 16 + kArrived;
    static constexpr int kClusterPerSm = kClusterBytes <= kFour && kPerSm >= 4 ? 4 : kClusterBytes <= kThree && kPerSm >= 3 ? 3 : kClusterBytes <= kTwo && kPerSm >= 2 ? 2 : kClusterBytes <= kOne ? 1 : 0;
};

__device__ __forceinline__ uint32_t word_at(const unsigned char *p) { return *reinterpret_cast<const uint32_t *>(p); }
__device__ __forceinline__ void copy4_async(uint32_t dst, const void *src, bool on)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
// Four codes of a 16-bit half as FP16 numbers; w: the codes of two keys or elements, one in each half.
// As they lie, at bits 2 to 5 or 6 to 9 once w is shifted: subnormal numbers, code 2^-22 (even NUMBER) and code 2^-18
template <int NUMBER> __device__ __forceinline__ uint32_t codes(uint32_t w) { return (NUMBER < 2 ? w << 2 : w >> 6) & (NUMBER % 2 ? 0x03C003C0u : 0x003C003Cu); }
// As normal numbers around zero, (code - 8) 2^-9
template <int NUMBER> __device__ __forceinline__ uint32_t centred_codes(uint32_t w)
{
    const uint32_t b = (NUMBER < 2 ? w : w >> 8) & (NUMBER % 2 ? 0x00F000F0u : 0x000F000Fu), by = NUMBER % 2 ? 0x68006800u : 0x78007800u, less = 0xA400A400u;
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&b), *reinterpret_cast<const __half2 *>(&by), *reinterpret_cast<const __half2 *>(&less));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// a b + c with FP32's subnormal numbers, which scores of very small keys pass through
__device__ __forceinline__ float mul_add(float a, float b, float c) { float r; asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// 2^8 / x of a power of two between 2^-118 and 2^126
__device__ __forceinline__ float two_to_8_over(float x) { return __uint_as_float((262u << 23) - __float_as_uint(x)); }

// Eight elements of a query, in memory's order, as the products take them: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ uint4 as_codes_lie(uint4 w)
{
    return make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410), __byte_perm(w.y, w.w, 0x7632));
}

// One query's operands: `row` is its place in shared memory, thread t of four has the words 4 j + t.  f: what the products are to be multiplied by;
// sums: of its elements, per group.
template <class T, int DP, int GROUPS>
__device__ __forceinline__ void query_operands(const unsigned char *row, int t, uint4 (&w)[DP / 32], float &f, float (&sums)[GROUPS])
{
    constexpr int J = DP / 32, PER = J / GROUPS;
#pragma unroll
    for (int j = 0; j < J; j++) w[j] = *reinterpret_cast<const uint4 *>(row + (4 * j + t) * 16);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < J; j++)
        most = __vmaxu2(__vmaxu2(__vmaxu2(w[j].x & 0x7FFF7FFFu, w[j].y & 0x7FFF7FFFu), __vmaxu2(w[j].z & 0x7FFF7FFFu, w[j].w & 0x7FFF7FFFu)), most);
    most = max(most & 0xFFFFu, most >> 16);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // e: FP32's exponent of the largest, of zero the least; elements times 2^(14 - e).  (Infinity and NaN stay what they are; of rows below 2^-100 nothing is lost that FP32 shows.)
    const float size = Half<T>::unpack(most).x;
    const int e = min(max((int)(__float_as_uint(size) >> 23), 27), 254);
    const float by = __uint_as_float((uint32_t)(268 - e) << 23);
    f = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
    for (int j = 0; j < J; j++) {
        uint32_t *const x = reinterpret_cast<uint32_t *>(&w[j]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 v = Half<T>::unpack(x[i]);
            x[i] = Half<__half>::pack(v.x * by, v.y * by);
        }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        float s = 0.f;
#pragma unroll
        for (int j = g * PER; j < (g + 1) * PER; j++) {
            const uint32_t *const x = reinterpret_cast<const uint32_t *>(&w[j]);
#pragma unroll
            for (int i = 0; i < 4; i++) { const float2 v = Half<__half>::unpack(x[i]); s += v.x + v.y; }
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        sums[g] = s;
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
        w[j] = as_codes_lie(w[j]);
        // what meets codes 2^-18 is a sixteenth
        const __half2 sixteenth = __float2half2_rn(0.0625f), y = __hmul2(*reinterpret_cast<const __half2 *>(&w[j].y), sixteenth), z = __hmul2(*reinterpret_cast<const __half2 *>(&w[j].w), sixteenth);
        w[j].y = *reinterpret_cast<const uint32_t *>(&y);
        w[j].w = *reinterpret_cast<const uint32_t *>(&z);
    }
}

template <class T, int DP, int NT, bool GROUPED, bool CLUSTER>
__global__ void __launch_bounds__(kAttnThreads, QuantisedShape<DP, NT, GROUPED>::kPerSm)
paged_attention_quantised_kernel(const __grid_constant__ QuantisedAttentionArgs args)
{
    using Shape = QuantisedShape<DP, NT, GROUPED>;
    // p vs in FP16 is off by up to 2^-11: as much as an FP16 output's rounding, and enough to round one BF16 output in twelve otherwise.  So the rest goes in too.
    constexpr int kParts = 2;
    constexpr int S = Shape::kStages, J = DP / 32, G = Shape::kGroups, CH = DP / 64, HALF = DP / 32 % 2;      // pieces of 32 elements, groups, chunks of 64 and a half one
    // The tensor core cuts its sums towards zero: where registers allow it they are of 32 keys, and FP32 adds them up.
    constexpr bool APART = NT == 1;
    constexpr int TILES = NT * DP <= 128 ? 2 : 1;                              // of 16 keys that are worked on together, as registers allow
    // Scales and zeros of values times kSmall, so that FP32 holds their sums with weights of up to 2^kSlack; what weights, and weights times scales in FP16, stay below
    constexpr float kSmall = std::is_same<T, __half>::value ? 1.f : 0x1p-16f, kMostWeight = 128.f, kMostProduct = 32768.f;
    static_assert(kSlack == 7.f, "log2 of kMostWeight");
    constexpr uint32_t kAll = 0xffffffffu, kHere = TILES == 2 ? kAll : 0xFFFFu;
    extern __shared__ __align__(128) unsigned char smem[];
    const AttentionArgs &a = args.a;
    const auto &d = a.d;
    const auto &c = args.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t4 = lane & 3, D = (int)d.head_dim;
    unsigned char *const ring = smem + warp * (S * Shape::kStage);
    unsigned char *const q_ring = smem + kAttnWarps * S * Shape::kStage;
    unsigned char *const operands = q_ring + S * Shape::kQ;                    // (of queries that do not stay in registers) [NT][J][32] x 16 bytes
    float2 *const sums = reinterpret_cast<float2 *>(operands + Shape::kOperands);
    const int inners = (int)d.kv_heads * a.groups, cta = blockIdx.x;
    float2 *const arrived_sums = reinterpret_cast<float2 *>(smem + (Shape::kBytes + 15) / 16 * 16);           // [ranks][rows]
    float4 *const arrived = reinterpret_cast<float4 *>(arrived_sums + Shape::kMostRanks * NT * 8);            // [ranks][this CTA's share]

    if constexpr (CLUSTER) cluster_arrive();
    auto others_started = [&]() { if constexpr (CLUSTER) { __syncwarp(); cluster_wait(); } };         // before anything is sent to them, once the first copies are under way
    griddep_wait();
    griddep_launch();

    [[maybe_unused]] long long per = 0, item_at = 0;                           // costs of a CTA; cost number of the item's first cost
    [[maybe_unused]] const int rank = CLUSTER ? (int)cluster_ctarank() : 0, ranks = CLUSTER ? (int)cluster_nctarank() : 1;
    Walk<kQUnitKeys> now = first_unit<kQUnitKeys, CLUSTER>(d, inners, a.ctas, rank, ranks, per, item_at);     // the unit that is computed
    if (now.left <= 0) {                         // (a share of one cost may be that of an item's start alone)
        others_started();
        if (!CLUSTER && tid == 0) a.cut[cta] = make_int4(0, 0, 0, 0);
    } else {
        // A CTA goes through its units in runs: those of one item that follow one another (in a cluster, every `ranks`-th of the item's)
        const int stride = CLUSTER ? ranks * kQUnitKeys : kQUnitKeys;
        auto run_of = [&](const Walk<kQUnitKeys> &w) {
            const int units = w.s.units - w.unit;
            return CLUSTER ? (units + ranks - 1) / ranks : w.left < units ? (int)w.left : units;
        };
        auto next_item = [&](Walk<kQUnitKeys> &w, int run) {                   // behind a run; false where there is none
            if (CLUSTER || w.unit + run < w.s.units) return false;
            w.left -= run + 1;
            if (w.left < 1) return false;
            w.unit = 0;
            if (++w.inner == inners) {
                w.inner = 0;
                do w.b++, w.s = w.b < d.batch ? span_of<kQUnitKeys>(d, w.b) : Span{0, 0, 1, 0}; while (w.s.units == 0);
            }
            return true;
        };
        // What the copies of a unit need; a lane has a key of the warp's 32, and looks its page up well ahead of its use
        struct Ticket { int b, inner, page, place; bool valid, queries; };
        Walk<kQUnitKeys> ahead = now;            // the run that the next ticket is of; what is left of it, this lane's next key, and the end of the keys
        bool more_tickets = true, first_of_run = true;
        int ahead_run = run_of(ahead), ahead_left = ahead_run, key = ahead.s.from + ahead.unit * kQUnitKeys + warp * kQWarpKeys + lane, end = ahead.s.n;
        const int32_t *pages = d.block_table + ahead.s.row * d.table_stride;
        auto ticket = [&]() {
            Ticket t = {(int)ahead.b, ahead.inner, -1, 0, more_tickets, first_of_run};
            if (more_tickets) {
                if (key < end) {
                    const int col = (int)a.by_page.quotient((uint32_t)key);
                    t.place = key - col * (int)d.page_size;
                    t.page = pages[col];
                }
                first_of_run = false;
                key += stride;
                if (--ahead_left == 0) {
                    more_tickets = next_item(ahead, ahead_run);
                    if (more_tickets) {
                        first_of_run = true;
                        ahead_run = ahead_left = run_of(ahead);
                        key = ahead.s.from + warp * kQWarpKeys + lane;
                        end = ahead.s.n;
                        pages = d.block_table + ahead.s.row * d.table_stride;
                    }
                }
            }
            return t;
        };
        int fresh_q = 0;                         // items issued so far: place in the ring of queries
        int inner_at = -1, head = 0, group = 0;  // the head group that is copied, and its head's first codes and scales
        const unsigned char *k = nullptr, *v = nullptr;
        const uint32_t *ks = nullptr, *vs = nullptr;
        const bool alike = c.k_page_stride == c.v_page_stride && c.k_slot_stride == c.v_slot_stride;
        const bool alike_s = c.ks_page_stride == c.vs_page_stride && c.ks_slot_stride == c.vs_slot_stride;
        auto issue = [&](const Ticket &t, int stage) {                         // -> which of the warp's keys are there
            uint32_t ok = 0;
            if (t.valid) {
                if (t.inner != inner_at) {
                    inner_at = t.inner;
                    head = t.inner / a.groups;
                    group = t.inner - head * a.groups;
                    k = (const unsigned char *)c.k + head * c.k_head_stride;
                    v = (const unsigned char *)c.v + head * c.v_head_stride;
                    ks = (const uint32_t *)c.k_scales + head * c.ks_head_stride;
                    vs = (const uint32_t *)c.v_scales + head * c.vs_head_stride;
                }
                const bool is_there = t.page >= 0 && t.page < d.pages;
                const uint32_t page = is_there ? t.page : 0, place = is_there ? t.place : 0;
                ok = __ballot_sync(kAll, is_there);
                const uint32_t dst = shared_addr(ring + stage * Shape::kStage);
                auto copy_scales = [&](const uint32_t *k_from, const uint32_t *v_from) {
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        copy4_async(dst + 2 * Shape::kCodes + lane * G * 8 + g * 8, k_from + g, is_there);
                        copy4_async(dst + 2 * Shape::kCodes + lane * G * 8 + g * 8 + 4, v_from + g, is_there);
                    }
                };
                // a lane's own key's place in the caches; the lanes that copy a row get it from there
                if (args.wide) {                 // in pieces of 16 bytes, and in scales with their zeros, which 32 bits number
                    const uint32_t ks_mine = page * args.ks_page + place * args.ks_slot, vs_mine = alike_s ? ks_mine : page * args.vs_page + place * args.vs_slot;
                    copy_scales(ks + ks_mine, vs + vs_mine);
                    const uint32_t k_mine = page * args.k_page + place * args.k_slot, v_mine = alike ? k_mine : page * args.v_page + place * args.v_slot;
#pragma unroll
                    for (int i = 0; i < Shape::kPieces; i++) {
                        const int at = i * 32 + lane, row = at / Shape::kPieces, piece = at % Shape::kPieces;
                        const uint32_t k_at = __shfl_sync(kAll, k_mine, row), v_at = alike ? k_at : __shfl_sync(kAll, v_mine, row);
                        const bool on = (ok >> row & 1) && piece * 32 < D;     // (else zeros; the address is that of the first page)
                        const int e = piece * 32 < D ? piece * 16 : 0;
                        copy16_async(dst + row * Shape::kPitch + piece * 16, k + e + (uint64_t)k_at * 16, on);
                        copy16_async(dst + Shape::kCodes + row * Shape::kPitch + piece * 16, v + e + (uint64_t)v_at * 16, on);
                    }
                } else {
                    copy_scales(ks + page * c.ks_page_stride + place * c.ks_slot_stride, vs + page * c.vs_page_stride + place * c.vs_slot_stride);
                    const int64_t k_mine = page * c.k_page_stride + place * c.k_slot_stride, v_mine = page * c.v_page_stride + place * c.v_slot_stride;
                    for (int at = lane; at < kQWarpKeys * (DP / 8); at += 32) {
                        const int row = at / (DP / 8), word = at % (DP / 8);
                        const int64_t k_at = __shfl_sync(kAll, k_mine, row), v_at = __shfl_sync(kAll, v_mine, row);
                        const bool on = (ok >> row & 1) && word * 8 < D;
                        const int e = word * 8 < D ? word * 4 : 0;
                        copy4_async(dst + row * Shape::kPitch + word * 4, k + k_at + e, on);
                        copy4_async(dst + Shape::kCodes + row * Shape::kPitch + word * 4, v + v_at + e, on);
                    }
                }
                if (t.queries) {                                               // its queries, a quarter per warp
                    const uint32_t qdst = shared_addr(q_ring + fresh_q * Shape::kQ);
                    const int h0 = head * (int)(d.q_heads / d.kv_heads) + group * a.per_group;
                    const int heads = min(a.per_group, (int)(d.q_heads / d.kv_heads) - group * a.per_group);
                    for (int at = tid; at < NT * DP; at += kAttnThreads) {
                        const int row = at / (DP / 8), chunk = at % (DP / 8);
                        const bool on = row < heads && chunk * 8 < D;
                        copy16_async(qdst + row * Shape::kQPitch + chunk * 16, (const T *)d.q + (int64_t)t.b * d.q_token_stride + (on ? (h0 + row) * d.q_head_stride + chunk * 8 : 0), on);
                    }
                    if (++fresh_q == S) fresh_q = 0;
                }
            }
            copy_commit();
            return ok;
        };
        Ticket pending;
        uint32_t oks[S - 1];                     // of the units that are under way
        {
            Ticket first[S - 1];
#pragma unroll
            for (int i = 0; i < S - 1; i++) first[i] = ticket();
            pending = ticket();
#pragma unroll
            for (int i = 0; i < S - 1; i++) oks[i] = issue(first[i], i);
        }
        others_started();

        uint4 q[Shape::kKeepQ ? NT : 1][Shape::kKeepQ ? J : 1];
        // of queries 2 (lane % 4) and the next: scale, power of two and log2 e; sums of elements.  Scores are in units of the codes' 2^-22 up to `factor`: FP32 holds them for keys of any size.
        float factor[NT][2], q_sum[NT][G][2];
        float o[2 * J][NT][4], sum[NT][2], zeros[NT][G][2];
        float base[NT][2];                       // what is taken off scores: the largest by the time, which weighs exactly one; kNone before the first
        float down[NT][2];                       // a power of two that brings the item's largest weight times scale by the time to 2^7 .. 2^15
        int stage = 0, q_at = -1;
        for (bool more = true; more;) {
            const bool started_here = now.unit == 0;                             // the item's first unit is this CTA's
            const int run = run_of(now);
            for (int u = 0; u < run; u++) {
                copy_wait<S - 2>();
                __syncwarp();
                if (u == 0) {
                    if (++q_at == S) q_at = 0;
                    __syncthreads();                 // every warp's part of the queries is there, and the sums of the item before are read
                    const unsigned char *const src = q_ring + q_at * Shape::kQ + r * Shape::kQPitch;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        uint4 w[J];
                        float f, s[G];
                        query_operands<T, DP, G>(src + t * 8 * Shape::kQPitch, t4, w, f, s);
                        if constexpr (Shape::kKeepQ) {
#pragma unroll
                            for (int j = 0; j < J; j++) q[t][j] = w[j];
                        } else if (t % kAttnWarps == warp) {
#pragma unroll
                            for (int j = 0; j < J; j++) reinterpret_cast<uint4 *>(operands)[(t * J + j) * 32 + lane] = w[j];
                        }
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            factor[t][e] = __shfl_sync(kAll, f, t4 * 8 + e * 4) * (a.scale_log2 * 0x1p22f);
#pragma unroll
                            for (int g = 0; g < G; g++) q_sum[t][g][e] = __shfl_sync(kAll, s[g], t4 * 8 + e * 4) * 0x1p-22f;
                        }
                        base[t][0] = base[t][1] = kNone;
                        down[t][0] = down[t][1] = 1.f;
                        sum[t][0] = sum[t][1] = 0.f;
#pragma unroll
                        for (int g = 0; g < G; g++) zeros[t][g][0] = zeros[t][g][1] = 0.f;
#pragma unroll
                        for (int i = 0; i < 2 * J; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[i][t][e] = 0.f;
                    }
                    if constexpr (!Shape::kKeepQ) __syncthreads();
                }
                const uint32_t ok = oks[0];
                const unsigned char *const keys = ring + stage * Shape::kStage, *const values = keys + Shape::kCodes, *const scales = values + Shape::kCodes;
#pragma unroll
                for (int i = 0; i + 1 < S - 1; i++) oks[i] = oks[i + 1];
                oks[S - 2] = issue(pending, stage == 0 ? S - 1 : stage - 1);
                pending = ticket();
#pragma unroll
                for (int h0 = 0; h0 < 2; h0 += TILES) {
                    const uint32_t there = ok >> (16 * h0) & kHere;
                    if (!there) continue;
                    // ---- scores of a tile of 16 keys, or of two: rows (keys) r and r + 8 of a tile, columns (queries) 2 t4 and the next
                    float s[TILES][NT][4];
                    float2 kv[TILES][2][G][2];           // scales and zeros: of key r or r + 8 of a tile, of the key and of the value
#pragma unroll
                    for (int h = 0; h < TILES; h++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int g = 0; g < G; g++) {
                                const uint2 w = *reinterpret_cast<const uint2 *>(scales + ((16 * (h0 + h) + 8 * i + r) * G + g) * 8);
                                kv[h][i][g][0] = Half<T>::unpack(w.x);
                                kv[h][i][g][1] = Half<T>::unpack(w.y);
                            }
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        float x[TILES][NT][4];
#pragma unroll
                        for (int h = 0; h < TILES; h++)
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int e = 0; e < 4; e++) x[h][t][e] = q_sum[t][g][e & 1] * -8.f;           // (8 off every code)
#pragma unroll
                        for (int j = g * (J / G); j < (g + 1) * (J / G); j++) {
#pragma unroll
                            for (int h = 0; h < TILES; h++) {
                                const unsigned char *const at = keys + (16 * (h0 + h) + r) * Shape::kPitch + t4 * 4 + j * 16;
                                const uint32_t w0 = word_at(at), w1 = word_at(at + 8 * Shape::kPitch);
                                const uint32_t lower[4] = {codes<0>(w0), codes<0>(w1), codes<1>(w0), codes<1>(w1)};
                                const uint32_t upper[4] = {codes<2>(w0), codes<2>(w1), codes<3>(w0), codes<3>(w1)};
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    uint4 b;
                                    if constexpr (Shape::kKeepQ) b = q[t][j];
                                    else b = reinterpret_cast<const uint4 *>(operands)[(t * J + j) * 32 + lane];
                                    Half<__half>::mma(x[h][t], lower, b.x, b.y);
                                    Half<__half>::mma(x[h][t], upper, b.z, b.w);
                                }
                            }
                        }
#pragma unroll
                        for (int h = 0; h < TILES; h++) {
                            const float2 a0 = kv[h][0][g][0], a1 = kv[h][1][g][0];
                            const float z0 = mul_add(8.f, a0.x, a0.y), z1 = mul_add(8.f, a1.x, a1.y);
#pragma unroll
                            for (int t = 0; t < NT; t++)
#pragma unroll
                                for (int e = 0; e < 2; e++) {
                                    s[h][t][e] = mul_add(a0.x, x[h][t][e], mul_add(z0, q_sum[t][g][e], g ? s[h][t][e] : 0.f));
                                    s[h][t][e + 2] = mul_add(a1.x, x[h][t][e + 2], mul_add(z1, q_sum[t][g][e], g ? s[h][t][e + 2] : 0.f));
                                }
                        }
                    }
                    // Weights relative to the reference, which moves where one is kSlack above it (and at the first number: kNone lies far below).  A weight times the value's scale has a
                    // reference of its own, because the products take it in FP16: what counts is how large it is beside the item's other keys.
                    float p[TILES][NT][4], most_scale = 0.f;
                    bool grows = false;
                    auto value_scale = [&](int h, int i) {
                        float m = fabsf(kv[h][i][0][1].x);
#pragma unroll
                        for (int g = 1; g < G; g++) m = fmaxf(m, fabsf(kv[h][i][g][1].x));
                        return m;
                    };
#pragma unroll
                    for (int h = 0; h < TILES; h++) most_scale = fmaxf(most_scale, fmaxf(value_scale(h, 0), value_scale(h, 1)));
                    most_scale *= kSmall;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
#pragma unroll
                        for (int h = 0; h < TILES; h++)
#pragma unroll
                            for (int e = 0; e < 4; e++) p[h][t][e] = mul_add(s[h][t][e], factor[t][e & 1], -base[t][e & 1]);
#pragma unroll
                        if (there != kHere) {        // keys that are not there
#pragma unroll
                            for (int h = 0; h < TILES; h++) {
                                const bool on0 = (there >> (16 * h + r)) & 1, on1 = (there >> (16 * h + r + 8)) & 1;
#pragma unroll
                                for (int e = 0; e < 4; e++) p[h][t][e] = (e < 2 ? on0 : on1) ? p[h][t][e] : -INFINITY;
                            }
                        }
#pragma unroll
                        for (int h = 0; h < TILES; h++)
#pragma unroll
                            for (int e = 0; e < 4; e++) p[h][t][e] = exp2_approx(p[h][t][e]);
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float m = fmaxf(p[0][t][e], p[0][t][e + 2]);
                            if constexpr (TILES == 2) m = fmaxf(m, fmaxf(p[TILES - 1][t][e], p[TILES - 1][t][e + 2]));
                            grows = grows || m > kMostWeight || m * down[t][e] * most_scale > kMostProduct;
                        }
                    }
                    if (__any_sync(kAll, grows)) {
                        auto over_rows = [](float m) {
                            m = fmaxf(m, __shfl_xor_sync(kAll, m, 4));
                            m = fmaxf(m, __shfl_xor_sync(kAll, m, 8));
                            return fmaxf(m, __shfl_xor_sync(kAll, m, 16));
                        };
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            float keep[2];
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                float m = -INFINITY;
                                auto score = [&](int h, int i) { return (there >> (16 * h + r + 8 * i)) & 1 ? mul_add(s[h][t][e + 2 * i], factor[t][e], 0.f) : -INFINITY; };
#pragma unroll
                                for (int h = 0; h < TILES; h++) m = fmaxf(m, fmaxf(score(h, 0), score(h, 1)));
                                m = over_rows(m);
                                keep[e] = 1.f;
                                if (m > base[t][e]) {
                                    keep[e] = exp2_approx(base[t][e] - m);
                                    base[t][e] = m;
                                }
                                m = 0.f;
#pragma unroll
                                for (int h = 0; h < TILES; h++)
#pragma unroll
                                    for (int i = 0; i < 2; i++) {
                                        p[h][t][e + 2 * i] = exp2_approx(score(h, i) - base[t][e]);
                                        m = fmaxf(m, p[h][t][e + 2 * i] * (value_scale(h, i) * kSmall));
                                    }
                                sum[t][e] *= keep[e];
#pragma unroll
                                for (int g = 0; g < G; g++) zeros[t][g][e] *= keep[e];
                                // the power of two at or above the largest weight times scale, between 2^-100 and 2^126: this goes to 2^8
                                keep[e] *= two_to_8_over(down[t][e]);
                                const uint32_t up = (__float_as_uint(fmaxf(over_rows(m), keep[e])) + 0x7FFFFFu) & 0x7F800000u;
                                down[t][e] = two_to_8_over(__uint_as_float(min(max(up, 27u << 23), 253u << 23)));
                                keep[e] *= down[t][e] * (1.f / 256.f);
                            }
#pragma unroll
                            for (int i = 0; i < 2 * J; i++) {
                                o[i][t][0] *= keep[0]; o[i][t][1] *= keep[1]; o[i][t][2] *= keep[0]; o[i][t][3] *= keep[1];
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < TILES; h++)
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int e = 0; e < 2; e++) sum[t][e] += p[h][t][e] + p[h][t][e + 2];
                    // ---- values: a lane's pairs of keys are 2 t4 and 2 t4 + 8 of a tile with the next ones each; it has the elements 8 r to 8 r + 7 of a chunk of 64
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        uint32_t hi[TILES][NT][2], lo[TILES][NT][2];
#pragma unroll
                        for (int h = 0; h < TILES; h++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const float f = kv[h][i][g][1].x * kSmall, z = kv[h][i][g][1].y * kSmall + 8.f * f;
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    const float p0 = p[h][t][2 * i], p1 = p[h][t][2 * i + 1], y0 = p0 * down[t][0] * f, y1 = p1 * down[t][1] * f;
                                    zeros[t][g][0] += p0 * z;
                                    zeros[t][g][1] += p1 * z;
                                    const uint32_t up = pack_half2(y0, y1);
                                    hi[h][t][i] = transpose8x8(up);
                                    const float2 w = Half<__half>::unpack(up);
                                    lo[h][t][i] = transpose8x8(pack_half2(y0 - w.x, y1 - w.y));
                                }
                            }
                        // Two tiles of 16 elements, from four codes each of a pair of keys and of the pair 8 behind; those of tile h from pair(h, x, y)
                        auto products = [&](int at, auto pair) {
                            float sums[2][NT][4];
#pragma unroll
                            for (int h = 0; h < TILES; h++) {
                                uint32_t x, y;
                                pair(h, x, y);
                                const uint32_t w[2][4] = {{centred_codes<0>(x), centred_codes<1>(x), centred_codes<0>(y), centred_codes<1>(y)},
                                                          {centred_codes<2>(x), centred_codes<3>(x), centred_codes<2>(y), centred_codes<3>(y)}};
#pragma unroll
                                for (int part = 0; part < kParts; part++)
#pragma unroll
                                    for (int i = 0; i < 2; i++)
#pragma unroll
                                        for (int t = 0; t < NT; t++) {
                                            if (APART && h == 0 && part == 0) { sums[i][t][0] = sums[i][t][1] = sums[i][t][2] = sums[i][t][3] = 0.f; }
                                            Half<__half>::mma(!APART ? o[at + i][t] : sums[i][t], w[i], part ? lo[h][t][0] : hi[h][t][0], part ? lo[h][t][1] : hi[h][t][1]);
                                        }
                            }
                            if (APART) {
#pragma unroll
                                for (int i = 0; i < 2; i++)
#pragma unroll
                                    for (int t = 0; t < NT; t++)
#pragma unroll
                                        for (int e = 0; e < 4; e++) o[at + i][t][e] += sums[i][t][e];
                            }
                        };
#pragma unroll
                        for (int ch = GROUPED ? g : 0; ch < (GROUPED ? g + 1 : CH); ch++) {
                            uint32_t w[TILES][4];
#pragma unroll
                            for (int h = 0; h < TILES; h++) {
                                const unsigned char *const at = values + (16 * (h0 + h) + 2 * t4) * Shape::kPitch + r * 4 + ch * 32;
                                w[h][0] = word_at(at); w[h][1] = word_at(at + Shape::kPitch); w[h][2] = word_at(at + 8 * Shape::kPitch); w[h][3] = word_at(at + 9 * Shape::kPitch);
                            }
#pragma unroll
                            for (int half = 0; half < 2; half++)
                                products(4 * ch + 2 * half, [&](int h, uint32_t &x, uint32_t &y) {
                                    x = __byte_perm(w[h][0], w[h][1], half ? 0x7632 : 0x5410);
                                    y = __byte_perm(w[h][2], w[h][3], half ? 0x7632 : 0x5410);
                                });
                        }
                        if constexpr (HALF) {        // the last 32 elements: 4 r to 4 r + 3
                            products(4 * CH, [&](int h, uint32_t &x, uint32_t &y) {
                                const unsigned char *const at = values + (16 * (h0 + h) + 2 * t4) * Shape::kPitch + CH * 32 + (r >> 1) * 4;
                                const uint32_t half = r & 1 ? 0x7632 : 0x5410;
                                x = __byte_perm(word_at(at), word_at(at + Shape::kPitch), half);
                                y = __byte_perm(word_at(at + 8 * Shape::kPitch), word_at(at + 9 * Shape::kPitch), half);
                            });
                        }
                    }
                }
                if (++stage == S) stage = 0;
            }
            const bool last = now.unit + run == now.s.units;
            // ---- the four warps' sums over their keys of this item become one.  They pass through the stage that was just used: its next copies are
            // issued behind the barrier above.  What `down` has made of the sums is undone here.
            const int head = now.inner / a.groups, group = now.inner - head * a.groups;
            const int64_t h0 = head * (d.q_heads / d.kv_heads) + group * a.per_group;
            const int heads = min(a.per_group, (int)(d.q_heads / d.kv_heads) - group * a.per_group);
            const bool whole = started_here && last;
            const int64_t slot = 2 * (int64_t)cta + (started_here ? 1 : 0);
            auto over_keys = [](float x) {
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                return x + __shfl_xor_sync(0xffffffffu, x, 16);
            };
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float l = over_keys(sum[t][e]);
                    if (lane < 4) sums[warp * NT * 8 + t * 8 + 2 * lane + e] = make_float2(base[t][e] == kNone ? -INFINITY : base[t][e] + AttnType<T>::lift, l);
#pragma unroll
                    for (int g = 0; g < G; g++) zeros[t][g][e] = over_keys(zeros[t][g][e]) * (1.f / kSmall);
                }
            const int used = stage == 0 ? S - 1 : stage - 1;
            float *const fold = reinterpret_cast<float *>(ring + used * Shape::kStage) + 2 * t4 * Shape::kFoldPitch;
            const float *const folds = reinterpret_cast<const float *>(smem + used * Shape::kStage);
            constexpr int WARP_FLOATS = S * Shape::kStage / 4;
            constexpr float kUp = 0x1p9f / kSmall;                                              // (of the codes' unit)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                __syncwarp();                // the warp has read its values
                if (t) __syncthreads();
#pragma unroll
                for (int i = 0; i < 2 * J; i++) {
                    const int el = i < 4 * CH ? (i / 4) * 64 + 8 * r + 2 * (i % 4) : CH * 64 + 4 * r + 2 * (i % 4);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float z = zeros[t][GROUPED ? i / 4 : 0][e], times = two_to_8_over(down[t][e]) * (1.f / 256.f);
                        *reinterpret_cast<float2 *>(fold + e * Shape::kFoldPitch + el) = make_float2(o[i][t][e] * kUp * times + z, o[i][t][e + 2] * kUp * times + z);
                    }
                }
                __syncthreads();
                add_warps<T, DP, NT, CLUSTER, WARP_FLOATS, Shape::kFoldPitch>(a, folds, sums, t, now.b, h0, heads, whole, slot, rank, ranks, arrived_sums, arrived);
            }
            const Walk<kQUnitKeys> was = now;
            more = next_item(now, run);
            if constexpr (!CLUSTER) {
                if (!more && tid == 0) a.cut[cta] = make_int4((int)was.b, was.inner, (int)((item_at + was.s.units) / per), started_here && !last ? 1 : 0);
                item_at += was.s.units + 1;
            }
        }
        copy_wait<0>();
    }
    if constexpr (CLUSTER) {
        // ---- the cluster's sums become one, a share of the elements in each CTA
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
    empty_rows<T, kQUnitKeys>(d);
}

// ---- host: which variant, how much workspace -----------------------------------------------------------------
template <class T> int launch_attention_quantised(const QuantisedAttentionArgs &a, const AttnPlan &p, bool grouped, cudaStream_t stream);

template <class T, int DP, int NT, bool GROUPED>
int launch_attention_quantised_as(const QuantisedAttentionArgs &a, const AttnPlan &p, cudaStream_t stream)
{
    using Shape = QuantisedShape<DP, NT, GROUPED>;
    const int dev = current_device_index();
    if (dev < 0) return ORTHO_B200_ERR_CUDA;
    static bool attr_set[kMaxDevices] = {};
    if (!attr_set[dev]) {
        OB_CUDA(cudaFuncSetAttribute(paged_attention_quantised_kernel<T, DP, NT, GROUPED, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes));
        if constexpr (Shape::kClusterPerSm > 0)
            OB_CUDA(cudaFuncSetAttribute(paged_attention_quantised_kernel<T, DP, NT, GROUPED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kClusterBytes));
        attr_set[dev] = true;
    }
    if constexpr (Shape::kClusterPerSm > 0) {
        if (p.cluster) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)a.a.ctas); cfg.blockDim = dim3(kAttnThreads); cfg.dynamicSmemBytes = Shape::kClusterBytes; cfg.stream = stream;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = (unsigned)p.cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
            cfg.attrs = attr; cfg.numAttrs = 2;
            OB_CUDA(cudaLaunchKernelEx(&cfg, paged_attention_quantised_kernel<T, DP, NT, GROUPED, true>, a));
            count_launch();
            return ORTHO_B200_OK;
        }
    }
    const int st = launch_dependent(paged_attention_quantised_kernel<T, DP, NT, GROUPED, false>, dim3((unsigned)a.a.ctas), kAttnThreads, Shape::kBytes, stream, a);
    if (st) return st;
    return launch_dependent(join_kernel<T>, dim3((unsigned)a.a.ctas, (unsigned)a.a.per_group), 128, 0, stream, a.a, NT * 8);
}

template <class T, int DP, bool GROUPED>
int launch_attention_quantised_dim(const QuantisedAttentionArgs &a, const AttnPlan &p, cudaStream_t stream)
{
    if (p.nt == 1) return launch_attention_quantised_as<T, DP, 1, GROUPED>(a, p, stream);
    if (p.nt == 2) return launch_attention_quantised_as<T, DP, 2, GROUPED>(a, p, stream);
    if constexpr (DP <= 128) return launch_attention_quantised_as<T, DP, 4, GROUPED>(a, p, stream);
    return ORTHO_B200_ERR_SHAPE;
}

#define OB_QUANTISED_DIMS(X) X(64) X(96) X(128) X(192) X(256)

template <class T>
int launch_attention_quantised(const QuantisedAttentionArgs &a, const AttnPlan &p, bool grouped, cudaStream_t stream)
{
#define OB_CASE(DP)                                                                                              \
    if (p.dp == DP) {                                                                                            \
        if constexpr (DP % kQuantGroup == 0 && DP > kQuantGroup)                                                 \
            if (grouped) return launch_attention_quantised_dim<T, DP, true>(a, p, stream);                       \
        return launch_attention_quantised_dim<T, DP, false>(a, p, stream);                                       \
    }
    OB_QUANTISED_DIMS(OB_CASE)
#undef OB_CASE
    return ORTHO_B200_ERR_SHAPE;
}

}  // namespace ob
