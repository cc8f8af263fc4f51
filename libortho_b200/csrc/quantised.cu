// Keys and values quantised to 4 bits as they are written to the paged cache, and a cache read back (quantised.cuh, include/ortho_b200.h: the format).
//
//     zero = round16(min x),  scale = round16((max x - min x) / 15),  code = clamp(rint((x - zero) / scale), 0, 15)      over a group of a head
//
// Rounding to 4 bits turns a difference in the last place of FP32 into a whole step wherever x lies next to a border, so the codes are those of exact
// arithmetic: FP32 does the work and knows its own error, and what lies within that of a border is taken again from the raw values: ties of values, which FP32 decides exactly
// (one BF16 value in 500), the rest in FP64 (a key in some 40000; the least or largest of an FP16 group in some 300).  A turned key is a c - b s of an 11-bit and a 24-bit factor
// each, exact in FP64 up to its last sum.
// Bound by instructions, not by HBM: some 450 for four heads of 128 elements in a warp.  4096 tokens of 32 query, key and value heads of 128 (155 MB): 56 us = 2.8 TB/s,
// of which queries and the copies alone take 28; 64 tokens of 64 + 2 x 8: 3.9 us, launch and the chain slot, position, angle, heads.  Tried (us, the same 4096 tokens):
// two items of a thread 75 (registers), rows ahead in registers instead of shared memory 75, all of an unsure head in FP64 64 (and 64 tokens 6.0).

#include "quantised.cuh"
#include "rotary.cuh"

namespace ob {

constexpr int kMostTogether = 4;                 // tokens of a CTA

struct QuantiseArgs {
    ortho_b200_rotary_append_desc d;
    ortho_b200_quantised_cache c;
    int turned, lanes_log2, together;            // items (two vectors) of a head that turn; lanes of a head, a power of two; tokens of a CTA
    FastDiv by_half;
};

template <class T> struct QuantType;
template <> struct QuantType<__half> {
    static constexpr float safe = 30000.f;                                     // below: neither a value nor zero + 15 scale comes near the type's end, nor a quotient FP32's
    static constexpr double beyond = 65520.0;                                  // rounds to infinity
    static __device__ __forceinline__ __half from_double(double v) { return __double2half(v); }
};
template <> struct QuantType<__nv_bfloat16> {
    static constexpr float safe = 1e28f;
    static constexpr double beyond = 3.3961775292304957e38;
    static __device__ __forceinline__ __nv_bfloat16 from_double(double v) { return __double2bfloat16(v); }
};
template <class T> __device__ __forceinline__ uint32_t bits16(T v) { return *reinterpret_cast<const uint16_t *>(&v); }

// Least and largest, NaN where one is
__device__ __forceinline__ float least_of(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float most_of(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float least_of(float a, float b, float c) { float r; asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float most_of(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// A group's scale and zero; `bits`: as they are stored.  A group that stands for NaN has scale 0 here, so that its codes come out as 0.
struct Held { float s, z; uint32_t bits; };
constexpr uint32_t kNoNumber = 0x7FFFu;

// From the least and largest of values that are each off by up to `tol` and are all below QuantType::safe; false where that could change a bit
template <class T>
__device__ __forceinline__ bool held_of(float lo, float hi, float tol, Held &h)
{
    const float q = (hi - lo) * (1.f / 15.f), tq = tol * (2.f / 15.f) + q * 0x1p-21f;
    h.bits = Half<T>::pack(q, lo);
    const float2 f = Half<T>::unpack(h.bits);
    h.s = f.x;
    h.z = f.y;
    return Half<T>::pack(q - tq, lo - tol) == Half<T>::pack(q + tq, lo + tol) && (q > 1e-28f || (lo == hi && tol == 0.f));
}
template <class T>
__device__ __forceinline__ Held held_of(double lo, double hi)
{
    Held h = {0.f, 0.f, kNoNumber};
    if (!(fabs(lo) < QuantType<T>::beyond && fabs(hi) < QuantType<T>::beyond)) return h;       // (NaN too)
    const T z = QuantType<T>::from_double(lo);
    T s = QuantType<T>::from_double((hi - lo) / 15.0);
    h.z = Half<T>::to_float(z);
    h.s = Half<T>::to_float(s);
    if (!((double)h.z + 15.0 * (double)h.s < QuantType<T>::beyond)) {
        const uint16_t below = (uint16_t)(bits16(s) - 1);
        s = *reinterpret_cast<const T *>(&below);
        h.s = Half<T>::to_float(s);
    }
    h.bits = bits16(s) | bits16(z) << 16;
    return h;
}

// Bytes from global to a thread's own place in shared memory
template <int BYTES> __device__ __forceinline__ void copy_own(uint32_t dst, const void *src)
{
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

constexpr int kAhead = 4;                   // rows of a thread that are under way

// A row is a head of a token; a warp has 32 / L of them at a time, L lanes each, a lane two vectors of VEC values.  The rows to come are copied ahead into a place of
// their thread's own in shared memory, so that neither registers nor barriers are spent on them and unsure values are read again from there.
template <class T, int VEC, bool INTERLEAVED, bool GROUPED>
__global__ void __launch_bounds__(256, 3)
quantise_append_kernel(const __grid_constant__ QuantiseArgs a)
{
    constexpr uint32_t kAll = 0xffffffffu;
    extern __shared__ __align__(16) unsigned char smem[];                      // [kAhead][2][256] vectors; [tokens][rotary]: cosines, then sines
    struct Places { unsigned char *to[3]; uint32_t *scales[3]; };              // of a token's queries, keys and values; no place in the cache: NULL
    __shared__ Places places[kMostTogether];
    __shared__ int64_t apart[3][2];              // heads in them: in bytes, in pairs
    float *const angles = reinterpret_cast<float *>(smem + kAhead * 2 * 256 * VEC * 2);
    const auto &d = a.d;
    const auto &c = a.c;
    const int64_t t0 = (int64_t)blockIdx.x * a.together;
    const int tokens = d.tokens - t0 < a.together ? (int)(d.tokens - t0) : a.together;
    const int R = (int)d.rotary, half = R / 2, D = (int)c.head_dim, q_heads = (int)d.q_heads, kv_heads = (int)c.kv_heads, heads = q_heads + 2 * kv_heads;
    const int L = 1 << a.lanes_log2, it = threadIdx.x & (L - 1), seg = (threadIdx.x & 31) >> a.lanes_log2, rows = 256 >> a.lanes_log2, step = (int)gridDim.y * rows;
    const bool turns = it < a.turned;
    int e0, e1;                                  // elements that this thread's vectors start with; -1: none
    if (!turns) { e0 = R + 2 * (it - a.turned) * VEC; e1 = e0 + VEC; }
    else if (INTERLEAVED) { e0 = 2 * it * VEC; e1 = e0 + VEC; }
    else { e0 = it * VEC; e1 = e0 + half; }
    if (e0 >= D) e0 = -1;
    if (e1 >= D) e1 = -1;
    const int groups = (int)c.groups, width = D / groups, g0 = GROUPED ? e0 / kQuantGroup : 0, g1 = GROUPED ? e1 / kQuantGroup : 0;
    // A segment has a head of one token after the other, then its next head; kinds 0 to 2 are queries, keys and values
    const int head0 = (int)blockIdx.y * rows + ((int)threadIdx.x >> 5) * (32 >> a.lanes_log2);                // the warp's first
    auto kind_of = [&](int h, int &own) {
        const int kind = (h >= q_heads) + (h >= q_heads + kv_heads);
        own = h - (kind == 0 ? 0 : kind == 1 ? q_heads : q_heads + kv_heads);
        return kind;
    };
    auto place = [&](int stage, int v) { return smem + ((stage * 2 + v) * 256 + threadIdx.x) * (VEC * 2); };
    int next_head = head0 + seg, next_token = 0;                               // of the row that is copied next
    const T *next = nullptr;
    int64_t next_step = 0;
    auto issue = [&](int stage) {
        if (next_head < heads && e0 >= 0) {
            if (next_token == 0) {
                int own;
                const int kind = kind_of(next_head, own);
                next_step = kind == 0 ? d.q_token_stride : kind == 1 ? d.k_token_stride : d.v_token_stride;
                next = (const T *)(kind == 0 ? d.q : kind == 1 ? d.k : d.v) + t0 * next_step
                     + (uint32_t)own * (kind == 0 ? d.q_head_stride : kind == 1 ? d.k_head_stride : d.v_head_stride);
            }
            copy_own<VEC * 2>(shared_addr(place(stage, 0)), next + e0);
            if (e1 >= 0) copy_own<VEC * 2>(shared_addr(place(stage, 1)), next + e1);
            next += next_step;
        }
        if (++next_token == tokens) { next_token = 0; next_head += step; }
        copy_commit();
    };
    griddep_wait();
    griddep_launch();
#pragma unroll
    for (int i = 0; i < kAhead - 1; i++) issue(i);
    if ((int)threadIdx.x < tokens) {
        const int64_t t = t0 + threadIdx.x, slot = d.slots[t];
        const bool kept = slot >= 0 && slot < c.pages * c.page_size;
        const int64_t page = !kept ? 0 : slot <= 0x7FFFFFFF ? (int64_t)((uint32_t)slot / (uint32_t)c.page_size) : slot / c.page_size, in = slot - page * c.page_size;
        Places &p = places[threadIdx.x];
        p.to[0] = (unsigned char *)((T *)d.q_out + t * d.out_token_stride);
        p.scales[0] = nullptr;
        p.to[1] = kept ? (unsigned char *)c.k + page * c.k_page_stride + in * c.k_slot_stride : nullptr;
        p.to[2] = kept ? (unsigned char *)c.v + page * c.v_page_stride + in * c.v_slot_stride : nullptr;
        p.scales[1] = kept ? (uint32_t *)c.k_scales + page * c.ks_page_stride + in * c.ks_slot_stride : nullptr;
        p.scales[2] = kept ? (uint32_t *)c.v_scales + page * c.vs_page_stride + in * c.vs_slot_stride : nullptr;
    }
    if (threadIdx.x == 0) {
        apart[0][0] = d.out_head_stride * 2;
        apart[1][0] = c.k_head_stride;
        apart[2][0] = c.v_head_stride;
        apart[1][1] = c.ks_head_stride;
        apart[2][1] = c.vs_head_stride;
    }
    angles_of(d, a.by_half, t0, tokens, angles);
    __syncthreads();

    int stage = 0, token = tokens - 1, head = head0 + seg - step, kind = 0;
    int64_t code_at = 0, scale_at = 0;
    // (a warp's segments go round the loop together: they meet in shuffles)
    for (;; stage = stage == kAhead - 1 ? 0 : stage + 1) {
        if (++token == tokens) {
            token = 0;
            head += step;
            if (head - seg >= heads) break;
            int own;
            kind = kind_of(head, own);
            code_at = (uint32_t)own * apart[kind][0];
            scale_at = (uint32_t)own * apart[kind][1];
        }
        issue(stage == 0 ? kAhead - 1 : stage - 1);
        copy_wait<kAhead - 1>();
        const bool mine = head < heads && e0 >= 0, is_value = kind == 2;
        const float *const angle = angles + token * R;
        unsigned char *const base = places[token].to[kind], *const to = base + code_at;
        const bool kept = mine && kind != 0 && base;
        float x[2][VEC];
        {
            Raw<VEC> r;
            r.load(place(stage, 0));
            r.template to<T>(x[0]);
            r.load(place(stage, 1));             // (what lies there, where there is no second vector, is not used)
            r.template to<T>(x[1]);
        }
        if (turns && !is_value) {
            const float *const at = angle + it * VEC;
            float cs[VEC], sn[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const float4 y = *reinterpret_cast<const float4 *>(at + i), z = *reinterpret_cast<const float4 *>(at + half + i);
                cs[i] = y.x; cs[i + 1] = y.y; cs[i + 2] = y.z; cs[i + 3] = y.w;
                sn[i] = z.x; sn[i + 1] = z.y; sn[i + 2] = z.z; sn[i + 3] = z.w;
            }
            if (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i + 1 < VEC; i += 2) {
                    turn_pair(x[0][i], x[0][i + 1], cs[i / 2], sn[i / 2]);
                    turn_pair(x[1][i], x[1][i + 1], cs[(VEC + i) / 2], sn[(VEC + i) / 2]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) turn_pair(x[0][i], x[1][i], cs[i], sn[i]);
            }
        }
        if (mine && kind == 0) {
            T *const dst = (T *)to;
            Raw<VEC> r;
            r.template from<T>(x[0]);
            r.store(dst + e0);
            r.template from<T>(x[1]);
            if (e1 >= 0) r.store(dst + e1);
        }
        if (!__any_sync(kAll, kept)) continue;
        // ---- least and largest value of this thread's vectors, then of their groups, and the largest size in the head
        float lo[2], hi[2], size;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            float l = least_of(x[v][0], x[v][1], x[v][2]), m = most_of(x[v][0], x[v][1], x[v][2]);
#pragma unroll
            for (int i = 3; i + 1 < VEC; i += 2) { l = least_of(l, x[v][i], x[v][i + 1]); m = most_of(m, x[v][i], x[v][i + 1]); }
            const bool some = kept && (v ? e1 : e0) >= 0;
            lo[v] = some ? least_of(l, x[v][VEC - 1]) : INFINITY;
            hi[v] = some ? most_of(m, x[v][VEC - 1]) : -INFINITY;
        }
        auto over_lanes = [&](float &l, float &m) {
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1)
                if (o < L) {
                    l = least_of(l, __shfl_xor_sync(kAll, l, o));
                    m = most_of(m, __shfl_xor_sync(kAll, m, o));
                }
        };
        if constexpr (GROUPED) {
            float own_lo[2] = {lo[0], lo[1]}, own_hi[2] = {hi[0], hi[1]};
            size = 0.f;
            for (int g = 0; g < groups; g++) {
                float l = least_of(g0 == g ? own_lo[0] : INFINITY, g1 == g ? own_lo[1] : INFINITY), m = most_of(g0 == g ? own_hi[0] : -INFINITY, g1 == g ? own_hi[1] : -INFINITY);
                over_lanes(l, m);
                if (g0 == g) { lo[0] = l; hi[0] = m; }
                if (g1 == g) { lo[1] = l; hi[1] = m; }
                size = most_of(size, -l, m);
            }
        } else {
            lo[0] = least_of(lo[0], lo[1]);
            hi[0] = most_of(hi[0], hi[1]);
            over_lanes(lo[0], hi[0]);
            lo[1] = lo[0];
            hi[1] = hi[0];
            size = most_of(-lo[0], hi[0]);
        }
        // A turned value a c - b s is off by at most 2^-24 (|b s| + |x|), and both are at most sqrt(c c + s s) |(a, b)| = |(x, y)| <= 2 size
        const float tol = is_value || R == 0 ? 0.f : 0x1p-22f * size;
        Held held[2];
        bool ends = false, sure = held_of<T>(lo[0], hi[0], tol, held[0]) && size < QuantType<T>::safe;
        if constexpr (GROUPED) sure = held_of<T>(lo[1], hi[1], tol, held[1]) && sure;
        else held[1] = held[0];
        // A value in FP64: of vector v, number i
        auto exact = [&](int v, int i) {
            const T *const raws = reinterpret_cast<const T *>(place(stage, v));
            const double raw = (double)Half<T>::to_float(raws[i]);
            if (!turns || is_value) return raw;
            const double other = (double)Half<T>::to_float(INTERLEAVED ? raws[i ^ 1] : reinterpret_cast<const T *>(place(stage, v ^ 1))[i]);
            const int pair = it * VEC + (INTERLEAVED ? (v * VEC + i) / 2 : i);
            const double co = (double)angle[pair], si = (double)angle[half + pair];
            return (INTERLEAVED ? i & 1 : v) ? raw * co + other * si : raw * co - other * si;
        };
        if (!__all_sync(kAll, sure || !kept)) {  // least and largest values once more in FP64, the warp together: of those that may be
            uint32_t may = 0;
#pragma unroll
            for (int v = 0; v < 2; v++)
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (kept && (v ? e1 : e0) >= 0 && !(x[v][i] > lo[v] + 2.f * tol && x[v][i] < hi[v] - 2.f * tol)) may |= 1u << (v * VEC + i);
#pragma unroll 1
            for (int g = 0; g < (GROUPED ? groups : 1); g++) {
                uint32_t now = may & ((g0 == g ? (1u << VEC) - 1 : 0u) | (g1 == g ? ((1u << VEC) - 1) << VEC : 0u));
                double l = INFINITY, m = -INFINITY;
                while (now) {
                    const int n = __ffs(now) - 1;
                    now &= now - 1;
                    const double y = exact(n / VEC, n % VEC);
                    l = y < l ? y : l;
                    m = y > m ? y : m;
                    if (!(fabs(y) < INFINITY)) m = INFINITY;
                }
                __syncwarp();
                for (int o = L >> 1; o >= 1; o >>= 1) {
                    const double l2 = __shfl_xor_sync(kAll, l, o), m2 = __shfl_xor_sync(kAll, m, o);
                    l = l2 < l ? l2 : l;
                    m = m2 > m ? m2 : m;
                }
                const Held h = held_of<T>(l, m);
                if (g0 == g) held[0] = h;
                if (g1 == g) held[1] = h;
                // quotients near the ends of FP32: all codes in FP64
                ends = ends || (h.s > 0.f && !(h.s > 0x1p-100f && size < QuantType<T>::safe));
            }
        }
        if (!kept) continue;
        // ---- codes: 15 times a saturated (x - zero) / (15 scale), and how far that is from a whole number.  Off by 15 2^-21.5 for the inverse and the sums' roundings, by
        // 2^-24 of the zero's own quotient, and for a key by tol: what is that near a half is taken again.
        uint32_t word[2], unsure = 0;
        float by, less, limit;
#pragma unroll
        for (int v = 0; v < 2; v++) {
            if (GROUPED || v == 0) {
                const float s = held[v].s, z = held[v].z, inverse = s > 0.f ? __fdividef(1.f, s) : 0.f;
                by = inverse * (1.f / 15.f);
                less = -z * by;
                limit = ends ? -1.f : (0.5f - 0x1p-17f) - (0x1p-23f * fabsf(z) + tol) * inverse;
                if (s == 0.f) limit = 1.f;       // (code 0)
            }
            uint32_t sum = 0;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float t = __saturatef(__fmaf_rn(x[v][i], by, less)), m = __fmaf_rn(t, 15.f, 12582912.f);        // (1.5 2^23: the sum's last bits are the code)
                if (!(fabsf(__fmaf_rn(t, 15.f, -(m - 12582912.f))) < limit)) unsure |= 1u << (v * VEC + i);
                sum += __float_as_uint(m) << (4 * i);
            }
            word[v] = sum - 0x4B400000u * (VEC == 8 ? 0x11111111u : 0x1111u);
        }
        if (e1 < 0) unsure &= (1u << VEC) - 1;
        while (unsure) {
            const int n = __ffs(unsure) - 1, v = n / VEC, i = n % VEC;
            unsure &= unsure - 1;
            const float s = v ? held[1].s : held[0].s, z = v ? held[1].z : held[0].z;
            const float raw = Half<T>::to_float(reinterpret_cast<const T *>(place(stage, v))[i]), y = raw - z;
            uint32_t code;
            if (is_value && !ends) {
                // A value: what is left behind a code is exact, and half a scale is a tie unless x - zero was rounded
                const float m = fminf(fmaxf(y * __fdividef(1.f, s), 0.f), 15.f) + 12582912.f, left = __fmaf_rn(-(m - 12582912.f), s, y);
                const float lost = (raw - (y + z)) + ((y + z) - y - z);                           // raw = z + y + lost
                const float over = fabsf(left) == 0.5f * s ? (left > 0.f ? lost : -lost) : fabsf(left) - 0.5f * s;
                code = __float_as_uint(m) & 15u;
                if (over > 0.f || (over == 0.f && (code & 1u))) code = (uint32_t)min(max((int)code + (left > 0.f ? 1 : -1), 0), 15);
            } else {
                const double q = rint((exact(v, i) - (double)z) / (double)s);
                code = q > 0.0 ? (q < 15.0 ? (uint32_t)q : 15u) : 0u;
            }
            const uint32_t keep = ~(15u << (4 * i)), put = code << (4 * i);
            if (v) word[1] = (word[1] & keep) | put;
            else word[0] = (word[0] & keep) | put;
        }
#pragma unroll
        for (int v = 0; v < 2; v++) {
            const int e = v ? e1 : e0;
            if (e >= 0) {
                if constexpr (VEC == 8) *reinterpret_cast<uint32_t *>(to + e / 2) = word[v];
                else *reinterpret_cast<uint16_t *>(to + e / 2) = (uint16_t)word[v];
            }
            if (e >= 0 && e % width == 0) (places[token].scales[kind] + scale_at)[v ? g1 : g0] = held[v].bits;
        }
    }
    copy_wait<0>();
}

template <class T, int VEC, bool GROUPED>
static int launch_quantise(QuantiseArgs &a, cudaStream_t stream)
{
    const int64_t heads = a.d.q_heads + 2 * a.c.kv_heads, rows = 256 >> a.lanes_log2, sms = device_sm_count(current_device_index());
    // as rotary_append_kernel does it: four tokens of a CTA where there are many, the heads of one over several CTAs where there are few
    a.together = a.d.tokens >= 2 * kMostTogether * sms ? kMostTogether : 1;
    const int64_t ctas = ceil_div(a.d.tokens, a.together), most = ceil_div(heads, rows);
    int64_t y = ceil_div(2 * sms, ctas);
    y = y < 1 ? 1 : y < most ? y : most;
    const dim3 grid((unsigned)ctas, (unsigned)y);
    const size_t smem = (size_t)(kAhead * 2 * 256 * VEC * 2 + a.together * a.d.rotary * 4);
    return a.d.interleaved ? launch_dependent(quantise_append_kernel<T, VEC, true, GROUPED>, grid, 256, smem, stream, a)
                           : launch_dependent(quantise_append_kernel<T, VEC, false, GROUPED>, grid, 256, smem, stream, a);
}

template <class T, int VEC>
static int launch_quantise_of(QuantiseArgs &a, cudaStream_t stream)
{
    return a.c.groups > 1 ? launch_quantise<T, VEC, true>(a, stream) : launch_quantise<T, VEC, false>(a, stream);
}

// ---- reading back: value = round16(zero + scale code), one multiply-add in the type itself ------------------------------------------------------
// An item is 8 codes of a head, 4 bytes in and 16 out.  A thread has an item of every token (or every few) of its CTA, whose places pass through shared memory.
// Bound by HBM, four fifths of it what is written, past the cache: 65536 tokens of 8 heads of 128, 344 MB: 58.5 us = 5.9 TB/s (83 with an item of a token at a time).
struct ReadArgs {
    ortho_b200_read_quantised_desc d;
    ortho_b200_quantised_cache c;
    int together;
    FastDiv by_token, by_chunk, by_group;        // items of a token, chunks of a head, chunks of a group
};
constexpr int kMostRead = 16;

// Two codes, one from each of the 16-bit halves of w, as numbers of the type: 1024 + code in FP16 and 128 + code in BF16, less that
template <class T> struct Codes;
template <> struct Codes<__half> {
    static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t s, uint32_t z)
    {
        const uint32_t b = (w & 0x000F000Fu) | 0x64006400u, off = 0x64006400u;
        const __half2 n = __hsub2(*reinterpret_cast<const __half2 *>(&b), *reinterpret_cast<const __half2 *>(&off));
        const __half2 r = __hfma2(n, *reinterpret_cast<const __half2 *>(&s), *reinterpret_cast<const __half2 *>(&z));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
};
template <> struct Codes<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t value(uint32_t w, uint32_t s, uint32_t z)
    {
        const uint32_t b = (w & 0x000F000Fu) | 0x43004300u, off = 0x43004300u;
        const __nv_bfloat162 n = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&b), *reinterpret_cast<const __nv_bfloat162 *>(&off));
        const __nv_bfloat162 r = __hfma2(n, *reinterpret_cast<const __nv_bfloat162 *>(&s), *reinterpret_cast<const __nv_bfloat162 *>(&z));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
};

template <class T>
__global__ void __launch_bounds__(256)
read_quantised_kernel(const __grid_constant__ ReadArgs a)
{
    constexpr int U = 4;                         // items of a thread in flight together
    struct Places { const unsigned char *codes[2]; const uint32_t *scales[2]; };                  // of a token's keys and values; outside the cache: NULL
    __shared__ Places places[kMostRead];
    const auto &d = a.d;
    const auto &c = a.c;
    const int64_t t0 = (int64_t)blockIdx.x * a.together;
    const int tokens = d.count - t0 < a.together ? (int)(d.count - t0) : a.together, chunks = (int)c.head_dim / 8, per_cache = (int)c.kv_heads * chunks, per_token = 2 * per_cache;
    griddep_wait();
    griddep_launch();
    if ((int)threadIdx.x < tokens) {
        const int64_t slot = d.slots[t0 + threadIdx.x];
        const bool in = slot >= 0 && slot < c.pages * c.page_size;
        const int64_t page = in ? slot / c.page_size : 0, place = slot - page * c.page_size;
        Places &p = places[threadIdx.x];
        p.codes[0] = in ? (const unsigned char *)c.k + page * c.k_page_stride + place * c.k_slot_stride : nullptr;
        p.codes[1] = in ? (const unsigned char *)c.v + page * c.v_page_stride + place * c.v_slot_stride : nullptr;
        p.scales[0] = (const uint32_t *)c.k_scales + page * c.ks_page_stride + place * c.ks_slot_stride;
        p.scales[1] = (const uint32_t *)c.v_scales + page * c.vs_page_stride + place * c.vs_slot_stride;
    }
    __syncthreads();
    // several tokens side by side where one has few items; the threads behind the last whole token rest
    const int row = (int)a.by_token.quotient(threadIdx.x), rows = per_token <= 256 ? 256 / per_token : 1;
    for (int at = (int)(blockIdx.y * 256 + threadIdx.x) - row * per_token; at < per_token && row < rows; at += (int)gridDim.y * 256) {
        const int is_value = at >= per_cache, rest = at - (is_value ? per_cache : 0), h = (int)a.by_chunk.quotient(rest), chunk = rest - h * chunks;
        const int64_t code_at = h * (is_value ? c.v_head_stride : c.k_head_stride) + chunk * 4;
        const int64_t scale_at = h * (is_value ? c.vs_head_stride : c.ks_head_stride) + (int)a.by_group.quotient(chunk);
        const int64_t stride = is_value ? d.v_token_stride : d.k_token_stride;
        T *const out = (T *)(is_value ? d.v_out : d.k_out) + t0 * stride + h * (is_value ? d.v_head_stride : d.k_head_stride) + chunk * 8;
        for (int token0 = row; token0 < tokens; token0 += U * rows) {
            uint32_t code[U], held[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int token = token0 + u * rows;
                code[u] = held[u] = 0;
                if (token >= tokens) break;
                const unsigned char *const codes = places[token].codes[is_value];
                if (!codes) continue;
                code[u] = *reinterpret_cast<const uint32_t *>(codes + code_at);
                held[u] = places[token].scales[is_value][scale_at];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int token = token0 + u * rows;
                if (token >= tokens) break;
                const uint32_t s = __byte_perm(held[u], 0, 0x1010), z = __byte_perm(held[u], 0, 0x3232), next = code[u] >> 4;
                uint4 y;                         // byte i of the codes in the low half, its upper code brought down in the high one
                y.x = Codes<T>::value(__byte_perm(code[u], next, 0x4400), s, z);
                y.y = Codes<T>::value(__byte_perm(code[u], next, 0x5511), s, z);
                y.z = Codes<T>::value(__byte_perm(code[u], next, 0x6622), s, z);
                y.w = Codes<T>::value(__byte_perm(code[u], next, 0x7733), s, z);
                __stcs(reinterpret_cast<uint4 *>(out + token * stride), y);
            }
        }
    }
}

}  // namespace ob

using namespace ob;

extern "C" int ortho_b200_rotary_append_quantised(const ortho_b200_rotary_append_desc *d, const ortho_b200_quantised_cache *c, void *stream)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    int st = check_quantised(c);
    if (st) return st;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->tokens < 0 || d->tokens > 0x7FFFFFFF || d->q_heads < 0 || d->q_heads > 65535 || d->kv_heads != c->kv_heads || d->head_dim != c->head_dim
        || d->rotary < 0 || d->rotary % 8 || d->rotary > d->head_dim) return ORTHO_B200_ERR_SHAPE;
    if (d->rotary) {
        if (d->axes < 1 || d->axes > ORTHO_B200_MAX_AXES || d->table_rows < 0 || d->section_ends[d->axes - 1] != d->rotary / 2) return ORTHO_B200_ERR_SHAPE;
        for (int i = 0; i < d->axes; i++)
            if (d->section_ends[i] < (i ? d->section_ends[i - 1] : 0)) return ORTHO_B200_ERR_SHAPE;
    }
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->k || !d->v || !d->slots || (d->q_heads && (!d->q || !d->q_out))) return ORTHO_B200_ERR_NULL;
    if (d->rotary && (!d->positions || (d->table_rows && !d->table))) return ORTHO_B200_ERR_NULL;
    // two vectors of eight or of four values are a thread's share of a head
    const int64_t strides[] = {d->q_heads ? d->q_token_stride : 0, d->q_heads ? d->q_head_stride : 0, d->k_token_stride, d->k_head_stride, d->v_token_stride, d->v_head_stride,
                               d->q_heads ? d->out_token_stride : 0, d->q_heads ? d->out_head_stride : 0};
    const void *bases[] = {d->q_heads ? d->q : nullptr, d->k, d->v, d->q_heads ? d->q_out : nullptr};
    int vec = d->rotary % 16 ? 4 : 8;
    for (int64_t s : strides) {
        if (s % 4) return ORTHO_B200_ERR_ALIGN;
        if (s % 8) vec = 4;
    }
    for (const void *p : bases) {
        if ((uintptr_t)p & 7u) return ORTHO_B200_ERR_ALIGN;
        if ((uintptr_t)p & 15u) vec = 4;
    }
    if (d->q_heads && (expanded(d->tokens, d->out_token_stride) || expanded(d->q_heads, d->out_head_stride))) return ORTHO_B200_ERR_SHAPE;
    st = check_written(*c);
    if (st) return st;
    st = check_device();
    if (st) return st;
    QuantiseArgs a;
    a.d = *d;
    a.c = *c;
    a.turned = (int)(d->rotary / 2 / vec);
    const int64_t items = a.turned + ceil_div(d->head_dim - d->rotary, 2 * vec);
    for (a.lanes_log2 = 0; 1 << a.lanes_log2 < items; a.lanes_log2++) {}       // (32 items at most)
    a.by_half = FastDiv((uint32_t)(d->rotary ? d->rotary / 2 : 1));
    const cudaStream_t s = (cudaStream_t)stream;
    if (d->type == ORTHO_B200_TYPE_F16) return vec == 8 ? launch_quantise_of<__half, 8>(a, s) : launch_quantise_of<__half, 4>(a, s);
    return vec == 8 ? launch_quantise_of<__nv_bfloat16, 8>(a, s) : launch_quantise_of<__nv_bfloat16, 4>(a, s);
}

extern "C" int ortho_b200_read_quantised(const ortho_b200_read_quantised_desc *d, const ortho_b200_quantised_cache *c, void *stream)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    int st = check_quantised(c);
    if (st) return st;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->count < 0 || d->count > 0x7FFFFFFF) return ORTHO_B200_ERR_SHAPE;
    if (d->count == 0) return ORTHO_B200_OK;
    if (!d->slots || !d->k_out || !d->v_out) return ORTHO_B200_ERR_NULL;
    if (((uintptr_t)d->k_out | (uintptr_t)d->v_out) & 15u) return ORTHO_B200_ERR_ALIGN;
    for (int64_t s : {d->k_token_stride, d->k_head_stride, d->v_token_stride, d->v_head_stride})
        if (s % 8) return ORTHO_B200_ERR_ALIGN;
    if (d->k_out == d->v_out || expanded(d->count, d->k_token_stride) || expanded(d->count, d->v_token_stride) || expanded(c->kv_heads, d->k_head_stride)
        || expanded(c->kv_heads, d->v_head_stride)) return ORTHO_B200_ERR_SHAPE;
    st = check_device();
    if (st) return st;
    ReadArgs a;
    a.d = *d;
    a.c = *c;
    const int64_t chunks = c->head_dim / 8, items = 2 * c->kv_heads * chunks, sms = device_sm_count(current_device_index());
    // eight CTAs an SM where there are tokens enough, and four items a thread
    const int64_t rows = items <= 256 ? 256 / items : 1, fair = ceil_div(d->count, 8 * sms), few = 4 * rows < kMostRead ? 4 * rows : kMostRead;
    a.together = (int)(fair < few ? fair : fair < kMostRead ? fair : kMostRead);
    const int64_t ctas = ceil_div(d->count, a.together), most = ceil_div(items, 256);
    int64_t y = ceil_div(4 * sms, ctas);
    y = y < 1 ? 1 : y < most ? y : most;
    a.by_token = FastDiv((uint32_t)items);
    a.by_chunk = FastDiv((uint32_t)chunks);
    a.by_group = FastDiv((uint32_t)(chunks / c->groups));
    const dim3 grid((unsigned)ctas, (unsigned)y);
    return d->type == ORTHO_B200_TYPE_F16 ? launch_dependent(read_quantised_kernel<__half>, grid, 256, 0, (cudaStream_t)stream, a)
                                          : launch_dependent(read_quantised_kernel<__nv_bfloat16>, grid, 256, 0, (cudaStream_t)stream, a);
}
