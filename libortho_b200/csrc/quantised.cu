// Keys and values quantised to 4 bits as they are written to the paged cache, and a cache read back (quantised.cuh, include/ortho_b200.h: the format).
//
//     zero = round16(min x),  scale = round16((max x - min x) / 15),  code = clamp(rint((x - zero) / scale), 0, 15)      over a group of a head
//
// Rounding to 4 bits turns a difference in the last place of FP32 into a whole step wherever x lies next to a border, so the codes are those of exact
// arithmetic: FP32 does the work and knows its own error, and what lies within that of a border is taken again in FP64 from the raw values (a key in
// some 1500 groups, and ties).  A turned key is a c - b s of an 11-bit and a 24-bit factor each, exact in FP64 up to its last sum.
#include "quantised.cuh"
#include "rotary.cuh"

namespace ob {

struct QuantiseArgs {
    ortho_b200_rotary_append_desc d;
    ortho_b200_quantised_cache c;
    int turned, items, lanes_log2, together;     // as in rotary.cu; lanes of a head (a power of two)
    FastDiv by_heads, by_half;
};

template <class T> struct QuantType;
template <> struct QuantType<__half> {
    static constexpr float safe = 30000.f;                                     // below: neither a value nor zero + 15 scale comes near the type's end
    static constexpr double beyond = 65520.0;                                  // rounds to infinity
    static __device__ __forceinline__ __half from_double(double v) { return __double2half(v); }
};
template <> struct QuantType<__nv_bfloat16> {
    static constexpr float safe = 1e38f;
    static constexpr double beyond = 3.3961775292304957e38;
    static __device__ __forceinline__ __nv_bfloat16 from_double(double v) { return __double2bfloat16(v); }
};
template <class T> __device__ __forceinline__ uint32_t bits16(T v) { return *reinterpret_cast<const uint16_t *>(&v); }

// Element e of a head in FP64, turned or not
template <class T, bool INTERLEAVED>
__device__ __noinline__ double exact_element(const T *src, int e, const float *angles, int rotary)
{
    if (e >= rotary) return (double)Half<T>::to_float(src[e]);
    const int half = rotary / 2, pair = INTERLEAVED ? e >> 1 : e < half ? e : e - half;
    const bool upper = INTERLEAVED ? e & 1 : e >= half;
    const double a = (double)Half<T>::to_float(src[INTERLEAVED ? 2 * pair : pair]), b = (double)Half<T>::to_float(src[INTERLEAVED ? 2 * pair + 1 : pair + half]);
    const double c = (double)angles[pair], s = (double)angles[half + pair];
    return upper ? b * c + a * s : a * c - b * s;
}

// A group's scale and zero; `bits`: as they are stored.  A group that stands for NaN has scale 0 here, so that its codes come out as 0.
struct Held { float s, z; uint32_t bits; };
constexpr uint32_t kNoNumber = 0x7FFFu;

// From the least and largest of values that are each off by up to `tol`; false where that, or an end of the type, could change a bit
template <class T>
__device__ __forceinline__ bool held_of(float lo, float hi, float tol, Held &h)
{
    const float q = (hi - lo) * (1.f / 15.f), tq = tol * (2.f / 15.f) + q * 0x1p-21f;
    const T z = Half<T>::from_float(lo), s = Half<T>::from_float(q);
    h.z = Half<T>::to_float(z);
    h.s = Half<T>::to_float(s);
    h.bits = bits16(s) | bits16(z) << 16;
    return bits16(Half<T>::from_float(lo - tol)) == bits16(Half<T>::from_float(lo + tol))
        && bits16(Half<T>::from_float(q - tq)) == bits16(Half<T>::from_float(q + tq))
        && fmaxf(fabsf(lo), fabsf(hi)) < QuantType<T>::safe && (q > 1e-30f || (lo == hi && tol == 0.f));
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

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 2)
quantise_append_kernel(const __grid_constant__ QuantiseArgs a)
{
    constexpr int U = 2;                         // rows of a segment whose values are in flight together
    constexpr uint32_t kAll = 0xffffffffu;
    extern __shared__ __align__(16) float angles[];                            // [tokens][rotary]: cosines, then sines
    __shared__ int64_t places[4][4];             // of a token in codes and scales of keys and values; the first -1 for none
    const auto &d = a.d;
    const auto &c = a.c;
    const int64_t t0 = (int64_t)blockIdx.x * a.together;
    const int tokens = d.tokens - t0 < a.together ? (int)(d.tokens - t0) : a.together;
    const int R = (int)d.rotary, half = R / 2, D = (int)c.head_dim, q_heads = (int)d.q_heads, kv_heads = (int)c.kv_heads, heads = q_heads + 2 * kv_heads, all = tokens * heads;
    const int L = 1 << a.lanes_log2, it = threadIdx.x & (L - 1), seg = (threadIdx.x & 31) >> a.lanes_log2, rows = 256 >> a.lanes_log2, step = (int)gridDim.y * rows;
    const int groups = (int)c.groups, width = D / groups;
    const bool some = it < a.items, turns = it < a.turned;
    int e0, e1;                                  // elements that this thread's two vectors start with
    if (!turns) { e0 = R + 2 * (it - a.turned) * VEC; e1 = e0 + VEC; }
    else if (INTERLEAVED) { e0 = 2 * it * VEC; e1 = e0 + VEC; }
    else { e0 = it * VEC; e1 = e0 + half; }
    const bool second = some && e1 < D;
    const int g0 = groups == 1 ? 0 : e0 / kQuantGroup, g1 = groups == 1 ? 0 : e1 / kQuantGroup;
    griddep_wait();
    griddep_launch();
    bool ready = false;
    // (a warp's segments go round the loop together: they meet in shuffles)
    for (int j0 = (int)blockIdx.y * rows + ((int)threadIdx.x >> 5) * (32 >> a.lanes_log2); j0 < all || !ready; j0 += U * step) {
        Raw<VEC> r0[U], r1[U];
        const T *from[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = j0 + u * step + seg;
            from[u] = nullptr;
            if (j >= all || !some) continue;
            const int token = (int)a.by_heads.quotient(j), h = j - token * heads;
            const int64_t t = t0 + token;
            const T *const src = h < q_heads ? (const T *)d.q + t * d.q_token_stride + h * d.q_head_stride
                               : h < q_heads + kv_heads ? (const T *)d.k + t * d.k_token_stride + (h - q_heads) * d.k_head_stride
                                                        : (const T *)d.v + t * d.v_token_stride + (h - q_heads - kv_heads) * d.v_head_stride;
            from[u] = src;
            r0[u].load(src + e0);
            if (second) r1[u].load(src + e1);
        }
        if (!ready) {                            // once, while the first values are under way
            ready = true;
            if ((int)threadIdx.x < tokens) {
                const int64_t slot = d.slots[t0 + threadIdx.x];
                const bool kept = slot >= 0 && slot < c.pages * c.page_size;
                const int64_t page = kept ? slot / c.page_size : 0, place = slot - page * c.page_size;
                places[threadIdx.x][0] = kept ? page * c.k_page_stride + place * c.k_slot_stride : -1;
                places[threadIdx.x][1] = page * c.v_page_stride + place * c.v_slot_stride;
                places[threadIdx.x][2] = page * c.ks_page_stride + place * c.ks_slot_stride;
                places[threadIdx.x][3] = page * c.vs_page_stride + place * c.vs_slot_stride;
            }
            angles_of(d, a.by_half, t0, tokens, angles);
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (j0 + u * step >= all) break;     // (the whole warp)
            const int j = j0 + u * step + seg, token = j < all ? (int)a.by_heads.quotient(j) : 0, h = j - token * heads;
            const bool is_query = h < q_heads, is_value = h >= q_heads + kv_heads;
            const float *const angle = angles + token * R;
            float x0[VEC], x1[VEC];
            if (from[u]) {
                r0[u].template to<T>(x0);
                if (second) r1[u].template to<T>(x1);
                if (turns && !is_value) {
                    float cs[VEC], sn[VEC];
                    const float *const at = angle + it * VEC;
#pragma unroll
                    for (int i = 0; i < VEC; i += 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(at + i), y = *reinterpret_cast<const float4 *>(at + half + i);
                        cs[i] = x.x; cs[i + 1] = x.y; cs[i + 2] = x.z; cs[i + 3] = x.w;
                        sn[i] = y.x; sn[i + 1] = y.y; sn[i + 2] = y.z; sn[i + 3] = y.w;
                    }
                    if (INTERLEAVED) {
#pragma unroll
                        for (int i = 0; i + 1 < VEC; i += 2) {
                            turn_pair(x0[i], x0[i + 1], cs[i / 2], sn[i / 2]);
                            turn_pair(x1[i], x1[i + 1], cs[(VEC + i) / 2], sn[(VEC + i) / 2]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; i++) turn_pair(x0[i], x1[i], cs[i], sn[i]);
                    }
                }
                if (is_query) {
                    r0[u].template from<T>(x0);
                    T *const dst = (T *)d.q_out + (t0 + token) * d.out_token_stride + h * d.out_head_stride;
                    r0[u].store(dst + e0);
                    if (second) {
                        r1[u].template from<T>(x1);
                        r1[u].store(dst + e1);
                    }
                }
            }
            const bool kept = from[u] && !is_query && places[token][0] >= 0;
            if (!__any_sync(kAll, kept)) continue;
            // ---- least and largest value of the groups of this thread's vectors, and largest size in the head
            float least[2] = {INFINITY, INFINITY}, most[2] = {-INFINITY, -INFINITY};
            if (kept) {
#pragma unroll
                for (int i = 0; i < VEC; i++) { least[0] = fminf(least[0], x0[i]); most[0] = fmaxf(most[0], x0[i]); }
                if (second) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) { least[1] = fminf(least[1], x1[i]); most[1] = fmaxf(most[1], x1[i]); }
                }
            }
            float lo[2], hi[2], size = 0.f;
            for (int g = 0; g < groups; g++) {
                float l = fminf(g0 == g ? least[0] : INFINITY, g1 == g ? least[1] : INFINITY), m = fmaxf(g0 == g ? most[0] : -INFINITY, g1 == g ? most[1] : -INFINITY);
                for (int o = L >> 1; o >= 1; o >>= 1) {
                    l = fminf(l, __shfl_xor_sync(kAll, l, o));
                    m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
                }
                if (g0 == g) { lo[0] = l; hi[0] = m; }
                if (g1 == g) { lo[1] = l; hi[1] = m; }
                size = fmaxf(size, fmaxf(fabsf(l), fabsf(m)));
            }
            if (!second) { lo[1] = lo[0]; hi[1] = hi[0]; }
            // A turned value a c - b s is off by at most 2^-24 (|b s| + |x|), and both are at most sqrt(c c + s s) |(a, b)| = |(x, y)| <= 2 size
            const float tol = is_value || R == 0 ? 0.f : 0x1p-22f * size;
            Held held[2] = {};
            bool sure = true;
            if (kept) {
                sure = held_of<T>(lo[0], hi[0], tol, held[0]);
                if (g1 == g0) held[1] = held[0];
                else sure = held_of<T>(lo[1], hi[1], tol, held[1]) && sure;
            }
            if (!__all_sync(kAll, sure)) {       // the same in FP64, for the whole warp
                double l0[2] = {INFINITY, INFINITY}, m0[2] = {-INFINITY, -INFINITY};
                if (kept) {
                    for (int v = 0; v < (second ? 2 : 1); v++)
#pragma unroll 1
                        for (int i = 0; i < VEC; i++) {
                            const double x = exact_element<T, INTERLEAVED>(from[u], (v ? e1 : e0) + i, angle, is_value ? 0 : R);
                            l0[v] = x < l0[v] ? x : l0[v];
                            m0[v] = x > m0[v] ? x : m0[v];
                            if (!(fabs(x) < INFINITY)) m0[v] = INFINITY;
                        }
                }
                for (int g = 0; g < groups; g++) {
                    double l = INFINITY, m = -INFINITY;
                    for (int v = 0; v < 2; v++)
                        if ((v ? g1 : g0) == g) { l = l0[v] < l ? l0[v] : l; m = m0[v] > m ? m0[v] : m; }
                    for (int o = L >> 1; o >= 1; o >>= 1) {
                        const double l2 = __shfl_xor_sync(kAll, l, o), m2 = __shfl_xor_sync(kAll, m, o);
                        l = l2 < l ? l2 : l;
                        m = m2 > m ? m2 : m;
                    }
                    if (!kept) continue;
                    if (g0 == g) held[0] = held_of<T>(l, m);
                    if (g1 == g) held[1] = held_of<T>(l, m);
                }
            }
            // ---- codes.  What is left of a value behind its code, x - zero - code scale, shows in FP32 whether the code is the next one; it is off by
            // tol and the rounding of x - zero (2^-24 of at most 15.5 scales; in a value it is 0 where there is a tie)
            uint32_t word[2] = {0, 0};
            bool odd[2] = {false, false};        // a value that is no number
            if (kept) {
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    if (v && !second) break;
                    const float s = held[v].s, z = held[v].z, inverse = s > 0.f ? __frcp_rn(s) : 0.f;
                    const float limit = s > 0.f ? 0.5f * s - (is_value ? 0.f : tol + s * 0x1p-20f) : INFINITY;
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        const float x = (v ? x1[i] : x0[i]) - z;
                        const float m = fminf(fmaxf(x * inverse, 0.f), 15.f) + 12582912.f;        // (1.5 2^23: the sum's last bits are the code)
                        uint32_t code = __float_as_uint(m) & 15u;
                        if (!(fabsf(__fmaf_rn(-(m - 12582912.f), s, x)) < limit)) {
                            const double exact = exact_element<T, INTERLEAVED>(from[u], (v ? e1 : e0) + i, angle, is_value ? 0 : R);
                            odd[v] = odd[v] || !(fabs(exact) < INFINITY);
                            const double y = rint((exact - (double)z) / (double)s);
                            code = s > 0.f && y > 0.0 ? (y < 15.0 ? (uint32_t)y : 15u) : 0u;
                        }
                        word[v] |= code << (4 * i);
                    }
                }
            }
            if (__any_sync(kAll, odd[0] || odd[1])) {
                for (int g = 0; g < groups; g++) {
                    const uint32_t who = __ballot_sync(kAll, (odd[0] && g0 == g) || (odd[1] && g1 == g));
                    if (!(who >> (seg << a.lanes_log2) & (L == 32 ? kAll : (1u << L) - 1))) continue;
                    if (g0 == g) { word[0] = 0; held[0].bits = kNoNumber; }
                    if (g1 == g) { word[1] = 0; held[1].bits = kNoNumber; }
                }
            }
            if (!kept) continue;
            const int hk = h - q_heads - (is_value ? kv_heads : 0);
            unsigned char *const codes = is_value ? (unsigned char *)c.v + places[token][1] + hk * c.v_head_stride : (unsigned char *)c.k + places[token][0] + hk * c.k_head_stride;
            uint32_t *const scales = is_value ? (uint32_t *)c.v_scales + places[token][3] + hk * c.vs_head_stride : (uint32_t *)c.k_scales + places[token][2] + hk * c.ks_head_stride;
#pragma unroll
            for (int v = 0; v < 2; v++) {
                if (v && !second) break;
                const int e = v ? e1 : e0;
                if constexpr (VEC == 8) *reinterpret_cast<uint32_t *>(codes + e / 2) = word[v];
                else *reinterpret_cast<uint16_t *>(codes + e / 2) = (uint16_t)word[v];
                if (e % width == 0) scales[v ? g1 : g0] = held[v].bits;
            }
        }
    }
}

template <class T, int VEC>
static int launch_quantise(QuantiseArgs &a, cudaStream_t stream)
{
    const int64_t heads = a.d.q_heads + 2 * a.c.kv_heads, rows = 256 >> a.lanes_log2, sms = device_sm_count(current_device_index());
    // as rotary_append_kernel does it: four tokens of a CTA where there are many, the heads of one over several CTAs where there are few
    a.together = a.d.tokens >= 8 * sms ? 4 : 1;
    const int64_t ctas = ceil_div(a.d.tokens, a.together), most = ceil_div(heads * a.together, rows);
    int64_t y = ceil_div(2 * sms, ctas);
    y = y < 1 ? 1 : y < most ? y : most;
    const dim3 grid((unsigned)ctas, (unsigned)y);
    const size_t smem = (size_t)(a.together * a.d.rotary * 4);
    return a.d.interleaved ? launch_dependent(quantise_append_kernel<T, VEC, true>, grid, 256, smem, stream, a)
                           : launch_dependent(quantise_append_kernel<T, VEC, false>, grid, 256, smem, stream, a);
}

// ---- reading back: value = round16(zero + scale code), one multiply-add in the type itself ------------------------------------------------------
// An item is 8 codes of a head, 4 bytes in and 16 out; a CTA has a few tokens, whose places pass through shared memory.  Bound by HBM, four fifths of it
// what is written.
struct ReadArgs {
    ortho_b200_read_quantised_desc d;
    ortho_b200_quantised_cache c;
    int together;
    FastDiv by_token, by_chunk, by_group;        // items of a token, chunks of a head, chunks of a group
};
constexpr int kMostRead = 32;

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
    __shared__ int64_t places[kMostRead][4];
    const auto &d = a.d;
    const auto &c = a.c;
    const int64_t t0 = (int64_t)blockIdx.x * a.together;
    const int tokens = d.count - t0 < a.together ? (int)(d.count - t0) : a.together, chunks = (int)c.head_dim / 8, per_cache = (int)c.kv_heads * chunks, all = tokens * 2 * per_cache;
    griddep_wait();
    griddep_launch();
    if ((int)threadIdx.x < tokens) {
        const int64_t slot = d.slots[t0 + threadIdx.x];
        const bool in = slot >= 0 && slot < c.pages * c.page_size;
        const int64_t page = in ? slot / c.page_size : 0, place = slot - page * c.page_size;
        places[threadIdx.x][0] = in ? page * c.k_page_stride + place * c.k_slot_stride : -1;
        places[threadIdx.x][1] = page * c.v_page_stride + place * c.v_slot_stride;
        places[threadIdx.x][2] = page * c.ks_page_stride + place * c.ks_slot_stride;
        places[threadIdx.x][3] = page * c.vs_page_stride + place * c.vs_slot_stride;
    }
    __syncthreads();
    for (int i0 = (int)(blockIdx.y * blockDim.x + threadIdx.x); i0 < all; i0 += U * (int)(gridDim.y * blockDim.x)) {
        uint32_t code[U], held[U];
        uint4 *to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * (int)(gridDim.y * blockDim.x);
            to[u] = nullptr;
            if (i >= all) break;
            const int token = (int)a.by_token.quotient(i), at = i - token * 2 * per_cache;
            const bool is_value = at >= per_cache;
            const int rest = at - (is_value ? per_cache : 0), h = (int)a.by_chunk.quotient(rest), chunk = rest - h * chunks, group = (int)a.by_group.quotient(chunk);
            to[u] = reinterpret_cast<uint4 *>((T *)(is_value ? d.v_out : d.k_out) + (t0 + token) * (is_value ? d.v_token_stride : d.k_token_stride)
                                              + h * (is_value ? d.v_head_stride : d.k_head_stride) + chunk * 8);
            code[u] = held[u] = 0;
            if (places[token][0] < 0) continue;
            code[u] = *reinterpret_cast<const uint32_t *>(is_value ? (const unsigned char *)c.v + places[token][1] + h * c.v_head_stride + chunk * 4
                                                                   : (const unsigned char *)c.k + places[token][0] + h * c.k_head_stride + chunk * 4);
            held[u] = *(is_value ? (const uint32_t *)c.v_scales + places[token][3] + h * c.vs_head_stride + group
                                 : (const uint32_t *)c.k_scales + places[token][2] + h * c.ks_head_stride + group);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!to[u]) break;
            const uint32_t s = __byte_perm(held[u], 0, 0x1010), z = __byte_perm(held[u], 0, 0x3232), next = code[u] >> 4;
            uint4 y;                             // byte i of the codes in the low half, its upper code brought down in the high one
            y.x = Codes<T>::value(__byte_perm(code[u], next, 0x4400), s, z);
            y.y = Codes<T>::value(__byte_perm(code[u], next, 0x5511), s, z);
            y.z = Codes<T>::value(__byte_perm(code[u], next, 0x6622), s, z);
            y.w = Codes<T>::value(__byte_perm(code[u], next, 0x7733), s, z);
            *to[u] = y;
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
    st = check_device();
    if (st) return st;
    QuantiseArgs a;
    a.d = *d;
    a.c = *c;
    a.turned = (int)(d->rotary / 2 / vec);
    a.items = a.turned + (int)ceil_div(d->head_dim - d->rotary, 2 * vec);
    for (a.lanes_log2 = 0; 1 << a.lanes_log2 < a.items; a.lanes_log2++) {}     // (32 items at most)
    a.by_heads = FastDiv((uint32_t)(d->q_heads + 2 * d->kv_heads));
    a.by_half = FastDiv((uint32_t)(d->rotary ? d->rotary / 2 : 1));
    const cudaStream_t s = (cudaStream_t)stream;
    if (d->type == ORTHO_B200_TYPE_F16) return vec == 8 ? launch_quantise<__half, 8>(a, s) : launch_quantise<__half, 4>(a, s);
    return vec == 8 ? launch_quantise<__nv_bfloat16, 8>(a, s) : launch_quantise<__nv_bfloat16, 4>(a, s);
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
    st = check_device();
    if (st) return st;
    ReadArgs a;
    a.d = *d;
    a.c = *c;
    const int64_t chunks = c->head_dim / 8, items = 2 * c->kv_heads * chunks, sms = device_sm_count(current_device_index());
    // some 4096 items to a CTA where there are enough of them; where there are few, a token's items over several CTAs
    const int64_t together = ceil_div(4096, items), fair = ceil_div(d->count, 8 * sms);
    a.together = (int)(together < fair ? together : fair);
    if (a.together > kMostRead) a.together = kMostRead;
    const int64_t ctas = ceil_div(d->count, a.together), most = ceil_div(items * a.together, 1024);
    int64_t y = ceil_div(4 * sms, ctas);
    y = y < 1 ? 1 : y < most ? y : most;
    a.by_token = FastDiv((uint32_t)items);
    a.by_chunk = FastDiv((uint32_t)chunks);
    a.by_group = FastDiv((uint32_t)(chunks / c->groups));
    const dim3 grid((unsigned)ctas, (unsigned)y);
    return d->type == ORTHO_B200_TYPE_F16 ? launch_dependent(read_quantised_kernel<__half>, grid, 256, 0, (cudaStream_t)stream, a)
                                          : launch_dependent(read_quantised_kernel<__nv_bfloat16>, grid, 256, 0, (cudaStream_t)stream, a);
}
