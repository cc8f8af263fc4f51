// Rotary positions of queries and keys on one to four axes, keys and values written into the paged cache.
//
//     pair i < R / 2 of a head:  (a, b) -> (a c - b s, b c + a s),  c = table[p][i], s = table[p][R / 2 + i],  p = positions[axis(i)][t]
//
// Every value is read and written once: bound by HBM.  An item is two vectors of VEC values of one head; a thread has one item and walks over the
// (token, head) pairs of its CTA, queries, keys and values alike.  Cosines and sines of the CTA's tokens pass through shared memory: in registers
// they leave too little room for values under way (4096 tokens of 96 heads of 128, 204 MB: 36.9 us = 5.5 TB/s; 40 us with a token a CTA and its angles in
// registers, 49 to 64 with values loaded ahead there).  64 tokens of 80 heads: 2.7 us, launch and the chain slot, position, angle.
#include "rotary.cuh"

namespace ob {

struct RotaryArgs {
    ortho_b200_rotary_append_desc d;
    int turned, items;                           // items of a head that turn, and all of them (two vectors each)
    int together;                                // tokens of a CTA
    FastDiv by_items, by_heads, by_half;
};

constexpr int kTurnsAhead = 2, kMostTogether = 4;  // turns of a thread whose values are in flight together; tokens of a CTA

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4)
rotary_append_kernel(const __grid_constant__ RotaryArgs a)
{
    constexpr int U = kTurnsAhead;
    extern __shared__ __align__(16) float angles[];                            // [tokens][rotary]: cosines, then sines
    __shared__ int64_t k_at[kMostTogether], v_at[kMostTogether];               // places in the caches, k_at -1 for none
    const auto &d = a.d;
    const int64_t t0 = (int64_t)blockIdx.x * a.together;
    const int tokens = d.tokens - t0 < a.together ? (int)(d.tokens - t0) : a.together;
    const int R = (int)d.rotary, half = R / 2, q_heads = (int)d.q_heads, kv_heads = (int)d.kv_heads, heads = q_heads + 2 * kv_heads, all = tokens * heads;
    // a thread's item, and the first of its (token, head) pairs; the threads behind the last whole row of items rest
    const int row = (int)a.by_items.quotient(threadIdx.x), rows = a.items <= 256 ? 256 / a.items : 1, step = (int)gridDim.y * rows;
    const int first = row < rows ? (int)blockIdx.y * rows + row : all;
    griddep_wait();
    griddep_launch();
    bool ready = false;
    for (int it0 = 0; it0 < a.items; it0 += 256) {
        const int it = it0 + (int)threadIdx.x - row * a.items;
        const bool some = it < a.items, turns = it < a.turned;
        // offsets of the two vectors
        int e0, e1;
        if (!turns) { e0 = R + 2 * (it - a.turned) * VEC; e1 = e0 + VEC; }
        else if (INTERLEAVED) { e0 = 2 * it * VEC; e1 = e0 + VEC; }
        else { e0 = it * VEC; e1 = e0 + half; }
        const bool second = e1 < d.head_dim;
        for (int j0 = some ? first : all; j0 < all || !ready; j0 += U * step) {
            Raw<VEC> r0[U], r1[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int j = j0 + u * step;
                if (j >= all) break;
                const int token = (int)a.by_heads.quotient(j), h = j - token * heads;
                const int64_t t = t0 + token;
                const T *const src = h < q_heads ? (const T *)d.q + t * d.q_token_stride + h * d.q_head_stride
                                   : h < q_heads + kv_heads ? (const T *)d.k + t * d.k_token_stride + (h - q_heads) * d.k_head_stride
                                                            : (const T *)d.v + t * d.v_token_stride + (h - q_heads - kv_heads) * d.v_head_stride;
                r0[u].load(src + e0);
                if (second) r1[u].load(src + e1);
            }
            if (!ready) {                        // once, while the first values are under way: the tokens' places, cosines and sines
                ready = true;
                if ((int)threadIdx.x < tokens) {
                    const int64_t slot = d.slots[t0 + threadIdx.x];
                    const bool kept = slot >= 0 && slot < d.pages * d.page_size;
                    const int64_t page = !kept ? 0 : slot <= 0x7FFFFFFF && d.page_size <= 0x7FFFFFFF ? (int64_t)((uint32_t)slot / (uint32_t)d.page_size) : slot / d.page_size;
                    const int64_t place = slot - page * d.page_size;
                    k_at[threadIdx.x] = kept ? page * d.k_page_stride + place * d.k_slot_stride : -1;
                    v_at[threadIdx.x] = kept ? page * d.v_page_stride + place * d.v_slot_stride : -1;
                }
                angles_of(d, a.by_half, t0, tokens, angles);
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int j = j0 + u * step;
                if (j >= all) break;
                const int token = (int)a.by_heads.quotient(j), h = j - token * heads;
                const bool is_value = h >= q_heads + kv_heads;
                if (turns && !is_value) {
                    float x0[VEC], x1[VEC], c[VEC], s[VEC];
                    const float *const at = angles + token * R + it * VEC;
                    if constexpr (VEC > 1) {               // (half is a multiple of VEC)
#pragma unroll
                        for (int i = 0; i < VEC; i += 4) {
                            const float4 x = *reinterpret_cast<const float4 *>(at + i), y = *reinterpret_cast<const float4 *>(at + half + i);
                            c[i] = x.x; c[i + 1] = x.y; c[i + 2] = x.z; c[i + 3] = x.w;
                            s[i] = y.x; s[i + 1] = y.y; s[i + 2] = y.z; s[i + 3] = y.w;
                        }
                    } else { c[0] = at[0]; s[0] = at[half]; }
                    r0[u].template to<T>(x0);
                    r1[u].template to<T>(x1);
                    if (INTERLEAVED && VEC > 1) {
#pragma unroll
                        for (int i = 0; i + 1 < VEC; i += 2) {
                            turn_pair(x0[i], x0[i + 1], c[i / 2], s[i / 2]);
                            turn_pair(x1[i], x1[i + 1], c[(VEC + i) / 2], s[(VEC + i) / 2]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; i++) turn_pair(x0[i], x1[i], c[i], s[i]);
                    }
                    r0[u].template from<T>(x0);
                    r1[u].template from<T>(x1);
                }
                const int64_t place = is_value ? v_at[token] : k_at[token];
                if (h >= q_heads && k_at[token] < 0) continue;                 // (no place in the cache)
                T *const dst = h < q_heads ? (T *)d.q_out + (t0 + token) * d.out_token_stride + h * d.out_head_stride
                             : !is_value ? (T *)d.k_cache + place + (h - q_heads) * d.k_cache_head_stride
                                         : (T *)d.v_cache + place + (h - q_heads - kv_heads) * d.v_cache_head_stride;
                r0[u].store(dst + e0);
                if (second) r1[u].store(dst + e1);
            }
        }
    }
}

template <class T, int VEC>
static int launch_rotary(RotaryArgs &a, cudaStream_t stream)
{
    const int64_t heads = a.d.q_heads + 2 * a.d.kv_heads, rows = a.items <= 256 ? 256 / a.items : 1, sms = device_sm_count(current_device_index());
    // Four tokens of a CTA share the time that their angles take to come; with few tokens one each, its heads over several CTAs until the GPU is full
    a.together = a.d.tokens >= 2 * kMostTogether * sms && a.d.rotary <= 2048 ? kMostTogether : 1;
    const int64_t ctas = ceil_div(a.d.tokens, a.together), most = ceil_div(heads * a.together, rows);
    int64_t y = ceil_div(2 * sms, ctas);
    y = y < 1 ? 1 : y < most ? y : most;
    const dim3 grid((unsigned)ctas, (unsigned)y);
    const size_t smem = (size_t)(a.together * a.d.rotary * 4);
    return a.d.interleaved ? launch_dependent(rotary_append_kernel<T, VEC, true>, grid, 256, smem, stream, a)
                           : launch_dependent(rotary_append_kernel<T, VEC, false>, grid, 256, smem, stream, a);
}

template <class T>
static int launch_rotary_of(RotaryArgs &a, int vec, cudaStream_t stream)
{
    return vec == 8 ? launch_rotary<T, 8>(a, stream) : vec == 4 ? launch_rotary<T, 4>(a, stream) : launch_rotary<T, 1>(a, stream);
}

}  // namespace ob

using namespace ob;

extern "C" int ortho_b200_rotary_append(const ortho_b200_rotary_append_desc *d, void *stream)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->tokens < 0 || d->q_heads < 0 || d->kv_heads < 1 || d->head_dim < 1 || d->pages < 0 || d->page_size < 1
        || d->tokens > 0x7FFFFFFF || d->q_heads > 65535 || d->kv_heads > 65535 || d->head_dim > 8192) return ORTHO_B200_ERR_SHAPE;
    if (d->rotary < 0 || d->rotary % 2 || d->rotary > d->head_dim) return ORTHO_B200_ERR_SHAPE;
    if (d->rotary) {
        if (d->axes < 1 || d->axes > ORTHO_B200_MAX_AXES || d->table_rows < 0 || d->section_ends[d->axes - 1] != d->rotary / 2) return ORTHO_B200_ERR_SHAPE;
        for (int i = 0; i < d->axes; i++)
            if (d->section_ends[i] < (i ? d->section_ends[i - 1] : 0)) return ORTHO_B200_ERR_SHAPE;
    }
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->k || !d->v || !d->slots || (d->pages && (!d->k_cache || !d->v_cache)) || (d->q_heads && (!d->q || !d->q_out))) return ORTHO_B200_ERR_NULL;
    if (d->rotary && (!d->positions || (d->table_rows && !d->table))) return ORTHO_B200_ERR_NULL;
    const int st = check_device();
    if (st) return st;
    // the widest vector that every address is a multiple of and that pairs and the rest of a head divide into
    const int64_t strides[] = {d->q_heads ? d->q_token_stride : 0, d->q_heads ? d->q_head_stride : 0, d->k_token_stride, d->k_head_stride, d->v_token_stride, d->v_head_stride,
                               d->q_heads ? d->out_token_stride : 0, d->q_heads ? d->out_head_stride : 0, d->k_page_stride, d->k_slot_stride, d->k_cache_head_stride,
                               d->v_page_stride, d->v_slot_stride, d->v_cache_head_stride, d->rotary / 2, d->head_dim};
    const void *bases[] = {d->q_heads ? d->q : nullptr, d->k, d->v, d->q_heads ? d->q_out : nullptr, d->k_cache, d->v_cache};
    int vec = 8;
    for (; vec > 1; vec = vec == 8 ? 4 : 1) {
        bool fits = true;
        for (int64_t s : strides) fits = fits && s % vec == 0;
        for (const void *p : bases) fits = fits && (uintptr_t)p % (2 * vec) == 0;
        if (fits) break;
    }
    RotaryArgs a;
    a.d = *d;
    a.turned = (int)(d->rotary / 2 / vec);
    a.items = a.turned + (int)ceil_div(d->head_dim - d->rotary, 2 * vec);
    a.by_items = FastDiv((uint32_t)a.items);
    a.by_heads = FastDiv((uint32_t)(d->q_heads + 2 * d->kv_heads));
    a.by_half = FastDiv((uint32_t)(d->rotary ? d->rotary / 2 : 1));
    return d->type == ORTHO_B200_TYPE_F16 ? launch_rotary_of<__half>(a, vec, (cudaStream_t)stream)
                                          : launch_rotary_of<__nv_bfloat16>(a, vec, (cudaStream_t)stream);
}
