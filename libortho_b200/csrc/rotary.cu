// Rotary positions of queries and keys on one to four axes, keys and values written into the paged cache.
//
//     pair i < R / 2 of a head:  (a, b) -> (a c - b s, b c + a s),  c = table[p][i], s = table[p][R / 2 + i],  p = positions[axis(i)][t]
//
// Every value is read and written once.  An item is two vectors of VEC values of one head; a thread keeps an item's cosines and sines and
// walks over the heads of its token, queries, keys and values alike.
#include "launch.cuh"

namespace ob {

struct RotaryArgs {
    ortho_b200_rotary_append_desc d;
    int turned, items;                           // items of a head that turn, and all of them (two vectors each)
    FastDiv by_items;
};

// VEC 16-bit values as they lie in memory
template <int VEC>
struct Raw {
    uint32_t w[VEC > 1 ? VEC / 2 : 1];
    __device__ __forceinline__ void load(const void *p)
    {
        if constexpr (VEC == 8) { const uint4 u = *reinterpret_cast<const uint4 *>(p); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
        else if constexpr (VEC == 4) { const uint2 u = *reinterpret_cast<const uint2 *>(p); w[0] = u.x; w[1] = u.y; }
        else w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
    __device__ __forceinline__ void store(void *p) const
    {
        if constexpr (VEC == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (VEC == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
    }
    template <class T> __device__ __forceinline__ void to(float (&o)[VEC]) const
    {
#pragma unroll
        for (int j = 0; j < (VEC + 1) / 2; j++) {
            const float2 f = Half<T>::unpack(w[j]);
            o[2 * j] = f.x;
            if (VEC > 1) o[VEC > 1 ? 2 * j + 1 : 0] = f.y;
        }
    }
    template <class T> __device__ __forceinline__ void from(const float (&o)[VEC])
    {
#pragma unroll
        for (int j = 0; j < (VEC + 1) / 2; j++) w[j] = Half<T>::pack(o[2 * j], VEC > 1 ? o[VEC > 1 ? 2 * j + 1 : 0] : 0.f);
    }
};

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256)
rotary_append_kernel(RotaryArgs a)
{
    const auto &d = a.d;
    const int64_t t = blockIdx.x;
    const int half = (int)d.rotary / 2, all_heads = (int)(d.q_heads + 2 * d.kv_heads);
    // a thread's item, and the first of its heads; the threads behind the last whole row of items rest
    const int row = (int)a.by_items.quotient(threadIdx.x), item = threadIdx.x - row * a.items, rows = a.items <= 256 ? 256 / a.items : 1;
    griddep_wait();
    griddep_launch();
    const int64_t slot = d.slots[t];
    const bool kept = slot >= 0 && slot < d.pages * d.page_size;
    int64_t page = 0, place = 0;
    if (kept) { page = slot / d.page_size; place = slot - page * d.page_size; }
    if (row >= rows) return;
    for (int it = item; it < a.items; it += 256) {
        const bool turns = it < a.turned;
        // offsets of the two vectors
        int e0, e1;
        if (!turns) { e0 = (int)d.rotary + 2 * (it - a.turned) * VEC; e1 = e0 + VEC; }
        else if (INTERLEAVED) { e0 = 2 * it * VEC; e1 = e0 + VEC; }
        else { e0 = it * VEC; e1 = e0 + half; }
        float c[VEC], s[VEC];
        if (turns) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int i = it * VEC + j;
                int axis = 0;
#pragma unroll
                for (int x = 0; x < ORTHO_B200_MAX_AXES - 1; x++) axis += x + 1 < d.axes && i >= d.section_ends[x];
                const int32_t p = d.positions[axis * d.position_stride + t];
                const bool in = p >= 0 && p < d.table_rows;
                c[j] = in ? d.table[(int64_t)p * d.rotary + i] : 1.f;
                s[j] = in ? d.table[(int64_t)p * d.rotary + half + i] : 0.f;
            }
        }
        const bool second = e1 < d.head_dim;
        for (int h = (int)blockIdx.y * rows + row; h < all_heads; h += (int)gridDim.y * rows) {
            const T *src;
            T *dst;
            bool turn = turns, write = true;
            if (h < d.q_heads) {
                src = (const T *)d.q + t * d.q_token_stride + h * d.q_head_stride;
                dst = (T *)d.q_out + t * d.out_token_stride + h * d.out_head_stride;
            } else if (h < d.q_heads + d.kv_heads) {
                const int g = h - (int)d.q_heads;
                src = (const T *)d.k + t * d.k_token_stride + g * d.k_head_stride;
                dst = (T *)d.k_cache + page * d.k_page_stride + place * d.k_slot_stride + g * d.k_cache_head_stride;
                write = kept;
            } else {
                const int g = h - (int)(d.q_heads + d.kv_heads);
                src = (const T *)d.v + t * d.v_token_stride + g * d.v_head_stride;
                dst = (T *)d.v_cache + page * d.v_page_stride + place * d.v_slot_stride + g * d.v_cache_head_stride;
                turn = false;
                write = kept;
            }
            if (!write) continue;
            Raw<VEC> r0, r1;
            r0.load(src + e0);
            if (second) r1.load(src + e1);
            if (turn) {
                float x0[VEC], x1[VEC];
                r0.template to<T>(x0);
                r1.template to<T>(x1);
                if (INTERLEAVED && VEC > 1) {
#pragma unroll
                    for (int j = 0; j + 1 < VEC; j += 2) {
                        const int i0 = j / 2, i1 = (VEC + j) / 2;
                        const float a0 = x0[j], b0 = x0[j + 1], a1 = x1[j], b1 = x1[j + 1];
                        x0[j] = a0 * c[i0] - b0 * s[i0]; x0[j + 1] = b0 * c[i0] + a0 * s[i0];
                        x1[j] = a1 * c[i1] - b1 * s[i1]; x1[j + 1] = b1 * c[i1] + a1 * s[i1];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const float lo = x0[j], hi = x1[j];
                        x0[j] = lo * c[j] - hi * s[j];
                        x1[j] = hi * c[j] + lo * s[j];
                    }
                }
                r0.template from<T>(x0);
                r1.template from<T>(x1);
            }
            r0.store(dst + e0);
            if (second) r1.store(dst + e1);
        }
    }
}

template <class T, int VEC>
static int launch_rotary(const RotaryArgs &a, cudaStream_t stream)
{
    const int64_t heads = a.d.q_heads + 2 * a.d.kv_heads, rows = a.items <= 256 ? 256 / a.items : 1;
    // heads of a token over several CTAs only where the tokens alone do not fill the GPU
    int64_t y = ceil_div(2 * device_sm_count(current_device_index()), a.d.tokens);
    const int64_t most = ceil_div(heads, rows);
    y = y < 1 ? 1 : y < most ? y : most;
    const dim3 grid((unsigned)a.d.tokens, (unsigned)y);
    return a.d.interleaved ? launch_dependent(rotary_append_kernel<T, VEC, true>, grid, 256, 0, stream, a)
                           : launch_dependent(rotary_append_kernel<T, VEC, false>, grid, 256, 0, stream, a);
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
        || d->tokens > 0x7FFFFFFF || d->q_heads > 65535 || d->kv_heads > 65535 || d->head_dim > 65536) return ORTHO_B200_ERR_SHAPE;
    if (d->rotary < 0 || d->rotary % 2 || d->rotary > d->head_dim) return ORTHO_B200_ERR_SHAPE;
    if (d->rotary) {
        if (d->axes < 1 || d->axes > ORTHO_B200_MAX_AXES || d->table_rows < 0 || d->section_ends[d->axes - 1] != d->rotary / 2) return ORTHO_B200_ERR_SHAPE;
        for (int i = 0; i < d->axes; i++)
            if (d->section_ends[i] < (i ? d->section_ends[i - 1] : 0)) return ORTHO_B200_ERR_SHAPE;
    }
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->k || !d->v || !d->k_cache || !d->v_cache || !d->slots || (d->q_heads && (!d->q || !d->q_out))) return ORTHO_B200_ERR_NULL;
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
    return d->type == ORTHO_B200_TYPE_F16 ? launch_rotary_of<__half>(a, vec, (cudaStream_t)stream)
                                          : launch_rotary_of<__nv_bfloat16>(a, vec, (cudaStream_t)stream);
}
