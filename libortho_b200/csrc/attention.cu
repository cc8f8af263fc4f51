// Attention of one new token per request over a paged key-value cache:
//
//     s_j = scale q . k_j,   out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max),   lse = max + log sum_j exp(s_j - max)
//
// One CTA per row and query head, keys in blocks of 128: a thread has the score of one key, then one or two elements of the output.
#include "launch.cuh"

namespace ob {

struct AttentionArgs {
    ortho_b200_paged_attention_desc d;
    FastDiv by_page;
};

template <class T>
__global__ void __launch_bounds__(128)
paged_attention_kernel(AttentionArgs a)
{
    const auto &d = a.d;
    __shared__ float q[256], p[128], red[4];
    __shared__ int32_t page_of[128];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = (int)d.head_dim;
    const int64_t b = blockIdx.x, h = blockIdx.y, g = h / (d.q_heads / d.kv_heads);
    griddep_wait();
    griddep_launch();
    const int64_t row = d.row_of ? d.row_of[b] : b;
    int64_t n = row >= 0 && row < d.rows ? d.lengths[b] : 0;
    n = n < 0 ? 0 : n < d.width * d.page_size ? n : d.width * d.page_size;
    const int64_t from = d.window > 0 && n > d.window ? n - d.window : 0;
    for (int i = tid; i < D; i += 128) q[i] = Half<T>::to_float(((const T *)d.q)[b * d.q_token_stride + h * d.q_head_stride + i]);
    float top = -INFINITY, sum = 0.f, o0 = 0.f, o1 = 0.f;
    for (int64_t j0 = from; j0 < n; j0 += 128) {
        __syncthreads();
        const int64_t j = j0 + tid;
        float s = -INFINITY;
        int32_t page = -1;
        if (j < n) {
            page = d.block_table[row * d.table_stride + j / d.page_size];
            if (page >= 0 && page < d.pages) {
                const T *k = (const T *)d.k_cache + page * d.k_page_stride + (j % d.page_size) * d.k_slot_stride + g * d.k_head_stride;
                s = 0.f;
                for (int i = 0; i < D; i++) s += q[i] * Half<T>::to_float(k[i]);
                s *= d.scale;
            } else page = -1;
        }
        float m = s;
#pragma unroll
        for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        if (lane == 0) red[warp] = m;
        __syncthreads();
        const float now = fmaxf(top, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = now == -INFINITY ? 0.f : now, keep = __expf(top - base);
        page_of[tid] = page;
        p[tid] = page >= 0 ? __expf(s - base) : 0.f;
        top = now;
        __syncthreads();
        sum *= keep; o0 *= keep; o1 *= keep;
        for (int i = 0; i < 128; i++) {
            if (page_of[i] < 0) continue;
            const T *v = (const T *)d.v_cache + page_of[i] * d.v_page_stride + ((j0 + i) % d.page_size) * d.v_slot_stride + g * d.v_head_stride;
            sum += p[i];
            if (tid < D) o0 += p[i] * Half<T>::to_float(v[tid]);
            if (tid + 128 < D) o1 += p[i] * Half<T>::to_float(v[tid + 128]);
        }
    }
    const float r = sum > 0.f ? 1.f / sum : 0.f;
    T *out = (T *)d.out + b * d.out_token_stride + h * d.out_head_stride;
    if (tid < D) out[tid] = Half<T>::from_float(sum == 0.f ? 0.f : o0 * r);
    if (tid + 128 < D) out[tid + 128] = Half<T>::from_float(sum == 0.f ? 0.f : o1 * r);
    if (d.lse && tid == 0) d.lse[b * d.q_heads + h] = sum == 0.f ? -INFINITY : top + __logf(sum);
}

static int check_attention(const ortho_b200_paged_attention_desc *d)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->batch < 0 || d->batch > 0x7FFFFFFF || d->q_heads < 1 || d->kv_heads < 1 || d->q_heads > 65535 || d->q_heads % d->kv_heads || d->head_dim < 8 || d->head_dim > 256 || d->head_dim % 8
        || d->rows < 0 || d->width < 0 || d->pages < 0 || d->page_size < 1 || d->window < 0 || d->width > 0x7FFFFFFF / d->page_size) return ORTHO_B200_ERR_SHAPE;
    if (d->batch == 0) return ORTHO_B200_OK;
    if (!d->q || !d->k_cache || !d->v_cache || !d->out || !d->lengths || (d->rows && d->width && !d->block_table)) return ORTHO_B200_ERR_NULL;
    if (((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache | (uintptr_t)d->out) & 15u) return ORTHO_B200_ERR_ALIGN;
    for (int64_t s : {d->q_token_stride, d->q_head_stride, d->out_token_stride, d->out_head_stride, d->k_page_stride, d->k_slot_stride, d->k_head_stride, d->v_page_stride, d->v_slot_stride, d->v_head_stride})
        if (s % 8) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

}  // namespace ob

using namespace ob;

extern "C" int64_t ortho_b200_paged_attention_workspace_bytes(const ortho_b200_paged_attention_desc *d)
{
    return check_attention(d) == ORTHO_B200_OK ? 0 : -1;
}

extern "C" int ortho_b200_paged_attention(const ortho_b200_paged_attention_desc *d, void *workspace, int64_t workspace_bytes, void *stream)
{
    (void)workspace; (void)workspace_bytes;
    int st = check_attention(d);
    if (st || d->batch == 0) return st;
    st = check_device();
    if (st) return st;
    AttentionArgs a;
    a.d = *d;
    a.by_page = FastDiv((uint32_t)d->page_size);
    const dim3 grid((unsigned)d->batch, (unsigned)d->q_heads);
    return d->type == ORTHO_B200_TYPE_F16 ? launch_dependent(paged_attention_kernel<__half>, grid, 128, 0, (cudaStream_t)stream, a)
                                          : launch_dependent(paged_attention_kernel<__nv_bfloat16>, grid, 128, 0, (cudaStream_t)stream, a);
}
