// Low-rank adapters of many requests beside a shared projection:
//
//     v[t] = scale_e (down_e x[t]),   out[t] = y[t] + up_e v[t],   e = ids[t]
//
// A warp per token and rank for v, a thread per output for the rest.
#include "launch.cuh"

namespace ob {

__device__ __forceinline__ int adapter_of(const ortho_b200_low_rank_desc &d, int64_t t)
{
    const int32_t e = d.ids[t];
    return e >= 0 && e < d.adapters ? e : -1;
}
__device__ __forceinline__ int rank_of(const ortho_b200_low_rank_desc &d, int e)
{
    const int64_t r = d.ranks ? ((int64_t)max(d.ranks[e], 0) + 7) / 8 * 8 : d.rank;
    return (int)(r < d.rank ? r : d.rank);
}

template <class T>
__global__ void __launch_bounds__(128)
low_rank_down_kernel(ortho_b200_low_rank_desc d, float *v)
{
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31;
    griddep_wait();
    griddep_launch();
    const int e = adapter_of(d, t);
    if (e < 0) return;
    const int rank = rank_of(d, e);
    for (int r = threadIdx.x >> 5; r < rank; r += 4) {
        const T *x = (const T *)d.x + t * d.x_stride, *w = (const T *)d.down + ((int64_t)e * d.rank + r) * d.K;
        float s = 0.f;
        for (int64_t k = lane; k < d.K; k += 32) s += Half<T>::to_float(x[k]) * Half<T>::to_float(w[k]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) v[t * d.rank + r] = s * (d.scales ? d.scales[e] : 1.f);
    }
}

template <class T>
__global__ void __launch_bounds__(256)
low_rank_up_kernel(ortho_b200_low_rank_desc d, const float *v)
{
    const int64_t t = blockIdx.x;
    griddep_wait();
    griddep_launch();
    const int e = adapter_of(d, t), rank = e < 0 ? 0 : rank_of(d, e);
    for (int64_t n = (int64_t)blockIdx.y * 256 + threadIdx.x; n < d.N; n += (int64_t)gridDim.y * 256) {
        const T y = ((const T *)d.y)[t * d.y_stride + n];
        const T *w = (const T *)d.up + ((int64_t)(e < 0 ? 0 : e) * d.N + n) * d.rank;
        float s = 0.f;
        for (int r = 0; r < rank; r++) s += v[t * d.rank + r] * Half<T>::to_float(w[r]);
        ((T *)d.out)[t * d.out_stride + n] = rank ? Half<T>::from_float(Half<T>::to_float(y) + s) : y;
    }
}

static int check_low_rank(const ortho_b200_low_rank_desc *d)
{
    if (!d) return ORTHO_B200_ERR_NULL;
    if (d->type != ORTHO_B200_TYPE_F16 && d->type != ORTHO_B200_TYPE_BF16) return ORTHO_B200_ERR_SHAPE;
    if (d->tokens < 0 || d->tokens > 0x7FFFFFFF || d->K < 8 || d->K % 8 || d->K > 0x7FFFFFFF || d->N < 1 || d->N > 0x7FFFFFFF || d->adapters < 1 || d->adapters > 65536 || d->rank < 8 || d->rank % 8 || d->rank > 256)
        return ORTHO_B200_ERR_SHAPE;
    if (d->tokens == 0) return ORTHO_B200_OK;
    if (!d->x || !d->y || !d->out || !d->down || !d->up || !d->ids) return ORTHO_B200_ERR_NULL;
    if ((((uintptr_t)d->x | (uintptr_t)d->down | (uintptr_t)d->up) & 15u) || d->x_stride % 8) return ORTHO_B200_ERR_ALIGN;
    return ORTHO_B200_OK;
}

template <class T>
static int launch_low_rank(const ortho_b200_low_rank_desc *d, float *v, cudaStream_t stream)
{
    int st = launch_dependent(low_rank_down_kernel<T>, dim3((unsigned)d->tokens), 128, 0, stream, *d, v);
    if (st) return st;
    return launch_dependent(low_rank_up_kernel<T>, dim3((unsigned)d->tokens, (unsigned)(ceil_div(d->N, 1024) < 65535 ? ceil_div(d->N, 1024) : 65535)), 256, 0, stream, *d, (const float *)v);
}

}  // namespace ob

using namespace ob;

extern "C" int64_t ortho_b200_low_rank_add_workspace_bytes(const ortho_b200_low_rank_desc *d)
{
    return check_low_rank(d) == ORTHO_B200_OK ? 4 * d->tokens * d->rank : -1;
}

extern "C" int ortho_b200_low_rank_add(const ortho_b200_low_rank_desc *d, void *workspace, int64_t workspace_bytes, void *stream)
{
    int st = check_low_rank(d);
    if (st || d->tokens == 0) return st;
    if (!workspace || workspace_bytes < ortho_b200_low_rank_add_workspace_bytes(d) || ((uintptr_t)workspace & 255u)) return ORTHO_B200_ERR_WORKSPACE;
    st = check_device();
    if (st) return st;
    return d->type == ORTHO_B200_TYPE_F16 ? launch_low_rank<__half>(d, (float *)workspace, (cudaStream_t)stream)
                                          : launch_low_rank<__nv_bfloat16>(d, (float *)workspace, (cudaStream_t)stream);
}
