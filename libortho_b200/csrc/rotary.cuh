// Vectors of 16-bit values and the turn of a pair, for the kernels that write the paged caches.
#pragma once

#include "launch.cuh"

namespace ob {

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

// (a c - b s, b c + a s), the same bits in every variant: two products are rounded, the other two are not
__device__ __forceinline__ void turn_pair(float &a, float &b, float c, float s)
{
    const float was = a;
    a = __fmaf_rn(a, c, -__fmul_rn(b, s));
    b = __fmaf_rn(b, c, __fmul_rn(was, s));
}

// Cosines and sines of a CTA's tokens, [tokens][rotary]: 1 and 0 where a position lies outside the table
__device__ __forceinline__ void angles_of(const ortho_b200_rotary_append_desc &d, const FastDiv &by_half, int64_t t0, int tokens, float *angles)
{
    const int R = (int)d.rotary, half = R / 2;
    for (int i = threadIdx.x; i < tokens * half; i += 256) {
        const int token = (int)by_half.quotient(i), pair = i - token * half;
        int axis = 0;
#pragma unroll
        for (int x = 0; x < ORTHO_B200_MAX_AXES - 1; x++) axis += x + 1 < d.axes && pair >= d.section_ends[x];
        const int32_t p = d.positions[axis * d.position_stride + t0 + token];
        const bool in = p >= 0 && p < d.table_rows;
        angles[token * R + pair] = in ? d.table[(int64_t)p * R + pair] : 1.f;
        angles[token * R + half + pair] = in ? d.table[(int64_t)p * R + half + pair] : 0.f;
    }
}

}  // namespace ob
