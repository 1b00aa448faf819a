// Device helpers of the cache operators: vectors of eight lanes in f32, f16 or bf16, and the rows of a sequence.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache.h"

namespace qb {

// ---------------------------------------------------------------------------------- eight values of a row
template <typename T> struct Vec8 { uint32_t w[sizeof(T) * 2]; };

template <typename T>
__device__ __forceinline__ Vec8<T> zero8()
{
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; i++) v.w[i] = 0;
    return v;
}

// wide: p is 16-byte aligned; else it has its type's own alignment only
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T *p, bool wide)
{
    Vec8<T> v;
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 u = __ldg((const uint4 *)p + i);
            v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
        }
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) v.w[i % (sizeof(T) * 2)] = ((const uint32_t *)p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v.w[i] = ((const uint16_t *)p)[2 * i] | (uint32_t)((const uint16_t *)p)[2 * i + 1] << 16;
    }
    return v;
}

__device__ __forceinline__ void unpack8(const Vec8<float> &x, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(x.w[i]);
}
__device__ __forceinline__ void unpack8(const Vec8<__half> &x, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __half2float(__ushort_as_half((unsigned short)(x.w[i] & 0xffffu)));
        v[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(x.w[i] >> 16)));
    }
}
__device__ __forceinline__ void unpack8(const Vec8<__nv_bfloat16> &x, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(x.w[i] << 16);
        v[2 * i + 1] = __uint_as_float(x.w[i] & 0xffff0000u);
    }
}

// The largest magnitude's bits, of eight values and of what was there: two 16-bit halves, or one word.
template <typename T>
__device__ __forceinline__ uint32_t largest8(const Vec8<T> &x, uint32_t bits)
{
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 2; i++) bits = sizeof(T) == 4 ? max(bits, x.w[i] & 0x7fffffffu) : __vmaxu2(bits, x.w[i] & 0x7fff7fffu);
    return bits;
}
__device__ __forceinline__ uint32_t largest_of(uint32_t bits, const float *) { return bits; }
__device__ __forceinline__ uint32_t largest_of(uint32_t bits, const void *) { return max(bits & 0xffffu, bits >> 16); }
__device__ __forceinline__ float magnitude(uint32_t bits, const float *) { return __uint_as_float(bits); }
__device__ __forceinline__ float magnitude(uint32_t bits, const __half *) { return __half2float(__ushort_as_half((unsigned short)bits)); }
__device__ __forceinline__ float magnitude(uint32_t bits, const __nv_bfloat16 *) { return __uint_as_float(bits << 16); }

__device__ __forceinline__ uint32_t bits_of(float x, const __half *) { return __half_as_ushort(__float2half_rn(x)); }
__device__ __forceinline__ uint32_t bits_of(float x, const __nv_bfloat16 *) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
__device__ __forceinline__ uint32_t bits_of(float x, const float *) { return __float_as_uint(x); }

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8], bool wide)
{
    if (sizeof(T) == 4) {
        if (wide) {
            ((float4 *)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            ((float4 *)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) ((float *)p)[i] = v[i];
        }
    } else {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = bits_of(v[i], p);
        if (wide) *(uint4 *)p = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        else {
#pragma unroll
            for (int i = 0; i < 8; i++) ((uint16_t *)p)[i] = (uint16_t)h[i];
        }
    }
}

// ---------------------------------------------------------------------------------- sequences
// The rows of sequence b, held to the rows there are; `bad` where what the caller gave does not fit.
__device__ __forceinline__ void seq_rows(const qb200_sequences_t &s, int b, int &row, int &n, bool &bad)
{
    if (!s.offsets) {
        row = b;
        n = 1;
        bad = false;
        return;
    }
    const int lo = s.offsets[b], hi = s.offsets[b + 1];
    bad = lo < 0 || hi < lo || hi > s.rows;
    row = max(0, min(lo, s.rows));
    n = max(row, min(hi, s.rows)) - row;           // (whatever hi is, the difference stays inside 32 bits)
}

}  // namespace qb
