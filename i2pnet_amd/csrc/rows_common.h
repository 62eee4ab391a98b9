// Storage types of the row operators (rms_norm.hip, token_logprobs.hip, grad_norm.hip): fp32, bf16 and fp16 in memory, fp32 arithmetic.
#pragma once
#include "bf16_common.h"

__host__ __device__ constexpr int i2p_esize(int dtype) { return dtype == I2P_F32 ? 4 : 2; }

// one element
template <int DT> __device__ __forceinline__ float ld1(const void *p, long long i) {
    if constexpr (DT == I2P_F32) return reinterpret_cast<const float *>(p)[i];
    else if constexpr (DT == I2P_BF16) return __uint_as_float((unsigned)reinterpret_cast<const unsigned short *>(p)[i] << 16);
    else return (float)reinterpret_cast<const _Float16 *>(p)[i];
}
// the value `f` has once stored in DT (round to nearest even)
template <int DT> __device__ __forceinline__ float round1(float f) {
    if constexpr (DT == I2P_F32) return f;
    else if constexpr (DT == I2P_BF16) return bf_round(f);
    else return (float)(_Float16)f;
}
template <int DT> __device__ __forceinline__ void st1(void *p, long long i, float f) {
    if constexpr (DT == I2P_F32) reinterpret_cast<float *>(p)[i] = f;
    else if constexpr (DT == I2P_BF16) reinterpret_cast<unsigned short *>(p)[i] = (unsigned short)bf_pack2(f, 0.f);
    else reinterpret_cast<_Float16 *>(p)[i] = (_Float16)f;
}

// sum / maximum over the block's waves; every thread gets the result.  red: one float per wave.  (All threads of the block call it; the
// trailing barrier lets the caller use `red` again.)
template <bool MAX> __device__ __forceinline__ float block_reduce(float v, float *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const float u = __shfl_xor(v, o, 64); v = MAX ? fmaxf(v, u) : v + u; }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) t = MAX ? fmaxf(t, red[w]) : t + red[w];
    __syncthreads();
    return t;
}

// four bytes of OCP e4m3 (round to nearest even, saturating at +-448; NaN stays NaN)
__device__ __forceinline__ float e4m3_clamp(float v) { return v > 448.f ? 448.f : (v < -448.f ? -448.f : v); }
__device__ __forceinline__ unsigned e4m3_pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(a), e4m3_clamp(b), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(c), e4m3_clamp(d), v, true);
}
