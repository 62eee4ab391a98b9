// Storage types of the row operators (rms_norm.hip, token_logprobs.hip, grad_norm.hip): fp32, bf16 and fp16 in memory, fp32 arithmetic.
//
// Rows are read and written in 16-byte vectors wherever they start: the hardware takes 16-byte accesses at any element's address.
#pragma once
#include "bf16_common.h"

__host__ __device__ constexpr int i2p_esize(int dtype) { return dtype == I2P_F32 ? 4 : 2; }
__host__ __device__ constexpr int i2p_vec(int dtype) { return 16 / i2p_esize(dtype); }       // elements of a vector

typedef _Float16 i2p_f16x2 __attribute__((ext_vector_type(2)));

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

// a vector's values and back (round to nearest even)
template <int DT> __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[i2p_vec(DT)]) {
    if constexpr (DT == I2P_F32) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
    else if constexpr (DT == I2P_BF16) bf_unpack8(v, f);
    else {
        const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) { const i2p_f16x2 h = __builtin_bit_cast(i2p_f16x2, u[k]); f[2 * k] = (float)h.x; f[2 * k + 1] = (float)h.y; }
    }
}
template <int DT> __device__ __forceinline__ uint4 pack(const float (&f)[i2p_vec(DT)]) {
    if constexpr (DT == I2P_F32) return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else if constexpr (DT == I2P_BF16) return bf_pack8(f);
    else {
        unsigned u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) { const i2p_f16x2 h = {(_Float16)f[2 * k], (_Float16)f[2 * k + 1]}; u[k] = __builtin_bit_cast(unsigned, h); }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// Vector number `n` of a row of `d` elements.  The last, partial one is moved back so that it ends with the row: it reads and writes whole,
// its first `skip` elements are the previous vector's (the same values, written twice), and are left out of sums.  A row shorter than a
// vector (TINY) is read and written element by element instead.
template <int DT, bool TINY = false> struct Col {
    static constexpr int VE = i2p_vec(DT), ES = i2p_esize(DT);
    int at, skip;
    bool in;
    __device__ __forceinline__ Col(int n, int d) {
        const int i = n * VE;
        in = i < d;
        at = TINY ? i : min(i, d - VE);
        skip = TINY ? 0 : i - at;
    }
    __device__ __forceinline__ uint4 load(const char *row, int d, unsigned fill = 0u) const {
        uint4 v = make_uint4(fill, fill, fill, fill);
        if (!in) return v;
        if (!TINY || at + VE <= d) __builtin_memcpy(&v, row + (long long)at * ES, 16);
        else {
            unsigned u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (at + e < d) {
                    if constexpr (ES == 4) u[e] = reinterpret_cast<const unsigned *>(row)[at + e];
                    else u[e >> 1] |= (unsigned)reinterpret_cast<const unsigned short *>(row)[at + e] << (16 * (e & 1));
                }
            v = make_uint4(u[0], u[1], u[2], u[3]);
        }
        return v;
    }
    __device__ __forceinline__ void store(char *row, int d, const uint4 &v) const {
        if (!in) return;
        if (!TINY || at + VE <= d) __builtin_memcpy(row + (long long)at * ES, &v, 16);
        else {
            const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (at + e < d) {
                    if constexpr (ES == 4) reinterpret_cast<unsigned *>(row)[at + e] = u[e];
                    else reinterpret_cast<unsigned short *>(row)[at + e] = (unsigned short)(u[e >> 1] >> (16 * (e & 1)));
                }
        }
    }
    // the same past the caches (a whole vector of a row that is aligned)
    __device__ __forceinline__ void store_stream(char *row, const uint4 &v) const { if (in) st_u4_stream(row + (long long)at * ES, v); }
    // does element `e` of the vector count (is it the row's, and not the previous vector's)?
    __device__ __forceinline__ bool counts(int e, int d) const { return in && e >= skip && (!TINY || at + e < d); }
};

// Butterfly reduction over groups of N = 2 .. 64 lanes; every lane gets the same bits.  Register moves only (DPP inside a row of 16 lanes, the
// lane swaps of gfx950 above): a reduction through ds_bpermute is some thirty instructions and six LDS round trips
template <int N, class Op> __device__ __forceinline__ unsigned lanes_reduce(unsigned v, Op op) {
    if constexpr (N >= 2) v = op(v, i2p_dpp_u32<0xB1>(v));
    if constexpr (N >= 4) v = op(v, i2p_dpp_u32<0x4E>(v));
    if constexpr (N >= 8) v = op(v, i2p_dpp_u32<0x141>(v));
    if constexpr (N >= 16) v = op(v, i2p_dpp_u32<0x140>(v));
    if constexpr (N >= 32) { const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false); v = op(r[0], r[1]); }
    if constexpr (N >= 64) { const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false); v = op(r[0], r[1]); }
    return v;
}
struct AddF { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); } };
struct MaxF { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); } };
struct MaxU { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; } };
template <int N> __device__ __forceinline__ float lanes_sum(float v) { return __uint_as_float(lanes_reduce<N>(__float_as_uint(v), AddF{})); }
template <int N> __device__ __forceinline__ float lanes_max(float v) { return __uint_as_float(lanes_reduce<N>(__float_as_uint(v), MaxF{})); }

// sum over the block's waves; every thread gets the result.  red: one float per wave.  (All threads of the block call it; the trailing barrier
// lets the caller use `red` again.)
__device__ __forceinline__ float block_total(float v, float *red) {
    v = lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) t += red[w];
    __syncthreads();
    return t;
}

// four bytes of OCP e4m3 (round to nearest even, saturating at +-448; NaN stays NaN)
__device__ __forceinline__ float e4m3_clamp(float v) { return v > 448.f ? 448.f : (v < -448.f ? -448.f : v); }
__device__ __forceinline__ unsigned e4m3_pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(a), e4m3_clamp(b), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(c), e4m3_clamp(d), v, true);
}
