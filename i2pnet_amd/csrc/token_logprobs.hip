// Log probabilities of given candidates of a row of scores, with the row's entropy and its best alternatives, and the gradient.
//
//   z = x - max,  S = sum e^z,  L = log S:   logp = z[id] - L,   H = L - (sum z e^z) / S,   top = the k largest, equal ones by lower index
//   dx_j = g_logp (delta_j,id - p_j) - g_H p_j (log p_j + H),   p_j = e^(z_j - L)
//
// The maximum and L are kept apart for the backward pass: rounded into one number, scores of a few hundred would lose the digits of L.
// A row without candidates (all -inf): logp -inf, H 0, gradient 0.  +inf or NaN in a row: logp, H, top_logp and the gradient are NaN.
#include "rows_common.h"

namespace {

constexpr int T = 256;

// order of the alternatives: by value, NaN above +inf, -0 equal to +0; then by lower index.  0 is below every key
__device__ __forceinline__ unsigned order_of(float x) {
    x += 0.f;
    if (x != x) return 0xffc00000u;
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ unsigned long long key_of(float x, unsigned col) { return ((unsigned long long)order_of(x) << 32) | (0xffffffffu - col); }

__device__ __forceinline__ float shift_of(float m) { return m == -__builtin_inff() ? 0.f : m; }
// z e^z with 0 in the limit z -> -inf
__device__ __forceinline__ float z_exp(float z, float e) { return fmaxf(z, -200.f) * e; }      // (e^-200 is 0)

template <int DT>
__global__ __launch_bounds__(T) void logprobs_fwd_kernel(long long rows, int v, const void *__restrict__ x, long long ldx,
                                                         const int64_t *__restrict__ ids, long long ignore, int top, float *__restrict__ logp,
                                                         float *__restrict__ entropy, float *__restrict__ stat, float *__restrict__ top_logp,
                                                         int64_t *__restrict__ top_ids) {
    __shared__ float red[T / 64];
    __shared__ unsigned long long kred[T / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long long id = ids[row], base = row * ldx;
        if (id == ignore) {
            if (threadIdx.x == 0) { logp[row] = 0.f; entropy[row] = 0.f; stat[2 * row] = 0.f; stat[2 * row + 1] = 0.f; }
            for (int k = threadIdx.x; k < top; k += T) { top_logp[row * top + k] = -__builtin_inff(); top_ids[row * top + k] = -1; }
            continue;
        }
        float m = -__builtin_inff();
        for (int i = threadIdx.x; i < v; i += T) m = fmaxf(m, ld1<DT>(x, base + i));
        m = block_reduce<true>(m, red);
        const float c = shift_of(m);
        float S = 0.f, U = 0.f;
        for (int i = threadIdx.x; i < v; i += T) { const float z = ld1<DT>(x, base + i) - c, e = __expf(z); S += e; U += z_exp(z, e); }
        S = block_reduce<false>(S, red);
        U = block_reduce<false>(U, red);
        const bool empty = S == 0.f;
        const float L = empty ? __builtin_inff() : logf(S);
        if (threadIdx.x == 0) {
            logp[row] = id < 0 || id >= v ? __builtin_nanf("") : (ld1<DT>(x, base + id) - c) - L;
            entropy[row] = empty ? 0.f : L - U / S;
            stat[2 * row] = c; stat[2 * row + 1] = L;
        }
        unsigned long long last = ~0ull;
        for (int k = 0; k < top; ++k) {
            unsigned long long best = 0;
            for (int i = threadIdx.x; i < v; i += T) { const unsigned long long key = key_of(ld1<DT>(x, base + i), i); if (key < last && key > best) best = key; }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) { const unsigned long long u = __shfl_xor(best, o, 64); best = u > best ? u : best; }
            if ((threadIdx.x & 63) == 0) kred[threadIdx.x >> 6] = best;
            __syncthreads();
#pragma unroll
            for (int wv = 0; wv < T / 64; ++wv) best = kred[wv] > best ? kred[wv] : best;
            __syncthreads();
            if (threadIdx.x == 0) {
                top_logp[row * top + k] = (value_of((unsigned)(best >> 32)) - c) - L;
                top_ids[row * top + k] = (int64_t)(0xffffffffu - (unsigned)best);
            }
            last = best;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(T) void logprobs_bwd_kernel(long long rows, int v, const void *__restrict__ x, long long ldx,
                                                         const int64_t *__restrict__ ids, long long ignore, const float *__restrict__ stat,
                                                         const float *__restrict__ entropy, const float *__restrict__ g_logp,
                                                         const float *__restrict__ g_entropy, void *__restrict__ dx) {
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long long id = ids[row];
        const bool skip = id == ignore;
        float gl = g_logp ? g_logp[row] : 0.f;
        const float gh = g_entropy ? g_entropy[row] : 0.f, H = entropy[row], c = stat[2 * row], L = stat[2 * row + 1];
        if (L == __builtin_inff()) gl = 0.f;                 // an empty row
        if (id < 0 || id >= v) gl = __builtin_nanf("");
        for (int i = threadIdx.x; i < v; i += T) {
            float g = 0.f;
            if (!skip) {
                const float lp = ld1<DT>(x, row * ldx + i) - c - L, p = __expf(lp);
                g = (i == id ? gl : 0.f) - p * (gl + gh * (fmaxf(lp, -200.f) + H));
            }
            st1<DT>(dx, row * v + i, g);
        }
    }
}

template <class F> void by_type(int dtype, F f) {
    if (dtype == I2P_F32) f(std::integral_constant<int, I2P_F32>{});
    else if (dtype == I2P_BF16) f(std::integral_constant<int, I2P_BF16>{});
    else f(std::integral_constant<int, I2P_F16>{});
}

}  // namespace

extern "C" long long i2p_token_logprobs_scratch(long long, int, int, int) { return 0; }

extern "C" int i2p_token_logprobs_fwd(long long rows, int v, int dtype, const void *x, long long ldx, const int64_t *ids, long long ignore, int top,
                                      float *logp, float *entropy, float *stat, float *top_logp, int64_t *top_ids, void *scratch,
                                      void *stream) {
    if (rows < 0 || v <= 0 || v > I2P_MAX_CANDIDATES || dtype < I2P_F32 || dtype > I2P_F16 || ldx < v || top < 0 || top > v || top > I2P_MAX_TOP) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !ids || !logp || !entropy || !stat || (top && (!top_logp || !top_ids))) return I2P_ERR_BAD_ARG;
    const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : (1 << 20));
    by_type(dtype, [&](auto dt) {
        hipLaunchKernelGGL((logprobs_fwd_kernel<dt.value>), dim3(grid), dim3(T), 0, (hipStream_t)stream, rows, v, x, ldx, ids, ignore, top, logp,
                           entropy, stat, top_logp, top_ids);
    });
    I2P_RETURN_LAUNCH_STATUS();
}

extern "C" int i2p_token_logprobs_bwd(long long rows, int v, int dtype, const void *x, long long ldx, const int64_t *ids, long long ignore,
                                      const float *stat, const float *entropy, const float *g_logp, const float *g_entropy, void *dx, void *stream) {
    if (rows < 0 || v <= 0 || v > I2P_MAX_CANDIDATES || dtype < I2P_F32 || dtype > I2P_F16 || ldx < v) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !ids || !stat || !entropy || !dx) return I2P_ERR_BAD_ARG;
    const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : (1 << 20));
    by_type(dtype, [&](auto dt) {
        hipLaunchKernelGGL((logprobs_bwd_kernel<dt.value>), dim3(grid), dim3(T), 0, (hipStream_t)stream, rows, v, x, ldx, ids, ignore, stat, entropy,
                           g_logp, g_entropy, dx);
    });
    I2P_RETURN_LAUNCH_STATUS();
}
