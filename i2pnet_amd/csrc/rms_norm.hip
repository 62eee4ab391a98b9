// Root-mean-square norm of rows with the residual's addition, forward, backward and with an 8-bit output.
//
//   s = round(x + res)             the residual stream, kept in the inputs' type: the norm is of the stream as it is stored
//   rstd = 1 / sqrt(mean(s^2) + eps),  y = round(s * rstd * w)
//   8 bits: scale = max |s rstd w| / 448 over a group of columns (1 where the group is all zero), q = e4m3(s rstd w / scale)
//   backward, t = gy * w, xh = s * rstd:  dx = dres = round(rstd * (t - xh * mean(t * xh)) + gs),  dw = sum over rows of gy * xh
//
// Sums are fp32.  dw is summed per block over the rows it owns and then over the blocks in index order: reproducible.
#include "rows_common.h"

namespace {

constexpr int T = 256;

template <int DT, int WT, bool Q8>
__global__ __launch_bounds__(T) void rms_fwd_kernel(long long rows, int d, const void *__restrict__ x, long long ldx, const void *__restrict__ res,
                                                    long long ldr, const void *__restrict__ w, float eps, void *__restrict__ s,
                                                    void *__restrict__ y, float *__restrict__ rstd_out, int group, unsigned char *__restrict__ q,
                                                    float *__restrict__ scale) {
    __shared__ float red[T / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        float acc = 0.f;
        auto at = [&](int i) {
            float v = ld1<DT>(x, row * ldx + i);
            if (res) v = round1<DT>(v + ld1<DT>(res, row * ldr + i));
            return v;
        };
        for (int i = threadIdx.x; i < d; i += T) {
            const float v = at(i);
            if (s) st1<DT>(s, row * d + i, v);
            acc += v * v;
        }
        const float rstd = 1.f / sqrtf(block_reduce<false>(acc, red) / (float)d + eps);
        auto val = [&](int i) { return at(i) * rstd * (w ? ld1<WT>(w, i) : 1.f); };
        if constexpr (!Q8) {
            if (rstd_out && threadIdx.x == 0) rstd_out[row] = rstd;
            for (int i = threadIdx.x; i < d; i += T) st1<DT>(y, row * d + i, val(i));
        } else {
            const int width = group ? group : d, ng = (d + width - 1) / width;
            for (int g = 0; g < ng; ++g) {
                const int hi = min(d, (g + 1) * width);
                float m = 0.f;
                bool nan = false;
                for (int i = g * width + threadIdx.x; i < hi; i += T) { const float v = fabsf(val(i)); m = fmaxf(m, v); nan |= v != v; }
                m = block_reduce<true>(nan ? __builtin_inff() : m, red);
                float sc = m / 448.f;
                if (!(sc > 0.f)) sc = 1.f;
                if (threadIdx.x == 0) scale[row * ng + g] = sc;
                for (int i = g * width + threadIdx.x; i < hi; i += T) q[row * d + i] = (unsigned char)e4m3_pack4(val(i) / sc, 0.f, 0.f, 0.f);
            }
        }
    }
}

template <int DT, int WT>
__global__ __launch_bounds__(T) void rms_bwd_kernel(long long rows, int d, const void *__restrict__ s, long long lds, const void *__restrict__ gy,
                                                    long long ldg, const void *__restrict__ gs, long long ldgs, const void *__restrict__ w,
                                                    const float *__restrict__ rstd_in, void *__restrict__ dx, float *__restrict__ part) {
    __shared__ float red[T / 64];
    float *my = part ? part + (long long)blockIdx.x * d : nullptr;
    if (my)
        for (int i = threadIdx.x; i < d; i += T) my[i] = 0.f;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const float rstd = rstd_in[row];
        float acc = 0.f;
        for (int i = threadIdx.x; i < d; i += T) {
            const float xh = ld1<DT>(s, row * lds + i) * rstd, g = ld1<DT>(gy, row * ldg + i);
            acc += g * (w ? ld1<WT>(w, i) : 1.f) * xh;
            if (my) my[i] += g * xh;
        }
        const float mean = block_reduce<false>(acc, red) / (float)d;
        for (int i = threadIdx.x; i < d; i += T) {
            const float xh = ld1<DT>(s, row * lds + i) * rstd, t = ld1<DT>(gy, row * ldg + i) * (w ? ld1<WT>(w, i) : 1.f);
            float v = rstd * (t - xh * mean);
            if (gs) v += ld1<DT>(gs, row * ldgs + i);
            st1<DT>(dx, row * d + i, v);
        }
    }
}

template <int WT> __global__ __launch_bounds__(T) void rms_dw_kernel(int nblk, int d, const float *__restrict__ part, void *__restrict__ dw) {
    const int i = blockIdx.x * T + threadIdx.x;
    if (i >= d) return;
    float t = 0.f;
    for (int b = 0; b < nblk; ++b) t += part[(long long)b * d + i];
    st1<WT>(dw, i, t);
}

inline long long bwd_blocks(long long rows) { return rows < 512 ? rows : 512; }
inline bool types_ok(int dtype, int wdtype) {
    return dtype >= I2P_F32 && dtype <= I2P_F16 && (wdtype == I2P_F32 || wdtype == dtype);
}

// calls f(DT, WT) as integral constants
template <class F> void by_type(int dtype, int wdtype, F f) {
    using std::integral_constant;
    if (dtype == I2P_F32) f(integral_constant<int, I2P_F32>{}, integral_constant<int, I2P_F32>{});
    else if (dtype == I2P_BF16) {
        if (wdtype == I2P_F32) f(integral_constant<int, I2P_BF16>{}, integral_constant<int, I2P_F32>{});
        else f(integral_constant<int, I2P_BF16>{}, integral_constant<int, I2P_BF16>{});
    } else {
        if (wdtype == I2P_F32) f(integral_constant<int, I2P_F16>{}, integral_constant<int, I2P_F32>{});
        else f(integral_constant<int, I2P_F16>{}, integral_constant<int, I2P_F16>{});
    }
}

}  // namespace

extern "C" int i2p_rms_norm_fwd(long long rows, int d, int dtype, int wdtype, const void *x, long long ldx, const void *res, long long ldr,
                                const void *w, float eps, void *s, void *y, float *rstd, void *stream) {
    if (rows < 0 || d <= 0 || !types_ok(dtype, wdtype) || ldx < d || (res && ldr < d) || (res != nullptr) != (s != nullptr)) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !y) return I2P_ERR_BAD_ARG;
    const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : (1 << 20));
    by_type(dtype, wdtype, [&](auto dt, auto wt) {
        hipLaunchKernelGGL((rms_fwd_kernel<dt.value, wt.value, false>), dim3(grid), dim3(T), 0, (hipStream_t)stream, rows, d, x, ldx, res, ldr, w,
                           eps, s, y, rstd, 0, (unsigned char *)nullptr, (float *)nullptr);
    });
    I2P_RETURN_LAUNCH_STATUS();
}

extern "C" int i2p_rms_norm_q8(long long rows, int d, int dtype, int wdtype, const void *x, long long ldx, const void *res, long long ldr,
                               const void *w, float eps, int group, void *s, unsigned char *q, float *scale, void *stream) {
    if (rows < 0 || d <= 0 || !types_ok(dtype, wdtype) || ldx < d || (res && ldr < d) || (res != nullptr) != (s != nullptr)) return I2P_ERR_BAD_ARG;
    if (group != 0 && (group < 32 || group > 512 || (group & (group - 1)))) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return I2P_ERR_BAD_ARG;
    const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : (1 << 20));
    by_type(dtype, wdtype, [&](auto dt, auto wt) {
        hipLaunchKernelGGL((rms_fwd_kernel<dt.value, wt.value, true>), dim3(grid), dim3(T), 0, (hipStream_t)stream, rows, d, x, ldx, res, ldr, w,
                           eps, s, (void *)nullptr, (float *)nullptr, group, q, scale);
    });
    I2P_RETURN_LAUNCH_STATUS();
}

extern "C" long long i2p_rms_norm_bwd_scratch(long long rows, int d) { return rows <= 0 || d <= 0 ? 0 : bwd_blocks(rows) * d * 4; }

extern "C" int i2p_rms_norm_bwd(long long rows, int d, int dtype, int wdtype, const void *s, long long lds, const void *gy, long long ldgy,
                                const void *gs, long long ldgs, const void *w, const float *rstd, void *dx, void *dw, void *scratch, void *stream) {
    if (rows <= 0 || d <= 0 || !types_ok(dtype, wdtype) || lds < d || ldgy < d || (gs && ldgs < d)) return I2P_ERR_BAD_ARG;
    if (!s || !gy || !rstd || !dx || (dw && !scratch)) return I2P_ERR_BAD_ARG;
    const int nblk = (int)bwd_blocks(rows);
    float *part = dw ? (float *)scratch : nullptr;
    by_type(dtype, wdtype, [&](auto dt, auto wt) {
        hipLaunchKernelGGL((rms_bwd_kernel<dt.value, wt.value>), dim3(nblk), dim3(T), 0, (hipStream_t)stream, rows, d, s, lds, gy, ldgy, gs, ldgs,
                           w, rstd, dx, part);
        if (dw)
            hipLaunchKernelGGL((rms_dw_kernel<wt.value>), dim3((d + T - 1) / T), dim3(T), 0, (hipStream_t)stream, nblk, d, part, dw);
    });
    I2P_RETURN_LAUNCH_STATUS();
}
