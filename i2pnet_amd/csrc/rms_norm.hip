// Root-mean-square norm of rows with the residual's addition, forward, backward and with an 8-bit output.
//
//   s = round(x + res)             the residual stream, kept in the inputs' type: the norm is of the stream as it is stored
//   rstd = 1 / sqrt(mean(s^2) + eps),  y = round(s * rstd * w)
//   8 bits: scale = max |s rstd w| / 448 over a group of columns (1 where that quotient is 0), q = e4m3(s rstd w / scale)
//   backward, t = gy * w, xh = s * rstd:  dx = dres = round(rstd * (t - xh * mean(t * xh)) + gs),  dw = sum over rows of gy * xh
//
// Sums are fp32.  Where the sum of squares passes fp32 (values of 1e19 and more), or would lose digits below it and eps does not cover that
// (values of 1e-12 and less with an eps below 1e-24), it is formed again from scaled values.
//
// All of it is bound by memory: a row lives in the registers of the TPR threads that share it (NV 16-byte vectors each, the 16-bit types
// packed), so every input is read once and every output written once.  Short rows are shared by 16 lanes or one wave (no barrier, several
// rows per block), longer ones by a block of 256 to 1024.  dw is summed per block over the rows it owns (fp32 registers),
// then over the blocks in index order: reproducible.
// 8192 x 4096 bf16 with residual: forward 45 us (6.0 TB/s, part of it from the last-level cache), backward 58 us (4.6 TB/s) and 4.6 for dw;
// 6001 x 5000 to 8 bits 48 us (4.4 TB/s); 28800 x 64 fp32 7.7, 7.1 and 3.6 us; one row of 4096 2.6 us.
// Not of that form: rows of more than 4096 vectors, and fp32 rows of more than 256 columns in groups of 512 (two waves' vectors), are walked
// by a block, one element a thread, and read twice (three times to 8 bits).  The backward of 16-bit rows of more than 16384 columns keeps its
// four vectors a thread, with their weight gradients, partly in scratch memory (80 registers).
#include "rows_common.h"
#include <algorithm>

namespace {

constexpr int DW_COLS = 32, DW_LANES = 32;      // dw reduction: columns and row lanes of a block

// sum (or maximum of non-negative values' bits) over the TPR threads of a row; every one gets it.  A block-wide row uses red[waves]; calls
// alternate between two such arrays, so that one barrier each is enough
template <int TPR, class Op> __device__ __forceinline__ unsigned row_reduce(unsigned v, unsigned *red, Op op) {
    v = lanes_reduce<(TPR < 64 ? TPR : 64)>(v, op);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) v = op(v, red[w]);
    }
    return v;
}
template <int TPR> __device__ __forceinline__ float row_sum(float v, unsigned *red) {
    return __uint_as_float(row_reduce<TPR>(__float_as_uint(v), red, AddF{}));
}

// the weights of a vector of columns (ones where there is no weight)
template <int DT, bool TINY> __device__ __forceinline__ void ld_weight(const void *w, int wdtype, const Col<DT, TINY> &c, int d, float (&f)[i2p_vec(DT)]) {
    constexpr int VE = i2p_vec(DT);
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = 1.f;
    if (!w || !c.in) return;
    if (wdtype == DT) unpack<DT>(c.load((const char *)w, d), f);
    else if (!TINY) {                            // fp32 weights of a 16-bit row: two vectors
        float4 a[2];
        __builtin_memcpy(a, (const float *)w + c.at, 4 * VE);
        f[0] = a[0].x; f[1] = a[0].y; f[2] = a[0].z; f[3] = a[0].w;
        if constexpr (VE == 8) { f[4] = a[1].x; f[5] = a[1].y; f[6] = a[1].z; f[7] = a[1].w; }
    } else
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (c.at + e < d) f[e] = ((const float *)w)[c.at + e];
}

// Rows of d <= 2^26 whose squares fp32 does not hold are summed again from their values times `by`:
//   2^-80 where the sum is inf: squares below 1e29, and a value whose own is lost does not count beside the others.  (A value inf: rstd 0)
//   2^90 where mean + eps is at most 2^-80: a sum below 2^126, and squares of the smallest subnormal numbers are 2^-118
struct Far {
    float by;
    bool is;
    __device__ __forceinline__ Far(float sum, float var) : by(sum > 3.40282347e38f ? 0x1p-80f : 0x1p90f), is(sum > 3.40282347e38f || var <= 0x1p-80f) {}
    __device__ __forceinline__ float rstd(float sum, int d, float eps) const { return by / sqrtf(sum / (float)d + eps * by * by); }
};

struct FwdArgs {
    long long rows; int d, wdtype; const char *x; long long ldx; const char *res; long long ldr; const void *w; float eps; char *s, *y;
    float *rstd; int group; unsigned char *q; float *scale;
};

__device__ __forceinline__ float scale_of(unsigned bits) {
    if (bits > 0x7f7fffffu) return __builtin_inff();
    const float sc = __uint_as_float(bits) / 448.f;
    return sc == 0.f ? 1.f : sc;
}
// v / sc = v * up * inv: the reciprocal of a scale below the smallest normal number may pass fp32, so both are taken 2^64 higher
struct Divide {
    float up, inv;
    bool small;
    __device__ __forceinline__ explicit Divide(float sc) : small(sc < 1.17549435e-38f) {
        up = small ? 0x1p64f : 1.f;
        inv = 1.f / (sc * up);
    }
    __device__ __forceinline__ float operator()(float v) const { return v * up * inv; }
};

template <int DT, int TPR, int NV, bool TINY, bool Q8>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, NV < 3 ? 8 : NV < 4 ? 6 : 4) void rms_fwd_kernel(FwdArgs a) {
    constexpr int VE = i2p_vec(DT), ES = i2p_esize(DT), BLOCK = TPR < 256 ? 256 : TPR;
    __shared__ unsigned red[TPR > 64 ? TPR / 64 : 1];
    __shared__ unsigned mred[TPR > 64 ? TPR / 64 : 1];
    const long long row = (long long)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
    if (TPR < BLOCK && row >= a.rows) return;                   // (a block-wide row always exists)
    const int t = threadIdx.x % TPR, d = a.d;
    auto col = [&](int j) { return Col<DT, TINY>(j * TPR + t, d); };
    const char *x = a.x + row * a.ldx * ES;
    uint4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = col(j).load(x, d);
    if (a.res) {
        const char *r = a.res + row * a.ldr * ES;
        uint4 u[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) u[j] = col(j).load(r, d);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE], g[VE];
            unpack<DT>(v[j], f); unpack<DT>(u[j], g);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] += g[e];
            v[j] = pack<DT>(f);
            col(j).store(a.s + row * d * ES, d, v[j]);
        }
    }
    float acc = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float f[VE];
        unpack<DT>(v[j], f);
        const Col<DT, TINY> c = col(j);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc += e >= c.skip ? f[e] * f[e] : 0.f;        // (what is past the row was read as 0)
    }
    acc = row_sum<TPR>(acc, red);
    const float var = acc / (float)d + a.eps;
    float rstd = 1.f / sqrtf(var);
    const Far far(acc, var);
    if (__builtin_expect(far.is, 0)) {                          // (the row's threads agree)
        acc = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE];
            unpack<DT>(v[j], f);
            const Col<DT, TINY> c = col(j);
#pragma unroll
            for (int e = 0; e < VE; ++e) { const float g = f[e] * far.by; acc += e >= c.skip ? g * g : 0.f; }
        }
        if constexpr (TPR > 64) __syncthreads();                // (all have read `red`)
        rstd = far.rstd(row_sum<TPR>(acc, red), d, a.eps);
    }
    if constexpr (!Q8) {
        if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE], w[VE];
            unpack<DT>(v[j], f);
            ld_weight<DT>(a.w, a.wdtype, col(j), d, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] = f[e] * rstd * w[e];
            col(j).store(a.y + row * d * ES, d, pack<DT>(f));
        }
    } else {
        unsigned char *q = a.q + row * d;
        unsigned m[NV], all = 0u;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Col<DT, TINY> c = col(j);
            float f[VE], w[VE];
            unpack<DT>(v[j], f);
            ld_weight<DT>(a.w, a.wdtype, c, d, w);
            m[j] = 0u;
#pragma unroll
            for (int e = 0; e < VE; ++e) { const unsigned b = __float_as_uint(f[e] * rstd * w[e]) & 0x7fffffffu; if (c.counts(e, d) && b > m[j]) m[j] = b; }
            all = m[j] > all ? m[j] : all;
        }
        // a group of columns is a run of group / VE <= TPR lanes of one vector number, or the whole row
        const bool whole = !a.group || a.group >= TPR * NV * VE;
        const int lanes = whole ? 0 : a.group / VE, ng = whole ? 1 : (d + a.group - 1) / a.group;
        if (whole) all = row_reduce<TPR>(all, mred, MaxU{});
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Col<DT, TINY> c = col(j);
            unsigned b = all;
            if (!whole) {
                b = m[j];
                b = lanes == 64 ? lanes_reduce<64>(b, MaxU{}) : lanes == 32 ? lanes_reduce<32>(b, MaxU{}) : lanes == 16 ? lanes_reduce<16>(b, MaxU{})
                    : lanes == 8 ? lanes_reduce<8>(b, MaxU{}) : lanes_reduce<4>(b, MaxU{});
            }
            if (!c.in) continue;
            const float sc = scale_of(b);
            const Divide by(sc);
            if (whole ? (t | j) == 0 : (t & (lanes - 1)) == 0) a.scale[row * ng + (whole ? 0 : (j * TPR + t) * VE / a.group)] = sc;
            float f[VE], w[VE];
            unpack<DT>(v[j], f);
            ld_weight<DT>(a.w, a.wdtype, c, d, w);
            unsigned u[VE / 4];
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] = f[e] * rstd * w[e];
            if (by.small)
#pragma unroll
                for (int e = 0; e < VE; ++e) f[e] *= by.up;
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] *= by.inv;
#pragma unroll
            for (int k = 0; k < VE / 4; ++k) u[k] = e4m3_pack4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
            if (!c.skip && c.at + VE <= d) __builtin_memcpy(q + c.at, u, VE);
            else {                               // (the elements before may belong to another group)
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (c.counts(e, d)) q[c.at + e] = (unsigned char)(u[e >> 2] >> (8 * (e & 3)));
            }
        }
    }
}

struct BwdArgs {
    long long rows; int d, wdtype; const char *s; long long lds; const char *gy; long long ldg; const char *gs; long long ldgs; const void *w;
    const float *rstd; char *dx; float *part;
};

// Every group of TPR threads walks rows in steps of the grid
template <int DT, int TPR, int NV, bool TINY>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_bwd_kernel(BwdArgs a) {
    constexpr int VE = i2p_vec(DT), ES = i2p_esize(DT), BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
    __shared__ unsigned red[2][TPR > 64 ? TPR / 64 : 1];
    __shared__ float cols[RPB > 1 ? BLOCK * VE : 1];
    const int t = threadIdx.x % TPR, d = a.d;
    auto col = [&](int j) { return Col<DT, TINY>(j * TPR + t, d); };
    const long long step = (long long)gridDim.x * RPB;
    float dw[NV][VE] = {};
    int flip = 0;
    for (long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += step, flip ^= 1) {
        uint4 xs[NV], gg[NV], ex[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            xs[j] = col(j).load(a.s + row * a.lds * ES, d);
            gg[j] = col(j).load(a.gy + row * a.ldg * ES, d);
            if (a.gs) ex[j] = col(j).load(a.gs + row * a.ldgs * ES, d);
        }
        const float rstd = a.rstd[row];
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Col<DT, TINY> c = col(j);
            float f[VE], g[VE], w[VE];
            unpack<DT>(xs[j], f); unpack<DT>(gg[j], g);
            ld_weight<DT>(a.w, a.wdtype, c, d, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) { const float p = g[e] * (f[e] * rstd); dw[j][e] += p; acc += e >= c.skip ? p * w[e] : 0.f; }
        }
        const float mean = row_sum<TPR>(acc, red[flip]) / (float)d;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE], g[VE], w[VE], h[VE] = {};
            unpack<DT>(xs[j], f); unpack<DT>(gg[j], g);
            if (a.gs) unpack<DT>(ex[j], h);
            ld_weight<DT>(a.w, a.wdtype, col(j), d, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] = rstd * (g[e] * w[e] - f[e] * rstd * mean) + h[e];
            col(j).store(a.dx + row * d * ES, d, pack<DT>(f));
        }
    }
    if (!a.part) return;
    float *out = a.part + (long long)blockIdx.x * d;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if constexpr (RPB > 1) {                 // the block's groups, summed in order
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VE; ++e) cols[threadIdx.x * VE + e] = dw[j][e];
            __syncthreads();
            if (threadIdx.x < TPR) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    float v = 0.f;
                    for (int g = 0; g < RPB; ++g) v += cols[(g * TPR + t) * VE + e];
                    dw[j][e] = v;
                }
            }
        }
        if (RPB == 1 || threadIdx.x < TPR) {
            const Col<DT, TINY> c = col(j);
            if (c.in && !c.skip && c.at + VE <= d) __builtin_memcpy(out + c.at, dw[j], 4 * VE);
            else
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (c.counts(e, d)) out[c.at + e] = dw[j][e];
        }
    }
}

__global__ __launch_bounds__(DW_COLS * DW_LANES) void rms_dw_kernel(int nblk, int d, const float *__restrict__ part, void *__restrict__ dw, int wdtype) {
    __shared__ float sum[DW_LANES][DW_COLS + 1];
    const int c = threadIdx.x % DW_COLS, l = threadIdx.x / DW_COLS, i = blockIdx.x * DW_COLS + c;
    float v = 0.f;
    if (i < d)
        for (int b = l; b < nblk; b += 16 * DW_LANES) {          // 16 loads in flight
#pragma unroll
            for (int u = 0; u < 16; ++u) { const int k = b + u * DW_LANES; v += k < nblk ? part[(long long)k * d + i] : 0.f; }
        }
    sum[l][c] = v;
    __syncthreads();
    if (l || i >= d) return;
    for (int k = 1; k < DW_LANES; ++k) v += sum[k][c];
    if (wdtype == I2P_F32) st1<I2P_F32>(dw, i, v);
    else if (wdtype == I2P_BF16) st1<I2P_BF16>(dw, i, v);
    else st1<I2P_F16>(dw, i, v);
}

// ---- rows longer than the registers of a block: 1024 threads walk them, reading twice --------------------------------------------------
constexpr int LT = 1024;

__device__ __forceinline__ float weight1(const void *w, int wdtype, int i) {
    return !w ? 1.f : wdtype == I2P_F32 ? ld1<I2P_F32>(w, i) : wdtype == I2P_BF16 ? ld1<I2P_BF16>(w, i) : ld1<I2P_F16>(w, i);
}

template <int DT, bool Q8> __global__ __launch_bounds__(LT) void rms_fwd_long_kernel(FwdArgs a) {
    constexpr int ES = i2p_esize(DT);
    __shared__ float red[LT / 64];
    const int d = a.d;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const char *x = a.x + row * a.ldx * ES, *r = a.res + row * a.ldr * ES;
        auto at = [&](int i) {
            float v = ld1<DT>(x, i);
            if (a.res) v = round1<DT>(v + ld1<DT>(r, i));
            return v;
        };
        float acc = 0.f;
        for (int i = threadIdx.x; i < d; i += LT) {
            const float v = at(i);
            if (a.s) st1<DT>(a.s, row * d + i, v);
            acc += v * v;
        }
        acc = block_total(acc, red);
        const float var = acc / (float)d + a.eps;
        float rstd = 1.f / sqrtf(var);
        const Far far(acc, var);
        if (far.is) {
            acc = 0.f;
            for (int i = threadIdx.x; i < d; i += LT) { const float v = at(i) * far.by; acc += v * v; }
            rstd = far.rstd(block_total(acc, red), d, a.eps);
        }
        auto val = [&](int i) { return at(i) * rstd * weight1(a.w, a.wdtype, i); };
        if constexpr (!Q8) {
            if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
            for (int i = threadIdx.x; i < d; i += LT) st1<DT>(a.y, row * d + i, val(i));
        } else if (a.group) {                    // a wave per group
            const int ng = (d + a.group - 1) / a.group, lane = threadIdx.x & 63;
            for (int g = threadIdx.x >> 6; g < ng; g += LT / 64) {
                const int hi = min(d, (g + 1) * a.group);
                unsigned m = 0u;
                for (int i = g * a.group + lane; i < hi; i += 64) { const unsigned b = __float_as_uint(val(i)) & 0x7fffffffu; m = b > m ? b : m; }
                m = row_reduce<64>(m, (unsigned *)nullptr, MaxU{});
                const float sc = scale_of(m);
                const Divide by(sc);
                if (lane == 0) a.scale[row * ng + g] = sc;
                for (int i = g * a.group + lane; i < hi; i += 64) a.q[row * d + i] = (unsigned char)e4m3_pack4(by(val(i)), 0.f, 0.f, 0.f);
            }
        } else {
            unsigned m = 0u;
            for (int i = threadIdx.x; i < d; i += LT) { const unsigned b = __float_as_uint(val(i)) & 0x7fffffffu; m = b > m ? b : m; }
            __syncthreads();
            m = row_reduce<LT>(m, (unsigned *)red, MaxU{});
            const float sc = scale_of(m);
            const Divide by(sc);
            if (threadIdx.x == 0) a.scale[row] = sc;
            for (int i = threadIdx.x; i < d; i += LT) a.q[row * d + i] = (unsigned char)e4m3_pack4(by(val(i)), 0.f, 0.f, 0.f);
            __syncthreads();
        }
    }
}

template <int DT> __global__ __launch_bounds__(LT) void rms_bwd_long_kernel(BwdArgs a) {
    constexpr int ES = i2p_esize(DT);
    __shared__ float red[LT / 64];
    const int d = a.d;
    float *my = a.part ? a.part + (long long)blockIdx.x * d : nullptr;
    if (my)
        for (int i = threadIdx.x; i < d; i += LT) my[i] = 0.f;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const char *s = a.s + row * a.lds * ES, *gy = a.gy + row * a.ldg * ES, *gs = a.gs + row * a.ldgs * ES;
        const float rstd = a.rstd[row];
        float acc = 0.f;
        for (int i = threadIdx.x; i < d; i += LT) {
            const float c = ld1<DT>(gy, i) * (ld1<DT>(s, i) * rstd);
            acc += c * weight1(a.w, a.wdtype, i);
            if (my) my[i] += c;
        }
        const float mean = block_total(acc, red) / (float)d;
        for (int i = threadIdx.x; i < d; i += LT) {
            float v = rstd * (ld1<DT>(gy, i) * weight1(a.w, a.wdtype, i) - ld1<DT>(s, i) * rstd * mean);
            if (a.gs) v += ld1<DT>(gs, i);
            st1<DT>(a.dx, row * d + i, v);
        }
    }
}

inline bool types_ok(int dtype, int wdtype) {
    return dtype >= I2P_F32 && dtype <= I2P_F16 && (wdtype == I2P_F32 || wdtype == dtype);
}

// Blocks of the backward pass for `rows` rows (or runs of rows) of a block of `threads`: as many as run at once (four waves a SIMD), but no
// more than 2^21 partial weight gradients, whose write and read cost as much as a row's (8192 x 4096 bf16: 512 blocks 63 us in both
// launches, 1024 67, 2048 70; 30000 x 1000: 512 blocks 65 us, 1024 51, 2048 55)
inline long long bwd_blocks(long long rows, int d, int threads) {
    const long long most = std::min(262144ll / threads, std::max(256ll, (1ll << 21) / d));
    return std::min(rows, most);
}

// f(DT, TPR, NV) for rows of d elements; false: the row does not fit the registers of a block
template <int DT, bool BWD, class F> bool by_width(int d, F f) {
    using std::integral_constant;
    const long long n = ((long long)d + i2p_vec(DT) - 1) / i2p_vec(DT);
#define I2P_ROW(TPR, NV, TINY) \
    { f(integral_constant<int, DT>{}, integral_constant<int, TPR>{}, integral_constant<int, NV>{}, std::bool_constant<TINY>{}); return true; }
    if (d < i2p_vec(DT)) I2P_ROW(8, 1, true)
    if (n <= 8) I2P_ROW(8, 1, false)
    if (n <= 16) I2P_ROW(16, 1, false)
    if (n <= 32) I2P_ROW(16, 2, false)
    if (n <= 64) I2P_ROW(64, 1, false)
    if (n <= 128) I2P_ROW(64, 2, false)
    if (n <= 256) I2P_ROW(256, 1, false)
    if constexpr (BWD) {
        // the weight gradients double the registers of a vector: more threads with one vector each (8192 x 4096 bf16 as 256 x 2: 62 us,
        // 512 x 1: 58; 4000 x 8000 as 512 x 2: 85, 1024 x 1: 57), unless many of them would have none (15000 x 2100: 65, 74)
        if (n <= 384) I2P_ROW(256, 2, false)
        if (n <= 512) I2P_ROW(512, 1, false)
        if (n <= 1024) I2P_ROW(1024, 1, false)
    }
    if (n <= 512) I2P_ROW(256, 2, false)
    if (n <= 768) I2P_ROW(256, 3, false)
    if (n <= 1024) I2P_ROW(512, 2, false)
    if (n <= 2048) I2P_ROW(1024, 2, false)
    if (n <= 4096) I2P_ROW(1024, 4, false)
#undef I2P_ROW
    return false;
}
template <bool BWD, class F, class G> void by_row(int dtype, int d, F f, G longer, int group = 0) {
    // (512 columns of fp32 are two waves' vectors: such groups take the long-row kernel unless they cover the row)
    if (dtype == I2P_F32) { if ((group > 256 && d > 256) || !by_width<I2P_F32, BWD>(d, f)) longer(std::integral_constant<int, I2P_F32>{}); }
    else if (dtype == I2P_BF16) { if (!by_width<I2P_BF16, BWD>(d, f)) longer(std::integral_constant<int, I2P_BF16>{}); }
    else if (!by_width<I2P_F16, BWD>(d, f)) longer(std::integral_constant<int, I2P_F16>{});
}

template <bool Q8> int launch_fwd(int dtype, const FwdArgs &a, void *stream) {
    by_row<false>(dtype, a.d, [&](auto dt, auto tpr, auto nv, auto tiny) {
        constexpr int BLOCK = tpr.value < 256 ? 256 : tpr.value, RPB = BLOCK / tpr.value;
        constexpr long long MOST = 1ll << 21;                   // blocks of a launch: a grid has fewer than 2^32 threads
        const long long es = i2p_esize(dt.value), ng = a.group ? (a.d + a.group - 1) / a.group : 1;
        for (long long r = 0; r < a.rows; r += MOST * RPB) {
            FwdArgs b = a;
            b.rows = a.rows - r < MOST * RPB ? a.rows - r : MOST * RPB;
            b.x += r * a.ldx * es;
            if (a.res) { b.res += r * a.ldr * es; b.s += r * a.d * es; }
            if (a.y) b.y += r * a.d * es;
            if (a.rstd) b.rstd += r;
            if (a.q) { b.q += r * a.d; b.scale += r * ng; }
            hipLaunchKernelGGL((rms_fwd_kernel<dt.value, tpr.value, nv.value, tiny.value, Q8>), dim3((unsigned)((b.rows + RPB - 1) / RPB)), dim3(BLOCK), 0,
                               (hipStream_t)stream, b);
        }
    }, [&](auto dt) {
        hipLaunchKernelGGL((rms_fwd_long_kernel<dt.value, Q8>), dim3((unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20))), dim3(LT), 0,
                           (hipStream_t)stream, a);
    }, a.group);
    I2P_RETURN_LAUNCH_STATUS();
}

}  // namespace

extern "C" int i2p_rms_norm_fwd(long long rows, int d, int dtype, int wdtype, const void *x, long long ldx, const void *res, long long ldr,
                                const void *w, float eps, void *s, void *y, float *rstd, void *stream) {
    if (rows < 0 || d <= 0 || d > I2P_MAX_ROW || !types_ok(dtype, wdtype) || ldx < d || (res && ldr < d) || (res != nullptr) != (s != nullptr)) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !y) return I2P_ERR_BAD_ARG;
    return launch_fwd<false>(dtype, FwdArgs{rows, d, wdtype, (const char *)x, ldx, (const char *)res, ldr, w, eps, (char *)s, (char *)y, rstd, 0,
                                            nullptr, nullptr}, stream);
}

extern "C" int i2p_rms_norm_q8(long long rows, int d, int dtype, int wdtype, const void *x, long long ldx, const void *res, long long ldr,
                               const void *w, float eps, int group, void *s, unsigned char *q, float *scale, void *stream) {
    if (rows < 0 || d <= 0 || d > I2P_MAX_ROW || !types_ok(dtype, wdtype) || ldx < d || (res && ldr < d) || (res != nullptr) != (s != nullptr)) return I2P_ERR_BAD_ARG;
    if (group != 0 && (group < 32 || group > 512 || (group & (group - 1)))) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return I2P_ERR_BAD_ARG;
    return launch_fwd<true>(dtype, FwdArgs{rows, d, wdtype, (const char *)x, ldx, (const char *)res, ldr, w, eps, (char *)s, nullptr, nullptr, group,
                                           q, scale}, stream);
}

extern "C" long long i2p_rms_norm_bwd_scratch(long long rows, int d) { return rows <= 0 || d <= 0 ? 0 : bwd_blocks(rows, d, 256) * d * 4; }

extern "C" int i2p_rms_norm_bwd(long long rows, int d, int dtype, int wdtype, const void *s, long long lds, const void *gy, long long ldgy,
                                const void *gs, long long ldgs, const void *w, const float *rstd, void *dx, void *dw, void *scratch, void *stream) {
    if (rows <= 0 || d <= 0 || d > I2P_MAX_ROW || !types_ok(dtype, wdtype) || lds < d || ldgy < d || (gs && ldgs < d)) return I2P_ERR_BAD_ARG;
    if (!s || !gy || !rstd || !dx || (dw && (!scratch || ((uintptr_t)scratch & 15)))) return I2P_ERR_BAD_ARG;
    const BwdArgs a{rows, d, wdtype, (const char *)s, lds, (const char *)gy, ldgy, (const char *)gs, ldgs, w, rstd, (char *)dx,
                    dw ? (float *)scratch : nullptr};
    long long nblk = 0;
    by_row<true>(dtype, d, [&](auto dt, auto tpr, auto nv, auto tiny) {
        constexpr int BLOCK = tpr.value < 256 ? 256 : tpr.value, RPB = BLOCK / tpr.value;
        nblk = bwd_blocks((rows + RPB - 1) / RPB, d, BLOCK);
        hipLaunchKernelGGL((rms_bwd_kernel<dt.value, tpr.value, nv.value, tiny.value>), dim3((unsigned)nblk), dim3(BLOCK), 0, (hipStream_t)stream, a);
    }, [&](auto dt) {
        nblk = bwd_blocks(rows, d, LT);
        hipLaunchKernelGGL((rms_bwd_long_kernel<dt.value>), dim3((unsigned)nblk), dim3(LT), 0, (hipStream_t)stream, a);
    });
    if (dw)
        hipLaunchKernelGGL(rms_dw_kernel, dim3((unsigned)((d + DW_COLS - 1) / DW_COLS)), dim3(DW_COLS * DW_LANES), 0, (hipStream_t)stream, (int)nblk, d,
                           a.part, dw, wdtype);
    I2P_RETURN_LAUNCH_STATUS();
}
