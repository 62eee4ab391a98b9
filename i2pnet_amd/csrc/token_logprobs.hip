// Log probabilities of given candidates of a row of scores, with the row's entropy and its best alternatives, and the gradient.
//
//   z = x - max,  S = sum e^z,  L = log S:   logp = z[id] - L,   H = L - (sum z e^z) / S,   top = the k largest, equal ones by lower index
//   dx_j = g_logp (delta_j,id - p_j) - g_H p_j (log p_j + H),   p_j = e^(z_j - L)
//
// The maximum and L are kept apart for the backward pass: rounded into one number, scores of a few hundred would lose the digits of L.
// A row without candidates (all -inf): logp -inf, H 0, gradient 0.  +inf or NaN in a row: logp, H, top_logp and the gradient are NaN.
//
// Forward: reads the scores once.  A row of more than 128 scores, or a slice of a long one, stays in the registers of a wave, of 4 or of 16
// waves (at most 32 scores a thread, 64 of the 16-bit types), so that the maximum is known before the first exponential; slices leave (max, S,
// sum z e^z) and their k best in the workspace and a second launch joins them.  8192 x 131072 bf16: 430 .. 470 us, 4.6 .. 5.0 TB/s (a plain sum
// of that much reads 4.0 TB/s here), and 13 to join; a wave issues 715 vector instructions for 64 scores a lane, in 75 % of the cycles, and the
// exponentials among them take four times a slot.  4096 x 32000: 58 + 6 us; a wave's fixed part weighs more in shorter slices (387 for 28 scores a lane).
// Best alternatives: the threads' maxima give 64 group maxima; the k-th largest of those (to 16 bits) is a value that at least k scores reach
// and that few others do.  The scores that reach it go to LDS and are ranked by counting.  Rows with many equal scores (or a NaN) overflow
// that list and are searched k times instead.  10000 x 2000 fp32: 15.2 us without alternatives, 20.0 with 8, 25.0 with 32; 777 x 50001 fp16:
// 22 + 4 us without, 26 + 5 with 5 (387 and 497 vector instructions a wave).
// Backward: elementwise from the saved maximum, L and H; bound by reading the scores again and writing as much: 8192 x 131072 bf16 755 us,
// 5.7 TB/s.
#include "rows_common.h"

namespace {

constexpr int LIST = 256;                       // scores ranked by counting

// order of the alternatives: by value, NaN above +inf, -0 equal to +0; then by lower index.  0 is below every key
typedef unsigned long long skey;
__device__ __forceinline__ unsigned order_of(float x) {
    x += 0.f;
    if (x != x) return 0xffc00000u;
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ skey key_of(float x, unsigned col) { return ((skey)order_of(x) << 32) | (0xffffffffu - col); }
__device__ __forceinline__ float score_of(skey k) { return value_of((unsigned)(k >> 32)); }
__device__ __forceinline__ int64_t col_of(skey k) { return (int64_t)(0xffffffffu - (unsigned)k); }

__device__ __forceinline__ float shift_of(float m) { return m == -__builtin_inff() ? 0.f : m; }

// The sums S = sum 2^y and U = sum y 2^y are formed with y = x log2(e) - c log2(e) in one multiply-add and one exponential per score.  The
// rounding of c log2(e) shifts every y by the same `off`; it is known exactly and taken out of the sums afterwards.  Beyond FAR, where that
// shift would grow, y = (x - c) log2(e) takes one operation more.
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f, FAR = 65536.f;
struct Shift {
    float c, c2, off;
    bool far;
    __device__ __forceinline__ explicit Shift(float m) : c(m), far(!(fabsf(m) < FAR)) {
        c2 = c * LOG2E;
        off = far ? 0.f : __builtin_fmaf(c, LOG2E, -c2);
    }
    template <bool FARAWAY> __device__ __forceinline__ void add(float x, float &S, float &U) const {
        const float y = FARAWAY ? (x - c) * LOG2E : __builtin_fmaf(x, LOG2E, -c2), e = __builtin_amdgcn_exp2f(y);
        S += e;
        U = __builtin_fmaf(fmaxf(y, -300.f), e, U);             // (2^-300 is 0, and so is y 2^y in the limit)
    }
    // S and U = sum z e^z of z = x - c
    __device__ __forceinline__ void finish(float &S, float &U) const {
        U = LN2 * __builtin_fmaf(-off, S, U);
        const float f = __builtin_amdgcn_exp2f(-off);
        S *= f; U *= f;
    }
};

struct FwdArgs {
    long long rows; int v; const char *x; long long ldx; const int64_t *ids; long long ignore; int top; float *logp, *entropy, *stat, *top_logp;
    int64_t *top_ids;
    int nsplit, slice;                          // slices of a row, scores of a slice
    float4 *part;                               // [rows][nsplit]: max, S, sum z e^z
    skey *keys;                                 // [rows][nsplit][top], best first
};

// what a row's results are, from its maximum and sums; one thread
__device__ __forceinline__ void finish_row(const FwdArgs &a, long long row, long long id, float xid, float c, float S, float U) {
    const bool empty = S == 0.f;
    const float L = empty ? __builtin_inff() : logf(S);
    a.logp[row] = id < 0 || id >= a.v ? __builtin_nanf("") : (xid - c) - L;
    a.entropy[row] = empty ? 0.f : L - U / S;
    if (a.stat) { a.stat[2 * row] = c; a.stat[2 * row + 1] = L; }
}
__device__ __forceinline__ void put_top(const FwdArgs &a, long long row, int rank, skey key, float c, float S) {
    a.top_logp[row * a.top + rank] = S == 0.f ? -__builtin_inff() : (score_of(key) - c) - logf(S);
    a.top_ids[row * a.top + rank] = col_of(key);
}
__device__ __forceinline__ void skip_row(const FwdArgs &a, long long row) {
    if (threadIdx.x == 0) { a.logp[row] = 0.f; a.entropy[row] = 0.f; if (a.stat) a.stat[2 * row] = a.stat[2 * row + 1] = 0.f; }
    for (int k = threadIdx.x; k < a.top; k += blockDim.x) { a.top_logp[row * a.top + k] = -__builtin_inff(); a.top_ids[row * a.top + k] = -1; }
}

template <int DT> __device__ __forceinline__ constexpr unsigned minus_inf() {
    return DT == I2P_F32 ? 0xff800000u : DT == I2P_BF16 ? 0xff80ff80u : 0xfc00fc00u;
}

// keeps the scores packed between the phases: the compiler would hold their fp32 values, and half as many waves would fit
template <int N> __device__ __forceinline__ void hold(uint4 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) asm volatile("" : "+v"(v[j].x), "+v"(v[j].y), "+v"(v[j].z), "+v"(v[j].w));
}

template <int DT, int W, int E>
__global__ __launch_bounds__(64 * W, E == 64 || (DT == I2P_F32 && E == 32 && W < 16) ? 6 : 8) void logprobs_fwd_kernel(FwdArgs a) {
    constexpr int T = 64 * W, VE = i2p_vec(DT), NV = E / VE;
    __shared__ float gmax[64], sums[2][W], bound;
    __shared__ skey list[LIST], best[W];
    __shared__ int count;
    const long long row = blockIdx.x / (unsigned)a.nsplit;      // (one row's slices stay together)
    const int part = (int)(blockIdx.x - (unsigned)row * (unsigned)a.nsplit), lo = part * a.slice, n = min(a.slice, a.v - lo);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long long id = a.ids[row];
    const char *x = a.x + (row * a.ldx + lo) * i2p_esize(DT);
    if (id == a.ignore) { if (a.nsplit == 1) skip_row(a, row); return; }
    uint4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const Col<DT> c(j * T + t, n);
        v[j] = c.load(x, n, minus_inf<DT>());
        if (c.skip) {                                           // what is not this vector's reads as -inf
            float f[VE];
            unpack<DT>(v[j], f);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] = c.counts(e, n) ? f[e] : -__builtin_inff();
            v[j] = pack<DT>(f);
        }
    }
    float xid = 0.f;
    if (a.nsplit == 1 && t == 0 && id >= 0 && id < a.v) xid = ld1<DT>(x, id);
    float vmax[NV], most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float f[VE];
        unpack<DT>(v[j], f);
        vmax[j] = f[0];
#pragma unroll
        for (int e = 1; e < VE; ++e) vmax[j] = fmaxf(vmax[j], f[e]);
        most = fmaxf(most, vmax[j]);
    }
    hold(v);
    // 64 groups of W lanes
    float g = lanes_max<W>(most);
    if constexpr (W > 1) {
        if ((t & (W - 1)) == 0) gmax[t / W] = g;
        if (t == 0) count = 0;
        __syncthreads();
        g = gmax[lane];
    } else if (t == 0) count = 0;
    const float m = lanes_max<64>(g), c = shift_of(m);
    // the largest value, to 16 bits of its order, that at least `top` groups reach
    float least = -__builtin_inff();
    if (a.top && wave == 0) {                                   // (the others read it behind the next barrier)
        const unsigned o = order_of(g);
        unsigned b = 0u;
#pragma unroll
        for (int k = 31; k >= 16; --k) {
            const unsigned next = b | (1u << k);
            if (__popcll(__ballot(o >= next)) >= a.top) b = next;
        }
        if (b > 0x007fffffu) least = value_of(b);               // (below: the order of -inf)
        if (W > 1 && lane == 0) bound = least;
    }
    const Shift sh(c);
    float S = 0.f, U = 0.f;
    if (!sh.far) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE];
            unpack<DT>(v[j], f);
#pragma unroll
            for (int e = 0; e < VE; ++e) sh.template add<false>(f[e], S, U);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float f[VE];
            unpack<DT>(v[j], f);
#pragma unroll
            for (int e = 0; e < VE; ++e) sh.template add<true>(f[e], S, U);
        }
    }
    hold(v);
    S = lanes_sum<64>(S); U = lanes_sum<64>(U);
    if constexpr (W > 1) {
        if (lane == 0) { sums[0][wave] = S; sums[1][wave] = U; }
        __syncthreads();
        S = U = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { S += sums[0][w]; U += sums[1][w]; }
    }
    sh.finish(S, U);
    if (t == 0) {
        if (a.nsplit == 1) finish_row(a, row, id, xid, c, S, U);
        else a.part[row * a.nsplit + part] = make_float4(m, S, U, 0.f);
    }
    if (!a.top) return;
    auto put = [&](int rank, skey key) {
        if (a.nsplit == 1) put_top(a, row, rank, key, c, S);
        else a.keys[(row * a.nsplit + part) * a.top + rank] = key;
    };
    if constexpr (W == 1) __syncthreads();                      // (`count`)
    else least = bound;
    const bool plain = S == S;                                  // no NaN, no +inf
    unsigned long long bits = 0ull;                             // which of the thread's scores reach the bound
    if (plain && most >= least) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!(vmax[j] >= least)) continue;
            const Col<DT> col(j * T + t, n);
            float f[VE];
            unpack<DT>(v[j], f);
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (f[e] >= least && (least > -__builtin_inff() || col.counts(e, n))) bits |= 1ull << (j * VE + e);
        }
    }
    for (;;) {                                                  // one of each lane a turn; its value is read again, from the caches
        const skey has = __ballot(bits != 0ull);
        if (!has) break;
        int base = 0;
        if (lane == 0) base = atomicAdd(&count, __popcll(has));
        base = __builtin_amdgcn_readfirstlane(base);
        if (base >= LIST) break;
        if (bits) {
            const int i = __ffsll(bits) - 1, at = base + __popcll(has & ((1ull << lane) - 1ull));
            bits &= bits - 1ull;
            const int col = Col<DT>(i / VE * T + t, n).at + i % VE;
            if (at < LIST) list[at] = key_of(ld1<DT>(x, col), (unsigned)(lo + col));
        }
    }
    __syncthreads();
    const int found = count;
    if (plain && found <= LIST) {
        for (int i = t; i < found; i += T) {
            const skey key = list[i];
            int rank = 0;
            for (int k = 0; k < found; ++k) rank += list[k] > key;
            if (rank < a.top) put(rank, key);
        }
        return;
    }
    skey last = ~0ull;                                          // (rare: the scores are read again, from the caches)
    for (int k = 0; k < a.top; ++k) {
        skey top = 0;
        for (int i = t; i < n; i += T) {
            const skey key = key_of(ld1<DT>(x, i), (unsigned)(lo + i));
            if (key < last && key > top) top = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { const skey u = __shfl_xor(top, o, 64); top = u > top ? u : top; }
        if (lane == 0) best[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) top = best[w] > top ? best[w] : top;
        __syncthreads();
        if (t == 0) put(k, top);
        last = top;
    }
}

// Rows of at most 128 scores: 16 lanes share one (8 scores each, lane by lane), so that a wave has four.  The alternatives are searched one
// after the other.  60000 x 32 fp32: 20.8 us with a wave per row, 5.5 here (41.7 and 12.7 with 3 alternatives)
constexpr int SMALL = 128;
__device__ __forceinline__ skey row16_best(skey k) {
    auto step = [&](unsigned lo, unsigned hi) { const skey u = ((skey)hi << 32) | lo; k = u > k ? u : k; };
    step(i2p_dpp_u32<0xB1>((unsigned)k), i2p_dpp_u32<0xB1>((unsigned)(k >> 32)));
    step(i2p_dpp_u32<0x4E>((unsigned)k), i2p_dpp_u32<0x4E>((unsigned)(k >> 32)));
    step(i2p_dpp_u32<0x141>((unsigned)k), i2p_dpp_u32<0x141>((unsigned)(k >> 32)));
    step(i2p_dpp_u32<0x140>((unsigned)k), i2p_dpp_u32<0x140>((unsigned)(k >> 32)));
    return k;
}

template <int DT> __global__ __launch_bounds__(256) void logprobs_small_kernel(FwdArgs a) {
    constexpr int E = SMALL / 16;
    const long long row = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    if (row >= a.rows) return;                                  // (16 lanes leave together: the reductions below stay among 16)
    const int t = threadIdx.x % 16;
    const long long id = a.ids[row];
    const char *x = a.x + row * a.ldx * i2p_esize(DT);
    if (id == a.ignore) {
        if (t == 0) { a.logp[row] = 0.f; a.entropy[row] = 0.f; if (a.stat) a.stat[2 * row] = a.stat[2 * row + 1] = 0.f; }
        for (int k = t; k < a.top; k += 16) { a.top_logp[row * a.top + k] = -__builtin_inff(); a.top_ids[row * a.top + k] = -1; }
        return;
    }
    float f[E], m = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * 16 + t;
        f[e] = i < a.v ? ld1<DT>(x, i) : -__builtin_inff();
        m = fmaxf(m, f[e]);
    }
    const float xid = t == 0 && id >= 0 && id < a.v ? ld1<DT>(x, id) : 0.f;
    const float c = shift_of(lanes_max<16>(m));
    float S = 0.f, U = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * 16 < a.v) {
            const float y = (f[e] - c) * LOG2E, p = __builtin_amdgcn_exp2f(y);
            S += p;
            U = __builtin_fmaf(fmaxf(y, -300.f), p, U);
        }
    S = lanes_sum<16>(S);
    U = LN2 * lanes_sum<16>(U);
    if (t == 0) finish_row(a, row, id, xid, c, S, U);
    skey last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        skey best = 0ull;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const skey key = e * 16 + t < a.v ? key_of(f[e], (unsigned)(e * 16 + t)) : 0ull;
            if (key < last && key > best) best = key;
        }
        last = row16_best(best);
        if (t == 0) put_top(a, row, k, last, c, S);
    }
}

// Joins the slices of a row, whose keys are in order.  Their q-th keys, q = top / slices rounded up, bound the row's best from below: where
// top / q slices, rounded up, have a q-th key of at least b, `top` keys are at least b
constexpr int JT = 256;                         // = most slices of a row
__global__ __launch_bounds__(JT) void logprobs_join_kernel(FwdArgs a, int dtype) {
    __shared__ float sums[3][JT / 64];
    __shared__ skey head[JT], list[I2P_MAX_TOP * I2P_MAX_TOP], bound;
    __shared__ int count;
    const long long row = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long long id = a.ids[row];
    if (id == a.ignore) { skip_row(a, row); return; }
    const float4 p = t < a.nsplit ? a.part[row * a.nsplit + t] : make_float4(-__builtin_inff(), 0.f, 0.f, 0.f);
    const skey *keys = a.keys + (row * a.nsplit + t) * a.top;
    const int q = a.top ? (a.top + a.nsplit - 1) / a.nsplit : 1, need = (a.top + q - 1) / q;
    const skey mine = a.top && t < a.nsplit ? keys[q - 1] : 0ull;
    float xid = 0.f;
    if (t == 0 && id >= 0 && id < a.v) {
        const long long i = row * a.ldx + id;
        xid = dtype == I2P_F32 ? ld1<I2P_F32>(a.x, i) : dtype == I2P_BF16 ? ld1<I2P_BF16>(a.x, i) : ld1<I2P_F16>(a.x, i);
    }
    float m = lanes_max<64>(p.x);
    if (lane == 0) sums[0][wave] = m;
    head[t] = mine;
    if (t == 0) { count = 0; bound = 0ull; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JT / 64; ++w) m = fmaxf(m, sums[0][w]);
    const float c = shift_of(m), shift = p.x - c, f = __expf(shift);
    float S = lanes_sum<64>(f * p.y), U = lanes_sum<64>(f * __builtin_fmaf(fmaxf(shift, -200.f), p.y, p.z));
    if (lane == 0) { sums[1][wave] = S; sums[2][wave] = U; }
    if (a.top && t < a.nsplit) {
        int rank = 0;
        for (int k = 0; k < a.nsplit; ++k) rank += head[k] > mine;
        if (rank == need - 1) bound = mine;
    }
    __syncthreads();
    S = U = 0.f;
#pragma unroll
    for (int w = 0; w < JT / 64; ++w) { S += sums[1][w]; U += sums[2][w]; }
    if (t == 0) finish_row(a, row, id, xid, c, S, U);
    if (!a.top) return;
    if (t < a.nsplit)
        for (int k = 0; k < a.top; ++k) {                       // (`need` slices have up to `top` keys that reach it, the others fewer than q)
            const skey key = keys[k];
            if (key < bound) break;
            list[atomicAdd(&count, 1)] = key;
        }
    __syncthreads();
    const int found = count;
    for (int i = t; i < found; i += JT) {
        const skey key = list[i];
        int rank = 0;
        for (int k = 0; k < found; ++k) rank += list[k] > key;
        if (rank < a.top) put_top(a, row, rank, key, c, S);
    }
}

struct BwdArgs {
    long long rows; int v; const char *x; long long ldx; const int64_t *ids; long long ignore; const float *stat, *entropy, *g_logp, *g_entropy;
    char *dx; bool stream; int pieces;          // pieces of a row, each BV vectors of the TPR threads that share it
};
constexpr int BV = 4;

template <int DT, int TPR>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(BwdArgs a) {
    constexpr int VE = i2p_vec(DT), ES = i2p_esize(DT);
    constexpr bool TINY = TPR == 16;
    const long long work = a.rows * a.pieces;
    const int t = threadIdx.x % TPR;
    for (long long k = (long long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; k < work; k += (long long)gridDim.x * (256 / TPR)) {
        const long long i = a.stream ? work - 1 - k : k;
        const long long row = a.pieces == 1 ? i : i / a.pieces;
        const int piece = (int)(i - row * a.pieces);
        const char *x = a.x + row * a.ldx * ES;
        const long long id = a.ids[row];
        uint4 u[BV];
        if (id != a.ignore)
#pragma unroll
            for (int j = 0; j < BV; ++j) u[j] = Col<DT, TINY>((piece * BV + j) * TPR + t, a.v).load(x, a.v);
        const float gh = a.g_entropy ? a.g_entropy[row] : 0.f, H = a.entropy[row], c = a.stat[2 * row], L = a.stat[2 * row + 1];
        float gl = a.g_logp ? a.g_logp[row] : 0.f;
        if (L == __builtin_inff()) gl = 0.f;                     // an empty row
        if (id < 0 || id >= a.v) gl = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < BV; ++j) {
            const Col<DT, TINY> col((piece * BV + j) * TPR + t, a.v);
            if (!col.in) break;
            float f[VE] = {};
            if (id != a.ignore) {
                unpack<DT>(u[j], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float lp = f[e] - c - L, p = __expf(lp);
                    f[e] = (col.at + e == id ? gl : 0.f) - p * __builtin_fmaf(gh, fmaxf(lp, -200.f) + H, gl);
                }
            }
            if (a.stream) col.store_stream(a.dx + row * a.v * ES, pack<DT>(f));
            else col.store(a.dx + row * a.v * ES, a.v, pack<DT>(f));
        }
    }
}

template <class F> void by_type(int dtype, F f) {
    if (dtype == I2P_F32) f(std::integral_constant<int, I2P_F32>{});
    else if (dtype == I2P_BF16) f(std::integral_constant<int, I2P_BF16>{});
    else f(std::integral_constant<int, I2P_F16>{});
}

constexpr int WHOLE = 32768;                    // scores that 16 waves hold
constexpr int FEW = 4096;                       // a slice where blocks are few
constexpr int SLICE = 8192;                     // 4 waves

// how a row is cut: few rows of up to 32768 scores stay whole, which saves the second launch (the 256 CUs hold two blocks of 16 waves each);
// otherwise slices of 4 waves, whose barriers stall less of a CU (4096 x 32000 bf16: whole 73.5 us, slices of 8192 57.5 + 6.1), shorter ones
// where there would be fewer than half as many as CUs (1 x 131072 fp32: 6.5 -> 5.3 us) and, of the 16-bit types, longer ones where they still
// fill the chip ten times (8192 x 131072: 508 -> 466 us; 4096 x 32000, which is five times: 58 -> 61)
inline void cut(long long rows, int v, int dtype, int &nsplit, int &slice) {
    nsplit = v <= WHOLE && rows <= 512 ? 1 : (v + SLICE - 1) / SLICE;
    if (dtype != I2P_F32 && nsplit > 1 && rows * ((nsplit + 1) / 2) >= 16384) nsplit = (v + 2 * SLICE - 1) / (2 * SLICE);
    if (nsplit > 1 && rows * nsplit <= 128 && v <= FEW * JT) nsplit = (v + FEW - 1) / FEW;
    slice = ((v + nsplit - 1) / nsplit + 7) & ~7;
    nsplit = (v + slice - 1) / slice;
}

inline bool sizes_ok(long long rows, int v, int dtype, long long ldx) {
    return rows >= 0 && v > 0 && v <= I2P_MAX_CANDIDATES && dtype >= I2P_F32 && dtype <= I2P_F16 && ldx >= v;
}

}  // namespace

extern "C" long long i2p_token_logprobs_scratch(long long rows, int v, int dtype, int top) {
    if (rows <= 0 || v <= 0 || v > I2P_MAX_CANDIDATES || top < 0 || top > I2P_MAX_TOP) return 0;
    int nsplit, slice;
    cut(rows, v, dtype, nsplit, slice);
    return nsplit == 1 ? 0 : rows * nsplit * (16 + 8ll * top);
}

extern "C" int i2p_token_logprobs_fwd(long long rows, int v, int dtype, const void *x, long long ldx, const int64_t *ids, long long ignore, int top,
                                      float *logp, float *entropy, float *stat, float *top_logp, int64_t *top_ids, void *scratch, void *stream) {
    if (!sizes_ok(rows, v, dtype, ldx) || top < 0 || top > v || top > I2P_MAX_TOP) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !ids || !logp || !entropy || (top && (!top_logp || !top_ids))) return I2P_ERR_BAD_ARG;
    int nsplit, slice;
    cut(rows, v, dtype, nsplit, slice);
    if (nsplit > 1 && (!scratch || ((uintptr_t)scratch & 15))) return I2P_ERR_BAD_ARG;
    hipStream_t st = (hipStream_t)stream;
    const long long most = (1 << 21) / nsplit;          // rows of a launch: a grid has fewer than 2^32 threads
    for (long long r = 0; r < rows; r += most) by_type(dtype, [&](auto dt) {
        const long long k = rows - r < most ? rows - r : most;
        const FwdArgs a{k, v, (const char *)x + r * ldx * i2p_esize(dtype), ldx, ids + r, ignore, top, logp + r, entropy + r, stat ? stat + 2 * r : nullptr,
                        top_logp + r * top, top_ids + r * top, nsplit, slice, (float4 *)scratch + r * nsplit,
                        (skey *)((char *)scratch + rows * nsplit * 16) + r * nsplit * top};
        const dim3 grid((unsigned)(k * nsplit));
        constexpr int DT = dt.value;
        if (v <= SMALL) hipLaunchKernelGGL((logprobs_small_kernel<DT>), dim3((unsigned)((k + 15) / 16)), dim3(256), 0, st, a);
        else if (slice <= 512) hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 1, 8>), grid, dim3(64), 0, st, a);
        else if (slice <= 2048) hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 1, 32>), grid, dim3(64), 0, st, a);
        else if (slice <= 4096) hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 4, 16>), grid, dim3(256), 0, st, a);
        else if (slice <= SLICE) hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 4, 32>), grid, dim3(256), 0, st, a);
        else if (DT != I2P_F32 && slice <= 2 * SLICE && (nsplit > 1 || rows > 512))
            hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 4, (DT == I2P_F32 ? 32 : 64)>), grid, dim3(256), 0, st, a);
        else if (slice <= 16384) hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 16, 16>), grid, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((logprobs_fwd_kernel<DT, 16, 32>), grid, dim3(1024), 0, st, a);
        if (nsplit > 1) hipLaunchKernelGGL(logprobs_join_kernel, dim3((unsigned)k), dim3(JT), 0, st, a, dtype);
    });
    I2P_RETURN_LAUNCH_STATUS();
}

extern "C" int i2p_token_logprobs_bwd(long long rows, int v, int dtype, const void *x, long long ldx, const int64_t *ids, long long ignore,
                                      const float *stat, const float *entropy, const float *g_logp, const float *g_entropy, void *dx, void *stream) {
    if (!sizes_ok(rows, v, dtype, ldx)) return I2P_ERR_BAD_ARG;
    if (rows == 0) return 0;
    if (!x || !ids || !stat || !entropy || !dx) return I2P_ERR_BAD_ARG;
    const long long pitch = (long long)v * i2p_esize(dtype);
    // A gradient that no cache would hold until it is used goes past them, and the rows are taken from the last: then what the forward read
    // last is still in the 256 MB last-level cache (kernels of forward + backward in turn, 4096 x 32000 bf16: 163 -> 150 us,
    // 8192 x 32000 343 -> 326: the forward's 72 and 145 become 58 and 123).  Rows that do not start on 16 bytes would be written in parts of lines
    const bool stream_out = pitch % 16 == 0 && ((uintptr_t)dx & 15) == 0 && rows * pitch >= (64ll << 20);
    by_type(dtype, [&](auto dt) {
        constexpr int DT = dt.value;
        const int nvec = (v + i2p_vec(DT) - 1) / i2p_vec(DT);
        auto go = [&](auto tpr) {
            constexpr int TPR = tpr.value;
            const BwdArgs a{rows, v, (const char *)x, ldx, ids, ignore, stat, entropy, g_logp, g_entropy, (char *)dx, stream_out,
                            (nvec + TPR * BV - 1) / (TPR * BV)};
            const long long blocks = (rows * a.pieces + 256 / TPR - 1) / (256 / TPR);
            hipLaunchKernelGGL((logprobs_bwd_kernel<DT, TPR>), dim3((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), dim3(256), 0,
                               (hipStream_t)stream, a);
        };
        if (nvec <= 16 * BV) go(std::integral_constant<int, 16>{});
        else if (nvec <= 64 * BV) go(std::integral_constant<int, 64>{});
        else go(std::integral_constant<int, 256>{});
    });
    I2P_RETURN_LAUNCH_STATUS();
}
