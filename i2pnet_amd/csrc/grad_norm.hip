// Global norm of many gradient tensors and clipping by it, in place or into one flat fp32 buffer.
//
//   total = sqrt(sum over all tensors of g^2)   or   max |g|;      c = min(1, max_norm / (total + 1e-6));      g <- round(c g)   or   out <- c g
//
// The tensors (any sizes, fp32 / bf16 / fp16 mixed) come as a host list; a launch takes a table of them by value, so the call can be captured:
// a captured launch holds its table.  Squares are summed in fp64: no overflow below the type's own range, and the order of the additions
// depends on the list's sizes and types alone: the norm is the same with clipping and without, in place or not.  A NaN or inf reaches the
// total and, through c, every gradient.
//
// Bound by memory where there is much (300 M elements, bf16 and fp32, into the flat buffer: norm 164 us = 4.3 TB/s read, clipping 370 us =
// 5.2 TB/s read and written) and by two launches where there is little (254 tensors of 845 k elements in place: 4.9 + 2.8 us of a call of 20:
// the rest is the host, which lists them).
#include "rows_common.h"
#include <algorithm>
#include <new>
#include <type_traits>

namespace {

constexpr int T = 256;
constexpr long long PART = 1ll << 30;           // a longer tensor is listed in parts of this many elements

// The tensors of a launch, by value (below the 4 KB of a kernel's arguments).  Where each starts in the flat output is listed only for a
// launch that writes there, so that in place and for the norm one launch takes 320 tensors
template <bool OUT> struct Table {
    static constexpr int CAP = OUT ? 192 : 320;
    unsigned long long ptr[CAP];                // address | (elements of the last chunk - 1) << 48
    unsigned long long off[OUT ? CAP : 1];
    unsigned first[CAP];                        // first chunk | dtype << 30
    unsigned n, chunks;
    int chunk;                                  // elements of a chunk
};

struct Piece { unsigned long long p; int dtype; unsigned count; unsigned long long off; };

// The piece of the table that chunk `c` of this launch covers.  Every wave finds it by itself: each lane counts the tensors of its share that
// start at or before the chunk (independent loads: a binary search is eight dependent ones, 2 .. 3 us of a 5 us kernel)
template <bool OUT> __device__ __forceinline__ Piece piece_of(const Table<OUT> &t, unsigned c) {
    constexpr int PER = Table<OUT>::CAP / 64;
    const int lane = threadIdx.x & 63;
    int before = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const unsigned i = k * 64 + lane;
        before += __popcll(__ballot(i < t.n && (t.first[i] & 0x3fffffffu) <= c));
    }
    const int at = __builtin_amdgcn_readfirstlane(before) - 1;
    const unsigned f = t.first[at], k = c - (f & 0x3fffffffu), end = at + 1 < (int)t.n ? (t.first[at + 1] & 0x3fffffffu) : t.chunks;
    const unsigned long long p = t.ptr[at];
    Piece r;
    r.dtype = (int)(f >> 30);
    r.p = (p & 0xffffffffffffull) + (unsigned long long)k * t.chunk * i2p_esize(r.dtype);
    r.count = c + 1 == end ? (unsigned)(p >> 48) + 1u : (unsigned)t.chunk;
    r.off = OUT ? t.off[at] + (unsigned long long)k * t.chunk : 0ull;
    return r;
}

__device__ __forceinline__ double nan_max(double a, double b) { return a != a ? a : (b > a || b != b ? b : a); }

template <bool MAX> __device__ __forceinline__ double block_sum(double v, double *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const double u = __shfl_xor(v, o, 64); v = MAX ? nan_max(v, u) : v + u; }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) t = MAX ? nan_max(t, red[w]) : t + red[w];
    return t;
}

// A piece is read in 16-byte vectors from wherever it starts, BATCH of a thread in flight; its last elements one by one
constexpr int BATCH = 4;
template <int DT, class F> __device__ __forceinline__ void for_vectors(const Piece &p, F f) {
    constexpr int VE = i2p_vec(DT);
    const char *base = (const char *)p.p;
    const unsigned nv = p.count / VE;
    for (unsigned v0 = threadIdx.x; v0 < nv; v0 += BATCH * T) {
        uint4 u[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (v0 + j * T < nv) __builtin_memcpy(&u[j], base + (size_t)(v0 + j * T) * 16, 16);
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (v0 + j * T < nv) { float g[VE]; unpack<DT>(u[j], g); f(g, (v0 + j * T) * VE); }
    }
}

template <int DT, bool MAX> __device__ __forceinline__ double norm_piece(const Piece &p) {
    constexpr int VE = i2p_vec(DT);
    double acc = 0.0;
    auto add = [&](float g) { acc = MAX ? nan_max(acc, (double)fabsf(g)) : __builtin_fma((double)g, (double)g, acc); };
    for_vectors<DT>(p, [&](const float (&g)[VE], unsigned) {
#pragma unroll
        for (int e = 0; e < VE; ++e) add(g[e]);
    });
    const unsigned rest = p.count / VE * VE + threadIdx.x;
    if (rest < p.count) add(ld1<DT>((const void *)p.p, rest));
    return acc;
}

template <bool MAX> __global__ __launch_bounds__(T) void grad_norm_kernel(Table<false> t, double *__restrict__ partials) {
    __shared__ double red[T / 64];
    const Piece p = piece_of(t, blockIdx.x);
    const double acc = p.dtype == I2P_F32 ? norm_piece<I2P_F32, MAX>(p) : p.dtype == I2P_BF16 ? norm_piece<I2P_BF16, MAX>(p) : norm_piece<I2P_F16, MAX>(p);
    const double s = block_sum<MAX>(acc, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// the partial norms in a fixed order, the same on every block of as many threads
template <bool MAX, int THREADS> __device__ __forceinline__ float total_of(unsigned n, const double *__restrict__ partials, double *red) {
    double acc = 0.0;
    for (unsigned i0 = threadIdx.x; i0 < n; i0 += 8 * THREADS) {      // eight loads in flight
        double p[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) p[u] = i0 + u * THREADS < n ? partials[i0 + u * THREADS] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) acc = MAX ? nan_max(acc, p[u]) : acc + p[u];
    }
    const double s = block_sum<MAX>(acc, red);
    return (float)(MAX ? s : sqrt(s));
}

template <bool MAX, int THREADS>
__global__ __launch_bounds__(THREADS) void grad_total_kernel(unsigned n, const double *__restrict__ partials, float *__restrict__ total) {
    __shared__ double red[THREADS / 64];
    const float t = total_of<MAX, THREADS>(n, partials, red);
    if (threadIdx.x == 0) total[0] = t;
}

template <int DT, bool OUT> __device__ __forceinline__ void clip_piece(const Piece &p, float c, float *out) {
    constexpr int VE = i2p_vec(DT);
    for_vectors<DT>(p, [&](const float (&g)[VE], unsigned i) {
        float h[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) h[e] = g[e] * c;
        if (OUT) __builtin_memcpy(out + p.off + i, h, 4 * VE);
        else { const uint4 u = pack<DT>(h); __builtin_memcpy((char *)p.p + (size_t)i * i2p_esize(DT), &u, 16); }
    });
    const unsigned rest = p.count / VE * VE + threadIdx.x;
    if (rest < p.count) {
        const float g = ld1<DT>((const void *)p.p, rest) * c;
        if (OUT) out[p.off + rest] = g;
        else st1<DT>((void *)p.p, rest, g);
    }
}

// OUT: into the flat buffer.  SUM 0: the total is there; 1, 2: every block forms it (2-norm, maximum) from the partial norms
template <bool OUT, int SUM>
__global__ __launch_bounds__(T) void grad_clip_kernel(Table<OUT> t, float max_norm, unsigned n, const double *__restrict__ partials, float *total, float *out) {
    __shared__ double red[T / 64];
    float norm;
    if constexpr (SUM != 0) {
        norm = total_of<SUM == 2, T>(n, partials, red);
        if (total && blockIdx.x == 0 && threadIdx.x == 0) total[0] = norm;
    } else norm = total[0];
    const float r = max_norm / (norm + 1e-6f), c = r > 1.f ? 1.f : r;                       // (NaN stays)
    if (c == 1.f && !OUT) return;                                                            // within the limit: the gradients stay as they are
    const Piece p = piece_of(t, blockIdx.x);
    if (p.dtype == I2P_F32) clip_piece<I2P_F32, OUT>(p, c, out);
    else if (p.dtype == I2P_BF16) clip_piece<I2P_BF16, OUT>(p, c, out);
    else clip_piece<I2P_F16, OUT>(p, c, out);
}

inline long long chunks_of(long long numel, int chunk) { return (numel + chunk - 1) / chunk; }

// A chunk is what a block reads (at most 65536 elements: 16 bits of `ptr` tell the last one's length): 4096 elements, one batch of loads a
// thread, while there are few; else 16384 (300 M elements: 541 us in all, 583 with 65536)
inline int chunk_for(int n, const long long *numel) {
    long long total = 0;
    for (int i = 0; i < n; ++i) total += numel[i];
    return total <= (4ll << 20) ? 4096 : 16384;
}

// Walks the list in tables and calls launch(table) for each
template <bool OUT, class F> void for_tables(int n, const void *const *grads, const long long *numel, const int *dtype, F launch) {
    Table<OUT> t;
    t.n = t.chunks = 0;
    t.chunk = chunk_for(n, numel);
    unsigned long long off = 0;
    for (int i = 0; i < n; ++i)
        for (long long done = 0; done < numel[i]; done += PART) {
            const long long k = std::min(PART, numel[i] - done);
            if (t.n == Table<OUT>::CAP || t.chunks + chunks_of(k, t.chunk) > (1 << 22)) { launch(t); t.n = t.chunks = 0; }
            const unsigned long long last = (unsigned long long)((k - 1) % t.chunk);
            t.ptr[t.n] = ((unsigned long long)grads[i] + (unsigned long long)done * i2p_esize(dtype[i])) | (last << 48);
            t.first[t.n] = t.chunks | ((unsigned)dtype[i] << 30);
            if (OUT) t.off[t.n] = off;
            off += (unsigned long long)k;
            ++t.n;
            t.chunks += (unsigned)chunks_of(k, t.chunk);
        }
    if (t.n) launch(t);
}

// partial norms that every clipping block sums itself: cheaper than a launch of one block for it.  That many are always summed by T threads
// and more by 1024, so that a norm without clipping adds them in the same order
constexpr unsigned FEW = 2048;

struct Range { unsigned long long lo, hi; };

// 0: fine; otherwise the status.  No two tensors may share memory: both would be scaled, in whatever order the blocks run
int check(int n, const void *const *grads, const long long *numel, const int *dtype, bool in_place, const float *out) {
    if (n < 0 || (n && (!grads || !numel || !dtype))) return I2P_ERR_BAD_ARG;
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        if (numel[i] < 0 || dtype[i] < I2P_F32 || dtype[i] > I2P_F16 || (numel[i] && !grads[i]) || numel[i] > (1ll << 44) - total) return I2P_ERR_BAD_ARG;
        const unsigned long long p = (unsigned long long)grads[i];
        if ((p >> 48) || (p & (i2p_esize(dtype[i]) - 1))) return I2P_ERR_BAD_ARG;
        total += numel[i];
    }
    Range *r = new (std::nothrow) Range[(size_t)n + 1];
    if (!r) return I2P_ERR_BAD_ARG;
    int k = 0;
    if (in_place || out)
        for (int i = 0; i < n; ++i)
            if (numel[i]) {
                const unsigned long long p = (unsigned long long)grads[i];
                r[k++] = {p, p + (unsigned long long)numel[i] * i2p_esize(dtype[i])};
            }
    if (out) {                                  // the flat buffer against every gradient
        const Range o{(unsigned long long)out, (unsigned long long)out + 4ull * (unsigned long long)total};
        for (int i = 0; i < k; ++i)
            if (r[i].lo < o.hi && o.lo < r[i].hi) { delete[] r; return I2P_ERR_OVERLAP; }
        k = 0;                                  // (only read: the same tensor may be listed twice)
    }
    const auto below = [](const Range &a, const Range &b) { return a.lo < b.lo; };
    if (!std::is_sorted(r, r + k, below)) std::sort(r, r + k, below);
    int rc = 0;
    for (int i = 1; i < k; ++i)
        if (r[i].lo < r[i - 1].hi) rc = I2P_ERR_OVERLAP;
    delete[] r;
    return rc;
}

}  // namespace

extern "C" long long i2p_grad_norm_scratch(int n, const long long *numel) {
    long long c = 0;
    if (n > 0 && numel) {
        const int chunk = chunk_for(n, numel);
        for (int i = 0; i < n; ++i)
            for (long long done = 0; done < numel[i]; done += PART) c += chunks_of(std::min(PART, numel[i] - done), chunk);
    }
    return 8 * std::max(c, 1ll);
}

extern "C" int i2p_clip_grad_norm(int n, const void *const *grads, const long long *numel, const int *dtype, int kind, int clip, float max_norm,
                                  float *out, void *scratch, float *total, void *stream) {
    const int bad = check(n, grads, numel, dtype, clip && !out, clip ? out : nullptr);
    if (bad) return bad;
    if (kind < 0 || kind > 1 || !scratch || ((uintptr_t)scratch & 15) || !total || (clip && !(max_norm >= 0.f))) return I2P_ERR_BAD_ARG;
    hipStream_t st = (hipStream_t)stream;
    double *partials = (double *)scratch;
    unsigned done = 0;
    for_tables<false>(n, grads, numel, dtype, [&](const Table<false> &t) {
        if (kind) hipLaunchKernelGGL((grad_norm_kernel<true>), dim3(t.chunks), dim3(T), 0, st, t, partials + done);
        else hipLaunchKernelGGL((grad_norm_kernel<false>), dim3(t.chunks), dim3(T), 0, st, t, partials + done);
        done += t.chunks;
    });
    const bool few = clip && done && done <= FEW;
    if (!few) {
        auto sum = [&](auto threads) {
            constexpr int THREADS = threads.value;
            if (kind) hipLaunchKernelGGL((grad_total_kernel<true, THREADS>), dim3(1), dim3(THREADS), 0, st, done, partials, total);
            else hipLaunchKernelGGL((grad_total_kernel<false, THREADS>), dim3(1), dim3(THREADS), 0, st, done, partials, total);
        };
        if (done <= FEW) sum(std::integral_constant<int, T>{});
        else sum(std::integral_constant<int, 1024>{});
    }
    if (clip) {
        float *sum = total;                     // the first launch's first block writes the total
        auto go = [&](auto with_out) {
            constexpr bool OUT = decltype(with_out)::value;
            for_tables<OUT>(n, grads, numel, dtype, [&](const Table<OUT> &t) {
                if (!few) hipLaunchKernelGGL((grad_clip_kernel<OUT, 0>), dim3(t.chunks), dim3(T), 0, st, t, max_norm, done, partials, total, out);
                else if (kind) hipLaunchKernelGGL((grad_clip_kernel<OUT, 2>), dim3(t.chunks), dim3(T), 0, st, t, max_norm, done, partials, sum, out);
                else hipLaunchKernelGGL((grad_clip_kernel<OUT, 1>), dim3(t.chunks), dim3(T), 0, st, t, max_norm, done, partials, sum, out);
                sum = nullptr;
            });
        };
        if (out) go(std::true_type{});
        else go(std::false_type{});
    }
    I2P_RETURN_LAUNCH_STATUS();
}
