// Global norm of many gradient tensors and clipping by it, in place or into one flat fp32 buffer.
//
//   total = sqrt(sum over all tensors of g^2)   or   max |g|;      c = min(1, max_norm / (total + 1e-6));      g <- round(c g)   or   out <- c g
//
// The tensors (any sizes, fp32 / bf16 / fp16 mixed) come as a host list; a launch takes a table of them by value, so the call can be captured:
// a captured launch holds its table.  Squares are summed in fp64: no overflow below the type's own range, and the order (chunk by
// chunk, partial sums in index order) does not depend on the launch.  A NaN or inf reaches the total and, through c, every gradient.
#include "rows_common.h"
#include <algorithm>
#include <new>

namespace {

constexpr int T = 256, CHUNK = 16384;
constexpr int CAP = 180;                        // 20 bytes each: the table stays below the 4 KB of a kernel's arguments
constexpr long long PART = 1ll << 30;           // a longer tensor is listed in parts of this many elements

struct Table {
    unsigned long long ptr[CAP];                // address | (elements of the last chunk - 1) << 48
    unsigned first[CAP];                        // first chunk | dtype << 30
    unsigned long long off[CAP];                // where it starts in the flat output
    unsigned n, chunks;
};

struct Piece { unsigned long long p; int dtype; unsigned count; unsigned long long off; };

// the piece of the table that chunk `c` of this launch covers
__device__ __forceinline__ Piece piece_of(const Table &t, unsigned c) {
    unsigned lo = 0, hi = t.n;                  // first[lo] <= c < first[hi]
    while (hi - lo > 1) { const unsigned mid = (lo + hi) >> 1; if ((t.first[mid] & 0x3fffffffu) <= c) lo = mid; else hi = mid; }
    const unsigned f = t.first[lo], k = c - (f & 0x3fffffffu), end = lo + 1 < t.n ? (t.first[lo + 1] & 0x3fffffffu) : t.chunks;
    const unsigned long long p = t.ptr[lo];
    Piece r;
    r.dtype = (int)(f >> 30);
    r.p = (p & 0xffffffffffffull) + (unsigned long long)k * CHUNK * i2p_esize(r.dtype);
    r.count = c + 1 == end ? (unsigned)(p >> 48) + 1u : (unsigned)CHUNK;
    r.off = t.off[lo] + (unsigned long long)k * CHUNK;
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

template <bool MAX> __global__ __launch_bounds__(T) void grad_norm_kernel(Table t, double *__restrict__ partials) {
    __shared__ double red[T / 64];
    const Piece p = piece_of(t, blockIdx.x);
    const double acc = p.dtype == I2P_F32 ? norm_piece<I2P_F32, MAX>(p) : p.dtype == I2P_BF16 ? norm_piece<I2P_BF16, MAX>(p) : norm_piece<I2P_F16, MAX>(p);
    const double s = block_sum<MAX>(acc, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

template <bool MAX> __global__ __launch_bounds__(1024) void grad_total_kernel(unsigned n, const double *__restrict__ partials, float *__restrict__ total) {
    __shared__ double red[16];
    double acc = 0.0;
    for (unsigned i = threadIdx.x; i < n; i += 1024) acc = MAX ? nan_max(acc, partials[i]) : acc + partials[i];
    const double s = block_sum<MAX>(acc, red);
    if (threadIdx.x == 0) total[0] = (float)(MAX ? s : sqrt(s));
}

template <int DT> __device__ __forceinline__ void clip_piece(const Piece &p, float c, float *out) {
    constexpr int VE = i2p_vec(DT);
    for_vectors<DT>(p, [&](const float (&g)[VE], unsigned i) {
        float h[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) h[e] = g[e] * c;
        if (out) __builtin_memcpy(out + p.off + i, h, 4 * VE);
        else { const uint4 u = pack<DT>(h); __builtin_memcpy((char *)p.p + (size_t)i * i2p_esize(DT), &u, 16); }
    });
    const unsigned rest = p.count / VE * VE + threadIdx.x;
    if (rest < p.count) {
        const float g = ld1<DT>((const void *)p.p, rest) * c;
        if (out) out[p.off + rest] = g;
        else st1<DT>((void *)p.p, rest, g);
    }
}

__global__ __launch_bounds__(T) void grad_clip_kernel(Table t, float max_norm, const float *__restrict__ total, float *out) {
    const float r = max_norm / (total[0] + 1e-6f), c = r > 1.f ? 1.f : r;                   // (NaN stays)
    if (c == 1.f && !out) return;                                                            // within the limit: the gradients stay as they are
    const Piece p = piece_of(t, blockIdx.x);
    if (p.dtype == I2P_F32) clip_piece<I2P_F32>(p, c, out);
    else if (p.dtype == I2P_BF16) clip_piece<I2P_BF16>(p, c, out);
    else clip_piece<I2P_F16>(p, c, out);
}

inline long long chunks_of(long long numel) { return (numel + CHUNK - 1) / CHUNK; }

// Walks the list in tables of at most CAP pieces and calls launch(table) for each
template <class F> void for_tables(int n, const void *const *grads, const long long *numel, const int *dtype, F launch) {
    Table t;
    t.n = t.chunks = 0;
    unsigned long long off = 0;
    for (int i = 0; i < n; ++i)
        for (long long done = 0; done < numel[i]; done += PART) {
            const long long k = std::min(PART, numel[i] - done);
            if (t.n == CAP || t.chunks + chunks_of(k) > (1 << 22)) { launch(t); t.n = t.chunks = 0; }
            const unsigned long long last = (unsigned long long)((k - 1) % CHUNK);
            t.ptr[t.n] = ((unsigned long long)grads[i] + (unsigned long long)done * i2p_esize(dtype[i])) | (last << 48);
            t.first[t.n] = t.chunks | ((unsigned)dtype[i] << 30);
            t.off[t.n] = off;
            off += (unsigned long long)k;
            ++t.n;
            t.chunks += (unsigned)chunks_of(k);
        }
    if (t.n) launch(t);
}

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
    std::sort(r, r + k, [](const Range &a, const Range &b) { return a.lo < b.lo; });
    int rc = 0;
    for (int i = 1; i < k; ++i)
        if (r[i].lo < r[i - 1].hi) rc = I2P_ERR_OVERLAP;
    delete[] r;
    return rc;
}

}  // namespace

extern "C" long long i2p_grad_norm_scratch(int n, const long long *numel) {
    long long c = 0;
    for (int i = 0; numel && i < n; ++i)
        for (long long done = 0; done < numel[i]; done += PART) c += chunks_of(std::min(PART, numel[i] - done));
    return 8 * std::max(c, 1ll);
}

extern "C" int i2p_clip_grad_norm(int n, const void *const *grads, const long long *numel, const int *dtype, int kind, int clip, float max_norm,
                                  float *out, void *scratch, float *total, void *stream) {
    const int bad = check(n, grads, numel, dtype, clip && !out, clip ? out : nullptr);
    if (bad) return bad;
    if (kind < 0 || kind > 1 || !scratch || !total || (clip && !(max_norm >= 0.f))) return I2P_ERR_BAD_ARG;
    hipStream_t st = (hipStream_t)stream;
    double *partials = (double *)scratch;
    unsigned done = 0;
    for_tables(n, grads, numel, dtype, [&](const Table &t) {
        if (kind) hipLaunchKernelGGL((grad_norm_kernel<true>), dim3(t.chunks), dim3(T), 0, st, t, partials + done);
        else hipLaunchKernelGGL((grad_norm_kernel<false>), dim3(t.chunks), dim3(T), 0, st, t, partials + done);
        done += t.chunks;
    });
    if (kind) hipLaunchKernelGGL((grad_total_kernel<true>), dim3(1), dim3(1024), 0, st, done, partials, total);
    else hipLaunchKernelGGL((grad_total_kernel<false>), dim3(1), dim3(1024), 0, st, done, partials, total);
    if (clip)
        for_tables(n, grads, numel, dtype, [&](const Table &t) {
            hipLaunchKernelGGL(grad_clip_kernel, dim3(t.chunks), dim3(T), 0, st, t, max_norm, total, out);
        });
    I2P_RETURN_LAUNCH_STATUS();
}
