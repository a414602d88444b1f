// Layer norm over the last axis of (rows, C) and its backward pass.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Both passes are bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx - each byte once.  32768 x 4096
// bf16: 103 us and 177 us (5.2 and 4.6 TB/s; a large copy reaches 5.0), and 5 us for the parameters' gradients.  Below a few
// megabytes latency counts: 1008 x 512 fp32 takes 3.9 us, and 5.9 + 4.6 us backward.  Rows beyond the registers (below) run at 1.0 to
// 2.8 TB/s.  A row stays in the registers of the threads
// that own it (64 to 1024 of them), so the variance is the two-pass one (the sum of squared differences from the mean, no
// cancellation) without a second read.  The differences are summed beside their squares and correct the mean: a sum's roundings leave
// it a few steps of x off, which for rows of nearly equal large values is as much as they differ (a constant row gave 0.93
// instead of 0; forward 90 us without it).  A thread owns the same columns of every row its workgroup takes: w and b are loaded once,
// and the column sums dw / db grow in its registers; the row groups of a workgroup are joined in LDS, the workgroups by a second
// launch in fixed order (no atomics: results do not change from run to run).  Statistics, sums and parameter gradients are fp32; y
// and dx are rounded once.
#include "lm_common.h"
#include "ssecg.h"

namespace {
using namespace ssecg_lm;

// Sum over the TPR threads of a row; every thread gets it.  `sh` holds a slot per wave; two slots sets alternate by `flip`, so
// one barrier per reduction is enough (a wave can be at most one reduction ahead of the others).
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* sh, int& flip) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / W * W;
        float* s = sh + flip * (16 * K);
        flip ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) s[wave * K + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) t += s[(first + w) * K + k];
            v[k] = t;
        }
    }
}

// a b, rounded: left to itself the compiler fuses the product into the differences from it and not into the mean
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// mean and 1 / deviation from an approximate mean and the means of the differences from it and of their squares
__device__ __forceinline__ void row_stats(float near, float d, float d2, float eps, float& mu, float& rs) {
    const float var = d2 - d * d;                     // d2 >= d^2 but for roundings
    mu = d == d ? near + d : near;                    // (a row with an infinity: its mean is infinite)
    rs = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);  // (a NaN stays one)
}

// a thread's share of a parameter vector (absent or beyond C: `none`)
template <typename T, int TPR, int NCH>
__device__ __forceinline__ void load_params(const float* __restrict__ p, int t, int C, float none, float (&v)[NCH][Vec<T>::N]) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const int c = (t + TPR * j) * V + i;
            Vec<float>::type q = {none, none, none, none};
            if (p && c < C) q = load_vec(p, c, C);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][i + k] = q[k];
        }
}

// a thread's share of a row
template <typename T, int TPR, int NCH>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int t, int C, typename Vec<T>::type (&v)[NCH]) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const int c0 = (t + TPR * j) * Vec<T>::N;
        if (c0 < C) {
            v[j] = load_vec(p, c0, C);
        } else {
#pragma unroll
            for (int i = 0; i < Vec<T>::N; ++i) v[j][i] = (T)0.f;
        }
    }
}

// A row group takes every gridDim-th row; the next row is requested before the current one is reduced, so that loads travel
// through the two reductions.
template <typename T, int TPR, int NT, int NCH>
__global__ __launch_bounds__(NT) void ln_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                    T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                    int64_t rows, int C, float eps) {
    constexpr int V = Vec<T>::N, G = NT / TPR;
    __shared__ float sh[2 * 32];
    int flip = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * G;
    typename Vec<T>::type cur[NCH], nxt[NCH];
    {
        const int64_t row = (int64_t)blockIdx.x * G + grp;
        load_row<T, TPR, NCH>(x + (row < rows ? row : rows - 1) * C, t, C, cur);
    }
    float wv[NCH][V], bv[NCH][V];
    load_params<T, TPR, NCH>(w, t, C, 1.f, wv);
    load_params<T, TPR, NCH>(b, t, C, 0.f, bv);
    const float invC = 1.f / (float)C;
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < rows; r0 += step) {   // uniform: every wave reaches each barrier
        const int64_t row = r0 + grp, after = row + step;
        const bool live = row < rows;
        if (r0 + step < rows) load_row<T, TPR, NCH>(x + (after < rows ? after : rows - 1) * C, t, C, nxt);
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += (float)cur[j][i];
        row_sum<TPR, 1>(s, sh, flip);
        const float near = product(s[0], invC);
        float q[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = (float)cur[j][i] - near;
                if ((t + TPR * j) * V + i < C) { q[0] += d; q[1] += d * d; }
            }
        row_sum<TPR, 2>(q, sh, flip);
        float mu, rs;
        row_stats(near, q[0] * invC, q[1] * invC, eps, mu, rs);
        if (live) {
            if (t == 0) { mean[row] = mu; rstd[row] = rs; }
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int c0 = (t + TPR * j) * V;
                if (c0 < C) {
                    typename Vec<T>::type o;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = (T)(((float)cur[j][i] - mu) * rs * wv[j][i] + bv[j][i]);
                    store_vec(y + row * C, c0, C, o);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) cur[j] = nxt[j];
    }
}

// any C: a workgroup walks its row three times (the second and third read come from the caches)
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                           T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                           int64_t rows, int C, float eps) {
    constexpr int V = Vec<T>::N;
    __shared__ float sh[2 * 32];
    int flip = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * C;
        float s[1] = {0.f};
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < C; c0 += 1024 * V) {
            const auto q = load_vec(xr, (int)c0, C);
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += (float)q[i];
        }
        row_sum<1024, 1>(s, sh, flip);
        const float near = s[0] / (float)C;
        float q2[2] = {0.f, 0.f};
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < C; c0 += 1024 * V) {
            const auto q = load_vec(xr, (int)c0, C);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = (float)q[i] - near;
                if (c0 + i < C) { q2[0] += d; q2[1] += d * d; }
            }
        }
        row_sum<1024, 2>(q2, sh, flip);
        float mu, rs;
        row_stats(near, q2[0] / (float)C, q2[1] / (float)C, eps, mu, rs);
        if (threadIdx.x == 0) { mean[row] = mu; rstd[row] = rs; }
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < C; c0 += 1024 * V) {
            const auto q = load_vec(xr, (int)c0, C);
            typename Vec<T>::type o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (int)c0 + i;
                const float wi = w && c < C ? w[c] : 1.f, bi = b && c < C ? b[c] : 0.f;
                o[i] = (T)(((float)q[i] - mu) * rs * wi + bi);
            }
            store_vec(y + row * C, (int)c0, C, o);
        }
    }
}

// partial: [gridDim.x][2][C] column sums {dy xh, dy} of the workgroup's rows, or null
template <typename T, int TPR, int NT, int NCH>
__global__ __launch_bounds__(NT) void ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                                                    const float* __restrict__ rstd, const float* __restrict__ w, T* __restrict__ dx,
                                                    float* __restrict__ partial, int64_t rows, int C) {
    constexpr int V = Vec<T>::N, G = NT / TPR;
    __shared__ float sh[2 * 32];
    extern __shared__ float col[];                    // [G / 2][C]: the join of the row groups
    int flip = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * G;
    typename Vec<T>::type xq[NCH], gq[NCH], xn[NCH], gn[NCH];
    float mu, rs, mun = 0.f, rsn = 0.f;
    {
        int64_t row = (int64_t)blockIdx.x * G + grp;
        row = row < rows ? row : rows - 1;
        load_row<T, TPR, NCH>(x + row * C, t, C, xq);
        load_row<T, TPR, NCH>(dy + row * C, t, C, gq);
        mu = mean[row];
        rs = rstd[row];
    }
    float wv[NCH][V], aw[NCH][V], ab[NCH][V];
    load_params<T, TPR, NCH>(w, t, C, 1.f, wv);
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) { aw[j][i] = 0.f; ab[j][i] = 0.f; }
    const float invC = 1.f / (float)C;
    for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < rows; r0 += step) {
        const int64_t row = r0 + grp;
        const bool live = row < rows;
        if (r0 + step < rows) {
            const int64_t after = row + step < rows ? row + step : rows - 1;
            load_row<T, TPR, NCH>(x + after * C, t, C, xn);
            load_row<T, TPR, NCH>(dy + after * C, t, C, gn);
            mun = mean[after];
            rsn = rstd[after];
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = ((float)xq[j][i] - mu) * rs, d = (float)gq[j][i], g = d * wv[j][i];   // beyond C: dy = 0
                s[0] += g;
                s[1] += g * xh;
                if (live) { aw[j][i] += d * xh; ab[j][i] += d; }
            }
        row_sum<TPR, 2>(s, sh, flip);
        const float c1 = s[0] * invC, c2 = s[1] * invC;
        if (live && dx != nullptr) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int c0 = (t + TPR * j) * V;
                if (c0 < C) {
                    typename Vec<T>::type o;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float xh = ((float)xq[j][i] - mu) * rs, g = (float)gq[j][i] * wv[j][i];
                        o[i] = (T)(rs * (g - c1 - xh * c2));
                    }
                    store_vec(dx + row * C, c0, C, o);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) { xq[j] = xn[j]; gq[j] = gn[j]; }
        mu = mun;
        rs = rsn;
    }
    if (partial == nullptr) return;
    if (G > 1) {                                      // the upper half of the groups to the lower half, down to one: fixed order
        auto join = [&](float (&a)[NCH][V]) {
#pragma unroll
            for (int half = G / 2; half > 0; half /= 2) {
                __syncthreads();
                if (grp >= half && grp < 2 * half)
#pragma unroll
                    for (int j = 0; j < NCH; ++j)
                        if ((t + TPR * j) * V < C)
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                if ((t + TPR * j) * V + i < C) col[(grp - half) * C + (t + TPR * j) * V + i] = a[j][i];
                __syncthreads();
                if (grp < half)
#pragma unroll
                    for (int j = 0; j < NCH; ++j)
                        if ((t + TPR * j) * V < C)
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                if ((t + TPR * j) * V + i < C) a[j][i] += col[grp * C + (t + TPR * j) * V + i];
            }
        };
        join(aw);
        join(ab);
    }
    if (grp == 0) {
        float* out = partial + (size_t)blockIdx.x * 2 * C;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const int c = (t + TPR * j) * V + i;
                if (c < C) {
                    Vec<float>::type p, q;
#pragma unroll
                    for (int k = 0; k < 4; ++k) { p[k] = aw[j][i + k]; q[k] = ab[j][i + k]; }
                    store_vec(out, c, C, p);
                    store_vec(out + C, c, C, q);
                }
            }
    }
}

// any C: dx alone, two reads of the row
template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, const float* __restrict__ w,
                                                           T* __restrict__ dx, int64_t rows, int C) {
    constexpr int V = Vec<T>::N;
    __shared__ float sh[2 * 32];
    int flip = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t at = row * C;
        const float mu = mean[row], rs = rstd[row];
        float s[2] = {0.f, 0.f};
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < C; c0 += 1024 * V) {
            const auto xq = load_vec(x + at, (int)c0, C);
            const auto gq = load_vec(dy + at, (int)c0, C);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (int)c0 + i;
                const float g = (float)gq[i] * (w && c < C ? w[c] : 1.f);
                s[0] += g;
                s[1] += g * (((float)xq[i] - mu) * rs);
            }
        }
        row_sum<1024, 2>(s, sh, flip);
        const float c1 = s[0] / (float)C, c2 = s[1] / (float)C;
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < C; c0 += 1024 * V) {
            const auto xq = load_vec(x + at, (int)c0, C);
            const auto gq = load_vec(dy + at, (int)c0, C);
            typename Vec<T>::type o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (int)c0 + i;
                const float g = (float)gq[i] * (w && c < C ? w[c] : 1.f);
                o[i] = (T)(rs * (g - c1 - (((float)xq[i] - mu) * rs) * c2));
            }
            store_vec(dx + at, (int)c0, C, o);
        }
    }
}

// any C: the column sums of a slab of rows, one thread per column
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, float* __restrict__ partial, int64_t rows, int C) {
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = per * blockIdx.y, r1 = r0 + per < rows ? r0 + per : rows;
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float aw = 0.f, ab = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float d = (float)dy[r * C + c];
        aw += d * (((float)x[r * C + c] - mean[r]) * rstd[r]);
        ab += d;
    }
    float* out = partial + (size_t)blockIdx.y * 2 * C;
    out[c] = aw;
    out[C + c] = ab;
}

// dw / db: columns of partial [parts][2][C] in fixed order; 32 columns x 32 row strands per workgroup
__global__ __launch_bounds__(1024) void ln_param_grads_kernel(const float* __restrict__ partial, int parts, int C, float* __restrict__ dw,
                                                              float* __restrict__ db) {
    __shared__ float sh[32][33];
    const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;       // column of the flattened [2][C]
    const int64_t W = 2 * (int64_t)C;
    float s = 0.f;
    if (c < W)
        for (int p = strand; p < parts; p += 32) s += partial[p * W + c];
    sh[strand][lane] = s;
    __syncthreads();
    if (strand == 0 && c < W) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += sh[k][lane];
        float* out = c < C ? dw : db;
        if (out) out[c < C ? c : c - C] = t;
    }
}

// Threads per row and 16-byte vectors per thread: the fewest threads whose registers hold the row beside the parameters (and, in the
// backward pass, the column sums and the next row: 128 registers a thread at 1024 threads).  One wave per row needs no barrier.
// Longer rows take the kernels that read a row two or three times.  Those cost 131 us forward and 155 us backward at 2000 x 16384
// bf16 where the registers take 30 and 97 (with 141 values spilled); at 2000 x 16384 fp32 they take 152 us backward, where four
// vectors a thread (251 spilled) took 181.
struct LnShape { int tpr, nch; };
inline LnShape ln_shape(int C, int V, bool bwd) {
    const int64_t vecs = ((int64_t)C + V - 1) / V;
    const int most = bwd ? (V == 8 ? 1 : 2) : (V == 8 ? 2 : 4);
    for (int tpr = 64; tpr <= 1024; tpr *= V == 8 || bwd ? 2 : 4)
        for (int n = 1; n <= most; n *= 2)
            if (vecs <= (int64_t)tpr * n) return {tpr, n};
    if (bwd && V == 8 && vecs <= 2048) return {1024, 2};
    return {0, 0};
}

template <typename T, int TPR, int NCH>
int launch_fwd(const void* x, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t rows, int C, float eps, hipStream_t st) {
    constexpr int NT = TPR > 256 ? TPR : 256, G = NT / TPR;
    const int64_t blocks = (rows + G - 1) / G, most = 256 * (1024 / NT);
    hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NT, NCH>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(NT), 0, st, (const T*)x, w, b,
                       (T*)y, mean, rstd, rows, C, eps);
    return (int)hipGetLastError();
}

// Workgroups of the backward pass: 1024 threads, one per CU, if that gives every CU one (16384 x 1024 bf16: 28.7 us; 512 of 256
// threads 31.4, 256 of them 44.3) or a row takes 512 threads (300 x 4096 fp32: 11.3 us; one row a workgroup, with twice the partial
// sums, 13.6); else 256 threads, so that few rows still reach many CUs (1008 x 512 bf16: 9.4 us; 1024 threads 11.2).
struct LnGrid { int nt, parts; };
inline LnGrid ln_grid(int64_t rows, int C, int dtype) {
    const LnShape s = ln_shape(C, dtype == kF32 ? 4 : 8, true);
    if (!s.tpr) return {1024, (int)(rows < 32 ? rows : 32)};           // very long rows: few slabs bound the workspace
    const int64_t g = 1024 / s.tpr, wide = (rows + g - 1) / g;
    if (s.tpr >= 512 || wide >= 256) return {1024, (int)(wide < 256 ? wide : 256)};
    return {256, (int)((rows * s.tpr + 255) / 256)};
}

template <typename T, int TPR, int NT, int NCH>
int launch_bwd_of(const void* dy, const void* x, const float* mean, const float* rstd, const float* w, void* dx, float* partial, int64_t rows,
                  int C, int parts, hipStream_t st) {
    const size_t lds = partial && TPR < NT ? (size_t)(NT / TPR / 2) * C * sizeof(float) : 0;
    hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NT, NCH>), dim3((unsigned)parts), dim3(NT), lds, st, (const T*)dy, (const T*)x, mean, rstd, w, (T*)dx,
                       partial, rows, C);
    return (int)hipGetLastError();
}
template <typename T, int TPR, int NCH>
int launch_bwd(const void* dy, const void* x, const float* mean, const float* rstd, const float* w, void* dx, float* partial, int64_t rows,
               int C, const LnGrid& g, hipStream_t st) {
    if constexpr (TPR <= 256)
        if (g.nt == 256) return launch_bwd_of<T, TPR, 256, NCH>(dy, x, mean, rstd, w, dx, partial, rows, C, g.parts, st);
    return launch_bwd_of<T, TPR, 1024, NCH>(dy, x, mean, rstd, w, dx, partial, rows, C, g.parts, st);
}

template <typename T>
int ln_fwd(const void* x, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t rows, int C, float eps, hipStream_t st) {
    const LnShape s = ln_shape(C, Vec<T>::N, false);
#define SSECG_LN_CASE(TPR, NCH) if (s.tpr == TPR && s.nch == NCH) return launch_fwd<T, TPR, NCH>(x, w, b, y, mean, rstd, rows, C, eps, st)
    SSECG_LN_CASE(64, 1); SSECG_LN_CASE(64, 2); SSECG_LN_CASE(256, 2); SSECG_LN_CASE(1024, 2);
    if constexpr (Vec<T>::N == 4) {
        SSECG_LN_CASE(64, 4); SSECG_LN_CASE(256, 4); SSECG_LN_CASE(1024, 4);
    } else {
        SSECG_LN_CASE(128, 2); SSECG_LN_CASE(512, 2);
    }
#undef SSECG_LN_CASE
    hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3((unsigned)(rows < 512 ? rows : 512)), dim3(1024), 0, st, (const T*)x, w, b, (T*)y, mean,
                       rstd, rows, C, eps);
    return (int)hipGetLastError();
}

template <typename T>
int ln_bwd(const void* dy, const void* x, const float* mean, const float* rstd, const float* w, void* dx, float* partial, int64_t rows, int C,
           const LnGrid& g, hipStream_t st) {
    const LnShape s = ln_shape(C, Vec<T>::N, true);
#define SSECG_LN_CASE(TPR, NCH) if (s.tpr == TPR && s.nch == NCH) return launch_bwd<T, TPR, NCH>(dy, x, mean, rstd, w, dx, partial, rows, C, g, st)
    SSECG_LN_CASE(64, 1); SSECG_LN_CASE(1024, 2);
    if constexpr (Vec<T>::N == 4) {
        SSECG_LN_CASE(64, 2); SSECG_LN_CASE(128, 2); SSECG_LN_CASE(256, 2); SSECG_LN_CASE(512, 2);
    } else {
        SSECG_LN_CASE(128, 1); SSECG_LN_CASE(256, 1); SSECG_LN_CASE(512, 1); SSECG_LN_CASE(1024, 1);
    }
#undef SSECG_LN_CASE
    if (dx)
        hipLaunchKernelGGL((ln_bwd_long_kernel<T>), dim3((unsigned)(rows < 512 ? rows : 512)), dim3(1024), 0, st, (const T*)dy, (const T*)x, mean,
                           rstd, w, (T*)dx, rows, C);
    if (partial)
        hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3((unsigned)((C + 255) / 256), (unsigned)g.parts), dim3(256), 0, st, (const T*)dy,
                           (const T*)x, mean, rstd, partial, rows, C);
    return (int)hipGetLastError();
}

constexpr int kMaxC = 1 << 24;

}  // namespace

extern "C" {

int ssecg_layer_norm_fwd(const void* x, const float* weight, const float* bias, int dtype, int64_t rows, int C, double eps, void* y,
                         float* mean, float* rstd, void* stream) {
    if (!x || !y || !mean || !rstd || !dtype_ok(dtype) || rows <= 0 || C <= 0 || C > kMaxC || !(eps >= 0.0)) return SSECG_E_INVAL;
    SSECG_LM_DTYPE(dtype, T, return ln_fwd<T>(x, weight, bias, y, mean, rstd, rows, C, (float)eps, (hipStream_t)stream));
}

size_t ssecg_layer_norm_bwd_workspace(int dtype, int64_t rows, int C) {
    if (!dtype_ok(dtype) || rows <= 0 || C <= 0 || C > kMaxC) return 0;
    return (size_t)ln_grid(rows, C, dtype).parts * 2 * C * sizeof(float);
}

int ssecg_layer_norm_bwd(const void* dy, const void* x, const float* mean, const float* rstd, const float* weight, int dtype, int64_t rows,
                         int C, void* dx, float* dweight, float* dbias, float* workspace, size_t workspace_bytes, void* stream) {
    const bool params = dweight || dbias;
    if (!dy || !x || !mean || !rstd || !(dx || params) || !dtype_ok(dtype) || rows <= 0 || C <= 0 || C > kMaxC) return SSECG_E_INVAL;
    if (params && (!workspace || workspace_bytes < ssecg_layer_norm_bwd_workspace(dtype, rows, C))) return SSECG_E_WORKSPACE;
    const LnGrid g = ln_grid(rows, C, dtype);
    float* partial = params ? workspace : nullptr;
    int rc = 0;
    SSECG_LM_DTYPE(dtype, T, rc = ln_bwd<T>(dy, x, mean, rstd, weight, dx, partial, rows, C, g, (hipStream_t)stream));
    if (rc != 0 || !params) return rc;
    hipLaunchKernelGGL(ln_param_grads_kernel, dim3((unsigned)((2 * (int64_t)C + 31) / 32)), dim3(1024), 0, (hipStream_t)stream, partial, g.parts,
                       C, dweight, dbias);
    return (int)hipGetLastError();
}

}  // extern "C"
