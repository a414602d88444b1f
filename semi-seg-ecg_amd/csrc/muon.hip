// Orthogonalised updates of weight matrices: the quintic Newton-Schulz iteration and the optimiser step built on it, for many
// matrices of any sizes in one chain of launches.
//
//   X = U / (|U|_F + eps), the shorter side first (m <= n);   repeat:  A = X X^T,  P = a I + b A + c A A,  X = P X
//   optimiser: v = mu v + g,  U = g + mu v (Nesterov) or v,  p = p (1 - lr wd) - lr s X,  s = 0.2 sqrt(max(rows, cols)) or
//   sqrt(max(1, rows / cols))
//
// Every product is mm_core.h's.  A and P are symmetric: only the tiles on and below the diagonal are computed, and the epilogue
// writes the mirrored tile too.  X is read along its rows for A and across for the update.  The identity is folded into P, so the
// update needs no third operand.
//
// Precision: the iteration multiplies errors along weak directions by up to a = 3.44 per step (485 over five), so 16-bit iterates
// would lose them.  All matrices are two fp16 planes times 2^13 - singular values stay below 1.21 and P's below 3.45, far inside
// fp16's range - with fp32 accumulators.  An entry of a matrix whose norm is 1 keeps 22 to 23 bits down to 2^-16, fewer below, none below
// 2^-38: entries of 10^-9 have 7 bits left, in a direction that ends as 5e-7 of the result.  For results in fp32 the tiles form
// every product and the polynomial's roundings are carried along (kFull): over 300 matrices of up to 64 rows the median error is 0.67 of
// that of 32-bit products; at 4096 x 4096, where long sums count for most, 3.7e-6 against 3.6e-6.
//
// Large matrices are bound by the products' main loop: 4096 x 4096 takes 3.65 to 3.8 ms for five steps; an update's product 340 to 360 us
// (1.15 to 1.21 PFLOP/s of fp16 products; a large library product reaches 1.3 to 1.6), a symmetric one 204 to 227 us (0.95 to 1.0 of those
// that count: 253 tiles of one workgroup each, four waves, fill the 256 CUs once).  A model's matrices are bound by the chain: the
// optimiser step of a 1D ResNet18 (21 matrices up to 512 x 1536) takes 270 to 285 us over 17 launches of 10 to 35 us, each as long as its longest
// tile, a few dozen stages of latency; its update has 111 tiles for 256 CUs.
#include <initializer_list>
#include <type_traits>
#include <utility>
#include "mm_core.h"
#include "ssecg.h"

namespace {
using namespace ssecg_lm;

constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;
constexpr int kScale = 13;

// Both planes of kC v + kB w (+ kA on the diagonal), all times 2^13.  The three cancel to a fifth of the largest.  FULL: the sums' roundings
// and the coefficients' own (2^-25, the same in every entry and step) are carried along; what is left is the planes' rounding.
template <bool FULL>
__device__ __forceinline__ uint32_t poly_planes(float v, float w, bool diagonal) {
    if constexpr (!FULL) {
        return planes16((float)kC * v + ((float)kB * w + (diagonal ? (float)kA * (float)(1 << kScale) : 0.f)), 0.f);
    } else {
#pragma clang fp contract(off)
        constexpr float b = (float)kB, bl = (float)(kB - (double)b), c = (float)kC, cl = (float)(kC - (double)c);
        constexpr double a64 = kA * (double)(1 << kScale);
        constexpr float a = (float)a64, al = (float)(a64 - (double)a);
        const float p = b * w, r = c * v, one = diagonal ? a : 0.f;
        const float s = p + r, sp = s - p, se = (p - (s - sp)) + (r - sp);
        const float d = one + s, ds = d - one, de = (one - (d - ds)) + (s - ds);
        const float rest = ((__builtin_fmaf(b, w, -p) + __builtin_fmaf(c, v, -r)) + (se + de)) +
                           (__builtin_fmaf(bl, w, cl * v) + (diagonal ? al : 0.f));
        return planes16(d, rest);
    }
}

// a number as the sum of two in fp32
struct Two {
    float h, l;
    explicit __device__ __forceinline__ Two(double v) : h((float)v), l((float)(v - (double)h)) {
        if (__builtin_isinf(h)) l = 0.f;
    }
    // both planes of u times it
    template <bool FULL> __device__ __forceinline__ uint32_t planes(float u) const {
        if constexpr (!FULL) {
            return planes16(u * h, 0.f);
        } else {
#pragma clang fp contract(off)
            const float p = u * h;
            return planes16(p, __builtin_fmaf(u, h, -p) + u * l);
        }
    }
};

// A result in fp32 is held to what 32-bit products give; in 16 bits its rounding, in the optimiser the parameter's is far larger.
template <typename S, bool MUON> constexpr bool kFull = std::is_same<S, float>::value && !MUON;
constexpr int kNormParts = 1024;                  // most workgroups that share one matrix's norm
constexpr int kMost = 32;                         // matrices of one chain of launches: their table travels in the kernel arguments

// By value in the kernel arguments (1.9 KB): no upload, nothing to keep for a captured launch.  first[w][k]: the first workgroup
// of matrix k in the launch of kind w.
enum { wPrep, wGram, wUpd };
struct Table {
    const void* src[kMost]; void* dst[kMost]; float* mom[kMost];
    int64_t offset[kMost];                        // of the matrix's planes in the workspace
    int rows[kMost], cols[kMost], first[3][kMost];
    int count;
};

struct Mat {
    const void* src; void* dst; float* mom;
    int rows, cols, m, n;
    int64_t pn, pm;                               // bytes of a row of X; of A and P
    char *X[2], *A, *P;                           // operands of two planes (mm_core.h); an update reads one X and writes the other
};

inline __host__ __device__ int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// of one matrix in the workspace
inline __host__ __device__ int64_t mat_bytes(int64_t rows, int64_t cols) {
    const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    const int64_t pn = up(n, 32) * 4, pm = up(m, 32) * 4;
    return up(2 * m * pn + 2 * m * pm, 256);
}

__device__ __forceinline__ Mat load_mat(const Table& table, int k, char* ws, int from) {   // X[0] is number `from`
    Mat t;
    t.src = table.src[k];
    t.dst = table.dst[k];
    t.mom = table.mom[k];
    t.rows = table.rows[k];
    t.cols = table.cols[k];
    t.m = t.rows < t.cols ? t.rows : t.cols;
    t.n = t.rows < t.cols ? t.cols : t.rows;
    t.pn = up(t.n, 32) * 4;
    t.pm = up(t.m, 32) * 4;
    char* base = ws + table.offset[k];
    t.X[0] = base + from * (t.m * t.pn);
    t.X[1] = base + (1 - from) * (t.m * t.pn);
    t.A = base + 2 * t.m * t.pn;
    t.P = t.A + t.m * t.pm;
    return t;
}

// the matrix whose workgroups of kind w hold workgroup q; every wave finds it by itself
__device__ __forceinline__ int find_mat(const Table& table, int w, int q, int& first) {
    const int lane = threadIdx.x & (kMost - 1);
    const unsigned long long le = __ballot((threadIdx.x & 63) < kMost && lane < table.count && table.first[w][lane] <= q);
    const int k = __builtin_amdgcn_readfirstlane(__popcll(le) - 1);
    first = table.first[w][k];
    return k;
}

struct Apply {                                    // the step's scalars; where they are on the device, a captured launch reads them anew
    double lr, weight_decay;
    int adjust;                                   // 0: sqrt(max(1, rows / cols)); 1: 0.2 sqrt(max(rows, cols))
    float momentum;
    const double* lr_dev;
    const double* scalars;                        // {lr, weight_decay, momentum}, or null
    __device__ __forceinline__ float mu() const { return scalars != nullptr ? (float)scalars[2] : momentum; }
    __device__ __forceinline__ double rate() const { return scalars != nullptr ? scalars[0] : lr_dev != nullptr ? lr_dev[0] : lr; }
    __device__ __forceinline__ double decay() const { return scalars != nullptr ? scalars[1] : weight_decay; }
};

// U of element i (momentum already advanced): Nesterov g + mu v, else v; without momentum g
template <typename S, bool MUON>
__device__ __forceinline__ float update_of(const Mat& t, int64_t i, float mu, int nesterov) {
    const float g = (float)reinterpret_cast<const S*>(t.src)[i];
    if (!MUON) return g;
    const float v = t.mom[i];
    return nesterov ? g + mu * v : v;
}

// momentum and the partial sums of |U|^2 (fp64: no gradient's scale overflows it); partial [count][gridDim.x]
template <typename S, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(Table table, Apply ap, int nesterov, const float* __restrict__ skip,
                                                      double* __restrict__ partial) {
    if (MUON && skip != nullptr && skip[0] != 0.f) return;
    const float mu = MUON ? ap.mu() : 0.f;
    const Mat t = load_mat(table, blockIdx.y, nullptr, 0);
    const int64_t n = (int64_t)t.rows * t.cols;
    constexpr int V = Vec<S>::N;
    const S* src = reinterpret_cast<const S*>(t.src);
    double s = 0.0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += (int64_t)gridDim.x * 256 * V) {
        const int left = n - i < V ? (int)(n - i) : V;
        const auto g = load_vec(src + i, 0, left);
        if constexpr (MUON) {
            auto v = load_vec(t.mom + i, 0, left);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = mu * v[j] + g[j];
                const float u = nesterov ? g[j] + mu * v[j] : v[j];
                s += (double)u * (double)u;               // beyond the end: zeros
            }
            store_vec(t.mom + i, 0, left, v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) s += (double)(float)g[j] * (double)(float)g[j];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __shared__ double sh[4];
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// U / (norm + eps) as an operand, the shorter side first; one workgroup: 64 x 64 elements, zeros up to the pitch
template <typename S, bool MUON>
__global__ __launch_bounds__(256) void ns_prep_kernel(Table table, char* __restrict__ ws, Apply ap, int nesterov,
                                                      int parts, double eps, const float* __restrict__ skip, const double* __restrict__ partial) {
    if (MUON && skip != nullptr && skip[0] != 0.f) return;
    const float mu = MUON ? ap.mu() : 0.f;
    __shared__ uint32_t tile[64][65];
    int first;
    const int k = find_mat(table, wPrep, blockIdx.x, first);
    const Mat t = load_mat(table, k, ws, 0);
    double s = 0.0;
    const int lane = threadIdx.x & 63, strand = threadIdx.x >> 6;
    for (int p = lane; p < parts; p += 64) s += partial[(int64_t)k * parts + p];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    const Two f((double)(1 << kScale) / (sqrt(s) + eps));
    const int tiles = (int)((up(t.cols, 32) + 63) / 64), q0 = blockIdx.x - first;
    const int64_t rb = (int64_t)(q0 / tiles) * 64, cb = (int64_t)(q0 % tiles) * 64;
    for (int i = strand; i < 64; i += 4) {
        const int64_t r = rb + i, c = cb + lane;
        uint32_t q = 0;
        if (r < t.rows && c < t.cols) q = f.planes<kFull<S, MUON>>(update_of<S, MUON>(t, r * t.cols + c, mu, nesterov));
        tile[i][lane] = q;
    }
    __syncthreads();
    const bool tall = t.rows > t.cols;
    const int64_t row0 = tall ? cb : rb, k0 = tall ? rb : cb;
    for (int u = threadIdx.x; u < 512; u += 256) {
        const int i = u >> 3, c8 = (u & 7) * 8;
        if (row0 + i >= t.m || kbyte<2>(k0 + c8) >= t.pn) continue;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = tall ? tile[c8 + j][i] : tile[i][c8 + j];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = (w[2 * j] >> 16 * q & 0xffffu) | w[2 * j + 1] >> 16 * q << 16;
            *reinterpret_cast<u32x4*>(t.X[0] + (row0 + i) * t.pn + kbyte<2>(k0 + c8, q)) = a;
        }
    }
}

// Tile q of the lower triangle of a square of tiles: row ti >= column tj
__device__ __forceinline__ void tri_tile(int q, int& ti, int& tj) {
    ti = (int)((sqrtf(8.f * (float)q + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > q) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= q) ++ti;
    tj = q - ti * (ti + 1) / 2;
}

// The same triangle of T rows of tiles in blocks of S x S tiles, so that the tiles of one XCD, which follow each other, share few rows of
// the operand: those of one row of tiles would each read different ones (4096 x 4096 in tiles of 64: 5.05 -> 4.63 ms, of 256: 4.63 ->
// 4.39; small matrices: the same).  S = 1 is the order by rows: tiles of 192 are better off with it at every size (five steps at 1500 /
// 3000 / 4096 / 6000 square: 866 / 2022 / 3647 / 13827 us; in blocks of 6: 903 / 2094 / 3706 / 14171).
template <int S>
__device__ __forceinline__ void tri_block(int q, int T, int& ti, int& tj) {
    tri_tile(q, ti, tj);
    const int I = ti / S, r0 = I * S, rows = T - r0 < S ? T - r0 : S, in = q - r0 * (r0 + 1) / 2;   // the rows before r0 come first either way
    if (in < rows * r0) {
        const int J = in / (rows * S), k = in - J * rows * S;
        ti = r0 + k % rows;
        tj = J * S + k / rows;
    } else {
        tri_tile(in - rows * r0, ti, tj);
        ti += r0;
        tj += r0;
    }
}

// POLY = false: A = X X^T.  POLY = true: P = a I + b A + c A A.
template <class M, bool POLY>
__global__ __launch_bounds__(M::NT, M::TM * M::TN > 8 ? 1 : 2) void ns_gram_kernel(Table table, char* __restrict__ ws, int from,
                                                        const float* __restrict__ skip) {
    if (skip != nullptr && skip[0] != 0.f) return;
    __shared__ __attribute__((aligned(16))) char lds[M::LDS];
    int first, ti, tj;
    const int tile = xcd_tile(blockIdx.x, gridDim.x);
    const Mat t = load_mat(table, find_mat(table, wGram, tile, first), ws, from);
    tri_block<(M::BM == 192 ? 1 : M::BM == 256 ? 6 : 8)>(tile - first, (t.m + M::BM - 1) / M::BM, ti, tj);
    const int a0 = ti * M::BM, b0 = tj * M::BN;
    const int64_t pitch = POLY ? t.pm : t.pn;
    const Operand op = {POLY ? t.A : t.X[0], pitch, t.m};
    f32x16 acc[M::TM][M::TN];
    if (!M::run(op, a0, op, b0, 0, (int)(pitch / M::STEP), lds, acc)) return;
    char* out = POLY ? t.P : t.A;
    constexpr float down = 1.f / (float)(1 << kScale);
#pragma unroll
    for (int j = 0; j < M::TN; ++j) {
        const int c = b0 + M::bcol(j);
#pragma unroll
        for (int i = 0; i < M::TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int r = a0 + M::arow(i, e);            // 4 consecutive rows
                float w[4] = {0.f, 0.f, 0.f, 0.f};
                if (POLY && c < t.m && r < t.m) {            // A[r..r+3][c] = A[c][r..r+3]
                    const char* s = t.A + (int64_t)c * t.pm;
                    _Float16 hi[4], lo[4];
                    u32x2 q = *reinterpret_cast<const u32x2*>(s + kbyte<2>(r));
                    __builtin_memcpy(hi, &q, 8);
                    q = *reinterpret_cast<const u32x2*>(s + kbyte<2>(r, 1));
                    __builtin_memcpy(lo, &q, 8);
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = (float)hi[k] + (float)lo[k];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {                // from here on both planes of the value, in its register
                    const float d = acc[i][j][e + k] * down;
                    const uint32_t q = POLY ? poly_planes<M::FULL>(d, w[k], r + k == c) : planes16(d, 0.f);
                    acc[i][j][e + k] = __builtin_bit_cast(float, r + k < t.m && c < t.m ? q : 0u);
                }
            }
    }
    using W = WaveStore<M>;
    char* reg = W::region(lds);
    const int r0 = a0 + M::wave_row(), c0 = b0 + M::wave_col();
    auto val = [&](int i, int j, int e, int q) -> uint16_t {
        const float both = acc[i][j][e];
        return (uint16_t)(__builtin_bit_cast(uint32_t, both) >> 16 * q);
    };
    auto put = [&](int r, int c, int q, u32x4 d) {
        if (r < t.m && kbyte<2>(c) < t.pm) *reinterpret_cast<u32x4*>(out + (int64_t)r * t.pm + kbyte<2>(c, q)) = d;
    };
    W::template store_rows<2>(reg, val, [&](int r, int c, int q, u32x4 d) { put(r0 + r, c0 + c, q, d); });
    // below the diagonal: the mirrored tile as well
    if (ti != tj) W::template store_cols<2>(reg, val, [&](int c, int r, int q, u32x4 d) { put(c0 + c, r0 + r, q, d); });
}

__device__ __forceinline__ double update_scale(const Mat& t, int adjust) {
    return adjust == 1 ? 0.2 * sqrt((double)t.n) : sqrt(t.rows > t.cols ? (double)t.rows / (double)t.cols : 1.0);
}

// X = P X, from X number `from` to the other, or the last one: the result / the parameter's update
template <class M, typename S, int LAST>          // LAST: 0 = planes, 1 = result, 2 = optimiser
__global__ __launch_bounds__(M::NT, M::TM * M::TN > 8 ? 1 : 2) void ns_update_kernel(Table table, char* __restrict__ ws, int from, Apply ap,
                                                          const float* __restrict__ skip) {
    if (skip != nullptr && skip[0] != 0.f) return;
    __shared__ __attribute__((aligned(16))) char lds[M::LDS];
    int first;
    const int tile = xcd_tile(blockIdx.x, gridDim.x);
    const Mat t = load_mat(table, find_mat(table, wUpd, tile, first), ws, from);
    const int tm = (t.m + M::BM - 1) / M::BM, q = tile - first;
    const int a0 = q % tm * M::BM, b0 = q / tm * M::BN;
    const Operand P = {t.P, t.pm, t.m}, X = {t.X[0], t.pn, t.m};
    f32x16 acc[M::TM][M::TN];
    if (!M::run(P, a0, X, b0, 0, (int)(t.pm / M::STEP), lds, acc)) return;
    constexpr float down = 1.f / (float)(1 << kScale);
    using W = WaveStore<M>;
    char* reg = W::region(lds);
    const int r0 = a0 + M::wave_row(), c0 = b0 + M::wave_col();
    if constexpr (LAST == 0) {
#pragma unroll
        for (int j = 0; j < M::TN; ++j) {
            const int c = b0 + M::bcol(j);
#pragma unroll
            for (int i = 0; i < M::TM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = a0 + M::arow(i, e) < t.m && c < t.n ? acc[i][j][e] * down : 0.f;
        }
        W::template store_rows<2>(reg, [&](int i, int j, int e, int q) -> uint16_t { return plane16(acc[i][j][e], q); },
                                  [&](int r, int c, int q, u32x4 d) {
                                      if (r0 + r < t.m && kbyte<2>(c0 + c) < t.pn)
                                          *reinterpret_cast<u32x4*>(t.X[1] + (int64_t)(r0 + r) * t.pn + kbyte<2>(c0 + c, q)) = d;
                                  });
        return;
    }
    const bool tall = t.rows > t.cols;
    if constexpr (LAST == 1 && sizeof(S) == 2) {
        auto val = [&](int i, int j, int e, int) -> uint16_t { return bits16((S)(acc[i][j][e] * (down * down))); };
        S* out = reinterpret_cast<S*>(t.dst);
        auto put = [&](int r, int c, u32x4 d) {
            if (r < t.rows && c < t.cols) store_vec(out + (int64_t)r * t.cols, c, t.cols, __builtin_bit_cast(typename Vec<S>::type, d));
        };
        if (tall) W::template store_cols<1>(reg, val, [&](int c, int r, int, u32x4 d) { put(c0 + c, r0 + r, d); });
        else W::template store_rows<1>(reg, val, [&](int r, int c, int, u32x4 d) { put(r0 + r, c0 + c, d); });
        return;
    }
    float step = 0.f, keep = 0.f;
    if (LAST == 2) {
        const double lr = ap.rate();
        step = (float)(lr * update_scale(t, ap.adjust));
        keep = (float)(1.0 - lr * ap.decay());
    }
    float* out = reinterpret_cast<float*>(t.dst);
#pragma unroll
    for (int j = 0; j < M::TN; ++j) {
        const int c = b0 + M::bcol(j);
#pragma unroll
        for (int i = 0; i < M::TM; ++i) {
            auto at = [&](int e) { const int64_t r = a0 + M::arow(i, e); return tall ? (int64_t)c * t.cols + r : r * t.cols + c; };
            float old[16];
            if (LAST == 2)                              // 16 loads in flight, then the stores
#pragma unroll
                for (int e = 0; e < 16; ++e) old[e] = c < t.n && a0 + M::arow(i, e) < t.m ? out[at(e)] : 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = acc[i][j][e] * (down * down);
                if (c < t.n && a0 + M::arow(i, e) < t.m) out[at(e)] = LAST == 1 ? v : old[e] * keep - step * v;
            }
        }
    }
}

// ---------------------------------------------------------------- small matrices: the whole iteration in one workgroup
// A matrix whose X, A and P fit the LDS of a CU (160 KB) needs no launch between the steps: 17 launches become one.  Five steps take
// 40 us at 64 x 192 (84 by the chain of launches), 59 at 64 x 400 (95), 53 at 32 x 1024 (109), 23 at 8 x 8 (58), and 41 for thirty of
// 64 x 192 (88); 16-bit results and the optimiser, which need no full precision, 36 at 64 x 192.  One matrix that does not fit sends all
// of a call's through the chain, where they cost nothing beside it.
// What bounds it is instructions: a phase lasts as long as its busiest wave.  So the 32 x 32 blocks of a product and shares of its k
// go over all sixteen waves, the sums meet in LDS in fp32, and every thread joins and splits four values of the result.  Rows are
// padded by 16 bytes, so that 16 rows read at one k lie in different banks.  X is updated in place, between two barriers.
constexpr int kSmallWaves = 16, kSmallLds = 160 * 1024 - 256;
constexpr int kSmallPairs = 2;                    // 32 x 32 blocks of X that a wave updates at most
inline __host__ __device__ int64_t small_planes(int64_t m, int64_t n) {
    const int64_t mp = up(m, 32), np = up(n, 32);
    return mp * (np * 4 + 16) + 2 * mp * (mp * 4 + 16);
}
// waves that share the k of a block of A: what LDS leaves for their sums (4 KB a block each), 8 at most
inline __host__ __device__ int small_shares(int64_t m, int64_t n) {
    const int64_t blocks = m > 32 ? 4 : 1;
    for (int s = m > 32 ? 4 : 8; s > 0; s /= 2)
        if (small_planes(m, n) + s * blocks * 4096 <= kSmallLds) return s;
    return 0;
}
inline bool small_ok(int64_t rows, int64_t cols) {
    const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    return m <= 64 && n <= 1024 && up(m, 32) / 32 * (up(n, 32) / 32) <= kSmallWaves * kSmallPairs && small_shares(m, n) > 0;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// rows r of a block at k 16 kk + 8 h .. + 7, plane q (k fast)
__device__ __forceinline__ f16x8 small_along(const char* base, int64_t pitch, int row, int kk, int h, int q) {
    return *reinterpret_cast<const f16x8*>(base + row * pitch + kbyte<2>(16 * kk + 8 * h, q));
}
// columns 32 blk + r at rows 16 kk + 8 h .. + 7, plane q (k slow)
__device__ __forceinline__ f16x8 small_across(const char* base, int64_t pitch, int lane, int blk, int kk, int q) {
    const int l = lane & 15, g = lane >> 4, k = 16 * kk + 8 * (g >> 1) + (l >> 2);
    const char* p = base + k * pitch + blk * 128 + q * 64 + 32 * (g & 1) + 8 * (l & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * pitch));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ void small_put(char* base, int64_t pitch, int row, int col, uint32_t q) {   // both planes
    char* d = base + row * pitch + (col >> 5) * 128 + (col & 31) * 2;
    *reinterpret_cast<uint16_t*>(d) = (uint16_t)q;
    *reinterpret_cast<uint16_t*>(d + 64) = (uint16_t)(q >> 16);
}

template <typename S, bool MUON>
__global__ __launch_bounds__(kSmallWaves * 64) void ns_small_kernel(Table table, int nesterov, int steps, double eps, Apply ap,
                                                                       const float* __restrict__ skip) {
    if (MUON && skip != nullptr && skip[0] != 0.f) return;
    const float mu = MUON ? ap.mu() : 0.f;
    __shared__ __attribute__((aligned(16))) char lds[kSmallLds];
    __shared__ double sums[kSmallWaves];
    constexpr bool FULL = kFull<S, MUON>;
    const Mat t = load_mat(table, blockIdx.x, nullptr, 0);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h = lane >> 5;
    const int mp = (int)up(t.m, 32), np = (int)up(t.n, 32), lb = mp >> 6, mb = 1 << lb;   // 32 or 64 rows: 1 or 2 blocks, lb = log2
    const int64_t px = np * 4 + 16, pa = mp * 4 + 16;
    char *X = lds, *A = X + mp * px, *P = A + mp * pa;
    float* scratch = reinterpret_cast<float*>(P + mp * pa);
    const bool tall = t.rows > t.cols;
    // norm and momentum; X's pads are zeros
    double s = 0.0;
    const int count = t.rows * t.cols;                             // at most 32 blocks of 1024
    constexpr int V = Vec<S>::N;
    const S* src = reinterpret_cast<const S*>(t.src);
#pragma unroll 2
    for (int i = threadIdx.x * V; i < count; i += kSmallWaves * 64 * V) {
        const int left = count - i < V ? count - i : V;
        const auto g = load_vec(src + i, 0, left);
        if constexpr (MUON) {
            auto v = load_vec(t.mom + i, 0, left);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = mu * v[j] + g[j];
                const float u = nesterov ? g[j] + mu * v[j] : v[j];
                s += (double)u * (double)u;                        // beyond the end: zeros
            }
            store_vec(t.mom + i, 0, left, v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) s += (double)(float)g[j] * (double)(float)g[j];
        }
    }
    for (int i = threadIdx.x * 16; i < mp * px; i += kSmallWaves * 64 * 16) *reinterpret_cast<u32x4*>(X + i) = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) s += sums[w];
    const Two f((double)(1 << kScale) / (sqrt(s) + eps));
#pragma unroll 2
    for (int i = threadIdx.x * V; i < count; i += kSmallWaves * 64 * V) {   // (a thread reads the momentum that it wrote)
        const int left = count - i < V ? count - i : V;
        const auto g = load_vec(src + i, 0, left);
        typename Vec<float>::type v = {};
        if constexpr (MUON) v = load_vec(t.mom + i, 0, left);
        int row = i / t.cols, col = i - row * t.cols;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float u = (float)g[j];
            if constexpr (MUON) u = nesterov ? u + mu * v[j] : v[j];
            if (j < left) small_put(X, px, tall ? col : row, tall ? row : col, f.planes<FULL>(u));
            if (++col == t.cols) { col = 0; ++row; }
        }
    }
    __syncthreads();
    constexpr float down = 1.f / (float)(1 << kScale);
    using F = Frag<_Float16>;
    const int blocks = mb * mb, shares = small_shares(t.m, t.n), pairs = mb * (np / 32);
    auto zero = [](f32x16& v) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0.f;
    };
    for (int step = 0; step < steps; ++step) {
#pragma unroll 1
        for (int phase = 0; phase < 2; ++phase) {         // A = X X^T, then P = a I + b A + c A A
            const char* src = phase == 0 ? X : A;
            const int64_t pitch = phase == 0 ? px : pa;
            const int b = wave & (blocks - 1), part = wave >> 2 * lb, i = b >> lb, j = b & (mb - 1), kks = phase == 0 ? np / 16 : mp / 16;
            if (part < shares) {
                f32x16 acc, low, cross;                       // one chain of products each: a chain's next product waits for its last
                zero(acc);
                zero(low);
                zero(cross);
#pragma unroll 1
                for (int kk = part; kk < kks; kk += shares) {
                    const f16x8 ah = small_along(src, pitch, 32 * i + r, kk, h, 0), al = small_along(src, pitch, 32 * i + r, kk, h, 1);
                    const f16x8 bh = small_along(src, pitch, 32 * j + r, kk, h, 0), bl = small_along(src, pitch, 32 * j + r, kk, h, 1);
                    if (FULL) low = F::mfma(al, bl, low);
                    cross = F::mfma(ah, bl, cross);
                    acc = F::mfma(ah, bh, acc);
                    low = F::mfma(al, bh, low);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) scratch[(part * blocks + b) * 1024 + e * 64 + lane] = acc[e] + (low[e] + cross[e]);
            }
            __syncthreads();
            for (int g = threadIdx.x; g < mp * mp / 4; g += kSmallWaves * 64) {
                const int row = g >> (3 + lb), col = (g & (mp / 4 - 1)) * 4, q = row & 31;
                const float* at = scratch + (((row >> 5) << lb) + (col >> 5)) * 1024 + ((q >> 3) * 4 + (q & 3)) * 64 + (q >> 2 & 1) * 32 + (col & 31);
                f32x4 v = *reinterpret_cast<const f32x4*>(at);
                for (int k = 1; k < shares; ++k) v += *reinterpret_cast<const f32x4*>(at + k * blocks * 1024);
                const int64_t off = row * pa + (col >> 5) * 128 + (col & 31) * 2;
                _Float16 hi[4], lo[4];
                if (phase == 1) {
                    __builtin_memcpy(hi, A + off, 8);
                    __builtin_memcpy(lo, A + off + 64, 8);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float d = v[k] * down;
                    uint32_t q = phase == 1 ? poly_planes<FULL>(d, (float)hi[k] + (float)lo[k], row == col + k) : planes16(d, 0.f);
                    q = row < t.m && col + k < t.m ? q : 0u;
                    hi[k] = __builtin_bit_cast(_Float16, (uint16_t)q);
                    lo[k] = __builtin_bit_cast(_Float16, (uint16_t)(q >> 16));
                }
                char* d = (phase == 0 ? A : P) + off;
                __builtin_memcpy(d, hi, 8);
                __builtin_memcpy(d + 64, lo, 8);
            }
            __syncthreads();
        }
        const bool last = step + 1 == steps;
        f32x16 acc[kSmallPairs];                          // X = P X: block (i, blk) is pair wave + 16 n
#pragma unroll
        for (int n = 0; n < kSmallPairs; ++n) {
            const int pair = wave + kSmallWaves * n, i = pair & (mb - 1), blk = pair >> lb;
            if (pair >= pairs) break;
            zero(acc[n]);
#pragma unroll 1
            for (int kk = 0; kk < mp / 16; ++kk) {
                const f16x8 bh = small_across(X, px, lane, blk, kk, 0), bl = small_across(X, px, lane, blk, kk, 1);
                const f16x8 ah = small_along(P, pa, 32 * i + r, kk, h, 0), al = small_along(P, pa, 32 * i + r, kk, h, 1);
                if (FULL) acc[n] = F::mfma(al, bl, acc[n]);
                acc[n] = F::mfma(al, bh, acc[n]);
                acc[n] = F::mfma(ah, bl, acc[n]);
                acc[n] = F::mfma(ah, bh, acc[n]);
            }
            __builtin_amdgcn_sched_barrier(0);            // (one block's fragments at a time: registers)
        }
        __syncthreads();                                  // every wave has read what it needs of X
#pragma unroll
        for (int n = 0; n < kSmallPairs; ++n) {
            const int pair = wave + kSmallWaves * n, i = pair & (mb - 1), blk = pair >> lb;
            if (pair >= pairs) break;
            char* d = X + (32 * i + 4 * h) * px + blk * 128 + r * (last ? 4 : 2);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = acc[n][e] * down;
                char* q = d + (8 * (e >> 2) + (e & 3)) * px;
                if (last) {                               // in fp32: rows of as many bytes
                    *reinterpret_cast<float*>(q) = v * down;
                } else {
                    const _Float16 hi = (_Float16)v;
                    *reinterpret_cast<_Float16*>(q) = hi;
                    *reinterpret_cast<_Float16*>(q + 64) = (_Float16)(v - (float)hi);
                }
            }
        }
        __syncthreads();
    }
    float lr_step = 0.f, keep = 0.f;
    if constexpr (MUON) {
        const double lr = ap.rate();
        lr_step = (float)(lr * update_scale(t, ap.adjust));
        keep = (float)(1.0 - lr * ap.decay());
    }
    S* dst = reinterpret_cast<S*>(t.dst);
#pragma unroll 2
    for (int i = threadIdx.x * V; i < count; i += kSmallWaves * 64 * V) {
        const int left = count - i < V ? count - i : V;
        typename Vec<S>::type o = {};
        if constexpr (MUON) o = load_vec(dst + i, 0, left);
        int row = i / t.cols, col = i - row * t.cols;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j < left) {
                const float v = *reinterpret_cast<const float*>(X + (tall ? col * px + row * 4 : row * px + col * 4));
                if constexpr (MUON) o[j] = o[j] * keep - lr_step * v;
                else o[j] = (S)v;
            }
            if (++col == t.cols) { col = 0; ++row; }
        }
        store_vec(dst + i, 0, left, o);
    }
}

template <bool FULL, bool TB> using Big = MmTile<_Float16, 2, 256, 256, 2, 4, 2, false, TB, 1, FULL>;
template <bool FULL> using Tri = MmTile<_Float16, 2, 192, 192, 2, 2, 3, false, false, 1, FULL>;   // 253 of them cover a triangle of 4096, one per CU
template <bool FULL, bool TB, int KG = 1> using Mid = MmTile<_Float16, 2, 128, 128, 2, 2, 2, false, TB, KG, FULL>;
template <bool FULL, bool TB, int KG = 1> using Small = MmTile<_Float16, 2, 64, 64, 2, 2, 4, false, TB, KG, FULL>;

#define SSECG_NS_LAUNCH(M, kernel, grid, st, ...)                                                                               \
    do {                                                                                                                        \
        hipLaunchKernelGGL(kernel, dim3((unsigned)(grid)), dim3(M::NT), 0, st, __VA_ARGS__);                               \
        const int rc_ = (int)hipGetLastError();                                                                                 \
        if (rc_ != 0) return rc_;                                                                                               \
    } while (0)

struct Plan {
    size_t bytes;
    int parts, prep, gram, upd, gramTile, updTile, gramGroups, updGroups;   // workgroups of the launches, tile sides, groups of waves
};

template <bool POLY, bool FULL>
int launch_gram(const Table& t, const Plan& p, char* ws, int from, const float* skip, hipStream_t st) {
#define SSECG_NS_GRAM(...) do { using M = __VA_ARGS__; SSECG_NS_LAUNCH(M, (ns_gram_kernel<M, POLY>), p.gram, st, t, ws, from, skip); } while (0)
    if (p.gramTile == 256) SSECG_NS_GRAM(Big<FULL, false>);
    else if (p.gramTile == 192) SSECG_NS_GRAM(Tri<FULL>);
    else if (p.gramTile == 128) SSECG_NS_GRAM(Mid<FULL, false>);
    else if (p.gramGroups == 2) SSECG_NS_GRAM(Small<FULL, false, 2>);
    else SSECG_NS_GRAM(Small<FULL, false>);
#undef SSECG_NS_GRAM
    return 0;
}

template <typename S, int LAST, bool FULL>
int launch_update(const Table& t, const Plan& p, char* ws, int from, const Apply& ap, const float* skip, hipStream_t st) {
#define SSECG_NS_UPDATE(...) \
    do { using M = __VA_ARGS__; SSECG_NS_LAUNCH(M, (ns_update_kernel<M, S, LAST>), p.upd, st, t, ws, from, ap, skip); } while (0)
    if (p.updTile == 256) SSECG_NS_UPDATE(Big<FULL, true>);
    else if (p.updTile == 128 && p.updGroups == 2) SSECG_NS_UPDATE(Mid<FULL, true, 2>);
    else if (p.updTile == 128) SSECG_NS_UPDATE(Mid<FULL, true>);
    else SSECG_NS_UPDATE(Small<FULL, true>);
#undef SSECG_NS_UPDATE
    return 0;
}

// mats: host rows {source, result or parameter, momentum, rows, cols} of at most kMost matrices
int make_plan(const int64_t* mats, int count, Table& t, Plan& p) {
    // the tile side that mm_time expects to be fastest: the two products of a step over a triangle of tiles, the update over all
    int64_t largest = 0;
    auto time = [&](int side, int groups, bool gram) {
        MmWork along, square, whole;
        for (int k = 0; k < count; ++k) {
            const int64_t a = mats[5 * k + 3], b = mats[5 * k + 4], m = a < b ? a : b, n = a < b ? b : a;
            const int64_t tm = (m + side - 1) / side, tn = (n + side - 1) / side;
            along.add(tm * (tm + 1) / 2, (n + 31) / 32);
            square.add(tm * (tm + 1) / 2, (m + 31) / 32);
            whole.add(tm * tn, (m + 31) / 32);
            largest = a * b > largest ? a * b : largest;
        }
        return gram ? mm_time(side, 2, along, groups) + mm_time(side, 2, square, groups) : mm_time(side, 2, whole, groups);
    };
    auto pick = [&](bool gram, int& tile, int& groups, std::initializer_list<std::pair<int, int>> of) {
        double least = 0.0;
        for (const auto& c : of) {
            const double t = time(c.first, c.second, gram);
            if (least == 0.0 || t < least) { least = t; tile = c.first; groups = c.second; }
        }
    };
    pick(true, p.gramTile, p.gramGroups, {{64, 1}, {64, 2}, {128, 1}, {192, 1}, {256, 1}});
    pick(false, p.updTile, p.updGroups, {{64, 1}, {128, 1}, {128, 2}, {256, 1}});
    p.parts = (int)(largest / 8192 < 1 ? 1 : largest / 8192 > kNormParts ? kNormParts : largest / 8192);
    t.count = count;
    int64_t at = up((int64_t)kMost * kNormParts * 8, 256), prep = 0, gram = 0, upd = 0;
    for (int k = 0; k < kMost; ++k) {
        const int64_t a = k < count ? mats[5 * k + 3] : 0, b = k < count ? mats[5 * k + 4] : 0, m = a < b ? a : b, n = a < b ? b : a;
        t.src[k] = k < count ? (const void*)mats[5 * k] : nullptr;
        t.dst[k] = k < count ? (void*)mats[5 * k + 1] : nullptr;
        t.mom[k] = k < count ? (float*)mats[5 * k + 2] : nullptr;
        t.rows[k] = (int)a;
        t.cols[k] = (int)b;
        t.offset[k] = at;
        t.first[wPrep][k] = (int)prep;
        t.first[wGram][k] = (int)gram;
        t.first[wUpd][k] = (int)upd;
        if (k >= count) continue;
        const int64_t tg = (m + p.gramTile - 1) / p.gramTile;
        at += mat_bytes(a, b);
        prep += ((up(a, 32) + 63) / 64) * ((up(b, 32) + 63) / 64);
        gram += tg * (tg + 1) / 2;
        upd += ((m + p.updTile - 1) / p.updTile) * ((n + p.updTile - 1) / p.updTile);
        if (prep >= INT32_MAX || gram >= INT32_MAX || upd >= INT32_MAX) return SSECG_E_INVAL;
    }
    p.bytes = (size_t)at;
    p.prep = (int)prep;
    p.gram = (int)gram;
    p.upd = (int)upd;
    return 0;
}

template <typename S, bool MUON>
int run_chain(const int64_t* mats, int count, int nesterov, int steps, double eps, const Apply& ap, const float* skip, char* ws,
              hipStream_t st) {
    Table t;
    Plan p;
    int rc = make_plan(mats, count, t, p);
    if (rc != 0) return rc;
    bool small = true;
    for (int k = 0; k < count; ++k) small = small && small_ok(mats[5 * k + 3], mats[5 * k + 4]);
    if (small) {
        hipLaunchKernelGGL((ns_small_kernel<S, MUON>), dim3(count), dim3(kSmallWaves * 64), 0, st, t, nesterov, steps, eps, ap, skip);
        return (int)hipGetLastError();
    }
    double* partial = reinterpret_cast<double*>(ws);
    hipLaunchKernelGGL((ns_norm_kernel<S, MUON>), dim3(p.parts, count), dim3(256), 0, st, t, ap, nesterov, skip, partial);
    hipLaunchKernelGGL((ns_prep_kernel<S, MUON>), dim3((unsigned)p.prep), dim3(256), 0, st, t, ws, ap, nesterov, p.parts, eps, skip, partial);
    rc = (int)hipGetLastError();
    for (int k = 0; k < steps && rc == 0; ++k) {
        constexpr bool FULL = kFull<S, MUON>;
        if ((rc = launch_gram<false, FULL>(t, p, ws, k & 1, skip, st)) != 0) break;
        if ((rc = launch_gram<true, FULL>(t, p, ws, k & 1, skip, st)) != 0) break;
        if (k + 1 < steps) rc = launch_update<S, 0, FULL>(t, p, ws, k & 1, ap, skip, st);
        else rc = launch_update<S, MUON ? 2 : 1, FULL>(t, p, ws, k & 1, ap, skip, st);
    }
    return rc;
}

constexpr int64_t kMaxSide = 1 << 20;

bool mats_ok(const int64_t* mats, int count, bool pointers, bool muon) {
    if (!mats || count <= 0) return false;
    for (int k = 0; k < count; ++k) {
        const int64_t* r = mats + 5 * (size_t)k;
        if (r[3] <= 0 || r[4] <= 0 || r[3] > kMaxSide || r[4] > kMaxSide) return false;
        if (pointers && (!r[0] || !r[1] || (muon && !r[2]))) return false;
    }
    return true;
}

}  // namespace

extern "C" {

size_t ssecg_orthogonalize_workspace(const int64_t* mats, int count) {
    if (!mats_ok(mats, count, false, false)) return 0;
    size_t most = 0;
    for (int k = 0; k < count; k += kMost) {
        Table t;
        Plan p;
        if (make_plan(mats + 5 * (size_t)k, count - k < kMost ? count - k : kMost, t, p) != 0) return 0;
        most = p.bytes > most ? p.bytes : most;
    }
    return most;
}

int ssecg_orthogonalize_multi(const int64_t* mats, int count, int dtype, int steps, double eps, void* workspace, size_t workspace_bytes,
                              void* stream) {
    if (!mats_ok(mats, count, true, false) || !dtype_ok(dtype) || steps < 1 || steps > 100 || !(eps >= 0.0) || !workspace ||
        ((uintptr_t)workspace & 255))
        return SSECG_E_INVAL;
    if (workspace_bytes < ssecg_orthogonalize_workspace(mats, count)) return SSECG_E_WORKSPACE;
    const Apply ap = {};
    for (int k = 0; k < count; k += kMost) {
        int rc = 0;
        SSECG_LM_DTYPE(dtype, S, rc = (run_chain<S, false>(mats + 5 * (size_t)k, count - k < kMost ? count - k : kMost, 0, steps, eps, ap, nullptr,
                                                          (char*)workspace, (hipStream_t)stream)));
        if (rc != 0) return rc;
    }
    return 0;
}

static int muon_multi(const int64_t* mats, int count, const Apply& ap, int nesterov, int steps, double eps, const float* skip_flag, void* workspace,
                      size_t workspace_bytes, void* stream) {
    if (!mats_ok(mats, count, true, true) || steps < 1 || steps > 100 || !(eps >= 0.0) || ap.adjust < 0 || ap.adjust > 1 || !workspace ||
        ((uintptr_t)workspace & 255))
        return SSECG_E_INVAL;
    if (workspace_bytes < ssecg_orthogonalize_workspace(mats, count)) return SSECG_E_WORKSPACE;
    for (int k = 0; k < count; k += kMost) {
        const int rc = run_chain<float, true>(mats + 5 * (size_t)k, count - k < kMost ? count - k : kMost, nesterov != 0, steps, eps, ap, skip_flag,
                                              (char*)workspace, (hipStream_t)stream);
        if (rc != 0) return rc;
    }
    return 0;
}

int ssecg_muon_multi(const int64_t* mats, int count, double lr, double momentum, int nesterov, double weight_decay, int adjust, int steps, double eps,
                     const float* skip_flag, const double* lr_dev, void* workspace, size_t workspace_bytes, void* stream) {
    if (!(momentum >= 0.0 && momentum < 1.0)) return SSECG_E_INVAL;
    return muon_multi(mats, count, {lr, weight_decay, adjust, (float)momentum, lr_dev, nullptr}, nesterov, steps, eps, skip_flag, workspace,
                      workspace_bytes, stream);
}

int ssecg_muon_multi_scalars(const int64_t* mats, int count, const double* scalars_dev, int nesterov, int adjust, int steps, double eps,
                             const float* skip_flag, void* workspace, size_t workspace_bytes, void* stream) {
    if (!scalars_dev) return SSECG_E_INVAL;
    return muon_multi(mats, count, {0.0, 0.0, adjust, 0.f, nullptr, scalars_dev}, nesterov, steps, eps, skip_flag, workspace, workspace_bytes,
                      stream);
}

}  // extern "C"
