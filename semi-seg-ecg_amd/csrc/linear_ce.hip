// A classifier and its softmax cross entropy over a large vocabulary, in pieces of the vocabulary, without keeping the logits:
//
//   z_nv = x_n . w_v (+ b_v),  lse_n = log sum_v exp z_nv,  row loss = g_n (lse_n - z_{n,t_n})
//   E_nv = g_n (exp(z_nv - lse_n) - [v = t_n]),  dx_n = f sum_v E_nv w_v,  dw_v = f sum_n E_nv x_n,  db_v = f sum_n E_nv
//
// g_n is 0 for an ignored position and for one whose confidence is below the threshold, else 1 (times the upstream gradient when
// the loss is not reduced); f = upstream / number of positions that are not ignored (mean), upstream (sum).
//
// Forward: one product whose epilogue keeps, per tile, the maximum and the sum of exponentials of a row and its target's logit.
// The vocabulary is the tile's register axis (operand A), so a lane reduces its own row without shuffles but one.  A second launch
// joins the tiles.  Backward: the logits of a piece are computed again, E is written in 16 bits and two products take it up, one
// along its rows, one across (mm_core.h reads an operand either way, so no operand is transposed in memory).  8 N V C
// multiplications and additions against the 6 N V C that keeping N V logits would need.
//
// 32-bit operands, and E between them, travel as three bf16 planes (mm_core.h): exact at every element's own exponent, so a row beside
// one 10^30 times larger, a class of probability 10^-30 and a position of a tiny upstream gradient are as precise as in a 32-bit
// product.  (Two fp16 planes and one scale per tensor took half the time, 231 us against 421 at 2000 x 512 x 8192, and lost them.)
//
// Roundings to fewer bits: for 16-bit operands E is held in their type, so that its products run at one 16-bit product's rate like those
// of x and w; more planes would write twice the bytes and triple dx's and dw's time.  The gradients' relative error against 64 bits is
// 1.7e-3 to 2.2e-3 in bf16 (1.7e-3 of it their own rounding at the end), 2.1e-4 to 2.8e-4 in fp16.  fp16 has no values below
// 2^-24: E, in [-1, 1], is held times 2^15, has fewer bits below 2^-29 and is zero below 2^-40 (of the largest |upstream gradient| where the
// loss is not reduced) - as f E x itself is in fp16 at a loss scale of 2^16.  Rows whose g_n is zero enter nothing: neither their values
// (which may be infinite or NaN) nor their products.
//
// Many positions are bound by the products' main loop, which keeps the matrix pipe busy 48 to 61 % of the cycles: 8192 x 1024 x 65536 bf16
// takes 1.13 ms forward (0.97 PFLOP/s) and 3.4 ms backward: E 1.42 ms, of which 0.3 for its 1 GiB and its exponentials, dx 0.95 (1.15
// PFLOP/s), dw 1.03.  fp32 is six such products each: 2000 x 512 x 8192 takes 93, 115, 135 and 144 us for the four (0.7 to 1.1 PFLOP/s).  Few
// positions are bound by the weights, read three times and written once: 8 x 1024 x 32768 fp16 takes 77 us, each pass over them 13
// to 20 us (4.7 to 3.4 TB/s).  The smallest calls are bound by their launches: 126 x 512 x 1000 fp32, 7 of them, 59 us.
#include <type_traits>
#include "mm_core.h"
#include "ssecg.h"

namespace {
using namespace ssecg_lm;

constexpr float kLog2e = 1.4426950408889634f;
// E is held times 2^15 where its type has few exponents
template <typename T> constexpr int kEScale = std::is_same<T, _Float16>::value ? 15 : 0;

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// ---------------------------------------------------------------- operands
struct Counts {                                   // which rows count: by the gate of the forward pass, by target and confidence, or all
    const float* gate;
    const int64_t* target; int64_t ignore;
    const float* conf; float thresh;
    __device__ __forceinline__ bool operator()(int64_t r) const {
        if (gate) return gate[r] != 0.f;
        return target == nullptr || (target[r] != ignore && (conf == nullptr || conf[r] >= thresh));
    }
};

// src (R, C) as an operand: its planes, zeros up to the pitch, and zeros for a row that does not count.  One thread: 8 values; one
// launch for all of a pass (blockIdx.y).
struct PackJob { const void* src; int64_t R; Counts counts; char* dst; };
struct PackJobs { PackJob job[2]; };
template <typename S, int P>
__global__ __launch_bounds__(256) void ce_pack_kernel(PackJobs jobs, int C, int64_t pitch) {
    const PackJob& job = jobs.job[blockIdx.y];
    const S* __restrict__ src = reinterpret_cast<const S*>(job.src);
    char* __restrict__ dst = job.dst;
    const Counts counts = job.counts;
    const int64_t R = job.R;
    const int per = (int)(pitch / 16);                     // threads of a row
    const int64_t plane = R * pitch;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < R * per; at += (int64_t)gridDim.x * 256) {
        const int64_t r = at / per;
        const int k = (int)(at - r * per) * 8;
        const bool live = counts(r);
        uint16_t q[8][P];
        constexpr int V = Vec<S>::N;
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            typename Vec<S>::type t = {};
            if (live && k + i < C) t = load_vec(src + r * C, k + i, C);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (P == 3) split3(t[j], q[i + j]);
                else q[i + j][0] = bits16(t[j]);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            u32x4 d;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = (unsigned)q[2 * j][p] | (unsigned)q[2 * j + 1][p] << 16;
            *reinterpret_cast<u32x4*>(dst + p * plane + r * pitch + k * 2) = d;
        }
    }
}

// f: upstream / count (mean), upstream (sum), or the power of two that ce_coef_kernel chose
struct Factor {
    const float* up; const float* count;
    __device__ __forceinline__ float operator()() const { return count ? up[0] / count[0] : up[0]; }
};

// ---------------------------------------------------------------- logits
struct LogitArgs {
    Operand W, X;                                // vocabulary rows (of the piece), position rows
    const float* bias;                           // of the piece, or null
    int V, N, tilesV, tilesN, stages;
    const int64_t* target;                       // class indices; v0 is the piece's first class
    int64_t v0;
    // forward: partial maxima and sums [parts][N], target logits [N]
    float* pm; float* ps; float* tl;
    // gradient: lse and g per row, E [rowsE][pitchE] (rows from N on are zeros), partial db [tilesN][V]
    const float* lse; const float* gate; const float* coef;
    char* E; int64_t pitchE, planeE;
    int rowsE;
    float* pdb;
    float* db; Factor f;                         // db itself where one tile holds all positions, times f
};

template <class M>
__device__ __forceinline__ void tile_of(int tilesA, int tilesB, int& ta, int& tb) {
    // operand A's tiles fastest within groups of 4 tiles of B: a group's rows of B stay in the L2 while A passes
    const int t = xcd_tile(blockIdx.x, tilesA * tilesB);
    const int grp = 4 * tilesA, g = t / grp, in = t - g * grp;
    const int width = tilesB - 4 * g < 4 ? tilesB - 4 * g : 4;
    ta = in / width;
    tb = 4 * g + in - ta * width;
}

template <class M>
__device__ __forceinline__ bool logits_tile(const LogitArgs& p, int a0, int b0, char* lds, f32x16 (&acc)[M::TM][M::TN]) {
    if (!M::run(p.W, a0, p.X, b0, 0, p.stages, lds, acc)) return false;
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < M::TM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int v = a0 + M::arow(i, e);
                const float b = p.bias[v < p.V ? v : p.V - 1];
#pragma unroll
                for (int j = 0; j < M::TN; ++j) acc[i][j][e] += b;
            }
            __builtin_amdgcn_sched_barrier(0);    // 16 loads at a time: all of them at once would spill the accumulators
        }
    }
    if (a0 + M::BM > p.V) {                       // the last tile: classes that do not exist
#pragma unroll
        for (int i = 0; i < M::TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool out = a0 + M::arow(i, e) >= p.V;
#pragma unroll
                for (int j = 0; j < M::TN; ++j) acc[i][j][e] = out ? -INFINITY : acc[i][j][e];
            }
    }
    __builtin_amdgcn_sched_barrier(0);
    return true;
}

// the label of a position as an offset from the lane's first class: register (i, e) holds it where offset == 32 i + 8 (e / 4) + e % 4
template <class M>
__device__ __forceinline__ int label_offset(int64_t t, int a0) {
    const int64_t off = t - a0 - M::arow(0, 0);
    return off >= 0 && off < 32 * M::TM ? (int)off : -1;
}
__device__ __forceinline__ constexpr int reg_offset(int i, int e) { return 32 * i + 8 * (e >> 2) + (e & 3); }

// (m, s): a maximum and the sum of exp(z - m), joined with another's.  Each is weighted by exp(m - max): 0 for a side without a finite
// logit (m = -inf, s = 0), whatever the other side's maximum is.  A NaN sum stays one.
__device__ __forceinline__ void join_lse(float& m, float& s, float m2, float s2) {
    const float mt = fmaxf(m, m2), mz = mt == -INFINITY ? 0.f : mt;
    s = s * exp2_fast((m - mz) * kLog2e) + s2 * exp2_fast((m2 - mz) * kLog2e);
    m = mt;
}

template <class M>
__global__ __launch_bounds__(M::NT, 2) void ce_lse_kernel(LogitArgs p) {
    __shared__ __attribute__((aligned(16))) char lds[M::LDS];
    int ta, tb;
    tile_of<M>(p.tilesV, p.tilesN, ta, tb);
    const int a0 = ta * M::BM, b0 = tb * M::BN;
    f32x16 acc[M::TM][M::TN];
    if (!logits_tile<M>(p, a0, b0, lds, acc)) return;
    const int wm = (threadIdx.x >> 6) / M::WN, h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int j = 0; j < M::TN; ++j) {
        const int n = b0 + M::bcol(j);
        const int off = n < p.N ? label_offset<M>(p.target[n], a0) : -1;
        float m = -INFINITY, hit = 0.f;
#pragma unroll
        for (int i = 0; i < M::TM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                m = fmaxf(m, acc[i][j][e]);
                hit = reg_offset(i, e) == off ? acc[i][j][e] : hit;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const float mm = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < M::TM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s += exp2_fast((acc[i][j][e] - mm) * kLog2e);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (off >= 0 && (off & 4) == 0 && a0 + M::arow(0, 0) + off < p.V) p.tl[n] = hit;
        // the lane's other half of the rows
        const float m2 = __shfl_xor(m, 32, 64), s2 = __shfl_xor(s, 32, 64);
        join_lse(m, s, m2, s2);
        if (h == 0 && n < p.N) {
            const int64_t part = (int64_t)ta * M::WM + wm;
            p.pm[part * p.N + n] = m;
            p.ps[part * p.N + n] = s;
        }
    }
}

struct Joined { float *lse, *gate, *row, *loss, *count; };
// loss (mean / sum; null: not reduced) and count from the sums of a workgroup of 1024; fixed order, fp64
__device__ __forceinline__ void ce_total(double s, int k, int mean, const Joined& out) {
    __shared__ double sh[16];
    __shared__ int shc[16];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); k += __shfl_xor(k, o, 64); }
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = s; shc[threadIdx.x >> 6] = k; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) { s += sh[w]; k += shc[w]; }
        const int c = k > 0 ? k : 1;
        out.count[0] = (float)c;
        if (out.loss) out.loss[0] = (float)(mean ? s / (double)c : s);
    }
}

// joins the parts of a row: lse, g and the row's loss.  A workgroup: ROWS rows, 1024 / ROWS strands of parts each.  WHOLE: it has all
// rows, and the total as well.
template <int ROWS, bool WHOLE>
__global__ __launch_bounds__(1024) void ce_join_kernel(const float* __restrict__ pm, const float* __restrict__ ps, const float* __restrict__ tl,
                                                       int parts, int N, int V, const int64_t* __restrict__ target, Counts counts, int mean,
                                                       Joined out) {
    constexpr int K = 1024 / ROWS, SPAN = ROWS < 64 ? 64 : ROWS, S = 1024 / SPAN;   // strands; threads whose strands meet in one wave
    __shared__ float sm[S][ROWS + 1], ss[S][ROWS + 1];
    const int c = threadIdx.x % ROWS, k = threadIdx.x / ROWS, n = blockIdx.x * ROWS + c;
    float m = -INFINITY, s = 0.f;
    if (n < N)
        for (int p = k; p < parts; p += 4 * K) {          // 4 loads in flight
            float m2[4], s2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = p + j * K < parts;
                m2[j] = in ? pm[(int64_t)(p + j * K) * N + n] : -INFINITY;
                s2[j] = in ? ps[(int64_t)(p + j * K) * N + n] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) join_lse(m, s, m2[j], s2[j]);
        }
#pragma unroll
    for (int o = ROWS; o < 64; o *= 2) {                  // the wave's strands
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        join_lse(m, s, m2, s2);
    }
    if (threadIdx.x % SPAN < ROWS) { sm[threadIdx.x / SPAN][c] = m; ss[threadIdx.x / SPAN][c] = s; }
    __syncthreads();
    double loss = 0.0;
    int kept = 0;
    if (k == 0 && n < N) {
        for (int q = 1; q < S; ++q) join_lse(m, s, sm[q][c], ss[q][c]);
        const int64_t t = target[n];
        const bool bad = t != counts.ignore && (t < 0 || t >= V);
        const float l = bad || m == -INFINITY ? NAN : m + logf(s);     // a label outside the vocabulary poisons its row: no silent loss
        const float g = counts(n) ? 1.f : 0.f, row = g != 0.f ? l - (bad ? 0.f : tl[n]) : 0.f;
        out.lse[n] = l;
        out.gate[n] = g;
        out.row[n] = row;
        loss = (double)row;
        kept = t != counts.ignore ? 1 : 0;
    }
    if (WHOLE) ce_total(loss, kept, mean, out);
}

__global__ __launch_bounds__(1024) void ce_total_kernel(const int64_t* __restrict__ target, int64_t ignore, int N, int mean, Joined out) {
    double s = 0.0;
    int k = 0;
    for (int i = threadIdx.x; i < N; i += 1024) {
        s += (double)out.row[i];
        k += target[i] != ignore ? 1 : 0;
    }
    ce_total(s, k, mean, out);
}

// ---------------------------------------------------------------- gradient
// Not reduced: coef[n] = g_n dloss[n] / s with s a power of two >= max |g dloss| (so that E stays in [-1, 1]); fscale[0] = s.
__global__ __launch_bounds__(1024) void ce_coef_kernel(const float* __restrict__ dloss, const float* __restrict__ gate, int N,
                                                       float* __restrict__ coef, float* __restrict__ fscale) {
    __shared__ float sh[16];
    float m = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        const float v = gate[i] != 0.f ? fabsf(dloss[i]) : 0.f;
        if (v < INFINITY) m = fmaxf(m, v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
    __syncthreads();
    m = sh[0];
    for (int k = 1; k < 16; ++k) m = fmaxf(m, sh[k]);
    int e = 0;
    if (m > 0.f) frexpf(m, &e);                        // m <= 2^e
    e = e > 127 ? 127 : (e < -126 ? -126 : e);
    for (int i = threadIdx.x; i < N; i += 1024) coef[i] = gate[i] != 0.f ? ldexpf(dloss[i], -e) : 0.f;
    if (threadIdx.x == 0) fscale[0] = ldexpf(1.f, e);
}

template <class M, bool DB>
__global__ __launch_bounds__(M::NT, 2) void ce_grad_kernel(LogitArgs p) {
    __shared__ __attribute__((aligned(16))) char lds[M::LDS];
    int ta, tb;
    tile_of<M>(p.tilesV, p.tilesN, ta, tb);
    const int a0 = ta * M::BM, b0 = tb * M::BN;
    using T = typename M::T;
    f32x16 acc[M::TM][M::TN];
    if (!logits_tile<M>(p, a0, b0, lds, acc)) return;
    const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % M::WN;
    float lse[M::TN], g[M::TN];
    int off[M::TN];
#pragma unroll
    for (int j = 0; j < M::TN; ++j) {
        const int n = b0 + M::bcol(j);
        const bool in = n < p.N;
        g[j] = in ? p.gate[n] : 0.f;
        if (in && p.coef) g[j] = p.coef[n];
        lse[j] = in ? p.lse[n] : 0.f;
        off[j] = in ? label_offset<M>(p.target[n] - p.v0, a0) : -1;
    }
    float* part = reinterpret_cast<float*>(lds);          // DB: column sums [WN][BM] of the waves
#pragma unroll
    for (int i = 0; i < M::TM; ++i) {
        float sums[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < M::TN; ++j) {
                const float pr = exp2_fast((acc[i][j][e] - lse[j]) * kLog2e) - (reg_offset(i, e) == off[j] ? 1.f : 0.f);
                const float q = g[j] != 0.f ? pr * g[j] : 0.f;      // a row that does not count enters as zero, whatever it holds
                acc[i][j][e] = q * (float)(1 << kEScale<T>);
                sum += q;
            }
            sums[e] = sum;
        }
        if (DB) {
            // column sums over the wave's 32 positions: at each exchange a lane keeps half of its sums and hands the others over (16
            // exchanges; 80 for one sum after the other).  Lane l ends with register (l / 2) % 16.
#pragma unroll
            for (int half = 8; half > 0; half >>= 1) {
                const bool upper = (lane & 2 * half) != 0;
#pragma unroll
                for (int k = 0; k < half; ++k) {
                    const float give = upper ? sums[k] : sums[k + half], keep = upper ? sums[k + half] : sums[k];
                    sums[k] = keep + __shfl_xor(give, 2 * half, 64);
                }
            }
            sums[0] += __shfl_xor(sums[0], 1, 64);
            if ((lane & 1) == 0) part[wn * M::BM + M::arow(i, (lane >> 1) & 15)] = sums[0];
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (DB) {
        __syncthreads();
        for (int r = threadIdx.x; r < M::BM; r += M::NW * 64) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < M::WN; ++k) sum += part[k * M::BM + r];
            if (a0 + r < p.V) {
                if (p.db) p.db[a0 + r] = sum * p.f();
                else p.pdb[(int64_t)tb * p.V + a0 + r] = sum;
            }
        }
        __syncthreads();
    }
    if (p.E == nullptr) return;
    using W = WaveStore<M>;
    char* reg = W::region(lds);
    const int v0 = a0 + M::wave_row(), n0 = b0 + M::wave_col();
    auto val = [&](int i, int j, int e, int q) -> uint16_t {
        if constexpr (M::P == 3) {
            uint16_t b[3];
            split3(acc[i][j][e], b);
            return b[q];
        } else {
            return bits16((T)acc[i][j][e]);
        }
    };
    // the pitch covers the whole tile: no condition on the class
    W::template store_cols<M::P>(reg, val, [&](int n, int v, int q, u32x4 d) {
        if (n0 + n < p.rowsE) *reinterpret_cast<u32x4*>(p.E + q * p.planeE + (n0 + n) * p.pitchE + (v0 + v) * 2) = d;
    });
}

// ---------------------------------------------------------------- products with E
struct ProdArgs {
    Operand A, B;
    int rows, cols, tilesA, tilesB, stages, splits;
    float* plane;                                // partial planes [splits][rows][cols], or null: write out
    int add;                                     // plane += instead of plane =
    void* out;                                   // (rows, cols) of the result's type
    Factor f;
};

template <typename O>
__device__ __forceinline__ O finish(float v, float f) { return (O)(v * f * (1.f / (float)(1 << kEScale<O>))); }

template <class M, typename O>
__global__ __launch_bounds__(M::NT, 2) void ce_prod_kernel(ProdArgs p) {
    __shared__ __attribute__((aligned(16))) char lds[M::LDS];
    int ta, tb;
    tile_of<M>(p.tilesA, p.tilesB, ta, tb);
    const int a0 = ta * M::BM, b0 = tb * M::BN;
    const int z = blockIdx.y, s0 = (int)((int64_t)p.stages * z / p.splits), s1 = (int)((int64_t)p.stages * (z + 1) / p.splits);
    f32x16 acc[M::TM][M::TN];
    if (!M::run(p.A, a0, p.B, b0, s0, s1 - s0, lds, acc)) return;
    const float f = p.plane ? 0.f : p.f();
    float* plane = p.plane ? p.plane + (int64_t)z * p.rows * p.cols : nullptr;
    if constexpr (sizeof(O) == 2) {
        if (!plane) {
            using W = WaveStore<M>;
            const int r0 = a0 + M::wave_row(), c0 = b0 + M::wave_col();
            W::template store_rows<1>(W::region(lds), [&](int i, int j, int e, int) -> uint16_t { return bits16(finish<O>(acc[i][j][e], f)); },
                          [&](int r, int c, int, u32x4 d) {
                              if (r0 + r < p.rows && c0 + c < p.cols)
                                  store_vec(reinterpret_cast<O*>(p.out) + (int64_t)(r0 + r) * p.cols, c0 + c, p.cols,
                                            __builtin_bit_cast(typename Vec<O>::type, d));
                          });
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < M::TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t r = a0 + M::arow(i, e);
            if (r >= p.rows) continue;
#pragma unroll
            for (int j = 0; j < M::TN; ++j) {
                const int c = b0 + M::bcol(j);
                if (c >= p.cols) continue;
                const int64_t at = r * p.cols + c;
                if (plane) plane[at] = p.add ? plane[at] + acc[i][j][e] : acc[i][j][e];
                else reinterpret_cast<O*>(p.out)[at] = finish<O>(acc[i][j][e], f);
            }
        }
}

// out = f (E's scale) sum of the planes, in their order; one launch for the results of a piece (blockIdx.y): dx and dweight of type O, dbias
// in fp32 (its planes are the tiles' column sums)
struct SumJob { const float* planes; int splits; int64_t n; int scaled; void* out; };   // scaled: O, from E
struct SumJobs { SumJob job[3]; };
template <typename O>
__global__ __launch_bounds__(256) void ce_sum_kernel(SumJobs jobs, Factor factor) {
    const SumJob& job = jobs.job[blockIdx.y];
    const float f = factor();
    const float* __restrict__ planes = job.planes;
    const int64_t n = job.n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        int k = 0;
        for (; k + 8 <= job.splits; k += 8) {             // 8 loads in flight
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = planes[(int64_t)(k + j) * n + i];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; k < job.splits; ++k) s += planes[(int64_t)k * n + i];
        if (job.scaled) reinterpret_cast<O*>(job.out)[i] = finish<O>(s, f);
        else reinterpret_cast<float*>(job.out)[i] = s * f;
    }
}

// ---------------------------------------------------------------- host side
template <typename S> struct Inner { using T = S; static constexpr int P = 1; };
template <> struct Inner<float> { using T = __bf16; static constexpr int P = 3; };
inline int planes_of(int dtype) { return dtype == kF32 ? 3 : 1; }

template <typename T, int P, bool TA = false, bool TB = false> using Big = MmTile<T, P, 256, 256, 2, 4, 2, TA, TB>;
template <typename T, int P, bool TA = false, bool TB = false, int KG = 1> using Mid = MmTile<T, P, 128, 128, 2, 2, 2, TA, TB, KG>;
template <typename T, int P, bool TA = false, bool TB = false, int KG = 1> using Small = MmTile<T, P, 64, 64, 2, 2, 4, TA, TB, KG>;

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// stages of a product over k
inline int64_t stages_of(int64_t k, int planes) { return up(k, 64) / 64 * (planes == 3 ? kTerms : 1); }

struct Blob {                                    // carves a workspace; a first pass with base 0 sizes it
    char* base; size_t at = 0;
    explicit Blob(void* p) : base((char*)p) {}
    template <typename T> T* take(size_t n) {
        char* q = base + at;
        at += (n * sizeof(T) + 255) & ~(size_t)255;
        return (T*)q;
    }
};

constexpr int64_t kMaxN = 1 << 21, kMaxV = 1 << 24, kMaxC = 1 << 16;
constexpr int64_t kMaxPiece = 1 << 21;           // classes of a piece
static_assert(kMaxC * 2 <= kMaxPitch && kMaxPiece * 2 <= kMaxPitch, "rows of every operand");
constexpr int64_t kMaxTiles = 1 << 22;           // of a launch: its 512 kMaxTiles threads stay below 2^32
inline int64_t tiles_of(int64_t n, int side) { return (n + side - 1) / side; }
inline bool shape_ok(int64_t N, int64_t C, int64_t V) {
    return N > 0 && C > 0 && V > 0 && N <= kMaxN && V <= kMaxV && C <= kMaxC && tiles_of(N, 256) * tiles_of(V, 256) <= kMaxTiles;
}

// Is the matrix an operand as it lies (16-bit, whole stages of k, aligned)?
inline bool direct(int dtype, const void* p, int64_t C) { return dtype != kF32 && C % 64 == 0 && ((uintptr_t)p & 15) == 0; }

// What forward leaves for backward beside the statistics: the operands that had to be copied (three planes, or k padded to a stage).
struct Packed {
    char *Xp, *Wp;                               // null where the tensor is an operand as it lies
    int64_t pitch;
    size_t bytes;
};

Packed plan_packed(void* base, const void* x, const void* w, int dtype, int64_t N, int64_t C, int64_t V) {
    Blob b(base);
    Packed p = {};
    const int P = planes_of(dtype);
    p.pitch = up(C, 64) * 2;
    if (!direct(dtype, x, C)) p.Xp = b.take<char>((size_t)(N * p.pitch * P));
    if (!direct(dtype, w, C)) p.Wp = b.take<char>((size_t)(V * p.pitch * P));
    p.bytes = b.at;
    return p;
}

// the tile side (256, 128, 64) of a product of a x b results with `stages` stages, and how many workgroups and how many groups of a
// workgroup's waves share the k of a tile
struct Choice { int side, splits, groups; };
inline Choice choose(int64_t a, int64_t b, int64_t stages, bool split) {
    Choice best = {256, 1, 1};
    double least = 0.0;
    for (int side = 256; side >= 64 && tiles_of(a, side) * tiles_of(b, side) <= kMaxTiles; side /= 2)
        for (int s = 1; s <= (split ? 64 : 1) && (s == 1 || stages / s >= 4); s += s < 8 ? 1 : s < 16 ? 2 : 8) {
            MmWork w;
            w.add(tiles_of(a, side) * tiles_of(b, side) * s, (stages + s - 1) / s);
            for (int g = 1; g <= (side < 256 ? 2 : 1); ++g) {
                // the planes of the parts are written and read again (4 TB/s), and a launch sums them
                const double t = mm_time(side, 1, w, g) + (s > 1 ? 4.0 + (double)a * b * s * 8 / 4e6 : 0.0);
                if (least == 0.0 || t < least) {
                    least = t;
                    best = {side, s, g};
                }
            }
        }
    return best;
}

struct FwdPlan {
    Choice c;
    int tilesV, tilesN, parts;
    float *pm, *ps, *tl, *row;
};

FwdPlan plan_fwd(Blob& ws, int dtype, int64_t N, int64_t C, int64_t V) {
    FwdPlan p;
    p.c = choose(V, N, stages_of(C, planes_of(dtype)), false);
    p.tilesV = (int)tiles_of(V, p.c.side);
    p.tilesN = (int)tiles_of(N, p.c.side);
    p.parts = p.tilesV * 2;                      // two waves of a tile along the classes
    p.pm = ws.take<float>((size_t)p.parts * N);
    p.ps = ws.take<float>((size_t)p.parts * N);
    p.tl = ws.take<float>((size_t)N);
    p.row = ws.take<float>((size_t)N);
    return p;
}

inline unsigned grid_for(int64_t n) {
    const int64_t b = (n + 255) / 256;
    return (unsigned)(b < 2048 ? b : 2048);
}

template <typename S>
int pack(const PackJobs& jobs, int count, int64_t C, int64_t pitch, hipStream_t st) {
    constexpr int P = Inner<S>::P;
    int64_t rows = jobs.job[0].R;
    if (count == 2 && jobs.job[1].R > rows) rows = jobs.job[1].R;
    hipLaunchKernelGGL((ce_pack_kernel<S, P>), dim3(grid_for(rows * (pitch / 16)), count), dim3(256), 0, st, jobs, (int)C,
                       pitch);
    return (int)hipGetLastError();
}

#define SSECG_CE_LAUNCH(M, kernel, grid, st, args)                                                                              \
    do {                                                                                                                        \
        hipLaunchKernelGGL(kernel, grid, dim3(M::NT), 0, st, args);                                                        \
        const int rc_ = (int)hipGetLastError();                                                                                 \
        if (rc_ != 0) return rc_;                                                                                               \
    } while (0)

// the tile of a choice
#define SSECG_CE_TILES(c, WITH, TA, TB)                                                \
    do {                                                                               \
        if ((c).side == 256) WITH(Big<T, P, TA, TB>);                                  \
        else if ((c).side == 128 && (c).groups == 2) WITH(Mid<T, P, TA, TB, 2>);       \
        else if ((c).side == 128) WITH(Mid<T, P, TA, TB>);                             \
        else if ((c).groups == 2) WITH(Small<T, P, TA, TB, 2>);                        \
        else WITH(Small<T, P, TA, TB>);                                                \
    } while (0)

template <typename S>
int ce_fwd(const void* x, const void* w, const float* bias, const int64_t* target, const float* conf, float thresh, int64_t ignore, int dtype,
           int64_t N, int64_t C, int64_t V, int reduction, float* loss, float* lse, float* gate, float* count, void* packed, void* ws,
           hipStream_t st) {
    using T = typename Inner<S>::T;
    constexpr int P = Inner<S>::P;
    Blob blob(ws);
    const Packed k = plan_packed(packed, x, w, dtype, N, C, V);
    const FwdPlan p = plan_fwd(blob, dtype, N, C, V);
    const Counts counts = {nullptr, target, ignore, conf, thresh};
    LogitArgs a = {};
    int rc = 0;
    PackJobs jobs = {};
    int copies = 0;
    if (k.Xp) jobs.job[copies++] = {x, N, counts, k.Xp};
    if (k.Wp) jobs.job[copies++] = {w, V, Counts{}, k.Wp};
    if (copies && (rc = pack<S>(jobs, copies, C, k.pitch, st)) != 0) return rc;
    a.X = {k.Xp ? k.Xp : (const char*)x, k.pitch, (int)N, N * k.pitch};
    a.W = {k.Wp ? k.Wp : (const char*)w, k.pitch, (int)V, V * k.pitch};
    a.bias = bias;
    a.V = (int)V; a.N = (int)N; a.tilesV = p.tilesV; a.tilesN = p.tilesN;
    a.stages = (int)stages_of(C, P);
    a.target = target; a.v0 = 0;
    a.pm = p.pm; a.ps = p.ps; a.tl = p.tl;
#define SSECG_CE_LSE(...) do { using M = __VA_ARGS__; SSECG_CE_LAUNCH(M, ce_lse_kernel<M>, dim3(p.tilesV * p.tilesN), st, a); } while (0)
    SSECG_CE_TILES(p.c, SSECG_CE_LSE, false, false);
#undef SSECG_CE_LSE
    const Joined out = {lse, gate, reduction == 0 ? loss : p.row, reduction == 0 ? nullptr : loss, count};
    const int mean = reduction == 1 ? 1 : 0;
#define SSECG_CE_JOIN(ROWS, WHOLE)                                                                                                        \
    hipLaunchKernelGGL((ce_join_kernel<ROWS, WHOLE>), dim3((unsigned)((N + ROWS - 1) / ROWS)), dim3(1024), 0, st, p.pm, p.ps, p.tl, p.parts, \
                       (int)N, (int)V, target, counts, mean, out)
    // Few rows whose parts one workgroup reads in a few rounds: the total in the same launch.  Forward passes over 64 columns in fp16, one
    // workgroup for all against many and a second launch: 8 rows and 500 / 2000 / 4096 parts 7.2 / 10.8 / 17.0 us against 9.4 / 12.1 / 17.3, 2 rows
    // and 2000 / 4096 parts 11.1 / 17.2 against 10.8 / 14.3; 16 to 128 rows and 32 / 126 / 500 parts 6.9 / 8.6 / 16.8 against 8.9 / 9.0 / 10.3.
    // Else up to 64 rows: more strands each (2 rows a workgroup against 16, 8 rows and 2000 / 4096 parts 12.1 / 17.3 us against 15.1 /
    // 23.4, 32 rows 15.2 / 23.6 against 16.0 / 25.7, 64 rows 16.4 / 26.4 against 16.7 / 26.0); more rows: whole sectors of their parts
    // (128 rows 14.2 / 20.7 against 14.8 / 22.5; 256 rows 17.4 / 26.7 against 18.3 / 28.3).
    if (N <= 8 && p.parts <= 2048) {
        SSECG_CE_JOIN(8, true);
        return (int)hipGetLastError();
    }
    if (N <= 128 && p.parts <= 128) {
        SSECG_CE_JOIN(128, true);
        return (int)hipGetLastError();
    }
    if (N <= 64) SSECG_CE_JOIN(2, false);
    else SSECG_CE_JOIN(16, false);
#undef SSECG_CE_JOIN
    hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(1024), 0, st, target, ignore, (int)N, mean, out);
    return (int)hipGetLastError();
}

constexpr size_t kPieceBytes = (size_t)1 << 30;  // of E

struct BwdPlan {
    int64_t Vc, rowsE, pitchE, planeE;           // classes per piece (a multiple of 256 unless there is one piece); E's rows and bytes
    int pieces;
    Choice cl, cx, cw;                           // E, dx, dw
    float *coef, *fscale, *pdb, *planeX, *planeW;
    char *Xg, *E;
};

BwdPlan plan_bwd(Blob& ws, int dtype, int64_t N, int64_t C, int64_t V, bool want_x, bool want_w, bool want_b, bool x_direct) {
    BwdPlan p;
    const int P = planes_of(dtype);
    p.rowsE = up(N, 64);
    int64_t most = (int64_t)(kPieceBytes / (size_t)(p.rowsE * 2 * P)) / 256 * 256;
    if (most < 256) most = 256;
    if (most > kMaxPiece) most = kMaxPiece;
    const int64_t pieces = (V + most - 1) / most;
    p.Vc = pieces == 1 ? V : up((V + pieces - 1) / pieces, 256);
    p.pieces = (int)((V + p.Vc - 1) / p.Vc);
    p.pitchE = up(p.Vc, 256) * 2;
    p.planeE = p.rowsE * p.pitchE;
    p.cl = choose(p.Vc, N, stages_of(C, P), false);
    p.cx = choose(N, C, stages_of(p.Vc, P), true);
    p.cw = choose(p.Vc, C, stages_of(N, P), true);
    p.coef = ws.take<float>((size_t)N);
    p.fscale = ws.take<float>(1);
    p.pdb = ws.take<float>(want_b ? (size_t)(tiles_of(N, p.cl.side) * p.Vc) : 0);
    p.planeX = ws.take<float>(want_x && (p.cx.splits > 1 || p.pieces > 1) ? (size_t)p.cx.splits * N * C : 0);
    p.planeW = ws.take<float>(want_w && p.cw.splits > 1 ? (size_t)p.cw.splits * p.Vc * C : 0);
    p.Xg = ws.take<char>(want_w && x_direct ? (size_t)(N * C * 2) : 0);
    p.E = ws.take<char>(want_x || want_w ? (size_t)(P * p.planeE) : 0);
    return p;
}

template <typename S, bool TA>
int product(const ProdArgs& q, const Choice& c, hipStream_t st) {
    using T = typename Inner<S>::T;
    constexpr int P = Inner<S>::P;
    const dim3 grid((unsigned)(q.tilesA * q.tilesB), (unsigned)q.splits);
#define SSECG_CE_PROD(...) do { using M = __VA_ARGS__; SSECG_CE_LAUNCH(M, (ce_prod_kernel<M, S>), grid, st, q); } while (0)
    SSECG_CE_TILES(c, SSECG_CE_PROD, TA, true);
#undef SSECG_CE_PROD
    return 0;
}

template <typename S>
int ce_bwd(const float* dloss, const void* x, const void* w, const float* bias, const int64_t* target, const float* lse, const float* gate,
           const float* count, int dtype, int64_t N, int64_t C, int64_t V, int reduction, void* dx, void* dw, float* db, void* packed, void* ws,
           hipStream_t st) {
    using T = typename Inner<S>::T;
    constexpr int P = Inner<S>::P;
    Blob blob(ws);
    const Packed k = plan_packed(packed, x, w, dtype, N, C, V);
    const BwdPlan p = plan_bwd(blob, dtype, N, C, V, dx != nullptr, dw != nullptr, db != nullptr, !k.Xp);
    const char *X = k.Xp ? k.Xp : (const char*)x, *W = k.Wp ? k.Wp : (const char*)w;
    int rc = 0;
    Factor f = {dloss, reduction == 1 ? count : nullptr};
    if (reduction == 0) {
        hipLaunchKernelGGL(ce_coef_kernel, dim3(1), dim3(1024), 0, st, dloss, gate, (int)N, p.coef, p.fscale);
        f = {p.fscale, nullptr};
    }
    const char* Xw = X;                          // of dw: rows that do not count are zeros (a copy made by the forward pass has them so)
    if (dw && !k.Xp) {
        const PackJobs jobs = {{{x, N, Counts{gate, nullptr, 0, nullptr, 0.f}, p.Xg}}};
        if ((rc = pack<S>(jobs, 1, C, k.pitch, st)) != 0) return rc;
        Xw = p.Xg;
    }
    for (int i = 0; i < p.pieces; ++i) {
        const int64_t v0 = i * p.Vc, vn = V - v0 < p.Vc ? V - v0 : p.Vc;
        LogitArgs a = {};
        a.X = {X, k.pitch, (int)N, N * k.pitch};
        a.W = {W + v0 * k.pitch, k.pitch, (int)vn, V * k.pitch};
        a.bias = bias ? bias + v0 : nullptr;
        a.V = (int)vn; a.N = (int)N;
        a.tilesV = (int)tiles_of(vn, p.cl.side); a.tilesN = (int)tiles_of(N, p.cl.side);
        a.stages = (int)stages_of(C, P);
        a.target = target; a.v0 = v0;
        a.lse = lse; a.gate = gate; a.coef = reduction == 0 ? p.coef : nullptr;
        a.E = dx || dw ? p.E : nullptr; a.pitchE = p.pitchE; a.planeE = p.planeE; a.rowsE = (int)p.rowsE;
        a.pdb = p.pdb;
        a.db = db && a.tilesN == 1 ? db + v0 : nullptr;
        a.f = f;
        const dim3 grid(a.tilesV * a.tilesN);
#define SSECG_CE_GRAD(...)                                                              \
    do {                                                                                \
        using M = __VA_ARGS__;                                                          \
        if (db) SSECG_CE_LAUNCH(M, (ce_grad_kernel<M, true>), grid, st, a);             \
        else SSECG_CE_LAUNCH(M, (ce_grad_kernel<M, false>), grid, st, a);               \
    } while (0)
        SSECG_CE_TILES(p.cl, SSECG_CE_GRAD, false, false);
#undef SSECG_CE_GRAD
        SumJobs jobs = {};
        int sums = 0;
        if (db && !a.db) jobs.job[sums++] = {p.pdb, a.tilesN, vn, 0, db + v0};
        if (dx) {                                // E along its rows, W across
            ProdArgs q = {};
            q.A = {p.E, p.pitchE, (int)N, p.planeE};
            q.B = {W + v0 * k.pitch, k.pitch, (int)vn, V * k.pitch};
            q.rows = (int)N; q.cols = (int)C;
            q.tilesA = (int)tiles_of(N, p.cx.side); q.tilesB = (int)tiles_of(C, p.cx.side);
            q.stages = (int)stages_of(vn, P); q.splits = p.cx.splits;
            q.plane = p.cx.splits > 1 || p.pieces > 1 ? p.planeX : nullptr;
            q.add = i > 0; q.out = dx; q.f = f;
            if ((rc = product<S, false>(q, p.cx, st)) != 0) return rc;
        }
        if (dw) {                                // both across
            ProdArgs q = {};
            q.A = {p.E, p.pitchE, (int)p.rowsE, p.planeE};
            q.B = {Xw, k.pitch, (int)N, N * k.pitch};
            q.rows = (int)vn; q.cols = (int)C;
            q.tilesA = (int)tiles_of(vn, p.cw.side); q.tilesB = (int)tiles_of(C, p.cw.side);
            q.stages = (int)stages_of(N, P); q.splits = p.cw.splits;
            q.plane = p.cw.splits > 1 ? p.planeW : nullptr;
            q.out = (S*)dw + v0 * C; q.f = f;
            if ((rc = product<S, true>(q, p.cw, st)) != 0) return rc;
            if (q.plane) jobs.job[sums++] = {p.planeW, p.cw.splits, vn * C, 1, (S*)dw + v0 * C};
        }
        if (dx && i + 1 == p.pieces && (p.cx.splits > 1 || p.pieces > 1)) jobs.job[sums++] = {p.planeX, p.cx.splits, N * C, 1, dx};
        if (sums) {
            int64_t most = 0;
            for (int n = 0; n < sums; ++n) most = jobs.job[n].n > most ? jobs.job[n].n : most;
            hipLaunchKernelGGL((ce_sum_kernel<S>), dim3(grid_for(most), sums), dim3(256), 0, st, jobs, f);
        }
    }
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t ssecg_linear_ce_packed_bytes(const void* x, const void* weight, int dtype, int64_t N, int64_t C, int64_t V) {
    if (!x || !weight || !dtype_ok(dtype) || !shape_ok(N, C, V)) return 0;
    return plan_packed(nullptr, x, weight, dtype, N, C, V).bytes;
}

size_t ssecg_linear_ce_fwd_workspace(int dtype, int64_t N, int64_t C, int64_t V) {
    if (!dtype_ok(dtype) || !shape_ok(N, C, V)) return 0;
    Blob b(nullptr);
    plan_fwd(b, dtype, N, C, V);
    return b.at;
}

int ssecg_linear_ce_fwd(const void* x, const void* weight, const float* bias, const int64_t* target, const float* conf, double thresh,
                        int64_t ignore_index, int dtype, int64_t N, int64_t C, int64_t V, int reduction, float* loss, float* lse, float* gate,
                        float* count, void* packed, size_t packed_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (!x || !weight || !target || !loss || !lse || !gate || !count || !workspace || !dtype_ok(dtype) || !shape_ok(N, C, V) || reduction < 0 ||
        reduction > 2 || ((uintptr_t)workspace & 255) || ((uintptr_t)packed & 255))
        return SSECG_E_INVAL;
    if (workspace_bytes < ssecg_linear_ce_fwd_workspace(dtype, N, C, V)) return SSECG_E_WORKSPACE;
    const size_t keep = ssecg_linear_ce_packed_bytes(x, weight, dtype, N, C, V);
    if (packed_bytes < keep || (keep && !packed)) return SSECG_E_WORKSPACE;
    SSECG_LM_DTYPE(dtype, S, return ce_fwd<S>(x, weight, bias, target, conf, (float)thresh, ignore_index, dtype, N, C, V, reduction, loss, lse, gate,
                                              count, packed, workspace, (hipStream_t)stream));
}

size_t ssecg_linear_ce_bwd_workspace(int dtype, int64_t N, int64_t C, int64_t V, int want_dx, int want_dw, int want_db) {
    if (!dtype_ok(dtype) || !shape_ok(N, C, V)) return 0;
    Blob b(nullptr);
    plan_bwd(b, dtype, N, C, V, want_dx != 0, want_dw != 0, want_db != 0, true);
    return b.at;
}

int ssecg_linear_ce_bwd(const float* dloss, const void* x, const void* weight, const float* bias, const int64_t* target, const float* lse,
                        const float* gate, const float* count, int dtype, int64_t N, int64_t C, int64_t V, int reduction, void* dx, void* dweight,
                        float* dbias, const void* packed, size_t packed_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (!dloss || !x || !weight || !target || !lse || !gate || !count || !workspace || (!dx && !dweight && !dbias) || !dtype_ok(dtype) ||
        !shape_ok(N, C, V) || reduction < 0 || reduction > 2 || ((uintptr_t)workspace & 255) || ((uintptr_t)packed & 255))
        return SSECG_E_INVAL;
    if (workspace_bytes < ssecg_linear_ce_bwd_workspace(dtype, N, C, V, dx != nullptr, dweight != nullptr, dbias != nullptr)) return SSECG_E_WORKSPACE;
    const size_t keep = ssecg_linear_ce_packed_bytes(x, weight, dtype, N, C, V);
    if (packed_bytes < keep || (keep && !packed)) return SSECG_E_WORKSPACE;
    SSECG_LM_DTYPE(dtype, S, return ce_bwd<S>(dloss, x, weight, bias, target, lse, gate, count, dtype, N, C, V, reduction, dx, dweight, dbias,
                                              (void*)packed, workspace, (hipStream_t)stream));
}

}  // extern "C"
