// The matrix product under linear_ce.hip and muon.hip: D[i][j] = sum_k A[i][k] B[j][k] on the bf16 / fp16 matrix pipe, both
// operands with k fastest.
//
// An operand is one or two PLANES of 16-bit values.  One plane: the data itself (bf16 or fp16).  Two planes (fp16): a 32-bit value
// v, scaled by a power of two into fp16's normal range, as hi = fp16(v) and lo = fp16(v - hi) - 22 to 23 significant bits - and
// D = hi hi + hi lo + lo hi in fp32 accumulators (the dropped lo lo is 2^-22 of the product and of random sign).  Three 16-bit
// products run at 1/3 of 2.5 PFLOP/s; the fp32 matrix pipe's peak is 0.157.  Two planes lie interleaved, 32 hi then 32 lo, so that
// a stage of a row is 128 consecutive bytes either way: 64 k of one plane or 32 k of both.
//
// Tile BM x BN by WM x WN waves, v_mfma_f32_32x32x16.  Stages travel by LDS-DMA (16 bytes a lane, no registers) into a ring of R
// slots, requested R - 1 stages ahead with counted waits and one barrier per stage; the fragments of a k step are read while the
// step before it is multiplied, across the barrier too.  A stage's LDS row is 8 chunks of 16 bytes.  Chunk c of row r lies at
// position c ^ (r & 7): the DMA writes positions in lane order, so the lane fetches the permuted chunk, and 8 rows read at one k by
// 8 lanes fall into 8 different bank groups.
//
// Bounds: a row index beyond the operand is clamped to its last row (the caller masks the result); k is padded with zeros in
// memory to a whole stage, so the loads have no other condition.  Offsets within a tile are 32 bits: 256 pitch < 2^32.
#pragma once
#include "lm_common.h"

namespace ssecg_lm {

struct Operand {
    const char* base;    // 16-byte aligned
    int64_t pitch;       // bytes of a row, a multiple of 128, below 2^24
    int rows;
};
constexpr int64_t kMaxPitch = (1 << 24) - 1;

// bytes of element k (a multiple of 8 within its 16 bytes) in plane q of a row
template <int P> __host__ __device__ __forceinline__ int64_t kbyte(int64_t k, int q = 0) {
    return P == 1 ? k * 2 : (k >> 5) * 128 + q * 64 + (k & 31) * 2;
}

// LDS-DMA: the lane's 16 bytes at base + off land at lds_wave_base + 16 lane.  From inline asm, so that hipcc's wait counts do not
// drain the queue before every LDS read; no register is written by the load, and the waits are MmTile::stage_wait's.
__device__ __forceinline__ void lds_dma16(const char* base, unsigned off, unsigned lds_wave_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(base), "s"(lds_wave_base) : "memory");
}

template <typename T> struct Frag;
template <> struct Frag<__bf16> {
    typedef bf16x8 type;
    static __device__ __forceinline__ f32x16 mfma(type a, type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<_Float16> {
    typedef f16x8 type;
    static __device__ __forceinline__ f32x16 mfma(type a, type b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

template <typename T_, int P_, int BM_, int BN_, int WM_, int WN_, int R_>
struct MmTile {
    using T = T_;
    using F = Frag<T>;
    using V8 = typename F::type;
    static constexpr int P = P_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, R = R_;
    static constexpr int NW = WM * WN, NT = NW * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    static constexpr int BK = P == 1 ? 64 : 32;                 // k of a stage
    static constexpr int STEP = 128;                            // bytes a row advances per stage
    static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, PPW = PA + PB;   // 1 KB pieces (8 rows) per wave and stage
    static constexpr int SLOT = (BM + BN) * 128;
    static constexpr int LDS = R * SLOT;
    static_assert(PA * NW * 8 == BM && PB * NW * 8 == BN, "every wave requests the same number of pieces");
    static_assert(R >= 2 && (R - 2) * PPW <= 63, "vmcnt counts to 63");

    template <int N> static __device__ __forceinline__ void stage_wait() {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
    }

    // acc += the tile at rows a0 of A and b0 of B over stages [s0, s0 + n); all waves of the workgroup call it together
    static __device__ __forceinline__ void run(const Operand& A, int a0, const Operand& B, int b0, int s0, int n, char* lds,
                                               f32x16 (&acc)[TM][TN]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN, r = lane & 31, h = lane >> 5;
        const unsigned ldsbase = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        unsigned off[PPW];
        const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
        for (int i = 0; i < PPW; ++i) {
            int row = (i < PA ? (wave * PA + i) * 8 : (wave * PB + i - PA) * 8) + (lane >> 3);
            const int last = i < PA ? A.rows - 1 - a0 : B.rows - 1 - b0;
            row = row < last ? row : last;
            off[i] = (unsigned)row * (unsigned)(i < PA ? A.pitch : B.pitch) + chunk * 16;
        }
        const char* pA = A.base + a0 * A.pitch + (int64_t)s0 * STEP;   // of the stage that is requested next
        const char* pB = B.base + b0 * B.pitch + (int64_t)s0 * STEP;
        const unsigned dstA = ldsbase + wave * PA * 1024, dstB = ldsbase + BM * 128 + wave * PB * 1024;
        auto issue = [&](int slot) {
#pragma unroll
            for (int i = 0; i < PPW; ++i)
                lds_dma16(i < PA ? pA : pB, off[i], (i < PA ? dstA + i * 1024 : dstB + (i - PA) * 1024) + slot * SLOT);
            pA += STEP;
            pB += STEP;
        };
#pragma unroll
        for (int s = 0; s < R - 1; ++s)
            if (s < n) issue(s);
        // fragment offsets: row (wave tile + 32 i + r), chunk (2 kk + h) of this lane
        const int swz = r & 7;
        const char* fa = lds + (wm * TM * 32 + r) * 128;
        const char* fb = lds + BM * 128 + (wn * TN * 32 + r) * 128;
        constexpr int KK = P == 1 ? 4 : 2;                      // k steps of 16 in a stage
        V8 a[2][P][TM], b[2][P][TN];                            // two sets: one is multiplied while the other is read
        auto frags = [&](int set, int slot, int kk) {
#pragma unroll
            for (int q = 0; q < P; ++q) {
                const int c = slot * SLOT + ((4 * q + 2 * kk + h) ^ swz) * 16;
#pragma unroll
                for (int i = 0; i < TM; ++i) a[set][q][i] = *reinterpret_cast<const V8*>(fa + i * 4096 + c);
#pragma unroll
                for (int j = 0; j < TN; ++j) b[set][q][j] = *reinterpret_cast<const V8*>(fb + j * 4096 + c);
            }
        };
        auto multiply = [&](int set) {
            // two planes: the small products first, each product over all blocks: no accumulator is used twice in a row
#pragma unroll
            for (int q = P == 1 ? 2 : 0; q < 3; ++q)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = F::mfma(a[set][q == 0 ? P - 1 : 0][i], b[set][q == 1 ? P - 1 : 0][j], acc[i][j]);
        };
        if (n > 0) {
            if (R > 3 && n > 2) stage_wait<(R > 3 ? 2 * PPW : 0)>();
            else if (R > 2 && n > 1) stage_wait<(R > 2 ? PPW : 0)>();
            else stage_wait<0>();
            frags(0, 0, 0);
        }
        int slot = 0;
        for (int s = 0; s < n; ++s) {
            const int next = slot + 1 == R ? 0 : slot + 1;
            // the stage that is requested R - 1 ahead goes into the slot of the stage before this one: every wave has read that one
            // (it passed the barrier below with no LDS read outstanding)
            if (s + R - 1 < n) issue(slot == 0 ? R - 1 : slot - 1);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (kk + 1 < KK) {
                    frags((kk + 1) & 1, slot, kk + 1);
                } else if (s + 1 < n) {
                    // the next stage has landed when only the pieces of the stages requested after it are outstanding
                    const int ahead = n - 2 - s < R - 2 ? n - 2 - s : R - 2;
                    if (R > 3 && ahead == 2) stage_wait<(R > 3 ? 2 * PPW : 0)>();
                    else if (R > 2 && ahead == 1) stage_wait<(R > 2 ? PPW : 0)>();
                    else stage_wait<0>();
                    frags((kk + 1) & 1, next, 0);
                }
                __builtin_amdgcn_sched_barrier(0);   // the reads above travel under the products below
                multiply(kk & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            slot = next;
        }
        // LDS may be reused by the caller behind this point (every wave has read its last stage)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }

    static __device__ __forceinline__ void zero(f32x16 (&acc)[TM][TN]) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    }
    // element e of acc[i][j] is row a0 + arow(i, e), column b0 + bcol(j)
    static __device__ __forceinline__ int arow(int i, int e) {
        const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / WN;
        return wm * TM * 32 + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    }
    static __device__ __forceinline__ int wave_row() { return (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WN) * TM * 32; }
    static __device__ __forceinline__ int wave_col() { return (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WN) * TN * 32; }
    static __device__ __forceinline__ int bcol(int j) {
        const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % WN;
        return wn * TN * 32 + j * 32 + (lane & 31);
    }
};

// The wave's tile as 16-bit values, 16 bytes a lane, through a region of LDS that only this wave uses (after MmTile::run): an
// accumulator's lanes run along B and its registers along A, so stores straight from it would be 2 bytes a lane (along B) or 8
// bytes to 32 different rows (along A).
//   store_rows: rows of A's index, B's index fastest;  dst(row, first column, 8 values), row and column relative to the wave's tile
//   store_cols: rows of B's index, A's index fastest;  dst(column, first row, 8 values)
template <class M> struct WaveStore {
    static constexpr int SI = M::TM > 1 ? 2 : 1;                          // 32-row blocks that store_cols takes at a time
    static constexpr int PC = SI * 64 + 16, PR = M::TN * 64 + 16;         // bytes of a row in LDS; the pad spreads the banks
    static constexpr int BYTES = M::TN * 32 * PC > 32 * PR ? M::TN * 32 * PC : 32 * PR;
    static_assert(M::NW * BYTES <= M::LDS, "the regions of all waves fit the tile's LDS");

    static __device__ __forceinline__ char* region(char* lds) { return lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * BYTES; }
    static __device__ __forceinline__ void fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

    template <typename VAL, typename DST> static __device__ __forceinline__ void store_rows(char* reg, VAL val, DST dst) {
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < M::TM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int j = 0; j < M::TN; ++j)
                    *reinterpret_cast<uint16_t*>(reg + (8 * (e >> 2) + 4 * h + (e & 3)) * PR + (j * 32 + r) * 2) = val(i, j, e);
            fence();
#pragma unroll
            for (int q = 0; q < M::TN * 2; ++q) {
                const int at = q * 64 + lane, row = at / (M::TN * 4), c = at % (M::TN * 4);
                dst(i * 32 + row, c * 8, *reinterpret_cast<const u32x4*>(reg + row * PR + c * 16));
            }
            fence();
        }
    }
    template <typename VAL, typename DST> static __device__ __forceinline__ void store_cols(char* reg, VAL val, DST dst) {
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i0 = 0; i0 < M::TM; i0 += SI) {
#pragma unroll
            for (int i = 0; i < SI; ++i)
#pragma unroll
                for (int j = 0; j < M::TN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        u32x2 v;
                        v[0] = (unsigned)val(i0 + i, j, 4 * g) | (unsigned)val(i0 + i, j, 4 * g + 1) << 16;
                        v[1] = (unsigned)val(i0 + i, j, 4 * g + 2) | (unsigned)val(i0 + i, j, 4 * g + 3) << 16;
                        *reinterpret_cast<u32x2*>(reg + (j * 32 + r) * PC + (i * 32 + 8 * g + 4 * h) * 2) = v;
                    }
            fence();
#pragma unroll
            for (int q = 0; q < M::TN * 2 * SI; ++q) {
                const int at = q * 64 + lane, row = at / (SI * 4), c = at % (SI * 4);
                dst(row, i0 * 32 + c * 8, *reinterpret_cast<const u32x4*>(reg + row * PC + c * 16));
            }
            fence();
        }
    }
};

// Consecutive workgroups run on different XCDs (8, round robin), each with an L2 of its own: give every XCD a contiguous range of
// tiles, so that neighbours share operand rows in one L2.  A permutation of [0, n).
__device__ __forceinline__ int xcd_tile(int bid, int n) {
    const int q = n >> 3, rem = n & 7, x = bid & 7, i = bid >> 3;
    return x * q + (x < rem ? x : rem) + i;
}

// The power of two that brings |amax| to [2^14, 2^15): its exponent
__device__ __forceinline__ int scale_exp(float amax) {
    if (!(amax > 0.f)) return 0;
    int e;
    frexpf(amax, &e);                       // amax = m 2^e, m in [0.5, 1)
    return 15 - e;
}

__device__ __forceinline__ uint16_t bits16(_Float16 v) { return __builtin_bit_cast(uint16_t, v); }
__device__ __forceinline__ uint16_t bits16(__bf16 v) { return __builtin_bit_cast(uint16_t, v); }

// plane q (0 = hi, 1 = lo) of v
__device__ __forceinline__ uint16_t plane16(float v, int q) {
    const _Float16 hi = (_Float16)v;
    if (q == 0) return bits16(hi);
    const float f = (float)hi;
    return __builtin_isinf(f) ? 0 : bits16((_Float16)(v - f));   // an infinity stays one instead of inf - inf
}

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    const float f = (float)hi;
    lo = __builtin_isinf(f) ? (_Float16)0.f : (_Float16)(v - f);   // an infinity stays one instead of inf - inf
}

}  // namespace ssecg_lm
