// The matrix product under linear_ce.hip and muon.hip: D[i][j] = sum_k A[i][k] B[j][k] on the bf16 / fp16 matrix pipe, both
// operands with k fastest.
//
// An operand is one or two PLANES of 16-bit values.  One plane: the data itself (bf16 or fp16).  Two planes (fp16): a 32-bit value
// v, scaled by a power of two into fp16's normal range, as hi = fp16(v) and lo = fp16(v - hi) - 22 to 23 significant bits - and
// D = hi hi + hi lo + lo hi in fp32 accumulators (the dropped lo lo is 2^-22 of the product and of random sign).  Three 16-bit
// products run at 1/3 of 2.5 PFLOP/s; the fp32 matrix pipe's peak is 0.157.
//
// Tile BM x BN by WM x WN waves, v_mfma_f32_32x32x16.  Stages travel by LDS-DMA (16 bytes a lane, no registers) into a ring of R
// slots, requested R - 1 stages ahead with counted waits and one barrier per stage.  A stage's LDS row is 128 bytes = 8 chunks of
// 16: 64 k of one plane, or 32 k of both.  Chunk c of row r lies at position c ^ (r & 7): the DMA writes positions in lane order,
// so the lane fetches the permuted chunk, and 8 rows read at one k by 8 lanes fall into 8 different bank groups.
//
// Bounds: a row index beyond the operand is clamped to its last row (the caller masks the result); k is padded with zeros in
// memory to a whole stage, so the loads have no other condition.
#pragma once
#include "lm_common.h"

namespace ssecg_lm {

struct Operand {
    const char* base;    // 16-byte aligned
    int64_t pitch;       // bytes of a row, multiple of 16
    int64_t plane;       // bytes from the hi plane to the lo plane
    int rows;
};

__device__ __forceinline__ void lds_dma16(const char* src, unsigned lds_wave_base) {
    // from inline asm, so that hipcc's wait counts do not drain the queue before every LDS read; m0 is left as it was.  No register
    // is written by the load; the waits are in MmTile::stage_wait.
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(lds_wave_base) : "memory");
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
    static constexpr int STEP = BK * 2;                         // bytes a row advances per stage
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
        const char* src[PPW];
        const int chunk = (lane & 7) ^ (lane >> 3);
        const int64_t off = P == 1 ? chunk * 16 : (chunk & 3) * 16;
#pragma unroll
        for (int i = 0; i < PPW; ++i) {
            const Operand& o = i < PA ? A : B;
            int row = i < PA ? a0 + (wave * PA + i) * 8 : b0 + (wave * PB + i - PA) * 8;
            row += lane >> 3;
            row = row < o.rows ? row : o.rows - 1;
            src[i] = o.base + row * o.pitch + (int64_t)s0 * STEP + off + (P == 2 && chunk >= 4 ? o.plane : 0);
        }
        const unsigned dstA = ldsbase + wave * PA * 1024, dstB = ldsbase + BM * 128 + wave * PB * 1024;
        auto issue = [&](int slot) {
#pragma unroll
            for (int i = 0; i < PPW; ++i) {
                lds_dma16(src[i], __builtin_amdgcn_readfirstlane((i < PA ? dstA + i * 1024 : dstB + (i - PA) * 1024) + slot * SLOT));
                src[i] += STEP;
            }
        };
#pragma unroll
        for (int s = 0; s < R - 1; ++s)
            if (s < n) issue(s);
        // fragment offsets: row (wave tile + 32 i + r), chunk (2 kk + h) of this lane
        const int swz = r & 7;
        const char* fa = lds + (wm * TM * 32 + r) * 128;
        const char* fb = lds + BM * 128 + (wn * TN * 32 + r) * 128;
        int slot = 0;
        for (int s = 0; s < n; ++s) {
            // stage s has landed when only the pieces of the stages requested after it are outstanding
            const int ahead = n - 1 - s < R - 2 ? n - 1 - s : R - 2;
            if (R > 3 && ahead == 2) stage_wait<(R > 3 ? 2 * PPW : 0)>();
            else if (R > 2 && ahead == 1) stage_wait<(R > 2 ? PPW : 0)>();
            else stage_wait<0>();
            int next = slot + R - 1;
            next = next >= R ? next - R : next;
            if (s + R - 1 < n) issue(next);
            const char* pa = fa + slot * SLOT;
            const char* pb = fb + slot * SLOT;
            if constexpr (P == 1) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const int c = ((2 * kk + h) ^ swz) * 16;
                    V8 a[TM], b[TN];
#pragma unroll
                    for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const V8*>(pa + i * 4096 + c);
#pragma unroll
                    for (int j = 0; j < TN; ++j) b[j] = *reinterpret_cast<const V8*>(pb + j * 4096 + c);
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(a[i], b[j], acc[i][j]);
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int ch = ((2 * kk + h) ^ swz) * 16, cl = ((4 + 2 * kk + h) ^ swz) * 16;
                    V8 ah[TM], al[TM], bh[TN], bl[TN];
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        ah[i] = *reinterpret_cast<const V8*>(pa + i * 4096 + ch);
                        al[i] = *reinterpret_cast<const V8*>(pa + i * 4096 + cl);
                    }
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        bh[j] = *reinterpret_cast<const V8*>(pb + j * 4096 + ch);
                        bl[j] = *reinterpret_cast<const V8*>(pb + j * 4096 + cl);
                    }
                    // the small products first, each product over all blocks: no accumulator is used twice in a row
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(al[i], bh[j], acc[i][j]);
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(ah[i], bl[j], acc[i][j]);
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(ah[i], bh[j], acc[i][j]);
                }
            }
            slot = slot + 1 == R ? 0 : slot + 1;
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
    static __device__ __forceinline__ int bcol(int j) {
        const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % WN;
        return wn * TN * 32 + j * 32 + (lane & 31);
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

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    const float f = (float)hi;
    lo = __builtin_isinf(f) ? (_Float16)0.f : (_Float16)(v - f);   // an infinity stays one instead of inf - inf
}

}  // namespace ssecg_lm
