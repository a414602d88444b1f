// The matrix product under linear_ce.hip and muon.hip: D[i][j] = sum_k A[i][k] B[j][k] on the bf16 / fp16 matrix pipe, both
// operands with k fastest.
//
// An operand is one to three PLANES of 16-bit values.
//   One: the data itself (bf16 or fp16).
//   Two (fp16), for values of a known range: v, scaled by a power of two into fp16's normal range, as hi = fp16(v) and
// lo = fp16(v - hi) - 22 to 23 significant bits - and D = hi hi + hi lo + lo hi in fp32 accumulators (the dropped lo lo is 2^-22 of
// the product and of random sign but on a Gram matrix's diagonal).  FULL tiles, of up to 4 blocks a wave, form lo lo too and sum the three
// small products apart, so that the large one takes one rounding per k step instead of three; beyond, registers do not allow it, and
// the roundings of longer sums count for more.  The planes lie interleaved, 32 hi then 32 lo, so that a stage of a row is 128
// consecutive bytes: 32 k.
//   Three (bf16), for any 32-bit values: b0 = bf16(v), b1 = bf16(v - b0), b2 = v - b0 - b1.  8 + 8 + 8 bits hold v exactly, and at
// its own exponent: no scale, no floor, each row and each element is as precise as in a 32-bit product whatever else the operand
// holds.  D is the six products down to 2^-18; the three dropped are at most 2^-26 of |a||b|.  The planes lie one behind the other, each
// like an operand of one plane, and a stage of 64 k is six stages, one per product.
// Three 16-bit products run at 1/3 of 2.5 PFLOP/s, six at 1/6; the fp32 matrix pipe's peak is 0.157.
//
// Tile BM x BN by WM x WN waves, v_mfma_f32_32x32x16.  Stages travel by LDS-DMA (16 bytes a lane, no registers) into a ring of R
// slots, requested R - 1 stages ahead with counted waits and one barrier per stage; the fragments of a k step are read while the
// step before it is multiplied, across the barrier too.  A stage's LDS row is 8 chunks of 16 bytes.  Chunk c of row r lies at
// position c ^ (r / 2 % 8): the DMA writes positions in lane order, so the lane fetches the permuted chunk, and the 16 rows that 16
// lanes read at one k cover the 64 banks once (two rows of 128 bytes are one pass over the banks).
//
// An operand may also lie with k SLOW (TA / TB): [k][index], its index padded in memory to whole chunks of 64.  Its stage in LDS is
// BK rows of the tile's indices; ds_read_b64_tr_b16 gives a lane 4 consecutive k of its index, so two of them are a fragment.  The
// chunks of a row are permuted by its row so that the 8 rows of a read fall into different banks.
//
// KG groups of waves, each with a ring of its own, may share a tile's k (group g takes its g-th share of the stages): half the chain
// of stages where there are too few tiles to fill the chip.  Their sums are joined in LDS, and the first group goes on alone.
//
// Bounds: an index beyond a k-fast operand is clamped to its last row, a chunk beyond a k-slow one to its row's last chunk (the
// caller masks the result).  k-fast operands are padded with zeros to a whole stage; of a k-slow operand rows beyond the last are
// read as the last one, and the other operand holds zeros there.  Offsets within a tile are 32 bits: 256 pitch < 2^32.
#pragma once
#include "lm_common.h"

namespace ssecg_lm {

struct Operand {
    const char* base;    // 16-byte aligned
    int64_t pitch;       // bytes of a row, a multiple of 128, below 2^24
    int rows;            // rows in memory: indices, or k of a k-slow operand
    int64_t plane = 0;   // three planes: bytes from one to the next
};
constexpr int64_t kMaxPitch = (1 << 24) - 1;

// bytes of element k (a multiple of 8 within its 16 bytes) in plane q of a row (three planes: in each of them)
template <int P> __host__ __device__ __forceinline__ int64_t kbyte(int64_t k, int q = 0) {
    return P != 2 ? k * 2 : (k >> 5) * 128 + q * 64 + (k & 31) * 2;
}

// Three planes: the products of a stage of 64 k, by the plane of A and of B; consecutive ones share a plane where they can.
constexpr int kTerms = 6;
constexpr unsigned kTermsA = 0u | 0u << 2 | 0u << 4 | 1u << 6 | 1u << 8 | 2u << 10;
constexpr unsigned kTermsB = 0u | 1u << 2 | 2u << 4 | 0u << 6 | 1u << 8 | 0u << 10;

// LDS-DMA: the lane's 16 bytes at base + off land at lds_wave_base + 16 lane.  From inline asm, so that hipcc's wait counts do not
// drain the queue before every LDS read; no register is written by the load, and the waits are MmTile::stage_wait's.
__device__ __forceinline__ void lds_dma16(const char* base, unsigned off, unsigned lds_wave_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(base), "s"(lds_wave_base) : "memory");
}

// a pointer that is the same in every lane, in scalar registers
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const char*)((uint64_t)hi << 32 | lo);
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

template <typename T_, int P_, int BM_, int BN_, int WM_, int WN_, int R_, bool TA_ = false, bool TB_ = false, int KG_ = 1, bool FULL_ = false>
struct MmTile {
    using T = T_;
    using F = Frag<T>;
    using V8 = typename F::type;
    static constexpr int P = P_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, R = R_;
    static constexpr int FP = P == 2 ? 2 : 1;                   // planes of a stage
    static constexpr bool TA = TA_, TB = TB_;
    static constexpr int KG = KG_, NW = WM * WN, NT = KG * NW * 64;   // waves of a group, threads of the workgroup
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    static constexpr bool FULL = FULL_, APART = FULL && P == 2 && TM * TN <= 4;
    static constexpr int BK = FP == 1 ? 64 : 32;                // k of a stage
    static constexpr int STEP = 128;                            // bytes of a k-fast row in a stage
    static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, PPW = PA + PB;   // 1 KB pieces (8 rows) per wave and stage
    static constexpr int SLOT = (BM + BN) * 128;
    static constexpr int LDS = KG * R * SLOT;
    static_assert(PA * NW * 8 == BM && PB * NW * 8 == BN, "every wave requests the same number of pieces");
    static_assert(R >= 2 && (R - 2) * PPW <= 63, "vmcnt counts to 63");

    // waits for every piece of this wave but those of `ahead` (uniform, at most AHEAD) stages, and for the other waves
    template <int AHEAD> static __device__ __forceinline__ void stage_wait(int ahead) {
        if constexpr (AHEAD > 0)
            if (ahead < AHEAD) return stage_wait<AHEAD - 1>(ahead);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(AHEAD * PPW) : "memory");
    }

    // k-slow stage: BK rows of ROW bytes (SIDE indices); position of chunk c of row k
    template <int SIDE> struct Slow {
        static constexpr int ROW = SIDE * 2 * FP, CH = ROW / 16;
        static __device__ __forceinline__ int swz(int k) { return ((k & 3) << 2 | (k >> 2 & 3)) & (CH - 1); }
        // lane's 4 indices x 4 k of the read that gives lane (r, h) the k 16 kk + 8 h + 4 part .. + 3 of index 32 blk + r, plane q
        static __device__ __forceinline__ int at(int lane, int blk, int kk, int part, int q) {
            const int l = lane & 15, g = lane >> 4;
            const int k = kk * 16 + 8 * (g >> 1) + 4 * part + (l >> 2);
            const int c = (blk * FP + q) * 4 + 2 * (g & 1) + ((l & 3) >> 1);
            return k * ROW + ((c ^ swz(k)) << 4) + 8 * (l & 1);
        }
    };
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ V8 read_tr(const char* lo, const char* hi) {
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi);
        return __builtin_bit_cast(V8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }

    // one operand's pieces of a stage: this wave's PC pieces of 1 KB, SIDE indices from i0
    template <int SIDE, int PC, bool SLOW, unsigned TERMS> struct Loader {
        unsigned off[PC];
        const char* base;                      // of the stage that is requested next
        const char* stage;                     // three planes: of its 64 k in the first plane
        int64_t plane;
        int term;
        unsigned dst;
        int64_t step;
        int left;                              // k-slow: rows from the stage that is requested next
        unsigned pitch;
        int row0;                              // k-slow: row of the lane in its first piece
        static constexpr int RPP = SLOW ? 1024 / Slow<SIDE>::ROW : 8;     // rows of a piece
        __device__ __forceinline__ Loader(const Operand& o, int i0, int s0, int lane, int wave, unsigned lds) {
            dst = lds + wave * PC * 1024;
            pitch = (unsigned)o.pitch;
            if constexpr (P == 3) {
                term = s0 % kTerms;
                s0 /= kTerms;
                plane = o.plane;
            }
            if constexpr (!SLOW) {
                base = o.base + i0 * o.pitch + (int64_t)s0 * STEP;
                step = STEP;
                const int last = o.rows - 1 - i0;
#pragma unroll
                for (int i = 0; i < PC; ++i) {
                    int row = (wave * PC + i) * 8 + (lane >> 3);
                    const int chunk = (lane & 7) ^ (row >> 1 & 7);
                    row = row < last ? row : last;
                    off[i] = (unsigned)row * pitch + (chunk << 4);
                }
            } else {
                using S = Slow<SIDE>;
                step = BK * o.pitch;
                base = o.base + s0 * step;
                left = o.rows - s0 * BK;
                const unsigned first = (unsigned)i0 * 2 * FP, most = pitch - 16;
                row0 = wave * PC * RPP + lane * 16 / S::ROW;
#pragma unroll
                for (int i = 0; i < PC; ++i) {
                    const int k = row0 + i * RPP;
                    const unsigned c = first + (((lane * 16 % S::ROW >> 4) ^ S::swz(k)) << 4);
                    off[i] = (unsigned)k * pitch + (c < most ? c : most);
                }
            }
            if constexpr (P == 3) {
                stage = base;
                base = stage + (TERMS >> 2 * term & 3) * plane;
            }
        }
        __device__ __forceinline__ void piece(int slot, int i, unsigned back = 0) {
            lds_dma16(uniform(base), off[i] - back, __builtin_amdgcn_readfirstlane(dst + i * 1024 + slot * SLOT));
        }
        __device__ __forceinline__ void advance() {
            if constexpr (P == 3) {
                if (++term == kTerms) {
                    term = 0;
                    stage += step;
                    if (SLOW) left -= BK;
                }
                base = stage + (TERMS >> 2 * term & 3) * plane;
            } else {
                base += step;
                if (SLOW) left -= BK;
            }
        }
        __device__ __forceinline__ void issue(int slot) {
            if (SLOW && left < BK) {           // the last stage: rows that do not exist are read as the last one
#pragma unroll
                for (int i = 0; i < PC; ++i) {
                    const int k = row0 + i * RPP;
                    piece(slot, i, k < left ? 0u : (unsigned)(k - left + 1) * pitch);
                }
            } else {
#pragma unroll
                for (int i = 0; i < PC; ++i) piece(slot, i);
            }
            advance();
        }
    };

    // acc = the tile at indices a0 of A and b0 of B over stages [s0, s0 + n); all waves of the workgroup call it together.  False for
    // the waves of the groups that are done: the tile is in the others' accumulators.
    static __device__ __forceinline__ bool run(const Operand& A, int a0, const Operand& B, int b0, int s0, int n, char* lds,
                                               f32x16 (&acc)[TM][TN]) {
        zero(acc);
        if constexpr (KG == 1) {
            sweep(A, a0, B, b0, s0, n, n, lds, acc);
            return true;
        } else {
            const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / NW, share = (n + KG - 1) / KG;
            const int from = group * share < n ? group * share : n, to = from + share < n ? from + share : n;
            sweep(A, a0, B, b0, s0 + from, to - from, share, lds + group * (R * SLOT), acc);
            // one group after the other leaves its sums in LDS, element-wise in lane order (no bank conflict)
            float* x = reinterpret_cast<float*>(lds) + (threadIdx.x & (NW * 64 - 1));
#pragma unroll
            for (int g = 1; g < KG; ++g) {
                if (group == g) {
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[((i * TN + j) * 16 + e) * (NW * 64)] = acc[i][j][e];
                }
                __syncthreads();
                if (group == 0) {
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[i][j][e] += x[((i * TN + j) * 16 + e) * (NW * 64)];
                }
                __syncthreads();
            }
            return group == 0;
        }
    }

    // a group's sweep over its n stages from s0; `most`: the stages of the largest group, whose barriers all waves meet
    static __device__ __forceinline__ void sweep(const Operand& A, int a0, const Operand& B, int b0, int s0, int n, int most, char* lds,
                                                 f32x16 (&acc)[TM][TN]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW;
        const int wm = wave / WN, wn = wave % WN, r = lane & 31, h = lane >> 5;
        const unsigned ldsbase = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        Loader<BM, PA, TA, kTermsA> la(A, a0, s0, lane, wave, ldsbase);
        Loader<BN, PB, TB, kTermsB> lb(B, b0, s0, lane, wave, ldsbase + BM * 128);
        auto issue = [&](int slot) {
            la.issue(slot);
            lb.issue(slot);
        };
#pragma unroll
        for (int s = 0; s < R - 1; ++s)
            if (s < n) issue(s);
        // fragment offsets, k fast: row (wave tile + 32 i + r), chunk (2 kk + h) of this lane
        const int swz = r >> 1 & 7;
        const char* fa = lds + (TA ? 0 : (wm * TM * 32 + r) * 128);
        const char* fb = lds + BM * 128 + (TB ? 0 : (wn * TN * 32 + r) * 128);
        constexpr int KK = BK / 16;                             // k steps of 16 in a stage
        constexpr bool AHEAD = !(P == 2 && TA && TB && TM * TN > 4);   // (there a second set of fragments would spill)
        V8 a[2][FP][TM], b[2][FP][TN];                          // two sets: one is multiplied while the other is read
        constexpr int NF = FP * (TM + TN);                       // fragments of a k step: in the order of their use, a k-slow B's last
        auto frag = [&](int set, int slot, int kk, int f) {
            const int q = f / (TM + TN), at = f % (TM + TN), i = TB || at == 0 ? at : at - TN, j = TB ? at - TM : at - 1;
            const int c = slot * SLOT + ((4 * q + 2 * kk + h) ^ swz) * 16;
            if (TB ? at < TM : at == 0 || at > TN) {
                if constexpr (TA)
                    a[set][q][i] = read_tr(fa + slot * SLOT + Slow<BM>::at(lane, wm * TM + i, kk, 0, q),
                                           fa + slot * SLOT + Slow<BM>::at(lane, wm * TM + i, kk, 1, q));
                else
                    a[set][q][i] = *reinterpret_cast<const V8*>(fa + i * 4096 + c);
            } else {
                if constexpr (TB)
                    b[set][q][j] = read_tr(fb + slot * SLOT + Slow<BN>::at(lane, wn * TN + j, kk, 0, q),
                                           fb + slot * SLOT + Slow<BN>::at(lane, wn * TN + j, kk, 1, q));
                else
                    b[set][q][j] = *reinterpret_cast<const V8*>(fb + j * 4096 + c);
            }
        };
        // Where a wave has its SIMD to itself, what else it issues is spread between the products of a k step, each of which keeps the
        // pipe busy for 32 cycles (A = X X^T at 4096: 230 -> 205 us); two waves cover for each other, and requests that leave
        // early count for more (8192 x 1024 x 65536 bf16: dx 951 us, 986 spread).
        constexpr bool SPREAD = TM * TN > 8;
        static_assert(!SPREAD || (!TA && !TB), "the spread requests are those of k-fast operands");
        f32x16 low[APART ? TM : 1][APART ? TN : 1];
        if constexpr (APART) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) low[i][j][e] = 0.f;
        }
        auto multiply = [&](int set, int extra, auto other) {
            constexpr int NM = (FP == 1 ? 1 : APART ? 4 : 3) * TM * TN;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                // two planes: the small products first, each product over all blocks: no accumulator is used twice in a row
                const int q = FP == 1 ? 2 : m / (TM * TN) - (APART ? 1 : 0), i = m % (TM * TN) / TN, j = m % TN;
                f32x16& to = APART && q < 2 ? low[APART ? i : 0][APART ? j : 0] : acc[i][j];
                to = F::mfma(a[set][q <= 0 ? FP - 1 : 0][i], b[set][q == 1 || q < 0 ? FP - 1 : 0][j], to);
                if (SPREAD) {
#pragma unroll
                    for (int x = m * extra / NM; x < (m + 1) * extra / NM; ++x) other(x);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        if (most > 0) {
            stage_wait<R - 2>(n < 1 ? 0 : n - 1 < R - 2 ? n - 1 : R - 2);
            if (AHEAD && n > 0)
#pragma unroll
                for (int f = 0; f < NF; ++f) frag(0, 0, 0, f);
        }
        int slot = 0, s = 0;
        for (; s < n; ++s) {
            // a stage is requested R - 1 ahead, into the slot of the stage before this one: every wave has read that one (it passed the
            // barrier below with no LDS read outstanding)
            const bool more = s + R - 1 < n;
            const int next = slot + 1 == R ? 0 : slot + 1, into = slot == 0 ? R - 1 : slot - 1;
            if (!SPREAD && more) issue(into);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (!AHEAD)
#pragma unroll
                    for (int f = 0; f < NF; ++f) frag(kk & 1, slot, kk, f);
                const bool within = kk + 1 < KK;
                // a fragment of the next k step (spread, behind the last stage: not used)
                auto read = [&](int f) { frag((kk + 1) & 1, within ? slot : next, within ? kk + 1 : 0, f); };
                auto read_all = [&]() {
                    if (AHEAD && !SPREAD)
#pragma unroll
                        for (int f = 0; f < NF; ++f) read(f);
                };
                if (within) {
                    read_all();
                } else if (s + 1 < n) {
                    // the next stage has landed when only the pieces of the stages requested after it are outstanding
                    const int ahead = n - 2 - s < R - 2 ? n - 2 - s : R - 2;
                    stage_wait<R - 2>(ahead);
                    read_all();
                }
                const int pieces = kk == 0 ? PPW : 0;
                __builtin_amdgcn_sched_barrier(0);   // the reads above travel under the products below
                multiply(kk & 1, NF + pieces, [&](int x) {
                    if (x >= pieces) read(x - pieces);
                    else if (more && x < PA) la.piece(into, x);
                    else if (more) lb.piece(into, x - PA);
                });
                if (SPREAD && more && kk == 0) {
                    la.advance();
                    lb.advance();
                }
            }
            slot = next;
        }
        if constexpr (APART) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] += low[i][j];
        }
        for (s = n < 1 ? 1 : n; s < most; ++s) __builtin_amdgcn_s_barrier();   // (a group with fewer stages)
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
        const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) % NW / WN;
        return wm * TM * 32 + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    }
    static __device__ __forceinline__ int wave_row() { return (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW / WN) * TM * 32; }
    static __device__ __forceinline__ int wave_col() { return (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WN) * TN * 32; }
    static __device__ __forceinline__ int bcol(int j) {
        const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % WN;
        return wn * TN * 32 + j * 32 + (lane & 31);
    }
};

// The wave's tile as 16-bit values, 16 bytes a lane, through a region of LDS that only this wave uses (after MmTile::run): an
// accumulator's lanes run along B and its registers along A, so stores straight from it would be 2 bytes a lane (along B) or 8
// bytes to 32 different rows (along A).
//   store_rows: rows of A's index, B's index fastest;  dst(row, first column, plane, 8 values), row and column of the wave's tile
//   store_cols: rows of B's index, A's index fastest;  dst(column, first row, plane, 8 values)
// val(i, j, e, plane) is the value of an accumulator.
template <class M> struct WaveStore {
    static constexpr int SI = M::TM % 2 == 0 ? 2 : 1;                     // 32-row blocks that store_cols takes at a time
    static constexpr int PC = SI * 64 + 16, PR = M::TN * 64 + 16;         // bytes of a row in LDS; the pad spreads the banks
    static constexpr int BYTES = M::TN * 32 * PC > 32 * PR ? M::TN * 32 * PC : 32 * PR;
    static_assert(M::NW * BYTES <= M::LDS, "the regions of all waves fit the tile's LDS");

    static __device__ __forceinline__ char* region(char* lds) { return lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * BYTES; }
    static __device__ __forceinline__ void fence() {   // the sched_barrier keeps the next strip's conversions out of this one's registers
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    template <int PLANES, typename VAL, typename DST> static __device__ __forceinline__ void store_rows(char* reg, VAL val, DST dst) {
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < M::TM; ++i)
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
#pragma unroll
                    for (int j = 0; j < M::TN; ++j)
                        *reinterpret_cast<uint16_t*>(reg + (8 * (e >> 2) + 4 * h + (e & 3)) * PR + (j * 32 + r) * 2) = val(i, j, e, p);
                fence();
#pragma unroll
                for (int q = 0; q < M::TN * 2; ++q) {
                    const int at = q * 64 + lane, row = at / (M::TN * 4), c = at % (M::TN * 4);
                    dst(i * 32 + row, c * 8, p, *reinterpret_cast<const u32x4*>(reg + row * PR + c * 16));
                }
                fence();
            }
    }
    template <int PLANES, typename VAL, typename DST> static __device__ __forceinline__ void store_cols(char* reg, VAL val, DST dst) {
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i0 = 0; i0 < M::TM; i0 += SI)
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
#pragma unroll
                for (int i = 0; i < SI; ++i)
#pragma unroll
                    for (int j = 0; j < M::TN; ++j)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            u32x2 v;
                            v[0] = (unsigned)val(i0 + i, j, 4 * g, p) | (unsigned)val(i0 + i, j, 4 * g + 1, p) << 16;
                            v[1] = (unsigned)val(i0 + i, j, 4 * g + 2, p) | (unsigned)val(i0 + i, j, 4 * g + 3, p) << 16;
                            *reinterpret_cast<u32x2*>(reg + (j * 32 + r) * PC + (i * 32 + 8 * g + 4 * h) * 2) = v;
                        }
                fence();
#pragma unroll
                for (int q = 0; q < M::TN * 2 * SI; ++q) {
                    const int at = q * 64 + lane, row = at / (SI * 4), c = at % (SI * 4);
                    dst(row, i0 * 32 + c * 8, p, *reinterpret_cast<const u32x4*>(reg + row * PC + c * 16));
                }
                fence();
            }
    }
};

// The time of a launch in microseconds, to choose a tile side by.  One stage of one workgroup takes `alone` us where it has the chip to
// itself and `full` us where the chip is full (two workgroups a CU up to 128), measured on products of 4096 x 4096 x 4096 (full:
// 120 / 155 / 200 us with one plane, 308 / 344 / 466 us with two, for sides of 256 / 128 / 64; a triangle of 192: 204) and 512 x 1536
// x 512 (alone; 128 with two planes, whose operands leave the L2 first: 2000 x 6000); between them it grows with the workgroups.  Three
// planes are timed as six stages of one: the side chosen so is within 3 % of the best of the three at eight shapes from 126 x 512 x 1000
// to 8192 x 512 x 16384.
struct MmWork {
    int64_t tiles = 0, stages = 0, longest = 0;      // workgroups, their stages together, the most stages of one
    void add(int64_t n, int64_t per) {
        tiles += n;
        stages += n * per;
        longest = longest < per ? per : longest;
    }
};
// groups: two groups of waves take a tile's stages in pairs (one workgroup a CU): a pair takes 1.25 us at a side of 128 with two
// planes and 0.42 us at 64 (ResNet18's matrices, A = X X^T over 240 tiles of 64 and 48 stages: 16 us against 21), and 1.45 times that
// where the tiles take more than one round (the iteration at 3000 x 3500: 2471 us by pairs, 2345 without, 2176 at a side of 128).
inline double mm_time(int side, int planes, const MmWork& w, int groups = 1) {
    const bool two = planes == 2;
    const double full = side == 256 ? (two ? 2.4 : 1.87) : side == 192 ? (two ? 1.65 : 1.3) : side == 128 ? (two ? 1.34 : 1.2) : (two ? 0.46 : 0.39);
    const double alone = side == 256 ? (two ? 1.9 : 1.5) : side == 192 ? (two ? 1.2 : 0.9) : side == 128 ? (two ? 0.9 : 0.6) : 0.3;
    const double pair = side == 128 ? (two ? 1.25 : 1.1) : (two ? 0.42 : 0.36);
    const int64_t slots = side > 128 || groups == 2 ? 256 : 512;
    const double rounds = (double)((w.tiles + slots - 1) / slots), mean = w.tiles ? (double)w.stages / (double)w.tiles : 0.0;
    if (groups == 2) return 4.0 + (rounds <= 1.0 ? (w.longest + 1) / 2 * pair : rounds * (mean * 0.5 * 1.45 * pair + 1.0));
    if (rounds <= 1.0) return 3.0 + w.longest * (alone + (full - alone) * (double)w.tiles / (double)slots);
    const double busy = rounds * mean * full, chain = w.longest * alone;
    return 3.0 + (busy > chain ? busy : chain);
}

// Consecutive workgroups run on different XCDs (8, round robin), each with an L2 of its own: give every XCD a contiguous range of
// tiles, so that neighbours share operand rows in one L2.  A permutation of [0, n).
__device__ __forceinline__ int xcd_tile(int bid, int n) {
    const int q = n >> 3, rem = n & 7, x = bid & 7, i = bid >> 3;
    return x * q + (x < rem ? x : rem) + i;
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

// both planes of v + rest, |rest| a few units of v's last place (hi in the lower half)
__device__ __forceinline__ uint32_t planes16(float v, float rest) {
    const _Float16 hi = (_Float16)v;
    const float f = (float)hi;
    return (uint32_t)bits16(hi) | (__builtin_isinf(f) ? 0u : (uint32_t)bits16((_Float16)((v - f) + rest)) << 16);
}

// v as three bf16 values that add up to it.  What rounds to infinity is cut off instead; infinities and NaN are in the first alone.
__device__ __forceinline__ void split3(float v, uint16_t (&q)[3]) {
    const __bf16 r = (__bf16)v;
    const bool finite = fabsf(v) < INFINITY;
    q[0] = finite && __builtin_isinf((float)r) ? (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16) : bits16(r);
    const float d = finite ? v - __builtin_bit_cast(float, (uint32_t)q[0] << 16) : 0.f;   // exact: at most 16 bits are left
    const __bf16 r1 = (__bf16)d;
    q[1] = bits16(r1);
    q[2] = bits16((__bf16)(d - (float)r1));                                               // exact: at most 8
}

}  // namespace ssecg_lm
