// product_core.hpp — the matrix-core mainloop of the operators that take 16-bit and 32-bit elements
// (grouped products, cross entropy).
//
//   D[m, n] = sum_k A[m, k] * B[k, n],   A and B of one type (bfloat16, half or float), sums in float.
//
// A workgroup owns a BM x BN tile, its WM x WN waves a (BM/WM) x (BN/WN) part each, made of 16 x 16
// accumulator tiles.  Reduction is walked in stages of 64 bytes of k per row (32 elements of 16 bits, 16
// floats): one stage is one v_mfma_f32_16x16x32 per accumulator tile (four v_mfma_f32_16x16x4 for floats).
//
// Feeding the matrix cores:
//   * global -> LDS without registers (buffer loads with the `lds` modifier, 16 bytes per lane).  S buffers
//     are filled in turn; S - 1 stages are in flight, so a stage may take S - 2 stage times to arrive.
//     Out-of-range lanes read zero by the buffer descriptor's bounds: rows behind a tile, the k past the end
//     and whole stages past the end need no other code.
//   * LDS -> registers one stage ahead: while the MFMAs of stage t run, the operands of stage t + 1 are read.
//     A wave therefore never waits for LDS between a barrier and its first MFMA, and there is one barrier per
//     stage.
//
// The first MFMA operand is B, so an accumulator lane holds one row m and, per tile, four consecutive n.  The columns of
// a wave's NT accumulator tiles are interleaved by eights: column of (tile j, operand row i) = 8 NT (i / 8) + 8 j + i % 8.
// Lanes l and l + 16 then hold the halves of 16-byte chunks of 16-bit elements, and a transposing read takes whole chunks.
//
// An operand lies in memory in one of two ways:
//   KMAJOR  k is contiguous (the rows of A; B stored transposed).  LDS tile: [row][64 bytes].
//   KROWS   k is the row index, m or n contiguous (A stored transposed; B as a plain matrix).  LDS tile:
//           [k][BM or BN elements].  16-bit elements are gathered by the transposing LDS read (ds_read_b64_tr_b16:
//           sixteen lanes read 4 k x 16 columns and get 4 k of one column each), floats by 32-bit reads.
// The 16-byte chunks of a tile row are permuted by XOR with a key of the row, chosen so that the lanes that an LDS
// read serves together (256 bytes a cycle: lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of each half wave for 128-bit
// reads, half waves for the 64-bit transposing ones; measured with pairs of lanes on one bank) never meet on a bank;
// the LDS side of a direct load is fixed (lane x 16 bytes), so the permutation is applied to the lanes' global addresses.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace t2sp {

typedef float pv4f __attribute__((ext_vector_type(4)));
typedef uint32_t pv4u __attribute__((ext_vector_type(4)));
typedef short pv4s __attribute__((ext_vector_type(4)));

enum : int { KMAJOR = 0, KROWS = 1 };

// 16 bytes of elements, and the same for an address that is aligned to an element only.
template <class O> struct Chunk {
    typedef O type __attribute__((ext_vector_type(16 / sizeof(O))));
    typedef O anywhere __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
};

template <class T> struct MatrixOp;
template <> struct MatrixOp<__bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ pv4f mul(pv4u a, pv4u b, pv4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
template <> struct MatrixOp<_Float16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ pv4f mul(pv4u a, pv4u b, pv4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
template <> struct MatrixOp<float> {
    static __device__ __forceinline__ pv4f mul(pv4u a, pv4u b, pv4f c) {
        const pv4f x = __builtin_bit_cast(pv4f, a), y = __builtin_bit_cast(pv4f, b);
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};

// What a tile reads of one operand: `p` its first element, `ld` bytes between rows (KMAJOR: of the tile; KROWS: of k),
// `count` rows of the tile that exist (KMAJOR) or elements from the tile's first column to the end of a row (KROWS);
// either may exceed the tile.  p, ld and, where elements are contiguous along it, the extent are whole 16-byte chunks,
// and 255 * ld < 2^31.  Nothing outside these rows, columns and the k_len of the product is read.
struct TileSource {
    const char *p;
    uint32_t ld;
    int count;
};

constexpr uint32_t OUT_OF_RANGE = 0x80000000u;      // a lane offset that the descriptors (2^31 - 1 bytes from the tile) do not cover

// 16 bytes per lane from `rsrc` + off to LDS at lds_base + lane * 16.  Not counted by the compiler: the caller
// waits with wait_loads().  (The m0 write needs one instruction between itself and the load.)
__device__ __forceinline__ void load_to_lds(pv4u rsrc, uint32_t off, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(off), "s"(rsrc), "s"(lds_base) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// s_barrier, with nothing moved across it by the compiler (the builtin alone says nothing about memory).
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ pv4u descriptor(const char *p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return pv4u{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
}

template <class T_, int BM_, int BN_, int WM_, int WN_, int AS_, int BS_, int S_>
struct ProductTile {
    using T = T_;
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, AS = AS_, BS = BS_, S = S_;
    static constexpr int NW = WM * WN, THREADS = NW * 64;
    static constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 16, NT = TN / 16;
    static constexpr int SZ = sizeof(T), KS = 64 / SZ, EPC = 16 / SZ;      // elements of k per stage, per chunk
    static constexpr int A_BYTES = BM * 64, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES, LDS = S * STAGE;
    static constexpr int A_LOADS = BM / 16 >= NW ? BM / 16 / NW : 1, B_LOADS = BN / 16 / NW;
    static constexpr int LOADS = A_LOADS + B_LOADS;                         // per wave and stage
    static constexpr bool TURNS = SZ == 2 && NW == 8 && AS == KMAJOR;        // see product_run
    static constexpr int A_READS = MT * (AS == KMAJOR ? 1 : SZ == 2 ? 2 : 4), B_READS = NT * (BS == KMAJOR ? 1 : SZ == 2 ? 2 : 4);
    static constexpr int LANE_N = 4 * NT;                                   // columns a lane ends up with, per row
    static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "whole accumulator tiles");
    static_assert(A_LOADS * NW * 16 == BM || (A_LOADS == 1 && NW % (BM / 16) == 0), "the waves share A's loads evenly");
    static_assert(B_LOADS >= 1 && B_LOADS * NW * 16 == BN, "the waves share B's loads evenly");
    static_assert(AS == KMAJOR || BM * SZ >= 256, "a KROWS tile row holds at least the sixteen chunks a key permutes");
    static_assert(BS == KMAJOR || BN * SZ >= 256, "a KROWS tile row holds at least the sixteen chunks a key permutes");
    static_assert(NT == 2 || NT == 4, "the B keys below are worked out for these");
    static_assert(SZ == 2 || MT * NT <= 16, "floats keep two sets of sums in registers");
    static_assert(S >= 3 && (S - 1) * LOADS < 63, "the wait counter has six bits");

    // Column of B's operand row i in accumulator tile 0 (tile j: + 8 j).
    static __device__ __forceinline__ int column(int i) { return 8 * NT * (i >> 3) + (i & 7); }
    // First of the four columns that a lane holds of accumulator tile 0.
    static __device__ __forceinline__ int lane_column(int lane) { return column(4 * (lane >> 4)); }

    // key of a KMAJOR row.  A read touches operand rows i = 0..15, whose rows of 64 bytes lie i % 4 quarters of 256 bytes
    // apart; of the four i / 4 = q, two come with one k chunk and two (1 and 2, or 0 and 3) with its neighbour, and the
    // keys 0, 3, 2, 1 send all four to different chunk positions.
    static __device__ __forceinline__ int key_kmajor(bool b, int r) {
        const int q = b ? ((r >> 2) & 1) | ((r / (8 * NT)) & 1) << 1 : (r >> 2) & 3;
        return (4 - q) & 3;
    }
    // key of a KROWS row.  16-bit: half a wave reads two chunks of each of eight k rows (k % 4 and k / 8 % 2), A: neighbours,
    // B: NT apart.  float: sixteen lanes read four chunks of one k row, the four sixteens of k rows 4 apart, A: neighbours, B:
    // two neighbours twice, 2 NT apart.  The keys use the bits of the chunk's position that the row's own chunks leave free.
    static __device__ __forceinline__ int key_krows(bool b, int k) {
        if (SZ == 2) {
            const int lo = k & 3, hi = (k >> 3) & 1;
            if (!b) return (lo | hi << 2) << 1;
            return NT == 4 ? lo | hi << 3 : (lo & 1) | (lo >> 1) << 2 | hi << 3;
        }
        const int q = (k >> 2) & 3;
        if (!b) return q << 2;
        return NT == 4 ? q << 1 : (q & 1) << 1 | (q >> 1) << 3;
    }

    // Byte offset (from the tile's first element) that lane `lane` fetches in wave-load `i` of a stage, OUT_OF_RANGE
    // where that row or column does not exist; sets the k of the chunk's first element within the stage.
    template <bool IS_B>
    static __device__ __forceinline__ uint32_t lane_source(int i, int lane, const TileSource &s, int *k_of) {
        constexpr int STYLE = IS_B ? BS : AS, ROWS = IS_B ? BN : BM;
        if (STYLE == KMAJOR) {
            const int r = i * 16 + (lane >> 2), c = (lane & 3) ^ key_kmajor(IS_B, r);
            *k_of = c * EPC;
            return r < s.count ? (uint32_t)r * s.ld + c * 16 : OUT_OF_RANGE;
        }
        constexpr int CPR = ROWS * SZ / 16;                                 // chunks per k row
        const int f = i * 64 + lane, k = f / CPR, c = (f % CPR) ^ key_krows(IS_B, k);
        *k_of = k;
        return c * EPC < s.count ? (uint32_t)k * s.ld + c * 16 : OUT_OF_RANGE;
    }

    struct Frags {
        pv4u a[MT], b[NT];
    };

    // One operand's fragments of the stage in LDS at `t`: for tile i the lane holds the 16 bytes of k that belong
    // to lane / 16, of row (or column) lane % 16 of the tile.
    template <bool IS_B, int COUNT>
    static __device__ __forceinline__ void read(const char *t, int first, int lane, pv4u (&out)[COUNT]) {
        constexpr int STYLE = IS_B ? BS : AS, ROWS = IS_B ? BN : BM;
        const int r = lane & 15, kg = lane >> 4;
        if (STYLE == KMAJOR) {
            const int row = first + (IS_B ? column(r) : r);
            const char *p = t + row * 64 + ((kg ^ key_kmajor(IS_B, row)) << 4);
#pragma unroll
            for (int i = 0; i < COUNT; i++) out[i] = *reinterpret_cast<const pv4u *>(p + i * (IS_B ? 8 * 64 : 16 * 64));
        } else if (SZ == 2) {
            constexpr int PITCH = ROWS * 2;
            typedef __attribute__((address_space(3))) pv4s lds_v4s;
            const int k = kg * 8 + (r >> 2), q = r & 3, key = key_krows(IS_B, k);
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                const int col = first + (IS_B ? column(4 * q) + 8 * i : 16 * i + 4 * q);
                const char *p = t + k * PITCH + (((col >> 3) ^ key) << 4) + ((col >> 2) & 1) * 8;
                const pv4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)p);
                const pv4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 4 * PITCH));   // (same key)
                typedef uint32_t v2u __attribute__((ext_vector_type(2)));
                const v2u l = __builtin_bit_cast(v2u, lo), h = __builtin_bit_cast(v2u, hi);
                out[i] = pv4u{l[0], l[1], h[0], h[1]};
            }
        } else {
            constexpr int PITCH = ROWS * 4;
            const int k = kg * 4, key = key_krows(IS_B, k);
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                const int col = first + (IS_B ? column(r) + 8 * i : 16 * i + r);
                const char *p = t + k * PITCH + (((col >> 2) ^ key) << 4) + (col & 3) * 4;
#pragma unroll
                for (int j = 0; j < 4; j++) out[i][j] = *reinterpret_cast<const uint32_t *>(p + j * PITCH);   // (same key)
            }
        }
    }
};

// acc[i][j] += the tile's product over k_len elements.  Every wave of the workgroup takes part; `smem` holds P::LDS
// bytes.  On return no load is outstanding and every wave has passed a barrier after its last LDS read.
template <class P>
__device__ __forceinline__ void product_run(const TileSource &A, const TileSource &B, int k_len, char *smem,
                                            pv4f (&acc)[P::MT][P::NT]) {
    using T = typename P::T;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first_m = (wave / P::WN) * P::TM, first_n = (wave % P::WN) * P::TN;
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem);

    uint32_t offA[P::A_LOADS], offB[P::B_LOADS];
    int kA[P::A_LOADS], kB[P::B_LOADS];
    uint32_t dstA[P::A_LOADS], dstB[P::B_LOADS];
#pragma unroll
    for (int i = 0; i < P::A_LOADS; i++) {
        const int w = P::BM / 16 >= P::NW ? i * P::NW + wave : wave % (P::BM / 16);     // (spare waves repeat a load)
        offA[i] = P::template lane_source<false>(w, lane, A, &kA[i]);
        dstA[i] = w * 1024;
    }
#pragma unroll
    for (int i = 0; i < P::B_LOADS; i++) {
        const int w = i * P::NW + wave;
        offB[i] = P::template lane_source<true>(w, lane, B, &kB[i]);
        dstB[i] = P::A_BYTES + w * 1024;
    }
    const int64_t stepA = P::AS == KMAJOR ? 64 : (int64_t)P::KS * A.ld, stepB = P::BS == KMAJOR ? 64 : (int64_t)P::KS * B.ld;
    const char *pa = A.p, *pb = B.p;
    int k_left = k_len;                              // elements of k from the next stage to load on
    uint32_t buf = lds0;
    auto issue = [&]() {
        if (k_left < P::KS) {                        // the last, partial stage and the empty ones behind it
#pragma unroll
            for (int i = 0; i < P::A_LOADS; i++) offA[i] = kA[i] >= k_left ? OUT_OF_RANGE : offA[i];
#pragma unroll
            for (int i = 0; i < P::B_LOADS; i++) offB[i] = kB[i] >= k_left ? OUT_OF_RANGE : offB[i];
        }
        const pv4u ra = descriptor(pa), rb = descriptor(pb);
#pragma unroll
        for (int i = 0; i < P::A_LOADS; i++) load_to_lds(ra, offA[i], buf + dstA[i]);
#pragma unroll
        for (int i = 0; i < P::B_LOADS; i++) load_to_lds(rb, offB[i], buf + dstB[i]);
        pa += stepA; pb += stepB; k_left -= P::KS;
        buf = buf + P::STAGE == lds0 + P::LDS ? lds0 : buf + P::STAGE;
    };
    const char *rd = smem;
    auto fetch = [&](typename P::Frags &f) {
        P::template read<false>(rd, first_m, lane, f.a);
        P::template read<true>(rd + P::A_BYTES, first_n, lane, f.b);
        rd = rd + P::STAGE == smem + P::LDS ? smem : rd + P::STAGE;
    };
    auto multiply = [&](const typename P::Frags &f) {
#pragma unroll
        for (int j = 0; j < P::NT; j++)
#pragma unroll
            for (int i = 0; i < P::MT; i++) acc[i][j] = MatrixOp<T>::mul(f.b[j], f.a[i], acc[i][j]);
    };
    // (left alone, the compiler moves the reads behind the MFMAs, next to their use, to save registers)
    auto fetch_and_multiply = [&](typename P::Frags &next, const typename P::Frags &now) {
        __builtin_amdgcn_sched_barrier(0);
        fetch(next);
        multiply(now);
        constexpr int READS = P::A_READS + P::B_READS, MULS = P::MT * P::NT * (P::SZ == 4 ? 4 : 1);
        constexpr int EACH = MULS / READS > 1 ? MULS / READS : 1;
#pragma unroll
        for (int r = 0; r < READS; r++) {
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);     // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);        // LDS read
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    const int stages = (k_len + P::KS - 1) / P::KS;
    if constexpr (P::TURNS) {
        // Two waves share a SIMD, one of each half of the workgroup, and take turns: while one multiplies (its 32 MFMAs
        // fill the SIMD's matrix unit for 512 cycles), the other reads its operands of the next stage from LDS and sends the loads
        // of a later one.  A barrier ends every turn, the second half of the waves runs one turn behind.  With both waves in step
        // the matrix units were idle a third of the time, around the barriers (8192 x 8192 x 4096, B's rows contiguous, on zeros: 1.73
        // PFLOP/s in step, 1.98 in turns; on random data the clock falls with the power drawn, to 2.0 of 2.4 GHz: 1.32 and 1.37).
        // A KROWS A has twice as many LDS reads, which do not fit a turn: such products keep the loop below (1.26 in turns, 1.32).
        // Stage t is read in the turns 2 t and 2 t + 1 and must have landed before them; its buffer is free in turn 2 t + 2,
        // where the loads of stage t + S are first sent.  A wave sees to its own loads of stage t + 1 at the end of its turn with t.
        const bool behind = wave >= P::NW / 2;
#pragma unroll
        for (int s = 0; s < P::S - 1; s++) issue();
        wait_loads<(P::S - 2) * P::LOADS>();
        meet();
        if (behind) meet();
        typename P::Frags f;
        for (int t = 0; t < stages; t++) {
            __builtin_amdgcn_sched_barrier(0);
            fetch(f);
            issue();
            wait_loads<(P::S - 2) * P::LOADS>();
            wait_lds_reads();
            meet();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply(f);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            meet();
        }
        if (!behind) meet();
        wait_loads<0>();
        meet();
        return;
    }
#pragma unroll
    for (int s = 0; s < P::S; s++) issue();
    wait_loads<(P::S - 1) * P::LOADS>();
    meet();
    typename P::Frags f0, f1;
    fetch(f0);
    // Sums of floats are taken in runs of RUN stages (256 elements of k) that are added up on the vector units: the error of
    // one running sum over k grows with sqrt(k), that of two levels with sqrt(256 + k / 256) (8192 of k: 1.0e-6 -> 3e-7
    // of the result's norm).  Results of 16-bit operands are rounded far above that.
    constexpr int RUN = 16;
    constexpr bool TWO_LEVELS = P::SZ == 4;
    pv4f whole[TWO_LEVELS ? P::MT : 1][TWO_LEVELS ? P::NT : 1];
    if constexpr (TWO_LEVELS)
#pragma unroll
        for (int i = 0; i < P::MT; i++)
#pragma unroll
            for (int j = 0; j < P::NT; j++) whole[i][j] = pv4f{0.f, 0.f, 0.f, 0.f};
    for (int t = 0; t < stages; t += 2) {            // (an odd number of stages ends with one of zeros)
        if constexpr (TWO_LEVELS)
            if (t % RUN == 0)
#pragma unroll
                for (int i = 0; i < P::MT; i++)
#pragma unroll
                    for (int j = 0; j < P::NT; j++) {
                        whole[i][j] += acc[i][j];
                        acc[i][j] = pv4f{0.f, 0.f, 0.f, 0.f};
                    }
        wait_loads<(P::S - 2) * P::LOADS>();          // stage t + 1 has landed
        wait_lds_reads();                             // this wave's operands of stage t are in registers:
        meet();                 // its buffer may be overwritten
        issue();
        fetch_and_multiply(f1, f0);
        wait_loads<(P::S - 2) * P::LOADS>();
        wait_lds_reads();
        meet();
        issue();
        fetch_and_multiply(f0, f1);
    }
    if constexpr (TWO_LEVELS)
#pragma unroll
        for (int i = 0; i < P::MT; i++)
#pragma unroll
            for (int j = 0; j < P::NT; j++) acc[i][j] += whole[i][j];
    wait_loads<0>();
    wait_lds_reads();
    meet();
}

// The position that workgroup `block` of `total` takes when every die works on a contiguous run of positions (workgroup
// ids are dealt to the dies in turn): neighbouring tiles share operands, and each die has an L2 of its own.
__device__ __forceinline__ unsigned die_run(unsigned block, unsigned total, unsigned dies) {
    const unsigned whole = total / dies, extra = total % dies, die = block % dies;
    return die * whole + (die < extra ? die : extra) + block / dies;
}

// Tile `at` of a row_tiles x col_tiles grid, walked in panels of eight rows of tiles, down the rows first: a die's 32
// tiles in flight are then 8 x 4, which read the least (12 panels of operands) among the shapes that cover 32.
__device__ __forceinline__ void panel_tile(int64_t at, int row_tiles, int col_tiles, int *row, int *col) {
    constexpr int PANEL = 8;
    const int panel = (int)(at / ((int64_t)PANEL * col_tiles)), rest = (int)(at % ((int64_t)PANEL * col_tiles));
    const int high = row_tiles - panel * PANEL < PANEL ? row_tiles - panel * PANEL : PANEL;
    *row = panel * PANEL + rest % high;
    *col = rest / high;
}

// x = {x0, x1, y0, y1}, y = {x2, x3, y2, y3}, indices counting the lanes' sixteens (permlane16_swap, used below, gives
// x = {x0, y0, x2, y2}, y = {x1, y1, x3, y3}).
__device__ __forceinline__ void swap_sixteens(pv4u &x, pv4u &y) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const auto r = __builtin_amdgcn_permlane32_swap(x[i], y[i], false, false);
        x[i] = r[0];
        y[i] = r[1];
    }
}

// Calls f(column, 16 bytes of the row from that column on, rounded to O) for a lane's share of row lane % 16 of
// accumulator row i, whose first column of the wave is n.  The four lanes of a row exchange parts first, such that one
// store (or load) of the wave covers 64 consecutive bytes of each row: chunks 64 bytes apart cost a memory request
// each (268 MB of float results of an 8192 x 8192 x 4096 product: 695 us stored so, 491 us exchanged).
template <class P, class O, class F>
__device__ __forceinline__ void row_chunks(int n, const pv4f (&acc)[P::NT], F f) {
    constexpr int CE = 16 / sizeof(O), C = P::LANE_N / CE;
    typedef typename Chunk<O>::type chunk;
    pv4u v[C];
    const int kg = (threadIdx.x >> 4) & 3;
    if constexpr (sizeof(O) == 4) {                  // v[j]: chunks 2 j, 2 j + 1, 2 NT + 2 j, 2 NT + 2 j + 1 in the sixteens
#pragma unroll
        for (int j = 0; j < P::NT; j++) v[j] = __builtin_bit_cast(pv4u, acc[j]);
#pragma unroll
        for (int j = 0; j < P::NT; j += 2) swap_sixteens(v[j], v[j + 1]);        // four neighbours each
#pragma unroll
        for (int j = 0; j < P::NT; j++) f(n + ((j & 1) * 2 * P::NT + (j >> 1) * 4 + kg) * CE, __builtin_bit_cast(chunk, v[j]));
    } else {                                         // halves of chunks j and j + 1 -> whole chunks j, j + 1, NT + j, NT + j + 1
        typedef O half_chunk __attribute__((ext_vector_type(4)));
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < P::NT; j += 2) {
            v2u x = __builtin_bit_cast(v2u, __builtin_convertvector(acc[j], half_chunk)),
                y = __builtin_bit_cast(v2u, __builtin_convertvector(acc[j + 1], half_chunk));
            const auto a = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false), b = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
            v[j / 2] = pv4u{a[0], b[0], a[1], b[1]};
        }
        if constexpr (C == 2) swap_sixteens(v[0], v[1]);
        static_assert(C <= 2, "four accumulator tiles");
#pragma unroll
        for (int c = 0; c < C; c++) f(n + (c * 4 + kg) * CE, __builtin_bit_cast(chunk, v[c]));
    }
}

// CE elements to p: one 16-byte store (memory takes it at any element's alignment), or those below n_end one by one.
template <class O>
__device__ __forceinline__ void store_chunk(O *p, int col, int n_end, typename Chunk<O>::type v) {
    constexpr int CE = 16 / sizeof(O);
    if (col + CE <= n_end) {
        *reinterpret_cast<typename Chunk<O>::anywhere *>(p + col) = v;
    } else {
#pragma unroll
        for (int i = 0; i < CE; i++)
            if (col + i < n_end) p[col + i] = v[i];
    }
}

// Row lane % 16 of accumulator row i to memory, columns below n_end, rounded to the output's type; `row` is the row's first
// element, n the wave's first column.
template <class P, class O>
__device__ __forceinline__ void store_row(char *row, int n, int n_end, const pv4f (&acc)[P::NT]) {
    row_chunks<P, O>(n, acc, [&](int col, typename Chunk<O>::type v) { store_chunk<O>(reinterpret_cast<O *>(row), col, n_end, v); });
}

template <class P>
__device__ __forceinline__ void clear(pv4f (&acc)[P::MT][P::NT]) {
#pragma unroll
    for (int i = 0; i < P::MT; i++)
#pragma unroll
        for (int j = 0; j < P::NT; j++) acc[i][j] = pv4f{0.f, 0.f, 0.f, 0.f};
}


// Tile shapes.  256 x 256 (16-bit) has the most arithmetic per byte from LDS and one workgroup per CU, whose 160 KB hold
// five stages (8192 x 8192 x 2048, bfloat16, both operands k-contiguous: 282 us with four stages, 235 with five); the
// smaller ones fill the chip when there are few rows or columns.  Floats, whose MFMAs are long, take two waves per SIMD
// instead of large wave tiles (128 x 128 x 1024 alone on a CU: 77 us with four waves, 70 with eight), and a 64 x 64 tile.
template <class T, int AS, int BS> using Tile256 = ProductTile<T, 256, 256, 2, 4, AS, BS, 5>;
template <class T, int AS, int BS> using Tile128 = ProductTile<T, 128, 128, 2, sizeof(T) == 2 ? 2 : 4, AS, BS, 5>;
template <class T, int BS> using Tile64 = ProductTile<T, 64, sizeof(T) == 2 ? 128 : 64, sizeof(T) == 2 ? 1 : 2, sizeof(T) == 2 ? 4 : 2, KMAJOR, BS, sizeof(T) == 2 ? 4 : 6>;

}  // namespace t2sp
