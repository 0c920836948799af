// grouped.hip — matrix products grouped by expert, with ragged group sizes.
//
//   forward   Y[r, :]  = X[r, :] * op(W[e])          for the rows offsets[e] <= r < offsets[e + 1] of group e
//   wgrad     dW[e]    = X_e^T * dY_e                (the rows of group e; zeros for an empty group)
//
// op(W[e]) is K x N, stored so or (opb) as N x K; the gradient of the rows is the forward product of dY with the other
// op.  The group sizes are on the device only, so the launch covers the largest number of row tiles they can make,
//   sum_e ceil(m_e / BM) <= floor(T / BM) + min(E, T),
// and every workgroup finds its group and tile by itself: the waves add up the tile counts of 64 groups at a time
// (a scan over the lanes); workgroups beyond the actual number end at once.  The tiles are then dealt to the dies in
// contiguous runs, since each die has an L2 of its own: neighbouring tiles read the same columns of one matrix.
//
// Offsets are clamped to 0 .. T and replaced by their running maximum before use: no value of theirs leads outside X or Y,
// no row belongs to two groups, and the tiles are never more than the launch covers.
#include "product_core.hpp"
#include "product_host.hpp"

#include <algorithm>
#include <cmath>

namespace t2sp {

struct GroupedArgs {
    const char *X, *W;
    char *Y;
    const void *offsets;
    int off64;                           // the offsets are 64-bit (else 32-bit) integers
    int T, E, K, N;
    int64_t ldx, ldw, sw, ldy;           // in elements; sw: between matrices
    int col_tiles, xcds;
    int die_cus;                         // CUs of a die
    int parts;                           // gradient of the matrices: parts of every group's rows, each with a plane of floats
    int64_t plane;
};

__device__ __forceinline__ int group_edge(const GroupedArgs &g, int e) {
    const int64_t v = g.off64 ? static_cast<const int64_t *>(g.offsets)[e] : (int64_t) static_cast<const int32_t *>(g.offsets)[e];
    return (int)(v < 0 ? 0 : v > g.T ? g.T : v);
}

struct GroupTile {
    int group, row0, rows, col_tile;     // rows: of the group from row0 on
    bool half;                           // only the first BM / 2 of them
};

// The output tile of workgroup `block`, false when there is none.  Every wave does the same work; the results are
// uniform over the wave.  HALVES: when the tiles that are left for a die's last round of workgroups would fill at most half of
// its CUs, each of them goes to two workgroups, by halves of its rows.
template <int BM, bool HALVES = false>
__device__ __forceinline__ bool find_tile(const GroupedArgs &g, unsigned block, GroupTile *out) {
    const int lane = threadIdx.x & 63;
    // The rows and tiles of group e0 + lane; `high` is the largest offset of the groups in front of e0, then of those behind.
    auto tiles_of = [&](int e0, int *high, int *start, int *rows) {
        int a = *high, b = a;
        if (e0 + lane < g.E) { a = group_edge(g, e0 + lane); b = group_edge(g, e0 + lane + 1); }
        if (__ballot(b < a || a < *high)) {              // (offsets that decrease, which a caller does not mean to pass)
            const int front = max(*high, __builtin_amdgcn_readlane(a, 0));
            b = max(b, front);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(b, d, 64);
                if (lane >= d) b = max(b, o);
            }
            a = __shfl_up(b, 1, 64);
            if (lane == 0) a = front;
        }
        *high = __builtin_amdgcn_readlane(b, 63);        // (used if there are groups behind these 64)
        *start = a;
        *rows = b - a;
        return (b - a + BM - 1) / BM;
    };
    auto scan = [&](int v) {                         // inclusive prefix sum over the wave
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(v, d, 64);
            if (lane >= d) v += o;
        }
        return v;
    };
    int high = 0, start, rows, n = tiles_of(0, &high, &start, &rows), sum = scan(n), high0 = high;
    int64_t total = __builtin_amdgcn_readlane(sum, 63);
    for (int e0 = 64; e0 < g.E; e0 += 64) {
        int s, r;
        total += __builtin_amdgcn_readlane(scan(tiles_of(e0, &high, &s, &r)), 63);
    }
    total *= g.col_tiles;
    const int64_t run = (total + g.xcds - 1) / g.xcds;
    const int64_t first = (block % g.xcds) * run;
    int64_t at = block / g.xcds;
    int half = -1;
    if (HALVES) {
        const int64_t mine = total - first < run ? total - first : run, whole = mine > 0 ? mine / g.die_cus * g.die_cus : 0;
        if (at >= whole && 2 * (mine - whole) <= g.die_cus) {
            half = (int)((at - whole) & 1);
            at = whole + (at - whole) / 2;
        }
    }
    const int64_t w = first + at;
    if (at >= run || w >= total) return false;
    int64_t before = 0;                              // tiles of the groups in front of this chunk of 64
    for (int e0 = 0; e0 < g.E;) {
        const int64_t end = (before + sum) * g.col_tiles;
        const uint64_t past = __ballot(end > w);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int mine = __builtin_amdgcn_readlane(n, l);
            const int64_t local = w - (before + __builtin_amdgcn_readlane(sum, l) - mine) * g.col_tiles;
            int m;
            panel_tile(local, mine, g.col_tiles, &m, &out->col_tile);
            out->group = e0 + l;
            out->row0 = __builtin_amdgcn_readlane(start, l) + m * BM;
            out->rows = __builtin_amdgcn_readlane(rows, l) - m * BM;
            out->half = half >= 0;
            if (half > 0) {
                out->row0 += BM / 2;
                out->rows -= BM / 2;
            }
            return out->rows > 0;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        e0 += 64;
        n = tiles_of(e0, &high0, &start, &rows);
        sum = scan(n);
    }
    return false;
}

template <class P, class O>
__device__ __forceinline__ void grouped_tile(const GroupedArgs &g, const GroupTile &t, int n0, char *smem) {
    const int have = t.half && t.rows > P::BM ? P::BM : t.rows;
    TileSource a, b;
    a.p = g.X + t.row0 * g.ldx * P::SZ;
    a.ld = (uint32_t)(g.ldx * P::SZ);
    a.count = have;
    b.p = g.W + t.group * g.sw * P::SZ + (P::BS == KMAJOR ? n0 * g.ldw : (int64_t)n0) * P::SZ;
    b.ld = (uint32_t)(g.ldw * P::SZ);
    b.count = g.N - n0;
    pv4f acc[P::MT][P::NT];
    clear<P>(acc);
    product_run<P>(a, b, g.K, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + (wave % P::WN) * P::TN;
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int m = (wave / P::WN) * P::TM + 16 * i + (lane & 15);
        if (m < have) store_row<P, O>(g.Y + (t.row0 + m) * g.ldy * sizeof(O), n, g.N, acc[i]);
    }
}

template <class P, class O>
__global__ void __launch_bounds__(P::THREADS) grouped_kernel(const GroupedArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    GroupTile t;
    if constexpr (P::BM == 256) {
        // Tiles of at most 128 rows, a group's last one or a half, take the same waves in half the time.  (16384 rows in 16 groups,
        // 2048 -> 4096: 4.5 rounds of workgroups, every fourth row tile a partial one: 280 us without, 272 with;
        // 4096 rows in 8 groups, 4096 -> 4096: 194 and 172)
        if (!find_tile<P::BM, true>(g, blockIdx.x, &t)) return;
        if (t.half || t.rows <= 128) {
            grouped_tile<ProductTile<typename P::T, 128, P::BN, P::WM, P::WN, P::AS, P::BS, P::S>, O>(g, t, t.col_tile * P::BN, smem);
            return;
        }
    } else {
        if (!find_tile<P::BM>(g, blockIdx.x, &t)) return;
    }
    grouped_tile<P, O>(g, t, t.col_tile * P::BN, smem);
}

// ------------------------------------------------------------------------------------------------ few rows per group
// Decoding: a group has a handful of rows, and what takes time is reading its matrix once.  A workgroup owns up to 16 MT
// rows of a group and a strip of columns; its eight waves take pieces of K in turn and are joined through LDS in a
// fixed order.  The matrix goes from memory straight into MFMA operands, 8 or 16 loads of 16 bytes per lane in flight, 64 or 128
// KB a workgroup (a CU needs about 50 KB in flight to draw its share of HBM's rate, and nothing is under way between two pieces).
// Two workgroups share a CU with 16 or 32 rows (80 to 111 registers), one with 64 and for 16-bit KROWS (160 to 219):
//   KMAJOR  32 columns; a lane's 16 bytes are k of its column, as the MFMA wants them; 256 bytes of a column per piece.
//   KROWS   16 EPC columns (128 of 16 bits, 64 floats): lane l reads EPC columns of k rows EPC (l / 16) + 0 .. EPC - 1, a block
//           that it transposes in its own registers (one v_perm per two elements; floats need none); accumulator tile j
//           then has the columns congruent to j modulo EPC.
// Rows that do not exist read as zeros without memory traffic, row tiles beyond the group's end are left out.
// 8 groups of one row, 2048 -> 1024, bfloat16 (34 MB): KMAJOR 9.0 us, KROWS 12.2, against 19 in 64 x 128 tiles; 32 groups of up to
// 16 rows, 4096 -> 2048 (0.5 GB): 115 to 128 us (KMAJOR) and 102 to 104 (KROWS) against 106 to 109 and 104.
__device__ __forceinline__ pv4u load_or_zeros(__amdgpu_buffer_rsrc_t rsrc, uint32_t off, bool valid) {
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(valid ? off : OUT_OF_RANGE), 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const char *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, 0x7fffffff, 0x00020000);
}

template <class T, int BS, int MT = 1>
struct FewRows {
    static constexpr int SZ = sizeof(T), EPC = 16 / SZ, STEP = 64 / SZ;     // k per MFMA step
    static constexpr int WAVES = 8, THREADS = 64 * WAVES;
    static constexpr int NT = BS == KMAJOR ? 2 : EPC, COLS = 16 * NT;
    static constexpr int LOADS = BS == KROWS && SZ == 2 && MT == 1 ? 16 : 8;  // of the matrix per piece
    static constexpr int STEPS = BS == KMAJOR ? LOADS / NT : LOADS / EPC;
    static constexpr int LDS = WAVES * 16 * COLS * 4;
};

template <class T, class O, int BS, int MT>
__global__ void __launch_bounds__(512) grouped_few_rows_kernel(const GroupedArgs g) {
    using F = FewRows<T, BS, MT>;
    constexpr int EPC = F::EPC, NT = F::NT, SZ = F::SZ;
    __shared__ __attribute__((aligned(16))) float joint[F::WAVES][16][F::COLS];
    GroupTile t;
    if (!find_tile<16 * MT>(g, blockIdx.x, &t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, kg = lane >> 4;
    const int n0 = t.col_tile * F::COLS, rows = t.rows < 16 * MT ? t.rows : 16 * MT;
    const char *x = g.X + t.row0 * g.ldx * SZ;
    const char *w = g.W + t.group * g.sw * SZ + (BS == KMAJOR ? n0 * g.ldw : (int64_t)n0) * SZ;
    const uint32_t ldx = (uint32_t)(g.ldx * SZ), ldw = (uint32_t)(g.ldw * SZ);
    const __amdgpu_buffer_rsrc_t xr = buffer_at(x);
    pv4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = pv4f{0.f, 0.f, 0.f, 0.f};
    constexpr int PIECE = F::STEP * F::STEPS;
    for (int k0 = wave * PIECE; k0 < g.K; k0 += F::WAVES * PIECE) {
        pv4u b[F::STEPS][BS == KMAJOR ? NT : EPC], a[F::STEPS][MT];
        if (BS == KMAJOR) {
            const __amdgpu_buffer_rsrc_t wr = buffer_at(w + (int64_t)k0 * SZ);
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int s = 0; s < F::STEPS; s++)
                    b[s][j] = load_or_zeros(wr, (uint32_t)(16 * j + r) * ldw + s * 64 + kg * 16, n0 + 16 * j + r < g.N && k0 + s * F::STEP + kg * EPC < g.K);
        } else {
            const __amdgpu_buffer_rsrc_t wr = buffer_at(w + (int64_t)k0 * ldw);
#pragma unroll
            for (int s = 0; s < F::STEPS; s++)
#pragma unroll
                for (int j = 0; j < EPC; j++) {
                    const int k = s * F::STEP + kg * EPC + j;
                    b[s][j] = load_or_zeros(wr, (uint32_t)k * ldw + r * 16, n0 + r * EPC < g.N && k0 + k < g.K);
                }
        }
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int s = 0; s < F::STEPS; s++)
                a[s][i] = load_or_zeros(xr, (uint32_t)(16 * i + r) * ldx + (uint32_t)k0 * SZ + s * 64 + kg * 16,
                                        16 * i + r < rows && k0 + s * F::STEP + kg * EPC < g.K);
        __builtin_amdgcn_sched_barrier(0);           // (every load is under way before the first is waited for)
#pragma unroll
        for (int s = 0; s < F::STEPS; s++) {
            pv4u f[NT];
            if constexpr (BS == KMAJOR) {
#pragma unroll
                for (int j = 0; j < NT; j++) f[j] = b[s][j];
            } else if constexpr (SZ == 2) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int p = 0; p < 4; p++)
                        f[j][p] = __builtin_amdgcn_perm(b[s][2 * p + 1][j >> 1], b[s][2 * p][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int p = 0; p < 4; p++) f[j][p] = b[s][p][j];
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
                if (16 * i >= rows) break;
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = MatrixOp<T>::mul(f[j], a[s][i], acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        if (16 * i >= rows) break;
        if (i) __syncthreads();
        // element e of tile j belongs to column 16 j + 4 kg + e (KMAJOR) or EPC (4 kg + e) + j (KROWS)
        if (BS == KMAJOR) {
#pragma unroll
            for (int j = 0; j < NT; j++) *reinterpret_cast<pv4f *>(&joint[wave][r][16 * j + 4 * kg]) = acc[i][j];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < NT; j += 4)
                    *reinterpret_cast<pv4f *>(&joint[wave][r][EPC * (4 * kg + e) + j]) = pv4f{acc[i][j][e], acc[i][j + 1 < NT ? j + 1 : 0][e],
                                                                                              acc[i][j + 2 < NT ? j + 2 : 0][e], acc[i][j + 3 < NT ? j + 3 : 0][e]};
        }
        __syncthreads();
        for (int q = threadIdx.x; q < 16 * F::COLS / 4; q += F::THREADS) {
            const int row = q / (F::COLS / 4), c = q % (F::COLS / 4) * 4;
            if (16 * i + row >= rows) continue;
            pv4f sum = *reinterpret_cast<const pv4f *>(&joint[0][row][c]);
#pragma unroll
            for (int v = 1; v < F::WAVES; v++) sum += *reinterpret_cast<const pv4f *>(&joint[v][row][c]);
            O *y = reinterpret_cast<O *>(g.Y + (t.row0 + 16 * i + row) * g.ldy * sizeof(O)) + n0 + c;
            typedef O quad __attribute__((ext_vector_type(4)));
            typedef O quad_anywhere __attribute__((ext_vector_type(4), aligned(sizeof(O))));
            if (n0 + c + 4 <= g.N) {
                *reinterpret_cast<quad_anywhere *>(y) = __builtin_convertvector(sum, quad);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n0 + c + e < g.N) y[e] = (O)sum[e];
            }
        }
    }
}

// The group that is `rank`-th in size (ties: the lower index first), its first row and the row behind its last; the first 64
// groups among themselves, as the groups behind them, which keep their places.  The results are uniform over the wave.
__device__ __forceinline__ int ranked_group(const GroupedArgs &g, int rank, int *first, int *last) {
    const int lane = threadIdx.x & 63, among = g.E < 64 ? g.E : 64;
    int a = 0, b = -1, e = rank;
    if (lane < among) { a = group_edge(g, lane); b = group_edge(g, lane + 1); }
    if (rank < 64) {
        const int size = b - a;
        int place = 0;
        for (int j = 0; j < among; j++) {
            const int other = __builtin_amdgcn_readlane(size, j);
            place += other > size || (other == size && j < lane);
        }
        e = __ffsll((unsigned long long)__ballot(lane < among && place == rank)) - 1;
    }
    if (e < 64 && !__ballot(lane < among && b < a)) {
        *first = __builtin_amdgcn_readlane(a, e);
        *last = __builtin_amdgcn_readlane(b, e);
    } else {                                         // the running maximum of the offsets up to e, and with e + 1
        int high = 0;
        for (int i = lane; i <= e; i += 64) high = max(high, group_edge(g, i));
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) high = max(high, __shfl_xor(high, m, 64));
        *first = __builtin_amdgcn_readfirstlane(high);
        *last = max(*first, group_edge(g, e + 1));
    }
    return e;
}

// dW[e] tile: rows of the tile are K (contiguous in X), columns N (contiguous in dY), the reduction runs over the
// rows of the group.  Here W is dY (ldw its row stride), Y is dW (ldy, sw its row and matrix strides).
template <class P, class O>
__global__ void __launch_bounds__(P::THREADS) grouped_wgrad_kernel(const GroupedArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // Every die takes its share of every group's tiles (dies that took whole groups would end with the largest one), the
    // workgroups of a die go through the groups from the largest to the smallest, so that short tiles come last.
    const int row_tiles = (g.K + P::BM - 1) / P::BM;
    const unsigned tiles = (unsigned)row_tiles * g.col_tiles, per_group = tiles * g.parts;
    int k0, n0, first, last;
    const unsigned rank = blockIdx.x / per_group, at = die_run(blockIdx.x % per_group, per_group, g.xcds), part = at / tiles;
    panel_tile(at % tiles, row_tiles, g.col_tiles, &k0, &n0);
    const int e = ranked_group(g, rank, &first, &last);
    k0 *= P::BM;
    n0 *= P::BN;
    if (g.parts > 1) {                               // this part's rows: whole stages
        const int stages = last > first ? (last - first + P::KS - 1) / P::KS : 0, per = (stages + g.parts - 1) / g.parts * P::KS;
        const int64_t from = first + (int64_t)part * per;
        first = from < last ? (int)from : last;
        last = last - first < per ? last : first + per;
    }
    const int rows = last > first ? last - first : 0;
    TileSource a, b;
    a.p = g.X + (first * g.ldx + k0) * P::SZ;
    a.ld = (uint32_t)(g.ldx * P::SZ);
    a.count = g.K - k0;
    b.p = g.W + (first * g.ldw + n0) * P::SZ;
    b.ld = (uint32_t)(g.ldw * P::SZ);
    b.count = g.N - n0;
    pv4f acc[P::MT][P::NT];
    clear<P>(acc);
    if (rows) product_run<P>(a, b, rows, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + (wave % P::WN) * P::TN;
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int k = k0 + (wave / P::WN) * P::TM + 16 * i + (lane & 15);
        if (k < g.K) store_row<P, O>(g.Y + (part * g.plane + e * g.sw + k * g.ldy) * (int64_t)sizeof(O), n, g.N, acc[i]);
    }
}

// ------------------------------------------------------------------------------------------------ padded copies
// Both operands' copies in one launch: they are independent, and small (2999 x 1365 and 5 matrices of 1000 x 1365, half: 15 us in two
// launches, 11 in one; the product with them 37.5 and 33.5).
struct PadArgs {
    const char *src;
    char *dst;
    int64_t rows, cols, ld, batch_stride, chunks_per_row, chunks;
    unsigned blocks;
};
template <class T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const PadArgs first, const PadArgs second) {
    constexpr int CE = 16 / sizeof(T);
    typedef typename Chunk<T>::type chunk;
    const bool other = blockIdx.x >= first.blocks;
    const PadArgs p = other ? second : first;
    for (int64_t i = (int64_t)(blockIdx.x - (other ? first.blocks : 0)) * 256 + threadIdx.x; i < p.chunks; i += (int64_t)p.blocks * 256) {
        const int64_t row = i / p.chunks_per_row, c = (i % p.chunks_per_row) * CE;
        const T *s = reinterpret_cast<const T *>(p.src) + (row / p.rows) * p.batch_stride + (row % p.rows) * p.ld + c;
        chunk v;
        if (c + CE <= p.cols) {                      // (memory takes 16 bytes at any element's alignment)
            v = *reinterpret_cast<const typename Chunk<T>::anywhere *>(s);
        } else {
#pragma unroll
            for (int j = 0; j < CE; j++) v[j] = c + j < p.cols ? s[j] : (T)0;
        }
        *reinterpret_cast<chunk *>(p.dst + i * 16) = v;
    }
}

int launch_pad_rows(const PadRows &a, const PadRows &b, int size, hipStream_t stream) {
    auto args = [&](const PadRows &p) {
        const int64_t per_row = padded_cols(p.cols, size) * size / 16, chunks = p.batch * p.rows * per_row;
        return PadArgs{static_cast<const char *>(p.src), static_cast<char *>(p.dst), p.rows, p.cols, p.ld, p.batch_stride, per_row, chunks,
                       (unsigned)std::min<int64_t>((chunks + 255) / 256, 65536)};
    };
    const PadArgs first = args(a), second = args(b);
    if (first.blocks + second.blocks == 0) return T2SP_OK;
    hipLaunchKernelGGL(size == 4 ? pad_rows_kernel<uint32_t> : pad_rows_kernel<uint16_t>, dim3(first.blocks + second.blocks), dim3(256), 0, stream,
                       first, second);
    return launched();
}

// ------------------------------------------------------------------------------------------------ joined planes
template <class O>
__global__ void __launch_bounds__(256) join_planes_kernel(const float *planes, int parts, int64_t plane, int64_t rows, int64_t cols, int64_t ldp, O *out,
                                                          int64_t ldo, int64_t batch_stride, int64_t quads) {
    const int64_t per = ldp / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per, c = i % per * 4;
        pv4f sum = *reinterpret_cast<const pv4f *>(planes + i * 4);
#pragma unroll 4
        for (int p = 1; p < parts; p++) sum += *reinterpret_cast<const pv4f *>(planes + p * plane + i * 4);
        O *o = out + row / rows * batch_stride + row % rows * ldo + c;
        typedef O quad __attribute__((ext_vector_type(4)));
        typedef O quad_anywhere __attribute__((ext_vector_type(4), aligned(sizeof(O))));
        if (c + 4 <= cols) {
            *reinterpret_cast<quad_anywhere *>(o) = __builtin_convertvector(sum, quad);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c + j < cols) o[j] = (O)sum[j];
        }
    }
}

int launch_join_planes(const float *planes, int parts, int64_t batch, int64_t rows, int64_t cols, int64_t ldp, void *out, int out_type,
                       int64_t ldo, int64_t batch_stride, hipStream_t stream) {
    const int64_t quads = batch * rows * (ldp / 4), blocks = std::min<int64_t>((quads + 255) / 256, 16384);
    return with_types(out_type, out_type, [&](auto *, auto *o) {
        using O = std::remove_pointer_t<decltype(o)>;
        hipLaunchKernelGGL(join_planes_kernel<O>, dim3((unsigned)blocks), dim3(256), 0, stream, planes, parts, batch * rows * ldp, rows, cols, ldp,
                           static_cast<O *>(out), ldo, batch_stride, quads);
        return launched();
    });
}

// ------------------------------------------------------------------------------------------------ launches
// The number of row tiles of `bm` rows that T rows in at most E groups can make.
static int64_t most_row_tiles(int T, int E, int bm) { return T / bm + (E < T ? E : T); }

template <class P, class O>
static int launch_forward(GroupedArgs g, hipStream_t stream) {
    g.col_tiles = (g.N + P::BN - 1) / P::BN;
    g.die_cus = std::max(1, machine().cus / g.xcds);
    // (halves: up to half a die's CUs more workgroups per die)
    const int64_t runs = (most_row_tiles(g.T, g.E, P::BM) * g.col_tiles + g.xcds - 1) / g.xcds + (P::BM == 256 ? (g.die_cus + 1) / 2 : 0);
    const int64_t blocks = runs * g.xcds;
    if (blocks > 0x7fffffff / P::THREADS) return T2SP_ERR_SHAPE;
    auto kern = grouped_kernel<P, O>;
    if (allow_lds(kern, P::LDS)) return T2SP_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(P::THREADS), P::LDS, stream, g);
    return launched();
}

template <class T, class O, int BS, int MT>
static int launch_few_rows(GroupedArgs g, hipStream_t stream) {
    g.col_tiles = (g.N + FewRows<T, BS>::COLS - 1) / FewRows<T, BS>::COLS;
    const int64_t blocks = (most_row_tiles(g.T, g.E, 16 * MT) * g.col_tiles + g.xcds - 1) / g.xcds * g.xcds;
    if (blocks > 0x7fffffff / 512) return T2SP_ERR_SHAPE;
    hipLaunchKernelGGL((grouped_few_rows_kernel<T, O, BS, MT>), dim3((unsigned)blocks), dim3(512), 0, stream, g);
    return launched();
}

template <class P, class O>
static int launch_wgrad(GroupedArgs g, hipStream_t stream) {
    g.col_tiles = (g.N + P::BN - 1) / P::BN;
    const int64_t blocks = (int64_t)g.E * ((g.K + P::BM - 1) / P::BM) * g.col_tiles * g.parts;
    if (blocks > 0x7fffffff / P::THREADS) return T2SP_ERR_SHAPE;
    auto kern = grouped_wgrad_kernel<P, O>;
    if (allow_lds(kern, P::LDS)) return T2SP_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(P::THREADS), P::LDS, stream, g);
    return launched();
}

// What a product takes in each form (microseconds), from the extents alone: as if every row chose its group freely, so that
// E (1 - exp(-T / E)) groups have rows, and their ends make half a row tile more than whole tiles would.  The workgroups share
// the CUs, n to a CU, and a stage of 64 bytes of k takes a + n (c + fill x the 16-row blocks that hold rows); `ends` stages go
// into start and store.  Beside that stands the reading of the matrices at `rate` TB/s: the larger of the two and a quarter of
// the smaller.  Fitted to measured products of 1 to 8192 rows in 1 to 64 groups of any sizes, 64 to 4096 x 64 to 4096, matrices not in
// the caches.  Over 60 other such products for each of bfloat16 and float in each layout, the form picked takes 2 to 5 percent more
// than the best of the six (geometric mean) and 7 to 20 at the 95th percentile; the worst (1.7 to 2 times) are
// mostly calls of 5 us with fewer rows than groups.
struct GroupShape {
    int rows, cols;
    double a, c, fill;
    int ends;
    double rate;
};
template <class T, int BS>
struct GroupShapes {
    static constexpr bool H = sizeof(T) == 2, KC = BS == KMAJOR;
    static constexpr int COLS = FewRows<T, BS>::COLS;
    static constexpr GroupShape FEW1 = H ? KC ? GroupShape{16, COLS, 0.046, 0.058, 0, 19, 8.9} : GroupShape{16, COLS, 0, 0.129, 0, 36, 5.9}
                                         : KC ? GroupShape{16, COLS, 0.031, 0.063, 0, 28, 8.7} : GroupShape{16, COLS, 0.048, 0.085, 0, 22, 6.5};
    static constexpr GroupShape FEW2 = H ? KC ? GroupShape{32, COLS, 0.048, 0.050, 0.023, 23, 7.4} : GroupShape{32, COLS, 0, 0.118, 0.021, 45, 5.8}
                                         : KC ? GroupShape{32, COLS, 0.039, 0.052, 0.027, 27, 7.4} : GroupShape{32, COLS, 0.037, 0.091, 0.030, 25, 6.9};
    static constexpr GroupShape FEW4 = H ? KC ? GroupShape{64, COLS, 0.027, 0.066, 0.024, 35, 5.5} : GroupShape{64, COLS, 0, 0.098, 0.035, 56, 5.4}
                                         : KC ? GroupShape{64, COLS, 0.017, 0.070, 0.032, 37, 5.7} : GroupShape{64, COLS, 0, 0.101, 0.044, 37, 6.5};
    static constexpr GroupShape T64 = H ? KC ? GroupShape{64, 128, 0.049, 0.248, 0, 8, 6.0} : GroupShape{64, 128, 0.091, 0.165, 0, 12, 6.4}
                                        : KC ? GroupShape{64, 64, 0.153, 0.234, 0, 9, 7.8} : GroupShape{64, 64, 0.134, 0.232, 0, 9, 8.0};
    static constexpr GroupShape T128 = H ? KC ? GroupShape{128, 128, 0.026, 0.253, 0, 14, 5.8} : GroupShape{128, 128, 0.015, 0.233, 0, 17, 8.5}
                                         : KC ? GroupShape{128, 128, 0.008, 0.958, 0, 6, 6.9} : GroupShape{128, 128, 0.062, 0.923, 0, 5, 7.0};
    static constexpr GroupShape T256 = KC ? GroupShape{256, 256, -0.171, 0.625, 0, 13, 5.6} : GroupShape{256, 256, -0.139, 0.548, 0, 17, 8.1};
};
static double grouped_cost(const GroupShape &s, int T, int E, int K, int N, int size) {
    const double groups = E == 1 ? 1 : E * (1 - std::exp(-(double)T / E)), k_bytes = (double)K * size, cus = machine().cus, per = T / groups;
    const double row_tiles = E == 1 ? std::ceil(per / s.rows) : groups * std::max(1.0, per / s.rows + 0.5);
    const double share = row_tiles * ((N + s.cols - 1) / s.cols) / cus, n = std::max(1.0, E == 1 ? std::ceil(share) : share + 0.3);
    const double work = (k_bytes / 64 + s.ends) * (s.a + n * (s.c + s.fill * std::min((double)s.rows, T / row_tiles) / 16));
    const double reads = groups * k_bytes * N / (s.rate * 1e6);
    return std::max(work, reads) + 0.25 * std::min(work, reads);
}

// The rows of a tile; `few`: straight from memory (16, 32 or 64 rows), else through LDS (64, 128 or 256).
struct GroupForm {
    int rows;
    bool few;
};
template <class T, int BS>
static GroupForm forward_form(int rows, int E, int K, int N) {
    typedef GroupShapes<T, BS> S;
    auto cost = [&](const GroupShape &s) { return grouped_cost(s, rows, E, K, N, sizeof(T)); };
    const double few1 = cost(S::FEW1), few2 = cost(S::FEW2), few4 = cost(S::FEW4), c64 = cost(S::T64), c128 = cost(S::T128),
                 c256 = sizeof(T) == 2 ? cost(S::T256) : 1e30;
    const double best = std::min({few1, few2, few4, c64, c128, c256});
    if (best == few1 || best == few2 || best == few4) return {best == few1 ? 16 : best == few2 ? 32 : 64, true};
    return {best == c256 ? 256 : best == c128 ? 128 : 64, false};
}
template <class T, class O, int BS>
static int forward_tiles(const GroupedArgs &g, hipStream_t stream) {
    const GroupForm form = forward_form<T, BS>(g.T, g.E, g.K, g.N);
    if (form.few) return form.rows == 16   ? launch_few_rows<T, O, BS, 1>(g, stream)
                         : form.rows == 32 ? launch_few_rows<T, O, BS, 2>(g, stream)
                                           : launch_few_rows<T, O, BS, 4>(g, stream);
    if constexpr (sizeof(T) == 2)
        if (form.rows == 256) return launch_forward<Tile256<T, KMAJOR, BS>, O>(g, stream);
    if (form.rows == 128) return launch_forward<Tile128<T, KMAJOR, BS>, O>(g, stream);
    return launch_forward<Tile64<T, BS>, O>(g, stream);
}

// Few and small matrices from many rows: the rows of every group are cut into parts, whose sums are joined in a fixed order.
// (8192 rows in one group, 512 x 512, bfloat16: 70 us whole, 22 in parts; float: 533 and 50)
static int wgrad_parts(int T, int E, int K, int N, int size) {
    const TileShape &s = size == 2 ? SHAPE_128 : SHAPE_128F;
    const double tiles = (double)E * ((K + 127) / 128) * ((N + 127) / 128);      // (extents up to 2^30 each: beyond 64 bits)
    return split_parts(tiles, machine().cus, (double)T / E * size / 64, s.a + s.c, 4.0 * E * K * N);
}
static int64_t plane_cols(int N) { return (N + 3) / 4 * 4; }
// The tile edge of sums that are not cut.
static int wgrad_tile(int T, int E, int K, int N, int size) { return pick_tile(E, K, N, (T + E - 1) / E, size, false); }

template <class T, class O>
static int wgrad_tiles(const GroupedArgs &g, float *planes, int out_type, hipStream_t stream) {
    if (g.parts > 1) {
        GroupedArgs p = g;
        p.Y = reinterpret_cast<char *>(planes);
        p.ldy = plane_cols(g.N);
        p.sw = g.K * p.ldy;
        p.plane = g.E * p.sw;
        if (int err = launch_wgrad<Tile128<T, KROWS, KROWS>, float>(p, stream)) return err;
        return launch_join_planes(planes, g.parts, g.E, g.K, g.N, p.ldy, g.Y, out_type, g.ldy, g.sw, stream);
    }
    if constexpr (sizeof(T) == 2)
        if (wgrad_tile(g.T, g.E, g.K, g.N, sizeof(T)) == 256) return launch_wgrad<Tile256<T, KROWS, KROWS>, O>(g, stream);
    return launch_wgrad<Tile128<T, KROWS, KROWS>, O>(g, stream);
}

}  // namespace t2sp

using namespace t2sp;

extern "C" size_t t2sp_gemm_grouped_workspace_bytes(int type, int opb, const void *X, const void *W, int T, int E, int K, int N,
                                                    int64_t ldx, int64_t ldw, int64_t sw) {
    const int size = type_bytes(type);
    if (!size || T < 0 || T > T2SP_MAX_EXTENT || !extent_ok(E) || !extent_ok(K) || !extent_ok(N) || !stride_ok(ldx) || !stride_ok(ldw) ||
        !stride_ok(sw) || (int64_t)E * (opb ? N : K) > T2SP_MAX_EXTENT)
        return 0;
    const int64_t wr = opb ? N : K, wc = opb ? K : N;
    size_t n = 0;
    if (!loadable(X, ldx, K, size)) n += round_up((size_t)T * padded_cols(K, size) * size, 16);
    if (!loadable(W, ldw, wc, size) || sw * size % 16) n += (size_t)E * wr * padded_cols(wc, size) * size;
    return n;
}

extern "C" int t2sp_gemm_grouped(int type, int out_type, int opb, const void *X, const void *W, const void *offsets, int offset_bits,
                                 void *Y, int T, int E, int K, int N, int64_t ldx, int64_t ldw, int64_t sw, int64_t ldy,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    const int size = type_bytes(type);
    const int64_t wr = opb ? N : K, wc = opb ? K : N;
    if (!size || !out_type_ok(type, out_type) || (offset_bits != 32 && offset_bits != 64) || T < 0 || T > T2SP_MAX_EXTENT || !extent_ok(E) ||
        !row_ok(K, size) || !extent_ok(N) || !row_ok(wc, size) || !stride_ok(ldx) || !stride_ok(ldw) || !stride_ok(sw) || !stride_ok(ldy) || ldx < K || ldw < wc ||
        ldy < N || (int64_t)E * wr > T2SP_MAX_EXTENT)
        return T2SP_ERR_SHAPE;
    if (T == 0) return T2SP_OK;
    if (!X || !W || !offsets || !Y) return T2SP_ERR_SHAPE;
    const size_t need = t2sp_gemm_grouped_workspace_bytes(type, opb, X, W, T, E, K, N, ldx, ldw, sw);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)) return T2SP_ERR_SHAPE;
    const hipStream_t st = (hipStream_t)stream;
    char *room = static_cast<char *>(workspace);
    PadRows px{}, pw{};
    if (!loadable(X, ldx, K, size)) {
        const int64_t pc = padded_cols(K, size);
        px = {X, room, 1, T, K, ldx, 0};
        X = room;
        ldx = pc;
        room += round_up((size_t)T * pc * size, 16);
    }
    if (!loadable(W, ldw, wc, size) || sw * size % 16) {
        const int64_t pc = padded_cols(wc, size);
        pw = {W, room, E, wr, wc, ldw, sw};
        W = room;
        ldw = pc;
        sw = wr * pc;
    }
    if (int err = launch_pad_rows(px, pw, size, st)) return err;
    // (a copy's padding is zeros, so the reduction may run over it; columns of Y stop at N)
    GroupedArgs g{};
    g.X = static_cast<const char *>(X); g.W = static_cast<const char *>(W); g.Y = static_cast<char *>(Y);
    g.offsets = offsets; g.off64 = offset_bits == 64;
    g.T = T; g.E = E; g.K = K; g.N = N;
    g.ldx = ldx; g.ldw = ldw; g.sw = sw; g.ldy = ldy;
    g.xcds = machine().xcds;
    return with_types(type, out_type, [&](auto *t, auto *o) {
        using TT = std::remove_pointer_t<decltype(t)>;
        using OO = std::remove_pointer_t<decltype(o)>;
        return opb ? forward_tiles<TT, OO, KMAJOR>(g, st) : forward_tiles<TT, OO, KROWS>(g, st);
    });
}

extern "C" size_t t2sp_gemm_grouped_wgrad_workspace_bytes(int type, const void *X, const void *dY, int T, int E, int K, int N, int64_t ldx,
                                                          int64_t ldy) {
    const int size = type_bytes(type);
    if (!size || T < 0 || T > T2SP_MAX_EXTENT || !extent_ok(E) || !extent_ok(K) || !extent_ok(N) || !stride_ok(ldx) || !stride_ok(ldy)) return 0;
    size_t n = 0;
    if (!loadable(X, ldx, K, size)) n += round_up((size_t)T * padded_cols(K, size) * size, 16);
    if (!loadable(dY, ldy, N, size)) n += round_up((size_t)T * padded_cols(N, size) * size, 16);
    if (const int parts = wgrad_parts(T, E, K, N, size); parts > 1) n += (size_t)parts * E * K * plane_cols(N) * sizeof(float);
    return n;
}

extern "C" int t2sp_gemm_grouped_wgrad(int type, int out_type, const void *X, const void *dY, const void *offsets, int offset_bits, void *dW,
                                       int T, int E, int K, int N, int64_t ldx, int64_t ldy, int64_t ldw, int64_t sw, void *workspace,
                                       size_t workspace_bytes, void *stream) {
    const int size = type_bytes(type);
    if (!size || !out_type_ok(type, out_type) || (offset_bits != 32 && offset_bits != 64) || T < 0 || T > T2SP_MAX_EXTENT || !extent_ok(E) ||
        !row_ok(K, size) || !row_ok(N, size) || !stride_ok(ldx) || !stride_ok(ldy) || !stride_ok(ldw) || !stride_ok(sw) || ldx < K || ldy < N || ldw < N ||
        (E > 1 && sw < (K - 1) * ldw + N))
        return T2SP_ERR_SHAPE;
    if (!offsets || !dW || (T && (!X || !dY))) return T2SP_ERR_SHAPE;
    const size_t need = t2sp_gemm_grouped_wgrad_workspace_bytes(type, X, dY, T, E, K, N, ldx, ldy);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)) return T2SP_ERR_SHAPE;
    const hipStream_t st = (hipStream_t)stream;
    char *room = static_cast<char *>(workspace);
    PadRows px{}, pd{};
    if (!loadable(X, ldx, K, size) && T) {
        const int64_t pc = padded_cols(K, size);
        px = {X, room, 1, T, K, ldx, 0};
        X = room;
        ldx = pc;
        room += round_up((size_t)T * pc * size, 16);
    }
    if (!loadable(dY, ldy, N, size) && T) {
        const int64_t pc = padded_cols(N, size);
        pd = {dY, room, 1, T, N, ldy, 0};
        dY = room;
        ldy = pc;
        room += round_up((size_t)T * pc * size, 16);
    }
    if (int err = launch_pad_rows(px, pd, size, st)) return err;
    GroupedArgs g{};
    g.X = static_cast<const char *>(X); g.W = static_cast<const char *>(dY); g.Y = static_cast<char *>(dW);
    g.offsets = offsets; g.off64 = offset_bits == 64;
    g.T = T; g.E = E; g.K = K; g.N = N;
    g.ldx = ldx; g.ldw = ldy; g.sw = sw; g.ldy = ldw;
    g.xcds = machine().xcds;
    g.parts = wgrad_parts(T, E, K, N, size);
    return with_types(type, out_type, [&](auto *t, auto *o) {
        return wgrad_tiles<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>>(g, reinterpret_cast<float *>(room), out_type, st);
    });
}

extern "C" int t2sp_gemm_grouped_plan(int type, int opb, int T, int E, int K, int N, int *few) {
    if (!type_bytes(type) || T < 1 || T > T2SP_MAX_EXTENT || !extent_ok(E) || !extent_ok(K) || !extent_ok(N) || !few) return T2SP_ERR_SHAPE;
    return with_types(type, type, [&](auto *t, auto *) {
        using TT = std::remove_pointer_t<decltype(t)>;
        const GroupForm form = opb ? forward_form<TT, KMAJOR>(T, E, K, N) : forward_form<TT, KROWS>(T, E, K, N);
        *few = form.few;
        return form.rows;
    });
}
extern "C" int t2sp_gemm_grouped_wgrad_plan(int type, int T, int E, int K, int N, int *parts) {
    if (!type_bytes(type) || T < 0 || T > T2SP_MAX_EXTENT || !extent_ok(E) || !extent_ok(K) || !extent_ok(N) || !parts) return T2SP_ERR_SHAPE;
    *parts = wgrad_parts(T, E, K, N, type_bytes(type));
    return *parts > 1 ? 128 : wgrad_tile(T, E, K, N, type_bytes(type));
}
