// gemv_w4.hip — a few rows times a matrix of 4-bit numbers with a scale (and maybe a zero point) per group of inputs.
//
//   y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / G]) * s[n, k / G],   q in 0 .. 15, z = 8 when there are none
//
// A token being decoded reads every weight once: the bound is HBM, N K / 2 bytes.  What has to be cheap is taking
// the numbers apart: at 6.5 TB/s a CU unpacks 21 of them per cycle.
//
// Numbers stay integers on their way into the matrix cores.  16 + q is a bfloat16 (and a half) whose upper bits are
// constant and whose mantissa holds q in place: 0x4180 | q << 3 (half: 0x4c00 | q << 6), so two numbers cost a shift
// and one v_and_or.  The 16 x 16 x 32 MFMA then sums x (16 + q) exactly but for float addition, over 32 inputs of 16
// rows of the matrix, for up to 16 rows of x at once, and a group ends with
//   y += s * (sum x (16 + q) - (16 + z) * sum x),
// the last sum from one more MFMA with ones.  Scales and zero points are thus applied in float, once per group.
// float rows of x go in as three bfloat16 pieces (24 bits together), each with its own MFMAs.  Their results are not rounded
// to 16 bits, so that what the difference above loses would show (rows whose elements have one sign, 4096 inputs: off by
// 5.6e-7 in norm); the numbers go in as 16 (q - 8) instead, a signed byte made a float, and
//   y += s * (sum x 16 (q - 8) / 16 - (z - 8) * sum x).
//
// Layout (t2sp_w4_pack, made once from plain numbers): blocks of 16 rows x 128 inputs, 1 KB, in which the 16 bytes of
// lane l are what that lane feeds to four MFMAs: row l % 16, inputs 32 f + 8 (l / 16) + 0..7 for f = 0..3; in a word the
// inputs 2 p and 2 p + 1 lie at bits 4 p and 4 p + 16.  A wave reads a block with one 16-byte load per lane, and any N
// and K become whole blocks (numbers behind K meet zeros of x).  Scales and zero points lie in the order in which a lane
// needs them: [tile of 16 rows][block][rows by fours][group of the block][four rows], the block's 4, 2 or 1 groups together
// (with [group][row] a block of 32-input groups took eight loads besides that of its numbers, and 8192 x 4096 13 us).
//
// One workgroup owns 16 * NT rows of the matrix and up to 16 * MT rows of x; its waves take the blocks of K in turn and
// are joined through LDS in a fixed order.
//
// Infinities in x, and values so large that x (16 + q) or a piece of a float leaves float's range though the result does not,
// end in a difference of infinities.  Results that are not finite are therefore computed again as they are written above, one
// input after the other, unless the row holds a NaN, which is then the result.  (16 rows, 4096 x 4096, bfloat16: 7 us; with an
// infinity in one row 1.1 ms, with a row of NaN 7.1 us, with one NaN at a row's end 32.)
#include "product_core.hpp"
#include "product_host.hpp"

namespace t2sp {

struct W4Args {
    const char *x;
    const uint8_t *Q;
    const char *S, *Z;                   // of x's type; Z may be NULL
    const int *ids;                      // row m takes matrix ids[m]; NULL: one matrix
    char *y;
    int M, N, K, E;
    int64_t ldx, ldy;                    // elements
    int blocks_k, tiles_n;               // of 128 inputs, of 16 rows
    int group_shift;                     // G = 32 << group_shift
    int group_blocks;                    // of scales (of 4, 2 or 1 groups)
    int vec_x;                           // rows of x are whole 16-byte chunks
};

// Pieces of x that go through the matrix cores, and 16 + q (float: 16 (q - 8)).
template <class T> struct W4Type;
template <> struct W4Type<__bf16> {
    using M = __bf16;
    static constexpr int PIECES = 1;
    static __device__ __forceinline__ uint32_t pair(uint32_t w, int p) {      // numbers at bits 4 p and 4 p + 16
        return ((p == 0 ? w << 3 : w >> (4 * p - 3)) & 0x00780078u) | 0x41804180u;
    }
    static constexpr uint32_t ONES = 0x3f803f80u;
};
template <> struct W4Type<_Float16> {
    using M = _Float16;
    static constexpr int PIECES = 1;
    static __device__ __forceinline__ uint32_t pair(uint32_t w, int p) {
        return ((p == 0 ? w << 6 : p == 1 ? w << 2 : w >> (4 * p - 6)) & 0x03c003c0u) | 0x4c004c00u;
    }
    static constexpr uint32_t ONES = 0x3c003c00u;
};
template <> struct W4Type<float> {
    using M = __bf16;
    static constexpr int PIECES = 3;
    static __device__ __forceinline__ uint32_t pair(uint32_t w, int p) {      // 16 (q - 8): the signed bytes with (q ^ 8) on top
        const uint32_t bytes = ((w ^ 0x88888888u) << (p & 1 ? 0 : 4)) & 0xf0f0f0f0u;
        const float lo = (float)(int8_t)(bytes >> (4 * (p & 2))), hi = (float)(int8_t)(bytes >> (4 * (p & 2) + 16));
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
    }
    static constexpr uint32_t ONES = W4Type<__bf16>::ONES;
};

// Eight inputs of a row of x at `k`, as MFMA operands: zeros behind K and for rows that do not exist.  VEC: rows are whole
// 16-byte chunks (the loads outside go past the descriptor's end and read zeros without memory traffic).
template <class T, bool VEC>
__device__ __forceinline__ void load_x(__amdgpu_buffer_rsrc_t rsrc, const T *x, uint32_t row, bool exists, int k, int K, pv4u (&raw)[sizeof(T) / 2]) {
    if (VEC) {
        const uint32_t off = exists && k < K ? row * (uint32_t)sizeof(T) + (uint32_t)k * (uint32_t)sizeof(T) : OUT_OF_RANGE;
#pragma unroll
        for (int c = 0; c < (int)sizeof(T) / 2; c++) raw[c] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(off + 16 * c), 0, 0);
    } else {
        T v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = exists && k + j < K ? x[row + k + j] : (T)0.f;
#pragma unroll
        for (int c = 0; c < (int)sizeof(T) / 2; c++) {
            typename Chunk<T>::type u;
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); j++) u[j] = v[c * (16 / sizeof(T)) + j];
            raw[c] = __builtin_bit_cast(pv4u, u);
        }
    }
}
template <class T>
__device__ __forceinline__ void pieces_of(const pv4u (&raw)[sizeof(T) / 2], pv4u (&out)[W4Type<T>::PIECES]) {
    if constexpr (sizeof(T) == 2) {
        out[0] = raw[0];
    } else {
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        b8 a, b, c;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = __builtin_bit_cast(pv4f, raw[j / 4])[j % 4];
            a[j] = (__bf16)v;
            const float r = v - (float)a[j];
            b[j] = (__bf16)r;
            c[j] = (__bf16)(r - (float)b[j]);
        }
        out[0] = __builtin_bit_cast(pv4u, a);
        out[1] = __builtin_bit_cast(pv4u, b);
        out[2] = __builtin_bit_cast(pv4u, c);
    }
}

// y[m, n] for the row of x at `x`, one input after the other.  Q, S, Z: of the row's matrix.
template <class T, int SHIFT>
__device__ __forceinline__ float one_result(const W4Args &g, const T *x, const uint8_t *Q, const T *S, const T *Z, int n) {
    constexpr int GROUPS = SHIFT == 0 ? 4 : SHIFT == 1 ? 2 : 1;
    const int64_t tile = n >> 4;
    const int r = n & 15;
    float sum = 0.f;
#pragma unroll 1
    for (int k = 0; k < g.K; k += 8) {
        const int block = k >> 7, f = (k >> 5) & 3;
        const uint32_t word = *reinterpret_cast<const uint32_t *>(Q + (tile * g.blocks_k + block) * 1024 + (((k >> 3) & 3) * 16 + r) * 16 + f * 4);
        const int64_t at = ((tile * g.group_blocks + (SHIFT == 2 ? (block * 4) >> g.group_shift : block)) * 4 + (r >> 2)) * (GROUPS * 4) +
                           f / (4 / GROUPS) * 4 + (r & 3);
        const float s = (float)S[at], z = Z ? (float)Z[at] : 8.f;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k + j < g.K) sum += (float)x[k + j] * (((float)((word >> (4 * (j >> 1) + 16 * (j & 1))) & 15) - z) * s);
    }
    return sum;
}

// MT: tiles of 16 rows of x, NT: of the matrix.  With many rows of x a workgroup takes several tiles of the matrix, which then
// share what it reads of x (16 rows of 4096 halves are 128 KB, four times a 16-row tile's numbers: 16384 x 4096 with 16 rows takes
// 24 us with one tile, 13 with four).  SHIFT: a group has 32 << SHIFT of a block's inputs (the whole block for groups of 128 and more).
// A wave has DEEP blocks of the matrix, their scales and their part of x under way before it waits for the first.
constexpr int W4_WAVES = 8;
template <class T, int MT, int NT, int SHIFT, bool VEC>
__global__ void __launch_bounds__(64 * W4_WAVES) gemv_w4_kernel(const W4Args g) {
    using Op = MatrixOp<typename W4Type<T>::M>;
    constexpr bool CENTRED = sizeof(T) == 4;
    constexpr int PIECES = W4Type<T>::PIECES, DEEP = MT * NT * sizeof(T) <= 2 ? 4 : MT * sizeof(T) <= 4 ? 2 : 1;
    constexpr int GROUPS = SHIFT == 0 ? 4 : SHIFT == 1 ? 2 : 1;         // of a block
    typedef T quad __attribute__((ext_vector_type(4)));
    typedef T quads __attribute__((ext_vector_type(4 * GROUPS)));
    __shared__ __attribute__((aligned(16))) pv4f joint[W4_WAVES - 1][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kg = lane >> 4;
    const int tile = blockIdx.x * NT, n0 = tile * 16 + 4 * kg;         // this lane ends with rows n0 .. n0 + 3 (+ 16 per tile) of x row r
    int m0 = blockIdx.y * 16 * MT, m_end = g.M;
    const uint8_t *Q = g.Q;
    const T *S = reinterpret_cast<const T *>(g.S), *Z = reinterpret_cast<const T *>(g.Z);
    const int64_t side = (int64_t)g.tiles_n * 16 * g.group_blocks * GROUPS;       // elements of S and of Z per matrix
    bool matrix = true;
    if (g.ids) {                                                        // one row of x per workgroup
        m0 = blockIdx.y;
        m_end = m0 + 1;
        const int e = g.ids[m0];
        matrix = e >= 0 && e < g.E;
        const int64_t at = matrix ? e : 0;
        Q += at * g.tiles_n * g.blocks_k * 1024;
        S += at * side;
        if (Z) Z += at * side;
    }
    const uint8_t *const Q0 = Q;
    const T *const S0 = S, *const Z0 = Z;
    Q += lane * 16;
    S += kg * GROUPS * 4;
    if (Z) Z += kg * GROUPS * 4;
    int64_t tile_q[NT], tile_s[NT];                                     // (tiles behind the last one repeat it and are not stored)
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int own = tile + t < g.tiles_n ? tile + t : g.tiles_n - 1;
        tile_q[t] = (int64_t)own * g.blocks_k * 1024;
        tile_s[t] = (int64_t)own * g.group_blocks;
    }
    const T *x = reinterpret_cast<const T *>(g.x) + (int64_t)m0 * g.ldx;
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(x), 0, 0x7fffffff, 0x00020000);
    pv4f y[MT * NT];
#pragma unroll
    for (int i = 0; i < MT * NT; i++) y[i] = pv4f{0.f, 0.f, 0.f, 0.f};
    const pv4u ones = pv4u{W4Type<T>::ONES, W4Type<T>::ONES, W4Type<T>::ONES, W4Type<T>::ONES};

    if (matrix)
        for (int b0 = wave; b0 < g.blocks_k; b0 += DEEP * W4_WAVES) {
            pv4u q[DEEP][NT], xs[DEEP][4][MT][sizeof(T) / 2];
            quads s[DEEP][NT], z[DEEP][NT];
#pragma unroll
            for (int d = 0; d < DEEP; d++) {                            // (blocks behind the last one repeat it against zeros)
                const int b = b0 + d * W4_WAVES, read = b < g.blocks_k ? b : g.blocks_k - 1;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    q[d][t] = __builtin_nontemporal_load(reinterpret_cast<const pv4u *>(Q + tile_q[t] + (int64_t)read * 1024));
                    const int64_t at = (tile_s[t] + (SHIFT == 2 ? (read * 4) >> g.group_shift : read)) * (16 * GROUPS);
                    s[d][t] = *reinterpret_cast<const quads *>(S + at);
                    if (Z) z[d][t] = *reinterpret_cast<const quads *>(Z + at);
                }
#pragma unroll
                for (int f = 0; f < 4; f++)
#pragma unroll
                    for (int i = 0; i < MT; i++)
                        load_x<T, VEC>(xr, x, (uint32_t)(16 * i + r) * (uint32_t)g.ldx, m0 + 16 * i + r < m_end, (b * 4 + f) * 32 + kg * 8, g.K, xs[d][f][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < DEEP; d++) {
                pv4f acc[MT * NT], sum[MT];
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    constexpr int LAST = 4 / GROUPS - 1;
                    if ((f & LAST) == 0) {
#pragma unroll
                        for (int i = 0; i < MT; i++) sum[i] = pv4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < MT * NT; i++) acc[i] = pv4f{0.f, 0.f, 0.f, 0.f};
                    }
                    pv4u p[MT][PIECES];
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        pieces_of<T>(xs[d][f][i], p[i]);
#pragma unroll
                        for (int c = 0; c < PIECES; c++) sum[i] = Op::mul(ones, p[i][c], sum[i]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const uint32_t word = q[d][t][f];
                        const pv4u w = pv4u{W4Type<T>::pair(word, 0), W4Type<T>::pair(word, 1), W4Type<T>::pair(word, 2), W4Type<T>::pair(word, 3)};
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int c = 0; c < PIECES; c++) acc[i * NT + t] = Op::mul(w, p[i][c], acc[i * NT + t]);
                    }
                    if ((f & LAST) == LAST) {
                        const int c = f / (4 / GROUPS);
#pragma unroll
                        for (int t = 0; t < NT; t++)
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const float less = CENTRED ? 8.f : -16.f, zz = (Z ? (float)z[d][t][4 * c + j] : 8.f) - less;
#pragma unroll
                                for (int i = 0; i < MT; i++)
                                    y[i * NT + t][j] += (float)s[d][t][4 * c + j] * ((CENTRED ? 0.0625f : 1.f) * acc[i * NT + t][j] - zz * sum[i][j]);
                            }
                    }
                }
            }
        }
    if (wave > 0)
#pragma unroll
        for (int i = 0; i < MT * NT; i++) joint[wave - 1][i][lane] = y[i];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < MT * NT; i++)
#pragma unroll
        for (int w = 0; w < W4_WAVES - 1; w++) y[i] += joint[w][i][lane];
    uint32_t again = 0;                                                 // results that are not finite
#pragma unroll
    for (int i = 0; i < MT * NT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) again |= fabsf(y[i][j]) < __builtin_inff() ? 0u : 1u << (4 * i + j);
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int m = m0 + 16 * i + r;
        if (m >= m_end) continue;
        T *row = reinterpret_cast<T *>(g.y) + m * g.ldy;
        typedef T quad_anywhere __attribute__((ext_vector_type(4), aligned(sizeof(T))));
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int n = n0 + 16 * t;
            if (n + 4 <= g.N) {
                *reinterpret_cast<quad_anywhere *>(row + n) = __builtin_convertvector(y[i * NT + t], quad);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (n + j < g.N) row[n + j] = (T)y[i * NT + t][j];
            }
        }
    }
    if (!__ballot(again != 0)) return;
#pragma unroll 1
    for (int i = 0; i < MT; i++) {
        const int m = m0 + 16 * i + r;
        const uint32_t mine = m < m_end ? (again >> (4 * NT * i)) & ((1u << (4 * NT - 1) << 1) - 1) : 0;
        auto rows_of = [](uint64_t lanes) { return (uint32_t)(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu; };
        const uint32_t wanted = rows_of(__ballot(mine != 0));
        uint32_t nans = 0;                                              // rows with a NaN
        for (int k = 0; k < g.K && (wanted & ~nans); k += 32) {
            pv4u raw[sizeof(T) / 2];
            bool nan = false;
            load_x<T, VEC>(xr, x, (uint32_t)(16 * i + r) * (uint32_t)g.ldx, m < m_end, k + kg * 8, g.K, raw);
#pragma unroll
            for (int c = 0; c < (int)sizeof(T) / 2; c++)
#pragma unroll
                for (int j = 0; j < 16 / (int)sizeof(T); j++) {
                    const float v = (float)__builtin_bit_cast(typename Chunk<T>::type, raw[c])[j];
                    nan |= v != v;
                }
            nans |= rows_of(__ballot(nan));
        }
        if (nans >> r & 1) continue;
        for (int j = 0; j < 4 * NT; j++) {
            const int n = n0 + 16 * (j >> 2) + (j & 3);
            if ((mine >> j & 1) && n < g.N)
                reinterpret_cast<T *>(g.y)[m * g.ldy + n] = (T)one_result<T, SHIFT>(g, x + (int64_t)(16 * i + r) * g.ldx, Q0, S0, Z0, n);
        }
    }
}

// ------------------------------------------------------------------------------------------------ packing
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t *q, int N, int K, int64_t ldq, int64_t sq, int blocks_k, int tiles_n, int64_t words,
                                                      uint32_t *Q) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int f = (int)(i & 3), lane = (int)(i >> 2) & 63;
        const int64_t block = i >> 8, b = block % blocks_k, t = block / blocks_k % tiles_n, e = block / blocks_k / tiles_n;
        const int64_t n = t * 16 + (lane & 15), k = b * 128 + f * 32 + (lane >> 4) * 8;
        uint32_t w = 0;
        if (n < N)
            for (int j = 0; j < 8; j++)
                if (k + j < K) w |= (uint32_t)(q[e * sq + n * ldq + k + j] & 15) << (4 * (j >> 1) + 16 * (j & 1));
        Q[i] = w;
    }
}

// dst in the kernel's order (see above), zeros for rows from N and groups behind the last.
template <class T>
__global__ void __launch_bounds__(256) w4_scales_kernel(const T *src, int N, int groups, int64_t ld, int64_t stride, int tiles_n, int group_blocks, int per_block,
                                                        int64_t total, T *dst) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t j = i & 3, c = (i >> 2) % per_block, rest = (i >> 2) / per_block, kg = rest & 3, b = (rest >> 2) % group_blocks,
                      t = (rest >> 2) / group_blocks % tiles_n, e = (rest >> 2) / group_blocks / tiles_n;
        const int64_t n = t * 16 + kg * 4 + j, g = b * per_block + c;
        dst[i] = n < N && g < groups ? src[e * stride + n * ld + g] : (T)0;
    }
}

static int group_shift_of(int group) {
    for (int s = 0; s <= 25; s++)
        if (group == 32 << s) return s;
    return -1;
}

// Groups of a block of 128 inputs, and the blocks of scales that K makes.
static int groups_per_block(int group) { return group == 32 ? 4 : group == 64 ? 2 : 1; }
static int64_t group_blocks_of(int K, int group) {
    const int64_t span = (int64_t)group * groups_per_block(group);
    return (K + span - 1) / span;
}

static unsigned blocks_for(int64_t n) { return (unsigned)(n < 256 * 65536 ? (n + 255) / 256 : 65536); }

}  // namespace t2sp

using namespace t2sp;

extern "C" int t2sp_w4_sizes(int N, int K, int group, int64_t *q_bytes, int64_t *scale_elements) {
    if (!extent_ok(N) || !extent_ok(K) || group_shift_of(group) < 0 || !q_bytes || !scale_elements) return T2SP_ERR_SHAPE;
    const int64_t tiles_n = ((int64_t)N + 15) / 16, blocks_k = ((int64_t)K + 127) / 128;
    *q_bytes = tiles_n * blocks_k * 1024;
    *scale_elements = tiles_n * 16 * group_blocks_of(K, group) * groups_per_block(group);
    return T2SP_OK;
}

extern "C" int t2sp_w4_pack(int type, const uint8_t *q, const void *scales, const void *zeros, int E, int N, int K, int group, int64_t ldq, int64_t sq,
                            int64_t lds, int64_t ss, int64_t ldz, int64_t sz, void *Q, void *S, void *Z, void *stream) {
    int64_t qb, se;
    const int size = type_bytes(type);
    if (!size || !extent_ok(E) || t2sp_w4_sizes(N, K, group, &qb, &se)) return T2SP_ERR_SHAPE;
    const int groups = (K + group - 1) / group;
    if (!q || !scales || !Q || !S || (zeros && !Z) || !stride_ok(ldq) || !stride_ok(sq) || !stride_ok(lds) || !stride_ok(ss) || ldq < K || lds < groups ||
        (zeros && (!stride_ok(ldz) || !stride_ok(sz) || ldz < groups)))
        return T2SP_ERR_SHAPE;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t words = qb / 4 * E, total = se * E;
    const int64_t padded_n = ((int64_t)N + 15) / 16 * 16;
    hipLaunchKernelGGL(w4_pack_kernel, dim3(blocks_for(words)), dim3(256), 0, st, q, N, K, ldq, sq, (int)(((int64_t)K + 127) / 128), (int)(padded_n / 16),
                       words, static_cast<uint32_t *>(Q));
    if (int err = launched()) return err;
    for (int i = 0; i < (zeros ? 2 : 1); i++) {
        const void *from = i ? zeros : scales;
        void *to = i ? Z : S;
        const int64_t ld = i ? ldz : lds, stride = i ? sz : ss;
        if (size == 4)
            hipLaunchKernelGGL(w4_scales_kernel<uint32_t>, dim3(blocks_for(total)), dim3(256), 0, st, static_cast<const uint32_t *>(from), N, groups, ld,
                               stride, (int)(padded_n / 16), (int)group_blocks_of(K, group), groups_per_block(group), total, static_cast<uint32_t *>(to));
        else
            hipLaunchKernelGGL(w4_scales_kernel<uint16_t>, dim3(blocks_for(total)), dim3(256), 0, st, static_cast<const uint16_t *>(from), N, groups, ld,
                               stride, (int)(padded_n / 16), (int)group_blocks_of(K, group), groups_per_block(group), total, static_cast<uint16_t *>(to));
        if (int err = launched()) return err;
    }
    return T2SP_OK;
}

namespace t2sp {
template <class T, int MT, int NT, int SHIFT, bool VEC>
static int launch_w4(const W4Args &g, hipStream_t st) {
    const int64_t rows = g.ids ? g.M : (g.M + 16 * MT - 1) / (16 * MT);
    if (rows > 65535) return T2SP_ERR_SHAPE;
    hipLaunchKernelGGL((gemv_w4_kernel<T, MT, NT, SHIFT, VEC>), dim3((unsigned)((g.tiles_n + NT - 1) / NT), (unsigned)rows), dim3(64 * W4_WAVES), 0, st, g);
    return launched();
}
template <class T, int MT, int NT, bool VEC>
static int launch_w4(const W4Args &g, hipStream_t st) {
    return g.group_shift == 0 ? launch_w4<T, MT, NT, 0, VEC>(g, st)
                              : g.group_shift == 1 ? launch_w4<T, MT, NT, 1, VEC>(g, st) : launch_w4<T, MT, NT, 2, VEC>(g, st);
}
// Several tiles of the matrix per workgroup where enough workgroups are left to fill the CUs.  16384 x 4096, bfloat16, groups of
// 128: 12.6 us with one row and one tile per workgroup, 11.3 with four; 64 rows: 67 us with one tile, 40 with two.  8192 x 4096 is
// the border: one row 7.4 us with one tile, 10.8 with four, 64 rows 35 and 21 with two.  Floats have no registers left for it but for one
// row tile and large groups (16384 x 4096: 24 us with one tile, 16 with four).
struct W4Form {
    int mt, nt;                              // tiles of 16 rows of x, of the matrix
};
static W4Form w4_form(int size, bool ids, int M, int tiles_n, int group_shift, bool vec_x) {
    const int cus = machine().cus;
    if (ids || M <= 16) return {1, vec_x && !ids && tiles_n >= 4 * cus && (size == 2 || group_shift >= 2) ? 4 : 1};
    if (!vec_x) return {2, 1};
    return {M <= 32 ? 2 : 4, size == 2 && tiles_n >= 2 * cus ? 2 : 1};
}
template <class T>
static int launch_w4(const W4Args &g, hipStream_t st) {
    const W4Form form = w4_form(sizeof(T), g.ids, g.M, g.tiles_n, g.group_shift, g.vec_x);
    if (!g.vec_x) return form.mt == 1 ? launch_w4<T, 1, 1, false>(g, st) : launch_w4<T, 2, 1, false>(g, st);
    if constexpr (sizeof(T) == 2) {
        if (form.nt == 4) return launch_w4<T, 1, 4, true>(g, st);
        if (form.nt == 2) return form.mt == 2 ? launch_w4<T, 2, 2, true>(g, st) : launch_w4<T, 4, 2, true>(g, st);
    } else {
        if (form.nt == 4) return launch_w4<T, 1, 4, 2, true>(g, st);
    }
    return form.mt == 1 ? launch_w4<T, 1, 1, true>(g, st) : form.mt == 2 ? launch_w4<T, 2, 1, true>(g, st) : launch_w4<T, 4, 1, true>(g, st);
}
}  // namespace t2sp

extern "C" int t2sp_gemv_w4(int type, const void *x, const void *Q, const void *S, const void *Z, const int *ids, void *y, int M, int N, int K, int E,
                            int group, int64_t ldx, int64_t ldy, void *stream) {
    const int size = type_bytes(type);
    int64_t qb, se;
    if (!size || M < 0 || M > T2SP_MAX_EXTENT || !extent_ok(E) || t2sp_w4_sizes(N, K, group, &qb, &se) || !stride_ok(ldx) || !stride_ok(ldy) || ldx < K ||
        ldy < N)
        return T2SP_ERR_SHAPE;
    if (M == 0) return T2SP_OK;
    if (!x || !Q || !S || !y || (!ids && E != 1)) return T2SP_ERR_SHAPE;
    if (M == 1) ldx = K;                                                 // (a single row's stride carries no information)
    if (ldx * size > T2SP_MAX_ROW_BYTES) return T2SP_ERR_SHAPE;          // (64 rows of x within 31 bits)
    if (reinterpret_cast<uintptr_t>(Q) % 16 || reinterpret_cast<uintptr_t>(S) % 16 || reinterpret_cast<uintptr_t>(Z) % 16) return T2SP_ERR_SHAPE;
    W4Args g{};
    g.x = static_cast<const char *>(x); g.Q = static_cast<const uint8_t *>(Q);
    g.S = static_cast<const char *>(S); g.Z = static_cast<const char *>(Z);
    g.ids = ids; g.y = static_cast<char *>(y);
    g.M = M; g.N = N; g.K = K; g.E = E;
    g.ldx = ldx; g.ldy = ldy;
    g.blocks_k = (int)(((int64_t)K + 127) / 128); g.tiles_n = (int)(((int64_t)N + 15) / 16);
    g.group_shift = group_shift_of(group);
    g.group_blocks = (int)group_blocks_of(K, group);
    g.vec_x = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * size % 16 == 0 && (int64_t)K % 8 == 0;
    const hipStream_t st = (hipStream_t)stream;
    return with_types(type, type, [&](auto *t, auto *) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_w4<T>(g, st);
    });
}

extern "C" int t2sp_gemv_w4_plan(int type, int ids, int M, int N, int K, int group, int *matrix_tiles) {
    int64_t qb, se;
    if (!type_bytes(type) || M < 1 || M > T2SP_MAX_EXTENT || t2sp_w4_sizes(N, K, group, &qb, &se) || !matrix_tiles) return T2SP_ERR_SHAPE;
    const W4Form form = w4_form(type_bytes(type), ids, M, (int)(((int64_t)N + 15) / 16), group_shift_of(group), K % 8 == 0);
    *matrix_tiles = form.nt;
    return form.mt;
}
