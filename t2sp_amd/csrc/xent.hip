// xent.hip — cross entropy of a softmax over a vocabulary, from hidden states, without keeping the logits.
//
//   z[t, v] = sum_d H[t, d] W[v, d]                         (T tokens, V words, D wide)
//   lse[t]  = log sum_v exp z[t, v],    loss[t] = lse[t] - z[t, label[t]]
//   g[t, v] = (exp(z[t, v] - lse[t]) - [v == label[t]]) * dloss[t]
//   dH = g W,   dW = g^T H
// A token whose label is outside 0 .. V - 1 has loss zero, no gradient and no part in dW.
//
// Forward: a 256 x 256 tile of z stays in the accumulators; its rows' maxima and sums of exponentials (both float) go
// to the workspace, 8 bytes per row and tile instead of 1024, and a second kernel joins them.
//
// Backward, for one piece of the vocabulary after the other: the tile of z is computed again, its epilogue writes
// p - [label], and the piece's rows of dW (complete) and its part of dH (added up in float) are two more products.
// p - [label] is a float, which the 16-bit matrix cores do not take: it goes in as the sum of two numbers of the operands'
// type, its rounding and the rounding of what that leaves (16 bits with bfloat16, 22 with half), and both products run over
// both.  12 T D V operations in all, of which 2 T D V pay for not holding T x V logits and 4 T D V for the second number.
// What they leave is below what the float sums of z do (8192 tokens, 4096 wide, 128000 words, bfloat16, float results, against
// float64: dH and dW are off by 6e-7 and 8e-7 in norm, by 9e-8 for the two numbers alone, by 5e-5 with one; a third number
// changes nothing; torch's products of floats: 6e-6 and 1.5e-6).  Callers who accept half a step of the type in p - [label]
// (t2sp_xent_grad_rounded) have one: 8 T D V, 26.7 ms instead of 39.8 there.
//
// Weights of the tokens.  dloss[t] = top m 2^x with top = max |dloss| and 1/2 <= |m| < 1 is a factor of both products' reductions
// or rows.  p - [label] is stored times m 2^b, the rows of H for dW are copied times 2^a, exactly, with a + b = x + C for one C of
// all tokens; dH's rows are multiplied by top 2^(x - b) at the end, dW by top 2^-C.  Equal weights, the usual case, thus change no
// bit of either matrix (with dloss itself for top m 2^x, and m some fraction in p - [label], the gradients of a mean over 7700 tokens
// were off by 2.4e-6 in norm instead of 6e-7).  bfloat16 and float: b = 0.  half has
// room between 2^-24 and 2^16 only, so its b is 15 (the probabilities of a large vocabulary reach far below 1, and together
// the two numbers go down to 2^-40 of that) and C is the largest for which no copied element exceeds 2^15, or half of
// that.  A lighter token's a is smaller by d = its distance, as a power of two, from the token that decides C.  Up to d = 20 that
// costs no bits of elements down to 2^-8 of the row's largest; the next 10 are taken from b; then a falls further.  So weights (times
// the size of the row) down to 2^-30 of the heaviest keep their bits, below that elements underflow.  (With dloss / max |dloss|
// rounded into the copy, weights of 1e-6 of the heaviest put dW off by 2 %.)
// With p - [label] rounded to one number m goes into the copy of H instead, and into dH's rows at the end.
// The copy of H also holds zeros for tokens without a label: what their rows hold (padding may be anything) reaches
// no sum.
#include "product_core.hpp"
#include "product_host.hpp"

namespace t2sp {

struct XentArgs {
    const char *H, *W;
    const void *labels;
    int lab64;
    int T, V, D;
    int64_t ldh, ldw;                    // elements
    int row_tiles, col_tiles, xcds;
    float2 *part;                        // [col_tiles][T]: maximum of z over the tile's columns, sum of exp(z - maximum)
    float *hit;                          // [T]: z at the label
    // backward
    const float *lse, *dloss;
    const struct Common *common;         // see the weights of the tokens above
    const int *row_exp;                  // half only
    char *G;                             // [numbers][T][ldg] p - [label] times m 2^b of the piece, zeros from vp to ldg
    int64_t ldg;
    int numbers;                         // of the type that p - [label] is the sum of
    int v0, vp;                          // the piece: words v0 .. v0 + vp - 1
};

__device__ __forceinline__ int64_t label_of(const void *labels, int lab64, int t) {
    return lab64 ? static_cast<const int64_t *>(labels)[t] : (int64_t) static_cast<const int32_t *>(labels)[t];
}

constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
// What is taken from z before the exponential, for a maximum of `top`: 0 where that is infinite (no word, all words at -inf, or
// one at inf, whose sum is then inf).
__device__ __forceinline__ float base_of(float top) { return fabsf(top) < __builtin_inff() ? top : 0.f; }
// sum (of exponentials above `top`) on the scale of `base`.
__device__ __forceinline__ float rescaled(float sum, float top, float base) {
    return sum * exp_of((top == -__builtin_inff() ? base : top) - base);
}

// The tile of logits of rows m0.., words v0 + n0..
template <class P>
__device__ __forceinline__ void logits_tile(const XentArgs &g, int m0, int n0, char *smem, pv4f (&acc)[P::MT][P::NT]) {
    TileSource a, b;
    a.p = g.H + m0 * g.ldh * P::SZ;
    a.ld = (uint32_t)(g.ldh * P::SZ);
    a.count = g.T - m0;
    b.p = g.W + (g.v0 + n0) * g.ldw * P::SZ;
    b.ld = (uint32_t)(g.ldw * P::SZ);
    b.count = g.vp - n0;
    clear<P>(acc);
    product_run<P>(a, b, g.D, smem, acc);
}

template <class P>
__global__ void __launch_bounds__(P::THREADS) xent_stats_kernel(const XentArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int m0, n0;
    panel_tile(die_run(blockIdx.x, gridDim.x, g.xcds), g.row_tiles, g.col_tiles, &m0, &n0);
    const int tile = n0;
    m0 *= P::BM;
    n0 *= P::BN;
    pv4f acc[P::MT][P::NT];
    logits_tile<P>(g, m0, n0, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first_m = (wave / P::WN) * P::TM, n = n0 + (wave % P::WN) * P::TN + P::lane_column(lane);
    float2 *joint = reinterpret_cast<float2 *>(smem);        // [WN][BM]; the product is done with its LDS
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int m = first_m + 16 * i + (lane & 15);
        const bool row = m0 + m < g.T;
        const int64_t hot = row ? label_of(g.labels, g.lab64, m0 + m) : -1;
        float top = -__builtin_inff();
#pragma unroll
        for (int c = 0; c < P::LANE_N; c++) {
            const float z = acc[i][c / 4][c % 4];
            const int v = n + 8 * (c / 4) + c % 4;
            if (v < g.V) top = fmaxf(top, z);
            if (v == hot && v < g.V) g.hit[m0 + m] = z;
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float base = base_of(top);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < P::LANE_N; c++)
            if (n + 8 * (c / 4) + c % 4 < g.V) sum += exp_of(acc[i][c / 4][c % 4] - base);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 16) joint[(wave % P::WN) * P::BM + m] = make_float2(top, sum);
    }
    __syncthreads();
    for (int m = threadIdx.x; m < P::BM && m0 + m < g.T; m += P::THREADS) {
        float2 v[P::WN];
        float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (int w = 0; w < P::WN; w++) {
            v[w] = joint[w * P::BM + m];
            top = fmaxf(top, v[w].x);
        }
        const float base = base_of(top);
#pragma unroll
        for (int w = 0; w < P::WN; w++) sum += rescaled(v[w].y, v[w].x, base);
        g.part[(int64_t)tile * g.T + m0 + m] = make_float2(top, sum);
    }
}

// Joins the tiles' maxima and sums: 64 rows per workgroup, 16 waves that take every sixteenth tile.
constexpr int JOIN_WAVES = 16;
__global__ void __launch_bounds__(64 * JOIN_WAVES) xent_join_kernel(const float2 *part, const float *hit, const void *labels, int lab64, int T,
                                                                    int V, int tiles, float *loss, float *lse) {
    __shared__ float2 joint[JOIN_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x * 64 + lane;
    float top = -__builtin_inff(), sum = 0.f;
    auto add = [&](float m, float s) {
        const float to = fmaxf(top, m), base = base_of(to);
        sum = rescaled(sum, top, base) + rescaled(s, m, base);
        top = to;
    };
    if (t < T) {
#pragma unroll 8
        for (int c = wave; c < tiles; c += JOIN_WAVES) {
            const float2 v = part[(int64_t)c * T + t];
            add(v.x, v.y);
        }
    }
    joint[wave][lane] = make_float2(top, sum);
    __syncthreads();
    if (wave == 0 && t < T) {
#pragma unroll
        for (int w = 1; w < JOIN_WAVES; w++) add(joint[w][lane].x, joint[w][lane].y);
        const float l = top + logf(sum);
        const int64_t label = label_of(labels, lab64, t);
        const bool valid = label >= 0 && label < V;
        if (lse) lse[t] = l;
        loss[t] = valid ? l - hit[t] : 0.f;
    }
}

// The weights of the tokens (see above).
constexpr int NO_EXPONENT = -0x7fffffff - 1;         // of a row without a finite element but zeros
struct Common {
    float top;
    int c;
};
struct TokenWeight {
    float m;                                         // (dloss itself where it is 0 or not finite)
    int a, b, u;                                     // u = x - b
};
template <class T>
__device__ __forceinline__ TokenWeight token_weight(float dloss, const int *row_exp, int t, Common common) {
    if (dloss == 0.f || !(fabsf(dloss) < __builtin_inff())) return {dloss, 0, 0, 0};
    int x;
    const float m = frexpf(dloss / common.top, &x);
    if constexpr (!std::is_same_v<T, _Float16>) return {m, x + common.c, 0, x};
    const int e = row_exp[t];
    if (e == NO_EXPONENT) return {m, 0, 15, x - 15};
    const int lighter = 30 - e - x - common.c, b = 15 - (lighter <= 20 ? 0 : lighter <= 30 ? lighter - 20 : 10);
    return {m, x + common.c - b, b, x - b};
}

// row_exp[t] = e: the largest finite |H[t, :]| is in 2^(e - 1) .. 2^e.  One wave per token.
__global__ void __launch_bounds__(256) xent_row_exponents_kernel(const _Float16 *H, int64_t ldh, int rows, int D, int *row_exp) {
    const int lane = threadIdx.x & 63;
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < rows; t += (int64_t)gridDim.x * 4) {
        const _Float16 *h = H + t * ldh;
        float top = 0.f;
        auto take = [&](_Float16 v) {
            const float f = fabsf((float)v);
            top = f < __builtin_inff() ? fmaxf(top, f) : top;
        };
        const int whole = D / 8 * 8;
        for (int c = lane * 8; c < whole; c += 512) {
            const Chunk<_Float16>::type v = *reinterpret_cast<const Chunk<_Float16>::anywhere *>(h + c);
#pragma unroll
            for (int j = 0; j < 8; j++) take(v[j]);
        }
        if (whole + lane < D) take(h[whole + lane]);
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
        int e = NO_EXPONENT;
        if (top > 0.f) frexpf(top, &e);
        if (lane == 0) row_exp[t] = e;
    }
}

// top and C, from the tokens with a label and a finite weight other than 0; in every thread of a workgroup.  The exponent of dloss / top
// is at most one more than the difference of the two exponents: with that half's C is found in the same pass over the tokens as top.
template <class T, int THREADS>
__device__ __forceinline__ Common common_weight(const float *dloss, const void *labels, int lab64, const int *row_exp, int rows, int V) {
    constexpr int WAVES = THREADS / 64, NONE = 0x7fffffff;
    __shared__ float tops[WAVES];
    __shared__ int joint[WAVES];
    float top = 0.f;
    int least = NONE;
    for (int t = threadIdx.x; t < rows; t += THREADS) {
        const int64_t label = label_of(labels, lab64, t);
        const float v = fabsf(dloss[t]);
        if (label < 0 || label >= V || !(v > 0.f && v < __builtin_inff())) continue;
        top = fmaxf(top, v);
        if constexpr (std::is_same_v<T, _Float16>) {
            int x;
            frexpf(v, &x);
            if (const int e = row_exp[t]; e != NO_EXPONENT) least = min(least, 30 - e - x);
        }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        top = fmaxf(top, __shfl_xor(top, m, 64));
        least = min(least, __shfl_xor(least, m, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x >> 6] = top;
        joint[threadIdx.x >> 6] = least;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        top = fmaxf(top, tops[w]);
        least = min(least, joint[w]);
    }
    if (!std::is_same_v<T, _Float16>) return {top, -1};
    int x;
    frexpf(top, &x);
    return {top, least == NONE ? 0 : least + x - 1};
}
template <class T>
__global__ void __launch_bounds__(1024) xent_common_kernel(const float *dloss, const void *labels, int lab64, const int *row_exp, int rows, int V,
                                                           Common *common) {
    const Common c = common_weight<T, 1024>(dloss, labels, lab64, row_exp, rows, V);
    if (threadIdx.x == 0) *common = c;
}

// Hz[t, :] = 2^a H[t, :] (one number: times m), zeros for tokens without a label and from D to ld.
// FIND: the workgroups look for top and C themselves, for the kernels behind too (up to FIND_ROWS tokens; a launch less, about 3 us
// of the host's time).
constexpr int FIND_ROWS = 2048;
template <class T, bool FIND>
__global__ void __launch_bounds__(256) xent_weighted_rows_kernel(const T *H, int64_t ldh, const void *labels, int lab64, const float *dloss,
                                                                 const int *row_exp, Common *common, int numbers, int rows, int V, int D, T *Hz,
                                                                 int64_t ld, int64_t chunks) {
    constexpr int CE = 16 / sizeof(T);
    typedef T chunk __attribute__((ext_vector_type(CE)));
    const int64_t per = ld / CE;
    const Common c0 = FIND ? common_weight<T, 256>(dloss, labels, lab64, row_exp, rows, V) : *common;
    if (FIND && blockIdx.x == 0 && threadIdx.x == 0) *common = c0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / per), c = (int)(i % per) * CE;
        const int64_t label = label_of(labels, lab64, t);
        chunk v;
        if (label >= 0 && label < V) {
            const TokenWeight w = token_weight<T>(dloss[t], row_exp, t, c0);
            const float m = sizeof(T) == 2 && numbers == 1 ? w.m : 1.f;
            const T *s = H + t * ldh + c;
            if (c + CE <= D) {
                v = *reinterpret_cast<const typename Chunk<T>::anywhere *>(s);
            } else {
#pragma unroll
                for (int j = 0; j < CE; j++) v[j] = c + j < D ? s[j] : (T)0.f;
            }
#pragma unroll
            for (int j = 0; j < CE; j++) v[j] = (T)ldexpf((float)v[j] * m, w.a);
        } else {
#pragma unroll
            for (int j = 0; j < CE; j++) v[j] = (T)0.f;
        }
        *reinterpret_cast<chunk *>(Hz + i * CE) = v;
    }
}

template <class P>
__global__ void __launch_bounds__(P::THREADS) xent_probabilities_kernel(const XentArgs g) {
    using T = typename P::T;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int m0, n0;
    panel_tile(die_run(blockIdx.x, gridDim.x, g.xcds), g.row_tiles, g.col_tiles, &m0, &n0);
    m0 *= P::BM;
    n0 *= P::BN;
    pv4f acc[P::MT][P::NT];
    logits_tile<P>(g, m0, n0, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Common common = *g.common;
    const int n = n0 + (wave % P::WN) * P::TN + P::lane_column(lane);
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int t = m0 + (wave / P::WN) * P::TM + 16 * i + (lane & 15);
        if (t >= g.T) continue;
        const int64_t label = label_of(g.labels, g.lab64, t);
        const bool valid = label >= 0 && label < g.V;
        const float lse = g.lse[t];
        const TokenWeight w = token_weight<T>(valid ? g.dloss[t] : 0.f, g.row_exp, t, common);
        const float weight = ldexpf(sizeof(T) == 2 && g.numbers == 1 ? 1.f : w.m, w.b);
        const int64_t hot = label - g.v0;
#pragma unroll
        for (int c = 0; c < P::LANE_N; c++) {
            const int v = n + 8 * (c / 4) + c % 4;
            const float p = exp_of(acc[i][c / 4][c % 4] - lse) - (v == hot ? 1.f : 0.f);
            acc[i][c / 4][c % 4] = valid && v < g.vp ? p * weight : 0.f;
        }
        char *row = g.G + t * g.ldg * (int64_t)sizeof(T);
        for (int j = 0; j < g.numbers; j++, row += g.T * g.ldg * (int64_t)sizeof(T)) {
            store_row<P, T>(row, n0 + (wave % P::WN) * P::TN, (int)g.ldg, acc[i]);
#pragma unroll
            for (int c = 0; c < P::LANE_N; c++) acc[i][c / 4][c % 4] -= (float)(T)acc[i][c / 4][c % 4];
        }
    }
}

struct XentProductArgs {
    const char *A, *B;
    char *out;
    int64_t lda, ldb, ldo;               // elements
    int rows, cols, k;                   // of the result; the reduction
    int numbers;                         // matrices that A is the sum of, `next` bytes apart
    int64_t next;
    int a_cols, b_cols;                  // elements in a row of A (dW) and B, whole 16-byte chunks
    int row_tiles, col_tiles, xcds;
    const Common *common;                // dW
    int splits;                          // the reduction in this many parts, each (dW: if more than one) with a plane of floats
    int64_t plane;
    int add;                             // dH: add to the planes (a later piece of the vocabulary)
};

// dW[v0 + m, n] = top 2^-C sum_t G[t, m] Hz[t, n], or one of several planes with the sums over part of the tokens
template <class P, class O>
__global__ void __launch_bounds__(P::THREADS) xent_dw_kernel(const XentProductArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int m0, n0;
    const unsigned at = die_run(blockIdx.x, gridDim.x, g.xcds), tiles = (unsigned)g.row_tiles * g.col_tiles, s = at / tiles;
    panel_tile(at % tiles, g.row_tiles, g.col_tiles, &m0, &n0);
    m0 *= P::BM;
    n0 *= P::BN;
    const int stages = (g.k + P::KS - 1) / P::KS, per = (stages + g.splits - 1) / g.splits * P::KS;
    const int k0 = (int64_t)s * per < g.k ? (int)s * per : g.k, k = g.k - k0 < per ? g.k - k0 : per;
    TileSource a{g.A + (k0 * g.lda + m0) * P::SZ, (uint32_t)(g.lda * P::SZ), g.a_cols - m0};
    const TileSource b{g.B + (k0 * g.ldb + n0) * P::SZ, (uint32_t)(g.ldb * P::SZ), g.b_cols - n0};
    pv4f acc[P::MT][P::NT];
    clear<P>(acc);
    if (k > 0)
        for (int i = 0; i < g.numbers; i++, a.p += g.next) product_run<P>(a, b, k, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + (wave % P::WN) * P::TN;
    const Common by = *g.common;
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int m = m0 + (wave / P::WN) * P::TM + 16 * i + (lane & 15);
        if (m >= g.rows) continue;
#pragma unroll
        for (int j = 0; j < P::NT; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[i][j][c] = by.top * ldexpf(acc[i][j][c], -by.c);
        store_row<P, O>(g.out + (s * g.plane + m * g.ldo) * (int64_t)sizeof(O), n, g.cols, acc[i]);
    }
}

// plane[s][t, n] (+)= sum over part s of the piece's words: G[t, v] W[v0 + v, n]
template <class P>
__global__ void __launch_bounds__(P::THREADS) xent_dh_kernel(const XentProductArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const unsigned at = die_run(blockIdx.x, gridDim.x, g.xcds), tiles = (unsigned)g.row_tiles * g.col_tiles, s = at / tiles;
    int m0, n0;
    panel_tile(at % tiles, g.row_tiles, g.col_tiles, &m0, &n0);
    m0 *= P::BM;
    n0 *= P::BN;
    const int stages = (g.k + P::KS - 1) / P::KS, per = (stages + g.splits - 1) / g.splits * P::KS;
    const int k0 = (int64_t)s * per < g.k ? (int)s * per : g.k, k = g.k - k0 < per ? g.k - k0 : per;
    TileSource a{g.A + (m0 * g.lda + k0) * P::SZ, (uint32_t)(g.lda * P::SZ), g.rows - m0};
    const TileSource b{g.B + (k0 * g.ldb + n0) * P::SZ, (uint32_t)(g.ldb * P::SZ), g.b_cols - n0};
    pv4f acc[P::MT][P::NT];
    clear<P>(acc);
    if (k > 0)
        for (int i = 0; i < g.numbers; i++, a.p += g.next) product_run<P>(a, b, k, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = n0 + (wave % P::WN) * P::TN;
#pragma unroll
    for (int i = 0; i < P::MT; i++) {
        const int m = m0 + (wave / P::WN) * P::TM + 16 * i + (lane & 15);
        if (m >= g.rows) continue;
        float *row = reinterpret_cast<float *>(g.out) + s * g.plane + m * g.ldo;
        row_chunks<P, float>(n, acc[i], [&](int col, pv4f v) {
            if (col >= g.ldo) return;                    // (planes have rows of whole 16-byte chunks)
            pv4f *p = reinterpret_cast<pv4f *>(row + col);
            *p = g.add ? *p + v : v;
        });
    }
}

// dH[t, n] = top 2^(x - b) (one number: m) sum_s plane[s][t, n], zeros for tokens without a label.
template <class T, class O>
__global__ void __launch_bounds__(256) xent_dh_join_kernel(const float *planes, int splits, int64_t plane, int64_t ld, const void *labels, int lab64,
                                                           const float *dloss, const int *row_exp, const Common *common, int numbers, int V, int D, O *dH, int64_t ldo,
                                                          int64_t chunks) {
    const int64_t per = ld / 4;
    typedef O quad __attribute__((ext_vector_type(4)));
    typedef O quad_anywhere __attribute__((ext_vector_type(4), aligned(sizeof(O))));
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / per), n = (int)(i % per) * 4;
        const int64_t label = label_of(labels, lab64, t);
        pv4f sum = pv4f{0.f, 0.f, 0.f, 0.f};
        if (label >= 0 && label < V) {
#pragma unroll 4
            for (int s = 0; s < splits; s++) sum += *reinterpret_cast<const pv4f *>(planes + s * plane + t * ld + n);
            const TokenWeight w = token_weight<T>(dloss[t], row_exp, t, *common);
            const float by = common->top * (sizeof(T) == 2 && numbers == 1 ? w.m : 1.f);
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] = by * ldexpf(sum[j], w.u);
        }
        O *o = dH + t * ldo + n;
        if (n + 4 <= D) {
            *reinterpret_cast<quad_anywhere *>(o) = __builtin_convertvector(sum, quad);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (n + j < D) o[j] = (O)sum[j];
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches
// What a call passes through its workspace, in this order (every part starts on 256 bytes).
struct XentRoom {
    size_t h, w;                         // padded copies of H and W (0: read where they lie)
    size_t part, hit;                    // forward
    size_t common, row_exp, hz, g, planes, dw;     // backward
    size_t total;
    int64_t ldd;                         // elements per row of hz and of the planes
    int piece, splits, dw_parts;
};

constexpr size_t ROOM_ALIGN = 256;
constexpr int64_t G_BYTES = 128 << 20;   // of the piece of p - [label]: it then stays in the 256 MB cache between its
                                         // kernel and the two products that read it ...
constexpr int MIN_PIECE = 4096;          // ... but a piece is long enough that adding up dH costs little beside it (beyond 8192
                                         // tokens it is therefore larger than G_BYTES: 2 GB at 131072 tokens)
// Numbers of the type that p - [label] takes.
static int numbers_of(int type, bool rounded) { return type_bytes(type) == 2 && !rounded ? 2 : 1; }

// The tile of the logits; 65536 exponentials are worth four stages (777 x 50001 x 1022, half: 129 us in 256 x 256 tiles, 120 in
// 128 x 128; 2048 x 32000 x 2048, bfloat16: 238 us in 256 x 256 tiles).
static int logits_shape(int64_t T, int64_t V, int64_t D, int size) { return pick_tile(1, T, V, D, size, true, 4); }
// Columns of the forward pass's tile.
static int tile_cols(int tile, int size) { return tile == 64 && size == 2 ? 128 : tile; }

// The tile of dH (the rows of T decide: its columns and the split fill the chip) and the parts of its reduction.
static int dh_tile(int T, int size) { return T > 128 && size == 2 ? 256 : T > 64 ? 128 : 64; }
static int dh_splits(int T, int D, int piece, int size, int numbers) {
    if (T == 0) return 1;
    const int bm = dh_tile(T, size), bn = tile_cols(bm, size), per_cu = bm == 256 ? 1 : bm == 128 ? 2 : 3;
    const int64_t tiles = (int64_t)((T + bm - 1) / bm) * ((D + bn - 1) / bn), slots = (int64_t)machine().cus * per_cu;
    const TileShape &s = size == 4 ? (bm == 128 ? SHAPE_128F : SHAPE_64F) : bm == 256 ? SHAPE_256 : bm == 128 ? SHAPE_128 : SHAPE_64;
    return split_parts(tiles, slots, (double)piece * size * numbers / 64, s.a + s.c * per_cu, 4.0 * T * D);
}
// The parts that the sums over tokens are cut into when dW has few tiles.  (Both gradients and the loss of 3155 tokens, 64 wide, 709
// words, float: 297 us whole, 74 in parts)
static int dw_splits(int T, int D, int piece, int size, int numbers) {
    const TileShape &s = size == 2 ? SHAPE_128 : SHAPE_128F;
    const int64_t tiles = (int64_t)((piece + 127) / 128) * ((D + 127) / 128);
    return split_parts(tiles, machine().cus, (double)T * size * numbers / 64, s.a + s.c, 4.0 * piece * D);
}

static int dw_tile(int T, int D, int piece, int size, int numbers) { return pick_tile(1, piece, D, (int64_t)T * numbers, size, false); }

static XentRoom xent_room(bool backward, int numbers, int type, const void *H, const void *W, int T, int V, int D, int64_t ldh, int64_t ldw) {
    const int size = type_bytes(type);
    XentRoom r{};
    r.ldd = padded_cols(D, size);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, ROOM_ALIGN);
        return here;
    };
    r.h = loadable(H, ldh, D, size) ? (size_t)-1 : take((size_t)T * r.ldd * size);
    r.w = loadable(W, ldw, D, size) ? (size_t)-1 : take((size_t)V * r.ldd * size);
    if (!backward) {
        const int cols = tile_cols(logits_shape(T, V, D, size), size);
        r.part = take((size_t)((V + cols - 1) / cols) * T * sizeof(float2));
        r.hit = take((size_t)T * sizeof(float));
    } else {
        int64_t piece = G_BYTES / ((int64_t)(T > 0 ? T : 1) * size * numbers) / 256 * 256;
        if (piece < MIN_PIECE) piece = MIN_PIECE;
        if (piece >= V) piece = V;
        else piece = round_up((V + (V + piece - 1) / piece - 1) / ((V + piece - 1) / piece), 256);     // equal pieces
        r.piece = (int)piece;
        r.splits = dh_splits(T, D, r.piece, size, numbers);
        r.common = take(sizeof(Common));
        r.row_exp = take(type == T2SP_TYPE_F16 ? (size_t)T * sizeof(int) : 0);
        r.hz = take((size_t)T * r.ldd * size);
        r.g = take((size_t)T * padded_cols(piece, size) * size * numbers);
        r.planes = take((size_t)r.splits * T * r.ldd * sizeof(float));
        r.dw_parts = dw_splits(T, D, r.piece, size, numbers);
        r.dw = take(r.dw_parts > 1 ? (size_t)r.dw_parts * r.piece * r.ldd * sizeof(float) : 0);
    }
    r.total = at;
    return r;
}

static bool xent_args_ok(int type, int T, int V, int D, int64_t ldh, int64_t ldw) {
    const int size = type_bytes(type);
    return size && T >= 0 && T <= T2SP_MAX_EXTENT && extent_ok(V) && row_ok(D, size) && stride_ok(ldh) && stride_ok(ldw) && ldh >= D && ldw >= D;
}

// Padded copies of the operands that need one; sets the pointers and leading dimensions of g.
static int xent_operands(XentArgs &g, const XentRoom &r, int size, char *room, const void *H, const void *W, int64_t ldh, int64_t ldw,
                         hipStream_t st) {
    g.H = static_cast<const char *>(H); g.W = static_cast<const char *>(W);
    g.ldh = ldh; g.ldw = ldw;
    PadRows ph{}, pw{};
    if (r.h != (size_t)-1) {
        ph = {H, room + r.h, 1, g.T, g.D, ldh, 0};
        g.H = room + r.h; g.ldh = r.ldd;
    }
    if (r.w != (size_t)-1) {
        pw = {W, room + r.w, 1, g.V, g.D, ldw, 0};
        g.W = room + r.w; g.ldw = r.ldd;
    }
    return launch_pad_rows(ph, pw, size, st);
}

#define T2SP_LAUNCH_TILES(P, kern, blocks, st, g)                                              \
    do {                                                                                       \
        const int64_t b_ = (blocks);                                                           \
        if (b_ > 0x7fffffff / P::THREADS) return T2SP_ERR_SHAPE;                               \
        auto k_ = kern;                                                                        \
        if (allow_lds(k_, P::LDS)) return T2SP_ERR_LAUNCH;                                     \
        hipLaunchKernelGGL(k_, dim3((unsigned)b_), dim3(P::THREADS), P::LDS, st, g);           \
        return launched();                                                                     \
    } while (0)

template <class P> static int launch_stats(XentArgs g, hipStream_t st) {
    g.row_tiles = (g.T + P::BM - 1) / P::BM;
    g.col_tiles = (g.V + P::BN - 1) / P::BN;
    T2SP_LAUNCH_TILES(P, xent_stats_kernel<P>, (int64_t)g.row_tiles * g.col_tiles, st, g);
}
template <class P> static int launch_probabilities(XentArgs g, hipStream_t st) {
    g.row_tiles = (g.T + P::BM - 1) / P::BM;
    g.col_tiles = (g.vp + P::BN - 1) / P::BN;
    T2SP_LAUNCH_TILES(P, xent_probabilities_kernel<P>, (int64_t)g.row_tiles * g.col_tiles, st, g);
}
template <class P, class O> static int launch_dw(XentProductArgs g, hipStream_t st) {
    g.row_tiles = (g.rows + P::BM - 1) / P::BM;
    g.col_tiles = (g.cols + P::BN - 1) / P::BN;
    T2SP_LAUNCH_TILES(P, (xent_dw_kernel<P, O>), (int64_t)g.row_tiles * g.col_tiles * g.splits, st, g);
}
template <class P> static int launch_dh(XentProductArgs g, hipStream_t st) {
    g.row_tiles = (g.rows + P::BM - 1) / P::BM;
    g.col_tiles = (g.cols + P::BN - 1) / P::BN;
    T2SP_LAUNCH_TILES(P, xent_dh_kernel<P>, (int64_t)g.row_tiles * g.col_tiles * g.splits, st, g);
}
#undef T2SP_LAUNCH_TILES

// The largest tile of a type (the choices above take 256 x 256 for 16-bit elements only).
template <class T, int AS, int BS> using Large = std::conditional_t<sizeof(T) == 2, Tile256<T, AS, BS>, Tile128<T, AS, BS>>;

template <class T>
static int xent_forward(XentArgs g, float *loss, float *lse, hipStream_t st) {
    const int tile = logits_shape(g.T, g.V, g.D, sizeof(T)), cols = tile_cols(tile, sizeof(T));
    int err = tile == 256 ? launch_stats<Large<T, KMAJOR, KMAJOR>>(g, st)
                          : tile == 128 ? launch_stats<Tile128<T, KMAJOR, KMAJOR>>(g, st) : launch_stats<Tile64<T, KMAJOR>>(g, st);
    if (err) return err;
    const int tiles = (g.V + cols - 1) / cols;
    hipLaunchKernelGGL(xent_join_kernel, dim3((g.T + 63) / 64), dim3(64 * JOIN_WAVES), 0, st, g.part, g.hit, g.labels, g.lab64, g.T, g.V, tiles,
                       loss, lse);
    return launched();
}

template <class T, class O>
static int xent_backward(XentArgs g, const XentRoom &r, char *room, const void *H, int64_t ldh, void *dH, void *dW, int out_type, int64_t lddh,
                         int64_t lddw, hipStream_t st) {
    constexpr int size = sizeof(T);
    float *planes = reinterpret_cast<float *>(room + r.planes);
    Common *common = reinterpret_cast<Common *>(room + r.common);
    int *row_exp = reinterpret_cast<int *>(room + r.row_exp);
    int err;
    g.common = common; g.row_exp = row_exp;
    if constexpr (std::is_same_v<T, _Float16>)
        if (g.T) {
            hipLaunchKernelGGL(xent_row_exponents_kernel, dim3((unsigned)std::min((g.T + 3) / 4, 16384)), dim3(256), 0, st, static_cast<const T *>(H), ldh,
                               g.T, g.D, row_exp);
            if ((err = launched())) return err;
        }
    const int64_t chunks = dW ? (int64_t)g.T * r.ldd * size / 16 : 0;
    const bool find = chunks && g.T <= FIND_ROWS;
    if (!find) {
        hipLaunchKernelGGL(xent_common_kernel<T>, dim3(1), dim3(1024), 0, st, g.dloss, g.labels, g.lab64, row_exp, g.T, g.V, common);
        if ((err = launched())) return err;
    }
    if (chunks) {
        auto kern = find ? xent_weighted_rows_kernel<T, true> : xent_weighted_rows_kernel<T, false>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(chunks < 256 * 16384 ? (chunks + 255) / 256 : 16384)), dim3(256), 0, st,
                           static_cast<const T *>(H), ldh, g.labels, g.lab64, g.dloss, row_exp, common, g.numbers, g.T, g.V, g.D,
                           reinterpret_cast<T *>(room + r.hz), r.ldd, chunks);
        if ((err = launched())) return err;
    }
    for (int v0 = 0; v0 < g.V; v0 += r.piece) {
        g.v0 = v0;
        g.vp = g.V - v0 < r.piece ? g.V - v0 : r.piece;
        g.G = room + r.g;
        g.ldg = padded_cols(g.vp, size);
        if (g.T) {
            const int tile = logits_shape(g.T, g.vp, g.D, size);
            err = tile == 256 ? launch_probabilities<Large<T, KMAJOR, KMAJOR>>(g, st)
                              : tile == 128 ? launch_probabilities<Tile128<T, KMAJOR, KMAJOR>>(g, st) : launch_probabilities<Tile64<T, KMAJOR>>(g, st);
            if (err) return err;
        }
        XentProductArgs p{};
        p.xcds = g.xcds;
        if (dW) {
            p.A = g.G; p.lda = g.ldg; p.a_cols = (int)g.ldg;
            p.B = room + r.hz; p.ldb = r.ldd; p.b_cols = (int)r.ldd;
            p.out = static_cast<char *>(dW) + v0 * lddw * (int64_t)sizeof(O); p.ldo = lddw;
            p.rows = g.vp; p.cols = g.D; p.k = g.T;
            p.numbers = g.numbers; p.next = g.T * g.ldg * (int64_t)size;
            p.common = common;
            p.splits = r.dw_parts;
            if (r.dw_parts > 1) {
                char *const out = p.out;
                p.out = room + r.dw; p.ldo = r.ldd; p.plane = p.rows * p.ldo;
                if (!(err = launch_dw<Tile128<T, KROWS, KROWS>, float>(p, st)))
                    err = launch_join_planes(reinterpret_cast<const float *>(room + r.dw), p.splits, 1, p.rows, p.cols, p.ldo, out, out_type, lddw, 0, st);
            } else {
                err = dw_tile(p.k, p.cols, p.rows, size, p.numbers) == 256 ? launch_dw<Large<T, KROWS, KROWS>, O>(p, st)
                                                                           : launch_dw<Tile128<T, KROWS, KROWS>, O>(p, st);
            }
            if (err) return err;
        }
        if (dH && g.T) {
            p.A = g.G; p.lda = g.ldg;
            p.B = g.W + v0 * g.ldw * size; p.ldb = g.ldw; p.b_cols = (int)r.ldd;
            p.out = reinterpret_cast<char *>(planes); p.ldo = r.ldd; p.plane = (int64_t)g.T * r.ldd;
            p.rows = g.T; p.cols = g.D; p.k = g.vp;
            p.numbers = g.numbers; p.next = g.T * g.ldg * (int64_t)size;
            p.splits = r.splits; p.add = v0 > 0;
            const int tile = dh_tile(g.T, size);
            err = tile == 256 ? launch_dh<Large<T, KMAJOR, KROWS>>(p, st)
                              : tile == 128 ? launch_dh<Tile128<T, KMAJOR, KROWS>>(p, st) : launch_dh<Tile64<T, KROWS>>(p, st);
            if (err) return err;
        }
    }
    if (dH && g.T) {
        const int64_t quads = (int64_t)g.T * r.ldd / 4;
        hipLaunchKernelGGL((xent_dh_join_kernel<T, O>), dim3((unsigned)(quads < 256 * 16384 ? (quads + 255) / 256 : 16384)), dim3(256), 0, st, planes,
                           r.splits, (int64_t)g.T * r.ldd, r.ldd, g.labels, g.lab64, g.dloss, row_exp, common, g.numbers, g.V, g.D, static_cast<O *>(dH), lddh, quads);
        return launched();
    }
    return T2SP_OK;
}

}  // namespace t2sp

using namespace t2sp;

extern "C" size_t t2sp_xent_workspace_bytes(int type, const void *H, const void *W, int T, int V, int D, int64_t ldh, int64_t ldw) {
    if (!xent_args_ok(type, T, V, D, ldh, ldw)) return 0;
    return xent_room(false, 1, type, H, W, T, V, D, ldh, ldw).total;
}

extern "C" int t2sp_xent(int type, const void *H, const void *W, const void *labels, int label_bits, float *loss, float *lse, int T, int V, int D,
                         int64_t ldh, int64_t ldw, void *workspace, size_t workspace_bytes, void *stream) {
    if (!xent_args_ok(type, T, V, D, ldh, ldw) || (label_bits != 32 && label_bits != 64)) return T2SP_ERR_SHAPE;
    if (T == 0) return T2SP_OK;
    if (!H || !W || !labels || !loss) return T2SP_ERR_SHAPE;
    const XentRoom r = xent_room(false, 1, type, H, W, T, V, D, ldh, ldw);
    if (!workspace || workspace_bytes < r.total || reinterpret_cast<uintptr_t>(workspace) % 16) return T2SP_ERR_SHAPE;
    const hipStream_t st = (hipStream_t)stream;
    char *room = static_cast<char *>(workspace);
    XentArgs g{};
    g.labels = labels; g.lab64 = label_bits == 64;
    g.T = T; g.V = V; g.D = D; g.vp = V;
    g.xcds = machine().xcds;
    g.part = reinterpret_cast<float2 *>(room + r.part);
    g.hit = reinterpret_cast<float *>(room + r.hit);
    if (int err = xent_operands(g, r, type_bytes(type), room, H, W, ldh, ldw, st)) return err;
    return with_types(type, type, [&](auto *t, auto *) { return xent_forward<std::remove_pointer_t<decltype(t)>>(g, loss, lse, st); });
}

extern "C" size_t t2sp_xent_grad_workspace_bytes(int type, const void *H, const void *W, int T, int V, int D, int64_t ldh, int64_t ldw) {
    if (!xent_args_ok(type, T, V, D, ldh, ldw)) return 0;
    const size_t full = xent_room(true, numbers_of(type, false), type, H, W, T, V, D, ldh, ldw).total;
    return std::max(full, xent_room(true, numbers_of(type, true), type, H, W, T, V, D, ldh, ldw).total);
}

static int xent_gradients(bool rounded, int type, int out_type, const void *H, const void *W, const void *labels, int label_bits, const float *lse,
                          const float *dloss, void *dH, void *dW, int T, int V, int D, int64_t ldh, int64_t ldw, int64_t lddh, int64_t lddw,
                          void *workspace, size_t workspace_bytes, void *stream) {
    if (!xent_args_ok(type, T, V, D, ldh, ldw) || !out_type_ok(type, out_type) || (label_bits != 32 && label_bits != 64) || !stride_ok(lddh) ||
        !stride_ok(lddw) || (dH && lddh < D) || (dW && lddw < D))
        return T2SP_ERR_SHAPE;
    if ((!dH && !dW) || (T == 0 && !dW)) return T2SP_OK;
    if (T && (!H || !W || !labels || !lse || !dloss)) return T2SP_ERR_SHAPE;
    const XentRoom r = xent_room(true, numbers_of(type, rounded), type, H, W, T, V, D, ldh, ldw);
    if (!workspace || workspace_bytes < r.total || reinterpret_cast<uintptr_t>(workspace) % 16) return T2SP_ERR_SHAPE;
    const hipStream_t st = (hipStream_t)stream;
    char *room = static_cast<char *>(workspace);
    XentArgs g{};
    g.labels = labels; g.lab64 = label_bits == 64;
    g.T = T; g.V = V; g.D = D;
    g.xcds = machine().xcds;
    g.lse = lse; g.dloss = dloss;
    g.numbers = numbers_of(type, rounded);
    if (T)
        if (int err = xent_operands(g, r, type_bytes(type), room, H, W, ldh, ldw, st)) return err;
    return with_types(type, out_type, [&](auto *t, auto *o) {
        return xent_backward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>>(g, r, room, H, ldh, dH, dW, out_type, lddh, lddw, st);
    });
}

extern "C" int t2sp_xent_grad(int type, int out_type, const void *H, const void *W, const void *labels, int label_bits, const float *lse,
                              const float *dloss, void *dH, void *dW, int T, int V, int D, int64_t ldh, int64_t ldw, int64_t lddh, int64_t lddw,
                              void *workspace, size_t workspace_bytes, void *stream) {
    return xent_gradients(false, type, out_type, H, W, labels, label_bits, lse, dloss, dH, dW, T, V, D, ldh, ldw, lddh, lddw, workspace,
                          workspace_bytes, stream);
}
extern "C" int t2sp_xent_grad_rounded(int type, int out_type, const void *H, const void *W, const void *labels, int label_bits, const float *lse,
                                      const float *dloss, void *dH, void *dW, int T, int V, int D, int64_t ldh, int64_t ldw, int64_t lddh,
                                      int64_t lddw, void *workspace, size_t workspace_bytes, void *stream) {
    return xent_gradients(true, type, out_type, H, W, labels, label_bits, lse, dloss, dH, dW, T, V, D, ldh, ldw, lddh, lddw, workspace,
                          workspace_bytes, stream);
}

extern "C" int t2sp_xent_plan(int type, int T, int V, int D) {
    return xent_args_ok(type, T, V, D, D, D) && T ? logits_shape(T, V, D, type_bytes(type)) : T2SP_ERR_SHAPE;
}
extern "C" int t2sp_xent_grad_plan(int type, int rounded, int T, int V, int D, int *out5) {
    if (!xent_args_ok(type, T, V, D, D, D) || !T || !out5) return T2SP_ERR_SHAPE;
    const int size = type_bytes(type), numbers = numbers_of(type, rounded);
    const XentRoom r = xent_room(true, numbers, type, nullptr, nullptr, T, V, D, D, D);
    out5[0] = logits_shape(T, r.piece, D, size);
    out5[1] = dh_tile(T, size);
    out5[2] = r.splits;
    out5[3] = r.dw_parts > 1 ? 128 : dw_tile(T, D, r.piece, size, numbers);
    out5[4] = r.dw_parts;
    return r.piece;
}
