// product_host.hpp — what the launchers of the 16/32-bit product operators (grouped.hip, xent.hip, gemv_w4.hip) share:
// element types, checks of arguments, and the padded copies of operands that the 16-byte loaders cannot take.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "machine.hpp"
#include "t2sp_hip.h"

namespace t2sp {

inline int type_bytes(int type) {
    return type == T2SP_TYPE_F32 ? 4 : type == T2SP_TYPE_F16 || type == T2SP_TYPE_BF16 ? 2 : 0;
}
inline bool out_type_ok(int type, int out_type) { return out_type == type || out_type == T2SP_TYPE_F32; }
inline bool extent_ok(int64_t e) { return e >= 1 && e <= T2SP_MAX_EXTENT; }
inline bool stride_ok(int64_t s) { return s >= 0 && stride_in_range(s); }

// Rows of a matrix the loaders of product_core.hpp can read where they lie: 16-byte chunks along the contiguous
// dimension, lane offsets of up to 255 rows inside 31 bits.
inline bool loadable(const void *p, int64_t ld, int64_t cols, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0 && cols * size % 16 == 0 && ld * size <= T2SP_MAX_ROW_BYTES;
}
// Extents along which elements are contiguous: a (padded) row within the loaders' reach.
inline bool row_ok(int64_t e, int size) { return e >= 1 && e * size <= T2SP_MAX_ROW_BYTES; }
// Elements per row of a padded copy.
inline int64_t padded_cols(int64_t cols, int size) { return (cols * size + 15) / 16 * 16 / size; }
inline size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// dst[b][r][0 .. padded) = src[b][r][0 .. cols), zeros behind: dense rows of whole 16-byte chunks.  Two copies in one launch; one
// that is not needed has no rows.
struct PadRows {
    const void *src;
    void *dst;
    int64_t batch, rows, cols, ld, batch_stride;
};
int launch_pad_rows(const PadRows &a, const PadRows &b, int size, hipStream_t stream);

// out[e][r][0 .. cols) = sum over parts of plane[part][e * rows + r][0 .. cols), in their order; rows of planes have ldp elements, a
// multiple of four.
int launch_join_planes(const float *planes, int parts, int64_t batch, int64_t rows, int64_t cols, int64_t ldp, void *out, int out_type,
                       int64_t ldo, int64_t batch_stride, hipStream_t stream);

template <class K> int allow_lds(K kern, int bytes) {
    if (bytes <= 64 * 1024) return T2SP_OK;
    return hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? T2SP_OK
                                                                                                               : T2SP_ERR_LAUNCH;
}
// Time in microseconds of a product in tiles, for choosing among tile shapes: `tiles` workgroups share the CUs, n to a
// CU, and a stage of 64 bytes of k then takes a + c n (fitted to sweeps of 1 to 4096 rows,
// k 512 to 4096, 1000 to 20000 columns; what it picks is within a tenth of the best shape there but for a few sizes at the borders).
struct TileShape {
    int rows, cols;
    double a, c;
    int ends = 4;
};
constexpr TileShape SHAPE_256{256, 256, -0.1, 0.75, 10}, SHAPE_128{128, 128, 0.1, 0.28, 7}, SHAPE_64{64, 128, 0.08, 0.205, 4};
constexpr TileShape SHAPE_128F{128, 128, 0.1, 1.02}, SHAPE_64F{64, 64, 0.12, 0.285};
inline double tiles_cost(const TileShape &s, int64_t tiles, int64_t k_bytes) {
    const int64_t cus = machine().cus, n = (tiles + cus - 1) / cus;
    return (double)(k_bytes / 64 + s.ends) * (s.a + s.c * (double)n);
}
inline double tiles_cost(const TileShape &s, int64_t groups, int64_t rows, int64_t cols, int64_t k_bytes) {
    // (groups differ in size: a twentieth more row tiles than equal ones would make)
    const int64_t row_tiles = groups * ((rows + s.rows - 1) / s.rows);
    return tiles_cost(s, (row_tiles + (groups > 1 ? row_tiles / 20 + 1 : 0)) * ((cols + s.cols - 1) / s.cols), k_bytes);
}
// The tile edge for a product of `rows` x `cols`: 256, 128 or 64 (64 only where its operand layouts have that tile).
// `epilogue`: stages that the 256 x 256 tile's epilogue takes beyond a plain store.
inline int pick_tile(int64_t groups, int64_t rows, int64_t cols, int64_t k, int size, bool small = true, int epilogue = 0) {
    TileShape large = SHAPE_256;
    large.ends += epilogue;
    const double c256 = size == 2 ? tiles_cost(large, groups, rows, cols, k * size) : 1e30;
    const double c128 = tiles_cost(size == 2 ? SHAPE_128 : SHAPE_128F, groups, rows, cols, k * size);
    const double c64 = small ? tiles_cost(size == 2 ? SHAPE_64 : SHAPE_64F, groups, rows, cols, k * size) : 1e30;
    return c256 <= c128 && c256 <= c64 ? 256 : c128 <= c64 ? 128 : 64;
}

// Parts that a reduction of `stages` stages is cut into when its output has fewer tiles than the `slots` workgroups that run at
// once: their planes of partial sums cost a write and a read at about 4 TB/s, a stage `unit` microseconds, the kernel
// that joins them four; a part has at least four stages.
inline int split_parts(double tiles, int64_t slots, double stages, double unit, double plane_bytes) {
    const double plane = plane_bytes / 2e6, most = std::min(std::floor((double)slots / std::max(tiles, 1.0)), stages / 4);
    const double parts = std::floor(std::min(most, std::sqrt(stages * unit / plane)));
    return parts >= 2 && stages * unit * (1 - 1 / parts) > 4 + parts * plane ? (int)parts : 1;
}

// f(element type, result type) as null pointers, for a pair that out_type_ok accepts.
template <class F>
int with_types(int type, int out_type, F f) {
    if (type == T2SP_TYPE_F32) return f((float *)nullptr, (float *)nullptr);
    if (type == T2SP_TYPE_F16) return out_type == type ? f((_Float16 *)nullptr, (_Float16 *)nullptr) : f((_Float16 *)nullptr, (float *)nullptr);
    return out_type == type ? f((__bf16 *)nullptr, (__bf16 *)nullptr) : f((__bf16 *)nullptr, (float *)nullptr);
}

inline int launched() { return hipGetLastError() == hipSuccess ? T2SP_OK : T2SP_ERR_LAUNCH; }

}  // namespace t2sp
