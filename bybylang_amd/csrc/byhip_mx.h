// byhip_mx.h - microscaled rows (8 or 4 bits with one power of two per 32 values) and the plan of an experts' call: what
// the kernels that write and read them share.
#pragma once

#include "byhip_cache.h"

namespace byhip {

inline bool is_mx(int dt) { return dt == BYHIP_MXFP8_KM || dt == BYHIP_MXFP4_KM; }
inline int mx_bits(int fmt) { return fmt == BYHIP_MXFP8_KM ? 8 : 4; }
// Bytes of the values of `rows` rows, and of the rows with their scales.
inline size_t mx_values(size_t rows, size_t K, int fmt) { return rows * K * mx_bits(fmt) / 8; }
inline size_t mx_bytes(size_t rows, size_t K, int fmt) { return mx_values(rows, K, fmt) + rows * (K / 32); }
// A buffer of microscaled rows: its format, width, alignment and span.
void check_mx(const void* p, size_t rows, size_t K, int fmt, const char* what);

// The larger magnitude of two values' bits: as whole numbers they are ordered as the magnitudes are, with infinity above
// every number and NaN above infinity, so that neither is lost in a maximum.
__device__ __forceinline__ uint32_t mag_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// Scale byte of a group whose largest magnitude has these bits: m 2^x (1 <= m < 2) is at most 448 = 1.75 2^8 times 2^(x - 8)
// where m <= 1.75, and at most 6 = 1.5 2^2 times 2^(x - 2) where m <= 1.5. 255 (NaN) for what is not finite.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale(uint32_t mag) {
    constexpr int step = FMT == BYHIP_MXFP8_KM ? 8 : 2;
    constexpr uint32_t most = FMT == BYHIP_MXFP8_KM ? 0x600000u : 0x400000u;
    const int e = (int)(mag >> 23) - step + ((mag & 0x7FFFFFu) > most);
    return mag >= 0x7F800000u ? 255u : (uint32_t)max(e, 0);
}
// The factor 2^(127 - byte) that brings the group's values into range: exact, both exponents being fp32's (bytes up to 253 occur).
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23); }

// Eight values of a group in memory order: lo are its elements j .. j + 3, hi the elements j + 16 .. j + 19 (j = 0, 4, 8, 12). out: the
// 8 bytes from 2 j on (8 bits), or in out[0] the 4 bytes from j on (4 bits). The conversions round to the nearest, ties
// to even, and see nothing out of their range; a group that is not finite has values 0 under its NaN scale.
template <int FMT>
__device__ __forceinline__ void mx_pack8(const float (&lo)[4], const float (&hi)[4], uint32_t byte, uint32_t (&out)[2]) {
    const float f = mx_inverse(byte);
    float a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = byte == 255u ? 0.0f : lo[e] * f;
        b[e] = byte == 255u ? 0.0f : hi[e] * f;
    }
    if constexpr (FMT == BYHIP_MXFP8_KM) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(a[2 * h], b[2 * h], 0, false);
            out[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a[2 * h + 1], b[2 * h + 1], w, true);
        }
    } else {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[0], b[0], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[1], b[1], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[2], b[2], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[3], b[3], 1.0f, 3);
        out[0] = w;
        out[1] = 0;
    }
}
__device__ __forceinline__ uint32_t mag8(const float (&lo)[4], const float (&hi)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, max(mag_bits(lo[e]), mag_bits(hi[e])));
    return m;
}
// The 8 values' place: 32 G + j of row `row` (j = 0, 4, 8, 12) in a buffer of K values per row.
template <int FMT>
__device__ __forceinline__ void mx_store8(uint8_t* y, size_t row, int K, int G, int j, const uint32_t (&out)[2]) {
    if constexpr (FMT == BYHIP_MXFP8_KM)
        *reinterpret_cast<uint2*>(y + row * K + 32 * G + 2 * j) = make_uint2(out[0], out[1]);
    else
        *reinterpret_cast<uint32_t*>(y + row * (K / 2) + 16 * G + j) = out[0];
}

// ── plans ──

constexpr int kMaxExperts = 1024;
// A unit of a product's work: rows `first` .. first + rows - 1 of the plan, all of one expert's.
struct MoeUnit {
    int expert, first, rows, pad;
};
// Rows of a unit of moe_rows, by the mean rows per expert, so that most experts fill one: a unit's rows share one pass over the expert's
// matrix, but 64 rows' own loads cost more than a second pass over it from the cache (us, one matrix of 4096 x 4096, 16 / 24 / 32 rows: units of 16 6.0 / 8.4 / 8.4, of 32 6.9 / 7.4 / 7.9;
// 64 / 128 / 256 rows: units of 32 10.5 / 14.4 / 22.4, of 64 12.4 / 14.8 / 19.3; 16 experts, 2080 to 2048 gates and ups, 8 / 16 rows each: units of 16 21.6 / 28.0, of 32 24.9 / 28.5;
// 128 / 192 rows each: of 32 82 / 117, of 64 82 / 105). moe_tiles' units have kTileRows.
inline int moe_unit_rows(long long rows, int experts) {
    const long long mean = (rows + experts - 1) / experts;
    return mean <= 16 ? 16 : mean <= 128 ? 32 : 64;
}
constexpr int kTileRows = 128;
// Units at most: an expert leaves one that is not full.
inline int moe_max_units(int rows, int experts, int unit) { return rows / unit + (rows < experts ? rows : experts); }
// The plan's buffer: offsets and order (the caller's to read), the numbers of units of both kinds and the units, and what the plan's
// kernels count in (one row of `experts` counts per block of assignments, and one of their sums).
struct MoePlan {
    int tokens, top_k, experts, rows, unit_rows, max_units, max_tiles, blocks;
    int *offsets, *order, *n_units, *counts;  // n_units: of units, of tiles
    MoeUnit *units, *tiles;
    size_t bytes;
};
constexpr int kPlanBlock = 1024;  // assignments per block of the plan's kernels
MoePlan moe_layout(const byhip_moe_plan* p);  // sizes checked (fail), the buffer not
MoePlan moe_plan_args(const byhip_moe_plan* p);

}  // namespace byhip
