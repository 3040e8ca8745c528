// byhip_cache.h - what the kernels over a paged cache share: descriptors by value, checks, and the search for
// a row's sequence.
#pragma once

#include "byhip_internal.h"
#include "byhip_kernels.h"

namespace byhip {

// One layer's cache as the kernels take it. A (page, head) block of page_size rows is contiguous; offsets are
// formed in 64 bits (a cache may pass 4 GiB).
struct CacheArgs {
    uint16_t* k;
    uint16_t* v;
    int pages, page_size, kv_heads, dim;
};

struct BatchArgs {
    const int* table;
    const int* starts;
    const int* lens;
    const int* granted;
    int batch, stride, rows;
};

// Host checks of the descriptors (their device spans included).
CacheArgs cache_args(const byhip_kv_cache* c);
BatchArgs batch_args(const byhip_kv_batch* b);
// Rows of `width` values, `stride` elements apart: the span the caller's buffer must hold.
void check_rows(const void* p, size_t rows, size_t width, size_t stride, int dtype, const char* what);

// The tokens of a sequence of `len` that its table has columns for.
__device__ __forceinline__ int in_table(const BatchArgs& s, const CacheArgs& c, int len) {
    const long long room = (long long)s.stride * c.page_size;
    return len > room ? (int)room : len;
}

// The rows that sequence b has room for at most: those of a refused cache_grow have no position, or they would be placed over the
// tokens before them.
__device__ __forceinline__ int rows_granted(const BatchArgs& s, int b) { return s.granted ? s.granted[b] : 0x7FFFFFFF; }

// The sequence of row t: the number of entries of starts[1 .. batch] that are <= t, `batch` when t belongs to
// none. The 64 lanes of a wave look at 64 entries at a time, so 4096 sequences take two dependent loads.
__device__ __forceinline__ int find_sequence(const int* starts, int batch, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = batch;
    while (n > 0) {
        const int step = (n + 63) / 64, at = (lane + 1) * step;
        const bool below = at <= n && starts[lo + at] <= t;
        const int count = __popcll(__ballot(below));
        lo += count * step;
        n = min(step - 1, n - count * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Value i of an array of dtype DT, and VEC (1 or 4) neighbours at once; DT is BYHIP_F32 / F16 / BF16.
template <int DT>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    if constexpr (DT == BYHIP_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == BYHIP_F16) return (float)static_cast<const _Float16*>(p)[i];
    else return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* p, size_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = load1<DT>(p, i);
    } else if constexpr (DT == BYHIP_F32) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        const uint32_t w[2] = {a.x, a.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t b = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
            v[e] = DT == BYHIP_F16 ? (float)bits_h((uint16_t)b) : __builtin_bit_cast(float, b << 16);
        }
    }
}
// The same for stores, the dtype known at run time (a branch that is the same for a whole launch).
template <int VEC>
__device__ __forceinline__ void store_vec(void* p, size_t i, const float (&v)[VEC], int dtype) {
    if constexpr (VEC == 1) {
        switch (dtype) {
        case BYHIP_F32: store_y<BYHIP_F32>(p, i, v[0]); break;
        case BYHIP_F16: store_y<BYHIP_F16>(p, i, v[0]); break;
        default: store_y<BYHIP_BF16>(p, i, v[0]); break;
        }
    } else if (dtype == BYHIP_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint2 w;
        if (dtype == BYHIP_F16) {
            w.x = h_bits((_Float16)v[0]) | (uint32_t)h_bits((_Float16)v[1]) << 16;
            w.y = h_bits((_Float16)v[2]) | (uint32_t)h_bits((_Float16)v[3]) << 16;
        } else {
            w.x = f32x2_to_bf16x2_bits(v[0], v[1]);
            w.y = f32x2_to_bf16x2_bits(v[2], v[3]);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = w;
    }
}

// Whether rows of dtype at p with this stride can be moved four values at a time.
inline bool aligned4(const void* p, size_t stride, int dtype) {
    const size_t bytes = 4 * dtype_bytes(dtype);  // 0: no dtype, which check_rows refuses
    return bytes && stride % 4 == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace byhip
