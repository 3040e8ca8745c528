// byhip_attn.h - what the kernels of byhip_paged_attention share: arguments, masks, the division of the work
// among blocks and the layout of partial results.
#pragma once

#include <algorithm>

#include "byhip_cache.h"

namespace byhip {

struct AttnArgs {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int q_dtype, out_dtype, cache_dtype, heads, window;
    float scale, softcap;
    const float* slopes;
    const int* prefix;
    CacheArgs c;
    BatchArgs s;
    int group;       // query heads per key head
    int q_vec;       // query rows can be read 16 bytes at a time
    int out_vec;     // output rows can be written 4 values at a time
    uint32_t page_mul;   // key / page_size as a product's high bits
    int page_shift;
    int min_rows, max_rows;  // rows (tokens x group) of the sequences this launch takes
    float* part;     // partial results
    int4* joins;     // one description per block
    const void* zeros;  // 16 zero bytes: what keys and values outside the cache read as
};

// Column of key j (below 2^31) in its table row. With l = ceil(log2(page size)) and page_mul = ceil(2^(31 + l) / page size),
// the product's error is under j / 2^(31 + l) < 1 / page size.
__device__ __forceinline__ int page_col(const AttnArgs& a, int j) {
    return (int)(__umulhi(2u * (uint32_t)j, a.page_mul) >> a.page_shift);
}

// Sequence b as a launch sees it.
struct SeqInfo {
    int len, first_pos, prefix;  // keys that can be read; position of the first row; keys that every row sees
    int rows;                    // tokens x group, 0 when the launch does not take the sequence
};

__device__ __forceinline__ SeqInfo seq_info(const AttnArgs& a, int b) {
    SeqInfo s;
    const int from = a.s.starts[b], to = a.s.starts[b + 1], len = a.s.lens[b], granted = rows_granted(a.s, b);  // loads that wait for each other cost a call 1 us
    const int n = from >= 0 && to <= a.s.rows ? max(0, to - from) : 0;  // rows outside the call's are no rows
    const int held = n <= granted ? len : 0;
    s.first_pos = held - n;
    s.len = max(0, in_table(a.s, a.c, held));
    s.prefix = a.prefix ? max(0, min(a.prefix[b], s.len)) : 0;
    const long long rows = (long long)n * a.group;
    s.rows = rows < a.min_rows || rows > a.max_rows ? 0 : (int)rows;
    return s;
}

__device__ __forceinline__ bool sees(const AttnArgs& a, const SeqInfo& s, int pos, int j) {
    return j < s.len && ((j <= pos && (a.window <= 0 || pos - j < a.window)) || j < s.prefix);
}

// The same for 32 keys j0 .. as bits, of those `there`. Formed without branches.
__device__ __forceinline__ uint32_t low_bits(int n) { return (uint32_t)((1ull << max(0, min(n, 32))) - 1); }
__device__ __forceinline__ uint32_t seen_keys(const AttnArgs& a, const SeqInfo& s, int pos, int j0, uint32_t there) {
    const int back = pos - j0;  // positions may lie below 0, so what a window near 2^31 leaves is not formed first
    const uint32_t gone = a.window > 0 && back >= a.window ? low_bits(back - a.window + 1) : 0u;
    return there & ((low_bits(pos + 1 - j0) & ~gone) | low_bits(s.prefix - j0));
}

// The key tiles (of T keys) that rows at positions p0 .. p1 need: first those of the open prefix below
// the window, then those from the window's start to the last key. At least one, so that every row is written.
template <int T>
struct TileRange {
    int prefix_tiles, start, tiles;
    __device__ __forceinline__ TileRange(const AttnArgs& a, const SeqInfo& s, int p0, int p1) {
        start = a.window > 0 && p0 >= a.window ? (p0 - a.window + 1) / T * T : 0;
        const int end = max(0, max(min(s.len, p1 + 1), s.prefix));
        start = min(start, end / T * T);
        prefix_tiles = min((s.prefix + T - 1) / T, start / T);
        tiles = max(1, prefix_tiles + (end - start + T - 1) / T);
    }
    __device__ __forceinline__ int key(int t) const { return t < prefix_tiles ? t * T : start + (t - prefix_tiles) * T; }
};

constexpr size_t kAttnJoinBytes = 65536;  // at the start of the workspace
constexpr int kAttnBatch = 1024;  // sequences per launch: their prefix sums lie in LDS

// A block whose share ends inside an item leaves {last block of the item, sequence, row tile, head}; .x = 0: none.
// Slot 2 w holds block w's part of an item that began before it, slot 2 w + 1 its part of one that goes on after it: R x DIM
// unnormalised sums, then R maxima (log2) and R sums of weights.
template <int R, int DIM>
__device__ __forceinline__ float* part_slot(float* part, int slot) {
    return part + (size_t)slot * R * (DIM + 2);
}

// Keys that a table's row has room for.
inline long long key_room(const AttnArgs& a) { return std::max(1LL, (long long)a.s.stride * a.c.page_size); }

// The launches, per type of the cache; `precise`: fp32 queries or outputs.
void launch_attn_rows_f16(const AttnArgs& a, bool precise);
void launch_attn_rows_bf16(const AttnArgs& a, bool precise);
void launch_attn_chunk_f16(const AttnArgs& a, bool precise);
void launch_attn_chunk_bf16(const AttnArgs& a, bool precise);

// Values that are the same in every lane, as the compiler cannot see where they come through LDS: loops over them then
// run on scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
    return (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

__device__ __forceinline__ uint32_t bit_mask(bool b) { return 0u - (uint32_t)b; }

// What block w leaves when its share ends inside an item it began: the block that holds the item's last unit.
__device__ __forceinline__ int4 join_of(long long last, long long blocks, long long total, int b, int rt, int h) {
    int w = (int)((last * blocks + blocks - 1) / total);
    while ((long long)w * total / blocks > last) --w;
    while ((long long)(w + 1) * total / blocks <= last) ++w;
    return make_int4(w, b, rt, h);
}

// Joins the parts of items of R rows that several blocks worked on. Grid: blocks x row groups. 16 lanes hold a row's values;
// the 4 lane groups of a wave, and with WAVES 4 those of the block's 4 waves, walk over its parts. With WAVES 1 each wave has
// rows of its own, and each lane group where the parts are few (the usual two: 17 us, 34 MB, with a wave per row, 8.6 us with a group).
template <int R, int DIM, int WAVES>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int V = DIM / 16;
    const int w = blockIdx.x;
    const int4 d = a.joins[w];
    if (d.x == 0) return;
    __shared__ float red[WAVES == 4 ? 4 : 1][DIM + 2];
    const int b = d.y, rt = d.z, h = d.w, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = (lane & 15) * V;
    const SeqInfo s = seq_info(a, b);
    const int rows = min(R, s.rows - rt * R), parts = d.x - w + 1;
    const bool alone = WAVES == 1 && parts <= 4;  // a lane group has its row alone
    const int groups = alone ? 1 : 4 * WAVES, group = alone ? 0 : WAVES == 4 ? threadIdx.x >> 4 : lane >> 4;
    const int own = WAVES == 4 ? 1 : alone ? 16 : 4, first = WAVES == 4 ? 0 : alone ? threadIdx.x >> 4 : wave;
    for (int r = blockIdx.y * own + first; r < rows; r += gridDim.y * own) {
        float acc[V] = {}, m = -INFINITY, l = 0.0f;
        const auto add = [&](float pm, float pl, const float (&x)[V]) {
            const float top = fmaxf(m, pm), base = top == -INFINITY ? 0.0f : top;
            const float fo = __builtin_amdgcn_exp2f(m - base), fn = __builtin_amdgcn_exp2f(pm - base);
            l = l * fo + pl * fn;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = acc[e] * fo + x[e] * fn;
            m = top;
        };
#pragma unroll 2
        for (int i = group; i < parts; i += groups) {
            const float* p = part_slot<R, DIM>(a.part, i == 0 ? 2 * w + 1 : 2 * (w + i));
            float x[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(p + r * DIM + col + e);
                x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
            }
            add(p[R * DIM + r], p[R * DIM + R + r], x);
        }
        for (int lanes = 16; !alone && lanes < 64; lanes <<= 1) {
            float x[V];
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = __shfl_xor(acc[e], lanes, 64);
            add(__shfl_xor(m, lanes, 64), __shfl_xor(l, lanes, 64), x);
        }
        if constexpr (WAVES == 4) {
            __syncthreads();
            if (lane < 16) {
#pragma unroll
                for (int e = 0; e < V; ++e) red[wave][col + e] = acc[e];
                if (lane == 0) { red[wave][DIM] = m; red[wave][DIM + 1] = l; }
            }
            __syncthreads();
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[V];
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = red[i][col + e];
                add(red[i][DIM], red[i][DIM + 1], x);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int q = rt * R + r, t = a.s.starts[b] + q / a.group;
        const size_t out = (size_t)t * a.out_stride + (size_t)(h * a.group + q % a.group) * a.c.dim + col;
        if (threadIdx.x < 16 || (WAVES == 1 && (alone || lane < 16))) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                if (col + e >= a.c.dim) continue;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = l == 0.0f ? 0.0f : acc[e + k] * inv;
                if (a.out_vec) {
                    store_vec<4>(a.out, out + e, v, a.out_dtype);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float one[1] = {v[k]};
                        store_vec<1>(a.out, out + e + k, one, a.out_dtype);
                    }
                }
            }
        }
    }
}

// The cache's 16-bit type in registers and the matrix instructions on it.
template <int CT> struct Half8;
template <> struct Half8<BYHIP_F16> {
    typedef _Float16 vec __attribute__((ext_vector_type(8)));
    typedef _Float16 one;
};
template <> struct Half8<BYHIP_BF16> {
    typedef __bf16 vec __attribute__((ext_vector_type(8)));
    typedef __bf16 one;
};
typedef float f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f4 mfma16(Half8<BYHIP_F16>::vec x, Half8<BYHIP_F16>::vec y, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(Half8<BYHIP_BF16>::vec x, Half8<BYHIP_BF16>::vec y, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
__device__ __forceinline__ f16v mfma32(Half8<BYHIP_F16>::vec x, Half8<BYHIP_F16>::vec y, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0); }
__device__ __forceinline__ f16v mfma32(Half8<BYHIP_BF16>::vec x, Half8<BYHIP_BF16>::vec y, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0); }

// x as NP terms of the cache's type, each the rounding of what the ones before it leave.
template <int CT, int NP>
__device__ __forceinline__ void split_terms(float x, typename Half8<CT>::one (&t)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        t[p] = (typename Half8<CT>::one)x;
        if (p + 1 < NP) x -= (float)t[p];
    }
}

// The power of two by which a row of fp32 queries is multiplied before it is split into fp16 terms: its largest value `top` comes
// to [2^14, 2^15). At most 2^100, so that scale / 2^shift stays a normal number (0 times a masked score of -infinity would be NaN):
// rows of zeros, and rows below 2^-86, whose terms then end at 2^-125 or so, far below what a weight can show.
__device__ __forceinline__ int query_shift(float top) { return min(fp16_range_shift(top), 100); }
// Value f of a row of queries, times 2^shift, as terms. A value too small for the first fp16 term still has its sign there (the second
// takes it back), for a product with an infinite key.
template <int CT, int NP>
__device__ __forceinline__ void query_terms(float f, int shift, typename Half8<CT>::one (&t)[NP]) {
    const float x = ldexpf(f, shift);
    split_terms<CT, NP>(x, t);
    if constexpr (CT == BYHIP_F16 && NP == 2) {
        if ((float)t[0] == 0.0f && f != 0.0f) {
            t[0] = (_Float16)copysignf(0x1p-24f, f);
            t[1] = (_Float16)(x - (float)t[0]);
        }
    }
}
constexpr float kLeastScale = 0x1p-20f;  // smaller scales (and those that are not positive) are applied before the masks

// Two 16-bit values, those that are not finite (all exponent bits `exp` set) as 0.
__device__ __forceinline__ uint32_t finite_only(uint32_t x, uint32_t exp) {
    x &= (x & exp) == exp ? 0xFFFF0000u : ~0u;
    return x & ((x >> 16 & exp) == exp ? 0xFFFFu : ~0u);
}

constexpr float kLog2e = 1.44269504f;

// tanh. Near 0 its Taylor sum (to y^15 below 1/2: remainder under 2e-8 of it), else 1 - 2 / (1 + e^2y).
template <bool PRECISE>
__device__ __forceinline__ float soft_tanh(float y) {
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
    const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e);
    if constexpr (!PRECISE) return far;
    const float z = y * y;
    float s = fmaf(z, -1.45583439e-3f, 3.59212804e-3f);
    s = fmaf(z, s, -8.86323553e-3f);
    s = fmaf(z, s, 2.18694885e-2f);
    s = fmaf(z, s, -5.39682540e-2f);
    s = fmaf(z, s, 1.33333333e-1f);
    s = fmaf(z, s, -3.33333333e-1f);
    return fabsf(y) < 0.5f ? fmaf(y * z, s, y) : far;
}

}  // namespace byhip
