// byhip_rope.hip - rotary positions and the append to a paged cache (gfx950).
//
// Pair i of a head turns by position * step_i, (a, b) -> m (a cos - b sin, a sin + b cos). step_i counts
// 2^-64ths of a turn, so the 64-bit product loses whole turns and nothing else: position 131,071 has its
// angle as exactly as position 1, where an fp32 product position * frequency is off by up to 0.004 rad there.
// The product's top 32 bits give the quadrant and the rest of the angle, x in [-pi/4, pi/4], whose sine and cosine
// are their Taylor sums to x^9 and x^8 (remainders 2e-9 and 2.5e-8).
//
// A row of QKV is read once and written once, queries to q_out and keys and values to their place in the
// pages. A thread owns one unit of 2 VEC values (VEC pairs, or as many values that pass through) and walks over the
// row's heads with it, so an angle's sine and cosine are formed once for all of them. Few rows are spread over
// more blocks, one head per thread.
//
// What bounds it: bytes (116 MB of prompts, bf16: 31 us, 3.7 TB/s, of rows that come from memory; 23 us, 5.1 TB/s, where they lie in
// the Infinity Cache); few rows the launch (32 rows: 4 us).
#include <algorithm>
#include <cmath>

#include "byhip_cache.h"

namespace byhip {
namespace {

struct RopeArgs {
    const void* x[3];      // q, k, v
    size_t stride[3];
    void* q_out;
    size_t q_out_stride;
    int q_out_dtype, cache_dtype;
    int heads, kv_heads, dim, has_cache;
    int layout, rot;
    float magnitude;
    const uint64_t* steps;
    CacheArgs c;
    BatchArgs s;
};

__device__ __forceinline__ void sincos_turns(uint32_t turns, float& sn, float& cs) {
    const uint32_t quadrant = (turns + 0x20000000u) >> 30;
    const float x = (float)(int)(turns - (quadrant << 30)) * 1.46291807926716e-9f;  // 2 pi / 2^32
    const float z = x * x;
    float s = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    s = fmaf(z, s, 8.33333333e-3f);
    s = fmaf(z, s, -1.66666667e-1f);
    s = fmaf(x * z, s, x);
    float c = fmaf(z, 2.48015873e-5f, -1.38888889e-3f);
    c = fmaf(z, c, 4.16666667e-2f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const bool swap = quadrant & 1;
    const float a = swap ? c : s, b = swap ? s : c;
    sn = quadrant & 2 ? -a : a;
    cs = (quadrant + 1) & 2 ? -b : b;
}

__device__ __forceinline__ void turn(float& x, float& y, float cs, float sn) {
    const float a = x * cs - y * sn;
    y = x * sn + y * cs;
    x = a;
}

// Grid: rows x head groups. Thread = (head, unit) of heads_at_once heads of `units` units.
template <int XT, int VEC>
__global__ __launch_bounds__(256) void rope_append(RopeArgs a, int units, int heads_at_once) {
    const int t = blockIdx.x;
    const int b = find_sequence(a.s.starts, a.s.batch, t);
    if (b >= a.s.batch) return;
    const int from = a.s.starts[b], to = a.s.starts[b + 1], pos = a.s.lens[b] - to + t;
    if (pos < 0 || from < 0 || to > a.s.rows || to - from > rows_granted(a.s, b)) return;  // rows outside the call's are no rows
    // the token's place in the pages
    size_t place = 0;
    bool in_cache = false;
    if (a.has_cache) {
        const int col = pos / a.c.page_size;
        const int page = col < a.s.stride ? a.s.table[(size_t)b * a.s.stride + col] : -1;
        in_cache = page >= 0 && page < a.c.pages;
        place = (size_t)page * a.kv_heads * a.c.page_size + (pos - col * a.c.page_size);
    }
    const int rotated = a.rot / (2 * VEC);
    const int total = a.heads + (a.has_cache ? 2 * a.kv_heads : 0);
    const int lane_head = threadIdx.x / units, first = threadIdx.x % units;
    if (lane_head >= heads_at_once) return;
    for (int u = first; u < units; u += 256) {  // more than 256 units only where heads_at_once is 1
        float sn[VEC], cs[VEC];
        int i0, i1;
        if (u < rotated) {
            i0 = a.layout == BYHIP_ROPE_HALVES ? u * VEC : 2 * u * VEC;
            i1 = a.layout == BYHIP_ROPE_HALVES ? i0 + a.rot / 2 : i0 + VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sincos_turns((uint32_t)((a.steps[u * VEC + e] * (uint64_t)pos) >> 32), sn[e], cs[e]);
                sn[e] *= a.magnitude;
                cs[e] *= a.magnitude;
            }
        } else {
            i0 = a.rot + (u - rotated) * 2 * VEC;
            i1 = i0 + VEC;
        }
        const bool two = i1 < a.dim;  // an odd head's last value has no partner
        for (int h = blockIdx.y * heads_at_once + lane_head; h < total; h += gridDim.y * heads_at_once) {
            const int part = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
            const int hl = part == 0 ? h : part == 1 ? h - a.heads : h - a.heads - a.kv_heads;
            if (part && !in_cache) continue;
            const size_t src = (size_t)t * a.stride[part] + (size_t)hl * a.dim;
            float p[VEC], q[VEC];
            load_vec<XT, VEC>(a.x[part], src + i0, p);
            if (two) load_vec<XT, VEC>(a.x[part], src + i1, q);
            else q[0] = 0.0f;
            if (u < rotated && part < 2) {
                if (VEC == 1 || a.layout == BYHIP_ROPE_HALVES) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) turn(p[e], q[e], cs[e], sn[e]);
                } else if constexpr (VEC == 4) {  // the unit's pairs 0 and 1 in p, 2 and 3 in q
                    turn(p[0], p[1], cs[0], sn[0]);
                    turn(p[2], p[3], cs[1], sn[1]);
                    turn(q[0], q[1], cs[2], sn[2]);
                    turn(q[2], q[3], cs[3], sn[3]);
                }
            }
            void* dst = part == 0 ? a.q_out : part == 1 ? (void*)a.c.k : (void*)a.c.v;
            const int dt = part == 0 ? a.q_out_dtype : a.cache_dtype;
            const size_t at = part == 0 ? (size_t)t * a.q_out_stride + (size_t)hl * a.dim
                                        : (place + (size_t)hl * a.c.page_size) * a.dim;
            store_vec<VEC>(dst, at + i0, p, dt);
            if (two) store_vec<VEC>(dst, at + i1, q, dt);
        }
    }
}

template <int XT>
void launch_rope(const RopeArgs& a, bool vec) {
    const int units = vec ? a.dim / 8 : a.rot / 2 + (a.dim - a.rot + 1) / 2;
    const int at_once = std::max(1, 256 / units);
    const int total = a.heads + (a.has_cache ? 2 * a.kv_heads : 0);
    const int passes = (total + at_once - 1) / at_once;
    // few rows: a block per pass, until the chip has a few blocks per CU
    const int spread = std::max(1, std::min(passes, 4 * compute_units() / std::max(1, a.s.rows)));
    const dim3 grid(a.s.rows, spread);
    if (vec) launch("rope_append", (rope_append<XT, 4>), grid, dim3(256), 0, a, units, at_once);
    else launch("rope_append", (rope_append<XT, 1>), grid, dim3(256), 0, a, units, at_once);
    BYHIP_LAUNCHED("rope_append");
}

}  // namespace

void check_rows(const void* p, size_t rows, size_t width, size_t stride, int dtype, const char* what) {
    if (!dtype_bytes(dtype)) fail("byhip: %s dtype %d", what, dtype);
    if (stride < width) fail("byhip: %s stride %zu below its width %zu", what, stride, width);
    if (rows == 0) return;
    check_span(p, ((rows - 1) * stride + width) * dtype_bytes(dtype), what);
}

CacheArgs cache_args(const byhip_kv_cache* c) {
    if (!c) fail("byhip: null cache");
    if (c->dtype != BYHIP_F16 && c->dtype != BYHIP_BF16)
        unsupported("byhip: a cache is fp16 or bf16 (dtype %d)", c->dtype);
    if (c->pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
        fail("byhip: cache of %d pages of %d tokens, %d heads of %d", c->pages, c->page_size, c->kv_heads, c->head_dim);
    const size_t bytes = (size_t)c->pages * c->page_size * c->kv_heads * c->head_dim * 2;
    check_span(c->k, bytes, "cache keys");
    check_span(c->v, bytes, "cache values");
    CacheArgs a;
    a.k = static_cast<uint16_t*>(c->k);
    a.v = static_cast<uint16_t*>(c->v);
    a.pages = c->pages; a.page_size = c->page_size; a.kv_heads = c->kv_heads; a.dim = c->head_dim;
    return a;
}

BatchArgs batch_args(const byhip_kv_batch* b) {
    if (!b) fail("byhip: null batch");
    if (b->batch < 0 || b->rows < 0 || b->table_stride <= 0)
        fail("byhip: batch of %d sequences, %d rows, %d pages each", b->batch, b->rows, b->table_stride);
    check_span(b->table, (size_t)b->batch * b->table_stride * 4, "page table");
    check_span(b->starts, ((size_t)b->batch + 1) * 4, "row starts");
    check_span(b->lens, (size_t)b->batch * 4, "lengths");
    if (b->granted) check_span(b->granted, (size_t)b->batch * 4, "granted tokens");
    BatchArgs a;
    a.table = b->table; a.starts = b->starts; a.lens = b->lens; a.granted = b->granted;
    a.batch = b->batch; a.stride = b->table_stride; a.rows = b->rows;
    return a;
}

}  // namespace byhip

using namespace byhip;

extern "C" {

int byhip_rope_steps(int rot_dim, double base, int scaling, double factor, double original_len, double slow,
                     double fast, uint64_t* steps, float* magnitude) {
    return guard([&] {
        if (!steps || !magnitude) fail("byhip: null rotary output");
        if (rot_dim < 0 || rot_dim % 2) fail("byhip: rotary dimension %d is not even", rot_dim);
        if (!(base > 1.0) || !std::isfinite(base)) fail("byhip: rotary base %g", base);
        if (scaling < BYHIP_ROPE_PLAIN || scaling > BYHIP_ROPE_PARTS) fail("byhip: rotary scaling %d", scaling);
        if (scaling != BYHIP_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
            fail("byhip: rotary scaling factor %g", factor);
        if (scaling == BYHIP_ROPE_PARTS && (!(original_len > 0.0) || !(fast > slow)))
            fail("byhip: rotary scaling over %g positions, %g to %g turns", original_len, slow, fast);
        if (scaling == BYHIP_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
        const double two_pi = 6.283185307179586476925;
        for (int i = 0; i < rot_dim / 2; ++i) {
            double f = std::pow(base, -2.0 * i / rot_dim) / two_pi;
            if (scaling == BYHIP_ROPE_LINEAR) f /= factor;
            if (scaling == BYHIP_ROPE_PARTS) {
                const double keep = std::min(1.0, std::max(0.0, (original_len * f - slow) / (fast - slow)));
                f = f / factor * (1.0 - keep) + f * keep;
            }
            steps[i] = (uint64_t)std::ldexp(f, 64);  // f <= 1 / (2 pi)
        }
        *magnitude = scaling == BYHIP_ROPE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    });
}

int byhip_rope_append(const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v,
                      size_t v_stride, int x_dtype, int heads, int head_dim, const byhip_rope* rope,
                      const byhip_kv_cache* cache, const byhip_kv_batch* batch, void* q_out,
                      size_t q_out_stride, int q_out_dtype) {
    return guard([&] {
        enter_compute();
        RopeArgs a{};
        a.s = batch_args(batch);
        a.has_cache = cache != nullptr;
        if (cache) a.c = cache_args(cache);
        if (cache && head_dim && head_dim != cache->head_dim)
            fail("byhip: heads of %d values, the cache's of %d", head_dim, cache->head_dim);
        a.dim = cache ? cache->head_dim : head_dim;
        a.heads = heads;
        a.kv_heads = cache ? cache->kv_heads : 0;
        if (heads <= 0 || a.dim <= 0) fail("byhip: %d heads of %d values", heads, a.dim);
        a.layout = rope ? rope->layout : BYHIP_ROPE_HALVES;
        a.rot = rope ? rope->rot_dim : 0;
        a.magnitude = rope ? rope->magnitude : 1.0f;
        a.steps = rope ? rope->steps : nullptr;
        if (a.layout != BYHIP_ROPE_HALVES && a.layout != BYHIP_ROPE_PAIRS) fail("byhip: rotary layout %d", a.layout);
        if (a.rot < 0 || a.rot % 2 || a.rot > a.dim) fail("byhip: %d of %d values rotated", a.rot, a.dim);
        if (a.rot) check_span(a.steps, (size_t)a.rot / 2 * 8, "rotary steps");
        const size_t rows = a.s.rows, qw = (size_t)heads * a.dim, kw = (size_t)a.kv_heads * a.dim;
        check_rows(q, rows, qw, q_stride, x_dtype, "queries");
        if (cache) {
            check_rows(k, rows, kw, k_stride, x_dtype, "keys");
            check_rows(v, rows, kw, v_stride, x_dtype, "values");
        }
        check_rows(q_out, rows, qw, q_out_stride, q_out_dtype, "rotated queries");
        if (q_out == q && (q_stride != q_out_stride || x_dtype != q_out_dtype))
            fail("byhip: queries rotated in place need the same stride and dtype");
        if (rows == 0 || a.s.batch == 0) return;
        a.x[0] = q; a.x[1] = k; a.x[2] = v;
        a.stride[0] = q_stride; a.stride[1] = k_stride; a.stride[2] = v_stride;
        a.q_out = q_out; a.q_out_stride = q_out_stride; a.q_out_dtype = q_out_dtype;
        a.cache_dtype = cache ? cache->dtype : BYHIP_F16;
        // four values at a time where every row, head and pair group starts on such a boundary
        bool vec = a.dim % 8 == 0 && a.rot % 8 == 0 && aligned4(q, q_stride, x_dtype) &&
                   aligned4(q_out, q_out_stride, q_out_dtype);
        if (cache)
            vec = vec && aligned4(k, k_stride, x_dtype) && aligned4(v, v_stride, x_dtype) &&
                  aligned4(a.c.k, 4, a.cache_dtype) && aligned4(a.c.v, 4, a.cache_dtype);
        note_device_write(q_out);
        if (cache) { note_device_write(a.c.k); note_device_write(a.c.v); }
        switch (x_dtype) {
        case BYHIP_F32: launch_rope<BYHIP_F32>(a, vec); break;
        case BYHIP_F16: launch_rope<BYHIP_F16>(a, vec); break;
        default: launch_rope<BYHIP_BF16>(a, vec); break;
        }
    });
}

}  // extern "C"
