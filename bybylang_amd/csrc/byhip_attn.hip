// byhip_attn.hip - attention of new rows over a paged cache: the entry point and the general kernel (gfx950).
//
// For row t of sequence b at position p and head h, over the keys j that the masks let it see:
//   s_j = scale q . k_j, capped to softcap tanh(s / softcap), less slope_h |p - j|
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m the largest s_j
// in one pass: m, the sum and the output are kept as of the keys seen so far, and scaled down when m grows.
#include <algorithm>

#include "byhip_attn.h"

namespace byhip {
namespace {

__device__ uint4 g_zeros;  // AttnArgs::zeros: zero from the start, so there is no write for a stream to wait for
void* zeros = nullptr;     // its address

constexpr int kGeneralMaxDim = 2048;  // queries and sums of 4 waves in 64 KB of LDS

// One wave per row and head, 64 keys at a time, a key per lane for the scores and a value per lane for the
// sums. It takes heads of any size.
template <int CT>
__global__ __launch_bounds__(256) void attn_general(AttnArgs a) {
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t item = (size_t)blockIdx.x * 4 + wave;
    if (item >= (size_t)a.s.rows * a.heads) return;
    const int t = __builtin_amdgcn_readfirstlane((int)(item / a.heads)), h = __builtin_amdgcn_readfirstlane((int)(item % a.heads));
    const int b = find_sequence(a.s.starts, a.s.batch, t);
    if (b >= a.s.batch) return;
    const SeqInfo s = seq_info(a, b);
    if (s.rows == 0) return;  // its rows pass the call's
    const int pos = s.first_pos + t - a.s.starts[b];
    const int D = a.c.dim, kvh = h / a.group;
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    float* q = lds + wave * 2 * D;
    float* acc = q + D;
    for (int d = lane; d < D; d += 64) {
        const size_t i = (size_t)t * a.q_stride + (size_t)h * D + d;
        q[d] = a.q_dtype == BYHIP_F32 ? load1<BYHIP_F32>(a.q, i) : load1<CT>(a.q, i);
        acc[d] = 0.0f;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave reads its lanes' queries
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, sum = 0.0f;
    for (int j0 = 0; j0 < s.len; j0 += 64) {
        const int j = j0 + lane;
        bool see = sees(a, s, pos, j);
        if (__ballot(see) == 0) continue;
        const int col = page_col(a, j);
        const int page = see ? a.s.table[(size_t)b * a.s.stride + col] : -1;
        see = page >= 0 && page < a.c.pages;
        const size_t row = ((size_t)page * a.c.kv_heads + kvh) * a.c.page_size + (j - col * a.c.page_size);
        float sc = -INFINITY;
        if (see) {
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot = fmaf(q[d], load1<CT>(a.c.k, row * D + d), dot);
            sc = dot * a.scale;
            if (a.softcap > 0.0f) sc = a.softcap * tanhf(sc / a.softcap);
            sc -= slope * fabsf((float)(pos - j));
        }
        float top = sc;
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float grown = fmaxf(m, top);
        const bool nan = __ballot(sc != sc) != 0;
        if (grown == -INFINITY && !nan) continue;
        const float base = grown == -INFINITY ? 0.0f : grown;
        const float w = see ? expf(sc - base) : 0.0f;
        const float fade = expf(m - base);
        sum = sum * fade + wave_sum(w);
        for (int d = lane; d < D; d += 64) acc[d] *= fade;
        m = grown;
        for (uint64_t left = __ballot(see); left; left &= left - 1) {
            const int l = __ffsll((unsigned long long)left) - 1;
            const float wj = __shfl(w, l, 64);
            const size_t rj = (size_t)__shfl((long long)row, l, 64);
            for (int d = lane; d < D; d += 64) {
                const float v = load1<CT>(a.c.v, rj * D + d);
                acc[d] = wj == 0.0f && !(fabsf(v) < INFINITY) ? acc[d] + v : fmaf(wj, v, acc[d]);  // no weight is 0, it may only round to it
            }
        }
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int d = lane; d < D; d += 64) {
        const float o[1] = {sum == 0.0f ? 0.0f : acc[d] * f};
        store_vec<1>(a.out, (size_t)t * a.out_stride + (size_t)h * D + d, o, a.out_dtype);
    }
}

void launch_general(const AttnArgs& a) {
    if (a.c.dim > kGeneralMaxDim) unsupported("byhip: attention heads of %d values (at most %d)", a.c.dim, kGeneralMaxDim);
    const size_t items = (size_t)a.s.rows * a.heads;
    const dim3 grid((unsigned)((items + 3) / 4));
    const size_t lds = (size_t)8 * a.c.dim * sizeof(float);
    if (a.cache_dtype == BYHIP_F16) launch("attn_general", attn_general<BYHIP_F16>, grid, dim3(256), lds, a);
    else launch("attn_general", attn_general<BYHIP_BF16>, grid, dim3(256), lds, a);
    BYHIP_LAUNCHED("attn_general");
}

// Rows per key head from which attn_chunk reads a sequence. attn_rows reads its keys once per 16 rows; attn_chunk reads them once
// per 256 but starts 10 us later, which is 56 MB at attn_rows' rate. 16 sequences of 4096 keys, 8 key heads of 128 values (268 MB),
// 16 rows: 64 us with attn_rows, 68 with attn_chunk; 32 rows: 100 and 68; one sequence of 600 keys, 32 rows: 15 and 25. With fp32
// rows, whose terms attn_chunk multiplies for 128 rows at least, 32 rows take 108 and 117 on bf16 (256 values: 204 and 403).
// The lengths are on the device, so the rule goes by the keys that the tables have room for: where they are much wider than their
// sequences, 17 to 32 rows go to attn_chunk for less (that one sequence of 600 keys in a table for 32000: 26 us).
int chunk_rows(const AttnArgs& a, bool precise) {
    const double bytes = (double)a.s.batch * key_room(a) * a.c.kv_heads * a.c.dim * 4.0;  // keys and values there is room for
    return !precise && bytes >= 56e6 ? 17 : 33;
}

// Whether the kernels on matrix instructions take the cache: whole 16-byte pieces of a head, cache rows that 32 bits count.
bool takes(const AttnArgs& a) {
    return a.c.dim % 8 == 0 && a.c.dim <= 256 && reinterpret_cast<uintptr_t>(a.c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.c.v) % 16 == 0 &&
           (double)a.c.pages * a.c.kv_heads * a.c.page_size < 4294967295.0;
}

void launch_tiled(AttnArgs a) {
    a.joins = static_cast<int4*>(attn_workspace());
    a.zeros = zeros;
    a.part = reinterpret_cast<float*>(static_cast<char*>(attn_workspace()) + kAttnJoinBytes);
    const bool precise = a.q_dtype == BYHIP_F32 || a.out_dtype == BYHIP_F32, f16 = a.cache_dtype == BYHIP_F16;
    // The lengths are on the device: one sequence has all rows; as many rows as sequences are decoding; else
    // sequences of few rows and of many go to a launch each, which passes over the others.
    const long long rows = (long long)a.s.rows * a.group;
    const bool one = a.s.batch == 1;
    const int from = chunk_rows(a, precise);
    const bool few = !one || rows < from, many = one ? rows >= from : a.s.rows > a.s.batch;
    const AttnArgs whole = a;
    for (int b0 = 0; b0 < whole.s.batch; b0 += kAttnBatch) {
        a.s.table = whole.s.table + (size_t)b0 * whole.s.stride;
        a.s.starts = whole.s.starts + b0;
        a.s.lens = whole.s.lens + b0;
        a.s.granted = whole.s.granted ? whole.s.granted + b0 : nullptr;
        a.s.batch = std::min(kAttnBatch, whole.s.batch - b0);
        a.prefix = whole.prefix ? whole.prefix + b0 : nullptr;
        a.min_rows = 1;
        a.max_rows = many ? from - 1 : 0x7FFFFFFF;
        if (few) (f16 ? launch_attn_rows_f16 : launch_attn_rows_bf16)(a, precise);
        a.min_rows = few ? from : 1;
        a.max_rows = 0x7FFFFFFF;
        if (many) (f16 ? launch_attn_chunk_f16 : launch_attn_chunk_bf16)(a, precise);
    }
}

}  // namespace

void attn_setup() {
    BYHIP_HIP(hipGetSymbolAddress(&zeros, HIP_SYMBOL(g_zeros)));
    if (!zeros) fail("byhip: attention's zeros have no device address");
}

}  // namespace byhip

using namespace byhip;

extern "C" int byhip_paged_attention(const void* q, size_t q_stride, int q_dtype, int heads, const byhip_attn* attn,
                                     const byhip_kv_cache* cache, const byhip_kv_batch* batch, void* out,
                                     size_t out_stride, int out_dtype) {
    return guard([&] {
        enter_compute();
        if (!attn) fail("byhip: null attention options");
        AttnArgs a{};
        a.c = cache_args(cache);
        a.s = batch_args(batch);
        if (heads <= 0 || heads % a.c.kv_heads) fail("byhip: %d heads over %d key heads", heads, a.c.kv_heads);
        if (q_dtype != BYHIP_F32 && (q_dtype == BYHIP_F16 || q_dtype == BYHIP_BF16) && q_dtype != cache->dtype)
            unsupported("byhip: 16-bit queries have the cache's dtype (%d, cache %d)", q_dtype, cache->dtype);
        if ((long long)a.s.rows * (heads / a.c.kv_heads) > 0x7FFFFFFF)  // the kernels count a key head's rows in 31 bits
            unsupported("byhip: attention of %d rows of %d heads over %d key heads in one call", a.s.rows, heads, a.c.kv_heads);
        const size_t width = (size_t)heads * a.c.dim;
        check_rows(q, a.s.rows, width, q_stride, q_dtype, "queries");
        check_rows(out, a.s.rows, width, out_stride, out_dtype, "attention output");
        if (!(attn->softcap >= 0.0f)) fail("byhip: softcap %g", (double)attn->softcap);
        if (attn->slopes) check_span(attn->slopes, (size_t)heads * 4, "slopes");
        if (attn->prefix) check_span(attn->prefix, (size_t)a.s.batch * 4, "prefix lengths");
        if (a.s.rows == 0 || a.s.batch == 0) return;
        a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride;
        a.q_dtype = q_dtype; a.out_dtype = out_dtype; a.cache_dtype = cache->dtype; a.heads = heads;
        a.scale = attn->scale; a.softcap = attn->softcap; a.window = attn->window;
        a.slopes = attn->slopes; a.prefix = attn->prefix;
        a.group = heads / a.c.kv_heads;
        a.max_rows = 0x7FFFFFFF;
        int log = 0;
        while ((1ll << log) < a.c.page_size) ++log;
        a.page_shift = log;
        a.page_mul = (uint32_t)(((1ull << (31 + log)) + a.c.page_size - 1) / a.c.page_size);
        a.q_vec = q_stride * dtype_bytes(q_dtype) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0;
        a.out_vec = aligned4(out, out_stride, out_dtype);
        note_device_write(out);
        if (takes(a)) launch_tiled(a);
        else launch_general(a);
    });
}
