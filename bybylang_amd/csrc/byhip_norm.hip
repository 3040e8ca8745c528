// byhip_norm.hip - the residual stream between two blocks (gfx950): h = res_scale res + gate . post(x),
// y = pre(h), post and pre RMS or layer norms.
//
// Every input is read once and every output written once: a row's values stay in its block's registers (at most
// 32 per thread) from the first norm to the last store. Sums are fp32; a variance is the mean of the squared
// deviations from the mean already formed, not a difference of two large sums. Rows too long for the registers
// of 1024 threads pass over x again for each sum.
#include <algorithm>

#include "byhip_mx.h"

namespace byhip {
namespace {

struct NormArgs {
    const void* x;
    const float* gate;
    const void* res;
    void* h;
    void* y;
    size_t x_stride, gate_stride, res_stride, h_stride, y_stride;
    byhip_norm post, pre;
    int has_post, has_pre, N, y_dtype, h_dtype, vec;
    long long M;
    float res_scale;
    uint8_t* y_scales;
};

// Sums over the block's threads, the same value in every thread. One barrier each: successive sums use the halves of `red`
// in turn, and a half is written again only after the barrier of the sum between.
struct BlockSum {
    float (*red)[16];
    int turn = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = wave_sum(v);
        const int waves = blockDim.x >> 6;
        if (waves == 1) return v;
        if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
        for (int i = 0; i < waves; ++i) v += red[turn][i];
        turn ^= 1;
        return v;
    }
};

// Loads, scales and stores of 4 values at column i, those past N left out (read as 0).
template <int DT>
__device__ __forceinline__ void read4(const void* p, size_t row, int i, int N, int vec, float (&v)[4]) {
    if (vec && i + 4 <= N) {
        load_vec<DT, 4>(p, row + i, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < N ? load1<DT>(p, row + i + e) : 0.0f;
    }
}
__device__ __forceinline__ void write4(void* p, size_t row, int i, int N, int vec, const float (&v)[4], int dtype) {
    if (vec && i + 4 <= N) {
        store_vec<4>(p, row + i, v, dtype);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < N) {
                const float one[1] = {v[e]};
                store_vec<1>(p, row + i + e, one, dtype);
            }
    }
}

// One norm over the row held in v (columns 4 (threads c + thread) ..).
template <int CH>
__device__ __forceinline__ void norm_row(float (&v)[CH][4], const byhip_norm& n, int N, int vec, int tid, BlockSum& block_sum) {
    const int TH = blockDim.x;
    float mean = 0.0f;
    if (n.kind == BYHIP_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += v[c][e];  // 0 past N
        mean = block_sum(s) / N;
    }
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float d = 4 * (TH * c + tid) + e < N ? v[c][e] - mean : 0.0f;
            s += d * d;
        }
    const float f = 1.0f / sqrtf(block_sum(s) / N + n.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = 4 * (TH * c + tid);
        float w[4] = {1.0f, 1.0f, 1.0f, 1.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (n.weight) read4<BYHIP_F32>(n.weight, 0, i, N, vec, w);
        if (n.bias) read4<BYHIP_F32>(n.bias, 0, i, N, vec, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c][e] = (v[c][e] - mean) * f * w[e] + b[e];
    }
}

// The lane's value of the lane 4 further on in its 8, or 4 back.
__device__ __forceinline__ uint32_t other_half(uint32_t v, bool upper) {
    const uint32_t up = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x104, 0xF, 0xF, false);    // row_shl:4
    const uint32_t down = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);  // row_shr:4
    return upper ? down : up;
}

// The row in v as microscaled values: 8 neighbouring lanes hold a group, and a lane's four elements and those of the lane 4 further on
// or back take turns in memory. (With a thread's eight values chosen so that they lie next to each other there, reads of 64 bytes at a time
// cost more than this exchange: 4099 x 5120 64 us.)
template <int FMT, int CH>
__device__ __forceinline__ void write_mx(const NormArgs& a, size_t row, int tid, int TH, const float (&v)[CH][4]) {
    const int t = tid & 7;
    const bool upper = t & 4;
    uint8_t* y = static_cast<uint8_t*>(a.y);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = 4 * (TH * c + tid), G = i >> 5;
        uint32_t m = max(max(mag_bits(v[c][0]), mag_bits(v[c][1])), max(mag_bits(v[c][2]), mag_bits(v[c][3])));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
        const uint32_t byte = mx_scale<FMT>(m);
        const float f = mx_inverse(byte);
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = byte == 255u ? 0.0f : v[c][e] * f;
        if constexpr (FMT == BYHIP_MXFP8_KM) {
            const int low = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
            const uint32_t own = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], low, true), far = other_half(own, upper);
            // Bytes 0 and 1 of both (the lower lane's first), or 2 and 3.
            const uint32_t out = upper ? __builtin_amdgcn_perm(own, far, 0x07030602u) : __builtin_amdgcn_perm(far, own, 0x05010400u);
            if (i < a.N) *reinterpret_cast<uint32_t*>(y + row * a.N + 32 * G + (upper ? 8 * (t - 4) + 4 : 8 * t)) = out;
        } else {
            uint32_t own = 0;
            own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, z[0], 0.0f, 1.0f, 0);
            own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, z[1], 0.0f, 1.0f, 1);
            own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, z[2], 0.0f, 1.0f, 2);
            own = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(own, z[3], 0.0f, 1.0f, 3);
            const uint32_t far = other_half(own, upper);
            if (i < a.N && !upper) *reinterpret_cast<uint32_t*>(y + row * (a.N / 2) + 16 * G + 4 * t) = own | far << 4;
        }
        if (i < a.N && t == 0) a.y_scales[row * (a.N / 32) + G] = (uint8_t)byte;
    }
}

template <int XT, int HT, int CH, bool MX = false>
__global__ __launch_bounds__(1024) void norm_block(NormArgs a) {
    __shared__ float red[2][16];
    BlockSum block_sum{red};
    const int tid = threadIdx.x, TH = blockDim.x;
    const size_t row = blockIdx.x;
    float v[CH][4], r[CH][4];
#pragma unroll
    for (int c = 0; c < CH; ++c) read4<XT>(a.x, row * a.x_stride, 4 * (TH * c + tid), a.N, a.vec, v[c]);
    if (a.res) {
#pragma unroll
        for (int c = 0; c < CH; ++c) read4<HT>(a.res, row * a.res_stride, 4 * (TH * c + tid), a.N, a.vec, r[c]);
    }
    if (a.has_post) norm_row<CH>(v, a.post, a.N, a.vec, tid, block_sum);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = 4 * (TH * c + tid);
        if (a.gate) {
            float g[4];
            read4<BYHIP_F32>(a.gate, row * a.gate_stride, i, a.N, a.vec, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] *= g[e];
        }
        if (a.res) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = a.res_scale * r[c][e] + v[c][e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c][e] = i + e < a.N ? v[c][e] : 0.0f;
        if (a.h) write4(a.h, row * a.h_stride, i, a.N, a.vec, v[c], HT);
    }
    if (!a.has_pre) return;
    norm_row<CH>(v, a.pre, a.N, a.vec, tid, block_sum);
    if constexpr (MX) {
        if (a.y_dtype == BYHIP_MXFP8_KM) write_mx<BYHIP_MXFP8_KM, CH>(a, row, tid, TH, v);
        else write_mx<BYHIP_MXFP4_KM, CH>(a, row, tid, TH, v);
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) write4(a.y, row * a.y_stride, 4 * (TH * c + tid), a.N, a.vec, v[c], a.y_dtype);
    }
}

// One value per lane of 32 neighbours (a half wave) that are a group: its byte, or with the lane 16 further on its byte of two.
template <int FMT>
__device__ __forceinline__ void write_mx1(const NormArgs& a, size_t row, int i, float v) {
    uint32_t m = mag_bits(v);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    const uint32_t byte = mx_scale<FMT>(m);
    const float z = byte == 255u ? 0.0f : v * mx_inverse(byte), far = __shfl_xor(z, 16);
    const int G = i >> 5, j = i & 31;
    uint8_t* y = static_cast<uint8_t*>(a.y);
    if constexpr (FMT == BYHIP_MXFP8_KM)
        y[row * a.N + 32 * G + 2 * (j & 15) + (j >> 4)] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(z, z, 0, false);
    else if (j < 16)
        y[row * (a.N / 2) + 16 * G + j] = (uint8_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, z, far, 1.0f, 0);
    if (j == 0) a.y_scales[row * (a.N / 32) + G] = (uint8_t)byte;
}

// Rows of any length: each sum walks over x (and res) again. h may be res's rows, so it is written last.
template <int XT, int HT>
__global__ __launch_bounds__(1024) void norm_block_long(NormArgs a) {
    __shared__ float red[2][16];
    BlockSum block_sum{red};
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x;
    const float inv = 1.0f / a.N;
    float mean = 0.0f, f = 1.0f;
    auto sum = [&](auto&& value) {
        float s = 0.0f;
        for (int i = tid; i < a.N; i += 1024) s += value(i);
        return block_sum(s);
    };
    auto x = [&](int i) { return load1<XT>(a.x, row * a.x_stride + i); };
    if (a.has_post) {
        if (a.post.kind == BYHIP_NORM_LAYER) mean = sum(x) * inv;
        f = 1.0f / sqrtf(sum([&](int i) { const float d = x(i) - mean; return d * d; }) * inv + a.post.eps);
    }
    auto h = [&](int i) {
        float v = x(i);
        if (a.has_post) v = (v - mean) * f * (a.post.weight ? a.post.weight[i] : 1.0f) + (a.post.bias ? a.post.bias[i] : 0.0f);
        if (a.gate) v *= a.gate[row * a.gate_stride + i];
        return a.res ? a.res_scale * load1<HT>(a.res, row * a.res_stride + i) + v : v;
    };
    float mean2 = 0.0f, f2 = 1.0f;
    if (a.has_pre) {
        if (a.pre.kind == BYHIP_NORM_LAYER) mean2 = sum(h) * inv;
        f2 = 1.0f / sqrtf(sum([&](int i) { const float d = h(i) - mean2; return d * d; }) * inv + a.pre.eps);
    }
    for (int i = tid; i < a.N; i += 1024) {
        const float v = h(i);
        const float hv[1] = {v};
        const float yv[1] = {(v - mean2) * f2 * (a.has_pre && a.pre.weight ? a.pre.weight[i] : 1.0f) +
                             (a.has_pre && a.pre.bias ? a.pre.bias[i] : 0.0f)};
        if (a.h) store_vec<1>(a.h, row * a.h_stride + i, hv, HT);
        if (!a.has_pre) continue;
        if (a.y_dtype == BYHIP_MXFP8_KM) write_mx1<BYHIP_MXFP8_KM>(a, row, i, yv[0]);
        else if (a.y_dtype == BYHIP_MXFP4_KM) write_mx1<BYHIP_MXFP4_KM>(a, row, i, yv[0]);
        else store_vec<1>(a.y, row * a.y_stride + i, yv, a.y_dtype);
    }
}

template <int XT, int HT>
void launch_norm(const NormArgs& a) {
    // Values per thread: many rows fill the card by themselves, and 16 per thread cost the fewest barriers per value (4099 x 5120
    // layer norms, 252 MB, half of what they read in the Infinity Cache: 67 us, with 8 per thread 74; all of it from memory 78 us, 3.2
    // TB/s); few rows take all the threads they can have (32 x 4096: 4.8 us, with 16 per
    // thread 5.2). What bounds the many is rows in flight: two rows a block that share the weights' loads took 103 us, the
    // weights' loads ahead of the sums 80 (both against the 67), for the registers that they hold.
    const bool few = a.M <= 2 * compute_units();
    const long long fours = ((long long)a.N + 3) / 4;
    const int ch = fours <= (few ? 1024 : 64) ? 1 : fours <= (few ? 2048 : 128) ? 2 : fours <= 4096 ? 4 : 8;
    const long long threads = ((fours + ch - 1) / ch + 63) / 64 * 64;
    const dim3 grid(a.M), block((unsigned)threads);
    if (a.has_pre && is_mx(a.y_dtype) && threads <= 1024) {
        if (ch == 1) launch("norm_block", (norm_block<XT, HT, 1, true>), grid, block, 0, a);
        else if (ch == 2) launch("norm_block", (norm_block<XT, HT, 2, true>), grid, block, 0, a);
        else if (ch == 4) launch("norm_block", (norm_block<XT, HT, 4, true>), grid, block, 0, a);
        else launch("norm_block", (norm_block<XT, HT, 8, true>), grid, block, 0, a);
        BYHIP_LAUNCHED("norm_block");
        return;
    }
    if (threads > 1024) launch("norm_block_long", (norm_block_long<XT, HT>), grid, dim3(1024), 0, a);
    else if (ch == 1) launch("norm_block", (norm_block<XT, HT, 1>), grid, block, 0, a);
    else if (ch == 2) launch("norm_block", (norm_block<XT, HT, 2>), grid, block, 0, a);
    else if (ch == 4) launch("norm_block", (norm_block<XT, HT, 4>), grid, block, 0, a);
    else launch("norm_block", (norm_block<XT, HT, 8>), grid, block, 0, a);
    BYHIP_LAUNCHED("norm_block");
}

template <int XT>
void launch_norm_x(const NormArgs& a) {
    switch (a.h_dtype) {
    case BYHIP_F32: launch_norm<XT, BYHIP_F32>(a); break;
    case BYHIP_F16: launch_norm<XT, BYHIP_F16>(a); break;
    default: launch_norm<XT, BYHIP_BF16>(a); break;
    }
}

void check_norm(const byhip_norm* n, int N, const char* what, int& vec) {
    if (n->kind != BYHIP_NORM_RMS && n->kind != BYHIP_NORM_LAYER) fail("byhip: %s norm kind %d", what, n->kind);
    if (!(n->eps >= 0.0f)) fail("byhip: %s norm eps %g", what, (double)n->eps);
    for (const float* p : {n->weight, n->bias}) {
        if (!p) continue;
        check_span(p, (size_t)N * 4, "norm weights");
        vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    }
}

}  // namespace
}  // namespace byhip

using namespace byhip;

extern "C" int byhip_norm_block(const void* x, size_t x_stride, int x_dtype, int M, int N, const byhip_norm* post,
                                const float* gate, size_t gate_stride, const void* res, size_t res_stride,
                                float res_scale, void* h, size_t h_stride, int h_dtype, const byhip_norm* pre,
                                void* y, size_t y_stride, int y_dtype) {
    return guard([&] {
        enter_compute();
        if (M < 0 || N <= 0) fail("byhip: norm of %d rows of %d values", M, N);
        if (!h && !pre) fail("byhip: norm_block without an output");
        NormArgs a{};
        a.M = M; a.N = N; a.res_scale = res_scale;
        check_rows(x, M, N, x_stride, x_dtype, "block output");
        int vec = aligned4(x, x_stride, x_dtype);
        if (!dtype_bytes(h_dtype)) fail("byhip: residual dtype %d", h_dtype);
        if (res) { check_rows(res, M, N, res_stride, h_dtype, "residual"); vec = vec && aligned4(res, res_stride, h_dtype); }
        if (h) { check_rows(h, M, N, h_stride, h_dtype, "residual output"); vec = vec && aligned4(h, h_stride, h_dtype); }
        if (h && h == res && h_stride != res_stride) fail("byhip: a residual updated in place needs one stride");
        if (gate) {
            if (gate_stride && gate_stride < (size_t)N) fail("byhip: gate stride %zu below its width %d", gate_stride, N);
            if (M) check_span(gate, ((size_t)(M - 1) * gate_stride + N) * 4, "gate");
            vec = vec && aligned4(gate, gate_stride, BYHIP_F32);
        }
        if (post) { check_norm(post, N, "post", vec); a.post = *post; a.has_post = 1; }
        if (pre) {
            check_norm(pre, N, "pre", vec);
            a.pre = *pre; a.has_pre = 1;
            if (is_mx(y_dtype)) {
                check_mx(y, M, N, y_dtype, "normed output");
                if (y_stride != (size_t)N) fail("byhip: normed output of %d values: microscaled rows have no stride of their own (%zu)", N, y_stride);
                a.y_scales = static_cast<uint8_t*>(y) + mx_values(M, N, y_dtype);
            } else {
                check_rows(y, M, N, y_stride, y_dtype, "normed output");
                vec = vec && aligned4(y, y_stride, y_dtype);
            }
        }
        if (M == 0) return;
        a.x = x; a.gate = gate; a.res = res; a.h = h; a.y = y; a.vec = vec;
        a.x_stride = x_stride; a.gate_stride = gate_stride; a.res_stride = res_stride;
        a.h_stride = h_stride; a.y_stride = y_stride; a.h_dtype = h_dtype; a.y_dtype = y_dtype;
        if (h) note_device_write(h);
        if (pre) note_device_write(y);
        switch (x_dtype) {
        case BYHIP_F32: launch_norm_x<BYHIP_F32>(a); break;
        case BYHIP_F16: launch_norm_x<BYHIP_F16>(a); break;
        default: launch_norm_x<BYHIP_BF16>(a); break;
        }
    });
}
