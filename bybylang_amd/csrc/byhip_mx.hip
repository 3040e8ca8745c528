// byhip_mx.hip - rows of 32 or 16 bits to microscaled rows (gfx950).
//
// One pass: a group's 32 values are read once, its largest magnitude is found across the 4 lanes that hold them, and the
// rounded values and the scale byte are written. Bound by memory.
#include "byhip_mx.h"

namespace byhip {
namespace {

struct QuantArgs {
    const void* x;
    uint8_t* y;
    uint8_t* scales;
    size_t stride;
    int K, M, groups, vec;
};

// Four lanes per group: lane t of them holds elements 4 t .. 4 t + 3 and 16 + 4 t .. + 3, which lie next to each other
// in memory order.
template <int XT, int FMT>
__global__ __launch_bounds__(256) void mx_quantize(QuantArgs a) {
    const int t = threadIdx.x & 3;
    const int G = blockIdx.x * 64 + (threadIdx.x >> 2);
    if (G >= a.groups) return;
    const size_t row = blockIdx.y;
    const int j = 4 * t;
    for (size_t r = row; r < (size_t)a.M; r += gridDim.y) {
        const size_t at = r * a.stride + 32 * (size_t)G + j;
        float lo[4], hi[4];
        if (a.vec) {
            load_vec<XT, 4>(a.x, at, lo);
            load_vec<XT, 4>(a.x, at + 16, hi);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo[e] = load1<XT>(a.x, at + e);
                hi[e] = load1<XT>(a.x, at + 16 + e);
            }
        }
        uint32_t m = mag8(lo, hi);
        m = max(m, (uint32_t)__shfl_xor((int)m, 1));
        m = max(m, (uint32_t)__shfl_xor((int)m, 2));
        const uint32_t byte = mx_scale<FMT>(m);
        uint32_t out[2];
        mx_pack8<FMT>(lo, hi, byte, out);
        mx_store8<FMT>(a.y, r, a.K, G, j, out);
        if (t == 0) a.scales[r * a.groups + G] = (uint8_t)byte;
    }
}

template <int XT>
void launch_quant(const QuantArgs& a, int fmt) {
    const dim3 grid((a.groups + 63) / 64, std::min(a.M, 65535));
    if (fmt == BYHIP_MXFP8_KM) launch("mx_quantize", (mx_quantize<XT, BYHIP_MXFP8_KM>), grid, dim3(256), 0, a);
    else launch("mx_quantize", (mx_quantize<XT, BYHIP_MXFP4_KM>), grid, dim3(256), 0, a);
    BYHIP_LAUNCHED("mx_quantize");
}

}  // namespace

void check_mx(const void* p, size_t rows, size_t K, int fmt, const char* what) {
    if (!is_mx(fmt)) fail("byhip: %s format %d", what, fmt);
    if (K == 0 || K % 32) fail("byhip: %s of %zu values, not a multiple of 32", what, K);
    if (rows == 0) return;
    check_span(p, mx_bytes(rows, K, fmt), what);
    if (reinterpret_cast<uintptr_t>(p) % 16) fail("byhip: %s must be 16-byte aligned", what);
}

}  // namespace byhip

using namespace byhip;

extern "C" int byhip_mx_quantize(const void* x, size_t x_stride, int x_dtype, int M, int K, void* y, int y_format) {
    return guard([&] {
        enter_compute();
        if (M < 0 || K <= 0) fail("byhip: quantisation of %d rows of %d values", M, K);
        check_rows(x, M, K, x_stride, x_dtype, "rows to quantise");
        check_mx(y, M, K, y_format, "microscaled rows");
        if (M == 0) return;
        uint8_t* out = static_cast<uint8_t*>(y);
        const QuantArgs a{x, out, out + mx_values(M, K, y_format), x_stride, K, M, K / 32, aligned4(x, x_stride, x_dtype)};
        note_device_write(y);
        switch (x_dtype) {
        case BYHIP_F32: launch_quant<BYHIP_F32>(a, y_format); break;
        case BYHIP_F16: launch_quant<BYHIP_F16>(a, y_format); break;
        default: launch_quant<BYHIP_BF16>(a, y_format); break;
        }
    });
}
