// byhip_moe.hip - entry points of the products of microscaled rows: with one matrix, and with each row's expert's.
#include "byhip_gemm.h"
#include "byhip_moe.h"

namespace byhip {
namespace {

// What both calls check; rows: x's rows, y_rows: y's.
MoeArgs product_args(const void* x, int x_format, const uint8_t* w, int experts, size_t rows, size_t y_rows, int K, int N, int flags,
                     void* y, size_t y_stride, int y_dtype) {
    const bool glu = flags & BYHIP_MOE_SWIGLU;
    if (K <= 0 || N <= 0) fail("byhip: a product of rows of %d values with %d outputs", K, N);
    MoeArgs a{};
    a.K = K; a.KG = K / 32; a.N = N;
    const long long R = glu ? 2ll * N : N;
    check_mx(x, rows, K, x_format, "rows of a product");
    // Offsets inside the rows and inside one matrix are 32-bit.
    if (mx_values(rows, K, x_format) >= 1ull << 31) fail("byhip: %zu rows of %d values: a product takes less than 2 GiB of them", rows, K);
    if (R > INT32_MAX / 2 || (unsigned long long)R * K / 2 >= 1ull << 31) fail("byhip: a matrix of %lld rows of %d values", R, K);
    a.R = (int)R;
    check_mx(w, (size_t)experts * R, K, BYHIP_MXFP4_KM, "matrices of a product");
    if (is_mx(y_dtype)) {
        check_mx(y, y_rows, N, y_dtype, "product");
        if (y_stride != (size_t)N) fail("byhip: product of %d values: microscaled rows have no stride of their own (%zu)", N, y_stride);
        a.ys = static_cast<uint8_t*>(y) + mx_values(y_rows, N, y_dtype);
    } else {
        check_rows(y, y_rows, N, y_stride, y_dtype, "product");
        // 1: four values at a time, 2: 16 bytes at a time
        const size_t bytes = dtype_bytes(y_dtype);
        a.vec = !aligned4(y, y_stride, y_dtype) ? 0 : reinterpret_cast<uintptr_t>(y) % 16 == 0 && y_stride * bytes % 16 == 0 ? 2 : 1;
    }
    a.x = static_cast<const uint8_t*>(x);
    a.x_bytes = (uint32_t)mx_values(rows, K, x_format);
    a.xs = a.x + a.x_bytes;
    a.xs_bytes = (uint32_t)(rows * a.KG);
    a.w = w;
    a.ws = w + mx_values((size_t)experts * R, K, BYHIP_MXFP4_KM);
    a.y = y; a.y_stride = y_stride; a.y_dtype = y_dtype;
    a.parts = x_format == BYHIP_MXFP8_KM && (y_dtype == BYHIP_F32 || flags & BYHIP_MOE_EXACT);
    return a;
}

// Whether tiles take a product: `units` is what can be told on the host of how many of 128 rows it has. A block of moe_tiles takes its time (30 us at K = 4096, 58 where 8-bit
// rows go in two parts) however few of its rows are real, so tiles need blocks enough and, where those do not fill the card, more products than moe_rows does in that
// time. Few rows per expert (us, moe_tiles / moe_rows; 128 experts, 2048 to 768 outputs of gates and ups, 6 / 8 / 10 / 12 / 24 each: 49 / 50 / 50 / 51 / 53 for
// 41 / 47 / 52 / 56 / 76; fp32: 16 / 24 / 32 each 77 / 77 / 79 for 65 / 77 / 90; 8 experts, 4096 to 14336, 8 / 12 each: 125 / 127 for 120 / 136). Few blocks (one matrix of 4096 x 4096, 256 / 384
// / 512 rows: 32 / 33 / 32 for 20 / 36 / 38, fp32 512 / 768 / 1024 rows: 60 / 61 / 61 for 38 / 56 / 72; 14336 x 4096, 64 / 96 / 128 rows: 31 / 32 / 32 for 22 / 32 / 40, fp32 128 / 256:
// 59 / 62 for 41 / 72; 8 experts, 14336 to 4096, 32 / 64 rows each: 123 / 130 for 98 / 153).
bool tiles_take(const MoeArgs& a, bool glu, long long rows, int units, int experts) {
    const int wide = glu ? 128 : 256;
    const long long blocks = (long long)units * ((a.N + wide - 1) / wide);
    return a.K % 128 == 0 && rows >= (a.parts ? 24ll : 10ll) * experts && (blocks >= 256 || rows * a.R >= (a.parts ? 3000000 : 1500000));
}

// Whether byhip_mxfp4_gemm's kernels take rows in 4 bits (with dense rows of 32 or 16 bits out): where there are more than one pass of moe_rows takes and products enough
// (us, mxfp4_gemm / here: 4096 x 4096, 16 / 64 / 80 / 192 / 512 rows 6.8 / 10.0 / 10.5 / 13.4 / 11.3 for 4.8 / 8.4 / 12.1 / 17.2 / 26.1; N = 14336, 16 / 32 / 64 / 256 rows 10.0 / 10.9 / 13.2
// / 18.9 for 9.3 / 11.1 / 24.4 / 29.2; K = 14336, 8 / 32 / 64 rows 9.7 / 10.9 / 13.3 for 10.2 / 15.4 / 19.8; 2048 x 2048, 64 / 256 rows 7.4 / 10.2 for 4.2 / 6.6). Rows of y
// that do not lie next to each other stay here.
bool mxfp4_takes(int M, int K, int N) {
    return K % 128 == 0 && M > 16 && (double)M * N * K >= 1.3e9 && mxfp4_fits(M, K, N);
}

}  // namespace
}  // namespace byhip

using namespace byhip;

extern "C" {

int byhip_mx_matmul(const void* x, int x_format, const uint8_t* w, int M, int K, int N, int flags, void* y, size_t y_stride,
                    int y_dtype) {
    return guard([&] {
        enter_compute();
        if (M < 0) fail("byhip: a product of %d rows", M);
        if (flags & ~(BYHIP_MOE_SWIGLU | BYHIP_MOE_EXACT)) fail("byhip: product flags %d without a plan", flags);
        const bool glu = flags & BYHIP_MOE_SWIGLU;
        MoeArgs a = product_args(x, x_format, w, 1, M, M, K, N, flags, y, y_stride, y_dtype);
        if (M == 0) return;
        note_device_write(y);
        if (x_format == BYHIP_MXFP4_KM && !glu && !is_mx(y_dtype) && y_stride == (size_t)N && mxfp4_takes(M, K, N)) {
            launch_mxfp4(a.x, a.xs, a.w, a.ws, y, y_dtype, M, K, N);
            return;
        }
        a.M = M; a.top_k = 1;
        const int tiles = (M + kTileRows - 1) / kTileRows;
        if (tiles_take(a, glu, M, tiles, 1)) {
            a.unit_rows = kTileRows;
            launch_moe_tiles(a, x_format, glu, tiles);
        } else {
            a.unit_rows = moe_unit_rows(M, 1);
            launch_moe_rows(a, x_format, glu, (M + a.unit_rows - 1) / a.unit_rows);
        }
    });
}

int byhip_moe_matmul(const void* x, int x_format, const uint8_t* w, const byhip_moe_plan* plan, int K, int N, int flags, void* y,
                     size_t y_stride, int y_dtype) {
    return guard([&] {
        enter_compute();
        const MoePlan p = moe_plan_args(plan);
        if (flags & ~(BYHIP_MOE_GATHER | BYHIP_MOE_SCATTER | BYHIP_MOE_SWIGLU | BYHIP_MOE_EXACT)) fail("byhip: product flags %d", flags);
        const bool glu = flags & BYHIP_MOE_SWIGLU, gather = flags & BYHIP_MOE_GATHER;
        MoeArgs a = product_args(x, x_format, w, p.experts, gather ? p.tokens : p.rows, p.rows, K, N, flags, y, y_stride, y_dtype);
        if (p.rows == 0) return;
        a.order = p.order;
        a.top_k = p.top_k; a.gather = gather; a.scatter = (flags & BYHIP_MOE_SCATTER) != 0;
        a.experts = p.experts; a.rows = p.rows;
        a.per_token = (uint32_t)(((1ull << 32) + p.top_k - 1) / p.top_k);
        note_device_write(y);
        if (tiles_take(a, glu, p.rows, p.max_tiles, p.experts)) {
            a.n_units = p.n_units + 1; a.units = p.tiles; a.max_units = p.max_tiles;
            a.unit_rows = kTileRows;
            launch_moe_tiles(a, x_format, glu, p.max_tiles);
        } else {
            a.n_units = p.n_units; a.units = p.units; a.max_units = p.max_units;
            a.unit_rows = p.unit_rows;
            launch_moe_rows(a, x_format, glu, p.max_units);
        }
    });
}

}  // extern "C"
