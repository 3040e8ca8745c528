// byhip_moe_tiles.hip - many rows per expert (gfx950): products in tiles of 256 matrix rows and 128 rows of x.
//
// Bound by the matrix instructions: v_mfma_scale_f32_32x32x64_f8f6f4, matrix first (operands as in byhip_moe_rows.hip with 2 lane
// groups instead of 4: lane (c, g) = (l % 32, l / 32) holds block g of row c; in 8 bits its two pieces are half g of block 0 and
// of block 1). A block of 4 waves holds the tile's sums in 128 accumulators per lane (wave: 128 matrix rows x 64 rows). A step is 128
// values: 16 products of 64 cycles per wave with rows in 8 bits, half of that in 4 bits.
//
// Two blocks share a CU, each wave of one on a SIMD with one of the other: while one looks its rows up, waits at a barrier, reads operands or
// writes its tile, the other multiplies. One block per CU that did all of that between its own products (operands read a step
// ahead, the next tile's loads out before this one's results) left the matrix unit idle for half of the time: 12000 of a tile's 34000
// cycles went outside the steps.
//
// With rows in 8 bits and outputs of 16 bits or fewer, the instructions' cut (split_bytes) stays: 5e-6 to 1e-5 of a product's norm, less than a hundredth of the
// rounding that follows. (Of outputs in 8 bits one in a thousand then takes the step next to its own: 0.0023 of their norm, where the steps' rounding is
// 0.026.) It is more where large terms cancel. In two parts, as with fp32 outputs and where the caller asks for it, they take half as long again: 4096 tokens, 6 of 64
// experts, 2048 to 1408, 246 us for 157.
//
// A step's data goes straight into LDS (16 bytes per lane) while the step before multiplies: two slots, one barrier per step. The
// order of the 16-byte pieces inside a row is turned by the row so that no cycle of the operand reads meets a bank twice.
#include <algorithm>

#include "byhip_moe.h"

namespace byhip {
namespace {

constexpr int kStep = 128, kTileW = 256, kTileX = kTileRows;
constexpr uint32_t kNoRow = 0x80000000u;  // past every range here (below 2 GiB), also with a step's offset added

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// LDS: two slots of a step's values, W (256 rows of 64 bytes) and X (128 rows of 128 or 64 bytes), then two buffers of scales (16 bytes per
// row of W and X: 4 steps of 4).
template <int XF>
struct Lds {
    static constexpr bool eight = XF == BYHIP_MXFP8_KM;
    static constexpr int w = kTileW * 64, x = kTileX * (eight ? 128 : 64);
    static constexpr int slot = w + x, scales = (kTileW + kTileX) * 16, scale_base = 2 * slot, bytes = scale_base + 2 * scales;
};

// How a row's pieces are turned (xor). Rows of 64 bytes: four fill all banks, so rows 4 apart differ; rows of 128 bytes: two do. In either 16 rows
// of one piece, and 8 rows of the two pieces that the lane groups read (2 apart in 64 bytes, next to each other in 128), meet 16 places.
__device__ __forceinline__ int turn4(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int turn8(int r) { return (r & 6) | (r >> 3 & 1); }

template <int XF, int H>  // H: the half, and the scales' byte
__device__ __forceinline__ f16v product(v4u w, v8i x, f16v c, int sw, int sx) {
    const v8i wide = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide, x, c, 4, XF == BYHIP_MXFP8_KM ? 0 : 4, H, sw, H, sx);
}

// Halves of a wave's registers changed over: x becomes (x of the lower lanes, y of the lower lanes), y the same of the upper lanes.
__device__ __forceinline__ void swap_halves(uint32_t& x, uint32_t& y) {
    const auto v = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = v[0];
    y = v[1];
}

// 32 outputs n .. n + 31 of a row, of which this lane holds 8 b + 4 lq .. + 3 (v[b]) and the lane 32 further on or back the rest: the
// two change over so that each stores 16 neighbouring bytes (of 16-bit outputs and 8-bit values).
template <int YT>
__device__ __forceinline__ void write_block(const MoeArgs& a, bool there, size_t row, int n, int lq, float (&v)[4][4]) {
    if constexpr (YT == BYHIP_MXFP8_KM || YT == BYHIP_MXFP4_KM) {
        uint8_t* y = static_cast<uint8_t*>(a.y);
        uint32_t mag = max(mag8(v[0], v[1]), mag8(v[2], v[3]));
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
        const uint32_t byte = mx_scale<YT>(mag);
        uint32_t p[2], q[2];
        mx_pack8<YT>(v[0], v[2], byte, p);
        mx_pack8<YT>(v[1], v[3], byte, q);
        swap_halves(p[0], q[0]);
        if constexpr (YT == BYHIP_MXFP8_KM) swap_halves(p[1], q[1]);
        if (!there) return;
        if constexpr (YT == BYHIP_MXFP8_KM) *reinterpret_cast<uint4*>(y + row * a.N + n + 16 * lq) = make_uint4(p[0], p[1], q[0], q[1]);
        else *reinterpret_cast<uint2*>(y + row * (a.N / 2) + n / 2 + 8 * lq) = make_uint2(p[0], q[0]);
        if (lq == 0) a.ys[row * (a.N / 32) + n / 32] = (uint8_t)byte;
    } else if (a.vec == 2 && n + 32 <= a.N) {
        if constexpr (YT == BYHIP_F32) {
            if (!there) return;
            float4* y = reinterpret_cast<float4*>(static_cast<float*>(a.y) + row * a.y_stride + n + 4 * lq);
#pragma unroll
            for (int b = 0; b < 4; ++b) y[2 * b] = make_float4(v[b][0], v[b][1], v[b][2], v[b][3]);
        } else {
            uint32_t w[4][2];
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    w[b][h] = YT == BYHIP_F16 ? h_bits((_Float16)v[b][2 * h]) | (uint32_t)h_bits((_Float16)v[b][2 * h + 1]) << 16 : f32x2_to_bf16x2_bits(v[b][2 * h], v[b][2 * h + 1]);
#pragma unroll
            for (int b = 0; b < 4; b += 2)
#pragma unroll
                for (int h = 0; h < 2; ++h) swap_halves(w[b][h], w[b + 1][h]);
            if (!there) return;
            uint16_t* y = static_cast<uint16_t*>(a.y) + row * a.y_stride + n + 8 * lq;
#pragma unroll
            for (int b = 0; b < 4; b += 2) *reinterpret_cast<uint4*>(y + 8 * b) = make_uint4(w[b][0], w[b][1], w[b + 1][0], w[b + 1][1]);
        }
    } else if (there) {
        for (int b = 0; b < 4; ++b) {
            float four[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) four[e] = b == 0 ? v[0][e] : b == 1 ? v[1][e] : b == 2 ? v[2][e] : v[3][e];
            const size_t at = row * a.y_stride + n + 8 * b + 4 * lq;
            for (int e = 0; e < 4; ++e)
                if (n + 8 * b + 4 * lq + e < a.N) store_y<YT>(a.y, at + e, e == 0 ? four[0] : e == 1 ? four[1] : e == 2 ? four[2] : four[3]);
        }
    }
}

template <int XF, bool GLU, int YT, bool FINE>
__global__ __launch_bounds__(256, 2) void moe_tiles(MoeArgs a) {
    typedef Lds<XF> L;
    constexpr bool eight = L::eight;
    static_assert(eight || !FINE, "rows in 4 bits are exact in one part");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[L::bytes];
    MoeUnit u;
    int strip;
    if (!MoeTiles(a).find(a, blockIdx.x >> 3, u, strip)) return;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wid >> 1, wt = wid & 1, lq = lane >> 5, lc = lane & 31;
    const uint32_t kb = (uint32_t)a.K / 2, xb = eight ? (uint32_t)a.K : kb, KG = (uint32_t)a.KG;
    const rsrc_t wr = make_rsrc(a.w + (size_t)u.expert * a.R * kb, (uint32_t)a.R * kb);
    const rsrc_t wsr = make_rsrc(a.ws + (size_t)u.expert * a.R * KG, (uint32_t)a.R * KG);
    const rsrc_t xr = make_rsrc(a.x, a.x_bytes), xsr = make_rsrc(a.xs, a.xs_bytes);

    // The matrix's row of the tile's row R: a wave's 128 are 64 gates and the ups of the same outputs.
    const int n0 = strip * (GLU ? kTileW / 2 : kTileW);
    auto matrix_row = [&](int R) {
        if constexpr (!GLU) return n0 + R;
        return ((R >> 6) & 1) * a.N + n0 + 64 * (R >> 7) + (R & 63);
    };
    // Offsets of this lane's loads, each 1 KB of a wave: rows of W 64 wid + 16 q + l / 4, rows of X 32 wid + 8 q + l / 8 (8 bits) or 32 wid + 16 q +
    // l / 4; a row past the matrix's or the unit's reads zeros.
    constexpr int kLoadsX = eight ? 4 : 2;
    uint32_t wo[4], xo[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int R = 64 * wid + 16 * q + (lane >> 2), n = matrix_row(R);
        wo[q] = n < a.R ? (uint32_t)n * kb + 16u * ((lane & 3) ^ turn4(R & 15)) : kNoRow;
    }
#pragma unroll
    for (int q = 0; q < kLoadsX; ++q) {
        const int R = eight ? 32 * wid + 8 * q + (lane >> 3) : 32 * wid + 16 * q + (lane >> 2);
        const uint32_t c = 16u * (eight ? (lane & 7) ^ turn8(R & 15) : (lane & 3) ^ turn4(R & 15));
        xo[q] = R < u.rows ? (uint32_t)moe_x_row(a, u.first + R) * xb + c : kNoRow;
    }
    const int swn = matrix_row(64 * wid + lane), sxr = 64 * wid + lane;
    const uint32_t wso = swn < a.R ? (uint32_t)swn * KG : kNoRow;
    const uint32_t xso = wid < 2 && sxr < u.rows ? (uint32_t)moe_x_row(a, u.first + sxr) * KG : kNoRow;

    const int nsteps = a.K / kStep;
    // Scales of steps 4 p .. 4 p + 3; past the last they are bytes that no step uses.
    auto load_scales = [&](int p) {
        uint8_t* buf = lds + L::scale_base + (p & 1) * L::scales;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (lds_void*)(buf + wid * 1024), 16, wso, 16 * p, 0, 0);
        if (wid < 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(xsr, (lds_void*)(buf + kTileW * 16 + wid * 1024), 16, xso, 16 * p, 0, 0);
    };
    auto load_step = [&](int s) {
        uint8_t* slot = lds + (s & 1) * L::slot;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(slot + (4 * wid + q) * 1024), 16, wo[q], 64 * s, 0, 0);
#pragma unroll
        for (int q = 0; q < kLoadsX; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(slot + L::w + (kLoadsX * wid + q) * 1024), 16, xo[q], (eight ? 128 : 64) * s, 0, 0);
    };

    // This lane's pieces of a step: of half h, group 2 g + h for the lane group g; of an 8-bit row, block b's.
    int w_at[2], x_at[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w_at[h] = 64 * (128 * wn + lc) + 16 * ((2 * lq + h) ^ turn4(lane & 15));
#pragma unroll
        for (int b = 0; b < 2; ++b)
            x_at[h][b] = L::w + (eight ? 128 * (64 * wt + lc) + 16 * ((4 * b + 2 * h + lq) ^ turn8(lane & 15)) : 64 * (64 * wt + lc) + 16 * ((2 * lq + h) ^ turn4(lane & 15)));
    }
    const int sw_at = L::scale_base + 16 * (128 * wn + lc) + 2 * lq, sx_at = L::scale_base + 16 * (kTileW + 64 * wt + lc) + 2 * lq;

    f16v acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
#ifdef __HIP_DEVICE_COMPILE__  // (the host's compiler has no such registers)
            asm volatile("" : "+v"(acc[i][j]));  // zeros in registers, not a constant addend (byhip_moe_rows.hip)
#endif
        }

    load_scales(0);
    load_step(0);
#pragma unroll 1
    for (int s = 0; s < nsteps; ++s) {
        // Step s has landed, and every wave is done with the slot (and the scales) that are loaded into now.
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < nsteps) load_step(s + 1);
        if ((s & 3) == 1) load_scales((s + 3) >> 2);
        [&](const uint8_t* __restrict__ slot, const uint8_t* __restrict__ sc) {
            int sw[4], sx[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) sw[i] = *reinterpret_cast<const uint16_t*>(sc + sw_at + 512 * i);
#pragma unroll
            for (int j = 0; j < 2; ++j) sx[j] = *reinterpret_cast<const uint16_t*>(sc + sx_at + 512 * j);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v8i x[2], small[2];
                v4u w[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const v4u p = *reinterpret_cast<const v4u*>(slot + x_at[h][0] + j * (eight ? 4096 : 2048));
                    const v4u q = eight ? *reinterpret_cast<const v4u*>(slot + x_at[h][1] + j * 4096) : v4u{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; ++e) { x[j][e] = (int)p[e]; x[j][4 + e] = (int)q[e]; }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const v4u*>(slot + w_at[h] + 2048 * i);
                auto add = [&](const v8i (&x)[2]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            acc[i][j] = h == 0 ? product<XF, 0>(w[i], x[j], acc[i][j], sw[i], sx[j]) : product<XF, 1>(w[i], x[j], acc[i][j], sw[i], sx[j]);
                };
                if constexpr (FINE) {
                    split_bytes(x[0], x[0], small[0]);
                    split_bytes(x[1], x[1], small[1]);
                    add(small);
                }
                add(x);
            }
        }(lds + (s & 1) * L::slot, lds + ((s >> 2) & 1) * L::scales + 4 * (s & 3));
    }

    // Lane (c, g) holds row c of block j of x; register r is matrix row 8 (r / 4) + 4 g + r % 4 of block i.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int R = 64 * wt + 32 * j + lc;
        const bool there = R < u.rows;
        const size_t row = there ? moe_y_row(a, u.first + R) : 0;
#pragma unroll
        for (int i = 0; i < (GLU ? 2 : 4); ++i) {
            float v[4][4];
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[b][e] = GLU ? swiglu(acc[i][j][4 * b + e], acc[GLU ? 2 + i : i][j][4 * b + e]) : acc[i][j][4 * b + e];
            const int n = n0 + (GLU ? 64 : 128) * wn + 32 * i;
            write_block<YT>(a, there && n < a.N, row, n, lq, v);
        }
    }
}

template <int XF, bool GLU, int YT>
void launch_tiles(const MoeArgs& a, const dim3& grid) {
    constexpr bool eight = XF == BYHIP_MXFP8_KM;
    if (eight && a.parts) launch("moe_tiles", (moe_tiles<XF, GLU, YT, eight>), grid, dim3(256), 0, a);
    else launch("moe_tiles", (moe_tiles<XF, GLU, YT, false>), grid, dim3(256), 0, a);
    BYHIP_LAUNCHED("moe_tiles");
}
template <int XF, bool GLU>
void launch_tiles_y(const MoeArgs& a, const dim3& grid) {
    switch (a.y_dtype) {
    case BYHIP_F32: launch_tiles<XF, GLU, BYHIP_F32>(a, grid); break;
    case BYHIP_F16: launch_tiles<XF, GLU, BYHIP_F16>(a, grid); break;
    case BYHIP_BF16: launch_tiles<XF, GLU, BYHIP_BF16>(a, grid); break;
    case BYHIP_MXFP8_KM: launch_tiles<XF, GLU, BYHIP_MXFP8_KM>(a, grid); break;
    default: launch_tiles<XF, GLU, BYHIP_MXFP4_KM>(a, grid); break;
    }
}

}  // namespace

void launch_moe_tiles(const MoeArgs& args, int x_format, bool glu, int max_units) {
    MoeArgs a = args;
    if (a.unit_rows != kTileX || a.K % kStep) fail("byhip: internal: units of %d rows, %d values", a.unit_rows, a.K);
    const int wide = glu ? kTileW / 2 : kTileW;
    a.strips = (a.N + wide - 1) / wide;
    const long long blocks = ((long long)max_units * a.strips + 7) / 8 * 8;
    if (blocks >= 1ll << 31) fail("byhip: a product of %d units of %d strips", max_units, a.strips);
    const dim3 grid((unsigned)blocks);
    if (x_format == BYHIP_MXFP4_KM) glu ? launch_tiles_y<BYHIP_MXFP4_KM, true>(a, grid) : launch_tiles_y<BYHIP_MXFP4_KM, false>(a, grid);
    else glu ? launch_tiles_y<BYHIP_MXFP8_KM, true>(a, grid) : launch_tiles_y<BYHIP_MXFP8_KM, false>(a, grid);
}

}  // namespace byhip
