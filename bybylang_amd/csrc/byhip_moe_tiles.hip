// byhip_moe_tiles.hip - many rows per expert (gfx950): products in tiles of 256 matrix rows and 128 rows of x.
//
// Bound by the matrix instructions: v_mfma_scale_f32_32x32x64_f8f6f4, matrix first (operands as in byhip_moe_rows.hip with 2 lane
// groups instead of 4: lane (c, g) = (l % 32, l / 32) holds block g of row c; in 8 bits its two pieces are half g of block 0 and
// of block 1). A block of 4 waves, one per SIMD, holds the tile's sums in 128 accumulators per lane (wave: 128 matrix rows x 64 rows). A
// step is 128 values: 16 products of 64 cycles per wave with rows in 8 bits, half of that in 4 bits.
//
// Loads go straight into LDS (16 bytes per lane, whole 128-byte lines: two steps of a matrix row at once), two pairs of
// steps ahead in two regions; scales follow once per 4 steps. During the products of step s the wave reads step s + 1's
// operands. One barrier per pair. The order of the loads inside a row's 128 (or 64) bytes is turned by the row so that no
// cycle of the operand reads meets a bank twice: 16 lanes read one place of 16 rows, which lie 128 bytes apart (8 bits), two to all 64
// banks, or 64 bytes apart (4 bits), four to all banks.
#include <algorithm>

#include "byhip_moe.h"

namespace byhip {
namespace {

constexpr int kStep = 128, kTileW = 256, kTileX = 128;
constexpr uint32_t kNoRow = 0x80000000u;  // past every range here (below 2 GiB), also with a step's offset added

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// LDS: two regions of W (256 rows, two steps: blocks of 8 rows, step e's 64 bytes of each in the first 512 bytes, step e + 1's in the second)
// and X (in 8 bits: step e's 128 rows of 128 bytes, then step e + 1's; in 4 bits as W), then two buffers of scales (16 bytes
// per row of W and X: 4 steps of 4).
template <int XF>
struct Lds {
    static constexpr bool eight = XF == BYHIP_MXFP8_KM;
    static constexpr int w = kTileW * 128, x_step = kTileX * 128, x = eight ? 2 * x_step : kTileX * 128;
    static constexpr int region = w + x, scales = (kTileW + kTileX) * 16, scale_base = 2 * region;
    static constexpr int bytes = scale_base + 2 * scales;
};

__device__ __forceinline__ int turn64(int r) { return (r ^ (r >> 2)) & 3; }
__device__ __forceinline__ int turn128(int r) { return (r >> 1) & 7; }

template <int N>
__device__ __forceinline__ void stage_barrier() {
    wait_vmcnt<N>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int XF>
struct Operands {
    v4u w[4][2];                                     // 4 blocks of 32 matrix rows, two halves of the step
    v4u x[2][2][XF == BYHIP_MXFP8_KM ? 2 : 1];       // 2 blocks of 32 rows
    int sw[4], sx[2];                                // scales of both halves
};

template <int XF, int H>
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

template <int XF, bool GLU, int YT>
__global__ __launch_bounds__(256) void moe_tiles(MoeArgs a) {
    typedef Lds<XF> L;
    constexpr bool eight = L::eight, FINE = eight && YT == BYHIP_F32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[L::bytes];
    const MoeTiles tiles(a);
    const int round = gridDim.x >> 3;
    int at = blockIdx.x >> 3;
    MoeUnit u;
    int strip;
    if (!tiles.find(a, at, u, strip)) return;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wid >> 1, wt = wid & 1, lq = lane >> 5, lc = lane & 31;
    const uint32_t kb = (uint32_t)a.K / 2, xb = eight ? (uint32_t)a.K : kb, KG = (uint32_t)a.KG;
    const rsrc_t xr = make_rsrc(a.x, a.x_bytes), xsr = make_rsrc(a.xs, a.xs_bytes);
    const int drow = lc >> 2;

    // A tile's rows of x for this lane's loads: rows of X 32 wid + 8 q + .. for its values, row 64 wid + lane for its scales; -1 past the
    // unit's. Asked for a tile ahead.
    auto ask_rows = [&](const MoeUnit& u, int (&rows)[5]) {
#pragma unroll
        for (int q = 0; q < 5; ++q) {
            const int R = q < 4 ? 32 * wid + 8 * q + (eight ? lane >> 3 : drow) : 64 * wid + lane;
            rows[q] = R >= u.rows ? -1 : a.gather ? a.order[u.first + R] : u.first + R;
        }
    };
    // Where a tile's operands are: offsets of this lane's loads, rows of W 64 wid + 8 q + ..; a row past the matrix's or the unit's reads
    // zeros.
    rsrc_t wr, wsr;
    uint32_t wo[8], xo[4], wso, xso;
    auto locate = [&](const MoeUnit& u, int strip, const int (&rows)[5]) {
        wr = make_rsrc(a.w + (size_t)u.expert * a.R * kb, (uint32_t)a.R * kb);
        wsr = make_rsrc(a.ws + (size_t)u.expert * a.R * KG, (uint32_t)a.R * KG);
        // The matrix's row of the tile's row R: a wave's 128 are 64 gates and the ups of the same outputs.
        const int n0 = strip * (GLU ? kTileW / 2 : kTileW);
        auto matrix_row = [&](int R) {
            if constexpr (!GLU) return n0 + R;
            return ((R >> 6) & 1) * a.N + n0 + 64 * (R >> 7) + (R & 63);
        };
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int R = 64 * wid + 8 * q + drow, n = matrix_row(R);
            wo[q] = n < a.R ? (uint32_t)n * kb + 16u * ((lane & 3) ^ turn64(R & 15)) + 64u * lq : kNoRow;
        }
        auto x_row = [&](int id) { return a.gather ? min((unsigned)id, (unsigned)a.rows - 1u) / (unsigned)a.top_k : (unsigned)id; };
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int R = 32 * wid + 8 * q + (eight ? lane >> 3 : drow);
            const uint32_t c = eight ? 16u * ((lane & 7) ^ turn128(R & 15)) : 16u * ((lane & 3) ^ turn64(R & 15)) + 64u * lq;
            xo[q] = R < u.rows ? x_row(rows[q]) * xb + c : kNoRow;
        }
        const int n = matrix_row(64 * wid + lane);
        wso = n < a.R ? (uint32_t)n * KG : kNoRow;
        xso = wid < 2 && 64 * wid + lane < u.rows ? x_row(rows[4]) * KG : kNoRow;
    };

    const int nsteps = a.K / kStep;
    // Loads past the last step read it again, or bytes that no step uses.
    auto load_scales = [&](int p, uint8_t* buf) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (lds_void*)(buf + wid * 1024), 16, wso, 16 * p, 0, 0);
        if (wid < 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(xsr, (lds_void*)(buf + kTileW * 16 + wid * 1024), 16, xso, 16 * p, 0, 0);
    };
    constexpr int kLoads = eight ? 16 : 12;  // per lane and pair of steps
    auto load_one = [&](int k, int e, uint8_t* reg) {
        const int s = min(e, nsteps - 1);
        if (k < 8) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(reg + (8 * wid + k) * 1024), 16, wo[k], s * 64, 0, 0);
        } else if constexpr (eight) {
            const int q = (k - 8) & 3, h = (k - 8) >> 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(reg + L::w + h * L::x_step + (4 * wid + q) * 1024), 16, xo[q], s * 128 + 128 * h, 0, 0);
        } else {
            const int q = k - 8;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(reg + L::w + (4 * wid + q) * 1024), 16, xo[q], s * 64, 0, 0);
        }
    };
    auto load_pair = [&](int e, uint8_t* reg) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) load_one(k, e, reg);
    };

    // Operand reads of a step: read k of 16 (8 bits) or 12.
    int at64[2], at128[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        at64[h] = 1024 * (lc >> 3) + 64 * (lane & 7) + 16 * ((2 * lq + h) ^ turn64(lane & 15));
#pragma unroll
        for (int b = 0; b < 2; ++b) at128[h][b] = 128 * lc + 16 * ((4 * b + 2 * h + lq) ^ turn128(lane & 15));
    }
    // `reg` is the step's region, `odd` whether it is the second of its pair.
    auto read_one = [&](Operands<XF>& o, const uint8_t* reg, int odd, int k) {
        if (k < 8) {
            const int F = k & 3, h = k >> 2;
            o.w[F][h] = *reinterpret_cast<const v4u*>(reg + 512 * odd + (16 * wn + 4 * F) * 1024 + at64[h]);
        } else if constexpr (eight) {
            const int J = k & 1, h = (k >> 2) & 1, b = (k >> 1) & 1;
            o.x[J][h][b] = *reinterpret_cast<const v4u*>(reg + L::w + odd * L::x_step + (64 * wt + 32 * J) * 128 + at128[h][b]);
        } else {
            const int J = k & 1, h = (k >> 1) & 1;
            o.x[J][h][0] = *reinterpret_cast<const v4u*>(reg + L::w + 512 * odd + (8 * wt + 4 * J) * 1024 + at64[h]);
        }
    };
    auto read_scale = [&](Operands<XF>& o, const uint8_t* sbuf, int T, int k) {
        if (k < 4) o.sw[k] = *reinterpret_cast<const uint16_t*>(sbuf + 16 * (128 * wn + 32 * k + lc) + 2 * lq + 4 * T);
        else o.sx[k - 4] = *reinterpret_cast<const uint16_t*>(sbuf + 16 * (kTileW + 64 * wt + 32 * (k - 4) + lc) + 2 * lq + 4 * T);
    };

    int rows[5];
    ask_rows(u, rows);
    locate(u, strip, rows);
    auto region_at = [&](int s) { return lds + ((s >> 1) & 1) * L::region; };
    auto sbuf_at = [&](int s) { return lds + L::scale_base + ((s >> 2) & 1) * L::scales; };
    load_scales(0, sbuf_at(0));
    load_pair(0, region_at(0));
    load_pair(2, region_at(2));
    bool more = true;
    while (more) {
    // The next tile's unit and rows are asked for now, and its first loads go out before this one's results are written.
    MoeUnit u1 = u;
    int strip1 = 0;
    at += round;
    more = tiles.find(a, at, u1, strip1);
    if (more) ask_rows(u1, rows);

    f16v acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
            asm volatile("" : "+v"(acc[i][j]));  // zeros in registers, not a constant addend (byhip_moe_rows.hip)
        }

    // At the start of step s `cur` holds its operands, and step s + 1's data and scales have landed. Step s reads them into `nxt`. An odd
    // step issues the loads of the pair s + 3, s + 4 into the region of the pair s - 1, s, whose last reads (for step s) were
    // in step s - 1, before the barrier that ended it; at s % 4 = 1 also the scales of period (s + 3) / 4. An even step ends with a
    // wait for all loads and the barrier. The pointers of a step are distinct, and __restrict__ says so: its reads need not wait
    // for its loads.
    Operands<XF> o0, o1;
    [&](const uint8_t* __restrict__ sc, const uint8_t* __restrict__ r0) {
        stage_barrier<kLoads>();  // the second pair, or what was written after it, may be on its way
#pragma unroll
        for (int k = 0; k < kLoads; ++k) read_one(o0, r0, 0, k);
#pragma unroll
        for (int k = 0; k < 6; ++k) read_scale(o0, sc, 0, k);
    }(sbuf_at(0), region_at(0));

    auto step = [&](auto Pc, int s, Operands<XF>& cur, Operands<XF>& nxt, uint8_t* __restrict__ dreg, uint8_t* __restrict__ sdst,
                    const uint8_t* __restrict__ src, const uint8_t* __restrict__ ssrc) {
        constexpr int P = decltype(Pc)::value;
        constexpr bool odd = P & 1;
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            const int h = m >> 3, j = (m >> 2) & 1, i = m & 3;
            v8i x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = (int)cur.x[j][h][0][e];
                x[4 + e] = eight ? (int)cur.x[j][h][eight ? 1 : 0][e] : 0;
            }
            if constexpr (FINE) {
                v8i large, small;
                split_bytes(x, large, small);
                acc[i][j] = h == 0 ? product<XF, 0>(cur.w[i][0], small, acc[i][j], cur.sw[i], cur.sx[j]) : product<XF, 1>(cur.w[i][1], small, acc[i][j], cur.sw[i], cur.sx[j]);
                x = large;
            }
            acc[i][j] = h == 0 ? product<XF, 0>(cur.w[i][0], x, acc[i][j], cur.sw[i], cur.sx[j]) : product<XF, 1>(cur.w[i][1], x, acc[i][j], cur.sw[i], cur.sx[j]);
            __builtin_amdgcn_sched_barrier(0);
            if (m < kLoads) read_one(nxt, src, !odd, m);
            if (m >= 10) read_scale(nxt, ssrc, (P + 1) & 3, m - 10);
            if constexpr (odd) {
                if (P == 1 && m == 1) load_scales((s + 3) >> 2, sdst);
                if (m < kLoads) load_one(m, s + 3, dreg);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!odd) stage_barrier<0>();
        __builtin_amdgcn_sched_barrier(0);
    };
#define BYHIP_STEP(P, S, CUR, NXT) \
    step(std::integral_constant<int, P>{}, S, CUR, NXT, region_at((S) + 3), sbuf_at((S) + 3), region_at((S) + 1), sbuf_at((S) + 1))
    int s = 0;
    for (; s + 3 < nsteps; s += 4) {
        BYHIP_STEP(0, s, o0, o1);
        BYHIP_STEP(1, s + 1, o1, o0);
        BYHIP_STEP(2, s + 2, o0, o1);
        BYHIP_STEP(3, s + 3, o1, o0);
    }
    if (s < nsteps) BYHIP_STEP(0, s, o0, o1);
    if (s + 1 < nsteps) BYHIP_STEP(1, s + 1, o1, o0);
    if (s + 2 < nsteps) BYHIP_STEP(2, s + 2, o0, o1);
#undef BYHIP_STEP
    // Every wave has read what its products need (the barrier of the last even step), and no load of this tile is left to land
    // on the next one's.
    wait_vmcnt<0>();
    if (more) {
        locate(u1, strip1, rows);
        load_scales(0, sbuf_at(0));
        load_pair(0, region_at(0));
        load_pair(2, region_at(2));
    }
    __builtin_amdgcn_sched_barrier(0);

    // Lane (c, g) holds row c of block j of x; register r is matrix row 8 (r / 4) + 4 g + r % 4 of block i.
    const int n0 = strip * (GLU ? kTileW / 2 : kTileW);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = 64 * wt + 32 * j + lc;
        const bool there = t < u.rows;
        const size_t row = there ? moe_y_row(a, u.first + t) : 0;
        constexpr int blocks = GLU ? 2 : 4;
#pragma unroll
        for (int i = 0; i < blocks; ++i) {
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
    u = u1;
    strip = strip1;
    }  // tiles
}

template <int XF, bool GLU, int YT>
void launch_tiles(const MoeArgs& a, const dim3& grid) {
    launch("moe_tiles", (moe_tiles<XF, GLU, YT>), grid, dim3(256), 0, a);
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

bool moe_tiles_take(const MoeArgs& a) { return a.unit_rows == kTileX && a.K % kStep == 0; }

void launch_moe_tiles(const MoeArgs& args, int x_format, bool glu, int max_units) {
    MoeArgs a = args;
    if (!moe_tiles_take(a)) fail("byhip: internal: units of %d rows, %d values", a.unit_rows, a.K);
    const int wide = glu ? kTileW / 2 : kTileW;
    a.strips = (a.N + wide - 1) / wide;
    const long long blocks = ((long long)max_units * a.strips + 7) / 8 * 8;
    if (blocks >= 1ll << 31) fail("byhip: a product of %d units of %d strips", max_units, a.strips);
    // One block per CU (its LDS holds one), each going through its XCD's tiles.
    const dim3 grid((unsigned)std::min<long long>(blocks, compute_units() / 8 * 8));
    if (x_format == BYHIP_MXFP4_KM) glu ? launch_tiles_y<BYHIP_MXFP4_KM, true>(a, grid) : launch_tiles_y<BYHIP_MXFP4_KM, false>(a, grid);
    else glu ? launch_tiles_y<BYHIP_MXFP8_KM, true>(a, grid) : launch_tiles_y<BYHIP_MXFP8_KM, false>(a, grid);
}

}  // namespace byhip
