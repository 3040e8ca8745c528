// byhip_moe_rows.hip - few rows per expert (gfx950): products that read each matrix once, in units of up to 64 rows.
//
// Bound by the matrices' bytes. A block takes a strip of a matrix (64 of its rows) and one unit's rows; its four waves share
// out the values' axis in windows of 512 (or 256) and add their sums in LDS at the end. A wave loads its window of the
// strip in 16-byte pieces straight into the operands of v_mfma_scale_f32_16x16x128_f8f6f4, 16 KB in flight before the first
// product, and the rows' values beside it (they come from L2: every strip of the expert reads them). Three waves per SIMD (six or seven with strips of 16) hide the latencies; loads
// of the first window ahead of the rows' look-up, with the registers they take, cost more than they saved (48 us for 33, 48 tokens, 128 experts).
//
// Operands (checked on the device): the matrix is the first, in 4 bits: lane (c, g) = (l % 16, l / 16) holds the 32 values of
// block g of row c. Rows in 4 bits are the same. Rows in 8 bits: lane (c, g) holds two pieces of 16 values, those of
// half g % 2 of blocks g / 2 and 2 + g / 2; scales go by block for both, lane (c, g)'s being block g's. Which 32 values of the
// window are block g of a step is free as long as both operands agree: step s takes groups 4 s .. 4 s + 3 of the window's 4 S, so
// that four lanes read 64 neighbouring bytes of a row (with group S g + s, 16 bytes of each 64 at a time: 37 us, 48 tokens, 128 experts, 2048 to 768, for 31). The result: lane (c, g) holds row c of x, matrix rows 4 g .. 4 g + 3.
//
// Sums are fp32. What the instructions add in one go is exact with rows in 4 bits; with rows in 8 bits they cut small products off, so those rows go in two
// parts (split_bytes), twice the products. With outputs of 16 bits or fewer one part would do for most rows (5e-6 to 1e-5 of a product's norm is cut off then), but not for
// rows whose large terms cancel, and it saves little here (us, two parts for one: 48 tokens, 128 experts, 2048 to 768 31.4 for 29.4, 800 to 2048 with 400 tokens
// 46 for 37; 1 / 16 / 64 rows of 4096 x 4096 5.1 / 5.8 / 10.8 for 4.8 / 5.5 / 9.9).
#include "byhip_moe.h"

namespace byhip {
namespace {

constexpr int kWaves = 4;

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v4u load16(rsrc_t r, uint32_t off) { return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); }

// The scale bytes of groups G + 4 s + g, s = 0 .. S - 1, of a row that starts at `row` (kOutOfRange: none). WORDS: rows start at whole words, and all lanes'
// bytes of the window come in one load; else a byte at a time. (No branch between loads: the compiler waits there for those under way.)
template <int S>
struct Scales {
    uint32_t word[S];
};
template <int S, bool WORDS>
__device__ __forceinline__ Scales<S> load_scales(rsrc_t r, uint32_t row, int G, int g, int KG) {
    Scales<S> v;
    if constexpr (WORDS) {
        const uint32_t at = row == kOutOfRange ? kOutOfRange : row + G;
        if constexpr (S == 4) {
            const v4u w = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
#pragma unroll
            for (int s = 0; s < S; ++s) v.word[s] = w[s];
        } else {
            const v2u w = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
#pragma unroll
            for (int s = 0; s < S; ++s) v.word[s] = w[s];
        }
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
            v.word[s] = __builtin_amdgcn_raw_buffer_load_b8(r, row == kOutOfRange || G + 4 * s + g >= KG ? kOutOfRange : row + G + 4 * s + g, 0, 0);
    }
    return v;
}
// Byte s: the s-th scale; 0 past the row's KG groups (a byte of the next row might be a NaN's).
template <int S, bool WORDS>
__device__ __forceinline__ uint32_t pick_scales(const Scales<S>& v, int G, int g, int KG) {
    const uint32_t byte = WORDS ? g : 0;
    auto from = [&](int s) { return G + 4 * s < KG ? byte + 4 * (s & 1) : 0x0Cu; };
    uint32_t p = __builtin_amdgcn_perm(v.word[1], v.word[0], 0x0C0C0000u | from(1) << 8 | from(0));
    if constexpr (S == 4) p |= __builtin_amdgcn_perm(v.word[3], v.word[2], 0x0C0Cu | from(3) << 24 | from(2) << 16);
    return p;
}

template <int XF, int B>  // B: the scales' byte
__device__ __forceinline__ f4v product(v8i w, v8i x, f4v c, int sw, int sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, XF == BYHIP_MXFP8_KM ? 0 : 4, B, sw, B, sx);
}

// MT blocks of 16 rows, NF blocks of 16 matrix rows (GLU: two of gates, two of ups), windows of S steps.
template <int XF, int MT, int NF, int S, bool WORDS, bool GLU>
__global__ __launch_bounds__(64 * kWaves) void moe_rows(MoeArgs a) {
    static_assert(!GLU || NF == 4, "gates and ups");
    __shared__ float4 part[kWaves][NF * MT][64];
    MoeUnit u;
    int strip;
    if (!MoeTiles(a).find(a, blockIdx.x >> 3, u, strip) || u.rows == 0) return;
    constexpr bool eight = XF == BYHIP_MXFP8_KM;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const uint32_t kb = (uint32_t)a.K / 2, xb = eight ? (uint32_t)a.K : kb;
    const rsrc_t wr = make_rsrc(a.w + (size_t)u.expert * a.R * kb, (uint32_t)a.R * kb);
    const rsrc_t wsr = make_rsrc(a.ws + (size_t)u.expert * a.R * a.KG, (uint32_t)a.R * a.KG);
    const rsrc_t xr = make_rsrc(a.x, a.x_bytes), xsr = make_rsrc(a.xs, a.xs_bytes);
    const int n0 = strip * (GLU ? 32 : 16 * NF);
    int n[NF];  // this lane's row of each block of the matrix
#pragma unroll
    for (int f = 0; f < NF; ++f) n[f] = GLU ? (f >> 1) * a.N + n0 + 16 * (f & 1) + c : n0 + 16 * f + c;
    const int windows = (a.KG + 4 * S - 1) / (4 * S);

    uint32_t x_at[MT], xs_at[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int i = 16 * m + c;
        const int row = i < u.rows ? moe_x_row(a, u.first + i) : -1;
        x_at[m] = row < 0 ? kOutOfRange : (uint32_t)row * xb;
        xs_at[m] = row < 0 ? kOutOfRange : (uint32_t)row * a.KG;
    }
    f4v acc[NF][MT];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            acc[f][m] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            // A product whose addend is the constant 0 may be given a result that overlaps its operands, which it then misreads:
            // the zeros stay in registers.
            asm volatile("" : "+v"(acc[f][m]));
        }
    for (int W = w; W < windows; W += kWaves) {
        const int G = 4 * S * W;  // the window's first group
        v4u wv[NF][S];
        Scales<S> wsv[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                wv[f][s] = load16(wr, n[f] < a.R && G + 4 * s + g < a.KG ? (uint32_t)n[f] * kb + 16 * (G + 4 * s + g) : kOutOfRange);
            wsv[f] = load_scales<S, WORDS>(wsr, n[f] < a.R ? (uint32_t)n[f] * a.KG : kOutOfRange, G, g, a.KG);
        }
        Scales<S> xsv[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xsv[m] = load_scales<S, WORDS>(xsr, xs_at[m], G, g, a.KG);
        // The rows' values go one step ahead of the products where a window has four (48 tokens, 128 experts, 2048 to 768: 31 us for 34; with
        // two, 768 to 2048: 23.0 for 22.5).
        constexpr bool ahead = S == 4;
        auto load_x = [&](int T, v8i (&x)[MT]) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                x[m] = v8i{0, 0, 0, 0, 0, 0, 0, 0};
                if constexpr (eight) {
                    const int g0 = G + 4 * T + (g >> 1), g1 = g0 + 2;
                    const v4u p = load16(xr, x_at[m] != kOutOfRange && g0 < a.KG ? x_at[m] + 32 * g0 + 16 * (g & 1) : kOutOfRange);
                    const v4u q = load16(xr, x_at[m] != kOutOfRange && g1 < a.KG ? x_at[m] + 32 * g1 + 16 * (g & 1) : kOutOfRange);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { x[m][e] = (int)p[e]; x[m][4 + e] = (int)q[e]; }
                } else {
                    const v4u p = load16(xr, x_at[m] != kOutOfRange && G + 4 * T + g < a.KG ? x_at[m] + 16 * (G + 4 * T + g) : kOutOfRange);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[m][e] = (int)p[e];
                }
            }
        };
        v8i xv[2][MT];
        if constexpr (ahead) load_x(0, xv[0]);
        uint32_t ws[NF], xs[MT];
        auto step = [&](auto Sc) {
            constexpr int T = decltype(Sc)::value;
            if constexpr (!ahead) load_x(T, xv[T & 1]);
            else if constexpr (T + 1 < S) load_x(T + 1, xv[(T + 1) & 1]);
            if constexpr (T == 0) {
                if constexpr (ahead) __builtin_amdgcn_sched_barrier(0);  // the loads are out
#pragma unroll
                for (int f = 0; f < NF; ++f) ws[f] = pick_scales<S, WORDS>(wsv[f], G, g, a.KG);
#pragma unroll
                for (int m = 0; m < MT; ++m) xs[m] = pick_scales<S, WORDS>(xsv[m], G, g, a.KG);
            }
            v8i large[MT], small[eight ? MT : 1];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (eight) split_bytes(xv[T & 1][m], large[m], small[m]);
                else large[m] = xv[T & 1][m];
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const v8i wf = {(int)wv[f][T][0], (int)wv[f][T][1], (int)wv[f][T][2], (int)wv[f][T][3], 0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (eight) acc[f][m] = product<XF, T>(wf, small[m], acc[f][m], (int)ws[f], (int)xs[m]);
                    acc[f][m] = product<XF, T>(wf, large[m], acc[f][m], (int)ws[f], (int)xs[m]);
                }
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        if constexpr (S > 2) {
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) part[w][f * MT + m][lane] = make_float4(acc[f][m][0], acc[f][m][1], acc[f][m][2], acc[f][m][3]);
    __syncthreads();
    auto whole = [&](int f, int m, float (&v)[4]) {
        v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float4 p = part[i][f * MT + m][lane];
            v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
        }
    };
    if constexpr (GLU) {
        for (int m = w; m < MT; m += kWaves) {
            const int i = 16 * m + c;
            float gate[4], up[4], h[2][4];
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                whole(f, m, gate);
                whole(2 + f, m, up);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[f][e] = swiglu(gate[e], up[e]);
            }
            const bool there = i < u.rows;
            const size_t row = there ? moe_y_row(a, u.first + i) : 0;
            if (is_mx_out(a.y_dtype)) {
                uint32_t mag = mag8(h[0], h[1]);
                mag = max(mag, (uint32_t)__shfl_xor((int)mag, 16));
                mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
                if (there) store_group(a, row, strip, 4 * g, g == 0, mag, h[0], h[1]);
            } else if (there) {
                moe_store4(a, row, n0 + 4 * g, h[0]);
                moe_store4(a, row, n0 + 16 + 4 * g, h[1]);
            }
        }
    } else if (NF > 1 && is_mx_out(a.y_dtype)) {
        for (int p = w; p < MT * (NF / 2); p += kWaves) {
            const int m = p / (NF > 1 ? NF / 2 : 1), q = p % (NF > 1 ? NF / 2 : 1), i = 16 * m + c;
            float h[2][4];
            whole(2 * q, m, h[0]);
            whole(NF > 1 ? 2 * q + 1 : 0, m, h[1]);
            uint32_t mag = mag8(h[0], h[1]);
            mag = max(mag, (uint32_t)__shfl_xor((int)mag, 16));
            mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
            if (i < u.rows && n0 + 32 * q < a.N) store_group(a, moe_y_row(a, u.first + i), n0 / 32 + q, 4 * g, g == 0, mag, h[0], h[1]);
        }
    } else {
        for (int p = w; p < MT * NF; p += kWaves) {
            const int m = p / NF, f = p % NF, i = 16 * m + c;
            float v[4];
            whole(f, m, v);
            if (i < u.rows) moe_store4(a, moe_y_row(a, u.first + i), n0 + 16 * f + 4 * g, v);
        }
    }
}

template <int XF, int MT, int NF, bool GLU>
void launch_rows_as(MoeArgs a, int max_units) {
    const int wide = GLU ? 32 : 16 * NF;
    a.strips = (a.N + wide - 1) / wide;
    const long long blocks = ((long long)max_units * a.strips + 7) / 8 * 8;
    if (blocks >= 1ll << 31) fail("byhip: a product of %d units of %d strips", max_units, a.strips);
    // Windows of 512 values, or of 256 where those would leave waves without one or with half of one (us, 512 / 256: 48 tokens, 128 experts, 2048 outputs, K = 768 / 1024 / 1408 / 1536 /
    // 2048 / 4096 22.2 / 24.6 / 27.1 / 31.1 / 43.0 / 79.4 for 19.0 / 21.5 / 29.0 / 32.1 / 44.6 / 95.6; one token, K = 1024 / 1536 / 2048 5.1 / 5.6 / 6.9 for 4.7 / 5.7 / 7.2; 256 rows of one
    // matrix, K = 1024 / 2048 8.6 / 11.7 for 7.7 / 12.7).
    const dim3 grid((unsigned)blocks), block(64 * kWaves);
    if (a.KG & 3) launch("moe_rows", (moe_rows<XF, MT, NF, 2, false, GLU>), grid, block, 0, a);
    else if (a.KG > 40) launch("moe_rows", (moe_rows<XF, MT, NF, 4, true, GLU>), grid, block, 0, a);
    else launch("moe_rows", (moe_rows<XF, MT, NF, 2, true, GLU>), grid, block, 0, a);
    BYHIP_LAUNCHED("moe_rows");
}

// Strips of 64, 32 or 16 outputs: the widest that gives half of the CUs a block, for rows are read once per strip (us, K = 4096, strips
// of 64 / 32 / 16: 16 rows, N = 4096 9.5 / 7.0 / 5.7, N = 4608 - / 7.3 / 8.8, N = 8192 10.3 / 8.3 / 9.4, N = 9216 10.4 / 11.7 / -, N = 14336 11.0 / 12.1 / 15.4; 32 rows, N =
// 4608 - / 9.7 / 12.9, N = 9216 13.4 / 16.2 / -; one row, N = 4608 - / 6.6 / 6.2). Gates and ups have 32 each. Eight waves per block took as long where
// one unit's strips are all there is (9.8 us for 10.5 at N = 14336, 9.6 for 9.7), longer elsewhere (33 us for 41, 48 tokens, 128 experts).
template <int XF, int MT, bool GLU>
void launch_rows_n(const MoeArgs& a, int max_units) {
    if constexpr (!GLU) {
        const long long strips = (a.N + 15) / 16, room = 130;
        if (strips / 4 * max_units < room) {
            if (strips / 2 * max_units < room && !is_mx(a.y_dtype)) launch_rows_as<XF, MT, 1, GLU>(a, max_units);
            else launch_rows_as<XF, MT, 2, GLU>(a, max_units);
            return;
        }
    }
    launch_rows_as<XF, MT, 4, GLU>(a, max_units);
}

template <int XF, bool GLU>
void launch_rows(const MoeArgs& a, int max_units) {
    // A block takes all of its unit's rows at once.
    if (a.unit_rows > 64) fail("byhip: internal: units of %d rows", a.unit_rows);
    if (a.unit_rows <= 16) launch_rows_n<XF, 1, GLU>(a, max_units);
    else if (a.unit_rows <= 32) launch_rows_n<XF, 2, GLU>(a, max_units);
    else launch_rows_n<XF, 4, GLU>(a, max_units);
}

}  // namespace

void launch_moe_rows(const MoeArgs& a, int x_format, bool glu, int max_units) {
    if (x_format == BYHIP_MXFP4_KM) glu ? launch_rows<BYHIP_MXFP4_KM, true>(a, max_units) : launch_rows<BYHIP_MXFP4_KM, false>(a, max_units);
    else glu ? launch_rows<BYHIP_MXFP8_KM, true>(a, max_units) : launch_rows<BYHIP_MXFP8_KM, false>(a, max_units);
}

}  // namespace byhip
