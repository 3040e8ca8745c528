// byhip_attn_chunk.h - attention of many rows per sequence over a paged cache: prompts and their chunks (gfx950).
//
// A sequence's rows that share a key head (tokens x group) form tiles of 32 per wave, 128 or 256 per block. A block walks over
// tiles of 64 keys, which direct global-to-LDS loads bring in one tile ahead (one lookup of the page table per key and
// wave, two tiles ahead), K and V row by row as the cache holds them, 16-byte pieces permuted within a row against
// bank conflicts:
//   S^T = K Q^T    v_mfma_f32_32x32x16, K from LDS, Q in registers; a lane holds one row's scores of half the keys
//   O^T = V^T P^T  contracts over the keys in the order in which S^T left them in each lane, so weights never leave it;
//                  V^T is read with gfx950's transposing LDS loads (ds_read_b64_tr_b16: 16 lanes turn 4 keys x 16 values)
// Rows keep their statistics in their own lane, as O^T does its columns: a maximum is exchanged (between the two lanes of a
// row) and the sums scaled down only when a score passes the row's reference by 2^8.
//
// The work is divided as in attn_rows: all (head, sequence, row tile) items laid end to end in tiles of 64 keys, every
// block an equal run of them, one block per CU; parts of items that a boundary cuts go to the workspace and attn_join adds them. Runs
// are head-major and dealt to the 8 XCDs in order, so that blocks on one XCD read the same head's keys through its L2.
//
// fp32 queries or outputs: two fp16 or three bf16 terms of queries and weights, a matrix instruction each, in blocks of 4
// waves with twice the registers.
#pragma once

#include <algorithm>

#include "byhip_attn.h"

namespace byhip {
namespace {

constexpr int kChunkKeys = 64;
constexpr int kXcds = 8;
__device__ __attribute__((aligned(64))) uint32_t zero_piece[16];  // what keys and values outside the cache read as

typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef float f8v __attribute__((ext_vector_type(8)));

// Workgroup barrier once this wave's direct loads have landed and its LDS reads are done.
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int CT, int NP, int DIM, int WAVES, bool EXTRA>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void attn_chunk(AttnArgs a) {
    typedef typename Half8<CT>::vec vec;
    constexpr int R = 32 * WAVES, T = kChunkKeys, NT = 64 * WAVES;
    constexpr int STEPS = DIM / 16, DT = DIM / 32, PIECES = DIM / 8, SW = (PIECES < 16 ? PIECES : 16) - 1;
    constexpr int ROW = DIM * 2, TILE = T * ROW;                  // bytes of a key, of a tile
    constexpr int NI = TILE / 1024 / WAVES, RPI = 1024 / ROW;     // direct loads per wave and tile, keys per load
    constexpr float kShift = CT == BYHIP_F16 ? 7.0f : 0.0f;       // log2 of the weights' factor
    constexpr float kRaise = 8.0f;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];  // K, V of one tile, then of the next
    __shared__ int row_tiles[kAttnBatch + 1];                         // row tiles of the sequences before each
    __shared__ long long units_before[NT + 1];                        // key tiles of the row tiles before each thread's run
    __shared__ long long wave_total[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, hf = lane >> 5;

    const auto positions = [&](const SeqInfo& s, int rt, int& p0, int& p1) {
        p0 = s.first_pos + rt * R / a.group;
        p1 = s.first_pos + (min(s.rows, (rt + 1) * R) - 1) / a.group;
    };
    const auto scan = [&](long long v) {  // exclusive over the block
        long long x = v;
        for (int o = 1; o < 64; o <<= 1) {
            const long long u = __shfl_up(x, o, 64);
            if (lane >= o) x += u;
        }
        if (lane == 63) wave_total[wave] = x;
        __syncthreads();
        long long base = x - v;
        for (int w = 0; w < wave; ++w) base += wave_total[w];
        __syncthreads();
        return base;
    };
    // 1. row tiles before each sequence, then key tiles before each thread's run of row tiles
    {
        const int per = (a.s.batch + NT - 1) / NT, b0 = min(tid * per, a.s.batch), b1 = min(b0 + per, a.s.batch);
        int sum = 0;
        for (int b = b0; b < b1; ++b) {
            row_tiles[b] = sum;
            sum += (seq_info(a, b).rows + R - 1) / R;
        }
        const int base = (int)scan(sum);
        for (int b = b0; b < b1; ++b) row_tiles[b] += base;
        if (tid == NT - 1) row_tiles[a.s.batch] = base + sum;
        __syncthreads();
    }
    const int all_row_tiles = row_tiles[a.s.batch];
    const int run = (all_row_tiles + NT - 1) / NT;
    const auto sequence_of = [&](int x) {  // the last one with row tiles before it <= x
        int lo = 0, hi = a.s.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (row_tiles[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    const auto tiles_at = [&](int x, int& b) {
        b = sequence_of(x);
        const SeqInfo s = seq_info(a, b);
        int p0, p1;
        positions(s, x - row_tiles[b], p0, p1);
        return TileRange<T>(a, s, p0, p1).tiles;
    };
    {
        long long sum = 0;
        int b;
        for (int x = tid * run; x < min((tid + 1) * run, all_row_tiles); ++x) sum += tiles_at(x, b);
        const long long base = scan(sum);
        units_before[tid] = base;
        if (tid == NT - 1) units_before[NT] = base + sum;
        __syncthreads();
    }
    const long long per_head = units_before[NT], total = per_head * a.c.kv_heads;
    const long long blocks = min((long long)gridDim.x, total);
    int w = blockIdx.x;
    if (blocks == (long long)gridDim.x && gridDim.x % kXcds == 0) w = (w % kXcds) * (gridDim.x / kXcds) + w / kXcds;
    if (w >= blocks) {
        if (tid == 0) a.joins[w] = make_int4(0, 0, 0, 0);
        return;
    }
    const long long u0 = total * w / blocks, u1 = total * (w + 1) / blocks;
    int4 join = make_int4(0, 0, 0, 0);

    // this lane's places in the LDS tiles
    int k_at[STEPS];  // pieces 2 st + hf of key c
#pragma unroll
    for (int st = 0; st < STEPS; ++st) k_at[st] = c * ROW + (((2 * st + hf) ^ (c & SW)) << 4);
    int v_at[DT][2];  // keys 8 j + 4 hf + (lane % 16) / 4, values 32 dt + 16 (lane / 16 % 2) + 4 (lane % 4)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int key = 8 * j + 4 * hf + (lane & 15) / 4, piece = 4 * dt + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
            v_at[dt][j] = key * ROW + ((piece ^ (key & SW)) << 4) + 8 * (lane & 1);
        }
    // and its share of the direct loads: key (wave NI + i) RPI + lane / PIECES, the piece that belongs at lane % PIECES
    const int load_key = wave * NI * RPI + lane / PIECES;
    lds_byte* const lds3 = (lds_byte*)lds;

    for (long long u = u0; u < u1;) {
        const int h = __builtin_amdgcn_readfirstlane((int)(u / per_head));
        long long in_head = u - h * per_head;
        int lo = 0, hi = NT - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (units_before[mid] <= in_head) lo = mid;
            else hi = mid - 1;
        }
        in_head -= units_before[lo];
        int x = lo * run, b, n_tiles = tiles_at(x, b);
        while (in_head >= n_tiles) {
            in_head -= n_tiles;
            n_tiles = tiles_at(++x, b);
        }
        x = __builtin_amdgcn_readfirstlane(x);
        b = __builtin_amdgcn_readfirstlane(b);
        const int rt = x - row_tiles[b], t0 = __builtin_amdgcn_readfirstlane((int)in_head);
        const SeqInfo s = seq_info(a, b);
        int p0, p1;
        positions(s, rt, p0, p1);
        const TileRange<T> range(a, s, p0, p1);
        const int t1 = __builtin_amdgcn_readfirstlane((int)min((long long)range.tiles, t0 + (u1 - u)));

        // 2. the wave's rows
        const int row0 = rt * R + wave * 32, row = row0 + c;
        const bool valid = row < s.rows;
        const int token = valid ? row / a.group : 0, hq = h * a.group + (valid ? row % a.group : 0);
        const int pos = s.first_pos + token;
        const int wp0 = s.first_pos + min(row0, s.rows - 1) / a.group, wp1 = s.first_pos + min(row0 + 31, s.rows - 1) / a.group;
        const float slope = EXTRA && a.slopes ? a.slopes[hq] * kLog2e : 0.0f;
        vec q[NP][STEPS];
        float factor;
        {
            const size_t base = (size_t)(a.s.starts[b] + token) * a.q_stride + (size_t)hq * a.c.dim;
            int shift = 0;
            if (NP > 1 && a.q_dtype == BYHIP_F32) {
                float top = 0.0f;
                const float* p = static_cast<const float*>(a.q) + base;
                if constexpr (CT == BYHIP_F16) {  // the row's largest value to [2^14, 2^15)
                    for (int d = 8 * hf; d < a.c.dim; d += 16)
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(p[d + e]));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    shift = fp16_range_shift(top);
                }
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const int d = 16 * st + 8 * hf;
                    const bool in = valid && d < a.c.dim;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        typename Half8<CT>::one t[NP];
                        split_terms<CT, NP>(in ? ldexpf(p[in ? d + e : 0], shift) : 0.0f, t);
#pragma unroll
                        for (int i = 0; i < NP; ++i) q[i][st][e] = t[i];
                    }
                }
            } else {
                const uint16_t* p = static_cast<const uint16_t*>(a.q) + base;
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const int d = 16 * st + 8 * hf;
                    const bool in = valid && d < a.c.dim;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (in) {
                        if (a.q_vec) {
                            v = *reinterpret_cast<const uint4*>(p + d);
                        } else {
                            v.x = p[d] | (uint32_t)p[d + 1] << 16; v.y = p[d + 2] | (uint32_t)p[d + 3] << 16;
                            v.z = p[d + 4] | (uint32_t)p[d + 5] << 16; v.w = p[d + 6] | (uint32_t)p[d + 7] << 16;
                        }
                    }
                    q[0][st] = __builtin_bit_cast(vec, v);
#pragma unroll
                    for (int i = 1; i < NP; ++i) q[i][st] = __builtin_bit_cast(vec, make_uint4(0, 0, 0, 0));
                }
            }
            factor = ldexpf(EXTRA ? a.scale : a.scale * kLog2e, -shift);
        }
        float m = -INFINITY, l = 0.0f;
        f16v o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;

        // 3. key tiles
        const auto page_of = [&](int t) {  // the page of key `lane` of tile t
            const int j = range.key(t) + lane, at = max(0, min(j, s.len - 1));
            return a.s.table[(size_t)b * a.s.stride + at / a.c.page_size];
        };
        const auto load = [&](int t, int page, int buf, uint64_t& there) {
            const int j = range.key(t) + lane, at = max(0, min(j, s.len - 1));
            const bool is = (j < s.len) & (page >= 0) & (page < a.c.pages);
            there = __ballot(is);
            const uint32_t key_row = is ? ((uint32_t)page * a.c.kv_heads + h) * a.c.page_size + at % a.c.page_size : ~0u;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int key = load_key + i * RPI;
                const uint32_t from = (uint32_t)__shfl((int)key_row, key, 64);
                const int piece = (lane % PIECES) ^ (key & SW);
                const bool in = (from != ~0u) & (8 * piece < a.c.dim);
                const size_t off = (size_t)from * a.c.dim + 8 * piece;
                const uint16_t* zero = reinterpret_cast<const uint16_t*>(zero_piece);
                const uint16_t* kp = in ? a.c.k + off : zero;
                const uint16_t* vp = in ? a.c.v + off : zero;
                lds_byte* dst = lds3 + buf * 2 * TILE + (wave * NI + i) * 1024;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)kp, (lds_void*)dst, 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vp, (lds_void*)(dst + TILE), 16, 0, 0);
            }
        };
        uint64_t there = 0, next_there = 0;
        int page = page_of(t0);
        tile_barrier();  // the item before may still be reading its last tile
        load(t0, page, 0, there);
        if (t0 + 1 < t1) page = page_of(t0 + 1);
        for (int t = t0; t < t1; ++t) {
            const int buf = (t - t0) & 1, j0 = range.key(t);
            tile_barrier();
            if (t + 1 < t1) load(t + 1, page, buf ^ 1, next_there);
            if (t + 2 < t1) page = page_of(t + 2);
            const uint8_t* kt = lds + buf * 2 * TILE;
            const uint8_t* vt = kt + TILE;
            const auto full = [&](int lo_pos, int hi_pos) {
                return there == ~0ull && ((j0 + T - 1 <= lo_pos && (a.window <= 0 || hi_pos - j0 < a.window)) || j0 + T <= s.prefix);
            };
            // values that are not finite and that a row does not see (or that meet weights of several terms) are added apart
            constexpr uint32_t kExp = CT == BYHIP_F16 ? 0x7C00u : 0x7F80u;
            bool odd = false;
            if (NP > 1 || !full(p0, p1)) {
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < TILE / 16 / NT; ++i) {
                    const uint4 v = *reinterpret_cast<const uint4*>(vt + (i * NT + tid) * 16);
                    for (const uint32_t x : {v.x, v.y, v.z, v.w}) any |= (uint32_t)((x & kExp) == kExp) | (uint32_t)((x >> 16 & kExp) == kExp);
                }
                odd = __syncthreads_or(any != 0);
            }
            const bool works = row0 < s.rows && (j0 <= wp1 || j0 < s.prefix);  // some row of the wave may see the tile
            f16v sc[2];
            if (works) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[kb][e] = 0.0f;
#pragma unroll
                    for (int st = 0; st < STEPS; ++st) {
                        const vec k = *reinterpret_cast<const vec*>(kt + k_at[st] + kb * 32 * ROW);
#pragma unroll
                        for (int i = NP - 1; i >= 0; --i) sc[kb] = mfma32(k, q[i][st], sc[kb]);
                    }
                }
                if constexpr (EXTRA) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float v = sc[kb][e] * factor;
                            if (a.softcap > 0.0f) v = a.softcap * soft_tanh<(NP > 1)>(v / a.softcap);
                            sc[kb][e] = v * kLog2e - slope * fabsf((float)(pos - (j0 + 32 * kb + 8 * (e / 4) + 4 * hf + e % 4)));
                        }
                }
                uint32_t see[2] = {~0u, ~0u};
                if (!full(wp0, wp1)) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        see[kb] = seen_keys(a, s, pos, j0 + 32 * kb, (uint32_t)(there >> (32 * kb)));
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[kb][e] = see[kb] >> (8 * (e / 4) + e % 4) >> (4 * hf) & 1u ? sc[kb][e] : -INFINITY;
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; e += 2) top = fmaxf(top, fmaxf(sc[kb][e], sc[kb][e + 1]));
                if (!EXTRA) top *= factor;
                if (__ballot(top > m + kRaise || (m == -INFINITY && top > m))) {
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float raised = fmaxf(m, top);
                    const float fade = raised == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
                    m = raised;
                    l *= fade;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[dt][e] *= fade;
                }
                if (odd) {
                    for (int key = 0; key < T; ++key) {
                        const uint32_t mine = (key < 32 ? see[0] >> key : see[1] >> (key - 32)) & 1u;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int g = 0; g < 4; ++g) {  // dimensions 32 dt + 8 g + 4 hf .. + 3
                                const int piece = (4 * dt + g) ^ (key & SW);
                                const uint2 v = *reinterpret_cast<const uint2*>(vt + key * ROW + piece * 16 + 8 * hf);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t bits = (e < 2 ? v.x : v.y) >> (16 * (e & 1)) & 0xFFFFu;
                                    const float val = CT == BYHIP_F16 ? (float)bits_h((uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
                                    o[dt][4 * g + e] += mine & (uint32_t)((bits & kExp) == kExp) ? val : 0.0f;
                                }
                            }
                    }
                }
                // weights, packed into the operands of the products with V
                const float base = m == -INFINITY ? 0.0f : m - kShift;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sc[kb][e] = __builtin_amdgcn_exp2f(EXTRA ? sc[kb][e] - base : fmaf(sc[kb][e], factor, -base));
                        l += sc[kb][e];
                    }
            }
            if (odd) {  // every wave has added what it sees of them: the tile's odd values become 0
                tile_barrier();
#pragma unroll
                for (int i = 0; i < TILE / 16 / NT; ++i) {
                    uint32_t* v = reinterpret_cast<uint32_t*>(lds + buf * 2 * TILE + TILE + (i * NT + tid) * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t x = v[e];
                        x &= (x & kExp) == kExp ? 0xFFFF0000u : ~0u;
                        x &= (x >> 16 & kExp) == kExp ? 0xFFFFu : ~0u;
                        v[e] = x;
                    }
                }
                tile_barrier();
            }
            if (works) {
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    vec wt[NP];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        typename Half8<CT>::one t[NP];
                        split_terms<CT, NP>(sc[st / 2][8 * (st & 1) + i], t);
#pragma unroll
                        for (int n = 0; n < NP; ++n) wt[n][i] = t[n];
                    }
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds3 + (buf * 2 + 1) * TILE + v_at[dt][0] + st * 16 * ROW));
                        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds3 + (buf * 2 + 1) * TILE + v_at[dt][1] + st * 16 * ROW));
                        const vec v = __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) o[dt] = mfma32(v, wt[n], o[dt]);
                    }
                }
            }
            there = next_there;
        }

        // 4. the wave's rows leave, whole or as a part
        const bool begins = t0 == 0, ends = t1 == range.tiles;
        l += __shfl_xor(l, 32, 64);
        if (begins && ends) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (valid) {
                const size_t out = (size_t)(a.s.starts[b] + token) * a.out_stride + (size_t)hq * a.c.dim;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int d = 32 * dt + 8 * g + 4 * hf;
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = l == 0.0f ? 0.0f : o[dt][4 * g + e] * inv;
                        if (d < a.c.dim) {
                            if (a.out_vec) {
                                store_vec<4>(a.out, out + d, x, a.out_dtype);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float one[1] = {x[e]};
                                    store_vec<1>(a.out, out + d + e, one, a.out_dtype);
                                }
                            }
                        }
                    }
            }
        } else {
            float* slot = part_slot<R, DIM>(a.part, begins ? 2 * w + 1 : 2 * w);
            const int r = wave * 32 + c;
            if (hf == 0) {
                slot[R * DIM + r] = m;
                slot[R * DIM + R + r] = l;
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f4*>(slot + r * DIM + 32 * dt + 8 * g + 4 * hf) =
                        (f4){o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
        }
        if (begins && !ends) join = join_of(u - t0 + range.tiles - 1, blocks, total, b, rt, h);
        u += t1 - t0;
    }
    if (tid == 0) a.joins[w] = join;
}

template <int CT, int NP, int DIM, int WAVES>
void launch_chunk(const AttnArgs& a) {
    constexpr size_t kSlots = (size_t)2 * 32 * WAVES * (DIM + 2) * sizeof(float);  // one block's
    const size_t room = (kAttnWorkspaceBytes - kAttnJoinBytes) / kSlots;
    const unsigned blocks = (unsigned)std::min<size_t>(room, compute_units());
    if (a.softcap > 0.0f || a.slopes || !(a.scale > 0.0f)) launch("attn_chunk", (attn_chunk<CT, NP, DIM, WAVES, true>), dim3(blocks), dim3(64 * WAVES), 0, a);
    else launch("attn_chunk", (attn_chunk<CT, NP, DIM, WAVES, false>), dim3(blocks), dim3(64 * WAVES), 0, a);
    BYHIP_LAUNCHED("attn_chunk");
    launch("attn_join", (attn_join<32 * WAVES, DIM>), dim3(blocks, 64), dim3(256), 0, a);
    BYHIP_LAUNCHED("attn_join");
}

// Blocks of 8 waves where two waves per SIMD have the registers they need, else of 4.
template <int CT, int NP>
void launch_chunk_dim(const AttnArgs& a) {
    if (a.c.dim <= 64) launch_chunk<CT, NP, 64, NP == 1 ? 8 : 4>(a);
    else if (a.c.dim <= 128) launch_chunk<CT, NP, 128, NP == 1 ? 8 : 4>(a);
    else launch_chunk<CT, NP, 256, 4>(a);
}

}  // namespace
}  // namespace byhip
