// byhip_attn_chunk.h - attention of many rows per sequence over a paged cache: prompts and their chunks (gfx950).
//
// A sequence's rows that share a key head (tokens x group) form tiles of 32 per wave, 128 or 256 per block. A block walks over
// tiles of 64 keys, which direct global-to-LDS loads bring in one or two tiles ahead (pages are looked up the same way, further
// ahead), K and V row by row as the cache holds them, 16-byte pieces turned within a row against bank conflicts:
//   S^T = K Q^T    v_mfma_f32_32x32x16, K from LDS, Q in registers; a lane holds one row's scores of half the keys
//   O^T = V^T P^T  contracts over the keys in the order in which S^T left them in each lane, so weights never leave it;
//                  V^T is read with gfx950's transposing LDS loads (ds_read_b64_tr_b16: 16 lanes turn 4 keys x 16 values)
// Rows keep their statistics in their own lane, as O^T does its columns. No maximum is searched for: weights are taken against the
// row's reference, their sum bounds the largest, and only where it passes a limit is the reference raised (a maximum
// exchanged between the two lanes of a row) and the sums scaled down.
//
// The work is divided as in attn_rows: all (head, sequence, row tile) items laid end to end in tiles of 64 keys, every
// block an equal run of them, one block per CU; parts of items that a boundary cuts go to the workspace and attn_join adds them.
// Where whole items leave the fullest block no more to do, none is cut. Runs are head-major and dealt to the 8 XCDs in
// order, so that blocks on one XCD read the same head's keys through its L2.
//
// What bounds it: the two phases of a tile, products and exponentials, which two waves per SIMD run in turn. 4096 rows x 16384
// keys, 32 heads of 128 values, bf16: 0.94 to 1.05 ms by the clock of the card, 920 to 1020 TFLOP/s, matrix instructions busy 47 to 49% of the cycles. With 64 values the
// exponentials outweigh the products (4 x 700 rows x 4000 keys, 24 heads: 117 us, 538 TFLOP/s; capped 169 us).
//
// fp32 queries or outputs: two fp16 or three bf16 terms of queries and weights, a matrix instruction each, in blocks of 4
// waves with twice the registers (30 x 255 rows x 2048 keys, 8 heads of 128 values: 94 us in bf16, 224 in fp32 on a bf16 cache). With
// 16-bit rows on both sides a weight is rounded once to the cache's type, as in attn_rows.
//
// Registers: heads of up to 128 values keep all vectors but 2 to 8 (fp32 forms: all); of 129 to 256 values 71 to 78 go to memory, 300
// of fp32 on fp16, 652 to 684 of fp32 on bf16 (4 x 700 rows x 4000 keys, 24 heads of 256: 411 us, 826, 1768), and every
// form keeps 150 to 390 scalars in vector lanes.
#pragma once

#include <algorithm>

#include "byhip_attn.h"

namespace byhip {
namespace {

#define INLINE __attribute__((always_inline))
constexpr int kChunkKeys = 64;
constexpr int kXcds = 8;
// What cutting an item costs the blocks that share it, in key tiles: the part's way to the workspace and back. (30 prompts of 255 rows x
// 1024 keys of 64 values: 135 us, with 4 150; 18 steps beside 6 prompts in a window: 64 us, with 16 77. It is too little for one prompt
// of 1000 rows: 77 us, with 16 44.)
constexpr int kCutTiles = 8;
// Key tiles a block should at least get before another one takes part. (100 rows x 2000 keys: 50 us, with 2 55, with 8 55; 3 prompts
// in fp32 59 us, with 8 65. It is too little where one item goes to hundreds of blocks, whose parts then take the join longer:
// 64 rows x 30000 keys of one key head 170 us, with 16 84.)
constexpr int kShareTiles = 4;

typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// Workgroup barrier after this wave's LDS reads, and unless LATEST < 0 once all its direct loads but the LATEST last ones have
// landed (they land in order; loads of the compiler's own among the last only make it wait for more).
template <int LATEST>
__device__ __forceinline__ void phase_barrier() {
    if constexpr (LATEST >= 0) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATEST) : "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 16 bytes per lane from memory to LDS byte `to` + 16 lane. Written as assembly because the compiler makes every later LDS
// read wait for such loads, which here belong to tiles still ahead; it has no output register, phase_barrier waits for
// it, and a wait of the compiler's own that counts it among its loads only waits longer. m0 (the LDS address) is an operand, so that
// the compiler knows what it holds; the s_nop is the wait state between its write and the load.
__device__ __forceinline__ void load_to_lds(const void* p, uint32_t to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(to) : "memory");
}
// The same for 4 bytes per lane.
__device__ __forceinline__ void word_to_lds(const void* p, uint32_t to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "{m0}"(to) : "memory");
}

template <int I> struct Index { static constexpr int value = I; };
template <int I, int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
    if constexpr (I < N) {
        f(Index<I>{});
        unrolled<I + 1, N>(f);
    }
}

// DIM: values a row takes in LDS and in a part, at least the head's; USED of them are multiplied.
template <int CT, int NP, int DIM, int USED, int WAVES, bool EXTRA>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void attn_chunk(AttnArgs a) {
    typedef typename Half8<CT>::vec vec;
    constexpr int R = 32 * WAVES, T = kChunkKeys, NT = 64 * WAVES;
    constexpr int STEPS = USED / 16, DT = USED / 32, PIECES = DIM / 8, SW = (PIECES < 16 ? PIECES : 16) - 1;
    constexpr int ROW = DIM * 2, TILE = T * ROW;                  // bytes of a key, of a tile
    constexpr int NI = TILE / 1024 / WAVES, RPI = 1024 / ROW;     // direct loads per wave and tile, keys per load
    constexpr bool PAIRED = WAVES == 8;                           // two waves per SIMD, half a tile apart
    constexpr int AHEAD = PAIRED ? 2 : 1;                         // tiles between the loads of one and its use
    // Loads go out between the products where those take less time than the weights (64 values: 146 us from 158, 4 x 700
    // rows x 4000 keys), else with the weights (128 values: 1.02 ms, from 1.04 between the products).
    constexpr bool EARLY = DIM <= 64;
    constexpr int BUFS = AHEAD + (EARLY || PAIRED ? 2 : 1);
    constexpr int SLOTS = 4;                                      // page lookups on their way and in use
    constexpr int BATCH = 2 * NI + 1;                             // a wave's direct loads per tile
    constexpr float kShift = CT == BYHIP_F16 ? 4.0f : 0.0f;       // log2 of the weights' factor
    constexpr float kLimit = 32768.0f;                            // a lane's weights of a tile may add up to this
    constexpr uint32_t kExp = CT == BYHIP_F16 ? 0x7C00u : 0x7F80u;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * BUFS * TILE];  // BUFS tiles of K, then of V
    __shared__ __attribute__((aligned(256))) int looked_up[WAVES][SLOTS][64];  // each wave's pages of the keys of tiles ahead
    __shared__ int row_tiles[kAttnBatch + 1];                                // row tiles of the sequences before each
    __shared__ long long units_before[NT + 1];                               // key tiles of the row tiles before each thread's run
    __shared__ long long wave_total[WAVES];
    __shared__ int not_finite;                                               // the last pass whose sums were not
    __shared__ int longest;                                                  // key tiles of the largest item
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
    const int all_row_tiles = uniform(row_tiles[a.s.batch]);
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
        int b, top = 0;
        if (tid == 0) longest = not_finite = 0;
        for (int x = tid * run; x < min((tid + 1) * run, all_row_tiles); ++x) {
            const int n = tiles_at(x, b);
            sum += n;
            top = max(top, n);
        }
        const long long base = scan(sum);
        if (top) atomicMax(&longest, top);
        units_before[tid] = base;
        if (tid == NT - 1) units_before[NT] = base + sum;
        __syncthreads();
    }
    const long long per_head = uniform(units_before[NT]), total = per_head * a.c.kv_heads;
    const long long items = (long long)all_row_tiles * a.c.kv_heads;
    // Whole items where the fullest block then has no more than with equal shares and their cuts (8 heads of 64 values, 255 rows x
    // 1024 keys: 240 items whole 46 us, cut 61; 264 items 68 and 63; 4 x 2100 rows x 4000 keys, 288 items: 155 and 119).
    const bool whole = (items + gridDim.x - 1) / gridDim.x * uniform(longest) <= max((long long)kShareTiles, total / gridDim.x) + kCutTiles;
    const long long blocks = min((long long)gridDim.x, whole ? items : max(1LL, total / kShareTiles));
    int w = blockIdx.x;
    if (blocks == (long long)gridDim.x && gridDim.x % kXcds == 0) w = (w % kXcds) * (gridDim.x / kXcds) + w / kXcds;
    if (w >= blocks || total == 0) {
        if (tid == 0) a.joins[w] = make_int4(0, 0, 0, 0);
        return;
    }
    const long long u0 = whole ? w : total * w / blocks, u1 = whole ? items : total * (w + 1) / blocks;
    int4 join = make_int4(0, 0, 0, 0);
    int pass = 0;

    // A key's pieces are turned within its row in LDS, so that what one cycle reads, 256 bytes, lies on different banks: K's, of
    // which 16 lanes read a piece each of 16 keys, and V's, of which 32 lanes read 64 bytes each of 4 keys. K's piece i of key j
    // lies at i ^ k_turn(j), V's at i ^ v_turn(j); turns of keys whose bits do not overlap combine.
    const auto k_turn = [](int j) INLINE { return (PIECES >= 16 ? j : j >> 1) & SW; };
    const auto v_turn = [](int j) INLINE { return (PIECES >= 16 ? 4 * j : 2 * j) & SW; };
    // This lane's places: pieces 2 st + hf of key c at k_at ^ 32 st, and keys 4 hf + (lane % 16) / 4 (+ 8 j + 16 st), values
    // 32 dt + 16 (lane / 16 % 2) + 4 (lane % 4) at v_at ^ 64 dt.
    const int k_at = c * ROW + ((hf ^ k_turn(c)) << 4);
    const int v_key = 4 * hf + (lane & 15) / 4;
    const int v_at = v_key * ROW + (((2 * (lane >> 4 & 1) + (lane & 3) / 2) ^ v_turn(v_key)) << 4) + 8 * (lane & 1);
    // and its share of the direct loads: keys load_key + i RPI, whose bits do not overlap, the piece that belongs at lane % PIECES
    const int load_key = wave * NI * RPI + lane / PIECES;
    const int k_piece = (lane % PIECES) ^ k_turn(load_key), v_piece = (lane % PIECES) ^ v_turn(load_key);
    lds_byte* const lds3 = (lds_byte*)lds;
    const uint32_t pages_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_byte*)looked_up[wave][0]);
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds3);

    for (long long u = u0; u < u1;) {
        int h, b, rt, t0, t1;
        if (whole) {
            h = (int)(u / all_row_tiles);
            const int x = (int)(u % all_row_tiles);
            b = uniform(sequence_of(x));
            rt = x - uniform(row_tiles[b]);
            t0 = 0;
        } else {
            h = (int)(u / per_head);
            long long in_head = u - h * per_head;
            int lo = 0, hi = NT - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (units_before[mid] <= in_head) lo = mid;
                else hi = mid - 1;
            }
            in_head -= units_before[lo];
            int x = lo * run, n_tiles = tiles_at(x, b);
            while (in_head >= n_tiles) {
                in_head -= n_tiles;
                n_tiles = tiles_at(++x, b);
            }
            b = uniform(b);
            rt = uniform(x - row_tiles[b]);
            t0 = uniform((int)in_head);
        }
        const SeqInfo s = seq_info(a, b);
        int p0, p1;
        positions(s, rt, p0, p1);
        const TileRange<T> range(a, s, p0, p1);
        t1 = whole ? range.tiles : (int)min((long long)range.tiles, t0 + (u1 - u));

        const auto page_at = [&](int t) INLINE {  // the table's entry of key `lane` of tile t
            const int at = max(0, min(range.key(t) + lane, s.len - 1));
            return a.s.table + (size_t)b * a.s.stride + page_col(a, at);
        };
        int first_pages[AHEAD + 2];
#pragma unroll
        for (int i = 0; i < AHEAD + 2; ++i) first_pages[i] = *page_at(t0 + i);

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
                    shift = query_shift(top);
                }
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    const int d = 16 * st + 8 * hf;
                    const bool in = valid && d < a.c.dim;
                    float f[8] = {};
                    if (in) {
                        if (a.q_vec) {
                            const float4 x = *reinterpret_cast<const float4*>(p + d), y = *reinterpret_cast<const float4*>(p + d + 4);
                            f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
                            f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] = p[d + e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        typename Half8<CT>::one t[NP];
                        query_terms<CT, NP>(f[e], shift, t);
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
        float m, l;
        // O^T as whole vectors throughout: a loop over its elements would have the compiler carry 16 scalars per vector and
        // copy them together for every product
        f16v o[DT];

        // 3. key tiles. A tile's work is two phases with a barrier after each: products (O^T += V^T P^T of the tile
        // before, S^T = K Q^T of this one) and weights (exponentials of S^T; the direct loads of K two tiles and V one tile
        // ahead). Of two waves on a SIMD one runs a phase behind the other, so that one's products go with the other's weights.
        const int n = t1 - t0;
        struct Keys {
            uint32_t row[NI];  // the cache rows this lane loads, ~0: none
            uint64_t there;    // bit j: key j exists; none past the share's last tile, whose loads are of zeros
        };
        const auto keys_of = [&](int t, int page) INLINE {
            Keys k;
            const int j = range.key(t) + lane, at = max(0, min(j, s.len - 1));
            const bool is = (t < t1) & (j < s.len) & (page >= 0) & (page < a.c.pages);
            k.there = __ballot(is);
            const uint32_t row = ((uint32_t)page * a.c.kv_heads + h) * a.c.page_size + (at - page_col(a, at) * a.c.page_size) | ~bit_mask(is);
#pragma unroll
            for (int i = 0; i < NI; ++i) k.row[i] = (uint32_t)__shfl((int)row, load_key + i * RPI, 64);
            return k;
        };
        const auto load = [&](const uint16_t* base, const Keys& k, int to, auto index, auto values) INLINE {
            constexpr int i = decltype(index)::value;
            const int piece = decltype(values)::value ? v_piece ^ v_turn(i * RPI) : k_piece ^ k_turn(i * RPI);
            // selected with masks, not with branches: a divergent branch in the loop would keep it off scalar control flow
            const uint32_t in = bit_mask(k.row[i] != ~0u) & bit_mask(8 * piece < a.c.dim);
            const uint64_t there_at = reinterpret_cast<uint64_t>(base) + ((uint64_t)k.row[i] * a.c.dim + 8 * piece) * 2;
            const uint64_t keep = (uint64_t)in << 32 | in;
            const void* p = reinterpret_cast<const void*>((there_at & keep) | (reinterpret_cast<uint64_t>(a.zeros) & ~keep));
            load_to_lds(p, lds_base + to + (wave * NI + i) * 1024);
        };
        const auto k_tile = [&](int i) { return i % BUFS * TILE; };
        const auto v_tile = [&](int i) { return (BUFS + i % BUFS) * TILE; };
        // With tile i goes a batch of loads: V of tile i + AHEAD, K of tile i + AHEAD + 1 and the pages of tile i + 2 AHEAD + 3.
        // The weights of tile i wait for batch i - AHEAD.
        constexpr int WAIT = EARLY ? AHEAD * BATCH : (AHEAD - 1) * BATCH;
        Keys v_keys, k_keys;
        uint64_t there[AHEAD + 1];  // of tiles i ..
        const auto look_up = [&](int i) INLINE { word_to_lds(page_at(t0 + i + 2 * AHEAD + 3), pages_base + (i + AHEAD + 1) % SLOTS * 256); };
        const auto next_keys = [&](int i) INLINE {  // where the next batch's loads are
            v_keys = k_keys;
            k_keys = keys_of(t0 + i + AHEAD + 2, looked_up[wave][i % SLOTS][lane]);
        };
        constexpr int PARTS = 2 * NI + 2;
        const auto load_part = [&](int i, auto part) INLINE {
            constexpr int P = decltype(part)::value;
            if constexpr (P < NI) load(a.c.v, v_keys, v_tile(i + AHEAD), Index<P>{}, Index<1>{});
            else if constexpr (P < 2 * NI) load(a.c.k, k_keys, k_tile(i + AHEAD + 1), Index<P - NI>{}, Index<0>{});
            else if constexpr (P == 2 * NI) look_up(i);
            else next_keys(i);
        };
        const auto load_batch = [&](int i) INLINE { unrolled<0, PARTS>([&](auto part) INLINE { load_part(i, part); }); };

        f16v sc[2];
        vec wt[NP][4];
        constexpr int LEAD = 4, NV = 4 * DT, NK = 2 * STEPS;  // operands read ahead of their use; operands of a tile's V and K
        const auto v_operand = [&](int tile, int k) INLINE {
            lds_byte* at = (lds_byte*)((uintptr_t)(lds3 + (v_at + tile)) ^ (64 * (k % DT)));
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + k / DT * 16 * ROW));
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + k / DT * 16 * ROW + 8 * ROW));
            return __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        const auto k_operand = [&](int tile, int k) INLINE {
            typedef __attribute__((address_space(3))) vec lds_vec;
            return *(lds_vec*)(((uintptr_t)(lds3 + (k_at + tile)) ^ (32 * (k / 2))) + k % 2 * 32 * ROW);
        };
        // O^T += V^T P^T of the tile at vt, then S^T = K Q^T of the tile at kt, in one run of reads and products, with batch `batch` of the loads spread between the products (where they are early)
        const auto products = [&](int vt, int kt, int batch, auto with_v, auto with_k) INLINE {
            constexpr int V0 = decltype(with_v)::value ? 0 : NV, N = decltype(with_k)::value ? NV + NK : NV;
            vec ring[LEAD + 1];
            const auto read = [&](auto k) INLINE {
                constexpr int K = decltype(k)::value;
                if constexpr (K < NV) ring[K % (LEAD + 1)] = v_operand(vt, K);
                else ring[K % (LEAD + 1)] = k_operand(kt, K - NV);
            };
            unrolled<V0, (V0 + LEAD < N ? V0 + LEAD : N)>(read);
            unrolled<V0, N>([&](auto k) INLINE {
                constexpr int K = decltype(k)::value;
                if constexpr (K + LEAD < N) read(Index<K + LEAD>{});
                __builtin_amdgcn_sched_barrier(0);
                const vec x = ring[K % (LEAD + 1)];
                if constexpr (K < NV) {
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) o[K % DT] = mfma32(x, wt[p][K / DT], o[K % DT]);
                } else {
                    constexpr int E = K - NV;
                    if constexpr (E / 2 == 0) sc[E % 2] = (f16v)(0.0f);
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) sc[E % 2] = mfma32(x, q[p][E / 2], sc[E % 2]);
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (EARLY && decltype(with_k)::value) {  // part P follows product V0 + (P + 1) (N - V0) / (PARTS + 1)
                    static_assert(PARTS < NK, "");
                    constexpr int P = ((K + 1 - V0) * (PARTS + 1) + N - V0 - 1) / (N - V0) - 1;
                    if constexpr (P < PARTS && (P + 1) * (N - V0) / (PARTS + 1) == K + 1 - V0) {
                        load_part(batch, Index<P>{});
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            });
        };
        uint32_t see[2];
        uint64_t here;  // of the tile at hand
        const auto next_there = [&]() INLINE {
            here = there[0];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) there[k] = there[k + 1];
            there[AHEAD] = v_keys.there;
        };
        const auto begin_weights = [&](int i) INLINE {  // the second phase, up to scores (log2, or raw ones that `factor` scales)
            const int j0 = range.key(t0 + i);
            if constexpr (EARLY) next_there();
            phase_barrier<WAIT>();
            if constexpr (!EARLY) {
                load_batch(i);
                next_there();
            }
            see[0] = see[1] = ~0u;
            if constexpr (EXTRA) {  // to capped and biased scores (log2)
                if (a.softcap > 0.0f && NP == 1) {
                    const float f = factor * (2.0f * kLog2e / a.softcap), top = a.softcap * kLog2e;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            sc[kb][e] = fmaf(-2.0f * top, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[kb][e] * f)), top);
                } else if (a.softcap > 0.0f) {
                    const float f = factor / a.softcap, top = a.softcap * kLog2e;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[kb][e] = top * soft_tanh<true>(sc[kb][e] * f);
                } else {
                    const float f = factor * kLog2e;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[kb][e] *= f;
                }
                if (a.slopes) {
                    const float back = (float)(pos - j0 - 4 * hf);
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[kb][e] = fmaf(-slope, fabsf(back - (float)(32 * kb + 8 * (e / 4) + e % 4)), sc[kb][e]);
                }
            }
            const bool full = here == ~0ull && ((j0 + T - 1 <= wp0 && (a.window <= 0 || wp1 - j0 < a.window)) || j0 + T <= s.prefix);
            if (!full) {  // without branches: all 64 lanes take part in what follows
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    see[kb] = seen_keys(a, s, pos, j0 + 32 * kb, (uint32_t)(here >> (32 * kb)));
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[kb][e] = (int)(see[kb] >> (4 * hf) << (31 - 8 * (e / 4) - e % 4)) < 0 ? sc[kb][e] : -INFINITY;
                }
            }
        };
        // Weights against the row's reference. Their sum bounds the largest of them: only where it passes the limit (or the row
        // has no reference yet) is a maximum looked for, the reference raised and the sums scaled down.
        float sum = 0.0f;
        const auto weigh = [&]() INLINE {
            const float base = m == -INFINITY ? 0.0f : m - kShift;
            sum = 0.0f;
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = sc[st / 2][8 * (st & 1) + e];
                    const float v = __builtin_amdgcn_exp2f(EXTRA ? x - base : fmaf(x, factor, -base));
                    sum += v;
                    typename Half8<CT>::one t[NP];
                    split_terms<CT, NP>(v, t);
#pragma unroll
                    for (int p = 0; p < NP; ++p) wt[p][st][e] = t[p];
                }
        };
        const auto past_limit = [&]() INLINE { return (int)__builtin_amdgcn_readfirstlane(__ballot((sum > kLimit) | (m == -INFINITY)) != 0); };
        const auto raise_reference = [&]() INLINE {
            float top = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[kb][e]);
            if (!EXTRA) top *= factor;
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float raised = fmaxf(m, top);
            const float fade = raised == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
            m = raised;
            l *= fade;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = o[dt] * (f16v)(fade);
        };
        const auto weights = [&](int i) INLINE {
            begin_weights(i);
            weigh();
            if (past_limit()) {
                raise_reference();
                weigh();
            }
            l += sum;
            phase_barrier<-1>();
        };
        const auto odd_values = [&](int i) INLINE {  // O^T += V^T P^T of the finite values, and the others where they are seen
            const uint8_t* vt = lds + v_tile(i);
            for (int key = 0; key < T; ++key) {
                const uint32_t mine = (key < 32 ? see[0] >> key : see[1] >> (key - 32)) & 1u;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    f16v add;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {  // dimensions 32 dt + 8 g + 4 hf .. + 3
                        const int piece = (4 * dt + g) ^ v_turn(key);
                        const uint2 v = *reinterpret_cast<const uint2*>(vt + key * ROW + piece * 16 + 8 * hf);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t bits = (e < 2 ? v.x : v.y) >> (16 * (e & 1)) & 0xFFFFu;
                            const float val = CT == BYHIP_F16 ? (float)bits_h((uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
                            add[4 * g + e] = mine & (uint32_t)((bits & kExp) == kExp) ? val : 0.0f;
                        }
                    }
                    o[dt] = o[dt] + add;
                }
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint4 v = __builtin_bit_cast(uint4, v_operand(v_tile(i), k));
                const vec x = __builtin_bit_cast(vec, make_uint4(finite_only(v.x, kExp), finite_only(v.y, kExp), finite_only(v.z, kExp), finite_only(v.w, kExp)));
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) o[k % DT] = mfma32(x, wt[p][k / DT], o[k % DT]);
            }
        };
        const auto careful_scores = [&](int i) INLINE {  // S^T = K Q^T, infinite keys with the queries' first terms alone, which have their signs
            if constexpr (EARLY) load_batch(i);
            unrolled<0, NK>([&](auto k) INLINE {
                constexpr int E = decltype(k)::value;
                const vec x = k_operand(k_tile(i), E);
                const uint4 v = __builtin_bit_cast(uint4, x);
                const vec y = __builtin_bit_cast(vec, make_uint4(finite_only(v.x, kExp), finite_only(v.y, kExp), finite_only(v.z, kExp), finite_only(v.w, kExp)));
                if constexpr (E / 2 == 0) sc[E % 2] = (f16v)(0.0f);
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) sc[E % 2] = mfma32(p ? y : x, q[p][E / 2], sc[E % 2]);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        // Values that are not finite spoil the sums of rows that do not see them (0 times infinity), and of rows that do where
        // weights have several terms (infinity less infinity), as infinite keys do where queries have. That shows in the sums,
        // so the tiles are not searched for them: a block whose sums are not finite works through them once more, carefully,
        // adding such values only where they are seen.
        bool careful = false;
        for (;;) {
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = (f16v)(0.0f);
            phase_barrier<0>();  // the item before has been read
            look_up(-AHEAD - 1);
            k_keys = keys_of(t0, first_pages[0]);
            unrolled<0, NI>([&](auto part) INLINE { load(a.c.k, k_keys, k_tile(0), part, Index<0>{}); });
#pragma unroll
            for (int i = -AHEAD; i < 0; ++i) {
                there[i + AHEAD] = k_keys.there;
                v_keys = k_keys;
                k_keys = keys_of(t0 + i + AHEAD + 1, first_pages[i + AHEAD + 1]);
                unrolled<0, PARTS - 1>([&](auto part) INLINE { load_part(i, part); });
            }
            there[AHEAD] = k_keys.there;
            v_keys = k_keys;
            k_keys = keys_of(t0 + AHEAD + 1, first_pages[AHEAD + 1]);
            phase_barrier<AHEAD * BATCH>();
            if (PAIRED && wave >= WAVES / 2) phase_barrier<-1>();
            if (row0 >= s.rows) {  // a wave without rows brings its share of the tiles
                for (int i = 0; i < n; ++i) {
                    if constexpr (EARLY) load_batch(i);
                    phase_barrier<WAIT>();
                    if constexpr (!EARLY) load_batch(i);
                    phase_barrier<-1>();
                }
            } else if (!careful) {  // a loop with one exit and no choice but the rare raise in it: with more, the compiler carries all sums twice
                products(0, k_tile(0), 0, Index<0>{}, Index<1>{});
                weights(0);
                int i = 0;
                while (i < n - 1) {
                    products(v_tile(i), k_tile(i + 1), i + 1, Index<1>{}, Index<1>{});
                    weights(++i);
                }
                products(v_tile(i), 0, 0, Index<1>{}, Index<0>{});
            } else {
                for (int i = 0; i < n; ++i) {
                    if constexpr (NP > 1) careful_scores(i);
                    else products(0, k_tile(i), i, Index<0>{}, Index<1>{});
                    weights(i);
                    odd_values(i);
                }
            }
            if (PAIRED && wave < WAVES / 2) phase_barrier<-1>();
            if (careful) break;
            uint32_t odd = 0;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) odd |= bit_mask(!(fabsf(o[dt][e]) < INFINITY));
            ++pass;
            if (__ballot(odd != 0 && valid) != 0 && lane == 0) not_finite = pass;
            phase_barrier<-1>();
            careful = uniform(not_finite) == pass;
            if (!careful) break;
        }

        // 4. the wave's rows leave, whole or as a part
        const bool begins = t0 == 0, ends = t1 == range.tiles;
        l += __shfl_xor(l, 32, 64);
        if (begins && ends) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const size_t at = (size_t)(a.s.starts[b] + token) * a.out_stride + (size_t)hq * a.c.dim + 4 * hf;
            const auto leave = [&](auto dtype, auto vector) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int d = 32 * dt + 8 * g;
                        if (d >= a.c.dim) continue;  // the same for all lanes: heads are multiples of 8
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = l == 0.0f ? 0.0f : o[dt][4 * g + e] * inv;
                        if constexpr (decltype(vector)::value) {
                            store_vec<4>(a.out, at + d, x, decltype(dtype)::value);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) store_y<decltype(dtype)::value>(a.out, at + d + e, x[e]);
                        }
                    }
            };
            const auto leave_as = [&](auto dtype) {
                if (a.out_vec) leave(dtype, Index<1>{});
                else leave(dtype, Index<0>{});
            };
            if (valid) {
                if (a.out_dtype == BYHIP_F32) leave_as(Index<BYHIP_F32>{});
                else if (a.out_dtype == BYHIP_F16) leave_as(Index<BYHIP_F16>{});
                else leave_as(Index<BYHIP_BF16>{});
            }
        } else if (valid) {
            const int r = wave * 32 + c;
            float* slot = part_slot<R, DIM>(a.part, begins ? 2 * w + 1 : 2 * w);
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
        u += whole ? blocks : t1 - t0;
    }
    if (tid == 0) a.joins[w] = join;
    phase_barrier<0>();  // no load on its way to LDS that is given back
}

template <int CT, int NP, int DIM, int USED, int WAVES>
void launch_chunk(const AttnArgs& a) {
    constexpr size_t kSlots = (size_t)2 * 32 * WAVES * (DIM + 2) * sizeof(float);  // one block's
    const size_t room = (kAttnWorkspaceBytes - kAttnJoinBytes) / kSlots;
    // no more than the tiles that the tables have room for
    const long long items = (a.s.batch + (long long)a.s.rows * a.group / (32 * WAVES)) * a.c.kv_heads;
    const long long tiles = items * ((key_room(a) + kChunkKeys - 1) / kChunkKeys);
    const unsigned blocks = (unsigned)std::min<long long>(std::min<long long>((long long)room, compute_units()), std::max(1LL, tiles));
    if (a.softcap > 0.0f || a.slopes || !(a.scale >= kLeastScale)) launch("attn_chunk", (attn_chunk<CT, NP, DIM, USED, WAVES, true>), dim3(blocks), dim3(64 * WAVES), 0, a);
    else launch("attn_chunk", (attn_chunk<CT, NP, DIM, USED, WAVES, false>), dim3(blocks), dim3(64 * WAVES), 0, a);
    BYHIP_LAUNCHED("attn_chunk");
    launch("attn_join", (attn_join<32 * WAVES, DIM, 1>), dim3(blocks, 16), dim3(256), 0, a);
    BYHIP_LAUNCHED("attn_join");
}

// Blocks of 8 waves where two waves per SIMD have the registers they need, else of 4.
template <int CT, int NP>
void launch_chunk_dim(const AttnArgs& a) {
    if (a.c.dim <= 64) launch_chunk<CT, NP, 64, 64, NP == 1 ? 8 : 4>(a);
    else if (a.c.dim <= 96) launch_chunk<CT, NP, 128, 96, NP == 1 ? 8 : 4>(a);
    else if (a.c.dim <= 128) launch_chunk<CT, NP, 128, 128, NP == 1 ? 8 : 4>(a);
    else launch_chunk<CT, NP, 256, 256, 4>(a);
}

}  // namespace
}  // namespace byhip
