// byhip_attn_rows.h - attention of few rows per sequence over a paged cache: decoding (gfx950).
//
// A sequence's rows that share a key head (tokens x group) form tiles of 16. A wave takes 32 keys at a
// time, straight from memory into the registers the matrix instructions read:
//   S^T = K Q^T  v_mfma_f32_16x16x32, twice 16 keys: lane c + 16 g holds key c's values 32 s + 8 g ..
//   O^T = V^T P^T  contracts over the 32 keys in the order in which S^T left them: lane group g holds keys 4 g + r and
//                  16 + 4 g + r, as exponentials and sums, without any exchange between lanes. V^T comes from the lane's own loads:
//                  it reads DIM / 16 neighbouring values of its 8 keys, and those 8 x DIM / 16 values are turned around
//                  with byte permutes; that column t of a lane is dimension c DIM / 16 + t only renames rows of O^T.
// The maximum of a row is kept as a reference that is raised (and the sums scaled down) only when a score passes it by
// 2^8, so most tiles exchange nothing between lanes at all. fp16 weights carry a factor 2^7 so that small ones stay clear
// of fp16's subnormals.
//
// What bounds it: bytes (64 sequences of 300 to 8192 keys, a row each, bf16: 205 us for 1.15 GB, 5.6 TB/s; 2 of up to 131072,
// fp32 on fp16: 186 us for 1.02 GB, 5.5 TB/s). Each key and value is read once per 16 rows, so the work is divided by keys, not by
// sequences: all (head, sequence, row tile) items are laid end to end in tiles of 32 keys and every block takes
// an equal run of them, whatever the lengths. A block therefore holds the end of one item and the start of another; their
// parts go to the workspace and attn_join adds them.
//
// fp32 queries or outputs: the queries as two fp16 terms (scaled per row to fp16's range) or three bf16 terms, the
// weights likewise, one matrix instruction per term; the memory still bounds it. With 16-bit rows on both sides a weight is
// rounded once to the cache's type, in which the matrix instruction takes it: the output is then off from 64 bits by 1.1 (fp16) to 1.4
// times (bf16) what its own rounding leaves, and a caller who needs less asks for fp32 output.
#pragma once

#include <algorithm>
#include <type_traits>

#include "byhip_attn.h"

namespace byhip {
namespace {

constexpr int kKeys = 32;      // keys per tile of a wave
constexpr int kWaves = 4;
constexpr int kRows = 16;
constexpr float kRaise = 8.0f;  // log2 by which a score may pass its row's reference

template <int CT, int NP, int DIM, bool EXTRA>
struct Rows {
    typedef typename Half8<CT>::vec vec;
    static constexpr int STEPS = DIM / 32, V = DIM / 16;
    static constexpr float kShift = CT == BYHIP_F16 ? 7.0f : 0.0f;  // log2 of the weights' factor
    static constexpr uint32_t kExp = CT == BYHIP_F16 ? 0x7C00u : 0x7F80u;
    typedef uint32_t KTile[2][STEPS][4];
    typedef uint32_t VTile[8][V / 2];

    const AttnArgs& a;
    const int lane, c, g;
    SeqInfo s;
    int head, pos;             // key head, this lane's row's position
    int koff[STEPS], voff[(V + 7) / 8];  // this lane's values of a key (those past the head's end read its first)
    uint32_t kmask[STEPS];     // 0 for those past the end
    float slope, factor;       // factor: scale (and the row's power of two), with log2 e unless EXTRA
    float inv_cap;
    bool valid;                // this lane's row exists
    bool again;                // the item's second pass (rows of one term)
    vec q[NP][STEPS];
    float m, l;                // reference (log2) of row c; this lane's sum of weights
    f4 o[V];

    __device__ __forceinline__ Rows(const AttnArgs& args) : a(args), lane(threadIdx.x & 63), c(lane & 15), g(lane >> 4) {
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            const bool in = 32 * st + 8 * g < a.c.dim;
            koff[st] = in ? 32 * st + 8 * g : 0;
            kmask[st] = in ? ~0u : 0u;
        }
#pragma unroll
        for (int e = 0; e < (V + 7) / 8; ++e) voff[e] = V * c + 8 * e < a.c.dim ? V * c + 8 * e : 0;
    }

    // The cache row of key j0 + lane % 32; `there`: bit j for the keys that exist (others read row 0). No branches:
    // all 64 lanes take part in what follows.
    __device__ __forceinline__ uint32_t key_row(int b, int j0, uint32_t& there) const {
        const int j = j0 + (lane & 31);
        const int at = max(0, min(j, s.len - 1)), col = page_col(a, at);
        const int page = a.s.table[(size_t)b * a.s.stride + col];
        const bool is = (j < s.len) & (page >= 0) & (page < a.c.pages);
        there = (uint32_t)__ballot(is);
        return (((uint32_t)page * a.c.kv_heads + head) * a.c.page_size + (at - col * a.c.page_size)) & bit_mask(is);
    }
    __device__ __forceinline__ void load_k(KTile& k, uint32_t rows) const {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const uint16_t* p = a.c.k + (size_t)(uint32_t)__shfl((int)rows, 16 * kb + c, 64) * a.c.dim;
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const uint4 x = *reinterpret_cast<const uint4*>(p + koff[st]);
                k[kb][st][0] = x.x; k[kb][st][1] = x.y; k[kb][st][2] = x.z; k[kb][st][3] = x.w;
            }
        }
    }
    __device__ __forceinline__ void load_v(VTile& v, uint32_t rows) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t* p = a.c.v + (size_t)(uint32_t)__shfl((int)rows, 16 * (i / 4) + 4 * g + i % 4, 64) * a.c.dim;
            if constexpr (V == 4) {
                const uint2 x = *reinterpret_cast<const uint2*>(p + voff[0]);
                v[i][0] = x.x; v[i][1] = x.y;
            } else {
#pragma unroll
                for (int e = 0; e < V / 8; ++e) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p + voff[e]);
                    v[i][4 * e] = x.x; v[i][4 * e + 1] = x.y; v[i][4 * e + 2] = x.z; v[i][4 * e + 3] = x.w;
                }
            }
        }
    }

    // Row c of tile rt: its position, its query as NP terms.
    __device__ __forceinline__ void begin(int b, int h, int rt) {
        s = seq_info(a, b);
        head = h;
        const int row = rt * kRows + c;
        valid = row < s.rows;
        const int token = valid ? row / a.group : 0, hq = h * a.group + (valid ? row % a.group : 0);
        pos = s.first_pos + token;
        slope = EXTRA && a.slopes ? a.slopes[hq] * kLog2e : 0.0f;
        const size_t base = (size_t)(a.s.starts[b] + token) * a.q_stride + (size_t)hq * a.c.dim;
        float x[STEPS][8];
        int shift = 0;
        if (a.q_dtype == BYHIP_F32) {
            float top = 0.0f;
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[st][e] = 0.0f;
                if (valid && kmask[st]) {
                    const float* p = static_cast<const float*>(a.q) + base + 32 * st + 8 * g;
                    if (a.q_vec) {
                        const float4 u = *reinterpret_cast<const float4*>(p), w = *reinterpret_cast<const float4*>(p + 4);
                        x[st][0] = u.x; x[st][1] = u.y; x[st][2] = u.z; x[st][3] = u.w;
                        x[st][4] = w.x; x[st][5] = w.y; x[st][6] = w.z; x[st][7] = w.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[st][e] = p[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[st][e]));
            }
            if constexpr (CT == BYHIP_F16) {  // the row's largest value to [2^14, 2^15)
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                shift = query_shift(top);
            }
#pragma unroll
            for (int st = 0; st < STEPS; ++st)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    typename Half8<CT>::one t[NP];
                    query_terms<CT, NP>(x[st][e], shift, t);
#pragma unroll
                    for (int p = 0; p < NP; ++p) q[p][st][e] = t[p];
                }
        } else {
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                uint4 u = make_uint4(0, 0, 0, 0);
                if (valid && kmask[st]) {
                    const uint16_t* p = static_cast<const uint16_t*>(a.q) + base + 32 * st + 8 * g;
                    if (a.q_vec) {
                        u = *reinterpret_cast<const uint4*>(p);
                    } else {
                        u.x = p[0] | (uint32_t)p[1] << 16; u.y = p[2] | (uint32_t)p[3] << 16;
                        u.z = p[4] | (uint32_t)p[5] << 16; u.w = p[6] | (uint32_t)p[7] << 16;
                    }
                }
                q[0][st] = __builtin_bit_cast(vec, u);
#pragma unroll
                for (int p = 1; p < NP; ++p) q[p][st] = __builtin_bit_cast(vec, make_uint4(0, 0, 0, 0));
            }
        }
        inv_cap = EXTRA && a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
        factor = ldexpf(EXTRA ? a.scale : a.scale * kLog2e, -shift);
    }
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < V; ++t) o[t] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ bool finite() const {  // whether all sums of the wave's rows are
        float none = 0.0f;  // NaN where a sum is infinite or NaN
#pragma unroll
        for (int t = 0; t < V; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) none = fmaf(o[t][e], 0.0f, none);
        return __ballot(none != 0.0f && valid) == 0;
    }

    // One tile of keys j0 ..; `there`: bit j of the keys that exist; `read`: called once k has been read.
    template <bool CAREFUL, typename F>
    __device__ __forceinline__ void tile(const KTile& k, VTile& v, int j0, uint32_t there, int p0, int p1, F&& read) {
        float x[8];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = k[kb][st][e] & kmask[st];
                        // the further terms of a query may have another sign than it has, or be 0: an infinite key meets the first alone
                        if (CAREFUL && p) w[e] = finite_only(w[e], kExp);
                    }
                    acc = mfma16(__builtin_bit_cast(vec, make_uint4(w[0], w[1], w[2], w[3])), q[p][st], acc);
                }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * kb + r] = acc[r] * factor;
        }
        read();
        if constexpr (EXTRA) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (a.softcap > 0.0f) x[i] = a.softcap * soft_tanh<(NP > 1)>(x[i] * inv_cap);
                x[i] = x[i] * kLog2e - slope * fabsf((float)(pos - (j0 + 16 * (i / 4) + 4 * g + i % 4)));
            }
        }
        const bool all = there == ~0u && ((j0 + kKeys - 1 <= p0 && (a.window <= 0 || p1 - j0 < a.window)) || j0 + kKeys <= s.prefix);
        uint32_t see = ~0u;
        if (!all) {  // without branches: all 64 lanes take part in what follows
            see = seen_keys(a, s, pos, j0, there);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = see >> (16 * (i / 4) + i % 4) >> (4 * g) & 1u ? x[i] : -INFINITY;
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__ballot(top > m + kRaise || (m == -INFINITY && top > m))) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float raised = fmaxf(m, top);
            const float fade = raised == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
            m = raised;
            l *= fade;
#pragma unroll
            for (int t = 0; t < V; ++t) o[t] *= fade;
        }
        if (CAREFUL || (NP == 1 && again) || !all) spare(v, see, there);
        const float base = m == -INFINITY ? 0.0f : m - kShift;
        vec w[NP];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(x[i] - base);
            l += e;
            typename Half8<CT>::one t[NP];
            split_terms<CT, NP>(e, t);
#pragma unroll
            for (int p = 0; p < NP; ++p) w[p][i] = t[p];
        }
#pragma unroll
        for (int t = 0; t < V; ++t) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                u[i] = __builtin_amdgcn_perm(v[2 * i + 1][t / 2], v[2 * i][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
            const vec vt = __builtin_bit_cast(vec, make_uint4(u[0], u[1], u[2], u[3]));
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) o[t] = mfma16(vt, w[p], o[t]);
        }
    }

    // A hidden value that is not finite would spoil the sums (0 times infinity), and so would one that is seen where
    // weights have several terms or round to 0: values of keys that do not exist are cleared, others that are not finite are taken out of V and
    // added to the rows that see them.
    __device__ __forceinline__ void spare(VTile& v, uint32_t see, uint32_t there) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t keep = there >> (16 * (i / 4) + 4 * g + i % 4) & 1u ? ~0u : 0u;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) v[i][e] &= keep;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t odd = 0;
#pragma unroll
            for (int e = 0; e < V / 2; ++e) odd |= (uint32_t)((v[i][e] & kExp) == kExp) | (uint32_t)((v[i][e] >> 16 & kExp) == kExp);
            if (!__ballot(odd != 0)) continue;
            for (int from = 0; from < 4; ++from) {
                const uint32_t mine = see >> (16 * (i / 4) + 4 * from + i % 4) & 1u;
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // o[t][r]: dimension V (4 g + r) + t of row c
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        const uint32_t word = (uint32_t)__shfl((int)v[i][e], 16 * from + 4 * g + r, 64);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t bits = word >> (16 * half) & 0xFFFFu;
                            const float val = CT == BYHIP_F16 ? (float)bits_h((uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
                            o[2 * e + half][r] += mine & (uint32_t)((bits & kExp) == kExp) ? val : 0.0f;
                        }
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                v[i][e] = finite_only(v[i][e], kExp);
            }
        }
    }
};

// Blocks resident per CU: two, but one where 256 registers per lane would not hold a tile (heads of 129 to 256 values; 4 sequences
// of 65536 keys, 8 key heads of 256, 2.15 GB: 372 us with one, 754 with two; fp32 398 and 1631). With one, 2 to 6 registers of the
// 16-bit forms still go to memory, 43 to 48 of fp32 on fp16, 100 of fp32 on bf16; no other form spills any.
constexpr int rows_blocks(int dim) { return dim > 128 ? 1 : 2; }

template <int CT, int NP, int DIM, bool EXTRA>
__global__ __launch_bounds__(256, rows_blocks(DIM)) void attn_rows(AttnArgs a) {
    constexpr int V = DIM / 16, kPitch = DIM + 4;
    __shared__ long long before[kAttnBatch + 1];  // units (tiles of 32 keys x row tiles) of the sequences before each
    __shared__ long long wave_sum_of[kWaves];
    __shared__ __attribute__((aligned(16))) float acc[kWaves][kRows][kPitch];
    __shared__ float top_of[kWaves][kRows], sum_of[kWaves][kRows];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;

    const auto tiles_of = [&](const SeqInfo& s) { return TileRange<kKeys>(a, s, s.first_pos, s.first_pos + s.rows / a.group - 1); };
    // 1. units before each sequence: a run of sequences per thread, then a scan over the block (1.2 us, so not for one)
    const bool one = a.s.batch == 1;
    long long all_units = 0;
    if (one) {
        const SeqInfo s = seq_info(a, 0);
        if (s.rows) all_units = (long long)((s.rows + kRows - 1) / kRows) * tiles_of(s).tiles;
    } else {
        const int per = (a.s.batch + 255) / 256, b0 = min(tid * per, a.s.batch), b1 = min(b0 + per, a.s.batch);
        long long sum = 0;
        for (int b = b0; b < b1; ++b) {
            const SeqInfo s = seq_info(a, b);
            before[b] = sum;
            if (s.rows) sum += (long long)((s.rows + kRows - 1) / kRows) * tiles_of(s).tiles;
        }
        long long scan = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const long long u = __shfl_up(scan, o, 64);
            if (lane >= o) scan += u;
        }
        if (lane == 63) wave_sum_of[wave] = scan;
        __syncthreads();
        long long base = scan - sum;
        for (int w = 0; w < wave; ++w) base += wave_sum_of[w];
        for (int b = b0; b < b1; ++b) before[b] += base;
        if (tid == 255) before[a.s.batch] = base + sum;
        __syncthreads();
        all_units = before[a.s.batch];
    }
    const long long per_head = uniform(all_units), total = per_head * a.c.kv_heads;
    // 2. this block's run of units
    const long long blocks = min((long long)gridDim.x, max(1LL, (total + kWaves - 1) / kWaves));
    const int w = blockIdx.x;
    if (w >= blocks || total == 0) {
        if (tid == 0) a.joins[w] = make_int4(0, 0, 0, 0);
        return;
    }
    const long long u0 = total * w / blocks, u1 = total * (w + 1) / blocks;
    int4 join = make_int4(0, 0, 0, 0);

    Rows<CT, NP, DIM, EXTRA> r(a);
    for (long long u = u0; u < u1;) {
        const int h = (int)(u / per_head);
        const long long in_head = u - h * per_head;
        int lo = 0, hi = a.s.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (before[mid] <= in_head) lo = mid;
            else hi = mid - 1;
        }
        const int b = uniform(lo);
        const long long local = one ? in_head : in_head - uniform(before[b]);
        SeqInfo s = seq_info(a, b);
        const auto range = tiles_of(s);
        const int rt = (int)(local / range.tiles), t0 = (int)(local % range.tiles);
        const int t1 = (int)min((long long)range.tiles, t0 + (u1 - u));
        r.begin(b, h, rt);
        const int p0 = s.first_pos + rt * kRows / a.group, p1 = s.first_pos + (min(s.rows, (rt + 1) * kRows) - 1) / a.group;

        // 3. the wave's tiles t0 + wave, + 4, ..: the next tile's keys and the one after's page lookups are under way
        // while one is worked on
        typename Rows<CT, NP, DIM, EXTRA>::KTile ka, kb;
        typename Rows<CT, NP, DIM, EXTRA>::VTile v;
        int t;
        uint32_t rows, next, there, next_there;
        const auto step = [&](auto& cur, auto& ahead, auto careful) __attribute__((always_inline)) {
            constexpr bool kOneTile = DIM > 128 || (DIM > 64 && NP > 1) || decltype(careful)::value;  // registers for one tile of keys: the next one's follow its last use
            r.load_v(v, rows);
            uint32_t after = 0, after_there = 0;
            if (t + 2 * kWaves < t1) after = r.key_row(b, range.key(t + 2 * kWaves), after_there);
            if (!kOneTile && t + kWaves < t1) r.load_k(ahead, next);
            r.template tile<decltype(careful)::value>(cur, v, range.key(t), there, p0, p1, [&] {
                if (kOneTile) r.load_k(cur, next);  // row 0 after the last tile
            });
            rows = next;
            there = next_there;
            next = after;
            next_there = after_there;
            t += kWaves;
        };
        const auto start = [&]() __attribute__((always_inline)) {
            r.clear();
            t = t0 + wave;
            rows = next = there = next_there = 0;
            if (t < t1) rows = r.key_row(b, range.key(t), there);
            if (t + kWaves < t1) next = r.key_row(b, range.key(t + kWaves), next_there);
            if (t < t1) r.load_k(ka, rows);
        };
        const auto walk = [&](auto careful) __attribute__((always_inline)) {
            while (t < t1) {
                step(ka, kb, careful);
                if (DIM > 128 || (DIM > 64 && NP > 1) || decltype(careful)::value) continue;
                if (t >= t1) break;
                step(kb, ka, careful);
            }
        };
        // Values that are not finite spoil the sums of rows where a weight is rounded to 0 (0 times infinity), or has several terms,
        // as infinite keys do where queries have. That shows in the sums, so full tiles are not searched for them: a wave whose
        // sums are not finite walks once more, carefully. (Two copies of the loop where weights have several terms: 398 us from
        // 504 with a search of every tile, 4 x 65536 keys of 8 heads of 256 values, fp32 on bf16; one copy where they have one, whose
        // loop for 128 values would spill registers beside another: 205 us and 223, 64 sequences of up to 8192 keys. The look at
        // the sums costs a call of one row 0.4 us; behind the waves' join, one look for the block, 1.0.)
        start();
        if constexpr (NP == 1) {
            r.again = false;
            for (;;) {
                walk(std::false_type{});
                if (r.again || r.finite()) break;
                r.again = true;
                start();
            }
        } else {
            walk(std::false_type{});
            if (!r.finite()) {
                start();
                walk(std::true_type{});
            }
        }

        // 4. the waves' sums join in LDS
        float l = r.l;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        __syncthreads();
        if (r.g == 0) { top_of[wave][r.c] = r.m; sum_of[wave][r.c] = l; }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < V; i += 4)
                *reinterpret_cast<f4*>(&acc[wave][r.c][V * (4 * r.g + e) + i]) = (f4){r.o[i][e], r.o[i + 1][e], r.o[i + 2][e], r.o[i + 3][e]};
        __syncthreads();
        const bool begins = t0 == 0, ends = t1 == range.tiles;
        const int row = tid >> 4, col = (tid & 15) * V, q = rt * kRows + row;
        if (q < s.rows) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) top = fmaxf(top, top_of[i][row]);
            const float base = top == -INFINITY ? 0.0f : top;
            float f[kWaves], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                f[i] = __builtin_amdgcn_exp2f(top_of[i][row] - base);
                sum += sum_of[i][row] * f[i];
            }
            float* slot = part_slot<kRows, DIM>(a.part, begins ? 2 * w + 1 : 2 * w);
            if (!(begins && ends) && col == 0) {
                slot[kRows * DIM + row] = top;
                slot[kRows * DIM + kRows + row] = sum;
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const size_t out = (size_t)(a.s.starts[b] + q / a.group) * a.out_stride + (size_t)(h * a.group + q % a.group) * a.c.dim;
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kWaves; ++j) x[e] += acc[j][row][col + i + e] * f[j];
                }
                if (!(begins && ends)) {
                    *reinterpret_cast<float4*>(slot + row * DIM + col + i) = make_float4(x[0], x[1], x[2], x[3]);
                } else if (col + i < a.c.dim) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = sum == 0.0f ? 0.0f : x[e] * inv;
                    if (a.out_vec) {
                        store_vec<4>(a.out, out + col + i, x, a.out_dtype);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float one[1] = {x[e]};
                            store_vec<1>(a.out, out + col + i + e, one, a.out_dtype);
                        }
                    }
                }
            }
        }
        if (begins && !ends) join = join_of(u - t0 + range.tiles - 1, blocks, total, b, rt, h);
        u += t1 - t0;
    }
    if (tid == 0) a.joins[w] = join;
}

template <int CT, int NP, int DIM>
void launch_rows(const AttnArgs& a) {
    // no more than the units that the tables have room for
    const long long row_tiles = a.s.batch + (long long)a.s.rows * a.group / kRows;
    const long long units = row_tiles * ((key_room(a) + kKeys - 1) / kKeys) * a.c.kv_heads;
    const unsigned blocks = (unsigned)std::min<long long>(compute_units() * rows_blocks(DIM), std::max(1LL, (units + kWaves - 1) / kWaves));
    // a token per sequence, as a rule, where there are no more rows than sequences: a tile then has the group's rows
    const unsigned join_rows = (unsigned)(a.s.rows <= a.s.batch ? std::min(kRows, a.group) : kRows);
    if (a.softcap > 0.0f || a.slopes) launch("attn_rows", (attn_rows<CT, NP, DIM, true>), dim3(blocks), dim3(256), 0, a);
    else launch("attn_rows", (attn_rows<CT, NP, DIM, false>), dim3(blocks), dim3(256), 0, a);
    BYHIP_LAUNCHED("attn_rows");
    launch("attn_join", (attn_join<kRows, DIM, 4>), dim3(blocks, join_rows), dim3(256), 0, a);
    BYHIP_LAUNCHED("attn_join");
}

template <int CT, int NP>
void launch_rows_dim(const AttnArgs& a) {
    if (a.c.dim <= 64) launch_rows<CT, NP, 64>(a);
    else if (a.c.dim <= 128) launch_rows<CT, NP, 128>(a);
    else launch_rows<CT, NP, 256>(a);
}

}  // namespace
}  // namespace byhip
