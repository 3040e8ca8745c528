// byhip_route.hip - routing to experts (gfx950): scores, the best of them per token, and the plan that orders the
// assignments by expert; and the sum of a token's rows afterwards.
//
// A wave routes a token: lane l holds the experts V l .. V l + V - 1 and the best of those not yet chosen, its head, so that a
// round of the selection looks at 64 heads and only the winner's lane looks for its next. Keys are compared as whole numbers with floats' order (0: not a choice); keys that are
// sums with a bias, or ranked by groups' sums, are formed in 64 bits, where their heads' 32-bit roundings tie the 64-bit
// values decide.
//
// The plan is a stable counting sort. A wave takes 64 assignments at a time and finds each one's rank among those of the same
// expert from ballots over the id's bits, so no atomic's order has a say in the result.
#include <algorithm>
#include <type_traits>

#include "byhip_mx.h"

namespace byhip {
namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;
    size_t stride;
    int T, E, k, score, groups, top_groups, group_by, renorm, vec;
    float scale;
    int* ids;
    float* weights;
};

// fp32 in an order of whole numbers: every number and infinity above 1, NaN 1, and 0 left for what is no choice.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 as 0
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// Orders a wave's LDS accesses: what its lanes wrote before is what its lanes read after.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The value that order_key made a key of (NaN: minus infinity).
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k <= 1u) return -INFINITY;
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The largest of the lanes' values, all in DPP (a shuffle through LDS would cost ten times the latency).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    auto step = [&](auto ctrl, auto mask) { v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(mask)::value, 0xF, false)); };
    typedef std::integral_constant<int, 0xF> All;
    step(std::integral_constant<int, 0xB1>{}, All{});   // quad_perm [1,0,3,2]
    step(std::integral_constant<int, 0x4E>{}, All{});   // quad_perm [2,3,0,1]
    step(std::integral_constant<int, 0x141>{}, All{});  // row_half_mirror
    step(std::integral_constant<int, 0x140>{}, All{});  // row_mirror
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15 into rows 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31 into rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float lane_sum(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_lane63(v)), 63));
}
__device__ __forceinline__ double wave_sumd(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double lane_d(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// 1 / y for y >= 1 (also infinity and NaN), within an ulp or two: the hardware's estimate and two steps of Newton's.
__device__ __forceinline__ double reciprocal(double y) {
    double r = __builtin_amdgcn_rcp(y);
    r = fma(r, fma(-y, r, 1.0), r);
    r = fma(r, fma(-y, r, 1.0), r);
    return y == (double)INFINITY ? 0.0 : r;
}

// The two largest of a and b, given those of two sets.
struct Two {
    double one, two;
};
__device__ __forceinline__ Two merge(Two a, Two b) {
    const bool over = b.one > a.one;
    const double low = over ? a.one : b.one, first = over ? b.one : a.one, second = b.two > a.two ? b.two : a.two;
    return Two{first, low > second ? low : second};
}
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ Two dpp_two(Two v) { return Two{dpp_d<CTRL>(v.one), dpp_d<CTRL>(v.two)}; }

// What a group's two largest keys make it worth: their sum that is no number (infinities of both signs) comes last, as such keys do.
__device__ __forceinline__ double group_worth(const RouteArgs& a, int size, double one, double two) {
    const double sum = a.group_by == 2 && size > 1 ? one + two : one;
    return sum == sum ? sum : -(double)INFINITY;
}

// The choices of token t by this wave. WIDE: keys in 64 bits (`group` holds E of them in LDS where groups are ranked).
template <int DT, int V, bool WIDE>
__device__ __forceinline__ void route_token(const RouteArgs& a, int t, double* group) {
    const int lane = threadIdx.x & 63, e0 = lane * V;
    const size_t row = (size_t)t * a.stride;
    float x[V];
    if (a.vec && V >= 4 && e0 + V <= a.E) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float four[4];
            load_vec<DT, 4>(a.logits, row + e0 + i, four);
#pragma unroll
            for (int q = 0; q < 4 && i + q < V; ++q) x[i + q] = four[q];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = e0 + i < a.E ? load1<DT>(a.logits, row + e0 + i) : -INFINITY;
    }
    // Softmax: exp(x - top) / sum. A logit of +infinity leaves weight to its like only; where all are -infinity, none has any.
    float top = 0.0f, sum = 1.0f;
    double sum_d = 1.0;
    const bool soft = a.score == BYHIP_MOE_SOFTMAX;
    bool nan_row = false;  // a softmax over a NaN
    auto lift = [&](float v) { return v == top ? 0.0f : v - top; };
    if (soft) {
        uint32_t most = 0;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            most = max(most, order_key(x[i]));
            nan = nan || x[i] != x[i];
        }
        top = key_value(wave_max(most));
        nan_row = __any(nan);
        if (WIDE || !a.renorm) {  // (it falls out of renormalised weights)
            float s = 0.0f;
            double sd = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (e0 + i >= a.E) continue;
                if constexpr (WIDE) sd += exp((double)(x[i] == top ? 0.0 : (double)x[i] - (double)top));
                else s += expf(lift(x[i]));
            }
            if constexpr (WIDE) { sum_d = wave_sumd(sd); sum = (float)sum_d; }
            else sum = lane_sum(s);
        }
        if (top == -INFINITY && !nan_row) { sum = INFINITY; sum_d = (double)INFINITY; }
    }
    auto score_f = [&](float v) { return soft ? expf(lift(v)) / sum : 1.0f / (1.0f + expf(-v)); };
    const double over_sum = soft ? 1.0 / sum_d : 1.0;
    auto score_d = [&](float v) {
        return soft ? exp(v == top ? 0.0 : (double)v - (double)top) * over_sum : reciprocal(1.0 + exp(-(double)v));
    };

    uint32_t key[V];
    double wide[WIDE ? V : 1];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (WIDE) {
            double c = -(double)INFINITY;
            if (e0 + i < a.E) c = score_d(x[i]) + (a.bias ? (double)a.bias[e0 + i] : 0.0);
            wide[i] = c;
            key[i] = e0 + i < a.E ? order_key(a.bias ? (float)c : x[i]) : 0u;
        } else {
            key[i] = e0 + i < a.E ? order_key(x[i]) : 0u;
        }
    }
    if (a.groups > 1) {
        const int size = a.E / a.groups;
        uint64_t in = 0;  // the groups that take part
        bool mine_in = false;
        const int span = size / V;  // lanes per group where they are whole
        if constexpr (WIDE) {
            const double none = -(double)INFINITY;
            if (span * V == size && (span & (span - 1)) == 0 && span <= 16) {
                // The lane's two best, then those of its neighbours of the group: 1, 2, 4, 8 lanes on. (By one lane per group from LDS: 23.4 us for
                // 19.4, 8191 tokens, 8 groups of 32.)
                Two best{none, none};
#pragma unroll
                for (int i = 0; i < V; ++i) best = merge(best, Two{wide[i] == wide[i] ? wide[i] : none, none});
                if (span > 1) best = merge(best, dpp_two<0xB1>(best));
                if (span > 2) best = merge(best, dpp_two<0x4E>(best));
                if (span > 4) best = merge(best, dpp_two<0x141>(best));
                if (span > 8) best = merge(best, dpp_two<0x140>(best));
                const double worth = group_worth(a, size, best.one, best.two);
                const int own = lane / span;
                int above = 0;
                for (int g = 0; g < a.groups; ++g) {
                    const double o = lane_d(worth, g * span);
                    above += o > worth || (o == worth && g < own);
                }
                mine_in = above < a.top_groups;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (e0 + i < a.E) group[e0 + i] = wide[i] == wide[i] ? wide[i] : none;
                wave_sync();
                double one = none, two = none;
                if (lane < a.groups)
                    for (int i = 0; i < size; ++i) {
                        const double c = group[lane * size + i];
                        if (c > one) { two = one; one = c; }
                        else if (c > two) two = c;
                    }
                const double worth = group_worth(a, size, one, two);
                int above = 0;
                for (int g = 0; g < a.groups; ++g) {
                    const double o = lane_d(worth, g);
                    above += o > worth || (o == worth && g < lane);
                }
                in = __ballot(lane < a.groups && above < a.top_groups);
                wave_sync();
            }
        } else {
            uint32_t* keys = reinterpret_cast<uint32_t*>(group);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (e0 + i < a.E) keys[e0 + i] = key[i];
            wave_sync();
            uint32_t worth = 0;
            if (lane < a.groups)
                for (int i = 0; i < size; ++i) worth = max(worth, keys[lane * size + i]);
            int above = 0;
            for (int g = 0; g < a.groups; ++g) {
                const uint32_t o = __builtin_amdgcn_readlane((int)worth, g);
                above += o > worth || (o == worth && g < lane);
            }
            in = __ballot(lane < a.groups && above < a.top_groups);
            wave_sync();
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i >= a.E || !(mine_in || ((in >> ((e0 + i) / size)) & 1))) key[i] = 0u;
    }
    // Rounds: the largest head; of several, in 64 bits the largest, then the lowest index (the lowest lane).
    int mine_id = 0;
    uint32_t head = 0;
    double head_wide = 0.0;
    int at = 0;
    auto find_head = [&] {
        head = key[0];
        at = 0;
        if constexpr (WIDE) head_wide = wide[0];
#pragma unroll
        for (int i = 1; i < V; ++i) {
            bool over = key[i] > head;
            if constexpr (WIDE) over = over || (key[i] == head && wide[i] > head_wide);
            head = over ? key[i] : head;
            at = over ? i : at;
            if constexpr (WIDE) head_wide = over ? wide[i] : head_wide;
        }
    };
    find_head();
    for (int j = 0; j < a.k; ++j) {
        const uint32_t best = wave_max(head);
        uint64_t who = __ballot(head == best);
        if constexpr (WIDE) {
            if (a.bias && __popcll(who) > 1 && best > 1u) {
                const double c = head == best ? head_wide : -(double)INFINITY;
                double m = c;
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o));
                who = __ballot(head == best && c == m);
            }
        }
        const int win = __ffsll((unsigned long long)who) - 1;
        const int pick = __builtin_amdgcn_readlane(at, win);
        if (lane == (j & 63)) mine_id = win * V + pick;
        if (lane == win) {
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = i == pick ? 0u : key[i];
            find_head();
        }
        // 64 choices at most are held.
        if ((j & 63) == 63 || j + 1 == a.k) {
            const int i = (j & ~63) + lane;
            if (i <= j) {
                a.ids[(size_t)t * a.k + i] = mine_id;
                if (!a.renorm) {
                    const float v = load1<DT>(a.logits, row + mine_id);
                    float s;
                    if constexpr (WIDE) s = (float)score_d(v);
                    else s = score_f(v);
                    a.weights[(size_t)t * a.k + i] = s * a.scale;
                }
            }
        }
    }
    if (!a.renorm) return;
    // Renormalised: scores of any size over their sum. They are taken relative to e^ref, ref the largest chosen logit (of a sigmoid where that is below 0), so
    // that the largest is 1/2 or more and neither it nor the sum vanishes where every score does in 32 bits.
    float v[4];  // choices lane, lane + 64, ..
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        v[c] = -INFINITY;
        const int i = 64 * c + lane;
        if (64 * c < a.k && i < a.k) {
            v[c] = load1<DT>(a.logits, row + (a.k <= 64 ? mine_id : a.ids[(size_t)t * a.k + i]));
            most = max(most, order_key(v[c]));
        }
    }
    const float largest = key_value(wave_max(most)), ref = soft ? largest : fminf(largest, 0.0f);
    auto share = [&](float x) {
        if constexpr (WIDE) {
            const double e = x == ref ? 0.0 : (double)x - (double)ref;
            return (float)(soft ? exp(e) : ref < 0.0f ? exp(e) * reciprocal(1.0 + exp((double)x)) : reciprocal(1.0 + exp(-(double)x)));
        } else {
            const float e = x == ref ? 0.0f : x - ref;
            return soft ? expf(e) : ref < 0.0f ? expf(e) / (1.0f + expf(x)) : 1.0f / (1.0f + expf(-x));
        }
    };
    float total = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (64 * c < a.k && 64 * c + lane < a.k) {
            v[c] = share(v[c]);
            total += v[c];
        }
    total = nan_row ? NAN : lane_sum(total);
    // Below e^-708 a score is taken for 0 (64-bit numbers end there), and so are the weights where all are.
    const float above = soft && largest != -INFINITY ? (largest == top ? 0.0f : largest - top) : largest;
    const float f = total != total ? total : above < -708.0f ? 0.0f : a.scale / total;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (64 * c < a.k && 64 * c + lane < a.k) a.weights[(size_t)t * a.k + 64 * c + lane] = v[c] * f;
}

constexpr int kTokensPerBlock = 4;

template <int DT, int V, bool WIDE>
__global__ __launch_bounds__(64 * kTokensPerBlock) void moe_route(RouteArgs a) {
    __shared__ double group[kTokensPerBlock][WIDE ? 64 * V : 32 * V];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.x * kTokensPerBlock + w;
    if (t >= a.T) return;
    route_token<DT, V, WIDE>(a, t, group[w]);
}

// ── the plan ──

// The `live` lanes whose id (below kMaxExperts) is this lane's.
__device__ __forceinline__ uint64_t same_id(int id, bool live) {
    uint64_t m = __ballot(live);
#pragma unroll
    for (int b = 0; 1 << b < kMaxExperts; ++b) {
        const bool bit = (id >> b) & 1;
        const uint64_t set = __ballot(bit);
        m &= bit ? set : ~set;
    }
    return m;
}
// How many of these lanes are below this one.
__device__ __forceinline__ int rank_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// Assignments lo .. hi - 1 in `waves` equal stretches of whole 64s; this wave's.
__device__ __forceinline__ void stretch(int lo, int hi, int waves, int w, int& from, int& to) {
    const int each = ((hi - lo + waves - 1) / waves + 63) & ~63;
    from = min(hi, lo + each * w);
    to = min(hi, from + each);
}

// How many assignments of its stretch each expert gets, added to the wave's counts.
__device__ __forceinline__ void count_ids(const int* ids, int from, int to, int E, int* counts) {
    const int lane = threadIdx.x & 63;
    for (int i = from + lane; i < to; i += 64) {
        const int id = ids[i];
        if ((unsigned)id < (unsigned)E) atomicAdd(&counts[id], 1);
    }
}

// Places the stretch's assignments: next[e] is where the wave's next assignment of expert e goes.
__device__ __forceinline__ void place_ids(const int* ids, int from, int to, int E, int* next, int* order) {
    const int lane = threadIdx.x & 63;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        int id = i < to ? ids[i] : -1;
        const bool live = (unsigned)id < (unsigned)E;
        id = live ? id : 0;
        const uint64_t peers = same_id(id, live);
        const int rank = rank_below(peers);
        if (live) order[next[id] + rank] = i;
        wave_sync();
        if (live && rank == 0) next[id] += __popcll(peers);
        wave_sync();
    }
}

// Inclusive prefix sums over the lanes, in DPP: within rows of 16 lanes, then across rows.
__device__ __forceinline__ int lane_prefix(int v) {
    auto step = [&](auto ctrl, auto mask) { v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(mask)::value, 0xF, false); };
    typedef std::integral_constant<int, 0xF> All;
    step(std::integral_constant<int, 0x111>{}, All{});  // row_shr:1, 2, 4, 8
    step(std::integral_constant<int, 0x112>{}, All{});
    step(std::integral_constant<int, 0x114>{}, All{});
    step(std::integral_constant<int, 0x118>{}, All{});
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15 into rows 1 and 3
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31 into rows 2 and 3
    return v;
}

// Where expert e (thread e) starts, from its count (0 past E); with `write` also the offsets and the units. Three prefix sums in one go, over as many
// waves as hold experts; part: one per wave, where: one per expert.
__device__ __forceinline__ int expert_starts(const MoePlan& p, int count, int4* part, int4* where, bool write) {
    const int e = threadIdx.x, lane = e & 63, w = e >> 6, waves = (p.experts + 63) >> 6;
    const int units = (count + p.unit_rows - 1) / p.unit_rows, tiles = (count + kTileRows - 1) / kTileRows;
    const int c = lane_prefix(count), u = lane_prefix(units), t = lane_prefix(tiles);
    __syncthreads();
    if (lane == 63) part[w] = make_int4(c, u, t, 0);
    __syncthreads();
    int4 before = make_int4(0, 0, 0, 0), total = before;
    for (int i = 0; i < waves; ++i) {
        const int4 v = part[i];
        if (i < w) { before.x += v.x; before.y += v.y; before.z += v.z; }
        total.x += v.x; total.y += v.y; total.z += v.z;
    }
    const int at = before.x + c - count;
    if (!write) return at;
    auto unit = [&](int e, int at, int count, int rows, int i) { return MoeUnit{e, at + i * rows, min(rows, count - i * rows), 0}; };
    constexpr int kFew = 4;
    const int4 mine = make_int4(at, count, before.y + u - units, before.z + t - tiles);
    if (e < p.experts) {
        p.offsets[e] = at;
        where[e] = mine;
        for (int i = 0; i < min(units, kFew); ++i) p.units[mine.z + i] = unit(e, at, count, p.unit_rows, i);
        for (int i = 0; i < min(tiles, kFew); ++i) p.tiles[mine.w + i] = unit(e, at, count, kTileRows, i);
    }
    if (e == 0) {
        p.offsets[p.experts] = total.x;
        p.n_units[0] = total.y;
        p.n_units[1] = total.z;
    }
    // Experts of more units: a wave writes one's.
    if (__syncthreads_or(units > kFew)) {
        for (int x = w; x < p.experts; x += (int)blockDim.x >> 6) {
            const int4 s = where[x];
            for (int i = kFew + lane; i * p.unit_rows < s.y; i += 64) p.units[s.z + i] = unit(x, s.x, s.y, p.unit_rows, i);
            for (int i = kFew + lane; i * kTileRows < s.y; i += 64) p.tiles[s.w + i] = unit(x, s.x, s.y, kTileRows, i);
        }
    }
    return at;
}

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// The whole plan in one block: counts per wave and expert, their sums, then the places.
__device__ __forceinline__ void plan_block(const MoePlan& p, const int* ids, int* counts, int4* part, int4* where) {
    const int w = threadIdx.x >> 6, E = p.experts;
    for (int i = threadIdx.x; i < kPlanWaves * E; i += kPlanThreads) counts[i] = 0;
    __syncthreads();
    int from, to;
    stretch(0, p.rows, kPlanWaves, w, from, to);
    count_ids(ids, from, to, E, counts + w * E);
    __syncthreads();
    int sum = 0;
    if ((int)threadIdx.x < E)
        for (int i = 0; i < kPlanWaves; ++i) {
            const int c = counts[i * E + threadIdx.x];
            counts[i * E + threadIdx.x] = sum;
            sum += c;
        }
    const int at = expert_starts(p, sum, part, where, true);
    if ((int)threadIdx.x < E)
        for (int i = 0; i < kPlanWaves; ++i) counts[i * E + threadIdx.x] += at;
    __syncthreads();
    place_ids(ids, from, to, E, counts + w * E, p.order);
}

__global__ __launch_bounds__(kPlanThreads) void moe_plan_one(MoePlan p, const int* ids) {
    __shared__ int counts[kPlanWaves * kMaxExperts];
    __shared__ int4 part[kPlanWaves], where[kMaxExperts];
    plan_block(p, ids, counts, part, where);
}

// Many assignments: counts per block of them, then the places; with few counts every block of the second forms the sums it needs from all blocks' counts,
// which costs less than a launch between (kSumCounts).
constexpr int kCountWaves = 4;
__global__ __launch_bounds__(64 * kCountWaves) void moe_plan_count(MoePlan p, const int* ids) {
    __shared__ int counts[kMaxExperts];
    const int E = p.experts, lo = blockIdx.x * kPlanBlock, hi = min(p.rows, lo + kPlanBlock);
    for (int i = threadIdx.x; i < E; i += 64 * kCountWaves) counts[i] = 0;
    __syncthreads();
    int from, to;
    stretch(lo, hi, kCountWaves, threadIdx.x >> 6, from, to);
    count_ids(ids, from, to, E, counts);
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += 64 * kCountWaves) p.counts[(size_t)blockIdx.x * E + i] = counts[i];
}
// Many blocks of them: the counts become each block's first places among its experts' assignments, with all blocks' sums in a row behind them. 64 experts per block, a
// stretch of the counts' rows per wave.
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void moe_plan_sums(MoePlan p) {
    __shared__ int sums[kSumWaves][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, E = p.experts, e = blockIdx.x * 64 + lane;
    const int each = (p.blocks + kSumWaves - 1) / kSumWaves, lo = min(p.blocks, each * w), hi = min(p.blocks, lo + each);
    int* const counts = p.counts + (e < E ? e : 0);
    int sum = 0;
    if (e < E) {
#pragma unroll 8
        for (int b = lo; b < hi; ++b) sum += counts[(size_t)b * E];
    }
    sums[w][lane] = sum;
    __syncthreads();
    if (e >= E) return;
    int at = 0, total = 0;
    for (int i = 0; i < kSumWaves; ++i) {
        const int v = sums[i][lane];
        at += i < w ? v : 0;
        total += v;
    }
    if (w == 0) counts[(size_t)p.blocks * E] = total;
    for (int b = lo; b < hi; b += 8) {
        int c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = b + i < hi ? counts[(size_t)(b + i) * E] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (b + i < hi) counts[(size_t)(b + i) * E] = at;
            at += c[i];
        }
    }
}
template <bool SUMS>  // whether moe_plan_sums has run
__global__ __launch_bounds__(kPlanThreads) void moe_plan_place(MoePlan p, const int* ids) {
    __shared__ int counts[kCountWaves * kMaxExperts];
    __shared__ int2 sums[SUMS ? 1 : kPlanThreads];
    __shared__ int4 part[kPlanWaves], where[kMaxExperts];
    const int w = threadIdx.x >> 6, e = threadIdx.x, E = p.experts, lo = blockIdx.x * kPlanBlock, hi = min(p.rows, lo + kPlanBlock);
    int from = 0, to = 0;
    for (int i = threadIdx.x; i < kCountWaves * E; i += kPlanThreads) counts[i] = 0;
    // Expert e's assignments in all blocks, and in those before this one.
    int sum = 0, before = 0;
    if constexpr (SUMS) {
        if (e < E) {
            sum = p.counts[(size_t)p.blocks * E + e];
            before = p.counts[(size_t)blockIdx.x * E + e];
        }
    } else {  // as many threads per expert as there are, a share of the blocks each
        const int room = (E + 63) & ~63, shares = kPlanThreads / room, share = e / room;
        if (e - share * room < E && share < shares) {
#pragma unroll 8
            for (int b = share; b < p.blocks; b += shares) {
                const int c = p.counts[(size_t)b * E + e - share * room];
                sum += c;
                before += b < (int)blockIdx.x ? c : 0;
            }
        }
        sums[e] = make_int2(sum, before);
        __syncthreads();
        sum = before = 0;
        if (e < E)
            for (int i = 0; i < shares; ++i) {
                sum += sums[i * room + e].x;
                before += sums[i * room + e].y;
            }
    }
    __syncthreads();
    if (w < kCountWaves) {
        stretch(lo, hi, kCountWaves, w, from, to);
        count_ids(ids, from, to, E, counts + w * E);
    }
    int at = expert_starts(p, sum, part, where, blockIdx.x == 0);
    __syncthreads();
    if (e < E) {
        at += before;
        for (int i = 0; i < kCountWaves; ++i) {
            const int c = counts[i * E + e];
            counts[i * E + e] = at;
            at += c;
        }
    }
    __syncthreads();
    if (w < kCountWaves) place_ids(ids, from, to, E, counts + w * E, p.order);
}

// Up to this many counts (blocks times experts) every block sums them all, whose reads grow with the square of the assignments; beyond, a launch sums them once (us, 256 experts,
// 128 / 256 / 512 / 2048 blocks: 15.2 / 18.7 / 30.5 / 256 by every block, 16.5 / 18.6 / 22.1 / 54 once; 64 experts, 256 blocks 11.2 and 13.5; 1024 experts, 128
// blocks 28.4 and 23.5).
constexpr long long kSumCounts = 65536;
void launch_plan(const MoePlan& p, const int* ids) {
    if (p.blocks <= 4) {
        launch("moe_plan_one", moe_plan_one, dim3(1), dim3(kPlanThreads), 0, p, ids);
    } else {
        launch("moe_plan_count", moe_plan_count, dim3(p.blocks), dim3(64 * kCountWaves), 0, p, ids);
        if ((long long)p.blocks * p.experts <= kSumCounts) {
            launch("moe_plan_place", moe_plan_place<false>, dim3(p.blocks), dim3(kPlanThreads), 0, p, ids);
        } else {
            launch("moe_plan_sums", moe_plan_sums, dim3((p.experts + 63) / 64), dim3(64 * kSumWaves), 0, p);
            launch("moe_plan_place", moe_plan_place<true>, dim3(p.blocks), dim3(kPlanThreads), 0, p, ids);
        }
    }
    BYHIP_LAUNCHED("moe_plan");
}

template <int DT, int V, bool WIDE>
void launch_route_v(const RouteArgs& a, const MoePlan& p) {
    // (A decode step's tokens and their plan in one block and one launch took longer: 12.4 us for 32 tokens of 128 experts, one CU's work,
    // where the two launches take 8.)
    launch("moe_route", (moe_route<DT, V, WIDE>), dim3((a.T + kTokensPerBlock - 1) / kTokensPerBlock), dim3(64 * kTokensPerBlock), 0, a);
    BYHIP_LAUNCHED("moe_route");
    launch_plan(p, a.ids);
}
template <int DT, bool WIDE>
void launch_route_w(const RouteArgs& a, const MoePlan& p) {
    if (a.E <= 64) launch_route_v<DT, 1, WIDE>(a, p);
    else if (a.E <= 128) launch_route_v<DT, 2, WIDE>(a, p);
    else if (a.E <= 256) launch_route_v<DT, 4, WIDE>(a, p);
    else if (a.E <= 512) launch_route_v<DT, 8, WIDE>(a, p);
    else launch_route_v<DT, 16, WIDE>(a, p);
}
template <int DT>
void launch_route(const RouteArgs& a, const MoePlan& p) {
    // Without a bias, and with groups ranked by one key, the logits have the keys' order.
    if (a.bias || (a.groups > 1 && a.group_by == 2)) launch_route_w<DT, true>(a, p);
    else launch_route_w<DT, false>(a, p);
}

// ── the sum of a token's rows ──

struct CombineArgs {
    const void* x;
    const int* ids;
    const float* weights;
    const void* res;
    void* y;
    size_t x_stride, res_stride, y_stride;
    int T, k, E, N, res_dtype, y_dtype, vec;
};

template <int DT, int W>
__device__ __forceinline__ void read_cols(const void* p, size_t at, int left, int vec, float (&v)[W]) {
#pragma unroll
    for (int q = 0; q < W; q += 4) {
        float four[4];
        if (vec && left >= W) {
            load_vec<DT, 4>(p, at + q, four);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) four[e] = q + e < left ? load1<DT>(p, at + q + e) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q + e] = four[e];
    }
}

// W columns per thread: 16 bytes of a row where it is aligned so.
template <int XT, int W>
__global__ __launch_bounds__(256) void moe_combine(CombineArgs a) {
    const int n = W * (blockIdx.x * 256 + threadIdx.x), left = a.N - n;
    if (left <= 0) return;
    for (int t = blockIdx.y; t < a.T; t += gridDim.y) {
        float s[W];
#pragma unroll
        for (int e = 0; e < W; ++e) s[e] = 0.0f;
        if (a.res) {
            const size_t at = (size_t)t * a.res_stride + n;
            if (a.res_dtype == BYHIP_F32) read_cols<BYHIP_F32, W>(a.res, at, left, a.vec, s);
            else if (a.res_dtype == BYHIP_F16) read_cols<BYHIP_F16, W>(a.res, at, left, a.vec, s);
            else read_cols<BYHIP_BF16, W>(a.res, at, left, a.vec, s);
        }
        // Four rows' loads at a time, then their sums.
        const size_t first = (size_t)t * a.k;
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            float w[4], v[4][W];
            bool live[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                live[j] = j0 + j < a.k && (unsigned)a.ids[first + min(j0 + j, a.k - 1)] < (unsigned)a.E;
                w[j] = a.weights[first + min(j0 + j, a.k - 1)];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (live[j]) read_cols<XT, W>(a.x, (first + j0 + j) * a.x_stride + n, left, a.vec, v[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < W; ++e) s[e] = live[j] ? fmaf(w[j], v[j][e], s[e]) : s[e];
        }
        const size_t at = (size_t)t * a.y_stride + n;
#pragma unroll
        for (int q = 0; q < W; q += 4) {
            const float four[4] = {s[q], s[q + 1], s[q + 2], s[q + 3]};
            if (a.vec && left >= W) {
                store_vec<4>(a.y, at + q, four, a.y_dtype);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (q + e < left) {
                        const float one[1] = {four[e]};
                        store_vec<1>(a.y, at + q + e, one, a.y_dtype);
                    }
            }
        }
    }
}

}  // namespace

MoePlan moe_layout(const byhip_moe_plan* p) {
    if (!p) fail("byhip: null plan");
    if (p->tokens < 0 || p->experts < 1 || p->experts > kMaxExperts || p->top_k < 1 || p->top_k > p->experts || p->top_k > 256 ||
        (long long)p->tokens * p->top_k >= 1 << 24)
        fail("byhip: a plan of %d tokens, %d of %d experts each", p->tokens, p->top_k, p->experts);
    MoePlan m{};
    m.tokens = p->tokens; m.top_k = p->top_k; m.experts = p->experts;
    m.rows = p->tokens * p->top_k;
    m.unit_rows = moe_unit_rows(m.rows, m.experts);
    m.max_units = moe_max_units(m.rows, m.experts, m.unit_rows);
    m.max_tiles = moe_max_units(m.rows, m.experts, kTileRows);
    m.blocks = (m.rows + kPlanBlock - 1) / kPlanBlock;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 15) / 16 * 16; return static_cast<char*>(p->plan) + here; };
    m.offsets = reinterpret_cast<int*>(take(((size_t)m.experts + 1 + m.rows) * 4));
    m.order = m.offsets + m.experts + 1;
    m.n_units = reinterpret_cast<int*>(take(8));
    m.units = reinterpret_cast<MoeUnit*>(take((size_t)m.max_units * sizeof(MoeUnit)));
    m.tiles = reinterpret_cast<MoeUnit*>(take((size_t)m.max_tiles * sizeof(MoeUnit)));
    m.counts = reinterpret_cast<int*>(take((size_t)(m.blocks + 1) * m.experts * 4));
    m.bytes = at;
    return m;
}

MoePlan moe_plan_args(const byhip_moe_plan* p) {
    const MoePlan m = moe_layout(p);
    check_span(p->plan, m.bytes, "plan");
    if (reinterpret_cast<uintptr_t>(p->plan) % 16) fail("byhip: a plan must be 16-byte aligned");
    return m;
}

}  // namespace byhip

using namespace byhip;

extern "C" {

unsigned long long byhip_moe_plan_bytes(int tokens, int top_k, int experts) {
    unsigned long long bytes = 0;
    guard([&] {
        const byhip_moe_plan p{tokens, top_k, experts, nullptr};
        bytes = moe_layout(&p).bytes;
    });
    return bytes;
}

int byhip_moe_route(const void* logits, size_t stride, int dtype, const byhip_moe_router* router, const byhip_moe_plan* plan,
                    int* ids, float* weights) {
    return guard([&] {
        enter_compute();
        const MoePlan p = moe_plan_args(plan);
        if (!router) fail("byhip: null router");
        const byhip_moe_router& r = *router;
        if (r.score != BYHIP_MOE_SOFTMAX && r.score != BYHIP_MOE_SIGMOID) fail("byhip: router score %d", r.score);
        if (r.groups < 1 || r.groups > 64 || p.experts % r.groups || r.top_groups < 1 || r.top_groups > r.groups)
            fail("byhip: the best %d of %d groups of %d experts", r.top_groups, r.groups, p.experts);
        if (r.groups > 1 && r.group_by != 1 && r.group_by != 2) fail("byhip: groups by their %d best", r.group_by);
        if (p.top_k > p.experts / r.groups * r.top_groups)
            fail("byhip: %d choices among %d experts", p.top_k, p.experts / r.groups * r.top_groups);
        check_rows(logits, p.tokens, p.experts, stride, dtype, "logits");
        if (r.bias) check_span(r.bias, (size_t)p.experts * 4, "router bias");
        if (p.rows) {
            check_span(ids, (size_t)p.rows * 4, "ids");
            check_span(weights, (size_t)p.rows * 4, "weights");
        }
        note_device_write(plan->plan);
        if (p.rows) {
            note_device_write(ids);
            note_device_write(weights);
            const RouteArgs a{logits, r.bias, stride, p.tokens, p.experts, p.top_k, r.score, r.groups, r.top_groups,
                              r.group_by, r.renorm, aligned4(logits, stride, dtype), r.scale, ids, weights};
            switch (dtype) {
            case BYHIP_F32: launch_route<BYHIP_F32>(a, p); break;
            case BYHIP_F16: launch_route<BYHIP_F16>(a, p); break;
            default: launch_route<BYHIP_BF16>(a, p); break;
            }
        } else {
            launch_plan(p, ids);
        }
    });
}

int byhip_moe_plan_ids(const int* ids, const byhip_moe_plan* plan) {
    return guard([&] {
        enter_compute();
        const MoePlan p = moe_plan_args(plan);
        if (p.rows) check_span(ids, (size_t)p.rows * 4, "ids");
        note_device_write(plan->plan);
        launch_plan(p, ids);
    });
}

int byhip_moe_combine(const void* x, size_t x_stride, int x_dtype, int N, const byhip_moe_plan* plan, const int* ids,
                      const float* weights, const void* res, size_t res_stride, int res_dtype, void* y, size_t y_stride,
                      int y_dtype) {
    return guard([&] {
        enter_compute();
        const MoePlan p = moe_layout(plan);
        if (N <= 0) fail("byhip: a sum of rows of %d values", N);
        check_rows(x, p.rows, N, x_stride, x_dtype, "experts' rows");
        if (res) check_rows(res, p.tokens, N, res_stride, res_dtype, "residual");
        check_rows(y, p.tokens, N, y_stride, y_dtype, "summed rows");
        if (res == y && res && (res_stride != y_stride || res_dtype != y_dtype)) fail("byhip: a residual updated in place needs one stride and dtype");
        if (p.rows == 0) return;
        check_span(ids, (size_t)p.rows * 4, "ids");
        check_span(weights, (size_t)p.rows * 4, "weights");
        const int vec = aligned4(x, x_stride, x_dtype) && (!res || aligned4(res, res_stride, res_dtype)) && aligned4(y, y_stride, y_dtype);
        const CombineArgs a{x, ids, weights, res, y, x_stride, res_stride, y_stride, p.tokens, p.top_k, p.experts, N, res_dtype, y_dtype, vec};
        note_device_write(y);
        const unsigned blocks = std::min(p.tokens, 65535);
        const dim3 four((N + 1023) / 1024, blocks), eight((N + 2047) / 2048, blocks);
        switch (x_dtype) {
        case BYHIP_F32: launch("moe_combine", (moe_combine<BYHIP_F32, 4>), four, dim3(256), 0, a); break;
        case BYHIP_F16: launch("moe_combine", (moe_combine<BYHIP_F16, 8>), eight, dim3(256), 0, a); break;
        default: launch("moe_combine", (moe_combine<BYHIP_BF16, 8>), eight, dim3(256), 0, a); break;
        }
        BYHIP_LAUNCHED("moe_combine");
    });
}

}  // extern "C"
