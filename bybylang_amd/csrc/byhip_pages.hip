// byhip_pages.hip - pages of a cache pool: fork, free, grow (with copy on write), compaction and copies
// (gfx950).
//
// Page tables, reference counts and lengths stay on the device, so these calls queue like any kernel, with no
// host round trip, and can be recorded. What has to be decided in order (which free page goes to whom, which
// of several sharers keeps a page) is decided by one block with prefix sums, so the outcome never depends on
// scheduling; the bytes then move in one copy kernel over all layers, at the rate of a plain copy (841 MB of live pages
// in 163 us, 5.2 TB/s; the planning blocks 8 to 10 us, a chain of reads and prefix sums; a grow of many slots, which
// compares them in pairs, 11 us for 64, 23 for 256, 80 for 1024).
#include <algorithm>

#include "byhip_cache.h"

namespace byhip {
namespace {

constexpr int kMaxRows = 1024;   // slots per call: one thread each in the planning block
constexpr int kLayersPerLaunch = 64;
constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 8;    // reference counts a planning thread looks at per turn

struct PoolArgs {
    int* refs;
    int* table;
    int* lens;
    int* status;
    int* granted;
    int slots, stride, pages, page_size;
};

// Lists the planning block leaves for the copy kernel: a count, then `room` sources and `room` destinations.
struct MoveList {
    int* count;
    int* src;
    int* dst;
};

__device__ __forceinline__ int pages_of(int tokens, int page_size) {
    return tokens <= 0 ? 0 : (int)(((long long)tokens + page_size - 1) / page_size);
}

// Exclusive prefix sum over the block's threads; the total in every thread. `red`: one value per wave.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* red, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T u = __shfl_up(s, o, 64);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        before += w < wave ? red[w] : 0;
        total += red[w];
    }
    return before + s - v;
}

// Slot rows[i] takes over parents[i]'s pages (parents null: none). A slot's pages are those its tokens
// need; entries past them are not looked at and become -1.
__global__ __launch_bounds__(256) void cache_assign(PoolArgs p, const int* parents, const int* rows, int n) {
    const int i = blockIdx.x, row = rows[i];
    const int parent = parents ? parents[i] : -1;
    bool bad = row < 0 || row >= p.slots || (parents && (parent < 0 || parent >= p.slots));
    for (int j = threadIdx.x; j < n; j += 256) {
        const int other = rows[j];
        bad = bad || (j < i && other == row) || (parents && other == parent);
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicAdd(&p.status[1], 1);
        return;
    }
    const int had = min(pages_of(p.lens[row], p.page_size), p.stride);
    const int len = parents ? p.lens[parent] : 0;
    const int gets = min(pages_of(len, p.page_size), p.stride);
    int* mine = p.table + (size_t)row * p.stride;
    const int* from = p.table + (size_t)(parents ? parent : row) * p.stride;
    for (int c = threadIdx.x; c < p.stride; c += 256) {
        const int old = c < had ? mine[c] : -1, now = c < gets ? from[c] : -1;
        if (old >= 0 && old < p.pages) atomicSub(&p.refs[old], 1);
        if (now >= 0 && now < p.pages) atomicAdd(&p.refs[now], 1);
        mine[c] = now;
    }
    __syncthreads();  // every thread has read the old length
    if (threadIdx.x == 0) p.lens[row] = len < 0 ? 0 : len;
}

// One block: room for add[i] more tokens in slot rows[i].
__global__ __launch_bounds__(kPlanThreads) void cache_grow_plan(PoolArgs p, const int* rows, const int* add, int n, int* free_list,
                                                                MoveList copies) {
    __shared__ int row_of[kMaxRows], last_of[kMaxRows], first_of[kMaxRows], sum_before[kMaxRows + 1];
    __shared__ int red[kPlanThreads / 64];
    __shared__ unsigned long long red_counts[kPlanThreads / 64];
    const int i = threadIdx.x;
    const int row = i < n ? rows[i] : -1, more = i < n ? add[i] : 0;
    row_of[i] = row;
    __syncthreads();
    // 1. what slot i wants
    bool bad = row < 0 || row >= p.slots;
    for (int j = 0; j < i && j < n; ++j) bad = bad || row_of[j] == row;
    bad = bad || i >= n;
    const int have = bad ? 0 : max(0, p.lens[row]);
    const long long want = (long long)have + more;
    int* mine = p.table + (size_t)(bad ? 0 : row) * p.stride;
    const bool too_long = !bad && more > 0 && want > min((long long)p.stride * p.page_size, 0x7FFFFFFFLL);
    const bool grows = !bad && !too_long && more > 0;
    int last = -1;  // the partly filled page it would append to
    if (grows && have % p.page_size) last = mine[have / p.page_size];
    if (last >= p.pages) last = -1;
    last_of[i] = last;
    __syncthreads();
    // 2. copy on write: of the slots that append to one page in this call, each copies unless it is the
    // page's last holder once those before it have theirs
    bool copy = false;
    if (last >= 0) {
        int before = 0;
        for (int j = 0; j < i; ++j) before += last_of[j] == last;
        copy = p.refs[last] - before > 1;
    }
    const int first = pages_of(have, p.page_size) - (copy ? 1 : 0);
    const int need = grows ? pages_of((int)want, p.page_size) - first : 0;
    int total;
    const int before = block_prefix(need, red, total);
    sum_before[i] = before;
    first_of[i] = first;
    if (i == 0) sum_before[kMaxRows] = total;
    // 3. the lowest `total` free pages, in order
    int found = 0;
    for (int base = 0; base < p.pages && found < total; base += kPlanThreads * kPerThread) {
        const int at = base + i * kPerThread;
        unsigned mask = 0;
#pragma unroll
        for (int e = 0; e < kPerThread; ++e)
            if (at + e < p.pages && p.refs[at + e] <= 0) mask |= 1u << e;
        int here;
        int rank = found + block_prefix((int)__popc(mask), red, here);
#pragma unroll
        for (int e = 0; e < kPerThread; ++e)
            if (mask >> e & 1) {
                if (rank < total) free_list[rank] = at + e;
                ++rank;
            }
        found += here;
    }
    // 4. slots are served up to the first that does not fit
    const bool served = grows && before + need <= found, refused = too_long || (grows && !served);
    __threadfence_block();
    // one sum for all counts: copies, refused and bad slots (11 bits each), pages taken (31)
    unsigned long long counts;
    const unsigned long long mine_before = block_prefix(
        (unsigned long long)(served && copy) | (unsigned long long)refused << 11 | (unsigned long long)(bad && i < n) << 22 |
            (unsigned long long)(served ? need : 0) << 33, red_counts, counts);
    const int copied = (int)(counts & 2047), n_refused = (int)(counts >> 11 & 2047), n_bad = (int)(counts >> 22 & 2047), taken = (int)(counts >> 33);
    for (int k = i; k < taken; k += kPlanThreads) {
        int lo = 0, hi = n - 1;  // the last slot whose sum before it is <= k and that takes pages
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (sum_before[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        const int page = free_list[k];
        const int col = first_of[lo] + (k - sum_before[lo]);
        p.table[(size_t)row_of[lo] * p.stride + col] = page;
        p.refs[page] = 1;
    }
    const int slot = (int)(mine_before & 2047);
    if (served && copy) {
        copies.src[slot] = last;
        copies.dst[slot] = free_list[before];
        atomicSub(&p.refs[last], 1);
    }
    if (served) p.lens[row] = (int)want;
    if (p.granted && !bad) p.granted[row] = served ? more : 0;
    // 5. slots that shrink release the pages past their new end
    if (!bad && more < 0) {
        const int keep = want < 0 ? 0 : (int)want;
        const int end = min(pages_of(have, p.page_size), p.stride);
        for (int c = pages_of(keep, p.page_size); c < end; ++c) {
            const int page = mine[c];
            if (page >= 0 && page < p.pages) atomicSub(&p.refs[page], 1);
            mine[c] = -1;
        }
        p.lens[row] = keep;
    }
    if (i == 0) {
        *copies.count = copied;
        if (n_refused) atomicAdd(&p.status[0], n_refused);
        if (n_bad) atomicAdd(&p.status[1], n_bad);
        if (copied) atomicAdd(&p.status[2], copied);
        if (taken) atomicAdd(&p.status[3], taken);
    }
}

// One block: the moves that bring all live pages to the front, the new reference counts and each page's new
// place.
__global__ __launch_bounds__(kPlanThreads) void cache_compact_plan(PoolArgs p, int* refs_out, int* remap, MoveList moves) {
    __shared__ int red[kPlanThreads / 64];
    const int i = threadIdx.x;
    int live = 0, holes = 0, movers = 0, total;
    for (int at = i; at < p.pages; at += kPlanThreads) live += p.refs[at] > 0;
    block_prefix(live, red, total);
    live = total;
    for (int base = 0; base < p.pages; base += kPlanThreads * kPerThread) {
        const int at = base + i * kPerThread;
        unsigned hole = 0, mover = 0;
#pragma unroll
        for (int e = 0; e < kPerThread; ++e)
            if (at + e < p.pages) {
                const int r = p.refs[at + e];
                if (at + e < live && r <= 0) hole |= 1u << e;
                if (at + e >= live && r > 0) mover |= 1u << e;
                remap[at + e] = at + e;
                if (refs_out != p.refs) refs_out[at + e] = r;
            }
        int both;  // a turn has at most 8192 of each: one sum for the two
        const int before = block_prefix((int)(__popc(hole) | __popc(mover) << 16), red, both);
        int hr = holes + (before & 0xFFFF), mr = movers + (before >> 16);
#pragma unroll
        for (int e = 0; e < kPerThread; ++e) {
            if (hole >> e & 1) moves.dst[hr++] = at + e;
            if (mover >> e & 1) moves.src[mr++] = at + e;
        }
        holes += both & 0xFFFF;
        movers += both >> 16;
    }
    __threadfence_block();
    __syncthreads();
    for (int k = i; k < movers; k += kPlanThreads) {
        const int src = moves.src[k], dst = moves.dst[k];
        remap[src] = dst;
        const int r = p.refs[src];
        refs_out[dst] = r;
        refs_out[src] = 0;
    }
    if (i == 0) {
        *moves.count = movers;
        if (movers) atomicAdd(&p.status[2], movers);
    }
}

// What the copy kernel does besides: tables follow their pages.
struct RemapArgs {
    const int* remap;
    const int* table;
    int* out;
    size_t entries;
    int blocks, pages;
};

struct CopyArgs {
    char* base[2 * kLayersPerLaunch];  // keys and values of each layer
    int bases, pages;
    size_t page_bytes;
    const int* src;
    const int* dst;
    const int* count;  // null: n
    int n;
};

constexpr size_t kPiece = 16384;  // bytes a block moves at a time

// T: the unit of a copy, 16 bytes where pages and buffers allow it, else 2.
template <typename T>
__global__ __launch_bounds__(256) void cache_copy(CopyArgs a, RemapArgs r) {
    if ((int)blockIdx.x < r.blocks) {
        for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < r.entries; e += (size_t)r.blocks * 256) {
            const int page = r.table[e];
            r.out[e] = page >= 0 && page < r.pages ? r.remap[page] : page;
        }
        return;
    }
    const int n = a.count ? min(*a.count, a.n) : a.n;
    const size_t pieces = (a.page_bytes + kPiece - 1) / kPiece;
    const size_t units = (size_t)n * a.bases * pieces;
    for (size_t u = blockIdx.x - r.blocks; u < units; u += gridDim.x - r.blocks) {
        const size_t piece = u % pieces, w = u / pieces;
        const int layer = (int)(w % a.bases), k = (int)(w / a.bases);
        const int src = a.src[k], dst = a.dst[k];
        if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages || src == dst) continue;
        const size_t off = piece * kPiece, bytes = min(kPiece, a.page_bytes - off);
        const T* s = reinterpret_cast<const T*>(a.base[layer] + (size_t)src * a.page_bytes + off);
        T* d = reinterpret_cast<T*>(a.base[layer] + (size_t)dst * a.page_bytes + off);
        const int words = (int)(bytes / sizeof(T));
        for (int e = threadIdx.x; e < words; e += 256) d[e] = s[e];
    }
}

struct Pool {
    PoolArgs p;
    const byhip_kv_pool* c;
    size_t page_bytes;
    bool wide;  // 16-byte copies
};

Pool pool_args(const byhip_kv_pool* pool, bool needs_caches) {
    if (!pool) fail("byhip: null pool");
    if (pool->n_caches <= 0 || !pool->caches) fail("byhip: a pool without caches");
    if (pool->slots <= 0 || pool->table_stride <= 0) fail("byhip: pool of %d slots of %d pages", pool->slots, pool->table_stride);
    const byhip_kv_cache& first = pool->caches[0];
    Pool a;
    a.c = pool;
    a.wide = true;
    for (int l = 0; l < pool->n_caches; ++l) {
        const byhip_kv_cache& c = pool->caches[l];
        if (c.dtype != first.dtype || c.pages != first.pages || c.page_size != first.page_size || c.kv_heads != first.kv_heads ||
            c.head_dim != first.head_dim)
            fail("byhip: layer %d's cache differs from the first's", l);
        if (needs_caches || l == 0) (void)cache_args(&c);
        a.wide = a.wide && reinterpret_cast<uintptr_t>(c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v) % 16 == 0;
    }
    check_span(pool->refs, (size_t)first.pages * 4, "reference counts");
    check_span(pool->table, (size_t)pool->slots * pool->table_stride * 4, "page table");
    check_span(pool->lens, (size_t)pool->slots * 4, "lengths");
    check_span(pool->status, 16, "pool status");
    if (pool->granted) check_span(pool->granted, (size_t)pool->slots * 4, "granted tokens");
    a.p.refs = pool->refs; a.p.table = pool->table; a.p.lens = pool->lens; a.p.status = pool->status; a.p.granted = pool->granted;
    a.p.slots = pool->slots; a.p.stride = pool->table_stride; a.p.pages = first.pages; a.p.page_size = first.page_size;
    a.page_bytes = (size_t)first.kv_heads * first.page_size * first.head_dim * 2;
    a.wide = a.wide && a.page_bytes % 16 == 0;
    for (void* w : {(void*)pool->refs, (void*)pool->table, (void*)pool->lens, (void*)pool->status, (void*)pool->granted}) note_device_write(w);
    return a;
}

void check_count(int n, int most) {
    if (n < 0 || n > most) fail("byhip: %d slots in one call (at most %d)", n, most);
}

// The lists in the library's workspace: 64 KB of copies, then what the plan needs.
constexpr size_t kListBytes = 65536;
MoveList small_list() {
    int* w = static_cast<int*>(workspace());
    return {w, w + 64, w + 64 + kMaxRows};
}

void launch_copies(const Pool& a, const int* src, const int* dst, const int* count, int n, RemapArgs r) {
    for (int l0 = 0; l0 < a.c->n_caches; l0 += kLayersPerLaunch) {
        CopyArgs c{};
        const int layers = std::min(kLayersPerLaunch, a.c->n_caches - l0);
        for (int l = 0; l < layers; ++l) {
            c.base[2 * l] = static_cast<char*>(a.c->caches[l0 + l].k);
            c.base[2 * l + 1] = static_cast<char*>(a.c->caches[l0 + l].v);
            note_device_write(c.base[2 * l]);
            note_device_write(c.base[2 * l + 1]);
        }
        c.bases = 2 * layers; c.pages = a.p.pages; c.page_bytes = a.page_bytes;
        c.src = src; c.dst = dst; c.count = count; c.n = n;
        const size_t units = (size_t)n * c.bases * ((a.page_bytes + kPiece - 1) / kPiece);
        const unsigned grid = (unsigned)std::min<size_t>(units, (size_t)compute_units() * 8);
        if (grid + r.blocks == 0) return;
        if (a.wide) launch("cache_copy", (cache_copy<uint4>), dim3(r.blocks + grid), dim3(256), 0, c, r);
        else launch("cache_copy", (cache_copy<uint16_t>), dim3(r.blocks + grid), dim3(256), 0, c, r);
        BYHIP_LAUNCHED("cache_copy");
        r = RemapArgs{};
    }
}

void assign(const byhip_kv_pool* pool, const int* parents, const int* rows, int n) {
    const Pool a = pool_args(pool, false);
    check_count(n, kMaxRows);
    if (n == 0) return;
    check_span(rows, (size_t)n * 4, "slots");
    launch("cache_assign", cache_assign, dim3(n), dim3(256), 0, a.p, parents, rows, n);
    BYHIP_LAUNCHED("cache_assign");
}

}  // namespace
}  // namespace byhip

using namespace byhip;

extern "C" {

int byhip_cache_fork(const byhip_kv_pool* pool, const int* parents, const int* rows, int n) {
    return guard([&] {
        enter_compute();
        if (n > 0) check_span(parents, (size_t)n * 4, "parents");
        assign(pool, parents, rows, n);
    });
}

int byhip_cache_free(const byhip_kv_pool* pool, const int* rows, int n) {
    return guard([&] {
        enter_compute();
        assign(pool, nullptr, rows, n);
    });
}

int byhip_cache_grow(const byhip_kv_pool* pool, const int* rows, const int* add, int n) {
    return guard([&] {
        enter_compute();
        const Pool a = pool_args(pool, true);
        check_count(n, kMaxRows);
        if (n == 0) return;
        check_span(rows, (size_t)n * 4, "slots");
        check_span(add, (size_t)n * 4, "token counts");
        if ((size_t)a.p.pages * 4 > kWorkspaceBytes - kListBytes)
            unsupported("byhip: a pool of %d pages is more than the library's workspace plans for", a.p.pages);
        if ((long long)n * (a.p.stride + 1LL) > 0x7FFFFFFF)  // the plan adds up the pages that the slots ask for
            unsupported("byhip: %d slots of %d pages in one call: more pages than 31 bits count", n, a.p.stride);
        const MoveList l = small_list();
        int* free_list = reinterpret_cast<int*>(static_cast<char*>(workspace()) + kListBytes);
        launch("cache_grow_plan", cache_grow_plan, dim3(1), dim3(kPlanThreads), 0, a.p, rows, add, n, free_list, l);
        BYHIP_LAUNCHED("cache_grow_plan");
        launch_copies(a, l.src, l.dst, l.count, n, RemapArgs{});
    });
}

int byhip_cache_compact(const byhip_kv_pool* pool, int* table_out, int* refs_out) {
    return guard([&] {
        enter_compute();
        const Pool a = pool_args(pool, true);
        const size_t entries = (size_t)a.p.slots * a.p.stride;
        if (table_out) check_span(table_out, entries * 4, "moved page table");
        if (refs_out) check_span(refs_out, (size_t)a.p.pages * 4, "moved reference counts");
        if ((size_t)a.p.pages * 12 > kWorkspaceBytes - kListBytes)
            unsupported("byhip: a pool of %d pages is more than the library's workspace plans for", a.p.pages);
        int* w = static_cast<int*>(workspace());
        int* remap = reinterpret_cast<int*>(static_cast<char*>(workspace()) + kListBytes);
        const MoveList l = {w, remap + a.p.pages, remap + 2 * (size_t)a.p.pages};
        note_device_write(table_out);
        note_device_write(refs_out);
        launch("cache_compact_plan", cache_compact_plan, dim3(1), dim3(kPlanThreads), 0, a.p, refs_out ? refs_out : a.p.refs, remap, l);
        BYHIP_LAUNCHED("cache_compact_plan");
        RemapArgs r;
        r.remap = remap; r.table = a.p.table; r.out = table_out ? table_out : a.p.table; r.entries = entries; r.pages = a.p.pages;
        r.blocks = (int)std::min<size_t>((entries + 255) / 256, (size_t)compute_units());
        launch_copies(a, l.src, l.dst, l.count, a.p.pages / 2, r);
    });
}

int byhip_cache_copy(const byhip_kv_pool* pool, const int* src, const int* dst, int n) {
    return guard([&] {
        enter_compute();
        const Pool a = pool_args(pool, true);
        if (n < 0) fail("byhip: %d page copies", n);
        if (n == 0) return;
        check_span(src, (size_t)n * 4, "source pages");
        check_span(dst, (size_t)n * 4, "destination pages");
        launch_copies(a, src, dst, nullptr, n, RemapArgs{});
    });
}

}  // extern "C"
