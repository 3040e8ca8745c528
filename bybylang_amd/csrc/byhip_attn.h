// byhip_attn.h - arguments and masks shared by the kernels of byhip_paged_attention.
#pragma once

#include "byhip_cache.h"

namespace byhip {

struct AttnArgs {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int q_dtype, out_dtype, cache_dtype, heads, window;
    float scale, softcap;
    const float* slopes;
    const int* prefix;
    CacheArgs c;
    BatchArgs s;
};

// Keys of sequence b that exist, and how many of them every row sees (the open prefix).
struct SeqInfo {
    int len, first_pos, prefix;  // first_pos: position of the call's first row
};

__device__ __forceinline__ SeqInfo seq_info(const AttnArgs& a, int b) {
    SeqInfo s;
    const int len = a.s.lens[b];
    s.first_pos = len - (a.s.starts[b + 1] - a.s.starts[b]);
    s.len = seq_len(a.s, a.c, b);
    s.prefix = a.prefix ? min(a.prefix[b], s.len) : 0;
    return s;
}

__device__ __forceinline__ bool sees(const AttnArgs& a, const SeqInfo& s, int pos, int j) {
    return j < s.len && ((j <= pos && (a.window <= 0 || pos - j < a.window)) || j < s.prefix);
}

}  // namespace byhip
