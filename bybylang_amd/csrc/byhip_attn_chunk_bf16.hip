// byhip_attn_chunk_bf16.hip - attn_chunk over bf16 caches.
#include "byhip_attn_chunk.h"

namespace byhip {

void launch_attn_chunk_bf16(const AttnArgs& a, bool precise) {
    if (precise) launch_chunk_dim<BYHIP_BF16, 3>(a);
    else launch_chunk_dim<BYHIP_BF16, 1>(a);
}

}  // namespace byhip
