// byhip_attn_chunk_f16.hip - attn_chunk over f16 caches.
#include "byhip_attn_chunk.h"

namespace byhip {

void launch_attn_chunk_f16(const AttnArgs& a, bool precise) {
    if (precise) launch_chunk_dim<BYHIP_F16, 2>(a);
    else launch_chunk_dim<BYHIP_F16, 1>(a);
}

}  // namespace byhip
