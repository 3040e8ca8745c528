// byhip_attn_rows_bf16.hip - attn_rows over bf16 caches.
#include "byhip_attn_rows.h"

namespace byhip {

void launch_attn_rows_bf16(const AttnArgs& a, bool precise) {
    if (precise) launch_rows_dim<BYHIP_BF16, 3>(a);
    else launch_rows_dim<BYHIP_BF16, 1>(a);
}

}  // namespace byhip
