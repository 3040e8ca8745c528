// byhip_attn_rows_f16.hip - attn_rows over f16 caches.
#include "byhip_attn_rows.h"

namespace byhip {

void launch_attn_rows_f16(const AttnArgs& a, bool precise) {
    if (precise) launch_rows_dim<BYHIP_F16, 2>(a);
    else launch_rows_dim<BYHIP_F16, 1>(a);
}

}  // namespace byhip
