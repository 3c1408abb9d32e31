// Attention over paged caches: bf16, head dim 256.
#include "dspark_paged_attn.h"

namespace dspark {
namespace paged {

DSPARK_PAGED_ATTN(BF16, 256) { return launch_rt<BF16, 256>(a, rt, codes, workgroups, most_rows, s); }

}  // namespace paged
}  // namespace dspark
