// Attention over paged caches: f16, head dim 128.
#include "dspark_paged_attn.h"

namespace dspark {
namespace paged {

DSPARK_PAGED_ATTN(F16, 128) { return launch_rt<F16, 128>(a, rt, codes, workgroups, most_rows, s); }

}  // namespace paged
}  // namespace dspark
