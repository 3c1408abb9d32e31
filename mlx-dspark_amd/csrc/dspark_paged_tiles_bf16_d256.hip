// Attention over paged caches, many rows: bf16, head dim 256.
#include "dspark_paged_tiles.h"

namespace dspark {
namespace paged {

DSPARK_PAGED_TILES(BF16, 256) { return codes ? launch_tiles_of<BF16, 256, true>(ta, items, s) : launch_tiles_of<BF16, 256, false>(ta, items, s); }

}  // namespace paged
}  // namespace dspark
