// Attention over paged caches, many rows: f16, head dim 256.
#include "dspark_paged_tiles.h"

namespace dspark {
namespace paged {

DSPARK_PAGED_TILES(F16, 256) { return codes ? launch_tiles_of<F16, 256, true>(ta, items, s) : launch_tiles_of<F16, 256, false>(ta, items, s); }

}  // namespace paged
}  // namespace dspark
