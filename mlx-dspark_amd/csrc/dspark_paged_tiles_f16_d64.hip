// Attention over paged caches, many rows: f16, head dim 64.
#include "dspark_paged_tiles.h"

namespace dspark {
namespace paged {

DSPARK_PAGED_TILES(F16, 64) { return codes ? launch_tiles_of<F16, 64, true>(ta, items, s) : launch_tiles_of<F16, 64, false>(ta, items, s); }

}  // namespace paged
}  // namespace dspark
