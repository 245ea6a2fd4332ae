// Attention over the paged cache where a batch's new tokens are trees: the tiles'
// kernels with masks (attn_paged.h).
#include "attn_paged.h"

namespace bch {

void launch_tree_tiles(const AttnCall &a) { launch_tiles<true>(a); }

}  // namespace bch
