// shared_tile_d64.hip -- the shared-keys MFMA kernel (shared_tile.hpp) at head_dim 64.
#include "shared_tile.hpp"

namespace vmc {

int shared_tile_d64(const TileParams& p, int src, bool q_bf16, unsigned grid, hipStream_t s) {
    return dispatch_tile<64>(p, src, q_bf16, grid, s);
}

}  // namespace vmc
