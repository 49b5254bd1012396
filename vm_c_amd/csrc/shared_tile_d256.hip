// shared_tile_d256.hip -- the shared-keys MFMA kernel (shared_tile.hpp) at head_dim 256.
#include "shared_tile.hpp"

namespace vmc {

int shared_tile_d256(const TileParams& p, int src, bool q_bf16, unsigned grid, hipStream_t s) {
    return dispatch_tile<256>(p, src, q_bf16, grid, s);
}

}  // namespace vmc
