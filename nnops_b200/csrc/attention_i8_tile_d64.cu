// Attention over an 8-bit cache for many rows a sequence, head size 64.
#include "attention_i8_tile.cuh"

namespace nnb200 {

cudaError_t launch_attention_tile_64(const TileCall& call, int blocks, cudaStream_t stream)
{
    return launch_tile_dim<64>(call, blocks, stream);
}

}  // namespace nnb200
