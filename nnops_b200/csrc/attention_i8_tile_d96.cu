// Attention over an 8-bit cache for many rows a sequence, head size 96.
#include "attention_i8_tile.cuh"

namespace nnb200 {

cudaError_t launch_attention_tile_96(const TileCall& call, int blocks, cudaStream_t stream)
{
    return launch_tile_dim<96>(call, blocks, stream);
}

}  // namespace nnb200
