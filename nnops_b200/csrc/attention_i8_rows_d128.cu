// Attention over an 8-bit cache for few rows a sequence, head size 128.
#include "attention_i8_rows.cuh"

namespace nnb200 {

cudaError_t launch_attention_rows_128(const RowsCall& call, int columns, int blocks, cudaStream_t stream)
{
    return launch_rows_dim<128>(call, columns, blocks, stream);
}

}  // namespace nnb200
