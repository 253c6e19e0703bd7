// Attention over a key/value cache in 8 bits: which kernel, and how it is launched.

#include "attention_i8_rows.cuh"

namespace nnb200 {

namespace {

// Tiles of 8, 16 or 32 query rows: as many as a sequence has, on average where lengths are the device's.  A wider tile reads
// the codes for more rows at once and holds more sums in registers (head size 256 and f32 rows: 16 at most).
RowsPlan rows_plan(const nnb200_attention_i8_args& a, const DeviceInfo& dev)
{
    const nnb200_cache_i8& c = a.cache;
    const int64_t rows = (c.rows + c.seqs - 1) / c.seqs * (a.q_heads / c.heads);
    RowsPlan p;
    p.columns = rows <= 8 ? 1 : (rows <= 16 || c.dim > 128 || a.float_type == NNB200_FLOAT_F32) ? 2 : 4;
    p.blocks = dev.sm_count * (p.columns == 1 && c.dim <= 128 ? 2 : 1);
    const size_t pieces = 2 * static_cast<size_t>(p.blocks);
    p.bytes = pieces * (sizeof(RowsPiece) + static_cast<size_t>(8 * p.columns) * static_cast<size_t>(c.dim + 2) * sizeof(float));
    return p;
}

}  // namespace

size_t attention_i8_workspace_bytes(const nnb200_attention_i8_args& a, const DeviceInfo& dev) { return rows_plan(a, dev).bytes; }

int launch_attention_i8(const nnb200_attention_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const RowsPlan p = rows_plan(a, dev);
    RowsCall call;
    call.a = a;
    call.error_word = dev.error_word;
    call.group = static_cast<int>(a.q_heads / a.cache.heads);
    call.factor = a.scale * 1.4426950408889634f;
    call.pieces = static_cast<RowsPiece*>(a.workspace);
    call.sums = reinterpret_cast<float*>(call.pieces + 2 * static_cast<size_t>(p.blocks));
    switch (a.cache.dim) {
    case 64: return cuda_status(launch_attention_rows_64(call, p.columns, p.blocks, stream));
    case 96: return cuda_status(launch_attention_rows_96(call, p.columns, p.blocks, stream));
    case 128: return cuda_status(launch_attention_rows_128(call, p.columns, p.blocks, stream));
    default: return cuda_status(launch_attention_rows_256(call, p.columns, p.blocks, stream));
    }
}

}  // namespace nnb200
