// Attention over a key/value cache in 8 bits: which kernel, and how it is launched.

#include "attention_i8_tile.cuh"

namespace nnb200 {

namespace {

constexpr int kEngineRows = 1;
constexpr int kEngineTile = 2;
// Clusters or the line with its second kernel, us, heads of 128, 8 of them: one sequence of 4096, 8192, 16384 and 32768 tokens 9.3 / 14.7, 12.4 / 17.4,
// 18.8 / 19.4 and 31.7 / 23.9; two of 4096, 8192 and 16384 12.1 / 15.7, 17.1 / 17.5 and 27.3 / 21.8; four 12.4 / 16.6, 17.3 / 21.0 and 28.6 / 35.4.
// What is known here is the table's reach, which sequences seldom fill.
constexpr int64_t kClusterTokens = 16384;
constexpr int64_t kMostTokens = int64_t{1} << 31;   // a sequence has fewer

// Query rows that share a sequence's head, on average where their numbers are the device's.  One kernel does the whole call, so a batch that mixes
// single tokens with a prompt's chunk is served by the one that suits neither: 63 tokens and a chunk of 200 or 512 rows, 4096 tokens each, 8 heads of 128
// with 8 rows, 344 and 391 us, as two calls 153 and 196.
int64_t rows_each(const nnb200_attention_i8_args& a)
{
    const nnb200_cache_i8& c = a.cache;
    return (c.rows + c.seqs - 1) / c.seqs * (a.q_heads / c.heads);
}

int page_shift(const nnb200_attention_i8_args& a)
{
    return a.cache.page_tokens == 16 ? 4 : a.cache.page_tokens == 32 ? 5 : a.cache.page_tokens == 64 ? 6 : 7;
}

int engine_of(const nnb200_attention_i8_args& a)
{
    if (a.float_type == NNB200_FLOAT_F32) {
        return kEngineRows;   // the tiles hold queries and weights as one f16
    }
    // The tiles take as long for one row as for all of theirs, the rows' kernel the longer the more rows and the larger the heads.
    // Heads of 64, 128 and 256, rows against tiles in us: 8 sequences of 4096 tokens, 64 and 96 rows 48 / 54 and 65 / 54; 48 and 64 rows
    // 61 / 62 and 83 / 63; 16 and 32 rows 65 / 80 and 96 / 82; one of 32768 tokens, 96 and 128 rows 59 / 64 and 73 / 65; 48 and 64
    // rows 60 / 72 and 76 / 72; 16 and 32 rows 68 / 91 and 93 / 91.
    return a.force_engine != 0 ? a.force_engine : rows_each(a) * a.cache.dim > 6144 ? kEngineTile : kEngineRows;
}

// Tiles of 8 to 32 query rows: as few of them as a sequence needs, all as wide.  A wider tile reads the codes for more rows at once
// and holds more sums in registers.
RowsPlan rows_plan(const nnb200_attention_i8_args& a, const DeviceInfo& dev)
{
    const nnb200_cache_i8& c = a.cache;
    const int64_t rows = rows_each(a);
    RowsPlan p;
    const bool split = a.float_type == NNB200_FLOAT_F32;
    const int most = rows_most_columns(c.dim, split);
    const int64_t tiles = (rows + 8 * most - 1) / (8 * most);
    p.columns = static_cast<int>((rows + 8 * tiles - 1) / (8 * tiles));
    p.blocks = dev.sm_count * rows_blocks(c.dim, p.columns, split);
    // Clusters where a warp has few groups whatever the lengths are: the most that the table, or the window, has room for.
    int64_t most_tokens = c.table_pages * c.page_tokens;
    if (a.window > 0 && a.window < most_tokens) {
        const int64_t seen = a.window + (a.sinks < most_tokens ? a.sinks : most_tokens) + c.rows / c.seqs + 32;
        most_tokens = seen < most_tokens ? seen : most_tokens;
    }
    // And where all of them are under way at once.  Eight blocks have to be on neighbouring SMs, so not every SM finds a cluster that it
    // fits: 32 of two blocks to an SM do, 16 of one do not (32 rows of 128 over 4096 tokens 22.0 us, on the line 15.8), 8 do.
    const int64_t clusters = c.seqs * c.heads * tiles, room = p.blocks > dev.sm_count ? p.blocks / 8 * 7 : p.blocks / 2;
    p.tiles = c.cu == nullptr && clusters * kRowsCluster <= room && most_tokens <= kClusterTokens ? static_cast<int>(tiles) : 0;
    if (p.tiles > 0) {
        p.blocks = static_cast<int>(clusters) * kRowsCluster;
        p.bytes = 0;
        return p;
    }
    const size_t blocks = static_cast<size_t>(p.blocks);
    p.bytes = blocks * (sizeof(RowsPiece) + 2 * static_cast<size_t>(8 * p.columns) * static_cast<size_t>(c.dim + 2) * sizeof(float));
    return p;
}

// Where the parts of the tile kernels' workspace lie, each at a multiple of 16 bytes.
struct TilePlan {
    size_t tiles, first_tile, pieces, sums, bytes;   // the line's lengths are at 0
    int64_t most_tiles;
};

TilePlan tile_plan(const nnb200_attention_i8_args& a, const DeviceInfo& dev)
{
    const nnb200_cache_i8& c = a.cache;
    const int64_t group = a.q_heads / c.heads, rows = tile_rows(c.dim);
    const int64_t most = c.cu == nullptr ? c.seqs * ((c.rows / c.seqs * group + rows - 1) / rows) : c.rows * group / rows + c.seqs;
    const auto up = [](size_t v) { return (v + 15) / 16 * 16; };
    const size_t pieces = 2 * static_cast<size_t>(dev.sm_count);
    TilePlan p;
    p.most_tiles = most;
    p.tiles = 16;
    p.first_tile = p.tiles + up(static_cast<size_t>(most) * sizeof(TileInfo));
    p.pieces = p.first_tile + up(static_cast<size_t>(c.seqs + 1) * sizeof(int32_t));
    p.sums = p.pieces + up(pieces * sizeof(TilePiece));
    p.bytes = p.sums + pieces * static_cast<size_t>(rows) * static_cast<size_t>(c.dim + 2) * sizeof(float);
    return p;
}

int run_rows(const nnb200_attention_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const RowsPlan p = rows_plan(a, dev);
    RowsCall call;
    call.a = a;
    call.error_word = dev.error_word;
    call.group = static_cast<int>(a.q_heads / a.cache.heads);
    call.factor = a.scale * 1.4426950408889634f;
    const int64_t per = a.float_type == NNB200_FLOAT_F32 ? 4 : 8;
    const auto multiple = [&](const void* p, uintptr_t bytes, int64_t row, int64_t head, int64_t values) {
        return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && row % values == 0 && head % values == 0 ? 1 : 0;
    };
    call.wide = multiple(a.q, 16, a.q_stride_row, a.q_stride_head, per);
    call.wide_out = multiple(a.out, 128 / per / 2, a.out_stride_row, a.out_stride_head, 4);
    call.page_shift = page_shift(a);
    call.tiles = p.tiles;
    call.pieces = static_cast<RowsPiece*>(a.workspace);
    call.sums = reinterpret_cast<float*>(call.pieces + p.blocks);
    switch (a.cache.dim) {
    case 64: return cuda_status(launch_attention_rows_64(call, p.columns, p.blocks, stream));
    case 96: return cuda_status(launch_attention_rows_96(call, p.columns, p.blocks, stream));
    case 128: return cuda_status(launch_attention_rows_128(call, p.columns, p.blocks, stream));
    default: return cuda_status(launch_attention_rows_256(call, p.columns, p.blocks, stream));
    }
}

int run_tile(const nnb200_attention_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const TilePlan p = tile_plan(a, dev);
    const auto wide = [](const void* q, int64_t row, int64_t head) {
        return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && row % 8 == 0 && head % 8 == 0;
    };
    TileCall call;
    call.a = a;
    call.error_word = dev.error_word;
    call.group = static_cast<int>(a.q_heads / a.cache.heads);
    call.factor = a.scale * 1.4426950408889634f;
    call.wide = wide(a.q, a.q_stride_row, a.q_stride_head) && wide(a.out, a.out_stride_row, a.out_stride_head) ? 1 : 0;
    call.wide_out = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0 && a.out_stride_row % 16 == 0 && a.out_stride_head % 16 == 0 ? 1 : 0;
    call.page_shift = page_shift(a);
    uint8_t* const base = static_cast<uint8_t*>(a.workspace);
    call.most_tiles = p.most_tiles;
    call.line = reinterpret_cast<int64_t*>(base);
    call.tiles = reinterpret_cast<TileInfo*>(base + p.tiles);
    call.first_tile = reinterpret_cast<int32_t*>(base + p.first_tile);
    call.pieces = reinterpret_cast<TilePiece*>(base + p.pieces);
    call.sums = reinterpret_cast<float*>(base + p.sums);
    switch (a.cache.dim) {
    case 64: return cuda_status(launch_attention_tile_64(call, dev.sm_count, stream));
    case 96: return cuda_status(launch_attention_tile_96(call, dev.sm_count, stream));
    case 128: return cuda_status(launch_attention_tile_128(call, dev.sm_count, stream));
    default: return cuda_status(launch_attention_tile_256(call, dev.sm_count, stream));
    }
}

}  // namespace

size_t attention_i8_workspace_bytes(const nnb200_attention_i8_args& a, const DeviceInfo& dev)
{
    return engine_of(a) == kEngineTile ? tile_plan(a, dev).bytes : rows_plan(a, dev).bytes;
}

int launch_attention_i8(const nnb200_attention_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    nnb200_attention_i8_args bounded = a;   // a window beyond every token is none; differences of positions and it stay within 64 bits
    bounded.window = a.window < kMostTokens ? a.window : kMostTokens;
    bounded.sinks = a.sinks < kMostTokens ? a.sinks : kMostTokens;
    return engine_of(a) == kEngineTile ? run_tile(bounded, dev, stream) : run_rows(bounded, dev, stream);
}

}  // namespace nnb200
