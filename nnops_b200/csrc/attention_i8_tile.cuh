// Attention over a key/value cache in 8 bits, for many rows a sequence (prompts, chunks of prompts): the same mathematics as
// attention_i8_rows.cuh, on the fifth-generation tensor cores.
//
// A block of the grid takes 256 query rows of a key head at a time (token by token, the heads of the group next to each
// other; 128 with head size 256) as one or two M = 128 operands of tcgen05.mma, and runs along the tokens in blocks of 128:
//
//     S = Q K^T           Q and K f16 in shared memory, S f32 in tensor memory
//     P = 2^(t - m)       a thread has a row: no exchange between threads; P f16 over S in tensor memory
//     O += P V            P from tensor memory, V f16 in shared memory (its dim contiguous: the MN-major form)
//
// The cache stays in 8 bits up to the SM: four warps copy codes, turn them into f16 integers (exact) and store them in the
// 128-byte-swizzled order that the MMAs read.  That work serves 256 rows, and is done while the tensor cores and the two
// groups of four softmax warps work on the block before.  The two halves of the rows alternate: one half's weights are computed while
// the other half's products run, and a half hands its weights over in two parts of 64 tokens, so that the products of the first run
// while the second is computed.  One warp issues all MMAs, in the order that the halves take turns in: scores come over the weights whose
// products it has issued before.  Another, the scout, looks up each block's pages and scales (one for each 16 tokens) ahead of everyone,
// marks blocks that some row does not see all of, and asks for the queries that come next.  Softmax warps need more registers than
// the rest: the groups of four trade them (152, 112 and 96 of a thread's; 128 at launch; 20 bytes are
// spilled with heads of 96, 56 and 48 with bf16 and heads of 128 and 256).
//
// The sums are rescaled only when a row's maximum has grown by more than 2^8 since they were last.  Weights are 2^7 times what the formula has, so
// that the largest is between 2^7 and 2^15 and f16 holds more of those far below it (attention_i8_rows.cuh).
//
// Sequences, tiles and heads are one line of 128-token blocks, cut into equal pieces, as in attention_i8_rows.cuh; a first
// kernel writes down which tiles there are.
//
// Bound by the chain from scores over weights to products, of which two are under way, on warps that issue in 46 % of the cycles; tensor cores, exponentials and
// integer units are busy for 38 % of the time each.  Measured on one B200: 8192 rows of 32 heads of 128, causal: 686 us, 802 TFLOP/s (0.48 of the measured
// bf16 rate); the same call again and again 652 us, 8 chunks of 288 rows over 9216 tokens 396 us, 2048 rows 79 us, 8192 rows of 64 540 us, of 96 600 us, 4096 of
// 256 488 us.  Not faster: scores of 64
// tokens at a time, also into tensor memory of their own (for heads of 64); one part instead of two; weights ahead of the maximum, made up for
// afterwards; two threads to a row; what a row sees of a block applied to registers instead of to tensor memory; a part of the exponentials as polynomials
// (one in eight 2 % slower, half 13 %); one issuing warp for each half, which would also need an order between the two.
#pragma once

#include "attention_i8_rows.cuh"

namespace nnb200 {

constexpr int kTileKeys = 128;
constexpr int kTileGroups = kTileKeys / 16;
constexpr int kParts = 2;       // of a block: the products of one with V run while the softmax is at the next
constexpr int kPartKeys = kTileKeys / kParts;
constexpr int kPartGroups = kPartKeys / 16;
// Blocks that a part of a tile costs besides its own: queries, first products, sums.  (2, 3, 8 and 12 were no faster.)
constexpr int kTileCost = 4;
constexpr int kMetaSlots = 4;   // blocks whose scales are kept: the one the softmax is at, and those the converters are ahead by

// One tile of query rows, of every head.
struct TileInfo {
    int32_t seq, tile, row0, n, len;   // the sequence's, as in SequenceRows
    int32_t blocks;                    // of 128 tokens, for each head
    int64_t before;                    // length of all tiles before this one, of one head: blocks, and kTileCost for each
};

// A part of a tile that was cut, as in RowsPiece, and the rows that it is of.
struct TilePiece {
    int32_t kind, head;
    int32_t row0;    // the sequence's first
    int32_t first;   // of the sequence's rows times heads of the group
    int32_t rows;
    int32_t unused[3];
};

struct TileCall {
    nnb200_attention_i8_args a;
    int32_t* error_word;
    int group;
    float factor;
    int wide;             // q's and out's rows and heads are 16-byte aligned
    int wide_out;         // out's 32-byte aligned
    int page_shift;       // log2 of the tokens of a page
    int64_t most_tiles;   // that `tiles` has room for: as many as the rows can make, unless `cu` names some of them twice
    int64_t* line;        // [0] tiles, [1] length of all tiles, of one head
    TileInfo* tiles;
    int32_t* first_tile;  // [seqs + 1]: tiles before each sequence's
    TilePiece* pieces;    // [blocks of the grid][2]
    float* sums;          // [blocks of the grid][2][dim / 4][rows][4], then m and l of each row
};

// What a tile's rows see, as a list of 16-token groups: the sinks' first, then those from first_group on.
struct TileRange {
    int sink_groups, first_group, groups;
    int least_pos[2], most_pos[2];   // of each 128 rows; without causality beyond every token
};

template <int ROWS>
__device__ __forceinline__ TileRange tile_range(const TileCall& call, int tile, int n, int len)
{
    const nnb200_attention_i8_args& a = call.a;
    const int all = n * call.group, first_pos = len - n;
    TileRange r;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int low = min(tile * ROWS + t * 128, all - 1), high = min(tile * ROWS + t * 128 + 127, all - 1);
        r.least_pos[t] = a.causal != 0 ? first_pos + low / call.group : 0x7FFFFFFF;
        r.most_pos[t] = a.causal != 0 ? first_pos + high / call.group : 0x7FFFFFFF;
    }
    const int last = ROWS == 256 ? 1 : 0;
    const int high = r.most_pos[last] < len ? max(r.most_pos[last] + 1, 0) : len;
    int64_t low = a.window > 0 ? static_cast<int64_t>(r.least_pos[0]) - a.window + 1 : 0;
    low = low < 0 ? 0 : low > high ? high : low;
    r.first_group = static_cast<int>(low) / 16;
    const int sinks = static_cast<int>(a.sinks < high ? a.sinks : high);
    r.sink_groups = a.window > 0 ? min((sinks + 15) / 16, r.first_group) : 0;
    r.groups = r.sink_groups + (high + 15) / 16 - r.first_group;
    return r;
}

// Which tiles there are, and where each begins on the line.  One block; what it has found out of the first 1024 sequences
// stays in shared memory.
template <int ROWS>
__global__ void __launch_bounds__(1024) attention_i8_plan_kernel(const TileCall call)
{
    constexpr int kKept = 1024;
    __shared__ int64_t part[2][32];
    __shared__ int kept_first[kKept + 1];
    __shared__ SequenceRows kept_rows[kKept];
    previous_kernel_done();
    const int seqs = static_cast<int>(call.a.cache.seqs), lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int turn = 0;
    // Of the threads before this one and of all, over the block.
    const auto before = [&](int64_t v, int64_t& total) {
        int64_t up = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t other = __shfl_up_sync(0xFFFFFFFFu, up, o);
            up += lane >= o ? other : 0;
        }
        if (lane == 31) {
            part[turn][warp] = up;
        }
        __syncthreads();
        int64_t warps = part[turn][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t other = __shfl_up_sync(0xFFFFFFFFu, warps, o);
            warps += lane >= o ? other : 0;
        }
        total = __shfl_sync(0xFFFFFFFFu, warps, 31);
        const int64_t earlier = __shfl_sync(0xFFFFFFFFu, warps, warp > 0 ? warp - 1 : 0);
        turn ^= 1;   // the next round's may be written while this one's are read
        return (warp > 0 ? earlier : 0) + up - v;
    };
    int64_t tiles = 0, total;
    for (int b0 = 0; b0 < seqs; b0 += 1024) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        SequenceRows s{};
        if (b < seqs) {
            s = sequence_rows(call.a.cache, b);
        }
        const int64_t first = tiles + before((s.n * call.group + ROWS - 1) / ROWS, total);
        if (b < seqs) {
            const int held = static_cast<int>(min(first, call.most_tiles));
            call.first_tile[b] = held;
            if (b < kKept) {
                kept_first[b] = held;
                kept_rows[b] = s;
            }
        }
        tiles += total;
    }
    __syncthreads();
    tiles = min(tiles, call.most_tiles);
    int64_t line = 0;
    for (int i0 = 0; i0 < tiles; i0 += 1024) {
        const int i = i0 + static_cast<int>(threadIdx.x);
        TileInfo info{};
        if (i < tiles) {
            int low = 0, high = seqs;   // first_tile[low] <= i, and below first_tile[high]
            while (high - low > 1) {
                const int mid = (low + high) / 2;
                ((mid < kKept ? kept_first[mid] : call.first_tile[mid]) <= i ? low : high) = mid;
            }
            const SequenceRows s = low < kKept ? kept_rows[low] : sequence_rows(call.a.cache, low);
            info.seq = low;
            info.tile = i - (low < kKept ? kept_first[low] : call.first_tile[low]);
            info.row0 = s.row0;
            info.n = s.n;
            info.len = s.len;
            info.blocks = max((tile_range<ROWS>(call, info.tile, s.n, s.len).groups + kTileGroups - 1) / kTileGroups, 1);
        }
        info.before = line + before(i < tiles ? info.blocks + kTileCost : 0, total);
        if (i < tiles) {
            call.tiles[i] = info;
        }
        line += total;
    }
    if (threadIdx.x == 0) {
        call.line[0] = tiles;
        call.line[1] = line;
    }
}

// A walk over this block's piece of the line: the same for every warp.
struct TileWalk {
    int64_t at, end;
    int tiles, index;    // index: of the tile that `at` lies in, or an earlier one
    // The part of a tile and head that comes next.
    TileInfo info;
    int head, off, count;
    bool begins, ends;

    // Warp-collective.
    __device__ __forceinline__ void begin(const TileCall& call, int block, int blocks)
    {
        tiles = static_cast<int>(call.line[0]);
        const int64_t line = call.line[1] * call.a.cache.heads, least = kTileCost;
        const int64_t most = (line + least - 1) / least < blocks ? (line + least - 1) / least : blocks;
        at = end = 0;
        index = 0;
        if (block >= most) {
            return;
        }
        at = line / most * block + line % most * block / most;
        end = line / most * (block + 1) + line % most * (block + 1) / most;
        // The last tile that begins at or before `at`, 32 probes at a time.
        int count_ = tiles;
        const int lane = static_cast<int>(threadIdx.x & 31);
        while (count_ > 1) {
            const int step = (count_ + 31) / 32;
            const bool before = lane * step < count_ && call.tiles[index + lane * step].before * call.a.cache.heads <= at;
            const int last = (__popc(__ballot_sync(0xFFFFFFFFu, before)) - 1) * step;
            index += last;
            count_ = min(step, count_ - last);
        }
    }

    __device__ __forceinline__ bool next(const TileCall& call)
    {
        while (at < end) {
            info = call.tiles[index];
            const int64_t heads = call.a.cache.heads;
            while (at >= (info.before + info.blocks + kTileCost) * heads) {
                info = call.tiles[++index];
            }
            const int length = info.blocks + kTileCost;
            const int64_t rel = at - info.before * heads;
            head = static_cast<int>(rel / length);
            const int from = static_cast<int>(rel % length);
            const int to = static_cast<int>(min(static_cast<int64_t>(length), from + (end - at)));
            at += to - from;
            off = max(from - kTileCost, 0);
            count = max(to - kTileCost, 0) - off;
            begins = off == 0;
            ends = off + count == info.blocks;
            if (count > 0) {
                return true;
            }
        }
        return false;
    }
};

struct GroupMeta {
    float k, v_log2, v_inv;
    int key0;   // first token; its low bits: 1 (2) if the first (second) 128 rows do not see all of its tokens
};

// What the scout says of a block besides: bits 0, 1: half h has more to do than t = s k + v_log2.
constexpr int kBlockLast = 4;   // of this block of the grid
constexpr int kBlockNone = 8;   // there is no block at all

template <int D>
struct TileShared {
    static constexpr int kHalves = D <= 128 ? 2 : 1;
    static constexpr int kRows = 128 * kHalves;
    static constexpr int kBlockBytes = 16384;   // 128 rows of 128 bytes: 64 f16 of each token
    static constexpr int kTileBytes = (D + 63) / 64 * kBlockBytes;
    static constexpr int kStages = D <= 128 ? 2 : 1;
    // Codes on their way: two units, of all 128 tokens of a block, or of 64 with head size 256.
    static constexpr int kUnits = D <= 128 ? 1 : 2;   // of a block's keys, and of its values
    static constexpr int kUnitBytes = kTileKeys * D / kUnits;
    static constexpr int kBytes = 1024 + (kHalves + 2 * kStages) * kTileBytes + 2 * kUnitBytes;
    static constexpr int kSoftmaxWarps = 4 * kHalves;
    static constexpr int kThreads = 32 * (kSoftmaxWarps + 8);   // and four for codes, the MMA issuer, the scout (and two to fill its group)
    // Registers of a thread: at launch, and of the three kinds of warps afterwards.
    static constexpr int kRegisters = kHalves == 2 ? 128 : 168;
    static constexpr int kSoftmaxRegisters = kHalves == 2 ? 152 : 200;
    static constexpr int kCodesRegisters = kHalves == 2 ? 112 : 168;
    static constexpr int kIssuerRegisters = kHalves == 2 ? 96 : 136;
    static_assert(kHalves * kSoftmaxRegisters + kCodesRegisters + kIssuerRegisters <= (kHalves + 2) * kRegisters, "a group would wait for registers");
    static constexpr int kOutColumn = 256;      // of the sums in tensor memory; S and P are below
    static_assert(kBytes <= 226 * 1024, "shared memory");
};

__device__ __forceinline__ void tile_mma_p(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tile_tmem_st_16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

__device__ __forceinline__ void tile_tmem_ld_16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tile_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The warpgroup's registers of a thread from here on.
template <int N>
__device__ __forceinline__ void more_registers()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair_of(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The same in every lane, and in a uniform register: what a reduction gives is, what a shuffle gives is not.
__device__ __forceinline__ uint32_t in_uniform(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }

// 16 codes as f16 into the swizzled tile: row `key`, dims [16 segment, + 16).
template <int D>
__device__ __forceinline__ void store_codes(uint8_t* tile, int key, int segment, const uint4& codes)
{
    uint32_t h[8];
    codes_to_half(codes.x, h[0], h[1]);
    codes_to_half(codes.y, h[2], h[3]);
    codes_to_half(codes.z, h[4], h[5]);
    codes_to_half(codes.w, h[6], h[7]);
    uint8_t* row = tile + segment / 4 * TileShared<D>::kBlockBytes + key * 128;
    const int chunk = 2 * segment & 7, turn = segment / 4 & 1;   // lanes of the two 64-dim blocks use different banks
    const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
    *reinterpret_cast<uint4*>(row + (((chunk + turn) ^ (key & 7)) << 4)) = turn ? b : a;
    *reinterpret_cast<uint4*>(row + (((chunk + 1 - turn) ^ (key & 7)) << 4)) = turn ? a : b;
}

template <int D, typename T>
__global__ void __launch_bounds__(TileShared<D>::kThreads, 1) attention_i8_tile_kernel(const TileCall call)
{
    using Shared = TileShared<D>;
    constexpr int kHalves = Shared::kHalves, kStages = Shared::kStages, kRows = Shared::kRows;
    constexpr int kPerThread = D / 16 / Shared::kUnits;   // 16-code segments of a unit that a converting thread has
    extern __shared__ uint8_t raw_shared[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][kParts], o_full[2][kParts];
    __shared__ __align__(8) uint64_t meta_full[kMetaSlots], meta_empty[kMetaSlots];
    __shared__ GroupMeta meta[kMetaSlots][kTileGroups], identity[kTileGroups];
    __shared__ int64_t where[kMetaSlots][kTileGroups];   // of a group's codes; -1: none
    __shared__ int state[kMetaSlots];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    uint8_t* const shared = raw_shared + (1024 - smem_u32(raw_shared) % 1024) % 1024;
    uint8_t* const q_tile = shared;
    uint8_t* const k_tile = q_tile + kHalves * Shared::kTileBytes;
    uint8_t* const v_tile = k_tile + kStages * Shared::kTileBytes;
    uint8_t* const codes_ring = v_tile + kStages * Shared::kTileBytes;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 128);
            mbar_init(&k_full[i], 128);
            mbar_init(&v_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            for (int part = 0; part < kParts; ++part) {
                mbar_init(&p_full[i][part], 128);
                mbar_init(&o_full[i][part], 1);
            }
        }
        for (int i = 0; i < kMetaSlots; ++i) {
            mbar_init(&meta_full[i], 1);
            mbar_init(&meta_empty[i], Shared::kSoftmaxWarps);
        }
        for (int i = 0; i < kTileGroups; ++i) {
            identity[i] = GroupMeta{1.0f, 0.0f, 0.0f, 0};
        }
        mbar_init_fence();
    }
    if (warp == Shared::kSoftmaxWarps + 4) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    previous_kernel_done();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    const nnb200_attention_i8_args& a = call.a;

    TileWalk walk;
    walk.begin(call, blockIdx.x, gridDim.x);

    if (warp < Shared::kSoftmaxWarps) {
        // ---------------- softmax: a thread has a row ----------------
        more_registers<Shared::kSoftmaxRegisters>();
        const int half = warp / 4, row = threadIdx.x & 127;
        const uint32_t s_addr = tmem + static_cast<uint32_t>((warp & 3) * 32 << 16) + static_cast<uint32_t>(half * 128);
        const uint32_t o_addr = tmem + static_cast<uint32_t>((warp & 3) * 32 << 16) + static_cast<uint32_t>(Shared::kOutColumn + half * 128);
        uint32_t n = 0;   // blocks
        int kinds[2] = {0, 0};
        // The row of the part that is next: its place in out, its tokens (those before `end`, and not before `low` unless before
        // `sinks`), its factor.
        bool there = false;
        int end = 0, low = 0;
        const int sinks = static_cast<int>(min(a.sinks, int64_t{0x7FFFFFFF}));
        int64_t place = 0;
        float factor = 0.0f;
        const auto load_queries = [&] {
            const int first = walk.info.tile * kRows + half * 128 + (warp & 3) * 32, all = walk.info.n * call.group;
            const auto source = [&](int r, int64_t stride_row, int64_t stride_head) {   // of this warp's r-th row
                const int token = (first + r) / call.group;
                return (walk.info.row0 + token) * stride_row + (walk.head * call.group + (first + r) - token * call.group) * stride_head;
            };
            there = first + lane < all;
            place = there ? source(lane, a.out_stride_row, a.out_stride_head) : 0;
            const int pos = walk.info.len - walk.info.n + (first + lane) / call.group;
            end = a.causal != 0 && pos < walk.info.len ? max(pos + 1, 0) : walk.info.len;
            low = a.window > 0 ? static_cast<int>(max(end - a.window, int64_t{0})) : 0;
            factor = call.factor;
            // Four lanes to a row, eight rows at a time: 64 bytes of each next to each other.  All are asked for before any is looked at.
            uint4 raw[4][D / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + lane / 4;
                const bool row_there = first + r < all;
                const T* src = static_cast<const T*>(a.q) + (row_there ? source(r, a.q_stride_row, a.q_stride_head) : 0) + lane % 4 * 8;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    raw[i][c] = row_there ? eight_of(reinterpret_cast<const uint16_t*>(src + c * 32), call.wide != 0) : make_uint4(0u, 0u, 0u, 0u);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + lane / 4;
                if constexpr (!std::is_same_v<T, __half>) {   // scaled by a power of two into f16
                    uint32_t top = 0;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        const uint32_t w[4] = {raw[i][c].x, raw[i][c].y, raw[i][c].z, raw[i][c].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            top = max(top, max(w[e] << 16 & 0x7FFF0000u, w[e] & 0x7FFF0000u));
                        }
                    }
                    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    const int e = row_exponent(top);
                    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    const float up = call.factor * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                    const float mine = __shfl_sync(0xFFFFFFFFu, up, lane % 8 * 4);
                    factor = lane / 8 == i ? mine : factor;
                    const auto scaled = [&](uint32_t w) {
                        float x, y;
                        unpack2<T>(w, x, y);
                        return pack2<__half>(x * down, y * down);
                    };
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        raw[i][c] = make_uint4(scaled(raw[i][c].x), scaled(raw[i][c].y), scaled(raw[i][c].z), scaled(raw[i][c].w));
                    }
                }
                uint8_t* const to = q_tile + half * Shared::kTileBytes + ((warp & 3) * 32 + r) * 128;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    const int chunk = c * 4 + lane % 4;
                    *reinterpret_cast<uint4*>(to + chunk / 8 * Shared::kBlockBytes + (((chunk & 7) ^ (r & 7)) << 4)) = raw[i][c];
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&q_full[half]);
        };
        // The part whose sums are next: where they go.
        bool had = false, whole = false, pending = false;
        int which = 0;
        T* dst = nullptr;
        TilePiece about{};
        constexpr float kTop = rows_top_weight(false);
        float m = 0.0f, l = 0.0f;   // m: the maximum less kTop
        bool ok = true, more = walk.next(call);
        while (more || pending) {
            // The scores of the part before are all there, so its queries may go, and the next one's first products come right
            // behind its last.
            if (more) {
                load_queries();
            }
            if (pending) {
                if (!wait_every_lane(&o_full[half][kParts - 1], (n - 1) & 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                float* piece = call.sums + (2 * static_cast<int64_t>(blockIdx.x) + which) * (kRows * (D + 2));
#pragma unroll 2
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld_32x32(o_addr + static_cast<uint32_t>(c * 32), o);
                    tmem_ld_wait();
                    if (had && whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                        }
                        const auto two = [&](int i) { return pack2<T>(__uint_as_float(o[i]), __uint_as_float(o[i + 1])); };
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (call.wide_out != 0) {   // whole sectors
                                st_global_32(dst + c * 32 + h * 16, two(16 * h), two(16 * h + 2), two(16 * h + 4), two(16 * h + 6), two(16 * h + 8), two(16 * h + 10),
                                             two(16 * h + 12), two(16 * h + 14));
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    dst[c * 32 + h * 16 + i] = from_float<T>(__uint_as_float(o[16 * h + i]));
                                }
                            }
                        }
                    } else if (had) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            reinterpret_cast<uint4*>(piece)[(c * 8 + i) * kRows + half * 128 + row] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }
                }
                if (!whole) {
                    if (had) {
                        piece[kRows * D + half * 128 + row] = m;
                        piece[kRows * (D + 1) + half * 128 + row] = l;
                    }
                    kinds[which] = about.kind;
                    if (threadIdx.x == 0) {
                        call.pieces[2 * blockIdx.x + which] = about;
                    }
                }
                tc_fence_before_sync();
                pending = false;
            }
            if (!more) {
                break;
            }
            m = -INFINITY;
            l = 0.0f;
            float most = kMostWeight;   // of a weight's log2; less where its own rounding may be more than half
            const int count = walk.count;
#pragma unroll 1
            for (int i = 0; i < kParts * count; ++i) {
                // Part i % kParts of block n.
                const int part = i % kParts;
                const uint32_t part_addr = s_addr + static_cast<uint32_t>(part * kPartKeys);
                if (part == 0) {
                    ok = wait_every_lane(&s_full[half], n & 1, &abort_flag) &&
                         wait_every_lane(&meta_full[n % kMetaSlots], n / kMetaSlots & 1, &abort_flag);   // long since: the products waited for it
                    if (!ok) {
                        break;
                    }
                    tc_fence_after_sync();
                }
                const GroupMeta* const groups = meta[n % kMetaSlots] + part * kPartGroups;
                const bool plain = (state[n % kMetaSlots] >> half & 1) == 0;
                const GroupMeta* const linear = plain ? groups : identity;
                if (!plain) {
                    // Scores become exponents in place, those that the row does not see -infinity.
#pragma unroll 1
                    for (int g = 0; g < kPartGroups; ++g) {
                        const GroupMeta of = groups[g];
                        const int key0 = of.key0 & ~15;
                        const auto first_bits = [&](int tokens) { return (1u << min(max(tokens - key0, 0), 16)) - 1u; };
                        // A bit for each token that the row sees.
                        const uint32_t seen = (of.key0 >> half & 1) == 0 ? 0xFFFFu : first_bits(end) & (~first_bits(low) | first_bits(sinks));
                        uint32_t s[16];
                        if (__any_sync(0xFFFFFFFFu, seen != 0)) {
                            tile_tmem_ld_16(part_addr + static_cast<uint32_t>(g * 16), s);
                            tmem_ld_wait();
                        }
                        const float k = of.k * factor;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            s[e] = (seen >> e & 1) != 0 ? __float_as_uint(__fmaf_rn(__uint_as_float(s[e]), k, of.v_log2)) : __float_as_uint(-INFINITY);
                        }
                        tile_tmem_st_16(part_addr + static_cast<uint32_t>(g * 16), s);
                    }
                    tile_tmem_st_wait();
                }
                uint32_t s[kPartKeys];
                float k[kPartGroups], add[kPartGroups], tops[kPartGroups];
                const float scale = plain ? factor : 1.0f;
#pragma unroll
                for (int c = 0; c < kPartKeys / 32; ++c) {
                    tmem_ld_32x32(part_addr + static_cast<uint32_t>(c * 32), *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                }
#pragma unroll
                for (int g = 0; g < kPartGroups; ++g) {
                    k[g] = linear[g].k * scale;
                    add[g] = linear[g].v_log2;
                }
                tmem_ld_wait();
#pragma unroll
                for (int g = 0; g < kPartGroups; ++g) {
                    float high = __uint_as_float(s[16 * g]), other = __uint_as_float(s[16 * g + 1]);
#pragma unroll
                    for (int e = 2; e < 14; e += 4) {
                        high = max3(high, __uint_as_float(s[16 * g + e]), __uint_as_float(s[16 * g + e + 1]));
                        other = max3(other, __uint_as_float(s[16 * g + e + 2]), __uint_as_float(s[16 * g + e + 3]));
                    }
                    high = max3(high, __uint_as_float(s[16 * g + 14]), __uint_as_float(s[16 * g + 15]));
                    tops[g] = __fmaf_rn(fmaxf(high, other), k[g], add[g]);
                }
                float top = tops[0];
#pragma unroll
                for (int g = 1; g < kPartGroups; ++g) {
                    top = fmaxf(top, tops[g]);
                }
                const bool grown = top - m > most;   // (not top > m + most: a sum that is rounded up would let a larger weight pass)
                if (__any_sync(0xFFFFFFFFu, grown)) {
                    const float next = grown ? (is_coarse(top) ? top : top - kTop) : m;
                    most = is_coarse(next) ? kMostWeight - kTop : kMostWeight;
                    const float alpha = grown ? exp2_fast(m - next) : 1.0f;
                    m = next;
                    l *= alpha;
                    if (i > 0) {
                        // The sums so far are complete: the next part's products wait for this one's weights.
                        if (!wait_every_lane(&o_full[half][(part + kParts - 1) % kParts], (part == 0 ? n - 1 : n) & 1, &abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tile_tmem_ld_16(o_addr + static_cast<uint32_t>(c * 16), o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            }
                            tile_tmem_st_16(o_addr + static_cast<uint32_t>(c * 16), o);
                        }
                    }
                }
                const float safe = m == -INFINITY ? 0.0f : m;
                uint64_t sums[kPartGroups];
#pragma unroll
                for (int c = 0; c < kPartGroups / 2; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int g = 2 * c + h;
                        const float less = add[g] - safe;
                        const uint64_t kk = pair_of(k[g], k[g]), aa = pair_of(less, less);
                        uint64_t sum[2] = {0, 0};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float x, y;
                            unpair(pair_fma(pair_of(__uint_as_float(s[16 * g + 2 * e]), __uint_as_float(s[16 * g + 2 * e + 1])), kk, aa), x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                            sum[e & 1] = e < 2 ? pair_of(x, y) : pair_add(sum[e & 1], pair_of(x, y));
                            p[8 * h + e] = pack2<__half>(x, y);
                        }
                        sums[g] = pair_add(sum[0], sum[1]);
                    }
                    tile_tmem_st_16(part_addr + static_cast<uint32_t>(c * 16), p);
                }
                tile_tmem_st_wait();
                tc_fence_before_sync();
                mbar_arrive(&p_full[half][part]);
#pragma unroll
                for (int g = 0; g < kPartGroups; ++g) {
                    float x, y;
                    unpair(sums[g], x, y);
                    x += y;
                    l += x == 0.0f ? 0.0f : x * groups[g].v_inv;   // (not 0 times what a block that is masked has for a scale)
                }
                if (part == kParts - 1) {
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&meta_empty[n % kMetaSlots]);
                    }
                    ++n;
                }
            }
            if (!ok) {
                break;
            }
            whole = walk.begins && walk.ends;
            had = there;
            which = walk.begins ? 1 : 0;
            about = TilePiece{walk.begins ? 1 : walk.ends ? 3 : 2, walk.head, walk.info.row0, walk.info.tile * kRows,
                              min(kRows, walk.info.n * call.group - walk.info.tile * kRows), {}};
            dst = static_cast<T*>(a.out) + place;
            pending = true;
            more = walk.next(call);
        }
        if (threadIdx.x < 2 && kinds[threadIdx.x] == 0) {
            call.pieces[2 * blockIdx.x + threadIdx.x].kind = 0;
        }
        if (!ok && lane == 0) {
            atomicCAS(call.error_word, 0, kErrEpilogueWait);
        }
        __syncwarp();
    } else if (warp < Shared::kSoftmaxWarps + 4) {
        // ---------------- codes into f16 tiles ----------------
        fewer_registers<Shared::kCodesRegisters>();
        const int t = threadIdx.x - 32 * Shared::kSoftmaxWarps;
        // A thread copies the 16-byte segments that it converts itself: what it waits for is its own copies.
        uint8_t* const my_codes = codes_ring + t * 16;
        const auto load = [&](const void* codes, uint32_t block, int part, int slot) {
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int idx = t + (part * kPerThread + i) * 128, key = idx / (D / 16), segment = idx % (D / 16);
                const int64_t base = where[block % kMetaSlots][key / 16];
                cp_async_16(my_codes + slot * Shared::kUnitBytes + i * 2048,
                            static_cast<const uint8_t*>(codes) + (base < 0 ? 0 : base + ((key & 15) * D + segment * 16)), base < 0 ? 0u : 16u);
            }
            cp_async_commit();
        };
        const auto store = [&](uint8_t* tile, int part, int slot) {
            cp_async_wait_group<1>();
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int idx = t + (part * kPerThread + i) * 128;
                store_codes<D>(tile, idx / (D / 16), idx % (D / 16), *reinterpret_cast<const uint4*>(my_codes + slot * Shared::kUnitBytes + i * 2048));
            }
        };
        bool ok = wait_every_lane(&meta_full[0], 0, &abort_flag);
        bool more = ok && (state[0] & kBlockNone) == 0;
        if (more) {
            load(a.cache.k, 0, 0, 0);
            load(Shared::kUnits == 1 ? a.cache.v : a.cache.k, 0, Shared::kUnits - 1, 1);
        }
        for (uint32_t n = 0; more; ++n) {
            const uint32_t slot = n % kStages, round = n / kStages & 1;
            const bool next = (state[n % kMetaSlots] & kBlockLast) == 0;
            ok = wait_every_lane(&k_empty[slot], round ^ 1, &abort_flag) &&
                 (!next || wait_every_lane(&meta_full[(n + 1) % kMetaSlots], (n + 1) / kMetaSlots & 1, &abort_flag));
            if (!ok) {
                break;
            }
#pragma unroll
            for (int part = 0; part < Shared::kUnits; ++part) {
                store(k_tile + slot * Shared::kTileBytes, part, part);
                if (Shared::kUnits == 2) {
                    load(a.cache.v, n, part, part);
                } else if (next) {
                    load(a.cache.k, n + 1, 0, 0);
                } else {
                    cp_async_commit();
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&k_full[slot]);
            ok = wait_every_lane(&v_empty[slot], round ^ 1, &abort_flag);
            if (!ok) {
                break;
            }
#pragma unroll
            for (int part = 0; part < Shared::kUnits; ++part) {
                store(v_tile + slot * Shared::kTileBytes, part, Shared::kUnits == 1 ? 1 : part);
                if (next) {
                    load(Shared::kUnits == 1 ? a.cache.v : a.cache.k, n + 1, part, Shared::kUnits == 1 ? 1 : part);
                } else {
                    cp_async_commit();
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&v_full[slot]);
            more = next;
        }
        cp_async_wait_group<0>();
        if (!ok && lane == 0) {
            atomicCAS(call.error_word, 0, kErrDequantWait);
        }
        __syncwarp();
    } else if (fewer_registers<Shared::kIssuerRegisters>(); warp == Shared::kSoftmaxWarps + 4) {
        // ---------------- MMA issuer ----------------
        const uint32_t base = in_uniform(tmem);
        constexpr uint32_t kIdescS = umma_idesc(1, 0, 0, 128, kTileKeys);
        constexpr uint32_t kIdescO = umma_idesc(1, 0, 0, 128, D) | kUmmaBMajorMN;
        const uint64_t q_desc = umma_desc_sw128_kmajor(smem_u32(q_tile));
        const uint64_t k_desc = umma_desc_sw128_kmajor(smem_u32(k_tile));
        const uint64_t v_desc = umma_desc_sw128_mnmajor(smem_u32(v_tile), Shared::kBlockBytes);
        constexpr uint64_t kTileStep = Shared::kTileBytes / 16, kBlockStep = Shared::kBlockBytes / 16;
        uint32_t failed = 0;
        const auto scores = [&](int half, uint32_t slot, bool last) {
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t step = static_cast<uint64_t>(k / 4) * kBlockStep + static_cast<uint64_t>(k % 4 * 2);
                    umma_f16(base + static_cast<uint32_t>(half * 128), q_desc + static_cast<uint64_t>(half) * kTileStep + step,
                             k_desc + slot * kTileStep + step, kIdescS, k > 0 ? 1u : 0u);
                }
                umma_commit_unless(&s_full[half], failed);
                if (last) {
                    umma_commit_unless(&k_empty[slot], failed);
                }
            }
            __syncwarp();
        };
        uint32_t n = 0, units = 0;
        // What steers the loops is made uniform in the compiler's eyes: the MMAs' operands then stay in uniform registers.
        while (in_uniform(walk.next(call) ? 1u : 0u) != 0) {
            const int count = static_cast<int>(in_uniform(static_cast<uint32_t>(walk.count)));
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                mbar_wait_converged<kErrMmaWait>(&q_full[h], units & 1, &abort_flag, failed);
                if (h == 0) {
                    mbar_wait_converged<kErrMmaWait>(&k_full[n % kStages], n / kStages & 1, &abort_flag, failed);
                }
                tc_fence_after_sync();
                scores(h, n % kStages, h == kHalves - 1);
            }
            for (int j = 0; j < count; ++j, ++n) {
                const bool next = j + 1 < count;
                const uint32_t slot = n % kStages, next_slot = (n + 1) % kStages;
                // One half after the other: while the products of one run, the softmax of the other does.
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    if (h == 0) {
                        mbar_wait_converged<kErrMmaWait>(&v_full[slot], n / kStages & 1, &abort_flag, failed);
                    }
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        mbar_wait_converged<kErrMmaWait>(&p_full[h][part], n & 1, &abort_flag, failed);
                        tc_fence_after_sync();
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < kPartKeys / 16; ++k) {
                                tile_mma_p(base + static_cast<uint32_t>(Shared::kOutColumn + h * 128),
                                           base + static_cast<uint32_t>(h * 128 + part * kPartKeys + k * 8),
                                           v_desc + slot * kTileStep + static_cast<uint64_t>((part * kPartKeys + k * 16) * 128 / 16), kIdescO,
                                           j > 0 || part > 0 || k > 0 ? 1u : 0u);
                            }
                            umma_commit_unless(&o_full[h][part], failed);
                            if (h == kHalves - 1 && part == kParts - 1) {
                                umma_commit_unless(&v_empty[slot], failed);
                            }
                        }
                        __syncwarp();
                    }
                    if (next) {
                        if (h == 0) {
                            mbar_wait_converged<kErrMmaWait>(&k_full[next_slot], (n + 1) / kStages & 1, &abort_flag, failed);
                            tc_fence_after_sync();
                        }
                        scores(h, next_slot, h == kHalves - 1);   // over the weights that have just been used
                    }
                }
            }
            ++units;
        }
        if (const uint32_t code = warp_failure(failed); code != 0) {
            if (lane == 0) {
                atomicCAS(call.error_word, 0, static_cast<int32_t>(code));
            }
            umma_settle_after_failure();
        }
        __syncwarp();
    } else if (warp == Shared::kSoftmaxWarps + 5) {
        // ---------------- scout: where the blocks' codes lie, and their scales ----------------
        const int tokens = static_cast<int>(a.cache.page_tokens);
        bool ok = true, more = walk.next(call);
        if (!more && lane == 0) {
            state[0] = kBlockNone;
            mbar_arrive(&meta_full[0]);
        }
        uint32_t n = 0;
        while (ok && more) {
            const TileRange range = tile_range<kRows>(call, walk.info.tile, walk.info.n, walk.info.len);
            const TileInfo info = walk.info;
            const int head = walk.head, off = walk.off, count = walk.count;
            more = walk.next(call);
            if (more) {   // the queries that come after this part's are on their way into L2 by the time they are asked for
                const int first = walk.info.tile * kRows, rows = min(kRows, walk.info.n * call.group - first);
                for (int r = lane; r < rows; r += 32) {
                    const int token = (first + r) / call.group;
                    const T* src = static_cast<const T*>(a.q) + (walk.info.row0 + token) * a.q_stride_row + (walk.head * call.group + (first + r) - token * call.group) * a.q_stride_head;
#pragma unroll
                    for (int byte = 0; byte < 2 * D; byte += 128) {
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(src) + byte));
                    }
                }
            }
            for (int j = 0; j < count; ++j, ++n) {
                // Lanes 0..7 have a group each.
                const int idx = (off + j) * kTileGroups + lane;
                // Where there is no group, or no page: behind every token, so that not even a query that is no number makes a weight of it.
                GroupMeta of{0.0f, -INFINITY, 0.0f, 0x7FFFFFF0 | (kHalves == 2 ? 3 : 1)};
                int64_t at = -1;
                if (lane < kTileGroups && idx < range.groups) {
                    const int key0 = (idx < range.sink_groups ? idx : idx - range.sink_groups + range.first_group) * 16;
                    const int page = page_at(a.cache, info.seq, key0 >> call.page_shift, call.error_word);
                    if (page >= 0) {
                        const int64_t scale = page * a.cache.scale_page_stride + head;
                        const float vs = a.cache.v_scale[scale], sure = vs < kLeastCacheScale ? kLeastCacheScale : vs;
                        of.k = a.cache.k_scale[scale];
                        of.v_log2 = log2f(sure);
                        of.v_inv = __fdiv_rn(1.0f, sure);
                        of.key0 = key0;
                        at = page * a.cache.page_stride + (static_cast<int64_t>(head) * tokens + (key0 & (tokens - 1))) * D;
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
                            const bool all_seen = key0 + 15 < info.len && key0 + 15 <= range.least_pos[h] &&
                                                  (a.window == 0 || key0 > range.most_pos[h] - a.window || key0 + 15 < a.sinks);
                            of.key0 |= all_seen ? 0 : 1 << h;
                        }
                    }
                }
                // A scale below zero turns the order of its scores round: those too are looked at one by one.
                const int odd = __reduce_or_sync(0xFFFFFFFFu, lane >= kTileGroups ? 0 : (of.key0 & 3) | (of.k * call.factor < 0.0f ? 3 : 0));
                const uint32_t slot = n % kMetaSlots;
                if (!wait_every_lane(&meta_empty[slot], (n / kMetaSlots & 1) ^ 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                if (lane < kTileGroups) {
                    meta[slot][lane] = of;
                    where[slot][lane] = at;
                }
                if (lane == 0) {
                    state[slot] = odd | (!more && j + 1 == count ? kBlockLast : 0);
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&meta_full[slot]);
                }
            }
        }
        if (!ok && lane == 0) {
            atomicCAS(call.error_word, 0, kErrProducerWait);
        }
        __syncwarp();
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == Shared::kSoftmaxWarps + 4) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the pieces of the tiles that were cut: blockIdx.x of the grid of the kernel before, 16 dims each block.
template <int D, typename T>
__global__ void __launch_bounds__(256) attention_i8_tile_join_kernel(const TileCall call)
{
    previous_kernel_done();
    constexpr int kRows = TileShared<D>::kRows;
    constexpr int64_t kPiece = kRows * (D + 2);
    const TilePiece mine = call.pieces[2 * blockIdx.x + 1];
    if (mine.kind != 1) {
        return;
    }
    const nnb200_attention_i8_args& a = call.a;
    int last = blockIdx.x + 1;
    while (last < static_cast<int>(gridDim.x) - 1 && call.pieces[2 * last].kind == 2) {
        ++last;
    }
    const float* first = call.sums + (2 * static_cast<int64_t>(blockIdx.x) + 1) * kPiece;
    const float* rest = call.sums + 2 * static_cast<int64_t>(blockIdx.x + 1) * kPiece;
    const int more = last - static_cast<int>(blockIdx.x), r = threadIdx.x, d = blockIdx.y * 16;
    if (r >= mine.rows) {
        return;
    }
    // A maximum that later turns out too small is made up for, so that a piece is read once.
    float top = -INFINITY, total = 0.0f;
    float4 sum[4] = {};
    for (int p = -1; p < more; ++p) {
        const float* piece = p < 0 ? first : rest + p * 2 * kPiece;
        const float m = piece[kRows * D + r], l = piece[kRows * (D + 1) + r];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = reinterpret_cast<const float4*>(piece)[(d / 4 + i) * kRows + r];
        }
        const float next = fmaxf(top, m), safe = next == -INFINITY ? 0.0f : next;
        const float old = exp2_fast(top - safe), share = exp2_fast(m - safe);
        top = next;
        total = __fmaf_rn(l, share, total * old);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i].x = __fmaf_rn(v[i].x, share, sum[i].x * old);
            sum[i].y = __fmaf_rn(v[i].y, share, sum[i].y * old);
            sum[i].z = __fmaf_rn(v[i].z, share, sum[i].z * old);
            sum[i].w = __fmaf_rn(v[i].w, share, sum[i].w * old);
        }
    }
    const int global = mine.first + r;
    T* dst = static_cast<T*>(a.out) + (mine.row0 + global / call.group) * a.out_stride_row + (mine.head * call.group + global % call.group) * a.out_stride_head + d;
    const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float f[8] = {sum[2 * i].x * inv, sum[2 * i].y * inv, sum[2 * i].z * inv, sum[2 * i].w * inv,
                            sum[2 * i + 1].x * inv, sum[2 * i + 1].y * inv, sum[2 * i + 1].z * inv, sum[2 * i + 1].w * inv};
        store8(dst + 8 * i, call.wide != 0, f);
    }
}

template <int D, typename T>
cudaError_t launch_tile_typed(const TileCall& call, int blocks, cudaStream_t stream)
{
    using Shared = TileShared<D>;
    const auto kernel = attention_i8_tile_kernel<D, T>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shared::kBytes);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return e;
    }
    // Groups trade registers within what the block is launched with; with less, one would wait for good.
    static const int registers = [&] {
        cudaFuncAttributes attributes;
        return cudaFuncGetAttributes(&attributes, kernel) == cudaSuccess ? attributes.numRegs : 0;
    }();
    if (registers != Shared::kRegisters) {
        return cudaErrorInvalidDeviceFunction;
    }
    const unsigned grid = static_cast<unsigned>(blocks);
    e = launch_overlapping(attention_i8_plan_kernel<Shared::kRows>, dim3(1), dim3(1024), 0, stream, 1, call);
    note_launch();
    if (e != cudaSuccess) {
        return e;
    }
    e = launch_overlapping(kernel, dim3(grid), dim3(Shared::kThreads), Shared::kBytes, stream, 1, call);
    note_launch();
    if (e != cudaSuccess) {
        return e;
    }
    e = launch_overlapping(attention_i8_tile_join_kernel<D, T>, dim3(grid, D / 16), dim3(Shared::kRows), 0, stream, 1, call);
    note_launch();
    return e;
}

template <int D>
cudaError_t launch_tile_dim(const TileCall& call, int blocks, cudaStream_t stream)
{
    return call.a.float_type == NNB200_FLOAT_F16 ? launch_tile_typed<D, __half>(call, blocks, stream)
                                                 : launch_tile_typed<D, __nv_bfloat16>(call, blocks, stream);
}

constexpr int tile_rows(int64_t dim) { return dim <= 128 ? 256 : 128; }

cudaError_t launch_attention_tile_64(const TileCall& call, int blocks, cudaStream_t stream);
cudaError_t launch_attention_tile_96(const TileCall& call, int blocks, cudaStream_t stream);
cudaError_t launch_attention_tile_128(const TileCall& call, int blocks, cudaStream_t stream);
cudaError_t launch_attention_tile_256(const TileCall& call, int blocks, cudaStream_t stream);

}  // namespace nnb200
