// Attention over a key/value cache in 8 bits, for few rows a sequence: the mathematics, the split and the kernel.
//
// For a row q of head a, tokens j, K-codes k_j with scale ks_j, V-codes v_j with scale vs_j (one of each for a page):
//
//     t_j = (q . k_j) ks_j c + log2 vs_j       c = scale * log2 e
//     m = max_j t_j,  w_j = 2^(t_j - m) <= 1,  l = sum_j w_j / vs_j,  out = (sum_j w_j v_j) / l
//
// which is the softmax with each block's V scale moved into the exponent: the weights that meet the codes are then at
// most 1 and the largest is 1 whatever the scales are, so that f16 holds them, and one exponential serves both sums.
// One pass over the tokens, with the running maximum; the sums are rescaled only when that has grown by more than 2^8 (f32 rows: 2^2), and the
// lanes of a row compare their maxima only then.  What is subtracted is not m but m - 7 (f32 rows: m - 13), which the quotient takes out
// again: the largest weights lie between 2^7 (2^13) and 2^15, the upper end of f16's range, so that half of its least step, which a weight far below the
// largest may be off by, is 2^-32 (2^-38) of the largest instead of 2^-25.  Of 8192 tokens the first with
// nothing for values and a score 14 higher than the others': with the largest weights at 1 outputs were 1.2e-3 off (f32 rows; f16 in tiles 2.5e-3), now
// 8.6e-7 (3.7e-4, f16's own steps).
//
// A warp takes 16 tokens at a time and is on its own: it copies their codes into its part of shared memory, a few groups ahead
// (16 tokens never leave a page, and one head's share of a page is contiguous), turns bytes into f16
// integers, which is exact, and feeds mma.m16n8k16 with the TOKENS as the 16-row operand: eight query rows (the heads
// of a group, a few proposed tokens) fill the narrow side, nothing is padded to 16 or 128.  The transposition between the
// two products is one movmatrix for 8 x 8 weights.  The order along dim and along the tokens inside an MMA is
// free, and chosen so that every thread's bytes are contiguous; where 16-byte pieces lie in shared memory is, too (code_offset),
// which is why the lanes copy 16 bytes each instead of one lane a block: with the rows as they come, accesses to shared memory took
// three times as long and the kernel 7 to 14 % longer.
//
// Bound by the reading of the codes, 2 D bytes for a token and head, and close behind it by instructions: about 280 of a warp for 16
// tokens of 64 dims and 8 rows, 440 of 128 dims, 50 to 75 more for each 8 rows more.  Measured on one B200: 64 sequences of 128 to 8192 tokens, 8 heads of
// 128, 8 rows: 108 us, 5.1 TB/s (0.79 of the measured copy rate; 98 us where the same call comes again and finds a part in L2); the same call again,
// 64 sequences of 4096 tokens, 8 heads: heads of 64 with 8, 16 and 32 rows 62, 86 and 130 us, heads of 128 with 8 rows 96 us, f32 rows 128; 16 sequences
// behind a window of 4096, 24 rows of 64: 37 us.
//
// The work of all sequences, row tiles and heads is one line of 16-token groups, cut into equal pieces, one for each block, so
// that lengths of any mix keep every SM busy to the end.  A row tile of a head that is cut leaves (m, l, sums) in the
// workspace, in a fixed order of blocks; a second kernel joins them, in that order: results do not depend on timing.
//
// A few row tiles over contexts that cannot be long, all sequences with as many rows, go to a cluster of eight blocks each instead:
// their sums meet in shared memory, without a workspace, a search for one's place or a second kernel.  One sequence of 4096 tokens, 8 heads of
// 128: 9.4 us, with the line and its second kernel 14.8.
#pragma once

#include "cache_i8.cuh"
#include "ptx_pair.cuh"

namespace nnb200 {

constexpr int kRowsThreads = 256; // of the joining kernel's blocks
// Groups that a part of a row tile costs besides its own: queries, the first copies, joining the warps.  With 16, 32 and 64, 8 heads of 128: 64 sequences of
// 128 to 8192 tokens 114, 96 and 98 us, 255 of 16 to 128 and one of 30000 70, 65 and 78, 120 of 100 and 8 of 20000 94, 78 and 95.
constexpr int kRowsCost = 32;
constexpr float kMostWeight = 15.0f;   // log2 of what a weight may be: f16 ends at 65504
// log2 of the largest weight when the sums have just been rescaled.
constexpr float rows_top_weight(bool split) { return split ? 13.0f : 7.0f; }
// From here on the steps of f32 are no longer small against the room above 2^15: the largest weight is 1 there.
constexpr float kCoarse = 4194304.0f;   // 2^22
__device__ __forceinline__ bool is_coarse(float m) { return fabsf(m) >= kCoarse && fabsf(m) < INFINITY; }

// By which power of two a row of bf16 or f32 is divided to be f16: its largest value, of these bits, comes to 2^13 (2^15 at the end of the range), so
// that values as far below it as a loud channel leaves the others keep their bits.  (Queries whose first channel is 2^20 times the others, where keys have
// zeros: 0.027 off with the largest at 1, now 0.0024, bf16's own step; f32 and 2^14: 4.6e-4, now 6.7e-7.)  2^-113 to 2^113: it and its reciprocal are normal.
__device__ __forceinline__ int row_exponent(uint32_t top) { return min(max(static_cast<int>(top >> 23) - 140, -113), 113); }

// A row tile of a head that begins in a block and ends in a later one.  What a block leaves of its sums: [0] the end or the middle of
// one that began in an earlier block, [1] the beginning of one that ends in a later block.
struct RowsPiece {
    int32_t more;    // blocks behind this one that have a part of it; 0: nothing begins here that does not end here
    int32_t head;
    int32_t row0;    // the sequence's first row
    int32_t first;   // of the sequence's rows times heads of the group
    int32_t rows;
    int32_t unused[3];
};

struct RowsPlan {
    int blocks;    // of the first kernel
    int columns;   // query rows of a tile / 8
    int tiles;     // of every sequence, if each row tile of a head has a cluster of its own; else 0
    size_t bytes;  // of the workspace: the pieces, then their sums ([tile rows][dim], m and l of each row)
};

struct RowsCall {
    nnb200_attention_i8_args a;
    int32_t* error_word;
    int group;           // query heads of a key head
    float factor;        // scale * log2 e
    int wide;            // q's rows and heads are 16-byte aligned
    int wide_out;        // out's are, to four values
    int page_shift;      // log2 of the tokens of a page
    int tiles;           // of every sequence, in clusters
    RowsPiece* pieces;   // [blocks]
    float* sums;         // [blocks][2][piece]
};

// One sequence's part of the line.  Its row tiles are all as long: from what its first row sees to its last token.  That is nothing to speak of for the
// few rows that this kernel is for; f32 prompts, which have no other, take up to twice the groups that they see (8192 rows of 32 heads of 128: 9.97 ms), and
// behind a window as many as without one (of 256: 10.4 ms).
struct SequenceWork {
    SequenceRows s;
    int sink_groups, first_group, groups;   // groups of a row tile: the sinks', then those from first_group on; 1 at least
    int tiles;
    int64_t total;   // length: of every item its groups and kRowsCost
};

__device__ __forceinline__ SequenceWork sequence_work(const RowsCall& call, int b, int tile_rows)
{
    const nnb200_attention_i8_args& a = call.a;
    SequenceWork w;
    w.s = sequence_rows(a.cache, b);
    int64_t low = a.window > 0 ? static_cast<int64_t>(w.s.len) - w.s.n - a.window + 1 : 0;
    low = low < 0 ? 0 : low;
    w.first_group = static_cast<int>(low < w.s.len ? low : w.s.len) / 16;
    const int sinks = static_cast<int>(a.sinks < w.s.len ? a.sinks : w.s.len);
    w.sink_groups = a.window > 0 ? min((sinks + 15) / 16, w.first_group) : 0;
    w.groups = max(w.sink_groups + (w.s.len + 15) / 16 - w.first_group, 1);
    w.tiles = (w.s.n * call.group + tile_rows - 1) / tile_rows;
    w.total = static_cast<int64_t>(a.cache.heads) * w.tiles * (w.groups + kRowsCost);
    return w;
}

// ---- pieces of the MMAs ---------------------------------------------------------------------

// Bytes of a word (signed) as f16 pairs: (0, 1) and (2, 3).  0x6400 | u is 1024 + u; u = byte + 128.
__device__ __forceinline__ uint32_t half2_minus(uint32_t v)
{
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void codes_to_half(uint32_t word, uint32_t& low, uint32_t& high)
{
    const uint32_t u = word ^ 0x80808080u;
    low = half2_minus(__byte_perm(u, 0x64646464u, 0x4140));
    high = half2_minus(__byte_perm(u, 0x64646464u, 0x4342));
}
// Bytes i of x and of y as the pair (x_i, y_i).
__device__ __forceinline__ void codes_to_half_pairs(uint32_t x, uint32_t y, uint32_t (&p)[4])
{
    x ^= 0x80808080u;
    y ^= 0x80808080u;
    const uint32_t a = __byte_perm(x, y, 0x5140), b = __byte_perm(x, y, 0x7362);
    p[0] = half2_minus(__byte_perm(a, 0x64646464u, 0x4140));
    p[1] = half2_minus(__byte_perm(a, 0x64646464u, 0x4342));
    p[2] = half2_minus(__byte_perm(b, 0x64646464u, 0x4140));
    p[3] = half2_minus(__byte_perm(b, 0x64646464u, 0x4342));
}

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// WORDS 32-bit words from shared memory, p aligned to the largest power of two that divides their bytes (up to 16).
template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[WORDS])
{
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (WORDS % 2 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        }
    }
}

// Where a token's 16 codes number `chunk` lie in a stage.  A product takes a chunk of 8 x 4 lanes at a time: for keys each of eight
// tokens' chunks of four places, for values the chunks of eight places of each of four tokens.  In rows one behind the other these are in
// the same banks (heads of 128: 2 and 4 times over); so the chunks of a row change places by the row's number, and each
// access takes as long as its bytes.  Heads of 96, whose rows begin in different banks, stay as they are.
template <int D>
__device__ __forceinline__ int code_offset(int row, int chunk)
{
    if constexpr (D == 64) {
        return (row >> 1) * 128 + (((row & 1) * 4 + chunk) ^ (row & 6)) * 16;
    } else if constexpr (D == 128) {
        return row * 128 + (chunk ^ (row & 7)) * 16;
    } else if constexpr (D == 256) {
        return row * 256 + (chunk >> 3) * 128 + ((chunk & 7) ^ (chunk >> 3) ^ ((row & 1) << 1 | (row >> 1 & 1) | (row & 4))) * 16;
    } else {
        return row * D + chunk * 16;
    }
}

// Four words, or eight 16-bit values, as they are; `wide`: the address is 16-byte aligned.
__device__ __forceinline__ uint4 four_words(const uint32_t* p, bool wide) { return wide ? *reinterpret_cast<const uint4*>(p) : make_uint4(p[0], p[1], p[2], p[3]); }
__device__ __forceinline__ uint4 eight_of(const uint16_t* p, bool wide)
{
    if (wide) {
        return *reinterpret_cast<const uint4*>(p);
    }
    const auto two = [&](int i) { return static_cast<uint32_t>(p[i]) | static_cast<uint32_t>(p[i + 1]) << 16; };
    return make_uint4(two(0), two(2), two(4), two(6));
}

template <typename T>
__device__ __forceinline__ void store_four(T* p, bool wide, float4 v)
{
    if (!wide) {
        p[0] = from_float<T>(v.x);
        p[1] = from_float<T>(v.y);
        p[2] = from_float<T>(v.z);
        p[3] = from_float<T>(v.w);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
    }
}
// This lane's part of a token's keys (those of `row`, dims [c D / 4, + D / 4)) and values (dims [g D / 8, + D / 8)).
template <int D>
__device__ __forceinline__ void load_keys(const uint8_t* stage, int row, int c, uint32_t (&w)[D / 16])
{
    if constexpr (D == 96) {
        load_words(stage + row * D + c * (D / 4), w);
    } else {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(stage + code_offset<D>(row, c * (D / 64) + i));
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}
template <int D>
__device__ __forceinline__ void load_values(const uint8_t* stage, int row, int g, uint32_t (&w)[D / 32])
{
    if constexpr (D == 96) {
        load_words(stage + row * D + g * (D / 8), w);
    } else if constexpr (D == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(stage + code_offset<D>(row, g >> 1) + (g & 1) * 8);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(stage + code_offset<D>(row, g * (D / 128) + i));
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}

// sum / total, or zeros where nothing was seen.
__device__ __forceinline__ void store_row(const RowsCall& call, int64_t i, float4 sum, float total)
{
    const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    const float4 v = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
    if (call.a.float_type == NNB200_FLOAT_F32) {
        store_four(static_cast<float*>(call.a.out) + i, call.wide_out != 0, v);
    } else if (call.a.float_type == NNB200_FLOAT_F16) {
        store_four(static_cast<__half*>(call.a.out) + i, call.wide_out != 0, v);
    } else {
        store_four(static_cast<__nv_bfloat16*>(call.a.out) + i, call.wide_out != 0, v);
    }
}

// (For the tiles' kernel.)  Every lane polls: the data behind the barrier is then every lane's.  Without a hint how long to sleep, which costs a
// hundred cycles on a barrier that is all but ready; within the limit that mbar_wait has.
__device__ __forceinline__ bool wait_every_lane(uint64_t* bar, uint32_t parity, volatile int* abort_flag)
{
    bool done = mbar_try_wait(bar, parity);
    if (!__all_sync(0xFFFFFFFFu, done)) {
        const long long t0 = clock64();
        bool give_up = false;
        for (uint32_t spins = 1; !done && !give_up; ++spins) {
            done = mbar_try_wait(bar, parity);
            if ((spins & 63u) == 0) {
                if (*abort_flag == 0 && clock64() - t0 > kWaitLimitCycles) {
                    *abort_flag = 1;
                }
                give_up = *abort_flag != 0;
            }
        }
        return __all_sync(0xFFFFFFFFu, done);
    }
    return true;
}

// What a warp's queries and sums take, in values a lane has 32nd parts of; and by that blocks on an SM and warps of a block: 16 warps with
// 128 registers a thread, 12 with 168 or 8 with 255.  (24 rows of heads of 64, 16 sequences behind a window of 4096: 8 warps 41 us, 10
// or 12, whose registers do not hold everything, 43 to 44.)
constexpr int rows_weight(int64_t dim, int columns, bool split) { return static_cast<int>(dim) * columns * (split ? 3 : 2) / 2; }
constexpr int rows_blocks(int64_t dim, int columns, bool split) { return columns == 1 && rows_weight(dim, columns, split) <= 128 ? 2 : 1; }
constexpr int rows_warps(int64_t dim, int columns, bool split)
{
    return rows_blocks(dim, columns, split) == 1 && rows_weight(dim, columns, split) <= 128 ? 12 : 8;
}

// At these the sums all but fit the registers (of a thread's 255, bytes that are spilled, on the line and in clusters: heads of 256 with 16 rows 308 and
// 188, of 96 with 32 rows 200 and 12, of 128 with 24 rows 8 and 0, all others none); with eight rows more they do not.
constexpr int rows_most_columns(int64_t dim, bool split) { return split ? (dim > 128 ? 1 : 2) : dim > 128 ? 2 : dim > 96 ? 3 : 4; }

template <int D, int NT, bool SPLIT>
struct RowsShared {   // bytes of the warps' rings, which hold the warps' sums when a piece is joined
    static constexpr int kWarps = rows_warps(D, NT, SPLIT);
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kStageBytes = 2 * 16 * D;
    static constexpr int kJoinBytes = kWarps * 8 * NT * D * 4;
    static constexpr int kWanted = (rows_blocks(D, NT, SPLIT) == 2 ? 96 : 192) * 1024;
    // Groups on their way or at work, of each warp.
    static constexpr int kStages = kWanted / (kWarps * kStageBytes) > 8 ? 8 : kWanted / (kWarps * kStageBytes);
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kSumBytes = 8 * NT * (D + 2) * 4;   // in a cluster: of a block
    static constexpr int kBytes = (kRing > kJoinBytes ? kRing : kJoinBytes);
    static constexpr int kClusterBytes = kRing > kJoinBytes + kSumBytes ? kRing : kJoinBytes + kSumBytes;
    static_assert(kStages >= 2 && rows_blocks(D, NT, SPLIT) * kBytes <= 200 * 1024, "ring");
};

struct StageScales {
    float k, v_log2, v_inv;
    int there;
};

constexpr int kRowsCluster = 8;

// Of numbers that are not negative: by 32-bit arithmetic where they allow it, which takes a fraction of the time.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b)
{
    return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

__device__ __forceinline__ float4 ld_shared_cluster_f32x4(uint32_t cluster_addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ float ld_shared_cluster_float(uint32_t cluster_addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

template <int D, int NT, bool SPLIT, bool CLUSTER>
__global__ void __launch_bounds__(RowsShared<D, NT, SPLIT>::kThreads, rows_blocks(D, NT, SPLIT))
attention_i8_rows_kernel(const RowsCall call)
{
    using Shared = RowsShared<D, NT, SPLIT>;
    constexpr int kStages = Shared::kStages, kWarps = Shared::kWarps, kThreads = Shared::kThreads;
    constexpr int kTile = 8 * NT;
    constexpr int kParts = SPLIT ? 2 : 1;
    constexpr float kTop = rows_top_weight(SPLIT);
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ StageScales scales[kWarps][kStages];
    __shared__ float join_m[kWarps][kTile], join_l[kWarps][kTile];
    __shared__ int64_t scan[kWarps + 1];
    __shared__ int64_t found_base;
    __shared__ int64_t cut[3];   // of the line: blocks, the least share of one, how many groups are over
    __shared__ int found_seq;

    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int g = lane / 4, c = lane & 3;
    previous_kernel_done();
    const nnb200_attention_i8_args& a = call.a;
    const int seqs = static_cast<int>(a.cache.seqs);

    int seq = 0;
    int64_t base = 0, at = 0, end = 1;
    const auto start_of = [&](int64_t block) { return cut[1] * block + quotient(cut[2] * block, cut[0]); };
    if constexpr (!CLUSTER) {
        // The line's length, and the sequence in which this block's piece begins.
        const auto block_sum_before = [&](int64_t v, int64_t& total) {   // of the threads before this one
            int64_t up = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t other = __shfl_up_sync(0xFFFFFFFFu, up, o);
                up += lane >= o ? other : 0;
            }
            __syncthreads();
            if (lane == 31) {
                scan[warp] = up;
            }
            __syncthreads();
            int64_t before = up - v;
            total = 0;
            for (int i = 0; i < kWarps; ++i) {
                before += i < warp ? scan[i] : 0;
                total += scan[i];
            }
            return before;
        };
        // Up to so many threads: everyone has its own sequence's place at once.
        int64_t line = 0, own = 0, own_before = 0;
        for (int b0 = 0; b0 < seqs; b0 += kThreads) {
            const int b = b0 + static_cast<int>(threadIdx.x);
            int64_t total;
            own = b < seqs ? sequence_work(call, b, kTile).total : 0;
            own_before = line + block_sum_before(own, total);
            line += total;
        }
        // Two groups a warp for a block, of eight, where there is no more to do: latency is what counts then.
        const int64_t share_at_least = 16;
        const int64_t most = (line + share_at_least - 1) / share_at_least;
        const int64_t blocks = most < gridDim.x ? most : gridDim.x;
        if (threadIdx.x == 0) {
            call.pieces[blockIdx.x].more = 0;
        }
        if (static_cast<int64_t>(blockIdx.x) >= blocks) {
            return;
        }
        if (threadIdx.x == 0) {
            cut[0] = blocks;
            cut[1] = quotient(line, blocks);
            cut[2] = line - cut[1] * blocks;
        }
        __syncthreads();
        at = start_of(blockIdx.x);
        end = start_of(blockIdx.x + 1);
        if (seqs <= kThreads) {
            if (own_before <= at && at < own_before + own) {
                found_seq = threadIdx.x;
                found_base = own_before;
            }
        } else {
            int64_t base = 0;
            for (int b0 = 0; b0 < seqs; b0 += kThreads) {
                const int b = b0 + static_cast<int>(threadIdx.x);
                own = b < seqs ? sequence_work(call, b, kTile).total : 0;
                int64_t total;
                own_before = base + block_sum_before(own, total);
                if (own_before <= at && at < own_before + own) {
                    found_seq = b;
                    found_base = own_before;
                }
                base += total;
            }
        }
        __syncthreads();
        seq = found_seq;
        base = found_base;
    }

    uint32_t issue_slot = 0, slot = 0;   // of the ring: the next to fill, the next to take
    uint8_t* const my_ring = ring + warp * kStages * Shared::kStageBytes;

    while (at < end) {
        SequenceWork work;
        int head, tile, off, count, length = 0;
        int64_t item = 0;
        if constexpr (CLUSTER) {
            // Sequence by sequence, tile by tile, head by head; as many tiles in each.
            const int cluster = static_cast<int>(blockIdx.x) / kRowsCluster, rank = static_cast<int>(blockIdx.x) % kRowsCluster;
            const int heads = static_cast<int>(a.cache.heads), each = cluster / heads;
            head = cluster - each * heads;
            seq = each / call.tiles;
            tile = each - seq * call.tiles;
            work = sequence_work(call, seq, kTile);
            off = static_cast<int>(static_cast<int64_t>(work.groups) * rank / kRowsCluster);
            count = static_cast<int>(static_cast<int64_t>(work.groups) * (rank + 1) / kRowsCluster) - off;
            at = end;
        } else {
            work = sequence_work(call, seq, kTile);
            if (at >= base + work.total) {
                base += work.total;
                ++seq;
                continue;
            }
            length = work.groups + kRowsCost;
            item = quotient(at - base, length);
            const int from = static_cast<int>(at - base - item * length);
            const int to = static_cast<int>(from + (end - at) < length ? from + (end - at) : length);
            at += to - from;
            off = max(from - kRowsCost, 0);
            count = max(to - kRowsCost, 0) - off;
            if (count <= 0) {
                continue;
            }
            head = static_cast<int>(quotient(item, work.tiles));
            tile = static_cast<int>(item - static_cast<int64_t>(head) * work.tiles);
        }

        const int rows = min(kTile, work.s.n * call.group - tile * kTile);
        const int first_pos = work.s.len - work.s.n;

        // This warp's groups of the piece: off + warp, off + warp + kWarps, ...
        const int mine = count > warp ? (count - warp + kWarps - 1) / kWarps : 0;
        const auto group_of = [&](int i) {
            const int idx = off + warp + i * kWarps;
            return idx < work.sink_groups ? idx : idx - work.sink_groups + work.first_group;
        };
        // Lane i has the i-th of 32 groups at a time: where its codes lie (-1: nowhere), its scales; and asks for them when their turn comes.
        int64_t ahead = -1;
        float ahead_k = 0.0f, ahead_log2 = 0.0f, ahead_inv = 0.0f;
        const auto issue = [&](int i) {
            if ((i & 31) == 0) {
                ahead = -1;
                const int key0 = group_of(i + lane) * 16;
                if (i + lane < mine && key0 < work.s.len) {
                    const int page = page_at(a.cache, seq, key0 >> call.page_shift, call.error_word);
                    if (page >= 0) {
                        const int64_t s = page * a.cache.scale_page_stride + head;
                        const float vs = a.cache.v_scale[s], sure = vs < kLeastCacheScale ? kLeastCacheScale : vs;
                        ahead_k = a.cache.k_scale[s];
                        ahead_log2 = log2f(sure);
                        ahead_inv = __fdiv_rn(1.0f, sure);
                        ahead = page * a.cache.page_stride +
                                ((static_cast<int64_t>(head) << call.page_shift) + (key0 & ((1 << call.page_shift) - 1))) * D;
                    }
                }
            }
            const int64_t from = __shfl_sync(0xFFFFFFFFu, ahead, i & 31);
            if (lane == (i & 31)) {
                scales[warp][issue_slot] = StageScales{ahead_k, ahead_log2, ahead_inv, ahead >= 0 ? 1 : 0};
            }
            if (from >= 0) {
                uint8_t* const dst = my_ring + issue_slot * Shared::kStageBytes;
                const uint8_t* const k = static_cast<const uint8_t*>(a.cache.k) + from + lane * 16;
                const uint8_t* const v = static_cast<const uint8_t*>(a.cache.v) + from + lane * 16;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const int to = code_offset<D>((j * 32 + lane) / (D / 16), (j * 32 + lane) % (D / 16));
                    cp_async_16(dst + to, k + j * 512, 16);
                    cp_async_16(dst + 16 * D + to, v + j * 512, 16);
                }
            }
            issue_slot = issue_slot + 1 == kStages ? 0 : issue_slot + 1;
        };
        // The query rows are asked for before the pages are looked up: this thread's part of row 8 nt + g, dims [c D / 4, + D / 4).
        uint4 raw[NT][SPLIT ? D / 16 : D / 32];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g, global = tile * kTile + r, token = global / call.group;
            const int64_t src = (work.s.row0 + token) * a.q_stride_row + (head * call.group + global - token * call.group) * a.q_stride_head + c * (D / 4);
#pragma unroll
            for (int i = 0; i < (SPLIT ? D / 16 : D / 32); ++i) {
                raw[nt][i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < rows) {
                    if constexpr (SPLIT) {
                        raw[nt][i] = four_words(static_cast<const uint32_t*>(a.q) + src + 4 * i, call.wide != 0);
                    } else {
                        raw[nt][i] = eight_of(static_cast<const uint16_t*>(a.q) + src + 8 * i, call.wide != 0);
                    }
                }
            }
        }
        // A group is committed for every turn, also without copies: what is waited for is then always the oldest of kStages.
        for (int i = 0; i < kStages; ++i) {
            if (i < mine) {
                issue(i);
            }
            cp_async_commit();
        }
        // In f16, bf16 and f32 scaled by a power of two.
        uint32_t q[NT][kParts][D / 16][2];
        float factor[NT][2];    // of the columns 2 c and 2 c + 1
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float v[D / 4];
#pragma unroll
            for (int i = 0; i < (SPLIT ? D / 16 : D / 32); ++i) {
                const uint32_t w[4] = {raw[nt][i].x, raw[nt][i].y, raw[nt][i].z, raw[nt][i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (SPLIT) {
                        v[4 * i + k] = __uint_as_float(w[k]);
                    } else if (a.float_type == NNB200_FLOAT_F16) {
                        unpack2<__half>(w[k], v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
                    } else {
                        unpack2<__nv_bfloat16>(w[k], v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
                    }
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
                top = max(top, magnitude_bits(v[i]));
            }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = a.float_type == NNB200_FLOAT_F16 ? 0 : row_exponent(top);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * call.factor;
#pragma unroll
            for (int w = 0; w < D / 16; ++w) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const float x = v[4 * w + 2 * p] * down, y = v[4 * w + 2 * p + 1] * down;
                    const __half2 h = __floats2half2_rn(x, y);
                    q[nt][0][w][p] = *reinterpret_cast<const uint32_t*>(&h);
                    if constexpr (SPLIT) {
                        const float2 f = __half22float2(h);
                        q[nt][kParts - 1][w][p] = pack2<__half>(x - f.x, y - f.y);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                factor[nt][j] = __shfl_sync(0xFFFFFFFFu, up, (2 * c + j) * 4);
                const int row = tile * kTile + nt * 8 + 2 * c + j;
                pos[nt][j] = a.causal != 0 ? first_pos + min(row, tile * kTile + rows - 1) / call.group : 0x7FFFFFFF;
            }
        }
        const int least_pos = a.causal != 0 ? first_pos + tile * kTile / call.group : 0x7FFFFFFF;
        const int most_pos = a.causal != 0 ? first_pos + (tile * kTile + rows - 1) / call.group : 0x7FFFFFFF;

        float m[NT][2], l[NT][2], o[NT][D / 16][4];   // m: the maximum less kTop
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
            }
        }

        for (int i = 0; i < mine; ++i) {
            cp_async_wait_group<kStages - 1>();
            __syncwarp();
            const StageScales sc = scales[warp][slot];
            if (sc.there != 0) {
                const uint8_t* kp = my_ring + slot * Shared::kStageBytes;
                const uint8_t* vp = kp + 16 * D;
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
                }
                {
                    uint32_t x[D / 16], y[D / 16];
                    load_keys<D>(kp, g, c, x);
                    load_keys<D>(kp + 8 * D, g, c, y);
#pragma unroll
                    for (int w = 0; w < D / 16; ++w) {
                        uint32_t f[4];
                        codes_to_half(x[w], f[0], f[2]);
                        codes_to_half(y[w], f[1], f[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int p = 0; p < kParts; ++p) {
                                mma_16x8x16(s[nt], f[0], f[1], f[2], f[3], q[nt][p][w][0], q[nt][p][w][1]);
                            }
                        }
                    }
                }
                const int key0 = group_of(i) * 16;
                const bool all_seen = key0 + 15 < work.s.len && key0 + 15 <= least_pos &&
                                      (a.window == 0 || key0 > most_pos - a.window || key0 + 15 < a.sinks);
                uint32_t pb[NT][kParts][2];
                // Element e of a tile of eight rows: token g (e < 2) or g + 8, column 2 c + (e & 1).
                float x[NT][4], largest = -INFINITY;
                uint32_t hidden = 0;   // a bit an element
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float kf[2] = {sc.k * factor[nt][0], sc.k * factor[nt][1]};
                    const float less[2] = {sc.v_log2 - m[nt][0], sc.v_log2 - m[nt][1]};   // +infinity until a row has seen something
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[nt][e] = __fmaf_rn(s[nt][e], kf[e & 1], less[e & 1]);
                    }
                }
                if (!all_seen) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + g + (e < 2 ? 0 : 8), at_pos = pos[nt][e & 1];
                            const bool seen = key < work.s.len && key <= at_pos && (a.window == 0 || key > at_pos - a.window || key < a.sinks);
                            x[nt][e] = seen ? x[nt][e] : -INFINITY;
                            hidden |= seen ? 0u : 1u << (nt * 4 + e);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    largest = fmaxf(largest, fmaxf(fmaxf(x[nt][0], x[nt][1]), fmaxf(x[nt][2], x[nt][3])));
                }
                if (__any_sync(0xFFFFFFFFu, largest > kMostWeight)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float alpha[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float kf = sc.k * factor[nt][j];
                            const float t0 = (hidden >> (nt * 4 + j) & 1) == 0 ? __fmaf_rn(s[nt][j], kf, sc.v_log2) : -INFINITY;
                            const float t1 = (hidden >> (nt * 4 + j + 2) & 1) == 0 ? __fmaf_rn(s[nt][j + 2], kf, sc.v_log2) : -INFINITY;
                            float top = fmaxf(t0, t1);
                            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                            const float next = fmaxf(m[nt][j], is_coarse(top) ? top : top - kTop), safe = next == -INFINITY ? 0.0f : next;
                            alpha[j] = exp2_fast(m[nt][j] - safe);
                            m[nt][j] = next;
                            l[nt][j] *= alpha[j];
                            x[nt][j] = t0 - safe;
                            x[nt][j + 2] = t1 - safe;
                        }
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
                            o[nt][d][0] *= alpha[0];
                            o[nt][d][1] *= alpha[1];
                            o[nt][d][2] *= alpha[0];
                            o[nt][d][3] *= alpha[1];
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        x[nt][j] = exp2_fast(x[nt][j]);
                        x[nt][j + 2] = exp2_fast(x[nt][j + 2]);
                        const float both = x[nt][j] + x[nt][j + 2];
                        l[nt][j] += both == 0.0f ? 0.0f : both * sc.v_inv;   // (not 0 times what a block that is masked has for a scale)
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const __half2 h = __floats2half2_rn(x[nt][2 * j], x[nt][2 * j + 1]);
                        pb[nt][0][j] = transposed_8x8(*reinterpret_cast<const uint32_t*>(&h));
                        if constexpr (SPLIT) {
                            const float2 f = __half22float2(h);
                            pb[nt][kParts - 1][j] = transposed_8x8(pack2<__half>(x[nt][2 * j] - f.x, x[nt][2 * j + 1] - f.y));
                        }
                    }
                }
                uint32_t v0[D / 32], v1[D / 32], v2[D / 32], v3[D / 32];
                load_values<D>(vp, 2 * c, g, v0);
                load_values<D>(vp, 2 * c + 1, g, v1);
                load_values<D>(vp + 8 * D, 2 * c, g, v2);
                load_values<D>(vp + 8 * D, 2 * c + 1, g, v3);
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    uint32_t e0[4], e1[4];
                    codes_to_half_pairs(v0[w], v1[w], e0);
                    codes_to_half_pairs(v2[w], v3[w], e1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int p = 0; p < kParts; ++p) {
                            mma_16x8x16(o[nt][2 * w], e0[0], e0[1], e1[0], e1[1], pb[nt][p][0], pb[nt][p][1]);
                            mma_16x8x16(o[nt][2 * w + 1], e0[2], e0[3], e1[2], e1[3], pb[nt][p][0], pb[nt][p][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (i + kStages < mine) {
                issue(i + kStages);
            }
            cp_async_commit();
            slot = slot + 1 == kStages ? 0 : slot + 1;
        }
        // The warps' sums, joined through the ring: every copy into it has been taken.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[nt][j] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][j], 4);
                l[nt][j] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][j], 8);
                l[nt][j] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][j], 16);
                if (g == 0) {
                    join_m[warp][nt * 8 + 2 * c + j] = m[nt][j];
                    join_l[warp][nt * 8 + 2 * c + j] = l[nt][j];
                }
            }
        }
        __syncthreads();
        float* join_o = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                float* dst = join_o + (warp * kTile + nt * 8 + 2 * c) * D + g * (D / 8) + 2 * i;
                *reinterpret_cast<float2*>(dst) = make_float2(o[nt][i][0], o[nt][i][2]);
                *reinterpret_cast<float2*>(dst + D) = make_float2(o[nt][i][1], o[nt][i][3]);
            }
        }
        __syncthreads();
        const bool begins = off == 0, ends = off + count == work.groups;   // (of no account in a cluster)
        const int which = begins ? 1 : 0;
        float* piece = call.sums + (2 * static_cast<int64_t>(blockIdx.x) + which) * (kTile * (D + 2));
        for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float top = join_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) {
                top = fmaxf(top, join_m[w][r]);
            }
            const float safe = top == -INFINITY ? 0.0f : top;
            float total = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float share = exp2_fast(join_m[w][r] - safe);
                const float4 v = *reinterpret_cast<const float4*>(join_o + (w * kTile + r) * D + d);
                total = __fmaf_rn(join_l[w][r], share, total);
                sum.x = __fmaf_rn(v.x, share, sum.x);
                sum.y = __fmaf_rn(v.y, share, sum.y);
                sum.z = __fmaf_rn(v.z, share, sum.z);
                sum.w = __fmaf_rn(v.w, share, sum.w);
            }
            if constexpr (CLUSTER) {
                float* mine_of = join_o + kWarps * kTile * D;   // behind the warps' sums
                *reinterpret_cast<float4*>(mine_of + r * D + d) = sum;
                if (d == 0) {
                    mine_of[kTile * D + r] = top;
                    mine_of[kTile * D + kTile + r] = total;
                }
            } else if (begins && ends) {
                const int global = tile * kTile + r;
                store_row(call, (work.s.row0 + global / call.group) * a.out_stride_row + (head * call.group + global % call.group) * a.out_stride_head + d, sum, total);
            } else {
                *reinterpret_cast<float4*>(piece + r * D + d) = sum;
                if (d == 0) {
                    piece[kTile * D + r] = top;
                    piece[kTile * D + kTile + r] = total;
                }
            }
        }
        if constexpr (CLUSTER) {
            // Every block takes an eighth of the row tile's sums, out of all eight.
            __syncwarp();
            cluster_sync_all();
            const uint32_t rank = cluster_cta_rank(), here = smem_u32(join_o + kWarps * kTile * D);
            for (int i = static_cast<int>(rank * kThreads + threadIdx.x); i < rows * (D / 4); i += kRowsCluster * kThreads) {
                const int r = i / (D / 4), d = i % (D / 4) * 4;
                float4 v[kRowsCluster];
                float m_of[kRowsCluster], l_of[kRowsCluster], top = -INFINITY;
#pragma unroll
                for (int k = 0; k < kRowsCluster; ++k) {
                    const uint32_t there = map_to_cta(here, k);
                    v[k] = ld_shared_cluster_f32x4(there + static_cast<uint32_t>(r * D + d) * 4);
                    m_of[k] = ld_shared_cluster_float(there + static_cast<uint32_t>(kTile * D + r) * 4);
                    l_of[k] = ld_shared_cluster_float(there + static_cast<uint32_t>(kTile * D + kTile + r) * 4);
                    top = fmaxf(top, m_of[k]);
                }
                const float safe = top == -INFINITY ? 0.0f : top;
                float total = 0.0f;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < kRowsCluster; ++k) {
                    const float part = exp2_fast(m_of[k] - safe);
                    total = __fmaf_rn(l_of[k], part, total);
                    sum.x = __fmaf_rn(v[k].x, part, sum.x);
                    sum.y = __fmaf_rn(v[k].y, part, sum.y);
                    sum.z = __fmaf_rn(v[k].z, part, sum.z);
                    sum.w = __fmaf_rn(v[k].w, part, sum.w);
                }
                const int global = tile * kTile + r;
                store_row(call, (work.s.row0 + global / call.group) * a.out_stride_row + (head * call.group + global % call.group) * a.out_stride_head + d, sum, total);
            }
            __syncwarp();
            cluster_sync_all();   // nobody leaves while his sums are read
            return;
        }
        if (begins && !ends && threadIdx.x == 0) {
            // The block in which it ends: the one that has the item's last place on the line.
            const int64_t place = base + (item + 1) * length - 1;
            int64_t block = quotient(place, cut[1] + 1);   // or a later one
            while (start_of(block + 1) <= place) {
                ++block;
            }
            call.pieces[blockIdx.x] = RowsPiece{static_cast<int32_t>(block - blockIdx.x), head, work.s.row0, tile * kTile, rows, {}};
        }
        __syncthreads();
    }
}

// Joins the pieces of the row tiles that were cut, one block for each block of the first kernel in which one begins.
template <int D, int TILE>
__global__ void __launch_bounds__(kRowsThreads) attention_i8_join_kernel(const RowsCall call)
{
    previous_kernel_done();
    const RowsPiece mine = call.pieces[blockIdx.x];
    const int more = mine.more, rows = mine.rows;
    if (more == 0) {
        return;
    }
    const nnb200_attention_i8_args& a = call.a;
    constexpr int64_t kPiece = TILE * (D + 2);
    const float* first = call.sums + (2 * static_cast<int64_t>(blockIdx.x) + 1) * kPiece;
    const float* rest = first + kPiece;   // and every second piece from there
    for (int i = threadIdx.x; i < rows * (D / 4); i += kRowsThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float top = first[TILE * D + r], total = first[TILE * D + TILE + r];
        float4 sum = *reinterpret_cast<const float4*>(first + r * D + d);
        constexpr int kAtOnce = 8;
        for (int p0 = 0; p0 < more; p0 += kAtOnce) {
            float m[kAtOnce], l[kAtOnce];
            float4 v[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float* piece = rest + min(p0 + k, more - 1) * 2 * kPiece;
                m[k] = p0 + k < more ? piece[TILE * D + r] : -INFINITY;
                l[k] = piece[TILE * D + TILE + r];
                v[k] = *reinterpret_cast<const float4*>(piece + r * D + d);
            }
            float next = top;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                next = fmaxf(next, m[k]);
            }
            const float safe = next == -INFINITY ? 0.0f : next, old = exp2_fast(top - safe);
            top = next;
            total *= old;
            sum = make_float4(sum.x * old, sum.y * old, sum.z * old, sum.w * old);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (p0 + k < more) {
                    const float share = exp2_fast(m[k] - safe);
                    total = __fmaf_rn(l[k], share, total);
                    sum.x = __fmaf_rn(v[k].x, share, sum.x);
                    sum.y = __fmaf_rn(v[k].y, share, sum.y);
                    sum.z = __fmaf_rn(v[k].z, share, sum.z);
                    sum.w = __fmaf_rn(v[k].w, share, sum.w);
                }
            }
        }
        const int global = mine.first + r;
        store_row(call, (mine.row0 + global / call.group) * a.out_stride_row + (mine.head * call.group + global % call.group) * a.out_stride_head + d, sum, total);
    }
}

template <int D, int NT, bool SPLIT, bool CLUSTER>
cudaError_t launch_rows(const RowsCall& call, int blocks, cudaStream_t stream)
{
    using Shared = RowsShared<D, NT, SPLIT>;
    constexpr int kBytes = CLUSTER ? Shared::kClusterBytes : Shared::kBytes;
    const auto kernel = attention_i8_rows_kernel<D, NT, SPLIT, CLUSTER>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return e;
    }
    e = launch_overlapping(kernel, dim3(static_cast<unsigned>(blocks)), dim3(Shared::kThreads), kBytes, stream, CLUSTER ? kRowsCluster : 1, call);
    note_launch();
    if (e != cudaSuccess || CLUSTER) {
        return e;
    }
    e = launch_overlapping(attention_i8_join_kernel<D, 8 * NT>, dim3(static_cast<unsigned>(blocks)), dim3(kRowsThreads), 0, stream, 1, call);
    note_launch();
    return e;
}

template <int D, bool SPLIT, int NT = 1>
cudaError_t launch_rows_columns(const RowsCall& call, int columns, int blocks, cudaStream_t stream)
{
    if constexpr (NT < rows_most_columns(D, SPLIT)) {
        if (columns > NT) {
            return launch_rows_columns<D, SPLIT, NT + 1>(call, columns, blocks, stream);
        }
    }
    return call.tiles > 0 ? launch_rows<D, NT, SPLIT, true>(call, blocks, stream) : launch_rows<D, NT, SPLIT, false>(call, blocks, stream);
}

template <int D>
cudaError_t launch_rows_dim(const RowsCall& call, int columns, int blocks, cudaStream_t stream)
{
    return call.a.float_type == NNB200_FLOAT_F32 ? launch_rows_columns<D, true>(call, columns, blocks, stream)
                                                 : launch_rows_columns<D, false>(call, columns, blocks, stream);
}

// One translation unit for each head size.
cudaError_t launch_attention_rows_64(const RowsCall& call, int columns, int blocks, cudaStream_t stream);
cudaError_t launch_attention_rows_96(const RowsCall& call, int columns, int blocks, cudaStream_t stream);
cudaError_t launch_attention_rows_128(const RowsCall& call, int columns, int blocks, cudaStream_t stream);
cudaError_t launch_attention_rows_256(const RowsCall& call, int columns, int blocks, cudaStream_t stream);

}  // namespace nnb200
