// Writing a key/value cache in 8 bits and reading it back.
//
// A unit of work is one page of one head, keys or values: it has one scale, so whoever quantises its new tokens has to see all
// of them.  A unit belongs to 1, 4, 8 or 16 warps, as many as let each thread hold its 64 values in registers: the values are
// read once, their largest magnitude is taken, and the codes are made from the registers.  Both directions are bound by memory
// (write: 3 bytes a value with f16, read: 3) once there are pages enough; a decode step's write touches one
// token in each of a few hundred units and costs its launch.
//
// The pages a call touches are counted on the device, as their number follows `cu` and `lens`.  With n rows in a
// sequence they are at most n / T + 2 (T tokens a page), so the places of sequence b are those from
// cu[b] / T + 2 b on: disjoint, in order, and their end rows / T + 2 seqs is known to the host.

#include <type_traits>

#include "cache_i8.cuh"

namespace nnb200 {

namespace {

constexpr int kVectors = 8;   // of 8 values, held by a thread

// The tokens of one page and head that a unit has to do with.
struct Unit {
    int page;          // -1: there is none
    int head, values;  // values: 1 for the values' half of the cache
    int row;           // of its first token
    int from, to;      // its tokens' places in the page
    bool begins;       // nothing of the page was there before
    int zero_row, zero_rows;   // rows without a token, which this unit answers for
};

// Warp-collective.
__device__ __forceinline__ Unit find_unit(const nnb200_cache_i8& c, int64_t index, int32_t* error_word)
{
    Unit u;
    u.values = static_cast<int>(index & 1);
    index >>= 1;
    const int tokens = static_cast<int>(c.page_tokens), seqs = static_cast<int>(c.seqs);
    u.head = static_cast<int>(index % c.heads);
    const int64_t place = index / c.heads;
    int b;
    int64_t j;
    if (c.cu == nullptr) {
        const int64_t slots = (c.rows / c.seqs + tokens - 2) / tokens + 1;
        b = static_cast<int>(place / slots);
        j = place - b * slots;
    } else {
        // The last b whose places begin at or before this one, 32 probes at a time.
        const auto begin = [&](int q) { return static_cast<int64_t>(max(c.cu[q], 0) / tokens) + 2 * q; };
        int low = 0, count = seqs;
        while (count > 1) {
            const int step = (count + 31) / 32, at = static_cast<int>(threadIdx.x & 31) * step;
            const bool before = at < count && begin(low + at) <= place;
            const int last = max(__popc(__ballot_sync(0xFFFFFFFFu, before)) - 1, 0) * step;
            low += last;
            count = min(step, count - last);
        }
        b = low;
        j = place - begin(low);
    }
    const SequenceRows s = sequence_rows(c, b);
    const int first = max(s.len - s.n, 0);   // position of the first row that has a token
    const int64_t slot = first / tokens + j;
    u.page = -1;
    u.zero_row = s.row0;
    u.zero_rows = j == 0 ? max(s.n - s.len, 0) : 0;
    if (s.n <= 0 || j < 0 || slot * tokens >= s.len) {
        return u;
    }
    const int start = static_cast<int>(slot) * tokens;
    u.from = max(first - start, 0);
    u.to = min(s.len - start, tokens);
    u.row = s.row0 + (start + u.from) - (s.len - s.n);
    u.begins = u.from == 0 && start >= first;
    u.page = page_at(c, b, static_cast<int>(slot), error_word);
    if (u.page < 0) {   // the tokens' rows have no page
        u.zero_row = u.row;
        u.zero_rows = u.to - u.from;
    }
    return u;
}

template <int WARPS>
__device__ __forceinline__ uint32_t largest_of_unit(uint32_t v)
{
    v = __reduce_max_sync(0xFFFFFFFFu, v);
    if constexpr (WARPS > 1) {
        __shared__ uint32_t part[WARPS];
        if ((threadIdx.x & 31) == 0) {
            part[threadIdx.x / 32] = v;
        }
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) {
            v = max(v, part[i]);
        }
    }
    return v;
}

constexpr int block_threads(int warps) { return warps == 1 ? 128 : 32 * warps; }

// `wide`: rows and heads of the floating side are 16-byte aligned.
template <typename T, int WARPS>
__global__ void __launch_bounds__(block_threads(WARPS))
cache_write_kernel(const nnb200_cache_rows_args a, const int64_t units, const int wide, int32_t* error_word)
{
    previous_kernel_done();
    constexpr int kThreads = 32 * WARPS;
    const nnb200_cache_i8& c = a.cache;
    const int64_t index = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32 : blockIdx.x;
    if (index >= units) {
        return;
    }
    const Unit u = find_unit(c, index, error_word);
    if (u.page < 0) {
        return;
    }
    const int t = threadIdx.x % kThreads;
    const int dim = static_cast<int>(c.dim), per_token = dim / 8;
    const int count = (u.to - u.from) * per_token;
    const int64_t stride_row = u.values ? a.v_stride_row : a.k_stride_row;
    const T* src = static_cast<const T*>(u.values ? a.v : a.k) + u.row * stride_row + u.head * (u.values ? a.v_stride_head : a.k_stride_head);
    float* scale = (u.values ? c.v_scale : c.k_scale) + u.page * c.scale_page_stride + u.head;
    int8_t* codes = static_cast<int8_t*>(u.values ? c.v : c.k) + u.page * c.page_stride + static_cast<int64_t>(u.head) * c.page_tokens * dim;

    const float before = u.begins ? 0.0f : *scale;
    float f[kVectors][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            load8(src + at / per_token * stride_row + at % per_token * 8, wide != 0, f[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = max(top, magnitude_bits(f[i][e]));
            }
        }
    }
    top = largest_of_unit<WARPS>(top);
    // A NaN or an infinity, of these tokens or of those before them, is the page's until it begins anew.
    float after = top >= kInfinityBits ? __uint_as_float(0x7FC00000u) : fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), kLeastCacheScale);
    after = before >= after || before != before ? before : after;
    const float inv = __frcp_rn(after);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            const uint2 q = make_uint2(codes4(f[i][0] * inv, f[i][1] * inv, f[i][2] * inv, f[i][3] * inv),
                                       codes4(f[i][4] * inv, f[i][5] * inv, f[i][6] * inv, f[i][7] * inv));
            *reinterpret_cast<uint2*>(codes + u.from * dim + at * 8) = q;
        }
    }
    if (after == before) {
        return;
    }
    if (t == 0) {
        *scale = after;
    }
    if (!u.begins) {   // the other tokens' codes, in the new scale
        const float ratio = __fdiv_rn(before, after);
        const int skip_from = u.from * per_token, skip_to = u.to * per_token;
        for (int at = t; at < static_cast<int>(c.page_tokens) * per_token; at += kThreads) {
            if (at < skip_from || at >= skip_to) {
                uint2* p = reinterpret_cast<uint2*>(codes + at * 8);
                const uint2 q = *p;
                *p = make_uint2(codes4(code_at(q.x, 0) * ratio, code_at(q.x, 1) * ratio, code_at(q.x, 2) * ratio, code_at(q.x, 3) * ratio),
                                codes4(code_at(q.y, 0) * ratio, code_at(q.y, 1) * ratio, code_at(q.y, 2) * ratio, code_at(q.y, 3) * ratio));
            }
        }
    }
}

template <typename T, int WARPS>
__global__ void __launch_bounds__(block_threads(WARPS))
cache_read_kernel(const nnb200_cache_rows_args a, const int64_t units, const int wide, int32_t* error_word)
{
    previous_kernel_done();
    constexpr int kThreads = 32 * WARPS;
    const nnb200_cache_i8& c = a.cache;
    const int64_t index = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32 : blockIdx.x;
    if (index >= units) {
        return;
    }
    const Unit u = find_unit(c, index, error_word);
    const int t = threadIdx.x % kThreads;
    const int dim = static_cast<int>(c.dim), per_token = dim / 8;
    const int64_t stride_row = u.values ? a.v_stride_row : a.k_stride_row;
    T* dst = static_cast<T*>(u.values ? a.v : a.k) + u.head * (u.values ? a.v_stride_head : a.k_stride_head);
    for (int64_t at = t; at < static_cast<int64_t>(u.zero_rows) * per_token; at += kThreads) {
        const float none[8] = {};
        store8(dst + (u.zero_row + at / per_token) * stride_row + at % per_token * 8, wide != 0, none);
    }
    if (u.page < 0) {
        return;
    }
    const int count = (u.to - u.from) * per_token;
    const float scale = (u.values ? c.v_scale : c.k_scale)[u.page * c.scale_page_stride + u.head];
    const int8_t* codes = static_cast<const int8_t*>(u.values ? c.v : c.k) + u.page * c.page_stride +
                          (static_cast<int64_t>(u.head) * c.page_tokens + u.from) * dim;
    dst += u.row * stride_row;
    uint2 q[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            q[i] = *reinterpret_cast<const uint2*>(codes + at * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = code_at(e < 4 ? q[i].x : q[i].y, e & 3) * scale;
            }
            store8(dst + at / per_token * stride_row + at % per_token * 8, wide != 0, f);
        }
    }
}

template <typename T, int WARPS, bool WRITE>
cudaError_t run_units(const nnb200_cache_rows_args& a, int64_t units, int wide, const DeviceInfo& dev, cudaStream_t stream)
{
    const int64_t blocks = WARPS == 1 ? (units + 3) / 4 : units;
    if (blocks > 0x7FFFFFFF) {
        return cudaErrorInvalidConfiguration;
    }
    if constexpr (WRITE) {
        return launch_overlapping(cache_write_kernel<T, WARPS>, dim3(static_cast<unsigned>(blocks)), dim3(block_threads(WARPS)), 0, stream, 1, a,
                                  units, wide, dev.error_word);
    } else {
        return launch_overlapping(cache_read_kernel<T, WARPS>, dim3(static_cast<unsigned>(blocks)), dim3(block_threads(WARPS)), 0, stream, 1, a,
                                  units, wide, dev.error_word);
    }
}

template <typename T, bool WRITE>
cudaError_t run_typed(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const nnb200_cache_i8& c = a.cache;
    const int64_t each = c.cu == nullptr ? c.rows / c.seqs : c.rows;   // a sequence has at most so many rows
    const int64_t places = c.cu == nullptr ? c.seqs * ((each + c.page_tokens - 2) / c.page_tokens + 1) : c.rows / c.page_tokens + 2 * c.seqs;
    const int64_t units = places * c.heads * 2;
    const int64_t values = (each < c.page_tokens ? each : c.page_tokens) * c.dim;
    const auto aligned = [](const void* p, int64_t s0, int64_t s1) {
        constexpr int64_t kPer = 16 / sizeof(T);
        return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && s0 % kPer == 0 && s1 % kPer == 0;
    };
    const int wide = aligned(a.k, a.k_stride_row, a.k_stride_head) && aligned(a.v, a.v_stride_row, a.v_stride_head) ? 1 : 0;
    constexpr int kPerWarp = 32 * 8 * kVectors;
    return values <= kPerWarp       ? run_units<T, 1, WRITE>(a, units, wide, dev, stream)
           : values <= 4 * kPerWarp ? run_units<T, 4, WRITE>(a, units, wide, dev, stream)
           : values <= 8 * kPerWarp ? run_units<T, 8, WRITE>(a, units, wide, dev, stream)
                                    : run_units<T, 16, WRITE>(a, units, wide, dev, stream);
}

template <bool WRITE>
int run(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const cudaError_t e = a.float_type == NNB200_FLOAT_F32   ? run_typed<float, WRITE>(a, dev, stream)
                          : a.float_type == NNB200_FLOAT_F16 ? run_typed<__half, WRITE>(a, dev, stream)
                                                             : run_typed<__nv_bfloat16, WRITE>(a, dev, stream);
    note_launch();
    return cuda_status(e);
}

}  // namespace

int launch_cache_write_i8(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream) { return run<true>(a, dev, stream); }
int launch_cache_read_i8(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream) { return run<false>(a, dev, stream); }

}  // namespace nnb200
