// Writing a key/value cache in 8 bits and reading it back.
//
// A unit of work is one page of one head, keys or values: it has one scale, so whoever quantises its new tokens has to see all
// of them.  A unit belongs to 1, 4, 8 or 16 warps, as many as let each thread hold its 64 values in registers: the values are
// read once, their largest magnitude is taken, and the codes are made from the registers.  Both directions are bound by memory
// (write: 3 bytes a value with f16, read: 3) once there are pages enough, and by the chain of loads before a unit's values are
// found (sequence, page, values) when there are few; a decode step's write touches one token in each of a few hundred
// units and costs its launch.  Small units come four to a block, those of neighbouring heads, and find their page together.
// Measured on one B200: 402 MB read back (134 MB of codes into f16) 71 us, 5.6 TB/s (0.87 of the measured copy rate), written 85 us; 8 prompts, 39 MB,
// 12.2 us written, 9.8 us read; a token each of 64 sequences 3.3 us.
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

// Warp-collective: the unit of `place` (a page that the call may touch) and `part` (head, keys or values).
__device__ __forceinline__ Unit find_unit(const nnb200_cache_i8& c, int place, int part, int32_t* error_word)
{
    Unit u;
    u.values = part & 1;
    u.head = part / 2;
    const int tokens = static_cast<int>(c.page_tokens), seqs = static_cast<int>(c.seqs);
    int b, j;
    if (c.cu == nullptr) {
        const int slots = (static_cast<int>(c.rows) / seqs + tokens - 2) / tokens + 1;
        b = place / slots;
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
        const int64_t from = begin(low);
        j = from <= place ? static_cast<int>(place - from) : -1;
    }
    const SequenceRows s = sequence_rows(c, b);
    const int first = max(s.len - s.n, 0);   // position of the first row that has a token
    const int64_t slot = static_cast<int64_t>(first / tokens) + j;
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
    if (u.page < 0) {   // the tokens' rows have no page; rows without a token stand directly before them
        u.zero_row = u.row - u.zero_rows;
        u.zero_rows += u.to - u.from;
    }
    return u;
}

// Division of numbers up to 4096 (the vectors of a unit) by one up to 32: n / 2^20 of the rounded-up 2^20 / d is off by less than 1 / 256.
struct Quotient {
    uint32_t by;
    __device__ __forceinline__ explicit Quotient(int d) : by(((1u << 20) + static_cast<uint32_t>(d) - 1u) / static_cast<uint32_t>(d)) {}
    __device__ __forceinline__ int operator()(int n) const { return static_cast<int>(static_cast<uint32_t>(n) * by >> 20); }
};

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
cache_write_kernel(const nnb200_cache_rows_args a, const int wide, int32_t* error_word)
{
    previous_kernel_done();
    constexpr int kThreads = 32 * WARPS;
    const nnb200_cache_i8& c = a.cache;
    const int part = WARPS == 1 ? static_cast<int>(blockIdx.y) * 4 + static_cast<int>(threadIdx.x) / 32 : static_cast<int>(blockIdx.y);
    if (part >= 2 * c.heads) {
        return;
    }
    const Unit u = find_unit(c, static_cast<int>(blockIdx.x), part, error_word);
    if (u.page < 0) {
        return;
    }
    const int t = threadIdx.x % kThreads;
    const int dim = static_cast<int>(c.dim), per_token = dim / 8;
    const int count = (u.to - u.from) * per_token;
    const Quotient divided(per_token);
    const int64_t stride_row = u.values ? a.v_stride_row : a.k_stride_row;
    const T* src = static_cast<const T*>(u.values ? a.v : a.k) + u.row * stride_row + u.head * (u.values ? a.v_stride_head : a.k_stride_head);
    float* scale = (u.values ? c.v_scale : c.k_scale) + u.page * c.scale_page_stride + u.head;
    int8_t* codes = static_cast<int8_t*>(u.values ? c.v : c.k) + u.page * c.page_stride + static_cast<int64_t>(u.head) * c.page_tokens * dim;

    const float before = u.begins ? 0.0f : *scale;
    Eight<T> x[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            const int token = divided(at);
            x[i].load(src + token * stride_row + (at - token * per_token) * 8, wide != 0);
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        if (t + i * kThreads < count) {
            float f[8];
            x[i].values(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = max(top, magnitude_bits(f[e]));
            }
        }
    }
    top = largest_of_unit<WARPS>(top);
    // A NaN or an infinity, of these tokens or of those before them, is the page's until it begins anew.
    float after = top >= kInfinityBits ? __uint_as_float(0x7FC00000u) : fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), kLeastCacheScale);
    after = before >= after || before != before ? before : after;
    const float inv = __frcp_rn(after);
    const bool number = after == after;   // else codes are zeros
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            float f[8];
            x[i].values(f);
            *reinterpret_cast<uint2*>(codes + u.from * dim + at * 8) = make_uint2(number ? codes4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv) : 0u,
                                                                                 number ? codes4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv) : 0u);
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
                const auto four = [&](uint32_t w) { return number ? codes4(code_at(w, 0) * ratio, code_at(w, 1) * ratio, code_at(w, 2) * ratio, code_at(w, 3) * ratio) : 0u; };
                *p = make_uint2(four(q.x), four(q.y));
            }
        }
    }
}

// A thread takes 16 codes at a time, all of its loads before its first store.
template <typename T, int WARPS>
__global__ void __launch_bounds__(block_threads(WARPS))
cache_read_kernel(const nnb200_cache_rows_args a, const int wide, int32_t* error_word)
{
    previous_kernel_done();
    constexpr int kThreads = 32 * WARPS;
    const nnb200_cache_i8& c = a.cache;
    const int part = WARPS == 1 ? static_cast<int>(blockIdx.y) * 4 + static_cast<int>(threadIdx.x) / 32 : static_cast<int>(blockIdx.y);
    if (part >= 2 * c.heads) {
        return;
    }
    const Unit u = find_unit(c, static_cast<int>(blockIdx.x), part, error_word);
    const int t = threadIdx.x % kThreads;
    const int dim = static_cast<int>(c.dim), per_token = dim / 16;
    const int64_t stride_row = u.values ? a.v_stride_row : a.k_stride_row;
    T* dst = static_cast<T*>(u.values ? a.v : a.k) + u.head * (u.values ? a.v_stride_head : a.k_stride_head);
    const auto store16 = [&](T* p, const float (&f)[16]) {
        store8(p, wide != 0, *reinterpret_cast<const float(*)[8]>(f));
        store8(p + 8, wide != 0, *reinterpret_cast<const float(*)[8]>(f + 8));
    };
    for (int64_t at = t; at < static_cast<int64_t>(u.zero_rows) * per_token; at += kThreads) {
        const float none[16] = {};
        store16(dst + (u.zero_row + at / per_token) * stride_row + at % per_token * 16, none);
    }
    if (u.page < 0) {
        return;
    }
    const int count = (u.to - u.from) * per_token;
    const Quotient divided(per_token);
    const float scale = (u.values ? c.v_scale : c.k_scale)[u.page * c.scale_page_stride + u.head];
    const int8_t* codes = static_cast<const int8_t*>(u.values ? c.v : c.k) + u.page * c.page_stride +
                          (static_cast<int64_t>(u.head) * c.page_tokens + u.from) * dim;
    dst += u.row * stride_row;
    uint4 q[kVectors / 2];
#pragma unroll
    for (int i = 0; i < kVectors / 2; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            q[i] = *reinterpret_cast<const uint4*>(codes + at * 16);
        }
    }
#pragma unroll
    for (int i = 0; i < kVectors / 2; ++i) {
        const int at = t + i * kThreads;
        if (at < count) {
            const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                f[e] = code_at(w[e / 4], e & 3) * scale;
            }
            const int token = divided(at);
            store16(dst + token * stride_row + (at - token * per_token) * 16, f);
        }
    }
}

template <typename T, int WARPS, bool WRITE>
cudaError_t run_units(const nnb200_cache_rows_args& a, int64_t places, int wide, const DeviceInfo& dev, cudaStream_t stream)
{
    const int64_t parts = 2 * a.cache.heads;
    const dim3 grid(static_cast<unsigned>(places), static_cast<unsigned>(WARPS == 1 ? (parts + 3) / 4 : parts));
    if constexpr (WRITE) {
        return launch_overlapping(cache_write_kernel<T, WARPS>, grid, dim3(block_threads(WARPS)), 0, stream, 1, a, wide, dev.error_word);
    } else {
        return launch_overlapping(cache_read_kernel<T, WARPS>, grid, dim3(block_threads(WARPS)), 0, stream, 1, a, wide, dev.error_word);
    }
}

template <typename T, bool WRITE>
cudaError_t run_typed(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const nnb200_cache_i8& c = a.cache;
    const int64_t each = c.cu == nullptr ? c.rows / c.seqs : c.rows;   // a sequence has at most so many rows
    const int64_t places = cache_places(c);
    const int64_t values = (each < c.page_tokens ? each : c.page_tokens) * c.dim;
    const auto aligned = [](const void* p, int64_t s0, int64_t s1) {
        constexpr int64_t kPer = 16 / sizeof(T);
        return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && s0 % kPer == 0 && s1 % kPer == 0;
    };
    const int wide = aligned(a.k, a.k_stride_row, a.k_stride_head) && aligned(a.v, a.v_stride_row, a.v_stride_head) ? 1 : 0;
    constexpr int kPerWarp = 32 * 8 * kVectors;
    return values <= kPerWarp       ? run_units<T, 1, WRITE>(a, places, wide, dev, stream)
           : values <= 4 * kPerWarp ? run_units<T, 4, WRITE>(a, places, wide, dev, stream)
           : values <= 8 * kPerWarp ? run_units<T, 8, WRITE>(a, places, wide, dev, stream)
                                    : run_units<T, 16, WRITE>(a, places, wide, dev, stream);
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
