// The key/value cache in 8 bits as its kernels see it: which tokens a call's rows are, which pages they lie in, and the
// floating types at its edges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.cuh"
#include "ptx.cuh"

namespace nnb200 {

constexpr float kLeastCacheScale = 8.673617379884035e-19f;  // 2^-60

// Pages that the rows of a call may touch, in all sequences.
inline int64_t cache_places(const nnb200_cache_i8& c)
{
    return c.cu == nullptr ? c.seqs * ((c.rows / c.seqs + c.page_tokens - 2) / c.page_tokens + 1) : c.rows / c.page_tokens + 2 * c.seqs;
}

int launch_cache_write_i8(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream);
int launch_cache_read_i8(const nnb200_cache_rows_args& a, const DeviceInfo& dev, cudaStream_t stream);
int launch_rms_norm_i8(const nnb200_rms_norm_i8_args& a, const DeviceInfo& dev, cudaStream_t stream);
size_t attention_i8_workspace_bytes(const nnb200_attention_i8_args& a, const DeviceInfo& dev);
int launch_attention_i8(const nnb200_attention_i8_args& a, const DeviceInfo& dev, cudaStream_t stream);

// ---- floating types -----------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v)
{
    if constexpr (sizeof(T) == 4) {
        return v;
    } else if constexpr (std::is_same_v<T, __half>) {
        return __float2half_rn(v);
    } else {
        return __float2bfloat16_rn(v);
    }
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b)
{
    if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x;
        b = f.y;
    } else {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// Eight consecutive values; `wide`: the address is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, float (&f)[8])
{
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[i] = to_float(p[i]);
        }
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        unpack2<T>(a.x, f[0], f[1]);
        unpack2<T>(a.y, f[2], f[3]);
        unpack2<T>(a.z, f[4], f[5]);
        unpack2<T>(a.w, f[6], f[7]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, const float (&f)[8])
{
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = from_float<T>(f[i]);
        }
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    }
}

// Eight values as they lie in memory, and one by one.
template <typename T>
struct Eight {
    uint4 raw[sizeof(T) / 2];

    __device__ __forceinline__ void load(const T* p, bool wide)
    {
        if (wide) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
                raw[i] = reinterpret_cast<const uint4*>(p)[i];
            }
        } else {
            uint32_t w[2 * sizeof(T)];
#pragma unroll
            for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) {
                if constexpr (sizeof(T) == 4) {
                    w[i] = reinterpret_cast<const uint32_t*>(p)[i];
                } else {
                    w[i] = static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[2 * i]) | static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[2 * i + 1]) << 16;
                }
            }
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
                raw[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
        }
    }
    __device__ __forceinline__ void values(float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    f[4 * i + k] = __uint_as_float(w[k]);
                } else {
                    unpack2<T>(w[k], f[2 * k], f[2 * k + 1]);
                }
            }
        }
    }
};

// Round half to even into s8, saturating; NaN gives 0.
__device__ __forceinline__ uint32_t code_of(float v)
{
    int32_t q;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(v));
    return static_cast<uint32_t>(q) & 0xFFu;
}

// The same of four values of which each rounds to a code: added to 1.5 * 2^23 they are rounded to an integer, whose low byte is the code.
// (Conversions take four times an addition's time.)
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d)
{
    constexpr float kInteger = 12582912.0f;
    const auto bits = [](float v) { return __float_as_uint(__fadd_rn(v, kInteger)); };
    return __byte_perm(__byte_perm(bits(a), bits(b), 0x0040), __byte_perm(bits(c), bits(d), 0x0040), 0x5410);
}

__device__ __forceinline__ float code_at(uint32_t word, int byte) { return static_cast<float>(static_cast<int8_t>(word >> (8 * byte))); }

// |v| ordered as a number, with every NaN above infinity.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kInfinityBits = 0x7F800000u;

// ---- sequences and pages ------------------------------------------------------------------

// Sequence b's rows of the call and its tokens, whatever the arrays hold: rows [row0, row0 + n) lie in [0, rows).
struct SequenceRows {
    int row0, n, len;
};

__device__ __forceinline__ SequenceRows sequence_rows(const nnb200_cache_i8& c, int b)
{
    SequenceRows s;
    const int rows = static_cast<int>(c.rows);
    if (c.cu != nullptr) {
        s.row0 = min(max(c.cu[b], 0), rows);
        s.n = min(max(c.cu[b + 1], s.row0), rows) - s.row0;
    } else {
        s.n = rows / static_cast<int>(c.seqs);
        s.row0 = s.n * b;
    }
    s.len = min(max(c.lens[b], 0), static_cast<int>(c.table_pages * c.page_tokens));
    return s;
}

// The page of a sequence's `slot`-th block of tokens; -1, recorded, where the table holds no page there.
__device__ __forceinline__ int page_at(const nnb200_cache_i8& c, int b, int slot, int32_t* error_word)
{
    const int page = c.page_table[b * c.table_stride + slot];
    if (page < 0 || page >= c.pages) {
        atomicCAS(error_word, 0, kErrBadPage);
        return -1;
    }
    return page;
}

}  // namespace nnb200
