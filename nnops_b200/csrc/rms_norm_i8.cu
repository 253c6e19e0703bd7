// RMS norm into 8 bits, with the residual's addition: the row of an int8 product out of the residual stream.
//
//   h = x + residual,  t = h * weight,  top = max |t|,  out = round(t * (127 / top)),  scale = top / (127 * sqrt(mean h^2 + eps))
//
// The reciprocal root is the same for the whole row, so it cancels out of the codes: they depend on no sum, only the
// scale does, and one pass over the row finds both what the sum and what the maximum need.  Squares are summed in
// 64 bits, which no f32 row can overflow.
//
// Bound by memory: with f16 rows 2 + 2 + 2 + 1 bytes an element.  4096 rows of 8192 with a residual: 37 us, 6.3 TB/s (0.98 of the measured copy
// rate); one row costs its launch.  A row is held in registers by one block (one warp, four rows
// a block, where a row has few vectors), every vector loaded before any is used (rows of more than 16384 columns spill: f32 244 bytes a thread, others with an
// f32 weight 96); rows off the 16-byte rule, or longer
// than 1024 threads hold, are read twice by an element-at-a-time kernel with the same arithmetic: 4096 x 8191 f16 197 us (1.2 TB/s), 1024 x 40000 bf16 323 us.

#include "cache_i8.cuh"

namespace nnb200 {

namespace {

constexpr float kLeastTop = 7.888609052210118e-31f;  // 2^-100: 127 / top stays finite

struct RowStats {
    double squares;
    uint32_t top;
};

__device__ __forceinline__ RowStats join_warp(RowStats s)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s.squares += __shfl_xor_sync(0xFFFFFFFFu, s.squares, o);
    }
    s.top = __reduce_max_sync(0xFFFFFFFFu, s.top);
    return s;
}

__device__ __forceinline__ RowStats join_block(RowStats s)
{
    __shared__ RowStats part[32];
    s = join_warp(s);
    const int warps = blockDim.x / 32;
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x / 32] = s;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    s = lane < warps ? part[lane] : RowStats{0.0, 0u};
    return join_warp(s);
}

// 127 / top of the row, or 0 where it holds something that is no number, and the row's scale.
__device__ __forceinline__ float finish_row(const RowStats& s, int64_t cols, float eps, float& scale)
{
    if (s.top >= kInfinityBits) {
        scale = __uint_as_float(0x7FC00000u);
        return 0.0f;
    }
    const float top = fmaxf(__uint_as_float(s.top), kLeastTop);
    scale = static_cast<float>(top * rsqrt(s.squares / static_cast<double>(cols) + static_cast<double>(eps)) / 127.0);
    return __fdiv_rn(127.0f, top);
}

// VECS vectors of 8 elements a thread, THREADS at most; WARP: a row is a warp's.
template <typename T, typename W, int VECS, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_i8_kernel(const nnb200_rms_norm_i8_args a)
{
    previous_kernel_done();
    const int per_row = WARP ? 32 : static_cast<int>(blockDim.x);
    const int t = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
    const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : static_cast<int64_t>(blockIdx.x);
    if (WARP && row >= a.rows) {
        return;
    }
    const int vectors = static_cast<int>(a.cols / 8);
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* residual = static_cast<const T*>(a.residual) + row * a.residual_stride;
    const W* weight = static_cast<const W*>(a.weight);
    Eight<T> raw[VECS], more[VECS];
    Eight<W> w[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int at = t + i * per_row;
        if (at < vectors) {
            raw[i].load(x + at * 8, true);
            if (a.residual != nullptr) {
                more[i].load(residual + at * 8, true);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int at = t + i * per_row;
        if (at < vectors) {
            w[i].load(weight + at * 8, true);
        }
    }
    float h[VECS][8];
    RowStats s{0.0, 0u};
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int at = t + i * per_row;
        if (at < vectors) {
            raw[i].values(h[i]);
            if (a.residual != nullptr) {
                float r[8];
                more[i].values(r);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[i][e] += r[e];
                }
            }
            if (a.residual_out != nullptr) {
                store8(static_cast<T*>(a.residual_out) + row * a.residual_out_stride + at * 8, true, h[i]);
            }
            float f[8];
            w[i].values(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double d = h[i][e];
                s.squares = fma(d, d, s.squares);
                h[i][e] *= f[e];
                s.top = max(s.top, magnitude_bits(h[i][e]));
            }
        }
    }
    s = WARP ? join_warp(s) : join_block(s);
    float scale;
    const float inv = finish_row(s, a.cols, a.eps, scale);
    if (t == 0) {
        a.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int at = t + i * per_row;
        if (at < vectors) {
            const uint2 q = make_uint2(inv != 0.0f ? codes4(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv) : 0u,
                                       inv != 0.0f ? codes4(h[i][4] * inv, h[i][5] * inv, h[i][6] * inv, h[i][7] * inv) : 0u);
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(a.out) + row * a.out_stride + at * 8) = q;
        }
    }
}

// Any row: read twice, residual_out written the second time, as it may be x or residual.
template <typename T, typename W>
__global__ void rms_norm_i8_twice_kernel(const nnb200_rms_norm_i8_args a)
{
    previous_kernel_done();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* residual = static_cast<const T*>(a.residual) + row * a.residual_stride;
    const W* weight = static_cast<const W*>(a.weight);
    const auto sum = [&](int64_t i) {
        const float v = to_float(x[i]);
        return a.residual != nullptr ? v + to_float(residual[i]) : v;
    };
    RowStats s{0.0, 0u};
    for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
        const float h = sum(i);
        const double d = h;
        s.squares = fma(d, d, s.squares);
        s.top = max(s.top, magnitude_bits(h * to_float(weight[i])));
    }
    s = join_block(s);
    float scale;
    const float inv = finish_row(s, a.cols, a.eps, scale);
    if (threadIdx.x == 0) {
        a.scale[row] = scale;
    }
    for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
        const float h = sum(i);
        if (a.residual_out != nullptr) {
            static_cast<T*>(a.residual_out)[row * a.residual_out_stride + i] = from_float<T>(h);
        }
        static_cast<int8_t*>(a.out)[row * a.out_stride + i] = static_cast<int8_t>(code_of(h * to_float(weight[i]) * inv));
    }
}

template <typename T, typename W>
cudaError_t run_typed(const nnb200_rms_norm_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    constexpr int64_t kPer = 16 / sizeof(T);
    const auto wide = [](const void* p, int64_t stride, int64_t per) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % per == 0; };
    const bool vectors_ok = a.cols % 8 == 0 && a.cols <= 8 * 4 * 1024 && wide(a.x, a.x_stride, kPer) &&
                            (a.residual == nullptr || wide(a.residual, a.residual_stride, kPer)) &&
                            (a.residual_out == nullptr || wide(a.residual_out, a.residual_out_stride, kPer)) && wide(a.weight, 0, 1) &&
                            (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0 && a.out_stride % 8 == 0;
    const unsigned rows = static_cast<unsigned>(a.rows);
    if (!vectors_ok) {
        const int64_t warps = (a.cols + 127) / 128;
        return launch_overlapping(rms_norm_i8_twice_kernel<T, W>, dim3(rows), dim3(static_cast<unsigned>(32 * (warps < 1 ? 1 : warps > 16 ? 16 : warps))), 0, stream,
                                  1, a);
    }
    const int64_t vectors = a.cols / 8;
    const auto threads = [&](int per) { return dim3(static_cast<unsigned>((vectors + 32 * per - 1) / (32 * per) * 32)); };
    if (vectors <= 64) {
        const dim3 grid((rows + 3) / 4);
        return vectors <= 32 ? launch_overlapping(rms_norm_i8_kernel<T, W, 1, true, 128>, grid, dim3(128), 0, stream, 1, a)
                             : launch_overlapping(rms_norm_i8_kernel<T, W, 2, true, 128>, grid, dim3(128), 0, stream, 1, a);
    }
    // Few rows: as many threads as there are vectors, for the latency.  Many: few threads with several vectors each, so that an
    // SM has more rows under way, some loading while others are summed or stored.
    const int64_t least = a.rows <= 2 * dev.sm_count ? 1 : (vectors + 255) / 256;
    const int64_t need = (vectors + 1023) / 1024, per = least > need ? least : need;
    return per <= 1         ? launch_overlapping(rms_norm_i8_kernel<T, W, 1, false, 1024>, dim3(rows), threads(1), 0, stream, 1, a)
           : per <= 2       ? launch_overlapping(rms_norm_i8_kernel<T, W, 2, false, 1024>, dim3(rows), threads(2), 0, stream, 1, a)
           : vectors <= 2048 ? launch_overlapping(rms_norm_i8_kernel<T, W, 4, false, 512>, dim3(rows), threads(4), 0, stream, 1, a)
                             : launch_overlapping(rms_norm_i8_kernel<T, W, 4, false, 1024>, dim3(rows), threads(4), 0, stream, 1, a);
}

}  // namespace

int launch_rms_norm_i8(const nnb200_rms_norm_i8_args& a, const DeviceInfo& dev, cudaStream_t stream)
{
    const bool wide_weight = a.weight_type == NNB200_FLOAT_F32;
    const cudaError_t e = a.float_type == NNB200_FLOAT_F32   ? run_typed<float, float>(a, dev, stream)
                          : a.float_type == NNB200_FLOAT_F16 ? (wide_weight ? run_typed<__half, float>(a, dev, stream) : run_typed<__half, __half>(a, dev, stream))
                          : wide_weight                      ? run_typed<__nv_bfloat16, float>(a, dev, stream)
                                                             : run_typed<__nv_bfloat16, __nv_bfloat16>(a, dev, stream);
    note_launch();
    return cuda_status(e);
}

}  // namespace nnb200
