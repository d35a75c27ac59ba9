// Products in 8-bit integers with one scale a token and one a channel (quantize_rows_i8_hip, mul_mat_i8_hip).
//
//   s_t = max_k |x_tk| r              q_tk = round_half_even(x_tk / s_t)        (0 where s_t is 0)
//   y_tm = (sum_k q_tk w_mk) s_t s_m + b_m
//
// r is the binary32 number nearest to 1/127; product and quotient are rounded to binary32.
// The sums are exact: |q|, |w| <= 128 and K <= 131071 keep them below 2^31.  The one rounding of a sum is its conversion to
// binary32, then one for either scale, one for the bias and one to the output's type.  Unlike the block format (q8.hip), whose
// every 32 products are settled in binary32, nothing but matrix instructions stands in the loop over k.
#include "elements.hpp"
#include "tile_product.hpp"

namespace ppmlhip {
namespace {

constexpr int I8_MAX_K = 131071;

// ------------------------------------------------------------------------------------------------------------ quantizer
// A wave per row.  The row is read twice, the second time from the cache: bound by the first.
struct I8Quantize {
    const void* x;
    const float* scale_in;    // x holds int8 already: its rows are only laid out anew
    int8_t* q;
    float* scale;
    int64_t rows, x_stride, q_stride;
    int K, Kq;                // elements per row, and how many to write (zero from K on)
};

__device__ __forceinline__ float i8_scale(float largest) {
    // (infinite or NaN: the row's results are NaN by its scale; its values are written as zeros)
    return largest <= 3.402823466e38f ? largest * (1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ int i8_value(float x, float scale) {
    const float q = __builtin_rintf(x / scale);
    return scale > 0.0f ? static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f)) : 0;
}
// the larger magnitude, NaN if either is one
__device__ __forceinline__ float max_or_nan(float a, float b) {
    return a != a ? a : (b != b ? b : fmaxf(a, b));
}

template <class T>
__global__ __launch_bounds__(256) void i8_quantize_kernel(const I8Quantize p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const T* const x = static_cast<const T*>(p.x) + row * p.x_stride;
    int8_t* const q = p.q + row * p.q_stride;
    if constexpr (sizeof(T) == 1) {
        for (int k = lane; k < p.Kq; k += 64) q[k] = k < p.K ? static_cast<int8_t>(x[k]) : static_cast<int8_t>(0);
        return;
    } else {
        float largest = 0.0f;
        for (int k = lane; k < p.K; k += 64) largest = max_or_nan(largest, __builtin_fabsf(to_f32(x[k])));
        largest = wave_butterfly(largest, [](float a, float b) { return max_or_nan(a, b); });
        const float scale = i8_scale(largest);
        for (int k = lane; k < p.Kq; k += 64) q[k] = static_cast<int8_t>(k < p.K ? i8_value(to_f32(x[k]), scale) : 0);
        if (lane == 0) p.scale[row] = scale;
    }
}

// ------------------------------------------------------------------------------------------------------------ product
struct I8Product {
    RowBytes w, x;            // rows: channels, tokens
    const float *w_scale, *x_scale, *bias;
    void* y;                  // [tokens][channels]
    int stages, tiles_w, tiles_x;
};

template <class T, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM * WN * 64) void i8_product_kernel(const I8Product p) {
    typedef TileLoop<StepI8, WM, WN, TM, TN> Loop;
    const int t = xcd_contiguous_index(blockIdx.x, p.tiles_w * p.tiles_x);
    const int m0 = (t % p.tiles_w) * Loop::BM, n0 = (t / p.tiles_w) * Loop::BN;
    v4i acc[TM][TN];
    Loop::run(p.w, p.x, m0, n0, p.stages, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mw = m0 + wave / WN * TM * 16 + (lane >> 4) * 4, nw = n0 + wave % WN * TN * 16 + (lane & 15);
    const int M = p.w.rows;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        float ws[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = mw + 16 * i + r < M ? mw + 16 * i + r : M - 1;
            ws[r] = p.w_scale[m];
            b[r] = p.bias ? p.bias[m] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + 16 * j;
            if (n >= p.x.rows) continue;
            const float xs = p.x_scale[n];
            T* const y = static_cast<T*>(p.y) + static_cast<int64_t>(n) * M;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = static_cast<float>(acc[i][j][r]) * xs * ws[r];
                if (mw + 16 * i + r < M) y[mw + 16 * i + r] = from_f32<T>(p.bias ? v + b[r] : v);
            }
        }
    }
}

int64_t i8_row_bytes(int64_t K) { return (K + TILE_K - 1) / TILE_K * TILE_K; }

int launch_quantize(const I8Quantize& p, int type, hipStream_t stream, const char* what) {
    const int64_t blocks = (p.rows + 3) / 4;
    if (blocks > 0x7fffffff) { set_error("%s: too many rows", what); return RC_BAD_ARGS; }
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    switch (type) {
        case PPML_ELEM_F32:  hipLaunchKernelGGL((i8_quantize_kernel<float>), grid, block, 0, stream, p); break;
        case PPML_ELEM_F16:  hipLaunchKernelGGL((i8_quantize_kernel<_Float16>), grid, block, 0, stream, p); break;
        case PPML_ELEM_BF16: hipLaunchKernelGGL((i8_quantize_kernel<__bf16>), grid, block, 0, stream, p); break;
        default:             hipLaunchKernelGGL((i8_quantize_kernel<int8_t>), grid, block, 0, stream, p); break;
    }
    return check_launch(what);
}

template <class T>
void launch_product(const I8Product& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.tiles_w * p.tiles_x));
    hipLaunchKernelGGL((i8_product_kernel<T, 2, 2, 4, 4>), grid, dim3(256), 0, stream, p);
}

bool float_type(int type) { return type == PPML_ELEM_F32 || type == PPML_ELEM_F16 || type == PPML_ELEM_BF16; }

}  // namespace
}  // namespace ppmlhip

using namespace ppmlhip;

extern "C" int quantize_rows_i8_hip(const void* x, int type, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t rows, int K,
                                    ppml_hip_stream_t stream) {
    const int64_t Kq = q_stride == i8_row_bytes(K) ? q_stride : K;
    if (!x || !q || !float_type(type) || !scale || rows <= 0 || K <= 0 || K > I8_MAX_K || x_stride < K || q_stride < K) {
        set_error("quantize_rows_i8_hip: bad arguments (rows=%lld K=%d type=%d)", (long long)rows, K, type);
        return RC_BAD_ARGS;
    }
    return launch_quantize(I8Quantize{x, nullptr, q, scale, rows, x_stride, q_stride, K, static_cast<int>(Kq)}, type, static_cast<hipStream_t>(stream),
                           "quantize_rows_i8_hip");
}

extern "C" size_t i8_weight_row_bytes_hip(int K) { return K > 0 && K <= I8_MAX_K ? static_cast<size_t>(i8_row_bytes(K)) : 0; }

extern "C" int i8_weight_pack_hip(const int8_t* w, int64_t w_stride, int M, int K, int8_t* packed, ppml_hip_stream_t stream) {
    if (!w || !packed || M <= 0 || K <= 0 || K > I8_MAX_K || w_stride < K) {
        set_error("i8_weight_pack_hip: bad arguments (M=%d K=%d)", M, K);
        return RC_BAD_ARGS;
    }
    const int64_t row = i8_row_bytes(K);
    return launch_quantize(I8Quantize{w, nullptr, packed, nullptr, M, w_stride, row, K, static_cast<int>(row)}, PPML_ELEM_I8, static_cast<hipStream_t>(stream),
                           "i8_weight_pack_hip");
}

extern "C" size_t mul_mat_i8_workspace_hip(int N, int K) {
    if (N <= 0 || K <= 0 || K > I8_MAX_K) return 0;
    return static_cast<size_t>(N) * static_cast<size_t>(i8_row_bytes(K)) + 4 * static_cast<size_t>(N);
}

extern "C" int mul_mat_i8_hip(const int8_t* packed, const float* w_scale, const void* x, int x_type, int64_t x_stride, const float* x_scale, const float* bias,
                              void* y, int y_type, int M, int N, int K, void* workspace, size_t workspace_bytes, ppml_hip_stream_t stream_) {
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (!packed || !w_scale || !x || !y || M <= 0 || N <= 0 || K <= 0 || K > I8_MAX_K || x_stride < K || !float_type(y_type) ||
        (x_type == PPML_ELEM_I8 ? !x_scale : !float_type(x_type)) || (reinterpret_cast<uintptr_t>(packed) & 15) != 0) {
        set_error("mul_mat_i8_hip: bad arguments (M=%d N=%d K=%d x_type=%d y_type=%d)", M, N, K, x_type, y_type);
        return RC_BAD_ARGS;
    }
    if (!workspace || workspace_bytes < mul_mat_i8_workspace_hip(N, K) || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
        set_error("mul_mat_i8_hip: needs %zu bytes of workspace, 16-byte aligned (got %zu)", mul_mat_i8_workspace_hip(N, K), workspace_bytes);
        return RC_BAD_ARGS;
    }
    StatsScope stats("i8", N, K, M, stream);
    const int64_t row = i8_row_bytes(K);
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scale = reinterpret_cast<float*>(q + static_cast<int64_t>(N) * row);
    const int rc = launch_quantize(I8Quantize{x, x_scale, q, scale, N, x_stride, row, K, static_cast<int>(row)}, x_type, stream, "mul_mat_i8_hip");
    if (rc != RC_OK) return rc;
    I8Product p{};
    p.w = RowBytes{reinterpret_cast<const uint8_t*>(packed), row, M};
    p.x = RowBytes{reinterpret_cast<const uint8_t*>(q), row, N};
    p.w_scale = w_scale;
    p.x_scale = x_type == PPML_ELEM_I8 ? x_scale : scale;
    p.bias = bias;
    p.y = y;
    p.stages = static_cast<int>(row / TILE_K);
    p.tiles_w = (M + 127) / 128;
    p.tiles_x = (N + 127) / 128;
    if (static_cast<int64_t>(p.tiles_w) * p.tiles_x > 0x7fffffff) { set_error("mul_mat_i8_hip: too many tiles"); return RC_BAD_ARGS; }
    switch (y_type) {
        case PPML_ELEM_F32:  launch_product<float>(p, stream); break;
        case PPML_ELEM_F16:  launch_product<_Float16>(p, stream); break;
        default:             launch_product<__bf16>(p, stream); break;
    }
    return check_launch("mul_mat_i8_hip");
}
