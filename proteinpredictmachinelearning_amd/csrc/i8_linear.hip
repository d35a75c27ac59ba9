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

constexpr int I8_MAX_K = 131071, I8_MAX_M = 1 << 22, I8_MAX_N = 0x7fffffff - 1023;      // (N: a tile's end stays an int)
constexpr int64_t LAUNCH_MOST_THREADS = 0xffffffffll;   // along x

// ------------------------------------------------------------------------------------------------------------ quantizer
struct I8Rows {
    const void* x;
    int type;                 // PPML_ELEM_*; I8: the rows are only laid out anew
    int64_t stride;
    const float* scale;       // I8: the rows' scales
    int64_t rows;
    int K;
};

// (the rows of any layout: four elements at the alignment of one)
template <class T> struct Quad { typedef T Raw __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

// the largest magnitude, NaN if there is one
__device__ __forceinline__ float largest_of(float m, float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_elementwise_maximum(m, x);
#else
    return m + x;
#endif
}
// A row's scale and what its values are divided with.  The quotient is x times the scale's reciprocal (rounded correctly, once a row), which is
// off by less than two units in the last place, with two corrections by the remainder: the first leaves less than one unit, the second is then
// the correctly rounded quotient (Markstein's theorem), provided that no intermediate leaves the normal numbers: rows whose largest is below
// 2^-40 are multiplied by 2^64 first, scale and all.  (A division per element cost a long row more than its way from memory, and a kernel of few
// tokens most of its time on fetching instructions: 32 tokens x 512 -> 512 12 us.)
struct RowScale {
    float scale;              // as it goes out
    float divisor, inverse, lift;
    uint32_t keep;            // 0 where the values are zeros: the scale is 0 or NaN

    __device__ __forceinline__ RowScale() : scale(0.0f), divisor(0.0f), inverse(0.0f), lift(1.0f), keep(0) {}
    __device__ __forceinline__ explicit RowScale(float largest) {
        // (infinite or NaN: the row's results are NaN by its scale)
        scale = largest <= 3.402823466e38f ? largest * (1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
        lift = largest < 0x1p-40f ? 0x1p64f : 1.0f;
        keep = scale > 0.0f ? ~0u : 0u;
        divisor = scale * lift;
        inverse = 1.0f / divisor;
    }
};
// Four quantized values, the first in the lowest byte.  Adding 1.5 * 2^23 rounds to whole numbers, halves to even, and leaves them in the lowest bits.
__device__ __forceinline__ uint32_t quantize4(const float (&x)[4], const RowScale& r) {
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = x[e] * r.lift, rough = y * r.inverse, near = fmaf(fmaf(-rough, r.divisor, y), r.inverse, rough);
        const float exact = fmaf(fmaf(-near, r.divisor, y), r.inverse, near);
        // (a scale that is itself a subnormal number may be far from the 127th part)
        q[e] = __float_as_uint(fminf(fmaxf(exact, -127.0f), 127.0f) + 12582912.0f);
    }
    const uint32_t low = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u), high = __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
    return (low | high) & r.keep;
}
// Four values that are whole numbers already
__device__ __forceinline__ uint32_t pack4(const float (&x)[4]) {
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __float_as_uint(x[e] + 12582912.0f);
    return __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
}

// Elements k to k + 3 of a row of four or more, zeros behind its end, in two steps: the load, which is made whatever k is (the row's last four where
// four from k on do not fit), and what becomes of it.  Loads under conditions, or with a use beside them, are waited for one after the other.
template <class T>
__device__ __forceinline__ typename Quad<T>::Raw fetch4(const T* row, int k, int K) {
    return *reinterpret_cast<const typename Quad<T>::Raw*>(row + (k + 4 <= K ? k : K - 4));
}
template <class T>
__device__ __forceinline__ void finish4(const typename Quad<T>::Raw& raw, int k, int K, float (&x)[4]) {
    const int by = k + 4 <= K ? 0 : k + 4 - K;          // places that the loaded four lie too low
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32(static_cast<T>(raw[e]));
    if (K & 3) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = by & 2 ? (e + 2 < 4 ? v[(e + 2) & 3] : 0.0f) : v[e];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = by & 1 ? (e + 1 < 4 ? v[(e + 1) & 3] : 0.0f) : v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = by < 4 ? v[e] : 0.0f;
}

// A wave's rows from `first` to `end`, of 4 to 256 R elements and at most G = 8 / R or 1 of them, kept in registers between the search for the largest and
// the quantizing.  put(row, k, four values) for every k of a whole number of 256, and scale_is(row, scale).
template <class T, int R, class Put, class ScaleIs>
__device__ __forceinline__ void quantize_resident(const I8Rows& p, int64_t first, int64_t end, const Put& put, const ScaleIs& scale_is) {
    constexpr int G = R >= 8 ? 1 : 8 / R;
    const int lane = threadIdx.x & 63;
    if (first >= end) return;
    typename Quad<T>::Raw raw[G][R];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const T* const row = static_cast<const T*>(p.x) + (first + g < end ? first + g : end - 1) * p.stride;
#pragma unroll
        for (int i = 0; i < R; ++i) raw[g][i] = fetch4<T>(row, 4 * (lane + 64 * i), p.K);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        if (first + g >= end) break;
        float x[R][4], largest = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) finish4<T>(raw[g][i], 4 * (lane + 64 * i), p.K, x[i]);
        if constexpr (sizeof(T) == 1) {
#pragma unroll
            for (int i = 0; i < R; ++i) put(first + g, 4 * (lane + 64 * i), pack4(x[i]));
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) largest = largest_of(largest, __builtin_fabsf(x[i][e]));
            largest = wave_butterfly(largest, [](float a, float b) { return largest_of(a, b); });
            const RowScale scale(largest);
#pragma unroll
            for (int i = 0; i < R; ++i) put(first + g, 4 * (lane + 64 * i), quantize4(x[i], scale));
            scale_is(first + g, scale.scale);
        }
    }
}
// Longer rows are read twice, the second time from the cache; rows of fewer than four elements as well
template <class T, class Put, class ScaleIs>
__device__ __forceinline__ void quantize_twice(const I8Rows& p, int64_t first, int64_t end, const Put& put, const ScaleIs& scale_is) {
    const int lane = threadIdx.x & 63;
    const auto load = [&](const T* row, int k, float (&x)[4]) {
        if (p.K >= 4) finish4<T>(fetch4<T>(row, k, p.K), k, p.K, x);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = k + e < p.K ? to_f32(row[k + e]) : 0.0f;
    };
    for (int64_t r = first; r < end; ++r) {
        const T* const row = static_cast<const T*>(p.x) + r * p.stride;
        RowScale scale;
        if constexpr (sizeof(T) > 1) {
            float largest = 0.0f;
            const auto meet = [&](const float (&x)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) largest = largest_of(largest, __builtin_fabsf(x[e]));
            };
            int k = 4 * lane;
            for (; k + 2048 <= p.K; k += 2048) {
                typename Quad<T>::Raw raw[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) raw[u] = fetch4<T>(row, k + 256 * u, p.K);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    float x[4];
                    finish4<T>(raw[u], k + 256 * u, p.K, x);
                    meet(x);
                }
            }
            for (; k < p.K; k += 256) {
                float x[4];
                load(row, k, x);
                meet(x);
            }
            largest = wave_butterfly(largest, [](float a, float b) { return largest_of(a, b); });
            scale = RowScale(largest);
            scale_is(r, scale.scale);
        }
        int k = 4 * lane;
        for (; k + 2048 <= p.K; k += 2048) {
            typename Quad<T>::Raw raw[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) raw[u] = fetch4<T>(row, k + 256 * u, p.K);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float x[4];
                finish4<T>(raw[u], k + 256 * u, p.K, x);
                put(r, k + 256 * u, sizeof(T) == 1 ? pack4(x) : quantize4(x, scale));
            }
        }
        for (; k < (p.K + 255) / 256 * 256; k += 256) {
            float x[4];
            load(row, k, x);
            put(r, k, sizeof(T) == 1 ? pack4(x) : quantize4(x, scale));
        }
    }
}

// `put` stores four values at k: all of them below the row's end, which is K or that up to a multiple of 128
__device__ __forceinline__ void put_row(int8_t* row, int k, int end, uint32_t v) {
    typedef uint32_t any32 __attribute__((aligned(1)));
    if (k + 4 <= end) *reinterpret_cast<any32*>(row + k) = v;
    else
        for (int e = 0; e < 4 && k + e < end; ++e) row[k + e] = static_cast<int8_t>(v >> 8 * e);
}

// A wave per row (R = 0: rows of any length).  Bound by memory, x read once and a byte an element written.  Traced: 8192 rows of 4096, bf16 20 us
// (5 TB/s).
template <class T, int R>
__global__ __launch_bounds__(256) void i8_quantize_kernel(const I8Rows p, int8_t* q, int64_t q_stride, int q_end, float* scales) {
    constexpr int G = R == 0 || R >= 8 ? 1 : 8 / R;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * G, end = first + G < p.rows ? first + G : p.rows;
    const auto put = [&](int64_t row, int k, uint32_t v) { put_row(q + row * q_stride, k, q_end, v); };
    const auto scale_is = [&](int64_t row, float scale) { if ((threadIdx.x & 63) == 0) scales[row] = scale; };
    if constexpr (R == 0) quantize_twice<T>(p, first, end, put, scale_is);
    else quantize_resident<T, R>(p, first, end, put, scale_is);
}

// Long rows, and few shorter ones: a work-group of eight waves per row, each with 256 R elements of it in registers.  bf16, without / with: 30 rows of 16384
// (read twice by one wave) 26.6 / 3.5 us, 8192 of 8192 65 / 37.5 (5.4 TB/s), 2048 of 32768 108 / 42; 64 of 4096 (one wave) 5.3 / 2.3, 1024 of 4096 6.1 / 3.8.
constexpr int I8_ROW_WAVES = 8;
template <class T, int R>
__global__ __launch_bounds__(I8_ROW_WAVES * 64) void i8_quantize_row_kernel(const I8Rows p, int8_t* q, int64_t q_stride, int q_end, float* scales) {
    __shared__ float parts[I8_ROW_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k0 = 4 * static_cast<int>(threadIdx.x);
    const T* const row = static_cast<const T*>(p.x) + static_cast<int64_t>(blockIdx.x) * p.stride;
    typename Quad<T>::Raw raw[R];
#pragma unroll
    for (int i = 0; i < R; ++i) raw[i] = fetch4<T>(row, k0 + I8_ROW_WAVES * 256 * i, p.K);
    float x[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) finish4<T>(raw[i], k0 + I8_ROW_WAVES * 256 * i, p.K, x[i]);
    RowScale scale;
    if constexpr (sizeof(T) > 1) {
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) largest = largest_of(largest, __builtin_fabsf(x[i][e]));
        largest = wave_butterfly(largest, [](float a, float b) { return largest_of(a, b); });
        if (lane == 0) parts[wave] = largest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < I8_ROW_WAVES; ++w) largest = largest_of(largest, parts[w]);
        scale = RowScale(largest);
        if (threadIdx.x == 0) scales[blockIdx.x] = scale.scale;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        put_row(q + static_cast<int64_t>(blockIdx.x) * q_stride, k0 + I8_ROW_WAVES * 256 * i, q_end, sizeof(T) == 1 ? pack4(x[i]) : quantize4(x[i], scale));
}

// ------------------------------------------------------------------------------------------------------------ product
struct I8Product {
    RowBytes w, x;            // rows: channels, tokens
    const float *w_scale, *x_scale, *bias;
    void* y;                  // [tokens][channels]
    int stages, tiles_w, tiles_x;
    // slices > 1: every tile is cut along k into work-groups of slice_stages stages, whose sums go to `sums`
    int slices, slice_stages;
    v4i* sums;                // [tile][slice][a wave's tiles of 16 x 16][thread]
};

// What a lane multiplies and adds to its channels of a wave's 16 TM from mw on
template <class T, int TM>
struct Channels {
    static constexpr int V = 16 / sizeof(T), ACROSS = TM * 16 / V;      // channels per lane, lanes per token
    static_assert(64 % ACROSS == 0, "a lane keeps its channels");
    float scale[V], bias[V];
    int m;
    __device__ __forceinline__ Channels(const I8Product& p, int mw) {
        m = mw + (threadIdx.x & 63) % ACROSS * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int at = m + e < p.w.rows ? m + e : p.w.rows - 1;
            scale[e] = p.w_scale[at];
            bias[e] = p.bias ? p.bias[at] : 0.0f;
        }
    }
};

// The outputs of a wave: TM x TN tiles of its channels and the tokens from nw on.  Sixteen tokens at a time go through LDS (16 (16 TM + 4)
// floats), where a lane's four consecutive channels become whole lines of the output: stored as the matrix instruction leaves
// them, a token's channels went out in pieces of 16 bytes (f32) and 8 (the alignment's projection 60 us instead of 22).
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
constexpr uint32_t OUTSIDE_ROWS = 0xfffffff0u;           // no resource here is that long
template <bool VEC, class T, int TM, int TN>
__device__ __forceinline__ void store_tokens(const I8Product& p, const Channels<T, TM>& ch, float* lds, int nw, const v4i (&acc)[TM][TN], const float* x_scale) {
    constexpr int PITCH = TM * 16 + 4;                  // floats: the rows of sixteen lanes' pieces in banks of their own
    constexpr int V = Channels<T, TM>::V, ACROSS = Channels<T, TM>::ACROSS;
    const int lane = threadIdx.x & 63, M = p.w.rows, c = lane % ACROSS * V, m = ch.m;
    // (stores outside, by their offsets, are none: without a condition around them the compiler knows how many there are, and waits for loads
    // that were requested before them without waiting for the stores)
    const int64_t left = (static_cast<int64_t>(p.x.rows) - nw) * M * sizeof(T), most = static_cast<int64_t>(TN * 16) * M * sizeof(T);
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(static_cast<T*>(p.y) + static_cast<int64_t>(nw) * M, 0,
                                                                          static_cast<int>(left < 0 ? 0 : left < most ? left : most), 0x00020000);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const float xs = x_scale[16 * j + (lane & 15)];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            v4f v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = static_cast<float>(acc[i][j][r]) * xs;
            *reinterpret_cast<v4f*>(lds + (lane & 15) * PITCH + 16 * i + (lane >> 4) * 4) = v;
        }
        wave_fence();
#pragma unroll
        for (int k = 0; k < 16 * ACROSS / 64; ++k) {
            const int token = (k * 64 + lane) / ACROSS;
            const uint32_t at = static_cast<uint32_t>((16 * j + token) * static_cast<int64_t>(M) + m) * static_cast<uint32_t>(sizeof(T));
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<v4f*>(v + e) = *reinterpret_cast<const v4f*>(lds + token * PITCH + c + e);
            typename Elements<T, V>::Raw raw;
#pragma unroll
            for (int e = 0; e < V; ++e) raw[e] = from_f32<T>(p.bias ? v[e] * ch.scale[e] + ch.bias[e] : v[e] * ch.scale[e]);
            if (VEC) {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, raw), rsrc, m < M ? at : OUTSIDE_ROWS, 0, 0);
            } else if (nw + 16 * j + token < p.x.rows) {
                // (rows of any length: the same stores at the alignment of an element, but for the last few channels)
                typedef T any __attribute__((ext_vector_type(V), aligned(sizeof(T))));
                T* const to = static_cast<T*>(p.y) + (static_cast<int64_t>(nw) + 16 * j + token) * M + m;
                if (m + V <= M) *reinterpret_cast<any*>(to) = raw;
                else
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (m + e < M) to[e] = raw[e];
            }
        }
        wave_fence();
    }
}
// whether outputs leave sixteen bytes at a time
template <class T>
__device__ __forceinline__ bool whole_stores(const I8Product& p) { return p.w.rows % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0; }

// Many tokens: tiles of quantized rows.  Bound by the matrix pipe and the power it may draw: 8192 tokens of 4096 onto 4096 channels, bf16, in tiles of 256 a
// side 116 us traced (2.4 POP/s, as the library's large product reaches; matrix instructions alone, on random numbers, 3.6, on zeros 4.4), output included.
template <class T, class Loop, bool DEEP>
__global__ __launch_bounds__(Loop::THREADS, Loop::STAGE * (DEEP ? 4 : 2) > 80 << 10 ? Loop::WAVES / 4 : 2) void i8_product_kernel(const I8Product p) {
    constexpr int WN = Loop::WN, TM = Loop::TM, TN = Loop::TN, PITCH = TM * 16 + 4;
    constexpr bool CUT = DEEP && Loop::BM == 64;
    __shared__ __attribute__((aligned(128))) uint8_t even[Loop::STAGE], odd[Loop::STAGE];
    __shared__ float x_scale[Loop::BN];
    int t = xcd_contiguous_index(blockIdx.x, p.tiles_w * p.tiles_x), tm, tn, stages = p.stages;
    RowBytes W = p.w, X = p.x;
    if (CUT && p.slices > 1) {
        // (slices of the same k on one XCD: they share rows of either operand)
        t = blockIdx.x / p.slices;
        const int first = (blockIdx.x % p.slices) * p.slice_stages;
        W.base += first * TILE_K;
        X.base += first * TILE_K;
        stages = stages - first < p.slice_stages ? stages - first : p.slice_stages;
    }
    tile_of(t, p.tiles_w, p.tiles_x, tm, tn);
    const int m0 = tm * Loop::BM, n0 = tn * Loop::BN;
    for (int i = threadIdx.x; i < Loop::BN; i += Loop::THREADS) x_scale[i] = p.x_scale[n0 + i < p.x.rows ? n0 + i : p.x.rows - 1];
    v4i acc[TM][TN];
    if constexpr (DEEP) {
        __shared__ __attribute__((aligned(128))) uint8_t third[Loop::STAGE], fourth[Loop::STAGE];
        Loop::run(W, X, m0, n0, stages, even, odd, third, fourth, acc);
        if (CUT && p.slices > 1) {
            v4i* const to = p.sums + static_cast<int64_t>(blockIdx.x) * (TM * TN * Loop::THREADS) + threadIdx.x;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) to[(i * TN + j) * Loop::THREADS] = acc[i][j];
            return;
        }
    } else {
        Loop::run(W, X, m0, n0, stages, even, odd, acc);
    }
    const int wave = threadIdx.x >> 6, nw = wave % WN * TN * 16;
    static_assert(Loop::WAVES / 2 * 16 * PITCH * 4 <= Loop::STAGE, "half of the waves' sixteen tokens fit a stage");
    __syncthreads();                                    // every wave has read its last stage
    float* const lds = reinterpret_cast<float*>(wave & 1 ? odd : even) + (wave >> 1) * 16 * PITCH;
    const Channels<T, TM> ch(p, m0 + wave / WN * TM * 16);
    if (whole_stores<T>(p)) store_tokens<true>(p, ch, lds, n0 + nw, acc, x_scale + nw);
    else                    store_tokens<false>(p, ch, lds, n0 + nw, acc, x_scale + nw);
}

// The tiles that were cut: a wave for each that one of their waves had, its slices' sums added (whole numbers: the same bits as uncut), then as above
template <class T, class Loop>
__global__ __launch_bounds__(64) void i8_join_kernel(const I8Product p) {
    constexpr int WN = Loop::WN, TM = Loop::TM, TN = Loop::TN, SUMS = TM * TN * Loop::THREADS;
    __shared__ __attribute__((aligned(16))) float lds[16 * (TM * 16 + 4)];
    __shared__ float x_scale[TN * 16];
    const int lane = threadIdx.x, wave = blockIdx.x % Loop::WAVES, t = blockIdx.x / Loop::WAVES;
    int tm, tn;
    tile_of(t, p.tiles_w, p.tiles_x, tm, tn);
    const int m0 = tm * Loop::BM + wave / WN * TM * 16, n0 = tn * Loop::BN + wave % WN * TN * 16;
    if (lane < TN * 16) x_scale[lane] = p.x_scale[n0 + lane < p.x.rows ? n0 + lane : p.x.rows - 1];
    const Channels<T, TM> ch(p, m0);
    const v4i* const from = p.sums + static_cast<int64_t>(t) * p.slices * SUMS + wave * 64 + lane;
    v4i acc[TM][TN] = {};
#pragma unroll 4
    for (int s = 0; s < p.slices; ++s)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] += from[static_cast<int64_t>(s) * SUMS + (i * TN + j) * Loop::THREADS];
    wave_fence();
    if (whole_stores<T>(p)) store_tokens<true>(p, ch, lds, n0, acc, x_scale);
    else                    store_tokens<false>(p, ch, lds, n0, acc, x_scale);
}

// Few tokens (at most 16) of long rows: what counts is the weight's way from memory.  A work-group takes 16 channels, its waves every WAVES-th stage of
// k, all requested before the first product.  The tokens are quantized in every work-group, into LDS, where they are few enough for that
// to cost less than a launch of its own.  Traced: one token, f32, 4096 x 4096 6.8 us (17 MB: 2.5 TB/s, an empty launch of 2.3 included): every work-group waits
// one way to memory for its token and one for its weight, whose 64 KB are all requested at once.
constexpr int I8_FEW_WAVES = 8, I8_FEW_PART = 2048;     // elements of a row that a wave quantizes at most
__host__ __device__ constexpr int few_share(int tokens) { return tokens <= 1 ? 8 : tokens <= 2 ? 4 : tokens <= 4 ? 2 : 1; }      // waves per token

// ROUNDS: tokens that a wave quantizes, eight or fewer tokens by shares of the waves, more by two each.  R quads of every lane hold a wave's part
// of a token.
template <class T, int ROUNDS, int R>
__global__ __launch_bounds__(I8_FEW_WAVES * 64) void i8_few_kernel(const I8Product p, const I8Rows rows) {
    constexpr int DEEP = 8, WAVES = I8_FEW_WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_q[];      // [tokens][row + 16], behind it the sums
    __shared__ float x_scale[16], parts_largest[WAVES];
    __shared__ int sums[WAVES][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tokens = p.x.rows, m0 = blockIdx.x * 16, row_bytes = p.stages * TILE_K, pitch = row_bytes + 16;
    const RowBytes W = p.w;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(W.base + m0 * W.stride), 0, 0x7fffffff, 0x00020000);
    const int last = W.rows - 1 - m0, r = (lane & 15) < last ? lane & 15 : last;
    const uint32_t from = static_cast<uint32_t>(r * W.stride) + (lane >> 4) * 16u;
    v4i a[DEEP][2];
    const auto request = [&](int first) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int stage = first + d * WAVES < p.stages ? first + d * WAVES : p.stages - 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) a[d][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, from, stage * TILE_K + h * 64, 0));
        }
    };
    const auto put = [&](int64_t row, int k, uint32_t v) { if (k < row_bytes) *reinterpret_cast<uint32_t*>(lds_q + row * pitch + k) = v; };
    const int share = few_share(tokens), part = wave % share, piece = (row_bytes / 4 + 64 * share - 1) / (64 * share) * 256;      // elements of a wave's part
    const int k0 = part * piece + 4 * lane;
    const auto each = [&](auto zero) {
        typedef decltype(zero) E;
        typename Quad<E>::Raw raw[ROUNDS][R];
        // the tokens ahead of the weight: loads come back in their order, and the weight's way is the longer one
#pragma unroll
        for (int o = 0; o < ROUNDS; ++o) {
            const int t = wave / share + o * WAVES;
            const E* const row = static_cast<const E*>(rows.x) + static_cast<int64_t>(t < tokens ? t : tokens - 1) * rows.stride;
#pragma unroll
            for (int i = 0; i < R; ++i) raw[o][i] = fetch4<E>(row, 256 * i < piece ? k0 + 256 * i : rows.K, rows.K);
        }
        request(wave);
#pragma unroll
        for (int o = 0; o < ROUNDS; ++o) {
            const int t = wave / share + o * WAVES;
            float x[R][4], largest = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) finish4<E>(raw[o][i], 256 * i < piece ? k0 + 256 * i : rows.K, rows.K, x[i]);
            RowScale scale;
            if constexpr (sizeof(E) > 1) {
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) largest = largest_of(largest, __builtin_fabsf(x[i][e]));
                largest = wave_butterfly(largest, [](float a, float b) { return largest_of(a, b); });
                if (ROUNDS == 1 && share > 1) {
                    if (lane == 0) parts_largest[wave] = largest;
                    __syncthreads();
                    largest = 0.0f;
                    for (int w = 0; w < share; ++w) largest = largest_of(largest, parts_largest[wave - part + w]);
                }
                scale = RowScale(largest);
                if (lane == 0 && part == 0 && t < tokens) x_scale[t] = scale.scale;
            }
            if (t < tokens) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (256 * i < piece) put(t, k0 + 256 * i, sizeof(E) == 1 ? pack4(x[i]) : quantize4(x[i], scale));
            }
        }
    };
    switch (rows.type) {
        case PPML_ELEM_F32:  each(0.0f); break;
        case PPML_ELEM_F16:  each(static_cast<_Float16>(0)); break;
        case PPML_ELEM_BF16: each(static_cast<__bf16>(0)); break;
        default:             each(static_cast<int8_t>(0)); break;
    }
    if (rows.type == PPML_ELEM_I8 && static_cast<int>(threadIdx.x) < tokens) x_scale[threadIdx.x] = rows.scale[threadIdx.x];
    __syncthreads();
    const uint8_t* const token = lds_q + ((lane & 15) < tokens ? lane & 15 : tokens - 1) * pitch + (lane >> 4) * 16;
    v4i acc{};
    for (int first = wave; first < p.stages; first += WAVES * DEEP) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int stage = first + d * WAVES;
            if (stage < p.stages) {
                const v4i b[2] = {*reinterpret_cast<const v4i*>(token + stage * TILE_K), *reinterpret_cast<const v4i*>(token + stage * TILE_K + 64)};
                StepI8::step<0>(a[d], b, acc);
                StepI8::step<1>(a[d], b, acc);
            }
        }
        if (first + WAVES * DEEP < p.stages) request(first + WAVES * DEEP);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][lane & 15][(lane >> 4) * 4 + e] = acc[e];
    __syncthreads();
    const int n = threadIdx.x >> 4, m = m0 + (threadIdx.x & 15);
    if (n >= tokens || m >= W.rows) return;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += sums[w][n][threadIdx.x & 15];
    const float v = static_cast<float>(sum) * x_scale[n] * p.w_scale[m];
    static_cast<T*>(p.y)[static_cast<int64_t>(n) * W.rows + m] = from_f32<T>(p.bias ? v + p.bias[m] : v);
}

// Short rows (at most 128 S elements) and more tokens: bound by the way of x and y from and to memory.  A wave keeps its 64 channels of the weight
// in registers, a work-group stays and takes every gridDim.x-th group of 4 WAVES tokens: their rows, requested a group ahead, are quantized
// into LDS by all its waves, and every wave multiplies them with its channels.  One launch, x read once (once per part of 64 WAVES channels).
// A wave quantizes four rows at a time, sixteen lanes each: the search for the largest then takes four steps for four rows (a row
// at a time by 64 lanes, six steps each, the alignment's projection was bound by it: 39 us).  Traced: 26368 tokens of 256, f32, onto 768 channels 24.3 us
// (4.4 TB/s); 408 onto 256 4.4 us.
template <class T, bool VEC, int S, int WAVES, int TM>
__global__ __launch_bounds__(WAVES * 64) void i8_stay_kernel(const I8Product p, const I8Rows rows) {
    constexpr int TN = WAVES / 4, TOKENS = TN * 16, PITCH = TM * 16 + 4, ROW = S * TILE_K, LDS_ROW = ROW + 16;
    constexpr int QUADS = ROW / 64;                     // of a row per lane
    __shared__ __attribute__((aligned(16))) float out_all[WAVES][16 * PITCH];
    __shared__ __attribute__((aligned(16))) uint8_t lds_q[2][TOKENS * LDS_ROW];
    __shared__ float x_scale[2][TOKENS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tokens = p.x.rows, groups = (tokens + TOKENS - 1) / TOKENS;
    const int mw = (blockIdx.y * WAVES + wave) * 16 * TM;
    const RowBytes W = p.w;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(W.base), 0, static_cast<int>(W.rows * W.stride), 0x00020000);
    v4i a[S][TM][2];
    {
        // (rows behind the last one lie outside the resource and read as nothing)
        const uint32_t from = static_cast<uint32_t>((mw + (lane & 15)) * W.stride) + (lane >> 4) * 16u;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a[s][i][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, from + static_cast<uint32_t>(16 * i * W.stride) + s * TILE_K + h * 64, 0, 0));
    }
    const Channels<T, TM> ch(p, mw);
    float* const out = out_all[wave];
    const int mine = wave * 4 + (lane >> 4), k0 = (lane & 15) * 4;      // the row of the group, and the first element, that this lane quantizes
    // (what is loaded once is here before the loop begins: waits for it inside would be waits for the rows requested there as well)
    __builtin_amdgcn_s_waitcnt(0x0f70);                 // vmcnt(0)
    const auto run = [&](auto zero) {
        typedef decltype(zero) E;
        typename Quad<E>::Raw raw[QUADS];
        float given = 0.0f;
        // (without a condition: past the last token the last one)
        const auto request = [&](int group) {
            const int64_t t = static_cast<int64_t>(group) * TOKENS + mine, at = t < tokens ? t : tokens - 1;
            const E* const row = static_cast<const E*>(rows.x) + at * rows.stride;
#pragma unroll
            for (int i = 0; i < QUADS; ++i) raw[i] = fetch4<E>(row, k0 + 64 * i, rows.K);
            if constexpr (sizeof(E) == 1) given = rows.scale[at];
        };
        int group = blockIdx.x, side = 0;
        request(group);
        for (; group < groups; group += gridDim.x, side ^= 1) {
            float x[QUADS][4];
            RowScale scale;
            scale.scale = given;
#pragma unroll
            for (int i = 0; i < QUADS; ++i) finish4<E>(raw[i], k0 + 64 * i, rows.K, x[i]);
            if constexpr (sizeof(E) > 1) {
                float largest = 0.0f;
#pragma unroll
                for (int i = 0; i < QUADS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) largest = largest_of(largest, __builtin_fabsf(x[i][e]));
                scale = RowScale(row16_butterfly(largest, [](float u, float v) { return largest_of(u, v); }));
            }
#pragma unroll
            for (int i = 0; i < QUADS; ++i)
                *reinterpret_cast<uint32_t*>(lds_q[side] + mine * LDS_ROW + k0 + 64 * i) = sizeof(E) == 1 ? pack4(x[i]) : quantize4(x[i], scale);
            if ((lane & 15) == 0) x_scale[side][mine] = scale.scale;
            request(group + gridDim.x);
            __syncthreads();                            // (the group before this one was read before the last one of these)
            v4i acc[TM][TN];
#pragma unroll
            for (int u = 0; u < TM; ++u)
#pragma unroll
                for (int v = 0; v < TN; ++v) acc[u][v] = v4i{};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                v4i b[TN][2];
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        b[j][h] = *reinterpret_cast<const v4i*>(lds_q[side] + (16 * j + (lane & 15)) * LDS_ROW + s * TILE_K + h * 64 + (lane >> 4) * 16);
                step_tiles<StepI8>(a[s], b, acc);
            }
            store_tokens<VEC>(p, ch, out, group * TOKENS, acc, x_scale[side]);
        }
    };
    switch (rows.type) {
        case PPML_ELEM_F32:  run(0.0f); break;
        case PPML_ELEM_F16:  run(static_cast<_Float16>(0)); break;
        case PPML_ELEM_BF16: run(static_cast<__bf16>(0)); break;
        default:             run(static_cast<int8_t>(0)); break;
    }
}

int64_t i8_row_bytes(int64_t K) { return (K + TILE_K - 1) / TILE_K * TILE_K; }

template <class T>
void launch_quantize(const I8Rows& p, int8_t* q, int64_t q_stride, int q_end, float* scale, int64_t waves, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((waves + 3) / 4)), block(256);
    const int pieces = (p.K + 255) / 256;
    // (rows that a wave holds as well, where there are few of them)
    if ((pieces > 16 ? p.rows <= LAUNCH_MOST_THREADS / (64 * I8_ROW_WAVES) : pieces > 4 && p.rows <= 4 * device_cu_count()) && pieces <= 16 * I8_ROW_WAVES) {
        const dim3 rows(static_cast<unsigned>(p.rows)), row(64 * I8_ROW_WAVES);
        if (pieces <= I8_ROW_WAVES)          hipLaunchKernelGGL((i8_quantize_row_kernel<T, 1>), rows, row, 0, stream, p, q, q_stride, q_end, scale);
        else if (pieces <= 2 * I8_ROW_WAVES) hipLaunchKernelGGL((i8_quantize_row_kernel<T, 2>), rows, row, 0, stream, p, q, q_stride, q_end, scale);
        else if (pieces <= 4 * I8_ROW_WAVES) hipLaunchKernelGGL((i8_quantize_row_kernel<T, 4>), rows, row, 0, stream, p, q, q_stride, q_end, scale);
        else if (pieces <= 8 * I8_ROW_WAVES) hipLaunchKernelGGL((i8_quantize_row_kernel<T, 8>), rows, row, 0, stream, p, q, q_stride, q_end, scale);
        else                                 hipLaunchKernelGGL((i8_quantize_row_kernel<T, 16>), rows, row, 0, stream, p, q, q_stride, q_end, scale);
    }
    else if (p.K < 4 || pieces > 16) hipLaunchKernelGGL((i8_quantize_kernel<T, 0>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
    else if (pieces <= 1)  hipLaunchKernelGGL((i8_quantize_kernel<T, 1>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
    else if (pieces <= 2)  hipLaunchKernelGGL((i8_quantize_kernel<T, 2>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
    else if (pieces <= 4)  hipLaunchKernelGGL((i8_quantize_kernel<T, 4>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
    else if (pieces <= 8)  hipLaunchKernelGGL((i8_quantize_kernel<T, 8>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
    else                   hipLaunchKernelGGL((i8_quantize_kernel<T, 16>), grid, block, 0, stream, p, q, q_stride, q_end, scale);
}
int launch_quantize(const I8Rows& p, int8_t* q, int64_t q_stride, int q_end, float* scale, hipStream_t stream, const char* what) {
    const int pieces = (p.K + 255) / 256, per_wave = p.K < 4 ? 1 : pieces <= 1 ? 8 : pieces <= 2 ? 4 : pieces <= 4 ? 2 : 1;
    if (p.rows > LAUNCH_MOST_THREADS / 256 * 4 * per_wave) { set_error("%s: too many rows (%lld)", what, (long long)p.rows); return RC_BAD_ARGS; }
    const int64_t waves = (p.rows + per_wave - 1) / per_wave;
    switch (p.type) {
        case PPML_ELEM_F32:  launch_quantize<float>(p, q, q_stride, q_end, scale, waves, stream); break;
        case PPML_ELEM_F16:  launch_quantize<_Float16>(p, q, q_stride, q_end, scale, waves, stream); break;
        case PPML_ELEM_BF16: launch_quantize<__bf16>(p, q, q_stride, q_end, scale, waves, stream); break;
        default:             launch_quantize<int8_t>(p, q, q_stride, q_end, scale, waves, stream); break;
    }
    return check_launch(what);
}

template <class T, class Loop, bool DEEP>
int launch_tiles(I8Product p, hipStream_t stream) {
    p.tiles_w = (p.w.rows + Loop::BM - 1) / Loop::BM;
    p.tiles_x = (p.x.rows + Loop::BN - 1) / Loop::BN;
    if (static_cast<int64_t>(p.tiles_w) * p.tiles_x * p.slices > LAUNCH_MOST_THREADS / Loop::THREADS) { set_error("mul_mat_i8_hip: too many tiles"); return RC_BAD_ARGS; }
    hipLaunchKernelGGL((i8_product_kernel<T, Loop, DEEP>), dim3(static_cast<unsigned>(p.tiles_w * p.tiles_x * p.slices)), dim3(Loop::THREADS), 0, stream, p);
    if constexpr (DEEP && Loop::BM == 64)
        if (p.slices > 1) hipLaunchKernelGGL((i8_join_kernel<T, Loop>), dim3(static_cast<unsigned>(p.tiles_w * p.tiles_x * Loop::WAVES)), dim3(64), 0, stream, p);
    return check_launch("mul_mat_i8_hip");
}

template <class T, int S, int WAVES, int TM>
void launch_stay_waves(const I8Product& p, const I8Rows& rows, hipStream_t stream) {
    constexpr int CHANNELS = 16 * TM * WAVES;
    const bool vec = p.w.rows % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
    const int parts = (p.w.rows + CHANNELS - 1) / CHANNELS, groups = (p.x.rows + 4 * WAVES - 1) / (4 * WAVES);
    // measured, 26368 tokens of 256: onto 256 channels 256 / 512 / 768 / 1024 work-groups of four waves 15.5 / 14.5 / 15.7 / 18.9 us (eight waves
    // 16.1), onto 768 work-groups of eight waves 25.6 / 30.0 / 33.5 / 36.9 (four waves 27.3 at best, twelve 32.5)
    int wgs = (WAVES == 4 ? 2 : 1) * device_cu_count() / parts;
    if (wgs < 1) wgs = 1;
    if (wgs > groups) wgs = groups;
    const dim3 grid(wgs, parts), block(64 * WAVES);
    if (vec) hipLaunchKernelGGL((i8_stay_kernel<T, true, S, WAVES, TM>), grid, block, 0, stream, p, rows);
    else     hipLaunchKernelGGL((i8_stay_kernel<T, false, S, WAVES, TM>), grid, block, 0, stream, p, rows);
}
template <class T, int S>
void launch_stay(const I8Product& p, const I8Rows& rows, hipStream_t stream) {
    // What a CU gets from memory by itself is some 40 GB/s, and the L2s begin every launch empty: the weight of a product of few tokens is spread over
    // small work-groups as long as the large ones are fewer than three quarters of the CUs (small / large, us: 32 tokens x 512 -> 512 5.3 / 12.2, 2601 x 512 ->
    // 512 10.0 / 13.1, 2601 x 500 -> 1001 12.8 / 15.3, 5000 x 256 -> 2048 19.3 / 16.6, 26368 x 256 -> 768 39.9 / 27.8).
    const int64_t large = static_cast<int64_t>((p.x.rows + 31) / 32) * ((p.w.rows + 511) / 512);
    if (4 * large <= 3 * device_cu_count()) launch_stay_waves<T, S, 4, 2>(p, rows, stream);
    else if (p.w.rows <= 256) launch_stay_waves<T, S, 4, 4>(p, rows, stream);
    else launch_stay_waves<T, S, 8, 4>(p, rows, stream);
}

// How a product is made
enum I8Form { I8_FEW, I8_STAY, I8_TILES };
constexpr int I8_FEW_LDS = 40 << 10, I8_STAY_STAGES = 4;
I8Form i8_form(int M, int N, int K) {
    const int64_t row = i8_row_bytes(K);
    if (K < 4) return I8_TILES;                         // (the rows are fetched four elements at a time)
    // (tiles behind a quantizing launch / staying, f16, us: 2601 tokens of 512 onto 512 channels 9.2 / 10.2, onto 1024 10.7 / 12.8, onto 4096 21.3 / 24.2; on either side of
    // the range 512 onto 1024 7.6 / 5.5, 10000 onto 1024 23.7 / 23.4, 30000 onto 512 29.9 / 27.4)
    const int64_t outputs = static_cast<int64_t>(N) * M;
    if (row > 2 * TILE_K && row <= I8_STAY_STAGES * TILE_K && M > 256 && outputs >= 1 << 20 && outputs <= 11 << 20) return I8_TILES;
    if (row <= I8_STAY_STAGES * TILE_K && (M + 511) * row < 0x7fffffff) return I8_STAY;
    if (N <= 16 && row <= I8_FEW_PART * few_share(N) && N * (row + 16) <= I8_FEW_LDS) return I8_FEW;
    return I8_TILES;
}

// Tiles of `side`; few of 64 under a long k are cut along it
struct I8Tiles { int side; CutTiles cut; };
I8Tiles i8_tiles(int64_t M, int64_t N, int K) {
    const auto tiles = [&](int side) { return (M + side - 1) / side * ((N + side - 1) / side); };
    const CutTiles few = cut_few_tiles(tiles(64), static_cast<int>(i8_row_bytes(K) / TILE_K));
    I8Tiles t{};
    t.side = tile_side([&](int side) { return static_cast<double>(tiles(side)); }, 2.2, 0.0, few.rounds);
    if (t.side == 64) t.cut = few;
    return t;
}

template <class T>
int launch_product(const I8Product& p, const I8Rows& rows, int8_t* q, float* scale, I8Form form, const I8Tiles& tiles, bool in_place, hipStream_t stream) {
    const int row = p.stages * TILE_K;
    if (form == I8_FEW) {
        const dim3 grid(static_cast<unsigned>((p.w.rows + 15) / 16));
        const size_t lds = static_cast<size_t>(p.x.rows) * (row + 16);
        const dim3 block(I8_FEW_WAVES * 64);
        if (p.x.rows > I8_FEW_WAVES)              hipLaunchKernelGGL((i8_few_kernel<T, 2, I8_FEW_PART / 256>), grid, block, lds, stream, p, rows);
        else if (row > 512 * few_share(p.x.rows)) hipLaunchKernelGGL((i8_few_kernel<T, 1, I8_FEW_PART / 256>), grid, block, lds, stream, p, rows);
        else                                      hipLaunchKernelGGL((i8_few_kernel<T, 1, 2>), grid, block, lds, stream, p, rows);
        return check_launch("mul_mat_i8_hip");
    }
    if (form == I8_STAY) {
        if (p.stages == 1)      launch_stay<T, 1>(p, rows, stream);
        else if (p.stages == 2) launch_stay<T, 2>(p, rows, stream);
        else                    launch_stay<T, 4>(p, rows, stream);
        return check_launch("mul_mat_i8_hip");
    }
    if (!in_place) {
        const int rc = launch_quantize(rows, q, row, row, scale, stream, "mul_mat_i8_hip");
        if (rc != RC_OK) return rc;
    }
    switch (tiles.side) {
        case 256: return launch_tiles<T, TilePingPong<StepI8>, false>(p, stream);
        case 128: return launch_tiles<T, TileDeep<StepI8, 2, 4, 4, 2>, true>(p, stream);
        default:  return launch_tiles<T, TileDeep<StepI8, 2, 2, 2, 2>, true>(p, stream);
    }
}

bool float_type(int type) { return type == PPML_ELEM_F32 || type == PPML_ELEM_F16 || type == PPML_ELEM_BF16; }

}  // namespace
}  // namespace ppmlhip

using namespace ppmlhip;

extern "C" int quantize_rows_i8_hip(const void* x, int type, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t rows, int K,
                                    ppml_hip_stream_t stream) {
    if (!x || !q || !float_type(type) || !scale || rows <= 0 || K <= 0 || K > I8_MAX_K || x_stride < K || q_stride < K) {
        set_error("quantize_rows_i8_hip: bad arguments (rows=%lld K=%d type=%d)", (long long)rows, K, type);
        return RC_BAD_ARGS;
    }
    const int end = q_stride == i8_row_bytes(K) ? static_cast<int>(q_stride) : K;
    return launch_quantize(I8Rows{x, type, x_stride, nullptr, rows, K}, q, q_stride, end, scale, static_cast<hipStream_t>(stream), "quantize_rows_i8_hip");
}

extern "C" size_t i8_weight_row_bytes_hip(int K) { return K > 0 && K <= I8_MAX_K ? static_cast<size_t>(i8_row_bytes(K)) : 0; }

extern "C" int i8_weight_pack_hip(const int8_t* w, int64_t w_stride, int M, int K, int8_t* packed, ppml_hip_stream_t stream) {
    if (!w || !packed || M <= 0 || K <= 0 || K > I8_MAX_K || w_stride < K) {
        set_error("i8_weight_pack_hip: bad arguments (M=%d K=%d)", M, K);
        return RC_BAD_ARGS;
    }
    const int64_t row = i8_row_bytes(K);
    return launch_quantize(I8Rows{w, PPML_ELEM_I8, w_stride, nullptr, M, K}, packed, row, static_cast<int>(row), nullptr, static_cast<hipStream_t>(stream),
                           "i8_weight_pack_hip");
}

// (the workspace: the quantized rows, their scales, and from here on the sums of tiles that are cut)
static int64_t i8_sums_at(int64_t N, int K) { return N * i8_row_bytes(K) + (4 * N + 15) / 16 * 16; }

extern "C" size_t mul_mat_i8_workspace_hip(int M, int N, int K) {
    if (M <= 0 || M > I8_MAX_M || N <= 0 || N > I8_MAX_N || K <= 0 || K > I8_MAX_K || i8_form(M, N, K) != I8_TILES) return 0;
    const CutTiles cut = i8_tiles(M, N, K).cut;
    return static_cast<size_t>(i8_sums_at(N, K)) + static_cast<size_t>(cut.left * cut.slices) * (64 * 64 * 4);
}

extern "C" int mul_mat_i8_hip(const int8_t* packed, const float* w_scale, const void* x, int x_type, int64_t x_stride, const float* x_scale, const float* bias,
                              void* y, int y_type, int M, int N, int K, void* workspace, size_t workspace_bytes, ppml_hip_stream_t stream_) {
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (!packed || !w_scale || !x || !y || M <= 0 || M > I8_MAX_M || N <= 0 || N > I8_MAX_N || K <= 0 || K > I8_MAX_K || x_stride < K || !float_type(y_type) ||
        (x_type == PPML_ELEM_I8 ? !x_scale : !float_type(x_type)) || (reinterpret_cast<uintptr_t>(packed) & 15) != 0) {
        set_error("mul_mat_i8_hip: bad arguments (M=%d N=%d K=%d x_type=%d y_type=%d)", M, N, K, x_type, y_type);
        return RC_BAD_ARGS;
    }
    const size_t need = mul_mat_i8_workspace_hip(M, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) {
        set_error("mul_mat_i8_hip: needs %zu bytes of workspace, 16-byte aligned (got %zu)", need, workspace_bytes);
        return RC_BAD_ARGS;
    }
    StatsScope stats("i8", N, K, M, stream);
    const int64_t row = i8_row_bytes(K);
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scale = q ? reinterpret_cast<float*>(q + static_cast<int64_t>(N) * row) : nullptr;
    I8Product p{};
    p.w = RowBytes{reinterpret_cast<const uint8_t*>(packed), row, M};
    p.x = RowBytes{reinterpret_cast<const uint8_t*>(q), row, N};
    p.w_scale = w_scale;
    p.x_scale = x_type == PPML_ELEM_I8 ? x_scale : scale;
    p.bias = bias;
    p.y = y;
    p.stages = static_cast<int>(row / TILE_K);
    const I8Rows rows{x, x_type, x_stride, x_scale, N, K};
    I8Form form = i8_form(M, N, K);
    // Quantized rows that lie as tiles read them are read where they are: tiles then need no launch before them, and no workspace where they are not cut
    const bool in_place = x_type == PPML_ELEM_I8 && K % TILE_K == 0 && x_stride % 16 == 0 && x_stride <= 1 << 20 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    if (in_place) {
        p.x = RowBytes{static_cast<const uint8_t*>(x), x_stride, N};
        // (tiles / staying, us: 2601 x 512 -> 1024 6.4 / 10.5, 30000 x 512 -> 512 16.7 / 24.5, 100 x 512 -> 1024 3.6 / 5.1, 30000 x 512 -> 128 8.0 / 15.7, 26368 x 256 -> 256
        // 11.2 / 12.0, -> 768 23.8 / 22.8, 5000 x 256 -> 2048 13.7 / 13.6, 10609 x 128 -> 512 9.6 / 8.4)
        if (form == I8_STAY && N >= 64 && (row > 2 * TILE_K || (row == 2 * TILE_K && static_cast<int64_t>(N) * M <= 8 << 20))) form = I8_TILES;
    }
    const I8Tiles tiles = form == I8_TILES ? i8_tiles(M, N, K) : I8Tiles{};
    p.slices = tiles.cut.left > 0 ? tiles.cut.slices : 1;
    p.slice_stages = tiles.cut.left > 0 ? tiles.cut.stages : p.stages;
    p.sums = p.slices > 1 ? reinterpret_cast<v4i*>(q + i8_sums_at(N, K)) : nullptr;
    switch (y_type) {
        case PPML_ELEM_F32:  return launch_product<float>(p, rows, q, scale, form, tiles, in_place, stream);
        case PPML_ELEM_F16:  return launch_product<_Float16>(p, rows, q, scale, form, tiles, in_place, stream);
        default:             return launch_product<__bf16>(p, rows, q, scale, form, tiles, in_place, stream);
    }
}
