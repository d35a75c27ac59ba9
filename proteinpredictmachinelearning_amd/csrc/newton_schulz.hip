// Updates orthogonalised by Newton-Schulz products (newton_schulz_hip).
//
//   X_0 = G / (|G| + eps)       |G| the Frobenius norm; G with its shorter side as rows
//   A = X X^T      B = b A + c A A      X <- a X + B X        `steps` times
//
// Every singular value s of G / (|G| + eps) becomes p(p(...p(s))), p(s) = a s + b s^3 + c s^5; its vectors stay.  A step
// multiplies small singular values by a (3.4 as a rule), and with them the errors made before: the arithmetic is binary32's in
// every step whatever the type of G.
//
// Between the products a matrix is kept as its operand, two halves x 2^e = h + l (to 2^-23, or 2^-25 absolute where below
// 2^-2): rows along k in groups of 32 elements, 64 bytes of upper parts and 64 of lower ones.  e is one exponent per matrix and step: no entry
// is larger than the spectral norm, which a bound on the singular values follows through the steps (next_bound), from |G| / (|G| + eps)
// on.  A and A A are symmetric: only the tiles on and above the diagonal are computed, and written twice.
//
// X is kept twice, by rows for A and as X^T for B X, both of whose operands have to run along k.
#include "elements.hpp"
#include "tile_product.hpp"

namespace ppmlhip {
namespace {

constexpr int NS_MOST_STEPS = 32, NS_NORM_BLOCKS = 64;
constexpr int64_t NS_MOST_SIDE = 1 << 20;

// (per matrix) what the launches multiply by: sums of products and the matrix that is added, to the next operand's scale
struct NsFactors { float of_sum[3 * NS_MOST_STEPS], of_added[3 * NS_MOST_STEPS]; };

struct NsCoefficients { float a, b, c; };

// the largest |p(s)| for 0 <= s <= v
__device__ double next_bound(double v, const NsCoefficients& k) {
    const auto p = [&](double s) { const double z = s * s; return fabs(s * (k.a + z * (k.b + z * k.c))); };
    double most = p(v);
    // p'(s) = a + 3 b z + 5 c z^2 = 0, z = s^2
    const double qa = 5.0 * k.c, qb = 3.0 * k.b, qc = k.a;
    double z[2] = {-1.0, -1.0};
    if (qa == 0.0) {
        if (qb != 0.0) z[0] = -qc / qb;
    } else {
        const double disc = qb * qb - 4.0 * qa * qc;
        if (disc >= 0.0) {
            z[0] = (-qb + sqrt(disc)) / (2.0 * qa);
            z[1] = (-qb - sqrt(disc)) / (2.0 * qa);
        }
    }
    for (const double x : z)
        if (x > 0.0 && x < v * v) most = fmax(most, p(sqrt(x)));
    return most;
}
// the largest |b z + c z^2| for 0 <= z <= v^2
__device__ double poly_bound(double v, const NsCoefficients& k) {
    const double z = v * v;
    double most = fabs(z * (k.b + z * k.c));
    if (k.c != 0.0f) {
        const double at = -k.b / (2.0 * k.c);
        if (at > 0.0 && at < z) most = fmax(most, fabs(at * (k.b + at * k.c)));
    }
    return most;
}
// the exponent under which entries of at most `bound` stay below 2^16
__device__ int operand_exponent(double bound) {
    if (!(bound > 0.0) || !(bound < 1e300)) return 0;
    int e;
    (void)frexp(bound * 1.01, &e);                      // bound 1.01 < 2^e (the hundredth: what the steps' roundings may add)
    e = 15 - e;
    return e < -100 ? -100 : (e > 100 ? 100 : e);
}

// ------------------------------------------------------------------------------------------------------------ norm
template <class T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* g, int64_t count, double* partial) {
    __shared__ double lds[256];
    const T* const x = g + blockIdx.y * count;
    double sum = 0.0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * 256) {
        const double v = static_cast<double>(to_f32(x[i]));
        sum = fma(v, v, sum);
    }
    lds[threadIdx.x] = sum;
    __syncthreads();
    for (int step = 128; step > 0; step >>= 1) {
        if (static_cast<int>(threadIdx.x) < step) lds[threadIdx.x] += lds[threadIdx.x + step];
        __syncthreads();
    }
    if (threadIdx.x == 0) partial[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = lds[0];
}

// ------------------------------------------------------------------------------------------------------------ operands
// Where an element lies in an operand: its upper half (the lower one 64 bytes behind)
__device__ __forceinline__ int64_t operand_at(int64_t row, int64_t stride, int k) { return row * stride + (k >> 5) * 128 + (k & 31) * 2; }
__device__ __forceinline__ float operand_value(const uint8_t* at) {
    return static_cast<float>(*reinterpret_cast<const _Float16*>(at)) + static_cast<float>(*reinterpret_cast<const _Float16*>(at + 64));
}
__device__ __forceinline__ void put_operand(uint8_t* at, float x) {
    const _Float16 h = static_cast<_Float16>(x);
    *reinterpret_cast<_Float16*>(at) = h;
    *reinterpret_cast<_Float16*>(at + 64) = static_cast<_Float16>(x - static_cast<float>(h));
}

struct NsStart {
    const void* g;
    const double* partial;
    uint8_t *x, *xt;
    NsFactors* factors;
    int rows, cols;           // of G as it lies
    int tall, steps, parts;
    int64_t x_stride, xt_stride, x_matrix, xt_matrix;      // X has min(rows, cols) rows
    float eps;
    NsCoefficients k;
};

// 64 x 64 elements of G per work-group: X_0 and its transpose, zeros behind the last column of either
template <class T>
__global__ __launch_bounds__(256) void ns_start_kernel(const NsStart p) {
    __shared__ float lds[64][65];
    const int64_t z = blockIdx.z;
    const int tid = threadIdx.x;
    double norm = 0.0;
    for (int i = 0; i < p.parts; ++i) norm += p.partial[z * p.parts + i];
    norm = sqrt(norm);
    const double inverse = norm < 1e300 ? 1.0 / (norm + static_cast<double>(p.eps)) : __longlong_as_double(0x7ff8000000000000ll);
    const double first = norm * inverse;
    const int e0 = operand_exponent(first);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
        NsFactors& f = p.factors[z];
        double bound = first;
        int ex = e0;
        for (int s = 0; s < p.steps; ++s) {
            const int ea = operand_exponent(bound * bound), eb = operand_exponent(poly_bound(bound, p.k));
            bound = next_bound(bound, p.k);
            const int en = s + 1 < p.steps ? operand_exponent(bound) : 0;      // (the last X leaves unscaled)
            f.of_sum[3 * s] = ldexpf(1.0f, ea - 2 * ex);
            f.of_added[3 * s] = 0.0f;
            f.of_sum[3 * s + 1] = ldexpf(p.k.c, eb - 2 * ea);
            f.of_added[3 * s + 1] = ldexpf(p.k.b, eb - ea);
            f.of_sum[3 * s + 2] = ldexpf(1.0f, en - eb - ex);
            f.of_added[3 * s + 2] = ldexpf(p.k.a, en - ex);
            ex = en;
        }
    }
    const double factor = ldexp(inverse, e0);
    const T* const g = static_cast<const T*>(p.g) + z * p.rows * p.cols;
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    // G as it lies goes to `same`, transposed to `turned`
    uint8_t* const same = p.tall ? p.xt + z * p.xt_matrix : p.x + z * p.x_matrix;
    uint8_t* const turned = p.tall ? p.x + z * p.x_matrix : p.xt + z * p.xt_matrix;
    const int64_t same_stride = p.tall ? p.xt_stride : p.x_stride, turned_stride = p.tall ? p.x_stride : p.xt_stride;
    for (int i = tid; i < 64 * 64; i += 256) {
        const int r = i >> 6, c = i & 63;
        float x = 0.0f;
        if (r0 + r < p.rows && c0 + c < p.cols) x = static_cast<float>(static_cast<double>(to_f32(g[static_cast<int64_t>(r0 + r) * p.cols + c0 + c])) * factor);
        lds[r][c] = x;
        if (r0 + r < p.rows && (c0 + c) < (p.cols + 31) / 32 * 32) put_operand(same + operand_at(r0 + r, same_stride, c0 + c), x);
    }
    __syncthreads();
    for (int i = tid; i < 64 * 64; i += 256) {
        const int c = i >> 6, r = i & 63;
        if (c0 + c < p.cols && r0 + r < (p.rows + 31) / 32 * 32) put_operand(turned + operand_at(c0 + c, turned_stride, r0 + r), lds[r][c]);
    }
}

// ------------------------------------------------------------------------------------------------------------ products
struct NsProduct {
    RowBytes a, b;            // of the first matrix of the batch
    const uint8_t* added;     // rows as the sum's, or null
    uint8_t *out, *turned;    // the sum as an operand and transposed (null: not wanted; symmetric: `out` is written twice)
    void* final;              // the last step: the result instead, [rows][cols], or [cols][rows] where G was turned
    int64_t a_matrix, b_matrix, added_matrix, added_stride, out_matrix, out_stride, turned_matrix, turned_stride, final_matrix;
    const NsFactors* factors;
    int which;                // 3 step + product
    int tiles_m, tiles_n, stages, symmetric, final_turned;
};

template <class T, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM * WN * 64) void ns_product_kernel(const NsProduct p) {
    typedef TileLoop<StepF16x2, WM, WN, TM, TN> Loop;
    const int64_t z = blockIdx.y;
    int t = xcd_contiguous_index(blockIdx.x, gridDim.x);
    int tm, tn;
    if (p.symmetric) {
        // the t-th tile on or above the diagonal, by rows
        tm = 0;
        while (t >= p.tiles_n - tm) { t -= p.tiles_n - tm; ++tm; }
        tn = tm + t;
    } else {
        tm = t % p.tiles_m;
        tn = t / p.tiles_m;
    }
    const int m0 = tm * Loop::BM, n0 = tn * Loop::BN;
    RowBytes A = p.a, B = p.b;
    A.base += z * p.a_matrix;
    B.base += z * p.b_matrix;
    v4f acc[TM][TN];
    Loop::run(A, B, m0, n0, p.stages, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mw = m0 + wave / WN * TM * 16 + (lane >> 4) * 4, nw = n0 + wave % WN * TN * 16 + (lane & 15);
    const float of_sum = p.factors[z].of_sum[p.which], of_added = p.factors[z].of_added[p.which];
    const int M = A.rows, N = B.rows, M32 = (M + 31) / 32 * 32, N32 = (N + 31) / 32 * 32;
    const bool mirror = p.symmetric && tm != tn;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = mw + 16 * i + r, n = nw + 16 * j;
                const bool inside = m < M && n < N;
                float v = 0.0f;
                if (inside) {
                    v = acc[i][j][r] * of_sum;
                    if (p.added) v = fmaf(operand_value(p.added + z * p.added_matrix + operand_at(m, p.added_stride, n)), of_added, v);
                }
                if (p.final) {
                    T* const y = static_cast<T*>(p.final) + z * p.final_matrix;
                    if (inside) y[p.final_turned ? static_cast<int64_t>(n) * M + m : static_cast<int64_t>(m) * N + n] = from_f32<T>(v);
                } else {
                    if (m < M && n < N32) put_operand(p.out + z * p.out_matrix + operand_at(m, p.out_stride, n), v);
                    if (mirror && n < N && m < M32) put_operand(p.out + z * p.out_matrix + operand_at(n, p.out_stride, m), v);
                    if (p.turned && n < N && m < M32) put_operand(p.turned + z * p.turned_matrix + operand_at(n, p.turned_stride, m), v);
                }
            }
}

// ------------------------------------------------------------------------------------------------------------ host side
struct NsLayout {
    int64_t m, n;             // m <= n
    int64_t x_stride, xt_stride, sq_stride;              // bytes of a row of X, of X^T and A
    int64_t x, xt, x2, xt2, a, b, partial, factors, total;
};
int64_t operand_row(int64_t k) { return (k + 31) / 32 * 128; }

NsLayout ns_layout(int64_t batch, int64_t rows, int64_t cols) {
    NsLayout l{};
    l.m = rows < cols ? rows : cols;
    l.n = rows < cols ? cols : rows;
    l.x_stride = operand_row(l.n);
    l.xt_stride = l.sq_stride = operand_row(l.m);
    int64_t at = 0;
    const auto take = [&](int64_t bytes) { const int64_t here = at; at += (bytes + 255) / 256 * 256; return here; };
    l.x = take(batch * l.m * l.x_stride);
    l.xt = take(batch * l.n * l.xt_stride);
    l.x2 = take(batch * l.m * l.x_stride);
    l.xt2 = take(batch * l.n * l.xt_stride);
    l.a = take(batch * l.m * l.sq_stride);
    l.b = take(batch * l.m * l.sq_stride);
    l.partial = take(batch * NS_NORM_BLOCKS * 8);
    l.factors = take(batch * static_cast<int64_t>(sizeof(NsFactors)));
    l.total = at;
    return l;
}

bool ns_fits(int64_t batch, int64_t rows, int64_t cols) {
    return batch > 0 && batch <= 65535 && rows > 0 && cols > 0 && rows <= NS_MOST_SIDE && cols <= NS_MOST_SIDE;
}

template <class T>
int run_newton_schulz(const void* g, void* out, int64_t batch, int64_t rows, int64_t cols, int steps, const NsCoefficients& k, float eps, uint8_t* ws,
                      hipStream_t stream) {
    const NsLayout l = ns_layout(batch, rows, cols);
    double* const partial = reinterpret_cast<double*>(ws + l.partial);
    NsFactors* const factors = reinterpret_cast<NsFactors*>(ws + l.factors);
    const int64_t count = rows * cols;
    int norm_blocks = static_cast<int>((count + 4095) / 4096 < NS_NORM_BLOCKS ? (count + 4095) / 4096 : NS_NORM_BLOCKS);
    hipLaunchKernelGGL((ns_norm_kernel<T>), dim3(norm_blocks, static_cast<unsigned>(batch)), dim3(256), 0, stream, static_cast<const T*>(g), count, partial);
    NsStart s{};
    s.g = g; s.partial = partial; s.x = ws + l.x; s.xt = ws + l.xt; s.factors = factors;
    s.rows = static_cast<int>(rows); s.cols = static_cast<int>(cols);
    s.tall = rows > cols; s.steps = steps; s.parts = norm_blocks;
    s.x_stride = l.x_stride; s.xt_stride = l.xt_stride; s.x_matrix = l.m * l.x_stride; s.xt_matrix = l.n * l.xt_stride;
    s.eps = eps; s.k = k;
    hipLaunchKernelGGL((ns_start_kernel<T>), dim3(static_cast<unsigned>((cols + 63) / 64), static_cast<unsigned>((rows + 63) / 64), static_cast<unsigned>(batch)), dim3(256),
                       0, stream, s);
    uint8_t *x = ws + l.x, *xt = ws + l.xt, *x2 = ws + l.x2, *xt2 = ws + l.xt2;
    const int64_t sq_matrix = l.m * l.sq_stride;
    const auto product = [&](NsProduct p) {
        p.factors = factors;
        p.tiles_m = (p.a.rows + 127) / 128;
        p.tiles_n = (p.b.rows + 127) / 128;
        const int64_t tiles = p.symmetric ? static_cast<int64_t>(p.tiles_n) * (p.tiles_n + 1) / 2 : static_cast<int64_t>(p.tiles_m) * p.tiles_n;
        hipLaunchKernelGGL((ns_product_kernel<T, 2, 2, 4, 4>), dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(batch)), dim3(256), 0, stream, p);
    };
    const int m = static_cast<int>(l.m), n = static_cast<int>(l.n);
    for (int step = 0; step < steps; ++step) {
        NsProduct gram{};
        gram.a = gram.b = RowBytes{x, l.x_stride, m};
        gram.a_matrix = gram.b_matrix = l.m * l.x_stride;
        gram.out = ws + l.a; gram.out_matrix = sq_matrix; gram.out_stride = l.sq_stride;
        gram.which = 3 * step; gram.symmetric = 1; gram.stages = static_cast<int>(l.x_stride / TILE_K);
        product(gram);
        NsProduct poly{};
        poly.a = poly.b = RowBytes{ws + l.a, l.sq_stride, m};
        poly.a_matrix = poly.b_matrix = sq_matrix;
        poly.added = ws + l.a; poly.added_matrix = sq_matrix; poly.added_stride = l.sq_stride;
        poly.out = ws + l.b; poly.out_matrix = sq_matrix; poly.out_stride = l.sq_stride;
        poly.which = 3 * step + 1; poly.symmetric = 1; poly.stages = static_cast<int>(l.sq_stride / TILE_K);
        product(poly);
        NsProduct next{};
        next.a = RowBytes{ws + l.b, l.sq_stride, m};
        next.b = RowBytes{xt, l.xt_stride, n};
        next.a_matrix = sq_matrix; next.b_matrix = l.n * l.xt_stride;
        next.added = x; next.added_matrix = l.m * l.x_stride; next.added_stride = l.x_stride;
        next.which = 3 * step + 2; next.stages = static_cast<int>(l.sq_stride / TILE_K);
        if (step + 1 < steps) {
            next.out = x2; next.out_matrix = l.m * l.x_stride; next.out_stride = l.x_stride;
            next.turned = xt2; next.turned_matrix = l.n * l.xt_stride; next.turned_stride = l.xt_stride;
        } else {
            next.final = out; next.final_matrix = count; next.final_turned = rows > cols;
        }
        product(next);
        uint8_t* const keep = x; x = x2; x2 = keep;
        uint8_t* const keep_t = xt; xt = xt2; xt2 = keep_t;
    }
    return check_launch("newton_schulz_hip");
}

}  // namespace
}  // namespace ppmlhip

using namespace ppmlhip;

extern "C" size_t newton_schulz_workspace_hip(int64_t batch, int64_t rows, int64_t cols) {
    return ns_fits(batch, rows, cols) ? static_cast<size_t>(ns_layout(batch, rows, cols).total) : 0;
}

extern "C" int newton_schulz_hip(const void* g, void* out, int type, int64_t batch, int64_t rows, int64_t cols, int steps, float a, float b, float c, float eps,
                                 void* workspace, size_t workspace_bytes, ppml_hip_stream_t stream_) {
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const auto finite = [](float x) { return x - x == 0.0f; };
    if (!g || !out || !ns_fits(batch, rows, cols) || steps < 1 || steps > NS_MOST_STEPS || !finite(a) || !finite(b) || !finite(c) || !finite(eps) || eps < 0.0f) {
        set_error("newton_schulz_hip: bad arguments (batch=%lld rows=%lld cols=%lld steps=%d)", (long long)batch, (long long)rows, (long long)cols, steps);
        return RC_BAD_ARGS;
    }
    if (!workspace || workspace_bytes < newton_schulz_workspace_hip(batch, rows, cols) || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) {
        set_error("newton_schulz_hip: needs %zu bytes of workspace, 256-byte aligned (got %zu)", newton_schulz_workspace_hip(batch, rows, cols), workspace_bytes);
        return RC_BAD_ARGS;
    }
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    const NsCoefficients k{a, b, c};
    switch (type) {
        case PPML_ELEM_F32:  return run_newton_schulz<float>(g, out, batch, rows, cols, steps, k, eps, ws, stream);
        case PPML_ELEM_F16:  return run_newton_schulz<_Float16>(g, out, batch, rows, cols, steps, k, eps, ws, stream);
        case PPML_ELEM_BF16: return run_newton_schulz<__bf16>(g, out, batch, rows, cols, steps, k, eps, ws, stream);
        default: break;
    }
    set_error("newton_schulz_hip: type %d", type);
    return RC_BAD_ARGS;
}
