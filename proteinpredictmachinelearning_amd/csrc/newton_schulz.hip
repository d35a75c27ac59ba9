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

#include <algorithm>
#include <type_traits>

namespace ppmlhip {
namespace {

constexpr int NS_MOST_STEPS = 32, NS_NORM_BLOCKS = 1024;
constexpr int64_t NS_MOST_SIDE = 1 << 20;

// (per matrix) what the launches multiply by: sums of products and the matrix that is added, to the next operand's scale
struct NsFactors { float of_sum[3 * NS_MOST_STEPS], of_added[3 * NS_MOST_STEPS]; };

struct NsCoefficients { float a, b, c; };

// the largest |p(s)| for 0 <= s <= v
__host__ __device__ double next_bound(double v, const NsCoefficients& k) {
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
// Each work-group a run of the matrix, its partial sum in 64 bits: no update is so large or so small that its norm leaves the range.
// Bound by memory: 4096 x 4096 f32 14 us (4.8 TB/s).
template <class T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* g, int64_t count, double* partial, int vec) {
    __shared__ double lds[4];
    const T* const x = g + blockIdx.y * count;
    double sum = 0.0;
    const auto add = [&](float v) { sum = fma(static_cast<double>(v), static_cast<double>(v), sum); };
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256, first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (vec) {
        int64_t i = first;
        for (; i + 3 * step < count / 4; i += 4 * step) {
            float v[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_f32<T, 4>(x + 4 * (i + u * step), v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) add(v[u][e]);
        }
        for (; i < count / 4; i += step) {
            float v[4];
            load_f32<T, 4>(x + 4 * i, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) add(v[e]);
        }
    } else {
        for (int64_t i = first; i < count; i += step) add(to_f32(x[i]));
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ------------------------------------------------------------------------------------------------------------ operands
// Where a group of 32 elements lies in an operand: their upper halves, the lower ones 64 bytes behind
__device__ __forceinline__ int64_t operand_at(int64_t row, int64_t stride, int k) { return row * stride + (k >> 5) * 128 + (k & 31) * 2; }

// Sixteen consecutive elements of a group
__device__ __forceinline__ void put_operand(uint8_t* at, const float (&x)[16]) {
#pragma unroll
    for (int o = 0; o < 16; o += 8) {
        v8h h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = static_cast<_Float16>(x[o + e]);
            l[e] = static_cast<_Float16>(x[o + e] - static_cast<float>(h[e]));
        }
        *reinterpret_cast<v8h*>(at + 2 * o) = h;
        *reinterpret_cast<v8h*>(at + 64 + 2 * o) = l;
    }
}
struct Operand16 {
    v8h h[2], l[2];
    __device__ __forceinline__ void fetch(const uint8_t* at) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            h[o] = *reinterpret_cast<const v8h*>(at + 16 * o);
            l[o] = *reinterpret_cast<const v8h*>(at + 64 + 16 * o);
        }
    }
    __device__ __forceinline__ float value(int e) const { return static_cast<float>(h[e >> 3][e & 7]) + static_cast<float>(l[e >> 3][e & 7]); }
};

struct NsStart {
    const void* g;
    const double* partial;
    uint8_t *x, *xt;
    NsFactors* factors;
    int rows, cols;           // of G as it lies
    int tall, steps, parts, vec;
    int64_t x_stride, xt_stride, x_matrix, xt_matrix;      // X has min(rows, cols) rows
    float eps;
    NsCoefficients k;
};

// 64 x 64 elements of G per work-group: X_0 and its transpose, zeros behind the last column of either.  The transpose goes through LDS, so that a lane has
// sixteen elements of a group of either; every work-group adds the norm's partial sums again, in their order, instead of waiting for a launch that does.
// Bound by what it writes, four bytes an element twice: 4096 x 4096 f32 50 us (200 MB, 4.0 TB/s), 24 x 512 x 128 bf16 11.4 us (14 MB).  Elements requested
// ahead of the norm and the factors made by a work-group of their own: the same within a per cent.
template <class T>
__global__ __launch_bounds__(256) void ns_start_kernel(const NsStart p) {
    __shared__ float lds[64][65];
    const int64_t z = blockIdx.z;
    const int tid = threadIdx.x;
    __shared__ double lds_norm[4];
    double norm = 0.0;
    for (int i = tid; i < p.parts; i += 256) norm += p.partial[z * p.parts + i];
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) norm += __shfl_xor(norm, w);
    if ((tid & 63) == 0) lds_norm[tid >> 6] = norm;
    __syncthreads();
    norm = sqrt((lds_norm[0] + lds_norm[1]) + (lds_norm[2] + lds_norm[3]));
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
    {
        const int r = tid >> 2, c = (tid & 3) * 16;     // sixteen elements each
        float x[16] = {};
        if (r0 + r < p.rows) {
            const T* const from = g + static_cast<int64_t>(r0 + r) * p.cols + c0 + c;
            if (p.vec && c0 + c + 16 <= p.cols) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) load_f32<T, 4>(from + e, *reinterpret_cast<float (*)[4]>(x + e));
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = c0 + c + e < p.cols ? to_f32(from[e]) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = c0 + c + e < p.cols ? static_cast<float>(static_cast<double>(x[e]) * factor) : 0.0f;
            if (c0 + c < (p.cols + 31) / 32 * 32) put_operand(same + operand_at(r0 + r, same_stride, c0 + c), x);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) lds[r][c + e] = x[e];
    }
    __syncthreads();
    {
        const int c = tid & 63, r = (tid >> 6) * 16;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = lds[r + e][c];
        if (c0 + c < p.cols && r0 + r < (p.rows + 31) / 32 * 32) put_operand(turned + operand_at(c0 + c, turned_stride, r0 + r), x);
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
    int tiles_m, tiles_n, stages, symmetric, final_turned, final_vec;
    // the tiles of all matrices from `whole` on are cut into slices of slice_stages stages, whose sums go to `sums` (slices = 1: none)
    int tiles, whole, slices, slice_stages;
    v4f* sums;                // [tile - whole][slice][a wave's tiles of 16 x 16][thread]
};

__device__ __forceinline__ void ns_tile_of(const NsProduct& p, int t, int& tm, int& tn) {
    if (p.symmetric) {
        // the t-th tile on or above the diagonal, by rows
        tm = 0;
        while (t >= p.tiles_n - tm) { t -= p.tiles_n - tm; ++tm; }
        tn = tm + t;
    } else {
        tile_of(t, p.tiles_m, p.tiles_n, tm, tn);
    }
}

constexpr int NS_PITCH = 33;                            // floats from row to row of a block in LDS: rows and columns both meet different banks

// What a lane adds to its half row of the block of 32 x 32 from (m0, n0) on
__device__ __forceinline__ void ns_fetch_added(const NsProduct& p, Operand16& added, int64_t z, int m0, int n0) {
    const int lane = threadIdx.x & 63, m = m0 + (lane >> 1), n = n0 + (lane & 1) * 16;
    if (p.added && m < p.a.rows && n0 < p.b.rows) added.fetch(p.added + z * p.added_matrix + operand_at(m, p.added_stride, n));
}

// A block of 32 x 32 sums, in LDS, becomes what the launch writes: by rows (half a row per lane), with what is added, then by columns.
template <class T>
__device__ __forceinline__ void ns_finish_block(const NsProduct& p, float* lds, int64_t z, int m0, int n0, bool mirror, float of_sum, float of_added, const Operand16& added) {
    const int lane = threadIdx.x & 63, line = lane >> 1, part = (lane & 1) * 16;
    const int M = p.a.rows, N = p.b.rows;
    T* const final = p.final ? static_cast<T*>(p.final) + z * p.final_matrix : nullptr;
    const auto put_final = [&](T* to, const float (&x)[16], int left) {
        if (p.final_vec && left >= 16) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) store_f32<T, 4>(to + e, *reinterpret_cast<const float (*)[4]>(x + e));
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e < left) to[e] = from_f32<T>(x[e]);
        }
    };
    float x[16];
    {
        const int m = m0 + line, n = n0 + part;
        float* const row = lds + line * NS_PITCH + part;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = row[e] * of_sum;
        if (p.added && m < M && n0 < N) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = fmaf(added.value(e), of_added, x[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if (m >= M || n + e >= N) x[e] = 0.0f;
            row[e] = x[e];
        }
        if (m < M && n0 < N) {
            if (!final) put_operand(p.out + z * p.out_matrix + operand_at(m, p.out_stride, n), x);
            else if (!p.final_turned) put_final(final + static_cast<int64_t>(m) * N + n, x, N - n);
        }
    }
    uint8_t* const turned = final ? nullptr : mirror ? p.out + z * p.out_matrix : p.turned ? p.turned + z * p.turned_matrix : nullptr;
    if (!turned && !(final && p.final_turned)) return;
    wave_fence();
    {
        const int n = n0 + line, m = m0 + part;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = lds[(part + e) * NS_PITCH + line];
        if (n < N && m0 < M) {
            if (turned) put_operand(turned + operand_at(n, mirror ? p.out_stride : p.turned_stride, m), x);
            else put_final(final + static_cast<int64_t>(n) * M + m, x, M - m);
        }
    }
}

// One of a step's three products.  Large matrices are bound by the matrix pipe and its power.  Traced at 4096 x 4096: B X in tiles of 256 a side 321 us (1.29
// PFLOP/s of f16 products; the library's large f16 product 1.37), A and A A in tiles of 128 on and above the diagonal 187 us and 8 of the join (1.14 without it).  Small
// matrices are a chain of 17 launches (22 with joins) of 4 to 6 us each (768 x 256): 2.3 of a launch, a way to memory, 4 to 8 stages, and the way out.
template <class T, class Loop, bool DEEP>
__global__ __launch_bounds__(Loop::THREADS, Loop::STAGE * (DEEP ? 4 : 2) > 80 << 10 ? Loop::WAVES / 4 : 2) void ns_product_kernel(const NsProduct p) {
    constexpr int WN = Loop::WN, TM = Loop::TM, TN = Loop::TN;
    __shared__ __attribute__((aligned(128))) uint8_t even[Loop::STAGE], odd[Loop::STAGE];
    int t = xcd_contiguous_index(blockIdx.x, p.whole), slice = -1, stages = p.stages;
    if (DEEP && static_cast<int>(blockIdx.x) >= p.whole) {
        const int i = blockIdx.x - p.whole;             // (slices of the same k on one XCD: they share rows of either operand)
        slice = i % p.slices;
        t = p.whole + i / p.slices;
    }
    const int64_t z = t / p.tiles;
    int tm, tn;
    ns_tile_of(p, t % p.tiles, tm, tn);
    const int m0 = tm * Loop::BM, n0 = tn * Loop::BN;
    RowBytes A = p.a, B = p.b;
    A.base += z * p.a_matrix;
    B.base += z * p.b_matrix;
    if (DEEP && slice >= 0) {
        const int first = slice * p.slice_stages;
        A.base += first * TILE_K;
        B.base += first * TILE_K;
        stages = stages - first < p.slice_stages ? stages - first : p.slice_stages;
    }
    v4f acc[TM][TN];
    if constexpr (DEEP) {
        __shared__ __attribute__((aligned(128))) uint8_t third[Loop::STAGE], fourth[Loop::STAGE];
        Loop::run(A, B, m0, n0, stages, even, odd, third, fourth, acc);
        if (slice >= 0) {
            v4f* const to = p.sums + (static_cast<int64_t>(t - p.whole) * p.slices + slice) * (TM * TN * Loop::THREADS) + threadIdx.x;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) to[(i * TN + j) * Loop::THREADS] = acc[i][j];
            return;
        }
    } else {
        Loop::run(A, B, m0, n0, stages, even, odd, acc);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float of_sum = p.factors[z].of_sum[p.which], of_added = p.factors[z].of_added[p.which];
    static_assert(Loop::WAVES / 2 * 32 * NS_PITCH * 4 <= Loop::STAGE, "a block for half of the waves fits a stage");
    __syncthreads();                                    // every wave has read its last stage
    float* const lds = reinterpret_cast<float*>(wave & 1 ? odd : even) + (wave >> 1) * 32 * NS_PITCH;
    const bool mirror = p.symmetric && tm != tn;
#pragma unroll
    for (int i = 0; i < TM; i += 2)
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
            const int mb = m0 + (wave / WN * TM + i) * 16, nb = n0 + (wave % WN * TN + j) * 16;
            Operand16 added{};
            ns_fetch_added(p, added, z, mb, nb);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int r = 0; r < 4; ++r) lds[(16 * u + (lane >> 4) * 4 + r) * NS_PITCH + 16 * v + (lane & 15)] = acc[i + u][j + v][r];
            wave_fence();
            ns_finish_block<T>(p, lds, z, mb, nb, mirror, of_sum, of_added, added);
            wave_fence();
        }
}

// The tiles that were cut: a wave per block of 32 x 32, its slices' sums added in their order, then as above.  16 tiles of 16 slices (4096 x 4096: 17 MB, most of
// it still in the caches) 8 us traced; four waves per block 7, and slower where there are fewer slices (2944 x 2944).
template <class T, class Loop>
__global__ __launch_bounds__(64) void ns_join_kernel(const NsProduct p) {
    constexpr int WN = Loop::WN, TM = Loop::TM, TN = Loop::TN, BLOCKS = TM / 2 * (TN / 2), SUMS = TM * TN * Loop::THREADS;
    __shared__ float lds[32 * NS_PITCH];
    const int lane = threadIdx.x, wave = blockIdx.x % Loop::WAVES, block = blockIdx.x / Loop::WAVES % BLOCKS, cut = blockIdx.x / (Loop::WAVES * BLOCKS);
    const int t = p.whole + cut, i = block / (TN / 2) * 2, j = block % (TN / 2) * 2;
    const int64_t z = t / p.tiles;
    int tm, tn;
    ns_tile_of(p, t % p.tiles, tm, tn);
    const int mb = tm * Loop::BM + (wave / WN * TM + i) * 16, nb = tn * Loop::BN + (wave % WN * TN + j) * 16;
    Operand16 added{};
    ns_fetch_added(p, added, z, mb, nb);
    const v4f* const from = p.sums + static_cast<int64_t>(cut) * p.slices * SUMS + wave * 64 + lane;
    v4f sum[4] = {};
#pragma unroll 4
    for (int s = 0; s < p.slices; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += from[static_cast<int64_t>(s) * SUMS + ((i + (q >> 1)) * TN + j + (q & 1)) * Loop::THREADS];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) lds[(16 * (q >> 1) + (lane >> 4) * 4 + r) * NS_PITCH + 16 * (q & 1) + (lane & 15)] = sum[q][r];
    wave_fence();
    ns_finish_block<T>(p, lds, z, mb, nb, p.symmetric && tm != tn, p.factors[z].of_sum[p.which], p.factors[z].of_added[p.which], added);
}

// ------------------------------------------------------------------------------------------------------------ host side
typedef TilePingPong<StepF16x2> NsLarge;
typedef TileDeep<StepF16x2, 2, 4, 4, 2> NsMiddle;
typedef TileDeep<StepF16x2, 2, 2, 2, 2> NsSmall;

// How a product of every matrix of the batch is made: tiles of `side`, the middle and small ones perhaps cut
struct NsPlan { int side, tiles; CutTiles cut; };
NsPlan ns_plan(int64_t batch, int64_t rows_a, int64_t rows_b, bool symmetric, int64_t row_bytes) {
    const auto tiles = [&](int side) {
        const int64_t m = (rows_a + side - 1) / side, n = (rows_b + side - 1) / side;
        return symmetric ? n * (n + 1) / 2 : m * n;
    };
    const int stages = static_cast<int>(row_bytes / TILE_K);
    const CutTiles cut = cut_tiles(batch * tiles(128), stages), few = cut_few_tiles(batch * tiles(64), stages);
    NsPlan plan{};
    plan.side = tile_side([&](int side) { return static_cast<double>(batch * tiles(side)); }, 2.55, cut.rounds, few.rounds);
    plan.tiles = static_cast<int>(tiles(plan.side));
    plan.cut = plan.side == 128 ? cut : plan.side == 64 ? few : CutTiles{batch * plan.tiles, 0, 1, stages, 0.0};
    return plan;
}

struct NsLayout {
    int64_t m, n;             // m <= n
    int64_t x_stride, xt_stride, sq_stride;              // bytes of a row of X, of X^T and A
    int64_t x, xt, x2, xt2, a, b, partial, factors, sums, total;
    NsPlan gram, poly, next;
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
    l.gram = ns_plan(batch, l.m, l.m, true, l.x_stride);
    l.poly = ns_plan(batch, l.m, l.m, true, l.sq_stride);
    l.next = ns_plan(batch, l.m, l.n, false, l.sq_stride);
    int64_t most = 0;
    for (const NsPlan* plan : {&l.gram, &l.poly, &l.next}) most = std::max(most, plan->cut.left * plan->cut.slices * plan->side * plan->side * 4);
    l.sums = take(most);
    l.total = at;
    return l;
}

// Work-groups that add up a matrix: 4096 elements each as long as all together stay below four per CU
int ns_norm_blocks(int64_t batch, int64_t count) {
    const int64_t wanted = (count + 4095) / 4096, most = 4 * device_cu_count() / batch;
    const int64_t n = wanted < most ? wanted : most;
    return static_cast<int>(n < 1 ? 1 : (n < NS_NORM_BLOCKS ? n : NS_NORM_BLOCKS));
}

// Whether singular values of up to 1 stay below 2^20 in every step: beyond, the bounds that the operands are scaled by say too little
bool ns_stays(int steps, const NsCoefficients& k) {
    double bound = 1.0;
    for (int s = 0; s < steps; ++s) {
        bound = next_bound(bound, k);
        if (!(bound <= 1048576.0)) return false;
    }
    return true;
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
    const int norm_blocks = ns_norm_blocks(batch, count);
    const int vec = cols % 4 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0, out_vec = cols % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    hipLaunchKernelGGL((ns_norm_kernel<T>), dim3(norm_blocks, static_cast<unsigned>(batch)), dim3(256), 0, stream, static_cast<const T*>(g), count, partial, vec);
    NsStart s{};
    s.g = g; s.partial = partial; s.x = ws + l.x; s.xt = ws + l.xt; s.factors = factors;
    s.rows = static_cast<int>(rows); s.cols = static_cast<int>(cols);
    s.tall = rows > cols; s.steps = steps; s.parts = norm_blocks; s.vec = vec;
    s.x_stride = l.x_stride; s.xt_stride = l.xt_stride; s.x_matrix = l.m * l.x_stride; s.xt_matrix = l.n * l.xt_stride;
    s.eps = eps; s.k = k;
    hipLaunchKernelGGL((ns_start_kernel<T>), dim3(static_cast<unsigned>((cols + 63) / 64), static_cast<unsigned>((rows + 63) / 64), static_cast<unsigned>(batch)), dim3(256),
                       0, stream, s);
    uint8_t *x = ws + l.x, *xt = ws + l.xt, *x2 = ws + l.x2, *xt2 = ws + l.xt2;
    const int64_t sq_matrix = l.m * l.sq_stride;
    const auto product = [&](NsProduct p, const NsPlan& plan) {
        p.factors = factors;
        p.final_vec = out_vec;
        p.tiles = plan.tiles;
        p.whole = static_cast<int>(plan.cut.whole);
        p.slices = plan.cut.slices;
        p.slice_stages = plan.cut.stages;
        p.sums = reinterpret_cast<v4f*>(ws + l.sums);
        const auto launch = [&](auto loop, auto deep) {
            typedef decltype(loop) Loop;
            p.tiles_m = (p.a.rows + Loop::BM - 1) / Loop::BM;
            p.tiles_n = (p.b.rows + Loop::BN - 1) / Loop::BN;
            hipLaunchKernelGGL((ns_product_kernel<T, Loop, decltype(deep)::value>), dim3(static_cast<unsigned>(plan.cut.whole + plan.cut.left * plan.cut.slices)),
                               dim3(Loop::THREADS), 0, stream, p);
        };
        switch (plan.side) {
            case 256: launch(NsLarge{}, std::false_type{}); break;
            case 128: launch(NsMiddle{}, std::true_type{}); break;
            default:  launch(NsSmall{}, std::true_type{}); break;
        }
        const auto join = [&](auto loop) {
            typedef decltype(loop) Loop;
            hipLaunchKernelGGL((ns_join_kernel<T, Loop>), dim3(static_cast<unsigned>(plan.cut.left * Loop::WAVES * (Loop::TM / 2) * (Loop::TN / 2))), dim3(64), 0, stream, p);
        };
        if (plan.cut.left > 0) {
            if (plan.side == 128) join(NsMiddle{});
            else join(NsSmall{});
        }
    };
    const int m = static_cast<int>(l.m), n = static_cast<int>(l.n);
    for (int step = 0; step < steps; ++step) {
        NsProduct gram{};
        gram.a = gram.b = RowBytes{x, l.x_stride, m};
        gram.a_matrix = gram.b_matrix = l.m * l.x_stride;
        gram.out = ws + l.a; gram.out_matrix = sq_matrix; gram.out_stride = l.sq_stride;
        gram.which = 3 * step; gram.symmetric = 1; gram.stages = static_cast<int>(l.x_stride / TILE_K);
        product(gram, l.gram);
        NsProduct poly{};
        poly.a = poly.b = RowBytes{ws + l.a, l.sq_stride, m};
        poly.a_matrix = poly.b_matrix = sq_matrix;
        poly.added = ws + l.a; poly.added_matrix = sq_matrix; poly.added_stride = l.sq_stride;
        poly.out = ws + l.b; poly.out_matrix = sq_matrix; poly.out_stride = l.sq_stride;
        poly.which = 3 * step + 1; poly.symmetric = 1; poly.stages = static_cast<int>(l.sq_stride / TILE_K);
        product(poly, l.poly);
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
        product(next, l.next);
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
    if (!ns_stays(steps, NsCoefficients{a, b, c})) {
        set_error("newton_schulz_hip: under coefficients %g, %g, %g singular values of up to 1 grow beyond 2^20 in %d steps", a, b, c, steps);
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
