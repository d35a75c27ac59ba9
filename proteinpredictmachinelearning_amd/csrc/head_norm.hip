// Norms of queries and keys for each head with the position rotation (qk_norm_rope_hip, qk_norm_rope_back_hip): from the
// projection's layout, a token's heads side by side, into attention's [B][h][L][d], and the gradients back.
//
// One head x of one token at position p, weights w, frequencies f (radians a position):
//   s = 1 / sqrt(mean(x^2) + eps)    n = x s    u = n w    y = R(p) u
// R turns the pairs (i, i + rot/2), or (2i, 2i+1) where they are interleaved, by p f_i; elements from rot on stay.
//   backward: v = R^T dy    dw = sum of v n    g = v w    dx = s (g - n mean(g n))
//
// Angles: p f_i may be millions of radians, of which binary32 would keep none of the fraction.  In units of a quarter turn,
// in 64 bits, the whole number (modulo 4) picks the quadrant and the rest, at most 1/2, becomes an angle of at most pi / 4 in binary32;
// sine and cosine there are their series up to the 11th and 10th power (next term below 2^-27 of the result).
//
// A group of G lanes takes a token and walks over its heads; each lane keeps its pairs' sines, cosines and weights.
#include "elements.hpp"

namespace ppmlhip {
namespace {

struct HeadSide {             // queries or keys
    const void* x;
    const void* dy;           // backward
    void* out;                // y, or dx
    const float* w;           // or null: ones
    int64_t x_b, x_l, x_h, dy_b, dy_l, dy_h, out_b, out_l, out_h;      // elements from batch to batch, token to token, head to head
    int heads;
};
struct HeadNorm {
    HeadSide side[2];
    const double* freqs;
    const void* positions;    // null: a token's place in its sequence
    int64_t pos_b;
    int pos_type;
    int64_t tokens;           // B L
    int L, d, rot, interleaved;
    float eps;
    int group;                // lanes per token: a power of two
    int heads_per_part;       // heads of queries and keys in one list, cut into gridDim.y parts
    float* partial;           // backward: [work-group][2][d]
};

// sine and cosine of p f, f in quarter turns a position
__device__ __forceinline__ void turn_of(double p, double f, float& sine, float& cosine) {
    const double t = p * f, whole = __builtin_rint(t);
    const float a = static_cast<float>((t - whole) * 1.5707963267948966), z = a * a;
    float s = -2.50521083854417188e-8f;
    s = fmaf(s, z, 2.75573192239858907e-6f);
    s = fmaf(s, z, -1.98412698412698413e-4f);
    s = fmaf(s, z, 8.33333333333333333e-3f);
    s = fmaf(s, z, -1.66666666666666667e-1f);
    s = fmaf(s * z, a, a);
    float c = -2.75573192239858907e-7f;
    c = fmaf(c, z, 2.48015873015873016e-5f);
    c = fmaf(c, z, -1.38888888888888889e-3f);
    c = fmaf(c, z, 4.16666666666666667e-2f);
    c = fmaf(c, z, -0.5f);
    c = fmaf(c, z, 1.0f);
    // (of a whole number of quarter turns the remainder modulo 4; beyond 2^53 it is a multiple of two)
    const int quarter = static_cast<int>(whole - 4.0 * __builtin_floor(whole * 0.25));
    const float x = quarter & 1 ? c : s, y = quarter & 1 ? s : c;
    sine = quarter & 2 ? -x : x;
    cosine = ((quarter + 1) & 2) ? -y : y;
}

// the sum over a group of lanes, in all of them
__device__ __forceinline__ float group_sum(float v, int group) {
#if defined(__HIP_DEVICE_COMPILE__)
#define PPML_DPP(CTRL) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true))
    if (group > 1) PPML_DPP(0xb1);                      // quad_perm [1, 0, 3, 2]
    if (group > 2) PPML_DPP(0x4e);                      // quad_perm [2, 3, 0, 1]
    if (group > 4) PPML_DPP(0x141);                     // row_half_mirror
    if (group > 8) PPML_DPP(0x140);                     // row_mirror
#undef PPML_DPP
    if (group > 16) v = fold16(v, v, [](float a, float b) { return a + b; });
    if (group > 32) v = fold32(v, v, [](float a, float b) { return a + b; });
#endif
    return v;
}

// What a lane holds of a head: R chunks of two times V elements.  A chunk's halves `a`, `b` are V pairs' first and second
// elements (half-split) or 2 V consecutive elements (interleaved, and behind the rotated ones).  FULL: a head is as many chunks as the group
// has lanes, so that none is outside, and no load or store stands under a condition (the compiler then waits for a head's loads alone, not
// for the stores behind them).
template <class T, int V, int R, bool FULL>
struct Chunks {
    typedef typename Elements<T, V>::Raw Raw;
    struct Head { Raw a[R], b[R]; };
    int at_a[R], at_b[R];     // -1: outside the head
    float sine[R][V], cosine[R][V];

    __device__ __forceinline__ void place(int lane, int group, int d, int rot, bool interleaved) {
        const int half = rot / 2, turning = interleaved ? 0 : half / V;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = lane + r * group;
            if (c < turning) {
                at_a[r] = c * V;
                at_b[r] = half + c * V;
            } else {
                at_a[r] = 2 * V * c;                    // (half-split: 2 V turning = rot)
                at_b[r] = at_a[r] + V;
            }
            if (at_a[r] >= d) at_a[r] = -1;
            if (at_b[r] >= d) at_b[r] = -1;
        }
    }
    __device__ __forceinline__ void angles(int lane, int group, const HeadNorm& p, double position) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int pair = (lane + r * group) * V + v;
                sine[r][v] = 0.0f;
                cosine[r][v] = 1.0f;
                if (pair < p.rot / 2) turn_of(position, p.freqs[pair] * 0.63661977236758134308, sine[r][v], cosine[r][v]);
            }
    }
    template <bool INTER, bool BACK>
    __device__ __forceinline__ void rotate(float (&a)[R][V], float (&b)[R][V]) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float sn = BACK ? -sine[r][v] : sine[r][v], cs = cosine[r][v];
                float& x = INTER && V > 1 ? (2 * v < V ? a[r][(2 * v) % V] : b[r][(2 * v) % V]) : a[r][v];
                float& y = INTER && V > 1 ? (2 * v + 1 < V ? a[r][(2 * v + 1) % V] : b[r][(2 * v + 1) % V]) : b[r][v];
                const float t = x * cs - y * sn;
                y = fmaf(y, cs, x * sn);
                x = t;
            }
    }
    __device__ __forceinline__ Head fetch(const T* head) const {
        Head x;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            x.a[r] = *reinterpret_cast<const Raw*>(head + (FULL || at_a[r] >= 0 ? at_a[r] : 0));
            x.b[r] = *reinterpret_cast<const Raw*>(head + (FULL || at_b[r] >= 0 ? at_b[r] : 0));
        }
        return x;
    }
    __device__ __forceinline__ void finish(const Head& x, float (&a)[R][V], float (&b)[R][V]) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (V == 1) { a[r][v] = to_f32(static_cast<T>(x.a[r])); b[r][v] = to_f32(static_cast<T>(x.b[r])); }
                else                  { a[r][v] = to_f32(static_cast<T>(x.a[r][v])); b[r][v] = to_f32(static_cast<T>(x.b[r][v])); }
                if (!FULL && at_a[r] < 0) a[r][v] = 0.0f;
                if (!FULL && at_b[r] < 0) b[r][v] = 0.0f;
            }
    }
    // of the norms' weights (a lane's own few, once)
    __device__ __forceinline__ void load_weights(const float* w, float (&a)[R][V], float (&b)[R][V]) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                a[r][v] = at_a[r] >= 0 ? w[at_a[r] + v] : 0.0f;
                b[r][v] = at_b[r] >= 0 ? w[at_b[r] + v] : 0.0f;
            }
    }
    template <class U>
    __device__ __forceinline__ void store(U* head, const float (&a)[R][V], const float (&b)[R][V]) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (FULL || at_a[r] >= 0) store_f32<U, V>(head + at_a[r], a[r]);
            if (FULL || at_b[r] >= 0) store_f32<U, V>(head + at_b[r], b[r]);
        }
    }
};

__device__ __forceinline__ double position_of(const HeadNorm& p, int64_t b, int64_t l) {
    if (!p.positions) return static_cast<double>(l);
    const int64_t at = b * p.pos_b + l;
    return p.pos_type == 4 ? static_cast<double>(static_cast<const int32_t*>(p.positions)[at])
                           : static_cast<double>(static_cast<const int64_t*>(p.positions)[at]);
}

// What both passes have of a head's elements
template <int R, int V>
__device__ __forceinline__ float squares_of(const float (&a)[R][V], const float (&b)[R][V]) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) sum = fmaf(a[r][v], a[r][v], fmaf(b[r][v], b[r][v], sum));
    return sum;
}

// Forward.  Bound by memory, a head read and written once: all of a token's heads pass through one group of lanes, so that the angles (64-bit work, as much as
// several heads') are made once, and the next head is on its way while one is normed.  Few tokens: the heads are cut into parts too (plan_heads),
// which make their angles again.  Measured: 26368 tokens of 16 heads of 32, f32 26.6 us (4.1 TB/s, where a large copy reaches 5.2; 19.0 where the last-level
// cache holds the tensors); 32768 of 40 heads of 128, bf16 155 us (4.3 TB/s); 103 tokens of 16 heads 4.2 us, an empty launch and one way to memory.
// Non-temporal loads and stores: the same or slower.
template <class T, int V, int R, bool INTER, bool FULL>
__global__ __launch_bounds__(256) void head_norm_kernel(const HeadNorm p) {
    const int lane = threadIdx.x & (p.group - 1);
    const int64_t token = static_cast<int64_t>(blockIdx.x) * (256 / p.group) + threadIdx.x / p.group;
    if (token >= p.tokens) return;                      // (whole groups)
    const int64_t b = token / p.L, l = token % p.L;
    Chunks<T, V, R, FULL> ch;
    ch.place(lane, p.group, p.d, p.rot, INTER);
    const int all = p.side[0].heads + p.side[1].heads;
    const int first = blockIdx.y * p.heads_per_part, end = first + p.heads_per_part < all ? first + p.heads_per_part : all;
    const float mean = 1.0f / static_cast<float>(p.d);
    bool turned = false;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const HeadSide& side = p.side[s];
        const int before = s == 0 ? 0 : p.side[0].heads;
        const int begin = first - before > 0 ? first - before : 0, stop = end - before < side.heads ? end - before : side.heads;
        if (begin >= stop) continue;
        const T* const x = static_cast<const T*>(side.x) + b * side.x_b + l * side.x_l;
        T* const y = static_cast<T*>(side.out) + b * side.out_b + l * side.out_l;
        typename Chunks<T, V, R, FULL>::Head next = ch.fetch(x + begin * side.x_h);
        if (!turned) ch.angles(lane, p.group, p, position_of(p, b, l));
        turned = true;
        float wa[R][V], wb[R][V];
        if (side.w) ch.load_weights(side.w, wa, wb);
        else
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) wa[r][v] = wb[r][v] = 1.0f;
        for (int h = begin; h < stop; ++h) {
            float xa[R][V], xb[R][V];
            ch.finish(next, xa, xb);
            next = ch.fetch(x + (h + 1 < stop ? h + 1 : h) * side.x_h);      // (past the last head, that one again)
            const float scale = rsqrtf(fmaf(group_sum(squares_of(xa, xb), p.group), mean, p.eps));
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    xa[r][v] *= scale * wa[r][v];
                    xb[r][v] *= scale * wb[r][v];
                }
            ch.template rotate<INTER, false>(xa, xb);
            ch.store(y + h * side.out_h, xa, xb);
        }
    }
}

// Backward, the norm's statistics made again (reading them back would cost as much as the rows they are of): x and dy in, dx out, one pass, bound by
// memory.  The weights' gradients stay in the lanes over all of a work-group's tokens and leave as one partial sum per work-group, in a fixed order: no
// atomics, the same bits every time.  Measured: 26368 tokens of 16 heads of 32, f32 42.8 us (3.8 TB/s; 34 where the last-level cache holds the tensors), of which
// 4.7 are the launch that adds the partial sums.
template <class T, int V, int R, bool INTER, bool FULL>
__global__ __launch_bounds__(256) void head_norm_back_kernel(const HeadNorm p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];      // [tokens of the work-group][d]
    const int lane = threadIdx.x & (p.group - 1), groups = 256 / p.group, mine = threadIdx.x / p.group;
    Chunks<T, V, R, FULL> ch;
    typedef typename Chunks<T, V, R, FULL>::Head Head;
    ch.place(lane, p.group, p.d, p.rot, INTER);
    const int all = p.side[0].heads + p.side[1].heads;
    const int first = blockIdx.y * p.heads_per_part, end = first + p.heads_per_part < all ? first + p.heads_per_part : all;
    const float mean = 1.0f / static_cast<float>(p.d);
    float wa[2][R][V], wb[2][R][V], dwa[2][R][V] = {}, dwb[2][R][V] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (p.side[s].w) ch.load_weights(p.side[s].w, wa[s], wb[s]);
        else
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) wa[s][r][v] = wb[s][r][v] = 1.0f;
    }
    for (int64_t token = static_cast<int64_t>(blockIdx.x) * groups + mine; token < p.tokens; token += static_cast<int64_t>(gridDim.x) * groups) {
        const int64_t b = token / p.L, l = token % p.L;
        bool turned = false;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const HeadSide& side = p.side[s];
            const int before = s == 0 ? 0 : p.side[0].heads;
            const int begin = first - before > 0 ? first - before : 0, stop = end - before < side.heads ? end - before : side.heads;
            if (begin >= stop) continue;
            const T* const x = static_cast<const T*>(side.x) + b * side.x_b + l * side.x_l;
            const T* const dy = static_cast<const T*>(side.dy) + b * side.dy_b + l * side.dy_l;
            T* const dx = static_cast<T*>(side.out) + b * side.out_b + l * side.out_l;
            Head next_x = ch.fetch(x + begin * side.x_h), next_g = ch.fetch(dy + begin * side.dy_h);
            if (!turned) ch.angles(lane, p.group, p, position_of(p, b, l));
            turned = true;
            for (int h = begin; h < stop; ++h) {
                float xa[R][V], xb[R][V], ga[R][V], gb[R][V];
                ch.finish(next_x, xa, xb);
                ch.finish(next_g, ga, gb);
                const int after = h + 1 < stop ? h + 1 : h;
                next_x = ch.fetch(x + after * side.x_h);
                next_g = ch.fetch(dy + after * side.dy_h);
                const float scale = rsqrtf(fmaf(group_sum(squares_of(xa, xb), p.group), mean, p.eps));
                ch.template rotate<INTER, true>(ga, gb);
                float along = 0.0f;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        xa[r][v] *= scale;
                        xb[r][v] *= scale;
                        dwa[s][r][v] = fmaf(ga[r][v], xa[r][v], dwa[s][r][v]);
                        dwb[s][r][v] = fmaf(gb[r][v], xb[r][v], dwb[s][r][v]);
                        ga[r][v] *= wa[s][r][v];
                        gb[r][v] *= wb[s][r][v];
                        along = fmaf(ga[r][v], xa[r][v], fmaf(gb[r][v], xb[r][v], along));
                    }
                along = group_sum(along, p.group) * mean;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        ga[r][v] = scale * fmaf(-xa[r][v], along, ga[r][v]);
                        gb[r][v] = scale * fmaf(-xb[r][v], along, gb[r][v]);
                    }
                ch.store(dx + h * side.out_h, ga, gb);
            }
        }
    }
    // the work-group's sums of dw, tokens in their order, in 64 bits: a few numbers per work-group, and sums of hundreds of thousands of terms
    if (!p.partial) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (!p.side[s].w) continue;
        __syncthreads();
        ch.template store<float>(lds + mine * p.d, dwa[s], dwb[s]);
        __syncthreads();
        for (int e = threadIdx.x; e < p.d; e += 256) {
            double sum = 0.0;
            for (int g = 0; g < groups; ++g) sum += static_cast<double>(lds[g * p.d + e]);
            p.partial[(static_cast<int64_t>(blockIdx.y * gridDim.x + blockIdx.x) * 2 + s) * p.d + e] = static_cast<float>(sum);
        }
    }
}

// dw[e] = the sum over `parts` work-groups of partial[part][side][e].  A work-group takes eight elements, 32 threads each: a thread every 32nd part,
// eight of them on their way at once (a chain of loads 21 us for 1024 parts of 32 elements).
__global__ __launch_bounds__(256) void head_norm_weights_kernel(const float* partial, int parts, int d, float* dwq, float* dwk) {
    __shared__ double lds[32][9];
    const int col = threadIdx.x & 7, run = threadIdx.x >> 3;
    const int e = blockIdx.x * 8 + col, s = blockIdx.y;
    float* const dw = s == 0 ? dwq : dwk;
    if (!dw) return;
    const float* const from = partial + s * d + (e < d ? e : d - 1);
    const int64_t step = 2 * static_cast<int64_t>(d);
    double sum = 0.0;
    for (int i = run; i < parts; i += 32 * 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = from[(i + 32 * u < parts ? i + 32 * u : run) * step];
#pragma unroll
        for (int u = 0; u < 8; ++u) sum += i + 32 * u < parts ? static_cast<double>(x[u]) : 0.0;
    }
    lds[run][col] = sum;
    __syncthreads();
    if (run == 0 && e < d) {
        for (int i = 1; i < 32; ++i) sum += lds[i][col];
        dw[e] = static_cast<float>(sum);
    }
}

constexpr int HEAD_MAX_D = 512;
constexpr int BACK_MOST_BLOCKS = 1024;

struct HeadPlan { int v, chunks_per_lane, group; bool full; unsigned blocks, parts; };

int elem_bytes(int type) { return type == PPML_ELEM_F32 ? 4 : 2; }

// How a head is dealt to lanes.  `aligned`: to how many elements at a time (1, 4, 8) addresses and strides are multiples of; sixteen bytes are
// taken where the head's parts are whole pieces of as many.
HeadPlan plan_heads(const ppml_qk_norm_desc& a, int aligned, bool back) {
    HeadPlan pl{};
    const auto whole = [&](int v) { return aligned % v == 0 && (a.interleaved ? a.d % (2 * v) == 0 && a.rot % (2 * v) == 0 : a.rot % (2 * v) == 0 && (a.d - a.rot) % (2 * v) == 0); };
    // Eight elements at a time halve the instructions per head and double the angles per lane: for tokens enough to fill the chip with half of the
    // lanes (bf16, 32768 tokens of 40 heads of 128 141 us, 182 with four; 16384 of 32 heads of 64 25.4 / 27.0; 26368 of 16 heads of 32 15.2 / 13.6; one token
    // 4.2 / 3.5)
    const int64_t tokens = a.B * a.L;
    pl.v = a.type != PPML_ELEM_F32 && whole(8) && tokens * (a.d / 16) >= 65536 ? 8 : whole(4) ? 4 : 1;
    const int chunks = (a.d + 2 * pl.v - 1) / (2 * pl.v);
    pl.group = 1;
    while (pl.group < 64 && pl.group < chunks) pl.group *= 2;
    pl.full = chunks == pl.group && a.d % (2 * pl.v) == 0;
    pl.chunks_per_lane = (chunks + pl.group - 1) / pl.group;
    const int64_t per_block = 256 / pl.group;
    int64_t blocks = (tokens + per_block - 1) / per_block;
    const int heads = a.hq + a.hk;
    if (back && blocks > BACK_MOST_BLOCKS) blocks = BACK_MOST_BLOCKS;
    int64_t parts = 1;
    while (parts < heads && blocks * parts < 1024) ++parts;
    pl.blocks = static_cast<unsigned>(blocks);
    pl.parts = static_cast<unsigned>(parts);
    return pl;
}

bool desc_ok(const ppml_qk_norm_desc* a) {
    return a && a->B > 0 && a->L > 0 && a->B <= INT64_MAX / a->L && a->L <= 0x7fffffff && a->hq >= 0 && a->hk >= 0 && a->hq + static_cast<int64_t>(a->hk) > 0 && a->hq <= 65535 && a->hk <= 65535 &&
           a->d > 0 && a->d <= HEAD_MAX_D && a->rot >= 0 && a->rot <= a->d && a->rot % 2 == 0 &&
           (a->type == PPML_ELEM_F32 || a->type == PPML_ELEM_F16 || a->type == PPML_ELEM_BF16) && a->eps >= 0.0f &&
           (a->position_bytes == 0 || a->position_bytes == 4 || a->position_bytes == 8) && a->B * a->L <= (int64_t{1} << 32);
}

// elements that all of a side's addresses and steps are multiples of: 8, 4 or 1
int side_aligned(const HeadSide& s, int elem, bool back) {
    if (s.heads == 0) return 8;
    for (const int v : {8, 4}) {
        const auto ok = [&](const void* ptr, int64_t b, int64_t l, int64_t h) {
            return reinterpret_cast<uintptr_t>(ptr) % static_cast<uintptr_t>(v * elem) == 0 && b % v == 0 && l % v == 0 && h % v == 0;
        };
        if (ok(s.x, s.x_b, s.x_l, s.x_h) && ok(s.out, s.out_b, s.out_l, s.out_h) && (!back || ok(s.dy, s.dy_b, s.dy_l, s.dy_h))) return v;
    }
    return 1;
}
int both_aligned(const HeadNorm& p, int elem, bool back) {
    const int q = side_aligned(p.side[0], elem, back), k = side_aligned(p.side[1], elem, back);
    return q < k ? q : k;
}

template <class T, int V, int R, bool FULL>
void launch_heads(const HeadNorm& p, const HeadPlan& pl, bool back, hipStream_t stream) {
    const dim3 grid(pl.blocks, pl.parts), block(256);
    const size_t lds = back ? static_cast<size_t>(256 / p.group) * p.d * 4 : 0;
    if (back) {
        if (p.interleaved) hipLaunchKernelGGL((head_norm_back_kernel<T, V, R, true, FULL>), grid, block, lds, stream, p);
        else               hipLaunchKernelGGL((head_norm_back_kernel<T, V, R, false, FULL>), grid, block, lds, stream, p);
    } else {
        if (p.interleaved) hipLaunchKernelGGL((head_norm_kernel<T, V, R, true, FULL>), grid, block, 0, stream, p);
        else               hipLaunchKernelGGL((head_norm_kernel<T, V, R, false, FULL>), grid, block, 0, stream, p);
    }
}

template <class T>
void launch_heads(const HeadNorm& p, const HeadPlan& pl, bool back, hipStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (pl.v == 8) return pl.full ? launch_heads<T, 8, 1, true>(p, pl, back, stream) : launch_heads<T, 8, 1, false>(p, pl, back, stream);
    if (pl.v == 4) return pl.full ? launch_heads<T, 4, 1, true>(p, pl, back, stream) : launch_heads<T, 4, 1, false>(p, pl, back, stream);
    if (pl.chunks_per_lane == 1) return launch_heads<T, 1, 1, false>(p, pl, back, stream);
    launch_heads<T, 1, 4, false>(p, pl, back, stream);
}

int run_heads(const ppml_qk_norm_desc& a, HeadNorm p, const HeadPlan& pl, bool back, hipStream_t stream, const char* what) {
    if (pl.blocks > 0xffffffffu / 256) {                // a launch's threads along x are counted in 32 bits
        set_error("%s: too many tokens (%lld)", what, (long long)p.tokens);
        return RC_BAD_ARGS;
    }
    p.group = pl.group;
    p.heads_per_part = (a.hq + a.hk + static_cast<int>(pl.parts) - 1) / static_cast<int>(pl.parts);
    switch (a.type) {
        case PPML_ELEM_F32: launch_heads<float>(p, pl, back, stream); break;
        case PPML_ELEM_F16: launch_heads<_Float16>(p, pl, back, stream); break;
        default:            launch_heads<__bf16>(p, pl, back, stream); break;
    }
    return check_launch(what);
}

HeadNorm describe(const ppml_qk_norm_desc& a, const double* freqs, const void* positions) {
    HeadNorm p{};
    p.freqs = freqs;
    p.positions = a.position_bytes ? positions : nullptr;
    p.pos_b = a.position_stride;
    p.pos_type = a.position_bytes;
    p.tokens = a.B * a.L;
    p.L = static_cast<int>(a.L);
    p.d = a.d;
    p.rot = a.rot;
    p.interleaved = a.interleaved;
    p.eps = a.eps;
    return p;
}

HeadSide side_of(const void* x, const int64_t* xs, const void* dy, const int64_t* dys, void* out, const int64_t* outs, const float* w, int heads) {
    HeadSide s{};
    s.x = x; s.dy = dy; s.out = out; s.w = w; s.heads = heads;
    s.x_b = xs[0]; s.x_l = xs[1]; s.x_h = xs[2];
    if (dys) { s.dy_b = dys[0]; s.dy_l = dys[1]; s.dy_h = dys[2]; }
    s.out_b = outs[0]; s.out_l = outs[1]; s.out_h = outs[2];
    return s;
}

}  // namespace
}  // namespace ppmlhip

using namespace ppmlhip;

extern "C" int qk_norm_rope_hip(const ppml_qk_norm_desc* a, const void* q, const void* k, const float* wq, const float* wk, const double* freqs,
                                const void* positions, void* q_out, void* k_out, ppml_hip_stream_t stream) {
    if (!desc_ok(a) || (a->hq > 0 && (!q || !q_out)) || (a->hk > 0 && (!k || !k_out)) || (a->rot > 0 && !freqs) || (a->position_bytes > 0 && !positions)) {
        set_error("qk_norm_rope_hip: bad arguments");
        return RC_BAD_ARGS;
    }
    HeadNorm p = describe(*a, freqs, positions);
    p.side[0] = side_of(q, a->q_strides, nullptr, nullptr, q_out, a->q_out_strides, wq, a->hq);
    p.side[1] = side_of(k, a->k_strides, nullptr, nullptr, k_out, a->k_out_strides, wk, a->hk);
    const HeadPlan pl = plan_heads(*a, both_aligned(p, elem_bytes(a->type), false), false);
    return run_heads(*a, p, pl, false, static_cast<hipStream_t>(stream), "qk_norm_rope_hip");
}

extern "C" size_t qk_norm_rope_back_workspace_hip(const ppml_qk_norm_desc* a) {
    if (!desc_ok(a)) return 0;
    size_t most = 0;
    for (const int aligned : {1, 4, 8}) {
        const HeadPlan pl = plan_heads(*a, aligned, true);
        const size_t bytes = static_cast<size_t>(pl.blocks) * pl.parts * 2 * static_cast<size_t>(a->d) * 4;
        if (bytes > most) most = bytes;
    }
    return most;
}

extern "C" int qk_norm_rope_back_hip(const ppml_qk_norm_desc* a, const void* dq, const void* dk, const void* q, const void* k, const float* wq, const float* wk,
                                     const double* freqs, const void* positions, void* q_grad, void* k_grad, float* wq_grad, float* wk_grad,
                                     void* workspace, size_t workspace_bytes, ppml_hip_stream_t stream_) {
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (!desc_ok(a) || (a->hq > 0 && (!q || !dq || !q_grad)) || (a->hk > 0 && (!k || !dk || !k_grad)) || (a->rot > 0 && !freqs) || (a->position_bytes > 0 && !positions) ||
        (wq_grad && !wq) || (wk_grad && !wk)) {
        set_error("qk_norm_rope_back_hip: bad arguments");
        return RC_BAD_ARGS;
    }
    const bool weights = wq_grad || wk_grad;
    if (weights && (!workspace || workspace_bytes < qk_norm_rope_back_workspace_hip(a) || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)) {
        set_error("qk_norm_rope_back_hip: needs %zu bytes of workspace (got %zu)", qk_norm_rope_back_workspace_hip(a), workspace_bytes);
        return RC_BAD_ARGS;
    }
    HeadNorm p = describe(*a, freqs, positions);
    p.side[0] = side_of(q, a->q_strides, dq, a->dq_strides, q_grad, a->q_out_strides, wq, a->hq);
    p.side[1] = side_of(k, a->k_strides, dk, a->dk_strides, k_grad, a->k_out_strides, wk, a->hk);
    p.partial = weights ? static_cast<float*>(workspace) : nullptr;
    const HeadPlan pl = plan_heads(*a, both_aligned(p, elem_bytes(a->type), true), true);
    const int rc = run_heads(*a, p, pl, true, stream, "qk_norm_rope_back_hip");
    if (rc != RC_OK || !weights) return rc;
    hipLaunchKernelGGL(head_norm_weights_kernel, dim3((a->d + 7) / 8, 2), dim3(256), 0, stream, static_cast<const float*>(workspace),
                       static_cast<int>(pl.blocks * pl.parts), a->d, wq_grad, wk_grad);
    return check_launch("qk_norm_rope_back_hip");
}
