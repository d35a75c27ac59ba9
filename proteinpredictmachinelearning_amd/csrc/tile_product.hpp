// The tile loop that the products of 8-bit integers (i8_linear.hip) and of binary32 numbers as two halves
// (newton_schulz.hip) share: both multiply rows of bytes, 128 of either operand at a time.
#pragma once
#include "split.hpp"

namespace ppmlhip {

// A dense operand: rows of bytes along k, zero from the last k on to a whole number of 128.
struct RowBytes {
    const uint8_t* base;
    int64_t stride;           // bytes from row to row: a multiple of 128
    int rows;
};

constexpr int TILE_K = 128;   // bytes of a row per stage

namespace {

typedef __attribute__((address_space(3))) void* lds_void;

// Sixteen bytes per lane from `voffset + soffset` of the resource to LDS, lane after lane from `to` (the same in all lanes)
__device__ __forceinline__ void load_to_lds(const __amdgpu_buffer_rsrc_t& rsrc, uint8_t* to, uint32_t voffset, uint32_t soffset) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void)to, 16, voffset, soffset, 0, 0);
#endif
}

// What a stage of 128 bytes contributes to a tile of 16 x 16: TERMS matrix instructions on the rows' two halves of 64 bytes each.  They are
// issued term by term over all tiles of a wave, so that no two in a row add into the same accumulator.
struct StepI8 {
    typedef v4i Acc;
    static constexpr int TERMS = 2;
    template <int TERM>
    __device__ static __forceinline__ void step(const v4i (&a)[2], const v4i (&b)[2], v4i& acc) {
#if defined(__HIP_DEVICE_COMPILE__)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[TERM], b[TERM], acc, 0, 0, 0);
#endif
    }
};
// The halves are the upper and lower parts of 32 elements; the product of the two lower parts is left out
struct StepF16x2 {
    typedef v4f Acc;
    static constexpr int TERMS = 3;
    template <int TERM>
    __device__ static __forceinline__ void step(const v4i (&a)[2], const v4i (&b)[2], v4f& acc) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int OF_A = TERM == 0 ? 1 : 0, OF_B = TERM == 1 ? 1 : 0;       // smallest first
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a[OF_A]), __builtin_bit_cast(v8h, b[OF_B]), acc, 0, 0, 0);
#endif
    }
};
template <class Step, int TERM = 0, int TM, int TN>
__device__ __forceinline__ void step_tiles(const v4i (&a)[TM][2], const v4i (&b)[TN][2], typename Step::Acc (&acc)[TM][TN]) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) Step::template step<TERM>(a[i], b[j], acc[i][j]);
    if constexpr (TERM + 1 < Step::TERMS) step_tiles<Step, TERM + 1>(a, b, acc);
}

// WM x WN waves, each with TM x TN tiles of 16 x 16.  In lane l, register r of acc[i][j] holds the product of A's row
// m0 + (wave's first) + 16 i + 4 (l / 16) + r and B's row n0 + (wave's first) + 16 j + l % 16.
//
// A row's 128 bytes lie in LDS as eight pieces of sixteen, piece p of row r in place p ^ (r / 2 & 7): sixteen lanes that read the
// same piece of sixteen rows meet all 64 banks once.  The loads to LDS put lane l's piece at place l, so it is the address that a lane
// loads from which is permuted.
template <class Step, int WM_, int WN_, int TM_, int TN_>
struct TileLoop {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int STAGE = (BM + BN) * TILE_K;
    static constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES;      // a load fetches eight rows
    static_assert(WAVES % 2 == 0 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads per wave");
    typedef typename Step::Acc Acc;

    // `even` and `odd` are LDS arrays of their own, of STAGE bytes each and aligned to 128: the compiler tells loads from the one from
    // stores to the other by their names, and lets the former pass loads to LDS that are still on their way to the latter.
    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, uint8_t* even, uint8_t* odd, Acc (&acc)[TM][TN]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        // (rows behind the last one are that row again: their products are nobody's)
        const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A.base + m0 * A.stride), 0, 0x7fffffff, 0x00020000);
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B.base + n0 * B.stride), 0, 0x7fffffff, 0x00020000);
        const int row8 = lane >> 3, piece = (lane & 7) ^ (4 * (wave & 1) + (row8 >> 1));
        uint32_t from_a[LOADS_A], from_b[LOADS_B];
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i) {
            const int r = (i * WAVES + wave) * 8 + row8, last = A.rows - 1 - m0;
            from_a[i] = static_cast<uint32_t>((r < last ? r : last) * A.stride) + piece * 16u;
        }
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i) {
            const int r = (i * WAVES + wave) * 8 + row8, last = B.rows - 1 - n0;
            from_b[i] = static_cast<uint32_t>((r < last ? r : last) * B.stride) + piece * 16u;
        }
        const auto request = [&](uint8_t* to, int stage) {
#pragma unroll
            for (int i = 0; i < LOADS_A; ++i) load_to_lds(ra, to + (i * WAVES + wave) * 8 * TILE_K, from_a[i], stage * TILE_K);
#pragma unroll
            for (int i = 0; i < LOADS_B; ++i) load_to_lds(rb, to + (BM + (i * WAVES + wave) * 8) * TILE_K, from_b[i], stage * TILE_K);
        };
        const int lane_at[2] = {(lane & 15) * TILE_K + (((lane >> 4) ^ ((lane & 15) >> 1)) * 16), (lane & 15) * TILE_K + (((4 + (lane >> 4)) ^ ((lane & 15) >> 1)) * 16)};
        const auto contract = [&](const uint8_t* from) {
            const uint8_t* const a_at = from + wm * TM * 16 * TILE_K;
            const uint8_t* const b_at = from + (BM + wn * TN * 16) * TILE_K;
            v4i a[TM][2], b[TN][2];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[i][h] = *reinterpret_cast<const v4i*>(a_at + i * 16 * TILE_K + lane_at[h]);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) b[j][h] = *reinterpret_cast<const v4i*>(b_at + j * 16 * TILE_K + lane_at[h]);
            step_tiles<Step>(a, b, acc);
        };
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Acc{};
        // A barrier says both "the stage is in LDS" (it waits for the loads) and "the one before has been read".
        request(even, 0);
        int stage = 0;
        for (; stage + 2 <= stages; stage += 2) {
            __syncthreads();
            request(odd, stage + 1);
            contract(even);
            __syncthreads();
            if (stage + 2 < stages) request(even, stage + 2);
            contract(odd);
        }
        if (stage < stages) {
            __syncthreads();
            contract(even);
        }
    }
};

// Large products: 256 x 256 outputs per work-group, eight waves of 128 x 64 in two groups of four, one of each group on every SIMD.
// While one group contracts a stage out of its registers, the other fetches the next one's 24 KB per wave from LDS, then they change
// places: matrix instructions of one or the other group are issued all the time.  In phases between barriers:
//
//   phase      group 0                                   group 1
//   2 s        read stage s from LDS                     contract stage s - 1      both first request stage s + 1 from memory
//   2 s + 1    contract stage s                          read stage s from LDS     both last wait for what they requested
//
// Stage s + 1 goes where stage s - 1 was, which group 1 has read in phase 2 s - 1.
template <class Step>
struct TilePingPong {
    static constexpr int WM = 2, WN = 4, TM = 8, TN = 4;
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int STAGE = (BM + BN) * TILE_K;
    static constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES;
    typedef typename Step::Acc Acc;

    __device__ static __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const RowBytes& x, int first) {
        const int left = x.rows - first < BM ? x.rows - first : BM;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(x.base + first * x.stride), 0, static_cast<int>(left * x.stride), 0x00020000);
    }
    // (nothing moves past it; the compiler puts no wait in front of it either)
    __device__ static __forceinline__ void barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
#endif
    }

    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, uint8_t* even, uint8_t* odd, Acc (&acc)[TM][TN]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;       // wm: the group
        // (the resources end behind the last rows, and a row's place is all in the lane's offset, which is what is checked against the end:
        // rows behind the last one read as nothing, and their products are nobody's)
        const __amdgpu_buffer_rsrc_t ra = rows_from(A, m0), rb = rows_from(B, n0);
        const int row8 = wave * 8 + (lane >> 3), piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
        const uint32_t from_a = static_cast<uint32_t>(row8 * A.stride) + piece * 16u, from_b = static_cast<uint32_t>(row8 * B.stride) + piece * 16u;
        const uint32_t step_a = static_cast<uint32_t>(WAVES * 8 * A.stride), step_b = static_cast<uint32_t>(WAVES * 8 * B.stride);
        const auto request = [&](uint8_t* to, int stage) {
            // (the eight offsets are added up anew for every stage: kept, they are registers that the tiles need)
            uint32_t sa = step_a, sb = step_b;
#if defined(__HIP_DEVICE_COMPILE__)
            asm volatile("" : "+s"(sa), "+s"(sb));
#endif
#pragma unroll
            for (int i = 0; i < LOADS_A; ++i) load_to_lds(ra, to + (i * WAVES + wave) * 8 * TILE_K, from_a + i * sa, stage * TILE_K);
#pragma unroll
            for (int i = 0; i < LOADS_B; ++i) load_to_lds(rb, to + (BM + (i * WAVES + wave) * 8) * TILE_K, from_b + i * sb, stage * TILE_K);
        };
        const int lane_at[2] = {(lane & 15) * TILE_K + (((lane >> 4) ^ ((lane & 15) >> 1)) * 16), (lane & 15) * TILE_K + (((4 + (lane >> 4)) ^ ((lane & 15) >> 1)) * 16)};
        v4i a[TM][2], b[TN][2];
        const auto read = [&](const uint8_t* from) {
            const uint8_t* const a_at = from + wm * TM * 16 * TILE_K;
            const uint8_t* const b_at = from + (BM + wn * TN * 16) * TILE_K;
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) b[j][h] = *reinterpret_cast<const v4i*>(b_at + j * 16 * TILE_K + lane_at[h]);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[i][h] = *reinterpret_cast<const v4i*>(a_at + i * 16 * TILE_K + lane_at[h]);
        };
        const auto contract = [&] {
#if defined(__HIP_DEVICE_COMPILE__)
            __builtin_amdgcn_s_setprio(1);
            step_tiles<Step>(a, b, acc);
            __builtin_amdgcn_s_setprio(0);
#endif
        };
        const auto wait_lds = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
        const auto wait_loads = [] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Acc{};
        request(even, 0);
        wait_loads();
        barrier();
        if (wm == 0) {
            const auto stage = [&](uint8_t* here, uint8_t* next, int s) {
                if (s + 1 < stages) request(next, s + 1);
                read(here);
                wait_lds();
                barrier();
                contract();
                wait_loads();
                barrier();
            };
            int s = 0;
#pragma unroll 1
            for (; s + 2 <= stages; s += 2) {
                stage(even, odd, s);
                stage(odd, even, s + 1);
            }
            if (s < stages) stage(even, odd, s);
        } else {
            const auto stage = [&](uint8_t* here, uint8_t* next, int s) {
                if (s + 1 < stages) request(next, s + 1);
                if (s > 0) contract();
                barrier();
                read(here);
                wait_lds();
                wait_loads();
                barrier();
            };
            int s = 0;
#pragma unroll 1
            for (; s + 2 <= stages; s += 2) {
                stage(even, odd, s);
                stage(odd, even, s + 1);
            }
            if (s < stages) stage(even, odd, s);
            contract();
        }
    }
};

// Few tiles: one tile of 16 TM x 16 TN per work-group, its WAVES waves take every WAVES-th stage each, straight from memory to registers.
// What bounds a small product is the way to memory and back, and all of a wave's stages travel it together (DEEP at a time).
// The waves' sums are the caller's to add.
template <class Step, int WAVES, int TM, int TN, int DEEP>
struct TileSplit {
    static constexpr int BM = TM * 16, BN = TN * 16, THREADS = WAVES * 64;
    typedef typename Step::Acc Acc;

    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, Acc (&acc)[TM][TN]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A.base + m0 * A.stride), 0, 0x7fffffff, 0x00020000);
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B.base + n0 * B.stride), 0, 0x7fffffff, 0x00020000);
        uint32_t from_a[TM], from_b[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int r = 16 * i + (lane & 15), last = A.rows - 1 - m0;
            from_a[i] = static_cast<uint32_t>((r < last ? r : last) * A.stride) + (lane >> 4) * 16u;
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int r = 16 * j + (lane & 15), last = B.rows - 1 - n0;
            from_b[j] = static_cast<uint32_t>((r < last ? r : last) * B.stride) + (lane >> 4) * 16u;
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Acc{};
        const auto load = [](const __amdgpu_buffer_rsrc_t& r, uint32_t at, int stage, int h) {
            return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at, stage * TILE_K + h * 64, 0));
        };
        for (int first = wave; first < stages; first += WAVES * DEEP) {
            v4i a[DEEP][TM][2], b[DEEP][TN][2];
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                // (a stage behind the last one is loaded again and not used)
                const int stage = first + d * WAVES < stages ? first + d * WAVES : first;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < TM; ++i) a[d][i][h] = load(ra, from_a[i], stage, h);
#pragma unroll
                    for (int j = 0; j < TN; ++j) b[d][j][h] = load(rb, from_b[j], stage, h);
                }
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
                if (first + d * WAVES < stages) step_tiles<Step>(a[d], b[d], acc);
        }
    }
};

}  // namespace
}  // namespace ppmlhip
