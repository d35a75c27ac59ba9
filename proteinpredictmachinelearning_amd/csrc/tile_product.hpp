// The tile loop that the products of 8-bit integers (i8_linear.hip) and of binary32 numbers as two halves
// (newton_schulz.hip) share: both multiply rows of bytes, 128 of either operand at a time.
#pragma once
#include "split.hpp"

#include <cmath>

namespace ppmlhip {

// An operand: rows of a whole number of 128 bytes along k, zero from the last k on.
struct RowBytes {
    const uint8_t* base;
    int64_t stride;           // bytes from row to row: a multiple of 16
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

// A barrier that nothing moves past and that waits for nothing by itself
__device__ __forceinline__ void bare_barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
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
// ... with between(n) after every TM of them, n = 0, 1, ...
template <class Step, int TERM = 0, int TM, int TN, class Between>
__device__ __forceinline__ void step_tiles_between(const v4i (&a)[TM][2], const v4i (&b)[TN][2], typename Step::Acc (&acc)[TM][TN], const Between& between) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int i = 0; i < TM; ++i) Step::template step<TERM>(a[i], b[j], acc[i][j]);
        between(TERM * TN + j);
    }
    if constexpr (TERM + 1 < Step::TERMS) step_tiles_between<Step, TERM + 1>(a, b, acc, between);
}

// A tile of the product: WM x WN waves, each with TM x TN tiles of 16 x 16.  In lane l, register r of acc[i][j] holds the product of A's row
// m0 + (wave's first) + 16 i + 4 (l / 16) + r and B's row n0 + (wave's first) + 16 j + l % 16.
//
// A row's 128 bytes lie in LDS as eight pieces of sixteen, piece p of row r in place p ^ (r / 2 & 7): sixteen lanes that read the
// same piece of sixteen rows meet all 64 banks once.  The loads to LDS put lane l's piece at place l, so it is the address that a
// lane loads from which is permuted.
//
// The stages' LDS arrays are the kernel's, each of STAGE bytes, aligned to 128 and declared by itself: the compiler tells loads from one from
// stores to another by their names, and lets the former pass loads to LDS that are still on their way to the latter.
//
// TileDeep: three stages are on their way while one is contracted (four arrays).  A work-group of a product of few tiles has a CU to itself and
// nothing else to do while a stage travels: with one on its way (two arrays) 1024 x 1024 x 1024 in two halves took 24 us instead of 12 in tiles of 64 x 64.
template <class Step, int WM_, int WN_, int TM_, int TN_>
struct TileDeep {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int STAGE = (BM + BN) * TILE_K;
    static constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES, LOADS = LOADS_A + LOADS_B;      // a load fetches eight rows
    static_assert(WAVES % 2 == 0 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads per wave");
    typedef typename Step::Acc Acc;

    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, uint8_t* s0, uint8_t* s1, uint8_t* s2, uint8_t* s3,
                                               Acc (&acc)[TM][TN]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
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
        // (past the last stage that one again, into an array nobody reads: as many loads are on their way in every iteration)
        const auto request = [&](uint8_t* to, int stage) {
            const int at = (stage < stages ? stage : stages - 1) * TILE_K;
#pragma unroll
            for (int i = 0; i < LOADS_A; ++i) load_to_lds(ra, to + (i * WAVES + wave) * 8 * TILE_K, from_a[i], at);
#pragma unroll
            for (int i = 0; i < LOADS_B; ++i) load_to_lds(rb, to + (BM + (i * WAVES + wave) * 8) * TILE_K, from_b[i], at);
        };
        const int lane_at[2] = {(lane & 15) * TILE_K + (((lane >> 4) ^ ((lane & 15) >> 1)) * 16), (lane & 15) * TILE_K + (((4 + (lane >> 4)) ^ ((lane & 15) >> 1)) * 16)};
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Acc{};
        // One barrier per stage: behind it the stage is in LDS (every wave has waited for its own part), and the one before has been read.
        const auto stage = [&](const uint8_t* here, uint8_t* free, int s) {
            static_assert(LOADS == 4 || LOADS == 8, "the wait below names 2 LOADS");
#if defined(__HIP_DEVICE_COMPILE__)
            if constexpr (LOADS == 4) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
            else                      asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)" ::: "memory");
#endif
            bare_barrier();
            request(free, s + 3);
            const uint8_t* const a_at = here + wm * TM * 16 * TILE_K;
            const uint8_t* const b_at = here + (BM + wn * TN * 16) * TILE_K;
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
        request(s0, 0);
        request(s1, 1);
        request(s2, 2);
        int s = 0;
#pragma unroll 1
        for (; s + 4 <= stages; s += 4) {
            stage(s0, s3, s);
            stage(s1, s0, s + 1);
            stage(s2, s1, s + 2);
            stage(s3, s2, s + 3);
        }
        if (s < stages) stage(s0, s3, s);
        if (s + 1 < stages) stage(s1, s0, s + 1);
        if (s + 2 < stages) stage(s2, s1, s + 2);
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (nothing is on its way to LDS when the caller uses it)
#endif
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
    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, uint8_t* even, uint8_t* odd, Acc (&acc)[TM][TN]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;       // wm: the group
        // (the resources end behind the last rows, and a row's place is all in the lane's offset, which is what is checked against the end:
        // rows behind the last one read as nothing, and their products are nobody's)
        const __amdgpu_buffer_rsrc_t ra = rows_from(A, m0), rb = rows_from(B, n0);
        const int row8 = wave * 8 + (lane >> 3), piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
        const uint32_t from_a = static_cast<uint32_t>(row8 * A.stride) + piece * 16u, from_b = static_cast<uint32_t>(row8 * B.stride) + piece * 16u;
        uint32_t step_a = static_cast<uint32_t>(WAVES * 8 * A.stride), step_b = static_cast<uint32_t>(WAVES * 8 * B.stride);
        // one of the LOADS_A + LOADS_B loads of a stage
        const auto request_one = [&](uint8_t* to, int stage, int n) {
            if (n < LOADS_A) load_to_lds(ra, to + (n * WAVES + wave) * 8 * TILE_K, from_a + n * step_a, stage * TILE_K);
            else             load_to_lds(rb, to + (BM + ((n - LOADS_A) * WAVES + wave) * 8) * TILE_K, from_b + (n - LOADS_A) * step_b, stage * TILE_K);
        };
        const auto request = [&](uint8_t* to, int stage) {
            // (the eight offsets are added up anew for every stage: kept, they are registers that the tiles need)
#if defined(__HIP_DEVICE_COMPILE__)
            asm volatile("" : "+s"(step_a), "+s"(step_b));
#endif
#pragma unroll
            for (int n = 0; n < LOADS_A + LOADS_B; ++n) request_one(to, stage, n);
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
        // with the next stage's loads one by one between the matrix instructions
        const auto contract_and_request = [&](uint8_t* to, int stage) {
#if defined(__HIP_DEVICE_COMPILE__)
            asm volatile("" : "+s"(step_a), "+s"(step_b));
            __builtin_amdgcn_s_setprio(1);
            step_tiles_between<Step>(a, b, acc, [&](int n) {
                __builtin_amdgcn_sched_barrier(0);
                if (n < LOADS_A + LOADS_B) request_one(to, stage, n);
                __builtin_amdgcn_sched_barrier(0);
            });
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
        bare_barrier();
        // (past the last stage that one is requested again, into an array that nobody reads any more; group 1 begins with a product of zeros:
        // conditions around either are branches at which the registers of all tiles have to meet)
        if (wm == 0) {
            const auto stage = [&](uint8_t* here, uint8_t* next, int s) {
                read(here);
                request(next, s + 1 < stages ? s + 1 : s);
                wait_lds();
                bare_barrier();
                contract();
                wait_loads();
                bare_barrier();
            };
            int s = 0;
#pragma unroll 1
            for (; s + 2 <= stages; s += 2) {
                stage(even, odd, s);
                stage(odd, even, s + 1);
            }
            if (s < stages) stage(even, odd, s);
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i) a[i][0] = a[i][1] = v4i{};
#pragma unroll
            for (int j = 0; j < TN; ++j) b[j][0] = b[j][1] = v4i{};
            const auto stage = [&](uint8_t* here, uint8_t* next, int s) {
                contract_and_request(next, s + 1 < stages ? s + 1 : s);
                bare_barrier();
                read(here);
                wait_lds();
                wait_loads();
                bare_barrier();
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

// The t-th tile of tiles_m x tiles_n: bands of eight rows of tiles, along the columns, so that the work-groups that run at once on one XCD (a run of
// numbers: xcd_contiguous_index) share rows and columns of both operands.
__device__ __forceinline__ void tile_of(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int BAND = 8;
    const int band = t / (BAND * tiles_n), left = tiles_m - band * BAND, rows = left < BAND ? left : BAND;
    t -= band * BAND * tiles_n;
    tm = band * BAND + t % rows;
    tn = t / rows;
}

// Tiles of 256 (TilePingPong), 128 or 64 (TileDeep) a side: whichever is done first.  A round of them over all CUs takes, per stage: `large`, 0.74 and
// 0.32 us; a round of few takes a bit more than half of that (alone, a work-group has the caches and the power to itself), and two work-groups of the
// smallest share a CU, so that a part of a round of those is just that part.  Measured: in two halves 4096 x 4096 x 4096 327 us with 256 a side and 397
// with 128 (its symmetric products 247 and 209), 2048 x 2048 x 2048 138, 49 and 81 with 64, 1536 x 1536 x 1536 symmetric 33 with 128 and 23 with 64; in
// 8-bit integers over 4096, N tokens onto 4096 channels, quantizer included: N = 256 55, 26 and 19, 1024 60, 33 and 49, 4096 85, 115 and 174.
// `cut`: what the last, partial round of tiles of 128 takes instead where its tiles are cut along k (CutTiles), in rounds, `few` the same of the round that
// fewer tiles of 64 than CUs are; 0: they are not.
inline double partial_round(double part) { return part > 0.0 ? 0.55 + 0.45 * part : 0.0; }
template <class Tiles>
int tile_side(const Tiles& tiles, double large, double cut = 0.0, double few = 0.0) {
    const double cus = device_cu_count();
    const auto time = [&](double round, double share, double last) {
        const double whole = std::floor(share), part = share - whole;
        return round * (whole + (last > 0.0 ? last : partial_round(part)));
    };
    const double t256 = time(large, tiles(256) / cus, 0.0), t128 = time(0.74, tiles(128) / cus, cut), t64 = 0.32 * (few > 0.0 ? few : std::fmax(1.0, tiles(64) / cus));
    return t256 <= t128 && t256 <= t64 ? 256 : t128 <= t64 ? 128 : 64;
}

// The tiles of 128 behind the last whole round, each cut along k into `slices` work-groups of `stages` stages (the last of them perhaps fewer), so that
// together they fill the CUs once; their sums are joined by a launch of its own, in their order.  slices = 1: not worth that launch and its way
// through memory, 10 us.  Measured, five steps of newton_schulz.hip without / with: 4096 x 4096 (528 tiles of a symmetric product) 3938 / 3465 us,
// 2944 x 2944 (276) 1963 / 1542; 3968 x 4096 (496: none are cut) 3345 / 3217 from tiles numbered through all matrices alone.
struct CutTiles { int64_t whole, left; int slices, stages; double rounds; };
inline CutTiles cut_tiles(int64_t tiles, int stages) {
    const int64_t cus = device_cu_count();
    CutTiles c{tiles, 0, 1, stages, 0.0};                // (none is)
    const int64_t left = tiles % cus;
    if (tiles < cus || left == 0) return c;
    int64_t slices = cus / left < stages / 4 ? cus / left : stages / 4;
    if (slices < 2) return c;
    const int each = static_cast<int>((stages + slices - 1) / slices);
    slices = (stages + each - 1) / each;
    const double rounds = (each + 10.0 / 0.74) / stages;
    if (rounds < partial_round(static_cast<double>(left) / static_cast<double>(cus))) c = CutTiles{tiles - left, left, static_cast<int>(slices), each, rounds};
    return c;
}

// ... and all tiles of 64 where they are few under a long k: a CU draws some 50 to 80 GB/s however much it has requested, so that a tile's stage of 16
// KB takes 0.2 us, and slices on other CUs draw beside it.  The join's launch and its way through memory are 3 us and
// one for every hundred slices.  Measured, five steps without / with: 256 x 768 (10 tiles) 104 / 100 us, 256 x 2048 149 / 115, 128 x 4096 197 / 100; where the rule
// refuses, 4 x 256 x 1024 (40) 126 / 128, 768 x 768 (78) 152 / 165; in 8-bit integers 128 x 8192 -> 1024 (32) 30.6 / 25.6, 32 x 4096 -> 1024 (16) 13.5 / 12.4,
// and 17 x 4096 -> 4096 (64), refused, 14.3 / 15.5.
inline CutTiles cut_few_tiles(int64_t tiles, int stages) {
    const int64_t cus = device_cu_count();
    CutTiles c{tiles, 0, 1, stages, 0.0};
    int64_t slices = tiles > 0 ? cus / tiles : 0;
    for (const int64_t most : {static_cast<int64_t>(stages / 4), int64_t{16}}) slices = slices < most ? slices : most;
    if (slices < 2) return c;
    const int each = static_cast<int>((stages + slices - 1) / slices);
    slices = (stages + each - 1) / each;
    const double rounds = (each + (3.0 + static_cast<double>(tiles * slices) / 100.0) / 0.2) / stages;
    if (rounds < 1.0) c = CutTiles{0, tiles, static_cast<int>(slices), each, rounds};
    return c;
}

}  // namespace
}  // namespace ppmlhip
