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

// One 16 x 16 x (128 bytes) product: `a`, `b` the two 64-byte halves of the rows
struct StepI8 {
    typedef v4i Acc;
    __device__ static __forceinline__ void step(const v4i (&a)[2], const v4i (&b)[2], v4i& acc) {
#if defined(__HIP_DEVICE_COMPILE__)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[0], b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[1], b[1], acc, 0, 0, 0);
#endif
    }
};
// The halves are the upper and lower parts of 32 elements; the product of the two lower parts is left out
struct StepF16x2 {
    typedef v4f Acc;
    __device__ static __forceinline__ void step(const v4i (&a)[2], const v4i (&b)[2], v4f& acc) {
#if defined(__HIP_DEVICE_COMPILE__)
        const v8h ah = __builtin_bit_cast(v8h, a[0]), al = __builtin_bit_cast(v8h, a[1]);
        const v8h bh = __builtin_bit_cast(v8h, b[0]), bl = __builtin_bit_cast(v8h, b[1]);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, acc, 0, 0, 0);
#endif
    }
};

// WM x WN waves, each with TM x TN tiles of 16 x 16.  In lane l, register r of acc[i][j] holds the product of A's row
// m0 + (wave's first) + 16 i + 4 (l / 16) + r and B's row n0 + (wave's first) + 16 j + l % 16.
//
// A row's 128 bytes lie in LDS as eight pieces of sixteen, piece p of row r in place p ^ (r & 7): sixteen lanes that read the
// same piece of sixteen rows meet all banks.  The loads to LDS put lane l's piece at place l, so it is the address that a lane
// loads from which is permuted.
template <class Step, int WM, int WN, int TM, int TN>
struct TileLoop {
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int STAGE = (BM + BN) * TILE_K;
    static constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES;      // a load fetches eight rows
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads per wave");
    typedef typename Step::Acc Acc;

    __device__ static __forceinline__ void run(const RowBytes& A, const RowBytes& B, int m0, int n0, int stages, Acc (&acc)[TM][TN]) {
        __shared__ __attribute__((aligned(128))) uint8_t even[STAGE], odd[STAGE];
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = wave / WN, wn = wave % WN;
        // (rows behind the last one are that row again: their products are nobody's)
        const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(A.base + m0 * A.stride), 0, 0x7fffffff, 0x00020000);
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(B.base + n0 * B.stride), 0, 0x7fffffff, 0x00020000);
        const int row8 = lane >> 3, piece = (lane & 7) ^ row8;
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
        const int lane_at[2] = {(lane & 15) * TILE_K + (((lane >> 4) ^ (lane & 7)) * 16), (lane & 15) * TILE_K + (((4 + (lane >> 4)) ^ (lane & 7)) * 16)};
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
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int i = 0; i < TM; ++i) Step::step(a[i], b[j], acc[i][j]);
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

}  // namespace
}  // namespace ppmlhip
