// tile_dma.h -- operand tiles of a matrix product copied straight from memory into LDS (gfx950), shared by muon.hip and int8.hip.
//
// A tile is R rows of RB bytes (RB = 64 or 128), rows ld bytes apart in memory, rows RB apart in LDS.  One wave instruction copies 1 KB: lane l
// supplies 16 bytes of its own choice, the hardware places them at (wave-uniform base) + 16 l.  So the permutation that makes the fragment reads
// free of bank conflicts is applied to the SOURCE address: the 16-byte chunk c of row r stands at chunk position c ^ swz(r), swz(r) =
// (r / (256 / RB)) mod (RB / 16).  A fragment read takes one chunk of 16 consecutive rows per quarter-wave pair: with this swz they cover the 64
// banks exactly once.
#pragma once
#include "common.h"

typedef __attribute__((address_space(3))) void *p2c_lds_ptr;
typedef const __attribute__((address_space(1))) void *p2c_glb_ptr;

template <int RB>
__device__ __forceinline__ int p2c_tile_swz(int r) { return (r / (256 / RB)) & (RB / 16 - 1); }

// byte offset in LDS of chunk c of row r
template <int RB>
__device__ __forceinline__ int p2c_tile_at(int r, int c) { return r * RB + ((c ^ p2c_tile_swz<RB>(r)) << 4); }

// Copies rows [0, R) x RB bytes with NW waves; `wave` must be wave-uniform.  src: first byte of row 0 at this k; rows past `last` are read from
// row `last` (their results are never stored).  Every wave issues exactly R * RB / 1024 / NW copies.
template <int R, int RB, int NW>
__device__ __forceinline__ void p2c_tile_copy(const char *src, long long ld, int last, char *lds, int wave, int lane)
{
    constexpr int ROWS = 1024 / RB, PIECES = R / ROWS;      // rows per instruction, instructions per tile
    static_assert(PIECES % NW == 0, "the same number of copies in every wave");
    const int r8 = lane / (RB / 16), p = lane & (RB / 16 - 1);
#pragma unroll
    for (int i = 0; i < PIECES / NW; ++i) {
        const int piece = wave + i * NW, r = piece * ROWS + r8;
        const char *g = src + (long long)min(r, last) * ld + ((p ^ p2c_tile_swz<RB>(r)) << 4);
        __builtin_amdgcn_global_load_lds((p2c_glb_ptr)g, (p2c_lds_ptr)(lds + piece * 1024), 16, 0, 0);
    }
}

// Waits until at most N of this wave's copies are in flight and every LDS read it issued has returned, then meets the workgroup.
template <int N>
__device__ __forceinline__ void p2c_tile_wait()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);         // (vmcnt N, lgkmcnt 0; as a builtin, so that the compiler knows what has arrived)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
