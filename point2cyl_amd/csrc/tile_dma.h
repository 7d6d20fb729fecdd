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

// Piece `piece` of a tile is 1 KB of it: 1024 / RB rows.  The byte that lane `lane` fetches for it, counted from row 0 at this k; rows past `last` are
// read from row `last` (their results are never stored).
template <int RB>
__device__ __forceinline__ unsigned p2c_tile_source(int piece, int ld, int last, int lane)
{
    const int r = piece * (1024 / RB) + lane / (RB / 16);
    return (unsigned)min(r, last) * (unsigned)ld + (((lane & (RB / 16 - 1)) ^ p2c_tile_swz<RB>(r)) << 4);
}
// one copy of one wave; lds (the piece's place) must be wave-uniform
__device__ __forceinline__ void p2c_tile_piece(const char *src, char *lds)
{
    __builtin_amdgcn_global_load_lds((p2c_glb_ptr)src, (p2c_lds_ptr)lds, 16, 0, 0);
}

// Waits until at most N of this wave's copies are in flight and every LDS read it issued has returned, then meets the workgroup.
template <int N>
__device__ __forceinline__ void p2c_tile_wait()
{
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);         // (vmcnt N, lgkmcnt 0; as a builtin, so that the compiler knows what has arrived)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
