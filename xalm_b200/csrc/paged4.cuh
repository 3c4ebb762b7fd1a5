// paged4.cuh — what the kernels of the paged cache of 4-bit numbers (xalm_cuda_paged4_*) share: where blocks lie in a page.
//
// A block is 32 neighbouring entries of a head, x = d (c - 8) with d in fp16 and codes c of 4 bits.  The kv heads of a page have a run of bytes each: the slots' key codes, the keys'
// scales, the values' codes, the values' scales.  A slot's codes fill 64, 128 or 256 entries.  They lie in the order in which the lanes of attention's products hold them, so that a lane reads its
// own from the copied tile in shared memory and no exchange is needed behind that: a key's block goes to 4 lanes, 8 entries (a word) to each, a value's to 8 lanes, 4 entries to each; and what a lane has
// of a slot's blocks lies together, 4 to 32 bytes by loads of up to 16.
#pragma once
#include "paged.cuh"

namespace xalm {
namespace paged {

struct Pool4 {
	uint8_t* at;
	long long page, head; // bytes
	int kg, vg;           // blocks of a slot's keys and values: 2, 4 or 8
};
__host__ __device__ __forceinline__ int blocks_of(int n) { return n <= 64 ? 2 : n <= 128 ? 4 : 8; }
// where in a run the sections begin, and the run's bytes: a block has 16 bytes of codes and 2 of scale
__host__ __device__ __forceinline__ int key_scales_at(int kg, int shift) { return (kg * 16) << shift; }
__host__ __device__ __forceinline__ int values_at(int kg, int shift) { return (kg * 18) << shift; }
__host__ __device__ __forceinline__ int value_scales_at(int kg, int vg, int shift) { return (kg * 18 + vg * 16) << shift; }
__host__ __device__ __forceinline__ int run_bytes(int kg, int vg, int shift) { return ((kg + vg) * 18) << shift; }

// Kernels by the type of the queries (bf16, fp16, fp32) and the (token, head) rows of a unit
enum Kind4 { B8, B16, H4, H16, F4, F16, TILE };
struct Shape4 {
	int rows, per_sm; // rows of a unit (0: none for such heads), CTAs to an SM
};
Shape4 attn4_shape(const Pool4& p, const BatchView& b, int kind);
int launch_attn4(const Attn& a, const Pool4& p, int part, int type, int kind, cudaStream_t s);
Shape4 tile4_shape(const Pool4& p);
int launch_attn4_tile(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s);

} // namespace paged
} // namespace xalm
