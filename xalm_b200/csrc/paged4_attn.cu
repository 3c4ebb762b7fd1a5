// paged4_attn.cu — attention over paged caches of 4-bit numbers (paged4.cuh).
#include "paged4.cuh"

#include <algorithm>
#include <type_traits>

namespace xalm {
namespace paged {

// =========================================================================================================================================
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, in one pass over the pages; k = d (c - 8), so that s_j = scale sum_blocks d sum_i q_i (c_i - 8), and the sums are of
// (p_j d_j) (c_j - 8), block by block.  The codes are the products' first operand as they are (16 keys, then 16 entries of the values, as rows), the (token, head) rows their columns: eight of
// them, or four with what rounding left of the second operand beside them.  So nothing is rounded that the cache holds, scales are applied in fp32, and a value that a row does not see, whatever
// its scale, is left out with the row's own scale of 0.
// A step of single tokens reads every key and value once for a handful of rows, 144 bytes for 128 entries of both, and needs 425 instructions for 16 keys and values and a warp (a third takes the codes
// apart), at 60 % of what an SM issues and 42 % of HBM's rate over the whole of a call of 64 tokens: what is between is waiting, and the pieces' ends.  So each of four warps has 16 keys of a tile, its own ring of four stages filled by cp.async, its own maxima and sums, and
// waits for nobody; the warps join at the end of a piece.  Registers bound the CTAs: four to an SM with eight rows, three with 16.
// Measured, heads of 128, 8 kv heads, four rows to each: 128 tokens behind 8000 to 32000 670 us, 4.4 TB/s (67 % of measured); 64 behind 1000 to 8000 94 us; eight rows to a kv head cost
// what four do (88 us, 64 behind 4096), 16 72 with half the kv heads; 32 sequences of three to six tokens of fp16 110.  Loads to registers instead of the ring: 206 us for the 64; codes as they lie in the word, for
// bf16, with 376 instructions: the same, since the ALU pipe, not the FMA pipe, is full then.
// =========================================================================================================================================
constexpr int FT = 128, FW = FT / 32, FK = KT / FW; // keys of a warp in every tile
constexpr int FP = 20;                              // floats between the probabilities of a warp's rows

// Kernels by the type of the queries and the rows of a unit.  How p d enters the second product: one fp16 number (bf16 results), two in turn, or two in columns of their own (SPLIT, where a tile of
// columns has four rows; fp32 queries enter the first product so too).  Its unit is taken from the largest scale that a row has seen, which leaves fp16 and bf16 results their bits wherever scales are
// less than 2^24 apart; fp32 results would lose some from 2^12 on, so there it follows the products themselves, down too where the maxima grow: 64 fp32 tokens behind 1000 to 8000 take 103 us with the one, 102
// with the other, 32 sequences of three to six 189 and 177.
template <int KG, int VG, int KIND>
struct Size4 {
	static constexpr bool WIDE = KIND == F4 || KIND == F16, SPLIT = WIDE || KIND == H4, TWO = KIND == H16;
	static constexpr int NT = KIND == B16 || KIND == H16 ? 2 : KIND == F16 ? (VG == 8 ? 2 : 4) : 1; // tiles of 8 columns
	static constexpr int M = SPLIT ? NT * 4 : NT * 8;                                                     // rows of a unit
	static constexpr int CTAS = NT == 1 ? (VG == 8 || KG == 8 ? 3 : 4) : NT == 2 && VG < 8 ? 3 : 2;       // to an SM, as registers allow
	static constexpr int OP = VG * 32 + 4;                                            // floats between rows of sums
	static constexpr int STAGE = (KG + VG) * 288, STAGES = 4, WARP = STAGES * STAGE > M * OP * 4 ? STAGES * STAGE : M * OP * 4; // bytes of 16 keys and values; of a warp's stages, whose place its sums take
	static constexpr size_t own = (size_t) FW * WARP + (NT * KG * 2 * 64 + FW * NT * 8 * FP + FW * M * 2 + NT * 8 * 2) * 4;
};

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
	             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
	             : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) { // added to nothing
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
	             : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
	             : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// N words of shared memory from an address that is a multiple of their size (of 16 bytes at most)
template <int N>
__device__ __forceinline__ void read_words(uint32_t p, uint32_t (&x)[N]) {
	if constexpr (N == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[0]) : "r"(p));
	else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(p));
	else
#pragma unroll
		for (int i = 0; i < N; i += 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]) : "r"(p + i * 4));
}
// A number that is kept in a register, not computed again wherever it is used
__device__ __forceinline__ uint32_t kept(uint32_t x) {
	asm volatile("" : "+r"(x));
	return x;
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool there) { // zeros where there is nothing
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __high2float(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
	uint32_t r;
	asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); } // -126 <= e <= 127
__device__ __forceinline__ void load8_any(const uint8_t* p, long long i, int type, float (&x)[8]) {
	if (type == XALM_F32) load8(reinterpret_cast<const float*>(p) + i, x);
	else if (type == XALM_F16) load8(reinterpret_cast<const __half*>(p) + i, x);
	else load8(reinterpret_cast<const __nv_bfloat16*>(p) + i, x);
}

// Codes of a word as four pairs of fp16 numbers (c - 8) 2^-10: codes 0 and 4, 1 and 5, 2 and 6, 3 and 7.  Where they lie in the word codes are numbers c 2^-24 and c 2^-20 below fp16's normal ones,
// which one multiplication and addition bring there without a rounding.  (As they are the products would be exact too, but a product's terms are lined up by the exponents that are written:
// results were 1.2e-5 off where these are 4e-7.)
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&h)[4]) {
	const uint32_t w8 = w >> 8;
#pragma unroll
	for (int i = 0; i < 4; i++) {
		const uint32_t x = (i < 2 ? w : w8) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
		const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), i & 1 ? __float2half2_rn(1024.f) : __float2half2_rn(16384.f), __float2half2_rn(-0.0078125f));
		h[i] = *reinterpret_cast<const uint32_t*>(&y);
	}
}
__device__ __forceinline__ float exp2_fast(float x) {
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}
// the larger magnitudes of two pairs; signs are of no use
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
	uint32_t r;
	asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
	return r;
}

// What a lane holds of 16 keys and values: of keys lane / 4 and 8 behind it a word of each block, of values lane % 4, and 4, 8 and 12 behind it, four entries of each
template <int KG>
struct Keys {
	uint32_t w[2][KG], s[2][KG / 2];
};
template <int VG>
struct Values {
	uint32_t w[4][VG / 2], s[4][VG / 2];
};

constexpr float NONE = -3.0e38f; // the maximum before the first key
constexpr int LEAST = -100;      // products of fp32 rows below 2^LEAST make the second product's unit no smaller: they are of keys far below others whose scales are zeros
// s f - m: in one step where that is off by less than 2^-6 from the rounded product, which m is one of; else in two, so that the largest score is 0 above itself
constexpr float COARSE = 262144.f;
__device__ __forceinline__ float above(float s, float f, float m, bool coarse) { return coarse ? __fsub_rn(__fmul_rn(s, f), m) : fmaf(s, f, -m); }

// A piece by one warp: its 16 keys of each tile, the unit's rows as columns of the products
template <typename Z, int KG, int VG>
__device__ __forceinline__ void piece4(const Attn& a, const Pool4& pool, const Piece& x, int vis, int least, const uint2* s_q, const float* s_fac, const int* s_lim, float* sp, uint8_t* stages, float2* s_ml) {
	constexpr int NT = Z::NT, STAGES = Z::STAGES, STAGE = Z::STAGE;
	constexpr bool SPLIT = Z::SPLIT, WIDE = Z::WIDE, TWO = Z::TWO;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane >> 2, t = lane & 3, P = 1 << a.c.shift;
	constexpr bool IN_REGS = NT == 1;
	uint2 q[IN_REGS ? KG * 2 : 1];
	float2 fac[NT];
	if constexpr (IN_REGS)
#pragma unroll
		for (int i = 0; i < KG * 2; i++) q[i] = s_q[i * 32 + lane];
	float acc[VG * 2][NT][4], m[NT][2], l[NT][2], mu[NT], room[NT]; // mu: what p d is multiplied with; room: the largest d (WIDE: p d) that it allows
#pragma unroll
	for (int n = 0; n < NT; n++) {
#pragma unroll
		for (int i = 0; i < VG * 2; i++)
#pragma unroll
			for (int e = 0; e < 4; e++) acc[i][n][e] = 0.f;
		fac[n] = *reinterpret_cast<const float2*>(s_fac + n * 8 + t * 2);
		m[n][0] = m[n][1] = NONE;
		l[n][0] = l[n][1] = 0.f;
		mu[n] = 1.f;
		room[n] = 0.f;
	}
	const int* table = a.b.table + (long long) x.s * a.b.table_row;
	int at = x.j0 * KT + warp * FK;
	const int end = min(x.j1 * KT, vis);
	auto id_at = [&](int key) { return key < end ? table[(x.key0 + key) >> a.c.shift] : 0; }; // looked at when its page is asked for
	// Copies, each lane's own 16 bytes at a time.  Values' 16 bytes lie in another order: those that four lanes t ask for at once, of keys t, in different banks.
	constexpr int VK = KG * 256, KS = VK + VG * 256, VS = KS + KG * 32; // sections of a stage
	auto turn = [](int key) { return VG == 8 ? (key & 3) * 32 : VG == 4 ? (key & 2) * 16 : 0; };
	const uint32_t ring = smem_u32(stages), to_k = kept(ring + lane * 16), to_v = kept(ring + VK + ((lane * 16) ^ turn(lane / VG)));
	const uint32_t k_lane = kept(ring + u * (KG * 16) + t * (KG * 4)), ks_lane = kept(ring + KS + u * (KG * 2)), v_lane = kept(ring + VK + t * (VG * 16) + ((u * (VG * 2)) ^ turn(t))),
	               vs_lane = kept(ring + VS + t * (VG * 2));
	const uint32_t p_write = kept(smem_u32(sp) + (t * 2 * FP + (u & 3) * 4 + (u >> 2)) * 4), p_read = kept(smem_u32(sp) + (u * FP + t * 4) * 4); // keys t, t + 4, .. side by side
	const int v_at = values_at(KG, a.c.shift), s_at = lane < KG * 2 ? key_scales_at(KG, a.c.shift) : value_scales_at(KG, VG, a.c.shift) - KG * 32, s_by = lane < KG * 2 ? KG * 2 : VG * 2;
	const uint8_t* from = pool.at + x.g * pool.head + lane * 16;
	auto bring = [&](int key, int id, int to) {
		const bool good = (unsigned) id < (unsigned) a.c.pages, there = good && key < end; // what is not there reads as zeros
		if (!good && lane == 0) report(a.c, ERR_PAGE);
		const uint8_t* run = from + (good ? id : 0) * pool.page;
		const int slot = (x.key0 + key) & (P - 1);
		const uint8_t *kw = run + slot * (KG * 16), *vw = run + (v_at + slot * (VG * 16));
#pragma unroll
		for (int i = 0; i < KG / 2; i++) copy16(to_k + to + i * 512, kw + i * 512, there);
#pragma unroll
		for (int i = 0; i < VG / 2; i++) copy16(to_v + to + i * 512, vw + i * 512, there);
		if ((KG + VG) * 2 == 32 || lane < (KG + VG) * 2) copy16(to_k + to + KS, run + (s_at + slot * s_by), there);
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	bool coarse = false;
	int id = id_at(at), full = 0, free = (STAGES - 1) * STAGE; // the stage to be read, and the one to be filled
#pragma unroll
	for (int i = 0; i < STAGES - 1; i++) {
		bring(at + i * KT, id, i * STAGE);
		id = id_at(at + (i + 1) * KT);
	}
	auto step = [&](auto edge) {
		constexpr bool EDGE = decltype(edge)::value; // some rows may not see some keys, or scores are large
		asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
		__syncwarp(); // the stage is there, and nobody reads the one before any more
		bring(at + (STAGES - 1) * KT, id, free);
		id = id_at(at + STAGES * KT);
		const int stage = full;
		free = full;
		full = full == (STAGES - 1) * STAGE ? 0 : full + STAGE;
		Keys<KG> k;
#pragma unroll
		for (int i = 0; i < 2; i++) {
			read_words<KG>(k_lane + stage + i * (KG * 128), k.w[i]);
			read_words<KG / 2>(ks_lane + stage + i * (KG * 16), k.s[i]);
		}
		// ---- scores: keys as rows of the product ----
		float s[NT][4];
#pragma unroll
		for (int n = 0; n < NT; n++)
#pragma unroll
			for (int e = 0; e < 4; e++) s[n][e] = 0.f;
#pragma unroll
		for (int g = 0; g < KG; g++) {
			uint32_t h0[4], h1[4];
			codes4(k.w[0][g], h0);
			codes4(k.w[1][g], h1);
			const float d0 = g & 1 ? half_hi(k.s[0][g / 2]) : half_lo(k.s[0][g / 2]), d1 = g & 1 ? half_hi(k.s[1][g / 2]) : half_lo(k.s[1][g / 2]);
#pragma unroll
			for (int n = 0; n < NT; n++) {
				uint2 qa, qb;
				if constexpr (IN_REGS) { qa = q[g * 2]; qb = q[g * 2 + 1]; }
				else {
					qa = s_q[((n * KG + g) * 2) * 32 + lane];
					qb = s_q[((n * KG + g) * 2 + 1) * 32 + lane];
				}
				float c[4];
				mma16_new(c, h0[0], h1[0], h0[1], h1[1], qa.x, qa.y);
				mma16(c, h0[2], h1[2], h0[3], h1[3], qb.x, qb.y);
				s[n][0] = fmaf(c[0], d0, s[n][0]);
				s[n][1] = fmaf(c[1], d0, s[n][1]);
				s[n][2] = fmaf(c[2], d1, s[n][2]);
				s[n][3] = fmaf(c[3], d1, s[n][3]);
			}
		}
		// ---- probabilities ----
		float p[NT][4];
		bool grow = false;
#pragma unroll
		for (int n = 0; n < NT; n++) {
			if constexpr (WIDE) // the rest of the queries has columns of its own
#pragma unroll
				for (int e = 0; e < 4; e++) s[n][e] += __shfl_xor_sync(0xffffffffu, s[n][e], 2);
#pragma unroll
			for (int e = 0; e < 4; e++) p[n][e] = above(s[n][e], e & 1 ? fac[n].y : fac[n].x, m[n][e & 1], EDGE && coarse);
			if constexpr (EDGE) {
				const int2 lim = *reinterpret_cast<const int2*>(s_lim + n * 8 + t * 2);
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (at + u + (e >> 1) * 8 >= (e & 1 ? lim.y : lim.x)) p[n][e] = -INFINITY;
			}
			grow = grow || fmaxf(fmaxf(p[n][0], p[n][1]), fmaxf(p[n][2], p[n][3])) > 2.f;
		}
		if (__any_sync(0xffffffffu, grow)) { // rare behind the first keys: probabilities may be up to 4
#pragma unroll
			for (int n = 0; n < NT; n++) {
				float up[2]; // what the maxima grow by, and the units with them
#pragma unroll
				for (int c = 0; c < 2; c++) {
					const float f0 = c ? fac[n].y : fac[n].x;
					float top = fmaxf(p[n][c] == -INFINITY ? NONE : __fmul_rn(s[n][c], f0), p[n][c + 2] == -INFINITY ? NONE : __fmul_rn(s[n][c + 2], f0));
#pragma unroll
					for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
					top = fmaxf(m[n][c], top);
					up[c] = top - m[n][c];
					m[n][c] = top;
					l[n][c] *= exp2f(-up[c]);
					coarse = coarse || (fabsf(top) > COARSE && top != NONE);
				}
				float g = 1.f;
				if constexpr (WIDE) { // all products so far are as much smaller: so is what they need room for
					const float up0 = __shfl_sync(0xffffffffu, up[0], u >> 1), up1 = __shfl_sync(0xffffffffu, up[1], u >> 1);
					if (room[n] > 0.f) {
						const int e = min((int) fminf(u & 1 ? up1 : up0, 100.f), (__float_as_int(room[n]) >> 23) - 127 - (LEAST + 2));
						g = pow2(e);
						mu[n] *= g;
						room[n] *= pow2(-e);
					}
				}
				const float f0 = exp2f(-up[0]) * (WIDE ? __shfl_sync(0xffffffffu, g, t * 8) : 1.f), f1 = exp2f(-up[1]) * (WIDE ? __shfl_sync(0xffffffffu, g, t * 8 + 4) : 1.f);
#pragma unroll
				for (int i = 0; i < VG * 2; i++) { acc[i][n][0] *= f0; acc[i][n][2] *= f0; acc[i][n][1] *= f1; acc[i][n][3] *= f1; }
			}
			coarse = __any_sync(0xffffffffu, coarse);
#pragma unroll
			for (int n = 0; n < NT; n++)
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (p[n][e] != -INFINITY) p[n][e] = above(s[n][e], e & 1 ? fac[n].y : fac[n].x, m[n][e & 1], coarse);
		}
		__syncwarp();
#pragma unroll
		for (int n = 0; n < NT; n++)
#pragma unroll
			for (int e = 0; e < 4; e++) {
				p[n][e] = exp2_fast(p[n][e]);
				l[n][e & 1] += p[n][e];
				asm volatile("st.shared.f32 [%0], %1;" ::"r"(p_write + ((n * 8 + (e & 1)) * FP + (e >> 1) * 2) * 4), "f"(p[n][e]) : "memory");
			}
		__syncwarp();
		// ---- sums: values' entries as rows of the product ----
		Values<VG> v;
#pragma unroll
		for (int i = 0; i < 4; i++) {
			read_words<VG / 2>(v_lane + stage + i * (VG * 64), v.w[i]);
			read_words<VG / 2>(vs_lane + stage + i * (VG * 8), v.s[i]);
		}
		uint32_t vs[NT][2 * VG];
		float4 p4[NT];
#pragma unroll
		for (int n = 0; n < NT; n++) {
#pragma unroll
			for (int i = 0; i < 2 * VG; i++) vs[n][i] = v.s[i / (VG / 2)][i % (VG / 2)];
			if constexpr (EDGE) { // what the row does not see may have any scale, a NaN too
				const int lim = s_lim[n * 8 + u];
#pragma unroll
				for (int i = 0; i < 4; i++)
					if (at + t + i * 4 >= lim)
#pragma unroll
						for (int w = 0; w < VG / 2; w++) vs[n][i * (VG / 2) + w] = 0;
			}
			asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(p4[n].x), "=f"(p4[n].y), "=f"(p4[n].z), "=f"(p4[n].w) : "r"(p_read + n * 8 * FP * 4));
			uint32_t big = vs[n][0];
#pragma unroll
			for (int i = 1; i < 2 * VG; i++) big = max_abs2(big, vs[n][i]);
			float top = fmaxf(fabsf(half_lo(big)), fabsf(half_hi(big)));
			if constexpr (WIDE) top *= fmaxf(fmaxf(p4[n].x, p4[n].y), fmaxf(p4[n].z, p4[n].w)); // no product of these keys is larger
			if (__any_sync(0xffffffffu, top > room[n])) {
				if constexpr (WIDE) { // the largest itself: a large scale of a key that has next to no weight takes no bits from the others
					top = 0.f;
#pragma unroll
					for (int i = 0; i < 4; i++) {
						uint32_t own = vs[n][i * (VG / 2)];
#pragma unroll
						for (int w = 1; w < VG / 2; w++) own = max_abs2(own, vs[n][i * (VG / 2) + w]);
						top = fmaxf(top, (i == 0 ? p4[n].x : i == 1 ? p4[n].y : i == 2 ? p4[n].z : p4[n].w) * fmaxf(fabsf(half_lo(own)), fabsf(half_hi(own))));
					}
				}
				float y = fmaxf(top, room[n]);
				y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
				y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
				float f = 1.f;
				if (y > room[n]) {
					const int e = max((__float_as_int(y) >> 23) - 127, LEAST); // 2^e <= y < 2^(e + 1): scales up to twice that have room, and products up to eight times
					const float to = pow2(11 - e);
					f = to / mu[n];
					mu[n] = to;
					room[n] = pow2(min(e + (WIDE ? 4 : 2), 127));
				}
				const float f0 = __shfl_sync(0xffffffffu, f, t * 8), f1 = __shfl_sync(0xffffffffu, f, t * 8 + 4);
#pragma unroll
				for (int i = 0; i < VG * 2; i++) { acc[i][n][0] *= f0; acc[i][n][2] *= f0; acc[i][n][1] *= f1; acc[i][n][3] *= f1; }
			}
			p4[n].x *= mu[n]; p4[n].y *= mu[n]; p4[n].z *= mu[n]; p4[n].w *= mu[n];
		}
#pragma unroll
		for (int g = 0; g < VG; g++) {
			const uint32_t sel = g & 1 ? 0x7632 : 0x5410;
			uint32_t ab[4], cd[4];
			codes4(__byte_perm(v.w[0][g / 2], v.w[1][g / 2], sel), ab);
			codes4(__byte_perm(v.w[2][g / 2], v.w[3][g / 2], sel), cd);
#pragma unroll
			for (int n = 0; n < NT; n++) {
				float y[4];
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const uint32_t w = vs[n][i * (VG / 2) + g / 2];
					y[i] = (i == 0 ? p4[n].x : i == 1 ? p4[n].y : i == 2 ? p4[n].z : p4[n].w) * (g & 1 ? half_hi(w) : half_lo(w));
				}
				uint32_t b0 = pack_half(y[0], y[1]), b1 = pack_half(y[2], y[3]), r0 = 0, r1 = 0;
				if constexpr (SPLIT || TWO) {
					r0 = pack_half(y[0] - half_lo(b0), y[1] - half_hi(b0));
					r1 = pack_half(y[2] - half_lo(b1), y[3] - half_hi(b1));
				}
				if constexpr (SPLIT) {
					b0 = u < 4 ? b0 : r0;
					b1 = u < 4 ? b1 : r1;
				}
#pragma unroll
				for (int i = 0; i < 2; i++) {
					mma16(acc[g * 2 + i][n], ab[2 * i], ab[2 * i + 1], cd[2 * i], cd[2 * i + 1], b0, b1);
					if constexpr (TWO) mma16(acc[g * 2 + i][n], ab[2 * i], ab[2 * i + 1], cd[2 * i], cd[2 * i + 1], r0, r1);
				}
			}
		}
	};
	for (; at + FK <= least && at < end && !coarse; at += KT) step(std::false_type());
	for (; at < end; at += KT) step(std::true_type());
	asm volatile("cp.async.wait_group 0;" ::: "memory");
	__syncwarp(); // the sums take the stages' place
	// ---- this warp's maxima, sums and rows ----
#pragma unroll
	for (int n = 0; n < NT; n++) {
#pragma unroll
		for (int c = 0; c < 2; c++)
#pragma unroll
			for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
		const float inv = 1024.f / mu[n]; // a power of two; codes were taken as 2^-10 each
		const float i0 = __shfl_sync(0xffffffffu, inv, t * 8), i1 = __shfl_sync(0xffffffffu, inv, t * 8 + 4);
		const int row = SPLIT ? n * 4 + t * 2 : n * 8 + t * 2;
		const bool mine = !SPLIT || t < 2;
		if (mine && u == 0) {
			s_ml[warp * Z::M + row] = make_float2(m[n][0] == NONE ? -INFINITY : m[n][0], l[n][0]);
			s_ml[warp * Z::M + row + 1] = make_float2(m[n][1] == NONE ? -INFINITY : m[n][1], l[n][1]);
		}
#pragma unroll
		for (int g = 0; g < VG; g++)
#pragma unroll
			for (int c = 0; c < 2; c++) { // the row's entries 4 u .. 4 u + 3 of the block
				float y[4] = {acc[g * 2][n][c], acc[g * 2][n][c + 2], acc[g * 2 + 1][n][c], acc[g * 2 + 1][n][c + 2]};
#pragma unroll
				for (int e = 0; e < 4; e++) {
					if constexpr (SPLIT) y[e] += __shfl_xor_sync(0xffffffffu, y[e], 2);
					y[e] *= c ? i1 : i0;
				}
				if (mine) *reinterpret_cast<float4*>(reinterpret_cast<float*>(stages) + (row + c) * Z::OP + g * 32 + u * 4) = make_float4(y[0], y[1], y[2], y[3]);
			}
	}
}

template <int KG, int VG, int KIND>
__global__ void __launch_bounds__(FT, Size4<KG, VG, KIND>::CTAS) paged4_attn_kernel(const __grid_constant__ Attn a, const __grid_constant__ Part part, const Pool4 pool, const int type) {
	using Z = Size4<KG, VG, KIND>;
	constexpr int M = Z::M, OP = Z::OP;
	extern __shared__ __align__(16) uint8_t smem[];
	uint8_t* s_ring = smem;                                            // [FW][WARP]
	uint2* s_q = reinterpret_cast<uint2*>(s_ring + FW * Z::WARP);      // [NT][KG][2][32]: queries as the product wants them
	float* s_p = reinterpret_cast<float*>(s_q + Z::NT * KG * 2 * 32);  // [FW][NT * 8][FP]
	float2* s_ml = reinterpret_cast<float2*>(s_p + FW * Z::NT * 8 * FP); // [FW][M]
	float* s_fac = reinterpret_cast<float*>(s_ml + FW * M);            // [NT * 8]: from a product to a score in units of log2
	int* s_lim = reinterpret_cast<int*>(s_fac + Z::NT * 8);            // [NT * 8]: keys that the column's row sees
	uint8_t* s_plan = reinterpret_cast<uint8_t*>(s_lim + Z::NT * 8);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dv = a.c.dv;
	Plan plan;
	pdl_launch_dependents();
	make_plan<FT>(a, part, s_plan, plan);
	Walk k;
	bool more = walk_begin(a, part, plan, k);
	if (tid == 0) write_head(a, part, k, more, more && k.x.seg >= a.b.n_groups && k.x.key0 == 0, plan.share);
	for (; more; more = walk_next(a, part, plan, k)) {
		const Piece& x = k.x;
		if (x.j0 == x.j1) continue; // the same for every thread
		const int shared = plan.shs[x.s];
		const bool prefix = x.seg < a.b.n_groups;
		const int rows = min(M, x.rows - x.t * M), h0 = x.g * a.rep;
		constexpr bool split = Z::SPLIT;
		auto keys_of = [&](int r) { return prefix ? shared : own_keys(x.q, shared, a.rep, x.t * M + r); };
		__syncthreads(); // the piece before is written
		for (int n = warp; n < Z::NT; n += FW) { // queries, a tile of columns to a warp: 8 entries of each block to a lane
			const int u = lane >> 2, t = lane & 3, r = split ? n * 4 + (u & 3) : n * 8 + u;
			const bool there = r < rows;
			if (t == 0) s_lim[n * 8 + u] = there ? keys_of(r) : 0;
			const int w = x.t * M + r;
			const long long at = there ? (long long) (x.row0 + w / a.rep) * a.q_row + (h0 + w % a.rep) * a.c.d : 0;
			float y[KG][8], top = 0.f;
#pragma unroll
			for (int g = 0; g < KG; g++) {
#pragma unroll
				for (int e = 0; e < 8; e++) y[g][e] = 0.f;
				if (there && g * 32 + t * 8 < a.c.d) load8_any(a.q, at + g * 32 + t * 8, type, y[g]);
#pragma unroll
				for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(y[g][e]));
			}
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
			// the row times a power of two, so that its largest entry is between 2^14 and 2^15
			const int e0 = (__float_as_int(top) >> 23) - 127, e = e0 == 128 ? 0 : min(14 - e0, 126);
			const float f = e0 == 128 ? NAN : pow2(e); // a row with an infinity is no number, whatever the keys' signs
			if (t == 0) s_fac[n * 8 + u] = fminf(fmaxf(a.scale * 1.4426950408889634f * pow2(10 - e), -3.0e38f), 3.0e38f);
#pragma unroll
			for (int g = 0; g < KG; g++) {
				float z[8];
#pragma unroll
				for (int i = 0; i < 8; i++) {
					const float full = y[g][i] * f;
					float h = __half2float(__float2half_rn(full));
					if (Z::WIDE && u >= 4) h = full - h; // the rest
					z[i] = h;
				}
				s_q[((n * KG + g) * 2) * 32 + lane] = make_uint2(pack_half(z[0], z[4]), pack_half(z[1], z[5]));
				s_q[((n * KG + g) * 2 + 1) * 32 + lane] = make_uint2(pack_half(z[2], z[6]), pack_half(z[3], z[7]));
			}
		}
		__syncthreads();
		const int vis = keys_of(rows - 1), least = keys_of(0); // the last row sees the most
		float* sp = s_p + warp * Z::NT * 8 * FP;
		piece4<Z, KG, VG>(a, pool, x, vis, least, s_q, s_fac, s_lim, sp, s_ring + warp * Z::WARP, s_ml);
		__syncthreads();
		const bool direct = x.j0 == 0 && x.j1 == x.w && !prefix && shared == 0;
		const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
		for (int i = tid; i < rows * (dv / 4); i += FT) {
			const int row = i / (dv / 4), col = i % (dv / 4) * 4, w = x.t * M + row;
			float mx = -INFINITY, l = 0.f;
			float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
			for (int e = 0; e < FW; e++) mx = fmaxf(mx, s_ml[e * M + row].x);
#pragma unroll
			for (int e = 0; e < FW; e++) {
				const float2 ml = s_ml[e * M + row];
				const bool some = ml.x != -INFINITY || ml.y != 0.f; // else nothing that the row sees; a sum that is NaN stays one
				const float f = !some ? 0.f : ml.x == -INFINITY ? 1.f : exp2f(ml.x - mx);
				const float4 o = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(s_ring + e * Z::WARP) + row * OP + col);
				l += ml.y * f;
				v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
			}
			const bool any = l > 0.f || l != l;
			const long long tok = x.row0 + w / a.rep;
			const int h = h0 + w % a.rep;
			if (direct) {
				const float f = any ? 1.f / l : 0.f; // 0: a row that sees nothing, whose sums are zeros
				const float y[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
				const long long o = tok * a.out_row + h * dv + col;
				if (type == XALM_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o) = make_float4(y[0], y[1], y[2], y[3]);
				else if (type == XALM_F16) *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(a.out) + o) = make_uint2(pack_half(y[0], y[1]), pack_half(y[2], y[3]));
				else {
					const __nv_bfloat162 b[2] = {__floats2bfloat162_rn(y[0], y[1]), __floats2bfloat162_rn(y[2], y[3])};
					*reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o) = *reinterpret_cast<const uint2*>(b);
				}
				if (a.lse && col == 0) a.lse[tok * a.H + h] = any ? (mx + log2f(l)) * 0.6931471805599453f : -INFINITY;
			} else if (slot < part.slots) {
				*reinterpret_cast<float4*>(part.o + (slot * M + row) * dv + col) = v;
				if (col == 0) part.ml[slot * M + row] = make_float2(mx, l);
			}
		}
	}
	pdl_wait(); // beside the kernel of many rows, whose inputs were complete before it began, but not ahead of it to the join
}

// CTAs to an SM by registers (launch bounds) and shared memory
template <int KG, int VG, int KIND>
static Shape4 shape_of(const BatchView& b) {
	using Z = Size4<KG, VG, KIND>;
	const size_t smem = Z::own + plan_bytes(b.B, b.n_groups);
	return Shape4{Z::M, std::max(1, std::min(Z::CTAS, (int) (226 * 1024 / (smem + 1024))))};
}
template <int KIND>
static Shape4 shape4(const Pool4& p, const BatchView& b) {
	switch (p.kg * 16 + p.vg) {
#define XALM_PAGED4(K, V) case K * 16 + V: return shape_of<K, V, KIND>(b);
		XALM_PAGED4(2, 2) XALM_PAGED4(2, 4) XALM_PAGED4(2, 8) XALM_PAGED4(4, 2) XALM_PAGED4(4, 4) XALM_PAGED4(4, 8) XALM_PAGED4(8, 2) XALM_PAGED4(8, 4) XALM_PAGED4(8, 8)
#undef XALM_PAGED4
	}
	return Shape4{0, 0};
}
Shape4 attn4_shape(const Pool4& p, const BatchView& b, int kind) {
	return kind == B8 ? shape4<B8>(p, b) : kind == B16 ? shape4<B16>(p, b) : kind == H4 ? shape4<H4>(p, b) : kind == H16 ? shape4<H16>(p, b) : kind == F4 ? shape4<F4>(p, b) : shape4<F16>(p, b);
}

template <int KG, int VG, int KIND>
static int launch_kind(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	const size_t smem = Size4<KG, VG, KIND>::own + plan_bytes(a.b.B, a.b.n_groups);
	XALM_CUDA_CHECK(allow_smem((const void*) paged4_attn_kernel<KG, VG, KIND>));
	XALM_CUDA_CHECK(launch(paged4_attn_kernel<KG, VG, KIND>, a.part[part].grid, FT, smem, s, part > 0, a, a.part[part], p, type));
	return XALM_OK;
}
template <int KIND>
static int launch_blocks(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	switch (p.kg * 16 + p.vg) {
#define XALM_PAGED4(K, V) case K * 16 + V: return launch_kind<K, V, KIND>(a, p, part, type, s);
		XALM_PAGED4(2, 2) XALM_PAGED4(2, 4) XALM_PAGED4(2, 8) XALM_PAGED4(4, 2) XALM_PAGED4(4, 4) XALM_PAGED4(4, 8) XALM_PAGED4(8, 2) XALM_PAGED4(8, 4) XALM_PAGED4(8, 8)
#undef XALM_PAGED4
	}
	return set_error(XALM_ERR_INVALID, "paged attention: %d and %d blocks", p.kg, p.vg);
}
int launch_attn4(const Attn& a, const Pool4& p, int part, int type, int kind, cudaStream_t s) {
	switch (kind) {
		case B8: return launch_blocks<B8>(a, p, part, type, s);
		case B16: return launch_blocks<B16>(a, p, part, type, s);
		case H4: return launch_blocks<H4>(a, p, part, type, s);
		case H16: return launch_blocks<H16>(a, p, part, type, s);
		case F4: return launch_blocks<F4>(a, p, part, type, s);
		default: return launch_blocks<F16>(a, p, part, type, s);
	}
}

} // namespace paged
} // namespace xalm
