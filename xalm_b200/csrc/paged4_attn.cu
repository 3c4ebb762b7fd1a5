// paged4_attn.cu — attention over paged caches of 4-bit numbers (paged4.cuh).
#include "paged4.cuh"

#include <algorithm>

namespace xalm {
namespace paged {

// =========================================================================================================================================
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, in one pass over the pages.
// =========================================================================================================================================
constexpr int FT = 128, FW = FT / 32, FK = KT / FW; // keys of a warp in every tile
constexpr int FP = 20;                              // floats between the probabilities of a warp's rows

enum { FEW, MANY, F32 };
template <int KG, int VG, int KIND>
struct Size4 {
	static constexpr int NT = KIND == FEW ? 2 : VG == 8 ? (KIND == F32 ? 2 : 0) : 4; // tiles of 8 columns that fit a lane's registers
	static constexpr int M = KIND == F32 ? NT * 4 : NT * 8;                           // rows of a unit
	static constexpr int OP = VG * 32 + 4;                                            // floats between rows of sums
	static constexpr int SUMS = FW * M * OP;
	static constexpr size_t own = (size_t) (NT * KG * 2 * 64 + NT * KG * 8 + SUMS + FW * NT * 8 * FP + FW * M * 2 + NT * 8 * 2) * 4;
};

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
	             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
	             : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// N words from an address that is a multiple of their size (of 16 bytes at most)
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&x)[N]) {
	if constexpr (N == 1) asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(x[0]) : "l"(p));
	else if constexpr (N == 2) asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "l"(p));
	else
#pragma unroll
		for (int i = 0; i < N; i += 4)
			asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]) : "l"(p + i * 4));
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short) w)); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short) (w >> 16))); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
	uint32_t r;
	asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); } // -126 <= e <= 127
__device__ __forceinline__ float load_any(const uint8_t* p, long long i, int type) {
	return type == XALM_F32 ? reinterpret_cast<const float*>(p)[i] : type == XALM_F16 ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void load8_any(const uint8_t* p, long long i, int type, float (&x)[8]) {
	if (type == XALM_F32) load8(reinterpret_cast<const float*>(p) + i, x);
	else if (type == XALM_F16) load8(reinterpret_cast<const __half*>(p) + i, x);
	else load8(reinterpret_cast<const __nv_bfloat16*>(p) + i, x);
}

// Codes of a word as four pairs of fp16 numbers: codes 0 and 4, 1 and 5, 2 and 6, 3 and 7.  Where they lie in the word they are numbers c 2^-20, below fp16's normal ones and exact; a product's
// terms are lined up by their exponents, so that up to 6 of its 24 bits are lost: for fp32 results codes become c - 8.
template <bool WIDE>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&h)[4]) {
	constexpr uint32_t M = 0x00f000f0u;
	h[0] = (w << 4) & M;
	h[1] = w & M;
	h[2] = (w >> 4) & M;
	h[3] = (w >> 8) & M;
	if constexpr (WIDE)
#pragma unroll
		for (int i = 0; i < 4; i++) {
			const uint32_t x = h[i] | 0x64006400u; // 1024 + 16 c
			const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
			h[i] = *reinterpret_cast<const uint32_t*>(&y);
		}
}

// What a lane holds of 16 keys and values as they come: of keys lane / 4 and 8 behind it a word of each block, of values 4 (lane % 4) .. + 3 four entries of each
template <int KG>
struct Keys {
	uint32_t w[2][KG], s[2][KG / 2];
};
template <int VG>
struct Values {
	uint32_t w[4][VG / 2], s[4 * VG / 2]; // scales: value by value
};

// A piece by one warp: its 16 keys of each tile, the unit's rows as columns of the products.
// SPLIT: tiles of four rows, whose columns 4 .. 7 have what rounding to fp16 left of the queries (fp32) and of the probabilities
template <int KG, int VG, int NT, bool SPLIT, bool WIDE>
__device__ __forceinline__ void piece4(const Attn& a, const Pool4& pool, const Piece& x, int vis, int least, const uint2* s_q, const float* s_init, const float* s_fac, const int* s_lim, float* sp,
                                       float* s_o, float2* s_ml, int op, int most_rows) {
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, u = lane >> 2, t = lane & 3, P = 1 << a.c.shift;
	const int ks_at = key_scales_at(KG, a.c.shift), v_at = values_at(KG, a.c.shift), vs_at = value_scales_at(KG, VG, a.c.shift);
	constexpr bool IN_REGS = NT == 1;
	uint2 q[IN_REGS ? KG * 2 : 1];
	float2 init[IN_REGS ? KG : 1];
	if constexpr (IN_REGS) {
#pragma unroll
		for (int i = 0; i < KG * 2; i++) q[i] = s_q[i * 32 + lane];
#pragma unroll
		for (int g = 0; g < KG; g++) init[g] = *reinterpret_cast<const float2*>(s_init + g * 8 + t * 2);
	}
	float acc[VG * 2][NT][4], part[NT][VG], m[NT][2], l[NT][2], mu[NT], room[NT]; // part: sums of the probabilities times scales; mu: what those are multiplied with; room: the largest scale it allows
#pragma unroll
	for (int n = 0; n < NT; n++) {
#pragma unroll
		for (int i = 0; i < VG * 2; i++)
#pragma unroll
			for (int e = 0; e < 4; e++) acc[i][n][e] = 0.f;
#pragma unroll
		for (int g = 0; g < VG; g++) part[n][g] = 0.f;
		m[n][0] = m[n][1] = -INFINITY;
		l[n][0] = l[n][1] = 0.f;
		mu[n] = 1.f;
		room[n] = 0.f;
	}
	const int* table = a.b.table + (long long) x.s * a.b.table_row;
	const uint8_t* head = pool.at + x.g * pool.head;
	auto id_at = [&](int at) { // the page of keys `at` .. of the segment
		if (at >= vis) return 0;
		const int id = table[(x.key0 + at) >> a.c.shift];
		return id;
	};
	Keys<KG> k;
	Values<VG> v;
	auto run_of = [&](int at, int id, bool& there) {
		there = id >= 0 && id < a.c.pages;
		return head + (there ? id : 0) * pool.page;
	};
	auto load_keys = [&](int at, int id) {
		if (at >= vis) return;
		bool there;
		const uint8_t* run = run_of(at, id, there);
		const int slot = (x.key0 + at) & (P - 1);
#pragma unroll
		for (int i = 0; i < 2; i++) {
			const int j = slot + u + i * 8;
			load_words<KG>(run + j * (KG * 16) + t * (KG * 4), k.w[i]);
			load_words<KG / 2>(run + ks_at + j * (KG * 2), k.s[i]);
		}
		if (!there) { // reads as zeros
			if (lane == 0) report(a.c, ERR_PAGE);
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll
				for (int g = 0; g < KG / 2; g++) k.s[i][g] = 0;
		}
	};
	auto load_values = [&](int at, int id) {
		if (at >= vis) return;
		bool there;
		const uint8_t* run = run_of(at, id, there);
		const int slot = (x.key0 + at) & (P - 1);
#pragma unroll
		for (int i = 0; i < 4; i++) load_words<VG / 2>(run + v_at + (slot + t * 4 + i) * (VG * 16) + u * (VG * 2), v.w[i]);
		load_words<2 * VG>(run + vs_at + (slot + t * 4) * (VG * 2), v.s);
		if (!there)
#pragma unroll
			for (int i = 0; i < 2 * VG; i++) v.s[i] = 0;
	};
	int at = x.j0 * KT + warp * FK;
	const int end = min(x.j1 * KT, vis);
	int id = id_at(at), id_next = id_at(at + KT);
	if (at < end) {
		load_keys(at, id);
		load_values(at, id);
	}
	for (; at < end; at += KT) {
		const bool all = at + FK <= least; // every row sees every key
		// ---- scores: keys as rows of the product ----
		float s[NT][4];
#pragma unroll
		for (int n = 0; n < NT; n++)
#pragma unroll
			for (int e = 0; e < 4; e++) s[n][e] = 0.f;
#pragma unroll
		for (int g = 0; g < KG; g++) {
			uint32_t h0[4], h1[4];
			codes4<WIDE>(k.w[0][g], h0);
			codes4<WIDE>(k.w[1][g], h1);
			const float d0 = g & 1 ? half_hi(k.s[0][g / 2]) : half_lo(k.s[0][g / 2]), d1 = g & 1 ? half_hi(k.s[1][g / 2]) : half_lo(k.s[1][g / 2]);
#pragma unroll
			for (int n = 0; n < NT; n++) {
				uint2 qa, qb;
				float2 from;
				if constexpr (IN_REGS) { qa = q[g * 2]; qb = q[g * 2 + 1]; from = init[g]; }
				else {
					qa = s_q[((n * KG + g) * 2) * 32 + lane];
					qb = s_q[((n * KG + g) * 2 + 1) * 32 + lane];
					from = *reinterpret_cast<const float2*>(s_init + (n * KG + g) * 8 + t * 2);
				}
				float c[4] = {from.x, from.y, from.x, from.y};
				mma16(c, h0[0], h1[0], h0[1], h1[1], qa.x, qa.y);
				mma16(c, h0[2], h1[2], h0[3], h1[3], qb.x, qb.y);
				s[n][0] = fmaf(c[0], d0, s[n][0]);
				s[n][1] = fmaf(c[1], d0, s[n][1]);
				s[n][2] = fmaf(c[2], d1, s[n][2]);
				s[n][3] = fmaf(c[3], d1, s[n][3]);
			}
		}
		id = id_next;
		load_keys(at + KT, id);
		id_next = id_at(at + 2 * KT);
		// ---- probabilities ----
		bool grow = false;
#pragma unroll
		for (int n = 0; n < NT; n++) {
			if constexpr (SPLIT && WIDE) // the rest of the queries has columns of its own
#pragma unroll
				for (int e = 0; e < 4; e++) s[n][e] += __shfl_xor_sync(0xffffffffu, s[n][e], 2);
			const float2 f = *reinterpret_cast<const float2*>(s_fac + n * 8 + t * 2);
#pragma unroll
			for (int e = 0; e < 4; e++) s[n][e] *= e & 1 ? f.y : f.x;
			if (!all) {
				const int2 lim = *reinterpret_cast<const int2*>(s_lim + n * 8 + t * 2);
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (at + u + (e >> 1) * 8 >= (e & 1 ? lim.y : lim.x)) s[n][e] = -INFINITY;
			}
			grow = grow || fmaxf(s[n][0], s[n][2]) - m[n][0] > 2.f || fmaxf(s[n][1], s[n][3]) - m[n][1] > 2.f; // false where both are -infinity
		}
		if (__any_sync(0xffffffffu, grow)) { // rare behind the first keys: probabilities may be up to 4
#pragma unroll
			for (int n = 0; n < NT; n++) {
				float f[2];
#pragma unroll
				for (int c = 0; c < 2; c++) {
					float top = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
					for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
					top = fmaxf(m[n][c], top);
					f[c] = m[n][c] == -INFINITY ? 0.f : exp2f(m[n][c] - top);
					m[n][c] = top;
					l[n][c] *= f[c];
#pragma unroll
					for (int i = 0; i < VG * 2; i++) { acc[i][n][c] *= f[c]; acc[i][n][c + 2] *= f[c]; }
				}
				const float fu = __shfl_sync(0xffffffffu, f[0], u >> 1), fv = __shfl_sync(0xffffffffu, f[1], u >> 1);
#pragma unroll
				for (int g = 0; g < VG; g++) part[n][g] *= u & 1 ? fv : fu;
			}
		}
		__syncwarp();
#pragma unroll
		for (int n = 0; n < NT; n++) {
			const float b0 = m[n][0] == -INFINITY ? 0.f : m[n][0], b1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
			for (int e = 0; e < 4; e++) {
				const float p = exp2f(s[n][e] - (e & 1 ? b1 : b0));
				l[n][e & 1] += p;
				sp[(n * 8 + t * 2 + (e & 1)) * FP + u + (e >> 1) * 8] = p;
			}
		}
		__syncwarp();
		// ---- sums: values' entries as rows of the product ----
#pragma unroll
		for (int n = 0; n < NT; n++) {
			uint32_t vs[2 * VG];
#pragma unroll
			for (int i = 0; i < 2 * VG; i++) vs[i] = v.s[i];
			if (!all) { // what the row does not see may have any scale, a NaN too
				const int lim = s_lim[n * 8 + u];
#pragma unroll
				for (int i = 0; i < 4; i++)
					if (at + t * 4 + i >= lim)
#pragma unroll
						for (int w = 0; w < VG / 2; w++) vs[i * (VG / 2) + w] = 0;
			}
			__half2 big = __float2half2_rn(0.f);
#pragma unroll
			for (int i = 0; i < 2 * VG; i++) {
				const uint32_t y = vs[i] & 0x7fff7fffu;
				big = __hmax2(big, *reinterpret_cast<const __half2*>(&y));
			}
			const float top = fmaxf(__low2float(big), __high2float(big));
			if (__any_sync(0xffffffffu, top > room[n])) {
				float y = fmaxf(top, room[n]);
				y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
				y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
				float f = 1.f;
				if (y > room[n]) {
					const int e = (__float_as_int(y) >> 23) - 127; // 2^e <= y < 2^(e + 1): scales up to twice that have room
					const float to = pow2(11 - e);
					f = to / mu[n];
					mu[n] = to;
					room[n] = pow2(min(e + 2, 127));
				}
				const float f0 = __shfl_sync(0xffffffffu, f, t * 8), f1 = __shfl_sync(0xffffffffu, f, t * 8 + 4);
#pragma unroll
				for (int i = 0; i < VG * 2; i++) { acc[i][n][0] *= f0; acc[i][n][2] *= f0; acc[i][n][1] *= f1; acc[i][n][3] *= f1; }
#pragma unroll
				for (int g = 0; g < VG; g++) part[n][g] *= f;
			}
			float4 p = *reinterpret_cast<const float4*>(sp + (n * 8 + u) * FP + t * 4);
			p.x *= mu[n]; p.y *= mu[n]; p.z *= mu[n]; p.w *= mu[n];
#pragma unroll
			for (int g = 0; g < VG; g++) {
				float y[4];
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const uint32_t w = vs[i * (VG / 2) + g / 2];
					y[i] = (i == 0 ? p.x : i == 1 ? p.y : i == 2 ? p.z : p.w) * (g & 1 ? half_hi(w) : half_lo(w));
				}
				if constexpr (!WIDE) part[n][g] += (y[0] + y[1]) + (y[2] + y[3]);
				const uint32_t hi0 = pack_half(y[0], y[1]), hi1 = pack_half(y[2], y[3]);
				const uint32_t lo0 = pack_half(y[0] - half_lo(hi0), y[1] - half_hi(hi0)), lo1 = pack_half(y[2] - half_lo(hi1), y[3] - half_hi(hi1));
				const uint32_t sel = g & 1 ? 0x7632 : 0x5410;
				uint32_t ab[4], cd[4];
				codes4<WIDE>(__byte_perm(v.w[0][g / 2], v.w[1][g / 2], sel), ab);
				codes4<WIDE>(__byte_perm(v.w[2][g / 2], v.w[3][g / 2], sel), cd);
#pragma unroll
				for (int i = 0; i < 2; i++) {
					if constexpr (SPLIT) mma16(acc[g * 2 + i][n], ab[2 * i], ab[2 * i + 1], cd[2 * i], cd[2 * i + 1], u < 4 ? hi0 : lo0, u < 4 ? hi1 : lo1);
					else {
						mma16(acc[g * 2 + i][n], ab[2 * i], ab[2 * i + 1], cd[2 * i], cd[2 * i + 1], hi0, hi1);
						mma16(acc[g * 2 + i][n], ab[2 * i], ab[2 * i + 1], cd[2 * i], cd[2 * i + 1], lo0, lo1);
					}
				}
			}
		}
		load_values(at + KT, id);
	}
	// ---- this warp's maxima, sums and rows ----
#pragma unroll
	for (int n = 0; n < NT; n++) {
#pragma unroll
		for (int c = 0; c < 2; c++)
#pragma unroll
			for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
		const float inv = 1.f / mu[n]; // a power of two
		const float i0 = __shfl_sync(0xffffffffu, inv, t * 8), i1 = __shfl_sync(0xffffffffu, inv, t * 8 + 4);
		const int row = SPLIT ? n * 4 + t * 2 : n * 8 + t * 2;
		const bool mine = (!SPLIT || t < 2) && row < most_rows;
		if (mine && u == 0) {
			s_ml[warp * most_rows + row] = make_float2(m[n][0], l[n][0]);
			s_ml[warp * most_rows + row + 1] = make_float2(m[n][1], l[n][1]);
		}
#pragma unroll
		for (int g = 0; g < VG; g++) {
			float z = part[n][g];
			z += __shfl_xor_sync(0xffffffffu, z, 1);
			z += __shfl_xor_sync(0xffffffffu, z, 2);
			const float z0 = __shfl_sync(0xffffffffu, z, t * 8), z1 = __shfl_sync(0xffffffffu, z, t * 8 + 4);
			float y[2][4]; // the row's entries 4 u .. 4 u + 3 of the block
#pragma unroll
			for (int c = 0; c < 2; c++) {
				y[c][0] = acc[g * 2][n][c];
				y[c][1] = acc[g * 2][n][c + 2];
				y[c][2] = acc[g * 2 + 1][n][c];
				y[c][3] = acc[g * 2 + 1][n][c + 2];
#pragma unroll
				for (int e = 0; e < 4; e++) {
					if constexpr (SPLIT) y[c][e] += __shfl_xor_sync(0xffffffffu, y[c][e], 2);
					if constexpr (!WIDE) y[c][e] = y[c][e] * 1048576.f - 8.f * (c ? z1 : z0); // codes were taken as 2^-20 each
					y[c][e] *= c ? i1 : i0;
				}
			}
			if (mine) {
				*reinterpret_cast<float4*>(s_o + (warp * most_rows + row) * op + g * 32 + u * 4) = make_float4(y[0][0], y[0][1], y[0][2], y[0][3]);
				*reinterpret_cast<float4*>(s_o + (warp * most_rows + row + 1) * op + g * 32 + u * 4) = make_float4(y[1][0], y[1][1], y[1][2], y[1][3]);
			}
		}
	}
}

template <int KG, int VG, int KIND>
__global__ void __launch_bounds__(FT, KIND == FEW && VG < 8 ? 3 : 2) paged4_attn_kernel(const __grid_constant__ Attn a, const __grid_constant__ Part part, const Pool4 pool, const int type) {
	using Z = Size4<KG, VG, KIND>;
	constexpr int M = Z::M, OP = Z::OP, TILE = KIND == F32 ? 4 : 8; // rows of a tile of columns
	extern __shared__ __align__(16) uint8_t smem[];
	uint2* s_q = reinterpret_cast<uint2*>(smem);                       // [NT][KG][2][32]: queries as the product wants them
	float* s_init = reinterpret_cast<float*>(s_q + Z::NT * KG * 2 * 32); // [NT][KG][8]: -8 times the sum of a block's queries
	float* s_o = s_init + Z::NT * KG * 8;                              // [FW][M][OP]
	float* s_p = s_o + Z::SUMS;                                        // [FW][NT * 8][FP]
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
		const bool split = KIND == F32 || (KIND == FEW && rows <= 4);
		const int per = split ? 4 : 8, tiles = (rows + per - 1) / per;
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
			const int e0 = (__float_as_int(top) >> 23) - 127, e = e0 == 128 ? 0 : min(14 - e0, 127);
			const float f = pow2(e);
			if (t == 0) s_fac[n * 8 + u] = fminf(fmaxf(a.scale * 1.4426950408889634f * pow2(12 - e) * (KIND == F32 ? 1.f / 4096.f : 256.f), -3.0e38f), 3.0e38f);
#pragma unroll
			for (int g = 0; g < KG; g++) {
				float z[8];
#pragma unroll
				for (int i = 0; i < 8; i++) {
					const float full = y[g][i] * f;
					float h = __half2float(__float2half_rn(full));
					if (KIND == F32 && u >= 4) h = full - h; // the rest
					z[i] = h;
				}
				const uint2 qa = make_uint2(pack_half(z[0], z[4]), pack_half(z[1], z[5])), qb = make_uint2(pack_half(z[2], z[6]), pack_half(z[3], z[7]));
				s_q[((n * KG + g) * 2) * 32 + lane] = qa;
				s_q[((n * KG + g) * 2 + 1) * 32 + lane] = qb;
				float sum = ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
				sum += __shfl_xor_sync(0xffffffffu, sum, 1);
				sum += __shfl_xor_sync(0xffffffffu, sum, 2);
				if (t == 0) s_init[(n * KG + g) * 8 + u] = KIND == F32 ? 0.f : sum * -7.62939453125e-6f; // 8 codes of 2^-20
			}
		}
		__syncthreads();
		const int vis = keys_of(rows - 1), least = keys_of(0); // the last row sees the most
		float* sp = s_p + warp * Z::NT * 8 * FP;
		if constexpr (KIND == F32) {
			if (tiles == 1) piece4<KG, VG, 1, true, true>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
			else if (tiles == 2) piece4<KG, VG, 2, true, true>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
			else if constexpr (Z::NT == 4) piece4<KG, VG, 4, true, true>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
		} else if constexpr (KIND == FEW) {
			if (split) piece4<KG, VG, 1, true, false>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
			else if (tiles == 1) piece4<KG, VG, 1, false, false>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
			else piece4<KG, VG, 2, false, false>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
		} else piece4<KG, VG, Z::NT, false, false>(a, pool, x, vis, least, s_q, s_init, s_fac, s_lim, sp, s_o, s_ml, OP, M);
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
				const float4 o = *reinterpret_cast<const float4*>(s_o + (e * M + row) * OP + col);
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
	if (Z::NT == 0) return Shape4{0, 0};
	const size_t smem = Z::own + plan_bytes(b.B, b.n_groups);
	const int most = KIND == FEW && VG < 8 ? 3 : 2;
	return Shape4{Z::M, std::max(1, std::min(most, (int) (226 * 1024 / (smem + 1024))))};
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
Shape4 attn4_few(const Pool4& p, const BatchView& b) { return shape4<FEW>(p, b); }
Shape4 attn4_many(const Pool4& p, const BatchView& b) { return shape4<MANY>(p, b); }
Shape4 attn4_f32(const Pool4& p, const BatchView& b) { return shape4<F32>(p, b); }

template <int KG, int VG, int KIND>
static int launch_kind(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	if constexpr (Size4<KG, VG, KIND>::NT > 0) {
		const size_t smem = Size4<KG, VG, KIND>::own + plan_bytes(a.b.B, a.b.n_groups);
		XALM_CUDA_CHECK(allow_smem((const void*) paged4_attn_kernel<KG, VG, KIND>));
		XALM_CUDA_CHECK(launch(paged4_attn_kernel<KG, VG, KIND>, a.part[part].grid, FT, smem, s, part > 0, a, a.part[part], p, type));
	}
	return XALM_OK;
}
int launch_attn4(const Attn& a, const Pool4& p, int part, int type, bool many, cudaStream_t s) {
	switch (p.kg * 16 + p.vg) {
#define XALM_PAGED4(K, V) \
	case K * 16 + V: return type == XALM_F32 ? launch_kind<K, V, F32>(a, p, part, type, s) : many ? launch_kind<K, V, MANY>(a, p, part, type, s) : launch_kind<K, V, FEW>(a, p, part, type, s);
		XALM_PAGED4(2, 2) XALM_PAGED4(2, 4) XALM_PAGED4(2, 8) XALM_PAGED4(4, 2) XALM_PAGED4(4, 4) XALM_PAGED4(4, 8) XALM_PAGED4(8, 2) XALM_PAGED4(8, 4) XALM_PAGED4(8, 8)
#undef XALM_PAGED4
	}
	return set_error(XALM_ERR_INVALID, "paged attention: %d and %d blocks", p.kg, p.vg);
}

} // namespace paged
} // namespace xalm
