// paged4_tile.cu — attention over paged caches of 4-bit numbers (paged4.cuh) for many rows: prompts, and groups of sequences over their shared pages.
#include <algorithm>
#include <type_traits>

#include "paged4.cuh"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// As in paged4_attn.cu, but 128 (token, head) rows to a unit, 16 to a warp, so that codes are taken apart once for all of them: the CTA turns a tile of 64 keys and values into fp16 numbers
// c - 8 in shared memory, while the tile before enters the products.  Scores by m16n8k16 with the rows as A, block by block, times the keys' scales in fp32; probabilities become A of the second
// product where they are, times the values' scales in fp32: what a row does not see may then have any scale, a NaN too, and is left out.
// p d is rounded once, to one fp16 number for bf16 results, to two in turn for fp16, whose own rounding one would add to: five prompts of fp16 take 580 us with two, 456 with one, whose results have 1.31
// times the root mean square error.  p is 2^lift times as large, so that the largest scale that its row has seen times 4 has room in p d, and small ones beside it keep their bits.  (With p rounded to
// fp16 too and the scales multiplied as pairs, 433 us, but 1.56 times the error, and sums of small scales lost; with d (c - 8) rounded to fp16 for the first product 15 % less time, but the logarithms
// of the denominators are off by 1e-5.)
// Bound by latency: with 255 registers to a thread an SM has eight warps, whose products keep the tensor pipe busy for a third of the time; one half of the warps converts the next tile before its
// products, the other behind them.  Five prompts of 150 to 700 tokens behind 1000 to 3000 take 456 us of bf16 (173 TFLOP/s), 64 tokens behind 8192 in common and up to 1500 alone 95.
// 12 warps of 168 registers, half a tile at a time, were 4 % quicker for prompts and a third slower for 128 tokens of two texts, since units of 192 rows are filled less often.
// =========================================================================================================================================
constexpr int GT = 256, GW = GT / 32, GM = GW * 16; // threads, warps, rows of a unit
constexpr int RING = 3;                             // tiles on their way or waiting as they come

template <int KG, int VG>
struct Tile4 {
	static constexpr int RAW = KT * (KG + VG) * 18, KH = KT * KG * 64, VH = KT * VG * 64; // bytes of a tile as it comes, of its keys and values as fp16
	static constexpr int VD = KT / 2 * VG * 8, KD = KT / 2 * KG * 8;                       // and of its values' scales, by pairs of keys, and its keys', in fp32
	static constexpr int QH = GM * KG * 64;                                                // of the queries
	static constexpr size_t own = (size_t) RING * RAW + 2 * (KH + VH + VD + KD) + QH + 2 * KT * 4 + 2 * 4 + 2 * GM * 4 + 24;
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
__device__ __forceinline__ void matrices(uint32_t at, uint32_t (&r)[4]) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void matrices_turned(uint32_t at, uint32_t (&r)[4]) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void copy16_if(uint32_t dst, const uint8_t* src, bool there) { // zeros where there is nothing
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
	uint32_t r;
	asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}
__device__ __forceinline__ uint32_t bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 halves(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ float ex2(float x) {
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}
// s f - m: in one step where that is off by less than 2^-6 from the rounded product, which m is one of; else in two, so that the largest score is 0 above itself
constexpr float COARSE = 262144.f;
__device__ __forceinline__ float above(float s, float f, float m, bool coarse) { return coarse ? __fsub_rn(__fmul_rn(s, f), m) : fmaf(s, f, -m); }
__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }
// A word's codes, c - 8, in the order 0 4 1 5 2 6 3 7: 1024 + c and 1024 + 16 c as they lie, brought there without a rounding
__device__ __forceinline__ void numbers(uint32_t w, __half2 (&h)[4]) {
	const uint32_t w8 = w >> 8;
#pragma unroll
	for (int i = 0; i < 4; i++) {
		const uint32_t x = ((i < 2 ? w : w8) & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
		h[i] = __hfma2(halves(x), __float2half2_rn(i & 1 ? 0.0625f : 1.f), __float2half2_rn(i & 1 ? -72.f : -1032.f));
	}
}

// TWO: p d in two parts, for fp16 results
template <int KG, int VG, bool TWO>
__global__ void __launch_bounds__(GT, 1) paged4_tile_kernel(const __grid_constant__ Attn a, const __grid_constant__ Part part, const Pool4 pool, const int type) {
	using Z = Tile4<KG, VG>;
	extern __shared__ __align__(128) uint8_t smem[];
	uint8_t* s_raw = smem;                                         // [RING][RAW]: key codes, value codes, key scales, value scales
	uint8_t* s_k = s_raw + RING * Z::RAW;                          // [2][KT][KG * 32] fp16, 16 bytes c of key j at c ^ (j & 7)
	uint8_t* s_v = s_k + 2 * Z::KH;                                // [2][KT][VG * 32], likewise
	uint8_t* s_vd = s_v + 2 * Z::VH;                               // [2][KT / 2][VG] pairs of values' scales in fp32
	uint8_t* s_kd = s_vd + 2 * Z::VD;                              // [2][KT / 2][KG] of keys'
	uint8_t* s_q = s_kd + 2 * Z::KD;                               // [GM][KG * 32], as the keys
	float* s_top = reinterpret_cast<float*>(s_q + Z::QH);          // [2][KT]: each value's largest scale
	float* s_most = s_top + 2 * KT;                                // [2]: the tile's
	int* s_lim = reinterpret_cast<int*>(s_most + 2);               // [GM]: keys that a row sees
	float* s_fac = reinterpret_cast<float*>(s_lim + GM);           // [GM]: from a product to a score in units of log2
	uint8_t* s_plan = reinterpret_cast<uint8_t*>(s_fac + GM);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, u = lane >> 2, t = lane & 3, dv = a.c.dv, P = 1 << a.c.shift, shift = a.c.shift;
	Plan plan;
	pdl_launch_dependents();
	make_plan<GT>(a, part, s_plan, plan);
	Walk k;
	bool more = walk_begin(a, part, plan, k);
	if (tid == 0) write_head(a, part, k, more, more && k.x.seg >= a.b.n_groups && k.x.key0 == 0, plan.share);
	const uint32_t raw = smem_u32(s_raw), kh = smem_u32(s_k), vh = smem_u32(s_v);
	for (; more; more = walk_next(a, part, plan, k)) {
		const Piece& x = k.x;
		if (x.j0 == x.j1) continue; // the same for every thread
		const int shared = plan.shs[x.s];
		const bool prefix = x.seg < a.b.n_groups;
		const int rows = min(GM, x.rows - x.t * GM), h0 = x.g * a.rep;
		auto keys_of = [&](int r) { return prefix ? shared : own_keys(x.q, shared, a.rep, x.t * GM + r); };
		__syncthreads(); // the piece before has been read
		if (tid < GM) s_lim[tid] = tid < rows ? keys_of(tid) : 0;
		const int vis = keys_of(rows - 1), first = x.j0 * KT, n_tiles = max(min(x.j1, (vis + KT - 1) / KT) - x.j0, 0);
		// ---- copies: 16 bytes of codes of a key and of a value to a thread, and of scales to some ----
		const int* table = a.b.table + (long long) x.s * a.b.table_row;
		const uint8_t* head = pool.at + x.g * pool.head;
		constexpr int KC = KT * KG / 8, VC = KT * VG / 8; // 16 bytes of scales
		// this thread's keys of a tile: of its 16 bytes of a key's codes, of a value's, of scales (16 bytes are several keys', all of one page)
		const int j_k = tid / KG, j_v = tid / VG, j_s = tid < KC ? tid * (8 / KG) : (tid - KC) * (8 / VG);
		auto id_at = [&](int i, int j) { return i < n_tiles ? table[(x.key0 + min(first + i * KT + j, vis - 1)) >> shift] : 0; };
		int id_k = id_at(0, j_k & (KT - 1)), id_v = KG == VG ? 0 : id_at(0, j_v & (KT - 1)), id_s = id_at(0, j_s & (KT - 1)); // looked at a tile ahead
		auto copy = [&](int i) {
			if (i < n_tiles) {
				const uint32_t to = raw + i % RING * Z::RAW;
				const int at = first + i * KT;
				auto run_of = [&](int j, int id, bool& there) {
					const bool good = (unsigned) id < (unsigned) a.c.pages;
					if (!good) report(a.c, ERR_PAGE); // reads as zeros
					there = good && at + j < vis;
					return head + (good ? id : 0) * pool.page;
				};
				bool there;
				if (KG == 4 || tid < KT * KG) { // 16 bytes c of key j at c ^ (j / 2 & 3) where a key has four: a quarter of a warp reads the same c of eight keys
					const int j = j_k, c = tid % KG, slot = (x.key0 + at + j) & (P - 1);
					const uint8_t* run = run_of(j, id_k, there);
					copy16_if(to + j * (KG * 16) + (KG == 4 ? c ^ (j >> 1 & 3) : c) * 16, run + slot * (KG * 16) + c * 16, there);
					if constexpr (KG == VG) copy16_if(to + KT * KG * 16 + j * (VG * 16) + (VG == 4 ? c ^ (j >> 1 & 3) : c) * 16, run + values_at(KG, shift) + slot * (VG * 16) + c * 16, there);
				}
				if constexpr (KG != VG)
					if (VG == 4 || tid < KT * VG) {
						const int j = j_v, c = tid % VG, slot = (x.key0 + at + j) & (P - 1);
						const uint8_t* run = run_of(j, id_v, there);
						copy16_if(to + KT * KG * 16 + j * (VG * 16) + (VG == 4 ? c ^ (j >> 1 & 3) : c) * 16, run + values_at(KG, shift) + slot * (VG * 16) + c * 16, there);
					}
				if (tid < KC + VC) {
					const bool value = tid >= KC;
					const int j = j_s, slot = (x.key0 + at + j) & (P - 1);
					const uint8_t* run = run_of(j, id_s, there);
					copy16_if(to + KT * (KG + VG) * 16 + tid * 16, run + (value ? value_scales_at(KG, VG, shift) + slot * (VG * 2) : key_scales_at(KG, shift) + slot * (KG * 2)), there);
				}
				id_k = id_at(i + 1, j_k & (KT - 1));
				if constexpr (KG != VG) id_v = id_at(i + 1, j_v & (KT - 1));
				if (tid < KC + VC) id_s = id_at(i + 1, j_s & (KT - 1));
			}
			asm volatile("cp.async.commit_group;" ::: "memory");
		};
		// ---- a tile as fp16: a fourth of a key and of a value to a thread ----
		auto convert = [&](int i) {
			const uint8_t* from = s_raw + i % RING * Z::RAW;
			const int b = i & 1, j = tid & (KT - 1), c = tid / KT;
			const uint32_t to_k = kh + b * Z::KH + j * (KG * 64), to_v = vh + b * Z::VH + j * (VG * 64);
			uint32_t w[KG], v[VG];
			if constexpr (KG == 4) {
				const uint4 y = *reinterpret_cast<const uint4*>(from + j * 64 + (c ^ (j >> 1 & 3)) * 16);
				w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w;
			} else {
				const uint2 y = *reinterpret_cast<const uint2*>(from + j * 32 + c * 8);
				w[0] = y.x; w[1] = y.y;
			}
			auto store = [&](uint32_t to, uint32_t word) {
				__half2 h[4];
				numbers(word, h);
				asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(bits(h[0])), "r"(bits(h[1])), "r"(bits(h[2])), "r"(bits(h[3])) : "memory");
			};
#pragma unroll
			for (int g = 0; g < KG; g++) store(to_k + (((g * 4 + c) ^ (j & 7)) * 16), w[g]);
			// entries 8 c .. 8 c + 7 of a value's block: 16 bits each at places 2 c and 2 c + 1
			if constexpr (VG == 4) {
				const uint4 y = *reinterpret_cast<const uint4*>(from + KT * KG * 16 + j * 64 + (c ^ (j >> 1 & 3)) * 16);
				v[0] = __byte_perm(y.x, y.z, 0x5410); v[1] = __byte_perm(y.x, y.z, 0x7632);
				v[2] = __byte_perm(y.y, y.w, 0x5410); v[3] = __byte_perm(y.y, y.w, 0x7632);
			} else {
				const uint2 y = *reinterpret_cast<const uint2*>(from + KT * KG * 16 + j * 32 + c * 8);
				v[0] = __byte_perm(y.x, y.y, 0x5410); v[1] = __byte_perm(y.x, y.y, 0x7632);
			}
#pragma unroll
			for (int g = 0; g < VG; g++) store(to_v + (((g * 4 + c) ^ (j & 7)) * 16), v[g]);
			if (warp == GW - 2) { // keys' scales, two keys to a lane
				const uint8_t* s = from + KT * (KG + VG) * 16 + lane * (KG * 4);
#pragma unroll
				for (int z = 0; z < KG / 2; z++) {
					const float2 y0 = __half22float2(*reinterpret_cast<const __half2*>(s + z * 4)), y1 = __half22float2(*reinterpret_cast<const __half2*>(s + KG * 2 + z * 4));
					*reinterpret_cast<float4*>(s_kd + b * Z::KD + (lane * KG + z * 2) * 8) = make_float4(y0.x, y1.x, y0.y, y1.y);
				}
			}
			if (warp == GW - 1) { // values' scales, two keys to a lane
				const uint8_t* s = from + KT * (KG + VG) * 16 + KT * KG * 2 + lane * (VG * 4);
				uint32_t e[2][VG / 2];
#pragma unroll
				for (int y = 0; y < 2; y++)
#pragma unroll
					for (int z = 0; z < VG / 2; z++) e[y][z] = *reinterpret_cast<const uint32_t*>(s + y * (VG * 2) + z * 4);
				float top[2];
#pragma unroll
				for (int y = 0; y < 2; y++) {
					__half2 m = __habs2(halves(e[y][0]));
#pragma unroll
					for (int z = 1; z < VG / 2; z++) m = __hmax2(m, __habs2(halves(e[y][z])));
					top[y] = fmaxf(__low2float(m), __high2float(m)); // NaN counts for nothing
				}
#pragma unroll
				for (int z = 0; z < VG / 2; z++) {
					const float2 y0 = __half22float2(halves(e[0][z])), y1 = __half22float2(halves(e[1][z]));
					*reinterpret_cast<float4*>(s_vd + b * Z::VD + (lane * VG + z * 2) * 8) = make_float4(y0.x, y1.x, y0.y, y1.y);
				}
				*reinterpret_cast<float2*>(s_top + b * KT + lane * 2) = make_float2(top[0], top[1]);
				const float all = warp_max(fmaxf(fmaxf(top[0], top[1]), 0.f));
				if (lane == 0) s_most[b] = all;
			}
		};
		copy(0);
		copy(1);
		copy(2);
		// ---- queries, each warp its own rows: eight entries to a lane, in the order of the keys' ----
		constexpr int QL = KG * 4; // lanes to a row
#pragma unroll 2
		for (int i = 0; i < 16; i += 32 / QL) {
			const int r = warp * 16 + i + lane / QL, c = lane % QL, w = x.t * GM + r;
			float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, top = 0.f;
			if (r < rows && c * 8 < a.c.d) {
				const long long at = (long long) (x.row0 + w / a.rep) * a.q_row + (h0 + w % a.rep) * a.c.d + c * 8;
				if (type == XALM_F16) load8(reinterpret_cast<const __half*>(a.q) + at, y);
				else load8(reinterpret_cast<const __nv_bfloat16*>(a.q) + at, y);
			}
#pragma unroll
			for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(y[e]));
#pragma unroll
			for (int o = 1; o < QL; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
			// the row times a power of two, so that its largest entry is between 2^14 and 2^15
			const int e0 = (__float_as_int(top) >> 23) - 127, e = e0 == 128 ? 0 : min(14 - e0, 126);
			const float f = e0 == 128 ? NAN : a.scale < 0.f ? -two_to(e) : two_to(e); // a negative scale turns the queries' signs; a row with an infinity is no number, whatever the keys' signs
			if (c == 0) s_fac[r] = fminf(fmaxf(fabsf(a.scale) * 1.4426950408889634f * two_to(-e), 1e-30f), 3.0e38f); // not 0: 0 times an infinity is no number
			*reinterpret_cast<uint4*>(s_q + r * (KG * 64) + ((c ^ (r & 7)) * 16)) =
				make_uint4(pack2(y[0] * f, y[4] * f), pack2(y[1] * f, y[5] * f), pack2(y[2] * f, y[6] * f), pack2(y[3] * f, y[7] * f));
		}
		__syncwarp();
		float fac[2], m[2], l[2], lift[2], room[2]; // p is 2^lift times as large, so that the largest scale that the row has seen is 2^11 to 2^12 in p d
		int lim[2];
		bool coarse = false;
		const int r0 = warp * 16 + u;
#pragma unroll
		for (int half = 0; half < 2; half++) {
			fac[half] = s_fac[r0 + half * 8];
			m[half] = -3.0e38f;
			l[half] = 0.f;
			lift[half] = 0.f;
			room[half] = 0.f;
		}
		const uint32_t q_at = smem_u32(s_q) + (warp * 16 + (lane & 15)) * (KG * 64);
		float acc[VG * 4][4];
#pragma unroll
		for (int c = 0; c < VG * 4; c++)
#pragma unroll
			for (int e = 0; e < 4; e++) acc[c][e] = 0.f;
		asm volatile("cp.async.wait_group 2;" ::: "memory");
		__syncthreads();
		lim[0] = s_lim[r0];
		lim[1] = s_lim[r0 + 8];
		const int least = s_lim[warp * 16], most = warp * 16 < rows ? s_lim[min(warp * 16 + 15, rows - 1)] : 0; // of this warp's rows
		if (n_tiles) convert(0);
		asm volatile("cp.async.wait_group 1;" ::: "memory");
		__syncthreads();
		auto compute = [&](int i, auto edge) { // false: to be done again, as an edge
			constexpr bool EDGE = decltype(edge)::value; // some rows may not see some keys, or scores are large
			const int b = i & 1, at = first + i * KT;
			// ---- scores ----
			float s[KT / 8][4];
#pragma unroll
			for (int c = 0; c < KG; c++) {
				uint32_t q[2][4];
#pragma unroll
				for (int e = 0; e < 2; e++) matrices(q_at + (((c * 4 + e * 2 + (lane >> 4)) ^ (lane & 7)) * 16), q[e]);
#pragma unroll
				for (int n = 0; n < KT / 8; n += 4) { // a block of four times eight keys, then their scales
					uint32_t r[4][4];
					float y[4][4];
#pragma unroll
					for (int i = 0; i < 4; i++) matrices(kh + b * Z::KH + ((n + i) * 8 + (lane & 7)) * (KG * 64) + (((c * 4 + (lane >> 3)) ^ (lane & 7)) * 16), r[i]);
#pragma unroll
					for (int i = 0; i < 4; i++) mma16_new(y[i], q[0][0], q[0][1], q[0][2], q[0][3], r[i][0], r[i][1]);
#pragma unroll
					for (int i = 0; i < 4; i++) mma16(y[i], q[1][0], q[1][1], q[1][2], q[1][3], r[i][2], r[i][3]);
#pragma unroll
					for (int i = 0; i < 4; i++) {
						const float2 d = *reinterpret_cast<const float2*>(s_kd + b * Z::KD + (((n + i) * 4 + t) * KG + c) * 8);
#pragma unroll
						for (int e = 0; e < 4; e++) s[n + i][e] = c ? fmaf(y[i][e], e & 1 ? d.y : d.x, s[n + i][e]) : y[i][e] * (e & 1 ? d.y : d.x);
					}
				}
			}
			// ---- the largest scale that a row has seen ----
			float top[2];
			top[0] = top[1] = s_most[b];
			if constexpr (EDGE) {
				top[0] = top[1] = 0.f;
#pragma unroll
				for (int n = 0; n < KT / 8; n++) {
					const float2 y = *reinterpret_cast<const float2*>(s_top + b * KT + n * 8 + t * 2);
#pragma unroll
					for (int h = 0; h < 2; h++) {
						if (at + n * 8 + t * 2 < lim[h]) top[h] = fmaxf(top[h], y.x);
						if (at + n * 8 + t * 2 + 1 < lim[h]) top[h] = fmaxf(top[h], y.y);
					}
				}
#pragma unroll
				for (int h = 0; h < 2; h++) {
					top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
					top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
				}
			}
			if (__any_sync(0xffffffffu, top[0] > room[0] || top[1] > room[1])) {
#pragma unroll
				for (int h = 0; h < 2; h++)
					if (top[h] > room[h]) {
						const int e = (__float_as_int(top[h]) >> 23) - 127; // 2^e <= top < 2^(e + 1): scales up to twice that have room
						const float to = (float) max(11 - e, -4), f = exp2f(to - lift[h]); // -4 for the largest finite scale, 35 for the smallest
						room[h] = two_to(min(e + 2, 127));
						l[h] *= f;
						lift[h] = to;
#pragma unroll
						for (int c = 0; c < VG * 4; c++) { acc[c][h * 2] *= f; acc[c][h * 2 + 1] *= f; }
					}
			}
			// ---- probabilities ----
			float big[2] = {-INFINITY, -INFINITY};
#pragma unroll
			for (int n = 0; n < KT / 8; n++)
#pragma unroll
				for (int e = 0; e < 4; e++) {
					if (EDGE && at + n * 8 + t * 2 + (e & 1) >= lim[e >> 1]) s[n][e] = -INFINITY;
					big[e >> 1] = fmaxf(big[e >> 1], s[n][e]);
				}
			if (__any_sync(0xffffffffu, above(big[0], fac[0], m[0], EDGE && coarse) > 2.f || above(big[1], fac[1], m[1], EDGE && coarse) > 2.f)) { // rare behind the first keys: probabilities may be up to 4
#pragma unroll
				for (int h = 0; h < 2; h++) {
					float y = big[h];
					y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
					y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
					y = fmaxf(m[h], __fmul_rn(y, fac[h]));
					coarse = coarse || (fabsf(y) > COARSE && y != -3.0e38f);
					const float f = exp2f(m[h] - y);
					m[h] = y;
					l[h] *= f;
#pragma unroll
					for (int c = 0; c < VG * 4; c++) { acc[c][h * 2] *= f; acc[c][h * 2 + 1] *= f; }
				}
				coarse = __any_sync(0xffffffffu, coarse);
				if (!EDGE && coarse) return false;
			}
			const float ml[2] = {m[0] - lift[0], m[1] - lift[1]};
			if (EDGE && coarse)
#pragma unroll
				for (int n = 0; n < KT / 8; n++)
#pragma unroll
					for (int e = 0; e < 4; e++) s[n][e] = __fsub_rn(__fmul_rn(s[n][e], fac[e >> 1]), m[e >> 1]) + lift[e >> 1];
#pragma unroll
			for (int n = 0; n < KT / 8; n++)
#pragma unroll
				for (int h = 0; h < 2; h++) {
					s[n][h * 2] = ex2(EDGE && coarse ? s[n][h * 2] : fmaf(s[n][h * 2], fac[h], -ml[h]));
					s[n][h * 2 + 1] = ex2(EDGE && coarse ? s[n][h * 2 + 1] : fmaf(s[n][h * 2 + 1], fac[h], -ml[h]));
					l[h] += s[n][h * 2] + s[n][h * 2 + 1];
				}
			// ---- sums ----
#pragma unroll
			for (int kk = 0; kk < KT / 16; kk++) {
				uint32_t seen[4];
				if constexpr (EDGE) {
#pragma unroll
					for (int e = 0; e < 4; e++) { // as the product's parts: rows u, u + 8 of the first eight keys, of the second
						const int key = at + kk * 16 + (e >> 1) * 8 + t * 2;
						seen[e] = (key < lim[e & 1] ? 0xffffu : 0u) | (key + 1 < lim[e & 1] ? 0xffff0000u : 0u);
					}
				}
				const uint32_t row = vh + b * Z::VH + (kk * 16 + (lane & 15)) * (VG * 64);
#pragma unroll
				for (int g = 0; g < VG; g++) {
					// scales of keys 2 t, 2 t + 1 and 8 behind them
					const float2 d0 = *reinterpret_cast<const float2*>(s_vd + b * Z::VD + ((kk * 8 + t) * VG + g) * 8), d1 = *reinterpret_cast<const float2*>(s_vd + b * Z::VD + ((kk * 8 + 4 + t) * VG + g) * 8);
					const float *p0 = s[kk * 2], *p1 = s[kk * 2 + 1];
					const float2 y[4] = {make_float2(p0[0] * d0.x, p0[1] * d0.y), make_float2(p0[2] * d0.x, p0[3] * d0.y), make_float2(p1[0] * d1.x, p1[1] * d1.y), make_float2(p1[2] * d1.x, p1[3] * d1.y)};
					uint32_t f[4];
					[[maybe_unused]] uint32_t rest[4];
#pragma unroll
					for (int e = 0; e < 4; e++) {
						f[e] = pack2(y[e].x, y[e].y);
						if constexpr (TWO) rest[e] = pack2(y[e].x - __low2float(halves(f[e])), y[e].y - __high2float(halves(f[e])));
						if constexpr (EDGE) {
							f[e] &= seen[e];
							if constexpr (TWO) rest[e] &= seen[e];
						}
					}
#pragma unroll
					for (int c = 0; c < 4; c += 2) {
						uint32_t r[4];
						matrices_turned(row + (((g * 4 + c + (lane >> 4)) ^ (lane & 7)) * 16), r);
						mma16(acc[g * 4 + c], f[0], f[1], f[2], f[3], r[0], r[1]);
						mma16(acc[g * 4 + c + 1], f[0], f[1], f[2], f[3], r[2], r[3]);
						if constexpr (TWO) {
							mma16(acc[g * 4 + c], rest[0], rest[1], rest[2], rest[3], r[0], r[1]);
							mma16(acc[g * 4 + c + 1], rest[0], rest[1], rest[2], rest[3], r[2], r[3]);
						}
					}
				}
			}
			return true;
		};
		for (int i = 0; i < n_tiles; i++) {
			copy(i + RING);
			const int at = first + i * KT;
			if (warp < GW / 2 && i + 1 < n_tiles) convert(i + 1); // the halves in turn: one's products beside the other's conversion
			if (at < most && (coarse || at + KT > least || !compute(i, std::false_type()))) compute(i, std::true_type());
			if (warp >= GW / 2 && i + 1 < n_tiles) convert(i + 1);
			asm volatile("cp.async.wait_group 1;" ::: "memory");
			__syncthreads();
		}
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		// ---- results: two neighbouring entries to a lane, which its neighbour has one of ----
		const bool direct = x.j0 == 0 && x.j1 == x.w && !prefix && shared == 0;
		const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
#pragma unroll
		for (int h = 0; h < 2; h++) {
			float sum = l[h];
			sum += __shfl_xor_sync(0xffffffffu, sum, 1);
			sum += __shfl_xor_sync(0xffffffffu, sum, 2);
			const int r = r0 + h * 8, w = x.t * GM + r;
			const bool any = sum > 0.f || sum != sum, there = r < rows;
			const float down = two_to(-(int) lift[h]), f = direct ? any ? 1.f / sum : 0.f : down;
			const long long tok = x.row0 + w / a.rep;
			const int hd = h0 + w % a.rep;
			if (there && t == 0) {
				const float top = m[h] == -3.0e38f ? -INFINITY : m[h];
				if (!direct) {
					if (slot < part.slots) part.ml[slot * GM + r] = make_float2(top, sum * down);
				} else if (a.lse) a.lse[tok * a.H + hd] = any ? (top + log2f(sum * down)) * 0.6931471805599453f : -INFINITY;
			}
#pragma unroll
			for (int c = 0; c < VG * 4; c++) {
				const float y0 = acc[c][h * 2] * f, y1 = acc[c][h * 2 + 1] * f, other = __shfl_xor_sync(0xffffffffu, t & 1 ? y0 : y1, 1);
				const int col = c * 8 + (t & 1 ? t + 3 : t);
				const float2 y = t & 1 ? make_float2(other, y1) : make_float2(y0, other);
				if (!there || c * 8 >= dv) continue;
				if (!direct) {
					if (slot < part.slots) *reinterpret_cast<float2*>(part.o + (slot * GM + r) * dv + col) = y;
				} else if (type == XALM_F16) *reinterpret_cast<uint32_t*>(reinterpret_cast<__half*>(a.out) + tok * a.out_row + hd * dv + col) = pack2(y.x, y.y);
				else *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(a.out) + tok * a.out_row + hd * dv + col) = __floats2bfloat162_rn(y.x, y.y);
			}
		}
	}
	pdl_wait(); // not ahead of the kernel before it to the join
}

template <int KG, int VG, bool TWO>
static int launch_parts(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	const size_t smem = Tile4<KG, VG>::own + plan_bytes(a.b.B, a.b.n_groups);
	XALM_CUDA_CHECK(allow_smem((const void*) paged4_tile_kernel<KG, VG, TWO>));
	XALM_CUDA_CHECK(launch(paged4_tile_kernel<KG, VG, TWO>, a.part[part].grid, GT, smem, s, part > 0, a, a.part[part], p, type));
	return XALM_OK;
}
template <int KG, int VG>
static int launch_tile(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	return type == XALM_F16 ? launch_parts<KG, VG, true>(a, p, part, type, s) : launch_parts<KG, VG, false>(a, p, part, type, s);
}
Shape4 tile4_shape(const Pool4& p) { return p.kg <= 4 && p.vg <= 4 ? Shape4{GM, 1} : Shape4{0, 0}; }
int launch_attn4_tile(const Attn& a, const Pool4& p, int part, int type, cudaStream_t s) {
	if (p.kg == 4) return p.vg == 4 ? launch_tile<4, 4>(a, p, part, type, s) : launch_tile<4, 2>(a, p, part, type, s);
	return p.vg == 4 ? launch_tile<2, 4>(a, p, part, type, s) : launch_tile<2, 2>(a, p, part, type, s);
}

} // namespace paged
} // namespace xalm
