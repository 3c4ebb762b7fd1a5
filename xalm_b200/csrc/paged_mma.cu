// paged_mma.cu — attention over paged caches of 16-bit elements, for few rows: a token, or the few (token, head) rows that fit one 16-row matrix tile.
#include <cuda.h>

#include "paged.cuh"
#include "paged_tma.cuh"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, in one pass over the pages.  A step of single tokens reads every key and value once
// for a handful of rows: HBM bounds it, and what the kernel has to do is to keep enough bytes on their way.  A warp brings tiles of 64 keys and values
// by TMA (a page's slots, 64 entries wide, swizzled) into a ring; four warps take 16 keys of a tile each (with 32 of every other tile a stage is held longer: 91 us in place of 79 for the
// 64 sequences below behind 8192 tokens in common), with maximum, sum and output of their own, so that
// none waits for another and a stage is free again after a quarter of a tile's work: scores and sums by mma.sync m16n8k16 with the 16 rows as A, queries and sums in registers.
// At the end of a piece the four join through shared memory.  (tcgen05 would want 64 rows or more: a step of four heads to a kv head has four.)
// 64 sequences of 1000 to 2000 tokens, 8 kv heads of 128: 78 us with the join, 5.0 TB/s, 128 of 4000 325 us, 6.5 TB/s, wherever the pages lie; 10700 lists of 16 pages of 64, which L2 has, 474 us,
// 12.4 TB/s.
// Probabilities enter the second product in two parts of the cache's type, rounded and what that left (one alone had 1.5 times the result's own rounding as its error): of up to eight rows
// the second part are rows 8 to 15 of the same product, of more it costs a product of its own.  Scores, maxima and sums are fp32.
// fp16 ends at 2^-24, so its probabilities are lifted by 2^12, its second part by 2^11 more into sums of its own: what a probability loses is below 2^-47 of the row's largest one, and
// thousands of small ones beside a large one whose value is 0 keep their sum.
// =========================================================================================================================================
constexpr int MM = 16, CW = 4, MT = (CW + 1) * 32;

struct MmaConfig {
	int stages, per_sm;
	size_t smem;
};
template <int D>
struct Sizes {
	static constexpr int TILE = KT * D * 2;         // bytes of a key or value tile
	static constexpr int STAGE = 2 * TILE;
	static constexpr int OS = D + 8;                // floats between rows of the join's buffer
	static constexpr int JOIN = CW * 4 * OS * 4;    // four rows of every warp
};
// Two CTAs of three or more stages on an SM, or one with what there is: bytes on their way count, not how many CTAs ask for them
template <int D>
static MmaConfig mma_config(size_t plan, int n_lists) {
	using Z = Sizes<D>;
	const size_t fixed = 1024 + Z::JOIN + CW * MM * 8 + 512 + (size_t) n_lists * 4 + 16 + plan;
	for (int per_sm = 2; per_sm >= 1; per_sm--) {
		const size_t room = per_sm == 2 ? 113 * 1024 : 226 * 1024;
		const int n = room > fixed ? (int) ((room - fixed) / Z::STAGE) : 0;
		if (n >= 3 || per_sm == 1) {
			const int stages = n > 8 ? 8 : n;
			return MmaConfig{stages, per_sm, fixed + (size_t) stages * Z::STAGE};
		}
	}
	return MmaConfig{};
}

// Not volatile: products may move behind the loads of others, which are kept in their order
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
	if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
		asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
	else
		asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// 16-byte chunk c of row r in a tile of 64-entry columns with `rows` rows each, as the copy engine's 128-byte swizzle lays it
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int rows, int r, int c) { return base + (uint32_t) ((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
	if constexpr (std::is_same<T, __half>::value) {
		const __half2 h = __floats2half2_rn(lo, hi);
		return *reinterpret_cast<const uint32_t*>(&h);
	} else {
		const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
		return *reinterpret_cast<const uint32_t*>(&h);
	}
}
// what is left of two numbers beside their rounded ones
template <typename T>
__device__ __forceinline__ float2 rest16(uint32_t rounded, float lo, float hi) {
	if constexpr (std::is_same<T, __half>::value) {
		const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
		return make_float2(lo - r.x, hi - r.y);
	} else return make_float2(lo - __uint_as_float(rounded << 16), hi - __uint_as_float(rounded & 0xffff0000u));
}
// rounding towards 0
__device__ __forceinline__ uint32_t cut_bf16(float lo, float hi) { return (uint32_t) __bfloat16_as_ushort(__float2bfloat16_rz(lo)) | (uint32_t) __bfloat16_as_ushort(__float2bfloat16_rz(hi)) << 16; }
constexpr float REST_LIFT = 2048.f; // of fp16: half a step of 2^15, the most a probability is, is 2^4
// the two parts of two probabilities
template <typename T>
__device__ __forceinline__ void parts16(float lo, float hi, uint32_t& rounded, uint32_t& rest) {
	if constexpr (std::is_same<T, __half>::value) {
		// no 0, beside which an infinite value would give no infinity: what this adds to the smallest, and to masked ones, the second part takes off again
		const uint32_t near = probs_f16(lo, hi);
		const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2*>(&near), __halves2half2(__ushort_as_half(1), __ushort_as_half(1)));
		rounded = *reinterpret_cast<const uint32_t*>(&h);
		const float2 r = rest16<T>(rounded, lo, hi);
		rest = probs_f16(r.x * REST_LIFT, r.y * REST_LIFT);
	} else {
		rounded = pack16<T>(lo, hi);
		const float2 r = rest16<T>(rounded, lo, hi);
		rest = pack16<T>(r.x, r.y);
	}
}
__device__ __forceinline__ float ex2(float x) {
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}

// WIDE: units may have more than eight rows.  Those of a list are one token's, so that the host knows; without the code for them 10700 lists of fp16 take 481 us, with it 518.
template <typename T, int D, bool LIST, bool WIDE>
__global__ void __launch_bounds__(MT, D == 256 ? 1 : 2) paged_mma_kernel(const __grid_constant__ Attn a, const __grid_constant__ Part part, const __grid_constant__ CUtensorMap kmap,
                                                                         const __grid_constant__ CUtensorMap vmap, const int stages) {
	using Z = Sizes<D>;
	extern __shared__ uint8_t raw[];
	uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
	uint8_t* ring = smem;
	float* s_o = reinterpret_cast<float*>(ring + (size_t) stages * Z::STAGE); // [CW][4][OS]
	float2* s_ml = reinterpret_cast<float2*>((uint8_t*) s_o + Z::JOIN);   // [CW][MM]
	uint64_t* full = reinterpret_cast<uint64_t*>(s_ml + CW * MM);         // [8]
	uint64_t* empty = full + 8;                                           // [8]
	State* state = reinterpret_cast<State*>(empty + 8);
	int* s_sent = reinterpret_cast<int*>(state + 1);                      // tiles whose copies were sent
	int* s_ids = s_sent + 1;                                              // [32]
	int* s_list = reinterpret_cast<int*>((uint8_t*) full + 512);          // [S]
	uint8_t* s_plan = reinterpret_cast<uint8_t*>(s_list) + ((LIST ? a.S * 4 : 0) + 15) / 16 * 16;
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	if (tid == 0) {
		for (int i = 0; i < stages; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], CW); }
		state->init();
		*s_sent = 0;
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
	}
	pdl_launch_dependents();
	const int dc = (a.c.d + 63) / 64, vc = (a.c.dv + 63) / 64;
	// Products run over all D entries, without a question between them (asking eight times took as long as the products).  Blocks that no copy fills are zeros.
	if (dc < D / 64 || vc < D / 64)
		for (int i = tid; i < stages * 2 * (D / 64) * (KT * 8); i += MT) {
			const int block = i / (KT * 8), of_tile = block % (D / 64);
			if (of_tile >= (block / (D / 64) % 2 ? vc : dc)) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
		}
	Plan plan;
	if (!LIST) make_plan<MT>(a, part, s_plan, plan);
	else if (blockIdx.x == 0) check_seqs(a.c, a.b, tid, MT);
	__syncthreads();
	const int P = 1 << a.c.shift, W = min(P, KT), per = KT / W; // slots of a box, boxes of a tile's column
	Walk k;
	bool more = LIST ? list_begin(a, part, k) : walk_begin(a, part, plan, k);
	if (tid == 0)
		write_head(a, part, k, more, LIST ? more && row_in_seq(k.x.q, k.x.row0) : more && k.x.seg >= a.b.n_groups && k.x.key0 == 0, LIST ? share_of(list_total(a, part), part.grid) : plan.share);
	int st = 0;         // the tile's stage, and how often the ring has come round
	uint32_t round = 0;
	auto advance = [&] {
		if (++st == stages) { st = 0; round ^= 1; }
	};

	if (warp == CW) { // ---- the copies: 32 boxes' pages in one asking, then one thread sends them ----
		int sent = 0; // tiles
		for (; more; more = LIST ? list_next(a, part, k) : walk_next(a, part, plan, k)) {
			const Piece& x = k.x;
			if (x.j0 == x.j1) continue;
			int vis;
			if (LIST) {
				if (!row_in_seq(x.q, x.row0)) continue;
				const int pos = x.q.len - x.q.n + x.row0 - x.q.a;
				bool own;
				vis = list_pages(a, x.row0, x.g, pos >= 0 ? pos >> a.c.shift : -1, s_list, &own) << a.c.shift;
				if (own) vis += (pos & (P - 1)) + 1 - P;
			} else if (x.seg < a.b.n_groups) vis = plan.shs[x.s];
			else vis = own_keys(x.q, x.key0, a.rep, min((x.t + 1) * MM, x.rows) - 1);
			const int j1 = min(x.j1, (vis + KT - 1) / KT), batch = 32 / per, key0 = x.key0, g = x.g;
			bool ok = true;
			for (int j = x.j0; j < j1 && ok; j += batch) {
				const int at = j * KT + lane * W, key = key0 + at;
				int id = -1;
				if (at < vis) {
					id = page_of(a.c, a.b, x.s, LIST ? s_list[key >> a.c.shift] : key >> a.c.shift);
					if (id < 0) report(a.c, ERR_PAGE);
				}
				s_ids[lane] = id;
				__syncwarp();
				const int count = min(batch, j1 - j);
				if (elect())
					for (int i = 0, st1 = st, round1 = round; i < count; i++) {
						if (!(ok = wait_alone<!LIST>(&empty[st1], round1 ^ 1, state, a.c))) break;
						mbar_expect_tx(&full[st1], (uint32_t) ((dc + vc) * KT * 128));
						const uint32_t dst = smem_u32(ring) + (uint32_t) st1 * Z::STAGE;
						const int slot = (key0 + (j + i) * KT) & (P - 1);
						copy_tile(dst, &kmap, a.c.d, g, slot, per, W, s_ids + i * per, a.c.pages, &full[st1]);
						copy_tile(dst + Z::TILE, &vmap, a.c.dv, g, slot, per, W, s_ids + i * per, a.c.pages, &full[st1]);
						if (++st1 == stages) { st1 = 0; round1 ^= 1; }
						*s_sent = sent + i + 1;
					}
				ok = __all_sync(0xffffffffu, ok);
				for (int i = 0; i < count; i++) advance();
				sent += count;
			}
			if (!ok) break;
		}
		if (*(volatile int*) &state->dead) { // gave up: copies still on their way end first
			__syncwarp();
			const int last = *(volatile int*) s_sent;
			for (int i = max(0, last - stages); i < last; i++) wait_some(&full[i % stages], (i / stages) & 1, state);
		}
		pdl_wait(); // beside the kernel of many rows, whose inputs were complete before it began, but not ahead of it to the join
		return;
	}

	// ---- the products ----
	const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;            // a negative scale turns the queries' signs
	const float c1 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f); // not 0: 0 times an infinity is no number
	constexpr bool HALF = std::is_same<T, __half>::value;
	constexpr float LIFT = HALF ? 12.f : 0.f, LAG = HALF ? 3.f : 11.5f; // in powers of two; fp16 ends at 2^16
	const float slack = LAG / c1;
	// where this lane's rows of ldmatrix lie in a tile: keys (lane & 7) + 8 (lane / 16) of this warp's 16, chunk (lane / 8) & 1; values lane & 15, chunk lane / 16.  Every two chunks
	// further on are two bits of the address turned over, every eight a block of columns.
	const int kr = (lane & 7) + (lane >> 4) * 8, vr = lane & 15;
	const uint32_t k_lane = (uint32_t) ((warp * 16 + kr) * 128 + ((((lane >> 3) & 1) ^ (kr & 7)) << 4));
	const uint32_t v_lane = (uint32_t) (Z::TILE + (warp * 16 + vr) * 128 + (((lane >> 4) ^ (vr & 7)) << 4));
	for (; more; more = LIST ? list_next(a, part, k) : walk_next(a, part, plan, k)) {
		const Piece& x = k.x;
		if (x.j0 == x.j1) continue;
		const bool prefix = !LIST && x.seg < a.b.n_groups;
		const int rows = min(MM, x.rows - x.t * MM), h0 = x.g * a.rep;
		int lim0, lim1, least, most; // keys that this lane's two rows see; that the first and the last row see
		if (LIST && !row_in_seq(x.q, x.row0)) continue;
		// queries as A: rows lane / 4 and lane / 4 + 8, entries 2 (lane % 4) and 8 more of every 16
		uint32_t qa[D / 16][4];
#pragma unroll
		for (int half = 0; half < 2; half++) {
			const int r = lane / 4 + half * 8, w = x.t * MM + r;
			const uint8_t* at = a.q + ((long long) (x.row0 + w / a.rep) * a.q_row + (h0 + w % a.rep) * a.c.d + (lane & 3) * 2) * 2;
#pragma unroll
			for (int kk = 0; kk < D / 16; kk++) {
				qa[kk][half] = r < rows && kk * 16 < a.c.d ? *reinterpret_cast<const uint32_t*>(at + kk * 32) ^ flip : 0;
				qa[kk][half + 2] = r < rows && kk * 16 + 8 < a.c.d ? *reinterpret_cast<const uint32_t*>(at + kk * 32 + 16) ^ flip : 0;
			}
		}
		if (LIST) {
			const int pos = x.q.len - x.q.n + x.row0 - x.q.a;
			bool own;
			const int pages = list_pages(a, x.row0, x.g, pos >= 0 ? pos >> a.c.shift : -1, nullptr, &own);
			least = most = lim0 = lim1 = (pages << a.c.shift) + (own ? (pos & (P - 1)) + 1 - P : 0);
		} else if (prefix) least = most = lim0 = lim1 = plan.shs[x.s];
		else {
			least = own_keys(x.q, x.key0, a.rep, x.t * MM);
			most = own_keys(x.q, x.key0, a.rep, x.t * MM + rows - 1);
			lim0 = own_keys(x.q, x.key0, a.rep, min(x.t * MM + lane / 4, x.rows - 1));
			lim1 = own_keys(x.q, x.key0, a.rep, min(x.t * MM + lane / 4 + 8, x.rows - 1));
		}
		float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, b0 = 0.f, b1 = 0.f; // maxima of the raw scores, and what is added to a score times c1
#pragma unroll
		for (int i = 0; i < D / 8; i++)
#pragma unroll
			for (int e = 0; e < 4; e++) o[i][e] = 0.f;
		const int j1 = min(x.j1, (most + KT - 1) / KT);
		const bool high = WIDE && rows > 8;
		bool there = false; // the next tile
		for (int j = x.j0; j < j1; j++, advance()) {
			if (!there && !wait_for<!LIST>(&full[st], round, state, a.c)) continue;
			const uint32_t tile = smem_u32(ring) + (uint32_t) st * Z::STAGE;
			const int base = j * KT + warp * 16; // this warp's 16 keys
			const bool tail = base + 16 > most;
			if (tail) { // slots that no row sees may hold anything: as zeros they add nothing
				const int from = max(most - base, 0);
				for (int i = lane; i < (16 - from) * vc * 8; i += 32) {
					const int r = from + i / (vc * 8), c = i % (vc * 8);
					asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(chunk_at(tile + Z::TILE + warp * 16 * 128, KT, r, c)), "r"(0) : "memory");
				}
				__syncwarp();
			}
			float s[2][4];
#pragma unroll
			for (int i = 0; i < 2; i++)
#pragma unroll
				for (int e = 0; e < 4; e++) s[i][e] = 0.f;
#pragma unroll
			for (int kk = 0; kk < D / 16; kk++)
			{
				uint32_t b[4];
				ldsm4(b, ((tile + k_lane) ^ ((kk * 2 & 7) << 4)) + (kk >> 2) * KT * 128);
				mma16<T>(s[0], qa[kk], b[0], b[1]);
				mma16<T>(s[1], qa[kk], b[2], b[3]);
			}
			if (base + 16 > least) {
#pragma unroll
				for (int i = 0; i < 2; i++)
#pragma unroll
					for (int e = 0; e < 4; e++)
						if (base + i * 8 + (lane & 3) * 2 + (e & 1) >= (e < 2 ? lim0 : lim1)) s[i][e] = -INFINITY;
			}
			// The maximum that probabilities are taken against may lag behind by 2^LAG: then no lane has to ask its neighbours, and sums stay as they are
			float t0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), t1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
			if (__any_sync(0xffffffffu, t0 > m0 + slack || t1 > m1 + slack)) {
#pragma unroll
				for (int w = 1; w < 4; w <<= 1) {
					t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
					t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
				}
				const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1), f0 = m0 == -INFINITY ? 0.f : ex2((m0 - n0) * c1), f1 = m1 == -INFINITY ? 0.f : ex2((m1 - n1) * c1);
				l0 *= f0;
				l1 *= f1;
#pragma unroll
				for (int i = 0; i < D / 8; i++) { o[i][0] *= f0; o[i][1] *= f0; o[i][2] *= high ? f1 : f0; o[i][3] *= high ? f1 : f0; }
				m0 = n0;
				m1 = n1;
				b0 = m0 == -INFINITY ? 0.f : fmaf(-m0, c1, LIFT);
				b1 = m1 == -INFINITY ? 0.f : fmaf(-m1, c1, LIFT);
			}
			// asked for here, known when this tile is done
			there = j + 1 < j1 && try_wait_once(&full[st + 1 == stages ? 0 : st + 1], round ^ (st + 1 == stages));
			uint32_t pa[4], rest[4]; // probabilities, and what their rounding left
#pragma unroll
			for (int i = 0; i < 2; i++) {
				const float x0 = ex2(fmaf(s[i][0], c1, b0)), x1 = ex2(fmaf(s[i][1], c1, b0));
				l0 += x0 + x1;
				parts16<T>(x0, x1, pa[2 * i], rest[2 * i]);
				pa[2 * i + 1] = rest[2 * i];
			}
			if constexpr (HALF) {
				if (high) {
#pragma unroll
					for (int i = 0; i < 2; i++) {
						const float x0 = ex2(fmaf(s[i][2], c1, b1)), x1 = ex2(fmaf(s[i][3], c1, b1));
						l1 += x0 + x1;
						parts16<T>(x0, x1, pa[2 * i + 1], rest[2 * i + 1]);
					}
#pragma unroll
					for (int c = 0; c < D / 16; c++) {
						uint32_t b[4];
						float t[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
						ldsm4_t(b, ((tile + v_lane) ^ ((c * 2 & 7) << 4)) + (c >> 2) * KT * 128);
						mma16<T>(t[0], rest, b[0], b[1]);
						mma16<T>(t[1], rest, b[2], b[3]);
#pragma unroll
						for (int i = 0; i < 2; i++)
#pragma unroll
							for (int e = 0; e < 4; e++) // what is not finite comes from the first part's product, none of whose probabilities is 0
								o[2 * c + i][e] = fabsf(t[i][e]) <= 3.4e38f ? fmaf(t[i][e], 1.f / REST_LIFT, o[2 * c + i][e]) : o[2 * c + i][e];
					}
				}
			} else if (high) { // both parts add to the same sums: neither is negative, nor 0 beside a probability that is not, so that an infinite value gives an infinity
#pragma unroll
				for (int i = 0; i < 4; i++) {
					constexpr float LEAST = 1.17549435e-38f; // the smallest number that a product does not take for 0
					float x[2];
#pragma unroll
					for (int e = 0; e < 2; e++) {
						x[e] = ex2(fmaf(s[i >> 1][(i & 1) * 2 + e], c1, i & 1 ? b1 : b0));
						if (i & 1) l1 += x[e];
						x[e] = x[e] > 0.f ? fmaxf(x[e], LEAST) : x[e];
					}
					pa[i] = cut_bf16(x[0], x[1]);
					const float2 left = rest16<T>(pa[i], x[0], x[1]);
					rest[i] = pack16<T>(x[0] > 0.f ? fmaxf(left.x, LEAST) : left.x, x[1] > 0.f ? fmaxf(left.y, LEAST) : left.y);
				}
#pragma unroll
				for (int c = 0; c < D / 16; c++) {
					uint32_t b[4];
					ldsm4_t(b, ((tile + v_lane) ^ ((c * 2 & 7) << 4)) + (c >> 2) * KT * 128);
					mma16<T>(o[2 * c], rest, b[0], b[1]);
					mma16<T>(o[2 * c + 1], rest, b[2], b[3]);
				}
			}
#pragma unroll
			for (int c = 0; c < D / 16; c++)
			{
				uint32_t b[4];
				ldsm4_t(b, ((tile + v_lane) ^ ((c * 2 & 7) << 4)) + (c >> 2) * KT * 128);
				mma16<T>(o[2 * c], pa, b[0], b[1]);
				mma16<T>(o[2 * c + 1], pa, b[2], b[3]);
			}
			if (tail) asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the zeros, before the next copy
			__syncwarp();
			if (lane == 0) mbar_arrive(&empty[st]);
		}
		if (!high)
#pragma unroll
			for (int i = 0; i < D / 8; i++) // what an infinite value made infinite stays so: the rest may be 0 or negative
#pragma unroll
				for (int e = 0; e < 2; e++) o[i][e] = fabsf(o[i][e]) <= 3.4e38f ? fmaf(o[i][e + 2], HALF ? 1.f / REST_LIFT : 1.f, o[i][e]) : o[i][e];
		m0 = fmaf(m0, c1, -LIFT); // in units of log2 from here on
		m1 = fmaf(m1, c1, -LIFT);
		// ---- the four warps' sums ----
#pragma unroll
		for (int w = 1; w < 4; w <<= 1) {
			l0 += __shfl_xor_sync(0xffffffffu, l0, w);
			l1 += __shfl_xor_sync(0xffffffffu, l1, w);
		}
		if ((lane & 3) == 0) {
			s_ml[warp * MM + lane / 4] = make_float2(m0, l0);
			s_ml[warp * MM + lane / 4 + 8] = make_float2(m1, l1);
		}
		bar_sync(1, CW * 32);
		const bool direct = x.j0 == 0 && x.j1 == x.w && !prefix && x.key0 == 0;
		const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
		const bool mixed = !LIST && !prefix && least < most && x.j1 * KT > least; // some row of the tile must not see what another does
		float f[2];
#pragma unroll
		for (int half = 0; half < 2; half++) {
			float mx = -INFINITY;
#pragma unroll
			for (int w = 0; w < CW; w++) mx = fmaxf(mx, s_ml[w * MM + lane / 4 + half * 8].x);
			const float mine = half ? m1 : m0;
			f[half] = mine == -INFINITY ? 0.f : ex2(mine - mx);
		}
#pragma unroll
		for (int four = 0; four < 4; four++) { // four rows at a time
			if (four * 4 >= rows) break;
			if ((lane >> 4) == (four & 1)) {
#pragma unroll
				for (int i = 0; i < D / 8; i++)
					if (i * 8 < a.c.dv)
						*reinterpret_cast<float2*>(s_o + (warp * 4 + (lane / 4) % 4) * Z::OS + i * 8 + (lane & 3) * 2) = make_float2(o[i][four & 2] * f[four >> 1], o[i][(four & 2) + 1] * f[four >> 1]);
			}
			bar_sync(1, CW * 32);
			const int rh = min(4, rows - four * 4), cols = a.c.dv / 4;
			for (int i = tid; i < rh * cols; i += CW * 32) {
				const int r = i / cols, c = i % cols * 4, row = four * 4 + r;
				float mx = -INFINITY, l = 0.f;
#pragma unroll
				for (int w = 0; w < CW; w++) mx = fmaxf(mx, s_ml[w * MM + row].x);
#pragma unroll
				for (int w = 0; w < CW; w++) {
					const float2 ml = s_ml[w * MM + row];
					l += ml.y * (ml.x == -INFINITY ? 0.f : ex2(ml.x - mx)); // a NaN stays one
				}
				float4 v = *reinterpret_cast<const float4*>(s_o + r * Z::OS + c);
#pragma unroll
				for (int w = 1; w < CW; w++) {
					const float4 u = *reinterpret_cast<const float4*>(s_o + (w * 4 + r) * Z::OS + c);
					v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
				}
				put_row<T>(a, part, x, MM, row, c, v, mx, l, direct, slot);
			}
			bar_sync(1, CW * 32);
		}
		if (mixed) {
			// A value that is not finite and that only later rows see has met probabilities of zero in the product: rows that do not see it are done again, key by key.
			bool again = false;
#pragma unroll
			for (int i = 0; i < D / 8; i++)
#pragma unroll
				for (int e = 0; e < 4; e++) again = again || !(fabsf(o[i][e]) <= 3.0e38f);
			if (tid == 0) s_ml[0].x = 0.f;
			bar_sync(1, CW * 32);
			if (again) s_ml[0].x = 1.f;
			bar_sync(1, CW * 32);
			const bool redo = s_ml[0].x != 0.f;
			bar_sync(1, CW * 32);
			const Piece y = x; // in memory only here
			if (redo) redo_rows<T, MM, MM>(a, part, y, 0, state, reinterpret_cast<int*>(s_ml), s_o, tid, 1);
		}
	}
}

template <int D>
static MmaConfig config_of(const Cache&, const BatchView& b, int n_lists) { return mma_config<D>(n_lists ? 0 : plan_bytes(b.B, b.n_groups), n_lists); }
static int padded(const Cache& c) {
	const int d = c.d > c.dv ? c.d : c.dv;
	return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}
int mma_ctas_per_sm(const Cache& c, const BatchView& b, int n_lists) {
	const int D = padded(c);
	return (D == 64 ? config_of<64>(c, b, n_lists) : D == 128 ? config_of<128>(c, b, n_lists) : config_of<256>(c, b, n_lists)).per_sm;
}

template <typename T, int D, bool LIST, bool WIDE>
static int launch_typed(const Attn& a, int part, int type, cudaStream_t s) {
	const MmaConfig cfg = config_of<D>(a.c, a.b, LIST ? a.S : 0);
	if (cfg.stages < 1) return set_error(XALM_ERR_INVALID, "paged attention: no shared memory left for pages beside %d sequences", a.b.B);
	CUtensorMap kmap, vmap;
	XALM_TRY(pool_map(a.c, type, true, &kmap));
	XALM_TRY(pool_map(a.c, type, false, &vmap));
	XALM_CUDA_CHECK(allow_smem((const void*) paged_mma_kernel<T, D, LIST, WIDE>));
	XALM_CUDA_CHECK(launch(paged_mma_kernel<T, D, LIST, WIDE>, a.part[part].grid, MT, cfg.smem, s, part > 0, a, a.part[part], kmap, vmap, cfg.stages));
	return XALM_OK;
}
template <typename T, int D>
static int launch_lists(const Attn& a, int part, int type, cudaStream_t s) {
	return !a.lists ? launch_typed<T, D, false, true>(a, part, type, s) : a.rep > 8 ? launch_typed<T, D, true, true>(a, part, type, s) : launch_typed<T, D, true, false>(a, part, type, s);
}
template <typename T>
static int launch_size(const Attn& a, int part, int type, cudaStream_t s) {
	switch (padded(a.c)) {
		case 64: return launch_lists<T, 64>(a, part, type, s);
		case 128: return launch_lists<T, 128>(a, part, type, s);
		default: return launch_lists<T, 256>(a, part, type, s);
	}
}
int launch_attn_mma(const Attn& a, int part, int type, cudaStream_t s) {
	return type == XALM_F16 ? launch_size<__half>(a, part, type, s) : launch_size<__nv_bfloat16>(a, part, type, s);
}

} // namespace paged
} // namespace xalm
