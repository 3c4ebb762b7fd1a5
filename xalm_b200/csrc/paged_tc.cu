// paged_tc.cu — attention over paged caches of 16-bit elements, for many rows: what a group of sequences has in common, prompts and their continuations.
#include "paged.cuh"
#include "paged_tma.cuh"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// The same sums as paged_mma_kernel for 256 (token, head) rows at a time, two halves of 128: S = Q K^T and O += P V by tcgen05 with S, P and O in tensor memory.
// One warp brings tiles of 64 keys and of 64 values by TMA, each read once for both halves; a warp to a half issues its products; four warps to a half turn S into P, a row to a
// thread.  At 128 channels a tile of a half takes the tensor pipe 622 cycles (431 of them the scores, which shared memory bounds) and the exponential unit 512, which the halves share by
// turns; one load of keys and values for 256 rows asks L2 for half of what 128 rows would.  One warp that issued both halves' products was what everything waited for:
// a product takes 30 cycles to issue and a wait that is over 150 (2800 cycles a tile).
// P lies in tensor memory where S lay (its first 32 columns), two S buffers to a half: the scores of the next tile are under way while this one's are worked on.
// O accumulates unscaled and is rescaled only when a row's maximum has grown by more than 2^LAG over the one its probabilities are taken against.
// Probabilities are rounded once to the cache's type (a second part would double the second product and want columns of tensor memory that there are none of); sums l are of the unrounded
// ones.  fp16 ends at 2^-24, so its probabilities are lifted (Lift) and the maximum lags by less: those below 2^-27 of the row's largest lose bits, those below 2^-38 count in l alone.
// V comes with its entries as the fast dimension, which the second product reads as it is (B transposed).
// Tensor memory: S of half h, buffer b at columns 128 h + 64 b; O of half h at 256 + 128 h: the whole 512 of an SM, so heads of more than 128 entries stay on mma.sync.
// What runs once to a piece is kept short and in loops: code that comes from memory for the first time costs more than it takes to run.
// =========================================================================================================================================
constexpr int TT = 384;            // copies, products of either half, none, 2 x 4 warps of softmax
constexpr int HALF_ROWS = 128;
constexpr int QB = HALF_ROWS * 128; // bytes of 64 entries of a half's queries
constexpr int KB = KT * 128;        // bytes of 64 entries of a key or value tile
constexpr int RING = 4;

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// D (+)= A B^T with A from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
	asm volatile(
	    "{\n"
	    ".reg .pred p;\n"
	    "setp.ne.b32 p, %4, 0;\n"
	    "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
	    "}\n" ::"r"(d),
	    "l"(a), "l"(b), "r"(idesc), "r"(add)
	    : "memory");
}
// with A from tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
	asm volatile(
	    "{\n"
	    ".reg .pred p;\n"
	    "setp.ne.b32 p, %4, 0;\n"
	    "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
	    "}\n" ::"r"(d),
	    "r"(a), "l"(b), "r"(idesc), "r"(add)
	    : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
	asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 128-byte swizzle.  Fast dimension = the summed one: 8-row groups 1024 bytes apart.  Fast dimension = the output's columns: groups of 8 summed rows 1024 bytes apart,
// blocks of 64 columns `block` bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t at) { return (uint64_t) ((at & 0x3FFFFu) >> 4) | ((uint64_t) (1024 >> 4) << 32) | (1ull << 46) | (2ull << 61); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t at, uint32_t block) { return desc_k(at) | ((uint64_t) (block >> 4) << 16); }
template <typename T>
__device__ __forceinline__ uint32_t instr(int n, bool b_transposed) {
	const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
	return (1u << 4) | (f << 7) | (f << 10) | ((b_transposed ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (HALF_ROWS >> 4) << 24);
}
#define XALM_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
__device__ __forceinline__ void ld32(uint32_t at, uint32_t* r) {
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
	    "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
	    : XALM_R8(r, 0), XALM_R8(r, 8), XALM_R8(r, 16), XALM_R8(r, 24)
	    : "r"(at));
}
#undef XALM_R8
// The loads issued so far have landed in these registers: none of them is used ahead of the wait
#define XALM_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void wait_ld(uint32_t* r) {
	asm volatile("tcgen05.wait::ld.sync.aligned;" : XALM_RW8(r, 0), XALM_RW8(r, 8), XALM_RW8(r, 16), XALM_RW8(r, 24)::"memory");
}
#undef XALM_RW8
#define XALM_R8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void st32(uint32_t at, const uint32_t* r) {
	asm volatile(
	    "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
	    "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n" ::XALM_R8(r, 0),
	    XALM_R8(r, 8), XALM_R8(r, 16), XALM_R8(r, 24), "r"(at)
	    : "memory");
}
#undef XALM_R8
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
	if constexpr (std::is_same<T, __half>::value) {
		const __half2 h = __floats2half2_rn(lo, hi);
		return *reinterpret_cast<const uint32_t*>(&h);
	} else {
		const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
		return *reinterpret_cast<const uint32_t*>(&h);
	}
}

// A piece as the three kinds of warps see it
struct TcPiece {
	bool prefix;
	int rows, most, j1; // rows of the unit, keys that its last row sees, last tile of the piece that any row sees
};
__device__ __forceinline__ TcPiece tc_piece(const Attn& a, const Plan& plan, const Piece& x) {
	TcPiece p;
	p.prefix = x.seg < a.b.n_groups;
	p.rows = min(TC_ROWS, x.rows - x.t * TC_ROWS);
	p.most = p.prefix ? plan.shs[x.s] : own_keys(x.q, x.key0, a.rep, x.t * TC_ROWS + p.rows - 1);
	p.j1 = min(x.j1, (p.most + KT - 1) / KT);
	return p;
}

struct TcShared {
	uint64_t full[RING], empty[RING];
	uint64_t drained[2], q_full[2], s_full[2][2], p_full[2][2], o_full[2][2]; // by half and by the tile's parity, so that nobody is ever two phases ahead of a wait
	uint32_t tmem;
	State state;
	int flag[2], ids[32], sent; // tiles whose copies were sent
	alignas(16) float buf[2][256]; // read 16 bytes at a time
};

// fp16 rounds probabilities to 0 beside which an infinite value should give an infinity: the infinities and NaNs of column after column that a lane's row sees are put where its sums go.  A
// whole warp, whose lanes look at 32 keys at a time; row: of the unit, lim, most: keys that the lane's row sees, and the unit's last; fix: whether the lane's row is in need of it
__device__ __noinline__ void put_infinities(const Attn& a, const Part& part, const Piece& x, int row, int lim, int most, bool fix) {
	const int lane = threadIdx.x & 31, P = 1 << a.c.shift, w = x.t * TC_ROWS + row, last = min(x.j1 * KT, most);
	const bool direct = x.j0 == 0 && x.j1 == x.w && x.seg >= a.b.n_groups && x.key0 == 0;
	const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
	for (int c = 0; c < a.c.dv; c += 8) {
		unsigned up = 0, down = 0; // a bit to a column; a NaN is both
#pragma unroll 4
		for (int kb = x.j0 * KT; kb < last; kb += 32) {
			const int key = x.key0 + kb + lane, pg = kb + lane < last ? page_of(a.c, a.b, x.s, key >> a.c.shift) : -1;
			uint4 u = make_uint4(0, 0, 0, 0);
			if (pg >= 0) u = *reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(a.c.v) + pg * a.c.v_page + (key & (P - 1)) * a.c.v_slot + x.g * a.c.v_head + c);
			const uint32_t word[4] = {u.x, u.y, u.z, u.w};
			unsigned bits = 0;
#pragma unroll
			for (int e = 0; e < 8; e++) {
				const uint32_t v = word[e >> 1] >> (e & 1) * 16;
				if ((v & 0x7c00u) == 0x7c00u) bits |= ((v & 0x3ffu ? 0x101u : v & 0x8000u ? 0x100u : 1u)) << e;
			}
			for (unsigned m = __ballot_sync(0xffffffffu, bits != 0); m; m &= m - 1) {
				const int from = __ffs(m) - 1;
				const unsigned b = __shfl_sync(0xffffffffu, bits, from);
				if (kb + from < lim) { up |= b & 0xff; down |= b >> 8; }
			}
		}
		if (fix)
			for (unsigned m = up | down; m; m &= m - 1) {
				const int e = __ffs(m) - 1;
				const float v = up >> e & down >> e & 1 ? NAN : up >> e & 1 ? INFINITY : -INFINITY;
				if (direct) reinterpret_cast<__half*>(a.out)[(long long) (x.row0 + w / a.rep) * a.out_row + (x.g * a.rep + w % a.rep) * a.c.dv + c + e] = __float2half_rn(v);
				else if (slot < part.slots) part.o[(slot * TC_ROWS + row) * a.c.dv + c + e] = v;
			}
	}
	__syncwarp();
}

template <typename T>
struct Lift { // in powers of two; fp16 ends at 2^16
	static constexpr float BY = 0.f, LAG = 11.5f;
};
template <>
struct Lift<__half> {
	static constexpr float BY = 13.f, LAG = 2.9f;
};

template <typename T>
__global__ void __launch_bounds__(TT, 1) paged_tc_kernel(const __grid_constant__ Attn a, const __grid_constant__ Part part, const __grid_constant__ CUtensorMap kmap,
                                                         const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap) {
	extern __shared__ uint8_t raw[];
	uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
	uint8_t* s_q = smem;                       // [half][2 blocks][128 rows][128 bytes]
	uint8_t* s_k = s_q + 4 * QB;               // [RING][2 blocks][64 keys][128 bytes]
	uint8_t* s_v = s_k + RING * 2 * KB;
	TcShared& sh = *reinterpret_cast<TcShared*>(s_v + RING * 2 * KB);
	uint8_t* s_plan = reinterpret_cast<uint8_t*>(&sh + 1);
	static_assert(sizeof(TcShared) % 16 == 0 && offsetof(TcShared, buf) % 16 == 0, "what slow_row reads");
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	if (tid == 0) {
		for (int i = 0; i < RING; i++) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 2); }
		for (int h = 0; h < 2; h++) {
			mbar_init(&sh.drained[h], 1);
			mbar_init(&sh.q_full[h], 1);
			for (int b = 0; b < 2; b++) { mbar_init(&sh.s_full[h][b], 1); mbar_init(&sh.p_full[h][b], 4); mbar_init(&sh.o_full[h][b], 1); }
		}
		sh.state.init();
		sh.sent = 0;
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
	}
	if (warp == 1) {
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
	}
	pdl_launch_dependents();
	Plan plan;
	make_plan<TT>(a, part, s_plan, plan);
	fence_before();
	__syncthreads();
	fence_after();
	const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
	const int dc = (a.c.d + 63) / 64, vc = (a.c.dv + 63) / 64, P = 1 << a.c.shift, W = min(P, KT), per = KT / W;
	const int h = warp < 4 ? warp - 1 : (warp - 4) >> 2; // the half of a warp that has one
	const int quad = warp & 3;                           // which lanes of tensor memory a softmax warp may read
	const uint32_t lanes = (uint32_t) (quad * 32) << 16, t_o = tmem + 256 + 128 * h;
	const bool negative = a.scale < 0.f;
	const float c1 = a.scale == 0.f ? 1e-30f : fabsf(a.scale) * 1.4426950408889634f; // a negative scale turns the scores' signs
	Walk k;
	// tiles of the CTA, tiles and pieces of this warp's half so far
	int n = 0, done = 0, pieces = 0;
	bool ok = true;
	bool more = walk_begin(a, part, plan, k);
	if (tid == 96) write_head(a, part, k, more, more && k.x.seg >= a.b.n_groups && k.x.key0 == 0, plan.share); // a warp with nothing else to do
	for (; more && (ok || warp >= 4); more = walk_next(a, part, plan, k)) { // softmax warps meet at barriers: they go on to the end whatever happens, and wait for nothing once a wait has given up
		const Piece& x = k.x;
		if (x.j0 == x.j1) continue;
		const TcPiece p = tc_piece(a, plan, x);
		const int tiles = max(p.j1 - x.j0, 0);
		const bool here = h >= 0 && h * HALF_ROWS < p.rows;
		if (warp == 0) { // ---- copies: 32 boxes' pages in one asking, then one thread sends them ----
			const int batch = 32 / per, key0 = x.key0, g = x.g;
			for (int j = 0; j < tiles && ok; j += batch) {
				const int at = (x.j0 + j) * KT + lane * W;
				int id = -1;
				if (at < p.most) {
					id = page_of(a.c, a.b, x.s, (key0 + at) >> a.c.shift);
					if (id < 0) report(a.c, ERR_PAGE);
				}
				sh.ids[lane] = id;
				__syncwarp();
				if (elect())
					for (int i = 0; i < min(batch, tiles - j); i++) {
						const int m = n + j + i, st = m % RING, slot = (key0 + (x.j0 + j + i) * KT) & (P - 1);
						if (!(ok = wait_alone(&sh.empty[st], ((m / RING) & 1) ^ 1, &sh.state, a.c))) break;
						mbar_expect_tx(&sh.full[st], (uint32_t) ((dc + vc) * KB));
						copy_tile(smem_u32(s_k) + st * 2 * KB, &kmap, a.c.d, g, slot, per, W, sh.ids + i * per, a.c.pages, &sh.full[st]);
						copy_tile(smem_u32(s_v) + st * 2 * KB, &vmap, a.c.dv, g, slot, per, W, sh.ids + i * per, a.c.pages, &sh.full[st]);
						sh.sent = m + 1;
					}
				ok = __all_sync(0xffffffffu, ok);
			}
		} else if (warp <= 2) { // ---- products: one thread issues them, with nothing to compute but two additions to a descriptor ----
			if (here && tiles) {
				__syncwarp();
				if (elect()) { // not `lane == 0`: in a branch that the compiler cannot tell to be one thread's, it does not keep the operands of unrolled products apart
					const uint32_t id_s = instr<T>(KT, false), id_o = instr<T>((a.c.dv + 15) / 16 * 16, true), t_s = tmem + 128 * h;
					const uint64_t q = desc_k(smem_u32(s_q)) + h * (2 * QB >> 4), k_at = desc_k(smem_u32(s_k)), v_at = desc_mn(smem_u32(s_v), KB);
					ok = wait_alone(&sh.q_full[h], pieces & 1, &sh.state, a.c);
					for (int j = -1; j < tiles && ok; j++) { // the scores of tile j + 1, then the second product of tile j
						const int m = n + j, c = done + j;
						if (j + 1 < tiles) {
							if (!(ok = wait_alone(&sh.full[(m + 1) % RING], ((m + 1) / RING) & 1, &sh.state, a.c))) break;
							// Their buffer holds the P of the product before: only products into one accumulator are sure to follow one another, so its end is waited for
							if (j > 0 && !(ok = wait_alone(&sh.o_full[h][(c - 1) & 1], ((c - 1) >> 1) & 1, &sh.state, a.c))) break;
							fence_after();
							const uint64_t kk = k_at + ((m + 1) % RING) * (2 * KB >> 4);
							const uint32_t d = t_s + 64 * ((c + 1) & 1);
#pragma unroll
							for (int s = 0; s < 4; s++) mma_ss(d, q + 2 * s, kk + 2 * s, id_s, s != 0); // queries are zeros behind the head's last entry, and so are keys
							if (dc > 1)
#pragma unroll
								for (int s = 0; s < 4; s++) mma_ss(d, q + (QB >> 4) + 2 * s, kk + (KB >> 4) + 2 * s, id_s, 1);
							commit(&sh.s_full[h][(c + 1) & 1]);
						}
						if (j < 0) continue;
						if (!(ok = wait_alone(&sh.p_full[h][c & 1], (c >> 1) & 1, &sh.state, a.c))) break;
						fence_after();
						const uint64_t v = v_at + (m % RING) * (2 * KB >> 4);
						const uint32_t prob = t_s + 64 * (c & 1);
#pragma unroll
						for (int s = 0; s < KT / 16; s++) mma_ts(t_o, prob + 8 * s, v + s * (2048 >> 4), id_o, j != 0 || s != 0);
						commit(&sh.o_full[h][c & 1]);
						commit(&sh.empty[m % RING]);
					}
				}
			} else if (lane == 0) // no rows in this half: the tiles are let go one by one all the same, so that this warp does not get ahead of their barriers' phases
				for (int j = n; j < n + tiles && ok; j++)
					if ((ok = wait_alone(&sh.full[j % RING], (j / RING) & 1, &sh.state, a.c))) mbar_arrive(&sh.empty[j % RING]);
			ok = __all_sync(0xffffffffu, ok);
		} else if (warp >= 4 && here) { // ---- softmax ----
			const int r = quad * 32 + lane, wt = tid & 127, row = h * HALF_ROWS + r, first = x.t * TC_ROWS + h * HALF_ROWS; // row of the half, of the unit; the half's first row of the segment
			const bool direct = x.j0 == 0 && x.j1 == x.w && !p.prefix && x.key0 == 0, mine = row < p.rows;
			const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
			const int row0 = x.row0, head0 = x.g * a.rep;
			float m = -INFINITY, l = 0.f;
			int lim = p.most, least = p.most;
			if (!p.prefix) {
				least = own_keys(x.q, x.key0, a.rep, first);
				lim = own_keys(x.q, x.key0, a.rep, min(first + r, x.t * TC_ROWS + p.rows - 1));
			}
			if (tiles) {
				if (HALF_ROWS % a.rep == 0) { // whole tokens: the copy engine brings them, those of other sequences behind the last too (rows that nobody asks for)
					asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // what the piece before has laid there on its way out
					bar_sync(2 + h, 128);
					if (wt < 32 && elect() && !*(volatile int*) &sh.state.dead) {
						mbar_expect_tx(&sh.q_full[h], (uint32_t) (dc * QB));
						for (int i = 0; i < dc; i++)
							asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(s_q + (h * 2 + i) * QB)),
							             "l"(&qmap), "r"(i * 64), "r"(0), "r"(row0 + first / a.rep), "r"(x.g), "r"(smem_u32(&sh.q_full[h]))
							             : "memory");
					}
				} else {
#pragma unroll 1
					for (int i = lane; i < 32 * dc * 8; i += 32) { // 16 bytes of one of this warp's rows
						const int rr = quad * 32 + i / (dc * 8), ch = i % (dc * 8), w = first + rr, tok = w / a.rep;
						uint4 v = make_uint4(0, 0, 0, 0);
						if (h * HALF_ROWS + rr < p.rows && ch * 8 < a.c.d) v = *reinterpret_cast<const uint4*>(a.q + ((long long) (row0 + tok) * a.q_row + (head0 + w - tok * a.rep) * a.c.d + ch * 8) * 2);
						*reinterpret_cast<uint4*>(s_q + (h * 2 + (ch >> 3)) * QB + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) = v;
					}
					asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
					bar_sync(2 + h, 128);
					if (wt == 0) mbar_arrive(&sh.q_full[h]);
				}
			}
			for (int j = 0; j < tiles; j++) {
				const int c = done + j, b = c & 1, base = (x.j0 + j) * KT;
				const uint32_t t_s = tmem + 128 * h + 64 * b + lanes;
				ok = wait_for(&sh.s_full[h][b], (c >> 1) & 1, &sh.state, a.c) && ok;
				fence_after();
				uint32_t s[KT];
				ld32(t_s, s);
				ld32(t_s + 32, s + 32);
				if (base + KT > p.most) { // slots that no row sees may hold anything: as zeros they add nothing
					const int st = (n + j) % RING;
					ok = wait_for(&sh.full[st], ((n + j) / RING) & 1, &sh.state, a.c) && ok;
					for (int i = wt; i < (base + KT - p.most) * vc * 8; i += 128) {
						const int rr = p.most - base + i / (vc * 8), cc = i % (vc * 8);
						*reinterpret_cast<uint4*>(s_v + (st * 2 + (cc >> 3)) * KB + rr * 128 + ((cc & 7) << 4)) = make_uint4(0, 0, 0, 0);
					}
					asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
				}
				__syncwarp();
				wait_ld(s);
				wait_ld(s + 32);
				if (negative) {
#pragma unroll
					for (int i = 0; i < KT; i++) s[i] ^= 0x80000000u;
				}
				if (base + KT > least) {
#pragma unroll
					for (int i = 0; i < KT; i++)
						if (base + i >= lim) s[i] = 0xff800000u;
				}
				float m8[8]; // eight chains: one of 64 would be waited for link by link
#pragma unroll
				for (int i = 0; i < 8; i++) m8[i] = __uint_as_float(s[i]);
#pragma unroll
				for (int i = 8; i < KT; i++) m8[i & 7] = fmaxf(m8[i & 7], __uint_as_float(s[i]));
				float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
				mx *= c1;
				const bool grow = mx > m + Lift<T>::LAG;
				if (j == 0) m = mx;
				else if (__any_sync(0xffffffffu, grow)) { // rare: the sums so far are complete before they are rescaled
					ok = wait_for(&sh.o_full[h][(c - 1) & 1], ((c - 1) >> 1) & 1, &sh.state, a.c) && ok;
					fence_after();
					const float to = grow ? mx : m, f = grow ? (m == -INFINITY ? 0.f : exp2_approx(m - to)) : 1.f;
#pragma unroll 1
					for (int i0 = 0; i0 < a.c.dv; i0 += 32) {
						uint32_t o[32];
						ld32(t_o + lanes + i0, o);
						wait_ld(o);
#pragma unroll
						for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
						st32(t_o + lanes + i0, o);
						wait_st();
					}
					l *= f;
					m = to;
				}
				const float nm = m == -INFINITY ? 0.f : Lift<T>::BY - m;
				const f32x2 c2 = pack2(c1, c1), n2 = pack2(nm, nm);
				f32x2 sum[4] = {pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f), pack2(0.f, 0.f)};
				uint32_t q[KT / 2];
#pragma unroll
				for (int i = 0; i < KT / 2; i++) { // two at a time where there is an instruction for two
					float p0, p1;
					unpack2(fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, n2), p0, p1);
					p0 = exp2_approx(p0);
					p1 = exp2_approx(p1);
					sum[i & 3] = add2(sum[i & 3], pack2(p0, p1));
					if constexpr (std::is_same<T, __half>::value) q[i] = probs_f16(p0, p1);
					else q[i] = pair16<T>(p0, p1);
				}
				{
					float e, o;
					unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), e, o);
					l += e + o;
				}
				st32(t_s, q);
				wait_st();
				fence_before();
				__syncwarp();
				if (lane == 0) mbar_arrive(&sh.p_full[h][b]);
			}
			// ---- the piece's sums: 32 columns at a time through this warp's rows of Q, which no product reads any more, so that what is written lies side by side ----
			if (tiles) ok = wait_for(&sh.o_full[h][(done + tiles - 1) & 1], ((done + tiles - 1) >> 1) & 1, &sh.state, a.c) && ok;
			fence_after();
			bool again = false;
			uint8_t* stage = s_q + h * 2 * QB + quad * 32 * 128; // 32 rows of 128 bytes
			const bool any = l > 0.f || l != l;
			const float inv = direct ? (any ? 1.f / l : 0.f) : 1.f;
			m -= Lift<T>::BY;
			if (mine) {
				if (!direct) {
					if (slot < part.slots) part.ml[slot * TC_ROWS + row] = make_float2(m, l);
				} else if (a.lse) {
					const int w = first + r, tok = w / a.rep;
					a.lse[(long long) (row0 + tok) * a.H + head0 + w - tok * a.rep] = any ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
				}
			}
			// where the rows go that this lane writes: four rows at a time, eight lanes to a row
			const int left = p.rows - h * HALF_ROWS - quad * 32 - (lane >> 3), ch = lane & 7;
#pragma unroll 1
			for (int c0 = 0; c0 < a.c.dv; c0 += 32) {
				uint32_t o[32];
#pragma unroll
				for (int i = 0; i < 32; i++) o[i] = 0;
				if (tiles) {
					ld32(t_o + lanes + c0, o);
					wait_ld(o);
				}
#pragma unroll
				for (int i = 0; i < 8; i++) {
					float4 v = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
					const float sum = fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w);
					again = again || (c0 + i * 4 < a.c.dv && !(sum <= 3.0e38f));
					if (direct) { v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv; }
					*reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = v;
				}
				__syncwarp();
				const int col = c0 + ch * 4;
				if (direct) {
#pragma unroll 1
					for (int i = 0; i < 8; i++) {
						const int rr = i * 4 + (lane >> 3), w = first + quad * 32 + rr, tok = w / a.rep;
						const float4 v = *reinterpret_cast<const float4*>(stage + rr * 128 + ((ch ^ (rr & 7)) << 4));
						if (4 * i < left && col < a.c.dv)
							*reinterpret_cast<uint2*>(a.out + ((long long) (row0 + tok) * a.out_row + (head0 + w - tok * a.rep) * a.c.dv + col) * 2) = make_uint2(pair16<T>(v.x, v.y), pair16<T>(v.z, v.w));
					}
				} else if (slot < part.slots) {
					float* po = part.o + (slot * TC_ROWS + h * HALF_ROWS + quad * 32 + (lane >> 3)) * a.c.dv + col;
#pragma unroll 2
					for (int i = 0; i < 8; i++) {
						const int rr = i * 4 + (lane >> 3);
						const float4 v = *reinterpret_cast<const float4*>(stage + rr * 128 + ((ch ^ (rr & 7)) << 4));
						if (4 * i < left && col < a.c.dv) *reinterpret_cast<float4*>(po + i * 4 * a.c.dv) = v;
					}
				}
				__syncwarp();
			}
			fence_before();
			if constexpr (std::is_same<T, __half>::value) {
				const bool fix = again && mine && l == l && tiles && ok; // not where a score is NaN: all columns are
				if (__any_sync(0xffffffffu, fix)) {
					const Piece y = x;
					if (lane == 0) atomicAdd(&sh.state.busy, 1);
					put_infinities(a, part, y, row, lim, p.most, fix);
					if (lane == 0) atomicAdd(&sh.state.busy, -1);
				}
			}
			if (!p.prefix && tiles && x.j1 * KT > least && least < p.most) {
				// A value that is not finite and that only later rows see has met probabilities of zero: rows that do not see it are done again, key by key
				if (wt == 0) sh.flag[h] = 0;
				bar_sync(2 + h, 128);
				if (again && mine && ok) sh.flag[h] = 1;
				bar_sync(2 + h, 128);
				const bool redo = *(volatile int*) &sh.flag[h] != 0;
				bar_sync(2 + h, 128);
				const Piece y = x; // in memory only here
				if (redo) redo_rows<T, TC_ROWS, HALF_ROWS>(a, part, y, h * HALF_ROWS, &sh.state, &sh.flag[h], sh.buf[h], wt, 2 + h);
			}
		}
		n += tiles;
		if (here) done += tiles;
		pieces += here && tiles;
	}
	fence_before();
	__syncthreads();
	if (*(volatile int*) &sh.state.dead) { // a wait gave up: what is still on its way into shared or tensor memory ends first
		if (warp == 0)
			for (int i = max(0, sh.sent - RING); i < sh.sent; i++) wait_some(&sh.full[i % RING], (i / RING) & 1, &sh.state);
		if (warp == 1 || warp == 2) {
			if (elect()) {
				commit(&sh.drained[h]);
				wait_some(&sh.drained[h], 0, &sh.state);
				if (pieces) wait_some(&sh.q_full[h], (pieces - 1) & 1, &sh.state);
			}
			__syncwarp();
		}
		__syncthreads();
	}
	if (warp == 1) {
		fence_after();
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
	}
}

static size_t tc_smem(const BatchView& b) { return 1024 + 4 * QB + 4 * RING * KB + sizeof(TcShared) + plan_bytes(b.B, b.n_groups); }
bool tc_fits(const Cache& c, const BatchView& b) { return c.d <= 128 && c.dv <= 128 && tc_smem(b) <= 226 * 1024; }

template <typename T>
static int launch_typed(const Attn& a, int part, int type, cudaStream_t s) {
	CUtensorMap kmap, vmap, qmap;
	XALM_TRY(pool_map(a.c, type, true, &kmap));
	XALM_TRY(pool_map(a.c, type, false, &vmap));
	{ // (entries, heads of a kv head, tokens, kv heads): 64 entries of 128 rows
		const int tokens = HALF_ROWS % a.rep == 0 ? HALF_ROWS / a.rep : 1;
		const cuuint64_t dims[4] = {(cuuint64_t) a.c.d, (cuuint64_t) a.rep, (cuuint64_t) a.b.N, (cuuint64_t) a.c.G};
		const cuuint64_t strides[3] = {(cuuint64_t) a.c.d * 2, (cuuint64_t) a.q_row * 2, (cuuint64_t) a.rep * a.c.d * 2};
		const cuuint32_t box[4] = {64, (cuuint32_t) (tokens > 1 || a.rep == HALF_ROWS ? a.rep : 1), (cuuint32_t) tokens, 1};
		XALM_TRY(encode_map(&qmap, type, 4, const_cast<uint8_t*>(a.q), dims, strides, box));
	}
	const size_t smem = tc_smem(a.b);
	XALM_CUDA_CHECK(allow_smem((const void*) paged_tc_kernel<T>));
	XALM_CUDA_CHECK(launch(paged_tc_kernel<T>, a.part[part].grid, TT, smem, s, false, a, a.part[part], kmap, vmap, qmap));
	return XALM_OK;
}
int launch_attn_tc(const Attn& a, int part, int type, cudaStream_t s) {
	return type == XALM_F16 ? launch_typed<__half>(a, part, type, s) : launch_typed<__nv_bfloat16>(a, part, type, s);
}

} // namespace paged
} // namespace xalm
