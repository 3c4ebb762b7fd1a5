// paged_attn.cu — attention over the paged cache: rows of fp32 caches by fp32 FMAs, and the join of what several CTAs have of the same rows.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// Attention by fp32 FMAs: up to 16 (token, head) rows of one kv head at a time, 32 keys at a time in shared memory.  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s = scale q.k;
// kept in log2 units: exp2((q.k - m') scale log2 e).  A tile's keys and values are on their way (16 bytes a copy, four threads to a key) while the tile before is worked on.
// A warp takes 8 of the 32 keys, with maximum, sum and output of its own, so that no warp waits for another inside a tile: scores by four lanes to a key, each every fourth 16 bytes of it;
// sums by four or eight neighbouring columns to a lane.  At the end of a piece the four join through shared memory.  Few rows (R = 4) are bound by latency, 16 by what shared memory
// delivers: 20 accesses to 64 FMAs of the scores, 8 to 64 of the sums.  Measured with 8 kv heads of 128: 16 sequences of 2500 tokens, four rows to a kv head, 79 us (4.2 TB/s), where a warp to
// four rows and all keys took 151; two prompts of 300 tokens behind 300 295 us (15 TFLOP/s): 255 registers leave eight warps to an SM.
// =========================================================================================================================================
constexpr int RM = 16, RK = 32, RT = 128, RW = RT / 32, WK = RK / RW; // keys of a warp
constexpr int RS = 20; // floats between a key's probabilities of 16 rows

__device__ __forceinline__ void copy16(float* dst, const float* src, bool there) { // zeros where there is nothing
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// A warp's 8 keys of a tile for R rows.  q: [R][d]; keys: [8][kp]; values: [8][dv], this lane's columns; sp: [8][RS] of the warp; lim: keys that the rows see, `base` before these
// COLS: 64, 128 or 256 columns of values; with 64 the lanes' halves take every other key
template <int R, int COLS>
__device__ __forceinline__ void rows_step(const float* q, const float* keys, const float* values, float* sp, const int* lim, int base, int n_keys, int d, int kp, int dv, int cols, float c1, int lane, float (&m)[R],
                                          float (&l)[R], float (&acc)[R][COLS == 256 ? 8 : 4]) {
	constexpr int C = COLS == 256 ? 2 : 1, BY = COLS == 64 ? 2 : 1;
	const int key = lane >> 2, part = (lane & 3) * 4;
	float s[R];
#pragma unroll
	for (int r = 0; r < R; r++) s[r] = 0.f;
#pragma unroll 2
	for (int c = part; c < d; c += 16) { // d is a multiple of 8: the last two lanes may have one step less
		const float4 k = *reinterpret_cast<const float4*>(keys + key * kp + c);
#pragma unroll
		for (int r = 0; r < R; r++) {
			const float4 x = *reinterpret_cast<const float4*>(q + r * d + c);
			s[r] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, s[r]))));
		}
	}
	bool grow = false;
#pragma unroll
	for (int r = 0; r < R; r++) {
		s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
		s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
		s[r] = base + key < lim[r] ? s[r] * c1 : -INFINITY;
		grow = grow || s[r] > m[r] + 8.f;
	}
	if (__any_sync(0xffffffffu, grow)) { // rare behind the first keys: probabilities may be up to 2^8
#pragma unroll
		for (int r = 0; r < R; r++) {
			float t = s[r];
#pragma unroll
			for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
			t = fmaxf(m[r], t);
			const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - t);
			l[r] *= f;
#pragma unroll
			for (int c = 0; c < 4 * C; c++) acc[r][c] *= f;
			m[r] = t;
		}
	}
	float p[R];
#pragma unroll
	for (int r = 0; r < R; r++) {
		p[r] = exp2f(s[r] - (m[r] == -INFINITY ? 0.f : m[r]));
		l[r] += p[r]; // of this lane's keys, four times each
	}
	__syncwarp();
	if ((lane & 3) == 0)
#pragma unroll
		for (int r = 0; r < R; r += 4) *reinterpret_cast<float4*>(sp + key * RS + r) = make_float4(p[r], p[r + 1], p[r + 2], p[r + 3]);
	__syncwarp();
	auto add = [&](int j, bool all) {
		float4 v[C];
#pragma unroll
		for (int c = 0; c < C; c++) v[c] = c * 128 < cols ? *reinterpret_cast<const float4*>(values + j * dv + c * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
		for (int r = 0; r < R; r += 4) {
			const float4 p4 = *reinterpret_cast<const float4*>(sp + j * RS + r);
			const float x[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
			for (int e = 0; e < 4; e++)
				if (all || base + j < lim[r + e]) {
#pragma unroll
					for (int c = 0; c < C; c++) {
						acc[r + e][4 * c] = fmaf(x[e], v[c].x, acc[r + e][4 * c]);
						acc[r + e][4 * c + 1] = fmaf(x[e], v[c].y, acc[r + e][4 * c + 1]);
						acc[r + e][4 * c + 2] = fmaf(x[e], v[c].z, acc[r + e][4 * c + 2]);
						acc[r + e][4 * c + 3] = fmaf(x[e], v[c].w, acc[r + e][4 * c + 3]);
					}
				}
		}
	};
	if (cols <= 0) return; // these lanes have no columns
	if (n_keys == WK && base + WK <= lim[0]) { // every row sees every key (rows that are not there see none, and are not written)
#pragma unroll
		for (int j = 0; j < WK; j += BY) add(j + (BY > 1 ? lane >> 4 : 0), true);
	} else // what a row does not see may be anything, an infinity or a NaN too
#pragma unroll 1
		for (int j = BY > 1 ? lane >> 4 : 0; j < n_keys; j += BY) add(j, false);
}
// Floats between keys: d, and then 16 modulo 32, so that two keys' 64 bytes share no bank
__host__ __device__ __forceinline__ int key_pitch(int d) { return d + (48 - d % 32) % 32; }

template <int COLS, bool LIST>
__global__ void __launch_bounds__(RT) paged_rows_kernel(const __grid_constant__ Attn a, const int buffers) {
	extern __shared__ __align__(16) uint8_t smem[];
	constexpr int C = COLS == 256 ? 2 : 1;
	const Part& part = a.part[0];
	const int d = a.c.d, dv = a.c.dv, kp = key_pitch(d), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int tile = RK * (kp + dv);                      // floats of a tile
	float* sq = reinterpret_cast<float*>(smem);           // [RM][d]
	float* st = sq + RM * d;                              // [buffers] of [RK][kp] keys and [RK][dv] values; then the warps' sums [RW][rows][dv]
	float* sp = st + max(buffers * tile, RW * RM * dv);   // [RK][RS]
	float2* s_ml = reinterpret_cast<float2*>(sp + RK * RS); // [RW][RM]
	int* s_lim = reinterpret_cast<int*>(s_ml + RW * RM);  // [RM] keys that a row sees
	int* s_list = s_lim + RM;                             // [S]
	uint8_t* s_plan = reinterpret_cast<uint8_t*>(s_list + ((LIST ? a.S : 0) + 1) / 2 * 2);
	Plan plan;
	pdl_wait();
	pdl_launch_dependents();
	if (!LIST) make_plan<RT>(a, part, s_plan, plan);
	else if (blockIdx.x == 0) check_seqs(a.c, a.b, tid, RT);
	Walk k;
	bool more = LIST ? list_begin(a, part, k) : walk_begin(a, part, plan, k);
	if (tid == 0)
		write_head(a, part, k, more, LIST ? more && row_in_seq(k.x.q, k.x.row0) : more && k.x.seg >= a.b.n_groups && k.x.key0 == 0, LIST ? share_of(list_total(a, part), part.grid) : plan.share);
	const int col0 = (COLS == 64 ? lane & 15 : lane) * 4; // this lane's columns of values
	const int key_of = tid >> 2, P = 1 << a.c.shift; // this thread's key of a tile, of which it brings every fourth 16 bytes
	constexpr int NONE = -0x7fffffff;
	for (; more; more = LIST ? list_next(a, part, k) : walk_next(a, part, plan, k)) {
		const Piece& x = k.x;
		if (x.j0 == x.j1) continue; // the same for every thread
		__syncthreads();
		int pos = 0, listed = 0;
		if (LIST) {
			if (!row_in_seq(x.q, x.row0)) continue;
			pos = x.q.len - x.q.n + x.row0 - x.q.a;
			bool own;
			const int n = list_pages(a, x.row0, x.g, pos >= 0 ? pos >> a.c.shift : -1, warp == 0 ? s_list : nullptr, &own);
			listed = own ? ((n - 1) << a.c.shift) + (pos & (P - 1)) + 1 : n << a.c.shift;
		}
		const int shared = LIST ? 0 : plan.shs[x.s];
		const bool prefix = !LIST && x.seg < a.b.n_groups;
		const int rows = min(RM, x.rows - x.t * RM);
		const int h0 = x.g * a.rep;
		auto keys_of = [&](int r) { return LIST ? listed : prefix ? shared : own_keys(x.q, shared, a.rep, x.t * RM + r); };
		if (tid < RM) s_lim[tid] = tid >= rows ? 0 : keys_of(tid);
		if (LIST) __syncthreads();
		const int first = x.j0 * KT, last = min(x.j1 * KT, keys_of(rows - 1)); // the last row sees the most
		auto page_at = [&](int kb) { // what the table has for this thread's key of the tile at kb, looked at when the tile is copied
			if (kb + key_of >= last) return NONE;
			const int key = x.key0 + kb + key_of, at = LIST ? s_list[key >> a.c.shift] : key >> a.c.shift;
			return a.b.table[(long long) x.s * a.b.table_row + at];
		};
		auto copy = [&](int kb, int page, float* to) {
			const bool there = page >= 0 && page < a.c.pages;
			if (!there && page != NONE) report(a.c, ERR_PAGE);
			const long long pg = there ? page : 0, slot = there ? (x.key0 + kb + key_of) & (P - 1) : 0;
			const float* kk = reinterpret_cast<const float*>(a.c.k) + pg * a.c.k_page + slot * a.c.k_slot + x.g * a.c.k_head;
			const float* vv = reinterpret_cast<const float*>(a.c.v) + pg * a.c.v_page + slot * a.c.v_slot + x.g * a.c.v_head;
#pragma unroll 4
			for (int c = (tid & 3) * 4; c < d; c += 16) copy16(to + key_of * kp + c, kk + c, there);
#pragma unroll 4
			for (int c = (tid & 3) * 4; c < dv; c += 16) copy16(to + RK * kp + key_of * dv + c, vv + c, there);
			asm volatile("cp.async.commit_group;" ::: "memory");
		};
		int page = page_at(first);
		for (int i = tid; i < RM * (d / 4); i += RT) {
			const int r = i / (d / 4), c = i % (d / 4) * 4;
			float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
			if (r < rows) {
				const int w = x.t * RM + r;
				v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + (long long) (x.row0 + w / a.rep) * a.q_row + (h0 + w % a.rep) * d + c);
			}
			*reinterpret_cast<float4*>(sq + r * d + c) = v;
		}
		copy(first, page, st);
		page = page_at(first + RK);
		const float c1 = a.scale * 1.4426950408889634f;
		auto run = [&](auto of) {
			constexpr int R = decltype(of)::value;
			float m[R], l[R], acc[R][4 * C];
#pragma unroll
			for (int r = 0; r < R; r++) {
				m[r] = -INFINITY;
				l[r] = 0.f;
#pragma unroll
				for (int c = 0; c < 4 * C; c++) acc[r][c] = 0.f;
			}
			float* now = st;
			for (int kb = first; kb < last; kb += RK) {
				asm volatile("cp.async.wait_group 0;" ::: "memory");
				__syncthreads(); // the tile is there, and nobody reads the one before any more
				float* next = buffers == 1 || now != st ? st : st + tile;
				if (buffers > 1) copy(kb + RK, page, next);
				page = page_at(kb + (buffers > 1 ? 2 : 1) * RK);
				const int base = kb + warp * WK;
				if (base < last)
					rows_step<R, COLS>(sq, now + warp * WK * kp, now + RK * kp + warp * WK * dv + col0, sp + warp * WK * RS, s_lim, base, min(WK, last - base), d, kp, dv, dv - col0, c1, lane, m, l, acc);
				if (buffers == 1) {
					__syncthreads();
					copy(kb + RK, page, next);
				}
				now = next;
			}
			asm volatile("cp.async.wait_group 0;" ::: "memory");
			__syncthreads();
#pragma unroll
			for (int r = 0; r < R; r++) {
#pragma unroll
				for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
				if (lane == 0) s_ml[warp * RM + r] = make_float2(m[r], l[r]);
				if (COLS == 64)
#pragma unroll
					for (int c = 0; c < 4; c++) acc[r][c] += __shfl_xor_sync(0xffffffffu, acc[r][c], 16);
#pragma unroll
				for (int c = 0; c < C; c++)
					if (c * 128 + col0 < dv) *reinterpret_cast<float4*>(st + (warp * R + r) * dv + c * 128 + col0) = make_float4(acc[r][4 * c], acc[r][4 * c + 1], acc[r][4 * c + 2], acc[r][4 * c + 3]);
			}
			return R;
		};
		const int R = rows <= 4 ? run(std::integral_constant<int, 4>()) : rows <= 8 ? run(std::integral_constant<int, 8>()) : run(std::integral_constant<int, 16>());
		__syncthreads();
		const bool direct = x.j0 == 0 && x.j1 == x.w && !prefix && shared == 0;
		const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
		for (int i = tid; i < rows * (dv / 4); i += RT) {
			const int row = i / (dv / 4), col = i % (dv / 4) * 4, w = x.t * RM + row;
			float mx = -INFINITY, l = 0.f;
			float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
			for (int e = 0; e < RW; e++) mx = fmaxf(mx, s_ml[e * RM + row].x);
#pragma unroll
			for (int e = 0; e < RW; e++) {
				const float2 ml = s_ml[e * RM + row];
				const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mx); // times 0 a NaN stays one
				const float4 o = *reinterpret_cast<const float4*>(st + (e * R + row) * dv + col);
				l += ml.y * f;
				v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
			}
			const bool any = l > 0.f || l != l;
			if (direct) {
				const float f = any ? 1.f / l : 0.f; // 0: a row that sees nothing, whose sums are zeros
				*reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + (long long) (x.row0 + w / a.rep) * a.out_row + (h0 + w % a.rep) * dv + col) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
				if (a.lse && col == 0) a.lse[(long long) (x.row0 + w / a.rep) * a.H + h0 + w % a.rep] = any ? (mx + log2f(l)) * 0.6931471805599453f : -INFINITY;
			} else if (slot < part.slots) {
				*reinterpret_cast<float4*>(part.o + (slot * RM + row) * dv + col) = v;
				if (col == 0) part.ml[slot * RM + row] = make_float2(mx, l);
			}
		}
	}
}

// =========================================================================================================================================
// The join of what several CTAs have of the same rows, a warp to a row.  A lane takes a piece's maximum and sum, then the pieces' rows are added with their weights, eight
// loads on their way at a time.  Two kinds of blocks: with groups, for rows that read shared pages; and for 16 rows
// of the units that a CTA's share begins inside (four to a warp, which for five long prompts take 143 us of all in place of 149).  Bound by the latency of three or four loads that depend on one another:
// 2048 rows of 128 entries in 12 us.
// =========================================================================================================================================
constexpr int JT = 128, JR = 16;

struct JoinUnit {
	int part, unit, at, cta, n; // which part, unit, row of the unit, first CTA, CTAs
};
// The unit of row `idx` of a segment: where its pieces lie
__device__ __forceinline__ bool join_unit(const Attn& a, const View& v, int i, int seg, int s_first, int idx, int g, JoinUnit& o) {
	const Part& p = a.part[i];
	int row0, s;
	const int rows = seg_rows(v, a.rep, seg, row0, s);
	const int total = p.cum_w[a.b.n_groups + a.b.B], seg_at = p.cum_w[seg], seg_w = p.cum_w[seg + 1] - seg_at;
	const int sh = p.shs[s_first], u0 = p.cum_u[seg];
	if (!in_part(p, rows) || !seg_w) return false;
	const int tiles = (rows + p.M - 1) / p.M, t = idx / p.M, lane = threadIdx.x & 31;
	if (idx < 0 || idx >= rows) return false;
	const Seq q = seq_of(v, s_first);
	const int w = unit_tiles(a, p, seg, rows, q, sh, t);
	if (!w) return false;
	int before = 0;
	if (t) {
		for (int j = lane; j < t; j += 32) before += unit_work(a, p, seg, rows, q, sh, j);
		before = __reduce_add_sync(0xffffffffu, before);
	}
	const int share = share_of(total, p.grid), w0 = seg_at + seg_w / a.c.G * g + before + p.lead;
	o.unit = u0 + g * tiles + t;
	o.cta = w0 / share;
	o.n = (w0 + w - 1) / share - o.cta + 1;
	o.part = i;
	o.at = idx - t * p.M;
	return true;
}

template <typename T, int NC> // NC x 128 columns
__device__ __forceinline__ void join_row(const Attn& a, const JoinUnit (&u)[2], int found, int row, int h) {
	const int lane = threadIdx.x & 31, dv = a.c.dv;
	const int n0 = found ? u[0].n : 0, n = n0 + (found > 1 ? u[1].n : 0); // pieces
	float m = -INFINITY;
	bool nan = false;
	auto piece = [&](int i, const float*& o) { // the i-th piece's maximum and sum, and where its row lies
		const JoinUnit& x = i < n0 ? u[0] : u[1];
		const Part& p = a.part[x.part];
		const int c = i < n0 ? i : i - n0;
		const long long slot = piece_slot(a, x.unit, x.cta + c, c == 0);
		float2 ml = make_float2(-INFINITY, 0.f);
		if (slot < p.slots) {
			ml = p.ml[slot * p.M + x.at];
			o = p.o + (slot * p.M + x.at) * dv;
		}
		return ml;
	};
	const float* o = a.part[0].o;
	for (int i = lane; i < n; i += 32) {
		const float2 ml = piece(i, o);
		nan = nan || ml.x != ml.x;
		m = fmaxf(m, ml.x);
	}
	m = warp_max(m);
	nan = __any_sync(0xffffffffu, nan);
	const float base = nan ? NAN : m == -INFINITY ? 0.f : m;
	float l = 0.f, acc[4 * NC];
#pragma unroll
	for (int i = 0; i < 4 * NC; i++) acc[i] = 0.f;
	for (int i0 = 0; i0 < n; i0 += 32) {
		float wgt = 0.f;
		bool some = false;
		const float* row_at = a.part[0].o;
		if (i0 + lane < n) {
			const float2 ml = piece(i0 + lane, row_at);
			some = ml.x != -INFINITY || ml.y != 0.f; // else nothing that the row sees
			wgt = !some || ml.x == -INFINITY ? 0.f : exp2f(ml.x - base);
			if (some) l += ml.y * wgt; // a sum that is NaN stays one
		}
		for (unsigned left = __ballot_sync(0xffffffffu, some); left;) {
			constexpr int NB = 8 / NC;
			float4 x[NB][NC];
			float f[NB];
#pragma unroll
			for (int j = 0; j < NB; j++) {
				const bool one = left != 0;
				const int from = one ? __ffs(left) - 1 : 0;
				left &= left - 1;
				f[j] = __shfl_sync(0xffffffffu, wgt, from);
				const float* at = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row_at), from));
				if (!one) f[j] = 0.f;
#pragma unroll
				for (int c = 0; c < NC; c++)
					x[j][c] = one && c * 128 + lane * 4 < dv ? *reinterpret_cast<const float4*>(at + c * 128 + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
			}
#pragma unroll
			for (int j = 0; j < NB; j++)
#pragma unroll
				for (int c = 0; c < NC; c++) {
					acc[4 * c] = fmaf(x[j][c].x, f[j], acc[4 * c]);
					acc[4 * c + 1] = fmaf(x[j][c].y, f[j], acc[4 * c + 1]);
					acc[4 * c + 2] = fmaf(x[j][c].z, f[j], acc[4 * c + 2]);
					acc[4 * c + 3] = fmaf(x[j][c].w, f[j], acc[4 * c + 3]);
				}
		}
	}
	l = warp_sum(l);
	const bool any = l > 0.f || l != l;
	const float inv = any ? 1.f / l : 0.f;
	T* out = reinterpret_cast<T*>(a.out) + (long long) row * a.out_row + h * dv;
#pragma unroll
	for (int c = 0; c < NC; c++)
		if (c * 128 + lane * 4 < dv) {
			T v[4];
#pragma unroll
			for (int e = 0; e < 4; e++) v[e] = from_f<T>(any ? acc[4 * c + e] * inv : 0.f);
			if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out + c * 128 + lane * 4) = *reinterpret_cast<const uint4*>(v);
			else *reinterpret_cast<uint2*>(out + c * 128 + lane * 4) = *reinterpret_cast<const uint2*>(v);
		}
	if (a.lse && lane == 0) a.lse[(long long) row * a.H + h] = any ? (base + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// Four neighbouring rows of a unit of up to eight pieces by a warp, eight lanes to a row's maxima and sums, four rows' loads on their way together.  at: rows of the unit; w: of the segment
template <typename T, int NC>
__device__ __forceinline__ void join_four(const Attn& a, const JoinUnit& u, int rows, int row0, int head0, int w) {
	const int lane = threadIdx.x & 31, mine = lane >> 3, c = lane & 7, dv = a.c.dv;
	const Part& p = a.part[u.part];
	auto slot_of = [&](int i) { return piece_slot(a, u.unit, u.cta + i, i == 0); };
	float2 ml = make_float2(-INFINITY, 0.f);
	if (mine < rows && c < u.n && slot_of(c) < p.slots) ml = p.ml[slot_of(c) * p.M + u.at + mine];
	const bool some = ml.x != -INFINITY || ml.y != 0.f; // else nothing that the row sees
	const unsigned there = __ballot_sync(0xffffffffu, some), nan = __ballot_sync(0xffffffffu, ml.x != ml.x);
	float m = ml.x;
#pragma unroll
	for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
	const float base = nan >> (mine * 8) & 0xff ? NAN : m == -INFINITY ? 0.f : m, wgt = !some || ml.x == -INFINITY ? 0.f : exp2f(ml.x - base);
	float l = some ? ml.y * wgt : 0.f; // a sum that is NaN stays one
#pragma unroll
	for (int o = 1; o < 8; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
	float4 acc[4][NC];
#pragma unroll
	for (int r = 0; r < 4; r++)
#pragma unroll
		for (int k = 0; k < NC; k++) acc[r][k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
	for (int i = 0; i < u.n; i++) {
		const float* o = p.o + (slot_of(i) * p.M + u.at) * dv + lane * 4;
		float4 x[4][NC];
#pragma unroll
		for (int r = 0; r < 4; r++)
#pragma unroll
			for (int k = 0; k < NC; k++)
				x[r][k] = (there >> (r * 8 + i) & 1) && k * 128 + lane * 4 < dv ? *reinterpret_cast<const float4*>(o + r * dv + k * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
		for (int r = 0; r < 4; r++) {
			const float f = __shfl_sync(0xffffffffu, wgt, r * 8 + i);
#pragma unroll
			for (int k = 0; k < NC; k++) {
				acc[r][k].x = fmaf(x[r][k].x, f, acc[r][k].x);
				acc[r][k].y = fmaf(x[r][k].y, f, acc[r][k].y);
				acc[r][k].z = fmaf(x[r][k].z, f, acc[r][k].z);
				acc[r][k].w = fmaf(x[r][k].w, f, acc[r][k].w);
			}
		}
	}
	const bool any = l > 0.f || l != l;
	const float inv = any ? 1.f / l : 0.f;
	if (a.lse && c == 0 && mine < rows) a.lse[(long long) (row0 + (w + mine) / a.rep) * a.H + head0 + (w + mine) % a.rep] = any ? (base + log2f(l)) * 0.6931471805599453f : -INFINITY;
#pragma unroll
	for (int r = 0; r < 4; r++) {
		const float f = __shfl_sync(0xffffffffu, inv, r * 8);
		T* out = reinterpret_cast<T*>(a.out) + (long long) (row0 + (w + r) / a.rep) * a.out_row + (head0 + (w + r) % a.rep) * dv + lane * 4;
#pragma unroll
		for (int k = 0; k < NC; k++)
			if (r < rows && k * 128 + lane * 4 < dv) {
				const float y[4] = {acc[r][k].x * f, acc[r][k].y * f, acc[r][k].z * f, acc[r][k].w * f};
				T v[4];
#pragma unroll
				for (int e = 0; e < 4; e++) v[e] = from_f<T>(f == 0.f ? 0.f : y[e]); // 0: a row that sees nothing
				if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out + k * 128) = *reinterpret_cast<const uint4*>(v);
				else *reinterpret_cast<uint2*>(out + k * 128) = *reinterpret_cast<const uint2*>(v);
			}
	}
}

// blocks of a part's boundaries: one to 16 rows of each
__host__ __device__ __forceinline__ int boundary_blocks(const Part& p) { return p.grid * (p.M > JR ? p.M / JR : 1); }

template <typename T, int NC>
__global__ void __launch_bounds__(JT) paged_join_kernel(const __grid_constant__ Attn a) {
	const int warp = threadIdx.x >> 5;
	int id = blockIdx.x;
	if (id < a.row_blocks) { // a warp to a (token, head) row
		const View v = view_of(a.c, a.b);
		const long long rows = (long long) a.b.N * a.H;
		bool waited = false;
		for (long long r = id * (JT / 32) + warp; r < rows; r += a.row_blocks * (JT / 32)) {
			const int tok = (int) (r / a.H), h = (int) (r - (long long) tok * a.H), g = h / a.rep;
			int s = 0, lo = 0; // its sequence and that one's group: the last that begin there or before
			for (int hi = a.b.B - 1; s < hi;) {
				const int mid = (s + hi + 1) >> 1;
				if (v.starts[mid] <= tok) s = mid;
				else hi = mid - 1;
			}
			for (int hi = a.b.n_groups - 1; lo < hi;) {
				const int mid = (lo + hi + 1) >> 1;
				if (v.bounds[mid] <= s) lo = mid;
				else hi = mid - 1;
			}
			const Seq q = seq_of(v, s);
			const int first = min(group_of(v, lo).x, a.b.B - 1), row0 = seq_of(v, first).a;
			if (!waited) pdl_wait(); // the caller's arrays were there already, the other kernels' are not
			waited = true;
			const int sh = a.part[0].shs[s], of_groups = a.part[0].cum_w[a.b.n_groups] | (a.n_parts > 1 ? a.part[1].cum_w[a.b.n_groups] : 0);
			if (!of_groups) return; // no group's pages are read once for all
			if (!row_in_seq(q, tok) || !sh) continue;
			JoinUnit u[2];
			int found = 0;
			for (int i = 0; i < a.n_parts && !found; i++) found = join_unit(a, v, i, lo, first, (tok - row0) * a.rep + h - g * a.rep, g, u[0]);
			const int had = found;
			for (int i = 0; i < a.n_parts && found == had; i++) found += join_unit(a, v, i, a.b.n_groups + s, s, (tok - q.a) * a.rep + h - g * a.rep, g, had ? u[1] : u[0]);
			join_row<T, NC>(a, u, found, tok, h);
		}
		return;
	}
	id -= a.row_blocks;
	pdl_wait();
	for (int i = 0; i < a.n_parts; i++) {
		const Part& p = a.part[i];
		const int blocks = boundary_blocks(p), chunks = blocks / p.grid;
		if (id >= blocks) {
			id -= blocks;
			continue;
		}
		const int cta = id / chunks;
		const Head x = p.head[cta];
		if (!x.j0 || x.j0 > x.share) return; // of the shares that begin inside a unit, the first joins it
		JoinUnit u[2];
		u[0].part = i;
		u[0].unit = x.u;
		u[0].cta = cta - 1;
		u[0].n = (x.share - x.j0 + x.w - 1) / x.share + 1;
		if (u[0].n <= 8) {
			const int r = (id - cta * chunks) * JR + warp * (JR / (JT / 32)), w = x.first + r;
			u[0].at = r;
			if (r < x.rows) join_four<T, NC>(a, u[0], min(4, x.rows - r), x.row0, x.g * a.rep, w);
			return;
		}
		for (int r = (id - cta * chunks) * JR + warp; r < min(x.rows, (id - cta * chunks) * JR + JR); r += JT / 32) {
			const int w = x.first + r, tok = w / a.rep;
			u[0].at = r;
			join_row<T, NC>(a, u, 1, x.row0 + tok, x.g * a.rep + w - tok * a.rep);
		}
		return;
	}
}

int launch_join(const Attn& a, int type, cudaStream_t s) {
	int grid = a.row_blocks;
	for (int i = 0; i < a.n_parts; i++) grid += boundary_blocks(a.part[i]);
	const bool wide = a.c.dv > 128;
	XALM_CUDA_CHECK(type == XALM_F32   ? (wide ? launch(paged_join_kernel<float, 2>, grid, JT, 0, s, true, a) : launch(paged_join_kernel<float, 1>, grid, JT, 0, s, true, a))
	                : type == XALM_F16 ? (wide ? launch(paged_join_kernel<__half, 2>, grid, JT, 0, s, true, a) : launch(paged_join_kernel<__half, 1>, grid, JT, 0, s, true, a))
	                                   : (wide ? launch(paged_join_kernel<__nv_bfloat16, 2>, grid, JT, 0, s, true, a) : launch(paged_join_kernel<__nv_bfloat16, 1>, grid, JT, 0, s, true, a)));
	return XALM_OK;
}

static size_t rows_smem(const Cache& c, const BatchView& b, int n_lists, int buffers) {
	return (size_t) (RM * c.d + std::max(buffers * RK * (key_pitch(c.d) + c.dv), RW * RM * c.dv) + RK * RS + 2 * RW * RM) * 4 + (RM + n_lists + 2) * 4 + 16 + (n_lists ? 0 : plan_bytes(b.B, b.n_groups));
}
// Two buffers where shared memory holds them, which it does not for the largest heads beside thousands of sequences; two CTAs to an SM where it holds those
static int rows_buffers(const Cache& c, const BatchView& b, int n_lists) { return rows_smem(c, b, n_lists, 2) <= 226 * 1024 ? 2 : 1; }
int rows_ctas_per_sm(const Cache& c, const BatchView& b, int n_lists) { return rows_smem(c, b, n_lists, rows_buffers(c, b, n_lists)) <= 113 * 1024 ? 2 : 1; }
template <int COLS>
static int rows_cols(const Attn& a, cudaStream_t s) {
	const int buffers = rows_buffers(a.c, a.b, a.S);
	const size_t smem = rows_smem(a.c, a.b, a.S, buffers);
	auto kernel = a.lists ? paged_rows_kernel<COLS, true> : paged_rows_kernel<COLS, false>;
	XALM_CUDA_CHECK(allow_smem((const void*) kernel));
	XALM_CUDA_CHECK(launch(kernel, a.part[0].grid, RT, smem, s, false, a, buffers));
	return XALM_OK;
}
int launch_attn_rows(const Attn& a, cudaStream_t s) { return a.c.dv <= 64 ? rows_cols<64>(a, s) : a.c.dv <= 128 ? rows_cols<128>(a, s) : rows_cols<256>(a, s); }

} // namespace paged
} // namespace xalm
