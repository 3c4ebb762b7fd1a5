// paged_attn.cu — attention over the paged cache: rows of fp32 caches by fp32 FMAs, and the join of what several CTAs have of the same rows.
#include "paged.cuh"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// Attention by fp32 FMAs: 16 (token, head) rows of one kv head at a time, 32 keys at a time in shared memory, one running maximum and
// sum per row.  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s = scale q.k; kept in log2 units: exp2((q.k - m') scale log2 e).
// A tile's keys and values are on their way (16 bytes a copy, four threads to a key) while the tile before is worked on.  Scores: a lane to a key, four rows to a warp.
// Sums: four neighbouring columns to a thread, CG threads side by side, the rows divided among the 128 / CG groups.  Few rows are bound by the latency of a tile's steps, many by
// what shared memory delivers: for 16 rows of 128 entries 1024 + 640 cycles a tile against 1024 of FMAs.
// =========================================================================================================================================
constexpr int RM = 16, RK = 32, RT = 128, RS = 20; // RS: floats between a key's probabilities, so that a warp's stores of four rows meet no bank twice

__device__ __forceinline__ void copy16(float* dst, const float* src, bool there) { // zeros where there is nothing
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int CG, bool LIST> // threads that share a value's columns
__global__ void __launch_bounds__(RT) paged_rows_kernel(const __grid_constant__ Attn a, const int buffers) {
	constexpr int RPT = RM * CG / RT; // rows of a thread's sums
	extern __shared__ __align__(16) uint8_t smem[];
	const Part& part = a.part[0];
	const int d = a.c.d, dv = a.c.dv, kp = d + 4, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int tile = RK * (kp + dv);                      // floats of a tile
	float* sq = reinterpret_cast<float*>(smem);           // [RM][d]
	float* st = sq + RM * d;                              // [buffers] of [RK][d + 4] keys and [RK][dv] values
	float* sp = st + buffers * tile;                      // [RK][RS]
	float* s_corr = sp + RK * RS;                         // [RM] factor of what a row has so far, then of its sum
	int* s_lim = reinterpret_cast<int*>(s_corr + RM);     // [RM] keys that a row sees
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
	const int cg = tid % CG, col = cg * 4, r0 = tid / CG * RPT;      // this thread's columns and rows
	const int key_of = tid >> 2, P = 1 << a.c.shift;                 // this thread's key of a tile, of which it brings every fourth 16 bytes
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
		auto page_at = [&](int kb) { // page of this thread's key of the tile at kb
			if (kb + key_of >= last) return -1;
			const int key = x.key0 + kb + key_of, pg = page_of(a.c, a.b, x.s, LIST ? s_list[key >> a.c.shift] : key >> a.c.shift);
			if (pg < 0) report(a.c, ERR_PAGE);
			return pg;
		};
		auto copy = [&](int kb, int pg, float* to) {
			const long long slot = (x.key0 + kb + key_of) & (P - 1);
			const float* kk = reinterpret_cast<const float*>(a.c.k) + (pg < 0 ? 0 : pg * a.c.k_page + slot * a.c.k_slot + x.g * a.c.k_head);
			const float* vv = reinterpret_cast<const float*>(a.c.v) + (pg < 0 ? 0 : pg * a.c.v_page + slot * a.c.v_slot + x.g * a.c.v_head);
#pragma unroll 4
			for (int c = (tid & 3) * 4; c < d; c += 16) copy16(to + key_of * kp + c, kk + c, pg >= 0);
#pragma unroll 4
			for (int c = (tid & 3) * 4; c < dv; c += 16) copy16(to + RK * kp + key_of * dv + c, vv + c, pg >= 0);
			asm volatile("cp.async.commit_group;" ::: "memory");
		};
		int page = page_at(first);
		copy(first, page, st);
		page = page_at(first + RK);
		for (int i = tid; i < RM * (d / 4); i += RT) {
			const int r = i / (d / 4), c = i % (d / 4) * 4;
			float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
			if (r < rows) {
				const int w = x.t * RM + r;
				v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + (long long) (x.row0 + w / a.rep) * a.q_row + (h0 + w % a.rep) * d + c);
			}
			*reinterpret_cast<float4*>(sq + r * d + c) = v;
		}
		float m[4], l[4], acc[RPT][4];
#pragma unroll
		for (int r = 0; r < 4; r++) { m[r] = -INFINITY; l[r] = 0.f; }
#pragma unroll
		for (int r = 0; r < RPT; r++)
#pragma unroll
			for (int c = 0; c < 4; c++) acc[r][c] = 0.f;
		const float c1 = a.scale * 1.4426950408889634f;
		const bool scores = warp * 4 < rows, sums = r0 < rows && col < dv;
		float* now = st;
		for (int kb = first; kb < last; kb += RK) {
			asm volatile("cp.async.wait_group 0;" ::: "memory");
			__syncthreads(); // the tile is there, and nobody reads the one before any more
			float* next = buffers == 1 || now != st ? st : st + tile;
			if (buffers > 1) copy(kb + RK, page, next);
			const int after = buffers > 1 ? page_at(kb + 2 * RK) : -1;
			if (scores) {
				float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
				for (int c = 0; c < d; c += 4) {
					const float4 kk = *reinterpret_cast<const float4*>(now + lane * kp + c);
#pragma unroll
					for (int r = 0; r < 4; r++) {
						const float4 qq = *reinterpret_cast<const float4*>(sq + (warp * 4 + r) * d + c);
						s[r] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, s[r]))));
					}
				}
				float p[4];
#pragma unroll
				for (int r = 0; r < 4; r++) {
					const float sc = kb + lane < s_lim[warp * 4 + r] ? s[r] * c1 : -INFINITY;
					const float mt = fmaxf(m[r], warp_max(sc)), base = mt == -INFINITY ? 0.f : mt, corr = exp2f(m[r] - base);
					p[r] = exp2f(sc - base);
					l[r] = l[r] * corr + p[r]; // of this lane's keys
					m[r] = mt;
					if (lane == 0) s_corr[warp * 4 + r] = corr;
				}
				*reinterpret_cast<float4*>(sp + lane * RS + warp * 4) = make_float4(p[0], p[1], p[2], p[3]);
			}
			__syncthreads();
			if (sums) {
				const int n_keys = min(RK, last - kb);
				const float* vv = now + RK * kp + col;
#pragma unroll
				for (int r = 0; r < RPT; r++) {
					const float f = s_corr[r0 + r];
#pragma unroll
					for (int c = 0; c < 4; c++) acc[r][c] *= f;
				}
				// rows that are not there see no key, and are not written
				if (kb + n_keys <= s_lim[0]) {
#pragma unroll 4
					for (int j = 0; j < RK; j++) { // values behind the last key are zeros, and so are their probabilities
						const float4 v = *reinterpret_cast<const float4*>(vv + j * dv);
#pragma unroll
						for (int r = 0; r < RPT; r++) {
							const float p = sp[j * RS + r0 + r];
							acc[r][0] = fmaf(p, v.x, acc[r][0]);
							acc[r][1] = fmaf(p, v.y, acc[r][1]);
							acc[r][2] = fmaf(p, v.z, acc[r][2]);
							acc[r][3] = fmaf(p, v.w, acc[r][3]);
						}
					}
				} else { // what a row does not see may be anything, an infinity or a NaN too
					for (int j = 0; j < n_keys; j++) {
						const float4 v = *reinterpret_cast<const float4*>(vv + j * dv);
#pragma unroll
						for (int r = 0; r < RPT; r++)
							if (kb + j < s_lim[r0 + r]) {
								const float p = sp[j * RS + r0 + r];
								acc[r][0] = fmaf(p, v.x, acc[r][0]);
								acc[r][1] = fmaf(p, v.y, acc[r][1]);
								acc[r][2] = fmaf(p, v.z, acc[r][2]);
								acc[r][3] = fmaf(p, v.w, acc[r][3]);
							}
					}
				}
			}
			if (buffers == 1) {
				__syncthreads();
				copy(kb + RK, page_at(kb + RK), next);
			}
			page = after;
			now = next;
		}
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		const bool direct = x.j0 == 0 && x.j1 == x.w && !prefix && shared == 0;
		const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
		__syncthreads(); // the factors have been read
		if (scores)
#pragma unroll
			for (int r = 0; r < 4; r++) {
				const int row = warp * 4 + r;
				const float sum = warp_sum(l[r]);
				const bool any = sum > 0.f || sum != sum;
				if (lane == 0) {
					s_corr[row] = direct ? (any ? 1.f / sum : 0.f) : 1.f;
					if (row < rows) {
						if (!direct) {
							if (slot < part.slots) part.ml[slot * RM + row] = make_float2(m[r], sum);
						} else if (a.lse) {
							const int w = x.t * RM + row;
							a.lse[(long long) (x.row0 + w / a.rep) * a.H + h0 + w % a.rep] = any ? (m[r] + log2f(sum)) * 0.6931471805599453f : -INFINITY;
						}
					}
				}
			}
		__syncthreads();
		if (sums) {
#pragma unroll
			for (int r = 0; r < RPT; r++) {
				const int row = r0 + r, w = x.t * RM + row;
				if (row >= rows) break;
				const float f = s_corr[row]; // 0: a row that sees nothing, whose sums are zeros
				float* to = direct ? reinterpret_cast<float*>(a.out) + (long long) (x.row0 + w / a.rep) * a.out_row + (h0 + w % a.rep) * dv + col : part.o + (slot * RM + row) * dv + col;
				if (direct || slot < part.slots) *reinterpret_cast<float4*>(to) = make_float4(acc[r][0] * f, acc[r][1] * f, acc[r][2] * f, acc[r][3] * f);
			}
		}
	}
}

// =========================================================================================================================================
// The join of what several CTAs have of the same rows, a warp to a row.  A lane takes a piece's maximum and sum, then the pieces' rows are added with their weights, eight
// loads on their way at a time.  Two kinds of blocks: with groups, for rows that read shared pages; and for 16 rows
// of the units that a CTA's share begins inside.  Bound by the latency of three or four loads that depend on one another.
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
	return (size_t) (RM * c.d + buffers * RK * (c.d + 4 + c.dv) + RK * RS + RM) * 4 + (RM + n_lists + 2) * 4 + 16 + (n_lists ? 0 : plan_bytes(b.B, b.n_groups));
}
// Two buffers where shared memory holds them, which it does not for the largest heads beside thousands of sequences; two CTAs to an SM where it holds those
static int rows_buffers(const Cache& c, const BatchView& b, int n_lists) { return rows_smem(c, b, n_lists, 2) <= 226 * 1024 ? 2 : 1; }
int rows_ctas_per_sm(const Cache& c, const BatchView& b, int n_lists) { return rows_smem(c, b, n_lists, rows_buffers(c, b, n_lists)) <= 113 * 1024 ? 2 : 1; }
template <int CG>
static int rows_cols(const Attn& a, cudaStream_t s) {
	const int buffers = rows_buffers(a.c, a.b, a.S);
	const size_t smem = rows_smem(a.c, a.b, a.S, buffers);
	auto kernel = a.lists ? paged_rows_kernel<CG, true> : paged_rows_kernel<CG, false>;
	XALM_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem));
	XALM_CUDA_CHECK(launch(kernel, a.part[0].grid, RT, smem, s, false, a, buffers));
	return XALM_OK;
}
int launch_attn_rows(const Attn& a, cudaStream_t s) { return a.c.dv <= 64 ? rows_cols<16>(a, s) : a.c.dv <= 128 ? rows_cols<32>(a, s) : rows_cols<64>(a, s); }

} // namespace paged
} // namespace xalm
