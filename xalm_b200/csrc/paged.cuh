// paged.cuh — what the kernels of the paged cache (xalm_cuda_paged_*) share: the cache and the batch as they see them, and the plan by which attention's
// CTAs divide their work.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace xalm {
namespace paged {

constexpr int KT = 64;              // keys of a tile, the unit in which attention counts its work
constexpr int MAX_SEGMENTS = 4096;  // sequences and groups of one call: the plan lies in shared memory
constexpr int MAX_LIST = 1024;      // pages that a list of attend_selected names
// Sequences of more rows than this on average fill units of their own: reading the shared pages once for each of them costs less than joining two results of every row.  Five sequences
// behind 2048 shared tokens and 500 of their own, 8 kv heads: with 64 rows to each 35 us as a group and 38 alone, with 256 56 and 47.
constexpr int ALONE_ROWS = 128;
constexpr int ERR_PAGE = 1, ERR_BATCH = 2, ERR_WAIT = 4; // bits of the cache's status word

struct Cache {
	uint8_t *k, *v, *means;
	long long k_page, k_slot, k_head, v_page, v_slot, v_head; // elements
	int pages, shift, G, d, dv;                               // page size 1 << shift
	int* status;
};
struct BatchView {
	int N, B, max_pages, n_groups;
	const int *starts, *lens, *table;
	long long table_row;
	const int *bounds, *shared;
};

__device__ __forceinline__ void report(const Cache& c, int bit) {
	if (c.status) atomicOr(c.status, bit);
}

// What says which rows and lengths the sequences have: in device memory, or a copy of it in shared memory
struct View {
	int N, B, n_groups, cap; // cap: positions that a table row has room for
	const int *starts, *lens, *bounds;
};
__device__ __forceinline__ View view_of(const Cache& c, const BatchView& b) {
	return View{b.N, b.B, b.n_groups, (int) min((long long) b.max_pages << c.shift, 0x7fffffffll), b.starts, b.lens, b.bounds};
}
// A sequence's rows [a, a + n) and its length.  Whatever the arrays hold, rows lie in [0, N) and positions in the table.
struct Seq {
	int a, n, len;
};
__device__ __forceinline__ Seq seq_of(const View& v, int s, int& whole) { // whole: its length, not cut to the table
	Seq q;
	q.a = min(max(v.starts[s], 0), v.N);
	q.n = min(max(v.starts[s + 1], q.a), v.N) - q.a;
	whole = max(v.lens[s], 0);
	q.len = min(whole, v.cap);
	return q;
}
__device__ __forceinline__ Seq seq_of(const View& v, int s) {
	int whole;
	return seq_of(v, s, whole);
}
__device__ __forceinline__ bool seq_ok(const View& v, int s) {
	const int a = v.starts[s], e = v.starts[s + 1], l = v.lens[s];
	return a >= 0 && e >= a && e <= v.N && l >= e - a && l <= v.cap;
}
// One CTA of a call looks all sequences over
__device__ __forceinline__ void check_seqs(const Cache& c, const BatchView& b, int tid, int threads) {
	const View v = view_of(c, b);
	for (int s = tid; s < b.B; s += threads)
		if (!seq_ok(v, s)) report(c, ERR_BATCH);
}
// The sequences of a group
__device__ __forceinline__ int2 group_of(const View& v, int i) {
	const int s0 = min(max(v.bounds[i], 0), v.B);
	return make_int2(s0, min(max(v.bounds[i + 1], s0), v.B));
}
// The sequence of a row: the last s with starts[s] <= row.  A whole warp asks, with 32 probes a round.
__device__ __forceinline__ int seq_of_row(const BatchView& b, int row) {
	const int lane = threadIdx.x & 31;
	if (row < b.B && b.starts[row] <= row && b.starts[row + 1] > row) return row; // steps of single tokens: one asking of memory
	int lo = 0, n = b.B; // the answer lies in [lo, lo + n)
	while (n > 1) {
		const int step = (n + 31) / 32, at = lane * step;
		const unsigned m = __ballot_sync(0xffffffffu, at < n && b.starts[lo + at] <= row);
		const int k = m ? 31 - __clz(m) : 0;
		lo += k * step;
		n = min(step, n - k * step);
	}
	return lo;
}
// Page of the pool that holds page j of a sequence; -1 when the table names none there
__device__ __forceinline__ int page_of(const Cache& c, const BatchView& b, int s, int j) {
	const int p = b.table[(long long) s * b.table_row + j];
	return p >= 0 && p < c.pages ? p : -1;
}

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
// eight neighbouring elements at a 16-byte boundary
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
	if constexpr (sizeof(T) == 4) {
		const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
		x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
	} else {
		const uint4 u = *reinterpret_cast<const uint4*>(p);
		const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
		for (int i = 0; i < 8; i++) x[i] = to_f(t[i]);
	}
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
	if constexpr (sizeof(T) == 4) {
		reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
		reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
	} else {
		uint4 u;
		T* t = reinterpret_cast<T*>(&u);
#pragma unroll
		for (int i = 0; i < 8; i++) t[i] = from_f<T>(x[i]);
		*reinterpret_cast<uint4*>(p) = u;
	}
}

// ---- attention's work --------------------------------------------------------------------------------------------------------------------
// A segment is a run of keys that the same rows read: a group's shared pages (segment i < n_groups: the rows of all its sequences, every row sees every
// key) or a sequence's pages behind them (segment n_groups + s: its own rows, causal).  Rows are (token, query head of the kv head) pairs, `rep` to a token.
// A segment's unit is one kv head and M of its rows; a unit's work is its tiles of KT keys.  The tiles of all units, laid end to end, are cut into as many equal
// parts as there are CTAs, whatever the sequences' lengths: a CTA walks its part, and writes, for each unit that it meets, a partial result into slot
// (unit + CTA) — both numbers only grow along the walk, so no two pieces share a slot.  A unit that one CTA holds whole, and whose rows read no other
// segment, goes straight to the output; paged_join_kernel joins the rest.
struct Head { // the unit inside which a CTA's share begins, and no other segment's business: what the join needs to know of it
	int u, j0, w, share, row0, first, rows, g; // number; tiles before the share (0: no such unit), all; tiles to a CTA; first token row; first and number of its (token, head) rows
};
struct Part {
	float* o;            // (slots, M, dv): sums of exp(s - m) v
	float2* ml;          // (slots, M): m (in units of log2), sum of exp
	int slots, M, grid, lead;
	int least_rows, most_rows; // segments of so many rows are this part's
	int *cum_w, *cum_u, *shs; // the plan, left by CTA 0 for the join: work and units before each segment, keys shared by each sequence
	Head* head;          // (grid)
};
struct Attn {
	Cache c;
	BatchView b;
	const uint8_t* q;
	uint8_t* out;
	long long q_row, out_row; // elements
	float* lse;
	int H, rep;
	float scale;
	const int* lists;         // (N, G, S): pages by their place in the sequence; NULL: all
	int S;
	int n_parts, row_blocks;  // blocks of the join that go over all rows
	Part part[2];
};
struct Plan {
	int *cum_w, *cum_u, *shs; // segments + 1, the same, sequences
	int segs;
	int total, share;
	int units;           // where each is a CTA's as a whole, else 0
	View v; // in shared memory
};
__host__ __device__ constexpr size_t plan_bytes(int B, int n_groups) { return (size_t) (5 * B + 3 * n_groups + 5 + 65) * 4; }

__host__ __device__ __forceinline__ int share_of(int total, int grid) { return (int) (((unsigned) total + grid - 1) / grid); }

// rows of a segment, its first row and the sequence whose table row names the pages: a group's first with rows, since those without need not have any pages
__device__ __forceinline__ int seg_rows(const View& v, int rep, int seg, int& row0, int& s_first) {
	if (seg < v.n_groups) {
		const int2 g = group_of(v, seg);
		s_first = min(g.x, v.B - 1);
		row0 = 0;
		if (g.x == g.y) return 0;
		row0 = seq_of(v, g.x).a;
		const Seq l = seq_of(v, g.y - 1);
		if (v.starts[g.x + 1] <= row0) { // the last that begins at the first row or before
			int hi = g.y - 1;
			while (s_first < hi) {
				const int mid = (s_first + hi + 1) >> 1;
				if (v.starts[mid] <= row0) s_first = mid;
				else hi = mid - 1;
			}
		}
		return max(l.a + l.n - row0, 0) * rep;
	}
	s_first = seg - v.n_groups;
	const Seq q = seq_of(v, s_first);
	row0 = q.a;
	return q.n * rep;
}
// keys of an own segment that the rows up to `last` of it see
__device__ __forceinline__ int own_keys(const Seq& q, int shared, int rep, int last) { return max(q.len - q.n + last / rep + 1 - shared, 0); }

__device__ __forceinline__ bool in_part(const Part& p, int rows) { return rows >= p.least_rows && rows <= p.most_rows; }

// tiles of unit t of a segment
__device__ __forceinline__ int unit_tiles(const Attn& a, const Part& part, int seg, int rows, const Seq& q, int shared, int t) {
	if (seg < a.b.n_groups) return (shared + KT - 1) / KT;
	return max((own_keys(q, shared, a.rep, min((t + 1) * part.M, rows) - 1) + KT - 1) / KT, 1); // rows that see nothing have to be written as well
}

// its work: nothing, or its tiles behind `lead`
__device__ __forceinline__ int unit_work(const Attn& a, const Part& part, int seg, int rows, const Seq& q, int shared, int t) {
	const int w = unit_tiles(a, part, seg, rows, q, shared, t);
	return w ? w + part.lead : 0;
}

// All threads of the CTA.  Shared keys of each group (whole pages, and no more than every row of its sequences sees; a group of one sequence, or of sequences with many rows each, has none;
// sequences without rows do not count), then a running sum over the segments.
template <int NT>
__device__ void make_plan(const Attn& a, const Part& part, uint8_t* smem, Plan& p) {
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.b.B, n = a.b.n_groups;
	p.segs = n + B;
	p.cum_w = reinterpret_cast<int*>(smem);
	p.cum_u = p.cum_w + p.segs + 1;
	p.shs = p.cum_u + p.segs + 1;
	int *starts = p.shs + B, *lens = starts + B + 1, *bounds = lens + B, *sum_w = bounds + n + 1, *sum_u = sum_w + 32, *longest = sum_u + 32;
	// the arrays come in at once: what follows asks for them in turn, and every asking of memory is most of a microsecond
	for (int i = tid; i <= B; i += NT) {
		starts[i] = a.b.starts[i];
		if (i < B) { lens[i] = a.b.lens[i]; p.shs[i] = 0; }
	}
	if (n)
		for (int i = tid; i <= n; i += NT) bounds[i] = a.b.bounds[i];
	p.v = view_of(a.c, a.b);
	p.v.starts = starts;
	p.v.lens = lens;
	p.v.bounds = bounds;
	__syncthreads();
	// rows that two sequences claim, or sequences that two groups do, would be work without bounds: then there is none
	bool bad = false;
	for (int i = tid; i < p.segs; i += NT) {
		if (i < n) bad = bad || bounds[i] > bounds[i + 1];
		else {
			const int s = i - n;
			bad = bad || starts[s] > starts[s + 1];
			if (blockIdx.x == 0 && !seq_ok(p.v, s)) report(a.c, ERR_BATCH);
		}
	}
	bad = __syncthreads_or(bad);
	if (bad && blockIdx.x == 0 && tid == 0) report(a.c, ERR_BATCH);
	if (n && !bad) {
		for (int i = warp; i < n; i += NT / 32) {
			int m = max(a.b.shared[i], 0);
			const int2 g = group_of(p.v, i);
			if (g.y - g.x < 2) continue;
			const Seq last = seq_of(p.v, g.y - 1);
			int some = 0;
			for (int s = g.x + lane; s < g.y; s += 32) {
				const Seq q = seq_of(p.v, s);
				if (q.n) {
					some++;
					m = min(m, max(q.len - q.n, 0));
				}
			}
			some = __reduce_add_sync(0xffffffffu, some);
			if (some < 2 || (float) (last.a + last.n - seq_of(p.v, g.x).a) * a.rep > (float) some * ALONE_ROWS) continue;
			m = __reduce_min_sync(0xffffffffu, m) >> a.c.shift << a.c.shift;
			for (int s = g.x + lane; s < g.y; s += 32) p.shs[s] = m;
		}
		__syncthreads();
	}
	int carry_w = 0, carry_u = 0;
	if (tid == 0) { p.cum_w[0] = 0; p.cum_u[0] = 0; *longest = 0; }
	int most = 0; // tiles of a unit
	for (int base = 0; base < p.segs; base += NT) {
		const int seg = base + tid;
		int w = 0, u = 0, in_seg = 0;
		bool wide = false; // own rows of many tiles: their sum is the whole warp's
		if (seg < p.segs && !bad) {
			int row0, s;
			const int rows = seg_rows(p.v, a.rep, seg, row0, s);
			if (in_part(part, rows)) {
				in_seg = (rows + part.M - 1) / part.M;
				if (seg < n) w = in_seg * unit_work(a, part, seg, rows, Seq(), p.shs[s], 0);
				else if (in_seg == 1) w = unit_work(a, part, seg, rows, seq_of(p.v, s), p.shs[s], 0);
				else wide = true;
				if (!n) most = max(most, wide ? unit_tiles(a, part, seg, rows, seq_of(p.v, s), p.shs[s], in_seg - 1) : w - part.lead); // the last rows see the most
			}
		}
		for (unsigned m = __ballot_sync(0xffffffffu, wide); m; m &= m - 1) {
			const int from = __ffs(m) - 1, wseg = base + (tid & ~31) + from, n_tiles = __shfl_sync(0xffffffffu, in_seg, from);
			const Seq q = seq_of(p.v, wseg - n);
			int sum = 0;
			for (int t = lane; t < n_tiles; t += 32) sum += unit_work(a, part, wseg, q.n * a.rep, q, p.shs[wseg - n], t);
			sum = __reduce_add_sync(0xffffffffu, sum);
			if (lane == from) w = sum;
		}
		w *= a.c.G;
		u = w ? in_seg * a.c.G : 0;
#pragma unroll
		for (int o = 1; o < 32; o <<= 1) {
			const int x = __shfl_up_sync(0xffffffffu, w, o), y = __shfl_up_sync(0xffffffffu, u, o);
			if (lane >= o) { w += x; u += y; }
		}
		if (lane == 31) { sum_w[warp] = w; sum_u[warp] = u; }
		__syncthreads();
		for (int i = 0; i < NT / 32; i++) {
			if (i == warp) { w += carry_w; u += carry_u; }
			carry_w += sum_w[i];
			carry_u += sum_u[i];
		}
		if (seg < p.segs) { p.cum_w[seg + 1] = w; p.cum_u[seg + 1] = u; }
		__syncthreads();
	}
	p.total = carry_w;
	p.share = share_of(p.total, part.grid);
	if (!n) atomicMax(longest, most);
	__syncthreads();
	// Where each unit can have a CTA to itself, and no more tiles than an equal share counts, none is divided and nothing has to be joined.  A prompt of 1024 tokens of 8 kv heads (128 units
	// of 16 tiles) 38 us in place of 48, 16 of 33 tokens behind 400 (128 of 7) 30 in place of 36; but 64 tokens behind 448 (8 of 8) 30 in place of 26.
	p.units = !n && carry_u <= part.grid && *longest <= p.share ? carry_u : 0;
	if (part.cum_w && blockIdx.x == 0) {
		for (int i = tid; i <= p.segs; i += NT) { part.cum_w[i] = p.cum_w[i]; part.cum_u[i] = p.cum_u[i]; }
		for (int i = tid; i < B; i += NT) part.shs[i] = p.shs[i];
	}
}

// One unit of a CTA's walk, with what both its producer and its consumers need to know of it
struct Piece {
	int seg, g, t, u;    // segment, kv head, rows [M t, M (t + 1)) of the segment, number among all units
	int j0, j1;          // tiles of the unit that are this CTA's
	int w;               // all tiles of the unit
	int row0, rows;      // first token row of the segment, (token, head) rows of the segment
	int s;               // whose table row holds the pages (SELECTED: the sequence)
	int key0;            // position of the segment's first key
	Seq q;
};
__device__ __forceinline__ long long piece_slot(const Attn& a, int unit, int cta, bool begins) { return a.b.n_groups && !a.lists ? (long long) unit + cta : 2ll * cta + begins; }
// The walk over a CTA's share of the work
struct Walk {
	int at, end;
	Piece x;
	int tiles;           // row tiles of the segment
};
__device__ __forceinline__ void walk_segment(const Attn& a, const Part& part, const Plan& p, Walk& k) {
	k.x.rows = seg_rows(p.v, a.rep, k.x.seg, k.x.row0, k.x.s);
	k.tiles = (k.x.rows + part.M - 1) / part.M;
	k.x.q = seq_of(p.v, k.x.s);
	k.x.key0 = k.x.seg < a.b.n_groups ? 0 : p.shs[k.x.s];
}
__device__ __forceinline__ void share_begin(int total, int share, Walk& k) {
	k.at = (int) min((unsigned long long) share * blockIdx.x, (unsigned long long) total);
	k.end = k.at + min(share, total - k.at);
}
// The piece of the unit at k.at, `in` of whose work lies behind the share's start; the walk's place moves behind it
__device__ __forceinline__ void walk_piece(const Part& part, Walk& k, int in) {
	const int left = k.x.w + part.lead - in, take = min(left, k.end - k.at); // tiles lie behind the lead
	k.x.j0 = max(in - part.lead, 0);
	k.x.j1 = max(in + take - part.lead, 0);
	k.at += take;
}
// false: nothing for this CTA
__device__ __forceinline__ bool walk_begin(const Attn& a, const Part& part, const Plan& p, Walk& k) {
	if (p.units) {
		k.at = k.end = 0;
		const int u = blockIdx.x;
		if (u >= p.units) return false;
		int lo = 0, hi = p.segs - 1; // the last segment whose units begin at or before this one
		while (lo < hi) {
			const int mid = (lo + hi + 1) >> 1;
			if (p.cum_u[mid] <= u) lo = mid;
			else hi = mid - 1;
		}
		k.x.seg = lo;
		walk_segment(a, part, p, k);
		k.x.g = (u - p.cum_u[lo]) / k.tiles;
		k.x.t = u - p.cum_u[lo] - k.x.g * k.tiles;
		k.x.u = u;
		k.x.j0 = 0;
		k.x.j1 = k.x.w = unit_tiles(a, part, lo, k.x.rows, k.x.q, p.shs[k.x.s], k.x.t);
		return true;
	}
	share_begin(p.total, p.share, k);
	if (k.at >= k.end) return false;
	int lo = 0, hi = p.segs - 1; // the last segment that begins at or before k.at
	while (lo < hi) {
		const int mid = (lo + hi + 1) >> 1;
		if (p.cum_w[mid] <= k.at) lo = mid;
		else hi = mid - 1;
	}
	k.x.seg = lo;
	walk_segment(a, part, p, k);
	int rem = k.at - p.cum_w[lo];
	const int per = (p.cum_w[lo + 1] - p.cum_w[lo]) / a.c.G;
	k.x.g = rem / per;
	rem -= per * k.x.g;
	const int lane = threadIdx.x & 31;
	if (k.tiles == 1) { // the only one of its kv head
		k.x.t = 0;
		k.x.w = per - part.lead;
	} else
	for (int t0 = 0;; t0 += 32) { // whole warps walk: 32 units at a time
		const int w = t0 + lane < k.tiles ? unit_work(a, part, lo, k.x.rows, k.x.q, p.shs[k.x.s], t0 + lane) : 0;
		int sum = w;
#pragma unroll
		for (int o = 1; o < 32; o <<= 1) {
			const int x = __shfl_up_sync(0xffffffffu, sum, o);
			if (lane >= o) sum += x;
		}
		const unsigned m = __ballot_sync(0xffffffffu, sum > rem);
		if (m || t0 + 32 >= k.tiles) {
			const int at = m ? __ffs(m) - 1 : 0, found = __shfl_sync(0xffffffffu, w, at);
			k.x.t = t0 + at;
			k.x.w = max(found - part.lead, 0);
			rem -= __shfl_sync(0xffffffffu, sum, at) - found;
			break;
		}
		rem -= __shfl_sync(0xffffffffu, sum, 31);
	}
	k.x.u = p.cum_u[lo] + k.x.g * k.tiles + k.x.t;
	walk_piece(part, k, rem);
	return true;
}
__device__ __forceinline__ bool walk_next(const Attn& a, const Part& part, const Plan& p, Walk& k) {
	if (k.at >= k.end) return false;
	do {
		if (++k.x.t == k.tiles) {
			k.x.t = 0;
			if (++k.x.g == a.c.G) {
				k.x.g = 0;
				do k.x.seg++;
				while (p.cum_w[k.x.seg + 1] == p.cum_w[k.x.seg]); // ends: k.at < k.end <= total
				walk_segment(a, part, p, k);
			}
		}
		k.x.w = unit_tiles(a, part, k.x.seg, k.x.rows, k.x.q, p.shs[k.x.s], k.x.t);
	} while (k.x.w == 0);
	k.x.u = p.cum_u[k.x.seg] + k.x.g * k.tiles + k.x.t;
	walk_piece(part, k, 0);
	return true;
}
// With lists: units are (row, kv head, M of its query heads), all of the same work
__device__ __forceinline__ int list_tiles(const Attn& a) { return (int) ((((long long) a.S << a.c.shift) + KT - 1) / KT); }
__device__ __forceinline__ int list_total(const Attn& a, const Part& part) { return a.b.N * a.c.G * ((a.rep + part.M - 1) / part.M) * (list_tiles(a) + part.lead); }
__device__ __forceinline__ void list_unit(const Attn& a, const Part& part, Walk& k, int unit, bool walking) {
	const int tiles = (a.rep + part.M - 1) / part.M;
	const int of = unit / tiles, row = of / a.c.G;
	k.x.u = unit;
	k.x.t = unit - of * tiles;
	k.x.g = of - row * a.c.G;
	const bool same_row = walking && row == k.x.row0;
	k.x.row0 = row;
	k.x.rows = a.rep;
	k.x.seg = 0;
	k.x.key0 = 0;
	k.x.w = list_tiles(a);
	if (!same_row) {
		k.x.s = seq_of_row(a.b, k.x.row0); // whole warps walk
		k.x.q = seq_of(view_of(a.c, a.b), k.x.s);
	}
}
__device__ __forceinline__ bool list_begin(const Attn& a, const Part& part, Walk& k) {
	const int total = list_total(a, part);
	share_begin(total, share_of(total, part.grid), k);
	if (k.at >= k.end) return false;
	const int w = list_tiles(a) + part.lead;
	list_unit(a, part, k, k.at / w, false);
	walk_piece(part, k, k.at % w);
	return true;
}
__device__ __forceinline__ bool list_next(const Attn& a, const Part& part, Walk& k) {
	if (k.at >= k.end) return false;
	list_unit(a, part, k, k.x.u + 1, true);
	walk_piece(part, k, 0);
	return true;
}
// by one thread of a CTA, before its first walk_next / list_next
__device__ __forceinline__ void write_head(const Attn& a, const Part& part, const Walk& k, bool any, bool alone, int share) {
	Head h = {};
	if (any && alone) h = Head{k.x.u, k.x.j0, k.x.w, share, k.x.row0, k.x.t * part.M, min(part.M, k.x.rows - k.x.t * part.M), k.x.g};
	part.head[blockIdx.x] = h;
}
__device__ __forceinline__ bool row_in_seq(const Seq& q, int row) { return row >= q.a && row < q.a + q.n; }

// The list of (row, kv head), by a whole warp: pages that the row sees, each once, in ascending order, into `pages` (NULL: counted only).  Lists that come
// so, with -1 behind, cost one pass; any other order, and pages named twice, cost a pass over the list for every page.  *own: whether the row's own page is among them.
__device__ __forceinline__ int list_pages(const Attn& a, int row, int g, int own_page, int* pages, bool* own) {
	const int lane = threadIdx.x & 31;
	const int* l = a.lists + ((long long) row * a.c.G + g) * a.S;
	const int most = min(own_page, a.b.max_pages - 1);
	int n = 0, before = -1;
	bool tidy = true, gap = false;
	*own = false;
	for (int i = 0; i < a.S; i += 32) {
		const int e = i + lane < a.S ? l[i + lane] : -1;
		const bool ok = e >= 0 && e <= most;
		const unsigned m = __ballot_sync(0xffffffffu, ok);
		int prev = __shfl_up_sync(0xffffffffu, e, 1);
		if (lane == 0) prev = before;
		tidy = tidy && (m & (m + 1)) == 0 && !(gap && m) && __all_sync(0xffffffffu, !ok || e > prev);
		gap = gap || m != 0xffffffffu;
		before = __shfl_sync(0xffffffffu, e, 31);
		if (pages && ok) pages[n + __popc(m & ((1u << lane) - 1))] = e;
		n += __popc(m);
		*own = *own || __any_sync(0xffffffffu, ok && e == own_page);
	}
	if (tidy) {
		__syncwarp();
		return n;
	}
	n = 0;
	for (int last = -1;;) { // the next larger entry, until there is none
		int m = 0x7fffffff;
		for (int i = lane; i < a.S; i += 32) {
			const int e = l[i];
			if (e > last && e <= most) m = min(m, e);
		}
		m = __reduce_min_sync(0xffffffffu, m);
		if (m == 0x7fffffff) break;
		if (pages && lane == 0) pages[n] = m;
		n++;
		last = m;
	}
	__syncwarp();
	return n;
}

// A kernel's limit of dynamic shared memory is the process's: it is set to the same number by every call, whatever the call needs, so that none lowers it between another thread's
// setting and launch.  own: shared memory that the kernel declares
inline cudaError_t allow_smem(const void* kernel, int own = 0) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - own); }
// Launches; `after`: may start while the kernel before it on the stream still runs (it waits for it itself).
template <typename K, typename... A>
inline cudaError_t launch(K kernel, dim3 grid, int block, size_t smem, cudaStream_t s, bool after, const A&... args) {
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid;
	cfg.blockDim = dim3((unsigned) block);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = s;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = after ? 1 : 0;
	return cudaLaunchKernelEx(&cfg, kernel, args...);
}
int launch_join(const Attn& a, int type, cudaStream_t s);
int launch_status(int* status, int* taken, cudaStream_t s);
// CTAs per SM that a kernel's shared memory leaves room for, and its launch: fp32 caches, 16-bit caches
int rows_ctas_per_sm(const Cache& c, const BatchView& b, int n_lists);
int launch_attn_rows(const Attn& a, cudaStream_t s);
int mma_ctas_per_sm(const Cache& c, const BatchView& b, int n_lists);
int launch_attn_mma(const Attn& a, int part, int type, cudaStream_t s);
constexpr int TC_ROWS = 256; // rows of a unit on tcgen05
bool tc_fits(const Cache& c, const BatchView& b);
int launch_attn_tc(const Attn& a, int part, int type, cudaStream_t s);

} // namespace paged
} // namespace xalm
