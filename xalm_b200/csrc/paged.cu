// paged.cu — the paged cache: entry points (include/xalm_cuda.h, xalm_cuda_paged_*), appending to pages, choosing pages.
//
// Several sequences share one pool of pages; a table names each sequence's pages.  Lengths and tables are read on the device, so that a captured graph serves
// every step of a batch; what the host has to know is how large the arrays are.
#include "paged.cuh"

#include <math.h>

#include <algorithm>

#include "family.h"
#include "paged_check.h"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// append: a row's position is p = len - n + i, its page table[p / P], its slot p % P.  Bound by HBM (every element in and out once), so a thread takes 16 or 32 bytes of a head
// with those half a rotation away that they are turned with, of R rows at once: R = 4 keeps enough bytes on their way in prompts; steps of few tokens
// have a CTA to a row.  9 prompts of 300 to 1500 tokens (209 MB) take 47 us, 4.4 TB/s; 16 rows of 32 and 8 heads 3.7, a launch and two dependent loads.  The angle
// p * freq is taken in 64 bits and brought into [-pi, pi] there: in 32 bits position 100000 is 0.004 rad off.
// =========================================================================================================================================
struct AppendArgs {
	Cache c;
	BatchView b;
	const uint8_t *k, *v, *q;
	long long k_row, v_row, q_row, q_out_row;
	uint8_t* q_out;
	int H;
	const float* freq;
	int rot;
	float mag;
	int neighbours;
	int paired;                 // halves whose chunks of eight pair up: a thread takes both
	int per_head, per_value;    // work items of a head of q or k, of v
	unsigned by_head, by_value; // 2^32 / those, rounded up (0 for one)
};

constexpr int AT = 256;

template <typename I>
struct Chunk { // eight elements as they came
	uint4 u[sizeof(I) / 2];
	__device__ __forceinline__ void load(const I* p) {
#pragma unroll
		for (int i = 0; i < (int) sizeof(I) / 2; i++) u[i] = reinterpret_cast<const uint4*>(p)[i];
	}
	__device__ __forceinline__ void floats(float (&x)[8]) const {
		const I* t = reinterpret_cast<const I*>(u);
#pragma unroll
		for (int i = 0; i < 8; i++) x[i] = to_f(t[i]);
	}
};

template <typename I, typename T, int R>
__global__ void __launch_bounds__(AT) paged_append_kernel(const __grid_constant__ AppendArgs a) {
	__shared__ float s_cos[R][128], s_sin[R][128];
	__shared__ int s_pos[R], s_page[R]; // position (-1: not a row of any sequence, or before its first token), page of the pool (-1: none)
	pdl_launch_dependents();
	const int row0 = blockIdx.x * R, tid = threadIdx.x, warp = tid >> 5, d = a.c.d, dv = a.c.dv, G = a.c.G;
	if (blockIdx.x == 0) check_seqs(a.c, a.b, tid, AT);
	if (warp < R) {
		const int row = row0 + warp;
		int pos = -1, page = -1;
		if (row < a.b.N) {
			const int s = seq_of_row(a.b, row);
			const View view = view_of(a.c, a.b);
			int whole;
			const Seq q = seq_of(view, s, whole);
			if (row_in_seq(q, row)) {
				pos = whole - q.n + row - q.a; // what lies behind the table is turned, and written nowhere
				if (pos >= 0 && pos < view.cap) {
					page = page_of(a.c, a.b, s, pos >> a.c.shift);
					if (page < 0 && (tid & 31) == 0) report(a.c, ERR_PAGE);
				}
			}
		}
		if ((tid & 31) == 0) { s_pos[warp] = pos; s_page[warp] = page; }
	}
	__syncthreads();
	for (int i = tid; i < R * a.rot; i += AT) {
		const int r = i / a.rot, f = i - r * a.rot;
		if (s_pos[r] < 0) continue;
		const double x = (double) s_pos[r] * (double) a.freq[f], turns = rint(x * 0.15915494309189535);
		float sn, cs;
		sincosf((float) fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, x)), &sn, &cs); // 2 pi as the sum of two doubles
		s_cos[r][f] = cs * a.mag;
		s_sin[r][f] = sn * a.mag;
	}
	__syncthreads();
	const int n_q = a.q ? a.H * a.per_head : 0, n_k = n_q + G * a.per_head, n_all = n_k + G * a.per_value, slot_mask = (1 << a.c.shift) - 1;
	for (int i = tid; i < n_all; i += AT) {
		const bool value = i >= n_k, key = !value && i >= n_q;
		const int j = value ? i - n_k : key ? i - n_q : i, per = value ? a.per_value : a.per_head;
		const int h = per == 1 ? j : (int) __umulhi((unsigned) j, value ? a.by_value : a.by_head), u = j - h * per;
		const int c = value || !a.paired || u * 8 < a.rot ? u * 8 : u * 8 + a.rot; // the item's first element; behind the pairs come the chunks that are not turned
		const bool pair = !value && a.paired && u * 8 < a.rot;
		const I* in = value ? reinterpret_cast<const I*>(a.v) + h * dv + c : key ? reinterpret_cast<const I*>(a.k) + h * d + c : reinterpret_cast<const I*>(a.q) + h * d + c;
		const long long step = value ? a.v_row : key ? a.k_row : a.q_row;
		Chunk<I> x[R], y[R];
		bool go[R];
#pragma unroll
		for (int r = 0; r < R; r++) {
			go[r] = s_pos[r] >= 0 && !((value || key) && s_page[r] < 0);
			if (!go[r]) continue;
			x[r].load(in + (row0 + r) * step);
			if (pair) y[r].load(in + (row0 + r) * step + a.rot);
		}
#pragma unroll
		for (int r = 0; r < R; r++) {
			if (!go[r]) continue;
			float lo[8], hi[8];
			x[r].floats(lo);
			T* out = value ? reinterpret_cast<T*>(a.c.v) + s_page[r] * a.c.v_page + (s_pos[r] & slot_mask) * a.c.v_slot + h * a.c.v_head + c
			         : key ? reinterpret_cast<T*>(a.c.k) + s_page[r] * a.c.k_page + (s_pos[r] & slot_mask) * a.c.k_slot + h * a.c.k_head + c
			               : reinterpret_cast<T*>(a.q_out) + (row0 + r) * a.q_out_row + h * d + c;
			if (pair) {
				y[r].floats(hi);
#pragma unroll
				for (int e = 0; e < 8; e++) {
					const float cs = s_cos[r][c + e], sn = s_sin[r][c + e], l = lo[e];
					lo[e] = l * cs - hi[e] * sn;
					hi[e] = hi[e] * cs + l * sn;
				}
				store8(out + a.rot, hi);
			} else if (!value && !a.paired && c < 2 * a.rot) {
				if (a.neighbours) {
#pragma unroll
					for (int e = 0; e < 8; e += 2) {
						const int f = (c + e) / 2;
						if (f < a.rot) {
							const float l = lo[e];
							lo[e] = l * s_cos[r][f] - lo[e + 1] * s_sin[r][f];
							lo[e + 1] = lo[e + 1] * s_cos[r][f] + l * s_sin[r][f];
						}
					}
				} else { // halves that end inside a chunk
					const I* head = in - c + (row0 + r) * step;
#pragma unroll
					for (int e = 0; e < 8; e++) {
						const int at = c + e;
						if (at >= 2 * a.rot) continue;
						const int f = at < a.rot ? at : at - a.rot;
						const float o = to_f(head[at < a.rot ? at + a.rot : f]);
						lo[e] = at < a.rot ? lo[e] * s_cos[r][f] - o * s_sin[r][f] : lo[e] * s_cos[r][f] + o * s_sin[r][f];
					}
				}
			}
			store8(out, lo);
		}
	}
}

// Mean keys of the pages whose last slot this call has written: a CTA per page that may be one and kv head.  Sequence s has room for
// floor(starts[s + 1] / P) - floor(starts[s] / P) + 1 such pages, numbered from floor(starts[s] / P) + s.  The sum runs over the stored keys, in an order that does
// not depend on which calls brought them.
template <typename T>
__global__ void __launch_bounds__(128) paged_means_kernel(const Cache c, const BatchView b) {
	__shared__ float part[128][9];
	pdl_wait();
	pdl_launch_dependents();
	const int tid = threadIdx.x, lane = tid & 31, g = blockIdx.y, item = blockIdx.x, P = 1 << c.shift;
	int lo = 0, n = b.B; // the last s whose pages begin at or before this one
	while (n > 1) {
		const int step = (n + 31) / 32, at = lane * step;
		const unsigned m = __ballot_sync(0xffffffffu, at < n && (b.starts[lo + at] >> c.shift) + lo + at <= item);
		const int k = m ? 31 - __clz(m) : 0;
		lo += k * step;
		n = min(step, n - k * step);
	}
	int whole;
	const Seq q = seq_of(view_of(c, b), lo, whole);
	const int first = max(whole - q.n, 0) >> c.shift; // page of the first new token
	const int j = first + item - ((q.a >> c.shift) + lo);
	if (q.n == 0 || j < first || (long long) (j + 1) << c.shift > q.len) return; // not filled
	const int page = page_of(c, b, lo, j);
	if (page < 0) return;
	const int dc = c.d / 8, groups = 128 / dc, ch = tid % dc, sl = tid / dc;
	float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
	const T* base = reinterpret_cast<const T*>(c.k) + page * c.k_page + g * c.k_head + ch * 8;
	if (sl < groups)
		for (int i = sl; i < P; i += groups) {
			float x[8];
			load8(base + i * c.k_slot, x);
#pragma unroll
			for (int e = 0; e < 8; e++) sum[e] += x[e];
		}
#pragma unroll
	for (int e = 0; e < 8; e++) part[tid][e] = sum[e];
	__syncthreads();
	if (sl) return;
	for (int i = 1; i < groups; i++)
#pragma unroll
		for (int e = 0; e < 8; e++) sum[e] += part[i * dc + ch][e];
#pragma unroll
	for (int e = 0; e < 8; e++) sum[e] *= 1.f / P;
	store8(reinterpret_cast<T*>(c.means) + ((long long) page * c.G + g) * c.d + ch * 8, sum);
}

// =========================================================================================================================================
// select: score_j = (sum over the kv head's queries) . mean_j, and of the pages between the first and the recent ones those with the largest scores, equal ones from the lowest
// place on.  Which page is the last to be taken must not hang on how a sum was rounded, and sums in 64 bits cost a conversion per mean and row (279 us for 1341
// tokens of 8 heads over 110 to 235 pages, which take 56 now).  So scores are taken in fp32, each off by at most E = (d + rep + 4) 2^-24 sum_i (sum_r |q_ri|) max |mean|; of the want-th largest, t, the true
// one is off by no more than E (no E holds where fp32 may overflow: all are summed in 64 bits then), so pages above t + 2 E are taken, those below t - 2 E are not, and only where those between are more than are wanted are they summed in 64 bits.
// Steps of single tokens: a CTA to (row, kv head), 8 lanes to a page.  Longer ones: R rows of a sequence to a CTA, so that a page's mean is read and converted once for
// all of them: 64 pages at a time in shared memory, a thread taking one page and R / 4 rows; then a warp to a row.  The want-th largest is found bit by bit from above, up to 512 keys in a warp's registers.
// =========================================================================================================================================
struct SelectArgs {
	Cache c;
	BatchView b;
	const uint8_t* q;
	long long q_row;
	int H, rep, top, first, recent;
	int* out;
};
constexpr int ST = 256, SP = 64;
typedef unsigned long long u64;

__device__ __forceinline__ u64 ordered(double x) { // the order of numbers as integers, from 1 to 2^64 - 2; NaN and -infinity as the lowest finite, +infinity as the largest
	const double big = 1.7976931348623157e308;
	x = x != x ? -big : fmin(fmax(x, -big), big) + 0.0;
	const long long b = __double_as_longlong(x);
	return b < 0 ? ~(u64) b : (u64) b | (1ull << 63);
}
__device__ __forceinline__ unsigned ordered32(float x) {
	const int b = __float_as_int(x + 0.f);
	return b < 0 ? ~(unsigned) b : (unsigned) b | (1u << 31);
}
__device__ __forceinline__ float unordered32(unsigned k) { return __int_as_float(k >> 31 ? (int) (k & 0x7fffffffu) : (int) ~k); }

// The threads that have a row: a warp, or the CTA
template <int TEAM>
__device__ __forceinline__ int team_sum(int x, int* buf) {
	x = __reduce_add_sync(0xffffffffu, x);
	if constexpr (TEAM > 32) {
		__syncthreads();
		if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
		__syncthreads();
		x = 0;
#pragma unroll
		for (int w = 0; w < TEAM / 32; w++) x += buf[w];
	}
	return x;
}
template <int TEAM>
__device__ __forceinline__ void team_sync() {
	if constexpr (TEAM > 32) __syncthreads();
	else __syncwarp();
}
// A number that exactly `want` keys of [lo, hi) reach, or where equal keys forbid that, the want-th largest key: bit by bit from above until it divides
template <int TEAM, typename K>
__device__ __forceinline__ K divide_keys(const u64* key, int lo, int hi, int want, int tid, int* buf) {
	K prefix = 0;
	for (int bit = sizeof(K) * 8 - 1; bit >= 0; bit--) {
		const K c = prefix | (K) 1 << bit;
		int n = 0;
		for (int j = lo + tid; j < hi; j += TEAM) n += (K) key[j] >= c;
		n = team_sum<TEAM>(n, buf);
		if (n >= want) prefix = c;
		if (n == want) break;
	}
	return prefix;
}
constexpr int IN_REGS = 16; // keys that a lane holds at most
// The want-th largest of keys [lo, hi) by one warp, N to a lane in registers.  Halving the scores' range divides them in six or seven counts where they are spread evenly, bits
// need fourteen; bits where that fails (equal scores, some far from all others, some not finite).
template <int N>
__device__ __forceinline__ unsigned nth_in_regs(const u64* key, int lo, int hi, int want) {
	const int lane = threadIdx.x & 31;
	unsigned k[N], top = 0, low = ~0u;
#pragma unroll
	for (int i = 0; i < N; i++) {
		const int j = lo + lane + 32 * i;
		k[i] = j < hi ? (unsigned) key[j] : 0u;
		top = max(top, k[i]);
		if (j < hi) low = min(low, k[i]);
	}
	float up = unordered32(__reduce_max_sync(0xffffffffu, top)), down = unordered32(__reduce_min_sync(0xffffffffu, low));
	unsigned cut = 0;
	for (int step = 0; step < 20; step++) {
		const float mid = 0.5f * up + 0.5f * down;
		const unsigned c = ordered32(mid);
		int n = 0;
#pragma unroll
		for (int i = 0; i < N; i++) n += k[i] >= c;
		n = __reduce_add_sync(0xffffffffu, n);
		if (n == want) { cut = c; break; }
		(n > want ? down : up) = mid;
	}
	if (!cut)
		for (int bit = 31; bit >= 0; bit--) {
			const unsigned c = cut | 1u << bit;
			int n = 0;
#pragma unroll
			for (int i = 0; i < N; i++) n += k[i] >= c;
			n = __reduce_add_sync(0xffffffffu, n);
			if (n >= want) cut = c;
			if (n == want) break;
		}
	unsigned least = ~0u;
#pragma unroll
	for (int i = 0; i < N; i++)
		if (k[i] >= cut) least = min(least, k[i]);
	return least;
}
// (sum of the row's queries) . mean of page j, in 64 bits, by a warp
template <typename T>
__device__ __forceinline__ double exact_score(const SelectArgs& a, int s, int row, int g, int j) {
	const int lane = threadIdx.x & 31, page = page_of(a.c, a.b, s, j);
	double x = 0;
	if (page >= 0)
		for (int i = lane; i < a.c.d; i += 32) {
			double qs = 0;
			for (int r = 0; r < a.rep; r++) qs += (double) to_f(reinterpret_cast<const T*>(a.q)[(long long) row * a.q_row + (g * a.rep + r) * a.c.d + i]);
			x = fma((double) to_f(reinterpret_cast<const T*>(a.c.means)[((long long) page * a.c.G + g) * a.c.d + i]), qs, x);
		}
#pragma unroll
	for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
	return x;
}

// A row's list.  key[j] holds ordered32 of the fp32 scores of pages [lo, hi).
template <typename T, int TEAM>
__device__ void pick_pages(const SelectArgs& a, const Seq& q, int s, int row, int g, float err, u64* key, int tid, int* buf) {
	const int lane = tid & 31;
	const int pos = q.len - q.n + row - q.a, last = pos < 0 ? -1 : pos >> a.c.shift;
	const int lo = min(a.first, last + 1), hi = max(last - a.recent, lo); // pages [lo, hi) are chosen by score, those before and from hi to last are always
	const int fixed = lo + last + 1 - hi, want = min(a.top - fixed, hi - lo);
	int* out = a.out + ((long long) row * a.c.G + g) * a.top;
	const bool by_score = want > 0 && want < hi - lo;
	u64 least = 0; // taken: keys above it, and the first `ties` of those equal to it
	int ties = 0;
	if (by_score) {
		unsigned least32 = ~0u; // the want-th largest: the least of those that reach the dividing number
		if (TEAM == 32 && hi - lo <= 256) least32 = nth_in_regs<8>(key, lo, hi, want);
		else if (TEAM == 32 && hi - lo <= 32 * IN_REGS) least32 = nth_in_regs<IN_REGS>(key, lo, hi, want);
		else {
			const unsigned cut = divide_keys<TEAM, unsigned>(key, lo, hi, want, tid, buf);
			for (int j = lo + tid; j < hi; j += TEAM)
				if ((unsigned) key[j] >= cut) least32 = min(least32, (unsigned) key[j]);
		}
		least32 = __reduce_min_sync(0xffffffffu, least32);
		if constexpr (TEAM > 32) {
			__syncthreads();
			if (lane == 0) buf[tid >> 5] = (int) least32;
			__syncthreads();
			for (int w = 0; w < TEAM / 32; w++) least32 = min(least32, (unsigned) buf[w]);
		}
		const float t = unordered32(least32), up = t + 2.f * err, down = t - 2.f * err;
		int sure = 0, near = 0;
		for (int j = lo + tid; j < hi; j += TEAM) {
			const float x = unordered32((unsigned) key[j]);
			const bool above = x > up, below = x < down; // both false where something is not finite
			sure += above;
			near += !above && !below;
			key[j] = above ? ~0ull : below ? 0ull : 1ull;
		}
		sure = team_sum<TEAM>(sure, buf);
		near = team_sum<TEAM>(near, buf);
		if (sure + near > want) { // the order of those between, in 64 bits
			team_sync<TEAM>();
			if (near <= 32) { // a lane holds one of them; what stands before it says whether it is taken
				if (tid < 32) {
					int n = 0, page = -1;
					double x = 0;
					for (int j0 = lo; j0 < hi; j0 += 32)
						for (unsigned m = __ballot_sync(0xffffffffu, j0 + lane < hi && key[min(j0 + lane, hi - 1)] == 1); m; m &= m - 1, n++) {
							const int j = j0 + __ffs(m) - 1;
							const double e = exact_score<T>(a, s, row, g, j);
							if (lane == n) { x = e; page = j; }
						}
					const u64 mine = page >= 0 ? ordered(x) : 0;
					int rank = 0;
					for (int i = 0; i < n; i++) {
						const u64 o = __shfl_sync(0xffffffffu, mine, i);
						rank += o > mine || (o == mine && i < lane);
					}
					__syncwarp();
					if (page >= 0) key[page] = rank < want - sure ? 1ull : 0ull;
				}
			} else {
				for (int j0 = lo + tid / 32; j0 < hi; j0 += TEAM / 32)
					if (key[j0] == 1) {
						const double x = exact_score<T>(a, s, row, g, j0);
						__syncwarp();
						if (lane == 0) key[j0] = ordered(x);
						__syncwarp();
					}
				team_sync<TEAM>();
				least = divide_keys<TEAM, u64>(key, lo, hi, want, tid, buf);
				int above = 0, equal = 0;
				for (int j = lo + tid; j < hi; j += TEAM) { above += key[j] > least; equal += key[j] == least; }
				above = team_sum<TEAM>(above, buf);
				equal = team_sum<TEAM>(equal, buf);
				ties = want - above;
			}
		}
	}
	team_sync<TEAM>();
	// in ascending order, a team's worth of pages at a time
	int written = 0, tied = 0;
	for (int base = 0; base <= last; base += TEAM) {
		const int j = base + tid;
		const bool mid = j >= lo && j < hi, tie = by_score && least && mid && key[j] == least;
		int rank = 0; // among the ties before it
		if (least) {
			const unsigned tm = __ballot_sync(0xffffffffu, tie);
			rank = tied + __popc(tm & ((1u << lane) - 1));
			if constexpr (TEAM > 32) {
				__syncthreads();
				if (lane == 0) buf[tid >> 5] = __popc(tm);
				__syncthreads();
				for (int w = 0; w < TEAM / 32; w++) {
					if (w < tid >> 5) rank += buf[w];
					tied += buf[w];
				}
			} else tied += __popc(tm);
		}
		const bool take = j <= last && (mid ? (by_score ? key[j] > least || (tie && rank < ties) : want > 0) : true);
		const unsigned om = __ballot_sync(0xffffffffu, take);
		int at = written + __popc(om & ((1u << lane) - 1));
		if constexpr (TEAM > 32) {
			__syncthreads();
			if (lane == 0) buf[tid >> 5] = __popc(om);
			__syncthreads();
			for (int w = 0; w < TEAM / 32; w++) {
				if (w < tid >> 5) at += buf[w];
				written += buf[w];
			}
		} else written += __popc(om);
		if (take && at < a.top) out[at] = j;
	}
	for (int i = written + tid; i < a.top; i += TEAM) out[i] = -1;
}

// max |mean|, as the bits of a number: of two without signs the larger one's are larger, and those of what is not finite larger than all others'
__device__ __forceinline__ unsigned grow_bound(unsigned m, const float (&v)[8]) {
#pragma unroll
	for (int e = 0; e < 8; e++) m = max(m, (unsigned) __float_as_int(v[e]) & 0x7fffffffu);
	return m;
}
// No bound where a sum may leave the range of fp32 on its way; products and sums below its normal numbers are off by half of the smallest each
__device__ __forceinline__ float score_error(int d, int rep, float abs_q, unsigned most) {
	const float size = abs_q * __int_as_float((int) most);
	return most >= 0x7f800000u || !(size < 3.0e38f) ? INFINITY : 1.1f * (float) (d + rep + 4) * 5.9604645e-8f * size + (float) (d + 4) * 1.4e-45f;
}

template <typename T>
__global__ void __launch_bounds__(ST) paged_select_step_kernel(const __grid_constant__ SelectArgs a) {
	extern __shared__ __align__(16) u64 keys[]; // one per page
	__shared__ __align__(16) float s_q[256];
	__shared__ float s_abs[ST / 32];
	__shared__ unsigned s_max[ST / 32];
	__shared__ int buf[ST / 32];
	pdl_launch_dependents();
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x, g = blockIdx.y, d = a.c.d;
	if (row == 0 && g == 0) check_seqs(a.c, a.b, tid, ST);
	const int s = seq_of_row(a.b, row);
	const Seq q = seq_of(view_of(a.c, a.b), s);
	if (!row_in_seq(q, row)) return;
	const int pos = q.len - q.n + row - q.a, last = pos < 0 ? -1 : pos >> a.c.shift, lo = min(a.first, last + 1), hi = max(last - a.recent, lo);
	float err = 0.f;
	if (hi - lo > a.top - (lo + last + 1 - hi)) {
		float abs_q = 0.f;
		for (int i = tid; i < d; i += ST) {
			float x = 0.f;
#pragma unroll 4
			for (int r = 0; r < a.rep; r++) {
				const float e = to_f(reinterpret_cast<const T*>(a.q)[(long long) row * a.q_row + (g * a.rep + r) * d + i]);
				x += e;
				abs_q += fabsf(e);
			}
			s_q[i] = x;
		}
		__syncthreads();
		for (int j = lo + tid; j < hi; j += ST) { // which pages, all at once: a mean's address hangs on it
			const int page = page_of(a.c, a.b, s, j);
			if (page < 0) report(a.c, ERR_PAGE);
			keys[j] = (u64) (unsigned) page;
		}
		__syncthreads();
		const int sub = lane & 7;
		unsigned most = 0;
		for (int j0 = lo + warp * 4 + (lane >> 3); j0 < hi; j0 += 4 * (ST / 8)) { // four pages of each eight lanes on their way together
			int page[4];
			float x[4];
#pragma unroll
			for (int u = 0; u < 4; u++) {
				const int j = j0 + u * (ST / 8);
				page[u] = j < hi ? (int) keys[j] : -1;
				x[u] = 0.f;
			}
			for (int c = sub * 8; c < d; c += 64) {
				float v[4][8];
#pragma unroll
				for (int u = 0; u < 4; u++) load8(reinterpret_cast<const T*>(a.c.means) + ((long long) max(page[u], 0) * a.c.G + g) * d + c, v[u]);
#pragma unroll
				for (int u = 0; u < 4; u++)
					if (page[u] >= 0) {
						most = grow_bound(most, v[u]);
#pragma unroll
						for (int e = 0; e < 8; e++) x[u] = fmaf(v[u][e], s_q[c + e], x[u]);
					}
			}
#pragma unroll
			for (int u = 0; u < 4; u++) {
				const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
				for (int o = 4; o; o >>= 1) x[u] += __shfl_xor_sync(mask, x[u], o); // all eight have read their page
				if (sub == 0 && j0 + u * (ST / 8) < hi) keys[j0 + u * (ST / 8)] = ordered32(x[u]);
			}
		}
		most = __reduce_max_sync(0xffffffffu, most);
		abs_q = warp_sum(abs_q);
		if (lane == 0) { s_max[warp] = most; s_abs[warp] = abs_q; }
		__syncthreads();
		abs_q = 0.f;
		for (int w = 0; w < ST / 32; w++) { most = max(most, s_max[w]); abs_q += s_abs[w]; }
		err = score_error(d, a.rep, abs_q, most);
	}
	if (hi - lo <= 32 * IN_REGS) {
		if (warp == 0) pick_pages<T, 32>(a, q, s, row, g, err, keys, lane, nullptr);
	} else pick_pages<T, ST>(a, q, s, row, g, err, keys, tid, buf);
}

template <typename T, int R>
__global__ void __launch_bounds__(ST) paged_select_rows_kernel(const __grid_constant__ SelectArgs a) {
	extern __shared__ __align__(16) uint8_t smem[];
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.y, d = a.c.d, dp = d + 4;
	u64* keys = reinterpret_cast<u64*>(smem);                              // [R][max_pages]
	float* s_q = reinterpret_cast<float*>(keys + (size_t) R * a.b.max_pages); // [R][d]
	float* s_m = s_q + R * d;                                              // [SP][d + 4]
	float* s_abs = s_m + SP * dp;                                          // [R][d / 8]
	unsigned* s_max = reinterpret_cast<unsigned*>(s_abs + R * (d / 8));    // [8]
	int* s_page = reinterpret_cast<int*>(s_max + ST / 32);                 // [max_pages]
	pdl_launch_dependents();
	if (blockIdx.x == 0 && g == 0) check_seqs(a.c, a.b, tid, ST);
	// sequence s has room for floor(starts[s + 1] / R) - floor(starts[s] / R) + 1 blocks of rows, from number floor(starts[s] / R) + s on
	int s = 0;
	for (int n = a.b.B; n > 1;) {
		const int step = (n + 31) / 32, at = lane * step;
		const unsigned m = __ballot_sync(0xffffffffu, at < n && max(a.b.starts[s + at], 0) / R + s + at <= (int) blockIdx.x);
		const int k = m ? 31 - __clz(m) : 0;
		s += k * step;
		n = min(step, n - k * step);
	}
	const Seq q = seq_of(view_of(a.c, a.b), s);
	const long long first = q.a + (long long) ((int) blockIdx.x - (q.a / R + s)) * R;
	if (first < q.a || first >= q.a + q.n) return;
	const int row0 = (int) first, rows = min(R, q.a + q.n - row0);
	const int dc = d / 8;
	for (int i = tid; i < R * dc; i += ST) { // eight entries of a row's sum
		const int r = i / dc, c = (i - r * dc) * 8;
		float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, abs_q = 0.f;
		if (r < rows) {
			const T* at = reinterpret_cast<const T*>(a.q) + (long long) (row0 + r) * a.q_row + g * a.rep * d + c;
#pragma unroll 4
			for (int h = 0; h < a.rep; h++) {
				float v[8];
				load8(at + h * d, v);
#pragma unroll
				for (int e = 0; e < 8; e++) { sum[e] += v[e]; abs_q += fabsf(v[e]); }
			}
		}
#pragma unroll
		for (int e = 0; e < 8; e++) s_q[r * d + c + e] = sum[e];
		s_abs[i] = abs_q;
	}
	const int last = (q.len - q.n + row0 + rows - 1 - q.a) >> a.c.shift; // of the last row; negative where it sees nothing
	const int lo = min(a.first, max(last + 1, 0)), hi = max(last - a.recent, lo);
	for (int j = lo + tid; j < hi; j += ST) { // which pages, all at once: a mean's address hangs on it
		s_page[j] = page_of(a.c, a.b, s, j);
		if (s_page[j] < 0) report(a.c, ERR_PAGE);
	}
	unsigned most = 0;
	for (int p0 = lo; p0 < hi; p0 += SP) {
		__syncthreads();
		for (int i0 = tid; i0 < SP * dc; i0 += 4 * ST) {
			float v[4][8];
#pragma unroll
			for (int u = 0; u < 4; u++) {
				const int i = i0 + u * ST, j = i / dc, page = i < SP * dc && p0 + j < hi ? s_page[p0 + j] : -1;
				load8(reinterpret_cast<const T*>(a.c.means) + ((long long) max(page, 0) * a.c.G + g) * d + (i - j * dc) * 8, v[u]);
				if (page < 0)
#pragma unroll
					for (int e = 0; e < 8; e++) v[u][e] = 0.f;
			}
#pragma unroll
			for (int u = 0; u < 4; u++) {
				const int i = i0 + u * ST, j = i / dc, c = (i - j * dc) * 8;
				if (i >= SP * dc) break;
				most = grow_bound(most, v[u]);
				*reinterpret_cast<float4*>(s_m + j * dp + c) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
				*reinterpret_cast<float4*>(s_m + j * dp + c + 4) = make_float4(v[u][4], v[u][5], v[u][6], v[u][7]);
			}
		}
		__syncthreads();
		const int j = tid & (SP - 1), r0 = tid / SP * (R / 4);
		float x[R / 4];
#pragma unroll
		for (int r = 0; r < R / 4; r++) x[r] = 0.f;
		for (int c = 0; c < d; c += 4) {
			const float4 m = *reinterpret_cast<const float4*>(s_m + j * dp + c);
#pragma unroll
			for (int r = 0; r < R / 4; r++) {
				const float4 e = *reinterpret_cast<const float4*>(s_q + (r0 + r) * d + c);
				x[r] = fmaf(m.x, e.x, fmaf(m.y, e.y, fmaf(m.z, e.z, fmaf(m.w, e.w, x[r]))));
			}
		}
		if (p0 + j < hi)
#pragma unroll
			for (int r = 0; r < R / 4; r++) keys[(size_t) (r0 + r) * a.b.max_pages + p0 + j] = ordered32(x[r]);
	}
	most = __reduce_max_sync(0xffffffffu, most);
	if (lane == 0) s_max[warp] = most;
	__syncthreads();
	for (int w = 0; w < ST / 32; w++) most = max(most, s_max[w]);
	for (int r = warp; r < rows; r += ST / 32) {
		const float abs_q = warp_sum(lane < dc ? s_abs[r * dc + lane] : 0.f);
		pick_pages<T, 32>(a, q, s, row0 + r, g, score_error(d, a.rep, abs_q, most), keys + (size_t) r * a.b.max_pages, lane, nullptr);
	}
}

template <typename T>
static int select_typed(const SelectArgs& a, int sms, cudaStream_t s) {
	// A CTA to a row for single tokens, and where there are no more rows than SMs: 32 rows of 8 kv heads over 200 pages 13 us (26 with 16 rows to a CTA), over 1000 35 (64 with 8); 1400 rows
	// of two sequences 160 (72), and 656 (386).  Else 16 rows, 8 where there are many pages (their scores are 8 bytes each: 1400 rows over 200 pages 72 and 76 us, over 1000 428 and 386) and
	// one where shared memory does not hold more.
	const int R = a.b.N <= a.b.B || a.b.N <= sms ? 1 : a.b.max_pages <= 512 ? 16 : a.b.max_pages <= 2048 ? 8 : 1;
	const size_t smem = (size_t) R * a.b.max_pages * 8 + (R > 1 ? (size_t) (R * a.c.d + SP * (a.c.d + 4) + R * a.c.d / 8 + ST / 32 + a.b.max_pages) * 4 : 0);
	const dim3 grid((unsigned) (R > 1 ? a.b.N / R + a.b.B : a.b.N), (unsigned) a.c.G);
	void (*kernel)(SelectArgs) = R == 16 ? paged_select_rows_kernel<T, 16> : R == 8 ? paged_select_rows_kernel<T, 8> : paged_select_step_kernel<T>;
	if (smem > 48 * 1024) XALM_CUDA_CHECK(allow_smem((const void*) kernel, 2048));
	kernel<<<grid, ST, smem, s>>>(a);
	XALM_CUDA_CHECK(cudaGetLastError());
	return XALM_OK;
}

__global__ void paged_status_kernel(int* status, int* taken) { *taken = atomicExch(status, 0); }
int launch_status(int* status, int* taken, cudaStream_t s) {
	paged_status_kernel<<<1, 1, 0, s>>>(status, taken);
	XALM_CUDA_CHECK(cudaGetLastError());
	return XALM_OK;
}

// ---- checks and launches -----------------------------------------------------------------------------------------------------------------------
static int check_strides(const char* what, int G, int P, int pages, int dim, int bytes, long long page, long long slot, long long head) {
	const long long most = 1ll << 40;
	if (page <= 0 || slot <= 0 || head <= 0 || page >= most || slot >= most || head >= most || page * bytes % 16 || slot * bytes % 16 || head * bytes % 16)
		return set_error(XALM_ERR_INVALID, "paged cache: strides of the %s are multiples of 16 bytes, above 0", what);
	const bool by_slot = (G == 1 || head >= dim) && (P == 1 || slot >= (G - 1) * head + dim) && (pages == 1 || page >= (P - 1) * slot + (G - 1) * head + dim);
	const bool by_head = slot >= dim && (G == 1 || head >= (P - 1) * slot + dim) && (pages == 1 || page >= (G - 1) * head + (P - 1) * slot + dim);
	if (!by_slot && !by_head) return set_error(XALM_ERR_INVALID, "paged cache: slots, heads or pages of the %s overlap", what);
	return XALM_OK;
}

static int check_cache(const xalm_paged_cache* c, Cache& o) {
	if (!c) return set_error(XALM_ERR_INVALID, "paged cache: cache is NULL");
	if (!is_type(c->type)) return set_error(XALM_ERR_UNSUPPORTED, "paged cache: type %d (F32, F16 and BF16)", c->type);
	if (c->pages <= 0 || c->kv_heads <= 0 || c->dim <= 0 || c->vdim <= 0 || c->dim > 256 || c->vdim > 256 || c->dim % 8 || c->vdim % 8 || c->kv_heads > 65535)
		return set_error(XALM_ERR_INVALID, "paged cache: %d pages, %d heads of %d and %d entries (multiples of 8, at most 256)", c->pages, c->kv_heads, c->dim, c->vdim);
	int shift = 4;
	while (shift < 8 && (1 << shift) != c->page_size) shift++;
	if ((1 << shift) != c->page_size) return set_error(XALM_ERR_INVALID, "paged cache: pages of %d slots (16, 32, 64, 128 or 256)", c->page_size);
	if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v) || !aligned16(c->means)) return set_error(XALM_ERR_INVALID, "paged cache: pools are at 16-byte boundaries, and not NULL");
	if (!aligned4(c->status)) return set_error(XALM_ERR_INVALID, "paged cache: the status word is not at a 4-byte boundary");
	const int e = element_bytes(c->type);
	XALM_TRY(check_strides("keys", c->kv_heads, c->page_size, c->pages, c->dim, e, c->k_page, c->k_slot, c->k_head));
	XALM_TRY(check_strides("values", c->kv_heads, c->page_size, c->pages, c->vdim, e, c->v_page, c->v_slot, c->v_head));
	o = Cache{(uint8_t*) c->k, (uint8_t*) c->v, (uint8_t*) c->means, c->k_page, c->k_slot, c->k_head, c->v_page, c->v_slot, c->v_head,
	          c->pages, shift, c->kv_heads, c->dim, c->vdim, c->status};
	return XALM_OK;
}
static Span pool_span(const char* what, const Cache& c, const void* p, int dim, int e, long long page, long long slot, long long head) {
	return Span{what, p, ((c.pages - 1) * page + ((1 << c.shift) - 1) * slot + (c.G - 1) * head + dim) * e};
}
static int check_apart_from_cache(const char* call, const Span& out, const Cache& c, const BatchView& b, int e) {
	return check_apart(call, out, {pool_span("the keys' pool", c, c.k, c.d, e, c.k_page, c.k_slot, c.k_head), pool_span("the values' pool", c, c.v, c.dv, e, c.v_page, c.v_slot, c.v_head),
	                               Span{"the mean keys", c.means, (long long) c.pages * c.G * c.d * e}, Span{"the status word", c.status, 4}, Span{"starts", b.starts, 4ll * (b.B + 1)},
	                               Span{"lens", b.lens, 4ll * b.B}, rows_span("the table", b.table, b.table_row, b.max_pages, b.B, 4),
	                               Span{"group_bounds", b.bounds, 4ll * (b.n_groups + 1)}, Span{"group_shared", b.shared, 4ll * b.n_groups}});
}

// Segments of up to 16 (token, head) rows fill one tile of mma.sync, more go to tcgen05's tiles of 256: with 32 rows for either, 8 prompts of 8 tokens behind 4000 take 66 us in place of 54,
// and four groups of 8 sequences behind 8192 shared tokens 70 in place of 57 (8 kv heads, 32 rows to each)
constexpr int SMALL_ROWS = 16;
// A call of no more rows than this to a kv head has no launch of tcgen05: one group behind 8192 tokens takes 25 us in place of 35 with 24 rows, 33 in place of 38 with 64, but 44 in place of
// 39 with 128
constexpr int FEW_ROWS = 64;
// What a piece costs beside its tiles, in tiles, when the work is divided.  mma.sync: 64 sequences behind 8192 shared tokens 97 us, with 2 109.  tcgen05: five prompts of 150 to 700 tokens
// behind 2048 shared ones 147 us, with 2 176.  fp32: 16 sequences of 2500 tokens 79 us, with 6 86.
constexpr int LEAD = 6, LEAD_TC = 12, LEAD_F32 = 1;
constexpr int JOIN_ROWS = 4, JOIN_BLOCKS = 8; // rows to a block of the join, and most blocks to an SM: 128 sequences of 32 heads in two groups 205 us, with 2 223; five long prompts 152, with 16 153

// ---- attention: parts, workspace --------------------------------------------------------------------------------------------------------------
static int plan_attn(const xalm_paged_cache* cache, const Cache& c, const BatchView& b, int heads, int n_lists, Attn& a, size_t* bytes) {
	if (heads <= 0 || heads % c.G) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	if (n_lists < 0 || n_lists > MAX_LIST) return set_error(XALM_ERR_INVALID, "paged attention: lists of %d pages (at most %d)", n_lists, MAX_LIST);
	int sms = 0;
	XALM_TRY(sm_count(cache->device, &sms));
	a = Attn{};
	a.c = c;
	a.b = b;
	a.H = heads;
	a.rep = heads / c.G;
	a.S = n_lists;
	// Two kernels divide the segments by their rows: up to 16 fill one 16-row tile, more go to tcgen05.  The second is launched only where some segment may have more.
	const bool f32 = cache->type == XALM_F32;
	const bool tc = !f32 && !n_lists && tc_fits(c, b) && (b.n_groups || b.N > b.B) && (long long) b.N * a.rep > FEW_ROWS;
	a.n_parts = tc ? 2 : 1;
	size_t at = 0;
	auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
	for (int i = 0; i < a.n_parts; i++) {
		Part& p = a.part[i];
		const bool big = tc && i == 0;
		p.M = big ? TC_ROWS : 16;
		p.grid = sms * (big ? 1 : f32 ? rows_ctas_per_sm(c, b, n_lists) : mma_ctas_per_sm(c, b, n_lists));
		p.lead = big ? LEAD_TC : f32 ? LEAD_F32 : LEAD;
		p.least_rows = big ? SMALL_ROWS + 1 : 1;
		p.most_rows = tc && !big ? SMALL_ROWS : 0x7fffffff;
		const long long rows = (long long) b.N * a.rep;
		// A segment has at most its rows / M + 1 tiles, in a part that takes short ones only it has one; and there are no more segments than have room for the part's least rows, of sequences
		// as of groups.  (128 single tokens of 32 heads of 128 over 8 in two groups: 69 MB; with a tile of 256 rows for every sequence 174.)
		const long long whole = tc && !big ? 0 : rows / p.M, most = rows / p.least_rows;
		const long long tiles = n_lists ? (long long) b.N * ((a.rep + p.M - 1) / p.M)
		                                : whole + std::min((long long) b.B, most) + (b.n_groups ? whole + std::min((long long) b.n_groups, most) : 0);
		if (tiles * c.G + p.grid > 0x7fffffff / p.M) return set_error(XALM_ERR_INVALID, "paged attention: %d rows of %d heads are too many for one call", b.N, heads);
		const long long keys = (long long) b.max_pages << c.shift, work = n_lists ? (((long long) n_lists << c.shift) + KT - 1) / KT : keys / KT + 1;
		if (tiles * c.G > 0x7fffffffll / (work + p.lead)) return set_error(XALM_ERR_INVALID, "paged attention: %d rows of %d heads over up to %lld keys are too many for one call", b.N, heads, work * KT);
		p.slots = n_lists || !b.n_groups ? 2 * p.grid : (int) (tiles * c.G) + p.grid;
		p.o = (float*) take((size_t) p.slots * p.M * c.dv * 4);
		p.ml = (float2*) take((size_t) p.slots * p.M * 8);
		p.head = (Head*) take((size_t) p.grid * sizeof(Head));
		if (!n_lists) {
			p.cum_w = (int*) take((size_t) (b.B + b.n_groups + 1) * 4);
			p.cum_u = (int*) take((size_t) (b.B + b.n_groups + 1) * 4);
			p.shs = (int*) take((size_t) b.B * 4);
		}
	}
	a.row_blocks = n_lists || !b.n_groups ? 0 : (int) std::min(((long long) b.N * heads + JOIN_ROWS - 1) / JOIN_ROWS, (long long) sms * JOIN_BLOCKS);
	*bytes = at;
	return XALM_OK;
}

static int attend(const xalm_paged_cache* cache, const xalm_paged_batch* batch, const void* q, long long q_row, int heads, const int* lists, int n_lists, float scale,
                  void* out, long long out_row, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
	Cache c;
	BatchView b;
	Attn a;
	size_t need = 0;
	XALM_TRY(check_cache(cache, c));
	XALM_TRY(check_batch(batch, c, b));
	if (heads <= 0 || heads > 65535) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	const int e = element_bytes(cache->type);
	if (b.N) {
		XALM_TRY(check_rows("q", q, q_row, heads * c.d, e));
		XALM_TRY(check_rows("out", out, out_row, heads * c.dv, e));
	}
	if (heads % c.G) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	if (n_lists > MAX_LIST) return set_error(XALM_ERR_INVALID, "paged attention: lists of %d pages (at most %d)", n_lists, MAX_LIST);
	if (!aligned4(lse) || !aligned4(lists)) return set_error(XALM_ERR_INVALID, "paged attention: lse and lists are at 4-byte boundaries");
	if (!isfinite(scale)) return set_error(XALM_ERR_INVALID, "paged attention: scale is not finite");
	if (b.N == 0 || b.B == 0) return XALM_OK;
	if (!workspace || ((uintptr_t) workspace & 255)) return set_error(XALM_ERR_INVALID, "paged attention: the workspace is NULL or not at a 256-byte boundary");
	XALM_TRY(plan_attn(cache, c, b, heads, n_lists, a, &need));
	if (rows_meet(q, q_row * e, (long long) heads * c.d * e, out, out_row * e, (long long) heads * c.dv * e, b.N)) return set_error(XALM_ERR_INVALID, "paged attention: out overlaps q");
	{
		const Span sq = rows_span("q", q, q_row, heads * c.d, b.N, e), so = rows_span("out", out, out_row, heads * c.dv, b.N, e), sl = {"lse", lse, 4ll * b.N * heads},
		           sp = {"the lists", lists, 4ll * b.N * c.G * n_lists}, sw = {"the workspace", workspace, (long long) need};
		for (const Span& x : {so, sl, sw}) XALM_TRY(check_apart_from_cache("paged attention", x, c, b, e));
		XALM_TRY(check_apart("paged attention", sw, {sq, so, sl, sp}));
		XALM_TRY(check_apart("paged attention", sl, {sq, so, sp}));
		XALM_TRY(check_apart("paged attention", so, {sp}));
	}
	if (workspace_bytes < need) return set_error(XALM_ERR_INVALID, "paged attention: a workspace of %zu bytes is needed, %zu given", need, workspace_bytes);
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	uint8_t* base = (uint8_t*) workspace;
	for (int i = 0; i < a.n_parts; i++) {
		Part& p = a.part[i];
		p.o = (float*) (base + (size_t) p.o);
		p.ml = (float2*) (base + (size_t) p.ml);
		p.head = (Head*) (base + (size_t) p.head);
		if (!n_lists) {
			p.cum_w = (int*) (base + (size_t) p.cum_w);
			p.cum_u = (int*) (base + (size_t) p.cum_u);
			p.shs = (int*) (base + (size_t) p.shs);
		}
	}
	a.q = (const uint8_t*) q;
	a.q_row = q_row;
	a.out = (uint8_t*) out;
	a.out_row = out_row;
	a.lse = lse;
	a.scale = scale;
	a.lists = lists;
	cudaStream_t s = (cudaStream_t) stream;
	if (cache->type == XALM_F32) XALM_TRY(launch_attn_rows(a, s));
	else {
		if (a.n_parts == 2) XALM_TRY(launch_attn_tc(a, 0, cache->type, s));
		XALM_TRY(launch_attn_mma(a, a.n_parts - 1, cache->type, s));
	}
	return launch_join(a, cache->type, s);
}

} // namespace paged
} // namespace xalm

using namespace xalm;
using namespace xalm::paged;

extern "C" {

int xalm_cuda_paged_append(const xalm_paged_cache* cache, const xalm_paged_batch* batch, const void* k, long long k_row, const void* v, long long v_row, const void* q,
                           long long q_row, int heads, int in_type, void* q_out, long long q_out_row, const float* freq, int rot_half, float rot_mag, int neighbours,
                           void* stream) {
	AppendArgs a = {};
	XALM_TRY(check_cache(cache, a.c));
	XALM_TRY(check_batch(batch, a.c, a.b));
	if (!is_type(in_type)) return set_error(XALM_ERR_UNSUPPORTED, "paged append: rows of type %d (F32, F16 and BF16)", in_type);
	if (!aligned4(freq)) return set_error(XALM_ERR_INVALID, "paged append: freq is not at a 4-byte boundary");
	if (rot_half < 0 || 2 * rot_half > a.c.d || (rot_half && !freq)) return set_error(XALM_ERR_INVALID, "paged append: rotation of %d pairs in heads of %d", rot_half, a.c.d);
	if (q && (heads <= 0 || heads > 65535)) return set_error(XALM_ERR_INVALID, "paged append: %d query heads", heads);
	if (a.b.N) {
		const int ei = element_bytes(in_type), e = element_bytes(cache->type);
		XALM_TRY(check_rows("k", k, k_row, a.c.G * a.c.d, ei));
		XALM_TRY(check_rows("v", v, v_row, a.c.G * a.c.dv, ei));
		if (q) {
			XALM_TRY(check_rows("q", q, q_row, heads * a.c.d, ei));
			XALM_TRY(check_rows("q_out", q_out, q_out_row, heads * a.c.d, e));
			// in place only where a thread has all that its results are made of
			const bool in_place = q == q_out && q_row == q_out_row && in_type == cache->type && (neighbours || rot_half % 8 == 0);
			if (!in_place && rows_meet(q, q_row * ei, (long long) heads * a.c.d * ei, q_out, q_out_row * e, (long long) heads * a.c.d * e, a.b.N))
				return set_error(XALM_ERR_INVALID, "paged append: q_out overlaps q (in place: the same rows of the cache's type, and halves of a multiple of 8 pairs or neighbours)");
		}
	}
	if (a.b.N == 0 || a.b.B == 0) return XALM_OK;
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	a.k = (const uint8_t*) k; a.v = (const uint8_t*) v; a.q = (const uint8_t*) q;
	a.k_row = k_row; a.v_row = v_row; a.q_row = q_row; a.q_out_row = q_out_row;
	a.q_out = (uint8_t*) q_out;
	a.H = heads;
	a.freq = freq; a.rot = rot_half; a.mag = rot_mag; a.neighbours = neighbours;
	cudaStream_t s = (cudaStream_t) stream;
	a.paired = !neighbours && rot_half % 8 == 0;
	a.per_head = (a.c.d - (a.paired ? rot_half : 0)) / 8;
	a.per_value = a.c.dv / 8;
	a.by_head = (unsigned) ((0x100000000ull + a.per_head - 1) / a.per_head);
	a.by_value = (unsigned) ((0x100000000ull + a.per_value - 1) / a.per_value);
	int sms = 0;
	XALM_TRY(sm_count(cache->device, &sms));
	if (q) {
		const int ei = element_bytes(in_type), e = element_bytes(cache->type);
		const long long width = (long long) heads * a.c.d * e;
		const Span out = rows_span("q_out", q_out, q_out_row, heads * a.c.d, a.b.N, e);
		XALM_TRY(check_apart_from_cache("paged append", out, a.c, a.b, e));
		XALM_TRY(check_apart("paged append", out, {Span{"freq", freq, 4ll * rot_half}}));
		if (rows_meet(k, k_row * ei, (long long) a.c.G * a.c.d * ei, q_out, q_out_row * e, width, a.b.N) || rows_meet(v, v_row * ei, (long long) a.c.G * a.c.dv * ei, q_out, q_out_row * e, width, a.b.N))
			return set_error(XALM_ERR_INVALID, "paged append: q_out overlaps k or v");
	}
	// Four rows to a CTA once that still gives every SM one.  32 and 8 heads of 128, one and four rows to a CTA: 256 rows 4.5 and 5.9 us, 576 4.9 and 5.9, 1024 8.0 and 7.1, 8192 43 and 39
	const bool many = a.b.N >= sms * 4;
	void (*kernel)(AppendArgs) = nullptr;
	switch (in_type * 16 + cache->type) {
#define XALM_PAGED_APPEND(I, IT, C, CT) case IT * 16 + CT: kernel = many ? paged_append_kernel<I, C, 4> : paged_append_kernel<I, C, 1>; break;
		XALM_PAGED_APPEND(float, XALM_F32, float, XALM_F32)
		XALM_PAGED_APPEND(float, XALM_F32, __half, XALM_F16)
		XALM_PAGED_APPEND(float, XALM_F32, __nv_bfloat16, XALM_BF16)
		XALM_PAGED_APPEND(__half, XALM_F16, float, XALM_F32)
		XALM_PAGED_APPEND(__half, XALM_F16, __half, XALM_F16)
		XALM_PAGED_APPEND(__half, XALM_F16, __nv_bfloat16, XALM_BF16)
		XALM_PAGED_APPEND(__nv_bfloat16, XALM_BF16, float, XALM_F32)
		XALM_PAGED_APPEND(__nv_bfloat16, XALM_BF16, __half, XALM_F16)
		XALM_PAGED_APPEND(__nv_bfloat16, XALM_BF16, __nv_bfloat16, XALM_BF16)
#undef XALM_PAGED_APPEND
	}
	kernel<<<many ? (a.b.N + 3) / 4 : a.b.N, AT, 0, s>>>(a);
	XALM_CUDA_CHECK(cudaGetLastError());
	if (a.c.means) {
		const dim3 grid((unsigned) ((a.b.N >> a.c.shift) + a.b.B), (unsigned) a.c.G);
		void (*means)(Cache, BatchView) = cache->type == XALM_F32   ? paged_means_kernel<float>
		                                  : cache->type == XALM_F16 ? paged_means_kernel<__half>
		                                                            : paged_means_kernel<__nv_bfloat16>;
		cudaLaunchConfig_t cfg = {};
		cfg.gridDim = grid;
		cfg.blockDim = dim3(128);
		cfg.stream = s;
		cudaLaunchAttribute at[1];
		at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
		at[0].val.programmaticStreamSerializationAllowed = 1;
		cfg.attrs = at;
		cfg.numAttrs = 1;
		XALM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, means, a.c, a.b));
	}
	return XALM_OK;
}

int xalm_cuda_paged_status(const xalm_paged_cache* cache, int* taken, void* stream) {
	Cache c;
	XALM_TRY(check_cache(cache, c));
	if (!taken || !c.status || !aligned4(taken)) return set_error(XALM_ERR_INVALID, "paged status: %s", !taken || !c.status ? "taken or the cache's status word is NULL" : "taken is not at a 4-byte boundary");
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	return launch_status(c.status, taken, (cudaStream_t) stream);
}

int xalm_cuda_paged_workspace(const xalm_paged_cache* cache, const xalm_paged_batch* batch, int heads, int n_lists, size_t* bytes) {
	Cache c;
	BatchView b;
	Attn a;
	if (!bytes) return set_error(XALM_ERR_INVALID, "paged attention: bytes is NULL");
	XALM_TRY(check_cache(cache, c));
	XALM_TRY(check_batch(batch, c, b));
	return plan_attn(cache, c, b, heads, n_lists, a, bytes);
}

int xalm_cuda_paged_attend(const xalm_paged_cache* cache, const xalm_paged_batch* batch, const void* q, long long q_row, int heads, float scale, void* out,
                           long long out_row, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
	return attend(cache, batch, q, q_row, heads, nullptr, 0, scale, out, out_row, lse, workspace, workspace_bytes, stream);
}

int xalm_cuda_paged_attend_selected(const xalm_paged_cache* cache, const xalm_paged_batch* batch, const void* q, long long q_row, int heads, const int* lists,
                                    int n_lists, float scale, void* out, long long out_row, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
	if (!lists || n_lists <= 0) return set_error(XALM_ERR_INVALID, "paged attention: lists is NULL or of %d pages", n_lists);
	return attend(cache, batch, q, q_row, heads, lists, n_lists, scale, out, out_row, lse, workspace, workspace_bytes, stream);
}

int xalm_cuda_paged_select(const xalm_paged_cache* cache, const xalm_paged_batch* batch, const void* q, long long q_row, int heads, int top, int first, int recent,
                           int* out, void* stream) {
	SelectArgs a = {};
	XALM_TRY(check_cache(cache, a.c));
	XALM_TRY(check_batch(batch, a.c, a.b));
	if (!a.c.means) return set_error(XALM_ERR_STATE, "paged select: the cache keeps no mean keys");
	if (heads <= 0 || heads % a.c.G || heads > 65535) return set_error(XALM_ERR_INVALID, "paged select: %d query heads over %d", heads, a.c.G);
	if (top <= 0 || top > MAX_LIST || first < 0 || recent < 0 || first > top || recent > top || first + recent + 1 > top)
		return set_error(XALM_ERR_INVALID, "paged select: %d pages, of them the first %d, %d recent ones and the token's own (at most %d)", top, first, recent, MAX_LIST);
	if (a.b.max_pages > 24576) return set_error(XALM_ERR_INVALID, "paged select: sequences of %d pages (at most 24576)", a.b.max_pages);
	if (a.b.N) {
		XALM_TRY(check_rows("q", q, q_row, heads * a.c.d, element_bytes(cache->type)));
		if (!out || !aligned4(out)) return set_error(XALM_ERR_INVALID, "paged select: out is NULL or not at a 4-byte boundary");
	}
	if (a.b.N == 0 || a.b.B == 0) return XALM_OK;
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	a.q = (const uint8_t*) q;
	a.q_row = q_row;
	a.H = heads;
	a.rep = heads / a.c.G;
	a.top = top;
	a.first = first;
	int sms = 0;
	XALM_TRY(sm_count(cache->device, &sms));
	{
		const int e = element_bytes(cache->type);
		const Span so = {"out", out, 4ll * a.b.N * a.c.G * top};
		XALM_TRY(check_apart_from_cache("paged select", so, a.c, a.b, e));
		XALM_TRY(check_apart("paged select", so, {rows_span("q", q, q_row, heads * a.c.d, a.b.N, e)}));
	}
	a.recent = recent;
	a.out = out;
	cudaStream_t s = (cudaStream_t) stream;
	return cache->type == XALM_F32 ? select_typed<float>(a, sms, s) : cache->type == XALM_F16 ? select_typed<__half>(a, sms, s) : select_typed<__nv_bfloat16>(a, sms, s);
}

} // extern "C"
