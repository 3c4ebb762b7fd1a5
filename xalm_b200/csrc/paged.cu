// paged.cu — the paged cache: entry points (include/xalm_cuda.h, xalm_cuda_paged_*), appending to pages, choosing pages.
//
// Several sequences share one pool of pages; a table names each sequence's pages.  Lengths and tables are read on the device, so that a captured graph serves
// every step of a batch; what the host has to know is how large the arrays are.
#include "paged.cuh"

#include <math.h>

#include <algorithm>

#include "family.h"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// append: a CTA per new token; row's position p = len - n + i, page table[p / P], slot p % P.  Bound by HBM (every element in and out once): a thread takes
// eight neighbouring elements of a head, and its partners of the rotation from the same 16 or 32 bytes or from the chunk half a rotation away (the second
// reading of a line hits L1).  The angle p * freq is taken in 64 bits and brought into [-pi, pi] there: in 32 bits position 100000 is 0.004 rad off.
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
};

constexpr int AT = 256;

template <typename I, typename T>
__global__ void __launch_bounds__(AT) paged_append_kernel(const AppendArgs a) {
	__shared__ float s_cos[128], s_sin[128];
	pdl_wait();
	pdl_launch_dependents();
	const int row = blockIdx.x, tid = threadIdx.x, d = a.c.d, dv = a.c.dv, G = a.c.G;
	const int s = seq_of_row(a.b, row);
	const View view = view_of(a.c, a.b);
	const Seq q = seq_of(view, s);
	const bool in = row >= q.a && row < q.a + q.n;
	if (tid == 0 && row == q.a && !seq_ok(view, s)) report(a.c, ERR_BATCH);
	if (!in) return; // behind the last sequence
	const int pos = q.len - q.n + row - q.a;
	if (pos < 0) return;
	const int page = page_of(a.c, a.b, s, pos >> a.c.shift), slot = pos & ((1 << a.c.shift) - 1);
	if (page < 0 && tid == 0) report(a.c, ERR_PAGE);
	for (int i = tid; i < a.rot; i += AT) {
		const double x = (double) pos * (double) a.freq[i], turns = rint(x * 0.15915494309189535);
		float sn, cs;
		sincosf((float) fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, x)), &sn, &cs); // 2 pi as the sum of two doubles
		s_cos[i] = cs * a.mag;
		s_sin[i] = sn * a.mag;
	}
	__syncthreads();
	const int dc = d / 8, vc = dv / 8, n_q = a.q ? a.H * dc : 0, n_k = n_q + G * dc, n_all = n_k + (page < 0 ? 0 : G * vc);
	for (int i = tid; i < n_all; i += AT) {
		float x[8];
		if (i >= n_k) { // a value
			const int h = (i - n_k) / vc, c = (i - n_k) % vc * 8;
			load8(reinterpret_cast<const I*>(a.v) + (long long) row * a.v_row + h * dv + c, x);
			store8(reinterpret_cast<T*>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot + h * a.c.v_head + c, x);
			continue;
		}
		const bool key = i >= n_q;
		if (key && page < 0) break;
		const int h = (key ? i - n_q : i) / dc, c = (key ? i - n_q : i) % dc * 8;
		const I* in_head = key ? reinterpret_cast<const I*>(a.k) + (long long) row * a.k_row + h * d : reinterpret_cast<const I*>(a.q) + (long long) row * a.q_row + h * d;
		load8(in_head + c, x);
		float y[8];
#pragma unroll
		for (int e = 0; e < 8; e++) y[e] = x[e];
		if (c < 2 * a.rot) {
			if (a.neighbours) {
#pragma unroll
				for (int e = 0; e < 8; e += 2) {
					const int f = (c + e) / 2;
					if (f < a.rot) {
						y[e] = x[e] * s_cos[f] - x[e + 1] * s_sin[f];
						y[e + 1] = x[e + 1] * s_cos[f] + x[e] * s_sin[f];
					}
				}
			} else {
				const bool low = c < a.rot;
				float p[8];
				if (a.rot % 8 == 0) load8(in_head + (low ? c + a.rot : c - a.rot), p); // a chunk lies in one half
#pragma unroll
				for (int e = 0; e < 8; e++) {
					const int at = c + e;
					if (at >= 2 * a.rot) continue;
					const int f = at < a.rot ? at : at - a.rot;
					const float o = a.rot % 8 == 0 ? p[e] : to_f(in_head[at < a.rot ? at + a.rot : at - a.rot]);
					y[e] = at < a.rot ? x[e] * s_cos[f] - o * s_sin[f] : x[e] * s_cos[f] + o * s_sin[f];
				}
			}
		}
		if (key) store8(reinterpret_cast<T*>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot + h * a.c.k_head + c, y);
		else store8(reinterpret_cast<T*>(a.q_out) + (long long) row * a.q_out_row + h * d + c, y);
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
	const Seq q = seq_of(view_of(c, b), lo);
	const int first = max(q.len - q.n, 0) >> c.shift; // page of the first new token
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
// select: a CTA per (row, kv head).  score_j = (sum over the head's queries) . mean_j, summed in 64 bits: which page is the last to be taken must not hang on the
// order of a sum.  The pages are taken by their scores as ordered integers, equal ones from the lowest index on; a NaN counts as the lowest finite number.
// =========================================================================================================================================
struct SelectArgs {
	Cache c;
	BatchView b;
	const uint8_t* q;
	long long q_row;
	int H, rep, top, first, recent;
	int* out;
};
constexpr int ST = 256;

__device__ __forceinline__ unsigned long long ordered(double x) {
	const double big = 1.7976931348623157e308;
	x = x != x ? -big : fmin(fmax(x, -big), big) + 0.0;
	const long long b = __double_as_longlong(x);
	return b < 0 ? ~(unsigned long long) b : (unsigned long long) b | (1ull << 63);
}

template <typename T>
__global__ void __launch_bounds__(ST) paged_select_kernel(const SelectArgs a) {
	extern __shared__ __align__(16) unsigned long long keys[]; // one per page
	__shared__ double s_q[256];
	__shared__ int s_hist[256], s_warp[ST / 32];
	__shared__ unsigned long long s_prefix;
	__shared__ int s_need;
	pdl_wait();
	pdl_launch_dependents();
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x, g = blockIdx.y, d = a.c.d;
	const int s = seq_of_row(a.b, row);
	const View view = view_of(a.c, a.b);
	const Seq q = seq_of(view, s);
	if (!row_in_seq(q, row)) return;
	const int pos = q.len - q.n + row - q.a, last = pos < 0 ? -1 : pos >> a.c.shift;
	if (tid == 0 && row == q.a && !seq_ok(view, s)) report(a.c, ERR_BATCH);
	int* out = a.out + ((long long) row * a.c.G + g) * a.top;
	const int lo = min(a.first, last + 1), hi = max(last - a.recent, lo); // pages [lo, hi) are chosen by score, those before and from hi to last are always
	const int fixed = lo + last + 1 - hi, want = min(a.top - fixed, hi - lo);
	unsigned long long least = 0; // keys above it are taken, of those equal to it the first `ties`
	int ties = 0;
	if (want > 0 && want < hi - lo) {
		for (int i = tid; i < d; i += ST) {
			double x = 0;
			for (int r = 0; r < a.rep; r++) x += (double) to_f(reinterpret_cast<const T*>(a.q)[(long long) row * a.q_row + (g * a.rep + r) * d + i]);
			s_q[i] = x;
		}
		__syncthreads();
		const int sub = lane & 7; // eight lanes to a page
		for (int j0 = lo + warp * 4; j0 < hi; j0 += ST / 8) {
			const int j = j0 + (lane >> 3);
			const int page = j < hi ? page_of(a.c, a.b, s, j) : -1;
			double x = 0;
			if (page >= 0) {
				const T* m = reinterpret_cast<const T*>(a.c.means) + ((long long) page * a.c.G + g) * d;
				for (int c = sub * 8; c < d; c += 64) {
					float v[8];
					load8(m + c, v);
#pragma unroll
					for (int e = 0; e < 8; e++) x = fma((double) v[e], s_q[c + e], x);
				}
			} else if (j < hi && sub == 0) report(a.c, ERR_PAGE);
#pragma unroll
			for (int o = 4; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
			if (sub == 0 && j < hi) keys[j] = ordered(x);
		}
		if (tid == 0) { s_prefix = 0; s_need = want; }
		// the want-th largest key, eight bits at a time
		for (int shift = 56; shift >= 0; shift -= 8) {
			s_hist[tid] = 0;
			__syncthreads();
			const unsigned long long prefix = s_prefix;
			for (int j = lo + tid; j < hi; j += ST)
				if (shift == 56 || keys[j] >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_hist[(int) (keys[j] >> shift) & 255], 1);
			__syncthreads();
			if (warp == 0) { // from the top bin down: lane l holds bins 255 - 8 l .. 248 - 8 l
				int n[8], sum = 0;
#pragma unroll
				for (int e = 0; e < 8; e++) { n[e] = s_hist[255 - lane * 8 - e]; sum += n[e]; }
				int before = sum;
#pragma unroll
				for (int o = 1; o < 32; o <<= 1) {
					const int x = __shfl_up_sync(0xffffffffu, before, o);
					if (lane >= o) before += x;
				}
				before -= sum;
				const int need = s_need;
				__syncwarp();
				if (before < need && before + sum >= need) {
					int acc = before;
#pragma unroll
					for (int e = 0; e < 8; e++) {
						if (acc < need && acc + n[e] >= need) {
							s_prefix = prefix | (unsigned long long) (255 - lane * 8 - e) << shift;
							s_need = need - acc;
						}
						acc += n[e];
					}
				}
			}
			__syncthreads();
		}
		least = s_prefix;
		ties = s_need;
	} else if (want > 0) {
		least = 0; // all of them
	}
	const bool by_score = want > 0 && want < hi - lo;
	// in ascending order, a block's worth of pages at a time
	int written = 0, tied = 0;
	for (int base = 0; base <= last; base += ST) {
		const int j = base + tid;
		const bool mid = j >= lo && j < hi;
		const bool tie = by_score && mid && keys[j] == least;
		// place among the ties before it
		const unsigned tm = __ballot_sync(0xffffffffu, tie);
		__syncthreads();
		if (lane == 0) s_warp[warp] = __popc(tm);
		__syncthreads();
		int rank = tied + __popc(tm & ((1u << lane) - 1));
		for (int w = 0; w < ST / 32; w++) {
			if (w < warp) rank += s_warp[w];
			tied += s_warp[w];
		}
		const bool take = j <= last && (mid ? (by_score ? keys[j] > least || (tie && rank < ties) : want > 0) : true);
		const unsigned om = __ballot_sync(0xffffffffu, take);
		__syncthreads();
		if (lane == 0) s_warp[warp] = __popc(om);
		__syncthreads();
		int at = written + __popc(om & ((1u << lane) - 1));
		for (int w = 0; w < ST / 32; w++) {
			if (w < warp) at += s_warp[w];
			written += s_warp[w];
		}
		if (take && at < a.top) out[at] = j;
	}
	for (int i = written + tid; i < a.top; i += ST) out[i] = -1;
}

// ---- checks and launches -----------------------------------------------------------------------------------------------------------------------
static int element_bytes(int type) { return type == XALM_F32 ? 4 : 2; }
static bool is_type(int type) { return type == XALM_F32 || type == XALM_F16 || type == XALM_BF16; }
static bool aligned16(const void* p) { return ((uintptr_t) p & 15) == 0; }

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
	const int e = element_bytes(c->type);
	XALM_TRY(check_strides("keys", c->kv_heads, c->page_size, c->pages, c->dim, e, c->k_page, c->k_slot, c->k_head));
	XALM_TRY(check_strides("values", c->kv_heads, c->page_size, c->pages, c->vdim, e, c->v_page, c->v_slot, c->v_head));
	o = Cache{(uint8_t*) c->k, (uint8_t*) c->v, (uint8_t*) c->means, c->k_page, c->k_slot, c->k_head, c->v_page, c->v_slot, c->v_head,
	          c->pages, shift, c->kv_heads, c->dim, c->vdim, c->status};
	return XALM_OK;
}
static int check_batch(const xalm_paged_batch* b, BatchView& o) {
	if (!b) return set_error(XALM_ERR_INVALID, "paged cache: batch is NULL");
	if (b->rows < 0 || b->seqs < 0 || b->max_pages < 0 || b->groups < 0 || b->table_row < b->max_pages)
		return set_error(XALM_ERR_INVALID, "paged cache: %d rows, %d sequences of %d pages (rows %lld apart), %d groups", b->rows, b->seqs, b->max_pages, b->table_row, b->groups);
	if ((long long) b->seqs + b->groups > MAX_SEGMENTS) return set_error(XALM_ERR_INVALID, "paged cache: %d sequences and %d groups are more than %d", b->seqs, b->groups, MAX_SEGMENTS);
	if (b->seqs && (!b->starts || !b->lens || (b->max_pages && !b->table))) return set_error(XALM_ERR_INVALID, "paged cache: starts/lens/table is NULL");
	if (b->groups && (!b->group_bounds || !b->group_shared)) return set_error(XALM_ERR_INVALID, "paged cache: group_bounds/group_shared is NULL");
	o = BatchView{b->rows, b->seqs, b->max_pages, b->groups, b->starts, b->lens, b->table, b->table_row, b->group_bounds, b->group_shared};
	return XALM_OK;
}
static int check_rows(const char* what, const void* p, long long row, int least, int bytes) {
	if (!p || !aligned16(p) || row < least || row * bytes % 16)
		return set_error(XALM_ERR_INVALID, "paged cache: rows of %s are at 16-byte boundaries, %d entries or more apart, and not NULL", what, least);
	return XALM_OK;
}

// The calling thread's device is what it was when the call returns
struct OnDevice {
	int before = -1;
	int set(int device) {
		XALM_CUDA_CHECK(cudaGetDevice(&before));
		if (before == device) before = -1;
		else {
			const cudaError_t e = cudaSetDevice(device);
			if (e != cudaSuccess) {
				before = -1;
				return set_error(XALM_ERR_CUDA, "cudaSetDevice(%d) failed: %s", device, cudaGetErrorString(e));
			}
		}
		return XALM_OK;
	}
	~OnDevice() {
		if (before >= 0) cudaSetDevice(before);
	}
};
static int sm_count(int device, int* n) {
	static int known[64]; // the same number whoever writes it
	if (device >= 0 && device < 64 && known[device]) { *n = known[device]; return XALM_OK; }
	XALM_CUDA_CHECK(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device));
	if (device >= 0 && device < 64) known[device] = *n;
	return XALM_OK;
}

constexpr int SMALL_ROWS = 16;
constexpr int LEAD = 2, LEAD_TC = 4;

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
	const bool tc = !f32 && !n_lists && tc_fits(c, b) && (b.n_groups || b.N > b.B) && (long long) b.N * a.rep > SMALL_ROWS;
	a.n_parts = tc ? 2 : 1;
	size_t at = 0;
	auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
	for (int i = 0; i < a.n_parts; i++) {
		Part& p = a.part[i];
		const bool big = tc && i == 0;
		p.M = big ? TC_ROWS : 16;
		p.grid = sms * (big ? 1 : f32 ? 2 : mma_ctas_per_sm(c, b, n_lists));
		p.lead = big ? LEAD_TC : LEAD;
		p.least_rows = big ? SMALL_ROWS + 1 : 1;
		p.most_rows = tc && !big ? SMALL_ROWS : 0x7fffffff;
		const long long rows = (long long) b.N * a.rep;
		// a segment of `rows` rows has at most rows / M + 1 tiles, a part that takes short ones only has one
		const long long tiles = n_lists ? (long long) b.N * ((a.rep + p.M - 1) / p.M) : (tc && !big ? 0 : rows / p.M) + b.B + (b.n_groups ? (tc && !big ? 0 : rows / p.M) + b.n_groups : 0);
		if (tiles * c.G + p.grid > 0x7fffffff / p.M) return set_error(XALM_ERR_INVALID, "paged attention: %d rows of %d heads are too many for one call", b.N, heads);
		p.slots = n_lists || !b.n_groups ? 2 * p.grid : (int) (tiles * c.G) + p.grid;
		p.o = (float*) take((size_t) p.slots * p.M * c.dv * 4);
		p.ml = (float2*) take((size_t) p.slots * p.M * 8);
		p.head = (Head*) take((size_t) p.grid * sizeof(Head));
		if (!n_lists) {
			p.cum_w = (long long*) take((size_t) (b.B + b.n_groups + 1) * 8);
			p.cum_u = (int*) take((size_t) (b.B + b.n_groups + 1) * 4);
			p.shs = (int*) take((size_t) b.B * 4);
		}
	}
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
	XALM_TRY(check_batch(batch, b));
	if (heads <= 0 || heads > 65535) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	const int e = element_bytes(cache->type);
	if (b.N) {
		XALM_TRY(check_rows("q", q, q_row, heads * c.d, e));
		XALM_TRY(check_rows("out", out, out_row, heads * c.dv, e));
	}
	if (heads % c.G) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	if (n_lists > MAX_LIST) return set_error(XALM_ERR_INVALID, "paged attention: lists of %d pages (at most %d)", n_lists, MAX_LIST);
	if (!isfinite(scale)) return set_error(XALM_ERR_INVALID, "paged attention: scale is not finite");
	if (b.N == 0 || b.B == 0) return XALM_OK;
	if (!workspace || ((uintptr_t) workspace & 255)) return set_error(XALM_ERR_INVALID, "paged attention: the workspace is NULL or not at a 256-byte boundary");
	XALM_TRY(plan_attn(cache, c, b, heads, n_lists, a, &need));
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
			p.cum_w = (long long*) (base + (size_t) p.cum_w);
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
	XALM_TRY(check_batch(batch, a.b));
	if (!is_type(in_type)) return set_error(XALM_ERR_UNSUPPORTED, "paged append: rows of type %d (F32, F16 and BF16)", in_type);
	if (rot_half < 0 || 2 * rot_half > a.c.d || (rot_half && !freq)) return set_error(XALM_ERR_INVALID, "paged append: rotation of %d pairs in heads of %d", rot_half, a.c.d);
	if (q && (heads <= 0 || heads > 65535)) return set_error(XALM_ERR_INVALID, "paged append: %d query heads", heads);
	if (a.b.N) {
		const int ei = element_bytes(in_type), e = element_bytes(cache->type);
		XALM_TRY(check_rows("k", k, k_row, a.c.G * a.c.d, ei));
		XALM_TRY(check_rows("v", v, v_row, a.c.G * a.c.dv, ei));
		if (q) {
			XALM_TRY(check_rows("q", q, q_row, heads * a.c.d, ei));
			XALM_TRY(check_rows("q_out", q_out, q_out_row, heads * a.c.d, e));
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
	void (*kernel)(AppendArgs) = nullptr;
	switch (in_type * 16 + cache->type) {
#define XALM_PAGED_APPEND(I, IT, C, CT) case IT * 16 + CT: kernel = paged_append_kernel<I, C>; break;
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
	kernel<<<a.b.N, AT, 0, s>>>(a);
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

int xalm_cuda_paged_workspace(const xalm_paged_cache* cache, const xalm_paged_batch* batch, int heads, int n_lists, size_t* bytes) {
	Cache c;
	BatchView b;
	Attn a;
	if (!bytes) return set_error(XALM_ERR_INVALID, "paged attention: bytes is NULL");
	XALM_TRY(check_cache(cache, c));
	XALM_TRY(check_batch(batch, b));
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
	XALM_TRY(check_batch(batch, a.b));
	if (!a.c.means) return set_error(XALM_ERR_STATE, "paged select: the cache keeps no mean keys");
	if (heads <= 0 || heads % a.c.G || heads > 65535) return set_error(XALM_ERR_INVALID, "paged select: %d query heads over %d", heads, a.c.G);
	if (top <= 0 || top > MAX_LIST || first < 0 || recent < 0 || first > top || recent > top || first + recent + 1 > top)
		return set_error(XALM_ERR_INVALID, "paged select: %d pages, of them the first %d, %d recent ones and the token's own (at most %d)", top, first, recent, MAX_LIST);
	const size_t smem = (size_t) a.b.max_pages * 8;
	if (smem > 192 * 1024) return set_error(XALM_ERR_INVALID, "paged select: sequences of %d pages (at most %d)", a.b.max_pages, 192 * 1024 / 8);
	if (a.b.N) {
		XALM_TRY(check_rows("q", q, q_row, heads * a.c.d, element_bytes(cache->type)));
		if (!out) return set_error(XALM_ERR_INVALID, "paged select: out is NULL");
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
	a.recent = recent;
	a.out = out;
	void (*kernel)(SelectArgs) = cache->type == XALM_F32 ? paged_select_kernel<float> : cache->type == XALM_F16 ? paged_select_kernel<__half> : paged_select_kernel<__nv_bfloat16>;
	XALM_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem));
	kernel<<<dim3((unsigned) a.b.N, (unsigned) a.c.G), ST, smem, (cudaStream_t) stream>>>(a);
	XALM_CUDA_CHECK(cudaGetLastError());
	return XALM_OK;
}

} // extern "C"
