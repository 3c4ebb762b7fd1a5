// paged4.cu — the paged cache of 4-bit numbers: entry points (include/xalm_cuda.h, xalm_cuda_paged4_*), appending to pages, reading rows back.
#include "paged4.cuh"

#include <math.h>

#include <algorithm>

#include "paged_check.h"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// append: keys turned by their positions, then blocks of 32 entries: M the entry of the largest magnitude (the positive one where both signs have it), d = fp16(-M / 8), code =
// clamp(rint(x / d) + 8, 0, 15).  What is stored does not depend on how a sum was rounded: a turned key is the fp32 number next to the turn in 64 bits, and x / d as fp32 rounds it is on the
// same side of every n + 1/2 as the quotient itself, because d (n + 1/2) has 16 bits: where x differs from it, then by a unit of x's last place at least, and the quotient by more than half
// a unit of its own.
// Queries are turned in fp32, by blocks of their own: nothing is decided by them, 16-bit rows show none of it, and fp32 rows are off by a unit or two of their last place.  Nine prompts of 300 to 1500 tokens, 32 and 8 heads of 128, take 60 us (173 MB, 2.9 TB/s; keys and queries by the same blocks 87, a division for each
// code 73), 16 rows 3.9.  No unit is full there (issue 55 %, ALU 38 %, DRAM 27 %): 80 registers leave three blocks to an SM, and their loads wait for the lookups in front of them.
// =========================================================================================================================================
struct Append4Args {
	Cache c;
	BatchView b;
	Pool4 pool;
	const uint8_t *k, *v, *q;
	long long k_row, v_row, q_row, q_out_row;
	uint8_t* q_out;
	int H;
	const float* freq;
	int rot;
	float mag;
	int neighbours;
	int paired;           // halves whose chunks of eight pair up: of queries a thread takes both
	int per_head;         // work items of a head of q
	unsigned by_head;     // 2^32 / that, rounded up (0 for one)
};

constexpr int A4T = 256;

template <typename I>
struct Chunk8 { // eight elements as they came
	uint4 u[sizeof(I) == 4 ? 2 : 1];
	__device__ __forceinline__ void load(const I* p) {
#pragma unroll
		for (int i = 0; i < (sizeof(I) == 4 ? 2 : 1); i++) u[i] = reinterpret_cast<const uint4*>(p)[i];
	}
	__device__ __forceinline__ void floats(float (&x)[8]) const {
		const I* t = reinterpret_cast<const I*>(u);
#pragma unroll
		for (int i = 0; i < 8; i++) x[i] = to_f(t[i]);
	}
};

// position of a row (-1: of no sequence, or before its first token) and the page of the pool that has it (-1: none); by a whole warp
__device__ __forceinline__ int2 place_of(const Cache& c, const BatchView& b, int row, bool& in_seq, bool paged = true) { // paged: its page too
	int pos = -1, page = -1;
	in_seq = false;
	if (row < b.N) {
		const int s = seq_of_row(b, row);
		const View view = view_of(c, b);
		int whole;
		const Seq q = seq_of(view, s, whole);
		if (row_in_seq(q, row)) {
			in_seq = true;
			pos = whole - q.n + row - q.a; // what lies behind the table is turned, and written nowhere
			if (paged && pos >= 0 && pos < view.cap) {
				page = page_of(c, b, s, pos >> c.shift);
				if (page < 0 && (threadIdx.x & 31) == 0) report(c, ERR_PAGE);
			}
		}
	}
	return make_int2(pos, page);
}

// Eight entries of a head from c on, turned in T (keys: 64 bits, queries: 32); other: what they are turned with where that is eight neighbours too (PAIRED)
template <typename I, typename T>
__device__ __forceinline__ void turn(const I* head, int c, const Append4Args& a, const T* cs, const T* sn, float (&x)[8], const float (&other)[8]) {
	if (c >= 2 * a.rot) return;
	if (a.paired) {
		const bool second = c >= a.rot;
		const int f = second ? c - a.rot : c;
		struct alignas(16) Two {
			T v[16 / sizeof(T)];
		};
		constexpr int N = 16 / sizeof(T);
#pragma unroll
		for (int e0 = 0; e0 < 8; e0 += N) {
			const Two co = *reinterpret_cast<const Two*>(cs + f + e0), si = *reinterpret_cast<const Two*>(sn + f + e0);
#pragma unroll
			for (int e = 0; e < N; e++) {
				const T y = (T) x[e0 + e] * co.v[e], z = (T) other[e0 + e] * si.v[e];
				x[e0 + e] = (float) (second ? y + z : y - z);
			}
		}
	} else if (a.neighbours) {
#pragma unroll
		for (int e = 0; e < 8; e += 2) {
			const int f = (c + e) >> 1;
			if (f < a.rot) {
				const T y = (T) x[e], z = (T) x[e + 1];
				x[e] = (float) (y * cs[f] - z * sn[f]);
				x[e + 1] = (float) (z * cs[f] + y * sn[f]);
			}
		}
	} else { // halves that end inside a chunk
#pragma unroll
		for (int e = 0; e < 8; e++) {
			const int i = c + e;
			if (i >= 2 * a.rot) continue;
			const int f = i < a.rot ? i : i - a.rot;
			const T y = (T) x[e] * cs[f], z = (T) to_f(head[i < a.rot ? i + a.rot : f]) * sn[f];
			x[e] = (float) (i < a.rot ? y - z : y + z);
		}
	}
}

// What four lanes have of a block, eight entries each: scale and codes (entry i at bit 4 i).  n = rint(x times the rounded 1 / d) is off from x / d by a rounding's worth; x - n d is exact in fp32, and
// where it is less than d / 2 for all, n is the nearest; elsewhere (a border, a scale that is at its end) the quotients themselves are rounded.
__device__ __forceinline__ uint32_t block4(const float (&x)[8], unsigned quad, __half& scale) {
	float hi = x[0], lo = x[0], none = 0.f;
#pragma unroll
	for (int e = 0; e < 8; e++) {
		hi = fmaxf(hi, x[e]);
		lo = fminf(lo, x[e]);
		none = fmaf(x[e], 0.f, none); // a NaN where something is not finite
	}
#pragma unroll
	for (int o = 1; o < 4; o <<= 1) {
		hi = fmaxf(hi, __shfl_xor_sync(quad, hi, o));
		lo = fminf(lo, __shfl_xor_sync(quad, lo, o));
		none += __shfl_xor_sync(quad, none, o);
	}
	scale = __float2half_rn(fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -65504.f), 65504.f));
	const float d = __half2float(scale);
	if (none != 0.f || d == 0.f) { // a block with what is no finite number reads as none
		if (none != 0.f) scale = __ushort_as_half((unsigned short) 0x7fff);
		return 0x88888888u;
	}
	const float inv = 1.f / d, magic = 12582912.f; // 1.5 2^23: sums with it are rounded to whole numbers
	float most = 0.f;
	uint32_t w = 0;
#pragma unroll
	for (int e = 0; e < 8; e++) {
		const float t = fminf(fmaxf(x[e] * inv, -9.f), 9.f) + magic, n = t - magic;
		most = fmaxf(most, fabsf(fmaf(-n, d, x[e])));
		w |= (uint32_t) min(max(__float_as_int(t) - 0x4b400000 + 8, 0), 15) << (4 * e);
	}
	if (!(most < fabsf(d) * 0.5f)) {
		w = 0;
#pragma unroll
		for (int e = 0; e < 8; e++) w |= (uint32_t) (int) fminf(fmaxf(rintf(__fdiv_rn(x[e], d)) + 8.f, 0.f), 15.f) << (4 * e);
	}
	return w;
}

// blockIdx.y: 0 for keys and values, 1 for queries
template <typename I, int R>
__global__ void __launch_bounds__(A4T, R > 1 ? 3 : 1) paged4_append_kernel(const __grid_constant__ Append4Args a) {
	__shared__ __align__(16) double s_cos[R][128], s_sin[R][128]; // of queries floats
	__shared__ int s_pos[R], s_page[R];             // position (-1: of no sequence, or before its first token), page of the pool (-1: none)
	const int row0 = blockIdx.x * R, tid = threadIdx.x, warp = tid >> 5, d = a.c.d, dv = a.c.dv, G = a.c.G, KG = a.pool.kg, VG = a.pool.vg, shift = a.c.shift;
	const bool queries = blockIdx.y == 1;
	if (blockIdx.x == 0 && !queries) check_seqs(a.c, a.b, tid, A4T);
	if (warp < R) {
		bool in_seq;
		const int2 p = place_of(a.c, a.b, row0 + warp, in_seq, !queries);
		if ((tid & 31) == 0) { s_pos[warp] = in_seq ? p.x : -1; s_page[warp] = p.y; }
	}
	__syncthreads();
	float (*q_cos)[128] = reinterpret_cast<float (*)[128]>(s_cos), (*q_sin)[128] = reinterpret_cast<float (*)[128]>(s_sin);
	for (int i = tid; i < R * a.rot; i += A4T) {
		const int r = i / a.rot, f = i - r * a.rot;
		if (s_pos[r] < 0) continue;
		const double pos = (double) s_pos[r], freq = (double) a.freq[f], x = pos * freq, rest = fma(pos, freq, -x); // x + rest is the product itself: it has 54 or 55 bits from position 2^29 on
		const double turns = rint(x * 0.15915494309189535), angle = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, x)) + rest; // 2 pi is the sum of two doubles
		if (queries) {
			float sn, cs;
			sincosf((float) angle, &sn, &cs);
			q_cos[r][f] = cs * a.mag;
			q_sin[r][f] = sn * a.mag;
		} else {
			double sn, cs;
			sincos(angle, &sn, &cs);
			s_cos[r][f] = cs * (double) a.mag;
			s_sin[r][f] = sn * (double) a.mag;
		}
	}
	__syncthreads();
	bool in[R], kept[R];
#pragma unroll
	for (int r = 0; r < R; r++) {
		in[r] = s_pos[r] >= 0;
		kept[r] = in[r] && s_page[r] >= 0; // keys and values
	}
	const int n_q = queries ? a.H * a.per_head : 0, n_k = G * KG * 4, n_v = G * VG * 4, slot_mask = (1 << shift) - 1;
	for (int i = tid; i < n_q; i += A4T) { // queries, in fp32
		const int h = a.per_head == 1 ? i : (int) __umulhi((unsigned) i, a.by_head), u = i - h * a.per_head;
		const bool pair = a.paired && u * 8 < a.rot;
		const int c = !a.paired || pair ? u * 8 : u * 8 + a.rot; // the item's first entry; behind the pairs come the chunks that are not turned
		const I* from = reinterpret_cast<const I*>(a.q) + h * d + c;
		Chunk8<I> x[R], y[R];
#pragma unroll
		for (int r = 0; r < R; r++)
			if (in[r]) {
				x[r].load(from + (row0 + r) * a.q_row);
				if (pair) y[r].load(from + (row0 + r) * a.q_row + a.rot);
			}
#pragma unroll
		for (int r = 0; r < R; r++) {
			if (!in[r]) continue;
			float lo[8], hi[8];
			x[r].floats(lo);
			I* to = reinterpret_cast<I*>(a.q_out) + (row0 + r) * a.q_out_row + h * d + c;
			if (pair) {
				y[r].floats(hi);
				float cs[8], sn[8];
				load8(&q_cos[r][c], cs);
				load8(&q_sin[r][c], sn);
#pragma unroll
				for (int e = 0; e < 8; e++) {
					const float l = lo[e];
					lo[e] = l * cs[e] - hi[e] * sn[e];
					hi[e] = hi[e] * cs[e] + l * sn[e];
				}
				store8(to + a.rot, hi);
			} else if (!a.paired) turn(from - c + (row0 + r) * a.q_row, c, a, q_cos[r], q_sin[r], lo, lo);
			store8(to, lo);
		}
	}
	if (queries) return;
	for (int i = tid; i < n_k + n_v; i += A4T) {
		const bool value = i >= n_k;
		const int j = value ? i - n_k : i, by = value ? VG == 2 ? 3 : VG == 4 ? 4 : 5 : KG == 2 ? 3 : KG == 4 ? 4 : 5; // chunks of eight to a head: 8, 16 or 32
		const int h = j >> by, chunk = j - (h << by), g = chunk >> 2, t = chunk & 3, c = chunk * 8;
		const bool there = c < (value ? dv : d), pair = there && !value && a.paired && c < 2 * a.rot;
		const I* from = value ? reinterpret_cast<const I*>(a.v) + h * dv + c : reinterpret_cast<const I*>(a.k) + h * d + c;
		const long long step = value ? a.v_row : a.k_row;
		Chunk8<I> x[R], y[R];
#pragma unroll
		for (int r = 0; r < R; r++)
			if (kept[r] && there) {
				x[r].load(from + (row0 + r) * step);
				if (pair) y[r].load(from + (row0 + r) * step + (c < a.rot ? a.rot : -a.rot));
			}
#pragma unroll
		for (int r = 0; r < R; r++) {
			if (!kept[r]) continue; // the same for the whole CTA
			float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
			if (there) {
				x[r].floats(z);
				if (!value) {
					float o[8];
					if (pair) y[r].floats(o);
					turn(from - c + (row0 + r) * step, c, a, s_cos[r], s_sin[r], z, o);
				}
			}
			__half scale;
			const uint32_t w = block4(z, 0xfu << (tid & 28), scale);
			const int slot = s_pos[r] & slot_mask;
			uint8_t* run = a.pool.at + s_page[r] * a.pool.page + h * a.pool.head;
			if (value) {
				uint8_t* at = run + values_at(KG, shift) + slot * (VG * 16) + g * 2;
				*reinterpret_cast<uint16_t*>(at + (2 * t) * (VG * 2)) = (uint16_t) w;
				*reinterpret_cast<uint16_t*>(at + (2 * t + 1) * (VG * 2)) = (uint16_t) (w >> 16);
				if (t == 0) *reinterpret_cast<__half*>(run + value_scales_at(KG, VG, shift) + slot * (VG * 2) + g * 2) = scale;
			} else {
				*reinterpret_cast<uint32_t*>(run + slot * (KG * 16) + t * (KG * 4) + g * 4) = w;
				if (t == 0) *reinterpret_cast<__half*>(run + key_scales_at(KG, shift) + slot * (KG * 2) + g * 2) = scale;
			}
		}
	}
}

// =========================================================================================================================================
// read: rows of keys and values as the blocks stand for them, d (c - 8), exact in fp32 and rounded once in 16 bits.  Bound by what it writes: 8475 rows of 8 heads of 128 and 128 in 15.9 us as
// fp32 (79 MB, 5.0 TB/s; 19.6 with eight entries to a thread, whose 32 bytes lie apart from its neighbours'), 12.3 as fp16.
// =========================================================================================================================================
struct Read4Args {
	Cache c;
	BatchView b;
	Pool4 pool;
	uint8_t *k, *v;
	long long k_row, v_row;
};
template <typename T, int R>
__global__ void __launch_bounds__(A4T) paged4_read_kernel(const __grid_constant__ Read4Args a) {
	__shared__ int s_slot[R], s_page[R]; // slot (-1: not to be written), page (-1: none)
	const int row0 = blockIdx.x * R, tid = threadIdx.x, warp = tid >> 5, d = a.c.d, dv = a.c.dv, G = a.c.G, KG = a.pool.kg, VG = a.pool.vg, shift = a.c.shift;
	if (blockIdx.x == 0) check_seqs(a.c, a.b, tid, A4T);
	if (warp < R) {
		bool in_seq;
		const int2 p = place_of(a.c, a.b, row0 + warp, in_seq);
		if ((tid & 31) == 0) { s_slot[warp] = in_seq && p.x >= 0 ? p.x & ((1 << shift) - 1) : -1; s_page[warp] = p.y; }
	}
	__syncthreads();
	constexpr int E = 16 / sizeof(T); // entries of an item: 16 bytes of the result, so that a warp's are side by side
	const int per_k = d / E, per_v = dv / E, n_k = G * per_k, n_all = n_k + G * per_v;
	for (int i = tid; i < n_all; i += A4T) {
		const bool value = i >= n_k;
		const int j = value ? i - n_k : i, per = value ? per_v : per_k, h = j / per, c = (j - h * per) * E, g = c >> 5, B = value ? VG : KG; // entries c ..
		const int code = value ? (c & 31) / 4 * (VG * 2) + g * 2 : (c & 31) / 8 * (KG * 4) + g * 4 + (c & 7) / 2, first = value ? values_at(KG, shift) : 0;
		const uint8_t* head = a.pool.at + h * a.pool.head;
		uint32_t w[R];
		__half scale[R];
#pragma unroll
		for (int r = 0; r < R; r++) {
			w[r] = 0x88888888u;
			scale[r] = __ushort_as_half((unsigned short) 0);
			if (s_slot[r] >= 0 && s_page[r] >= 0) {
				const uint8_t *run = head + s_page[r] * a.pool.page, *at = run + first + s_slot[r] * (B * 16) + code;
				if (E == 4) w[r] = *reinterpret_cast<const uint16_t*>(at);
				else w[r] = value ? *reinterpret_cast<const uint16_t*>(at) | (uint32_t) *reinterpret_cast<const uint16_t*>(at + VG * 2) << 16 : *reinterpret_cast<const uint32_t*>(at);
				scale[r] = *reinterpret_cast<const __half*>(run + (value ? value_scales_at(KG, VG, shift) : key_scales_at(KG, shift)) + s_slot[r] * (B * 2) + g * 2);
			}
		}
#pragma unroll
		for (int r = 0; r < R; r++) {
			if (s_slot[r] < 0) continue;
			const float f = __half2float(scale[r]);
			T x[E];
#pragma unroll
			for (int e = 0; e < E; e++) x[e] = from_f<T>(f * (float) ((int) (w[r] >> (4 * e) & 15) - 8));
			*reinterpret_cast<uint4*>(reinterpret_cast<T*>(value ? a.v : a.k) + (row0 + r) * (value ? a.v_row : a.k_row) + h * (value ? dv : d) + c) = *reinterpret_cast<const uint4*>(x);
		}
	}
}

// ---- checks and launches -----------------------------------------------------------------------------------------------------------------------
static int check_cache4(const xalm_paged4_cache* c, Cache& o, Pool4& p) {
	if (!c) return set_error(XALM_ERR_INVALID, "paged cache: cache is NULL");
	if (c->pages <= 0 || c->kv_heads <= 0 || c->dim <= 0 || c->vdim <= 0 || c->dim > 256 || c->vdim > 256 || c->dim % 8 || c->vdim % 8 || c->kv_heads > 65535)
		return set_error(XALM_ERR_INVALID, "paged cache: %d pages, %d heads of %d and %d entries (multiples of 8, at most 256)", c->pages, c->kv_heads, c->dim, c->vdim);
	int shift = 4;
	while (shift < 8 && (1 << shift) != c->page_size) shift++;
	if ((1 << shift) != c->page_size) return set_error(XALM_ERR_INVALID, "paged cache: pages of %d slots (16, 32, 64, 128 or 256)", c->page_size);
	if (!c->pool || !aligned16(c->pool)) return set_error(XALM_ERR_INVALID, "paged cache: the pool is at a 16-byte boundary, and not NULL");
	if (!aligned4(c->status)) return set_error(XALM_ERR_INVALID, "paged cache: the status word is not at a 4-byte boundary");
	p = Pool4{(uint8_t*) c->pool, c->page, c->head, blocks_of(c->dim), blocks_of(c->vdim)};
	const long long most = 1ll << 40, run = run_bytes(p.kg, p.vg, shift);
	if (c->page <= 0 || c->head <= 0 || c->page >= most || c->head >= most || c->page % 16 || c->head % 16)
		return set_error(XALM_ERR_INVALID, "paged cache: strides of the pool are multiples of 16 bytes, above 0");
	const bool by_head = (c->kv_heads == 1 || c->head >= run) && (c->pages == 1 || c->page >= (c->kv_heads - 1) * c->head + run);
	const bool by_page = (c->pages == 1 || c->page >= run) && (c->kv_heads == 1 || c->head >= (c->pages - 1) * c->page + run);
	if (!by_head && !by_page) return set_error(XALM_ERR_INVALID, "paged cache: pages or heads of the pool overlap (a page has %lld bytes for each)", run);
	o = Cache{p.at, nullptr, nullptr, 0, 0, 0, 0, 0, 0, c->pages, shift, c->kv_heads, c->dim, c->vdim, c->status};
	return XALM_OK;
}
static int check_apart_from_cache4(const char* call, const Span& out, const Cache& c, const Pool4& p, const BatchView& b) {
	return check_apart(call, out, {Span{"the pool", p.at, (c.pages - 1) * p.page + (c.G - 1) * p.head + run_bytes(p.kg, p.vg, c.shift)}, Span{"the status word", c.status, 4},
	                               Span{"starts", b.starts, 4ll * (b.B + 1)}, Span{"lens", b.lens, 4ll * b.B}, rows_span("the table", b.table, b.table_row, b.max_pages, b.B, 4),
	                               Span{"group_bounds", b.bounds, 4ll * (b.n_groups + 1)}, Span{"group_shared", b.shared, 4ll * b.n_groups}});
}

// What a piece costs beside its tiles, in tiles (64 sequences behind 1000 to 8000 tokens: 94 us, with 2 97, with 14 98; 32 of three to six tokens of fp16 111, 114 and 120; five prompts 456, 474 and 486)
constexpr int LEAD4 = 6, LEAD4_TILE = 6;
// Segments of more rows are the kernel's of many.  32 sequences behind 4096 tokens, by the kernel of few rows and by this: of 48 rows to a kv head 190 and 280 us (fp16 226 and 341), of 64 243 and 289 (290 and
// 346), of 80 293 and 342 (353 and 443), of 96 348 and 353 (418 and 451), of 128 452 and 383 (545 and 481)
constexpr int TILE_ROWS = 64;
// rows to a block of the join, a warp to each, and most blocks to an SM (64 tokens behind 8192 in common: 94.6 us, with 2 101, with 4 or 16 the same; 128 in two groups 129.8, 144, 131 and 129.8)
constexpr int JOIN_ROWS4 = 4, JOIN_BLOCKS4 = 8;

static int plan_attn4(int device, const Cache& c, const Pool4& p, const BatchView& b, int type, int heads, Attn& a, size_t* bytes, int (&kinds)[2]) {
	if (heads <= 0 || heads % c.G || heads > 65535) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	if (!is_type(type)) return set_error(XALM_ERR_UNSUPPORTED, "paged attention: queries of type %d (F32, F16 and BF16)", type);
	int sms = 0;
	XALM_TRY(sm_count(device, &sms));
	a = Attn{};
	a.c = c;
	a.b = b;
	a.H = heads;
	a.rep = heads / c.G;
	// One kernel for segments of few rows, by the rows that one has on average, and where some may have more than TILE_ROWS, the one of many rows for those.  32 sequences behind 4096 tokens: of 4 rows to a kv
	// head fp16 56.7 us by units of 4 and 79.8 by units of 16, fp32 58 and 143; of 8 rows fp16 108 and 88, fp32 104 and 147; of 8 rows bf16 60 by units of 8 and 75 by units of 16, of 12 102 and 77.
	const long long rows_all = (long long) b.N * a.rep, each = (rows_all + b.B - 1) / std::max(b.B, 1);
	const int few_kind = type == XALM_F32 ? each <= 4 ? F4 : F16 : type == XALM_F16 ? each <= 4 ? H4 : H16 : each <= 8 ? B8 : B16;
	const Shape4 few = attn4_shape(p, b, few_kind), more = tile4_shape(p);
	const bool many = type != XALM_F32 && more.rows && (b.n_groups || b.N > b.B || a.rep > TILE_ROWS) && rows_all > TILE_ROWS;
	kinds[0] = many ? TILE : few_kind;
	kinds[1] = few_kind;
	a.n_parts = many ? 2 : 1;
	size_t at = 0;
	auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
	for (int i = 0; i < a.n_parts; i++) {
		Part& t = a.part[i];
		const bool big = many && i == 0;
		t.M = big ? more.rows : few.rows;
		t.grid = sms * (big ? more.per_sm : few.per_sm);
		t.lead = big ? LEAD4_TILE : LEAD4;
		t.least_rows = big ? TILE_ROWS + 1 : 1;
		t.most_rows = many && !big ? TILE_ROWS : 0x7fffffff;
		// a segment has at most its rows / M + 1 tiles, and there are no more segments than have room for the part's least rows, of sequences as of groups; in a part for few rows they have no more
		// than those.  (Five prompts of 2000 tokens in all, 32 heads of 128 over 8, in a group: 83 MB for both parts, without the second bound 147.)
		const long long rows = rows_all, most = rows / t.least_rows;
		auto tiles_of = [&](long long n) { return std::min(rows, many && !big ? n * TILE_ROWS : rows) / t.M + std::min(n, most); };
		const long long tiles = tiles_of(b.B) + (b.n_groups ? tiles_of(b.n_groups) : 0);
		if (tiles * c.G + t.grid > 0x7fffffff / t.M) return set_error(XALM_ERR_INVALID, "paged attention: %d rows of %d heads are too many for one call", b.N, heads);
		const long long work = ((long long) b.max_pages << c.shift) / KT + 1;
		if (tiles * c.G > 0x7fffffffll / (work + t.lead)) return set_error(XALM_ERR_INVALID, "paged attention: %d rows of %d heads over up to %lld keys are too many for one call", b.N, heads, work * KT);
		t.slots = !b.n_groups ? 2 * t.grid : (int) (tiles * c.G) + t.grid;
		t.o = (float*) take((size_t) t.slots * t.M * c.dv * 4);
		t.ml = (float2*) take((size_t) t.slots * t.M * 8);
		t.head = (Head*) take((size_t) t.grid * sizeof(Head));
		t.cum_w = (int*) take((size_t) (b.B + b.n_groups + 1) * 4);
		t.cum_u = (int*) take((size_t) (b.B + b.n_groups + 1) * 4);
		t.shs = (int*) take((size_t) b.B * 4);
	}
	a.row_blocks = !b.n_groups ? 0 : (int) std::min(((long long) b.N * heads + JOIN_ROWS4 - 1) / JOIN_ROWS4, (long long) sms * JOIN_BLOCKS4);
	*bytes = at;
	return XALM_OK;
}

} // namespace paged
} // namespace xalm

using namespace xalm;
using namespace xalm::paged;

extern "C" {

int xalm_cuda_paged4_append(const xalm_paged4_cache* cache, const xalm_paged_batch* batch, const void* k, long long k_row, const void* v, long long v_row, const void* q,
                            long long q_row, int heads, int type, void* q_out, long long q_out_row, const float* freq, int rot_half, float rot_mag, int neighbours, void* stream) {
	Append4Args a = {};
	XALM_TRY(check_cache4(cache, a.c, a.pool));
	XALM_TRY(check_batch(batch, a.c, a.b));
	if (!is_type(type)) return set_error(XALM_ERR_UNSUPPORTED, "paged append: rows of type %d (F32, F16 and BF16)", type);
	if (!aligned4(freq)) return set_error(XALM_ERR_INVALID, "paged append: freq is not at a 4-byte boundary");
	if (rot_half < 0 || 2 * rot_half > a.c.d || (rot_half && !freq)) return set_error(XALM_ERR_INVALID, "paged append: rotation of %d pairs in heads of %d", rot_half, a.c.d);
	if (q && (heads <= 0 || heads > 65535)) return set_error(XALM_ERR_INVALID, "paged append: %d query heads", heads);
	const int e = element_bytes(type);
	if (a.b.N) {
		XALM_TRY(check_rows("k", k, k_row, a.c.G * a.c.d, e));
		XALM_TRY(check_rows("v", v, v_row, a.c.G * a.c.dv, e));
		if (q) {
			XALM_TRY(check_rows("q", q, q_row, heads * a.c.d, e));
			XALM_TRY(check_rows("q_out", q_out, q_out_row, heads * a.c.d, e));
		}
	}
	if (a.b.N == 0 || a.b.B == 0) return XALM_OK;
	if (q) {
		const long long width = (long long) heads * a.c.d * e;
		if (rows_meet(q, q_row * e, width, q_out, q_out_row * e, width, a.b.N)) return set_error(XALM_ERR_INVALID, "paged append: q_out overlaps q");
		const Span out = rows_span("q_out", q_out, q_out_row, heads * a.c.d, a.b.N, e);
		XALM_TRY(check_apart_from_cache4("paged append", out, a.c, a.pool, a.b));
		XALM_TRY(check_apart("paged append", out, {Span{"freq", freq, 4ll * rot_half}}));
		if (rows_meet(k, k_row * e, (long long) a.c.G * a.c.d * e, q_out, q_out_row * e, width, a.b.N) || rows_meet(v, v_row * e, (long long) a.c.G * a.c.dv * e, q_out, q_out_row * e, width, a.b.N))
			return set_error(XALM_ERR_INVALID, "paged append: q_out overlaps k or v");
	}
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	a.k = (const uint8_t*) k; a.v = (const uint8_t*) v; a.q = (const uint8_t*) q;
	a.k_row = k_row; a.v_row = v_row; a.q_row = q_row; a.q_out_row = q_out_row;
	a.q_out = (uint8_t*) q_out;
	a.H = heads;
	a.freq = freq; a.rot = rot_half; a.mag = rot_mag; a.neighbours = neighbours;
	a.paired = !neighbours && rot_half % 8 == 0;
	a.per_head = (a.c.d - (a.paired ? rot_half : 0)) / 8;
	a.by_head = (unsigned) ((0x100000000ull + a.per_head - 1) / a.per_head);
	int sms = 0;
	XALM_TRY(sm_count(cache->device, &sms));
	const bool several = a.b.N >= sms * 4; // four rows to a block once that still gives every SM one, as in paged_append
	void (*kernel)(Append4Args) = type == XALM_F32   ? several ? paged4_append_kernel<float, 4> : paged4_append_kernel<float, 1>
	                              : type == XALM_F16 ? several ? paged4_append_kernel<__half, 4> : paged4_append_kernel<__half, 1>
	                                                 : several ? paged4_append_kernel<__nv_bfloat16, 4> : paged4_append_kernel<__nv_bfloat16, 1>;
	kernel<<<dim3((unsigned) (several ? (a.b.N + 3) / 4 : a.b.N), q ? 2 : 1), A4T, 0, (cudaStream_t) stream>>>(a);
	XALM_CUDA_CHECK(cudaGetLastError());
	return XALM_OK;
}

int xalm_cuda_paged4_read(const xalm_paged4_cache* cache, const xalm_paged_batch* batch, int type, void* k, long long k_row, void* v, long long v_row, void* stream) {
	Read4Args a = {};
	XALM_TRY(check_cache4(cache, a.c, a.pool));
	XALM_TRY(check_batch(batch, a.c, a.b));
	if (!is_type(type)) return set_error(XALM_ERR_UNSUPPORTED, "paged read: rows of type %d (F32, F16 and BF16)", type);
	const int e = element_bytes(type);
	if (a.b.N) {
		XALM_TRY(check_rows("k", k, k_row, a.c.G * a.c.d, e));
		XALM_TRY(check_rows("v", v, v_row, a.c.G * a.c.dv, e));
	}
	if (a.b.N == 0 || a.b.B == 0) return XALM_OK;
	if (rows_meet(k, k_row * e, (long long) a.c.G * a.c.d * e, v, v_row * e, (long long) a.c.G * a.c.dv * e, a.b.N)) return set_error(XALM_ERR_INVALID, "paged read: k overlaps v");
	for (const Span& x : {rows_span("k", k, k_row, a.c.G * a.c.d, a.b.N, e), rows_span("v", v, v_row, a.c.G * a.c.dv, a.b.N, e)}) XALM_TRY(check_apart_from_cache4("paged read", x, a.c, a.pool, a.b));
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	a.k = (uint8_t*) k; a.v = (uint8_t*) v;
	a.k_row = k_row; a.v_row = v_row;
	int sms = 0;
	XALM_TRY(sm_count(cache->device, &sms));
	const bool several = a.b.N >= sms * 4;
	void (*kernel)(Read4Args) = type == XALM_F32   ? several ? paged4_read_kernel<float, 4> : paged4_read_kernel<float, 1>
	                            : type == XALM_F16 ? several ? paged4_read_kernel<__half, 4> : paged4_read_kernel<__half, 1>
	                                               : several ? paged4_read_kernel<__nv_bfloat16, 4> : paged4_read_kernel<__nv_bfloat16, 1>;
	kernel<<<several ? (a.b.N + 3) / 4 : a.b.N, A4T, 0, (cudaStream_t) stream>>>(a);
	XALM_CUDA_CHECK(cudaGetLastError());
	return XALM_OK;
}

int xalm_cuda_paged4_status(const xalm_paged4_cache* cache, int* taken, void* stream) {
	Cache c;
	Pool4 p;
	XALM_TRY(check_cache4(cache, c, p));
	if (!taken || !c.status || !aligned4(taken)) return set_error(XALM_ERR_INVALID, "paged status: %s", !taken || !c.status ? "taken or the cache's status word is NULL" : "taken is not at a 4-byte boundary");
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	return launch_status(c.status, taken, (cudaStream_t) stream);
}

int xalm_cuda_paged4_workspace(const xalm_paged4_cache* cache, const xalm_paged_batch* batch, int type, int heads, size_t* bytes) {
	Cache c;
	Pool4 p;
	BatchView b;
	Attn a;
	int kinds[2];
	if (!bytes) return set_error(XALM_ERR_INVALID, "paged attention: bytes is NULL");
	XALM_TRY(check_cache4(cache, c, p));
	XALM_TRY(check_batch(batch, c, b));
	return plan_attn4(cache->device, c, p, b, type, heads, a, bytes, kinds);
}

int xalm_cuda_paged4_attend(const xalm_paged4_cache* cache, const xalm_paged_batch* batch, const void* q, long long q_row, int heads, int type, float scale, void* out,
                            long long out_row, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
	Cache c;
	Pool4 p;
	BatchView b;
	Attn a;
	int kinds[2];
	size_t need = 0;
	XALM_TRY(check_cache4(cache, c, p));
	XALM_TRY(check_batch(batch, c, b));
	if (!is_type(type)) return set_error(XALM_ERR_UNSUPPORTED, "paged attention: queries of type %d (F32, F16 and BF16)", type);
	if (heads <= 0 || heads % c.G || heads > 65535) return set_error(XALM_ERR_INVALID, "paged attention: %d query heads over %d", heads, c.G);
	const int e = element_bytes(type);
	if (b.N) {
		XALM_TRY(check_rows("q", q, q_row, heads * c.d, e));
		XALM_TRY(check_rows("out", out, out_row, heads * c.dv, e));
	}
	if (!aligned4(lse)) return set_error(XALM_ERR_INVALID, "paged attention: lse is not at a 4-byte boundary");
	if (!isfinite(scale)) return set_error(XALM_ERR_INVALID, "paged attention: scale is not finite");
	if (b.N == 0 || b.B == 0) return XALM_OK;
	if (!workspace || ((uintptr_t) workspace & 255)) return set_error(XALM_ERR_INVALID, "paged attention: the workspace is NULL or not at a 256-byte boundary");
	if (rows_meet(q, q_row * e, (long long) heads * c.d * e, out, out_row * e, (long long) heads * c.dv * e, b.N)) return set_error(XALM_ERR_INVALID, "paged attention: out overlaps q");
	const Span sq = rows_span("q", q, q_row, heads * c.d, b.N, e), so = rows_span("out", out, out_row, heads * c.dv, b.N, e), sl = {"lse", lse, 4ll * b.N * heads};
	for (const Span& x : {so, sl}) XALM_TRY(check_apart_from_cache4("paged attention", x, c, p, b));
	XALM_TRY(check_apart("paged attention", sl, {sq, so}));
	XALM_TRY(plan_attn4(cache->device, c, p, b, type, heads, a, &need, kinds));
	const Span sw = {"the workspace", workspace, (long long) need};
	XALM_TRY(check_apart_from_cache4("paged attention", sw, c, p, b));
	XALM_TRY(check_apart("paged attention", sw, {sq, so, sl}));
	if (workspace_bytes < need) return set_error(XALM_ERR_INVALID, "paged attention: a workspace of %zu bytes is needed, %zu given", need, workspace_bytes);
	OnDevice on;
	XALM_TRY(on.set(cache->device));
	uint8_t* base = (uint8_t*) workspace;
	for (int i = 0; i < a.n_parts; i++) {
		Part& t = a.part[i];
		t.o = (float*) (base + (size_t) t.o);
		t.ml = (float2*) (base + (size_t) t.ml);
		t.head = (Head*) (base + (size_t) t.head);
		t.cum_w = (int*) (base + (size_t) t.cum_w);
		t.cum_u = (int*) (base + (size_t) t.cum_u);
		t.shs = (int*) (base + (size_t) t.shs);
	}
	a.q = (const uint8_t*) q;
	a.q_row = q_row;
	a.out = (uint8_t*) out;
	a.out_row = out_row;
	a.lse = lse;
	a.scale = scale;
	cudaStream_t s = (cudaStream_t) stream;
	for (int i = 0; i < a.n_parts; i++) XALM_TRY(kinds[i] == TILE ? launch_attn4_tile(a, p, i, type, s) : launch_attn4(a, p, i, type, kinds[i], s));
	return launch_join(a, type, s);
}

} // extern "C"
