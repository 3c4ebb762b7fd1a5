// paged_tma.cuh — pages through the copy engine, waits that end, and what the tensor-core kernels over paged caches share at the end of a piece.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "paged.cuh"

namespace xalm {
namespace paged {

// A pool as the copy engine sees it: (64 entries, slots, blocks of 64 entries, heads, pages), boxes of min(page, 64) slots of one head with all their blocks, one behind the other.  Heads whose
// last block is not full are (entries, slots, 1, heads, pages) and come block by block: entries behind the last read as zeros, as pages behind the pool's last do.
__host__ __device__ __forceinline__ bool whole_heads(int dim) { return dim % 64 == 0; }
static inline int encode_map(CUtensorMap* map, int type, int n, void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
	typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
	                           CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
	static const Encode encode = [] {
		void* f = nullptr;
		cudaDriverEntryPointQueryResult q;
		if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
			cudaGetLastError();
			return (Encode) nullptr;
		}
		return (Encode) f;
	}();
	if (!encode) return set_error(XALM_ERR_CUDA, "paged attention: this driver has no cuTensorMapEncodeTiled");
	const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
	const CUresult r = encode(map, type == XALM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t) n, base, dims, strides, box, steps,
	                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
	if (r != CUDA_SUCCESS) return set_error(XALM_ERR_CUDA, "paged attention: cuTensorMapEncodeTiled failed (%d)", (int) r);
	return XALM_OK;
}
static inline int pool_map(const Cache& c, int type, bool keys, CUtensorMap* map) {
	const int P = 1 << c.shift, dim = keys ? c.d : c.dv, blocks = P >= KT && whole_heads(dim) ? dim / 64 : 1;
	const cuuint64_t dims[5] = {(cuuint64_t) (dim / blocks), (cuuint64_t) P, (cuuint64_t) blocks, (cuuint64_t) c.G, (cuuint64_t) c.pages};
	const cuuint64_t strides[4] = {(cuuint64_t) (keys ? c.k_slot : c.v_slot) * 2, 128, (cuuint64_t) (keys ? c.k_head : c.v_head) * 2, (cuuint64_t) (keys ? c.k_page : c.v_page) * 2};
	const cuuint32_t box[5] = {64, (cuuint32_t) (P < KT ? P : KT), (cuuint32_t) blocks, 1, 1};
	return encode_map(map, type, 5, keys ? c.k : c.v, dims, strides, box);
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page, uint64_t* bar) {
	asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map), "r"(x), "r"(slot),
	             "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
	             : "memory");
}
// One thread: keys or values of a tile, `per` runs of W slots whose pages are id[0 .. per) (-1: none), into [block][64 slots][128 bytes] at dst
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap* map, int dim, int head, int slot, int per, int W, const int* id, int none, uint64_t* bar) {
	if (per == 1 && whole_heads(dim)) copy_box(dst, map, 0, slot, head, id[0] < 0 ? none : id[0], bar);
	else
		for (int i = 0; i < per; i++)
			for (int x = 0; x < dim; x += 64) copy_box(dst + (x / 64 * KT + i * W) * 128, map, x, slot, head, id[i] < 0 ? none : id[i], bar);
}
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

__device__ __forceinline__ bool elect() { // one thread of a converged warp, in a way that the compiler knows for one
	uint32_t pred;
	asm volatile(
	    "{\n"
	    ".reg .pred p;\n"
	    "elect.sync _|p, 0xffffffff;\n"
	    "selp.u32 %0, 1, 0, p;\n"
	    "}\n"
	    : "=r"(pred));
	return pred != 0;
}
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
	uint32_t ok;
	asm volatile(
	    "{\n"
	    ".reg .pred p;\n"
	    "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
	    "selp.u32 %0, 1, 0, p;\n"
	    "}\n"
	    : "=r"(ok)
	    : "r"(smem_u32(bar)), "r"(parity)
	    : "memory");
	return ok != 0;
}
// The same, without waiting; a whole warp agrees
__device__ __forceinline__ bool try_wait_once(uint64_t* bar, uint32_t parity) {
	uint32_t ok;
	asm volatile(
	    "{\n"
	    ".reg .pred p;\n"
	    "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
	    "selp.u32 %0, 1, 0, p;\n"
	    "}\n"
	    : "=r"(ok)
	    : "r"(smem_u32(bar)), "r"(parity)
	    : "memory");
	return __all_sync(0xffffffffu, ok != 0);
}
// How the warps of a CTA stand with one another, in shared memory
struct State {
	int dead; // a wait has given up: nobody waits any more
	int busy; // warps that go over rows again key by key, which ends by itself but takes as long as it takes: no wait gives up meanwhile
	unsigned since[12]; // of each warp's wait
	__device__ __forceinline__ void init() { dead = busy = 0; }
};
// A wait gives up after two seconds, far beyond what a copy or a product takes.  By the clock: a try may be over at once (2^18 of them in 50 ms) or after microseconds.  The clock is looked at
// every 4096 tries, by a call where the loops around it are short of registers (single tokens 49.3 us in place of 49.9, a group's 64 80.5 in place of 82.3), in the loop itself in the kernel
// of lists (476 us in place of 502), which does no rows again.
constexpr int WAIT_TRIES = 1 << 30, LOOK = 4096;
__device__ __forceinline__ unsigned clock_us() { // nearly
	unsigned long long ns;
	asm volatile("mov.u64 %0, %globaltimer;" : "=l"(ns));
	return (unsigned) (ns >> 10);
}
constexpr unsigned WAIT_US = 2000000;
static __device__ __noinline__ bool waited_long(State* st, int tries) {
	const unsigned now = clock_us();
	volatile unsigned* since = &st->since[threadIdx.x >> 5];
	if (tries < LOOK || *(volatile int*) &st->busy) *since = now;
	return now - *since > WAIT_US;
}
template <bool CALL>
__device__ __forceinline__ bool gives_up(State* st, int tries, unsigned& since) {
	if ((tries & LOOK - 1) != LOOK - 1) return false;
	if constexpr (CALL) return waited_long(st, tries);
	const unsigned now = clock_us();
	if (tries < LOOK) since = now;
	return now - since > WAIT_US;
}
__device__ __forceinline__ bool wait_some(uint64_t* bar, uint32_t parity, State* st) {
	unsigned since = 0;
	for (int i = 0; i < WAIT_TRIES; i++) {
		if (try_wait(bar, parity)) return true;
		if (gives_up<true>(st, i, since)) return false;
	}
	return false;
}
// A wait of a whole warp that ends: when it gives up, or another of the CTA has, the status word says so and nobody waits any more
template <bool CALL = true>
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, State* st, const Cache& c) {
	bool ok = false;
	unsigned since = 0;
	for (int i = 0; i < WAIT_TRIES && !(ok = try_wait(bar, parity)); i++)
		if (*(volatile int*) &st->dead || gives_up<CALL>(st, i, since)) break;
	ok = __all_sync(0xffffffffu, ok);
	if (!ok && !*(volatile int*) &st->dead) {
		*(volatile int*) &st->dead = 1;
		report(c, ERR_WAIT);
	}
	return ok;
}

// The same for one thread
template <bool CALL = true>
__device__ __forceinline__ bool wait_alone(uint64_t* bar, uint32_t parity, State* st, const Cache& c) {
	unsigned since = 0;
	for (int i = 0; i < WAIT_TRIES; i++) {
		if (try_wait(bar, parity)) return true;
		if (*(volatile int*) &st->dead) return false;
		if (gives_up<CALL>(st, i, since)) break;
	}
	*(volatile int*) &st->dead = 1;
	report(c, ERR_WAIT);
	return false;
}

// Four neighbouring sums of one row of a piece, with the row's maximum (log2 units) and sum: to the output, or to the slot that the join reads
template <typename T>
__device__ __forceinline__ void put_row(const Attn& a, const Part& part, const Piece& x, int M, int row, int c, float4 v, float m, float l, bool direct, long long slot) {
	if (direct) {
		const int w = x.t * M + row, h = x.g * a.rep + w % a.rep;
		const long long token = x.row0 + w / a.rep;
		const bool any = l > 0.f || l != l;
		const float inv = any ? 1.f / l : 0.f;
		T t[4] = {from_f<T>(any ? v.x * inv : 0.f), from_f<T>(any ? v.y * inv : 0.f), from_f<T>(any ? v.z * inv : 0.f), from_f<T>(any ? v.w * inv : 0.f)};
		*reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + token * a.out_row + h * a.c.dv + c) = *reinterpret_cast<const uint2*>(t);
		if (a.lse && c == 0) a.lse[token * a.H + h] = any ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
	} else if (slot < part.slots) {
		*reinterpret_cast<float4*>(part.o + (slot * M + row) * a.c.dv + c) = v;
		if (c == 0) part.ml[slot * M + row] = make_float2(m, l);
	}
}

// Two probabilities of fp16, no infinities: where scores are so large that fp32 holds them to half a unit, one may be above what it is meant to be at most
__device__ __forceinline__ uint32_t probs_f16(float lo, float hi) {
	uint32_t r;
	asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}

// Two 16-bit numbers of a word, one of them not finite
template <typename T>
__device__ __forceinline__ bool infinite16(uint32_t w) {
	constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
	return (w & E) == E || (w >> 16 & E) == E;
}
// Of keys [from, to) of a piece's segment the last whose value is not finite in some entry, among those that this one of 128 threads looks at; -1: none
template <typename T>
__device__ __noinline__ int last_infinite(const Attn& a, const Piece& x, int from, int to, int tid) {
	const int chunks = a.c.dv / 8, P = 1 << a.c.shift;
	int last = -1;
#pragma unroll 4
	for (int i = tid; i < (to - from) * chunks; i += 128) {
		const int at = from + i / chunks, key = x.key0 + at, pg = page_of(a.c, a.b, x.s, key >> a.c.shift);
		if (pg < 0) continue;
		const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.c.v) + pg * a.c.v_page + (key & (P - 1)) * a.c.v_slot + x.g * a.c.v_head + i % chunks * 8);
		if (infinite16<T>(u.x) || infinite16<T>(u.y) || infinite16<T>(u.z) || infinite16<T>(u.w)) last = at;
	}
	return last;
}

// One row of a piece by fp32 FMAs, with only the keys that it sees: for rows that a value which is not finite has spoilt.  128 threads, which share
// barrier `bar`; `buf`: 256 floats.
template <typename T>
__device__ __noinline__ void slow_row(const Attn& a, const Part& part, const Piece& x, int M, int row, int lim, float* buf, bool direct, long long slot, int tid, int bar) {
	const int lane = tid & 31, warp = tid >> 5, w = x.t * M + row, P = 1 << a.c.shift;
	const T* q = reinterpret_cast<const T*>(a.q) + (long long) (x.row0 + w / a.rep) * a.q_row + (x.g * a.rep + w % a.rep) * a.c.d;
	const int first = x.j0 * KT, last = min(x.j1 * KT, lim);
	float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
	for (int kb = first; kb < last; kb += 128) {
		float s = -INFINITY;
		if (kb + tid < last) {
			const int key = x.key0 + kb + tid, pg = page_of(a.c, a.b, x.s, key >> a.c.shift);
			s = 0.f;
			if (pg >= 0) {
				const T* kk = reinterpret_cast<const T*>(a.c.k) + pg * a.c.k_page + (key & (P - 1)) * a.c.k_slot + x.g * a.c.k_head;
#pragma unroll 8
				for (int i = 0; i < a.c.d; i += 8) {
					float u[8], w[8];
					load8(q + i, u);
					load8(kk + i, w);
#pragma unroll
					for (int e = 0; e < 8; e++) s = fmaf(u[e], w[e], s);
				}
			}
			s *= a.scale * 1.4426950408889634f;
		}
		float mx = warp_max(s);
		if (__any_sync(0xffffffffu, s != s)) mx = NAN;
		bar_sync(bar, 128);
		if (lane == 0) buf[128 + warp] = mx;
		bar_sync(bar, 128);
		float top = m;
		for (int i = 0; i < 4; i++) top = top != top || buf[128 + i] != buf[128 + i] ? NAN : fmaxf(top, buf[128 + i]);
		const float base = top == -INFINITY ? 0.f : top, f = m == -INFINITY ? 0.f : exp2f(m - base);
		buf[tid] = exp2f(s - base);
		bar_sync(bar, 128);
		m = top;
		l *= f;
		acc[0] *= f;
		acc[1] *= f;
		const int n = min(128, last - kb);
		int next = page_of(a.c, a.b, x.s, (x.key0 + kb) >> a.c.shift);
		for (int i0 = 0; i0 < n; i0 += 16) { // the values of sixteen keys, which lie in one page, on their way at a time, and the number of the next ones' page
			const int pg = next, key = x.key0 + kb + i0;
			if (i0 + 16 < n) next = page_of(a.c, a.b, x.s, (key + 16) >> a.c.shift);
			const T* at = reinterpret_cast<const T*>(a.c.v) + max(pg, 0) * a.c.v_page + (key & (P - 1)) * a.c.v_slot + x.g * a.c.v_head;
			float p[16], v[16][2];
#pragma unroll
			for (int e = 0; e < 16; e++) {
				p[e] = i0 + e < n ? buf[i0 + e] : 0.f;
#pragma unroll
				for (int c = 0; c < 2; c++) v[e][c] = pg >= 0 && i0 + e < n && c * 128 + tid < a.c.dv ? to_f(at[e * a.c.v_slot + c * 128 + tid]) : 0.f;
			}
#pragma unroll
			for (int e = 0; e < 16; e++) {
				l += p[e];
				acc[0] = fmaf(p[e], v[e][0], acc[0]);
				acc[1] = fmaf(p[e], v[e][1], acc[1]);
			}
		}
		bar_sync(bar, 128);
	}
	bar_sync(bar, 128);
	for (int c = 0; c < 2; c++)
		if (c * 128 + tid < a.c.dv) buf[c * 128 + tid] = acc[c];
	bar_sync(bar, 128);
	for (int c = tid * 4; c < a.c.dv; c += 512) put_row<T>(a, part, x, M, row, c, *reinterpret_cast<const float4*>(buf + c), m, l, direct, slot);
	bar_sync(bar, 128);
}

// ROWS rows from r0 on of an own segment's unit of M, some of which did not come out finite: of the keys that not all of the unit's rows see, the last whose value is not finite is looked for, and
// the rows that do not see it are done again.  128 threads; mark: an int in shared memory.  (What can be told from the piece is, in here: more arguments took half a microsecond from short calls.)
// A row takes some 30 us to 128 keys: 96 rows behind 1600 tokens 39 ms.
template <typename T, int M, int ROWS>
__device__ __noinline__ void redo_rows(const Attn& a, const Part& part, const Piece& x, int r0, State* st, int* mark, float* buf, int tid, int bar) {
	const int rows = min(M, x.rows - x.t * M);
	const bool direct = x.j0 == 0 && x.j1 == x.w && x.key0 == 0;
	const long long slot = piece_slot(a, x.u, blockIdx.x, x.j0 == 0);
	auto seen = [&](int r) { return own_keys(x.q, x.key0, a.rep, x.t * M + r); };
	if (tid == 0) {
		*mark = -1;
		atomicAdd(&st->busy, 1);
	}
	bar_sync(bar, 128);
	const int found = last_infinite<T>(a, x, max(seen(0), x.j0 * KT), min(seen(rows - 1), x.j1 * KT), tid);
	if (found >= 0) atomicMax(mark, found);
	bar_sync(bar, 128);
	const int last = *(volatile int*) mark;
	bar_sync(bar, 128);
	for (int r = r0; r < min(rows, r0 + ROWS); r++)
		if (seen(r) <= last) slow_row<T>(a, part, x, M, r, seen(r), buf, direct, slot, tid, bar);
	if (tid == 0) atomicAdd(&st->busy, -1);
}

} // namespace paged
} // namespace xalm
