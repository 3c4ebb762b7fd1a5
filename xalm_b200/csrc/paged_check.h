// paged_check.h — what the entry points of the paged caches check their arguments with, and what they ask of the device.
#pragma once
#include "family.h"
#include "paged.cuh"

namespace xalm {
namespace paged {

inline int element_bytes(int type) { return type == XALM_F32 ? 4 : 2; }
inline bool is_type(int type) { return type == XALM_F32 || type == XALM_F16 || type == XALM_BF16; }
inline bool aligned16(const void* p) { return ((uintptr_t) p & 15) == 0; }
inline bool aligned4(const void* p) { return ((uintptr_t) p & 3) == 0; }


inline int check_batch(const xalm_paged_batch* b, const Cache& c, BatchView& o) {
	if (!b) return set_error(XALM_ERR_INVALID, "paged cache: batch is NULL");
	if (b->rows < 0 || b->seqs < 0 || b->max_pages < 0 || b->groups < 0 || b->table_row < b->max_pages)
		return set_error(XALM_ERR_INVALID, "paged cache: %d rows, %d sequences of %d pages (rows %lld apart), %d groups", b->rows, b->seqs, b->max_pages, b->table_row, b->groups);
	if ((long long) b->seqs + b->groups > MAX_SEGMENTS) return set_error(XALM_ERR_INVALID, "paged cache: %d sequences and %d groups are more than %d", b->seqs, b->groups, MAX_SEGMENTS);
	if ((long long) b->max_pages << c.shift > 1ll << 30) return set_error(XALM_ERR_INVALID, "paged cache: tables of %d pages of %d tokens (at most 2^30 tokens)", b->max_pages, 1 << c.shift);
	if (b->seqs && (!b->starts || !b->lens || (b->max_pages && !b->table))) return set_error(XALM_ERR_INVALID, "paged cache: starts/lens/table is NULL");
	if (b->groups && (!b->group_bounds || !b->group_shared)) return set_error(XALM_ERR_INVALID, "paged cache: group_bounds/group_shared is NULL");
	for (const int* p : {b->starts, b->lens, b->table, b->group_bounds, b->group_shared})
		if (!aligned4(p)) return set_error(XALM_ERR_INVALID, "paged cache: starts, lens, table and groups are at 4-byte boundaries");
	o = BatchView{b->rows, b->seqs, b->max_pages, b->groups, b->starts, b->lens, b->table, b->table_row, b->group_bounds, b->group_shared};
	return XALM_OK;
}
inline int check_rows(const char* what, const void* p, long long row, int least, int bytes) {
	if (!p || !aligned16(p) || row < least || row * bytes % 16)
		return set_error(XALM_ERR_INVALID, "paged cache: rows of %s are at 16-byte boundaries, %d entries or more apart, and not NULL", what, least);
	return XALM_OK;
}

// Whether n rows of so many bytes each meet: rows that lie side by side in wider ones of the same stride do not
inline bool rows_meet(const void* p, long long p_row, long long p_bytes, const void* q, long long q_row, long long q_bytes, int n) {
	const uintptr_t a = (uintptr_t) p, b = (uintptr_t) q;
	if (a >= b + (n - 1) * q_row + q_bytes || b >= a + (n - 1) * p_row + p_bytes) return false;
	if (p_row != q_row) return true;
	const long long off = (long long) (b - a) % p_row, at = off < 0 ? off + p_row : off; // from a row of p to the next of q
	return at < p_bytes || at + q_bytes > p_row;
}

// What a call writes lies apart from what it reads and from what else it writes
struct Span {
	const char* what;
	const void* at;
	long long bytes;
};
inline Span rows_span(const char* what, const void* p, long long row, long long width, int n, int bytes) { return Span{what, p, ((n - 1) * row + width) * bytes}; }
template <int N>
inline int check_apart(const char* call, const Span& out, const Span (&others)[N]) {
	const uintptr_t a = (uintptr_t) out.at;
	for (const Span& x : others) {
		const uintptr_t b = (uintptr_t) x.at;
		if (a && b && out.bytes > 0 && x.bytes > 0 && a < b + x.bytes && b < a + out.bytes) return set_error(XALM_ERR_INVALID, "%s: %s overlaps %s", call, out.what, x.what);
	}
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
inline int sm_count(int device, int* n) {
	static int known[64]; // the same number whoever writes it
	if (device >= 0 && device < 64 && known[device]) { *n = known[device]; return XALM_OK; }
	XALM_CUDA_CHECK(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device));
	if (device >= 0 && device < 64) known[device] = *n;
	return XALM_OK;
}

} // namespace paged
} // namespace xalm
