// verify.cu — drafted tokens against the target's probabilities (include/xalm_cuda.h, xalm_cuda_verify_drafts).
#include <cooperative_groups.h>

#include "paged_check.h"

namespace xalm {
namespace paged {

// =========================================================================================================================================
// Sequence s has rows a .. b - 1: row a is the token it had, those behind it its drafts, and row i has the target's distribution p_i of the token behind it.  The draft x behind row i, drawn from
// q_i, is taken where u_i q_i(x) < p_i(x); behind the last one taken a token is drawn from max(p - q, 0) (p where all are taken) by the inverse of its sums: the lowest token up to which they
// pass r times their total.  Tokens drawn so have the target's distribution.
// A cluster of CTAs has a sequence, each a part of the vocabulary, each warp a run of it, so that it is read once: sums in 64 bits (p - q is exact there, and a token's sum is off by less than
// its own probability's last bits), the parts' totals by the cluster's shared memory; then the CTA in whose part the goal lies goes over that warp's run again, which is in L2.
// Bound by latency: four loads that depend on one another before the row is known, then the row.  64 sequences over 131072 tokens, with the drafts' distributions, 20 us (3.3 TB/s), eight
// over 32000 6.3; with 16 warps to a CTA everywhere, so that not all have room at once, and one warp for the second look, 30.
// =========================================================================================================================================
struct VerifyArgs {
	int type, B, N, V;
	const int *starts, *tokens;
	const uint8_t *p, *q;
	long long p_row, q_row;
	const float *accept, *pick;
	int *out, *taken;
};
// four neighbouring weights from place i on, of places k .. k + V - 1 (the row lies k entries behind a boundary of four); WIDE: both rows do
template <typename T, bool WIDE>
__device__ __forceinline__ void weights4(const T* p, const T* q, int i, int k, int V, int without, double (&w)[4]) {
	float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
	if (WIDE && i >= k && i + 4 <= V + k) {
		if constexpr (sizeof(T) == 4) {
			const float4 a = *reinterpret_cast<const float4*>(p + i);
			x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
			if (q) {
				const float4 b = *reinterpret_cast<const float4*>(q + i);
				y[0] = b.x; y[1] = b.y; y[2] = b.z; y[3] = b.w;
			}
		} else {
			const uint2 a = *reinterpret_cast<const uint2*>(p + i);
#pragma unroll
			for (int e = 0; e < 4; e++) x[e] = to_f(reinterpret_cast<const T*>(&a)[e]);
			if (q) {
				const uint2 b = *reinterpret_cast<const uint2*>(q + i);
#pragma unroll
				for (int e = 0; e < 4; e++) y[e] = to_f(reinterpret_cast<const T*>(&b)[e]);
			}
		}
	} else
#pragma unroll
		for (int e = 0; e < 4; e++) {
			const bool there = i + e >= k && i + e < V + k;
			x[e] = there ? to_f(p[i + e]) : 0.f;
			if (q) y[e] = there ? to_f(q[i + e]) : 0.f;
		}
#pragma unroll
	for (int e = 0; e < 4; e++) {
		const float b = y[e] > 0.f ? y[e] : 0.f; // what is negative or no number counts as zero
		w[e] = x[e] > b && i + e != without ? (double) x[e] - (double) b : 0.0;
	}
}
__device__ __forceinline__ double warp_sum64(double x) {
#pragma unroll
	for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
	return x;
}

template <typename T, int VT>
__global__ void __launch_bounds__(VT) verify_kernel(const __grid_constant__ VerifyArgs a) {
	namespace cg = cooperative_groups;
	constexpr int VW = VT / 32;
	cg::cluster_group cluster = cg::this_cluster();
	const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), s = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	__shared__ double s_warp[VW], s_sum, s_run[VW];
	__shared__ int s_taken, s_found;
	const int first = min(max(a.starts[s], 0), a.N), n = min(max(a.starts[s + 1], first), a.N) - first;
	const T *target = reinterpret_cast<const T*>(a.p), *draft = reinterpret_cast<const T*>(a.q);
	if (warp == 0) { // how many drafts are taken: the first that is not
		int at = 0;
		for (; at < n - 1; at += 32) {
			const int i = at + lane;
			bool refused = true;
			if (i < n - 1) {
				const long long row = first + i;
				const int x = a.tokens[row + 1];
				if (x >= 0 && x < a.V) {
					const float q = draft ? to_f(draft[row * a.q_row + x]) : 1.f, p = to_f(target[row * a.p_row + x]); // what is negative or no number counts as zero, as below
					refused = !((double) a.accept[row] * (q > 0.f ? (double) q : 0.0) < (p > 0.f ? (double) p : 0.0));
				}
			}
			const unsigned m = __ballot_sync(0xffffffffu, refused);
			if (m) {
				at += __ffs(m) - 1;
				break;
			}
		}
		if (lane == 0) s_taken = max(min(at, n - 1), 0);
	}
	__syncthreads();
	const int taken = s_taken;
	if (rank == 0) {
		if (tid == 0) a.taken[s] = taken;
		for (int i = tid; i < n; i += VT)
			if (i != taken) a.out[first + i] = i < taken ? a.tokens[first + i + 1] : -1;
	}
	if (n == 0) return; // the whole cluster
	const long long row = first + taken;
	const bool refused = taken < n - 1;
	constexpr unsigned MASK = 4 * sizeof(T) - 1;
	// places: from the boundary of four entries that the row begins at or behind
	const int k = (int) (((uintptr_t) (target + row * a.p_row) & MASK) / sizeof(T)), k_draft = draft ? (int) (((uintptr_t) (draft + row * a.q_row) & MASK) / sizeof(T)) : k;
	const T* p = target + row * a.p_row - k;
	const int places = a.V + k, part = ((places + ranks * VW - 1) / (ranks * VW) + 127) / 128 * 128; // a warp's run
	auto run_of = [&](int w, int& lo, int& hi) {
		const long long from = ((long long) rank * VW + w) * part;
		lo = (int) min(from, (long long) places);
		hi = (int) min(from + part, (long long) places);
	};
	const double r = (double) a.pick[s];
	for (int round = 0; round < 2; round++) { // the second where the draft has all that the target has: from the target's own distribution
		const T* q = refused && draft && !round ? draft + row * a.q_row - k : nullptr;
		const int x_without = refused && !draft && !round ? a.tokens[row + 1] : -1, without = x_without >= 0 && x_without < a.V ? x_without + k : -1;
		const bool wide = !q || k == k_draft;
		int lo, hi;
		run_of(warp, lo, hi);
		double sums[4] = {0.0, 0.0, 0.0, 0.0};
		if (wide)
#pragma unroll 4
			for (int i = lo + lane * 4; i < hi; i += 128) {
				double w[4];
				weights4<T, true>(p, q, i, k, a.V, without, w);
#pragma unroll
				for (int e = 0; e < 4; e++) sums[e] += w[e];
			}
		else
#pragma unroll 2
			for (int i = lo + lane * 4; i < hi; i += 128) {
				double w[4];
				weights4<T, false>(p, q, i, k, a.V, without, w);
#pragma unroll
				for (int e = 0; e < 4; e++) sums[e] += w[e];
			}
		const double sum = warp_sum64((sums[0] + sums[1]) + (sums[2] + sums[3]));
		if (lane == 0) s_warp[warp] = sum;
		__syncthreads();
		if (tid == 0) {
			double x = 0.0;
			for (int w = 0; w < VW; w++) x += s_warp[w];
			s_sum = x;
			s_found = 0x7fffffff;
		}
		cluster.sync();
		double before = 0.0, total = 0.0;
		int last_rank = 0; // that has any weight
		for (int i = 0; i < ranks; i++) {
			const double x = *cluster.map_shared_rank(&s_sum, i);
			if (i == rank) before = total;
			if (x > 0.0) last_rank = i;
			total += x;
		}
		cluster.sync(); // every CTA has read every other's: they may be written again, and their owners may end
		if (!(total > 0.0)) {
			if (round == 0 && refused) continue;
			if (rank == 0 && tid == 0) a.out[row] = -1;
			return;
		}
		const double goal = r < 1.0 ? r > 0.0 ? r * total : 0.0 : INFINITY;
		// the run in which the sums pass the goal: of the CTA where they do, the first warp's
		const bool none = !(total > goal); // r is no number below 1 (a NaN neither), or the total is infinite: the last token that has a weight
		if (none ? s_sum <= 0.0 || rank != last_rank : !(before + s_sum > goal) || before > goal) return;
		int mine = -1, last = -1;
		double base = 0.0, x = 0.0;
		for (int w = 0; w < VW; w++) {
			if (s_warp[w] > 0.0) last = w;
			if (mine < 0) base = x;
			x += s_warp[w];
			if (mine < 0 && before + x > goal) mine = w;
		}
		if (mine < 0) {
			mine = last;
			base = 0.0;
			for (int w = 0; w < last; w++) base += s_warp[w];
		}
		// the CTA goes over it again, four places to a thread
		run_of(mine, lo, hi);
		int some = -1; // the last with a weight
		for (int i0 = lo; i0 < hi; i0 += VT * 4) {
			const int i = i0 + tid * 4;
			double w[4] = {0.0, 0.0, 0.0, 0.0};
			if (i < hi) {
				if (wide) weights4<T, true>(p, q, i, k, a.V, without, w);
				else weights4<T, false>(p, q, i, k, a.V, without, w);
			}
			double run = (w[0] + w[1]) + (w[2] + w[3]), own = run;
#pragma unroll
			for (int o = 1; o < 32; o <<= 1) {
				const double y = __shfl_up_sync(0xffffffffu, run, o);
				if (lane >= o) run += y;
			}
			if (lane == 31) s_run[warp] = run;
			__syncthreads();
			double y = base + (run - own);
			for (int v = 0; v < VW; v++) {
				if (v < warp) y += s_run[v];
				base += s_run[v];
			}
			int hit = 0x7fffffff;
#pragma unroll
			for (int e = 0; e < 4; e++) {
				y += w[e];
				if (w[e] > 0.0) {
					some = i + e;
					if (hit == 0x7fffffff && before + y > goal) hit = i + e;
				}
			}
			if (hit != 0x7fffffff) atomicMin(&s_found, hit);
			__syncthreads();
			if (s_found != 0x7fffffff) break;
		}
		if (s_found == 0x7fffffff) { // rounded otherwise here: the run's last
			__syncthreads();
			if (tid == 0) s_taken = -1;
			__syncthreads();
			atomicMax(&s_taken, some);
			__syncthreads();
			if (tid == 0) a.out[row] = s_taken - k;
		} else if (tid == 0) a.out[row] = s_found - k;
		return;
	}
}

template <typename T>
static int launch_verify(const VerifyArgs& a, int sms, cudaStream_t s) {
	// CTAs to a sequence: one to every 2048 tokens, up to eight (eight sequences over 32000 tokens 6.2 us, with four 7.0, with two 8.2; one over 131072 8.5, 11.1 and 15.8; over 8000 tokens 256 sequences take 11.3 with
	// four and 8.1 with two, 128 over 32000 13.4 with eight and 9.8 with four); and of eight warps, of sixteen where all of them have room at once (one over 131072 8.5, with eight 10.1; 33 over 50021 8.3 and
	// 7.4; 64 over 131072, which have none, 16.3 with eight and 20.5 with sixteen).  Times with all rows in L2.
	int ranks = 1;
	while (ranks < 8 && ranks * 2048 < a.V) ranks *= 2;
	const bool large = a.B * ranks <= 2 * sms;
	void (*kernel)(VerifyArgs) = large ? verify_kernel<T, 512> : verify_kernel<T, 256>;
	const int VT = large ? 512 : 256;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned) (a.B * ranks));
	cfg.blockDim = dim3(VT);
	cfg.stream = s;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeClusterDimension;
	at[0].val.clusterDim.x = (unsigned) ranks;
	at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	XALM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, a));
	return XALM_OK;
}

} // namespace paged
} // namespace xalm

using namespace xalm;
using namespace xalm::paged;

extern "C" int xalm_cuda_verify_drafts(int device, int type, int seqs, int rows, int vocab, const int* starts, const int* tokens, const void* target, long long target_row, const void* draft,
                                       long long draft_row, const float* accept, const float* pick, int* out, int* taken, void* stream) {
	if (!is_type(type)) return set_error(XALM_ERR_UNSUPPORTED, "verify: probabilities of type %d (F32, F16 and BF16)", type);
	if (seqs < 0 || rows < 0 || vocab <= 0 || seqs > 65535 || vocab > 1 << 30) return set_error(XALM_ERR_INVALID, "verify: %d sequences, %d rows of %d tokens (at most 65535 sequences, 2^30 tokens)", seqs, rows, vocab);
	if (target_row < vocab || (draft && draft_row < vocab) || target_row > 1ll << 40 || (draft && draft_row > 1ll << 40))
		return set_error(XALM_ERR_INVALID, "verify: rows of %d probabilities are %lld and %lld apart", vocab, target_row, draft_row);
	if (seqs == 0) return XALM_OK;
	const int e = element_bytes(type);
	if (!starts || !taken || !pick || (rows && (!tokens || !target || !accept || !out))) return set_error(XALM_ERR_INVALID, "verify: starts/tokens/target/accept/pick/out/taken is NULL");
	for (const void* p : {(const void*) starts, (const void*) tokens, (const void*) accept, (const void*) pick, (const void*) out, (const void*) taken})
		if (!aligned4(p)) return set_error(XALM_ERR_INVALID, "verify: arrays of int and float are at 4-byte boundaries");
	if (((uintptr_t) target | (uintptr_t) draft) & (e - 1)) return set_error(XALM_ERR_INVALID, "verify: probabilities are not at a boundary of their size");
	const long long n = rows > 0 ? rows : 0;
	const Span so = {"out", out, 4 * n}, st = {"taken", taken, 4ll * seqs};
	for (const Span& x : {so, st})
		XALM_TRY(check_apart("verify", x, {Span{"starts", starts, 4ll * (seqs + 1)}, Span{"tokens", tokens, 4 * n}, Span{"target", target, n ? ((n - 1) * target_row + vocab) * e : 0},
		                                   Span{"draft", draft, n ? ((n - 1) * draft_row + vocab) * e : 0}, Span{"accept", accept, 4 * n}, Span{"pick", pick, 4ll * seqs}}));
	XALM_TRY(check_apart("verify", so, {st}));
	OnDevice on;
	XALM_TRY(on.set(device));
	const VerifyArgs a = {type, seqs, rows, vocab, starts, tokens, (const uint8_t*) target, (const uint8_t*) draft, target_row, draft_row, accept, pick, out, taken};
	int sms = 0;
	XALM_TRY(sm_count(device, &sms));
	cudaStream_t s = (cudaStream_t) stream;
	return type == XALM_F32 ? launch_verify<float>(a, sms, s) : type == XALM_F16 ? launch_verify<__half>(a, sms, s) : launch_verify<__nv_bfloat16>(a, sms, s);
}
