// SPDX-License-Identifier: Apache-2.0
//
// logprobs.cu - log-probabilities of given tokens, their ranks, the entropy
// and the top alternatives of each row of logits, in one pass over them.
// The reference has no counterpart: its sampler keeps one token and no
// probability (userspace/decode/decode_loop.c:58-185).
//
// With c = log2(e) / T every thread keeps, over its logits l,
//   m = max l,  S = sum 2^((l - m) c),  W = sum 2^((l - m) c) (l - m) c
// and raises m a batch at a time: for d = (m' - m) c the sums become S' = 2^-d S,
// W' = 2^-d (W - d S). Triples of threads, warps and CTAs join by the same
// rule; then lse = m / T + log2 S ln 2 and the entropy is (log2 S - W / S) ln 2.
// The maximum is subtracted before the product: the sums do not depend on the
// logits' size, and m c may pass fp32's range where the logits do not (a row
// masked with the type's lowest value). A log-probability is the distance to the
// maximum, (l - m) / T - log2 S ln 2, for the same reason: z - lse would round at
// the size of z.
//
// Top alternatives, in the same pass. The elements fall into 32 groups by lane,
// and each group's maximum so far is kept; the k-th largest of those, tau, is
// an element that k elements reach, so all of the k largest are >= tau at any
// time. A batch's elements >= tau are collected (some 30 of the first batches'
// 16 thousand for k = 20, fewer as tau rises, a hundred or two in all), and at
// the end those that reach the k-th largest of 32 group maxima among them are
// ordered by counting the better ones. When too many are collected (long runs
// of equal logits, masks of the type's lowest value) the row is read again with
// the last tau, and selected exactly by radix if that is too many as well: by one
// CTA, one after another, and slow (one row of 128,256 fp32 logits with seven
// tokens allowed under a finite mask 475 us, 256 such rows 970 us; 999 bf16 rows of
// 32,003 440 us; masks of -inf take no longer than none).
// (Segment maxima in the pass and a second look at the best segments took 9 us
// of 37 on 256 rows of 128,256: the second look waits behind other rows' loads.)
//
// A row is one thread-block cluster of 1, 2, 4 or 8 CTAs, chosen so that few
// rows still cover the GPU; the CTAs share maxima, sums and candidates through
// distributed shared memory, so no workspace and no atomic on global memory is
// needed and the result does not depend on the order in which CTAs finish.
// Floor: HBM, each logit read once. No unit is full: a scheduler issues in 49 % (256
// fp32 rows of 128,256) or 58 % (999 bf16 rows of 32,003) of its cycles, with 15 to
// 20 instructions an element for ranks and alternatives (without them the same pass
// runs at 5.2 TB/s). Of the 12.7 (10.0) cycles between two instructions of a warp it
// waits 3.8 (2.0) for loads, as a batch is used up before the next is loaded, 2.1
// (2.0) for the instruction before and 2.0 (1.1) at barriers, mostly a row's end.
// Measured, with a target and 20 alternatives (three targets and five): 34 us, 3.9
// TB/s (35 us, 1.8 TB/s).

#include "kllm_device.cuh"
#include "kllm_internal.h"
#include "kllm_topk.cuh"

#include <cfloat>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kllm {
namespace {

constexpr int kCandCap = 1024;        // candidates ordered by counting
constexpr int kMaxCluster = 8;
constexpr int kTgtMax = KLLM_MAX_TARGETS_I;

struct LpSmem {
	float wm[16], ws[16], ww[16];         // per warp
	int wr[16][kTgtMax];
	// rank 0 of the cluster gathers here; each CTA writes its own slot
	float cm[kMaxCluster], cs[kMaxCluster], cw[kMaxCluster];
	int cr[kMaxCluster][kTgtMax];
	uint32_t gkey[32];                    // group maxima of this CTA's part, as ordered keys
	uint32_t all_key[32];                 // rank 0's: of the whole row
	float cand_v[kCandCap];               // rank 0's
	int cand_i[kCandCap];
	int n_cand;                           // rank 0's
	int short_list[kCandCap];             // candidates that reach the last threshold
	int n_short;
	float tl[kTgtMax];                    // the targets' logits (+inf: no such target)
	int ti[kTgtMax];                      // their indices
	float tau_run;                        // the last threshold a warp found, only ever raised
	float tau;
	float top, ln_s;                      // the row's maximum and ln S, 0 in an empty row
	uint32_t hist[256];
	uint32_t prefix;
	int remain, base_eq;
	int done;                             // radix_candidates: nothing more to find
	int wcnt[16];
};

template <int BF16>
struct Elem;
template <>
struct Elem<0> {
	static constexpr int kVec = 4;       // elements per 16 bytes
	static constexpr int kFly = 8;       // vectors of a batch: 32 elements a lane
	using T = float;
	static __device__ __forceinline__ float get(const T *p) { return __ldcg(p); }
	// elements of a batch that are > t, or >= t
	static __device__ __forceinline__ int count(const uint4 (&raw)[kFly], float t, bool equal)
	{
		int n = 0;
		if (equal) {
#pragma unroll
			for (int q = 0; q < kFly; ++q)
				n += (__uint_as_float(raw[q].x) >= t) + (__uint_as_float(raw[q].y) >= t) +
				     (__uint_as_float(raw[q].z) >= t) + (__uint_as_float(raw[q].w) >= t);
		} else {
#pragma unroll
			for (int q = 0; q < kFly; ++q)
				n += (__uint_as_float(raw[q].x) > t) + (__uint_as_float(raw[q].y) > t) +
				     (__uint_as_float(raw[q].z) > t) + (__uint_as_float(raw[q].w) > t);
		}
		return n;
	}
	static __device__ __forceinline__ float vmax(uint4 v)
	{
		return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
			     fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
	}
	static __device__ __forceinline__ void unpack(uint4 v, float (&x)[4])
	{
		x[0] = __uint_as_float(v.x);
		x[1] = __uint_as_float(v.y);
		x[2] = __uint_as_float(v.z);
		x[3] = __uint_as_float(v.w);
	}
};
template <>
struct Elem<1> {
	static constexpr int kVec = 8, kFly = 4;
	using T = uint16_t;
	static __device__ __forceinline__ float get(const T *p)
	{
		return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16);
	}
	// The comparisons of two elements give two bf16 ones or zeros, whose sums
	// (at most 32 each) are exact.
	static __device__ __forceinline__ int count(const uint4 (&raw)[kFly], float t, bool equal)
	{
		const __nv_bfloat162 t2 = __float2bfloat162_rn(t);       // t is a bf16 value
		__nv_bfloat162 n = __float2bfloat162_rn(0.f);
#pragma unroll
		for (int q = 0; q < kFly; ++q) {
			const uint32_t w[4] = {raw[q].x, raw[q].y, raw[q].z, raw[q].w};
#pragma unroll
			for (int i = 0; i < 4; ++i) {
				const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162 *>(&w[i]);
				n = __hadd2(n, equal ? __hge2(v, t2) : __hgt2(v, t2));
			}
		}
		return (int)(__low2float(n) + __high2float(n));
	}
	static __device__ __forceinline__ float vmax(uint4 v)
	{
		auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };
		const __nv_bfloat162 m = __hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w)));
		return fmaxf(__low2float(m), __high2float(m));
	}
	static __device__ __forceinline__ void unpack(uint4 v, float (&x)[8])
	{
		const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			x[2 * i] = __uint_as_float(w[i] << 16);
			x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
		}
	}
};

// Elements u .. u + kVec - 1 of the row in aligned coordinates (element index
// i = u - mis), as 16 raw bytes: one load when all are inside the row, single
// loads of those that are otherwise; the rest read as -inf.
template <int BF16>
__device__ __forceinline__ uint4 load_raw(const typename Elem<BF16>::T *row, int mis, int V, int u)
{
	constexpr int kVec = Elem<BF16>::kVec;
	const int i = u - mis;
	if (i >= 0 && i + kVec <= V)
		return __ldcg(reinterpret_cast<const uint4 *>(row + i));
	uint32_t w[4];
#pragma unroll
	for (int q = 0; q < 4; ++q) {
		if constexpr (BF16) {
			uint32_t h[2];
#pragma unroll
			for (int z = 0; z < 2; ++z) {
				const int j = i + 2 * q + z;
				h[z] = (j >= 0 && j < V)
				    ? (uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(row + j)) : 0xFF80u;
			}
			w[q] = h[0] | (h[1] << 16);
		} else {
			const int j = i + q;
			w[q] = (j >= 0 && j < V) ? __float_as_uint(__ldcg(reinterpret_cast<const float *>(row) + j))
						 : 0xFF800000u;
		}
	}
	return make_uint4(w[0], w[1], w[2], w[3]);
}

// The order of the top list and of ranks: value descending, NaN as -inf.
__device__ __forceinline__ float order_val(float l)
{
	return l != l ? -CUDART_INF_F : l;
}
__device__ __forceinline__ uint32_t order_bits(float l)
{
	return key_of(order_val(l));
}

// Exact selection by one CTA over the whole row: the k-th largest order key by
// four 8-bit radix passes, then the elements above it and the first of its
// equals in index order. Leaves k candidates. Rare: runs of equal logits.
template <int BF16, int TH>
__device__ __noinline__ void radix_candidates(const typename Elem<BF16>::T *row, int V, int k, LpSmem &sm)
{
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	if (tid == 0) {
		sm.prefix = 0u;
		sm.remain = k;
	}
	__syncthreads();
	for (int pass = 0; pass < 4; ++pass) {
		const int shift = 24 - 8 * pass;
		const uint32_t mask = pass ? 0xFFFFFFFFu << (32 - 8 * pass) : 0u;
		for (int i = tid; i < 256; i += TH)
			sm.hist[i] = 0u;
		__syncthreads();
		const uint32_t prefix = sm.prefix;
		for (int base = 0; base < V; base += TH) {
			const int i = base + tid;
			const uint32_t key = i < V ? order_bits(Elem<BF16>::get(row + i)) : 0u;
			const bool hit = i < V && (key & mask) == prefix;
			const unsigned act = __ballot_sync(0xffffffffu, hit);
			if (hit) {
				const uint32_t bin = (key >> shift) & 0xFFu;
				const unsigned peers = __match_any_sync(act, bin);
				if (__ffs(peers) - 1 == lane)
					atomicAdd(&sm.hist[bin], (uint32_t)__popc(peers));
			}
		}
		__syncthreads();
		if (tid == 0) {
			int rem = sm.remain, bin = 255;
			for (; bin > 0 && (int)sm.hist[bin] < rem; --bin)
				rem -= (int)sm.hist[bin];
			sm.prefix = prefix | ((uint32_t)bin << shift);
			sm.remain = rem;
		}
		__syncthreads();
	}
	const uint32_t kth = sm.prefix;
	const int need_eq = sm.remain, n_gt = k - need_eq;
	if (tid == 0) {
		sm.n_cand = 0;
		sm.base_eq = 0;               // equals taken so far
	}
	__syncthreads();
	// in index order, TH elements at a time: equals keep their order
	for (int base = 0; base < V; base += TH) {
		const int i = base + tid;
		const float l = i < V ? Elem<BF16>::get(row + i) : 0.f;
		const uint32_t key = i < V ? order_bits(l) : 0u;
		const bool gt = i < V && key > kth, eq = i < V && key == kth;
		if (gt) {
			const int at = atomicAdd(&sm.n_cand, 1);      // fewer than k of them
			sm.cand_v[at] = order_val(l);
			sm.cand_i[at] = i;
		}
		const unsigned be = __ballot_sync(0xffffffffu, eq);
		if (lane == 0)
			sm.wcnt[warp] = __popc(be);
		__syncthreads();
		int before = sm.base_eq, all = 0;
#pragma unroll
		for (int w = 0; w < (TH / 32); ++w) {
			if (w < warp)
				before += sm.wcnt[w];
			all += sm.wcnt[w];
		}
		const int at = before + __popc(be & ((1u << lane) - 1u));
		if (eq && at < need_eq) {
			sm.cand_v[n_gt + at] = order_val(l);
			sm.cand_i[n_gt + at] = i;
		}
		__syncthreads();
		// One thread decides for all, while no warp can be counting: a warp of the
		// next round would change n_cand under the others' test of it.
		if (tid == 0) {
			sm.base_eq += all;
			sm.done = sm.base_eq >= need_eq && sm.n_cand >= n_gt;
		}
		__syncthreads();
		if (sm.done)
			break;
	}
	if (tid == 0)
		sm.n_cand = k;
	__syncthreads();
}

// The k-th largest of 32 group maxima (every lane gets it).
__device__ __forceinline__ float group_tau(const uint32_t *gkey, int k, int lane)
{
	const uint32_t key = *reinterpret_cast<const volatile uint32_t *>(gkey + lane);
	const float top = warp_sort_desc(key ? value_of(key) : -CUDART_INF_F, lane);
	return __shfl_sync(0xffffffffu, top, k - 1);
}

// Too many candidates: the row once more, by one CTA, with the tau of all its
// elements; radix selection when that leaves too many as well.
template <int BF16, int TH>
__device__ __noinline__ void recollect(const typename Elem<BF16>::T *row, int V, int mis, int k, LpSmem &sm)
{
	constexpr int kVec = Elem<BF16>::kVec;
	__syncthreads();
	const float tau = group_tau(sm.all_key, k, threadIdx.x & 31);
	if (threadIdx.x == 0)
		sm.n_cand = 0;
	__syncthreads();
	for (int u = threadIdx.x * kVec; u < V + mis; u += TH * kVec) {
		float x[kVec];
		Elem<BF16>::unpack(load_raw<BF16>(row, mis, V, u), x);
#pragma unroll
		for (int z = 0; z < kVec; ++z)
			if (x[z] >= tau && x[z] > -CUDART_INF_F) {
				const int at = atomicAdd(&sm.n_cand, 1);
				if (at < kCandCap) {
					sm.cand_v[at] = x[z];
					sm.cand_i[at] = u - mis + z;
				}
			}
	}
	__syncthreads();
	if (sm.n_cand > kCandCap)
		radix_candidates<BF16, TH>(row, V, k, sm);
}

// TH threads.
template <int BF16, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH)
logprobs_kernel(const kllm_logprobs_args a)
{
	constexpr int kVec = Elem<BF16>::kVec, kFly = Elem<BF16>::kFly, kWarps = TH / 32;
	constexpr int kStep = 32 * kVec;              // elements a warp loads at once
	constexpr int kBatch = kFly * kStep;          // elements of a batch of loads
	using T = typename Elem<BF16>::T;
	__shared__ LpSmem sm;
	cg::cluster_group cl = cg::this_cluster();
	const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
	const int r = blockIdx.x / CL;
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int V = a.vocab, k = a.top_n, nt = a.num_targets;
	const T *row = static_cast<const T *>(a.logits) + (long long)r * a.row_stride;
	const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
	const int U = V + mis;
	LpSmem *lead = cl.map_shared_rank(&sm, 0);
	if (tid < 32)
		sm.gkey[tid] = sm.all_key[tid] = 0u;  // below every number's key
	if (tid == 0) {
		sm.n_cand = sm.n_short = 0;
		sm.tau_run = -CUDART_INF_F;
	}
	// every CTA of the cluster runs, its memory set, before another writes to it
	if (CL > 1)
		cl.sync();
	else
		__syncthreads();

	const int stride = CL * kWarps * kBatch, b0 = (rank * kWarps + warp) * kBatch;
	const float temp = a.temperature ? a.temperature[r] : 1.f;
	const float inv_t = temp > 0.f ? fminf(1.f / temp, FLT_MAX) : 1.f;
	const float c = fminf(kLog2e * inv_t, FLT_MAX);

	// ---- one pass: this thread's (m, S, W), ranks, group maxima, candidates ----
	// A batch at a time: one maximum, one look at the reference and one at each
	// target's place for its 32 elements (a vector at a time these took 35
	// instructions an element, and the pass was bound by them). Its loads are in
	// flight together; the 32 warps of an SM hide each other's.
	// What rarely happens is a rolled loop that reads its vector again: unrolled
	// over the batch and the targets it was half of the instructions, and the
	// fetches of its code stalled the rest (999 rows of 32,003 bf16: 41 us, 35 so).
	float m = -CUDART_INF_F, S = 0.f, W = 0.f, tau = -CUDART_INF_F;
	int rank_n = 0;                               // lane j: target j's rank so far
#pragma unroll 1
	for (int it = 0, here = b0; it == 0 || here < U; ++it, here += stride) {
		uint4 raw[kFly];
		if (here >= mis && here + kBatch <= U) {               // the same for the whole warp
			const uint4 *p = reinterpret_cast<const uint4 *>(row + (here - mis)) + lane;
#pragma unroll
			for (int q = 0; q < kFly; ++q)
				raw[q] = __ldcg(p + q * 32);
		} else {
#pragma unroll
			for (int q = 0; q < kFly; ++q)
				raw[q] = load_raw<BF16>(row, mis, V, here + q * kStep + lane * kVec);
		}                                                      // past the end: all -inf
		if (it == 0 && tid < nt) {
			const int t = a.targets[(size_t)r * nt + tid];
			const bool in = t >= 0 && t < V;
			sm.ti[tid] = in ? t : -1;
			sm.tl[tid] = in ? Elem<BF16>::get(row + t) : CUDART_INF_F;
		}
		float bm = -CUDART_INF_F;
#pragma unroll
		for (int q = 0; q < kFly; ++q)
			bm = fmaxf(bm, Elem<BF16>::vmax(raw[q]));
		if (bm > m) {
			if (m > -CUDART_INF_F) {
				const float d = raise_of(m, bm, c), f = ex2_approx(-d);
				W = f * fmaf(-d, S, W);
				S *= f;
			}
			m = bm;
		}
		const float ref = m == -CUDART_INF_F ? 0.f : m;
		// two elements an instruction where the hardware has it
		const uint64_t c2 = pack2(c, c), r2 = pack2(-ref, -ref);
		uint64_t s2 = 0ull, w2 = 0ull;
#pragma unroll
		for (int q = 0; q < kFly; ++q) {
			float x[kVec];
			Elem<BF16>::unpack(raw[q], x);
#pragma unroll
			for (int z = 0; z < kVec; z += 2) {
				float d0, d1;
				unpack2(mul2(add2(pack2(x[z], x[z + 1]), r2), c2), d0, d1);
				const uint64_t e2 = pack2(ex2_approx(d0), ex2_approx(d1));
				s2 = add2(s2, e2);
				w2 = fma2(e2, pack2(fmaxf(d0, -1000.f), fmaxf(d1, -1000.f)), w2);  // 0 x -inf counts 0
			}
		}
		float sa, sb, wa, wb;
		unpack2(s2, sa, sb);
		unpack2(w2, wa, wb);
		S += sa + sb;
		W += wa + wb;
		if (k > 0)
			atomicMax(&sm.gkey[lane], key_of(bm));
		if (it == 0)
			__syncthreads();  // the targets are here, all warps' first batches in the groups
		// A target counts the elements above it, and its equals at lower indices:
		// >= in the batches before the one it lies in, > in those after it, and one
		// by one in that one. A batch below the target counts nothing.
#pragma unroll 1
		for (int j = 0; j < nt; ++j) {
			const float t = sm.tl[j];
			if (!__any_sync(0xffffffffu, bm >= t))
				continue;
			const int rel = sm.ti[j] + mis - here;             // place in the batch
			int n;
			if (rel >= kBatch) {                               // the same for the whole warp
				n = Elem<BF16>::count(raw, t, true);
			} else if (rel < 0) {
				n = Elem<BF16>::count(raw, t, false);
			} else {
				n = 0;
#pragma unroll
				for (int q = 0; q < kFly; ++q) {
					float y[kVec];
					Elem<BF16>::unpack(raw[q], y);
#pragma unroll
					for (int z = 0; z < kVec; ++z)
						n += (int)(y[z] > t) |
						     ((int)(y[z] == t) & (int)(q * kStep + lane * kVec + z < rel));
				}
			}
			n = __reduce_add_sync(0xffffffffu, n);
			if (lane == j)
				rank_n += n;
		}
		if (k > 0) {
			if (it == 0) {
				tau = group_tau(sm.gkey, k, lane);
			} else if ((it & (it + 1)) == 0 && __popc(it) % kWarps == warp) {
				// after 2, 4, 8 .. batches, by one warp for all: an old threshold
				// only collects more
				tau = group_tau(sm.gkey, k, lane);
				if (lane == 0)
					*reinterpret_cast<volatile float *>(&sm.tau_run) = tau;
			} else {
				tau = fmaxf(tau, *reinterpret_cast<volatile float *>(&sm.tau_run));
			}
			const float reach = fmaxf(tau, -FLT_MAX);          // and not -inf
			if (__any_sync(0xffffffffu, bm >= reach)) {
				uint32_t todo = 0;                             // vectors with a candidate
#pragma unroll
				for (int q = 0; q < kFly; ++q)
					todo |= Elem<BF16>::vmax(raw[q]) >= reach ? 1u << q : 0u;
				while (todo) {
					const int u = here + (__ffs(todo) - 1) * kStep + lane * kVec;
					todo &= todo - 1u;
					float y[kVec];
					Elem<BF16>::unpack(load_raw<BF16>(row, mis, V, u), y);
#pragma unroll
					for (int z = 0; z < kVec; ++z)
						if (y[z] >= reach) {
							const int at = atomicAdd(&lead->n_cand, 1);
							if (at < kCandCap) {
								lead->cand_v[at] = y[z];
								lead->cand_i[at] = u + z - mis;
							}
						}
				}
			}
		}
	}

	// ---- join: warp, CTA, cluster ----------------------------------------------------
#pragma unroll
	for (int o = 16; o; o >>= 1) {
		const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
		const float s2 = __shfl_xor_sync(0xffffffffu, S, o);
		const float w2 = __shfl_xor_sync(0xffffffffu, W, o);
		join(m, S, W, m2, s2, w2, c);
	}
	if (lane == 0) {
		sm.wm[warp] = m;
		sm.ws[warp] = S;
		sm.ww[warp] = W;
	}
	if (lane < nt)
		sm.wr[warp][lane] = rank_n;
	__syncthreads();
	if (warp == 0) {
		float M = -CUDART_INF_F, s = 0.f, w = 0.f;
		if (lane < kWarps) {
			M = sm.wm[lane];
			s = sm.ws[lane];
			w = sm.ww[lane];
		}
#pragma unroll
		for (int o = kWarps / 2; o; o >>= 1) {
			const float m2 = __shfl_xor_sync(0xffffffffu, M, o);
			const float s2 = __shfl_xor_sync(0xffffffffu, s, o);
			const float w2 = __shfl_xor_sync(0xffffffffu, w, o);
			join(M, s, w, m2, s2, w2, c);
		}
		if (k > 0)
			atomicMax(&lead->all_key[lane], sm.gkey[lane]);
		if (lane == 0) {
			lead->cm[rank] = M;
			lead->cs[rank] = s;
			lead->cw[rank] = w;
		}
		if (lane < nt) {
			int n = 0;
#pragma unroll
			for (int i = 0; i < kWarps; ++i)
				n += sm.wr[i][lane];
			lead->cr[rank][lane] = n;
		}
	}
	if (CL > 1)
		cl.sync();
	else
		__syncthreads();

	// ---- rank 0: the row's numbers ------------------------------------------------------
	if (rank != 0)
		return;
	if (warp == 0) {
		float M = -CUDART_INF_F, s = 0.f, w = 0.f;
		if (lane < CL) {
			M = sm.cm[lane];
			s = sm.cs[lane];
			w = sm.cw[lane];
		}
#pragma unroll
		for (int o = kMaxCluster / 2; o; o >>= 1) {
			const float m2 = __shfl_xor_sync(0xffffffffu, M, o);
			const float s2 = __shfl_xor_sync(0xffffffffu, s, o);
			const float w2 = __shfl_xor_sync(0xffffffffu, w, o);
			join(M, s, w, m2, s2, w2, c);
		}
		const bool dead = M == -CUDART_INF_F && s == 0.f;
		const float l2 = log2f(s), top = dead ? 0.f : M, ln_s = dead ? 0.f : l2 * kLn2;
		if (lane == 0) {
			sm.top = top;
			sm.ln_s = ln_s;
			if (a.lse)
				a.lse[r] = dead ? -CUDART_INF_F : fmaf(M, inv_t, ln_s);
			if (a.entropy)
				a.entropy[r] = dead ? 0.f : (l2 - w / s) * kLn2;
		}
		if (lane < nt) {
			const bool in = sm.ti[lane] >= 0;
			const float l = in ? sm.tl[lane] : -CUDART_INF_F;
			a.target_lp[(size_t)r * nt + lane] = in ? fmaf(l - top, inv_t, -ln_s) : -CUDART_INF_F;
			if (a.target_rank) {
				int n = 0;
				for (int i = 0; i < CL; ++i)
					n += sm.cr[i][lane];
				if (l == -CUDART_INF_F)
					n -= mis;                   // the padding before the row read as -inf
				a.target_rank[(size_t)r * nt + lane] = in && l == l ? n : -1;
			}
		}
	}
	if (k == 0)
		return;

	// ---- the k largest of the candidates -------------------------------------------------
	if (sm.n_cand > kCandCap)                           // the same for every thread
		recollect<BF16, TH>(row, V, mis, k, sm);
	int n = sm.n_cand;
	if (n < k) {
		// fewer than k elements above -inf: the rest are -inf (or NaN), lowest
		// index first; the first k elements hold enough of them
		__syncthreads();
		if (warp == 1) {
			const bool low = lane < k && order_val(Elem<BF16>::get(row + min(lane, V - 1))) ==
							 -CUDART_INF_F;
			const unsigned b = __ballot_sync(0xffffffffu, low);
			const int at = n + __popc(b & ((1u << lane) - 1u));
			if (low && at < k) {
				sm.cand_v[at] = -CUDART_INF_F;
				sm.cand_i[at] = lane;
			}
		}
		n = k;
	}
	__syncthreads();                                    // and sm.top is set
	if (warp == 0) {
		float top = -CUDART_INF_F;
		for (int i = lane; i < n; i += 32)
			top = fmaxf(top, sm.cand_v[i]);
		top = warp_sort_desc(top, lane);
		if (lane == k - 1)
			sm.tau = top;
	}
	__syncthreads();
	const float last = sm.tau;
	for (int i = tid; i < n; i += TH)
		if (sm.cand_v[i] >= last)
			sm.short_list[atomicAdd(&sm.n_short, 1)] = i;
	__syncthreads();
	const int ns = sm.n_short;
	for (int i = tid; i < ns; i += TH) {
		const int me = sm.short_list[i], id = sm.cand_i[me];
		const float v = sm.cand_v[me];
		int at = 0;
#pragma unroll 4
		for (int j = 0; j < ns; ++j) {
			const int other = sm.short_list[j];
			const float o = sm.cand_v[other];
			at += (int)(o > v) | ((int)(o == v) & (int)(sm.cand_i[other] < id));
		}
		if (at < k) {
			a.top_ids[(size_t)r * k + at] = id;
			a.top_lp[(size_t)r * k + at] = fmaf(v - sm.top, inv_t, -sm.ln_s);
		}
	}
}

template <int BF16, int TH>
cudaError_t launch_lp(const kllm_logprobs_args &a, int cluster, cudaStream_t st)
{
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)a.num_rows * (unsigned)cluster);
	cfg.blockDim = dim3(TH);
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeClusterDimension;
	at[0].val.clusterDim.x = (unsigned)cluster;
	at[0].val.clusterDim.y = 1;
	at[0].val.clusterDim.z = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	return cudaLaunchKernelEx(&cfg, logprobs_kernel<BF16, TH>, a);
}

template <int BF16>
cudaError_t launch_rows(const kllm_logprobs_args &a, int num_sms, cudaStream_t st)
{
	// A row ends in a chain of a microsecond or two that loads nothing. Long rows
	// take 512 threads; short ones 128, so that eight share an SM and one row's
	// end runs under the others' loads.
	const bool wide = a.vocab >= 65536;
	const int th = wide ? 512 : 128, batch = 32 * Elem<BF16>::kVec * Elem<BF16>::kFly;
	// CTAs per row: enough to half fill the SMs, none without half a batch a warp
	int cluster = 1;
	while (cluster < kMaxCluster && (long long)a.num_rows * cluster * th < 512ll * num_sms &&
	       a.vocab / (cluster * 2) >= th / 32 * batch / 2)
		cluster *= 2;
	return wide ? launch_lp<BF16, 512>(a, cluster, st) : launch_lp<BF16, 128>(a, cluster, st);
}

}  // namespace
}  // namespace kllm

using namespace kllm;

extern "C" int kllm_logprobs_launch(const struct kllm_logprobs_args *a, int num_sms, void *stream)
{
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	return (int)(a->bf16 ? launch_rows<1>(*a, num_sms, st) : launch_rows<0>(*a, num_sms, st));
}
