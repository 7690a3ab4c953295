// SPDX-License-Identifier: Apache-2.0
//
// logprobs.cu - log-probabilities of given tokens, their ranks, the entropy
// and the top alternatives of each row of logits, in one pass over them.
// The reference has no counterpart: its sampler keeps one token and no
// probability (userspace/decode/decode_loop.c:58-185).
//
// With y = l x log2(e) / T (l: logit) every thread keeps, over its elements,
//   m = max y,  S = sum 2^(y - m),  W = sum 2^(y - m) (y - m)
// and raises m a batch at a time: for m' = m + d the sums become S' = 2^-d S,
// W' = 2^-d (W - d S). Triples of threads, warps and CTAs join by the same
// rule; then lse = (m + log2 S) ln 2 and the entropy is (log2 S - W / S) ln 2.
//
// Top alternatives. The row is cut into segments; the pass also leaves each
// segment's maximum. The k-th largest of those, tau, is an element, so at
// least k elements are >= tau and all of the k largest are; only segments
// whose maximum reaches tau (about k of up to 1,024) hold any. A second look
// at those segments, which are still in the L2, collects the elements >= tau,
// and each finds its place by counting the better ones. Rows whose candidates
// do not fit (long runs of equal logits) are selected exactly by radix.
//
// A row is one thread-block cluster of 1, 2, 4 or 8 CTAs, chosen so that few
// rows still cover the GPU; the CTAs share maxima, sums and candidates through
// distributed shared memory, so no workspace and no atomic on global memory is
// needed and the result does not depend on the order in which CTAs finish.
// Bound: HBM, each logit read once (the segments looked at twice come from L2).

#include "kllm_device.cuh"
#include "kllm_internal.h"
#include "kllm_topk.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kllm {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kMaxSeg = 1024;         // segments of a row, over the cluster
constexpr int kCandCap = 1024;        // candidates sorted by counting
constexpr int kMaxCluster = 8;
constexpr int kTgtMax = KLLM_MAX_TARGETS_I;

struct LpSmem {
	float wm[kLpWarps], ws[kLpWarps], ww[kLpWarps];
	int wr[kLpWarps][kTgtMax];
	// rank 0 of the cluster gathers here; each CTA writes its own slot
	float cm[kMaxCluster], cs[kMaxCluster], cw[kMaxCluster];
	int cr[kMaxCluster][kTgtMax];
	float segmax[kMaxSeg];                // rank 0's: every segment of the row
	float cand_v[kCandCap];               // rank 0's
	int cand_i[kCandCap];
	int n_cand;                           // rank 0's
	int seg_list[kMaxSeg];                // own segments to look at again
	int n_list;
	float merge[kLpWarps / 2][32];
	float tau;
	float fin[3];                         // lse, floor (lse, or 0 in an empty row), 1 / T
	uint32_t hist[256];
	uint32_t prefix;
	int remain, base_gt;
	int wcnt[2][kLpWarps];
};

template <int BF16>
struct Elem;
template <>
struct Elem<0> {
	static constexpr int kVec = 4;       // elements per 16 bytes
	using T = float;
	static __device__ __forceinline__ float get(const T *p) { return __ldcg(p); }
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
	static constexpr int kVec = 8;
	using T = uint16_t;
	static __device__ __forceinline__ float get(const T *p)
	{
		return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16);
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

// Elements u .. u + kVec - 1 of the row in aligned coordinates: element index
// i = u - mis. One 16-byte load when all are inside the row, single loads of
// those that are otherwise; the rest read as -inf.
template <int BF16>
__device__ __forceinline__ void load_vec(const typename Elem<BF16>::T *row, int mis, int V, int u,
					 float (&x)[Elem<BF16>::kVec])
{
	constexpr int kVec = Elem<BF16>::kVec;
	const int i = u - mis;
	if (i >= 0 && i + kVec <= V) {
		Elem<BF16>::unpack(__ldcg(reinterpret_cast<const uint4 *>(row + i)), x);
	} else {
#pragma unroll
		for (int q = 0; q < kVec; ++q)
			x[q] = (i + q >= 0 && i + q < V) ? Elem<BF16>::get(row + i + q) : -CUDART_INF_F;
	}
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

__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
	for (int o = 16; o; o >>= 1)
		x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
	return x;
}

// Exact selection by one CTA over the whole row: the k-th largest order key by
// four 8-bit radix passes, then the elements above it and the first of its
// equals in index order. Leaves k candidates. Rare: runs of equal logits.
template <int BF16>
__device__ void radix_candidates(const typename Elem<BF16>::T *row, int V, int k, LpSmem &sm)
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
		for (int i = tid; i < 256; i += kLpThreads)
			sm.hist[i] = 0u;
		__syncthreads();
		const uint32_t prefix = sm.prefix;
		for (int base = 0; base < V; base += kLpThreads) {
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
		sm.base_gt = 0;               // equals taken so far
	}
	__syncthreads();
	// in index order, 512 elements at a time: equals keep their order
	for (int base = 0; base < V; base += kLpThreads) {
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
			sm.wcnt[0][warp] = __popc(be);
		__syncthreads();
		int before = sm.base_gt, all = 0;
#pragma unroll
		for (int w = 0; w < kLpWarps; ++w) {
			if (w < warp)
				before += sm.wcnt[0][w];
			all += sm.wcnt[0][w];
		}
		const int at = before + __popc(be & ((1u << lane) - 1u));
		if (eq && at < need_eq) {
			sm.cand_v[n_gt + at] = order_val(l);
			sm.cand_i[n_gt + at] = i;
		}
		__syncthreads();
		if (tid == 0)
			sm.base_gt += all;
		__syncthreads();
		if (sm.base_gt >= need_eq && sm.n_cand >= n_gt)
			break;
	}
	if (tid == 0)
		sm.n_cand = k;
	__syncthreads();
}

// NT: targets counted in the pass (0, 1, or up to kTgtMax).
template <int BF16, int NT>
__global__ void __launch_bounds__(kLpThreads, 2)
logprobs_kernel(const kllm_logprobs_args a, int seg_len)
{
	constexpr int kVec = Elem<BF16>::kVec;
	constexpr int kStep = 32 * kVec;              // elements a warp loads at once
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
	const int n_seg = (U + seg_len - 1) / seg_len;
	LpSmem *lead = cl.map_shared_rank(&sm, 0);

	if (CL > 1)
		cl.sync();                  // every CTA of the cluster runs before its memory is written
	const float temp = a.temperature ? a.temperature[r] : 1.f;
	const float inv_t = temp > 0.f ? 1.f / temp : 1.f;
	const float c = kLog2e * inv_t;

	constexpr int NTA = NT > 0 ? NT : 1;
	float tl[NTA];
	int ti[NTA], cnt[NTA];
	if constexpr (NT > 0) {
#pragma unroll
		for (int j = 0; j < NT; ++j) {
			const int t = j < nt ? a.targets[(size_t)r * nt + j] : -1;
			ti[j] = (t >= 0 && t < V) ? t : -1;
			tl[j] = ti[j] >= 0 ? Elem<BF16>::get(row + ti[j]) : CUDART_INF_F;
			cnt[j] = 0;
		}
	}

	// ---- one pass: this thread's (m, S, W), ranks, segment maxima --------------
	float m = -CUDART_INF_F, S = 0.f, W = 0.f;
	for (int sg = rank * kLpWarps + warp; sg < n_seg; sg += CL * kLpWarps) {
		float smax = -CUDART_INF_F;
		for (int u0 = sg * seg_len; u0 < min((sg + 1) * seg_len, U); u0 += kStep) {
			float x[kVec];
			const int u = u0 + lane * kVec;
			load_vec<BF16>(row, mis, V, u, x);
			float bm = x[0];
#pragma unroll
			for (int q = 1; q < kVec; ++q)
				bm = fmaxf(bm, x[q]);
			smax = fmaxf(smax, bm);
			const float ym = bm * c;
			if (ym > m) {
				if (m > -CUDART_INF_F) {
					const float d = ym - m, f = ex2_approx(-d);
					W = f * fmaf(-d, S, W);
					S *= f;
				}
				m = ym;
			}
			const float ref = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
			for (int q = 0; q < kVec; ++q) {
				const float d = fmaf(x[q], c, -ref);
				const float e = ex2_approx(d);
				S += e;
				W = fmaf(e, fmaxf(d, -1000.f), W);      // 0 x -inf counts 0
				if constexpr (NT > 0) {
#pragma unroll
					for (int j = 0; j < NT; ++j)
						cnt[j] += (x[q] > tl[j] ||
							   (x[q] == tl[j] && u - mis + q < ti[j])) ? 1 : 0;
				}
			}
		}
		if (k > 0) {
			smax = warp_max(smax);
			if (lane == 0)
				lead->segmax[sg] = smax;
		}
	}

	// ---- join: warp, CTA, cluster ----------------------------------------------------
#pragma unroll
	for (int o = 16; o; o >>= 1) {
		const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
		const float s2 = __shfl_xor_sync(0xffffffffu, S, o);
		const float w2 = __shfl_xor_sync(0xffffffffu, W, o);
		join(m, S, W, m2, s2, w2);
		if constexpr (NT > 0) {
#pragma unroll
			for (int j = 0; j < NT; ++j)
				cnt[j] += __shfl_xor_sync(0xffffffffu, cnt[j], o);
		}
	}
	if (lane == 0) {
		sm.wm[warp] = m;
		sm.ws[warp] = S;
		sm.ww[warp] = W;
		if constexpr (NT > 0) {
#pragma unroll
			for (int j = 0; j < NT; ++j)
				sm.wr[warp][j] = cnt[j];
		}
	}
	if (tid == 0)
		sm.n_list = sm.n_cand = 0;
	__syncthreads();
	if (tid == 0) {
		float M = sm.wm[0], s = sm.ws[0], w = sm.ww[0];
#pragma unroll 1
		for (int i = 1; i < kLpWarps; ++i)
			join(M, s, w, sm.wm[i], sm.ws[i], sm.ww[i]);
		lead->cm[rank] = M;
		lead->cs[rank] = s;
		lead->cw[rank] = w;
	}
	if constexpr (NT > 0) {
		if (tid < NT) {
			int n = 0;
#pragma unroll 1
			for (int i = 0; i < kLpWarps; ++i)
				n += sm.wr[i][tid];
			lead->cr[rank][tid] = n;
		}
	}
	cl.sync();

	// ---- rank 0: the row's numbers, and tau -------------------------------------------
	if (rank == 0) {
		if (tid == 0) {
			float M = sm.cm[0], s = sm.cs[0], w = sm.cw[0];
			for (int i = 1; i < CL; ++i)
				join(M, s, w, sm.cm[i], sm.cs[i], sm.cw[i]);
			const float l2 = log2f(s);
			const bool dead = M == -CUDART_INF_F && s == 0.f;
			const float lse = dead ? -CUDART_INF_F : (M + l2) * kLn2;
			sm.fin[0] = lse;
			sm.fin[1] = dead ? 0.f : lse;
			if (a.lse)
				a.lse[r] = lse;
			if (a.entropy)
				a.entropy[r] = dead ? 0.f : (l2 - w / s) * kLn2;
			sm.tau = -CUDART_INF_F;
		}
		__syncthreads();
		if constexpr (NT > 0) {
			if (tid < nt) {
				const int t = a.targets[(size_t)r * nt + tid];
				const bool in = t >= 0 && t < V;
				const float l = in ? Elem<BF16>::get(row + t) : -CUDART_INF_F;
				a.target_lp[(size_t)r * nt + tid] = in ? l * inv_t - sm.fin[1] : -CUDART_INF_F;
				if (a.target_rank) {
					int n = 0;
					for (int i = 0; i < CL; ++i)
						n += sm.cr[i][tid];
					if (l == -CUDART_INF_F)
						n -= mis;       // the padding before the row read as -inf
					a.target_rank[(size_t)r * nt + tid] = in && l == l ? n : -1;
				}
			}
		}
		// the k-th largest segment maximum: each warp sorts its share, then the
		// warps' 32 largest are merged pair by pair
		if (k > 0 && k <= n_seg) {
			float top = -CUDART_INF_F;
			for (int i = tid; i - lane < n_seg; i += kLpThreads) {
				const float x = warp_sort_desc(i < n_seg ? sm.segmax[i] : -CUDART_INF_F, lane);
				top = i == tid ? x : warp_merge_desc(top, x, lane);
			}
			for (int half = kLpWarps / 2; half; half >>= 1) {
				if (warp >= half && warp < 2 * half)
					sm.merge[warp - half][lane] = top;
				__syncthreads();
				if (warp < half)
					top = warp_merge_desc(top, sm.merge[warp][lane], lane);
				__syncthreads();
			}
			if (warp == 0 && lane == k - 1)
				sm.tau = top;
		}
	}
	if (k == 0)
		return;
	cl.sync();

	// ---- candidates: every element >= tau (above -inf when that is all tau says) --------
	const float tau = lead->tau;
	for (int sg = tid; sg < n_seg; sg += kLpThreads) {
		if (sg % (CL * kLpWarps) / kLpWarps != rank)
			continue;
		const float v = lead->segmax[sg];
		if (v >= tau && v > -CUDART_INF_F)
			sm.seg_list[atomicAdd(&sm.n_list, 1)] = sg;
	}
	__syncthreads();
	const int n_list = sm.n_list;
	for (int li = warp; li < n_list; li += kLpWarps) {
		const int sg = sm.seg_list[li];
		for (int u0 = sg * seg_len; u0 < min((sg + 1) * seg_len, U); u0 += kStep) {
			float x[kVec];
			const int u = u0 + lane * kVec;
			load_vec<BF16>(row, mis, V, u, x);
#pragma unroll
			for (int q = 0; q < kVec; ++q)
				if (x[q] >= tau && x[q] > -CUDART_INF_F) {
					const int at = atomicAdd(&lead->n_cand, 1);
					if (at < kCandCap) {
						lead->cand_v[at] = x[q];
						lead->cand_i[at] = u - mis + q;
					}
				}
		}
	}
	cl.sync();
	if (rank != 0)
		return;
	if (sm.n_cand > kCandCap)
		radix_candidates<BF16>(row, V, k, sm);
	int n = sm.n_cand;
	__syncthreads();
	if (n < k) {
		// fewer than k elements above -inf: the rest are -inf (or NaN), lowest
		// index first; the first k elements hold enough of them
		if (warp == 0) {
			const bool low = lane < k && order_val(Elem<BF16>::get(row + min(lane, V - 1))) ==
							 -CUDART_INF_F;
			const unsigned b = __ballot_sync(0xffffffffu, low);
			const int at = n + __popc(b & ((1u << lane) - 1u));
			if (low && at < k) {
				sm.cand_v[at] = -CUDART_INF_F;
				sm.cand_i[at] = lane;
			}
		}
		__syncthreads();
		n = k;
	}
	for (int i = tid; i < n; i += kLpThreads) {
		const float v = sm.cand_v[i];
		const int id = sm.cand_i[i];
		int at = 0;
		for (int j = 0; j < n; ++j) {
			const float o = sm.cand_v[j];
			at += (o > v || (o == v && sm.cand_i[j] < id)) ? 1 : 0;
		}
		if (at < k) {
			a.top_ids[(size_t)r * k + at] = id;
			a.top_lp[(size_t)r * k + at] = v * inv_t - sm.fin[1];
		}
	}
}

template <int BF16, int NT>
cudaError_t launch_lp(const kllm_logprobs_args &a, int cluster, int seg_len, cudaStream_t st)
{
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)a.num_rows * (unsigned)cluster);
	cfg.blockDim = dim3(kLpThreads);
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeClusterDimension;
	at[0].val.clusterDim.x = (unsigned)cluster;
	at[0].val.clusterDim.y = 1;
	at[0].val.clusterDim.z = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	return cudaLaunchKernelEx(&cfg, logprobs_kernel<BF16, NT>, a, seg_len);
}

}  // namespace
}  // namespace kllm

using namespace kllm;

extern "C" int kllm_logprobs_launch(const struct kllm_logprobs_args *a, int num_sms, void *stream)
{
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	// segments of 256 elements, longer ones when the vocabulary has more than 1,024
	int seg_len = 256;
	while ((a->vocab + 7 + seg_len - 1) / seg_len > kMaxSeg)
		seg_len *= 2;
	// CTAs per row: enough for two CTAs on every SM, none with under 4,096 elements
	int cluster = 1;
	while (cluster < kMaxCluster && (long long)a->num_rows * cluster < 2ll * num_sms &&
	       a->vocab / (cluster * 2) >= 4096)
		cluster *= 2;
	const int nt = a->num_targets;
	cudaError_t e;
	if (a->bf16)
		e = nt == 0 ? launch_lp<1, 0>(*a, cluster, seg_len, st)
			    : nt == 1 ? launch_lp<1, 1>(*a, cluster, seg_len, st)
				      : launch_lp<1, kTgtMax>(*a, cluster, seg_len, st);
	else
		e = nt == 0 ? launch_lp<0, 0>(*a, cluster, seg_len, st)
			    : nt == 1 ? launch_lp<0, 1>(*a, cluster, seg_len, st)
				      : launch_lp<0, kTgtMax>(*a, cluster, seg_len, st);
	return (int)e;
}
