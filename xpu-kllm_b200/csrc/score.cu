// SPDX-License-Identifier: Apache-2.0
//
// score.cu - log-probabilities, entropy and top alternatives of given tokens
// straight from hidden states and the vocabulary matrix: the logits of a
// prompt (rows x vocabulary, gigabytes) are never stored. The reference has no
// counterpart (its GPU path returns zero logits,
// userspace/compute/infer_gpu.c:212-229).
//
//   l[r][v] = sum_k hidden[r][k] weight[v][k]     bf16 in, fp32 sums, tcgen05
// and per row, over its logits as they leave the tensor core, with c = log2(e) /
// T: m = max l, S = sum 2^((l - m) c), W = sum 2^((l - m) c) (l - m) c, joined as
// in logprobs.cu; lse = m / T + log2 S ln 2, entropy = (log2 S - W / S) ln 2, and a
// log-probability is (l - m) / T - log2 S ln 2.
//
// score_kernel: a CTA owns 128 rows and a contiguous range of the vocabulary
// (in units of 64 columns, so ranges differ by one unit at most), taken as
// tiles of up to 256 columns. One thread holds one row for the whole range, so
// its (m, S, W) and its list of largest logits live across tiles. A list is a
// column of 64 (value, index) pairs in shared memory: a logit above the row's
// threshold is appended; when a list of the warp is nearly full every list is
// cut to little more than top_n by a bisection on the values, which also
// raises the thresholds. A row appends about top_n (1 + ln(columns / top_n))
// logits in all. Ranges of up to 16 row blocks run side by side, so that a
// vocabulary tile is read from HBM once and by its other row blocks from L2.
// Warps: 0 TMA producer, 1 TMEM allocation and MMA issue, 2-5 the rows' sums,
// 6-9 their lists (in one warp the two took 1.5k cycles for 32 columns). Two
// accumulators of 256 TMEM columns let the epilogue of a tile run under the
// next one's products. Waits are bounded in wall time (KLLM_ERR_TIMEOUT).
//
// score_join_kernel: one CTA per row joins the ranges' triples, keeps the list
// entries that reach two thresholds (the largest that any range reports: it
// alone holds top_n logits that reach it; and with top_n ranges or more the
// top_n-th largest of their maxima), orders them, and takes each target's
// logit as a dot product of its own.
//
// Bound: HBM for few rows (24 rows of 4,096 against 128,256: 200 us, 5.3 TB/s of
// the matrix's 1.05 GB, of which 6 us are the last tile's lists and 7 the join),
// shared-memory bandwidth for many (a stage's 48 KB and its reads; 2,048 rows:
// 1.75 ms, 1,230 TFLOP/s, at the power cap). 333 rows of 1,024 against 32,003: 41
// us, 530 TFLOP/s, 2.5 tiles a CTA, so first products and last lists are bare.

#include "kllm_device.cuh"
#include "kllm_internal.h"
#include "kllm_topk.cuh"
#include "kllm_umma.cuh"

#include <cfloat>

namespace kllm {
namespace {

constexpr int kSR = 128;                   // rows per CTA (MMA M)
constexpr int kSU = 64;                    // vocabulary columns per unit
constexpr int kSN = 256;                   // columns per tile (MMA N), 4 units
constexpr int kSK = 64;                    // hidden elements per stage
constexpr int kSStages = 3;
constexpr int kScThreads = 320;
constexpr int kListCap = 64;
constexpr int kListTrig = 48;              // a list above this is cut (16 more may come)
constexpr int kSlack = 4;                  // a cut keeps top_n .. top_n + kSlack entries
constexpr uint64_t kScWaitNs = 200000000ull;

struct ScoreSmem {
	uint8_t a[kSStages][kSR * kSK * 2];
	uint8_t b[kSStages][kSN * kSK * 2];
	// (value, index) of a row's largest logits so far; one more for list_offer
	uint2 list[kListCap + 1][kSR];
	uint64_t full[kSStages], empty[kSStages];
	uint64_t acc_full[2], acc_empty[2], drain;
	uint32_t tmem_base;
	int abort;
};

__device__ bool sc_wait(ScoreSmem &sm, uint64_t *bar, uint32_t parity, uint32_t *err)
{
	if (mbar_try_wait(bar, parity))
		return true;
	const uint64_t t0 = global_ns();
	for (;;) {
		if (mbar_try_wait_sleep(bar, parity, 2000))
			return true;
		if (*reinterpret_cast<volatile int *>(&sm.abort))
			return false;
		if (global_ns() - t0 > kScWaitNs) {
			*reinterpret_cast<volatile int *>(&sm.abort) = 1;
			if (err)
				atomicOr(err, KLLM_ERR_TIMEOUT_BIT);
			return false;
		}
	}
}

// Range of units of split s out of q.
__device__ __forceinline__ int unit_at(int s, int q, int units)
{
	return (int)((long long)s * units / q);
}

// Cuts this thread's list (n keys, in index order) to its largest: k to k +
// kSlack of them, or exactly k when equal keys leave no such cut (the lowest
// indices of the equals stay). tau becomes a value that k kept entries reach,
// so a later logit has to be larger to matter. Called by whole warps; a lane
// with n < k keeps its list. The list is held in registers: counting in shared
// memory, an entry at a time, took 15k cycles a cut.
struct Cut {
	int n;                // entries kept
	float tau;
};

constexpr uint32_t kListStep = kSR * sizeof(uint2);    // from one entry of a row to its next

// Entries by their address in shared memory: the compiler takes the list for
// generic memory and an append for a branch, which was most of the epilogue
// (333 rows of 32,003 took 70 us with it and 53 without).
__device__ __forceinline__ uint2 list_get(uint32_t at)
{
	uint2 x;
	asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(at) : "memory");
	return x;
}
__device__ __forceinline__ void list_put(uint32_t at, float v, uint32_t id)
{
	asm volatile("st.shared.v2.u32 [%0], {%1, %2};" :: "r"(at), "r"(__float_as_uint(v)), "r"(id) : "memory");
}
// Puts (v, id) at `at` and advances it when `stays`. The store is
// unconditional: under a predicate the 32 of a chunk took 300 cycles more.
__device__ __forceinline__ void list_offer(uint32_t &at, float v, uint32_t id, bool stays)
{
	list_put(at, v, id);
	at += stays ? kListStep : 0u;
}

// CAP: entries looked at (n <= CAP). KEEP false: only the threshold.
template <int CAP, bool KEEP>
__device__ __noinline__ Cut cut_list(uint32_t list, int k, int n, float tau)
{
	uint32_t key[CAP];
	uint32_t lo = 0xffffffffu, hi = 0u;
#pragma unroll
	for (int e = 0; e < CAP; ++e) {
		key[e] = key_of(__uint_as_float(list_get(list + e * kListStep).x));
		if (e >= n)
			key[e] = 0u;                       // below every number's key
		else
			lo = min(lo, key[e]);
		hi = max(hi, key[e]);
	}
	// count(>= lo) >= k and count(>= hi) < k throughout: ends early on a count
	// of at most k + kSlack, else with hi = lo + 1, lo the k-th largest key
	const bool work = n >= k;
	hi = hi + 1u;                              // keys of numbers stay below 2^32 - 1
	bool done = !work || (KEEP && n <= k + kSlack);
	bool equals = false;
	while (!__all_sync(0xffffffffu, done)) {
		const uint32_t mid = lo + ((hi - lo) >> 1);
		int c[4] = {0, 0, 0, 0};
#pragma unroll
		for (int e = 0; e < CAP; ++e)
			c[e & 3] += key[e] >= mid ? 1 : 0;
		const int above = (c[0] + c[1]) + (c[2] + c[3]);
		if (!done) {
			if (mid == lo) {
				equals = done = true;
			} else if (above >= k) {
				lo = mid;
				done = above <= k + kSlack;
			} else {
				hi = mid;
			}
		}
	}
	if (work)
		tau = value_of(lo);
	if constexpr (!KEEP)
		return {n, tau};
	// the entries that stay move down; none does before it has been read
	const uint32_t least = work ? lo : 1u;     // a list with n < k stays as it is
	uint32_t at = list;
	int budget = 0;                            // of entries equal to lo
	const bool ties = __any_sync(0xffffffffu, equals);
	if (ties) {
		budget = equals ? k : CAP;
		if (equals)
#pragma unroll
			for (int e = 0; e < CAP; ++e)
				budget -= key[e] > lo ? 1 : 0;
	}
#pragma unroll
	for (int e0 = 0; e0 < CAP; e0 += 16) {
		uint2 x[16];
#pragma unroll
		for (int e = 0; e < 16; ++e)
			x[e] = list_get(list + (e0 + e) * kListStep);
		if (ties)
#pragma unroll
			for (int e = 0; e < 16; ++e)
				if (key[e0 + e] == least && work && --budget < 0)
					key[e0 + e] = 0u;
#pragma unroll
		for (int e = 0; e < 16; ++e)
			list_offer(at, __uint_as_float(x[e].x), x[e].y, key[e0 + e] >= least);
	}
	return {(int)((at - list) / kListStep), tau};
}

__global__ void __launch_bounds__(kScThreads, 1)
score_kernel(const kllm_score_args a, const __grid_constant__ CUtensorMap tm_h,
	     const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w1)
{
	extern __shared__ __align__(1024) uint8_t smem_raw[];
	ScoreSmem &sm = *reinterpret_cast<ScoreSmem *>(
	    (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const int KT = a.hidden_dim / kSK;
	const int per_group = a.group_rb * a.splits;
	const int n_items = (a.row_blocks + a.group_rb - 1) / a.group_rb * per_group;

	grid_launch_dependents();
	if (tid == 0) {
		for (int s = 0; s < kSStages; ++s) {
			mbar_init(&sm.full[s], 1);
			mbar_init(&sm.empty[s], 1);
		}
		for (int b = 0; b < 2; ++b) {
			mbar_init(&sm.acc_full[b], 1);
			mbar_init(&sm.acc_empty[b], a.top_n > 0 ? 256 : 128);
		}
		mbar_init(&sm.drain, 1);
		sm.abort = 0;
		fence_mbar_init();
	}
	if (warp == 1) {
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
			     :: "r"(smem_u32(&sm.tmem_base)), "r"(512u));
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = sm.tmem_base;

	// item -> row block and unit range; false for the gaps of a last group
	auto item_range = [&](int item, int &rb, int &split, int &u0, int &u1) {
		const int g = item / per_group, rem = item - g * per_group;
		split = rem / a.group_rb;
		rb = g * a.group_rb + rem % a.group_rb;
		u0 = unit_at(split, a.splits, a.units);
		u1 = unit_at(split + 1, a.splits, a.units);
		return rb < a.row_blocks;
	};

	if (warp == 0) {
		// ================= TMA producer ==============================================
		if (elect_one()) {
			// stage st is filled for the (round + 1)-th time; armed: fills of
			// each stage whose copies were issued, for the drain
			int st = 0, armed[kSStages];
			uint32_t round = 0;
#pragma unroll
			for (int s = 0; s < kSStages; ++s)
				armed[s] = 0;
			bool ok = true;
			for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
				int rb, split, u0, u1;
				if (!item_range(item, rb, split, u0, u1))
					continue;
				for (int u = u0; u < u1 && ok; u += 4) {
					const int nu = min(4, u1 - u);
					for (int kt = 0; kt < KT; ++kt) {
						if (round > 0 &&
						    !sc_wait(sm, &sm.empty[st], (round - 1) & 1, a.err)) {
							ok = false;
							break;
						}
#pragma unroll
						for (int s = 0; s < kSStages; ++s)
							armed[s] += s == st ? 1 : 0;
						mbar_arrive_expect_tx(&sm.full[st],
								      kSR * kSK * 2 + nu * kSU * kSK * 2);
						tma_load_2d(sm.a[st], &tm_h, kt * kSK, rb * kSR, &sm.full[st]);
						if (nu == 4)
							tma_load_2d(sm.b[st], &tm_w, kt * kSK, u * kSU, &sm.full[st]);
						else
							for (int i = 0; i < nu; ++i)
								tma_load_2d(sm.b[st] + i * kSU * kSK * 2, &tm_w1, kt * kSK,
									    (u + i) * kSU, &sm.full[st]);
						if (++st == kSStages) {
							st = 0;
							++round;
						}
					}
				}
			}
			// after an abort, wait (bounded) for this CTA's own tensor copies
			if (*reinterpret_cast<volatile int *>(&sm.abort))
#pragma unroll
				for (int s = 0; s < kSStages; ++s)
					if (armed[s] > 0)
						mbar_wait_ns(&sm.full[s], (uint32_t)((armed[s] - 1) & 1), kScWaitNs);
		}
		__syncwarp();
	} else if (warp == 1) {
		// ================= MMA issue ===================================================
		const bool leader = elect_one();
		int st = 0, it = 0;
		uint32_t ph = 0;
		bool ok = true;
		for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
			int rb, split, u0, u1;
			if (!item_range(item, rb, split, u0, u1))
				continue;
			for (int u = u0; u < u1 && ok; u += 4, ++it) {
				const int buf = it & 1;
				const uint32_t idesc = umma_idesc_bf16(kSR, min(4, u1 - u) * kSU, false);
				if (it >= 2)
					ok = __all_sync(0xffffffffu, sc_wait(sm, &sm.acc_empty[buf],
									     (uint32_t)(((it >> 1) - 1) & 1), a.err));
				tc_fence_after();
				for (int kt = 0; kt < KT && ok; ++kt) {
					ok = __all_sync(0xffffffffu, sc_wait(sm, &sm.full[st], ph, a.err));
					if (!ok)
						break;
					tc_fence_after();
					const uint64_t da = umma_desc(smem_u32(sm.a[st]), 16u, 1024u);
					const uint64_t db = umma_desc(smem_u32(sm.b[st]), 16u, 1024u);
#pragma unroll
					for (int kk = 0; kk < kSK / 16; ++kk) {
						const uint64_t off = (uint64_t)(kk * 32) >> 4;
						if (leader)
							umma_f16(tmem + (uint32_t)(buf * kSN), da + off, db + off, idesc,
								 (kt > 0 || kk > 0) ? 1u : 0u);
					}
					__syncwarp();
					if (leader)
						umma_commit(&sm.empty[st]);
					__syncwarp();
					if (++st == kSStages) {
						st = 0;
						ph ^= 1u;
					}
				}
				if (ok && leader)
					umma_commit(&sm.acc_full[buf]);
				__syncwarp();
			}
		}
		// every MMA issued by the leader completes before TMEM is freed
		if (leader)
			umma_commit(&sm.drain);
		__syncwarp();
		mbar_wait_ns(&sm.drain, 0u, kScWaitNs);
	} else {
		// ================= epilogue: one row a thread ==================================
		// Warps 2-5 keep the row's sums, warps 6-9 its list.
		const int q = warp & 3, t = q * 32 + lane;
		const int k = a.top_n, V = a.vocab;
		const bool lists = warp >= 6;
		const uint32_t list = smem_u32(&sm.list[0][t]);
		int it = 0;
		bool ok = !lists || k > 0;
		for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
			int rb, split, u0, u1;
			if (!item_range(item, rb, split, u0, u1))
				continue;
			const int row = rb * kSR + t;            // past the last: a row of zeros
			const float T = (row < a.num_rows && a.temperature) ? a.temperature[row] : 1.f;
			const float c = fminf(kLog2e * (T > 0.f ? 1.f / T : 1.f), FLT_MAX);
			float m = -CUDART_INF_F, S = 0.f, W = 0.f, tau = -CUDART_INF_F;
			uint32_t at = list;                // where the next entry goes
			for (int u = u0; u < u1; u += 4, ++it) {
				const int buf = it & 1, nc = min(4, u1 - u) * (kSU / 32);
				if (!__all_sync(0xffffffffu, sc_wait(sm, &sm.acc_full[buf],
								     (uint32_t)((it >> 1) & 1), a.err))) {
					ok = false;
					break;
				}
				tc_fence_after();
				const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kSN);
				// 32 columns of the row; those past the vocabulary read as -inf
				auto columns = [&](int ch, float (&v)[32]) {
					tmem_ld32(acc + (uint32_t)(ch * 32), v);
					const int nb = u * kSU + ch * 32;
					if (nb + 32 > V) {
#pragma unroll
						for (int i = 0; i < 32; ++i)
							if (nb + i >= V)
								v[i] = -CUDART_INF_F;
					}
				};
				if (lists && u == u0 && 4 * nc >= k) {
					// A range's first threshold: the k-th largest of its first tile's
					// maxima over 8 columns (the list holds them meanwhile). From -inf
					// the first tile alone would need several cuts.
#pragma unroll 1
					for (int ch = 0; ch < nc; ++ch) {
						float v[32];
						columns(ch, v);
#pragma unroll
						for (int g = 0; g < 4; ++g) {
							float gm = v[8 * g];
#pragma unroll
							for (int i = 1; i < 8; ++i)
								gm = fmaxf(gm, v[8 * g + i]);
							list_put(list + (4 * ch + g) * kListStep,
								 gm == gm ? gm : -CUDART_INF_F, 0u);
						}
					}
					tau = cut_list<kSN / 8, false>(list, k, 4 * nc, tau).tau;
					if (tau > -CUDART_INF_F)                 // its equals are wanted
						tau = value_below(tau);
				}
#pragma unroll 1
				for (int ch = 0; ch < nc; ++ch) {
					float v[32];
					const int nb = u * kSU + ch * 32;
					if (nb >= V)
						break;                 // nothing but padding
					columns(ch, v);
					if (lists) {
#pragma unroll
						for (int half = 0; half < 2; ++half) {
#pragma unroll
							for (int i = 16 * half; i < 16 * half + 16; ++i)
								list_offer(at, v[i], (uint32_t)(nb + i), v[i] > tau);
							const int n = (int)((at - list) / kListStep);
							if (__any_sync(0xffffffffu, n > kListTrig)) {
								const Cut cut = cut_list<kListCap, true>(list, k, n, tau);
								at = list + cut.n * kListStep;
								tau = cut.tau;
							}
						}
						continue;
					}
					float c4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
					for (int i = 4; i < 32; ++i)
						c4[i & 3] = fmaxf(c4[i & 3], v[i]);
					const float bm = fmaxf(fmaxf(c4[0], c4[1]), fmaxf(c4[2], c4[3]));
					if (bm > m) {
						if (m > -CUDART_INF_F) {
							const float d = raise_of(m, bm, c), f = ex2_approx(-d);
							W = f * fmaf(-d, S, W);
							S *= f;
						}
						m = bm;
					}
					// sums of 32, then of the chunks: a range has thousands of
					// terms, and one running fp32 sum over them lost 2e-6
					const float ref = m == -CUDART_INF_F ? 0.f : m;
					// two columns an instruction where the hardware has it
					const uint64_t c2 = pack2(c, c), r2 = pack2(-ref, -ref);
					uint64_t s2[2] = {0ull, 0ull}, w2[2] = {0ull, 0ull};
#pragma unroll
					for (int i = 0; i < 32; i += 2) {
						float d0, d1;
						unpack2(mul2(add2(pack2(v[i], v[i + 1]), r2), c2), d0, d1);
						const uint64_t e2 = pack2(ex2_approx(d0), ex2_approx(d1));
						const int z = (i >> 1) & 1;
						s2[z] = add2(s2[z], e2);
						w2[z] = fma2(e2, pack2(fmaxf(d0, -1000.f), fmaxf(d1, -1000.f)), w2[z]);
					}
					float s0, s1, w0, w1;
					unpack2(add2(s2[0], s2[1]), s0, s1);
					unpack2(add2(w2[0], w2[1]), w0, w1);
					S += s0 + s1;
					W += w0 + w1;
				}
				tc_fence_before();
				mbar_arrive(&sm.acc_empty[buf]);
			}
			if (!ok)
				break;
			const size_t to = (size_t)split * a.row_blocks * kSR + (size_t)rb * kSR + t;
			float *part = static_cast<float *>(a.part) + 4 * to;
			if (lists) {
				const Cut cut = cut_list<kListCap, true>(list, k, (int)((at - list) / kListStep), tau);
				const size_t stride = (size_t)a.splits * a.row_blocks * kSR;
				part[3] = cut.tau;
				a.part_n[to] = cut.n;
				for (int e = 0; e < cut.n; ++e)
					static_cast<uint2 *>(a.part_list)[(size_t)e * stride + to] =
					    list_get(list + e * kListStep);
			} else {
				*reinterpret_cast<float2 *>(part) = make_float2(m, S);
				part[2] = W;
			}
		}
	}

	tc_fence_before();
	__syncthreads();
	if (warp == 1) {
		__syncwarp();
		tc_fence_after();
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
			     :: "r"(tmem), "r"(512u));
	}
}

// ---- joining the ranges ---------------------------------------------------------

constexpr int kJoinThreads = 128;
// The join's candidates of a row: its shared memory grows with the ranges and
// stays within what a launch may have without an attribute, which is the
// function's for all callers of a device and so cannot follow one call's size.
constexpr int kMaxSplits = 160;
constexpr size_t join_smem(int splits, int top_n)
{
	return (size_t)splits * ((size_t)(top_n + kSlack) * 8 + 4);
}
static_assert(join_smem(kMaxSplits, KLLM_MAX_TOP_N_I) + 1024 <= 48 * 1024, "join's shared memory");

__device__ __forceinline__ float dot8(uint4 x, uint4 y, float acc)
{
	const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		acc = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), acc);
		acc = fmaf(__uint_as_float(a[i] & 0xFFFF0000u), __uint_as_float(b[i] & 0xFFFF0000u), acc);
	}
	return acc;
}

__global__ void __launch_bounds__(kJoinThreads)
score_join_kernel(const kllm_score_args a)
{
	extern __shared__ __align__(8) uint8_t join_raw[];
	const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int k = a.top_n, nt = a.num_targets, K8 = a.hidden_dim / 8, per = k + kSlack;
	float *cv = reinterpret_cast<float *>(join_raw);               // [splits * per]
	int *ci = reinterpret_cast<int *>(cv + (size_t)a.splits * per);
	int *ranges = ci + (size_t)a.splits * per;                     // [splits]
	__shared__ float red[4][4];
	__shared__ float dots[KLLM_MAX_TARGETS_I][4];
	__shared__ int n_cand, n_ranges;
	__shared__ float max_tau;
	const size_t rows = (size_t)a.row_blocks * kSR, stride = (size_t)a.splits * rows;
	const float4 *part = static_cast<const float4 *>(a.part) + r;
	const float T = a.temperature ? a.temperature[r] : 1.f;
	const float inv_t = T > 0.f ? fminf(1.f / T, FLT_MAX) : 1.f, c = fminf(kLog2e * inv_t, FLT_MAX);
	if (tid == 0)
		n_cand = n_ranges = 0;

	// the targets' logits
	const uint4 *h = reinterpret_cast<const uint4 *>(a.hidden) + (size_t)r * K8;
	for (int j = 0; j < nt; ++j) {
		const int t = a.targets[(size_t)r * nt + j];
		float acc = 0.f;
		if (t >= 0 && t < a.vocab) {
			const uint4 *w = reinterpret_cast<const uint4 *>(a.weight) + (size_t)t * K8;
#pragma unroll 4
			for (int i = tid; i < K8; i += kJoinThreads)
				acc = dot8(__ldg(h + i), __ldg(w + i), acc);
		}
#pragma unroll
		for (int o = 16; o; o >>= 1)
			acc += __shfl_xor_sync(0xffffffffu, acc, o);
		if (lane == 0)
			dots[j][warp] = acc;
	}
	grid_dependency_wait();                // the ranges' results
	// With at least top_n ranges, the top_n-th largest of the ranges' maxima is
	// a threshold that top_n logits reach; warp 0 finds it
	if (warp == 0 && k > 0) {
		float top = -CUDART_INF_F;
		for (int s = lane; s - lane < a.splits; s += 32) {
			const float d = warp_sort_desc(s < a.splits ? part[(size_t)s * rows].x : -CUDART_INF_F, lane);
			top = s == lane ? d : warp_merge_desc(top, d, lane);
		}
		const float kth = __shfl_sync(0xffffffffu, top, k - 1);
		if (lane == 0)
			max_tau = a.splits >= k ? kth : -CUDART_INF_F;
	}
	// the ranges' triples and the largest threshold any of them reports
	float m = -CUDART_INF_F, S = 0.f, W = 0.f, tau = -CUDART_INF_F;
	for (int s = tid; s < a.splits; s += kJoinThreads) {
		const float4 p = part[(size_t)s * rows];
		join(m, S, W, p.x, p.y, p.z, c);
		tau = fmaxf(tau, p.w);
	}
#pragma unroll
	for (int o = 16; o; o >>= 1) {
		const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
		const float s2 = __shfl_xor_sync(0xffffffffu, S, o);
		const float w2 = __shfl_xor_sync(0xffffffffu, W, o);
		join(m, S, W, m2, s2, w2, c);
		tau = fmaxf(tau, __shfl_xor_sync(0xffffffffu, tau, o));
	}
	if (lane == 0) {
		red[warp][0] = m;
		red[warp][1] = S;
		red[warp][2] = W;
		red[warp][3] = tau;
	}
	__syncthreads();
	m = red[0][0];
	S = red[0][1];
	W = red[0][2];
	tau = red[0][3];
#pragma unroll
	for (int i = 1; i < 4; ++i) {
		join(m, S, W, red[i][0], red[i][1], red[i][2], c);
		tau = fmaxf(tau, red[i][3]);
	}
	const bool dead = m == -CUDART_INF_F && S == 0.f;
	const float l2 = log2f(S), top = dead ? 0.f : m, ln_s = dead ? 0.f : l2 * kLn2;
	if (tid == 0) {
		if (a.lse)
			a.lse[r] = dead ? -CUDART_INF_F : fmaf(m, inv_t, ln_s);
		if (a.entropy)
			a.entropy[r] = dead ? 0.f : (l2 - W / S) * kLn2;
	}
	if (tid < nt) {
		const int t = a.targets[(size_t)r * nt + tid];
		const float l = dots[tid][0] + dots[tid][1] + dots[tid][2] + dots[tid][3];
		// this sum's order is not the tensor core's: l may round above the maximum
		a.target_lp[(size_t)r * nt + tid] =
		    (t >= 0 && t < a.vocab) ? fmaf(fminf(l - top, 0.f), inv_t, -ln_s) : -CUDART_INF_F;
	}
	if (k == 0)
		return;
	// the ranges whose maximum reaches the threshold, and their entries that do
	const float least = fmaxf(max_tau, tau);
	for (int s = tid; s < a.splits; s += kJoinThreads)
		if (part[(size_t)s * rows].x >= least)
			ranges[atomicAdd(&n_ranges, 1)] = s;
	__syncthreads();
	const int total = n_ranges * per;
#pragma unroll 4
	for (int i = tid; i < total; i += kJoinThreads) {
		const int g = i / per, e = i - g * per;
		const size_t at = (size_t)ranges[g] * rows + r;
		if (e < a.part_n[at]) {
			const uint2 x = static_cast<const uint2 *>(a.part_list)[(size_t)e * stride + at];
			const float v = __uint_as_float(x.x);
			if (v >= least) {
				const int p = atomicAdd(&n_cand, 1);
				cv[p] = v;
				ci[p] = (int)x.y;
			}
		}
	}
	__syncthreads();
	const int n = n_cand;
	for (int i = tid; i < n; i += kJoinThreads) {
		const float v = cv[i];
		const int id = ci[i];
		int at = 0;
#pragma unroll 4
		for (int j = 0; j < n; ++j)
			at += (int)(cv[j] > v) | ((int)(cv[j] == v) & (int)(ci[j] < id));
		if (at < k) {
			a.top_ids[(size_t)r * k + at] = id;
			a.top_lp[(size_t)r * k + at] = fmaf(v - top, inv_t, -ln_s);
		}
	}
	for (int i = n + tid; i < k; i += kJoinThreads) {   // fewer logits above -inf than top_n
		a.top_ids[(size_t)r * k + i] = -1;
		a.top_lp[(size_t)r * k + i] = -CUDART_INF_F;
	}
}

// [rows][hidden] bf16, box kSK x box_rows, 128-byte swizzle, zero fill past rows
bool make_rows_map(CUtensorMap *m, const void *base, int rows, int hidden, int box_rows)
{
	auto enc = get_encode();
	if (!enc)
		return false;
	cuuint64_t dims[2] = {(cuuint64_t)hidden, (cuuint64_t)rows};
	cuuint64_t strides[1] = {(cuuint64_t)hidden * 2};
	cuuint32_t box[2] = {(cuuint32_t)kSK, (cuuint32_t)box_rows};
	cuuint32_t estr[2] = {1, 1};
	return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims,
		   strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
		   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
		   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace kllm

using namespace kllm;

extern "C" void kllm_score_plan(int num_rows, int vocab, int num_sms, struct kllm_score_args *a)
{
	a->row_blocks = (num_rows + kSR - 1) / kSR;
	a->units = (vocab + kSU - 1) / kSU;
	const int groups = (a->row_blocks + 15) / 16;
	a->group_rb = (a->row_blocks + groups - 1) / groups;
	int q = num_sms / a->group_rb;
	if (q < 1)
		q = 1;
	if (q > kMaxSplits)
		q = kMaxSplits;
	if (q > a->units)
		q = a->units;
	a->splits = q;
}

extern "C" uint64_t kllm_score_workspace(const struct kllm_score_args *a)
{
	const uint64_t n = (uint64_t)a->splits * a->row_blocks * kSR;
	return n * 16u + (a->top_n > 0 ? n * 4u + n * 8u * (uint64_t)(a->top_n + kSlack) : 0u);
}

extern "C" int kllm_score_launch(struct kllm_score_args *a, void *workspace, void *stream)
{
	const uint64_t n = (uint64_t)a->splits * a->row_blocks * kSR;
	uint8_t *ws = static_cast<uint8_t *>(workspace);
	a->part = ws;
	a->part_list = ws + 16u * n;
	a->part_n = reinterpret_cast<int *>(ws + 16u * n + 8u * n * (uint64_t)(a->top_n + kSlack));
	CUtensorMap mh, mw, mw1;
	if (!make_rows_map(&mh, a->hidden, a->num_rows, a->hidden_dim, kSR) ||
	    !make_rows_map(&mw, a->weight, a->vocab, a->hidden_dim, kSN) ||
	    !make_rows_map(&mw1, a->weight, a->vocab, a->hidden_dim, kSU))
		return (int)cudaErrorInvalidValue;
	const size_t smem = sizeof(ScoreSmem) + 1024;
	cudaError_t e = cudaFuncSetAttribute(score_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
					     (int)smem);
	if (e != cudaSuccess)
		return (int)e;
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	score_kernel<<<a->group_rb * a->splits, kScThreads, smem, st>>>(*a, mh, mw, mw1);
	e = cudaGetLastError();
	if (e != cudaSuccess)
		return (int)e;
	// starts as the ranges' CTAs leave, with the targets' logits, which need none of them
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)a->num_rows);
	cfg.blockDim = dim3(kJoinThreads);
	cfg.dynamicSmemBytes = join_smem(a->splits, a->top_n);
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	return (int)cudaLaunchKernelEx(&cfg, score_join_kernel, (const struct kllm_score_args)*a);
}
