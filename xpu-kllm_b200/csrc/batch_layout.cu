// SPDX-License-Identifier: Apache-2.0
//
// batch_layout.cu - one scheduler step laid out on the GPU from the requests'
// lengths: block-table entries for the new blocks, and for every new token its
// row, position and slot (what the KV append and the chunked prefill take).
// The reference's scheduler does this on the host, one request at a time
// (userspace/reactor/batch_scheduler.c:258-263).
//
//   first[s] = sum of blocks wanted by the rows before s
//   cu[s]    = sum of new tokens of the rows before s
// are exclusive sums over at most 4,096 rows. Every CTA computes them for
// itself in shared memory (four rows a thread, one block scan), so that one
// launch does the whole step: a second launch to share one scan would cost
// more than the scan. Then the tokens are spread over the grid; a warp finds
// the row of its first token by a binary search in shared memory and its lanes
// walk on from there. Block j of a row is new exactly when token j *
// block_size is one of the row's new tokens, so the thread of that token writes
// the entry. Forked rows copy their parent's entries, one warp a row; a parent
// does not fork itself and its copied blocks are old ones, so no thread of the
// launch writes what another reads.

#include "kllm_device.cuh"
#include "kllm_internal.h"

namespace kllm {
namespace {

constexpr int kLayThreads = 1024;
constexpr int kLayRows = KLLM_MAX_SEQS_LAUNCH;
constexpr int kPerThread = kLayRows / kLayThreads;

struct LayEntry {
	unsigned long long k, v;
	long long valid;          // int valid + 4 bytes of padding
};

struct LaySmem {
	int ctx[kLayRows];        // effective lengths
	int cu[kLayRows + 1];     // exclusive sums of new tokens (cut at INT32_MAX)
	int first[kLayRows];      // exclusive sums of wanted blocks
	unsigned long long warp_sum[32];
};

// ctx and new of row s after clamping and the fork rules. Two rows' lengths
// are read at most; flags gains the error bits.
__device__ __forceinline__ void row_lengths(const kllm_layout_args &a, int s, int &ctx, int &nw,
					    int &parent, uint32_t &flags)
{
	const int cap = a.max_blocks * a.block_size;
	int c = max(a.ctx_lens[s], 0), n = max(a.new_lens[s], 0);
	if (c > cap || n > cap - min(c, cap))
		flags |= KLLM_ERR_SEQ_TOO_LONG_BIT;
	c = min(c, cap);
	n = min(n, cap - c);
	parent = a.fork_from ? a.fork_from[s] : -1;
	if (parent >= 0) {
		bool ok = parent < a.num_seqs && parent != s && c % a.block_size == 0;
		if (ok)
			ok = a.fork_from[parent] < 0 && c <= min(max(a.ctx_lens[parent], 0), cap);
		if (!ok) {
			c = n = 0;
			parent = -1;
			flags |= KLLM_ERR_LAYOUT_BIT;
		}
	}
	ctx = c;
	nw = n;
}

// Entry of the slot that free_slots names at `at`; false when there is none.
__device__ __forceinline__ bool free_entry(const kllm_layout_args &a, long long at, long long &slot,
					   LayEntry &e)
{
	slot = at < a.num_free ? (long long)a.free_slots[at] : -1;
	if (slot < 0 || (unsigned long long)slot >= a.total_slots) {
		e.k = e.v = 0ull;
		e.valid = 0;
		slot = -1;
		return false;
	}
	const unsigned long long base = a.arena_base + (unsigned long long)slot * a.slot_bytes;
	e.k = base + a.k_offset;
	e.v = base + a.v_offset;
	e.valid = 1;
	return true;
}

__device__ __forceinline__ unsigned long long warp_incl(unsigned long long x, int lane)
{
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
		if (lane >= o)
			x += y;
	}
	return x;
}

__global__ void __launch_bounds__(kLayThreads)
layout_kernel(const kllm_layout_args a)
{
	extern __shared__ __align__(16) uint8_t lay_raw[];
	LaySmem &sm = *reinterpret_cast<LaySmem *>(lay_raw);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int S = a.num_seqs, bs = a.block_size;
	const int gw = blockIdx.x * (kLayThreads / 32) + warp;      // warp of the grid
	const int n_warps = gridDim.x * (kLayThreads / 32);
	uint32_t flags = 0;

	// ---- lengths and their exclusive sums -------------------------------------
	// 64-bit sums: 4,096 rows of up to 2^30 tokens pass 32 bits
	int ctx[kPerThread], nw[kPerThread], need[kPerThread];
	unsigned long long tok = 0, blk = 0;
#pragma unroll
	for (int i = 0; i < kPerThread; ++i) {
		const int s = tid * kPerThread + i;
		ctx[i] = nw[i] = need[i] = 0;
		if (s < S) {
			int parent;
			row_lengths(a, s, ctx[i], nw[i], parent, flags);
			need[i] = (int)(((long long)ctx[i] + nw[i] + bs - 1) / bs -
					((long long)ctx[i] + bs - 1) / bs);
			sm.ctx[s] = ctx[i];
		}
		tok += (unsigned long long)nw[i];
		blk += (unsigned long long)need[i];
	}
	unsigned long long total[2];
	unsigned long long mine[2] = {tok, blk};
#pragma unroll
	for (int q = 0; q < 2; ++q) {
		const unsigned long long incl = warp_incl(mine[q], lane);
		if (lane == 31)
			sm.warp_sum[warp] = incl;
		__syncthreads();
		if (warp == 0)
			sm.warp_sum[lane] = warp_incl(sm.warp_sum[lane], lane);
		__syncthreads();
		const unsigned long long before = (warp ? sm.warp_sum[warp - 1] : 0ull) + incl - mine[q];
		total[q] = sm.warp_sum[31];
		unsigned long long run = before;
#pragma unroll
		for (int i = 0; i < kPerThread; ++i) {
			const int s = tid * kPerThread + i;
			if (s < S) {
				const int v = (int)min(run, 0x7fffffffull);
				if (q == 0)
					sm.cu[s] = v;
				else
					sm.first[s] = v;
			}
			run += (unsigned long long)(q == 0 ? nw[i] : need[i]);
		}
		__syncthreads();
	}
	if (tid == 0)
		sm.cu[S] = (int)min(total[0], 0x7fffffffull);
	__syncthreads();
	const int n_tok = sm.cu[S];
	if (total[0] > (unsigned long long)a.token_capacity)
		flags |= KLLM_ERR_LAYOUT_BIT;
	if (total[1] > (unsigned long long)a.num_free)
		flags |= KLLM_ERR_LAYOUT_BIT;

	if (blockIdx.x == 0) {
#pragma unroll
		for (int i = 0; i < kPerThread; ++i) {
			const int s = tid * kPerThread + i;
			if (s < S) {
				a.seq_lens[s] = ctx[i] + nw[i];
				a.cu_seqlens[s] = sm.cu[s];
			}
		}
		if (tid == 0) {
			a.cu_seqlens[S] = n_tok;
			if (a.counts) {
				a.counts[0] = n_tok;
				a.counts[1] = (int)min(total[1], 0x7fffffffull);
			}
		}
	}
	LayEntry *table = reinterpret_cast<LayEntry *>(a.table);

	// ---- forked rows: the parent's whole blocks ---------------------------------
	if (a.fork_from) {
		for (int s = gw; s < S; s += n_warps) {
			const int parent = a.fork_from[s];
			if (parent < 0 || parent >= S)
				continue;
			const int n = sm.ctx[s] / bs;     // 0 for a row that was refused
			const unsigned long long *src = reinterpret_cast<const unsigned long long *>(
			    table + (size_t)parent * a.max_blocks);
			unsigned long long *dst = reinterpret_cast<unsigned long long *>(
			    table + (size_t)s * a.max_blocks);
			for (int w = lane; w < 3 * n; w += 32)
				dst[w] = src[w];
		}
	}

	// ---- tokens ------------------------------------------------------------------
	const long long span = max((long long)n_tok, (long long)a.token_capacity);
	for (long long t0 = (long long)gw * 32; t0 < span; t0 += (long long)n_warps * 32) {
		const long long t = t0 + lane;
		if (t >= n_tok) {
			if (t < a.token_capacity) {
				a.token_seq[t] = -1;
				a.token_pos[t] = 0;
				if (a.slot_map)
					a.slot_map[t] = -1;
			}
			continue;
		}
		// the last row whose tokens start at or before t
		int lo = 0, hi = S - 1;
		while (lo < hi) {
			const int mid = (lo + hi + 1) >> 1;
			if ((long long)sm.cu[mid] <= t)
				lo = mid;
			else
				hi = mid - 1;
		}
		const int s = lo, c = sm.ctx[s], pos = c + (int)(t - sm.cu[s]);
		const int j = pos / bs, off = pos - j * bs, old = (int)(((long long)c + bs - 1) / bs);
		long long slot;
		if (j >= old) {
			LayEntry e;
			if (!free_entry(a, (long long)sm.first[s] + (j - old), slot, e))
				flags |= KLLM_ERR_LAYOUT_BIT;
			if (off == 0)
				table[(size_t)s * a.max_blocks + j] = e;
		} else {
			const LayEntry *e = table + (size_t)s * a.max_blocks + j;
			const bool ok = (int)(e->valid & 0xffffffffll) != 0;
			const unsigned long long at = (e->k - a.arena_base - a.k_offset) / a.slot_bytes;
			slot = ok && at < a.total_slots ? (long long)at : -1;
		}
		if (t < a.token_capacity) {
			a.token_seq[t] = s;
			a.token_pos[t] = pos;
			if (a.slot_map)
				a.slot_map[t] = slot < 0 ? -1 : slot * bs + off;
		}
	}
	if (flags && a.err)
		atomicOr(a.err, flags);
}

}  // namespace
}  // namespace kllm

using namespace kllm;

extern "C" int kllm_layout_launch(const struct kllm_layout_args *a, int num_sms, void *stream)
{
	cudaError_t e = cudaFuncSetAttribute(layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
					     (int)sizeof(LaySmem));
	if (e != cudaSuccess)
		return (int)e;
	// one CTA per 1,024 token rows, at most one per SM: each repeats the scan
	const long long by_tok = ((long long)a->token_capacity + kLayThreads - 1) / kLayThreads;
	const long long by_fork = a->fork_from ? (a->num_seqs + 31) / 32 : 1;
	long long grid = by_tok > by_fork ? by_tok : by_fork;
	if (grid > num_sms)
		grid = num_sms;
	if (grid < 1)
		grid = 1;
	layout_kernel<<<(int)grid, kLayThreads, sizeof(LaySmem),
			static_cast<cudaStream_t>(stream)>>>(*a);
	return (int)cudaGetLastError();
}
