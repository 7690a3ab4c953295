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
// more than the scan. Then each warp takes a contiguous run of tokens, finds the
// row of its first one by 32 probes a round in shared memory and walks on from
// there. Block j of a row is new exactly when token j *
// block_size is one of the row's new tokens, so the thread of that token writes
// the entry. Forked rows copy their parent's entries, one warp a row; a parent
// does not fork itself and its copied blocks are old ones, so no thread of the
// launch writes what another reads.
//
// Bound: the instructions that every CTA repeats (lengths, scan: a scheduler issues
// in 54 % of its cycles) and their latency (of 13 cycles between two instructions
// of a warp 2.8 wait for the one before, 2.1 for L2, 1.8 for shared memory); the
// bytes are 2 us of HBM. Measured: 4,096 rows, one in five forked, with 528,000
// token rows (13.6 MB) 18 us, 0.8 TB/s; 16 rows 6 us behind other work, 11.6 us as
// a call by itself, which is the host's part.

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
	unsigned long long warp_tok[32], warp_blk[32];
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

// Blocks of n tokens; n is at most 2^31 - 1 and the sum stays in 32 bits unsigned.
__device__ __forceinline__ int blocks_of(int n, int bs)
{
	return (int)(((unsigned)n + (unsigned)bs - 1u) / (unsigned)bs);
}

// x / d for quotients below 2^52, inv = 1 / d: a 64-bit division is some 100
// instructions, and a decode step's tokens all need one.
__device__ __forceinline__ unsigned long long div_small(unsigned long long x, unsigned long long d, double inv)
{
	unsigned long long q = (unsigned long long)((double)x * inv);    // off by one at most
	if (q * d > x)
		--q;
	else if (x - q * d >= d)
		++q;
	return q;
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
			need[i] = blocks_of(ctx[i] + nw[i], bs) - blocks_of(ctx[i], bs);
			sm.ctx[s] = ctx[i];
		}
		tok += (unsigned long long)nw[i];
		blk += (unsigned long long)need[i];
	}
	const unsigned long long it = warp_incl(tok, lane), ib = warp_incl(blk, lane);
	if (lane == 31) {
		sm.warp_tok[warp] = it;
		sm.warp_blk[warp] = ib;
	}
	__syncthreads();
	if (warp < 2) {
		unsigned long long *w = warp ? sm.warp_blk : sm.warp_tok;
		w[lane] = warp_incl(w[lane], lane);
	}
	__syncthreads();
	const unsigned long long total[2] = {sm.warp_tok[31], sm.warp_blk[31]};
	unsigned long long run_t = (warp ? sm.warp_tok[warp - 1] : 0ull) + it - tok;
	unsigned long long run_b = (warp ? sm.warp_blk[warp - 1] : 0ull) + ib - blk;
#pragma unroll
	for (int i = 0; i < kPerThread; ++i) {
		const int s = tid * kPerThread + i;
		if (s < S) {
			sm.cu[s] = (int)min(run_t, 0x7fffffffull);
			sm.first[s] = (int)min(run_b, 0x7fffffffull);
		}
		run_t += (unsigned long long)nw[i];
		run_b += (unsigned long long)need[i];
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
				if (a.seq_lens)
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
			// a batch of loads before its stores: one at a time, a row of 1,000
			// blocks was 96 round trips and most of the launch
			constexpr int kFly = 12;
			for (int w0 = lane; w0 < 3 * n; w0 += 32 * kFly) {
				unsigned long long v[kFly];
#pragma unroll
				for (int q = 0; q < kFly; ++q)
					if (w0 + 32 * q < 3 * n)
						v[q] = src[w0 + 32 * q];
#pragma unroll
				for (int q = 0; q < kFly; ++q)
					if (w0 + 32 * q < 3 * n)
						dst[w0 + 32 * q] = v[q];
			}
		}
	}

	// ---- tokens ------------------------------------------------------------------
	// Each warp takes a contiguous run of them. It finds the row of its first
	// token by 32 probes a round, and from there on a lane looks only between the
	// rows of the warp's first and last token.
	const long long span = max((long long)n_tok, (long long)a.token_capacity);
	const long long per = ((span + n_warps - 1) / n_warps + 31) / 32 * 32;
	const long long end = min(span, (gw + 1) * per);
	const double inv_slot = 1.0 / (double)a.slot_bytes;
	// the last row whose tokens start at or before t < n_tok
	auto row_of = [&](int t) {
		int lo = 0, hi = S - 1;
		while (lo < hi) {
			const int step = (hi - lo + 31) / 32;              // rows lo + 1 .. hi
			const int at = lo + 1 + lane * step;
			const unsigned b = __ballot_sync(0xffffffffu, at <= hi && sm.cu[min(at, hi)] <= t);
			const int n = __popc(b);                           // the first n probes hold
			hi = n ? min(hi, lo + n * step) : lo;
			lo = n ? lo + 1 + (n - 1) * step : lo;
		}
		return lo;
	};
	int s0 = -1;
	for (long long t0 = (long long)gw * per; t0 < end; t0 += 32) {
		const long long t = t0 + lane;
		int s1 = s0;
		if (t0 < n_tok) {
			if (s0 < 0)
				s0 = row_of((int)t0);
			s1 = row_of((int)min(t0 + 31, (long long)n_tok - 1));
		}
		if (t >= n_tok) {
			if (t < a.token_capacity) {
				a.token_seq[t] = -1;
				a.token_pos[t] = 0;
				if (a.slot_map)
					a.slot_map[t] = -1;
			}
			continue;
		}
		int lo = s0, hi = s1;
		while (lo < hi) {
			const int mid = (lo + hi + 1) >> 1;
			if (sm.cu[mid] <= (int)t)
				lo = mid;
			else
				hi = mid - 1;
		}
		s0 = s1;
		const int s = lo, c = sm.ctx[s], pos = c + (int)(t - sm.cu[s]);
		const int j = pos / bs, off = pos - j * bs, old = blocks_of(c, bs);
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
			const unsigned long long at = div_small(e->k - a.arena_base - a.k_offset, a.slot_bytes, inv_slot);
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

// seq_lens alone, where it overlaps the lengths: one CTA, which has read every
// row before it writes one.
__global__ void __launch_bounds__(kLayThreads)
lengths_kernel(const kllm_layout_args a)
{
	int len[kPerThread];
#pragma unroll
	for (int i = 0; i < kPerThread; ++i) {
		const int s = threadIdx.x * kPerThread + i;
		int ctx = 0, nw = 0, parent;
		uint32_t flags = 0;        // the main launch sets them
		if (s < a.num_seqs)
			row_lengths(a, s, ctx, nw, parent, flags);
		len[i] = ctx + nw;
	}
	__syncthreads();
#pragma unroll
	for (int i = 0; i < kPerThread; ++i) {
		const int s = threadIdx.x * kPerThread + i;
		if (s < a.num_seqs)
			a.seq_lens[s] = len[i];
	}
}

}  // namespace
}  // namespace kllm

using namespace kllm;

// Two arrays of n ints share an element.
static bool overlap(const int *x, const int *y, size_t n)
{
	const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
	return a < b + 4 * n && b < a + 4 * n;
}

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
	// Lengths updated in place: every CTA reads all of them, and none knows when the
	// others have, so seq_lens waits for a launch of its own (a single CTA reads
	// before it writes). 4,096 rows with 528,000 token rows take 22 us so, 600 when
	// one CTA does all.
	const size_t n = (size_t)a->num_seqs;
	const bool after = grid > 1 && (overlap(a->seq_lens, a->ctx_lens, n) ||
					overlap(a->seq_lens, a->new_lens, n));
	struct kllm_layout_args b = *a;
	if (after)
		b.seq_lens = nullptr;
	layout_kernel<<<(int)grid, kLayThreads, sizeof(LaySmem),
			static_cast<cudaStream_t>(stream)>>>(b);
	e = cudaGetLastError();
	if (e != cudaSuccess || !after)
		return (int)e;
	lengths_kernel<<<1, kLayThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
	return (int)cudaGetLastError();
}
