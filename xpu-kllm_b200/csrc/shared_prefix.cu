// SPDX-License-Identifier: Apache-2.0
//
// shared_prefix.cu - decode attention of a batch whose groups of sequences
// share their leading pages (many samples of one prompt, one system prompt for
// all): the shared pages are read and multiplied once per group instead of
// once per sequence. The reference attends every sequence on its own
// (userspace/gpu/paged_attention.cu:24-119); the result is the same.
//
// For a row (sequence s, query head) of group g the context splits into the
// group's prefix of P tokens (whole pages) and the row's own suffix:
//   o = (sum_prefix 2^(x_i - M) v_i + sum_suffix 2^(x_i - M) v_i) / (same sums of 1)
// with x = scale log2(e) q.k, so (max, sum, o) triples of the two parts, and of
// any pieces of the prefix, join exactly. Four steps per call:
//
// plan_kernel     per row: its group, suffix length and suffix block table; per
//                 group: the row whose table names the prefix pages, the work.
// prefix_kernel   the prefix. All rows of a group that use one kv head (G
//                 query heads x its sequences) are the M dimension of the
//                 products: S = Q K^T and O += P V on tcgen05, 128 keys at a
//                 time. Below.
// decode kernels  the suffixes, by the split-KV decode over the suffix tables.
// join_kernel     both parts' triples -> the output rows.
//
// prefix_kernel. A unit is (group, kv head, up to 256 rows). Its key blocks are
// laid end to end over all units, and each of one CTA per SM takes an equal
// contiguous share (pieces leave fp32 partials). A unit of more than 128 rows
// runs as two query tiles that share every K/V block; a smaller one as two
// streams of one query tile that take alternate blocks, so that in both shapes
// one stream's products run under the other's softmax. Warps:
//   0-3 / 4-7  softmax of stream 0 / 1 (one row a thread)
//   8-11       producers: queries, then K and V blocks into the swizzled
//              operand layout (MX: dequantised to f16 from staged raw pages;
//              BF16: copied by cp.async)
//   12         TMEM allocation and MMA issue
//   13         page lookup and bulk copies of raw pages (three stages)
// MX computes in f16 like the decode: K and V are payload x scale / 4, the
// query row times a power of two; P is one f16 (11 bits; its 2^-12 stays under
// the output's 2^-9) built 2^7 larger, so that what underflows is below 2^-32
// of the row's largest. BF16 pages keep P as bf16 hi + lo: one bf16 P would add
// as much error as the output's own rounding.
// Every wait is bounded in wall time; a timeout sets KLLM_ERR_TIMEOUT.

#include "kllm_device.cuh"
#include "kllm_internal.h"
#include "kllm_umma.cuh"

#include <math_constants.h>

namespace kllm {
namespace {

constexpr int kPRows = 128, kPKeys = 128;
constexpr int kUnitRows = 256;
constexpr int kPThreads = 14 * 32;
constexpr int kWarpProd = 8, kWarpMma = 12;
constexpr int kRaw = 3;                       // raw stages (MX) / page-address stages (BF16)
constexpr float kRaise = 8.f;                 // slack of the lazy reference maximum, log2
constexpr float kPShift = 7.f;                // f16 P is built 2^7 larger
constexpr uint64_t kPWaitNs = 200000000ull;
constexpr float kPLog2e = 1.4426950408889634f;

struct PGroup {
	long long x0;         // first work step of the group's units
	long long r0;         // first partial row
	int row0, nseq;       // its sequences
	int nblk;             // 128-key blocks of the prefix (0: nothing shared)
	int npages;
	int leader;           // the sequence whose table names the prefix pages
	int tiles;            // 256-row units per kv head
	int wgt;              // work steps per block: 1 up to 128 rows, 2 above
	int alloc;            // partial rows per kv head
};
struct PHeader {
	long long T;          // work steps of the call
	int W;                // CTAs that share them
	int pad[13];
};
static_assert(sizeof(PHeader) == 64 && sizeof(PGroup) == 48, "workspace layout");

struct DevEntry {
	unsigned long long k, v;
	int valid;
	int pad;
};

// ---- plan ------------------------------------------------------------------------

constexpr int kPlanThreads = 256;

// Tokens of group g's prefix that are whole pages inside the table.
__device__ __forceinline__ int prefix_tokens(const kllm_prefix_args &a, int g)
{
	const int cap = a.max_blocks * a.block_size;
	return min(max(a.prefix_lens[g], 0), cap) / a.block_size * a.block_size;
}

__device__ __forceinline__ int row_length(const kllm_prefix_args &a, int s, bool &too_long)
{
	const int cap = a.max_blocks * a.block_size, L = a.seq_lens[s];
	too_long |= L > cap;
	return min(max(L, 0), cap);
}

__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const kllm_prefix_args a)
{
	__shared__ int leader[kPlanThreads];
	__shared__ long long sx[kPlanThreads / 32], sr[kPlanThreads / 32];
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int S = a.num_seqs, NG = a.num_groups;
	grid_launch_dependents();
	bool bad = false, too_long = false;
	for (int g = tid; g < NG; g += kPlanThreads) {
		const int b = a.group_starts[g], e = a.group_starts[g + 1];
		bad |= b < 0 || e < b || e > S;
	}
	// groups out of order or out of range: nothing is shared (the result stays
	// right) and the call is flagged
	bad = __syncthreads_or(bad);

	if (blockIdx.x == 0) {
		PHeader *hd = static_cast<PHeader *>(a.header);
		PGroup *gr = static_cast<PGroup *>(a.groups);
		long long run_x = 0, run_r = 0;
		for (int base = 0; base < NG; base += kPlanThreads) {
			// the first row of each group that holds the whole prefix
			for (int i = warp; i < kPlanThreads && base + i < NG; i += kPlanThreads / 32) {
				const int g = base + i, b = a.group_starts[g], e = a.group_starts[g + 1];
				int who = -1;
				if (!bad && e - b >= a.min_share) {
					const int P = prefix_tokens(a, g);
					for (int s0 = b; P > 0 && s0 < e && who < 0; s0 += 32) {
						const unsigned m = __ballot_sync(
						    0xffffffffu, s0 + lane < e && a.seq_lens[min(s0 + lane, e - 1)] >= P);
						if (m)
							who = s0 + __ffs(m) - 1;
					}
				}
				if (lane == 0)
					leader[i] = who;
			}
			__syncthreads();
			const int g = base + tid;
			PGroup p = {};
			long long x = 0, r = 0;
			if (g < NG) {
				p.row0 = a.group_starts[g];
				p.nseq = bad ? 0 : a.group_starts[g + 1] - p.row0;
				p.leader = leader[tid];
				const int rows = p.nseq * a.group;
				p.tiles = (rows + kUnitRows - 1) / kUnitRows;
				p.wgt = rows > kPRows ? 2 : 1;
				p.alloc = rows > kPRows ? rows : 2 * rows;
				if (p.leader >= 0) {
					p.npages = prefix_tokens(a, g) / a.block_size;
					const int ppb = kPKeys / a.block_size;
					p.nblk = (p.npages + ppb - 1) / ppb;
					x = (long long)a.num_kv_heads * p.tiles * p.nblk * p.wgt;
					r = (long long)a.num_kv_heads * p.alloc;
				}
			}
			// exclusive sums of x and r over the groups
			long long ix = x, ir = r;
#pragma unroll
			for (int o = 1; o < 32; o <<= 1) {
				const long long nx = __shfl_up_sync(0xffffffffu, ix, o);
				const long long nr = __shfl_up_sync(0xffffffffu, ir, o);
				if (lane >= o) {
					ix += nx;
					ir += nr;
				}
			}
			if (lane == 31) {
				sx[warp] = ix;
				sr[warp] = ir;
			}
			__syncthreads();
			long long bx = run_x, br = run_r;
			for (int w = 0; w < kPlanThreads / 32; ++w) {
				if (w < warp) {
					bx += sx[w];
					br += sr[w];
				}
				run_x += sx[w];
				run_r += sr[w];
			}
			if (g < NG) {
				p.x0 = bx + ix - x;
				p.r0 = br + ir - r;
				gr[g] = p;
			}
			__syncthreads();
		}
		if (tid == 0) {
			hd->T = run_x;
			hd->W = (int)(run_x < a.ctas ? run_x : a.ctas);
			if (bad && a.err)
				atomicOr(a.err, KLLM_ERR_LAYOUT_BIT);
		}
		return;
	}

	// one warp per row
	for (int s = (blockIdx.x - 1) * (kPlanThreads / 32) + warp; s < S;
	     s += (gridDim.x - 1) * (kPlanThreads / 32)) {
		const int L = row_length(a, s, too_long);
		int g = -1, P = 0;
		if (!bad && NG > 0) {
			int lo = 0, hi = NG - 1;            // the last group that starts at or before s
			while (lo < hi) {
				const int mid = (lo + hi + 1) >> 1;
				if (a.group_starts[mid] <= s)
					lo = mid;
				else
					hi = mid - 1;
			}
			const int b = a.group_starts[lo], e = a.group_starts[lo + 1];
			if (b <= s && s < e && e - b >= a.min_share) {
				P = prefix_tokens(a, lo);
				if (P > 0 && L >= P)
					g = lo;
				else
					P = 0;                  // too short a row: all of it is suffix
			}
		}
		const int j0 = P / a.block_size;
		const int n = (L - P + a.block_size - 1) / a.block_size;
		if (lane == 0) {
			a.row_group[s] = g;
			a.suf_lens[s] = L - P;
		}
		const unsigned long long *src = reinterpret_cast<const unsigned long long *>(
		    static_cast<const DevEntry *>(a.table) + (size_t)s * a.max_blocks + j0);
		unsigned long long *dst = reinterpret_cast<unsigned long long *>(
		    static_cast<DevEntry *>(a.suf_table) + (size_t)s * a.max_blocks);
		for (int w = lane; w < 3 * n; w += 32)
			dst[w] = src[w];
	}
	if (too_long && lane == 0 && a.err)
		atomicOr(a.err, KLLM_ERR_SEQ_TOO_LONG_BIT);
}

// ---- prefix ------------------------------------------------------------------------

template <int D, int KVT>
struct PG {
	static constexpr bool MX = KVT == 1;
	static constexpr int NH = D / 64;                     // 64-column halves
	static constexpr int HALF = kPRows * 128;             // bytes of one half tile
	static constexpr int TILE = NH * HALF;
	static constexpr int KB = MX ? 1 : 2;                 // K operand buffers
	static constexpr int RAW = MX ? kPKeys * D * 9 / 8 : 16;
	static constexpr int LPR = D / 8;                     // producer lanes per row
};

template <int D, int KVT>
struct PrefixSmem {
	using G = PG<D, KVT>;
	uint8_t q[2][G::TILE];
	uint8_t k[G::KB][G::TILE];
	uint8_t v[2][G::TILE];
	uint8_t raw[kRaw][G::RAW];
	float qf[2][2][kPRows];               // 2^-e of each query row (MX), by piece parity
	unsigned long long pg[kRaw][2][8];    // page addresses of a block (BF16)
	uint32_t slot_ok[kRaw];               // pages present, one bit each
	uint32_t key_ok[4][4];                // key masks of the last four blocks
	uint64_t q_full, q_empty;
	uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
	uint64_t raw_full[kRaw], raw_empty[kRaw];
	uint64_t s_full[2], p_half[2], p_full[2], o_full[2];
	uint64_t drain;
	uint32_t tmem_base;
	int abort;
};

__device__ __forceinline__ bool p_wait(int *abort_flag, uint64_t *bar, uint32_t parity,
				       uint32_t *err)
{
	if (mbar_try_wait(bar, parity))
		return true;
	const uint64_t t0 = global_ns();
	for (;;) {
		if (mbar_try_wait_sleep(bar, parity, 20000))
			return true;
		if (*reinterpret_cast<volatile int *>(abort_flag))
			return false;
		if (global_ns() - t0 > kPWaitNs) {
			*reinterpret_cast<volatile int *>(abort_flag) = 1;
			if (err)
				atomicOr(err, KLLM_ERR_TIMEOUT_BIT);
			return false;
		}
	}
}

// The pieces of one CTA's share of the work, in order: every role walks them.
struct Piece {
	int g, h, tile;       // group, kv head, 256-row unit of the head's rows
	int b0, nb;           // first block and number of blocks
	int rows;             // rows of the unit
	bool solo;            // one query tile, two streams of alternate blocks
	long long slot;       // first partial row
	int row0, leader, npages;
};

__device__ __forceinline__ int group_of_step(const PGroup *gr, int ng, long long x)
{
	int lo = 0, hi = ng - 1;
	while (lo < hi) {
		const int mid = (lo + hi + 1) >> 1;
		if (gr[mid].x0 <= x)
			lo = mid;
		else
			hi = mid - 1;
	}
	return lo;
}

// The piece that starts at step x < xe; advances x to its end.
__device__ __forceinline__ Piece next_piece(const kllm_prefix_args &a, long long &x, long long xe,
					    int cta)
{
	const PGroup *gr = static_cast<const PGroup *>(a.groups);
	Piece p;
	p.g = group_of_step(gr, a.num_groups, x);
	const PGroup G = gr[p.g];
	const long long cost = (long long)G.nblk * G.wgt;
	const long long u = (x - G.x0) / cost;
	const long long ux = G.x0 + u * cost;
	const long long end = min(xe, ux + cost);
	p.h = (int)(u / G.tiles);
	p.tile = (int)(u - (long long)p.h * G.tiles);
	p.b0 = (int)((x - ux) / G.wgt);
	p.nb = (int)((end - ux) / G.wgt) - p.b0;
	const int all = G.nseq * a.group;
	p.rows = min(kUnitRows, all - p.tile * kUnitRows);
	p.solo = G.wgt == 1;
	p.slot = G.r0 + (long long)p.h * G.alloc + p.tile * kUnitRows + (long long)kUnitRows * cta;
	p.row0 = G.row0;
	p.leader = G.leader;
	p.npages = G.npages;
	x = end;
	return p;
}

template <int KVT>
__device__ __forceinline__ uint32_t p_idesc(int n, bool b_mn_major)
{
	// kind::f16 with fp32 accumulators; operand types f16 (MX) or bf16
	const uint32_t types = KVT == 1 ? 0u : (1u << 7) | (1u << 10);
	return (1u << 4) | types | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
	       ((uint32_t)(kPRows >> 4) << 24);
}

__device__ __forceinline__ uint32_t swz(int row, int chunk16)
{
	return (uint32_t)row * 128u + (uint32_t)((chunk16 ^ (row & 7)) << 4);
}

// Two words (8 codes) of an MX block and its scale -> 8 f16 values payload x
// scale / 4. The hardware conversion reads codes 0x7F / 0xFF as NaN; the
// format's decoder reads them as +-480 (userspace/compute/mx_dequant.h:30-55),
// so a word that holds one is converted by placing the bits: s.eeee.mmm as
// s.0eeee.mmm0000000 is the value x 2^-8 for every code.
__device__ __forceinline__ uint4 mx8_to_f16(uint2 w, uint32_t sc)
{
	const uint32_t bits = ((sc & 0x80u) << 8) | ((sc & 0x7Fu) << 7);
	const uint32_t s = f16x2_mul(bits | (bits << 16), 0x54005400u);     // x 64: scale / 4
	uint4 o;
	o.x = e4m3x2_lo_to_f16x2(w.x);
	o.y = e4m3x2_hi_to_f16x2(w.x);
	o.z = e4m3x2_lo_to_f16x2(w.y);
	o.w = e4m3x2_hi_to_f16x2(w.y);
	const uint32_t t0 = (w.x & 0x7F7F7F7Fu) + 0x01010101u, t1 = (w.y & 0x7F7F7F7Fu) + 0x01010101u;
	if ((t0 | t1) & 0x80808080u) {
		const uint32_t ww[2] = {w.x, w.y};
		uint32_t r[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const uint32_t x = __byte_perm(ww[i >> 1], 0u, (i & 1) ? 0x4342u : 0x4140u);
			const uint32_t p = ((x & 0x007F007Fu) << 7) | ((x & 0x00800080u) << 8);
			r[i] = f16x2_mul(p, 0x5C005C00u);                           // x 2^8: exact
		}
		o = make_uint4(r[0], r[1], r[2], r[3]);
	}
	o.x = f16x2_mul(o.x, s);
	o.y = f16x2_mul(o.y, s);
	o.z = f16x2_mul(o.z, s);
	o.w = f16x2_mul(o.w, s);
	return o;
}

// One raw block (pages of bs tokens: payload rows, then scale rows) -> the
// operand tile [128 keys][D] f16, 128-byte swizzle. Absent pages give zeros.
template <int D>
__device__ __forceinline__ void dequant_block(uint8_t *dst, const uint8_t *raw, uint32_t ok, int bs,
					      int pt)
{
	constexpr int LPR = D / 8, RPP = 128 / LPR;      // rows per pass of 128 threads
	const int l = pt % LPR, sec = bs * D * 9 / 8;
	int row = pt / LPR, page = 0, tok = row;         // row < 16 <= bs
	uint8_t *out = dst + (l >> 3) * (kPRows * 128);
#pragma unroll 4
	for (int i = 0; i < kPKeys / RPP; ++i) {
		uint4 o = make_uint4(0u, 0u, 0u, 0u);
		if ((ok >> page) & 1u) {
			const uint8_t *p = raw + page * sec;
			const uint2 w = *reinterpret_cast<const uint2 *>(p + tok * D + l * 8);
			o = mx8_to_f16(w, p[bs * D + tok * LPR + l]);
		}
		*reinterpret_cast<uint4 *>(out + swz(row, l & 7)) = o;
		row += RPP;
		tok += RPP;
		if (tok >= bs) {
			tok -= bs;
			++page;
		}
	}
}

__device__ __forceinline__ void cp_async16(void *dst, const void *src)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
		     :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit()
{
	asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
	asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// Loads two 32-column chunks of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64])
{
	uint32_t r[64];
#pragma unroll
	for (int q = 0; q < 4; ++q)
		tmem_ld16_nowait(taddr + 16 * q, *reinterpret_cast<uint32_t (*)[16]>(&r[16 * q]));
#pragma unroll
	for (int q = 0; q < 4; ++q)
		asm volatile("tcgen05.wait::ld.sync.aligned;"
			     : "+r"(r[16 * q]), "+r"(r[16 * q + 1]), "+r"(r[16 * q + 2]),
			       "+r"(r[16 * q + 3]), "+r"(r[16 * q + 4]), "+r"(r[16 * q + 5]),
			       "+r"(r[16 * q + 6]), "+r"(r[16 * q + 7]), "+r"(r[16 * q + 8]),
			       "+r"(r[16 * q + 9]), "+r"(r[16 * q + 10]), "+r"(r[16 * q + 11]),
			       "+r"(r[16 * q + 12]), "+r"(r[16 * q + 13]), "+r"(r[16 * q + 14]),
			       "+r"(r[16 * q + 15])
			     :: "memory");
#pragma unroll
	for (int i = 0; i < 64; ++i)
		v[i] = __uint_as_float(r[i]);
}

// Masked scores of half `half` of a block: absent keys are -inf.
__device__ __forceinline__ void mask64(float (&v)[64], uint32_t m0, uint32_t m1)
{
#pragma unroll
	for (int i = 0; i < 64; ++i)
		if (!(((i < 32 ? m0 : m1) >> (i & 31)) & 1u))
			v[i] = -CUDART_INF_F;
}

// One 128-key block of one row: S in the TMEM columns of tS -> P over them
// (f16 pairs in columns 0-63, or bf16 groups of 8 hi + 8 lo). The row's block
// maximum is known before any P is written, so raising the reference rescales
// only O and l. Warp-collective; branches around TMEM accesses are
// warp-uniform. Returns through m_ref and l_sum.
template <int D, int KVT>
__device__ __forceinline__ void softmax_rows(uint32_t tS, uint32_t tO, const uint32_t *mask,
					     float sl2, bool o_live, float &m_ref, float &l_sum,
					     uint64_t *p_half)
{
	constexpr bool MX = KVT == 1;
	constexpr float shift = MX ? kPShift : 0.f;
	const uint32_t k0 = mask[0], k1 = mask[1], k2 = mask[2], k3 = mask[3];
	const bool full = (k0 & k1 & k2 & k3) == 0xFFFFFFFFu;   // the same for every lane
	float v[64];
	float mx = -CUDART_INF_F;
#pragma unroll
	for (int half = 0; half < 2; ++half) {
		tmem_ld64(tS + 64 * half, v);
		if (!full)
			mask64(v, half ? k2 : k0, half ? k3 : k1);
		float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
		for (int i = 4; i < 64; ++i)
			m4[i & 3] = fmaxf(m4[i & 3], v[i]);
		mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
	}
	const float gl = mx * sl2;
	const bool raise = gl > m_ref + kRaise;
	if (__any_sync(0xffffffffu, raise)) {
		const float f = raise ? exp2f(m_ref - gl) : 1.f;
		if (o_live) {
#pragma unroll 1
			for (int c = 0; c < D / 16; ++c) {
				float o[16];
				tmem_ld16(tO + 16 * c, o);
#pragma unroll
				for (int i = 0; i < 16; ++i)
					o[i] *= f;
				tmem_st16(tO + 16 * c, o);
			}
		}
		l_sum *= f;
		if (raise)
			m_ref = gl;
	}
	// no key present yet (m_ref = -inf): every p is 0, not exp2(-inf + inf)
	const float moff = m_ref == -CUDART_INF_F ? -CUDART_INF_F : shift - m_ref;
	float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int half = 0; half < 2; ++half) {
		tmem_ld64(tS + 64 * half, v);
		if (!full)
			mask64(v, half ? k2 : k0, half ? k3 : k1);
#pragma unroll
		for (int c = 0; c < 64; c += MX ? 32 : 16) {
			float w[16];
			if constexpr (MX) {
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					const float p0 = ex2_approx(fmaf(v[c + 2 * i], sl2, moff));
					const float p1 = ex2_approx(fmaf(v[c + 2 * i + 1], sl2, moff));
					sum[i & 3] += p0 + p1;
					w[i] = __uint_as_float(pack_f16x2(p0, p1));
				}
				tmem_st16_nowait(tS + 32 * half + c / 2, w);
			} else {
#pragma unroll
				for (int i = 0; i < 8; ++i) {
					const float p0 = ex2_approx(fmaf(v[c + 2 * i], sl2, moff));
					const float p1 = ex2_approx(fmaf(v[c + 2 * i + 1], sl2, moff));
					sum[i & 3] += p0 + p1;
					const uint32_t hi = pack_bf16x2(p0, p1);
					w[i] = __uint_as_float(hi);
					w[8 + i] = __uint_as_float(
					    pack_bf16x2(p0 - __uint_as_float(hi << 16),
							p1 - __uint_as_float(hi & 0xFFFF0000u)));
				}
				tmem_st16_nowait(tS + 64 * half + c, w);
			}
		}
		tmem_wait_st();
		if (half == 0) {
			tc_fence_before();
			mbar_arrive(p_half);
		}
	}
	l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int D, int KVT>
__global__ void __launch_bounds__(kPThreads, 1)
prefix_kernel(const kllm_prefix_args a)
{
	using G = PG<D, KVT>;
	using Sm = PrefixSmem<D, KVT>;
	extern __shared__ __align__(1024) uint8_t smem_raw[];
	Sm &sm = *reinterpret_cast<Sm *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
					 ~(uintptr_t)1023);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

	if (tid == 0) {
		mbar_init(&sm.q_full, 128);
		mbar_init(&sm.q_empty, 1);
		for (int i = 0; i < 2; ++i) {
			mbar_init(&sm.k_full[i], 128);
			mbar_init(&sm.k_empty[i], 1);
			mbar_init(&sm.v_full[i], 128);
			mbar_init(&sm.v_empty[i], 1);
			mbar_init(&sm.s_full[i], 1);
			mbar_init(&sm.p_half[i], 128);
			mbar_init(&sm.p_full[i], 128);
			mbar_init(&sm.o_full[i], 1);
		}
		for (int i = 0; i < kRaw; ++i) {
			mbar_init(&sm.raw_full[i], 1);
			mbar_init(&sm.raw_empty[i], 128);
		}
		mbar_init(&sm.drain, 1);
		sm.abort = 0;
		fence_mbar_init();
	}
	// the plan this launch reads is written by the kernel before it
	grid_dependency_wait();
	grid_launch_dependents();
	const PHeader *hd = static_cast<const PHeader *>(a.header);
	const long long T = hd->T;
	const int W = hd->W, cta = blockIdx.x;
	if (cta >= W)
		return;                            // uniform: no barrier has been used yet
	if (warp == kWarpMma) {
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
			     :: "r"(smem_u32(&sm.tmem_base)), "r"(512u));
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = sm.tmem_base;
	auto col_s = [](int t) { return (uint32_t)(t * 128); };
	auto col_o = [](int t) { return (uint32_t)(256 + t * 128); };
	long long x = cta * T / W;
	const long long xe = (cta + 1) * T / W;
	const int bs = a.block_size, ppb = kPKeys / bs;
	const int sec = bs * (G::MX ? D * 9 / 8 : D * 2);
	auto wait = [&](uint64_t *bar, uint32_t parity) { return p_wait(&sm.abort, bar, parity, a.err); };

	if (warp < kWarpProd) {
		// ================= softmax of stream t ========================================
		const int t = warp >> 2, rr = (warp & 3) * 32 + lane;
		const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
		const uint32_t tS = lane_base + col_s(t), tO = lane_base + col_o(t);
		int kf = 0, n_s = 0, n_o = 0, np = 0;        // K fills, S tiles, O tiles, pieces
		bool ok = true;
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			const int qt = p.solo ? 0 : t;
			const int row = qt * kPRows + rr;            // row of the unit
			const bool warp_live = qt * kPRows + (warp & 3) * 32 < p.rows;
			float m_ref = -CUDART_INF_F, l_sum = 0.f, sl2 = 0.f;
			bool first = true;
			for (int j = p.solo ? t : 0; j < p.nb; j += p.solo ? 2 : 1, ++n_s) {
				if (!__all_sync(0xffffffffu, wait(&sm.s_full[t], (uint32_t)(n_s & 1)))) {
					ok = false;
					break;
				}
				tc_fence_after();
				if (first)
					sl2 = a.scale_log2 * (G::MX ? sm.qf[np & 1][qt][rr] * KLLM_MX_DEC_UNBIAS : 1.f);
				if (warp_live)
					softmax_rows<D, KVT>(tS, tO, sm.key_ok[(kf + j) & 3], sl2, !first, m_ref,
							     l_sum, &sm.p_half[t]);
				else
					mbar_arrive(&sm.p_half[t]);
				tc_fence_before();
				mbar_arrive(&sm.p_full[t]);
				first = false;
			}
			kf += p.nb;
			++np;
			if (!ok)
				break;
			// ---- this piece's partial: m, l, O -------------------------------------
			const long long at = p.slot + (p.solo && t == 1 ? p.rows : 0);
			const bool live = row < p.rows;
			if (!first) {
				if (!__all_sync(0xffffffffu, wait(&sm.o_full[t], (uint32_t)(n_o & 1)))) {
					ok = false;
					break;
				}
				++n_o;
				tc_fence_after();
				if (warp_live) {
					// [D / 4][rows][4]: the warp's lanes store 512 contiguous bytes
					float *po = a.po + at * D + (size_t)row * 4;
#pragma unroll 2
					for (int c = 0; c < D / 16; ++c) {
						float o[16];
						tmem_ld16(tO + 16 * c, o);
						if (live)
#pragma unroll
							for (int i = 0; i < 4; ++i)
								*reinterpret_cast<float4 *>(po + (size_t)(4 * c + i) * p.rows * 4) =
								    make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
					}
					tc_fence_before();
				}
			}
			if (live) {
				a.pm[at + row] = m_ref - (G::MX ? kPShift : 0.f);
				a.pl[at + row] = l_sum;
			}
		}
	} else if (warp < kWarpMma) {
		// ================= producers ====================================================
		const int pt = tid - kWarpProd * 32;
		int np = 0, kf = 0, vf = 0, rf = 0;              // pieces, K fills, V fills, raw stages
		bool ok = true;
		// a warp leaves as a whole: the query loads shuffle across it
		auto wait_warp = [&](uint64_t *bar, uint32_t parity) {
			return __all_sync(0xffffffffu, wait(bar, parity));
		};
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			// ---- queries ------------------------------------------------------------
			if (np > 0 && !wait_warp(&sm.q_empty, (uint32_t)((np - 1) & 1)))
				break;
			{
				const int l = pt % G::LPR;
				const int all = p.rows;
				for (int t = 0; t < (p.solo ? 1 : 2); ++t)
					for (int r = pt / G::LPR; r < kPRows; r += 128 / G::LPR) {
						const int ru = t * kPRows + r;               // row of the unit
						const int rh = p.tile * kUnitRows + ru;      // row of the head
						const int seq = p.row0 + rh / a.group, hh = rh % a.group;
						uint4 w = make_uint4(0u, 0u, 0u, 0u);
						if (ru < all && a.row_group[seq] == p.g)
							w = __ldg(reinterpret_cast<const uint4 *>(
								static_cast<const uint8_t *>(a.q) +
								(((size_t)seq * a.num_heads + (size_t)p.h * a.group + hh) * D +
								 l * 8) * 2));
						if constexpr (G::MX) {
							// the row times 2^e, its largest in [2^14, 2^15)
							const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
							float mx = 0.f;
#pragma unroll
							for (int i = 0; i < 4; ++i)
								mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(ww[i] << 16)),
										     fabsf(__uint_as_float(ww[i] & 0xFFFF0000u))));
#pragma unroll
							for (int o = 1; o < G::LPR; o <<= 1)
								mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
							const int E = mx > 0.f ? (int)((__float_as_uint(mx) >> 23) & 0xFFu) - 127 : 0;
							const int e = min(max(14 - E, -100), 100);
							const float f = __uint_as_float((uint32_t)(e + 127) << 23);
							uint32_t o4[4];
#pragma unroll
							for (int i = 0; i < 4; ++i)
								o4[i] = pack_f16x2(__uint_as_float(ww[i] << 16) * f,
										   __uint_as_float(ww[i] & 0xFFFF0000u) * f);
							w = make_uint4(o4[0], o4[1], o4[2], o4[3]);
							if (l == 0)
								sm.qf[np & 1][t][r] = __uint_as_float((uint32_t)(127 - e) << 23);
						}
						*reinterpret_cast<uint4 *>(sm.q[t] + (l >> 3) * G::HALF + swz(r, l & 7)) = w;
					}
			}
			fence_async_smem();
			mbar_arrive(&sm.q_full);
			++np;
			// ---- K and V blocks ---------------------------------------------------------
			auto write_mask = [&](uint32_t okm) {
				if (pt < 4) {
					uint32_t m = 0;
#pragma unroll
					for (int i = 0; i < 2; ++i) {
						const int page = (32 * pt + 16 * i) / bs;
						if (page < ppb && ((okm >> page) & 1u))
							m |= 0xFFFFu << (16 * i);
					}
					sm.key_ok[kf & 3][pt] = m;
				}
			};
			if constexpr (G::MX) {
				for (int j = 0; j < p.nb && ok; ++j)
					for (int which = 0; which < 2; ++which, ++rf) {
						const int st = rf % kRaw;
						ok = wait_warp(&sm.raw_full[st], (uint32_t)((rf / kRaw) & 1));
						if (which == 0)
							ok = ok && (kf == 0 || wait_warp(&sm.k_empty[0], (uint32_t)((kf - 1) & 1)));
						else
							ok = ok && (vf < 2 || wait_warp(&sm.v_empty[vf & 1],
										   (uint32_t)(((vf >> 1) - 1) & 1)));
						if (!ok)
							break;
						const uint32_t okm = sm.slot_ok[st];
						dequant_block<D>(which ? sm.v[vf & 1] : sm.k[0], sm.raw[st], okm, bs, pt);
						if (which == 0)
							write_mask(okm);
						fence_async_smem();
						mbar_arrive(&sm.raw_empty[st]);
						if (which == 0) {
							mbar_arrive(&sm.k_full[0]);
							++kf;
						} else {
							mbar_arrive(&sm.v_full[vf & 1]);
							++vf;
						}
					}
			} else {
				// fills run two ahead of their arrival: K0 V0 K1 V1 ...
				const int l = pt % G::LPR;
				const int kf0 = kf, n_fill = 2 * p.nb;
				auto arrive_fill = [&](int f) {
					const int b = (kf0 + (f >> 1)) & 1;
					mbar_arrive((f & 1) ? &sm.v_full[b] : &sm.k_full[b]);
				};
				for (int f = 0; f < n_fill; ++f) {
					const int which = f & 1, st = rf % kRaw;
					int &cnt = which ? vf : kf;
					uint64_t *empty = which ? &sm.v_empty[cnt & 1] : &sm.k_empty[cnt & 1];
					if (which == 0)
						ok = wait_warp(&sm.raw_full[st], (uint32_t)((rf / kRaw) & 1));
					ok = ok && (cnt < 2 || wait_warp(empty, (uint32_t)(((cnt >> 1) - 1) & 1)));
					if (!ok)
						break;
					const uint32_t okm = sm.slot_ok[st];
					uint8_t *dst = (which ? sm.v[cnt & 1] : sm.k[cnt & 1]) + (l >> 3) * G::HALF;
					int row = pt / G::LPR, page = 0, tok = row;
					for (int i = 0; i < kPKeys * G::LPR / 128; ++i) {
						uint8_t *o = dst + swz(row, l & 7);
						if ((okm >> page) & 1u)
							cp_async16(o, reinterpret_cast<const uint8_t *>(sm.pg[st][which][page]) +
									  (size_t)tok * D * 2 + l * 16);
						else
							*reinterpret_cast<uint4 *>(o) = make_uint4(0u, 0u, 0u, 0u);
						row += 128 / G::LPR;
						tok += 128 / G::LPR;
						if (tok >= bs) {
							tok -= bs;
							++page;
						}
					}
					cp_async_commit();
					if (which == 0)
						write_mask(okm);
					else {
						mbar_arrive(&sm.raw_empty[st]);
						++rf;
					}
					++cnt;
					if (f >= 2) {
						cp_async_wait<2>();
						fence_async_smem();
						arrive_fill(f - 2);
					}
				}
				// the piece's last two fills
				cp_async_wait<0>();
				fence_async_smem();
				if (ok) {
					if (n_fill >= 2)
						arrive_fill(n_fill - 2);
					arrive_fill(n_fill - 1);
				}
			}
		}
	} else if (warp == kWarpMma) {
		// ================= MMA issue =======================================================
		// The whole warp runs this role (descriptors stay warp-uniform); one
		// elected lane issues.
		const bool leader = elect_one();
		const uint32_t id_s = p_idesc<KVT>(kPKeys, false), id_pv = p_idesc<KVT>(D, true);
		const uint64_t dq0 = umma_desc(smem_u32(sm.q[0]), 16u, 1024u);
		const uint64_t dq1 = umma_desc(smem_u32(sm.q[1]), 16u, 1024u);
		const uint64_t dk0 = umma_desc(smem_u32(sm.k[0]), 16u, 1024u);
		const uint64_t dk1 = umma_desc(smem_u32(sm.k[G::KB - 1]), 16u, 1024u);
		const uint64_t dv0 = umma_desc(smem_u32(sm.v[0]), (uint32_t)G::HALF, 1024u);
		const uint64_t dv1 = umma_desc(smem_u32(sm.v[1]), (uint32_t)G::HALF, 1024u);
		int kf = 0, vf = 0, np = 0, n_p[2] = {0, 0};
		auto wait_all = [&](uint64_t *bar, uint32_t parity) {
			return __all_sync(0xffffffffu, wait(bar, parity));
		};
		auto commit = [&](uint64_t *bar) {
			if (leader)
				umma_commit(bar);
			__syncwarp();
		};
		auto wait_k = [&]() {
			const int b = G::KB == 1 ? 0 : kf & 1, round = G::KB == 1 ? kf : kf >> 1;
			return wait_all(&sm.k_full[b], (uint32_t)(round & 1));
		};
		auto free_k = [&]() {
			commit(&sm.k_empty[G::KB == 1 ? 0 : kf & 1]);
			++kf;
		};
		auto issue_s = [&](int t, int qt) {
			const uint64_t dq = qt ? dq1 : dq0, dk = (G::KB == 2 && (kf & 1)) ? dk1 : dk0;
#pragma unroll
			for (int kk = 0; kk < D / 16; ++kk) {
				const uint64_t off = ((uint64_t)(kk >> 2) * G::HALF + (uint64_t)(kk & 3) * 32u) >> 4;
				if (leader)
					umma_f16(tmem + col_s(t), dq + off, dk + off, id_s, kk > 0);
			}
			__syncwarp();
			commit(&sm.s_full[t]);
		};
		auto issue_pv = [&](int t, bool first, int half) {
			const uint64_t dv = (vf & 1) ? dv1 : dv0;
			const uint32_t d = tmem + col_o(t), pa = tmem + col_s(t);
#pragma unroll
			for (int g = half * 4; g < half * 4 + 4; ++g) {        // 16-key groups
				if constexpr (G::MX) {
					if (leader)
						umma_f16_ts(d, pa + 8u * g, dv + (uint64_t)((g * 2048) >> 4), id_pv,
							    (first && g == 0) ? 0u : 1u);
				} else {
#pragma unroll
					for (int lo = 0; lo < 2; ++lo)
						if (leader)
							umma_f16_ts(d, pa + 16u * g + 8u * lo, dv + (uint64_t)((g * 2048) >> 4),
								    id_pv, (first && g == 0 && lo == 0) ? 0u : 1u);
				}
			}
			__syncwarp();
		};
		// P of stream t's next block -> O, in two halves of 64 keys
		auto take_p = [&](int t, bool first) {
			if (!wait_all(&sm.p_half[t], (uint32_t)(n_p[t] & 1)))
				return false;
			tc_fence_after();
			issue_pv(t, first, 0);
			if (!wait_all(&sm.p_full[t], (uint32_t)(n_p[t] & 1)))
				return false;
			tc_fence_after();
			issue_pv(t, first, 1);
			++n_p[t];
			return true;
		};
		bool ok = true;
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			ok = wait_all(&sm.q_full, (uint32_t)(np & 1)) && wait_k();
			if (!ok)
				break;
			++np;
			tc_fence_after();
			issue_s(0, 0);
			if (!p.solo)
				issue_s(1, 1);
			free_k();
			if (p.solo && p.nb > 1) {
				ok = wait_k();
				if (!ok)
					break;
				tc_fence_after();
				issue_s(1, 0);
				free_k();
			}
			if (p.nb <= (p.solo ? 2 : 1))
				commit(&sm.q_empty);
			for (int j = 0; j < p.nb && ok; ++j) {
				ok = wait_all(&sm.v_full[vf & 1], (uint32_t)((vf >> 1) & 1));
				if (!ok)
					break;
				if (p.solo) {
					const int t = j & 1;
					ok = take_p(t, j < 2);
					if (!ok)
						break;
					commit(&sm.v_empty[vf & 1]);
					if (j + 2 < p.nb) {
						ok = wait_k();
						if (!ok)
							break;
						tc_fence_after();
						issue_s(t, 0);
						free_k();
						if (j + 3 == p.nb)
							commit(&sm.q_empty);
					} else {
						commit(&sm.o_full[t]);
					}
				} else {
					for (int t = 0; t < 2 && ok; ++t) {
						ok = take_p(t, j == 0);
						if (!ok)
							break;
						if (t == 1)
							commit(&sm.v_empty[vf & 1]);
						if (j + 1 < p.nb) {
							if (t == 0)
								ok = wait_k();
							if (!ok)
								break;
							tc_fence_after();
							issue_s(t, t);
							if (t == 1) {
								free_k();
								if (j + 2 == p.nb)
									commit(&sm.q_empty);
							}
						} else {
							commit(&sm.o_full[t]);
						}
					}
				}
				++vf;
			}
		}
		// every MMA issued completes before TMEM is freed
		commit(&sm.drain);
		mbar_wait_ns(&sm.drain, 0u, kPWaitNs);
	} else {
		// ================= page lookup and raw copies ========================================
		int rf = 0;
		uint32_t armed[kRaw] = {0, 0, 0};
		bool ok = true;
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			const DevEntry *tb = static_cast<const DevEntry *>(a.table) +
					     (size_t)p.leader * a.max_blocks;
			auto load = [&](int b, DevEntry &e) {
				const int page = b * ppb + lane;
				e.k = e.v = 0ull;
				e.valid = 0;
				if (lane < ppb && page < p.npages) {
					e.k = __ldg(&tb[page].k);
					e.v = __ldg(&tb[page].v);
					e.valid = __ldg(&tb[page].valid);
				}
			};
			DevEntry nxt;
			load(p.b0, nxt);
			for (int j = 0; j < p.nb && ok; ++j) {
				const DevEntry e = nxt;
				if (j + 1 < p.nb)
					load(p.b0 + j + 1, nxt);
				const bool present = e.valid && e.k != 0ull;
				const bool aligned = ((e.k | e.v) & 15ull) == 0ull;
				if (present && !aligned && a.err)
					atomicOr(a.err, 0x2u);
				const unsigned long long off = a.layer_off + (unsigned long long)p.h * sec;
				bool here = present && aligned;
				if (here && !(in_arenas(a.arenas, e.k + off, sec) &&
					      in_arenas(a.arenas, e.v + off, sec))) {
					here = false;
					if (a.err)
						atomicOr(a.err, KLLM_ERR_PAGE_RANGE_BIT);
				}
				const uint32_t mask = __ballot_sync(0xffffffffu, here);
				for (int which = 0; which < (G::MX ? 2 : 1); ++which, ++rf) {
					const int st = rf % kRaw;
					if (rf >= kRaw)
						ok = __all_sync(0xffffffffu, wait(&sm.raw_empty[st],
										  (uint32_t)((rf / kRaw - 1) & 1)));
					if (!ok)
						break;
					if constexpr (G::MX) {
						if (lane == 0) {
							sm.slot_ok[st] = mask;
							mbar_arrive_expect_tx(&sm.raw_full[st], (uint32_t)(__popc(mask) * sec));
						}
#pragma unroll
						for (int i = 0; i < kRaw; ++i)
							armed[i] += i == st ? 1u : 0u;
						__syncwarp();
						if (here)
							bulk_g2s(sm.raw[st] + lane * sec,
								 reinterpret_cast<const void *>((which ? e.v : e.k) + off),
								 (uint32_t)sec, &sm.raw_full[st]);
					} else {
						if (lane < 8) {
							sm.pg[st][0][lane] = e.k + off;
							sm.pg[st][1][lane] = e.v + off;
						}
						if (lane == 0)
							sm.slot_ok[st] = mask;
						__syncwarp();
						if (lane == 0)
							mbar_arrive(&sm.raw_full[st]);
					}
				}
			}
		}
		// after an abort, wait (bounded) for this CTA's own bulk copies
		if (G::MX && *reinterpret_cast<volatile int *>(&sm.abort))
#pragma unroll
			for (int i = 0; i < kRaw; ++i)
				if (armed[i] > 0)
					mbar_wait_ns(&sm.raw_full[i], (armed[i] - 1) & 1u, kPWaitNs);
	}

	tc_fence_before();
	__syncthreads();
	if (warp == kWarpMma) {
		__syncwarp();
		tc_fence_after();
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
			     :: "r"(tmem), "r"(512u));
	}
}

// ---- join -----------------------------------------------------------------------------

constexpr int kJThreads = 256;
constexpr int kJRows = 32;

// One CTA: 32 consecutive rows (sequence-major) of one kv head. Phase 1: a lane
// per row, a warp per chunk of 4 dims: the prefix pieces' sums against their
// maximum (the partials hold [D / 4][rows][4], so a warp reads 512 contiguous
// bytes). Phase 2: eight threads per row add the suffix triple and store.
template <int D>
__global__ void __launch_bounds__(kJThreads)
join_kernel(const kllm_prefix_args a, float unbias)
{
	__shared__ float acc_s[kJRows][D + 4];
	__shared__ float m_s[kJRows], l_s[kJRows];
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int h = blockIdx.y, rows = a.num_seqs * a.group;
	grid_dependency_wait();
	const PHeader *hd = static_cast<const PHeader *>(a.header);
	const long long T = hd->T, W = hd->W;
	const int i = blockIdx.x * kJRows + lane;
	{
		const int seq = i / a.group;
		const int g = i < rows ? a.row_group[seq] : -1;
		float M = -CUDART_INF_F, L = 0.f;
		float acc[D / 32][4];
#pragma unroll
		for (int c = 0; c < D / 32; ++c)
#pragma unroll
			for (int q = 0; q < 4; ++q)
				acc[c][q] = 0.f;
		if (g >= 0) {
			const PGroup G = static_cast<const PGroup *>(a.groups)[g];
			const int lr = (seq - G.row0) * a.group + i % a.group;
			const bool solo = G.wgt == 1;
			const int tile = lr / kUnitRows, r = lr - tile * kUnitRows;
			const int urows = min(kUnitRows, G.nseq * a.group - tile * kUnitRows);
			const long long cost = (long long)G.nblk * G.wgt;
			const long long ux = G.x0 + ((long long)h * G.tiles + tile) * cost;
			const long long c0 = ((ux + 1) * W - 1) / T, c1 = ((ux + cost) * W - 1) / T;
			const long long base = G.r0 + (long long)h * G.alloc + tile * kUnitRows;
			for (int pass = 0; pass < 2; ++pass)
				for (long long c = c0; c <= c1; ++c) {
					const long long lo = max(c * T / W, ux), hi = min((c + 1) * T / W, ux + cost);
					if ((hi - ux) / G.wgt <= (lo - ux) / G.wgt)
						continue;              // no whole block in this share
					for (int st = 0; st < (solo ? 2 : 1); ++st) {
						const long long at = base + (long long)kUnitRows * c + st * urows;
						const float l = __ldcg(a.pl + at + r), m = __ldcg(a.pm + at + r);
						if (!(l != 0.f))
							continue;
						if (pass == 0) {
							M = fmaxf(M, m);
							continue;
						}
						const float e = exp2f(m - M);
						L = fmaf(l, e, L);
						const float *po = a.po + at * D + (size_t)r * 4;
#pragma unroll
						for (int q = 0; q < D / 32; ++q) {
							const float4 o = __ldcg(reinterpret_cast<const float4 *>(
							    po + (size_t)(warp + 8 * q) * urows * 4));
							acc[q][0] = fmaf(o.x, e, acc[q][0]);
							acc[q][1] = fmaf(o.y, e, acc[q][1]);
							acc[q][2] = fmaf(o.z, e, acc[q][2]);
							acc[q][3] = fmaf(o.w, e, acc[q][3]);
						}
					}
				}
		}
#pragma unroll
		for (int q = 0; q < D / 32; ++q)
			*reinterpret_cast<float4 *>(&acc_s[lane][4 * (warp + 8 * q)]) =
			    make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
		if (warp == 0) {
			m_s[lane] = M;
			l_s[lane] = L;
		}
	}
	__syncthreads();
	const int r = tid >> 3, part = tid & 7, ii = blockIdx.x * kJRows + r;
	if (ii >= rows)
		return;
	const size_t row = (size_t)(ii / a.group) * a.num_heads + (size_t)h * a.group + ii % a.group;
	const float Ms = a.sm[row] * kPLog2e, Ls = a.sl[row], Mp = m_s[r], Lp = l_s[r];
	const float M = fmaxf(Ls > 0.f ? Ms : -CUDART_INF_F, Lp > 0.f ? Mp : -CUDART_INF_F);
	const float wp = Lp > 0.f ? exp2f(Mp - M) : 0.f;
	const float ws = Ls > 0.f ? Ls * exp2f(Ms - M) : 0.f;
	const float den = fmaf(Lp, wp, ws);
	const float fp = den > 0.f ? wp * unbias / den : 0.f, fs = den > 0.f ? ws / den : 0.f;
	constexpr int N = D / 8;                      // dims per thread
	const float *so = a.so + row * D + part * N;
	uint32_t o[N / 2];
#pragma unroll
	for (int c = 0; c < N; c += 4) {
		const float4 s = *reinterpret_cast<const float4 *>(so + c);
		const float4 p = *reinterpret_cast<const float4 *>(&acc_s[r][part * N + c]);
		o[c / 2] = pack_bf16x2(fmaf(p.x, fp, s.x * fs), fmaf(p.y, fp, s.y * fs));
		o[c / 2 + 1] = pack_bf16x2(fmaf(p.z, fp, s.z * fs), fmaf(p.w, fp, s.w * fs));
	}
	uint4 *out = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(a.out) + (row * D + part * N) * 2);
#pragma unroll
	for (int c = 0; c < N / 8; ++c)
		out[c] = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem,
			     cudaStream_t st, int dependent, Args... args)
{
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid;
	cfg.blockDim = dim3((unsigned)block);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = dependent ? 1 : 0;
	return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int KVT>
cudaError_t launch_prefix(const kllm_prefix_args &a, cudaStream_t st)
{
	// more than half an SM's shared memory, so that one CTA has the SM's TMEM
	size_t smem = sizeof(PrefixSmem<D, KVT>) + 1024;
	if (smem < 120u * 1024u)
		smem = 120u * 1024u;
	const cudaError_t e = cudaFuncSetAttribute(
	    prefix_kernel<D, KVT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
	if (e != cudaSuccess)
		return e;
	return launch_dependent(prefix_kernel<D, KVT>, dim3((unsigned)a.ctas), kPThreads, smem, st, 1, a);
}

}  // namespace
}  // namespace kllm

using namespace kllm;

static uint64_t up256(uint64_t x) { return (x + 255u) & ~(uint64_t)255u; }

extern "C" uint64_t kllm_prefix_workspace(int num_seqs, int num_heads, int head_dim, int max_blocks,
					  int ctas, void *base, struct kllm_prefix_args *a)
{
	uint8_t *p = static_cast<uint8_t *>(base);
	const uint64_t S = (uint64_t)num_seqs, rows = S * num_heads;
	const uint64_t part = 2u * rows + (uint64_t)kUnitRows * ctas;
	uint64_t at = 0;
	auto take = [&](uint64_t bytes) {
		uint8_t *q = p + at;
		at += up256(bytes);
		return q;
	};
	uint8_t *header = take(sizeof(PHeader)), *groups = take(S * sizeof(PGroup));
	uint8_t *rg = take(S * 4), *sl = take(S * 4), *stb = take(S * max_blocks * 24);
	uint8_t *sm = take(rows * 4), *sll = take(rows * 4), *so = take(rows * head_dim * 4);
	uint8_t *pm = take(part * 4), *pl = take(part * 4), *po = take(part * head_dim * 4);
	if (a) {
		a->header = header;
		a->groups = groups;
		a->row_group = reinterpret_cast<int *>(rg);
		a->suf_lens = reinterpret_cast<int *>(sl);
		a->suf_table = stb;
		a->sm = reinterpret_cast<float *>(sm);
		a->sl = reinterpret_cast<float *>(sll);
		a->so = reinterpret_cast<float *>(so);
		a->pm = reinterpret_cast<float *>(pm);
		a->pl = reinterpret_cast<float *>(pl);
		a->po = reinterpret_cast<float *>(po);
	}
	return at;
}

extern "C" int kllm_prefix_launch(const struct kllm_prefix_args *a, void *stream)
{
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	const int wpb = kPlanThreads / 32;
	const int row_ctas = (a->num_seqs + wpb - 1) / wpb;
	plan_kernel<<<1 + (row_ctas < 512 ? row_ctas : 512), kPlanThreads, 0, st>>>(*a);
	cudaError_t e = cudaGetLastError();
	if (e != cudaSuccess)
		return (int)e;
	if (a->head_dim == 128)
		e = a->kv_dtype ? launch_prefix<128, 1>(*a, st) : launch_prefix<128, 0>(*a, st);
	else
		e = a->kv_dtype ? launch_prefix<64, 1>(*a, st) : launch_prefix<64, 0>(*a, st);
	return (int)e;
}

extern "C" int kllm_prefix_join_launch(const struct kllm_prefix_args *a, void *stream)
{
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	const dim3 grid((unsigned)(((long long)a->num_seqs * a->group + kJRows - 1) / kJRows),
			(unsigned)a->num_kv_heads);
	const float unbias = a->kv_dtype ? KLLM_MX_DEC_UNBIAS : 1.f;
	if (a->head_dim == 128)
		return (int)launch_dependent(join_kernel<128>, grid, kJThreads, 0, st, 1, *a, unbias);
	return (int)launch_dependent(join_kernel<64>, grid, kJThreads, 0, st, 1, *a, unbias);
}
