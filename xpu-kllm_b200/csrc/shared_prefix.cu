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
// any pieces of either, join exactly. Three launches per call:
//
// plan_kernel     per row: its group and suffix; per group: the row whose table
//                 names the prefix pages, the work; how many CTAs take which part.
// attend_kernel   one CTA per SM. The first ones take the prefixes
//                 (prefix_role), the others the suffixes (suffix_role), so that
//                 the two run at the same time instead of one after the other.
// join_kernel     both parts' triples -> the output rows.
//
// prefix_role. All rows of a group that use one kv head (G query heads x its
// sequences) are the M dimension of the products: S = Q K^T and O += P V on
// tcgen05, 128 keys at a time. A unit is (group, kv head, up to 256 rows). Its
// key blocks are laid end to end over all units, and each CTA takes an equal
// contiguous share (pieces leave fp32 partials). A unit of more than 128 rows
// runs as two query tiles that share every K/V block; a smaller one as two
// streams of one query tile that take alternate blocks, so that in both shapes
// one stream's products run under the other's softmax. Warps:
//   0-3 / 4-7  one row a thread: queries into the operand tile, softmax of
//              stream 0 / 1, the piece's partial
//   8-13       producers, each on its own items of 16 keys: K and V into the
//              swizzled operand layout. MX codes come from L2 into registers an
//              item ahead and are placed as f16; BF16 rows are copied by cp.async,
//              whose completion arrives on the tile's barrier by itself. With all
//              producers on one staged tile at a time a pair of blocks took 6k
//              cycles, 5k so (softmax 2.5-3.7k, products 1.3k).
//   14         TMEM allocation and MMA issue
//   15         page lookup, and the pages on their way to L2
// MX computes in f16 like the decode: K and V are payload x scale / 4, the
// query row times a power of two, P built 2^7 larger, so that what underflows is
// below 2^-32 of the row's largest. P is a hi + lo pair of V's type as in the
// decode (f16: 21 bits, bf16: 16) and takes two products: with one f16 an output
// left over from values of 4,000 that cancel missed 1e-3 + 2e-2 |out| by 15x.
//
// suffix_role. The decode's tiles (16 tokens of one sequence and kv head, all G
// query heads, m16n8k16) laid end to end; each warp takes an equal contiguous
// range, as the split-KV decode does, but leaves every piece as a partial for
// the join, which reads them anyway: no counters, no last-arriver merge. 16
// warps a CTA (MX) read 1.26 GB at 5.2 TB/s, 12 read it at 4.8 TB/s.
// Every wait is bounded in wall time; a timeout sets KLLM_ERR_TIMEOUT.
//
// Bound: the floor is HBM (each shared page once, each own page once) or, for
// many rows, the tensor core; what holds is each stream's chain softmax -> P V
// -> S -> softmax, some 5k cycles for a pair of blocks (with a P of one f16 4-5k,
// of which the products took 1.5-2k; they take twice that for P V now), and some
// 30 us of plan, first block, last block and join. Measured, 32 query heads on 8
// kv heads, d 128, MX, pages not in L2: 64 rows that share 8,192 tokens (93 MB)
// 60-64 us, 1.5 TB/s; 256 rows (34.8 GFLOP) 114 us, 305 TFLOP/s (with one f16
// 56 and 100); 8 rows that share 512 tokens 20.5 us.

#include "kllm_decode_tile.cuh"
#include "kllm_device.cuh"
#include "kllm_internal.h"
#include "kllm_umma.cuh"

#include <cfloat>
#include <math_constants.h>

namespace kllm {
namespace {

constexpr int kPRows = 128, kPKeys = 128;
constexpr int kUnitRows = 256;
constexpr int kPThreads = 16 * 32;
constexpr int kWarpProd = 8, kWarpMma = 14, kWarpLoad = 15;
constexpr int kPW = 6;                        // producer warps
// Registers: 512 threads launch with 128 each, all of an SM's. A softmax thread
// holds 128 scores (256 x 160 + 256 x 96); a suffix warp's MX tile takes the 128,
// its BF16 tile 184 (256 x 184 + 256 x 72).
constexpr int kRegsLaunch = 128;
constexpr int kPg = 4;                        // blocks whose page addresses are known
constexpr float kRaise = 8.f;                 // slack of the lazy reference maximum, log2
constexpr float kPShift = 7.f;                // f16 P is built 2^7 larger
constexpr uint64_t kPWaitNs = 200000000ull;

// Moves registers between warps 0 .. FIRST - 1 (HI a thread from now on) and
// the others (LO). All warps of a warpgroup have to execute the same setmaxnreg,
// so this stands before the roles split and FIRST is a multiple of four; what
// one side takes, the other gives up. True in the warps below FIRST.
template <int FIRST, int HI, int LO>
__device__ __forceinline__ bool split_registers(int warp)
{
	constexpr int rest = kPThreads / 32 - FIRST;
	static_assert(FIRST % 4 == 0 && rest % 4 == 0, "a warpgroup takes one setmaxnreg");
	static_assert(FIRST * HI + rest * LO <= kPThreads / 32 * kRegsLaunch, "more than the launch holds");
	static_assert(HI % 8 == 0 && LO % 8 == 0 && HI >= kRegsLaunch && LO <= kRegsLaunch, "inc and dec");
	if (warp < FIRST) {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(HI));
		return true;
	}
	asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(LO));
	return false;
}

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
	long long T;          // work steps of the prefixes
	long long N;          // suffix tiles, kv heads counted
	int W;                // CTAs that share the steps
	int n_prefix;         // CTAs set aside for them; the rest take suffixes
	int WS;               // warps that share the tiles
	int pad[9];
};
static_assert(sizeof(PHeader) == 64 && sizeof(PGroup) == 48, "workspace layout");

// ---- plan ------------------------------------------------------------------------

constexpr int kPlanThreads = 256;
// A CTA's time for n steps or for n tiles a warp, in ns, as measured on the
// whole chip: set-up, then the rate. They only balance the two parts: steps of
// 1,500 and 1,800 ns give 105 and 102 us for 256 rows of 8,192 shared tokens, 53
// and 55 us for 64 rows.
constexpr float kStepSetNs = 10500.f, kStepNsMx = 1500.f, kStepNsBf16 = 2700.f;
constexpr float kTileSetNs = 5000.f, kTileNs = 2500.f;
// Each further unit that a CTA works on (64 rows with 16 or 128 shared tokens:
// 54 us without this term, 36 with it).
constexpr float kPieceNs = 4500.f;

struct PlanSmem {
	long long w0[32], w1[32];
	int leader[KLLM_MAX_SEQS_LAUNCH];
	unsigned long long best;
	int units;
};

// Tokens of group g's prefix that are whole pages inside the table.
__device__ __forceinline__ int prefix_tokens(const kllm_prefix_args &a, int g)
{
	const int cap = a.max_blocks * a.block_size;
	return min(max(a.prefix_lens[g], 0), cap) / a.block_size * a.block_size;
}

// Exclusive sums of x and y over the block's threads, on top of run_x, run_y,
// which advance by the totals.
__device__ __forceinline__ void block_scan2(PlanSmem &sm, long long x, long long y, long long &ex,
					    long long &ey, long long &run_x, long long &run_y)
{
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	long long ix = x, iy = y;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const long long nx = __shfl_up_sync(0xffffffffu, ix, o);
		const long long ny = __shfl_up_sync(0xffffffffu, iy, o);
		if (lane >= o) {
			ix += nx;
			iy += ny;
		}
	}
	__syncthreads();
	if (lane == 31) {
		sm.w0[warp] = ix;
		sm.w1[warp] = iy;
	}
	__syncthreads();
	long long bx = lane < kPlanThreads / 32 ? sm.w0[lane] : 0, by = lane < kPlanThreads / 32 ? sm.w1[lane] : 0;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const long long nx = __shfl_up_sync(0xffffffffu, bx, o);
		const long long ny = __shfl_up_sync(0xffffffffu, by, o);
		if (lane >= o) {
			bx += nx;
			by += ny;
		}
	}
	const long long px = __shfl_sync(0xffffffffu, bx, max(warp - 1, 0));
	const long long py = __shfl_sync(0xffffffffu, by, max(warp - 1, 0));
	ex = run_x + (warp ? px : 0) + ix - x;
	ey = run_y + (warp ? py : 0) + iy - y;
	run_x += __shfl_sync(0xffffffffu, bx, 31);
	run_y += __shfl_sync(0xffffffffu, by, 31);
}

__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const kllm_prefix_args a)
{
	__shared__ PlanSmem sm;
	const int tid = threadIdx.x;
	const int S = a.num_seqs, NG = a.num_groups, bs = a.block_size;
	grid_launch_dependents();
	// groups out of order or out of range: nothing is shared (the result stays
	// right) and the call is flagged
	bool bad = false, too_long = false;
	for (int g = tid; g < NG; g += kPlanThreads) {
		const int b = a.group_starts[g], e = a.group_starts[g + 1];
		bad |= b < 0 || e < b || e > S;
		sm.leader[g] = 0x7fffffff;
	}
	if (tid == 0)
		sm.units = 0;
	bad = __syncthreads_or(bad);

	// ---- rows: group, suffix, exclusive sums of the suffixes' tiles --------------
	const int cap = a.max_blocks * bs;
	long long tiles = 0, none = 0;
	for (int base = 0; base < S; base += kPlanThreads) {
		const int s = base + tid;
		int n_tiles = 0;
		if (s < S) {
			const int len = a.seq_lens[s], L = min(max(len, 0), cap);
			too_long |= len > cap;
			int g = -1, P = 0;
			if (!bad && NG > 0) {
				int lo = 0, hi = NG - 1;        // the last group that starts at or before s
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
					// A row without the whole prefix may have pages of its own, the
					// prefix's whole pages included: all of it is suffix.
					if (P > 0 && L >= a.prefix_lens[lo]) {
						g = lo;
						atomicMin(&sm.leader[lo], s);
					} else {
						P = 0;
					}
				}
			}
			n_tiles = (L - P + kTile - 1) / kTile;
			a.row_group[s] = g;
			a.suf_start[s] = P / bs;
			a.suf_lens[s] = L - P;
		}
		long long et, en;
		block_scan2(sm, n_tiles, 0, et, en, tiles, none);
		if (s < S)
			a.tile_pre[s] = (int)et;
	}
	__syncthreads();                           // sm.leader is complete

	// ---- groups: exclusive sums of steps and partial rows ---------------------------
	PGroup *gr = static_cast<PGroup *>(a.groups);
	long long run_x = 0, run_r = 0;
	for (int base = 0; base < NG; base += kPlanThreads) {
		const int g = base + tid;
		PGroup p = {};
		long long x = 0, r = 0;
		if (g < NG) {
			p.row0 = a.group_starts[g];
			p.nseq = bad ? 0 : a.group_starts[g + 1] - p.row0;
			p.leader = sm.leader[g];
			const int rows = p.nseq * a.group;
			p.tiles = (rows + kUnitRows - 1) / kUnitRows;
			p.wgt = rows > kPRows ? 2 : 1;
			p.alloc = rows > kPRows ? rows : 2 * rows;
			if (p.leader != 0x7fffffff) {
				p.npages = prefix_tokens(a, g) / bs;
				const int ppb = kPKeys / bs;
				p.nblk = (p.npages + ppb - 1) / ppb;
				x = (long long)a.num_kv_heads * p.tiles * p.nblk * p.wgt;
				r = (long long)a.num_kv_heads * p.alloc;
				atomicAdd(&sm.units, a.num_kv_heads * p.tiles);
			}
		}
		block_scan2(sm, x, r, p.x0, p.r0, run_x, run_r);
		if (g < NG)
			gr[g] = p;
	}

	// ---- CTAs for each part: the split whose slower part is fastest -----------------
	const long long T = run_x, N = tiles * a.num_kv_heads;
	if (tid == 0)
		sm.best = ~0ull;
	__syncthreads();
	if (tid <= a.ctas) {
		const int n = tid;                         // CTAs for the prefixes
		const bool possible = (T > 0) == (n > 0) && (N == 0 || n < a.ctas);
		if (possible) {
			float t = 0.f;
			if (n > 0)
				t = kStepSetNs + (a.kv_dtype ? kStepNsMx : kStepNsBf16) * ceilf((float)T / (float)n) +
				    kPieceNs * (ceilf((float)sm.units / (float)n) - 1.f);
			if (N > 0)
				t = fmaxf(t, kTileSetNs + kTileNs * ceilf((float)N / (float)((a.ctas - n) * a.suf_warps)));
			atomicMin(&sm.best, ((unsigned long long)__float_as_uint(t) << 32) | (unsigned)n);
		}
	}
	__syncthreads();
	if (tid == 0) {
		PHeader *hd = static_cast<PHeader *>(a.header);
		const int n = (int)(sm.best & 0xffffffffull);
		const long long ws = (long long)(a.ctas - n) * a.suf_warps;
		hd->T = T;
		hd->N = N;
		hd->n_prefix = n;
		hd->W = (int)(T < n ? T : n);
		hd->WS = (int)(N < ws ? N : ws);
		a.tile_pre[S] = (int)tiles;
		if (bad && a.err)
			atomicOr(a.err, KLLM_ERR_LAYOUT_BIT);
	}
	if (too_long && a.err)
		atomicOr(a.err, KLLM_ERR_SEQ_TOO_LONG_BIT);
}

// ---- prefix ------------------------------------------------------------------------

template <int D, int KVT>
struct PG {
	static constexpr bool MX = KVT == 1;
	static constexpr int NH = D / 64;                     // 64-column halves
	static constexpr int HALF = kPRows * 128;             // bytes of one half tile
	static constexpr int TILE = NH * HALF;
	static constexpr int FILL = kPKeys / 16 * (MX ? 1 : 32);  // arrivals that fill a tile
	static constexpr int LPR = MX ? D / 16 : D / 8;       // 16-byte pieces of a row
};

template <int D, int KVT>
struct PrefixSmem {
	using G = PG<D, KVT>;
	uint8_t q[2][G::TILE];
	uint8_t k[2][G::TILE];
	uint8_t v[2][G::TILE];
	float qf[2][kPRows];                  // 2^-e of a solo piece's query rows, by piece parity
	unsigned long long pg[kPg][2][8];     // section addresses of a block's pages, 0: absent
	alignas(16) uint32_t key_ok[8][4];    // key masks of the last eight blocks
	uint64_t q_full, q_empty;
	uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
	uint64_t pg_full[kPg], pg_empty[kPg];
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

// a / b, in 32 bits where the values allow (a 64-bit division costs several
// times as much, and the pieces are found before the first load)
__device__ __forceinline__ long long div_steps(long long x, long long y)
{
	return (unsigned long long)(x | y) >> 32 ? x / y : (long long)((uint32_t)x / (uint32_t)y);
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
	const long long u = div_steps(x - G.x0, cost);
	const long long ux = G.x0 + u * cost;
	const long long end = min(xe, ux + cost);
	p.h = (int)div_steps(u, G.tiles);
	p.tile = (int)(u - (long long)p.h * G.tiles);
	p.b0 = (int)((x - ux) >> (G.wgt - 1));
	p.nb = (int)((end - ux) >> (G.wgt - 1)) - p.b0;
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

// Two E4M3 codes in bytes 0 and 2 -> f16x2 of value x 2^-8: the bits s.eeee.mmm
// placed as s.0eeee.mmm0000000, exact for every code (subnormals land on f16
// subnormals, 0x7F / 0xFF give +-480 as the format's decoder has it,
// userspace/compute/mx_dequant.h:30-55). Shifted by 7 the sign sits in bit 14;
// adding that bit moves it to bit 15. Integer instructions, because the hardware
// conversion shares its unit with the softmax's exponentials.
__device__ __forceinline__ uint32_t place_pair(uint32_t x)
{
	const uint32_t h = x << 7;
	return h + (h & 0x40004000u);
}

// Sixteen codes (two scale blocks, their codes in bytes 0 and 2 of sc) of a row
// -> 16 f16 values payload x scale / 4, the second block's eight in `hi`: the
// scale is placed and multiplied by 2^14, which makes it x 64, and x 64 x 2^-8
// is / 4.
__device__ __forceinline__ void mx16_to_f16(uint2 wl, uint2 wh, uint32_t sc, uint4 &lo, uint4 &hi)
{
	const uint32_t s = f16x2_mul(place_pair(sc), 0x74007400u);
	const uint32_t s0 = __byte_perm(s, 0u, 0x1010u), s1 = __byte_perm(s, 0u, 0x3232u);
	lo.x = f16x2_mul(place_pair(__byte_perm(wl.x, 0u, 0x4140u)), s0);
	lo.y = f16x2_mul(place_pair(__byte_perm(wl.x, 0u, 0x4342u)), s0);
	lo.z = f16x2_mul(place_pair(__byte_perm(wl.y, 0u, 0x4140u)), s0);
	lo.w = f16x2_mul(place_pair(__byte_perm(wl.y, 0u, 0x4342u)), s0);
	hi.x = f16x2_mul(place_pair(__byte_perm(wh.x, 0u, 0x4140u)), s1);
	hi.y = f16x2_mul(place_pair(__byte_perm(wh.x, 0u, 0x4342u)), s1);
	hi.z = f16x2_mul(place_pair(__byte_perm(wh.y, 0u, 0x4140u)), s1);
	hi.w = f16x2_mul(place_pair(__byte_perm(wh.y, 0u, 0x4342u)), s1);
}

__device__ __forceinline__ void cp_async16(void *dst, const void *src)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
		     :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void bulk_prefetch_l2(const void *src, uint32_t bytes)
{
	asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit()
{
	asm volatile("cp.async.commit_group;" ::: "memory");
}
// One arrival on `bar` (counted at its initialisation) once this thread's copies
// so far are done.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar)
{
	asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
	asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// The 128 scores of this thread's TMEM lane, all loads in flight; keys whose bit
// in mask is clear read as -inf.
__device__ __forceinline__ void load_scores(uint32_t taddr, bool full, const uint32_t *mask,
					    uint32_t (&r)[8][16])
{
#pragma unroll
	for (int q = 0; q < 8; ++q)
		tmem_ld16_nowait(taddr + 16 * q, r[q]);
#pragma unroll
	for (int q = 0; q < 8; ++q)
		asm volatile("tcgen05.wait::ld.sync.aligned;"
			     : "+r"(r[q][0]), "+r"(r[q][1]), "+r"(r[q][2]), "+r"(r[q][3]),
			       "+r"(r[q][4]), "+r"(r[q][5]), "+r"(r[q][6]), "+r"(r[q][7]),
			       "+r"(r[q][8]), "+r"(r[q][9]), "+r"(r[q][10]), "+r"(r[q][11]),
			       "+r"(r[q][12]), "+r"(r[q][13]), "+r"(r[q][14]), "+r"(r[q][15])
			     :: "memory");
	if (!full)
#pragma unroll
		for (int w = 0; w < 4; ++w) {
			const uint32_t m = mask[w];
#pragma unroll
			for (int i = 0; i < 32; ++i)
				if (!((m >> i) & 1u))
					r[2 * w + (i >> 4)][i & 15] = 0xFF800000u;
		}
}

// One 128-key block of one row: S in the TMEM columns of tS -> P over them, 16
// columns for 16 keys: 8 of hi pairs, 8 of lo pairs. The row's block
// maximum is known before any P is written, so raising the reference rescales
// only O and l. Warp-collective; branches around TMEM accesses are
// warp-uniform. Returns through m_ref and l_sum. Keys 0-63 are announced on
// p_half as soon as they are written, so their products can start. The scores
// stay in registers between the maximum and the exponentials: read a second
// time they cost 0.9k of 3.3k cycles a block in TMEM round trips.
template <int D, int KVT>
__device__ __forceinline__ void softmax_rows(uint32_t tS, uint32_t tO, const uint32_t *mask,
					     float sl2, bool o_live, float &m_ref, float &l_sum,
					     uint64_t *p_half)
{
	constexpr bool MX = KVT == 1;
	constexpr float shift = MX ? kPShift : 0.f;
	const bool full = (mask[0] & mask[1] & mask[2] & mask[3]) == 0xFFFFFFFFu;  // same in all lanes
	uint32_t r[8][16];
	load_scores(tS, full, mask, r);
	float m4[4];
#pragma unroll
	for (int i = 0; i < 4; ++i)
		m4[i] = __uint_as_float(r[0][i]);
#pragma unroll
	for (int k = 4; k < 128; ++k)
		m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(r[k >> 4][k & 15]));
	const float gl = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
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
	// two keys an instruction where the hardware has it
	const uint64_t sl2_2 = pack2(sl2, sl2), moff_2 = pack2(moff, moff);
	float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int c = 0; c < 128; c += 16) {
		float w[16];
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			const int k = c + 2 * i;
			float x0, x1;
			unpack2(fma2(pack2(__uint_as_float(r[k >> 4][k & 15]),
					   __uint_as_float(r[k >> 4][(k & 15) + 1])), sl2_2, moff_2), x0, x1);
			const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
			if constexpr (MX) {
				float &s0 = sum[2 * (i & 1)], &s1 = sum[2 * (i & 1) + 1];
				unpack2(add2(pack2(s0, s1), pack2(p0, p1)), s0, s1);
				// hi: P cut to f16's 11 bits; lo: what that leaves off
				const float n0 = __uint_as_float((__float_as_uint(p0) & 0xFFFFE000u) | 0x80000000u);
				const float n1 = __uint_as_float((__float_as_uint(p1) & 0xFFFFE000u) | 0x80000000u);
				float l0, l1;
				unpack2(add2(pack2(p0, p1), pack2(n0, n1)), l0, l1);
				w[i] = __uint_as_float(pack_f16x2_rz(p0, p1));
				w[8 + i] = __uint_as_float(pack_f16x2(l0, l1));
			} else {
				sum[i & 3] += p0 + p1;
				const uint32_t hi = pack_bf16x2(p0, p1);
				w[i] = __uint_as_float(hi);
				w[8 + i] = __uint_as_float(pack_bf16x2(p0 - __uint_as_float(hi << 16),
								       p1 - __uint_as_float(hi & 0xFFFF0000u)));
			}
		}
		tmem_st16_nowait(tS + c, w);
		if (c + 16 == 64) {
			tmem_wait_st();
			tc_fence_before();
			mbar_arrive(p_half);
		}
	}
	tmem_wait_st();
	l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A warp's 32 query rows into the operand tile: bf16 as they are, or for MX f16
// after a power of two that puts a row's largest element in [2^14, 2^15);
// returns the inverse of that factor for row `lane`. off: where row `lane`
// starts in q, in elements (-1: a row of zeros). neg: the rows change sign, for a
// softmax scale below 0 (the softmax takes |scale|: absent keys are -inf before
// it, and the largest product is the largest score). Copied in by whole lines, then
// converted in place, a row a lane (the swizzle spreads eight rows over all
// banks). The loops stay rolled: this code runs once a piece, and unrolled it
// spent 10k cycles on instruction fetches alone.
template <int D, int KVT>
__device__ __forceinline__ float load_queries(uint8_t *tile, int r0, int lane, const void *q,
					      long long off, bool neg)
{
	constexpr int LPR = D / 8, RPP = 32 / LPR;
	const int l = lane % LPR, sub = lane / LPR;
#pragma unroll 2
	for (int i = 0; i < 32; i += RPP) {
		const long long o = __shfl_sync(0xffffffffu, off, i + sub);
		uint8_t *dst = tile + (l >> 3) * (kPRows * 128) + swz(r0 + i + sub, l & 7);
		if (o >= 0)
			cp_async16(dst, static_cast<const uint8_t *>(q) + o * 2 + l * 16);
		else
			*reinterpret_cast<uint4 *>(dst) = make_uint4(0u, 0u, 0u, 0u);
	}
	cp_async_commit();
	cp_async_wait<0>();
	__syncwarp();
	const int r = r0 + lane;
	if constexpr (KVT == 0) {
		if (neg)
#pragma unroll 1
			for (int c = 0; c < LPR; ++c) {
				uint4 *p = reinterpret_cast<uint4 *>(tile + (c >> 3) * (kPRows * 128) + swz(r, c & 7));
				const uint4 w = *p;
				*p = make_uint4(w.x ^ 0x80008000u, w.y ^ 0x80008000u, w.z ^ 0x80008000u, w.w ^ 0x80008000u);
			}
		return 1.f;
	}
	uint32_t mb = 0u;                                // bf16 magnitudes order as integers
#pragma unroll 4
	for (int c = 0; c < LPR; ++c) {
		const uint4 w = *reinterpret_cast<const uint4 *>(tile + (c >> 3) * (kPRows * 128) + swz(r, c & 7));
		const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
		for (int i = 0; i < 4; ++i)
			mb = max(mb, max((ww[i] << 16) & 0x7FFF0000u, ww[i] & 0x7FFF0000u));
	}
	const int E = mb ? (int)(mb >> 23) - 127 : 0;
	const int e = min(max(14 - E, -100), 100);
	const float f = __uint_as_float(((uint32_t)(e + 127) << 23) | (neg ? 0x80000000u : 0u));
#pragma unroll 2
	for (int c = 0; c < LPR; ++c) {
		uint4 *p = reinterpret_cast<uint4 *>(tile + (c >> 3) * (kPRows * 128) + swz(r, c & 7));
		const uint4 w = *p;
		uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
		for (int i = 0; i < 4; ++i)
			ww[i] = pack_f16x2(__uint_as_float(ww[i] << 16) * f,
					   __uint_as_float(ww[i] & 0xFFFF0000u) * f);
		*p = make_uint4(ww[0], ww[1], ww[2], ww[3]);
	}
	return __uint_as_float((uint32_t)(127 - e) << 23);
}

template <int D, int KVT>
__device__ __forceinline__ void init_prefix(PrefixSmem<D, KVT> &sm)
{
	mbar_init(&sm.q_full, 256);
	mbar_init(&sm.q_empty, 1);
	for (int i = 0; i < 2; ++i) {
		mbar_init(&sm.k_full[i], PG<D, KVT>::FILL);
		mbar_init(&sm.k_empty[i], 1);
		mbar_init(&sm.v_full[i], PG<D, KVT>::FILL);
		mbar_init(&sm.v_empty[i], 1);
		mbar_init(&sm.s_full[i], 1);
		mbar_init(&sm.p_half[i], 128);
		mbar_init(&sm.p_full[i], 128);
		mbar_init(&sm.o_full[i], 1);
	}
	for (int i = 0; i < kPg; ++i) {
		mbar_init(&sm.pg_full[i], 1);
		mbar_init(&sm.pg_empty[i], kPW);
	}
	mbar_init(&sm.drain, 1);
	sm.abort = 0;
	fence_mbar_init();
}

// CTA `cta` of the W that share the T steps of the prefixes. The barriers are
// initialised; every thread of the CTA calls it.
template <int D, int KVT>
__device__ __forceinline__ void prefix_role(const kllm_prefix_args &a, PrefixSmem<D, KVT> &sm, int cta,
					    long long T, int W)
{
	using G = PG<D, KVT>;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
	long long x = div_steps(cta * T, W);
	const long long xe = div_steps((cta + 1) * T, W);
	const int bs = a.block_size, ppb = kPKeys / bs;
	const int sec = bs * (G::MX ? D * 9 / 8 : D * 2);
	auto wait = [&](uint64_t *bar, uint32_t parity) { return p_wait(&sm.abort, bar, parity, a.err); };

	if (split_registers<kWarpProd, 160, 96>(warp)) {
		// ================= softmax of stream t ========================================
		const int t = warp >> 2, rr = (warp & 3) * 32 + lane;
		const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
		const uint32_t tS = lane_base + col_s(t), tO = lane_base + col_o(t);
		int kf = 0, n_s = 0, n_o = 0, np = 0;        // K fills, S tiles, O tiles, pieces
		bool ok = true;
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			const int qt = p.solo ? 0 : t;
			const int row = qt * kPRows + rr;            // row of the unit
			if (p.nb <= 0) {                             // a share without a whole block
				if (row < p.rows) {
					const long long e = p.slot + (p.solo && t == 1 ? p.rows : 0) + row;
					a.pm[e] = -CUDART_INF_F;
					a.pl[e] = 0.f;
				}
				continue;
			}
			const bool warp_live = qt * kPRows + (warp & 3) * 32 < p.rows;
			// ---- this row's query (a solo piece has one tile: stream 0 loads it) -------
			// Rows of sequences that do not take part are computed too; nothing
			// reads them.
			if (np > 0 && !__all_sync(0xffffffffu, wait(&sm.q_empty, (uint32_t)((np - 1) & 1)))) {
				ok = false;
				break;
			}
			float qf = 1.f;
			if (!p.solo || t == 0) {
				const int rh = p.tile * kUnitRows + row;         // row of the kv head
				const int seq = p.row0 + rh / a.group, hh = rh % a.group;
				const long long off = row < p.rows
				    ? ((long long)seq * a.num_heads + (long long)p.h * a.group + hh) * D : -1;
				qf = load_queries<D, KVT>(sm.q[qt], (warp & 3) * 32, lane, a.q, off,
							  a.scale_log2 < 0.f);
				if (G::MX && p.solo)
					sm.qf[np & 1][rr] = qf;
				fence_async_smem();
			}
			mbar_arrive(&sm.q_full);
			float m_ref = -CUDART_INF_F, l_sum = 0.f, sl2 = 0.f;
			bool first = true;
			for (int j = p.solo ? t : 0; j < p.nb; j += p.solo ? 2 : 1, ++n_s) {
				if (!__all_sync(0xffffffffu, wait(&sm.s_full[t], (uint32_t)(n_s & 1)))) {
					ok = false;
					break;
				}
				tc_fence_after();
				if (first) {
					sl2 = fabsf(a.scale_log2) *
					      (G::MX ? (p.solo && t ? sm.qf[np & 1][rr] : qf) * KLLM_MX_DEC_UNBIAS
						     : 1.f);
					// scale 0: the least factor that keeps an absent key at -inf
					if (sl2 < FLT_MIN)
						sl2 = FLT_MIN;
				}
				if (warp_live)
					softmax_rows<D, KVT>(tS, tO, sm.key_ok[(kf + j) & 7], sl2, !first, m_ref,
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
		// An item is 16 keys of K or V of one block (never more than one page), 16
		// items a block, and each warp takes every kPW-th on its own: with all
		// warps on one tile at a time, half of the time went into its barriers.
		constexpr int RP = 32 / G::LPR, NP = 16 / RP;      // rows a pass, passes of an item
		const int pw = warp - kWarpProd, l = lane % G::LPR, sub = lane / G::LPR;
		// (key / 16) x inv16 / 256 = key / bs for keys below 128 and the block sizes
		// 16, 32 .. 128
		const int inv16 = 256 / (bs >> 4) + 1;
		int gb0 = 0;                                 // blocks of the pieces before
		bool ok = true;
		auto wait_warp = [&](uint64_t *bar, uint32_t parity) {
			return __all_sync(0xffffffffu, wait(bar, parity));
		};
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			const int n_it = p.nb * 16;
			int cur = -1;                            // block whose addresses are here
			// this lane's first byte of item i; 0 when its page is absent. The first
			// item of a block waits for its addresses, the last one frees them.
			auto locate = [&](int i, int &row) {
				const int j = i >> 4, slot = (gb0 + j) % kPg, key = (i & 7) * 16;
				if (j != cur) {
					ok = ok && wait_warp(&sm.pg_full[slot], (uint32_t)(((gb0 + j) / kPg) & 1));
					cur = j;
				}
				const int page = ((key >> 4) * inv16) >> 8;
				row = key - page * bs + sub;
				const unsigned long long at = ok ? sm.pg[slot][(i >> 3) & 1][page] : 0ull;
				__syncwarp();
				if (((i + kPW) >> 4) != j && lane == 0)
					mbar_arrive(&sm.pg_empty[slot]);
				return at;
			};
			auto full_bar = [&](int i) {
				const int b = (gb0 + (i >> 4)) & 1;
				return (i & 8) ? &sm.v_full[b] : &sm.k_full[b];
			};
			auto tile_of = [&](int i) {
				const int b = (gb0 + (i >> 4)) & 1;
				return (i & 8) ? sm.v[b] : sm.k[b];
			};
			auto empty_bar = [&](int i) {
				const int b = (gb0 + (i >> 4)) & 1;
				return (i & 8) ? &sm.v_empty[b] : &sm.k_empty[b];
			};
			if constexpr (G::MX) {
				// an item's codes and scales go to registers while the item before is
				// placed
				uint4 cw[NP], nw[NP];
				uint32_t cs[NP], ns[NP];
				auto fetch = [&](int i, uint4 (&w)[NP], uint32_t (&sc)[NP]) {
					int row;
					const unsigned long long at = locate(i, row);
					const uint8_t *pay = reinterpret_cast<const uint8_t *>(at) + row * D + l * 16;
					const uint8_t *scl = reinterpret_cast<const uint8_t *>(at) + bs * D + row * (D / 8) + 2 * l;
#pragma unroll
					for (int u = 0; u < NP; ++u) {
						w[u] = make_uint4(0u, 0u, 0u, 0u);
						sc[u] = 0u;
						if (at) {
							w[u] = __ldcg(reinterpret_cast<const uint4 *>(pay + u * RP * D));
							sc[u] = __ldcg(reinterpret_cast<const unsigned short *>(scl + u * RP * (D / 8)));
						}
					}
				};
				// Lanes of the upper 64 columns store their second chunk first, so that
				// the eight lanes of a row never store to one bank.
				const bool swap = l >= 4;
				const uint32_t pick = swap ? 0x4041u : 0x4140u;
				const int c0 = (2 * l) & 7, half = (l >> 2) * G::HALF;
				auto place = [&](int i, const uint4 (&w)[NP], const uint32_t (&sc)[NP]) {
					const int cnt = gb0 + (i >> 4);
					ok = ok && (cnt < 2 || wait_warp(empty_bar(i), (uint32_t)(((cnt >> 1) - 1) & 1)));
					if (!ok)
						return;
					uint8_t *dst = tile_of(i) + half;
#pragma unroll
					for (int u = 0; u < NP; ++u) {
						const uint2 wa = make_uint2(w[u].x, w[u].y), wb = make_uint2(w[u].z, w[u].w);
						uint4 lo, hi;
						mx16_to_f16(swap ? wb : wa, swap ? wa : wb, __byte_perm(sc[u], 0u, pick), lo, hi);
						const int row = (i & 7) * 16 + u * RP + sub;
						*reinterpret_cast<uint4 *>(dst + swz(row, c0 + (swap ? 1 : 0))) = lo;
						*reinterpret_cast<uint4 *>(dst + swz(row, c0 + (swap ? 0 : 1))) = hi;
					}
					fence_async_smem();
					__syncwarp();
					if (lane == 0)
						mbar_arrive(full_bar(i));
				};
				fetch(pw, cw, cs);
#pragma unroll 1
				for (int i = pw; i < n_it && ok; i += 2 * kPW) {
					if (i + kPW < n_it)
						fetch(i + kPW, nw, ns);
					place(i, cw, cs);
					if (i + 2 * kPW < n_it)
						fetch(i + 2 * kPW, cw, cs);
					if (i + kPW < n_it && ok)
						place(i + kPW, nw, ns);
				}
			} else {
				// copies run as far ahead as buffers are free; their completion arrives
				// on the barrier by itself, and the MMA warp has the proxy fence
				for (int i = pw; i < n_it; i += kPW) {
					int row;
					const unsigned long long at = locate(i, row);
					const int cnt = gb0 + (i >> 4);
					ok = ok && (cnt < 2 || wait_warp(empty_bar(i), (uint32_t)(((cnt >> 1) - 1) & 1)));
					if (!ok)
						break;
					uint8_t *dst = tile_of(i) + (l >> 3) * G::HALF;
					const uint8_t *src = reinterpret_cast<const uint8_t *>(at) + row * (D * 2) + l * 16;
#pragma unroll
					for (int u = 0; u < NP; ++u) {
						uint8_t *o = dst + swz((i & 7) * 16 + u * RP + sub, l & 7);
						if (at)
							cp_async16(o, src + u * RP * (D * 2));
						else
							*reinterpret_cast<uint4 *>(o) = make_uint4(0u, 0u, 0u, 0u);
					}
					if (at)
						cp_async_arrive(full_bar(i));
					else
						mbar_arrive(full_bar(i));
				}
				cp_async_commit();
				cp_async_wait<0>();
			}
			gb0 += p.nb;
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
		const uint64_t dk1 = umma_desc(smem_u32(sm.k[1]), 16u, 1024u);
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
			const int b = kf & 1, round = kf >> 1;
			if (!wait_all(&sm.k_full[b], (uint32_t)(round & 1)))
				return false;
			if constexpr (!G::MX)
				fence_async_smem();
			return true;
		};
		auto free_k = [&]() {
			commit(&sm.k_empty[kf & 1]);
			++kf;
		};
		auto issue_s = [&](int t, int qt) {
			const uint64_t dq = qt ? dq1 : dq0, dk = (kf & 1) ? dk1 : dk0;
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
#pragma unroll
				for (int lo = 0; lo < 2; ++lo)
					if (leader)
						umma_f16_ts(d, pa + 16u * g + 8u * lo, dv + (uint64_t)((g * 2048) >> 4),
							    id_pv, (first && g == 0 && lo == 0) ? 0u : 1u);
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
				if constexpr (!G::MX)
					fence_async_smem();
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
	} else if (warp == kWarpLoad) {
		// ================= page lookup and raw copies ========================================
		int gb = 0;                                  // blocks posted
		bool ok = true;
		while (x < xe && ok) {
			const Piece p = next_piece(a, x, xe, cta);
			if (p.nb <= 0)
				continue;
			const DevEntry *tb = static_cast<const DevEntry *>(a.table) +
					     (size_t)p.leader * a.max_blocks;
			const unsigned long long off = a.layer_off + (unsigned long long)p.h * sec;
			auto load = [&](int b) {
				DevEntry e;
				const int page = b * ppb + lane;
				e.k = e.v = 0ull;
				e.valid = 0;
				if (b < p.b0 + p.nb && lane < ppb && page < p.npages) {
					e.k = __ldg(&tb[page].k);
					e.v = __ldg(&tb[page].v);
					e.valid = __ldg(&tb[page].valid);
				}
				return e;
			};
			// this lane's page of a block as section addresses (valid 0: absent)
			auto check = [&](DevEntry &e) {
				const bool present = e.valid && e.k != 0ull;
				const bool aligned = ((e.k | e.v) & 15ull) == 0ull;
				if (present && !aligned && a.err)
					atomicOr(a.err, 0x2u);
				bool here = present && aligned;
				e.k += off;
				e.v += off;
				if (here && !(in_arenas(a.arenas, e.k, sec) && in_arenas(a.arenas, e.v, sec))) {
					here = false;
					if (a.err)
						atomicOr(a.err, KLLM_ERR_PAGE_RANGE_BIT);
				}
				e.valid = here ? 1 : 0;
			};
			DevEntry cur = load(p.b0), nxt = load(p.b0 + 1);
			check(cur);
			for (int j = 0; j < p.nb && ok; ++j) {
				const DevEntry e = cur;
				const uint32_t mask = __ballot_sync(0xffffffffu, e.valid);
				const int slot = gb % kPg;
				if (gb >= kPg)
					ok = __all_sync(0xffffffffu, wait(&sm.pg_empty[slot], (uint32_t)((gb / kPg - 1) & 1)));
				if (!ok)
					break;
				if (lane < 8) {
					sm.pg[slot][0][lane] = e.valid ? e.k : 0ull;
					sm.pg[slot][1][lane] = e.valid ? e.v : 0ull;
				}
				if (lane < 4) {                        // keys 32 lane .. 32 lane + 31
					uint32_t m = 0;
#pragma unroll
					for (int i = 0; i < 2; ++i) {
						const int page = (32 * lane + 16 * i) / bs;
						if (page < ppb && ((mask >> page) & 1u))
							m |= 0xFFFFu << (16 * i);
					}
					sm.key_ok[gb & 7][lane] = m;
				}
				__syncwarp();
				if (lane == 0)
					mbar_arrive(&sm.pg_full[slot]);
				++gb;
				cur = nxt;
				nxt = load(p.b0 + j + 2);
				check(cur);
				// On its way to L2 up to five blocks ahead of the producers; not the
				// second block, whose address they already wait for (the two requests
				// of 16 pages take the warp 1.2k cycles).
				if (j > 0 && cur.valid) {
					bulk_prefetch_l2(reinterpret_cast<const void *>(cur.k), (uint32_t)sec);
					bulk_prefetch_l2(reinterpret_cast<const void *>(cur.v), (uint32_t)sec);
				}
			}
		}
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

// ---- suffixes --------------------------------------------------------------------------

// Warps of a suffix CTA that work (the BF16 tile needs more registers).
template <int KVT>
struct SW {
	static constexpr int N = KVT == 1 ? 16 : 8;
};

struct SufSeg {
	int s, h, j, ts;      // sequence, kv head, tile of its suffix, tiles of it
};

// The sequence, head and tile of step x of the tiles laid end to end
// (sequence-major, then kv head); pre: exclusive sums of tiles per sequence.
__device__ __forceinline__ SufSeg locate_suffix(const int *pre, int S, int H, long long x)
{
	int lo = 0, hi = S - 1;
	while (lo < hi) {
		const int mid = (lo + hi + 1) >> 1;
		if ((long long)pre[mid] * H <= x)
			lo = mid;
		else
			hi = mid - 1;
	}
	SufSeg c;
	c.s = lo;
	c.ts = pre[lo + 1] - pre[lo];
	const int rel = (int)(x - (long long)pre[lo] * H);   // below ts x H: 32 bits
	c.h = rel / c.ts;
	c.j = rel - c.h * c.ts;
	return c;
}

// Tiles j0 .. j1 - 1 of one (sequence, kv head) by a warp, exactly, in fp32
// with plain loads: for pieces whose tile loop was not finite because a page
// holds payload 0x7F / 0xFF (which the hardware conversion reads as NaN). No
// writer emits those codes, but pages that arrive from a store are raw bytes.
template <int D>
__device__ __noinline__ void suffix_exact(const kllm_prefix_args &a, int s, int h, int j0, int j1,
					  float sl2, float *xm, float *xl, float *xo)
{
	constexpr int NV = D / 32;
	const int lane = threadIdx.x & 31, bs = a.block_size;
	const size_t sec = (size_t)bs * D * 9 / 8;
	for (int hh = 0; hh < a.group; ++hh) {
		const uint16_t *qp = static_cast<const uint16_t *>(a.q) +
				     ((size_t)s * a.num_heads + (size_t)h * a.group + hh) * D + lane * NV;
		float q[NV], o[NV], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			q[i] = __uint_as_float((uint32_t)qp[i] << 16);
			o[i] = 0.f;
		}
		const int t1 = min(j1 * kTile, a.suf_lens[s]);
		for (int t = j0 * kTile; t < t1; ++t) {
			const int page = a.suf_start[s] + t / bs, r = t % bs;
			const DevEntry *e = static_cast<const DevEntry *>(a.table) + (size_t)s * a.max_blocks + page;
			const unsigned long long off = a.layer_off + (unsigned long long)h * sec;
			if (!e->valid || !e->k || ((e->k | e->v) & 15ull) ||
			    !(in_arenas(a.arenas, e->k + off, sec) && in_arenas(a.arenas, e->v + off, sec)))
				continue;                        // skipped by the tile loop as well
			const uint8_t *kb = reinterpret_cast<const uint8_t *>(e->k + off);
			const uint8_t *vb = reinterpret_cast<const uint8_t *>(e->v + off);
			const size_t so = (size_t)bs * D + (size_t)r * (D / 8) + lane * NV / 8;
			const float ksc = e4m3_ref_to_f32(kb[so]), vsc = e4m3_ref_to_f32(vb[so]);
			float dot = 0.f;
#pragma unroll
			for (int i = 0; i < NV; ++i)
				dot = fmaf(q[i], e4m3_ref_to_f32(kb[(size_t)r * D + lane * NV + i]) * ksc, dot);
#pragma unroll
			for (int w = 16; w; w >>= 1)
				dot += __shfl_xor_sync(0xffffffffu, dot, w);
			const float x = dot * sl2, mn = fmaxf(m, x);
			const float f = exp2f(m - mn), pw = exp2f(x - mn);
			l = fmaf(l, f, pw);
#pragma unroll
			for (int i = 0; i < NV; ++i)
				o[i] = fmaf(o[i], f, pw * e4m3_ref_to_f32(vb[(size_t)r * D + lane * NV + i]) * vsc);
			m = mn;
		}
		// the join multiplies MX values by what the tile loop leaves off
#pragma unroll
		for (int i = 0; i < NV; ++i)
			xo[(size_t)hh * D + lane * NV + i] = o[i] * (1.f / KLLM_MX_DEC_UNBIAS);
		if (lane == 0) {
			xm[hh] = m;
			xl[hh] = l;
		}
	}
}

// rows whose tile sums a suffix CTA keeps in shared memory; more are read from L2
constexpr int kSufSeqs = 2040;

template <int D, int KVT>
struct SufLayout {
	using Gm = Geom<D, KVT>;
	static constexpr int NW = SW<KVT>::N, NST = 3;
	static constexpr size_t ring = 0, bar = (size_t)NW * NST * Gm::STAGE, meta = bar + 8 * NW * NST;
	static constexpr size_t lut = meta + 4 * NW * NST, pre = lut + 4 * 256;
	static constexpr size_t total = pre + 4 * (kSufSeqs + 1);
};

// CTA `cta` of those that share the N tiles of the suffixes among WS warps.
// smem: SufLayout bytes, 128-byte aligned; its barriers are initialised here.
template <int D, int KVT>
__device__ __forceinline__ void suffix_role(const kllm_prefix_args &a, uint8_t *smem, int cta, long long N,
					    int WS)
{
	using Gm = Geom<D, KVT>;
	using Lay = SufLayout<D, KVT>;
	constexpr int NW = Lay::NW, NST = Lay::NST;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const int S = a.num_seqs, H = a.num_kv_heads, tpp = a.block_size / kTile;
	uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Lay::bar);
	int *meta = reinterpret_cast<int *>(smem + Lay::meta);
	uint32_t *lut = reinterpret_cast<uint32_t *>(smem + Lay::lut);
	int *spre = reinterpret_cast<int *>(smem + Lay::pre);
	if (cta * NW >= WS)
		return;                                    // uniform over the CTA
	const bool local = S <= kSufSeqs;
	if (local)
		for (int i = tid; i <= S; i += kPThreads)
			spre[i] = a.tile_pre[i];
	if constexpr (Gm::MX)
		for (int i = tid; i < 256; i += kPThreads)
			lut[i] = mx_scale_lut_entry_f16((uint32_t)i);
	if (warp < NW && lane == 0) {
		for (int i = 0; i < NST; ++i)
			mbar_init(&bars[warp * NST + i], 1);
		fence_mbar_init();
	}
	__syncthreads();
	if constexpr (!Gm::MX)
		if (!split_registers<NW, 184, 72>(warp))
			return;
	const int *pre = local ? spre : a.tile_pre;
	const int w = cta * NW + warp;
	if (w >= WS)
		return;
	const long long xa = div_steps(w * N, WS);
	const int n = (int)(div_steps((w + 1) * N, WS) - xa);
	uint8_t *ring = smem + Lay::ring + (size_t)warp * NST * Gm::STAGE;
	uint64_t *bar = bars + warp * NST;
	int *ntoks = meta + warp * NST;
	const size_t sec = Gm::MX ? (size_t)a.block_size * D * 9 / 8 : (size_t)a.block_size * D * 2;

	// block-table entries of 32 consecutive tiles, one a lane: loaded a batch
	// ahead (raw), turned into section addresses when their turn comes
	unsigned long long ck = 0, cv = 0, nk, nv;
	int cvalid = 0, cpack = 0, nvalid, npack;
	auto load = [&](int base, unsigned long long &ek, unsigned long long &ev, int &valid, int &pack) {
		const int pos = base + lane;
		ek = ev = 0ull;
		valid = pack = 0;
		if (pos < n) {
			const SufSeg c = locate_suffix(pre, S, H, xa + pos);
			const int ntok = min(a.suf_lens[c.s] - c.j * kTile, kTile);
			const int page = c.j / tpp, sub = c.j - page * tpp;
			const DevEntry *e = static_cast<const DevEntry *>(a.table) +
					    (size_t)c.s * a.max_blocks + a.suf_start[c.s] + page;
			ek = __ldg(&e->k);
			ev = __ldg(&e->v);
			valid = __ldg(&e->valid);
			pack = ntok | (sub << 8) | (c.h << 16);
		}
	};
	auto finish = [&]() {
		const int ntok = cpack & 0xFF, sub = (cpack >> 8) & 0xFF, h = cpack >> 16;
		const bool present = cvalid && ck != 0ull, aligned = ((ck | cv) & 15ull) == 0ull;
		if (present && !aligned && a.err)
			atomicOr(a.err, 0x2u);
		bool ok = present && aligned && ntok > 0;
		const unsigned long long off = a.layer_off + (unsigned long long)h * sec;
		if (ok && !(in_arenas(a.arenas, ck + off, sec) && in_arenas(a.arenas, cv + off, sec))) {
			ok = false;
			if (a.err)
				atomicOr(a.err, KLLM_ERR_PAGE_RANGE_BIT);
		}
		ck += off;
		cv += off;
		cpack = (ok ? ntok : 0) | (sub << 8);
	};
	load(0, ck, cv, cvalid, cpack);
	load(32, nk, nv, nvalid, npack);
	finish();
	int pb = 0;
	auto issue = [&](int pos) {
		int bi = pos - pb;
		if (bi >= 32) {
			ck = nk;
			cv = nv;
			cvalid = nvalid;
			cpack = npack;
			finish();
			pb += 32;
			bi -= 32;
			load(pb + 32, nk, nv, nvalid, npack);
		}
		const unsigned long long ek = __shfl_sync(0xffffffffu, ck, bi);
		const unsigned long long ev = __shfl_sync(0xffffffffu, cv, bi);
		const int pack = __shfl_sync(0xffffffffu, cpack, bi);
		if (lane == 0) {
			const int st = pos % NST, ntok = pack & 0xFF, sub = pack >> 8;
			ntoks[st] = ntok;
			if (ntok) {
				const uint64_t policy = l2_evict_first_policy();
				mbar_arrive_expect_tx(&bar[st], Gm::STAGE);
				uint8_t *dK = ring + (size_t)st * Gm::STAGE, *dV = dK + Gm::KV;
				const uint8_t *sK = reinterpret_cast<const uint8_t *>(ek);
				const uint8_t *sV = reinterpret_cast<const uint8_t *>(ev);
				if (Gm::MX && tpp == 1) {       // payload and scales in one run
					bulk_g2s_stream(dK, sK, Gm::KV, &bar[st], policy);
					bulk_g2s_stream(dV, sV, Gm::KV, &bar[st], policy);
				} else {
					bulk_g2s_stream(dK, sK + (size_t)sub * Gm::PAY, Gm::PAY, &bar[st], policy);
					bulk_g2s_stream(dV, sV + (size_t)sub * Gm::PAY, Gm::PAY, &bar[st], policy);
				}
				if (Gm::MX && tpp > 1) {
					const size_t so = (size_t)a.block_size * D + (size_t)sub * Gm::SCL;
					bulk_g2s_stream(dK + Gm::PAY, sK + so, Gm::SCL, &bar[st], policy);
					bulk_g2s_stream(dV + Gm::PAY, sV + so, Gm::SCL, &bar[st], policy);
				}
			} else {
				mbar_arrive(&bar[st]);
			}
		}
	};
	int p = 0;
	for (; p < n && p < NST - 1; ++p)
		issue(p);

	SufSeg cc = locate_suffix(pre, S, H, xa);
	bool redo = false;
	uint32_t q[D / 8];
	load_q<D>(q, a, cc.s, cc.h, lane);
	const float scale = a.scale_log2 * (Gm::MX ? KLLM_MX_DEC_UNBIAS : 1.f);
	float sl2 = scale;
	if constexpr (Gm::MX)
		sl2 = scale * q_to_f16<D>(q);
	float o[D / 16][4];
#pragma unroll
	for (int mt = 0; mt < D / 16; ++mt)
		o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
	float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
	float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
	const int g = lane >> 2, c = lane & 3;

#pragma unroll 1
	for (int i = 0; i < n; ++i) {
		if (p < n) {
			issue(p);
			++p;
		}
		const int st = i % NST;
		if (!__all_sync(0xffffffffu, mbar_wait_ns(&bar[st], (uint32_t)((i / NST) & 1), kPWaitNs))) {
			if (lane == 0 && a.err)
				atomicOr(a.err, KLLM_ERR_TIMEOUT_BIT);
			for (int j = i + 1; j < p; ++j)        // this warp's copies in flight
				mbar_wait_ns(&bar[j % NST], (uint32_t)((j / NST) & 1), kPWaitNs);
			return;
		}
		const int ntok = *reinterpret_cast<volatile int *>(&ntoks[st]);
		if (ntok > 0) {
			const uint8_t *sK = ring + (size_t)st * Gm::STAGE;
			tile_compute<D, KVT>(sK, sK + Gm::KV, lut, ntok, q, o, m0, m1, l0, l1, mx0, mx1, sl2,
					     lane);
		}
		__syncwarp();
		const bool seg_end = cc.j + 1 == cc.ts, last = i + 1 == n;
		if (!(seg_end || last)) {
			++cc.j;
			continue;
		}
		// ---- piece finished: its partial, against its exact maximum ----------------
#pragma unroll
		for (int off = 4; off < 32; off <<= 1) {
			mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
			mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
		}
		const float f0 = mx0 > m0 ? exp2f(m0 - mx0) : 1.f, f1 = mx1 > m1 ? exp2f(m1 - mx1) : 1.f;
		m0 = fmaxf(m0, mx0);
		m1 = fmaxf(m1, mx1);
		float L0 = l0 * f0, L1 = l1 * f1;
#pragma unroll
		for (int off = 4; off < 32; off <<= 1) {
			L0 += __shfl_xor_sync(0xffffffffu, L0, off);
			L1 += __shfl_xor_sync(0xffffffffu, L1, off);
		}
		// (sequence, head) + warp numbers the pieces without gaps or clashes
		const size_t slot = (size_t)cc.s * H + cc.h + w;
		float *xm = a.xm + slot * a.group, *xl = a.xl + slot * a.group, *xo = a.xo + slot * a.group * D;
		if constexpr (Gm::MX) {
			// not finite: the piece is marked by its sum and done again at the end
			bool bad = !isfinite(L0) || !isfinite(L1);
#pragma unroll
			for (int mt = 0; mt < D / 16; ++mt)
				bad |= !isfinite(o[mt][0] + o[mt][1] + o[mt][2] + o[mt][3]);
			if (__any_sync(0xffffffffu, bad)) {
				L0 = L1 = CUDART_INF_F;
				redo = true;
			}
		}
#pragma unroll
		for (int hp = 0; hp < 2; ++hp) {
			const int hh = 2 * c + hp;
			if (hh < a.group) {
				const float f = hp ? f1 : f0;
				float *dst = xo + (size_t)hh * D + g * (D / 8);
#pragma unroll
				for (int mt = 0; mt < D / 16; mt += 2)
					*reinterpret_cast<float4 *>(dst + 2 * mt) =
					    make_float4(o[mt][hp] * f, o[mt][2 + hp] * f,
							o[mt + 1][hp] * f, o[mt + 1][2 + hp] * f);
				if (g == 0) {
					xm[hh] = hp ? m1 : m0;
					xl[hh] = hp ? L1 : L0;
				}
			}
		}
		if (last)
			break;
		cc.j = 0;
		if (++cc.h == H) {
			cc.h = 0;
			do {
				++cc.s;
			} while (pre[cc.s + 1] == pre[cc.s]);
			cc.ts = pre[cc.s + 1] - pre[cc.s];
		}
		load_q<D>(q, a, cc.s, cc.h, lane);
		if constexpr (Gm::MX)
			sl2 = scale * q_to_f16<D>(q);
#pragma unroll
		for (int mt = 0; mt < D / 16; ++mt)
			o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
		m0 = m1 = mx0 = mx1 = -CUDART_INF_F;
		l0 = l1 = 0.f;
	}
	if constexpr (Gm::MX) {
		if (redo) {                    // rare: the marked pieces of this warp, exactly
			__syncwarp();
			const PHeader *hd = static_cast<const PHeader *>(a.header);
			const long long xb = div_steps((w + 1) * hd->N, hd->WS);
			for (long long x = xa; x < xb;) {
				const SufSeg e = locate_suffix(pre, S, H, x);
				const int nt = (int)min((long long)(e.ts - e.j), xb - x);
				const size_t slot = ((size_t)e.s * H + e.h + w) * a.group;
				if (__ldcg(a.xl + slot) == CUDART_INF_F)
					suffix_exact<D>(a, e.s, e.h, e.j, e.j + nt, a.scale_log2, a.xm + slot,
							a.xl + slot, a.xo + slot * D);
				x += nt;
			}
		}
	}
}

template <int D, int KVT>
__global__ void __launch_bounds__(kPThreads, 1)
attend_kernel(const kllm_prefix_args a)
{
	extern __shared__ __align__(1024) uint8_t smem_raw[];
	// an offset, not a rounded pointer: the compiler keeps to shared-memory loads
	uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
	// the plan this launch reads is written by the kernel before it
	grid_dependency_wait();
	grid_launch_dependents();
	const PHeader *hd = static_cast<const PHeader *>(a.header);
	const int cta = blockIdx.x, n_prefix = hd->n_prefix;
	if (cta < n_prefix) {
		const long long T = hd->T;
		const int W = hd->W;
		if (cta >= W)
			return;
		PrefixSmem<D, KVT> &sm = *reinterpret_cast<PrefixSmem<D, KVT> *>(smem);
		if (threadIdx.x == 0)
			init_prefix(sm);
		prefix_role<D, KVT>(a, sm, cta, T, W);
	} else {
		suffix_role<D, KVT>(a, smem, cta - n_prefix, hd->N, hd->WS);
	}
}

// ---- join -----------------------------------------------------------------------------

constexpr int kJRows = 16;

// A running (max, sum, 4 dims of o) and the fold of pieces into it; a piece
// with l = 0 counts nothing (its o is not written).
struct JoinAcc {
	float M, L, o[4];
};
template <int N>
__device__ __forceinline__ void fold(JoinAcc &A, const float (&l)[N], const float (&m)[N], const float4 (&o)[N])
{
	float mb = A.M;
#pragma unroll
	for (int u = 0; u < N; ++u)
		if (l[u] != 0.f)
			mb = fmaxf(mb, m[u]);
	if (mb > A.M) {
		const float f = exp2f(A.M - mb);               // 0 while M is -inf
		A.L *= f;
#pragma unroll
		for (int q = 0; q < 4; ++q)
			A.o[q] *= f;
		A.M = mb;
	}
#pragma unroll
	for (int u = 0; u < N; ++u)
		if (l[u] != 0.f) {
			const float e = exp2f(m[u] - A.M);
			A.L = fmaf(l[u], e, A.L);
			A.o[0] = fmaf(o[u].x, e, A.o[0]);
			A.o[1] = fmaf(o[u].y, e, A.o[1]);
			A.o[2] = fmaf(o[u].z, e, A.o[2]);
			A.o[3] = fmaf(o[u].w, e, A.o[3]);
		}
}

// One CTA: 16 consecutive rows (sequence-major) of one kv head, a thread 4 dims
// of a row. Phase 1, rows fastest: the prefix pieces, kFly pieces' loads in
// flight (the partials hold [D / 4][rows][4], so 16 lanes read 256 contiguous
// bytes). Phase 2, dims fastest: the suffix pieces (rows of D), and the store.
// kFly 8 takes 86 registers, one CTA an SM, and is the faster one when no SM
// gets a second CTA (64 rows of 8,192 shared tokens 47.4 us against 49.3); kFly
// 6 takes 64, two CTAs (256 rows: 93 us against 99).
template <int D, int kFly>
__global__ void __launch_bounds__(kJRows * D / 4, kFly == 8 ? 1 : 256 / D)
join_kernel(const kllm_prefix_args a, float unbias)
{
	constexpr int kFlyS = kFly / 2;
	__shared__ float acc_s[kJRows][D + 4];
	__shared__ float m_s[kJRows], l_s[kJRows];
	const int tid = threadIdx.x;
	const int h = blockIdx.y, H = a.num_kv_heads, rows = a.num_seqs * a.group;
	// The plan is complete here: the attention's CTAs let this kernel start only
	// after they have waited for it. Its partials need the wait below.
	const PHeader *hd = static_cast<const PHeader *>(a.header);
	const int lr1 = tid % kJRows, ch1 = tid / kJRows, i = blockIdx.x * kJRows + lr1;
	const int lr2 = tid / (D / 4), ch2 = tid % (D / 4), ii = blockIdx.x * kJRows + lr2;
	const int seq2 = min(ii, rows - 1) / a.group;
	const int t0 = a.tile_pre[seq2], ts = a.tile_pre[seq2 + 1] - t0;
	const long long N = hd->N, WS = hd->WS;
	{
		const int seq = i / a.group;
		const int g = i < rows ? a.row_group[seq] : -1;
		JoinAcc A = {-CUDART_INF_F, 0.f, {0.f, 0.f, 0.f, 0.f}};
		if (g < 0) {
			grid_dependency_wait();
		} else {
			const long long T = hd->T, W = hd->W;
			const PGroup G = static_cast<const PGroup *>(a.groups)[g];
			const int lr = (seq - G.row0) * a.group + i % a.group;
			const bool solo = G.wgt == 1;
			const int tile = lr / kUnitRows, r = lr - tile * kUnitRows;
			const int urows = min(kUnitRows, G.nseq * a.group - tile * kUnitRows);
			const long long cost = (long long)G.nblk * G.wgt;
			const long long ux = G.x0 + ((long long)h * G.tiles + tile) * cost;
			// the shares that overlap the unit; solo pieces are two streams
			const long long c0 = div_steps((ux + 1) * W - 1, T), c1 = div_steps((ux + cost) * W - 1, T);
			const long long base = G.r0 + (long long)h * G.alloc + tile * kUnitRows + kUnitRows * c0;
			const int sh = solo ? 1 : 0, np = (int)(c1 - c0 + 1) << sh;
			grid_dependency_wait();
			for (int p0 = 0; p0 < np; p0 += kFly) {
				float l[kFly], m[kFly];
				float4 o[kFly];
#pragma unroll
				for (int u = 0; u < kFly; ++u) {
					const int p = p0 + u;
					l[u] = 0.f;
					m[u] = -CUDART_INF_F;
					if (p < np) {
						const long long at = base + (long long)kUnitRows * (p >> sh) +
								     (solo && (p & 1) ? urows : 0);
						l[u] = __ldcg(a.pl + at + r);
						m[u] = __ldcg(a.pm + at + r);
						o[u] = __ldcg(reinterpret_cast<const float4 *>(
						    a.po + at * D + ((size_t)ch1 * urows + r) * 4));
					}
				}
				fold(A, l, m, o);
			}
		}
		*reinterpret_cast<float4 *>(&acc_s[lr1][4 * ch1]) = make_float4(A.o[0], A.o[1], A.o[2], A.o[3]);
		if (ch1 == 0) {
			m_s[lr1] = A.M;
			l_s[lr1] = A.L;
		}
	}
	__syncthreads();
	if (ii >= rows)
		return;
	const int seq = seq2, hh = ii - seq * a.group;
	JoinAcc A;
	A.M = m_s[lr2];
	A.L = l_s[lr2];
	*reinterpret_cast<float4 *>(A.o) = *reinterpret_cast<const float4 *>(&acc_s[lr2][4 * ch2]);
	if (ts > 0) {
		const long long x0 = (long long)t0 * H + (long long)h * ts;
		const long long w0 = div_steps((x0 + 1) * WS - 1, N), w1 = div_steps((x0 + ts) * WS - 1, N);
		const size_t slot = (size_t)seq * H + h + w0;
		const int np = (int)(w1 - w0 + 1);
		for (int p0 = 0; p0 < np; p0 += kFlyS) {
			float l[kFlyS], m[kFlyS];
			float4 o[kFlyS];
#pragma unroll
			for (int u = 0; u < kFlyS; ++u) {
				l[u] = 0.f;
				m[u] = -CUDART_INF_F;
				if (p0 + u < np) {
					const size_t at = (slot + p0 + u) * a.group + hh;
					l[u] = __ldcg(a.xl + at);
					m[u] = __ldcg(a.xm + at);
					o[u] = __ldcg(reinterpret_cast<const float4 *>(a.xo + at * D + 4 * ch2));
				}
			}
			fold(A, l, m, o);
		}
	}
	const float inv = A.L != 0.f ? unbias / A.L : 0.f;    // an empty row gives zeros
	const size_t row = (size_t)seq * a.num_heads + (size_t)h * a.group + hh;
	*reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.out) + (row * D + 4 * ch2) * 2) =
	    make_uint2(pack_bf16x2(A.o[0] * inv, A.o[1] * inv), pack_bf16x2(A.o[2] * inv, A.o[3] * inv));
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
cudaError_t launch_attend(const kllm_prefix_args &a, cudaStream_t st)
{
	// at least half an SM's shared memory, so that one CTA has the SM's TMEM
	size_t smem = sizeof(PrefixSmem<D, KVT>);
	if (smem < SufLayout<D, KVT>::total)
		smem = SufLayout<D, KVT>::total;
	smem += 1024;
	if (smem < 120u * 1024u)
		smem = 120u * 1024u;
	const cudaError_t e = cudaFuncSetAttribute(
	    attend_kernel<D, KVT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
	if (e != cudaSuccess)
		return e;
	return launch_dependent(attend_kernel<D, KVT>, dim3((unsigned)a.ctas), kPThreads, smem, st, 1, a);
}

}  // namespace
}  // namespace kllm

using namespace kllm;

static uint64_t up256(uint64_t x) { return (x + 255u) & ~(uint64_t)255u; }

extern "C" uint64_t kllm_prefix_workspace(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
					  int ctas, void *base, struct kllm_prefix_args *a)
{
	uint8_t *p = static_cast<uint8_t *>(base);
	const uint64_t S = (uint64_t)num_seqs, G = (uint64_t)(num_heads / num_kv_heads);
	// prefix partials: two streams of a row, and a unit's rows for every CTA
	// boundary; suffix partials: one per (sequence, kv head) and one per warp
	const uint64_t part = 2u * S * num_heads + (uint64_t)kUnitRows * ctas;
	const uint64_t suf = (S * num_kv_heads + (uint64_t)ctas * 16u) * G;
	uint64_t at = 0;
	auto take = [&](uint64_t bytes) {
		uint8_t *q = p + at;
		at += up256(bytes);
		return q;
	};
	uint8_t *header = take(sizeof(PHeader)), *groups = take(S * sizeof(PGroup));
	uint8_t *rg = take(S * 4), *ss = take(S * 4), *sl = take(S * 4), *tp = take((S + 1) * 4);
	uint8_t *xm = take(suf * 4), *xl = take(suf * 4), *xo = take(suf * head_dim * 4);
	uint8_t *pm = take(part * 4), *pl = take(part * 4), *po = take(part * head_dim * 4);
	if (a) {
		a->header = header;
		a->groups = groups;
		a->row_group = reinterpret_cast<int *>(rg);
		a->suf_start = reinterpret_cast<int *>(ss);
		a->suf_lens = reinterpret_cast<int *>(sl);
		a->tile_pre = reinterpret_cast<int *>(tp);
		a->xm = reinterpret_cast<float *>(xm);
		a->xl = reinterpret_cast<float *>(xl);
		a->xo = reinterpret_cast<float *>(xo);
		a->pm = reinterpret_cast<float *>(pm);
		a->pl = reinterpret_cast<float *>(pl);
		a->po = reinterpret_cast<float *>(po);
	}
	return at;
}

extern "C" int kllm_prefix_launch(struct kllm_prefix_args *a, void *stream)
{
	cudaStream_t st = static_cast<cudaStream_t>(stream);
	a->suf_warps = a->kv_dtype ? SW<1>::N : SW<0>::N;
	plan_kernel<<<1, kPlanThreads, 0, st>>>(*a);
	cudaError_t e = cudaGetLastError();
	if (e != cudaSuccess)
		return (int)e;
	if (a->head_dim == 128)
		e = a->kv_dtype ? launch_attend<128, 1>(*a, st) : launch_attend<128, 0>(*a, st);
	else
		e = a->kv_dtype ? launch_attend<64, 1>(*a, st) : launch_attend<64, 0>(*a, st);
	if (e != cudaSuccess)
		return (int)e;
	const dim3 grid((unsigned)(((long long)a->num_seqs * a->group + kJRows - 1) / kJRows),
			(unsigned)a->num_kv_heads);
	const float unbias = a->kv_dtype ? KLLM_MX_DEC_UNBIAS : 1.f;
	const bool one = (long long)grid.x * grid.y <= a->ctas;
	if (a->head_dim == 128)
		return (int)launch_dependent(one ? join_kernel<128, 8> : join_kernel<128, 6>, grid, kJRows * 32,
					     0, st, 1, *a, unbias);
	return (int)launch_dependent(one ? join_kernel<64, 8> : join_kernel<64, 6>, grid, kJRows * 16, 0, st,
				     1, *a, unbias);
}
