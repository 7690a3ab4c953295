// SPDX-License-Identifier: Apache-2.0
//
// kllm_decode_tile.cuh - the 16-token tile of the paged decode, shared by the
// split-KV decode and the suffixes of the shared-prefix attention: staging
// geometry, query fragments, and the scores, softmax update and PV of a tile.
#pragma once

#include "kllm_device.cuh"
#include "kllm_internal.h"

#include <math_constants.h>

namespace kllm {
namespace {

#ifndef KLLM_DEC_STAGES
#define KLLM_DEC_STAGES 2       // bulk-copy ring depth per warp
#endif
#ifndef KLLM_DEC_MIN_CTAS_MX
#define KLLM_DEC_MIN_CTAS_MX 4  // resident MX decode CTAs per SM (register cap)
#endif

constexpr int kTile = 16;
constexpr float kLazyLog2 = 8.f;                // reference max slack (p <= 256)

template <int D, int KVT>
struct Geom {
	static constexpr bool MX = (KVT == 1);
	static constexpr int PAY = MX ? kTile * D : kTile * D * 2;  // payload / tile
	static constexpr int SCL = MX ? kTile * D / 8 : 0;          // scales / tile
	static constexpr int KV = PAY + SCL;                        // one of K, V
	static constexpr int STAGE = 2 * KV;
	static constexpr int NST = KLLM_DEC_STAGES;                 // ring depth
	static constexpr int MIN_CTAS = MX ? KLLM_DEC_MIN_CTAS_MX : 2;  // per SM
};

struct DevEntry {  // userspace/gpu/paged_attention.cu:18-22 (24 bytes)
	unsigned long long k, v;
	int valid;
	int pad;
};

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t *p)
{
	if constexpr (N % 4 == 0) {
#pragma unroll
		for (int i = 0; i < N / 4; ++i) {
			uint4 v = reinterpret_cast<const uint4 *>(p)[i];
			w[4 * i] = v.x;
			w[4 * i + 1] = v.y;
			w[4 * i + 2] = v.z;
			w[4 * i + 3] = v.w;
		}
	} else if constexpr (N == 2) {
		uint2 v = *reinterpret_cast<const uint2 *>(p);
		w[0] = v.x;
		w[1] = v.y;
	} else {
		w[0] = *reinterpret_cast<const uint32_t *>(p);
	}
}

template <int D, typename Args>
__device__ __forceinline__ void load_q(uint32_t (&q)[D / 8],
				       const Args &a, int s, int h,
				       int lane)
{
	const int g = lane >> 2, c = lane & 3;
	if (g < a.group) {
		const uint8_t *p = reinterpret_cast<const uint8_t *>(a.q) +
			(((size_t)s * a.num_heads + (size_t)h * a.group + g) * D +
			 (size_t)c * (D / 4)) * 2;
#pragma unroll
		for (int i = 0; i < D / 32; ++i) {
			uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i);
			q[4 * i] = v.x;
			q[4 * i + 1] = v.y;
			q[4 * i + 2] = v.z;
			q[4 * i + 3] = v.w;
		}
	} else {
#pragma unroll
		for (int i = 0; i < D / 8; ++i)
			q[i] = 0u;
	}
}

// MX path: the segment's query rows (bf16, as load_q leaves them) -> f16,
// multiplied by 2^e so that the largest |q| lies in [2^14, 2^15): no
// overflow, and every bf16 value of at least 2^-28 of that maximum converts
// exactly. Returns 2^-e, which multiplies the softmax scale.
template <int D>
__device__ __forceinline__ float q_to_f16(uint32_t (&q)[D / 8])
{
	float mx = 0.f;
#pragma unroll
	for (int i = 0; i < D / 8; ++i)
		mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(q[i] << 16)),
				     fabsf(__uint_as_float(q[i] & 0xFFFF0000u))));
#pragma unroll
	for (int off = 1; off < 32; off <<= 1)
		mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
	const int E = mx > 0.f ? (int)((__float_as_uint(mx) >> 23) & 0xFFu) - 127 : 0;
	int e = 14 - E;
	e = e < -100 ? -100 : (e > 100 ? 100 : e);
	const float f = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
	for (int i = 0; i < D / 8; ++i)
		q[i] = pack_f16x2(__uint_as_float(q[i] << 16) * f,
				  __uint_as_float(q[i] & 0xFFFF0000u) * f);
	return __uint_as_float((uint32_t)(127 - e) << 23);
}

// One 16-token tile: scores, online-softmax update and PV accumulation.
template <int D, int KVT>
__device__ __forceinline__ void tile_compute(
    const uint8_t *sK, const uint8_t *sV, const uint32_t *lut, int ntok,
    const uint32_t (&q)[D / 8], float (&o)[D / 16][4], float &m0, float &m1,
    float &l0, float &l1, float &mx0, float &mx1, float scale_log2, int lane)
{
	using Gm = Geom<D, KVT>;
	const int g = lane >> 2, c = lane & 3;

	// ---- S^T[tok][head] = K . Q^T ------------------------------------------
	float s[4] = {0.f, 0.f, 0.f, 0.f};
	float s2[4] = {0.f, 0.f, 0.f, 0.f};  // odd k-steps: halves the MMA chain
	if constexpr (Gm::MX) {
		constexpr int KW = D / 16;
		uint32_t k0[KW], k1[KW];
		lds_words<KW>(k0, sK + g * D + c * (D / 4));
		lds_words<KW>(k1, sK + (g + 8) * D + c * (D / 4));
		uint32_t sw0, sw1;
		if constexpr (D == 128) {
			sw0 = *reinterpret_cast<const uint32_t *>(sK + kTile * D + g * 16 + c * 4);
			sw1 = *reinterpret_cast<const uint32_t *>(sK + kTile * D + (g + 8) * 16 + c * 4);
		} else {
			sw0 = *reinterpret_cast<const uint16_t *>(sK + kTile * D + g * 8 + c * 2);
			sw1 = *reinterpret_cast<const uint16_t *>(sK + kTile * D + (g + 8) * 8 + c * 2);
		}
		uint32_t sc0[D / 32], sc1[D / 32];
#pragma unroll
		for (int b = 0; b < D / 32; ++b) {
			sc0[b] = lut[__byte_perm(sw0, 0u, 0x4440u | b)];
			sc1[b] = lut[__byte_perm(sw1, 0u, 0x4440u | b)];
		}
#pragma unroll
		for (int j = 0; j < D / 16; ++j) {
			// word j = dims 4j..4j+3 of this lane's chunk: (0,1) -> a0/a1, (2,3) -> a2/a3
			const uint32_t a0 = f16x2_mul(e4m3x2_lo_to_f16x2(k0[j]), sc0[j >> 1]);
			const uint32_t a2 = f16x2_mul(e4m3x2_hi_to_f16x2(k0[j]), sc0[j >> 1]);
			const uint32_t a1 = f16x2_mul(e4m3x2_lo_to_f16x2(k1[j]), sc1[j >> 1]);
			const uint32_t a3 = f16x2_mul(e4m3x2_hi_to_f16x2(k1[j]), sc1[j >> 1]);
			if (j & 1)
				mma_f16(s2, a0, a1, a2, a3, q[2 * j], q[2 * j + 1]);
			else
				mma_f16(s, a0, a1, a2, a3, q[2 * j], q[2 * j + 1]);
		}
	} else {
		constexpr int KW = D / 8;
		uint32_t k0[KW], k1[KW];
		lds_words<KW>(k0, sK + (g * D + c * (D / 4)) * 2);
		lds_words<KW>(k1, sK + ((g + 8) * D + c * (D / 4)) * 2);
#pragma unroll
		for (int j = 0; j < D / 16; ++j) {
			if (j & 1)
				mma_bf16(s2, k0[2 * j], k1[2 * j], k0[2 * j + 1],
					 k1[2 * j + 1], q[2 * j], q[2 * j + 1]);
			else
				mma_bf16(s, k0[2 * j], k1[2 * j], k0[2 * j + 1],
					 k1[2 * j + 1], q[2 * j], q[2 * j + 1]);
		}
	}
#pragma unroll
	for (int i = 0; i < 4; ++i)
		s[i] += s2[i];

	// ---- online softmax (log2 domain, lazy reference max) ---------------------
	// m0/m1 are warp-uniform reference maxima per head. They are raised only
	// when some lane's score exceeds them by more than kLazyLog2, so most tiles
	// skip the cross-lane max and the O rescale; p then stays <= 2^kLazyLog2.
	// mx0/mx1 track each lane's exact running maximum for the final triple.
	const bool v0 = g < ntok, v1 = g + 8 < ntok;
	const float x0 = v0 ? s[0] * scale_log2 : -CUDART_INF_F;  // tok g,   head 2c
	const float x1 = v0 ? s[1] * scale_log2 : -CUDART_INF_F;  // tok g,   head 2c+1
	const float x2 = v1 ? s[2] * scale_log2 : -CUDART_INF_F;  // tok g+8, head 2c
	const float x3 = v1 ? s[3] * scale_log2 : -CUDART_INF_F;  // tok g+8, head 2c+1
	float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
	mx0 = fmaxf(mx0, t0);
	mx1 = fmaxf(mx1, t1);
	if (__any_sync(0xffffffffu, t0 > m0 + kLazyLog2 || t1 > m1 + kLazyLog2)) {
#pragma unroll
		for (int off = 4; off < 32; off <<= 1) {
			t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
			t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
		}
		const float mn0 = fmaxf(m0, t0), mn1 = fmaxf(m1, t1);  // finite: ntok >= 1
		const float al0 = exp2f(m0 - mn0), al1 = exp2f(m1 - mn1);
		l0 *= al0;
		l1 *= al1;
		m0 = mn0;
		m1 = mn1;
#pragma unroll
		for (int mt = 0; mt < D / 16; ++mt) {
			o[mt][0] *= al0;
			o[mt][1] *= al1;
			o[mt][2] *= al0;
			o[mt][3] *= al1;
		}
	}
	const float p0 = exp2f(x0 - m0), p2 = exp2f(x2 - m0);
	const float p1 = exp2f(x1 - m1), p3 = exp2f(x3 - m1);
	l0 += p0 + p2;
	l1 += p1 + p3;
	// P as a hi + lo pair of the V operand's type (bf16: 16 significant bits,
	// f16: 22): one rounded P misses the 1e-3 absolute bound on outputs built
	// from a few large, cancelling V values.
	uint32_t h01, h23, l01, l23;
	if constexpr (Gm::MX) {
		h01 = pack_f16x2(p0, p1);
		h23 = pack_f16x2(p2, p3);
		const float2 f01 = __half22float2(*reinterpret_cast<const __half2 *>(&h01));
		const float2 f23 = __half22float2(*reinterpret_cast<const __half2 *>(&h23));
		l01 = pack_f16x2(p0 - f01.x, p1 - f01.y);
		l23 = pack_f16x2(p2 - f23.x, p3 - f23.y);
	} else {
		h01 = pack_bf16x2(p0, p1);
		h23 = pack_bf16x2(p2, p3);
		l01 = pack_bf16x2(p0 - __uint_as_float(h01 << 16),
				  p1 - __uint_as_float(h01 & 0xFFFF0000u));
		l23 = pack_bf16x2(p2 - __uint_as_float(h23 << 16),
				  p3 - __uint_as_float(h23 & 0xFFFF0000u));
	}
	const uint32_t b0 = movmatrix_trans(h01);   // tok 2c,2c+1;   head g
	const uint32_t b1 = movmatrix_trans(h23);   // tok 2c+8,2c+9; head g
	const uint32_t c0 = movmatrix_trans(l01);
	const uint32_t c1 = movmatrix_trans(l23);

	// ---- O^T[dim][head] += V^T . P^T -----------------------------------------
	const int r0 = 2 * c, r1 = 2 * c + 1, r2 = 2 * c + 8, r3 = 2 * c + 9;
	if constexpr (Gm::MX) {
		constexpr int VW = D / 32;
		uint32_t w0[VW], w1[VW], w2[VW], w3[VW];
		lds_words<VW>(w0, sV + r0 * D + g * (D / 8));
		lds_words<VW>(w1, sV + r1 * D + g * (D / 8));
		lds_words<VW>(w2, sV + r2 * D + g * (D / 8));
		lds_words<VW>(w3, sV + r3 * D + g * (D / 8));
		if (ntok < kTile) {  // zero rows past the context (payload 0 == 0.0)
#pragma unroll
			for (int i = 0; i < VW; ++i) {
				if (r0 >= ntok) w0[i] = 0u;
				if (r1 >= ntok) w1[i] = 0u;
				if (r2 >= ntok) w2[i] = 0u;
				if (r3 >= ntok) w3[i] = 0u;
			}
		}
		constexpr int NB = D / 64;  // scale blocks per lane chunk
		uint32_t s01[NB], s23[NB];
		const uint8_t *sS = sV + kTile * D;
#pragma unroll
		for (int bb = 0; bb < NB; ++bb) {
			const int col = g * NB + bb;
			s01[bb] = __byte_perm(lut[sS[r0 * (D / 8) + col]],
					      lut[sS[r1 * (D / 8) + col]], 0x5410u);
			s23[bb] = __byte_perm(lut[sS[r2 * (D / 8) + col]],
					      lut[sS[r3 * (D / 8) + col]], 0x5410u);
		}
#pragma unroll
		for (int i = 0; i < VW; ++i) {
			const int bb = i >> 1;  // m-tiles 2i, 2i+1 -> dims 4i..4i+3 -> block (4i)/8
			const uint32_t c01a = __byte_perm(w0[i], w1[i], 0x5140u);
			const uint32_t c01b = __byte_perm(w0[i], w1[i], 0x7362u);
			const uint32_t c23a = __byte_perm(w2[i], w3[i], 0x5140u);
			const uint32_t c23b = __byte_perm(w2[i], w3[i], 0x7362u);
			// (R0,R1) / (R2,R3) token pairs of dims 4i, 4i+1 (x) and 4i+2, 4i+3 (y)
			const uint32_t e0 = f16x2_mul(e4m3x2_lo_to_f16x2(c01a), s01[bb]);
			const uint32_t e1 = f16x2_mul(e4m3x2_hi_to_f16x2(c01a), s01[bb]);
			const uint32_t e2 = f16x2_mul(e4m3x2_lo_to_f16x2(c23a), s23[bb]);
			const uint32_t e3 = f16x2_mul(e4m3x2_hi_to_f16x2(c23a), s23[bb]);
			mma_f16(o[2 * i], e0, e1, e2, e3, b0, b1);
			mma_f16(o[2 * i], e0, e1, e2, e3, c0, c1);
			const uint32_t f0 = f16x2_mul(e4m3x2_lo_to_f16x2(c01b), s01[bb]);
			const uint32_t f1 = f16x2_mul(e4m3x2_hi_to_f16x2(c01b), s01[bb]);
			const uint32_t f2 = f16x2_mul(e4m3x2_lo_to_f16x2(c23b), s23[bb]);
			const uint32_t f3 = f16x2_mul(e4m3x2_hi_to_f16x2(c23b), s23[bb]);
			mma_f16(o[2 * i + 1], f0, f1, f2, f3, b0, b1);
			mma_f16(o[2 * i + 1], f0, f1, f2, f3, c0, c1);
		}
	} else {
		constexpr int VW = D / 16;
		uint32_t w0[VW], w1[VW], w2[VW], w3[VW];
		lds_words<VW>(w0, sV + (r0 * D + g * (D / 8)) * 2);
		lds_words<VW>(w1, sV + (r1 * D + g * (D / 8)) * 2);
		lds_words<VW>(w2, sV + (r2 * D + g * (D / 8)) * 2);
		lds_words<VW>(w3, sV + (r3 * D + g * (D / 8)) * 2);
		if (ntok < kTile) {  // rows past the context may hold any bits
#pragma unroll
			for (int i = 0; i < VW; ++i) {
				if (r0 >= ntok) w0[i] = 0u;
				if (r1 >= ntok) w1[i] = 0u;
				if (r2 >= ntok) w2[i] = 0u;
				if (r3 >= ntok) w3[i] = 0u;
			}
		}
#pragma unroll
		for (int mt = 0; mt < D / 16; ++mt) {
			const uint32_t e0 = __byte_perm(w0[mt], w1[mt], 0x5410u);
			const uint32_t e1 = __byte_perm(w0[mt], w1[mt], 0x7632u);
			const uint32_t e2 = __byte_perm(w2[mt], w3[mt], 0x5410u);
			const uint32_t e3 = __byte_perm(w2[mt], w3[mt], 0x7632u);
			mma_bf16(o[mt], e0, e1, e2, e3, b0, b1);
			mma_bf16(o[mt], e0, e1, e2, e3, c0, c1);
		}
	}
}

}  // namespace
}  // namespace kllm
