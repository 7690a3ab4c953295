// SPDX-License-Identifier: Apache-2.0
//
// kllm_topk.cuh - pieces shared by the scoring kernels: joining softmax sums,
// the fp32 order as integers, and sorted lists of 32 values in a warp.
#pragma once

#include "kllm_device.cuh"

#include <math_constants.h>

namespace kllm {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// Softmax sums of a set of logits l, c = log2(e) / T: m = max l, S = sum 2^((l -
// m) c), W = sum 2^((l - m) c) (l - m) c. join adds the set (m2, s2, w2) to (m, s,
// w): for a maximum raised by d = (M - m) c the sums become 2^-d S and 2^-d (W - d
// S). A set without elements has m = -inf, S = 0. A raise is cut where 2^-d is 0
// (M - m may be infinite).
__device__ __forceinline__ float raise_of(float m, float M, float c)
{
	return fminf((M - m) * c, 1000.f);
}
__device__ __forceinline__ void join(float &m, float &s, float &w, float m2, float s2, float w2, float c)
{
	const float M = fmaxf(m, m2);
	if (M == -CUDART_INF_F) {     // nothing finite on either side (NaN sums stay NaN)
		s += s2;
		w += w2;
		return;
	}
	const float d1 = m == -CUDART_INF_F ? 0.f : raise_of(m, M, c);
	const float d2 = m2 == -CUDART_INF_F ? 0.f : raise_of(m2, M, c);
	const float f1 = ex2_approx(-d1), f2 = ex2_approx(-d2);
	w = f1 * fmaf(-d1, s, w) + f2 * fmaf(-d2, s2, w2);
	s = f1 * s + f2 * s2;
	m = M;
}

// fp32 values as unsigned integers of the same order (-0 as +0), and back.
__device__ __forceinline__ uint32_t key_of(float v)
{
	const uint32_t u = __float_as_uint(v + 0.f);
	return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key)
{
	return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// The largest value below v. The key below +0 stands for -0, which compares
// equal to it, so zero steps over that one.
__device__ __forceinline__ float value_below(float v)
{
	const uint32_t key = key_of(v) - 1u;
	return value_of(key == 0x7fffffffu ? key - 1u : key);
}

// 32 values, one a lane, sorted descending over the warp (bitonic network).
__device__ __forceinline__ float bitonic_step(float x, int stride, bool keep_max)
{
	const float o = __shfl_xor_sync(0xffffffffu, x, stride);
	return keep_max ? fmaxf(x, o) : fminf(x, o);
}
__device__ __forceinline__ float warp_sort_desc(float x, int lane)
{
#pragma unroll
	for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
		for (int stride = size >> 1; stride; stride >>= 1)
			x = bitonic_step(x, stride, ((lane & stride) == 0) == ((lane & size) == 0));
	return x;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ float warp_merge_desc(float a, float b, int lane)
{
	a = fmaxf(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
	for (int stride = 16; stride; stride >>= 1)
		a = bitonic_step(a, stride, (lane & stride) == 0);
	return a;
}

}  // namespace
}  // namespace kllm
