// SPDX-License-Identifier: GPL-2.0-or-later
// rmsnorm of a batch of rows with the residual's addition and a q8_0 output
// (charsiu_gpu_norm_quantise_dev).
//
//   s = fl(x + add), ss = the sequential fp32 sum of fl(s_i^2),
//   scale = fl(1 / sqrt(fl(fl(ss / k) + eps))), v = fl(fl(s scale) w),
//   then the quantiser of each 32-block of v (charsiu_act_set).
//
// Every row's bits are the decode step's (fwd_norm_quant_kernel): the sum of
// squares keeps the reference's order.
#pragma once

#include "rowops.cuh"

namespace cgpu {

constexpr uint32_t NORM_ROWS_MAX_K = 8192;
constexpr int NORM_ROWS_THREADS = 512;

inline size_t norm_rows_smem(uint32_t k)
{
	return (size_t)3 * k * sizeof(float);
}

// One CTA a row: s and its squares in shared memory, the ordered sum by the CTA.
__global__ void __launch_bounds__(NORM_ROWS_THREADS)
norm_rows_kernel(const float *x, const float *add, const float *__restrict__ w, uint32_t k,
		 float eps, float *x_out, int8_t *__restrict__ q, float *__restrict__ d)
{
	extern __shared__ __align__(16) float nrsm[];
	float *xs = nrsm, *sq = nrsm + k, *ws = nrsm + 2 * k;
	__shared__ float scale_s;
	const size_t row = blockIdx.x;
	pdl_wait();
	pdl_launch_dependents();
	for (uint32_t i = threadIdx.x * 4; i < k; i += blockDim.x * 4)
		cp_async16(ws + i, w + i);
	norm_quant_cta(x + row * k, add ? add + row * k : nullptr, k, eps, xs, sq, ws, &scale_s,
		       q + row * k, d + row * (k / 32));
	if (x_out)
		for (uint32_t i = threadIdx.x; i < k; i += blockDim.x)
			x_out[row * k + i] = xs[i];
}

} // namespace cgpu
