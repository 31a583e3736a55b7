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

// 4, 8 or 16 rows a CTA (SW = 1, 2 or 4): the ordered sum of each by one thread (a lane of
// the chain's warp a row), as the other eight warps bring the squares in, 256 columns
// at a time into a ring, each warp's loads a chunk ahead of its stores. A row's sum is k
// dependent adds, but the chains of a warp's lanes and of the other CTAs run beside it,
// where the CTA form above spends a whole CTA on one row. The rows themselves are not
// kept: the quantiser reads s again, out of L2 (13 rows of 4096 a multiprocessor is what shared
// memory would hold: 47 us). 2048 rows of 4096 with the residual: 36 us, 3.1 TB/s of the 110 MB;
// 10 us of that is a row's chain, 4.6 cycles an add.
constexpr int NORM_CHAIN_THREADS = 288;
constexpr uint32_t NORM_CHAIN_COLS = 256, NORM_CHAIN_STAGES = 4, NORM_CHAIN_LOADERS = 8;
constexpr uint32_t NORM_CHAIN_PITCH = NORM_CHAIN_COLS + 4;      // (16 bytes on: other banks)
constexpr int NORM_ERR_CHAIN = 26;

inline size_t norm_chain_smem(uint32_t rows)
{
	return (size_t)NORM_CHAIN_STAGES * rows * NORM_CHAIN_PITCH * sizeof(float);
}

__device__ __forceinline__ float4 add4_rn(const float4 &a, const float4 &b)
{
	return make_float4(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y), __fadd_rn(a.z, b.z), __fadd_rn(a.w, b.w));
}

template <int SW>
__global__ void __launch_bounds__(NORM_CHAIN_THREADS)
norm_chain_kernel(const float *x, const float *add, const float *__restrict__ w, uint32_t m,
		  uint32_t k, float eps, float *x_out, int8_t *__restrict__ q, float *__restrict__ d,
		  int *err)
{
	constexpr uint32_t NS = NORM_CHAIN_STAGES, R = 4 * SW;
	extern __shared__ __align__(16) float ncsm[];
	__shared__ __align__(8) uint64_t b_full[NS], b_free[NS];
	__shared__ float s_scale[R];
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const uint32_t chunks = (k + NORM_CHAIN_COLS - 1) / NORM_CHAIN_COLS;
	const size_t row0 = (size_t)blockIdx.x * R;
	const uint32_t n = (uint32_t)(m - row0 < R ? m - row0 : R);
	if (threadIdx.x < NS) {
		mbar_init(&b_full[threadIdx.x], NORM_CHAIN_LOADERS);
		mbar_init(&b_free[threadIdx.x], 1);
	}
	__syncthreads();
	pdl_wait();
	// (No early start of the kernel after this one: its CTAs, waiting beside these, took 2048
	// rows of 4096 from 36 to 44 us.)
	bool ok = true;
	if (warp == NORM_CHAIN_LOADERS) {
		float ss = 0.0f;
		for (uint32_t c = 0; c < chunks; c++) {
			ok = __all_sync(0xffffffffu, mbar_wait_bounded(&b_full[c % NS], c / NS & 1, WAIT_LIMIT_NS));
			if (!ok)
				break;
			if (lane < n) {
				// (a row's last chunk is filled up with zeros, which leave the sum as it is)
				const float4 *t = reinterpret_cast<const float4 *>(ncsm + (c % NS * R + lane) * NORM_CHAIN_PITCH);
#pragma unroll 16
				for (uint32_t i = 0; i < NORM_CHAIN_COLS / 4; i++) {
					const float4 v = t[i];
					ss = __fadd_rn(ss, v.x);
					ss = __fadd_rn(ss, v.y);
					ss = __fadd_rn(ss, v.z);
					ss = __fadd_rn(ss, v.w);
				}
			}
			__syncwarp();
			if (lane == 0)
				mbar_arrive(&b_free[c % NS]);
		}
		if (lane < n)
			s_scale[lane] = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)k), eps)));
	} else {
		// this warp's pieces of 128 columns of a chunk: rows 4 j + warp / 2, half warp % 2
		const uint32_t o = warp % 2 * 128 + lane * 4;
		const size_t at0 = (row0 + warp / 2) * k + o;
		float4 now[SW], plus[SW];
		auto load = [&](uint32_t c) {
#pragma unroll
			for (int j = 0; j < SW; j++) {
				const bool in = warp / 2 + 4 * j < n && c * NORM_CHAIN_COLS + o < k;
				const size_t at = at0 + (size_t)4 * j * k + c * NORM_CHAIN_COLS;
				now[j] = in ? *(const float4 *)(x + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				if (add)
					plus[j] = in ? *(const float4 *)(add + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			}
		};
		load(0);
		for (uint32_t c = 0; c < chunks; c++) {
			float4 v[SW];
#pragma unroll
			for (int j = 0; j < SW; j++)
				v[j] = add ? add4_rn(now[j], plus[j]) : now[j];
			if (c + 1 < chunks)
				load(c + 1);
			if (c >= NS)
				ok = __all_sync(0xffffffffu, mbar_wait_bounded(&b_free[c % NS], (c / NS - 1) & 1, WAIT_LIMIT_NS));
			if (!ok)
				break;
#pragma unroll
			for (int j = 0; j < SW; j++) {
				if (x_out && warp / 2 + 4 * j < n && c * NORM_CHAIN_COLS + o < k)
					*(float4 *)(x_out + at0 + (size_t)4 * j * k + c * NORM_CHAIN_COLS) = v[j];
				*(float4 *)(ncsm + (c % NS * R + warp / 2 + 4 * j) * NORM_CHAIN_PITCH + o) =
					make_float4(__fmul_rn(v[j].x, v[j].x), __fmul_rn(v[j].y, v[j].y),
						    __fmul_rn(v[j].z, v[j].z), __fmul_rn(v[j].w, v[j].w));
			}
			__syncwarp();
			if (lane == 0)
				mbar_arrive(&b_full[c % NS]);
		}
	}
	if (!ok && lane == 0)
		*(volatile int *)err = NORM_ERR_CHAIN;
	__syncthreads();
	// the quantiser: 8 lanes a 32-block, 4 blocks a warp at a time, 4 rows together, the next
	// four's loads ahead. The two divisions of a block are done once, by the lane of its
	// 8 that has the row's number.
	const uint32_t segs = (k + 127) / 128, units = segs * SW;
	float4 now[4], g = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
	auto load = [&](uint32_t u) {
		const uint32_t i = u / SW * 128 + lane * 4, r0 = u % SW * 4;
		if (i < k)
			g = *(const float4 *)(w + i);
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const size_t at = (row0 + r0 + j) * k + i;
			now[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			if (i < k && r0 + j < n) {
				now[j] = x_out ? *(const float4 *)(x_out + at) : *(const float4 *)(x + at);
				if (!x_out && add)
					now[j] = add4_rn(now[j], *(const float4 *)(add + at));
			}
		}
	};
	if (warp < units)
		load(warp);
	for (uint32_t u = warp; u < units; u += NORM_CHAIN_THREADS / 32) {
		const uint32_t i = u / SW * 128 + lane * 4, r0 = u % SW * 4;
		const bool in = i < k;
		float4 v[4];
		float top[4];
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float s = s_scale[r0 + j];
			v[j].x = __fmul_rn(__fmul_rn(now[j].x, s), g.x);
			v[j].y = __fmul_rn(__fmul_rn(now[j].y, s), g.y);
			v[j].z = __fmul_rn(__fmul_rn(now[j].z, s), g.z);
			v[j].w = __fmul_rn(__fmul_rn(now[j].w, s), g.w);
			top[j] = fmaxf(fmaxf(fabsf(v[j].x), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
		}
		if (u + NORM_CHAIN_THREADS / 32 < units)
			load(u + NORM_CHAIN_THREADS / 32);
#pragma unroll
		for (int o = 4; o; o >>= 1)
#pragma unroll
			for (int j = 0; j < 4; j++)
				top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
		const uint32_t who = lane & 3;
		const float mine = who == 0 ? top[0] : who == 1 ? top[1] : who == 2 ? top[2] : top[3];
		const float dd = __fdiv_rn(mine, 127.0f);
		const float inv_mine = dd != 0.0f ? __fdiv_rn(1.0f, dd) : 0.0f;
		if (in && (lane & 4) == 0 && r0 + who < n)
			d[(row0 + r0 + who) * (k / 32) + i / 32] = dd;
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float inv = __shfl_sync(0xffffffffu, inv_mine, (lane & ~7u) | j);
			if (in && r0 + j < n) {
				const uint32_t a = (uint8_t)__float2int_rn(__fmul_rn(v[j].x, inv));
				const uint32_t b = (uint8_t)__float2int_rn(__fmul_rn(v[j].y, inv));
				const uint32_t c = (uint8_t)__float2int_rn(__fmul_rn(v[j].z, inv));
				const uint32_t e = (uint8_t)__float2int_rn(__fmul_rn(v[j].w, inv));
				*(uint32_t *)(q + (row0 + r0 + j) * k + i) = a | b << 8 | c << 16 | e << 24;
			}
		}
	}
}

} // namespace cgpu
