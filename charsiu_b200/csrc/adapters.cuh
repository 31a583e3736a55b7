// SPDX-License-Identifier: GPL-2.0-or-later
// Low-rank adapters of many requests beside a shared projection
// (charsiu_gpu_adapters_dev): y_r = base_r + scale_a B_a (A_a x_r), a = which[r].
//
// Two launches. The first makes t_r = A_a x_r (rank numbers a row): K is cut into
// pieces, one a CTA, whose sums go to scratch. The second adds the pieces up and
// makes y. Both take tiles of 16 rows, as mma.sync's m; a tile's rows may want
// different adapters, so a tile goes over the distinct ones among its rows, each
// product made into accumulators of its own and kept only for the rows that want
// it (whatever an adapter's weights are, they reach no other row).
//
// Bound by memory: an adapter's weights are used for few rows, and y is read and
// written for rank / 4 multiply-adds a byte.
//
// Precision: x is q d with q int8, exact in both 16-bit types, so a 32-block's
// products with A are exact and its sum is taken in fp32 before d scales it. t
// stays fp32: for its product with B it is cut into two tf32 parts of 11 bits each
// (the second the remainder), and B is exact in tf32, so what is lost is 2^-22 of a
// term.
#pragma once

#include "attn.cuh"
#include "charsiu_gpu.h"
#include "ptx.cuh"

namespace cgpu {

constexpr int ADAPT_MAX_SETS = 8;
constexpr uint32_t ADAPT_ROWS = 16;
constexpr uint32_t ADAPT_WARPS = 4;

struct AdaptSet {
	const void *a, *b;
	const int32_t *rank;
	const float *scale;
	const float *base;
	float *y;
	uint32_t n, slots, max_rank;
	uint32_t block_end;     // the expansion's column blocks up to this set's last
};

struct AdaptArgs {
	AdaptSet s[ADAPT_MAX_SETS];
	const int8_t *q;
	const float *d;
	const int32_t *which;
	float *t;               // [set][piece][row][RT]
	uint32_t n_sets, m, k, pieces, blocks;
};

// The next distinct adapter of the tile after those in `done` (bits of rows): its
// number, and the rows that want it; -1 none. `mine` is the adapter of row lane % 16.
__device__ __forceinline__ int32_t adapt_next(int32_t mine, uint32_t &done, uint32_t *rows)
{
	const uint32_t left = __ballot_sync(0xffffffffu, mine >= 0) & ~done & 0xffffu;
	if (!left)
		return -1;
	const int32_t a = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
	*rows = __ballot_sync(0xffffffffu, mine == a) & 0xffffu;
	done |= *rows;
	return a;
}

__device__ __forceinline__ int32_t adapt_which(const AdaptArgs &a, const AdaptSet &s, uint32_t row)
{
	if (row >= a.m)
		return -1;
	const int32_t w = a.which[row];
	return w >= 0 && (uint32_t)w < s.slots ? w : -1;
}

__device__ __forceinline__ uint32_t adapt_rank(const AdaptSet &s, int32_t a)
{
	const int32_t r = s.rank[a];
	return r < 0 ? 0 : (uint32_t)r > s.max_rank ? s.max_rank : (uint32_t)r;
}

// two int8 of a word as a pair of T
template <typename T>
__device__ __forceinline__ uint32_t int8_pair(uint32_t w, int at)
{
	const float lo = (float)(int8_t)(w >> (8 * at)), hi = (float)(int8_t)(w >> (8 * at + 8));
	return pack_pair<T>(lo, hi);
}

// t of one tile of rows and one piece of K, for one set. RT: ranks, padded to a
// multiple of 8. The warps take 32-blocks of the piece in turn. Within a block the
// mma's k is permuted alike for x and A so that a lane's 8 elements are
// consecutive (one 16-byte load of A).
template <typename T, int RT>
__global__ void __launch_bounds__(ADAPT_WARPS * 32)
adapt_shrink_kernel(const __grid_constant__ AdaptArgs a)
{
	constexpr int NT = RT / 8;
	__shared__ float s_t[ADAPT_WARPS][ADAPT_ROWS][RT];
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t row0 = blockIdx.x * ADAPT_ROWS, piece = blockIdx.y;
	const AdaptSet &set = a.s[blockIdx.z];
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t nb = a.k / 32, each = (nb + a.pieces - 1) / a.pieces;
	const uint32_t b0 = piece * each, b1 = min(b0 + each, nb);
	const int32_t mine = adapt_which(a, set, row0 + (lane & 15));
	float keep[NT][4];
#pragma unroll
	for (int n = 0; n < NT; n++)
		keep[n][0] = keep[n][1] = keep[n][2] = keep[n][3] = 0.0f;
	uint32_t done = 0, rows;
	for (int32_t ad; (ad = adapt_next(mine, done, &rows)) >= 0;) {
		const uint32_t rank = adapt_rank(set, ad);
		const T *w = (const T *)set.a + (size_t)ad * set.max_rank * a.k;
		float acc[NT][4];
#pragma unroll
		for (int n = 0; n < NT; n++)
			acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
		for (uint32_t b = b0 + warp; b < b1; b += ADAPT_WARPS) {
			uint32_t x[2][2] = {{0, 0}, {0, 0}};
			float dd[2] = {0.0f, 0.0f};
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const uint32_t r = row0 + lane / 4 + 8 * h;
				if (r < a.m) {
					const uint2 v = *(const uint2 *)(a.q + (size_t)r * a.k + b * 32 + c * 8);
					x[h][0] = v.x;
					x[h][1] = v.y;
					dd[h] = a.d[(size_t)r * nb + b];
				}
			}
			uint32_t fa[2][4];
#pragma unroll
			for (int s = 0; s < 2; s++) {
				fa[s][0] = int8_pair<T>(x[0][s], 0);
				fa[s][1] = int8_pair<T>(x[1][s], 0);
				fa[s][2] = int8_pair<T>(x[0][s], 2);
				fa[s][3] = int8_pair<T>(x[1][s], 2);
			}
#pragma unroll
			for (int n = 0; n < NT; n++) {
				const uint32_t r = n * 8 + lane / 4;
				uint4 v = make_uint4(0, 0, 0, 0);
				if (r < rank)
					v = *(const uint4 *)(w + (size_t)r * a.k + b * 32 + c * 8);
				float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
				mma_16816<T>(part, fa[0], v.x, v.y);
				mma_16816<T>(part, fa[1], v.z, v.w);
#pragma unroll
				for (int e = 0; e < 4; e++)
					acc[n][e] = __fmaf_rn(dd[e >> 1], part[e], acc[n][e]);
			}
		}
#pragma unroll
		for (int n = 0; n < NT; n++)
#pragma unroll
			for (int e = 0; e < 4; e++)
				if (rows >> (lane / 4 + 8 * (e >> 1)) & 1)
					keep[n][e] = acc[n][e];
	}
#pragma unroll
	for (int n = 0; n < NT; n++)
#pragma unroll
		for (int e = 0; e < 4; e++)
			s_t[warp][lane / 4 + 8 * (e >> 1)][n * 8 + c * 2 + (e & 1)] = keep[n][e];
	__syncthreads();
	float *t = a.t + (((size_t)blockIdx.z * a.pieces + piece) * a.m + row0) * RT;
	for (uint32_t i = threadIdx.x; i < ADAPT_ROWS * RT; i += ADAPT_WARPS * 32) {
		const uint32_t r = i / RT;
		if (row0 + r >= a.m)
			break;
		float v = 0.0f;
#pragma unroll
		for (int w = 0; w < (int)ADAPT_WARPS; w++)
			v += s_t[w][r][i % RT];
		t[i] = v;
	}
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
					 uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, "
		     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// y of one tile of rows and ADAPT_COLS columns of one set: each warp 8-column groups.
// The ranks are permuted alike for t and B so that a lane's RT / 4 are consecutive.
constexpr uint32_t ADAPT_COLS = 128;

template <typename T, int RT>
__global__ void __launch_bounds__(ADAPT_WARPS * 32)
adapt_expand_kernel(const __grid_constant__ AdaptArgs a)
{
	constexpr int SP = RT / 4, KS = RT / 8;          // ranks a lane; k steps
	__shared__ float s_t[ADAPT_ROWS][RT];
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t row0 = blockIdx.x * ADAPT_ROWS;
	uint32_t si = 0;
	while (blockIdx.y >= a.s[si].block_end)
		si++;
	const AdaptSet &set = a.s[si];
	const uint32_t col0 = (blockIdx.y - (si ? a.s[si - 1].block_end : 0)) * ADAPT_COLS;
	pdl_wait();
	pdl_launch_dependents();
	const int32_t mine = adapt_which(a, set, row0 + (lane & 15));
	const uint32_t wants = __ballot_sync(0xffffffffu, mine >= 0);
	for (uint32_t i = threadIdx.x; i < ADAPT_ROWS * RT; i += ADAPT_WARPS * 32) {
		float v = 0.0f;
		if (row0 + i / RT < a.m)
			for (uint32_t p = 0; p < a.pieces; p++)
				v += a.t[(((size_t)si * a.pieces + p) * a.m + row0) * RT + i];
		s_t[i / RT][i % RT] = v;
	}
	__syncthreads();
	uint32_t hi[KS][4], lo[KS][4];
#pragma unroll
	for (int ks = 0; ks < KS; ks++)
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float v = s_t[lane / 4 + 8 * (j & 1)][c * SP + 2 * ks + (j >> 1)];
			hi[ks][j] = __float_as_uint(v) & 0xffffe000u;
			lo[ks][j] = __float_as_uint(__fsub_rn(v, __uint_as_float(hi[ks][j])));
		}
	for (uint32_t n0 = col0 + warp * 8; n0 < min(col0 + ADAPT_COLS, set.n); n0 += ADAPT_WARPS * 8) {
		float keep[4] = {0.0f, 0.0f, 0.0f, 0.0f};
		uint32_t done = 0, rows;
		for (int32_t ad; (ad = adapt_next(mine, done, &rows)) >= 0;) {
			const uint32_t rank = adapt_rank(set, ad);
			const float scale = set.scale[ad];
			const uint32_t n = n0 + lane / 4;
			T w[SP];
#pragma unroll
			for (int j = 0; j < SP; j += SP < 8 ? SP : 8) {
				const T *src = (const T *)set.b + ((size_t)ad * set.n + n) * set.max_rank + c * SP + j;
				const bool ok = n < set.n && c * SP + j < rank;
				if (SP == 2) {
					*(uint32_t *)(w + j) = ok ? *(const uint32_t *)src : 0u;
				} else if (SP == 4) {
					*(uint2 *)(w + j) = ok ? *(const uint2 *)src : make_uint2(0, 0);
				} else {
					*(uint4 *)(w + j) = ok ? *(const uint4 *)src : make_uint4(0, 0, 0, 0);
				}
			}
			float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
			for (int ks = 0; ks < KS; ks++) {
				const float w0 = c * SP + 2 * ks < rank ? to_float<T>(w[2 * ks]) : 0.0f;
				const float w1 = c * SP + 2 * ks + 1 < rank ? to_float<T>(w[2 * ks + 1]) : 0.0f;
				mma_tf32(acc, lo[ks], __float_as_uint(w0), __float_as_uint(w1));
				mma_tf32(acc, hi[ks], __float_as_uint(w0), __float_as_uint(w1));
			}
#pragma unroll
			for (int e = 0; e < 4; e++)
				if (rows >> (lane / 4 + 8 * (e >> 1)) & 1)
					keep[e] = __fmul_rn(scale, acc[e]);
		}
#pragma unroll
		for (int e = 0; e < 4; e++) {
			const uint32_t r = row0 + lane / 4 + 8 * (e >> 1), n = n0 + c * 2 + (e & 1);
			if (r < a.m && n < set.n) {
				const size_t at = (size_t)r * set.n + n;
				const float base = set.base[at];       // (a row of no adapter keeps its bits)
				set.y[at] = wants >> (lane / 4 + 8 * (e >> 1)) & 1 ? __fadd_rn(base, keep[e])
										   : base;
			}
		}
	}
}

} // namespace cgpu
