// SPDX-License-Identifier: GPL-2.0-or-later
// Low-rank adapters of many requests beside a shared projection
// (charsiu_gpu_adapters_dev): y_r = base_r + scale_a B_a (A_a x_r), a = which[r].
//
// The first launch makes t_r = A_a x_r (rank numbers a row): K is cut into pieces whose sums
// go to scratch. The last adds the pieces up and makes y (where that is much to read a launch
// between them adds up). Both take tiles of 16 rows, as mma.sync's m, in long batches four of them. A
// tile's rows may want different adapters: each of its distinct ones is a product of its
// own over all 16 rows, of which only the rows that want it are kept (so whatever an
// adapter's weights are, they reach no other row). In a long prompt a tile has one; in a
// decode step of many requests they are spread over warps and CTAs.
//
// The bytes are few for the time they take (y is read and written for rank / 4 multiply-adds
// a byte, a decode step's adapters are a few MB): what bounds both is latency. 16 rows, K =
// N = 2048 and two of 512, rank 16: 12 us, of which two launches of 3 and in each a chain of
// four dependent loads (which adapter, its rank, its weights, ...). 2000 rows, K = N = 4096,
// rank 64: 44 us, t 16, its pieces 3, y 25 (66 MB of bases and outputs: 10 us at the copy rate).
//
// Precision: x is q d with q int8, exact in both 16-bit types, so a 32-block's products
// with A are exact and its sum is taken in fp32 before d scales it. t stays fp32: for its
// product with B it is cut into parts of which each product with B is exact, two of tf32
// (what is lost is less than 2^-21 of a term: the last two bits of fp32's 24), in long
// batches two or three of B's type (see there).
#pragma once

#include "attn.cuh"
#include "batch_checks.h"
#include "charsiu_gpu.h"
#include "ptx.cuh"

namespace cgpu {

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
	uint32_t n_sets, m, k;
	uint32_t pieces;        // of K
	uint32_t left;          // of them, for the last launch to add up: all, or 1 behind adapt_sum_kernel
	uint32_t parts;         // the first launch: CTAs that share a tile's distinct adapters
	uint32_t cols;          // the second: columns a CTA, a multiple of 32
	uint32_t blocks;        // and CTAs over all sets' columns
};

// A tile's distinct adapters: number, rows (a bit each), rank and scale
struct AdaptTile {
	int32_t ad[ADAPT_ROWS];
	uint32_t rows[ADAPT_ROWS], rank[ADAPT_ROWS];
	float scale[ADAPT_ROWS];
	uint32_t n, wants;      // how many; the rows that want one
};

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

// by one warp
__device__ __forceinline__ void adapt_tile(const AdaptArgs &a, const AdaptSet &s, uint32_t row0,
					   AdaptTile &t)
{
	const uint32_t lane = threadIdx.x & 31;
	const int32_t mine = lane < ADAPT_ROWS ? adapt_which(a, s, row0 + lane) : -1;
	const uint32_t same = __match_any_sync(0xffffffffu, mine);
	const bool first = mine >= 0 && (int)lane == __ffs(same) - 1;
	const uint32_t firsts = __ballot_sync(0xffffffffu, first), wants = __ballot_sync(0xffffffffu, mine >= 0);
	if (first) {
		const uint32_t at = __popc(firsts & ((1u << lane) - 1));
		t.ad[at] = mine;
		t.rows[at] = same;
		t.rank[at] = adapt_rank(s, mine);
		t.scale[at] = s.scale[mine];
	}
	if (lane == 0) {
		t.n = __popc(firsts);
		t.wants = wants;
	}
}

// Two int8 of a word, bytes `at` and at + 1, as a pair of T. By their bits: a conversion
// instruction takes 8 cycles a warp. u = the byte with its sign flipped (value + 128) in the low
// bits of 1024 (fp16) or 2^23 (fp32) is that plus u, the difference is exact, and so is an
// int8's bf16, the high half of its fp32.
template <typename T>
__device__ __forceinline__ uint32_t int8_pair(uint32_t w, int at)
{
	const uint32_t u = w ^ 0x80808080u;
	if (std::is_same<T, __half>::value) {
		const uint32_t x = __byte_perm(u, 0x64006400u, at ? 0x5352 : 0x5150);
		const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&x), __floats2half2_rn(1152.0f, 1152.0f));
		return *reinterpret_cast<const uint32_t *>(&v);
	}
	const float lo = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + at)), 8388736.0f);
	const float hi = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + at)), 8388736.0f);
	return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
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
	__shared__ AdaptTile s_tile;
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t row0 = blockIdx.x * ADAPT_ROWS, piece = blockIdx.y / a.parts, part = blockIdx.y % a.parts;
	const AdaptSet &set = a.s[blockIdx.z];
	pdl_wait();
	pdl_launch_dependents();
	if (warp == 0)
		adapt_tile(a, set, row0, s_tile);
	__syncthreads();
	const uint32_t nb = a.k / 32, each = (nb + a.pieces - 1) / a.pieces;
	const uint32_t b0 = min(piece * each, nb), b1 = min(b0 + each, nb);
	const int8_t *xq[2];
	const float *xd[2];
	bool real[2];
#pragma unroll
	for (int h = 0; h < 2; h++) {
		const uint32_t r = row0 + lane / 4 + 8 * h;
		real[h] = r < a.m;
		xq[h] = a.q + (size_t)(real[h] ? r : row0) * a.k + c * 8;
		xd[h] = a.d + (size_t)(real[h] ? r : row0) * nb;
	}
	for (uint32_t j = part; j < s_tile.n; j += a.parts) {
		const uint32_t rank = s_tile.rank[j], rows = s_tile.rows[j];
		const T *w = (const T *)set.a + ((size_t)s_tile.ad[j] * set.max_rank + lane / 4) * a.k + c * 8;
		float acc[NT][4];
#pragma unroll
		for (int n = 0; n < NT; n++)
			acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
		// the next block's loads go out before this one's products
		struct Block {
			uint2 x[2];
			float d[2];
			uint4 w[NT];
		};
		auto load = [&](Block &k, uint32_t b) {
#pragma unroll
			for (int h = 0; h < 2; h++) {
				k.x[h] = real[h] ? *(const uint2 *)(xq[h] + b * 32) : make_uint2(0, 0);
				k.d[h] = real[h] ? xd[h][b] : 0.0f;
			}
#pragma unroll
			for (int n = 0; n < NT; n++)
				k.w[n] = n * 8 + lane / 4 < rank ? *(const uint4 *)(w + (size_t)n * 8 * a.k + b * 32)
								 : make_uint4(0, 0, 0, 0);
		};
		Block now, next;
		if (b0 + warp < b1)
			load(now, b0 + warp);
		for (uint32_t b = b0 + warp; b < b1; b += ADAPT_WARPS) {
			if (b + ADAPT_WARPS < b1)
				load(next, b + ADAPT_WARPS);
			uint32_t fa[2][4];
#pragma unroll
			for (int s = 0; s < 2; s++) {
				const uint32_t x0 = s ? now.x[0].y : now.x[0].x, x1 = s ? now.x[1].y : now.x[1].x;
				fa[s][0] = int8_pair<T>(x0, 0);
				fa[s][1] = int8_pair<T>(x1, 0);
				fa[s][2] = int8_pair<T>(x0, 2);
				fa[s][3] = int8_pair<T>(x1, 2);
			}
#pragma unroll
			for (int n = 0; n < NT; n++) {
				float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
				mma_16816<T>(sum, fa[0], now.w[n].x, now.w[n].y);
				mma_16816<T>(sum, fa[1], now.w[n].z, now.w[n].w);
#pragma unroll
				for (int e = 0; e < 4; e++)
					acc[n][e] = __fmaf_rn(now.d[e >> 1], sum[e], acc[n][e]);
			}
			now = next;
		}
		__syncthreads();                  // (the last adapter's sums have been read)
#pragma unroll
		for (int n = 0; n < NT; n++)
#pragma unroll
			for (int e = 0; e < 4; e += 2)
				*(float2 *)&s_t[warp][lane / 4 + 4 * e][n * 8 + c * 2] = make_float2(acc[n][e], acc[n][e + 1]);
		__syncthreads();
		float *t = a.t + (((size_t)blockIdx.z * a.pieces + piece) * a.m + row0) * RT;
		for (uint32_t i = threadIdx.x; i < ADAPT_ROWS * RT; i += ADAPT_WARPS * 32) {
			float v = 0.0f;
#pragma unroll
			for (int x = 0; x < (int)ADAPT_WARPS; x++)
				v += s_t[x][i / RT][i % RT];
			// (behind the rank 0, which an infinite d times the sum's 0 is not)
			if (rows >> (i / RT) & 1)
				t[i] = i % RT < rank ? v : 0.0f;
		}
	}
}

// Rows row0 + r of y, r a bit of `rows`, columns [col0, end): the base's bits, by threads
// `at` of `n`; eight on their way at a time. (One after another, a prompt without an
// adapter between others took the whole launch 60 us.)
__device__ __forceinline__ void adapt_copy(const AdaptSet &s, uint32_t row0, uint32_t rows, uint32_t col0,
					   uint32_t end, uint32_t at, uint32_t n)
{
	if (!rows || s.base == s.y)
		return;
	const bool fours = s.n % 4 == 0 && !(((uintptr_t)s.base | (uintptr_t)s.y) & 15);
	const uint32_t each = fours ? 4 : 1, wide = (end - col0) / each, words = ADAPT_ROWS * wide;
	for (uint32_t x0 = at; x0 < words; x0 += 8 * n) {
		float4 v[8];
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const uint32_t x = x0 + j * n, r = x / wide, c = col0 + (x - r * wide) * each;
			if (x < words && (rows >> r & 1)) {
				const float *b = s.base + (size_t)(row0 + r) * s.n + c;
				if (fours)
					v[j] = *(const float4 *)b;
				else
					v[j].x = *b;
			}
		}
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const uint32_t x = x0 + j * n, r = x / wide, c = col0 + (x - r * wide) * each;
			if (x < words && (rows >> r & 1)) {
				float *y = s.y + (size_t)(row0 + r) * s.n + c;
				if (fours)
					*(float4 *)y = v[j];
				else
					*y = v[j].x;
			}
		}
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

// y of one tile of rows and a.cols columns of one set. An item of work is a distinct
// adapter of the tile and 8 columns; the warps take them in turn, the next one's loads
// on their way before this one's products. The ranks are permuted alike for t and B so
// that a lane's RT / 4 are consecutive.
template <typename T, int RT>
__global__ void __launch_bounds__(ADAPT_WARPS * 32)
adapt_expand_kernel(const __grid_constant__ AdaptArgs a)
{
	constexpr int SP = RT / 4, KS = RT / 8;          // ranks a lane; k steps
	__shared__ float s_t[ADAPT_ROWS][RT];
	__shared__ AdaptTile s_tile;
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t row0 = blockIdx.x * ADAPT_ROWS;
	uint32_t si = 0;
	while (blockIdx.y >= a.s[si].block_end)
		si++;
	const AdaptSet &set = a.s[si];
	const uint32_t col0 = (blockIdx.y - (si ? a.s[si - 1].block_end : 0)) * a.cols;
	pdl_wait();
	pdl_launch_dependents();
	if (warp == 0)
		adapt_tile(a, set, row0, s_tile);
	{
		const float *t = a.t + ((size_t)si * a.pieces * a.m + row0) * RT;
		const uint32_t filled = min(a.m - row0, ADAPT_ROWS) * RT;
		for (uint32_t i = threadIdx.x; i < ADAPT_ROWS * RT; i += ADAPT_WARPS * 32) {
			float v = 0.0f;
#pragma unroll 4
			for (uint32_t p = 0; p < a.left; p++)
				v += i < filled ? t[(size_t)p * a.m * RT + i] : 0.0f;
			s_t[i / RT][i % RT] = v;          // (rows that want no adapter: never used)
		}
	}
	__syncthreads();
	const uint32_t end = min(col0 + a.cols, set.n), groups = (end - col0 + 7) / 8;
	// a column of 4 ranks, beside sets whose ranks make RT, is 8 bytes of B, all of them lane 0's
	const bool narrow = set.max_rank < 8;
	// two columns a load and store
	const bool pairs = set.n % 2 == 0 && !(((uintptr_t)set.base | (uintptr_t)set.y) & 7);
	// rows of no adapter keep the base's bits
	const uint32_t there = a.m - row0 < ADAPT_ROWS ? (1u << (a.m - row0)) - 1 : 0xffffu;
	adapt_copy(set, row0, there & ~s_tile.wants, col0, end, threadIdx.x, ADAPT_WARPS * 32);
	uint32_t hi[KS][4], lo[KS][4];
#pragma unroll
	for (int ks = 0; ks < KS; ks++)
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float v = s_t[lane / 4 + 8 * (j & 1)][c * SP + 2 * ks + (j >> 1)];
			hi[ks][j] = __float_as_uint(v) & 0xffffe000u;
			// (an infinite t is infinite in hi, and its rest is 0, not inf - inf)
			const float top = __uint_as_float(hi[ks][j]);
			lo[ks][j] = v == top ? 0u : __float_as_uint(__fsub_rn(v, top));
		}
	struct Item {
		uint32_t w[SP / 2];
		float base[4];
	};
	auto load = [&](Item &it, uint32_t item) {
		const uint32_t j = item / groups, n0 = col0 + (item - j * groups) * 8, n = n0 + lane / 4;
		const uint32_t rank = s_tile.rank[j], rows = s_tile.rows[j];
		const T *src = (const T *)set.b + ((size_t)s_tile.ad[j] * set.n + n) * set.max_rank + c * SP;
#pragma unroll
		for (int x = 0; x < SP; x += SP < 8 ? SP : 8) {
			const bool ok = n < set.n && c * SP + x < rank;
			if (SP == 2) {
				it.w[0] = ok ? *(const uint32_t *)src : 0u;
			} else if (SP == 4) {
				*(uint2 *)it.w = ok ? *(const uint2 *)src : make_uint2(0, 0);
			} else if (!narrow) {
				*(uint4 *)(it.w + x / 2) = ok ? *(const uint4 *)(src + x) : make_uint4(0, 0, 0, 0);
			} else {
				const uint2 v = ok ? *(const uint2 *)src : make_uint2(0, 0);
				*(uint4 *)(it.w + x / 2) = make_uint4(v.x, v.y, 0, 0);
			}
		}
#pragma unroll
		for (int h = 0; h < 2; h++) {
			const uint32_t r = lane / 4 + 8 * h, col = n0 + c * 2;
			const float *b = set.base + (size_t)(row0 + r) * set.n + col;
			it.base[2 * h] = it.base[2 * h + 1] = 0.0f;
			if (rows >> r & 1) {
				if (pairs && col < set.n) {
					const float2 v = *(const float2 *)b;
					it.base[2 * h] = v.x;
					it.base[2 * h + 1] = v.y;
				} else if (col < set.n) {
					it.base[2 * h] = b[0];
					it.base[2 * h + 1] = col + 1 < set.n ? b[1] : 0.0f;
				}
			}
		}
	};
	const uint32_t items = s_tile.n * groups;
	Item now, next;
	if (warp < items)
		load(now, warp);
	for (uint32_t item = warp; item < items; item += ADAPT_WARPS) {
		if (item + ADAPT_WARPS < items)
			load(next, item + ADAPT_WARPS);
		const uint32_t j = item / groups, n0 = col0 + (item - j * groups) * 8;
		const uint32_t rank = s_tile.rank[j], rows = s_tile.rows[j];
		const float scale = s_tile.scale[j];
		float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
		for (int ks = 0; ks < KS; ks++) {
			T w[2];
			*(uint32_t *)w = now.w[ks];
			const uint32_t w0 = c * SP + 2 * ks < rank ? __float_as_uint(to_float<T>(w[0])) : 0u;
			const uint32_t w1 = c * SP + 2 * ks + 1 < rank ? __float_as_uint(to_float<T>(w[1])) : 0u;
			mma_tf32(low, lo[ks], w0, w1);
			mma_tf32(acc, hi[ks], w0, w1);
		}
#pragma unroll
		for (int h = 0; h < 2; h++) {
			const uint32_t r = lane / 4 + 8 * h, col = n0 + c * 2;
			if (!(rows >> r & 1) || col >= set.n)
				continue;
			const float v0 = __fadd_rn(now.base[2 * h], __fmul_rn(scale, acc[2 * h] + low[2 * h]));
			const float v1 = __fadd_rn(now.base[2 * h + 1], __fmul_rn(scale, acc[2 * h + 1] + low[2 * h + 1]));
			float *y = set.y + (size_t)(row0 + r) * set.n + col;
			if (pairs) {
				*(float2 *)y = make_float2(v0, v1);
			} else {
				y[0] = v0;
				if (col + 1 < set.n)
					y[1] = v1;
			}
		}
		now = next;
	}
}

// ---- long batches: 64 rows a CTA -----------------------------------------------------
//
// The same two steps where there are rows enough: each of four warps has 16 rows, and the
// adapter's weights pass through shared memory once for all of them (a prompt's rows
// share their adapter; where they do not, a warp without rows of an adapter sits
// it out). 2000 rows, K = N = 4096, rank 64: 16 + 3 + 25 us, against 28 + 58 by the kernels
// above (then without a sum of their own), which read every weight again for each 16 rows. Adapters one at a time, not two:
// 48 us for that, 145 against 113 for 1000 rows of 8 mixed adapters (but 38 against 42 for
// 2000 rows of one).
constexpr uint32_t ADAPT_LONG_ROWS = 64, ADAPT_STAGES = 3;

__device__ __forceinline__ void cp_async16_zero(void *dst, const void *src, bool ok)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
		     :: "r"(smem_addr(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// The distinct adapters of 64 rows, in order; by warp 0. which: the rows' in shared memory.
__device__ __forceinline__ uint32_t adapt_distinct(const int32_t *which, int32_t *list)
{
	const uint32_t lane = threadIdx.x & 31, below = (1u << lane) - 1;
	const int32_t v0 = which[lane], v1 = which[lane + 32];
	const uint32_t same0 = __match_any_sync(0xffffffffu, v0), same1 = __match_any_sync(0xffffffffu, v1);
	const bool f0 = v0 >= 0 && (int)lane == __ffs(same0) - 1;
	bool f1 = v1 >= 0 && (int)lane == __ffs(same1) - 1;
	const uint32_t firsts0 = __ballot_sync(0xffffffffu, f0);
	for (uint32_t left = firsts0; left; left &= left - 1) {
		const int32_t v = __shfl_sync(0xffffffffu, v0, __ffs(left) - 1);     // (by all lanes)
		f1 = f1 && v1 != v;
	}
	const uint32_t firsts1 = __ballot_sync(0xffffffffu, f1);
	if (f0)
		list[__popc(firsts0 & below)] = v0;
	if (f1)
		list[__popc(firsts0) + __popc(firsts1 & below)] = v1;
	return __popc(firsts0) + __popc(firsts1);
}

// The weights of two of the tile's adapters pass together (a tile where one request's rows end
// and the next one's begin takes as long as others so): each warp takes those that
// its rows want.
constexpr uint32_t ADAPT_PASS = 2;

template <int RT>
struct AdaptLong {
	static constexpr uint32_t A_STAGES = 3, A_PART = RT * 128, A_STAGE = ADAPT_PASS * A_PART;      // 64 k of a rank
	static constexpr uint32_t B_COLS = 64, B_PITCH = RT * 2 + 16;
	static constexpr uint32_t B_PART = B_COLS * B_PITCH, B_STAGE = ADAPT_PASS * B_PART;
	static constexpr size_t A_SMEM = A_STAGES * A_STAGE, B_SMEM = ADAPT_STAGES * B_STAGE;
};

struct AdaptLongTile {
	int32_t which[ADAPT_LONG_ROWS], list[ADAPT_LONG_ROWS];
	uint32_t rank[ADAPT_LONG_ROWS];
	float scale[ADAPT_LONG_ROWS];
	uint32_t n;
};

// by the CTA; ends with a barrier
__device__ __forceinline__ void adapt_long_tile(const AdaptArgs &a, const AdaptSet &s, uint32_t tile0,
						AdaptLongTile &t)
{
	const uint32_t lane = threadIdx.x & 31;
	if (threadIdx.x < ADAPT_LONG_ROWS)
		t.which[threadIdx.x] = adapt_which(a, s, tile0 + threadIdx.x);
	__syncthreads();
	if (threadIdx.x < 32) {
		const uint32_t n = adapt_distinct(t.which, t.list);
		__syncwarp();
		for (uint32_t j = lane; j < n; j += 32) {
			t.rank[j] = adapt_rank(s, t.list[j]);
			t.scale[j] = s.scale[t.list[j]];
		}
		if (lane == 0)
			t.n = n;
	}
	__syncthreads();
}

template <typename T, int RT>
__global__ void __launch_bounds__(ADAPT_WARPS * 32, 3)
adapt_shrink_long_kernel(const __grid_constant__ AdaptArgs a)
{
	using L = AdaptLong<RT>;
	constexpr int NT = RT / 8;
	constexpr uint32_t NS = L::A_STAGES;
	extern __shared__ __align__(128) uint8_t adapt_raw[];
	__shared__ AdaptLongTile s_tile;
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t tile0 = blockIdx.x * ADAPT_LONG_ROWS, row0 = tile0 + warp * ADAPT_ROWS, piece = blockIdx.y;
	const AdaptSet &set = a.s[blockIdx.z];
	pdl_wait();
	pdl_launch_dependents();
	adapt_long_tile(a, set, tile0, s_tile);
	// the piece in steps of two 32-blocks
	const uint32_t nb = a.k / 32, steps_all = (nb + 1) / 2, each = (steps_all + a.pieces - 1) / a.pieces;
	const uint32_t s0 = min(piece * each, steps_all), steps = min(s0 + each, steps_all) - s0;
	const int32_t mine = s_tile.which[warp * ADAPT_ROWS + (lane & 15)];
	const int8_t *xq[2];
	const float *xd[2];
#pragma unroll
	for (int h = 0; h < 2; h++) {
		const uint32_t r = min(row0 + lane / 4 + 8 * h, a.m - 1);     // (rows past the last: not kept)
		xq[h] = a.q + (size_t)r * a.k + c * 8;
		xd[h] = a.d + (size_t)r * nb;
	}
	float *t = a.t + (((size_t)blockIdx.z * a.pieces + piece) * a.m + row0) * RT;
	for (uint32_t j = 0; j < s_tile.n; j += ADAPT_PASS) {
		const uint32_t two = min(s_tile.n - j, ADAPT_PASS);
		const int32_t ad0 = s_tile.list[j], ad1 = two > 1 ? s_tile.list[j + 1] : -2;
		const uint32_t rows0 = __ballot_sync(0xffffffffu, mine == ad0) & 0xffffu;
		const uint32_t rows1 = __ballot_sync(0xffffffffu, mine == ad1) & 0xffffu;
		const uint32_t rows = rows0 | rows1;
		auto fetch = [&](uint32_t s) {
			// 8 words of 16 bytes a rank, an odd rank's halves swapped (other banks)
			for (uint32_t x = threadIdx.x; s < steps && x < two * RT * 8; x += ADAPT_WARPS * 32) {
				const uint32_t r = x / 8 % RT, k = (s0 + s) * 64 + x % 8 * 8;
				const bool ok = r < set.max_rank && k < a.k;
				const size_t row = (size_t)(x / 8 < RT ? ad0 : ad1) * set.max_rank + (ok ? r : 0);
				cp_async16_zero(adapt_raw + s % NS * L::A_STAGE + x / 8 * 128 + ((x % 8) ^ (r & 1) * 4) * 16,
						(const T *)set.a + row * a.k + (ok ? k : 0), ok);
			}
			asm volatile("cp.async.commit_group;" ::: "memory");
		};
		float acc[NT][4];
#pragma unroll
		for (int n = 0; n < NT; n++)
			acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
		struct Rows {
			uint2 x[2][2];        // [block][row]
			float d[2][2];
		};
		auto load = [&](Rows &v, uint32_t s) {
#pragma unroll
			for (int b = 0; b < 2; b++)
#pragma unroll
				for (int h = 0; h < 2; h++) {
					const uint32_t block = (s0 + s) * 2 + b;
					const bool ok = s < steps && block < nb;
					v.x[b][h] = ok ? *(const uint2 *)(xq[h] + block * 32) : make_uint2(0, 0);
					v.d[b][h] = ok ? xd[h][block] : 0.0f;
				}
		};
		__syncthreads();                  // (the last adapters' stages have been read)
		Rows buf[NS];
#pragma unroll
		for (uint32_t s = 0; s < NS - 1; s++) {
			fetch(s);
			if (rows)
				load(buf[s], s);
		}
		for (uint32_t s4 = 0; s4 < steps; s4 += NS)
#pragma unroll
			for (uint32_t u = 0; u < NS; u++) {
				const uint32_t s = s4 + u;
				if (s >= steps)
					break;
				asm volatile("cp.async.wait_group %0;" :: "n"((int)NS - 2) : "memory");
				__syncthreads();
				fetch(s + NS - 1);
				if (!rows)
					continue;
				load(buf[(u + NS - 1) % NS], s + NS - 1);
				const Rows &now = buf[u];
				uint32_t fa[2][2][4];
#pragma unroll
				for (int b = 0; b < 2; b++)
#pragma unroll
					for (int x = 0; x < 2; x++) {
						const uint32_t x0 = x ? now.x[b][0].y : now.x[b][0].x, x1 = x ? now.x[b][1].y : now.x[b][1].x;
						fa[b][x][0] = int8_pair<T>(x0, 0);
						fa[b][x][1] = int8_pair<T>(x1, 0);
						fa[b][x][2] = int8_pair<T>(x0, 2);
						fa[b][x][3] = int8_pair<T>(x1, 2);
					}
#pragma unroll 1
				for (uint32_t g = 0; g < two; g++) {
					const uint32_t in = g ? rows1 : rows0;
					if (!in)
						continue;
					const bool take[2] = {(in >> (lane / 4) & 1) != 0, (in >> (lane / 4 + 8) & 1) != 0};
					const uint8_t *stage = adapt_raw + u * L::A_STAGE + g * L::A_PART;
#pragma unroll
					for (int b = 0; b < 2; b++)
#pragma unroll
						for (int n = 0; n < NT; n++) {
							const uint32_t r = n * 8 + lane / 4;
							const uint4 v = *(const uint4 *)(stage + r * 128 + ((b * 4 + c) ^ (r & 1) * 4) * 16);
							float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
							mma_16816<T>(sum, fa[b][0], v.x, v.y);
							mma_16816<T>(sum, fa[b][1], v.z, v.w);
#pragma unroll
							for (int e = 0; e < 4; e++)
								acc[n][e] = take[e >> 1] ? __fmaf_rn(now.d[b][e >> 1], sum[e], acc[n][e]) : acc[n][e];
						}
				}
			}
		asm volatile("cp.async.wait_group 0;" ::: "memory");
		// (what lies behind a rank reached its own columns of t only: 0)
#pragma unroll
		for (int h = 0; h < 2; h++) {
			const uint32_t r = lane / 4 + 8 * h, rank = s_tile.rank[j + (rows1 >> r & 1)];
			if (rows >> r & 1)
#pragma unroll
				for (int n = 0; n < NT; n++) {
					const uint32_t i = n * 8 + c * 2;
					*(float2 *)(t + r * RT + i) = make_float2(i < rank ? acc[n][2 * h] : 0.0f,
										  i + 1 < rank ? acc[n][2 * h + 1] : 0.0f);
				}
		}
	}
}

// The pieces of t added up, in order, into the first: every CTA of the columns reads them
__global__ void __launch_bounds__(256)
adapt_sum_kernel(float4 *t, uint32_t pieces, uint32_t each)
{
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t i = blockIdx.x * 256 + threadIdx.x;
	if (i >= each)
		return;
	float4 *at = t + (size_t)blockIdx.y * pieces * each + i;
	float4 v = at[0];
#pragma unroll 8
	for (uint32_t p = 1; p < pieces; p++) {
		const float4 u = at[(size_t)p * each];
		v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
	}
	at[0] = v;
}

// t as a sum of numbers of B's type, for exact products with B: fp16 in two parts, the row scaled by a
// power of two so that its largest is in [2^13, 2^14) (what is lost is 2^-24 of a term, or 2^-38
// of the row's largest), bf16 in three (2^-27). Against two tf32 parts that is 2 or 3 MMAs for 16
// ranks, not 4 of half the rate, and B needs no conversion.
template <typename T>
__host__ __device__ constexpr int adapt_parts()
{
	return std::is_same<T, __half>::value ? 2 : 3;
}

template <typename T>
__device__ __forceinline__ float adapt_largest()
{
	return std::is_same<T, __half>::value ? 65504.0f : __uint_as_float(0x7f7f0000u);
}

// the power of two for a row whose largest is `top`; 1 where that is 0. (Of inf, 2^-114: the row's finite
// numbers stay finite in 16 bits.)
__device__ __forceinline__ float adapt_lift(float top)
{
	const int e = min((int)(__float_as_uint(top) >> 23 & 255) - 127, 127);
	if (!(top > 0.0f))
		return 1.0f;
	const int x = min(max(13 - e, -126), 126);
	return __uint_as_float((uint32_t)(x + 127) << 23);
}

template <typename T, int RT>
__global__ void __launch_bounds__(ADAPT_WARPS * 32, 3)
adapt_expand_long_kernel(const __grid_constant__ AdaptArgs a)
{
	using L = AdaptLong<RT>;
	constexpr int SP = RT / 4, PAIRS = SP / 2, KS = RT < 16 ? 1 : RT / 16;      // ranks a lane; k steps
	constexpr int PARTS = adapt_parts<T>();
	extern __shared__ __align__(128) uint8_t adapt_raw[];
	__shared__ AdaptLongTile s_tile;
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
	const uint32_t tile0 = blockIdx.x * ADAPT_LONG_ROWS, row0 = tile0 + warp * ADAPT_ROWS;
	uint32_t si = 0;
	while (blockIdx.y >= a.s[si].block_end)
		si++;
	const AdaptSet &set = a.s[si];
	const uint32_t col0 = (blockIdx.y - (si ? a.s[si - 1].block_end : 0)) * a.cols;
	const uint32_t end = min(col0 + a.cols, set.n), steps = (end - col0 + L::B_COLS - 1) / L::B_COLS;
	const bool fours = set.n % 4 == 0 && !(((uintptr_t)set.base | (uintptr_t)set.y) & 15);
	pdl_wait();
	pdl_launch_dependents();
	adapt_long_tile(a, set, tile0, s_tile);
	// this warp's t, straight into the fragments: of the 16 ranks of k step s lane c has ranks
	// c SP + 4 s ... + 3, of t and of B alike
	uint32_t part[PARTS][KS][4];
	float back[2];
#pragma unroll
	for (int h = 0; h < 2; h++) {
		const uint32_t r = row0 + lane / 4 + 8 * h;
		float v[SP];
#pragma unroll
		for (int i = 0; i < SP; i++)
			v[i] = 0.0f;
		if (r < a.m) {
			const float *t = a.t + ((size_t)si * a.pieces * a.m + r) * RT + c * SP;
#pragma unroll
			for (int i = 0; i < SP; i += SP < 4 ? 2 : 4) {
				if (SP < 4)
					*(float2 *)v = *(const float2 *)t;
				else
					*(float4 *)(v + i) = *(const float4 *)(t + i);
			}
		}
		back[h] = 1.0f;
		if (PARTS == 2) {
			float top = 0.0f;
#pragma unroll
			for (int i = 0; i < SP; i++)
				top = fmaxf(top, fabsf(v[i]));
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
			const float lift = adapt_lift(top);
			back[h] = __uint_as_float((254u << 23) - __float_as_uint(lift));      // 1 / lift
#pragma unroll
			for (int i = 0; i < SP; i++)
				v[i] = __fmul_rn(v[i], lift);
		}
#pragma unroll
		for (int p = 0; p < PARTS; p++)
#pragma unroll
			for (int i = 0; i < 2 * KS; i++) {
				uint32_t two = 0;
				if (i < PAIRS) {
					// (no part but the last is infinite, or the rest would be inf - inf: what is
					// beyond T, infinities and NaN too, is left to the last)
					float x0 = v[2 * i], x1 = v[2 * i + 1];
					if (p < PARTS - 1) {
						x0 = fminf(fmaxf(x0, -adapt_largest<T>()), adapt_largest<T>());
						x1 = fminf(fmaxf(x1, -adapt_largest<T>()), adapt_largest<T>());
					}
					two = pack_pair<T>(x0, x1);
					T x[2];
					*(uint32_t *)x = two;
					v[2 * i] = __fsub_rn(v[2 * i], to_float<T>(x[0]));
					v[2 * i + 1] = __fsub_rn(v[2 * i + 1], to_float<T>(x[1]));
				}
				part[p][i / 2][h + 2 * (i % 2)] = two;
			}
	}
	const int32_t mine = s_tile.which[warp * ADAPT_ROWS + (lane & 15)];
	const uint32_t wants = __ballot_sync(0xffffffffu, mine >= 0) & 0xffffu;
	// rows of no adapter keep the base's bits
	const uint32_t there = row0 >= a.m ? 0 : a.m - row0 < ADAPT_ROWS ? (1u << (a.m - row0)) - 1 : 0xffffu;
	adapt_copy(set, row0, there & ~wants, col0, end, lane, 32);
	for (uint32_t j = 0; j < s_tile.n; j += ADAPT_PASS) {
		const uint32_t two = min(s_tile.n - j, ADAPT_PASS);
		const int32_t ad0 = s_tile.list[j], ad1 = two > 1 ? s_tile.list[j + 1] : -2;
		const uint32_t rows0 = __ballot_sync(0xffffffffu, mine == ad0) & 0xffffu;
		const uint32_t rows1 = __ballot_sync(0xffffffffu, mine == ad1) & 0xffffu;
		const uint32_t rows = rows0 | rows1;
		// what is behind a rank counts as 0: words of 8 by the copies, the rest by hand
		const uint32_t rank0 = s_tile.rank[j], rank1 = two > 1 ? s_tile.rank[j + 1] : 0;
		const bool ragged = (rank0 | rank1) % 8;
		auto fetch = [&](uint32_t s) {
			constexpr uint32_t WORDS = RT / 8;
			for (uint32_t x = threadIdx.x; s < steps && x < two * L::B_COLS * WORDS; x += ADAPT_WARPS * 32) {
				const uint32_t r = x / WORDS, i = x % WORDS, n = col0 + s * L::B_COLS + r % L::B_COLS;
				const bool first = r < L::B_COLS, ok = n < end && i * 8 < (first ? rank0 : rank1);
				const size_t col = (size_t)(first ? ad0 : ad1) * set.n + (ok ? n : 0);
				cp_async16_zero(adapt_raw + s % ADAPT_STAGES * L::B_STAGE + r * L::B_PITCH + i * 16,
						(const T *)set.b + col * set.max_rank + (ok ? i * 8 : 0), ok);
			}
			asm volatile("cp.async.commit_group;" ::: "memory");
		};
		// Columns are dealt to the MMAs so that a thread has runs of four: column
		// 16 x + 4 (n / 2) + 2 (g % 2) + n % 2 is the n-th of group g, x = g / 2, so of
		// groups 2 x and 2 x + 1 thread c has 16 x + 4 c ... + 3. A row's 64 bytes then
		// move together (not 32, as in the order of the fragments). The bases of a step are on
		// their way from the step before.
		struct Bases {
			float v[4][2][4];
		};
		auto load = [&](Bases &to, uint32_t s) {
#pragma unroll
			for (int x = 0; x < 4; x++)
#pragma unroll
				for (int h = 0; h < 2; h++) {
					const uint32_t r = lane / 4 + 8 * h, col = col0 + s * L::B_COLS + c * 4 + x * 16;
					const float *b = set.base + (size_t)(row0 + r) * set.n + col;
					const bool mine_too = rows >> r & 1;
					float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
					if (fours) {
						if (mine_too && col < end)
							v = *(const float4 *)b;
					} else if (mine_too) {
						v.x = col < end ? b[0] : 0.0f;
						v.y = col + 1 < end ? b[1] : 0.0f;
						v.z = col + 2 < end ? b[2] : 0.0f;
						v.w = col + 3 < end ? b[3] : 0.0f;
					}
					*(float4 *)to.v[x][h] = v;
				}
		};
		__syncthreads();                  // (the last adapters' stages have been read)
		for (uint32_t s = 0; s < ADAPT_STAGES - 1; s++)
			fetch(s);
		auto step = [&](const Bases &now, Bases &next, uint32_t s) {
			if (s + 1 < steps)
				load(next, s + 1);
			asm volatile("cp.async.wait_group %0;" :: "n"((int)ADAPT_STAGES - 2) : "memory");
			__syncthreads();
			uint8_t *stage0 = adapt_raw + s % ADAPT_STAGES * L::B_STAGE;
			if (ragged) {
				for (uint32_t r = threadIdx.x; r < two * L::B_COLS; r += ADAPT_WARPS * 32) {
					const uint32_t rank = r < L::B_COLS ? rank0 : rank1;
					for (uint32_t i = rank; i % 8; i++)
						*(uint16_t *)(stage0 + r * L::B_PITCH + i * 2) = 0;
				}
				__syncthreads();
			}
			fetch(s + ADAPT_STAGES - 1);
#pragma unroll 1
			for (uint32_t which = 0; which < two; which++) {
				const uint32_t in = which ? rows1 : rows0;
				if (!in)
					continue;
				const float scale = s_tile.scale[j + which];
				const uint8_t *stage = stage0 + which * L::B_PART;
#pragma unroll
				for (int x = 0; x < 4; x++) {
					float acc[2][4], low[2][4];
					uint32_t wv[2][PAIRS];
#pragma unroll
					for (int g = 0; g < 2; g++) {
						const uint32_t n = lane / 4, col = 16 * x + 4 * (n / 2) + 2 * g + n % 2;
						const uint8_t *src = stage + col * L::B_PITCH + c * SP * 2;
#pragma unroll
						for (int i = 0; i < PAIRS; i += PAIRS < 4 ? PAIRS : 4) {
							if (PAIRS == 1)
								wv[g][0] = *(const uint32_t *)src;
							else if (PAIRS == 2)
								*(uint2 *)wv[g] = *(const uint2 *)src;
							else
								*(uint4 *)(wv[g] + i) = *(const uint4 *)(src + i * 4);
						}
#pragma unroll
						for (int e = 0; e < 4; e++)
							acc[g][e] = low[g][e] = 0.0f;
					}
#pragma unroll
					for (int ks = 0; ks < KS; ks++)
#pragma unroll
						for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
							for (int g = 0; g < 2; g++)
								mma_16816<T>(p ? low[g] : acc[g], part[p][ks], wv[g][2 * ks],
									     2 * ks + 1 < PAIRS ? wv[g][(2 * ks + 1) % PAIRS] : 0u);
#pragma unroll
					for (int h = 0; h < 2; h++) {
						const uint32_t r = lane / 4 + 8 * h, col = col0 + s * L::B_COLS + c * 4 + x * 16;
						if (!(in >> r & 1))
							continue;
						float v[4];
#pragma unroll
						for (int e = 0; e < 4; e++) {
							const float sum = acc[e / 2][2 * h + e % 2] + low[e / 2][2 * h + e % 2];
							v[e] = __fadd_rn(now.v[x][h][e], __fmul_rn(scale, __fmul_rn(sum, back[h])));
						}
						float *y = set.y + (size_t)(row0 + r) * set.n + col;
						if (fours) {
							if (col < end)
								*(float4 *)y = make_float4(v[0], v[1], v[2], v[3]);
						} else {
#pragma unroll
							for (int e = 0; e < 4; e++)
								if (col + e < end)
									y[e] = v[e];
						}
					}
				}
			}
		};
		// (two buffers by name: a copy of one into the other would wait for its loads)
		Bases even, odd;
		load(even, 0);
		for (uint32_t s = 0; s < steps; s += 2) {
			step(even, odd, s);
			if (s + 1 < steps)
				step(odd, even, s + 1);
		}
		asm volatile("cp.async.wait_group 0;" ::: "memory");
	}
}

} // namespace cgpu
