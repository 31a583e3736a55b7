// SPDX-License-Identifier: GPL-2.0-or-later
// A cache of K and V in pages (charsiu_gpu_pages_*): the bookkeeping that a
// batch's sequences need (grow, fork, free, compact), and RoPE with the append
// of new positions.
//
// The tables and reference counts live on the device and every decision about
// them is made there, so a captured graph can replay a step whatever the
// lengths have become. Fresh pages are the free ones of the lowest numbers: a
// scan of the reference counts finds them, and its order (not the order in
// which threads happen to run) says which item gets which page.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "batch_checks.h"
#include "charsiu_gpu.h"
#include "ptx.cuh"

namespace cgpu {

constexpr int PAGES_PLAN_THREADS = 1024;

// The words of `work`: [0] the refused items so far; [1] the moves of a compaction.
// Then the lists that a planner leaves for the kernel after it:
//   fork     four words an item: source slot (-1: refused), full pages, filled
//            positions of the last page, its fresh page
//   compact  (from, to) of every move; and, n_pages words on, where a page went
//   grow     the fresh pages
constexpr uint32_t PAGES_WORK_LIST = 16;
constexpr uint32_t PAGES_FORK_WORDS = 4;

inline size_t pages_work_words(uint32_t n_pages)
{
	return PAGES_WORK_LIST + (size_t)PAGES_FORK_WORDS * PAGES_MAX_ITEMS + 2 * (size_t)n_pages;
}

// exclusive prefix sum over the CTA's PAGES_PLAN_THREADS threads; *total in all.
// sh: 32 words. Barriers before and after, so sh can be used again at once.
__device__ __forceinline__ uint32_t pages_scan(uint32_t v, uint32_t *sh, uint32_t *total)
{
	const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
	uint32_t inc = v;
	for (int o = 1; o < 32; o <<= 1) {
		const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
		if (lane >= (uint32_t)o)
			inc += y;
	}
	__syncthreads();
	if (lane == 31)
		sh[wid] = inc;
	__syncthreads();
	uint32_t w = sh[lane], winc = w;
	for (int o = 1; o < 32; o <<= 1) {
		const uint32_t y = __shfl_up_sync(0xffffffffu, winc, o);
		if (lane >= (uint32_t)o)
			winc += y;
	}
	const uint32_t before = __shfl_sync(0xffffffffu, winc - w, wid);
	*total = __shfl_sync(0xffffffffu, winc, 31);
	return before + inc - v;
}

// The first `want` free pages, in order, into list (global memory); returns how
// many there are, at most `want`. The whole CTA; ends with a barrier.
__device__ __forceinline__ uint32_t pages_find_free(const int32_t *ref, uint32_t n_pages,
						    uint32_t want, int32_t *list, uint32_t *sh)
{
	constexpr uint32_t EACH = 4;
	uint32_t found = 0;
	for (uint32_t p0 = 0; p0 < n_pages && found < want; p0 += EACH * PAGES_PLAN_THREADS) {
		const uint32_t p = p0 + threadIdx.x * EACH;
		uint32_t mask = 0;
#pragma unroll
		for (uint32_t j = 0; j < EACH; j++)
			if (p + j < n_pages && ref[p + j] == 0)
				mask |= 1u << j;
		uint32_t here;
		uint32_t at = found + pages_scan(__popc(mask), sh, &here);
		for (; mask && at < want; mask &= mask - 1, at++)
			list[at] = (int32_t)(p + __ffs(mask) - 1);
		found += here;
	}
	__syncthreads();
	return found < want ? found : want;
}

// Whether an item before this one lists the same slot; slots in shared memory.
__device__ __forceinline__ bool pages_listed_before(const int32_t *slots, uint32_t i)
{
	bool dup = false;
	for (uint32_t j = 0; j < i; j++)
		dup |= slots[j] == slots[i];
	return dup;
}

__device__ __forceinline__ bool pages_slot_ok(const charsiu_gpu_pages &p, int32_t slot)
{
	return slot >= 0 && (uint32_t)slot < p.n_seq;
}

__global__ void __launch_bounds__(PAGES_PLAN_THREADS)
pages_grow_kernel(const __grid_constant__ charsiu_gpu_pages p, const int32_t *__restrict__ slots,
		  uint32_t n, uint32_t add)
{
	__shared__ uint32_t sh[32];
	__shared__ int32_t s_slot[PAGES_MAX_ITEMS];
	__shared__ uint32_t s_at[PAGES_MAX_ITEMS], s_have[PAGES_MAX_ITEMS], s_need[PAGES_MAX_ITEMS];
	const uint32_t i = threadIdx.x;
	pdl_wait();
	pdl_launch_dependents();
	if (i < n)
		s_slot[i] = slots[i];
	__syncthreads();
	uint32_t need = 0, have = 0;
	int64_t grown = 0;
	bool ok = false;
	if (i < n && pages_slot_ok(p, s_slot[i]) && !pages_listed_before(s_slot, i)) {
		const int64_t len = p.len[s_slot[i]];
		grown = len + add;
		if (len >= 0 && grown <= (int64_t)p.max_pages * p.page && grown <= 0x7fffffff) {
			ok = true;
			have = (uint32_t)((len + p.page - 1) / p.page);
			need = (uint32_t)((grown + p.page - 1) / p.page) - have;
			// (more than the pool has is more, however many: the sum of 1024 needs stays in 32 bits)
			need = need <= p.n_pages ? need : p.n_pages + 1;
		}
	}
	uint32_t total;
	const uint32_t at = pages_scan(need, sh, &total);
	int32_t *list = p.work + PAGES_WORK_LIST;
	const uint32_t want = total < p.n_pages ? total : p.n_pages;
	const uint32_t found = want ? pages_find_free(p.ref, p.n_pages, want, list, sh) : 0;
	if (need && at + need > found) {
		ok = false;
		need = 0;
	}
	if (ok)
		p.len[s_slot[i]] = (int32_t)grown;
	else if (i < n)
		atomicAdd(&p.work[0], 1);
	if (!want)
		return;
	if (i < n) {
		s_at[i] = at;
		s_have[i] = have;
		s_need[i] = need;
	}
	__syncthreads();
	for (uint32_t it = i >> 5; it < n; it += PAGES_PLAN_THREADS / 32) {
		int32_t *row = p.table + (size_t)(s_need[it] ? s_slot[it] : 0) * p.max_pages + s_have[it];
		for (uint32_t j = i & 31; j < s_need[it]; j += 32) {
			const int32_t page = list[s_at[it] + j];
			row[j] = page;
			p.ref[page] = 1;
		}
	}
}

// Which forks go ahead, and the fresh page of each that needs one.
__global__ void __launch_bounds__(PAGES_PLAN_THREADS)
pages_fork_plan_kernel(const __grid_constant__ charsiu_gpu_pages p,
		       const int32_t *__restrict__ from, const int32_t *__restrict__ to, uint32_t n)
{
	__shared__ uint32_t sh[32];
	__shared__ int32_t s_to[PAGES_MAX_ITEMS], s_free[PAGES_MAX_ITEMS];
	const uint32_t i = threadIdx.x;
	pdl_wait();
	pdl_launch_dependents();
	if (i < n)
		s_to[i] = to[i];
	__syncthreads();
	const int32_t src = i < n ? from[i] : -1;
	uint32_t rest = 0, whole = 0;
	bool ok = false;
	int32_t len = 0;
	if (i < n && pages_slot_ok(p, s_to[i]) && pages_slot_ok(p, src) && p.len[s_to[i]] == 0 &&
	    !pages_listed_before(s_to, i)) {
		len = p.len[src];
		whole = (uint32_t)len / p.page;
		rest = (uint32_t)len % p.page;
		ok = len >= 0 && whole + (rest != 0) <= p.max_pages;
	}
	uint32_t total;
	const uint32_t at = pages_scan(ok && rest, sh, &total);     // (its barriers: every len read)
	int32_t *list = p.work + PAGES_WORK_LIST + PAGES_FORK_WORDS * PAGES_MAX_ITEMS;
	const uint32_t want = total < p.n_pages ? total : p.n_pages;
	const uint32_t found = want ? pages_find_free(p.ref, p.n_pages, want, list, sh) : 0;
	if (i < found)
		s_free[i] = list[i];
	__syncthreads();
	if (i >= n)
		return;
	if (ok && rest && at >= found)
		ok = false;
	int32_t *item = p.work + PAGES_WORK_LIST + PAGES_FORK_WORDS * i;
	item[0] = ok ? src : -1;
	item[1] = (int32_t)whole;
	item[2] = (int32_t)rest;
	item[3] = ok && rest ? s_free[at] : -1;
	if (ok)
		p.len[s_to[i]] = len;
	else
		atomicAdd(&p.work[0], 1);
}

// Positions [0, rows) of page `from` to page `to`, K (which 0) or V of one layer,
// by the CTA. The elements of a page come in runs without a gap: the whole
// page, one a head or position, or one a row of head_dim.
__device__ __forceinline__ void pages_copy(const charsiu_gpu_pages &p, uint32_t layer,
					   uint32_t which, uint32_t from, uint32_t to, uint32_t rows)
{
	uint8_t *base = (uint8_t *)(which ? p.v : p.k) + 2 * layer * p.layer_stride;
	const uint4 *src = (const uint4 *)(base + 2 * from * p.page_stride);
	uint4 *dst = (uint4 *)(base + 2 * to * p.page_stride);
	const uint32_t hv = p.head_dim / 8;              // 16-byte words a row of head_dim
	uint32_t run = hv, inner = 1;
	uint64_t s_in = 0, s_out = 0;                      // strides of the runs, in words
	if (p.head_stride == p.head_dim) {                 // [position][head]
		run = hv * p.n_head_kv;
		s_out = p.pos_stride / 8;
		if (p.pos_stride == (uint64_t)p.head_dim * p.n_head_kv)
			run *= rows;
	} else if (p.pos_stride == p.head_dim) {           // [head][position]
		run = hv * rows;
		s_out = p.head_stride / 8;
	} else {
		inner = p.n_head_kv;
		s_in = p.head_stride / 8;
		s_out = p.pos_stride / 8;
	}
	// (four words on their way at a time: a load behind a store would wait for the one before it)
	const uint32_t total = rows * p.n_head_kv * hv;
	for (uint32_t j0 = threadIdx.x; j0 < total; j0 += 4 * blockDim.x) {
		uint64_t o[4];
		uint4 v[4];
#pragma unroll
		for (uint32_t e = 0; e < 4; e++) {
			const uint32_t j = j0 + e * blockDim.x;
			if (run == total) {
				o[e] = j;
			} else {
				const uint32_t r = j / run, w = j - r * run;
				o[e] = (r / inner) * s_out + (r % inner) * s_in + w;
			}
			if (j < total)
				v[e] = src[o[e]];
		}
#pragma unroll
		for (uint32_t e = 0; e < 4; e++)
			if (j0 + e * blockDim.x < total)
				dst[o[e]] = v[e];
	}
}

// (256 forks of 32 sequences, 16 of 32 positions of the last page on average, 16 layers of 8 heads
// of 64: the whole beam step 47 us, with one word a thread at a time 55, with eight 60; 134 MB are
// written in runs of 2 KB, 34 us of it cold. The planners, one
// CTA each, take 4 to 7 us by their chain of loads: slots, lengths, reference counts.)
//
// The forks that pages_fork_plan_kernel let through: one CTA per (item, layer, K
// or V) copies the filled positions of the last page, and the first CTA of
// each item also fills the new table row and counts the pages.
__global__ void __launch_bounds__(256)
pages_fork_kernel(const __grid_constant__ charsiu_gpu_pages p, const int32_t *__restrict__ to)
{
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t i = blockIdx.x, part = blockIdx.y;
	const int32_t *item = p.work + PAGES_WORK_LIST + PAGES_FORK_WORDS * i;
	const int32_t src = item[0], rest = item[2], fresh = item[3];
	if (src < 0)
		return;
	const uint32_t whole = (uint32_t)item[1];
	const int32_t *row = p.table + (size_t)src * p.max_pages;
	if (part == 0) {
		int32_t *out = p.table + (size_t)to[i] * p.max_pages;
		for (uint32_t j = threadIdx.x; j < whole; j += blockDim.x) {
			const int32_t page = row[j];
			out[j] = page;
			if ((uint32_t)page < p.n_pages)
				atomicAdd(&p.ref[page], 1);
		}
		if (threadIdx.x == 0 && rest) {
			out[whole] = fresh;
			p.ref[fresh] = 1;
		}
	}
	if (rest && (uint32_t)row[whole] < p.n_pages)
		pages_copy(p, part >> 1, part & 1, (uint32_t)row[whole], (uint32_t)fresh, (uint32_t)rest);
}

// One CTA a listed slot. Whoever takes a slot's length frees its pages, so a
// slot listed twice is freed once.
__global__ void __launch_bounds__(128)
pages_free_kernel(const __grid_constant__ charsiu_gpu_pages p, const int32_t *__restrict__ slots)
{
	__shared__ int32_t s_len;
	pdl_wait();
	pdl_launch_dependents();
	const int32_t slot = slots[blockIdx.x];
	if (!pages_slot_ok(p, slot)) {
		if (threadIdx.x == 0)
			atomicAdd(&p.work[0], 1);
		return;
	}
	if (threadIdx.x == 0)
		s_len = atomicExch(&p.len[slot], 0);
	__syncthreads();
	if (s_len <= 0)
		return;
	uint32_t held = (uint32_t)(((int64_t)s_len + p.page - 1) / p.page);
	held = held < p.max_pages ? held : p.max_pages;
	const int32_t *row = p.table + (size_t)slot * p.max_pages;
	for (uint32_t j = threadIdx.x; j < held; j += blockDim.x)
		if ((uint32_t)row[j] < p.n_pages)
			atomicSub(&p.ref[row[j]], 1);
}

// What moves where: the i-th live page from `live` on to the i-th free one below.
__global__ void __launch_bounds__(PAGES_PLAN_THREADS)
pages_compact_plan_kernel(const __grid_constant__ charsiu_gpu_pages p, int32_t *n_live)
{
	constexpr uint32_t EACH = 4, STEP = EACH * PAGES_PLAN_THREADS;
	__shared__ uint32_t sh[32];
	pdl_wait();
	pdl_launch_dependents();
	uint32_t mine = 0, live, none;
	for (uint32_t p0 = threadIdx.x * EACH; p0 < p.n_pages; p0 += STEP)
#pragma unroll
		for (uint32_t j = 0; j < EACH; j++)
			mine += p0 + j < p.n_pages && p.ref[p0 + j] != 0;
	pages_scan(mine, sh, &live);
	int32_t *moves = p.work + PAGES_WORK_LIST;
	int32_t *went = moves + PAGES_FORK_WORDS * PAGES_MAX_ITEMS + p.n_pages;
	// both kinds in one pass over their own ranges, in order
	uint32_t holes = 0, movers = 0;
	for (uint32_t p0 = 0; p0 < live; p0 += STEP) {
		const uint32_t at0 = p0 + threadIdx.x * EACH;
		uint32_t mask = 0;
#pragma unroll
		for (uint32_t j = 0; j < EACH; j++)
			if (at0 + j < live && p.ref[at0 + j] == 0)
				mask |= 1u << j;
		uint32_t at = holes + pages_scan(__popc(mask), sh, &none);
		for (; mask; mask &= mask - 1, at++)
			moves[2 * at + 1] = (int32_t)(at0 + __ffs(mask) - 1);
		holes += none;
	}
	for (uint32_t p0 = live; p0 < p.n_pages; p0 += STEP) {
		const uint32_t at0 = p0 + threadIdx.x * EACH;
		uint32_t mask = 0;
#pragma unroll
		for (uint32_t j = 0; j < EACH; j++)
			if (at0 + j < p.n_pages && p.ref[at0 + j] != 0)
				mask |= 1u << j;
		uint32_t at = movers + pages_scan(__popc(mask), sh, &none);
		for (; mask; mask &= mask - 1, at++)
			moves[2 * at] = (int32_t)(at0 + __ffs(mask) - 1);
		movers += none;
	}
	__syncthreads();
	for (uint32_t j = threadIdx.x; j < movers; j += PAGES_PLAN_THREADS) {
		const int32_t a = moves[2 * j], b = moves[2 * j + 1];
		went[a] = b;
		p.ref[b] = p.ref[a];
		p.ref[a] = 0;
	}
	if (threadIdx.x == 0) {
		p.work[1] = (int32_t)movers;
		p.work[2] = (int32_t)live;
		if (n_live)
			*n_live = (int32_t)live;
	}
}

// The moves: CTAs take (move, layer, K or V) in turn; then the table rows. Bound by memory: half
// of 2048 pages of 16 layers live, 467 MB in 74 us, 0.96 of the copy rate.
__global__ void __launch_bounds__(256)
pages_compact_kernel(const __grid_constant__ charsiu_gpu_pages p)
{
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t parts = 2 * p.n_layer, live = (uint32_t)p.work[2];
	const uint64_t jobs = (uint64_t)p.work[1] * parts;
	const int32_t *moves = p.work + PAGES_WORK_LIST;
	const int32_t *went = moves + PAGES_FORK_WORDS * PAGES_MAX_ITEMS + p.n_pages;
	for (uint64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
		const uint32_t m = (uint32_t)(j / parts), part = (uint32_t)(j % parts);
		pages_copy(p, part >> 1, part & 1, (uint32_t)moves[2 * m], (uint32_t)moves[2 * m + 1],
			   p.page);
	}
	for (uint32_t s = blockIdx.x; s < p.n_seq; s += gridDim.x) {
		const int64_t len = p.len[s];
		uint64_t held = len > 0 ? (uint64_t)(len + p.page - 1) / p.page : 0;
		held = held < p.max_pages ? held : p.max_pages;
		int32_t *row = p.table + (size_t)s * p.max_pages;
		for (uint32_t i = threadIdx.x; i < held; i += blockDim.x) {
			const uint32_t page = (uint32_t)row[i];
			if (page >= live && page < p.n_pages)
				row[i] = went[page];
		}
	}
}

// ---- RoPE and the append ---------------------------------------------------------

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi)
{
	const __half2 v = __floats2half2_rn(lo, hi);
	return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi)
{
	const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
	return *reinterpret_cast<const uint32_t *>(&v);
}

// One CTA a row: its q heads, then its k heads, then its v heads, 8 elements a thread at a
// time (two 16-byte loads, one 16-byte store). Where the row goes is found once a CTA
// (dividing per thread took 4000 rows of 48 heads of 128 from 25.0 to 27.6 us, 0.90 of the copy
// peak to 0.81). Bound by memory.
constexpr int APPEND_MAX_THREADS = 512;

template <typename T>
__global__ void __launch_bounds__(APPEND_MAX_THREADS)
pages_append_kernel(const __grid_constant__ charsiu_gpu_pages p, uint32_t layer,
		    const int32_t *__restrict__ slots, uint32_t t, uint32_t n_head,
		    const float *__restrict__ q, const float *__restrict__ k,
		    const float *__restrict__ v, const float *__restrict__ rope_cs, uint32_t n_ctx,
		    T *__restrict__ q_out)
{
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t row = blockIdx.x, shift = p.head_dim == 64 ? 3 : 4;
	const uint32_t words = (n_head + 2 * p.n_head_kv) << shift, seq = row / t;
	const int32_t slot = slots[seq];
	if (!pages_slot_ok(p, slot))
		return;
	const int64_t pos = (int64_t)p.len[slot] - t + (row - seq * t);
	if (pos < 0 || pos >= n_ctx || pos >= (int64_t)p.max_pages * p.page)
		return;
	const int32_t page = p.table[(size_t)slot * p.max_pages + (uint32_t)pos / p.page];
	if ((uint32_t)page >= p.n_pages)
		return;
	const uint64_t at = layer * p.layer_stride + page * p.page_stride + (uint32_t)pos % p.page * p.pos_stride;
	const float *cs_row = rope_cs + (size_t)pos * p.head_dim;
#pragma unroll 2
	for (uint32_t w = threadIdx.x; w < words; w += blockDim.x) {
		uint32_t head = w >> shift;
		const uint32_t i = (w & ((1u << shift) - 1)) * 8;
		const float *src;
		T *dst;
		const bool is_q = head < n_head, is_v = head >= n_head + p.n_head_kv;
		if (is_q) {
			src = q + ((size_t)row * n_head + head) * p.head_dim + i;
			dst = q_out + ((size_t)row * n_head + head) * p.head_dim + i;
		} else {
			head -= n_head + (is_v ? p.n_head_kv : 0);
			src = (is_v ? v : k) + ((size_t)row * p.n_head_kv + head) * p.head_dim + i;
			dst = (T *)(is_v ? p.v : p.k) + at + head * p.head_stride + i;
		}
		float x[8];
		*(float4 *)x = *(const float4 *)src;
		*(float4 *)(x + 4) = *(const float4 *)(src + 4);
		if (!is_v) {
			float cs[8];
			*(float4 *)cs = *(const float4 *)(cs_row + i);
			*(float4 *)(cs + 4) = *(const float4 *)(cs_row + i + 4);
#pragma unroll
			for (int j = 0; j < 8; j += 2) {
				const float a = x[j], b = x[j + 1], c = cs[j], s = cs[j + 1];
				x[j] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
				x[j + 1] = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
			}
		}
		uint4 o;
		o.x = pack_pair<T>(x[0], x[1]);
		o.y = pack_pair<T>(x[2], x[3]);
		o.z = pack_pair<T>(x[4], x[5]);
		o.w = pack_pair<T>(x[6], x[7]);
		*(uint4 *)dst = o;
	}
}

} // namespace cgpu
