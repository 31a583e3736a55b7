// SPDX-License-Identifier: GPL-2.0-or-later
// Attention of a batch over a paged cache, sequences of a group sharing their
// first pages (charsiu_gpu_attention_dev).
//
//   o = softmax(scale q K^T) V over the keys a query sees
//
// The keys of a query are cut into pieces: its group's shared pages (a prefix,
// the same for every query of the group, so read once for a tile of many
// queries), and the rest of its own sequence. Each piece is cut again where the
// batch is too small to fill the GPU. A piece gives, per query and head, its
// normalised output o_j = sum_t e^(x_t - m) v_t / l and the logarithm of its
// weight, m + log l, in one pass with a running maximum and sum; a last kernel
// joins the pieces: o = sum_j w_j o_j, w_j proportional to the weights.
//
// The weights e^(x - m) are rounded to the cache's type for their product with V, since
// the tensor cores take both operands in one type of 16 bits; l sums them unrounded. Each is off by
// at most half a step (2^-8 of it in bf16, 2^-11 in fp16), to either side, so a result with
// random V is off by about as much as by its own rounding: rms 1.5e-3 in bf16 over 16384 keys,
// 1.9e-4 in fp16 over 3000 (measured with fp32 results), where the 16-bit result's own is 1.7e-3
// and 2.1e-4. Weights in two parts would double the products with V, which with the
// exponentials are what the shared prefix is bound by.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "attn_cut.h"
#include "charsiu_gpu.h"
#include "pages.cuh"
#include "ptx.cuh"

namespace cgpu {

constexpr uint32_t ATTN_TILE_ROWS = 16;      // rows of a unit: the m of mma.m16n8k16
constexpr uint32_t ATTN_WARPS = 4;
constexpr uint32_t ATTN_GRAIN = 128;         // keys: pieces are cut to multiples of it
constexpr uint32_t ATTN_MAX_SPLITS = 32;     // pieces of a sequence's own keys; of a prefix twice as many
constexpr uint32_t ATTN_MAX_PIECES = 3 * ATTN_MAX_SPLITS;

struct AttnArgs {
	charsiu_gpu_pages p;
	const int32_t *slots, *group, *shared;
	const void *q;
	void *out;
	float *part_o;        // [row][pieces][hd], row = (sequence * n_tok + token) * n_head + head
	float *part_w;        // [row][pieces]: log2 of the piece's weight, -inf: nothing in it
	uint32_t layer, n_seq, n_tok, n_head, n_group, gqa;
	uint32_t pre_splits, own_splits;      // pieces of the prefix and of the rest
	uint32_t own_grain;                   // keys: the least a piece of the rest has
	uint32_t pre_units, own_tiles;        // units of the prefix at most; row tiles a sequence
	uint32_t rows_splits;                 // pieces of the prefix that the rows kernel makes
	uint32_t out_type;
	uint32_t behind;      // the rows kernel: behind the prefix's launch, no wait for it
	uint32_t early;       // and its CTAs that fit beside that launch's
	float scale;          // scale * log2(e)
	int *err;             // a wait that gave up says so here
};

// (Lengths, tables and queries are read past L1: the rows kernel may start without a wait
// of its own, see there.)

// the length of a slot; 0 for none
__device__ __forceinline__ int32_t attn_slot_len(const AttnArgs &a, int32_t slot)
{
	if (!pages_slot_ok(a.p, slot))
		return 0;
	const int64_t len = __ldcg(&a.p.len[slot]), most = (int64_t)a.p.max_pages * a.p.page;
	return (int32_t)(len < 0 ? 0 : len > most ? most : len);
}

// the length of sequence s of the batch; 0 for a padded one
__device__ __forceinline__ int32_t attn_len(const AttnArgs &a, uint32_t s)
{
	return attn_slot_len(a, __ldcg(&a.slots[s]));
}

// What the queries of a group share: sequences [s0, s1), their `keys` first keys
// (whole pages that every one of their queries sees), from slot `slot`'s table.
struct AttnGroup {
	uint32_t s0, s1;
	int32_t keys, slot;
};

// of the group with these bounds and told shared pages; by a whole warp
__device__ __forceinline__ AttnGroup attn_group(const AttnArgs &a, int32_t b0, int32_t b1, int32_t told)
{
	AttnGroup r;
	r.s0 = b0 < 0 ? 0 : b0 > (int32_t)a.n_seq ? a.n_seq : (uint32_t)b0;
	r.s1 = b1 < (int32_t)r.s0 ? r.s0 : b1 > (int32_t)a.n_seq ? a.n_seq : (uint32_t)b1;
	int32_t least = 0x7fffffff, mine = -1;
	uint32_t first = 0xffffffffu;
	for (uint32_t s = r.s0 + (threadIdx.x & 31); s < r.s1; s += 64) {
		// two at a time: their slots, then their lengths
		const int32_t sl[2] = {__ldcg(&a.slots[s]), s + 32 < r.s1 ? __ldcg(&a.slots[s + 32]) : -1};
		const int32_t len[2] = {attn_slot_len(a, sl[0]), attn_slot_len(a, sl[1])};
#pragma unroll
		for (int j = 0; j < 2; j++)
			if (len[j] > 0) {
				least = min(least, len[j] - (int32_t)a.n_tok + 1);
				if (s + 32 * j < first) {
					first = s + 32 * j;
					mine = sl[j];
				}
			}
	}
	least = __reduce_min_sync(0xffffffffu, least);
	const uint32_t lowest = __reduce_min_sync(0xffffffffu, first);
	const uint32_t who = __ballot_sync(0xffffffffu, first == lowest && mine >= 0);
	r.keys = 0;
	r.slot = -1;
	if (who && least > 0) {
		int32_t pages = min(told, (int32_t)a.p.max_pages);
		pages = min(pages, least / (int32_t)a.p.page);
		r.keys = pages > 0 ? pages * (int32_t)a.p.page : 0;
		r.slot = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
	}
	return r;
}

// the group of sequence s, or none (its keys 0); by a whole warp
__device__ __forceinline__ AttnGroup attn_group_of(const AttnArgs &a, uint32_t s)
{
	for (uint32_t g0 = 0; g0 < a.n_group; g0 += 32) {
		const uint32_t g = g0 + (threadIdx.x & 31);
		const bool real = g < a.n_group;
		const int32_t b0 = real ? __ldcg(&a.group[g]) : 0, b1 = real ? __ldcg(&a.group[g + 1]) : 0;
		const int32_t told = real ? __ldcg(&a.shared[g]) : 0;
		const uint32_t who = __ballot_sync(0xffffffffu, b0 <= (int32_t)s && (int32_t)s < b1);
		if (who) {
			const int src = __ffs(who) - 1;
			return attn_group(a, __shfl_sync(0xffffffffu, b0, src), __shfl_sync(0xffffffffu, b1, src),
					  __shfl_sync(0xffffffffu, told, src));
		}
	}
	AttnGroup r;
	r.s0 = r.s1 = s;
	r.keys = 0;
	r.slot = -1;
	return r;
}

// Unit u of all groups' row tiles (`rows` rows each): its group's bounds and told shared
// pages, and the tile in it; false past the last. By a whole warp.
struct AttnUnit {
	int32_t b0, b1, told;
	uint32_t tile;
};

__device__ __forceinline__ bool attn_find_unit(const AttnArgs &a, uint32_t u, uint32_t rows, AttnUnit *at)
{
	const uint32_t lane = threadIdx.x & 31;
	uint32_t before = 0;
	for (uint32_t g0 = 0; g0 < a.n_group; g0 += 32) {
		const bool real = g0 + lane < a.n_group;
		const int32_t b0 = real ? __ldcg(&a.group[g0 + lane]) : 0;
		const int32_t b1 = real ? __ldcg(&a.group[g0 + lane + 1]) : 0;
		const int32_t told = real ? __ldcg(&a.shared[g0 + lane]) : 0;
		const int32_t c0 = max(b0, 0), c1 = min(b1, (int32_t)a.n_seq);
		const uint32_t n = c1 > c0 ? ((uint32_t)(c1 - c0) * a.n_tok * a.gqa + rows - 1) / rows : 0;
		uint32_t inc = n;
		for (int o = 1; o < 32; o <<= 1) {
			const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
			if (lane >= (uint32_t)o)
				inc += y;
		}
		const uint32_t lo = before + inc - n;
		const uint32_t who = __ballot_sync(0xffffffffu, u >= lo && u < lo + n);
		if (who) {
			const int src = __ffs(who) - 1;
			at->tile = u - __shfl_sync(0xffffffffu, lo, src);
			at->b0 = __shfl_sync(0xffffffffu, b0, src);
			at->b1 = __shfl_sync(0xffffffffu, b1, src);
			at->told = __shfl_sync(0xffffffffu, told, src);
			return true;
		}
		before += __shfl_sync(0xffffffffu, inc, 31);
	}
	return false;
}

// ---- mma.sync pieces ---------------------------------------------------------------

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
					  uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
							 uint32_t b0, uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
		     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4],
						  uint32_t b0, uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
		     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
		     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
		     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v)
{
	return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v)
{
	return __bfloat162float(v);
}

// ---- rows of 16 ----------------------------------------------------------------------
//
// Items of work: 16 rows (queries of one KV head: sequence, token, head of the group)
// against one piece of keys, of a sequence's own or of a prefix. Bound by memory:
// a key's K and V serve few rows, so what counts is that enough of them are on
// their way at all times. Each of a persistent grid's CTAs takes items in turn; one
// warp runs ahead through its items (lengths, tables, then tensor copies of K and
// V page by page, and of the item's queries) into a ring of stages, so the latency
// of one item's start hides behind the work on the ones before. Four warps take a quarter of a
// stage's keys each (mma.m16n8k16, scores and outputs in registers,
// one pass with a running maximum and sum) and are joined through the item's last
// stage before it is given back. 64 sequences of up to 512 keys of their own, 8 KV heads of 128,
// on the 56 multiprocessors that a prefix leaves: 78 MB in 40 us, 35 GB/s a multiprocessor (an even
// share of the copy rate is 44). A CTA an item instead: 128 us for what takes 27 on all.
template <int HD>
struct AttnRing {
	static constexpr uint32_t KEYS = HD == 128 ? 64 : 128;      // a stage's; 32 KB of K and V
	static constexpr uint32_t WKEYS = KEYS / ATTN_WARPS;        // a warp's
	static constexpr uint32_t STAGES = 3;
	static constexpr uint32_t SLAB = KEYS * 128;                // 64 elements of each key
	static constexpr uint32_t HALF = KEYS * HD * 2;             // K, then V
	static constexpr uint32_t STAGE = 2 * HALF;
	static constexpr uint32_t Q_ROW = HD * 2 + 16;              // (16 bytes on: other banks)
	static constexpr uint32_t Q_AT = STAGES * STAGE, Q_STAGE = ATTN_TILE_ROWS * Q_ROW;
	static constexpr size_t SMEM = Q_AT + (size_t)STAGES * Q_STAGE;
};

// positions a tensor copy takes of one page
__host__ __device__ inline uint32_t attn_box(uint32_t page)
{
	return page < 64 ? page : 64;
}

struct AttnStage {
	uint32_t kind;        // 1: an item's first stage, 2: its last, 8: the end, 16: of a prefix
	uint32_t s0, n_rows, tile, kvh, slot_at;
	int32_t key0, k1;     // the stage's first key; the piece's end
	int32_t len;          // the sequence's length (a prefix is seen whole)
};

// a box of (64 elements, positions of a page) of one head of one page
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, int x, int y, int z, int w,
					    uint64_t *bar)
{
	asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
		     " [%0], [%1, {%2, %3, %4, %5}], [%6];"
		     :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
		     : "memory");
}

constexpr int ATTN_THREADS = (ATTN_WARPS + 1) * 32;

// How many CTAs of the rows kernel take items. Beside the prefix's launch the first a.early of
// them start with it, the others when its CTAs end: where the sequences' own keys are
// little work, the first take it all while the prefix is computed. The estimate is in
// microseconds: a stage of keys takes a CTA 0.8, an item 2 more, the prefix's steps of 64
// keys 0.9 each and 10 around them. Every CTA comes to the same answer. By a whole warp.
template <int HD>
__device__ __forceinline__ uint32_t attn_takers(const AttnArgs &a)
{
	const uint32_t lane = threadIdx.x & 31;
	if (!a.behind || a.early >= gridDim.x || a.n_seq > 128 || a.n_group > 32)
		return gridDim.x;
	const bool real = lane < a.n_group;
	const int32_t b0 = real ? __ldcg(&a.group[lane]) : 0, b1 = real ? __ldcg(&a.group[lane + 1]) : 0;
	const int32_t told = real ? __ldcg(&a.shared[lane]) : 0;
	int32_t slot[4], own[4];
#pragma unroll
	for (int j = 0; j < 4; j++)
		slot[j] = lane + 32 * j < a.n_seq ? __ldcg(&a.slots[lane + 32 * j]) : -1;
#pragma unroll
	for (int j = 0; j < 4; j++)
		own[j] = attn_slot_len(a, slot[j]);
	float keys = 0.0f, longest = 0.0f;
	for (uint32_t g = 0; g < a.n_group; g++) {
		const int32_t c0 = __shfl_sync(0xffffffffu, b0, g), c1 = __shfl_sync(0xffffffffu, b1, g);
		const int32_t pages = min(__shfl_sync(0xffffffffu, told, g), (int32_t)a.p.max_pages);
		const int32_t shared = max(pages, 0) * (int32_t)a.p.page;
		longest = fmaxf(longest, (float)shared);
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const int32_t s = (int32_t)lane + 32 * j;
			if (s >= c0 && s < c1)
				own[j] = max(own[j] - shared, 0);
		}
	}
#pragma unroll
	for (int j = 0; j < 4; j++)
		keys += (float)own[j];
	for (int o = 16; o; o >>= 1)
		keys += __shfl_xor_sync(0xffffffffu, keys, o);
	const float items = (float)a.own_tiles * a.p.n_head_kv;
	const float t_own = items * (0.8f * keys / AttnRing<HD>::KEYS + 2.0f * a.n_seq) / a.early;
	const float t_prefix = 10.0f + 0.9f * longest / 64.0f / (a.pre_splits / 2);
	return t_own <= 1.2f * t_prefix ? a.early : gridDim.x;
}

// codes of a wait that gave up, after the batched matvec's (5 to 13)
constexpr int ATTN_ERR_RING = 24, ATTN_ERR_ROWS = 25;

template <typename T, int HD>
__global__ void __launch_bounds__(ATTN_THREADS, 2)
attn_rows_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap,
		 const __grid_constant__ CUtensorMap vmap)
{
	using R = AttnRing<HD>;
	constexpr uint32_t NS = R::STAGES;
	constexpr int NT = HD / 8, KS = HD / 16;
	extern __shared__ __align__(1024) uint8_t rows_raw[];
	__shared__ __align__(8) uint64_t b_full[NS], b_free[NS];
	__shared__ __align__(8) uint64_t b_join;
	__shared__ AttnStage s_stage[NS];
	// (two items' maxima and sums: one warp may be at the next while another reads the last's)
	__shared__ float s_m[2][ATTN_WARPS][ATTN_TILE_ROWS], s_l[2][ATTN_WARPS][ATTN_TILE_ROWS];
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const uint32_t ring = smem_addr(rows_raw);
	uint8_t *ring_ptr = rows_raw;
	const uint32_t kvh_n = a.p.n_head_kv, tg = a.n_tok * a.gqa, pieces = a.pre_splits + a.own_splits;
	if (threadIdx.x == 0) {
		for (uint32_t i = 0; i < NS; i++) {
			mbar_init(&b_full[i], 1);
			mbar_init(&b_free[i], ATTN_WARPS);
		}
		mbar_init(&b_join, ATTN_WARPS);
		fence_mbar_init();
	}
	__syncthreads();
	// Behind the prefix's launch of the same call this one starts once all of that one's CTAs
	// are past their own wait, so what came before both is done; what it writes, that
	// one does not touch. It ends after that one, as the join counts on.
	if (!a.behind)
		pdl_wait();
	const uint32_t pre_items = a.pre_units * kvh_n * a.rows_splits;
	const uint32_t own_items = a.n_seq * a.own_tiles * kvh_n * a.own_splits, items = pre_items + own_items;

	if (warp == ATTN_WARPS) {
		// ---- the items, and their K, V and queries into the ring
		const uint32_t box = attn_box(a.p.page), row_bytes = HD * 2;
		uint32_t c = 0;
		bool ok = true;
		// `ids`: pages first_page, first_page + 1, ... of the sequence, one a lane
		constexpr uint32_t PAGES_HELD = 24;     // of 32 looked up: a stage starts in these, and has at most 8
		auto push = [&](AttnStage h, uint32_t ids, uint32_t first_page) {
			const uint32_t st = c % NS, base = ring + st * R::STAGE;
			if (c >= NS)
				ok = __all_sync(0xffffffffu,
						mbar_wait_bounded(&b_free[st], (c / NS - 1) & 1, WAIT_LIMIT_NS));
			if (!ok)
				return;
			const uint32_t keys = min((uint32_t)(h.k1 - h.key0), R::KEYS), boxes = (keys + box - 1) / box;
			const uint32_t q_rows = h.kind & 1 ? min(h.n_rows - h.tile * ATTN_TILE_ROWS, ATTN_TILE_ROWS) : 0;
			// this lane's box: which positions, which 64 elements; K and V alike
			const uint32_t mine = lane % (R::KEYS / 16), slab = lane / (R::KEYS / 16);
			const uint32_t pos = (uint32_t)h.key0 + mine * box;
			// (no page: zeros)
			const int page = (int)min(__shfl_sync(0xffffffffu, ids, pos / a.p.page - first_page), a.p.n_pages);
			if (lane == 0) {
				s_stage[st] = h;
				mbar_arrive_expect_tx(&b_full[st], 2 * boxes * box * row_bytes + q_rows * row_bytes);
			}
			__syncwarp();
			if (mine < boxes && slab < HD / 64) {
				const uint32_t dst = base + slab * R::SLAB + mine * box * 128;
				tma_load_4d(dst, &kmap, (int)(slab * 64), (int)(pos % a.p.page), (int)h.kvh, page,
					    &b_full[st]);
				tma_load_4d(dst + R::HALF, &vmap, (int)(slab * 64), (int)(pos % a.p.page), (int)h.kvh,
					    page, &b_full[st]);
			}
			if (lane < q_rows) {
				const uint32_t r = h.tile * ATTN_TILE_ROWS + lane, s = h.s0 + r / tg, x = r % tg;
				const T *src = (const T *)a.q + ((size_t)(s * a.n_tok + x / a.gqa) * a.n_head +
								 h.kvh * a.gqa + x % a.gqa) * HD;
				bulk_g2s(ring_ptr + R::Q_AT + st * R::Q_STAGE + lane * R::Q_ROW, src, row_bytes,
					 &b_full[st]);
			}
			__syncwarp();
			c++;
		};
		const uint32_t ctas = attn_takers<HD>(a);
		// a lane an item, 32 items' lengths and groups on their way at a time
		for (uint64_t at = blockIdx.x < ctas ? blockIdx.x : items; at < items && ok; at += 32ull * ctas) {
			const uint64_t it = at + (uint64_t)lane * ctas;
			const bool own = it >= pre_items && it < items;
			const uint32_t splits = own ? a.own_splits : max(a.rows_splits, 1u);
			uint32_t b = own ? (uint32_t)(it - pre_items) : (uint32_t)min(it, (uint64_t)items);
			const uint32_t per = kvh_n * splits * (own ? a.own_tiles : 1);
			AttnStage h = {};
			h.s0 = b / per;                         // (of a prefix: the unit)
			b -= h.s0 * per;
			h.tile = b / (kvh_n * splits);
			b -= h.tile * kvh_n * splits;
			uint32_t piece = b / kvh_n;
			h.kvh = b - piece * kvh_n;
			h.n_rows = tg;
			int32_t slot = own ? __ldcg(&a.slots[h.s0]) : -1, shared = 0;
			// the groups of own items: each looked up once for all lanes in it
			for (uint32_t left = a.n_group ? __ballot_sync(0xffffffffu, own) : 0; left;) {
				const uint32_t s = __shfl_sync(0xffffffffu, h.s0, __ffs(left) - 1);
				const AttnGroup gr = attn_group_of(a, s);
				const bool in = own && (h.s0 == s || (h.s0 >= gr.s0 && h.s0 < gr.s1));
				shared = in ? gr.keys : shared;
				left &= ~__ballot_sync(0xffffffffu, in);
			}
			h.len = attn_slot_len(a, slot);
			int32_t k0 = h.len ? shared : 0;
			uint32_t kind = own ? (!piece && !k0 ? 32u : 0u) : 16u;  // 32: no prefix, its first piece says so
			// (no keys behind the tile's last query's position: 4 prompts of 1000 tokens, 32 heads of
			// 128, pages of 16, 393 us, with all the sequence's keys for every tile 658)
			const uint32_t last = (min((h.tile + 1) * ATTN_TILE_ROWS, tg) - 1) / a.gqa;
			h.k1 = max(h.len - (int32_t)a.n_tok + (int32_t)last + 1, 0);
			h.slot_at = (own ? a.pre_splits : 0) + piece;
			if (own)
				attn_piece(k0, h.k1, piece, a.own_splits, a.own_grain);
			const uint32_t rows = min(tg - h.tile * ATTN_TILE_ROWS, ATTN_TILE_ROWS);
			if (own && (k0 >= h.k1 || (kind & 32)))
				// no keys, or no prefix: the weights say so
				for (uint32_t i = 0; i < rows; i++) {
					const uint32_t x = h.tile * ATTN_TILE_ROWS + i;
					float *w = a.part_w + ((size_t)(h.s0 * a.n_tok + x / a.gqa) * a.n_head +
							       h.kvh * a.gqa + x % a.gqa) * pieces;
					if (k0 >= h.k1)
						w[h.slot_at] = -INFINITY;
					for (uint32_t j = 0; (kind & 32) && j < a.pre_splits; j++)
						w[j] = -INFINITY;
				}
			uint32_t left = __ballot_sync(0xffffffffu, it < items && (!own || k0 < h.k1));
			for (; left && ok; left &= left - 1) {
				const int j = __ffs(left) - 1;
				AttnStage g;
				g.s0 = __shfl_sync(0xffffffffu, h.s0, j);
				g.tile = __shfl_sync(0xffffffffu, h.tile, j);
				g.kvh = __shfl_sync(0xffffffffu, h.kvh, j);
				g.n_rows = tg;
				g.slot_at = __shfl_sync(0xffffffffu, h.slot_at, j);
				g.k1 = __shfl_sync(0xffffffffu, h.k1, j);
				g.len = __shfl_sync(0xffffffffu, h.len, j);
				const uint32_t what = __shfl_sync(0xffffffffu, kind, j);
				int32_t from = __shfl_sync(0xffffffffu, k0, j), of = __shfl_sync(0xffffffffu, slot, j);
				if (what & 16) {
					// a prefix's unit
					AttnUnit at;
					if (!attn_find_unit(a, g.s0, ATTN_TILE_ROWS, &at))
						continue;
					const AttnGroup gr = attn_group(a, at.b0, at.b1, at.told);
					if (!gr.keys)
						continue;
					g.tile = at.tile;
					g.s0 = gr.s0;
					g.n_rows = (gr.s1 - gr.s0) * tg;
					g.len = 0x7fffffff;
					of = gr.slot;
					from = 0;
					g.k1 = gr.keys;
					attn_piece(from, g.k1, g.slot_at, a.rows_splits, ATTN_GRAIN);
					const uint32_t r = g.tile * ATTN_TILE_ROWS + lane, s = g.s0 + r / tg, x = r % tg;
					if (from >= g.k1 && lane < ATTN_TILE_ROWS && r < g.n_rows && attn_len(a, s))
						a.part_w[((size_t)(s * a.n_tok + x / a.gqa) * a.n_head + g.kvh * a.gqa +
							  x % a.gqa) * pieces + g.slot_at] = -INFINITY;
				}
				const int32_t *row = a.p.table + (size_t)of * a.p.max_pages;
				uint32_t ids = 0, more = 0, at_page = 0;
				const uint32_t pages = g.k1 > from ? (uint32_t)(g.k1 - 1) / a.p.page + 1 : 0;
				auto pages_from = [&](uint32_t p) {
					return p + lane < pages ? (uint32_t)__ldcg(&row[p + lane]) : 0u;
				};
				if (from < g.k1) {
					at_page = (uint32_t)from / a.p.page;
					ids = pages_from(at_page);
					more = pages_from(at_page + PAGES_HELD);
				}
				for (int32_t key0 = from; key0 < g.k1 && ok; key0 += (int32_t)R::KEYS) {
					g.kind = (what & 16) | (key0 == from ? 1u : 0u) |
						 (key0 + (int32_t)R::KEYS >= g.k1 ? 2u : 0u);
					g.key0 = key0;
					// (a stage's pages lie within 32 from at_page on)
					while ((uint32_t)key0 / a.p.page >= at_page + PAGES_HELD) {
						at_page += PAGES_HELD;
						ids = more;
						more = pages_from(at_page + PAGES_HELD);
					}
					push(g, ids, at_page);
				}
			}
		}
		// the end; then every copy issued lands before the CTA leaves
		AttnStage end = {};
		end.kind = 8;
		if (ok)
			push(end, 0, 0);
		if (!ok && lane == 0)
			*(volatile int *)a.err = ATTN_ERR_RING;
		for (uint32_t i = c > NS ? c - NS : 0; i < c; i++)
			if (!mbar_wait_bounded(&b_full[i % NS], (i / NS) & 1, WAIT_LIMIT_NS) && lane == 0)
				*(volatile int *)a.err = ATTN_ERR_RING;
	} else {
		// ---- rows
		const uint32_t q4 = lane & 3;
		uint32_t qa[KS][4];
		float o[NT][4], m[2], l[2];
		int32_t limit[2], least = 0;
		uint32_t joins = 0;
		bool ended = false;
		auto together = [&]() {                 // the four warps, as a barrier that can give up
			__syncwarp();
			if (lane == 0)
				mbar_arrive(&b_join);
			return (bool)__all_sync(0xffffffffu, mbar_wait_bounded(&b_join, joins++ & 1, WAIT_LIMIT_NS));
		};
		for (uint32_t c = 0;; c++) {
			const uint32_t st = c % NS;
			if (!__all_sync(0xffffffffu, mbar_wait_bounded(&b_full[st], (c / NS) & 1, WAIT_LIMIT_NS)))
				break;
			const AttnStage h = s_stage[st];
			if (h.kind & 8) {
				ended = true;
				break;
			}
			if (h.kind & 1) {
				m[0] = m[1] = -INFINITY;
				l[0] = l[1] = 0.0f;
#pragma unroll
				for (int n = 0; n < NT; n++)
					o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
				// this thread's rows of the accumulators: lane / 4 and 8 more
#pragma unroll
				for (int e = 0; e < 2; e++) {
					const uint32_t r = h.tile * ATTN_TILE_ROWS + lane / 4 + 8 * e;
					// (a prefix is seen whole)
					limit[e] = r < h.n_rows && !(h.kind & 16)
							   ? h.len - (int32_t)a.n_tok + (int32_t)(r / a.gqa) + 1
							   : h.k1;
				}
				least = min(min(__reduce_min_sync(0xffffffffu, limit[0]),
						__reduce_min_sync(0xffffffffu, limit[1])), h.k1);
				const uint32_t rows = min(h.n_rows - h.tile * ATTN_TILE_ROWS, ATTN_TILE_ROWS);
				const uint8_t *qs = ring_ptr + R::Q_AT + st * R::Q_STAGE;
#pragma unroll
				for (int ks = 0; ks < KS; ks++)
#pragma unroll
					for (int j = 0; j < 4; j++) {
						const uint32_t r = lane / 4 + 8 * (j & 1);
						qa[ks][j] = r < rows ? *(const uint32_t *)(qs + r * R::Q_ROW + ks * 32 +
											   (j >> 1) * 16 + q4 * 4)
								     : 0u;
					}
			}
			const uint32_t ks_ = ring + st * R::STAGE, vs = ks_ + R::HALF, w0 = warp * R::WKEYS;
			const int32_t key0 = h.key0 + (int32_t)w0;
			if (key0 < h.k1) {
				constexpr int NK = R::WKEYS / 8;
				float s[NK][4];
#pragma unroll
				for (int j = 0; j < NK; j++) {
					s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
					float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // (two chains of MMAs, not one)
					const uint32_t key = w0 + j * 8 + (lane & 7);
#pragma unroll
					for (int k2 = 0; k2 < KS / 2; k2++) {
						const uint32_t w = k2 * 4 + lane / 8;
						uint32_t kb[4];
						ldmatrix_x4(kb, ks_ + (w / 8) * R::SLAB + key * 128 + (((w % 8) ^ (key & 7)) << 4));
						mma_16816<T>(s[j], qa[2 * k2], kb[0], kb[1]);
						mma_16816<T>(odd, qa[2 * k2 + 1], kb[2], kb[3]);
					}
#pragma unroll
					for (int e = 0; e < 4; e++)
						s[j][e] += odd[e];
				}
				const bool ragged = key0 + (int32_t)R::WKEYS > least;
				float mx[2] = {m[0], m[1]};
#pragma unroll
				for (int j = 0; j < NK; j++)
#pragma unroll
					for (int e = 0; e < 4; e++) {
						s[j][e] *= a.scale;
						if (ragged && key0 + j * 8 + (int32_t)q4 * 2 + (e & 1) >= min(limit[e >> 1], h.k1))
							s[j][e] = -INFINITY;
						mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
					}
#pragma unroll
				for (int e = 0; e < 2; e++) {
					mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
					mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
				}
				if (__any_sync(0xffffffffu, mx[0] != m[0] || mx[1] != m[1])) {
#pragma unroll
					for (int e = 0; e < 2; e++) {
						const float keep = mx[e] == m[e] ? 1.0f : exp2_approx(m[e] - mx[e]);
						m[e] = mx[e];
						l[e] *= keep;
#pragma unroll
						for (int n = 0; n < NT; n++) {
							o[n][2 * e] *= keep;
							o[n][2 * e + 1] *= keep;
						}
					}
				}
#pragma unroll
				for (int e = 0; e < 2; e++) {
					const float base = m[e] == -INFINITY ? 0.0f : m[e];
#pragma unroll
					for (int j = 0; j < NK; j++) {
						s[j][2 * e] = exp2_approx(s[j][2 * e] - base);
						s[j][2 * e + 1] = exp2_approx(s[j][2 * e + 1] - base);
						l[e] += s[j][2 * e] + s[j][2 * e + 1];
					}
				}
				// A weight of 0 must take nothing from its key, and 0 * inf is NaN. Keys
				// behind the piece's end are cleared; where some row does not see some
				// key that others do, V is searched for inf and NaN, and such a tile
				// goes key by key.
				bool plain = true;
				if (ragged && key0 + (int32_t)R::WKEYS > h.k1) {
					const uint32_t end = (uint32_t)(h.k1 - key0);
					for (uint32_t x = lane; x < (R::WKEYS - end) * (HD / 8); x += 32) {
						const uint32_t key = w0 + end + x / (HD / 8), w = x % (HD / 8);
						asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};"
							     :: "r"(vs + (w / 8) * R::SLAB + key * 128 + (w % 8) * 16), "r"(0)
							     : "memory");
					}
					fence_proxy_async_smem();
					__syncwarp();
				}
				if (ragged && least < h.k1) {
					bool bad = false;
					for (uint32_t x = lane; x < R::WKEYS * (HD / 2); x += 32) {
						const uint32_t key = w0 + x / (HD / 2), w = x % (HD / 2);
						uint32_t two;
						asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two)
							     : "r"(vs + (w / 32) * R::SLAB + key * 128 + (w % 32) * 4) : "memory");
						const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
						bad |= (two & e) == e || ((two >> 16) & e) == e;
					}
					plain = !__any_sync(0xffffffffu, bad);
				}
				if (plain) {
#pragma unroll
					for (int k16 = 0; k16 < NK / 2; k16++) {
						const uint32_t pa[4] = {pack_pair<T>(s[2 * k16][0], s[2 * k16][1]),
									pack_pair<T>(s[2 * k16][2], s[2 * k16][3]),
									pack_pair<T>(s[2 * k16 + 1][0], s[2 * k16 + 1][1]),
									pack_pair<T>(s[2 * k16 + 1][2], s[2 * k16 + 1][3])};
						const uint32_t key = w0 + k16 * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
						for (int n2 = 0; n2 < NT / 2; n2++) {
							const uint32_t w = n2 * 2 + (lane >> 4);
							uint32_t vb[4];
							ldmatrix_x4_trans(vb, vs + (w / 8) * R::SLAB + key * 128 +
									  (((w % 8) ^ (key & 7)) << 4));
							mma_16816<T>(o[2 * n2], pa, vb[0], vb[1]);
							mma_16816<T>(o[2 * n2 + 1], pa, vb[2], vb[3]);
						}
					}
				} else {
#pragma unroll 1
					for (int key = 0; key < (int)R::WKEYS; key++) {
						float w[2];
#pragma unroll
						for (int e = 0; e < 2; e++) {
							float x = 0.0f;
#pragma unroll
							for (int j = 0; j < NK; j++)
								if (key / 8 == j)
									x = key & 1 ? s[j][2 * e + 1] : s[j][2 * e];
							w[e] = to_float<T>(T(__shfl_sync(0xffffffffu, x, (lane & ~3u) + (key % 8) / 2)));
						}
						const uint32_t kk = w0 + key;
#pragma unroll
						for (int n = 0; n < NT; n++) {
							uint32_t two;
							asm volatile("ld.shared.u32 %0, [%1];"
								     : "=r"(two)
								     : "r"(vs + (n / 8) * R::SLAB + kk * 128 +
									   (((n % 8) ^ (kk & 7)) << 4) + q4 * 4)
								     : "memory");
							T v[2];
							*(uint32_t *)v = two;
#pragma unroll
							for (int e = 0; e < 4; e++)
								if (key0 + key < min(limit[e >> 1], h.k1))
									o[n][e] = __fmaf_rn(w[e >> 1], to_float<T>(v[e & 1]), o[n][e]);
						}
					}
				}
			}
			if (h.kind & 2) {
				// the warps joined: maxima and sums, then the outputs through this stage
				const uint32_t row0 = h.tile * ATTN_TILE_ROWS, turn = joins / 2 & 1;
				const uint32_t rows = min(h.n_rows - row0, ATTN_TILE_ROWS);
#pragma unroll
				for (int e = 0; e < 2; e++) {
					l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
					l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
					if (q4 == 0) {
						s_m[turn][warp][lane / 4 + 8 * e] = m[e];
						s_l[turn][warp][lane / 4 + 8 * e] = l[e];
					}
				}
				if (!together())                           // all have read the stage
					break;
				float *os = reinterpret_cast<float *>(ring_ptr + st * R::STAGE);     // [warps][16][HD]
#pragma unroll
				for (int e = 0; e < 2; e++)
					if (lane / 4 + 8 * e < rows)
#pragma unroll
						for (int n = 0; n < NT; n++)
							*(float2 *)(os + (warp * ATTN_TILE_ROWS + lane / 4 + 8 * e) * HD +
								    ((n * 8) ^ ((lane / 4 & 3) * 8)) + q4 * 2) =
								make_float2(o[n][2 * e], o[n][2 * e + 1]);
				if (!together())
					break;
				for (uint32_t x = threadIdx.x; x < rows * (HD / 4); x += ATTN_WARPS * 32) {
					const uint32_t r = x / (HD / 4), i = x % (HD / 4) * 4, rr = row0 + r;
					const uint32_t ss = h.kind & 16 ? rr / tg : 0, in = rr - ss * tg, tok = in / a.gqa;
					if ((h.kind & 16) && !attn_len(a, h.s0 + ss))
						continue;              // (its own pieces say that it sees nothing)
					float top = -INFINITY, sum = 0.0f, f[ATTN_WARPS];
#pragma unroll
					for (int w = 0; w < (int)ATTN_WARPS; w++)
						top = fmaxf(top, s_m[turn][w][r]);
					const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
					for (int w = 0; w < (int)ATTN_WARPS; w++) {
						f[w] = exp2_approx(s_m[turn][w][r] - base);
						sum += f[w] * s_l[turn][w][r];
					}
					const size_t at = ((size_t)((h.s0 + ss) * a.n_tok + tok) * a.n_head + h.kvh * a.gqa +
							   in - tok * a.gqa) * pieces;
					const float inv = sum != 0.0f ? __fdiv_rn(1.0f, sum) : 0.0f;
					if (i == 0)
						a.part_w[at + h.slot_at] = sum != 0.0f ? base + log2f(sum) : -INFINITY;
					float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
					for (int w = 0; w < (int)ATTN_WARPS; w++) {
						const float4 p = *(const float4 *)(os + (w * ATTN_TILE_ROWS + r) * HD +
										   (i ^ ((r & 3) * 8)));
						v[0] += f[w] * p.x;
						v[1] += f[w] * p.y;
						v[2] += f[w] * p.z;
						v[3] += f[w] * p.w;
					}
					*(float4 *)(a.part_o + (at + h.slot_at) * HD + i) =
						make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
				}
				fence_proxy_async_smem();
			}
			__syncwarp();
			if (lane == 0)
				mbar_arrive(&b_free[st]);
		}
		if (!ended && lane == 0)
			*(volatile int *)a.err = ATTN_ERR_ROWS;
	}
	// (Only now: the join's CTAs, waiting beside this kernel from its start, took 32 sequences on 16384
	// shared keys of hd 128 from 41 to 53 us.)
	pdl_launch_dependents();
	if (a.behind)
		pdl_wait();
}

// The pieces of each row joined: one warp a row (sequence, token, head). Bound by latency, its
// weights and then its outputs, four at a time: 2048 rows of up to 31 pieces 5 us (8 of them cold),
// 12.8 MB.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_join_kernel(const __grid_constant__ AttnArgs a)
{
	pdl_wait();
	const uint32_t lane = threadIdx.x & 31;
	const size_t row = (size_t)blockIdx.x * 8 + threadIdx.x / 32;
	if (row >= (size_t)a.n_seq * a.n_tok * a.n_head)
		return;
	constexpr int EACH = HD / 32;
	const uint32_t pieces = a.pre_splits + a.own_splits;
	float v[EACH];
#pragma unroll
	for (int e = 0; e < EACH; e++)
		v[e] = 0.0f;
	// lane j has the weights of pieces j, j + 32, ...
	constexpr int WORDS = ATTN_MAX_PIECES / 32;
	const float *w = a.part_w + row * pieces;
	float mine[WORDS], top = -INFINITY;
	bool any = false;                               // (a NaN is no maximum, but it is a weight)
#pragma unroll
	for (int j = 0; j < WORDS; j++) {
		mine[j] = lane + 32 * j < pieces ? w[lane + 32 * j] : -INFINITY;
		top = fmaxf(top, mine[j]);
		any |= mine[j] != -INFINITY;
	}
	for (int o = 16; o; o >>= 1)
		top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
	top = top == -INFINITY ? 0.0f : top;
	if (__any_sync(0xffffffffu, any)) {
		float sum = 0.0f;
#pragma unroll
		for (int j = 0; j < WORDS; j++) {
			const bool has = mine[j] != -INFINITY;
			mine[j] = exp2_approx(mine[j] - top);
			sum += mine[j];
			for (uint32_t left = __ballot_sync(0xffffffffu, has); left;) {
				float f[4], p[4][EACH];          // four pieces' outputs on their way at a time
#pragma unroll
				for (int k = 0; k < 4; k++, left &= left - 1) {
					const int src = left ? __ffs(left) - 1 : 0;
					f[k] = __shfl_sync(0xffffffffu, mine[j], src);
					const float *o = a.part_o + (row * pieces + 32 * j + src) * HD + lane * EACH;
#pragma unroll
					for (int e = 0; e < EACH; e++)
						p[k][e] = left ? o[e] : 0.0f;
					f[k] = left ? f[k] : 0.0f;
				}
#pragma unroll
				for (int k = 0; k < 4; k++)
#pragma unroll
					for (int e = 0; e < EACH; e++)
						v[e] += f[k] * p[k][e];
			}
		}
		for (int o = 16; o; o >>= 1)
			sum += __shfl_xor_sync(0xffffffffu, sum, o);
		const float inv = __fdiv_rn(1.0f, sum);
#pragma unroll
		for (int e = 0; e < EACH; e++)
			v[e] *= inv;
	}
#pragma unroll
	for (int e = 0; e < EACH; e += 2) {
		const size_t at = row * HD + lane * EACH + e;
		if (a.out_type == 0)
			*(float2 *)((float *)a.out + at) = make_float2(v[e], v[e + 1]);
		else
			*(uint32_t *)((T *)a.out + at) = pack_pair<T>(v[e], v[e + 1]);
	}
}

} // namespace cgpu
