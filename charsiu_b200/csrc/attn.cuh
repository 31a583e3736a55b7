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
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "charsiu_gpu.h"
#include "pages.cuh"
#include "ptx.cuh"

namespace cgpu {

constexpr uint32_t ATTN_TILE_ROWS = 16;      // rows of a unit: the m of mma.m16n8k16
constexpr uint32_t ATTN_WARPS = 4;
constexpr uint32_t ATTN_KEYS = 32;           // keys a warp takes at a time
constexpr uint32_t ATTN_GRAIN = ATTN_WARPS * ATTN_KEYS;

struct AttnArgs {
	charsiu_gpu_pages p;
	const int32_t *slots, *group, *shared;
	const void *q;
	void *out;
	float *part_o;        // [row][pieces][hd], row = (sequence * n_tok + token) * n_head + head
	float *part_w;        // [row][pieces]: log2 of the piece's weight, -inf: nothing in it
	uint32_t layer, n_seq, n_tok, n_head, n_group, gqa;
	uint32_t pre_splits, own_splits;      // pieces of the prefix and of the rest
	uint32_t pre_units, own_tiles;        // units of the prefix at most; row tiles a sequence
	uint32_t out_type;
	uint32_t beside;      // the prefix is another launch's, before this one: no wait for it
	float scale;          // scale * log2(e)
	int *err;             // a wait that gave up says so here
};

// (Lengths, tables and queries are read past L1: the rows kernel may start without
// a wait of its own, see there.)

// the length of sequence s of the batch; 0 for a padded one
__device__ __forceinline__ int32_t attn_len(const AttnArgs &a, uint32_t s)
{
	const int32_t slot = __ldcg(&a.slots[s]);
	if (!pages_slot_ok(a.p, slot))
		return 0;
	const int64_t len = __ldcg(&a.p.len[slot]), most = (int64_t)a.p.max_pages * a.p.page;
	return (int32_t)(len < 0 ? 0 : len > most ? most : len);
}

// What the queries of a group share: sequences [s0, s1), their `keys` first keys
// (whole pages that every one of their queries sees), from slot `slot`'s table.
struct AttnGroup {
	uint32_t s0, s1;
	int32_t keys, slot;
};

// by a whole warp
__device__ __forceinline__ AttnGroup attn_group(const AttnArgs &a, uint32_t g)
{
	AttnGroup r;
	const int32_t b0 = __ldcg(&a.group[g]), b1 = __ldcg(&a.group[g + 1]);
	r.s0 = b0 < 0 ? 0 : b0 > (int32_t)a.n_seq ? a.n_seq : (uint32_t)b0;
	r.s1 = b1 < (int32_t)r.s0 ? r.s0 : b1 > (int32_t)a.n_seq ? a.n_seq : (uint32_t)b1;
	int32_t least = 0x7fffffff;
	uint32_t first = 0xffffffffu;
	for (uint32_t s = r.s0 + (threadIdx.x & 31); s < r.s1; s += 32) {
		const int32_t len = attn_len(a, s);
		if (len > 0) {
			least = min(least, len - (int32_t)a.n_tok + 1);
			first = min(first, s);
		}
	}
	least = __reduce_min_sync(0xffffffffu, least);
	first = __reduce_min_sync(0xffffffffu, first);
	r.keys = 0;
	r.slot = -1;
	if (first != 0xffffffffu && least > 0) {
		int32_t pages = __ldcg(&a.shared[g]);
		pages = min(pages, (int32_t)a.p.max_pages);
		pages = min(pages, least / (int32_t)a.p.page);
		r.keys = pages > 0 ? pages * (int32_t)a.p.page : 0;
		r.slot = __ldcg(&a.slots[first]);
	}
	return r;
}

// the group of sequence s, or none (its keys 0); by a whole warp
__device__ __forceinline__ AttnGroup attn_group_of(const AttnArgs &a, uint32_t s)
{
	for (uint32_t g0 = 0; g0 < a.n_group; g0 += 32) {
		const uint32_t g = g0 + (threadIdx.x & 31);
		const bool in = g < a.n_group && __ldcg(&a.group[g]) <= (int32_t)s &&
				(int32_t)s < __ldcg(&a.group[g + 1]);
		const uint32_t who = __ballot_sync(0xffffffffu, in);
		if (who)
			return attn_group(a, g0 + __ffs(who) - 1);
	}
	AttnGroup r;
	r.s0 = r.s1 = s;
	r.keys = 0;
	r.slot = -1;
	return r;
}

// Unit u of all groups' row tiles (`rows` rows each): its group and the tile in
// it; false past the last. By a whole warp.
__device__ __forceinline__ bool attn_find_unit(const AttnArgs &a, uint32_t u, uint32_t rows,
					       uint32_t *g, uint32_t *tile)
{
	const uint32_t lane = threadIdx.x & 31;
	uint32_t before = 0;
	for (uint32_t g0 = 0; g0 < a.n_group; g0 += 32) {
		uint32_t n = 0;
		if (g0 + lane < a.n_group) {
			const int32_t b0 = max(__ldcg(&a.group[g0 + lane]), 0);
			const int32_t b1 = min(__ldcg(&a.group[g0 + lane + 1]), (int32_t)a.n_seq);
			if (b1 > b0)
				n = ((uint32_t)(b1 - b0) * a.n_tok * a.gqa + rows - 1) / rows;
		}
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
			*g = g0 + src;
			*tile = u - __shfl_sync(0xffffffffu, lo, src);
			return true;
		}
		before += __shfl_sync(0xffffffffu, inc, 31);
	}
	return false;
}

// Piece `i` of `n` of the keys [k0, k1): whole grains
__device__ __forceinline__ void attn_piece(int32_t &k0, int32_t &k1, uint32_t i, uint32_t n,
					   uint32_t grain)
{
	const int32_t keys = k1 - k0;
	const int32_t grains = (keys + (int32_t)grain - 1) / (int32_t)grain;
	const int32_t each = (grains + (int32_t)n - 1) / (int32_t)n * (int32_t)grain;
	const int64_t b = (int64_t)k0 + (int64_t)i * each, e = b + each;
	const int32_t last = k1;
	k0 = (int32_t)(b < last ? b : last);
	k1 = (int32_t)(e < last ? e : last);
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

// 16 bytes global -> shared, or zeros (nothing is read then)
__device__ __forceinline__ void cp_async16_or_zero(uint32_t smem, const void *gmem, bool ok)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
		     :: "r"(smem), "l"(gmem), "r"(ok ? 16 : 0) : "memory");
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

template <int HD>
constexpr size_t attn_rows_smem()
{
	return (size_t)ATTN_WARPS * 2 * 2 * ATTN_KEYS * HD * 2;      // warps, stages, K and V
}

// 16 rows (queries of one KV head: sequence, token, head of the group) against one
// piece of keys. Four warps, each with 32-key tiles of its own (every fourth) that
// it copies to shared memory two deep; scores, weights and outputs stay in
// registers; the warps' results are joined at the end. Shared rows are swizzled
// by 16-byte words (word ^ (key & 7)), so ldmatrix meets no bank conflict.
template <typename T, int HD>
__global__ void __launch_bounds__(ATTN_WARPS * 32)
attn_rows_kernel(const __grid_constant__ AttnArgs a)
{
	extern __shared__ __align__(128) uint8_t asm_[];
	__shared__ float s_m[ATTN_WARPS][ATTN_TILE_ROWS], s_l[ATTN_WARPS][ATTN_TILE_ROWS];
	constexpr int KW = HD / 8;                       // 16-byte words a key
	constexpr int NT = HD / 8, KS = HD / 16;
	const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const uint32_t kvh_n = a.p.n_head_kv, tg = a.n_tok * a.gqa;
	// Beside the prefix's launch this one starts once all of that one's CTAs are past
	// their own wait, so what came before both is done; what it writes, that one
	// does not touch. It ends after that one, as the join counts on.
	struct EndAfter {
		bool late;
		__device__ ~EndAfter()
		{
			if (late)
				pdl_wait();
		}
	} end_after{a.beside != 0};
	if (!a.beside)
		pdl_wait();
	pdl_launch_dependents();

	// which rows, which keys
	uint32_t b = blockIdx.x, s0, s1, tile, piece, kvh, slot_at;
	int32_t k0, k1, slot;
	const uint32_t pre_blocks = a.pre_units * kvh_n * a.pre_splits;
	if (b < pre_blocks) {
		const uint32_t u = b / (kvh_n * a.pre_splits);
		b -= u * kvh_n * a.pre_splits;
		piece = b / kvh_n;
		kvh = b - piece * kvh_n;
		uint32_t g;
		if (!attn_find_unit(a, u, ATTN_TILE_ROWS, &g, &tile))
			return;
		const AttnGroup gr = attn_group(a, g);
		if (!gr.keys)
			return;
		s0 = gr.s0;
		s1 = gr.s1;
		slot = gr.slot;
		k0 = 0;
		k1 = gr.keys;
		attn_piece(k0, k1, piece, a.pre_splits, ATTN_GRAIN);
		slot_at = piece;
	} else {
		b -= pre_blocks;
		const uint32_t per = a.own_tiles * kvh_n * a.own_splits;
		s0 = b / per;
		b -= s0 * per;
		tile = b / (kvh_n * a.own_splits);
		b -= tile * kvh_n * a.own_splits;
		piece = b / kvh_n;
		kvh = b - piece * kvh_n;
		s1 = s0 + 1;
		k1 = attn_len(a, s0);
		if (k1 == 0)
			return;
		slot = __ldcg(&a.slots[s0]);
		k0 = attn_group_of(a, s0).keys;
		attn_piece(k0, k1, piece, a.own_splits, ATTN_GRAIN);
		slot_at = a.pre_splits + piece;
	}
	const uint32_t n_rows = (s1 - s0) * tg, pieces = a.pre_splits + a.own_splits;

	// this thread's two rows of the accumulators: lane / 4 and 8 more
	int32_t limit[2];
	const T *qp[2];
	const uint32_t c = lane & 3;
#pragma unroll
	for (int h = 0; h < 2; h++) {
		const uint32_t r = tile * ATTN_TILE_ROWS + lane / 4 + 8 * h;
		limit[h] = k1;
		qp[h] = nullptr;
		if (r < n_rows) {
			const uint32_t s = s0 + r / tg, t = r % tg / a.gqa;
			const int32_t len = attn_len(a, s);
			if (len > 0)
				limit[h] = len - (int32_t)a.n_tok + (int32_t)t + 1;
			qp[h] = (const T *)a.q + ((size_t)(s * a.n_tok + t) * a.n_head + kvh * a.gqa +
						  r % a.gqa) * HD;
		}
	}
	const int32_t least = min(min(__reduce_min_sync(0xffffffffu, limit[0]),
				      __reduce_min_sync(0xffffffffu, limit[1])), k1);

	uint32_t qa[KS][4];
#pragma unroll
	for (int ks = 0; ks < KS; ks++)
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const T *src = qp[j & 1];
			qa[ks][j] = src ? __ldcg((const uint32_t *)(src + ks * 16 + (j >> 1) * 8 + c * 2)) : 0u;
		}

	float o[NT][4];
	float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
	for (int n = 0; n < NT; n++)
		o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

	constexpr uint32_t TILE_BYTES = ATTN_KEYS * HD * 2;
	uint8_t *stage0 = asm_ + (size_t)warp * 4 * TILE_BYTES;
	const T *kbase = (const T *)a.p.k + a.layer * a.p.layer_stride + kvh * a.p.head_stride;
	const T *vbase = (const T *)a.p.v + a.layer * a.p.layer_stride + kvh * a.p.head_stride;
	const int32_t *row = a.p.table + (size_t)slot * a.p.max_pages;

	auto load = [&](int st, int32_t key0) {
		const uint32_t ks = smem_addr(stage0 + st * 2 * TILE_BYTES), vs = ks + TILE_BYTES;
#pragma unroll
		for (int it = 0; it < (int)ATTN_KEYS * KW / 32; it++) {
			const uint32_t key = it * (32 / KW) + lane / KW, w = lane % KW;
			const int32_t pos = key0 + (int32_t)key;
			bool ok = pos < k1;
			int32_t page = 0;
			if (ok) {
				page = __ldcg(&row[pos / a.p.page]);
				ok = (uint32_t)page < a.p.n_pages;
				page = ok ? page : 0;
			}
			const uint64_t off = page * a.p.page_stride +
					     (uint32_t)(pos % a.p.page) * a.p.pos_stride + w * 8;
			const uint32_t dst = key * HD * 2 + ((w ^ (key & 7)) << 4);
			cp_async16_or_zero(ks + dst, kbase + off, ok);
			cp_async16_or_zero(vs + dst, vbase + off, ok);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};

	const int32_t first = k0 + (int32_t)(warp * ATTN_KEYS), step = (int32_t)ATTN_GRAIN;
	if (first < k1)
		load(0, first);
	int st = 0;
	for (int32_t key0 = first; key0 < k1; key0 += step, st ^= 1) {
		if (key0 + step < k1) {
			load(st ^ 1, key0 + step);
			asm volatile("cp.async.wait_group 1;" ::: "memory");
		} else {
			asm volatile("cp.async.wait_group 0;" ::: "memory");
		}
		__syncwarp();
		const uint32_t ks = smem_addr(stage0 + st * 2 * TILE_BYTES), vs = ks + TILE_BYTES;
		float s[4][4];
#pragma unroll
		for (int j = 0; j < 4; j++) {
			s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
			const uint32_t key = j * 8 + (lane & 7);
#pragma unroll
			for (int k2 = 0; k2 < KS / 2; k2++) {
				uint32_t kb[4];
				ldmatrix_x4(kb, ks + key * HD * 2 + (((k2 * 4 + lane / 8) ^ (key & 7)) << 4));
				mma_16816<T>(s[j], qa[2 * k2], kb[0], kb[1]);
				mma_16816<T>(s[j], qa[2 * k2 + 1], kb[2], kb[3]);
			}
		}
		const bool ragged = key0 + (int32_t)ATTN_KEYS > least;
		float mx[2] = {m[0], m[1]};
#pragma unroll
		for (int j = 0; j < 4; j++)
#pragma unroll
			for (int e = 0; e < 4; e++) {
				s[j][e] *= a.scale;
				if (ragged && key0 + j * 8 + (int32_t)c * 2 + (e & 1) >= min(limit[e >> 1], k1))
					s[j][e] = -INFINITY;
				mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
			}
#pragma unroll
		for (int h = 0; h < 2; h++) {
			mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
			mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
			const float base = mx[h] == -INFINITY ? 0.0f : mx[h];
			const float keep = exp2_approx(m[h] - base);
			m[h] = mx[h];
			l[h] *= keep;
#pragma unroll
			for (int n = 0; n < NT; n++) {
				o[n][2 * h] *= keep;
				o[n][2 * h + 1] *= keep;
			}
#pragma unroll
			for (int j = 0; j < 4; j++) {
				s[j][2 * h] = exp2_approx(s[j][2 * h] - base);
				s[j][2 * h + 1] = exp2_approx(s[j][2 * h + 1] - base);
				l[h] += s[j][2 * h] + s[j][2 * h + 1];
			}
		}
		// A weight of 0 must take nothing from its key, and 0 * inf is NaN: where
		// some row of the tile does not see some key that others do, V is
		// searched for inf and NaN, and such a tile goes key by key.
		bool plain = true;
		if (ragged && key0 + (int32_t)ATTN_KEYS > least && least < k1) {
			bool bad = false;
			for (uint32_t w = lane; w < TILE_BYTES / 4; w += 32) {
				uint32_t two;
				asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(vs + w * 4) : "memory");
				const uint32_t e = sizeof(T) && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
				bad |= (two & e) == e || ((two >> 16) & e) == e;
			}
			plain = !__any_sync(0xffffffffu, bad);
		}
		if (plain) {
#pragma unroll
			for (int k16 = 0; k16 < 2; k16++) {
				const uint32_t pa[4] = {pack_pair<T>(s[2 * k16][0], s[2 * k16][1]),
							pack_pair<T>(s[2 * k16][2], s[2 * k16][3]),
							pack_pair<T>(s[2 * k16 + 1][0], s[2 * k16 + 1][1]),
							pack_pair<T>(s[2 * k16 + 1][2], s[2 * k16 + 1][3])};
				const uint32_t key = k16 * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
				for (int n2 = 0; n2 < NT / 2; n2++) {
					uint32_t vb[4];
					ldmatrix_x4_trans(vb, vs + key * HD * 2 +
							  (((n2 * 2 + (lane >> 4)) ^ (key & 7)) << 4));
					mma_16816<T>(o[2 * n2], pa, vb[0], vb[1]);
					mma_16816<T>(o[2 * n2 + 1], pa, vb[2], vb[3]);
				}
			}
		} else {
#pragma unroll 1
			for (int key = 0; key < (int)ATTN_KEYS; key++) {
				float w[2];
#pragma unroll
				for (int h = 0; h < 2; h++) {
					float x = 0.0f;
#pragma unroll
					for (int j = 0; j < 4; j++)
						if (key / 8 == j)
							x = key & 1 ? s[j][2 * h + 1] : s[j][2 * h];
					w[h] = to_float<T>(T(__shfl_sync(0xffffffffu, x, (lane & ~3u) + (key % 8) / 2)));
				}
#pragma unroll
				for (int n = 0; n < NT; n++) {
					uint32_t two;
					asm volatile("ld.shared.u32 %0, [%1];"
						     : "=r"(two)
						     : "r"(vs + key * HD * 2 + ((n ^ (key & 7)) << 4) + c * 4)
						     : "memory");
					T v[2];
					*(uint32_t *)v = two;
#pragma unroll
					for (int e = 0; e < 4; e++)
						if (key0 + key < min(limit[e >> 1], k1))
							o[n][e] = __fmaf_rn(w[e >> 1], to_float<T>(v[e & 1]), o[n][e]);
				}
			}
		}
		__syncwarp();
	}
	// join the warps: rows' maxima and sums, then the outputs through shared memory
#pragma unroll
	for (int h = 0; h < 2; h++) {
		l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
		l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
		if (c == 0) {
			s_m[warp][lane / 4 + 8 * h] = m[h];
			s_l[warp][lane / 4 + 8 * h] = l[h];
		}
	}
	__syncthreads();
	float *os = reinterpret_cast<float *>(asm_);        // [warps][16][HD]
#pragma unroll
	for (int n = 0; n < NT; n++)
#pragma unroll
		for (int h = 0; h < 2; h++)
			*(float2 *)(os + ((size_t)warp * ATTN_TILE_ROWS + lane / 4 + 8 * h) * HD + n * 8 +
				    c * 2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
	__syncthreads();
	const uint32_t r = tid / 8, rr = tile * ATTN_TILE_ROWS + r;
	if (rr >= n_rows)
		return;
	float top = -INFINITY, sum = 0.0f, f[ATTN_WARPS];
#pragma unroll
	for (int w = 0; w < (int)ATTN_WARPS; w++)
		top = fmaxf(top, s_m[w][r]);
	const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
	for (int w = 0; w < (int)ATTN_WARPS; w++) {
		f[w] = exp2_approx(s_m[w][r] - base);
		sum += f[w] * s_l[w][r];
	}
	const size_t at = ((size_t)((s0 + rr / tg) * a.n_tok + rr % tg / a.gqa) * a.n_head +
			   kvh * a.gqa + rr % a.gqa) * pieces + slot_at;
	const float inv = sum != 0.0f ? __fdiv_rn(1.0f, sum) : 0.0f;
	if (tid % 8 == 0)
		a.part_w[at] = sum != 0.0f ? base + log2f(sum) : -INFINITY;
	for (uint32_t i = (tid % 8) * 4; i < HD; i += 32) {
		float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
		for (int w = 0; w < (int)ATTN_WARPS; w++)
#pragma unroll
			for (int e = 0; e < 4; e++)
				v[e] += f[w] * os[((size_t)w * ATTN_TILE_ROWS + r) * HD + i + e];
		*(float4 *)(a.part_o + at * HD + i) =
			make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
	}
}

// The pieces of each row joined: one warp a row (sequence, token, head).
template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_join_kernel(const __grid_constant__ AttnArgs a)
{
	pdl_wait();
	pdl_launch_dependents();
	const uint32_t lane = threadIdx.x & 31;
	const size_t row = (size_t)blockIdx.x * 8 + threadIdx.x / 32;
	if (row >= (size_t)a.n_seq * a.n_tok * a.n_head)
		return;
	constexpr int EACH = HD / 32;
	const uint32_t s = (uint32_t)(row / ((size_t)a.n_tok * a.n_head)), pieces = a.pre_splits + a.own_splits;
	float v[EACH];
#pragma unroll
	for (int e = 0; e < EACH; e++)
		v[e] = 0.0f;
	if (attn_len(a, s) > 0) {
		const uint32_t first = attn_group_of(a, s).keys ? 0 : a.pre_splits;
		const float *w = a.part_w + row * pieces;
		float top = -INFINITY, sum = 0.0f;
		bool any = false;                       // (a NaN is no maximum, but it is a weight)
		for (uint32_t j = first; j < pieces; j++) {
			top = fmaxf(top, w[j]);
			any |= w[j] != -INFINITY;
		}
		top = top == -INFINITY ? 0.0f : top;
		if (any) {
			for (uint32_t j = first; j < pieces; j++) {
				if (w[j] == -INFINITY)
					continue;
				const float f = exp2_approx(w[j] - top);
				sum += f;
				const float *o = a.part_o + (row * pieces + j) * HD + lane * EACH;
#pragma unroll
				for (int e = 0; e < EACH; e++)
					v[e] += f * o[e];
			}
			const float inv = __fdiv_rn(1.0f, sum);
#pragma unroll
			for (int e = 0; e < EACH; e++)
				v[e] *= inv;
		}
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
