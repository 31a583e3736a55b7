// SPDX-License-Identifier: GPL-2.0-or-later
// The shared prefix of a group on the tensor cores (tcgen05): up to 256 rows
// (queries of one KV head: sequence, token, head of the group) against one piece of
// the prefix's keys, one CTA.
//
// With r rows sharing K and V, a key costs 4 r hd operations for its 4 hd bytes: at
// 256 rows the tensor cores and HBM are about balanced, and the softmax's r
// exponentials a key (16 a cycle and multiprocessor) cost as much as the products
// of hd = 128. So the three must overlap:
//
//   warp 9      copies K and V tiles of 128 keys, page by page, by tensor copies
//               (128-byte swizzle) into a ring
//   warp 8      issues the MMAs, in steps of 64 keys (half a tile): S = Q K^T (M = 128
//               rows, N = 64 keys) into tensor memory, and O += P V with P read
//               from tensor memory, where it lies over the S it was made of, and V
//               as an operand whose N (hd) is the contiguous side
//   warps 0-7   two streams of 128 rows, a thread a row: scores out of tensor
//               memory, maximum, exponentials, the sum, P back
//
// A stream's scores have two buffers and run two steps ahead of its outputs, so the
// exponentials of a step find their scores ready, and the tensor cores work for
// one stream while the other is in its exponentials. With more than 128 rows in the
// unit the streams are its two halves; with fewer they are the same rows over the
// even and the odd tiles, joined with the other pieces at the end.
//
// The MMA thread must do next to nothing between MMAs: one takes 64 cycles (N = 128, at
// the tensor cores' full rate; 48 for scores of N = 64, by the shared memory they read),
// and descriptors put together in 64 bits for each cost 120 to 170. Here a descriptor's
// high word is a constant and its low word a running sum.
//
// What bounds it: a step of 2 x 128 rows by 64 keys takes 0.9 us, of which 0.54 are the
// exponentials alone and 0.68 the MMAs alone; they overlap across the two streams but not with
// a stream's own tensor memory loads. 64 sequences of 4 rows on 16384 keys, 8 KV heads of 128, on 88
// multiprocessors: 38 us, 17.2 GFLOP, 450 TFLOP/s (0.45 of those multiprocessors' share of
// the measured bf16 rate), every key read once (67 MB). With scores of 128 keys in one
// buffer a tile takes 2.4 us, not 1.8; with two threads a row the whole spills, 38 against
// 31 us at that time.
//
// O is scaled only where a row's maximum has grown by more than 2^8 since it was
// last taken (P stays below 2^8, exact enough in both types); the weight of the
// piece is taken with the same maximum, so the result is the same.
#pragma once

#include "attn.cuh"
#include "tcgen05.cuh"

namespace cgpu {

constexpr uint32_t ATC_KEYS = 128, ATC_ROWS = 256;
constexpr uint32_t ATC_STEP = 64;                    // keys of a step: half a tile
constexpr int ATC_THREADS = 320;
constexpr uint32_t ATC_SLAB = ATC_KEYS * 128;        // 128 rows of 64 elements

// Tiles in the ring: what fits beside Q; one more where Q is 128 rows (a half of it is a tile)
template <int HD>
__host__ __device__ constexpr uint32_t atc_ring()
{
	return HD == 128 ? 5 : 10;
}

template <int HD>
constexpr size_t atc_smem()
{
	return ((size_t)ATC_ROWS + atc_ring<HD>() * ATC_KEYS) * HD * 2;      // on a 1024-byte boundary
}

// Shared-memory descriptors, 128-byte swizzle (8 rows of 128 bytes an atom, 1024 bytes on to
// the next 8 rows), version 1 (sm_100): the low word has the address and, for an
// N-major operand, the distance between 64-element columns of atoms.
constexpr uint32_t ATC_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);

__device__ __forceinline__ uint32_t atc_desc_lo(uint32_t addr, uint32_t lbo)
{
	return (addr >> 4) | ((lbo >> 4) << 16);
}

// dense kind::f16 MMA, D fp32, M = 128: A and B both fp16 (0) or both bf16 (1); B
// N-major where b_mn
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t bf16, uint32_t n, bool b_mn)
{
	return (1u << 4) | (bf16 << 7) | (bf16 << 10) | ((uint32_t)b_mn << 16) | ((n >> 3) << 17) |
	       ((128u >> 4) << 24);
}

// D (+)= A B^T, descriptors by their low words
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
					   uint32_t accumulate)
{
	asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
		     "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
		     "setp.ne.b32 p, %5, 0;\n\t"
		     "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
		     :: "r"(d), "r"(a_lo), "r"(b_lo), "r"(ATC_DESC_HI), "r"(idesc), "r"(accumulate) : "memory");
}

// A from tensor memory: 16 bits a value, two a word, a row a lane
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc,
					   uint32_t accumulate)
{
	asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
		     "mov.b64 b, {%2, %3};\n\t"
		     "setp.ne.b32 p, %5, 0;\n\t"
		     "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
		     :: "r"(d), "r"(a), "r"(b_lo), "r"(ATC_DESC_HI), "r"(idesc), "r"(accumulate) : "memory");
}

// one lane of a converged warp
__device__ __forceinline__ bool elect_lane()
{
	uint32_t r;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
	return r;
}

// 32 lanes x 32 consecutive columns
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *r)
{
	uint32_t *u = reinterpret_cast<uint32_t *>(r);
	asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
		     "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
		     "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
		     : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
		       "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]),
		       "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
		       "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
		       "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]),
		       "=r"(u[31])
		     : "r"(taddr));
}

// The wait for such loads does not name their registers, so nothing would keep the
// compiler from using them before it: this makes them its results.
__device__ __forceinline__ void tmem_loaded32(float *r)
{
	uint32_t *u = reinterpret_cast<uint32_t *>(r);
#pragma unroll
	for (int i = 0; i < 32; i += 8)
		asm volatile("" : "+r"(u[i]), "+r"(u[i + 1]), "+r"(u[i + 2]), "+r"(u[i + 3]), "+r"(u[i + 4]),
				  "+r"(u[i + 5]), "+r"(u[i + 6]), "+r"(u[i + 7]));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *u)
{
	asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
		     "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
		     "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
		     :: "r"(taddr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
		     "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]),
		     "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
		     "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]),
		     "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
		     : "memory");
}

// codes of a wait that gave up, after the batched matvec's (5 to 13)
constexpr int ATC_ERR_RING = 21, ATC_ERR_MMA = 22, ATC_ERR_ROWS = 23;

template <typename T, int HD>
__global__ void __launch_bounds__(ATC_THREADS, 1)
attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap,
	       const __grid_constant__ CUtensorMap vmap)
{
	constexpr uint32_t NB = atc_ring<HD>(), SLABS = HD / 64, TILE = ATC_KEYS * HD * 2;
	constexpr uint32_t COL_S = 0, COL_O = 256;      // S (and P) 128 columns a stream, then O
	extern __shared__ __align__(1024) uint8_t atc_raw[];
	__shared__ __align__(8) uint64_t b_full[NB + 1], b_free[NB + 1], b_q, b_s[2][2], b_p[2][2], b_o[2], b_end;
	__shared__ uint32_t s_tmem, s_row[ATC_ROWS];
	constexpr uint32_t NO_ROW = 0xffffffffu;
	const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const uint32_t q_at = smem_addr(atc_raw);
	uint8_t *q_ptr = atc_raw;

	pdl_wait();
	pdl_launch_dependents();

	// which rows, which keys (every warp for itself). The launch has room for more units
	// than there may be (each group can end in a part of one): those leave at once.
	const uint32_t kvh_n = a.p.n_head_kv, tg = a.n_tok * a.gqa, splits = a.pre_splits / 2;
	uint32_t b = blockIdx.x;
	const uint32_t u = b / (kvh_n * splits);
	b -= u * kvh_n * splits;
	const uint32_t piece = b / kvh_n, kvh = b - piece * kvh_n;
	AttnUnit unit;
	if (!attn_find_unit(a, u, ATC_ROWS, &unit))
		return;
	const uint32_t tile = unit.tile;
	if (warp == 8) {
		if (lane == 0) {
			for (uint32_t i = 0; i <= NB; i++) {
				mbar_init(&b_full[i], 1);
				mbar_init(&b_free[i], 1);
			}
			mbar_init(&b_q, 256);
			mbar_init(&b_end, 1);
			for (int i = 0; i < 2; i++) {
				for (int h = 0; h < 2; h++) {
					mbar_init(&b_s[i][h], 1);
					mbar_init(&b_p[i][h], 128);
				}
				mbar_init(&b_o[i], 1);
			}
			fence_mbar_init();
		}
		__syncwarp();
		tmem_alloc(&s_tmem, 512);
		tmem_relinquish();
	}
	const AttnGroup gr = attn_group(a, unit.b0, unit.b1, unit.told);
	int32_t k0 = 0, k1 = gr.keys;
	attn_piece(k0, k1, piece, splits, ATC_KEYS);
	const uint32_t n_rows = (gr.s1 - gr.s0) * tg, row0 = tile * ATC_ROWS;
	const bool halves = n_rows - row0 > 128;
	const uint32_t q_slab = halves ? 256 * 128 : 128 * 128, ring = q_at + q_slab * SLABS;
	// copy c's place in the ring, and which time round
	auto at_of = [&](uint32_t c) { return halves ? c % NB : c % (NB + 1); };
	auto turn_of = [&](uint32_t c) { return halves ? c / NB : c / (NB + 1); };
	const uint32_t tiles = (uint32_t)(k1 - k0 + (int32_t)ATC_KEYS - 1) / ATC_KEYS;
	const uint32_t pieces = a.pre_splits + a.own_splits;
	// a row of the unit by its number among q's rows: (sequence, token, head)
	if (threadIdx.x < ATC_ROWS) {
		// (none: behind the last, or a query that sees nothing, as its own pieces say)
		const uint32_t r = row0 + threadIdx.x, s = gr.s0 + r / tg, x = r % tg;
		s_row[threadIdx.x] = r < n_rows && attn_len(a, s)
					     ? (s * a.n_tok + x / a.gqa) * a.n_head + kvh * a.gqa + x % a.gqa
					     : NO_ROW;
	}
	// the steps of stream i: its tiles' halves, but a last one without keys
	auto count = [&](uint32_t i) {
		const uint32_t n = halves ? tiles : (tiles + 1 - i) / 2;
		const bool last = halves || (tiles - 1) % 2 == i;
		return 2 * n - (last && (uint32_t)(k1 - k0) <= (tiles - 1) * ATC_KEYS + ATC_STEP);
	};
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = s_tmem;

	if (!tiles) {
		// nothing in this piece (a group with fewer rows or keys than the launch has room for)
		if (gr.keys && threadIdx.x < ATC_ROWS && s_row[threadIdx.x] != NO_ROW) {
			float *w = a.part_w + (size_t)s_row[threadIdx.x] * pieces + 2 * piece;
			w[0] = w[1] = -INFINITY;
		}
	} else if (warp == 9) {
		// ---- K and V tiles into the ring, in the order in which they are asked for: a tile's K,
		// then its V; of two streams on the same rows, both their K first
		const uint32_t box = attn_box(a.p.page), per = ATC_KEYS / box;     // positions; boxes a tile
		const int32_t *row = a.p.table + (size_t)gr.slot * a.p.max_pages;
		const uint32_t my_box = lane % per, my_slab = lane / per;
		bool ok = true;
		uint32_t c = 0, issued = 0, turns = 0;           // (bits by place: copied to, the turn's parity)
		// a page past the piece, or no page at all, reads as zeros
		auto pos_of = [&](uint32_t j) { return (uint32_t)k0 + j * ATC_KEYS + my_box * box; };
		auto page_of = [&](uint32_t j) {
			const uint32_t pos = pos_of(j);
			const uint32_t page = pos < (uint32_t)k1 ? (uint32_t)__ldcg(&row[pos / a.p.page]) : a.p.n_pages;
			return (int)min(page, a.p.n_pages);
		};
		const uint32_t group = halves ? 1 : 2;
		int page[2] = {page_of(0), page_of(1)};
		for (uint32_t j = 0; j < tiles && ok; j += group) {
			const int next[2] = {page_of(j + group), page_of(j + group + 1)};
			for (uint32_t x = 0; x < 2 * group; x++, c++) {
				const uint32_t v = x / group, t = x % group;
				if (j + t >= tiles)
					continue;                  // (of the last pair, where tiles is odd)
				const uint32_t at = at_of(c), turn = turn_of(c);
				if (turn)
					ok = __all_sync(0xffffffffu, mbar_wait_bounded(&b_free[at], (turn - 1) & 1,
										       WAIT_LIMIT_NS));
				if (!ok)
					break;
				if (lane == 0)
					mbar_arrive_expect_tx(&b_full[at], TILE);
				__syncwarp();
				if (my_slab < SLABS)
					tma_load_4d(ring + at * TILE + my_slab * ATC_SLAB + my_box * box * 128,
						    v ? &vmap : &kmap, (int)(my_slab * 64),
						    (int)(pos_of(j + t) % a.p.page), (int)kvh, page[t], &b_full[at]);
				__syncwarp();
				issued |= 1u << at;
				turns = (turns & ~(1u << at)) | (turn & 1) << at;
			}
			page[0] = next[0];
			page[1] = next[1];
		}
		// every copy issued lands before the CTA leaves (already so unless a wait gave up)
		if (!ok && lane == 0)
			*(volatile int *)a.err = ATC_ERR_RING;
		for (uint32_t i = 0; i <= NB; i++)
			if ((issued >> i & 1) && !mbar_wait_bounded(&b_full[i], turns >> i & 1, WAIT_LIMIT_NS) &&
			    lane == 0)
				*(volatile int *)a.err = ATC_ERR_RING;
	} else if (warp == 8) {
		if (elect_lane()) {
			// ---- the MMAs
			constexpr uint32_t BF = std::is_same<T, __nv_bfloat16>::value;
			constexpr uint32_t id_s = idesc_f16(BF, ATC_STEP, false), id_o = idesc_f16(BF, HD, true);
			bool ok = mbar_wait_bounded(&b_q, 0, WAIT_LIMIT_NS);
			tc_fence_after();
			const uint32_t n0 = count(0), n1 = count(1), q_next = q_slab >> 4;
			// where each stream's next tile of K and of V is in the ring; waited for, and
			// given back after its second half, once a tile
			const uint32_t nb = halves ? NB : NB + 1;
			struct Place {
				uint32_t at, turn;
			} kp[2] = {{0, 0}, {halves ? 0u : 1u, 0}}, vp[2] = {{halves ? 1u : 2u, 0}, {halves ? 1u : 3u, 0}};
			auto advance = [&](Place &p) {
				p.at += halves ? 2 : 4;
				if (p.at >= nb) {
					p.at -= nb;
					p.turn ^= 1;
				}
			};
			auto scores = [&](uint32_t i, uint32_t n) {      // S of stream i's step n
				Place &p = kp[i];
				if (!(n & 1))
					ok = ok && mbar_wait_bounded(&b_full[p.at], p.turn, WAIT_LIMIT_NS);
				if (!ok)
					return;
				const uint32_t qa = atc_desc_lo(q_at + (halves ? i * 128 * 128 : 0), 16);
				const uint32_t ka = atc_desc_lo(ring + p.at * TILE + (n & 1) * (ATC_STEP * 128), 16);
				const uint32_t d = tmem + COL_S + i * 128 + (n & 1) * ATC_STEP;
#pragma unroll
				for (uint32_t k = 0; k < HD / 16; k++)
					mma_f16_ss(d, qa + (k / 4) * q_next + (k % 4) * 2,
						   ka + (k / 4) * (ATC_SLAB >> 4) + (k % 4) * 2, id_s, k != 0);
				mma_commit(&b_s[i][n & 1]);
				if (n & 1) {
					if (!halves || i == 1)
						mma_commit(&b_free[p.at]);
					advance(p);
				}
			};
			auto outputs = [&](uint32_t i, uint32_t n) {     // O += P V of the same
				Place &p = vp[i];
				if (!(n & 1))
					ok = ok && mbar_wait_bounded(&b_full[p.at], p.turn, WAIT_LIMIT_NS);
				ok = ok && mbar_wait_bounded(&b_p[i][n & 1], (n / 2) & 1, WAIT_LIMIT_NS);
				if (!ok)
					return;
				tc_fence_after();
				const uint32_t va = atc_desc_lo(ring + p.at * TILE + (n & 1) * (ATC_STEP * 128), ATC_SLAB);
				const uint32_t d = tmem + COL_O + i * HD, pa = tmem + COL_S + i * 128 + (n & 1) * ATC_STEP;
#pragma unroll
				for (uint32_t k = 0; k < ATC_STEP / 16; k++)
					mma_f16_ts(d, pa + k * 8, va + k * (16 * 128 >> 4), id_o, k ? 1 : n);
				mma_commit(&b_o[i]);
				if (n & 1) {
					if (!halves || i == 1)
						mma_commit(&b_free[p.at]);
					advance(p);
				}
			};
			// scores two steps ahead of the outputs
			for (uint32_t n = 0; n < 2; n++) {
				if (n < n0)
					scores(0, n);
				if (n < n1)
					scores(1, n);
			}
#pragma unroll 2
			for (uint32_t n = 0; n < n0 && ok; n++) {
				outputs(0, n);
				if (n + 2 < n0)
					scores(0, n + 2);
				if (n < n1)
					outputs(1, n);
				if (n + 2 < n1)
					scores(1, n + 2);
			}
			// all MMAs done before tensor memory is freed
			mma_commit(&b_end);
			if (!mbar_wait_bounded(&b_end, 0, WAIT_LIMIT_NS) || !ok)
				*(volatile int *)a.err = ATC_ERR_MMA;
		}
		__syncwarp();
	} else {
		// ---- rows: Q into shared memory first (swizzled as the tensor copies would)
		const uint32_t rows = halves ? 256 : 128;
		// scale > 0 from here on: Q's sign takes the scale's, and of a scale of 0 Q is 0 (0 times
		// the -inf of a key behind the end would be NaN)
		const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale != 0.0f ? 0xffffffffu : 0u;
		constexpr uint32_t QW = HD / 8, EACH = 128 * QW / 256;      // words a row; a thread's in 128 rows
		const uint32_t w = threadIdx.x % QW;
		for (uint32_t r0 = 0; r0 < rows; r0 += 128) {
			uint4 v[EACH];
#pragma unroll
			for (uint32_t e = 0; e < EACH; e++) {
				const uint32_t row = s_row[r0 + e * (256 / QW) + threadIdx.x / QW];
				v[e] = row == NO_ROW ? make_uint4(0, 0, 0, 0)
						     : __ldcg((const uint4 *)((const T *)a.q + (size_t)row * HD + w * 8));
			}
#pragma unroll
			for (uint32_t e = 0; e < EACH; e++) {
				const uint32_t r = r0 + e * (256 / QW) + threadIdx.x / QW;
				*(uint4 *)(q_ptr + (w / 8) * q_slab + r * 128 + (((w % 8) ^ (r & 7)) << 4)) =
					make_uint4((v[e].x ^ flip) & keep, (v[e].y ^ flip) & keep, (v[e].z ^ flip) & keep,
						   (v[e].w ^ flip) & keep);
			}
		}

		const uint32_t i = warp / 4, quarter = warp % 4, mine = count(i);
		const uint32_t lanes = (quarter * 32) << 16, my = s_row[(halves ? i * 128 : 0) + quarter * 32 + lane];
		const uint32_t ts = tmem + lanes + COL_S + i * 128, to = tmem + lanes + COL_O + i * HD;
		const float scale = keep ? fabsf(a.scale) : 1.0f;
		float m = -INFINITY, l = 0.0f;
		bool ok = true;
		fence_proxy_async_smem();
		mbar_arrive(&b_q);
		for (uint32_t n = 0; n < mine; n++) {
			ok = __all_sync(0xffffffffu, mbar_wait_bounded(&b_s[i][n & 1], (n / 2) & 1, WAIT_LIMIT_NS));
			if (!ok)
				break;
			tc_fence_after();
			const uint32_t tn = ts + (n & 1) * ATC_STEP;
			float s[64];
			tmem_ld32(tn, s);
			tmem_ld32(tn + 32, s + 32);
			tmem_wait_ld();
			tmem_loaded32(s);
			tmem_loaded32(s + 32);
			const uint32_t j = halves ? n / 2 : 2 * (n / 2) + i;
			const int32_t in_step = k1 - k0 - (int32_t)(j * ATC_KEYS + (n & 1) * ATC_STEP);
			if (in_step < (int32_t)ATC_STEP) {
#pragma unroll
				for (int c = 0; c < 64; c++)
					if (c >= in_step)
						s[c] = -INFINITY;
			}
			float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
			for (int c = 0; c < 64; c++)
				mx[c & 3] = fmaxf(mx[c & 3], s[c]);
			mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
			if (n == 0) {
				m = mx[0];
			} else if (__any_sync(0xffffffffu, (mx[0] - m) * scale > 8.0f)) {
				const float f = mx[0] == m ? 1.0f : exp2_approx((m - mx[0]) * scale);
				ok = __all_sync(0xffffffffu,
						mbar_wait_bounded(&b_o[i], (n - 1) & 1, WAIT_LIMIT_NS));
				if (!ok)
					break;
				tc_fence_after();
#pragma unroll 1
				for (int c = 0; c < HD / 32; c++) {
					float o[32];
					tmem_ld32(to + 32 * c, o);
					tmem_wait_ld();
					tmem_loaded32(o);
#pragma unroll
					for (int e = 0; e < 32; e++)
						o[e] *= f;
					tmem_st32(to + 32 * c, reinterpret_cast<uint32_t *>(o));
				}
				l *= f;
				m = mx[0];
			}
			const float base = m == -INFINITY ? 0.0f : -m * scale;
			const uint64_t scale2 = pack2(scale, scale), base2 = pack2(base, base);
			uint64_t sum[2] = {0, 0};                // pairs of sums
			uint32_t p[32];
#pragma unroll
			for (int c = 0; c < 32; c++) {
				const uint64_t x = fma2_rn(pack2(s[2 * c], s[2 * c + 1]), scale2, base2);
				const float e0 = exp2_approx(lo2(x)), e1 = exp2_approx(hi2(x));
				sum[c & 1] = add2_rn(sum[c & 1], pack2(e0, e1));
				p[c] = pack_pair<T>(e0, e1);
			}
			tmem_st32(tn, p);
			l += (lo2(sum[0]) + hi2(sum[0])) + (lo2(sum[1]) + hi2(sum[1]));
			tmem_wait_st();
			tc_fence_before();
			mbar_arrive(&b_p[i][n & 1]);
		}
		// all MMAs are done: the outputs go out through the ring, 32 columns of a warp's 32
		// rows at a time, so that a row's 128 bytes leave together
		ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(&b_end, 0, WAIT_LIMIT_NS));
		if (!ok && lane == 0)
			*(volatile int *)a.err = ATC_ERR_ROWS;
		if (ok) {
			tc_fence_after();
			const uint32_t col = 2 * piece + (halves ? 0 : i);
			const float inv = l != 0.0f ? __fdiv_rn(1.0f, l) : 0.0f;
			if (my != NO_ROW) {
				float *pw = a.part_w + (size_t)my * pieces + col;
				pw[0] = l != 0.0f ? (m == -INFINITY ? 0.0f : m * scale) + log2f(l) : -INFINITY;
				if (halves)
					pw[1] = -INFINITY;
			}
			float *stage = reinterpret_cast<float *>(q_ptr + (ring - q_at)) + warp * (32 * 36);
#pragma unroll 1
			for (int c = 0; mine && c < HD / 32; c++) {
				float o[32];
				tmem_ld32(to + 32 * c, o);
				tmem_wait_ld();
				tmem_loaded32(o);
#pragma unroll
				for (int e = 0; e < 32; e += 4)
					*(float4 *)(stage + lane * 36 + e) = make_float4(o[e] * inv, o[e + 1] * inv,
											 o[e + 2] * inv, o[e + 3] * inv);
				__syncwarp();
#pragma unroll
				for (int e = 0; e < 8; e++) {
					const uint32_t row = e * 4 + lane / 8, at = __shfl_sync(0xffffffffu, my, row);
					if (at != NO_ROW)
						*(float4 *)(a.part_o + ((size_t)at * pieces + col) * HD + 32 * c +
							    (lane % 8) * 4) =
							*(float4 *)(stage + row * 36 + (lane % 8) * 4);
				}
				__syncwarp();
			}
		}
		tc_fence_before();
	}
	__syncthreads();
	if (warp == 8) {
		tc_fence_after();
		tmem_dealloc(tmem, 512);
	}
}

} // namespace cgpu
