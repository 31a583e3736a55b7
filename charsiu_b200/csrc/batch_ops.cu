// SPDX-License-Identifier: GPL-2.0-or-later
// The operators of a batched step: argument checks, launch shapes and the C entry
// points of include/charsiu_gpu.h. The kernels are in norm_rows.cuh, pages.cuh,
// attn.cuh, attn_tc.cuh and adapters.cuh.
//
// Every launch has the programmatic attribute, and every kernel waits for its
// predecessor before it reads or writes anything of the caller's (one, behind a launch
// of its own call, waits at its end: attn_rows_kernel).
#include <cuda_runtime.h>
#include <cudaTypedefs.h>          // PFN_cuTensorMapEncodeTiled

#include <atomic>
#include <cstdio>
#include <type_traits>

#include "charsiu_gpu.h"

#include "adapters.cuh"
#include "attn.cuh"
#include "attn_tc.cuh"
#include "batch_checks.h"
#include "layer_internal.h"
#include "norm_rows.cuh"
#include "pages.cuh"

using namespace cgpu;

namespace {

// The layer's GPU for the length of a call; the caller's current one after it.
struct OnDevice {
	int before = -1, device;
	explicit OnDevice(const charsiu_gpu *g) : device(layer_device(g))
	{
		if (cudaGetDevice(&before) != cudaSuccess)
			before = -1;
		if (before != device)
			cudaSetDevice(device);
	}
	~OnDevice()
	{
		if (before >= 0 && before != device)
			cudaSetDevice(before);
	}
};

int refuse(charsiu_gpu *g, const char *why)
{
	layer_whine(g, why);
	return -1;
}

template <typename K, typename... Args>
bool launch(charsiu_gpu *g, void *stream, K kernel, dim3 grid, unsigned block, size_t smem,
	    Args... args)
{
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid;
	cfg.blockDim = dim3(block);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream ? (cudaStream_t)stream : layer_stream(g);
	cudaLaunchAttribute attr[1];
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = attr;
	cfg.numAttrs = layer_no_pdl(g) ? 0 : 1;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
	if (e != cudaSuccess) {
		cudaGetLastError();
		char why[160];
		snprintf(why, sizeof(why), "the launch failed: %s", cudaGetErrorString(e));
		layer_whine(g, why);
		return false;
	}
	layer_launched(g, 1);
	return true;
}

// more than 48 KB of shared memory, asked for once a kernel and device; and the whole of a
// multiprocessor's as shared memory, so that CTAs of different kernels find room on one
template <typename K>
bool allow_smem(charsiu_gpu *g, K kernel, size_t bytes, std::atomic<uint64_t> &done)
{
	const uint64_t bit = 1ull << (layer_device(g) & 63);
	if (done & bit)
		return true;
	if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
		    cudaSuccess ||
	    cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
				 cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
		cudaGetLastError();
		layer_whine(g, "a kernel's shared memory was refused");
		return false;
	}
	done |= bit;
	return true;
}

// the start of every call on a cache: 0 to go on
int pages_check(charsiu_gpu *g, const charsiu_gpu_pages *p, bool lists)
{
	if (!g || layer_dead(g))
		return -1;
	const char *why = pages_fault(p);
	if (*why)
		return refuse(g, why);
	if (lists && !p->work)
		return refuse(g, "the cache has no work array");
	return 0;
}

int slots_check(charsiu_gpu *g, const charsiu_gpu_pages *p, const int32_t *slots, unsigned n)
{
	if (pages_check(g, p, true))
		return -1;
	const char *why = slots_fault(slots, n);
	return *why ? refuse(g, why) : 0;
}

template <typename T>
int append(charsiu_gpu *g, const charsiu_gpu_pages *p, unsigned layer, const int32_t *slots,
	   unsigned n, unsigned t, unsigned n_head, const float *q, const float *k, const float *v,
	   const float *rope_cs, unsigned n_ctx, void *q_out, void *stream)
{
	// two words a thread, as far as a CTA goes
	const uint64_t words = (n_head + 2ull * p->n_head_kv) * (p->head_dim / 8), half = (words / 2 + 31) / 32 * 32;
	const unsigned threads = half < APPEND_MAX_THREADS ? (unsigned)half : APPEND_MAX_THREADS;
	return launch(g, stream, pages_append_kernel<T>, dim3(n * t), threads, 0, *p, (uint32_t)layer, slots,
		      (uint32_t)t, (uint32_t)n_head, q, k, v, rope_cs, (uint32_t)n_ctx, (T *)q_out)
		       ? 0
		       : -1;
}

// ---- attention ------------------------------------------------------------------

constexpr uint32_t ATTN_CTAS_PER_SM = 2;     // of the rows kernel, by its shared memory
constexpr uint32_t ATTN_LONG = 2048;         // keys: about the most in a piece of a sequence

// How the work is cut. Returns whether the prefixes go to the tensor cores.
bool attention_plan(charsiu_gpu *g, const charsiu_gpu_pages *p, const charsiu_gpu_attention *b,
		    AttnArgs *a)
{
	const uint32_t gqa = b->n_head / p->n_head_kv, rows = b->n_tok * gqa;
	const uint32_t sms = (uint32_t)layer_sms(g);
	const uint64_t all = (uint64_t)b->n_seq * rows;
	auto splits = [&](uint64_t ctas, uint64_t aim, uint64_t pieces) {
		uint64_t n = ctas ? aim / ctas : 1;
		n = n > ATTN_MAX_SPLITS ? ATTN_MAX_SPLITS : n < 1 ? 1 : n;
		return (uint32_t)(n < pieces ? n : pieces);
	};
	a->gqa = gqa;
	a->own_tiles = (rows + ATTN_TILE_ROWS - 1) / ATTN_TILE_ROWS;
	a->own_splits = splits((uint64_t)b->n_seq * a->own_tiles * p->n_head_kv, ATTN_CTAS_PER_SM * sms,
			       b->max_len / ATTN_GRAIN + 1);
	// in a large batch a long sequence is cut all the same, or it would be the last to end
	a->own_grain = a->own_splits > 1 ? ATTN_GRAIN : 4 * ATTN_GRAIN;
	const uint32_t by_length = b->max_len / ATTN_LONG < ATTN_MAX_SPLITS ? b->max_len / ATTN_LONG : ATTN_MAX_SPLITS;
	a->own_splits = a->own_splits > by_length ? a->own_splits : by_length;
	a->pre_units = a->pre_splits = a->rows_splits = 0;
	if (!b->n_group)
		return false;
	// The tensor cores' form from 32 rows of a KV head on, over all groups; measured with one group. (Of
	// many small groups each fills a unit of its own, and the splits below, made from the rows of all, come
	// out as for one.) Measured with 4 rows a sequence, hd 64, against
	// 16 rows at a time in the rows kernel: 256 shared keys, 2 sequences 9.2 against 8.6 us, 16
	// 10.0 / 13.5; 4096, 8 20.7 / 17.4, 32 23.6 / 24.1, 64 27 / 37; 16384, 8 30.9 / 26.7, 16
	// 32 / 35, 64 40 / 100. Of hd 128, 256, 8 11.5 / 13.1; 16384, 4 36 / 31, 8 37 / 40, 64 49 / 176.
	const bool tc = all >= 32;
	const uint32_t unit = tc ? ATC_ROWS : ATTN_TILE_ROWS;
	const uint32_t units = (uint32_t)((all + unit - 1) / unit);
	// (three eighths of the multiprocessors are left to the rows kernel beside it: 48 queries of
	// 4 on 3 x 3000 keys of hd 64 take 37 us with the prefix on all and the rest after it,
	// 34 with a quarter left, 28 with three eighths; 64 on 16384 of hd 128 55, 58, 51)
	a->pre_splits = tc ? 2 * splits((uint64_t)units * p->n_head_kv, sms * 5 / 8, b->max_len / ATC_KEYS + 1)
			   : splits((uint64_t)units * p->n_head_kv, ATTN_CTAS_PER_SM * sms,
				    b->max_len / ATTN_GRAIN + 1);
	a->rows_splits = tc ? 0 : a->pre_splits;
	a->pre_units = (uint32_t)((all + (uint64_t)b->n_group * (unit - 1)) / unit);     // each group may end in a part of one
	return tc;
}

// Scratch for the pieces of this batch and of any smaller one: fewer sequences are
// cut finer, but n sequences of c CTAs each give at most n + aim / c pieces of
// each kind, which grows with n.
size_t attention_bytes(charsiu_gpu *g, const charsiu_gpu_pages *p, const charsiu_gpu_attention *b)
{
	const uint64_t kv = p->n_head_kv, n = b->n_seq, rows = (uint64_t)b->n_tok * (b->n_head / kv);
	const uint64_t tiles = (rows + ATTN_TILE_ROWS - 1) / ATTN_TILE_ROWS, most = ATTN_MAX_SPLITS * n;
	const uint64_t sms = (uint64_t)layer_sms(g);
	uint64_t parts = n + ATTN_CTAS_PER_SM * sms / (tiles * kv) + 1;
	parts = parts < most ? parts : most;
	const uint64_t by_length = n * (b->max_len / ATTN_LONG);
	parts = parts > by_length ? parts : by_length < most ? by_length : most;
	if (b->n_group) {
		const uint64_t pre = 2 * (n + sms * ATC_ROWS / (rows * kv) + 1);
		parts += pre < 2 * most ? pre : 2 * most;
	}
	return (size_t)(parts * b->n_tok * b->n_head * (p->head_dim + 1) * sizeof(float) + 15) / 16 * 16;
}

// K or V of one layer as (element, position, head, page); boxes of 64 elements and
// attn_box positions of a page. A dimension of one element has no stride to speak of.
bool attention_map(CUtensorMap *map, const charsiu_gpu_pages *p, const void *base, unsigned layer)
{
	const auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode());
	if (!enc)
		return false;
	const cuuint64_t dims[4] = {p->head_dim, p->page, p->n_head_kv, p->n_pages};
	const cuuint64_t row = 2ull * p->head_dim;
	const cuuint64_t strides[3] = {2 * p->pos_stride, p->n_head_kv > 1 ? 2 * p->head_stride : row,
				       p->n_pages > 1 ? 2 * p->page_stride : row};
	const cuuint32_t box[4] = {64, attn_box(p->page), 1, 1}, ones[4] = {1, 1, 1, 1};
	return enc(map, p->type == TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
		   4, (uint8_t *)const_cast<void *>(base) + 2 * layer * p->layer_stride, dims, strides, box, ones,
		   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
		   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
int attention(charsiu_gpu *g, AttnArgs &a, bool tc, void *stream)
{
	static std::atomic<uint64_t> smem_done, tc_done, join_done;
	CUtensorMap kmap, vmap;
	if (!attention_map(&kmap, &a.p, a.p.k, a.layer) || !attention_map(&vmap, &a.p, a.p.v, a.layer))
		return refuse(g, "the cache's strides cannot be described to the copy engine");
	if (!allow_smem(g, attn_rows_kernel<T, HD>, AttnRing<HD>::SMEM, smem_done) ||
	    !allow_smem(g, attn_tc_kernel<T, HD>, atc_smem<HD>(), tc_done) ||
	    !allow_smem(g, attn_join_kernel<T, HD>, 0, join_done))
		return -1;
	if (tc && !launch(g, stream, attn_tc_kernel<T, HD>,
			  dim3(a.pre_units * a.p.n_head_kv * (a.pre_splits / 2)), ATC_THREADS, atc_smem<HD>(), a,
			  kmap, vmap))
		return -1;
	if (tc) {
		// (without the room for groups' ends, whose CTAs leave at once)
		const uint64_t busy = (((uint64_t)a.n_seq * a.n_tok * a.gqa + ATC_ROWS - 1) / ATC_ROWS) *
				      a.p.n_head_kv * (a.pre_splits / 2);
		const uint64_t sms = layer_sms(g);
		a.pre_units = 0;
		a.behind = 1;
		a.early = busy + 8 <= sms ? (uint32_t)(ATTN_CTAS_PER_SM * (sms - busy)) : 0xffffffffu;
	}
	const uint64_t items = (uint64_t)a.p.n_head_kv * ((uint64_t)a.pre_units * a.rows_splits +
							  (uint64_t)a.n_seq * a.own_tiles * a.own_splits);
	const uint64_t grid = ATTN_CTAS_PER_SM * (uint64_t)layer_sms(g);
	const uint64_t rows = (uint64_t)a.n_seq * a.n_tok * a.n_head;
	return launch(g, stream, attn_rows_kernel<T, HD>, dim3((unsigned)(items < grid ? items : grid)),
		      ATTN_THREADS, AttnRing<HD>::SMEM, a, kmap, vmap) &&
			       launch(g, stream, attn_join_kernel<T, HD>,
				      dim3((unsigned)((rows + 7) / 8)), 256, 0, a)
		       ? 0
		       : -1;
}

// ---- adapters --------------------------------------------------------------------

// ranks a kernel holds: the largest of the sets', padded
uint32_t adapters_ranks(const charsiu_gpu_adapters *s, unsigned n)
{
	uint32_t most = 0;
	for (unsigned i = 0; i < n; i++)
		most = s[i].max_rank > most ? s[i].max_rank : most;
	return most <= 8 ? 8 : most <= 16 ? 16 : most <= 32 ? 32 : most <= 64 ? 64 : 128;
}

constexpr uint32_t ADAPT_CTAS_PER_SM = 4, ADAPT_MAX_PIECES = 16, ADAPT_LONG_CTAS_PER_SM = 3;
constexpr unsigned ADAPT_LONG_M = 512;
constexpr uint32_t ADAPT_SUM_BYTES = 32768;

// Whether the rows go 64 to a CTA. Measured, K = N = 4096, 16 rows a CTA against 64: 256 rows of rank
// 16, 32, 64 12.6 / 18.6, 17.8 / 21.2, 25 / 28 us; 512 rows 17.5 / 18.4, 24 / 21, 37 / 32; 1000 rows
// 31 / 29, 40 / 31, 51 / 38. With 8 adapters mixed over the rows, 256 rows 32 / 35, 43 / 42, 58 / 56;
// 512 rows 54 / 45, 74 / 55, 102 / 90.
bool adapters_long(const charsiu_gpu_adapters *s, unsigned n, unsigned m)
{
	for (unsigned i = 0; i < n; i++)
		if (s[i].max_rank % 8)          // (weights are copied by 16 bytes)
			return false;
	return m >= ADAPT_LONG_M && adapters_ranks(s, n) <= 64;
}

uint64_t adapters_tiles(bool lng, unsigned m)
{
	const uint64_t rows = lng ? ADAPT_LONG_ROWS : ADAPT_ROWS;
	return (m + rows - 1) / rows;
}

// CTAs that fill the GPU
uint64_t adapters_aim(charsiu_gpu *g, bool lng)
{
	return (uint64_t)(lng ? ADAPT_LONG_CTAS_PER_SM : ADAPT_CTAS_PER_SM) * layer_sms(g);
}

// columns a CTA of the last launch: as wide as still fills the GPU
uint32_t adapters_cols(charsiu_gpu *g, const charsiu_gpu_adapters *s, unsigned n, unsigned m)
{
	const bool lng = adapters_long(s, n, m);
	const uint64_t tiles = adapters_tiles(lng, m), aim = adapters_aim(g, lng);
	uint64_t columns = 0;
	for (unsigned i = 0; i < n; i++)
		columns += s[i].n;
	if (lng) {
		// (as many as are on it at once: twice as many, of half the columns, take 2000 rows of
		// rank 64 from 45 to 48 us, 1000 of mixed adapters from 113 to 128)
		const uint64_t cols = (tiles * columns / aim + 63) / 64 * 64;
		return cols < 64 ? 64 : cols > 1024 ? 1024 : (uint32_t)cols;
	}
	uint32_t cols = 256;
	while (cols > 32 && tiles * columns / cols < aim)
		cols /= 2;
	return cols;
}

// "" or why a call of m rows would be refused for its size
const char *adapters_size_fault(charsiu_gpu *g, const charsiu_gpu_adapters *s, unsigned n, unsigned m)
{
	if (m > (1u << 24))
		return "adapters: more rows than a call takes";
	const uint32_t cols = adapters_cols(g, s, n, m);
	uint64_t blocks = 0;
	for (unsigned i = 0; i < n; i++)
		blocks += ((uint64_t)s[i].n + cols - 1) / cols;
	return blocks > 65535 ? "adapters: more columns than a call takes" : "";
}

// pieces of K: enough CTAs to fill the GPU, at least one 32-block a warp
uint32_t adapters_pieces(charsiu_gpu *g, const charsiu_gpu_adapters *s, unsigned n, unsigned m)
{
	const bool lng = adapters_long(s, n, m);
	const uint64_t tiles = n * adapters_tiles(lng, m);
	uint64_t want = adapters_aim(g, lng) / (tiles ? tiles : 1);
	const uint32_t most = (s->k / 32 + ADAPT_WARPS - 1) / ADAPT_WARPS;
	want = want < most ? want : most;
	want = want < ADAPT_MAX_PIECES ? want : ADAPT_MAX_PIECES;
	return want < 1 ? 1 : (uint32_t)want;
}

// scratch for m rows, and for any fewer: pieces * m is at most the CTAs aimed at and a
// tile's more, in rows, and at most the most pieces a row
size_t adapters_bytes(charsiu_gpu *g, const charsiu_gpu_adapters *s, unsigned n, unsigned m)
{
	const size_t rows = ((size_t)m + ADAPT_LONG_ROWS - 1) / ADAPT_LONG_ROWS * ADAPT_LONG_ROWS;
	const size_t a = ADAPT_MAX_PIECES * rows * n;
	const size_t b = (size_t)ADAPT_LONG_CTAS_PER_SM * layer_sms(g) * ADAPT_LONG_ROWS + n * rows;
	return (a < b ? a : b) * adapters_ranks(s, n) * sizeof(float);
}

template <typename T, int RT>
int adapters(charsiu_gpu *g, AdaptArgs &a, bool lng, void *stream)
{
	if constexpr (RT <= 64) {
		if (lng) {
			const unsigned tiles = (a.m + ADAPT_LONG_ROWS - 1) / ADAPT_LONG_ROWS;
			const uint32_t each = a.m * (RT / 4);
			constexpr size_t a_smem = AdaptLong<RT>::A_SMEM, b_smem = AdaptLong<RT>::B_SMEM;
			static std::atomic<uint64_t> a_done, b_done;
			return allow_smem(g, adapt_shrink_long_kernel<T, RT>, a_smem, a_done) &&
					       allow_smem(g, adapt_expand_long_kernel<T, RT>, b_smem, b_done) &&
					       launch(g, stream, adapt_shrink_long_kernel<T, RT>,
						      dim3(tiles, a.pieces, a.n_sets), ADAPT_WARPS * 32, a_smem, a) &&
					       (a.pieces == 1 ||
						launch(g, stream, adapt_sum_kernel, dim3((each + 255) / 256, a.n_sets), 256, 0,
						       (float4 *)a.t, a.pieces, each)) &&
					       launch(g, stream, adapt_expand_long_kernel<T, RT>, dim3(tiles, a.blocks),
						      ADAPT_WARPS * 32, b_smem, a)
				       ? 0
				       : -1;
		}
	}
	const unsigned tiles = (a.m + ADAPT_ROWS - 1) / ADAPT_ROWS;
	// Every CTA of the columns adds the pieces of its rows up, or a launch before them does, where that
	// is much to read. Measured, K = N = 4096, 16 pieces, in the CTAs against by a launch: 16
	// rows of rank 16 (16 KB a CTA) 10.8 against 12.6 us, of rank 32 13.0 / 13.0, 64 20 / 16, 128
	// 33 / 23; 128 rows 11.4 / 12.6, 18 / 16, 31 / 22, 89 / 48; 4 rows of rank 32 8.0 / 10.3,
	// 128 17.4 / 17.2.
	const bool sum = a.pieces > 1 && (a.m < ADAPT_ROWS ? a.m : ADAPT_ROWS) * RT * sizeof(float) * a.pieces >=
						 ADAPT_SUM_BYTES;
	const uint32_t each = a.m * (RT / 4);
	a.left = sum ? 1 : a.pieces;
	return launch(g, stream, adapt_shrink_kernel<T, RT>, dim3(tiles, a.pieces * a.parts, a.n_sets),
		      ADAPT_WARPS * 32, 0, a) &&
			       (!sum || launch(g, stream, adapt_sum_kernel, dim3((each + 255) / 256, a.n_sets), 256, 0,
					       (float4 *)a.t, a.pieces, each)) &&
			       launch(g, stream, adapt_expand_kernel<T, RT>, dim3(tiles, a.blocks),
				      ADAPT_WARPS * 32, 0, a)
		       ? 0
		       : -1;
}

template <typename T>
int adapters_of(charsiu_gpu *g, AdaptArgs &a, uint32_t ranks, bool lng, void *stream)
{
	switch (ranks) {
	case 8: return adapters<T, 8>(g, a, lng, stream);
	case 16: return adapters<T, 16>(g, a, lng, stream);
	case 32: return adapters<T, 32>(g, a, lng, stream);
	case 64: return adapters<T, 64>(g, a, lng, stream);
	default: return adapters<T, 128>(g, a, lng, stream);
	}
}

} // namespace

extern "C" {

int charsiu_gpu_norm_quantise_dev(struct charsiu_gpu *g, const float *x, const float *add,
				  const float *w, unsigned m, unsigned k, float eps, float *x_out,
				  int8_t *q, float *d, void *stream)
{
	if (!g || layer_dead(g))
		return -1;
	if (!x || !w || !q || !d)
		return refuse(g, "norm_quantise lacks an array");
	if (!k || k % 32 || k > NORM_ROWS_MAX_K)
		return refuse(g, "norm_quantise takes rows of a multiple of 32 up to 8192");
	if (misaligned(x, 16) || misaligned(add, 16) || misaligned(w, 16) || misaligned(x_out, 16) ||
	    misaligned(q, 16) || misaligned(d, 4))
		return refuse(g, "norm_quantise: an array is misaligned");
	if (m > 0x7fffffffu)
		return refuse(g, "norm_quantise: more rows than a call takes");
	if (!m)
		return 0;
	OnDevice on(g);
	// A CTA a row where the rows are few and long: one row of 2048 / 4096 / 8192 takes it
	// 8.5 / 12.6 / 16.7 us and the chains 10.6 / 18.7 / 35; at 296 rows of 4096 it is
	// 33 us against 20. The chains: as few rows a CTA (three of them a multiprocessor) as
	// hold all rows at once: 2048 rows of 4096 take 41 us by 4, 37 by 8, 41 by 16.
	const uint64_t sms = layer_sms(g), cta = 3;
	if (k >= 2048 && 4 * (uint64_t)m <= 3 * sms) {
		static std::atomic<uint64_t> smem_done;
		if (!allow_smem(g, norm_rows_kernel, norm_rows_smem(NORM_ROWS_MAX_K), smem_done))
			return -1;
		return launch(g, stream, norm_rows_kernel, dim3(m), NORM_ROWS_THREADS, norm_rows_smem(k), x, add, w,
			      (uint32_t)k, eps, x_out, q, d)
			       ? 0
			       : -1;
	}
	auto chains = [&](auto kernel, uint32_t rows, std::atomic<uint64_t> &smem_done) {
		return allow_smem(g, kernel, norm_chain_smem(rows), smem_done) &&
				       launch(g, stream, kernel, dim3((unsigned)(((uint64_t)m + rows - 1) / rows)),
					      NORM_CHAIN_THREADS, norm_chain_smem(rows), x, add, w, (uint32_t)m,
					      (uint32_t)k, eps, x_out, q, d, layer_kernel_error(g))
			       ? 0
			       : -1;
	};
	static std::atomic<uint64_t> done4, done8, done16;
	return m <= 4 * cta * sms   ? chains(norm_chain_kernel<1>, 4, done4)
	       : m <= 8 * cta * sms ? chains(norm_chain_kernel<2>, 8, done8)
				    : chains(norm_chain_kernel<4>, 16, done16);
}

size_t charsiu_gpu_pages_work(const struct charsiu_gpu_pages *p)
{
	return *pages_fault(p) ? 0 : pages_work_words(p->n_pages) * sizeof(int32_t);
}

int charsiu_gpu_pages_grow_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
			       const int32_t *slots, unsigned n, unsigned add, void *stream)
{
	if (slots_check(g, p, slots, n))
		return -1;
	if (add > 0x7fffffffu)
		return refuse(g, "a slot cannot grow that far");
	if (!n || !add)
		return 0;
	OnDevice on(g);
	return launch(g, stream, pages_grow_kernel, dim3(1), PAGES_PLAN_THREADS, 0, *p, slots,
		      (uint32_t)n, (uint32_t)add)
		       ? 0
		       : -1;
}

int charsiu_gpu_pages_fork_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
			       const int32_t *from, const int32_t *to, unsigned n, void *stream)
{
	if (slots_check(g, p, from, n) || slots_check(g, p, to, n))
		return -1;
	if (!n)
		return 0;
	OnDevice on(g);
	return launch(g, stream, pages_fork_plan_kernel, dim3(1), PAGES_PLAN_THREADS, 0, *p, from, to,
		      (uint32_t)n) &&
			       launch(g, stream, pages_fork_kernel, dim3(n, 2 * p->n_layer), 256, 0, *p, to)
		       ? 0
		       : -1;
}

int charsiu_gpu_pages_free_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
			       const int32_t *slots, unsigned n, void *stream)
{
	if (slots_check(g, p, slots, n))
		return -1;
	if (!n)
		return 0;
	OnDevice on(g);
	return launch(g, stream, pages_free_kernel, dim3(n), 128, 0, *p, slots) ? 0 : -1;
}

int charsiu_gpu_pages_compact_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
				  int32_t *live, void *stream)
{
	if (pages_check(g, p, true))
		return -1;
	if (misaligned(live, 4))
		return refuse(g, "an array is misaligned");
	OnDevice on(g);
	return launch(g, stream, pages_compact_plan_kernel, dim3(1), PAGES_PLAN_THREADS, 0, *p, live) &&
			       launch(g, stream, pages_compact_kernel, dim3(8 * layer_sms(g)), 256, 0, *p)
		       ? 0
		       : -1;
}

int charsiu_gpu_pages_append_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
				 unsigned layer, const int32_t *slots, unsigned n, unsigned t,
				 unsigned n_head, const float *q, const float *k, const float *v,
				 const float *rope_cs, unsigned n_ctx, void *q_out, void *stream)
{
	if (pages_check(g, p, false))
		return -1;
	if (layer >= p->n_layer)
		return refuse(g, "the cache has no such layer");
	if (!n || !t)
		return 0;
	if (!slots || !q || !k || !v || !rope_cs || !q_out)
		return refuse(g, "append lacks an array");
	if (!n_head || n_head % p->n_head_kv)
		return refuse(g, "n_head is no multiple of n_head_kv");
	if (misaligned(q, 16) || misaligned(k, 16) || misaligned(v, 16) || misaligned(rope_cs, 16) ||
	    misaligned(q_out, 16) || misaligned(slots, 4))
		return refuse(g, "append: an array is misaligned");
	if ((uint64_t)n * t > 0x7fffffffull || n_head > 1u << 20)
		return refuse(g, "append: more rows than a call takes");
	OnDevice on(g);
	return p->type == TYPE_F16
		       ? append<__half>(g, p, layer, slots, n, t, n_head, q, k, v, rope_cs, n_ctx, q_out, stream)
		       : append<__nv_bfloat16>(g, p, layer, slots, n, t, n_head, q, k, v, rope_cs, n_ctx,
					       q_out, stream);
}

size_t charsiu_gpu_attention_work(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
				  const struct charsiu_gpu_attention *a)
{
	if (!g || *attention_fault(p, a))
		return 0;
	return attention_bytes(g, p, a);
}

int charsiu_gpu_attention_dev(struct charsiu_gpu *g, const struct charsiu_gpu_pages *p,
			      unsigned layer, const struct charsiu_gpu_attention *b, const void *q,
			      void *out, void *stream)
{
	if (pages_check(g, p, false))
		return -1;
	const char *why = attention_fault(p, b);
	if (*why)
		return refuse(g, why);
	if (layer >= p->n_layer)
		return refuse(g, "the cache has no such layer");
	if (!b->n_seq)
		return 0;
	if (!q || !out || misaligned(q, 16) || misaligned(out, 16) || misaligned(b->slots, 4) ||
	    misaligned(b->group, 4) || misaligned(b->shared, 4))
		return refuse(g, "attention: an array is missing or misaligned");
	AttnArgs a = {};
	const bool tc = attention_plan(g, p, b, &a);
	if (!b->work || misaligned(b->work, 16) || b->work_bytes < attention_bytes(g, p, b))
		return refuse(g, "attention: the work array is missing, misaligned or too small");
	a.p = *p;
	a.slots = b->slots;
	a.group = b->group;
	a.shared = b->shared;
	a.q = q;
	a.out = out;
	a.part_o = (float *)b->work;
	a.part_w = a.part_o + (size_t)b->n_seq * b->n_tok * b->n_head * (a.pre_splits + a.own_splits) *
				      p->head_dim;
	a.layer = layer;
	a.n_seq = b->n_seq;
	a.n_tok = b->n_tok;
	a.n_head = b->n_head;
	a.n_group = b->n_group;
	a.out_type = b->out_type;
	a.scale = b->scale * 1.4426950408889634f;
	a.err = layer_kernel_error(g);
	OnDevice on(g);
	if (p->type == TYPE_F16)
		return p->head_dim == 64 ? attention<__half, 64>(g, a, tc, stream)
					 : attention<__half, 128>(g, a, tc, stream);
	return p->head_dim == 64 ? attention<__nv_bfloat16, 64>(g, a, tc, stream)
				 : attention<__nv_bfloat16, 128>(g, a, tc, stream);
}

size_t charsiu_gpu_adapters_work(struct charsiu_gpu *g, const struct charsiu_gpu_adapters *sets,
				 unsigned n, unsigned m)
{
	return !g || *adapters_fault(sets, n) || *adapters_size_fault(g, sets, n, m) ? 0 : adapters_bytes(g, sets, n, m);
}

int charsiu_gpu_adapters_dev(struct charsiu_gpu *g, const struct charsiu_gpu_adapters *sets,
			     unsigned n, unsigned m, const int8_t *q, const float *d,
			     const int32_t *which, const float *const *bases, float *const *ys,
			     void *work, size_t work_bytes, void *stream)
{
	if (!g || layer_dead(g))
		return -1;
	const char *why = adapters_fault(sets, n);
	if (*why)
		return refuse(g, why);
	if (!m)
		return 0;
	if (!q || !d || !which || !ys || misaligned(q, 16) || misaligned(d, 4) || misaligned(which, 4))
		return refuse(g, "adapters: an array is missing or misaligned");
	if (*(why = adapters_size_fault(g, sets, n, m)))
		return refuse(g, why);
	if (!work || misaligned(work, 16) || work_bytes < adapters_bytes(g, sets, n, m))
		return refuse(g, "adapters: the work array is missing, misaligned or too small");
	AdaptArgs a = {};
	uint32_t slots = 0;
	for (unsigned i = 0; i < n; i++) {
		AdaptSet &s = a.s[i];
		s.a = sets[i].a;
		s.b = sets[i].b;
		s.rank = sets[i].rank;
		s.scale = sets[i].scale;
		s.y = ys[i];
		s.base = bases ? bases[i] : ys[i];
		if (!s.y || !s.base || misaligned(s.y, 4) || misaligned(s.base, 4))
			return refuse(g, "adapters: an output is missing or misaligned");
		for (unsigned j = 0; j < i; j++)
			if (s.y == a.s[j].y || s.base == a.s[j].y || s.y == a.s[j].base)
				return refuse(g, "adapters: two sets share an output, or one's base is another's");
		s.n = sets[i].n;
		s.slots = sets[i].slots;
		s.max_rank = sets[i].max_rank;
		slots = slots > s.slots ? slots : s.slots;
	}
	const bool lng = adapters_long(sets, n, m);
	const uint64_t tiles = adapters_tiles(lng, m), aim = adapters_aim(g, lng);
	a.cols = adapters_cols(g, sets, n, m);
	uint32_t blocks = 0;
	for (unsigned i = 0; i < n; i++) {
		blocks += (a.s[i].n + a.cols - 1) / a.cols;
		a.s[i].block_end = blocks;
	}
	a.q = q;
	a.d = d;
	a.which = which;
	a.t = (float *)work;
	a.n_sets = n;
	a.m = m;
	a.k = sets[0].k;
	a.pieces = adapters_pieces(g, sets, n, m);
	// few tiles: their distinct adapters over several CTAs, as far as the GPU has room
	uint64_t parts = aim / (tiles * n * a.pieces);
	parts = parts < ADAPT_ROWS ? parts : ADAPT_ROWS;
	parts = parts < slots ? parts : slots;
	parts = parts < m ? parts : m;
	a.parts = parts < 1 ? 1 : (uint32_t)parts;
	a.blocks = blocks;
	OnDevice on(g);
	const uint32_t ranks = adapters_ranks(sets, n);
	return sets[0].type == TYPE_F16 ? adapters_of<__half>(g, a, ranks, lng, stream)
					: adapters_of<__nv_bfloat16>(g, a, ranks, lng, stream);
}

} // extern "C"
