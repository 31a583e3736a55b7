/* SPDX-License-Identifier: GPL-2.0-or-later */
#ifndef CHARSIU_GPU_H
#define CHARSIU_GPU_H

/*
 * The GPU device layer: a drop-in for charsiu's NPU device layer on NVIDIA
 * B200 (sm_100a).
 *
 * Every call below is the GPU twin of one charsiu_npu_* call (declared in the
 * reference at include/charsiu_llm.h:186-200, implemented in src/npudev.c),
 * with the same conventions:
 *
 *   - NULL / -1 on failure, never abort. A failed call leaves the caller's
 *     output undefined and the caller recomputes on the CPU, as llama.c does
 *     for the NPU (src/llama.c:269-282).
 *   - Three slow or failed calls in a row retire the layer; every call after
 *     that returns -1 (src/npudev.c:560-602). The first refusal is printed once
 *     (src/npudev.c:124-138) and the report says if nothing ran on the GPU.
 *   - Not re-entrant: one decode thread calls it, before any pool fan-out
 *     (src/llama.c:261-282).
 *
 * The NPU layer takes the NPU's own per-channel int8 format; this layer takes
 * the GGUF tensor itself and computes charsiu's GGML block arithmetic
 * (src/gguf.c:1061-1107, 1149-1171) exactly: q8_0 or q4_0 weights against the
 * q8_0 activation of charsiu_act_set, int32 block dots, and the fp32 sum of
 * (d_w * d_a) * dot in block order, so y is bit-identical to gguf_matvec.
 * Weights are repacked once, at add time, into a coalesced device layout.
 *
 * The struct types are charsiu's own (include/charsiu_llm.h:51-59, 100-119;
 * include/charsiu.h:113-119, 194-225); this header only names them. Callers
 * without those headers use the flat forms (plain pointers and sizes).
 */

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define CHARSIU_GPU_API __attribute__((visibility("default")))
#else
#define CHARSIU_GPU_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

struct gguf_tensor;
struct charsiu_act;
struct charsiu_job;
struct charsiu_gpu;

/* ---- lifetime ------------------------------------------------------------ */

/* charsiu_npu_open (include/charsiu_llm.h:188-189, src/npudev.c:140-233).
 * Device 0, the whole of every tensor. max_k: a multiple of 32, at most
 * 14336. NULL: no usable GPU; stay on the CPU. */
CHARSIU_GPU_API struct charsiu_gpu *charsiu_gpu_open(unsigned max_k, unsigned max_n,
				     unsigned max_tensors);

/* The same on `device`, holding only column slab `rank` of `world` of every
 * tensor added: rows [rank*N/world, (rank+1)*N/world) rounded to whole
 * 8-row groups. No counterpart in the reference (one board, one NPU); it is
 * the N-split the vendor runtime uses across NPU cores (docs/vendor-dispatch.md:43-58). */
CHARSIU_GPU_API struct charsiu_gpu *charsiu_gpu_open_ex(unsigned max_k, unsigned max_n,
					unsigned max_tensors, int device,
					unsigned rank, unsigned world);

/* charsiu_npu_close (include/charsiu_llm.h:190). NULL-safe. */
CHARSIU_GPU_API void charsiu_gpu_close(struct charsiu_gpu *g);

/* ---- weights ------------------------------------------------------------- */

/* charsiu_npu_add (include/charsiu_llm.h:191, src/npudev.c:389-461), for the
 * GGUF tensor: q8_0 or q4_0 with ne[0] = K a multiple of 32, or q6_K (the
 * head of a llama.cpp q4_0 file) with K a multiple of 256; ne[1] = N. The host
 * tensor stays the caller's. Returns an id >= 0, or -1 (tensor stays on the
 * CPU). Adding the same tensor again returns its existing id. */
CHARSIU_GPU_API int charsiu_gpu_add(struct charsiu_gpu *g, const struct gguf_tensor *w);

/* Flat form of charsiu_gpu_add: `blocks` is N rows of GGML blocks (34 bytes
 * a 32-weight q8_0 block, 18 q4_0, 210 a 256-weight q6_K super-block), row
 * major, as in a GGUF file. */
CHARSIU_GPU_API int charsiu_gpu_add_blocks(struct charsiu_gpu *g, uint32_t type, uint64_t k,
			   uint64_t n, const void *blocks, const char *name);

/* Rows this GPU holds of tensor `id`: [*row0, *row0 + *nrows). */
CHARSIU_GPU_API int charsiu_gpu_rows(const struct charsiu_gpu *g, int id, uint64_t *row0,
		     uint64_t *nrows);

/* ---- the matvec ---------------------------------------------------------- */

/* charsiu_npu_matvec (include/charsiu_llm.h:192-193, src/npudev.c:463-607):
 * y = W x from a->q and a->d (a->quantised must be set, a->n = K). y holds
 * this GPU's rows of the output (all N on an unsharded layer). */
CHARSIU_GPU_API int charsiu_gpu_matvec(struct charsiu_gpu *g, int id,
		       const struct charsiu_act *a, float *y);

/* charsiu_npu_matvec_group (include/charsiu_llm.h:195-196,
 * src/npudev.c:621-716): up to 8 projections of one activation, one launch
 * and one fence. -1: the caller falls back to single calls. */
CHARSIU_GPU_API int charsiu_gpu_matvec_group(struct charsiu_gpu *g, const int *ids, unsigned n,
			     const struct charsiu_act *a, float **ys);

/* Flat form of the group call: q is K int8 (K/32 blocks), d K/32 fp32. */
CHARSIU_GPU_API int charsiu_gpu_matvec_q(struct charsiu_gpu *g, const int *ids, unsigned n,
			 const int8_t *q, const float *d, unsigned k,
			 float **ys);

/* Batched: m activations q[m][K], d[m][K/32] against tensor id; y[m][rows].
 * Each y[i] is bit-identical to the single matvec of activation i. No
 * counterpart in the reference, which decodes one token at a time. */
CHARSIU_GPU_API int charsiu_gpu_matvec_batch(struct charsiu_gpu *g, int id, unsigned m,
			     const int8_t *q, const float *d, unsigned k,
			     float *y);

/* ---- the int8 matmul with the NPU's output stage ------------------------- */

/* What charsiu_emit_job + charsiu_submit compute for an int8 job
 * (include/charsiu.h:194-235; arithmetic of tools/charsiu_matmul.c:41-81 and
 * the output stage of src/job.c:137-177): a u8 [m][k], w u8 [n][k] (int8
 * weights, job->mm.wdtype CHARSIU_INT8), bias i32 [n]; out i8 [m][n] row
 * major, out = clamp(max(requant, 0) + offset, -128, 127). Byte-exact
 * against cpu_reference. */
CHARSIU_GPU_API int charsiu_gpu_matmul_i8(struct charsiu_gpu *g, const struct charsiu_job *job,
			  const uint8_t *a, const uint8_t *w,
			  const int32_t *bias, int8_t *out);

/* Flat form of charsiu_gpu_matmul_i8. */
CHARSIU_GPU_API int charsiu_gpu_matmul_i8_flat(struct charsiu_gpu *g, unsigned m, unsigned k,
			       unsigned n, const uint8_t *a, const uint8_t *w,
			       const int32_t *bias, float in_scale,
			       float wt_scale, float out_scale, int in_zp,
			       int wt_zp, int out_zp, int8_t *out);

/* ---- device-resident forms ------------------------------------------------ */
/*
 * For callers that keep the activation in HBM (a decode loop on the device).
 * All pointers are device pointers; the work is queued on `stream` (a
 * cudaStream_t, NULL for the layer's own) with no host synchronisation, so a
 * caller may capture it in a CUDA graph. Return 0 when queued.
 */
CHARSIU_GPU_API int charsiu_gpu_matvec_dev(struct charsiu_gpu *g, const int *ids, unsigned n,
			   const int8_t *q, const float *d, float *const *ys,
			   void *stream);
CHARSIU_GPU_API int charsiu_gpu_matvec_batch_dev(struct charsiu_gpu *g, int id, unsigned m,
				 const int8_t *q, const float *d, float *y,
				 void *stream);
/* The batched twin of charsiu_gpu_matvec_group (include/charsiu_llm.h:194-196
 * for one activation): m activations (q [m][K] int8, d [m][K/32] fp32) against
 * n <= 8 tensors of the same K, ys[i] = [m][rows of ids[i]]. From 9
 * activations, q8_0 tensors share one packing of the activations and one
 * tensor-core launch; below, the tensors of each quant type share one CUDA-core
 * launch a chunk of 8, 4 or 2 activations. */
CHARSIU_GPU_API int charsiu_gpu_matvec_batch_group_dev(struct charsiu_gpu *g, const int *ids,
						       unsigned n, unsigned m, const int8_t *q,
						       const float *d, float *const *ys,
						       void *stream);
/* ---- the matvec fused with its all-gather ------------------------------------ */
/*
 * For a layer opened with charsiu_gpu_open_ex(..., rank, world) in each of
 * `world` processes, one a GPU, that need every rank to hold the whole y (the
 * column-split decode). No counterpart in the reference (charsiu has one
 * device).
 *
 * Buffers the peers write are allocated here (charsiu_gpu_ipc_alloc: plain
 * device memory, zeroed) and shared with a 64-byte handle
 * (charsiu_gpu_ipc_handle; exchange the bytes between processes, then
 * charsiu_gpu_ipc_open gives this process's pointer to a peer's buffer;
 * charsiu_gpu_ipc_free releases either kind).
 *
 * charsiu_gpu_matvec_gather_dev runs the matvec of this rank's slab and
 * stores each y into every rank's full output full_ys[r * n + i] (tensor
 * ids[i], rank r: the whole N floats), then adds the groups it finished to
 * word signal_idx of every rank's sync array syncs[r] (uint32). With
 * wait_mult > 0 it first waits, on this GPU, until its own word wait_idx
 * reaches (epoch + wait_adj) * wait_mult, epoch being word 0, which
 * charsiu_gpu_gather_epoch_dev adds 1 to (call it at each token's start). The
 * wait gives up after one second (the layer then retires). The launches run
 * without programmatic dependence. 0 when queued on `stream`.
 */
CHARSIU_GPU_API void *charsiu_gpu_ipc_alloc(struct charsiu_gpu *g, size_t bytes);
CHARSIU_GPU_API int charsiu_gpu_ipc_handle(struct charsiu_gpu *g, void *ptr,
					   unsigned char *handle);
CHARSIU_GPU_API void *charsiu_gpu_ipc_open(struct charsiu_gpu *g, const unsigned char *handle);
CHARSIU_GPU_API void charsiu_gpu_ipc_free(struct charsiu_gpu *g, void *ptr, int opened);
/* Copy `bytes` of device memory (this GPU's, or a peer's opened above) to the
 * host; waits for it. 0 on success. */
CHARSIU_GPU_API int charsiu_gpu_read_device(struct charsiu_gpu *g, const void *dev_ptr,
					    void *host, size_t bytes);
CHARSIU_GPU_API int charsiu_gpu_gather_epoch_dev(struct charsiu_gpu *g, uint32_t *sync_local,
						 void *stream);
/* The first nonzero code a kernel of the _dev forms wrote since the last
 * call (a bounded wait that gave up), then clears it; a nonzero code retires
 * the layer, as a host call's would. 0: none. */
CHARSIU_GPU_API int charsiu_gpu_kernel_error(struct charsiu_gpu *g);
CHARSIU_GPU_API int charsiu_gpu_matvec_gather_dev(struct charsiu_gpu *g, const int *ids,
						  unsigned n, const int8_t *q, const float *d,
						  float *const *full_ys, uint32_t *const *syncs,
						  unsigned signal_idx, unsigned wait_idx,
						  unsigned wait_mult, int wait_adj, void *stream);
/* The batched form of charsiu_gpu_matvec_gather_dev: m activations (q [m][K]
 * int8, d [m][K/32] fp32, m at least CHARSIU_GPU_QMM_MIN_M, so on the tensor
 * cores) against n <= 8 q8_0 tensors of one K. Each rank's rows go straight
 * into every rank's full output full_ys[r * n + i] ([m][N] floats) from the
 * tensor-core epilogue; the waits and the arrival words are as above, except
 * that each rank adds 1 a launch (so wait_mult is the world size). No
 * counterpart in the reference. */
CHARSIU_GPU_API int charsiu_gpu_matvec_batch_gather_dev(struct charsiu_gpu *g, const int *ids,
							unsigned n, unsigned m, const int8_t *q,
							const float *d, float *const *full_ys,
							uint32_t *const *syncs, unsigned signal_idx,
							unsigned wait_idx, unsigned wait_mult,
							int wait_adj, void *stream);

/* The batched matvec of charsiu_gpu_matvec_batch_dev, for callers that
 * cannot allocate GPU memory while they run -- a server whose own memory
 * pool already owns the GPU's free memory, or a latency-bound loop that must
 * not take cudaMalloc's implicit device synchronisation (the _dev form grows
 * a staging buffer with cudaMalloc on first use). This call allocates
 * nothing: its scratch is a fixed 1 MiB array inside the library, held on
 * every GPU that loads it until exit. q8_0 tensors only; the m activations
 * are always packed into that array first, in tiles of 16 or 32 (the _dev
 * form reads them from q and d by tensor copies where it can), and must fit
 * it (m <= 64 up to
 * K = 14336), else -1 with the reason in charsiu_gpu_error. All calls on a GPU
 * share the array, so two calls running on it at the same time race. A
 * layer's first call looks up the array's device address (on the layer's
 * GPU) and keeps it; make that call before any stream capture. Every m, from
 * 1, runs on the tensor cores here (charsiu_gpu_matvec_batch_dev takes m
 * below CHARSIU_GPU_QMM_MIN_M to the CUDA cores); both are gguf_matvec bit
 * for bit, so the results are the same. No counterpart in the reference. */
CHARSIU_GPU_API int charsiu_gpu_matvec_batch_noalloc(struct charsiu_gpu *g, int id, unsigned m,
						     const int8_t *q, const float *d, float *y,
						     void *stream);
/* charsiu_act_set (src/gguf.c:829-882) on the device, bit-exact: x fp32
 * [m][k] -> q int8 [m][k rounded up to 32], d fp32 [m][k/32]. */
CHARSIU_GPU_API int charsiu_gpu_act_quantise_dev(struct charsiu_gpu *g, const float *x,
				 unsigned m, unsigned k, int8_t *q, float *d,
				 void *stream);

/* gguf_row_f32 (src/gguf.c:1217-1256) of one row of tensor id -- the
 * embedding lookup -- from the layer's copy, bit-exact: out fp32 [K]. The row
 * index is read from device memory (*row), so a captured graph can take a new
 * token each replay; an index outside the tensor writes a nonzero code that
 * charsiu_gpu_kernel_error returns. The whole tensor must be on this GPU
 * (world 1). */
CHARSIU_GPU_API int charsiu_gpu_row_dev(struct charsiu_gpu *g, int id, const int32_t *row,
					float *out, void *stream);

/* ---- the decode step on the device ------------------------------------------ */
/*
 * llama_forward (src/llama.c:743-856) with every step on the GPU: the
 * embedding row, rmsnorm, the activation quantiser, the projections (this
 * layer's matvecs), RoPE and the KV cache, attention, SiLU, the residual adds,
 * the head and llama_argmax, replayed as one CUDA graph a token. The logits
 * are the reference's bit for bit: every sum keeps the reference's order and
 * rounding, and expf is a table of the host C library's own expf over every
 * float where it is neither 1, 0 nor inf (2.2 GB of device memory, built once
 * a process and GPU, checked against expf for every float it leaves out).
 * No counterpart in the reference, which runs these steps on the CPU.
 *
 * The model: projection ids (tensors added to g) per layer in the order q, k,
 * v, o, gate, up, down; the embedding and head ids (the same tensor when the
 * head is tied); host fp32 norm weights, copied at creation; rope_cs the
 * (cos, sin) pair i of every position, [n_ctx][head_dim], as
 * src/llama.c:364-383 computes them. Requires n_head * head_dim = n_embd,
 * head_dim a multiple of 32 and at most 256, n_embd and n_ff multiples of 32, n_embd at most
 * 8192, and a layer opened with world 1.
 */
struct charsiu_gpu_decoder;

struct charsiu_gpu_decoder_desc {
	uint32_t n_embd, n_layer, n_head, n_head_kv, n_ff, head_dim, n_vocab, n_ctx;
	float rms_eps;
	int embd_id, head_id;
	const int *proj_ids;               /* [n_layer][7] */
	const float *const *attn_norm;     /* [n_layer] -> n_embd floats */
	const float *const *ffn_norm;      /* [n_layer] -> n_embd floats */
	const float *out_norm;             /* n_embd floats */
	const float *rope_cs;              /* [n_ctx][head_dim] */
};

CHARSIU_GPU_API struct charsiu_gpu_decoder *charsiu_gpu_decoder_new(
	struct charsiu_gpu *g, const struct charsiu_gpu_decoder_desc *desc);
/* The same step in charsiu's NPU number format (CHARSIU_NPU_QUANT,
 * src/llama.c:110-312): proj_ids and head_id are tensors added to npu (the
 * charsiu_npu_* layer of include/charsiu_npu.h, on g's GPU), each fed the
 * single-scale activation of charsiu_act_set (src/gguf.c:883-910) of the
 * rmsnorm, attention and SiLU outputs, computed on the device; embd_id is
 * still a tensor of g. */
struct charsiu_npu;
CHARSIU_GPU_API struct charsiu_gpu_decoder *charsiu_gpu_decoder_new_npu(
	struct charsiu_gpu *g, struct charsiu_npu *npu, const struct charsiu_gpu_decoder_desc *desc);
CHARSIU_GPU_API void charsiu_gpu_decoder_free(struct charsiu_gpu_decoder *dec);
/* One token at pos (positions run 0, 1, 2, ... as llama_forward's callers
 * step them): *next gets llama_argmax of its logits; with want_logits the
 * logits are also copied back, readable at charsiu_gpu_decoder_logits until
 * the next step. 0 on success, -1 on failure (charsiu_gpu_error says why). */
CHARSIU_GPU_API int charsiu_gpu_decoder_step(struct charsiu_gpu_decoder *dec, int32_t token,
					     int pos, int want_logits, int32_t *next);
/* The greedy loop of tools/charsiu_run.c:295-317 with the host taken out:
 * n steps from `token` at `pos`, each step's argmax the next step's token at
 * the next position, all queued at once (the argmax never leaves the device
 * between steps); out[i] gets the argmax of step i, so out[0] is what
 * charsiu_gpu_decoder_step would return for (token, pos). pos + n must not
 * pass the context. *device_ms (if given) gets the device time of the n
 * steps, from CUDA events on the decoder's stream. 0 on success, -1 on
 * failure. No counterpart in the reference. */
CHARSIU_GPU_API int charsiu_gpu_decoder_generate(struct charsiu_gpu_decoder *dec, int32_t token,
						 int pos, unsigned n, int32_t *out,
						 float *device_ms);
CHARSIU_GPU_API const float *charsiu_gpu_decoder_logits(const struct charsiu_gpu_decoder *dec);
/* kernels one step launches */
CHARSIU_GPU_API unsigned charsiu_gpu_decoder_launches(const struct charsiu_gpu_decoder *dec);

/* ---- the operators of a batched step ------------------------------------------ */
/*
 * What a server that batches sequences runs between its projections
 * (charsiu_gpu_matvec_batch_group_dev): the norm before them, low-rank adapters
 * beside them, and a paged cache with the attention that reads it. The manner is
 * the device-resident forms': device pointers, work queued on `stream` (NULL for
 * the layer's own), no host synchronisation, no allocation, capturable in a CUDA
 * graph; 0 when queued, -1 with the reason in charsiu_gpu_error. Every buffer,
 * scratch included, is the caller's: calls that may run at the same time (two
 * streams, two captured graphs) need scratch of their own. Arrays that say where
 * to read or write (slots, tables, adapter numbers) are device memory and are
 * checked there: an index out of range reads and writes nothing. A wait inside a
 * kernel that gave up (after a second; none does in a sound run) leaves wrong
 * results and shows in charsiu_gpu_kernel_error only, which a caller asks once a
 * step or so, after synchronising.
 * No counterpart in the reference, which decodes one token at a time.
 */

/* rmsnorm of m rows with the residual's addition, and the q8_0 activation of the
 * result: s = x + add (x alone if add is NULL), q and d what charsiu_act_set
 * gives of rmsnorm(s) with gains w (src/llama.c:316-326, src/gguf.c:829-882).
 * Every row is bit-identical to the decode step's. x, add fp32 [m][k], w [k],
 * q int8 [m][k], d fp32 [m][k/32]; x_out fp32 [m][k] gets s (it may be x or add;
 * NULL: not wanted). k a multiple of 32, at most 8192; x, add, w, x_out and q
 * 16-byte aligned, d 4. m 0 does nothing. */
CHARSIU_GPU_API int charsiu_gpu_norm_quantise_dev(struct charsiu_gpu *g, const float *x,
						  const float *add, const float *w, unsigned m,
						  unsigned k, float eps, float *x_out, int8_t *q,
						  float *d, void *stream);

/* A cache of K and V in pages. All memory is the caller's; pointers are device
 * pointers. Element (layer, page, position, head, i) of K is
 * k[layer * layer_stride + page * page_stride + position * pos_stride + head *
 * head_stride + i] (strides in elements), the same for V: both [page][position]
 * [head] and [page][head][position] orders can be told. Elements of two
 * (layer, page, position, head) must not overlap.
 *
 * A sequence lives in a slot 0..n_seq-1: len[slot] positions, in the pages
 * table[slot * max_pages + j], j < ceil(len / page). ref[page] counts the slots
 * that hold a page; 0 is free. Start with len and ref all 0.
 *
 * A call that lists slots takes them in order; one that cannot be done (a slot out
 * of range or listed before, no room in the table, no free page) is left as it was
 * and counted in the first int32 of `work`, which only the caller clears. Lists of
 * slots are 4-byte aligned. Fresh pages are the free ones of the lowest numbers, so
 * results never depend on timing. */
struct charsiu_gpu_pages {
	void *k, *v;                       /* 16-byte aligned */
	int32_t *table;                    /* [n_seq][max_pages] */
	int32_t *len;                      /* [n_seq] */
	int32_t *ref;                      /* [n_pages] */
	int32_t *work;                     /* charsiu_gpu_pages_work bytes, cleared once */
	uint64_t layer_stride, page_stride, pos_stride, head_stride;   /* multiples of 8 */
	uint32_t type;                     /* GGML's number: 1 fp16, 30 bf16 */
	uint32_t n_layer, n_pages;         /* n_pages at most 2^21 */
	uint32_t page;                     /* positions a page: 16, 32, 64 or 128 */
	uint32_t n_head_kv, head_dim;      /* head_dim 64 or 128 */
	uint32_t n_seq, max_pages;
};
/* bytes of `work`; 0 for a cache that the calls would refuse */
CHARSIU_GPU_API size_t charsiu_gpu_pages_work(const struct charsiu_gpu_pages *p);
/* Slots slots[0..n) grow by `add` positions: len, and the pages for them. Once the
 * free pages run out at one slot, the later ones that need a page are refused too.
 * n at most 1024. */
CHARSIU_GPU_API int charsiu_gpu_pages_grow_dev(struct charsiu_gpu *g,
					       const struct charsiu_gpu_pages *p,
					       const int32_t *slots, unsigned n, unsigned add,
					       void *stream);
/* Slot to[i] becomes a fork of slot from[i], for i < n <= 1024: it shares the full
 * pages and gets a copy, in all layers, of the filled positions of a last page that
 * is not full. to[i] must be empty (len 0). Every source is taken as it was before
 * the call. Refusals for want of pages as above. */
CHARSIU_GPU_API int charsiu_gpu_pages_fork_dev(struct charsiu_gpu *g,
					       const struct charsiu_gpu_pages *p,
					       const int32_t *from, const int32_t *to, unsigned n,
					       void *stream);
/* Slots slots[0..n) become empty; pages that no slot holds any more are free. A
 * slot listed twice, or empty already, is freed once and not counted as refused. */
CHARSIU_GPU_API int charsiu_gpu_pages_free_dev(struct charsiu_gpu *g,
					       const struct charsiu_gpu_pages *p,
					       const int32_t *slots, unsigned n, void *stream);
/* Packs the pages in use into 0..live-1: the live pages from `live` on, in order,
 * go to the free ones below it, in order, in all layers; tables and ref follow.
 * *live (device, may be NULL) gets their number. */
CHARSIU_GPU_API int charsiu_gpu_pages_compact_dev(struct charsiu_gpu *g,
						  const struct charsiu_gpu_pages *p, int32_t *live,
						  void *stream);
/* RoPE and the cache's rows, for one layer: row i * t + j of q, k, v (fp32 [n*t]
 * [heads * head_dim]) is position len - t + j of slot slots[i] (grow the slots
 * first). q and k are rotated by the position's (cos, sin) pairs of rope_cs
 * (fp32 [n_ctx][head_dim], as charsiu_gpu_decoder_desc has them), products and
 * sums in fp32 with the reference's roundings (src/llama.c:364-383), then rounded
 * once to the cache's type: q to q_out [n*t][n_head][head_dim], k and v into the
 * pages. A row whose slot, position (negative, or n_ctx and more) or page is out
 * of range writes nothing. Slots must differ. q, k, v, rope_cs, q_out 16-byte
 * aligned. */
CHARSIU_GPU_API int charsiu_gpu_pages_append_dev(struct charsiu_gpu *g,
						 const struct charsiu_gpu_pages *p, unsigned layer,
						 const int32_t *slots, unsigned n, unsigned t,
						 unsigned n_head, const float *q, const float *k,
						 const float *v, const float *rope_cs,
						 unsigned n_ctx, void *q_out, void *stream);

/* Attention of a batch over the pages of one layer: n_seq sequences (slots; -1
 * pads) of n_tok queries each. Query t of sequence i is row i * n_tok + t of q and
 * stands at position len - n_tok + t of its slot: it sees that position and all
 * before it. Query head h reads KV head h / (n_head / n_head_kv).
 *   out = softmax(scale * q K^T) V
 * with fp32 scores, maxima, sums and accumulators; the weights are rounded to the
 * cache's type for their product with V (whatever out_type is), the result once to
 * out_type. A query that sees nothing (position below 0, an empty or padded slot)
 * gives zeros, and so does one all of whose scores are -inf. What lies behind a
 * query's position never reaches its result, NaN and inf included.
 *
 * Sequences that share their first pages: group g is sequences group[g] to
 * group[g + 1] - 1 (ascending, device), whose slots hold the same first shared[g]
 * pages, as charsiu_gpu_pages_fork_dev leaves them. Those pages are then read once
 * for all of the group's queries. (Only pages that every query of the group sees
 * whole are taken so; the rest is read through each sequence's own table.)
 * n_group 0: group and shared may be NULL. Sequences outside all groups share
 * nothing. n_seq is at most 65536, n_group 4096 and no more than n_seq, n_seq *
 * n_tok * n_head 2^25.
 *
 * max_len: about the longest length; results hold for any, the split of the work
 * over the GPU is chosen by it. */
struct charsiu_gpu_attention {
	const int32_t *slots;              /* [n_seq] */
	const int32_t *group;              /* [n_group + 1] */
	const int32_t *shared;             /* [n_group], pages */
	void *work;                        /* charsiu_gpu_attention_work bytes, 16-byte aligned */
	size_t work_bytes;
	uint32_t n_seq, n_tok, n_head, n_group;
	uint32_t max_len;
	uint32_t out_type;                 /* 0 fp32, or the cache's */
	float scale;
};
/* bytes of `work`, enough for a batch of fewer sequences or groups too; 0 for one
 * that would be refused */
CHARSIU_GPU_API size_t charsiu_gpu_attention_work(struct charsiu_gpu *g,
						  const struct charsiu_gpu_pages *p,
						  const struct charsiu_gpu_attention *a);
/* q [n_seq * n_tok][n_head][head_dim] in the cache's type, out the same shape in
 * out_type; both 16-byte aligned. */
CHARSIU_GPU_API int charsiu_gpu_attention_dev(struct charsiu_gpu *g,
					      const struct charsiu_gpu_pages *p, unsigned layer,
					      const struct charsiu_gpu_attention *a, const void *q,
					      void *out, void *stream);

/* Low-rank adapters of one projection of K inputs and N outputs: adapter s is
 * A = a[s] (the first rank[s] rows of [max_rank][K]) and B = b[s] (the first
 * rank[s] columns of [N][max_rank]), the orders of a GGUF adapter's lora_a and
 * lora_b. What lies behind rank[s] is not used. Device memory, 16-byte aligned. */
struct charsiu_gpu_adapters {
	const void *a;                     /* [slots][max_rank][k] */
	const void *b;                     /* [slots][n][max_rank] */
	const int32_t *rank;               /* [slots], 0..max_rank */
	const float *scale;                /* [slots], alpha / rank */
	uint32_t k, n;                     /* k a multiple of 32 */
	uint32_t slots, max_rank;          /* max_rank 4, or a multiple of 8 up to 128 */
	uint32_t type;                     /* GGML's number: 1 fp16, 30 bf16 */
};
/* bytes of scratch for a call of up to m rows; 0 for one that would be refused */
CHARSIU_GPU_API size_t charsiu_gpu_adapters_work(struct charsiu_gpu *g,
						 const struct charsiu_gpu_adapters *sets, unsigned n,
						 unsigned m);
/* ys[i][r] = bases[i][r] + scale * B (A x_r) of adapter which[r] of sets[i], for the
 * m rows of the q8_0 activation x = q d that the projections read (q int8 [m][K],
 * d fp32 [m][K/32]), against n <= 8 sets of the same K (each with slots and a
 * max_rank of its own; m at most 2^24, the sets' N about 2^24 in all). bases and
 * ys: n device pointers to fp32 [m][N]; bases[i] may be ys[i], and bases NULL means
 * ys: the projections' outputs get the adapters added. No set's output may overlap
 * another's output or base. A row whose `which` is no adapter (-1) is its base.
 * Products are exact, sums and A x fp32. Before its product with B, A x loses less
 * than 2^-21 of a component below 512 rows and where a max_rank is 4 or above 64;
 * else 2^-27 in bf16, and in fp16 what is below 2^-24 of a component or 2^-38 of its
 * row's largest (a component smaller than that adds nothing).
 * work: 16-byte aligned, as q is (d 4). */
CHARSIU_GPU_API int charsiu_gpu_adapters_dev(struct charsiu_gpu *g,
					     const struct charsiu_gpu_adapters *sets, unsigned n,
					     unsigned m, const int8_t *q, const float *d,
					     const int32_t *which, const float *const *bases,
					     float *const *ys, void *work, size_t work_bytes,
					     void *stream);

/* ---- accounting ----------------------------------------------------------- */

/* charsiu_npu_submits (include/charsiu_llm.h:197): calls that ran. */
CHARSIU_GPU_API unsigned long charsiu_gpu_calls(const struct charsiu_gpu *g);
/* kernels this layer has launched */
CHARSIU_GPU_API unsigned long charsiu_gpu_launches(const struct charsiu_gpu *g);
/* charsiu_npu_report (include/charsiu_llm.h:198, src/npudev.c:272-295) */
CHARSIU_GPU_API void charsiu_gpu_report(const struct charsiu_gpu *g);
/* the last failure, in words ("" if none) */
CHARSIU_GPU_API const char *charsiu_gpu_error(const struct charsiu_gpu *g);
/* 1 once the layer has retired itself */
CHARSIU_GPU_API int charsiu_gpu_dead(const struct charsiu_gpu *g);

/* ---- test hooks ------------------------------------------------------------ */

/* The integer block dots of tensor id against q: dots[r][K/32], int32, for
 * this GPU's rows. Bit-exact against dotq_q8_0 / dotq_q4_0's t. */
CHARSIU_GPU_API int charsiu_gpu_block_dots(struct charsiu_gpu *g, int id, const int8_t *q,
			   int32_t *dots);

/* The decode step's ordered sum on the device: the sequential fp32 sum
 * fl(...fl(fl(0 + a[0]) + a[1]) ... + a[n-1]) (rmsnorm's sum of squares,
 * src/llama.c:321-322, and the softmax sum), in both of the step's forms:
 * out[0] by one thread, out[1] by one CTA (the form the rmsnorm uses; exact
 * for non-negative finite terms, and the one-thread sum for any others).
 * a and out (2 floats) are device pointers, n <= 8192. Queued on `stream`. */
CHARSIU_GPU_API int charsiu_gpu_ordered_sum_dev(struct charsiu_gpu *g, const float *a,
						unsigned n, float *out, void *stream);

/* Host-side fault injection (no GPU fault is ever made): from call number
 * `at` on (1-based, counting matvec/group/batch/matmul calls), `count` calls
 * fail as `kind` says: 1 = the launch reports an error, 2 = the call is slow
 * (counts as a watchdog strike), 3 = the device allocation fails (at add).
 * count 0 disarms. */
CHARSIU_GPU_API int charsiu_gpu_inject(struct charsiu_gpu *g, unsigned long at,
		       unsigned long count, int kind);

#ifdef __cplusplus
}
#endif

#endif /* CHARSIU_GPU_H */
