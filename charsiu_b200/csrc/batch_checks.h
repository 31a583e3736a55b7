// SPDX-License-Identifier: GPL-2.0-or-later
// What the operators of a batched step refuse of their descriptions: the structs'
// sizes, types, strides and pointers, by themselves (no layer, no GPU).
#pragma once

#include <cstdint>

#include "charsiu_gpu.h"

namespace cgpu {

constexpr uint32_t TYPE_F32 = 0, TYPE_F16 = 1, TYPE_BF16 = 30;      // GGML's numbers

inline bool misaligned(const void *p, uintptr_t to)
{
	return (uintptr_t)p & (to - 1);
}

constexpr uint32_t PAGES_MAX_ITEMS = 1024;      // slots a call lists, one a thread of its planner

// "" or why the calls would refuse this cache
inline const char *pages_fault(const charsiu_gpu_pages *p)
{
	if (!p || !p->k || !p->v || !p->table || !p->len || !p->ref)
		return "the cache lacks an array";
	if (p->type != TYPE_F16 && p->type != TYPE_BF16)
		return "the cache's type is neither fp16 nor bf16";
	if (p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128)
		return "the cache's pages are not of 16, 32, 64 or 128 positions";
	if (p->head_dim != 64 && p->head_dim != 128)
		return "the cache's head_dim is neither 64 nor 128";
	if (!p->n_layer || !p->n_pages || !p->n_head_kv || !p->n_seq || !p->max_pages)
		return "the cache has a size of 0";
	if (p->n_layer > 32767 || p->n_pages > (1u << 21) || p->n_head_kv > 1024 || p->n_seq > (1u << 20) ||
	    (uint64_t)p->max_pages * p->page > 0x7fffff00ull)
		return "the cache is larger than the calls take";
	if (misaligned(p->k, 16) || misaligned(p->v, 16) || misaligned(p->table, 4) ||
	    misaligned(p->len, 4) || misaligned(p->ref, 4) || misaligned(p->work, 4))
		return "an array of the cache is misaligned";
	if (p->layer_stride % 8 || p->page_stride % 8 || p->pos_stride % 8 || p->head_stride % 8)
		return "a stride of the cache is not a multiple of 8";
	if (p->pos_stride < p->head_dim || p->head_stride < p->head_dim)
		return "the cache's positions or heads overlap";
	return "";
}

// "" or why the calls would refuse this list of slots
inline const char *slots_fault(const int32_t *slots, unsigned n)
{
	if (n && !slots)
		return "no slots";
	if (n > PAGES_MAX_ITEMS)
		return "more slots than a call takes";
	if (n && misaligned(slots, 4))
		return "a list of slots is misaligned";
	return "";
}

// Every CTA looks its group up among all, and a group's shared length among its sequences: with
// these at their most that is 0.1 ms an item (2^25 sequences in as many groups would take hours).
constexpr uint32_t ATTN_MAX_SEQS = 65536, ATTN_MAX_GROUPS = 4096, ATTN_MAX_ROWS = 1u << 25;

inline const char *attention_fault(const charsiu_gpu_pages *p, const charsiu_gpu_attention *a)
{
	const char *why = pages_fault(p);
	if (*why)
		return why;
	if (!a || !a->slots || (a->n_group && (!a->group || !a->shared)))
		return "the batch lacks an array";
	if (!a->n_tok || !a->n_head || a->n_head % p->n_head_kv)
		return "n_tok is 0, or n_head no multiple of n_head_kv";
	// (each factor by itself first: the product of three stays in 64 bits then)
	if (a->n_seq > ATTN_MAX_SEQS || a->n_tok > ATTN_MAX_ROWS || a->n_head > ATTN_MAX_ROWS ||
	    (uint64_t)a->n_seq * a->n_tok > ATTN_MAX_ROWS ||
	    (uint64_t)a->n_seq * a->n_tok * a->n_head > ATTN_MAX_ROWS || a->n_group > a->n_seq ||
	    a->n_group > ATTN_MAX_GROUPS)
		return "the batch is larger than the call takes";
	if (a->out_type != TYPE_F32 && a->out_type != p->type)
		return "out_type is neither fp32 nor the cache's type";
	return "";
}

constexpr int ADAPT_MAX_SETS = 8;

inline const char *adapters_fault(const charsiu_gpu_adapters *s, unsigned n)
{
	if (!s || !n || n > (unsigned)ADAPT_MAX_SETS)
		return "a call takes 1 to 8 adapter sets";
	for (unsigned i = 0; i < n; i++) {
		if (!s[i].a || !s[i].b || !s[i].rank || !s[i].scale)
			return "an adapter set lacks an array";
		if (s[i].type != s[0].type || (s[i].type != TYPE_F16 && s[i].type != TYPE_BF16))
			return "the adapters' types are not all fp16 or all bf16";
		if (!s[i].k || s[i].k % 32 || s[i].k != s[0].k || !s[i].n || s[i].n > 0x7fffff00u)
			return "the adapters' K is not one multiple of 32, or an N is 0";
		if (!s[i].max_rank || s[i].max_rank > 128 || (s[i].max_rank != 4 && s[i].max_rank % 8))
			return "an adapter set's max_rank is not 4 or a multiple of 8 up to 128";
		if (misaligned(s[i].a, 16) || misaligned(s[i].b, 16) || misaligned(s[i].rank, 4) ||
		    misaligned(s[i].scale, 4))
			return "an array of an adapter set is misaligned";
		if (s[i].slots > 0x7fffffffu)
			return "an adapter set is larger than the call takes";
	}
	return "";
}

} // namespace cgpu
