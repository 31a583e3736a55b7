// SPDX-License-Identifier: GPL-2.0-or-later
// CPU check of what the operators of a batched step refuse
// (charsiu_b200/csrc/batch_checks.h), built and run by tests/test_batch_ops_cpu.py.
// Prints "ok <checks>" and exits 0, or every wrong answer and 1.
#include <cstdio>
#include <initializer_list>

#include "batch_checks.h"

using namespace cgpu;

namespace {

int checks, wrong;

void expect(bool refused, const char *why, const char *what, unsigned long long a = 0, unsigned long long b = 0,
	    unsigned long long c = 0)
{
	checks++;
	if ((*why != 0) != refused) {
		wrong++;
		printf("%s %llu %llu %llu: %s\n", what, a, b, c, *why ? why : "accepted");
	}
}

template <typename T>
T *at(uintptr_t address)
{
	return reinterpret_cast<T *>(address);
}

charsiu_gpu_pages cache()
{
	charsiu_gpu_pages p = {};
	p.k = at<void>(1 << 20);
	p.v = at<void>(1 << 21);
	p.table = p.len = p.ref = p.work = at<int32_t>(1 << 12);
	p.layer_stride = 1 << 16;
	p.page_stride = 8192;
	p.pos_stride = 512;
	p.head_stride = 64;
	p.type = TYPE_BF16;
	p.n_layer = 2;
	p.n_pages = 8;
	p.page = 16;
	p.n_head_kv = 1;
	p.head_dim = 64;
	p.n_seq = 4;
	p.max_pages = 4;
	return p;
}

charsiu_gpu_attention batch(uint32_t n_seq, uint32_t n_tok, uint32_t n_head)
{
	charsiu_gpu_attention a = {};
	a.slots = at<const int32_t>(64);
	a.n_seq = n_seq;
	a.n_tok = n_tok;
	a.n_head = n_head;
	a.out_type = TYPE_F32;
	return a;
}

// n_seq * n_tok * n_head is at most 2^25, also where the product of the three passes 64 bits
void attention_sizes()
{
	const charsiu_gpu_pages p = cache();
	const uint32_t powers[] = {0, 1, 4, 5, 12, 13, 15, 16, 17, 24, 25, 26, 30, 31};
	for (uint32_t s : powers)
		for (uint32_t t : powers)
			for (uint32_t h : powers)
				for (uint32_t less = 0; less < 2; less++) {
					const charsiu_gpu_attention a = batch(1u << s, 1u << t, (1u << h) - (less && h));
					// (exact: at most 93 bits)
					const bool fits = (unsigned __int128)a.n_seq * a.n_tok * a.n_head <= 1u << 25 && a.n_seq <= 65536;
					expect(!fits, attention_fault(&p, &a), "attention", a.n_seq, a.n_tok, a.n_head);
				}
	for (uint32_t n_seq : {3u, 4u, 65536u}) {
		const charsiu_gpu_attention a = batch(n_seq, 0xffffffffu, 0xffffffffu);
		expect(true, attention_fault(&p, &a), "attention", n_seq, a.n_tok, a.n_head);
	}
	const charsiu_gpu_attention none = batch(0, 5, 8);
	expect(false, attention_fault(&p, &none), "attention of nothing");
}

// a list that the planners would read misaligned (a fault there) is refused on the host
void lists_of_slots()
{
	for (uintptr_t off = 0; off < 8; off++)
		expect(off % 4 != 0, slots_fault(at<const int32_t>(4096 + off), 3), "slots at", off);
	expect(false, slots_fault(at<const int32_t>(4098), 0), "no slots");
	expect(true, slots_fault(nullptr, 1), "null slots");
	expect(false, slots_fault(at<const int32_t>(4096), 1024), "1024 slots");
	expect(true, slots_fault(at<const int32_t>(4096), 1025), "1025 slots");
}

} // namespace

int main()
{
	lists_of_slots();
	attention_sizes();
	if (wrong)
		return 1;
	printf("ok %d\n", checks);
	return 0;
}
