// SPDX-License-Identifier: GPL-2.0-or-later
// CPU check of cgpu::attn_piece (charsiu_b200/csrc/attn_cut.h), built and run by
// tests/test_batch_ops_cpu.py: for lengths up to the longest that a cache may tell, the
// pieces are the keys, each once, in order, cut at whole grains. Prints "ok <cuts>" and
// exits 0, or the first wrong cut and 1.
#include <cstdio>
#include <initializer_list>

#define __host__
#define __device__
#define __forceinline__ inline
#include "attn_cut.h"

int main()
{
	int cuts = 0;
	const long long longest = 0x7fffff00;
	for (long long from : {0ll, 16ll, 4096ll, longest - 128, longest})
		for (long long to : {0ll, 1ll, 16ll, 127ll, 128ll, 129ll, 511ll, 513ll, 5000ll, 1ll << 20, (1ll << 30) + 1, 0x7ffffd00ll,
				   0x7ffffe00ll, 0x7ffffe01ll, 0x7ffffe80ll, 0x7ffffeffll, longest})
			for (uint32_t n : {1u, 2u, 3u, 7u, 31u, 32u})
				for (uint32_t grain : {128u, 512u}) {
					int64_t at = from < to ? from : to;
					for (uint32_t i = 0; i < n; i++, cuts++) {
						int32_t k0 = (int32_t)from, k1 = (int32_t)to;
						cgpu::attn_piece(k0, k1, i, n, grain);
						const bool good = k0 == at && k1 >= k0 && k1 <= to &&
								  (k1 == to || (k1 - from) % grain == 0);
						if (!good) {
							printf("keys %lld to %lld, piece %u of %u by %u: %d to %d, not from %lld\n",
							       (long long)from, (long long)to, i, n, grain, k0, k1, (long long)at);
							return 1;
						}
						at = k1;
					}
					if (at != to) {
						printf("keys %lld to %lld in %u by %u: up to %lld\n", (long long)from, (long long)to, n,
						       grain, (long long)at);
						return 1;
					}
				}
	printf("ok %d\n", cuts);
	return 0;
}
