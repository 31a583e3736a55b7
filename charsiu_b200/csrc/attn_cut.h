// SPDX-License-Identifier: GPL-2.0-or-later
// How the keys of an item of attention are cut into pieces.
#pragma once

#include <cstdint>

namespace cgpu {

// Piece `i` of `n` of the keys [k0, k1): whole grains, but for the last. Unsigned, and the ends in 64
// bits: a sequence may have up to 0x7fffff00 keys, and a grain more does not fit 31 bits.
__host__ __device__ __forceinline__ void attn_piece(int32_t &k0, int32_t &k1, uint32_t i, uint32_t n,
						    uint32_t grain)
{
	if (k0 >= k1) {
		k0 = k1;
		return;
	}
	const uint32_t grains = ((uint32_t)(k1 - k0) - 1) / grain + 1, each = ((grains - 1) / n + 1) * grain;
	const int64_t b = k0 + (int64_t)i * each, e = b + each;
	const int32_t last = k1;
	k0 = (int32_t)(b < last ? b : last);
	k1 = (int32_t)(e < last ? e : last);
}

} // namespace cgpu
