// SPDX-License-Identifier: GPL-2.0-or-later
// What the decode step (decoder.cu) and the operators of a batched step
// (batch_ops.cu) read of a GPU layer beyond the C ABI.
// Hidden symbols of the library, not part of include/charsiu_gpu.h.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

struct charsiu_gpu;

namespace cgpu {

int layer_device(const charsiu_gpu *g);
bool layer_no_pdl(const charsiu_gpu *g);
bool layer_whole(const charsiu_gpu *g);
bool layer_tensor(const charsiu_gpu *g, int id, uint64_t *k, uint64_t *rows, uint32_t *type);
void layer_whine(charsiu_gpu *g, const char *why);
bool layer_dead(const charsiu_gpu *g);
int layer_sms(const charsiu_gpu *g);
cudaStream_t layer_stream(const charsiu_gpu *g);
int *layer_kernel_error(const charsiu_gpu *g);   // the device word a wait that gave up writes
void layer_launched(charsiu_gpu *g, unsigned n);
void *tensor_map_encode();      // the driver's cuTensorMapEncodeTiled, or null

} // namespace cgpu
