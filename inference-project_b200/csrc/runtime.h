// Host-side helpers shared by the translation units of libinf.so.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/inf.h"

namespace inf {

// Records a description of the failure for inf_last_error_detail() and returns err.
Error_t fail(Error_t err, const char* fmt, ...);

#define INF_CUDA_TRY(expr)                                                                                  \
	do {                                                                                                    \
		cudaError_t inf_e_ = (expr);                                                                        \
		if (inf_e_ != cudaSuccess)                                                                          \
			return ::inf::fail(ErrorCuda, "%s:%d %s: %s", __FILE__, __LINE__, #expr, cudaGetErrorString(inf_e_)); \
	} while (0)

#define INF_TRY(expr)                          \
	do {                                       \
		Error_t inf_r_ = (expr);               \
		if (inf_r_ != Success) return inf_r_;  \
	} while (0)

bool is_device_ptr(const void* p);
// Whether p is memory the current device's kernels may be given: device memory of that device, or
// managed memory.
bool is_local_device_ptr(const void* p);

// The Error_t of a device error word (DevErr), with its description recorded.
Error_t map_dev_err(int v);

// A layer's paged K or V pool [pages][KV][blk][hd] as a 4-D tensor (hd, row, head, page) with boxes
// of 64 head dims x blk rows x 1 head x box_pages pages, SWIZZLE_128B.
Error_t tensor_map_kv(CUtensorMap* m, const void* base, u32 hd, u32 blk, u32 kv, u32 pages, u32 box_pages);
// Rows of `heads` heads of hd, `stride` elements apart, as a 3-D tensor (dim, head, token) with boxes of 64 dims x
// box_heads x box_tokens, SWIZZLE_128B.
Error_t tensor_map_q(CUtensorMap* m, const void* base, u32 tokens, u32 heads, u32 hd, u64 stride, u32 box_heads, u32 box_tokens);
// A K or V pool as a 5-D tensor (64 dims of a row, 8 rows, head_dim / 64, blk / 8, page), SWIZZLE_128B: a box is
// box_groups 8-row groups of one head of box_pages consecutive pages, and lands as [box_pages * box_groups][head_dim / 64][8 rows x 128 bytes], an even
// stride between the 8-row groups of all pages.  The second coordinate is head * blk.
Error_t tensor_map_kv_groups(CUtensorMap* m, const void* base, u32 hd, u32 blk, u32 kv, u32 pages, u32 box_pages, u32 box_groups);

// Whether inf_set_sampling turned sampling on for this model (false for NULL).
bool model_sampling_on(const Model* m);

// inf_forward_batch; single_batched runs even one sequence through the batched tensor-core
// step (inf_forward_batch gives a lone sequence the batch-1 decode kernels instead), so a
// sequence's results do not depend on how many others share the step.
Error_t forward_batch(Model* model, u32 n_seqs, const u32* seq_slots, const u32* ids, const u32* positions,
                      f32* logits_out, u32* argmax_out, bool single_batched);

// After an inf_forward of `slot` whose new token sits at pos_new: replaces *id (the token the
// forward chose) by a draw under the slot's inf_set_slot_sampling settings, when they sample.
Error_t sample_slot_token(Model* model, u32 slot, u32 pos_new, u32* id);

} // namespace inf
