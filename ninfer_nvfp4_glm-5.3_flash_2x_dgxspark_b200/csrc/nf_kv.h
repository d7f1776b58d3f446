// nf_kv.h -- what the operators of the drafted-token step share: the checks of
// their host arguments, the thread's error message, and the launchers that the
// entry points and the decoder stack both use.
#pragma once

#include "nf_moe.h"

#include <cuda_runtime.h>
#include <stdint.h>

namespace nf {

// Sets the thread's message (nf_kv_last_error) and returns `status`.
int kv_fail(int status, const char* fmt, ...);
void kv_clear_error();
// The cache description alone: kind, shape, pointers, alignment.
int kv_check_cache(const nf_kv_cache* c);

// The launchers check nothing.  `slices` F32 matrices slice_stride elements
// apart are summed into qkv (a split-K projection's parts).
cudaError_t launch_kv_write(const nf_kv_cache& c, const nf_rope& rope, const void* qkv, int qkv_type,
                            int64_t row_stride, int tokens, int q_heads, const float* q_norm, const float* k_norm,
                            float eps, const int32_t* pos, const int32_t* seq, const int32_t* slot, uint16_t* q,
                            int32_t* status, cudaStream_t st, int slices = 1, int64_t slice_stride = 0);
// BF16 rows [n][head_dim] as E4M3 codes with a scale each (a cache's layout).
cudaError_t launch_kv_quantize(const uint16_t* x, int64_t n, int head_dim, uint8_t* codes, float* scale, cudaStream_t st);
// The rows of a batch of sequences: their sequence, cache slot (prefix + row
// of the sequence) and rotary position (prefix + depth); rows behind the last
// sequence get slot -1, those of a sequence that does not fit places that
// launch_kv_write refuses.
cudaError_t launch_kv_places(int rows, int max_context, const int32_t* row_start, int batch, const int32_t* prefix, const int32_t* depth,
                             int32_t* seq, int32_t* slot, int32_t* pos, cudaStream_t st);
cudaError_t launch_tree_attention(const nf_kv_cache& c, const uint16_t* q, int rows, int q_heads,
                                  const int32_t* row_start, int batch, const int32_t* prefix, const int32_t* cache_seq,
                                  const uint64_t* mask, int mask_words, float scale, uint16_t* out, void* work,
                                  int32_t* status, cudaStream_t st);
// With `epoch`: the logits lie epoch_bytes further when *epoch is odd.
cudaError_t launch_token_logprobs(const void* logits, int type, int64_t stride, int rows, int64_t vocab,
                                  const int32_t* target, int top, float* logprob, float* entropy, int32_t* top_idx,
                                  float* top_lp, cudaStream_t st, const uint32_t* epoch = nullptr,
                                  int64_t epoch_bytes = 0);
cudaError_t launch_kv_accept(const nf_kv_cache* caches, int layers, const int32_t* prefix, const int32_t* path,
                             int max_path, const int32_t* path_len, const int32_t* cache_seq, int batch,
                             int32_t* status, cudaStream_t st);

}  // namespace nf
