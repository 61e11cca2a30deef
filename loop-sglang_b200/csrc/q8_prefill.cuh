// Attention of requests with several query rows over the 8-bit KV cache: the launcher that
// lsb_paged_attention_q8 dispatches prompts to.
#pragma once

#include "q8.cuh"

namespace lsb {

struct Q8PrefillParams {
  bf16* out;
  int64_t out_stride;
  const bf16* q;
  int64_t q_stride;
  const uint8_t *k, *v;
  int64_t slot_stride, num_slots;
  const float *ks, *vs;
  int block_shift;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t *cache_seqlens, *cu_seqlens_q;
  int num_reqs;
  int64_t rows;
  int hkv, group, page_size;
  int64_t max_seqlen;
  float scale_log2;
  int* error_flag;
};

int launch_q8_prefill(const Q8PrefillParams& p, int head_dim, bool int8, cudaStream_t stream);

}  // namespace lsb
