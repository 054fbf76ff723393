// Internal interface between the layer engine (layers_kernel.hip) and the packed-sequence attention
// (packed_kernel.hip); not part of the exported C header.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// Causal attention of the prefill's queries over packed prompts: num_seqs sequences of lengths[i] tokens
// (HOST array), their rows one after the other. Queries as the engine keeps them (bf16 hi/lo pair,
// [rows][16 * 128]); layer `layer` of sequence i's keys and values in its cache, seq_stride elements
// after that of sequence i - 1 ([layers][8][max_seq][128]). The normalised output goes to the next
// product's fragments: frag 1 or 2 of attn_out (layers_kernel.hip).
struct MkPackedPrefill {
  const uint16_t *qh, *ql, *k_cache, *v_cache;
  uint16_t *oh, *ol;
  int frag, layer, max_seq;
  int64_t seq_stride;
  const int32_t* lengths;
  int num_seqs;
};
hipError_t mkp_attention_prefill(const MkPackedPrefill& a, hipStream_t stream);
