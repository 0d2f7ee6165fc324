// Arguments of the attention over packed sequences (packed_attn.hip) and its launches, shared with the entry points.
#pragma once
#include "common.hpp"

namespace fvsr {

template <typename E>
struct HeadView {   // (tokens, heads, D) with D contiguous
  E* p;
  int64_t t, h;     // elements between tokens and between heads
};

struct PackedArgs {
  HeadView<const bf16> q, k, v, d_o;
  HeadView<bf16> o, dq, dk, dv;   // o is read by the backward pass
  float* lse;                     // (heads, tq), natural logarithms; may be null in the forward pass
  bf16* stat;                     // (heads, tq, 8) stat_parts of the queries, from the dQ kernel to the dK, dV kernel
  float* part;                    // partial results of the split walk, or of dK and dV
  int dkv_whole, dkv_parts;       // blocks of keys before the first whose queries are cut, and the parts that they are cut into
  const int32_t *cu_q, *cu_k, *used_k;   // used_k may be null
  int seqs, tq, tk;
  int heads, kv_heads, group, D, causal;
  int clear;                      // rows of no sequence: 1, o's or the gradients' are set to zeros; 2, lse's to -inf; or both
  int max_parts;                  // workgroups of the split walk
  float c, scale;                 // scale * log2(e), scale
};

size_t packed_forward_workspace(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads, int D);
int launch_packed_forward(PackedArgs a, void* ws, hipStream_t stream);
size_t packed_backward_workspace(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads, int D, bool causal);
int launch_packed_backward(PackedArgs a, void* ws, hipStream_t stream);

}  // namespace fvsr
