// Launchers of attention over packed sequences and its gradient (each returns 0 or a
// negative blt_status).
#pragma once
#include "rowops.hpp"

namespace blt {

// heads of [total, heads, d], strides in elements
struct PackedHeads {
  const void* x;
  int64_t st, sh;
};
struct PackedAttnArgs {
  PackedHeads q, k, v, o;  // (o is written)
  float* lse;              // [total, H] or null
  int dtype;
  int64_t total;
  int H, Hkv, d;
  const int32_t* starts;
  int64_t B;
  int causal, window;
  float scale;
  int tail;  // o behind the last sequence: 0 = left alone, 1 = zeros (lse: -inf)
};
int64_t packed_attention_workspace_bytes(int64_t B, int64_t total, int H, int Hkv, int dtype);
int launch_packed_attention(const PackedAttnArgs& a, void* ws, hipStream_t s);

// a.o and a.lse are the forward's; g: the output's gradient; dq, dk, dv are written
struct PackedGradArgs {
  PackedHeads g, dq, dk, dv;
};
int64_t packed_attention_backward_workspace_bytes(int64_t total, int H, int Hkv, int d, int dtype);
int launch_packed_attention_backward(const PackedAttnArgs& a, const PackedGradArgs& g, void* ws,
                                     hipStream_t s);

}  // namespace blt
