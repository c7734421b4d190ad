// Launchers of the incremental operators: rotary positions, writes into the
// paged cache, attention over it and its page maintenance (each returns 0 or a
// negative blt_status).
#pragma once
#include "rowops.hpp"

namespace blt {

// ---- k_rotary.hip ------------------------------------------------------------
// Heads of one tensor of a rotary launch: `heads` of them from `x`, rotated
// into `y`; strides in elements.
struct RotarySet {
  const void* x;
  void* y;
  int heads;
  int64_t sb_x, sh_x, st_x, sb_y, sh_y, st_y;
};
struct RotaryArgs {
  RotarySet q, k;
  int64_t B, T;
  int d;
  const int32_t* pos;  // position of token t of row b: pos[b * sb_pos + t]
  int64_t sb_pos;
  blt_rotary r;
  int backward;
};
int launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s);

struct AppendArgs {
  const void *q, *k, *v;
  void* q_out;
  int Hq;
  int64_t st_q, sh_q, st_qo, sh_qo, st_k, sh_k, st_v, sh_v;
  const int32_t *starts, *seqs;
  int64_t B, total;
  int layer;
  blt_rotary r;
};
int launch_append(const blt_paged_cache& c, const AppendArgs& a, hipStream_t s);

// status bits that hold back writes until they are cleared
constexpr int kCachePending =
    BLT_CACHE_FULL | BLT_CACHE_TOO_LONG | BLT_CACHE_BAD_INDEX | BLT_CACHE_BUSY;

// ---- k_pages.hip -------------------------------------------------------------
constexpr int kPageListMax = 8192;  // sequences of one maintenance call
constexpr int kMaxSeqs = 65536;
int64_t cache_workspace_bytes(const blt_paged_cache& c, int64_t n);
int launch_cache_reserve(const blt_paged_cache& c, const int32_t* seqs, const int32_t* counts,
                         int64_t n, hipStream_t s);
int launch_cache_trim(const blt_paged_cache& c, const int32_t* seqs, const int32_t* lens,
                      int64_t n, void* ws, hipStream_t s);
int launch_cache_fork(const blt_paged_cache& c, const int32_t* src, const int32_t* dst, int64_t n,
                      hipStream_t s);
int launch_cache_compact(const blt_paged_cache& c, void* ws, hipStream_t s);
int launch_cache_copy_pages(const blt_paged_cache& c, const int32_t* src, const int32_t* dst,
                            int64_t n, hipStream_t s);

// ---- k_paged_attn.hip --------------------------------------------------------
struct PagedAttnArgs {
  const void* q;
  void* o;
  int64_t st_q, sh_q, st_o, sh_o;
  int H;
  const int32_t *starts, *seqs;
  int64_t B, total;
  int layer, causal, window;
  float scale;
};
int64_t paged_attention_workspace_bytes(const blt_paged_cache& c, int64_t B, int64_t total,
                                        int H);
int launch_paged_attention(const blt_paged_cache& c, const PagedAttnArgs& a, void* ws,
                           hipStream_t s);

inline int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

}  // namespace blt
