// Rotary positions: (x1, x2) -> (x1 cos a - x2 sin a, x1 sin a + x2 cos a) per pair
// and position, a = position * frequency, on q and k of any strides
// (rotary_kernel) and on new tokens on their way into the paged cache
// (append_kernel).
//
// The angle needs no table and no range reduction: a frequency is a 64-bit
// fraction of a turn, so the low 64 bits of position * frequency are the angle
// modulo a turn, to 2^-33 for any 32-bit position.  The upper word's quarter turn
// picks the quadrant, its remainder (|x| <= pi / 4) goes through the Taylor series
// of sine and cosine in f32 (first terms left out: x^11 / 11! and x^12 / 12!, below
// 2e-9).  Both kernels move bytes; a block computes the angles of its tokens once, into
// LDS, and applies them to every head.  [16, 24 heads, 8192, 64] bf16: 143 us, 5.6 TB/s; 5001
// f32 gradients of 40 heads of 128: 36 us, 5.7 TB/s (41 and 5.0 with cold inputs); 7418 tokens
// of 32 / 8 heads of 128 into the cache: 34 us, 5.3 TB/s (a large copy: 6.15).
#include <math.h>

#include "paged.hpp"

namespace blt {

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <typename T>
struct Conv;
template <>
struct Conv<float> {
  __device__ static float in(float x) { return x; }
  __device__ static float out(float x) { return x; }
};
template <>
struct Conv<uint16_t> {
  __device__ static float in(uint16_t x) { return bf16_to_f32(x); }
  __device__ static uint16_t out(float x) { return f32_to_bf16(x); }
};

// V elements moved at once (16 bytes, or one element)
template <typename T, int V>
struct Piece {
  T e[V];
};
template <typename T, int V>
__device__ inline Piece<T, V> load_piece(const T* p) {
  Piece<T, V> r;
  if constexpr (V == 1) {
    r.e[0] = *p;
  } else {
    static_assert(sizeof(T) * V == 16, "16-byte pieces");
    r = __builtin_bit_cast(Piece<T, V>, *reinterpret_cast<const u32x4_t*>(p));
  }
  return r;
}
template <typename T, int V>
__device__ inline void store_piece(T* p, const Piece<T, V>& r) {
  if constexpr (V == 1)
    *p = r.e[0];
  else
    *reinterpret_cast<u32x4_t*>(p) = __builtin_bit_cast(u32x4_t, r);
}

// cosine and sine of pos * freq (a 64-bit fraction of a turn)
__device__ inline void angle_of(int pos, uint64_t freq, float& c, float& s) {
  const uint64_t angle = (uint64_t)(int64_t)pos * freq;
  const uint32_t hi = (uint32_t)((angle + 0x80000000ull) >> 32);  // rounded
  const uint32_t quad = (hi + 0x20000000u) >> 30;                // nearest quarter turn
  const int rem = (int)(hi - (quad << 30));                      // [-2^29, 2^29)
  const float x = (float)rem * 1.46291807926715968e-9f;          // pi / 2^31
  const float z = x * x;
  const float sn = x * (1.f + z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880)))));
  const float cs = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float a = quad & 1 ? sn : cs, b = quad & 1 ? cs : sn;
  c = (quad + 1) & 2 ? -a : a;
  s = quad & 2 ? -b : b;
}

// A unit of a head: two pieces.  The rotary_dim / (2 V) first ones rotate V pairs, the
// others ((d - rotary_dim) / (2 V) of them) are copied.
template <int V>
struct Unit {
  int a, b;  // element offsets of its pieces
  bool rot;
  int pair;  // its first pair
};
template <int V>
__device__ inline Unit<V> unit_of(int u, const blt_rotary& r) {
  Unit<V> t;
  const int nr = r.rotary_dim / (2 * V);
  t.rot = u < nr;
  t.pair = u * V;
  if (t.rot && !r.interleaved) {
    t.a = u * V;
    t.b = t.a + r.rotary_dim / 2;
  } else {
    t.a = 2 * u * V;
    t.b = t.a + V;
  }
  return t;
}

// The (cosine, sine) pairs of a token, times the magnitude, into `out`: its `step` threads
// take them in turn.
__device__ inline void token_angles(const blt_rotary& r, int pos, int first, int step,
                                    bool backward, f32x2_t* out) {
  for (int i = first; i < r.rotary_dim / 2; i += step) {
    float c, s;
    angle_of(pos, r.freq[i], c, s);
    out[i] = f32x2_t{c * r.magnitude, s * (backward ? -r.magnitude : r.magnitude)};
  }
}

// one pair, with its roundings written out: every variant gives the same bits
__device__ inline void turn(float x, float y, float c, float s, float& a, float& b) {
  a = fmaf(x, c, -(y * s));
  b = fmaf(x, s, y * c);
}
template <typename T, int V>
__device__ inline void rotate(Piece<T, V>& a, Piece<T, V>& b, const f32x2_t* cs,
                              bool interleaved) {
  float p, q;
  if (!interleaved) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      turn(Conv<T>::in(a.e[e]), Conv<T>::in(b.e[e]), cs[e].x, cs[e].y, p, q);
      a.e[e] = Conv<T>::out(p);
      b.e[e] = Conv<T>::out(q);
    }
  } else if constexpr (V == 1) {
    turn(Conv<T>::in(a.e[0]), Conv<T>::in(b.e[0]), cs[0].x, cs[0].y, p, q);
    a.e[0] = Conv<T>::out(p);
    b.e[0] = Conv<T>::out(q);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      Piece<T, V>& w = e < V / 2 ? a : b;
      const int i = 2 * (e % (V / 2));
      turn(Conv<T>::in(w.e[i]), Conv<T>::in(w.e[i + 1]), cs[e].x, cs[e].y, p, q);
      w.e[i] = Conv<T>::out(p);
      w.e[i + 1] = Conv<T>::out(q);
    }
  }
}

// heads whose pieces a thread of rotary_kernel has in flight
template <typename T>
constexpr int kBatch = sizeof(T) == 2 ? 4 : 6;

// How a block's threads are dealt: `units` of a head side by side, `hg` heads (each
// thread takes every hg-th), then `tb` tokens.
struct Deal {
  int units, hg, tb;
  int64_t blocks;
};
// Where the tokens fill the chip by themselves a thread of rotary_kernel takes one batch of
// heads, otherwise (and in append_kernel always) every head has its own thread, as far
// as a block has room.  [16, 24 heads, 8192, 64] bf16 takes 143 us with batches of four,
// 144 with six, 150 with eight, 169 with one; 5001 f32 gradients of 40 heads of 128, half
// rotated, 40 us with four and 38 with six.  7418 tokens of 32 / 8 heads of 128 into the
// cache take 35 us with one head a thread, 36 with two, 38 with three, 41 with four.
inline Deal deal(int d, int v, int heads, int64_t tokens, int batch) {
  Deal t;
  t.units = d / (2 * v);
  const int most = t.units >= 256 ? 1 : 256 / t.units;
  if (tokens * t.units < (int64_t)256 * 1024) batch = 1;
  const int64_t want = (heads + batch - 1) / batch;
  t.hg = (int)(want < most ? want : most);
  t.tb = 256 / (t.units * t.hg);
  if (t.tb < 1) t.tb = 1;
  if (t.tb > tokens) t.tb = (int)tokens;
  t.blocks = (tokens + t.tb - 1) / t.tb;
  return t;
}

template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p, Deal dl) {
  const int tid = threadIdx.x;
  const int u0 = tid % dl.units, rest = tid / dl.units;
  const int h0 = rest % dl.hg, tt = rest / dl.hg;
  __shared__ __attribute__((aligned(16))) f32x2_t angles[256 * V];  // (tb * rotary_dim / 2 of them)
  const int64_t tokens = p.B * p.T;
  const int64_t tok = (int64_t)blockIdx.x * dl.tb + tt;
  const bool mine = tt < dl.tb && tok < tokens;
  const int64_t b = tok / p.T, t = tok - b * p.T;
  const Unit<V> un = unit_of<V>(u0, p.r);
  const f32x2_t* cs = angles + tt * (p.r.rotary_dim / 2) + un.pair;
  if (mine)
    token_angles(p.r, p.pos[b * p.sb_pos + t], h0 * dl.units + u0, dl.units * dl.hg, p.backward,
                 angles + tt * (p.r.rotary_dim / 2));
  __syncthreads();
  if (!mine) return;
  const int heads = p.q.heads + p.k.heads;
  for (int hb = h0; hb < heads; hb += kBatch<T> * dl.hg) {
    Piece<T, V> a[kBatch<T>], w[kBatch<T>];
#pragma unroll
    for (int i = 0; i < kBatch<T>; ++i) {
      const int h = hb + i * dl.hg;
      if (h < heads) {
        const bool iq = h < p.q.heads;
        const T* x = iq ? (const T*)p.q.x + b * p.q.sb_x + t * p.q.st_x + h * p.q.sh_x
                        : (const T*)p.k.x + b * p.k.sb_x + t * p.k.st_x + (h - p.q.heads) * p.k.sh_x;
        a[i] = load_piece<T, V>(x + un.a);
        w[i] = load_piece<T, V>(x + un.b);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch<T>; ++i) {
      const int h = hb + i * dl.hg;
      if (h < heads) {
        const bool iq = h < p.q.heads;
        T* y = iq ? (T*)p.q.y + b * p.q.sb_y + t * p.q.st_y + h * p.q.sh_y
                  : (T*)p.k.y + b * p.k.sb_y + t * p.k.st_y + (h - p.q.heads) * p.k.sh_y;
        if (un.rot) rotate<T, V>(a[i], w[i], cs, p.r.interleaved);
        store_piece<T, V>(y + un.a, a[i]);
        store_piece<T, V>(y + un.b, w[i]);
      }
    }
  }
}

struct AppendKernelArgs {
  AppendArgs a;
  blt_paged_cache c;
  int lps;         // log2 page_size
  int64_t layer0;  // the layer's first element
};

// New tokens into the cache: heads 0 .. Hq - 1 of a token are q's (rotated into q_out),
// then k's (rotated into its page), then v's (copied).
template <typename T, int V>
__global__ __launch_bounds__(256) void append_kernel(AppendKernelArgs p, Deal dl) {
  const AppendArgs& a = p.a;
  const blt_paged_cache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int u0 = tid % dl.units, rest = tid / dl.units;
  const int h0 = rest % dl.hg, tt = rest / dl.hg;
  const int64_t tok0 = (int64_t)blockIdx.x * dl.tb, tok = tok0 + tt;
  const bool mine = tt < dl.tb && tok < a.total;
  // The token's row b: the number of starts[1 ..] at or below it; its first token and
  // length.  Up to 64 rows a wave holds them all, one round of loads ahead of the page's;
  // beyond that every wave counts for the block's first token and goes on from there.
  int64_t s0 = 0, n = 0;
  int seq = -1, len = 0;
  bool found = false;
  bool crossed = false;  // starts that do not ascend within the tokens
  if (a.B <= 64) {
    const int i = lane < a.B ? lane : (int)a.B - 1;
    const int lo = a.starts[i], hi = a.starts[i + 1];
    const int sq = a.seqs ? a.seqs[i] : i;
    const int ln = c.lens[sq >= 0 && sq < c.max_seqs ? sq : 0];
    crossed = lo < 0 || hi < lo || hi > a.total;
    int b = __popcll(__ballot(lane < a.B && hi <= tok0));
    // (every lane takes part in the shuffles; tokens past the last row stop at 64)
    for (int next = __shfl(hi, b & 63); __any(b < a.B && next <= tok); next = __shfl(hi, b & 63))
      b += b < a.B && next <= tok ? 1 : 0;
    s0 = __shfl(lo, b & 63);
    n = __shfl(hi, b & 63) - s0;
    seq = __shfl(sq, b & 63);
    len = __shfl(ln, b & 63);
    found = mine && b < a.B;  // (else behind the last row)
  } else {
    int b = 0;
    for (int64_t i = 0; i < a.B; i += 64) {
      const bool le = i + lane < a.B && a.starts[i + lane + 1] <= tok0;
      const uint64_t m = __ballot(le);
      b += __popcll(m);
      if (m != ~0ull) break;
    }
    while (mine && b < a.B && a.starts[b + 1] <= tok) ++b;
    if (blockIdx.x == 0)
      for (int64_t i = tid; i < a.B; i += 256)
        crossed = crossed || a.starts[i] < 0 || a.starts[i + 1] < a.starts[i] ||
                  a.starts[i + 1] > a.total;
    found = mine && b < a.B;
    if (found) {
      s0 = a.starts[b];
      n = a.starts[b + 1] - s0;
      seq = a.seqs ? a.seqs[b] : b;
      len = c.lens[seq >= 0 && seq < c.max_seqs ? seq : 0];
    }
  }
  found = found && tok >= s0;
  const bool known = seq >= 0 && seq < c.max_seqs;
  const int64_t pos = (known ? len : 0) - n + (tok - s0);
  // where k and v go: no page where an index is out of range or a failure is pending
  // (looked at behind the angles, which need not wait for it)
  const bool inside = found && known && pos >= 0 && (pos >> p.lps) < c.max_pages;
  const int page = inside ? c.page_table[(int64_t)seq * c.max_pages + (pos >> p.lps)] : -1;
  const int status = *c.status;

  const Unit<V> un = unit_of<V>(u0, a.r);
  __shared__ __attribute__((aligned(16))) f32x2_t angles[256 * V];
  const f32x2_t* cs = angles + tt * (a.r.rotary_dim / 2) + un.pair;
  if (found)
    token_angles(a.r, (int)pos, h0 * dl.units + u0, dl.units * dl.hg, false,
                 angles + tt * (a.r.rotary_dim / 2));
  if (blockIdx.x == 0 && __any(crossed) && lane == 0) atomicOr(c.status, BLT_CACHE_BAD_INDEX);
  __syncthreads();
  if (!found) return;
  const bool bad = page < 0 || page >= c.num_pages;
  if (bad && u0 == 0 && h0 == 0) atomicOr(c.status, BLT_CACHE_NO_PAGE);
  const int Hk = c.n_kv_heads, heads = a.Hq + 2 * Hk;
  const int64_t sh_page = (int64_t)c.head_dim << p.lps;
  const int64_t at = bad || (status & kCachePending)
                         ? -1
                         : p.layer0 + (int64_t)page * c.n_kv_heads * sh_page +
                               (pos & (c.page_size - 1)) * c.head_dim;
  for (int h = h0; h < heads; h += dl.hg) {
    const T* src = h < a.Hq ? (const T*)a.q + tok * a.st_q + h * a.sh_q
                   : h < a.Hq + Hk ? (const T*)a.k + tok * a.st_k + (h - a.Hq) * a.sh_k
                                   : (const T*)a.v + tok * a.st_v + (h - a.Hq - Hk) * a.sh_v;
    Piece<T, V> x = load_piece<T, V>(src + un.a), y = load_piece<T, V>(src + un.b);
    T* dst;
    if (h < a.Hq) {
      dst = (T*)a.q_out + tok * a.st_qo + h * a.sh_qo;
    } else {
      if (at < 0) continue;
      dst = h < a.Hq + Hk ? (T*)c.k + at + (h - a.Hq) * sh_page
                          : (T*)c.v + at + (h - a.Hq - Hk) * sh_page;
    }
    if (un.rot && h < a.Hq + Hk) rotate<T, V>(x, y, cs, a.r.interleaved);
    store_piece<T, V>(dst + un.a, x);
    store_piece<T, V>(dst + un.b, y);
  }
}

inline bool whole(int64_t stride, int v) { return stride % v == 0; }
inline bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s) {
  const int64_t tokens = a.B * a.T;
  const int heads = a.q.heads + a.k.heads;
  if (tokens == 0 || heads == 0) return 0;
  const int v = dtype == BLT_DTYPE_BF16 ? 8 : 4;
  bool vec = a.r.rotary_dim % (2 * v) == 0 && (a.d - a.r.rotary_dim) % (2 * v) == 0;
  for (const RotarySet* x : {&a.q, &a.k})
    if (x->heads)
      vec = vec && aligned(x->x) && aligned(x->y) && whole(x->sb_x, v) && whole(x->sh_x, v) &&
            whole(x->st_x, v) && whole(x->sb_y, v) && whole(x->sh_y, v) && whole(x->st_y, v);
  const Deal dl = deal(a.d, vec ? v : 1, heads, tokens,
                       dtype == BLT_DTYPE_BF16 ? kBatch<uint16_t> : kBatch<float>);
  if (dl.blocks > 0x7fffffff) return fail(BLT_ERR_SHAPE, "fused_rotary: too many tokens");
  const dim3 g((unsigned)dl.blocks), b(256);
  if (dtype == BLT_DTYPE_BF16) {
    if (vec) hipLaunchKernelGGL((rotary_kernel<uint16_t, 8>), g, b, 0, s, a, dl);
    else hipLaunchKernelGGL((rotary_kernel<uint16_t, 1>), g, b, 0, s, a, dl);
  } else {
    if (vec) hipLaunchKernelGGL((rotary_kernel<float, 4>), g, b, 0, s, a, dl);
    else hipLaunchKernelGGL((rotary_kernel<float, 1>), g, b, 0, s, a, dl);
  }
  BLT_LAUNCH_CHECK("rotary_kernel");
  return 0;
}

int launch_append(const blt_paged_cache& c, const AppendArgs& a, hipStream_t s) {
  if (a.total == 0 || a.B == 0) return 0;
  const int v = c.dtype == BLT_DTYPE_BF16 ? 8 : 4;
  const int d = c.head_dim;
  bool vec = a.r.rotary_dim % (2 * v) == 0 && aligned(a.k) && aligned(a.v) && whole(a.st_k, v) &&
             whole(a.sh_k, v) && whole(a.st_v, v) && whole(a.sh_v, v);
  if (a.Hq)
    vec = vec && aligned(a.q) && aligned(a.q_out) && whole(a.st_q, v) && whole(a.sh_q, v) &&
          whole(a.st_qo, v) && whole(a.sh_qo, v);
  const Deal dl = deal(d, vec ? v : 1, a.Hq + 2 * c.n_kv_heads, a.total, 1);
  if (dl.blocks > 0x7fffffff) return fail(BLT_ERR_SHAPE, "cache_append: too many tokens");
  AppendKernelArgs p{a, c, log2_of(c.page_size), 0};
  p.layer0 = (int64_t)a.layer * c.num_pages * c.n_kv_heads * c.page_size * d;
  const dim3 g((unsigned)dl.blocks), b(256);
  if (c.dtype == BLT_DTYPE_BF16) {
    if (vec) hipLaunchKernelGGL((append_kernel<uint16_t, 8>), g, b, 0, s, p, dl);
    else hipLaunchKernelGGL((append_kernel<uint16_t, 1>), g, b, 0, s, p, dl);
  } else {
    if (vec) hipLaunchKernelGGL((append_kernel<float, 4>), g, b, 0, s, p, dl);
    else hipLaunchKernelGGL((append_kernel<float, 1>), g, b, 0, s, p, dl);
  }
  BLT_LAUNCH_CHECK("append_kernel");
  return 0;
}

}  // namespace blt
