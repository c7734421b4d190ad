// One token a row from logits, by temperature, top-k, top-p and min-p, from given random
// numbers.
//
// With tokens ranked by logit (descending, equal ones by index) and weights
// w_i = e^((x_i - max) / temperature), the tokens kept are the first n ranks: at most top_k;
// those whose running sum before them is below top_p times the sum of the top_k; those with
// w >= min_p.  The token drawn is the lowest index whose running sum of kept weights, in the order
// of the indices, passes u times their sum.
//
// No sorting: all three rules keep a prefix of the ranks, so a row's choice is a cut, the last
// kept (logit, index), found by counting.  Weights are exponentials in 64 bits rounded to
// fixed point (the largest is 2^scale, scale = 62 - ceil(log2 vocab), so that a row's sum stays below
// 2^63): sums of integers do not depend on their order, so the tokens are the same in every run
// whatever adds up first.  A weight is off by less than 2^-44 of itself (see weight) and by its
// rounding, 2^-(scale + 1) of the largest.
//
// By the size of the vocabulary: up to 1024 a wave holds a row in registers and bisects
// the cut over the bits of the logits; up to 16384 a block holds it in LDS and counts bins; above that rows are
// cut into parts, in five launches.
#include <algorithm>

#include "sample.hpp"

namespace blt {

namespace {

struct Found;
struct Entry;
struct SArgs {
  const void* x;
  int64_t st;  // row stride
  int64_t rows;
  int V;
  const float* u;
  SampleSetting s;
  int32_t* out;
  int scale;
  // parts of rows
  int parts;
  float* pmax;      // [rows][parts], NaN where a logit is
  uint64_t* pmass;  // [rows][parts]
  uint64_t* hm;     // [rows][parts][NB]
  uint32_t* hc;     // [rows][parts][NB]
  Found* found;  // [rows]
  Entry* list;   // [rows][parts][NT]
  int* count;           // [rows][parts]: entries of it
};

template <typename T>
__device__ inline float logit(const void* x, int64_t i) {
  if constexpr (sizeof(T) == 2) return bf16_to_f32(((const uint16_t*)x)[i]);
  else return ((const float*)x)[i];
}
// an integer that orders as the value does (-0 as 0)
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// the last kept (logit, index): tokens with a larger key, or the same and an index up to this
struct Cut {
  uint32_t key;
  int index;
};
__device__ inline bool kept(const Cut& c, uint32_t key, int i) {
  return key > c.key || (key == c.key && i <= c.index);
}

// ---- a row's rules ---------------------------------------------------------------------
struct Rules {
  double a;     // log2(e) / temperature
  double p;     // top_p; 1 or more: off
  uint64_t m;   // smallest weight kept
  int k;        // 0: off
  float bins;   // bins per logit (see bin_of)
  bool good;
};
constexpr int NB = 2048;
__device__ inline Rules rules_of(const SArgs& g, int64_t row) {
  const SampleSetting& s = g.s;
  const double t = s.temperatures ? (double)s.temperatures[row] : s.temperature;
  const double p = s.top_ps ? (double)s.top_ps[row] : s.top_p;
  const double m = s.min_ps ? (double)s.min_ps[row] : s.min_p;
  const int k = s.top_ks ? s.top_ks[row] : s.top_k;
  Rules r;
  r.good = t >= 0. && t < (double)INFINITY && p > 0. && m >= 0. && m <= 1. && k >= 0 &&
           g.u[row] == g.u[row];
  r.a = t > 0. ? 1.4426950408889634074 / t : 1.;
  r.p = p;
  r.m = (uint64_t)ceil(ldexp(m, g.scale));
  r.k = t > 0. ? k : 1;  // (temperature 0: the first of the largest)
  if (r.k >= g.V) r.k = 0;
  // weights below 2^-63 share the last bin
  r.bins = (float)((NB - 1) / 63. * r.a);
  return r;
}
// 2^(j / 64), which a block keeps in LDS
struct Powers {
  double of[64];
};
__device__ inline void fill(Powers& p) {  // (a barrier before their use)
  if (threadIdx.x < 64) p.of[threadIdx.x] = exp2((double)threadIdx.x / 64.);
}
// 2^(scale - (top - x) a) as an integer: 2^y with y = k / 64 + f, |f| <= 1 / 128, is 2^(k / 64) times
// the series of 2^f up to f^4, off by less than 2^-44; its mantissa is shifted to its place.
// The largest logit has 2^scale exactly, equal ones equal weights.
__device__ inline uint64_t weight(float x, float top, const Rules& r, int scale, const Powers& pw) {
  if (x == top) return (uint64_t)1 << scale;
  // (in 64 bits here too: at temperatures near the ends of f32's range x - top or 1 / temperature passes
  // it where the weight does not vanish)
  const double y = ((double)x - (double)top) * r.a;
  if (!(y > -70.)) return 0;  // (scale <= 62)
  constexpr double L = 0.693147180559945309417;
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4;
  constexpr double M = 1.5 * 70368744177664.;  // 2^46: the sum below is a multiple of 1 / 64
  const double t = y + M, f = y - (t - M);
  const int k = (int)(uint32_t)__double_as_longlong(t);
  const double v = pw.of[k & 63] * fma(fma(fma(fma(c4, f, c3), f, c2), f, L), f, 1.);
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  // mantissa times 2^(exponent - 52 + k / 64 + scale), half of the last place up
  const uint64_t m = (b & 0xfffffffffffffull) | 0x10000000000000ull;
  const int shift = 52 + 1023 - scale - (int)(b >> 52) - (k >> 6);  // >= -10
  return shift > 0 ? ((m >> (min(shift, 55) - 1)) + 1) >> 1 : m << -shift;
}
// a bin of about the same logits, the largest ones first; the order of bins is that of logits
__device__ inline float place_of(float x, float top, const Rules& r) {
  const float t = (top - x) * r.bins;
  return x == top ? 0.f : t < (float)(NB - 1) ? t : (float)(NB - 1);
}
__device__ inline int bin_of(float x, float top, const Rules& r) { return (int)place_of(x, top, r); }
__device__ inline uint64_t wanted(double p, uint64_t sum) {  // least running sum >= p * sum
  const double x = ceil(p * (double)sum);
  return x >= (double)sum ? sum : x < 1. ? 1 : (uint64_t)x;
}
// u of the sum: the token is the first whose running sum is above
__device__ inline uint64_t aim_of(float u, uint64_t sum) {
  const double x = floor((double)fminf(fmaxf(u, 0.f), 1.f) * (double)sum);
  return x >= (double)sum ? sum - 1 : (uint64_t)x;
}

// ---- 64-bit sums over a wave -------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ inline uint64_t dpp_u64(uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
  return (uint64_t)hi << 32 | lo;
}
__device__ inline uint64_t lane_u64(uint64_t x, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
}
__device__ inline uint64_t incl_scan_u64(uint64_t v) {  // (as wave_incl_scan)
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
__device__ inline uint64_t sum_u64(uint64_t v) { return lane_u64(incl_scan_u64(v), 63); }
__device__ inline uint32_t wave_min_u32(uint32_t x) {
  return ~((uint32_t)wave_max_i32((int)(~x ^ 0x80000000u)) ^ 0x80000000u);
}
__device__ inline uint32_t wave_max_u32(uint32_t x) {
  return (uint32_t)wave_max_i32((int)(x ^ 0x80000000u)) ^ 0x80000000u;
}
__device__ inline int below(uint64_t mask) {  // set bits below this lane
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
__device__ inline int bits(uint64_t mask) { return __popcll((unsigned long long)mask); }

// ---- up to 1024 tokens: one wave a row ------------------------------------------------------
// A row of logits is in registers before anything else happens; what follows are dependent steps on it
// (weights, their sum, the cut bit by bit with a ballot each, running sums).  260 tokens with top_k, top_p and
// min_p: one row 7.4 us, of which a launch is 3; 4096 rows 15.6 us (4.3 MB, so 0.27 TB/s: vector units
// 50 % busy, the rest the chains of one wave).  N = 5 for up to 320: a byte's vocabulary with its special tokens.
template <typename T, int N>
__global__ __launch_bounds__(256) void sample_wave_kernel(SArgs g) {
  __shared__ Powers pw;
  fill(pw);
  __syncthreads();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= g.rows) return;
  const int lane = threadIdx.x & 63;
  const char* x = (const char*)g.x + row * g.st * (int64_t)sizeof(T);
  float v[N];
  uint32_t key[N];
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    v[j] = lane + 64 * j < g.V ? logit<T>(x, lane + 64 * j) : -INFINITY;
    nan |= v[j] != v[j];
    key[j] = lane + 64 * j < g.V ? key_of(v[j]) : 0;  // (a logit's is never 0)
    top = fmaxf(top, v[j]);
  }
  top = wave_max(top);
  const Rules r = rules_of(g, row);
  if (__any(nan) || top == -INFINITY || !r.good) {
    if (lane == 0) g.out[row] = -1;
    return;
  }
  uint64_t w[N];
#pragma unroll
  for (int j = 0; j < N; ++j) w[j] = weight(v[j], top, r, g.scale, pw);
  auto count = [&](uint32_t c) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += bits(__ballot(key[j] >= c));
    return n;
  };
  auto mass = [&](uint32_t c) {
    uint64_t m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m += key[j] >= c ? w[j] : 0;
    return sum_u64(m);
  };
  // The largest c whose tokens of key >= c are enough, as far as it matters: down to one
  // token or one key between lo (enough) and hi (not); `over` tokens at or above hi.
  uint32_t lo = 1;
  int at = g.V;            // tokens of key >= lo
  int ties = 0x7fffffff;   // kept ones of the smallest key >= lo
  if (r.k) {
    uint32_t hi = key_of(top) + 1;
    int over = 0;
    while (hi - lo > 1 && at - over > 1 && at != r.k) {
      const uint32_t mid = lo + ((hi - lo) >> 1);
      const int n = count(mid);
      if (n >= r.k) {
        lo = mid;
        at = n;
      } else {
        hi = mid;
        over = n;
      }
    }
    if (at != r.k) ties = r.k - over;  // (of at - over with the one key that is left)
  }
  if (r.p < 1.) {
    uint64_t sum = mass(lo);
    if (ties < 0x7fffffff) {
      const uint64_t above = mass(lo + 1);
      sum = above + (sum - above) / (uint64_t)(at - (r.k - ties)) * (uint64_t)ties;
    }
    const uint64_t want = wanted(r.p, sum);
    const uint32_t first = lo;
    uint32_t hi = key_of(top) + 1;
    int over = 0;
    uint64_t above = 0;
    while (hi - lo > 1 && at - over > 1) {
      const uint32_t mid = lo + ((hi - lo) >> 1);
      const uint64_t m = mass(mid);
      if (m >= want) {
        lo = mid;
        at = count(mid);
      } else {
        hi = mid;
        over = count(mid);
        above = m;
      }
    }
    // one key is left; its tokens' weight is not 0, for with them the sum reaches `want`
    const uint64_t each = (mass(lo) - above) / (uint64_t)(at - over);
    const uint64_t need = (want - above + each - 1) / each;
    const int n = need < (uint64_t)(at - over) ? (int)need : at - over;
    ties = lo == first ? min(ties, n) : n;
  }
  // kept weights, the ties in the order of their indices
  uint64_t total = 0;
  {
    uint32_t tie = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < N; ++j) tie = key[j] >= lo ? min(tie, key[j]) : tie;
    tie = wave_min_u32(tie);
    int before = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint64_t here = __ballot(key[j] == tie);
      const bool in = key[j] > tie || (key[j] == tie && before + below(here) < ties);
      w[j] = in && w[j] >= r.m ? w[j] : 0;
      before += bits(here);
      total += w[j];
    }
  }
  total = sum_u64(total);
  const uint64_t aim = aim_of(g.u[row], total);
  uint64_t run = 0;
  int token = -1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint64_t s = incl_scan_u64(w[j]);
    const uint64_t hit = __ballot(run + s > aim);
    if (token < 0 && hit) token = 64 * j + __ffsll((unsigned long long)hit) - 1;
    run += lane_u64(s, 63);
  }
  if (lane == 0) g.out[row] = token;
}

// ---- blocks of 1024 threads ------------------------------------------------------------------
constexpr int NT = 1024, NW = NT / 64;
constexpr int PART = 16 * NT;  // tokens that a block holds in registers

// Tokens [0, n) of a row in the registers of a block, or in memory; wave w has a run of them, so
// that the waves' runs, and the groups of 64 within one, follow each other. each(f) calls
// f(x, index, j) in that order in all lanes, with index < 0 where there is no token; j counts
// the calls.
template <typename T, int N>
struct Held {
  float x[N];
  int first, n;
  __device__ inline Held(const void* row, int64_t from, int n_) : n(n_) {
    first = (int)(threadIdx.x >> 6) * 64 * N + (int)(threadIdx.x & 63);
#pragma unroll
    for (int j = 0; j < N; ++j)
      x[j] = first + 64 * j < n ? logit<T>(row, from + first + 64 * j) : -INFINITY;
  }
  template <typename F>
  __device__ inline void each(F f) const {
#pragma unroll
    for (int j = 0; j < N; ++j) f(x[j], first + 64 * j < n ? first + 64 * j : -1, j);
  }
};
struct InLds {
  const float* x;
  int n, run;
  __device__ inline InLds(const float* x_, int n_) : x(x_), n(n_) {
    run = ((n + NW - 1) / NW + 63) & ~63;
  }
  template <typename F>
  __device__ inline void each(F f) const {
    const int a = (int)(threadIdx.x >> 6) * run, lane = threadIdx.x & 63;
#pragma unroll 2
    for (int j = 0; j < run; j += 64) {
      const int i = a + j + lane;
      f(i < n ? x[i] : -INFINITY, i < n ? i : -1, j / 64);
    }
  }
};
template <typename T>
struct InMemory {
  const void* row;
  int n, run;
  __device__ inline InMemory(const void* row_, int n_) : row(row_), n(n_) {
    run = ((n + NW - 1) / NW + 63) & ~63;
  }
  template <typename F>
  __device__ inline void each(F f) const {
    const int a = (int)(threadIdx.x >> 6) * run, lane = threadIdx.x & 63;
#pragma unroll 2
    for (int j = 0; j < run; j += 64) {  // (longer unrolled the kernels' code takes longer to fetch)
      const int i = a + j + lane;
      f(i < n ? logit<T>(row, i) : -INFINITY, i < n ? i : -1, j / 64);
    }
  }
};

constexpr int FEW = 64;
struct Room {
  uint64_t m[NB];  // bins: sum of weights and tokens
  uint32_t c[NB];
  uint64_t lc[FEW], lw[FEW];  // a bin's tokens, when they are few
  uint64_t wm[NW];            // of the waves
  uint32_t wc[NW], wx[NW];
  int n;
  uint64_t code, sum;
  // a bin, and what lies above it
  int bin, bin0;
  uint32_t above_c, in_c;
  uint64_t above_m;
  Powers pw;
};
__device__ inline void zero_bins(Room& s) {
  for (int i = threadIdx.x; i < NB; i += NT) {
    s.m[i] = 0;
    s.c[i] = 0;
  }
}
__device__ inline void add_to_bin(Room& s, int b, uint64_t w, bool count = true) {
  if (count) atomicAdd(&s.c[b], 1u);
  if (w) atomicAdd((unsigned long long*)&s.m[b], (unsigned long long)w);
}
// Two bins of a thread and what lies above them.
struct Bins {
  uint32_t c[2], above_c;
  uint64_t m[2], above_m;
  uint64_t total_m;
};
// of the bins in s, complete; a barrier before and two within
__device__ inline Bins scan_bins(Room& s) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  Bins b;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    b.c[q] = s.c[2 * tid + q];
    b.m[q] = s.m[2 * tid + q];
  }
  const uint32_t ic = (uint32_t)wave_incl_scan((int)(b.c[0] + b.c[1]));
  const uint64_t im = incl_scan_u64(b.m[0] + b.m[1]);
  if (lane == 63) {
    s.wc[w] = ic;
    s.wm[w] = im;
  }
  __syncthreads();
  b.above_c = ic - b.c[0] - b.c[1];
  b.above_m = im - b.m[0] - b.m[1];
  b.total_m = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (i < w) {
      b.above_c += s.wc[i];
      b.above_m += s.wm[i];
    }
    b.total_m += s.wm[i];
  }
  __syncthreads();
  return b;
}
// The bin where the running count (or sum) reaches `want`, into s.
__device__ inline void locate(Room& s, const Bins& b, bool by_count, uint64_t want) {
  uint32_t c = b.above_c;
  uint64_t m = b.above_m;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint64_t at = by_count ? c : m, here = by_count ? b.c[q] : b.m[q];
    if (at < want && want <= at + here) {
      s.bin = 2 * (int)threadIdx.x + q;
      s.above_c = c;
      s.above_m = m;
      s.in_c = b.c[q];
    }
    c += b.c[q];
    m += b.m[q];
  }
  __syncthreads();
}
// Tokens have a code, an integer of their own whose order is that of the selection:
// their rank's (logits descending, then indices ascending) or their index.
__device__ inline uint64_t rank_code(float x, int i) {
  return (uint64_t)~key_of(x) << 32 | (uint32_t)i;
}
__device__ inline Cut cut_of(uint64_t code) {
  return Cut{~(uint32_t)(code >> 32), (int)(uint32_t)code};
}
// The code at which the running count (or sum of weights) of the tokens that code_of takes
// (it gives false for others) reaches `want`, in the order of the codes, and that sum.  s.in_c: how many they
// are, at most (with in_c above FEW any number); s.above_c, s.above_m: what counts as before
// them.  More than a few are put into bins over the bits of their codes, until there are
// few in one; those find their own places.
template <typename Row, typename Code>
__device__ uint64_t select(const Row& row, Room& s, Code code_of, bool by_count, uint64_t want,
                           uint64_t& sum) {
  const int tid = threadIdx.x;
  uint64_t lo = 0, hi = ~(uint64_t)0;
  for (bool first = true;; first = false) {
    const uint32_t n = s.in_c, above_c = s.above_c;
    const uint64_t above_m = s.above_m;
    if (n <= FEW) {
      if (tid == 0) s.n = 0;
      __syncthreads();
      row.each([&](float x, int i, int) {
        uint64_t c, w;
        if (i >= 0 && code_of(x, i, c, w) && c >= lo && c <= hi) {
          const int at = atomicAdd(&s.n, 1);
          s.lc[at] = c;
          s.lw[at] = w;
        }
      });
      __syncthreads();
      const int m = s.n;
      if (tid < m) {
        const uint64_t c = s.lc[tid], w = s.lw[tid];
        uint32_t rank = above_c;
        uint64_t before = above_m;
        for (int j = 0; j < m; ++j) {
          const bool better = s.lc[j] < c;
          rank += better ? 1 : 0;
          before += better ? s.lw[j] : 0;
        }
        if (by_count ? rank + 1 == (uint32_t)want : before < want && want <= before + w) {
          s.code = c;
          s.sum = before + w;
        }
      }
      __syncthreads();
      const uint64_t c = s.code;
      sum = s.sum;
      __syncthreads();
      return c;
    }
    if (first) {  // the range of their upper halves, and of the lower ones if those are equal
      uint32_t a = 0xffffffffu, b = 0, a0 = 0xffffffffu, b0 = 0;
      row.each([&](float x, int i, int) {
        uint64_t c, w;
        if (i >= 0 && code_of(x, i, c, w)) {
          a = min(a, (uint32_t)(c >> 32));
          b = max(b, (uint32_t)(c >> 32));
          a0 = min(a0, (uint32_t)c);
          b0 = max(b0, (uint32_t)c);
        }
      });
      if (tid == 0) {
        s.wc[0] = s.wx[0] = 0xffffffffu;
        s.wc[1] = s.wx[1] = 0;
      }
      a = wave_min_u32(a);
      b = wave_max_u32(b);
      a0 = wave_min_u32(a0);
      b0 = wave_max_u32(b0);
      __syncthreads();
      if ((tid & 63) == 0) {
        atomicMin(&s.wc[0], a);
        atomicMax(&s.wc[1], b);
        atomicMin(&s.wx[0], a0);
        atomicMax(&s.wx[1], b0);
      }
      __syncthreads();
      const bool one = s.wc[0] == s.wc[1];
      lo = (uint64_t)s.wc[0] << 32 | (one ? s.wx[0] : 0);
      hi = (uint64_t)s.wc[1] << 32 | (one ? s.wx[1] : 0xffffffffu);
      __syncthreads();
    }
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
    zero_bins(s);
    __syncthreads();
    row.each([&](float x, int i, int) {
      uint64_t c, w;
      if (i >= 0 && code_of(x, i, c, w) && c >= lo && c <= hi) add_to_bin(s, (int)((c - lo) >> shift), w);
    });
    __syncthreads();
    const Bins b = scan_bins(s);
    locate(s, b, by_count, want - (by_count ? above_c : above_m));
    lo += (uint64_t)s.bin << shift;
    hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
    __syncthreads();
    if (tid == 0) {
      s.above_c += above_c;
      s.above_m += above_m;
    }
    __syncthreads();
  }
}
// The cut of a row whose bins are in s.
template <typename Row>
__device__ Cut find_cut(const Row& row, Room& s, const Rules& r, float top, int scale) {
  Cut c{0, 0x7fffffff};
  if (!r.k && !(r.p < 1.)) return c;
  const Bins b = scan_bins(s);
  uint64_t sum = b.total_m, unused;
  auto in_bin = [&](float x, int i, uint64_t& code, uint64_t& w) {
    if (bin_of(x, top, r) != s.bin0) return false;
    code = rank_code(x, i);
    w = weight(x, top, r, scale, s.pw);
    return true;
  };
  auto end_of = [&](bool by_count, uint64_t want, uint64_t& upto) {
    locate(s, b, by_count, want);
    if (threadIdx.x == 0) s.bin0 = s.bin;
    __syncthreads();
    return cut_of(select(row, s, in_bin, by_count, want, upto));
  };
  if (r.k) c = end_of(true, (uint64_t)r.k, sum);
  if (r.p < 1.) c = end_of(false, wanted(r.p, sum), unused);
  return c;
}
// The token: the first whose running sum of kept weights is above u times their sum.
template <typename Row>
__device__ int draw(const Row& row, Room& s, const Rules& r, float top, int scale, const Cut& cut,
                    float u) {
  const int wid = threadIdx.x >> 6;
  auto mass = [&](float x, int i) {
    const uint64_t w = i >= 0 && kept(cut, key_of(x), i) ? weight(x, top, r, scale, s.pw) : 0;
    return w >= r.m ? w : 0;
  };
  uint64_t mine = 0;
  row.each([&](float x, int i, int) { mine += mass(x, i); });
  mine = sum_u64(mine);
  if ((threadIdx.x & 63) == 0) s.wm[wid] = mine;
  if (threadIdx.x == 0) s.n = -1;
  __syncthreads();
  uint64_t run = 0, total = 0;
  for (int i = 0; i < NW; ++i) {
    run += i < wid ? s.wm[i] : 0;
    total += s.wm[i];
  }
  const uint64_t aim = aim_of(u, total);
  if (run <= aim && aim < run + mine) {  // (one wave's run)
    int token = -1;
    row.each([&](float x, int i, int) {
      const uint64_t at = incl_scan_u64(mass(x, i));
      const uint64_t hit = __ballot(run + at > aim);
      if (token < 0 && hit) token = __builtin_amdgcn_readlane(i, __ffsll((unsigned long long)hit) - 1);
      run += lane_u64(at, 63);
    });
    if ((threadIdx.x & 63) == 0) s.n = token;
  }
  __syncthreads();
  return s.n;
}
// The same for up to PART tokens of a row, the thread's ones beside each other, where the
// sum is known: the first above `aim`.
template <typename T>
__device__ int draw_part(const void* row, int64_t from, int n, Room& s, const Rules& r, float top,
                         int scale, const Cut& cut, uint64_t aim) {
  constexpr int E = PART / NT;
  const int tid = threadIdx.x, lane = tid & 63, i0 = tid * E;
  auto mass = [&](float x, int i) {
    const uint64_t w = i < n && kept(cut, key_of(x), i) ? weight(x, top, r, scale, s.pw) : 0;
    return w >= r.m ? w : 0;
  };
  uint64_t mine = 0;
  float x[E];
#pragma unroll
  for (int j = 0; j < E; ++j) x[j] = i0 + j < n ? logit<T>(row, from + i0 + j) : -INFINITY;
#pragma unroll
  for (int j = 0; j < E; ++j) mine += mass(x[j], i0 + j);
  const uint64_t at = incl_scan_u64(mine);
  if (lane == 63) s.wm[tid >> 6] = at;
  __syncthreads();
  uint64_t run = at - mine;
  for (int i = 0; i < (tid >> 6); ++i) run += s.wm[i];
  const uint64_t here = __ballot(run <= aim && aim < run + mine);
  if (here) {  // one thread's tokens: one each for lanes of its wave
    const int l = __ffsll((unsigned long long)here) - 1, i = __builtin_amdgcn_readlane(i0, l) + lane;
    const bool has = lane < E && i < n;
    const uint64_t w = has ? mass(logit<T>(row, from + i), i) : 0;
    const uint64_t hit = __ballot(has && lane_u64(run, l) + incl_scan_u64(w) > aim);
    if (lane == 0) s.n = i + __ffsll((unsigned long long)hit) - 1;
  }
  __syncthreads();
  return s.n;
}
// the largest over a block; NaN where one is
__device__ inline float block_top(Room& s, float x, bool nan) {
  x = wave_max(x);
  if (__any(nan)) x = NAN;
  if ((threadIdx.x & 63) == 0) s.wc[threadIdx.x >> 6] = __float_as_uint(x);
  __syncthreads();
  float top = -INFINITY;
  bool bad = false;
  for (int i = 0; i < NW; ++i) {
    const float y = __uint_as_float(s.wc[i]);
    bad |= y != y;
    top = fmaxf(top, y);
  }
  __syncthreads();
  return bad ? NAN : top;
}

// ---- up to 16384 tokens: one block a row -------------------------------------------------------
// The row is kept in LDS (in registers it spilled), weights are made where they are counted.  64 rows with
// top_p: of 1025 logits 10.5 us, of 4096 14, of 16384 31 (one row 30; with top_k 50 26): one row's chain of
// counts and scans; 1024 rows of 16384 120 us, 67 MB, four rounds of one block a CU (92 KB of LDS).
template <typename T>
__global__ __launch_bounds__(NT) void sample_block_kernel(SArgs g) {
  __shared__ Room s;
  __shared__ float held[PART];
  const int64_t row = blockIdx.x;
  fill(s.pw);
  float m = -INFINITY;
  bool nan = false;
  {
    const char* from = (const char*)g.x + row * g.st * (int64_t)sizeof(T);
    float v[PART / NT];
#pragma unroll
    for (int j = 0; j < PART / NT; ++j) {
      const int i = (int)threadIdx.x + NT * j;
      v[j] = i < g.V ? logit<T>(from, i) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < PART / NT; ++j) {
      if ((int)threadIdx.x + NT * j < g.V) held[threadIdx.x + NT * j] = v[j];
      m = fmaxf(m, v[j]);
      nan |= v[j] != v[j];
    }
  }
  const float top = block_top(s, m, nan);
  const Rules r = rules_of(g, row);
  if (!(top > -INFINITY) || !r.good) {
    if (threadIdx.x == 0) g.out[row] = -1;
    return;
  }
  const InLds x(held, g.V);
  if (r.k || r.p < 1.) {
    zero_bins(s);
    __syncthreads();
    x.each([&](float v, int i, int) {
      if (i >= 0) add_to_bin(s, bin_of(v, top, r), r.p < 1. ? weight(v, top, r, g.scale, s.pw) : 0);
    });
    __syncthreads();
  }
  const Cut cut = find_cut(x, s, r, top, g.scale);
  const int token = draw(x, s, r, top, g.scale, cut, g.u[row]);
  if (threadIdx.x == 0) g.out[row] = token;
}

// ---- more: parts of rows ------------------------------------------------------------------------
// The launches: every part's largest logit; the bins of every part; for every row the bins in
// which its rules end, from their sums; of every part the tokens that decide (listed) and the
// weights that are kept whatever they decide; for every row the token.  What is listed:
//   with top_k     all tokens down to the bin in which it ends: they decide everything
//   with top_p     those of the bin in which it ends; what lies above is kept
// Where that are more than a block ranks at once, the cut is found by passes over the row.
// 64 rows of 131072 f32 logits with top_p, 33.5 MB, which the last-level cache holds after the first
// launch: 60 us, of which top 4.5 (7.4 TB/s), bins 17 (vector units 52 % busy with weights in 64 bits and
// LDS atomics), find 7, lists and kept weights 11, pick 19 (64 blocks, chains of scans; a launch's
// start is in each).  Three reads of the row and five launches take 34 us at those rates; one launch
// a row (the form above, in passes) 123.  With top_k 50 as well 47: bins by
// counts alone (with weights 9 more), lists from registers (in passes over memory 9 more).  With
// top_k 4000, beyond a list, 155, of which find 101, and with top_p too 268 and 217: one block walks all of its
// row several times.
enum Way { ALL, TOP, BIN, CUT };  // (no rule but min_p; lists; a cut that is known)
struct Found {
  int way, bin;
  uint32_t above_c, key;
  int index;
  uint32_t pad;
  uint64_t above_m, want;  // want: of top_p
};
struct Entry {
  float x;
  int index;
  uint64_t w;
};
__device__ inline float row_top(const SArgs& g, int64_t row) {
  float m = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x & 63; i < g.parts; i += 64) {
    const float x = g.pmax[row * g.parts + i];
    m = fmaxf(m, x);
    nan |= x != x;
  }
  m = wave_max(m);
  return __any(nan) ? NAN : m;
}
template <typename T>
__device__ inline Held<T, 16> part_of(const SArgs& g, int64_t row, int part) {
  return Held<T, 16>((const char*)g.x + row * g.st * (int64_t)sizeof(T), (int64_t)part * PART,
                     min(PART, g.V - part * PART));
}
template <typename T>
__global__ __launch_bounds__(NT) void sample_top_kernel(SArgs g) {
  __shared__ Room s;
  const int64_t row = blockIdx.x / g.parts;
  const int part = (int)(blockIdx.x - row * g.parts);
  const Held<T, 16> x = part_of<T>(g, row, part);
  float m = -INFINITY;
  bool nan = false;
  x.each([&](float v, int, int) {
    m = fmaxf(m, v);
    nan |= v != v;
  });
  const float top = block_top(s, m, nan);
  if (threadIdx.x == 0) g.pmax[row * g.parts + part] = top;
}
template <typename T>
__global__ __launch_bounds__(NT) void sample_bins_kernel(SArgs g) {
  __shared__ Room s;
  const int64_t row = blockIdx.x / g.parts;
  const int part = (int)(blockIdx.x - row * g.parts);
  const Held<T, 16> x = part_of<T>(g, row, part);
  const float top = row_top(g, row);
  const Rules r = rules_of(g, row);
  if (!(top > -INFINITY) || !r.good || (!r.k && !(r.p < 1.))) return;
  fill(s.pw);
  zero_bins(s);
  __syncthreads();
  x.each([&](float v, int i, int) {
    if (i >= 0)
      add_to_bin(s, bin_of(v, top, r), r.k ? 0 : weight(v, top, r, g.scale, s.pw), r.k > 0);
  });
  __syncthreads();
  const int64_t at = (row * g.parts + part) * NB;
  for (int i = threadIdx.x; i < NB; i += NT) {
    // (where top_k ends goes by counts; the weights of its tokens are taken from the list)
    if (r.k) g.hc[at + i] = s.c[i];
    else g.hm[at + i] = s.m[i];
  }
}
template <typename T>
__global__ __launch_bounds__(NT) void sample_find_kernel(SArgs g) {
  __shared__ Room s;
  const int64_t row = blockIdx.x;
  const float top = row_top(g, row);
  const Rules r = rules_of(g, row);
  if (!(top > -INFINITY) || !r.good) return;
  Found f{};
  f.way = ALL;
  if (r.k || r.p < 1.) {
    uint64_t m[2] = {0, 0};
    uint32_t c[2] = {0, 0};
    for (int part = 0; part < g.parts; ++part) {
      const int64_t at = (row * g.parts + part) * NB + 2 * threadIdx.x;
      if (r.k) {
        c[0] += g.hc[at];
        c[1] += g.hc[at + 1];
      } else {
        m[0] += g.hm[at];
        m[1] += g.hm[at + 1];
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      s.m[2 * threadIdx.x + q] = m[q];
      s.c[2 * threadIdx.x + q] = c[q];
    }
    __syncthreads();
    const Bins b = scan_bins(s);
    if (r.k) {
      locate(s, b, true, (uint64_t)r.k);
      f.way = s.above_c + s.in_c <= NT ? TOP : CUT;
      f.bin = s.bin;
    } else {
      f.want = wanted(r.p, b.total_m);
      locate(s, b, false, f.want);
      f.way = BIN;
      f.bin = s.bin;
      f.above_m = s.above_m;
    }
    if (f.way == CUT) {  // (top_k beyond a list)
      const InMemory<T> x((const char*)g.x + row * g.st * (int64_t)sizeof(T), g.V);
      fill(s.pw);
      __syncthreads();
      if (r.p < 1.) {  // (the bins have no weights yet)
        x.each([&](float v, int i, int) {
          if (i >= 0) add_to_bin(s, bin_of(v, top, r), weight(v, top, r, g.scale, s.pw), false);
        });
        __syncthreads();
      }
      const Cut cut = find_cut(x, s, r, top, g.scale);
      f.key = cut.key;
      f.index = cut.index;
    }
  }
  if (threadIdx.x == 0) g.found[row] = f;
}
// weights kept of a part, and its list
template <typename T>
__global__ __launch_bounds__(NT) void sample_part_kernel(SArgs g) {
  __shared__ uint64_t wm[NW];
  __shared__ int listed;
  __shared__ Powers pw;
  const int64_t row = blockIdx.x / g.parts;
  const int part = (int)(blockIdx.x - row * g.parts);
  const Held<T, 16> x = part_of<T>(g, row, part);
  const float top = row_top(g, row);
  const Rules r = rules_of(g, row);
  if (!(top > -INFINITY) || !r.good) return;
  const Found f = g.found[row];
  if (threadIdx.x == 0) listed = 0;
  fill(pw);
  __syncthreads();
  const Cut cut{f.key, f.index - part * PART};
  Entry* list = g.list + (row * g.parts + part) * NT;
  uint64_t m = 0;
  // (without min_p the weights above the bin are those of the part's bins)
  const bool sums = f.way == BIN && r.m == 0;
  if (sums) {
    const uint64_t* bins = g.hm + (row * g.parts + part) * NB;
    for (int i = threadIdx.x; i < f.bin; i += NT) m += bins[i];
  }
  auto enter = [&](float v, int i) {
    const int at = atomicAdd(&listed, 1);
    if (at < NT) list[at] = Entry{v, part * PART + i, weight(v, top, r, g.scale, pw)};
  };
  if (sums || f.way == TOP) {
    const float end = (float)f.bin + 1.f, from = f.way == TOP ? -INFINITY : (float)f.bin;
    uint32_t hits = 0;
    x.each([&](float v, int i, int j) {
      const float t = place_of(v, top, r);
      hits |= t >= from && t < end && i >= 0 ? 1u << j : 0;
    });
    while (hits) {
      const int i = x.first + 64 * (__ffs((int)hits) - 1);
      hits &= hits - 1;
      enter(logit<T>((const char*)g.x + row * g.st * (int64_t)sizeof(T), (int64_t)part * PART + i), i);
    }
  } else {
    const InMemory<T> again((const char*)g.x + (row * g.st + (int64_t)part * PART) * (int64_t)sizeof(T),
                            x.n);
    again.each([&](float v, int i, int) {
      if (i < 0) return;
      const int bin = f.way == BIN ? bin_of(v, top, r) : 0;
      const bool keep = f.way == ALL || (f.way == CUT && kept(cut, key_of(v), i)) ||
                        (f.way == BIN && bin < f.bin);
      if (keep) {
        const uint64_t w = weight(v, top, r, g.scale, pw);
        m += w >= r.m ? w : 0;
      }
      if (f.way == BIN && bin == f.bin) enter(v, i);
    });
  }
  m = sum_u64(m);
  if ((threadIdx.x & 63) == 0) wm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint64_t all = 0;
    for (int i = 0; i < NW; ++i) all += wm[i];
    g.pmass[row * g.parts + part] = all;
    g.count[row * g.parts + part] = listed;
  }
}
// the lists' tokens, one each in a thread's registers
struct Listed {
  float x;
  int index;  // -1: none
  template <typename F>
  __device__ inline void each(F f) const { f(x, index, 0); }
};
template <typename T>
__global__ __launch_bounds__(NT) void sample_pick_kernel(SArgs g) {
  __shared__ Room s;
  __shared__ uint64_t extra[64];  // kept weights of the bin, by parts
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  // (everything whose address is known is on its way at once; of a row without a token it is
  // whatever lies there)
  const Found f = g.found[row];
  const int n_of = lane < g.parts ? g.count[row * g.parts + lane] : 0;
  const uint64_t above = lane < g.parts ? g.pmass[row * g.parts + lane] : 0;
  const float top = row_top(g, row);
  const Rules r = rules_of(g, row);
  if (!(top > -INFINITY) || !r.good) {
    if (threadIdx.x == 0) g.out[row] = -1;
    return;
  }
  Cut cut{f.key, f.way == ALL ? 0x7fffffff : f.index};
  fill(s.pw);
  if (tid < 64) extra[tid] = 0;
  if (f.way == TOP || f.way == BIN) {
    // the parts' lists one behind the other (parts <= 64: 2^20 tokens)
    const bool over = __any(n_of > NT);
    const int upto = wave_incl_scan(min(n_of, NT)), n = __builtin_amdgcn_readlane(upto, 63);
    if (tid == 0) {
      s.above_c = 0;
      s.above_m = f.way == BIN ? f.above_m : 0;
      s.in_c = over ? 0xffffffffu : (uint32_t)n;
    }
    __syncthreads();
    uint64_t sum;
    if (over || n > NT) {  // (top_p's bin beyond a list)
      const InMemory<T> x((const char*)g.x + row * g.st * (int64_t)sizeof(T), g.V);
      auto in_bin = [&](float v, int i, uint64_t& c, uint64_t& w) {
        if (bin_of(v, top, r) != f.bin) return false;
        c = rank_code(v, i);
        w = weight(v, top, r, g.scale, s.pw);
        return true;
      };
      cut = cut_of(select(x, s, in_bin, false, f.want, sum));
      x.each([&](float v, int i, int) {
        if (i < 0 || bin_of(v, top, r) != f.bin || !kept(cut, key_of(v), i)) return;
        const uint64_t w = weight(v, top, r, g.scale, s.pw);
        if (w >= r.m) atomicAdd((unsigned long long*)&extra[i / PART], (unsigned long long)w);
      });
    } else {
      int part = 0, before_part = 0;
      for (int i = 0; i < g.parts; ++i) {
        const int end = __builtin_amdgcn_readlane(upto, i);
        part += end <= tid ? 1 : 0;
        before_part = end <= tid ? end : before_part;
      }
      Entry e{0.f, -1, 0};
      if (tid < n) e = g.list[(row * g.parts + part) * NT + tid - before_part];
      const Listed x{e.x, e.index};
      // the selections of the list, one after the other: where top_k ends, where top_p ends,
      // and of a list of all that is kept the token
      enum { BY_K, BY_P, TOKEN };
      uint64_t want = f.way == TOP ? (uint64_t)r.k : f.want;
      bool in = true;
      int stage = f.way == TOP ? BY_K : BY_P;
      for (;;) {
        const uint64_t code =
            select(x, s,
                   [&](float v, int i, uint64_t& c, uint64_t& w) {
                     c = stage == TOKEN ? (uint32_t)i : rank_code(v, i);
                     w = e.w;
                     return in;
                   },
                   stage == BY_K, want, sum);
        if (stage == TOKEN) {
          if (tid == 0) g.out[row] = (int)code;
          return;
        }
        cut = cut_of(code);
        if (stage == BY_K && r.p < 1.) {
          stage = BY_P;
          want = wanted(r.p, sum);
        } else {
          in = e.index >= 0 && kept(cut, key_of(e.x), e.index) && e.w >= r.m;
          if (f.way == BIN) break;
          stage = TOKEN;
          sum = sum_u64(in ? e.w : 0);
          if (lane == 0) s.wm[tid >> 6] = sum;
          __syncthreads();
          sum = 0;
          for (int i = 0; i < NW; ++i) sum += s.wm[i];
          want = aim_of(g.u[row], sum) + 1;
        }
        if (tid == 0) {
          s.above_c = 0;
          s.above_m = 0;
          s.in_c = (uint32_t)n;
        }
        __syncthreads();
      }
      if (in) atomicAdd((unsigned long long*)&extra[e.index / PART], (unsigned long long)e.w);
    }
  }
  __syncthreads();
  const uint64_t m = above + extra[lane];
  const uint64_t at = incl_scan_u64(m);
  const uint64_t aim = aim_of(g.u[row], lane_u64(at, 63));
  const uint64_t hit = __ballot(at > aim);
  const int part = __ffsll((unsigned long long)hit) - 1;
  const uint64_t before = lane_u64(at - m, part);
  const int token = draw_part<T>((const char*)g.x + row * g.st * (int64_t)sizeof(T),
                                 (int64_t)part * PART, min(PART, g.V - part * PART), s, r, top,
                                 g.scale, Cut{cut.key, cut.index - part * PART}, aim - before);
  if (tid == 0) g.out[row] = part * PART + token;
}

int parts_of(int vocab) { return vocab <= PART ? 0 : (vocab + PART - 1) / PART; }

template <typename T>
int run(const SArgs& g, hipStream_t s) {
  if (g.V <= 1024) {
    const dim3 grid(ceil_div(g.rows, 4)), block(256);
    if (g.V <= 64)
      hipLaunchKernelGGL((sample_wave_kernel<T, 1>), grid, block, 0, s, g);
    else if (g.V <= 128)
      hipLaunchKernelGGL((sample_wave_kernel<T, 2>), grid, block, 0, s, g);
    else if (g.V <= 320)
      hipLaunchKernelGGL((sample_wave_kernel<T, 5>), grid, block, 0, s, g);
    else if (g.V <= 512)
      hipLaunchKernelGGL((sample_wave_kernel<T, 8>), grid, block, 0, s, g);
    else
      hipLaunchKernelGGL((sample_wave_kernel<T, 16>), grid, block, 0, s, g);
  } else if (g.V <= PART) {
    hipLaunchKernelGGL((sample_block_kernel<T>), dim3((unsigned)g.rows), dim3(NT), 0, s, g);
  } else {
    const dim3 all((unsigned)(g.rows * g.parts)), one((unsigned)g.rows), block(NT);
    hipLaunchKernelGGL((sample_top_kernel<T>), all, block, 0, s, g);
    // (without top_k and top_p for any row there is nothing to find)
    if (g.s.top_ks || g.s.top_ps || g.s.temperatures || g.s.temperature == 0. || g.s.top_k > 0 ||
        g.s.top_p < 1.)
      hipLaunchKernelGGL((sample_bins_kernel<T>), all, block, 0, s, g);
    hipLaunchKernelGGL((sample_find_kernel<T>), one, block, 0, s, g);
    hipLaunchKernelGGL((sample_part_kernel<T>), all, block, 0, s, g);
    hipLaunchKernelGGL((sample_pick_kernel<T>), one, block, 0, s, g);
  }
  BLT_LAUNCH_CHECK("sample");
  return 0;
}

}  // namespace

// Rows of one round of launches: where they are in parts, 8192 of these fill the chip four times, and
// what they leave behind (41 KB each) stays below 340 MB; else 2^31 work-items (a launch takes less than
// 2^32), a wave a row or a block.
static int64_t rows_at_once(int64_t rows, int vocab) {
  const int64_t parts = parts_of(vocab);
  return std::min<int64_t>(rows, parts ? 8192 / parts : vocab <= 1024 ? 1 << 25 : 1 << 21);
}
int64_t sample_workspace_bytes(int64_t rows, int vocab) {
  const int64_t parts = parts_of(vocab);
  rows = rows_at_once(rows, vocab);
  return parts ? rows * (parts * (12 * (int64_t)NB + sizeof(Entry) * NT + 16) + sizeof(Found)) : 0;
}

int launch_sample(const SampleArgs& a, void* ws, hipStream_t s) {
  SArgs g{};
  g.st = a.row_stride; g.V = a.vocab; g.s = a.set;
  int l = 0;
  while (((int64_t)1 << l) < a.vocab) ++l;
  g.scale = 62 - l;
  g.parts = parts_of(a.vocab);
  if (a.rows > 0x7fffffff) return fail(BLT_ERR_SHAPE, "fused_sample: too many rows");
  const int64_t each = rows_at_once(a.rows, a.vocab), n = each * g.parts;
  if (g.parts) {
    g.hm = (uint64_t*)ws;
    g.pmass = g.hm + n * NB;
    g.list = (Entry*)(g.pmass + n);
    g.found = (Found*)(g.list + n * NT);
    g.hc = (uint32_t*)(g.found + each);
    g.pmax = (float*)(g.hc + n * NB);
    g.count = (int*)(g.pmax + n);
  }
  const bool bf16 = a.dtype == BLT_DTYPE_BF16;
  for (int64_t row = 0; row < a.rows; row += each) {
    g.rows = std::min(each, a.rows - row);
    g.x = (const char*)a.logits + row * a.row_stride * (bf16 ? 2 : 4);
    g.u = a.uniform + row;
    g.out = a.out + row;
    if (a.set.temperatures) g.s.temperatures = a.set.temperatures + row;
    if (a.set.top_ps) g.s.top_ps = a.set.top_ps + row;
    if (a.set.min_ps) g.s.min_ps = a.set.min_ps + row;
    if (a.set.top_ks) g.s.top_ks = a.set.top_ks + row;
    if (int rc = bf16 ? run<uint16_t>(g, s) : run<float>(g, s)) return rc;
  }
  return 0;
}

}  // namespace blt
