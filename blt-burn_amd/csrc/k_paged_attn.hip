// Attention of a chunk of new tokens per sequence over the paged cache: one pass
// over the keys with a running max and sum, head_dim 64 or 128, grouped heads, any
// chunk length from one token up.
//
// Rows and items.  The query heads that share a key head are packed with the tokens
// into rows (row = token * G + head), so one key tile serves all of them and a
// single token with grouped heads still fills matrix rows.  An item is a row tile of
// one (sequence, key head) and, where the call has too few of them to fill the chip, a
// part of its keys; the part that ends last joins the parts' unnormalised outputs (join_parts).  Lengths
// live on the device (the call can be captured and replayed as they grow), so every wave
// works out its item itself: the number of key tiles an item may have (C) follows from
// the total work, then a scan over the sequences finds the item of a block.  The host
// only bounds the grid: items <= row tiles + the blocks that are to be filled (2 * resident,
// where find_item spills 4 * resident), parts in need of joining <= twice those blocks (every
// one of them has more than half of C).
#include <type_traits>

#include "paged.hpp"

namespace blt {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
#define LDS_PTR(p) ((__attribute__((address_space(3))) s16x4_t*)(p))

// x / d for 0 <= x < 2^31 by one product: m = floor(2^s / d) + 1 with s = 31 + ceil(log2 d)
// is at most 2^s / d + 1, so x m / 2^s passes x / d by less than 1 / d.
struct Divisor {
  uint32_t m;
  int s;
};
inline Divisor divisor_of(int d) {
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return Divisor{(uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)d + 1), 31 + l};
}
__device__ inline int over(int x, const Divisor& d) {
  return (int)(((uint64_t)(uint32_t)x * d.m) >> d.s);
}

struct KArgs {
  const void *q, *k, *v;  // k, v: the layer's first element
  void* o;
  int64_t st_q, sh_q, st_o, sh_o;
  const int32_t *starts, *seqs, *lens, *table;
  int B, total, Hkv, G;
  Divisor by_g;
  int tokens_max;  // tokens that a row tile touches, at most
  int max_seqs, max_pages, num_pages, lps, cap;  // cap: tokens max_pages hold
  int causal, window;                            // window 0: none
  float c;        // log2(e) * scale
  int resident, cmin, spill;  // see Shape
  int* sync;      // a counter for every row tile with parts; all zero between calls
  int32_t* status;
  float* part;    // [slots][rows of a tile][D], unnormalised outputs
  float* ml;      // [slots][rows of a tile][2], their max (before the scale) and sum
};

// ---- which item ----------------------------------------------------------------

struct Seq {
  int s0, n, len, slot;  // first token in q, tokens, keys, sequence
};
// lost: a row without a sequence; crossed: starts that do not ascend within q (what bounds
// the grid and the workspace rests on that)
__device__ inline Seq seq_at(const KArgs& p, int b, bool& lost, bool& crossed) {
  Seq q{0, 0, 0, 0};
  if (b < p.B) {
    // (loads that wait for no comparison: all of them are on their way at once)
    const int slot = p.seqs ? p.seqs[b] : b;
    const bool known = slot >= 0 && slot < p.max_seqs;
    int len = p.lens[known ? slot : 0];
    const int a = p.starts[b], e = p.starts[b + 1];
    crossed = crossed || a < 0 || e < a || e > p.total;
    lost = lost || !known;
    len = len < 0 ? 0 : len > p.cap ? p.cap : len;
    if (a >= 0 && e > a && e <= p.total && known) q = Seq{a, e - a, len, slot};
  }
  return q;
}
// row tiles of a sequence, and the key tiles one of them may have to read
template <int BQ, int BKV>
__device__ inline void tiles_of(const KArgs& p, const Seq& q, int& nrt, int& kt) {
  nrt = (int)(((uint32_t)(q.n * p.G) + BQ - 1) / BQ);
  kt = (int)(((uint32_t)q.len + BKV - 1) / BKV);
  if (p.window) {
    const int tokens = q.n < p.tokens_max ? q.n : p.tokens_max;
    const int most = (int)((uint32_t)(p.window + tokens + BKV - 2) / BKV) + 1;
    kt = kt < most ? kt : most;
  }
  kt = kt < 1 ? 1 : kt;
}
struct Item {
  Seq q;
  int kvh, rt, split, ns;  // key head, row tile, part and number of parts
  int nrt;                 // row tiles of the sequence
  int pslot, join;         // first partial slot and first counter of its row tiles
};
__device__ inline int lane_of(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ inline float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// The item of block `bid`, false if it has none.  (Up to 64 rows a lane holds each; beyond that
// every wave walks all rows three times or more, so that a call grows with the square of its
// rows: single tokens over up to 200 keys, 12 heads, 64 of them 10 us, 256 50, 1024 406,
// 4096 5200.)  Every wave computes it by itself, in
// the same order, so all agree.
template <int BQ, int BKV>
__device__ bool find_item(const KArgs& p, unsigned bid, Item& it) {
  const int lane = threadIdx.x & 63;
  Seq q;
  int nrt, kt;
  float work = 0.f, tiles = 0.f, longest = 0.f;
  bool lost = false, crossed = false;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    q = seq_at(p, b0 + lane, lost, crossed);
    tiles_of<BQ, BKV>(p, q, nrt, kt);
    work += (float)nrt * (float)kt;
    longest = fmaxf(longest, nrt ? (float)kt : 0.f);
    tiles += (float)nrt;
  }
  if (__any(lost || crossed)) {
    if (bid == 0 && threadIdx.x == 0) atomicOr(p.status, BLT_CACHE_BAD_INDEX);
    if (__any(crossed)) return false;
  }
  // (one value for the wave, in scalar registers: what follows from it stays there too)
  work = uniform(wave_sum(work)) * (float)p.Hkv;
  tiles = uniform(wave_sum(tiles)) * (float)p.Hkv;
  // Items should fill the chip's resident blocks once, or twice where there are so many row
  // tiles that items of a single round would differ much in size and that round is a long
  // one (64 single tokens over up to 3000 keys, 12 heads, 56 us in one round and 52 in two;
  // over up to 500, 15 and 19).  Row tiles that are no whole number of C make half an
  // item more each, on average: so work / C = blocks - tiles / 2.  (0.1 % above the exact
  // quotient: the bounds on the grid and the slots hold whatever the rounding of the sums.)
  // Row tiles just above one round would leave the next one nearly empty: four rounds of parts,
  // where these are not too short (see shape_of).
  const bool spill = p.spill && tiles > (float)p.resident && tiles <= 1.5f * (float)p.resident &&
                     work >= 32.f * tiles;
  const bool twice = 2.f * tiles > (float)p.resident && work >= 12.f * p.resident;
  const float blocks = (spill ? 4.f : twice ? 2.f : 1.f) * p.resident;
  const float fill = fmaxf(blocks - 0.5f * tiles, 0.5f * (float)p.resident);
  int C = max(p.cmin, (int)fminf(ceilf(work * 1.001f / fill), 1e9f));
  // Row tiles that fill a round between them and are of about one length stay whole: parts of
  // them would only add a round that is not full (16 chunks of 128 over 8192 keys, 32 / 8
  // heads of 128: 308 us, 380 in parts; with a window of 3000 keys 113 and 210).
  longest = uniform(wave_max(longest));
  if ((BQ >= 128 || tiles <= (float)p.resident) && !spill && longest * (float)p.resident <= 1.25f * work)
    C = max(C, (int)longest);
  int ns;
  auto parts_of = [&]() {
    // (a part costs as much as a few key tiles to write and join, in proportion to its rows:
    // one chunk of 1578, 12 heads, 28 us with a quarter of them, 21 with a sixteenth; and the
    // more there are of one row tile, the longer their joining takes: one token over 8192 keys, 12 heads, 16.0 us in parts of
    // four tiles and 17.8 in parts of two, over 1000 keys 10.4 and 8.7)
    const int r = q.n * p.G, long_row = BKV < 64 || kt < 64 ? 0 : max(2, kt >> 6);
    const int most = max(C, p.cmin + long_row + (r < BQ ? r : BQ) / 16);
    ns = (int)((uint32_t)(kt + most - 1) / (uint32_t)most);
  };
  // Items, partial slots and counters of one key head.  Key heads are the outermost order of
  // the items, and dispatch places block i on XCD i % 8, of which each takes a contiguous
  // run of items: the row tiles of one (sequence, key head) share an L2, and every XCD gets
  // its share of the long sequences (2 chunks of 2048 over 16384 and 11854 keys, 8 key
  // heads: 795 us, 940 with the sequences outermost).
  int items, inc;  // of all sequences; with up to 64 of them, those up to the lane's own
  for (int tries = 0;; ++tries) {
    items = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      if (p.B > 64) {
        q = seq_at(p, b0 + lane, lost, crossed);
        tiles_of<BQ, BKV>(p, q, nrt, kt);
      }
      parts_of();
      items += nrt * ns;
    }
    inc = wave_incl_scan(items);
    items = lane_of(inc, 63);
    // a few items above a whole round would take one of their own: fewer, larger parts
    // (8 sequences of 49152 keys, 12 heads: 1056 items 295 us, 960 of them 213)
    const float excess = (float)items * (float)p.Hkv / blocks;
    if (excess <= 1.f || tiles > blocks || tries == 3) break;
    C = max(C + 1, (int)(excess * (float)C));
  }
  // partial slots, and counters above them: at most 8192 and 2048 of a call
  auto joined = [&]() { return ns > 1 ? nrt * ns + (nrt << 16) : 0; };
  int join = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (p.B > 64) {
      q = seq_at(p, b0 + lane, lost, crossed);
      tiles_of<BQ, BKV>(p, q, nrt, kt);
      parts_of();
    }
    join += joined();
  }
  int jinc = wave_incl_scan(join);
  const int joins = lane_of(jinc, 63);
  const int all = items * p.Hkv, per = (all + 7) >> 3;
  const int id = (int)(bid & 7) * per + (int)(bid >> 3);
  if ((int)(bid >> 3) >= per || id >= all) return false;
  it.kvh = (int)((uint32_t)id / (uint32_t)items);
  const int rem = id - it.kvh * items;
  int base = 0, jbase = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (p.B > 64) {
      q = seq_at(p, b0 + lane, lost, crossed);
      tiles_of<BQ, BKV>(p, q, nrt, kt);
      parts_of();
      join = joined();
      inc = wave_incl_scan(nrt * ns);
      jinc = wave_incl_scan(join);
    }
    const uint64_t above = __ballot(base + inc > rem);
    if (above) {
      const int l = __ffsll((unsigned long long)above) - 1;
      it.q = Seq{lane_of(q.s0, l), lane_of(q.n, l), lane_of(q.len, l), lane_of(q.slot, l)};
      it.nrt = lane_of(nrt, l);
      it.ns = lane_of(ns, l);
      const int before = jbase + lane_of(jinc - join, l);
      it.pslot = it.kvh * (joins & 0xffff) + (before & 0xffff);
      it.join = it.kvh * (joins >> 16) + (before >> 16);
      const int at = rem - (base + lane_of(inc - nrt * ns, l));
      it.split = (int)((uint32_t)at / (uint32_t)it.nrt);
      it.rt = it.nrt - 1 - (at - it.split * it.nrt);  // the longest causal rows first
      return true;
    }
    base += lane_of(inc, 63);
    jbase += lane_of(jinc, 63);
  }
  return false;
}
// The key tiles [t0, t1) of an item: its part of the `cnt` ones from t_lo on.
__device__ inline void part_of(const Item& it, int t_lo, int cnt, int& t0, int& t1) {
  const int each = (int)((uint32_t)cnt / (uint32_t)it.ns), more = cnt - each * it.ns;
  t0 = t_lo + it.split * each + min(it.split, more);
  t1 = t0 + each + (it.split < more ? 1 : 0);
}
__device__ inline int64_t slot_of(const Item& it, int split) {
  return it.pslot + (int64_t)split * it.nrt + it.rt;
}

// The keys rows r0 .. r1 (of one sequence) see between them: [lo, hi].
__device__ inline void key_range(const KArgs& p, const Seq& q, int r0, int r1, int& lo, int& hi) {
  const int first = q.len - q.n;  // position of token 0
  hi = q.len - 1;
  lo = 0;
  if (p.causal) {
    const int last = first + over(r1, p.by_g);
    hi = last < hi ? last : hi;
    if (p.window) {
      const int l = first + over(r0, p.by_g) - p.window + 1;
      lo = l > 0 ? l : 0;
    }
  }
}

// ---- pages of a sequence in LDS --------------------------------------------------
// A run of PT entries of the sequence's page table, clamped to the pool, so that a
// tile's addresses come from LDS: a load from the table itself would have to be
// waited for behind the tiles in flight.
constexpr int PT = 512;
__device__ inline void stage_pages(const KArgs& p, const Seq& q, int base, int* ptab, int tid,
                                   int threads) {
  const int cols = (q.len + (1 << p.lps) - 1) >> p.lps;
  for (int i = tid; i < PT; i += threads) {
    int page = base + i < cols ? p.table[(int64_t)q.slot * p.max_pages + base + i] : 0;
    page = page < 0 ? 0 : page;
    ptab[i] = page < p.num_pages ? page : p.num_pages - 1;
  }
}

// Words of two bf16 values: the largest exponents seen so far; whether one of them is an
// infinite value's or a NaN's; a word with such values zeroed.
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ inline uint32_t exponents2(uint32_t seen, uint32_t x) {
  return __builtin_bit_cast(
      uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, seen),
                                          __builtin_bit_cast(u16x2_t, x & 0x7f807f80u)));
}
__device__ inline bool not_finite2(uint32_t seen) {
  return (seen & 0xffffu) == 0x7f80u || (seen >> 16) == 0x7f80u;
}
__device__ inline uint32_t finite2(uint32_t x) {
  x = (x & 0x7f800000u) == 0x7f800000u ? x & 0xffffu : x;
  return (x & 0x7f80u) == 0x7f80u ? x & 0xffff0000u : x;
}

// ---- joining the parts of a row tile ----------------------------------------------
// Every block that has written its part counts itself; the one that finds all others
// counted joins them, in the order of the parts (so the result does not depend on who
// is last), and sets the counter back to zero.
//   o = sum_i w_i o_i / sum_i w_i l_i,  w_i = e^(scale (m_i - max))
// The blocks may sit on different XCDs, whose L2s are not coherent for ordinary accesses,
// so parts are written and read by relaxed atomics of agent scope: they pass the L2s, a
// write is complete when the wave's counter of stores says so.  (Ordinary accesses
// between fences write back and invalidate whole L2s: 48 single tokens over up to 8192
// keys, 12 heads, took 333 us that way, 135 with a second launch that joins, 128 so.)
__device__ inline void put2(float* at, float x, float y) {
  const uint64_t v = (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(at), v, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void put4(float* at, f32x4_t v) {
  put2(at, v.x, v.y);
  put2(at + 2, v.z, v.w);
}
__device__ inline void get2(const float* at, float& x, float& y) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  x = __uint_as_float((uint32_t)v);
  y = __uint_as_float((uint32_t)(v >> 32));
}
__device__ inline f32x4_t get4(const float* at) {
  f32x4_t v;
  float x, y;
  get2(at, x, y);
  v.x = x; v.y = y;
  get2(at + 2, x, y);
  v.z = x; v.w = y;
  return v;
}
// Every thread of the block has written its share of the part: is it the last one?
__device__ inline bool last_part(const KArgs& p, const Item& it) {
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's share, before the count
  __syncthreads();
  int* counter = p.sync + it.join + it.rt;
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           it.ns - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last;
}
// The forms for few rows: parts [rows][D].
// A thread takes four columns of a row at a time; where that leaves threads over and there
// are many parts, groups of threads take runs of them and meet in `room` (6 NT words of LDS
// that nobody uses any more).  Called by all threads of a block of NT.
struct Joined {
  float m, l;
  f32x4_t o;
};
__device__ inline void join(Joined& a, const Joined& b, float c) {
  const float mx = fmaxf(a.m, b.m), off = mx == -INFINITY ? 0.f : mx;
  const float wa = __builtin_amdgcn_exp2f((a.m - off) * c);
  const float wb = __builtin_amdgcn_exp2f((b.m - off) * c);
  a.m = mx;
  a.l = fmaf(a.l, wa, wb * b.l);
  a.o = a.o * wa + wb * b.o;
}
template <int D, int BQ, int NT, typename T>
__device__ void join_parts(const KArgs& p, const Item& it, int nr, float* room) {
  if (!last_part(p, it)) return;
  // U parts at a time, everything of them in flight at once (a read that passes the L2 takes
  // about 1 us), with a running max; past the last part: the last one again, without weight.
  // Its infinite values become NaN by that: where a sum is none, the parts are added up once
  // more, those past the last as empty ones (0.2 us a call if it is always done so).
  const int64_t step = (int64_t)it.nrt * BQ;
  auto sum = [&](int i, int x0, int x1, auto at_once, auto odd) {
    constexpr int U = decltype(at_once)::value;
    const int64_t s0 = slot_of(it, 0) * BQ + i / (D / 4);
    const int dd = (i % (D / 4)) * 4;
    Joined a{-INFINITY, 0.f, f32x4_t{0.f, 0.f, 0.f, 0.f}};
    for (int x = x0; x < x1; x += U) {
      float m[U], l[U];
      f32x4_t o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = s0 + min(x + u, x1 - 1) * step;
        get2(p.ml + at * 2, m[u], l[u]);
        o[u] = get4(p.part + at * D + dd);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (x + u < x1) continue;
        m[u] = -INFINITY;
        if constexpr (decltype(odd)::value) {
          l[u] = 0.f;
          o[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
      }
      float mn = a.m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, m[u]);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f((a.m - mu) * p.c);
      a.m = mn;
      a.l *= alpha;
      a.o *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __builtin_amdgcn_exp2f((m[u] - mu) * p.c);
        a.l = fmaf(w, l[u], a.l);
        a.o += w * o[u];
      }
    }
    return a;
  };
  auto run = [&](int i, int x0, int x1, auto at_once) {
    const Joined a = sum(i, x0, x1, at_once, std::false_type{});
    const float all = (a.o.x + a.o.y) + (a.o.z + a.o.w) + a.l;
    return all == all ? a : sum(i, x0, x1, at_once, std::true_type{});
  };
  auto store = [&](int i, const Joined& a) {
    const int r = i / (D / 4), dd = (i % (D / 4)) * 4;
    const int row = it.rt * BQ + r, t = over(row, p.by_g), g = row - t * p.G;
    const int64_t at =
        (int64_t)(it.q.s0 + t) * p.st_o + (int64_t)(it.kvh * p.G + g) * p.sh_o + dd;
    const f32x4_t x = a.l == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : a.o / a.l;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2_t*>((uint16_t*)p.o + at) =
          u32x2_t{pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w)};
    else
      *reinterpret_cast<f32x4_t*>((float*)p.o + at) = x;
  };
  constexpr std::integral_constant<int, 8> eight{};
  constexpr std::integral_constant<int, BQ <= 32 && sizeof(T) == 2 ? 16 : 8> more{};
  const int work = nr * (D / 4);
  if (it.ns <= 8) {
    for (int i = threadIdx.x; i < work; i += NT) store(i, run(i, 0, it.ns, eight));
    return;
  }
  if (2 * work > NT) {
    for (int i = threadIdx.x; i < work; i += NT) store(i, run(i, 0, it.ns, more));
    return;
  }
  const int groups = NT / work, per = (it.ns + groups - 1) / groups;
  const int i = threadIdx.x % work, g = threadIdx.x / work;
  const int x0 = min(g * per, it.ns);
  Joined a = run(i, x0, g < groups ? min(x0 + per, it.ns) : x0, eight);
  *reinterpret_cast<f32x4_t*>(room + threadIdx.x * 4) = a.o;
  room[4 * NT + threadIdx.x] = a.m;
  room[5 * NT + threadIdx.x] = a.l;
  __syncthreads();
  if (g > 0) return;
  for (int x = 1; x < groups; ++x) {
    const int th = i + x * work;
    join(a, Joined{room[4 * NT + th], room[5 * NT + th], *reinterpret_cast<f32x4_t*>(room + th * 4)},
         p.c);
  }
  store(i, a);
}

// The forms for 128 rows, a wave with 32 of them and o in the accumulators' layout.  A part is
// laid out as the threads hold it, [D / 4][256] pairs, so that whole lines are written and
// read: the last block's threads take up the values of their own rows.  (By rows, with every
// lane's 16 bytes in another line, 4 chunks of 512 over 4096 keys, 12 heads, took 64 us
// instead of 53.)  False where the thread has nothing to store; else o, total are the row's.
template <int D>
__device__ inline bool join_tiles(const KArgs& p, const Item& it, bool active,
                                  f32x16_t (&o)[D / 32], float m, float& total) {
  constexpr int BQ = 128, PAIRS = D / 4;
  const int tid = threadIdx.x, trow = (tid >> 6) * 32 + (tid & 31);
  if (active) {
    const int64_t slot = slot_of(it, it.split);
    float* at = p.part + slot * BQ * D + tid * 2;
#pragma unroll
    for (int k = 0; k < PAIRS; ++k)
      put2(at + k * 512, o[k >> 3][2 * (k & 7)], o[k >> 3][2 * (k & 7) + 1]);
    if (!(tid & 32)) put2(p.ml + (slot * BQ + trow) * 2, m, total);
  }
  if (!last_part(p, it) || !active) return false;
  constexpr int U = 2;  // parts in flight at once (more would cost a block a CU)
  float mx = -INFINITY;
  total = 0.f;
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[j][r] = 0.f;
  for (int x0 = 0; x0 < it.ns; x0 += U) {
    float pm[U], pl[U], v[U][D / 2];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the last part: the last one again, left out)
      const int64_t slot = slot_of(it, min(x0 + u, it.ns - 1));
      const float* at = p.part + slot * BQ * D + tid * 2;
      get2(p.ml + (slot * BQ + trow) * 2, pm[u], pl[u]);
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) get2(at + k * 512, v[u][2 * k], v[u][2 * k + 1]);
    }
    float mn = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) mn = fmaxf(mn, pm[u]);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((mx - mu) * p.c);
    mx = mn;
    total *= alpha;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[j][r] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (x0 + u < it.ns) {
        const float w = __builtin_amdgcn_exp2f((pm[u] - mu) * p.c);
        total = fmaf(w, pl[u], total);
#pragma unroll
        for (int k = 0; k < D / 2; ++k) o[k >> 4][k & 15] = fmaf(w, v[u][k], o[k >> 4][k & 15]);
      }
  }
  return true;
}

// p = 2^(s c - m c) is one fma with m c rounded, which is off by 2^-24 |m c| in the exponent: much
// where scores are large (beyond 2^31 the largest key's p would overflow or vanish).  From here
// on m is taken from s first, which is exact.  Only looked at where a wave's offsets move.
constexpr float kFar = 1024.f;

// ---- bf16, tiles of rows ---------------------------------------------------------
// One block = 4 waves of 32 rows each; key tiles of 64 keys go global -> LDS by DMA
// through NST stages shared by the waves.  As in attn_fwd_kernel the scores are taken
// transposed, S^T = K . Q^T, so a lane owns one row: its max and sum need one
// cross-lane step, P^T feeds the second product from registers, and V's operand is
// read with the LDS transposing read.  Unlike there q keeps its own bf16 values (scaling it
// before its rounding costs as much accuracy as the output's rounding): the scale and the
// running max go into one fma before exp2.
// p is rounded to bf16 for the second product, and the sum takes the rounded values: the
// outputs are 2.3e-3 off (relative, rms; their own rounding alone is 1.7e-3).  As two halves,
// as in the form below, the chunks named next take 1080 us.
// Chunks of 2048 and 1598 tokens over 16384 and 11854 keys, 32 / 8 heads of 128: 795 us,
// 1.0 PFLOP/s of the visible pairs (an 8192^3 library product reaches 1.4); the matrix cores
// are busy 46 % of the time and the vector units 43 %, hardly ever both.  With 64 rows a wave
// (1.2 ms for 0.96 then), three stages, or 32-key tiles at three waves a SIMD it was slower.
template <int D, int NST>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(KArgs p) {
  constexpr int BKV = 64, QPW = 32, BQ = 4 * QPW;
  constexpr int TILE = BKV * D;        // elements of a K (or V) tile
  constexpr int STAGE = 2 * TILE;
  constexpr int NOP = 4 * (D / 64);    // DMA instructions of a wave per tile
  constexpr int KS = D / 16, DS = D / 32;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[NST * STAGE];
  __shared__ int ptab[PT];

  Item it;
  if (!find_item<BQ, BKV>(p, blockIdx.x, it)) return;
  const Seq& sq = it.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int rows = sq.n * p.G;
  const int first = sq.len - sq.n;

  // the block's key tiles [t0, t1)
  int lo, hi;
  const int r0 = it.rt * BQ, r1 = min(r0 + BQ, rows) - 1;
  key_range(p, sq, r0, r1, lo, hi);
  const int t_lo = lo / BKV, cnt = hi < 0 ? 0 : hi / BKV - t_lo + 1;
  int t0, t1;
  part_of(it, t_lo, cnt, t0, t1);
  // the wave's
  const int rw = r0 + wid * QPW;
  const bool wave_active = rw < rows;
  int wlo = 0, whi = -1;
  const int rwl = min(rw + QPW, rows) - 1;
  if (wave_active) key_range(p, sq, rw, rwl, wlo, whi);
  const int pos_first = first + over(rw, p.by_g);  // lowest position in the wave
  const int lo_last = p.window ? first + over(rwl, p.by_g) - p.window + 1 : 0;  // highest lower bound

  // Q fragments (B operand): row rw + lrow, d = 16 ks + 8 lhalf .. + 8
  bf16x8_t qf[KS];
  const int row = rw + lrow;
  const int tok = over(min(row, rows - 1), p.by_g), head = it.kvh * p.G + min(row, rows - 1) - tok * p.G;
  {
    const uint16_t* qrow =
        (const uint16_t*)p.q + (int64_t)(sq.s0 + tok) * p.st_q + (int64_t)head * p.sh_q;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[ks] = __builtin_bit_cast(
          bf16x8_t, *reinterpret_cast<const u32x4_t*>(qrow + ks * 16 + lhalf * 8));
  }
  // the row's visible keys
  const int khi = p.causal ? min(first + tok, sq.len - 1) : sq.len - 1;
  const int klo = p.window ? first + tok - p.window + 1 : 0;
  int wbase = (t0 * BKV) >> p.lps;
  if (t0 < t1) stage_pages(p, sq, wbase, ptab, tid, 256);
  // consumed here, before any DMA is in flight (see attn_fwd_kernel)
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[ks]));
  __syncthreads();

  // DMA.  Wave w moves keys 16 w .. 16 w + 15 of a tile, eight (one page) at a time.  LDS
  // rows are D elements without padding; 16-byte chunk c of a row is stored at c ^ (a
  // swizzle of the row) so that the operand reads spread over all banks.
  const unsigned lds_base = (unsigned)(uintptr_t)lds;
  constexpr int CPR = D / 8;                     // chunks of a row
  const int kin = lane / CPR, slot = lane % CPR;  // key within one instruction, chunk slot
  // rows k of K: D = 64 (k >> 1) & 7, D = 128 k & 15; of V: 4 ((k >> 1) & 1), 4 (k & 3)
  const int kx = slot ^ (D == 64 ? kin >> 1 : kin);
  const int vx = slot ^ (4 * (D == 64 ? (kin >> 1) & 1 : kin & 3));
  auto issue = [&](int t, int stage) {
    const unsigned sb = lds_base + (unsigned)(stage * STAGE * 2);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key0 = t * BKV + 16 * wid + 8 * g;
      const int kc = min(key0, (sq.len - 1) & ~7);  // the group that is read
      const int page = __builtin_amdgcn_readfirstlane(ptab[(kc >> p.lps) - wbase]);
      const int64_t off =
          (((((int64_t)page * p.Hkv + it.kvh) << p.lps) + (kc & ((1 << p.lps) - 1))) * D) * 2;
      const char* kb = (const char*)p.k + off;
      const char* vb = (const char*)p.v + off;
      const bool all = key0 + 8 <= sq.len;  // else rows past the end read the last key
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        int row = kin + (D == 128 ? 4 * h : 0);
        if (!all) row = min(key0 + row, sq.len - 1) - kc;
        const int kch = kx ^ (D == 64 ? 4 * g : 8 * g + 4 * h);
        const unsigned la = sb + (unsigned)((16 * wid + 8 * g) * D * 2 + h * 1024);
        dma16_so(kb, (unsigned)(row * D * 2 + kch * 16), la);
        dma16_so(vb, (unsigned)(row * D * 2 + vx * 16), la + TILE * 2);
      }
    }
  };
  // lanes' LDS offsets: K row of key lrow, V's transposing reads (see attn_fwd_kernel)
  const int s16 = lane & 15;
  int vt[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds)
    vt[ds] = (4 * lhalf + (s16 >> 2)) * D + 32 * (ds ^ (D == 64 ? s16 >> 3 : s16 >> 2)) +
             16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
  const int kswz = D == 64 ? (lrow >> 1) & 7 : lrow & 15;

  f32x16_t o[DS];
  float m = -INFINITY, l = 0.f;  // the row's offset (-inf until its first visible key), its sum
  float mc = 0.f;                // -m c, or 0 where m is taken from the scores themselves (far)
  bool far = false;
#pragma unroll
  for (int j = 0; j < DS; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[j][r] = 0.f;
  const bf16x2_t ones2 = {(__bf16)1.0f, (__bf16)1.0f};
  const float c = p.c, grow_at = 8.f / p.c;

  // pages of tile t are in ptab (refilled, rarely, when the run is used up; every wave is
  // past its reads of the old run at the barrier before issue(t))
  auto need = [&](int t) {
    const int last = min(t * BKV + BKV - 1, sq.len - 1) >> p.lps;
    if (last >= wbase + PT) {
      wbase = (t * BKV) >> p.lps;
      stage_pages(p, sq, wbase, ptab, tid, 256);
      __syncthreads();
    }
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (t0 + i < t1) issue(t0 + i, i);  // (a run of pages covers the first tiles)
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // tile t has landed and every wave is past tile t - 1, whose stage is free
    if (NST > 2 && t + 1 < t1) dma_wait_barrier<NOP*(NST - 2)>(); else dma_wait_barrier<0>();
    if (t + NST - 1 < t1) {
      need(t + NST - 1);
      issue(t + NST - 1, stage == 0 ? NST - 1 : stage - 1);
    }
    const int kb = t * BKV;
    if (wave_active && kb <= whi && kb + BKV > wlo) {
      const uint16_t* sk = lds + stage * STAGE;
      const uint16_t* sv = sk + TILE;
      const bool mask_hi = kb + BKV - 1 > (p.causal ? pos_first : sq.len - 1) ||
                           kb + BKV > sq.len;
      const bool mask_lo = p.window && kb < lo_last;
      // All of K's fragments are read before the first product and all of V's under the
      // softmax: against that, 2 chunks over up to 16384 keys (d = 128) take 4 % longer with
      // V's read between the products of the second, 85 % with K's among those of the first.
      bf16x8_t f[2][KS];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          f[sub][ks] = *reinterpret_cast<const bf16x8_t*>(
              sk + (sub * 32 + lrow) * D + (((2 * ks + lhalf) ^ kswz) << 3));
      f32x16_t s[2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
          s[sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              f[sub][ks], qf[ks], ks == 0 ? f32x16_t{} : s[sub], 0, 0, 0);
      u32x4_t vf[DS][2][2];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint16_t* vp = sv + (sub * 32 + u * 16) * D + vt[ds];
            const u32x2_t w0 =
                __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(vp)));
            const u32x2_t w1 = __builtin_bit_cast(
                u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(vp + 8 * D)));
            vf[ds][sub][u] = u32x4_t{w0.x, w0.y, w1.x, w1.y};
          }
      if (mask_hi) {
        const int rel = khi - kb - 4 * lhalf;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[sub][r] = sub * 32 + 8 * (r >> 2) + (r & 3) <= rel ? s[sub][r] : -INFINITY;
      }
      if (mask_lo) {
        const int rel = klo - kb - 4 * lhalf;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[sub][r] = sub * 32 + 8 * (r >> 2) + (r & 3) >= rel ? s[sub][r] : -INFINITY;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[sub][r]);
      {
        float a, b;
        swap_pair<32>(mt, a, b);
        mt = fmaxf(a, b);
      }
      // the offset moves only when the max is more than 2^8 over it (far: in every tile)
      if (__any(mt > m + grow_at) || far) {
        const float m_new = fmaxf(m, mt);
        const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int j = 0; j < DS; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[j][r] *= alpha;
        mc = m == -INFINITY ? 0.f : -m * c;
        far = __any(fabsf(mc) > kFar);
        if (__builtin_expect(far, false)) {
          const float mu = m == -INFINITY ? 0.f : m;
          mc = 0.f;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[sub][r] -= mu;
        }
      }
      // A weight of zero does not silence an infinite or NaN value: where rows see different
      // keys of a tile that holds one, it is taken out of the product and added to the
      // rows that see it (behind the rescaling, whose factor may be zero).
      if (mask_hi || mask_lo) {
        uint32_t seen = 0;
#pragma unroll
        for (int i = 0; i < DS * 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            seen = exponents2(seen, vf[i >> 2][(i >> 1) & 1][i & 1][e]);
        if (__any(not_finite2(seen))) {
#pragma unroll
          for (int i = 0; i < DS * 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vf[i >> 2][(i >> 1) & 1][i & 1][e] = finite2(vf[i >> 2][(i >> 1) & 1][i & 1][e]);
          for (int j = 0; j < BKV; ++j) {
            const bool sees = kb + j <= khi && kb + j >= klo;
            const int swz = 4 * (D == 64 ? (j >> 1) & 1 : j & 3);
#pragma unroll
            for (int i = 0; i < DS * 4; ++i) {  // columns 8 i + 4 lhalf .. + 3
              const u32x2_t x =
                  *reinterpret_cast<const u32x2_t*>(sv + j * D + ((i ^ swz) << 3) + 4 * lhalf);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = bf16_to_f32((uint16_t)(x[e >> 1] >> (16 * (e & 1))));
                o[i >> 2][4 * (i & 3) + e] += sees && !(fabsf(v) < INFINITY) ? v : 0.f;
              }
            }
          }
        }
      }
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[sub][8 * u + e], c, mc));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[sub][8 * u + e + 1], c, mc));
            w[e >> 1] = pack_bf16x2(p0, p1);
            l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[e >> 1]), ones2, l,
                                                false);
          }
          const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{w[0], w[1], w[2], w[3]});
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)  // (independent chains)
            o[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(bf16x8_t, vf[ds][sub][u]), pb, o[ds], 0, 0, 0);
        }
    }
    stage = stage + 1 < NST ? stage + 1 : 0;
  }

  float a, b;
  swap_pair<32>(l, a, b);
  const float lt = a + b;
  float total = lt;
  if (it.ns > 1 && !join_tiles<D>(p, it, wave_active, o, m, total)) return;
  if (row < rows) {
    uint16_t* orow = (uint16_t*)p.o + (int64_t)(sq.s0 + tok) * p.st_o + (int64_t)head * p.sh_o;
    // hardware reciprocal (1 ulp): the output is rounded to bf16
    const float inv = total > 0.f ? __builtin_amdgcn_rcpf(total) : total == total ? 0.f : total;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x2_t w;
        w.x = pack_bf16x2(o[ds][4 * j] * inv, o[ds][4 * j + 1] * inv);
        w.y = pack_bf16x2(o[ds][4 * j + 2] * inv, o[ds][4 * j + 3] * inv);
        *reinterpret_cast<u32x2_t*>(orow + ds * 32 + 8 * j + 4 * lhalf) = w;
      }
  }
}

// ---- bf16, few rows ----------------------------------------------------------------
// Up to 16 NR rows (single tokens, short chunks): bound by reading K and V once, so the
// waves of a block share nothing and wait for nothing but their own loads: each takes
// every NW-th 32-key tile of the item through its own LDS ring of two tiles, filled by DMA
// while the tiles before are consumed, and they meet once at the end.  16 x 16 x 32
// MFMAs, scores transposed as above (a lane owns a row, the key blocks' registers are the
// second product's operand).  p goes into that product as two bf16 halves (p cut off, and
// what that left, rounded): the matrix cores have nothing else to do, and p is off by 2^-15 at
// most, against 2^-8 of the output's own rounding.  Cut off and not rounded, and the rest with
// 2^-22 p on top, so that both halves are above zero: an infinite value times zero or a
// negative rest would be NaN (below p = 2^-104, where the rest may vanish, it still is).
// 48 single tokens over up to 8192 keys, 12 heads of 64: 128 us, 5.0 TB/s; 16 over up to 32768
// keys, 32 / 8 heads of 128: 169 us, 5.5 TB/s (a large copy: 6.15).  One token over 1000 keys,
// 12 heads: 8.9 us of dependent steps: launch 1.7, find_item 0.5, pages 0.6, tiles 2.1, the
// waves' merge 1.3, join 2.6; over 8192 keys 15.4 us, over 32768 26.8.
constexpr float kAbove1 = 1.f + 0x1p-22f;
template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int D, int NR, int NW>
__global__ __launch_bounds__(64 * NW) void paged_attn_few_kernel(KArgs p) {
  constexpr int KT = 32, BKV = 64, BQ = 16 * NR, TILE = KT * D, NST = 2;
  constexpr int OPS = 4 * (D / 64);  // DMA instructions of a K (or V) tile
  constexpr int KS = D / 32, DB = D / 16, OP = D + 4, PTF = 1024;
  constexpr int RING = NW * NST * 2 * TILE;  // elements
  static_assert(RING * 2 >= NW * BQ * OP * 4, "the waves' outputs fit the rings");
  __shared__ __attribute__((aligned(1024))) uint16_t lds[RING];
  __shared__ float sm[NW][BQ], sl[NW][BQ];
  __shared__ int ptab[PTF];

  Item it;
  if (!find_item<BQ, BKV>(p, blockIdx.x, it)) return;
  const Seq& sq = it.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  const int r0 = it.rt * BQ, r1 = min(r0 + BQ, rows) - 1;
  int lo, hi;
  key_range(p, sq, r0, r1, lo, hi);
  // the item's key tiles [t0, t1), of 32 keys here
  const int t_lo = lo / KT, cnt = hi < 0 ? 0 : hi / KT - t_lo + 1;
  int t0, t1;
  part_of(it, t_lo, cnt, t0, t1);

  bf16x8_t qf[NR][KS];
  int klo[NR], khi[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = min(r0 + 16 * n + col, rows - 1);
    const int t = over(r, p.by_g), g = r - t * p.G;
    const uint16_t* qrow = (const uint16_t*)p.q + (int64_t)(sq.s0 + t) * p.st_q +
                           (int64_t)(it.kvh * p.G + g) * p.sh_q;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[n][ks] = __builtin_bit_cast(
          bf16x8_t, *reinterpret_cast<const u32x4_t*>(qrow + ks * 32 + g4 * 8));
    khi[n] = p.causal ? min(first + t, sq.len - 1) : sq.len - 1;
    klo[n] = p.window ? first + t - p.window + 1 : 0;
  }
  // every row sees [all_lo, all_hi]
  const int all_hi = p.causal ? min(first + over(r0, p.by_g), sq.len - 1) : sq.len - 1;
  const int all_lo = p.window ? first + over(r1, p.by_g) - p.window + 1 : 0;

  // DMA of one tile: eight keys (one page) at a time, chunks swizzled for the operand reads
  const unsigned ring = (unsigned)(uintptr_t)lds + (unsigned)(w * NST * 2 * TILE * 2);
  constexpr int CPR = D / 8;
  const int kin = lane / CPR, slot = lane % CPR;
  const int kx = slot ^ (D == 64 ? kin >> 1 : kin);
  const int vx = slot ^ (D == 64 ? 2 * (kin >> 1) : 2 * kin);
  int wbase = 0;
  // byte offsets of a tile's groups of eight keys in K and V (past the end: the last group)
  struct Groups {
    int64_t at[4];
  };
  auto group = [&](int t, int g) { return min(t * KT + 8 * g, (sq.len - 1) & ~7); };
  auto place = [&](int t) {
    int pg[4];
    Groups x;
#pragma unroll
    for (int g = 0; g < 4; ++g) pg[g] = ptab[(group(t, g) >> p.lps) - wbase];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int page = __builtin_amdgcn_readfirstlane(pg[g]);
      x.at[g] = (((((int64_t)page * p.Hkv + it.kvh) << p.lps) +
                  (group(t, g) & ((1 << p.lps) - 1))) * D) * 2;
    }
    return x;
  };
  auto issue = [&](int t, int stage, const Groups& x, auto of_v) {
    constexpr bool V = decltype(of_v)::value;
    const unsigned sb = ring + (unsigned)(stage * 2 * TILE * 2) + (V ? TILE * 2 : 0);
    // (this wave's operand reads of the stage are done)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const char* base = (const char*)(V ? p.v : p.k) + x.at[g];
      const int key0 = t * KT + 8 * g;
      const bool all = key0 + 8 <= sq.len;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        int row = kin + (D == 128 ? 4 * h : 0);
        if (!all) row = min(key0 + row, sq.len - 1) - group(t, g);
        const int ch = V ? (D == 64 ? vx : vx ^ (8 * h))
                         : kx ^ (D == 64 ? 4 * (g & 1) : 8 * (g & 1) + 4 * h);
        dma16_so(base, (unsigned)(row * D * 2 + ch * 16),
                 sb + (unsigned)(8 * g * D * 2 + h * 1024));
      }
    }
  };
  constexpr std::false_type of_k{};
  constexpr std::true_type of_v{};
  // operand reads: K row `col` of a 16-key block; V rows 4 g4 + col / 4, 16 columns at 16 db
  const int kswz = D == 64 ? (col >> 1) & 7 : col;
  const int vrow = 4 * g4 + (col >> 2);
  const int vswz = D == 64 ? (vrow >> 1) & 3 : vrow & 7;  // of 16-column blocks
  const int vlane = vrow * D + 4 * (col & 3);

  f32x4_t o[NR][DB];
  float l[NR], m[NR];
  float mc[NR];  // (as in paged_attn_kernel)
  bool far[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = -INFINITY;
    mc[n] = 0.f;
    far[n] = false;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[n][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const float c = p.c, grow_at = 8.f / p.c;

  // Tile t of this wave; `more` follow.  A half of the ring is refilled as soon as
  // it is read: K of tile t + 2 under the softmax of t, V behind its second product, so
  // three halves or more are on their way at any time.
  auto tile = [&](int t, int stage, int more) {
    if (more >= 1) wait_loads<3 * OPS>(); else wait_loads<OPS>();  // K has landed
    const uint16_t* sk = lds + (w * NST + stage) * 2 * TILE;
    const uint16_t* sv = sk + TILE;
    const int kb = t * KT;
    f32x4_t s[NR][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(
            sk + (16 * b + col) * D + (((4 * ks + g4) ^ kswz) << 3));
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              a, qf[n][ks], ks == 0 ? f32x4_t{} : s[n][b], 0, 0, 0);
        }
      }
    Groups next{};
    if (more >= 2) {
      next = place(t + 2 * NW);
      issue(t + 2 * NW, stage, next, of_k);
    }
    const bool mask = kb + KT - 1 > all_hi || kb < all_lo;
    bf16x8_t ph[NR], pl[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (mask) {
        const int up = khi[n] - kb - 4 * g4, dn = klo[n] - kb - 4 * g4;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[n][b][r] = 16 * b + r <= up && 16 * b + r >= dn ? s[n][b][r] : -INFINITY;
      }
      float mt = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      {
        float a, b;
        swap_pair<16>(mt, a, b);
        mt = fmaxf(a, b);
        swap_pair<32>(mt, a, b);
        mt = fmaxf(a, b);
      }
      if (__any(mt > m[n] + grow_at) || far[n]) {
        const float m_new = fmaxf(m[n], mt);
        const float alpha = m[n] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[n] - m_new) * c);
        m[n] = m_new;
        l[n] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[n][d] *= alpha;
        mc[n] = m_new == -INFINITY ? 0.f : -m_new * c;
        far[n] = __any(fabsf(mc[n]) > kFar);
        if (__builtin_expect(far[n], false)) {
          const float mu = m_new == -INFINITY ? 0.f : m_new;
          mc[n] = 0.f;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][b][r] -= mu;
        }
      }
      uint32_t wh[4], wl[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][e & 3], c, mc[n]));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][(e & 3) + 1], c, mc[n]));
        l[n] += p0 + p1;
        const uint32_t x0 = __float_as_uint(p0), x1 = __float_as_uint(p1);
        wh[e >> 1] = __builtin_amdgcn_perm(x1, x0, 0x07060302);  // their upper halves
        wl[e >> 1] = pack_bf16x2(fmaf(p0, kAbove1, -__uint_as_float(x0 & 0xffff0000u)),
                                 fmaf(p1, kAbove1, -__uint_as_float(x1 & 0xffff0000u)));
      }
      ph[n] = __builtin_bit_cast(bf16x8_t, u32x4_t{wh[0], wh[1], wh[2], wh[3]});
      pl[n] = __builtin_bit_cast(bf16x8_t, u32x4_t{wl[0], wl[1], wl[2], wl[3]});
    }
    if (more >= 2) wait_loads<3 * OPS>(); else if (more == 1) wait_loads<2 * OPS>(); else wait_loads<0>();
    u32x4_t vf[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint16_t* vp = sv + vlane + 16 * (d ^ vswz);
      const u32x2_t w0 =
          __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(vp)));
      const u32x2_t w1 = __builtin_bit_cast(
          u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(vp + 16 * D)));
      vf[d] = u32x4_t{w0.x, w0.y, w1.x, w1.y};
    }
    if (mask) {  // (as in paged_attn_kernel: no infinite value behind a mask)
      uint32_t seen = 0;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) seen = exponents2(seen, vf[d][e]);
      if (__any(not_finite2(seen))) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[d][e] = finite2(vf[d][e]);
        for (int j = 0; j < KT; ++j) {
          const int swz = D == 64 ? (j >> 1) & 3 : j & 7;
#pragma unroll
          for (int d = 0; d < DB; ++d) {  // columns 16 d + 4 g4 .. + 3
            const u32x2_t x =
                *reinterpret_cast<const u32x2_t*>(sv + j * D + 16 * (d ^ swz) + 4 * g4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = bf16_to_f32((uint16_t)(x[e >> 1] >> (16 * (e & 1))));
#pragma unroll
              for (int n = 0; n < NR; ++n)
                o[n][d][e] +=
                    kb + j <= khi[n] && kb + j >= klo[n] && !(fabsf(v) < INFINITY) ? v : 0.f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const bf16x8_t a = __builtin_bit_cast(bf16x8_t, vf[d]);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ph[n], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pl[n], o[n][d], 0, 0, 0);
      }
    }
    if (more >= 2) issue(t + 2 * NW, stage, next, of_v);
  };

  // runs of tiles whose pages ptab holds (one, but for very long parts)
  const int run = ((PTF - 1) << p.lps) / KT;
  for (int ta = t0; ta < t1; ta += run) {
    const int tb = min(ta + run, t1);
    if (ta > t0) __syncthreads();
    wbase = (ta * KT) >> p.lps;
    {
      const int cols = (sq.len + (1 << p.lps) - 1) >> p.lps;
      const int n = min(PTF, ((min(tb * KT, sq.len) - 1) >> p.lps) - wbase + 1);
      for (int i = tid; i < n; i += 64 * NW) {
        int page = wbase + i < cols ? p.table[(int64_t)sq.slot * p.max_pages + wbase + i] : 0;
        page = page < 0 ? 0 : page;
        ptab[i] = page < p.num_pages ? page : p.num_pages - 1;
      }
    }
    __syncthreads();
    const int mine = (tb - ta - w + NW - 1) / NW;  // this wave's tiles
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i < mine) {
        const Groups x = place(ta + w + i * NW);
        issue(ta + w + i * NW, i, x, of_k);
        issue(ta + w + i * NW, i, x, of_v);
      }
    for (int i = 0; i < mine; ++i) tile(ta + w + i * NW, i & 1, mine - 1 - i);
  }

  // ---- the waves' partial results ----
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float a, b;
    swap_pair<16>(l[n], a, b);
    l[n] = a + b;
    swap_pair<32>(l[n], a, b);
    l[n] = a + b;
    if (g4 == 0) {
      sm[w][16 * n + col] = m[n];
      sl[w][16 * n + col] = l[n];
    }
  }
  __syncthreads();  // every wave is past its ring
  float* so = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *reinterpret_cast<f32x4_t*>(so + (w * BQ + 16 * n + col) * OP + 16 * d + 4 * g4) = o[n][d];
  __syncthreads();
  const int nr = r1 - r0 + 1;
  const int64_t at = it.ns > 1 ? slot_of(it, it.split) * BQ : 0;
  for (int i = tid; i < nr * (D / 4); i += 64 * NW) {
    const int r = i / (D / 4), dd = (i % (D / 4)) * 4;
    float mx = sm[0][r];
#pragma unroll
    for (int x = 1; x < NW; ++x) mx = fmaxf(mx, sm[x][r]);
    const float off = mx == -INFINITY ? 0.f : mx;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    float lt = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float wt = __builtin_amdgcn_exp2f((sm[x][r] - off) * c);
      lt += wt * sl[x][r];
      acc += wt * *reinterpret_cast<const f32x4_t*>(so + (x * BQ + r) * OP + dd);
    }
    if (it.ns > 1) {
      put4(p.part + (at + r) * D + dd, acc);
      if (dd == 0) put2(p.ml + (at + r) * 2, mx, lt);
    } else {
      const int t = over(r0 + r, p.by_g), g = (r0 + r) - t * p.G;
      uint16_t* dst = (uint16_t*)p.o + (int64_t)(sq.s0 + t) * p.st_o +
                      (int64_t)(it.kvh * p.G + g) * p.sh_o + dd;
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{pack_bf16x2(acc.x * inv, acc.y * inv),
                                                 pack_bf16x2(acc.z * inv, acc.w * inv)};
    }
  }
  if (it.ns > 1) join_parts<D, BQ, 64 * NW, uint16_t>(p, it, nr, so);
}

// ---- f32 -------------------------------------------------------------------------
// As attn_f32_kernel (k_attn.hip): both products on the f32 matrix cores, one block = 32
// rows, its four waves take every fourth 32-key tile with operands straight from global
// memory, and meet once at the end.  Chunks of 100, 97 and 87 tokens over 1500, 350 and 87 keys,
// 12 heads: 22.5 us; two tiles a wave, each 64 MFMAs of 64 cycles behind its loads, then the
// merge and the join.  A single token fills a whole tile of 32 rows: one over 8192 keys 22.4 us.
template <int ND>
__global__ __launch_bounds__(256) void paged_attn_f32_kernel(KArgs p) {
  constexpr int D = 32 * ND, NW = 4, NC = 4 * ND, OP = D + 4, BQ = 32, BKV = 32;
  __shared__ __attribute__((aligned(16))) float so[NW * 32 * OP];
  __shared__ float sm[NW][32], sl[NW][32];
  __shared__ int ptab[PT];
  Item it;
  if (!find_item<BQ, BKV>(p, blockIdx.x, it)) return;
  const Seq& sq = it.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  const int r0 = it.rt * BQ, r1 = min(r0 + BQ, rows) - 1;
  int lo, hi;
  key_range(p, sq, r0, r1, lo, hi);
  const int t_lo = lo / BKV, cnt = hi < 0 ? 0 : hi / BKV - t_lo + 1;
  int t0, t1;
  part_of(it, t_lo, cnt, t0, t1);

  const int r = min(r0 + l31, rows - 1);
  const int tok = over(r, p.by_g), g = r - tok * p.G;
  const int khi = p.causal ? min(first + tok, sq.len - 1) : sq.len - 1;
  const int klo = p.window ? first + tok - p.window + 1 : 0;
  f32x4_t qf[NC], kf[NC];
  {
    const float* qrow = (const float*)p.q + (int64_t)(sq.s0 + tok) * p.st_q +
                        (int64_t)(it.kvh * p.G + g) * p.sh_q;
#pragma unroll
    for (int j = 0; j < NC; ++j) qf[j] = *reinterpret_cast<const f32x4_t*>(qrow + 8 * j + 4 * h);
  }
  const int mask = (1 << p.lps) - 1;
  int wbase = 0;
  // element offset of a key's row; keys past the end give the last one
  auto row_at = [&](int key) -> int64_t {
    key = min(key, sq.len - 1);
    const int page = ptab[(key >> p.lps) - wbase];
    return ((((int64_t)page * p.Hkv + it.kvh) << p.lps) + (key & mask)) * D;
  };
  auto load_k = [&](int t) {
    const float* row = (const float*)p.k + row_at(t * BKV + l31);
#pragma unroll
    for (int j = 0; j < NC; ++j) kf[j] = *reinterpret_cast<const f32x4_t*>(row + 8 * j + 4 * h);
  };
  // V in VW-wide pieces: row i of O^T block n is column VW i + n % VW + 32 VW (n / VW)
  constexpr int VW = ND % 4 == 0 ? 4 : 2, NV = ND / VW;
  typedef float vf_t __attribute__((ext_vector_type(VW)));

  f32x16_t oacc[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[n][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = p.c;
  // every row sees [all_lo, all_hi]
  const int all_hi = p.causal ? min(first + over(r0, p.by_g), sq.len - 1) : sq.len - 1;
  const int all_lo = p.window ? first + over(r1, p.by_g) - p.window + 1 : 0;
  // one tile; the next one's K (of `next`) is loaded under the second product
  auto tile = [&](int t, int next) {
    const int k0 = t * BKV;
    // V of key k0 + 8 (i / 4) + 4 h + i % 4: four neighbours lie in one page
    vf_t vf[NV][16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = k0 + 8 * j + 4 * h;
      const bool whole = key + 3 < sq.len;
      const float* row = (const float*)p.v + row_at(key) + VW * l31;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // past the end: the group's last valid row (masked; a value that no query sees
        // must not reach the product)
        const int step = whole ? e : max(0, min(key + e, sq.len - 1) - key);
#pragma unroll
        for (int n = 0; n < NV; ++n)
          vf[n][4 * j + e] = *reinterpret_cast<const vf_t*>(row + step * D + 32 * VW * n);
      }
    }
    f32x16_t s, s1;  // two chains of alternate chunks: less rounding in each
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = s1[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f32x16_t& a = j & 1 ? s1 : s;
        a = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j][e], qf[j][e], a, 0, 0, 0);
      }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] += s1[i];
    load_k(next);
    const int up = khi - k0 - 4 * h, dn = klo - k0 - 4 * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 8 * (i >> 2) + (i & 3);
      s[i] = key <= up && key >= dn ? s[i] : -INFINITY;
    }
    bool odd = false;  // a value that is not finite, where rows see different keys
    if (k0 + BKV - 1 > all_hi || k0 < all_lo) {  // (as in paged_attn_kernel)
      uint32_t seen = 0;  // the largest magnitude, as bits
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int u = 0; u < VW; ++u)
            seen = max(seen, __float_as_uint(vf[n][i][u]) & 0x7fffffffu);
      odd = __any(seen >= 0x7f800000u);
      if (odd)
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int u = 0; u < VW; ++u) {
              const float v = vf[n][i][u];
              vf[n][i][u] = fabsf(v) < INFINITY ? v : 0.f;
            }
    }
    float mt = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
    {
      float a, b;
      swap_pair<32>(mt, a, b);
      mt = fmaxf(a, b);
    }
    const float m_new = fmaxf(m, mt);
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f((m - mu) * c);
    m = m_new;
    float ls = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f((s[i] - mu) * c);
      ls += s[i];
    }
    l = l * alpha + ls;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[n][i] *= alpha;
    if (odd) {  // (behind the rescaling: the row's first tile has a factor of zero there)
      for (int j = 0; j < BKV; ++j) {
        const float* vrow = (const float*)p.v + row_at(k0 + j);
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v =
                vrow[VW * (8 * (i >> 2) + 4 * h + (i & 3)) + n % VW + 32 * VW * (n / VW)];
            oacc[n][i] += k0 + j <= khi && k0 + j >= klo && !(fabsf(v) < INFINITY) ? v : 0.f;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int n = 0; n < ND; ++n)
        oacc[n] =
            __builtin_amdgcn_mfma_f32_32x32x2f32(vf[n / VW][i][n % VW], s[i], oacc[n], 0, 0, 0);
  };
  // runs of tiles whose pages ptab holds
  const int run = ((PT - 1) << p.lps) / BKV;
  for (int ta = t0; ta < t1; ta += run) {
    const int tb = min(ta + run, t1);
    if (ta > t0) __syncthreads();
    wbase = (ta * BKV) >> p.lps;
    stage_pages(p, sq, wbase, ptab, tid, 256);
    __syncthreads();
    if (ta + w < tb) load_k(ta + w);
    for (int t = ta + w; t < tb; t += NW) tile(t, t + NW < tb ? t + NW : t);
  }

  // ---- the four waves' partial results ----
  {
    float a, b;
    swap_pair<32>(l, a, b);
    l = a + b;
  }
  if (h == 0) {
    sm[w][l31] = m;
    sl[w][l31] = l;
  }
  __syncthreads();
  float mx = sm[0][l31];
#pragma unroll
  for (int i = 1; i < NW; ++i) mx = fmaxf(mx, sm[i][l31]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  const float wt = __builtin_amdgcn_exp2f((m - mu) * c);
  float lt = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) lt += sl[i][l31] * __builtin_amdgcn_exp2f((sm[i][l31] - mu) * c);
  float* orow = so + (w * 32 + l31) * OP;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      vf_t x;
#pragma unroll
      for (int u = 0; u < VW; ++u) x[u] = oacc[n * VW + u][i] * wt;
      *reinterpret_cast<vf_t*>(orow + VW * (8 * (i >> 2) + 4 * h + (i & 3)) + 32 * VW * n) = x;
    }
  __syncthreads();
  if (w == 0 && h == 0) {
    sm[0][l31] = mx;
    sl[0][l31] = lt;
  }
  __syncthreads();
  const int nq = r1 - r0 + 1;
  const int64_t at = it.ns > 1 ? slot_of(it, it.split) * BQ : 0;
  for (int i = tid; i < nq * (D / 4); i += 256) {
    const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
    f32x4_t x[NW];
#pragma unroll
    for (int k = 0; k < NW; ++k)
      x[k] = *reinterpret_cast<const f32x4_t*>(so + (k * 32 + rr) * OP + cc);
    const f32x4_t sum = (x[0] + x[1]) + (x[2] + x[3]);
    const float tot = sl[0][rr];
    if (it.ns > 1) {
      put4(p.part + (at + rr) * D + cc, sum);
      if (cc == 0) put2(p.ml + (at + rr) * 2, sm[0][rr], tot);
    } else {
      const int t = over(r0 + rr, p.by_g), gg = (r0 + rr) - t * p.G;
      *reinterpret_cast<f32x4_t*>((float*)p.o + (int64_t)(sq.s0 + t) * p.st_o +
                                  (int64_t)(it.kvh * p.G + gg) * p.sh_o + cc) =
          tot == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sum / tot;
    }
  }
  if (it.ns > 1) join_parts<D, BQ, 256, float>(p, it, nq, so);
}

// ---- f32, tiles of rows ----------------------------------------------------------
// Many long chunks with d = 128, where the form above has one block a CU: as in
// paged_attn_kernel a block has 4 waves of 32 rows each that share key tiles (of 32 keys here)
// moved by LDS DMA through two stages, two blocks a CU, with the f32 products of the form
// above; a quarter of its reads of K and V, and nothing to merge.  32 / 8 heads: chunks of up
// to 107 tokens in 25 sequences 50 us (80 in the form above), of up to 1025 over up to 2045
// keys in two, window 300, 125 (182), 4 of up to 1024 265 (316).  With few row tiles their keys
// take too long one after the other (7 chunks of up to 566, 4 / 2 heads, 61 and 53), and with
// d = 64 the form above has two blocks a CU itself (10 of up to 400, 12 heads, 58 and 39).
// At 256 registers 91 values a lane stay in scratch memory, in the main loop (q's fragments,
// scores and outputs alone are 160).
__global__ __launch_bounds__(256, 2) void paged_attn_f32_tiles_kernel(KArgs p) {
  constexpr int D = 128, BKV = 32, QPW = 32, BQ = 4 * QPW, ND = D / 32, NC = D / 8;
  constexpr int TILE = BKV * D, STAGE = 2 * TILE, NST = 2;
  constexpr int CPR = D / 4, RPI = 64 / CPR, NI = 8 / RPI;  // chunks of a row; rows of a DMA
  constexpr int VW = 4, NV = ND / VW;                       // V's columns as in the form above
  typedef float vf_t __attribute__((ext_vector_type(VW)));
  __shared__ __attribute__((aligned(1024))) float lds[NST * STAGE];
  __shared__ int ptab[PT];

  Item it;
  if (!find_item<BQ, BKV>(p, blockIdx.x, it)) return;
  const Seq& sq = it.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  int lo, hi;
  const int r0 = it.rt * BQ, r1 = min(r0 + BQ, rows) - 1;
  key_range(p, sq, r0, r1, lo, hi);
  const int t_lo = lo / BKV, cnt = hi < 0 ? 0 : hi / BKV - t_lo + 1;
  int t0, t1;
  part_of(it, t_lo, cnt, t0, t1);
  // the wave's rows and keys
  const int rw = r0 + wid * QPW, rwl = min(rw + QPW, rows) - 1;
  const bool wave_active = rw < rows;
  int wlo = 0, whi = -1;
  if (wave_active) key_range(p, sq, rw, rwl, wlo, whi);
  const int pos_first = first + over(rw, p.by_g);
  const int lo_last = p.window ? first + over(rwl, p.by_g) - p.window + 1 : 0;

  const int row = min(rw + l31, rows - 1);
  const int tok = over(row, p.by_g), head = it.kvh * p.G + row - tok * p.G;
  const int khi = p.causal ? min(first + tok, sq.len - 1) : sq.len - 1;
  const int klo = p.window ? first + tok - p.window + 1 : 0;
  f32x4_t qf[NC];
  {
    const float* qrow =
        (const float*)p.q + (int64_t)(sq.s0 + tok) * p.st_q + (int64_t)head * p.sh_q;
#pragma unroll
    for (int j = 0; j < NC; ++j) qf[j] = *reinterpret_cast<const f32x4_t*>(qrow + 8 * j + 4 * h);
  }
  int wbase = (t0 * BKV) >> p.lps;
  if (t0 < t1) stage_pages(p, sq, wbase, ptab, tid, 256);
  // consumed here, before any DMA is in flight
#pragma unroll
  for (int j = 0; j < NC; ++j) asm volatile("" ::"v"(qf[j]));
  __syncthreads();

  // DMA.  Wave w moves keys 8 w .. 8 w + 7 of a tile (one page), RPI at a time.  16-byte
  // chunk c of K's row k is stored at c ^ (k & 15), so that 16 lanes' reads of one chunk
  // of 16 rows spread over all banks; V is read along its rows.
  const unsigned lds_base = (unsigned)(uintptr_t)lds;
  const int kin = lane / CPR, slot = lane % CPR;
  auto issue = [&](int t, int stage) {
    const int key0 = t * BKV + 8 * wid;
    const int kc = min(key0, (sq.len - 1) & ~7);  // the group that is read
    const int page = __builtin_amdgcn_readfirstlane(ptab[(kc >> p.lps) - wbase]);
    const int64_t off =
        (((((int64_t)page * p.Hkv + it.kvh) << p.lps) + (kc & ((1 << p.lps) - 1))) * D) * 4;
    const unsigned la = lds_base + (unsigned)(stage * STAGE + 8 * wid * D) * 4;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int k = kin + RPI * i;
      // rows past the end read the last key
      const int from = key0 + 8 <= sq.len ? k : min(key0 + k, sq.len - 1) - kc;
      const int kch = slot ^ ((8 * wid + k) & 15);
      dma16_so((const char*)p.k + off, (unsigned)(from * D * 4 + kch * 16), la + i * 1024);
      dma16_so((const char*)p.v + off, (unsigned)(from * D * 4 + slot * 16),
               la + TILE * 4 + i * 1024);
    }
  };
  f32x16_t o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = p.c;

  // operand reads are not moved over it: all of a tile's would not fit the registers
  auto some_at_once = [] { asm volatile("" ::: "memory"); };
  auto need = [&](int t) {  // (as in paged_attn_kernel)
    const int last = min(t * BKV + BKV - 1, sq.len - 1) >> p.lps;
    if (last >= wbase + PT) {
      wbase = (t * BKV) >> p.lps;
      stage_pages(p, sq, wbase, ptab, tid, 256);
      __syncthreads();
    }
  };
  if (t0 < t1) issue(t0, 0);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // tile t has landed and every wave is past tile t - 1, whose stage is free
    dma_wait_barrier<0>();
    if (t + 1 < t1) {
      need(t + 1);
      issue(t + 1, stage ^ 1);
    }
    const int kb = t * BKV;
    if (wave_active && kb <= whi && kb + BKV > wlo) {
      const float* sk = lds + stage * STAGE;
      const float* sv = sk + TILE;
      const bool mask = kb + BKV - 1 > (p.causal ? pos_first : sq.len - 1) ||
                        kb + BKV > sq.len || kb < lo_last;
      f32x16_t s, s1;  // two chains of alternate chunks: less rounding in each
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = s1[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const f32x4_t kf =
            *reinterpret_cast<const f32x4_t*>(sk + l31 * D + (((2 * j + h) ^ (l31 & 15)) << 2));
        f32x16_t& a = j & 1 ? s1 : s;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          a = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[j][e], a, 0, 0, 0);
        if ((j & 3) == 3) some_at_once();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] += s1[i];
      if (mask) {
        const int up = khi - kb - 4 * h, dn = klo - kb - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 8 * (i >> 2) + (i & 3);
          s[i] = key <= up && key >= dn ? s[i] : -INFINITY;
        }
      }
      float mt = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
      {
        float a, b;
        swap_pair<32>(mt, a, b);
        mt = fmaxf(a, b);
      }
      if (__any(mt > m)) {
        const float m_new = fmaxf(m, mt);
        const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[n][i] *= alpha;
      }
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f((s[i] - mu) * c);
        l += s[i];
      }
      // V of key kb + 8 (i / 4) + 4 h + i % 4
      auto v_at = [&](int i, int n) {
        return *reinterpret_cast<const vf_t*>(sv + (8 * (i >> 2) + 4 * h + (i & 3)) * D +
                                              VW * l31 + 32 * VW * n);
      };
      bool odd = false;  // a value that is not finite, where rows see different keys
      if (mask) {
        uint32_t seen = 0;  // the largest magnitude, as bits
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const vf_t x = v_at(i, n);
#pragma unroll
            for (int u = 0; u < VW; ++u) seen = max(seen, __float_as_uint(x[u]) & 0x7fffffffu);
          }
        odd = __any(seen >= 0x7f800000u);
      }
      if (!odd) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const vf_t x = v_at(i, n);
#pragma unroll
            for (int u = 0; u < VW; ++u)
              o[n * VW + u] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[u], s[i], o[n * VW + u], 0, 0, 0);
          }
          if ((i & 3) == 3) some_at_once();
        }
      } else {  // (as in paged_attn_kernel: added to the rows that see it, out of the product)
        for (int j = 0; j < BKV; ++j) {
          const bool sees = kb + j <= khi && kb + j >= klo;
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x =
                  sv[j * D + VW * (8 * (i >> 2) + 4 * h + (i & 3)) + n % VW + 32 * VW * (n / VW)];
              o[n][i] += sees && !(fabsf(x) < INFINITY) ? x : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const vf_t x = v_at(i, n);
#pragma unroll
            for (int u = 0; u < VW; ++u)
              o[n * VW + u] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                  fabsf(x[u]) < INFINITY ? x[u] : 0.f, s[i], o[n * VW + u], 0, 0, 0);
          }
      }
    }
    stage ^= 1;
  }

  float a, b;
  swap_pair<32>(l, a, b);
  float total = a + b;
  if (it.ns > 1 && !join_tiles<D>(p, it, wave_active, o, m, total)) return;
  if (rw + l31 < rows) {
    float* orow = (float*)p.o + (int64_t)(sq.s0 + tok) * p.st_o + (int64_t)head * p.sh_o;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        vf_t x;
#pragma unroll
        for (int u = 0; u < VW; ++u) x[u] = total == 0.f ? 0.f : o[n * VW + u][i] / total;
        *reinterpret_cast<vf_t*>(orow + VW * (8 * (i >> 2) + 4 * h + (i & 3)) + 32 * VW * n) = x;
      }
  }
}

// ---- launch ------------------------------------------------------------------------
enum Form { FORM_TILES, FORM_FEW16, FORM_FEW32, FORM_F32, FORM_F32_TILES };
struct Shape {
  Form form;
  int bq, bkv;
  int resident;  // blocks the chip holds at once
  int cmin;      // key tiles of the smallest part
  int spill;     // the row tiles may be just above one round
};
// resident: blocks the chip holds at once by their registers and LDS (f32 with d = 128: one
// per CU; with two assumed, 3 chunks of 100 tokens over 1500 keys, 32 / 8 heads, took 85 us
// instead of 68; tiles of 128 rows with d = 64 three, one chunk of 1473 over 8319 keys, 12
// heads, 69 us with two assumed and 62).  A counter for every row tile with parts: at most 2 * resident (two parts
// or more of each) or, with a spill, 1.5 * resident of them, <= BLT_CACHE_SYNC_WORDS.  The form goes by the rows a sequence has on average: a tile of 16 rows costs the
// matrix cores half of one of 32, and 128 rows share what they read; every form takes any
// chunk, in more row tiles (63 single tokens and a chunk of 900 over 4000 keys: 194 us in one
// call, 192 in two, 12 heads; 285 and 263, 32 / 8 heads of 128).
int64_t row_tiles(const blt_paged_cache& c, int64_t B, int64_t total, int H, int bq) {
  return total * (H / c.n_kv_heads) / bq + B;
}
// spill: 72 single tokens over 8000 keys, 32 / 8 heads of 128, are 576 row tiles for 512
// blocks: 590 us in two rounds, 432 in four; 96 over 4000 keys, 12 heads, 266 and 224.  From
// half a round more on it costs (128: 291 and 309), and in the form for 128 rows always
// (5 chunks of 512 over 8192 keys, 32 / 8 heads: 415 and 455).
Shape shape_of(const blt_paged_cache& c, int64_t B, int64_t total, int H) {
  const int64_t rows = total * (H / c.n_kv_heads);  // of all sequences, per key head
  const int few = c.head_dim == 64 ? 1024 : 512;  // 32 and 64 KB of rings
  Shape s{FORM_TILES, 128, 64, c.head_dim == 64 ? 768 : 512, 2, 0};
  // (enough of the larger row tiles for half the chip, with d = 128: see the form)
  if (c.dtype == BLT_DTYPE_F32 && c.head_dim == 128 && rows > 64 * B &&
      row_tiles(c, B, total, H, 128) * c.n_kv_heads >= 256)
    s = Shape{FORM_F32_TILES, 128, 32, 512, 4, 0};
  else if (c.dtype == BLT_DTYPE_F32) s = Shape{FORM_F32, 32, 32, few / 2, 4, 0};
  else if (rows <= 16 * B) s = Shape{FORM_FEW16, 16, 64, few, 2, 0};
  else if (rows <= 32 * B) s = Shape{FORM_FEW32, 32, 64, few, 2, 0};
  s.spill = s.bq < 128 && 5 * B * c.n_kv_heads <= 7 * s.resident &&
            row_tiles(c, B, total, H, s.bq) * c.n_kv_heads > s.resident;
  return s;
}
// Most parts a row tile can have: one for every cmin key tiles of a full sequence.
int64_t most_parts(const blt_paged_cache& c, const Shape& s) {
  const int64_t tiles = ((int64_t)c.max_pages * c.page_size + s.bkv - 1) / s.bkv;
  return (tiles + s.cmin - 1) / s.cmin;
}
// Bounds for what find_item makes of lengths that only the device knows: blocks, and
// slots for parts (none where no row tile can have two).
int64_t blocks_of(const blt_paged_cache& c, const Shape& s, int64_t B, int64_t total, int H) {
  const int64_t rt = row_tiles(c, B, total, H, s.bq) * c.n_kv_heads;
  const int64_t fill = (s.spill ? 4 : 2 * rt > s.resident ? 2 : 1) * (int64_t)s.resident;
  const int64_t most = most_parts(c, s);
  return most < 2 ? rt : rt * most < rt + fill ? rt * most : rt + fill;
}
int64_t slots_of(const blt_paged_cache& c, const Shape& s, int64_t B, int64_t total, int H) {
  const int64_t rt = row_tiles(c, B, total, H, s.bq) * c.n_kv_heads;
  const int64_t most = most_parts(c, s), all = (s.bq < 128 ? 8 : 4) * (int64_t)s.resident;
  return most < 2 ? 0 : rt * most < all ? rt * most : all;
}

template <int D>
int run_paged(const KArgs& p, const Shape& sh, unsigned nb, hipStream_t s) {
  const dim3 grid(nb), block(256);
  switch (sh.form) {
    case FORM_TILES:
      hipLaunchKernelGGL((paged_attn_kernel<D, 2>), grid, block, 0, s, p);
      break;
    case FORM_FEW16:
      hipLaunchKernelGGL((paged_attn_few_kernel<D, 1, 2>), grid, dim3(128), 0, s, p);
      break;
    case FORM_FEW32:
      hipLaunchKernelGGL((paged_attn_few_kernel<D, 2, 2>), grid, dim3(128), 0, s, p);
      break;
    case FORM_F32_TILES:
      hipLaunchKernelGGL(paged_attn_f32_tiles_kernel, grid, block, 0, s, p);
      break;
    default:
      hipLaunchKernelGGL((paged_attn_f32_kernel<D / 32>), grid, block, 0, s, p);
  }
  BLT_LAUNCH_CHECK("paged_attn_kernel");
  return 0;
}

}  // namespace

int64_t paged_attention_workspace_bytes(const blt_paged_cache& c, int64_t B, int64_t total,
                                        int H) {
  const Shape s = shape_of(c, B, total, H);
  return slots_of(c, s, B, total, H) * s.bq * (c.head_dim + 2) * 4;
}

int launch_paged_attention(const blt_paged_cache& c, const PagedAttnArgs& a, void* ws,
                           hipStream_t s) {
  Shape sh = shape_of(c, a.B, a.total, a.H);
  const int d = c.head_dim;
  KArgs p{};
  const int64_t es = c.dtype == BLT_DTYPE_BF16 ? 2 : 4;
  const int64_t layer = (int64_t)a.layer * c.num_pages * c.n_kv_heads * c.page_size * d * es;
  p.q = a.q; p.o = a.o;
  p.k = (const char*)c.k + layer; p.v = (const char*)c.v + layer;
  p.st_q = a.st_q; p.sh_q = a.sh_q; p.st_o = a.st_o; p.sh_o = a.sh_o;
  p.starts = a.starts; p.seqs = a.seqs; p.lens = c.lens; p.table = c.page_table;
  p.B = (int)a.B; p.total = (int)a.total; p.Hkv = c.n_kv_heads; p.G = a.H / c.n_kv_heads;
  p.by_g = divisor_of(p.G);
  p.tokens_max = sh.bq / p.G + 2;
  p.max_seqs = c.max_seqs; p.max_pages = c.max_pages; p.num_pages = c.num_pages;
  p.lps = log2_of(c.page_size); p.cap = c.max_pages * c.page_size;
  p.causal = a.causal; p.window = a.causal ? a.window : 0;
  if (p.window > (1 << 30)) p.window = 0;  // longer than any sequence
  p.c = (float)(1.44269504088896340736 * (double)a.scale);
  if (p.window && p.window < 24 * sh.bkv) sh.spill = 0;  // (too short: its blocks would only exit)
  p.resident = sh.resident; p.cmin = sh.cmin; p.spill = sh.spill;
  const int64_t slots = slots_of(c, sh, a.B, a.total, a.H);
  p.sync = c.sync; p.status = c.status;
  p.part = (float*)ws;
  p.ml = p.part + slots * sh.bq * d;
  const int64_t nb = (blocks_of(c, sh, a.B, a.total, a.H) + 7) / 8 * 8;
  if (nb > 0x7fffffff) return fail(BLT_ERR_SHAPE, "paged_attention: too many row tiles");
  return d == 64 ? run_paged<64>(p, sh, (unsigned)nb, s)
                 : run_paged<128>(p, sh, (unsigned)nb, s);
}

}  // namespace blt
