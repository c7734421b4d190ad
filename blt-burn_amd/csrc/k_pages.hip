// Page maintenance of the paged cache: reserve, trim, fork, compact, copy.
//
// All bookkeeping is on the device (page table, lengths, reference counts), so a
// decode step can grow, branch and drop sequences without the host.  What has to
// be decided in order (which free page goes to whom) is a block of 1024 threads
// walking the reference counts with a block scan: latency-bound, 4 us for a reserve of 24
// sequences in a pool of 1700 pages, an empty launch (2) among them.  Free pages are always taken lowest index first, so results
// do not depend on timing.  What moves data (page contents of every layer, the shared
// rows of the table) runs on many blocks: a fork's blocks each decide for themselves,
// from state that only the one that ends last writes; the others read a list that a
// first kernel made.
#include "paged.hpp"

namespace blt {

namespace {

constexpr int NT = 1024;     // threads of a bookkeeping block
constexpr int PER = 4;       // reference counts a thread reads per step
constexpr int LIST = 4096;   // free pages of one call held in LDS
constexpr int CLAIM = (int)0x80000000;  // sign bit of a length, while trim_split_kernel runs

// Workspace words: [0] number of copies; then three lists of `cap` words (source page,
// destination page, tokens to copy) and, for compact, the page map.
struct Lists {
  int32_t* count;
  int32_t *src, *dst, *fill, *map;
};
inline int64_t list_cap(const blt_paged_cache& c, int64_t n) {
  return n > 0 ? n : (int64_t)c.num_pages / 2 + 1;
}
inline Lists lists_of(const blt_paged_cache& c, int64_t n, void* ws) {
  int32_t* w = reinterpret_cast<int32_t*>(ws);
  const int64_t cap = list_cap(c, n);
  return Lists{w, w + 16, w + 16 + cap, w + 16 + 2 * cap, w + 16 + 3 * cap};
}

// Exclusive sum over the block's threads; `total` is the block's.  `part`: NT / 64 + 1
// words of LDS.  Two barriers.
__device__ inline int block_excl(int v, int* part, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int inc = wave_incl_scan(v);
  if (lane == 63) part[w] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    const int x = part[i];
    before += i < w ? x : 0;
    all += x;
  }
  __syncthreads();
  total = all;
  return before + inc - v;
}

struct Refs {
  int r[PER];
};
// reference counts of pages p .. p + PER - 1 (past the end: none free, none used)
template <bool FREE>
__device__ inline Refs load_refs(const int32_t* ref, int P, int p) {
  Refs x;
#pragma unroll
  for (int i = 0; i < PER; ++i) x.r[i] = p + i < P ? ref[p + i] : FREE ? 1 : 0;
  return x;
}
// Walk the reference counts in ascending order of page until f has been called for
// `most` free pages (or `used` ones, FREE false): f(page, ordinal).  Returns how many
// there were, at most those of the step that reached `most`.  x: the first step's.
template <bool FREE, typename F>
__device__ int walk_pages(const int32_t* ref, int P, int most, int* part, Refs x, F f) {
  int seen = 0;
  for (int p0 = 0; p0 < P && seen < most; p0 += NT * PER) {
    const int p = p0 + (int)threadIdx.x * PER;
    if (p0) x = load_refs<FREE>(ref, P, p);
    int hit[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      hit[i] = (FREE ? x.r[i] == 0 : x.r[i] != 0) ? 1 : 0;
      mine += hit[i];
    }
    int total;
    int at = seen + block_excl(mine, part, total);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (hit[i]) {
        if (at < most) f(p + i, at);
        ++at;
      }
    seen += total;
  }
  return seen;
}
template <bool FREE, typename F>
__device__ int walk_pages(const int32_t* ref, int P, int most, int* part, F f) {
  return walk_pages<FREE>(ref, P, most, part, load_refs<FREE>(ref, P, (int)threadIdx.x * PER), f);
}

// which sequences a call has named: a bit for each, in LDS
constexpr int kSeqWords = kMaxSeqs / 32;
__device__ inline bool named_before(uint32_t* bits, int s) {
  return atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1;
}
__device__ inline bool named(const uint32_t* bits, int s) { return bits[s >> 5] >> (s & 31) & 1; }

__device__ inline int pages_of(int tokens, int lps) {
  return (int)(((int64_t)tokens + (1 << lps) - 1) >> lps);
}

// ---- reserve -------------------------------------------------------------------
__global__ __launch_bounds__(NT) void reserve_kernel(blt_paged_cache c, int lps,
                                                     const int32_t* seqs, const int32_t* counts,
                                                     int n) {
  __shared__ int first[kPageListMax + 1];  // pages wanted by the entries before
  __shared__ int held[kPageListMax];       // pages an entry's sequence has
  __shared__ int list[LIST];
  __shared__ uint32_t bits[kSeqWords];
  __shared__ int part[NT / 64];
  __shared__ int bad;
  const int tid = threadIdx.x;
  const Refs refs = load_refs<true>(c.refcount, c.num_pages, tid * PER);
  // (in a register: `bad` takes the entries' errors as soon as the barrier is passed)
  const bool pending = *c.status & kCachePending;
  if (tid == 0) bad = 0;
  for (int i = tid; i < kSeqWords; i += NT) bits[i] = 0;
  __syncthreads();
  if (pending) return;
  int need_all = 0;
  for (int i0 = 0; i0 < n; i0 += NT) {
    const int i = i0 + tid;
    int need = 0, err = 0;
    if (i < n) {
      const int s = seqs ? seqs[i] : i, cnt = counts[i];
      if (s < 0 || s >= c.max_seqs || cnt < 0) {
        err = BLT_CACHE_BAD_INDEX;
      } else {
        const int len = c.lens[s];
        if (named_before(bits, s)) err = BLT_CACHE_BUSY;
        const int64_t want = ((int64_t)len + cnt + (1 << lps) - 1) >> lps;
        if (len < 0) err |= BLT_CACHE_BAD_INDEX;  // (a column before the sequence's row)
        else if (want > c.max_pages) err |= BLT_CACHE_TOO_LONG;
        else need = (int)want - pages_of(len, lps);
        held[i] = pages_of(len, lps);
      }
    }
    if (err) atomicOr(&bad, err);
    int total;
    const int at = block_excl(need, part, total);
    if (i < n) first[i] = need_all + at;
    // past any pool: too many for this call, and no overflow
    need_all = total > c.num_pages - need_all ? c.num_pages + 1 : need_all + total;
  }
  __syncthreads();
  // ordinal o of the new pages: the last entry with first[entry] <= o
  auto assign = [&](int page, int o) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= o) lo = mid; else hi = mid;
    }
    const int s = seqs ? seqs[lo] : lo;
    c.page_table[(int64_t)s * c.max_pages + held[lo] + o - first[lo]] = page;
    c.refcount[page] = 1;
  };
  if (!bad && need_all > 0) {
    const int have = walk_pages<true>(c.refcount, c.num_pages, need_all, part, refs,
                                      [&](int page, int o) { if (o < LIST) list[o] = page; });
    if (have < need_all && tid == 0) bad = BLT_CACHE_FULL;
    __syncthreads();
    if (!bad && need_all <= LIST)
      for (int o = tid; o < need_all; o += NT) assign(list[o], o);
    else if (!bad)
      walk_pages<true>(c.refcount, c.num_pages, need_all, part, refs, assign);
  }
  __syncthreads();
  if (bad) {
    if (tid == 0) atomicOr(c.status, bad);
  } else {
    for (int i = tid; i < n; i += NT) c.lens[seqs ? seqs[i] : i] += counts[i];
  }
}

// ---- copies --------------------------------------------------------------------
// The first `fill` tokens of a page in one layer's k or v, by 256 threads (this one is
// `tid`): 16 bytes a lane, four in flight.  Callers' grids walk (pair, layer, k or v, part):
// a few pages of more than 32 KB go in parts, so that they are not a few teams' work (one
// started 393 KB page in 14 layers: a fork of four, growth and drop 36 us in one part, 18 so).
// Whole pages (compaction, copy_pages) are moved past the caches: 400 MB of them take 167 us
// so and 175 us through the caches (6.15 TB/s is a large plain copy).  The started pages of a
// fork or a trim are read by the next step's attention and stay cached.
struct Parts {
  int n, pieces;  // parts of a page, 16-byte pieces of each
};
// pages: of one layer's k or v, to be copied
__host__ __device__ inline Parts page_parts(const blt_paged_cache& c, int64_t pages, int es) {
  const int pieces = c.n_kv_heads * (c.page_size * c.head_dim * es / 16);
  const int most = (pieces + 2047) / 2048;
  if (most == 1 || pages >= 1024) return Parts{1, pieces};
  const int n = pages < 1 ? most : 2048 / (int)pages;
  const int parts = n < most ? n : most;
  return Parts{parts, (pieces + parts - 1) / parts};
}
// Item `it` of a walk: its pair, layer, k or v, and first piece.
struct CopyItem {
  int64_t pair;
  int layer, kv, first;
};
__device__ inline CopyItem copy_item(int64_t it, int n_layers, const Parts& parts) {
  if (it >> 32) {  // (parts.n is 1 where there are so many)
    const int64_t pair = it / (n_layers * 2);
    const int r = (int)(it - pair * (n_layers * 2));
    return CopyItem{pair, r >> 1, r & 1, 0};
  }
  const uint32_t page = parts.n == 1 ? (uint32_t)it : (uint32_t)it / (uint32_t)parts.n;
  const uint32_t pair = page / (uint32_t)(n_layers * 2);
  const int r = (int)(page - pair * (n_layers * 2));
  return CopyItem{pair, r >> 1, r & 1, (int)((uint32_t)it - page * parts.n) * parts.pieces};
}
template <bool WHOLE>
__device__ inline void copy_rows(const char* from, char* to, int64_t head_b, int row, int first,
                                 int all, int tid) {
  auto off = [&](int i) -> int64_t {
    return WHOLE ? (int64_t)i * 16 : (i / row) * head_b + (int64_t)(i % row) * 16;
  };
  constexpr int U = 4;
  for (int i = first + tid; i < all; i += U * 256) {
    u32x4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * 256 < all) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(from + off(i + u * 256));
        x[u] = WHOLE ? __builtin_nontemporal_load(p) : *p;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * 256 < all) {
        u32x4_t* p = reinterpret_cast<u32x4_t*>(to + off(i + u * 256));
        if (WHOLE) __builtin_nontemporal_store(x[u], p);
        else *p = x[u];
      }
  }
}
template <bool WHOLE>
__device__ inline void copy_tokens(const blt_paged_cache& c, int64_t src, int64_t dst, int fill,
                                   const CopyItem& x, const Parts& parts, int es, int tid) {
  const int64_t page_b = (int64_t)c.n_kv_heads * c.page_size * c.head_dim * es;
  const int64_t head_b = (int64_t)c.page_size * c.head_dim * es;
  char* base =
      reinterpret_cast<char*>(x.kv ? c.v : c.k) + (int64_t)x.layer * c.num_pages * page_b;
  const char* from = base + src * page_b;
  char* to = base + dst * page_b;
  const int row = fill * c.head_dim * es / 16;  // 16-byte pieces of a head
  const int all = min(row * c.n_kv_heads, x.first + parts.pieces);
  copy_rows<WHOLE>(from, to, head_b, row, x.first, all, tid);
}
template <bool WHOLE>
__device__ inline void copy_listed(const blt_paged_cache& c, const Lists& l, int es) {
  const int64_t pages = (int64_t)*l.count * c.n_layers * 2;
  const Parts parts = page_parts(c, pages, es);
  const int64_t items = pages * parts.n;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const CopyItem x = copy_item(it, c.n_layers, parts);
    copy_tokens<WHOLE>(c, l.src[x.pair], l.dst[x.pair], WHOLE ? c.page_size : l.fill[x.pair], x,
                       parts, es, threadIdx.x);
  }
}
__global__ __launch_bounds__(256) void copy_list_kernel(blt_paged_cache c, Lists l, int es) {
  copy_listed<false>(c, l, es);
}
__global__ __launch_bounds__(256) void copy_pages_kernel(blt_paged_cache c, const int32_t* src,
                                                         const int32_t* dst, int64_t n, int es) {
  const Parts parts = page_parts(c, n * c.n_layers * 2, es);
  const int64_t items = n * c.n_layers * 2 * parts.n;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const CopyItem x = copy_item(it, c.n_layers, parts);
    const int a = src[x.pair], b = dst[x.pair];
    if (a < 0 || a >= c.num_pages || b < 0 || b >= c.num_pages) {
      if (threadIdx.x == 0 && x.layer + x.kv + x.first == 0)
        atomicOr(c.status, BLT_CACHE_BAD_INDEX);
      continue;
    }
    if (a != b) copy_tokens<true>(c, a, b, c.page_size, x, parts, es, threadIdx.x);
  }
}

// ---- fork ----------------------------------------------------------------------
// Every block decides for itself, from the lengths and reference counts as they were:
// the pages of the pairs whose source ends inside one, and whether the call can be carried
// out.  Then the blocks share the work: entries of the shared rows (their pages are in
// use, so the counts they raise change no decision) and the copies.  The block that ends
// last, behind all decisions, writes what they rest on: the new pages' counts and
// the lengths.  24 pairs of 14 layers take 10 us, 4 us less than a deciding kernel and a
// copying one.
__global__ __launch_bounds__(NT) void fork_kernel(blt_paged_cache c, int lps, const int32_t* src,
                                                  const int32_t* dst, int n, int es) {
  __shared__ int first[kPageListMax];  // partial pages of the pairs before
  __shared__ int list[kPageListMax];   // their new pages, old pages and tokens, by ordinal
  __shared__ int olds[kPageListMax];
  __shared__ short fills[kPageListMax];
  __shared__ uint32_t bits[kSeqWords];
  __shared__ int part[NT / 64];
  __shared__ int bad, last;
  const int tid = threadIdx.x, mask = c.page_size - 1;
  const Refs refs = load_refs<true>(c.refcount, c.num_pages, tid * PER);
  // (in a register, as in reserve_kernel; the status changes behind all blocks' reads)
  const bool pending = *c.status & kCachePending;
  if (tid == 0) bad = 0;
  for (int i = tid; i < kSeqWords; i += NT) bits[i] = 0;
  __syncthreads();
  auto page_at = [&](int s, int col) {
    const int page = c.page_table[(int64_t)s * c.max_pages + col];
    return page < 0 ? 0 : page < c.num_pages ? page : c.num_pages - 1;
  };
  int need_all = 0;
  if (!pending) {
    auto known = [&](int s) { return s >= 0 && s < c.max_seqs; };
    for (int i0 = 0; i0 < n; i0 += NT) {
      const int i = i0 + tid;
      int need = 0, err = 0, old = 0, fill = 0;
      if (i < n) {
        const int a = src[i], b = dst[i];
        if (!known(a) || !known(b)) {
          err = BLT_CACHE_BAD_INDEX;
        } else {
          if (named_before(bits, b) || c.lens[b] != 0) err = BLT_CACHE_BUSY;
          const int len = c.lens[a];
          if (len < 0 || pages_of(len, lps) > c.max_pages) {
            err |= BLT_CACHE_BAD_INDEX;
          } else {
            fill = len & mask;
            need = fill ? 1 : 0;
            if (fill) old = page_at(a, len >> lps);
          }
        }
      }
      if (err) atomicOr(&bad, err);
      int total;
      const int at = block_excl(need, part, total);
      if (i < n) first[i] = need_all + at;
      if (need) {
        olds[need_all + at] = old;
        fills[need_all + at] = (short)fill;
      }
      need_all += total;
    }
    __syncthreads();
    // no source may be a destination of the same call
    for (int i = tid; i < n; i += NT)
      if (known(src[i]) && named(bits, src[i])) atomicOr(&bad, BLT_CACHE_BUSY);
    int have = 0;
    if (need_all > 0)
      have = walk_pages<true>(c.refcount, c.num_pages, need_all, part, refs,
                              [&](int page, int o) { list[o] = page; });
    if (have < need_all && tid == 0) atomicOr(&bad, BLT_CACHE_FULL);
    __syncthreads();
  }
  const bool go = !pending && !bad;
  if (go) {
    const int64_t cols = c.max_pages;
    for (int64_t x = (int64_t)blockIdx.x * NT + tid; x < n * cols; x += (int64_t)gridDim.x * NT) {
      const int i = (int)(x / cols), col = (int)(x - i * cols);
      const int len = c.lens[src[i]];
      int page = -1;
      if (col < len >> lps) {
        page = page_at(src[i], col);
        atomicAdd(&c.refcount[page], 1);
      } else if (col == len >> lps && (len & mask)) {
        page = list[first[i]];
      }
      if (page >= 0) c.page_table[(int64_t)dst[i] * cols + col] = page;
    }
    const int64_t pages = (int64_t)need_all * c.n_layers * 2;  // four teams of 256 threads
    const Parts parts = page_parts(c, pages, es);
    const int64_t items = pages * parts.n;
    for (int64_t it = (int64_t)blockIdx.x * 4 + (tid >> 8); it < items;
         it += (int64_t)gridDim.x * 4) {
      const CopyItem x = copy_item(it, c.n_layers, parts);
      copy_tokens<false>(c, olds[x.pair], list[x.pair], fills[x.pair], x, parts, es, tid & 255);
    }
  }
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(c.sync, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(c.sync, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!go) {
    if (tid == 0 && !pending) atomicOr(c.status, bad);
    return;
  }
  for (int o = tid; o < need_all; o += NT) c.refcount[list[o]] = 1;
  for (int i = tid; i < n; i += NT) c.lens[dst[i]] = c.lens[src[i]];
}

// ---- trim ----------------------------------------------------------------------
// One block per entry.  atomicMin hands every entry the length before it, so a
// sequence listed twice frees each of its pages once.
__global__ __launch_bounds__(256) void trim_kernel(blt_paged_cache c, int lps, const int32_t* seqs,
                                                   const int32_t* lens) {
  __shared__ int old_len;
  const int i = blockIdx.x;
  const int s = seqs ? seqs[i] : i, want = lens ? lens[i] : 0;
  if (s < 0 || s >= c.max_seqs || want < 0) {
    if (threadIdx.x == 0) atomicOr(c.status, BLT_CACHE_BAD_INDEX);
    return;
  }
  if (threadIdx.x == 0) {
    old_len = atomicMin(&c.lens[s], want);
    if (old_len < 0) {  // no length: none from here on (trim_split_kernel uses the sign)
      atomicMax(&c.lens[s], 0);
      atomicOr(c.status, BLT_CACHE_BAD_INDEX);
    }
  }
  __syncthreads();
  int hi = pages_of(old_len, lps);
  if (hi > c.max_pages) hi = c.max_pages;
  for (int col = pages_of(want, lps) + threadIdx.x; col < hi; col += 256) {
    const int page = c.page_table[(int64_t)s * c.max_pages + col];
    if (page >= 0 && page < c.num_pages) atomicSub(&c.refcount[page], 1);
  }
}
// Sequences that now end inside a page that others use get a copy of it.  Those
// sharers that were cut into the same page in one call each get their own.
__global__ __launch_bounds__(NT) void trim_split_kernel(blt_paged_cache c, int lps,
                                                        const int32_t* seqs, int n, Lists l) {
  __shared__ int first[kPageListMax];  // splits of the entries before; -1: no split
  __shared__ int part[NT / 64];
  const int tid = threadIdx.x, mask = c.page_size - 1;
  auto entry = [&](int64_t s, int len) {
    const int page = c.page_table[s * c.max_pages + (len >> lps)];
    return page >= 0 && page < c.num_pages ? page : -1;
  };
  int need_all = 0;
  for (int i0 = 0; i0 < n; i0 += NT) {
    const int i = i0 + tid;
    int need = 0;
    if (i < n) {
      const int s = seqs ? seqs[i] : i;
      if (s >= 0 && s < c.max_seqs) {
        const int old = atomicOr(&c.lens[s], CLAIM);
        if (!(old & CLAIM) && (old & mask) && (old >> lps) < c.max_pages) {
          const int page = entry(s, old);
          need = page >= 0 && c.refcount[page] > 1 ? 1 : 0;
        }
      }
    }
    int total;
    const int at = block_excl(need, part, total);
    if (i < n) first[i] = need ? need_all + at : -1;
    need_all += total;
  }
  __syncthreads();
  int have = 0;
  if (need_all > 0)
    have = walk_pages<true>(c.refcount, c.num_pages, need_all, part,
                            [&](int page, int o) { l.dst[o] = page; });
  if (have > need_all) have = need_all;
  __syncthreads();
  for (int o = tid; o < have; o += NT) c.refcount[l.dst[o]] = 1;
  for (int i = tid; i < n; i += NT) {
    const int o = first[i];
    if (o < 0) continue;
    const int s = seqs ? seqs[i] : i;
    const int len = c.lens[s] & ~CLAIM;
    const int page = entry(s, len);
    atomicSub(&c.refcount[page], 1);
    if (o < have) {
      l.src[o] = page;
      l.fill[o] = len & mask;
      c.page_table[(int64_t)s * c.max_pages + (len >> lps)] = l.dst[o];
    } else {
      atomicExch(&c.lens[s], (len & ~mask) | CLAIM);
    }
  }
  if (tid == 0) {
    *l.count = have;
    if (have < need_all) atomicOr(c.status, BLT_CACHE_FULL);
  }
  __syncthreads();
  for (int i = tid; i < n; i += NT) {
    const int s = seqs ? seqs[i] : i;
    if (s >= 0 && s < c.max_seqs) atomicAnd(&c.lens[s], ~CLAIM);
  }
}

// ---- compact -------------------------------------------------------------------
// With n pages in use, the used ones at n and above move into the free ones below, both
// ascending.  As in a fork every block decides for itself and the last one writes the
// counts.  The lists are in LDS where the pool is small enough (FIT: one launch); for
// larger ones compact_kernel writes them, and the map of the pages, for compact_copy_kernel.
// 400 MB of pages move in 165 us, 4.9 TB/s.
constexpr int FIT = 8192;  // pairs whose lists fit: pools of up to twice as many pages
// f(page, ordinal) of the holes, g of the movers; returns how many, and n
template <typename F, typename G>
__device__ int find_pairs(const blt_paged_cache& c, int* part, int& live, F f, G g) {
  const int P = c.num_pages;
  live = walk_pages<false>(c.refcount, P, P, part, [](int, int) {});
  const int holes = walk_pages<true>(c.refcount, live, P, part, f);
  const int n = live;
  walk_pages<false>(c.refcount + n, P - n, P, part, [&](int page, int o) { g(page + n, o); });
  return holes;
}
__global__ __launch_bounds__(NT) void compact_fit_kernel(blt_paged_cache c, int lps, int es) {
  __shared__ int hole[FIT], mover[FIT];
  __shared__ int part[NT / 64];
  __shared__ int last;
  const int tid = threadIdx.x;
  int live;
  const int pairs = find_pairs(
      c, part, live, [&](int page, int o) { hole[o] = page; },
      [&](int page, int o) { mover[o] = page; });
  __syncthreads();
  if (pairs > 0) {
    const int64_t cols = c.max_pages, threads = (int64_t)gridDim.x * NT;
    for (int64_t x = (int64_t)blockIdx.x * NT + tid; x < c.max_seqs * cols; x += threads) {
      const int64_t s = x / cols;
      if (x - s * cols >= pages_of(c.lens[s], lps)) continue;
      const int page = c.page_table[x];
      if (page < live) continue;
      int lo = 0, hi = pairs;  // mover[lo] <= page
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (mover[mid] <= page) lo = mid; else hi = mid;
      }
      if (mover[lo] == page) c.page_table[x] = hole[lo];
    }
    const int64_t pages = (int64_t)pairs * c.n_layers * 2;  // four teams of 256 threads
    const Parts parts = page_parts(c, pages, es);
    const int64_t items = pages * parts.n;
    for (int64_t it = (int64_t)blockIdx.x * 4 + (tid >> 8); it < items;
         it += (int64_t)gridDim.x * 4) {
      const CopyItem x = copy_item(it, c.n_layers, parts);
      copy_tokens<true>(c, mover[x.pair], hole[x.pair], c.page_size, x, parts, es, tid & 255);
    }
  }
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(c.sync, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(c.sync, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int o = tid; o < pairs; o += NT) {
    c.refcount[hole[o]] = c.refcount[mover[o]];
    c.refcount[mover[o]] = 0;
  }
}
__global__ __launch_bounds__(NT) void compact_kernel(blt_paged_cache c, Lists l) {
  __shared__ int part[NT / 64];
  const int tid = threadIdx.x;
  int live;
  const int pairs = find_pairs(
      c, part, live, [&](int page, int o) { l.dst[o] = page; },
      [&](int page, int o) { l.src[o] = page; });
  __syncthreads();
  for (int o = tid; o < pairs; o += NT) {
    const int from = l.src[o], to = l.dst[o];
    c.refcount[to] = c.refcount[from];
    c.refcount[from] = 0;
    l.map[from] = to;
  }
  if (tid == 0) {
    l.count[0] = pairs;
    l.count[1] = live;
  }
}
__global__ __launch_bounds__(256) void compact_copy_kernel(blt_paged_cache c, int lps, Lists l,
                                                           int es) {
  if (*l.count == 0) return;
  const int live = l.count[1];
  const int64_t threads = (int64_t)gridDim.x * 256, cols = c.max_pages;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < c.max_seqs * cols; x += threads) {
    const int64_t s = x / cols;
    if (x - s * cols >= pages_of(c.lens[s], lps)) continue;
    const int page = c.page_table[x];
    if (page >= live && page < c.num_pages) c.page_table[x] = l.map[page];
  }
  copy_listed<true>(c, l, es);
}

constexpr int kCopyBlocks = 2048;  // eight 256-thread blocks on each of 256 CUs

// ---- common prefix -----------------------------------------------------------------
// Whole pages that all listed sequences with tokens have in common, in tokens (0 with fewer than
// two of them).  One block, once a step: what it costs are the rounds of loads (48 sequences of 512 pages,
// 100 KB: a thread has 24 entries).
__global__ __launch_bounds__(NT) void common_prefix_kernel(blt_paged_cache c, int lps,
                                                           const int32_t* seqs, int n,
                                                           int32_t* tokens) {
  __shared__ int full, count, first, bad, slots[NT];
  const int tid = threadIdx.x;
  if (tid == 0) {
    full = c.max_pages;
    count = 0;
    first = n;
    bad = 0;
  }
  __syncthreads();
  // the sequence of entry i, -1 if it has no tokens; *pages: its whole pages
  auto slot_at = [&](int i, int* pages) {
    const int s = seqs ? seqs[i] : i;
    const bool known = s >= 0 && s < c.max_seqs;
    const int len = known ? c.lens[s] : 0;
    if (!known) atomicOr(&bad, 1);
    *pages = len >> lps;
    return len > 0 ? s : -1;
  };
  for (int i = tid; i < n; i += NT) {
    int pages;
    if (slot_at(i, &pages) >= 0) {
      atomicMin(&full, pages);
      atomicAdd(&count, 1);
      atomicMin(&first, i);
    }
  }
  __syncthreads();
  if (bad || count < 2) {
    if (tid == 0) {
      tokens[0] = 0;
      if (bad) atomicOr(c.status, BLT_CACHE_BAD_INDEX);
    }
    return;
  }
  const int32_t* own = c.page_table + (int64_t)(seqs ? seqs[first] : first) * c.max_pages;
  // 1024 sequences at a time, a thread has entries (sequence, column) of all of them
  for (int i0 = 0; i0 < n; i0 += NT) {
    int pages;
    __syncthreads();
    slots[tid] = i0 + tid < n ? slot_at(i0 + tid, &pages) : -1;
    // (the same for all threads, which divide the entries by it: read before the barrier, behind
    // which `full` may shrink; what lies behind does not matter then)
    const int cols = full;
    __syncthreads();
    const int64_t all = (int64_t)min(NT, n - i0) * cols;
    int j = cols ? tid / cols : 0, at = cols ? tid - j * cols : 0;
    const int dj = cols ? NT / cols : 0, dat = cols ? NT - dj * cols : 0;
    constexpr int U = 16;  // entries in flight
    for (int64_t e = tid; e < all; e += (int64_t)U * NT) {
      int x[U], y[U], col[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = e + (int64_t)u * NT < all ? slots[j] : -1;
        col[u] = at;
        x[u] = s < 0 ? 0 : own[at];
        y[u] = s < 0 ? 0 : c.page_table[(int64_t)s * c.max_pages + at];
        j += dj;
        at += dat;
        if (at >= cols) {
          at -= cols;
          ++j;
        }
        j = min(j, NT - 1);
      }
      int most = 0x7fffffff;
#pragma unroll
      for (int u = 0; u < U; ++u) most = x[u] != y[u] ? min(most, col[u]) : most;
      if (most != 0x7fffffff) atomicMin(&full, most);
    }
  }
  __syncthreads();
  if (tid == 0) tokens[0] = full << lps;
}

}  // namespace

int64_t cache_workspace_bytes(const blt_paged_cache& c, int64_t n) {
  if (n == 0 && c.num_pages <= 2 * FIT) return 0;
  return (16 + 3 * list_cap(c, n) + (n > 0 ? 0 : (int64_t)c.num_pages)) * 4;
}

int launch_cache_reserve(const blt_paged_cache& c, const int32_t* seqs, const int32_t* counts,
                         int64_t n, hipStream_t s) {
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(NT), 0, s, c, log2_of(c.page_size), seqs,
                     counts, (int)n);
  BLT_LAUNCH_CHECK("reserve_kernel");
  return 0;
}

inline int elem_size(const blt_paged_cache& c) { return c.dtype == BLT_DTYPE_BF16 ? 2 : 4; }
inline unsigned copy_blocks(const blt_paged_cache& c, int64_t pairs) {
  // (at most `pairs`: fewer may be cut into more parts)
  const int64_t items = pairs * c.n_layers * 2 * page_parts(c, 1, elem_size(c)).n;
  return (unsigned)(items < 1 ? 1 : items < kCopyBlocks ? items : kCopyBlocks);
}

int launch_cache_trim(const blt_paged_cache& c, const int32_t* seqs, const int32_t* lens,
                      int64_t n, void* ws, hipStream_t s) {
  const int lps = log2_of(c.page_size);
  hipLaunchKernelGGL(trim_kernel, dim3((unsigned)n), dim3(256), 0, s, c, lps, seqs, lens);
  BLT_LAUNCH_CHECK("trim_kernel");
  if (lens == nullptr) return 0;
  const Lists l = lists_of(c, n, ws);
  hipLaunchKernelGGL(trim_split_kernel, dim3(1), dim3(NT), 0, s, c, lps, seqs, (int)n, l);
  BLT_LAUNCH_CHECK("trim_split_kernel");
  hipLaunchKernelGGL(copy_list_kernel, dim3(copy_blocks(c, n)), dim3(256), 0, s, c, l,
                     elem_size(c));
  BLT_LAUNCH_CHECK("copy_list_kernel");
  return 0;
}

int launch_cache_fork(const blt_paged_cache& c, const int32_t* src, const int32_t* dst, int64_t n,
                      hipStream_t s) {
  const unsigned nb = (copy_blocks(c, n) + 3) / 4;
  hipLaunchKernelGGL(fork_kernel, dim3(nb < 256 ? nb : 256), dim3(NT), 0, s, c,
                     log2_of(c.page_size), src, dst, (int)n, elem_size(c));
  BLT_LAUNCH_CHECK("fork_kernel");
  return 0;
}

int launch_cache_compact(const blt_paged_cache& c, void* ws, hipStream_t s) {
  if (c.num_pages <= 2 * FIT) {
    const unsigned nb = (copy_blocks(c, c.num_pages / 2) + 3) / 4;
    hipLaunchKernelGGL(compact_fit_kernel, dim3(nb < 512 ? nb : 512), dim3(NT), 0, s, c,
                       log2_of(c.page_size), elem_size(c));
    BLT_LAUNCH_CHECK("compact_fit_kernel");
    return 0;
  }
  const Lists l = lists_of(c, 0, ws);
  hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(NT), 0, s, c, l);
  BLT_LAUNCH_CHECK("compact_kernel");
  hipLaunchKernelGGL(compact_copy_kernel, dim3(copy_blocks(c, c.num_pages / 2)), dim3(256), 0, s, c,
                     log2_of(c.page_size), l, elem_size(c));
  BLT_LAUNCH_CHECK("compact_copy_kernel");
  return 0;
}

int launch_cache_common_prefix(const blt_paged_cache& c, const int32_t* seqs, int64_t n,
                               int32_t* tokens, hipStream_t s) {
  hipLaunchKernelGGL(common_prefix_kernel, dim3(1), dim3(NT), 0, s, c, log2_of(c.page_size), seqs,
                     (int)n, tokens);
  BLT_LAUNCH_CHECK("common_prefix_kernel");
  return 0;
}

int launch_cache_copy_pages(const blt_paged_cache& c, const int32_t* src, const int32_t* dst,
                            int64_t n, hipStream_t s) {
  hipLaunchKernelGGL(copy_pages_kernel, dim3(copy_blocks(c, n)), dim3(256), 0, s, c, src, dst, n,
                     elem_size(c));
  BLT_LAUNCH_CHECK("copy_pages_kernel");
  return 0;
}

}  // namespace blt
