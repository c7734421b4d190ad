// Attention of a chunk of new tokens per sequence over the paged cache: one pass
// over the keys with a running max and sum, head_dim 64 or 128, grouped heads, any
// chunk length from one token up.
//
// Rows and items.  The query heads that share a key head are packed with the tokens
// into rows (row = token * G + head), so one key tile serves all of them and a
// single token with grouped heads still fills matrix rows.  An item is a row tile of
// one (sequence, key head) and, where the call has too few of them to fill the chip, a
// part of its keys; the parts' unnormalised outputs meet in combine_kernel.  Lengths
// live on the device (the call can be captured and replayed as they grow), so every wave
// works out its item itself: the number of key tiles an item may have (C) follows from
// the total work, then a scan over the sequences finds the item of a block.  The host
// only bounds the grid: items <= target + row tiles, parts in need of
// joining <= 2 * target (every one of them has more than half of C).
#include <type_traits>

#include "paged.hpp"

namespace blt {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
#define LDS_PTR(p) ((__attribute__((address_space(3))) s16x4_t*)(p))

struct KArgs {
  const void *q, *k, *v;  // k, v: the layer's first element
  void* o;
  int64_t st_q, sh_q, st_o, sh_o;
  const int32_t *starts, *seqs, *lens, *table;
  int B, total, H, Hkv, G;
  int max_seqs, max_pages, num_pages, lps, cap;  // cap: tokens max_pages hold
  int causal, window;                            // window 0: none
  float c;        // log2(e) * scale
  int target, cmin;
  float* part;    // [slots][rows of a tile][D], unnormalised outputs
  float* ml;      // [slots][rows of a tile][2], their max (before the scale) and sum
};

// ---- which item ----------------------------------------------------------------

struct Seq {
  int s0, n, len, slot;  // first token in q, tokens, keys, sequence
};
__device__ inline Seq seq_at(const KArgs& p, int b) {
  Seq q{0, 0, 0, 0};
  if (b < p.B) {
    const int a = p.starts[b], e = p.starts[b + 1];
    const int slot = p.seqs ? p.seqs[b] : b;
    if (a >= 0 && e > a && e <= p.total && slot >= 0 && slot < p.max_seqs) {
      int len = p.lens[slot];
      len = len < 0 ? 0 : len > p.cap ? p.cap : len;
      q = Seq{a, e - a, len, slot};
    }
  }
  return q;
}
// row tiles of a sequence, and the key tiles one of them may have to read
template <int BQ, int BKV>
__device__ inline void tiles_of(const KArgs& p, const Seq& q, int& nrt, int& kt) {
  nrt = (int)(((int64_t)q.n * p.G + BQ - 1) / BQ);
  kt = (q.len + BKV - 1) / BKV;
  if (p.window) {
    const int tokens = q.n < BQ / p.G + 2 ? q.n : BQ / p.G + 2;
    const int most = (p.window + tokens + BKV - 2) / BKV + 1;
    kt = kt < most ? kt : most;
  }
  kt = kt < 1 ? 1 : kt;
}
struct Item {
  Seq q;
  int kvh, rt, split, ns;  // key head, row tile, part and number of parts
  int nrt, pslot;          // row tiles of the sequence; first partial slot of the sequence
};
__device__ inline int lane_of(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// The item of block `bid`, false if it has none.  JOIN: the row tiles whose parts have
// to be joined instead.  Every wave computes it by itself, in the same order, so all
// agree.
template <int BQ, int BKV, bool JOIN>
__device__ bool find_item(const KArgs& p, unsigned bid, Item& it) {
  const int lane = threadIdx.x & 63;
  Seq q;
  int nrt, kt;
  float work = 0.f;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    q = seq_at(p, b0 + lane);
    tiles_of<BQ, BKV>(p, q, nrt, kt);
    work += (float)nrt * (float)kt;
  }
  work = wave_sum(work) * (float)p.Hkv;
  // (0.1 % above the exact quotient: the bounds on the grid and the slots hold
  // whatever the rounding of the sums)
  const int C = max(p.cmin, (int)fminf(ceilf(work * (1.001f / (float)p.target)), 1e9f));
  auto counts = [&](int& ns, int& items, int& parts) {
    ns = (kt + C - 1) / C;
    items = JOIN ? (ns > 1 ? nrt * p.Hkv : 0) : nrt * ns * p.Hkv;
    parts = ns > 1 ? nrt * ns * p.Hkv : 0;
  };
  int ns, items, parts;
  int id = (int)bid;
  if constexpr (!JOIN) {
    // dispatch places block i on XCD i % 8: each XCD takes a contiguous run of items, so
    // the row tiles of one key head share its L2
    int mine = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      if (p.B > 64) {
        q = seq_at(p, b0 + lane);
        tiles_of<BQ, BKV>(p, q, nrt, kt);
      }
      counts(ns, items, parts);
      mine += items;
    }
    const int all = lane_of(wave_incl_scan(mine), 63);
    const int per = (all + 7) >> 3;
    id = (int)(bid & 7) * per + (int)(bid >> 3);
    if ((int)(bid >> 3) >= per || id >= all) return false;
  }
  int base = 0, pbase = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (p.B > 64) {
      q = seq_at(p, b0 + lane);
      tiles_of<BQ, BKV>(p, q, nrt, kt);
    }
    counts(ns, items, parts);
    const int inc = wave_incl_scan(items), pinc = wave_incl_scan(parts);
    const uint64_t above = __ballot(base + inc > id);
    if (above) {
      const int l = __ffsll((unsigned long long)above) - 1;
      it.q = Seq{lane_of(q.s0, l), lane_of(q.n, l), lane_of(q.len, l), lane_of(q.slot, l)};
      it.nrt = lane_of(nrt, l);
      it.ns = lane_of(ns, l);
      it.pslot = pbase + lane_of(pinc - parts, l);
      int at = id - (base + lane_of(inc - items, l));
      it.rt = it.nrt - 1 - at % it.nrt;  // the longest causal rows first
      at /= it.nrt;
      it.split = JOIN ? 0 : at % it.ns;
      it.kvh = JOIN ? at : at / it.ns;
      return true;
    }
    base += lane_of(inc, 63);
    pbase += lane_of(pinc, 63);
  }
  return false;
}
__device__ inline int64_t slot_of(const Item& it, int split) {
  return it.pslot + ((int64_t)it.kvh * it.ns + split) * it.nrt + it.rt;
}

// The keys rows r0 .. r1 (of one sequence) see between them: [lo, hi].
__device__ inline void key_range(const KArgs& p, const Seq& q, int r0, int r1, int& lo, int& hi) {
  const int first = q.len - q.n;  // position of token 0
  hi = q.len - 1;
  lo = 0;
  if (p.causal) {
    const int last = first + r1 / p.G;
    hi = last < hi ? last : hi;
    if (p.window) {
      const int l = first + r0 / p.G - p.window + 1;
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

// ---- bf16, tiles of rows ---------------------------------------------------------
// One block = 4 waves of 32 NQ rows each; key tiles of 64 keys go global -> LDS by DMA
// through NST stages shared by the waves.  As in attn_fwd_kernel the scores are taken
// transposed, S^T = K . Q^T, so a lane owns one row: its max and sum need one
// cross-lane step, P^T feeds the second product from registers, and V's operand is
// read with the LDS transposing read.  Unlike there q keeps its own bf16 values (scaling it
// before its rounding costs as much accuracy as the output's rounding): the scores come
// out of the matrix core minus the running max, and the scale is one multiply before exp2.
template <int D, int NQ, int NST>
__global__ __launch_bounds__(256) void paged_attn_kernel(KArgs p) {
  constexpr int BKV = 64, QPW = 32 * NQ, BQ = 4 * QPW;
  constexpr int TILE = BKV * D;        // elements of a K (or V) tile
  constexpr int STAGE = 2 * TILE;
  constexpr int NOP = 4 * (D / 64);    // DMA instructions of a wave per tile
  constexpr int KS = D / 16, DS = D / 32;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[NST * STAGE];
  __shared__ int ptab[PT];

  Item it;
  if (!find_item<BQ, BKV, false>(p, blockIdx.x, it)) return;
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
  const int t0 = t_lo + (int)((int64_t)cnt * it.split / it.ns);
  const int t1 = t_lo + (int)((int64_t)cnt * (it.split + 1) / it.ns);
  // the wave's
  const int rw = r0 + wid * QPW;
  const bool wave_active = rw < rows;
  int wlo = 0, whi = -1;
  const int rwl = min(rw + QPW, rows) - 1;
  if (wave_active) key_range(p, sq, rw, rwl, wlo, whi);
  const int pos_first = first + rw / p.G;  // lowest position in the wave
  const int lo_last = p.window ? first + rwl / p.G - p.window + 1 : 0;  // highest lower bound

  // Q fragments (B operand): row rw + 32 qq + lrow, d = 16 ks + 8 lhalf .. + 8
  bf16x8_t qf[NQ][KS];
  int klo[NQ], khi[NQ];  // the row's visible keys
#pragma unroll
  for (int qq = 0; qq < NQ; ++qq) {
    const int r = min(rw + 32 * qq + lrow, rows - 1);
    const int t = r / p.G, g = r - t * p.G;
    const uint16_t* qrow = (const uint16_t*)p.q + (int64_t)(sq.s0 + t) * p.st_q +
                           (int64_t)(it.kvh * p.G + g) * p.sh_q;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[qq][ks] = __builtin_bit_cast(
          bf16x8_t, *reinterpret_cast<const u32x4_t*>(qrow + ks * 16 + lhalf * 8));
    khi[qq] = p.causal ? min(first + t, sq.len - 1) : sq.len - 1;
    klo[qq] = p.window ? first + t - p.window + 1 : 0;
  }
  // consumed here, before any DMA is in flight (see attn_fwd_kernel)
#pragma unroll
  for (int qq = 0; qq < NQ; ++qq)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[qq][ks]));

  int wbase = (t0 * BKV) >> p.lps;
  if (t0 < t1) stage_pages(p, sq, wbase, ptab, tid, 256);
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

  f32x16_t o[NQ][DS], negm[NQ];
  float m[NQ], mu[NQ], l[NQ];
#pragma unroll
  for (int qq = 0; qq < NQ; ++qq) {
    m[qq] = -INFINITY;
    mu[qq] = 0.f;
    l[qq] = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) negm[qq][r] = 0.f;
#pragma unroll
    for (int j = 0; j < DS; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[qq][j][r] = 0.f;
  }
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
      f32x16_t s[NQ][2];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const bf16x8_t a = *reinterpret_cast<const bf16x8_t*>(
              sk + (sub * 32 + lrow) * D + (((2 * ks + lhalf) ^ kswz) << 3));
#pragma unroll
          for (int qq = 0; qq < NQ; ++qq)
            s[qq][sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                a, qf[qq][ks], ks == 0 ? negm[qq] : s[qq][sub], 0, 0, 0);
        }
      const bool mask_hi = kb + BKV - 1 > (p.causal ? pos_first : sq.len - 1) ||
                           kb + BKV > sq.len;
      const bool mask_lo = p.window && kb < lo_last;
      bf16x8_t pb[NQ][2][2];
#pragma unroll
      for (int qq = 0; qq < NQ; ++qq) {
        if (mask_hi) {
          const int rel = khi[qq] - kb - 4 * lhalf;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[qq][sub][r] = sub * 32 + 8 * (r >> 2) + (r & 3) <= rel ? s[qq][sub][r] : -INFINITY;
        }
        if (mask_lo) {
          const int rel = klo[qq] - kb - 4 * lhalf;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[qq][sub][r] = sub * 32 + 8 * (r >> 2) + (r & 3) >= rel ? s[qq][sub][r] : -INFINITY;
        }
        float mt = -INFINITY;  // this tile's max, relative to mu
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[qq][sub][r]);
        {
          float a, b;
          swap_pair<32>(mt, a, b);
          mt = fmaxf(a, b);
        }
        // the offset mu moves only when the max grows by more than 2^8 over it
        const bool grow = mt > grow_at || (m[qq] == -INFINITY && mt > -INFINITY);
        if (__any(grow)) {
          const float m_new = fmaxf(m[qq], mt + mu[qq]);
          const float alpha =
              m[qq] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mu[qq] - m_new) * c);
          m[qq] = m_new;
          const float mu_new = m_new == -INFINITY ? 0.f : m_new;
          const float shift = mu_new - mu[qq];
          mu[qq] = mu_new;
          l[qq] *= alpha;
#pragma unroll
          for (int j = 0; j < DS; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[qq][j][r] *= alpha;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[qq][sub][r] -= shift;
#pragma unroll
          for (int r = 0; r < 16; ++r) negm[qq][r] = -mu_new;
        }
        float ls = l[qq];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float p0 = __builtin_amdgcn_exp2f(s[qq][sub][8 * u + e] * c);
              const float p1 = __builtin_amdgcn_exp2f(s[qq][sub][8 * u + e + 1] * c);
              w[e >> 1] = pack_bf16x2(p0, p1);
              ls = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[e >> 1]), ones2,
                                                   ls, false);
            }
            pb[qq][sub][u] = __builtin_bit_cast(bf16x8_t, u32x4_t{w[0], w[1], w[2], w[3]});
          }
        l[qq] = ls;
      }
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
            const bf16x8_t a = __builtin_bit_cast(bf16x8_t, u32x4_t{w0.x, w0.y, w1.x, w1.y});
#pragma unroll
            for (int qq = 0; qq < NQ; ++qq)
              o[qq][ds] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb[qq][sub][u], o[qq][ds], 0, 0, 0);
          }
    }
    stage = stage + 1 < NST ? stage + 1 : 0;
  }

  if (!wave_active) return;
#pragma unroll
  for (int qq = 0; qq < NQ; ++qq) {
    float a, b;
    swap_pair<32>(l[qq], a, b);
    const float lt = a + b;
    const int r = rw + 32 * qq + lrow;
    if (r >= rows) continue;
    if (it.ns > 1) {
      const int64_t at = slot_of(it, it.split) * BQ + (r - r0);
      float* dst = p.part + at * D;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4_t*>(dst + ds * 32 + 8 * j + 4 * lhalf) =
              f32x4_t{o[qq][ds][4 * j], o[qq][ds][4 * j + 1], o[qq][ds][4 * j + 2],
                      o[qq][ds][4 * j + 3]};
      if (lhalf == 0) {
        p.ml[at * 2] = m[qq] == -INFINITY ? -INFINITY : mu[qq];
        p.ml[at * 2 + 1] = lt;
      }
    } else {
      const int t = r / p.G, g = r - t * p.G;
      uint16_t* orow = (uint16_t*)p.o + (int64_t)(sq.s0 + t) * p.st_o +
                       (int64_t)(it.kvh * p.G + g) * p.sh_o;
      // hardware reciprocal (1 ulp): the output is rounded to bf16
      const float inv = lt > 0.f ? __builtin_amdgcn_rcpf(lt) : lt == lt ? 0.f : lt;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u32x2_t w;
          w.x = pack_bf16x2(o[qq][ds][4 * j] * inv, o[qq][ds][4 * j + 1] * inv);
          w.y = pack_bf16x2(o[qq][ds][4 * j + 2] * inv, o[qq][ds][4 * j + 3] * inv);
          *reinterpret_cast<u32x2_t*>(orow + ds * 32 + 8 * j + 4 * lhalf) = w;
        }
    }
  }
}

// ---- f32 -------------------------------------------------------------------------
// As attn_f32_kernel (k_attn.hip): both products on the f32 matrix cores, one block = 32
// rows, its four waves take every fourth 32-key tile with operands straight from global
// memory, and meet once at the end.
template <int ND>
__global__ __launch_bounds__(256) void paged_attn_f32_kernel(KArgs p) {
  constexpr int D = 32 * ND, NW = 4, NC = 4 * ND, OP = D + 4, BQ = 32, BKV = 32;
  __shared__ __attribute__((aligned(16))) float so[NW * 32 * OP];
  __shared__ float sm[NW][32], sl[NW][32];
  Item it;
  if (!find_item<BQ, BKV, false>(p, blockIdx.x, it)) return;
  const Seq& sq = it.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int rows = sq.n * p.G, first = sq.len - sq.n;
  const int r0 = it.rt * BQ, r1 = min(r0 + BQ, rows) - 1;
  int lo, hi;
  key_range(p, sq, r0, r1, lo, hi);
  const int t_lo = lo / BKV, cnt = hi < 0 ? 0 : hi / BKV - t_lo + 1;
  const int t0 = t_lo + (int)((int64_t)cnt * it.split / it.ns);
  const int t1 = t_lo + (int)((int64_t)cnt * (it.split + 1) / it.ns);

  const int r = min(r0 + l31, rows - 1);
  const int tok = r / p.G, g = r - tok * p.G;
  const int khi = p.causal ? min(first + tok, sq.len - 1) : sq.len - 1;
  const int klo = p.window ? first + tok - p.window + 1 : 0;
  f32x4_t qf[NC], kf[NC];
  {
    const float* qrow = (const float*)p.q + (int64_t)(sq.s0 + tok) * p.st_q +
                        (int64_t)(it.kvh * p.G + g) * p.sh_q;
#pragma unroll
    for (int j = 0; j < NC; ++j) qf[j] = *reinterpret_cast<const f32x4_t*>(qrow + 8 * j + 4 * h);
  }
  const int32_t* table = p.table + (int64_t)sq.slot * p.max_pages;
  const int mask = (1 << p.lps) - 1;
  // element offset of a key's row; keys past the end give the last one
  auto row_at = [&](int key) -> int64_t {
    key = min(key, sq.len - 1);
    int page = table[key >> p.lps];
    page = page < 0 ? 0 : page < p.num_pages ? page : p.num_pages - 1;
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
  if (t0 + w < t1) load_k(t0 + w);
  for (int t = t0 + w; t < t1; t += NW) {
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
    load_k(t + NW < t1 ? t + NW : t);
    const int up = khi - k0 - 4 * h, dn = klo - k0 - 4 * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 8 * (i >> 2) + (i & 3);
      s[i] = key <= up && key >= dn ? s[i] : -INFINITY;
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
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int n = 0; n < ND; ++n)
        oacc[n] =
            __builtin_amdgcn_mfma_f32_32x32x2f32(vf[n / VW][i][n % VW], s[i], oacc[n], 0, 0, 0);
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
  for (int i = tid; i < nq * D; i += 256) {
    const int rr = i / D, cc = i - rr * D;
    const float* x = so + rr * OP + cc;
    const float sum = (x[0] + x[32 * OP]) + (x[64 * OP] + x[96 * OP]);
    const float tot = sl[0][rr];
    if (it.ns > 1) {
      p.part[(at + rr) * D + cc] = sum;
      if (cc == 0) {
        p.ml[(at + rr) * 2] = sm[0][rr];
        p.ml[(at + rr) * 2 + 1] = tot;
      }
    } else {
      const int t = (r0 + rr) / p.G, gg = (r0 + rr) - t * p.G;
      ((float*)p.o)[(int64_t)(sq.s0 + t) * p.st_o + (int64_t)(it.kvh * p.G + gg) * p.sh_o + cc] =
          tot == 0.f ? 0.f : sum / tot;
    }
  }
}

// ---- joining the parts of a row tile ----------------------------------------------
// One block per row tile with parts, a wave per row: o = sum_i w_i o_i / sum_i w_i l_i,
// w_i = e^(scale (m_i - max)).
template <int D, int BQ, int BKV, typename T>
__global__ __launch_bounds__(256) void combine_kernel(KArgs p) {
  Item it;
  if (!find_item<BQ, BKV, true>(p, blockIdx.x, it)) return;
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int rows = it.q.n * p.G;
  const int r0 = it.rt * BQ, nr = min(BQ, rows - r0);
  const int64_t step = (int64_t)it.nrt * BQ, s0 = slot_of(it, 0) * BQ;
  for (int r = w; r < nr; r += 4) {
    float mx = -INFINITY;
    for (int i = lane; i < it.ns; i += 64) mx = fmaxf(mx, p.ml[(s0 + i * step + r) * 2]);
    mx = wave_max(mx);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float acc[E], lt = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < it.ns; i0 += 64) {
      float wt = 0.f;
      if (i0 + lane < it.ns) {
        const float* ml = p.ml + (s0 + (i0 + lane) * step + r) * 2;
        wt = __builtin_amdgcn_exp2f((ml[0] - mu) * p.c);
        lt += wt * ml[1];
      }
      const int n = min(64, it.ns - i0);
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float wi =
            __builtin_bit_cast(float, lane_of(__builtin_bit_cast(int, wt), i));
        const float* src = p.part + (s0 + (i0 + i) * step + r) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(wi, src[e], acc[e]);
      }
    }
    lt = wave_sum(lt);
    const int t = (r0 + r) / p.G, g = (r0 + r) - t * p.G;
    const int64_t at = (int64_t)(it.q.s0 + t) * p.st_o + (int64_t)(it.kvh * p.G + g) * p.sh_o;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = lt == 0.f ? 0.f : acc[e] / lt;
      if constexpr (sizeof(T) == 2) ((uint16_t*)p.o)[at + lane * E + e] = f32_to_bf16(x);
      else ((float*)p.o)[at + lane * E + e] = x;
    }
  }
}

// ---- launch ------------------------------------------------------------------------
struct Shape {
  int bq, bkv, target, cmin;
};
// resident blocks: 3 per CU where LDS (48 KB of stages) and registers allow, 2 for
// head_dim 128 and f32
Shape shape_of(const blt_paged_cache& c) {
  if (c.dtype == BLT_DTYPE_F32) return Shape{32, 32, 512, 4};
  return Shape{128, 64, c.head_dim == 64 ? 768 : 512, 2};
}
int64_t row_tiles(const blt_paged_cache& c, int64_t B, int64_t total, int H, int bq) {
  return total * (H / c.n_kv_heads) / bq + B;
}
// parts: none where not even a full sequence has more than cmin key tiles
int64_t slots_of(const blt_paged_cache& c, const Shape& s) {
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  return cap <= (int64_t)s.cmin * s.bkv ? 0 : 2 * (int64_t)s.target;
}

}  // namespace

int64_t paged_attention_workspace_bytes(const blt_paged_cache& c, int64_t, int64_t, int) {
  const Shape s = shape_of(c);
  return slots_of(c, s) * s.bq * (c.head_dim + 2) * 4;
}

int launch_paged_attention(const blt_paged_cache& c, const PagedAttnArgs& a, void* ws,
                           hipStream_t s) {
  const Shape sh = shape_of(c);
  const int d = c.head_dim;
  KArgs p{};
  const int64_t es = c.dtype == BLT_DTYPE_BF16 ? 2 : 4;
  const int64_t layer = (int64_t)a.layer * c.num_pages * c.n_kv_heads * c.page_size * d * es;
  p.q = a.q; p.o = a.o;
  p.k = (const char*)c.k + layer; p.v = (const char*)c.v + layer;
  p.st_q = a.st_q; p.sh_q = a.sh_q; p.st_o = a.st_o; p.sh_o = a.sh_o;
  p.starts = a.starts; p.seqs = a.seqs; p.lens = c.lens; p.table = c.page_table;
  p.B = (int)a.B; p.total = (int)a.total; p.H = a.H; p.Hkv = c.n_kv_heads; p.G = a.H / c.n_kv_heads;
  p.max_seqs = c.max_seqs; p.max_pages = c.max_pages; p.num_pages = c.num_pages;
  p.lps = log2_of(c.page_size); p.cap = c.max_pages * c.page_size;
  p.causal = a.causal; p.window = a.causal ? a.window : 0;
  if (p.window > (1 << 30)) p.window = 0;  // longer than any sequence
  p.c = (float)(1.44269504088896340736 * (double)a.scale);
  p.target = sh.target; p.cmin = sh.cmin;
  const int64_t slots = slots_of(c, sh);
  p.part = (float*)ws;
  p.ml = p.part + slots * sh.bq * d;
  const int64_t rt = row_tiles(c, a.B, a.total, a.H, sh.bq) * c.n_kv_heads;
  const int64_t nb = (rt + (slots ? sh.target : 0) + 7) / 8 * 8;
  if (nb > 0x7fffffff) return fail(BLT_ERR_SHAPE, "paged_attention: too many row tiles");
  const dim3 grid((unsigned)nb), block(256);
  const int64_t nj = rt < sh.target ? rt : sh.target;  // row tiles with parts
  const dim3 jgrid((unsigned)nj);
  if (c.dtype == BLT_DTYPE_BF16) {
    if (d == 64) hipLaunchKernelGGL((paged_attn_kernel<64, 1, 3>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_attn_kernel<128, 1, 2>), grid, block, 0, s, p);
    BLT_LAUNCH_CHECK("paged_attn_kernel");
    if (slots) {
      if (d == 64) hipLaunchKernelGGL((combine_kernel<64, 128, 64, uint16_t>), jgrid, block, 0, s, p);
      else hipLaunchKernelGGL((combine_kernel<128, 128, 64, uint16_t>), jgrid, block, 0, s, p);
      BLT_LAUNCH_CHECK("combine_kernel");
    }
  } else {
    if (d == 64) hipLaunchKernelGGL((paged_attn_f32_kernel<2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_attn_f32_kernel<4>), grid, block, 0, s, p);
    BLT_LAUNCH_CHECK("paged_attn_f32_kernel");
    if (slots) {
      if (d == 64) hipLaunchKernelGGL((combine_kernel<64, 32, 32, float>), jgrid, block, 0, s, p);
      else hipLaunchKernelGGL((combine_kernel<128, 32, 32, float>), jgrid, block, 0, s, p);
      BLT_LAUNCH_CHECK("combine_kernel");
    }
  }
  return 0;
}

}  // namespace blt
