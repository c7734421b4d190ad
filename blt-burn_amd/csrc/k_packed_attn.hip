// Attention of whole sequences packed behind each other, of different lengths, grouped
// heads, head_dim 64 or 128: one pass over the keys with a running max and sum.
//
// Tokens, rows and tiles.  Tokens are counted over the whole pack, so that "key j is visible to
// token i" is klo(i) <= j <= khi(i) with the two bounds from the sequence that i lies in, found
// once per row.  The query heads that share a key head are packed with the tokens into rows
// (row = token * G + head): one key tile serves all of them, and no tile has fewer rows
// because a sequence ends in it: tiles of rows run over the ends of sequences, so that the grid
// follows from the number of tokens alone and many short sequences share a tile.  A wave passes the
// key tiles that none of its rows sees.
#include <algorithm>
#include <type_traits>

#include "attn_tiles.hpp"
#include "packed.hpp"

namespace blt {

namespace {

struct PArgs {
  const void *q, *k, *v;
  void* o;
  float* lse;
  int64_t st_q, sh_q, st_k, sh_k, st_v, sh_v, st_o, sh_o;
  const int32_t* starts;
  int B, total, rows, H, G;  // rows: total * G
  Divisor by_g;
  int causal, window;  // window 0: none
  float scale, c;      // c: log2(e) * scale
  int tail;
  int tiles, residues, units;  // row (or key) tiles; see tile_of
  const int* order;            // the tiles, longest first, or null: see packed_order_kernel
};

// The key head and the tile of block `bid`.  Dispatch places block i on XCD i % 8; a
// unit, the tiles of one key head with one residue modulo `residues`, belongs to one XCD, whose L2 its
// keys share.  Every XCD has the same number of units (`units`), and residues rather than
// runs so that all units have about the same work.  Without an order, the last tiles first (`down`)
// or the first ones: the long ones of a single causal sequence.
__device__ inline bool tile_of(const PArgs& p, bool down, int& kvh, int& tile) {
  const uint32_t x = blockIdx.x & 7, l = blockIdx.x >> 3;
  const uint32_t step = l / (uint32_t)p.units;
  const uint32_t u = x * (uint32_t)p.units + (l - step * (uint32_t)p.units);
  kvh = (int)(u / (uint32_t)p.residues);
  const int residue = (int)(u - (uint32_t)kvh * (uint32_t)p.residues);
  const int rank = residue + p.residues * (int)step;
  if (rank >= p.tiles) return false;
  tile = p.order ? p.order[rank] : down ? p.tiles - 1 - rank : rank;
  return true;
}

// The sequence [a, e) of token `tok`, false if it lies in none.  Starts that do not ascend
// give some sequence, within the tokens.  Called by whole waves.
__device__ inline bool sequence_of(const PArgs& p, int tok, int& a, int& e) {
  int b = 0;
  if (p.B <= 64) {  // (one load, then no more dependent ones)
    const int lane = threadIdx.x & 63;
    const int s = p.starts[min(lane, p.B)];
    const int all = p.starts[p.B];
    for (int i = 1; i <= p.B; ++i)
      b += (i < 64 ? __builtin_amdgcn_readlane(s, i) : all) <= tok ? 1 : 0;
    a = __shfl(s, min(b, 63));
    e = b + 1 < 64 ? __shfl(s, min(b + 1, 63)) : all;
  } else {
    int hi = p.B;  // the first b with starts[b + 1] > tok
    while (__any(b < hi)) {
      const int mid = (b + hi) >> 1;
      if (b < hi) {
        if (p.starts[mid + 1] > tok) hi = mid; else b = mid + 1;
      }
    }
    a = p.starts[min(b, p.B)];
    e = p.starts[min(b + 1, p.B)];
  }
  a = max(a, 0);
  e = min(e, p.total);
  return b < p.B && a <= tok && tok < e;
}
// The keys that a token sees.
__device__ inline bool keys_of(const PArgs& p, int tok, int& klo, int& khi) {
  int a, e;
  const bool in = sequence_of(p, tok, a, e);
  klo = a;
  khi = p.causal ? tok : e - 1;
  if (p.window) klo = max(klo, tok - p.window + 1);
  if (!in) {
    klo = 0;
    khi = -1;
  }
  return in;
}

// Tiles by their lengths, longest first, so that the blocks that start last are short ones (12
// documents of up to 8192 tokens, 12 heads of 64: 423 us in the order of the tokens, whose last blocks are
// the first document's long ones, and 403 in this one; the order itself takes 5).  Block 0: the row tiles,
// block 1: the key tiles (null: not asked for).  Tiles of one of 256 lengths in any order: it does not change
// what they hold.
constexpr int kOrderTiles = 8192, kOrderStarts = 4096;
__global__ __launch_bounds__(1024) void packed_order_kernel(PArgs p, int rows, int keys, int* row_order,
                                                            int* key_order) {
  constexpr int PER = kOrderTiles / 1024;
  __shared__ int starts[kOrderStarts + 1], hist[256], longest;
  const bool of_rows = blockIdx.x == 0;
  int* out = of_rows ? row_order : key_order;
  if (!out) return;
  const int each = of_rows ? rows : keys, n = of_rows ? p.rows : p.total;
  const int tiles = (n + each - 1) / each, tid = threadIdx.x;
  const int32_t* at = p.starts;
  if (p.B <= kOrderStarts) {
    for (int i = tid; i <= p.B; i += 1024) starts[i] = p.starts[i];
    at = starts;
  }
  if (tid < 256) hist[tid] = 0;
  if (tid == 0) longest = 1;
  __syncthreads();
  // the sequence of a token (the last one for those behind it)
  auto sequence = [&](int tok, int& a, int& e) {
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at[mid + 1] > tok) hi = mid; else lo = mid + 1;
    }
    a = min(max(at[lo], 0), tok);
    e = max(at[lo + 1], tok + 1);
  };
  int length[PER], most = 1;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + 1024 * j;
    length[j] = 0;
    if (i >= tiles) continue;
    const int x0 = i * each, x1 = min(x0 + each, n) - 1;
    const int t0 = of_rows ? over(x0, p.by_g) : x0, t1 = of_rows ? over(x1, p.by_g) : x1;
    int a, e, a1, e1;
    sequence(t0, a, e);
    sequence(t1, a1, e1);
    int64_t lo, hi;  // tokens on the other side
    if (of_rows) {
      lo = p.window ? max(a, t0 - p.window + 1) : a;
      hi = p.causal ? t1 : e1 - 1;
    } else {
      lo = p.causal ? t0 : a;
      hi = p.window ? min((int64_t)e1 - 1, (int64_t)t1 + p.window - 1) : e1 - 1;
    }
    length[j] = (int)min((hi - lo) / 32 + 1, (int64_t)1 << 24);
    most = max(most, length[j]);
  }
  most = wave_max_i32(most);
  if ((tid & 63) == 0) atomicMax(&longest, most);
  __syncthreads();
  int cls[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    cls[j] = 255 - (int)((int64_t)length[j] * 255 / longest);
    if (tid + 1024 * j < tiles) atomicAdd(&hist[cls[j]], 1);
  }
  __syncthreads();
  if (tid < 64) {  // exclusive sums of 256 counts
    int v[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = sum;
      sum += hist[4 * tid + i];
    }
    const int before = wave_incl_scan(sum) - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) hist[4 * tid + i] = before + v[i];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (tid + 1024 * j < tiles) out[atomicAdd(&hist[cls[j]], 1)] = tid + 1024 * j;
}

// LDS tiles have rows of D elements without padding; 16-byte chunk c of row r is stored at
// c ^ swz(r), which spreads both the reads of one chunk of 16 rows and the transposing reads
// of four rows' neighbouring chunks over all banks.
template <int D>
__device__ inline int swz(int r) {
  return D == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}
template <int D>
__device__ inline bf16x8_t row_chunk(const uint16_t* tile, int r, int chunk) {
  return *reinterpret_cast<const bf16x8_t*>(tile + r * D + ((chunk ^ swz<D>(r)) << 3));
}
// Transposing reads: the wave's 16-row blocks as the first operand of a product over rows.
// Lane offsets for 32 columns at 32 ds: rows 4 (lane / 32) + lane % 16 / 4 (and 8 further),
// columns 16 (lane / 16 % 2) + 4 (lane % 4).
template <int D>
struct Transposed {
  int at[D / 32][2];
  __device__ inline Transposed(int lane) {
    const int s16 = lane & 15, r = 4 * (lane >> 5) + (s16 >> 2);
#pragma unroll
    for (int ds = 0; ds < D / 32; ++ds)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int chunk = 4 * ds + 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
        at[ds][h] = (r + 8 * h) * D + ((chunk ^ swz<D>(r + 8 * h)) << 3) + 4 * (s16 & 1);
      }
  }
  // rows r0 .. r0 + 15 (r0 a multiple of 16): [k] = row 8 (k / 4) + 4 (lane / 32) + k % 4
  __device__ inline u32x4_t read(const uint16_t* tile, int r0, int ds) const {
    const u32x2_t w0 = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(tile + r0 * D + at[ds][0])));
    const u32x2_t w1 = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(tile + r0 * D + at[ds][1])));
    return u32x4_t{w0.x, w0.y, w1.x, w1.y};
  }
};
// The order of a block's LDS reads and matrix products: `ahead` reads, then `each` reads behind every
// one of the first `n` products.  (Left alone the compiler reads an operand right before its
// product and waits for it every time.)
template <int AHEAD, int N, int EACH, int LAST>
__device__ inline void reads_ahead() {
  constexpr int MFMA = 0x008, READ = 0x100;
  __builtin_amdgcn_sched_group_barrier(READ, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    __builtin_amdgcn_sched_group_barrier(READ, EACH, 0);
  }
  __builtin_amdgcn_sched_group_barrier(MFMA, LAST, 0);
}
__device__ inline bf16x8_t bf8(u32x4_t x) { return __builtin_bit_cast(bf16x8_t, x); }

// Bounds of the keys that the rows of a wave and of its block see.
struct Bounds {
  int wlo, whi;    // some row of the wave sees these keys
  int lo_max, hi_min;  // every row sees [lo_max, hi_min]
  int lo, hi;      // some row of the block
};
template <int NW>
__device__ inline Bounds bounds_of(int klo, int khi, bool in) {
  Bounds b;
  b.wlo = -wave_max_i32(in ? -klo : -0x7fffffff);
  b.whi = wave_max_i32(khi);
  b.lo_max = wave_max_i32(klo);
  b.hi_min = -wave_max_i32(-khi);
  b.lo = b.wlo;
  b.hi = b.whi;
  if constexpr (NW > 1) {  // (the waves have rows of their own)
    __shared__ int lo_of[NW], hi_of[NW];
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      lo_of[w] = b.wlo;
      hi_of[w] = b.whi;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      b.lo = min(b.lo, lo_of[i]);
      b.hi = max(b.hi, hi_of[i]);
    }
  }
  b.lo = __builtin_amdgcn_readfirstlane(b.lo);
  b.hi = __builtin_amdgcn_readfirstlane(b.hi);
  return b;
}

// ---- bf16 --------------------------------------------------------------------------
// One block = 4 waves of 32 rows; key tiles of 64 keys go global -> LDS by DMA through two
// stages shared by the waves.  Scores are taken transposed, S^T = K . Q^T, so a lane owns one
// row: its max and sum need one cross-lane step and P^T feeds the second product from
// registers; V's operand is read with the LDS transposing read.  p is rounded to bf16 for the second
// product, and without LSE the sum takes the rounded values, so that the weights of a row
// add up to one; with it the sum is of p itself, which a gradient's weights go by.
// d = 64: bound by the vector units (an exponential, and 2.5 more instructions, for each score
// take longer than its 256 FLOP): 12 sequences of up to 8192, 12 heads, 403 us, 0.77 PFLOP/s, vector units
// 65 % and matrix cores 39 % busy, rarely both.  d = 128: two sequences of 16384 and 11603, 32 / 8
// heads, 3.07 ms, 1.08 PFLOP/s (the library's 8192^3 product: 1.21), 49 % and 55 %.  Short ones: 156 tokens of
// 12 heads 7.2 us, a launch and three tiles' dependent steps.
template <int D, bool LSE>
__global__ __launch_bounds__(256, 2) void packed_attn_kernel(PArgs p) {
  constexpr int BKV = 64, QPW = 32, BQ = 4 * QPW;
  constexpr int TILE = BKV * D, STAGE = 2 * TILE, NST = 2;
  constexpr int KS = D / 16, DS = D / 32, CPR = D / 8, RPI = 64 / CPR;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[NST * STAGE];

  int kvh, tile;
  if (!tile_of(p, true, kvh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int rw = tile * BQ + wid * QPW;
  const int row = min(rw + lrow, p.rows - 1);
  const int tok = over(row, p.by_g), head = kvh * p.G + row - tok * p.G;

  bf16x8_t qf[KS];
  {
    const uint16_t* qrow =
        (const uint16_t*)p.q + (int64_t)tok * p.st_q + (int64_t)head * p.sh_q;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[ks] = bf8(*reinterpret_cast<const u32x4_t*>(qrow + ks * 16 + lhalf * 8));
  }
  int klo, khi;
  const bool in = keys_of(p, tok, klo, khi);
  const Bounds bd = bounds_of<4>(klo, khi, in);
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BKV, t1 = bd.hi < 0 ? 0 : bd.hi / BKV + 1;
  // consumed here, before any DMA is in flight
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[ks]));

  // DMA: wave w moves keys 16 w .. 16 w + 15 of a tile, RPI at a time
  const unsigned lds_base = (unsigned)(uintptr_t)lds;
  const int kin = lane / CPR, slot = lane % CPR;
  const char* kbase = (const char*)p.k + (int64_t)kvh * p.sh_k * 2;
  const char* vbase = (const char*)p.v + (int64_t)kvh * p.sh_v * 2;
  auto issue = [&](int t, int stage) {
    const unsigned sb = lds_base + (unsigned)(stage * STAGE * 2);
    const int last = p.total - 1 - t * BKV;
    const char* kt = kbase + (int64_t)t * BKV * p.st_k * 2;
    const char* vt = vbase + (int64_t)t * BKV * p.st_v * 2;
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const int r = 16 * wid + RPI * i + kin, from = min(r, last);
      const unsigned ch = (unsigned)((slot ^ swz<D>(r)) * 16);
      const unsigned la = sb + (unsigned)((16 * wid + RPI * i) * D * 2);
      dma16_so(kt, (unsigned)from * (unsigned)(p.st_k * 2) + ch, la);
      dma16_so(vt, (unsigned)from * (unsigned)(p.st_v * 2) + ch, la + TILE * 2);
    }
  };
  const Transposed<D> tr(lane);

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

  if (t0 < t1) issue(t0, 0);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    // tile t has landed and every wave is past tile t - 1, whose stage is free
    dma_wait_barrier<0>();
    if (t + 1 < t1) issue(t + 1, stage ^ 1);
    const int kb = t * BKV;
    if (kb <= bd.whi && kb + BKV > bd.wlo) {
      const uint16_t* sk = lds + stage * STAGE;
      const uint16_t* sv = sk + TILE;
      const bool mask_hi = kb + BKV - 1 > bd.hi_min, mask_lo = kb < bd.lo_max;
      bf16x8_t f[2][KS];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          f[sub][ks] = row_chunk<D>(sk, sub * 32 + lrow, 2 * ks + lhalf);
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
          for (int u = 0; u < 2; ++u) vf[ds][sub][u] = tr.read(sv, sub * 32 + u * 16, ds);
      // (d = 64: one side at a time, since hardly a tile needs both: eleven sequences of up to 2047,
      // window 512, 12 heads, 38.7 us for 41.2; d = 128: 201 for 195)
      const int up = khi - kb - 4 * lhalf, dn = klo - kb - 4 * lhalf;
      if (D == 64 ? mask_hi : mask_hi || mask_lo) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = sub * 32 + 8 * (r >> 2) + (r & 3);
            s[sub][r] = key <= up && (D == 64 || key >= dn) ? s[sub][r] : -INFINITY;
          }
      }
      if (D == 64 && mask_lo) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[sub][r] = sub * 32 + 8 * (r >> 2) + (r & 3) >= dn ? s[sub][r] : -INFINITY;
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
#pragma unroll
            for (int i = 0; i < DS * 4; ++i) {  // columns 8 i + 4 lhalf .. + 3
              const u32x2_t x = *reinterpret_cast<const u32x2_t*>(
                  sv + j * D + ((i ^ swz<D>(j)) << 3) + 4 * lhalf);
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
            if constexpr (LSE)
              l += p0 + p1;
            else
              l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[e >> 1]), ones2,
                                                  l, false);
          }
          const bf16x8_t pb = bf8(u32x4_t{w[0], w[1], w[2], w[3]});
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)  // (independent chains)
            o[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf8(vf[ds][sub][u]), pb, o[ds], 0, 0,
                                                            0);
        }
    }
    stage ^= 1;
  }

  float a, b;
  swap_pair<32>(l, a, b);
  const float total = a + b;
  if (rw + lrow < p.rows && (in || p.tail)) {
    uint16_t* orow = (uint16_t*)p.o + (int64_t)tok * p.st_o + (int64_t)head * p.sh_o;
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
  // (behind the last sequence too, whatever `tail` says of o)
  if (LSE && rw + lrow < p.rows && lhalf == 0)
    p.lse[(int64_t)tok * p.H + head] = total == 0.f ? -INFINITY : fmaf(m, p.scale, logf(total));
}

// ---- f32 -----------------------------------------------------------------------------
// Both products on the f32 matrix cores, one block = 32 rows, its four waves take every
// fourth 32-key tile with operands straight from global memory, and meet once at the end.
// Bound by the loads in front of the products, with two waves a SIMD to cover them: five sequences of up to
// 1501, 12 heads of 64, 142 us, 79 TFLOP/s (an f32 library product: 136), matrix cores 53 % busy.  d = 128, one
// wave a SIMD: sequences of 2000 and 1441, 8 / 1 heads, 175 us, 71 TFLOP/s; of 1000, 721, 1 and 303, 32 / 8 heads,
// 209, 63.
template <int ND>
__global__ __launch_bounds__(256) void packed_attn_f32_kernel(PArgs p) {
  constexpr int D = 32 * ND, NW = 4, NC = 4 * ND, OP = D + 4, BKV = 32;
  __shared__ __attribute__((aligned(16))) float so[NW * 32 * OP];
  __shared__ float sm[NW][32], sl[NW][32];
  int kvh, rt;
  if (!tile_of(p, true, kvh, rt)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int r0 = rt * 32, row = min(r0 + l31, p.rows - 1);
  const int tok = over(row, p.by_g), head = kvh * p.G + row - tok * p.G;
  int klo, khi;
  const bool in = keys_of(p, tok, klo, khi);
  const Bounds bd = bounds_of<1>(klo, khi, in);  // (every wave has the same rows)
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BKV, t1 = bd.hi < 0 ? 0 : bd.hi / BKV + 1;

  f32x4_t qf[NC], kf[NC];
  {
    const float* qrow = (const float*)p.q + (int64_t)tok * p.st_q + (int64_t)head * p.sh_q;
#pragma unroll
    for (int j = 0; j < NC; ++j) qf[j] = *reinterpret_cast<const f32x4_t*>(qrow + 8 * j + 4 * h);
  }
  const float* kbase = (const float*)p.k + (int64_t)kvh * p.sh_k;
  const float* vbase = (const float*)p.v + (int64_t)kvh * p.sh_v;
  auto load_k = [&](int t) {
    const float* r = kbase + (int64_t)min(t * BKV + l31, p.total - 1) * p.st_k;
#pragma unroll
    for (int j = 0; j < NC; ++j) kf[j] = *reinterpret_cast<const f32x4_t*>(r + 8 * j + 4 * h);
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
  // one tile; the next one's K (of `next`) is loaded under the second product
  auto tile = [&](int t, int next) {
    const int k0 = t * BKV;
    // V of key k0 + 8 (i / 4) + 4 h + i % 4 (past the end: the last one, masked)
    vf_t vf[NV][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float* r = vbase +
                       (int64_t)min(k0 + 8 * (i >> 2) + 4 * h + (i & 3), p.total - 1) * p.st_v +
                       VW * l31;
#pragma unroll
      for (int n = 0; n < NV; ++n) vf[n][i] = *reinterpret_cast<const vf_t*>(r + 32 * VW * n);
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
    if (k0 + BKV - 1 > bd.hi_min || k0 < bd.lo_max) {  // (as in packed_attn_kernel)
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
        const float* vrow = vbase + (int64_t)min(k0 + j, p.total - 1) * p.st_v;
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
  if (t0 + w < t1) load_k(t0 + w);
  for (int t = t0 + w; t < t1; t += NW) tile(t, t + NW < t1 ? t + NW : t);

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
  __shared__ int write[32];
  if (w == 0 && h == 0) {
    sl[0][l31] = lt;
    write[l31] = r0 + l31 < p.rows && (in || p.tail);
    if (p.lse && r0 + l31 < p.rows)  // (behind the last sequence too)
      p.lse[(int64_t)tok * p.H + head] = lt == 0.f ? -INFINITY : fmaf(mx, p.scale, logf(lt));
  }
  __syncthreads();
  for (int i = tid; i < 32 * (D / 4); i += 256) {
    const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
    if (!write[rr]) continue;
    f32x4_t x[NW];
#pragma unroll
    for (int k = 0; k < NW; ++k)
      x[k] = *reinterpret_cast<const f32x4_t*>(so + (k * 32 + rr) * OP + cc);
    const f32x4_t sum = (x[0] + x[1]) + (x[2] + x[3]);
    const float tot = sl[0][rr];
    const int t = over(r0 + rr, p.by_g), gg = (r0 + rr) - t * p.G;
    *reinterpret_cast<f32x4_t*>((float*)p.o + (int64_t)t * p.st_o +
                                (int64_t)(kvh * p.G + gg) * p.sh_o + cc) =
        tot == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sum / tot;
  }
}

// ---- gradient ------------------------------------------------------------------------
// With p_ij = e^(scale s_ij - L_i) and D_i = do_i . o_i
//   ds_ij = p_ij (do_i . v_j - D_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// in two kernels that recompute p from L: one with rows in registers and the keys passing by, for dq
// (and D), one with keys in registers and the rows that see them passing by, which sums
// dk and dv over tokens and a key head's query heads by itself.  That makes seven products of the
// size of S instead of the five of one kernel, which would have to add up dq in memory in
// an order that changes from run to run.
struct GArgs {
  PArgs a;  // (o and lse are read)
  const void* g;  // of the output
  void *dq, *dk, *dv;
  int64_t st_g, sh_g, st_dq, sh_dq, st_dk, sh_dk, st_dv, sh_dv;
  // for 64 rows each: -L log2(e) of them, then -D
  float* stats;
  int stat_tiles;  // of a key head
  float* part;     // dk and dv of one of several blocks of a tile's rows: see packed_join_kernel
};
__device__ inline float* stats_of(const GArgs& p, int kvh, int row) {
  return p.stats + (((int64_t)kvh * p.stat_tiles + (row >> 6)) * 128 + (row & 63));
}
// -L log2(e) for e^(scale s - L) = 2^(s c + this); -inf where the row has no sum: all its
// scores are -inf
__device__ inline float offset_of(float lse) {
  return lse == -INFINITY ? lse : -1.44269504088896340736f * lse;
}
__device__ inline float dot8(u32x4_t x, u32x4_t y) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
    s = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), s);
  }
  return s;
}
// The rows that see a key, as keys_of.
__device__ inline bool rows_of(const PArgs& p, int key, int& rlo, int& rhi) {
  int a, e;
  const bool in = sequence_of(p, key, a, e);
  const int lo = p.causal ? key : a;
  const int hi = p.window ? min(e - 1, key + p.window - 1) : e - 1;
  rlo = in ? lo * p.G : 0;
  rhi = in ? (hi + 1) * p.G - 1 : -1;
  return in;
}

// dq, bf16: as packed_attn_kernel, with two score products, V . dO^T beside K . Q^T, and
// dQ^T = K^T . dS^T, whose first operand is read by transposing reads of the same K tile.
// dS goes into its product as two bf16 halves (cut off, and what that left, rounded), and as it
// adds up to 0 over a row but for what D is off by, with o rounded to bf16, that sum corrects D for the
// other kernel.  So both gradients are 2.3e-3 off or less (relative, rms; their own rounding is
// 1.7e-3), and not 2.5e-3 or, in short sequences, 3e-3.
// Four sequences of up to 4096 (9 k tokens), 32 / 8 heads of 128: 435 us, four products (dS twice) at
// 1.1 PFLOP/s, matrix cores 55 % and vector units 47 % busy; eleven of up to 2047, window 512, 12 heads of
// 64: 48 us, ten key tiles behind each other in 1.5 rounds of blocks (52 with 64 keys at a time, whether
// seen or not, and both sides of the mask in one).
template <int D>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(GArgs ga) {
  const PArgs& p = ga.a;
  constexpr int BKV = 64, QPW = 32, BQ = 4 * QPW;
  constexpr int TILE = BKV * D, STAGE = 2 * TILE, NST = 2;
  constexpr int KS = D / 16, DS = D / 32, CPR = D / 8, RPI = 64 / CPR;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[NST * STAGE];

  int kvh, tile;
  if (!tile_of(p, true, kvh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int rw = tile * BQ + wid * QPW;
  const int row = min(rw + lrow, p.rows - 1);
  const int tok = over(row, p.by_g), head = kvh * p.G + row - tok * p.G;

  bf16x8_t qf[KS], gf[KS];
  float delta = 0.f;
  {
    const uint16_t* qrow =
        (const uint16_t*)p.q + (int64_t)tok * p.st_q + (int64_t)head * p.sh_q;
    const uint16_t* grow =
        (const uint16_t*)ga.g + (int64_t)tok * ga.st_g + (int64_t)head * ga.sh_g;
    const uint16_t* orow =
        (const uint16_t*)p.o + (int64_t)tok * p.st_o + (int64_t)head * p.sh_o;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = bf8(*reinterpret_cast<const u32x4_t*>(qrow + ks * 16 + lhalf * 8));
      const u32x4_t g = *reinterpret_cast<const u32x4_t*>(grow + ks * 16 + lhalf * 8);
      gf[ks] = bf8(g);
      delta += dot8(g, *reinterpret_cast<const u32x4_t*>(orow + ks * 16 + lhalf * 8));
    }
    float a, b;
    swap_pair<32>(delta, a, b);
    delta = a + b;
  }
  const float mc = offset_of(p.lse[(int64_t)tok * p.H + head]);
  int klo, khi;
  const bool in = keys_of(p, tok, klo, khi);
  const Bounds bd = bounds_of<4>(klo, khi, in);
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BKV, t1 = bd.hi < 0 ? 0 : bd.hi / BKV + 1;
  // (everything consumed before any DMA is in flight)
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[ks]), "v"(gf[ks]));

  const unsigned lds_base = (unsigned)(uintptr_t)lds;
  const int kin = lane / CPR, slot = lane % CPR;
  const char* kbase = (const char*)p.k + (int64_t)kvh * p.sh_k * 2;
  const char* vbase = (const char*)p.v + (int64_t)kvh * p.sh_v * 2;
  auto issue = [&](int t, int stage) {
    const unsigned sb = lds_base + (unsigned)(stage * STAGE * 2);
    const int last = p.total - 1 - t * BKV;
    const char* kt = kbase + (int64_t)t * BKV * p.st_k * 2;
    const char* vt = vbase + (int64_t)t * BKV * p.st_v * 2;
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const int r = 16 * wid + RPI * i + kin, from = min(r, last);
      const unsigned ch = (unsigned)((slot ^ swz<D>(r)) * 16);
      const unsigned la = sb + (unsigned)((16 * wid + RPI * i) * D * 2);
      dma16_so(kt, (unsigned)from * (unsigned)(p.st_k * 2) + ch, la);
      dma16_so(vt, (unsigned)from * (unsigned)(p.st_v * 2) + ch, la + TILE * 2);
    }
  };
  const Transposed<D> tr(lane);
  f32x16_t acc[DS];
#pragma unroll
  for (int j = 0; j < DS; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
  const float c = p.c;
  float rest = 0.f;  // sum of the row's dS

  if (t0 < t1) issue(t0, 0);
  int stage = 0;
  for (int t = t0; t < t1; ++t) {
    dma_wait_barrier<0>();
    if (t + 1 < t1) issue(t + 1, stage ^ 1);
    const int kb = t * BKV;
    if (kb <= bd.whi && kb + BKV > bd.wlo) {
      const uint16_t* sk = lds + stage * STAGE;
      const uint16_t* sv = sk + TILE;
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) {
        const int k0 = kb + sub * 32;
        if (k0 > bd.whi || k0 + 32 <= bd.wlo) continue;
        const bool mask_hi = k0 + 31 > bd.hi_min, mask_lo = k0 < bd.lo_max;
        f32x16_t s, dp;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              row_chunk<D>(sk, sub * 32 + lrow, 2 * ks + lhalf), qf[ks],
              ks == 0 ? f32x16_t{} : s, 0, 0, 0);
          dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              row_chunk<D>(sv, sub * 32 + lrow, 2 * ks + lhalf), gf[ks], ks == 0 ? f32x16_t{} : dp, 0,
              0, 0);
        }
        u32x4_t kt[DS][2];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int u = 0; u < 2; ++u) kt[ds][u] = tr.read(sk, sub * 32 + u * 16, ds);
        // A weight of zero does not silence a key that is not finite (as in packed_attn_kernel),
        // which shows in every row's score of it; where it is seen the result is NaN.
        bool odd = false;
        if (mask_hi || mask_lo) {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum = fmaf(s[r], 0.f, sum);
          odd = __any(sum != sum);
        }
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, mc)) * (dp[r] - delta);
        if (mask_hi || mask_lo) {
          const int up = khi - k0 - 4 * lhalf, dn = klo - k0 - 4 * lhalf;
          if (mask_hi) {
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = 8 * (r >> 2) + (r & 3) <= up ? e[r] : 0.f;
          }
          if (mask_lo) {
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = 8 * (r >> 2) + (r & 3) >= dn ? e[r] : 0.f;
          }
          if (odd) {
#pragma unroll
            for (int i = 0; i < DS * 2; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x) kt[i >> 1][i & 1][x] = finite2(kt[i >> 1][i & 1][x]);
            for (int j = 32 * sub; j < 32 * sub + 32; ++j) {
              const bool sees = kb + j <= khi && kb + j >= klo;
#pragma unroll
              for (int i = 0; i < DS * 4; ++i) {
                const u32x2_t x = *reinterpret_cast<const u32x2_t*>(
                    sk + j * D + ((i ^ swz<D>(j)) << 3) + 4 * lhalf);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const float v = bf16_to_f32((uint16_t)(x[y >> 1] >> (16 * (y & 1))));
                  acc[i >> 2][4 * (i & 3) + y] += sees ? v - v : 0.f;
                }
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t w[4], l[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float e0 = e[8 * u + 2 * x], e1 = e[8 * u + 2 * x + 1];
            const uint32_t x0 = __float_as_uint(e0), x1 = __float_as_uint(e1);
            rest += e0 + e1;
            w[x] = __builtin_amdgcn_perm(x1, x0, 0x07060302);  // their upper halves
            l[x] = pack_bf16x2(e0 - __uint_as_float(x0 & 0xffff0000u),
                               e1 - __uint_as_float(x1 & 0xffff0000u));
          }
          const bf16x8_t hi = bf8(u32x4_t{w[0], w[1], w[2], w[3]});
          const bf16x8_t lo = bf8(u32x4_t{l[0], l[1], l[2], l[3]});
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)
            acc[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf8(kt[ds][u]), hi, acc[ds], 0, 0, 0);
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)
            acc[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf8(kt[ds][u]), lo, acc[ds], 0, 0, 0);
        }
      }
    }
    stage ^= 1;
  }
  {
    float a, b;
    swap_pair<32>(rest, a, b);
    rest = a + b;
  }
  if (lhalf == 0 && rw + lrow < p.rows) {
    float* st = stats_of(ga, kvh, row);
    st[0] = mc;
    st[64] = -(delta + rest);
  }
  if (rw + lrow < p.rows) {
    uint16_t* out = (uint16_t*)ga.dq + (int64_t)tok * ga.st_dq + (int64_t)head * ga.sh_dq;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<u32x2_t*>(out + ds * 32 + 8 * j + 4 * lhalf) =
            u32x2_t{pack_bf16x2(acc[ds][4 * j] * p.scale, acc[ds][4 * j + 1] * p.scale),
                    pack_bf16x2(acc[ds][4 * j + 2] * p.scale, acc[ds][4 * j + 3] * p.scale)};
  }
}

// Where a slice's part of dk (0) or dv (1) of a key lies, in rows of head_dim f32.
__device__ inline int64_t part_at(const PArgs& p, int slice, int kvh, int what, int key) {
  return (((int64_t)slice * (p.H / p.G) + kvh) * 2 + what) * p.total + key;
}

// dk and dv, bf16.  One block = KW x RW waves: 32 keys each, and one RW-th of the rows of a tile
// each; tiles of BR rows, Q beside dO, pass through LDS.  S = Q . K^T and dP = dO . V^T put a key into
// a lane and rows into registers, from which P and dS feed dV^T = dO^T . P and dK^T = Q^T . dS.
// The shares are added up at the end; with SLICED a block takes every gridDim.y-th row tile and leaves its sums
// to packed_join_kernel (a kernel of its own: the few registers more would be spilled, beside DMA in
// flight, by all calls).  For d = 128, K and the two sums fill the registers and V is read from LDS.
// Same calls as dq's above: 510 us, four products at 0.96 PFLOP/s, matrix cores 45 % busy, the rest waits
// for LDS operands (16 reads of 16 bytes for 16 products of 32 cycles) and the exponentials between them;
// and 51 us, 23 %.
template <int D, int KW, int RW, int BR, bool SLICED>
__global__ __launch_bounds__(64 * KW * RW, D == 64 ? 3 : 2) void packed_dkdv_kernel(GArgs ga) {
  const PArgs& p = ga.a;
  constexpr int NW = KW * RW, KPW = 32, BK = KW * KPW, SHARE = BR / RW;
  constexpr bool V_LDS = D == 128;  // (its fragments would not fit the registers)
  constexpr int TILE = BR * D, STAGE = 2 * TILE + 512, NST = 2;  // 512: 1 KB of stats
  constexpr int KS = D / 16, DS = D / 32, CPR = D / 8, RPI = 64 / CPR, RPW = BR / NW;
  // (the sums that meet: (RW - 1) x KW x 64 x DS x 16 floats)
  static_assert(NST * STAGE >= (RW - 1) * KW * 64 * DS * 32, "they fit the stages");
  __shared__ __attribute__((aligned(1024))) uint16_t lds[NST * STAGE + (V_LDS ? BK * D : 0)];

  int kvh, tile;
  if (!tile_of(p, false, kvh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wid % KW, wr = wid / KW;
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int kw = tile * BK + wk * KPW;
  const int key = min(kw + lrow, p.total - 1);
  bf16x8_t kf[KS], vf[V_LDS ? 1 : KS];
  {
    const uint16_t* krow = (const uint16_t*)p.k + (int64_t)key * p.st_k + (int64_t)kvh * p.sh_k;
    const uint16_t* vrow = (const uint16_t*)p.v + (int64_t)key * p.st_v + (int64_t)kvh * p.sh_v;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = bf8(*reinterpret_cast<const u32x4_t*>(krow + ks * 16 + lhalf * 8));
      if constexpr (!V_LDS)
        vf[ks] = bf8(*reinterpret_cast<const u32x4_t*>(vrow + ks * 16 + lhalf * 8));
    }
  }
  int rlo, rhi;
  const bool in = rows_of(p, key, rlo, rhi);
  const Bounds bd = bounds_of<NW>(rlo, rhi, in);
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BR, t1 = bd.hi < 0 ? 0 : bd.hi / BR + 1;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(kf[ks]), "v"(vf[V_LDS ? 0 : ks]));

  const unsigned lds_base = (unsigned)(uintptr_t)lds;
  const int kin = lane / CPR, slot = lane % CPR;
  const char* qbase = (const char*)p.q + (int64_t)kvh * p.G * p.sh_q * 2;
  const char* gbase = (const char*)ga.g + (int64_t)kvh * p.G * ga.sh_g * 2;
  const char* sbase = (const char*)(ga.stats + (int64_t)kvh * ga.stat_tiles * 128);
  auto issue = [&](int t, int stage) {
    const unsigned sb = lds_base + (unsigned)(stage * STAGE * 2);
    const int tok0 = over(t * BR, p.by_g);
    const char* qt = qbase + (int64_t)tok0 * p.st_q * 2;
    const char* gt = gbase + (int64_t)tok0 * ga.st_g * 2;
#pragma unroll
    for (int i = 0; i < RPW / RPI; ++i) {
      const int r = RPW * wid + RPI * i + kin, from = min(t * BR + r, p.rows - 1);
      const int tok = over(from, p.by_g), g = from - tok * p.G;
      const unsigned ch = (unsigned)((slot ^ swz<D>(r)) * 16);
      const unsigned la = sb + (unsigned)((RPW * wid + RPI * i) * D * 2);
      dma16_so(qt, (unsigned)((tok - tok0) * (int)p.st_q + g * (int)p.sh_q) * 2u + ch, la);
      dma16_so(gt, (unsigned)((tok - tok0) * (int)ga.st_g + g * (int)ga.sh_g) * 2u + ch,
               la + TILE * 2);
    }
    // the stats of 64 rows are 512 bytes (twice, where a tile has no more; behind the last: the
    // last ones)
    if (wid == 0) {
      const int at = min(t * (BR / 64) + (BR == 128 ? lane >> 5 : 0), ga.stat_tiles - 1);
      dma16_so(sbase + (int64_t)t * (BR / 64) * 512,
               (unsigned)((at - t * (BR / 64)) * 512 + (lane & 31) * 16), sb + 2 * TILE * 2);
    }
  };
  const uint16_t* sv = lds + NST * STAGE;  // V of the block's keys
  const int slices = SLICED ? (int)gridDim.y : 1;
  const int from = SLICED ? t0 + (int)blockIdx.y : t0;  // (and every slices-th tile)
  if (V_LDS && from < t1) {
    const char* vt = (const char*)p.v + ((int64_t)tile * BK * p.st_v + (int64_t)kvh * p.sh_v) * 2;
#pragma unroll
    for (int i = 0; i < BK / NW / RPI; ++i) {
      const int r = BK / NW * wid + RPI * i + kin, row = min(r, p.total - 1 - tile * BK);
      dma16_so(vt, (unsigned)row * (unsigned)(p.st_v * 2) + (unsigned)((slot ^ swz<D>(r)) * 16),
               lds_base + (unsigned)(NST * STAGE + (BK / NW * wid + RPI * i) * D) * 2);
    }
  }
  const Transposed<D> tr(lane);
  f32x16_t dk[DS], dv[DS];
#pragma unroll
  for (int j = 0; j < DS; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[j][r] = dv[j][r] = 0.f;
  const float c = p.c;

  // P and dS of 32 rows at row r0 of the tile at sq, as the second products' operands: false
  // where no row of them sees a key.  odd: values that are not finite are to be left out.
  auto first = [&](int t, const uint16_t* sq, int r0, bf16x8_t (&bw)[2], bf16x8_t (&be)[2],
                   bool& odd) {
    const uint16_t* sg = sq + TILE;
    const int rb = t * BR + r0;
    odd = false;
    if (rb > bd.whi || rb + 32 <= bd.wlo) return false;
    const float* st = reinterpret_cast<const float*>(sg + TILE) + (r0 >> 6) * 128 + (r0 & 63);
    const bool mask_hi = rb + 31 > bd.hi_min, mask_lo = rb < bd.lo_max, mask = mask_hi || mask_lo;
    f32x16_t s, dp;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // (dP starts from -D)
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(st + 64 + 8 * j + 4 * lhalf);
#pragma unroll
      for (int i = 0; i < 4; ++i) dp[4 * j + i] = x[i];
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_chunk<D>(sq, r0 + lrow, 2 * ks + lhalf),
                                                  kf[ks], ks == 0 ? f32x16_t{} : s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          row_chunk<D>(sg, r0 + lrow, 2 * ks + lhalf),
          V_LDS ? row_chunk<D>(sv, wk * 32 + lrow, 2 * ks + lhalf) : vf[V_LDS ? 0 : ks], dp, 0, 0,
          0);
    }
    // (2 KS products, 2 KS reads and the 4 of -D; with D = 128 there are no registers for it)
    if constexpr (!V_LDS) reads_ahead<8, 2 * KS - 4, 1, 4>();
    if (mask) {
      // A weight of zero does not silence a row of Q or dO that is not finite, to the keys that
      // it does not see (as in packed_attn_kernel); such a row shows in S or dP of every key.
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum = fmaf(s[r], 0.f, fmaf(dp[r], 0.f, sum));
      odd = __any(sum != sum);
    }
    float w[16], e[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(st + 8 * j + 4 * lhalf);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * j + i;
        w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, x[i]));
        e[r] = w[r] * dp[r];
      }
    }
    if (mask) {
      const int up = rhi - rb - 4 * lhalf, dn = rlo - rb - 4 * lhalf;
      if (mask_hi) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool sees = 8 * (r >> 2) + (r & 3) <= up;
          w[r] = sees ? w[r] : 0.f;
          e[r] = sees ? e[r] : 0.f;
        }
      }
      if (mask_lo) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool sees = 8 * (r >> 2) + (r & 3) >= dn;
          w[r] = sees ? w[r] : 0.f;
          e[r] = sees ? e[r] : 0.f;
        }
      }
      if (odd) {
        for (int j = r0; j < r0 + 32; ++j) {
          const bool sees = t * BR + j <= rhi && t * BR + j >= rlo;
#pragma unroll
          for (int i = 0; i < DS * 4; ++i) {
            const int at = j * D + ((i ^ swz<D>(j)) << 3) + 4 * lhalf;
            const u32x2_t x = *reinterpret_cast<const u32x2_t*>(sg + at);
            const u32x2_t y = *reinterpret_cast<const u32x2_t*>(sq + at);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float a = bf16_to_f32((uint16_t)(x[z >> 1] >> (16 * (z & 1))));
              const float b = bf16_to_f32((uint16_t)(y[z >> 1] >> (16 * (z & 1))));
              dv[i >> 2][4 * (i & 3) + z] += sees && !(fabsf(a) < INFINITY) ? a : 0.f;
              dk[i >> 2][4 * (i & 3) + z] += sees ? b - b : 0.f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t pw[4], pe[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        pw[x] = pack_bf16x2(w[8 * u + 2 * x], w[8 * u + 2 * x + 1]);
        pe[x] = pack_bf16x2(e[8 * u + 2 * x], e[8 * u + 2 * x + 1]);
      }
      bw[u] = bf8(u32x4_t{pw[0], pw[1], pw[2], pw[3]});
      be[u] = bf8(u32x4_t{pe[0], pe[1], pe[2], pe[3]});
    }
    return true;
  };
  auto products = [&](const uint16_t* sq, int r0, const bf16x8_t (&bw)[2],
                      const bf16x8_t (&be)[2], auto some_odd) {
    const uint16_t* sg = sq + TILE;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        u32x4_t x = tr.read(sg, r0 + u * 16, ds), y = tr.read(sq, r0 + u * 16, ds);
        if constexpr (decltype(some_odd)::value) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = finite2(x[j]);
            y[j] = finite2(y[j]);
          }
        }
        dv[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf8(x), bw[u], dv[ds], 0, 0, 0);
        dk[ds] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf8(y), be[u], dk[ds], 0, 0, 0);
      }
    // (4 DS products and 8 DS reads)
    if constexpr (!decltype(some_odd)::value) reads_ahead<8, 4 * DS - 4, 2, 4>();
  };
  auto second = [&](const uint16_t* sq, int r0, const bf16x8_t (&bw)[2], const bf16x8_t (&be)[2],
                    bool odd) {
    if (__builtin_expect(odd, false))
      products(sq, r0, bw, be, std::true_type{});
    else
      products(sq, r0, bw, be, std::false_type{});
  };

  if (from < t1) issue(from, 0);
  int stage = 0;
  for (int t = from; t < t1; t += slices) {
    // tile t has landed and every wave is past the one before, whose stage is free
    dma_wait_barrier<0>();
    if (t + slices < t1) issue(t + slices, stage ^ 1);
    const uint16_t* sq = lds + stage * STAGE;
    stage ^= 1;
#pragma unroll 1
    for (int r0 = wr * SHARE; r0 < wr * SHARE + SHARE; r0 += 32) {
      bf16x8_t bw[2], be[2];
      bool odd = false;
      if (first(t, sq, r0, bw, be, odd)) second(sq, r0, bw, be, odd);
    }
  }
  // the rows' shares meet, through LDS
  float* meet = reinterpret_cast<float*>(lds) + (wk * 64 + lane) * 4;
  constexpr int PIECE = KW * 64 * 4, ALL = DS * 4 * PIECE;
  auto add = [&](f32x16_t (&x)[DS]) {
    __syncthreads();
    if (wr) {
#pragma unroll
      for (int i = 0; i < DS * 4; ++i)
        *reinterpret_cast<f32x4_t*>(meet + (wr - 1) * ALL + i * PIECE) =
            f32x4_t{x[i >> 2][4 * (i & 3)], x[i >> 2][4 * (i & 3) + 1], x[i >> 2][4 * (i & 3) + 2],
                    x[i >> 2][4 * (i & 3) + 3]};
    }
    __syncthreads();
    if (wr) return;
#pragma unroll
    for (int i = 0; i < DS * 4; ++i)
#pragma unroll
      for (int w = 0; w < RW - 1; ++w) {
        const f32x4_t y = *reinterpret_cast<f32x4_t*>(meet + w * ALL + i * PIECE);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i >> 2][4 * (i & 3) + e] += y[e];
      }
  };
  if constexpr (RW > 1) {
    add(dk);
    add(dv);
  }
  if (SLICED && wr == 0 && kw + lrow < p.total) {
    float* ok = ga.part + part_at(p, (int)blockIdx.y, kvh, 0, key) * D + 4 * lhalf;
    float* ov = ga.part + part_at(p, (int)blockIdx.y, kvh, 1, key) * D + 4 * lhalf;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<f32x4_t*>(ok + ds * 32 + 8 * j) = f32x4_t{
            dk[ds][4 * j], dk[ds][4 * j + 1], dk[ds][4 * j + 2], dk[ds][4 * j + 3]};
        *reinterpret_cast<f32x4_t*>(ov + ds * 32 + 8 * j) = f32x4_t{
            dv[ds][4 * j], dv[ds][4 * j + 1], dv[ds][4 * j + 2], dv[ds][4 * j + 3]};
      }
  } else if (wr == 0 && kw + lrow < p.total) {
    uint16_t* ok = (uint16_t*)ga.dk + (int64_t)key * ga.st_dk + (int64_t)kvh * ga.sh_dk;
    uint16_t* ov = (uint16_t*)ga.dv + (int64_t)key * ga.st_dv + (int64_t)kvh * ga.sh_dv;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = ds * 32 + 8 * j + 4 * lhalf;
        *reinterpret_cast<u32x2_t*>(ok + at) =
            u32x2_t{pack_bf16x2(dk[ds][4 * j] * p.scale, dk[ds][4 * j + 1] * p.scale),
                    pack_bf16x2(dk[ds][4 * j + 2] * p.scale, dk[ds][4 * j + 3] * p.scale)};
        *reinterpret_cast<u32x2_t*>(ov + at) =
            u32x2_t{pack_bf16x2(dv[ds][4 * j], dv[ds][4 * j + 1]),
                    pack_bf16x2(dv[ds][4 * j + 2], dv[ds][4 * j + 3])};
      }
  }
}

// f32, as packed_attn_f32_kernel: a block has 32 rows (dq) or 32 keys (dk, dv) in registers, its four
// waves take every fourth tile of 32 of the others from global memory and add up at the end.  Bound by
// those loads: 12 heads of 64, five sequences of up to 1501, dq 223 us, 76 TFLOP/s, dk and dv 370, 61 (one
// wave a SIMD 440, blocks of eight waves 422); 12 / 4 heads, 1000 + 780 + 439 tokens, 70 and 139; heads of 128,
// 2000 + 1441 tokens, 8 / 1 heads, 314 and 537 with the join, 1000 + 721 + 1 + 303, 32 / 8 heads, 370 and 452.
// Sum of the waves' [D][32] results, scaled, into rows out(i).
template <int ND, typename F>
__device__ inline void add_waves(float* so, const f32x16_t (&acc)[ND], float scale, F out) {
  constexpr int D = 32 * ND, OP = D + 4, VW = ND % 4 == 0 ? 4 : 2, NV = ND / VW;
  typedef float vf_t __attribute__((ext_vector_type(VW)));
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, h = lane >> 5;
  __syncthreads();
  float* row = so + (w * 32 + l31) * OP;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      vf_t x;
#pragma unroll
      for (int u = 0; u < VW; ++u) x[u] = acc[n * VW + u][i];
      *reinterpret_cast<vf_t*>(row + VW * (8 * (i >> 2) + 4 * h + (i & 3)) + 32 * VW * n) = x;
    }
  __syncthreads();
  for (int i = tid; i < 32 * (D / 4); i += 256) {
    const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
    float* to = out(rr);
    if (!to) continue;
    f32x4_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      x[k] = *reinterpret_cast<const f32x4_t*>(so + (k * 32 + rr) * OP + cc);
    *reinterpret_cast<f32x4_t*>(to + cc) = ((x[0] + x[1]) + (x[2] + x[3])) * scale;
  }
}

template <int ND>
__global__ __launch_bounds__(256) void packed_dq_f32_kernel(GArgs ga) {
  const PArgs& p = ga.a;
  constexpr int D = 32 * ND, NW = 4, NC = 4 * ND, OP = D + 4, BKV = 32;
  constexpr int VW = ND % 4 == 0 ? 4 : 2, NV = ND / VW;
  typedef float vf_t __attribute__((ext_vector_type(VW)));
  __shared__ __attribute__((aligned(16))) float so[NW * 32 * OP];
  int kvh, rt;
  if (!tile_of(p, true, kvh, rt)) return;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int r0 = rt * 32, row = min(r0 + l31, p.rows - 1);
  const int tok = over(row, p.by_g), head = kvh * p.G + row - tok * p.G;
  f32x4_t qf[NC], gf[NC];
  float delta = 0.f;
  {
    const float* qrow = (const float*)p.q + (int64_t)tok * p.st_q + (int64_t)head * p.sh_q;
    const float* grow = (const float*)ga.g + (int64_t)tok * ga.st_g + (int64_t)head * ga.sh_g;
    const float* orow = (const float*)p.o + (int64_t)tok * p.st_o + (int64_t)head * p.sh_o;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      qf[j] = *reinterpret_cast<const f32x4_t*>(qrow + 8 * j + 4 * h);
      gf[j] = *reinterpret_cast<const f32x4_t*>(grow + 8 * j + 4 * h);
      const f32x4_t o = *reinterpret_cast<const f32x4_t*>(orow + 8 * j + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) delta = fmaf(gf[j][e], o[e], delta);
    }
    float a, b;
    swap_pair<32>(delta, a, b);
    delta = a + b;
  }
  const float mc = offset_of(p.lse[(int64_t)tok * p.H + head]);
  if (w == 0 && h == 0 && r0 + l31 < p.rows) {
    float* st = stats_of(ga, kvh, row);
    st[0] = mc;
    st[64] = -delta;
  }
  int klo, khi;
  const bool in = keys_of(p, tok, klo, khi);
  const Bounds bd = bounds_of<1>(klo, khi, in);
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BKV, t1 = bd.hi < 0 ? 0 : bd.hi / BKV + 1;
  const float* kbase = (const float*)p.k + (int64_t)kvh * p.sh_k;
  const float* vbase = (const float*)p.v + (int64_t)kvh * p.sh_v;
  f32x16_t acc[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
  for (int t = t0 + w; t < t1; t += NW) {
    const int k0 = t * BKV;
    const int64_t at = min(k0 + l31, p.total - 1);
    const float *kr = kbase + at * p.st_k, *vr = vbase + at * p.st_v;
    f32x16_t s, dp;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = 0.f;
      dp[i] = -delta;
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(kr + 8 * j + 4 * h);
      const f32x4_t vf = *reinterpret_cast<const f32x4_t*>(vr + 8 * j + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[j][e], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[e], gf[j][e], dp, 0, 0, 0);
      }
    }
    const int up = khi - k0 - 4 * h, dn = klo - k0 - 4 * h;
    const bool mask = k0 + BKV - 1 > bd.hi_min || k0 < bd.lo_max;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 8 * (i >> 2) + (i & 3);
      const float e = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, mc)) * dp[i];
      s[i] = key <= up && key >= dn ? e : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
      const float* r = kbase + (int64_t)min(key, p.total - 1) * p.st_k + VW * l31;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        vf_t x = *reinterpret_cast<const vf_t*>(r + 32 * VW * n);
#pragma unroll
        for (int u = 0; u < VW; ++u) {
          if (mask) {
            // a weight of zero does not silence a key that is not finite: it is taken out, and
            // the rows that see it become NaN below
            x[u] = fabsf(x[u]) < INFINITY ? x[u] : 0.f;
          }
          acc[n * VW + u] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[u], s[i], acc[n * VW + u], 0, 0, 0);
        }
      }
    }
    if (mask) {
      // (a key that is not finite makes its score NaN or infinite: a row that sees it has NaN
      // weights or a weight of zero, whose product with it is NaN too)
      bool odd = false;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const f32x4_t kf = *reinterpret_cast<const f32x4_t*>(kr + 8 * j + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= !(fabsf(kf[e]) < INFINITY);
      }
      if (__any(odd)) {
        for (int j = 0; j < BKV; ++j) {
          const float* r = kbase + (int64_t)min(k0 + j, p.total - 1) * p.st_k;
          const bool sees = k0 + j <= khi && k0 + j >= klo;
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x =
                  r[VW * (8 * (i >> 2) + 4 * h + (i & 3)) + n % VW + 32 * VW * (n / VW)];
              acc[n][i] += sees ? x - x : 0.f;
            }
        }
      }
    }
  }
  add_waves<ND>(so, acc, p.scale, [&](int rr) -> float* {
    if (r0 + rr >= p.rows) return nullptr;
    const int t = over(r0 + rr, p.by_g), g = r0 + rr - t * p.G;
    return (float*)ga.dq + (int64_t)t * ga.st_dq + (int64_t)(kvh * p.G + g) * ga.sh_dq;
  });
}

// (d = 64: 256 registers, so that a SIMD has two waves; the compiler takes two more unasked)
template <int ND>
__global__ __launch_bounds__(256, ND == 2 ? 2 : 1) void packed_dkdv_f32_kernel(GArgs ga) {
  const PArgs& p = ga.a;
  constexpr int D = 32 * ND, NW = 4, NC = 4 * ND, OP = D + 4, BR = 32;
  constexpr int VW = ND % 4 == 0 ? 4 : 2, NV = ND / VW;
  typedef float vf_t __attribute__((ext_vector_type(VW)));
  __shared__ __attribute__((aligned(16))) float so[NW * 32 * OP];
  int kvh, tile;
  if (!tile_of(p, false, kvh, tile)) return;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  const int j0 = tile * 32, key = min(j0 + l31, p.total - 1);
  f32x4_t kf[NC], vf[NC];
  {
    const float* krow = (const float*)p.k + (int64_t)key * p.st_k + (int64_t)kvh * p.sh_k;
    const float* vrow = (const float*)p.v + (int64_t)key * p.st_v + (int64_t)kvh * p.sh_v;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      kf[j] = *reinterpret_cast<const f32x4_t*>(krow + 8 * j + 4 * h);
      vf[j] = *reinterpret_cast<const f32x4_t*>(vrow + 8 * j + 4 * h);
    }
  }
  int rlo, rhi;
  const bool in = rows_of(p, key, rlo, rhi);
  const Bounds bd = bounds_of<1>(rlo, rhi, in);
  const int t0 = bd.hi < 0 ? 0 : bd.lo / BR, t1 = bd.hi < 0 ? 0 : bd.hi / BR + 1;
  auto row_at = [&](const void* x, int64_t st, int64_t sh, int row) {
    row = min(row, p.rows - 1);
    const int tok = over(row, p.by_g), g = row - tok * p.G;
    return (const float*)x + (int64_t)tok * st + (int64_t)(kvh * p.G + g) * sh;
  };
  f32x16_t dk[ND], dv[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[n][i] = dv[n][i] = 0.f;
  const int slice = (int)blockIdx.y, slices = (int)gridDim.y;
  for (int t = t0 + slice * NW + w; t < t1; t += NW * slices) {
    const int rb = t * BR;
    const float* qr = row_at(p.q, p.st_q, p.sh_q, rb + l31);
    const float* gr = row_at(ga.g, ga.st_g, ga.sh_g, rb + l31);
    const float* st = stats_of(ga, kvh, rb);
    f32x16_t s, dp;
    float mc[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(st + 8 * j + 4 * h);
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(st + 64 + 8 * j + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mc[4 * j + i] = x[i];
        dp[4 * j + i] = y[i];
        s[4 * j + i] = 0.f;
      }
    }
    bool odd = false;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const f32x4_t q = *reinterpret_cast<const f32x4_t*>(qr + 8 * j + 4 * h);
      const f32x4_t g = *reinterpret_cast<const f32x4_t*>(gr + 8 * j + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        odd |= !(fabsf(q[e]) < INFINITY) || !(fabsf(g[e]) < INFINITY);
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(q[e], kf[j][e], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x2f32(g[e], vf[j][e], dp, 0, 0, 0);
      }
    }
    const int up = rhi - rb - 4 * h, dn = rlo - rb - 4 * h;
    odd = (rb + BR - 1 > bd.hi_min || rb < bd.lo_max) && __any(odd);
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int at = 8 * (i >> 2) + (i & 3);
      const bool sees = at <= up && at >= dn;
      const float x = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, mc[i]));
      s[i] = sees ? x : 0.f;
      e[i] = sees ? x * dp[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = rb + 8 * (i >> 2) + 4 * h + (i & 3);
      const float* q = row_at(p.q, p.st_q, p.sh_q, row) + VW * l31;
      const float* g = row_at(ga.g, ga.st_g, ga.sh_g, row) + VW * l31;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        vf_t x = *reinterpret_cast<const vf_t*>(g + 32 * VW * n);
        vf_t y = *reinterpret_cast<const vf_t*>(q + 32 * VW * n);
#pragma unroll
        for (int u = 0; u < VW; ++u) {
          if (odd) {  // (see packed_dq_f32_kernel)
            x[u] = fabsf(x[u]) < INFINITY ? x[u] : 0.f;
            y[u] = fabsf(y[u]) < INFINITY ? y[u] : 0.f;
          }
          const int k = n * VW + u;
          dv[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[u], s[i], dv[k], 0, 0, 0);
          dk[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(y[u], e[i], dk[k], 0, 0, 0);
        }
      }
    }
    if (odd) {
      for (int j = 0; j < BR; ++j) {
        const float* q = row_at(p.q, p.st_q, p.sh_q, rb + j);
        const float* g = row_at(ga.g, ga.st_g, ga.sh_g, rb + j);
        const bool sees = rb + j <= rhi && rb + j >= rlo;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int col = VW * (8 * (i >> 2) + 4 * h + (i & 3)) + n % VW + 32 * VW * (n / VW);
            const float x = g[col], y = q[col];
            dv[n][i] += sees && !(fabsf(x) < INFINITY) ? x : 0.f;
            dk[n][i] += sees ? y - y : 0.f;
          }
      }
    }
  }
  if (slices > 1) {
    auto part = [&](int what, int i) {
      return j0 + i < p.total ? ga.part + part_at(p, slice, kvh, what, j0 + i) * D : nullptr;
    };
    add_waves<ND>(so, dk, 1.f, [&](int i) { return part(0, i); });
    add_waves<ND>(so, dv, 1.f, [&](int i) { return part(1, i); });
    return;
  }
  auto out = [&](void* x, int64_t st, int64_t sh, int i) -> float* {
    return j0 + i < p.total ? (float*)x + (int64_t)(j0 + i) * st + (int64_t)kvh * sh : nullptr;
  };
  add_waves<ND>(so, dk, p.scale, [&](int i) { return out(ga.dk, ga.st_dk, ga.sh_dk, i); });
  add_waves<ND>(so, dv, 1.f, [&](int i) { return out(ga.dv, ga.st_dv, ga.sh_dv, i); });
}

// dk and dv from the parts of their tiles' blocks, in the blocks' order: a thread 4 values of one
template <int D, typename T>
__global__ __launch_bounds__(256) void packed_join_kernel(GArgs ga, int slices) {
  const PArgs& p = ga.a;
  const int kvh = (int)blockIdx.y, what = (int)blockIdx.z;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= (int64_t)p.total * D) return;
  const float* x = ga.part + part_at(p, 0, kvh, what, 0) * D + i;
  const int64_t step = part_at(p, 1, 0, 0, 0) * D;
  f32x4_t sum = *reinterpret_cast<const f32x4_t*>(x);
  for (int k = 1; k < slices; ++k) sum += *reinterpret_cast<const f32x4_t*>(x + k * step);
  if (!what) sum *= p.scale;
  T* to = (T*)(what ? ga.dv : ga.dk) + i / D * (what ? ga.st_dv : ga.st_dk) +
          kvh * (what ? ga.sh_dv : ga.sh_dk) + i % D;
  if constexpr (std::is_same<T, float>::value)
    *reinterpret_cast<f32x4_t*>(to) = sum;
  else
    *reinterpret_cast<u32x2_t*>(to) =
        u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
}

// ---- launch ----------------------------------------------------------------------------
// Tiles of `each` out of n, and the grid over them (see tile_of).
int64_t plan_tiles(PArgs& p, int64_t n, int each, int Hkv) {
  p.tiles = (int)((n + each - 1) / each);
  p.residues = 1;
  while (Hkv * p.residues % 8) p.residues *= 2;
  p.units = Hkv * p.residues / 8;
  return (int64_t)8 * p.units * ((p.tiles + p.residues - 1) / p.residues);
}
PArgs args_of(const PackedAttnArgs& a) {
  PArgs p{};
  p.q = a.q.x; p.k = a.k.x; p.v = a.v.x; p.o = const_cast<void*>(a.o.x); p.lse = a.lse;
  p.st_q = a.q.st; p.sh_q = a.q.sh; p.st_k = a.k.st; p.sh_k = a.k.sh;
  p.st_v = a.v.st; p.sh_v = a.v.sh; p.st_o = a.o.st; p.sh_o = a.o.sh;
  p.starts = a.starts; p.B = (int)a.B; p.total = (int)a.total; p.H = a.H; p.G = a.H / a.Hkv;
  p.rows = p.total * p.G;
  p.by_g = divisor_of(p.G);
  p.causal = a.causal; p.window = a.causal && a.window < (1 << 30) ? a.window : 0;
  p.scale = a.scale;
  p.c = (float)(1.44269504088896340736 * (double)a.scale);
  p.tail = a.tail;
  return p;
}

// An order for n rows (or keys) in tiles of `each`: for several sequences, where the blocks are
// more than two of a CU and there is room for it.
bool ordered(int64_t B, int64_t n, int each, int Hkv) {
  const int64_t tiles = (n + each - 1) / each;
  return B > 1 && tiles * Hkv >= 512 && tiles <= kOrderTiles;
}
// Keys of a tile of dk and dv.  With few tiles the longest takes longer than a CU's share of the work:
// half as many keys, and twice the rows at a time (32 / 8 heads of 128: one sequence of 4096
// 331 us, 440 with 128 keys; four of up to 4096, 10.8 k tokens, 696 and 665).
int key_tile(int64_t total, int Hkv, int d, bool f32) {
  return f32 ? 32 : d == 128 && Hkv * ((total + 127) / 128) <= 512 ? 64 : 128;
}

}  // namespace

int64_t packed_attention_workspace_bytes(int64_t B, int64_t total, int H, int Hkv, int dtype) {
  const int64_t rows = total * (H / Hkv);
  const int each = dtype == BLT_DTYPE_F32 ? 32 : 128;
  return ordered(B, rows, each, Hkv) ? (rows + each - 1) / each * 4 : 0;
}

int launch_packed_attention(const PackedAttnArgs& a, void* ws, hipStream_t s) {
  PArgs p = args_of(a);
  const bool f32 = a.dtype == BLT_DTYPE_F32;
  const int each = f32 ? 32 : 128;
  const int64_t nb = plan_tiles(p, p.rows, each, a.Hkv);
  if (nb > 0x7fffffff) return fail(BLT_ERR_SHAPE, "packed_attention: too many tiles");
  if (ordered(a.B, p.rows, each, a.Hkv)) {
    hipLaunchKernelGGL(packed_order_kernel, dim3(1), dim3(1024), 0, s, p, each, 0, (int*)ws, nullptr);
    p.order = (const int*)ws;
  }
  const dim3 grid((unsigned)nb), block(256);
  if (f32 && a.d == 64)
    hipLaunchKernelGGL((packed_attn_f32_kernel<2>), grid, block, 0, s, p);
  else if (f32)
    hipLaunchKernelGGL((packed_attn_f32_kernel<4>), grid, block, 0, s, p);
  else if (a.d == 64 && p.lse)
    hipLaunchKernelGGL((packed_attn_kernel<64, true>), grid, block, 0, s, p);
  else if (a.d == 64)
    hipLaunchKernelGGL((packed_attn_kernel<64, false>), grid, block, 0, s, p);
  else if (p.lse)
    hipLaunchKernelGGL((packed_attn_kernel<128, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((packed_attn_kernel<128, false>), grid, block, 0, s, p);
  BLT_LAUNCH_CHECK("packed_attn_kernel");
  return 0;
}

// Blocks that share a key tile's rows, each every so-many-th row tile: where the tiles are fewer than
// keep the device even, at most 8 (`seen`: about how many rows a key has, 0 for unknown: a block
// gets 256 of them or more; f32 with d = 128, whose tiles take longest, 128: 54 sequences of up to
// 93, 8 / 1 heads, 72 us and 126, but 20 of 100, 12 / 4 heads of 64, 40 and 35).  Their parts cost a
// join of 4 to 10 us.  dk and dv, sliced with the join and in one block:
//   f32   12 / 4 heads of 64: 1000 + 77 + 439 tokens 110 and 191 us, 1000 + 780 + 439 139 and 195;
//         8 / 1 heads of 128: 2 x 2000 827 and 1880; but with more blocks 12 / 12 of 64, 2 x 1000,
//         133 and 124
//   bf16  12 / 4 heads of 64: the first of these 33 and 87, 8 x 1000 78 and 120; 12 heads: 1 x
//         4096 99 and 131; 8 / 1 heads of 128: 2 x 2000 89 and 268; 32 / 8 of 128: 1 x 2048 106 and
//         133, but 4 x 500 68 and 52 (so fewer where keys have few rows), 4 x 100 31 and 20
int key_slices(int64_t total, int Hkv, int d, bool f32, int64_t seen) {
  const int each = key_tile(total, Hkv, d, f32);
  const int64_t blocks = (total + each - 1) / each * Hkv;
  const int64_t fill = f32 ? 1024 : d == 64 ? 768 : seen == 0 || seen >= 4096 ? 512 : 256;
  if (blocks < 1 || blocks >= fill) return 1;
  const int64_t most = seen > 0 ? std::max<int64_t>(seen / (f32 && d == 128 ? 128 : 256), 1) : 8;
  return (int)std::min<int64_t>(std::min<int64_t>(fill / blocks, 8), most);
}
// the stats of 64 rows each, the orders of row and key tiles, then the parts of dk and dv
int64_t stats_bytes(int64_t total, int H, int Hkv) {
  return (int64_t)Hkv * ((total * (H / Hkv) + 63) / 64) * 512 + 2 * kOrderTiles * 4;
}
int64_t packed_attention_backward_workspace_bytes(int64_t total, int H, int Hkv, int d, int dtype) {
  const int slices = key_slices(total, Hkv, d, dtype == BLT_DTYPE_F32, 0);
  return stats_bytes(total, H, Hkv) +
         (slices > 1 ? slices * total * Hkv * 8 * d : 0);
}

int launch_packed_attention_backward(const PackedAttnArgs& a, const PackedGradArgs& g, void* ws,
                                     hipStream_t s) {
  GArgs p{};
  p.a = args_of(a);
  p.g = g.g.x; p.st_g = g.g.st; p.sh_g = g.g.sh;
  p.dq = const_cast<void*>(g.dq.x); p.st_dq = g.dq.st; p.sh_dq = g.dq.sh;
  p.dk = const_cast<void*>(g.dk.x); p.st_dk = g.dk.st; p.sh_dk = g.dk.sh;
  p.dv = const_cast<void*>(g.dv.x); p.st_dv = g.dv.st; p.sh_dv = g.dv.sh;
  p.stats = (float*)ws;
  p.stat_tiles = (p.a.rows + 63) / 64;
  const bool f32 = a.dtype == BLT_DTYPE_F32;
  const int bk = key_tile(a.total, a.Hkv, a.d, f32), bq = f32 ? 32 : 128;
  const int64_t mean = a.total / std::max<int64_t>(a.B, 1);
  const int64_t seen = std::max<int64_t>(p.a.window ? std::min<int64_t>(mean, p.a.window + bk) : mean,
                                         1) * p.a.G;
  const int slices = key_slices(a.total, a.Hkv, a.d, f32, seen);
  int* orders = (int*)(p.stats + (int64_t)a.Hkv * p.stat_tiles * 128);
  const bool by_rows = ordered(a.B, p.a.rows, bq, a.Hkv), by_keys = ordered(a.B, a.total, bk, a.Hkv * slices);
  if (by_rows || by_keys) {
    hipLaunchKernelGGL(packed_order_kernel, dim3(2), dim3(1024), 0, s, p.a, bq, bk,
                       by_rows ? orders : nullptr, by_keys ? orders + kOrderTiles : nullptr);
  }
  GArgs pk = p;
  const int64_t nq = plan_tiles(p.a, p.a.rows, bq, a.Hkv);
  const int64_t nk = plan_tiles(pk.a, a.total, bk, a.Hkv);
  if (by_rows) p.a.order = orders;
  if (by_keys) pk.a.order = orders + kOrderTiles;
  if (nq > 0x7fffffff || nk > 0x7fffffff)
    return fail(BLT_ERR_SHAPE, "packed_attention_backward: too many tiles");
  pk.part = (float*)((char*)ws + stats_bytes(a.total, a.H, a.Hkv));
  const dim3 gq((unsigned)nq), gk((unsigned)nk, slices), block(256);
  if (f32 && a.d == 64) {
    hipLaunchKernelGGL((packed_dq_f32_kernel<2>), gq, block, 0, s, p);
    hipLaunchKernelGGL((packed_dkdv_f32_kernel<2>), gk, block, 0, s, pk);
  } else if (f32) {
    hipLaunchKernelGGL((packed_dq_f32_kernel<4>), gq, block, 0, s, p);
    hipLaunchKernelGGL((packed_dkdv_f32_kernel<4>), gk, block, 0, s, pk);
  } else if (a.d == 64) {
    hipLaunchKernelGGL((packed_dq_kernel<64>), gq, block, 0, s, p);
    if (slices > 1)
      hipLaunchKernelGGL((packed_dkdv_kernel<64, 4, 1, 64, true>), gk, block, 0, s, pk);
    else
      hipLaunchKernelGGL((packed_dkdv_kernel<64, 4, 1, 64, false>), gk, block, 0, s, pk);
  } else {
    hipLaunchKernelGGL((packed_dq_kernel<128>), gq, block, 0, s, p);
    if (slices > 1)  // (never where tiles have 128 keys: they are too many for it)
      hipLaunchKernelGGL((packed_dkdv_kernel<128, 2, 4, 128, true>), gk, dim3(512), 0, s, pk);
    else if (bk == 64)
      hipLaunchKernelGGL((packed_dkdv_kernel<128, 2, 4, 128, false>), gk, dim3(512), 0, s, pk);
    else
      hipLaunchKernelGGL((packed_dkdv_kernel<128, 4, 2, 64, false>), gk, dim3(512), 0, s, pk);
  }
  if (slices > 1) {
    const dim3 grid((unsigned)((a.total * a.d + 1023) / 1024), (unsigned)a.Hkv, 2);
    if (f32 && a.d == 64)
      hipLaunchKernelGGL((packed_join_kernel<64, float>), grid, block, 0, s, pk, slices);
    else if (f32)
      hipLaunchKernelGGL((packed_join_kernel<128, float>), grid, block, 0, s, pk, slices);
    else if (a.d == 64)
      hipLaunchKernelGGL((packed_join_kernel<64, uint16_t>), grid, block, 0, s, pk, slices);
    else
      hipLaunchKernelGGL((packed_join_kernel<128, uint16_t>), grid, block, 0, s, pk, slices);
  }
  BLT_LAUNCH_CHECK("packed_dq_kernel, packed_dkdv_kernel");
  return 0;
}

}  // namespace blt
