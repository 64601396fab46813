// Attention of a chunk of new tokens over the paged K/V cache: prompts whose first pages
// are cached already, the next chunk of a long prompt, single tokens.
//
// Sequence b brings rows cu[b] .. cu[b + 1] of a flat batch; its last row is token
// ctx_lens[b] - 1 of the sequence, whose keys and values are in the cache, the new ones
// among them. Row i sees the keys 0 .. its own position:
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m),  m the running maximum.
//
// A workgroup owns a kv head and a block of rows that are (token, query head of the
// group) pairs, tokens outermost: K and V are read once for all heads of the group, and a
// block ends few tokens behind its first, so that little of the diagonal is computed in
// vain. Products and softmax are those of the learner's attention (attention_tiles.h). Three
// kernels share them: a light one, one for many rows over long contexts and one for few.
//
// Weights go into the second product as two bf16 terms, 17 bits, as those of single tokens
// do (paged_attn.hip); the result's error against 64 bits is then that of its own rounding
// (0.00166, with one term 0.0023). It costs half as much matrix work again. us, one card,
// one term and two: 2 x 4096 behind 8192, 64/8 heads of 128 2729 and 3584 (1150 TFLOP/s with
// the second terms, a product of 8192^3 1296); 2048 behind 14336, 28/4 501 and 647; 30 single
// tokens and 2 x 512 behind up to 2900, 32/8 102 and 119; 16 x 20..121 behind 1040, 28/4 43
// and 51. The first of these keeps matrix cores and vector units busy for 58 % of the time
// each; little of one wave's products hides behind the vector work of the SIMD's other.
// Tried there, with one term (2690): 128 rows a workgroup 2796, the light kernel 2975, 64 rows
// a wave (one wave a SIMD) 3755, twelve waves of 32 (three a SIMD) 2856 for 2767, priorities
// of waves even. 6 single tokens behind 20 to 32 thousand, 40/8 heads 129 us = 4.5 TB/s, K and
// V read once. 16 x 20..121 behind 1040 and 10 x 200..350 behind none, 28/4 (24 us): a
// workgroup's start (lengths, pages, rows, one behind the other) and up to 36 blocks or 6
// tiles. 5 tokens behind 1040, 14/2 of 64 10.8: two launches of such chains.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "attention_tiles.h"

namespace {

constexpr int BLOCK = 32, RING = 4;     // keys of a block of the deep kernel, blocks in LDS
constexpr int AHEAD = 1024;             // keys whose cache rows are looked up at once
constexpr int TILE = 64;        // keys of a tile
constexpr int LEAST = 256;      // of a slice, at least

// x / n for 0 <= x < 2^30 as a product: ceil(2^(31 + shift) / n), shift = ceil(log2(n)), is
// too large by less than 1 and x times that less than 2^(31 + shift), so the result is exact.
struct Divisor {
  int n;
  uint32_t inverse;
  int shift;
  Divisor(int64_t n = 1) : n((int)n), shift(0) {
    while ((1ll << shift) < n) ++shift;
    inverse = (uint32_t)(((1ull << (31 + shift)) + n - 1) / n);
  }
  DEV_INLINE int of(int x) const { return (int)(__umulhi(2u * x, inverse) >> shift); }
};

struct Chunk {
  const __hip_bfloat16* q;      // (T, H, D), heads and rows these elements apart
  int64_t q_t, q_h;
  const __hip_bfloat16 *key, *value;    // (pages, block, KV, D)
  const int *tables, *cu, *ctx;         // (B, width), (B + 1), (B)
  __hip_bfloat16* out;                  // (T, H, D)
  float *o_part, *ml_part;              // (slices, T, H, D), (slices, T, H, 2)
  int T, B, H, KV, width, pages, block;
  Divisor by_block, by_group;           // group: query heads of a kv head
  float scale_log2;

  DEV_INLINE int first(int b) const { return min(max(cu[b], 0), T); }
};

// The sequence whose rows block `s` of the launch holds: its first row, end and keys, its
// number, and the block it starts at. Sequence b starts at block floor(cu[b] G / ROWS) + b:
// as many as it may need and no sum over those before it.
struct Sequence { int b, first, end, ctx, start; };

template <int ROWS>
DEV_INLINE int start_of(const Chunk& a, int row, int b) { return row * a.by_group.n / ROWS + b; }

template <int ROWS>
DEV_INLINE Sequence sequence_of(const Chunk& a, int s) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.B;
  while (n > 64) {              // 64 candidates a turn
    const int step = (n + 63) / 64, i = lane * step;
    const bool before = i < n && start_of<ROWS>(a, a.first(lo + i), lo + i) <= s;
    const int k = max(1, (int)__popcll(__ballot(before)));
    lo += (k - 1) * step;
    n = min(step, n - (k - 1) * step);
  }
  // of the last 64 all that is wanted is on its way at once: one behind the other the
  // three numbers are a microsecond each
  const int b = lo + min(lane, n - 1);
  const int first = a.first(b), end = a.first(b + 1), ctx = a.ctx[b];
  const int start = start_of<ROWS>(a, first, b);
  const int k = max(1, (int)__popcll(__ballot(lane < n && start <= s))) - 1;
  return {lo + k, __builtin_amdgcn_readlane(first, k), __builtin_amdgcn_readlane(end, k),
          __builtin_amdgcn_readlane(ctx, k), __builtin_amdgcn_readlane(start, k)};
}

// Rows that no sequence has are zeros: of this kv head, by workgroup `mine` of `all`.
template <int D>
DEV_INLINE void clear_rows(const Chunk& a, int kv, int group, int mine, int all) {
  const int from = a.first(a.B), to = a.first(0), units = group * D / 8;
  const int64_t n = (int64_t)(to + a.T - from) * units;
  for (int64_t i = (int64_t)mine * blockDim.x + threadIdx.x; i < n; i += (int64_t)all * blockDim.x) {
    const int row = (int)(i / units), t = row < to ? row : from + row - to;
    *reinterpret_cast<u32x4*>(a.out + ((int64_t)t * a.H + kv * group) * D + i % units * 8) =
        u32x4{0, 0, 0, 0};
  }
}

template <typename T>
using LDS = __attribute__((address_space(3))) T;
template <typename T>
DEV_INLINE LDS<T>* at(uint32_t lds) { return (LDS<T>*)(uintptr_t)lds; }

// What a workgroup works on: rows block0 .. of sequence q's (token, head) pairs, and a slice
// of the keys that its last row sees. Of those a lane's own row: token t, its head, and
// keys; least: keys that all rows of the wave see.
struct Work {
  Sequence q;
  int rows, block0, t, head, mine, least, begin, end;
  bool live;
};

// Whether there is any work; if not, rows of no sequence have been cleared. NW waves own 32
// rows each, or one block of them is every wave's.
template <int D, int NW>
DEV_INLINE bool find_work(const Chunk& a, Work& w) {
  constexpr int ROWS = NW * WROWS;
  const int group = a.by_group.n, blocks = gridDim.x / a.KV;
  const int kv = blockIdx.x % a.KV, s = blocks - 1 - blockIdx.x / a.KV;   // longest first
  const int none = start_of<ROWS>(a, a.first(a.B), a.B);
  w.q = sequence_of<ROWS>(a, s);
  if (s >= none) {
    if (blockIdx.y == 0) clear_rows<D>(a, kv, group, s - none, blocks - none);
    return false;
  }
  w.block0 = (s - w.q.start) * ROWS;
  w.rows = (w.q.end - w.q.first) * group;
  if (w.block0 < 0 || w.block0 >= w.rows) return false;
  const int before = w.q.ctx - (w.q.end - w.q.first);
  const int reach = (int)min((int64_t)a.width * a.block, (int64_t)1 << 30);
  auto keys_of = [&](int r) { return max(0, min(before + a.by_group.of(r) + 1, reach)); };
  const int r0 = w.block0 + (NW == 1 ? 0 : wave_id() * WROWS), row = r0 + (threadIdx.x & 31);
  const int r = min(row, w.rows - 1), of = a.by_group.of(r);
  w.live = row < w.rows;
  w.t = w.q.first + of;
  w.head = kv * group + r - of * group;
  w.mine = keys_of(r);
  w.least = keys_of(min(r0, w.rows - 1));
  const int all = keys_of(min(w.block0 + ROWS, w.rows) - 1), slices = gridDim.y;
  const int per = max(LEAST, ((all + slices - 1) / slices + TILE - 1) / TILE * TILE);
  w.begin = blockIdx.y * per;
  w.end = min(all, w.begin + per);
  return true;
}

template <int D>
DEV_INLINE void load_queries(const Chunk& a, const Work& w, bf16v8 (&qf)[D / 16]) {
  const __hip_bfloat16* qp = a.q + w.t * a.q_t + w.head * a.q_h + ((threadIdx.x & 63) >> 5) * 8;
  #pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const bf16v8*>(qp + ks * 16);
}

// Scores of keys that this lane's row does not see; k0: the first
DEV_INLINE void hide(f32x16& st, const Work& w, int k0) {
  const int seen = min(w.mine, w.end) - k0 - 4 * ((int)(threadIdx.x & 63) >> 5);
  #pragma unroll
  for (int j = 0; j < 16; ++j)
    if (seen <= acc_row(j, 0)) st[j] = -1e30f;
}

// The second term of weights 8 k .. 8 k + 7, whose first is hi = pack8(p, k): p = hi + lo,
// off by 2^-16 of p at most. (Made and used beside the products with hi: with those of both
// terms behind it all 2 x 4096 behind 8192 take 3689 us for 3583.)
DEV_INLINE bf16v8 rest8(const f32x16& p, const bf16v8& hi, int k) {
  f32x16 rest;
  #pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = p[8 * k + j] - (float)hi[j];
  return pack8(rest, 0);
}

// acc += values of 16 keys times a term of their weights
template <int D>
DEV_INLINE void add_values(f32x16 (&acc)[D / 32], const bf16v8 (&v)[D / 32], const bf16v8& p) {
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = mfma(v[dt], p, acc[dt]);
}

// Scores into weights, first terms into hi. They carry 2^-m of their own, and their sum; what m moved by is
// returned, and what was weighed before is to be rescaled by 2 to that.
// m is a whole number and may lag by 8: weights that differ by powers of two round alike,
// so that tiles and slices do not change the result beyond the order of fp32 sums, and
// sums are hardly ever rescaled. Nothing is lost by a leading weight that is not 1, as its
// two terms carry 17 bits of it.
template <int NS>
DEV_INLINE float weigh(f32x16 (&st)[NS], bf16v8 (&hi)[NS][2], float& m, float& sum, float scale_log2) {
  float mx = st[0][0];
  #pragma unroll
  for (int n = 0; n < NS; ++n)
    #pragma unroll
    for (int j = 0; j < 16; ++j) mx = fmaxf(mx, st[n][j]);
  mx = halves_max(mx) * scale_log2;
  const float to = mx > m + 8.f ? ceilf(mx) : m, fall = m - to;
  m = to;
  sum = 0.f;
  #pragma unroll
  for (int n = 0; n < NS; ++n) {
    #pragma unroll
    for (int j = 0; j < 16; ++j) {
      st[n][j] = __builtin_amdgcn_exp2f(st[n][j] * scale_log2 - m);
      sum += st[n][j];
    }
    #pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) hi[n][k2] = pack8(st[n], k2);
  }
  return fall;
}

template <int D>
DEV_INLINE void rescale(float fall, float& lsum, f32x16 (&acc)[D / 32]) {
  const float alpha = __builtin_amdgcn_exp2f(fall);
  lsum *= alpha;
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
    #pragma unroll
    for (int j = 0; j < 16; ++j) acc[dt][j] *= alpha;
}

// The sum of a part in which a row sees no key; told by its bits, as a sum that is no number
// (a query's that is none) is neither more nor less than any.
constexpr float NONE = -1.f;
DEV_INLINE bool is_none(float sum) { return __float_as_uint(sum) == __float_as_uint(NONE); }

// This lane's row, or its part of it, into memory.
template <int D>
DEV_INLINE void finish(const Chunk& a, const Work& w, float m, float lsum, f32x16 (&acc)[D / 32]) {
  const bool seen = w.mine > w.begin;
  lsum = halves_sum(lsum);
  if (__any(!seen)) {           // what its masked scores became is no number
    lsum = seen ? lsum : 0.f;
    #pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
      #pragma unroll
      for (int j = 0; j < 16; ++j) acc[dt][j] = seen ? acc[dt][j] : 0.f;
  }
  const int64_t at = (int64_t)w.t * a.H + w.head;
  if (gridDim.y == 1) {
    store_rows<D>(acc, seen ? 1.f / lsum : 0.f, a.out + at * D, w.live);
    return;
  }
  const int64_t part = blockIdx.y * (int64_t)a.T * a.H + at;
  if (w.begin < w.end) store_rows_f32<D>(acc, a.o_part + part * D, w.live);
  if ((threadIdx.x & 63) < 32 && w.live) {
    a.ml_part[part * 2] = m;
    a.ml_part[part * 2 + 1] = seen ? lsum : NONE;
  }
}

// Rows of K and V of a tile: fetched into registers, then stored to LDS. Rows
// past the end and pages that are none read as zeros.
template <int D, int KEYS, int NT>
struct Staged {
  static constexpr int UN = D / 8, STEP = NT / UN, PER = KEYS / STEP;
  static_assert(KEYS % STEP == 0, "tile does not divide");
  u32x4 k[PER], v[PER];
  int page[PER];                // of the rows that are fetched next
  int there;                    // a bit a row: k and v hold it

  DEV_INLINE static int row(int i) { return i * STEP + threadIdx.x / UN; }

  DEV_INLINE void look(const Chunk& a, const int* table, int at, int end) {
    #pragma unroll
    for (int i = 0; i < PER; ++i) page[i] = table[a.by_block.of(min(at + row(i), end - 1))];
  }
  DEV_INLINE void fetch(const Chunk& a, int kv, int at, int end) {
    there = 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = at + row(i), in = j - a.by_block.of(j) * a.block;
      const bool ok = (j < end) & ((unsigned)page[i] < (unsigned)a.pages);
      const int64_t off = ((int64_t)(ok ? page[i] * a.block + in : 0) * a.KV + kv) * D +
                          threadIdx.x % UN * 8;
      there |= (int)ok << i;
      k[i] = *reinterpret_cast<const u32x4*>(a.key + off);
      v[i] = *reinterpret_cast<const u32x4*>(a.value + off);
    }
  }
  DEV_INLINE void store(char* kt, char* vt) {
    if (__any(there != (1 << PER) - 1)) {
      #pragma unroll
      for (int i = 0; i < PER; ++i)
        if (!(there >> i & 1)) k[i] = v[i] = u32x4{0, 0, 0, 0};
    }
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = row(i) * (2 * D) + ((threadIdx.x % UN ^ swz<D>(row(i))) << 4);
      *reinterpret_cast<u32x4*>(kt + at) = k[i];
      *reinterpret_cast<u32x4*>(vt + at) = v[i];
    }
  }
};

// Shorter contexts and fewer rows: tiles of 64 keys, the next one on its way into registers
// while this one's scores, weights and values follow one another. It starts in half the
// time of the kernel below. (Two waves a workgroup and tiles of 32, with weights of one term:
// 10 x 200..350 behind none, 28/4 heads 22.7 us for 22.1, 80 x 100 33.8 for 37.4, 4 x 1200 85
// for 67.)
template <int D, int NW>
__global__ __launch_bounds__(NW * 64, 2)
void chunk_attn_kernel(Chunk a) {
  constexpr int NS = TILE / 32, TB = TILE * D * 2;
  Work w;
  if (!find_work<D, NW>(a, w)) return;
  const int kv = blockIdx.x % a.KV;
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const Frags<D> fr;
  bf16v8 qf[D / 16];
  load_queries<D>(a, w, qf);
  float m = -1e30f, lsum = 0.f;
  f32x16 acc[D / 32];
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = zero16();

  if (w.begin < w.end) {
    const int* table = a.tables + (int64_t)w.q.b * a.width;
    const int most = __builtin_amdgcn_readlane(w.mine, 31);       // of the wave's rows
    Staged<D, TILE, NW * 64> tile;
    tile.look(a, table, w.begin, w.end);
    tile.fetch(a, kv, w.begin, w.end);
    tile.look(a, table, w.begin + TILE, w.end);
    tile.store(smem, smem + TB);
    __syncthreads();
    int turn = 0;
    for (int k0 = w.begin; k0 < w.end; k0 += TILE, turn ^= 1) {
      char *kt = smem + turn * (2 * TB), *vt = kt + TB;
      const bool more = k0 + TILE < w.end;
      if (more) {
        tile.fetch(a, kv, k0 + TILE, w.end);
        tile.look(a, table, k0 + 2 * TILE, w.end);
      }
      if (k0 < most && w.block0 + wave_id() * WROWS < w.rows) {   // wave-uniform
        f32x16 st[NS];
        #pragma unroll
        for (int n = 0; n < NS; ++n) {
          st[n] = zero16();
          #pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) st[n] = mfma(fr.row(kt, n, ks), qf[ks], st[n]);
        }
        if (k0 + TILE > min(w.least, w.end)) {          // the diagonal, or the end
          #pragma unroll
          for (int n = 0; n < NS; ++n) hide(st[n], w, k0 + n * 32);
        }
        bf16v8 hi[NS][2];
        float sum;
        const float fall = weigh(st, hi, m, sum, a.scale_log2);
        if (__any(fall < 0.f)) rescale<D>(fall, lsum, acc);
        lsum += sum;
        #pragma unroll
        for (int n = 0; n < NS; ++n)
          #pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            bf16v8 v[D / 32];
            #pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) v[dt] = fr.col(vt, n * 32 + k2 * 16, dt);
            add_values<D>(acc, v, hi[n][k2]);
            add_values<D>(acc, v, rest8(st[n], hi[n][k2], k2));
          }
      }
      if (more) {
        char* next = smem + (turn ^ 1) * (2 * TB);
        tile.store(next, next + TB);
        __syncthreads();
      }
    }
  }
  finish<D>(a, w, m, lsum, acc);
}

// Few rows of a sequence, as single tokens: a workgroup's four waves have the same 32 rows
// and 32 keys of a tile of 128 each, with a softmax of their own, joined at the end. (One
// wave for all keys of a tile is a chain four times as long, beside three that wait.)
template <int D>
__global__ __launch_bounds__(256, 2)
void chunk_few_kernel(Chunk a) {
  constexpr int NW = 4, KEYS = NW * 32, TB = KEYS * D * 2, LD = D + 4;
  Work w;
  if (!find_work<D, 1>(a, w)) return;
  const int kv = blockIdx.x % a.KV, wave = wave_id();
  extern __shared__ __attribute__((aligned(256))) char smem[];
  const Frags<D> fr;
  bf16v8 qf[D / 16];
  load_queries<D>(a, w, qf);
  float m = -1e30f, lsum = 0.f;
  f32x16 acc[D / 32];
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = zero16();

  if (w.begin < w.end) {
    const int* table = a.tables + (int64_t)w.q.b * a.width;
    Staged<D, KEYS, NW * 64> tile;
    tile.look(a, table, w.begin, w.end);
    tile.fetch(a, kv, w.begin, w.end);
    tile.look(a, table, w.begin + KEYS, w.end);
    for (int t0 = w.begin; t0 < w.end; t0 += KEYS) {
      tile.store(smem, smem + TB);
      __syncthreads();
      if (t0 + KEYS < w.end) {
        tile.fetch(a, kv, t0 + KEYS, w.end);
        tile.look(a, table, t0 + 2 * KEYS, w.end);
      }
      const int k0 = t0 + wave * 32;
      if (k0 < w.end) {                                 // wave-uniform
        f32x16 st[1] = {zero16()};
        #pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) st[0] = mfma(fr.row(smem, wave, ks), qf[ks], st[0]);
        if (k0 + 32 > min(w.least, w.end)) hide(st[0], w, k0);
        bf16v8 hi[1][2];
        float sum;
        const float fall = weigh(st, hi, m, sum, a.scale_log2);
        if (__any(fall < 0.f)) rescale<D>(fall, lsum, acc);
        lsum += sum;
        #pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          bf16v8 v[D / 32];
          #pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) v[dt] = fr.col(smem + TB, wave * 32 + k2 * 16, dt);
          add_values<D>(acc, v, hi[0][k2]);
          add_values<D>(acc, v, rest8(st[0], hi[0][k2], k2));
        }
      }
      __syncthreads();
    }
  }

  float* parts = reinterpret_cast<float*>(smem);        // (waves, 32, LD), then (waves, 32, 2)
  float* ml = parts + NW * WROWS * LD;
  const int l = threadIdx.x & 63;
  lsum = halves_sum(lsum);
  store_rows_f32<D>(acc, parts + (wave * WROWS + (l & 31)) * LD, true);
  if (l < 32) {
    const bool seen = min(w.mine, w.end) > w.begin + wave * 32;
    ml[(wave * WROWS + l) * 2] = seen ? m : -1e30f;
    ml[(wave * WROWS + l) * 2 + 1] = seen ? lsum : NONE;
  }
  __syncthreads();
  const int row = threadIdx.x / 8, r = w.block0 + row, of = a.by_group.of(r);
  if (r >= w.rows) return;
  float top = -1e30f, total = 0.f, f[NW];
  bool seen[NW], any = false;
  #pragma unroll
  for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[(i * WROWS + row) * 2]);
  #pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float sum = ml[(i * WROWS + row) * 2 + 1];
    seen[i] = !is_none(sum);
    any |= seen[i];
    f[i] = __builtin_amdgcn_exp2f(ml[(i * WROWS + row) * 2] - top);
    total += seen[i] ? f[i] * sum : 0.f;
  }
  const int64_t at = (int64_t)(w.q.first + of) * a.H + kv * a.by_group.n + r - of * a.by_group.n;
  const int64_t part = blockIdx.y * (int64_t)a.T * a.H + at;
  #pragma unroll
  for (int d0 = 0; d0 < D / 8; d0 += 4) {
    const int d = threadIdx.x % 8 * 4 + d0 * 8;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    #pragma unroll
    for (int i = 0; i < NW; ++i)
      if (seen[i])              // else what is there is no number
        o += f[i] * *reinterpret_cast<const f32x4*>(parts + (i * WROWS + row) * LD + d);
    if (gridDim.y > 1) {
      *reinterpret_cast<f32x4*>(a.o_part + part * D + d) = o;
      continue;
    }
    const float inv = any ? 1.f / total : 0.f;
    bf16v4 y;
    #pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (__bf16)(o[j] * inv);
    *reinterpret_cast<bf16v4*>(a.out + at * D + d) = y;
  }
  if (gridDim.y > 1 && threadIdx.x % 8 == 0) {
    a.ml_part[part * 2] = top;
    a.ml_part[part * 2 + 1] = any ? total : NONE;
  }
}

// Addresses of a block's fragments, in registers: which block it is goes into the
// instructions' offsets.
template <int D>
struct Places {
  uint32_t row, lo[D / 32], hi[D / 32];
  DEV_INLINE explicit Places(uint32_t lds) {
    const Frags<D> f;
    keep(row = lds + f.row_off);        // lds ends on 256 bytes
    #pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      keep(lo[dt] = lds + (f.tr_lo ^ (dt << 6)));
      keep(hi[dt] = lds + (f.tr_hi ^ (dt << 6)));
    }
  }
  DEV_INLINE static void keep(uint32_t& x) { asm volatile("" : "+v"(x)); }
  DEV_INLINE bf16v8 keys(uint32_t block, int ks) const { return *at<bf16v8>((row ^ (ks << 5)) + block); }
  DEV_INLINE bf16v8 values(uint32_t block, int k0, int dt) const {
    const bf16v4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at<bf16v4>(lo[dt] + block + k0 * (2 * D)));
    const bf16v4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(at<bf16v4>(hi[dt] + block + k0 * (2 * D)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Not to be moved behind what follows
DEV_INLINE void hold(bf16v8& x) {
  u32x4 w = __builtin_bit_cast(u32x4, x);
  asm volatile("" : "+v"(w));
  x = __builtin_bit_cast(bf16v8, w);
}

// 16 B a lane from `from` into LDS at lds + 16 * lane. m0 is lost to the compiler, which
// warns that nothing keeps it: nothing has to.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
DEV_INLINE void load_to_lds(uint32_t lds, uint64_t from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(from) : "m0");
}
#pragma clang diagnostic pop
// Until at most VM of this wave's loads are on their way and its LDS accesses are done.
template <int VM>
DEV_INLINE void landed() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(VM) : "memory"); }
DEV_INLINE void meet() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Rows of K and V on pages straight into LDS, a block of BLOCK at a time. Which cache row a
// key is in stands in LDS for two runs of AHEAD keys; a row that is none (past the end, or
// its page is outside the cache) has the sign bit there and is overwritten with zeros once
// it has landed.
template <int D, int NW>
struct Paged {
  static constexpr int UN = D / 8, PER = BLOCK * UN / (NW * 64);   // lanes of a row, loads of a wave
  static_assert(PER * NW * 64 == BLOCK * UN, "block does not divide");
  static constexpr int TB = BLOCK * D * 2, BYTES = 2 * RING * TB + 2 * AHEAD * 4 + 16;
  uint32_t lds;
  uint64_t k[PER];              // key of row 0, this lane's 16 bytes
  uint64_t value;               // from there to the value
  uint32_t step;                // bytes from cache row to row

  DEV_INLINE int row(int n) const { return (wave_id() * PER + n) * (64 / UN) + (threadIdx.x & 63) / UN; }
  DEV_INLINE Paged(const Chunk& a, uint32_t lds, int kv)
      : lds(lds), value(reinterpret_cast<uint64_t>(a.value) - reinterpret_cast<uint64_t>(a.key)),
        step(a.KV * D * 2) {
    #pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int64_t off = (int64_t)kv * D + ((threadIdx.x % UN) ^ swz<D>(row(n))) * 8;
      k[n] = reinterpret_cast<uint64_t>(a.key + off);
    }
  }
  DEV_INLINE uint32_t keys(int slot) const { return lds + (slot & (RING - 1)) * TB; }
  DEV_INLINE uint32_t values(int slot) const { return lds + (RING + (slot & (RING - 1))) * TB; }
  DEV_INLINE LDS<int>* lines() const { return at<int>(lds + 2 * RING * TB); }
  DEV_INLINE LDS<int>* bad() const { return lines() + 2 * AHEAD; }   // the first key on no page
  DEV_INLINE int line(int block, int n) const { return lines()[(block * BLOCK + row(n)) & (2 * AHEAD - 1)]; }

  // key j's row of the cache, or the sign bit
  DEV_INLINE static int row_of(const Chunk& a, const int* table, int j, int end) {
    const int of = a.by_block.of(j), page = j < end ? table[of] : -1;
    return (unsigned)page < (unsigned)a.pages ? page * a.block + j - of * a.block : (int)0x80000000;
  }
  // the cache rows of keys begin + from .. + AHEAD
  template <int UNROLL>
  DEV_INLINE void look(const Chunk& a, const int* table, int begin, int from, int end) const {
    #pragma unroll UNROLL
    for (int i = 0; i < AHEAD; i += NW * 64) {
      const int x = from + i + (int)threadIdx.x, j = begin + x, row = row_of(a, table, j, end);
      lines()[x & (2 * AHEAD - 1)] = row;
      if ((row < 0) & (j < end)) __hip_atomic_fetch_min(bad(), j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  struct Lines { int of[PER]; };
  DEV_INLINE Lines lines_of(int block) const {
    Lines l;
    #pragma unroll
    for (int n = 0; n < PER; ++n) l.of[n] = line(block, n);
    return l;
  }
  // the same from the table, before lines are there
  DEV_INLINE Lines look_up(const Chunk& a, const int* table, int begin, int block, int end) const {
    Lines l;
    #pragma unroll
    for (int n = 0; n < PER; ++n) l.of[n] = row_of(a, table, begin + block * BLOCK + row(n), end);
    return l;
  }
  DEV_INLINE void load(uint32_t to, uint64_t more, const Lines& l) const {
    #pragma unroll
    for (int n = 0; n < PER; ++n)
      load_to_lds(__builtin_amdgcn_readfirstlane(to + (wave_id() * PER + n) * 1024),
                  k[n] + more + (uint64_t)(uint32_t)(l.of[n] & 0x7fffffff) * step);
  }
  DEV_INLINE void load_keys(int slot, const Lines& l) const { load(keys(slot), 0, l); }
  DEV_INLINE void load_values(int slot, const Lines& l) const { load(values(slot), value, l); }
  // zeros for the rows that are none; this wave's have landed
  DEV_INLINE void mend(uint32_t slot, const Lines& l) const {
    #pragma unroll
    for (int n = 0; n < PER; ++n)
      if (l.of[n] < 0)
        *at<u32x4>(slot + (wave_id() * PER + n) * 1024 + (threadIdx.x & 63) * 16) = u32x4{0, 0, 0, 0};
  }
};

// Many rows and long contexts: keys come in blocks of 32 through rings of four in LDS. A
// turn of the loop makes the weights of block i beside the products with the keys of block
// i + 1, which wait in registers, then adds the values of block i while the keys of block
// i + 2 are read; the keys of block i + 5 and the values of i + 3 set out meanwhile.
template <int D, int NW>
__global__ __launch_bounds__(NW * 64, 2)
void chunk_deep_kernel(Chunk a) {
  Work w;
  if (!find_work<D, NW>(a, w)) return;
  const int kv = blockIdx.x % a.KV, begin = w.begin, end = w.end;
  extern __shared__ __attribute__((aligned(256))) char smem[];   // all of LDS: from 0 on
  const uint32_t lds = (uint32_t)(uintptr_t)(LDS<char>*)smem;
  const Places<D> fr(lds);
  bf16v8 qf[D / 16];
  load_queries<D>(a, w, qf);
  float m = -1e30f, lsum = 0.f;
  f32x16 acc[D / 32];
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = zero16();

  if (begin < end) {
    const int* table = a.tables + (int64_t)w.q.b * a.width;
    const Paged<D, NW> tile(a, lds, kv);
    constexpr int PER = Paged<D, NW>::PER;
    auto l1 = tile.look_up(a, table, begin, 0, end), l2 = tile.look_up(a, table, begin, 1, end),
         l3 = tile.look_up(a, table, begin, 2, end), l4 = tile.look_up(a, table, begin, 3, end),
         l5 = tile.look_up(a, table, begin, 4, end);
    if (threadIdx.x == 0) *tile.bad() = 0x7fffffff;
    __syncthreads();
    tile.template look<AHEAD / (NW * 64)>(a, table, begin, 0, end);
    tile.load_keys(0, l1);
    tile.load_keys(1, l2);
    tile.load_keys(2, l3);
    tile.load_values(0, l1);
    tile.load_keys(3, l4);
    tile.load_values(1, l2);
    landed<2 * PER>();
    tile.mend(tile.keys(0), l1);
    tile.mend(tile.keys(1), l2);
    tile.mend(tile.keys(2), l3);
    tile.mend(tile.values(0), l1);
    landed<2 * PER>();
    meet();
    bf16v8 kf[D / 16];
    auto read_keys = [&](int block) {
      #pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) kf[ks] = fr.keys(tile.keys(block) - lds, ks);
    };
    auto scores = [&](f32x16& to) {
      to = zero16();
      #pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) to = mfma(kf[ks], qf[ks], to);
    };
    f32x16 s0[1], s1[1];
    read_keys(0);
    scores(s0[0]);
    read_keys(1);
    landed<2 * PER>();
    meet();                     // block 4's keys land where block 0's are
    tile.load_keys(4, l5);
    tile.load_values(2, l3);
    l3 = l4;                    // of the values that set out next
    l4 = l5;
    l5 = tile.lines_of(5);      // and of the keys
    int whole = 0;              // keys before this one all rows see, and their pages are there
    // Block i, whose scores are st; the next one's into next.
    auto turn = [&](int i, f32x16 (&st)[1], f32x16& next) {
      const int k0 = begin + i * BLOCK;
      // keys that not all rows see, or rows that are none in what lands by the turn's end
      const bool careful = k0 + 4 * BLOCK > whole;
      tile.load_keys(i + 5, l5);
      tile.load_values(i + 3, l3);
      l3 = l4;
      l4 = l5;
      l5 = tile.lines_of(i + 6);
      bf16v8 v[2][D / 32];
      auto read_values = [&](int k2) {
        #pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) v[k2][dt] = fr.values(tile.values(i) - lds, k2 * 16, dt);
      };
      read_values(0);
      if (careful) hide(st[0], w, k0);
      scores(next);             // past the end of what lies there, unused
      bf16v8 hi[1][2];
      float sum;
      const float fall = weigh(st, hi, m, sum, a.scale_log2);
      // here, and not behind the branch
      hold(hi[0][0]);
      hold(hi[0][1]);
      #pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) hold(v[0][dt]);
      if (__any(fall < 0.f)) rescale<D>(fall, lsum, acc);
      lsum += sum;
      read_values(1);
      read_keys(i + 2);
      #pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) add_values<D>(acc, v[k2], hi[0][k2]);
      #pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) add_values<D>(acc, v[k2], rest8(st[0], hi[0][k2], k2));
      landed<4 * PER>();
      if (careful) {
        tile.mend(tile.keys(i + 3), tile.lines_of(i + 3));
        tile.mend(tile.values(i + 1), tile.lines_of(i + 1));
        landed<4 * PER>();
      }
      meet();
    };
    for (int i = 0; begin + i * BLOCK < end; i += 2) {   // an even number: the last may be empty
      // the next run of cache rows, of which the last turns look past the end
      if (i % (AHEAD / BLOCK) == AHEAD / BLOCK / 2) {
        const int from = i * BLOCK + AHEAD / 2;
        if (begin + from < end + 8 * BLOCK) tile.template look<1>(a, table, begin, from, end);
      }
      whole = min(min(w.least, end), __builtin_amdgcn_readfirstlane(*tile.bad()));
      turn(i, s0, s1[0]);
      turn(i + 1, s1, s0[0]);
    }
    landed<0>();                        // nothing may land in LDS that is another's
  }

  finish<D>(a, w, m, lsum, acc);
}

// The slices of a row joined; eight elements a thread.
template <int D>
__global__ __launch_bounds__(256)
void chunk_join_kernel(Chunk a, int slices) {
  const int64_t n = (int64_t)a.T * a.H, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (D / 8);
  if (row >= n) return;
  const int t = (int)(row / a.H);
  if (t < a.first(0) || t >= a.first(a.B)) return;
  float m = -1e30f, l = 0.f, o[8] = {};
  bool any = false;
  for (int z = 0; z < slices; ++z) {
    const float2 ml = reinterpret_cast<const float2*>(a.ml_part)[z * n + row];
    if (is_none(ml.y)) continue;
    any = true;
    const float m_new = fmaxf(m, ml.x);
    const float keep = __builtin_amdgcn_exp2f(m - m_new), add = __builtin_amdgcn_exp2f(ml.x - m_new);
    const f32x4* p = reinterpret_cast<const f32x4*>(a.o_part + (z * n + row) * D + i % (D / 8) * 8);
    #pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = o[j] * keep + p[j / 4][j % 4] * add;
    l = l * keep + ml.y * add;
    m = m_new;
  }
  bf16x8 out;
  #pragma unroll
  for (int j = 0; j < 8; ++j) out.v[j] = f2bf(any ? o[j] / l : 0.f);
  *reinterpret_cast<bf16x8*>(a.out + row * D + i % (D / 8) * 8) = out;
}

// q's rows where 16 B loads can walk them, else a copy of them
torch::Tensor rows_on_16(const torch::Tensor& q) {
  const bool ok = q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  return ok ? q : q.clone(at::MemoryFormat::Contiguous);
}

}  // namespace

// q (T, H, D) in any strides; caches (pages, block, KV, D); block_tables (B, width); cu (B + 1)
// the first row of every sequence and the end; ctx_lens (B) tokens in the cache, the rows'
// own among them. longest: the most rows of one sequence, which picks the kernel alone.
torch::Tensor paged_attention_chunk(torch::Tensor q, torch::Tensor kcache, torch::Tensor vcache,
                                    torch::Tensor block_tables, torch::Tensor cu,
                                    torch::Tensor ctx_lens, double scale, int64_t longest) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16,
              "paged_attention_chunk: q (rows, heads, head_dim) in bfloat16 on the GPU");
  TORCH_CHECK(kcache.dim() == 4 && kcache.sizes() == vcache.sizes() && kcache.is_contiguous() &&
              vcache.is_contiguous() && kcache.scalar_type() == at::kBFloat16 &&
              vcache.scalar_type() == at::kBFloat16,
              "paged_attention_chunk: caches (pages, block, kv heads, head_dim), contiguous bfloat16");
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2), KV = kcache.size(2);
  TORCH_CHECK(D == 64 || D == 128, "paged_attention_chunk: head_dim 64 or 128");
  TORCH_CHECK(kcache.size(3) == D && KV > 0 && H % KV == 0 && kcache.size(1) > 0,
              "paged_attention_chunk: heads or head_dim of q and the cache");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt &&
              block_tables.is_contiguous(), "paged_attention_chunk: block_tables (sequences, pages), int32");
  const int64_t B = block_tables.size(0), width = block_tables.size(1);
  TORCH_CHECK(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.dim() == 1 &&
              cu.numel() == B + 1 && ctx_lens.scalar_type() == at::kInt && ctx_lens.is_contiguous() &&
              ctx_lens.dim() == 1 && ctx_lens.numel() == B,
              "paged_attention_chunk: cu (sequences + 1) and context_lens (sequences), int32");
  for (const auto* t : {&kcache, &vcache, &block_tables, &cu, &ctx_lens})
    TORCH_CHECK(t->device() == q.device(), "paged_attention_chunk: all on q's device");
  for (const auto* t : {&kcache, &vcache})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "paged_attention_chunk: caches on 16 bytes");
  // hidden scores are -1e30 before they are scaled, and have to be far below the others then;
  // scaled ones have to stay within 2^29, as a larger maximum's rounding is no weight's
  // exponent any more
  TORCH_CHECK(scale >= 1e-12 && scale <= 1e6, "paged_attention_chunk: a scale of 1e-12 to 1e6");
  TORCH_CHECK(longest >= 0, "paged_attention_chunk: longest");
  TORCH_CHECK(T * H < (1ll << 30) && kcache.size(0) * kcache.size(1) < (1ll << 31) && B < (1 << 24),
              "paged_attention_chunk: too many rows");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = torch::empty({T, H, D}, q.options());
  if (T == 0 || H == 0) return out;
  if (B == 0 || width == 0 || kcache.size(0) == 0) return out.zero_();   // no key at all
  auto rows = rows_on_16(q);
  const int64_t block = kcache.size(1);
  Chunk a{};
  auto bf = [](const torch::Tensor& t) { return reinterpret_cast<__hip_bfloat16*>(t.data_ptr()); };
  a.q = bf(rows);
  a.q_t = rows.stride(0);
  a.q_h = rows.stride(1);
  a.key = bf(kcache);
  a.value = bf(vcache);
  a.tables = block_tables.data_ptr<int>();
  a.cu = cu.data_ptr<int>();
  a.ctx = ctx_lens.data_ptr<int>();
  a.out = bf(out);
  a.T = T;
  a.B = B;
  a.H = H;
  a.KV = KV;
  a.width = width;
  a.pages = kcache.size(0);
  a.block = block;
  a.by_block = Divisor(block);
  a.by_group = Divisor(H / KV);
  a.scale_log2 = (float)scale * LOG2E;
  // one block more than the sequences can have, which clears the rows of none
  auto grid_of = [&](int64_t rows) { return (T * (H / KV) / rows + B + 1) * KV; };
  const int64_t most = width * block;           // keys at most
  auto stream = at::cuda::getCurrentCUDAStream();
  auto check = [](int64_t grid) {
    TORCH_CHECK(grid < (1ll << 31), "paged_attention_chunk: too many rows");
    return grid;
  };
  auto deep = [&] {
    constexpr int DIM = 128, NW = 8, lds = Paged<DIM, NW>::BYTES;
    static const hipError_t raised = hipFuncSetAttribute(
        reinterpret_cast<const void*>(chunk_deep_kernel<DIM, NW>),
        hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    TORCH_CHECK(raised == hipSuccess, "paged_attention_chunk: LDS");
    hipLaunchKernelGGL((chunk_deep_kernel<DIM, NW>), dim3(check(grid_of(NW * WROWS))),
                       dim3(NW * 64), lds, stream, a);
    HIP_CHECK_LAST();
  };
  auto sliced = [&](auto d_, auto few_) {
    constexpr int DIM = decltype(d_)::value;
    constexpr bool FEWS = decltype(few_)::value;
    const int64_t grid = check(grid_of(FEWS ? WROWS : 4 * WROWS));
    // Slices where the workgroups leave CUs idle (a CU holds two of four waves, with heads
    // of 64 four), of 256 keys at least and from three of them on: the join is a launch of 4
    // us. 5 tokens behind 1040, 14/2 heads of 64 11.2 us, one slice 12.8. Half, so and twice
    // as many: 36 x 43..68 behind up to 8435, 8/2 of 64 109, 68 and 63, 2 x 36..826 behind
    // 6000, 32/8 of 128 45.4, 43.5 and 45.6, 6 x 1 behind 20 to 32 thousand, 40/8 209, 129 and 133.
    const int slices = most < 3 * LEAST ? 1 : (int)std::max<int64_t>(
        1, std::min<int64_t>({(DIM == 64 ? 1024 : 512) / grid, (most + LEAST - 1) / LEAST, 64}));
    torch::Tensor part;
    if (slices > 1) {
      const int64_t n = slices * T * H;
      part = torch::empty({n * (D + 2)}, q.options().dtype(at::kFloat));
      a.o_part = part.data_ptr<float>();
      a.ml_part = a.o_part + n * D;
    }
    const dim3 launch(grid, slices);
    if constexpr (FEWS) {
      constexpr int lds = 4 * WROWS * (DIM + 6) * 4;
      static_assert(lds >= 4 * 4 * WROWS * DIM, "tile and join share LDS");
      static const hipError_t raised = hipFuncSetAttribute(
          reinterpret_cast<const void*>(chunk_few_kernel<DIM>),
          hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      TORCH_CHECK(raised == hipSuccess, "paged_attention_chunk: LDS");
      hipLaunchKernelGGL(chunk_few_kernel<DIM>, launch, dim3(256), lds, stream, a);
    } else {
      hipLaunchKernelGGL((chunk_attn_kernel<DIM, 4>), launch, dim3(256), 4 * TILE * DIM * 2, stream, a);
    }
    HIP_CHECK_LAST();
    if (slices > 1) {
      hipLaunchKernelGGL(chunk_join_kernel<DIM>, dim3(CDIV(T * H * (DIM / 8), 256)), dim3(256), 0,
                         stream, a, slices);
      HIP_CHECK_LAST();
    }
  };
  // By rows of a sequence, keys a row sees on average (if sequences are alike and their
  // tables as wide as they need) and workgroups. us, light and deep kernel, 128 rows and
  // 256 a workgroup: 2 x 4096 behind 8192, 64/8 heads 3820 and 3580; 2048 behind 14336, 28/4
  // 701 and 631; 8192 behind none, 28/4 693 and 661; 16 x 20..121 behind 1040, 28/4 53.2 and
  // 50.5; but 2 x 1024 behind 2048, 40/8 185 and 199, 4 x 1200 behind none, 28/4 80 and 89,
  // 512 behind 4096 67 and 167, 10 x 200..350 24.0 and 33.3, single tokens among two chunks
  // 118 and 162.
  // Up to 64 rows a sequence, where a step waits for chains and not for memory. us, light
  // kernel and few rows: a token behind 1000, 14/2 heads of 64 11.5 and 9.9, 40/8 of 128
  // 14.2 and 12.3; 64 x 1 behind 500, 14/2 12.1 and 7.8, behind 3000 31 and 28; of 128, where a
  // CU's LDS holds two workgroups, it depends on the batch: 8 x 1 behind 2000, 28/4 18.7
  // and 19.9, 8 x 5 behind 1040 16.5 and 17.9, 4 x 1 behind 20000, 40/8 72 and 81, 64 x 1
  // behind 3000, 28/4 103 and 118, but 40/8 223 and 187, 2 x 2 behind 500, 28/4 16.9 and 11.6,
  // 64 x 5 behind 500, 12/2 17.6 and 12.7.
  const bool few = longest * (H / KV) <= 64 && (D == 64 || B == 1);
  auto by_rows = [&](auto d_) {
    if (few) sliced(d_, std::true_type{});
    else sliced(d_, std::false_type{});
  };
  if (D == 128 && T * (H / KV) >= 256 * B && most - T / (2 * B) >= 1024 && grid_of(256) >= 160)
    deep();
  else if (D == 128)
    by_rows(std::integral_constant<int, 128>{});
  else
    by_rows(std::integral_constant<int, 64>{});
  return out;
}
