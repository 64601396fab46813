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
// vain. Products and softmax are those of the learner's attention (attention_tiles.h).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "attention_tiles.h"

namespace {

constexpr int KEYS = 64;        // of a tile
constexpr int LEAST = 256;      // keys of a slice, at least

struct Chunk {
  const __hip_bfloat16* q;      // (T, H, D), heads and rows these elements apart
  int64_t q_t, q_h;
  const __hip_bfloat16 *key, *value;    // (pages, block, KV, D)
  const int *tables, *cu, *ctx;         // (B, width), (B + 1), (B)
  __hip_bfloat16* out;                  // (T, H, D)
  float *o_part, *ml_part;              // (slices, T, H, D), (slices, T, H, 2)
  int T, B, H, KV, width, pages, block, shift;
  float scale_log2;

  DEV_INLINE int first(int b) const { return min(max(cu[b], 0), T); }
};

// The sequence whose rows block `s` of the launch holds. Sequence b's blocks start at
// floor(cu[b] G / ROWS) + b: as many as it may need and no sum over those before it.
template <int ROWS>
DEV_INLINE int start_of(const Chunk& a, int b, int group) { return a.first(b) * group / ROWS + b; }

template <int ROWS>
DEV_INLINE int sequence_of(const Chunk& a, int s, int group) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.B;
  while (n > 1) {               // 64 candidates a turn
    const int step = (n + 63) / 64, b = lane * step;
    const bool before = b < n && start_of<ROWS>(a, lo + b, group) <= s;
    const int k = max(1, (int)__popcll(__ballot(before)));
    lo += (k - 1) * step;
    n = min(step, n - (k - 1) * step);
  }
  return lo;
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

// Rows of K and V of a tile, which lie on pages: fetched into registers, then stored to
// LDS. Rows past the end and pages that are none read as zeros.
template <int D, int NT>
struct Paged {
  static constexpr int UN = D / 8, STEP = NT / UN, PER = KEYS / STEP;
  u32x4 k[PER], v[PER];
  int page[PER];                // of the rows that are fetched next
  int there;                    // a bit a row: k and v hold it

  DEV_INLINE static int row(int i) { return i * STEP + threadIdx.x / UN; }

  DEV_INLINE void look(const Chunk& a, const int* table, int at, int end) {
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = min(at + row(i), end - 1);
      page[i] = table[a.shift >= 0 ? j >> a.shift : j / a.block];
    }
  }
  DEV_INLINE void fetch(const Chunk& a, int kv, int at, int end) {
    there = 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = at + row(i);
      const bool ok = j < end && (unsigned)page[i] < (unsigned)a.pages;
      const int in = a.shift >= 0 ? j & (a.block - 1) : j % a.block;
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

template <int D, int NW>
__global__ __launch_bounds__(NW * 64, 2)
void chunk_attn_kernel(Chunk a) {
  constexpr int ROWS = NW * WROWS, NS = KEYS / 32, TB = KEYS * D * 2;
  const int group = a.H / a.KV, blocks = gridDim.x / a.KV;
  const int kv = blockIdx.x % a.KV, s = blocks - 1 - blockIdx.x / a.KV;   // longest first
  const int slices = gridDim.y, z = blockIdx.y;
  const int none = start_of<ROWS>(a, a.B, group);
  if (s >= none) {
    if (z == 0) clear_rows<D>(a, kv, group, s - none, blocks - none);
    return;
  }
  const int b = __builtin_amdgcn_readfirstlane(sequence_of<ROWS>(a, s, group));
  const int row0 = a.first(b), tokens = a.first(b + 1) - row0;
  const int block0 = (s - start_of<ROWS>(a, b, group)) * ROWS, rows = tokens * group;
  if (block0 < 0 || block0 >= rows) return;

  const int wave = wave_id(), l = threadIdx.x & 63, half = l >> 5;
  const int before = a.ctx[b] - tokens, reach = (int)min((int64_t)a.width * a.block, (int64_t)1 << 30);
  auto keys_of = [&](int r) { return max(0, min(before + r / group + 1, reach)); };
  const int r0 = block0 + wave * WROWS, r = r0 + (l & 31);
  const int rr = min(r, rows - 1), t = row0 + rr / group, head = kv * group + rr % group;
  const int mine = keys_of(rr);                                 // keys this lane's row sees
  const int least = keys_of(min(r0, rows - 1)), most = keys_of(min(r0 + WROWS, rows) - 1);
  const int all = keys_of(min(block0 + ROWS, rows) - 1);        // of the workgroup
  // slices of the workgroup's own keys
  const int per = max(LEAST, ((all + slices - 1) / slices + KEYS - 1) / KEYS * KEYS);
  const int begin = z * per, end = min(all, begin + per);

  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Frags<D> fr;
  bf16v8 qf[D / 16];
  {
    const __hip_bfloat16* qp = a.q + t * a.q_t + head * a.q_h;
    #pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      qf[ks] = *reinterpret_cast<const bf16v8*>(qp + ks * 16 + half * 8);
  }
  float m = -1e30f, lsum = 0.f;
  f32x16 acc[D / 32];
  #pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = zero16();

  if (begin < end) {
    const int* table = a.tables + (int64_t)b * a.width;
    Paged<D, NW * 64> tile;
    tile.look(a, table, begin, end);
    tile.fetch(a, kv, begin, end);
    tile.look(a, table, begin + KEYS, end);
    tile.store(smem, smem + TB);
    __syncthreads();
    int turn = 0;
    for (int k0 = begin; k0 < end; k0 += KEYS, turn ^= 1) {
      char *kt = smem + turn * (2 * TB), *vt = kt + TB;
      const bool more = k0 + KEYS < end;
      if (more) {
        tile.fetch(a, kv, k0 + KEYS, end);
        tile.look(a, table, k0 + 2 * KEYS, end);
      }
      if (k0 < most && r0 < rows) {                     // wave-uniform
        f32x16 st[NS];
        #pragma unroll
        for (int n = 0; n < NS; ++n) {
          st[n] = zero16();
          #pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) st[n] = mfma(fr.row(kt, n, ks), qf[ks], st[n]);
        }
        if (k0 + KEYS > least) {                        // the diagonal, or the end
          #pragma unroll
          for (int n = 0; n < NS; ++n)
            #pragma unroll
            for (int i = 0; i < 16; ++i)
              if (k0 + n * 32 + acc_row(i, half) >= mine) st[n][i] = -1e30f;
        }
        float mx = st[0][0];
        #pragma unroll
        for (int n = 0; n < NS; ++n)
          #pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[n][i]);
        const float m_new = fmaxf(m, halves_max(mx) * a.scale_log2);
        if (__any(m_new > m)) {
          const float alpha = __builtin_amdgcn_exp2f(m - m_new);
          lsum *= alpha;
          #pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
            #pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
          m = m_new;
        }
        #pragma unroll
        for (int n = 0; n < NS; ++n)
          #pragma unroll
          for (int i = 0; i < 16; ++i) {
            st[n][i] = __builtin_amdgcn_exp2f(st[n][i] * a.scale_log2 - m);
            lsum += st[n][i];
          }
        #pragma unroll
        for (int n = 0; n < NS; ++n)
          #pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const bf16v8 p = pack8(st[n], k2);
            #pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
              acc[dt] = mfma(fr.col(vt, n * 32 + k2 * 16, dt), p, acc[dt]);
          }
      }
      if (more) {
        char* next = smem + (turn ^ 1) * (2 * TB);
        tile.store(next, next + TB);
        __syncthreads();
      }
    }
  }

  const bool live = r < rows, seen = mine > begin;      // else no key of this slice
  lsum = halves_sum(lsum);
  if (__any(!seen)) {           // what its masked scores became is no number
    lsum = seen ? lsum : 0.f;
    #pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
      #pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] = seen ? acc[dt][i] : 0.f;
  }
  const int64_t at = (int64_t)t * a.H + head;
  if (slices == 1) {
    store_rows<D>(acc, seen ? 1.f / lsum : 0.f, a.out + at * D, live);
    return;
  }
  const int64_t part = z * (int64_t)a.T * a.H + at;
  if (begin < end) store_rows_f32<D>(acc, a.o_part + part * D, live);
  if (half == 0 && live) {
    a.ml_part[part * 2] = seen ? m : -1e30f;
    a.ml_part[part * 2 + 1] = lsum;
  }
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
  for (int z = 0; z < slices; ++z) {
    const float2 ml = reinterpret_cast<const float2*>(a.ml_part)[z * n + row];
    if (ml.y == 0.f) continue;
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
  for (int j = 0; j < 8; ++j) out.v[j] = f2bf(l > 0.f ? o[j] / l : 0.f);
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
  TORCH_CHECK(scale > 0. && scale < 1e30, "paged_attention_chunk: a positive scale");
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
  a.shift = (block & (block - 1)) == 0 ? __builtin_ctzll(block) : -1;
  a.scale_log2 = (float)scale * LOG2E;
  constexpr int NW = 4, ROWS = NW * WROWS;
  // one block more than the sequences can have, which clears the rows of none
  const int64_t blocks = T * (H / KV) / ROWS + B + 1, grid = blocks * KV;
  TORCH_CHECK(grid < (1ll << 31), "paged_attention_chunk: too many rows");
  const int64_t most = width * block;
  const int slices = (int)std::max<int64_t>(1, std::min<int64_t>({512 / grid, (most + LEAST - 1) / LEAST, 64}));
  torch::Tensor part, ml;
  if (slices > 1) {
    part = torch::empty({slices, T, H, D}, q.options().dtype(at::kFloat));
    ml = torch::empty({slices, T, H, 2}, part.options());
    a.o_part = part.data_ptr<float>();
    a.ml_part = ml.data_ptr<float>();
  }
  auto stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto d_) {
    constexpr int DIM = decltype(d_)::value;
    hipLaunchKernelGGL((chunk_attn_kernel<DIM, NW>), dim3(grid, slices), dim3(NW * 64),
                       4 * KEYS * DIM * 2, stream, a);
    HIP_CHECK_LAST();
    if (slices > 1) {
      hipLaunchKernelGGL(chunk_join_kernel<DIM>, dim3(CDIV(T * H * (DIM / 8), 256)), dim3(256), 0,
                         stream, a, slices);
      HIP_CHECK_LAST();
    }
  };
  if (D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  return out;
}
