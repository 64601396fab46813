// Where a step's new tokens lie in the paged cache, from the requests' lengths: rows of
// the flat batch, positions, cache rows, and the block tables' next pages.
//
// Request b has ctx[b] tokens in the cache and brings new[b]; its pages are ceil(n / block)
// entries of its table, of which held[b] are there. What it is short of comes from a list
// of free pages, one request's behind the other's:
//   cu[b] = sum of new[< b],  opened[b] = sum of (ceil((ctx + new) / block) - held)[< b].
// Every workgroup forms both sums for itself in LDS (lengths of 1000 requests are 12 KB, in
// every L2 after the first), so that one launch is all; then a thread takes four neighbouring
// tokens, or a page that is opened, and looks for its request there.
// Bound: the chain of lengths, sums, search and page, 5 us, which calls of up to 100
// thousand tokens wait for in full (a call 7 us with its launch and outputs); 2 million
// tokens 15 us, 1.7 TB/s of what is written. A token a thread took 19.3.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.h"

namespace {

constexpr int THREADS = 256, RUN = 4;
constexpr int MOST = 8192;      // requests: two sums of 32 KB in LDS

struct Slots {
  int* tables;                  // (B, width)
  const int *ctx, *fresh, *held, *pages;        // held: or null, what ctx fills
  int *positions, *cu, *context;
  int64_t *slots, *last;
  int B, width, block, free, rows;
};

// Sums stop at MANY: lengths may be any numbers, and there are fewer rows and free pages.
constexpr uint32_t MANY = 0x7fffffff;
struct Need {
  int tokens, pages;
  DEV_INLINE static int sum(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, MANY); }
  DEV_INLINE void operator+=(const Need& n) {
    tokens = sum(tokens, n.tokens);
    pages = sum(pages, n.pages);
  }
};

DEV_INLINE int pages_of(uint32_t n, int block) {
  return n == 0 ? 0 : (int)min((n - 1) / (uint32_t)block + 1, MANY);
}
DEV_INLINE int held_of(const Slots& a, int b) {
  return max(0, a.held ? a.held[b] : pages_of(max(0, a.ctx[b]), a.block));
}
DEV_INLINE Need need_of(const Slots& a, int b) {
  const int n = max(0, a.fresh[b]);
  const int64_t with = (int64_t)a.ctx[b] + n;           // below 2^32
  return {n, max(0, pages_of((uint32_t)max(with, (int64_t)0), a.block) - held_of(a, b))};
}

// the largest b < n with sum[b] <= i; sums never fall, sum[0] = 0
DEV_INLINE int find(const int* sum, int n, int i) {
  int lo = 0;
  while (n > 1) {
    const int h = n / 2;
    if (sum[lo + h] <= i) {
      lo += h;
      n -= h;
    } else {
      n = h;
    }
  }
  return lo;
}

// Where token i of request b lies: its page's number of the last look-up is kept, as
// neighbours share it.
struct Place {
  int b = -1, page_index = -1, page = -1, ctx = 0, held = 0;

  DEV_INLINE int64_t slot(const Slots& a, const int* cu, const int* opened, int request, int i,
                          int& position) {
    if (request != b) {
      b = request;
      page_index = -1;
      ctx = a.ctx[b];
      held = held_of(a, b);
    }
    position = (int)((uint32_t)ctx + (uint32_t)(i - cu[b]));
    if (position < 0) return -1;
    const int p = position / a.block;
    if (p != page_index) {
      page_index = p;
      const uint32_t from = (uint32_t)opened[b] + (uint32_t)(p - held);
      page = p >= a.width ? -1
             : p < held   ? a.tables[(int64_t)b * a.width + p]
             : from < (uint32_t)a.free ? a.pages[from] : -1;
    }
    return page >= 0 ? (int64_t)page * a.block + (position - p * a.block) : -1;
  }
};

__global__ __launch_bounds__(THREADS)
void chunk_slots_kernel(Slots a) {
  extern __shared__ int lds[];
  int *cu = lds, *opened = lds + a.B + 1;
  __shared__ Need wave_sum_of[THREADS / WAVE];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
  #pragma unroll 4
  for (int b = tid; b < a.B; b += THREADS) {
    const Need n = need_of(a, b);
    cu[b] = n.tokens;
    opened[b] = n.pages;
  }
  __syncthreads();
  // a run of requests a thread, then the runs' sums over the workgroup
  const int run = CDIV(a.B, THREADS), b0 = min(tid * run, a.B), b1 = min(b0 + run, a.B);
  Need sum{0, 0};
  for (int b = b0; b < b1; ++b) sum += Need{cu[b], opened[b]};
  Need to = sum;                // inclusive over the wave
  #pragma unroll
  for (int off = 1; off < WAVE; off <<= 1) {
    const Need before{__shfl_up(to.tokens, off, WAVE), __shfl_up(to.pages, off, WAVE)};
    if (lane >= off) to += before;
  }
  if (lane == WAVE - 1) wave_sum_of[wave] = to;
  __syncthreads();
  Need at{__shfl_up(to.tokens, 1, WAVE), __shfl_up(to.pages, 1, WAVE)};
  if (lane == 0) at = Need{0, 0};
  for (int w = 0; w < wave; ++w) at += wave_sum_of[w];
  for (int b = b0; b < b1; ++b) {
    const Need n{cu[b], opened[b]};
    cu[b] = at.tokens;
    opened[b] = at.pages;
    at += n;
  }
  if (tid == THREADS - 1) {
    cu[a.B] = at.tokens;
    opened[a.B] = at.pages;
  }
  __syncthreads();

  // RUN neighbouring tokens a thread: one search, one page for most of them, whole stores
  const int total = cu[a.B], stride = gridDim.x * THREADS, me = blockIdx.x * THREADS + tid;
  for (int64_t i0 = (int64_t)me * RUN; i0 < a.rows; i0 += (int64_t)stride * RUN) {
    int b = find(cu, a.B, (int)i0);
    Place place;
    int position[RUN];
    int64_t slot[RUN];
    #pragma unroll
    for (int j = 0; j < RUN; ++j) {
      const int i = (int)i0 + j;
      position[j] = 0;
      slot[j] = -1;
      if (i < total) {
        while (b + 1 < a.B && cu[b + 1] <= i) ++b;
        slot[j] = place.slot(a, cu, opened, b, i, position[j]);
      }
    }
    if (i0 + RUN <= a.rows) {
      *reinterpret_cast<int4*>(a.positions + i0) = int4{position[0], position[1], position[2], position[3]};
      #pragma unroll
      for (int j = 0; j < RUN; j += 2)
        *reinterpret_cast<longlong2*>(a.slots + i0 + j) = longlong2{slot[j], slot[j + 1]};
    } else {
      for (int j = 0; j < (int)(a.rows - i0); ++j) {
        a.positions[i0 + j] = position[j];
        a.slots[i0 + j] = slot[j];
      }
    }
  }
  const int64_t entries = (int64_t)a.B * a.width;
  if (opened[a.B] <= entries) {
    for (int64_t i = me; i < opened[a.B]; i += stride) {
      const int b = find(opened, a.B, (int)i);
      const int64_t p = held_of(a, b) + i - opened[b];
      if (p < a.width) a.tables[(int64_t)b * a.width + p] = i < a.free ? a.pages[i] : -1;
    }
  } else {                      // more than the tables can take: by their entries
    for (int64_t e = me; e < entries; e += stride) {
      const int b = (int)(e / a.width), of = (int)(e - (int64_t)b * a.width) - held_of(a, b);
      if ((uint32_t)of >= (uint32_t)need_of(a, b).pages) continue;
      const uint32_t from = (uint32_t)opened[b] + (uint32_t)of;
      a.tables[e] = from < (uint32_t)a.free ? a.pages[from] : -1;
    }
  }
  for (int b = me; b <= a.B; b += stride) {
    a.cu[b] = min(cu[b], a.rows);
    if (b == a.B) break;
    a.context[b] = (int)((uint32_t)a.ctx[b] + (uint32_t)max(0, a.fresh[b]));
    a.last[b] = min(max(cu[b + 1], 1), max(a.rows, 1)) - 1;
  }
}

}  // namespace

// {positions (rows) int32, slots (rows) int64, cu (B + 1) int32, context lengths after the
// step (B) int32, each request's last row (B) int64}; block_tables <- the opened pages.
std::vector<torch::Tensor> chunk_slots(torch::Tensor block_tables, torch::Tensor ctx_lens,
                                       torch::Tensor new_lens, torch::Tensor pages,
                                       int64_t block_size, int64_t rows,
                                       c10::optional<torch::Tensor> held) {
  TORCH_CHECK(block_tables.is_cuda() && block_tables.dim() == 2,
              "chunk_slots: block_tables (requests, pages) on the GPU");
  const int64_t B = block_tables.size(0), width = block_tables.size(1);
  auto check = [&](const torch::Tensor& t, int64_t n, const char* what) {
    TORCH_CHECK(t.device() == block_tables.device() && t.scalar_type() == at::kInt &&
                t.is_contiguous() && t.numel() == n, "chunk_slots: ", what, ": device, type, size or layout");
  };
  check(block_tables, B * width, "block_tables");
  check(ctx_lens, B, "context_lens");
  check(new_lens, B, "new_lens");
  check(pages, pages.numel(), "pages");
  if (held) check(*held, B, "held");
  TORCH_CHECK(block_size > 0 && block_size < (1ll << 31), "chunk_slots: block_size");
  TORCH_CHECK(rows >= 0 && rows < (1ll << 31) - (1 << 24) && pages.numel() < (1ll << 31),
              "chunk_slots: rows");
  TORCH_CHECK(B <= MOST, "chunk_slots: up to ", MOST, " requests");
  const c10::cuda::CUDAGuard guard(block_tables.device());
  auto ints = block_tables.options();
  auto longs = ints.dtype(at::kLong);
  auto positions = torch::empty({rows}, ints), cu = torch::empty({B + 1}, ints);
  auto context = torch::empty({B}, ints);
  auto slots = torch::empty({rows}, longs), last = torch::empty({B}, longs);
  Slots a{};
  a.tables = block_tables.data_ptr<int>();
  a.ctx = ctx_lens.data_ptr<int>();
  a.fresh = new_lens.data_ptr<int>();
  a.held = held ? held->data_ptr<int>() : nullptr;
  a.pages = pages.data_ptr<int>();
  a.positions = positions.data_ptr<int>();
  a.cu = cu.data_ptr<int>();
  a.context = context.data_ptr<int>();
  a.slots = slots.data_ptr<int64_t>();
  a.last = last.data_ptr<int64_t>();
  a.B = B;
  a.width = width;
  a.block = block_size;
  a.free = pages.numel();
  a.rows = rows;
  const int64_t work = std::max(std::max<int64_t>(CDIV(rows, RUN), B + 1),
                                std::min<int64_t>(pages.numel(), B * width));
  // up to four workgroups a CU, each of which forms the sums for itself: 2 million tokens
  // of 1000 requests 19.3 us with 512 of them, 15.0 so and with 2048
  hipLaunchKernelGGL(chunk_slots_kernel, dim3(std::min<int64_t>(CDIV(work, THREADS), 1024)),
                     dim3(THREADS), 2 * (B + 1) * sizeof(int), at::cuda::getCurrentCUDAStream(), a);
  HIP_CHECK_LAST();
  return {positions, slots, cu, context, last};
}
