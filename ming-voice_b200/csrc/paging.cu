// Pages of the next step on the device (mv_plan_step, mv_release_pages).
//
// Integers only. Two prefix sums over the batch (tokens, pages taken) give every packed token its slot and every new page
// its place on the free stack; all else is a copy. Bound: latency (a step of a few hundred sequences moves some kilobytes).
// One CTA checks the step, sums and writes the counters; what grows with the tokens and the page table's width is written by a
// second kernel over the whole card, which takes page ids from the state as it was before the step, so that nothing in it
// depends on the order of its threads. Measured on a B200: one token of each of 61 sequences 9.6 us as called (4.8 in a graph, one
// launch), 16001 tokens of 9 prompts 12.8 (7.8), 2000 tokens of 1000 sequences with their rows of 516 pages gathered 12.9 (12.3); the
// host side of a call is 8 to 9 us.
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_common.cuh"
#include "common.cuh"

namespace mv {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxSeqs = 1 << 18;

struct PlanArgs {
  const int *new_tokens, *seqs, *lens, *n_free;
  int *free_pages, *pages, *lens_out, *n_free_out, *cu, *kv_lens, *table;
  long long* slots;
  int *positions, *ok, *scratch;  // scratch: the batch's first pages on the stack [B + 1], then the stack's height before the step
  long long pages_st, table_st;
  int B, max_seqs, max_pages, page_shift, max_len, num_pages, T;
  bool prompts;  // tokens only for sequences that have none
};

__device__ __forceinline__ int pages_of(int tokens, int shift) {
  return static_cast<int>((static_cast<unsigned int>(tokens) + (1u << shift) - 1) >> shift);
}

// Inclusive sums of (a, b) over the CTA's threads; `total` receives the sums over all. Two barriers.
__device__ __forceinline__ void scan2(int& a, int& b, int2& total, int2* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pa = __shfl_up_sync(0xffffffffu, a, o), pb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += pa, b += pb;
  }
  if (lane == 31) part[warp] = make_int2(a, b);
  __syncthreads();
  int2 s = part[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pa = __shfl_up_sync(0xffffffffu, s.x, o), pb = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += pa, s.y += pb;
  }
  total = make_int2(__shfl_sync(0xffffffffu, s.x, 31), __shfl_sync(0xffffffffu, s.y, 31));
  const int bx = __shfl_sync(0xffffffffu, s.x, (warp + 31) & 31), by = __shfl_sync(0xffffffffu, s.y, (warp + 31) & 31);
  if (warp > 0) a += bx, b += by;
  __syncthreads();
}

__device__ __forceinline__ long long block_sum(long long v, long long* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  long long s = part[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  return s;
}

// The page of column `col` of batch entry b after the step. `have`: the columns that it owned before.
__device__ __forceinline__ int page_at(const PlanArgs& a, int s, int col, int have, int first, int height) {
  return col < have ? a.pages[s * a.pages_st + col] : a.free_pages[height - 1 - (first + col - have)];
}

// The last b with start[b] <= i among b < n (start ascends, start[0] = 0 <= i).
__device__ __forceinline__ int owner_of(const int* start, int n, int i) {
  int lo = 0, hi = n;  // start[lo] <= i, start[hi] > i or hi = n
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// What a step writes besides the counters: slot and position of token t; new entry i of the page table; cell of a gathered table.
__device__ __forceinline__ void write_token(const PlanArgs& a, int t, int height) {
  long long slot = -1;
  int pos = 0;
  if (t < a.cu[a.B]) {
    const int b = owner_of(a.cu, a.B, t);
    const int s = a.seqs != nullptr ? a.seqs[b] : b;
    const int end = a.kv_lens[b], old = end - (a.cu[b + 1] - a.cu[b]);
    pos = old + t - a.cu[b];
    const int page = page_at(a, s, pos >> a.page_shift, pages_of(old, a.page_shift), a.scratch[b], height);
    slot = (static_cast<long long>(page) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__device__ __forceinline__ void write_page(const PlanArgs& a, int i, int height) {
  const int b = owner_of(a.scratch, a.B, i);
  const int s = a.seqs != nullptr ? a.seqs[b] : b;
  const int old = a.kv_lens[b] - (a.cu[b + 1] - a.cu[b]);
  a.pages[s * a.pages_st + pages_of(old, a.page_shift) + i - a.scratch[b]] = a.free_pages[height - 1 - i];
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const PlanArgs a, bool all_here) {
  extern __shared__ unsigned int seen[];  // a bit per sequence: the step has it
  __shared__ int2 part2[32];
  __shared__ long long part[32];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (a.seqs != nullptr) {
    for (int i = tid; i < (a.max_seqs + 31) / 32; i += kThreads) seen[i] = 0u;
    __syncthreads();
  }
  const int height = *a.n_free;
  const int limit = static_cast<int>(min(static_cast<long long>(a.max_len), static_cast<long long>(a.max_pages) << a.page_shift));
  long long tokens = 0, taken = 0;
  bool bad = height < 0 || height > a.num_pages;
  for (int b = tid; b < a.B; b += kThreads) {
    const int s = a.seqs != nullptr ? a.seqs[b] : b, n = a.new_tokens[b];
    if (s < 0 || s >= a.max_seqs || n < 0) {
      bad = true;
      continue;
    }
    if (a.seqs != nullptr && (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u)) bad = true;
    const int old = a.lens[s];
    if (old < 0 || n > limit - min(old, limit) || (a.prompts && n > 0 && old > 0)) {
      bad = true;
      continue;
    }
    tokens += n;
    taken += pages_of(old + n, a.page_shift) - pages_of(old, a.page_shift);
  }
  const bool any_bad = __syncthreads_or(bad);
  tokens = block_sum(tokens, part);
  taken = block_sum(taken, part);
  const bool ok = !any_bad && tokens <= a.T && taken <= height;

  // the state of sequences that the step does not have
  if (a.lens_out != a.lens)
    for (int s = tid; s < a.max_seqs; s += kThreads)
      if (!ok || (a.seqs != nullptr ? !(seen[s >> 5] >> (s & 31) & 1u) : s >= a.B)) a.lens_out[s] = a.lens[s];
  int2 base = make_int2(0, 0);
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    int s = -1, n = 0, old = 0, more = 0;
    if (b < a.B) {
      s = a.seqs != nullptr ? a.seqs[b] : b;
      if (s >= 0 && s < a.max_seqs) old = a.lens[s];
      if (ok) {
        n = a.new_tokens[b];
        more = pages_of(old + n, a.page_shift) - pages_of(old, a.page_shift);
      }
    }
    int ends = n, last = more;
    int2 total;
    scan2(ends, last, total, part2);
    if (b < a.B) {
      a.cu[b + 1] = base.x + ends;
      a.scratch[b] = base.y + last - more;
      a.kv_lens[b] = old + n;
      if (ok) a.lens_out[s] = old + n;
    }
    base.x += total.x, base.y += total.y;
  }
  if (tid == 0) {
    a.cu[0] = 0;
    a.scratch[a.B] = base.y;
    a.scratch[a.B + 1] = height;
    *a.n_free_out = ok ? height - base.y : height;
    *a.ok = ok;
  }
  if (!all_here) return;
  __syncthreads();
  for (int i = tid; i < base.y; i += kThreads) write_page(a, i, height);
  for (int t = tid; t < a.T; t += kThreads) write_token(a, t, height);
}

// The rest of a large step. The first `token_blocks` CTAs write tokens and new pages, the others rows of a gathered table.
__global__ void __launch_bounds__(256) spread_kernel(const PlanArgs a, int token_blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const int height = a.scratch[a.B + 1];
  if (static_cast<int>(blockIdx.x) < token_blocks) {
    const int n = token_blocks * 256, i0 = blockIdx.x * 256 + threadIdx.x;
    const int taken = a.scratch[a.B];
    for (int i = i0; i < taken; i += n) write_page(a, i, height);
    for (long long t = i0; t < a.T; t += n) write_token(a, static_cast<int>(t), height);
    return;
  }
  for (int b = blockIdx.x - token_blocks; b < a.B; b += gridDim.x - token_blocks) {
    const int s = a.seqs[b];
    const bool known = s >= 0 && s < a.max_seqs;
    const int end = a.kv_lens[b], old = end - (a.cu[b + 1] - a.cu[b]);
    const int have = pages_of(max(old, 0), a.page_shift), need = known ? pages_of(max(end, 0), a.page_shift) : 0;
    const int first = a.scratch[b];
    int* row = a.table + b * a.table_st;
    for (int col = threadIdx.x; col < a.max_pages; col += 256)
      row[col] = col < need ? page_at(a, s, col, have, first, height) : 0;
  }
}

__global__ void __launch_bounds__(kThreads) release_kernel(const PlanArgs a) {
  extern __shared__ unsigned int seen[];
  __shared__ int2 part2[32];
  __shared__ long long part[32];
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  for (int i = tid; i < (a.max_seqs + 31) / 32; i += kThreads) seen[i] = 0u;
  __syncthreads();
  const int height = *a.n_free;
  bool bad = height < 0 || height > a.num_pages;
  long long given = 0;
  for (int b = tid; b < a.B; b += kThreads) {
    const int s = a.seqs[b];
    if (s < 0 || s >= a.max_seqs || (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u)) {
      bad = true;
      continue;
    }
    const int n = pages_of(max(a.lens[s], 0), a.page_shift);
    if (a.lens[s] < 0 || n > a.max_pages) bad = true;
    given += n;
  }
  const bool any_bad = __syncthreads_or(bad);
  given = block_sum(given, part);
  const bool ok = !any_bad && given <= a.num_pages - height;
  if (ok) {
    int base = height;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + tid;
      const int s = b < a.B ? a.seqs[b] : 0;
      const int n = b < a.B ? pages_of(a.lens[s], a.page_shift) : 0;
      int ends = n, unused = 0;
      int2 total;
      scan2(ends, unused, total, part2);
      // a warp gives back the pages of its 32 sequences one after another, its lanes side by side
      for (int j = 0; j < 32; ++j) {
        const int sj = __shfl_sync(0xffffffffu, s, j), nj = __shfl_sync(0xffffffffu, n, j);
        const int at = base + __shfl_sync(0xffffffffu, ends, j) - nj;
        for (int i = lane; i < nj; i += 32) a.free_pages[at + i] = a.pages[sj * a.pages_st + i];
      }
      base += total.x;
    }
  }
  __syncthreads();  // all lengths are read
  for (int s = tid; s < a.max_seqs; s += kThreads) {
    const bool given_back = ok && (seen[s >> 5] >> (s & 31) & 1u);
    if (given_back)
      a.lens_out[s] = 0;
    else if (a.lens_out != a.lens)
      a.lens_out[s] = a.lens[s];
  }
  if (tid == 0) {
    *a.n_free_out = ok ? height + static_cast<int>(given) : height;
    *a.ok = ok;
  }
}

int check_state(const mv_plan_args* x, const char* who) {
  if (x->B < 0 || x->max_seqs < 0 || x->B > x->max_seqs || x->max_seqs > kMaxSeqs || x->max_pages < 0 ||
      x->num_pages < 0)
    return fail(MV_ERR_INVALID, "%s: bad B=%d / max_seqs=%d (at most %d) / max_pages=%d / num_pages=%d", who, x->B,
                x->max_seqs, kMaxSeqs, x->max_pages, x->num_pages);
  if (x->page_size < 8 || x->page_size > 256 || (x->page_size & (x->page_size - 1)) != 0)
    return fail(MV_ERR_UNSUPPORTED, "%s: page_size=%d must be a power of two in 8..256", who, x->page_size);
  if (x->n_free == nullptr || x->n_free_out == nullptr || x->ok == nullptr ||
      (x->max_seqs > 0 && (x->lens == nullptr || x->lens_out == nullptr)) ||
      (x->max_pages > 0 && x->max_seqs > 0 && x->pages == nullptr) || (x->num_pages > 0 && x->free_pages == nullptr))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (x->max_seqs > 1 && x->pages_st < x->max_pages)
    return fail(MV_ERR_INVALID, "%s: page table row stride %lld shorter than max_pages=%d", who, x->pages_st, x->max_pages);
  return MV_OK;
}

PlanArgs state_of(const mv_plan_args* x) {
  PlanArgs a{};
  a.new_tokens = x->new_tokens, a.seqs = x->seqs, a.lens = x->lens, a.n_free = x->n_free;
  a.free_pages = x->free_pages, a.pages = x->pages, a.lens_out = x->lens_out, a.n_free_out = x->n_free_out;
  a.cu = x->cu_seqlens, a.kv_lens = x->kv_lens, a.table = x->table, a.slots = x->slots, a.positions = x->positions;
  a.ok = x->ok, a.scratch = x->scratch, a.pages_st = x->pages_st, a.table_st = x->table_st;
  a.B = x->B, a.max_seqs = x->max_seqs, a.max_pages = x->max_pages, a.page_shift = attn::log2_of(x->page_size);
  a.max_len = x->max_len, a.num_pages = x->num_pages, a.T = x->T, a.prompts = x->prompts != 0;
  return a;
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" int mv_plan_step(const mv_plan_args* x, void* stream) {
  const char* who = "mv_plan_step";
  if (x == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const int rc = check_state(x, who);
  if (rc != MV_OK) return rc;
  if (x->T < 0 || x->max_len < 0) return fail(MV_ERR_INVALID, "%s: bad T=%d / max_len=%d", who, x->T, x->max_len);
  if (x->cu_seqlens == nullptr || x->scratch == nullptr || (x->B > 0 && (x->new_tokens == nullptr || x->kv_lens == nullptr)) ||
      (x->T > 0 && (x->slots == nullptr || x->positions == nullptr)))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (x->seqs == nullptr && x->B != 0 && x->B != x->max_seqs)
    return fail(MV_ERR_INVALID, "%s: B=%d without seqs must be max_seqs=%d", who, x->B, x->max_seqs);
  const bool gather = x->seqs != nullptr && x->B > 0 && x->max_pages > 0;
  if (gather && (x->table == nullptr || (x->B > 1 && x->table_st < x->max_pages)))
    return fail(MV_ERR_INVALID, "%s: table is null, or its rows are shorter than max_pages=%d", who, x->max_pages);
  PlanArgs a = state_of(x);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = a.seqs != nullptr ? (static_cast<size_t>(a.max_seqs) + 31) / 32 * 4 : 0;
  const bool all_here = !gather && a.T <= 2 * kThreads;
  const int rc2 = attn::launch_pdl(plan_kernel, dim3(1), kThreads, smem, st, "mv_plan_step launch", a, all_here);
  if (rc2 != MV_OK || all_here) return rc2;
  const int token_blocks = (a.T + 1023) / 1024 < 256 ? (a.T + 1023) / 1024 + 1 : 256;
  const int row_blocks = gather ? (a.B < 592 ? a.B : 592) : 0;
  return attn::launch_pdl(spread_kernel, dim3(token_blocks + row_blocks), 256, 0, st, "mv_plan_step launch", a,
                          token_blocks);
}

extern "C" int mv_release_pages(const mv_plan_args* x, void* stream) {
  const char* who = "mv_release_pages";
  if (x == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const int rc = check_state(x, who);
  if (rc != MV_OK) return rc;
  if (x->B > 0 && x->seqs == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  PlanArgs a = state_of(x);
  const size_t smem = (static_cast<size_t>(a.max_seqs) + 31) / 32 * 4;
  return attn::launch_pdl(release_kernel, dim3(1), kThreads, smem, static_cast<cudaStream_t>(stream),
                          "mv_release_pages launch", a);
}
