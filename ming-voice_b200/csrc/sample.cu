// Drawing tokens from logits with temperature, top-k, top-p and min-p (mv_sample).
//
// Mathematics. Tokens are ordered by (logit descending, index ascending), as one 64-bit number `place`: the logit's bits, mapped
// so that unsigned comparison orders them, in the upper half and the index in the lower. Each filter keeps a prefix of that order,
// so all that is kept is given by one place, the border, and a least weight. Weights 2^t, t = (logit - max) log2(e) / temperature,
// are whole numbers of 2^-shift (shift 44 for vocabularies of 2^17, more for smaller ones up to 51; 2^f from a table of 32 values and a polynomial of degree 5
// that interpolates 2^g at the Chebyshev nodes of [-1/64, 1/64], off by 2^-52 of it), so that sums do not depend on their order: each border and each draw comes out
// the same whatever the split. A weight is off by half a unit at most (below that it is 0), so a sum of V by V 2^-(shift + 1) of the
// largest weight: 2^-28 for 2^17 tokens; from 2^19 on (2^-24) a random number of 24 bits may resolve it.
//
// Steps, a cluster of CTAs for each row, the row in their shared memory:
//   1. read the row once; the first of the order, and (top-k) a key with at least top_k logits at or above it: the least over
//      the CTAs of the one that top_k / C of its threads' largest logits reach
//   2. few candidates (a small top_k, or min_p without top_p): they are brought together in the first CTA, which finds the
//      borders and draws by itself
//   3. else the borders: a histogram of t with 2048 bins (counts for top-k; for top-p weights, as three sums of 15 bits, since
//      64-bit additions in shared memory cost seven times three of 32 bits), added up in the first CTA, which finds the bin with the border; that bin's tokens
//      are brought together there. A bin with more than the list holds (runs of equal logits) is searched over all CTAs.
//   4. each CTA adds up what is kept of its part; the CTA in which the sum passes u times the total finds the token.
// A border among listed tokens is found over their places, by finer and finer bins and by comparing the last few with one another.
//
// Bound: many rows by the weights (a 64-bit exponential is some 60 cycles of a quarter SM for 32 logits; every logit has one where top-p
// or nothing is asked for) and by the steps of a row that wait for one another; one row by those steps alone (a cluster barrier and the
// reads behind it are 1 us, and there are 4 to 12). Measured on a B200, call after call: one row of 131072 f32 with all filters 10.9 us,
// 192 rows of 131072 bf16 with min_p 40 (a copy of them 7.8), 48 rows of 100277 f32 with top-p over a flat distribution 50, 128 rows of
// 50257 bf16 with settings of their own 46.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_common.cuh"
#include "common.cuh"

namespace mv {
namespace {

namespace cg = cooperative_groups;

struct SampleArgs {
  const void* logits;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  long long* tokens;
  float* logprob;
  long long st;
  float temperature_value, top_p_value, min_p_value;
  int top_k_value, V, shift;
  int slice;     // elements of a CTA's part of the row, a multiple of 8
  bool in_smem;  // the part fits in shared memory
  bool vectors;  // rows start at 16-byte addresses
};

// A CTA's threads and what goes by them: 512 for few rows, else 256, four of which share an SM (launch_rows).
template <int kThreads>
struct Cta {
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kBins = 4 * kThreads, kList = 8 * kThreads;
  static constexpr int kFine = kThreads == 256 ? 8 : 9;   // log2 of the finer bins, one for each thread
  static constexpr int kMostMaxima = kThreads * 3 / 4;    // of the threads, in finding the key of step 1
  static_assert(1 << kFine == kThreads, "a finer bin for each thread");
};
constexpr unsigned int kFew = 128;  // tokens that are put in order by comparing all with all (n * n / 128 steps of some 12 instructions)
constexpr uint32_t kNone = 0x007fffffu;  // the key of -inf

__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 -> +0
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) {
  return static_cast<uint64_t>(~key) << 32 | static_cast<uint32_t>(i);
}

// Weights of one row as whole numbers. Logits are compared as fp32 numbers (an integer operation costs twice as much).
struct Weights {
  double m, c;          // largest logit, log2(e) / temperature
  float top, least;     // the largest logit, and the least that can have a weight
  const double* table;  // 2^(j / 32 + shift)
  // 2^t in units of 2^-shift, rounded, for a logit from `least` on; of others what comes out
  __device__ __forceinline__ uint64_t of(float l) const {
    constexpr double kRound = 211106232532992.0;  // 1.5 * 2^47: the low word of a sum with it counts 32nds, rounded
    // (the largest logit may be infinite; roundings are spelled out, so that each use of this gives the same weight)
    const double t = l == top ? 0.0 : __dmul_rn(__dsub_rn(static_cast<double>(l), m), c);
    const double r = __dadd_rn(t, kRound);
    const double g = __dsub_rn(t, __dsub_rn(r, kRound));
    const int n = __double2loint(r);
    double p = 0.0013333604694153824;
    p = fma(p, g, 0.009618176115571158);
    p = fma(p, g, 0.05550410866453748);
    p = fma(p, g, 0.24022650695623157);
    p = fma(p, g, 0.6931471805599453);
    p = fma(p, g, 1.0);
    const double b = table[n & 31];
    const double s = __hiloint2double(__double2hiint(b) + (n & ~31) * 32768, __double2loint(b));  // 20 - 5 bits up
    return static_cast<uint64_t>(__double_as_longlong(fma(p, s, 4503599627370496.0))) & 0xfffffffffffffull;  // 2^52
  }
  // The least logit whose weight is 2^t or more. Rounded up, so that it is no lighter either, however far apart the numbers of its
  // size lie: lighter ones have no bin, and their powers of two leave the exponent's range.
  __device__ __forceinline__ float logit_at(double t) const {
    if (isinf(top)) return top;  // beside an infinite logit only its equals have a weight
    const double l = m + t / c * 1.0000001;
    return l > -3.4e38 ? __double2float_ru(l) : -3.4028235e38f;
  }
};

// three additions of 27, 27 and 10 bits, which a warp does in one instruction each
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
  const unsigned int a = __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(v) & 0x7ffffffu);
  const unsigned int b = __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(v >> 27) & 0x7ffffffu);
  const unsigned int c = __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(v >> 54));
  return a + (static_cast<uint64_t>(b) << 27) + (static_cast<uint64_t>(c) << 54);
}

template <int kThreads>
struct Shared : Cta<kThreads> {
  using C = Cta<kThreads>;
  union {
    unsigned int bins[4][C::kBins];  // counts, or the weights' bits 0-14, 15-29 and 30-51
    unsigned long long list[C::kList];
  };
  unsigned long long part[C::kWarps], total, border, kept, least_place, most_place, best, bin_before;
  double table[32];
  unsigned int fine[4][kThreads], counts[C::kWarps], n_list, n_left, pivot, nan, bin, bin_count_before, part_n, bin_from, bin_to;
  int bin_here;  // the bin, where this CTA has found it
};

// Sums of (w, n) over the CTA in every thread. Two barriers.
template <int kThreads>
__device__ __forceinline__ void block_sum(uint64_t& w, unsigned int& n, Shared<kThreads>& s) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  w = warp_sum(w);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) s.part[warp] = w, s.counts[warp] = n;
  __syncthreads();
  w = lane < kWarps ? s.part[lane] : 0ull;
  n = lane < kWarps ? s.counts[lane] : 0u;
  w = warp_sum(w);
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
}

// Sums of (w, n) over the threads before this one, in thread order, and over all. Two barriers.
template <int kThreads>
__device__ __forceinline__ void block_before(uint64_t& w, unsigned int& n, uint64_t& total_w, unsigned int& total_n,
                                             Shared<kThreads>& s) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t w0 = w;
  const unsigned int n0 = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t pw = __shfl_up_sync(0xffffffffu, w, o);
    const unsigned int pn = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) w += pw, n += pn;
  }
  if (lane == 31) s.part[warp] = w, s.counts[warp] = n;
  __syncthreads();
  uint64_t sw = lane < kWarps ? s.part[lane] : 0ull;
  unsigned int sn = lane < kWarps ? s.counts[lane] : 0u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t pw = __shfl_up_sync(0xffffffffu, sw, o);
    const unsigned int pn = __shfl_up_sync(0xffffffffu, sn, o);
    if (lane >= o) sw += pw, sn += pn;
  }
  total_w = __shfl_sync(0xffffffffu, sw, 31);
  total_n = __shfl_sync(0xffffffffu, sn, 31);
  const uint64_t bw = __shfl_sync(0xffffffffu, sw, (warp + 31) & 31);
  const unsigned int bn = __shfl_sync(0xffffffffu, sn, (warp + 31) & 31);
  w = w - w0 + (warp > 0 ? bw : 0ull);
  n = n - n0 + (warp > 0 ? bn : 0u);
  __syncthreads();
}

// Tokens of a list in the registers of one CTA's threads.
template <int kThreads>
struct Listed {
  using Shared = Shared<kThreads>;
  static constexpr int kEach = Cta<kThreads>::kList / kThreads, kFine = Cta<kThreads>::kFine;
  uint64_t place[kEach], w[kEach];  // ~0 and 0 where there is no token
  int rows;                         // of them that are in use

  // from the list; weights where they are asked for
  __device__ __forceinline__ void load(unsigned int count, const Weights& wt, bool weights, const Shared& s) {
    rows = (count + kThreads - 1) / kThreads;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      place[i] = ~0ull, w[i] = 0;
      const unsigned int at = threadIdx.x + i * kThreads;
      if (i >= rows || at >= count) continue;
      place[i] = s.list[at];
      const uint32_t key = ~static_cast<uint32_t>(place[i] >> 32);
      if (weights) w[i] = wt.of(of_key(key));
    }
  }
  // sums over all tokens up to place `last`
  __device__ __forceinline__ void up_to(uint64_t last, uint64_t& sum, unsigned int& n, Shared& s) const {
    sum = 0, n = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < rows && place[i] <= last && place[i] != ~0ull) ++n, sum += w[i];
    block_sum(sum, n, s);
  }

  // The first place up to which there are at least need_n tokens (by_count) or weights of at least need_w, among the `count`
  // tokens, which lie in from .. to; it exists. Overwrites the list.
  __device__ __forceinline__ uint64_t border(bool by_count, unsigned int need_n, uint64_t need_w, unsigned int count, uint64_t from,
                                             uint64_t to, Shared& s) const {
    const int tid = threadIdx.x;
    // (n_left, not n_list: other CTAs may still be reading how long the list was)
    uint64_t w_before = 0;  // of what lies before what is still looked at
    unsigned int n_before = 0;
    __syncthreads();
    // a bin for each thread over the range of the places that are left, until few of them are
    while (count > kFew) {
      s.fine[0][tid] = 0u, s.fine[1][tid] = 0u, s.fine[2][tid] = 0u, s.fine[3][tid] = 0u;
      if (tid == 0) s.n_left = 0u;
      __syncthreads();
      const int shift = max(0, 64 - __clzll(to - from) - kFine);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (i >= rows || place[i] < from || place[i] > to) continue;
        const unsigned int b = static_cast<unsigned int>((place[i] - from) >> shift);
        atomicAdd(&s.fine[0][b], 1u);
        if (by_count) continue;
        atomicAdd(&s.fine[1][b], static_cast<unsigned int>(w[i]) & 0x7fffu);
        atomicAdd(&s.fine[2][b], static_cast<unsigned int>(w[i] >> 15) & 0x7fffu);
        atomicAdd(&s.fine[3][b], static_cast<unsigned int>(w[i] >> 30));
      }
      __syncthreads();
      const unsigned int n_bin = s.fine[0][tid];
      const uint64_t w_bin = s.fine[1][tid] + (static_cast<uint64_t>(s.fine[2][tid]) << 15) + (static_cast<uint64_t>(s.fine[3][tid]) << 30);
      unsigned int n = n_bin, all_n;
      uint64_t wb = w_bin, all_w;
      block_before(wb, n, all_w, all_n, s);
      n += n_before, wb += w_before;
      if (by_count ? n < need_n && n + n_bin >= need_n : wb < need_w && wb + w_bin >= need_w) {
        s.bin_before = wb, s.bin_count_before = n, s.n_left = n_bin;
        const uint64_t least = from + (static_cast<uint64_t>(tid) << shift), most = least + ((1ull << shift) - 1);
        s.least_place = least;
        // The last bin of a wide range ends behind 2^64; ~0 is no place. (Held to `to` instead, one row with top-p takes 0.4 us more.)
        s.most_place = most < least ? ~0ull - 1 : most;
      }
      __syncthreads();
      from = s.least_place, to = s.most_place, w_before = s.bin_before, n_before = s.bin_count_before, count = s.n_left;
      __syncthreads();
      if (count == 0u) break;  // (no place has what is asked for: it does not happen, and must not hold the loop)
    }
    // by comparing with all that are left
    if (tid == 0) s.n_left = 0u, s.border = to;
    __syncthreads();
    if (count == 0u) return to;
    unsigned long long *places = s.list, *weights = places + kFew;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < rows && place[i] >= from && place[i] <= to) {
        const unsigned int at = atomicAdd(&s.n_left, 1u);
        places[at] = place[i], weights[at] = w[i];
      }
    __syncthreads();
    if (tid < count) {
      const uint64_t mine = places[tid], own = weights[tid];
#pragma unroll 4
      for (unsigned int j = 0; j < count; ++j)
        if (places[j] < mine) ++n_before, w_before += weights[j];
      if (by_count ? n_before == need_n - 1 : w_before < need_w && w_before + own >= need_w) s.border = mine;
    }
    __syncthreads();
    return s.border;
  }
};

template <int DT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const SampleArgs a) {
  using Shared = Shared<kThreads>;
  constexpr int kWarps = Shared::kWarps, kBins = Shared::kBins, kList = Shared::kList, kMostMaxima = Shared::kMostMaxima;
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  using T = typename std::conditional<DT == MV_F32, float, uint16_t>::type;
  T* held = reinterpret_cast<T*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int r = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Shared& s0 = *cluster.map_shared_rank(&s, 0);
  pdl_launch_dependents();
  pdl_wait();
  const float temp = a.temperature != nullptr ? a.temperature[r] : a.temperature_value;
  const float top_p = a.top_p != nullptr ? a.top_p[r] : a.top_p_value;
  const float min_p = a.min_p != nullptr ? a.min_p[r] : a.min_p_value;
  const int top_k = a.top_k != nullptr ? a.top_k[r] : a.top_k_value;
  const float u0 = a.u[r];
  const float u = u0 > 0.f ? fminf(u0, 0.99999994f) : 0.f;  // at most the largest value below 1
  const bool greedy = !(temp > 0.f) || top_k == 1 || top_p <= 0.f || min_p > 1.f;  // the first of the order alone
  const bool by_k = !greedy && top_k > 0 && top_k < a.V, by_p = !greedy && top_p < 1.f;

  const int start = min(static_cast<long long>(a.V), static_cast<long long>(rank) * a.slice);
  const int len = min(a.slice, a.V - start), len4 = (len + 3) / 4 * 4;
  const T* src = static_cast<const T*>(a.logits) + r * a.st + start;
  auto value = [](T x) {
    if constexpr (DT == MV_F32) return x;
    else if constexpr (DT == MV_BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
    else return __half2float(__ushort_as_half(x));
  };
  const T minus_inf = [] {
    if constexpr (DT == MV_F32) return -INFINITY;
    else return static_cast<uint16_t>(DT == MV_BF16 ? 0xff80 : 0xfc00);
  }();
  // f(four logits, index of the first in the part) for this thread's share of the part; behind its end -inf
  auto each = [&](auto&& f) {
    for (int i = tid * 4; i < len4; i += kThreads * 4) {
      alignas(16) T v[4];
      if (a.in_smem) {
        if constexpr (DT == MV_F32)
          *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(held + i);
        else
          *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(held + i);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < len ? src[i + k] : minus_inf;
      }
      float l[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) l[k] = value(v[k]);
      f(l, i);
    }
  };

  // ---- 1. the row, the first of its order
  if (tid == 0) s.nan = 0u, s.n_list = 0u, s.best = ~0ull;
  if (warp == 1) s.table[lane] = exp2(lane / 32.0 + a.shift);
  __syncthreads();
  uint32_t top = 0u;
  int top_at = 0;
  bool nan = false;
  auto meet = [&](float l, int i) {  // (a thread meets its logits in the order of their indices)
    nan |= l != l;
    const uint32_t key = key_of(l);
    if (key > top) top = key, top_at = i;
  };
  if (a.in_smem) {
    constexpr int kVec = 16 / sizeof(T);
    int done = 0;
    if (a.vectors) {
      const uint4* v = reinterpret_cast<const uint4*>(src);
      done = len / kVec;
#pragma unroll 4
      for (int i = tid; i < done; i += kThreads) {
        const uint4 x = __ldcs(v + i);
        reinterpret_cast<uint4*>(held)[i] = x;
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int k = 0; k < kVec; ++k) meet(value(e[k]), i * kVec + k);
      }
      done *= kVec;
    }
#pragma unroll 4
    for (int i = done + tid; i < len4; i += kThreads) {
      const T x = i < len ? src[i] : minus_inf;
      held[i] = x;
      meet(value(x), i);
    }
  } else {
    each([&](const float (&l)[4], int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) meet(l[k], i + k);
    });
  }
  uint64_t best = top == 0u ? ~0ull : place_of(top, start + top_at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) {
    if (best != ~0ull) atomicMin(&s.best, static_cast<unsigned long long>(best));
    if (nan) s.nan = 1u;
  }
  // a key that at least `share` of this CTA's logits reach
  const int share = by_k ? (top_k + C - 1) / C : kMostMaxima + 1;
  if (share <= kMostMaxima) {
    uint32_t pivot = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t mid = pivot | 1u << bit;
      const int n = __syncthreads_count(top >= mid);
      if (n >= share) pivot = mid;
      if (n >= share && n <= share + share / 8) break;
    }
    if (tid == 0) s.pivot = pivot;
  }
  cluster_sync();
  best = ~0ull;
  unsigned int any_nan = 0;
  uint32_t pivot = 0xffffffffu;
  if (lane < C) {
    const Shared& p = *cluster.map_shared_rank(&s, lane);
    best = p.best, any_nan = p.nan;
    if (share <= kMostMaxima) pivot = p.pivot;
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
  best = __shfl_sync(0xffffffffu, best, 0);
  any_nan = __any_sync(0xffffffffu, any_nan != 0u);
  pivot = __reduce_min_sync(0xffffffffu, pivot);
  top = best == ~0ull ? 0u : ~static_cast<uint32_t>(best >> 32);
  const bool nothing = any_nan || top <= kNone;
  if (nothing || greedy) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = nothing ? -1 : static_cast<int>(static_cast<uint32_t>(best));
      if (a.logprob != nullptr) a.logprob[r] = nothing ? -INFINITY : 0.f;
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  Weights wt;
  wt.top = of_key(top), wt.table = s.table;
  wt.m = wt.top, wt.c = 1.4426950408889634 / static_cast<double>(temp);
  const double lim = -static_cast<double>(a.shift + 2);
  wt.least = wt.logit_at(lim);
  const double one = static_cast<double>(1ull << a.shift);
  const uint64_t least_w = min_p > 0.f ? static_cast<uint64_t>(fmax(ceil(static_cast<double>(min_p) * one), 1.0)) : 1;
  // logits below this are not kept whatever the other filters do
  const float least_logit = min_p > 0.f ? fmaxf(wt.least, wt.logit_at(fmax(log2(static_cast<double>(min_p)) - 1e-9, lim))) : wt.least;
  auto draw = [&](uint64_t total) {  // the sum up to the token drawn is the first above this
    const uint64_t t = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total));
    return t < total ? t : total - 1;
  };
  auto answer = [&](int token, float l, uint64_t total) {
    a.tokens[r] = token;
    // from the logit: its weight of few units would be off by half of one
    const double z = l == wt.top ? 0.0 : (static_cast<double>(l) - wt.m) / static_cast<double>(temp);
    if (a.logprob != nullptr) a.logprob[r] = static_cast<float>(z - log(static_cast<double>(total) / one));
  };

  // a place with its halves exchanged: kept tokens in the order of their indices
  auto by_index = [](uint64_t place) { return place << 32 | place >> 32; };
  auto logit_of = [](uint64_t at) { return of_key(~static_cast<uint32_t>(at)); };

  // ---- 2. few candidates
  if (share <= kMostMaxima || (!by_k && !by_p && min_p > 0.f)) {
    const float from = fmaxf(by_k ? of_key(pivot) : -INFINITY, by_p ? wt.least : least_logit);
    each([&](const float (&l)[4], int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!(l[k] >= from)) continue;
        const unsigned int at = atomicAdd(&s0.n_list, 1u);
        if (at < kList) s0.list[at] = place_of(key_of(l[k]), start + i + k);
      }
    });
    cluster_sync();
    const unsigned int count = s0.n_list;
    if (count <= kList) {
      cluster_arrive();
      if (rank > 0) return;
      if (count <= 2 * kFew) {
        // a thread for each: its place among them, and the weights before it, by comparing with all
        unsigned long long *places = s.list, *weights = places + 2 * kFew, *index = weights + 2 * kFew, *kept = index + 2 * kFew;
        uint64_t place = ~0ull, w = 0, w_before = 0;
        unsigned int n_before = 0;
        if (tid < count) {
          place = places[tid];
          const uint32_t key = ~static_cast<uint32_t>(place >> 32);
          weights[tid] = w = wt.of(of_key(key));
        }
        __syncthreads();
        if (warp * 32 < count) {
#pragma unroll 4
          for (unsigned int j = 0; j < count; ++j)
            if (places[j] < place) ++n_before, w_before += weights[j];
        }
        const unsigned int most = by_k ? min(count, static_cast<unsigned int>(top_k)) : count;
        if (tid < count && n_before == most - 1) s.kept = w_before + w;
        __syncthreads();
        bool keep = tid < count && n_before < most && w >= least_w;
        if (by_p) keep &= w_before < static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(s.kept)));
        const unsigned int n_kept = __syncthreads_count(keep);
        if (keep) {
          index[n_before] = by_index(place), kept[n_before] = w;
          if (n_before == n_kept - 1) s.total = w_before + w;
        }
        __syncthreads();
        if (tid < n_kept) {
          // the weights up to a token in the order of the indices
          const uint64_t at = index[tid], own = kept[tid], target = draw(s.total);
          uint64_t run = 0;
#pragma unroll 4
          for (unsigned int j = 0; j < n_kept; ++j)
            if (index[j] < at) run += kept[j];
          if (target >= run && target < run + own) answer(static_cast<int>(at >> 32), logit_of(at), s.total);
        }
        cluster_wait();
        return;
      }
      Listed<kThreads> list;
      list.load(count, wt, true, s);
      const uint64_t first = best, last = place_of(key_of(from), -1);  // the list's places lie between these
      uint64_t border = ~0ull - 1, sum;
      unsigned int n;
      if (by_k && count > static_cast<unsigned int>(top_k)) border = list.border(true, top_k, 0, count, first, last, s);
      if (by_p) {
        // the first place up to which the weights reach top_p of top-k's; its tokens before that are all top-k's
        list.up_to(border, sum, n, s);
        border = list.border(false, 0, static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(sum))), count, first,
                             last, s);
      }
      // kept tokens in the order of their indices: the draw's is the first up to which the sum is above the target
#pragma unroll
      for (int i = 0; i < Listed<kThreads>::kEach; ++i) {
        if (list.place[i] > border || list.w[i] < least_w) list.place[i] = ~0ull, list.w[i] = 0;
        if (list.place[i] != ~0ull) list.place[i] = by_index(list.place[i]);
      }
      uint64_t total;
      list.up_to(~0ull - 1, total, n, s);
      const uint64_t at = list.border(false, 0, draw(total) + 1, n, 0, (static_cast<uint64_t>(a.V) << 32) - 1, s);
      if (tid == 0) answer(static_cast<int>(at >> 32), logit_of(at), total);
      cluster_wait();
      return;
    }
    cluster_sync();  // all have read the count
  }

  // ---- 3. the borders
  uint64_t border = ~0ull;
  const bool bins = a.slice <= (1 << 17);  // 15 bits of as many weights fit in 32
  // the bin of a logit with a weight: how far it lies below the largest, in fp32, whose roundings keep the order (both factors are
  // held finite: distances of logits at the type's two ends, temperatures below 2^-122)
  const float per = static_cast<float>(fmin(static_cast<double>(kBins) / (a.shift + 4.0) * wt.c, 3.4e38));
  auto bin_of = [&](float l) -> unsigned int {
    return l == wt.top ? 0u : __float_as_uint(fmaf(fminf(wt.top - l, 3.4e38f), per, 8388608.0f)) & (kBins * 2 - 1);  // 2^23
  };
  // first top-k's border, then top-p's among what top-k keeps
  for (int phase = by_k ? 0 : 1; phase < (by_p ? 2 : 1); ++phase) {
    // what the last phase kept: logits above `from`, and equal ones up to an index
    const uint32_t from_key = max(key_of(wt.least), ~static_cast<uint32_t>(border >> 32));
    const float from = of_key(from_key);
    const unsigned int from_last = from_key == ~static_cast<uint32_t>(border >> 32) ? static_cast<uint32_t>(border) : 0xffffffffu;
    auto is_in = [&](float l, int i) { return l > from || (l == from && static_cast<unsigned int>(start + i) <= from_last); };
    uint64_t need_w = ~0ull, w;  // top-p keeps a token while the weights before it are less
    const unsigned int need_n = static_cast<unsigned int>(top_k);
    unsigned int bin = 0xffffffffu, n;
    uint32_t bin_from = 0u, bin_to = 0xffffffffu;
    if (tid == 0) s.n_list = 0u, s.bin = bin, s.bin_here = -1, s.least_place = ~0ull, s.most_place = 0ull;
    if (bins) {
      for (int i = tid; i < 4 * kBins; i += kThreads) s.bins[0][i] = 0u;
      __syncthreads();
      each([&](const float (&l)[4], int i) {
        if (phase == 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (is_in(l[k], i + k)) atomicAdd(&s.bins[0][bin_of(l[k])], 1u);
        } else {
          uint64_t x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = wt.of(l[k]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (!is_in(l[k], i + k)) continue;
            const unsigned int b = bin_of(l[k]);
            atomicAdd(&s.bins[1][b], static_cast<unsigned int>(x[k]) & 0x7fffu);
            atomicAdd(&s.bins[2][b], static_cast<unsigned int>(x[k]) >> 15 & 0x7fffu);
            atomicAdd(&s.bins[3][b], static_cast<unsigned int>(x[k] >> 30));
          }
        }
      });
      cluster_sync();
      // each CTA adds up a share of the bins over all CTAs, a few neighbours to a thread
      constexpr int kPer = kBins / kThreads;
      const int share_bins = (kBins + C - 1) / C, per_thread = (share_bins + kThreads - 1) / kThreads;
      const int share_end = min(kBins, (rank + 1) * share_bins);
      uint64_t wb[kPer] = {}, all_w;
      unsigned int nb[kPer] = {}, all_n;
      w = 0, n = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int b = rank * share_bins + tid * per_thread + i;
        if (i >= per_thread || b >= share_end) continue;
        unsigned int x[3][8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            x[q][c] = 0u;
            if (c < C && (q == 0 || phase == 1)) x[q][c] = cluster.map_shared_rank(&s, c)->bins[phase == 0 ? 0 : q + 1][b];
          }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (phase == 0)
            nb[i] += x[0][c];
          else
            wb[i] += x[0][c] + (static_cast<uint64_t>(x[1][c]) << 15) + (static_cast<uint64_t>(x[2][c]) << 30);
        }
        w += wb[i], n += nb[i];
      }
      block_before(w, n, all_w, all_n, s);
      if (tid == 0) s.total = all_w, s.part_n = all_n;
      cluster_sync();
      {
        uint64_t of_lane = 0;
        unsigned int n_lane = 0;
        if (lane < C) {
          const Shared& p = *cluster.map_shared_rank(&s, lane);
          of_lane = p.total, n_lane = p.part_n;
        }
        all_w = warp_sum(of_lane);
        w += warp_sum(lane < rank ? of_lane : 0ull);
        n += __reduce_add_sync(0xffffffffu, lane < rank ? n_lane : 0u);
      }
      need_w = static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(all_w)));
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (phase == 0 ? n < need_n && n + nb[i] >= need_n : w < need_w && w + wb[i] >= need_w) {
          s0.bin = rank * share_bins + tid * per_thread + i, s0.bin_before = w, s0.bin_count_before = n;
          s.bin_here = rank * share_bins + tid * per_thread + i;
        }
        w += wb[i], n += nb[i];
      }
      __syncthreads();
      if (warp < 2 && s.bin_here >= 0) {
        // the bin's least and largest keys: a key's bin falls as the key rises
        const unsigned int b = s.bin_here;
        const unsigned int most = warp == 0 ? b : b - 1;  // the least key with at most this bin, which the largest logit's is
        uint32_t key = top;
        if (b > 0u || warp == 0) {
          // where the rounding to the bin turns it is near; else 32 keys at a time are tried
          const double l0 = wt.m - (most + 0.5) / static_cast<double>(per);
          const uint32_t guess = key_of(l0 > -3.4e38 ? static_cast<float>(l0) : -3.4e38f);
          uint32_t lo = from_key, hi = top;
          uint32_t tried = min(max(static_cast<int64_t>(guess) - 16 + lane, static_cast<int64_t>(from_key)), static_cast<int64_t>(top));
          unsigned int in = __ballot_sync(0xffffffffu, bin_of(of_key(tried)) <= most);
          if (in != 0u && !(in & 1u)) {
            lo = hi = __shfl_sync(0xffffffffu, tried, __ffs(in) - 1);
          }
          while (lo < hi) {
            const uint32_t part = (hi - lo) / 32 + 1;
            tried = min(static_cast<uint64_t>(lo) + static_cast<uint64_t>(part) * lane, static_cast<uint64_t>(hi));
            in = __ballot_sync(0xffffffffu, bin_of(of_key(tried)) <= most);
            if (in == 0u) {
              lo = __shfl_sync(0xffffffffu, tried, 31) + 1;
            } else {
              const int k = __ffs(in) - 1;
              hi = __shfl_sync(0xffffffffu, tried, k);
              lo = k == 0 ? hi : __shfl_sync(0xffffffffu, tried, k - 1) + 1;
            }
          }
          key = warp == 0 ? hi : hi - 1;
        }
        if (lane == 0) (warp == 0 ? s0.bin_from : s0.bin_to) = key;
      }
      cluster_sync();
      bin = s0.bin;
      if (bin == 0xffffffffu) continue;  // top_k keeps all that has a weight
      bin_from = s0.bin_from, bin_to = s0.bin_to;
      const uint64_t w_before = s0.bin_before;
      const unsigned int n_before = s0.bin_count_before;
      const float bin_least = of_key(bin_from), bin_most = of_key(bin_to);
      each([&](const float (&l)[4], int i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!(l[k] >= bin_least && l[k] <= bin_most && is_in(l[k], i + k))) continue;
          const unsigned int at = atomicAdd(&s0.n_list, 1u);
          if (at < kList) s0.list[at] = place_of(key_of(l[k]), start + i + k);
        }
      });
      cluster_sync();
      const unsigned int count = s0.n_list;
      if (count <= kList) {
        if (rank == 0) {
          Listed<kThreads> list;
          list.load(count, wt, phase == 1, s);
          list.border(phase == 0, need_n - n_before, need_w - w_before, count, place_of(bin_to, 0), place_of(bin_from, -1), s);
        }
        cluster_sync();
        border = s0.border;
        continue;
      }
    }
    // the same over all CTAs' parts; counts and weights of what lies before `end`
    auto before = [&](uint64_t end) {
      w = 0, n = 0;
      each([&](const float (&l)[4], int i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!is_in(l[k], i + k) || place_of(key_of(l[k]), start + i + k) >= end) continue;
          ++n;
          if (phase == 1) w += wt.of(l[k]);
        }
      });
      block_sum(w, n, s);
      if (tid == 0) s.total = w, s.part_n = n;
      cluster_sync();
      w = 0, n = 0;
      if (lane < C) {
        const Shared& p = *cluster.map_shared_rank(&s, lane);
        w = p.total, n = p.part_n;
      }
      w = warp_sum(w), n = __reduce_add_sync(0xffffffffu, n);
      cluster_sync();
    };
    if (!bins) {
      before(~0ull);
      if (phase == 0 && n < need_n) continue;
      need_w = static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(w)));
    }
    uint64_t first = ~0ull, last = 0;
    each([&](const float (&l)[4], int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t key = key_of(l[k]);
        const uint64_t place = place_of(key, start + i + k);
        if (!is_in(l[k], i + k) || key < bin_from || key > bin_to) continue;
        first = min(first, place), last = max(last, place);
      }
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    if (lane == 0 && first != ~0ull) {
      atomicMin(&s.least_place, static_cast<unsigned long long>(first));
      atomicMax(&s.most_place, static_cast<unsigned long long>(last));
    }
    cluster_sync();
    first = ~0ull, last = 0;
    if (lane < C) {
      const Shared& p = *cluster.map_shared_rank(&s, lane);
      first = p.least_place, last = p.most_place;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    first = __shfl_sync(0xffffffffu, first, 0), last = __shfl_sync(0xffffffffu, last, 0);
    int bit = first == last ? -1 : 63 - __clzll(first ^ last);
    uint64_t low = bit < 0 ? first : first >> bit >> 1 << bit << 1;
    for (; bit >= 0; --bit) {
      before(low | 1ull << bit);
      if (phase == 0 ? n < need_n : w < need_w) low |= 1ull << bit;
    }
    border = low;
    cluster_sync();  // all have read the first CTA's places
  }

  // ---- 4. the draw
  const uint32_t last_key = max(~static_cast<uint32_t>(border >> 32), key_of(least_logit));
  const float last_logit = of_key(last_key);
  const unsigned int last_index = last_key == ~static_cast<uint32_t>(border >> 32) ? static_cast<uint32_t>(border) : 0xffffffffu;
  auto load = [&](int i) { return value(a.in_smem ? held[i] : src[i]); };
  // weights of four elements from i on, `step` apart, that lie before `end`; 0 for those not kept
  auto kept = [&](int i, int step, int end, uint64_t (&w)[4]) {
    float l[4];
    bool any = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      l[k] = -INFINITY, w[k] = 0;
      if (i + k * step < end) l[k] = load(i + k * step);
      any |= l[k] >= last_logit;
    }
    if (!any) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t x = wt.of(l[k]);
      if (l[k] > last_logit || (l[k] == last_logit && static_cast<unsigned int>(start + i + k * step) <= last_index)) w[k] = x;
    }
    if (least_w > 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (w[k] < least_w) w[k] = 0;
    }
  };
  // warp w owns a contiguous range of the part
  const int range = (len4 + kWarps * 4 - 1) / (kWarps * 4) * 4, range_end = min(len, (warp + 1) * range);
  uint64_t mine = 0, w4[4];
  for (int i = warp * range + lane; i < range_end; i += 128) {
    kept(i, 32, range_end, w4);
    mine += w4[0] + w4[1] + w4[2] + w4[3];
  }
  mine = warp_sum(mine);
  if (lane == 0) s.part[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const uint64_t all = warp_sum(lane < kWarps ? s.part[lane] : 0ull);
    if (lane == 0) s.total = all;
  }
  cluster_sync();
  const uint64_t of_lane = lane < C ? cluster.map_shared_rank(&s, lane)->total : 0ull;
  const uint64_t total = warp_sum(of_lane);
  uint64_t before = warp_sum(lane < rank ? of_lane : 0ull);
  const uint64_t target = draw(total), own = s.total;
  cluster_sync();  // no CTA leaves while another reads its total
  if (target < before || target >= before + own) return;
  int part = 0;
  while (part < kWarps - 1 && target >= before + s.part[part]) before += s.part[part++];
  __syncthreads();
  // the range's elements in order: a thread takes neighbours
  const int i0 = part * range, i1 = min(len, i0 + range), per_thread = (i1 - i0 + kThreads - 1) / kThreads;
  const int lo = min(i0 + tid * per_thread, i1), hi = min(lo + per_thread, i1);
  uint64_t mass = 0, all_w;
  unsigned int n = 0, all_n;
  for (int i = lo; i < hi; i += 4) {
    kept(i, 1, hi, w4);
    mass += w4[0] + w4[1] + w4[2] + w4[3];
  }
  const uint64_t have = mass;
  block_before(mass, n, all_w, all_n, s);
  uint64_t run = before + mass;
  if (target < run || target >= run + have) return;
  for (int i = lo; i < hi; i += 4) {
    kept(i, 1, hi, w4);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (target >= run && target < run + w4[k]) answer(start + i + k, load(i + k), total);
      run += w4[k];
    }
  }
}

constexpr size_t kSm = 227 * 1024;  // shared memory of an SM, of which a CTA takes 1 KB for itself

template <int kThreads>
constexpr size_t fixed_smem() {
  return (sizeof(Shared<kThreads>) + 15) / 16 * 16;
}

template <int DT, int kThreads>
int launch(SampleArgs a, int B, int C, cudaStream_t st) {
  const int size = DT == MV_F32 ? 4 : 2;
  a.slice = ((a.V + C - 1) / C + 7) / 8 * 8;
  a.in_smem = static_cast<size_t>(a.slice) * size <= kSm - fixed_smem<kThreads>();
  const size_t smem = fixed_smem<kThreads>() + (a.in_smem ? static_cast<size_t>(a.slice) * size : 0);
  auto fn = sample_kernel<DT, kThreads>;
  // the most that any call takes: the limit is the kernel's, not the launch's, and another thread may be about to launch
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSm));
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(mv_sample)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned int>(B) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, fn, a), "mv_sample launch");
}

// CTAs of a row. Few rows: CTAs of 512 threads, as many a row as fill 5/7 of the SMs, which is what clusters find together (16 rows of
// 131072, top-p, us: 6 CTAs a row 36, 7 63, 8 42; one row: 28, and 34 with 256 threads). More rows: up to four CTAs of 256 share an SM,
// some of which read or wait while others compute (48 rows of 100277, three on an SM, top-p, us: 45; two of 512 65): at least as many a
// row as leaves room for four, or eight, and more up to 7/8 of the places. Where three of eight CTAs' parts find no room on an SM, two of
// 512 threads (192 rows of 131072 in f32, min_p: 61 us; two of 256 65).
template <int DT>
int launch_rows(const SampleArgs& a, int B, cudaStream_t st) {
  const int size = DT == MV_F32 ? 4 : 2, sms = num_sms();
  if (4LL * B <= sms * 5 / 7) {
    const int C = sms * 5 / 7 / B;
    return launch<DT, 512>(a, B, C < 8 ? C : 8, st);
  }
  // whether n CTAs' parts, c of them a row, find room on an SM
  const auto fits = [&](int c, int n, size_t fixed) { return (static_cast<size_t>(a.V) / c + 8) * size <= kSm / n - 1024 - fixed; };
  int C = 1;
  if (!fits(8, 3, fixed_smem<256>())) {
    while (C < 8 && !fits(C, 2, fixed_smem<512>())) ++C;
    return launch<DT, 512>(a, B, C, st);
  }
  while (C < 8 && (!fits(C, 4, fixed_smem<256>()) || static_cast<long long>(B) * (C + 1) <= sms * 7 / 2)) ++C;
  return launch<DT, 256>(a, B, C, st);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" size_t mv_sample_scratch_bytes(int, int) { return 0; }

extern "C" int mv_sample(const mv_sample_args* x, void* stream) {
  const char* who = "mv_sample";
  if (x == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (x->dtype != MV_BF16 && x->dtype != MV_F16 && x->dtype != MV_F32)
    return fail(MV_ERR_UNSUPPORTED, "%s: logits must be bf16, f16 or f32", who);
  if (x->B < 0 || x->B > (1 << 27) || x->V < 0 || x->V > (1 << 30))
    return fail(MV_ERR_INVALID, "%s: bad B=%d / V=%d", who, x->B, x->V);
  if (x->B == 0) return MV_OK;
  if (x->u == nullptr || x->tokens == nullptr || (x->V > 0 && x->logits == nullptr))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (x->B > 1 && x->st < 0) return fail(MV_ERR_INVALID, "%s: negative row stride %lld", who, x->st);
  const int size = x->dtype == MV_F32 ? 4 : 2;
  SampleArgs a{};
  a.logits = x->logits, a.u = x->u, a.temperature = x->temperature, a.top_p = x->top_p, a.min_p = x->min_p;
  a.top_k = x->top_k, a.tokens = x->tokens, a.logprob = x->logprob, a.st = x->B > 1 ? x->st : 0;
  a.temperature_value = x->temperature_value, a.top_p_value = x->top_p_value, a.min_p_value = x->min_p_value;
  a.top_k_value = x->top_k_value, a.V = x->V;
  // Weights stay below 2^52, and sums of V of them within 2^61: those of their bits from 30 on (2^31) fit in 32, for a list that holds
  // the whole row too. It goes by V alone, so that a row's weights do not depend on the batch or the split.
  a.shift = 61 - attn::log2_of(x->V > 1 ? x->V : 2);
  if (a.shift > 51) a.shift = 51;
  a.vectors = aligned16(x->logits) && a.st * size % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x->dtype == MV_F32) return launch_rows<MV_F32>(a, x->B, st);
  return x->dtype == MV_BF16 ? launch_rows<MV_BF16>(a, x->B, st) : launch_rows<MV_F16>(a, x->B, st);
}
