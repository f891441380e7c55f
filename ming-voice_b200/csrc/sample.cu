// Drawing tokens from logits with temperature, top-k, top-p and min-p (mv_sample).
//
// Mathematics. Tokens are ordered by (logit descending, index ascending), as one 64-bit number `place`: the logit's bits, mapped
// so that unsigned comparison orders them, in the upper half and the index in the lower. Each filter keeps a prefix of that order,
// so all that is kept is given by one place, the border, and a least weight. Weights 2^t, t = (logit - max) log2(e) / temperature,
// are whole numbers of 2^-shift (shift 45 for vocabularies up to 2^17; the polynomial for 2^f, by interpolation at the Chebyshev
// nodes of [-1/2, 1/2], is off by 2^-44 of it at most), so that sums do not depend on their order: each border and each draw comes out
// the same whatever the split, and a weight below 2^-shift / 2, which no 24-bit random number can draw, is 0.
//
// Steps, a cluster of CTAs for each row, the row in their shared memory:
//   1. read the row once; the largest logit
//   2. (top-k, top-p) a histogram of t: counts and weights of 2048 bins, added up in the first CTA, which finds the bin with
//      the border; that bin's tokens are brought together there, and their ranks and weight sums by counting give the border.
//      A bin with more tokens than the list holds (runs of equal logits) is searched bit by bit over all CTAs.
//   3. each CTA adds up what is kept of its part; the CTA in which the sum passes u times the total finds the token.
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

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kList = 4096;
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

// Weights of one row as whole numbers.
struct Weights {
  double m, c, lim;  // largest logit, log2(e) / temperature, least t that has a weight
  uint32_t top, least;  // keys: of the largest logit, and of the least that can have a weight
  int shift;
  __device__ __forceinline__ double t_of(float l) const { return (static_cast<double>(l) - m) * c; }
  // 2^t in units of 2^-shift, for -48 <= t <= 0 (lower ones: 0)
  __device__ __forceinline__ uint64_t of(float l, double t) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the low word of a sum with it is the number, rounded
    if (t < lim) return 0;
    const double r = t + kRound;
    const int n = __double2loint(r);
    const double f = t - (r - kRound);
    double p = 1.0203121063391729e-07;
    p = fma(p, f, 1.3255224878668817e-06);
    p = fma(p, f, 1.525268684626772e-05);
    p = fma(p, f, 0.00015403455852453838);
    p = fma(p, f, 0.0013333558179043112);
    p = fma(p, f, 0.009618129159402558);
    p = fma(p, f, 0.055504108664760424);
    p = fma(p, f, 0.2402265069581299);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    const double s = __hiloint2double((1023 + n + shift) << 20, 0);
    return static_cast<uint64_t>(__double_as_longlong(fma(p, s, 4503599627370496.0))) & 0xfffffffffffffull;  // 2^52
  }
  __device__ __forceinline__ uint64_t of(float l) const { return of(l, t_of(l)); }
};

__device__ __forceinline__ uint64_t shfl_down(uint64_t v, int o) { return __shfl_down_sync(0xffffffffu, v, o); }

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  unsigned long long weight[kBins];
  unsigned long long list[kList];
  unsigned long long part[kWarps], total, border, found_weight;
  unsigned long long bin_before;  // of the bin that is looked into: weights of the bins before it
  unsigned int count[kBins];
  unsigned int counts[kWarps];
  unsigned int n_list, top, nan, bin, bin_count_before, bin_count;
  unsigned long long need, kept, least_place, most_place;
  unsigned int part_n;
  int token;
};

// Sums of (w, n) over the CTA in every thread. Two barriers.
__device__ __forceinline__ void block_sum(uint64_t& w, unsigned int& n, Shared& s) {
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
__device__ __forceinline__ void block_before(uint64_t& w, unsigned int& n, uint64_t& total_w, unsigned int& total_n, Shared& s) {
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

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
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
  // f(logit, index in the part) for this thread's share of the part; behind its end -inf
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
#pragma unroll
      for (int k = 0; k < 4; ++k) f(value(v[k]), i + k);
    }
  };

  // ---- 1. the row, its largest logit
  if (tid == 0) s.top = 0u, s.nan = 0u, s.n_list = 0u, s.token = 0x7fffffff, s.border = ~0ull;
  if (by_k || by_p)
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0u, s.weight[i] = 0ull;
  __syncthreads();
  uint32_t top = 0u;
  bool nan = false;
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
        for (int k = 0; k < kVec; ++k) {
          const float l = value(e[k]);
          nan |= l != l;
          top = max(top, key_of(l));
        }
      }
      done *= kVec;
    }
    for (int i = done + tid; i < len4; i += kThreads) {
      const T x = i < len ? src[i] : minus_inf;
      held[i] = x;
      const float l = value(x);
      nan |= l != l;
      top = max(top, key_of(l));
    }
  } else {
    each([&](float l, int) {
      nan |= l != l;
      top = max(top, key_of(l));
    });
  }
  top = __reduce_max_sync(0xffffffffu, top);
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) {
    atomicMax(&s.top, top);
    if (nan) s.nan = 1u;
  }
  cluster.sync();
  top = 0u;
  unsigned int any_nan = 0;
  for (int i = 0; i < C; ++i) {
    const Shared& p = *cluster.map_shared_rank(&s, i);
    top = max(top, p.top);
    any_nan |= p.nan;
  }
  if (any_nan || top <= kNone) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprob != nullptr) a.logprob[r] = -INFINITY;
    }
    cluster.sync();
    return;
  }
  if (greedy) {
    int first = 0x7fffffff;
    each([&](float l, int i) {
      if (key_of(l) == top) first = min(first, i);
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first != 0x7fffffff) atomicMin(&s0.token, start + first);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      a.tokens[r] = s.token;
      if (a.logprob != nullptr) a.logprob[r] = 0.f;
    }
    return;
  }
  Weights wt;
  wt.top = top, wt.shift = a.shift;
  wt.m = of_key(top), wt.c = 1.4426950408889634 / static_cast<double>(temp);
  wt.lim = -static_cast<double>(a.shift + 2);
  // logits below `least` have no weight for certain (rounded down; where the maximum is infinite, all others have none)
  {
    const double l = wt.m + wt.lim / wt.c * 1.0000001;
    float f = l > -3.4e38 ? __double2float_rd(l) : -3.4028235e38f;
    if (top == 0xff800000u) f = INFINITY;
    wt.least = key_of(f);
  }
  const uint64_t one = 1ull << a.shift;
  // the weight of a logit whose key is at least `least`
  auto weight = [&](float l, uint32_t key) { return key == top ? one : wt.of(l); };

  // ---- 2. the border
  uint64_t border = ~0ull;
  if (by_k || by_p) {
    const double per = -static_cast<double>(kBins) / (a.shift + 4.0);
    auto bin_of = [&](float l, uint32_t key) { return key == top ? 0 : __double2int_rz(fmax(wt.t_of(l), wt.lim) * per); };
    each([&](float l, int) {
      const uint32_t key = key_of(l);
      if (key < wt.least) return;
      const int b = bin_of(l, key);
      atomicAdd(&s.count[b], 1u);
      atomicAdd(&s.weight[b], static_cast<unsigned long long>(weight(l, key)));
    });
    __syncthreads();
    if (rank > 0)
      for (int i = tid; i < kBins; i += kThreads)
        if (s.count[i] != 0u) {
          atomicAdd(&s0.count[i], s.count[i]);
          atomicAdd(&s0.weight[i], s.weight[i]);
        }
    uint64_t need = ~0ull;  // top-p keeps a token while the weights before it are less
    unsigned int need_n = by_k ? static_cast<unsigned int>(top_k) : 0xffffffffu;
    // first top-k's border, whose weights top-p is a share of, then top-p's
    for (int phase = by_k ? 0 : 1; phase < (by_p ? 2 : 1); ++phase) {
      cluster.sync();
      if (rank == 0) {
        constexpr int kPer = kBins / kThreads;
        uint64_t w = 0, sum;
        unsigned int n = 0, all;
        for (int i = 0; i < kPer; ++i) w += s.weight[tid * kPer + i], n += s.count[tid * kPer + i];
        block_before(w, n, sum, all, s);
        if (phase == 1) {
          // (after top-k: of the weights that it kept)
          const uint64_t kept = by_k ? s.kept : sum;
          need = static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(kept)));
        }
        __syncthreads();
        if (tid == 0) {
          s.bin = 0xffffffffu, s.n_list = 0u, s.border = border, s.need = need;
          s.least_place = ~0ull, s.most_place = 0ull;
        }
        __syncthreads();
        if (phase == 0 && all < need_n && tid == 0) s.kept = sum;  // all that has a weight is kept
        for (int i = 0; i < kPer; ++i) {
          const int b = tid * kPer + i;
          const uint64_t wb = s.weight[b];
          const unsigned int nb = s.count[b];
          const bool here = phase == 0 ? n < need_n && n + nb >= need_n : w < need && w + wb >= need;
          if (here) s.bin = b, s.bin_before = w, s.bin_count_before = n, s.bin_count = nb;
          w += wb, n += nb;
        }
      }
      cluster.sync();
      const unsigned int bin = s0.bin;
      if (bin == 0xffffffffu) continue;
      need = s0.need;
      const uint64_t w_before = s0.bin_before;
      const unsigned int n_before = s0.bin_count_before, n_bin = s0.bin_count;
      if (n_bin <= kList) {
        each([&](float l, int i) {
          const uint32_t key = key_of(l);
          if (key < wt.least || bin_of(l, key) != static_cast<int>(bin)) return;
          s0.list[atomicAdd(&s0.n_list, 1u)] = place_of(key, start + i);
        });
        cluster.sync();
        if (rank == 0) {
          // each thread has some of the list's tokens; the border is found bit by bit from the first that differs
          constexpr int kEach = kList / kThreads;
          uint64_t place[kEach], w[kEach], first = ~0ull, last = 0;
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            const unsigned int at = tid + i * kThreads;
            place[i] = ~0ull, w[i] = 0;
            if (at >= n_bin) continue;
            place[i] = s.list[at];
            const uint32_t key = ~static_cast<uint32_t>(place[i] >> 32);
            w[i] = weight(of_key(key), key);
            first = min(first, place[i]), last = max(last, place[i]);
          }
          if (first != ~0ull) {
            atomicMin(&s.least_place, static_cast<unsigned long long>(first));
            atomicMax(&s.most_place, static_cast<unsigned long long>(last));
          }
          __syncthreads();
          first = s.least_place, last = s.most_place;
          int bit = first == last ? -1 : 63 - __clzll(first ^ last);
          uint64_t low = bit < 0 ? first : first >> bit >> 1 << bit << 1;
          unsigned int n_low = 0, n_high = n_bin;  // tokens before low, and before the end of what is left
          for (; bit >= 0 && n_high - n_low > 1; --bit) {
            const uint64_t mid = low | 1ull << bit;
            uint64_t sum = 0;
            unsigned int n = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
              if (place[i] < mid) ++n, sum += w[i];
            block_sum(sum, n, s);
            if (phase == 0 ? n_before + n < need_n : w_before + sum < need)
              low = mid, n_low = n;
            else
              n_high = n;
          }
          // one token is left at or behind low, and what lies before low
          const uint64_t end = bit < 0 ? low + 1 : low + (2ull << bit);
          uint64_t sum = 0;
          unsigned int n = 0;
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            if (place[i] >= low && place[i] < end && place[i] != ~0ull) s.border = min(place[i], border);
            if (place[i] < end) sum += w[i];
          }
          block_sum(sum, n, s);
          if (tid == 0) s.kept = w_before + sum;
        }
        cluster.sync();
      } else {
        // the same over all CTAs' parts
        uint64_t first = ~0ull, last = 0;
        each([&](float l, int i) {
          const uint32_t key = key_of(l);
          if (key < wt.least || bin_of(l, key) != static_cast<int>(bin)) return;
          const uint64_t o = place_of(key, start + i);
          first = min(first, o), last = max(last, o);
        });
        if (first != ~0ull) {
          atomicMin(&s0.least_place, static_cast<unsigned long long>(first));
          atomicMax(&s0.most_place, static_cast<unsigned long long>(last));
        }
        cluster.sync();
        first = s0.least_place, last = s0.most_place;
        // counts and weights of what lies before `end`, over all CTAs
        auto before = [&](uint64_t end, uint64_t& w, unsigned int& n) {
          w = 0, n = 0;
          each([&](float l, int i) {
            const uint32_t key = key_of(l);
            if (key < wt.least || place_of(key, start + i) >= end) return;
            ++n;
            w += weight(l, key);
          });
          block_sum(w, n, s);
          if (tid == 0) s.total = w, s.part_n = n;
          cluster.sync();
          w = 0, n = 0;
          for (int i = 0; i < C; ++i) {
            const Shared& p = *cluster.map_shared_rank(&s, i);
            w += p.total, n += p.part_n;
          }
          cluster.sync();
        };
        int bit = first == last ? -1 : 63 - __clzll(first ^ last);
        uint64_t low = bit < 0 ? first : first >> bit >> 1 << bit << 1, w;
        unsigned int n;
        for (; bit >= 0; --bit) {
          before(low | 1ull << bit, w, n);
          if (phase == 0 ? n < need_n : w < need) low |= 1ull << bit;
        }
        if (phase == 0) before(low + 1, w, n);
        if (rank == 0 && tid == 0) s.border = min(low, border), s.kept = w;
        cluster.sync();
      }
      border = s0.border;
      // (the next phase's first barrier comes before the first CTA changes it)
    }
  }

  // ---- 3. the draw
  const uint64_t least_w = min_p > 0.f ? static_cast<uint64_t>(fmax(ceil(static_cast<double>(min_p) * static_cast<double>(one)), 1.0)) : 1;
  const uint32_t last_key = max(~static_cast<uint32_t>(border >> 32), wt.least);
  auto kept = [&](float l, int i) -> uint64_t {
    const uint32_t key = key_of(l);
    if (key < last_key || place_of(key, start + i) > border) return 0;
    const uint64_t w = weight(l, key);
    return w >= least_w ? w : 0;
  };
  // warp w owns a contiguous range of the part
  const int range = (len4 + kWarps * 4 - 1) / (kWarps * 4) * 4;
  uint64_t mine = 0;
  for (int i = warp * range + lane; i < min(len, (warp + 1) * range); i += 32)
    mine += kept(value(a.in_smem ? held[i] : src[i]), i);
  mine = warp_sum(mine);
  if (lane == 0) s.part[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const uint64_t all = warp_sum(lane < kWarps ? s.part[lane] : 0ull);
    if (lane == 0) s.total = all;
  }
  cluster.sync();
  uint64_t before = 0, total = 0;
  for (int i = 0; i < C; ++i) {
    const uint64_t t = cluster.map_shared_rank(&s, i)->total;
    if (i < rank) before += t;
    total += t;
  }
  // the sum up to the token is the first above this
  uint64_t target = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total));
  target = target < total ? target : total - 1;
  const uint64_t own = s.total;
  cluster.sync();  // no CTA leaves, or writes part[], while another reads its total
  if (target < before || target >= before + own) return;
  int w = 0;
  while (w < kWarps - 1 && target >= before + s.part[w]) before += s.part[w++];
  // the range's elements in order: a thread takes neighbours
  const int i0 = w * range, n_range = min(len, i0 + range) - i0, per = (n_range + kThreads - 1) / kThreads;
  const int lo = min(i0 + tid * per, i0 + n_range), hi = min(lo + per, i0 + n_range);
  uint64_t mass = 0, unused_w;
  unsigned int n = 0, unused_n;
  for (int i = lo; i < hi; ++i) mass += kept(value(a.in_smem ? held[i] : src[i]), i);
  const uint64_t have = mass;
  __syncthreads();
  block_before(mass, n, unused_w, unused_n, s);
  uint64_t run = before + mass;
  if (target < run || target >= run + have) return;
  for (int i = lo; i < hi; ++i) {
    const uint64_t x = kept(value(a.in_smem ? held[i] : src[i]), i);
    if (target < run + x) {
      a.tokens[r] = start + i;
      if (a.logprob != nullptr) a.logprob[r] = static_cast<float>(log(static_cast<double>(x) / static_cast<double>(total)));
      break;
    }
    run += x;
  }
}

template <int DT>
int launch(SampleArgs a, int B, cudaStream_t st) {
  const int size = DT == MV_F32 ? 4 : 2;
  constexpr size_t kFixed = (sizeof(Shared) + 15) / 16 * 16;
  constexpr size_t kMost = 227 * 1024;
  // as many CTAs a row as keep the card busy, more where the row does not fit in their shared memory
  int C = 1;
  while (C < 8 && (static_cast<long long>(B) * C * 2 <= num_sms() || (static_cast<size_t>(a.V) / C + 8) * size > kMost - kFixed)) C *= 2;
  a.slice = ((a.V + C - 1) / C + 7) / 8 * 8;
  a.in_smem = static_cast<size_t>(a.slice) * size <= kMost - kFixed;
  const size_t smem = kFixed + (a.in_smem ? static_cast<size_t>(a.slice) * size : 0);
  auto fn = sample_kernel<DT>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
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
  // sums of V weights stay below 2^62, weights below 2^52
  a.shift = 62 - attn::log2_of(x->V > 1 ? x->V : 2);
  if (a.shift > 45) a.shift = 45;
  a.vectors = aligned16(x->logits) && a.st * size % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x->dtype == MV_F32) return launch<MV_F32>(a, x->B, st);
  return x->dtype == MV_BF16 ? launch<MV_BF16>(a, x->B, st) : launch<MV_F16>(a, x->B, st);
}
