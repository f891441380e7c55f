// Drawing tokens from logits with temperature, top-k, top-p and min-p (mv_sample).
//
// Mathematics: the order (logit descending, index ascending) makes each filter a prefix of it, so what is kept is one border:
// a key, and the last index that is kept among the logits equal to it. Keys are the logits' bits, mapped so that unsigned
// comparison orders them (the two zeros are one key). The border of top-k is the largest key with at least k logits at or
// above it; that of top-p the largest key at or above which the weights reach top_p times their sum; both are found bit by bit.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_common.cuh"
#include "common.cuh"

namespace mv {
namespace {

struct SampleArgs {
  const void* logits;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  long long* tokens;
  float* logprob;
  long long st;
  float temperature_value, top_p_value, min_p_value;
  int top_k_value, V;
};

constexpr int kThreads = 1024;

template <int DT>
__device__ __forceinline__ float logit(const void* row, int i) {
  if (DT == MV_F32) return static_cast<const float*>(row)[i] + 0.f;  // -0 -> +0
  if (DT == MV_BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16) + 0.f;
  return __half2float(static_cast<const __half*>(row)[i]) + 0.f;
}

__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}

struct Pair {
  double w;
  long long n;
};

__device__ __forceinline__ Pair block_sum(Pair v, Pair* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
    v.n += __shfl_xor_sync(0xffffffffu, v.n, o);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & 31];
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
    v.n += __shfl_xor_sync(0xffffffffu, v.n, o);
  }
  return v;
}

// Exclusive sums over the threads before this one, in thread order.
__device__ __forceinline__ Pair block_before(Pair v, Pair* part) {
  __shared__ Pair all[kThreads];
  all[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    Pair s{0.0, 0};
    for (int i = 0; i < kThreads; ++i) {
      const Pair t = all[i];
      all[i] = s;
      s.w += t.w, s.n += t.n;
    }
  }
  __syncthreads();
  const Pair r = all[threadIdx.x];
  __syncthreads();
  return r;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  __shared__ Pair part[32];
  __shared__ uint32_t s_key;
  __shared__ int s_idx;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, tid = threadIdx.x, V = a.V;
  const void* row = static_cast<const uint8_t*>(a.logits) + r * a.st * (DT == MV_F32 ? 4 : 2);
  const float temp = a.temperature != nullptr ? a.temperature[r] : a.temperature_value;
  const float top_p = a.top_p != nullptr ? a.top_p[r] : a.top_p_value;
  const float min_p = a.min_p != nullptr ? a.min_p[r] : a.min_p_value;
  const int top_k = a.top_k != nullptr ? a.top_k[r] : a.top_k_value;
  const float u0 = a.u[r];
  const double u = u0 > 0.f ? fminf(u0, 0.99999994f) : 0.f;  // the largest value below 1

  if (tid == 0) s_key = 0u, s_idx = 0x7fffffff;
  __syncthreads();
  uint32_t top = 0u;
  bool nan = false;
  for (int i = tid; i < V; i += kThreads) {
    const float l = logit<DT>(row, i);
    nan |= l != l;
    top = max(top, key_of(l));
  }
  atomicMax(&s_key, top);
  const bool any_nan = __syncthreads_or(nan);
  top = s_key;
  if (any_nan || V == 0 || top <= key_of(-INFINITY)) {
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprob != nullptr) a.logprob[r] = -INFINITY;
    }
    return;
  }
  const float m = __uint_as_float((top & 0x80000000u) ? top ^ 0x80000000u : ~top);
  const double t = temp;
  const bool greedy = !(temp > 0.f);
  auto weight = [&](float l) { return l == m ? 1.0 : exp((static_cast<double>(l) - static_cast<double>(m)) / t); };
  // sums of weights and counts of the logits whose key is at least k
  auto above = [&](uint32_t k) {
    Pair s{0.0, 0};
    for (int i = tid; i < V; i += kThreads) {
      const float l = logit<DT>(row, i);
      if (key_of(l) >= k) s.w += weight(l), s.n += 1;
    }
    return block_sum(s, part);
  };
  uint32_t border = 0u;            // kept: keys above the border, and the first `ties` of those equal to it
  long long ties = 0x7fffffffffffll;
  if (greedy) {
    border = top, ties = 1;
  } else {
    if (top_k > 0 && top_k < V) {
      for (int bit = 31; bit >= 0; --bit)
        if (above(border | 1u << bit).n >= top_k) border |= 1u << bit;
      ties = top_k - (border == 0xffffffffu ? 0 : above(border + 1).n);
    }
    if (top_p < 1.f) {
      const uint32_t k_border = border;
      const long long k_ties = ties;
      const float bl = __uint_as_float((k_border & 0x80000000u) ? k_border ^ 0x80000000u : ~k_border);
      const bool cut = top_k > 0 && top_k < V;
      const double wk = cut ? weight(bl) : 0.0;
      const double sum = cut ? above(k_border + 1).w + static_cast<double>(k_ties) * wk : above(0).w;
      const double need = fmax(static_cast<double>(top_p), 0.0) * sum;
      uint32_t p = 0u;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t k = p | 1u << bit;
        if (k > k_border || !cut) {
          if (above(k).w >= need) p = k;
        } else {
          p = k;  // all that top_k kept is at or above its border
        }
      }
      if (p > top) p = top;
      const double over = above(p + 1).w;
      const double w = weight(__uint_as_float((p & 0x80000000u) ? p ^ 0x80000000u : ~p));
      long long n = need > over && w > 0.0 ? static_cast<long long>(fmin(ceil((need - over) / w), 4.0e9)) : 0;
      if (p == top && n < 1) n = 1;
      if (p != k_border || !cut || n < k_ties) ties = n;
      border = p;
    }
  }
  if (min_p > 1.f) border = top, ties = 1;
  const double floor_w = min_p > 0.f && min_p <= 1.f && !greedy ? static_cast<double>(min_p) : 0.0;

  // the last kept index of the border's ties, then the draw: threads own contiguous ranges, so their order is the indices'
  const int share = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, tid * share), i1 = min(V, i0 + share);
  Pair eq{0.0, 0};
  for (int i = i0; i < i1; ++i) eq.n += key_of(logit<DT>(row, i)) == border;
  long long left = ties - block_before(eq, part).n;
  auto kept = [&](float l, long long& ties_left) {
    const uint32_t k = key_of(l);
    if (k < border) return 0.0;
    if (k == border && ties_left-- <= 0) return 0.0;
    const double w = greedy ? 1.0 : weight(l);
    return w >= floor_w ? w : 0.0;
  };
  Pair mine{0.0, 0};
  long long lt = left;
  for (int i = i0; i < i1; ++i) mine.w += kept(logit<DT>(row, i), lt);
  const Pair before = block_before(mine, part);
  const double total = block_sum(mine, part).w;
  const double target = u * total;
  double run = before.w;
  lt = left;
  for (int i = i0; i < i1; ++i) {
    const double w = kept(logit<DT>(row, i), lt);
    run += w;
    if (w > 0.0 && run > target) {
      atomicMin(&s_idx, i);
      break;
    }
  }
  __syncthreads();
  if (tid == 0) {
    const int i = s_idx;
    a.tokens[r] = i;
    if (a.logprob != nullptr) a.logprob[r] = static_cast<float>(greedy ? 0.0 : log(weight(logit<DT>(row, i)) / total));
  }
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
  if (x->B < 0 || x->V < 0 || x->V > (1 << 30)) return fail(MV_ERR_INVALID, "%s: bad B=%d / V=%d", who, x->B, x->V);
  if (x->B == 0) return MV_OK;
  if (x->u == nullptr || x->tokens == nullptr || (x->V > 0 && x->logits == nullptr))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (x->B > 1 && x->st < 0) return fail(MV_ERR_INVALID, "%s: negative row stride %lld", who, x->st);
  SampleArgs a{x->logits, x->u, x->temperature, x->top_p, x->min_p, x->top_k, x->tokens, x->logprob, x->st,
               x->temperature_value, x->top_p_value, x->min_p_value, x->top_k_value, x->V};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto fn = x->dtype == MV_F32 ? sample_kernel<MV_F32> : x->dtype == MV_BF16 ? sample_kernel<MV_BF16> : sample_kernel<MV_F16>;
  return attn::launch_pdl(fn, dim3(x->B), kThreads, 0, st, "mv_sample launch", a);
}
