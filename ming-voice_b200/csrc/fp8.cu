// Products with 8-bit floating-point weights and a scale for each block of 128 (mv_fp8_linear; the products are in fp8_gemm.cu), and
// the rounding of activations and weights to that form (mv_quantize_fp8, mv_quantize_fp8_weight).
//
// An activation block's scale is a power of two: x / scale is exact, so the rounded values do not depend on how the quotient is
// taken, and an e4m3 number has as many significant bits at any power of two (down to 2^-6 of 448). Bound: memory; 16001 x 2048 in 19.6
// us, 5.0 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "attn_common.cuh"
#include "common.cuh"
#include "fp8.cuh"

namespace mv {
namespace fp8 {
namespace {

// ---------------------------------------------------------------------------------------------- rounding

// Activations: a half warp owns a token's block of 128 columns, 8 values a lane. VEC: values of one load (16, 8 or 4 bytes of
// a 16-bit type), by the alignment of the rows. Scales as fp32 numbers, or as their exponents' bytes: a block that is not finite
// has NaNs among its rounded values, so the products are NaN whatever its exponent says. Bound: memory.
// UNITS: blocks of a CTA, 16 or 64; of 64 a thread takes four, 16 apart, whose loads are under way together (16001 x 2048: 19.6 us
// against 22.1; 300 x 2048, where it leaves SMs idle: 2.1 against 1.8).
template <int DT, int VEC, typename S, int UNITS>
__global__ void __launch_bounds__(256) quantize_kernel(const void* __restrict__ x, long long x_st, int T, int K, int blocks,
                                                       uint8_t* __restrict__ q, long long q_st, S* __restrict__ scale,
                                                       long long s_st) {
  pdl_wait();
  // where this is a product's first half, its second may be scheduled
  if (sizeof(S) == 1) pdl_launch_dependents();
  const int sub = threadIdx.x & 15;
  const long long first = static_cast<long long>(blockIdx.x) * UNITS;
  const int t0 = static_cast<int>(first / blocks), b0 = static_cast<int>(first % blocks);
  float v[UNITS / 16][8];
  int ts[UNITS / 16], bs[UNITS / 16];
#pragma unroll
  for (int i = 0; i < UNITS / 16; ++i) {
    const int at = b0 + i * 16 + (threadIdx.x >> 4);
    ts[i] = t0 + at / blocks, bs[i] = at % blocks;
    load8<DT, VEC>(x, min(ts[i], T - 1) * x_st, bs[i] * kBlock + sub * 8, ts[i] < T ? K : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < UNITS / 16; ++i) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[i][k]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    float up, down;
    block_scale(top, up, down);
    if (ts[i] >= T) continue;
    *reinterpret_cast<uint2*>(q + ts[i] * q_st + bs[i] * kBlock + sub * 8) = round8(v[i], down);
    if (sub == 0) {
      if constexpr (sizeof(S) == 1)
        scale[bs[i] * s_st + ts[i]] = static_cast<uint8_t>(__float_as_uint(up) >> 23);
      else
        scale[bs[i] * s_st + ts[i]] = up;
    }
  }
}

// Weights: a CTA owns a block of 128 x 128. Done once for a model, so by single elements: 131072 x 2048 bf16 in 521 us, 1.5 TB/s.
template <int DT>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const void* __restrict__ w, long long w_st, int N, int K,
                                                              uint8_t* __restrict__ q, long long q_st,
                                                              float* __restrict__ scale, long long s_st) {
  __shared__ float part[8];
  const int k0 = blockIdx.x * kBlock, n0 = blockIdx.y * kBlock;
  const int rows = min(kBlock, N - n0), cols = min(kBlock, K - k0);
  float top = 0.f;
  bool nan = false;
  for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
    const int r = i / kBlock, c = i % kBlock;
    if (r >= rows || c >= cols) continue;
    const float v = fabsf(load1<DT>(w, (n0 + r) * w_st + k0 + c));
    nan |= !(v <= FLT_MAX);
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  const bool any_nan = __syncthreads_or(nan);
  top = part[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, part[i]);
  const float s = fmaxf(__fdiv_rn(top, 448.f), 7.888609052210118e-31f);  // 2^-100
  if (threadIdx.x == 0) scale[blockIdx.y * s_st + blockIdx.x] = any_nan ? __int_as_float(0x7fc00000) : s;
  for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
    const int r = i / kBlock, c = i % kBlock;
    if (r >= rows || c >= cols) continue;
    q[(n0 + r) * q_st + k0 + c] = static_cast<uint8_t>(e4m3x2(__fdiv_rn(load1<DT>(w, (n0 + r) * w_st + k0 + c), s), 0.f) & 0xff);
  }
}

template <int DT, typename S>
int launch_quantize(const void* x, long long x_st, int T, int K, uint8_t* q, long long q_st, S* scale, long long s_st,
                    cudaStream_t st) {
  const int blocks = (K + kBlock - 1) / kBlock;
  const long long units = static_cast<long long>(T) * blocks;
  const int per_cta = units >= 64LL * 8 * num_sms() ? 64 : 16;
  const long long ctas = (units + per_cta - 1) / per_cta;
  if (ctas > 0x7fffffffLL) return fail(MV_ERR_INVALID, "mv_quantize_fp8: T=%d x K=%d is too large", T, K);
  const int size = DT == MV_F32 ? 4 : 2;
  const uintptr_t step = reinterpret_cast<uintptr_t>(x) | (T > 1 ? static_cast<uintptr_t>(x_st) * size : 0);
  auto fn = per_cta == 64 ? quantize_kernel<DT, 1, S, 64> : quantize_kernel<DT, 1, S, 16>;
  if (step % 16 == 0 && K % 8 == 0)
    fn = per_cta == 64 ? quantize_kernel<DT, 8, S, 64> : quantize_kernel<DT, 8, S, 16>;
  else if (step % 8 == 0 && K % 4 == 0 && DT != MV_F32)
    fn = per_cta == 64 ? quantize_kernel<DT, 4, S, 64> : quantize_kernel<DT, 4, S, 16>;
  return attn::launch_pdl(fn, dim3(static_cast<unsigned int>(ctas)), 256, 0, st, "mv_quantize_fp8 launch", x, x_st, T, K, blocks,
                          q, q_st, scale, s_st);
}

template <typename S>
int quantize(const void* x, int dtype, long long x_st, int T, int K, uint8_t* q, long long q_st, S* scale, long long s_st,
             cudaStream_t st) {
  if (dtype == MV_BF16) return launch_quantize<MV_BF16>(x, x_st, T, K, q, q_st, scale, s_st, st);
  if (dtype == MV_F16) return launch_quantize<MV_F16>(x, x_st, T, K, q, q_st, scale, s_st, st);
  return launch_quantize<MV_F32>(x, x_st, T, K, q, q_st, scale, s_st, st);
}

// whether two [rows, cols] tensors (row strides and widths in bytes) have a byte in common; columns of one buffer side by side
// have none
bool overlap(const void* p, long long p_st, long long p_w, const void* q, long long q_st, long long q_w, int rows) {
  const long long a = static_cast<long long>(reinterpret_cast<uintptr_t>(p)), b = static_cast<long long>(reinterpret_cast<uintptr_t>(q));
  if (a + (rows - 1) * p_st + p_w <= b || b + (rows - 1) * q_st + q_w <= a) return false;
  if (rows < 2 || p_st != q_st || p_st <= 0) return true;
  const long long d = ((b - a) % p_st + p_st) % p_st;
  return d < p_w || d + q_w > p_st;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace fp8
}  // namespace mv

using namespace mv;
using namespace mv::fp8;

extern "C" int mv_quantize_fp8(const void* x, int x_dtype, long long x_st, int T, int K, void* q, long long q_st, float* scale,
                               long long s_st, void* stream) {
  const char* who = "mv_quantize_fp8";
  if (T < 0 || K < 0) return fail(MV_ERR_INVALID, "%s: bad T=%d / K=%d", who, T, K);
  if (x_dtype != MV_BF16 && x_dtype != MV_F16 && x_dtype != MV_F32)
    return fail(MV_ERR_UNSUPPORTED, "%s: x must be bf16, f16 or f32", who);
  if (T == 0 || K == 0) return MV_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (reinterpret_cast<uintptr_t>(x) % (x_dtype == MV_F32 ? 4 : 2) != 0 || !aligned16(q) || q_st % 16 != 0)
    return fail(MV_ERR_ALIGN, "%s: q must be 16-byte aligned with rows of whole 16 bytes", who);
  if ((T > 1 && x_st < 0) || q_st < (static_cast<long long>(K) + kBlock - 1) / kBlock * kBlock || s_st < T)
    return fail(MV_ERR_INVALID, "%s: a row stride is too short for T=%d, K=%d", who, T, K);
  return quantize(x, x_dtype, x_st, T, K, static_cast<uint8_t*>(q), q_st, scale, s_st, static_cast<cudaStream_t>(stream));
}

extern "C" int mv_quantize_fp8_weight(const void* w, int w_dtype, long long w_st, int N, int K, void* q, long long q_st,
                                      float* scale, long long s_st, void* stream) {
  const char* who = "mv_quantize_fp8_weight";
  if (N < 0 || K < 0 || N > 65535 * kBlock) return fail(MV_ERR_INVALID, "%s: bad N=%d / K=%d", who, N, K);
  if (w_dtype != MV_BF16 && w_dtype != MV_F16 && w_dtype != MV_F32)
    return fail(MV_ERR_UNSUPPORTED, "%s: w must be bf16, f16 or f32", who);
  if (N == 0 || K == 0) return MV_OK;
  if (w == nullptr || q == nullptr || scale == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const int kb = (K + kBlock - 1) / kBlock, nb = (N + kBlock - 1) / kBlock;
  if ((N > 1 && (w_st < K || q_st < K)) || (nb > 1 && s_st < kb))
    return fail(MV_ERR_INVALID, "%s: a row stride is too short for N=%d, K=%d", who, N, K);
  auto fn = w_dtype == MV_F32 ? quantize_weight_kernel<MV_F32>
            : w_dtype == MV_F16 ? quantize_weight_kernel<MV_F16>
                                : quantize_weight_kernel<MV_BF16>;
  fn<<<dim3(kb, nb), 256, 0, static_cast<cudaStream_t>(stream)>>>(w, w_st, N, K, static_cast<uint8_t*>(q), q_st, scale, s_st);
  return cuda_status(cudaGetLastError(), "mv_quantize_fp8_weight launch");
}

extern "C" size_t mv_fp8_linear_scratch_bytes(int T, int N, int K) {
  if (T <= 0 || K <= 0) return 0;
  const size_t blocks = (static_cast<size_t>(K) + kBlock - 1) / kBlock;
  LinearArgs a{};
  a.T = T, a.N = N, a.K = K, a.blocks = static_cast<int>(blocks);
  if (one_launch(a)) return 0;
  return align256(static_cast<size_t>(T) * blocks * kBlock) + align256(blocks * scale_stride(T));
}

extern "C" int mv_fp8_linear(const mv_fp8_linear_args* x, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "mv_fp8_linear";
  if (x == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const int T = x->T, N = x->N, K = x->K;
  if (T < 0 || N < 0 || K < 1) return fail(MV_ERR_INVALID, "%s: bad T=%d / N=%d / K=%d", who, T, N, K);
  if (x->x_dtype != MV_BF16 && x->x_dtype != MV_F16) return fail(MV_ERR_UNSUPPORTED, "%s: x must be bf16 or f16", who);
  if (x->out_dtype != MV_BF16 && x->out_dtype != MV_F16 && x->out_dtype != MV_F32)
    return fail(MV_ERR_UNSUPPORTED, "%s: the result must be bf16, f16 or f32", who);
  if (T == 0 || N == 0) return MV_OK;
  if (x->x == nullptr || x->wq == nullptr || x->ws == nullptr || x->out == nullptr)
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const long long blocks = (static_cast<long long>(K) + kBlock - 1) / kBlock;
  if ((T > 1 && (x->x_st < 0 || x->o_st < N || (x->residual != nullptr && x->r_st < 0))) || (N > 1 && x->w_st < K) ||
      (N > kBlock && x->ws_st < blocks))
    return fail(MV_ERR_INVALID, "%s: a row stride is too short for T=%d, N=%d, K=%d", who, T, N, K);
  if (!aligned16(x->wq) || (N > 1 && x->w_st % 16 != 0))
    return fail(MV_ERR_ALIGN, "%s: wq must be 16-byte aligned with rows of whole 16 bytes", who);
  const int size = elem_size(x->out_dtype);
  if (overlap(x->out, x->o_st * size, static_cast<long long>(N) * size, x->x, x->x_st * 2, K * 2LL, T))
    return fail(MV_ERR_INVALID, "%s: out overlaps x", who);
  if (x->residual != nullptr && !(x->residual == x->out && (T == 1 || x->r_st == x->o_st)) &&
      overlap(x->out, x->o_st * size, static_cast<long long>(N) * size, x->residual, x->r_st * size, static_cast<long long>(N) * size, T))
    return fail(MV_ERR_INVALID, "%s: residual overlaps out without being it", who);
  if (workspace == nullptr || workspace_bytes < kWsHeaderBytes)
    return fail(MV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, kWsHeaderBytes);
  const size_t scratch_bytes = mv_fp8_linear_scratch_bytes(T, N, K);
  if (scratch_bytes > 0 && (x->scratch == nullptr || x->scratch_bytes < scratch_bytes ||
                            (reinterpret_cast<uintptr_t>(x->scratch) & 255u)))
    return fail(MV_ERR_WORKSPACE, "%s: 256-byte aligned scratch of %zu bytes needed", who, scratch_bytes);
  LinearArgs a{};
  a.q_st = blocks * kBlock, a.s_st = scale_stride(T), a.blocks = static_cast<int>(blocks);
  uint8_t* scratch = static_cast<uint8_t*>(x->scratch);
  a.q = scratch, a.scale = scratch + align256(static_cast<size_t>(T) * a.q_st);
  a.w = static_cast<const uint8_t*>(x->wq), a.w_st = N > 1 ? x->w_st : a.q_st, a.ws = x->ws, a.ws_st = x->ws_st;
  a.residual = x->residual, a.r_st = x->r_st, a.out = x->out, a.o_st = x->o_st;
  a.T = T, a.N = N, a.K = K, a.header = static_cast<WsHeader*>(workspace);
  a.x = x->x, a.x_st = T > 1 ? x->x_st : 0, a.x_dtype = x->x_dtype;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (one_launch(a)) return run_product(a, x->out_dtype, st);
  const int rc = quantize(x->x, x->x_dtype, x->x_st, T, K, a.q, a.q_st, a.scale, a.s_st, st);
  if (rc != MV_OK) return rc;
  return run_product(a, x->out_dtype, st);
}
