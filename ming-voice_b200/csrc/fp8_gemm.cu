// The products of mv_fp8_linear on the 5th-generation tensor cores.
//
// y[t, n] = sum_b sx[t, b] ws[n / 128, b] * (q[t, block b] . w[n, block b]). The tensor cores give one block's product at a
// time in TMEM (kind::f8f6f4, 128 values of K: four instructions); the epilogue warps read it while the next block runs in the
// other buffer, and add it in fp32 registers with its factor. Two forms of the same pipeline (TMA warp, issuing warp, epilogue
// warps; a ring of stages with one weight tile and one activation tile each):
//   few tokens  weights are the 128-row operand and up to 128 tokens the columns, so a tile is a weight stream of 16 KB
//               blocks; a cluster shares a tile's blocks of K where there are fewer tiles than SMs and adds the parts over
//               distributed shared memory in rank order.
//   many tokens 256 tokens are the rows and 256 weight rows the columns of a pair of CTAs: an epilogue thread owns one token, so
//               a block's factor is one number per thread.
// Bound and measured (B200; graph replays): few tokens by the weights' bytes, 131072 x 2048 for one token 50 us (5.4 TB/s, 83 % of the
// measured copy; the rest is the start of 4 us and the last wave of tiles), for 64 tokens 65 us; many tokens by the tensor pipe
// and the hand-over of each block between it and the epilogue, 16001 x 5632 x 2048 195 to 203 us by card with the
// activations' rounding (1.82 to 1.89 PFLOP/s), 4096 x 5632 x 8192 178 to 185 (2.0 to 2.1; products added up in TMEM instead, which one
// scale a row would allow, take 148).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "attn_common.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "tc.cuh"

namespace mv {
namespace fp8 {
namespace {

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 operands, fp32 accumulation, 32 values of K; issued by one thread.
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), both operands e4m3 (0) and K-major, N >> 3 (17-22), M >> 4 (24-28)
constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// the 16-byte aligned 1-D copy that brings a block's activation scales along with its tiles
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 32 lanes x 64 consecutive 32-bit columns
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, "
      "%42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr));
}

// the exponent byte `i` of `w` as a power of two
__device__ __forceinline__ float power(uint32_t w, int i) { return __uint_as_float((w >> (8 * i) & 0xffu) << 23); }

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 16)
    tc::tmem_ld16(addr, r);
  else
    tc::tmem_ld32(addr, r);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// four values at shared address `addr` of the cluster's CTA `rank`
__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// mbar_wait inline: a call would save the epilogue's 128 sums around it
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, WsHeader* h, unsigned int info) {
  uint64_t t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    const uint64_t now = globaltimer_ns();  // (reading it takes longer than most waits)
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      raise_error(h, kErrTimeout, info);
      return false;
    }
  }
}

// the loads into d have landed: what uses d comes behind it for the compiler too
__device__ __forceinline__ void landed(uint32_t (&d)[64]) {
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 64; i += 16)
    asm volatile("" : "+r"(d[i + 0]), "+r"(d[i + 1]), "+r"(d[i + 2]), "+r"(d[i + 3]), "+r"(d[i + 4]), "+r"(d[i + 5]), "+r"(d[i + 6]), "+r"(d[i + 7]), "+r"(d[i + 8]), "+r"(d[i + 9]), "+r"(d[i + 10]), "+r"(d[i + 11]), "+r"(d[i + 12]), "+r"(d[i + 13]), "+r"(d[i + 14]), "+r"(d[i + 15]) : : "memory");
}

constexpr size_t kMostSmem = 226 * 1024;       // dynamic shared memory of a CTA, beside the barriers
constexpr int kTile = 128;                     // rows of the 128-row operand
constexpr uint32_t kTileBytes = kTile * kBlock;  // 16 KB

// ------------------------------------------------------------------------------------------------ few tokens

struct FewArgs {
  const float* ws;
  const uint8_t* scale;
  const void* residual;
  void* out;
  long long ws_st, s_st, r_st, o_st;
  int T, N, blocks, n_tiles, t_tiles, split;
  bool x_bf16;                // type of the activations that the kernel rounds itself
  bool out_lines, res_lines;  // whole lines of `out` and `residual` go through their tensor maps
  WsHeader* header;
};

// Adds the parts [cols][128] of a cluster's CTAs in rank order, each CTA a share of the columns; the loads of all parts are under way
// together (one after another they took 64 x 2048 x 2048 14.5 us).
template <int ODT>
__device__ __forceinline__ void join_parts(const FewArgs& a, uint32_t part, int n0, int t0, int cols, int rank, int threads) {
  for (int i = (threadIdx.x + rank * threads) * 4; i < cols * kTile; i += threads * a.split * 4) {
    const int t = t0 + i / kTile, n = n0 + i % kTile;
    float4 p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < a.split) p[r] = ld_peer(part + i * 4, r);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < a.split) v[0] += p[r].x, v[1] += p[r].y, v[2] += p[r].z, v[3] += p[r].w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k >= a.N) break;
      if (a.residual != nullptr) v[k] += load1<ODT>(a.residual, t * a.r_st + n + k);
      store1<ODT>(a.out, t * a.o_st + n + k, v[k]);
    }
  }
}

// NT token columns of a tile. Stage: weight tile, activation tile, activation scales.
template <int NT>
struct Few {
  static constexpr int kStages = NT <= 32 ? 9 : NT == 64 ? 8 : 6;
  static constexpr uint32_t kXBytes = NT * kBlock;
  static constexpr uint32_t kStageBytes = kTileBytes + kXBytes;
  static constexpr int kHalves = NT >= 64 ? 2 : 1;  // epilogue warps per 32 rows
  static constexpr int kCols = NT / kHalves;         // columns of an epilogue thread
  static constexpr int kThreads = 64 + 128 * kHalves;
  static constexpr int kBufs = NT == 128 ? 4 : 8;    // blocks' products in TMEM
  static constexpr uint32_t kTmemCols = kBufs * NT;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kStages) * (kStageBytes + NT);
};

template <int NT, int ODT>
__global__ void __launch_bounds__(Few<NT>::kThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const FewArgs a) {
  using F = Few<NT>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* scales = smem + F::kStages * F::kStageBytes;  // [stage][NT]
  __shared__ alignas(8) uint64_t full[F::kStages], empty[F::kStages], acc_full[F::kBufs], acc_empty[F::kBufs];
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kEpiWarps = 4 * F::kHalves;
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1 + kEpiWarps);
    for (int i = 0; i < F::kBufs; ++i) mbar_init(&acc_full[i], 2), mbar_init(&acc_empty[i], kEpiWarps);
    fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem_base, F::kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int first = blockIdx.x / a.split, step = gridDim.x / a.split;
  const int tiles = a.n_tiles * a.t_tiles;
  // the cluster's CTAs take equal contiguous shares of the blocks of K
  const int b0 = a.blocks * rank / a.split, b1 = a.blocks * (rank + 1) / a.split;
  pdl_launch_dependents();

  if (warp == 0) {
    if (tc::elect_one()) {
      tc::prefetch_tmap(&wmap);
      tc::prefetch_tmap(&xmap);
      pdl_wait();
      int it = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        const int n0 = tile / a.t_tiles * kTile, t0 = tile % a.t_tiles * NT;
        const uint32_t sb = static_cast<uint32_t>(min(static_cast<long long>(NT), a.s_st - t0));
        for (int b = b0; b < b1; ++b, ++it) {
          const int s = it % F::kStages;
          if (it >= F::kStages && !wait(&empty[s], (it / F::kStages + 1) & 1, a.header, 0x800u)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * F::kStageBytes;
          mbar_arrive_expect_tx(&full[s], F::kStageBytes + sb);
          tc::tma_load_2d(st, &wmap, &full[s], b * kBlock, n0);
          tc::tma_load_2d(st + kTileBytes, &xmap, &full[s], b * kBlock, t0);
          bulk_load(scales + s * NT, a.scale + b * a.s_st + t0, sb, &full[s]);
        }
      }
    }
  } else if (warp == 1) {
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += step) {
      for (int b = b0; b < b1; ++b, ++it) {
        const int s = it % F::kStages, buf = it % F::kBufs;
        if (!wait(&full[s], (it / F::kStages) & 1, a.header, 0x801u) ||
            (it >= F::kBufs && !wait(&acc_empty[buf], (it / F::kBufs + 1) & 1, a.header, 0x802u))) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        if (tc::elect_one()) {
          const uint32_t base = smem_u32(smem + s * F::kStageBytes);
          const uint64_t ad = tc::sw128_desc(base), bd = tc::sw128_desc(base + kTileBytes);
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k) mma_f8(tmem + buf * NT, ad + 2 * k, bd + 2 * k, idesc_e4m3(kTile, NT), k > 0);
          tc::mma_commit(&empty[s]);
          tc::mma_commit(&acc_full[buf]);
          // The epilogue reads the stage's scales, and a commit hands on nothing but its products: this thread, which has waited for
          // the copies, arrives too (a wait of each epilogue warp for the copies took 61 x 100277 x 1500 3 us).
          mbar_arrive(&acc_full[buf]);
        }
        __syncwarp();
      }
    }
  } else {
    const int e = warp - 2, quarter = warp & 3, c0 = e / 4 * F::kCols;  // the warp reads TMEM lanes 32 * quarter ..
    const int row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c0;
    pdl_wait();
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < tiles; tile += step) {
      const int n0 = tile / a.t_tiles * kTile, t0 = tile % a.t_tiles * NT;
      float acc[F::kCols];
#pragma unroll
      for (int c = 0; c < F::kCols; ++c) acc[c] = 0.f;
      const float* ws = a.ws + n0 / kBlock * a.ws_st;
      float w_next = b0 < b1 ? ws[b0] : 0.f;
      for (int b = b0; b < b1 && ok; ++b, ++it) {
        const int s = it % F::kStages, buf = it % F::kBufs;
        const float w = w_next;
        if (b + 1 < b1) w_next = ws[b + 1];
        if (!wait(&acc_full[buf], (it / F::kBufs) & 1, a.header, 0x803u)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        constexpr int kLd = F::kCols < 32 ? 16 : 32;
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(scales + s * NT + c0);
#pragma unroll
        for (int c = 0; c < F::kCols; c += kLd) {
          uint32_t d[kLd];
          tmem_load<kLd>(lanes + buf * NT + c, d);
          tc::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < kLd; i += 4) {
            const uint32_t f = sc[(c + i) / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[c + i + k] = fmaf(__uint_as_float(d[i + k]), power(f, k) * w, acc[c + i + k]);
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&acc_empty[buf]);
          mbar_arrive(&empty[s]);
        }
      }
      const int n = n0 + row;
      if (a.split == 1) {
        if (n < a.N && ok) {
#pragma unroll
          for (int c = 0; c < F::kCols; ++c) {
            const int t = t0 + c0 + c;
            if (t >= a.T) break;
            float v = acc[c];
            if (a.residual != nullptr) v += load1<ODT>(a.residual, t * a.r_st + n);
            store1<ODT>(a.out, t * a.o_st + n, v);
          }
        }
      } else {
        // the parts lie where the ring was: its copies have landed and its products are done
        float* part = reinterpret_cast<float*>(smem);  // [NT][128]
        named_bar(1, 128 * F::kHalves);
#pragma unroll
        for (int c = 0; c < F::kCols; ++c) part[(c0 + c) * kTile + row] = acc[c];
      }
    }
  }
  if (a.split > 1) {
    __syncwarp();
    pdl_wait();
    cluster_sync();
    const int tile = first;
    join_parts<ODT>(a, smem_u32(smem), tile / a.t_tiles * kTile, tile % a.t_tiles * NT, min(NT, a.T - tile % a.t_tiles * NT), rank,
                    F::kThreads);
    cluster_sync();
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, F::kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------ a few tokens, few rows
//
// The same with the activations rounded by the epilogue warps while the first weights are on their way: one launch, and no
// activation traffic in the ring. All blocks of a CTA's share of K lie in shared memory; a cluster has one tile (one_launch).

constexpr int kTokenN = 16, kTokenBlocks = 32, kTokenStages = 12;
constexpr int kTokenBufs = 8;  // blocks' products in TMEM: the issuing warp does not wait for the epilogue of the last two
constexpr uint32_t kTokenXBytes = kTokenN * kBlock;  // of a block

inline size_t token_smem(int blocks, int stages) {
  return 1024 + static_cast<size_t>(stages) * kTileBytes + static_cast<size_t>(blocks) * (kTokenXBytes + kTokenN * 4);
}

struct TokenArgs {
  FewArgs f;
  const void* x;
  long long x_st;
  int K, stages, vec;
};

template <int XDT, int VEC>
__device__ __forceinline__ void round_tokens(const TokenArgs& a, int b0, int b1, uint8_t* xs, float* scales, int tid) {
  // a half warp has a token's block; eight blocks at a time are under way
  const int sub = tid & 15, units = (b1 - b0) * a.f.T;
  constexpr int kDeep = 4;
  for (int u0 = tid >> 4; u0 < units + (tid >> 4); u0 += 8 * kDeep) {
    float v[kDeep][8];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int u = u0 + 8 * i, b = u / a.f.T, t = u % a.f.T;
      load8<XDT, VEC>(a.x, t * a.x_st, (b0 + b) * kBlock + sub * 8, u < units ? a.K : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int u = u0 + 8 * i, b = u / a.f.T, t = u % a.f.T;
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[i][k]) & 0x7fffffffu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      float up, down;
      block_scale(top, up, down);
      if (u >= units) continue;
      // the 128-byte swizzle of the operand's layout: 16-byte piece j of row t at j ^ (t & 7)
      *reinterpret_cast<uint2*>(xs + b * kTokenXBytes + t * kBlock + (((sub >> 1) ^ (t & 7)) << 4) + (sub & 1) * 8) =
          round8(v[i], down);
      if (sub == 0) scales[b * kTokenN + t] = up;
    }
  }
}

template <int ODT>
__global__ void __launch_bounds__(192, 1) token_kernel(const __grid_constant__ CUtensorMap wmap, const TokenArgs g) {
  const FewArgs& a = g.f;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int rank = static_cast<int>(cluster_rank());
  const int b0 = a.blocks * rank / a.split, b1 = a.blocks * (rank + 1) / a.split;
  uint8_t* xs = smem + g.stages * kTileBytes;                                     // [block][token][128], swizzled
  float* scales = reinterpret_cast<float*>(xs + (b1 - b0) * kTokenXBytes);        // [block][token]
  __shared__ alignas(8) uint64_t full[kTokenStages], empty[kTokenStages], acc_full[kTokenBufs], acc_empty[kTokenBufs], x_full;
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < kTokenBufs; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 4);
    mbar_init(&x_full, 4);
    fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem_base, kTokenBufs * kTokenN);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int tile = blockIdx.x / a.split;
  pdl_launch_dependents();

  if (warp == 0) {
    if (tc::elect_one()) {
      tc::prefetch_tmap(&wmap);
      // weights too: the kernel in front may be what writes them (their copies ahead of the wait save 0.02 of 5.4 us)
      pdl_wait();
      for (int b = b0, it = 0; b < b1; ++b, ++it) {
        const int s = it % g.stages;
        if (it >= g.stages && !wait(&empty[s], (it / g.stages + 1) & 1, a.header, 0x820u)) break;
        mbar_arrive_expect_tx(&full[s], kTileBytes);
        tc::tma_load_2d(smem + s * kTileBytes, &wmap, &full[s], b * kBlock, tile * kTile);
      }
    }
  } else if (warp == 1) {
    const bool rounded = wait(&x_full, 0, a.header, 0x824u);
    for (int b = b0, it = 0; b < b1 && rounded; ++b, ++it) {
      const int s = it % g.stages, buf = it % kTokenBufs;
      if (!wait(&full[s], (it / g.stages) & 1, a.header, 0x821u) ||
          (it >= kTokenBufs && !wait(&acc_empty[buf], (it / kTokenBufs + 1) & 1, a.header, 0x822u)))
        break;
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint64_t ad = tc::sw128_desc(smem_u32(smem + s * kTileBytes));
        const uint64_t bd = tc::sw128_desc(smem_u32(xs + (b - b0) * kTokenXBytes));
#pragma unroll
        for (int k = 0; k < kBlock / 32; ++k)
          mma_f8(tmem + buf * kTokenN, ad + 2 * k, bd + 2 * k, idesc_e4m3(kTile, kTokenN), k > 0);
        tc::mma_commit(&empty[s]);
        tc::mma_commit(&acc_full[buf]);
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3, row = quarter * 32 + lane, tid = threadIdx.x - 64;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    pdl_wait();
    if (g.vec == 8)
      g.f.x_bf16 ? round_tokens<MV_BF16, 8>(g, b0, b1, xs, scales, tid) : round_tokens<MV_F16, 8>(g, b0, b1, xs, scales, tid);
    else
      g.f.x_bf16 ? round_tokens<MV_BF16, 1>(g, b0, b1, xs, scales, tid) : round_tokens<MV_F16, 1>(g, b0, b1, xs, scales, tid);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&x_full);
    named_bar(1, 128);  // the scales of all four warps
    float acc[kTokenN];
#pragma unroll
    for (int c = 0; c < kTokenN; ++c) acc[c] = 0.f;
    // lane l: the weights' scale of block b0 + l
    const float ws_lane = b0 + lane < b1 ? a.ws[tile * a.ws_st + b0 + lane] : 0.f;
    for (int b = b0, it = 0; b < b1; ++b, ++it) {
      const int buf = it % kTokenBufs;
      const float w = __shfl_sync(0xffffffffu, ws_lane, b - b0);
      if (!wait(&acc_full[buf], (it / kTokenBufs) & 1, a.header, 0x823u)) break;
      tc::fence_after_sync();
      uint32_t d[kTokenN];
      tc::tmem_ld16(lanes + buf * kTokenN, d);
      tc::tmem_ld_wait();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
      const float4* sc = reinterpret_cast<const float4*>(scales + (b - b0) * kTokenN);
#pragma unroll
      for (int i = 0; i < kTokenN; i += 4) {
        if (i >= a.T) break;
        const float4 f = sc[i / 4];
        acc[i] = fmaf(__uint_as_float(d[i]), f.x * w, acc[i]);
        acc[i + 1] = fmaf(__uint_as_float(d[i + 1]), f.y * w, acc[i + 1]);
        acc[i + 2] = fmaf(__uint_as_float(d[i + 2]), f.z * w, acc[i + 2]);
        acc[i + 3] = fmaf(__uint_as_float(d[i + 3]), f.w * w, acc[i + 3]);
      }
    }
    // the parts lie where the ring was: its copies have landed and its products are done
    float* part = reinterpret_cast<float*>(smem);  // [token][128]
    named_bar(1, 128);
#pragma unroll
    for (int t = 0; t < kTokenN; ++t) part[t * kTile + row] = acc[t];
  }
  pdl_wait();
  cluster_sync();
  join_parts<ODT>(a, smem_u32(smem), tile * kTile, 0, a.T, rank, 192);
  cluster_sync();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTokenBufs * kTokenN);
  }
}

// ------------------------------------------------------------------------------------------------ many tokens
//
// Two CTAs of a cluster work on one tile of 256 tokens x 256 weight rows (cta_group::2): each brings 128 rows of either
// operand, 32 KB a block instead of 48, and holds the products of its 128 tokens (16001 x 5632 x 2048: 222 us with one CTA's tiles of 128 x
// 256, 195 with pairs). The products of a block's 256 columns are handed over together: halves of 128, four buffers instead
// of two, took 253 us, since a hand-over costs more than the reads behind it. The pair's epilogue frees a buffer by a plain arrive
// on the first CTA's barrier: with .release.cluster, which waits for all earlier memory operations, it took 394 us.

constexpr int kManyStages = 5, kManyN = 256, kManyT = 256;
constexpr uint32_t kManyStageBytes = 2 * kTileBytes;  // 32 KB
constexpr uint32_t kLineBytes = 32 * 128;             // 32 rows of a warp's staging, two of these per warp
// A slot of scales is written when the products five blocks back are done, so the epilogue is done with those seven back.
constexpr int kScaleSlots = 8;
constexpr size_t kManySmem = 1024 + kManyStages * kManyStageBytes + 8 * 2 * kLineBytes + kScaleSlots * 128;
constexpr int kManyThreads = 128 + 256;

__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}

// a tile into this CTA's shared memory, counted on the barrier at cluster address `bar`
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// arrives on `bar` in both CTAs when the products issued so far are done
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}

// 32 rows of 128 bytes from shared memory to (x, y) of a tensor; what lies outside it is left out
__device__ __forceinline__ void store_lines(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// all but the last N stores have been read from shared memory
template <int N>
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// 16 bytes of a warp's staging: 32 rows of 128 bytes, chunk j of row r at j ^ (r & 7), so that both a row per lane and a
// line per 8 lanes are without bank conflicts
__device__ __forceinline__ uint4* staged(uint8_t* buf, int r, int j) {
  return reinterpret_cast<uint4*>(buf + r * 128 + ((j ^ (r & 7)) * 16));
}

// Moves 32 rows x 128 bytes between the staging and global memory, whole lines at a time where rows start at 16-byte addresses
// (aligned), else an element per lane. `rows` and `cols`: what lies inside the tensor.
template <int SIZE, bool STORE>
__device__ __forceinline__ void move_lines(uint8_t* buf, void* global, long long stride, int rows, int cols, bool aligned, int lane) {
  constexpr int kElems = 128 / SIZE, kChunk = 16 / SIZE;
  uint8_t* g = static_cast<uint8_t*>(global);
  if (aligned) {
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + lane / 8, j = lane % 8;
      if (r >= rows) continue;
      uint8_t* p = g + (r * stride) * SIZE + j * 16;
      if ((j + 1) * kChunk <= cols) {
        if (STORE)
          *reinterpret_cast<uint4*>(p) = *staged(buf, r, j);
        else
          *staged(buf, r, j) = *reinterpret_cast<const uint4*>(p);
      } else {
        uint8_t* q = reinterpret_cast<uint8_t*>(staged(buf, r, j));
        for (int c = 0; j * kChunk + c < cols && c < kChunk; ++c) {
          if (SIZE == 4) {
            if (STORE) reinterpret_cast<uint32_t*>(p)[c] = reinterpret_cast<uint32_t*>(q)[c];
            else reinterpret_cast<uint32_t*>(q)[c] = reinterpret_cast<uint32_t*>(p)[c];
          } else {
            if (STORE) reinterpret_cast<uint16_t*>(p)[c] = reinterpret_cast<uint16_t*>(q)[c];
            else reinterpret_cast<uint16_t*>(q)[c] = reinterpret_cast<uint16_t*>(p)[c];
          }
        }
      }
    }
    return;
  }
  for (int r = 0; r < rows; ++r) {
#pragma unroll
    for (int c = lane; c < kElems; c += 32) {
      if (c >= cols) continue;
      uint8_t* p = g + (r * stride + c) * SIZE;
      uint8_t* q = reinterpret_cast<uint8_t*>(staged(buf, r, c / kChunk)) + c % kChunk * SIZE;
      if (SIZE == 4) {
        if (STORE) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(q);
        else *reinterpret_cast<uint32_t*>(q) = *reinterpret_cast<uint32_t*>(p);
      } else {
        if (STORE) *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<uint16_t*>(q);
        else *reinterpret_cast<uint16_t*>(q) = *reinterpret_cast<uint16_t*>(p);
      }
    }
  }
}

// 64 TMEM columns times the factor (a pair of equal halves), added to the pairs acc[0..31]
__device__ __forceinline__ void add64(const uint32_t (&d)[64], uint64_t f, uint64_t (&acc)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%1, %2};\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}" : "+l"(acc[i]) : "r"(d[2 * i]), "r"(d[2 * i + 1]), "l"(f));
}

template <int ODT>
__global__ void __launch_bounds__(kManyThreads, 1)
    many_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                const __grid_constant__ CUtensorMap smap, const __grid_constant__ CUtensorMap omap,
                const __grid_constant__ CUtensorMap rmap, const FewArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* scales = smem + kManyStages * kManyStageBytes + 8 * 2 * kLineBytes;  // [slot][128]
  __shared__ alignas(8) uint64_t full[kManyStages], empty[kManyStages], acc_full[2], acc_empty[2], res_full[8], scale_full[kScaleSlots];
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kManyStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 2), mbar_init(&acc_empty[i], 16);
    for (int i = 0; i < 8; ++i) mbar_init(&res_full[i], 1);
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&scale_full[i], 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  const int tiles = a.n_tiles * a.t_tiles, first = blockIdx.x / 2, step = gridDim.x / 2;
  pdl_launch_dependents();

  // 384 threads start with 168 registers each (64512); the epilogue's 256 take 224, the other 128 keep 40 (62464)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      if (tc::elect_one()) {
        tc::prefetch_tmap(&wmap);
        tc::prefetch_tmap(&xmap);
        tc::prefetch_tmap(&smap);
        tc::prefetch_tmap(&omap);
        pdl_wait();
        int it = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
          const int t0 = tile % a.t_tiles * kManyT + rank * 128, n0 = tile / a.t_tiles * kManyN + rank * 128;
          for (int b = 0; b < a.blocks; ++b, ++it) {
            const int s = it % kManyStages;
            if (it >= kManyStages && !wait(&empty[s], (it / kManyStages + 1) & 1, a.header, 0x810u)) {
              ok = false;
              break;
            }
            // the first CTA's barrier counts both CTAs' tiles
            uint8_t* st = smem + s * kManyStageBytes;
            const uint32_t bar = peer_addr(&full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kManyStageBytes);
            pair_load(st, &xmap, bar, b * kBlock, t0);
            mbar_arrive_expect_tx(&scale_full[it % kScaleSlots], 128);
            tc::tma_load_2d(scales + it % kScaleSlots * 128, &smap, &scale_full[it % kScaleSlots], t0, b);
            pair_load(st + kTileBytes, &wmap, bar, b * kBlock, n0);
          }
        }
      }
    } else if (warp == 1 && rank == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        for (int b = 0; b < a.blocks; ++b, ++it) {
          const int s = it % kManyStages, buf = it & 1;
          if (!wait(&full[s], (it / kManyStages) & 1, a.header, 0x811u) ||
              (it >= 2 && !wait(&acc_empty[buf], (it / 2 + 1) & 1, a.header, 0x812u))) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t base = smem_u32(smem + s * kManyStageBytes);
            const uint64_t ad = tc::sw128_desc(base), bd = tc::sw128_desc(base + kTileBytes);
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
              pair_mma(tmem + buf * kManyN, ad + 2 * k, bd + 2 * k, idesc_e4m3(kManyT, kManyN), k > 0);
            pair_commit(&empty[s]);
            pair_commit(&acc_full[buf]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 2) {
      // The scales' hand-over: a commit, the other CTA's on top of it, hands on nothing but its products, so a block's products are there
      // for the epilogue once its scales are too. (A wait of each epilogue warp for the scales took 16001 x 5632 x 2048 8 to 14 us.)
      if (tc::elect_one()) {
        int it = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
          for (int b = 0; b < a.blocks; ++b, ++it) {
            // (an arrival ahead of the block two back would end that one's phase)
            if ((it >= 2 && !wait(&acc_full[it & 1], (it / 2 + 1) & 1, a.header, 0x815u)) ||
                !wait(&scale_full[it % kScaleSlots], (it / kScaleSlots) & 1, a.header, 0x816u)) {
              ok = false;
              break;
            }
            mbar_arrive(&acc_full[it & 1]);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    constexpr int kSize = ODT == MV_F32 ? 4 : 2, kPart = 128 / kSize;  // columns that a row of the staging holds
    const int half = (warp - 4) / 4, quarter = warp & 3;  // a warp has 32 tokens and half of the tile's columns
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
    uint8_t* lines = smem + kManyStages * kManyStageBytes + (warp - 4) * 2 * kLineBytes;
    const uint32_t freed = peer_addr(&acc_empty[0], 0);
    pdl_wait();
    // lane l's scale of the weights of block b + l
    auto load_ws = [&](int tile, int b) {
      const int n0 = tile / a.t_tiles * kManyN + half * 128;
      return b + lane < a.blocks && n0 < a.N ? a.ws[n0 / kBlock * a.ws_st + b + lane] : 0.f;
    };
    int it = 0, turn = 0, fetched = 0;
    bool ok = true;
    float ws_next = load_ws(first, 0);
    for (int tile = first; tile < tiles && ok; tile += step) {
      const int t0 = tile % a.t_tiles * kManyT + rank * 128 + quarter * 32, n0 = tile / a.t_tiles * kManyN + half * 128;
      const int rows = min(32, a.T - t0), cols_here = a.N - n0;
      // the residual's first two lines come while the products are made
      const bool fetch = a.res_lines && rows > 0 && cols_here > 0;
      if (fetch && lane == 0) {
        stores_read<0>();
        const int n = cols_here > kPart ? 2 : 1;
        uint8_t* to[2] = {lines + (turn & 1) * kLineBytes, lines + ((turn + 1) & 1) * kLineBytes};
        mbar_arrive_expect_tx(&res_full[warp - 4], n * kLineBytes);
        for (int i = 0; i < n; ++i) tc::tma_load_2d(to[i], &rmap, &res_full[warp - 4], n0 + i * kPart, t0);
      }
      float ws_now = ws_next;
      if (tile + step < tiles) ws_next = load_ws(tile + step, 0);
      uint64_t acc[2][32];  // pairs of columns
#pragma unroll
      for (int c = 0; c < 32; ++c) acc[0][c] = acc[1][c] = 0;
      for (int b = 0; b < a.blocks && ok; ++b, ++it) {
        const int buf = it & 1;
        if ((b & 31) == 0 && b > 0) ws_now = load_ws(tile, b);
        const float w_now = __shfl_sync(0xffffffffu, ws_now, b & 31);
        if (!wait(&acc_full[buf], (it / 2) & 1, a.header, 0x813u)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const float f1 = power(scales[it % kScaleSlots * 128 + quarter * 32 + lane], 0) * w_now;
        uint64_t f;
        asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "f"(f1));
        uint32_t d[64];
        tmem_ld64(lanes + buf * kManyN, d);
        landed(d);
        add64(d, f, acc[0]);
        tmem_ld64(lanes + buf * kManyN + 64, d);
        landed(d);
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(freed + buf * 8) : "memory");
        add64(d, f, acc[1]);
      }
      if (fetch && !wait(&res_full[warp - 4], fetched++ & 1, a.header, 0x814u)) ok = false;
      if (rows <= 0 || !ok) continue;
#pragma unroll
      for (int p = 0; p < 128 / kPart; ++p) {
        const int h = p / (64 / kPart), c = p % (64 / kPart) * kPart;
        const int n = n0 + p * kPart, cols = a.N - n;
        if (cols <= 0) break;
        uint8_t* line = lines + (turn++ & 1) * kLineBytes;
        if (a.out_lines && lane == 0 && !(fetch && p < 2)) stores_read<1>();  // the store before the last was from here
        __syncwarp();
        if (a.residual != nullptr && !(fetch && p < 2)) {
          move_lines<kSize, false>(line, static_cast<uint8_t*>(const_cast<void*>(a.residual)) + (t0 * a.r_st + n) * kSize,
                                   a.r_st, rows, cols, a.res_lines, lane);
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4* slot = staged(line, lane, j);
          float v[16 / kSize];
#pragma unroll
          for (int i = 0; i < 8 / kSize; ++i)
            asm("mov.b64 {%0, %1}, %2;" : "=f"(v[2 * i]), "=f"(v[2 * i + 1]) : "l"(acc[h][(c + j * (16 / kSize)) / 2 + i]));
          if constexpr (kSize == 4) {
            float4 o = make_float4(v[0], v[1], v[2], v[3]);
            if (a.residual != nullptr) {
              const float4 r = *reinterpret_cast<const float4*>(slot);
              o.x += r.x, o.y += r.y, o.z += r.z, o.w += r.w;
            }
            *reinterpret_cast<float4*>(slot) = o;
          } else {
            uint32_t w[4];
            uint4 r = make_uint4(0u, 0u, 0u, 0u);
            if (a.residual != nullptr) r = *slot;
            const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 add = unpack<ODT>(rr[i]);
              w[i] = pack<ODT>(v[2 * i] + add.x, v[2 * i + 1] + add.y);
            }
            *slot = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        // a tensor store writes whole 16 bytes: a line that ends inside them would reach into what lies behind it
        if (a.out_lines && cols >= kPart) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) store_lines(&omap, line, n, t0);
        } else {
          __syncwarp();
          move_lines<kSize, true>(line, static_cast<uint8_t*>(a.out) + (t0 * a.o_st + n) * kSize, a.o_st, rows, cols, a.out_lines, lane);
          if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // (an empty one, for stores_read's count)
          // all lanes have read the line before the next residual's copy may come into it
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc::fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ host

// a [rows, cols] tensor of `size`-byte elements (1, 2 or 4; rows of `stride` bytes) in boxes of 128 bytes x box_rows
int row_map(CUtensorMap* m, const void* base, int size, int cols, int rows, long long stride, int box_rows, const char* what,
            bool swizzle = true) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  if (enc == nullptr) return fail(MV_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(box_rows)}, estr[2] = {1, 1};
  const CUtensorMapDataType type = size == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT32;
  const auto encode = [&] {
    return enc(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT && bind_context()) r = encode();
  if (r != CUDA_SUCCESS) return fail(MV_ERR_INVALID, "tensor map for %s rejected (CUresult %d)", what, static_cast<int>(r));
  return MV_OK;
}

template <typename... P, typename... A>
int launch(void (*fn)(P...), int grid, int threads, size_t smem, int cluster, cudaStream_t st, const A&... args) {
  // the most that any call takes: the limit is the kernel's, not the launch's, and another thread may be about to launch
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem));
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(mv_fp8_linear)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, fn, args...), "mv_fp8_linear launch");
}

// CTAs that share a tile's blocks of K: as many as find place at once, which clusters do on some 5/7 of the SMs (64 x 2048 x 2048, 16
// tiles: clusters of 4 7.8 us, of 8 12.2)
int split_of(long long tiles, int blocks) {
  int split = 1;
  while (split < 8 && tiles * split * 2 <= num_sms() * 5 / 7 && split * 2 <= blocks) split *= 2;
  return split;
}

template <int ODT>
int run_token(const LinearArgs& x, cudaStream_t st) {
  TokenArgs g{};
  g.f = FewArgs{x.ws, nullptr, x.residual, x.out, x.ws_st, 0, x.r_st, x.o_st, x.T, x.N, x.blocks, (x.N + kTile - 1) / kTile, 1, 1,
                x.x_dtype == MV_BF16, false, false, x.header};
  g.x = x.x, g.x_st = x.x_st, g.K = x.K;
  g.vec = ((reinterpret_cast<uintptr_t>(x.x) | static_cast<uintptr_t>(x.x_st * 2)) & 15) == 0 && x.K % 8 == 0 ? 8 : 1;
  g.f.split = split_of(g.f.n_tiles, x.blocks);
  const int share = (x.blocks + g.f.split - 1) / g.f.split;
  g.stages = kTokenStages;
  while (token_smem(share, g.stages) > kMostSmem) --g.stages;
  CUtensorMap wm;
  const int rc = row_map(&wm, x.w, 1, x.K, x.N, x.w_st, kTile, "wq");
  if (rc != MV_OK) return rc;
  return launch(token_kernel<ODT>, g.f.n_tiles * g.f.split, 192, token_smem(share, g.stages), g.f.split, st, wm, g);
}

template <int NT, int ODT>
int run_few(const LinearArgs& x, cudaStream_t st) {
  FewArgs a{x.ws, x.scale, x.residual, x.out, x.ws_st, x.s_st, x.r_st, x.o_st, x.T, x.N, x.blocks, 0, 0, 1, x.x_dtype == MV_BF16, false, false, x.header};
  a.n_tiles = (x.N + kTile - 1) / kTile;
  a.t_tiles = (x.T + NT - 1) / NT;
  CUtensorMap wm, xm;
  int rc = row_map(&wm, x.w, 1, x.K, x.N, x.w_st, kTile, "wq");
  if (rc == MV_OK) rc = row_map(&xm, x.q, 1, static_cast<int>(x.q_st), x.T, x.q_st, NT, "the activations");
  if (rc != MV_OK) return rc;
  const long long tiles = static_cast<long long>(a.n_tiles) * a.t_tiles;
  if (tiles > 0x7fffffffLL) return fail(MV_ERR_INVALID, "mv_fp8_linear: T=%d x N=%d is too large", x.T, x.N);
  const int sms = num_sms();
  a.split = split_of(tiles, a.blocks);
  const int grid = a.split > 1 ? static_cast<int>(tiles) * a.split : static_cast<int>(tiles < sms ? tiles : sms);
  return launch(few_kernel<NT, ODT>, grid, Few<NT>::kThreads, Few<NT>::kSmem, a.split, st, wm, xm, a);
}

template <int ODT>
int run_typed(const LinearArgs& x, cudaStream_t st) {
  if (one_launch(x)) return run_token<ODT>(x, st);
  if (x.T <= 16) return run_few<16, ODT>(x, st);
  if (x.T <= 32) return run_few<32, ODT>(x, st);
  if (x.T <= 64) return run_few<64, ODT>(x, st);
  const long long tiles = static_cast<long long>((x.N + kManyN - 1) / kManyN) * ((x.T + kManyT - 1) / kManyT);
  if (tiles > 0x7fffffffLL) return fail(MV_ERR_INVALID, "mv_fp8_linear: T=%d x N=%d is too large", x.T, x.N);
  const int pairs = num_sms() / 2;
  if (tiles < pairs / 2) return run_few<128, ODT>(x, st);
  FewArgs a{x.ws, x.scale, x.residual, x.out, x.ws_st, x.s_st, x.r_st, x.o_st, x.T, x.N, x.blocks, 0, 0, 1, x.x_dtype == MV_BF16, false, false, x.header};
  a.n_tiles = (x.N + kManyN - 1) / kManyN;
  a.t_tiles = (x.T + kManyT - 1) / kManyT;
  const int size = ODT == MV_F32 ? 4 : 2;
  a.out_lines = aligned16(x.out) && x.o_st * size % 16 == 0;
  CUtensorMap wm, xm, sm, om, rm;
  int rc = row_map(&wm, x.w, 1, x.K, x.N, x.w_st, 128, "wq");
  if (rc == MV_OK) rc = row_map(&xm, x.q, 1, static_cast<int>(x.q_st), x.T, x.q_st, 128, "the activations");
  if (rc == MV_OK) rc = row_map(&sm, x.scale, 1, static_cast<int>(x.s_st), x.blocks, x.s_st, 1, "the scales", false);
  a.res_lines = x.residual != nullptr && aligned16(x.residual) && x.r_st * size % 16 == 0 && (x.T == 1 || x.r_st >= x.N);
  om = rm = xm;
  if (rc == MV_OK && a.out_lines) rc = row_map(&om, x.out, size, x.N, x.T, x.o_st * size, 32, "out");
  if (rc == MV_OK && a.res_lines) rc = row_map(&rm, x.residual, size, x.N, x.T, x.r_st * size, 32, "residual");
  if (rc != MV_OK) return rc;
  return launch(many_kernel<ODT>, static_cast<int>(tiles < pairs ? tiles : pairs) * 2, kManyThreads, kManySmem, 2, st, wm, xm,
                sm, om, rm, a);
}

}  // namespace

// Up to four tokens over rows that do not fill the card by themselves: one launch less is 3 us as called (2560 x 2048, one token:
// 10.7 -> 7.6; in a graph 5.6 / 5.5). 16 tokens take longer to round in each CTA than once before (7.4 us against 6.6), and over a
// vocabulary the activations' place in shared memory is missed by the ring (131072 x 2048: 52.4 us against 50.1).
bool one_launch(const LinearArgs& x) {
  const int split = split_of((x.N + kTile - 1) / kTile, x.blocks);
  if (x.T > 4 || split == 1) return false;
  return (x.blocks + split - 1) / split <= kTokenBlocks;  // shared memory for the rounded activations
}

int run_product(const LinearArgs& x, int out_dtype, cudaStream_t st) {
  if (out_dtype == MV_F32) return run_typed<MV_F32>(x, st);
  if (out_dtype == MV_F16) return run_typed<MV_F16>(x, st);
  return run_typed<MV_BF16>(x, st);
}

}  // namespace fp8
}  // namespace mv
