// Attention of few rows per key head (a decode step, drafted tokens): mma.sync kernel, keys streamed once.
//
// Mathematics: out = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m), t_j = scale log2(e) q . k_j, with a running maximum m
// and sum per row: when a key tile raises m, what has been summed is multiplied by 2^(m_old - m_new).
//
// Measured on a B200, call after call (16 query / 4 key heads of 128 unless said): one token over 812 keys 9.1 to 10.2 us (8.6
// in a graph), over 130501 keys (12 / 2 heads) 29.9 us (134 MB, 4.48 TB/s), 61 sequences of 301061 keys together 105 us (617 MB,
// 5.88 TB/s, 91 % of the measured copy; 100 us in a graph).
//
// Bound: memory. A key row of 2 D values serves the G query heads of its key head (4 G D flops per 4 D bytes), so at
// G = 4..8 the cache has to stream at HBM speed and the products need a few percent of the tensor pipe. Both
// products are taken transposed, S^T = K Q^T and O^T = V^T P^T, with the keys (the head's values) in the 16-row
// operand and the query rows in the 8-column one: 8 rows fill an instruction where the untransposed form would fill
// half of it. (Two such columns of 8 rows still pay: 16 query heads to one key head over 48 x 5000 keys 38.9 us, the 128-row
// kernel 40.4. Four did not: 32 heads 82.2 and 40.7.) The cost of that is one movmatrix per 8 x 8 block of P.
//
// Split: one CTA per SM takes an equal share of all key tiles (attn_common.cuh). Producer warps keep a ring of
// key tiles filled by TMA (a box per page and 64 values, 128-byte swizzle); each of the consumer warps takes whole
// tiles in turn with its own maximum, sum and output in registers, so the warps meet only at the end of a piece.
// Pieces of an item that ranges cut go to the workspace and join_kernel joins them in CTA order.
#include "attn_common.cuh"

namespace mv {
namespace attn {
namespace {

template <int D, int NT>
struct Cfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kBN = D == 128 ? 32 : 64;             // keys of a tile
  static constexpr int kWarps = 8;                            // consumer warps
  // producer warps, a tile each in turn: issuing a tile's copies is a chain of some 800 cycles for one warp, which
  // would hold the ring to 16 KB per 0.43 us (5.6 TB/s over the card, before anything else is in the way)
  static constexpr int kProd = 4;
  static constexpr int kThreads = 32 * (kWarps + kProd);
  static constexpr int kTile = kBN * D * 2;                   // bytes of a key (or value) tile
  static constexpr int kStage = 2 * kTile;
  // a ring slot is always read by the same warp (tile i: slot i % kStages, warp i % kWarps), so a warp never waits
  // for a slot whose previous copy it has not seen complete
  static constexpr int kStages = 131072 / kStage;
  static_assert(kStages % kWarps == 0, "ring slots of one warp");
  static constexpr int kOS = D + 4;                           // row stride of the merge buffer (no bank conflicts)
  static constexpr int kMerge = kWarps * kRows * kOS * 4;
  static constexpr int kPiece = kRows * (D + 2);              // floats of a piece: output, maxima, sums
  // shared memory: ring | merge | Q fragments | per-warp maxima and sums | row weights | schedule | barriers
  static constexpr int oMerge = kStages * kStage;
  static constexpr int oQ = oMerge + kMerge;
  static constexpr int oM = oQ + (D / 16) * NT * 32 * 8;
  static constexpr int oL = oM + kWarps * kRows * 4;
  static constexpr int oPre = oL + kWarps * kRows * 4;
  static constexpr int oTmp = oPre + (kMaxB + 4) * 4;
  static constexpr int oBar = oTmp + 32 * 4;
  static constexpr int kSmem = oBar + 2 * kStages * 8 + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// out and lse of values d .. d + 3 of a row from its joined sums
template <bool BF16>
__device__ __forceinline__ void store_row(const Problem& p, long long row, int head, int d, bool sees, const float4& acc,
                                          float M, float L) {
  const float inv = 1.f / L;
  uint2 v = make_uint2(0u, 0u);
  if (sees) v = make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
  *reinterpret_cast<uint2*>(p.out + row * p.o_st + head * p.o_sh + d) = v;
  if (p.lse != nullptr && d == 0) p.lse[row * p.Hq + head] = sees ? M * kLn2 + logf(L) : -INFINITY;
}

// Joins parts of a row: (M, L, acc) and (m, l, v), weights 2^(m - M); a part without a visible key has sum 0.
__device__ __forceinline__ void join(float& M, float& L, float4& acc, float m, float l, const float4& v) {
  if (l == 0.f) return;
  const float Mn = fmaxf(M, m);
  const float a = L != 0.f ? exp2_approx(M - Mn) : 0.f, f = exp2_approx(m - Mn);
  M = Mn;
  L = L * a + f * l;
  acc.x = acc.x * a + f * v.x, acc.y = acc.y * a + f * v.y, acc.z = acc.z * a + f * v.z, acc.w = acc.w * a + f * v.w;
}

template <int D, int NT, bool BF16, bool kLong>
__global__ void __launch_bounds__(Cfg<D, NT>::kThreads, 1)
    split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Problem p,
                 int box) {
  using C = Cfg<D, NT>;
  constexpr int R = C::kRows, NW = C::kWarps, NS = C::kStages, OS = C::kOS, kBN = C::kBN, MT = kBN / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sO = reinterpret_cast<float*>(smem + C::oMerge);
  uint2* sQ = reinterpret_cast<uint2*>(smem + C::oQ);
  float* sM = reinterpret_cast<float*>(smem + C::oM);
  float* sL = reinterpret_cast<float*>(smem + C::oL);
  unsigned int* pre = reinterpret_cast<unsigned int*>(smem + C::oPre);
  unsigned int* tmp = reinterpret_cast<unsigned int*>(smem + C::oTmp);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::oBar);
  uint64_t* empty = full + NS;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int box_shift = 31 - __clz(box);
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    fence_mbar_init();
    tc::prefetch_tmap(&tmK);
    tc::prefetch_tmap(&tmV);
  }
  pdl_launch_dependents();
  pdl_wait();
  build_schedule<kBN, kLong>(p, pre, tmp);  // its barriers also publish the mbarriers
  const unsigned int W = pre[p.B];
  if (W == 0) {
    if (threadIdx.x == 0) p.cuts[blockIdx.x].n = 0;
    return;
  }
  const Cut cut(p, W, kLong && pre[p.B + 1], gridDim.x);
  Walk<kBN, kLong> wk(p, pre, cut, blockIdx.x);

  if (warp >= NW) {
    // ---------------------------------------------------------------- producers: lane 0 issues all copies
    const int turn = warp - NW;
    int it = 0, issued = 0;
    bool ok = true;
    Pages pages;
    for (; wk.more() && ok; wk.next()) {
      const int kend = wk.kend();
      const int i0 = wk.i0, i1 = min(wk.i1, (kend + kBN - 1) / kBN);
      const int skip = (turn - it) & (C::kProd - 1);  // tile `it` of the CTA is producer it % kProd's
      pages.next = Pages::read(p, wk.b, (i0 + skip) * kBN + lane * box, kend);
      const int base = it - i0;
      for (int i = i0 + skip; i < i1; i += C::kProd) {
        const int stage = (base + i) % NS;
        const int live = min(kBN, kend - i * kBN + box - 1) >> box_shift;  // boxes with a key
        pages.step(p, 0x710u);
        pages.next = Pages::read(p, wk.b, (i + C::kProd) * kBN + lane * box, kend);
        ok = __all_sync(0xffffffffu, wait_bar(&empty[stage], (((base + i) / NS) & 1) ^ 1, p.ws, 0x720u));
        if (!ok) break;
        if (tc::elect_one()) mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(live * box * D * 4));
        for (int bx = 0; bx < live; ++bx) {
          const int j = i * kBN + bx * box, page = pages.of(bx);
          const int row = p.page_table != nullptr ? j & ((1 << p.page_shift) - 1) : wk.s.k0 + j;
          if (tc::elect_one()) {
            uint8_t* dst = smem + stage * C::kStage + bx * box * (2 * D);
            tc::tma_load_5d(dst, &tmK, &full[stage], 0, row, 0, wk.h, page);
            tc::tma_load_5d(dst + C::kTile, &tmV, &full[stage], 0, row, 0, wk.h, page);
          }
        }
        issued = base + i + 1;
      }
      it += max(i1 - i0, 0);
    }
    // its last copies land before the CTA exits: tiles issued - 1, issued - 1 - kProd, ..
    if (tc::elect_one())
      for (int i = issued - 1; i >= 0 && i > issued - 1 - NS; i -= C::kProd)
        wait_bar(&full[i % NS], (i / NS) & 1, p.ws, 0x721u);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, t4 = lane & 3;
  const int tid = threadIdx.x;
  constexpr int NTH = 32 * NW;
  // a tile in shared memory is [box of a page][64-value part][key][64 values]
  const int half_step = box * 128;
  auto row_at = [&](int r) { return (r >> box_shift) * (box * 2 * D) + (r & (box - 1)) * 128; };
  int k_row[MT], v_row[MT];  // the rows this lane addresses for the two products
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    k_row[mt] = row_at(mt * 16 + (lane & 7) + ((lane >> 3) & 1) * 8);
    v_row[mt] = row_at(mt * 16 + (lane & 7) + (lane >> 4) * 8);
  }
  int it = 0;      // tiles of the CTA so far
  bool ok = true;  // a wait that ran out: no more tiles, but every barrier is still met
  CutItem mine{};
  for (; wk.more(); wk.next()) {
    const int kend = wk.kend(), ntok = wk.ntok(), rows = ntok * p.G, first = wk.i0;
    const int i1 = min(wk.i1, (kend + kBN - 1) / kBN);
    // Q as the 8-column operand's fragments: row n = lane / 4, values 16 ks + 2 (lane % 4) + {0, 1} and + {8, 9}
    for (int e = tid; e < (D / 16) * NT * 32; e += NTH) {
      const int l = e & 31, nt = (e >> 5) % NT, ks = (e >> 5) / NT;
      const int r = nt * 8 + (l >> 2);
      uint2 v = make_uint2(0u, 0u);
      if (r < rows) {
        const uint16_t* src = p.q + (wk.s.q0 + wk.tok0() + r / p.G) * p.q_st + (wk.h * p.G + r % p.G) * p.q_sh +
                              ks * 16 + (l & 3) * 2;
        v.x = *reinterpret_cast<const uint32_t*>(src);
        v.y = *reinterpret_cast<const uint32_t*>(src + 8);
      }
      sQ[e] = v;
    }
    named_bar(1, NTH);

    // keys seen by the thread's rows (columns of S^T): 8 nt + 2 t4 + {0, 1}
    int lim[NT][2];
    int lim_min = kend;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + t4 * 2 + c;
        lim[nt][c] = keys_seen(p, wk.s, wk.tok0() + min(r / p.G, ntok - 1) + 1);
        lim_min = min(lim_min, lim[nt][c]);
      }
    float m[NT][2], l[NT][2], o[D / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][nt][c] = 0.f;
    }

    const int base = it - first;  // tile i of the item is the CTA's tile base + i
    it = base + max(i1, first);
    const int skip = ((warp - (base + first)) % NW + NW) % NW;
    for (int i = first + skip; i < i1 && ok; i += NW) {
      const int cta_tile = base + i, stage = cta_tile % NS;
      ok = __all_sync(0xffffffffu, wait_bar(&full[stage], (cta_tile / NS) & 1, p.ws, 0x730u));
      if (!ok) break;
      const uint32_t kt = smem_u32(smem + stage * C::kStage), vt = kt + C::kTile;
      const int nv = min(kBN, kend - i * kBN);  // keys of the tile
      const int blocks = (nv + 15) / 16;
      if (nv < blocks * 16) {
        // rows behind the last key hold anything (an older page's values, NaN): their weights are 0, and 0 * NaN
        // is not, so the values are cleared
        constexpr int kVec = D / 8;
        for (int e = lane; e < (blocks * 16 - nv) * kVec; e += 32) {
          const int r = nv + e / kVec, c = e % kVec;
          *reinterpret_cast<uint4*>(smem + stage * C::kStage + C::kTile + row_at(r) + (c / 8) * half_step +
                                    (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
      // S^T = K Q^T
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
      {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint2 qf[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) qf[nt] = sQ[(ks * NT + nt) * 32 + lane];
          const uint32_t a0 = kt + (ks / 4) * half_step + ((((ks & 3) * 2 + ch) ^ (r & 7)) << 4);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            if (mt < blocks) {
              uint32_t a[4];
              ldsm4(a, a0 + k_row[mt]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<BF16>(s[mt][nt], a, qf[nt].x, qf[nt].y);
            }
        }
      }
      // masks, running maximum, weights
      const int j0 = i * kBN;
      const bool masked = j0 + blocks * 16 > lim_min;
      float tmax[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) tmax[nt][0] = tmax[nt][1] = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (mt < blocks)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float x = s[mt][nt][c] * p.scale_log2;
              if (masked && j0 + mt * 16 + g + (c >> 1) * 8 >= lim[nt][c & 1]) x = -INFINITY;
              s[mt][nt][c] = x;
              tmax[nt][c & 1] = fmaxf(tmax[nt][c & 1], x);
            }
      bool grow = false;
      float base_m[NT][2], alpha[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = tmax[nt][c];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float mn = fmaxf(m[nt][c], x);
          base_m[nt][c] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every weight is 2^-inf = 0
          alpha[nt][c] = exp2_approx(m[nt][c] - base_m[nt][c]);
          grow = grow || mn != m[nt][c];
          m[nt][c] = mn;
          l[nt][c] *= alpha[nt][c];
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[j][nt][c] *= alpha[nt][c & 1];
      }
      uint32_t pb[MT][NT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (mt < blocks)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              e[c] = exp2_approx(s[mt][nt][c] - base_m[nt][c & 1]);
              l[nt][c & 1] += e[c];
            }
            // the weights are rounded to the element type here, as the second product's 16-bit operands (32-bit ones would
            // double its work; the outputs' mean relative error against 64 bits is 1.7e-3 for 1.6e-3 in bf16, the latter
            // the result's own rounding, and 2.2e-4 for 2.1e-4 in f16)
            pb[mt][nt][0] = transpose8(pack2<BF16>(e[0], e[1]));
            pb[mt][nt][1] = transpose8(pack2<BF16>(e[2], e[3]));
          }
      // O^T += V^T P^T
      {
        const int r = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          if (mt < blocks) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              uint32_t a[4];
              ldsm4_t(a, vt + v_row[mt] + (j / 4) * half_step + ((((j & 3) * 2 + ch) ^ (r & 7)) << 4));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<BF16>(o[j][nt], a, pb[mt][nt][0], pb[mt][nt][1]);
            }
          }
      }
      if (nv < blocks * 16) fence_proxy_async_smem();  // this warp's stores before the ring slot's next copy
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }

    // sums over the 8 lanes that share a row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) {
          sM[warp * R + nt * 8 + t4 * 2 + c] = m[nt][c];
          sL[warp * R + nt * 8 + t4 * 2 + c] = x;
        }
      }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sO[(warp * R + nt * 8 + t4 * 2 + (c & 1)) * OS + j * 16 + g + (c >> 1) * 8] = o[j][nt][c];
    named_bar(1, NTH);

    // the warps' parts of a row, joined in warp order: weights 2^(m_w - M); a part without a key has sum 0
    const bool whole = wk.whole();
    float* part = p.parts + (blockIdx.x * 2 + (first > 0 ? 0 : 1)) * C::kPiece;
    constexpr int kVecs = D / 4;
    for (int e = tid; e < rows * kVecs; e += NTH) {
      const int r = e / kVecs, d = (e % kVecs) * 4;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w)
        if (sL[w * R + r] != 0.f) M = fmaxf(M, sM[w * R + r]);
      float L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float lw = sL[w * R + r];
        if (lw != 0.f) {
          const float f = exp2_approx(sM[w * R + r] - M);
          const float4 v = *reinterpret_cast<const float4*>(sO + (w * R + r) * OS + d);
          L += f * lw;
          acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
        }
      }
      if (whole) {
        const int i = r / p.G;
        store_row<BF16>(p, wk.s.q0 + wk.tok0() + i, wk.h * p.G + r % p.G, d, keys_seen(p, wk.s, wk.tok0() + i + 1) > 0,
                        acc, M, L);
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = acc;
        if (d == 0) {
          part[R * D + r] = M;
          part[R * D + R + r] = L;
        }
      }
    }
    if (!whole && first == 0) mine = wk.cut_item(cut, blockIdx.x);
    named_bar(1, NTH);  // the merge buffer and Q are free again
  }
  if (tid == 0) p.cuts[blockIdx.x] = mine;
}

// Joins the pieces of the item that starts in CTA blockIdx.x's range and ends in a later one's, rows blockIdx.y NT .. + NT - 1.
// A few rows of many pieces (74 of one long sequence) are a chain of L2 latencies for one CTA (9 us for a single CTA that
// did it all), so every row has 8 warps: warp w joins pieces w, w + 8, .. in order, then the warps' results are joined. 64
// registers, so that four CTAs, of which most find nothing to do, fit an SM (batch of 61 sequences 101.9 -> 100.0 us).
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(256, 4) join_kernel(const Problem p) {
  constexpr int R = 8 * NT, kPiece = R * (D + 2), kLanes = D / 4, kAhead = 5;
  __shared__ float sM[8], sL[8];
  __shared__ float4 sV[8][kLanes];
  pdl_wait();
  const CutItem c = p.cuts[blockIdx.x];
  if (c.n <= 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = blockIdx.y * NT; r < blockIdx.y * NT + NT && r < c.ntok * p.G; ++r) {
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = warp; i0 < c.n; i0 += 8 * kAhead) {
      float m[kAhead], l[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + 8 * k;
        l[k] = 0.f;
        if (i < c.n) {
          // the first piece is CTA blockIdx.x's last (slot 1), the others are their CTAs' first (slot 0)
          const float* pc = p.parts + (static_cast<size_t>(blockIdx.x + i) * 2 + (i == 0)) * kPiece;
          m[k] = pc[R * D + r];
          l[k] = pc[R * D + R + r];
          if (lane < kLanes) v[k] = reinterpret_cast<const float4*>(pc + r * D)[lane];
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i0 + 8 * k < c.n) join(M, L, acc, m[k], l[k], v[k]);
    }
    if (lane == 0) sM[warp] = M, sL[warp] = L;
    if (lane < kLanes) sV[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && lane < kLanes) {
#pragma unroll
      for (int w = 1; w < 8; ++w) join(M, L, acc, sM[w], sL[w], sV[w][lane]);
      const int i = r / p.G;
      store_row<BF16>(p, c.row0 + i, c.h * p.G + r % p.G, lane * 4, i >= c.first, acc, M, L);
    }
    __syncthreads();
  }
}

template <int D, int NT>
int launch_split(Problem& p, const Source& src, bool bf16, int grid, cudaStream_t st) {
  using C = Cfg<D, NT>;
  CUtensorMap mk, mv_;
  const int box = src.box < C::kBN ? src.box : C::kBN;
  p.can_cut = src.max_keys > C::kBN;
  const int rc = make_kv_maps(&mk, &mv_, src, p.Hkv, D, bf16, box, D / 64);
  if (rc != MV_OK) return rc;
  const bool lng = may_be_long(p, src, C::kBN);
  auto fn = bf16 ? (lng ? split_kernel<D, NT, true, true> : split_kernel<D, NT, true, false>)
                 : (lng ? split_kernel<D, NT, false, true> : split_kernel<D, NT, false, false>);
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(attention split)");
  const int rc2 = launch_pdl(fn, dim3(grid), C::kThreads, C::kSmem, st, "attention split launch", mk, mv_, p, box);
  if (rc2 != MV_OK || !p.can_cut) return rc2;
  return launch_pdl(bf16 ? join_kernel<D, NT, true> : join_kernel<D, NT, false>, dim3(grid, 8), 256, 0, st,
                    "attention join launch", p);
}

}  // namespace

// The kernel for `rows_hint` rows (at most 16) per (sequence, key head); any number is computed rightly (tiles of tok tokens).
int run_split(Problem& p, const Source& src, int D, bool bf16, int rows_hint, int grid, cudaStream_t st) {
  const int nt = rows_hint <= 8 && p.G <= 8 ? 1 : 2;
  p.tok = 8 * nt / p.G;
  // Fewer items than CTAs: cutting is what fills the card, and the less a CTA has the sooner it is done (one token over
  // 812 keys, 4 key heads: 9.3 us with 2 and 7, 10.6 with 6 and 14). More: an item counts for what it costs besides its
  // tiles, so that CTAs with several short items get less (61 sequences of 300000 keys: 101.9 us with 6, 104.3 with 2).
  const bool few = static_cast<long long>(p.B) * p.Hkv < grid;
  if (few) cut_rule<2, 7>(p);
  else cut_rule<6, 14>(p);
  if (D == 128)
    return nt == 1 ? launch_split<128, 1>(p, src, bf16, grid, st) : launch_split<128, 2>(p, src, bf16, grid, st);
  return nt == 1 ? launch_split<64, 1>(p, src, bf16, grid, st) : launch_split<64, 2>(p, src, bf16, grid, st);
}

}  // namespace attn
}  // namespace mv
