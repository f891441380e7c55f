// Attention of many rows per key head (prompts, chunks of new tokens) on the 5th-generation tensor cores.
//
// Mathematics: as in attn_split.cu, a running maximum and sum per row over tiles of 128 keys. The maximum that the
// weights are taken against is raised only when a tile exceeds it by more than 8 (in powers of two): weights then stay
// below 2^8, nothing overflows, and the accumulator is rarely rescaled; out = sum p v / sum p is the same.
//
// Bound: the tensor pipe and the exponential unit together. A 128 x 128 tile of scores takes 2 x 128^2 x D
// multiply-adds (512 + 512 cycles at D = 128) and 16384 exponentials (1024 cycles at 16 a cycle and SM), so the two
// have to run side by side.
//
// Measured on a B200, call after call: 20000 causal tokens in 2 prompts, 16 / 4 heads of 128, bf16: 998 us (1050 TFLOP/s, 62 % of
// the measured burst and 73 % of the sustained peak: power is the bound; 855 us in a few calls after a pause); 2043 new tokens
// over 45000 cached 249 us (913; 210); 9999 tokens, all pairs, 16 / 16 heads of 64, f16: 192 us (598; the exponential unit is
// busy 75 % of the time).
//
// Layout of a CTA (one per SM): a work item is two tiles of 128 rows (row = token * G + head) of one sequence and key
// head, which share the key and value tiles in shared memory.
//   warps 0, 2   TMA producers: Q and K tiles, V tiles, into two rings of slots (a box per page and 64 values). One
//                warp fills all slots of a ring: its wait for a free slot knows the slot's last use by parity, which
//                holds only for a warp that has itself issued that use
//   warps 1, 3   MMA issuers: S_t = Q_t K^T and O_t += P_t V, both into TMEM; P_t is the TMEM operand. D = 128: warp 1
//                for both row tiles in turn; D = 64: a warp each
//   warps 4..7   softmax of tile 0, warps 8..11 of tile 1: a thread owns a row (a TMEM lane). S -> weights P in TMEM;
//                the row's sum and maximum stay in registers; at the end O / sum -> global memory.
// D = 128: while one tile's scores are in the softmax, the other tile's products run. TMEM columns: S_0 | S_1 | O_0 | O_1,
// 128 each; P_t overwrites S_t, so QK(j + 1) follows PV(j), and the one issuer keeps the tiles half a period apart. (An
// issuer per tile let them fall into step, both in the exponentials and then both waiting: 1155 us instead of 891 for
// 20000 causal tokens, 16 / 4 heads.)
// D = 64: the softmax is the bound. S_0 | S_1 (128) | P_0 | P_1 | O_0 | O_1 (64): QK(j + 1) needs only S_t to be in
// registers, so the softmax finds its next scores ready, and PV(j) starts when half of the weights are there.
//
// Split: equal shares of all (item, key tile) units (attn_common.cuh). Pieces of a cut item go to the workspace and
// combine_kernel joins them in CTA order.
#include "attn_common.cuh"

namespace mv {
namespace attn {
namespace {

constexpr int kBN = 128;        // keys of a tile
constexpr int kM = 128;         // rows of a tile
constexpr int kThreads = 384;
constexpr float kHuge = 16777216.f;
constexpr float kGrow = 8.f;    // growth of the maximum, in powers of two, that is not followed at once

template <int D>
struct Cfg {
  static constexpr int kTile = kBN * D * 2;         // bytes of a K or V tile
  static constexpr int kQ = kM * D * 2;             // bytes of a Q tile
  static constexpr int kSlots = 65536 / kTile;      // of each ring
  static constexpr int oK = 2 * kQ;
  static constexpr int oV = oK + kSlots * kTile;
  static constexpr int oPre = oV + kSlots * kTile;
  static constexpr int oTmp = oPre + (kMaxB + 4) * 4;
  static constexpr int oBar = oTmp + 32 * 4;
  static constexpr int kBars = 4 * kSlots + 2 + 10 + 1;
  static constexpr int oTmem = oBar + kBars * 8;
  static constexpr int oOut = (oTmem + 31) / 16 * 16;  // a buffer per softmax warp: 32 rows of 64 B, 80 B apart
  static constexpr int kOutWarp = 32 * 80;
  static constexpr int kSmem = oOut + 8 * kOutWarp + 1024;
  static_assert(kSmem <= 232448, "shared memory");
  static constexpr bool kEarly = D == 64;  // P has columns of its own
  static constexpr int kIssuers = kEarly ? 2 : 1;
  __device__ __forceinline__ static uint32_t tmem_p(uint32_t base, int t) {
    return kEarly ? base + 256 + t * 64 : base + t * 128;
  }
  __device__ __forceinline__ static uint32_t tmem_o(uint32_t base, int t) {
    return kEarly ? base + 384 + t * 64 : base + 256 + t * 128;
  }
};

// D[tmem] (+)= A[tmem] * B[smem], 16-bit operands, fp32 accumulation; issued by one thread.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of V as the MN-major operand (N = head values, contiguous; K = keys): atoms of 8 keys x 64 values
// (8 x 128 B, 128-byte swizzle). Leading offset (bits 16-29): to the next 64 values; stride offset (32-45): to the
// next 8 keys, 1024 B.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr, uint32_t half_bytes) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(half_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// kind::f16 instruction descriptor (tc.cuh's fields) for either element type; b_mn: B is MN-major (bit 16).
__host__ __device__ constexpr uint32_t idesc16(bool bf16, int M, int N, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The row's weights 2^(s scale + base) of a tile into TMEM, rounded to the element type there; returns their fp32 sum. They are
// rounded because the second product takes 16-bit operands: 32-bit ones (tf32) run at half the rate and would need twice the
// TMEM columns, which are all taken. The mean relative error of the outputs against 64 bits goes from 1.6e-3 (the result's own
// rounding) to 2.2e-3 in bf16 (20000 tokens), from 2.1e-4 to 2.9e-4 in f16 (2000 tokens, all pairs).
// Bound by the exponential unit: 8 cycles an instruction and scheduler, 1052 for the 128 of a row. (Handing 2 to 8 of 16 pairs
// to a polynomial of degree 4 or 5 on the FMA pipe gave 1075 to 1219, and longer kernels: the clamp, the rounding and the
// packed multiplies cost what they relieve.)
template <typename C, bool BF16>
__device__ __forceinline__ float weights(const uint32_t (&s)[4][32], float base, float scale, uint32_t tP,
                                         uint64_t* half_done) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float x0 = base, x1 = base;
      ffma2(x0, x1, __uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1]), scale, scale);
      x0 = exp2_approx(x0);
      x1 = exp2_approx(x1);
      ffma2(sum[(e & 1) * 2], sum[(e & 1) * 2 + 1], x0, x1, 1.f, 1.f);
      pk[e] = pack2<BF16>(x0, x1);
    }
    tmem_st16(tP + c * 16, pk);
    if (C::kEarly && c == 1) {
      tmem_st_wait();
      tc::fence_before_sync();
      mbar_arrive(half_done);
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Key tiles of a piece: [wk.i0, end), of which row tile t sees [wk.i0, end_of[t]).
struct Tiles {
  int kend, end, end_of[2];
  template <bool kLong>
  __device__ __forceinline__ Tiles(const Problem& p, const Walk<kBN, kLong>& wk, int half_tok) {
    kend = wk.kend();
    const int ntok = wk.ntok();
    end = min(wk.i1, (kend + kBN - 1) / kBN);
    end_of[0] = min(wk.i1, (keys_seen(p, wk.s, wk.tok0() + min(ntok, half_tok)) + kBN - 1) / kBN);
    end_of[1] = ntok > half_tok ? end : 0;
  }
};

template <int D, bool BF16, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const Problem p, int box) {
  using C = Cfg<D>;
  constexpr int NS = C::kSlots, kHalves = D / 64, kHalfBytes = kBN * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* kring = smem + C::oK;
  uint8_t* vring = smem + C::oV;
  unsigned int* pre = reinterpret_cast<unsigned int*>(smem + C::oPre);
  unsigned int* tmp = reinterpret_cast<unsigned int*>(smem + C::oTmp);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::oBar);
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* q_full = v_empty + NS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;  // [2] scores of tile t are in TMEM (D = 128: and the product before them is complete)
  uint64_t* s_free = s_full + 2;   // [2] D = 64: the scores of tile t are in registers
  uint64_t* p_half = s_free + 2;   // [2] the first half of tile t's weights is in TMEM, its accumulator may be added to
  uint64_t* p_full = p_half + 2;   // [2] and the second half
  uint64_t* o_full = p_full + 2;   // [2] tile t's product with V is complete (D = 128: the piece's last one)
  uint64_t* done = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::oTmem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], C::kIssuers);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], C::kIssuers);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, C::kIssuers);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], kM);
      mbar_init(&p_half[t], kM);
      mbar_init(&p_full[t], kM);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(done, C::kIssuers);
    fence_mbar_init();
    tc::prefetch_tmap(&tmQ);
    tc::prefetch_tmap(&tmK);
    tc::prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  const int half_tok = p.tok / 2;       // tokens of a 128-row tile
  const int rows_used = half_tok * p.G;
  if (rows_used < kM) {  // Q rows that no copy writes: any finite values
    for (int e = threadIdx.x; e < 2 * kHalves * (kM - rows_used) * 8; e += kThreads) {
      const int c = e & 7, r = rows_used + (e >> 3) % (kM - rows_used), hf = (e >> 3) / (kM - rows_used);
      *reinterpret_cast<uint4*>(smem + hf * kHalfBytes + r * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  tc::fence_before_sync();
  pdl_launch_dependents();
  pdl_wait();
  build_schedule<kBN, kLong>(p, pre, tmp);
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const unsigned int W = pre[p.B];
  const Cut cut(p, W, kLong && pre[p.B + 1], gridDim.x);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    Walk<kBN, kLong> wk(p, pre, cut, blockIdx.x);
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------------- TMA producers: lane 0 issues all copies
      const bool is_v = warp == 2;
      const CUtensorMap* map = is_v ? &tmV : &tmK;
      uint8_t* ring = is_v ? vring : kring;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      const int box_shift = 31 - __clz(box);
      int it = 0, qn = 0;  // tiles and items so far
      bool ok = true;
      Pages pages;
      for (; wk.more() && ok; wk.next()) {
        const int kend = wk.kend(), ntok = wk.ntok();
        const int i0 = wk.i0, i1 = min(wk.i1, (kend + kBN - 1) / kBN);
        if (i0 >= i1) continue;
        pages.next = Pages::read(p, wk.b, i0 * kBN + lane * box, kend);
        if (!is_v) {
          const int nt = ntok > half_tok ? 2 : 1;
          ok = __all_sync(0xffffffffu, wait_bar(q_empty, (qn & 1) ^ 1, p.ws, 0x740u));
          if (!ok) break;
          if (tc::elect_one()) {
            mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(nt * kHalves * rows_used * 128));
            for (int t = 0; t < nt; ++t)
              for (int hf = 0; hf < kHalves; ++hf)
                tc::tma_load_3d(smem + t * C::kQ + hf * kHalfBytes, &tmQ, q_full, hf * 64, wk.h * p.G,
                                wk.s.q0 + wk.tok0() + t * half_tok);
          }
          ++qn;
        }
        for (int i = i0; i < i1; ++i, ++it) {
          const int slot = it % NS;
          const int live = min(kBN, kend - i * kBN + box - 1) >> box_shift;  // boxes with a key
          pages.step(p, 0x711u);
          pages.next = Pages::read(p, wk.b, (i + 1) * kBN + lane * box, kend);
          ok = __all_sync(0xffffffffu, wait_bar(&empty[slot], ((it / NS) & 1) ^ 1, p.ws, 0x741u));
          if (!ok) break;
          if (tc::elect_one()) mbar_arrive_expect_tx(&full[slot], static_cast<uint32_t>(live * box * D * 2));
          for (int bx = 0; bx < live; ++bx) {
            const int j = i * kBN + bx * box, page = pages.of(bx);
            const int row = p.page_table != nullptr ? j & ((1 << p.page_shift) - 1) : wk.s.k0 + j;
            if (tc::elect_one())
#pragma unroll
              for (int hf = 0; hf < kHalves; ++hf)
                tc::tma_load_5d(ring + slot * C::kTile + hf * kHalfBytes + bx * box * 128, map, &full[slot], 0, row,
                                hf, wk.h, page);
          }
        }
      }
      // copies in flight land before the CTA exits
      if (tc::elect_one()) {
        if (qn > 0) wait_bar(q_full, (qn - 1) & 1, p.ws, 0x742u);
        for (int i = 0; i < NS && i < it; ++i)
          wait_bar(&full[i], static_cast<uint32_t>(((it - 1 - i) / NS) & 1), p.ws, 0x743u);
      }
    } else if (C::kEarly || warp == 1) {
      // ---------------------------------------------------------------- MMA issuers (one elected lane)
      constexpr uint32_t id_qk = idesc16(BF16, kM, kBN, false), id_pv = idesc16(BF16, kM, D, true);
      int kt = 0, vt = 0, qn = 0;  // K, V tiles and items so far
      uint32_t pn[2] = {0, 0};     // weights taken
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int info) {
        ok = ok && __all_sync(0xffffffffu, wait_bar(bar, parity, p.ws, info));
        tc::fence_after_sync();
        return ok;
      };
      // this warp's part of a slot's release: behind its products, or at once where it has none
      auto release = [&](uint64_t* bar, bool used) {
        if (tc::elect_one()) {
          if (used) tc::mma_commit(bar);
          else mbar_arrive(bar);
        }
      };
      auto qk = [&](int t, int slot) {
        if (tc::elect_one()) {
          const uint32_t qa = smem_u32(smem + t * C::kQ), ka = smem_u32(kring + slot * C::kTile);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            tc::mma_bf16(tmem + t * 128, tc::sw128_desc(qa + (ks / 4) * kHalfBytes) + 2 * (ks & 3),
                         tc::sw128_desc(ka + (ks / 4) * kHalfBytes) + 2 * (ks & 3), id_qk, ks != 0);
          tc::mma_commit(&s_full[t]);
        }
      };
      // O_t (+)= P_t V over keys [16 k0, 16 k1) of the tile
      auto pv = [&](int t, int slot, int k0, int k1, bool first) {
        if (tc::elect_one()) {
          const uint64_t vd = v_desc(smem_u32(vring + slot * C::kTile), kHalfBytes);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k >= k0 && k < k1)
              mma_ts(C::tmem_o(tmem, t), C::tmem_p(tmem, t) + k * 8, vd + k * (2048 >> 4), id_pv, !first || k > 0);
        }
      };
      // rows behind the last of a V tile's nv keys hold anything (an older page's values, NaN, another sequence's): their
      // weights are 0, and 0 * NaN is not, so the values are cleared up to the product's 16 keys (where there are two
      // issuers, by both: the same zeros)
      auto clear_tail = [&](int slot, int nv) {
        const int up = (nv + 15) & ~15;
        if (nv == up) return;
        for (int e = lane; e < (up - nv) * kHalves * 8; e += 32) {
          const int c = e & 7, hf = (e >> 3) % kHalves, r = nv + (e >> 3) / kHalves;
          *reinterpret_cast<uint4*>(vring + slot * C::kTile + hf * kHalfBytes + r * 128 + c * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      };
      if constexpr (C::kEarly) {
        // a warp per row tile; QK(j + 1) before PV(j)
        const int t = warp >> 1;
        for (; wk.more() && ok; wk.next()) {
          const Tiles tl(p, wk, half_tok);
          const int all = tl.end - wk.i0, my = tl.end_of[t] - wk.i0;  // tiles loaded, tiles this row tile sees
          if (all <= 0) continue;
          if (!wait(q_full, qn & 1, 0x750u) || !wait(&k_full[kt % NS], (kt / NS) & 1, 0x751u)) break;
          ++qn;
          if (my > 0) qk(t, kt % NS);
          release(&k_empty[kt % NS], my > 0);
          if (my <= 1) release(q_empty, my > 0);
          ++kt;
          for (int i = 0; i < all; ++i, ++vt) {
            const int vs = vt % NS, ks = kt % NS;
            if (i + 1 < all) {
              if (!wait(&k_full[ks], (kt / NS) & 1, 0x752u)) break;
              if (i + 1 < my) {
                if (!wait(&s_free[t], pn[t] & 1, 0x753u)) break;
                qk(t, ks);
              }
              release(&k_empty[ks], i + 1 < my);
              if (i + 2 == my) release(q_empty, true);
              ++kt;
            }
            if (!wait(&v_full[vs], (vt / NS) & 1, 0x754u)) break;
            if (i < my) {
              const int nv = min(kBN, tl.kend - (wk.i0 + i) * kBN), k16 = (nv + 15) / 16;
              clear_tail(vs, nv);
              if (!wait(&p_half[t], pn[t] & 1, 0x755u)) break;
              pv(t, vs, 0, min(k16, 4), i == 0);
              if (!wait(&p_full[t], pn[t] & 1, 0x756u)) break;
              pv(t, vs, 4, k16, i == 0);
              ++pn[t];
              release(&o_full[t], true);
            }
            release(&v_empty[vs], i < my);
          }
        }
      } else {
        // one warp for both row tiles, which keeps them half a period apart: one in the softmax, one in the products
        for (; wk.more() && ok; wk.next()) {
          const Tiles tl(p, wk, half_tok);
          const int all = tl.end - wk.i0;
          const int my[2] = {tl.end_of[0] - wk.i0, tl.end_of[1] - wk.i0};
          if (all <= 0) continue;
          if (!wait(q_full, qn & 1, 0x750u) || !wait(&k_full[kt % NS], (kt / NS) & 1, 0x751u)) break;
          ++qn;
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (my[t] > 0) qk(t, kt % NS);
          release(&k_empty[kt % NS], true);
          if (all == 1) release(q_empty, true);
          ++kt;
          for (int i = 0; i < all; ++i, ++vt) {
            const int vs = vt % NS, ks = kt % NS;
            const bool more = i + 1 < all;
            if (!wait(&v_full[vs], (vt / NS) & 1, 0x752u)) break;
            if (more && !wait(&k_full[ks], (kt / NS) & 1, 0x753u)) break;
            const int nv = min(kBN, tl.kend - (wk.i0 + i) * kBN);
            clear_tail(vs, nv);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (i >= my[t] || !wait(&p_full[t], pn[t] & 1, 0x754u)) continue;
              ++pn[t];
              pv(t, vs, 0, (nv + 15) / 16, i == 0);
              if (i + 1 == my[t]) release(&o_full[t], true);
              if (i + 1 < my[t]) qk(t, ks);
            }
            if (!ok) break;
            release(&v_empty[vs], true);
            if (more) release(&k_empty[ks], true);
            if (i + 2 == all) release(q_empty, true);
            kt += more;
          }
        }
      }
      // every issued product retires before the TMEM is released
      release(done, true);
      if (warp == 1) wait_bar(done, 0u, p.ws, 0x757u);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax: tile t, a thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    Walk<kBN, kLong> wk(p, pre, cut, blockIdx.x);
    const int t = warp >= 8, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + t * 128, tP = C::tmem_p(tmem, t) + lanes, tO = C::tmem_o(tmem, t) + lanes;
    uint32_t sn = 0, on = 0;  // scores taken, products waited for
    bool ok = true;
    const int my_tok = t * half_tok + r / p.G, my_head = r % p.G;
    CutItem mine{};
    for (; wk.more() && ok; wk.next()) {
      const Tiles tl(p, wk, half_tok);
      const int ntok = wk.ntok(), i0 = wk.i0, i1 = tl.end_of[t];
      const bool whole = wk.whole();
      if (!whole && i0 == 0) mine = wk.cut_item(cut, blockIdx.x);
      if (t == 1 && ntok <= half_tok) continue;
      const bool live = r < rows_used && my_tok < ntok;
      // keys the row sees; rows that are not there see what the last one does
      const int lim = keys_seen(p, wk.s, wk.tok0() + min(my_tok, ntok - 1) + 1);
      const int lim_min = keys_seen(p, wk.s, wk.tok0() + t * half_tok + 1);
      float m = -INFINITY, l = 0.f;
      for (int i = i0; i < i1; ++i) {
        ok = __all_sync(0xffffffffu, wait_bar(&s_full[t], sn & 1, p.ws, 0x760u));
        if (!ok) break;
        ++sn;
        tc::fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld32(tS + c * 32, s[c]);
        tc::tmem_ld_wait();
        if (C::kEarly) {
          tc::fence_before_sync();
          mbar_arrive(&s_free[t]);
        }
        if ((i + 1) * kBN > lim_min) {
          const int left = lim - i * kBN;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= left) s[c][e] = 0xff800000u;  // -inf
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2)
            mx[c] = max3(mx[c], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
          mx[c] = fmaxf(mx[c], __uint_as_float(s[c][31]));
        }
        const float tile_max = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
        const bool grow = (tile_max - m) * p.scale_log2 > kGrow;  // m = -inf: the difference is inf, or NaN if both are
        // weights 2^(s scale + base), one fused multiply-add each; the rounding of base is the same for all of a row's
        // weights and cancels in the quotient, unless it is so large that they overflow: then s - m is taken first
        float base = m == -INFINITY ? 0.f : -m * p.scale_log2;  // nothing seen yet: every weight is 2^-inf = 0
        if (C::kEarly && i > i0) {  // P_t and O_t are this row tile's again
          ok = __all_sync(0xffffffffu, wait_bar(&o_full[t], on & 1, p.ws, 0x762u));
          if (!ok) break;
          ++on;
          tc::fence_after_sync();
        }
        if (__any_sync(0xffffffffu, grow || fabsf(base) > kHuge)) {
          const float alpha = grow ? exp2_approx((m - tile_max) * p.scale_log2) : 1.f;
          if (grow) m = tile_max;
          l *= alpha;
          if (i > i0) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tc::tmem_ld16(tO + c * 16, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(tO + c * 16, o);
            }
          }
          base = m == -INFINITY ? 0.f : -m * p.scale_log2;
          if (fabsf(base) > kHuge) {
            base = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e) s[c][e] = __float_as_uint(__uint_as_float(s[c][e]) - m);
          }
        }
        l += weights<C, BF16>(s, base, p.scale_log2, tP, &p_half[t]);
        tmem_st_wait();
        tc::fence_before_sync();
        mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      const int slot = i0 > 0 ? 0 : 1;
      float* part = p.parts + (static_cast<size_t>(blockIdx.x) * 2 + slot) * (256 * (128 + 2));
      const float m2 = m * p.scale_log2;
      if (i1 > i0) {
        ok = __all_sync(0xffffffffu, wait_bar(&o_full[t], on & 1, p.ws, 0x761u));
        if (!ok) break;
        ++on;
        tc::fence_after_sync();
      }
      const long long row = wk.s.q0 + wk.tok0() + my_tok;
      const int head = wk.h * p.G + my_head;
      const bool sees = lim > 0;
      const float inv = sees ? 1.f / l : 0.f;
      // Output rows go through shared memory 64 B at a time: from registers, a row per lane, every store would touch 32
      // lines; so it touches 8. Lane x stores 16 B of rows x / 4 + 8 i of the warp's.
      const long long off = live ? row * p.o_st + head * p.o_sh : -1;
      uint8_t* buf = smem + C::oOut + (warp - 4) * C::kOutWarp;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (i1 > i0) {
          tc::tmem_ld32(tO + c * 32, o);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (whole) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = sees ? pack2<BF16>(__uint_as_float(o[v * 8 + 2 * e]) * inv, __uint_as_float(o[v * 8 + 2 * e + 1]) * inv)
                          : 0u;
            *reinterpret_cast<uint4*>(buf + lane * 80 + v * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int x = v * 8 + (lane >> 2);
            const long long to = __shfl_sync(0xffffffffu, off, x);
            const uint4 w = *reinterpret_cast<const uint4*>(buf + x * 80 + (lane & 3) * 16);
            if (to >= 0) *reinterpret_cast<uint4*>(p.out + to + c * 32 + (lane & 3) * 8) = w;
          }
          __syncwarp();
        } else {
          // a piece is [4 values][row]: neighbouring lanes write neighbouring 16 B
          float4* dst = reinterpret_cast<float4*>(part) + c * 8 * 256 + t * kM + r;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            dst[v * 256] = make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                                       __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
        }
      }
      if (live) {
        if (whole) {
          if (p.lse != nullptr) p.lse[row * p.Hq + head] = sees ? m2 * kLn2 + logf(l) : -INFINITY;
        } else {
          part[256 * D + t * kM + r] = m2;
          part[256 * D + 256 + t * kM + r] = l;
        }
      }
      tc::fence_before_sync();  // the accumulator is read before the next item's first product is allowed
    }
    if (threadIdx.x == 128) p.cuts[blockIdx.x] = mine;
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the item that starts in CTA blockIdx.x's range and ends in a later one's: rows blockIdx.y * 32 ..
// + 31 of its 256, a lane each, D / 8 values per warp; weights 2^(m_piece - M), pieces in CTA order. 64 registers: most of
// the grid's CTAs find nothing to join, and four of them fit an SM beside each other instead of two.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 4) combine_kernel(const Problem p) {
  pdl_wait();
  const CutItem c = p.cuts[blockIdx.x];
  if (c.n <= 1) return;
  const int half_tok = p.tok / 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int R = blockIdx.y * 32 + lane, t = R / kM, r = R % kM;
  const int tok = t * half_tok + r / p.G;
  if (r >= half_tok * p.G || tok >= c.ntok) return;
  constexpr size_t kPiece = 256 * (128 + 2);
  constexpr int kVec = D / 32;                 // float4 per lane
  constexpr int kAhead = 8 / kVec;             // pieces read at a time: most items have two or three
  // the first piece is CTA blockIdx.x's last (slot 1), the others are their CTAs' first (slot 0)
  auto piece = [&](int i) { return p.parts + (static_cast<size_t>(blockIdx.x + i) * 2 + (i == 0)) * kPiece; };
  float M = -INFINITY, L = 0.f;
  float4 acc[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < c.n; i0 += kAhead) {
    float pm[kAhead], pl[kAhead];
    float4 pv[kAhead][kVec];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* pc = piece(min(i0 + i, c.n - 1));
      pm[i] = pc[256 * D + R];
      pl[i] = i0 + i < c.n ? pc[256 * D + 256 + R] : 0.f;
#pragma unroll
      for (int v = 0; v < kVec; ++v) pv[i][v] = reinterpret_cast<const float4*>(pc)[(warp * kVec + v) * 256 + R];
    }
    float Mn = M;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (pl[i] != 0.f) Mn = fmaxf(Mn, pm[i]);  // a piece without a visible key counts for nothing
    const float a = L != 0.f ? exp2_approx(M - Mn) : 0.f;
    M = Mn;
    L *= a;
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v].x *= a, acc[v].y *= a, acc[v].z *= a, acc[v].w *= a;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (pl[i] == 0.f) continue;
      const float f = exp2_approx(pm[i] - M);
      L += f * pl[i];
#pragma unroll
      for (int v = 0; v < kVec; ++v)
        acc[v].x += f * pv[i][v].x, acc[v].y += f * pv[i][v].y, acc[v].z += f * pv[i][v].z, acc[v].w += f * pv[i][v].w;
    }
  }
  const bool sees = tok >= c.first;
  const float inv = 1.f / L;
  const long long row = c.row0 + tok;
  const int head = c.h * p.G + r % p.G;
  uint16_t* dst = p.out + row * p.o_st + head * p.o_sh + warp * (D / 8);
#pragma unroll
  for (int v = 0; v < kVec; v += 2) {
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (sees)
      w = make_uint4(pack2<BF16>(acc[v].x * inv, acc[v].y * inv), pack2<BF16>(acc[v].z * inv, acc[v].w * inv),
                     pack2<BF16>(acc[v + 1].x * inv, acc[v + 1].y * inv),
                     pack2<BF16>(acc[v + 1].z * inv, acc[v + 1].w * inv));
    *reinterpret_cast<uint4*>(dst + v * 4) = w;
  }
  if (p.lse != nullptr && warp == 0) p.lse[row * p.Hq + head] = sees ? M * kLn2 + logf(L) : -INFINITY;
}

template <int D, bool BF16>
int launch_tile(const Problem& p, const Source& src, int grid, cudaStream_t st) {
  using C = Cfg<D>;
  CUtensorMap mq, mk, mv_;
  const int box = src.box < kBN ? src.box : kBN;
  int rc = make_kv_maps(&mk, &mv_, src, p.Hkv, D, BF16, box, 1);
  if (rc == MV_OK) rc = make_q_map(&mq, p, D, BF16, p.tok / 2);
  if (rc != MV_OK) return rc;
  auto fn = may_be_long(p, src, kBN) ? tile_kernel<D, BF16, true> : tile_kernel<D, BF16, false>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(attention tile)");
  rc = launch_pdl(fn, dim3(grid), kThreads, C::kSmem, st, "attention tile launch", mq, mk, mv_, p, box);
  if (rc != MV_OK || !p.can_cut) return rc;
  return launch_pdl(combine_kernel<D, BF16>, dim3(grid, 8), 256, 0, st, "attention combine launch", p);
}

}  // namespace

int run_tile(Problem& p, const Source& src, int D, bool bf16, int grid, cudaStream_t st) {
  p.tok = 2 * (kM / p.G);
  // Short prompts are items of one to four tiles, where most of the time goes into beginning and finishing them: fewer cuts
  // (8 prompts, 2043 tokens: 24.1 us with 5 and 6, 25.9 with 2 and 3). Elsewhere cuts are worth more (24 sequences of a few
  // tokens over 2500 keys: 23.1 us with 2 and 3, 27.2 with 5 and 6; 9999 tokens in 5 prompts 190 and 197). The host knows the
  // mean length only, and of a paged cache not even that: a batch that it takes for the other kind is some us slower.
  const bool brief = p.page_table == nullptr && src.max_keys < 512ll * p.B;
  if (brief) cut_rule<5, 6>(p);
  else cut_rule<2, 3>(p);
  p.can_cut = src.max_keys > kBN;
  if (D == 128)
    return bf16 ? launch_tile<128, true>(p, src, grid, st) : launch_tile<128, false>(p, src, grid, st);
  return bf16 ? launch_tile<64, true>(p, src, grid, st) : launch_tile<64, false>(p, src, grid, st);
}

}  // namespace attn
}  // namespace mv
