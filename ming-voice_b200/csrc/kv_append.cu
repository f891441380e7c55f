// Appending to a paged cache with the position rotation on the way (mv_kv_append).
//
// Mathematics: each pair of a head's first rot_dim values is a point turned by its position's angle,
//   (a, b) -> (a cos - b sin, b cos + a sin), in fp32, rounded once to the element type; the rest is copied.
// Bound: memory (every value is read and written once). A lane owns the same 16 values (two 16-byte vectors) of
// several heads of one token, so a table row is read once per token and not once per head, and the vectors of all
// its heads are in flight together. Measured on a B200: 16001 tokens of 16 / 4 heads of 128, 205 MB, 35.3 us call after call
// (5.8 TB/s, 90 % of the measured copy; 34.3 us in a graph); one token 6.6 to 7.1 us as called, 2.8 us in a graph.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_common.cuh"
#include "common.cuh"

namespace mv {
namespace {

struct AppendArgs {
  const uint16_t *k, *v, *q;
  uint16_t *qo, *kc, *vc;
  long long k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh;
  long long kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  const int *page_table, *cu, *kv_lens, *positions;
  const float* cos_sin;
  long long pt_stride, cs_stride;
  int T, B, Hq, Hkv, max_pages, page_shift, num_pages, max_pos, rot;
  bool interleaved;
  WsHeader* ws;
};

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) return make_float2(bf16lo(w), bf16hi(w));
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return __half22float2(h);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The sequence that owns row t: the last b with cu[b] <= t (-1 if none, B when t lies behind the last sequence).
// The warp compares 32 boundaries at a time, so up to 32 sequences cost one load and up to 1024 two.
__device__ __forceinline__ int find_seq(const int* __restrict__ cu, int B, int t, int lane) {
  int lo = 0, n = B + 1;  // boundaries lo .. lo + n - 1 remain; cu[lo - 1] <= t
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int i = lane * step + step - 1;  // the last boundary of the lane's share
    const bool le = i < n && cu[lo + i] <= t;
    const int full = __popc(__ballot_sync(0xffffffffu, le));  // shares wholly <= t (cu ascends)
    lo += full * step;
    n = min(step - 1, max(0, n - full * step));
    if (step == 1) break;
  }
  return lo - 1;
}

// One warp per (token, group of heads). U = head_dim / 16 lanes share a head, 16 values each; a warp does 32 / U heads
// side by side, kBatch times. The heads of a token are numbered queries, keys, values.
constexpr int kBatch = 4;

template <int D, bool BF16>
__global__ void __launch_bounds__(128) kv_append_kernel(const AppendArgs a) {
  constexpr int U = D / 16, HL = 32 / U;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (t >= a.T) return;
  const int u = lane % U;
  const int nrot = a.rot / 16;
  const bool turn = u < nrot;
  // the lane's two vectors of 8: the two halves of 8 split pairs, or 16 neighbours (8 interleaved pairs, or a copy)
  const int v0 = (turn && !a.interleaved) ? u : 2 * u;
  const int v1 = (turn && !a.interleaved) ? u + nrot : 2 * u + 1;
  const int h0 = blockIdx.y * (HL * kBatch) + lane / U;
  const int n_heads = a.Hq + 2 * a.Hkv;

  // the data does not depend on where it goes: its loads start before the sequence is looked up
  uint4 x0[kBatch], x1[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int h = h0 + i * HL;
    if (h >= n_heads) break;
    const uint16_t* src = h < a.Hq           ? a.q + t * a.q_st + h * a.q_sh
                          : h < a.Hq + a.Hkv ? a.k + t * a.k_st + (h - a.Hq) * a.k_sh
                                             : a.v + t * a.v_st + (h - a.Hq - a.Hkv) * a.v_sh;
    x0[i] = *reinterpret_cast<const uint4*>(src + v0 * 8);
    x1[i] = *reinterpret_cast<const uint4*>(src + v1 * 8);
  }

  const int b = find_seq(a.cu, a.B, t, lane);
  if (b < 0 || b >= a.B) return;
  const int s = a.kv_lens[b] - (a.cu[b + 1] - t);
  const int s_page = s >> a.page_shift;
  bool ok = s >= 0 && s_page < a.max_pages;
  int page = 0, pos = s;
  if (ok) page = a.page_table[b * a.pt_stride + s_page];
  ok = ok && page >= 0 && page < a.num_pages;
  if (nrot > 0) {
    if (a.positions != nullptr) pos = a.positions[t];
    ok = ok && pos >= 0 && pos < a.max_pos;
  }
  if (!ok) {
    if (lane == 0) raise_error(a.ws, kErrBadPage, 0x700u);
    return;
  }
  float cs[8], sn[8];
  if (turn) {
    const float4* row = reinterpret_cast<const float4*>(a.cos_sin + pos * a.cs_stride + u * 8);
    const float4* row2 = row + a.rot / 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = row[i], d = row2[i];
      cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
      sn[4 * i] = d.x, sn[4 * i + 1] = d.y, sn[4 * i + 2] = d.z, sn[4 * i + 3] = d.w;
    }
  }
  const int slot = s & ((1 << a.page_shift) - 1);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int h = h0 + i * HL;
    if (h >= n_heads) break;
    uint16_t* dst = h < a.Hq           ? a.qo + t * a.qo_st + h * a.qo_sh
                    : h < a.Hq + a.Hkv ? a.kc + page * a.kc_sp + slot * a.kc_st + (h - a.Hq) * a.kc_sh
                                       : a.vc + page * a.vc_sp + slot * a.vc_st + (h - a.Hq - a.Hkv) * a.vc_sh;
    if (turn && h < a.Hq + a.Hkv) {
      uint32_t w0[4] = {x0[i].x, x0[i].y, x0[i].z, x0[i].w};
      uint32_t w1[4] = {x1[i].x, x1[i].y, x1[i].z, x1[i].w};
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = unpack2<BF16>(w0[j]), r = unpack2<BF16>(w1[j]);
          w0[j] = pack2<BF16>(p.x * cs[j] - p.y * sn[j], p.y * cs[j] + p.x * sn[j]);
          w1[j] = pack2<BF16>(r.x * cs[j + 4] - r.y * sn[j + 4], r.y * cs[j + 4] + r.x * sn[j + 4]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = unpack2<BF16>(w0[j]), r = unpack2<BF16>(w1[j]);
          const float c0 = cs[2 * j], c1 = cs[2 * j + 1], s0 = sn[2 * j], s1 = sn[2 * j + 1];
          w0[j] = pack2<BF16>(p.x * c0 - r.x * s0, p.y * c1 - r.y * s1);
          w1[j] = pack2<BF16>(r.x * c0 + p.x * s0, r.y * c1 + p.y * s1);
        }
      }
      x0[i] = make_uint4(w0[0], w0[1], w0[2], w0[3]);
      x1[i] = make_uint4(w1[0], w1[1], w1[2], w1[3]);
    }
    *reinterpret_cast<uint4*>(dst + v0 * 8) = x0[i];
    *reinterpret_cast<uint4*>(dst + v1 * 8) = x1[i];
  }
}

template <int D, bool BF16>
int launch(const AppendArgs& a, cudaStream_t st) {
  constexpr int per_warp = 32 / (D / 16) * kBatch;
  const dim3 grid((a.T + 3) / 4, (a.Hq + 2 * a.Hkv + per_warp - 1) / per_warp);
  return attn::launch_pdl(kv_append_kernel<D, BF16>, grid, 128, 0, st, "mv_kv_append launch", a);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" int mv_kv_append(const mv_kv_append_args* x, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "mv_kv_append";
  if (x == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const mv_paged_kv* c = x->cache;
  int rc = attn::check_cache(c, who);
  if (rc != MV_OK) return rc;
  const int T = x->T, B = x->B, Hq = x->Hq, rot = x->rot_dim, D = c->head_dim;
  if (T < 0 || B < 0 || x->max_pages < 0 || Hq < 0 || Hq > 4096)
    return fail(MV_ERR_INVALID, "%s: bad T=%d / B=%d / max_pages=%d / Hq=%d", who, T, B, x->max_pages, Hq);
  if (T == 0 || B == 0) return MV_OK;
  if (x->k == nullptr || x->v == nullptr || (Hq > 0 && (x->q == nullptr || x->q_out == nullptr)) ||
      x->cu_seqlens == nullptr || x->kv_lens == nullptr || (x->page_table == nullptr && x->max_pages > 0))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (rot < 0 || rot > D || rot % 16 != 0)
    return fail(MV_ERR_INVALID, "%s: rot_dim=%d must be a multiple of 16 in 0..%d", who, rot, D);
  if (rot > 0 && (x->cos_sin == nullptr || x->max_pos < 1 || (x->max_pos > 1 && x->cs_stride < rot)))
    return fail(MV_ERR_INVALID, "%s: rot_dim=%d needs a cos_sin table of rows >= rot_dim", who, rot);
  if (rot > 0 && (!aligned16(x->cos_sin) || (x->max_pos > 1 && x->cs_stride % 4 != 0)))
    return fail(MV_ERR_ALIGN, "%s: cos_sin rows must be 16-byte aligned", who);
  if (x->max_pages > 1 && x->pt_stride < x->max_pages && B > 1)
    return fail(MV_ERR_INVALID, "%s: page table row stride %lld shorter than max_pages=%d", who, x->pt_stride,
                x->max_pages);
  if ((rc = attn::check_rows(x->k, x->k_st, x->k_sh, c->n_kv_heads, T, D, "k", who)) != MV_OK) return rc;
  if ((rc = attn::check_rows(x->v, x->v_st, x->v_sh, c->n_kv_heads, T, D, "v", who)) != MV_OK) return rc;
  if (Hq > 0) {
    if ((rc = attn::check_rows(x->q, x->q_st, x->q_sh, Hq, T, D, "q", who)) != MV_OK) return rc;
    if ((rc = attn::check_rows(x->q_out, x->qo_st, x->qo_sh, Hq, T, D, "q_out", who)) != MV_OK) return rc;
  }
  if (workspace == nullptr || workspace_bytes < kWsHeaderBytes)
    return fail(MV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, kWsHeaderBytes);
  AppendArgs a{};
  a.k = static_cast<const uint16_t*>(x->k), a.v = static_cast<const uint16_t*>(x->v);
  a.q = static_cast<const uint16_t*>(x->q), a.qo = static_cast<uint16_t*>(x->q_out);
  a.kc = static_cast<uint16_t*>(c->k), a.vc = static_cast<uint16_t*>(c->v);
  a.k_st = x->k_st, a.k_sh = x->k_sh, a.v_st = x->v_st, a.v_sh = x->v_sh;
  a.q_st = x->q_st, a.q_sh = x->q_sh, a.qo_st = x->qo_st, a.qo_sh = x->qo_sh;
  a.kc_sp = c->k_sp, a.kc_st = c->k_st, a.kc_sh = c->k_sh;
  a.vc_sp = c->v_sp, a.vc_st = c->v_st, a.vc_sh = c->v_sh;
  a.page_table = x->page_table, a.cu = x->cu_seqlens, a.kv_lens = x->kv_lens, a.positions = x->positions;
  a.cos_sin = x->cos_sin, a.pt_stride = x->pt_stride, a.cs_stride = x->cs_stride;
  a.T = T, a.B = B, a.Hq = Hq, a.Hkv = c->n_kv_heads, a.max_pages = x->max_pages;
  a.page_shift = attn::log2_of(c->page_size), a.num_pages = c->num_pages, a.max_pos = x->max_pos;
  a.rot = rot, a.interleaved = x->interleaved != 0;
  a.ws = static_cast<WsHeader*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = c->dtype == MV_BF16;
  if (D == 128) return bf ? launch<128, true>(a, st) : launch<128, false>(a, st);
  return bf ? launch<64, true>(a, st) : launch<64, false>(a, st);
}
