// Entry points of attention over the paged cache and over packed prompts: argument checks, tensor maps, the choice of
// the kernel.
#include "attn_common.cuh"

namespace mv {
namespace attn {

int check_rows(const void* p, long long st, long long sh, int heads, int rows, int d, const char* name,
               const char* who) {
  if (!aligned16(p) || (rows > 1 && st % 8 != 0) || (heads > 1 && sh % 8 != 0))
    return fail(MV_ERR_ALIGN, "%s: %s must be 16-byte aligned with row and head strides of whole 16 bytes", who, name);
  if ((rows > 1 && st < d) || (heads > 1 && sh < d))
    return fail(MV_ERR_INVALID, "%s: %s has a row or head stride shorter than head_dim=%d", who, name, d);
  return MV_OK;
}

int check_cache(const mv_paged_kv* c, const char* who) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr) return fail(MV_ERR_INVALID, "%s: null cache", who);
  if (c->dtype != MV_BF16 && c->dtype != MV_F16)
    return fail(MV_ERR_UNSUPPORTED, "%s: the cache must be bf16 or f16", who);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(MV_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, c->head_dim);
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(MV_ERR_UNSUPPORTED, "%s: page_size=%d must be a power of two in 8..256", who, c->page_size);
  if (c->num_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 4096)
    return fail(MV_ERR_INVALID, "%s: bad num_pages=%d / n_kv_heads=%d", who, c->num_pages, c->n_kv_heads);
  int rc = check_rows(c->k, c->k_st, c->k_sh, c->n_kv_heads, c->page_size, c->head_dim, "cache k", who);
  if (rc == MV_OK) rc = check_rows(c->v, c->v_st, c->v_sh, c->n_kv_heads, c->page_size, c->head_dim, "cache v", who);
  if (rc != MV_OK) return rc;
  if (c->num_pages > 1 && (c->k_sp % 8 != 0 || c->v_sp % 8 != 0))
    return fail(MV_ERR_ALIGN, "%s: cache page strides must be whole 16 bytes", who);
  if (c->num_pages > 1 && (c->k_sp < c->head_dim || c->v_sp < c->head_dim))
    return fail(MV_ERR_INVALID, "%s: cache page stride shorter than head_dim", who);
  return MV_OK;
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

static int make_map(CUtensorMap* m, const void* base, bool bf16, int d, int tokens, int heads, int pages, long long st,
                    long long sh, long long sp, int box, int parts, const char* what) {
  auto enc = encode_fn();
  if (enc == nullptr) return fail(MV_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  // the stride of an axis of one element is never used: a valid one stands in for it
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(d / 64),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(tokens > 1 ? st : d) * 2, 128,
                                 static_cast<cuuint64_t>(heads > 1 ? sh : d) * 2,
                                 static_cast<cuuint64_t>(pages > 1 ? sp : d) * 2};
  const cuuint32_t boxes[5] = {64, static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(parts), 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                         const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B,
                         // a head's row and no more: with 128-byte rows, 256 bytes would fetch the next head's too
                         d == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(MV_ERR_INVALID, "tensor map for %s rejected (CUresult %d)", what, static_cast<int>(r));
  return MV_OK;
}

int make_kv_maps(CUtensorMap* mk, CUtensorMap* mv_, const Source& s, int heads, int d, bool bf16, int box, int parts) {
  const int rc = make_map(mk, s.k, bf16, d, s.tokens, heads, s.pages, s.k_st, s.k_sh, s.k_sp, box, parts, "k");
  if (rc != MV_OK) return rc;
  return make_map(mv_, s.v, bf16, d, s.tokens, heads, s.pages, s.v_st, s.v_sh, s.v_sp, box, parts, "v");
}

int make_q_map(CUtensorMap* m, const Problem& p, int d, bool bf16, int tok) {
  auto enc = encode_fn();
  if (enc == nullptr) return fail(MV_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(p.Hq), static_cast<cuuint64_t>(p.T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.Hq > 1 ? p.q_sh : d) * 2,
                                 static_cast<cuuint64_t>(p.T > 1 ? p.q_st : d) * 2};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(tok)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<uint16_t*>(p.q), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MV_ERR_INVALID, "tensor map for q rejected (CUresult %d)", static_cast<int>(r));
  return MV_OK;
}

int run_split(Problem& p, const Source& src, int D, bool bf16, int rows_hint, int grid, cudaStream_t st);
int run_tile(Problem& p, const Source& src, int D, bool bf16, int grid, cudaStream_t st);

namespace {

constexpr size_t kCutsBytes = (kMaxCtas * sizeof(CutItem) + 255) / 256 * 256;
constexpr size_t kPartsBytes = size_t(kMaxCtas) * 2 * 256 * (128 + 2) * 4;  // two pieces of 256 rows per CTA

// The shared part of the two entry points: `src` describes the keys, D / dtype / Hkv their heads.
int run(const mv_attention_args* a, const Source& src, int D, int dtype, int Hkv, void* workspace,
        size_t workspace_bytes, cudaStream_t st, const char* who) {
  if (!(a->scale > 0.f) || a->scale > 3.0e38f)
    return fail(MV_ERR_INVALID, "%s: scale must be positive and finite", who);
  if (a->Hq < 1 || a->Hq % Hkv != 0 || a->Hq / Hkv > 64)
    return fail(MV_ERR_INVALID, "%s: Hq=%d must be 1..64 times Hkv=%d", who, a->Hq, Hkv);
  int rc = check_rows(a->q, a->q_st, a->q_sh, a->Hq, a->T, D, "q", who);
  if (rc == MV_OK) rc = check_rows(a->out, a->o_st, a->o_sh, a->Hq, a->T, D, "out", who);
  if (rc != MV_OK) return rc;
  if (workspace == nullptr || workspace_bytes < mv_attention_workspace_bytes() ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(MV_ERR_WORKSPACE, "%s: 256-byte aligned workspace of %zu bytes needed", who,
                mv_attention_workspace_bytes());
  const bool paged = a->cache != nullptr;
  Problem p{};
  p.q = static_cast<const uint16_t*>(a->q), p.out = static_cast<uint16_t*>(a->out), p.lse = a->lse;
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.T = a->T, p.Tk = a->Tk, p.Hq = a->Hq, p.Hkv = Hkv, p.G = a->Hq / Hkv, p.causal = a->causal != 0;
  p.scale_log2 = a->scale * kLog2e;
  if (paged) {
    p.max_pages = a->max_pages, p.pt_stride = a->pt_stride;
    p.page_shift = log2_of(src.tokens), p.num_pages = src.pages;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.ws = reinterpret_cast<WsHeader*>(ws);
  p.cuts = reinterpret_cast<CutItem*>(ws + kWsHeaderBytes);
  p.parts = reinterpret_cast<float*>(ws + kWsHeaderBytes + kCutsBytes);
  const bool bf16 = dtype == MV_BF16;
  int grid = num_sms();
  if (grid > kMaxCtas) grid = kMaxCtas;
  const int* cu_k = a->cu_seqlens_k != nullptr ? a->cu_seqlens_k : a->cu_seqlens;
  const int rows = a->max_q > 0 && a->max_q < 64 ? a->max_q * p.G : 64 * p.G;
  for (int b0 = 0; b0 < a->B; b0 += kMaxB) {
    p.B = a->B - b0 < kMaxB ? a->B - b0 : kMaxB;
    p.cu_q = a->cu_seqlens + b0;
    if (paged) {
      p.kv_lens = a->kv_lens + b0;
      p.page_table = a->page_table + b0 * a->pt_stride;
    } else {
      p.cu_k = cu_k + b0;
    }
    // the few-row kernel up to 16 rows per key head, the 128-row kernel above (attn_split.cu has both sides measured)
    rc = rows <= 16 ? run_split(p, src, D, bf16, rows, grid, st) : run_tile(p, src, D, bf16, grid, st);
    if (rc != MV_OK) return rc;
  }
  return MV_OK;
}

}  // namespace
}  // namespace attn
}  // namespace mv

using namespace mv;
using namespace mv::attn;

extern "C" size_t mv_attention_workspace_bytes(void) { return kWsHeaderBytes + kCutsBytes + kPartsBytes; }

extern "C" int mv_paged_attention(const mv_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "mv_paged_attention";
  if (a == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const mv_paged_kv* c = a->cache;
  const int rc = check_cache(c, who);
  if (rc != MV_OK) return rc;
  if (a->T < 0 || a->B < 0 || a->max_pages < 0 || a->max_q < 0)
    return fail(MV_ERR_INVALID, "%s: bad T=%d / B=%d / max_pages=%d / max_q=%d", who, a->T, a->B, a->max_pages,
                a->max_q);
  if (a->T == 0 || a->B == 0) return MV_OK;
  if (a->q == nullptr || a->out == nullptr || a->cu_seqlens == nullptr || a->kv_lens == nullptr ||
      (a->page_table == nullptr && a->max_pages > 0))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (a->max_pages > 1 && a->B > 1 && a->pt_stride < a->max_pages)
    return fail(MV_ERR_INVALID, "%s: page table row stride %lld shorter than max_pages=%d", who, a->pt_stride,
                a->max_pages);
  const Source src{c->k, c->v, c->k_st, c->k_sh, c->k_sp, c->v_st, c->v_sh, c->v_sp, c->page_size, c->num_pages,
                   c->page_size, static_cast<long long>(a->max_pages) * c->page_size};
  return run(a, src, c->head_dim, c->dtype, c->n_kv_heads, workspace, workspace_bytes,
             static_cast<cudaStream_t>(stream), who);
}

extern "C" int mv_prompt_attention(const mv_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "mv_prompt_attention";
  if (a == nullptr) return fail(MV_ERR_INVALID, "%s: null pointer", who);
  const int D = a->head_dim;
  if (a->cache != nullptr) return fail(MV_ERR_INVALID, "%s: cache must be NULL", who);
  if (a->dtype != MV_BF16 && a->dtype != MV_F16)
    return fail(MV_ERR_UNSUPPORTED, "%s: tensors must be bf16 or f16", who);
  if (D != 64 && D != 128) return fail(MV_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, D);
  if (a->T < 0 || a->Tk < 0 || a->B < 0 || a->max_q < 0 || a->Hkv < 1 || a->Hkv > 4096)
    return fail(MV_ERR_INVALID, "%s: bad T=%d / Tk=%d / B=%d / max_q=%d / Hkv=%d", who, a->T, a->Tk, a->B, a->max_q,
                a->Hkv);
  if (a->T == 0 || a->B == 0) return MV_OK;
  if (a->q == nullptr || a->out == nullptr || a->cu_seqlens == nullptr ||
      (a->Tk > 0 && (a->k == nullptr || a->v == nullptr)))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (a->Tk > 0) {
    int rc = check_rows(a->k, a->k_st, a->k_sh, a->Hkv, a->Tk, D, "k", who);
    if (rc == MV_OK) rc = check_rows(a->v, a->v_st, a->v_sh, a->Hkv, a->Tk, D, "v", who);
    if (rc != MV_OK) return rc;
  }
  // without a key every row is empty and no copy runs: the maps then stand on one row of q
  const Source src = a->Tk > 0 ? Source{a->k, a->v, a->k_st, a->k_sh, 0, a->v_st, a->v_sh, 0, a->Tk, 1, 128, a->Tk}
                               : Source{a->q, a->q, D, D, 0, D, D, 0, 1, 1, 128, 0};
  return run(a, src, D, a->dtype, a->Hkv, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), who);
}
