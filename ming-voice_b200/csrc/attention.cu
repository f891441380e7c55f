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
                    long long sh, long long sp, int box, const char* what) {
  auto enc = encode_fn();
  if (enc == nullptr) return fail(MV_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  // the stride of an axis of one element is never used: a valid one stands in for it
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(tokens),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(tokens > 1 ? st : d) * 2,
                                 static_cast<cuuint64_t>(heads > 1 ? sh : d) * 2,
                                 static_cast<cuuint64_t>(pages > 1 ? sp : d) * 2};
  const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(MV_ERR_INVALID, "tensor map for %s rejected (CUresult %d)", what, static_cast<int>(r));
  return MV_OK;
}

int make_kv_maps(CUtensorMap* mk, CUtensorMap* mv_, const Source& s, int heads, int d, bool bf16, int box) {
  const int rc = make_map(mk, s.k, bf16, d, s.tokens, heads, s.pages, s.k_st, s.k_sh, s.k_sp, box, "k");
  if (rc != MV_OK) return rc;
  return make_map(mv_, s.v, bf16, d, s.tokens, heads, s.pages, s.v_st, s.v_sh, s.v_sp, box, "v");
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

constexpr size_t kCountersBytes = 1024 + kMaxCtas * 32;                     // arrival counters, cut items
constexpr size_t kPartsBytes = size_t(kMaxCtas) * 2 * 256 * (128 + 2) * 4;  // two pieces of 256 rows per CTA

int run(Problem& p, const Source& src, int D, int dtype, int B, const int* cu_q, const int* cu_k, const int* kv_lens,
        int max_q, float scale, void* workspace, size_t workspace_bytes, cudaStream_t st, const char* who) {
  if (!(scale > 0.f) || scale > 3.0e38f) return fail(MV_ERR_INVALID, "%s: scale must be positive and finite", who);
  if (p.Hq < 1 || p.Hq % p.Hkv != 0 || p.Hq / p.Hkv > 64)
    return fail(MV_ERR_INVALID, "%s: Hq=%d must be 1..64 times Hkv=%d", who, p.Hq, p.Hkv);
  if (workspace == nullptr || workspace_bytes < mv_attention_workspace_bytes() ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(MV_ERR_WORKSPACE, "%s: 256-byte aligned workspace of %zu bytes needed", who,
                mv_attention_workspace_bytes());
  p.G = p.Hq / p.Hkv;
  p.scale_log2 = scale * kLog2e;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.ws = reinterpret_cast<WsHeader*>(ws);
  p.counters = reinterpret_cast<unsigned int*>(ws + kWsHeaderBytes);
  p.parts = reinterpret_cast<float*>(ws + kWsHeaderBytes + kCountersBytes);
  const bool bf16 = dtype == MV_BF16;
  int grid = num_sms();
  if (grid > kMaxCtas) grid = kMaxCtas;
  int rc = MV_OK;
  const long long pt_row = p.pt_stride;
  const int* table = p.page_table;
  const int rows = max_q > 0 && max_q < 64 ? max_q * p.G : 64 * p.G;
  for (int b0 = 0; b0 < B; b0 += kMaxB) {
    p.B = B - b0 < kMaxB ? B - b0 : kMaxB;
    p.cu_q = cu_q + b0;
    p.cu_k = cu_k == nullptr ? nullptr : cu_k + b0;
    p.kv_lens = kv_lens == nullptr ? nullptr : kv_lens + b0;
    p.page_table = table == nullptr ? nullptr : table + b0 * pt_row;
    rc = rows <= 32 ? run_split(p, src, D, bf16, rows, grid, st) : run_tile(p, src, D, bf16, grid, st);
    if (rc != MV_OK) return rc;
  }
  return MV_OK;
}

}  // namespace
}  // namespace attn
}  // namespace mv

using namespace mv;
using namespace mv::attn;

extern "C" size_t mv_attention_workspace_bytes(void) { return kWsHeaderBytes + kCountersBytes + kPartsBytes; }

extern "C" int mv_paged_attention(const mv_paged_kv* c, const void* q, long long q_st, long long q_sh, int Hq, int T,
                                  const int* page_table, long long pt_stride, int max_pages, const int* cu_seqlens,
                                  const int* kv_lens, int B, int max_q, float scale, int causal, void* out,
                                  long long o_st, long long o_sh, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* who = "mv_paged_attention";
  int rc = check_cache(c, who);
  if (rc != MV_OK) return rc;
  if (T < 0 || B < 0 || max_pages < 0 || max_q < 0)
    return fail(MV_ERR_INVALID, "%s: bad T=%d / B=%d / max_pages=%d / max_q=%d", who, T, B, max_pages, max_q);
  if (T == 0 || B == 0) return MV_OK;
  if (q == nullptr || out == nullptr || cu_seqlens == nullptr || kv_lens == nullptr || page_table == nullptr)
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  if (max_pages > 1 && B > 1 && pt_stride < max_pages)
    return fail(MV_ERR_INVALID, "%s: page table row stride %lld shorter than max_pages=%d", who, pt_stride, max_pages);
  if ((rc = check_rows(q, q_st, q_sh, Hq, T, c->head_dim, "q", who)) != MV_OK) return rc;
  if ((rc = check_rows(out, o_st, o_sh, Hq, T, c->head_dim, "out", who)) != MV_OK) return rc;
  Problem p{};
  p.q = static_cast<const uint16_t*>(q), p.out = static_cast<uint16_t*>(out), p.lse = lse;
  p.q_st = q_st, p.q_sh = q_sh, p.o_st = o_st, p.o_sh = o_sh;
  p.page_table = page_table, p.pt_stride = pt_stride, p.max_pages = max_pages;
  p.page_shift = log2_of(c->page_size), p.num_pages = c->num_pages;
  p.T = T, p.Hq = Hq, p.Hkv = c->n_kv_heads, p.causal = causal != 0;
  const Source src{c->k, c->v, c->k_st, c->k_sh, c->k_sp, c->v_st, c->v_sh, c->v_sp, c->page_size, c->num_pages,
                   c->page_size};
  return run(p, src, c->head_dim, c->dtype, B, cu_seqlens, nullptr, kv_lens, max_q, scale, workspace, workspace_bytes,
             static_cast<cudaStream_t>(stream), who);
}

extern "C" int mv_prompt_attention(const void* q, long long q_st, long long q_sh, const void* k, long long k_st,
                                   long long k_sh, const void* v, long long v_st, long long v_sh, int dtype, int Tq,
                                   int Tk, int Hq, int Hkv, int head_dim, const int* cu_seqlens,
                                   const int* cu_seqlens_k, int B, int max_q, float scale, int causal, void* out,
                                   long long o_st, long long o_sh, float* lse, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const char* who = "mv_prompt_attention";
  if (dtype != MV_BF16 && dtype != MV_F16) return fail(MV_ERR_UNSUPPORTED, "%s: tensors must be bf16 or f16", who);
  if (head_dim != 64 && head_dim != 128) return fail(MV_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, head_dim);
  if (Tq < 0 || Tk < 0 || B < 0 || max_q < 0 || Hkv < 1 || Hkv > 4096)
    return fail(MV_ERR_INVALID, "%s: bad Tq=%d / Tk=%d / B=%d / max_q=%d / Hkv=%d", who, Tq, Tk, B, max_q, Hkv);
  if (Tq == 0 || B == 0) return MV_OK;
  if (q == nullptr || out == nullptr || cu_seqlens == nullptr || (Tk > 0 && (k == nullptr || v == nullptr)))
    return fail(MV_ERR_INVALID, "%s: null pointer", who);
  int rc = check_rows(q, q_st, q_sh, Hq, Tq, head_dim, "q", who);
  if (rc == MV_OK) rc = check_rows(out, o_st, o_sh, Hq, Tq, head_dim, "out", who);
  if (rc == MV_OK && Tk > 0) rc = check_rows(k, k_st, k_sh, Hkv, Tk, head_dim, "k", who);
  if (rc == MV_OK && Tk > 0) rc = check_rows(v, v_st, v_sh, Hkv, Tk, head_dim, "v", who);
  if (rc != MV_OK) return rc;
  Problem p{};
  p.q = static_cast<const uint16_t*>(q), p.out = static_cast<uint16_t*>(out), p.lse = lse;
  p.q_st = q_st, p.q_sh = q_sh, p.o_st = o_st, p.o_sh = o_sh;
  p.T = Tq, p.Tk = Tk, p.Hq = Hq, p.Hkv = Hkv, p.causal = causal != 0;
  // without a key every row is empty and no copy runs: the maps then stand on one row of q
  const Source src = Tk > 0 ? Source{k, v, k_st, k_sh, 0, v_st, v_sh, 0, Tk, 1, 64}
                            : Source{q, q, head_dim, head_dim, 0, head_dim, head_dim, 0, 1, 1, 64};
  return run(p, src, head_dim, dtype, B, cu_seqlens, cu_seqlens_k != nullptr ? cu_seqlens_k : cu_seqlens, nullptr,
             max_q, scale, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), who);
}
