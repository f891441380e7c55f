// Shared pieces of the attention kernels: the problem description, the split of its work over the CTAs, and the
// host's checks and tensor maps.
//
// Work split. The rows of a tile are `tok` consecutive tokens of one sequence times the G query heads of one key
// head (row = token * G + head): they read the same keys, so a key tile is loaded once for all of them. An item is
// (sequence, key head, token tile); its units are the key tiles of kBN keys that any of its rows sees. All units of
// all items, in order, form one sequence that is cut into one equal contiguous range per CTA, so every SM streams
// the same share of the cache whatever the lengths are, and nothing about the lengths has to be known on the host.
// An item cut by a range boundary leaves pieces (unnormalised fp32 output, running maximum and sum of each row),
// which are joined in CTA order: the result does not depend on the run.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "tc.cuh"

namespace mv {
namespace attn {

constexpr int kMaxB = 1024;      // sequences of one launch (more: several launches)
constexpr int kMaxCtas = 148;    // CTAs the workspace is laid out for: one per SM
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.442695040888963407f;

struct Problem {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  long long q_st, q_sh, o_st, o_sh;
  const int* cu_q;
  const int* cu_k;        // packed prompts: bounds of the keys; NULL for a paged cache
  const int* kv_lens;     // paged cache: lengths; NULL for packed prompts
  const int* page_table;  // NULL for packed prompts (the keys are one page of Tk rows)
  long long pt_stride;
  int max_pages, page_shift, num_pages;
  int B, T, Tk, Hq, Hkv, G;
  int tok;                // tokens of a tile
  int causal;
  int min_share;          // least units worth a CTA of their own
  float scale_log2;       // scale * log2(e): softmax in powers of two
  WsHeader* ws;
  unsigned int* counters;  // [kMaxCtas] arrivals of the split item that starts in a CTA's range (left zeroed)
  float* parts;            // [kMaxCtas][2] pieces
};

struct Seq {
  int q0, nq, k0, n;  // first query row, queries, first key row (packed prompts), keys
};

// What does not fit the tensors is clamped, so that no index derived from it leaves them. `report` names the fault.
__device__ __forceinline__ Seq seq_of(const Problem& p, int b, bool report) {
  Seq s;
  const int a0 = p.cu_q[b], a1 = p.cu_q[b + 1];
  s.q0 = min(max(a0, 0), p.T);
  s.nq = max(min(a1, p.T) - s.q0, 0);
  bool bad = s.q0 != a0 || s.q0 + s.nq != a1;
  if (p.kv_lens != nullptr) {
    const int n = p.kv_lens[b];
    s.k0 = 0;
    s.n = static_cast<int>(min(static_cast<long long>(max(n, 0)), static_cast<long long>(p.max_pages) << p.page_shift));
    bad = bad || s.n != n;
  } else {
    const int c0 = p.cu_k[b], c1 = p.cu_k[b + 1];
    s.k0 = min(max(c0, 0), p.Tk);
    s.n = max(min(c1, p.Tk) - s.k0, 0);
    bad = bad || s.k0 != c0 || s.k0 + s.n != c1;
  }
  if (bad && report) raise_error(p.ws, kErrBadSeq, static_cast<unsigned int>(b));
  return s;
}

// Keys seen by the last of tokens [0, end) of a sequence: the end of the item's key range.
__device__ __forceinline__ int keys_seen(const Problem& p, const Seq& s, int end) {
  return p.causal ? min(s.n, max(s.n - s.nq + end, 0)) : s.n;
}

template <int BN>
__device__ __forceinline__ int item_units(const Problem& p, const Seq& s, int t) {
  const int kend = keys_seen(p, s, min(s.nq, (t + 1) * p.tok));
  return max((kend + BN - 1) / BN, 1);  // an item without a visible key still has its rows to write
}

// Exclusive prefix sums of the sequences' units into pre[0 .. B], by all threads of the CTA; `tmp` [32].
template <int BN>
__device__ __forceinline__ void build_schedule(const Problem& p, unsigned long long* pre, unsigned long long* tmp) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = (nt + 31) / 32;
  unsigned long long carry = 0;
  for (int base = 0; base < p.B; base += nt) {
    const int b = base + tid;
    unsigned long long u = 0;
    if (b < p.B) {
      const Seq s = seq_of(p, b, blockIdx.x == 0);
      const int tiles = (s.nq + p.tok - 1) / p.tok;
      for (int t = 0; t < tiles; ++t) u += item_units<BN>(p, s, t);
      u *= p.Hkv;
    }
    unsigned long long x = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) tmp[warp] = x;
    __syncthreads();
    unsigned long long before = carry, all = carry;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before += tmp[w];
      all += tmp[w];
    }
    if (b < p.B) pre[b] = before + x - u;
    carry = all;
    __syncthreads();
  }
  if (tid == 0) pre[p.B] = carry;
  __syncthreads();
}

// a / b: a 64-bit division is a long subroutine, and nearly all counts here fit 32 bits
__device__ __forceinline__ unsigned long long quot(unsigned long long a, unsigned long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned int>(a) / static_cast<unsigned int>(b);
  return a / b;
}

// The CTAs' ranges: [bound(c), bound(c + 1)) of W units over the first `ctas` CTAs of the grid, the first `rest` of
// them one unit longer.
struct Cut {
  unsigned long long share;
  unsigned int ctas, rest;
  __device__ __forceinline__ Cut(unsigned long long W, int grid, int min_share) {
    ctas = static_cast<unsigned int>(min(quot(W + min_share - 1, min_share), static_cast<unsigned long long>(grid)));
    if (ctas == 0) ctas = 1;
    share = quot(W, ctas);
    rest = static_cast<unsigned int>(W - share * ctas);
  }
  __device__ __forceinline__ unsigned long long bound(unsigned int c) const {
    c = min(c, ctas);
    return c * share + min(c, rest);
  }
  // the CTA whose range holds unit x
  __device__ __forceinline__ unsigned int cta_of(unsigned long long x) const {
    const unsigned long long long_part = rest * (share + 1);
    if (x < long_part) return static_cast<unsigned int>(quot(x, share + 1));
    return rest + static_cast<unsigned int>(quot(x - long_part, share));
  }
};

// Walks the pieces of a CTA's range. Every role of the CTA walks on its own and sees the same pieces.
template <int BN>
struct Walk {
  const Problem& p;
  unsigned long long at, end;      // units of the range still to do
  unsigned long long item_start;   // unit at which the current item starts
  int b, h, t, units;
  Seq s;

  __device__ __forceinline__ Walk(const Problem& p_, const unsigned long long* pre, unsigned long long a,
                                  unsigned long long e)
      : p(p_), at(a), end(e), b(0), h(0), t(0), units(1) {
    if (at >= end) return;
    int lo = 0, hi = p.B - 1;  // the last sequence with pre[b] <= at (it has units: the next one starts behind at)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pre[mid] <= at) lo = mid; else hi = mid - 1;
    }
    b = lo;
    s = seq_of(p, b, false);
    const unsigned long long per_head = quot(pre[b + 1] - pre[b], p.Hkv);
    unsigned long long off = at - pre[b];
    h = static_cast<int>(quot(off, per_head));
    off -= per_head * h;
    for (t = 0;; ++t) {
      units = item_units<BN>(p, s, t);
      if (off < static_cast<unsigned long long>(units)) break;
      off -= units;
    }
    item_start = at - off;
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  __device__ __forceinline__ int first() const { return static_cast<int>(at - item_start); }
  __device__ __forceinline__ int last() const {  // one past the piece's last unit
    return static_cast<int>(min(end - item_start, static_cast<unsigned long long>(units)));
  }
  __device__ __forceinline__ int tok0() const { return t * p.tok; }
  __device__ __forceinline__ int ntok() const { return min(p.tok, s.nq - t * p.tok); }
  __device__ __forceinline__ int kend() const { return keys_seen(p, s, min(s.nq, (t + 1) * p.tok)); }
  __device__ __forceinline__ bool whole() const { return first() == 0 && last() == units; }
  __device__ __forceinline__ void next() {
    at = item_start + last();
    if (at >= end) return;
    item_start = at;
    if ((t + 1) * p.tok < s.nq) {
      ++t;
    } else {
      t = 0;
      if (++h == p.Hkv) {
        h = 0;
        do {
          s = seq_of(p, ++b, false);
        } while (s.nq == 0);
      }
    }
    units = item_units<BN>(p, s, t);
  }
};

// Bounded wait, in line: a call would hold the caller's registers to the calling convention.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, WsHeader* h, unsigned int info) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      raise_error(h, kErrTimeout, info);
      return false;
    }
  return true;
}

// A producer warp's view of the page table: lane x holds the page of box x of the tile at hand, and the next tile's
// are on their way while this one's copies are issued (a table read between any two tiles would cost an L2 latency
// each). Packed prompts are one page.
struct Pages {
  int ids, next;
  // lane x: the page of the box that holds keys [j, j + box) of sequence b (j < kend), as read from the table
  __device__ __forceinline__ static int read(const Problem& p, int b, int j, int kend) {
    return p.page_table != nullptr && j < kend ? p.page_table[b * p.pt_stride + (j >> p.page_shift)] : 0;
  }
  // takes over the ids read ahead. One outside the cache is reported and becomes num_pages, which lies outside the
  // tensor map and reads as zeros.
  __device__ __forceinline__ void step(const Problem& p, unsigned int info) {
    ids = next;
    if (p.page_table != nullptr && (ids < 0 || ids >= p.num_pages)) {
      raise_error(p.ws, kErrBadPage, info);
      ids = p.num_pages;
    }
  }
  __device__ __forceinline__ int of(int box) const { return __shfl_sync(0xffffffffu, ids, box); }
};

// Value conversions of the element types
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------------------ host

inline int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// a [rows, heads, d] tensor's pointer and strides: 16-byte vectors and tensor maps need 16-byte steps
int check_rows(const void* p, long long st, long long sh, int heads, int rows, int d, const char* name,
               const char* who);
int check_cache(const mv_paged_kv* c, const char* who);

// Where keys and values lie: `pages` pages of `tokens` rows (packed prompts: one page), copies of `box` rows at most.
struct Source {
  const void *k, *v;
  long long k_st, k_sh, k_sp, v_st, v_sh, v_sp;
  int tokens, pages, box;
};

// 5-D maps over keys and values [page][head][64-value part of a head][token][64 values], 128-byte swizzle, box of
// 64 values x `box` tokens x `parts` parts: in shared memory [part][token][64 values]
int make_kv_maps(CUtensorMap* mk, CUtensorMap* mv_, const Source& src, int heads, int d, bool bf16, int box, int parts);

// 3-D map over queries [token][head][d], 128-byte swizzle, box of 64 values x the G heads of a key head x `tok` tokens
int make_q_map(CUtensorMap* m, const Problem& p, int d, bool bf16, int tok);

}  // namespace attn
}  // namespace mv
