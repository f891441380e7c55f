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
constexpr unsigned int kMaxUnits = 0x7fffffffu;  // sums of units stop here: two of them still add up in 32 bits
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
  int extra;              // units an item counts besides its key tiles
  int min_share;          // least units worth a CTA of their own
  bool can_cut;           // an item may have more than one tile, so that the joining kernel is needed
  float scale_log2;       // scale * log2(e): softmax in powers of two
  WsHeader* ws;
  struct CutItem* cuts;  // [kMaxCtas]
  float* parts;          // [kMaxCtas][2] pieces: slot 1 starts its item, slot 0 starts inside it
};

// The cut rule of a launch. A range is then never shorter than `extra`, so that of two cuts one at most lies within the last
// `extra` units of an item: there it moves to the item's end, and last_cta() names the range before it. (A shorter range could
// move two cuts to the same end. A range may still be left empty, by cuts that move to both of its ends.)
template <int kExtra, int kMinShare>
inline void cut_rule(Problem& p) {
  static_assert(kMinShare >= kExtra, "two cuts could move to one end");
  p.extra = kExtra;
  p.min_share = kMinShare;
}

// What the joining kernel needs of a cut item, left by the CTA whose range holds its start; written by every CTA.
struct CutItem {
  int n;         // pieces: this CTA's and those of the n - 1 next (0: no item is cut behind its start here)
  int row0;      // first token's row
  int ntok;      // tokens
  int h;         // key head
  int first;     // first token that sees a key
  int pad[3];
};
static_assert(sizeof(CutItem) == 32, "");

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

// Key tiles of token tile t; at least one, as an item without a visible key still has its rows to write.
template <int BN>
__device__ __forceinline__ int item_tiles(const Problem& p, const Seq& s, int t) {
  return max((keys_seen(p, s, min(s.nq, (t + 1) * p.tok)) + BN - 1) / BN, 1);
}

// sum of floor((a i + b) / m) over 0 <= i < n (a, b >= 0): the number of lattice points (i, y), y >= 1, on or under the line
// (a i + b) / m. Whole multiples of m in a and b are counted outright; then both are below m, and the points are counted along
// y instead, where the line's slope is m / a: the pair (m, a) shrinks as in Euclid's algorithm. (The reciprocity of such sums:
// Graham, Knuth, Patashnik, Concrete Mathematics, section 3.5.)
__device__ __forceinline__ unsigned int floor_sum(unsigned int n, unsigned int m, unsigned int a, unsigned int b) {
  unsigned int sum = 0;
  while (n > 0) {
    sum += (n * (n - 1) / 2) * (a / m) + n * (b / m);
    a %= m, b %= m;
    const unsigned int top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const unsigned int t = m;
    m = a, a = t;
  }
  return sum;
}

// Units of all token tiles of one key head of a sequence.
template <int BN>
__device__ __forceinline__ unsigned int head_units(const Problem& p, const Seq& s) {
  const int tiles = (s.nq + p.tok - 1) / p.tok;
  if (tiles == 0) return 0;
  const unsigned int last = item_tiles<BN>(p, s, tiles - 1);
  if (!p.causal) return tiles * (last + p.extra);
  // tile t < tiles - 1 sees c + (t + 1) tok keys; the first `ones` of them at most BN
  const int c = s.n - s.nq;
  const int ones = min(tiles - 1, max(0, (BN - c) / p.tok));
  const int rest = tiles - 1 - ones;
  unsigned int u = last + ones + tiles * p.extra;
  if (rest > 0) u += floor_sum(rest, BN, p.tok, c + (ones + 1) * p.tok + BN - 1);
  return u;
}

// Exclusive prefix sums of the sequences' units (kByItem: items) into pre[0 .. B], by all threads of the CTA; `tmp` [32].
// Returns whether they fit 32 bits (pre[B] is 0 otherwise).
template <int BN, bool kByItem>
__device__ __forceinline__ bool prefix_units(const Problem& p, unsigned int* pre, unsigned int* tmp) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = (nt + 31) / 32;
  unsigned int carry = 0;
  for (int base = 0; base < p.B; base += nt) {
    const int b = base + tid;
    unsigned int u = 0;
    if (b < p.B) {
      const Seq s = seq_of(p, b, blockIdx.x == 0);
      const unsigned long long items = static_cast<unsigned long long>((s.nq + p.tok - 1) / p.tok) * p.Hkv;
      const unsigned long long most = kByItem ? items : items * ((s.n + BN - 1) / BN + 1 + p.extra);
      u = most >= kMaxUnits ? kMaxUnits : kByItem ? static_cast<unsigned int>(items) : head_units<BN>(p, s) * p.Hkv;
    }
    unsigned int x = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = min(x + y, kMaxUnits);
    }
    if (lane == 31) tmp[warp] = x;
    __syncthreads();
    unsigned int before = carry, all = carry;
    const int used = min(nw, (p.B - base + 31) / 32);  // warps that hold a sequence
    for (int w = 0; w < used; ++w) {
      if (w < warp) before = min(before + tmp[w], kMaxUnits);
      all = min(all + tmp[w], kMaxUnits);
    }
    if (b < p.B) pre[b] = before + x - u;
    carry = all;
    if (base + nt < p.B) __syncthreads();
  }
  if (tid == 0) pre[p.B] = carry < kMaxUnits ? carry : 0;
  __syncthreads();
  return carry < kMaxUnits;
}

// The schedule into pre[0 .. B]. All sequences of a launch share 32 bits of units, whatever part of them each takes. kLong, for
// launches whose tensors could hold more work than that (3 s and more of it): where the lengths do, an item counts as one unit, is
// not cut, and the CTAs share the items by number. (pre[B + 1] tells; items fit, as each has query rows of its own.) Bounds that
// do not ascend can claim rows many times over: where their sum does not fit nothing is computed, and that is reported.
template <int BN, bool kLong>
__device__ __forceinline__ void build_schedule(const Problem& p, unsigned int* pre, unsigned int* tmp) {
  bool fits = prefix_units<BN, false>(p, pre, tmp);
  if (kLong) {
    const bool by_item = !fits;
    if (by_item) fits = prefix_units<BN, true>(p, pre, tmp);
    if (threadIdx.x == 0) pre[p.B + 1] = by_item;
    __syncthreads();
  }
  if (!fits && threadIdx.x == 0 && blockIdx.x == 0) raise_error(p.ws, kErrOverflow, 0x701u);
}

// The CTAs' ranges [bound(c), bound(c + 1)) of the W units, bound(c) = floor(W c / ctas), before cuts move to nearby ends
// of items.
struct Cut {
  unsigned int W, ctas, share, rest;  // ctas: CTAs of the grid that have a range; W = share ctas + rest
  __device__ __forceinline__ Cut(const Problem& p, unsigned int total, bool by_item, int grid) {
    W = total;
    ctas = min(by_item ? W : W / p.min_share, static_cast<unsigned int>(grid));
    // one sequence: its heads' items are alike, and so many cuts for each fall on their ends
    if (p.B == 1 && ctas > p.Hkv) ctas -= ctas % p.Hkv;
    if (ctas == 0) ctas = 1;
    share = W / ctas;
    rest = W - share * ctas;
  }
  __device__ __forceinline__ unsigned int bound(unsigned int c) const {
    c = min(c, ctas);
    return c * share + c * rest / ctas;
  }
  // the CTA whose range holds unit x: the estimate in floats is off by one at most
  __device__ __forceinline__ unsigned int cta_of(unsigned int x) const {
    unsigned int c = min(static_cast<unsigned int>((static_cast<float>(x) + 0.5f) * ctas / W), ctas - 1);
    if (c > 0 && bound(c) > x) --c;
    if (bound(c + 1) <= x) ++c;
    return c;
  }
};

// Walks the pieces of a CTA's range, warp by warp: every warp of the CTA walks on its own and sees the same pieces.
template <int BN, bool kLong>
struct Walk {
  const Problem& p;
  const unsigned int* pre;
  unsigned int end;                // end of the range
  unsigned int start;              // unit at which the current item starts
  int b, h, t, tiles;
  int i0, i1;                      // the piece: key tiles [i0, i1) of the item's `tiles`
  bool live;
  Seq s;

  __device__ __forceinline__ Walk(const Problem& p_, const unsigned int* pre_, const Cut& cut, unsigned int c)
      : p(p_), pre(pre_), end(cut.bound(c + 1)), start(cut.bound(c)), b(0), h(0), t(0), tiles(1), i0(0), i1(0) {
    live = start < end;
    if (!live) return;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = p.B - 1;  // the last sequence with pre[b] <= start (it has units: the next starts behind it)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pre[mid] <= start) lo = mid; else hi = mid - 1;
    }
    b = lo;
    s = seq_of(p, b, false);
    const unsigned int per_head = (pre[b + 1] - pre[b]) / p.Hkv;
    unsigned int off = start - pre[b];
    h = static_cast<int>(off / per_head);
    off -= per_head * h;
    int n_t = (s.nq + p.tok - 1) / p.tok;
    if (by_item()) n_t = 1, t = static_cast<int>(off), off = 0;
    for (int t0 = 0; n_t > 1; t0 += 32) {  // 32 token tiles at a time
      const unsigned int u = t0 + lane < n_t ? item_tiles<BN>(p, s, t0 + lane) + p.extra : 0;
      unsigned int x = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned int over = __ballot_sync(0xffffffffu, x > off);
      if (over) {
        const int l = __ffs(over) - 1;
        t = t0 + l;
        off -= __shfl_sync(0xffffffffu, x, l) - __shfl_sync(0xffffffffu, u, l);
        break;
      }
      off -= __shfl_sync(0xffffffffu, x, 31);
    }
    tiles = item_tiles<BN>(p, s, t);
    start -= off;
    // the range's first cut, moved to an end of the item if that is near
    const int o = static_cast<int>(off);
    if (o > p.extra && tiles + p.extra - o <= p.extra) {
      advance();
    } else {
      i0 = o <= p.extra ? 0 : o - p.extra;
      finish();
    }
  }
  __device__ __forceinline__ bool by_item() const { return kLong && pre[p.B + 1] != 0; }
  __device__ __forceinline__ unsigned int units() const { return by_item() ? 1u : tiles + p.extra; }
  // the piece's end: the item's, or the range's where that lies well inside the item
  __device__ __forceinline__ void finish() {
    i1 = tiles;
    if (end < start + units()) {
      const int o = static_cast<int>(end > start ? end - start : 0);
      if (o <= p.extra) live = false;  // the cut has moved to the item's start: the next CTA's
      else if (tiles + p.extra - o > p.extra) i1 = o - p.extra;
    }
  }
  __device__ __forceinline__ void advance() {
    start += units();
    live = start < end;
    if (!live) return;
    if ((t + 1) * p.tok < s.nq) {
      ++t;
    } else {
      t = 0;
      if (++h == p.Hkv) {
        h = 0;
        do ++b; while (pre[b + 1] == pre[b]);
        s = seq_of(p, b, false);
      }
    }
    tiles = item_tiles<BN>(p, s, t);
    i0 = 0;
    finish();
  }
  __device__ __forceinline__ bool more() const { return live; }
  __device__ __forceinline__ void next() {
    if (i1 < tiles) live = false;  // cut: the range ends inside this item
    else advance();
  }
  __device__ __forceinline__ bool whole() const { return i0 == 0 && i1 == tiles; }
  __device__ __forceinline__ int tok0() const { return t * p.tok; }
  __device__ __forceinline__ int ntok() const { return min(p.tok, s.nq - t * p.tok); }
  __device__ __forceinline__ int kend() const { return keys_seen(p, s, min(s.nq, (t + 1) * p.tok)); }
  // of a cut item, seen by CTA c that holds its first piece
  __device__ __forceinline__ CutItem cut_item(const Cut& cut, unsigned int c) const {
    return CutItem{static_cast<int>(last_cta(cut) - c) + 1, s.q0 + tok0(), ntok(), h,
                   p.causal ? max(0, s.nq - s.n - tok0()) : 0, {0, 0, 0}};
  }
  __device__ __forceinline__ unsigned int last_cta(const Cut& cut) const {
    const unsigned int e = start + tiles + p.extra;
    const unsigned int c = cut.cta_of(e - 1);
    return e - cut.bound(c) <= static_cast<unsigned int>(p.extra) ? c - 1 : c;
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

// Launches fn as a programmatic dependent of the stream's previous kernel: its CTAs may start while that one drains, and
// wait (pdl_wait) before they touch global memory.
template <typename... P, typename... A>
int launch_pdl(void (*fn)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const char* what, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, fn, args...), what);
}

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
  long long max_keys;  // no sequence has more
};

// Whether the tensors could hold more units than the schedule counts: every sequence with all of its keys, token tiles of
// `bn` keys each. (The lengths are on the device; up to this bound, the kernels without the other schedule are right for all.)
inline bool may_be_long(const Problem& p, const Source& src, int bn) {
  const double items = (static_cast<double>(p.T) / p.tok + p.B) * p.Hkv;
  return items * (static_cast<double>(src.max_keys) / bn + 2 + p.extra) >= static_cast<double>(kMaxUnits);
}

// 5-D maps over keys and values [page][head][64-value part of a head][token][64 values], 128-byte swizzle, box of
// 64 values x `box` tokens x `parts` parts: in shared memory [part][token][64 values]
int make_kv_maps(CUtensorMap* mk, CUtensorMap* mv_, const Source& src, int heads, int d, bool bf16, int box, int parts);

// 3-D map over queries [token][head][d], 128-byte swizzle, box of 64 values x the G heads of a key head x `tok` tokens
int make_q_map(CUtensorMap* m, const Problem& p, int d, bool bf16, int tok);

}  // namespace attn
}  // namespace mv
