// paged.h -- a paged key/value cache as the kernels see it, shared by the attention kernels that
// read it (sdpa_paged*.hip) and the kernels that write it (kv_pages.hip).
//
// Sequence b holds len[b] keys; its n = start[b + 1] - start[b] new tokens are the last of them and
// rows start[b] .. of q, o and of an append's inputs.  Key j of it is slot j % page_size of page
// table[b][j / page_size].  Tables, lengths and starts are device memory that a captured graph reads
// at its replay, so the kernels bound whatever they find there: an entry outside 0 .. num_pages - 1 is
// a page that is not held (its keys are neither read nor written), starts are clamped to the rows
// there are and lengths to the table's width.
//
// Which keys a row sees: with c = len[b] - n, row i of a chain is at position c + i and sees key j
// <= its position; row i of a tree of drafts (parent[i] < i, or -1) is at position c + its number of
// ancestors and sees keys below c, itself and its ancestors.  Of those, with window > 0, it sees the
// ones less than window positions back and the ones in the first `sinks` positions.
#pragma once
#include "bch_internal.h"

#include <algorithm>

namespace bch {

constexpr int kMaxDrafts = 128;  // rows of one sequence's tree: its ancestor masks are four words

constexpr long long kMaxKeys = 0x7fffff00;  // of a sequence: a block's last key still has a 32-bit number

struct KvPages {
  const float *k, *v;
  SdpaLayout kl, vl;  // (page, head, row) strides
  int num_pages, page_size;
  unsigned mul;  // j / page_size = (j * mul) >> shift
  int shift;
  const int* table;  // null: sequence b is page b, whole (dense operands)
  int width;
};

struct KvSeqs {
  const int *start, *len;  // null: max_new rows and dense_len keys each (dense operands)
  int total, max_new, dense_len;
};

struct PagedCall {
  int B, H, Hkv, D;
  float qscale;  // scale * log2(e): the kernels' exponentials are powers of two
  int window, sinks;
  const int* parent;
  KvPages kv;
  KvSeqs seqs;
  const float* q;
  float* o;
  SdpaLayout ql, ol;  // (batch, head, row) strides; batch 0 where rows are numbered through
};

// The multiplier of an exact division by d of any 0 <= j < 2^31: with 2^s >= d, mul = ceil(2^(31 + s) / d)
// exceeds 2^(31 + s) / d by less than 1, so j * mul / 2^(31 + s) exceeds j / d by less than 2^-s <= 1 / d.
inline void set_page_size(KvPages& kv, int d) {
  kv.page_size = d;
  int s = 0;
  while ((1LL << s) < d) ++s;
  kv.shift = 31 + s;
  kv.mul = (unsigned)(((1ULL << kv.shift) + d - 1) / d);
}

// One sequence: its rows begin at row0, first = c (negative if there are more rows than keys).
struct Seq {
  int row0, n, len, first;
};
__device__ __forceinline__ Seq load_seq(const KvPages& kv, const KvSeqs& s, int b) {
  Seq r;
  if (!s.start) {
    r.row0 = 0;
    r.n = s.max_new;
    r.len = s.dense_len;
    r.first = r.len - r.n;
    return r;
  }
  const int a = min(max(s.start[b], 0), s.total), e = min(max(s.start[b + 1], a), s.total);
  const long long most = (long long)kv.width * kv.page_size;
  r.row0 = a;
  r.len = (int)min((long long)max(s.len[b], 0), min(most, kMaxKeys));
  r.first = r.len - (e - a);
  r.n = min(e - a, s.max_new);
  return r;
}

// The first key that the window leaves a row at position pos (negative: a row that sees nothing).
__device__ __forceinline__ int window_begin(int pos, int window) {
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}

// Page and slot of key j >= 0 of sequence b; page < 0 where it is not held.
struct Slot {
  int page, slot;
};
__device__ __forceinline__ Slot key_slot(const KvPages& kv, int b, int j) {
  if (!kv.table) return {b, j};
  const int i = (int)(((unsigned long long)(unsigned)j * kv.mul) >> kv.shift);
  if (i >= kv.width) return {-1, 0};
  const int p = kv.table[(long long)b * kv.width + i];
  return {(unsigned)p < (unsigned)kv.num_pages ? p : -1, j - i * kv.page_size};
}
__device__ __forceinline__ long long slot_offset(const SdpaLayout& l, Slot s) {
  return s.page * l.batch + s.slot * l.row;
}

// Ancestor masks of a tree's n <= kMaxDrafts drafts, by pointer jumping: every step joins a draft's
// ancestors with those of its furthest one so far, so seven steps reach the root.  A parent that is not
// below its draft (or is negative) makes it a root.  All threads of the workgroup (kMaxDrafts at
// least) call; mask[i] then holds i and the ancestors that the window leaves, depth[i] their number.
struct TreeMasks {
  unsigned mask[kMaxDrafts][4];
  int next[kMaxDrafts], depth[kMaxDrafts];
};
__device__ __forceinline__ void tree_masks(TreeMasks& t, const int* parent, const Seq& s, int window, int sinks) {
  const int i = threadIdx.x;
  const bool on = i < s.n && i < kMaxDrafts;
  if (on) {
    const int p = parent[s.row0 + i];
    t.next[i] = p >= 0 && p < i ? p : -1;
#pragma unroll
    for (int w = 0; w < 4; ++w) t.mask[i][w] = (i >> 5) == w ? 1u << (i & 31) : 0u;
  }
  __syncthreads();
  for (int step = 1; step < kMaxDrafts; step *= 2) {
    const int p = on ? t.next[i] : -1;
    unsigned m[4] = {0, 0, 0, 0};
    int np = -1;
    if (p >= 0) {
      np = t.next[p];
#pragma unroll
      for (int w = 0; w < 4; ++w) m[w] = t.mask[p][w];
    }
    __syncthreads();
    if (p >= 0) {
      t.next[i] = np;
#pragma unroll
      for (int w = 0; w < 4; ++w) t.mask[i][w] |= m[w];
    }
    __syncthreads();
  }
  if (on) {
    int c = -1;
#pragma unroll
    for (int w = 0; w < 4; ++w) c += __popc(t.mask[i][w]);
    t.depth[i] = c;
  }
  __syncthreads();
  if (on && window > 0 && window <= t.depth[i]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      unsigned m = t.mask[i][w], keep = 0;
      while (m) {
        const int a = __ffs(m) - 1;
        m &= m - 1;
        const int d = t.depth[32 * w + a];
        if (t.depth[i] - d < window || s.first + d < sinks) keep |= 1u << a;
      }
      t.mask[i][w] = keep;
    }
  }
  __syncthreads();
}

// ---- a block of rows and the keys that it reads ----
// Rows of a sequence and key/value head: token t, query head hk * group + g is row t * group + g.  The keys
// that any of the tokens t_lo .. t_hi sees, [0, s_hi) and [lo, hi), as a list of n blocks of BLK keys (each
// starting at a multiple of BLK), the first ns of them the sinks'.
struct KeyList {
  int hi, lo, s_hi, ns, m0, n;
  template <int BLK>
  __device__ __forceinline__ int key0(int t) const {
    return (t < ns ? t : t - ns + m0) * BLK;
  }
  __device__ __forceinline__ bool any(int j) const { return j < hi && (j >= lo || j < s_hi); }
};
template <int BLK>
__device__ __forceinline__ KeyList key_list(const Seq& s, int t_lo, int t_hi, int window, int sinks, bool tree) {
  KeyList k;
  k.hi = s.first + t_hi + 1;
  k.lo = window_begin(tree ? s.first : s.first + t_lo, window);
  k.s_hi = min(min(sinks, k.lo), k.hi);
  k.m0 = k.lo / BLK;
  k.ns = k.s_hi > 0 ? min((k.s_hi - 1) / BLK + 1, k.m0) : 0;
  k.n = k.hi > 0 ? k.ns + (k.hi - 1) / BLK + 1 - k.m0 : 0;
  return k;
}

// How a call is cut: row blocks of block_rows (the most of any sequence: tiles), the list of each block's
// keys over at most `splits` workgroups of at least min_blocks key blocks.
struct PagedPlan {
  int max_rows, block_rows, tiles, block_keys, min_blocks, splits;
};
__device__ __forceinline__ int split_count(int blocks, const PagedPlan& p) {
  return min(p.splits, max(1, (blocks + p.min_blocks - 1) / p.min_blocks));
}
// The most keys that a row block of the call reads.
inline long long most_keys(const PagedCall& c, int max_len) {
  return c.window > 0 ? std::min<long long>(max_len, (long long)c.window + c.sinks + c.seqs.max_new) : max_len;
}
inline size_t paged_part_bytes(const PagedCall& c, const PagedPlan& p) {
  return p.splits > 1 ? sizeof(float) * (size_t)c.B * c.Hkv * p.splits * sdpa_part_floats(p.max_rows, c.D) : 0;
}
// o = the splits' results joined, for the rows whose keys were split (sdpa_paged_rows.hip).
hipError_t launch_paged_combine(hipStream_t s, const PagedCall& c, const PagedPlan& p, const float* part);

// ws: the results of split keys; with less than sdpa_paged_workspace_bytes it runs unsplit.  max_len:
// the longest sequence, for the plan.
hipError_t launch_sdpa_paged(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes);
size_t sdpa_paged_workspace_bytes(const PagedCall& c, int max_len);
// More than kTileRows rows a key/value head, 8 <= D <= 128 (sdpa_paged_tile.hip).
constexpr int kTileRows = 64;
bool sdpa_paged_tile_applies(const PagedCall& c);
hipError_t launch_sdpa_paged_tile(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes);
size_t sdpa_paged_tile_workspace_bytes(const PagedCall& c, int max_len);
// 4 <= D <= 256 (sdpa_paged_rows.hip).
bool sdpa_paged_rows_applies(const PagedCall& c);
hipError_t launch_sdpa_paged_rows(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes);
size_t sdpa_paged_rows_workspace_bytes(const PagedCall& c, int max_len);

// ---- the cache's own calls (kv_pages.hip) ----
hipError_t launch_kv_append(hipStream_t s, const KvPages& kv, float* k, float* v, const KvSeqs& seqs, int B, int Hkv,
                            int D, const float* nk, const SdpaLayout& nkl, const float* nv, const SdpaLayout& nvl);
// Pages dst[x] = src[x], of `layers` layers; host arrays.
hipError_t launch_kv_copy_pages(hipStream_t s, const KvPages& kv, float* k, float* v, int layers, long long k_layer,
                                long long v_layer, int Hkv, int D, int n, const int* src, const int* dst);
// Key to[b] + i = key keep[start[b] + i], of `layers` layers, in ascending i.
hipError_t launch_kv_keep(hipStream_t s, const KvPages& kv, float* k, float* v, int layers, long long k_layer,
                          long long v_layer, int Hkv, int D, int B, int total, const int* start, const int* keep,
                          const int* to);

}  // namespace bch
