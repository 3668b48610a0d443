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

constexpr int kMaxSeqs = 1 << 24;  // of a call: workgroups look through them 64 at a time

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

// a / b of a >= 0, b > 0; the 64-bit division takes a microsecond.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// The sequence that row `row` of q is one of, by 64 lanes: the first that ends behind it, or the last (where starts
// do not ascend, any of the call's).
__device__ __forceinline__ int seq_of_row(const KvSeqs& s, int B, long long row, int lane) {
  if (!s.start) return (int)quotient(row, s.max_new);
  int lo = 0, n = B;  // it is one of lo .. lo + n - 1, or the last
  while (n > 1) {
    const int step = (n - 1) / 64 + 1;  // lane l asks whether sequence lo + (l + 1) step - 1 ends at or before the row
    const int at = (lane + 1) * step;
    const int below = __popcll(__ballot(at < n && s.start[lo + min(at, n)] <= row));
    lo += below * step;
    n = min(step, n - below * step);
  }
  return lo;
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
// ancestors with those of its furthest one so far, so log2(n) steps reach the root.  A parent that is not
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
  for (int step = 1; step < s.n; step *= 2) {
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

// ---- equal shares ----
// The lists of all row blocks, key/value heads and sequences stand in one line, a list as long as its key
// blocks and `over` more (what a workgroup spends on beginning and ending one, in blocks); the line is cut
// into equal shares, a workgroup each, whatever the lengths of the sequences.  A share may hold the end of
// one list, whole ones and the beginning of another; the parts of a list that was cut meet in
// paged_combine.  Where there are few lists or little to do, each list is cut into equal parts by itself
// instead and a workgroup has one of them: no workgroup then begins two.  And where lists are to be taken whole
// but there might be more than a grid has workgroups (most of them empty: a list for each row block that a
// sequence might have), the lists that there are stand in the line, each with length 1.
struct SharePlan {
  int row_min, row_max;  // rows a key/value head of the sequences served
  int rows, tiles;       // rows of a row block, row blocks of the longest sequence
  int part_rows;         // rows of a part: a row block's, if any sequence has as many
  int shares;            // workgroups of the line; 0 (no workspace): a workgroup a list
  int min_share;         // of a share, in blocks; 0: the line's lists are not cut (no workspace either)
  __host__ __device__ bool whole() const { return min_share == 0; }
};
// Workspace: for every list the workgroup of its first part and the number of its parts (in that workgroup and
// the ones behind it), then two parts a workgroup, the one that ends a list begun before its share and the one
// that its share leaves unended: rows of O, then (reference max, sum) pairs.
__host__ __device__ inline long long part_floats(const SharePlan& p, int D) { return (long long)p.part_rows * (D + 2); }
__host__ __device__ inline long long notes_floats(long long lists) { return (2 * lists + 63) / 64 * 64; }
__host__ __device__ inline long long part_at(const SharePlan& p, int first, int u, int D) {
  return (2LL * (first + u) + (u == 0)) * part_floats(p, D);
}
inline long long lists_of(const PagedCall& c, const SharePlan& p) { return (long long)c.B * c.Hkv * p.tiles; }
// A grid has fewer than 2^32 threads.
inline bool fits_grid(long long workgroups, int threads) { return workgroups < (1LL << 32) / threads; }
inline size_t share_bytes(const PagedCall& c, const SharePlan& p) {
  if (p.shares == 0 || p.whole()) return 0;
  const long long lists = lists_of(c, p);
  return sizeof(float) * (size_t)(notes_floats(lists) + 2LL * p.shares * part_floats(p, c.D));
}

// Lists taken whole by workgroups of `threads`: through a line of `workgroups` where a grid cannot have one a list.
inline void deal_whole(const PagedCall& c, SharePlan& p, int threads, int workgroups) {
  if (p.shares > 0 || fits_grid(lists_of(c, p), threads)) return;
  p.shares = workgroups;
  p.min_share = 0;
}

// The lists of 64 sequences from b0 on, one sequence a lane.
struct Lane64 {
  Seq seq;
  int tiles, length;  // a list's place in the line
  long long sum;      // of all lists up to and with this sequence's
};
// A workgroup's piece of work: part `slot` of `count` (0: none left) of a list.
struct Piece {
  Seq seq;
  int b, hk, rb, p0, p1, slot, count;
  int parts;  // not 0: p0 is the part's number; else p0 .. p1 of the list's length
  // its blocks, of the n that the row block's list has
  __device__ __forceinline__ void blocks(int n, int over, int& t0, int& t1) const {
    t0 = parts ? (int)((long long)n * p0 / count) : min(max(p0 - over, 0), n);
    t1 = parts ? (int)((long long)n * (p0 + 1) / count) : min(max(p1 - over, 0), n);
  }
};
// Where a workgroup is in its share [.., end): the next place x, the sequences around it (b0 on, `before` the
// line before them), and the piece it has and the next one, in turn.
struct Share {
  Lane64 seqs[64];
  long long share, x, end, before;
  int b0;
  int part;  // blocks a part, where each list is cut by itself (the line is then one of parts); else 0
  Piece piece[2];
};
__device__ __forceinline__ long long uniform(long long v) {
  return (long long)(((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                     (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// BLK keys a block, ROWS rows a block, OVER blocks for a list's beginning and end.
template <int BLK, int ROWS, int OVER, bool TREE>
struct Shares {
  static __device__ __forceinline__ Lane64 line(const PagedCall& c, const SharePlan& plan, int b0, int lane, int part) {
    Lane64 r{{0, 0, 0, 0}, 0, 1, 0};
    if (b0 + lane < c.B) {
      const Seq s = r.seq = load_seq(c.kv, c.seqs, b0 + lane);
      const long long rows = (long long)s.n * (c.H / c.Hkv);
      if (rows > 0 && rows >= plan.row_min && rows <= plan.row_max) {
        r.tiles = ((int)rows - 1) / ROWS + 1;
        // (that of all rows of the sequence; a row block's own list may be shorter, never longer)
        r.length = key_list<BLK>(s, 0, s.n - 1, c.window, c.sinks, TREE).n + OVER;
        if (part) r.length = (r.length - 1) / part + 1;
        r.sum = (long long)c.Hkv * r.tiles * r.length;
      }
    }
    add_up(r, lane);
    return r;
  }
  static __device__ __forceinline__ void add_up(Lane64& r, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const long long up = __shfl_up(r.sum, d);
      if (lane >= d) r.sum += up;
    }
  }

  // By the first wavefront.  The state is kept in LDS: held in registers, it would cost the loops over the
  // keys some.
  static __device__ __forceinline__ void begin(Share& f, const PagedCall& c, const SharePlan& plan, int lane) {
    Lane64 seqs;
    long long total = 0, lists = 0;
    int part = plan.whole() ? 0x7fffffff : 0;  // (that many blocks are any list)
    for (int b0 = 0; b0 < c.B; b0 += 64) {
      seqs = line(c, plan, b0, lane, part);
      total += uniform(__shfl(seqs.sum, 63));
      int n = seqs.tiles;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d);
      lists += (long long)c.Hkv * __builtin_amdgcn_readfirstlane(n);
    }
    const long long grid = gridDim.x;
    long long share = max((long long)max(plan.min_share, 1), quotient(total + grid - 1, grid));
    // parts of one list each: ceil(w / part) <= w / part + 1 of them, in all no more than workgroups; up to a
    // twentieth longer than the shares
    if (!plan.whole() && lists < grid) {
      const long long p = max((long long)plan.min_share, quotient(total + grid - lists - 1, grid - lists));
      if (20 * p <= 21 * share && p <= 0x7fffffff) part = (int)p;
    }
    if (part || c.B > 64) seqs = line(c, plan, 0, lane, part);
    f.seqs[lane] = seqs;
    if (part && !plan.whole()) {
      share = 1;
      total = 0;
      for (int b0 = 0; b0 < c.B; b0 += 64)
        total += uniform(__shfl(b0 == 0 ? seqs.sum : line(c, plan, b0, lane, part).sum, 63));
    }
    if (lane == 0) {
      f.share = share;
      f.x = blockIdx.x * share;
      f.end = min(total, f.x + share);
      f.before = 0;
      f.b0 = 0;
      f.part = part;
    }
  }

  // The next list of the share, or the part of one, into piece[turn]; by the first wavefront, a barrier behind
  // it.  It is called one piece ahead, so that its time does not stand between two pieces.
  static __device__ __forceinline__ void next(Share& f, const PagedCall& c, const SharePlan& plan, int lane, int turn) {
    asm volatile("" ::: "memory");
    const long long x = uniform(f.x), x1 = uniform(f.end), share = uniform(f.share);
    int count = 0;
    if (x < x1) {
      const long long x0 = blockIdx.x * share;
      long long before = uniform(f.before);
      int b0 = __builtin_amdgcn_readfirstlane(f.b0);
      Lane64 seqs = f.seqs[lane];
      for (long long sum; before + (sum = uniform(__shfl(seqs.sum, 63))) <= x;) {
        before += sum;
        b0 += 64;
        seqs = line(c, plan, b0, lane, __builtin_amdgcn_readfirstlane(f.part));
        f.seqs[lane] = seqs;
      }
      const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before + seqs.sum <= x)));
      const int tiles = __builtin_amdgcn_readlane(seqs.tiles, at), length = __builtin_amdgcn_readlane(seqs.length, at);
      const long long off = x - before - (at > 0 ? uniform(__shfl(seqs.sum, at - 1)) : 0);
      const int list = (int)quotient(off, length), p0 = (int)(off - (long long)list * length);
      const int p1 = (int)min((long long)length, p0 + x1 - x);
      // parts: the list begins at x - p0 and is cut at multiples of the share
      const long long begin = x - p0;
      const int slot = begin >= x0 ? 0 : (int)quotient(x0 - begin + share - 1, share);
      count = begin + length <= x0 + share ? slot + 1 : slot + 1 + (int)quotient(begin + length - x0 - 1, share);
      if (lane == at) f.piece[turn] = {seqs.seq, b0 + at, list / tiles, list % tiles, p0, p1, slot, count, f.part};
      if (lane == 0) {
        f.x = x + p1 - p0;
        f.before = before;
        f.b0 = b0;
      }
    }
    if (lane == 0 && count == 0) f.piece[turn].count = 0;
  }
};

__device__ __forceinline__ Piece read_piece(const Piece& f) {
  auto u = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return {{u(f.seq.row0), u(f.seq.n), u(f.seq.len), u(f.seq.first)}, u(f.b), u(f.hk), u(f.rb), u(f.p0), u(f.p1),
          u(f.slot), u(f.count), u(f.parts)};
}
// Where a workgroup leaves its part of a list that was cut, and (the first part's) the list's note; ws is null where
// no list is.
__device__ __forceinline__ float* part_of(float* ws, const PagedCall& c, const SharePlan& plan, const Piece& p) {
  return ws + notes_floats((long long)c.B * c.Hkv * plan.tiles) +
         part_at(plan, (int)blockIdx.x - p.slot, p.slot, c.D);
}
__device__ __forceinline__ void note_list(float* ws, const PagedCall& c, const SharePlan& plan, const Piece& p) {
  if (ws && p.slot == 0) {
    int* note = reinterpret_cast<int*>(ws) + 2 * (((long long)p.b * c.Hkv + p.hk) * plan.tiles + p.rb);
    note[0] = blockIdx.x;
    note[1] = p.count;
  }
}
constexpr int kShortRows = 16, kTileRows = 256, kWideRows = 128;  // rows of a row block of the kernels
constexpr int kTileDim = 128;                                     // the bf16 parts' widest, f32 tiles from there on
// What a list's beginning and end cost an f32 tile, in blocks: 13 tokens behind 2048 keys, 4 sequences, 8 heads on
// 2, D 256, 50 us with 2, 67 with 4.
constexpr int kWideOver = 2;
// Where a workgroup takes a tile whole: tile and b * Hkv + hk of workgroup n, last tiles first (without a window the
// longest), a tile's sequences and heads together; with Hkv a multiple of 8 the tiles of a head share an XCD's L2.
// The sequences go round by one from tile to tile: workgroups are dealt out in turn to the XCDs and to the four
// engines of one, and with B a multiple of 4 one engine would else get all tiles of the longest sequence.
struct Tile {
  int rb, bk;
};
__device__ __forceinline__ Tile tile_of(const PagedCall& c, const SharePlan& plan, unsigned n) {
  const unsigned nbk = (unsigned)c.B * c.Hkv, at = n / nbk;
  return {(int)(plan.tiles - 1 - at), (int)((n - at * nbk + at % c.B * c.Hkv) % nbk)};
}
inline int tile_rows(int D) { return D <= kTileDim ? kTileRows : kWideRows; }

// The most keys that a row block of the call reads.
inline long long most_keys(const PagedCall& c, int max_len) {
  return c.window > 0 ? std::min<long long>(max_len, (long long)c.window + c.sinks + c.seqs.max_new) : max_len;
}

// ws: the results of split keys; with less than sdpa_paged_workspace_bytes it runs unsplit.  max_len:
// the longest sequence, for the plan.
hipError_t launch_sdpa_paged(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes);
size_t sdpa_paged_workspace_bytes(const PagedCall& c, int max_len);
// The kernels of the call, rows of a row block and shares (the least of one in blocks) of each; with a workspace.
const char* sdpa_paged_kernel_name(const PagedCall& c, int max_len);
// The sequences with more than kFewRows rows a key/value head, 8 <= D <= 256 (sdpa_paged_tile.hip, above 128
// sdpa_paged_wide.hip), and the
// ones with up to row_limit, 4 <= D <= 256 (sdpa_paged_rows.hip).  A plan's workspace: share_bytes.
// Measured, the first / the second kernel, us (8 sequences of 4096 keys, 32 heads on 8, D 128): 32 rows 113 / 63,
// 48 117 / 103 (90 and 128 with 16 rows a workgroup, as in batches with longer chunks; 64 so 116 / 170); through a
// window of 512, 48 rows 40 / 34, 64 41 / 41.  D 256:
// 32 rows 185 by the second, 48 - / 299, 52 208 / -; 4 sequences of 2048 keys, 8 heads on 2, 48 - / 41, 52 50 / -.
constexpr int kFewRows = 48;
bool sdpa_paged_tile_applies(const PagedCall& c);
SharePlan sdpa_paged_tile_plan(const PagedCall& c, int max_len, bool may_split);
hipError_t launch_sdpa_paged_tile(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws);
hipError_t launch_sdpa_paged_wide(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws);
bool sdpa_paged_rows_applies(const PagedCall& c, int row_limit);
SharePlan sdpa_paged_rows_plan(const PagedCall& c, int max_len, int row_limit, bool may_split);
hipError_t launch_sdpa_paged_rows(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws);

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
