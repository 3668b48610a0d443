// sdpa_paged_rows.hip -- attention over a paged cache for few rows a sequence: a decode step, a small
// tree of drafts, a short chunk (paged.h says which keys a row sees).
//
// What bounds it: reading the visible K and V once: 4 sequences of 65536 keys, 8 heads of 128, 2.15 GB, 369 us,
// 5.8 TB/s; 32 of up to 16384 keys through a window of 4096, 389 MB, 84 us, 4.6 TB/s, where the beginnings of
// 256 lists count.  As in sdpa_decode.hip:
//   * Rows: token t, query head hk * group + g of a key/value head is row t * group + g (tokens outermost,
//     so that the rows of a block stand close together and share the ends of their windows), taken 16 or 32
//     at a time; K and V are read once for all of them.
//   * Keys: the sink blocks and the window's blocks of 16 keys of a row block are one list, and the lists of
//     all row blocks, key/value heads and sequences one line that is cut into equal shares, a workgroup
//     each, whatever the lengths of the sequences: a share may hold the end of one list, whole ones and the
//     beginning of another.  The four wavefronts of a workgroup (eight, where it takes one list whole) take a
//     list's blocks in turn.  K and V go from global memory
//     straight into the operand registers of v_mfma_f32_16x16x4_f32, the next block's loads in flight and
//     the page numbers of the one after that.  No barrier until the end.
//   * S^T = K Q^T: lane (g = l / 16, i = l % 16) holds K[key i][16 c + 4 g .. + 3] and q[row i] alike; value r
//     of the result is key 4 g + r of row i.  O^T += V^T P^T: step r contracts key 4 g + r; the lane holds
//     V[key 4 g + r][4 (i + 16 h) .. + 3], component e feeding O block 4 h + e, whose value r' is
//     d = 4 (4 g + r' + 16 h) + e.
//   * Lane i of the first sixteen looks key i's page up; the others get the row's offset by a lane
//     permutation.
//   * Keys that no row of the block sees (behind the last row, between sinks and window, in a page that is
//     not held) have their V rows zeroed, whatever stands there; masked scores are -inf.  A weight of 0
//     still turns an infinite V that only some rows see into NaN, so a wavefront whose result is not
//     finite does its blocks again with those values added by the vector unit, to the rows that see them.
//   * Each wavefront keeps its own lazily moved reference maximum, sum and O; they meet in LDS, and the
//     results of a list that was cut in paged_combine.  Fixed cuts and order: deterministic.
#include "paged.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

using bch::f32x4;
using bch::PagedCall;
using bch::SharePlan;

constexpr float kLazy = 8.0f;  // log2 headroom before the reference max moves
constexpr int kRows = bch::kShortRows;  // rows per workgroup
constexpr int kBlk = 16;       // keys per block

__device__ __forceinline__ float quad_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows are read in fours from d0 = 0, 4, ... on.  FULL: D == DP; otherwise D >= 4, and a four that would
// reach past D is the row's last one: its columns below d0 are in the four before too, so they are zero
// in q (and count once in the scores), and come out twice, alike, in O.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// (inside: known to be below D without looking; only the last 64 columns of a class of D need the comparison,
// and the others' addresses no registers of their own: 4 x 2048 keys of 8 heads on 2, D 200, a token
// each, 51 and 40 us)
template <bool FULL>
__device__ __forceinline__ int four(int d0, int D, bool inside) {
  return FULL || inside ? d0 : min(d0, D - 4);
}
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4u*>(p); }
template <bool FULL>
__device__ __forceinline__ f32x4 once(f32x4 x, int d0, int D) {
  if (!FULL) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = min(d0, D - 4) + e >= d0 ? x[e] : 0.0f;
  }
  return x;
}

// What a list's beginning and end (the trips to memory for its pages and its first keys, the wavefronts'
// results) cost in blocks when the chip is full: 32 ragged sequences (389 MB) took 110 us with 3, 84 with 8 to
// 12, 85 with 16.
constexpr int kOver = 8;

template <int DP, int kWaves, int RB, bool FULL, bool TREE>
__global__ __launch_bounds__(64 * kWaves, DP * RB > 128 ? 1 : 2) void sdpa_paged_rows_kernel(PagedCall c, SharePlan plan,
                                                                                      float* __restrict__ ws) {
  constexpr int NC = DP / 16, NH = DP / 64, kIn = DP - 64;  // D > kIn
  constexpr int ROWS = kRows * RB;
  __shared__ float red_m[kWaves][ROWS], red_l[kWaves][ROWS];
  __shared__ float red_o[kWaves - 1][ROWS][DP + 4];
  __shared__ std::conditional_t<TREE, bch::TreeMasks, int> tree;
  __shared__ bch::Share find;

  const int D = c.D, group = c.H / c.Hkv;

  using Line = bch::Shares<kBlk, ROWS, kOver, TREE>;
  if (plan.shares > 0 && threadIdx.x < 64) {
    Line::begin(find, c, plan, threadIdx.x);
    Line::next(find, c, plan, threadIdx.x, 0);
  }

  int tree_of = -1;
  bool more = true;
  for (int turn = 0; more; turn ^= 1) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // what follows from it is not held in registers from one piece to the next
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    bch::Piece piece;
    if (plan.shares > 0) {
      __syncthreads();
      piece = bch::read_piece(find.piece[turn]);
      if (piece.count == 0) break;
      if (wave == 0) Line::next(find, c, plan, lane, turn ^ 1);
    } else {
      const int bk = blockIdx.x / plan.tiles;
      piece = {bch::load_seq(c.kv, c.seqs, bk / c.Hkv), bk / c.Hkv, bk % c.Hkv, (int)(blockIdx.x % plan.tiles), 0, 0, 0, 1, 1};
      more = false;
    }
    const int b = piece.b, hk = piece.hk, rb = piece.rb, count = piece.count;
    const bch::Seq s = piece.seq;
    const int rows = s.n * group;
    if (plan.shares == 0 && (rb * ROWS >= rows || rows > plan.row_max)) break;
    if constexpr (TREE) {
      static_assert(64 * kWaves >= bch::kMaxDrafts, "tree_masks");
      if (b != tree_of) bch::tree_masks(tree, c.parent, s, c.window, c.sinks);
      tree_of = b;
    }
    const int t_lo = rb * ROWS / group, t_hi = (min(rb * ROWS + ROWS, rows) - 1) / group;
    const bch::KeyList keys = bch::key_list<kBlk>(s, t_lo, t_hi, c.window, c.sinks, TREE);
    int t0, t1;
    piece.blocks(keys.n, kOver, t0, t1);
    const float* kh = c.kv.k + hk * c.kv.kl.head;
    const float* vh = c.kv.v + hk * c.kv.vl.head;

    // ---- rows ROWS rb + 16 a + i (rows past the end repeat the last one and are not stored) ----
    int tok[RB], pos[RB];
    f32x4 qf[RB][NC];
    auto lane_row = [&](int a) { return min(rb * ROWS + 16 * a + i, rows - 1); };
    auto row_offset = [&](const bch::SdpaLayout& l, int a) {
      return b * l.batch + (long long)(s.row0 + tok[a]) * l.row + (long long)(hk * group + lane_row(a) - tok[a] * group) * l.head;
    };
#pragma unroll
    for (int a = 0; a < RB; ++a) {
      tok[a] = lane_row(a) / group;
      pos[a] = s.first + [&] {
        if constexpr (TREE) return tree.depth[tok[a]];
        else return tok[a];
      }();
      const float* qr = c.q + row_offset(c.ql, a);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int d0 = 16 * n + 4 * g;
        qf[a][n] = once<FULL>(load4(qr + four<FULL>(d0, D, 16 * n + 16 <= kIn)), d0, D) * c.qscale;
      }
    }

    const int p_lo = TREE ? s.first : s.first + t_lo, p_hi = s.first + t_hi;
    auto key0 = [&](int t) { return keys.key0<kBlk>(t); };

    f32x4 acc[RB][4 * NH];
    float m_ref[RB], l_run[RB];
    auto reset = [&]() {
#pragma unroll
      for (int a = 0; a < RB; ++a) {
#pragma unroll
        for (int n = 0; n < 4 * NH; ++n) acc[a][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
        m_ref[a] = -INFINITY;
        l_run[a] = 0.0f;
      }
    };
    reset();

    f32x4 kf[2][NC], vf[2][4 * NH];
    unsigned there[2];  // bit j: key j of the block is one that a row sees, in a page that is held
    long long voff;     // of this lane's key (i) of the block loaded last
    int entry = 0;      // the table's entry for this lane's key of the block to be loaded next
    auto fetch = [&](int t) {
      const int j = key0(t) + i, n = (int)(((unsigned long long)(unsigned)j * c.kv.mul) >> c.kv.shift);
      if (c.kv.table) entry = c.kv.table[(long long)b * c.kv.width + min(n, c.kv.width - 1)];
    };
    auto load = [&](int u, int t, int next) {
      const int j = key0(t) + i, n = (int)(((unsigned long long)(unsigned)j * c.kv.mul) >> c.kv.shift);
      bch::Slot slot{b, j};
      if (c.kv.table) slot = {entry, j - n * c.kv.page_size};
      const bool on = keys.any(j) && (unsigned)slot.page < (unsigned)c.kv.num_pages;
      if (!on) slot = {0, 0};
      there[u] = (unsigned)__ballot(on) & 0xffffu;
      const float* kr = kh + bch::slot_offset(c.kv.kl, slot);
      voff = bch::slot_offset(c.kv.vl, slot);
#pragma unroll
      for (int x = 0; x < NC; ++x) kf[u][x] = load4(kr + four<FULL>(16 * x + 4 * g, D, 16 * x + 16 <= kIn));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float* vr = vh + __shfl(voff, 4 * g + r);
#pragma unroll
        for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = load4(vr + four<FULL>(4 * (i + 16 * h), D, 64 * h + 64 <= kIn));
      }
      fetch(next);
    };

    // careful: adds values that are not finite by the vector unit, to the rows that see their key
    auto block = [&](auto careful, int u, int t) {
      const int kb = key0(t);
      f32x4 sc[RB];
#pragma unroll
      for (int a = 0; a < RB; ++a) sc[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        // (0 times an infinite K would be NaN, not the score)
        const f32x4 kx = decltype(careful)::value ? once<FULL>(kf[u][x], 16 * x + 4 * g, D) : kf[u][x];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int a = 0; a < RB; ++a) sc[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[e], qf[a][x][e], sc[a], 0, 0, 0);
      }
      const unsigned on = there[u] >> (4 * g);
      if (there[u] != 0xffffu) {  // uniform
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(on >> r & 1)) {
#pragma unroll
            for (int a = 0; a < RB; ++a) sc[a][r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = (f32x4){0.f, 0.f, 0.f, 0.f};
          }
      }
      // rows that differ in what they see of this block
      const bool cut = c.window > 0 && kb <= p_hi - c.window && kb + kBlk > c.sinks;
      if (kb + kBlk - 1 > p_lo - (TREE ? 1 : 0) || cut) {
#pragma unroll
        for (int a = 0; a < RB; ++a)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = kb + 4 * g + r;
            bool see = j <= pos[a] && (c.window == 0 || pos[a] - j < c.window || j < c.sinks);
            if constexpr (TREE) {
              const int n = j - s.first;
              if (n >= 0) see = n < bch::kMaxDrafts && (tree.mask[tok[a]][(n >> 5) & 3] >> (n & 31) & 1);
            }
            if (!see) sc[a][r] = -INFINITY;
          }
      }
      unsigned seen[RB];
#pragma unroll
      for (int a = 0; a < RB; ++a) {
        const float bm = quad_max(fmaxf(fmaxf(sc[a][0], sc[a][1]), fmaxf(sc[a][2], sc[a][3])));
        const bool move = bm > m_ref[a] + kLazy;  // -inf reference: any finite block max moves it
        if (__any(move)) {
          const float m_new = move ? bm : m_ref[a];
          const float alpha = m_ref[a] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_ref[a] - m_new);
          l_run[a] *= alpha;
#pragma unroll
          for (int n = 0; n < 4 * NH; ++n) acc[a][n] *= alpha;
          m_ref[a] = m_new;
        }
        const float m_use = m_ref[a] == -INFINITY ? 0.0f : m_ref[a];
        seen[a] = 0;
        float rs = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (decltype(careful)::value) seen[a] |= sc[a][r] == -INFINITY ? 0u : 1u << r;
          sc[a][r] = __builtin_amdgcn_exp2f(sc[a][r] - m_use);
          rs += sc[a][r];
        }
        l_run[a] += quad_sum(rs);
      }
      if constexpr (decltype(careful)::value) {
        unsigned odd = 0;  // keys with values that are not finite
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float z = 0.0f;
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) z = fmaf(vf[u][r * NH + h][e], 0.0f, z);
          const unsigned long long lanes = __ballot(z != 0.0f);
          for (int g2 = 0; g2 < 4; ++g2)
            if (lanes >> (16 * g2) & 0xffffu) odd |= 1u << (4 * g2 + r);
          if (odd >> (4 * g + r) & 1) {
#pragma unroll
            for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = (f32x4){0.f, 0.f, 0.f, 0.f};
          }
        }
#pragma unroll 1
        for (; odd; odd &= odd - 1) {
          const int key = __ffs(odd) - 1, r = key & 3, from = 16 * (key >> 2) + i;
          const float* vr = vh + __shfl(voff, key);
#pragma unroll
          for (int a = 0; a < RB; ++a) {
            const float p = __shfl(r == 0 ? sc[a][0] : r == 1 ? sc[a][1] : r == 2 ? sc[a][2] : sc[a][3], from);
            const bool see = __shfl((int)seen[a], from) >> r & 1;
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
              for (int r2 = 0; r2 < 4; ++r2) {
                const f32x4 x = load4(vr + four<FULL>(4 * (4 * g + r2 + 16 * h), D, 64 * h + 64 <= kIn));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (see) acc[a][4 * h + e][r2] = fmaf(p, x[e], acc[a][4 * h + e][r2]);
              }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int a = 0; a < RB; ++a)
              acc[a][4 * h + e] =
                  __builtin_amdgcn_mfma_f32_16x16x4f32(vf[u][r * NH + h][e], sc[a][r], acc[a][4 * h + e], 0, 0, 0);
    };

    // wavefront w takes blocks t0 + w, t0 + w + 4, ...; loads past the last one repeat it
    if (t0 + wave < t1) {
      int t = t0 + wave;
      fetch(t);
      load(0, t, min(t + kWaves, t1 - 1));
      for (; t < t1; t += 2 * kWaves) {
        load(1, min(t + kWaves, t1 - 1), min(t + 2 * kWaves, t1 - 1));
        block(std::false_type{}, 0, t);
        if (t + kWaves >= t1) break;
        load(0, min(t + 2 * kWaves, t1 - 1), min(t + 3 * kWaves, t1 - 1));
        block(std::false_type{}, 1, t + kWaves);
      }
      float z = 0.0f;
#pragma unroll
      for (int a = 0; a < RB; ++a) {
        z = fmaf(l_run[a], 0.0f, z);
#pragma unroll
        for (int n = 0; n < 4 * NH; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) z = fmaf(acc[a][n][r], 0.0f, z);
      }
      if (__any(z != 0.0f)) {
        reset();
#pragma unroll 1
        for (t = t0 + wave; t < t1; t += kWaves) {
          fetch(t);
          load(0, t, t);
          block(std::true_type{}, 0, t);
        }
      }
    }

    // ---- the wavefronts' results, in wavefront order ----
#pragma unroll
    for (int a = 0; a < RB; ++a) {
      if (g == 0) {
        red_m[wave][16 * a + i] = m_ref[a];
        red_l[wave][16 * a + i] = l_run[a];
      }
      if (wave > 0) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) red_o[wave - 1][16 * a + i][4 * (4 * g + r + 16 * h) + e] = acc[a][4 * h + e][r];
      }
    }
    __syncthreads();
    if (wave == 0) {
      if (lane == 0) bch::note_list(ws, c, plan, piece);
#pragma unroll
      for (int a = 0; a < RB; ++a) {
        const int at = 16 * a + i;
        float m = red_m[0][at];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red_m[w][at]);
        const float m_use = m == -INFINITY ? 0.0f : m;
        // a wavefront without a key has m = -inf: its factor is 0 and so is its O
        float f = __builtin_amdgcn_exp2f(m_ref[a] - m_use), l = f * l_run[a];
#pragma unroll
        for (int n = 0; n < 4 * NH; ++n) acc[a][n] *= f;
#pragma unroll 1
        for (int w = 1; w < kWaves; ++w) {
          f = __builtin_amdgcn_exp2f(red_m[w][at] - m_use);
          l += f * red_l[w][at];
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[a][4 * h + e][r] += f * red_o[w - 1][at][4 * (4 * g + r + 16 * h) + e];
        }

        if (rb * ROWS + at < rows) {
          float* dst;
          float inv = 1.0f;
          if (count > 1) {
            float* p = bch::part_of(ws, c, plan, piece);
            dst = p + (long long)at * D;
            if (g == 0) {
              p[plan.part_rows * D + 2 * at] = m;
              p[plan.part_rows * D + 2 * at + 1] = l;
            }
          } else {
            dst = c.o + row_offset(c.ol, a);
            inv = l == 0.0f ? 0.0f : 1.0f / l;
          }
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int d0 = 4 * (4 * g + r + 16 * h);
              f32x4 x;
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = acc[a][4 * h + e][r] * inv;
              if (FULL || d0 < D) *reinterpret_cast<f32x4u*>(dst + four<FULL>(d0, D, 64 * h + 64 <= kIn)) = x;
            }
        }
      }
    }
    // (the next barrier, at the top, comes before anything here is written again)
  }
}

// Workgroups that are resident at once, so that equal shares end together.
int resident(int D, int rows) {
  return (rows > kRows ? (D <= 64 ? 2 : 1) : D <= 64 ? 3 : D <= 128 ? 2 : 1) * bch::device_cu_count();
}

template <int DP, int WAVES, int RB>
void launch_dp(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  const dim3 grid((unsigned)(p.shares > 0 ? (long long)p.shares : bch::lists_of(c, p))), block(64 * WAVES);
  const bool full = c.D == DP, tree = c.parent != nullptr;
  auto kern = full ? (tree ? sdpa_paged_rows_kernel<DP, WAVES, RB, true, true> : sdpa_paged_rows_kernel<DP, WAVES, RB, true, false>)
                   : (tree ? sdpa_paged_rows_kernel<DP, WAVES, RB, false, true> : sdpa_paged_rows_kernel<DP, WAVES, RB, false, false>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, c, p, ws);
}
// A list that one workgroup takes whole: eight wavefronts, where the registers leave that many room.
template <int DP>
void launch_waves(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  if (p.shares == 0 && DP <= 128) launch_dp<DP, DP <= 128 ? 8 : 4, 1>(s, c, p, ws);
  else if (p.rows > kRows) launch_dp<DP, 4, DP <= 128 ? 2 : 1>(s, c, p, ws);
  else launch_dp<DP, 4, 1>(s, c, p, ws);
}

}  // namespace

namespace bch {

// A share is at least 128 keys.  A workgroup takes a list whole, which saves the second launch, up to 384 keys
// of 128 floats, and up to 1024 where there is a list a CU; of narrower ones in proportion more.  Measured,
// whole / shared, us a decode step (32 heads on 8, D 128): 8 lists of 256 / 384 / 512 keys 15.5 / 18.8 / 22.0
// against 17.0 / 18.4 / 18.3; 256 lists of 512 / 1024 / 2048 28.6 / 45.8 / 96 against 36.8 / 54.3 / 107 (beyond,
// lists of unequal lengths gain more from shares); 8 lists of 500 keys, D 64, 13.9 against 16.8.
// Shared lists of more than 16 rows: 32 rows a workgroup, so that K and V are read once for them, where the lists'
// keys together take longer than a workgroup's beginning, which they lengthen (only D <= 128 leaves the registers;
// not in batches with longer chunks, most of whose sequences here may have one token).  16 / 32 rows, us (32 heads
// on 8, 8 tokens a sequence): D 128, 16 sequences of 8192 keys 302 / 202, 32 of 1500 120 / 86, one of 32768 92 / 67, of 4096
// 33.5 / 30.3, of 2048 22.5 / 28.3; D 64, 8 sequences of 2048 keys 36 / 30, of 1024 26.7 / 26.7, one of 2048 17.8 / 21.2.
SharePlan sdpa_paged_rows_plan(const PagedCall& c, int max_len, int row_limit, bool may_split) {
  SharePlan p;
  const int group = c.H / c.Hkv;
  p.row_min = 1;
  p.row_max = row_limit;
  const int most = (int)std::min((long long)c.seqs.max_new * group, (long long)row_limit / group * group);
  p.rows = kRows;
  p.tiles = (most + kRows - 1) / kRows;
  p.min_share = 8 + kOver;
  p.shares = 0;
  const long long whole = lists_of(c, p) >= device_cu_count() ? 1024 : 384, width = c.D <= 64 ? 64 : c.D <= 128 ? 128 : c.D <= 192 ? 192 : 256;
  if (may_split && p.tiles > 0 && most_keys(c, max_len) * width > whole * 128) p.shares = resident(c.D, p.rows);
  if (p.shares > 0 && c.D <= 128 && most > kRows && c.seqs.max_new * (long long)group <= row_limit &&
      most_keys(c, max_len) * c.B * c.Hkv >= (c.D <= 64 ? 131072 : 32768)) {
    p.rows = 2 * kRows;
    p.tiles = (most + p.rows - 1) / p.rows;
    p.shares = resident(c.D, p.rows);
  }
  p.part_rows = std::min(most, p.rows);
  deal_whole(c, p, 512, resident(c.D, p.rows));
  return p;
}

bool sdpa_paged_rows_applies(const PagedCall& c, int row_limit) {
  const long long rows = std::min((long long)c.seqs.max_new * (c.H / c.Hkv), (long long)row_limit);
  return c.D >= 4 && c.D <= 256 && rows <= 0x7fffffff - kRows &&
         (long long)c.Hkv * ((rows + kRows - 1) / kRows) <= 0x7fffffff;
}

hipError_t launch_sdpa_paged_rows(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  if (p.tiles == 0) return hipSuccess;  // a token alone has more rows than the limit
  if (c.D <= 64) launch_waves<64>(s, c, p, ws);
  else if (c.D <= 128) launch_waves<128>(s, c, p, ws);
  else if (c.D <= 192) launch_waves<192>(s, c, p, ws);
  else launch_waves<256>(s, c, p, ws);
  return hipGetLastError();
}

}  // namespace bch
