// sdpa_paged_rows.hip -- attention over a paged cache for few rows a sequence: a decode step, a small
// tree of drafts, a short chunk (paged.h says which keys a row sees).
//
// What bounds it: reading the visible K and V once.  As in sdpa_decode.hip:
//   * Rows: token t, query head hk * group + g of a key/value head is row t * group + g (tokens outermost,
//     so that the rows of a block stand close together and share the ends of their windows), taken 16 at a
//     time; K and V are read once for all 16.
//   * Keys: the sink blocks and the window's blocks of 16 keys are one list, cut evenly over the
//     workgroups of a sequence and dealt to the four wavefronts of each.  K and V go from global memory
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
//   * Each wavefront keeps its own lazily moved reference maximum, sum and O; the four meet in LDS, and the
//     workgroups' results in paged_combine.  Fixed split and order: deterministic.
#include "paged.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

using bch::f32x4;
using bch::PagedCall;
using bch::PagedPlan;

constexpr float kLazy = 8.0f;  // log2 headroom before the reference max moves
constexpr int kRows = 16;      // rows per workgroup
constexpr int kBlk = 16;       // keys per block
constexpr int kWaves = 4;

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

template <bool FULL>
__device__ __forceinline__ int four(int d0, int D) {
  return FULL ? d0 : min(d0, D - 4);
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

template <int DP, bool FULL, bool TREE>
__global__ __launch_bounds__(64 * kWaves, DP > 128 ? 1 : 2) void sdpa_paged_rows_kernel(PagedCall c, PagedPlan plan,
                                                                                      float* __restrict__ part) {
  constexpr int NC = DP / 16, NH = DP / 64;
  __shared__ float red_m[kWaves][kRows], red_l[kWaves][kRows];
  __shared__ float red_o[kWaves - 1][kRows][DP + 4];
  __shared__ std::conditional_t<TREE, bch::TreeMasks, int> tree;

  // row blocks of one split are neighbours on one XCD (round-robin dispatch over 8), sharing its L2's
  // copy of the keys
  const int nb = gridDim.x;
  int L = blockIdx.x;
  if ((nb & 7) == 0) L = (L & 7) * (nb >> 3) + (L >> 3);
  const int rb = L % plan.tiles;
  const int sp = L / plan.tiles % plan.splits;
  const int bk = L / plan.tiles / plan.splits;
  const int b = bk / c.Hkv, hk = bk - b * c.Hkv;
  const bch::Seq s = bch::load_seq(c.kv, c.seqs, b);
  const int group = c.H / c.Hkv, rows = s.n * group;
  if (rb * kRows >= rows) return;
  const int t_lo = rb * kRows / group, t_hi = (min(rb * kRows + kRows, rows) - 1) / group;
  const bch::KeyList keys = bch::key_list<kBlk>(s, t_lo, t_hi, c.window, c.sinks, TREE);
  const int splits = bch::split_count(keys.n, plan);
  if (sp >= splits) return;
  if constexpr (TREE) {
    static_assert(64 * kWaves >= bch::kMaxDrafts, "tree_masks");
    bch::tree_masks(tree, c.parent, s, c.window, c.sinks);
  }

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int D = c.D;
  const float* kh = c.kv.k + hk * c.kv.kl.head;
  const float* vh = c.kv.v + hk * c.kv.vl.head;

  // ---- row rb * 16 + i (rows past the end repeat the last one and are not stored) ----
  const int row = min(rb * kRows + i, rows - 1), tok = row / group;
  const int pos = s.first + [&] {
    if constexpr (TREE) return tree.depth[tok];
    else return tok;
  }();
  const float* qr = c.q + b * c.ql.batch + (long long)(s.row0 + tok) * c.ql.row +
                    (long long)(hk * group + row - tok * group) * c.ql.head;
  f32x4 qf[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int d0 = 16 * n + 4 * g;
    qf[n] = once<FULL>(load4(qr + four<FULL>(d0, D)), d0, D) * c.qscale;
  }

  const int p_lo = TREE ? s.first : s.first + t_lo, p_hi = s.first + t_hi;
  const int t0 = (int)((long long)keys.n * sp / splits), t1 = (int)((long long)keys.n * (sp + 1) / splits);
  auto key0 = [&](int t) { return keys.key0<kBlk>(t); };

  f32x4 acc[4 * NH];
  float m_ref, l_run;
  auto reset = [&]() {
#pragma unroll
    for (int n = 0; n < 4 * NH; ++n) acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    m_ref = -INFINITY;
    l_run = 0.0f;
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
    for (int x = 0; x < NC; ++x) kf[u][x] = load4(kr + four<FULL>(16 * x + 4 * g, D));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float* vr = vh + __shfl(voff, 4 * g + r);
#pragma unroll
      for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = load4(vr + four<FULL>(4 * (i + 16 * h), D));
    }
    fetch(next);
  };

  // careful: adds values that are not finite by the vector unit, to the rows that see their key
  auto block = [&](auto careful, int u, int t) {
    const int kb = key0(t);
    f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      // (0 times an infinite K would be NaN, not the score)
      const f32x4 kx = decltype(careful)::value ? once<FULL>(kf[u][x], 16 * x + 4 * g, D) : kf[u][x];
#pragma unroll
      for (int e = 0; e < 4; ++e) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[e], qf[x][e], sc, 0, 0, 0);
    }
    const unsigned on = there[u] >> (4 * g);
    if (there[u] != 0xffffu) {  // uniform
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!(on >> r & 1)) {
          sc[r] = -INFINITY;
#pragma unroll
          for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
    // rows that differ in what they see of this block
    const bool cut = c.window > 0 && kb <= p_hi - c.window && kb + kBlk > c.sinks;
    if (kb + kBlk - 1 > p_lo - (TREE ? 1 : 0) || cut) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = kb + 4 * g + r;
        bool see = j <= pos && (c.window == 0 || pos - j < c.window || j < c.sinks);
        if constexpr (TREE) {
          const int a = j - s.first;
          if (a >= 0) see = a < bch::kMaxDrafts && (tree.mask[tok][(a >> 5) & 3] >> (a & 31) & 1);
        }
        if (!see) sc[r] = -INFINITY;
      }
    }
    const float bm = quad_max(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
    const bool move = bm > m_ref + kLazy;  // -inf reference: any finite block max moves it
    if (__any(move)) {
      const float m_new = move ? bm : m_ref;
      const float alpha = m_ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_ref - m_new);
      l_run *= alpha;
#pragma unroll
      for (int n = 0; n < 4 * NH; ++n) acc[n] *= alpha;
      m_ref = m_new;
    }
    const float m_use = m_ref == -INFINITY ? 0.0f : m_ref;
    unsigned seen = 0;
    float rs = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (decltype(careful)::value) seen |= sc[r] == -INFINITY ? 0u : 1u << r;
      sc[r] = __builtin_amdgcn_exp2f(sc[r] - m_use);
      rs += sc[r];
    }
    l_run += quad_sum(rs);
    if constexpr (decltype(careful)::value) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float z = 0.0f;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) z = fmaf(vf[u][r * NH + h][e], 0.0f, z);
        const unsigned long long odd = __ballot(z != 0.0f);
        for (int g2 = 0; g2 < 4; ++g2) {
          if (!(odd >> (16 * g2) & 0xffffu)) continue;
          if (g == g2) {
#pragma unroll
            for (int h = 0; h < NH; ++h) vf[u][r * NH + h] = (f32x4){0.f, 0.f, 0.f, 0.f};
          }
          const float p = __shfl(sc[r], 16 * g2 + i);
          const bool see = __shfl((int)seen, 16 * g2 + i) >> r & 1;
          const float* vr = vh + __shfl(voff, 4 * g2 + r);
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r2 = 0; r2 < 4; ++r2) {
              const int d0 = 4 * (4 * g + r2 + 16 * h);
              const f32x4 x = load4(vr + four<FULL>(d0, D));
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (see) acc[4 * h + e][r2] = fmaf(p, x[e], acc[4 * h + e][r2]);
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
          acc[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[u][r * NH + h][e], sc[r], acc[4 * h + e], 0, 0, 0);
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
    float z = l_run * 0.0f;
#pragma unroll
    for (int n = 0; n < 4 * NH; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) z = fmaf(acc[n][r], 0.0f, z);
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

  // ---- the four wavefronts' results, in wavefront order ----
  if (g == 0) {
    red_m[wave][i] = m_ref;
    red_l[wave][i] = l_run;
  }
  if (wave > 0) {
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) red_o[wave - 1][i][4 * (4 * g + r + 16 * h) + e] = acc[4 * h + e][r];
  }
  __syncthreads();
  if (wave > 0) return;
  float m = red_m[0][i];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red_m[w][i]);
  const float m_use = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float a[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    // a wavefront without a key has m = -inf: its factor is 0 and so is its O
    a[w] = __builtin_amdgcn_exp2f(red_m[w][i] - m_use);
    l += a[w] * red_l[w][i];
  }
#pragma unroll
  for (int n = 0; n < 4 * NH; ++n) acc[n] *= a[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[4 * h + e][r] += a[w] * red_o[w - 1][i][4 * (4 * g + r + 16 * h) + e];

  const int my = rb * kRows + i;
  if (my >= rows) return;
  float* dst;
  float inv = 1.0f;
  if (splits > 1) {
    float* p = part + ((long long)bk * plan.splits + sp) * bch::sdpa_part_floats(plan.max_rows, D);
    dst = p + (long long)my * D;
    if (g == 0) {
      p[(long long)plan.max_rows * D + 2 * my] = m;
      p[(long long)plan.max_rows * D + 2 * my + 1] = l;
    }
  } else {
    dst = c.o + b * c.ol.batch + (long long)(s.row0 + tok) * c.ol.row +
          (long long)(hk * group + row - tok * group) * c.ol.head;
    inv = l == 0.0f ? 0.0f : 1.0f / l;
  }
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d0 = 4 * (4 * g + r + 16 * h);
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[4 * h + e][r] * inv;
      if (FULL || d0 < D) *reinterpret_cast<f32x4u*>(dst + four<FULL>(d0, D)) = x;
    }
}

// o[row] = sum over splits of 2^(m_s - m) O_s / sum of 2^(m_s - m) l_s, in split order: a wavefront per
// row, lane s the maximum and sum of split s.  A split without a key that the row sees has l = 0 and
// counts nothing; a row without any gives zeros.  Rows whose keys were not split are there already.
template <int BLK, bool TREE>
__global__ __launch_bounds__(64) void paged_combine(PagedCall c, PagedPlan plan, const float* __restrict__ part) {
  const int bk = blockIdx.x / plan.max_rows, row = blockIdx.x % plan.max_rows;
  const int b = bk / c.Hkv, hk = bk - b * c.Hkv;
  const bch::Seq s = bch::load_seq(c.kv, c.seqs, b);
  const int group = c.H / c.Hkv, rows = s.n * group;
  if (row >= rows) return;
  const int r0 = row / plan.block_rows * plan.block_rows;
  const int splits = bch::split_count(
      bch::key_list<BLK>(s, r0 / group, (min(r0 + plan.block_rows, rows) - 1) / group, c.window, c.sinks, TREE).n, plan);
  if (splits == 1) return;
  const long long per = bch::sdpa_part_floats(plan.max_rows, c.D);
  const float* p = part + (long long)bk * plan.splits * per;
  const float* ml = p + (long long)plan.max_rows * c.D + 2 * row;
  const int lane = threadIdx.x;
  const bool on = lane < splits;
  const float ms = on ? ml[lane * per] : -INFINITY, ls = on ? ml[lane * per + 1] : 0.0f;
  const float m = bch::wave_allreduce(ms, bch::OpMax());
  const float as = __builtin_amdgcn_exp2f(ms - (m == -INFINITY ? 0.0f : m));
  const float l = bch::wave_allreduce(as * ls, bch::OpSum());
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int tok = row / group;
  float* dst = c.o + b * c.ol.batch + (long long)(s.row0 + tok) * c.ol.row +
               (long long)(hk * group + row - tok * group) * c.ol.head;
  for (int d0 = 0; d0 < c.D; d0 += 64) {
    const int d = d0 + lane;
    const float* po = p + (long long)row * c.D + min(d, c.D - 1);
    float x = 0.0f;
    int u = 0;
    for (; u + 8 <= splits; u += 8) {
      float v[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) v[w] = po[(u + w) * per];
#pragma unroll
      for (int w = 0; w < 8; ++w) x = fmaf(bch::readlane(as, u + w), v[w], x);
    }
    for (; u < splits; ++u) x = fmaf(bch::readlane(as, u), po[u * per], x);
    if (d < c.D) dst[d] = x * inv;
  }
}

// Four workgroups per CU where the sequences may differ in length (the plan knows the longest alone), two
// where there is one; a split keeps at least 128 keys (two blocks a wavefront) and there are at most 64,
// whose results one wavefront still adds quickly.
PagedPlan rows_plan(const PagedCall& c, int max_len, bool may_split) {
  PagedPlan p;
  p.max_rows = c.seqs.max_new * (c.H / c.Hkv);
  p.block_rows = kRows;
  p.tiles = (p.max_rows + kRows - 1) / kRows;
  p.block_keys = kBlk;
  p.min_blocks = 8;
  const long long units = (long long)c.B * c.Hkv * p.tiles;
  const long long want = may_split ? ((c.B > 1 ? 4LL : 2LL) * bch::device_cu_count() + units - 1) / units : 1;
  p.splits = (int)std::max(1LL, std::min({want, bch::most_keys(c, max_len) / (kBlk * p.min_blocks), 64LL}));
  return p;
}

template <int DP>
void launch_dp(hipStream_t s, const PagedCall& c, const PagedPlan& p, float* part) {
  const dim3 grid((unsigned)((long long)c.B * c.Hkv * p.tiles * p.splits)), block(64 * kWaves);
  const bool full = c.D == DP, tree = c.parent != nullptr;
  auto kern = full ? (tree ? sdpa_paged_rows_kernel<DP, true, true> : sdpa_paged_rows_kernel<DP, true, false>)
                   : (tree ? sdpa_paged_rows_kernel<DP, false, true> : sdpa_paged_rows_kernel<DP, false, false>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, c, p, part);
}

}  // namespace

namespace bch {

bool sdpa_paged_rows_applies(const PagedCall& c) {
  const long long rows = (long long)c.seqs.max_new * (c.H / c.Hkv);
  const long long blocks = (long long)c.B * c.Hkv * ((rows + kRows - 1) / kRows);
  return c.D >= 4 && c.D <= 256 && rows <= 0x7fffffff - kRows && blocks * 64 <= 0x7fffffffLL &&
         (long long)c.B * c.Hkv * rows <= 0x7fffffffLL;
}

size_t sdpa_paged_rows_workspace_bytes(const PagedCall& c, int max_len) {
  return paged_part_bytes(c, rows_plan(c, max_len, true));
}

hipError_t launch_sdpa_paged_rows(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes) {
  const PagedPlan p = rows_plan(c, max_len, ws_bytes >= sdpa_paged_rows_workspace_bytes(c, max_len));
  float* part = static_cast<float*>(ws);
  if (c.D <= 64) launch_dp<64>(s, c, p, part);
  else if (c.D <= 128) launch_dp<128>(s, c, p, part);
  else launch_dp<256>(s, c, p, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  return launch_paged_combine(s, c, p, part);
}

hipError_t launch_paged_combine(hipStream_t s, const PagedCall& c, const PagedPlan& p, const float* part) {
  const bool tree = c.parent != nullptr;
  auto kern = p.block_keys == 16 ? (tree ? paged_combine<16, true> : paged_combine<16, false>)
                                 : (tree ? paged_combine<32, true> : paged_combine<32, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)((long long)c.B * c.Hkv * p.max_rows)), dim3(64), 0, s, c, p, part);
  return hipGetLastError();
}

}  // namespace bch
