// sdpa_paged_wide.hip -- attention over a paged cache for many rows a sequence, 128 < D <= 256 (paged.h
// says which keys a row sees).
//
// At these widths the bf16 parts of q, K and V leave no room in registers and LDS for two wavefronts a SIMD
// (sdpa_paged_tile.hip), so the products are f32 ones, v_mfma_f32_16x16x4_f32, whose rate bounds it: a prompt of
// 4096 tokens, 32 heads on 8, D 256, 2.37 ms, 116 TFLOP/s, 74% of the instruction's peak (D 192 1.75 ms); 9.4 and
// 4.9 ms with the 16-row kernel, which reads K and V from L2 for every 16 rows.
//   * A workgroup = eight wavefronts of 16 rows of one key/value head (token t, query head hk * group + g is
//     row t * group + g); q and O stay in registers, D / 4 floats a lane each.  K and V in blocks of 32 keys
//     through LDS as they are, double-buffered (131 KB at D = 256: a workgroup a CU), one barrier a block,
//     loaded two blocks ahead; a wavefront in turn looks up the places of the keys three ahead.
//   * S^T = K Q^T, chains sb = 0, 1 of 16 keys: lane (g = l / 16, i = l % 16) holds K[16 sb + i][16 x + 4 g ..
//     + 3] and q[row i] alike; value r of the result is key 16 sb + 4 g + r of row i.  O^T += V^T P^T: step
//     (sb, r) contracts that key; the lane holds V[key][4 (i + 16 h) .. + 3], component e feeding O block
//     4 h + e, whose value r' is d = 4 (4 g + r' + 16 h) + e.  All reads of LDS are 128 bits (a row of
//     K is 4 floats longer against bank conflicts, which are a quarter of LDS's busy cycles, and those are a sixth
//     of the kernel's), each feeding four matrix instructions.
//   * Online softmax with a lazily moved reference maximum; a wavefront passes over blocks that none of its
//     rows sees.  Lists of blocks, shares and their joining as in the other two kernels.
//   * Columns in fours; one that would reach past D is the row's last one, with the columns that the four
//     before has too zero in q.  Where a result is not finite (a weight of 0 times an infinite V that only
//     other rows see), the workgroup does the list again and adds values that are not finite by the vector
//     unit, to the rows that see their key.
#include "paged.h"

#include <math.h>

#include <type_traits>

namespace {

using bch::f32x4;
using bch::PagedCall;
using bch::SharePlan;

constexpr int kBKV = 32;       // keys per block
constexpr float kLazy = 8.0f;  // log2 headroom before the reference max moves
constexpr int kRows = bch::kWideRows, kNT = 4 * kRows;
constexpr int kOver = bch::kWideOver;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4u*>(p); }
__device__ __forceinline__ f32x4 once(f32x4 x, int d0, int D) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = min(d0, D - 4) + e >= d0 ? x[e] : 0.0f;
  return x;
}

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

struct Ring {
  long long k[4][kBKV], v[4][kBKV];  // offsets of a block's keys; block t in place t % 4
  unsigned there[4];
};

template <int DP, bool TREE>
__global__ __launch_bounds__(kNT, 2) void sdpa_paged_wide_kernel(PagedCall c, SharePlan plan, float* __restrict__ ws) {
  constexpr int NC = DP / 16, NH = DP / 64, NQ = DP / 4, CH = kBKV * NQ / kNT;
  static_assert(kBKV * NQ % kNT == 0, "fours a thread");
  __shared__ __attribute__((aligned(16))) float k_lds[2][kBKV][DP + 4], v_lds[2][kBKV][DP];
  __shared__ Ring ring;
  __shared__ std::conditional_t<TREE, bch::TreeMasks, int> tree;
  __shared__ bch::Share share;
  __shared__ int odd_seen;

  using Line = bch::Shares<kBKV, kRows, kOver, TREE>;
  if (plan.shares > 0 && threadIdx.x < 64) {
    Line::begin(share, c, plan, threadIdx.x);
    Line::next(share, c, plan, threadIdx.x, 0);
  }

  int tree_of = -1;
  bool more = true;
  for (int turn = 0; more; turn ^= 1) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // what follows from it is not held in registers from one piece to the next
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    bch::Piece mine;
    if (plan.shares > 0) {
      __syncthreads();
      mine = bch::read_piece(share.piece[turn]);
      if (mine.count == 0) break;
      if (wave == 0) Line::next(share, c, plan, lane, turn ^ 1);
    } else {
      const bch::Tile own = bch::tile_of(c, plan, blockIdx.x);
      const int of = own.bk / c.Hkv;
      mine = {bch::load_seq(c.kv, c.seqs, of), of, own.bk - of * c.Hkv, own.rb, 0, 0, 0, 1, 1};
      more = false;
    }
    const int b = mine.b, hk = mine.hk, tile = mine.rb;
    const bch::Seq s = mine.seq;
    const int D = c.D, group = c.H / c.Hkv, rows = s.n * group;
    if (plan.shares == 0 && (rows < plan.row_min || tile * kRows >= rows)) break;
    const bch::KeyList keys = bch::key_list<kBKV>(s, tile * kRows / group, (min(tile * kRows + kRows, rows) - 1) / group,
                                                  c.window, c.sinks, TREE);
    if constexpr (TREE) {
      static_assert(kNT >= bch::kMaxDrafts, "tree_masks");
      if (b != tree_of) bch::tree_masks(tree, c.parent, s, c.window, c.sinks);
      tree_of = b;
    }
    const float* kh = c.kv.k + hk * c.kv.kl.head;
    const float* vh = c.kv.v + hk * c.kv.vl.head;
    int t0, t1;
    mine.blocks(keys.n, kOver, t0, t1);

    // ---- a lane's row (past the end: the last one again, not stored), the wavefront's positions ----
    const int r0w = tile * kRows + 16 * wave;
    const int row = min(r0w + i, rows - 1), tok = row / group;
    const int pos = s.first + [&] {
      if constexpr (TREE) return tree.depth[tok];
      else return tok;
    }();
    const int pw_lo = TREE ? s.first : s.first + min(r0w, rows - 1) / group;
    const int pw_hi = s.first + min(r0w + 15, rows - 1) / group;
    auto row_offset = [&](const bch::SdpaLayout& l) {
      return b * l.batch + (long long)(s.row0 + tok) * l.row + (long long)(hk * group + row - tok * group) * l.head;
    };
    f32x4 qf[NC];
    {
      const float* qr = c.q + row_offset(c.ql);
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        const int d0 = 16 * x + 4 * g;
        qf[x] = once(load4(qr + min(d0, D - 4)), d0, D) * c.qscale;
      }
    }

    // ---- where block t's keys stand: lanes 0 .. 31 of the calling wavefront ----
    struct Found {
      bch::Slot slot;
      bool on;
    };
    auto last = [&](int t) { return min(t, t1 - 1); };
    auto find = [&](int t) {
      const int j = keys.key0<kBKV>(t) + (lane & 31);
      Found f;
      f.on = keys.any(j);
      f.slot = f.on ? bch::key_slot(c.kv, b, j) : bch::Slot{-1, 0};
      f.on = f.slot.page >= 0;
      if (!f.on) f.slot = {0, 0};
      return f;
    };
    auto note = [&](int t, const Found& f) {
      const unsigned there = (unsigned)__ballot(f.on);
      if (lane < kBKV) {
        ring.k[t & 3][lane] = bch::slot_offset(c.kv.kl, f.slot);
        ring.v[t & 3][lane] = bch::slot_offset(c.kv.vl, f.slot);
        if (lane == 0) ring.there[t & 3] = there;
      }
    };
    auto there = [&](int t) { return (unsigned)__builtin_amdgcn_readfirstlane(ring.there[t & 3]); };

    // ---- global -> registers -> LDS: four ch of a block is key ch / NQ, d 4 (ch % NQ) .. + 3 ----
    f32x4 rk[CH], rv[CH];
    auto load = [&](int t) {
#pragma unroll
      for (int n = 0; n < CH; ++n) {
        const int ch = tid + n * kNT, key = ch / NQ, d = min(4 * (ch % NQ), D - 4);
        rk[n] = load4(kh + ring.k[t & 3][key] + d);
        rv[n] = load4(vh + ring.v[t & 3][key] + d);
      }
    };
    auto store = [&](int t, int buf) {
      const unsigned on = there(t);
#pragma unroll
      for (int n = 0; n < CH; ++n) {
        const int ch = tid + n * kNT, key = ch / NQ, d = 4 * (ch % NQ);
        const bool is = on >> key & 1;
        *reinterpret_cast<f32x4*>(&k_lds[buf][key][d]) = is ? rk[n] : (f32x4){0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<f32x4*>(&v_lds[buf][key][d]) = is ? rv[n] : (f32x4){0.f, 0.f, 0.f, 0.f};
      }
    };

    f32x4 acc[4 * NH];
    float m_ref, l_run;
    // careful: adds values that are not finite by the vector unit, to the rows that see their key
    auto block = [&](auto careful, int t, int buf) {
      const int kb = keys.key0<kBKV>(t);
      f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        f32x4 kx[2];
#pragma unroll
        for (int sb = 0; sb < 2; ++sb) {
          kx[sb] = *reinterpret_cast<const f32x4*>(&k_lds[buf][16 * sb + i][16 * x + 4 * g]);
          // (0 times an infinite K would be NaN, not the score)
          if (decltype(careful)::value) kx[sb] = once(kx[sb], 16 * x + 4 * g, D);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int sb = 0; sb < 2; ++sb)
            sc[sb] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[sb][e], qf[x][e], sc[sb], 0, 0, 0);
      }
      // rows that differ in what they see of this block, or keys that are not there
      const unsigned on = there(t);
      const bool cut = c.window > 0 && kb <= max(pw_hi, 0) - c.window && kb + kBKV > c.sinks;
      if (on != ~0u || kb + kBKV - 1 > pw_lo - (TREE ? 1 : 0) || cut) {
        const int low = c.window > 0 ? pos - c.window : -1;  // keys above it, or sinks (pos >= 0 where any key is)
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int o = 16 * sb + 4 * g + r, j = kb + o;
            bool see = j <= pos && (j > low || j < c.sinks);
            if constexpr (TREE) {
              const int a = j - s.first;
              if (a >= 0) see = a < bch::kMaxDrafts && (tree.mask[tok][(a >> 5) & 3] >> (a & 31) & 1);
            }
            if (!see || !(on >> o & 1)) sc[sb][r] = -INFINITY;
          }
      }
      float bm = sc[0][0];
#pragma unroll
      for (int n = 1; n < 8; ++n) bm = fmaxf(bm, sc[n >> 2][n & 3]);
      bm = quad_max(bm);
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
      unsigned seen = 0;  // bit 4 sb + r
      float rs = 0.0f;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float x = sc[n >> 2][n & 3];
        if (decltype(careful)::value) seen |= x == -INFINITY ? 0u : 1u << n;
        sc[n >> 2][n & 3] = __builtin_amdgcn_exp2f(x - m_use);
        rs += sc[n >> 2][n & 3];
      }
      l_run += quad_sum(rs);
      unsigned odd = 0;  // keys with values that are not finite
      if constexpr (decltype(careful)::value) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float* vr = &v_lds[buf][16 * (n >> 2) + 4 * g + (n & 3)][4 * i];
          float z = 0.0f;
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) z = fmaf(vr[64 * h + e], 0.0f, z);
          const unsigned long long lanes = __ballot(z != 0.0f);
          for (int g2 = 0; g2 < 4; ++g2)
            if (lanes >> (16 * g2) & 0xffffu) odd |= 1u << (16 * (n >> 2) + 4 * g2 + (n & 3));
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int key = 16 * (n >> 2) + 4 * g + (n & 3);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          f32x4 vx = *reinterpret_cast<const f32x4*>(&v_lds[buf][key][4 * i + 64 * h]);
          if (decltype(careful)::value && (odd >> key & 1)) vx = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[e], sc[n >> 2][n & 3], acc[4 * h + e], 0, 0, 0);
        }
      }
      if constexpr (decltype(careful)::value) {
#pragma unroll 1
        for (; odd; odd &= odd - 1) {
          const int key = __ffs(odd) - 1, at = 4 * (key >> 4) + (key & 3), from = 4 * (key & 12) + i;
          float p = sc[0][0];
#pragma unroll
          for (int n = 1; n < 8; ++n) p = n == at ? sc[n >> 2][n & 3] : p;
          p = __shfl(p, from);
          const bool see = __shfl((int)seen, from) >> at & 1;
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (see) acc[4 * h + e][r] = fmaf(p, v_lds[buf][key][4 * (4 * g + r + 16 * h) + e], acc[4 * h + e][r]);
        }
      }
    };
    auto unseen = [&](int kb) {  // no row of the wavefront sees any of the block
      return r0w >= rows || kb > pw_hi || (c.window > 0 && kb + kBKV - 1 <= max(pw_lo, 0) - c.window && kb >= c.sinks);
    };

    // Block t: the next one to the other buffer (which the last barrier released), the loads of the one after
    // it, the places of the one after that.  Blocks past the end are the last one again, never read.
    auto run = [&](auto careful) {
#pragma unroll
      for (int n = 0; n < 4 * NH; ++n) acc[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
      m_ref = -INFINITY;
      l_run = 0.0f;
      if (t0 >= t1) return;
      if (wave < 3) note(t0 + wave, find(last(t0 + wave)));
      __syncthreads();
      load(t0);
      store(t0, 0);
      load(t0 + 1);
      __syncthreads();
#pragma unroll 1
      for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        const bool turn_to_look = wave == (t & 7);
        Found f{};
        if (turn_to_look) f = find(last(t + 3));
        store(t + 1, cur ^ 1);
        load(t + 2);
        if (!unseen(keys.key0<kBKV>(t))) block(careful, t, cur);
        if (turn_to_look) note(t + 3, f);
        __syncthreads();
      }
    };
    if (tid == 0) odd_seen = 0;
    run(std::false_type{});
    {
      float z = l_run * 0.0f;
#pragma unroll
      for (int n = 0; n < 4 * NH; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = fmaf(acc[n][r], 0.0f, z);
      if (z != 0.0f) odd_seen = 1;
      __syncthreads();
      if (odd_seen) run(std::true_type{});
    }

    // ---- epilogue: value r of block 4 h + e is d = 4 (4 g + r + 16 h) + e ----
    if (tid == 0) bch::note_list(ws, c, plan, mine);
    if (r0w + i < rows) {
      float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
      float* dst;
      if (mine.count > 1) {
        float* p = bch::part_of(ws, c, plan, mine);
        const int at = row - tile * kRows;
        dst = p + (long long)at * D;
        inv = 1.0f;
        if (g == 0) {
          p[(long long)plan.part_rows * D + 2 * at] = m_ref;
          p[(long long)plan.part_rows * D + 2 * at + 1] = l_run;
        }
      } else {
        dst = c.o + row_offset(c.ol);
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d0 = 4 * (4 * g + r + 16 * h);
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = acc[4 * h + e][r] * inv;
          if (d0 < D) *reinterpret_cast<f32x4u*>(dst + min(d0, D - 4)) = x;
        }
    }
  }
}

template <int DP>
void launch_dp(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  const dim3 grid((unsigned)(p.shares > 0 ? (long long)p.shares : bch::lists_of(c, p))), block(kNT);
  auto kern = c.parent ? sdpa_paged_wide_kernel<DP, true> : sdpa_paged_wide_kernel<DP, false>;
  hipLaunchKernelGGL(kern, grid, block, 0, s, c, p, ws);
}

}  // namespace

namespace bch {

hipError_t launch_sdpa_paged_wide(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  if (c.D <= 192) launch_dp<192>(s, c, p, ws);
  else launch_dp<256>(s, c, p, ws);
  return hipGetLastError();
}

}  // namespace bch
