// sdpa_paged_tile.hip -- attention over a paged cache for many rows a sequence: prompts, chunks of
// them, large trees of drafts (paged.h says which keys a row sees).  8 <= D <= 128.
//
// What bounds it: the matrix cores at the clock that the power limit leaves them: a 16384-token prompt, window
// 4096, 32 heads on 8, D 128, 4.56 ms, 211 TFLOP/s of f32 products, matrix cores busy 61% of the cycles at 1.92
// GHz.  A list's beginning and end cost about 16 us, most of the time of a list of six blocks.
//
// Both products on the bf16 matrix cores, three exact bf16 parts per f32 and six part products
// accumulated in f32 (bch_internal.h, split8), arranged as in sdpa_fwd.hip:
//   * A workgroup = eight wavefronts of 32 rows of one key/value head: token t, query head hk * group + g is
//     row t * group + g, so that the query heads that share K and V share their conversion too, and a
//     workgroup's rows stand close together: a window adds few keys that only some of them see.  Key
//     blocks of 32 are split into parts on their way into LDS, once per workgroup, double-buffered, one
//     barrier per block, loaded two blocks ahead.
//   * S^T = K Q^T (32 keys x 32 rows): each lane holds 16 scores of its row; O^T += V^T P^T takes P from
//     the same registers.  Online softmax with a lazily moved reference maximum.
//   * The blocks of the sinks and of the window's keys are one list; a wavefront passes over the ones that
//     none of its rows sees and masks only those that some do not see whole.
//   * Where the keys stand: each iteration one wavefront looks up the 32 keys of the block three ahead
//     and leaves their offsets, and a word that says which are there, in a ring in LDS.  Keys that are
//     not there are staged as zeros.
//   * Where the parts cannot stand for the operands (|q scale log2(e)| or |K| from 2^43 on, or a result
//     that is not finite), the wavefront does its rows again on v_mfma_f32_32x32x2_f32 from global memory,
//     and there adds values that are not finite by the vector unit, to the rows that see them: a
//     weight of 0 times an infinity must not reach the rows that do not.
#include "paged.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace {

using bch::bf16_mm;
using bch::f32x16;
using bch::PagedCall;
using bch::SharePlan;
using bch::split8;
using bch::u32x4;

constexpr int kBKV = 32;       // keys per block
constexpr float kLazy = 8.0f;  // log2 headroom before the reference max moves
// 128 products of operands below this, scaled by 2^32, stay below 2^127 (sdpa_fwd.hip).
constexpr float kScoreBig = 0x1p43f;

__device__ __forceinline__ float half_swap_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS of one key block, three parts each of K, [d octet][32 keys][8 d] (a key's place permuted by the
// octet, key ^ octet % 8), and of V, [4 key octets][DP][8 keys].  At DP = 128 the smallest part of q for
// QL of the eight 16-d steps is kept in LDS too, which leaves two wavefronts per SIMD their registers.
template <int DP>
struct TileCfg {
  static constexpr int NW = 8, NT = 64 * NW, BQ = bch::kTileRows;
  static_assert(BQ == 32 * NW, "32 rows a wavefront");
  static constexpr int NO = DP / 8;
  static constexpr int KSTR = kBKV * 16, VSTR = DP * 16;
  static constexpr int KBYTES = 3 * NO * KSTR, VBYTES = 3 * 4 * VSTR;
  static constexpr int QL = DP == 128 ? 7 : 0;
  static constexpr int NCH = kBKV * NO;           // octets of K, and of V, per block
  static constexpr int CH = (NCH + NT - 1) / NT;  // per thread
};
// A list's beginning and end take about as long as four blocks.
constexpr int kOver = 4;
struct Ring {
  long long k[4][kBKV], v[4][kBKV];  // offsets of a block's keys; block t in place t % 4
  unsigned there[4];
};

// FULL: D == DP; otherwise D >= 8 and an octet of columns that would reach past D is the row's last
// one, with its columns below the octet's zero in q (they count in the octet before).
template <int DP, bool FULL, bool TREE>
__global__ __launch_bounds__(TileCfg<DP>::NT) void sdpa_paged_tile_kernel(PagedCall c, SharePlan plan,
                                                                          float* __restrict__ ws) {
  using G = TileCfg<DP>;
  constexpr int NT = G::NT, NW = G::NW, NO = G::NO, NC = DP / 16, NBK = DP / 32;
  __shared__ __attribute__((aligned(16))) char k_lds[2 * G::KBYTES], v_lds[2 * G::VBYTES];
  __shared__ u32x4 q_lds[G::QL > 0 ? G::QL * NT : 1];
  __shared__ Ring ring;
  __shared__ std::conditional_t<TREE, bch::TreeMasks, int> tree;
  __shared__ bch::Share share;
  __shared__ int big_seen;

  // a lane number computed anew wherever this is called: what follows from it is not held in registers
  // through the loops in between
  auto anew = [](int l) {
    asm volatile("" : "+v"(l));
    return l;
  };
  using Line = bch::Shares<kBKV, G::BQ, kOver, TREE>;
  if (plan.shares > 0 && threadIdx.x < 64) {
    Line::begin(share, c, plan, threadIdx.x);
    Line::next(share, c, plan, threadIdx.x, 0);
  }

  int tree_of = -1;
  bool more = true;
  for (int turn = 0; more; turn ^= 1) {
    const int tid = anew(threadIdx.x);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
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
    const int group = c.H / c.Hkv, rows = s.n * group;
    if (plan.shares == 0 && (rows < plan.row_min || tile * G::BQ >= rows)) break;
    const bch::KeyList keys = bch::key_list<kBKV>(s, tile * G::BQ / group, (min(tile * G::BQ + G::BQ, rows) - 1) / group,
                                                  c.window, c.sinks, TREE);
    if constexpr (TREE) {
      static_assert(NT >= bch::kMaxDrafts, "tree_masks");
      if (b != tree_of) bch::tree_masks(tree, c.parent, s, c.window, c.sinks);
      tree_of = b;
    }
    const int D = c.D;
    const float* kh = c.kv.k + hk * c.kv.kl.head;
    const float* vh = c.kv.v + hk * c.kv.vl.head;

    // a lane's row (past the end: the last one again, not stored), and the wavefront's tokens
    const int r0w = tile * G::BQ + wave * 32;
    struct Row {
      int row, tok;
    };
    auto lane_row = [&](int l) {
      const int row = min(r0w + (l & 31), rows - 1);
      return Row{row, row / group};
    };
    auto row_offset = [&](const bch::SdpaLayout& l, Row r) {
      return b * l.batch + (long long)(s.row0 + r.tok) * l.row + (long long)(hk * group + r.row - r.tok * group) * l.head;
    };
    const int tok = lane_row(lane).tok;
    const int pos = s.first + [&] {
      if constexpr (TREE) return tree.depth[tok];
      else return tok;
    }();
    const int pw_lo = TREE ? s.first : s.first + min(r0w, rows - 1) / group;
    const int pw_hi = s.first + min(r0w + 31, rows - 1) / group;

    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    auto row8 = [&](const float* p, int d0, float (&x)[8]) {
      const int d = FULL ? d0 : min(d0, D - 8);
      const f32x4u a = *reinterpret_cast<const f32x4u*>(p + d), e4 = *reinterpret_cast<const f32x4u*>(p + d + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = a[e];
        x[4 + e] = e4[e];
      }
    };
    auto once = [&](int d0, float (&x)[8]) {
      if (!FULL) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = min(d0, D - 8) + e >= d0 ? x[e] : 0.0f;
      }
    };

    f32x16 oacc[NBK];
    float m_ref, l_run;
    auto reset = [&]() {
#pragma unroll
      for (int n = 0; n < NBK; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[n][r] = 0.0f;
      m_ref = -INFINITY;
      l_run = 0.0f;
    };
    reset();

    int t0, t1;
    mine.blocks(keys.n, kOver, t0, t1);

    // ---- where block t's keys stand: lanes 0 .. 31 of the calling wavefront ----
    struct Found {
      bch::Slot slot;
      bool on;
    };
    auto find = [&](int t) {
      const int j = keys.key0<kBKV>(t) + li;
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
        ring.k[t & 3][li] = bch::slot_offset(c.kv.kl, f.slot);
        ring.v[t & 3][li] = bch::slot_offset(c.kv.vl, f.slot);
        if (lane == 0) ring.there[t & 3] = there;
      }
    };
    auto there = [&](int t) { return (unsigned)__builtin_amdgcn_readfirstlane(ring.there[t & 3]); };

    // ---- global -> registers -> parts in LDS ----
    // octet ch of K: key ch / NO, d 8 (ch % NO) .. + 7; of V: column ch % DP, key octet ch / DP (keys
    // 16 (oct / 2) + 4 (oct % 2) + {0..3, 8..11})
    float rk[G::CH][8], rv[G::CH][8];
    float mk = 0.0f;  // largest magnitude of the K that this thread has split
    auto load_k = [&](int t) {
#pragma unroll
      for (int n = 0; n < G::CH; ++n) {
        const int ch = (G::NCH % NT == 0) ? tid + n * NT : min(tid + n * NT, G::NCH - 1);
        row8(kh + ring.k[t & 3][ch / NO], 8 * (ch % NO), rk[n]);
      }
    };
    auto load_v = [&](int t) {
#pragma unroll
      for (int n = 0; n < G::CH; ++n) {
        const int ch = (G::NCH % NT == 0) ? tid + n * NT : min(tid + n * NT, G::NCH - 1);
        const int oct = ch / DP, d = FULL ? ch % DP : min(ch % DP, D - 1);
        const long long* off = ring.v[t & 3] + 16 * (oct >> 1) + 4 * (oct & 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) rv[n][e] = (vh + off[(e & 3) + 8 * (e >> 2)])[d];
      }
    };
    auto zero_missing = [&](unsigned on) {
#pragma unroll
      for (int n = 0; n < G::CH; ++n) {
        const int ch = (G::NCH % NT == 0) ? tid + n * NT : min(tid + n * NT, G::NCH - 1);
        const int oct = ch / DP, k0 = 16 * (oct >> 1) + 4 * (oct & 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!(on >> (ch / NO) & 1)) rk[n][e] = 0.0f;
          if (!(on >> (k0 + (e & 3) + 8 * (e >> 2)) & 1)) rv[n][e] = 0.0f;
        }
      }
    };
    // The first trips to memory go together: q and the places of three blocks, then the first block's K and V
    // while q is split.
    auto last = [&](int t) { return min(t, t1 - 1); };
    // ---- q parts: step n holds q[row][16 n + 8 lh .. + 7] * scale * log2(e) ----
    const float* const q0 = c.q + row_offset(c.ql, lane_row(lane));
    float qx[NC][8];
#pragma unroll
    for (int n = 0; n < NC; ++n) row8(q0, 16 * n + 8 * lh, qx[n]);

    if (tid == 0) big_seen = 0;
    // (past the end: the last block's places under a number that is never read)
    if (t0 < t1 && wave < 3) note(t0 + wave, find(last(t0 + wave)));
    __syncthreads();
    if (t0 < t1) {
      load_k(t0);
      load_v(t0);
    }
    u32x4 qf[NC][3];
    float mq = 0.0f;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      once(16 * n + 8 * lh, qx[n]);
#pragma unroll
      for (int e = 0; e < 8; ++e) mq = fmaxf(mq, fabsf(qx[n][e] * c.qscale));
      split8(qx[n], qf[n], c.qscale * bch::kSplitScale);
      if (n < G::QL) q_lds[n * NT + tid] = qf[n][2];  // read back by this lane alone
    }
    const bool q_big = __any(mq >= kScoreBig);  // settled here: later, the floats of q would stay in registers

    u32x4 kp[G::CH][3], vp[G::CH][3];
    // one of the 8 CH pairs of floats of this thread's octets: V's first, then K's
    constexpr int UNITS = 8 * G::CH;
    auto split_unit = [&](int u) {
      const int n = (u >> 2) % G::CH, e = u & 3;
      float& x = u < UNITS / 2 ? rv[n][2 * e] : rk[n][2 * e];
      float& y = u < UNITS / 2 ? rv[n][2 * e + 1] : rk[n][2 * e + 1];
      if (u >= UNITS / 2) mk = fmaxf(mk, fmaxf(fabsf(x), fabsf(y)));
      x *= bch::kSplitScale;
      y *= bch::kSplitScale;
      bch::split2(x, y, u < UNITS / 2 ? vp[n] : kp[n], e);
    };
    auto store_k = [&](int buf) {
      char* p = k_lds + buf * G::KBYTES;
#pragma unroll
      for (int n = 0; n < G::CH; ++n) {
        const int ch = tid + n * NT;
        if (G::NCH % NT == 0 || ch < G::NCH) {
#pragma unroll
          for (int p3 = 0; p3 < 3; ++p3)
            *reinterpret_cast<u32x4*>(p + (p3 * NO + ch % NO) * G::KSTR + ((ch / NO) ^ (ch % NO & 7)) * 16) = kp[n][p3];
        }
      }
    };
    auto store_v = [&](int buf) {
      char* p = v_lds + buf * G::VBYTES;
#pragma unroll
      for (int n = 0; n < G::CH; ++n) {
        const int ch = tid + n * NT;
        if (G::NCH % NT == 0 || ch < G::NCH) {
#pragma unroll
          for (int p3 = 0; p3 < 3; ++p3)
            *reinterpret_cast<u32x4*>(p + (p3 * 4 + ch / DP) * G::VSTR + (ch % DP) * 16) = vp[n][p3];
        }
      }
    };

    // value r of a score block: key kb + 8 (r / 4) + 4 lh + r % 4 of this lane's row
    auto mask = [&](f32x16& x, int kb, unsigned on) {
      const int low = c.window > 0 ? pos - c.window : -1;  // keys above it, or sinks (pos >= 0 where any key is)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int o = 8 * (r >> 2) + 4 * lh + (r & 3), j = kb + o;
        bool see = j <= pos && (j > low || j < c.sinks);
        if constexpr (TREE) {
          const int a = j - s.first;
          if (a >= 0) see = a < bch::kMaxDrafts && (tree.mask[tok][(a >> 5) & 3] >> (a & 31) & 1);
        }
        if (!see || !(on >> o & 1)) x[r] = -INFINITY;
      }
    };
    auto cut = [&](int kb) {  // some row of the wavefront does not see some key of the block
      return kb + kBKV - 1 > pw_lo - (TREE ? 1 : 0) ||
             (c.window > 0 && kb <= max(pw_hi, 0) - c.window && kb + kBKV > c.sinks);
    };
    auto unseen = [&](int kb) {  // none sees any
      return r0w >= rows || kb > pw_hi || (c.window > 0 && kb + kBKV - 1 <= max(pw_lo, 0) - c.window && kb >= c.sinks);
    };

    // Scores -> probabilities against the reference max, which moves when a block exceeds it by more than
    // 2^kLazy, and their parts pf, in kPieces pieces.  unit: the scores' scale.  alpha: what the results so
    // far are to be multiplied by.
    u32x4 pf[2][3];
    float bm, m_use, rs, alpha;
    constexpr int kPieces = 20;
    auto piece = [&](float unit, f32x16& x, int i) {
      if (i == 0) {
        bm = x[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) bm = fmaxf(bm, x[r]);
      } else if (i == 1) {
#pragma unroll
        for (int r = 8; r < 16; ++r) bm = fmaxf(bm, x[r]);
        bm = half_swap_max(bm) * unit;
      } else if (i == 2) {
        const bool move = bm > m_ref + kLazy;  // -inf reference: any finite block max moves it
        const float m_new = move ? bm : m_ref;
        alpha = move ? (m_ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_ref - m_new)) : 1.0f;
        m_ref = m_new;
        m_use = (m_ref == -INFINITY) ? 0.0f : m_ref;
        rs = 0.0f;
      } else if (i < 11) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 2 * (i - 3) + e;
          x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], unit, -m_use));
          rs += x[r];
        }
      } else if (i == 11) {
        l_run = l_run * alpha + half_swap_sum(rs);
      } else {
        const int u = i - 12, h = u >> 2, e = u & 3;
        float y = x[8 * h + 2 * e] * bch::kSplitScale, z = x[8 * h + 2 * e + 1] * bch::kSplitScale;
        bch::split2(y, z, pf[h], e);
      }
    };
    auto softmax = [&](float unit, f32x16& x) {  // without the parts
#pragma unroll
      for (int i = 0; i < 12; ++i) piece(unit, x, i);
      return alpha;
    };
    auto rescale = [&](float a) {
      if (__any(a != 1.0f)) {
#pragma unroll
        for (int n = 0; n < NBK; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[n][r] *= a;
      }
    };

    // the scores of the block in buffer buf, with work(i) behind MFMA i of 6 NC
    auto qk = [&](int buf, f32x16& x, auto&& work) {
      const char* ks = k_lds + buf * G::KBYTES + lh * G::KSTR;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = 0.0f;
      u32x4 kf[2][3], q2[2];
      auto read = [&](int n) {  // octet 2 n + lh
        const int key = li ^ ((2 * n + lh) & 7);
#pragma unroll
        for (int p3 = 0; p3 < 3; ++p3)
          kf[n & 1][p3] = *reinterpret_cast<const u32x4*>(ks + (p3 * NO + 2 * n) * G::KSTR + key * 16);
        q2[n & 1] = n < G::QL ? q_lds[n * NT + tid] : qf[n][2];
      };
      read(0);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        if (n + 1 < NC) read(n + 1);
#pragma unroll
        for (int y = 0; y < 6; ++y) {
          const int pb = bch::kPartB[y];
          x = bf16_mm(kf[n & 1][bch::kPartA[y]], pb == 2 ? q2[n & 1] : qf[n][pb], x);
          work(6 * n + y);
        }
      }
    };
    // O += V^T P^T of the block in buffer buf
    auto pv = [&](int buf) {
      const char* vs = v_lds + buf * G::VBYTES + lh * G::VSTR + li * 16;
      u32x4 vf[2][3];
      auto read = [&](int i) {  // 16-k step i / NBK, O block i % NBK
#pragma unroll
        for (int p3 = 0; p3 < 3; ++p3)
          vf[i & 1][p3] = *reinterpret_cast<const u32x4*>(vs + (p3 * 4 + 2 * (i / NBK)) * G::VSTR + (i % NBK) * 512);
      };
      read(0);
#pragma unroll
      for (int i = 0; i < 2 * NBK; ++i) {
        if (i + 1 < 2 * NBK) read(i + 1);
#pragma unroll
        for (int y = 0; y < 6; ++y)
          oacc[i % NBK] = bf16_mm(vf[i & 1][bch::kPartA[y]], pf[i / NBK][bch::kPartB[y]], oacc[i % NBK]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    // Block t: its scores run over the conversion of block t + 1's K and V (stored to the other buffers,
    // which the previous barrier released), then the softmax and the PV product.  Blocks past the end are clamped to the last one (reloaded, never read).
    if (t0 < t1) {
      if (there(t0) != ~0u) zero_missing(there(t0));
#pragma unroll
      for (int u = 0; u < UNITS; ++u) split_unit(u);
      store_v(0);
      store_k(0);
      load_k(t0 + 1);
      load_v(t0 + 1);
    }
    __syncthreads();
    // block t + 1 to the other buffers, block t + 2's loads, block t + 3's places
    auto stage = [&](int t, bool turn, const Found& f) {
      const int nxt = (t - t0 + 1) & 1;
      store_v(nxt);
      store_k(nxt);
      load_k(t + 2);
      load_v(t + 2);
      if (turn) note(t + 3, f);
    };
    auto look = [&](int t, Found& f) {
      const bool turn = wave == (t & (NW - 1));
      if (turn) f = find(last(t + 3));
      if (there(t + 1) != ~0u) zero_missing(there(t + 1));
      return turn;
    };
    // The blocks that this wavefront's rows see are the sinks' and a run of the window's; past the others it
    // only stages.
    int t = t0;
    while (t < t1) {
#pragma unroll 1
      for (; t < t1 && !unseen(keys.key0<kBKV>(t)); ++t) {
        const int cur = (t - t0) & 1, kb = keys.key0<kBKV>(t);
        constexpr int NQ = 6 * NC;
        Found f;
        const bool turn = look(t, f);
        f32x16 x;
        qk(cur, x, [&](int i) {
#pragma unroll
          for (int u = 0; u < UNITS; ++u)
            if (u * NQ / UNITS == i) split_unit(u);
          __builtin_amdgcn_sched_barrier(0);
        });
        stage(t, turn, f);
        __builtin_amdgcn_sched_barrier(0);
        const unsigned th = there(t);
        if (th != ~0u || cut(kb)) mask(x, kb, th);
        rescale(softmax(bch::kSplitUnscale, x));
#pragma unroll
        for (int i = 12; i < kPieces; ++i) piece(bch::kSplitUnscale, x, i);
        __builtin_amdgcn_sched_barrier(0);
        pv(cur);
        __syncthreads();
      }
#pragma unroll 1
      for (; t < t1 && unseen(keys.key0<kBKV>(t)); ++t) {
        Found f;
        const bool turn = look(t, f);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) split_unit(u);
        stage(t, turn, f);
        __syncthreads();
      }
    }

    // ---- O scaled back; where the parts cannot stand for the operands, these rows again in f32 ----
    bool redo;
    {
      float z = l_run * 0.0f;
#pragma unroll
      for (int n = 0; n < NBK; ++n) {
        oacc[n] *= bch::kSplitUnscale;
#pragma unroll
        for (int r = 0; r < 16; ++r) z = fmaf(oacc[n][r], 0.0f, z);
      }
      if (mk >= kScoreBig) big_seen = 1;
      __syncthreads();
      redo = q_big || big_seen != 0 || __any(z != 0.0f);
    }
    if (redo && r0w < rows) {
      reset();
      const float* const qr = c.q + row_offset(c.ql, lane_row(anew(lane)));
#pragma unroll 1
      for (int t = t0; t < t1; ++t) {
        const int kb = keys.key0<kBKV>(t);
        if (unseen(kb)) continue;
        const Found f = find(t);
        const unsigned th = (unsigned)__ballot(f.on);  // lanes 0 .. 31
        const float* kr = kh + bch::slot_offset(c.kv.kl, f.slot);
        const long long voff = bch::slot_offset(c.kv.vl, f.slot);
        f32x16 x;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.0f;
#pragma unroll 1
        for (int d0 = 0; d0 < DP; d0 += 16) {
          float y[8], w[8];
          row8(kr, d0 + 8 * lh, y);
          once(d0 + 8 * lh, y);
          row8(qr, d0 + 8 * lh, w);
          once(d0 + 8 * lh, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) x = __builtin_amdgcn_mfma_f32_32x32x2f32(y[e], w[e] * c.qscale, x, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        mask(x, kb, th);
        unsigned seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) seen |= x[r] == -INFINITY ? 0u : 1u << r;
        rescale(softmax(1.0f, x));
        unsigned odd = 0;  // keys with values that are not finite
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int o = 8 * (r >> 2) + 4 * lh + (r & 3);
          const float* vr = vh + __shfl(voff, o);
          float y[NBK], z = 0.0f;
#pragma unroll
          for (int n = 0; n < NBK; ++n) {
            y[n] = th >> o & 1 ? vr[min(32 * n + li, D - 1)] : 0.0f;
            z = fmaf(y[n], 0.0f, z);
          }
          const unsigned long long lanes = __ballot(z != 0.0f);
          odd |= ((unsigned)lanes ? 1u : 0u) << (8 * (r >> 2) + (r & 3));
          odd |= ((unsigned)(lanes >> 32) ? 1u : 0u) << (8 * (r >> 2) + 4 + (r & 3));
#pragma unroll
          for (int n = 0; n < NBK; ++n)
            oacc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(odd >> o & 1 ? 0.0f : y[n], x[r], oacc[n], 0, 0, 0);
        }
#pragma unroll 1
        for (; odd; odd &= odd - 1) {
          const int o = __ffs(odd) - 1, at = 4 * (o >> 3) + (o & 3), from = 8 * (o & 4) + li;
          float p = x[0];
#pragma unroll
          for (int r = 1; r < 16; ++r) p = r == at ? x[r] : p;
          p = __shfl(p, from);
          const bool see = __shfl((int)seen, from) >> at & 1;
          const float* wr = vh + __shfl(voff, o);
#pragma unroll
          for (int n = 0; n < NBK; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float w = wr[min(32 * n + 8 * (e >> 2) + 4 * lh + (e & 3), D - 1)];
              if (see) oacc[n][e] = fmaf(p, w, oacc[n][e]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- epilogue: value r of block n is d = 32 n + 8 (r / 4) + 4 lh + r % 4 ----
    if (tid == 0) bch::note_list(ws, c, plan, mine);
    const Row me = lane_row(anew(lane));
    if (r0w + li < rows) {
      float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
      float* dst;
      if (mine.count > 1) {
        float* p = bch::part_of(ws, c, plan, mine);
        const int at = me.row - tile * G::BQ;
        dst = p + (long long)at * D;
        inv = 1.0f;
        if (lh == 0) {
          p[(long long)plan.part_rows * D + 2 * at] = m_ref;
          p[(long long)plan.part_rows * D + 2 * at + 1] = l_run;
        }
      } else {
        dst = c.o + row_offset(c.ol, me);
      }
#pragma unroll
      for (int n = 0; n < NBK; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int d = 32 * n + 2 * r + 4 * lh;
          if (FULL || d + 3 < D) {
            *reinterpret_cast<f32x4u*>(dst + d) =
                f32x4u{oacc[n][r] * inv, oacc[n][r + 1] * inv, oacc[n][r + 2] * inv, oacc[n][r + 3] * inv};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < D) dst[d + e] = oacc[n][r + e] * inv;
          }
        }
    }
  }
}

template <int DP>
void launch_dp(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  const long long lists = bch::lists_of(c, p);
  const dim3 grid((unsigned)(p.shares > 0 ? (long long)p.shares : lists)), block(TileCfg<DP>::NT);
  const bool full = c.D == DP, tree = c.parent != nullptr;
  auto kern = full ? (tree ? sdpa_paged_tile_kernel<DP, true, true> : sdpa_paged_tile_kernel<DP, true, false>)
                   : (tree ? sdpa_paged_tile_kernel<DP, false, true> : sdpa_paged_tile_kernel<DP, false, false>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, c, p, ws);
}

}  // namespace

namespace bch {

// Up to a tile for every second CU: equal shares of their key blocks, a workgroup each, a share four blocks
// at least.  More: a workgroup a tile, last ones first; a prompt's lists differ in length, which shares do not
// know.  Up to two tiles a CU shares too where that hardly matters (keys more than twice the new tokens) and the
// lists are long: whole ones leave CUs idle where sequences differ.  Measured, a workgroup a tile / shares, us (32 heads on 8, D 128): 64 tiles of a 512-token prompt 84 / 66,
// behind 3584 keys 514 / 202; 128 tiles, 1024 tokens 146 / 123 (window 512: 93 / 111); 256 tiles, 2048 tokens
// 276 / 298, eight prompts of 256 55 / 76.  Chunks: four of up to 700 tokens, 2048 keys, 271 / 201; eight of up to 256,
// 4096 keys, 509 / 191, all of 256 627 / 654; sixteen of 128, window 512, 109 / 126.  Four prompts of up to 2048 tokens
// 281 / 359 (D 256, three chunks of up to 600, 5000 keys: 1378 / 886).
SharePlan sdpa_paged_tile_plan(const PagedCall& c, int max_len, bool may_split) {
  SharePlan p;
  const int group = c.H / c.Hkv;
  const long long cu = device_cu_count();
  p.row_min = kFewRows + 1;
  p.row_max = 0x7fffffff;
  const int most = c.seqs.max_new * group;
  p.rows = tile_rows(c.D);
  p.tiles = (most - 1) / p.rows + 1;
  p.part_rows = std::min(most, p.rows);
  p.min_share = c.D <= kTileDim ? 4 + kOver : 2 + kWideOver;
  // full tiles that there are: a batch's rows, or every sequence's
  const long long rows = (long long)c.Hkv * group * (c.seqs.start ? c.seqs.total : (long long)c.B * c.seqs.max_new);
  const long long full = rows / p.rows, keys = most_keys(c, max_len);
  const bool alike = keys >= 1024 && keys > 2LL * c.seqs.max_new;
  p.shares = may_split && full <= (alike ? 2 * cu : cu / 2) ? (int)cu : 0;
  deal_whole(c, p, TileCfg<32>::NT, (int)cu);
  return p;
}

bool sdpa_paged_tile_applies(const PagedCall& c) {
  const long long rows = (long long)c.seqs.max_new * (c.H / c.Hkv);
  return c.D >= 8 && c.D <= 256 && rows > kFewRows && rows <= 0x7fffffff - 256 &&
         (long long)c.Hkv * ((rows - 1) / tile_rows(c.D) + 1) <= 0x7fffffff;
}

hipError_t launch_sdpa_paged_tile(hipStream_t s, const PagedCall& c, const SharePlan& p, float* ws) {
  if (c.D <= 32) launch_dp<32>(s, c, p, ws);
  else if (c.D <= 64) launch_dp<64>(s, c, p, ws);
  else if (c.D <= 96) launch_dp<96>(s, c, p, ws);
  else if (c.D <= kTileDim) launch_dp<128>(s, c, p, ws);
  else return launch_sdpa_paged_wide(s, c, p, ws);
  return hipGetLastError();
}

}  // namespace bch
