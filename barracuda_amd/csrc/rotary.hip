// rotary.hip -- rotary positions: pairs of a head's columns turned by an angle that grows with the
// row's position, for dense operands and for the new tokens of a paged cache (paged.h), whose turned
// keys go straight into their pages.  The reference has no positions; these stand beside its
// attention ops and the cache's append.
//
// The pair (a, b) of columns i, i + dim/2 (interleaved: 2i, 2i + 1) of a row at position p becomes
//   scale (a cos t - b sin t), scale (a sin t + b cos t),  t = p freq[i]
// and columns from dim on are copied.  The inverse takes -t: it is also the gradient of the turn.
//
// HBM bounds the large calls (8 bytes an element, 6 FLOP a pair), the launch the small ones.  A thread keeps
// one token and four pairs, so it computes their sines once and turns every head with them: no table, and
// the trigonometry is a small part of a call with a few heads or more.  Angles are products in 64 bits (a
// position of 2^20 in 32 would be off by 2^-4 of a radian); only what is left after taking out quarter
// turns is rounded to 32 bits.
#include "paged.h"

#include <algorithm>

namespace {

using bch::KvPages;
using bch::KvSeqs;
using bch::RotaryPlan;
using bch::SdpaLayout;

constexpr int kThreads = 256;
constexpr int kHeads = 2;  // heads of a thread in flight (4: 8.8 instead of 6.9 us for 16 trees, 1 and 2 alike, 8 10.4)

// cos and sin of t, times scale.  n quarter turns are taken out of t in 64 bits (pi/2 in two parts: t up to 2^31 keeps
// 2^-50), what remains lies within pi/4 and goes through Taylor's series to x^9 and x^10: off by 2^-28 there, below the
// rounding of the last operation (2^-24 of a value near 1).
__device__ __forceinline__ void turn(double t, float scale, float& c, float& s) {
  const double n = rint(t * 0.63661977236758134308);
  double r = fma(n, -1.57079632679489661923, t);
  r = fma(n, -6.12323399573676603587e-17, r);
  const int q = (int)(n - 4.0 * floor(n * 0.25));
  const float x = (float)r, x2 = x * x;
  float sn = fmaf(x2, 2.75573192e-6f, -1.98412698e-4f);
  sn = fmaf(x2, sn, 8.33333333e-3f);
  sn = fmaf(x2, sn, -1.66666667e-1f);
  sn = fmaf(x * x2, sn, x);
  float cs = fmaf(x2, -2.75573192e-7f, 2.48015873e-5f);
  cs = fmaf(x2, cs, -1.38888889e-3f);
  cs = fmaf(x2, cs, 4.16666667e-2f);
  cs = fmaf(x2, cs, -0.5f);
  cs = fmaf(x2, cs, 1.0f);
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  c = scale * ((q + 1) & 2 ? -a : a);
  s = scale * (q & 2 ? -b : b);
}

// What a launch turns: rows of q (dense: of x), H heads into o; for a paged cache also Hkv heads of nk into the pages and
// Hkv heads of nv, as they are.
struct Call {
  RotaryPlan r;
  int D, H, Hkv;
  int pairs, items;       // a row's items: the first `pairs` of them VEC pairs each, the others VEC (interleaved or not) columns
  int width_log, tn_log;  // a row's items on 2^width_log threads, 2^tn_log tokens a workgroup, the other threads on other heads
  int chunks;             // workgroups that share a token's heads
  const float *q, *nk, *nv;
  float *o, *k, *v;
  SdpaLayout ql, ol, nkl, nvl;
  // dense
  long long tokens, first;
  int S;
  const int* positions;
  // paged
  KvPages kv;
  KvSeqs seqs;
  int B, tiles;
  const int* parent;
};

template <int VEC>
struct Elem;
template <>
struct Elem<1> {
  typedef float type;
};
template <>
struct Elem<4> {
  typedef bch::f32x4 type;
};
template <bool NT, typename T>
__device__ __forceinline__ T load(const float* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  return *reinterpret_cast<const T*>(p);
}
template <bool NT, typename T>
__device__ __forceinline__ void store(T x, float* p) {
  if constexpr (NT)
    __builtin_nontemporal_store(x, reinterpret_cast<T*>(p));
  else
    *reinterpret_cast<T*>(p) = x;
}
template <int VEC, typename T>
__device__ __forceinline__ float& at(T& x, int i) {
  if constexpr (VEC == 1)
    return x;
  else
    return reinterpret_cast<float*>(&x)[i];
}

// One thread's token: turn (or copy) its items of the heads hs, hs + step, ...
// find(h, src, dst): where head h of the token is and goes, and whether it is turned; dst null: nowhere.
template <int VEC, bool IL, bool NT, typename Find>
__device__ __forceinline__ void turn_heads(const Call& c, double pos, int e0, int hs, int step, int heads, Find find) {
  typedef typename Elem<VEC>::type T;
  for (int e = e0; e < c.items; e += 1 << c.width_log) {
    const bool pair = e < c.pairs;
    float cs[VEC], sn[VEC];
    int d0, d1;  // the item's first columns: of the pairs' both halves, or the one copied
    if (pair) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) turn(pos * c.r.freq[e * VEC + i], c.r.scale, cs[i], sn[i]);
      d0 = IL ? 2 * VEC * e : VEC * e;
      d1 = IL ? d0 + VEC : d0 + c.r.dim / 2;
    } else {
      d0 = d1 = c.r.dim + (e - c.pairs) * VEC;
    }
    for (int h0 = hs; h0 < heads; h0 += kHeads * step) {
      T x[kHeads], y[kHeads];
      const float* src[kHeads];
      float* dst[kHeads];
      bool turned[kHeads];
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + u * step;
        dst[u] = nullptr;
        if (h < heads) find(h, src[u], dst[u], turned[u]);
        if (dst[u]) {
          x[u] = load<NT, T>(src[u] + d0);
          y[u] = load<NT, T>(src[u] + d1);
        }
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        if (!dst[u]) continue;
        if (pair && turned[u]) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            // interleaved: the item's 2 VEC columns in order, x the first VEC
            float& a = IL ? (2 * i < VEC ? at<VEC>(x[u], 2 * i) : at<VEC>(y[u], 2 * i - VEC)) : at<VEC>(x[u], i);
            float& b = IL ? (2 * i + 1 < VEC ? at<VEC>(x[u], 2 * i + 1) : at<VEC>(y[u], 2 * i + 1 - VEC)) : at<VEC>(y[u], i);
            const float a0 = a, b0 = b;
            a = fmaf(a0, cs[i], -(b0 * sn[i]));
            b = fmaf(a0, sn[i], b0 * cs[i]);
          }
        }
        store<NT, T>(x[u], dst[u] + d0);
        if (pair) store<NT, T>(y[u], dst[u] + d1);
      }
    }
  }
}

template <int VEC, bool IL, bool NT>
__global__ __launch_bounds__(kThreads) void rotary_dense_kernel(Call c) {
  const int e = threadIdx.x & ((1 << c.width_log) - 1), slot = threadIdx.x >> c.width_log;
  const int t = slot & ((1 << c.tn_log) - 1), hn = kThreads >> (c.width_log + c.tn_log);
  const int hs = (slot >> c.tn_log) + hn * blockIdx.y;
  for (long long tok = ((long long)blockIdx.x << c.tn_log) + t; tok < c.tokens; tok += (long long)gridDim.x << c.tn_log) {
    const long long b = bch::quotient(tok, c.S), i = tok - b * c.S;
    const double p = c.positions ? (double)c.positions[tok] : (double)(c.first + i);
    const float* x = c.q + b * c.ql.batch + i * c.ql.row;
    float* o = c.o + b * c.ol.batch + i * c.ol.row;
    turn_heads<VEC, IL, NT>(c, c.r.inverse ? -p : p, e, hs, hn * c.chunks, c.H,
                            [&](int h, const float*& src, float*& dst, bool& turned) {
                              src = x + h * c.ql.head;
                              dst = o + h * c.ol.head;
                              turned = true;
                            });
  }
}

// FIND: tokens of all rows that there are, whose sequences each thread looks for: where batch times the longest sequence's
// tiles is beyond a grid.
template <int VEC, bool IL, bool NT, bool FIND>
__global__ __launch_bounds__(kThreads) void rotary_append_kernel(Call c, long long block0) {
  __shared__ int next[bch::kMaxDrafts], depth[bch::kMaxDrafts];
  const int e = threadIdx.x & ((1 << c.width_log) - 1), slot = threadIdx.x >> c.width_log;
  const int t = slot & ((1 << c.tn_log) - 1), hn = kThreads >> (c.width_log + c.tn_log);
  const int hs = (slot >> c.tn_log) + hn * blockIdx.y;
  int b, i;  // the thread's sequence, and its token of that
  bch::Seq s;
  if constexpr (FIND) {
    const long long row = ((block0 + blockIdx.x) << c.tn_log) + t;
    if (row >= c.seqs.total) return;
    int lo = 0, n = c.B;  // the first sequence that ends behind the row, or the last
    while (n > 1) {
      const int half = n / 2;
      const bool below = c.seqs.start[lo + half] <= row;
      lo = below ? lo + half : lo;
      n = below ? n - half : half;
    }
    b = lo;
    s = bch::load_seq(c.kv, c.seqs, b);
    if (row < s.row0) return;
    i = (int)row - s.row0;
  } else {
    b = (int)(blockIdx.x / c.tiles);
    i = ((int)(blockIdx.x % c.tiles) << c.tn_log) + t;
    s = bch::load_seq(c.kv, c.seqs, b);
  }
  long long pos = (long long)s.first + i;
  if (c.parent) {
    if constexpr (FIND) {
      int up = i < s.n ? c.parent[s.row0 + i] : -1, below = i;
      pos = s.first;
      while (up >= 0 && up < below) {
        ++pos;
        below = up;
        up = c.parent[s.row0 + up];
      }
    } else {
      // depths by pointer jumping: each step adds the depth of a draft's furthest ancestor so far
      const int x = threadIdx.x, n = min(s.n, bch::kMaxDrafts);
      if (x < n) {
        const int p = c.parent[s.row0 + x];
        next[x] = p >= 0 && p < x ? p : -1;
        depth[x] = next[x] >= 0;
      }
      __syncthreads();
      for (int step = 1; step < n; step *= 2) {
        const int p = x < n ? next[x] : -1;
        const int more = p >= 0 ? depth[p] : 0, far = p >= 0 ? next[p] : -1;
        __syncthreads();
        if (x < n) {
          depth[x] += more;
          next[x] = far;
        }
        __syncthreads();
      }
      if (i < s.n) pos = (long long)s.first + depth[i];
    }
  }
  if (i >= s.n) return;
  const long long row = s.row0 + i;
  const int j = s.first + i;
  const bch::Slot at = j >= 0 ? bch::key_slot(c.kv, b, j) : bch::Slot{-1, 0};
  turn_heads<VEC, IL, NT>(c, (double)pos, e, hs, hn * c.chunks, c.H + 2 * c.Hkv,
                          [&](int h, const float*& src, float*& dst, bool& turned) {
                            turned = h < c.H + c.Hkv;
                            if (h < c.H) {
                              src = c.q + row * c.ql.row + h * c.ql.head;
                              dst = c.o + row * c.ol.row + h * c.ol.head;
                            } else if (at.page >= 0) {
                              const int g = turned ? h - c.H : h - c.H - c.Hkv;
                              const SdpaLayout &nl = turned ? c.nkl : c.nvl, &l = turned ? c.kv.kl : c.kv.vl;
                              src = (turned ? c.nk : c.nv) + row * nl.row + g * nl.head;
                              dst = (turned ? c.k : c.v) + bch::slot_offset(l, at) + g * l.head;
                            }
                          });
}

bool mult4(const SdpaLayout& l) { return l.batch % 4 == 0 && l.head % 4 == 0 && l.row % 4 == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_up(long long x) {
  int l = 0;
  while ((1LL << l) < x) ++l;
  return l;
}

// Items, and how 256 threads share a row's items, tokens and heads.  Tokens first (neighbouring rows of a head lie
// together), then heads.
void plan(Call& c, int vec, long long tokens_each, int heads) {
  c.pairs = c.r.dim / 2 / vec;
  c.items = c.pairs + (c.D - c.r.dim + vec - 1) / vec;
  c.width_log = std::min(8, log2_up(c.items));
  c.tn_log = std::min(8 - c.width_log, log2_up(tokens_each));
  const int hn = kThreads >> (c.width_log + c.tn_log);
  c.chunks = (heads + hn - 1) / hn;  // at most; fewer where there are workgroups enough
}
// Workgroups enough.  Fewer leave loads unhidden, more compute the sines of a token again: 48 a CU for streams (4 x 32 heads x 2048 rows
// of 128: 47 us, 54 with 8; a prompt's 10031 tokens of 32 + 2 x 8 heads 91, 95 with 8, 97 with 64), three for small
// calls (3069 rows of 12 heads of 80 7.7 us, 8.8 with 1, 8.4 with 16).
void share_heads(Call& c, long long blocks, bool stream) {
  const long long want = (stream ? 48LL : 3LL) * bch::device_cu_count();
  c.chunks = (int)std::max(1LL, std::min({(long long)c.chunks, (want + blocks - 1) / std::max(1LL, blocks), 65535LL}));
}

constexpr double kNtBytes = 64.0 * 1048576;  // streams at least this large bypass the caches

}  // namespace

namespace bch {

hipError_t launch_rotary(hipStream_t s, int B, int H, int S, int D, const RotaryPlan& r, long long first,
                         const int* positions, const float* x, const SdpaLayout& xl, float* o, const SdpaLayout& ol) {
  Call c{};
  c.r = r;
  c.D = D;
  c.H = H;
  c.q = x;
  c.o = o;
  c.ql = xl;
  c.ol = ol;
  c.tokens = (long long)B * S;
  c.first = first;
  c.S = S;
  c.positions = positions;
  const bool vec = D % 4 == 0 && r.dim % 8 == 0 && aligned16(x) && aligned16(o) && mult4(xl) && mult4(ol);
  const bool nt = 8.0 * B * S * H * D >= kNtBytes;
  plan(c, vec ? 4 : 1, c.tokens, H);
  const long long blocks = ((c.tokens - 1) >> c.tn_log) + 1;
  share_heads(c, blocks, nt);
  const dim3 grid((unsigned)std::min(blocks, 1LL << 20), c.chunks), block(kThreads);
#define BCH_ROTARY(V, IL) (nt ? rotary_dense_kernel<V, IL, true> : rotary_dense_kernel<V, IL, false>)
  auto kern = r.interleaved ? (vec ? BCH_ROTARY(4, true) : BCH_ROTARY(1, true))
                            : (vec ? BCH_ROTARY(4, false) : BCH_ROTARY(1, false));
#undef BCH_ROTARY
  hipLaunchKernelGGL(kern, grid, block, 0, s, c);
  return hipGetLastError();
}

hipError_t launch_kv_append_rotary(hipStream_t s, const KvPages& kv, float* k, float* v, const KvSeqs& seqs, int B,
                                   const int* parent, const RotaryPlan& r, int H, int Hkv, int D, const float* q,
                                   const SdpaLayout& ql, float* o, const SdpaLayout& ol, const float* nk,
                                   const SdpaLayout& nkl, const float* nv, const SdpaLayout& nvl) {
  Call c{};
  c.r = r;
  c.D = D;
  c.H = H;
  c.Hkv = Hkv;
  c.q = q;
  c.nk = nk;
  c.nv = nv;
  c.o = o;
  c.k = k;
  c.v = v;
  c.ql = ql;
  c.ol = ol;
  c.nkl = nkl;
  c.nvl = nvl;
  c.kv = kv;
  c.seqs = seqs;
  c.B = B;
  c.parent = parent;
  const bool vec = D % 4 == 0 && r.dim % 8 == 0 && aligned16(k) && aligned16(v) && mult4(kv.kl) && mult4(kv.vl) &&
                   aligned16(nk) && aligned16(nv) && mult4(nkl) && mult4(nvl) &&
                   (H == 0 || (aligned16(q) && aligned16(o) && mult4(ql) && mult4(ol)));
  const bool nt = 8.0 * seqs.total * D * (H + 2.0 * Hkv) >= kNtBytes;
  plan(c, vec ? 4 : 1, seqs.max_new, H + 2 * Hkv);
  c.tiles = ((seqs.max_new - 1) >> c.tn_log) + 1;
  const bool find = !fits_grid((long long)c.tiles * B, kThreads);
  const long long blocks = find ? ((seqs.total - 1LL) >> c.tn_log) + 1 : (long long)c.tiles * B;
  // of many sequences with room for long chunks most workgroups are empty: the rows that there are count
  share_heads(c, std::min(blocks, ((seqs.total - 1LL) >> c.tn_log) + 1 + B), nt);
#define BCH_ROTARY(V, IL)                                                                         \
  (find ? (nt ? rotary_append_kernel<V, IL, true, true> : rotary_append_kernel<V, IL, false, true>) \
        : (nt ? rotary_append_kernel<V, IL, true, false> : rotary_append_kernel<V, IL, false, false>))
  auto kern = r.interleaved ? (vec ? BCH_ROTARY(4, true) : BCH_ROTARY(1, true))
                            : (vec ? BCH_ROTARY(4, false) : BCH_ROTARY(1, false));
#undef BCH_ROTARY
  const long long most = find ? 1 << 23 : blocks;
  for (long long at = 0; at < blocks; at += most) {
    const dim3 grid((unsigned)std::min(most, blocks - at), c.chunks), block(kThreads);
    hipLaunchKernelGGL(kern, grid, block, 0, s, c, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace bch
