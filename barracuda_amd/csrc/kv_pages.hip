// kv_pages.hip -- what writes a paged key/value cache (paged.h): new tokens appended, whole pages
// copied, keys moved down within their sequences.  The reference has no cache; these stand beside its
// attention ops as bch_copy and the head permutations do.
//
// All three only move data: 16 bytes of K and V a column read and written, so HBM bounds the large
// calls and the launch the small ones.  Rows go as 16-byte accesses where D, the strides and the
// pointers allow (VEC 4), else as single floats.
#include "paged.h"

#include <algorithm>

namespace {

using bch::KvPages;
using bch::KvSeqs;
using bch::SdpaLayout;

constexpr int kThreads = 256;

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

// ---- append: row i of sequence b is key len[b] - n + i ----
// A workgroup takes kAppend tokens of one sequence; a thread the same columns of each, K and V, with
// all of its loads ahead of its stores, past the caches (8 ragged prompts, 8128 tokens of 8 KB, 133 MB: 23.8 us,
// 5.6 TB/s; through them, four tokens 29; past them, one token 28.8, four 24.9).
constexpr int kAppend = 2;

// FIND: kAppend rows of all that there are (from the at0'th kAppend on), whose sequences it looks for: where batch
// times the longest sequence's new tokens is beyond a grid.  In ordinary batches the search costs some: a workgroup a
// sequence and kAppend of its tokens / all rows, 8 ragged prompts 23.9 / 24.6 us, 16 sequences of up to 64 drafts in four
// layers, with their keep, 28.5 / 29.7.  (Beside a long chunk it would save: 127 tokens and a chunk of 8192 take 207 us
// by sequence, 7 and 23 apart.)
template <int VEC, bool FIND>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvPages kv, float* k, float* v, KvSeqs seqs, int B,
                                                             int tiles, long long at0, int Hkv, int D,
                                                             const float* __restrict__ nk, SdpaLayout nkl,
                                                             const float* __restrict__ nv, SdpaLayout nvl) {
  typedef typename Elem<VEC>::type T;
  bch::Slot slot[kAppend];
  long long rows[kAppend];
  if constexpr (FIND) {
#pragma unroll
    for (int u = 0; u < kAppend; ++u) {
      const long long at = (at0 + blockIdx.x) * kAppend + u;
      rows[u] = min(at, (long long)seqs.total - 1);
      const int b = __builtin_amdgcn_readfirstlane(bch::seq_of_row(seqs, B, rows[u], threadIdx.x & 63));
      const bch::Seq s = bch::load_seq(kv, seqs, b);
      const long long i = rows[u] - s.row0, j = s.first + i;
      slot[u] = at < seqs.total && i >= 0 && i < s.n && j >= 0 ? bch::key_slot(kv, b, (int)j) : bch::Slot{-1, 0};
    }
  } else {
    const int b = blockIdx.x / tiles, i0 = (blockIdx.x % tiles) * kAppend;
    const bch::Seq s = bch::load_seq(kv, seqs, b);
    if (i0 >= s.n) return;
#pragma unroll
    for (int u = 0; u < kAppend; ++u) {
      const int j = s.first + i0 + u;
      slot[u] = i0 + u < s.n && j >= 0 ? bch::key_slot(kv, b, j) : bch::Slot{-1, 0};
      rows[u] = s.row0 + min(i0 + u, s.n - 1);
    }
  }
  const int dv = D / VEC;
  for (int e = threadIdx.x; e < Hkv * dv; e += kThreads) {
    const int h = e / dv, d = (e - h * dv) * VEC;
    T x[kAppend], y[kAppend];
#pragma unroll
    for (int u = 0; u < kAppend; ++u) {
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const T*>(nk + rows[u] * nkl.row + h * nkl.head + d));
      y[u] = __builtin_nontemporal_load(reinterpret_cast<const T*>(nv + rows[u] * nvl.row + h * nvl.head + d));
    }
#pragma unroll
    for (int u = 0; u < kAppend; ++u)
      if (slot[u].page >= 0) {
        __builtin_nontemporal_store(x[u], reinterpret_cast<T*>(k + bch::slot_offset(kv.kl, slot[u]) + h * kv.kl.head + d));
        __builtin_nontemporal_store(y[u], reinterpret_cast<T*>(v + bch::slot_offset(kv.vl, slot[u]) + h * kv.vl.head + d));
      }
  }
}

// ---- copy of whole pages ----
// The pairs travel as kernel arguments: a captured graph holds them, and no copy of them to the device
// is waited for.  A page is [n1][n2][run] floats with strides s1, s2 (merged where they are dense).
constexpr int kPairs = 480;
struct Pairs {
  int src[kPairs], dst[kPairs];
};
struct PageShape {
  float* base;
  long long page, layer, s1, s2;
  int n2;
  long long run, total;  // floats
};

// One access a thread, past the caches (1500 pages of 64 KB, K and V, 393 MB: 75 us, 5.2 TB/s; through them
// 95; two or four accesses a thread past them 83, eight 131).
template <int VEC>
__global__ __launch_bounds__(kThreads) void kv_copy_kernel(PageShape ks, PageShape vs, Pairs pairs) {
  typedef typename Elem<VEC>::type T;
  const PageShape& p = blockIdx.z & 1 ? vs : ks;
  const long long e = ((long long)blockIdx.x * kThreads + threadIdx.x) * VEC;
  if (e >= p.total) return;
  long long off = e;
  if (p.run != p.total) {
    const long long r = e / p.run;
    off = (r / p.n2) * p.s1 + (r % p.n2) * p.s2 + (e - r * p.run);
  }
  float* base = p.base + (blockIdx.z >> 1) * p.layer + off;
  const T x = __builtin_nontemporal_load(reinterpret_cast<const T*>(base + pairs.src[blockIdx.y] * p.page));
  __builtin_nontemporal_store(x, reinterpret_cast<T*>(base + pairs.dst[blockIdx.y] * p.page));
}

PageShape page_shape(float* base, const SdpaLayout& l, long long layer, int Hkv, int page_size, int D) {
  PageShape p{base, l.batch, layer, l.head, l.row, page_size, D, (long long)Hkv * page_size * D};
  int n1 = Hkv;
  if (p.s1 < p.s2) {  // heads inside keys
    std::swap(p.s1, p.s2);
    std::swap(n1, p.n2);
  }
  if (p.s2 == p.run || p.n2 == 1) {
    p.run *= p.n2;
    p.n2 = n1;
    p.s2 = p.s1;
    p.s1 = 0;
    if (p.s2 == p.run || p.n2 == 1) {
      p.run *= p.n2;
      p.n2 = 1;
      p.s2 = 0;
    }
  }
  return p;
}

// ---- keep: key to[b] + i = key keep[start[b] + i] ----
// A thread owns its columns of a sequence's keys and moves them in ascending i, kKeep at a time, so
// that a key is read before a later one of the same call takes its place (keep ascends and no key moves
// up: to[b] + i <= keep[i] < keep[i + 1]).  Where the keys read lie behind all that are written, their order
// does not matter, and `chunks` workgroups share them.
constexpr int kKeep = 8;

template <int VEC>
__global__ __launch_bounds__(kThreads) void kv_keep_kernel(KvPages kv, float* k, float* v, long long k_layer,
                                                           long long v_layer, int Hkv, int D, int chunks, int total,
                                                           const int* start, const int* keep, const int* to) {
  typedef typename Elem<VEC>::type T;
  const int b = blockIdx.y, chunk = blockIdx.x % chunks;
  const bool is_v = blockIdx.z & 1;
  const SdpaLayout& l = is_v ? kv.vl : kv.kl;
  float* base = (is_v ? v : k) + (blockIdx.z >> 1) * (is_v ? v_layer : k_layer);
  const int a = min(max(start[b], 0), total), n = min(max(start[b + 1], a), total) - a;
  const int t0 = to[b], dv = D / VEC;
  const int e = blockIdx.x / chunks * kThreads + threadIdx.x;
  if (n == 0 || e >= Hkv * dv) return;
  const bool apart = keep[a] >= (long long)t0 + n;
  if (!apart && chunk > 0) return;
  const int per = apart ? ((n - 1) / chunks / kKeep + 1) * kKeep : n;
  const int i1 = (int)min((long long)n, ((long long)chunk + 1) * per);
  float* col = base + (e / dv) * l.head + (e % dv) * VEC;
  for (int i0 = chunk * per; i0 < i1; i0 += kKeep) {
    T x[kKeep];
    bch::Slot dst[kKeep];
#pragma unroll
    for (int u = 0; u < kKeep; ++u) {
      const int i = min(i0 + u, i1 - 1), j = keep[a + i];
      const long long to_j = (long long)t0 + i;
      const bool on = i0 + u < i1 && j > to_j && to_j >= 0;
      const bch::Slot src = on ? bch::key_slot(kv, b, j) : bch::Slot{-1, 0};
      dst[u] = src.page >= 0 ? bch::key_slot(kv, b, (int)to_j) : src;
      if (dst[u].page >= 0) x[u] = *reinterpret_cast<const T*>(col + bch::slot_offset(l, src));
    }
#pragma unroll
    for (int u = 0; u < kKeep; ++u)
      if (dst[u].page >= 0) *reinterpret_cast<T*>(col + bch::slot_offset(l, dst[u])) = x[u];
  }
}

bool mult4(const SdpaLayout& l) { return l.batch % 4 == 0 && l.head % 4 == 0 && l.row % 4 == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool vec4(const KvPages& kv, const float* k, const float* v, int D) {
  return D % 4 == 0 && aligned16(k) && aligned16(v) && mult4(kv.kl) && mult4(kv.vl);
}

}  // namespace

namespace bch {

hipError_t launch_kv_append(hipStream_t s, const KvPages& kv, float* k, float* v, const KvSeqs& seqs, int B, int Hkv,
                            int D, const float* nk, const SdpaLayout& nkl, const float* nv, const SdpaLayout& nvl) {
  if ((long long)Hkv * D > 0x7fffffffLL - kThreads) return hipErrorInvalidConfiguration;
  const int tiles = (seqs.max_new - 1) / kAppend + 1;
  const bool vec = vec4(kv, k, v, D) && aligned16(nk) && aligned16(nv) && nkl.row % 4 == 0 && nkl.head % 4 == 0 &&
                   nvl.row % 4 == 0 && nvl.head % 4 == 0;
  const bool find = !fits_grid((long long)tiles * B, kThreads);
  const long long all = find ? (seqs.total - 1LL) / kAppend + 1 : (long long)tiles * B, most = find ? 1 << 23 : all;
  auto kern = find ? (vec ? kv_append_kernel<4, true> : kv_append_kernel<1, true>)
                   : (vec ? kv_append_kernel<4, false> : kv_append_kernel<1, false>);
  for (long long at = 0; at < all; at += most) {
    const dim3 grid((unsigned)std::min(most, all - at)), block(kThreads);
    hipLaunchKernelGGL(kern, grid, block, 0, s, kv, k, v, seqs, B, tiles, at, Hkv, D, nk, nkl, nv, nvl);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_kv_copy_pages(hipStream_t s, const KvPages& kv, float* k, float* v, int layers, long long k_layer,
                                long long v_layer, int Hkv, int D, int n, const int* src, const int* dst) {
  const bool vec = vec4(kv, k, v, D) && k_layer % 4 == 0 && v_layer % 4 == 0;
  const PageShape ks = page_shape(k, kv.kl, k_layer, Hkv, kv.page_size, D);
  const PageShape vs = page_shape(v, kv.vl, v_layer, Hkv, kv.page_size, D);
  const long long per = (long long)kThreads * (vec ? 4 : 1);
  const long long chunks = (ks.total + per - 1) / per;
  if (chunks > 0x7fffffffLL / kThreads) return hipErrorInvalidConfiguration;
  for (int l0 = 0; l0 < layers; l0 += 16384) {
    const int nl = std::min(layers - l0, 16384);
    PageShape kl = ks, vl = vs;
    kl.base += l0 * k_layer;
    vl.base += l0 * v_layer;
    for (int p0 = 0; p0 < n; p0 += kPairs) {
      const int np = std::min(n - p0, kPairs);
      Pairs pairs;
      std::copy(src + p0, src + p0 + np, pairs.src);
      std::copy(dst + p0, dst + p0 + np, pairs.dst);
      const dim3 grid((unsigned)chunks, np, 2 * nl), block(kThreads);
      if (vec)
        hipLaunchKernelGGL(kv_copy_kernel<4>, grid, block, 0, s, kl, vl, pairs);
      else
        hipLaunchKernelGGL(kv_copy_kernel<1>, grid, block, 0, s, kl, vl, pairs);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

hipError_t launch_kv_keep(hipStream_t s, const KvPages& kv, float* k, float* v, int layers, long long k_layer,
                          long long v_layer, int Hkv, int D, int B, int total, const int* start, const int* keep,
                          const int* to) {
  const bool vec = vec4(kv, k, v, D) && k_layer % 4 == 0 && v_layer % 4 == 0;
  const long long cols = (long long)Hkv * D / (vec ? 4 : 1);
  if (cols > 0x7fffffffLL - kThreads || B > 65535 || layers > 32767) return hipErrorInvalidConfiguration;
  // 32 keys or more a workgroup on the average
  const int chunks = (int)std::max(1LL, std::min(64LL, (long long)total / B / 32));
  const long long blocks = (cols + kThreads - 1) / kThreads * chunks;
  if (!fits_grid(blocks * B, kThreads) || !fits_grid(blocks * B * 2 * layers, 1)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks, B, 2 * layers), block(kThreads);
  if (vec)
    hipLaunchKernelGGL(kv_keep_kernel<4>, grid, block, 0, s, kv, k, v, k_layer, v_layer, Hkv, D, chunks, total, start, keep, to);
  else
    hipLaunchKernelGGL(kv_keep_kernel<1>, grid, block, 0, s, kv, k, v, k_layer, v_layer, Hkv, D, chunks, total, start, keep, to);
  return hipGetLastError();
}

}  // namespace bch
