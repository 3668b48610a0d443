// sdpa_paged.hip -- attention over a paged key/value cache, with a sliding window, sinks and trees of
// drafts (paged.h says which keys a row sees):
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j,
// over the keys j that row i sees; zeros where it sees none.  The reference has no such op; the ones it
// has (ops/causal_attn/mod.rs:64-158, ops/grouped_query_attention/mod.rs:52-147) are the case of one
// page a sequence and no window.
#include "paged.h"

#include <math.h>

#include <algorithm>

namespace {

using bch::PagedCall;
using bch::Seq;

constexpr int kAnyWaves = 4;

// A wavefront per row and query head, lane l the columns l + 64 t: one key after the other, its score
// by a reduction over the wavefront.  Reads nothing that the row does not see.
template <int T>
__global__ __launch_bounds__(64 * kAnyWaves) void sdpa_paged_any_kernel(PagedCall c, int tiles) {
  __shared__ bch::TreeMasks tree;
  const int b = blockIdx.x / tiles;
  const Seq s = bch::load_seq(c.kv, c.seqs, b);
  if (c.parent) bch::tree_masks(tree, c.parent, s, c.window, c.sinks);

  const int lane = threadIdx.x & 63;
  const long long r = (long long)(blockIdx.x % tiles) * kAnyWaves + (threadIdx.x >> 6);
  if (r >= (long long)s.n * c.H) return;
  const int i = (int)(r / c.H), h = (int)(r % c.H), hk = h / (c.H / c.Hkv);
  const float* kh = c.kv.k + hk * c.kv.kl.head;
  const float* vh = c.kv.v + hk * c.kv.vl.head;
  const long long row = s.row0 + i;
  const float* q = c.q + b * c.ql.batch + row * c.ql.row + h * c.ql.head;
  float* o = c.o + b * c.ol.batch + row * c.ol.row + h * c.ol.head;

  float qv[T], acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int d = lane + 64 * t;
    qv[t] = d < c.D ? q[d] * c.qscale : 0.0f;
    acc[t] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  auto key = [&](int j) {
    const bch::Slot sl = bch::key_slot(c.kv, b, j);
    if (sl.page < 0) return;
    const float* kr = kh + bch::slot_offset(c.kv.kl, sl);
    const float* vr = vh + bch::slot_offset(c.kv.vl, sl);
    float p = 0.0f, x[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int d = lane + 64 * t;
      p = fmaf(qv[t], d < c.D ? kr[d] : 0.0f, p);
      x[t] = d < c.D ? vr[d] : 0.0f;
    }
    p = bch::wave_allreduce(p, bch::OpSum());
    if (p == -INFINITY) return;
    const float mn = p > m ? p : m;  // NaN: the sum below becomes NaN and stays it
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float e = __builtin_amdgcn_exp2f(p - (mn == -INFINITY ? 0.0f : mn));
    m = mn;
    l = l * a + e;
#pragma unroll
    for (int t = 0; t < T; ++t) acc[t] = fmaf(e, x[t], acc[t] * a);
  };

  const int pos = s.first + (c.parent ? tree.depth[i] : i);
  const int hi = c.parent ? s.first : pos + 1;  // committed keys (or the chain's) below hi
  const int lo = bch::window_begin(pos, c.window);
  for (int j = 0; j < min(min(c.sinks, lo), hi); ++j) key(j);
  for (int j = lo; j < hi; ++j) key(j);
  if (c.parent)
    for (int w = 0; w < 4; ++w)
      for (unsigned bits = tree.mask[i][w]; bits; bits &= bits - 1) {
        const int j = s.first + 32 * w + __ffs(bits) - 1;
        if (j >= 0) key(j);
      }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int d = lane + 64 * t;
    if (d < c.D) o[d] = l == 0.0f ? 0.0f : acc[t] * inv;
  }
}

}  // namespace

namespace bch {

size_t sdpa_paged_workspace_bytes(const PagedCall& c, int max_len) {
  if (sdpa_paged_tile_applies(c)) return sdpa_paged_tile_workspace_bytes(c, max_len);
  return sdpa_paged_rows_applies(c) ? sdpa_paged_rows_workspace_bytes(c, max_len) : 0;
}

hipError_t launch_sdpa_paged(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes) {
  if (sdpa_paged_tile_applies(c)) return launch_sdpa_paged_tile(s, c, max_len, ws, ws_bytes);
  if (sdpa_paged_rows_applies(c)) return launch_sdpa_paged_rows(s, c, max_len, ws, ws_bytes);
  const long long tiles = ((long long)c.seqs.max_new * c.H + kAnyWaves - 1) / kAnyWaves;
  if (tiles * c.B > 0x7fffffffLL) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)(tiles * c.B)), block(64 * kAnyWaves);
#define BCH_ANY(T_) hipLaunchKernelGGL(sdpa_paged_any_kernel<T_>, grid, block, 0, s, c, (int)tiles)
  if (c.D <= 64) BCH_ANY(1);
  else if (c.D <= 128) BCH_ANY(2);
  else if (c.D <= 256) BCH_ANY(4);
  else if (c.D <= 512) BCH_ANY(8);
  else if (c.D <= 1024) BCH_ANY(16);
  else return hipErrorInvalidValue;
#undef BCH_ANY
  return hipGetLastError();
}

}  // namespace bch
