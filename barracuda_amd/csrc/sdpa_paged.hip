// sdpa_paged.hip -- attention over a paged key/value cache, with a sliding window, sinks and trees of
// drafts (paged.h says which keys a row sees):
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j,
// over the keys j that row i sees; zeros where it sees none.  The reference has no such op; the ones it
// has (ops/causal_attn/mod.rs:64-158, ops/grouped_query_attention/mod.rs:52-147) are the case of one
// page a sequence and no window.
#include "paged.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

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

// o[row] = sum over a list's parts of 2^(m_s - m) O_s / sum of 2^(m_s - m) l_s, in their order: a
// wavefront four rows, lane s the maximum and sum of part s, lane d (and on by 64) the columns.  A part
// without a key that the row sees has l = 0 and counts nothing; a row without any gives zeros.  Rows of a
// list that was not cut are there already.  Trips to memory bound it, so a wavefront's four rows make
// them together.
template <int ROWS>
__global__ __launch_bounds__(256) void paged_combine(PagedCall c, bch::SharePlan plan, const float* __restrict__ ws) {
  constexpr int R = 4, Q = ROWS / 16;
  const int list = blockIdx.x / Q;
  const int rb = list % plan.tiles, bk = list / plan.tiles, b = bk / c.Hkv, hk = bk - b * c.Hkv;
  const Seq s = bch::load_seq(c.kv, c.seqs, b);
  const int group = c.H / c.Hkv;
  const long long rows = (long long)s.n * group;
  const int lane = threadIdx.x & 63, r0 = (blockIdx.x % Q) * 16 + (threadIdx.x >> 6) * R;  // within the row block
  if ((long long)rb * ROWS + r0 >= rows || rows < plan.row_min || rows > plan.row_max) return;
  const int count = reinterpret_cast<const int*>(ws)[list];
  if (count <= 1) return;
  const long long per = bch::part_floats(plan, c.D);
  const float* p = ws + bch::counts_floats((long long)c.B * c.Hkv * plan.tiles) + (long long)list * plan.slots * per;
  const int last = (int)min(rows - (long long)rb * ROWS, (long long)plan.part_rows) - 1;
  const float *ml[R], *po[R];
  float m[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = min(r0 + j, last);
    ml[j] = p + (long long)plan.part_rows * c.D + 2 * r;
    po[j] = p + (long long)r * c.D;
    m[j] = -INFINITY;
  }
  for (int u0 = 0; u0 < count; u0 += 64) {
    float v[R];
#pragma unroll
    for (int j = 0; j < R; ++j) v[j] = u0 + lane < count ? ml[j][(u0 + lane) * per] : -INFINITY;
#pragma unroll
    for (int j = 0; j < R; ++j) m[j] = fmaxf(m[j], bch::wave_allreduce(v[j], bch::OpMax()));
  }
  for (int d0 = 0; d0 < c.D; d0 += 128) {
    const int da = min(d0 + lane, c.D - 1), db = min(d0 + lane + 64, c.D - 1);
    float x[R], y[R], l[R];
#pragma unroll
    for (int j = 0; j < R; ++j) x[j] = y[j] = l[j] = 0.0f;
    for (int u0 = 0; u0 < count; u0 += 64) {
      const bool on = u0 + lane < count;
      const int n = min(64, count - u0);
      float a[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const float ms = on ? ml[j][(u0 + lane) * per] : -INFINITY, ls = on ? ml[j][(u0 + lane) * per + 1] : 0.0f;
        a[j] = __builtin_amdgcn_exp2f(ms - (m[j] == -INFINITY ? 0.0f : m[j]));
        l[j] += bch::wave_allreduce(a[j] * ls, bch::OpSum());
      }
      auto add = [&](auto width, int u) {  // the next U parts, their rows loaded before they are added
        constexpr int U = decltype(width)::value;
        float vx[U][R], vy[U][R];
#pragma unroll
        for (int w = 0; w < U; ++w)
#pragma unroll
          for (int j = 0; j < R; ++j) {
            vx[w][j] = po[j][(u0 + u + w) * per + da];
            vy[w][j] = po[j][(u0 + u + w) * per + db];
          }
#pragma unroll
        for (int w = 0; w < U; ++w)
#pragma unroll
          for (int j = 0; j < R; ++j) {
            const float f = bch::readlane(a[j], u + w);
            x[j] = fmaf(f, vx[w][j], x[j]);
            y[j] = fmaf(f, vy[w][j], y[j]);
          }
      };
      int u = 0;
      for (; u + 4 <= n; u += 4) add(std::integral_constant<int, 4>{}, u);
      for (; u < n; ++u) add(std::integral_constant<int, 1>{}, u);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int row = rb * ROWS + r0 + j, tok = row / group;
      if (r0 + j > last) break;
      float* dst = c.o + b * c.ol.batch + (long long)(s.row0 + tok) * c.ol.row +
                   (long long)(hk * group + row - tok * group) * c.ol.head;
      if (d0 + lane < c.D) dst[d0 + lane] = l[j] == 0.0f ? 0.0f : x[j] / l[j];
      if (d0 + lane + 64 < c.D) dst[d0 + lane + 64] = l[j] == 0.0f ? 0.0f : y[j] / l[j];
    }
  }
}

}  // namespace

namespace bch {

hipError_t launch_paged_combine(hipStream_t s, const PagedCall& c, const SharePlan& p, int rows, const float* ws) {
  // row blocks with rows in them: a part's rows are all that there are if they are fewer
  const long long groups = lists_of(c, p) * (rows / 16);
  if (groups > 0x7fffffffLL) return hipErrorInvalidConfiguration;
  if (rows == 16)
    hipLaunchKernelGGL(paged_combine<16>, dim3((unsigned)groups), dim3(256), 0, s, c, p, ws);
  else
    hipLaunchKernelGGL(paged_combine<256>, dim3((unsigned)groups), dim3(256), 0, s, c, p, ws);
  return hipGetLastError();
}

namespace {

// Which kernels a call takes.  The tile kernel does 64 rows or fewer of a sequence as slowly as 256; a batch
// may mix prompts and single tokens, so each kernel serves its own sequences.
struct Route {
  bool tile, rows;
  int row_limit;
};
Route route(const PagedCall& c) {
  Route r;
  r.tile = sdpa_paged_tile_applies(c);
  r.row_limit = r.tile ? kTileRows : 0x7fffffff;
  // dense operands: every sequence has max_new rows
  r.rows = r.tile ? c.seqs.start != nullptr : sdpa_paged_rows_applies(c, r.row_limit);
  return r;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t sdpa_paged_workspace_bytes(const PagedCall& c, int max_len) {
  const Route r = route(c);
  return (r.tile ? up256(sdpa_paged_tile_workspace_bytes(c, max_len)) : 0) +
         (r.rows ? sdpa_paged_rows_workspace_bytes(c, max_len, r.row_limit) : 0);
}

hipError_t launch_sdpa_paged(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes) {
  const Route r = route(c);
  if (r.tile || r.rows) {
    if (ws_bytes < sdpa_paged_workspace_bytes(c, max_len)) ws_bytes = 0;
    const size_t at = r.tile ? std::min(ws_bytes, up256(sdpa_paged_tile_workspace_bytes(c, max_len))) : 0;
    hipError_t e = r.tile ? launch_sdpa_paged_tile(s, c, max_len, ws, at) : hipSuccess;
    if (e != hipSuccess || !r.rows) return e;
    return launch_sdpa_paged_rows(s, c, max_len, r.row_limit, static_cast<char*>(ws) + at, ws_bytes - at);
  }
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
