// sdpa_paged.hip -- attention over a paged key/value cache, with a sliding window, sinks and trees of
// drafts (paged.h says which keys a row sees):
//   o_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j,
// over the keys j that row i sees; zeros where it sees none.  The reference has no such op; the ones it
// has (ops/causal_attn/mod.rs:64-158, ops/grouped_query_attention/mod.rs:52-147) are the case of one
// page a sequence and no window.
#include "paged.h"

#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <type_traits>

namespace {

using bch::PagedCall;
using bch::Seq;

constexpr int kAnyWaves = 4;

// Head dimensions that the matrix-core kernels do not take (below 4, and 257 to 1024): a workgroup per row of q and
// query head, which looks for the row's sequence; its wavefronts four keys in turn each, lane l the columns l + 64 t;
// a score is a reduction over the wavefront, four of them under way at a time.  Reads nothing that the row does not
// see.  Every row reads its own K and V: 4 sequences of 2048 keys, 8 heads on 2, D 512, a token each: 1914 us with a
// wavefront per row and one key at a time, 276 so; 64 tokens each 2241 and 837 (D 2: 787 and 131, 810 and 511).
template <int T>
__global__ __launch_bounds__(64 * kAnyWaves) void sdpa_paged_any_kernel(PagedCall c, long long at0) {
  constexpr int U = 4;  // keys at a time
  __shared__ bch::TreeMasks tree;
  __shared__ float red_m[kAnyWaves], red_l[kAnyWaves], red_o[kAnyWaves][64 * T];
  const long long at = at0 + blockIdx.x;  // row of q * H + query head
  const long long of = bch::quotient(at, c.H);
  const int h = (int)(at - of * c.H), hk = h / (c.H / c.Hkv);
  const int b = __builtin_amdgcn_readfirstlane(bch::seq_of_row(c.seqs, c.B, of, threadIdx.x & 63));
  const Seq s = bch::load_seq(c.kv, c.seqs, b);
  const long long i_ = of - (c.seqs.start ? s.row0 : (long long)b * c.seqs.max_new);
  if (i_ < 0 || i_ >= s.n) return;
  const int i = (int)i_;
  if (c.parent) bch::tree_masks(tree, c.parent, s, c.window, c.sinks);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  // keys j .. min(j + U, end) - 1
  auto some = [&](int j, int end) {
    bool on[U];
    float p[U], x[U][T];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      bch::Slot sl{-1, 0};
      if (j + u < end) sl = bch::key_slot(c.kv, b, j + u);
      on[u] = sl.page >= 0;
      if (!on[u]) sl = {0, 0};
      const float* kr = kh + bch::slot_offset(c.kv.kl, sl);
      const float* vr = vh + bch::slot_offset(c.kv.vl, sl);
      p[u] = 0.0f;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int d = lane + 64 * t;
        p[u] = fmaf(qv[t], on[u] && d < c.D ? kr[d] : 0.0f, p[u]);
        x[u][t] = on[u] && d < c.D ? vr[d] : 0.0f;
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = bch::wave_allreduce(p[u], bch::OpSum());
      if (!on[u]) p[u] = -INFINITY;
      mn = p[u] > mn ? p[u] : mn;  // (NaN: its weight below is NaN, and so is the sum)
    }
    const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), use = mn == -INFINITY ? 0.0f : mn;
    m = mn;
    l *= a;
#pragma unroll
    for (int t = 0; t < T; ++t) acc[t] *= a;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p[u] == -INFINITY) continue;  // not seen: whatever its value
      const float e = __builtin_amdgcn_exp2f(p[u] - use);
      l += e;
#pragma unroll
      for (int t = 0; t < T; ++t) acc[t] = fmaf(e, x[u][t], acc[t]);
    }
  };

  const int pos = s.first + (c.parent ? tree.depth[i] : i);
  const int hi = c.parent ? s.first : pos + 1;  // committed keys (or the chain's) below hi
  const int lo = bch::window_begin(pos, c.window), s_hi = min(min(c.sinks, lo), hi);
  for (int j = U * wave; j < s_hi; j += U * kAnyWaves) some(j, s_hi);
  for (long long j = lo + U * wave; j < hi; j += U * kAnyWaves) some((int)j, hi);
  if (c.parent) {
    int turn = 0;
    for (int w = 0; w < 4; ++w)
      for (unsigned bits = tree.mask[i][w]; bits; bits &= bits - 1) {
        const int j = s.first + 32 * w + __ffs(bits) - 1;
        if (j >= 0 && turn++ % kAnyWaves == wave) some(j, j + 1);
      }
  }
  if (lane == 0) {
    red_m[wave] = m;
    red_l[wave] = l;
  }
#pragma unroll
  for (int t = 0; t < T; ++t) red_o[wave][lane + 64 * t] = acc[t];
  __syncthreads();
  m = red_m[0];
#pragma unroll
  for (int w = 1; w < kAnyWaves; ++w) m = fmaxf(m, red_m[w]);
  float f[kAnyWaves];
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < kAnyWaves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(red_m[w] - (m == -INFINITY ? 0.0f : m));
    l += f[w] * red_l[w];
  }
  for (int d = threadIdx.x; d < c.D; d += 64 * kAnyWaves) {
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kAnyWaves; ++w) x = fmaf(f[w], red_o[w][d], x);
    o[d] = l == 0.0f ? 0.0f : x / l;
  }
}

// o[row] = sum over a list's parts of 2^(m_s - m) O_s / sum of 2^(m_s - m) l_s, in their order: a
// wavefront per row, lane s the maximum and sum of part s, lane d (and on by 64) the columns.  A part
// without a key that the row sees has l = 0 and counts nothing; a row without any gives zeros.  Rows of a
// list that was not cut are there already.  Trips to memory bound it: the rows of eight parts are loaded
// before they are added (32 decode steps 4.9 us, a tree of 64 rows in 32 parts 10.6).  Both kernels' rows in one launch, a wavefront per row of q that there is (with one
// per row that a sequence might have, those with nothing to do took 12 of 20 us for seven ragged chunks).
struct Combined {
  bch::SharePlan plan;
  const float* ws;
};
// most > 0: the tokens of a sequence that are looked at; else all rows of q.
__global__ __launch_bounds__(256) void paged_combine(PagedCall c, Combined tile, Combined few, int most) {
  const int lane = threadIdx.x & 63;
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  int tok0 = (int)(at / c.H);
  const int h = (int)(at - (long long)tok0 * c.H);
  // the token's sequence b, with rows row0 .. end - 1 (as load_seq)
  int b = 0, row0 = 0, end = 0;
  if (most > 0) {
    b = tok0 / most;
    if (b >= c.B) return;
    row0 = c.seqs.start[b];
    end = c.seqs.start[b + 1];
    tok0 = max(row0, 0) + tok0 % most;
  } else if (c.seqs.start) {
    if (tok0 >= c.seqs.total) return;
    for (int b0 = 0; b0 < c.B; b0 += 64) {
      const int e = c.seqs.start[min(b0 + lane, c.B - 1) + 1], first = b0 == 0 ? c.seqs.start[0] : end;
      const int n = __popcll(__ballot(b0 + lane < c.B && e <= tok0));
      b += n;
      row0 = n > 0 ? __shfl(e, n - 1) : first;
      end = __shfl(e, min(n, 63));
      if (n < 64) break;
    }
  } else {
    b = tok0 / c.seqs.max_new;
    row0 = b * c.seqs.max_new;
    end = row0 + c.seqs.max_new;
  }
  row0 = max(row0, 0);
  const int n = min(min(end, c.seqs.start ? c.seqs.total : end) - row0, c.seqs.max_new), tok = tok0 - row0;
  if (b >= c.B || tok < 0 || tok >= n) return;
  const int group = c.H / c.Hkv, hk = h / group;
  const long long rows = (long long)n * group, row = (long long)tok * group + h - hk * group;
  const bool is_tile = tile.plan.shares > 0 && rows >= tile.plan.row_min;
  if (!is_tile && (few.plan.shares == 0 || rows > few.plan.row_max)) return;
  bch::SharePlan plan = few.plan;
  if (is_tile) plan = tile.plan;
  const float* const ws = is_tile ? tile.ws : few.ws;
  const long long list = ((long long)b * c.Hkv + hk) * plan.tiles + row / plan.rows;
  const int r = (int)(row % plan.rows);
  // (starts that do not ascend name lists that nobody noted: still no more than there is room for)
  const int2 note = reinterpret_cast<const int2*>(ws)[list];
  const int first = min(max(note.x, 0), plan.shares - 1), count = min(note.y, plan.shares - first);
  if (count <= 1) return;
  const float* const parts = ws + bch::notes_floats((long long)c.B * c.Hkv * plan.tiles);
  auto ml = [&](int u) { return parts + bch::part_at(plan, first, u, c.D) + (long long)plan.part_rows * c.D + 2 * r; };
  float ms = ml(min(lane, count - 1))[0], ls = ml(min(lane, count - 1))[1];
  float m = bch::wave_allreduce(lane < count ? ms : -INFINITY, bch::OpMax());
  for (int u0 = 64; u0 < count; u0 += 64)
    m = fmaxf(m, bch::wave_allreduce(u0 + lane < count ? ml(u0 + lane)[0] : -INFINITY, bch::OpMax()));
  float* dst = c.o + (c.seqs.start ? (long long)tok0 * c.ol.row : b * c.ol.batch + (long long)tok * c.ol.row) +
               h * c.ol.head;
  for (int d0 = 0; d0 < c.D; d0 += 128) {
    const int da = min(d0 + lane, c.D - 1), db = min(d0 + lane + 64, c.D - 1);
    float x = 0.0f, y = 0.0f, l = 0.0f;
    for (int u0 = 0; u0 < count; u0 += 64) {
      const bool on = u0 + lane < count;
      const int n = min(64, count - u0);
      if (count > 64) {
        ms = ml(min(u0 + lane, count - 1))[0];
        ls = ml(min(u0 + lane, count - 1))[1];
      }
      const float a = on ? __builtin_amdgcn_exp2f(ms - (m == -INFINITY ? 0.0f : m)) : 0.0f;
      l += bch::wave_allreduce(on ? a * ls : 0.0f, bch::OpSum());
      for (int u = 0; u < n; u += 8) {
        float vx[8], vy[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) {  // past the last part: it again, not added
          const float* po = parts + bch::part_at(plan, first, u0 + min(u + w, n - 1), c.D) + (long long)r * c.D;
          vx[w] = po[da];
          vy[w] = po[db];
        }
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (u + w < n) {
            const float f = bch::readlane(a, u + w);
            x = fmaf(f, vx[w], x);
            y = fmaf(f, vy[w], y);
          }
      }
    }
    if (d0 + lane < c.D) dst[d0 + lane] = l == 0.0f ? 0.0f : x / l;
    if (d0 + lane + 64 < c.D) dst[d0 + lane + 64] = l == 0.0f ? 0.0f : y / l;
  }
}

// Which kernels a call takes.  The tile kernel does a few rows of a sequence nearly as slowly as 256; a batch may
// mix prompts and single tokens, so each kernel serves its own sequences (16 ragged trees of up to 64 drafts: 320
// us on tiles alone, 282 on both, 118 with shares).
struct Route {
  bool tile, rows;
  bch::SharePlan tile_plan, rows_plan;
  size_t tile_bytes, bytes;
};
Route route(const PagedCall& c, int max_len, bool may_split) {
  const long long all = (c.seqs.start ? (long long)c.seqs.total : (long long)c.B * c.seqs.max_new) * c.H;
  if (!bch::fits_grid(all / 4 + 1, 256)) may_split = false;  // paged_combine's
  Route r{};
  // (a batch's short sequences are the other kernel's)
  r.tile = bch::sdpa_paged_tile_applies(c) && (!c.seqs.start || bch::sdpa_paged_rows_applies(c, bch::kFewRows));
  const int row_limit = r.tile ? bch::kFewRows : 0x7fffffff;
  // dense operands: every sequence has max_new rows
  r.rows = bch::sdpa_paged_rows_applies(c, row_limit) && !(r.tile && !c.seqs.start);
  if (r.tile) {
    r.tile_plan = bch::sdpa_paged_tile_plan(c, max_len, may_split);
    r.tile_bytes = (bch::share_bytes(c, r.tile_plan) + 255) / 256 * 256;
  }
  if (r.rows) r.rows_plan = bch::sdpa_paged_rows_plan(c, max_len, row_limit, may_split);
  r.bytes = r.tile_bytes + (r.rows ? bch::share_bytes(c, r.rows_plan) : 0);
  return r;
}

}  // namespace

namespace bch {

size_t sdpa_paged_workspace_bytes(const PagedCall& c, int max_len) { return route(c, max_len, true).bytes; }

const char* sdpa_paged_kernel_name(const PagedCall& c, int max_len) {
  thread_local char text[256];
  const Route r = route(c, max_len, true);
  int at = 0;
  auto add = [&](const char* name, const SharePlan& p) {
    at += snprintf(text + at, sizeof text - at, "%s%s rows=%d", at > 0 ? " + " : "", name, p.rows);
    if (p.whole()) at += snprintf(text + at, sizeof text - at, " dealt=%d", p.shares);
    else if (p.shares > 0) at += snprintf(text + at, sizeof text - at, " shares=%d least=%d", p.shares, p.min_share);
    else at += snprintf(text + at, sizeof text - at, " whole");
  };
  text[0] = 0;
  if (r.tile) add(c.D <= kTileDim ? "sdpa_paged_tile_kernel" : "sdpa_paged_wide_kernel", r.tile_plan);
  if (r.rows && r.rows_plan.tiles > 0) add("sdpa_paged_rows_kernel", r.rows_plan);
  if (r.bytes > 0) snprintf(text + at, sizeof text - at, " + paged_combine");
  else if (at == 0) snprintf(text, sizeof text, "sdpa_paged_any_kernel");
  return text;
}

hipError_t launch_sdpa_paged(hipStream_t s, const PagedCall& c, int max_len, void* ws, size_t ws_bytes) {
  Route r = route(c, max_len, true);
  if (ws_bytes < r.bytes) r = route(c, max_len, false);
  if (r.tile || r.rows) {
    float* tile_ws = r.tile_bytes > 0 ? static_cast<float*>(ws) : nullptr;
    float* rows_ws = r.bytes > r.tile_bytes ? static_cast<float*>(ws) + r.tile_bytes / sizeof(float) : nullptr;
    hipError_t e = r.tile ? launch_sdpa_paged_tile(s, c, r.tile_plan, tile_ws) : hipSuccess;
    if (e == hipSuccess && r.rows) e = launch_sdpa_paged_rows(s, c, r.rows_plan, rows_ws);
    if (e != hipSuccess || r.bytes == 0) return e;
    Combined a{r.tile_plan, tile_ws}, b{r.rows_plan, rows_ws};
    if (a.plan.whole()) a.plan.shares = 0;  // nothing of it to join
    if (b.plan.whole()) b.plan.shares = 0;
    const long long rows = (c.seqs.start ? (long long)c.seqs.total : (long long)c.B * c.seqs.max_new) * c.H;
    // where only short sequences can have been cut, their first tokens, if those are fewer
    const int group = c.H / c.Hkv, few = std::min(kFewRows / group, c.seqs.max_new);
    const bool only_few = r.tile && a.plan.shares == 0 && (long long)c.B * few * c.H < rows;
    const long long waves = only_few ? (long long)c.B * few * c.H : rows;
    if (waves == 0) return hipSuccess;
    hipLaunchKernelGGL(paged_combine, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, c, a, b, only_few ? few : 0);
    return hipGetLastError();
  }
  // the rows that there are, 2^23 workgroups a launch
  auto any = c.D <= 64    ? sdpa_paged_any_kernel<1>
             : c.D <= 256 ? nullptr  // the other kernels'
             : c.D <= 512 ? sdpa_paged_any_kernel<8>
                          : sdpa_paged_any_kernel<16>;
  const long long tokens = c.seqs.start ? (long long)c.seqs.total : (long long)c.B * c.seqs.max_new, most = 1LL << 23;
  if (!any || c.D > 1024 || tokens > (1LL << 40) / c.H) return hipErrorInvalidConfiguration;
  for (long long at = 0; at < tokens * c.H; at += most) {
    const dim3 grid((unsigned)std::min(most, tokens * c.H - at)), block(64 * kAnyWaves);
    hipLaunchKernelGGL(any, grid, block, 0, s, c, at);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace bch
