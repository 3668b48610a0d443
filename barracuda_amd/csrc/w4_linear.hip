// w4_linear.hip -- y = act(x W^T + bias) with 4-bit weights (w4.h), and the packing of such weights.  The reference's linear
// layer (shaders/misc/linear_f64.wgsl) has f32 weights only; this stands beside it (bch_sgemm_ex) for layers whose
// weights are most of what a step reads.
#include "w4.h"

#include <algorithm>

namespace {

using bch::W4;

constexpr int kThreads = 256;

// ---- packing: a thread a word of codes, then one a scale ----
__global__ __launch_bounds__(kThreads) void w4_pack_codes(W4 w, const unsigned char* __restrict__ codes, long long ld,
                                                          const unsigned char* __restrict__ zero, unsigned* out) {
  const long long total = 256LL * w.tiles * w.blocks, stride = (long long)gridDim.x * kThreads;
  const int real = (w.k - 1) / w.group + 1;
  for (long long at = (long long)blockIdx.x * kThreads + threadIdx.x; at < total; at += stride) {
    const int j = at & 3, lane = (int)(at >> 2) & 63;
    const long long block = at >> 8, tile = block / w.blocks;
    const long long o = 16 * tile + (lane & 15);
    const int i0 = 128 * (int)(block - tile * w.blocks) + 32 * j + 8 * (lane >> 4);
    unsigned word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = i0 + e;
      unsigned c = 8;
      if (o < w.n && i < w.k)
        c = (codes[o * ld + (i >> 1)] >> (4 * (i & 1))) & 15;
      else if (zero && o < w.n && i / w.group < real)
        c = zero[o * real + i / w.group] & 15;
      word |= c << (4 * (e / 2 + 4 * (e % 2)));
    }
    out[at] = word;
  }
}
__global__ __launch_bounds__(kThreads) void w4_pack_scales(W4 w, const float* __restrict__ scale,
                                                           const unsigned char* __restrict__ zero, float* s, unsigned char* z) {
  const long long total = 16LL * w.tiles * w.groups, stride = (long long)gridDim.x * kThreads;
  const int real = (w.k - 1) / w.group + 1;
  for (long long at = (long long)blockIdx.x * kThreads + threadIdx.x; at < total; at += stride) {
    const long long tg = at >> 4, tile = tg / w.groups, o = 16 * tile + (at & 15);
    const int g = (int)(tg - tile * w.groups);
    const bool on = o < w.n && g < real;
    s[at] = on ? scale[o * real + g] : 0.0f;
    z[at] = on && zero ? zero[o * real + g] & 15 : 8;
  }
}

}  // namespace

namespace bch {

hipError_t launch_w4_pack(hipStream_t s, const W4& w, const unsigned char* codes, long long ld, const float* scale,
                          const unsigned char* zero, void* out) {
  const W4 o = w4_of(w.n, w.k, w.group, out);
  const long long words = 256LL * w.tiles * w.blocks, scales = 16LL * w.tiles * w.groups;
  const unsigned most = 1u << 16;
  hipLaunchKernelGGL(w4_pack_codes, dim3((unsigned)std::min<long long>(most, (words - 1) / kThreads + 1)), dim3(kThreads), 0, s, w,
                     codes, ld, zero, static_cast<unsigned*>(out));
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(w4_pack_scales, dim3((unsigned)std::min<long long>(most, (scales - 1) / kThreads + 1)), dim3(kThreads), 0, s,
                     w, scale, zero, const_cast<float*>(o.scale), const_cast<unsigned char*>(o.zero));
  return hipGetLastError();
}

namespace {

// Scratch that a call of many rows asks for at most; more rows go through it in turn.
constexpr size_t kMostBytes = (size_t)256 << 20;

// The rows that go together, and how: kernels for few rows as long as their models say that they are done earlier.
struct Way {
  int rows;
  bool tile;
  W4Plan plan;
  size_t bytes;
};
Way way_of(int m, const W4& w, size_t most) {
  const int cus = device_cu_count(), few = std::min(m, kW4Few);
  for (const bool split : {true, false}) {
    const W4Plan f = w4_skinny_plan(few, w, cus, split), t = m > kW4Few ? w4_tile_plan(m, w, cus, split) : W4Plan{};
    if (m <= kW4Few || f.cost * ((m - 1) / few + 1) < t.cost) {
      if (w4_skinny_bytes(few, w, f) <= most) return {few, false, f, w4_skinny_bytes(few, w, f)};
    } else if (w4_tile_bytes(m, w, t) <= most) {
      return {m, true, t, w4_tile_bytes(m, w, t)};
    }
  }
  // as many rows as the scratch holds, in whole tiles where it holds one
  int rows = (int)std::min<long long>(m, (long long)(most / (w4_parts_bytes(128, w) / 128 + 1)));
  if (rows >= 128) {
    rows = rows / 128 * 128;
    return {rows, true, w4_tile_plan(rows, w, cus, false), w4_parts_bytes(rows, w)};
  }
  rows = std::min(rows / 8 * 8 - 8, kW4Few);
  if (rows < 8) return {0, false, {}, 0};
  const W4Plan p = w4_skinny_plan(rows, w, cus, false);
  return w4_skinny_bytes(rows, w, p) <= most ? Way{rows, false, p, w4_skinny_bytes(rows, w, p)} : Way{0, false, {}, 0};
}

}  // namespace

size_t w4_linear_workspace_bytes(int m, const W4& w) { return m <= 2 ? 0 : way_of(m, w, kMostBytes).bytes; }

hipError_t launch_w4_linear(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, size_t ws_bytes) {
  for (int at = 0; at < m;) {
    const int left = m - at;
    const Way way = left <= 2 ? Way{0, false, {}, 0} : way_of(left, w, std::min(ws_bytes, kMostBytes));
    const float* xs = x + at * ldx;
    float* ys = y + at * ldy;
    const int rows = way.rows > 0 ? std::min(left, way.rows) : std::min(left, 2);
    const hipError_t e = way.rows == 0 ? launch_w4_line(s, rows, w, xs, ldx, bias, act, ys, ldy)
                         : way.tile    ? launch_w4_tile(s, rows, w, xs, ldx, bias, act, ys, ldy, ws, way.plan)
                                       : launch_w4_skinny(s, rows, w, xs, ldx, bias, act, ys, ldy, ws, way.plan);
    if (e != hipSuccess) return e;
    at += rows;
  }
  return hipSuccess;
}

}  // namespace bch
