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

// ---- a few rows of x: f32 multiplications ----
// A workgroup takes 16 outputs and MT rows; its wavefronts share the blocks of inputs.  A lane holds 32 codes of its output,
// and its sums over a group's codes before they are scaled.
template <int MT>
__global__ __launch_bounds__(kThreads) void w4_rows_kernel(W4 w, int m, const float* __restrict__ x, long long ldx,
                                                           bool vec, const float* __restrict__ bias, int act, float* y,
                                                           long long ldy) {
  __shared__ float part[4][MT][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kb = lane >> 4;
  const int tile = blockIdx.x % w.tiles;
  const long long m0 = (long long)(blockIdx.x / w.tiles) * MT;
  float acc[MT] = {};
  for (int b = wave; b < w.blocks; b += 4) {
    const bch::u32x4 c = w.codes[((long long)tile * w.blocks + b) * 64 + lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i0 = 128 * b + 32 * j + 8 * kb;
      const long long g = (long long)tile * w.groups + (128 * b + 32 * j) / w.group;
      const float s = w.scale[16 * g + r];
      const int z = w.zero[16 * g + r];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)((int)((c[j] >> (4 * (e / 2 + 4 * (e % 2)))) & 15) - z);
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const float* row = x + min(m0 + u, (long long)m - 1) * ldx;
        float q[8];
        if (vec) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 t = i0 + 4 * h < w.k ? *reinterpret_cast<const float4*>(row + i0 + 4 * h) : make_float4(0, 0, 0, 0);
            q[4 * h] = t.x;
            q[4 * h + 1] = t.y;
            q[4 * h + 2] = t.z;
            q[4 * h + 3] = t.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = i0 + e < w.k ? row[i0 + e] : 0.0f;
        }
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[e], q[e], sum);
        acc[u] = fmaf(s, sum, acc[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    acc[u] += __shfl_xor(acc[u], 16);
    acc[u] += __shfl_xor(acc[u], 32);
    if (kb == 0) part[wave][u][r] = acc[u];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < 16 * MT; t += kThreads) {
    const int u = t >> 4, rr = t & 15, o = 16 * tile + rr;
    if (m0 + u >= m || o >= w.n) continue;
    float sum = (part[0][u][rr] + part[1][u][rr]) + (part[2][u][rr] + part[3][u][rr]);
    if (bias) sum += bias[o];
    y[(m0 + u) * ldy + o] = bch::activate(sum, act);
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

// Rows from which the matrix cores' tiles are taken.
constexpr int kTileFrom = 64;
// Scratch of a call: the parts of its rows, or of as many as take this much.
constexpr size_t kPartsMost = (size_t)256 << 20;

// The rows whose parts ws_bytes hold, in whole tiles of 128 where that is not all of them.
int rows_in(int m, const W4& w, size_t ws_bytes) {
  if (w4_parts_bytes(m, w) <= ws_bytes) return m;
  const long long fit = (long long)(ws_bytes / (w4_parts_bytes(128, w) / 128 + 1)) / 128 * 128;
  return (int)std::min<long long>(fit, m);
}

size_t w4_linear_workspace_bytes(int m, const W4& w) {
  if (m < kTileFrom) return 0;
  return std::min(w4_parts_bytes(m, w), std::max(kPartsMost, 2 * w4_parts_bytes(128, w)));
}

hipError_t launch_w4_linear(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, size_t ws_bytes) {
  const int fit = m < kTileFrom ? 0 : rows_in(m, w, ws_bytes);
  if (fit > 0) {
    for (int at = 0; at < m; at += fit) {
      const hipError_t e = launch_w4_tile(s, std::min(fit, m - at), w, x + at * ldx, ldx, bias, act, y + at * ldy, ldy, ws);
      if (e != hipSuccess || m - at <= fit) return e;
    }
  }
  const bool vec = w.k % 4 == 0 && ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int mt = m >= 8 ? 8 : m >= 4 ? 4 : m >= 2 ? 2 : 1;
  const long long per = (1LL << 23) / w.tiles * mt;  // rows a launch
  for (long long at = 0; at < m; at += per) {
    const int mm = (int)std::min<long long>(per, m - at);
    const dim3 grid((unsigned)((long long)w.tiles * ((mm - 1) / mt + 1))), block(kThreads);
    auto kern = mt == 8 ? w4_rows_kernel<8> : mt == 4 ? w4_rows_kernel<4> : mt == 2 ? w4_rows_kernel<2> : w4_rows_kernel<1>;
    hipLaunchKernelGGL(kern, grid, block, 0, s, w, mm, x + at * ldx, ldx, vec, bias, act, y + at * ldy, ldy);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace bch
