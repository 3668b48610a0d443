// w4_tile.hip -- many rows through a linear layer of 4-bit weights (w4.h) on the bf16 matrix cores.
//
// code - zero is a whole number within 15, exact in bf16; x is three bf16 parts (x = x0 + x1 + x2 exactly, as
// bch_internal.h splits both operands of an f32 product), so a product is three part products where one of f32
// weights is six, and all three are exact.  A group's sum is accumulated in f32 by the matrix cores and joins the output's sum times
// its scale: 64 FMAs a wavefront and group.
//
// x is split once, by a kernel of its own (x is read by every column of tiles), each row scaled by a power of two that puts its
// largest value between 2^30 and 2^31: parts below bf16's smallest then are 2^-140 of it, and a sum of 2^20 products stays far
// from f32's largest.  The outputs are scaled back by an exponent.  An infinity or a NaN is its first part alone, so that it
// gives what it gives in f32: the row's other outputs' sums do not see it.
#include "w4.h"

#include <algorithm>

namespace {

using bch::f32x16;
using bch::u32x4;
using bch::W4;

// ---- x into parts ----
// Part p, inputs 8 o .. 8 o + 7 of row r: 16 bytes at ((p octets + o) rows + r): neighbouring rows lie together, as the matrix
// cores take them.  A workgroup has 8 rows; a thread every 64th octet of one.
constexpr int kSplitThreads = 512, kSplitRows = 8, kSplitHeld = 8;

__device__ __forceinline__ void load8(float (&v)[8], const float* row, int i0, int k, bool vec) {
  if (vec) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 t = i0 + 4 * h < k ? *reinterpret_cast<const float4*>(row + i0 + 4 * h) : make_float4(0, 0, 0, 0);
      v[4 * h] = t.x;
      v[4 * h + 1] = t.y;
      v[4 * h + 2] = t.z;
      v[4 * h + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i0 + e < k ? row[i0 + e] : 0.0f;
  }
}
__device__ __forceinline__ unsigned top_bits(const float (&v)[8], unsigned top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned b = __builtin_bit_cast(unsigned, v[e]) & 0x7fffffffu;
    if (b < 0x7f800000u) top = max(top, b);  // finite
  }
  return top;
}

__global__ __launch_bounds__(kSplitThreads) void w4_split_kernel(int m, int k, int octets, int rows, const float* __restrict__ x,
                                                                 long long ldx, bool vec, u32x4* parts, int* exponent) {
  __shared__ unsigned tops[8][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rr = threadIdx.x & 7, o0 = threadIdx.x >> 3;
  const int r = blockIdx.x * kSplitRows + rr;
  const float* row = x + min(r, m - 1) * ldx;
  float held[kSplitHeld][8];
  unsigned top = 0;
#pragma unroll
  for (int h = 0; h < kSplitHeld; ++h) {
    if (o0 + 64 * h < octets) {
      load8(held[h], row, 8 * (o0 + 64 * h), k, vec);
      top = top_bits(held[h], top);
    }
  }
  for (int o = o0 + 64 * kSplitHeld; o < octets; o += 64) {
    float v[8];
    load8(v, row, 8 * o, k, vec);
    top = top_bits(v, top);
  }
#pragma unroll
  for (int d = 8; d < 64; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if (lane < 8) tops[wave][lane] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, tops[w][rr]);
  // the largest is below 2^e
  int e = 0;
  if (top) (void)frexpf(__builtin_bit_cast(float, top), &e);
  if (threadIdx.x < 8 && r < m) exponent[r] = e - 31;
  auto put = [&](float (&v)[8], int o) {
    u32x4 p[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = ldexpf(v[2 * i], 31 - e), b = ldexpf(v[2 * i + 1], 31 - e);
      const bool fa = __builtin_isfinite(a), fb = __builtin_isfinite(b);
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        p[q][i] = bch::bf16_pack(a, b);
        if (q < 2) {
          a = fa ? a - __builtin_bit_cast(float, p[q][i] << 16) : 0.0f;
          b = fb ? b - __builtin_bit_cast(float, p[q][i] & 0xffff0000u) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) parts[((long long)q * octets + o) * rows + r] = p[q];
  };
  if (r >= rows) return;
#pragma unroll
  for (int h = 0; h < kSplitHeld; ++h)
    if (o0 + 64 * h < octets) put(held[h], o0 + 64 * h);
  for (int o = o0 + 64 * kSplitHeld; o < octets; o += 64) {
    float v[8];
    load8(v, row, 8 * o, k, vec);
    put(v, o);
  }
}

// ---- the product ----
// A workgroup has 128 rows and 256 outputs, 2 x 4 wavefronts of 64 x 64.  A pass is 32 inputs: the parts of x through LDS (double
// buffered, [part][octet][row], free of bank conflicts), the codes straight from memory into the wavefront that takes
// them apart, 128 inputs ahead.
constexpr int kRows = 128, kCols = 256, kThreads = 512;
constexpr int kPassBytes = 3 * 4 * kRows * 16;

// Eight codes as bf16 of code - zero: bytes to floats, and the floats' upper halves.
__device__ __forceinline__ u32x4 decode(unsigned c, float zero) {
  const unsigned lo = c & 0x0f0f0f0fu, hi = (c >> 4) & 0x0f0f0f0fu;
  float v[8];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const unsigned t = s & 1 ? hi : lo;
    v[2 * s] = (float)((t >> (8 * (s >> 1))) & 0xffu) - zero;
    v[2 * s + 1] = (float)((t >> (8 * (s >> 1) + 16)) & 0xffu) - zero;
  }
  u32x4 p;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    p[s] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, v[2 * s + 1]), __builtin_bit_cast(unsigned, v[2 * s]), 0x07060302u);
  return p;
}

// FL: passes of one group in every 128 inputs (4: the group is a multiple of 128, 2: of 64, 1: of 32).
template <int FL>
__global__ __launch_bounds__(kThreads, 2) void w4_tile_kernel(W4 w, int m, int rows, int octets, const u32x4* __restrict__ parts,
                                                              const int* __restrict__ exponent, const float* __restrict__ bias,
                                                              int act, float* y, long long ldy, int mt, int nt) {
  extern __shared__ u32x4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1, l32 = lane & 31, kh = lane >> 5;
  // the workgroups of an XCD (each eighth of them) take a contiguous range of tiles, rows first
  const int wgs = mt * nt, per = wgs / 8, extra = wgs % 8, xcd = blockIdx.x % 8;
  const int at = xcd * per + min(xcd, extra) + blockIdx.x / 8;
  const int r0 = (at % mt) * kRows, c0 = (at / mt) * kCols + 64 * wn;
  // this thread's three pieces of a pass: octet and row of each part
  const int po = threadIdx.x >> 7, pr = threadIdx.x & 127;
  const u32x4* px = parts + (long long)po * rows + min(r0 + pr, rows - 1);
  const long long part = (long long)octets * rows;
  // codes of the wavefront's two blocks of 32 outputs: tile of 16, and this lane's 16 bytes of the block for each half pass
  const u32x4* pc[2];
  const float* ps[2];
  const unsigned char* pz[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int tile = min((c0 + 32 * b + l32) / 16, w.tiles - 1);
    pc[b] = w.codes + (long long)tile * w.blocks * 64 + kh * 16 + (lane & 15);
    ps[b] = w.scale + (long long)tile * w.groups * 16 + (lane & 15);
    pz[b] = w.zero + (long long)tile * w.groups * 16 + (lane & 15);
  }
  f32x16 acc[2][2] = {}, sum[2][2];
  u32x4 stage[3], codes[2][2];
  const int passes = 4 * w.blocks;
  auto fetch = [&](int t) {
#pragma unroll
    for (int q = 0; q < 3; ++q) stage[q] = px[q * part + (long long)t * 4 * rows];
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int q = 0; q < 3; ++q) lds[buf * (kPassBytes / 16) + q * 4 * kRows + threadIdx.x] = stage[q];
  };
  auto fetch_codes = [&](u32x4 (&c)[2][2], int block) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) c[b][h] = pc[b][(long long)block * 64 + h * 32];
  };
  fetch(0);
  fetch_codes(codes, 0);
  put(0);
  fetch(min(1, passes - 1));
  __syncthreads();
  for (int block = 0; block < w.blocks; ++block) {
    u32x4 next[2][2];
    fetch_codes(next, min(block + 1, w.blocks - 1));
    float scale[2], zero[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * block + j, buf = j & 1;
      if (j % FL == 0) {
        const int g = (128 * block + 32 * j) / w.group;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          scale[b] = ps[b][16LL * g];
          zero[b] = (float)pz[b][16LL * g];
        }
      }
      put(buf ^ 1);
      fetch(min(t + 2, passes - 1));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 a[2][3], v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 3; ++q)
            a[i][q] = lds[buf * (kPassBytes / 16) + (q * 4 + 2 * h + kh) * kRows + 64 * wm + 32 * i + l32];
#pragma unroll
        for (int b = 0; b < 2; ++b) v[b] = decode(codes[b][h][j], zero[b]);
#pragma unroll
        for (int q = 2; q >= 0; --q)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const bool fresh = j % FL == 0 && h == 0 && q == 2;
              sum[i][b] = bch::bf16_mm(a[i][q], v[b], fresh ? f32x16{} : sum[i][b]);
            }
      }
      if (j % FL == FL - 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][b][e] = fmaf(scale[b], sum[i][b][e], acc[i][b][e]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) codes[b][h] = next[b][h];
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int o = c0 + 32 * b + l32;
    if (o >= w.n) continue;
    const float add = bias ? bias[o] : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = r0 + 64 * wm + 32 * i + 8 * (e / 4) + 4 * kh + e % 4;
        if (r < m) {
          float v = ldexpf(acc[i][b][e], exponent[r]);
          if (bias) v += add;
          y[r * ldy + o] = bch::activate(v, act);
        }
      }
  }
}

int up(int x, int to) { return (x - 1) / to * to + to; }

}  // namespace

namespace bch {

size_t w4_parts_bytes(int m, const W4& w) {
  return 3ULL * 16 * w.blocks * up(m, kSplitRows) * 16 + 4ULL * up(m, 64);
}

hipError_t launch_w4_split(hipStream_t s, int m, const W4& w, const float* x, long long ldx, void* ws, const u32x4** parts,
                           const int** exponent) {
  const int rows = up(m, kSplitRows), octets = 16 * w.blocks;
  u32x4* p = static_cast<u32x4*>(ws);
  int* e = reinterpret_cast<int*>(p + 3LL * octets * rows);
  const bool vec = w.k % 4 == 0 && ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  hipLaunchKernelGGL(w4_split_kernel, dim3(rows / kSplitRows), dim3(kSplitThreads), 0, s, m, w.k, octets, rows, x, ldx, vec, p, e);
  *parts = p;
  *exponent = e;
  return hipGetLastError();
}

hipError_t launch_w4_tile(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy, void* ws) {
  const u32x4* parts;
  const int* exponent;
  hipError_t e = launch_w4_split(s, m, w, x, ldx, ws, &parts, &exponent);
  if (e != hipSuccess) return e;
  const int rows = up(m, kSplitRows), mt = (m - 1) / kRows + 1, nt = (w.n - 1) / kCols + 1;
  auto kern = w.group % 128 == 0 ? w4_tile_kernel<4> : w.group % 64 == 0 ? w4_tile_kernel<2> : w4_tile_kernel<1>;
  const int bytes = 2 * kPassBytes;
  hipLaunchKernelGGL(kern, dim3(mt * nt), dim3(kThreads), bytes, s, w, m, rows, 16 * w.blocks, parts, exponent, bias, act, y,
                     ldy, mt, nt);
  return hipGetLastError();
}

}  // namespace bch
