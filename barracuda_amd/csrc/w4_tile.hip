// w4_tile.hip -- many rows through a linear layer of 4-bit weights (w4.h) on the bf16 matrix cores.
//
// code - zero is a whole number within 15, exact in bf16; x is three bf16 parts (w4.h), so a product is three part products
// where one of f32 weights is six, and all three are exact.  A group's sum is accumulated in f32 by the matrix cores and
// joins the output's sum times its scale: 64 FMAs a wavefront and group.
//
// x is split once, by a kernel of its own (x is read by every column of tiles), each row by a power of two of its own.
#include "w4.h"

#include <algorithm>

namespace {

using bch::f32x16;
using bch::u32x4;
using bch::W4;

// ---- x into parts ----
// Part p, inputs 8 o .. 8 o + 7 of row r: 16 bytes at ((p octets + o) rows + r): neighbouring rows lie together, as the matrix
// cores take them.  A workgroup has ROWS rows, and a row THREADS / ROWS threads in turn: eight rows store whole lines of 128 bytes
// (2048 rows of 4096: 15 us), four have four times the threads where few rows leave CUs idle (65 rows, 11008 -> 4096: a
// call 66 us, 80 by eights).
constexpr int kSplitRows = 8, kSplitHeld = 8;

template <int ROWS, int THREADS>
__global__ __launch_bounds__(THREADS) void w4_split_kernel(int m, int k, int octets, int rows, const float* __restrict__ x,
                                                           long long ldx, bool vec, u32x4* parts, int* exponent) {
  constexpr int kStep = THREADS / ROWS;
  __shared__ unsigned tops[THREADS / 64][ROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rr = threadIdx.x % ROWS, o0 = threadIdx.x / ROWS;
  const int r = blockIdx.x * ROWS + rr;
  const float* row = x + min(r, m - 1) * ldx;
  float held[kSplitHeld][8];
  unsigned top = 0;
#pragma unroll
  for (int h = 0; h < kSplitHeld; ++h) {
    if (o0 + kStep * h < octets) {
      bch::w4_load8(held[h], row, 8 * (o0 + kStep * h), k, vec);
      top = bch::w4_top(held[h], top);
    }
  }
  for (int o = o0 + kStep * kSplitHeld; o < octets; o += kStep) {
    float v[8];
    bch::w4_load8(v, row, 8 * o, k, vec);
    top = bch::w4_top(v, top);
  }
#pragma unroll
  for (int d = ROWS; d < 64; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if (lane < ROWS) tops[wave][lane] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) top = max(top, tops[w][rr]);
  const int e = bch::w4_exponent(top);
  if ((int)threadIdx.x < ROWS && r < m) exponent[r] = bch::kW4Unit - e;
  auto put = [&](const float (&v)[8], int o) {
    u32x4 p[3];
    bch::w4_split(v, e, p);
#pragma unroll
    for (int q = 0; q < 3; ++q) parts[((long long)q * octets + o) * rows + r] = p[q];
  };
#pragma unroll
  for (int h = 0; h < kSplitHeld; ++h)
    if (o0 + kStep * h < octets) put(held[h], o0 + kStep * h);
  for (int o = o0 + kStep * kSplitHeld; o < octets; o += kStep) {
    float v[8];
    bch::w4_load8(v, row, 8 * o, k, vec);
    put(v, o);
  }
}

// ---- the product ----
// A workgroup has 128 rows and 256 outputs, 2 x 4 wavefronts of 64 x 64.  A pass is 32 inputs: the parts of x through LDS (double
// buffered, [part][octet][row], free of bank conflicts), the codes straight from memory into the wavefront that takes
// them apart, 128 inputs ahead.
constexpr int kRows = 128, kCols = 256, kThreads = 512;
constexpr int kPassBytes = 3 * 4 * kRows * 16, kTileBytes = 4 * kRows * kCols;
static_assert(kTileBytes >= 2 * kPassBytes, "two passes, then the results");

// FL: passes of one group in every 128 inputs (4: the group is a multiple of 128, 2: of 64, 1: of 32).
template <int FL>
__global__ __launch_bounds__(kThreads, 2) void w4_tile_kernel(W4 w, int m, int rows, int octets, const u32x4* __restrict__ parts,
                                                              const int* __restrict__ exponent, const float* __restrict__ bias,
                                                              int act, float* y, long long ldy, int mt, int nt, int per,
                                                              float* partial) {
  extern __shared__ u32x4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1, l32 = lane & 31, kh = lane >> 5;
  // the workgroups of an XCD (each eighth of them) take a contiguous range of tiles, rows first
  const int wgs = gridDim.x, share = wgs / 8, extra = wgs % 8, xcd = blockIdx.x % 8;
  const int at = xcd * share + min(xcd, extra) + blockIdx.x / 8;
  const int r0 = (at % mt) * kRows, c0 = (at / mt % nt) * kCols + 64 * wn, slice = at / mt / nt;
  const int b0 = slice * per, b1 = min(w.blocks, b0 + per);
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
  const int first = 4 * b0, last = 4 * b1 - 1;
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
  fetch(first);
  fetch_codes(codes, b0);
  put(0);
  fetch(min(first + 1, last));
  __syncthreads();
  for (int block = b0; block < b1; ++block) {
    u32x4 next[2][2];
    fetch_codes(next, min(block + 1, b1 - 1));
    float scale[2];
    unsigned zero[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 4 * block + j, buf = j & 1;
      if (j % FL == 0) {
        const int g = bch::w4_group(w, 4 * block + j);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          scale[b] = ps[b][16LL * g];
          zero[b] = bch::w4_zero(pz[b][16LL * g]);
        }
      }
      put(buf ^ 1);
      fetch(min(t + 2, last));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 a[2][3], v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 3; ++q)
            a[i][q] = lds[buf * (kPassBytes / 16) + (q * 4 + 2 * h + kh) * kRows + 64 * wm + 32 * i + l32];
#pragma unroll
        for (int b = 0; b < 2; ++b) v[b] = bch::w4_decode(codes[b][h][j], zero[b]);
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
  // out through LDS (the last pass has left it): whole rows of 256, and a loop of few instructions, not 64 times an activation's
  float* tile = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        tile[(64 * wm + 32 * i + 8 * (e / 4) + 4 * kh + e % 4) * kCols + 64 * wn + 32 * b + l32] = acc[i][b][e];
  __syncthreads();
  float* out = partial ? partial + (long long)slice * m * w.n : y;
  const long long ld = partial ? w.n : ldy;
  const bool wide = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll 1
  for (int j = threadIdx.x; j < kRows * kCols / 4; j += kThreads) {
    const int r = r0 + j / (kCols / 4), o = c0 - 64 * wn + j % (kCols / 4) * 4;
    if (r >= m) break;
    if (o >= w.n) continue;
    const int up = exponent[r];
    bch::f32x4 v = *reinterpret_cast<const bch::f32x4*>(tile + 4 * j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = ldexpf(v[e], up);
      if (!partial) {
        if (bias && o + e < w.n) v[e] += bias[o + e];
        v[e] = bch::activate(v[e], act);
      }
    }
    float* to = out + r * ld + o;
    if (wide && o + 3 < w.n) {
      *reinterpret_cast<bch::f32x4*>(to) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (o + e < w.n) to[e] = v[e];
    }
  }
}

// y = act(the slices' sums, in their order, + bias).
__global__ __launch_bounds__(256) void w4_reduce_kernel(int m, int n, int slices, const float* __restrict__ partial,
                                                        const float* __restrict__ bias, int act, float* y, long long ldy) {
  const long long total = (long long)m * n, stride = (long long)gridDim.x * 256;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += stride) {
    const long long r = at / n;
    const int o = (int)(at - r * n);
    float v = partial[at];
#pragma unroll 8
    for (int s = 1; s < slices; ++s) v += partial[s * total + at];
    if (bias) v += bias[o];
    y[r * ldy + o] = bch::activate(v, act);
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
  if (rows / kSplitRows < device_cu_count())
    hipLaunchKernelGGL((w4_split_kernel<4, 1024>), dim3(rows / 4), dim3(1024), 0, s, m, w.k, octets, rows, x, ldx, w4_vec(w, x, ldx), p, e);
  else
    hipLaunchKernelGGL((w4_split_kernel<8, 512>), dim3(rows / 8), dim3(512), 0, s, m, w.k, octets, rows, x, ldx, w4_vec(w, x, ldx), p, e);
  *parts = p;
  *exponent = e;
  return hipGetLastError();
}

hipError_t launch_w4_reduce(hipStream_t s, int m, int n, int slices, const float* partial, const float* bias, int act, float* y,
                            long long ldy) {
  const long long total = (long long)m * n;
  hipLaunchKernelGGL(w4_reduce_kernel, dim3((unsigned)std::min(4096LL, (total - 1) / 256 + 1)), dim3(256), 0, s, m, n, slices,
                     partial, bias, act, y, ldy);
  return hipGetLastError();
}

// The slices of inputs: 4.9 us for a round of workgroups and 128 inputs (2048 rows, or 128, 4096 -> 11008), 5 for the sums over
// the slices and their bytes, written and read, at 4 TB/s.  Up to 32 of them (65 rows, 11008 -> 4096: 17 slices 50 us, 8 66).
W4Plan w4_tile_plan(int m, const W4& w, int cus, bool may_split) {
  W4Plan best{0, 1, 0.0};
  const long long tiles = (long long)((m - 1) / kRows + 1) * ((w.n - 1) / kCols + 1);
  for (int s = 1; s <= (may_split ? 32 : 1) && s <= w.blocks; ++s) {
    const int per = (w.blocks - 1) / s + 1, slices = (w.blocks - 1) / per + 1;
    if (s > 1 && 4.0 * slices * m * w.n > 256e6) break;
    const double c = (double)((tiles * slices - 1) / cus + 1) * per * 4.9 +
                     (slices > 1 ? 5.0 + 2e-6 * slices * m * w.n : 0.0);
    if (best.cost == 0.0 || c < best.cost) best = {0, s, c};
  }
  best.cost += 3.0 + 1e-6 * 3.5 * m * w.k / 2;
  return best;
}
size_t w4_tile_bytes(int m, const W4& w, const W4Plan& p) {
  return w4_parts_bytes(m, w) + (p.slices > 1 ? 4ULL * p.slices * m * w.n : 0);
}

hipError_t launch_w4_tile(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy, void* ws, const W4Plan& p) {
  const u32x4* parts;
  const int* exponent;
  hipError_t e = launch_w4_split(s, m, w, x, ldx, ws, &parts, &exponent);
  if (e != hipSuccess) return e;
  const int rows = up(m, kSplitRows), mt = (m - 1) / kRows + 1, nt = (w.n - 1) / kCols + 1;
  const int per = (w.blocks - 1) / p.slices + 1, slices = (w.blocks - 1) / per + 1;
  float* partial = slices > 1 ? reinterpret_cast<float*>(static_cast<char*>(ws) + w4_parts_bytes(m, w)) : nullptr;
  auto kern = w.group % 128 == 0 ? w4_tile_kernel<4> : w.group % 64 == 0 ? w4_tile_kernel<2> : w4_tile_kernel<1>;
  e = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), kTileBytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)mt * nt * slices), dim3(kThreads), kTileBytes, s, w, m, rows, 16 * w.blocks, parts, exponent,
                     bias, act, y, ldy, mt, nt, per, partial);
  e = hipGetLastError();
  if (e != hipSuccess || slices == 1) return e;
  return launch_w4_reduce(s, m, w.n, slices, partial, bias, act, y, ldy);
}

}  // namespace bch
