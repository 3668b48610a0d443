// w4_skinny.hip -- few rows through a linear layer of 4-bit weights (w4.h): the weights' stream bounds it.
//
// Up to two rows: f32 multiplications.  From three on the bf16 matrix cores, 16 x 16 x 32, with x in three parts that a kernel of
// its own has made (w4_tile.hip).
#include "w4.h"

#include <algorithm>

namespace {

using bch::u32x4;
using bch::W4;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
constexpr int kThreads = 512, kWaves = 8;

__device__ __forceinline__ f32x4_t mm16(u32x4 a, u32x4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bch::bf16x8, a), __builtin_bit_cast(bch::bf16x8, b), c, 0, 0, 0);
}

// ---- one or two rows: f32 multiplications ----
// A workgroup has 16 outputs, its wavefronts every 16th or eighth block of inputs, two of them in flight each; x lies in LDS.  What
// bounds it: the launch, the first trip to memory, the codes' stream.  One row, 4096 -> 11008 / 50000 and back, us: 16 wavefronts
// 9.2 / 31 / 9.2, eight 8.9 / 25 to 26 / 10.9; two rows 11.2 / 36 / 10.9 and 12.1 / 38 / 12.  So eight where one row has more workgroups than two
// a CU, else 16.  Four blocks in flight: eight wavefronts 9.8 / 33 / 10.4, 16 12.6 and 9.5.
constexpr int kLineBlocks = 64;  // blocks of x in LDS at a time

// Code e of a word is nibble e / 2 + 4 (e % 2): its byte of the masked word, as a float.
__device__ __forceinline__ void codes_of(unsigned c, float zero, float (&v)[8]) {
  unsigned lo = c & 0x0f0f0f0fu, hi = (c >> 4) & 0x0f0f0f0fu;
  // (kept as they are: a byte of them converts in one instruction, four bits of c in two)
  asm("" : "+v"(lo), "+v"(hi));
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const unsigned t = s & 1 ? hi : lo;
    v[2 * s] = (float)((t >> (8 * (s >> 1))) & 0xffu) - zero;
    v[2 * s + 1] = (float)((t >> (8 * (s >> 1) + 16)) & 0xffu) - zero;
  }
}

// A group's inputs times its whole numbers are added up before the scale: up to 2^11 times an input, and what a small scale would bring
// back into f32's range may have left it.  Such rows are computed again times 2^-kDown: this lane's part of an output's sum of
// blocks b0, b0 + step, ..  (codes, scales and zeros are the lane's.)
constexpr int kDown = 12;
__device__ __forceinline__ float line_again(const W4& w, const u32x4* codes, const float* scales, const unsigned char* zeros,
                                            const float* row, bool vec, int b0, int b1, int step) {
  const int kb = (threadIdx.x & 63) >> 4;
  float sum = 0.0f;
#pragma unroll 1
  for (int b = b0; b < b1; b += step) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const long long g = bch::w4_group(w, 4 * b + j);
      float v[8], q[8], one = 0.0f;
      codes_of(reinterpret_cast<const unsigned*>(codes + (long long)b * 64)[j], (float)zeros[16 * g], v);
      bch::w4_load8(q, row, 128 * b + 32 * j + 8 * kb, w.k, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) one = fmaf(v[e], ldexpf(q[e], -kDown), one);
      sum = fmaf(scales[16 * g], one, sum);
    }
  }
  sum += __shfl_xor(sum, 16);
  return sum + __shfl_xor(sum, 32);
}

template <int MT, int FL, int THREADS>
__global__ __launch_bounds__(THREADS) void w4_line_kernel(W4 w, const float* __restrict__ x, long long ldx, bool vec,
                                                           const float* __restrict__ bias, int act, float* y, long long ldy) {
  constexpr int kOf = THREADS / 64;
  __shared__ float4 xs[MT][kLineBlocks * 32];
  __shared__ float part[kOf][MT][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, kb = lane >> 4;
  const int tile = blockIdx.x;
  const u32x4* codes = w.codes + (long long)tile * w.blocks * 64 + lane;
  const float* scales = w.scale + (long long)tile * w.groups * 16 + r;
  const unsigned char* zeros = w.zero + (long long)tile * w.groups * 16 + r;
  constexpr int kFlight = 2, kPer = 4 / FL;  // blocks in flight, groups of one
  float acc[MT] = {};
  for (int base = 0; base < w.blocks; base += kLineBlocks) {
    const int end = min(w.blocks, base + kLineBlocks);
    u32x4 c[kFlight];
    float s[kFlight][kPer], z[kFlight][kPer];
    auto fetch = [&](int b0) {
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int b = min(b0 + kOf * f, end - 1);
        c[f] = __builtin_nontemporal_load(codes + (long long)b * 64);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const long long g = bch::w4_group(w, 4 * b + FL * i);
          s[f][i] = scales[16 * g];
          z[f][i] = (float)zeros[16 * g];
        }
      }
    };
    fetch(min(base + wave, end - 1));
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MT; ++u)
      for (int i = threadIdx.x; i < (end - base) * 16; i += THREADS) {
        float v[8];
        bch::w4_load8(v, x + u * ldx, 128 * base + 8 * i, w.k, vec);
        xs[u][2 * i] = make_float4(v[0], v[1], v[2], v[3]);
        xs[u][2 * i + 1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    __syncthreads();
    for (int b0 = base + wave; b0 < end; b0 += kOf * kFlight) {
      u32x4 cc[kFlight];
      float ss[kFlight][kPer], zz[kFlight][kPer];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        cc[f] = c[f];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          ss[f][i] = s[f][i];
          zz[f][i] = z[f][i];
        }
      }
      if (b0 + kOf * kFlight < end) fetch(b0 + kOf * kFlight);
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int b = b0 + kOf * f;
        if (b >= end) break;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          float sum[MT] = {};
#pragma unroll
          for (int jj = 0; jj < FL; ++jj) {
            const int j = FL * i + jj;
            float v[8];
            codes_of(cc[f][j], zz[f][i], v);
#pragma unroll
            for (int u = 0; u < MT; ++u) {
              const float4* q = &xs[u][(b - base) * 32 + 8 * j + 2 * kb];
              const float4 q0 = q[0], q1 = q[1];
              sum[u] = fmaf(v[0], q0.x, sum[u]);
              sum[u] = fmaf(v[1], q0.y, sum[u]);
              sum[u] = fmaf(v[2], q0.z, sum[u]);
              sum[u] = fmaf(v[3], q0.w, sum[u]);
              sum[u] = fmaf(v[4], q1.x, sum[u]);
              sum[u] = fmaf(v[5], q1.y, sum[u]);
              sum[u] = fmaf(v[6], q1.z, sum[u]);
              sum[u] = fmaf(v[7], q1.w, sum[u]);
            }
          }
#pragma unroll
          for (int u = 0; u < MT; ++u) acc[u] = fmaf(ss[f][i], sum[u], acc[u]);
        }
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
  if (wave > 0) return;
  const int o = 16 * tile + r;
  const bool on = kb < MT && o < w.n;
  float sum = 0.0f;
  if (on) {
#pragma unroll
    for (int v = 0; v < kOf; ++v) sum += part[v][kb][r];
  }
  if (__any(!(fabsf(sum) < INFINITY))) {
#pragma unroll 1
    for (int u = 0; u < MT; ++u) {
      const bool lost = kb == u && !(fabsf(sum) < INFINITY);
      if (!__any(lost)) continue;
      // lost before the scale, if the row's inputs are finite (a row with one that is not: 11 us instead of 9, two 15 instead of 11)
      const float* row = x + u * ldx;
      bool finite = true;
#pragma unroll 1
      for (unsigned i = lane; i < (unsigned)w.k; i += 64 * 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row[min(i + 64 * e, (unsigned)w.k - 1)];
#pragma unroll
        for (int e = 0; e < 8; ++e) finite &= fabsf(v[e]) < INFINITY;
      }
      if (!__all(finite)) continue;
      const float again = ldexpf(line_again(w, codes, scales, zeros, row, vec, 0, w.blocks, 1), kDown);
      if (lost) sum = again;
    }
  }
  if (on) {
    if (bias) sum += bias[o];
    y[kb * ldy + o] = bch::activate(sum, act);
  }
}

// ---- up to 64 rows ----
// x's parts are of 2^kUp x here, whatever the row: no row has to be read whole before the first part is written.  2^kUp takes back
// kW4Unit: sums are what they stand for, finite wherever f32 is, and subnormal numbers keep their bits.  A value
// from 2^36 on would leave bf16's range; its row and chunk are noted, and the product computes such rows again in f32.
constexpr int kUp = bch::kW4Unit;
constexpr float kMost = 0x1p36f;
constexpr int kSplitThreads = 256, kSplitRows = 8, kSplitOctets = kSplitThreads / kSplitRows;

__global__ __launch_bounds__(kSplitThreads) void w4_split_few_kernel(int m, int k, int octets, int rows, const float* __restrict__ x,
                                                                     long long ldx, bool vec, u32x4* parts, unsigned* big) {
  const int r = blockIdx.y * kSplitRows + threadIdx.x % kSplitRows, o = blockIdx.x * kSplitOctets + threadIdx.x / kSplitRows;
  float v[8];
  bool large = false;
  if (o < octets) {
    bch::w4_load8(v, x + min(r, m - 1) * ldx, 8 * o, k, vec);
    u32x4 p[3];
    bch::w4_split(v, kUp, p);
#pragma unroll
    for (int q = 0; q < 3; ++q) parts[((long long)q * octets + o) * rows + r] = p[q];
#pragma unroll
    for (int e = 0; e < 8; ++e) large |= fabsf(v[e]) >= kMost && fabsf(v[e]) < INFINITY;
  }
  // bit r of the word of 8 rows and this chunk
  __shared__ unsigned rowbits[kSplitThreads / 64];
  unsigned long long any = __ballot(large);
#pragma unroll
  for (int d = 32; d >= 8; d /= 2) any |= any >> d;
  if (threadIdx.x % 64 == 0) rowbits[threadIdx.x / 64] = (unsigned)any & 0xff;
  __syncthreads();
  if (threadIdx.x == 0) big[blockIdx.y * gridDim.x + blockIdx.x] = rowbits[0] | rowbits[1] | rowbits[2] | rowbits[3];
}

// A workgroup has 16 T outputs of 16 MB rows and a range of blocks of inputs (`per` of them; others have the rest, blockIdx.x /
// groups).  Its eight wavefronts take every eighth block each: operands come straight from memory in the layouts that the matrix
// cores take, codes kAhead blocks before they are taken, x's parts kSteps - 1 steps of 32 inputs before, and no
// wavefront waits for another until their sums meet in LDS.  What bounds it: the first 4.5 us go by until data has come to all
// wavefronts, then 3 KB of x's parts for every 32 inputs and 16 rows of each T tiles of weights.
// Measured, 4096 -> 11008, us at 16 / 32 / 64 rows: this 15.2 / 20.8 / 33.1; with two steps of x's parts instead of four 19.8 / 26.0
// / 33.1; x split by the workgroup itself, through LDS, inputs over six workgroups 18.8 / 24.6 / 40.1.
constexpr int kAhead = 2;

template <int MB, int T, int FL>
__global__ __launch_bounds__(kThreads, 2) void w4_skinny_kernel(W4 w, int m, int rows, int octets,
                                                                const u32x4* __restrict__ parts, const unsigned* __restrict__ big,
                                                                const float* __restrict__ x, long long ldx, bool vec,
                                                                const float* __restrict__ bias, int act, float* y, long long ldy,
                                                                int groups, int per, float* partial) {
  constexpr int kPer = 4 / FL, kSteps = MB <= 2 ? 4 : 2;
  extern __shared__ f32x4_t meet[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, kb = lane >> 4;
  const int group = blockIdx.x % groups, slice = blockIdx.x / groups;
  const int b0 = slice * per, b1 = min(w.blocks, b0 + per);
  const u32x4* codes[T];
  const float* scales[T];
  const unsigned char* zeros[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = min(group * T + t, w.tiles - 1);
    codes[t] = w.codes + (long long)tile * w.blocks * 64 + lane;
    scales[t] = w.scale + (long long)tile * w.groups * 16 + l16;
    zeros[t] = w.zero + (long long)tile * w.groups * 16 + l16;
  }
  const u32x4* px[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) px[mb] = parts + kb * rows + min(16 * mb + l16, rows - 1);
  const long long part = (long long)octets * rows;
  f32x4_t acc[T][MB] = {};
  u32x4 c[kAhead][T], a[kSteps][MB][3];
  float s[kAhead][T][kPer];
  unsigned char z[kAhead][T][kPer];
  auto fetch_codes = [&](int n, int b) {
    b = min(b, b1 - 1);
#pragma unroll
    for (int t = 0; t < T; ++t) c[n][t] = __builtin_nontemporal_load(codes[t] + (long long)b * 64);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const long long g = bch::w4_group(w, 4 * b + FL * i);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        s[n][t][i] = scales[t][16 * g];
        z[n][t][i] = zeros[t][16 * g];
      }
    }
  };
  // step j of block b, or of the wavefront's next
  auto fetch_x = [&](int b, int j) {
    const long long at = (long long)(4 * (4 * min(j < 4 ? b : b + kWaves, b1 - 1) + j % 4)) * rows;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int q = 0; q < 3; ++q) a[j % kSteps][mb][q] = px[mb][q * part + at];
  };
  if (b0 + wave < b1) {
    fetch_codes(0, b0 + wave);
#pragma unroll
    for (int j = 0; j < kSteps - 1; ++j) fetch_x(b0 + wave, j);
#pragma unroll
    for (int n = 1; n < kAhead; ++n) fetch_codes(n, b0 + wave + n * kWaves);
  }
  for (int base = b0 + wave; base < b1; base += kAhead * kWaves) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int b = base + n * kWaves;
      if (b >= b1) break;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        f32x4_t sum[T][MB];
        unsigned zz[T];
#pragma unroll
        for (int t = 0; t < T; ++t) zz[t] = bch::w4_zero(z[n][t][i]);
#pragma unroll
        for (int jj = 0; jj < FL; ++jj) {
          const int j = FL * i + jj;
          fetch_x(b, j + kSteps - 1);
          u32x4 v[T];
#pragma unroll
          for (int t = 0; t < T; ++t) v[t] = bch::w4_decode(c[n][t][j], zz[t]);
#pragma unroll
          for (int q = 2; q >= 0; --q)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int t = 0; t < T; ++t)
                sum[t][mb] = mm16(a[j % kSteps][mb][q], v[t], jj == 0 && q == 2 ? f32x4_t{} : sum[t][mb]);
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][mb][e] = fmaf(s[n][t][i], sum[t][mb][e], acc[t][mb][e]);
      }
      fetch_codes(n, b + kAhead * kWaves);
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) meet[(wave * T * MB + t * MB + mb) * 64 + lane] = acc[t][mb];
  // which rows hold values too large (of any chunk)
  const int chunks = (octets - 1) / kSplitOctets + 1;
  unsigned found = 0;
  for (int i = threadIdx.x; i < rows / 8 * chunks; i += kThreads) found |= big[i];
  const bool again = __syncthreads_or(found != 0);
  float* p = partial ? partial + (long long)slice * m * w.n : nullptr;
  for (int i = threadIdx.x; i < T * MB * 64; i += kThreads) {
    f32x4_t sum = meet[i];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) sum += meet[v * T * MB * 64 + i];
    const int o = 16 * (group * T + i / 64 / MB) + (i & 15), r0 = 16 * (i / 64 % MB) + 4 * (i >> 4 & 3);
    if (o >= w.n) continue;
    const float add = bias ? bias[o] : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = r0 + e;
      if (r >= m) continue;
      float v = sum[e];
      if (p) {
        p[(long long)r * w.n + o] = v;
      } else {
        if (bias) v += add;
        y[r * ldy + o] = bch::activate(v, act);
      }
    }
  }
  if (!again) return;
  for (int r = 0; r < m; ++r) {
    unsigned bits = 0;
    for (int i = threadIdx.x; i < chunks; i += kThreads) bits |= big[r / 8 * chunks + i];
    __syncthreads();  // (the sums of the row before have been read)
    if (!__syncthreads_or(bits >> (r % 8) & 1)) continue;
    float* f = reinterpret_cast<float*>(meet);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float sum = 0.0f;
      for (int b = b0 + wave; b < b1; b += kWaves) {
        const u32x4 cc = codes[t][(long long)b * 64];
        for (int j = 0; j < 4; ++j) {
          const long long g = bch::w4_group(w, 4 * b + j);
          float v[8], q[8], one = 0.0f;
          codes_of(cc[j], (float)zeros[t][16 * g], v);
          bch::w4_load8(q, x + r * ldx, 128 * b + 32 * j + 8 * kb, w.k, vec);
#pragma unroll
          for (int e = 0; e < 8; ++e) one = fmaf(v[e], ldexpf(q[e], -kDown), one);
          sum = fmaf(scales[t][16 * g], one, sum);
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (kb == 0) f[(wave * T + t) * 16 + l16] = sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * T; i += kThreads) {
      const int o = 16 * group * T + i;
      if (o >= w.n) continue;
      float v = 0.0f;
#pragma unroll
      for (int u = 0; u < kWaves; ++u) v += f[u * T * 16 + i];
      v = ldexpf(v, kDown);
      if (p) {
        p[(long long)r * w.n + o] = v;
      } else {
        if (bias) v += bias[o];
        y[r * ldy + o] = bch::activate(v, act);
      }
    }
  }
}

typedef void (*SkinnyKernel)(W4, int, int, int, const u32x4*, const unsigned*, const float*, long long, bool, const float*, int, float*, long long, int, int, float*);

template <int MB, int T>
SkinnyKernel by_group(int group) {
  return group % 128 == 0 ? w4_skinny_kernel<MB, T, 4>
         : group % 64 == 0 ? w4_skinny_kernel<MB, T, 2>
                           : w4_skinny_kernel<MB, T, 1>;
}

}  // namespace

namespace bch {

hipError_t launch_w4_line(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy) {
#define BCH_LINE(M, N) \
  (w.group % 128 == 0 ? w4_line_kernel<M, 4, N> : w.group % 64 == 0 ? w4_line_kernel<M, 2, N> : w4_line_kernel<M, 1, N>)
  const bool wide = m == 1 && w.tiles > 2 * device_cu_count();
  auto kern = m == 2 ? BCH_LINE(2, 1024) : wide ? BCH_LINE(1, 512) : BCH_LINE(1, 1024);
#undef BCH_LINE
  hipLaunchKernelGGL(kern, dim3(w.tiles), dim3(wide ? 512 : 1024), 0, s, w, x, ldx, w4_vec(w, x, ldx), bias, act, y, ldy);
  return hipGetLastError();
}

// How much a call of m rows takes, in us, with t tiles of 16 outputs a workgroup and the inputs cut into `slices`: what a wavefront's
// block takes (0.6 for 16 rows of x's parts, 0.5 and 0.12 for 16 rows for each tile), for all that a CU's workgroups
// have of them, and 3.5 for the sums over the slices.  Fitted at 16 to 64 rows, 4096 -> 11008 and back.
namespace {
double skinny_cost(int m, const W4& w, int t, int slices, int cus) {
  const int mb = (m - 1) / 16 + 1, per = (w.blocks - 1) / slices + 1;
  const long long groups = (long long)((w.tiles - 1) / t + 1) * ((w.blocks - 1) / per + 1);
  const double rounds = (double)((groups - 1) / cus + 1) * ((per - 1) / kWaves + 1);
  return rounds * (0.6 * mb + t * (0.5 + 0.12 * mb)) + (slices > 1 ? 3.5 + 2e-6 * slices * m * w.n : 0.0);
}
}  // namespace

W4Plan w4_skinny_plan(int m, const W4& w, int cus, bool may_split) {
  W4Plan best{1, 1, 0.0};
  const int most = m > 32 ? 3 : 4;
  for (int t = 1; t <= most; ++t)
    for (int s = 1; s <= (may_split ? 8 : 1) && s <= w.blocks; ++s) {
      const double c = skinny_cost(m, w, t, s, cus);
      if (best.cost == 0.0 || c < best.cost) best = {t, s, c};
    }
  best.cost += 8.0;
  return best;
}

static size_t few_bytes(int m, const W4& w) {
  const long long rows = (m + 7) / 8 * 8, octets = 16LL * w.blocks, chunks = (octets - 1) / kSplitOctets + 1;
  return (size_t)(48 * octets * rows + (4 * chunks * rows / 8 + 255) / 256 * 256);
}
size_t w4_skinny_bytes(int m, const W4& w, const W4Plan& p) {
  return few_bytes(m, w) + (p.slices > 1 ? 4ULL * p.slices * m * w.n : 0);
}

hipError_t launch_w4_skinny(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, const W4Plan& p) {
  const int mb = (m - 1) / 16 + 1, rows = (m + 7) / 8 * 8, octets = 16 * w.blocks, chunks = (octets - 1) / kSplitOctets + 1;
  SkinnyKernel kern = nullptr;
#define BCH_W4(MB, T) if (mb == MB && p.t == T) kern = by_group<MB, T>(w.group);
  BCH_W4(1, 1) BCH_W4(1, 2) BCH_W4(1, 3) BCH_W4(1, 4) BCH_W4(2, 1) BCH_W4(2, 2) BCH_W4(2, 3) BCH_W4(2, 4)
  BCH_W4(3, 1) BCH_W4(3, 2) BCH_W4(3, 3) BCH_W4(4, 1) BCH_W4(4, 2) BCH_W4(4, 3)
#undef BCH_W4
  if (!kern) return hipErrorInvalidValue;
  u32x4* parts = static_cast<u32x4*>(ws);
  unsigned* big = reinterpret_cast<unsigned*>(parts + 3LL * octets * rows);
  const bool vec = w4_vec(w, x, ldx);
  hipLaunchKernelGGL(w4_split_few_kernel, dim3(chunks, rows / 8), dim3(kSplitThreads), 0, s, m, w.k, octets, rows, x, ldx, vec, parts, big);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int groups = (w.tiles - 1) / p.t + 1, per = (w.blocks - 1) / p.slices + 1, slices = (w.blocks - 1) / per + 1;
  const int bytes = kWaves * p.t * mb * 1024;
  float* partial = slices > 1 ? reinterpret_cast<float*>(static_cast<char*>(ws) + few_bytes(m, w)) : nullptr;
  e = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3(groups * slices), dim3(kThreads), bytes, s, w, m, rows, octets, parts, big, x, ldx, vec, bias, act, y,
                     ldy, groups, per, partial);
  e = hipGetLastError();
  if (e != hipSuccess || slices == 1) return e;
  return launch_w4_reduce(s, m, w.n, slices, partial, bias, act, y, ldy);
}

}  // namespace bch
