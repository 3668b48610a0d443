// w4.h -- linear layers whose weights have 4 bits and a scale and a zero point for each group of inputs, as the kernels
// see them: W[o][i] = scale[o][i / group] * (code[o][i] - zero[o][i / group]).
//
// The packed weights lie as a 16 x 32 operand of the matrix cores is held: by 16 outputs and 128 inputs a block of 1 KB, of
// which lane l's 16 bytes are output l % 16; their word j holds inputs 32 j + 8 (l / 16) .. + 7 of the block, input e of them in
// the bits from 4 (e / 2 + 4 (e % 2)) on, so that two neighbours come out of one mask in the two halves of a register.  A wavefront
// reads a block as 1024 consecutive bytes, every 32 inputs of one group together.  Behind the blocks lie the scales and
// behind those the zero points, [outputs / 16][groups][16].  Outputs and inputs beyond the layer's are codes equal to their
// zero point; their groups have scale 0.
#pragma once
#include "bch_internal.h"

namespace bch {

struct W4 {
  int n, k, group;
  int tiles, blocks, groups;  // of 16 outputs, of 128 inputs, of `group` inputs (those of the blocks)
  const u32x4* codes;
  const float* scale;
  const unsigned char* zero;
  unsigned mul;  // of an exact division by group / 32: group of inputs 32 c .. 32 c + 31 = (c * mul) >> shift
  int shift;
};

inline W4 w4_of(int n, int k, int group, const void* data) {
  W4 w;
  w.n = n;
  w.k = k;
  w.group = group;
  w.tiles = (n - 1) / 16 + 1;
  w.blocks = (k - 1) / 128 + 1;
  w.groups = (int)((128LL * w.blocks - 1) / group) + 1;
  const char* p = static_cast<const char*>(data);
  w.codes = reinterpret_cast<const u32x4*>(p);
  w.scale = reinterpret_cast<const float*>(p + 1024LL * w.tiles * w.blocks);
  w.zero = reinterpret_cast<const unsigned char*>(w.scale + 16LL * w.tiles * w.groups);
  // 2^l >= d: mul exceeds 2^(31 + l) / d by less than 1, so c mul / 2^(31 + l) exceeds c / d by less than 1 / d for c < 2^31
  const int d = group / 32;
  int l = 0;
  while ((1LL << l) < d) ++l;
  w.shift = 31 + l;
  w.mul = (unsigned)(((1ULL << w.shift) + d - 1) / d);
  return w;
}
inline size_t w4_bytes(int n, int k, int group) {
  const W4 w = w4_of(n, k, group, nullptr);
  return 1024ULL * w.tiles * w.blocks + 80ULL * w.tiles * w.groups;
}

__device__ __forceinline__ int w4_group(const W4& w, int c) { return (int)(((unsigned long long)(unsigned)c * w.mul) >> w.shift); }

// ---- codes and inputs as the bf16 matrix cores take them ----
// A code alone in the low bits of an f16 is code * 2^-24 (four bits higher up, 16 times that): one packed f16 multiplication and
// addition makes two of them (code - zero) * 2^-11, exactly.  Three bits down, its exponent (4 to 7, or 0) and mantissa are
// a bf16's.  The sign comes from where it was, and with it bit 12, where the shift leaves the sign: there it is 1 for those
// exponents and 0 for 0, so the bf16 is (code - zero) * 2^-91 in every case.  17 operations take eight codes apart;
// converting bytes to f32, subtracting and packing takes 23 (2048 rows of 4096 -> 11008: 479 and 494 us).
// Codes as bf16 below its smallest normal number would take 9 to 11 (sign and magnitude are what a packed f16 addition of such numbers
// leaves), but the matrix cores add their products as if each magnitude began at bit 7: up to three bits of a small
// code's are lost.
constexpr int kW4Unit = 91;  // a sum of products with such weights is 2^-91 of what it stands for

__device__ __forceinline__ unsigned w4_fma(unsigned a, unsigned b, unsigned c) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b),
                                                                __builtin_bit_cast(f16x2, c)));
}
// Two f16 of -zero * 2^-11.
__device__ __forceinline__ unsigned w4_zero(unsigned char z) {
  return w4_fma(0x80008000u | (unsigned)z * 0x00010001u, 0x70007000u, 0u);
}
__device__ __forceinline__ u32x4 w4_decode(unsigned c, unsigned zero) {
  constexpr unsigned k13 = 0x70007000u, k9 = 0x60006000u;  // two f16 of 2^13, of 2^9
  const unsigned d = c >> 8;
  const unsigned h[4] = {w4_fma(c & 0x000f000fu, k13, zero), w4_fma(c & 0x00f000f0u, k9, zero), w4_fma(d & 0x000f000fu, k13, zero),
                         w4_fma(d & 0x00f000f0u, k9, zero)};
  unsigned mask = 0x90009000u;
  asm("" : "+s"(mask));  // (not a constant to the compiler, which would take more operations for one)
  u32x4 v;
#pragma unroll
  for (int s = 0; s < 4; ++s) v[s] = (mask & h[s]) | (~mask & (h[s] >> 3));
  return v;
}

// Eight inputs times 2^e as three bf16 parts, x = x0 + x1 + x2 exactly (split8 of bch_internal.h).  An infinity or NaN is its first part alone (the differences that are NaN
// become 0: med3 of them and 0 is the least number), so that it gives what it gives in f32.
__device__ __forceinline__ void w4_split(const float (&v)[8], int e, u32x4 (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = ldexpf(v[2 * i], e), b = ldexpf(v[2 * i + 1], e);
    p[0][i] = bf16_pack(a, b);
    a -= __builtin_bit_cast(float, p[0][i] << 16);
    b -= __builtin_bit_cast(float, p[0][i] & 0xffff0000u);
    asm("v_med3_f32 %0, %0, %0, 0" : "+v"(a));
    asm("v_med3_f32 %0, %0, %0, 0" : "+v"(b));
    p[1][i] = bf16_pack(a, b);
    a -= __builtin_bit_cast(float, p[1][i] << 16);
    b -= __builtin_bit_cast(float, p[1][i] & 0xffff0000u);
    p[2][i] = bf16_pack(a, b);
  }
}
// Inputs i0 .. i0 + 7 of a row of k; vec: k and the rows are multiples of 4 floats, 16-byte aligned.
__device__ __forceinline__ void w4_load8(float (&v)[8], const float* row, int i0, int k, bool vec) {
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
// The magnitude's bits of the largest finite of them and `top`.
__device__ __forceinline__ unsigned w4_top(const float (&v)[8], unsigned top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned b = __builtin_bit_cast(unsigned, v[e]) & 0x7fffffffu;
    if (b < 0x7f800000u) top = max(top, b);
  }
  return top;
}
// The e of a row whose largest value has these bits: all below 2^kW4Top, as high as bf16 reaches, so that values far below the largest
// keep their bits (all of them from 2^-160 of it on: a product's last lies 114 below its value, f32's at 2^-149).  Not beyond
// kW4Unit: sums then never exceed what they stand for, and f32 holds them wherever it holds that.
constexpr int kW4Top = 127;
__device__ __forceinline__ int w4_exponent(unsigned top) { return min(kW4Unit, kW4Top + 126 - (int)(top >> 23)); }
inline bool w4_vec(const W4& w, const float* x, long long ldx) {
  return w.k % 4 == 0 && ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

// codes [n][ld bytes], input i in the low (even i) or high half of byte i / 2; scale and zero [n][groups of k], zero
// null: 8.
hipError_t launch_w4_pack(hipStream_t s, const W4& w, const unsigned char* codes, long long ld, const float* scale,
                          const unsigned char* zero, void* out);

// y[m][n] = act(x W^T + bias); bias nullable, act as launch_sgemm_ex.  ws: w4_linear_workspace_bytes, or less, with which it runs
// slower.
hipError_t launch_w4_linear(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, size_t ws_bytes);
size_t w4_linear_workspace_bytes(int m, const W4& w);

// ---- its kernels ----
struct W4Plan {
  int t, slices;  // tiles of 16 outputs a workgroup (few rows), slices that the inputs are cut into
  double cost;    // us
};
// One or two rows (w4_skinny.hip), no scratch.
hipError_t launch_w4_line(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy);
// Up to kW4Few rows (w4_skinny.hip).
constexpr int kW4Few = 64;
W4Plan w4_skinny_plan(int m, const W4& w, int cus, bool may_split);
size_t w4_skinny_bytes(int m, const W4& w, const W4Plan& p);
hipError_t launch_w4_skinny(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, const W4Plan& p);
// Any (w4_tile.hip).
W4Plan w4_tile_plan(int m, const W4& w, int cus, bool may_split);
size_t w4_parts_bytes(int m, const W4& w);
size_t w4_tile_bytes(int m, const W4& w, const W4Plan& p);
hipError_t launch_w4_tile(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy, void* ws, const W4Plan& p);
// y = act(the slices' partial sums [slices][m][n], in their order, + bias).
hipError_t launch_w4_reduce(hipStream_t s, int m, int n, int slices, const float* partial, const float* bias, int act, float* y,
                            long long ldy);

}  // namespace bch
