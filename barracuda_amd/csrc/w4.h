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
  return w;
}
inline size_t w4_bytes(int n, int k, int group) {
  const W4 w = w4_of(n, k, group, nullptr);
  return 1024ULL * w.tiles * w.blocks + 80ULL * w.tiles * w.groups;
}

// codes [n][ld bytes], input i in the low (even i) or high half of byte i / 2; scale and zero [n][groups of k], zero
// null: 8.
hipError_t launch_w4_pack(hipStream_t s, const W4& w, const unsigned char* codes, long long ld, const float* scale,
                          const unsigned char* zero, void* out);

// y[m][n] = act(x W^T + bias); bias nullable, act as launch_sgemm_ex.
hipError_t launch_w4_linear(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                            float* y, long long ldy, void* ws, size_t ws_bytes);
size_t w4_linear_workspace_bytes(int m, const W4& w);


// More rows, on the matrix cores (w4_tile.hip): ws holds w4_parts_bytes(m, w).
size_t w4_parts_bytes(int m, const W4& w);
hipError_t launch_w4_tile(hipStream_t s, int m, const W4& w, const float* x, long long ldx, const float* bias, int act,
                          float* y, long long ldy, void* ws);

}  // namespace bch
