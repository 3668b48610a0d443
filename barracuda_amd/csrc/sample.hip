// sample.hip -- a token for each row of logits: temperature, top-k, top-p, min-p, and the draw from given numbers.  The
// reference ends at the softmax; this stands beside it for programs that generate.
//
// With m a row's largest logit a token weighs w = exp((x - m) / temperature).  In the order of descending logits (equal ones by
// ascending index) top_k leaves the first k; top_p of these the shortest beginning that holds that part of their
// weight; min_p of these the ones with w >= min_p.  The token is the first in index order whose cumulative weight
// exceeds u times all that is left.
//
// Weights are whole numbers of 2^-U (2^-44 for 131072 tokens; 62 bits hold their sum): from 64-bit arithmetic, rounded once.  Sums of
// them are exact, so neither the order in which threads add nor how a row is cut up changes a choice, and the
// roundings move a border by 2^-45 of the largest weight a token.  What is below half of 2^-U is never drawn.
#include "sample.h"

#include <algorithm>

namespace {

using bch::SampleCall;
using bch::SampleRule;
typedef unsigned long long u64;

// ---- order and weight of a logit ----

// NaN counts as -inf, -0 as 0.
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
// Ascending with x.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(unsigned key) {
  return __builtin_bit_cast(float, key ^ ((int)key < 0 ? 0x80000000u : 0xffffffffu));
}
constexpr unsigned kNothing = 0x007fffffu;  // key_of(-inf)

struct Scale {
  float m;        // the row's largest logit
  double per;     // log2(e) / temperature
  double min_p;
  int unit_log;   // U
};
// 2^-t for t = (m - x) per: the whole part of t is an exponent, the rest, within 1/2, goes through the series of exp to the
// eleventh power (off by 2^-47).  A token of an infinite distance weighs nothing.
__device__ __forceinline__ double weight_of(const Scale& s, float x) {
  const double d = x == s.m ? 0.0 : (double)s.m - (double)x, t = d * s.per;
  if (!(t < 64.0)) return 0.0;
  const double n = rint(t), r = (n - t) * 0.69314718055994530942;
  double p = fma(r, 2.50521083854417187751e-08, 2.75573192239858906526e-07);
  p = fma(r, p, 2.75573192239858906526e-06);
  p = fma(r, p, 2.48015873015873015873e-05);
  p = fma(r, p, 1.98412698412698412698e-04);
  p = fma(r, p, 1.38888888888888888889e-03);
  p = fma(r, p, 8.33333333333333333333e-03);
  p = fma(r, p, 4.16666666666666666667e-02);
  p = fma(r, p, 1.66666666666666666667e-01);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return ldexp(p, -(int)n);
}
// In units: 2^52 is added, which leaves the whole number in the low bits (U <= 51).
__device__ __forceinline__ u64 units(const Scale& s, double w) {
  return __builtin_bit_cast(u64, ldexp(w, s.unit_log) + 0x1p52) - 0x4330000000000000ull;
}

// ---- sums over a workgroup ----
constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

struct Cut {
  unsigned key;  // tokens above it stay,
  unsigned ties; // and of those on it the first so many
};

struct Shared {
  u64 weight[kBins];
  unsigned count[kBins];
  u64 sums[2][kWaves];
  u64 found[4];
  int bin;
};

// Exclusive sums of a and b over the threads, and their totals.
__device__ __forceinline__ void block_scan(Shared& s, u64& a, u64& b, u64& all_a, u64& all_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 ia = wave_scan(a, lane), ib = wave_scan(b, lane);
  __syncthreads();
  if (lane == 63) {
    s.sums[0][wave] = ia;
    s.sums[1][wave] = ib;
  }
  __syncthreads();
  u64 ba = 0, bb = 0;
  all_a = all_b = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) {
      ba = all_a;
      bb = all_b;
    }
    all_a += s.sums[0][w];
    all_b += s.sums[1][w];
  }
  a = ba + ia - a;
  b = bb + ib - b;
}

// The cut behind the shortest beginning of the order that holds `target` tokens (BY_COUNT), or units of weight: the key's digits
// from the top, each by a histogram of the tokens that share the digits before it.  total: the weight of what the search is in; the
// target is given for it by `aim`.  Returns the weight that the cut leaves.
template <bool BY_COUNT, typename Aim>
__device__ u64 find_cut(Shared& s, const float* row, int vocab, const Scale& sc, Aim aim, Cut& cut) {
  unsigned prefix = 0;
  u64 target = 0, above_weight = 0, tie_weight = 0;
  constexpr int kShift[4] = {32, 21, 10, 0};
#pragma unroll
  for (int level = 0; level < 3; ++level) {
    const int shift = kShift[level + 1], bins = 1 << (kShift[level] - shift);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) {
      s.weight[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const float x = clean(row[i]);
      const unsigned key = key_of(x);
      if (level > 0 && key >> kShift[level] != prefix) continue;
      const int b = (key >> shift) & (bins - 1);
      atomicAdd(&s.count[b], 1u);
      const u64 w = units(sc, weight_of(sc, x));
      if (w) atomicAdd(&s.weight[b], w);
    }
    __syncthreads();
    // from the top: thread t has the bins below bins - 1 - per t
    const int per = bins / kThreads, hi = bins - 1 - per * (int)threadIdx.x;
    u64 c = 0, w = 0;
    for (int b = hi; b > hi - per; --b) {
      c += s.count[b];
      w += s.weight[b];
    }
    u64 all_c, all_w;
    block_scan(s, c, w, all_c, all_w);
    if (level == 0) target = aim(all_w);
    for (int b = hi; b > hi - per; --b) {
      const u64 before = BY_COUNT ? c : w, in = BY_COUNT ? s.count[b] : s.weight[b];
      if (before < target && target <= before + in) {
        s.bin = b;
        s.found[0] = before;
        s.found[1] = w;
        s.found[2] = s.count[b];
        s.found[3] = s.weight[b];
      }
      c += s.count[b];
      w += s.weight[b];
    }
    __syncthreads();
    prefix = level == 0 ? s.bin : (prefix << (kShift[level] - shift)) | s.bin;
    target -= s.found[0];
    above_weight += s.found[1];
    tie_weight = s.found[2] ? s.found[3] / s.found[2] : 0;
  }
  cut.key = prefix;
  cut.ties = BY_COUNT ? (unsigned)target : (unsigned)((target + tie_weight - 1) / tie_weight);
  return above_weight + cut.ties * tie_weight;
}

// ---- one workgroup a row ----
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleCall c) {
  __shared__ Shared s;
  const long long r = blockIdx.x;
  const float* row = c.logits + r * c.stride;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the largest logit, of equal ones the lowest index
  u64 top = 0;
  for (int i = threadIdx.x; i < c.vocab; i += kThreads)
    top = max(top, (u64)key_of(clean(row[i])) << 32 | (0xffffffffu - (unsigned)i));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max(top, __shfl_xor(top, d));
  if (lane == 0) s.sums[0][wave] = top;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) top = max(top, s.sums[0][w]);
  const unsigned top_key = (unsigned)(top >> 32);
  const bool nothing = top_key == kNothing, one = !(rule.temperature > 0.0f) || rule.top_k == 1 || rule.top_p <= 0.0f;
  if (nothing || one) {
    if (threadIdx.x == 0) {
      c.tokens[r] = nothing ? -1 : (int)(0xffffffffu - (unsigned)top);
      if (c.probs) c.probs[r] = nothing ? 0.0f : 1.0f;
    }
    return;
  }
  const Scale sc{logit_of(top_key), 1.44269504088896340736 / (double)rule.temperature,
                 rule.min_p > 0.0f ? fmin((double)rule.min_p, 1.0) : 0.0, c.unit_log};
  Cut cut{0, 0};
  u64 left = 0;
  const bool by_count = rule.top_k > 0 && rule.top_k < c.vocab;
  if (by_count) left = find_cut<true>(s, row, c.vocab, sc, [&](u64) { return (u64)rule.top_k; }, cut);
  if (rule.top_p < 1.0f)
    find_cut<false>(s, row, c.vocab, sc,
                    [&](u64 all) {
                      const u64 of = by_count ? left : all;
                      return min(of, max((u64)1, (u64)ceil((double)rule.top_p * (double)of)));
                    },
                    cut);
  // the draw: the part of the row that the target falls into, sixteen times smaller each time
  u64 target = 0, whole = 0;
  unsigned ties = 0;  // on the cut, before the part
  int lo = 0, hi = c.vocab;
  for (bool first = true; first || hi - lo > 64; first = false) {
    const int per = ((hi - lo - 1) / kThreads + 1) * 64, a = (int)min((long long)hi, lo + (long long)per * wave),
              b = (int)min((long long)hi, (long long)a + per);
    u64 sum = 0;
    unsigned on = 0;
    double tie = 0.0;
    for (int i = a + lane; i < b; i += 64) {
      const float x = clean(row[i]);
      const unsigned key = key_of(x);
      if (key < cut.key) continue;
      if (key == cut.key) {
        ++on;
      } else {
        const double w = weight_of(sc, x);
        if (w >= sc.min_p) sum += units(sc, w);
      }
    }
    tie = weight_of(sc, logit_of(cut.key));
    const u64 tie_weight = cut.ties && tie >= sc.min_p ? units(sc, tie) : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      sum += __shfl_xor(sum, d);
      on += __shfl_xor(on, d);
    }
    __syncthreads();
    if (lane == 0) {
      s.sums[0][wave] = sum;
      s.sums[1][wave] = on;
    }
    __syncthreads();
    u64 part[kWaves];
    unsigned before[kWaves + 1];
    before[0] = ties;
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const unsigned n = (unsigned)s.sums[1][w];
      const unsigned keep = cut.ties > before[w] ? min(n, cut.ties - before[w]) : 0;
      before[w + 1] = before[w] + n;
      part[w] = s.sums[0][w] + keep * tie_weight;
      all += part[w];
    }
    if (first) {
      whole = all;
      const double u = c.u[r];  // NaN counts as 0
      target = u > 0.0 ? (u64)(fmin(u, 1.0) * (double)whole) : 0;
      target = min(target, whole - 1);
    }
    int pick = 0;
    bool found = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (!found && target < part[w]) {
        pick = w;
        found = true;
      }
      if (!found) target -= part[w];
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (w == pick) ties = before[w];
    const int from = (int)min((long long)hi, lo + (long long)per * pick);
    hi = (int)min((long long)hi, (long long)from + per);
    lo = from;
  }
  if (wave == 0) {
    const int i = lo + lane;
    u64 w = 0;
    bool on = false;
    float x = 0.0f;
    if (i < hi) {
      x = clean(row[i]);
      on = key_of(x) == cut.key;
    }
    const u64 mask = __ballot(on);
    const unsigned rank = ties + (unsigned)__popcll(mask & ((1ull << lane) - 1));
    if (i < hi && (key_of(x) > cut.key || (on && rank < cut.ties))) {
      const double v = weight_of(sc, x);
      if (v >= sc.min_p) w = units(sc, v);
    }
    const u64 run = wave_scan(w, lane);
    const u64 beyond = __ballot(run > target);
    if (beyond && lane == __ffsll(beyond) - 1) {
      c.tokens[r] = i;
      if (c.probs) c.probs[r] = (float)((double)w / (double)whole);
    }
  }
}

}  // namespace

namespace bch {

int sample_unit_log(int vocab) {
  int bits = 1;
  while (bits < 31 && (1LL << bits) <= vocab) ++bits;
  return std::min(51, 62 - bits);
}

size_t sample_workspace_bytes(const SampleCall&) { return 0; }

hipError_t launch_sample(hipStream_t s, const SampleCall& call, int rows, void* ws, size_t ws_bytes) {
  constexpr int kMost = 1 << 21;
  for (int at = 0; at < rows; at += kMost) {
    SampleCall c = call;
    c.logits += at * call.stride;
    if (c.rules) c.rules += at;
    c.u += at;
    c.tokens += at;
    if (c.probs) c.probs += at;
    hipLaunchKernelGGL(sample_row_kernel, dim3((unsigned)std::min(kMost, rows - at)), dim3(kThreads), 0, s, c);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace bch
