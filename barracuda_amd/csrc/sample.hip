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
// roundings move a border by 2^-45 of the largest weight a token.  What is below half of 2^-U is never drawn.  (The whole
// weight of a row of which nothing but top_p, or nothing at all, leaves some is added up from spans of 512 logits, whole
// numbers of 2^-51 of each span's largest, and rows that nothing cuts are drawn from these: the same spans and order for every
// row of that length, whichever kernels take it.)
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
#pragma clang fp contract(off)  // (the same bits wherever it is inlined)
  const double d = x == s.m ? 0.0 : (double)s.m - (double)x, t = d * s.per;
  if (!(t < 64.0)) return 0.0;
  const double n = rint(t), r = fma(-d, s.per, n) * 0.69314718055994530942;
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
// A key below which no token reaches min_p of the largest's weight (v_log_f32 is right to 2^-20 here; what it may be off by is taken off
// many times over), or 0.
__device__ __forceinline__ unsigned least_key(const SampleRule& rule, const Scale& s) {
  const double t = -(double)__builtin_amdgcn_logf(rule.min_p), x = (double)s.m - (t + 1e-4 * (t + 1.0)) / s.per;
  return fabs(x) < 3e38 ? key_of((float)x - 1e-6f * fabsf((float)x)) - 1 : 0;
}
// In units: 2^52 is added, which leaves the whole number in the low bits (U <= 51).
__device__ __forceinline__ u64 units(const Scale& s, double w) {
  return __builtin_bit_cast(u64, ldexp(w, s.unit_log) + 0x1p52) - 0x4330000000000000ull;
}

// ---- sums over a workgroup ----
// A workgroup goes through most of its code once, and much of its time is the fetching of that code.  So what a thread has several
// of goes through loops in turn, with one copy of weight_of in each (16 rows of 50021 logits, 4900 of them finite, top_p 0.98: the
// last step took 25 us, and 48 with the loops unrolled and eight weights a thread in scratch memory).
constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {  // inclusive
#pragma unroll 1
  for (int d = 1; d < 64; d *= 2) {
    const u64 o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

typedef u64 Sums[2][kWaves];

// Exclusive sum of v over the threads, and the total.
__device__ __forceinline__ u64 block_scan(Sums& sums, u64 v, u64& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 in = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) sums[0][wave] = in;
  __syncthreads();
  u64 before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const u64 one = sums[0][w];
    before += w < wave ? one : 0;
    all += one;
  }
  return before + in - v;
}

// ---- rules ----

__device__ __forceinline__ bool one_token(const SampleRule& rule) {
  return !(rule.temperature > 0.0f) || rule.top_k == 1 || rule.top_p <= 0.0f;
}
__device__ __forceinline__ bool by_count(const SampleRule& rule, int vocab) { return rule.top_k > 0 && rule.top_k < vocab; }
__device__ __forceinline__ bool by_weight(const SampleRule& rule) { return rule.top_p < 1.0f; }
__device__ __forceinline__ Scale scale_of(const SampleCall& c, const SampleRule& rule, float m) {
  return {m, 1.44269504088896340736 / (double)rule.temperature, rule.min_p > 0.0f ? fmin((double)rule.min_p, 1.0) : 0.0,
          c.unit_log};
}
// The part of `whole` that u is.  NaN counts as 0.
__device__ __forceinline__ double draw_at(const SampleCall& c, long long r, double whole) {
  const double u = c.u[r];
  return u > 0.0 ? fmin(u, 1.0) * whole : 0.0;
}
__device__ __forceinline__ u64 draw_units(const SampleCall& c, long long r, u64 whole) {
  return min((u64)draw_at(c, r, (double)whole), whole - 1);
}
// The weight that top_p asks for of `of` units.
__device__ __forceinline__ u64 part_units(const SampleRule& rule, double of) {
  return max((u64)1, (u64)ceil((double)rule.top_p * of));
}
__device__ __forceinline__ void answer(const SampleCall& c, long long r, int token, double prob) {
  c.tokens[r] = token;
  if (c.probs) c.probs[r] = (float)prob;
}

// ---- a row by one workgroup, whatever its rule and its logits ----
struct Cut {
  unsigned key;  // tokens above it stay,
  unsigned ties; // and of those on it the first so many
};

struct General {
  u64 weight[kBins];
  unsigned count[kBins];
  u64 found[4];
  int bin;
};

// The cut behind the shortest beginning of the order that holds `target` tokens (BY_COUNT), or units of weight: the key's digits
// from the top, each by a histogram of the tokens that share the digits before it.  total: the weight of what the search is in; the
// target is given for it by `aim`.  Returns the weight that the cut leaves.
template <bool BY_COUNT, typename Aim>
__device__ u64 find_cut(General& s, Sums& sums, const float* row, int vocab, const Scale& sc, Aim aim, Cut& cut) {
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
    c = block_scan(sums, c, all_c);
    w = block_scan(sums, w, all_w);
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

// For a rule that leaves more than one token, and not all.  whole_row: the row's weight in units, where only a weight cuts.
__device__ void general_row(General& s, Sums& sums, const SampleCall& c, long long r, const SampleRule& rule, const Scale& sc,
                            double whole_row) {
  const float* row = c.logits + r * c.stride;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Cut cut{0, 0};
  u64 left = 0;
  const bool count_cut = by_count(rule, c.vocab);
  if (count_cut) left = find_cut<true>(s, sums, row, c.vocab, sc, [&](u64) { return (u64)rule.top_k; }, cut);
  if (by_weight(rule))
    find_cut<false>(s, sums, row, c.vocab, sc,
                    [&](u64 all) {
                      return min(count_cut ? left : all, part_units(rule, count_cut ? (double)left : whole_row));
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
      sums[0][wave] = sum;
      sums[1][wave] = on;
    }
    __syncthreads();
    u64 part[kWaves];
    unsigned before[kWaves + 1];
    before[0] = ties;
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const unsigned n = (unsigned)sums[1][w];
      const unsigned keep = cut.ties > before[w] ? min(n, cut.ties - before[w]) : 0;
      before[w + 1] = before[w] + n;
      part[w] = sums[0][w] + keep * tie_weight;
      all += part[w];
    }
    if (first) {
      whole = all;
      target = draw_units(c, r, whole);
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
      answer(c, r, i, (double)w / (double)whole);
    }
  }
}

// ---- the same from the largest logits of every 512 ----
// Most rules leave few tokens of many.  A wavefront takes 512 logits, read once: it notes its largest, what its weights add up to
// against that (where the rule needs it), and a list of its largest: those from its lanes' R-th largest maximum on.  All of the
// row's tokens from the largest such bound of any wavefront on (`tau`) then are on lists, and where the rule's cuts are found
// among them, they alone decide.  Where they are not, the rows of the next section go on there and others (thousands of equal
// logits, more than 32 of a top_k's tokens in one span) to general_row.
// What bounds it (64 rows of 131072): the lists 15.5 us, some 350 vector operations a 512 logits, 80% of the
// cycles, where the stream takes 6; the choice 8 us a row for tens of entries, 12 to 20 for some hundreds, exchanges between wavefronts and trips to memory one behind the other.
constexpr int kSpan = 512, kListMost = 128, kListedMost = 2048;
constexpr int kSpanUnit = 51;  // 512 weights in units of 2^-51 stay below 2^61

struct Record {
  unsigned top, tau;  // keys; tau 0xffffffff: the list is not whole
  int count, first;   // of the list; the lowest index of the largest
  u64 weight;
};

// Does the top_k-th largest of the spans' largest logits bound the row's top_k largest?
constexpr int kTopsMost = 512;
__device__ __forceinline__ bool tops_tell(const SampleRule& rule, int vocab, int spans) {
  return by_count(rule, vocab) && rule.top_k < spans && spans <= kTopsMost;
}
// How many of a wavefront's lanes are to hold a token from tau on: top_k where the spans' largest bound what is taken of them (so
// up to 32 of the row's top_k may lie in one span); else the largest of the wavefronts' bounds leaves a good deal more than top_k
// tokens of the row, or, where there is no top_k, 1000 to 1500 of any number of spans (of independent logits; more than kListedMost
// would be of no use).
__device__ __forceinline__ int list_rank(const SampleRule& rule, int vocab, int spans) {
  if (one_token(rule)) return 1;
  if (tops_tell(rule, vocab, spans)) return min(32, max(8, rule.top_k));
  if (by_count(rule, vocab)) return (int)min(48LL, 5 + (4LL * rule.top_k + spans - 1) / spans);
  return min(32, max(4, (int)(192.0f * __builtin_amdgcn_rsqf((float)spans))));
}
__device__ __forceinline__ bool needs_whole(const SampleRule& rule, int vocab) {
  return !one_token(rule) && !by_count(rule, vocab) && (by_weight(rule) || !(rule.min_p > 0.0f));
}

// f of each of eight values, one copy of it.
template <typename F>
__device__ __forceinline__ void each(const float (&x)[8], F f) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x[e];
#pragma unroll 1
  for (int n = 0; n < 8; ++n) {
    f(y[0]);
#pragma unroll
    for (int e = 0; e < 7; ++e) y[e] = y[e + 1];
  }
}

// Four logits from index i on, wherever they lie (16-byte loads need 4-byte alignment); -inf behind the last.
__device__ __forceinline__ void load_four(const SampleCall& c, const float* row, int i, float* x) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  if (i + 3 < c.vocab) {
    const f32x4_any t = *reinterpret_cast<const f32x4_any*>(row + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = clean(t[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = row[min(i + e, c.vocab - 1)];
      x[e] = i + e < c.vocab ? clean(t) : -INFINITY;
    }
  }
}
// The logits of a span: this lane's 4 lane .. + 3 and 256 + 4 lane .. + 3.
__device__ __forceinline__ void load_span(const SampleCall& c, const float* row, int base, float (&x)[8]) {
  const int lane = threadIdx.x & 63;
  load_four(c, row, base + 4 * lane, x);
  load_four(c, row, base + 256 + 4 * lane, x + 4);
}
__device__ __forceinline__ void load_eight(const SampleCall& c, const float* row, int i, float (&x)[8]) {
  load_four(c, row, i, x);
  load_four(c, row, i + 4, x + 4);
}
__device__ __forceinline__ int span_index(int base, int e) {
  return base + 256 * (e / 4) + 4 * (int)(threadIdx.x & 63) + e % 4;
}

// What the logits of a wavefront's span, the largest of them `top`, weigh against that one, in units of 2^-kSpanUnit.
template <bool MANY>
__device__ __forceinline__ u64 weigh(const SampleCall& c, const SampleRule& rule, const float (&x)[8], unsigned top) {
  Scale sc = scale_of(c, rule, logit_of(top));
  sc.unit_log = kSpanUnit;
  u64 sum = 0;
  if constexpr (MANY) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += units(sc, weight_of(sc, x[e]));
  } else {
    each(x, [&](float v) { sum += units(sc, weight_of(sc, v)); });
  }
#pragma unroll 1
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  return sum;
}
// The largest logit and the weight of span `at`, by one wavefront, where no record holds them.
__device__ __forceinline__ Record weigh_span(const SampleCall& c, const float* row, const SampleRule& rule, int at) {
  float x[8];
  load_span(c, row, at * kSpan, x);
  unsigned mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) mine = max(mine, key_of(x[e]));
  Record q{};
  q.top = key_of(bch::wave_allreduce(logit_of(mine), bch::OpMax()));
  if (q.top != kNothing) q.weight = weigh<true>(c, rule, x, q.top);
  return q;
}
// A span's weight against the row's largest logit, in units of 2^-kSpanUnit.
__device__ __forceinline__ double span_weight(const Scale& s, const Record& q) {
#pragma clang fp contract(off)
  return q.top == kNothing ? 0.0 : (double)q.weight * weight_of(s, logit_of(q.top));
}

// Span `at` of a row, by one wavefront: its record, and its list (keys in the upper half, 2^32 - 1 - index in the lower).
// MANY: a launch of many wavefronts, whose code is fetched once for all of them: its weights without a loop.
template <bool MANY>
__device__ __forceinline__ void list_span(const SampleCall& c, const float* row, const SampleRule& rule, int spans, int at,
                                          Record* record, u64* list) {
  const int lane = threadIdx.x & 63, base = at * kSpan;
  float x[8];
  load_span(c, row, base, x);
  unsigned key[8], mine = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    key[e] = key_of(x[e]);
    mine = max(mine, key[e]);
  }
  const unsigned top = key_of(bch::wave_allreduce(logit_of(mine), bch::OpMax()));
  int first = 0x7fffffff;
  if (one_token(rule)) {
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (key[e] == top) first = span_index(base, e);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
  }
  unsigned tau = top;
  int count = 0;
  if (!one_token(rule)) {
    // the R-th largest of the lanes' maxima, bit by bit (the upper half of them: a little below it is as good)
    const int rank = list_rank(rule, c.vocab, spans);
    tau = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; --bit) {
      const unsigned next = tau | 1u << bit;
      if (__popcll(__ballot(mine >= next)) >= rank) tau = next;
    }
    tau = max(tau, kNothing + 1);  // -inf is never chosen
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool on = key[e] >= tau;
      const u64 mask = __ballot(on);
      const int slot = count + __popcll(mask & ((1ull << lane) - 1));
      if (on && slot < kListMost) list[slot] = (u64)key[e] << 32 | (0xffffffffu - (unsigned)span_index(base, e));
      count += __popcll(mask);
    }
  }
  u64 sum = 0;
  if (needs_whole(rule, c.vocab) && top != kNothing) sum = weigh<MANY>(c, rule, x, top);
  if (lane == 0) *record = {top, count > kListMost ? 0xffffffffu : tau, min(count, kListMost), first, sum};
}

// Of lane ^ D, without LDS: exchanges, mirrors and a rotation within 16 lanes.
template <int D>
__device__ __forceinline__ unsigned across(unsigned v) {
  constexpr int kCtrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x128;
  v = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, true);
  if constexpr (D == 4) v = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x1B, 0xF, 0xF, true);  // (a mirror of 8, then of 4)
  return v;
}
template <int D>
__device__ __forceinline__ u64 across(u64 v) {
  return (u64)across<D>((unsigned)(v >> 32)) << 32 | across<D>((unsigned)v);
}

constexpr int kFew = kThreads / 4, kSlots = kThreads;
struct Lists {
  u64 entry[kListedMost], weight[kListedMost];
  u64 slot[kSlots];
  u64 few[kFew], few_value[kFew];
};
union Work {
  General general;
  Lists lists;
};
struct Common {
  Sums sums;
  int n, pick, large;
  unsigned least;
  double before;
  u64 want;
  u64 chunk[kThreads];
};

// The threads' sums of their spans' weights.  HELD: of records; else each thread's spans are weighed by a wavefront, in the same
// order.  spans_of(thread, i): that thread's i-th span, or -1.
template <bool HELD, typename Of>
__device__ __forceinline__ double thread_weight(Common& m, const SampleCall& c, const float* row, const SampleRule& rule, const Scale& sc,
                                                const Record* records, Of spans_of) {
#pragma clang fp contract(off)
  if constexpr (HELD) {
    double sum = 0.0;
    for (int i = 0, at; (at = spans_of((int)threadIdx.x, i)) >= 0; ++i) sum += span_weight(sc, records[at]);
    return sum;
  } else {
    for (int t = threadIdx.x >> 6; t < kThreads; t += kWaves) {
      double sum = 0.0;
      for (int i = 0, at; (at = spans_of(t, i)) >= 0; ++i) sum += span_weight(sc, weigh_span(c, row, rule, at));
      if ((threadIdx.x & 63) == 0) m.chunk[t] = __builtin_bit_cast(u64, sum);
    }
    __syncthreads();
    return __builtin_bit_cast(double, m.chunk[threadIdx.x]);
  }
}
// A row's weight in units.  (Behind a barrier since sums were read.)
template <bool HELD>
__device__ __forceinline__ double row_weight(Common& m, const SampleCall& c, const float* row, const SampleRule& rule, const Scale& sc,
                                             int spans, const Record* records) {
#pragma clang fp contract(off)
  double whole = thread_weight<HELD>(m, c, row, rule, sc, records, [&](int t, int i) {
    const long long at = t + (long long)kThreads * i;
    return at < spans ? (int)at : -1;
  });
#pragma unroll
  for (int d = 1; d < 64; d *= 2) whole += __shfl_xor(whole, d);
  if ((threadIdx.x & 63) == 0) m.sums[0][threadIdx.x >> 6] = __builtin_bit_cast(u64, whole);
  __syncthreads();
  whole = 0.0;
  for (int i = 0; i < kWaves; ++i) whole += __builtin_bit_cast(double, m.sums[0][i]);
  return ldexp(whole, c.unit_log - kSpanUnit);
}

// A row of which all tokens stay: the span that the target falls into, then the token in it.
template <bool HELD>
__device__ void draw_span(Common& m, const SampleCall& c, long long r, const SampleRule& rule, const Scale& sc, int spans,
                          const Record* records) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* row = c.logits + r * c.stride;
  // a thread's spans lie together; weights in units of 2^-kSpanUnit of the row's largest
  const int per = (spans - 1) / kThreads + 1;
  const double mine = thread_weight<HELD>(m, c, row, rule, sc, records, [&](int t, int i) {
    const long long at = (long long)per * t + i;
    return i < per && at < spans ? (int)at : -1;
  });
  double run = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  if (lane == 63) m.sums[0][wave] = __builtin_bit_cast(u64, run);
  if (threadIdx.x == 0) {
    m.pick = kThreads;
    m.n = 0;
  }
  __syncthreads();
  double whole = 0.0, before = 0.0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) before = whole;
    whole += __builtin_bit_cast(double, m.sums[0][w]);
  }
  run += before;
  const double target = draw_at(c, r, whole);
  // the first thread whose spans end beyond the target; of a target at the end (sums in other orders may fall short of it), the
  // last with any weight
  if (mine > 0.0 && run > target) atomicMin(&m.pick, (int)threadIdx.x);
  if (mine > 0.0) atomicMax(&m.n, (int)threadIdx.x);
  __syncthreads();
  const int chosen = m.pick < kThreads ? m.pick : m.n;
  if ((int)threadIdx.x == chosen) m.before = run - mine;
  __syncthreads();
  if (wave > 0) return;
  auto span = [&](int i) {
    if constexpr (HELD)
      return records[i];
    else
      return weigh_span(c, row, rule, i);
  };
  const int lo = per * chosen, hi = (int)min((long long)spans, (long long)lo + per);
  double at = m.before;
  int i = lo, last = lo;
  for (; i < hi; ++i) {
    const double w = span_weight(sc, span(i));
    if (w > 0.0) last = i;
    if (at + w > target) break;
    at += w;
  }
  if (i == hi) {
    i = last;
    at -= span_weight(sc, span(i));
  }
  const Record q = span(i);
  const double of = weight_of(sc, logit_of(q.top));
  u64 left = min((u64)fmax((target - at) / of, 0.0), q.weight - 1);
  Scale own = scale_of(c, rule, logit_of(q.top));
  own.unit_log = kSpanUnit;
  // eight tokens a lane, in index order
  float x[8];
  i = i * kSpan + 8 * lane;
  load_eight(c, row, i, x);
  u64 sum = 0;
  each(x, [&](float v) { sum += units(own, weight_of(own, v)); });
  left -= wave_scan(sum, lane) - sum;
  const u64 here = __ballot(left < sum);  // (what has become less than 0 is large)
  if (!here) return;
  // and of that lane's eight a lane one
  const int owner = __ffsll((long long)here) - 1;
  left = __shfl(left, owner);
  i = __shfl(i, owner) + lane;
  const u64 w = lane < 8 && i < c.vocab ? units(own, weight_of(own, clean(row[i]))) : 0, end = wave_scan(w, lane);
  if (left < end && left >= end - w) answer(c, r, i, (double)w * of / whole);
}

// The choice from all of a few tokens, without a sort: 4 to 16 threads a token compare it with the others.  Its place and the weight
// before it decide whether it stays, and the weight of the tokens with lower indexes whether it is drawn.  `whole`: the row's
// weight where only a weight cuts; complete: nothing else is in the row.  False if the tokens do not tell.
__device__ __forceinline__ int few_log(int n) { return n <= kThreads / 16 ? 4 : n <= kThreads / 8 ? 3 : n <= kThreads / 4 ? 2 : 1; }
template <typename T>
__device__ __forceinline__ T over_parts(T v, int log) {
  v += across<1>(v);
  if (log > 1) v += across<2>(v);
  if (log > 2) v += across<4>(v);
  if (log > 3) v += across<8>(v);
  return v;
}
__device__ __forceinline__ bool choose_few(Lists& lists, Common& m, const SampleCall& c, long long r, const SampleRule& rule,
                                           const Scale& sc, int n, double whole, bool complete) {
  const bool count_cut = by_count(rule, c.vocab), weight_cut = by_weight(rule);
  const int log = few_log(n), parts = 1 << log, i = threadIdx.x >> log, part = threadIdx.x & (parts - 1);
  if ((int)threadIdx.x < n) {
    const double real = weight_of(sc, logit_of((unsigned)(lists.entry[threadIdx.x] >> 32)));
    lists.weight[threadIdx.x] = units(sc, real);
    const int large = __popcll(__ballot(real >= sc.min_p));
    if ((threadIdx.x & 63) == 0) atomicAdd(&m.large, large);
  }
  __syncthreads();
  const int of = count_cut ? min(n, rule.top_k) : n;
  const u64 own = i < n ? lists.entry[i] : 0, weight = i < n ? lists.weight[i] : 0;
  unsigned place = 0;
  u64 before = 0;
  if (i < n) {
#pragma unroll 1
    for (int j = part; j < n; j += parts) {
      const u64 w = lists.weight[j];
      const bool above = lists.entry[j] > own;
      place += above;
      before += above ? w : 0;
    }
    place = over_parts(place, log);
    before = over_parts(before, log);
    if (part == 0 && (int)place == of - 1) m.want = before + weight;
  }
  __syncthreads();
  const u64 listed = m.want, target = part_units(rule, count_cut ? (double)listed : whole);
  const int large = sc.min_p > 0.0 ? m.large : n;
  const bool short_of_min = sc.min_p > 0.0 && (complete || large < n);
  if (count_cut ? !(complete || n >= rule.top_k) : !(short_of_min || (weight_cut && (complete || listed >= target)))) return false;
  const bool stays = i < n && (int)place < min(of, large) && (!weight_cut || before < target);
  if (part == 0 && i < n) lists.weight[i] = stays ? weight : 0;
  __syncthreads();
  u64 left = 0;
  before = 0;
  if (i < n) {
#pragma unroll 1
    for (int j = part; j < n; j += parts) {
      const u64 w = lists.weight[j];
      const unsigned low = (unsigned)lists.entry[j];
      left += w;
      before += low > (unsigned)own ? w : 0;
    }
    left = over_parts(left, log);
    before = over_parts(before, log);
    const u64 at = draw_units(c, r, left);
    if (part == 0 && stays && at >= before && at < before + weight)
      answer(c, r, (int)(0xffffffffu - (unsigned)own), (double)weight / (double)left);
  }
  return true;
}

// Of n entries those with fewer than k larger logits above them; how many that are.  Comparing keys alone, two operations a pair, it
// spares choose_few most of its pairs (191 entries, k = 40: a call of one row 16.1 -> 12.8 us).
constexpr int kKeysMost = kThreads / 2;
constexpr int kFewMost = 208;  // about where choose_few, whose time grows with the square, takes the 7 us of choose_many
__device__ __forceinline__ int largest_of(Lists& lists, Common& m, int n, int k) {
  unsigned* keys = reinterpret_cast<unsigned*>(lists.weight);
  const int log = few_log(n), parts = 1 << log, i = threadIdx.x >> log, part = threadIdx.x & (parts - 1);
  keys[threadIdx.x] = (int)threadIdx.x < n ? (unsigned)(lists.entry[threadIdx.x] >> 32) : 0;
  if (threadIdx.x == 0) m.pick = 0;
  __syncthreads();
  bool on = false;
  u64 own = 0;
  if (i < n) {
    own = lists.entry[i];
    const unsigned key = (unsigned)(own >> 32);
    int above = 0;
#pragma unroll 2
    for (int j = part; 4 * j < n; j += parts) {
      const uint4 q = reinterpret_cast<const uint4*>(keys)[j];
      above += (q.x > key) + (q.y > key) + (q.z > key) + (q.w > key);
    }
    on = over_parts((unsigned)above, log) < (unsigned)k && part == 0;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const u64 mask = __ballot(on);
  int slot = 0;
  if (lane == 0 && mask) slot = atomicAdd(&m.pick, __popcll(mask));
  slot = __shfl(slot, 0) + __popcll(mask & ((1ull << lane) - 1));
  if (on) lists.entry[slot] = own;
  __syncthreads();
  return m.pick;
}

// Entries in kSlots bins of their logits, evenly from the largest down; never descending with the logit, whatever the numbers.
struct Bins {
  float m, per, from;
};
__device__ __forceinline__ int slot_of(const Bins& b, u64 entry) {
  const float x = logit_of((unsigned)(entry >> 32));
  return x == b.m ? 0 : (int)fminf(fmaxf((b.m - x) * b.per - b.from, 0.0f), (float)(kSlots - 1));
}
// Of n entries with their weights those that are at least `floor`, in descending order: the one with which their weights (or, counts:
// their number) reach `target`, 0 if they do not.  The bins tell between which it lies, one bin's are compared with
// each other.  False if those are too many.
__device__ bool list_cut(Lists& lists, Common& m, const Bins& bins, int n, u64 floor, bool counts, u64 target, u64& last) {
  __syncthreads();
  lists.slot[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    m.pick = n <= kFew ? 0 : -1;  // few entries are one bin
    m.large = 0;
    m.want = target;
  }
  __syncthreads();
  if (n > kFew) {
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 e = lists.entry[i], w = counts ? 1 : lists.weight[i];
      if (e >= floor) atomicAdd(&lists.slot[slot_of(bins, e)], w);
    }
    __syncthreads();
    const u64 own = lists.slot[threadIdx.x];
    u64 all;
    const u64 before = block_scan(m.sums, own, all);
    if (before < target && before + own >= target) {
      m.pick = threadIdx.x;
      m.want = target - before;
    }
    __syncthreads();
  }
  const int at = m.pick;
  const u64 want = m.want;
  last = 0;
  if (at < 0) return true;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const u64 e = lists.entry[i];
    if (e >= floor && (n <= kFew || slot_of(bins, e) == at)) {
      const int to = atomicAdd(&m.large, 1);
      if (to < kFew) {
        lists.few[to] = e;
        lists.few_value[to] = counts ? 1 : lists.weight[i];
      }
    }
  }
  __syncthreads();
  const int few = m.large;
  if (few > kFew) return false;
  if (threadIdx.x == 0) m.want = 0;
  __syncthreads();
  const int log = few_log(few), parts = 1 << log, i = threadIdx.x >> log, part = threadIdx.x & (parts - 1);
  if (i < few) {
    const u64 mine = lists.few[i];
    u64 above = 0;
#pragma unroll 1
    for (int j = part; j < few; j += parts) {
      const u64 w = lists.few_value[j];
      above += lists.few[j] > mine ? w : 0;
    }
    above = over_parts(above, log);
    if (part == 0 && above < want && above + lists.few_value[i] >= want) m.want = mine;
  }
  __syncthreads();
  last = m.want;
  return true;
}
// The draw from the entries that are at least `last`: bins of their indexes tell between which it falls.
__device__ bool list_draw(Lists& lists, Common& m, const SampleCall& c, long long r, int n, u64 last) {
  const int shift = max(0, 22 - __clz(c.vocab - 1 | 1));  // kSlots parts of the row
  __syncthreads();
  lists.slot[threadIdx.x] = 0;
  if (threadIdx.x == 0) m.large = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const u64 e = lists.entry[i];
    if (e >= last) atomicAdd(&lists.slot[(0xffffffffu - (unsigned)e) >> shift], lists.weight[i]);
  }
  __syncthreads();
  const u64 own = lists.slot[threadIdx.x];
  u64 all;
  const u64 before = block_scan(m.sums, own, all), target = draw_units(c, r, all);
  if (target >= before && target < before + own) {
    m.pick = threadIdx.x;
    m.want = target - before;
  }
  __syncthreads();
  const unsigned at = (unsigned)m.pick;
  const u64 want = m.want;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const u64 e = lists.entry[i];
    if (e >= last && (0xffffffffu - (unsigned)e) >> shift == at) {
      const int to = atomicAdd(&m.large, 1);
      if (to < kFew) {
        lists.few[to] = e;
        lists.few_value[to] = lists.weight[i];
      }
    }
  }
  __syncthreads();
  const int few = m.large, log = few_log(few), parts = 1 << log, i = threadIdx.x >> log, part = threadIdx.x & (parts - 1);
  if (few > kFew) return false;
  if (i < few) {
    const u64 mine = lists.few[i], weight = lists.few_value[i];
    u64 below = 0;
#pragma unroll 1
    for (int j = part; j < few; j += parts) {
      const u64 w = lists.few_value[j];
      below += (unsigned)lists.few[j] > (unsigned)mine ? w : 0;
    }
    below = over_parts(below, log);
    if (part == 0 && want >= below && want < below + weight)
      answer(c, r, (int)(0xffffffffu - (unsigned)mine), (double)weight / (double)all);
  }
  return true;
}
// choose_few for up to kListedMost tokens, none below key `tau`.  Their bins reach down to that, or of a row whose tokens are all listed,
// where it is f32's lowest, to the least of them (else all would be in one bin); for weights to where they end.
__device__ __forceinline__ bool choose_many(Lists& lists, Common& m, const SampleCall& c, long long r, const SampleRule& rule,
                                            const Scale& sc, int n, unsigned tau, double whole, bool complete) {
  const bool count_cut = by_count(rule, c.vocab), weight_cut = by_weight(rule);
  if (count_cut && !complete && n < rule.top_k) return false;
  if (threadIdx.x == 0) m.least = 0xffffffffu;
  __syncthreads();
  u64 mine = 0, listed;
  unsigned lowest = key_of(INFINITY);
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned key = (unsigned)(lists.entry[i] >> 32);
    const double real = weight_of(sc, logit_of(key));
    mine += lists.weight[i] = units(sc, real);
    lowest = min(lowest, key);
    if (sc.min_p > 0.0) {
      if (real >= sc.min_p)
        atomicMin(&m.least, key);
      else
        m.large = 1;
    }
  }
  block_scan(m.sums, mine, listed);
  const unsigned least = m.least;
  const bool short_of_min = sc.min_p > 0.0 && (complete || m.large > 0);
  if (!count_cut && !short_of_min && !(weight_cut && (complete || listed >= part_units(rule, whole)))) return false;
  float end = logit_of(tau);
  if (tau <= kNothing + 1) {
    end = -bch::wave_allreduce(-logit_of(lowest), bch::OpMax());
    if ((threadIdx.x & 63) == 0) m.sums[1][threadIdx.x >> 6] = key_of(end);
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) lowest = min(lowest, (unsigned)m.sums[1][w]);
    end = logit_of(lowest);
  }
  const float end_weight = fmaxf(end, sc.m - 44.4f * rule.temperature);  // (2^-64 there)
  u64 last = 0, more = 0;
  if (count_cut && n > rule.top_k) {
    if (!list_cut(lists, m, Bins{sc.m, (float)kSlots / (sc.m - end), 0.0f}, n, 0, true, rule.top_k, last)) return false;
    if (weight_cut) {
      mine = 0;
      for (int i = threadIdx.x; i < n; i += kThreads) mine += lists.entry[i] >= last ? lists.weight[i] : 0;
      block_scan(m.sums, mine, listed);
    }
  }
  if (weight_cut) {
    if (!list_cut(lists, m, Bins{sc.m, (float)kSlots / (sc.m - end_weight), 0.0f}, n, last, false,
                  part_units(rule, count_cut ? (double)listed : whole), more))
      return false;
    last = max(last, more);
  }
  if (sc.min_p > 0.0) last = max(last, (u64)least << 32);
  return list_draw(lists, m, c, r, n, last);
}

// A row's token from its records and lists (list of span i at lists + i * kListMost).  False if they do not tell; `top`: the
// largest logit's key, `whole`: the row's weight in units, where only a weight cuts.
__device__ bool choose(Work& work, Common& m, const SampleCall& c, long long r, const SampleRule& rule, int spans, const Record* records,
                       const u64* lists, unsigned& top, double& whole) {
  whole = 0.0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the beginnings of the lists, 16 lanes a span: of up to four spans a thread, or more of fewer
  constexpr int kFlight = 4, kAt = kThreads / 16;
  const int glog = spans <= kAt ? 0 : spans <= 2 * kAt ? 1 : 2, j0 = threadIdx.x % 16, rounds = kFlight >> glog;
  int count[kFlight];
  u64 e[kFlight];
  auto span_at = [&](int i0, int f) { return i0 + (f & ((1 << glog) - 1)) * kAt + (int)threadIdx.x / 16; };
  auto fetch = [&](int i0) {
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int i = span_at(i0, f), at = min(i, spans - 1);
      count[f] = i < spans ? records[at].count : 0;
      e[f] = lists[(long long)at * kListMost + j0 + 16 * (f >> glog)];
    }
  };
  fetch(0);
  // the largest logit and its lowest index; the bound from which the lists are whole
  unsigned tau = 0;
  u64 best = 0;
  for (int i = threadIdx.x; i < spans; i += kThreads) {
    const Record q = records[i];
    best = max(best, (u64)q.top << 32 | (0xffffffffu - (unsigned)q.first));
    tau = max(tau, q.tau);
  }
  const unsigned mine = (unsigned)(best >> 32);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    best = max(best, __shfl_xor(best, d));
    tau = max(tau, (unsigned)__shfl_xor((int)tau, d));
  }
  if (lane == 0) {
    m.sums[0][wave] = best;
    m.sums[1][wave] = tau;
  }
  unsigned* tops = reinterpret_cast<unsigned*>(work.lists.slot);
  const bool by_tops = tops_tell(rule, c.vocab, spans);
  if (by_tops && (int)threadIdx.x < kTopsMost) tops[threadIdx.x] = (int)threadIdx.x < spans ? mine : 0;
  if (threadIdx.x == 0) m.n = m.large = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    best = max(best, m.sums[0][i]);
    tau = max(tau, (unsigned)m.sums[1][i]);
  }
  top = (unsigned)(best >> 32);
  // as few tokens as hold all that can stay: from the top_k-th largest of the spans' largest on (its upper half), or from min_p on
  if (by_tops) {
    if (wave == 0) {
      unsigned v[kTopsMost / 64], from = 0;
#pragma unroll
      for (int f = 0; f < kTopsMost / 64; ++f) v[f] = tops[64 * f + lane];
      const int differ = 31 - __clz((int)((tau ^ top) | 1u));  // above it any bound from tau on is as top
      from = differ < 31 ? top >> (differ + 1) << (differ + 1) : 0;
#pragma unroll 1
      for (int bit = differ; bit >= 16; --bit) {
        const unsigned next = from | 1u << bit;
        int n = 0;
#pragma unroll
        for (int f = 0; f < kTopsMost / 64; ++f)
          if (64 * f < spans) n += __popcll(__ballot(v[f] >= next));
        if (n >= rule.top_k) from = next;
      }
      if (lane == 0) m.least = from;
    }
    __syncthreads();
    tau = max(tau, m.least);
  }
  __syncthreads();
  if (top == kNothing || one_token(rule)) {
    if (threadIdx.x == 0) {
      const bool any = top != kNothing;
      answer(c, r, any ? (int)(0xffffffffu - (unsigned)best) : -1, any ? 1.0 : 0.0);
    }
    return true;
  }
  const Scale sc = scale_of(c, rule, logit_of(top));
  const bool count_cut = by_count(rule, c.vocab), weight_cut = by_weight(rule);
  if (!count_cut && !weight_cut && sc.min_p == 0.0) {
    draw_span<true>(m, c, r, rule, sc, spans, records);
    return true;
  }
  bool covers_min = false;
  if (sc.min_p > 0.0 && !count_cut) {
    const unsigned from = least_key(rule, sc);
    covers_min = from >= tau;
    tau = max(tau, from);
  }
  // the lists' tokens from tau on
  auto take = [&](u64 e, bool on) {
    on = on && (unsigned)(e >> 32) >= tau;
    const u64 mask = __ballot(on);
    int slot = 0;
    if (lane == 0 && mask) slot = atomicAdd(&m.n, __popcll(mask));
    slot = __shfl(slot, 0) + __popcll(mask & ((1ull << lane) - 1));
    if (on && slot < kListedMost) work.lists.entry[slot] = e;
  };
#pragma unroll 1
  for (int i0 = 0; i0 < spans; i0 += kAt << glog) {
    if (i0 > 0) fetch(i0);
    for (int j = j0;; j += 16 * rounds) {
      u64 now[kFlight];
      bool on[kFlight], more = false;
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int k = j + 16 * (f >> glog), then = k + 16 * rounds;
        now[f] = e[f];
        on[f] = k < count[f];
        if (then < count[f]) {
          more = true;
          e[f] = lists[(long long)span_at(i0, f) * kListMost + then];
        }
      }
#pragma unroll
      for (int f = 0; f < kFlight; ++f) take(now[f], on[f]);
      if (!__any(more)) break;
    }
  }
  if (!count_cut && weight_cut) whole = row_weight<true>(m, c, c.logits + r * c.stride, rule, sc, spans, records);
  __syncthreads();
  int n = m.n;
  const bool complete = tau <= kNothing + 1 || covers_min;  // all that can stay is on the lists
  const bool found = n > 0 && n <= kListedMost;
  if (count_cut && n > 64 && n > rule.top_k && rule.top_k <= 128 && n <= kKeysMost) n = largest_of(work.lists, m, n, rule.top_k);
  if (found && n <= kFewMost ? choose_few(work.lists, m, c, r, rule, sc, n, whole, complete)
                         : found && choose_many(work.lists, m, c, r, rule, sc, n, tau, whole, complete))
    return true;
  __syncthreads();
  return false;
}

// ---- rows of which thousands of tokens stay ----
// Where only weights cut a row (top_p or min_p, no top_k), its weights are sorted into kBins bins of their logarithm, a chunk of kChunk
// logits a workgroup; then one workgroup a row finds the bin that the cut falls into, collects that bin's tokens and cuts among them,
// and draws: the bins hold each chunk's weight above the cut, so one chunk is read again.  What bounds it: of 20 us for 16 rows of
// 50021 (23 for one of 131072) the bins' sums take 3, the collecting 4 (7; 17 with eight logits a thread in flight instead of 32), the
// chunks' sums 2, the weights of the one chunk 5.
constexpr int kChunk = 8192, kChunksMost = kThreads;

__device__ __forceinline__ bool binned(const SampleRule& rule, int vocab) {
  return !by_count(rule, vocab) && !(by_weight(rule) && rule.min_p > 0.0f);
}
// Descending with x; a weight of 0 falls into the last.
__device__ __forceinline__ float bins_per(const Scale& s) { return (float)(s.per * (kBins / 50.0)); }
__device__ __forceinline__ int bin_of(const Scale& s, float x) {
  return x == s.m ? 0 : (int)fminf((s.m - x) * bins_per(s), (float)(kBins - 1));
}

// hist (LDS): the weights of a chunk's tokens, of those that min_p leaves.
__device__ void bin_chunk(u64* hist, const SampleCall& c, const float* row, const Scale& sc, int chunk) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) hist[i] = 0;
  float x[8];
  load_eight(c, row, chunk * kChunk + 8 * threadIdx.x, x);
  __syncthreads();
  each(x, [&](float t) {
    const double v = weight_of(sc, t);
    const u64 w = v >= sc.min_p ? units(sc, v) : 0;
    if (w) atomicAdd(&hist[bin_of(sc, t)], w);
  });
  __syncthreads();
}

// The row's token from its chunks' bins (chunk i's at hist + i * kBins); whole_row as general_row's.
__device__ void choose_binned(Work& work, Common& m, const SampleCall& c, long long r, const SampleRule& rule, const Scale& sc,
                              const u64* hist, double whole_row) {
  const float* row = c.logits + r * c.stride;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, chunks = (c.vocab - 1) / kChunk + 1;
  if (chunks > kChunksMost || c.vocab < 4) {
    general_row(work.general, m.sums, c, r, rule, sc, whole_row);
    return;
  }
  int cut = kBins;   // the bin that the cut falls into: tokens of lower ones stay,
  u64 last = ~0ull;  // and of its tokens those at or above this entry
  int stay = 0;
  if (by_weight(rule)) {
    const int i0 = 2 * threadIdx.x;
    u64 w0 = 0, w1 = 0;
#pragma unroll 8
    for (int i = 0; i < chunks; ++i) {
      w0 += hist[(long long)i * kBins + i0];
      w1 += hist[(long long)i * kBins + i0 + 1];
    }
    u64 whole;
    u64 before = block_scan(m.sums, w0 + w1, whole);
    const u64 target = min(whole, part_units(rule, whole_row));
    if (before < target && before + w0 + w1 >= target) {
      const bool second = before + w0 < target;
      m.pick = second ? i0 + 1 : i0;
      m.want = target - before - (second ? w0 : 0);
    }
    if (threadIdx.x == 0) m.n = m.large = 0;
    __syncthreads();
    cut = m.pick;
    const u64 want = m.want;
    // 32 logits a thread in flight (a CU has its share of the memory only so); fours that hold one near the bin are noted (its ends as
    // logits, with room for what bin_of rounds), and then looked at
    const float g = bins_per(sc), from = (float)cut / g, to = cut == kBins - 1 ? INFINITY : ((float)cut + 1.0f) / g;
    float low = sc.m - to - 2e-6f * (fabsf(sc.m) + to), high = sc.m - from + 2e-6f * (fabsf(sc.m) + from);
    low = low == low ? low : -INFINITY;
    high = high == high ? high : INFINITY;
    int* near = reinterpret_cast<int*>(work.lists.slot);
    constexpr int kFours = 8, kNearMost = 2 * kSlots;
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 1
    for (int at = 4 * threadIdx.x; at < c.vocab; at += 4 * kThreads * kFours) {
      f32x4_any x[kFours];
#pragma unroll
      for (int f = 0; f < kFours; ++f)  // (a four that would end behind the row: the row's last, and with them all that it has)
        x[f] = *reinterpret_cast<const f32x4_any*>(row + min(at + 4 * kThreads * f, c.vocab - 4));
#pragma unroll
      for (int f = 0; f < kFours; ++f) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= x[f][e] >= low && x[f][e] <= high;
        if (any && at + 4 * kThreads * f < c.vocab) {
          const int to = atomicAdd(&m.large, 1);
          if (to < kNearMost) near[to] = at + 4 * kThreads * f;
        }
      }
    }
    __syncthreads();
    const int fours = m.large;
#pragma unroll 1
    for (int j = threadIdx.x; j < 4 * min(fours, kNearMost); j += kThreads) {
      const int i = near[j / 4] + j % 4;
      if (i >= c.vocab) continue;
      const float t = clean(row[i]);
      if (t > -INFINITY && bin_of(sc, t) == cut) {
        const int to = atomicAdd(&m.n, 1);
        if (to < kListedMost) work.lists.entry[to] = (u64)key_of(t) << 32 | (0xffffffffu - (unsigned)i);
      }
    }
    __syncthreads();
    const int n = m.n;
    if (n > kListedMost || fours > kNearMost) {
      __syncthreads();
      general_row(work.general, m.sums, c, r, rule, sc, whole_row);
      return;
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kThreads)
      work.lists.weight[i] = units(sc, weight_of(sc, logit_of((unsigned)(work.lists.entry[i] >> 32))));
    // (the bin's own kSlots parts)
    if (!list_cut(work.lists, m, Bins{sc.m, g * (float)kSlots, (float)cut * (float)kSlots}, n, 0, false, want, last)) {
      __syncthreads();
      general_row(work.general, m.sums, c, r, rule, sc, whole_row);
      return;
    }
    stay = n;
  }
  // what stays of each chunk
  __syncthreads();
  for (int i = wave; i < chunks; i += kWaves) {
    u64 sum = 0;
#pragma unroll 8
    for (int b = 0; b < kBins; b += 64) sum += b + lane < cut ? hist[(long long)i * kBins + b + lane] : 0;
    for (int j = lane; j < stay; j += 64)
      if (work.lists.entry[j] >= last && (int)((0xffffffffu - (unsigned)work.lists.entry[j]) / kChunk) == i)
        sum += work.lists.weight[j];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) m.chunk[i] = sum;
  }
  __syncthreads();
  const u64 mine = (int)threadIdx.x < chunks ? m.chunk[threadIdx.x] : 0;
  u64 whole;
  const u64 before = block_scan(m.sums, mine, whole), target = draw_units(c, r, whole);
  if (target >= before && target < before + mine) {
    m.pick = threadIdx.x;
    m.want = target - before;
  }
  __syncthreads();
  // of that chunk's tokens each thread has eight, in index order
  int i = m.pick * kChunk + 8 * threadIdx.x;
  u64 want = m.want, sum = 0;
  float x[8];
  load_eight(c, row, i, x);
  const auto weight = [&](float t, int at) -> u64 {
    const int b = bin_of(sc, t);
    if (b > cut || (b == cut && ((u64)key_of(t) << 32 | (0xffffffffu - (unsigned)at)) < last)) return 0;
    const double v = weight_of(sc, t);
    return v >= sc.min_p ? units(sc, v) : 0;
  };
  int at = i;
  each(x, [&](float t) { sum += weight(t, at++); });
  u64 all;
  const u64 start = block_scan(m.sums, sum, all);
  if (want >= start && want - start < sum) {
    m.pick = i;
    m.want = want - start;
  }
  __syncthreads();
  if (wave > 0) return;
  // and of those eight a lane one
  i = m.pick + lane;
  const u64 w = lane < 8 ? weight(i < c.vocab ? clean(row[i]) : -INFINITY, i) : 0, end = wave_scan(w, lane);
  want = m.want;
  if (want < end && want >= end - w) answer(c, r, i, (double)w / (double)whole);
}

// Spans of all rows, four a workgroup.
__global__ __launch_bounds__(256) void sample_list_kernel(SampleCall c, int spans, int groups, Record* records, u64* lists) {
  const long long r = blockIdx.x / groups;
  const int at = (int)(blockIdx.x % groups) * 4 + (threadIdx.x >> 6);
  if (at >= spans) return;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  list_span<true>(c, c.logits + r * c.stride, rule, spans, at, records + r * spans + at,
            lists + (r * spans + at) * kListMost);
}
// A row that the lists do not tell: its weight as choose gives it, and its largest logit's key, or 0 for a row that is done.
struct Left {
  double whole;
  unsigned top;
};
// later: such rows are left to the next two kernels where their rule allows.
__global__ __launch_bounds__(kThreads) void sample_choose_kernel(SampleCall c, int spans, const Record* records, const u64* lists,
                                                                 bool later, Left* left) {
  __shared__ Work work;
  __shared__ Common common;
  const long long r = blockIdx.x;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  unsigned top;
  double whole;
  const bool done = choose(work, common, c, r, rule, spans, records + r * spans, lists + r * spans * kListMost, top, whole);
  const bool leave = !done && later && binned(rule, c.vocab);
  if (threadIdx.x == 0) left[r] = {whole, leave ? top : 0};
  if (!done && !leave) general_row(work.general, common.sums, c, r, rule, scale_of(c, rule, logit_of(top)), whole);
}
__global__ __launch_bounds__(kThreads) void sample_bin_kernel(SampleCall c, int chunks, const Left* left, u64* hists) {
  __shared__ u64 hist[kBins];
  const long long r = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const unsigned top = left[r].top;
  if (!top) return;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  bin_chunk(hist, c, c.logits + r * c.stride, scale_of(c, rule, logit_of(top)), chunk);
  u64* to = hists + (r * chunks + chunk) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) to[i] = hist[i];
}
__global__ __launch_bounds__(kThreads) void sample_binned_kernel(SampleCall c, int chunks, const Left* left, const u64* hists) {
  __shared__ Work work;
  __shared__ Common common;
  const long long r = blockIdx.x;
  const unsigned top = left[r].top;
  if (!top) return;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  choose_binned(work, common, c, r, rule, scale_of(c, rule, logit_of(top)), hists + r * chunks * kBins,
                left[r].whole);
}

// All of it for a row of up to kWaves spans.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleCall c, int spans) {
  __shared__ Work work;
  __shared__ Common common;
  __shared__ Record records[kWaves];
  __shared__ u64 lists[kWaves * kListMost];  // and then the bins
  static_assert(kWaves * kListMost >= kBins && kWaves * kSpan <= kChunk, "bins of one chunk in the lists' place");
  const long long r = blockIdx.x;
  const float* row = c.logits + r * c.stride;
  const SampleRule rule = c.rules ? c.rules[r] : c.rule;
  const int wave = threadIdx.x >> 6;
  if (wave < spans) list_span<false>(c, row, rule, spans, wave, &records[wave], &lists[wave * kListMost]);
  __syncthreads();
  unsigned top;
  double whole;
  if (choose(work, common, c, r, rule, spans, records, lists, top, whole)) return;
  const Scale sc = scale_of(c, rule, logit_of(top));
  if (binned(rule, c.vocab)) {
    bin_chunk(lists, c, row, sc, 0);
    choose_binned(work, common, c, r, rule, sc, lists, whole);
  } else {
    general_row(work.general, common.sums, c, r, rule, sc, whole);
  }
}

// A row of any length where there is no room for records.
__global__ __launch_bounds__(kThreads) void sample_whole_kernel(SampleCall c, int spans) {
  __shared__ General general;
  __shared__ Common common;
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
  if (lane == 0) common.sums[0][wave] = top;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) top = max(top, common.sums[0][w]);
  __syncthreads();
  const unsigned top_key = (unsigned)(top >> 32);
  if (top_key == kNothing || one_token(rule)) {
    const bool any = top_key != kNothing;
    if (threadIdx.x == 0) answer(c, r, any ? (int)(0xffffffffu - (unsigned)top) : -1, any ? 1.0 : 0.0);
    return;
  }
  const Scale sc = scale_of(c, rule, logit_of(top_key));
  const bool count_cut = by_count(rule, c.vocab), weight_cut = by_weight(rule);
  if (!count_cut && !weight_cut && sc.min_p == 0.0) {
    draw_span<false>(common, c, r, rule, sc, spans, nullptr);
    return;
  }
  const double whole = !count_cut && weight_cut ? row_weight<false>(common, c, row, rule, sc, spans, nullptr) : 0.0;
  general_row(general, common.sums, c, r, rule, sc, whole);
}

}  // namespace

namespace bch {

int sample_unit_log(int vocab) {
  int bits = 1;
  while (bits < 31 && (1LL << bits) <= vocab) ++bits;
  return std::min(51, 62 - bits);
}

// Of a row: lists, records, what is left of it, and bins; none where a workgroup holds them.
struct RowBytes {
  size_t lists, records, bins, all;
};
static RowBytes row_bytes(const SampleCall& c) {
  const size_t spans = (size_t)(c.vocab - 1) / kSpan + 1, chunks = (size_t)(c.vocab - 1) / kChunk + 1;
  if (spans <= kWaves) return {0, 0, 0, 0};
  RowBytes b{spans * kListMost * sizeof(u64), spans * sizeof(Record), chunks > kChunksMost ? 0 : chunks * kBins * sizeof(u64), 0};
  b.all = b.lists + b.records + b.bins + sizeof(Left);
  return b;
}
constexpr size_t kMostBytes = (size_t)64 << 20;  // rows go through it in turn

size_t sample_workspace_bytes(const SampleCall& call, int rows) {
  const size_t each = row_bytes(call).all;
  return std::min(each * (size_t)rows, std::max(kMostBytes, each));
}

hipError_t launch_sample(hipStream_t s, const SampleCall& call, int rows, void* ws, size_t ws_bytes) {
  const int spans = (call.vocab - 1) / kSpan + 1, groups = (spans - 1) / 4 + 1, chunks = (call.vocab - 1) / kChunk + 1;
  const RowBytes each = row_bytes(call);
  const bool listed = each.all > 0 && ws_bytes >= each.all;
  // the two kernels for rows that the lists do not tell: not if the host knows that a count cuts every row, or nothing does
  const SampleRule& rule = call.rule;
  const bool later = each.bins > 0 && (call.rules || ((rule.top_k == 0 || rule.top_k >= call.vocab) && rule.temperature > 0.0f &&
                                                      (rule.top_p < 1.0f) != (rule.min_p > 0.0f)));
  long long most = 1 << 21;
  if (listed)
    most = std::min({most, (long long)(std::min(ws_bytes, std::max(kMostBytes, each.all)) / each.all), (1LL << 21) / groups + 1});
  for (long long at = 0; at < rows; at += most) {
    const int n = (int)std::min(most, rows - at);
    SampleCall c = call;
    c.logits += at * call.stride;
    if (c.rules) c.rules += at;
    c.u += at;
    c.tokens += at;
    if (c.probs) c.probs += at;
    hipError_t e;
    if (listed) {
      u64* lists = static_cast<u64*>(ws);
      u64* hists = lists + n * each.lists / sizeof(u64);
      Record* records = reinterpret_cast<Record*>(hists + n * each.bins / sizeof(u64));
      Left* left = reinterpret_cast<Left*>(records + (size_t)n * spans);
      hipLaunchKernelGGL(sample_list_kernel, dim3((unsigned)(n * (long long)groups)), dim3(256), 0, s, c, spans, groups, records, lists);
      if ((e = hipGetLastError()) != hipSuccess) return e;
      hipLaunchKernelGGL(sample_choose_kernel, dim3(n), dim3(kThreads), 0, s, c, spans, records, lists, later, left);
      if ((e = hipGetLastError()) != hipSuccess) return e;
      if (later) {
        hipLaunchKernelGGL(sample_bin_kernel, dim3((unsigned)(n * (long long)chunks)), dim3(kThreads), 0, s, c, chunks, left, hists);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        hipLaunchKernelGGL(sample_binned_kernel, dim3(n), dim3(kThreads), 0, s, c, chunks, left, hists);
      }
    } else if (spans <= kWaves) {
      hipLaunchKernelGGL(sample_row_kernel, dim3(n), dim3(kThreads), 0, s, c, spans);
    } else {
      hipLaunchKernelGGL(sample_whole_kernel, dim3(n), dim3(kThreads), 0, s, c, spans);
    }
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace bch
