// The C++ host API's windowed attention (include/barracuda_hip_ops.hpp): its checks, and its result against the
// sums written out, on a GPU.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "barracuda_hip_ops.hpp"

using namespace barracuda;

static int g_fail = 0;
#define REQUIRE(x)                                      \
  do {                                                  \
    if (!(x)) {                                         \
      std::printf("FAIL line %d: %s\n", __LINE__, #x);  \
      ++g_fail;                                         \
    }                                                   \
  } while (0)

static void checks() {
  using W = SlidingWindowAttention;
  REQUIRE(!W::validate({1, 8, 4, 16}, {1, 2, 9, 16}, {1, 2, 9, 16}));
  REQUIRE(W::validate({8, 4, 16}, {1, 2, 9, 16}, {1, 2, 9, 16})->kind == ErrorKind::InvalidInput);
  REQUIRE(W::validate({1, 8, 4, 16}, {1, 3, 9, 16}, {1, 3, 9, 16})->kind == ErrorKind::InvalidInput);
  REQUIRE(W::validate({1, 8, 4, 16}, {2, 2, 9, 16}, {2, 2, 9, 16})->kind == ErrorKind::ShapeMismatch);
  REQUIRE(W::validate({1, 8, 4, 16}, {1, 2, 9, 16}, {1, 2, 8, 16})->kind == ErrorKind::ShapeMismatch);
  std::printf("PASS window_checks\n");
}

static void result(const std::shared_ptr<HipDevice>& dev) {
  const size_t B = 2, H = 4, Hkv = 2, Sq = 21, Skv = 50, D = 8, window = 7, sinks = 2;
  std::vector<float> q(B * H * Sq * D), k(B * Hkv * Skv * D), v(k.size());
  auto fill = [](std::vector<float>& x, float f) {
    for (size_t i = 0; i < x.size(); ++i) x[i] = std::sin(f * (float)(i + 1));
  };
  fill(q, 0.7f);
  fill(k, 1.3f);
  fill(v, 0.31f);
  auto tq = Tensor::from_data(q, {B, H, Sq, D}, dev).unwrap();
  auto tk = Tensor::from_data(k, {B, Hkv, Skv, D}, dev).unwrap();
  auto tv = Tensor::from_data(v, {B, Hkv, Skv, D}, dev).unwrap();
  const auto got = tq.sliding_window_attention(tk, tv, window, sinks).unwrap().to_vec().unwrap();
  double worst = 0.0;
  for (size_t b = 0; b < B; ++b)
    for (size_t h = 0; h < H; ++h)
      for (size_t i = 0; i < Sq; ++i) {
        const size_t kv = (b * Hkv + h / (H / Hkv)) * Skv, pos = Skv - Sq + i;
        std::vector<double> o(D, 0.0);
        double sum = 0.0;
        for (size_t j = 0; j <= pos; ++j) {
          if (pos - j >= window && j >= sinks) continue;
          double s = 0.0;
          for (size_t d = 0; d < D; ++d) s += (double)q[((b * H + h) * Sq + i) * D + d] * k[(kv + j) * D + d];
          const double e = std::exp(s / std::sqrt((double)D));
          sum += e;
          for (size_t d = 0; d < D; ++d) o[d] += e * v[(kv + j) * D + d];
        }
        for (size_t d = 0; d < D; ++d)
          worst = std::max(worst, std::fabs(o[d] / sum - got[((b * H + h) * Sq + i) * D + d]));
      }
  // values up to 1, scores up to 3: a few tens of roundings of 2^-24
  REQUIRE(worst <= 64 * 0x1p-24);
  auto empty = Tensor::empty({0, 2, 5, 8}, dev).unwrap();
  REQUIRE(empty.sliding_window_attention(empty, empty, 3).is_ok());
  std::printf("PASS window_result\n");
}

int main(int argc, char** argv) {
  checks();
  if (argc > 1 && std::strcmp(argv[1], "--gpu") == 0) {
    auto dev = HipDevice::create(0);
    REQUIRE(dev.is_ok());
    if (dev.is_ok()) result(dev.value());
  }
  return g_fail == 0 ? 0 : 1;
}
