// Host build of the softmax helpers of the tree attention (det_dev.cuh),
// compared here with the general forms; each returns the number of differences.
#include <cstdint>

#include "det_dev.cuh"

using namespace rdet;

static uint64_t mix(uint64_t z) {
  z += 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

extern "C" {
// every distance below the maximum that has a term
int64_t exp_all(int32_t max_logit) {
  int64_t bad = 0;
  for (uint32_t D = 0; D < (16u << 16); ++D)
    if ((int64_t)max_logit - D >= INT32_MIN)
      bad += (D ? (int64_t)exp_term_below(D) : kOneAcc) != exp_term((int32_t)((int64_t)max_logit - D), max_logit);
  return bad;
}
// the largest term below 2^32: the code 2^32 - 1 stands for 2^32 alone
uint64_t exp_second() { return exp_term_below(1); }

static int64_t one(uint64_t e, uint64_t sum) {
  const uint32_t coded = e >> 32 ? 0xffffffffu : (uint32_t)e;
  int32_t w;
  return softmax_weight_near(coded, softmax_inverse(sum), &w) && w != softmax_weight((int64_t)e, (int64_t)sum);
}
// the branch-free rounding, around every power of two, at every tie beside the
// ends of the range and at random
int64_t requantize_random(uint64_t seed, int64_t n) {
  int64_t bad = 0;
  auto check = [&](uint64_t v) { bad += requantize_flat((int64_t)v) != requantize((int64_t)v); };
  for (int sh = 0; sh < 64; ++sh)
    for (int64_t o = -70000; o <= 70000; ++o) {
      check((1ull << sh) + (uint64_t)o);
      check(0 - (1ull << sh) + (uint64_t)o);
    }
  for (int64_t i = 0; i < n; ++i) {
    const uint64_t v = mix(seed + i);
    check(v);
    check((uint64_t)((int64_t)v >> (i % 64)));
    check((uint64_t)((int64_t)v >> 16) & ~0xffffull | 0x8000u);
  }
  return bad;
}
// digit sums with an addend, against the same in 64 bits: random ones and ones
// beside the ends of the range
int64_t digits_random(uint64_t seed, int64_t n) {
  int64_t bad = 0;
  for (int64_t i = 0; i < n; ++i) {
    int32_t c[7];
    for (int g = 0; g < 7; ++g) {
      const uint64_t z = mix(seed + 16 * i + g);
      c[g] = (int32_t)(z >> 37) - (1 << 26);
      if (z % 5 == 0) c[g] = 0;
      if (z % 7 == 0) c[g] = z & 64 ? 1 << 26 : -(1 << 26);
      if ((i & 3) && g > 3) c[g] = (int32_t)(z % 3) - 1;
    }
    uint64_t v = 0;
    for (int g = 0; g < 7; ++g) v += (uint64_t)(int64_t)c[g] << (8 * g);
    uint64_t add = mix(seed + 16 * i + 8) >> (i % 64);
    if (i % 3 == 0) {  // the sum at a chosen place
      const uint64_t at = mix(seed + 16 * i + 9);
      add = ((at & 1 ? 1ull : ~0ull) << (at >> 8) % 64) + (uint64_t)((int64_t)((at >> 16) % 262144) - 131072) - v;
    }
    bad += requantize_digits(c[0], c[1], c[2], c[3], c[4], c[5], c[6], (int32_t)(add & 0xffff),
                             (int32_t)(add >> 16 & 0xffff), (int32_t)(add >> 32)) != requantize((int64_t)(v + add));
  }
  return bad;
}
// how many of n random weights the reciprocal leaves open
int64_t weights_open(uint64_t seed, int64_t n) {
  int64_t open = 0;
  for (int64_t i = 0; i < n; ++i) {
    const uint64_t a = mix(seed + 2 * i), b = mix(seed + 2 * i + 1);
    int32_t w;
    open += !softmax_weight_near((uint32_t)(b >> (32 + b % 16)), softmax_inverse((1ull << 32) + (a >> 24)), &w);
  }
  return open;
}
// random sums and terms
int64_t weights_random(uint64_t seed, int64_t n) {
  int64_t bad = 0;
  for (int64_t i = 0; i < n; ++i) {
    const uint64_t a = mix(seed + 2 * i), b = mix(seed + 2 * i + 1);
    const uint64_t sum = (1ull << 32) + (a >> (8 + a % 56)) % (1ull << 50);
    const uint64_t e = b % 3 == 0 ? (1ull << 32) : (b >> (32 + b % 31));
    bad += one(e, sum);
  }
  return bad;
}
// terms whose weight lies at k + 1/2, and their neighbours, for sums of every size
int64_t weights_ties(uint64_t seed, int64_t n) {
  int64_t bad = 0;
  for (int64_t i = 0; i < n; ++i) {
    const uint64_t a = mix(seed + i);
    const uint64_t sum = (1ull << 32) + (a >> 8) % (1ull << (1 + a % 49));
    const uint64_t k = mix(a) % 65536;
    // e 2^16 / sum = k + 1/2  ->  e = (2 k + 1) sum / 2^17
    const unsigned __int128 p = (unsigned __int128)(2 * k + 1) * sum;
    const uint64_t e0 = (uint64_t)(p >> 17);
    for (int64_t d = -3; d <= 4; ++d) {
      const uint64_t e = e0 + d;
      // terms are at most 2^32 - 2^15, or 2^32
      if ((int64_t)e >= 0 && e <= (1ull << 32) - (1ull << 15) && e <= sum) bad += one(e, sum);
    }
    // quotients at k + 1/2 exactly: sum a multiple of 2^17
    const uint64_t s2 = (sum >> 17 << 17) + (1ull << 32), e2 = (2 * k + 1) * (s2 >> 17);
    for (int64_t d = -2; d <= 2; ++d)
      if (e2 + d <= (1ull << 32) - (1ull << 15)) bad += one(e2 + d, s2);
  }
  return bad;
}
// a term equal or almost equal to the sum
int64_t weights_one(int64_t n) {
  int64_t bad = 0;
  for (int64_t i = 0; i < n; ++i) {
    bad += one(1ull << 32, (1ull << 32) + i);
    bad += one(1ull << 32, (1ull << 32) + i * 257);
    bad += one((1ull << 32) - (1ull << 15) - i, (1ull << 32));
  }
  return bad;
}
}
