// fp4_plan.h -- how a product of 4-bit matrices is divided (host arithmetic
// only; k_fp4.cu launches by it): M tokens, n result columns (a gated
// product's F), K values, sms multiprocessors.
#pragma once

#include <stdint.h>

constexpr int SPLIT_MAX_CLUSTER = 8;
constexpr int SPLIT_FUSED_MAX_SL = 8;  // stages of a slice whose activations the kernel quantises itself

// How a product is divided for the split kernel.
struct SplitPlan {
  int NT, CS, SL, rt;
  int64_t ctas;
  double us;  // estimate
};
// Tiles of 64 or 128 tokens where one does not hold them all.
inline SplitPlan split_plan(bool glu, int M, int n, int K, int most, int sms) {
  SplitPlan q;
  q.NT = M <= most ? (M + 7) / 8 * 8 : most;
  q.rt = (n + 127) / 128;
  const int64_t tiles = (int64_t)q.rt * ((M + q.NT - 1) / q.NT);
  const int S = (K + 255) / 256;
  // clusters have to fit the GPCs: of 8 CTAs not more than two thirds of the
  // SMs can be used at once (1024 x 4096, 256 tokens in tiles of 128: 128 CTAs
  // in clusters of 8 13.5 us, 96 in clusters of 4 for 384 tokens 8.4 us)
  int cs = 1;
  while (cs < SPLIT_MAX_CLUSTER && tiles * cs * 2 <= (cs == 4 ? sms * 2 / 3 : sms * 7 / 8) && S >= cs * 2) cs *= 2;
  q.SL = (S + cs - 1) / cs;
  q.CS = (S + q.SL - 1) / q.SL;
  q.ctas = tiles * q.CS;
  // microseconds, fitted to the measured times of up to 512 tokens: 512 x 512
  // 3.3 (16 tokens), 4.6 (64); 8192 x 8192 9.8 (16), 13.8 (128), 18.7 (256)
  const double waves = (double)((q.ctas + sms - 1) / sms);
  q.us = 2.6 + waves * ((glu ? 0.045 : 0.030) * q.NT + (glu ? 0.7 : 0.4) * q.SL);
  return q;
}

// The same for the pair kernel: 256 tokens 512 x 512 4.8, 1024 x 4096 8.9,
// 8192 x 8192 14.1; gated 512 x 512 5.5, 4096 x 4096 10.1.  Too short for many
// tokens (4096: 8192 x 64 9.6 for 14.5, 8192 x 8192 77 for 97), where the choice
// is the same all the same; elsewhere the chosen kernel is within about 8 % of
// the better one.
inline double pair_us(bool glu, int M, int n, int K, int sms) {
  const int64_t tiles = (int64_t)((M + 255) / 256) * (glu ? (n + 127) / 128 : (n + 255) / 256);
  return 3.9 + (double)((tiles + sms / 2 - 1) / (sms / 2)) * ((glu ? 1.1 : 0.5) + 0.31 * ((K + 255) / 256));
}

// The split kernel's plan if it is the faster one (CS 0: the pair kernel is).
inline SplitPlan choose(bool glu, int M, int n, int K, int sms) {
  SplitPlan q = split_plan(glu, M, n, K, 64, sms);
  if (!glu && M > 64) {
    const SplitPlan r = split_plan(glu, M, n, K, 128, sms);
    if (r.us < q.us) q = r;
  }
  if (pair_us(glu, M, n, K, sms) <= q.us) q.CS = 0;
  return q;
}

// Whether the split kernel may run a plan: what its layout of tensor and shared
// memory takes for granted.  A tile's first token has to lie on an even scale
// column (a multiple of 64 tokens): the MMA faults on an odd one.
inline bool split_plan_ok(const SplitPlan &q, bool glu, bool fused, int M, int n, int K) {
  const int S = (K + 255) / 256;
  if (q.NT < 8 || q.NT % 8 || q.NT > (glu || fused ? 64 : 128)) return false;
  if (M > q.NT && (q.NT % 64 || fused)) return false;
  if (q.CS < 1 || q.CS > SPLIT_MAX_CLUSTER || q.SL < 1) return false;
  if ((int64_t)q.CS * q.SL < S || (int64_t)(q.CS - 1) * q.SL >= S) return false;  // no slice left out, none empty
  if (fused && q.SL > SPLIT_FUSED_MAX_SL) return false;
  return q.rt == (n + 127) / 128 && q.ctas == (int64_t)q.rt * ((M + (int64_t)q.NT - 1) / q.NT) * q.CS;
}
