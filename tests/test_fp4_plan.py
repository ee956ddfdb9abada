"""How 4-bit products are divided (csrc/fp4_plan.h), compiled and swept on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SWEEP = r"""
#include <cstdio>
#include <vector>
#include "fp4_plan.h"

int main() {
  std::vector<int> m, n, k;
  for (int i = 1; i <= 300; ++i) m.push_back(i);
  for (int i : {333, 384, 511, 512, 513, 700, 1000, 1024, 1072, 2048, 4099, 65536, 1 << 20, (1 << 30) - 1}) m.push_back(i);
  for (int i : {1, 16, 127, 128, 129, 257, 512, 1001, 4096, 8192, 20001, 1 << 20, (1 << 30) - 1}) n.push_back(i);
  for (int i : {1, 64, 255, 256, 257, 512, 700, 1024, 1281, 1793, 2048, 4096, 8192, 70000, 1 << 20}) k.push_back(i);
  long plans = 0, split = 0, bad = 0, taken = 0, tampered = 0;
  for (int glu = 0; glu < 2; ++glu)
    for (int sms : {148, 132, 20})
      for (int M : m)
        for (int N : n)
          for (int K : k) {
            const int f = glu ? (N + 1) / 2 : N;
            const SplitPlan q = choose(glu, M, f, K, sms);
            ++plans;
            if (!q.CS) continue;
            ++split;
            if (!split_plan_ok(q, glu, false, M, f, K)) ++bad;
            const bool fused = M <= 64 && q.SL <= SPLIT_FUSED_MAX_SL;
            if (fused && !split_plan_ok(q, glu, true, M, f, K)) ++bad;
            // plans that must not run: several tiles of another width, a slice left out or empty
            auto refuse = [&](SplitPlan r) {
              r.ctas = (int64_t)r.rt * ((M + (int64_t)r.NT - 1) / r.NT) * r.CS;
              ++tampered;
              if (split_plan_ok(r, glu, false, M, f, K)) ++taken;
            };
            for (int w : {8, 32, 48, 96, 120})
              if (M > w) {
                SplitPlan r = q;
                r.NT = w;
                refuse(r);
              }
            SplitPlan r = q;
            r.NT = 192;
            refuse(r);
            r = q, r.CS += 1, refuse(r);
            r = q, r.CS -= 1, refuse(r);
            r = q, r.CS = 16, r.SL = 1, refuse(r);
          }
  printf("%ld %ld %ld %ld %ld\n", plans, split, bad, tampered, taken);
}
"""


def test_every_chosen_plan_may_run_and_others_are_refused(tmp_path):
    src, exe = tmp_path / "sweep.cpp", tmp_path / "sweep"
    src.write_text(SWEEP)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "t0_web_b200", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    plans, split, bad, tampered, taken = map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    assert plans > 100000 and split > 10000 and tampered > 50000
    assert bad == 0 and taken == 0


def test_the_launch_asks_first():
    """The host refuses a plan before it builds a launch from it."""
    src = open(os.path.join(ROOT, "t0_web_b200", "csrc", "k_fp4.cu")).read()
    body = src[src.index("cudaError_t launch_split("):]
    body = body[:body.index("cudaLaunchKernelEx")]
    assert "if (!split_plan_ok(q, GLU, FUSED, a.M, a.n, a.K)) return cudaErrorInvalidConfiguration;" in body
