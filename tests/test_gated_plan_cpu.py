"""The plan of the gated backward pass's second products, checked without a device: over many shapes, numbers of CTA pairs and
choices of gradients, every step of every output tile's reduction belongs to exactly one unit, and every part has its place."""
import os
import subprocess

from conftest import ROOT

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>
#include "ql_gated_plan.cuh"
using namespace ql;

static const char *check(int M, int I, int K, bool want_x, bool want_w, int pairs) {
  const GradPlan p = plan_grads(M, I, K, want_x, want_w, pairs);
  const GradArgs &a = p.a;
  if (a.layers != 1 && (a.layers != 2 || M > 128)) return "layers";
  if (p.clusters < 1 || p.clusters > pairs) return "clusters";
  const int tm[2] = {(M + 255) / 256, 2 * ((I + 255) / 256)}, tn = (K + 255) / 256;
  const int steps[2] = {2 * ((I + 63) / 64), a.layers * ((M + 63) / 64)};
  const int parts[2] = {a.x_split, a.w_split};
  const bool want[2] = {want_x, want_w};
  if (a.x_steps != steps[0] || a.w_steps != steps[1]) return "steps";
  std::vector<int> begin[2], end[2]; // of each tile's parts
  for (int k = 0; k < 2; k++) {
    if (parts[k] < 1 || parts[k] > 32 || parts[k] > steps[k]) return "parts";
    begin[k].assign((size_t)tm[k] * tn * parts[k], -1);
    end[k].assign((size_t)tm[k] * tn * parts[k], -1);
  }
  Unit u;
  for (int c = 0; c < p.clusters; c++) {
    for (int j = 0; get_unit(a, c, p.clusters, j, &u); j++) {
      const int k = u.is_x ? 0 : 1;
      if (!want[k]) return "a unit of a gradient nobody wants";
      if (u.is_x && u.up) return "up";
      const int mt = u.row0 / 256 + (u.up ? tm[1] / 2 : 0), nt = u.col0 / 256;
      if (u.row0 < 0 || u.row0 % 256 || u.col0 % 256 || mt >= tm[k] || nt >= tn || u.row0 >= (k ? I : M) || u.col0 >= K) return "tile";
      if (u.part < 0 || u.part >= parts[k] || u.step0 < 0 || u.step0 >= u.step1 || u.step1 > steps[k]) return "part";
      const size_t at = ((size_t)mt * tn + nt) * parts[k] + u.part;
      if (begin[k][at] != -1) return "a unit twice";
      begin[k][at] = u.step0, end[k][at] = u.step1;
    }
  }
  for (int k = 0; k < 2; k++)
    for (size_t tile = 0; want[k] && tile < (size_t)tm[k] * tn; tile++)
      for (int q = 0, next = 0; q < parts[k]; q++) {
        if (begin[k][tile * parts[k] + q] != next) return "a step twice or never";
        next = end[k][tile * parts[k] + q];
        if (q == parts[k] - 1 && next != steps[k]) return "steps at the end";
      }
  // a layer of f32 for each part (and each of the remainders' layers), or none
  const int64_t x_layers = (int64_t)parts[0] * a.layers, w_layers = 2ll * parts[1];
  if (p.x_part_floats != (want_x && x_layers > 1 ? x_layers * M * K : 0)) return "room for the parts of dX";
  if (p.w_part_floats != (want_w && parts[1] > 1 ? w_layers * I * K : 0)) return "room for the parts of dW";
  return nullptr;
}

int main() {
  std::mt19937 rng(1234);
  const int many[] = {74, 73, 66, 37, 148, 7, 2, 1};
  auto size = [&](double low, double high) {
    return (int)std::exp(std::uniform_real_distribution<double>(std::log(low), std::log(high))(rng));
  };
  int cases = 0;
  for (int i = 0; i < 12000; i++) {
    int M = size(1, 9000), I = (size(8, 30000) + 7) / 8 * 8, K = (size(8, 9000) + 7) / 8 * 8;
    if (i % 4 == 0) M = size(1, 200);
    if (i % 16 == 1) I = 8 + 8 * (i / 16 % 40), K = 8 + 8 * (i / 640);
    const int pairs = i % 3 ? 74 : many[i / 3 % 8];
    for (int wants = 1; wants < 4; wants++, cases++) {
      const char *wrong = check(M, I, K, wants & 1, wants & 2, pairs);
      if (wrong) {
        printf("%d x %d x %d, dX %d, dW %d, %d pairs: %s\n", M, I, K, wants & 1, wants >> 1, pairs, wrong);
        return 1;
      }
    }
  }
  printf("%d cases\n", cases);
  return 0;
}
"""


def test_every_step_of_every_tile_once(tmp_path):
    source, program = tmp_path / "plan.cc", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "tensorrt-incubator_b200", "csrc"), "-o", str(program), str(source)], check=True)
    r = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    assert r.stdout == "36000 cases\n"
