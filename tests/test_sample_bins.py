"""The sampler's choice of the histogram bins that can hold the top-p threshold: the threads of a CTA, run one after
another on the host, name one bin each way, and the threshold lies between the two."""
from __future__ import annotations

import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "wavefront-decoding_b200" / "csrc"

HARNESS = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "wfd_sample_bins.cuh"
using namespace wfd;
typedef unsigned long long ull;
constexpr int THREADS = 512, PER = 4, BINS = THREADS * PER;

struct Row {
  std::vector<unsigned> cnt;
  float g;
  double low;
  std::vector<SampleBounds<PER>> b;
  std::vector<ull> lo0, hi0;
  ull lo_all = 0, hi_all = 0;
  Row(std::vector<unsigned> c, float g_, double low_) : cnt(c), g(g_), low(low_) {
    for (int t = 0; t < THREADS; ++t) {
      const unsigned q[PER] = {cnt[4 * t], cnt[4 * t + 1], cnt[4 * t + 2], cnt[4 * t + 3]};
      b.push_back(sample_bounds(q, 4 * t, g, low));
      lo0.push_back(lo_all);
      hi0.push_back(hi_all);
      lo_all += b[t].lo_sum;
      hi_all += b[t].hi_sum;
    }
  }
  // bins named by each thread
  void bracket(float tp, std::vector<int>& first, std::vector<int>& last) const {
    first.clear();
    last.clear();
    for (int t = 0; t < THREADS; ++t)
      sample_bracket(b[t], lo0[t], hi0[t], lo_all, hi_all, tp, 4 * t, [&](int x) { first.push_back(x); },
                     [&](int x) { last.push_back(x); });
  }
};

int main() {
  std::mt19937_64 rng(7);
  auto uni = [&] { return std::uniform_real_distribution<double>(0, 1)(rng); };
  std::vector<int> first, last;
  long many = 0, none = 0, outside = 0, calls = 0;
  for (int trial = 0; trial < 40; ++trial) {
    std::vector<unsigned> c(BINS, 0);
    const double dense = uni();
    for (int i = 0; i < BINS; ++i)
      if (uni() < dense) c[i] = (unsigned)(1 + uni() * (trial % 4 == 3 ? 200 : 3));
    c[0] = std::max(c[0], 1u);
    const float g = trial % 5 == 4 ? 0.f : (float)(45.0 / BINS * uni());
    const Row row(c, g, trial % 10 == 9 ? 0.0 : 0.9999);
    // every border between two threads, from either side and for the numbers next to it
    std::vector<float> tps = {0.f, -1.f, 1e-30f, 0.99999994f, 0.5f, -__builtin_inff()};
    for (int t = 0; t < THREADS; ++t) {
      for (double at : {(double)row.hi0[t] / std::max(1.0, (double)row.lo_all), (double)row.lo0[t] / (double)row.hi_all}) {
        float tp = (float)at;
        for (int k = 0; k < 6; ++k) tp = nextafterf(tp, 0.f);
        for (int k = 0; k < 60 && tp < 1.f; ++k) {  // (the margin moves a crossing by some of these steps)
          tps.push_back(tp);
          tp = nextafterf(tp, 1.f);
        }
      }
    }
    // weights somewhere inside their bins, summed as the exact pass does
    std::vector<ull> mass(BINS, 0);
    ull Z = 0;
    for (int i = 0; i < BINS; ++i) {
      for (unsigned k = 0; k < c[i]; ++k) {
        const double x = row.low == 0.0 ? 45.0 * uni() : g * std::max(0.0, i - 0.5 + uni());
        mass[i] += (ull)(std::exp2(-x) * 17592186044416.0 + 0.5);
      }
      Z += mass[i];
    }
    for (float tp : tps) {
      ++calls;
      row.bracket(tp, first, last);
      many += first.size() > 1 || last.size() > 1;
      none += first.empty();
      const int b0 = first.empty() ? BINS - 1 : first[0], b1 = last.empty() ? BINS - 1 : last[0];
      const ull need = std::max<ull>(1, tp > 0.f ? (ull)std::ceil((double)tp * (double)Z) : 1);
      ull run = 0;
      int at = BINS - 1;
      for (int i = 0; i < BINS; ++i) {
        if (run < need && run + mass[i] >= need) {
          at = i;
          break;
        }
        run += mass[i];
      }
      outside += at < b0 || at > b1;
    }
  }
  std::printf("calls %ld many %ld none %ld outside %ld\n", calls, many, none, outside);
  return many || none || outside;
}
"""


def test_one_bin_each_way_and_the_threshold_between(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "bins.cpp"
    src.write_text(HARNESS)
    exe = tmp_path / "bins"
    subprocess.run([cxx, "-O2", "-std=c++17", "-D__host__=", "-D__device__=", "-D__forceinline__=inline", "-I", str(CSRC),
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout.split()[1]) > 1000000, out.stdout
