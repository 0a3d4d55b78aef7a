"""A host program over the checks of tensors that share memory
(csrc/row_overlap.h), against every element of small tensors: no shared element is
missed, and slices of one buffer that share none are told apart, also where a dim
has one row and any stride."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "frisk_amd", "csrc")

MAIN = """
#include "%s/row_overlap.h"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
using frisk::Rows;
static std::set<int64_t> bytes_of(const Rows& r, int64_t row, int es) {
  std::set<int64_t> out;
  for (int64_t i = 0; i < r.n[0]; ++i)
    for (int64_t j = 0; j < r.n[1]; ++j)
      for (int64_t k = 0; k < r.n[2]; ++k)
        for (int64_t e = 0; e < row * es; ++e)
          out.insert((int64_t)r.p + (i * r.s[0] + j * r.s[1] + k * r.s[2]) * es + e);
  return out;
}
static bool share(const std::set<int64_t>& a, const std::set<int64_t>& b) {
  for (int64_t x : a)
    if (b.count(x)) return true;
  return false;
}
int main(int, char** v) {
  std::mt19937 rng(atoi(v[2]));
  const auto pick = [&](int lo, int hi) { return (int64_t)(lo + rng() %% (unsigned)(hi - lo + 1)); };
  int missed = 0, refused = 0, apart = 0, met = 0;
  for (int n = 0; n < 4000; ++n) {
    const int64_t row = pick(1, 4), es = 2;
    Rows a{(void*)1000, {pick(1, 3), pick(1, 3), pick(1, 3)}, {}}, b{nullptr, {pick(1, 3), pick(1, 3), pick(1, 3)}, {}};
    if (v[1][0] == 'r') {  // any strides
      for (int i = 0; i < 3; ++i) a.s[i] = pick(0, 30), b.s[i] = rng() & 1 ? a.s[i] : pick(0, 30);
      b.p = (void*)(1000 + pick(-60, 60));
    } else {  // heads of one buffer [batch, tokens, heads, row], in any order of the dims
      const int64_t heads = 8, tokens = 3;
      int64_t st[3] = {tokens * heads * row, row, heads * row};
      const int turn = (int)pick(0, 2);
      for (int i = 0; i < 3; ++i) a.s[i] = b.s[i] = st[(i + turn) %% 3];
      const int64_t at = pick(0, 5) * row + pick(0, 2) * heads * row;
      b.p = (void*)(1000 + at * es);
      for (int i = 0; i < 3; ++i) {
        if (a.n[i] == 1 && rng() & 1) a.s[i] = pick(0, 100);
        if (b.n[i] == 1 && rng() & 1) b.s[i] = pick(0, 100);
        if (rng() %% 8 == 0) b.s[i] = 0;  // repeated
      }
    }
    const bool truth = share(bytes_of(a, row, es), bytes_of(b, row, es));
    for (const bool said : {frisk::rows_share(a, b, row, es), frisk::rows_share(b, a, row, es)}) {
      missed += truth && !said;
      refused += !truth && said;
    }
    (truth ? met : apart)++;
  }
  printf("%%d %%d %%d %%d\\n", missed, refused, apart, met);
}"""


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "main.cpp").write_text(MAIN % CSRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", str(d / "main.cpp"),
                    "-o", str(d / "main")], check=True)
    return lambda *args: [int(x) for x in subprocess.run([str(d / "main"), *map(str, args)], check=True,
                                                         capture_output=True, text=True).stdout.split()]


@pytest.mark.parametrize("seed", range(3))
def test_no_shared_element_is_missed(overlap, seed):
    missed, _, apart, met = overlap("random", seed)
    assert missed == 0 and min(apart, met) > 500


@pytest.mark.parametrize("seed", range(3))
def test_slices_of_one_buffer_are_told_apart(overlap, seed):
    missed, refused, apart, met = overlap("slices", seed)
    assert missed == 0 and refused == 0 and min(apart, met) > 500
