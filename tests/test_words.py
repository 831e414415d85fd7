"""Ranges of order-preserving words (csrc/words.h): the rounds in which a threshold is
found among a row's entries, on the CPU, where a range ends beside zero."""

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "attention_nn_amd", "csrc")

PROGRAM = r"""
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#include "words.h"
using namespace ann;

static const uint32_t ZERO = 0x80000000u, BELOW = 0x7fffffffu;   // 0's word, and -0's, which no number has

// The largest word t from lo on with `want` entries or more at t or above, by rounds over 2048
// bins; 1 where a round leaves no smaller range or an entry passes the bins.
static int rounds(const std::vector<float>& v, uint32_t lo, uint32_t hi, size_t want, uint32_t* t) {
  WordRange r = {lo, hi};
  size_t above = 0;
  while (r.lo != r.hi) {
    const int s = r.shift();
    std::vector<size_t> bins(2048, 0);
    for (float x : v) {
      int part;
      if (!r.has(x, s, part)) continue;
      if (part < 0 || part > 2047) return 1;
      ++bins[part];
    }
    int at = -1;
    for (int b = 2047; b >= 0 && at < 0; --b) {
      if (above + bins[b] >= want) at = b;
      else above += bins[b];
    }
    if (at < 0) return 2;
    const WordRange to = r.part(at, s);
    if (to.lo < r.lo || to.hi > r.hi || to.lo > to.hi || to.hi - to.lo >= r.hi - r.lo) return 3;
    r = to;
  }
  *t = r.lo;
  return 0;
}

static int check(const std::vector<float>& v, uint32_t lo) {
  std::vector<uint32_t> words;
  for (float x : v)
    if (x == x && word_of(x + 0.f) >= lo) words.push_back(word_of(x + 0.f));
  if (words.empty()) return 0;
  std::sort(words.rbegin(), words.rend());
  for (size_t want : {(size_t)1, (words.size() + 1) / 2, words.size() * 3 / 4 + 1, words.size()}) {
    if (want > words.size()) continue;
    uint32_t t = 0;
    const int rc = rounds(v, lo, words[0], want, &t);
    if (rc || t != words[want - 1]) {
      printf("lo %08x want %zu of %zu: rc %d, %08x for %08x\n", lo, want, words.size(), rc, t, words[want - 1]);
      return 1;
    }
  }
  return 0;
}

int main() {
  // words keep the order, and 0 lies in no range that ends below it
  const float some[] = {-FLT_MAX, -1.f, -FLT_MIN, -1e-45f, 0.f, 1e-45f, FLT_MIN, 1.f, FLT_MAX, INFINITY};
  for (int i = 1; i < 10; ++i)
    if (word_of(some[i]) <= word_of(some[i - 1]) || word_value(word_of(some[i])) != some[i]) return 1;
  int part;
  for (uint32_t lo : {0x00800000u, 0x7fe00000u, 0x7ffffffeu, BELOW}) {
    const WordRange r = {lo, BELOW};
    if (r.has(0.f, r.shift(), part) || r.has(-0.f, r.shift(), part) || r.has(1.f, r.shift(), part)) return 2;
    if (r.has(NAN, r.shift(), part) || r.has(-NAN, r.shift(), part) || r.has(-INFINITY, r.shift(), part)) return 3;
    if (r.has(-1e-45f, r.shift(), part) != (lo < BELOW)) return 4;
    const WordRange z = {lo, ZERO};
    if (!z.has(0.f, z.shift(), part) || !z.has(-0.f, z.shift(), part)) return 5;
  }
  if (word_most(BELOW) != -1e-45f || word_most(ZERO) != 0.f || word_most(ZERO - 2) != -1e-45f) return 6;
  if (!(0.f > word_most(BELOW)) || word_most(word_of(1.5f)) != 1.5f) return 7;

  // zeros beside negative subnormal numbers: a bin of the first round ends at 0x7fffffff
  std::vector<float> v(100, 0.f);
  v.insert(v.end(), 200, -1e-45f);
  if (check(v, 0x00800000u)) return 8;
  srand(3);
  for (int t = 0; t < 3000; ++t) {
    v.clear();
    const int n = 1 + rand() % 60;
    for (int i = 0; i < n; ++i) {
      const uint32_t low = rand() % (1 << (1 + rand() % 23)), sign = (uint32_t)(rand() % 4 != 0) << 31;
      const float tiny = word_value(word_of(0.f) + low);       // subnormal, or just above
      const int kind = rand() % 8;
      v.push_back(kind < 2 ? 0.f : kind == 2 ? -0.f : kind == 3 ? (float)(rand() % 5 - 2)
                  : kind == 4 && t % 3 == 0 ? NAN : kind == 5 && t % 5 == 0 ? -INFINITY : sign ? -tiny : tiny);
    }
    // from the lowest number's word, one so placed that a bin of s bits ends at 0x7fffffff, or any
    const int s = rand() % 21;
    const uint32_t lo[3] = {0x00800000u, ZERO - ((1u + rand() % 2047) << s), 0x00800000u + (uint32_t)rand() % 0x7f000000u};
    for (uint32_t l : lo)
      if (check(v, std::max(l, 0x00800000u))) return 9;
  }
  return 0;
}
"""


def test_rounds_beside_zero(tmp_path):
    src, exe = tmp_path / "t.cpp", str(tmp_path / "t")
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0, (got.returncode, got.stdout)
