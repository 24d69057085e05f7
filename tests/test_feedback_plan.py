"""The host's sort of a preference plan's pairs: against a plain listing, and
with every one of its allocations failing in turn."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <new>
#include <vector>
#include "feedback_plan.h"

static std::atomic<long> seen{0}, fails{-1};  // allocations so far, the one that fails

static void* take(size_t n) {
  if (seen.fetch_add(1) == fails.load()) throw std::bad_alloc();
  if (void* p = malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void* operator new(size_t n) { return take(n); }
void* operator new[](size_t n) { return take(n); }
void operator delete(void* p) noexcept { free(p); }
void operator delete[](void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }
void operator delete[](void* p, size_t) noexcept { free(p); }

// fails the program with a name
static void want(bool ok, const char* what) {
  if (!ok) {
    printf("wrong: %s\n", what);
    exit(1);
  }
}

int main(int, char** argv) {
  const long long n = atoll(argv[1]), np = atoll(argv[2]);
  const bool weighted = atoi(argv[3]);
  std::vector<int64_t> w(np), l(np);
  std::vector<float> weights(np);
  unsigned long long x = 88172645463325252ull;
  auto next = [&](long long m) {
    x ^= x << 13, x ^= x >> 7, x ^= x << 17;
    return (long long)(x % (unsigned long long)m);
  };
  for (long long p = 0; p < np; ++p) {
    w[p] = p % 3 == 0 ? n / 2 : p % 3 == 1 ? next(std::min(n, 20ll)) : next(n);  // one huge item, some long ones
    do l[p] = next(n);
    while (l[p] == w[p]);
    if (next(2)) std::swap(w[p], l[p]);
    weights[p] = (float)next(5);
  }
  const float* wp = weighted ? weights.data() : nullptr;
  std::vector<std::vector<std::pair<int, int>>> of(n);
  std::vector<int> zero;
  for (long long p = 0; p < np; ++p) {
    if (wp && wp[p] == 0) {
      zero.push_back((int)p);
      continue;
    }
    of[w[p]].push_back({(int)l[p], (int)p});
    of[l[p]].push_back({(int)w[p] | (int)0x80000000, (int)p});
  }
  auto run = [&] { return mtb::sort_pairs(w.data(), l.data(), wp, np, n); };
  seen = 0;
  {
    const mtb::SortedPairs s = run();
    const int from = mtb::pairs_long_from(s.n_entries, n), huge = std::max(mtb::kHugeItem, from);
    long long at = 0, n_long = 0, n_huge = 0;
    for (long long i = 0; i < n; ++i) {
      want(s.offsets[i] == at, "offsets");
      for (auto& e : of[i]) {
        want(s.entries[at].x == e.first && s.entries[at].y == e.second, "entries");
        want(!wp || s.weights[at] == wp[e.second], "weights");
        ++at;
      }
      const long long m = (long long)of[i].size();
      if (m >= huge) want(n_huge < s.n_huge && s.huge_items[n_huge++] == i, "huge items");
      else if (m >= from) want(n_long < s.n_long && s.long_items[n_long++] == i, "long items");
    }
    want(s.offsets[n] == at && s.n_entries == at && n_long == s.n_long && n_huge == s.n_huge, "counts");
    want(s.n_zero == (long long)zero.size() && std::equal(zero.begin(), zero.end(), s.zero_pairs.get()), "pairs of weight 0");
    want(!wp == !s.weights, "weights");
    printf("%lld entries, %lld long, %lld huge, ", at, n_long, n_huge);
  }
  seen = 0;
  run();
  const long n_allocations = seen;
  for (long k = 0; k < n_allocations; ++k) {
    bool caught = false;
    seen = 0;
    fails = k;
    try {
      run();
    } catch (const std::bad_alloc&) {
      caught = true;
    }
    fails = -1;
    want(caught, "a failed allocation");
  }
  printf("%ld allocations\n", n_allocations);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(PROGRAM)
    csrc = os.path.join(ROOT, "mojoboost_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O2", "-fopenmp", "-I", csrc, "-I", "/usr/local/cuda/include", str(at / "plan.cpp"),
                    os.path.join(csrc, "feedback_plan.cpp"), "-o", str(at / "plan")], check=True)
    return str(at / "plan")


@pytest.mark.parametrize("n,pairs", [(2, 1), (2, 5000), (70, 3), (1000, 10_000), (100_000, 60_000), (5000, 200_000), (40, 300_000)])
@pytest.mark.parametrize("weighted", [0, 1])
def test_sorted_pairs(program, n, pairs, weighted):
    """The entries of each item in the pairs' order; a failed allocation is an
    exception that the caller gets, from parallel sorts too."""
    r = subprocess.run([program, str(n), str(pairs), str(weighted)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "allocations" in r.stdout, (r.returncode, r.stdout, r.stderr[-400:])
