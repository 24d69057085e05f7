// Sorting a preference plan's pairs by item.
#include "feedback_plan.h"

#include <algorithm>
#include <vector>

namespace mtb {

// Two passes of a counting sort, both in the pairs' order and on all host
// threads: pairs into ranges of items, then each range's by item, within a
// core's cache.  An exception that leaves a thread of a parallel loop ends the
// process, so all memory is taken outside of them.
SortedPairs sort_pairs(const int64_t* winners, const int64_t* losers, const float* weights, long long np,
                       long long ni) {
  struct Entry {
    int item;
    int2 e;
    float w;
  };
  constexpr int kRanges = 256, kMostThreads = 64;
  const int parts = (int)std::min<long long>(kMostThreads, 1 + np / 16384);
  const long long range = std::max<long long>(1, (ni + kRanges - 1) / kRanges);
  std::vector<long long> count((size_t)parts * kRanges, 0), zeros(parts, 0);
  auto slice = [&](int t) { return np * t / parts; };
#pragma omp parallel for schedule(static, 1) if (parts > 1)
  for (int t = 0; t < parts; ++t) {
    long long* c = &count[(size_t)t * kRanges];
    for (long long p = slice(t); p < slice(t + 1); ++p) {
      if (weights && weights[p] == 0.0f) {
        ++zeros[t];
        continue;
      }
      ++c[winners[p] / range];
      ++c[losers[p] / range];
    }
  }
  std::vector<long long> start(kRanges + 1, 0), zero_at(parts + 1, 0);
  long long total = 0;
  for (int q = 0; q < kRanges; ++q) {
    start[q] = total;
    for (int t = 0; t < parts; ++t) {
      const long long c = count[(size_t)t * kRanges + q];
      count[(size_t)t * kRanges + q] = total;
      total += c;
    }
  }
  start[kRanges] = total;
  for (int t = 0; t < parts; ++t) zero_at[t + 1] = zero_at[t] + zeros[t];
  std::unique_ptr<Entry[]> sorted(new Entry[std::max(1ll, total)]);
  SortedPairs s;
  s.n_entries = total;
  s.n_zero = zero_at[parts];
  s.zero_pairs.reset(new int[std::max(1ll, s.n_zero)]);
  s.offsets.reset(new int[(size_t)ni + 1]);
  s.entries.reset(new int2[std::max(1ll, total)]);
  if (weights) s.weights.reset(new float[std::max(1ll, total)]);
#pragma omp parallel for schedule(static, 1) if (parts > 1)
  for (int t = 0; t < parts; ++t) {
    long long* c = &count[(size_t)t * kRanges];
    long long z = zero_at[t];
    for (long long p = slice(t); p < slice(t + 1); ++p) {
      const int a = (int)winners[p], b = (int)losers[p];
      const float w = weights ? weights[p] : 1.0f;
      if (w == 0.0f) {
        s.zero_pairs[z++] = (int)p;
        continue;
      }
      sorted[c[a / range]++] = {a, {b, (int)p}, w};
      sorted[c[b / range]++] = {b, {a | (int)0x80000000, (int)p}, w};
    }
  }
  const int from = pairs_long_from(total, ni), huge_from = std::max(kHugeItem, from);
  std::vector<long long> n_long(kRanges + 1, 0), n_huge(kRanges + 1, 0);
#pragma omp parallel for schedule(dynamic, 1) if (parts > 1)
  for (int q = 0; q < kRanges; ++q) {
    const long long i0 = std::min(ni, q * range), i1 = std::min(ni, i0 + range);
    if (i0 >= i1) continue;
    // the range's offsets count its items' entries, then say where each item's
    // next entry goes, and are put back at the end
    int* const at = &s.offsets[i0];
    int2* const entries = s.entries.get();
    float* const entry_w = s.weights.get();
    const Entry* const first = &sorted[start[q]];
    const Entry* const last = first + (start[q + 1] - start[q]);
    std::fill(at, at + (i1 - i0), 0);
    for (const Entry* e = first; e < last; ++e) ++at[e->item - i0];
    int sum = (int)start[q];
    for (long long i = 0; i < i1 - i0; ++i) {
      const int n = at[i];
      at[i] = sum;
      sum += n;
      if (n >= from) ++(n >= huge_from ? n_huge : n_long)[q];
    }
    for (const Entry* e = first; e < last; ++e) {
      const int to = at[e->item - i0]++;
      entries[to] = e->e;
      if (entry_w) entry_w[to] = e->w;
    }
    for (long long i = i1 - i0 - 1; i > 0; --i) at[i] = at[i - 1];
    at[0] = (int)start[q];
  }
  s.offsets[ni] = (int)total;
  auto places = [](std::vector<long long>& n) {  // from counts to where each range's begin
    long long sum = 0;
    for (long long& v : n) {
      const long long c = v;
      v = sum;
      sum += c;
    }
    return sum;
  };
  s.n_long = places(n_long);
  s.n_huge = places(n_huge);
  s.long_items.reset(new int[std::max(1ll, s.n_long)]);
  s.huge_items.reset(new int[std::max(1ll, s.n_huge)]);
  if (s.n_long + s.n_huge > 0) {
#pragma omp parallel for schedule(dynamic, 1) if (parts > 1)
    for (int q = 0; q < kRanges; ++q) {
      const long long i0 = std::min(ni, q * range), i1 = std::min(ni, i0 + range);
      long long l = n_long[q], h = n_huge[q];
      if (l == n_long[q + 1] && h == n_huge[q + 1]) continue;
      for (long long i = i0; i < i1; ++i) {
        const int n = s.offsets[i + 1] - s.offsets[i];
        if (n >= huge_from) s.huge_items[h++] = (int)i;
        else if (n >= from) s.long_items[l++] = (int)i;
      }
    }
  }
  return s;
}

}  // namespace mtb
