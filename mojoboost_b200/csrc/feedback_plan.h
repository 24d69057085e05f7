// The host's part of a preference plan: the pairs listed item by item.
#pragma once
#include <stdint.h>
#include <vector_types.h>

#include <memory>

namespace mtb {

// Lanes an item, by the mean number of an item's pairs: about eight steps of a
// lane, so that an item's own loads, sums of lanes and stores are shared by
// few instructions (all pairs in groups of 64, float64: 53 us with 32 lanes,
// 41 us with 8).
inline int pair_lanes(long long mean) { return mean < 8 ? 1 : mean < 32 ? 4 : mean < 128 ? 8 : 32; }

// Items of more pairs than their lanes take in 24 steps have a block to
// themselves, or from 2048 pairs a cluster of 8: a lane's steps are one after
// the other, and a long item in a warp would be the last to end.  Pairs of
// popular items, 12, 24 and 48 steps: 100000 of 3000 float32 items 20.6, 21.0,
// 30.0 us; 1M of 20000 float64 48, 46, 52; 4M of 300001 float32 122, 130, 131.
// Clusters from 512, 2048 and 8192 pairs: 21.3, 21.0, 21.1; 58, 46, 47; 152,
// 130, 118.
inline int pairs_long_from(long long n_entries, long long n_items) {
  return 24 * pair_lanes(n_entries / (n_items > 1 ? n_items : 1)) + 1;
}
constexpr int kHugeItem = 2048;

struct SortedPairs {
  long long n_entries = 0, n_zero = 0, n_long = 0, n_huge = 0;
  std::unique_ptr<int[]> offsets;    // [n_items + 1] into the entries
  std::unique_ptr<int2[]> entries;   // the other item, sign bit set where this item lost; the pair
  std::unique_ptr<float[]> weights;  // of the entries; null without weights
  std::unique_ptr<int[]> zero_pairs, long_items, huge_items;
};

// Pairs that passed PreferencePlan::check; an item's entries in the pairs'
// order.  Throws std::bad_alloc.
SortedPairs sort_pairs(const int64_t* winners, const int64_t* losers, const float* weights, long long n_pairs,
                       long long n_items);

}  // namespace mtb
