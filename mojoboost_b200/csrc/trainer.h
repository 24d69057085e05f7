// GPU trainer entry point (host side).
#pragma once
#include <stddef.h>

#include <stdexcept>
#include <string>

#include "model.h"

namespace mtb {

// A request the device path does not cover (maps to MOJOTREES_ERROR_UNSUPPORTED).
struct Unsupported : std::runtime_error {
  explicit Unsupported(const std::string& m) : std::runtime_error(m) {}
};

struct BinMapper;

// What the objectives preference and policy learn from, in place of labels.
// Host arrays, checked by the caller; per-row ones have n_rows values, and
// null ones the meaning given here.
struct Feedback {
  const int32_t* actions = nullptr;  // class each row took (null: one score per row); policy: -1 takes no part
  const double* initial = nullptr;   // [n_rows][num_class] raw scores to start from (null: 0)
  // policy
  const double* advantages = nullptr;
  const double* old_logp = nullptr;  // null: under the initial scores
  const double* ref_logp = nullptr;  // null: under the initial scores
  const double* weights = nullptr;   // null: 1
  // preference: rows winners[p] preferred to rows losers[p]
  const int64_t* winners = nullptr;
  const int64_t* losers = nullptr;
  const float* pair_weights = nullptr;  // null: 1
  int64_t n_pairs = 0;
  const double* reference = nullptr;  // a reference model's scores or log probabilities (null: 0)
};

struct BinnedInput {
  const uint8_t* bins_fm;   // feature-major bins[f * n_rows + r], host memory
  long long n_rows;
  int n_features;
  int n_bins;               // histogram width (<= 256)
  const int* missing_bin;   // [n_features], -1 when none
  const int* n_cats;        // [n_features], -1 numeric, else kept categories
  const double* labels;     // [n_rows]
  // Data-parallel fits (one process per GPU): this device's rows are global
  // rows [row_offset, row_offset + n_rows); every shard but the last holds a
  // multiple of 1024 rows.  coll == nullptr for a single-device fit.
  long long row_offset = 0;
  long long n_rows_global = 0;
  class Collective* coll = nullptr;
  // Dense entry point: instead of bins_fm, float64 columns dense_fm[f * n_rows
  // + r] (host memory) binned on the device with `mapper`.
  const double* dense_fm = nullptr;
  const BinMapper* mapper = nullptr;
  // Set for the objectives that learn from feedback; labels is null then.
  const Feedback* feedback = nullptr;
};

// Trains on the current (or configured) CUDA device; fills model.trees,
// base_scores and stats.  Throws Unsupported or std::runtime_error.
void train_gpu(const BinnedInput& in, const TrainConfig& cfg, Model& model);

// Device memory of the per-process cache that fits take theirs from, on the
// current device: `bytes` becomes the size of the block, 2 MB at least, which
// it is returned with.  Returning a block, on the device it came from, waits
// for the device's work.
void* take_device_memory(size_t* bytes);
void give_device_memory(void* p, size_t bytes);

// Number of CUDA devices visible (0 when the driver or a device is absent).
int cuda_device_count();

}  // namespace mtb
