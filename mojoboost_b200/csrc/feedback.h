// Losses that learn from feedback instead of labels: the clipped policy loss
// of logged decisions, the paired preference loss, and the log probabilities
// of taken classes that both start from.  Launchers shared by the C entry
// points (feedback_api.cpp) and the trainer.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace mtb {

enum ScoreType : int { SCORE_F64 = 0, SCORE_F32 = 1, SCORE_F16 = 2, SCORE_BF16 = 3 };
enum PreferenceKind : int { PREFERENCE_LOGISTIC = 0, PREFERENCE_SQUARED = 1 };

// Most classes of a row: what a cluster's registers hold in float32.
constexpr long long kMaxClasses = 1 << 18;

// Scores [n][K] (rows `stride` elements apart, classes next to each other)
// and the class each row took.  All pointers are device memory.
struct ScoreRows {
  const void* scores;
  int type;  // ScoreType
  long long n;
  int K;
  long long stride;
  const void* actions;  // int32 or int64
  bool actions64;
};

// Derivatives with respect to the scores: element (r, k) at r * row_stride +
// k * class_stride; float for float64 and float32 scores, else the scores'
// type.  hess may be null.
struct ScoreDerivatives {
  void* grad;
  void* hess;
  long long row_stride;
  long long class_stride;
};

struct PolicyTerms {
  const void* advantages;  // double for float64 scores, else float; as all per-row arrays here
  const void* old_logp;
  const void* ref_logp;    // null: no KL term
  const void* weights;     // null: 1
  double clip_low, clip_high, kl_coef;
  void* loss;  // may be null
  void* logp;  // may be null
};

// Each launcher returns how many kernels it launched.
int launch_logprobs(const ScoreRows& in, void* logp, void* stats, cudaStream_t st);
int launch_logprobs_grad(const ScoreRows& in, const void* stats, const float* grad_logp, const float* hess_logp,
                          const ScoreDerivatives& out, cudaStream_t st);
// out.grad null: the loss alone.
int launch_policy(const ScoreRows& in, const PolicyTerms& t, const ScoreDerivatives& out, cudaStream_t st);

// The pairs of a preference loss, laid out on a device per item, so that an
// item's derivatives are one sum in a fixed order (no atomics).
struct PreferencePlan {
  int device = 0;
  long long n_items = 0, n_pairs = 0, n_entries = 0;
  // Device arrays, all in `memory`.  Pairs of weight 0 have no entries.
  int* offsets = nullptr;    // [n_items + 1] into the entries
  int2* entries = nullptr;   // [n_entries] the other item, sign bit set where this item lost; the pair
  float* entry_w = nullptr;  // [n_entries] weights, or null
  int* zero_pairs = nullptr;  // pairs of weight 0
  int* long_items = nullptr;  // items of many pairs, and of very many
  int* huge_items = nullptr;
  long long n_zero = 0, n_long = 0, n_huge = 0;
  void* memory = nullptr;
  size_t memory_bytes = 0;
  PreferencePlan() = default;
  PreferencePlan(const PreferencePlan&) = delete;
  PreferencePlan& operator=(const PreferencePlan&) = delete;
  ~PreferencePlan();
  // Throws std::invalid_argument for an item out of range, an item paired
  // with itself, or a weight that is negative or not finite.
  static void check(const int64_t* winners, const int64_t* losers, const float* weights, long long n_pairs,
                    long long n_items);
  // Host arrays that passed check().  Allocates on the current device and
  // waits for the copies.
  void build(const int64_t* winners, const int64_t* losers, const float* weights, long long n_pairs,
             long long n_items);
};

struct PreferenceTerms {
  const void* scores;     // double or float [n_items]
  const void* reference;  // same type, or null
  int type;               // SCORE_F64 or SCORE_F32
  double beta, smoothing;
  int kind;      // PreferenceKind
  void* loss;    // [n_pairs] in the scores' type, or null
  float* grad;   // [n_items]
  float* hess;   // [n_items]
};

int launch_preference(const PreferencePlan& plan, const PreferenceTerms& t, cudaStream_t st);

}  // namespace mtb
