// C entry points of the losses from feedback (declared in include/mojotrees.h).
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <memory>
#include <stdexcept>
#include <string>

#include "../../include/mojotrees.h"
#include "capi_util.h"
#include "feedback.h"
#include "trainer.h"

struct MojoTreesPreferencePlan {
  mtb::PreferencePlan plan;
};

namespace {

using mtb::Unsupported;

template <typename F>
int32_t checked(MojoTreesError* error, F&& fn) {
  mtb::capi_clear_error(error);
  try {
    fn();
    return MOJOTREES_OK;
  } catch (const std::invalid_argument& e) {
    mtb::capi_set_error(error, e.what());
    return MOJOTREES_ERROR_INVALID_ARGUMENT;
  } catch (const Unsupported& e) {
    mtb::capi_set_error(error, e.what());
    return MOJOTREES_ERROR_UNSUPPORTED;
  } catch (const std::exception& e) {
    mtb::capi_set_error(error, e.what());
    return MOJOTREES_ERROR_TRAINING;
  }
}

void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

void require_cuda() {
  if (mtb::cuda_device_count() < 1) throw Unsupported("no CUDA device is available");
}

void check(cudaError_t e) {
  if (e != cudaSuccess) throw std::runtime_error(std::string("CUDA error: ") + cudaGetErrorString(e));
}

// Makes a device current for a call, and the caller's again after it.
struct DeviceScope {
  int before = -1;
  bool moved = false;
  explicit DeviceScope(int dev) {
    check(cudaGetDevice(&before));
    if (dev >= 0 && dev != before) {
      check(cudaSetDevice(dev));
      moved = true;
    }
  }
  ~DeviceScope() {
    if (moved) cudaSetDevice(before);
  }
};

// The device that holds `p`; every array of a call has to be there.
int device_of(const void* p) {
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    throw std::invalid_argument("array is not in device memory");
  }
  require(a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged, "array is not in device memory");
  return a.device;
}

void require_aligned(int bytes, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays) require((uintptr_t)p % bytes == 0, "array is not aligned to its element size");
}

int common_device(std::initializer_list<const void*> arrays) {
  int dev = -1;
  for (const void* p : arrays) {
    if (!p) continue;
    const int d = device_of(p);
    require(dev < 0 || d == dev, "arrays of one call are on different devices");
    dev = d;
  }
  return dev;
}

// Element sizes by score type: scores, per-row values, derivatives.
int score_bytes(int32_t type) { return type == mtb::SCORE_F64 ? 8 : type == mtb::SCORE_F32 ? 4 : 2; }
int row_bytes(int32_t type) { return type == mtb::SCORE_F64 ? 8 : 4; }
int out_bytes(int32_t type) { return std::min(score_bytes(type), 4); }

mtb::ScoreRows score_rows(const void* scores, int32_t type, int64_t n_rows, int64_t n_classes, int64_t stride,
                          const void* actions, int32_t action_bytes) {
  require(type >= mtb::SCORE_F64 && type <= mtb::SCORE_BF16, "unknown score type");
  require(n_rows >= 0, "n_rows must be non-negative");
  require(n_classes >= 1 && n_classes <= mtb::kMaxClasses, "n_classes must be in [1, 262144]");
  require(stride >= n_classes, "row_stride must be at least n_classes");
  require(n_rows == 0 || stride <= (int64_t)1 << 46 && n_rows <= ((int64_t)1 << 46) / stride, "scores are too large");
  require(action_bytes == 4 || action_bytes == 8, "actions must be 4 or 8 byte integers");
  require(n_rows == 0 || (scores && actions), "null pointer argument");
  require_aligned(score_bytes(type), {scores});
  require_aligned(action_bytes, {actions});
  return {scores, type, n_rows, (int)n_classes, stride, actions, action_bytes == 8};
}

mtb::ScoreDerivatives derivatives(void* grad, void* hess, int64_t n_rows, int64_t n_classes, int64_t stride) {
  require(stride >= n_classes, "out_stride must be at least n_classes");
  require(n_rows == 0 || stride <= (int64_t)1 << 46 && n_rows <= ((int64_t)1 << 46) / stride, "derivatives are too large");
  return {grad, hess, stride, 1};
}

}  // namespace

extern "C" {

int32_t mojotrees_b200_action_logprobs(const void* scores, int32_t score_type, int64_t n_rows, int64_t n_classes,
                                       int64_t row_stride, const void* actions, int32_t action_bytes, void* out_logp,
                                       void* out_stats, void* stream, MojoTreesError* error) {
  return checked(error, [&] {
    const mtb::ScoreRows in = score_rows(scores, score_type, n_rows, n_classes, row_stride, actions, action_bytes);
    require(n_rows == 0 || (out_logp && out_stats), "null pointer argument");
    require_aligned(row_bytes(score_type), {out_logp, out_stats});
    require_cuda();
    if (n_rows == 0) return;
    DeviceScope on(common_device({scores, actions, out_logp, out_stats}));
    mtb::launch_logprobs(in, out_logp, out_stats, static_cast<cudaStream_t>(stream));
  });
}

int32_t mojotrees_b200_action_logprobs_grad(const void* scores, int32_t score_type, int64_t n_rows, int64_t n_classes,
                                            int64_t row_stride, const void* actions, int32_t action_bytes,
                                            const void* stats, const float* grad_logp, const float* hess_logp,
                                            void* out_grad, void* out_hess, int64_t out_stride, void* stream,
                                            MojoTreesError* error) {
  return checked(error, [&] {
    const mtb::ScoreRows in = score_rows(scores, score_type, n_rows, n_classes, row_stride, actions, action_bytes);
    require(n_rows == 0 || (stats && grad_logp && out_grad), "null pointer argument");
    require(!hess_logp == !out_hess, "hess_logp and out_hess go together");
    require_aligned(row_bytes(score_type), {stats});
    require_aligned(4, {grad_logp, hess_logp});
    require_aligned(out_bytes(score_type), {out_grad, out_hess});
    const mtb::ScoreDerivatives out = derivatives(out_grad, out_hess, n_rows, n_classes, out_stride);
    require_cuda();
    if (n_rows == 0) return;
    DeviceScope on(common_device({scores, actions, stats, grad_logp, hess_logp, out_grad, out_hess}));
    mtb::launch_logprobs_grad(in, stats, grad_logp, hess_logp, out, static_cast<cudaStream_t>(stream));
  });
}

int32_t mojotrees_b200_policy_loss(const void* scores, int32_t score_type, int64_t n_rows, int64_t n_classes,
                                   int64_t row_stride, const void* actions, int32_t action_bytes,
                                   const void* advantages, const void* old_logp, const void* ref_logp,
                                   const void* weights, double clip_low, double clip_high, double kl_coef,
                                   void* out_loss, void* out_logp, void* out_grad, void* out_hess, int64_t out_stride,
                                   void* stream, MojoTreesError* error) {
  return checked(error, [&] {
    const mtb::ScoreRows in = score_rows(scores, score_type, n_rows, n_classes, row_stride, actions, action_bytes);
    require(n_rows == 0 || (advantages && old_logp && out_loss), "null pointer argument");
    require(clip_low >= 0.0 && clip_low <= 1.0, "clip_low must be in [0, 1]");
    require(clip_high >= 0.0, "clip_high must be non-negative");
    require(kl_coef >= 0.0 && std::isfinite(kl_coef), "kl_coef must be finite and non-negative");
    require(kl_coef == 0.0 || ref_logp || n_rows == 0, "kl_coef needs ref_logp");
    require(out_grad || !out_hess, "out_hess needs out_grad");
    require_aligned(row_bytes(score_type), {advantages, old_logp, ref_logp, weights, out_loss, out_logp});
    require_aligned(out_bytes(score_type), {out_grad, out_hess});
    const mtb::ScoreDerivatives out =
        out_grad ? derivatives(out_grad, out_hess, n_rows, n_classes, out_stride) : mtb::ScoreDerivatives{};
    require_cuda();
    if (n_rows == 0) return;
    DeviceScope on(common_device({scores, actions, advantages, old_logp, ref_logp, weights, out_loss, out_logp,
                                  out_grad, out_hess}));
    const mtb::PolicyTerms t = {advantages, old_logp, kl_coef > 0.0 ? ref_logp : nullptr, weights, clip_low,
                                clip_high, kl_coef, out_loss, out_logp};
    mtb::launch_policy(in, t, out, static_cast<cudaStream_t>(stream));
  });
}

int32_t mojotrees_b200_preference_plan_create(const int64_t* winners, const int64_t* losers, const float* weights,
                                              int64_t n_pairs, int64_t n_items, int32_t gpu_device_id,
                                              MojoTreesPreferencePlan** out_plan, MojoTreesError* error) {
  return checked(error, [&] {
    require(out_plan, "null pointer argument");
    require(n_pairs >= 0 && n_items >= 0, "n_pairs and n_items must be non-negative");
    require(n_items < (int64_t)1 << 31, "more than 2^31-1 items");
    require(n_pairs < (int64_t)1 << 29, "more than 2^29-1 pairs");  // entry numbers and steps beyond them fit 32 bits
    require(n_pairs == 0 || (winners && losers), "null pointer argument");
    mtb::PreferencePlan::check(winners, losers, weights, n_pairs, n_items);
    require_cuda();
    require(gpu_device_id < mtb::cuda_device_count(), "gpu_device_id out of range");
    DeviceScope on(gpu_device_id);
    std::unique_ptr<MojoTreesPreferencePlan> h(new MojoTreesPreferencePlan());
    h->plan.build(winners, losers, weights, n_pairs, n_items);
    *out_plan = h.release();
  });
}

void mojotrees_b200_preference_plan_free(MojoTreesPreferencePlan* plan) { delete plan; }

int32_t mojotrees_b200_preference_loss(const MojoTreesPreferencePlan* plan, const void* scores, const void* reference,
                                       int32_t score_type, double beta, double label_smoothing, int32_t loss_kind,
                                       void* out_loss, float* out_grad, float* out_hess, void* stream,
                                       MojoTreesError* error) {
  return checked(error, [&] {
    require(plan, "null pointer argument");
    require(score_type == mtb::SCORE_F64 || score_type == mtb::SCORE_F32, "preference scores are float64 or float32");
    require(beta > 0.0 && std::isfinite(beta), "beta must be positive");
    require(score_type == mtb::SCORE_F64 || beta <= FLT_MAX, "beta is beyond float32 scores");
    require(label_smoothing >= 0.0 && label_smoothing <= 0.5, "label_smoothing must be in [0, 0.5]");
    require(loss_kind == mtb::PREFERENCE_LOGISTIC || loss_kind == mtb::PREFERENCE_SQUARED, "unknown preference loss");
    const mtb::PreferencePlan& p = plan->plan;
    require(p.n_items == 0 || scores, "null pointer argument");
    require(!out_grad == !out_hess, "out_grad and out_hess go together");
    require_aligned(score_bytes(score_type), {scores, reference, out_loss});
    require_aligned(4, {out_grad, out_hess});
    require_cuda();
    if (p.n_items == 0) return;
    const int dev = common_device({scores, reference, out_loss, out_grad, out_hess});
    require(dev == p.device, "arrays are not on the plan's device");
    DeviceScope on(dev);
    const mtb::PreferenceTerms t = {scores, reference, score_type, beta, label_smoothing, loss_kind, out_loss,
                                    out_grad, out_hess};
    mtb::launch_preference(p, t, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
