// The losses' row by row arithmetic, and what their kernels are given.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "feedback.h"
#include "feedback_math.cuh"

namespace mtb {
namespace {

// Per score type: C computes a row's exponentials, Row holds per-row values,
// Out the derivatives.  float64 scores are computed in float64 throughout and
// narrowed to float32 derivatives, as the trainer's other objectives are;
// 16-bit scores are widened to float32 and only the stored derivatives are
// rounded back.
template <typename T>
struct Types {
  using C = float;
  using Row = float;
  using Out = T;
};
template <>
struct Types<double> {
  using C = double;
  using Row = double;
  using Out = float;
};

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void narrow(double v, float& o) { o = (float)v; }
__device__ __forceinline__ void narrow(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T>
struct RowPointers {
  const T* scores;
  const int* actions32;
  const long long* actions64;
  long long n, stride;
  int K;
  __device__ __forceinline__ long long action(long long r) const {
    return actions64 ? actions64[r] : (long long)actions32[r];
  }
};

template <typename T>
struct OutPointers {
  typename Types<T>::Out* grad;
  typename Types<T>::Out* hess;
  long long row_stride, class_stride;
};

template <typename T>
struct PolicyPointers {
  using Row = typename Types<T>::Row;
  const Row *advantages, *old_logp, *ref_logp, *weights;
  double log_low, log_high;    // log of the clip range's ends
  double clip_low, clip_high;  // the ends
  double kl;
  Row *loss, *logp;
};

// The gradient on l jumps at the ends of the clip range, so there l has to be
// right beyond the accuracy of a float32 sum: a row whose log ratio is this
// near to an end sums its exponentials again in float64.  A float32 sum of
// exponentials adds at most `adds` of them one after the other (2^-24 each),
// and each is off by (2 + 1.173 |d|) 2^-23 for d = z - m (__expf's documented
// bound), d itself by |d| 2^-24; weighted by the probabilities |d| averages
// below log K <= 12.5.
__host__ __device__ constexpr double border_slack(int adds, double log_k) {
  return 1.1 * (adds * 0x1p-24 + (2.0 + 1.173 * log_k) * 0x1p-23 + log_k * 0x1p-24);
}

struct RowDerivative {
  double g, h;
};

// Loss of a row with log probability l, and its derivatives in l.
template <typename T, typename Exp>
__device__ __forceinline__ RowDerivative policy_terms(const PolicyPointers<T>& t, double l, double adv, double old,
                                                      double ref, double w, double* loss, Exp exp_f) {
  const double d = l - old;
  const double ra = exp_f(d) * adv;
  const bool active = adv >= 0.0 ? d <= t.log_high : d >= t.log_low;
  double v = active ? -ra : (adv >= 0.0 ? -t.clip_high * adv : -t.clip_low * adv);
  double g = active ? -ra : 0.0;
  if (ra != ra) v = g = ra;
  double h = g > 0.0 ? g : 0.0;
  if (t.ref_logp) {
    const double e = exp_f(ref - l);
    v += t.kl * (e - 1.0 - (ref - l));
    g -= t.kl * (e - 1.0);
    h += t.kl * e;
  }
  *loss = w * v;
  return {w * g, w * h};
}

// Whether the float32 sum leaves open on which side of an end of the clip
// range the row lies.
template <typename T>
__device__ __forceinline__ bool near_border(const PolicyPointers<T>& t, double d, double adv, double slack) {
  return fabs(d - (adv >= 0.0 ? t.log_high : t.log_low)) < slack;
}

enum RowOp : int { ROW_LOGPROBS = 0, ROW_BACK = 1, ROW_POLICY = 2 };

template <typename T>
struct RowArgs {
  RowPointers<T> in;
  OutPointers<T> out;
  PolicyPointers<T> pol;
  typename Types<T>::Row* logp;         // ROW_LOGPROBS
  typename Types<T>::Row* stats;        // ROW_LOGPROBS (written), ROW_BACK (read)
  const float *grad_logp, *hess_logp;   // ROW_BACK
};

}  // namespace
}  // namespace mtb
