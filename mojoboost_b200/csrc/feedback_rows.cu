// Losses of one row's scores that learn from feedback instead of labels: log
// probabilities of taken classes and the clipped policy loss, each with its
// gradient and hessian.
//
// With z a row's scores, a the class it took, p = softmax(z):
//   log probability  l = z_a - m - log sum exp(z - m), m = max z
//   back to scores   G_k = g ([k = a] - p_k)
//                    H_k = h ([k = a] - p_k)^2 + |g| p_k (1 - p_k)
// for g = dL/dl, h = d2L/dl2.  H is the diagonal of the Hessian with the
// curvature of l, -p_k (1 - p_k), taken with weight |g| instead of -g, so it
// is never negative; for cross entropy (g = -1, h = 0) it is p_k (1 - p_k).
//
// A row takes no part when its class is negative, its weight is 0 or every
// score is -inf (all classes masked), and for the policy loss when the class
// it took is masked: its outputs are 0, whatever else the row holds.  A class
// of n_classes or more gives NaN in that row.
#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "feedback_large.cuh"
#include "feedback_small.cuh"

namespace mtb {
namespace {

// ---------------------------------------------------------------------------
// float64 scores of more than 512 classes, which only callers with scores of
// their own have (a fit has 64 classes at most), stay with the simplest kernel:
// three passes, the later ones out of L2.  2000 x 2000: log probabilities 21 us
// (5 at the copy rate), their gradient 19 (7), the policy loss with gradient 40
// (7); 200 x 50000: 172 (18).  Bound is the latency of 256 threads' passes.
// ---------------------------------------------------------------------------

constexpr int kRowThreads = 256;

__device__ __forceinline__ double add_f64(double a, double b) { return a + b; }

__device__ __forceinline__ double max_f64(double a, double b) { return (b > a || b != b) ? b : a; }  // NaN when either is

template <typename F>
__device__ __forceinline__ double block_reduce(double v, double* sm, F f) {
  for (int k = 16; k > 0; k >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, k));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int i = 1; i < kRowThreads / 32; ++i) v = f(v, sm[i]);
  return v;
}

// One block per row: the maximum, the sum, the derivatives, each a pass over
// the row.
template <int OP>
__global__ void __launch_bounds__(kRowThreads) k_feedback_rows(const RowArgs<double> A) {
  __shared__ double sm[kRowThreads / 32];
  const int K = A.in.K;
  for (long long r = blockIdx.x; r < A.in.n; r += gridDim.x) {
    const double* z = A.in.scores + r * A.in.stride;
    const long long a = A.in.action(r);
    const bool bad = a >= K;
    bool part = a >= 0;
    if (OP == ROW_POLICY && A.pol.weights) part = part && A.pol.weights[r] != 0.0;
    double m = 0.0, rest = -1.0;
    if (OP == ROW_BACK) {
      m = A.stats[2 * r];
      rest = A.stats[2 * r + 1];
      part = part && rest != -1.0;
    } else if (part && !bad) {
      double mx = -INFINITY;
      for (int k = threadIdx.x; k < K; k += kRowThreads) mx = max_f64(mx, z[k]);
      mx = block_reduce(mx, sm, max_f64);
      if (mx == -INFINITY) {
        part = false;
      } else {
        m = mx;
        double s = 0.0, ties = 0.0;
        for (int k = threadIdx.x; k < K; k += kRowThreads) {
          const double e = exp(z[k] - m);
          if (e != 1.0) s += e;
          else ties += 1.0;
        }
        s = block_reduce(s, sm, add_f64);
        rest = s + (block_reduce(ties, sm, add_f64) - 1.0);
      }
    }
    RowDerivative row = {0.0, 0.0};
    double l = 0.0, loss = 0.0;
    if (OP == ROW_BACK) {
      if (part) row = {(double)A.grad_logp[r], A.hess_logp ? (double)A.hess_logp[r] : 0.0};
    } else if (part && bad) {
      l = loss = NAN;
    } else if (part) {
      l = z[a] - m - log1p(rest);
      if (OP == ROW_POLICY) {
        part = z[a] != -INFINITY;  // the class taken is masked
        if (part)
          row = policy_terms(A.pol, l, A.pol.advantages[r], A.pol.old_logp[r], A.pol.ref_logp ? A.pol.ref_logp[r] : 0.0,
                             A.pol.weights ? A.pol.weights[r] : 1.0, &loss, [](double d) { return exp(d); });
      }
    }
    if (OP == ROW_LOGPROBS && threadIdx.x == 0) {
      A.logp[r] = l;
      A.stats[2 * r] = part && bad ? NAN : m;
      A.stats[2 * r + 1] = part && bad ? NAN : part ? rest : -1.0;
    }
    if (OP == ROW_POLICY && threadIdx.x == 0) {
      if (A.pol.loss) A.pol.loss[r] = loss;
      if (A.pol.logp) A.pol.logp[r] = l;
    }
    if (OP != ROW_LOGPROBS && A.out.grad) {
      float* gp = A.out.grad + r * A.out.row_stride;
      float* hp = A.out.hess ? A.out.hess + r * A.out.row_stride : nullptr;
      const double inv = 1.0 / (1.0 + rest), share = rest / (1.0 + rest);
      for (int k = threadIdx.x; k < K; k += kRowThreads) {
        double g = part && bad ? NAN : 0.0, h = g;
        if (part && !bad) {
          const double e = exp(z[k] - m), p = e * inv, left = e == 1.0 ? share : 1.0 - p, q = k == a ? left : -p;
          g = row.g * q;
          h = row.h * q * q + fabs(row.g) * p * left;
        }
        gp[k * A.out.class_stride] = (float)g;
        if (hp) hp[k * A.out.class_stride] = (float)h;
      }
    }
    __syncthreads();
  }
}

template <typename T, int OP>
void launch_rows_t(const RowArgs<T>& A, cudaStream_t st) {
  if (A.in.n == 0) return;
  if (A.in.K <= kSmallClasses<T>) {
    launch_small<T, OP>(A, st);
    MTB_CUDA_FB(cudaGetLastError());
    return;
  }
  if constexpr (sizeof(T) == 8) {
    k_feedback_rows<OP><<<(unsigned)std::min<long long>(A.in.n, 1 << 20), kRowThreads, 0, st>>>(A);
    MTB_CUDA_FB(cudaGetLastError());
  } else {
    launch_large<T, OP>(A, st);
  }
}

template <typename T>
RowArgs<T> row_args(const ScoreRows& in) {
  RowArgs<T> A = {};
  A.in.scores = static_cast<const T*>(in.scores);
  (in.actions64 ? (const void*&)A.in.actions64 : (const void*&)A.in.actions32) = in.actions;
  A.in.n = in.n;
  A.in.K = in.K;
  A.in.stride = in.stride;
  return A;
}

template <typename T>
void set_out(RowArgs<T>& A, const ScoreDerivatives& out) {
  using Out = typename Types<T>::Out;
  A.out = {static_cast<Out*>(out.grad), static_cast<Out*>(out.hess), out.row_stride, out.class_stride};
}

template <typename F>
void by_type(int type, F&& f) {
  switch (type) {
    case SCORE_F64: f((double*)nullptr); break;
    case SCORE_F32: f((float*)nullptr); break;
    case SCORE_F16: f((__half*)nullptr); break;
    case SCORE_BF16: f((__nv_bfloat16*)nullptr); break;
    default: throw std::invalid_argument("unknown score type");
  }
}

}  // namespace

int launch_logprobs(const ScoreRows& in, void* logp, void* stats, cudaStream_t st) {
  by_type(in.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RowArgs<T> A = row_args<T>(in);
    A.logp = static_cast<typename Types<T>::Row*>(logp);
    A.stats = static_cast<typename Types<T>::Row*>(stats);
    launch_rows_t<T, ROW_LOGPROBS>(A, st);
  });
  return in.n > 0 ? 1 : 0;
}

int launch_logprobs_grad(const ScoreRows& in, const void* stats, const float* grad_logp, const float* hess_logp,
                          const ScoreDerivatives& out, cudaStream_t st) {
  by_type(in.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    RowArgs<T> A = row_args<T>(in);
    A.stats = const_cast<typename Types<T>::Row*>(static_cast<const typename Types<T>::Row*>(stats));
    A.grad_logp = grad_logp;
    A.hess_logp = hess_logp;
    set_out(A, out);
    launch_rows_t<T, ROW_BACK>(A, st);
  });
  return in.n > 0 ? 1 : 0;
}

int launch_policy(const ScoreRows& in, const PolicyTerms& t, const ScoreDerivatives& out, cudaStream_t st) {
  by_type(in.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    using Row = typename Types<T>::Row;
    RowArgs<T> A = row_args<T>(in);
    A.pol.advantages = static_cast<const Row*>(t.advantages);
    A.pol.old_logp = static_cast<const Row*>(t.old_logp);
    A.pol.ref_logp = static_cast<const Row*>(t.ref_logp);
    A.pol.weights = static_cast<const Row*>(t.weights);
    A.pol.log_low = log1p(-t.clip_low);
    A.pol.log_high = log1p(t.clip_high);
    A.pol.clip_low = 1.0 - t.clip_low;
    A.pol.clip_high = 1.0 + t.clip_high;
    A.pol.kl = t.kl_coef;
    A.pol.loss = static_cast<Row*>(t.loss);
    A.pol.logp = static_cast<Row*>(t.logp);
    set_out(A, out);
    launch_rows_t<T, ROW_POLICY>(A, st);
  });
  return in.n > 0 ? 1 : 0;
}

}  // namespace mtb
