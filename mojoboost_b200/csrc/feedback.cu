// Losses that learn from feedback instead of labels, each with its gradient
// and hessian: kernels, launchers and C entry points.
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
#include "feedback.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <memory>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/mojotrees.h"
#include "capi_util.h"
#include "trainer.h"

namespace mtb {
namespace {

#define MTB_CUDA_FB(call)                                                                    \
  do {                                                                                       \
    cudaError_t e_ = (call);                                                                 \
    if (e_ != cudaSuccess)                                                                   \
      throw std::runtime_error(std::string("CUDA error: ") + cudaGetErrorString(e_) + " at " \
                               + #call);                                                     \
  } while (0)

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

__device__ __forceinline__ double exp_c(double d) { return exp(d); }
__device__ __forceinline__ float exp_c(float d) { return __expf(d); }

// The larger of two values, NaN when either is.
template <typename C>
__device__ __forceinline__ C max_nan(C a, C b) {
  return (b > a || b != b) ? b : a;
}

// A row's softmax sum as sum exp(z - m) = 1 + rest: `rest` leaves out one
// class at the maximum, so it keeps its relative accuracy when one class has
// nearly all of the probability, and with it 1 - p of that class.
template <typename C>
struct RowSum {
  C m;
  double rest;
};

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

// Derivatives at class k from e = exp(z_k - m) and the row's sum.  e is 1 for
// a class at the maximum (or one so near to it that its term of the sum is 1).
template <typename C>
__device__ __forceinline__ void derivative(C e, C inv_total, C rest_share, bool taken, C g, C h, bool want_h, C* grad,
                                           C* hess) {
  const C p = e * inv_total;
  const C left = e == (C)1 ? rest_share : (C)1 - p;  // 1 - p
  const C q = taken ? left : -p;
  *grad = g * q;
  if (want_h) *hess = h * q * q + fabs(g) * p * left;
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

constexpr int kRowThreads = 256;

__device__ __forceinline__ double add_f64(double a, double b) { return a + b; }

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* sm, F f) {
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
template <typename T, int OP>
__global__ void __launch_bounds__(kRowThreads) k_feedback_rows(const RowArgs<T> A) {
  using C = typename Types<T>::C;
  using Row = typename Types<T>::Row;
  __shared__ C sm_c[kRowThreads / 32];
  __shared__ double sm_d[kRowThreads / 32];
  const int K = A.in.K;
  for (long long r = blockIdx.x; r < A.in.n; r += gridDim.x) {
    const T* z = A.in.scores + r * A.in.stride;
    const long long a = A.in.action(r);
    const bool bad = a >= K;
    bool part = a >= 0;
    if (OP == ROW_POLICY && A.pol.weights) part = part && A.pol.weights[r] != (Row)0;
    C m = 0;
    double rest = -1.0;
    if (OP == ROW_BACK) {
      m = A.stats[2 * r];
      rest = (double)A.stats[2 * r + 1];
      part = part && rest != -1.0;
    } else if (part && !bad) {
      C mx = -INFINITY;
      for (int k = threadIdx.x; k < K; k += kRowThreads) mx = max_nan<C>(mx, widen(z[k]));
      mx = block_reduce(mx, sm_c, max_nan<C>);
      if (mx == (C)-INFINITY) {
        part = false;
      } else {
        m = mx;
        C s = 0;
        int ties = 0;
        for (int k = threadIdx.x; k < K; k += kRowThreads) {
          const C e = exp_c((C)widen(z[k]) - m);
          if (e != (C)1) s += e;
          else ++ties;
        }
        const double others = block_reduce((double)s, sm_d, add_f64);
        rest = others + (block_reduce((double)ties, sm_d, add_f64) - 1.0);
      }
    }
    RowDerivative row = {0.0, 0.0};
    if (OP == ROW_LOGPROBS) {
      if (threadIdx.x == 0) {
        const double l = part ? (bad ? (double)NAN : (double)widen(z[a]) - (double)m - log1p(rest)) : 0.0;
        A.logp[r] = (Row)l;
        A.stats[2 * r] = part && bad ? (Row)NAN : (Row)m;
        A.stats[2 * r + 1] = part ? (bad ? (Row)NAN : (Row)rest) : (Row)-1;
      }
      __syncthreads();
      continue;
    } else if (OP == ROW_BACK) {
      row = {part ? (double)A.grad_logp[r] : 0.0, part && A.hess_logp ? (double)A.hess_logp[r] : 0.0};
    } else {
      double l = 0.0, loss = 0.0;
      if (part && bad) {
        l = loss = row.g = row.h = NAN;
      } else if (part) {
        const double za = (double)widen(z[a]);
        l = za - (double)m - log1p(rest);
        if (za == -INFINITY) {
          part = false;
        } else {
          const double adv = (double)A.pol.advantages[r], old = (double)A.pol.old_logp[r];
          if (sizeof(C) == 4 && near_border(A.pol, l - old, adv, border_slack(kMaxClasses / kRowThreads + 16, 12.5))) {
            double s = 0.0;
            for (int k = threadIdx.x; k < K; k += kRowThreads) s += exp((double)widen(z[k]) - (double)m);
            l = za - (double)m - log(block_reduce(s, sm_d, add_f64));
          }
          row = policy_terms(A.pol, l, adv, old, A.pol.ref_logp ? (double)A.pol.ref_logp[r] : 0.0,
                             A.pol.weights ? (double)A.pol.weights[r] : 1.0, &loss,
                             [](double d) { return exp(d); });
        }
      }
      if (threadIdx.x == 0) {
        if (A.pol.loss) A.pol.loss[r] = (Row)loss;
        if (A.pol.logp) A.pol.logp[r] = (Row)l;
      }
    }
    if (OP == ROW_POLICY && !A.out.grad) {
      __syncthreads();
      continue;
    }
    auto* gp = A.out.grad + r * A.out.row_stride;
    auto* hp = A.out.hess ? A.out.hess + r * A.out.row_stride : nullptr;
    const C g = (C)row.g, h = (C)row.h, inv = (C)(1.0 / (1.0 + rest)), left = (C)(rest / (1.0 + rest));
    for (int k = threadIdx.x; k < K; k += kRowThreads) {
      C dg = 0, dh = 0;
      if (part && bad) dg = dh = (C)NAN;
      else if (part) derivative<C>(exp_c((C)widen(z[k]) - m), inv, left, k == a, g, h, hp != nullptr, &dg, &dh);
      narrow(dg, gp[k * A.out.class_stride]);
      if (hp) narrow(dh, hp[k * A.out.class_stride]);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Rows of up to 128 classes
//
// A warp copies 32 / L whole rows into shared memory, L lanes take a row each
// (class l + L e in lane l, at most 16 a lane), and the derivatives go back
// through the same memory, so every array crosses the memory system once and
// in one piece per warp.  With L = 1 (up to 16 classes) no lane waits for
// another.  A row's float64 scalars, a logarithm, two exponentials and a
// quotient, cost as much as ten classes; every lane of a row computes them.
// ---------------------------------------------------------------------------

constexpr int kSmallThreads = 128;
constexpr int kSmallPer = 16;  // classes a lane
constexpr int kSmallClasses = 8 * kSmallPer;

// exp and log1p in float64 by tables in shared memory and polynomials (P. T. P.
// Tang, "Table-driven implementation of the exponential function in IEEE
// floating-point arithmetic", ACM TOMS 15(2), 1989, and "... of the logarithm
// function ...", ACM TOMS 16(4), 1990): both without a branch, so that the
// work of a lane's classes overlaps.
struct MathTables {
  double two[65];     // 2^(j / 64) for j < 64, then 0
  double inv_c[64];   // 1 / c, c = 1 + j / 64
  double log_c[64];
};

struct TableMath {
  MathTables* t;
  // The whole block calls it; used: whether any of the tables is.
  __device__ __forceinline__ explicit TableMath(MathTables& tables, bool used = true) : t(&tables) {
    if (!used) return;
    for (int j = threadIdx.x; j < 65; j += blockDim.x) t->two[j] = j < 64 ? exp2(j / 64.0) : 0.0;
    for (int j = threadIdx.x; j < 64; j += blockDim.x) {
      t->inv_c[j] = 64.0 / (64 + j);
      t->log_c[j] = log(1.0 + j / 64.0);
    }
    __syncthreads();
  }
  // exp(d), d <= 709.78: d = (n / 64) ln 2 + r, exp(d) = 2^(n / 64) (1 + r +
  // ... + r^5 / 120), |r| <= ln 2 / 128, truncation below 2^-54.  NaN stays;
  // below -708 (3e-308) the value is 0.
  __device__ __forceinline__ double exp(double d) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const bool none = d < -708.0;
    d = __hiloint2double(none ? 0 : __double2hiint(d), __double2loint(d));
    const double k0 = fma(d, 92.332482616893656, kRound);
    const int n = __double2loint(k0);
    const double k = k0 - kRound;
    double r = fma(k, -1.0830424696249145e-2, d);  // ln 2 / 64, and its rounding error
    r = fma(k, -3.6235106466348430e-19, r);
    double q = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(q, r, 1.0 / 6.0);
    q = fma(q, r, 0.5);
    q = fma(q, r * r, r);
    const double two_n = t->two[none ? 64 : n & 63];
    const double scaled = __hiloint2double(__double2hiint(two_n) + (n >> 6 << 20), __double2loint(two_n));
    return fma(scaled, q, scaled);
  }
  __device__ __forceinline__ float exp(float d) const { return __expf(d); }
  __device__ __forceinline__ double operator()(double d) const { return d > 709.78 ? INFINITY : exp(d); }
  // log(1 + x), 0 <= x < 2^1000: 1 + x = 2^e c (1 + f), c the multiple of 1/64
  // next to its significand, |f| <= 1 / 128; f - f^2 / 2 + ... - f^8 / 8,
  // truncation below 2^-59.  Next to 1, f is x itself.
  __device__ __forceinline__ double log1p(double x) const {
    const double s = 1.0 + x;
    const int hi = __double2hiint(s) + 0x2000;
    const int j = hi >> 14 & 63, e = (hi >> 20) - 1023;
    const double c = __hiloint2double(hi & ~0x3fff, 0);
    const double inv = t->inv_c[j];
    const double f = c == 1.0 ? x : (s - c) * __hiloint2double(__double2hiint(inv) - (e << 20), __double2loint(inv));
    double q = fma(f, -1.0 / 8.0, 1.0 / 7.0);
    q = fma(q, f, -1.0 / 6.0);
    q = fma(q, f, 1.0 / 5.0);
    q = fma(q, f, -1.0 / 4.0);
    q = fma(q, f, 1.0 / 3.0);
    q = fma(q, f, -1.0 / 2.0);
    return fma((double)e, 0.6931471805599453, t->log_c[j]) + fma(q, f * f, f);
  }
  // 1 / s for 1 <= s < 2^100, by Newton's iteration from a float32 quotient.
  __device__ __forceinline__ static double inverse(double s) {
    double r = (double)__fdividef(1.0f, (float)s);
    r = fma(r, fma(-s, r, 1.0), r);
    return fma(r, fma(-s, r, 1.0), r);
  }
};

// Rows in shared memory: a row of a multiple of 16 bytes starts at an odd
// multiple of 16, so that lanes reading the same class of different rows meet
// at most four to a bank; other rows follow each other directly.
struct TileRows {
  int bytes, stride;
  __host__ __device__ explicit TileRows(int row_bytes)
      : bytes(row_bytes), stride(row_bytes % 16 == 0 ? (row_bytes / 16 | 1) * 16 : row_bytes) {}
};

// A lane's walk over the elements lane, lane + 32, ... of rows of `width`.
struct RowWalk {
  int row, col, width, step_row, step_col;
  __device__ __forceinline__ RowWalk(int lane, int w)
      : row(lane / w), col(lane % w), width(w), step_row(32 / w), step_col(32 % w) {}
  __device__ __forceinline__ void next() {
    row += step_row;
    col += step_col;
    if (col >= width) {
      col -= width;
      ++row;
    }
  }
};

// Bulk copies between global and shared memory, of multiples of 16 bytes that
// start on 16 bytes; those to shared memory count down a barrier.
__device__ __forceinline__ unsigned shared_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bulk_in(void* shared, const void* global, int bytes, unsigned long long* barrier) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   shared_address(shared)),
               "l"(global), "r"(bytes), "r"(shared_address(barrier))
               : "memory");
}

__device__ __forceinline__ void bulk_out(void* global, const void* shared, int bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(global), "r"(shared_address(shared)),
               "r"(bytes)
               : "memory");
}

// Starts the copy of `rows` rows, row_stride apart, into shared memory (`at`
// walks over their elements); rows_wait ends it.  The whole warp calls both.  vec: the rows are
// one piece of global memory that starts on 16 bytes, copied whole, or row by
// row where they lie apart in shared memory.
template <typename E>
__device__ __forceinline__ void rows_in(const E* global, unsigned char* tile, TileRows R, int rows, RowWalk at,
                                        long long row_stride, bool vec, unsigned long long* barrier) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    const int bytes = rows * R.bytes & ~15;
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(barrier)), "r"(bytes)
                   : "memory");
    __syncwarp();
    if (R.stride != R.bytes) {
      if (lane < rows) bulk_in(tile + lane * R.stride, reinterpret_cast<const char*>(global) + lane * R.bytes, R.bytes, barrier);
    } else {
      if (lane == 0 && bytes) bulk_in(tile, global, bytes, barrier);
      const int j = bytes / (int)sizeof(E) + lane;  // fewer than 16 bytes are left
      if (j < rows * at.width) reinterpret_cast<E*>(tile)[j] = global[j];
    }
  } else {
    while (at.row < rows) {  // four loads in flight
      E x[4];
      E* to[4];
#pragma unroll
      for (int q = 0; q < 4; ++q, at.next()) {
        to[q] = nullptr;
        if (at.row < rows) {
          to[q] = reinterpret_cast<E*>(tile + at.row * R.stride) + at.col;
          x[q] = global[at.row * row_stride + at.col];
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (to[q]) *to[q] = x[q];
    }
  }
}

// False when the copies did not end within the limit (about a second).
__device__ __forceinline__ bool rows_wait(bool vec, unsigned long long* barrier, unsigned phase) {
  unsigned done = vec ? 0 : 1;
  for (int i = 0; i < 1 << 20 && !done; ++i)
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(shared_address(barrier)), "r"(phase)
        : "memory");
  __syncwarp();
  return done != 0;
}

// Rows from shared memory to global memory, elements row_stride and
// class_stride apart; vec as above.  The whole warp calls it, after writing
// the rows; out_wait before they are overwritten.
template <int ROWS, typename E>
__device__ __forceinline__ void rows_out(E* global, const unsigned char* tile, TileRows R, int rows, RowWalk at,
                                         long long row_stride, long long class_stride, bool vec) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    const int bytes = rows * R.bytes & ~15;
    if (R.stride != R.bytes) {
      if (lane < rows) bulk_out(reinterpret_cast<char*>(global) + lane * R.bytes, tile + lane * R.stride, R.bytes);
    } else {
      if (lane == 0 && bytes) bulk_out(global, tile, bytes);
      const int j = bytes / (int)sizeof(E) + lane;
      if (j < rows * at.width) global[j] = reinterpret_cast<const E*>(tile)[j];
    }
  } else if (class_stride == 1) {
    for (; at.row < rows; at.next())
      global[at.row * row_stride + at.col] = reinterpret_cast<const E*>(tile + at.row * R.stride)[at.col];
  } else {  // classes apart: rows next to each other
    const int row = lane % ROWS;
    if (row < rows)
      for (int k = lane / ROWS; k < at.width; k += 32 / ROWS)
        global[row * row_stride + k * class_stride] = reinterpret_cast<const E*>(tile + row * R.stride)[k];
  }
}

// Ends the reads of this lane's copies out of shared memory.
__device__ __forceinline__ void out_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

struct SmallLayout {
  int tile;              // bytes of a tile; a warp has two
  bool vec_in, vec_out;  // see rows_in
};

// A row's own values, loaded a step ahead of their use.
struct RowValues {
  long long a;
  double adv, old, ref, w;  // ROW_POLICY
  double m, rest, g, h;     // ROW_BACK
};

template <int OP, typename T>
__device__ __forceinline__ RowValues load_row(const RowArgs<T>& A, long long r, bool there) {
  RowValues v = {-1, 0.0, 0.0, 0.0, 1.0, 0.0, -1.0, 0.0, 0.0};
  if (there) {
    v.a = A.in.action(r);
    if (OP == ROW_POLICY) {
      v.adv = (double)A.pol.advantages[r];
      v.old = (double)A.pol.old_logp[r];
      if (A.pol.ref_logp) v.ref = (double)A.pol.ref_logp[r];
      if (A.pol.weights) v.w = (double)A.pol.weights[r];
    }
    if (OP == ROW_BACK) {
      v.m = (double)A.stats[2 * r];
      v.rest = (double)A.stats[2 * r + 1];
      v.g = (double)A.grad_logp[r];
      if (A.hess_logp) v.h = (double)A.hess_logp[r];
    }
  }
  return v;
}

// L lanes a row, P classes a lane: K <= L P.
template <typename T, int OP, int L, int P>
__global__ void __launch_bounds__(kSmallThreads) k_feedback_small(const RowArgs<T> A, const SmallLayout lay) {
  using C = typename Types<T>::C;
  using Row = typename Types<T>::Row;
  using Out = typename Types<T>::Out;
  constexpr int kRows = 32 / L;
  // In float64 a sum that holds the 1 of the largest class gives the others'
  // to 2^-43 of it unless it is below 2^-10, far beyond what the float32
  // derivatives keep; the statistics keep it whole.
  constexpr bool kExact = sizeof(C) == 4 || OP == ROW_LOGPROBS;
  constexpr double kNearOne = 0x1p-10;
  extern __shared__ __align__(16) unsigned char small_smem[];
  __shared__ MathTables tables;
  __shared__ __align__(8) unsigned long long barriers[kSmallThreads / 32][2];
  const TableMath math(tables);
  const int lane = threadIdx.x & 31, l = lane % L, i = lane / L;  // this lane's row of a batch
  const int K = A.in.K;
  unsigned char* tile = small_smem + (threadIdx.x >> 5) * (2 * lay.tile);
  int other = lay.tile;  // from this batch's tile to the next one's
  const TileRows in_rows(K * (int)sizeof(T)), out_rows(K * (int)sizeof(Out));
  const RowWalk walk(lane, K);
  const long long step = (long long)gridDim.x * (kSmallThreads / 32) * kRows;
  long long base = ((long long)blockIdx.x * (kSmallThreads / 32) + (threadIdx.x >> 5)) * kRows;
  auto rows_at = [&](long long b) { return (int)max(0ll, min((long long)kRows, A.in.n - b)); };
  // a barrier per tile; the warp waits for tile q of its barrier in phase q mod 2
  unsigned long long* barrier = barriers[threadIdx.x >> 5];
  if (lane < 2)
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(barrier + lane)) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  RowValues next = load_row<OP>(A, base + i, i < rows_at(base));
  if (base < A.in.n)
    rows_in(A.in.scores + base * A.in.stride, tile, in_rows, rows_at(base), walk, A.in.stride, lay.vec_in, barrier);
  unsigned turn = 0;  // bit 0: the tile's barrier, bit 1: its phase
  for (; base < A.in.n; base += step, tile += other, other = -other, turn = (turn + 1) & 3) {
    const int rows = rows_at(base);
    const bool mine = i < rows;  // the lanes of a missing row compute on what lies there, and store nothing
    const long long r = base + i;
    const RowValues now = next;
    next = load_row<OP>(A, r + step, i < rows_at(base + step));
    const bool arrived = rows_wait(lay.vec_in, barrier + (turn & 1), turn >> 1);
    const T* z = reinterpret_cast<const T*>(tile + i * in_rows.stride);
    RowDerivative row = {now.g, now.h};
    C m = (C)now.m;
    double rest = now.rest;
    bool part = now.a >= 0 && now.w != 0.0 && (OP != ROW_BACK || rest != -1.0);
    const bool bad = part && (now.a >= K || !arrived);
    const int taken = part && !bad ? (int)now.a : 0;
    const double za = (double)widen(z[taken]);
    C v[P];
    int top = -1;  // a class of this lane at the maximum
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] = l + e * L < K ? (C)widen(z[l + e * L]) : (C)-INFINITY;
    if (OP != ROW_BACK) {
      C mx = v[0];
#pragma unroll
      for (int e = 1; e < P; ++e) mx = !(v[e] <= mx) ? v[e] : mx;  // may lose a NaN: the sum does not
#pragma unroll
      for (int k = L / 2; k > 0; k >>= 1) {
        const C o = __shfl_xor_sync(0xffffffffu, mx, k);
        mx = o > mx ? o : mx;
      }
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = math.exp(v[e] - mx);
      // the sum less the 1 of one class at the maximum
      double others = 0.0;
      bool exact = kExact;  // a matter of this row alone, whatever the warp's others are
      if (!kExact) {
        C sum = v[0];
#pragma unroll
        for (int e = 1; e < P; ++e) sum += v[e];
#pragma unroll
        for (int k = L / 2; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        others = (double)sum - 1.0;
        exact = others < kNearOne;
      }
      if (kExact || __any_sync(0xffffffffu, exact)) {
        C sum = 0;
        int ties = 0;
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const bool one = v[e] == (C)1;
          sum += one ? (C)0 : v[e];
          ties += one ? 1 : 0;
          top = one && exact ? l + e * L : top;
        }
#pragma unroll
        for (int k = L / 2; k > 0; k >>= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, k);
          ties += __shfl_xor_sync(0xffffffffu, ties, k);
        }
        if (exact) others = (double)sum + (double)(ties - 1);
      }
      if (mx == (C)-INFINITY && part && !bad) {  // no class, unless a NaN hides among them
        part = false;
        for (int k = 0; k < K; ++k) part = part || widen(z[k]) != (C)-INFINITY;
      }
      m = 0;
      if (part) {
        m = mx;
        rest = others;
      }
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = math.exp(v[e] - m);
      const bool exact = kExact || rest < kNearOne;
#pragma unroll
      for (int e = 0; e < P; ++e) top = v[e] == (C)1 && exact ? l + e * L : top;
    }
    // the next rows into the other tile, whose derivatives are on their way by now
    out_wait();
    __syncwarp();
    if (base + step < A.in.n)
      rows_in(A.in.scores + (base + step) * A.in.stride, tile + other, in_rows, rows_at(base + step), walk, A.in.stride,
              lay.vec_in, barrier + (turn + 1 & 1));

    if (OP == ROW_LOGPROBS) {
      if (mine && l == 0) {
        const double lp = part && !bad ? za - (double)m - math.log1p(rest) : 0.0;
        A.logp[r] = bad ? (Row)NAN : (Row)lp;
        A.stats[2 * r] = bad ? (Row)NAN : (Row)m;
        A.stats[2 * r + 1] = bad ? (Row)NAN : part ? (Row)rest : (Row)-1;
      }
      __syncwarp();
      continue;
    }
    if (OP == ROW_POLICY) {
      double lp = 0.0, loss = 0.0;
      if (part && !bad) {
        lp = za - (double)m - math.log1p(rest);
        part = za != -INFINITY;  // the class taken is masked
      }
      if (sizeof(C) == 4) {
        const bool near = part && !bad && near_border(A.pol, lp - now.old, now.adv, border_slack(P + 3, 4.9));
        if (__any_sync(0xffffffffu, near)) {
          double sum = 0.0;
          for (int k = l; k < K && near; k += L) sum += exp((double)widen(z[k]) - (double)m);
#pragma unroll
          for (int k = L / 2; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
          if (near) lp = za - (double)m - log(sum);
        }
      }
      if (bad) lp = loss = NAN;
      else if (part)
        row = policy_terms(A.pol, lp, now.adv, now.old, now.ref, now.w, &loss, math);
      if (mine && l == 0) {
        if (A.pol.loss) A.pol.loss[r] = (Row)loss;
        if (A.pol.logp) A.pol.logp[r] = (Row)lp;
      }
      if (!A.out.grad) {
        __syncwarp();
        continue;
      }
    }
    __syncwarp();  // the scores are used up: the derivatives take their place
    const bool want_h = A.out.hess != nullptr;
    unsigned char* tile_h = tile + kRows * out_rows.stride;
    Out* to_g = reinterpret_cast<Out*>(tile + i * out_rows.stride);
    Out* to_h = reinterpret_cast<Out*>(tile_h + i * out_rows.stride);
    const double inv_total = TableMath::inverse(1.0 + rest);
    const C inv = (C)inv_total, share = (C)(rest * inv_total), g = (C)row.g, h = (C)row.h;
    if (part && !bad) {
      // every class as one that was not taken, and with 1 - p as it comes
      const C down = -g * inv, ag = fabs(g), bend = h - ag;
#pragma unroll
      for (int e = 0; e < P; ++e)
        if (l + e * L < K) narrow(v[e] * down, to_g[l + e * L]);
      if (want_h) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const C p = v[e] * inv;
          if (l + e * L < K) narrow(p * fma(p, bend, ag), to_h[l + e * L]);
        }
      }
      // a class with more than half of the probability is alone at the
      // maximum, and 1 - p is the others' share; then the class taken
      const C pt = inv, lt = share;
      if (want_h && inv > (C)0.5 && top >= 0) narrow(pt * (ag * lt + h * pt), to_h[top]);
    }
    __syncwarp();
    if (l == 0 && part && !bad) {
      const C e = math.exp((C)(za - (double)m)), p = e * inv, q = e == (C)1 ? share : (C)1 - p;
      narrow(g * q, to_g[taken]);
      if (want_h) narrow(q * (h * q + fabs(g) * p), to_h[taken]);
    }
    if (!part || bad) {
      for (int k = l; k < K; k += L) {
        narrow(bad ? (C)NAN : (C)0, to_g[k]);
        if (want_h) narrow(bad ? (C)NAN : (C)0, to_h[k]);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    const long long to = base * A.out.row_stride;
    rows_out<kRows>(A.out.grad + to, tile, out_rows, rows, walk, A.out.row_stride, A.out.class_stride, lay.vec_out);
    if (want_h)
      rows_out<kRows>(A.out.hess + to, tile_h, out_rows, rows, walk, A.out.row_stride, A.out.class_stride, lay.vec_out);
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    __syncwarp();
  }
  out_wait();
}

inline bool on16(const void* p) { return (uintptr_t)p % 16 == 0; }

int multiprocessors() {
  constexpr int kMostDevices = 64;
  static std::atomic<int> known[kMostDevices];
  int dev = 0, n = 0;
  MTB_CUDA_FB(cudaGetDevice(&dev));
  if (dev < kMostDevices && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  MTB_CUDA_FB(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  if (dev < kMostDevices) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int OP, int L, int P>
void launch_small_t(const RowArgs<T>& A, cudaStream_t st) {
  using Out = typename Types<T>::Out;
  constexpr int rows = 32 / L, warps = kSmallThreads / 32;
  const int K = A.in.K;
  const TileRows in(K * (int)sizeof(T)), out(K * (int)sizeof(Out));
  SmallLayout lay;
  const int back = OP == ROW_LOGPROBS || !A.out.grad ? 0 : rows * out.stride * (A.out.hess ? 2 : 1);
  lay.tile = (std::max(rows * in.stride, back) + 15) / 16 * 16;
  lay.vec_in = on16(A.in.scores) && A.in.stride == K && rows * in.bytes % 16 == 0;
  lay.vec_out = on16(A.out.grad) && on16(A.out.hess) && A.out.row_stride == K && A.out.class_stride == 1 &&
                rows * out.bytes % 16 == 0;
  const long long blocks = (A.in.n + rows * warps - 1) / (rows * warps);
  const unsigned grid = (unsigned)std::min<long long>(blocks, 16ll * multiprocessors());
  k_feedback_small<T, OP, L, P><<<grid, kSmallThreads, (size_t)lay.tile * 2 * warps, st>>>(A, lay);
}

// Few classes fit one lane; a class too many in P costs a float64 exponential
// a row (20 instructions of about 100 a class), a float32 one next to nothing.
template <typename T, int OP>
void launch_small(const RowArgs<T>& A, cudaStream_t st) {
  const int K = A.in.K;
  if (K > 64) return launch_small_t<T, OP, 8, 16>(A, st);
  if (K > 32) return launch_small_t<T, OP, 4, 16>(A, st);
  if (K > 16) return launch_small_t<T, OP, 2, 16>(A, st);
  if constexpr (sizeof(T) == 8) {
    if (K <= 2) return launch_small_t<T, OP, 1, 2>(A, st);
    if (K <= 4) return launch_small_t<T, OP, 1, 4>(A, st);
    if (K <= 6) return launch_small_t<T, OP, 1, 6>(A, st);
    if (K <= 8) return launch_small_t<T, OP, 1, 8>(A, st);
    if (K <= 10) return launch_small_t<T, OP, 1, 10>(A, st);
    if (K <= 12) return launch_small_t<T, OP, 1, 12>(A, st);
  } else if constexpr (sizeof(T) == 4) {
    if (K <= 4) return launch_small_t<T, OP, 1, 4>(A, st);
    if (K <= 8) return launch_small_t<T, OP, 1, 8>(A, st);
  }
  launch_small_t<T, OP, 1, 16>(A, st);
}

// ---------------------------------------------------------------------------
// Rows of more than 128 classes, scores of 32 and 16 bits
//
// A block (or a cluster of up to 8 of them, where a row is longer than 8192
// vectors of 16 bytes, or rows are too few to fill the GPU) holds a row in its
// registers: the scores are read once.  Bound are the memory system and, for
// 16-bit scores, the exponentials, two a class (the sum's, and the gradient's
// again: kept in float32 they would take twice the registers).  Each warp sums
// relative to its own maximum, so one barrier joins maxima and sums; the next
// row is fetched into L2 meanwhile.
//
// Measured, policy loss with gradient of 8192 x 32768 bfloat16 (1.07 GB,
// 164 us at the copy rate): 246 us; the gradient's pass alone, which needs no
// sum, takes 200.  Rows kept in shared memory instead, three blocks an SM,
// took 60% longer (more instructions a class); clusters of 2 or 4 smaller
// blocks a row 6% and 55% longer (their barriers); 50001 classes in one block
// of 1024 threads rather than two of 512: 129 -> 120 us.
// ---------------------------------------------------------------------------

__device__ __forceinline__ float max_nan32(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two float32 values in one register pair, with the paired instructions.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ static Pair of(float x, float y) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
    return p;
  }
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
  __device__ __forceinline__ Pair operator+(Pair o) const {
    Pair p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(v), "l"(o.v));
    return p;
  }
  __device__ __forceinline__ Pair times_plus(Pair o, Pair c) const {
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(v), "l"(o.v), "l"(c.v));
    return p;
  }
  __device__ __forceinline__ Pair operator*(Pair o) const {
    Pair p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(v), "l"(o.v));
    return p;
  }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ __half low_of(__half2 x) { return __low2half(x); }
__device__ __forceinline__ __half high_of(__half2 x) { return __high2half(x); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 x) { return __low2bfloat16(x); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 x) { return __high2bfloat16(x); }

// 16 bytes of scores.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ unsigned word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
  __device__ __forceinline__ Pair pair(int i) const {  // elements 2 i, 2 i + 1
    if constexpr (sizeof(T) == 4) {
      return Pair::of(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return Pair::of(__uint_as_float(word(i) << 16), __uint_as_float(word(i) & 0xffff0000u));
    } else {
      const unsigned w = word(i);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
      return Pair::of(f.x, f.y);
    }
  }
  __device__ __forceinline__ void set(int i, Pair p) {  // rounds elements 2 i, 2 i + 1
    const float2 f = p.get();
    unsigned* w = reinterpret_cast<unsigned*>(&raw);
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const unsigned*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(f.x, f.y);
      w[i] = *reinterpret_cast<const unsigned*>(&b);
    }
  }
  __device__ __forceinline__ float max() const {  // NaN when one is
    if constexpr (sizeof(T) == 4) {
      return max_nan32(max_nan32(__uint_as_float(raw.x), __uint_as_float(raw.y)),
                       max_nan32(__uint_as_float(raw.z), __uint_as_float(raw.w)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* w = reinterpret_cast<const T2*>(&raw);
      const T2 x = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
      return max_nan32(widen(low_of(x)), widen(high_of(x)));
    }
  }
  // Hides the value's history, so that what an earlier pass made of it is not
  // kept in registers for a later one.
  __device__ __forceinline__ void forget() {
    asm volatile("" : "+r"(raw.x), "+r"(raw.y), "+r"(raw.z), "+r"(raw.w));
  }
  __device__ __forceinline__ static Vec lowest() {  // every element -inf
    const unsigned w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u;
    return {make_uint4(w, w, w, w)};
  }
};

// A part of a row: its maximum m, and a sum of 2^(log2(e) z - c) for a float32
// c next to log2(e) m, `shift` being log2(e) m - c.  One rounding takes each
// score to its exponent that way, and the error of c is a factor of the whole
// sum, which the scalars take out again.
struct Part {
  double sum;
  float m, shift;
  int ones;  // terms at the maximum that a later sum leaves out
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

// c of the comment above, negated.
__device__ __forceinline__ float exponent_offset(float m) { return -__fmul_rn(m, kLog2e); }

enum RowState : int { ROW_EMPTY = 0, ROW_DONE = 1, ROW_SLOW = 2, ROW_NEAR = 3 };

template <int THREADS>
struct LargeShared {
  MathTables tables;
  Part warp[2][THREADS / 32], slow[2][THREADS / 32];  // by the parity of the row, as all arrays here
  Part block[2], slow_block[2];                       // read by the cluster
  double near[2][THREADS / 32], near_block[2];
  int state;  // RowState, and what goes with it
  float m, g, h, inv, share;
};

// The parts of lanes below n joined: the maximum, the sum of exp(z - maximum).
__device__ __forceinline__ Part join_parts(Part p, int n, const TableMath& math) {
  const bool there = (int)(threadIdx.x & 31) < n;
  float m = there ? p.m : -INFINITY;
  for (int k = 16; k > 0; k >>= 1) m = max_nan32(m, __shfl_xor_sync(0xffffffffu, m, k));
  double s = 0.0;
  if (there && p.m != -INFINITY) s = p.sum * math.exp((double)p.m - (double)m - (double)p.shift * kLn2);
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  return {s, m, 0.0f, 0};
}

// Sums of parts relative to one maximum.
__device__ __forceinline__ Part add_parts(Part p, int n) {
  if ((int)(threadIdx.x & 31) >= n) p.sum = 0.0, p.ones = 0;
  for (int k = 16; k > 0; k >>= 1) {
    p.sum += __shfl_xor_sync(0xffffffffu, p.sum, k);
    p.ones += __shfl_xor_sync(0xffffffffu, p.ones, k);
  }
  return p;
}

// A vector's elements one by one, for derivatives whose vectors do not start
// on 16 bytes where the scores' do.
template <typename T>
__device__ __noinline__ void store_elements(T* to, Vec<T> v) {
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) to[i] = reinterpret_cast<const T*>(&v)[i];
}

// per: whole vectors of a row that a block takes at most.
template <typename T, int OP, bool HESS, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_feedback_large(const RowArgs<T> A, const int per) {
  namespace cg = cooperative_groups;
  using Row = typename Types<T>::Row;
  constexpr int N = Vec<T>::N, kWarps = THREADS / 32;
  __shared__ LargeShared<THREADS> S;
  const TableMath math(S.tables);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = A.in.K;
  const Pair scale = Pair::of(kLog2e, kLog2e);
  const long long clusters = gridDim.x / blocks;
  int parity = 0;
  for (long long r = blockIdx.x / blocks; r < A.in.n; r += clusters) {
    // The row's whole vectors of 16 bytes are divided among the blocks.  The
    // up to 2 (N - 1) elements before and behind them lie with the first
    // block's first warp: head ones in the lanes from 0, tail ones from 16.
    const T* z = A.in.scores + r * A.in.stride;
    const int lead = (int)(-(uintptr_t)z / sizeof(T) % N);  // elements before the first whole vector
    const int vecs = (int)((unsigned)(K - lead) / N);
    const int v0 = min(vecs, rank * per), v1 = min(vecs, v0 + per);
    const int tail = K - lead - vecs * N;
    int edge = -1;
    if (warp == 0 && rank == 0) edge = lane < lead ? lane : lane >= 16 && lane < 16 + tail ? K - tail + lane - 16 : -1;
    const T* zv = z + lead + (long long)(v0 + (int)threadIdx.x) * N;
    const int mine = v1 - v0 - (int)threadIdx.x;  // vector j is this thread's if j * THREADS < mine
    const long long a = A.in.action(r);
    const bool bad = a >= K;
    bool part = a >= 0;
    if (OP == ROW_POLICY && A.pol.weights) part = part && A.pol.weights[r] != (Row)0;
    float m = 0.0f, g = 0.0f, h = 0.0f, inv = 0.0f, share = 0.0f;
    if (OP == ROW_BACK) {
      m = A.stats[2 * r];
      const float rest = A.stats[2 * r + 1];
      part = part && rest != -1.0f;
      if (part && !bad) {
        g = A.grad_logp[r];
        if (HESS) h = A.hess_logp[r];
        const float inv_total = __frcp_rn(1.0f + rest);
        inv = inv_total * exp2_approx(-fmaf(m, kLog2e, exponent_offset(m)));
        share = rest * inv_total;
      }
    }
    bool live = part && !bad;
    Vec<T> v[NV];
    float ze = -INFINITY, za = 0.0f;
    if (live) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        v[j] = Vec<T>::lowest();
        if (j * THREADS < mine) v[j].raw = *reinterpret_cast<const uint4*>(zv + j * THREADS * N);
      }
      if (edge >= 0) ze = widen(z[edge]);
      za = widen(z[a]);
    }
    if (threadIdx.x == 0 && r + clusters < A.in.n) {  // the next row's vectors of this block
      const T* zn = z + clusters * A.in.stride;
      const int ln = (int)(-(uintptr_t)zn / sizeof(T) % N);
      const int e = min(v1, (K - ln) / N);
      if (v0 < e)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(zn + ln + v0 * N), "r"((e - v0) * 16) : "memory");
    }

    if (OP != ROW_BACK && live) {
      parity ^= 1;
      float adv = 0.0f, old = 0.0f, ref = 0.0f, w = 1.0f;
      if (OP == ROW_POLICY && warp == 0) {
        adv = A.pol.advantages[r];
        old = A.pol.old_logp[r];
        if (A.pol.ref_logp) ref = A.pol.ref_logp[r];
        if (A.pol.weights) w = A.pol.weights[r];
      }
      // the first warp's end of a row; near: l is right whatever the border
      auto finish = [&](float top, double rest, double lp, bool near_known) {
        const double total = 1.0 + rest, inv_total = TableMath::inverse(total);
        if (OP == ROW_LOGPROBS) {
          if (threadIdx.x == 0) {
            S.state = ROW_DONE;
            if (rank == 0) {
              A.logp[r] = (Row)lp;
              A.stats[2 * r] = top;
              A.stats[2 * r + 1] = (Row)rest;
            }
          }
          return;
        }
        const bool masked = za == -INFINITY;
        const bool near = !near_known && !masked && near_border(A.pol, lp - (double)old, (double)adv,
                                                                border_slack(NV * N / 2 + 8, 12.5));
        double loss = 0.0;
        RowDerivative d = {0.0, 0.0};
        if (!near && !masked)
          d = policy_terms(A.pol, lp, (double)adv, (double)old, (double)ref, (double)w, &loss, math);
        if (threadIdx.x == 0) {
          const double shift = (double)fmaf(top, kLog2e, exponent_offset(top));
          S.state = near ? ROW_NEAR : masked ? ROW_EMPTY : ROW_DONE;
          S.m = top;
          S.g = (float)d.g;
          S.h = (float)d.h;
          S.inv = (float)(inv_total * math.exp(-shift * kLn2));
          S.share = (float)(rest * inv_total);
          if (rank == 0 && !near) {
            if (A.pol.loss) A.pol.loss[r] = (Row)loss;
            if (A.pol.logp) A.pol.logp[r] = (Row)lp;
          }
        }
      };

      // the warp's maximum, and its sum relative to it
      float wm = ze;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        wm = max_nan32(wm, v[j].max());
        v[j].forget();
      }
      for (int k = 16; k > 0; k >>= 1) wm = max_nan32(wm, __shfl_xor_sync(0xffffffffu, wm, k));
      Part p = {0.0, wm, 0.0f, 0};
      if (wm != -INFINITY) {
        const float c = exponent_offset(wm);
        const Pair offset = Pair::of(c, c);
        Pair sum = Pair::of(exp2_approx(fmaf(ze, kLog2e, c)), 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            const float2 d = v[j].pair(i).times_plus(scale, offset).get();
            sum = sum + Pair::of(exp2_approx(d.x), exp2_approx(d.y));
          }
          v[j].forget();
        }
        float s = sum.get().x + sum.get().y;
        for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        p.sum = (double)s;
        p.shift = fmaf(wm, kLog2e, c);
      }
      if (lane == 0) S.warp[parity][warp] = p;
      __syncthreads();
      Part all;
      if (kWarps == 1) all = {p.sum * math.exp(-(double)p.shift * kLn2), wm, 0.0f, 0};
      else if (warp == 0) all = join_parts(S.warp[parity][lane < kWarps ? lane : 0], kWarps, math);
      if (blocks > 1) {
        if (threadIdx.x == 0) S.block[parity] = all;
        cluster.sync();
        if (warp == 0) all = join_parts(*cluster.map_shared_rank(&S.block[parity], lane < blocks ? lane : 0), blocks, math);
      }
      if (warp == 0) {
        const double rest = all.sum - 1.0;
        if (all.m == -INFINITY || rest < 1.0) {
          if (lane == 0) {
            S.state = all.m == -INFINITY ? ROW_EMPTY : ROW_SLOW;
            S.m = all.m;
            if (OP == ROW_POLICY && rank == 0 && S.state == ROW_EMPTY) {
              if (A.pol.loss) A.pol.loss[r] = 0.0f;
              if (A.pol.logp) A.pol.logp[r] = 0.0f;
            }
          }
        } else {
          finish(all.m, rest, (double)za - (double)all.m - math.log1p(rest), false);
        }
      }
      __syncthreads();
      if (S.state == ROW_SLOW) {
        // One class has more than half, and its 1 took the last bits of the
        // others: the sum without the terms at the maximum, of the warps that
        // have any.
        const float top = S.m;
        if (wm == top) {
          const float c = exponent_offset(top);
          float s = ze == top ? 0.0f : exp2_approx(fmaf(ze, kLog2e, c));
          int ones = ze == top ? 1 : 0;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              const float2 f = v[j].pair(i).get();
              s += f.x == top ? 0.0f : exp2_approx(fmaf(f.x, kLog2e, c));
              s += f.y == top ? 0.0f : exp2_approx(fmaf(f.y, kLog2e, c));
              ones += (f.x == top ? 1 : 0) + (f.y == top ? 1 : 0);
            }
            v[j].forget();
          }
          for (int k = 16; k > 0; k >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, k);
            ones += __shfl_xor_sync(0xffffffffu, ones, k);
          }
          p.sum = (double)s;
          p.ones = ones;
        }
        if (wm != -INFINITY) p.sum *= math.exp((double)wm - (double)top - (double)p.shift * kLn2);
        if (lane == 0) S.slow[parity][warp] = p;
        __syncthreads();
        if (warp == 0) p = add_parts(S.slow[parity][lane < kWarps ? lane : 0], kWarps);
        if (blocks > 1) {
          if (threadIdx.x == 0) S.slow_block[parity] = p;
          cluster.sync();
          if (warp == 0) p = add_parts(*cluster.map_shared_rank(&S.slow_block[parity], lane < blocks ? lane : 0), blocks);
        }
        if (warp == 0) {
          const double rest = p.sum + (double)(p.ones - 1);
          finish(top, rest, (double)za - (double)top - math.log1p(rest), false);
        }
        __syncthreads();
      }
      if (OP == ROW_POLICY && S.state == ROW_NEAR) {
        const float top = S.m;
        const double share64 = (double)S.share, inv64 = (double)S.inv;
        double sum = ze == -INFINITY ? 0.0 : math.exp((double)ze - (double)top);
        for (int k = threadIdx.x; k < (v1 - v0) * N; k += THREADS)
          sum += math.exp((double)widen(z[lead + v0 * N + k]) - (double)top);
        for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        if (lane == 0) S.near[parity][warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int i = 0; i < kWarps; ++i) sum += S.near[parity][i];
        if (blocks > 1) {
          if (threadIdx.x == 0) S.near_block[parity] = sum;
          cluster.sync();
          sum = 0.0;
          for (int i = 0; i < blocks; ++i) sum += *cluster.map_shared_rank(&S.near_block[parity], i);
        }
        if (warp == 0) finish(top, sum - 1.0, (double)za - (double)top - log(sum), true);
        if (threadIdx.x == 0) {  // as the row's other paths have them
          S.share = (float)share64;
          S.inv = (float)inv64;
        }
        __syncthreads();
      }
      live = part = S.state == ROW_DONE;
      if (live && OP == ROW_POLICY) {
        m = S.m;
        g = S.g;
        h = S.h;
        inv = S.inv;
        share = S.share;
      }
    }
    if (OP != ROW_BACK && !live && threadIdx.x == 0 && rank == 0) {
      const float none = part && bad ? NAN : 0.0f;
      if (OP == ROW_LOGPROBS) {
        A.logp[r] = none;
        A.stats[2 * r] = none;
        A.stats[2 * r + 1] = part && bad ? NAN : -1.0f;
      } else if (za != -INFINITY) {  // else the row's values are written
        if (A.pol.loss) A.pol.loss[r] = none;
        if (A.pol.logp) A.pol.logp[r] = none;
      }
    }
    if (OP == ROW_LOGPROBS || !A.out.grad) continue;

    T* to_g = A.out.grad + r * A.out.row_stride;
    T* to_h = HESS ? A.out.hess + r * A.out.row_stride : nullptr;
    if (!live) {
      T fill;
      narrow(part && bad ? NAN : 0.0f, fill);
      for (int k = rank * THREADS + threadIdx.x; k < K; k += blocks * THREADS) {
        to_g[k] = fill;
        if (HESS) to_h[k] = fill;
      }
      continue;
    }
    const bool whole = (uintptr_t)(to_g + lead) % 16 == 0 && (!HESS || (uintptr_t)(to_h + lead) % 16 == 0);
    const float c = exponent_offset(m), down = -g * inv, ag = fabsf(g);
    const Pair offset = Pair::of(c, c), times = Pair::of(down, down);
    const long long at = lead + (long long)(v0 + (int)threadIdx.x) * N;
    auto hess_of = [&](float score, float e) {
      const float p = e * inv;
      return p * (ag * (score == m ? share : 1.0f - p) + h * p);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * THREADS < mine) {
        Vec<T> og, oh;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 d = v[j].pair(i).times_plus(scale, offset).get();
          const Pair e = Pair::of(exp2_approx(d.x), exp2_approx(d.y));
          og.set(i, e * times);
          if (HESS) {
            const float2 f = v[j].pair(i).get();
            oh.set(i, Pair::of(hess_of(f.x, e.get().x), hess_of(f.y, e.get().y)));
          }
        }
        T* pg = to_g + at + j * THREADS * N;
        T* ph = HESS ? to_h + at + j * THREADS * N : nullptr;
        if (whole) {
          *reinterpret_cast<uint4*>(pg) = og.raw;
          if (HESS) *reinterpret_cast<uint4*>(ph) = oh.raw;
        } else {
          store_elements(pg, og);
          if (HESS) store_elements(ph, oh);
        }
      }
    }
    if (edge >= 0) {
      const float e = exp2_approx(fmaf(ze, kLog2e, c));
      narrow(e * down, to_g[edge]);
      if (HESS) narrow(hess_of(ze, e), to_h[edge]);
    }
    // the class taken, by the thread that has just stored it
    const int taken = (int)a, tv = taken >= lead ? (taken - lead) / N : vecs;
    if (edge == taken || (tv >= v0 && tv < v1 && (tv - v0) % THREADS == (int)threadIdx.x)) {
      const float p = exp2_approx(fmaf(za, kLog2e, c)) * inv, q = za == m ? share : 1.0f - p;
      narrow(g * q, to_g[taken]);
      if (HESS) narrow(q * (h * q + ag * p), to_h[taken]);
    }
  }
  if (blocks > 1) cluster.sync();  // the others may still read this block's parts
}

template <typename T, int OP, bool HESS, int THREADS, int NV>
void launch_large_t(const RowArgs<T>& A, int blocks, int per, cudaStream_t st) {
  const long long most = (long long)multiprocessors() * (1024 / THREADS) / blocks;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(std::min(A.in.n, most) * blocks));
  lc.blockDim = dim3(THREADS);
  lc.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  lc.attrs = attr;
  lc.numAttrs = blocks > 1 ? 1 : 0;
  MTB_CUDA_FB(cudaLaunchKernelEx(&lc, k_feedback_large<T, OP, HESS, THREADS, NV>, A, per));
}

template <typename T, int OP, bool HESS>
void launch_large_h(const RowArgs<T>& A, int blocks, int per, cudaStream_t st) {
  if (per > 4096) launch_large_t<T, OP, HESS, 1024, 8>(A, blocks, per, st);
  else if (per > 2048) launch_large_t<T, OP, HESS, 512, 8>(A, blocks, per, st);
  else if (per > 1024) launch_large_t<T, OP, HESS, 512, 4>(A, blocks, per, st);
  else if (per > 512) launch_large_t<T, OP, HESS, 256, 4>(A, blocks, per, st);
  else if (per > 128) launch_large_t<T, OP, HESS, 128, 4>(A, blocks, per, st);
  else launch_large_t<T, OP, HESS, 32, 4>(A, blocks, per, st);
}

// False when a row does not fit a cluster's registers, or its derivatives are
// not next to each other.
template <typename T, int OP>
bool launch_large(const RowArgs<T>& A, cudaStream_t st) {
  const int vecs = A.in.K / Vec<T>::N;  // or one fewer, where a row does not start on 16 bytes
  if (OP != ROW_LOGPROBS && A.out.grad && A.out.class_stride != 1) return false;
  int blocks = 1;
  while (blocks < 8 && (vecs > 8192 * blocks || (vecs > 512 * blocks && A.in.n * blocks * 2 <= multiprocessors()))) blocks *= 2;
  const int per = (vecs + blocks - 1) / blocks;
  if (per > 8192) return false;
  if constexpr (OP == ROW_LOGPROBS) launch_large_h<T, OP, false>(A, blocks, per, st);
  else if (A.out.hess) launch_large_h<T, OP, true>(A, blocks, per, st);
  else launch_large_h<T, OP, false>(A, blocks, per, st);
  return true;
}

template <typename T, int OP>
void launch_rows_t(const RowArgs<T>& A, cudaStream_t st) {
  if (A.in.n == 0) return;
  if (A.in.K <= kSmallClasses) {
    launch_small<T, OP>(A, st);
    MTB_CUDA_FB(cudaGetLastError());
    return;
  }
  if constexpr (sizeof(T) <= 4)
    if (launch_large<T, OP>(A, st)) return;
  const unsigned grid = (unsigned)std::min<long long>(A.in.n, 1 << 20);
  k_feedback_rows<T, OP><<<grid, kRowThreads, 0, st>>>(A);
  MTB_CUDA_FB(cudaGetLastError());
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

// ---------------------------------------------------------------------------
// Paired preference loss
// ---------------------------------------------------------------------------

// With u = (s_w - s_l) - (ref_w - ref_l) and x = beta u:
//   logistic  L = (1 - e) softplus(-x) + e softplus(x)
//             L' = beta (e sig(x) - (1 - e) sig(-x))
//             L'' = beta^2 sig(x) sig(-x)
//   squared   L = (u - 1 / (2 beta))^2
//
// An item's derivatives are a sum over its pairs, which the plan lists item by
// item: no atomics, and the same bits at every call.  Each pair's terms are
// computed for both of its items (a hundred instructions) rather than once and
// stored, which would take memory that calls share; the winner's side also
// writes the pair's loss.  What bounds it is the other item's score and
// reference, a sector of L2 each per entry, and the terms' arithmetic.
struct PairMath {
  double beta, smoothing, target;  // target: 1 / (2 beta)
  int kind;
};

template <typename T>
struct PairTerms {
  T g, h, loss;
};

// float64 scores: float64 throughout.  float32 scores: u is as good as exact
// (see Lean), and what follows is float32 arithmetic of a few steps' error.
__device__ __forceinline__ double pair_exp(double x, const TableMath& math) { return math.exp(x); }
__device__ __forceinline__ float pair_exp(float x, const TableMath&) { return expf(x); }
__device__ __forceinline__ double pair_inverse(double x) { return TableMath::inverse(x); }
__device__ __forceinline__ float pair_inverse(float x) { return __frcp_rn(x); }
__device__ __forceinline__ double pair_log1p(double x, const TableMath& math) { return math.log1p(x); }
__device__ __forceinline__ float pair_log1p(float x, const TableMath&) { return log1pf(x); }
__device__ __forceinline__ double flip(double x, int by) {  // x, negated where by is negative
  return __hiloint2double(__double2hiint(x) ^ (by & 0x80000000), __double2loint(x));
}
__device__ __forceinline__ float flip(float x, int by) { return __uint_as_float(__float_as_uint(x) ^ (by & 0x80000000u)); }

template <typename T>
__device__ __forceinline__ PairTerms<T> pair_terms(const PairMath& pm, T u, bool want_loss, const TableMath& math) {
  PairTerms<T> t;
  if (pm.kind == PREFERENCE_SQUARED) {
    const T d = u - (T)pm.target;
    return {(T)2 * d, (T)2, d * d};
  }
  const T beta = (T)pm.beta, x = beta * u, e = pair_exp(-fabs(x), math), r = pair_inverse((T)1 + e), er = e * r;
  const T down = x >= (T)0 ? er : r;  // sig(-x)
  const T keep = (T)(1.0 - pm.smoothing);
  t.g = -(beta * keep) * down;
  t.h = beta * beta * er * r;
  t.loss = (T)0;
  if (want_loss) {
    const T soft = pair_log1p(e, math);
    t.loss = keep * (soft + (x < (T)0 ? -x : (T)0));
    if (pm.smoothing > 0.0) t.loss += (T)pm.smoothing * (soft + (x > (T)0 ? x : (T)0));
    if (x != x) t.loss = x;
  }
  // apart, since an infinite x times a smoothing of 0 would be NaN
  if (pm.smoothing > 0.0) t.g += beta * (T)pm.smoothing * (x >= (T)0 ? r : er);
  return t;
}

template <typename T>
struct PreferenceArgs {
  const int* offsets;
  const int2* entries;
  const float* entry_w;
  const int* zero_pairs;
  int n_zero, n_items, long_from;
  const T *s, *ref;
  PairMath pm;
  T* loss;
  float *grad, *hess;
};

// An item's distance to its reference.  The difference of two float32 log
// probabilities of whole answers loses what the pair's difference needs, so it
// is kept with its rounding error (O. Moller, "Quasi double-precision in
// floating point addition", BIT 5, 1965).
template <typename T>
struct Lean;
template <>
struct Lean<double> {
  double v;
  __device__ __forceinline__ Lean(double s, double r) : v(s - r) {}
  __device__ __forceinline__ double minus(const Lean& o) const { return v - o.v; }
};
template <>
struct Lean<float> {
  float v, err;
  __device__ __forceinline__ Lean(float s, float r) {
    v = s - r;
    const float b = v - s;
    err = (s - (v - b)) - (r + b);
  }
  __device__ __forceinline__ float minus(const Lean& o) const {
    const float d = v - o.v, b = d - v;
    const float low = ((v - (d - b)) - (o.v + b)) + (err - o.err);
    return low == low ? d + low : d;  // infinities have no error terms
  }
};

template <typename T>
__device__ __forceinline__ Lean<T> lean(const PreferenceArgs<T>& A, int i) {
  return Lean<T>(A.s[i], A.ref ? A.ref[i] : (T)0);
}

// One entry of an item's list; `own` is the item's own distance to its reference.
template <typename T>
__device__ __forceinline__ void add_entry(const PreferenceArgs<T>& A, int2 entry, T w, const Lean<T>& own,
                                          const Lean<T>& other, const TableMath& math, double* g, double* h) {
  const PairTerms<T> t = pair_terms<T>(A.pm, flip(own.minus(other), entry.x), A.loss != nullptr, math);
  *g += (double)flip(w * t.g, entry.x);
  *h += (double)(w * t.h);
  if (A.loss && entry.x >= 0) A.loss[entry.y] = w * t.loss;
}

constexpr int kPairThreads = 256;
constexpr int kLongThreads = 128;
constexpr int kHugeThreads = 512;
constexpr int kPairCluster = 8;

// Lanes an item, by the mean number of an item's pairs: about eight steps of a
// lane, so that an item's own loads, sums of lanes and stores are shared by
// few instructions (all pairs in groups of 64, float64: 53 us with 32 lanes,
// 41 us with 8).
int pair_lanes(long long mean) { return mean < 8 ? 1 : mean < 32 ? 4 : mean < 128 ? 8 : 32; }

}  // namespace

// Items of more pairs than their lanes take in 24 steps have a block to
// themselves, or from 2048 pairs a cluster of 8: a lane's steps are one after
// the other, and a long item in a warp would be the last to end.
int PreferencePlan::long_from(long long n_entries, long long n_items) {
  return 24 * pair_lanes(n_entries / std::max(1ll, n_items)) + 1;
}

namespace {

constexpr int kHuge = 2048;

// The launches for huge, long and other items write apart from one another,
// so each lets the next begin at once; each ends only when the one before it
// has, so that the last one's end is the call's.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// G lanes an item.
template <typename T, int G>
__global__ void __launch_bounds__(kPairThreads) k_preference_items(const PreferenceArgs<T> A) {
  __shared__ MathTables tables;
  const TableMath math(tables, sizeof(T) == 8);
  const long long thread = (long long)blockIdx.x * kPairThreads + threadIdx.x;
  const long long threads = (long long)gridDim.x * kPairThreads;
  if (A.loss)
    for (long long z = thread; z < A.n_zero; z += threads) A.loss[A.zero_pairs[z]] = (T)0;
  const int l = threadIdx.x % G;
  for (long long at = thread / G; at < (A.n_items + 31) / 32 * 32ll; at += threads / G) {  // whole warps
    const int i = (int)min(at, (long long)A.n_items - 1);
    const int e0 = A.offsets[i], e1 = A.offsets[i + 1];
    const bool skip = at >= A.n_items || e1 - e0 >= A.long_from;
    double g = 0.0, h = 0.0;
    if (!skip && e0 + l < e1) {
      const Lean<T> own = lean(A, i);
      int2 c = A.entries[e0 + l];
      Lean<T> other = lean(A, c.x & 0x7fffffff);
      T w = A.entry_w ? (T)A.entry_w[e0 + l] : (T)1;
      for (int e = e0 + l; e < e1; e += G) {  // the next entry's loads while this one is computed
        const bool more = e + G < e1;
        const int2 cn = more ? A.entries[e + G] : c;
        const Lean<T> on = more ? lean(A, cn.x & 0x7fffffff) : other;
        const T wn = more && A.entry_w ? (T)A.entry_w[e + G] : w;
        add_entry(A, c, w, own, other, math, &g, &h);
        c = cn;
        other = on;
        w = wn;
      }
    }
#pragma unroll
    for (int k = G / 2; k > 0; k >>= 1) {
      g += __shfl_xor_sync(0xffffffffu, g, k);
      h += __shfl_xor_sync(0xffffffffu, h, k);
    }
    if (!skip && l == 0 && A.grad) {
      A.grad[i] = (float)g;
      A.hess[i] = (float)h;
    }
  }
  wait_for_previous();
}

// A block or cluster an item of the list.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_preference_long(const PreferenceArgs<T> A, const int* __restrict__ items,
                                                             const int n) {
  namespace cg = cooperative_groups;
  __shared__ MathTables tables;
  __shared__ double sm[2][2][THREADS / 32], sum[2][2];  // by the parity of the item
  let_next_begin();
  const TableMath math(tables, sizeof(T) == 8);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  int parity = 0;
  for (int at = blockIdx.x / blocks; at < n; at += gridDim.x / blocks, parity ^= 1) {
    const int i = items[at], e1 = A.offsets[i + 1], step = blocks * THREADS;
    const Lean<T> own = lean(A, i);
    double g = 0.0, h = 0.0;
    for (int e = A.offsets[i] + rank * THREADS + threadIdx.x; e < e1; e += 4 * step) {
      int2 c[4];
      T w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool there = e1 - e > q * step;
        c[q] = there ? A.entries[e + q * step] : make_int2(i, -1);
        w[q] = there && A.entry_w ? (T)A.entry_w[e + q * step] : (T)1;
      }
      const Lean<T> o[4] = {lean(A, c[0].x & 0x7fffffff), lean(A, c[1].x & 0x7fffffff), lean(A, c[2].x & 0x7fffffff),
                            lean(A, c[3].x & 0x7fffffff)};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c[q].y >= 0) add_entry(A, c[q], w[q], own, o[q], math, &g, &h);
    }
    for (int k = 16; k > 0; k >>= 1) {
      g += __shfl_xor_sync(0xffffffffu, g, k);
      h += __shfl_xor_sync(0xffffffffu, h, k);
    }
    if ((threadIdx.x & 31) == 0) {
      sm[parity][0][threadIdx.x >> 5] = g;
      sm[parity][1][threadIdx.x >> 5] = h;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      double t = 0.0;
      for (int k = 0; k < THREADS / 32; ++k) t += sm[parity][threadIdx.x][k];
      sum[parity][threadIdx.x] = t;
    }
    if (blocks > 1) cluster.sync();
    if (rank == 0 && threadIdx.x < 2 && A.grad) {
      double t = 0.0;
      for (int k = 0; k < blocks; ++k) t += *cluster.map_shared_rank(&sum[parity][threadIdx.x], k);
      (threadIdx.x ? A.hess : A.grad)[i] = (float)t;
    }
  }
  if (blocks > 1) cluster.sync();  // until the first block has read the sums
  wait_for_previous();
}

// after: this call's launch before this one, which it need not wait for.
template <typename K, typename... Args>
void launch_pairs(K kernel, unsigned grid, int threads, int blocks, bool after, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(grid);
  lc.blockDim = dim3(threads);
  lc.stream = st;
  cudaLaunchAttribute attr[2];
  lc.attrs = attr;
  lc.numAttrs = 0;
  if (blocks > 1) {
    cudaLaunchAttribute& a = attr[lc.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = blocks;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
  }
  if (after) {
    cudaLaunchAttribute& a = attr[lc.numAttrs++];
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
  }
  MTB_CUDA_FB(cudaLaunchKernelEx(&lc, kernel, args...));
}

template <typename T, int G>
void launch_preference_items(const PreferenceArgs<T>& A, bool after, cudaStream_t st) {
  const long long blocks = ((long long)A.n_items * G + kPairThreads - 1) / kPairThreads;
  const unsigned grid = (unsigned)std::min<long long>(blocks, 16ll * multiprocessors());
  launch_pairs(k_preference_items<T, G>, grid, kPairThreads, 1, after, st, A);
}

template <typename T>
void launch_preference_t(const PreferencePlan& plan, const PreferenceTerms& t, cudaStream_t st) {
  if (plan.n_items == 0) return;
  PreferenceArgs<T> A;
  A.offsets = plan.offsets;
  A.entries = plan.entries;
  A.entry_w = plan.entry_w;
  A.zero_pairs = plan.zero_pairs;
  A.n_zero = (int)plan.n_zero;
  A.n_items = (int)plan.n_items;
  A.long_from = PreferencePlan::long_from(plan.n_entries, plan.n_items);
  A.s = static_cast<const T*>(t.scores);
  A.ref = static_cast<const T*>(t.reference);
  A.pm = {t.beta, t.smoothing, 1.0 / (2.0 * t.beta), t.kind};
  A.loss = static_cast<T*>(t.loss);
  A.grad = t.grad;
  A.hess = t.hess;
  // long items first: they take longest
  const bool huge = plan.n_huge > 0, any = huge || plan.n_long > 0;
  if (huge)
    launch_pairs(k_preference_long<T, kHugeThreads>,
                 (unsigned)std::min<long long>(plan.n_huge, multiprocessors() / 4) * kPairCluster, kHugeThreads,
                 kPairCluster, false, st, A, (const int*)plan.huge_items, (int)plan.n_huge);
  if (plan.n_long > 0)
    launch_pairs(k_preference_long<T, kLongThreads>,
                 (unsigned)std::min<long long>(plan.n_long, 8ll * multiprocessors()), kLongThreads, 1, huge, st, A,
                 (const int*)plan.long_items, (int)plan.n_long);
  switch (pair_lanes(plan.n_entries / plan.n_items)) {
    case 1: launch_preference_items<T, 1>(A, any, st); break;
    case 4: launch_preference_items<T, 4>(A, any, st); break;
    case 8: launch_preference_items<T, 8>(A, any, st); break;
    default: launch_preference_items<T, 32>(A, any, st);
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

PreferencePlan::~PreferencePlan() { cudaFree(memory); }

void PreferencePlan::check(const int64_t* winners, const int64_t* losers, const float* weights, long long np,
                           long long ni) {
  int fault = 0;  // the largest of: 1 weight, 2 itself, 3 range
#pragma omp parallel for schedule(static) reduction(max : fault) if (np > 65536)
  for (long long p = 0; p < np; ++p) {
    const int64_t a = winners[p], b = losers[p];
    if (a < 0 || a >= ni || b < 0 || b >= ni) fault = std::max(fault, 3);
    else if (a == b) fault = std::max(fault, 2);
    else if (weights && !(weights[p] >= 0.0f && std::isfinite(weights[p]))) fault = std::max(fault, 1);
  }
  if (fault == 3) throw std::invalid_argument("pair item out of range");
  if (fault == 2) throw std::invalid_argument("an item is paired with itself");
  if (fault == 1) throw std::invalid_argument("pair weights must be finite and non-negative");
}

// Two passes of a counting sort, both in the pairs' order and on all host
// threads: pairs into ranges of items, then each range's by item, within a
// core's cache.
void PreferencePlan::build(const int64_t* winners, const int64_t* losers, const float* weights, long long np,
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
  std::vector<int> zero((size_t)zero_at[parts]), off((size_t)ni + 1);
  std::unique_ptr<int2[]> ent(new int2[std::max(1ll, total)]);
  std::unique_ptr<float[]> ew(new float[weights ? std::max(1ll, total) : 1]);
#pragma omp parallel for schedule(static, 1) if (parts > 1)
  for (int t = 0; t < parts; ++t) {
    long long* c = &count[(size_t)t * kRanges];
    long long z = zero_at[t];
    for (long long p = slice(t); p < slice(t + 1); ++p) {
      const int a = (int)winners[p], b = (int)losers[p];
      const float w = weights ? weights[p] : 1.0f;
      if (w == 0.0f) {
        zero[z++] = (int)p;
        continue;
      }
      sorted[c[a / range]++] = {a, make_int2(b, (int)p), w};
      sorted[c[b / range]++] = {b, make_int2(a | (int)0x80000000, (int)p), w};
    }
  }
#pragma omp parallel for schedule(dynamic, 1) if (parts > 1)
  for (int q = 0; q < kRanges; ++q) {
    const long long i0 = std::min(ni, q * range), i1 = std::min(ni, i0 + range);
    if (i0 >= i1) continue;
    std::vector<int> at((size_t)(i1 - i0) + 1, 0);
    for (long long e = start[q]; e < start[q + 1]; ++e) ++at[sorted[e].item - i0 + 1];
    int sum = (int)start[q];
    for (long long i = i0; i < i1; ++i) {
      off[i] = sum;
      const int n = at[i - i0 + 1];
      at[i - i0] = sum;
      sum += n;
    }
    for (long long e = start[q]; e < start[q + 1]; ++e) {
      const int to = at[sorted[e].item - i0]++;
      ent[to] = sorted[e].e;
      if (weights) ew[to] = sorted[e].w;
    }
  }
  off[ni] = (int)total;
  std::vector<int> lng, huge;
  const int from = long_from(total, ni);
  for (long long i = 0; i < ni; ++i) {
    const int d = off[i + 1] - off[i];
    if (d < from) continue;
    (d >= std::max(kHuge, from) ? huge : lng).push_back((int)i);
  }
  // one allocation, each array on 256 bytes
  MTB_CUDA_FB(cudaGetDevice(&device));
  size_t bytes = 0;
  struct Copy {
    const void* from;
    size_t n, at;
  };
  std::vector<Copy> copies;
  auto add = [&](const void* from, size_t n) {
    copies.push_back({from, n, bytes});
    bytes += (n + 255) / 256 * 256;
    return copies.back().at;
  };
  const size_t at_off = add(off.data(), 4 * off.size()), at_ent = add(ent.get(), 8 * (size_t)total),
               at_w = add(ew.get(), weights ? 4 * (size_t)total : 0), at_zero = add(zero.data(), 4 * zero.size()),
               at_long = add(lng.data(), 4 * lng.size()), at_huge = add(huge.data(), 4 * huge.size());
  MTB_CUDA_FB(cudaMalloc(&memory, bytes));
  char* base = static_cast<char*>(memory);
  for (const Copy& c : copies)
    if (c.n) MTB_CUDA_FB(cudaMemcpy(base + c.at, c.from, c.n, cudaMemcpyHostToDevice));
  n_items = ni;
  n_pairs = np;
  n_entries = total;
  n_zero = (long long)zero.size();
  n_long = (long long)lng.size();
  n_huge = (long long)huge.size();
  offsets = reinterpret_cast<int*>(base + at_off);
  entries = reinterpret_cast<int2*>(base + at_ent);
  entry_w = weights ? reinterpret_cast<float*>(base + at_w) : nullptr;
  zero_pairs = reinterpret_cast<int*>(base + at_zero);
  long_items = reinterpret_cast<int*>(base + at_long);
  huge_items = reinterpret_cast<int*>(base + at_huge);
}

int launch_preference(const PreferencePlan& plan, const PreferenceTerms& t, cudaStream_t st) {
  if (t.type == SCORE_F64) launch_preference_t<double>(plan, t, st);
  else launch_preference_t<float>(plan, t, st);
  return plan.n_items > 0 ? 1 + (plan.n_huge > 0 ? 1 : 0) + (plan.n_long > 0 ? 1 : 0) : 0;
}

}  // namespace mtb

// ---------------------------------------------------------------------------
// C entry points
// ---------------------------------------------------------------------------

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

// Makes a device current for a call, and the caller's again after it.
struct DeviceScope {
  int before = -1;
  bool moved = false;
  explicit DeviceScope(int dev) {
    MTB_CUDA_FB(cudaGetDevice(&before));
    if (dev >= 0 && dev != before) {
      MTB_CUDA_FB(cudaSetDevice(dev));
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
    require(label_smoothing >= 0.0 && label_smoothing <= 0.5, "label_smoothing must be in [0, 0.5]");
    require(loss_kind == mtb::PREFERENCE_LOGISTIC || loss_kind == mtb::PREFERENCE_SQUARED, "unknown preference loss");
    require(loss_kind == mtb::PREFERENCE_LOGISTIC || label_smoothing == 0.0, "label_smoothing needs the logistic loss");
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
