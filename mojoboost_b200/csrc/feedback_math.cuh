// Shared by the kernels of the losses from feedback: error checks and float64
// functions by table.
#pragma once
#include <cuda_runtime.h>
#include <math.h>

#include <atomic>
#include <stdexcept>
#include <string>

namespace mtb {
namespace {

#define MTB_CUDA_FB(call)                                                                    \
  do {                                                                                       \
    cudaError_t e_ = (call);                                                                 \
    if (e_ != cudaSuccess)                                                                   \
      throw std::runtime_error(std::string("CUDA error: ") + cudaGetErrorString(e_) + " at " \
                               + #call);                                                     \
  } while (0)

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

}  // namespace
}  // namespace mtb
