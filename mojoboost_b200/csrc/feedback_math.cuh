// Shared by the kernels of the losses from feedback: error checks and float64
// functions by table.
#pragma once
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
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

// 2^(j / 64), then 0; rounded from 50 digits, as the tables below.
__device__ const double kTwoTo[65] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138, 1.0556451783605572,
    1.0671404006768237, 1.0787607977571199, 1.0905077326652577, 1.102382583307841, 1.1143867425958924,
    1.1265216186082418, 1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687, 1.241857812073484, 1.255380757024691,
    1.2690509571917332, 1.2828700160787783, 1.2968395546510096, 1.3109612115247644, 1.3252366431597413,
    1.339667524053303, 1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647, 1.4768261459394993,
    1.4929077282912648, 1.5091644275934228, 1.5255981507445384, 1.5422108254079407, 1.559004400237837,
    1.5759808451078865, 1.593142151342267, 1.6104903319492543, 1.6280274218573478, 1.645755478153965,
    1.6636765803267364, 1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989, 1.8340080864093424,
    1.8539791250833855, 1.8741676341103, 1.8945759815869656, 1.9152065613971474, 1.9360617934922943,
    1.9571441241754002, 1.978456026387951, 0.0};
// 64 / (64 + j).
__device__ const double kInverse[64] = {
    1.0, 0.9846153846153847, 0.9696969696969697, 0.9552238805970149, 0.9411764705882353, 0.927536231884058,
    0.9142857142857143, 0.9014084507042254, 0.8888888888888888, 0.8767123287671232, 0.8648648648648649,
    0.8533333333333334, 0.8421052631578947, 0.8311688311688312, 0.8205128205128205, 0.810126582278481, 0.8,
    0.7901234567901234, 0.7804878048780488, 0.7710843373493976, 0.7619047619047619, 0.7529411764705882,
    0.7441860465116279, 0.735632183908046, 0.7272727272727273, 0.7191011235955056, 0.7111111111111111,
    0.7032967032967034, 0.6956521739130435, 0.6881720430107527, 0.6808510638297872, 0.6736842105263158,
    0.6666666666666666, 0.6597938144329897, 0.6530612244897959, 0.6464646464646465, 0.64, 0.6336633663366337,
    0.6274509803921569, 0.6213592233009708, 0.6153846153846154, 0.6095238095238096, 0.6037735849056604,
    0.5981308411214953, 0.5925925925925926, 0.5871559633027523, 0.5818181818181818, 0.5765765765765766,
    0.5714285714285714, 0.5663716814159292, 0.5614035087719298, 0.5565217391304348, 0.5517241379310345,
    0.5470085470085471, 0.5423728813559322, 0.5378151260504201, 0.5333333333333333, 0.5289256198347108,
    0.5245901639344263, 0.5203252032520326, 0.5161290322580645, 0.512, 0.5079365079365079, 0.5039370078740157};
// log((64 + j) / 64).
__device__ const double kLog[64] = {
    0.0, 0.015504186535965254, 0.030771658666753687, 0.0458095360312942, 0.06062462181643484, 0.07522342123758753,
    0.08961215868968714, 0.10379679368164356, 0.11778303565638346, 0.13157635778871926, 0.1451820098444979,
    0.15860503017663857, 0.17185025692665923, 0.184922338494012, 0.19782574332991987, 0.21056476910734964,
    0.22314355131420976, 0.2355660713127669, 0.24783616390458127, 0.25995752443692605, 0.27193371548364176,
    0.2837681731306446, 0.2954642128938359, 0.3070250352949119, 0.3184537311185346, 0.329753286372468,
    0.3409265869705932, 0.3519764231571782, 0.3629054936893685, 0.37371640979358406, 0.38441169891033206,
    0.394993808240869, 0.4054651081081644, 0.415827895143711, 0.4260843953109001, 0.43623676677491807,
    0.44628710262841953, 0.4562374334815876, 0.46608972992459924, 0.4758459048699639, 0.4855078157817008,
    0.4950772667978515, 0.5045560107523953, 0.5139457511022343, 0.5232481437645479, 0.5324647988694718,
    0.5415972824327444, 0.5506471179526623, 0.5596157879354227, 0.5685047353526688, 0.5773153650348236,
    0.5860490450035782, 0.5947071077466928, 0.6032908514380843, 0.6118015411059929, 0.6202404097518576,
    0.6286086594223741, 0.6369074622370692, 0.6451379613735847, 0.6533012720127457, 0.661398482245365,
    0.6694306539426292, 0.6773988235918061, 0.6853040030989194};

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
    for (int j = threadIdx.x; j < 65; j += blockDim.x) t->two[j] = kTwoTo[j];
    for (int j = threadIdx.x; j < 64; j += blockDim.x) {
      t->inv_c[j] = kInverse[j];
      t->log_c[j] = kLog[j];
    }
    __syncthreads();
  }
  // exp(d) / 2^less, d <= 709 + less: d = (n / 64) ln 2 + r, exp(d) = 2^(n / 64)
  // (1 + r + ... + r^5 / 120), |r| <= ln 2 / 128, truncation below 2^-54.  NaN
  // stays; below -708 (3e-308) the value is 0.
  __device__ __forceinline__ double exp(double d, int less = 0) const {
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
    const double scaled = __hiloint2double(__double2hiint(two_n) + ((n >> 6) - less << 20), __double2loint(two_n));
    return fma(scaled, q, scaled);
  }
  __device__ __forceinline__ float exp(float d) const { return __expf(d); }
  // exp(d) for any d: the last binade by its half, whose scale still has an exponent.
  __device__ __forceinline__ double operator()(double d) const {
    const int less = d > 709.0 ? 1 : 0;
    const double e = exp(d, less);
    return d > 709.79 ? INFINITY : less ? e + e : e;
  }
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

// Blocks of a kernel that an SM holds at once, for the grids of kernels whose
// blocks loop: each block's start (tables, the first rows' way from memory)
// is paid once.  The registers are asked for once per kernel.
template <typename K>
int resident_blocks(K kernel, int threads, size_t dynamic_smem, std::atomic<int>& known) {
  int packed = known.load(std::memory_order_relaxed);  // registers a thread, and static shared memory in 16 bytes
  if (packed == 0) {
    cudaFuncAttributes a;
    MTB_CUDA_FB(cudaFuncGetAttributes(&a, kernel));
    packed = a.numRegs | (int)((a.sharedSizeBytes + 15) / 16) << 8;
    known.store(packed, std::memory_order_relaxed);
  }
  const int warps = threads / 32, regs = ((packed & 255) + 7) / 8 * 8 * 32 * warps;
  const size_t smem = dynamic_smem + 16 * (size_t)(packed >> 8) + 1024;
  const int by_smem = (int)(228 * 1024 / smem);
  return std::max(1, std::min(std::min(65536 / regs, by_smem), std::min(64 / warps, 32)));
}

}  // namespace
}  // namespace mtb
