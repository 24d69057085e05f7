// The paired preference loss with its gradient and hessian, and the plan of
// its pairs.
#include <cooperative_groups.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <stdexcept>
#include <vector>

#include "feedback.h"
#include "feedback_math.cuh"
#include "feedback_plan.h"
#include "trainer.h"

namespace mtb {
namespace {

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
//
// Measured: 1M pairs of 2M items, float64 with reference, 36 us (64 MB of
// arrays, 10 us at the copy rate; 4M random sectors); 2M pairs within groups of
// 64, 39 us (issue slots 64% busy); 4M pairs of popular items, float32, 129 us.
struct PairMath {
  double beta, smoothing, target;  // target: 1 / (2 beta)
  int kind;
};

template <typename T>
struct PairTerms {
  T g, h, loss;
};

// float64 scores: float64 throughout.  float32 scores: u is as good as exact
// (see Lean), the squared loss's distance to its target is rounded once, and
// what follows is float32 arithmetic of a few steps' error.
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

// A pair's difference: hi + low, low being what float32 scores' hi leaves out.
template <typename T>
struct Difference {
  T hi, low;
  __device__ __forceinline__ T value() const { return hi + low; }
  __device__ __forceinline__ T less(double target) const { return (T)((double)hi - target + (double)low); }
};
template <>
struct Difference<double> {
  double hi;
  __device__ __forceinline__ double value() const { return hi; }
  __device__ __forceinline__ double less(double target) const { return hi - target; }
};
__device__ __forceinline__ Difference<double> flip(Difference<double> d, int by) { return {flip(d.hi, by)}; }
__device__ __forceinline__ Difference<float> flip(Difference<float> d, int by) { return {flip(d.hi, by), flip(d.low, by)}; }

template <typename T>
__device__ __forceinline__ PairTerms<T> pair_terms(const PairMath& pm, Difference<T> u, bool want_loss, const TableMath& math) {
  PairTerms<T> t;
  if (pm.kind == PREFERENCE_SQUARED) {
    const T d = u.less(pm.target);
    return {(T)2 * d, (T)2, d * d};
  }
  const T beta = (T)pm.beta, x = beta * u.value(), e = pair_exp(-fabs(x), math), r = pair_inverse((T)1 + e), er = e * r;
  const T down = x >= (T)0 ? er : r;  // sig(-x)
  const T keep = (T)(1.0 - pm.smoothing);
  t.g = -(beta * keep) * down;
  t.h = beta * er * (beta * r);  // beta's square may be beyond the type where this is 0
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
  __device__ __forceinline__ Difference<double> minus(const Lean& o) const { return {v - o.v}; }
};
template <>
struct Lean<float> {
  float v, err;
  __device__ __forceinline__ Lean(float s, float r) {
    v = s - r;
    const float b = v - s;
    err = (s - (v - b)) - (r + b);
  }
  __device__ __forceinline__ Difference<float> minus(const Lean& o) const {
    const float d = v - o.v, b = d - v;
    const float low = ((v - (d - b)) - (o.v + b)) + (err - o.err);
    return {d, low == low ? low : 0.0f};  // infinities have no error terms
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
  // One block an SM's place, whose start is then paid once (1M pairs apart: 41
  // -> 36 us); with long items about, items differ enough that blocks queueing
  // for places balance better (popular items: 135 -> 127 us).
  static std::atomic<int> known{0};
  const int resident = after ? 16 : resident_blocks(k_preference_items<T, G>, kPairThreads, 0, known);
  const long long most = (long long)multiprocessors() * resident;
  launch_pairs(k_preference_items<T, G>, (unsigned)std::min(blocks, most), kPairThreads, 1, after, st, A);
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
  A.long_from = pairs_long_from(plan.n_entries, plan.n_items);
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

// The memory comes from the fits' cache: allocating and freeing took 0.6 ms a
// plan, more than the loss of most batches.
PreferencePlan::~PreferencePlan() {
  if (!memory) return;
  int before = -1;
  const bool known = cudaGetDevice(&before) == cudaSuccess;
  if (cudaSetDevice(device) == cudaSuccess) give_device_memory(memory, memory_bytes);
  if (known) cudaSetDevice(before);
}

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

void PreferencePlan::build(const int64_t* winners, const int64_t* losers, const float* weights, long long np,
                           long long ni) {
  const SortedPairs s = sort_pairs(winners, losers, weights, np, ni);
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
  const size_t at_off = add(s.offsets.get(), 4 * ((size_t)ni + 1)), at_ent = add(s.entries.get(), 8 * (size_t)s.n_entries),
               at_w = add(s.weights.get(), weights ? 4 * (size_t)s.n_entries : 0),
               at_zero = add(s.zero_pairs.get(), 4 * (size_t)s.n_zero),
               at_long = add(s.long_items.get(), 4 * (size_t)s.n_long),
               at_huge = add(s.huge_items.get(), 4 * (size_t)s.n_huge);
  memory_bytes = bytes;
  memory = take_device_memory(&memory_bytes);
  char* base = static_cast<char*>(memory);
  // A copy from pageable memory may return before it has arrived, and the
  // streams that will read the plan need not be ordered behind this one: the
  // copies are waited for.
  const cudaStream_t st = cudaStreamPerThread;
  if (bytes <= 1 << 20) {  // a copy costs more than its bytes
    std::vector<char> all(bytes);
    for (const Copy& c : copies)
      if (c.n) memcpy(&all[c.at], c.from, c.n);
    MTB_CUDA_FB(cudaMemcpyAsync(base, all.data(), bytes, cudaMemcpyHostToDevice, st));
    MTB_CUDA_FB(cudaStreamSynchronize(st));
  } else {
    for (const Copy& c : copies)
      if (c.n) MTB_CUDA_FB(cudaMemcpyAsync(base + c.at, c.from, c.n, cudaMemcpyHostToDevice, st));
    MTB_CUDA_FB(cudaStreamSynchronize(st));
  }
  n_items = ni;
  n_pairs = np;
  n_entries = s.n_entries;
  n_zero = s.n_zero;
  n_long = s.n_long;
  n_huge = s.n_huge;
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
