// Row kernels for many classes.
#pragma once
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "feedback_rows.cuh"

namespace mtb {
namespace {

// ---------------------------------------------------------------------------
// Rows of more than 128 classes, scores of 32 and 16 bits
//
// A block (or a cluster of up to 8 of them, where a row is longer than 8192
// vectors of 16 bytes, or rows are too few to fill the GPU) holds a row in its
// registers: the scores are read once.  A class takes two exponentials (the
// sum's, and the gradient's again: kept in float32 they would take twice the
// registers).  Each warp sums relative to its own maximum, so one barrier joins
// maxima and sums; the next row is fetched into L2 meanwhile.
//
// Measured, policy loss with gradient of 8192 x 32768 bfloat16 (1.07 GB,
// 164 us at the copy rate): 233 us.  No unit is full (DRAM 55%, exponentials
// 55%, issue slots 50%): the block waits for its row's scalars, which one warp
// makes (a quarter of the stalls), and 64 registers a thread spill 122 bytes out
// and 146 back in.  The gradient's pass alone, which needs no sum, takes 200, and
// for 2047 x 50001 69 of 62 at the copy rate.  Rows kept in shared memory instead, three blocks an SM,
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

// Up to 2^24, c is within 1 of log2(e) m.  Far beyond, `shift` would leave
// float32's exponents, and c itself at the type's end.  A warp that lies
// farther than kFarWarp leaves its sum out (0, with its maximum): it matters
// only to a row whose own maximum is farther than kFarRow, as a warp of masked
// classes is e^-8000000 of any other row.  Such rows are left to far_rows, which
// takes their exponentials of z - m.  float16 holds no such score.
constexpr float kFarWarp = 0x1p24f, kFarRow = 0x1p23f;

template <typename T>
__device__ __forceinline__ bool is_far(float m) {
  return !std::is_same<T, __half>::value && fabsf(m) > kFarRow;
}

enum RowState : int { ROW_EMPTY = 0, ROW_DONE = 1, ROW_SLOW = 2, ROW_NEAR = 3, ROW_FAR = 4 };

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

// A far row's derivatives; 0 without `live`.
template <typename T, bool HESS>
__device__ __noinline__ void far_derivatives(const RowArgs<T>& A, long long r, float m, float g, float h, float inv,
                                             float share, bool live) {
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const T* z = A.in.scores + r * A.in.stride;
  const long long a = A.in.action(r), to = r * A.out.row_stride;
  for (int k = cluster.thread_rank(); k < A.in.K; k += cluster.num_threads()) {
    const float f = widen(z[k]), p = exp2_approx((f - m) * kLog2e) * inv, left = f == m ? share : 1.0f - p;
    const float q = k == a ? left : -p;
    narrow(live ? g * q : 0.0f, A.out.grad[to + k]);
    if (HESS) narrow(live ? h * q * q + fabsf(g) * p * left : 0.0f, A.out.hess[to + k]);
  }
}

// The far rows among this block's or cluster's, after all others: their
// elements are read again, and summed in float64.  Apart from the loop over
// rows, which has no registers left for it: called in there it took 2 to 10%
// more time for other rows, called behind it 1 to 3%, inlined there -3 to 4%.
template <typename T, int OP, bool HESS, int THREADS>
__device__ __forceinline__ void far_rows(const RowArgs<T>& A, LargeShared<THREADS>& S, const TableMath math) {
  namespace cg = cooperative_groups;
  using Row = typename Types<T>::Row;
  constexpr int kWarps = THREADS / 32;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = A.in.K;
  // Every block of the cluster sums what every block has: no joins between blocks.
  for (long long r = blockIdx.x / blocks; r < A.in.n; r += gridDim.x / blocks) {
    const T* z = A.in.scores + r * A.in.stride;
    const long long a = A.in.action(r);
    if (a < 0 || a >= K || (OP == ROW_POLICY && A.pol.weights && A.pol.weights[r] == (Row)0)) continue;
    float m = -INFINITY;
    for (int k = threadIdx.x; k < K; k += THREADS) m = max_nan32(m, widen(z[k]));
    for (int k = 16; k > 0; k >>= 1) m = max_nan32(m, __shfl_xor_sync(0xffffffffu, m, k));
    __syncthreads();
    if (lane == 0) S.warp[0][warp].m = m;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) m = max_nan32(m, S.warp[0][i].m);
    if (!is_far<T>(m) || m == -INFINITY) continue;
    double sum = 0.0;  // less the terms at the maximum
    int ones = 0;
    for (int k = threadIdx.x; k < K; k += THREADS) {
      const double d = (double)widen(z[k]) - (double)m;  // NaN at a maximum of infinity
      if (d == 0.0) ++ones;
      else sum += math.exp(d);
    }
    const Part p = add_parts({sum, m, 0.0f, ones}, 32);
    if (lane == 0) S.slow[0][warp] = p;
    __syncthreads();
    sum = 0.0;
    ones = -1;
    for (int i = 0; i < kWarps; ++i) {
      sum += S.slow[0][i].sum;
      ones += S.slow[0][i].ones;
    }
    const double rest = sum + (double)ones, za = (double)widen(z[a]), lp = za - (double)m - math.log1p(rest);
    if (OP == ROW_LOGPROBS) {
      if (rank == 0 && threadIdx.x == 0) {
        A.logp[r] = (Row)lp;
        A.stats[2 * r] = m;
        A.stats[2 * r + 1] = (Row)rest;
      }
      continue;
    }
    double loss = 0.0;
    RowDerivative d = {0.0, 0.0};
    const bool live = za != -INFINITY;
    if (live)
      d = policy_terms(A.pol, lp, (double)A.pol.advantages[r], (double)A.pol.old_logp[r],
                       A.pol.ref_logp ? (double)A.pol.ref_logp[r] : 0.0, A.pol.weights ? (double)A.pol.weights[r] : 1.0,
                       &loss, math);
    if (rank == 0 && threadIdx.x == 0) {
      if (A.pol.loss) A.pol.loss[r] = (Row)loss;
      if (A.pol.logp) A.pol.logp[r] = (Row)lp;
    }
    if (!A.out.grad) continue;
    const double inv64 = TableMath::inverse(1.0 + rest);
    const float g = (float)d.g, h = (float)d.h, inv = (float)inv64, share = (float)(rest * inv64);
    far_derivatives<T, HESS>(A, r, m, g, h, inv, share, live);
  }
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
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_feedback_large(const __grid_constant__ RowArgs<T> A,
                                                                             const int per) {
  namespace cg = cooperative_groups;
  using Row = typename Types<T>::Row;
  constexpr int N = Vec<T>::N, kWarps = THREADS / 32;
  __shared__ LargeShared<THREADS> S;
  const TableMath math(S.tables, OP != ROW_BACK);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = A.in.K;
  const Pair scale = Pair::of(kLog2e, kLog2e);
  const long long clusters = gridDim.x / blocks;
  int parity = 0;
  bool far = false;
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
        if (is_far<T>(m)) {
          far_derivatives<T, HESS>(A, r, m, g, h, inv_total, rest * inv_total, true);
          continue;
        }
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
      if (!(fabsf(wm) > kFarWarp)) {
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
        if (all.m == -INFINITY || rest < 1.0 || is_far<T>(all.m)) {
          if (lane == 0) {
            S.state = all.m == -INFINITY ? ROW_EMPTY : is_far<T>(all.m) ? ROW_FAR : ROW_SLOW;
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
      if (!std::is_same<T, __half>::value && S.state == ROW_FAR) {
        far = true;
        continue;
      }
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
  if constexpr (!std::is_same<T, __half>::value && OP != ROW_BACK) {
    if (far) far_rows<T, OP, HESS, THREADS>(A, S, math);
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

// The smallest block that holds the row: as many rows as possible are under way
// an SM.  One size up, policy loss of 200M bfloat16 scores: 200 classes 870 ->
// 1099 us, 400 577 -> 1534, 2000 371 -> 684, 6000 270 -> 484, 12000 274 -> 366,
// 24000 210 -> 369.
template <typename T, int OP, bool HESS>
void launch_large_h(const RowArgs<T>& A, int blocks, int per, cudaStream_t st) {
  if (per > 4096) launch_large_t<T, OP, HESS, 1024, 8>(A, blocks, per, st);
  else if (per > 2048) launch_large_t<T, OP, HESS, 512, 8>(A, blocks, per, st);
  else if (per > 1024) launch_large_t<T, OP, HESS, 512, 4>(A, blocks, per, st);
  else if (per > 512) launch_large_t<T, OP, HESS, 256, 4>(A, blocks, per, st);
  else if (per > 128) launch_large_t<T, OP, HESS, 128, 4>(A, blocks, per, st);
  else if (per > 32) launch_large_t<T, OP, HESS, 32, 4>(A, blocks, per, st);
  else launch_large_t<T, OP, HESS, 32, 1>(A, blocks, per, st);
}

// Derivatives next to each other (class_stride 1), as every caller with such
// scores has them.  Clusters for few rows, kernel time of float16 policy rows
// with one block a row, and with these clusters: 1 x 131072 12.2, 6.8 us; 18 x
// 131072 12.7, 8.4; 37 x 20000 9.3, 7.3; 37 x 8000 5.3, 5.9.  From 128 vectors a
// block on instead of 512: 37 x 2000 5.5 -> 7.2.
template <typename T, int OP>
void launch_large(const RowArgs<T>& A, cudaStream_t st) {
  const int vecs = A.in.K / Vec<T>::N;  // or one fewer, where a row does not start on 16 bytes
  static_assert(kMaxClasses / 4 <= 8 * 8192, "a cluster's registers hold the longest float32 row");
  int blocks = 1;
  while (blocks < 8 && (vecs > 8192 * blocks || (vecs > 512 * blocks && A.in.n * blocks * 2 <= multiprocessors()))) blocks *= 2;
  const int per = (vecs + blocks - 1) / blocks;
  if constexpr (OP == ROW_LOGPROBS) launch_large_h<T, OP, false>(A, blocks, per, st);
  else if (A.out.hess) launch_large_h<T, OP, true>(A, blocks, per, st);
  else launch_large_h<T, OP, false>(A, blocks, per, st);
}

}  // namespace
}  // namespace mtb
