// Row kernels for few classes.
#pragma once
#include <algorithm>

#include "feedback_rows.cuh"

namespace mtb {
namespace {

// ---------------------------------------------------------------------------
// Rows of up to 128 classes, of float64 scores up to 512
//
// A warp copies 32 / L whole rows into shared memory, L lanes take a row each
// (class l + L e in lane l, at most 16 a lane), and the derivatives go back
// through the same memory, so every array crosses the memory system once and
// in one piece per warp.  With L = 1 (up to 16 classes) no lane waits for
// another.  A row's float64 scalars, a logarithm, two exponentials and a
// quotient, cost as much as ten classes; every lane of a row computes them.
//
// Measured, policy loss with gradient and hessian of 4M x 10 float64 (816 MB,
// 125 us at the copy rate): 190 us.  What is left is latency: 120 registers
// leave room for a quarter of the warps an SM could hold, which fill 62% of the
// issue slots and 47% of DRAM with about 1050 instructions for 32 rows, a third
// of them float64.  A block per row took 20.2 ms; rows spread
// over four lanes' registers 396 us; a branch per class 309 us, and classes
// fixed at compile time with the next rows' copy in flight 224 us, since a
// lane's exponentials then overlap; bulk copies and the branch-free functions
// of TableMath 195 us.  Fewer registers for five or six blocks an SM instead
// of four cost 10 and 13%.
// ---------------------------------------------------------------------------

constexpr int kSmallThreads = 128;
constexpr int kSmallPer = 16;  // classes a lane
// Most classes: with 16 and 32 lanes a row, float64 rows are still five times as
// fast as a block per row (50000 x 200, log probabilities: 33 us against 196);
// 16-bit rows gain nothing on a warp that holds them as whole vectors (100000 x
// 400 bfloat16: 64 us against 62, the gradient 84 against 55).
template <typename T>
constexpr int kSmallClasses = (sizeof(T) == 8 ? 32 : 8) * kSmallPer;

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
  // How many of a lane's classes every row of this variant has (launch_small):
  // no guards for them.
  constexpr int kSure = L > 1 ? P / 2 : sizeof(T) == 2 ? 1 : sizeof(T) == 4 ? (P == 4 ? 1 : P / 2 + 1) : P == 16 ? 13 : P - 1;
  auto has = [&](int e, int l, int K) { return e < kSure || l + e * L < K; };
  // In float64 a sum that holds the 1 of the largest class gives the others'
  // to 2^-43 of it unless it is below 2^-10, far beyond what the float32
  // derivatives keep; the statistics keep it whole.
  constexpr bool kExact = sizeof(C) == 4 || OP == ROW_LOGPROBS;
  constexpr double kNearOne = 0x1p-10;
  extern __shared__ __align__(16) unsigned char small_smem[];
  __shared__ MathTables tables;
  __shared__ __align__(8) unsigned long long barriers[kSmallThreads / 32][2];
  const TableMath math(tables, sizeof(C) == 8 || OP != ROW_BACK);
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
    for (int e = 0; e < P; ++e) v[e] = has(e, l, K) ? (C)widen(z[l + e * L]) : (C)-INFINITY;
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
      if (kExact || __any_sync(0xffffffffu, exact)) {
#pragma unroll
        for (int e = 0; e < P; ++e) top = v[e] == (C)1 && exact ? l + e * L : top;
      }
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
        const bool near = part && !bad && near_border(A.pol, lp - now.old, now.adv, border_slack(P + 5, 6.3));
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
      const C down = -g * inv, ag = fabs(g), bend = ag < (C)INFINITY ? h - ag : (C)0;
#pragma unroll
      for (int e = 0; e < P; ++e)
        if (has(e, l, K)) narrow(v[e] * down, to_g[l + e * L]);
      if (want_h) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const C p = v[e] * inv;
          if (has(e, l, K)) narrow(p * fma(p, bend, ag), to_h[l + e * L]);
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
  const size_t smem = (size_t)lay.tile * 2 * warps;
  static std::atomic<int> known{0};
  const long long most = (long long)multiprocessors() * resident_blocks(k_feedback_small<T, OP, L, P>, kSmallThreads, smem, known);
  k_feedback_small<T, OP, L, P><<<(unsigned)std::min(blocks, most), kSmallThreads, smem, st>>>(A, lay);
}

// Few classes fit one lane; a class too many in P costs a float64 exponential
// a row (20 instructions of about 100 a class), a float32 one next to nothing.
template <typename T, int OP>
void launch_small(const RowArgs<T>& A, cudaStream_t st) {
  const int K = A.in.K;
  if constexpr (sizeof(T) == 8) {
    if (K > 256) return launch_small_t<T, OP, 32, 16>(A, st);
    if (K > 128) return launch_small_t<T, OP, 16, 16>(A, st);
  }
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

}  // namespace
}  // namespace mtb
