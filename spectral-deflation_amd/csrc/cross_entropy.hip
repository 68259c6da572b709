// Cross entropy over the classes of a vocabulary, with its gradient.
//
//   lse  = log sum exp z
//   loss = lse - (1 - eps) z_y - eps mean(z) + zeta lse^2
//   dz   = (p (1 + 2 zeta lse) - (1 - eps) delta_y - eps / V) * g,     p = exp(z - lse)
//
// with m = max z and s = sum exp(z - m) computed as
//
//   loss = log s + (m - z_y) - eps mean(z - z_y) + zeta (m + log s)^2,     p = exp(z - m) / s
//
// so that what all logits of a row have in common cancels before anything is rounded: lse itself
// in 32 bits is off by half a last place of the logits' size, more than the whole loss of a row
// that is sure of its target.
//
// eps is the label smoothing, zeta the weight of the z-loss; g is grad_scale, divided by the
// number of rows that have a target for a mean.  A row whose target is ignore_index has loss 0
// and gradient 0 whatever its logits hold; any other target outside [0, V) makes both NaN.  A
// row of -inf alone has no softmax: its loss and gradient are NaN.
#include "train_ops.h"

namespace dmh {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

enum { RED_NONE = 0, RED_MEAN = 1, RED_SUM = 2 };

struct XentArgs {
  const void* z;
  const void* targets;
  void* dz;              // or null
  float* row_loss;
  float* row_max;        // per row, written (forward) or read (gradient): its maximum, and
  float* row_sum;        // sum exp(z - maximum); lse and 1 if row_sum is null.  Both may be null
                         // in the forward pass
  const float* count;    // rows that have a target, or null
  int counts;            // the rows' launch counts them itself
  const float* gout;     // gradient of the loss (gradient kernel): one, or one a row
  long long rows, zs, ds, ignore;
  int classes, t64, gout_rows;
  float eps, zeta, gscale;
};

constexpr float INF = __builtin_inff();

// exp(x - m) by the hardware's 2^x (results below 2^-126 are zero)
__device__ __forceinline__ float exp_diff(float x, float m) {
  return __builtin_amdgcn_exp2f((x - m) * LOG2E);
}

// The sum of one value a thread over THREADS threads: part of a wave, a wave, or a workgroup of as
// many.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int d = (THREADS < 64 ? THREADS : 64) / 2; d; d >>= 1) v += __shfl_xor(v, d);
  constexpr int W = THREADS / 64;
  if (W <= 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) s += lds[w];
  return s;
}

// Parts of a row: m their maximum, s = sum exp(z - m); (-inf, 0) for none, and for values of
// -inf alone.  A NaN ends in s.
struct Part {
  float m, s;
};
__device__ __forceinline__ Part join(Part a, Part b) {
  const float m = fmaxf(a.m, b.m);
  // nothing to scale where the maximum stays; both -inf must not give inf - inf
  const float fa = a.m == m ? 1.f : exp_diff(a.m, m), fb = b.m == m ? 1.f : exp_diff(b.m, m);
  return {m, a.s * fa + b.s * fb};
}
template <int THREADS>
__device__ __forceinline__ Part block_join(Part p, Part* lds) {
#pragma unroll
  for (int d = (THREADS < 64 ? THREADS : 64) / 2; d; d >>= 1)
    p = join(p, {__shfl_xor(p.m, d), __shfl_xor(p.s, d)});
  constexpr int W = THREADS / 64;
  if (W <= 1) return p;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = p;
  __syncthreads();
  // every wave joins the waves' parts in the same way
  p = (threadIdx.x & 63) < W ? lds[threadIdx.x & 63] : Part{-INF, 0.f};
#pragma unroll
  for (int d = W / 2; d; d >>= 1) p = join(p, {__shfl_xor(p.m, d), __shfl_xor(p.s, d)});
  return {__shfl(p.m, 0), __shfl(p.s, 0)};
}

// The number of rows that have a target, in every thread of the workgroup.  One workgroup goes
// through all rows, so it has AHEAD loads a thread on their way.
template <int THREADS, int AHEAD>
__device__ __forceinline__ float count_targets(const XentArgs& a, float* lds) {
  int n = 0;
  const int rows = (int)a.rows;
  auto count = [&](auto* targets) {
    int i = threadIdx.x;
    for (; i + (AHEAD - 1) * THREADS < rows; i += AHEAD * THREADS) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) n += targets[i + k * THREADS] != a.ignore;
    }
    for (; i < rows; i += THREADS) n += targets[i] != a.ignore;
  };
  if (a.t64) count((const long long*)a.targets); else count((const int*)a.targets);
  return block_sum<THREADS>((float)n, lds);   // exact: below 2^24 rows
}

// (One workgroup: 8192 rows are counted in 4.6 us and summed in 5.1, most of it latency.  It is made
// for the rows of a vocabulary: of 256 16-bit classes, 2^18 rows take 31 us themselves, 22 to
// sum and 29 to count, 2^20 rows 133, 80 and 155.)
__global__ __launch_bounds__(1024) void xent_count(XentArgs a, float* count) {
  __shared__ float lds[16];
  const float n = count_targets<1024, 8>(a, lds);
  if (threadIdx.x == 0) *count = n;
}

// The sum of the rows' losses, divided by the number of rows with a target for a mean, which it
// counts if no launch before has (COUNT).
template <bool COUNT>
__global__ __launch_bounds__(1024) void xent_reduce(XentArgs a, float* count, float* loss) {
  __shared__ float lds[16];
  constexpr int AHEAD = 16;
  const int rows = (int)a.rows;
  float s = 0.f;
  int i = threadIdx.x;
  for (; i + (AHEAD - 1) * 1024 < rows; i += AHEAD * 1024) {
    float v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) v[k] = a.row_loss[i + k * 1024];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) s += v[k];
  }
  for (; i < rows; i += 1024) s += a.row_loss[i];
  s = block_sum<1024>(s, lds);
  const float n = COUNT ? count_targets<1024, 8>(a, lds) : count ? *count : 1.f;
  if (threadIdx.x == 0) {
    if (COUNT) *count = n;
    *loss = s / n;
  }
}

// What a row's statistics say: its loss, and the factors of its gradient
// d = exp(z - m) ps + base (+ top at the target).
struct Grad {
  float ps, base, top;
};
// Differences to the target's logit are summed up 2^-28 times their size, which costs nothing in a
// fused multiply-add: classes at the lowest and the highest values of the type do not overflow.
constexpr float SMALL = 0x1p-28f, BIG = 0x1p28f;
__device__ __forceinline__ float small_diff(float z, float zy) {
  return fmaf(z, SMALL, zy * -SMALL);
}
// zsum: the sum of small_diff(z, zy); from 0 in place of a zy that is not finite, whose loss
// is not either
__device__ __forceinline__ float row_loss(const XentArgs& a, float m, float log_s, float zy,
                                          float zsum) {
  float loss = log_s + (m - zy);
  if (a.eps != 0.f) loss -= zsum * (a.eps / a.classes) * BIG;
  const float lse = m + log_s;
  if (a.zeta != 0.f) loss += a.zeta * lse * lse;
  return loss;
}
// (Each store under a condition of its own: from an if and an else with three stores ROCm 7.2's
// compiler made one whose address was the wrong array's.)
__device__ __forceinline__ void put_stats(const XentArgs& a, long long row, float m, float s,
                                          float log_s) {
  if (a.row_max) a.row_max[row] = a.row_sum ? m : m + log_s;
  if (a.row_sum) a.row_sum[row] = s;
}
__device__ __forceinline__ Grad row_grad(const XentArgs& a, float g, float m, float s,
                                         float log_s) {
  return {g * (1.f + 2.f * a.zeta * (m + log_s)) / s, -g * (a.eps / a.classes),
          -g * (1.f - a.eps)};
}

// A row in aligned pieces of 16 bytes, and the classes before the first and behind the last one,
// up to seven on each side, which the first sixteen threads of a row take one by one.  Rows of an
// odd number of classes start anywhere; with pieces from the row's start instead the loads
// and stores of bf16 rows of 50257 took 13% longer.
template <class T>
struct Row {
  static constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::type type;
  int head, pieces, classes;
  __device__ __forceinline__ Row(const T* z, int v) : classes(v) {
    head = (int)(-((uintptr_t)z / sizeof(T)) & (N - 1));
    head = head < v ? head : v;
    pieces = (v - head) / N;
  }
  __device__ __forceinline__ int piece_class(int i) const { return head + i * N; }
  // the single class of thread t, or -1
  __device__ __forceinline__ int edge(int t) const {
    const int c = t < 8 ? (t < head ? t : -1) : piece_class(pieces) + t - 8;
    return c < classes && t < 16 ? c : -1;
  }
  // the thread that writes class c
  template <int THREADS>
  __device__ __forceinline__ int owner(int c) const {
    const int i = (c - head) / N;
    return c < head ? c : i < pieces ? i % THREADS : 8 + c - piece_class(pieces);
  }
};

// Bound by the memory, and close to it by arithmetic: 8192 bf16 rows of 50257 with gradient take
// 296 us (1647 MB, 5.6 TB/s), the vector units busy 85% of the time; the loss alone 141 us for half
// the bytes.  A sweep of its own each for the maximum, the sum and the gradient took 1270 us.
//
// One row by THREADS threads that hold all of it in registers, HELD pieces each: it is read
// once, and with GRAD its gradient written once.  Every thread first takes the maximum and the
// sum of its own classes, and one exchange joins them.  Between the steps the row stays packed
// (`repack`: what a step has unpacked may not stay in registers for the next), so that two
// workgroups of 1024 fit a compute unit up to 65536 16-bit classes and one's loads run under
// the other's arithmetic: with the unpacked values kept, 8192 bf16 rows of 50257 took 381
// instead of 332 us.
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <int HELD>
__device__ __forceinline__ void repack(i32x4 (&x)[HELD]) {
#pragma unroll
  for (int k = 0; k < HELD; ++k) asm volatile("" : "+v"(x[k]));
}

template <class T, int THREADS, int HELD, bool GRAD, bool COUNT>
__global__ __launch_bounds__(THREADS < 128 ? 256 : THREADS, HELD > 16      ? 2
                                                            : HELD > 8      ? 4
                                                            : THREADS < 128 ? 7
                                                                            : 8)
void xent_row(XentArgs a) {
  __shared__ Part parts[16];
  __shared__ float lds[16];
  constexpr int N = Piece<T>::N, GROUP = THREADS < 128 ? 256 : THREADS;
  float count = 1.f;
  if (COUNT)
    count = count_targets<GROUP, 2>(a, lds);
  else if (a.count)
    count = *a.count;
  const long long row = THREADS == GROUP
                            ? (long long)blockIdx.x
                            : (long long)blockIdx.x * (GROUP / THREADS) + (threadIdx.x / THREADS);
  if (row >= a.rows) return;
  const int t = THREADS == GROUP ? threadIdx.x : threadIdx.x % THREADS;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = GRAD ? (T*)a.dz + row * a.ds : nullptr;
  const Row<T> r(z, a.classes);
  const long long y = load_index(a.targets, a.t64, row);
  typedef typename Row<T>::type type;
  i32x4 x[HELD] = {};
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = k * THREADS + t;
    if (i < r.pieces) x[k] = __builtin_bit_cast(i32x4, *(const type*)(z + r.piece_class(i)));
  }
  const int ec = r.edge(t);
  const float ex = ec >= 0 ? (float)z[ec] : -INF;
  if (y == a.ignore) {
    if (t == 0) {
      a.row_loss[row] = 0.f;
      put_stats(a, row, 0.f, 1.f, 0.f);
    }
    if (GRAD) {
      const type zero = {};
      for (int i = t; i < r.pieces; i += THREADS)
        *(type*)(dz + r.piece_class(i)) = zero;
      if (ec >= 0) dz[ec] = (T)0.f;
    }
    return;
  }
  const bool known = y >= 0 && y < a.classes;
  const float zy = known ? (float)z[y] : __builtin_nanf("");
  const float ref = fabsf(zy) < INF ? zy : 0.f;
  float zsum = ec >= 0 ? small_diff(ex, ref) : 0.f;
  if (a.eps != 0.f) {
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      if (k * THREADS + t < r.pieces) {
        const type v = __builtin_bit_cast(type, x[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) zsum += small_diff((float)v[j], ref);
      }
    }
  }
  repack(x);
  Part p = {fmaxf(ex, -INF), 0.f};   // not a NaN
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    if (k * THREADS + t < r.pieces) {
      const type v = __builtin_bit_cast(type, x[k]);
#pragma unroll
      for (int j = 0; j < N; ++j) p.m = fmaxf(p.m, (float)v[j]);
    }
  }
  repack(x);
  const float m0 = p.m == -INF ? 0.f : p.m;
  p.s = exp_diff(ex, m0);
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    if (k * THREADS + t < r.pieces) {
      const type v = __builtin_bit_cast(type, x[k]);
#pragma unroll
      for (int j = 0; j < N; ++j) p.s += exp_diff((float)v[j], m0);
    }
  }
  repack(x);
  p = block_join<THREADS>(p, parts);
  if (a.eps != 0.f) zsum = block_sum<THREADS>(zsum, lds);
  const float log_s = __builtin_amdgcn_logf(p.s) * LN2;
  if (t == 0) {
    a.row_loss[row] = row_loss(a, p.m, log_s, zy, zsum);
    put_stats(a, row, p.m, p.s, log_s);
  }
  if (!GRAD) return;
  const Grad g = row_grad(a, known ? a.gscale / count : __builtin_nanf(""), p.m, p.s, log_s);
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = k * THREADS + t;
    if (i < r.pieces) {
      const type v = __builtin_bit_cast(type, x[k]);
      type d;
#pragma unroll
      for (int j = 0; j < N; ++j) d[j] = (T)fmaf(exp_diff((float)v[j], p.m), g.ps, g.base);
      *(type*)(dz + r.piece_class(i)) = d;
    }
  }
  if (ec >= 0) dz[ec] = (T)fmaf(exp_diff(ex, p.m), g.ps, g.base);
  // the target's element again, by the thread that has just written it
  if (known && t == r.template owner<THREADS>((int)y))
    dz[y] = (T)(fmaf(exp_diff(zy, p.m), g.ps, g.base) + g.top);
}

// Rows that no workgroup's registers hold, and long rows without gradient, which need not be held:
// a workgroup reads its row for the statistics and again for the gradient.  5.5 TB/s of what it
// reads and writes for 131072 fp32 classes.
template <class T, bool GRAD>
__global__ __launch_bounds__(1024) void xent_stream(XentArgs a) {
  __shared__ Part parts[16];
  __shared__ float lds[16];
  constexpr int N = Piece<T>::N, AHEAD = 4;
  typedef typename Row<T>::type type;
  const long long row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = GRAD ? (T*)a.dz + row * a.ds : nullptr;
  const Row<T> r(z, a.classes);
  const long long y = load_index(a.targets, a.t64, row);
  const int ec = r.edge(threadIdx.x);
  const type zero = {};
  if (y == a.ignore) {
    if (threadIdx.x == 0) {
      a.row_loss[row] = 0.f;
      put_stats(a, row, 0.f, 1.f, 0.f);
    }
    if (GRAD) {
      for (int i = threadIdx.x; i < r.pieces; i += 1024) *(type*)(dz + r.piece_class(i)) = zero;
      if (ec >= 0) dz[ec] = (T)0.f;
    }
    return;
  }
  const bool known = y >= 0 && y < a.classes;
  const float zy = known ? (float)z[y] : __builtin_nanf("");
  const float ex = ec >= 0 ? (float)z[ec] : -INF;
  const float ref = fabsf(zy) < INF ? zy : 0.f;
  float zsum = ec >= 0 ? small_diff(ex, ref) : 0.f;
  Part p = {fmaxf(ex, -INF), 0.f};
  p.s = exp_diff(ex, p.m == -INF ? 0.f : p.m);
  for (int i0 = threadIdx.x; i0 < r.pieces; i0 += AHEAD * 1024) {
    type x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * 1024;
      x[k] = *(const type*)(z + r.piece_class(i < r.pieces ? i : i0));
    }
    float m = p.m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, (float)x[k][j]);
    const float m0 = m == -INF ? 0.f : m;
    p.s *= p.m == m ? 1.f : exp_diff(p.m, m);
    p.m = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const bool in = i0 + k * 1024 < r.pieces;
      float e = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        e += exp_diff((float)x[k][j], m0);
        if (a.eps != 0.f) zsum += in ? small_diff((float)x[k][j], ref) : 0.f;
      }
      p.s += in ? e : 0.f;
    }
  }
  p = block_join<1024>(p, parts);
  zsum = block_sum<1024>(zsum, lds);   // also: every read of z[y] is before dz, which may be z
  const float log_s = __builtin_amdgcn_logf(p.s) * LN2;
  if (threadIdx.x == 0) {
    a.row_loss[row] = row_loss(a, p.m, log_s, zy, zsum);
    put_stats(a, row, p.m, p.s, log_s);
  }
  if (!GRAD) return;
  const float count = a.count ? *a.count : 1.f;
  const Grad g = row_grad(a, known ? a.gscale / count : __builtin_nanf(""), p.m, p.s, log_s);
  for (int i0 = threadIdx.x; i0 < r.pieces; i0 += AHEAD * 1024) {
    type x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * 1024;
      x[k] = *(const type*)(z + r.piece_class(i < r.pieces ? i : i0));
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * 1024;
      type d;
#pragma unroll
      for (int j = 0; j < N; ++j) d[j] = (T)fmaf(exp_diff((float)x[k][j], p.m), g.ps, g.base);
      if (i < r.pieces) *(type*)(dz + r.piece_class(i)) = d;
    }
  }
  if (ec >= 0) dz[ec] = (T)fmaf(exp_diff(ex, p.m), g.ps, g.base);
  if (known && (int)threadIdx.x == r.template owner<1024>((int)y))
    dz[y] = (T)(fmaf(exp_diff(zy, p.m), g.ps, g.base) + g.top);
}

// The gradient from a forward pass's statistics, element by element: THREADS threads a row, AHEAD
// pieces each.  Bound by the memory: 78 us for 2000 fp32 rows of 32003 (512 MB, 6.6 TB/s; the
// logits are partly in the last-level cache still).
template <class T, int THREADS>
__global__ __launch_bounds__(256) void xent_grad(XentArgs a) {
  constexpr int N = Piece<T>::N, AHEAD = 4;
  typedef typename Row<T>::type type;
  const long long row = (long long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (row >= a.rows) return;
  const int t = threadIdx.x % THREADS;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = (T*)a.dz + row * a.ds;
  const Row<T> r(z, a.classes);
  const int i0 = blockIdx.y * THREADS * AHEAD + t;
  const int ec = blockIdx.y == 0 ? r.edge(t) : -1;
  type x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    if (r.pieces) x[k] = *(const type*)(z + r.piece_class(i < r.pieces ? i : 0));
  }
  const float ex = ec >= 0 ? (float)z[ec] : 0.f;
  const long long y = load_index(a.targets, a.t64, row);
  const bool live = y != a.ignore, known = y >= 0 && y < a.classes;
  const float m = a.row_max[row], s = a.row_sum ? a.row_sum[row] : 1.f;
  float go = a.gout[a.gout_rows ? row : 0];
  if (a.count) go /= *a.count;
  const Grad g = row_grad(a, known ? go : __builtin_nanf(""), m, s,
                          __builtin_amdgcn_logf(s) * LN2);
  auto grad = [&](float v, int c) {
    float d = fmaf(exp_diff(v, m), g.ps, g.base);
    if (c == (int)y) d += g.top;
    return (T)(live ? d : 0.f);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    type d;
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = grad((float)x[k][j], r.piece_class(i) + j);
    if (i < r.pieces) *(type*)(dz + r.piece_class(i)) = d;
  }
  if (ec >= 0) dz[ec] = grad(ex, ec);
}

// The fewest threads that hold a row, eight pieces each, so that several rows share a compute unit
// whatever their length; TB/s of bf16 rows' losses against the next larger variant: 256 classes 4.1
// / 1.3 (a wave a row), 5000 4.9 / 3.9 (256 threads), 17000 4.9 / 3.3 (1024).  Longer rows are
// held for the gradient as far as registers go (70000 fp32 classes 4.5 TB/s, streamed 3.7), and
// streamed for the loss alone (70000 bf16 classes 4.6, held 3.8).
template <class T, bool GRAD, bool COUNT>
static void launch_rows(hipStream_t stream, const XentArgs& a) {
  const int pieces = a.classes / Piece<T>::N, rows = (int)a.rows;   // at most
#define DMH_ROWS(THREADS, HELD)                                                           \
  if (pieces <= THREADS * HELD) {                                                         \
    constexpr int PER = THREADS < 128 ? 256 / THREADS : 1;                                \
    hipLaunchKernelGGL((xent_row<T, THREADS, HELD, GRAD, COUNT>), dim3(ceil_div(rows, PER)), \
                       dim3(PER * THREADS), 0, stream, a);                                \
    return;                                                                               \
  }
  DMH_ROWS(16, 8)
  DMH_ROWS(64, 8)
  DMH_ROWS(128, 8)
  DMH_ROWS(256, 8)
  DMH_ROWS(512, 8)
  DMH_ROWS(1024, 8)
  if constexpr (GRAD) {
    DMH_ROWS(1024, 16)
    DMH_ROWS(512, 48)
  }
#undef DMH_ROWS
  hipLaunchKernelGGL((xent_stream<T, GRAD>), dim3(rows), dim3(1024), 0, stream, a);
}
template <class T>
static void launch_xent(hipStream_t stream, const XentArgs& a) {
  if (a.dz && a.counts)
    launch_rows<T, true, true>(stream, a);
  else if (a.dz)
    launch_rows<T, true, false>(stream, a);
  else
    launch_rows<T, false, false>(stream, a);
}
template <class T>
static void launch_xent_grad(hipStream_t stream, const XentArgs& a) {
  const int whole = a.classes / Piece<T>::N, rows = (int)a.rows;
  if (whole <= 64 * 4)
    hipLaunchKernelGGL((xent_grad<T, 64>), dim3(ceil_div(rows, 4)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((xent_grad<T, 256>), dim3(rows, ceil_div(whole, 256 * 4)), dim3(256), 0,
                       stream, a);
}

// Rows up to here are counted by every workgroup itself, two loads a thread, which saves a launch
// of 4.6 us.
constexpr long long COUNT_ROWS = 2048;

// what launch_rows asks of xent_row
static bool row_in_registers(int dtype, long long classes) {
  return classes / (dtype == DMH_F32 ? 4 : 8) <= 512 * 48;
}

static bool xent_shape(long long rows, long long classes) {
  return rows >= 0 && rows < (1LL << 22) && classes >= 1 && classes <= (1LL << 27);
}

}  // namespace dmh

using namespace dmh;

extern "C" {

int dmh_cross_entropy_workspace_size(long long rows, long long classes, size_t* bytes) {
  if (!bytes || !xent_shape(rows, classes)) {
    set_error("dmh_cross_entropy_workspace_size: bad arguments (rows=%lld classes=%lld)", rows,
              classes);
    return DMH_EINVAL;
  }
  *bytes = 4 * (size_t)rows;
  return DMH_OK;
}

}  // extern "C"

static int xent_forward(hipStream_t stream, const void* logits, int dtype, long long rows,
                        long long classes, long long z_rstride, const void* targets,
                        int targets_64, long long ignore_index, float smoothing, float z_loss,
                        int reduction, float grad_scale, float* loss, float* count, float* row_max,
                        float* row_sum, void* dlogits, long long d_rstride, void* ws,
                        size_t ws_bytes) {
  if (!xent_shape(rows, classes) || z_rstride < 0 || d_rstride < 0 || !float_code(dtype) ||
      reduction < RED_NONE || reduction > RED_SUM) {
    set_error("dmh_cross_entropy: bad arguments (rows=%lld classes=%lld dtype=%d reduction=%d)",
              rows, classes, dtype, reduction);
    return DMH_EINVAL;
  }
  if (!loss || (reduction == RED_MEAN && !count) || (rows > 0 && (!logits || !targets))) {
    set_error("dmh_cross_entropy: null tensor");
    return DMH_EINVAL;
  }
  size_t need;
  dmh_cross_entropy_workspace_size(rows, classes, &need);
  if (reduction != RED_NONE && need > 0 && (!ws || ws_bytes < need)) {
    set_error("dmh_cross_entropy: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return DMH_EWORKSPACE;
  }
  XentArgs a{};
  a.z = logits;
  a.targets = targets;
  a.dz = dlogits;
  a.row_loss = reduction == RED_NONE ? loss : (float*)ws;
  a.row_max = row_max;
  a.row_sum = row_sum;
  a.count = reduction == RED_MEAN ? count : nullptr;
  a.rows = rows;
  a.zs = z_rstride;
  a.ds = d_rstride;
  a.ignore = ignore_index;
  a.classes = (int)classes;
  a.t64 = targets_64 != 0;
  a.eps = smoothing;
  a.zeta = z_loss;
  a.gscale = grad_scale;
  // a mean's gradient needs the count at the start, its loss in the end
  const bool mean = reduction == RED_MEAN;
  a.counts = mean && dlogits && rows <= COUNT_ROWS && row_in_registers(dtype, classes);
  const bool before = mean && dlogits && rows > 0 && !a.counts;
  if (before) {
    hipLaunchKernelGGL(xent_count, dim3(1), dim3(1024), 0, stream, a, count);
    DMH_CHECK_LAUNCH("xent_count");
  }
  if (rows > 0) {
    DMH_FOR_TYPE(dtype, T, (launch_xent<T>(stream, a)))
    DMH_CHECK_LAUNCH("xent_row");
  }
  if (reduction != RED_NONE) {
    if (mean && !before)
      hipLaunchKernelGGL(xent_reduce<true>, dim3(1), dim3(1024), 0, stream, a, count, loss);
    else
      hipLaunchKernelGGL(xent_reduce<false>, dim3(1), dim3(1024), 0, stream, a,
                         mean ? count : nullptr, loss);
    DMH_CHECK_LAUNCH("xent_reduce");
  }
  return DMH_OK;
}

static int xent_backward(hipStream_t stream, const void* logits, int dtype, long long rows,
                         long long classes, long long z_rstride, const void* targets,
                         int targets_64, long long ignore_index, float smoothing, float z_loss,
                         const float* row_max, const float* row_sum, const float* count,
                         const float* grad_out, int grad_out_rows, void* dlogits,
                         long long d_rstride) {
  if (!xent_shape(rows, classes) || z_rstride < 0 || d_rstride < 0 || !float_code(dtype)) {
    set_error("dmh_cross_entropy_grad: bad arguments (rows=%lld classes=%lld dtype=%d)", rows,
              classes, dtype);
    return DMH_EINVAL;
  }
  if (rows == 0) return DMH_OK;
  if (!logits || !targets || !row_max || !grad_out || !dlogits) {
    set_error("dmh_cross_entropy_grad: null tensor");
    return DMH_EINVAL;
  }
  XentArgs a{};
  a.z = logits;
  a.targets = targets;
  a.dz = dlogits;
  a.row_max = (float*)row_max;
  a.row_sum = (float*)row_sum;
  a.count = count;
  a.gout = grad_out;
  a.gout_rows = grad_out_rows != 0;
  a.rows = rows;
  a.zs = z_rstride;
  a.ds = d_rstride;
  a.ignore = ignore_index;
  a.classes = (int)classes;
  a.t64 = targets_64 != 0;
  a.eps = smoothing;
  a.zeta = z_loss;
  DMH_FOR_TYPE(dtype, T, (launch_xent_grad<T>(stream, a)))
  DMH_CHECK_LAUNCH("xent_grad");
  return DMH_OK;
}

extern "C" {

int dmh_cross_entropy(hipStream_t stream, const void* logits, int dtype, long long rows,
                      long long classes, long long z_rstride, const void* targets,
                      int targets_64, long long ignore_index, float smoothing, float z_loss,
                      int reduction, float grad_scale, float* loss, float* count, float* lse,
                      void* dlogits, long long d_rstride, void* ws, size_t ws_bytes) {
  return xent_forward(stream, logits, dtype, rows, classes, z_rstride, targets, targets_64,
                      ignore_index, smoothing, z_loss, reduction, grad_scale, loss, count, lse,
                      nullptr, dlogits, d_rstride, ws, ws_bytes);
}

int dmh_cross_entropy_stats(hipStream_t stream, const void* logits, int dtype, long long rows,
                            long long classes, long long z_rstride, const void* targets,
                            int targets_64, long long ignore_index, float smoothing,
                            float z_loss, int reduction, float grad_scale, float* loss,
                            float* count, float* row_max, float* row_sum, void* dlogits,
                            long long d_rstride, void* ws, size_t ws_bytes) {
  if (rows > 0 && (!row_max || !row_sum)) {
    set_error("dmh_cross_entropy_stats: null statistics");
    return DMH_EINVAL;
  }
  return xent_forward(stream, logits, dtype, rows, classes, z_rstride, targets, targets_64,
                      ignore_index, smoothing, z_loss, reduction, grad_scale, loss, count, row_max,
                      row_sum, dlogits, d_rstride, ws, ws_bytes);
}

int dmh_cross_entropy_grad(hipStream_t stream, const void* logits, int dtype, long long rows,
                           long long classes, long long z_rstride, const void* targets,
                           int targets_64, long long ignore_index, float smoothing, float z_loss,
                           const float* lse, const float* count, const float* grad_out,
                           int grad_out_rows, void* dlogits, long long d_rstride) {
  return xent_backward(stream, logits, dtype, rows, classes, z_rstride, targets, targets_64,
                       ignore_index, smoothing, z_loss, lse, nullptr, count, grad_out,
                       grad_out_rows, dlogits, d_rstride);
}

int dmh_cross_entropy_grad_stats(hipStream_t stream, const void* logits, int dtype,
                                 long long rows, long long classes, long long z_rstride,
                                 const void* targets, int targets_64, long long ignore_index,
                                 float smoothing, float z_loss, const float* row_max,
                                 const float* row_sum, const float* count,
                                 const float* grad_out, int grad_out_rows, void* dlogits,
                                 long long d_rstride) {
  if (rows > 0 && !row_sum) {
    set_error("dmh_cross_entropy_grad_stats: null statistics");
    return DMH_EINVAL;
  }
  return xent_backward(stream, logits, dtype, rows, classes, z_rstride, targets, targets_64,
                       ignore_index, smoothing, z_loss, row_max, row_sum, count, grad_out,
                       grad_out_rows, dlogits, d_rstride);
}

}  // extern "C"
