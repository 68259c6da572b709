// Log probabilities of given tokens, the entropy and the largest classes of rows of logits, with
// the logits' gradient.
//
//   x = z / tau,  m = max x,  s = sum exp(x - m),  p = exp(x - m) / s
//   log p_y = (x_y - m) - log s
//   H       = log s - (1/s) sum exp(x - m) (x - m)
//   dz      = (1/tau) (sum over outputs i: g_i delta_i - p (sum of the g_i) - g_H p (log p + H))
//
// with the g_i the gradients of log p_y and of the top classes' log probabilities.  Everything is
// formed from differences to the maximum, so that what the logits have in common costs nothing; the
// entropy is a sum of two parts that are not negative.
//
// The largest classes go by the logits themselves, ties by the lower class; -0 and 0 are equal.
// A row whose token is `ignore` gives 0 everywhere and `ignore` for its classes.  A row without a
// softmax (a NaN, an infinity, -inf alone) gives NaN and the classes 0 to K - 1.
#include <type_traits>

#include "rows.h"

namespace dmh {

constexpr int TOP_MAX = 256;

struct LogProbArgs {
  const void* z;
  const void* tokens;    // or null
  float* lp;             // (rows), or null without tokens
  float* ent;            // (rows), or null
  float* top_lp;         // (rows, top)
  long long* top_ids;    // (rows, top)
  float* stats;          // (3, rows): maximum, sum, entropy; or null
  long long rows, zs, ignore;
  int classes, t64, top;
  float itau, c2;        // 1 / tau; log2(e) / tau
};

// Parts of a row in units of 2: e = 2^d, d = (z - m) c2: s = sum e, t = sum e d.
struct Part3 {
  float m, s, t;
};
constexpr float LOWEST = -200.f;   // 2^d is 0 here and below; d itself may be -inf there

__device__ __forceinline__ void rescale(Part3& p, float m, float c2) {
  if (p.m != m) {   // never for two of -inf
    const float d = (p.m - m) * c2, f = __builtin_amdgcn_exp2f(d);
    p.t = f * fmaf(p.s, fmaxf(d, LOWEST), p.t);
    p.s *= f;
    p.m = m;
  }
}
__device__ __forceinline__ Part3 join(Part3 a, Part3 b, float c2) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, c2);
  rescale(b, m, c2);
  return {m, a.s + b.s, a.t + b.t};
}
template <int THREADS>
__device__ __forceinline__ Part3 block_join(Part3 p, float c2, Part3* lds) {
#pragma unroll
  for (int d = (THREADS < 64 ? THREADS : 64) / 2; d; d >>= 1)
    p = join(p, {__shfl_xor(p.m, d), __shfl_xor(p.s, d), __shfl_xor(p.t, d)}, c2);
  constexpr int W = THREADS / 64;
  if (W <= 1) return p;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = p;
  __syncthreads();
  p = (threadIdx.x & 63) < W ? lds[threadIdx.x & 63] : Part3{-INF, 0.f, 0.f};
#pragma unroll
  for (int d = W / 2; d; d >>= 1)
    p = join(p, {__shfl_xor(p.m, d), __shfl_xor(p.s, d), __shfl_xor(p.t, d)}, c2);
  return {__shfl(p.m, 0), __shfl(p.s, 0), __shfl(p.t, 0)};
}

// ---- the largest classes ----------------------------------------------------------------------
typedef unsigned long long u64;

// Floats in their order as whole numbers; -0 counts as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// ... and by class among equals.  Never 0: classes stay below 2^27.
__device__ __forceinline__ u64 rank_key(float x, int c) {
  return (u64)order_key(x) << 32 | (uint32_t)~c;
}

struct TopLds {
  u64 cand[1024];
  int slots[96];   // a counter for each step of a search
  int n;
};
constexpr int CANDS = 1024;

// The number over the whole workgroup, through counter `slot` (zero before).
__device__ __forceinline__ int block_count(int n, int* slot) {
#pragma unroll
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  if ((threadIdx.x & 63) == 0 && n) atomicAdd(slot, n);
  __syncthreads();
  return *slot;
}

// The K largest classes of a row by one workgroup; each(f) calls f(value, class) for every class of
// the thread, `largest` is their maximum (-inf for none).
template <int THREADS, class Each>
__device__ __forceinline__ void select_top(int K, float largest, const Each& each, TopLds& l) {
  for (int i = threadIdx.x; i < 96; i += THREADS) l.slots[i] = 0;
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  // K threads have a class that is at least the K-th largest of the threads' maxima, so K
  // classes are: a bit at a time, until few more threads are left
  const uint32_t mine = order_key(largest);
  uint32_t cut = 0;
  int step = 0;
  const int enough = K + K / 4 + 4;
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = cut | 1u << b;
    const int n = block_count(mine >= c, &l.slots[step++]);
    if (n >= K) {
      cut = c;
      if (n <= enough) break;
    }
  }
  u64 from = (u64)cut << 32;
  auto gather = [&]() {
    each([&](float v, int c) {
      const u64 k = rank_key(v, c);
      if (k >= from) {
        const int at = atomicAdd(&l.n, 1);
        if (at < CANDS) l.cand[at] = k;
      }
    });
    __syncthreads();
  };
  gather();
  if (l.n > CANDS) {
    // few threads with many large classes, or many equal ones: the same over all classes
    step = 32;
    from = 0;
    for (int b = 63; b >= 0; --b) {
      const u64 t = from | 1ull << b;
      int n = 0;
      each([&](float v, int c) { n += rank_key(v, c) >= t; });
      n = block_count(n, &l.slots[step++]);
      if (n >= K) {
        from = t;
        if (n <= CANDS) break;
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) l.n = 0;
    __syncthreads();
    gather();
  }
}

// Rows of any length: a workgroup reads its row for the sums, and again for its largest classes.
template <class T, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void log_prob_row(LogProbArgs a) {
  __shared__ Part3 parts[16];
  __shared__ typename std::conditional<TOP, TopLds, char>::type top;
  constexpr int N = Piece<T>::N, AHEAD = 4;
  typedef typename Row<T>::type type;
  const long long row = blockIdx.x;
  const int t = threadIdx.x, K = a.top;
  const T* z = (const T*)a.z + row * a.zs;
  const Row<T> r(z, a.classes);
  const long long y = a.tokens ? load_index(a.tokens, a.t64, row) : 0;
  if (a.tokens && y == a.ignore) {
    if (t == 0) {
      a.lp[row] = 0.f;
      if (a.ent) a.ent[row] = 0.f;
    }
    if (t < 3 && a.stats) a.stats[t * a.rows + row] = t == 1 ? 1.f : 0.f;
    for (int i = t; i < K; i += THREADS) {
      a.top_lp[row * K + i] = 0.f;
      a.top_ids[row * K + i] = a.ignore;
    }
    return;
  }
  const int ec = r.edge(t);
  const float ex = ec >= 0 ? (float)z[ec] : -INF;
  Part3 p = {fmaxf(ex, -INF), 0.f, 0.f};
  auto add = [&](float v, float m0) {
    const float d = (v - m0) * a.c2, e = __builtin_amdgcn_exp2f(d);
    p.s += e;
    p.t = fmaf(e, fmaxf(d, LOWEST), p.t);
  };
  if (ec >= 0) add(ex, p.m == -INF ? 0.f : p.m);
  for (int i0 = t; i0 < r.pieces; i0 += AHEAD * THREADS) {
    type x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * THREADS;
      x[k] = *(const type*)(z + r.piece_class(i < r.pieces ? i : i0));
    }
    float m = p.m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, (float)x[k][j]);
    rescale(p, m, a.c2);
    const float m0 = m == -INF ? 0.f : m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i0 + k * THREADS < r.pieces) {
#pragma unroll
        for (int j = 0; j < N; ++j) add((float)x[k][j], m0);
      }
  }
  const float largest = p.m;
  p = block_join<THREADS>(p, a.c2, parts);
  const float log_s = __builtin_amdgcn_logf(p.s) * LN2;
  const bool good = p.s >= 0.5f;   // the maximum alone gives 1
  if (t == 0) {
    const float ent = log_s - LN2 * (p.t / p.s);
    if (a.ent) a.ent[row] = ent;
    if (a.stats) a.stats[row] = p.m;
    if (a.stats) a.stats[a.rows + row] = p.s;
    if (a.stats) a.stats[2 * a.rows + row] = ent;
    if (a.tokens)
      a.lp[row] = y >= 0 && y < a.classes ? ((float)z[y] - p.m) * a.itau - log_s
                                          : __builtin_nanf("");
  }
  if constexpr (TOP) {
    if (!good) {
      for (int i = t; i < K; i += THREADS) {
        a.top_lp[row * K + i] = __builtin_nanf("");
        a.top_ids[row * K + i] = i;
      }
      return;
    }
    auto each = [&](auto f) {
      if (ec >= 0) f(ex, ec);
      for (int i = t; i < r.pieces; i += THREADS) {
        const type x = *(const type*)(z + r.piece_class(i));
#pragma unroll
        for (int j = 0; j < N; ++j) f((float)x[j], r.piece_class(i) + j);
      }
    };
    select_top<THREADS>(K, largest, each, top);
    const int n = top.n;
    for (int i = t; i < n; i += THREADS) {
      const u64 k = top.cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += top.cand[j] > k;
      if (before < K) {
        a.top_lp[row * K + before] = (key_value((uint32_t)(k >> 32)) - p.m) * a.itau - log_s;
        a.top_ids[row * K + before] = (uint32_t)~k;
      }
    }
  }
}

template <class T>
static void launch_log_probs(hipStream_t stream, const LogProbArgs& a) {
  const dim3 rows((unsigned)a.rows);
  if (a.classes <= 8192) {
    if (a.top)
      hipLaunchKernelGGL((log_prob_row<T, 256, true>), rows, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((log_prob_row<T, 256, false>), rows, dim3(256), 0, stream, a);
  } else if (a.top) {
    hipLaunchKernelGGL((log_prob_row<T, 1024, true>), rows, dim3(1024), 0, stream, a);
  } else {
    hipLaunchKernelGGL((log_prob_row<T, 1024, false>), rows, dim3(1024), 0, stream, a);
  }
}

// ---- gradient -----------------------------------------------------------------------------------
struct LogProbGradArgs {
  const void* z;
  const void* tokens;            // or null
  const long long* top_ids;      // (rows, top)
  const float* stats;            // (3, rows), of the forward pass
  const float *glp, *gent, *gtop;   // each may be null
  void* dz;
  long long rows, zs, ds, ignore;
  int classes, t64, top;
  float itau, c2;
};

// Element by element, 256 threads for four pieces each of a row; the listed classes (the token and
// the top ones) are written again behind a barrier, each by one thread with the sum of its terms.
template <class T>
__global__ __launch_bounds__(256) void log_prob_grad(LogProbGradArgs a) {
  constexpr int N = Piece<T>::N, AHEAD = 4, THREADS = 256;
  __shared__ float lds[16];
  __shared__ int ids[TOP_MAX + 1];
  __shared__ float terms[TOP_MAX + 1];
  __shared__ uint32_t marks[THREADS];
  __shared__ uint32_t edge_marks;
  __shared__ int twice;
  typedef typename Row<T>::type type;
  const long long row = blockIdx.x;
  const int t = threadIdx.x, K = a.gtop ? a.top : 0;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = (T*)a.dz + row * a.ds;
  const Row<T> r(z, a.classes);
  const int first = blockIdx.y * THREADS * AHEAD, i0 = first + t;
  const int ec = blockIdx.y == 0 ? r.edge(t) : -1;
  const long long y = a.tokens ? load_index(a.tokens, a.t64, row) : 0;
  if (a.tokens && y == a.ignore) {
    const type zero = {};
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i0 + k * THREADS < r.pieces) *(type*)(dz + r.piece_class(i0 + k * THREADS)) = zero;
    if (ec >= 0) dz[ec] = (T)0.f;
    return;
  }
  type x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    if (r.pieces) x[k] = *(const type*)(z + r.piece_class(i < r.pieces ? i : 0));
  }
  const float ex = ec >= 0 ? (float)z[ec] : 0.f;
  const float m = a.stats[row], s = a.stats[a.rows + row], ent = a.stats[2 * a.rows + row];
  const float gy = a.glp ? a.glp[row] : 0.f, gh = a.gent ? a.gent[row] : 0.f;
  // the list: what is outside the classes is not in it
  marks[t] = 0;
  if (t == 0) {
    edge_marks = 0;
    twice = 0;
  }
  float push = 0.f;
  for (int j = t; j <= K; j += THREADS) {
    const bool top = j < K;
    const long long c = top ? a.top_ids[row * K + j] : a.glp ? y : -1;
    const float g = top ? a.gtop[row * K + j] : gy;
    push += g;
    ids[j] = c >= 0 && c < a.classes ? (int)c : -1;
    terms[j] = g * a.itau;
  }
  push = block_sum<THREADS>(push, lds);
  const bool known = !a.tokens || (y >= 0 && y < a.classes);
  const float scale = known ? -a.itau / s : __builtin_nanf("");
  const float log_s = __builtin_amdgcn_logf(s) * LN2;
  const float A = scale * (push + gh * (ent - log_s)), B = scale * gh * LN2;
  auto grad = [&](float v) {
    const float d = (v - m) * a.c2;
    return __builtin_amdgcn_exp2f(d) * fmaf(B, fmaxf(d, LOWEST), A);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    type d;
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = (T)grad((float)x[k][j]);
    if (i < r.pieces) *(type*)(dz + r.piece_class(i)) = d;
  }
  if (ec >= 0) dz[ec] = (T)grad(ex);
  __syncthreads();   // also: the list is written
  uint32_t firsts = 0;
  int it = 0;
  for (int j = t; j <= K; j += THREADS, ++it) {
    uint32_t *word, bit;
    if (ids[j] >= 0 && find_mark(r, ids[j], first, THREADS * AHEAD, blockIdx.y == 0, marks,
                                 &edge_marks, word, bit)) {
      if (atomicOr(word, bit) & bit) twice = 1;
      else firsts |= 1u << it;
    }
  }
  __syncthreads();
  it = 0;
  for (int j = t; j <= K; j += THREADS, ++it) {
    if (firsts >> it & 1) {
      const int c = ids[j];
      float g = terms[j];
      if (twice) {   // a class listed more than once: its terms in their order
        g = 0.f;
        for (int i = 0; i <= K; ++i) g += ids[i] == c ? terms[i] : 0.f;
      }
      dz[c] = (T)(grad((float)z[c]) + g);
    }
  }
}

template <class T>
static void launch_log_prob_grad(hipStream_t stream, const LogProbGradArgs& a) {
  const int whole = a.classes / Piece<T>::N;
  hipLaunchKernelGGL((log_prob_grad<T>),
                     dim3((unsigned)a.rows, (unsigned)(whole ? ceil_div(whole, 1024) : 1)),
                     dim3(256), 0, stream, a);
}

static bool log_prob_shape(long long rows, long long classes, long long top) {
  return rows >= 0 && rows < (1LL << 22) && classes >= 1 && classes <= (1LL << 27) && top >= 0 &&
         top <= TOP_MAX && top <= classes;
}
static bool temperature_ok(float tau) { return tau >= 1e-6f && tau <= 1e6f; }

}  // namespace dmh

using namespace dmh;

extern "C" {

int dmh_log_probs(hipStream_t stream, const void* logits, int dtype, long long rows,
                  long long classes, long long z_rstride, const void* tokens, int tokens_64,
                  long long ignore_index, float temperature, int top, float* log_probs,
                  float* entropy, float* top_log_probs, long long* top_ids, float* stats) {
  if (!log_prob_shape(rows, classes, top) || z_rstride < 0 || !float_code(dtype) ||
      !temperature_ok(temperature)) {
    set_error("dmh_log_probs: bad arguments (rows=%lld classes=%lld dtype=%d top=%d "
              "temperature=%g)", rows, classes, dtype, top, (double)temperature);
    return DMH_EINVAL;
  }
  if (rows == 0) return DMH_OK;
  if (!logits || (tokens && !log_probs) || (top && (!top_log_probs || !top_ids))) {
    set_error("dmh_log_probs: null tensor");
    return DMH_EINVAL;
  }
  LogProbArgs a{};
  a.z = logits;
  a.tokens = tokens;
  a.lp = log_probs;
  a.ent = entropy;
  a.top_lp = top_log_probs;
  a.top_ids = top_ids;
  a.stats = stats;
  a.rows = rows;
  a.zs = z_rstride;
  a.ignore = ignore_index;
  a.classes = (int)classes;
  a.t64 = tokens_64 != 0;
  a.top = top;
  a.itau = (float)(1.0 / temperature);
  a.c2 = (float)(1.4426950408889634 / temperature);
  DMH_FOR_TYPE(dtype, T, (launch_log_probs<T>(stream, a)))
  DMH_CHECK_LAUNCH("log_prob_row");
  return DMH_OK;
}

int dmh_log_probs_grad(hipStream_t stream, const void* logits, int dtype, long long rows,
                       long long classes, long long z_rstride, const void* tokens, int tokens_64,
                       long long ignore_index, float temperature, int top,
                       const long long* top_ids, const float* stats, const float* grad_log_probs,
                       const float* grad_entropy, const float* grad_top, void* dlogits,
                       long long d_rstride) {
  if (!log_prob_shape(rows, classes, top) || z_rstride < 0 || d_rstride < 0 ||
      !float_code(dtype) || !temperature_ok(temperature)) {
    set_error("dmh_log_probs_grad: bad arguments (rows=%lld classes=%lld dtype=%d top=%d "
              "temperature=%g)", rows, classes, dtype, top, (double)temperature);
    return DMH_EINVAL;
  }
  if (rows == 0) return DMH_OK;
  if (!logits || !stats || !dlogits || (grad_log_probs && !tokens) || (grad_top && !top_ids)) {
    set_error("dmh_log_probs_grad: null tensor");
    return DMH_EINVAL;
  }
  LogProbGradArgs a{};
  a.z = logits;
  a.tokens = tokens;
  a.top_ids = top_ids;
  a.stats = stats;
  a.glp = grad_log_probs;
  a.gent = grad_entropy;
  a.gtop = grad_top;
  a.dz = dlogits;
  a.rows = rows;
  a.zs = z_rstride;
  a.ds = d_rstride;
  a.ignore = ignore_index;
  a.classes = (int)classes;
  a.t64 = tokens_64 != 0;
  a.top = top;
  a.itau = (float)(1.0 / temperature);
  a.c2 = (float)(1.4426950408889634 / temperature);
  DMH_FOR_TYPE(dtype, T, (launch_log_prob_grad<T>(stream, a)))
  DMH_CHECK_LAUNCH("log_prob_grad");
  return DMH_OK;
}

}  // extern "C"
