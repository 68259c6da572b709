// Distillation: the divergence of rows of logits from a teacher's lists of classes, with its
// gradient.
//
//   x = z / tau,  p = softmax(x),  lists of classes i_j with log probabilities t_j
//   q = softmax(t)                     loss = tau^2 sum_j q_j (log q_j - log p_{i_j})
//                                      dz   = tau (p - sum over j with i_j = v of q_j)
//
// or with the classes outside the list (the rest, R) as one more,
//
//   q = exp(t), r = max(0, 1 - sum q)  loss = tau^2 (sum_j q_j (log q_j - log p_{i_j})
//                                                    + r (log r - log p_R)),  p_R = sum_R p
//                                      dz   = tau (w p - q),  w = sum q + r, on the list
//                                             tau (w p - r p / p_R)          off it
//
// The rest has a maximum and a sum of its own, m_R and s_R: p / p_R = exp(x - m_R) / s_R and
// log p_R = m_R + log s_R - lse, where 1 - sum p would have lost all digits for a student that is
// sure of the list.  Off the list, dz is one exponential times one factor of the row.
//
// Where no class is off the list, or only ones of -inf, there is no rest and r is 0.  So it is within
// the rounding of sum q: what that leaves of a teacher's 1 would otherwise be infinitely far from a
// student whose rest is masked, and count a million times over where the mask is -1e9.
//
// An entry whose class is `ignore` is left out, also where that is one of the V classes (then `none`,
// by which token_log_probs marks its lists, is left out too); a row whose first entry is has no
// teacher, loss 0 and gradient 0.  Another class outside [0, V) makes its row NaN, as does a row
// without a softmax.  What has q_j = 0 (or r = 0) adds nothing, whatever p is.  A class that is
// listed twice has two terms.
#include "rows.h"

namespace dmh {

enum { RED_NONE = 0, RED_MEAN = 1, RED_SUM = 2 };

constexpr int LIST_MAX = 1024;

struct DistillArgs {
  const void* z;
  const void* ids;       // (rows, k)
  const void* teacher;   // (rows, k)
  void* dz;              // or null
  float* row_loss;
  float* row_has;        // 1 for a row with a teacher, 0 without; or null
  float* stats;          // (6, rows), written (forward; may be null) or read (gradient)
  const float* counts;   // COUNTS parts of the number of rows that have a teacher, or null
  int self_count;        // the rows' launch counts them itself
  const float* count;    // ... their sum (gradient kernel), or null
  const float* gout;     // gradient of the loss (gradient kernel): one, or one a row
  long long rows, zs, ds, ignore, none;   // none: stands for no class
  int classes, k, i64 /* 0 or 1 */, ttype, gout_rows;
  int skip;              // `ignore` where it is a class, else -1: one register in a comparison
  float itau, c2;        // 1 / tau; log2(e) / tau
  float lscale, gscale;  // tau^2; tau times the gradient's scale
  float slack;           // a rest up to here is the list's rounding
};

// An entry of a list as it is in memory, of any of the types: loaded without a branch, which would
// wait for the value before the row behind it is on its way.
struct RawEntry {
  int lo, hi;             // of the class
  unsigned short a, b;    // the upper and the lower half of an fp32 value; a 16-bit one, twice
  __device__ __forceinline__ void load(const DistillArgs& d, long long i) {
    const int* id = (const int*)d.ids + (i << d.i64);
    lo = id[0];
    hi = id[d.i64];
    const int wide = d.ttype == DMH_F32;
    const unsigned short* t = (const unsigned short*)d.teacher + (i << wide);
    a = t[wide];
    b = t[0];
  }
  __device__ __forceinline__ long long id(const DistillArgs& d) const {
    return (long long)((unsigned long long)(uint32_t)(d.i64 ? hi : lo >> 31) << 32 | (uint32_t)lo);
  }
  __device__ __forceinline__ float value(const DistillArgs& d) const {
    const float f = __builtin_bit_cast(
        float, (uint32_t)a << 16 | (d.ttype == DMH_F32 ? (uint32_t)b : 0u));
    return d.ttype == DMH_F16 ? (float)__builtin_bit_cast(fp16, a) : f;
  }
};

__device__ __forceinline__ bool left_out(const DistillArgs& a, long long id) {
  return id == a.none || id == a.ignore;
}

// A mean's gradient needs the number of rows that have a teacher at the start.  Up to SELF_ROWS
// every workgroup of the rows' launch counts them itself; else a launch does, by the rows' first
// entries, which lie k apart: in COUNTS parts, of one workgroup each (8192 rows, k = 64: 16 us by
// one workgroup alone, 3 by these).
constexpr int COUNTS = 64, SELF_ROWS = 256;

__device__ __forceinline__ bool has_teacher(const DistillArgs& a, long long row) {
  RawEntry e;
  e.load(a, row * a.k);
  return !left_out(a, e.id(a));
}
__global__ __launch_bounds__(256) void distill_count(DistillArgs a, float* counts) {
  __shared__ float lds[4];
  int n = 0;
  for (long long i = blockIdx.x * 256 + threadIdx.x; i < a.rows; i += COUNTS * 256)
    n += has_teacher(a, i);
  const float s = wave_sum((float)n);   // exact: below 2^24 rows
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

// The sum of the rows' losses, for a mean divided by the number of rows with a teacher.
__global__ __launch_bounds__(1024) void distill_reduce(DistillArgs a, float* loss, float* count) {
  __shared__ float lds[16];
  constexpr int AHEAD = 16;
  const int rows = (int)a.rows;
  auto total = [&](const float* v) {
    float s = 0.f;
    int i = threadIdx.x;
    for (; i + (AHEAD - 1) * 1024 < rows; i += AHEAD * 1024) {
      float x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) x[k] = v[i + k * 1024];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) s += x[k];
    }
    for (; i < rows; i += 1024) s += v[i];
    return block_sum<1024>(s, lds);
  };
  const float s = total(a.row_loss), n = a.row_has ? total(a.row_has) : 1.f;
  if (threadIdx.x == 0) {
    if (count) *count = n;
    *loss = s / n;
  }
}

// What a row's gradient needs: off the list 2^((z - ref) c2) coef, on it
// 2^((z - m) c2) ws - q, q = 2^((t - tm) log2 e) qs, all times tau and the loss's gradient.
struct RowStats {
  float ref, coef, m, ws, tm, qs;
};

__device__ __forceinline__ float natural_exp(float x) {
  return __builtin_amdgcn_exp2f(x * LOG2E);
}
__device__ __forceinline__ float natural_log(float x) { return __builtin_amdgcn_logf(x) * LN2; }

// One row by THREADS threads that hold it in registers, HELD pieces each, packed between the
// steps: it is read once, and its gradient written once.  With HELD = 0 a workgroup streams its
// row, twice with a gradient.
//
// Thread j deals with entries j, j + THREADS, ... of the list, while the row is on its way.  A
// bitmap of the classes says which entry of a class is its first (the others add nothing to the list's
// sum, and the first writes the gradient), and with REST which logits are not the rest's: they
// become -inf before the row is summed.
//
// Bound by the memory: 8192 bf16 rows of 50257 with gradient, lists of 64, take 297 us (5.5 TB/s) and
// with REST 307, of an odd stride 310 and 325; the losses alone 142 and 165, there the vector units
// too (passes among others, their two small launches included; the shortest of five averages).  The
// listed classes' second writes are 4 to 15 us of these.  (Put into their pieces before the first and
// only write they cost as much in waiting for the list: 1% less, but 2% more for 2048 rows of 131072,
// and 10% more where rows are few or short.)
template <class T, int THREADS, int HELD, bool REST, bool GRAD, bool PAST>
__global__ __launch_bounds__(THREADS, HELD > 16 ? 2 : HELD > 8 ? 4 : 8)
void distill_row(DistillArgs a) {
  constexpr int N = Piece<T>::N, AHEAD = 4, W = THREADS / 64;
  constexpr int SPAN = HELD ? HELD * THREADS : 32768;
  // the waves' maxima and sums: of the row, the list, the teacher; their losses
  __shared__ float row_max[16], list_max[16], teacher_max[16];
  __shared__ float row_sum[16], list_sum[16], teacher_sum[16], losses[16], counted[16];
  __shared__ int ids[LIST_MAX];
  // the list's logits; log probabilities, then q
  __shared__ float zs[LIST_MAX], ts[LIST_MAX];
  __shared__ __attribute__((aligned(16))) uint32_t marks[SPAN / 4];   // of SPAN pieces
  __shared__ float edge_logits[16];
  __shared__ uint32_t edge_marks;
  __shared__ int twice;
  typedef typename Row<T>::type type;
  const long long row = blockIdx.x;
  const int t = threadIdx.x, wave = t >> 6, K = a.k;
  const int list_waves = K < THREADS ? (K + 63) >> 6 : W;   // the waves with a part of the list
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = GRAD ? (T*)a.dz + row * a.ds : nullptr;
  const Row<T> r(z, a.classes);
  const int edge = r.edge(t);
  RawEntry named;
  named.load(a, row * K);
  // the thread's first entry is on its way before the row, which the list's logits follow
  RawEntry first_entry;
  first_entry.load(a, row * K + (t < K ? t : 0));
  float z0 = 0.f;
  i32x4 x[HELD ? HELD : 1] = {};
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = k * THREADS + t;
    if (i < r.pieces) x[k] = load_piece<T, PAST>(z + r.piece_class(i));
  }
  if (edge >= 0) edge_logits[t] = (float)z[edge];   // (registers are few)
  if (left_out(a, named.id(a))) {
    if (t == 0) a.row_loss[row] = 0.f;
    if (t == 0 && a.row_has) a.row_has[row] = 0.f;
    if (t < 6 && a.stats) a.stats[t * a.rows + row] = 0.f;
    if (GRAD) {
      const type zero = {};
      for (int i = t; i < r.pieces; i += THREADS) *(type*)(dz + r.piece_class(i)) = zero;
      if (edge >= 0) dz[edge] = (T)0.f;
    }
    return;
  }
  // One wave of entries clears the marks that it sets itself, other lanes than set them: without a
  // barrier, but in this order.
  if (t == 0) {
    edge_marks = 0;
    twice = 0;
  }
  const int marking = K <= 64 ? 64 : THREADS;
  const int words = ((r.pieces < SPAN ? r.pieces : SPAN) + 15) / 16;
  if (t < marking)
    for (int i = t; i < words; i += marking) ((i32x4*)marks)[i] = i32x4{0, 0, 0, 0};
  if (REST || !HELD) {
    if (marking > 64) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // the list; entries that are left out have no class
  float most_t = -INF, bad = 0.f;   // a NaN where a class is outside
  auto entry = [&](int j, long long c, float q) {
    const bool known = c >= 0 && c < a.classes, in = known && (int)c != a.skip;
    if (!known && c != a.none) bad = __builtin_nanf("");
    ids[j] = in ? (int)c : -1;
    ts[j] = in ? q : -INF;
    if (!REST && in) most_t = maximum(most_t, q);
    return in;
  };
  if (t < K && entry(t, first_entry.id(a), first_entry.value(a))) z0 = (float)z[ids[t]];
  for (int j = t + THREADS; j < K; j += THREADS) {
    RawEntry e;
    e.load(a, row * K + j);
    if (entry(j, e.id(a), e.value(a))) zs[j] = (float)z[ids[j]];
  }
  // the first entry of each class among SPAN pieces from `first` on
  uint32_t firsts = 0;
  auto mark_list = [&](int first) {
    int it = 0;
    for (int j = t; j < K; j += THREADS, ++it) {
      uint32_t *word, bit;
      if (ids[j] >= 0 &&
          find_mark(r, ids[j], first, SPAN, first == 0, marks, &edge_marks, word, bit)) {
        if (atomicOr(word, bit) & bit) twice = 1;
        else firsts |= 1u << it;
      }
    }
  };
  const uint8_t* byte_marks = (const uint8_t*)marks;
  auto without_listed = [&](i32x4 v, uint32_t listed) {
    type e = __builtin_bit_cast(type, v);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (listed >> j & 1) e[j] = (T)-INF;
    return __builtin_bit_cast(i32x4, e);
  };
  if (REST || !HELD) {
    mark_list(0);
    __syncthreads();
  }
  if (t < K) zs[t] = z0;
  // the thread's class beside the pieces, if it is the row's
  auto edge_logit = [&]() {
    return r.edge(t) < 0 || (REST && edge_marks >> t & 1) ? -INF : edge_logits[t];
  };
  // (with 48 pieces a thread 2% less, of 2048 bf16 rows of 151936; with fewer up to 1% more)
  auto here = [&]() { return HELD > 16 ? anew(r.pieces) : r.pieces; };
  Part p = {edge_logit(), 0.f};
  if constexpr (HELD > 0) {
    int pieces = here();
    if constexpr (REST) {
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const int i = k * THREADS + t;
        const uint32_t listed = i < pieces ? byte_marks[i] : 0;
        if (listed) x[k] = without_listed(x[k], listed);
      }
      repack(x);
      pieces = here();
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (k * THREADS + t < pieces) p.m = maximum(p.m, piece_max<T>(x[k]));
    repack(x);
  } else {
    p.s = __builtin_amdgcn_exp2f((p.m - (p.m == -INF ? 0.f : p.m)) * a.c2);
    for (int first = 0; first < r.pieces; first += SPAN) {
      const int last = first + SPAN < r.pieces ? first + SPAN : r.pieces;
      if (first > 0) {
        __syncthreads();
        for (int i = t; i < (last - first + 3) / 4; i += THREADS) marks[i] = 0;
        __syncthreads();
        mark_list(first);
        __syncthreads();
      }
      for (int i0 = first + t; i0 < last; i0 += AHEAD * THREADS) {
        i32x4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          v[k] = load_piece<T, PAST>(z + r.piece_class(i < last ? i : i0));
        }
        float m = p.m;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS < last ? i0 + k * THREADS : i0;
          if (REST) {
            const uint32_t listed = byte_marks[i - first];
            if (listed) v[k] = without_listed(v[k], listed);
          }
          m = maximum(m, piece_max<T>(v[k]));
        }
        rescale(p, m, a.c2);
        const float m0 = m == -INF ? 0.f : m;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (i0 + k * THREADS < last) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              p.s += __builtin_amdgcn_exp2f((element<T>(v[k], j) - m0) * a.c2);
          }
      }
    }
  }
  const float wave_m = wave_max(p.m);
  if ((t & 63) == 0) row_max[wave] = wave_m;
  if (wave < list_waves) {
    float most_l = -INF;
    if (REST) {
      int it = 0;
      for (int j = t; j < K; j += THREADS, ++it)
        if (firsts >> it & 1) most_l = maximum(most_l, zs[j]);
      most_l = wave_max(most_l);
    } else {
      most_t = wave_max(most_t);
    }
    if ((t & 63) == 0) (REST ? list_max : teacher_max)[wave] = REST ? most_l : most_t;
  }
  __syncthreads();
  const float m = waves_max(row_max, W), m0 = m == -INF ? 0.f : m;
  const float ml = REST ? waves_max(list_max, list_waves) : -INF;
  const float tm = REST ? 0.f : waves_max(teacher_max, list_waves);
  if constexpr (HELD > 0) {
    p.s = __builtin_amdgcn_exp2f((edge_logit() - m0) * a.c2);
    const int pieces = here();
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      if (k * THREADS + t < pieces) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          p.s += __builtin_amdgcn_exp2f((element<T>(x[k], j) - m0) * a.c2);
      }
    }
    repack(x);
  } else {
    rescale(p, m, a.c2);
  }
  float count = 1.f;
  if (GRAD && a.counts) count = a.counts[t & 63];
  if (GRAD && a.self_count) {
    const float n = wave_sum(t < a.rows && has_teacher(a, t) ? 1.f : 0.f);
    if ((t & 63) == 0) counted[wave] = n;
  }
  const float wave_s = wave_sum(p.s);
  if ((t & 63) == 0) row_sum[wave] = wave_s;
  if (wave < list_waves) {
    if (!REST && HELD && GRAD) mark_list(0);
    float sl = 0.f, st = bad;
    int it = 0;
    for (int j = t; j < K; j += THREADS, ++it) {
      if (REST && firsts >> it & 1)
        sl += ml == -INF ? 0.f : __builtin_amdgcn_exp2f((zs[j] - ml) * a.c2);
      if (ids[j] >= 0) st += natural_exp(ts[j] - tm);
    }
    st = wave_sum(st);
    if (REST) sl = wave_sum(sl);
    if ((t & 63) == 0) teacher_sum[wave] = st;
    if ((t & 63) == 0) list_sum[wave] = sl;
  }
  __syncthreads();
  p = {m, waves_sum(row_sum, W)};
  const float qsum = waves_sum(teacher_sum, list_waves);
  Part all = p;
  if (REST) {
    all.m = maximum(m, ml);
    const float sl = waves_sum(list_sum, list_waves);
    all.s = (m == -INF ? 0.f : p.s * __builtin_amdgcn_exp2f((m - all.m) * a.c2)) +
            (ml == -INF ? 0.f : sl * __builtin_amdgcn_exp2f((ml - all.m) * a.c2));
  }
  // coefficients
  const float log_s = natural_log(all.s);
  const bool others = REST && m != -INF;
  const float left = others && 1.f - qsum > a.slack ? 1.f - qsum : 0.f;
  float w = !REST ? qsum / qsum : others && qsum <= 1.f ? 1.f : qsum;
  if (!(all.s >= 0.5f) || (REST && !others && qsum == 0.f)) w = __builtin_nanf("");
  RowStats st;
  st.m = all.m;
  st.ws = w / all.s;
  st.tm = tm;
  st.qs = REST ? 1.f : 1.f / qsum;
  st.ref = m0;
  st.coef = st.ws;
  if (REST) {
    st.coef = st.ws * (m == -INF ? 0.f : __builtin_amdgcn_exp2f((m - all.m) * a.c2));
    if (left > 0.f) st.coef -= left / p.s;
  }
  if (wave < list_waves) {
    float loss = 0.f;
    const float log_q = REST ? 0.f : natural_log(qsum);
    for (int j = t; j < K; j += THREADS) {
      const float q = ids[j] >= 0 ? natural_exp(ts[j] - tm) * st.qs : 0.f;
      // not below: a NaN goes on
      if (!(q <= 0.f)) loss += q * ((ts[j] - tm - log_q) - ((zs[j] - all.m) * a.itau - log_s));
      ts[j] = q;
    }
    loss = wave_sum(loss);
    if ((t & 63) == 0) losses[wave] = loss;
  }
  if constexpr (GRAD) {
    if (a.counts) count = wave_sum(count);
    if (a.self_count) count = waves_sum(counted, W);
    const float g = a.gscale / count;
    const float coef = st.coef * g;
    auto gradient = [&](i32x4 v) {
      type d;
#pragma unroll
      for (int j = 0; j < N; ++j)
        d[j] = (T)(__builtin_amdgcn_exp2f((element<T>(v, j) - st.ref) * a.c2) * coef);
      return __builtin_bit_cast(i32x4, d);
    };
    if constexpr (HELD > 0) {
      const int pieces = here();
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const int i = k * THREADS + t;
        if (i < pieces) store_piece<T, PAST>(dz + r.piece_class(i), gradient(x[k]));
      }
    } else {
      for (int i0 = t; i0 < r.pieces; i0 += AHEAD * THREADS) {
        i32x4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          v[k] = load_piece<T, PAST>(z + r.piece_class(i < r.pieces ? i : i0));
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          if (i < r.pieces) store_piece<T, PAST>(dz + r.piece_class(i), gradient(v[k]));
        }
      }
    }
    if (r.edge(t) >= 0)
      dz[r.edge(t)] = (T)(__builtin_amdgcn_exp2f((edge_logits[t] - st.ref) * a.c2) * coef);
    __syncthreads();   // the losses; and the listed classes again, by the first entry of each
    int it = 0;
    for (int j = t; j < K; j += THREADS, ++it) {
      if (firsts >> it & 1) {
        float q = ts[j];
        if (twice) {   // a class listed more than once: its terms in their order
          q = 0.f;
          for (int i = 0; i < K; ++i) q += ids[i] == ids[j] ? ts[i] : 0.f;
        }
        dz[ids[j]] = (T)((__builtin_amdgcn_exp2f((zs[j] - st.m) * a.c2) * st.ws - q) * g);
      }
    }
  } else {
    __syncthreads();
  }
  if (t == 0) {
    float loss = losses[0];
    for (int i = 1; i < list_waves; ++i) loss += losses[i];
    if (REST && left > 0.f)
      loss += left * (natural_log(left) - ((m - all.m) * a.itau + natural_log(p.s) - log_s));
    a.row_loss[row] = w == w ? loss * a.lscale : w;
    if (a.row_has) a.row_has[row] = 1.f;
    if (a.stats) a.stats[row] = st.ref;
    if (a.stats) a.stats[a.rows + row] = st.coef;
    if (a.stats) a.stats[2 * a.rows + row] = st.m;
    if (a.stats) a.stats[3 * a.rows + row] = st.ws;
    if (a.stats) a.stats[4 * a.rows + row] = st.tm;
    if (a.stats) a.stats[5 * a.rows + row] = st.qs;
  }
}

// The fewest threads that hold a row; longer rows are held for the gradient as far as registers
// go, and streamed for the loss alone.  (2048 bf16 rows with gradient: of 131072 233 us, of 151936 298,
// of 200064, which are read twice, 440.)  Rows of few classes are bound by a workgroup's latency:
// 16384 of 256 to 2000 bf16 classes take 30 us, with gradient 52 to 57.
template <class T, bool REST, bool GRAD, bool PAST>
static void launch_rows(hipStream_t stream, const DistillArgs& a) {
  const int pieces = a.classes / Piece<T>::N;   // at most
  const dim3 rows((unsigned)a.rows);
#define DMH_ROWS(THREADS, HELD)                                                                   \
  if (pieces <= THREADS * HELD) {                                                                 \
    hipLaunchKernelGGL((distill_row<T, THREADS, HELD, REST, GRAD, PAST>), rows, dim3(THREADS), 0, \
                       stream, a);                                                                \
    return;                                                                                       \
  }
  DMH_ROWS(256, 8)
  DMH_ROWS(1024, 8)
  if constexpr (GRAD) {
    DMH_ROWS(1024, 16)
    DMH_ROWS(512, 48)
  }
#undef DMH_ROWS
  hipLaunchKernelGGL((distill_row<T, 1024, 0, REST, GRAD, PAST>), rows, dim3(1024), 0, stream, a);
}
template <class T, bool REST, bool GRAD>
static void launch_sized(hipStream_t stream, const DistillArgs& a) {
  if (!a.stats && past_caches<T>(a.rows, a.classes))   // (with statistics, the gradient comes next)
    launch_rows<T, REST, GRAD, true>(stream, a);
  else
    launch_rows<T, REST, GRAD, false>(stream, a);
}
template <class T>
static void launch_distill(hipStream_t stream, const DistillArgs& a, bool rest) {
  if (rest)
    a.dz ? launch_sized<T, true, true>(stream, a) : launch_sized<T, true, false>(stream, a);
  else
    a.dz ? launch_sized<T, false, true>(stream, a) : launch_sized<T, false, false>(stream, a);
}

// The gradient from a forward pass's statistics, element by element, 256 threads for four pieces
// each of a row; the listed classes are written again behind a barrier.  Bound by the memory: 78 us
// for 2000 fp32 rows of 32003 (512 MB, 6.6 TB/s; the logits are partly in the last-level cache
// still).  Not more than 64 registers: with two more only seven waves fit.
template <class T, bool PAST>
__global__ __launch_bounds__(256, 8) void distill_grad(DistillArgs a) {
  constexpr int N = Piece<T>::N, AHEAD = 4, THREADS = 256;
  __shared__ int ids[LIST_MAX];
  __shared__ float qs[LIST_MAX];
  __shared__ uint32_t marks[THREADS];
  __shared__ uint32_t edge_marks;
  __shared__ int twice;
  typedef typename Row<T>::type type;
  const long long row = blockIdx.x;
  const int t = threadIdx.x, K = a.k;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = (T*)a.dz + row * a.ds;
  const Row<T> r(z, a.classes);
  const int first = blockIdx.y * THREADS * AHEAD, i0 = first + t;
  const int ec = blockIdx.y == 0 ? r.edge(t) : -1;
  if (left_out(a, load_index(a.ids, a.i64, row * K))) {
    const type zero = {};
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i0 + k * THREADS < r.pieces) *(type*)(dz + r.piece_class(i0 + k * THREADS)) = zero;
    if (ec >= 0) dz[ec] = (T)0.f;
    return;
  }
  i32x4 x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    if (r.pieces) x[k] = load_piece<T, PAST>(z + r.piece_class(i < r.pieces ? i : 0));
  }
  const float ex = ec >= 0 ? (float)z[ec] : 0.f;
  RowStats st;
  st.ref = a.stats[row];
  st.coef = a.stats[a.rows + row];
  st.m = a.stats[2 * a.rows + row];
  st.ws = a.stats[3 * a.rows + row];
  st.tm = a.stats[4 * a.rows + row];
  st.qs = a.stats[5 * a.rows + row];
  float g = a.gout[a.gout_rows ? row : 0] * a.gscale;
  if (a.count) g /= *a.count;
  marks[t] = 0;
  if (t == 0) {
    edge_marks = 0;
    twice = 0;
  }
  for (int j = t; j < K; j += THREADS) {
    RawEntry e;
    e.load(a, row * K + j);
    const long long c = e.id(a);
    const bool in = c >= 0 && c < a.classes && (int)c != a.skip;
    ids[j] = in ? (int)c : -1;
    qs[j] = in ? natural_exp(e.value(a) - st.tm) * st.qs : 0.f;
  }
  const float coef = st.coef * g;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    type d;
#pragma unroll
    for (int j = 0; j < N; ++j)
      d[j] = (T)(__builtin_amdgcn_exp2f((element<T>(x[k], j) - st.ref) * a.c2) * coef);
    if (i < r.pieces)
      store_piece<T, PAST>(dz + r.piece_class(i), __builtin_bit_cast(i32x4, d));
  }
  if (ec >= 0) dz[ec] = (T)(__builtin_amdgcn_exp2f((ex - st.ref) * a.c2) * coef);
  __syncthreads();   // also: the list is written
  uint32_t firsts = 0;
  int it = 0;
  for (int j = t; j < K; j += THREADS, ++it) {
    uint32_t *word, bit;
    if (ids[j] >= 0 && find_mark(r, ids[j], first, THREADS * AHEAD, blockIdx.y == 0, marks,
                                 &edge_marks, word, bit)) {
      if (atomicOr(word, bit) & bit) twice = 1;
      else firsts |= 1u << it;
    }
  }
  __syncthreads();
  it = 0;
  for (int j = t; j < K; j += THREADS, ++it) {
    if (firsts >> it & 1) {
      const int c = ids[j];
      float q = qs[j];
      if (twice) {
        q = 0.f;
        for (int i = 0; i < K; ++i) q += ids[i] == c ? qs[i] : 0.f;
      }
      dz[c] = (T)((__builtin_amdgcn_exp2f(((float)z[c] - st.m) * a.c2) * st.ws - q) * g);
    }
  }
}

template <class T>
static void launch_distill_grad(hipStream_t stream, const DistillArgs& a) {
  const int whole = a.classes / Piece<T>::N;
  const dim3 grid((unsigned)a.rows, (unsigned)(whole ? ceil_div(whole, 1024) : 1));
  if (past_caches<T>(a.rows, a.classes))
    hipLaunchKernelGGL((distill_grad<T, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((distill_grad<T, false>), grid, dim3(256), 0, stream, a);
}

static bool distill_shape(long long rows, long long classes, long long k) {
  return rows >= 0 && rows < (1LL << 22) && classes >= 1 && classes <= (1LL << 27) && k >= 1 &&
         k <= LIST_MAX;
}

static DistillArgs distill_args(const void* logits, long long rows, long long classes,
                                long long z_rstride, const void* ids, int ids_64, int k,
                                const void* teacher, int teacher_dtype, long long ignore_index,
                                float temperature, float* stats, const float* count,
                                void* dlogits, long long d_rstride) {
  DistillArgs a{};
  a.z = logits;
  a.ids = ids;
  a.teacher = teacher;
  a.dz = dlogits;
  a.stats = stats;
  a.count = count;
  a.rows = rows;
  a.zs = z_rstride;
  a.ds = d_rstride;
  a.none = no_class(ignore_index, classes);
  a.ignore = ignore_index;
  a.skip = a.none == ignore_index ? -1 : (int)ignore_index;
  a.classes = (int)classes;
  a.k = k;
  a.i64 = ids_64 != 0;
  a.ttype = teacher_dtype;
  a.itau = (float)(1.0 / temperature);
  a.c2 = (float)(1.4426950408889634 / temperature);
  a.lscale = temperature * temperature;
  a.gscale = temperature;
  // Each of q's exponents t is off by half a last place and its product by another, 2^-24 |t| each,
  // and sum q |t| is at most log k where sum q is 1; 8 for the exponentials and their sum.
  a.slack = (float)(8.0 + 2.0 * log((double)k)) * 0x1p-24f;
  return a;
}

}  // namespace dmh

using namespace dmh;

extern "C" {

int dmh_distill_workspace_size(long long rows, size_t* bytes) {
  if (!bytes || !distill_shape(rows, 1, 1)) {
    set_error("dmh_distill_workspace_size: bad arguments (rows=%lld)", rows);
    return DMH_EINVAL;
  }
  *bytes = 4 * (2 * (size_t)rows + COUNTS);
  return DMH_OK;
}

int dmh_distill(hipStream_t stream, const void* logits, int dtype, long long rows,
                long long classes, long long z_rstride, const void* ids, int ids_64, int k,
                const void* teacher, int teacher_dtype, long long ignore_index, float temperature,
                int rest, int reduction, float grad_scale, float* loss, float* count,
                float* stats, void* dlogits, long long d_rstride, void* ws, size_t ws_bytes) {
  if (!distill_shape(rows, classes, k) || z_rstride < 0 || d_rstride < 0 || !float_code(dtype) ||
      !float_code(teacher_dtype) || !(temperature >= 1e-6f && temperature <= 1e6f) ||
      reduction < RED_NONE || reduction > RED_SUM) {
    set_error("dmh_distill: bad arguments (rows=%lld classes=%lld dtype=%d k=%d teacher_dtype=%d "
              "temperature=%g reduction=%d)", rows, classes, dtype, k, teacher_dtype,
              (double)temperature, reduction);
    return DMH_EINVAL;
  }
  if (!loss || (reduction == RED_MEAN && !count) ||
      (rows > 0 && (!logits || !ids || !teacher))) {
    set_error("dmh_distill: null tensor");
    return DMH_EINVAL;
  }
  size_t need;
  dmh_distill_workspace_size(rows, &need);
  if (reduction != RED_NONE && need > 0 && (!ws || ws_bytes < need)) {
    set_error("dmh_distill: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return DMH_EWORKSPACE;
  }
  const bool mean = reduction == RED_MEAN;
  DistillArgs a = distill_args(logits, rows, classes, z_rstride, ids, ids_64, k, teacher,
                               teacher_dtype, ignore_index, temperature, stats, nullptr, dlogits,
                               d_rstride);
  a.row_loss = reduction == RED_NONE ? loss : (float*)ws;
  a.gscale *= grad_scale;
  if (mean) a.row_has = (float*)ws + rows;
  if (mean && dlogits && rows > SELF_ROWS) {
    float* counts = (float*)ws + 2 * rows;
    hipLaunchKernelGGL(distill_count, dim3(COUNTS), dim3(256), 0, stream, a, counts);
    DMH_CHECK_LAUNCH("distill_count");
    a.counts = counts;
  }
  a.self_count = mean && dlogits && rows <= SELF_ROWS;
  if (rows > 0) {
    DMH_FOR_TYPE(dtype, T, (launch_distill<T>(stream, a, rest != 0)))
    DMH_CHECK_LAUNCH("distill_row");
  }
  if (reduction != RED_NONE) {
    hipLaunchKernelGGL(distill_reduce, dim3(1), dim3(1024), 0, stream, a, loss,
                       mean ? count : nullptr);
    DMH_CHECK_LAUNCH("distill_reduce");
  }
  return DMH_OK;
}

int dmh_distill_grad(hipStream_t stream, const void* logits, int dtype, long long rows,
                     long long classes, long long z_rstride, const void* ids, int ids_64, int k,
                     const void* teacher, int teacher_dtype, long long ignore_index,
                     float temperature, const float* stats, const float* count,
                     const float* grad_out, int grad_out_rows, void* dlogits,
                     long long d_rstride) {
  if (!distill_shape(rows, classes, k) || z_rstride < 0 || d_rstride < 0 || !float_code(dtype) ||
      !float_code(teacher_dtype) || !(temperature >= 1e-6f && temperature <= 1e6f)) {
    set_error("dmh_distill_grad: bad arguments (rows=%lld classes=%lld dtype=%d k=%d "
              "teacher_dtype=%d temperature=%g)", rows, classes, dtype, k, teacher_dtype,
              (double)temperature);
    return DMH_EINVAL;
  }
  if (rows == 0) return DMH_OK;
  if (!logits || !ids || !teacher || !stats || !grad_out || !dlogits) {
    set_error("dmh_distill_grad: null tensor");
    return DMH_EINVAL;
  }
  if (dlogits == logits) {   // the listed classes' are read again
    set_error("dmh_distill_grad: the gradient cannot take the logits' place");
    return DMH_EINVAL;
  }
  DistillArgs a = distill_args(logits, rows, classes, z_rstride, ids, ids_64, k, teacher,
                               teacher_dtype, ignore_index, temperature, (float*)stats, count,
                               dlogits, d_rstride);
  a.gout = grad_out;
  a.gout_rows = grad_out_rows != 0;
  DMH_FOR_TYPE(dtype, T, (launch_distill_grad<T>(stream, a)))
  DMH_CHECK_LAUNCH("distill_grad");
  return DMH_OK;
}

}  // extern "C"
