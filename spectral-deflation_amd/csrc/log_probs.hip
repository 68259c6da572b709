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
// A row whose token is `ignore` gives 0 everywhere and `none` for its classes.  A row without a
// softmax (a NaN, an infinity, -inf alone) gives NaN and the classes 0 to K - 1.
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
  long long rows, zs, ignore, none;   // none: what stands for no class
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

// The largest of each of HELD pieces, for later: two 16-bit values a register, while fp32 ones are
// found again from the piece, in three instructions.  (A register for each piece made the compiler
// spill a few others, whose reloads made the 8192 rows below 60% slower.)
template <class T, int HELD>
struct PieceMaxima {
  typedef T pair __attribute__((ext_vector_type(2)));
  int m[HELD ? HELD / 2 : 1];
  __device__ __forceinline__ void put(int k, float even, float odd) {   // of pieces k and k + 1
    if constexpr (std::is_same<T, bf16>::value)
      m[k / 2] = (int)__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, odd),
                                            __builtin_bit_cast(uint32_t, even), 0x07060302u);
    else
      m[k / 2] = __builtin_bit_cast(int, pair{(T)even, (T)odd});
  }
  __device__ __forceinline__ float get(int k, i32x4) const {
    return element<T>(i32x4{m[k / 2], 0, 0, 0}, k & 1);
  }
};
template <int HELD>
struct PieceMaxima<float, HELD> {
  __device__ __forceinline__ void put(int, float, float) {}
  __device__ __forceinline__ float get(int, i32x4 x) const { return piece_max<float>(x); }
};
// What a value with an order_key of at least cut is at least.
__device__ __forceinline__ float cut_value(uint32_t cut) {
  return cut < 0x007FFFFFu ? -INF : key_value(cut);
}

// The smallest of a wave's, in all lanes.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t lesser(uint32_t v) {
  const uint32_t o = __builtin_amdgcn_update_dpp(-1, (int)v, CTRL, ROWS, 0xF, false);
  return o < v ? o : v;
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  v = lesser<0x118>(lesser<0x114>(lesser<0x112>(lesser<0x111>(v))));
  return __builtin_amdgcn_readlane(lesser<0x143, 0xC>(lesser<0x142, 0xA>(v)), 63);
}

constexpr int SEGMENTS = 8;   // of a thread's part of a long row, whose maxima are kept
constexpr int CANDS = 1024;   // what is sorted out in the end, K <= TOP_MAX of them kept

struct TopLds {
  uint32_t keys[512];   // of groups of threads
  u64 cand[CANDS];
  uint32_t cut, most;
  int slots[128];        // a counter for each step of the search over all classes
  int n;
};

// A lower bound of the K-th largest of a row, by the first wave: the K-th largest of the maxima of
// 64 PER groups of threads, since K groups have a class that large.  Halving what lies between the
// smallest of them and the largest (bit by bit from the first one on, the 64 largest of 8009 classes
// took 6% longer, two bits at a time 17%), and no further than to a few groups more than K: their
// classes are ranked by comparing all with all (with K / 4 groups more, 256 of 50257 classes took
// 19% longer).  The other waves go on with the row's sum.
template <int PER>
__device__ __forceinline__ void group_cut(int K, uint32_t high, TopLds& l) {
  uint32_t k[PER], low = ~0u;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    k[i] = l.keys[i * 64 + (threadIdx.x & 63)];
    low = k[i] < low ? k[i] : low;
  }
  low = wave_min(low);
  if (threadIdx.x == 0) l.most = high;
  const int enough = K + K / 16 + 1;
  __builtin_amdgcn_s_setprio(3);   // the others wait for this one in the end
  while (low < high) {   // ends: low grows or high falls
    const uint32_t c = low + (high - low) / 2 + 1;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(k[i] >= c));
    if (n >= K) {
      low = c;
      if (n <= enough) break;
    } else {
      high = c - 1;
    }
  }
  if (threadIdx.x == 0) l.cut = low;
}

// The threads' maxima by groups: 256, or 512 for more than 64 classes.  (Of 256 and K = 64, about
// 74 classes are as large as the 64th group's; of 512 and K = 256, about 355.)  Zeroes the counters
// of what follows.
template <int THREADS>
__device__ __forceinline__ void put_group(int K, float largest, TopLds& l) {
  uint32_t k = order_key(largest), o;
  int t = threadIdx.x;
  if (THREADS == 1024) {
    o = __builtin_amdgcn_mov_dpp((int)k, 0xB1, 0xF, 0xF, true);   // lane ^ 1
    k = o > k ? o : k;
    t >>= 1;
    if (K <= 64) {
      o = __builtin_amdgcn_mov_dpp((int)k, 0x4E, 0xF, 0xF, true);   // lane ^ 2
      k = o > k ? o : k;
      t >>= 1;
    }
  }
  l.keys[t] = k;   // the same from all threads of a group
  if (threadIdx.x == 0) l.n = 0;
  if (threadIdx.x < 128) l.slots[threadIdx.x] = 0;
}
template <int THREADS>
__device__ __forceinline__ void find_cut(int K, float largest, TopLds& l) {
  const uint32_t high = __builtin_amdgcn_readfirstlane(order_key(largest));
  if (THREADS == 256 || K <= 64) group_cut<4>(K, high, l);
  else group_cut<8>(K, high, l);
}

// A candidate from each lane that has one; all lanes of the wave come here.
__device__ __forceinline__ void put_candidate(bool has, u64 key, TopLds& l) {
  const u64 who = __ballot(has);
  if (who == 0) return;
  int at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(&l.n, __popcll(who));
  at = __builtin_amdgcn_readfirstlane(at) +
       __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                 __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
  if (has && at < CANDS) l.cand[at] = key;
}

// Pieces with a class that is large enough, gathered by a wave, 64 at most: their elements side by
// side in the lanes, 64 at a time.
struct PieceList {
  i32x4 data[64];
  int first[64];   // class of a piece's first element
};
template <class T>
__device__ __forceinline__ void put_pieces(int count, u64 from, const PieceList& p, TopLds& l) {
  constexpr int N = Piece<T>::N;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int e = threadIdx.x & 63; (e & ~63) < count * N; e += 64) {
    const bool in = e < count * N;
    const int q = in ? e : 0;
    const u64 k = rank_key((float)((const T*)p.data)[q], p.first[q / N] + q % N);
    put_candidate(in && k >= from, k, l);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The candidates where more than CANDS classes are above the cut: many large ones in few groups, or
// many equal ones.  each(cut, first, last, f) calls f(key, class) for the thread's classes from
// first to last - 1 whose order_key is at least cut.
//
// First the K-th largest value.  The groups' is the row's where equal classes are the cause; else a
// bit at a time between it and the largest, which only threads with such classes have to look at.
// Then, if its classes are still too many, the first of them: twice as far each time, and the last
// step halved.
template <int THREADS, class Each>
__device__ __forceinline__ void search_top(int K, int classes, const Each& each, TopLds& l) {
  uint32_t value = l.cut;
  const uint32_t most = l.most;
  int step = 0;
  auto count = [&](uint32_t least, uint32_t up_to, int first, int last) {
    int n = 0;
    each(least, first, last, [&](uint32_t k, int) { n += k <= up_to; });
    const float s = wave_sum((float)n);   // exact: a wave has fewer than 2^24 classes
    if ((threadIdx.x & 63) == 0 && s != 0.f) atomicAdd(&l.slots[step], (int)s);
    __syncthreads();
    return l.slots[step++];
  };
  auto gather = [&](uint32_t least, int first, int last, uint32_t equal, int end) {
    each(least, first, last, [&](uint32_t k, int c) {
      if (k != equal || c < end) {
        const int at = atomicAdd(&l.n, 1);
        if (at < CANDS) l.cand[at] = (u64)k << 32 | (uint32_t)~c;
      }
    });
  };
  __syncthreads();   // everyone has seen that there are too many
  if (threadIdx.x == 0) l.n = 0;
  int above = value == most ? 0 : count(value + 1, most, 0, classes);
  if (above >= K) {
    int n = above;
    value += 1;
    if (n > CANDS) {
      const int high = value == most ? -1 : 31 - __clz(value ^ most);
      value = high < 0 ? most : most & ~((2u << high) - 1u);
      for (int b = high; b >= 0; --b) {
        const uint32_t c = value | 1u << b;
        const int now = count(c, most, 0, classes);
        if (now >= K) {
          value = c;
          n = now;
          if (n <= CANDS) break;
        }
      }
    }
    if (n <= CANDS) {
      gather(value, 0, classes, 0, 0);
      __syncthreads();
      return;
    }
    above = value == most ? 0 : count(value + 1, most, 0, classes);
  }
  int first = 0, last = classes < 512 ? classes : 512, before = 0, here;
  // (both loops end, and all stores stay inside, also if someone writes to the row meanwhile)
  while (before + (here = count(value, value, first, last)) < K - above && last < classes) {
    before += here;
    first = last;
    last = last < classes / 2 ? 2 * last : classes;
  }
  while (above + before + here > CANDS && last - first > 1) {
    const int middle = first + (last - first) / 2, n = count(value, value, first, middle);
    if (before + n < K - above) {
      before += n;
      here -= n;
      first = middle;
    } else {
      here = n;
      last = middle;
    }
  }
  if (above > 0)
    gather(value, 0, classes, value, last);
  else
    gather(value, 0, last, value, last);
  __syncthreads();
}

// The K largest candidates in their order: put(place, value, class).  A candidate's place is the
// number of larger ones, which as many threads as there are for each count together.
template <int THREADS, class Put>
__device__ __forceinline__ void put_top(int K, const Put& put, const TopLds& l) {
  const int n = l.n < CANDS ? l.n : CANDS;
  int share = 1;
  while (share < 64 && 2 * share * n <= THREADS) share *= 2;
  const int part = threadIdx.x & (share - 1);
  for (int i = threadIdx.x / share; i < n; i += THREADS / share) {
    const u64 k = l.cand[i];
    int before = 0;
#pragma unroll 4
    for (int j = part; j < n; j += share) before += l.cand[j] > k;
    for (int d = share >> 1; d; d >>= 1) before += __shfl_xor(before, d);
    if (part == 0 && before < K) put(before, key_value((uint32_t)(k >> 32)), (int)~(uint32_t)k);
  }
}

// One row by THREADS threads that hold it in registers, HELD pieces each (packed between the
// steps), or for HELD = 0 a workgroup that streams it.
//
// (Figures: a pass among others, the shortest of five averages of 30, three sets of logits in turn.)
//
// Without a top it reads each logit once and is bound by the memory, the vector units not far
// behind: 8192 bf16 rows of 50257 take 143 us (5.8 TB/s), 1000 fp32 rows of 131072 82 (6.4).  Two
// barriers and reductions by lane shifts, one for the maximum and one for the sums, take less of
// them than one that joins parts of different maxima (a fifth more).  Rows of few classes are bound
// by the workgroups' own latency: 16384 of 256, 600, 1000 or 2000 bf16 classes all take 19 to 22 us.
//
// Top classes: the threads' maxima, which the sums need anyway, give a lower bound of the K-th
// largest class that few classes reach, whatever the distribution; those are gathered, piece by
// piece, and ranked by comparing all with all.  The 64 largest take 176 us of the same rows, the
// largest alone 160, 256 of them 312.  Where too many reach the bound (equal logits, or many large
// ones in one thread's classes) the row is read again, as far as needed: 426 us for 8192 rows of
// zeros, 634 where a mask leaves 20 classes of them (181 without a top: such rows are summed twice).
// Long rows keep the maxima of SEGMENTS parts of each thread's pieces, and read again only the parts
// that reach the bound (20 of 131072 classes: 87 us, a fifth more with all parts of such threads).
// Of few classes, 20 take 16384 rows to 57 us: a workgroup's latency again.
template <class T, int THREADS, int HELD, bool TOP, bool PAST>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? 6 : 8) void log_prob_row(LogProbArgs a) {
  __shared__ float maxes[16], sums[16], weights[16];   // of the waves
  __shared__ typename std::conditional<TOP, TopLds, char>::type top;
  __shared__ typename std::conditional<(TOP && HELD > 0), PieceList, char>::type
      lists[TOP && HELD ? THREADS / 64 : 1];
  __shared__ float segments[TOP && !HELD ? SEGMENTS * THREADS : 1];
  constexpr int N = Piece<T>::N, AHEAD = 4;
  const long long row = blockIdx.x;
  const int t = threadIdx.x, K = a.top;
  const T* z = (const T*)a.z + row * a.zs;
  const Row<T> r(z, a.classes);
  const long long y = a.tokens ? load_index(a.tokens, a.t64, row) : 0;
  i32x4 x[HELD ? HELD : 1] = {};
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = k * THREADS + t;
    if (i < r.pieces) x[k] = load_piece<T, PAST>(z + r.piece_class(i));
  }
  const int ec = r.edge(t);
  const float ex = ec >= 0 ? (float)z[ec] : -INF;
  if (a.tokens && y == a.ignore) {
    if (t == 0) {
      a.lp[row] = 0.f;
      if (a.ent) a.ent[row] = 0.f;
    }
    if (t < 3 && a.stats) a.stats[t * a.rows + row] = t == 1 ? 1.f : 0.f;
    for (int i = t; i < K; i += THREADS) {
      a.top_lp[row * K + i] = 0.f;
      a.top_ids[row * K + i] = a.none;
    }
    return;
  }
  // a long row's rounds of AHEAD pieces a thread, by segment
  constexpr int ROUND = AHEAD * THREADS;
  const int segment_rounds = (r.pieces + ROUND * SEGMENTS - 1) / (ROUND * SEGMENTS);
  const bool known = a.tokens && y >= 0 && y < a.classes;
  const float zy = known ? (float)z[y] : __builtin_nanf("");
  Part3 p = {ex, 0.f, 0.f};
  // (a logit of -inf gives 0 * -inf in t, a NaN, which the end mends)
  auto add = [&](float v, float m0) {
    const float d = (v - m0) * a.c2, e = __builtin_amdgcn_exp2f(d);
    p.s += e;
    p.t = fmaf(e, d, p.t);
  };
  PieceMaxima<T, HELD> maxima;
  float m = 0.f, largest = 0.f;   // of the row and of the thread
  auto join_max = [&]() {
    largest = p.m;
    const float w = wave_max(p.m);
    if ((t & 63) == 0) maxes[t >> 6] = w;
    if constexpr (TOP) put_group<THREADS>(K, p.m, top);
    __syncthreads();
    m = waves_max(maxes, THREADS / 64);
    if constexpr (TOP)
      if (t < 64) find_cut<THREADS>(K, m, top);
  };
  if constexpr (HELD > 0) {
    // a small workgroup's waves pass over pieces behind the row (7% less for the 64 largest of 8009
    // classes; at 1024 threads up to 1% more)
    const int wave = __builtin_amdgcn_readfirstlane(t);
    int pieces = anew(r.pieces);
#pragma unroll
    for (int k = 0; k < HELD; k += 2) {
      float m0 = -INF, m1 = -INF;
      if (THREADS > 256 || k * THREADS + wave < pieces) {
        m0 = k * THREADS + t < pieces ? piece_max<T>(x[k]) : -INF;
        m1 = (k + 1) * THREADS + t < pieces ? piece_max<T>(x[k + 1]) : -INF;
        p.m = maximum(p.m, maximum(m0, m1));
      }
      if constexpr (TOP) maxima.put(k, m0, m1);
    }
    repack(x);
    join_max();
    const float m0 = m == -INF ? 0.f : m;
    if (ec >= 0) add(ex, m0);
    pieces = anew(pieces);
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      if (k * THREADS + t < pieces) {
#pragma unroll
        for (int j = 0; j < N; ++j) add(element<T>(x[k], j), m0);
      }
    }
    repack(x);
  } else {
    if (ec >= 0) add(ex, p.m == -INF ? 0.f : p.m);
    int segment = t, left = segment_rounds;
    if constexpr (TOP)
      for (int s = 0; s < SEGMENTS; ++s) segments[s * THREADS + t] = -INF;
    float of_segment = -INF;
    for (int i0 = t; i0 < r.pieces; i0 += AHEAD * THREADS) {
      i32x4 v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + k * THREADS;
        v[k] = load_piece<T, PAST>(z + r.piece_class(i < r.pieces ? i : i0));
      }
      float most = -INF;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) most = maximum(most, piece_max<T>(v[k]));
      if constexpr (TOP) {
        of_segment = maximum(of_segment, most);
        segments[segment] = of_segment;
        if (--left == 0) {
          segment += THREADS;
          left = segment_rounds;
          of_segment = -INF;
        }
      }
      most = maximum(most, p.m);
      rescale(p, most, a.c2);
      const float m0 = most == -INF ? 0.f : most;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i0 + k * THREADS < r.pieces) {
#pragma unroll
          for (int j = 0; j < N; ++j) add(element<T>(v[k], j), m0);
        }
    }
    join_max();
    rescale(p, m, a.c2);
  }
  if (!(p.t == p.t)) {   // the thread's sums again, its logits of -inf apart
    p.s = p.t = 0.f;
    const float m0 = m == -INF ? 0.f : m;
    auto again = [&](float v) {
      const float d = (v - m0) * a.c2, e = __builtin_amdgcn_exp2f(d);
      p.s += e;
      p.t = fmaf(e, fmaxf(d, LOWEST), p.t);
    };
    if (r.edge(t) >= 0) again((float)z[r.edge(t)]);
    if constexpr (HELD > 0) {
      const int pieces = anew(r.pieces);
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        if (k * THREADS + t < pieces) {
#pragma unroll
          for (int j = 0; j < N; ++j) again(element<T>(x[k], j));
        }
      }
      repack(x);
    } else {
      for (int i0 = t; i0 < r.pieces; i0 += AHEAD * THREADS) {
        i32x4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          v[k] = load_piece<T, false>(z + r.piece_class(i < r.pieces ? i : i0));
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (i0 + k * THREADS < r.pieces) {
#pragma unroll
            for (int j = 0; j < N; ++j) again(element<T>(v[k], j));
          }
      }
    }
  }
  const float ws = wave_sum(p.s), wt = wave_sum(p.t);
  if ((t & 63) == 0) {
    sums[t >> 6] = ws;
    weights[t >> 6] = wt;
  }
  if (TOP && t < 64) __builtin_amdgcn_s_setprio(0);
  __syncthreads();
  p = {m, waves_sum(sums, THREADS / 64), waves_sum(weights, THREADS / 64)};
  const float log_s = __builtin_amdgcn_logf(p.s) * LN2;
  if (t == 0) {
    const float ent = log_s - LN2 * (p.t / p.s);
    if (a.ent) a.ent[row] = ent;
    if (a.stats) a.stats[row] = p.m;
    if (a.stats) a.stats[a.rows + row] = p.s;
    if (a.stats) a.stats[2 * a.rows + row] = ent;
    if (a.tokens) a.lp[row] = (zy - p.m) * a.itau - log_s;
  }
  if constexpr (TOP) {
    if (!(p.s >= 0.5f)) {   // no softmax: the maximum alone gives 1
      for (int i = t; i < K; i += THREADS) {
        a.top_lp[row * K + i] = __builtin_nanf("");
        a.top_ids[row * K + i] = i;
      }
      return;
    }
    // (by value: what a lambda refers to may end in memory)
    auto each = [=](uint32_t cut, int first, int last, auto f) {
      if (order_key(largest) < cut) return;
      auto visit = [&](float v, int c) {
        const uint32_t k = order_key(v);
        if (k >= cut && c >= first && c < last) f(k, c);
      };
      if (r.edge(t) >= 0) visit((float)z[r.edge(t)], r.edge(t));
      const int begin = first > r.head ? (first - r.head) / N : 0;
      const int end = last > r.head ? (last - r.head + N - 1) / N : 0;
      const int stop = end < r.pieces ? end : r.pieces;
      const float least = cut_value(cut);
      // the thread's own pieces, which `largest` is of
      for (int i0 = begin + ((t - begin) & (THREADS - 1)); i0 < stop; i0 += AHEAD * THREADS) {
        i32x4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          v[k] = load_piece<T, false>(z + r.piece_class(i < stop ? i : i0));
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int i = i0 + k * THREADS;
          if (i < stop && piece_max<T>(v[k]) >= least) {
#pragma unroll
            for (int j = 0; j < N; ++j) visit(element<T>(v[k], j), r.piece_class(i) + j);
          }
        }
      }
    };
    const uint32_t cut = top.cut;
    const u64 from = (u64)cut << 32;
    if constexpr (HELD > 0) {
      PieceList& list = lists[t >> 6];
      const float least = cut_value(cut);
      if (t < 64) {   // (read again: it would wait in a register all the time)
        const int c = r.edge(t);
        const u64 key = c >= 0 ? rank_key((float)z[c], c) : 0;
        put_candidate(key != 0 && key >= from, key, top);
      }
      int count = 0;
      const int pieces = anew(r.pieces);
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const bool has = k * THREADS + t < pieces && maxima.get(k, x[k]) >= least;
        const u64 who = __ballot(has);
        if (who) {
          const int at = count + __builtin_amdgcn_mbcnt_hi(
              (uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
          if (has && at < 64) {
            list.data[at] = x[k];
            list.first[at] = r.piece_class(k * THREADS + t);
          }
          count += __popcll(who);
        }
      }
      if (count <= 64)
        put_pieces<T>(count, from, list, top);
      else if ((t & 63) == 0)
        atomicAdd(&top.n, CANDS + 1);   // more than this wave's list holds: search_top
    } else {
      // every thread goes through those of its own segments that have a large class
      auto put = [&](float v, int c) {
        const u64 k = rank_key(v, c);
        if (k >= from) {
          const int at = atomicAdd(&top.n, 1);
          if (at < CANDS) top.cand[at] = k;
        }
      };
      const float least = cut_value(cut);
      if (r.edge(t) >= 0) put((float)z[r.edge(t)], r.edge(t));
      uint32_t has = 0;
#pragma unroll
      for (int s = 0; s < SEGMENTS; ++s)
        has |= (uint32_t)(segments[s * THREADS + t] >= least) << s;
      while (has) {
        const int s = __builtin_ctz(has);
        has &= has - 1;
        for (int n = 0; n < segment_rounds; ++n) {
          const int i0 = t + (s * segment_rounds + n) * AHEAD * THREADS;
          if (i0 >= r.pieces) break;
          i32x4 v[AHEAD];
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k * THREADS;
            v[k] = load_piece<T, false>(z + r.piece_class(i < r.pieces ? i : i0));
          }
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k * THREADS;
            if (i < r.pieces && piece_max<T>(v[k]) >= least) {
#pragma unroll
              for (int j = 0; j < N; ++j) put(element<T>(v[k], j), r.piece_class(i) + j);
            }
          }
        }
      }
    }
    __syncthreads();
    if (top.n > CANDS) search_top<THREADS>(K, a.classes, each, top);
    put_top<THREADS>(K, [&](int place, float v, int c) {
      a.top_lp[row * K + place] = (v - p.m) * a.itau - log_s;
      a.top_ids[row * K + place] = c;
    }, top);
  }
}

// 256 threads where they hold a row (of 8009 bf16 classes, 64 largest: 85 us for 16384 rows) and
// have groups enough, else 1024 (the 128 largest of those: 142 us, by 1024 threads twice that; 256:
// 464).  Rows of 17000 bf16 classes give 1024 threads two of their eight pieces each, and take 65 us
// for 8192 (4.3 TB/s); workgroups between the two, or of less than 256, were not tried.
template <class T, bool TOP, bool PAST>
static void launch_rows(hipStream_t stream, const LogProbArgs& a) {
  const int pieces = a.classes / Piece<T>::N;   // at most
  const dim3 rows((unsigned)a.rows);
  if (pieces <= 256 * 8 && a.top <= 128)
    hipLaunchKernelGGL((log_prob_row<T, 256, 8, TOP, PAST>), rows, dim3(256), 0, stream, a);
  else if (pieces <= 1024 * 8)
    hipLaunchKernelGGL((log_prob_row<T, 1024, 8, TOP, PAST>), rows, dim3(1024), 0, stream, a);
  else
    hipLaunchKernelGGL((log_prob_row<T, 1024, 0, TOP, PAST>), rows, dim3(1024), 0, stream, a);
}
template <class T>
static void launch_log_probs(hipStream_t stream, const LogProbArgs& a) {
  // (the gradient's launch comes next, and finds a part of the logits still in the cache: both 206
  // instead of 232 us for 4096 bf16 rows of 50257, 432 instead of 454 for 8192)
  if (!a.stats && past_caches<T>(a.rows, a.classes))
    a.top ? launch_rows<T, true, true>(stream, a) : launch_rows<T, false, true>(stream, a);
  else
    a.top ? launch_rows<T, true, false>(stream, a) : launch_rows<T, false, false>(stream, a);
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
// Bound by the memory: 4096 bf16 rows of 50257 take 134 us (823 MB, 6.1 TB/s).
template <class T, bool PAST>
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
  i32x4 x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = i0 + k * THREADS;
    if (r.pieces) x[k] = load_piece<T, PAST>(z + r.piece_class(i < r.pieces ? i : 0));
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
  const bool known = !a.glp || (y >= 0 && y < a.classes);
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
    for (int j = 0; j < N; ++j) d[j] = (T)grad(element<T>(x[k], j));
    if (i < r.pieces)
      store_piece<T, PAST>(dz + r.piece_class(i), __builtin_bit_cast(i32x4, d));
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
  const dim3 grid((unsigned)a.rows, (unsigned)(whole ? ceil_div(whole, 1024) : 1));
  if (past_caches<T>(a.rows, a.classes))
    hipLaunchKernelGGL((log_prob_grad<T, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((log_prob_grad<T, false>), grid, dim3(256), 0, stream, a);
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
  a.none = no_class(ignore_index, classes);
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
  if (dlogits == logits) {   // the listed classes' are read again
    set_error("dmh_log_probs_grad: the gradient cannot take the logits' place");
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
