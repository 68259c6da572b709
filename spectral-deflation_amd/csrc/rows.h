// Rows of logits: the reductions, the exponentials and the pieces that the operators over the
// classes of a vocabulary share.
#pragma once

#include <type_traits>

#include "train_ops.h"

namespace dmh {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

constexpr float INF = __builtin_inff();

typedef int i32x4 __attribute__((ext_vector_type(4)));

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

// The same in units of 2: s = sum 2^((z - m) c2), c2 = log2(e) / temperature.
__device__ __forceinline__ void rescale(Part& p, float m, float c2) {
  if (p.m != m) {   // never for two of -inf
    p.s *= __builtin_amdgcn_exp2f((p.m - m) * c2);
    p.m = m;
  }
}

// ---- reductions by lane shifts: in the last lane of a row of 16, then of the wave --------------
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float shifted(float v, float none) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                         CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float lane(float v, int i) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}
// (a NaN goes on)
__device__ __forceinline__ float maximum(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}
__device__ __forceinline__ float row16_max(float v) {
  v = maximum(v, shifted<0x111>(v, -INF));
  v = maximum(v, shifted<0x112>(v, -INF));
  v = maximum(v, shifted<0x114>(v, -INF));
  return maximum(v, shifted<0x118>(v, -INF));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += shifted<0x111>(v, 0.f);
  v += shifted<0x112>(v, 0.f);
  v += shifted<0x114>(v, 0.f);
  return v + shifted<0x118>(v, 0.f);
}
__device__ __forceinline__ float wave_max(float v) {
  v = row16_max(v);
  v = maximum(v, shifted<0x142, 0xA>(v, -INF));
  return lane(maximum(v, shifted<0x143, 0xC>(v, -INF)), 63);
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row16_sum(v);
  v += shifted<0x142, 0xA>(v, 0.f);
  return lane(v + shifted<0x143, 0xC>(v, 0.f), 63);
}
// Of the first `waves` waves' values in LDS, behind a barrier, by every wave alike.
__device__ __forceinline__ float waves_max(const float* lds, int waves) {
  const int i = threadIdx.x & 15;
  return lane(row16_max(i < waves ? lds[i] : -INF), 15);
}
__device__ __forceinline__ float waves_sum(const float* lds, int waves) {
  const int i = threadIdx.x & 15;
  return lane(row16_sum(i < waves ? lds[i] : 0.f), 15);
}

// What stands for no class in lists of classes: ignore_index, unless that is a class.
inline long long no_class(long long ignore, long long classes) {
  return ignore < 0 || ignore >= classes ? ignore : -100;
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

// Logits of much more than the last-level cache's 256 MB are read, and their gradient written, as
// what no cache need keep.  Bf16 rows of 50257, a distilled step with the rest, us a pass through the
// caches and by them, logits from memory:
//   rows                      2000 (191 MiB)  3000       3800 (364 MiB)  4300       8192
//   step                      91, 87          128, 123   158, 151        176, 169   322, 307
//   ... in place              77, 76          140, 111   178, 141        201, 161   390, 304
//   loss alone                47, 48          66, 66     80, 81          91, 91     164, 165
// Below the switch it is the caches that may still hold the logits: 46 instead of 48 us for a step of
// 1024 rows that they hold, 43 instead of 46 for the losses of 2000.
template <class T>
inline bool past_caches(long long rows, long long classes) {
  return rows * classes * (long long)sizeof(T) >= 384LL << 20;
}
// A piece of a row; with PAST as one that the caches need not keep.
template <class T, bool PAST>
__device__ __forceinline__ i32x4 load_piece(const T* at) {
  typedef typename Piece<T>::type type;
  return __builtin_bit_cast(i32x4, PAST ? __builtin_nontemporal_load((const type*)at)
                                        : *(const type*)at);
}
template <class T, bool PAST>
__device__ __forceinline__ void store_piece(T* at, i32x4 x) {
  typedef typename Piece<T>::type type;
  if (PAST)
    __builtin_nontemporal_store(__builtin_bit_cast(type, x), (type*)at);
  else
    *(type*)at = __builtin_bit_cast(type, x);
}

// Element j of a piece.  bf16 by its bits: from converted values the compiler makes 16-bit maxima,
// which it then has to convert back and forth.
template <class T>
__device__ __forceinline__ float element(i32x4 x, int j) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_bit_cast(float, j & 1 ? x[j / 2] & (int)0xFFFF0000u : x[j / 2] << 16);
  else
    return (float)__builtin_bit_cast(typename Piece<T>::type, x)[j];
}
// The largest of a piece, or a NaN.  (Packed 16-bit integers would take one and a half instructions
// for two elements in place of three, and took 4% longer for the whole row.)
template <class T>
__device__ __forceinline__ float piece_max(i32x4 x) {
  float m = element<T>(x, 0);
#pragma unroll
  for (int j = 1; j < Piece<T>::N; ++j) m = maximum(m, element<T>(x, j));
  return m;
}

// Marks of listed classes in LDS: a byte for each of `count` pieces from `first` on, a bit for each
// class of a piece, and (edges) a word for the classes before and behind the pieces, bit t that of
// the class of thread t.  False where class c has no mark here.
template <class T>
__device__ __forceinline__ bool find_mark(const Row<T>& r, int c, int first, int count, bool edges,
                                          uint32_t* marks, uint32_t* edge, uint32_t*& word,
                                          uint32_t& bit) {
  const int i = (c - r.head) / Row<T>::N;
  if (c < r.head || i >= r.pieces) {
    word = edge;
    bit = 1u << (c < r.head ? c : 8 + c - r.piece_class(r.pieces));
    return edges;
  }
  const int q = i - first;
  word = marks + (q >> 2);
  bit = 1u << ((q & 3) * 8 + (c - r.head) % Row<T>::N);
  return q >= 0 && q < count;
}

// A row that stays packed in registers between the steps: what one has unpacked may not stay there
// for the next.
template <int HELD>
__device__ __forceinline__ void repack(i32x4 (&x)[HELD]) {
#pragma unroll
  for (int k = 0; k < HELD; ++k) asm volatile("" : "+v"(x[k]));
}

// The same number, which the compiler takes for another: what is compared with it is compared where it
// is needed.  The comparisons of a thread's eight pieces with their number, kept from the loads to the
// end, are 16 scalar registers; those that did not fit cost rows with a top up to 6%.
__device__ __forceinline__ int anew(int uniform) {
  asm volatile("" : "+s"(uniform));
  return uniform;
}

}  // namespace dmh
