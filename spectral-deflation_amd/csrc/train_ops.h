// Shared pieces of the training operators (dropout, embedding, cross entropy): their element
// types, eight-element accesses and the counter-based generator.
#pragma once

#include "common.h"

namespace dmh {

typedef _Float16 fp16;

// dtype codes of the C entries
enum { DMH_F32 = 0, DMH_BF16 = 1, DMH_F16 = 2 };
inline bool float_code(int d) { return d == DMH_F32 || d == DMH_BF16 || d == DMH_F16; }

// A 16-byte piece of a tensor.  Its address may have the element's alignment only: rows of an
// odd width start anywhere, and global accesses of this size need no more on amdhsa (the
// unaligned access mode).
template <class T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// eight consecutive elements, as they are in memory
template <class T>
struct Raw8 {
  typename Piece<T>::type p[8 / Piece<T>::N];
  __device__ __forceinline__ void load(const T* at) {
#pragma unroll
    for (int k = 0; k < 8 / Piece<T>::N; ++k)
      p[k] = *(const typename Piece<T>::type*)(at + k * Piece<T>::N);
  }
  __device__ __forceinline__ float operator[](int j) const {
    return (float)p[j / Piece<T>::N][j % Piece<T>::N];
  }
};

// ... and as fp32
template <class T>
__device__ __forceinline__ void load8(const T* at, float (&v)[8]) {
  Raw8<T> x;
  x.load(at);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x[j];
}

// back, each rounded to nearest even
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  constexpr int N = Piece<T>::N;
#pragma unroll
  for (int k = 0; k < 8 / N; ++k) {
    typename Piece<T>::type x;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (T)v[k * N + j];
    *(typename Piece<T>::type*)(p + k * N) = x;
  }
}

// the first `n` of eight elements (n < 8: a row's end)
template <class T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
}
template <class T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) p[j] = (T)v[j];
}

// ids, positions and targets: int32 or int64
__device__ __forceinline__ long long load_index(const void* p, int is64, long long i) {
  return is64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// ---- dropout ------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): a 128-bit counter through ten rounds of two 32 x 32 -> 64 bit products under a
// 64-bit key.  Eight 16-bit draws a block: element e of the tensor (flat index) takes half
// (e & 1) of word (e >> 1) & 3 of block e >> 3.  16 bits fix p to 1/65536, which the scale
// takes into account exactly, and halve the integer work, which with 32 bits a draw would
// take longer than moving 16-bit data does.
struct Rng {
  unsigned long long seed, offset;
  const unsigned long long* state;   // {seed, offset} in device memory instead, or null
  unsigned cut;                      // dropped if draw < cut: 0 (none) .. 65536 (all)
  float scale;                       // 65536 / (65536 - cut); 0 where all are dropped
};

inline Rng make_rng(unsigned long long seed, unsigned long long offset, const void* state,
                    int cut) {
  Rng r;
  r.seed = seed;
  r.offset = offset;
  r.state = (const unsigned long long*)state;
  r.cut = (unsigned)cut;
  r.scale = cut < 65536 ? (float)(65536.0 / (65536 - cut)) : 0.f;
  return r;
}

// the key and the counter's upper half, once a thread
struct RngKey {
  uint32_t k0, k1, c2, c3;
};
__device__ __forceinline__ RngKey rng_key(const Rng& r) {
  unsigned long long s = r.seed, o = r.offset;
  if (r.state) {
    s = r.state[0];
    o = r.state[1];
  }
  return {(uint32_t)s, (uint32_t)(s >> 32), (uint32_t)o, (uint32_t)(o >> 32)};
}

__device__ __forceinline__ void philox(const RngKey& key, unsigned long long block,
                                       uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.c2, c3 = key.c3;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u;
    const unsigned long long b = (unsigned long long)c2 * 0xCD9E8D57u;
    // (x ^ y ^ z in one instruction)
    c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), c1, k0, 0x96);
    c1 = (uint32_t)b;
    c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), c3, k1, 0x96);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// The kept elements of a block as bits: element j has bit (j >> 1) + 16 (j & 1), that is, its
// word's number in the half that its draw comes from: two packed 16-bit instructions a word
// and three to join them, where a comparison for each draw takes twice as many.  cut >= 1.
__device__ __forceinline__ uint32_t keep_bits(const Rng& r, const RngKey& key,
                                              unsigned long long block) {
  uint32_t w[4], m = 0;
  philox(key, block, w);
  const uint32_t least = (r.cut - 1) * 0x10001u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // draw - (cut - 1), not below zero, is positive where the element is kept
    uint32_t t;
    asm("v_pk_sub_u16 %0, %1, %2 clamp" : "=v"(t) : "v"(w[k]), "s"(least));
    asm("v_pk_min_u16 %0, %1, %2" : "=v"(t) : "v"(t), "s"(0x10001u));
    m |= t << k;
  }
  return m;
}

// ... of the eight elements from flat index e on.  SPLIT: e may lie inside a block, and the next
// one has the rest.
template <bool SPLIT>
__device__ __forceinline__ uint32_t keep_bits_at(const Rng& r, const RngKey& key,
                                                 unsigned long long e) {
  uint32_t m = keep_bits(r, key, e >> 3);
  if (SPLIT) {
    m |= keep_bits(r, key, (e >> 3) + 1) << 4;   // the halves' bits of 16 elements
    const int t = (int)(e & 7) >> 1;
    const uint32_t even = m >> t, odd = (m >> 16 >> t & 15) | (m >> (t + 1) & 15) << 16;
    m = e & 1 ? odd : even & 0x000F000Fu;
  }
  return m;
}

// x where element j is kept, else zero: what is dropped is replaced, not multiplied, so an
// infinity or NaN there leaves nothing behind
__device__ __forceinline__ float kept(uint32_t bits, int j, float x) {
  const int all = (int)(bits << (31 - (j >> 1) - 16 * (j & 1))) >> 31;
  return __builtin_bit_cast(float, all & __builtin_bit_cast(int, x));
}

}  // namespace dmh

// a call for one of the three element types
#define DMH_FOR_TYPE(code, T, ...)      \
  switch (code) {                       \
    case dmh::DMH_F32: {                \
      using T = float;                  \
      __VA_ARGS__;                      \
      break;                            \
    }                                   \
    case dmh::DMH_BF16: {               \
      using T = dmh_bf16_t;             \
      __VA_ARGS__;                      \
      break;                            \
    }                                   \
    default: {                          \
      using T = dmh::fp16;              \
      __VA_ARGS__;                      \
      break;                            \
    }                                   \
  }
typedef bf16 dmh_bf16_t;
