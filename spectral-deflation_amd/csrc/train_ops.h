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

// eight consecutive elements as fp32
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  constexpr int N = Piece<T>::N;
#pragma unroll
  for (int k = 0; k < 8 / N; ++k) {
    const typename Piece<T>::type x = *(const typename Piece<T>::type*)(p + k * N);
#pragma unroll
    for (int j = 0; j < N; ++j) v[k * N + j] = (float)x[j];
  }
}

// ... and back, each rounded to nearest even
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
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// dropout of the eight elements of one block: what is dropped is replaced, not multiplied, so
// an infinity or NaN there leaves nothing behind
__device__ __forceinline__ void drop_block(const Rng& r, const RngKey& key,
                                           unsigned long long block, float (&v)[8]) {
  uint32_t w[4];
  philox(key, block, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t draw = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
    v[j] = draw >= r.cut ? v[j] * r.scale : 0.f;
  }
}

// ... of eight elements from flat index e on, which two blocks may hold
__device__ __forceinline__ void drop_at(const Rng& r, const RngKey& key, unsigned long long e,
                                        float (&v)[8]) {
  const int skip = (int)(e & 7);
  if (skip == 0) {
    drop_block(r, key, e >> 3, v);
    return;
  }
  uint32_t keep = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
    philox(key, (e >> 3) + h, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t draw = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
      keep |= (draw >= r.cut ? 1u : 0u) << (8 * h + j);
    }
  }
  keep >>= skip;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (keep >> j & 1) ? v[j] * r.scale : 0.f;
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
