// Embedding lookup with scaling, and its gradients by sorted tokens.
//
//   out[i, :]  = D(scale * W[id_i, :] + P[pos_i, :])
//   dW[v, :]  (+)= scale * sum over i with id_i = v of D(g)[i, :]
//   dP[t, :]  (+)= sum over i with pos_i = t of D(g)[i, :]
//
// D is dropout over the flat index i * dim + column (train_ops.h), evaluated again in the
// backward pass.  Sums are held in fp32 and taken in the order of the tokens: no atomics, the
// same gradient every time.  An id or position outside its table gives a row of NaN, and no
// gradient.
#include "train_ops.h"

namespace dmh {

struct EmbedArgs {
  const void* ids;
  const void* pos;        // positions, or null: i % seq
  const void* w;
  const void* p;          // position table, or null
  void* out;
  long long tokens, vocab, wstride, prows, pstride;
  int is64, seq, dim;
  float scale;
  Rng rng;
};

// Eight columns of one token a thread.
template <class TW, class TO, bool POS, bool DROP>
__global__ __launch_bounds__(256) void embed_rows(EmbedArgs a) {
  const int d8 = (a.dim + 7) / 8;
  const long long items = a.tokens * d8, step = (long long)gridDim.x * 256;
  const RngKey key = DROP ? rng_key(a.rng) : RngKey{};
  for (long long it = (long long)blockIdx.x * 256 + threadIdx.x; it < items; it += step) {
    const long long i = it / d8;
    const int c = (int)(it - i * d8) * 8, n = a.dim - c < 8 ? a.dim - c : 8;
    const long long id = load_index(a.ids, a.is64, i);
    const long long t = !POS ? 0 : a.pos ? load_index(a.pos, a.is64, i) : i % a.seq;
    float v[8];
    if ((unsigned long long)id < (unsigned long long)a.vocab &&
        (!POS || (unsigned long long)t < (unsigned long long)a.prows)) {
      const TW* w = (const TW*)a.w + id * a.wstride + c;
      if (n == 8) load8(w, v); else load_some(w, n, v);
      if (POS) {
        float p[8];
        const TW* pr = (const TW*)a.p + t * a.pstride + c;
        if (n == 8) load8(pr, p); else load_some(pr, n, p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], a.scale, p[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= a.scale;
      }
      if (DROP) drop_at(a.rng, key, (unsigned long long)(i * a.dim + c), v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_nanf("");
    }
    TO* o = (TO*)a.out + i * a.dim + c;
    if (n == 8) store8(o, v); else store_some(o, n, v);
  }
}

// ---- gradient -----------------------------------------------------------------------------
// The tokens in the order of (id, index): each token's place is the number of tokens before it
// in that order.  Ids that take no gradient (padding, outside the table) become `vocab`.
__device__ __forceinline__ int sort_key(const void* ids, int is64, long long i, long long vocab,
                                        long long padding) {
  const long long id = load_index(ids, is64, i);
  return (unsigned long long)id < (unsigned long long)vocab && id != padding ? (int)id
                                                                               : (int)vocab;
}

constexpr int RANK_TILE = 2048;

__global__ __launch_bounds__(256) void embed_rank(const void* ids, int is64, int tokens,
                                                  long long vocab, long long padding, int* keys,
                                                  int* order) {
  __shared__ int tile[RANK_TILE];
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int mine = i < tokens ? sort_key(ids, is64, i, vocab, padding) : 0;
  int before = 0;
  for (int t0 = 0; t0 < tokens; t0 += RANK_TILE) {
    const int n = tokens - t0 < RANK_TILE ? tokens - t0 : RANK_TILE;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += 256)
      tile[j] = sort_key(ids, is64, t0 + j, vocab, padding);
    __syncthreads();
    for (int j = 0; j < n; ++j)
      before += (tile[j] < mine) | ((tile[j] == mine) & (t0 + j < i));
  }
  if (i < tokens) {
    keys[before] = mine;
    order[before] = i;
  }
}

struct EmbedGradArgs {
  const int* keys;        // sorted; null for implicit positions (id_i = i % seq)
  const int* order;
  const void* g;
  void* out;
  long long rows, gstride;
  int tokens, seq, dim, accumulate;
  float scale;
  Rng rng;
};

// first place in the sorted keys that is not below v
__device__ __forceinline__ int first_at(const int* keys, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

constexpr int GRAD_ROWS = 16;   // table rows a workgroup

// A wave takes a row of the table and 512 of its columns, eight a lane.
template <class TG, class TO, bool DROP>
__global__ __launch_bounds__(256) void embed_grad(EmbedGradArgs a) {
  __shared__ int first[GRAD_ROWS + 1];
  const long long v0 = (long long)blockIdx.x * GRAD_ROWS;
  if (a.keys) {
    if (threadIdx.x <= GRAD_ROWS)
      first[threadIdx.x] = first_at(a.keys, a.tokens, (int)(v0 + threadIdx.x));
    __syncthreads();
  }
  const RngKey key = DROP ? rng_key(a.rng) : RngKey{};
  const int wave = threadIdx.x >> 6, c = (blockIdx.y * 64 + (threadIdx.x & 63)) * 8;
  if (c >= a.dim) return;
  const int n = a.dim - c < 8 ? a.dim - c : 8;
  for (int r = wave; r < GRAD_ROWS; r += 4) {
    const long long v = v0 + r;
    if (v >= a.rows) return;
    int s0, s1;
    if (a.keys) {
      s0 = first[r];
      s1 = first[r + 1];
    } else {   // tokens v, v + seq, ...
      s0 = 0;
      s1 = v < a.seq ? (a.tokens - (int)v + a.seq - 1) / a.seq : 0;
    }
    if (a.accumulate && s0 == s1) continue;
    float sum[8] = {};
    for (int s = s0; s < s1; ++s) {
      const long long i = a.keys ? a.order[s] : v + (long long)s * a.seq;
      float x[8];
      const TG* g = (const TG*)a.g + i * a.gstride + c;
      if (n == 8) load8(g, x); else load_some(g, n, x);
      if (DROP) drop_at(a.rng, key, (unsigned long long)(i * a.dim + c), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += x[j];
    }
    TO* o = (TO*)a.out + v * a.dim + c;
    float old[8] = {};
    if (a.accumulate) {
      if (n == 8) load8(o, old); else load_some(o, n, old);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = fmaf(sum[j], a.scale, old[j]);
    if (n == 8) store8(o, sum); else store_some(o, n, sum);
  }
}

template <class TW, class TO>
static void launch_rows(hipStream_t stream, const EmbedArgs& a) {
  const long long groups = (a.tokens * ((a.dim + 7) / 8) + 255) / 256;
  const dim3 grid((unsigned)(groups < (1 << 22) ? groups : (1 << 22))), block(256);
  if (a.p && a.rng.cut)
    hipLaunchKernelGGL((embed_rows<TW, TO, true, true>), grid, block, 0, stream, a);
  else if (a.p)
    hipLaunchKernelGGL((embed_rows<TW, TO, true, false>), grid, block, 0, stream, a);
  else if (a.rng.cut)
    hipLaunchKernelGGL((embed_rows<TW, TO, false, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((embed_rows<TW, TO, false, false>), grid, block, 0, stream, a);
}

template <class TG, class TO>
static void launch_grad(hipStream_t stream, const EmbedGradArgs& a) {
  const dim3 grid((unsigned)ceil_div(a.rows, GRAD_ROWS), ceil_div(a.dim, 512)), block(256);
  if (a.rng.cut)
    hipLaunchKernelGGL((embed_grad<TG, TO, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((embed_grad<TG, TO, false>), grid, block, 0, stream, a);
}

static bool grad_shape(long long tokens, long long rows, int dim) {
  return tokens >= 0 && tokens < (1LL << 31) - 65536 && rows >= 0 && rows < (1LL << 31) - 65536 &&
         dim >= 0 && dim <= 65535 * 512;
}

}  // namespace dmh

using namespace dmh;

extern "C" {

int dmh_embedding(hipStream_t stream, const void* ids, int ids_64, long long tokens, int seq,
                  const void* weight, int dtype, long long vocab, int dim, long long w_rstride,
                  const void* pos_weight, long long pos_rows, long long p_rstride,
                  const void* positions, float scale, int cut, unsigned long long seed,
                  unsigned long long offset, const void* rng_state, void* out, int out_dtype) {
  if (tokens < 0 || vocab < 0 || dim < 0 || w_rstride < 0 || pos_rows < 0 || p_rstride < 0 ||
      !float_code(dtype) || !float_code(out_dtype) || cut < 0 || cut > 65536 ||
      tokens > (1LL << 40) || vocab > (1LL << 40) ||
      (tokens > 0 && pos_weight && !positions && seq < 1)) {
    set_error("dmh_embedding: bad arguments (tokens=%lld seq=%d vocab=%lld dim=%d dtypes=%d,%d "
              "cut=%d)", tokens, seq, vocab, dim, dtype, out_dtype, cut);
    return DMH_EINVAL;
  }
  if (tokens == 0 || dim == 0) return DMH_OK;
  if (!ids || !out || (!weight && vocab)) {
    set_error("dmh_embedding: null tensor");
    return DMH_EINVAL;
  }
  EmbedArgs a;
  a.ids = ids;
  a.pos = positions;
  a.w = weight;
  a.p = pos_weight;
  a.out = out;
  a.tokens = tokens;
  a.vocab = vocab;
  a.wstride = w_rstride;
  a.prows = pos_rows;
  a.pstride = p_rstride;
  a.is64 = ids_64 != 0;
  a.seq = seq;
  a.dim = dim;
  a.scale = scale;
  a.rng = make_rng(seed, offset, rng_state, cut);
  DMH_FOR_TYPE(dtype, TW, DMH_FOR_TYPE(out_dtype, TO, (launch_rows<TW, TO>(stream, a))))
  DMH_CHECK_LAUNCH("embed_rows");
  return DMH_OK;
}

int dmh_embedding_grad_workspace_size(long long tokens, long long rows, int dim, size_t* bytes) {
  if (!bytes || !grad_shape(tokens, rows, dim)) {
    set_error("dmh_embedding_grad_workspace_size: bad arguments (tokens=%lld rows=%lld dim=%d)",
              tokens, rows, dim);
    return DMH_EINVAL;
  }
  *bytes = 8 * (size_t)tokens;
  return DMH_OK;
}

int dmh_embedding_grad(hipStream_t stream, const void* ids, int ids_64, long long tokens, int seq,
                       const void* grad, int dtype, long long g_rstride, long long rows, int dim,
                       long long padding_idx, float scale, int cut, unsigned long long seed,
                       unsigned long long offset, const void* rng_state, void* out,
                       int out_dtype, int accumulate, void* ws, size_t ws_bytes) {
  if (!grad_shape(tokens, rows, dim) || g_rstride < 0 || !float_code(dtype) ||
      !float_code(out_dtype) || cut < 0 || cut > 65536 || (!ids && tokens > 0 && seq < 1)) {
    set_error("dmh_embedding_grad: bad arguments (tokens=%lld seq=%d rows=%lld dim=%d "
              "dtypes=%d,%d cut=%d)", tokens, seq, rows, dim, dtype, out_dtype, cut);
    return DMH_EINVAL;
  }
  if (rows == 0 || dim == 0) return DMH_OK;
  if (!out || (tokens > 0 && !grad)) {
    set_error("dmh_embedding_grad: null tensor");
    return DMH_EINVAL;
  }
  size_t need;
  dmh_embedding_grad_workspace_size(tokens, rows, dim, &need);
  if (ids && need > 0 && (!ws || ws_bytes < need)) {
    set_error("dmh_embedding_grad: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return DMH_EWORKSPACE;
  }
  EmbedGradArgs a;
  a.keys = ids ? (const int*)ws : nullptr;
  a.order = ids ? (const int*)ws + tokens : nullptr;
  a.g = grad;
  a.out = out;
  a.rows = rows;
  a.gstride = g_rstride;
  a.tokens = (int)tokens;
  a.seq = seq < 1 ? 1 : seq;
  a.dim = dim;
  a.accumulate = accumulate != 0;
  a.scale = scale;
  a.rng = make_rng(seed, offset, rng_state, cut);
  if (ids && tokens > 0) {
    hipLaunchKernelGGL(embed_rank, dim3(ceil_div(tokens, 256)), dim3(256), 0, stream, ids,
                       ids_64 != 0, (int)tokens, rows, padding_idx, (int*)ws, (int*)ws + tokens);
    DMH_CHECK_LAUNCH("embed_rank");
  }
  DMH_FOR_TYPE(dtype, TG, DMH_FOR_TYPE(out_dtype, TO, (launch_grad<TG, TO>(stream, a))))
  DMH_CHECK_LAUNCH("embed_grad");
  return DMH_OK;
}

}  // extern "C"
