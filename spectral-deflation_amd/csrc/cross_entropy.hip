// Cross entropy over the classes of a vocabulary, with its gradient.
//
//   lse  = log sum exp z
//   loss = lse - (1 - eps) z_y - eps mean(z) + zeta lse^2
//   dz   = (p (1 + 2 zeta lse) - (1 - eps) delta_y - eps / V) * g,     p = exp(z - lse)
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
  float* lse;            // per row, written (forward) or read (gradient); may be null in the
                         // forward pass
  const float* count;    // rows that have a target, or null
  const float* gout;     // gradient of the loss (gradient kernel): one, or one a row
  long long rows, zs, ds, ignore;
  int classes, t64, gout_rows;
  float eps, zeta, gscale;
};

// The sum of one value a thread over a workgroup, the same in every thread.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  constexpr int W = THREADS / 64;
  if (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) s += lds[w];
  return s;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  constexpr int W = THREADS / 64;
  if (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) s = fmaxf(s, lds[w]);
  return s;
}

// The number of rows that have a target.
__global__ __launch_bounds__(1024) void xent_count(const void* targets, int t64, long long rows,
                                                   long long ignore, float* count) {
  __shared__ float lds[16];
  int n = 0;
  for (long long i = threadIdx.x; i < rows; i += 1024)
    n += load_index(targets, t64, i) != ignore;
  // exact: a thread's and a workgroup's counts stay far below 2^24 up to 2^24 rows, and are
  // off by their last place beyond
  const float s = block_sum<1024>((float)n, lds);
  if (threadIdx.x == 0) *count = s;
}

// The sum of the rows' losses, divided by the count for a mean.
__global__ __launch_bounds__(1024) void xent_reduce(const float* row_loss, long long rows,
                                                    const float* count, float* loss) {
  __shared__ float lds[16];
  float s = 0.f;
  for (long long i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
  s = block_sum<1024>(s, lds);
  if (threadIdx.x == 0) *loss = count ? s / *count : s;
}

// One workgroup a row: maximum, sum and gradient, a sweep each.
template <class T, bool GRAD>
__global__ __launch_bounds__(256) void xent_row(XentArgs a) {
  __shared__ float lds[4];
  const long long row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = GRAD ? (T*)a.dz + row * a.ds : nullptr;
  const long long y = load_index(a.targets, a.t64, row);
  const int v = a.classes;
  if (y == a.ignore) {
    if (threadIdx.x == 0) {
      a.row_loss[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    if (GRAD)
      for (int c = threadIdx.x; c < v; c += 256) dz[c] = (T)0.f;
    return;
  }
  float m = -__builtin_inff(), zsum = 0.f;
  for (int c = threadIdx.x; c < v; c += 256) {
    const float x = (float)z[c];
    m = fmaxf(m, x);
    zsum += x;
  }
  m = block_max<256>(m, lds);
  float s = 0.f;
  for (int c = threadIdx.x; c < v; c += 256) s += exp2f(((float)z[c] - m) * LOG2E);
  s = block_sum<256>(s, lds);
  if (a.eps != 0.f) zsum = block_sum<256>(zsum, lds);
  const float lse = m + log2f(s) * LN2;
  const bool known = y >= 0 && y < v;
  const float zy = known ? (float)z[y] : __builtin_nanf("");
  if (threadIdx.x == 0) {
    float loss = lse - (1.f - a.eps) * zy;
    if (a.eps != 0.f) loss -= a.eps * (zsum / v);
    if (a.zeta != 0.f) loss += a.zeta * lse * lse;
    a.row_loss[row] = loss;
    if (a.lse) a.lse[row] = lse;
  }
  if (GRAD) {
    float g = a.gscale;
    if (a.count) g /= *a.count;
    if (!known) g = __builtin_nanf("");
    const float ps = g * (1.f + 2.f * a.zeta * lse) / s, base = -g * (a.eps / v);
    const float top = -g * (1.f - a.eps);
    __syncthreads();   // z[y] is read before dz, which may be z, is written
    for (int c = threadIdx.x; c < v; c += 256) {
      float d = fmaf(exp2f(((float)z[c] - m) * LOG2E), ps, base);
      if (c == (int)y) d += top;
      dz[c] = (T)d;
    }
  }
}

// The gradient from a forward pass's lse: element by element.
template <class T>
__global__ __launch_bounds__(256) void xent_grad(XentArgs a) {
  const long long row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.zs;
  T* dz = (T*)a.dz + row * a.ds;
  const long long y = load_index(a.targets, a.t64, row);
  const int v = a.classes;
  const bool live = y != a.ignore, known = y >= 0 && y < v;
  const float lse = a.lse[row];
  float g = a.gout[a.gout_rows ? row : 0];
  if (a.count) g /= *a.count;
  if (!known) g = __builtin_nanf("");
  const float ps = g * (1.f + 2.f * a.zeta * lse), base = -g * (a.eps / v);
  const float top = -g * (1.f - a.eps);
  for (int c = threadIdx.x; c < v; c += 256) {
    float d = fmaf(exp2f(((float)z[c] - lse) * LOG2E), ps, base);
    if (c == (int)y) d += top;
    dz[c] = (T)(live ? d : 0.f);
  }
}

static bool xent_shape(long long rows, long long classes) {
  return rows >= 0 && rows < (1LL << 23) && classes >= 1 && classes < (1LL << 31) - 65536;
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

int dmh_cross_entropy(hipStream_t stream, const void* logits, int dtype, long long rows,
                      long long classes, long long z_rstride, const void* targets,
                      int targets_64, long long ignore_index, float smoothing, float z_loss,
                      int reduction, float grad_scale, float* loss, float* count, float* lse,
                      void* dlogits, long long d_rstride, void* ws, size_t ws_bytes) {
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
  if (reduction == RED_MEAN) {
    hipLaunchKernelGGL(xent_count, dim3(1), dim3(1024), 0, stream, targets, targets_64 != 0, rows,
                       ignore_index, count);
    DMH_CHECK_LAUNCH("xent_count");
  }
  XentArgs a{};
  a.z = logits;
  a.targets = targets;
  a.dz = dlogits;
  a.row_loss = reduction == RED_NONE ? loss : (float*)ws;
  a.lse = lse;
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
  if (rows > 0) {
    const dim3 grid((unsigned)rows), block(256);
    if (dlogits) {
      DMH_FOR_TYPE(dtype, T, hipLaunchKernelGGL((xent_row<T, true>), grid, block, 0, stream, a))
    } else {
      DMH_FOR_TYPE(dtype, T, hipLaunchKernelGGL((xent_row<T, false>), grid, block, 0, stream, a))
    }
    DMH_CHECK_LAUNCH("xent_row");
  }
  if (reduction != RED_NONE) {
    hipLaunchKernelGGL(xent_reduce, dim3(1), dim3(1024), 0, stream, (const float*)ws, rows,
                       (const float*)a.count, loss);
    DMH_CHECK_LAUNCH("xent_reduce");
  }
  return DMH_OK;
}

int dmh_cross_entropy_grad(hipStream_t stream, const void* logits, int dtype, long long rows,
                           long long classes, long long z_rstride, const void* targets,
                           int targets_64, long long ignore_index, float smoothing, float z_loss,
                           const float* lse, const float* count, const float* grad_out,
                           int grad_out_rows, void* dlogits, long long d_rstride) {
  if (!xent_shape(rows, classes) || z_rstride < 0 || d_rstride < 0 || !float_code(dtype)) {
    set_error("dmh_cross_entropy_grad: bad arguments (rows=%lld classes=%lld dtype=%d)", rows,
              classes, dtype);
    return DMH_EINVAL;
  }
  if (rows == 0) return DMH_OK;
  if (!logits || !targets || !lse || !grad_out || !dlogits) {
    set_error("dmh_cross_entropy_grad: null tensor");
    return DMH_EINVAL;
  }
  XentArgs a{};
  a.z = logits;
  a.targets = targets;
  a.dz = dlogits;
  a.lse = (float*)lse;
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
  DMH_FOR_TYPE(dtype, T, hipLaunchKernelGGL((xent_grad<T>), dim3((unsigned)rows), dim3(256), 0,
                                            stream, a))
  DMH_CHECK_LAUNCH("xent_grad");
  return DMH_OK;
}

}  // extern "C"
