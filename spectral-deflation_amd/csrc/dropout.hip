// Dropout from a counter-based generator, with the residual's addition.
//
//   y[e] = residual[e] + (draw(e) >= cut ? x[e] * scale : 0)
//
// The mask is a function of (seed, offset, e) alone (train_ops.h), so nothing is stored for the
// backward pass: it is the same call on the gradient, without the residual.
#include "train_ops.h"

namespace dmh {

struct DropArgs {
  const void* x;
  const void* res;
  void* out;
  long long numel, cols, xs, rs;   // rows of `cols` elements, strides of x and the residual
  Rng rng;
};

// Bound by the memory: 27.4 us for 8192 x 5120 bf16 (168 MB, 6.1 TB/s), 17.4 us for 8192 x 1280
// bf16 added to an fp32 residual (105 MB, 6.0 TB/s); the generator keeps the vector units busy for
// 64% of the former.
//
// One block of eight flat elements a thread: one evaluation of the generator.  FLAT: x and the
// residual are contiguous; otherwise a block finds its row by a division and takes its elements
// one by one where a row ends inside it: 11.5 us for 8192 rows of 1280 bf16 columns out of 2560,
// 12.7 for 1281 out of 1283, where contiguous rows take 10.4.
template <class TX, class TO, bool RES, bool FLAT>
__global__ __launch_bounds__(256) void dropout(DropArgs a) {
  const TX* x = (const TX*)a.x;
  const TO* res = (const TO*)a.res;
  TO* out = (TO*)a.out;
  const RngKey key = rng_key(a.rng);
  const long long step = (long long)gridDim.x * 256;
  for (long long b = (long long)blockIdx.x * 256 + threadIdx.x; b * 8 < a.numel; b += step) {
    const long long e = b * 8;
    const int n = a.numel - e < 8 ? (int)(a.numel - e) : 8;
    float v[8], r[8];
    if (FLAT && n == 8) {
      load8(x + e, v);
      if (RES) load8(res + e, r);
    } else if (FLAT) {
      load_some(x + e, n, v);
      if (RES) load_some(res + e, n, r);
    } else {
      long long row = e / a.cols, col = e - row * a.cols;
      if (n == 8 && col + 8 <= a.cols) {
        load8(x + row * a.xs + col, v);
        if (RES) load8(res + row * a.rs + col, r);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = j < n ? (float)x[row * a.xs + col] : 0.f;
          if (RES) r[j] = j < n ? (float)res[row * a.rs + col] : 0.f;
          if (++col == a.cols) {
            col = 0;
            ++row;
          }
        }
      }
    }
    const uint32_t bits = a.rng.cut ? keep_bits(a.rng, key, (unsigned long long)b) : ~0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = kept(bits, j, v[j] * a.rng.scale);
      if (RES) v[j] += r[j];
    }
    if (n == 8)
      store8(out + e, v);
    else
      store_some(out + e, n, v);
  }
}

template <class TX, class TO>
static void launch_dropout(hipStream_t stream, const DropArgs& a) {
  // one block of eight elements a thread up to 2^30 threads
  const long long groups = (a.numel + 2047) / 2048;
  const dim3 grid((unsigned)(groups < (1 << 22) ? groups : (1 << 22))), block(256);
  const bool flat = a.xs == a.cols && (!a.res || a.rs == a.cols);
  if (a.res && flat)
    hipLaunchKernelGGL((dropout<TX, TO, true, true>), grid, block, 0, stream, a);
  else if (a.res)
    hipLaunchKernelGGL((dropout<TX, TO, true, false>), grid, block, 0, stream, a);
  else if (flat)
    hipLaunchKernelGGL((dropout<TX, TO, false, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((dropout<TX, TO, false, false>), grid, block, 0, stream, a);
}

}  // namespace dmh

using namespace dmh;

extern "C" int dmh_dropout(hipStream_t stream, const void* x, int x_dtype, long long rows,
                           long long cols, long long x_rstride, const void* residual,
                           long long res_rstride, void* out, int out_dtype, int cut,
                           unsigned long long seed, unsigned long long offset,
                           const void* rng_state) {
  if (rows < 0 || cols < 0 || x_rstride < 0 || res_rstride < 0 || !float_code(x_dtype) ||
      !float_code(out_dtype) || cut < 0 || cut > 65536) {
    set_error("dmh_dropout: bad arguments (rows=%lld cols=%lld dtypes=%d,%d cut=%d)", rows, cols,
              x_dtype, out_dtype, cut);
    return DMH_EINVAL;
  }
  if (rows == 0 || cols == 0) return DMH_OK;
  if (!x || !out) {
    set_error("dmh_dropout: null tensor");
    return DMH_EINVAL;
  }
  if (rows > (1LL << 60) / cols) {
    set_error("dmh_dropout: %lld x %lld elements are too many", rows, cols);
    return DMH_EINVAL;
  }
  DropArgs a;
  a.x = x;
  a.res = residual;
  a.out = out;
  a.numel = rows * cols;
  a.cols = cols;
  a.xs = rows == 1 ? cols : x_rstride;
  a.rs = rows == 1 ? cols : res_rstride;
  a.rng = make_rng(seed, offset, rng_state, cut);
  DMH_FOR_TYPE(x_dtype, TX, DMH_FOR_TYPE(out_dtype, TO, (launch_dropout<TX, TO>(stream, a))))
  DMH_CHECK_LAUNCH("dropout");
  return DMH_OK;
}
