// Rows of floating-point activations to int8 codes and one scale per row, the
// step before an int8 linear layer:
//   a = max |x[k]|,  code[k] = rint(127 x[k] / a) (half to even),  scale = a / 127.
// A row whose largest magnitude is below 2^-100 gives zeros and scale 0; a row
// that holds an infinity or NaN gives zeros and scale NaN, so that everything
// computed from it is NaN.
#include <hip/hip_runtime.h>

#include <string>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"
#include "quantize_tile.hpp"

namespace i8conv {
namespace {

// A workgroup per row; the row is read twice, the second time from the caches.
template <int TYPE, bool kVec>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void *x, int64_t ldx, int k,
                                                            int8_t *codes, float *scales) {
  const int64_t row = blockIdx.x;
  __shared__ uint32_t tops[kThreads / 64];
  uint32_t top = 0;
  for (int i = int(threadIdx.x) * 8; i < k; i += kThreads * 8) {
    float v[8];
    load8<TYPE, kVec>(x, row * ldx + i, v);
    top = max(top, top8(v));
  }
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) top = max(top, tops[i]);
  const RowStep step = row_step(top);
  if (threadIdx.x == 0) scales[row] = step.scale;
  for (int i = int(threadIdx.x) * 8; i < k; i += kThreads * 8) {
    float v[8];
    load8<TYPE, kVec>(x, row * ldx + i, v);
    *reinterpret_cast<v2u *>(codes + row * k + i) = codes8(v, step);
  }
}

template <int TYPE>
void launch_type(const void *x, int64_t ldx, int rows, int k, bool vec, int8_t *codes,
                 float *scales, hipStream_t s) {
  if (vec)
    I8_LAUNCH((quantize_kernel<TYPE, true>), dim3(rows), dim3(kThreads), 0, s, x, ldx, k, codes,
              scales);
  else
    I8_LAUNCH((quantize_kernel<TYPE, false>), dim3(rows), dim3(kThreads), 0, s, x, ldx, k, codes,
              scales);
}

}  // namespace

int launch_quantize(const void *x, int type, int64_t ldx, int rows, int k, int8_t *codes,
                    float *scales, void *stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int per16 = 16 / type_size(type);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx % per16 == 0;
  if (type == I8CONV_BF16)
    launch_type<I8CONV_BF16>(x, ldx, rows, k, vec, codes, scales, s);
  else if (type == I8CONV_FP16)
    launch_type<I8CONV_FP16>(x, ldx, rows, k, vec, codes, scales, s);
  else
    launch_type<I8CONV_FP32>(x, ldx, rows, k, vec, codes, scales, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string("quantize launch: ") + hipGetErrorString(e));
    return I8CONV_HIP_ERROR;
  }
  return I8CONV_OK;
}

}  // namespace i8conv
