// Rows of floating-point activations to int8 codes and one scale per row, the
// step before an int8 linear layer:
//   a = max |x[k]|,  code[k] = rint(127 x[k] / a) (half to even),  scale = a / 127.
// A row whose largest magnitude is below 2^-100 gives zeros and scale 0; a row
// that holds an infinity or NaN gives zeros and scale NaN, so that everything
// computed from it is NaN.
//
// Bound by memory: a row is read once and stays in registers between its
// largest value and its codes (rows too long for that are read again, from the
// caches).  A wave takes a row to itself where there are many of them, with
// nothing to wait for but its own loads; few rows are spread over a workgroup
// each.  16384 x 8192 bf16: 74 us, 5.4 TB/s of reading and writing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"
#include "quantize_tile.hpp"

namespace i8conv {
namespace {

// TPR threads to a row (a wave or the workgroup), NV pieces of eight values in
// each one's registers.
template <int TYPE, bool kVec, int TPR, int NV>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void *x, int64_t ldx, int64_t rows,
                                                            int k, int8_t *codes, float *scales) {
  constexpr int kRows = kThreads / TPR;
  __shared__ uint32_t tops[2][kThreads / 64];
  const int t = int(threadIdx.x) % TPR;
  int parity = 0;
  for (int64_t row = int64_t(blockIdx.x) * kRows + int(threadIdx.x) / TPR; row < rows;
       row += int64_t(gridDim.x) * kRows, parity ^= 1) {
    float v[NV][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (i * TPR + t) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
      if (at < k) load8<TYPE, kVec>(x, row * ldx + at, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, top8(v[i]));
    for (int at = (NV * TPR + t) * 8; at < k; at += TPR * 8) {
      float w[8];
      load8<TYPE, kVec>(x, row * ldx + at, w);
      top = max(top, top8(w));
    }
    top = wave_max(top);
    if constexpr (TPR > 64) {
      // (two sets in turn: a wave may be a row ahead of another's reads)
      if ((threadIdx.x & 63) == 0) tops[parity][threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i) top = max(top, tops[parity][i]);
    }
    const RowStep step = row_step(top);
    if (t == 0) scales[row] = step.scale;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (i * TPR + t) * 8;
      if (at < k) *reinterpret_cast<v2u *>(codes + row * k + at) = codes8(v[i], step);
    }
    for (int at = (NV * TPR + t) * 8; at < k; at += TPR * 8) {
      float w[8];
      load8<TYPE, kVec>(x, row * ldx + at, w);
      *reinterpret_cast<v2u *>(codes + row * k + at) = codes8(w, step);
    }
  }
}

template <int TYPE, bool kVec, int TPR, int NV>
void launch_form(const void *x, int64_t ldx, int rows, int k, int8_t *codes, float *scales,
                 hipStream_t s) {
  constexpr int kRows = kThreads / TPR;
  const unsigned blocks = unsigned(std::min<int64_t>((int64_t(rows) + kRows - 1) / kRows, 1 << 22));
  I8_LAUNCH((quantize_kernel<TYPE, kVec, TPR, NV>), dim3(blocks), dim3(kThreads), 0, s, x, ldx,
            int64_t(rows), k, codes, scales);
}

template <int TYPE>
void launch_type(const void *x, int64_t ldx, int rows, int k, bool vec, int8_t *codes,
                 float *scales, hipStream_t s) {
  if (!vec) {
    launch_form<TYPE, false, kThreads, 1>(x, ldx, rows, k, codes, scales, s);
    return;
  }
  // A wave to a row where there are many and its registers hold it: bf16, us with
  // a wave and with a workgroup, 512 x 1024 2.9 and 3.0, 1024 x 1024 3.0 and 3.2,
  // 32768 x 1024 17.9 and 31.9; 1024 x 2048 3.7 and 3.4, 2048 x 2048 4.2 and 4.7,
  // 4096 x 2048 5.6 and 7.1.
  if (rows >= 512 && k <= 64 * 8 * 2) {
    launch_form<TYPE, true, 64, 2>(x, ldx, rows, k, codes, scales, s);
  } else if (rows >= 2048 && k <= 64 * 8 * 4) {
    launch_form<TYPE, true, 64, 4>(x, ldx, rows, k, codes, scales, s);
  } else if (k <= kThreads * 8) {
    launch_form<TYPE, true, kThreads, 1>(x, ldx, rows, k, codes, scales, s);
  } else if (k <= kThreads * 8 * 2) {
    launch_form<TYPE, true, kThreads, 2>(x, ldx, rows, k, codes, scales, s);
  } else {
    launch_form<TYPE, true, kThreads, 4>(x, ldx, rows, k, codes, scales, s);
  }
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
