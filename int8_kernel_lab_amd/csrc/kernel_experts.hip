// What stands before and after the products of a layer of experts: the stable
// sort of the tokens' choices by expert, and each token's weighted sum of its
// experts' rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"

namespace i8conv {
namespace {

// A workgroup per expert e.  It reads all ids twice: first each wave counts, in
// its part of them, those of experts before e and those of e; then it gives
// e's their rows in order.  Workgroup 0 does what belongs to no expert as well:
// the places of dropped choices, and the sources past the last row.
constexpr int kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;
__global__ __launch_bounds__(kRouteThreads) void route_kernel(const int32_t *ids, int count,
                                                              int choices, int experts,
                                                              int32_t *offsets, int32_t *sources,
                                                              int32_t *places) {
  __shared__ int less_of[kRouteWaves], mine_of[kRouteWaves], all_of[kRouteWaves];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = ((count + kRouteWaves - 1) / kRouteWaves + 63) / 64 * 64;
  const int begin = min(count, wave * part), end = min(count, begin + part);
  int less = 0, mine = 0, all = 0;
  for (int i = begin + lane; i < end; i += 64) {
    const int id = ids[i];
    less += id >= 0 && id < e;
    mine += id == e;
    all += id >= 0 && id < experts;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    less += __shfl_xor(less, d);
    mine += __shfl_xor(mine, d);
    all += __shfl_xor(all, d);
  }
  if (lane == 0) less_of[wave] = less, mine_of[wave] = mine, all_of[wave] = all;
  __syncthreads();
  int base = 0, next = 0, total = 0;
  for (int w = 0; w < kRouteWaves; ++w) {
    base += less_of[w];
    if (w < wave) next += mine_of[w];
    total += all_of[w];
  }
  if (threadIdx.x == 0) {
    offsets[e] = base;
    if (e == 0) offsets[experts] = total;
  }
  next += base;
  for (int i0 = begin; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const int id = i < end ? ids[i] : e;
    const bool hit = i < end && id == e;
    const uint64_t hits = __ballot(hit);
    if (hit) {
      const int row = next + __popcll(hits & ((uint64_t(1) << lane) - 1));
      places[i] = row;
      sources[row] = i / choices;
    }
    if (e == 0 && (id < 0 || id >= experts)) places[i] = -1;
    next += __popcll(hits);
  }
  if (e == 0)
    for (int i = total + int(threadIdx.x); i < count; i += kRouteThreads) sources[i] = -1;
}

// A workgroup per token and 1024 outputs, four outputs a thread.
__global__ __launch_bounds__(kThreads) void combine_kernel(const void *x, const int32_t *places,
                                                           const float *weights,
                                                           const void *residual, void *y,
                                                           int choices, int n, int rows,
                                                           int in_type, int out_type, int vec) {
  const int64_t t = blockIdx.x;
  const int c0 = (int(blockIdx.y) * kThreads + int(threadIdx.x)) * 4;
  if (c0 >= n) return;
  const int live = min(4, n - c0);
  v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = 0; c < choices; ++c) {
    const int row = places[t * choices + c];
    if (row < 0 || row >= rows) continue;
    const float wt = weights[t * choices + c];
    const int64_t at = int64_t(row) * n + c0;
    if (vec) {
      const v4f v = load_values4(x, at, in_type);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(wt, v[e], sum[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < live) sum[e] = fmaf(wt, load_value(x, at + e, in_type), sum[e]);
    }
  }
  const int64_t at = t * n + c0;
  if (vec) {
    if (residual) sum += load_values4(residual, at, out_type);
    store_values4(y, at, out_type, sum);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < live)
        store_value(y, at + e, out_type,
                    residual ? sum[e] + load_value(residual, at + e, out_type) : sum[e]);
  }
}

int done(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return I8CONV_OK;
  set_error(std::string(what) + ": " + hipGetErrorString(e));
  return I8CONV_HIP_ERROR;
}

}  // namespace

int launch_route(const int32_t *ids, int tokens, int choices, int experts, int32_t *offsets,
                 int32_t *sources, int32_t *places, void *stream) {
  I8_LAUNCH(route_kernel, dim3(unsigned(experts)), dim3(kRouteThreads), 0,
            static_cast<hipStream_t>(stream), ids, tokens * choices, choices, experts, offsets,
            sources, places);
  return done("route launch");
}

int launch_combine(const void *x, int in_type, const int32_t *places, const float *weights,
                   const void *residual, void *y, int out_type, int tokens, int choices, int n,
                   void *stream) {
  const bool vec = linear_vec_ok(x, n, n, type_size(in_type), 4) &&
                   linear_vec_ok(y, n, n, type_size(out_type), 4) &&
                   (!residual || linear_vec_ok(residual, n, n, type_size(out_type), 4));
  const unsigned parts = unsigned((n + 4 * kThreads - 1) / (4 * kThreads));
  I8_LAUNCH(combine_kernel, dim3(unsigned(tokens), parts), dim3(kThreads), 0,
            static_cast<hipStream_t>(stream), x, places, weights, residual, y, choices, n,
            tokens * choices, in_type, out_type, int(vec));
  return done("combine launch");
}

}  // namespace i8conv
