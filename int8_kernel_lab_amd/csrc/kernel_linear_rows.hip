// Int8 linear layers of few rows: every weight is read once and multiplied
// with all rows, so the time is the weights' way from memory.
//
// A workgroup takes 16 output channels (gated: 16 of each half); its eight
// waves split the reduction and add their sums up through LDS.  On
// v_mfma_i32_16x16x64_i8 with the channels as its rows: lane l loads 16 bytes
// of channel l % 16 straight from memory into the operand, a batch of k-steps
// at a time and the next one before the first is used, and ends with four
// consecutive channels of row l % 16.
//
// The rows come as codes, from memory like the weights (kDirect), or as floating-point
// values that the workgroup quantizes itself into LDS (kFused), while its first
// weights are on the way: every workgroup does that work again, but a launch
// and the codes' way through memory are saved.
//
// By expert: a workgroup row (blockIdx.y) takes the y-th of the experts that
// have rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"
#include "quantize_tile.hpp"

namespace i8conv {
namespace {

constexpr int kRowsWaves = 8, kRowsThreads = 64 * kRowsWaves;
constexpr int kFusedChunks = 4;  // 8-value pieces of x a thread holds
constexpr int kFusedLds = 256;   // bytes of their largest values and the rows' scales
static_assert(kFusedChunks * (kRowsWaves + 1) * 4 <= kFusedLds, "fits");

// Bytes between rows of codes in LDS: 16-byte units in a step of 2 x odd, so
// that a fragment read (16 rows, two chunks per 32 lanes) has no bank conflicts.
__host__ __device__ inline int fused_pitch(int k) {
  const int units = k / 16;
  return 16 * (units + ((2 - units % 4) + 4) % 4);
}

// The y-th expert with rows, and those rows; false if there are fewer.
struct Group {
  int expert, begin, end;
};
__device__ __forceinline__ bool find_group(const int32_t *offsets, int experts, int rows, int y,
                                           int lane, Group *g) {
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < experts) lo = offsets[e], hi = min(offsets[e + 1], rows);
    const uint64_t live = __ballot(lo >= 0 && lo < hi);
    const int count = __popcll(live);
    if (y < count) {
      const bool mine = (live >> lane & 1) && __popcll(live & ((uint64_t(1) << lane) - 1)) == y;
      const int at = __ffsll((unsigned long long)__ballot(mine)) - 1;
      g->expert = e0 + at;
      g->begin = __shfl(lo, at);
      g->end = __shfl(hi, at);
      return true;
    }
    y -= count;
  }
  return false;
}

// MF: fragments of 16 rows taken together; U: k-steps of 64 bytes per batch.
template <bool kGated, bool kExperts, bool kFused, int MF, int U>
__global__ __launch_bounds__(kRowsThreads, 2) void linear_rows_kernel(LinearArgs a) {
  constexpr int F = kGated ? 2 : 1;
  // LDS: the waves' sums; kFused: the pieces' largest values, the rows' scales
  // and their codes [step_rows][pitch]
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  v4i(*const sums)[F * MF][64] = reinterpret_cast<v4i(*)[F * MF][64]>(smem);
  int8_t *const extra = smem + sizeof(v4i) * kRowsWaves * F * MF * 64;
  uint32_t(*const tops)[kRowsWaves] = reinterpret_cast<uint32_t(*)[kRowsWaves]>(extra);
  float *const row_scale = reinterpret_cast<float *>(extra + kFusedChunks * kRowsWaves * 4);
  int8_t *const codes = extra + kFusedLds;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Group group = {0, 0, a.rows};
  if constexpr (kExperts) {
    if (!find_group(a.offsets, a.experts, a.rows, int(blockIdx.y), lane, &group)) return;
    group.expert = __builtin_amdgcn_readfirstlane(group.expert);
    group.begin = __builtin_amdgcn_readfirstlane(group.begin);
    group.end = __builtin_amdgcn_readfirstlane(group.end);
  }
  const bool gather = kExperts && a.sources != nullptr;
  const int q = lane & 15, kq = 16 * (lane >> 4);
  const int c0 = int(blockIdx.x) * 16;

  // this wave's part of the reduction
  const int steps = (a.k + 63) / 64, per = (steps + kRowsWaves - 1) / kRowsWaves;
  const int k0 = wave * per * 64, k1 = min(a.k, k0 + per * 64);

  const auto wr = make_rsrc(a.w + int64_t(group.expert) * a.wide * a.k, uint32_t(a.wide) * uint32_t(a.k));
  uint32_t woff[F];
#pragma unroll
  for (int f = 0; f < F; ++f)
    woff[f] = c0 + q < a.n ? uint32_t(c0 + q + (f ? a.n : 0)) * uint32_t(a.k) + uint32_t(kq) : kOutOfRange;
  auto load_w = [&](v4i (&wv)[U][F], int k) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const bool ok = k + 64 * u + kq < k1 && woff[f] != kOutOfRange;
        wv[u][f] = load16(wr, ok ? woff[f] + uint32_t(k + 64 * u) : kOutOfRange);
      }
  };

  const int pitch = fused_pitch(a.k);
  // rows of x per pass
  const int chunks = (a.k + 8 * kRowsThreads - 1) / (8 * kRowsThreads);
  const int step_rows = kFused ? kFusedChunks / chunks : 16 * MF;
  for (int row0 = group.begin; row0 < group.end; row0 += step_rows) {
    const int rows = min(step_rows, group.end - row0);

    // kDirect: this lane's row of each fragment
    uint32_t xoff[MF];
    const int8_t *const xbase =
        static_cast<const int8_t *>(a.x) + (gather || kFused ? 0 : int64_t(row0) * a.ldx);
    const auto xr = make_rsrc(xbase, kFused ? 0u
                                     : gather ? uint32_t(int64_t(a.x_rows - 1) * a.ldx + a.k)
                                              : uint32_t((rows - 1) * uint32_t(a.ldx) + a.k));
    if constexpr (!kFused) {
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        uint32_t r = uint32_t(16 * m + q);
        bool ok = int(r) < rows;
        if (gather && ok) {
          r = uint32_t(a.sources[row0 + int(r)]);
          ok = r < uint32_t(a.x_rows);
        }
        xoff[m] = ok ? r * uint32_t(a.ldx) + uint32_t(kq) : kOutOfRange;
      }
    }

    v4i acc[F][MF];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int m = 0; m < MF; ++m) acc[f][m] = v4i{0, 0, 0, 0};

    v4i wv[2][U][F], xv[2][U][MF];
    auto load_x = [&](v4i (&dst)[U][MF], int k) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          const bool ok = k + 64 * u + kq < k1;
          if constexpr (kFused)
            dst[u][m] = ok ? *reinterpret_cast<const v4i *>(codes + min(q, rows - 1) * pitch + k + 64 * u + kq)
                           : v4i{0, 0, 0, 0};
          else
            dst[u][m] = load16(xr, ok && xoff[m] != kOutOfRange ? xoff[m] + uint32_t(k + 64 * u)
                                                               : kOutOfRange);
        }
    };
    auto multiply = [&](const v4i (&w)[U][F], const v4i (&x)[U][MF]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int m = 0; m < MF; ++m) acc[f][m] = mfma16(w[u][f], x[u][m], acc[f][m]);
    };

    if constexpr (kFused) {
      // the values first, then the first weights: loads return in order
      v4f v[kFusedChunks][2];
      const int piece = int(threadIdx.x) * 8;
      auto read = [&](auto type) {
        int r = 0, c = 0;  // piece i is piece c of row r
#pragma unroll
        for (int i = 0; i < kFusedChunks; ++i, ++c) {
          if (c == chunks) c = 0, ++r;
          const int k = piece + c * 8 * kRowsThreads;
          float t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (r < rows && k < a.k) {
            int64_t src = row0 + r;
            if (gather) src = a.sources[src];
            if (uint64_t(src) < uint64_t(a.x_rows)) load8<decltype(type)::value, true>(a.x, src * a.ldx + k, t);
          }
          v[i][0] = v4f{t[0], t[1], t[2], t[3]};
          v[i][1] = v4f{t[4], t[5], t[6], t[7]};
        }
      };
      if (a.x_type == I8CONV_BF16)
        read(std::integral_constant<int, I8CONV_BF16>{});
      else if (a.x_type == I8CONV_FP16)
        read(std::integral_constant<int, I8CONV_FP16>{});
      else
        read(std::integral_constant<int, I8CONV_FP32>{});
      load_w(wv[0], k0);
      auto piece_of = [&](int i, float (&t)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = v[i][e / 4][e % 4];
      };
#pragma unroll
      for (int i = 0; i < kFusedChunks; ++i) {
        float t[8];
        piece_of(i, t);
        const uint32_t top = wave_max(top8(t));
        if (lane == 0) tops[i][wave] = top;
      }
      __syncthreads();
      int r = 0, c = 0;
#pragma unroll
      for (int i = 0; i < kFusedChunks; ++i, ++c) {
        if (c == chunks) c = 0, ++r;
        const int k = piece + c * 8 * kRowsThreads;
        if (r >= rows) break;
        uint32_t top = 0;
        for (int j = 0; j < chunks; ++j)
#pragma unroll
          for (int w = 0; w < kRowsWaves; ++w) top = max(top, tops[r * chunks + j][w]);
        const RowStep step = row_step(top);
        if (threadIdx.x == 0) row_scale[r] = step.scale;
        float t[8];
        piece_of(i, t);
        if (k < a.k) *reinterpret_cast<v2u *>(codes + r * pitch + k) = codes8(t, step);
      }
      __syncthreads();
      load_x(xv[0], k0);
    } else {
      load_w(wv[0], k0);
      load_x(xv[0], k0);
    }
    for (int k = k0; k < k1; k += 128 * U) {
      if (k + 64 * U < k1) {
        load_w(wv[1], k + 64 * U);
        load_x(xv[1], k + 64 * U);
      }
      multiply(wv[0], xv[0]);
      if (k + 64 * U >= k1) break;
      if (k + 128 * U < k1) {
        load_w(wv[0], k + 128 * U);
        load_x(xv[0], k + 128 * U);
      }
      multiply(wv[1], xv[1]);
    }

#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int m = 0; m < MF; ++m) sums[wave][f * MF + m][lane] = acc[f][m];
    __syncthreads();
    if (wave < MF) {
      const int m = wave, r = 16 * m + q, ch = c0 + 4 * (lane >> 4);
      v4i s[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        s[f] = sums[0][f * MF + m][lane];
#pragma unroll
        for (int w = 1; w < kRowsWaves; ++w) s[f] += sums[w][f * MF + m][lane];
      }
      if (r < rows && ch < a.n) {
        float xs;
        if constexpr (kFused) {
          xs = row_scale[r];
        } else {
          const int src = gather ? a.sources[row0 + r] : row0 + r;
          xs = uint32_t(src) < uint32_t(a.x_rows) ? a.xs[src] : 0.0f;
        }
        float v[4], u[4];
        const int64_t p = int64_t(group.expert) * a.wide + ch;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = ch + e < a.n;
          v[e] = fmaf(float(s[0][e]) * xs, ok ? a.ws[p + e] : 0.0f, ok && a.bias ? a.bias[p + e] : 0.0f);
          if constexpr (kGated)
            u[e] = fmaf(float(s[F - 1][e]) * xs, ok ? a.ws[p + a.n + e] : 0.0f,
                        ok && a.bias ? a.bias[p + a.n + e] : 0.0f);
        }
        activate(v, a.activation);
        if constexpr (kGated) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= u[e];
        }
        const int64_t row = row0 + r;
        if (a.vec4) {
          v4f o = {v[0], v[1], v[2], v[3]};
          if (a.residual) o += load_values4(a.residual, row * a.ldr + ch, a.out_type);
          store_values4(a.y, row * a.ldy + ch, a.out_type, o);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (ch + e >= a.n) break;
            float o = v[e];
            if (a.residual) o += load_value(a.residual, row * a.ldr + ch + e, a.out_type);
            store_value(a.y, row * a.ldy + ch + e, a.out_type, o);
          }
        }
      }
    }
    if (row0 + step_rows < group.end) __syncthreads();  // sums and codes are read
  }
}

template <bool kGated, bool kExperts, bool kFused, int MF, int U>
int launch_rows(const LinearArgs &a, hipStream_t s) {
  auto kern = linear_rows_kernel<kGated, kExperts, kFused, MF, U>;
  const size_t lds = size_t(kRowsWaves) * (kGated ? 2 : 1) * MF * 1024 +
                     (kFused ? kFusedLds + size_t(fused_rows(a.k)) * fused_pitch(a.k) : 0);
  static LdsLimit limit;
  if (const int rc = limit.raise(kern, lds); rc != I8CONV_OK) return rc;
  const dim3 grid(unsigned((a.n + 15) / 16), unsigned(kExperts ? std::min(a.experts, a.rows) : 1));
  I8_LAUNCH(kern, grid, dim3(kRowsThreads), lds, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string("linear rows kernel launch: ") + hipGetErrorString(e));
    return I8CONV_HIP_ERROR;
  }
  return I8CONV_OK;
}

template <bool kGated, bool kExperts>
int launch_any(const LinearArgs &a, bool fused, hipStream_t s) {
  if (fused) return launch_rows<kGated, kExperts, true, 1, 8>(a, s);
  if (kExperts || a.rows <= 16) return launch_rows<kGated, kExperts, false, 1, 8>(a, s);
  if (a.rows <= 32) return launch_rows<kGated, kExperts, false, 2, 4>(a, s);
  return launch_rows<kGated, kExperts, false, 4, 4>(a, s);
}

}  // namespace

// Rows that a workgroup quantizes itself at a time.
int fused_rows(int k) {
  const int chunks = (k + 8 * kRowsThreads - 1) / (8 * kRowsThreads);
  return chunks > kFusedChunks ? 0 : kFusedChunks / chunks;
}

int launch_linear_rows(const LinearArgs &a, bool gated, bool fused, void *stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.experts > 0) return gated ? launch_any<true, true>(a, fused, s) : launch_any<false, true>(a, fused, s);
  return gated ? launch_any<true, false>(a, fused, s) : launch_any<false, false>(a, fused, s);
}

}  // namespace i8conv
