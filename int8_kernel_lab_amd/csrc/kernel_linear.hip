// The product of an int8 linear layer, dense or by expert:
//   y[m][n] = act(x[m] . w[n] * xs[m] * ws[n] + bias[n]) [* gated half] + residual[m][n]
// on v_mfma_i32_32x32x32_i8 (rows of x are the MFMA's rows, channels its
// columns; mfma32_tile.hpp), int32 sums exact for k < 2^17.
//
// Persistent workgroups over BM x BN tiles; 128-byte k-stages of the weight
// and activation rows come by LDS-DMA into two stage buffers, as in
// kernel_gemm32.hip.  Gated layers: a wave's first blocks of channels are gate
// rows of w and its last ones the rows `n` further, the other halves of the
// same outputs, so a lane holds both.
//
// By expert: the rows are sorted by expert and `offsets` says where each
// expert's begin; it is read on the device, so the host never waits for it.  A
// tile lies inside one expert's rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"
#include "mfma32_tile.hpp"

namespace i8conv {
namespace {

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void barrier_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 4 x 4 transpose of floats over the lanes of a quad.
__device__ __forceinline__ v4f quad_transpose_f(v4f v, int lane) {
  return __builtin_bit_cast(v4f, quad_transpose4(__builtin_bit_cast(v4i, v), lane));
}

// BM rows x BN rows of w over WM x WN waves.
template <int BM, int BN, int WM, int WN, int kOcc, bool kGated, bool kExperts>
__global__ __launch_bounds__(64 * WM * WN, kOcc) void linear_kernel(LinearArgs a, int tiles_m_max) {
  constexpr int P = kStageBytes, KS = P / 32, RPC = 1024 / P;
  constexpr int kWaves = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  constexpr int FO = kGated ? FN / 2 : FN;      // output blocks of 32 channels per wave
  constexpr int BO = kGated ? BN / 2 : BN;      // output channels per tile
  constexpr int kTile = (BM + BN) * P;
  constexpr int CPW = (BM + BN) / RPC / kWaves, CPA = BN / RPC / kWaves, CPB = CPW - CPA;
  static_assert(CPA >= 1 && CPB >= 1 && BN % (RPC * kWaves) == 0 && kWaves % 4 == 0, "tile shape");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const uint32_t lds0 = lds_addr(smem);
  const int stages = (a.k + P - 1) / P;
  const int tiles_n = (a.n + BO - 1) / BO;
  int *const first = reinterpret_cast<int *>(smem + 2 * kTile);  // by expert: its first row tile

  int tiles_m = tiles_m_max;
  if constexpr (kExperts) {
    // first[e] = row tiles of the experts before e (one wave, 64 at a time)
    if (wave == 0) {
      int total = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int count = 0;
        if (e < a.experts) count = (max(0, a.offsets[e + 1] - a.offsets[e]) + BM - 1) / BM;
        int sum = count;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int up = __shfl_up(sum, d);
          sum += lane >= d ? up : 0;
        }
        if (e < a.experts) first[e] = total + sum - count;
        total += __shfl(sum, 63);
      }
      if (lane == 0) first[a.experts] = total;
    }
    __syncthreads();
    tiles_m = min(tiles_m_max, first[a.experts]);
  }
  const TileRun run = xcd_tile_run(tiles_m * tiles_n, int(gridDim.x), int(blockIdx.x));

  const int crow = lane / (P / 16);
  const int lk = 16 * ((lane % (P / 16)) ^ swz32_f(wave * RPC + crow));
  const int frow = lane & 31, ff = swz32_f(frow);
  int koff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = frow * P + 16 * ((2 * ks + (lane >> 5)) ^ ff);
  const int abuf = wn * TN * P, bbuf = (BN + wm * TM) * P;

  for (int t = run.first; t < run.last; t += run.step) {
    const int tm = t / tiles_n, n0 = (t % tiles_n) * BO;
    int row0 = tm * BM, row_end = a.rows, expert = 0;
    if constexpr (kExperts) {
      int lo = 0, hi = a.experts;  // the last e with first[e] <= tm
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= tm)
          lo = mid;
        else
          hi = mid;
      }
      expert = __builtin_amdgcn_readfirstlane(lo);
      row0 = __builtin_amdgcn_readfirstlane(a.offsets[expert] + (tm - first[expert]) * BM);
      row_end = __builtin_amdgcn_readfirstlane(min(a.offsets[expert + 1], a.rows));
      if (row0 < 0 || row0 >= row_end) continue;  // offsets that are no offsets
    }
    const int rows = min(BM, row_end - row0);

    // rows of w and x that this lane copies: byte offsets from the tile's bases
    const bool gather = kExperts && a.sources != nullptr;
    const int8_t *const wbase = a.w + int64_t(expert) * a.wide * a.k;
    const v4u wd = make_desc(wbase, uint32_t(a.wide) * uint32_t(a.k));
    const int8_t *const xbase =
        static_cast<const int8_t *>(a.x) + (gather ? 0 : int64_t(row0) * a.ldx);
    const v4u xd = make_desc(xbase, gather ? uint32_t(int64_t(a.x_rows - 1) * a.ldx + a.k)
                                           : uint32_t((rows - 1) * uint32_t(a.ldx) + a.k));
    uint32_t aoff[CPA], boff[CPB];
#pragma unroll
    for (int j = 0; j < CPA; ++j) {
      const int lr = (wave + kWaves * j) * RPC + crow;
      const int w_of = lr / TN, b = lr % TN / 32, q = lr % 32;
      const int ch = n0 + w_of * (32 * FO) + (kGated ? b % FO : b) * 32 + q;
      const uint32_t r = uint32_t(ch) + (kGated && b >= FO ? uint32_t(a.n) : 0u);
      aoff[j] = ch < a.n ? r * uint32_t(a.k) + uint32_t(lk) : kOutOfRange;
    }
#pragma unroll
    for (int j = 0; j < CPB; ++j) {
      const int m = (wave + kWaves * j) * RPC + crow;
      uint32_t r = uint32_t(m);
      bool ok = m < rows;
      if (gather && ok) {
        r = uint32_t(a.sources[row0 + m]);
        ok = r < uint32_t(a.x_rows);
      }
      boff[j] = ok ? r * uint32_t(a.ldx) + uint32_t(lk) : kOutOfRange;
    }
    auto copy_stage = [&](int s) {
      const uint32_t buf = lds0 + uint32_t((s & 1) * kTile);
      const bool live = lk < a.k - s * P;
#pragma unroll
      for (int j = 0; j < CPW; ++j) {
        const uint32_t off = (j < CPA ? aoff[j] : boff[j - CPA]);
        lds_copy16(j < CPA ? wd : xd, buf + uint32_t(wave + kWaves * j) * 1024u,
                   live && off != kOutOfRange ? off + uint32_t(s * P) : kOutOfRange);
      }
    };

    barrier_lds();  // every wave has read the last tile's stages
    copy_stage(0);
    if (stages > 1) copy_stage(1);

    v16i acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    for (int s = 0; s < stages; ++s) {
      if (s + 1 < stages)
        wait_vm<CPW>();
      else
        wait_vm<0>();
      barrier_lds();
      const int8_t *const buf = smem + (s & 1) * kTile;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        v4i fa[FN], fb[FM];
#pragma unroll
        for (int i = 0; i < FN; ++i)
          fa[i] = *reinterpret_cast<const v4i *>(buf + koff[ks] + abuf + 32 * P * i);
#pragma unroll
        for (int j = 0; j < FM; ++j)
          fb[j] = *reinterpret_cast<const v4i *>(buf + koff[ks] + bbuf + 32 * P * j);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FM; ++j) acc[i][j] = mfma32(fb[j], fa[i], acc[i][j]);
      }
      if (s + 2 < stages) {
        barrier_lds();
        copy_stage(s + 2);
      }
    }

    // lane: channel lane % 32 of rows 8 g + 4 (lane / 32) + e of each block
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < FO; ++i) {
      const int c0 = n0 + wn * (32 * FO) + 32 * i, ch = c0 + (lane & 31);
      if (c0 >= a.n) break;
      const bool ok = ch < a.n;
      const int64_t p = int64_t(expert) * a.wide + (ok ? ch : 0);
      const float ws = a.ws[p], bias = a.bias ? a.bias[p] : 0.0f;
      const float ws2 = kGated ? a.ws[p + a.n] : 0.0f;
      const float bias2 = kGated && a.bias ? a.bias[p + a.n] : 0.0f;
#pragma unroll
      for (int j = 0; j < FM; ++j) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int r = wm * TM + 32 * j + 8 * g + 4 * half;
          float v[4], u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float xs = 0.0f;
            if (r + e < rows) {
              int src = row0 + r + e;
              if (gather) src = a.sources[src];
              xs = uint32_t(src) < uint32_t(a.x_rows) ? a.xs[src] : 0.0f;
            }
            v[e] = fmaf(float(acc[i][j][4 * g + e]) * xs, ws, bias);
            if constexpr (kGated)
              u[e] = fmaf(float(acc[FO + i][j][4 * g + e]) * xs, ws2, bias2);
          }
          activate(v, a.activation);
          if constexpr (kGated) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= u[e];
          }
          if (a.vec) {
            v4f o = quad_transpose_f(v4f{v[0], v[1], v[2], v[3]}, lane);
            const int m = r + (lane & 3), c = c0 + (lane & 28);
            if (m < rows && c < a.n) {
              if (a.residual) o += load_values4(a.residual, int64_t(row0 + m) * a.ldr + c, a.out_type);
              store_values4(a.y, int64_t(row0 + m) * a.ldy + c, a.out_type, o);
            }
          } else if (ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (r + e >= rows) break;
              float o = v[e];
              if (a.residual) o += load_value(a.residual, int64_t(row0 + r + e) * a.ldr + ch, a.out_type);
              store_value(a.y, int64_t(row0 + r + e) * a.ldy + ch, a.out_type, o);
            }
          }
        }
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int kOcc, int kGroups, bool kGated, bool kExperts>
int launch_tile(const LinearArgs &a, hipStream_t s) {
  auto kern = linear_kernel<BM, BN, WM, WN, kOcc, kGated, kExperts>;
  const size_t lds = 2 * size_t(BM + BN) * kStageBytes + (kExperts ? size_t(a.experts + 1) * 4 : 0);
  constexpr int BO = kGated ? BN / 2 : BN;
  // by expert: every group may end in a part of a tile
  int64_t tiles_m = (int64_t(a.rows) + BM - 1) / BM;
  if (kExperts) tiles_m = int64_t(a.rows) / BM + std::min(a.experts, a.rows);
  const int64_t tiles = tiles_m * ((int64_t(a.n) + BO - 1) / BO);
  static LdsLimit limit;
  if (const int rc = limit.raise(kern, lds); rc != I8CONV_OK) return rc;
  I8_LAUNCH(kern, dim3(unsigned(std::min<int64_t>(tiles, 256 * kGroups))), dim3(64 * WM * WN), lds, s,
            a, int(tiles_m));
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string("linear kernel launch: ") + hipGetErrorString(e));
    return I8CONV_HIP_ERROR;
  }
  return I8CONV_OK;
}

template <bool kGated, bool kExperts>
int launch_any(const LinearArgs &a, hipStream_t s) {
  return launch_tile<128, 128, 2, 2, 2, 2, kGated, kExperts>(a, s);
}

}  // namespace

int launch_linear_tiles(const LinearArgs &a, bool gated, void *stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.experts > 0) return gated ? launch_any<true, true>(a, s) : launch_any<false, true>(a, s);
  return gated ? launch_any<true, false>(a, s) : launch_any<false, false>(a, s);
}

}  // namespace i8conv
