// The product of an int8 linear layer, dense or by expert:
//   y[m][n] = act(x[m] . w[n] * xs[m] * ws[n] + bias[n]) [* gated half] + residual[m][n]
// on v_mfma_i32_32x32x32_i8 (rows of x are the MFMA's rows, channels its
// columns; mfma32_tile.hpp), int32 sums exact for k < 2^17.
//
// Persistent workgroups over BM x BN tiles; 128-byte k-stages of the weight
// and activation rows come by LDS-DMA into R stage buffers, and fragments of
// the next k-step are read while the present one multiplies, as in
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
#include <type_traits>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"
#include "mfma32_tile.hpp"

namespace i8conv {
namespace {

template <int N>
using Set = std::integral_constant<int, N>;

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void barrier_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The value of the lane's neighbour (lane ^ 1).
__device__ __forceinline__ float neighbour(float v) {
  return bits_f32(uint32_t(__builtin_amdgcn_update_dpp(0, int(f32_bits(v)), 0xb1, 0xf, 0xf, false)));
}

// A descriptor of wave-uniform values, in scalar registers.
__device__ __forceinline__ v4u uniform_desc(const void *base, uint32_t bytes) {
  const v4u d = make_desc(base, bytes);
  return v4u{uint32_t(__builtin_amdgcn_readfirstlane(int(d[0]))),
             uint32_t(__builtin_amdgcn_readfirstlane(int(d[1]))),
             uint32_t(__builtin_amdgcn_readfirstlane(int(d[2]))), d[3]};
}

// Row tiles taken together: the workgroups of an XCD run walk kRowGroup row
// tiles before the next column tile, so that a round of them shares both its
// rows of x and its rows of w in the XCD's L2.
constexpr int kRowGroup = 8;

// BM rows x BN rows of w over WM x WN waves; KG groups of such waves, each with
// stage buffers of its own, take the k-stages in turn and add their sums up
// through LDS; fragments read GS k-steps of 32 bytes at a time.
template <int BM, int BN, int WM, int WN, int R, int KG, int GS, int kOcc, bool kGated, bool kExperts>
__global__ __launch_bounds__(64 * WM * WN * KG, kOcc) void linear_kernel(LinearArgs a) {
  constexpr int P = kStageBytes, KS = P / 32, RPC = 1024 / P;
  constexpr int kWaves = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  constexpr int FO = kGated ? FN / 2 : FN;  // output blocks of 32 channels per wave
  constexpr int BO = kGated ? BN / 2 : BN;  // output channels per tile
  constexpr int kTile = (BM + BN) * P;
  constexpr int CPW = (BM + BN) / RPC / kWaves, CPA = BN / RPC / kWaves, CPB = CPW - CPA;
  // Two blocks of a wave hold the even and the odd ones of 64 channels, so that
  // a lane has pairs of neighbours: a row's 64 outputs leave as whole lines.
  constexpr bool kPair = FO % 2 == 0;
  constexpr int kParams = 2 * BN + BM;  // floats: weight scales, biases, row scales
  static_assert(CPA >= 1 && CPB >= 1 && BN % (RPC * kWaves) == 0 && kWaves % 4 == 0, "tile shape");
  static_assert(!kGated || FN % 2 == 0, "both halves of an output in one wave");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];

  const int lane = threadIdx.x & 63;
  const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave_id / kWaves, wave = wave_id % kWaves;
  // (waves of different rows share a SIMD, so that one gains by the other's rest)
  const int wm = wave / WN, wn = wave % WN;
  int8_t *const bufs = smem + group * R * kTile;
  const uint32_t lds0 = lds_addr(bufs);
  float *const params = reinterpret_cast<float *>(smem + KG * R * kTile);  // two slots
  // by expert: its first row and its first row tile
  int *const begins = reinterpret_cast<int *>(params + 2 * kParams);
  int *const first = begins + a.experts + 1;
  // stages per group (the last ones may lie past the reduction: zeros)
  const int stages = (a.k + KG * P - 1) / (KG * P);
  const int tiles_n = (a.n + BO - 1) / BO;
  const bool gather = kExperts && a.sources != nullptr;

  int tiles_m = (a.rows + BM - 1) / BM;
  if constexpr (kExperts) {
    // first[e] = row tiles of the experts before e (one wave, 64 at a time)
    if (wave_id == 0) {
      int total = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int count = 0;
        if (e < a.experts) {
          const int begin = a.offsets[e], end = a.offsets[e + 1];
          count = min(max(0, end - begin), a.rows);
          count = count / BM + (count % BM != 0);
          begins[e] = begin;
          if (e + 1 == a.experts) begins[a.experts] = end;
        }
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
    // (no more than there can be, whatever the offsets say)
    tiles_m = __builtin_amdgcn_readfirstlane(
        min(first[a.experts], a.rows / BM + min(a.experts, a.rows)));
  }
  const TileRun run = xcd_tile_run(tiles_m * tiles_n, int(gridDim.x), int(blockIdx.x));

  // copies: this lane's row within a copy's eight and its chunk of the row
  const int crow = lane / (P / 16);
  const int lk = 16 * ((lane % (P / 16)) ^ swz32_f(wave * RPC + crow));
  // fragment reads: row lane % 32, chunk 2 ks + lane / 32
  const int frow = lane & 31, ff = swz32_f(frow);
  int koff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = frow * P + 16 * ((2 * ks + (lane >> 5)) ^ ff);
  const int abuf = wn * TN * P, bbuf = (BN + wm * TM) * P;

  // the tile whose copies are being issued
  int n0 = 0, row0 = 0, rows = 0, expert = 0;
  v4u wd, xd;
  uint32_t abase = 0, bbase = 0;
  uint32_t boff[kExperts ? CPB : 1];

  // Channels past n and rows past the tile's last read whatever lies there
  // inside the tensors: their sums go nowhere.  Chunks past k have to be zero
  // in one operand, and are in x.
  auto setup = [&](int t) {
    const int in_group = kRowGroup * tiles_n, g = t / in_group, m0 = g * kRowGroup;
    const int gm = min(kRowGroup, tiles_m - m0), at = t - g * in_group;
    const int tm = m0 + at % gm;
    n0 = at / gm * BO;
    row0 = tm * BM;
    int row_end = a.rows;
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
      row0 = __builtin_amdgcn_readfirstlane(begins[expert] + (tm - first[expert]) * BM);
      row_end = __builtin_amdgcn_readfirstlane(min(begins[expert + 1], a.rows));
      if (row0 < 0) row0 = row_end = 0;  // offsets that are no offsets
    }
    rows = max(0, min(BM, row_end - row0));
    wd = uniform_desc(static_cast<const int8_t *>(a.w) + int64_t(expert) * a.wide * a.k,
                   uint32_t(a.wide) * uint32_t(a.k));
    xd = uniform_desc(static_cast<const int8_t *>(a.x) + (gather ? 0 : int64_t(row0) * a.ldx),
                   rows == 0 ? 0u
                   : gather  ? uint32_t(int64_t(a.x_rows - 1) * a.ldx + a.k)
                             : uint32_t(rows - 1) * uint32_t(a.ldx) + uint32_t(a.k));
    abase = uint32_t(n0 + crow * (kPair ? 2 : 1)) * uint32_t(a.k) + uint32_t(lk);
    bbase = uint32_t(wave * RPC + crow) * uint32_t(a.ldx) + uint32_t(lk);
    if constexpr (kExperts) {
#pragma unroll
      for (int j = 0; j < CPB; ++j) {
        const int m = (wave + kWaves * j) * RPC + crow;
        uint32_t r = uint32_t(m);
        if (gather) r = m < rows ? uint32_t(a.sources[row0 + m]) : ~0u;
        boff[j] = (gather ? r < uint32_t(a.x_rows) : m < rows) ? r * uint32_t(a.ldx) + uint32_t(lk)
                                                              : kOutOfRange;
      }
    }
  };
  // copy j of the group's stage s into stage buffer `ring`
  auto copy = [&](int s, int ring, int j) {
    const uint32_t dst = lds0 + uint32_t(ring * kTile) + uint32_t(wave + kWaves * j) * 1024u;
    const int k = (s * KG + group) * P;
    if (j < CPA) {
      // eight rows of one 32-channel block (wave-uniform)
      const int lr = (wave + kWaves * j) * RPC, b = lr % TN / 32, bo = kGated ? b % FO : b;
      const int ch = lr / TN * (32 * FO) +
                     (kPair ? bo / 2 * 64 + bo % 2 + 2 * (lr % 32) : bo * 32 + lr % 32);
      const uint32_t r = uint32_t(ch) + (kGated && b >= FO ? uint32_t(a.n) : 0u);
      lds_copy16(wd, dst, abase + r * uint32_t(a.k) + uint32_t(k));
    } else if constexpr (kExperts) {
      const uint32_t off = boff[j - CPA];
      lds_copy16(xd, dst, lk < a.k - k && off != kOutOfRange ? off + uint32_t(k) : kOutOfRange);
    } else {
      lds_copy16(xd, dst, lk < a.k - k ? bbase + uint32_t(kWaves * RPC * (j - CPA)) * uint32_t(a.ldx) + uint32_t(k)
                                       : kOutOfRange);
    }
  };
  // scales and biases of the tile into parameter slot `slot`
  auto copy_params = [&](int slot) {
    const uint32_t dst = lds_addr(params + slot * kParams);
    const int64_t p = int64_t(expert) * a.wide;
    const v4u sd = uniform_desc(a.ws + p, uint32_t(a.wide) * 4u);
    const v4u bd = uniform_desc(a.bias ? a.bias + p : a.ws, a.bias ? uint32_t(a.wide) * 4u : 0u);
    const v4u rd = make_desc(a.xs, uint32_t(a.x_rows) * 4u);
    for (int i0 = wave_id * 64; i0 < BN + BM; i0 += 64 * kWaves * KG) {
      if (i0 < BN) {
        const int c = i0 + lane, half = kGated && c >= BO;
        const int ch = n0 + c - (half ? BO : 0);
        const uint32_t off = ch < a.n ? uint32_t(ch + (half ? a.n : 0)) * 4u : kOutOfRange;
        lds_copy4(sd, dst + uint32_t(i0) * 4u, off);
        lds_copy4(bd, dst + uint32_t(BN + i0) * 4u, off);
      } else {
        const int m = i0 - BN + lane;
        uint32_t r = uint32_t(row0 + m);
        if (m < rows && gather) r = uint32_t(a.sources[row0 + m]);
        lds_copy4(rd, dst + uint32_t(BN + i0) * 4u, m < rows && r < uint32_t(a.x_rows) ? r * 4u : kOutOfRange);
      }
    }
  };
  auto prologue = [&](int slot) {
    copy_params(slot);
#pragma unroll
    for (int s = 0; s < R; ++s) {
      if (s >= stages) break;
#pragma unroll
      for (int j = 0; j < CPW; ++j) copy(s, s, j);
    }
  };

  int t = run.first;
  if (t >= run.last) return;
  setup(t);
  int slot = 0;
  bool later = false;  // a tile after the first: stores may follow its copies
  prologue(slot);
  for (;;) {
    // the first stage has landed
    if (!later && stages >= R)
      wait_vm<(R - 1) * CPW>();
    else
      wait_vm<0>();
    barrier_lds();

    v16i acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // Fragments of GS k-steps, two sets: one feeds the MFMAs while the other
    // is read.
    constexpr int NP = KS / GS;
    v4i fa[2][GS][FN], fb[2][GS][FM];
    auto read = [&](auto set, const int8_t *buf, int part, int q) {
      const int ks = q / (FN + FM), n = q % (FN + FM);
      const int8_t *const p = buf + koff[part * GS + ks];
      if (n < FN)
        fa[set.value][ks][n] = *reinterpret_cast<const v4i *>(p + abuf + 32 * P * n);
      else
        fb[set.value][ks][n - FN] = *reinterpret_cast<const v4i *>(p + bbuf + 32 * P * (n - FN));
    };
    constexpr int kMfma = GS * FN * FM, kReads = GS * (FN + FM);
    int ring = 0;
    // a wave whose rows all lie past the tile's last only copies
    const bool idle = FM * FN >= 4 && wm * TM >= rows;
    if (idle) {
      for (int s = 0; s < stages; ++s) {
        if (s + R <= stages)
          wait_vm<(R - 2) * CPW>();
        else if (s + 1 < stages)
          wait_vm<0>();
        barrier_lds();
        if (s + R < stages) {
#pragma unroll
          for (int q = 0; q < CPW; ++q) copy(s + R, ring, q);
        }
        ring = ring + 1 == R ? 0 : ring + 1;
      }
    } else {
#pragma unroll
      for (int q = 0; q < kReads; ++q) read(Set<0>{}, bufs, 0, q);
    for (int s = 0; s < stages; ++s) {
      const int8_t *const buf = bufs + ring * kTile;
      const int next = ring + 1 == R ? 0 : ring + 1;
      const int8_t *const nbuf = bufs + next * kTile;
      const bool more = s + R < stages;
      auto part = [&](auto set, auto last, int pt) {
        if (last.value) {
          // every wave has read all of stage s, and stage s + 1 has landed
          // (of the copies in flight only the R - 2 stages after that may be)
          if (s + R <= stages)
            wait_vm<(R - 2) * CPW>();
          else if (s + 1 < stages)
            wait_vm<0>();
          barrier_lds();
        }
#pragma unroll
        for (int n = 0; n < kMfma; ++n) {
#pragma unroll
          for (int q = n * kReads / kMfma; q < (n + 1) * kReads / kMfma; ++q)
            read(Set<1 - set.value>{}, last.value ? nbuf : buf, last.value ? 0 : pt + 1, q);
          if (last.value && more) {
#pragma unroll
            for (int q = n * CPW / kMfma; q < (n + 1) * CPW / kMfma; ++q) copy(s + R, ring, q);
          }
          const int ks = n / (FN * FM), i = n / FM % FN, j = n % FM;
          acc[i][j] = mfma32(fb[set.value][ks][j], fa[set.value][ks][i], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      static_assert(NP == 2 || NP == 4, "an even number of sets per stage");
      part(Set<0>{}, std::false_type{}, 0);
      if constexpr (NP == 4) {
        part(Set<1>{}, std::false_type{}, 1);
        part(Set<0>{}, std::false_type{}, 2);
      }
      part(Set<1>{}, std::true_type{}, NP - 1);
      ring = next;
    }
    }

    const int out_n = n0, out_row = row0, out_rows = rows;
    const float *const pr = params + slot * kParams;
    t += run.step;
    const bool again = t < run.last;

    // Outputs of rows 8 g + 4 (lane / 32) + e of the wave's output block i (kPair:
    // of i and i + 1), row block j, from the lane's sums of quad g (all in 32 bits)
    constexpr int B = kPair ? 2 : 1;
    const int half = lane >> 5;
    // Q quads, from g0 on, of row block j: their sums sg (and su, the other
    // halves'), for each of the B blocks
    constexpr int Q = kGated || kOcc == 3 ? 1 : 2;  // (two spill there)
    auto finish = [&](int i, int j, int g0, const v4i (&sg)[B][Q], const v4i (&su)[B][Q]) {
      const int ct = wn * (32 * FO) + (kPair ? i * 32 + 2 * (lane & 31) : 32 * i + (lane & 31));
      const int ch = out_n + ct;
      const int r0 = wm * TM + 32 * j + 4 * half + 8 * g0;
      // windows over this step's rows, its first one at 0: rows past the tile's
      // last are out of their range, and so is the column of a channel past n
      const int size = a.out_type == I8CONV_FP32 ? 4 : 2;
      const int w0 = wm * TM + 32 * j + 8 * g0, left = out_rows - w0;
      const uint32_t yp = uint32_t(a.ldy) * uint32_t(size), rp = uint32_t(a.ldr) * uint32_t(size);
      const auto window = [&](const void *base, int64_t ld, uint32_t pitch) {
        const int in = min(left, 8 * Q);
        return make_rsrc(static_cast<const int8_t *>(base) + (out_row + w0) * ld * size,
                         in > 0 && base ? uint32_t(in - 1) * pitch + uint32_t(a.n) * uint32_t(size) : 0u);
      };
      const auto yr = window(a.y, a.ldy, yp), rr = window(a.residual, a.ldr, rp);
      auto row_of = [&](int e) { return 4 * half + 8 * (e / 4) + e % 4; };
      // 16-bit outputs leave two channels to a dword, at any alignment (buffer
      // accesses need none).  Single blocks: of every two rows an even lane takes
      // the first and its odd neighbour the second.  With n odd the last channel
      // is alone.
      const int odd = kPair ? 0 : lane & 1, pair = ch - odd;
      constexpr int W = kPair ? 4 * Q : 2 * Q;  // dwords
      auto word_row = [&](int w) { return kPair ? row_of(w) : row_of(2 * w) + odd; };
      const uint32_t cw = pair + 1 < a.n ? uint32_t(pair) * uint32_t(size) : kOutOfRange;
      const uint32_t alone = pair + 1 == a.n ? uint32_t(pair) * uint32_t(size) : kOutOfRange;
      const bool any_alone = __builtin_amdgcn_ballot_w64(alone != kOutOfRange) != 0;
      uint32_t cb[B];
#pragma unroll
      for (int b = 0; b < B; ++b) cb[b] = ch + b < a.n ? uint32_t(ch + b) * uint32_t(size) : kOutOfRange;

      // the residual, on its way while the sums are worked on
      uint32_t res[B][4 * Q];
      if (a.residual) {
        if (size == 2) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            res[0][w] = __builtin_amdgcn_raw_buffer_load_b32(rr, cw + uint32_t(word_row(w)) * rp, 0, 0);
          if (any_alone) {
#pragma unroll
            for (int w = 0; w < W; ++w)
              res[0][w] |= __builtin_amdgcn_raw_buffer_load_b16(rr, alone + uint32_t(word_row(w)) * rp, 0, 0);
          }
        } else {
#pragma unroll
          for (int b = 0; b < B; ++b)
#pragma unroll
            for (int e = 0; e < 4 * Q; ++e)
              res[b][e] = __builtin_amdgcn_raw_buffer_load_b32(rr, cb[b] + uint32_t(row_of(e)) * rp, 0, 0);
        }
      }

      float v[B][4 * Q];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const float ws = pr[ct + b], bias = pr[BN + ct + b];
        float u[4 * Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const v4f xs = *reinterpret_cast<const v4f *>(pr + 2 * BN + r0 + 8 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[b][4 * q + e] = fmaf(float(sg[b][q][e]) * xs[e], ws, bias);
          if constexpr (kGated) {
            const float ws2 = pr[BO + ct + b], bias2 = pr[BN + BO + ct + b];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              u[4 * q + e] = fmaf(float(su[b][q][e]) * xs[e], ws2, bias2);
          }
        }
        activate(v[b], a.activation);
        if constexpr (kGated) {
#pragma unroll
          for (int e = 0; e < 4 * Q; ++e) v[b][e] *= u[e];
        }
      }
      if (size == 4) {
#pragma unroll
        for (int e = 0; e < 4 * Q; ++e) {
          if (a.residual) {
#pragma unroll
            for (int b = 0; b < B; ++b) v[b][e] += bits_f32(res[b][e]);
          }
          const uint32_t row = uint32_t(row_of(e)) * yp;
          if constexpr (kPair) {
            __builtin_amdgcn_raw_buffer_store_b64(v2u{f32_bits(v[0][e]), f32_bits(v[1][e])}, yr, cw + row, 0, 0);
            if (any_alone)
              __builtin_amdgcn_raw_buffer_store_b32(f32_bits(v[0][e]), yr, alone + row, 0, 0);
          } else {
            __builtin_amdgcn_raw_buffer_store_b32(f32_bits(v[0][e]), yr, cb[0] + row, 0, 0);
          }
        }
        return;
      }
      auto store16 = [&](auto kind) {  // (the type once for all, not per value)
        constexpr int T = decltype(kind)::value;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          float lo, hi;
          if constexpr (kPair) {
            lo = v[0][w], hi = v[B - 1][w];
          } else {
            const float got = neighbour(odd ? v[0][2 * w] : v[0][2 * w + 1]);
            lo = odd ? got : v[0][2 * w];
            hi = odd ? v[0][2 * w + 1] : got;
          }
          if (a.residual) {
            lo += from_half(res[0][w] & 0xffffu, T);
            hi += from_half(res[0][w] >> 16, T);
          }
          const uint32_t word = to_halves(lo, hi, T), row = uint32_t(word_row(w)) * yp;
          __builtin_amdgcn_raw_buffer_store_b32(word, yr, cw + row, 0, 0);
          if (any_alone) __builtin_amdgcn_raw_buffer_store_b16(uint16_t(word), yr, alone + row, 0, 0);
        }
      };
      if (a.out_type == I8CONV_BF16)
        store16(Set<I8CONV_BF16>{});
      else
        store16(Set<I8CONV_FP16>{});
    };
    if constexpr (KG == 1) {
      // the next tile's copies go out before this tile's stores
      if (again) {
        setup(t);
        prologue(slot ^ 1);
      }
      // One copy of the code for all blocks: a step's sums are moved into
      // registers of their own first.  (Unrolled over the blocks it took 112 KB
      // and spilled 104 registers: 1024 rows of 8 tiles each, 16384 x 2048 ->
      // 8192, 434 us; 270 with one output type's code only.)
      constexpr int U = 4 / Q, kSteps = FM * (FO / B) * U;
#pragma unroll 1
      for (int st = idle ? kSteps : 0; st < kSteps; ++st) {
        v4i sg[B][Q], su[B][Q];
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          if (st != c) continue;
          asm volatile("" ::: "memory");  // a branch: selects would run through every block's registers
          const int j = c / U % FM, i = c / U / FM * B, g0 = c % U * Q;
#pragma unroll
          for (int b = 0; b < B; ++b)
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sg[b][q][e] = acc[i + b][j][4 * (g0 + q) + e];
                if constexpr (kGated) su[b][q][e] = acc[FO + i + b][j][4 * (g0 + q) + e];
              }
        }
        finish(st / U / FM * B, st / U % FM, st % U * Q, sg, su);
      }
    } else {
      // each wave's sums go to the first stage buffers (every wave has read
      // its last stage), four elements per 1 KB; then the groups take the
      // steps (two quads of a block) in turn
      auto part_of = [&](int grp, int b, int q) {
        return reinterpret_cast<v4i *>(smem + grp * R * kTile + (wave * FN * FM + b) * 4096 + q * 1024 +
                                       lane * 16);
      };
      static_assert(KG == 1 || kWaves * FN * FM * 4096 <= R * kTile, "sums fit the stage buffers");
      barrier_lds();
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *part_of(group, i * FM + j, q) = v4i{acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                                 acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      barrier_lds();
      auto total = [&](int f, int m, int q) {
        const int b = f * FM + m;
        v4u sum = *reinterpret_cast<const v4u *>(part_of(0, b, q));
#pragma unroll
        for (int g = 1; g < KG; ++g) sum += *reinterpret_cast<const v4u *>(part_of(g, b, q));
        return __builtin_bit_cast(v4i, sum);
      };
      constexpr int U = 4 / Q, kSteps = FM * (FO / B) * U;
#pragma unroll 1
      for (int st = group; st < kSteps; st += KG) {
        const int j = st / U % FM, i = st / U / FM * B, g0 = st % U * Q;
        v4i sg[B][Q], su[B][Q];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            sg[b][q] = total(i + b, j, g0 + q);
            if constexpr (kGated) su[b][q] = total(FO + i + b, j, g0 + q);
          }
        finish(i, j, g0, sg, su);
      }
      if (again) {
        barrier_lds();
        setup(t);
        prologue(slot ^ 1);
      }
    }
    if (!again) return;
    slot ^= 1;
    later = true;
  }
}

template <int BM, int BN, int WM, int WN, int R, int KG, int GS, int kOcc, int kGroups, bool kGated,
          bool kExperts>
int launch_tile(const LinearArgs &a, hipStream_t s) {
  auto kern = linear_kernel<BM, BN, WM, WN, R, KG, GS, kOcc, kGated, kExperts>;
  const size_t lds = size_t(KG) * R * (BM + BN) * kStageBytes + 2 * size_t(2 * BN + BM) * 4 +
                     (kExperts ? size_t(a.experts + 1) * 8 : 0);
  constexpr int BO = kGated ? BN / 2 : BN;
  // by expert: every group may end in a part of a tile
  int64_t tiles_m = (int64_t(a.rows) + BM - 1) / BM;
  if (kExperts) tiles_m = int64_t(a.rows) / BM + std::min(a.experts, a.rows);
  const int64_t tiles = tiles_m * ((int64_t(a.n) + BO - 1) / BO);
  static LdsLimit limit;
  if (const int rc = limit.raise(kern, lds); rc != I8CONV_OK) return rc;
  I8_LAUNCH(kern, dim3(unsigned(std::min<int64_t>(tiles, 256 * kGroups))), dim3(64 * WM * WN * KG), lds,
            s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string("linear kernel launch: ") + hipGetErrorString(e));
    return I8CONV_HIP_ERROR;
  }
  return I8CONV_OK;
}

template <bool kGated, bool kExperts>
int launch_any(const LinearArgs &a, int tile, hipStream_t s) {
  switch (tile) {
    case kTile256x256: return launch_tile<256, 256, 4, 2, 2, 1, 1, 2, 1, kGated, kExperts>(a, s);
    case kTile128x256: return launch_tile<128, 256, 2, 4, 3, 1, 1, 2, 1, kGated, kExperts>(a, s);
    case kTile128x128: return launch_tile<128, 128, 2, 2, 2, 1, 1, 2, 2, kGated, kExperts>(a, s);
    case kTile128x64: return launch_tile<128, 64, 4, 1, 2, 1, 2, 3, 3, kGated, kExperts>(a, s);
  }
  if constexpr (kGated) {
    if (tile == kTile128x64Pair) return launch_tile<128, 64, 4, 1, 3, 2, 2, 2, 1, true, kExperts>(a, s);
  } else {
    switch (tile) {
      case kTile64x64: return launch_tile<64, 64, 2, 2, 2, 1, 2, 4, 4, false, kExperts>(a, s);
      case kTile64x64Deep: return launch_tile<64, 64, 2, 2, 4, 1, 2, 2, 2, false, kExperts>(a, s);
      case kTile64x64Pair: return launch_tile<64, 64, 2, 2, 4, 2, 2, 2, 1, false, kExperts>(a, s);
    }
  }
  set_error("linear: unsupported tile " + std::to_string(tile));
  return I8CONV_BAD_ARGUMENT;
}

}  // namespace

int launch_linear_tiles(const LinearArgs &a, bool gated, int tile, void *stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.experts > 0) return gated ? launch_any<true, true>(a, tile, s) : launch_any<false, true>(a, tile, s);
  return gated ? launch_any<true, false>(a, tile, s) : launch_any<false, false>(a, tile, s);
}

}  // namespace i8conv
