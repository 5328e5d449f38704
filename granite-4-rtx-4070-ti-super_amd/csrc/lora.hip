// lora.hip - low-rank adapters of many requests beside a shared projection.
//
// granite4_lora_add: row m of x carries the number of its adapter (or none);
//   y[m][n] = base[m][n] + mult * alpha[a] * sum_r t[m][r] B[a][n][r],
//   t[m][r] = sum_k x[m][k] A[a][part(n)][r][k],  a = adapter[m],
// where part(n) is the weight block (q | k | v, gate | up) of output column n.
// Rows may name adapters in any order: a 16- or 32-row tile takes the distinct
// adapters of its rows one after another and keeps, of each product, the rows
// that asked for it. A tile of one session's rows has one.
//
// Two launches. lora_shrink_kernel: t, the rank-side product over K, 8 waves
// of a workgroup over K, joined in LDS (f32 sums in a fixed order).
// lora_expand_kernel: 64 output columns per wave over the rank, the base added
// in f32 and rounded once. Between them t is two bf16 terms, t = hi + lo to
// 2^-17 of it: as one bf16 it would add 2^-9 of the adapter's part to an f32
// output, and the second product costs nothing beside the loads.
#include "attn_rows.h"
#include "g4_common.h"
#include "g4_hw.h"
#include "g4_math.h"
#include "granite4_layerops.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

namespace g4 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kMaxRank = 128;
constexpr int kShrinkWaves = 8;

struct LoraArgs {
  const void* x;          // [M][ldx] bf16, or e4m3 codes under *xs
  int ldx;
  const float* xs;
  const uint16_t* A;      // [adapters][parts][rank][K]
  const uint16_t* B;      // [adapters][N][rank]
  const float* alpha;     // [adapters]
  const int* adapter;     // [M]
  int adapters, rank, parts;
  int M, N, K, seg1, seg2;
  const void* base;       // [M][ldb] (bf16 or f32, as the output), or nullptr: 0
  int ldb;
  float mult;
  void* y;
  int ldy;
  int keep;               // rows without an adapter are in place already
  uint16_t* t_hi;         // [M][parts * rank]
  uint16_t* t_lo;
};

// Eight x elements as bf16 (e4m3 values are bf16 values).
template <bool FP8>
__device__ __forceinline__ bf16x8_t x_frag(const u32x4_t& r) {
  if constexpr (!FP8) {
    return __builtin_bit_cast(bf16x8_t, r);
  } else {
    u32x4_t o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(r[i]), false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(r[i]), true);
      o[2 * i] = pack_bf16_hw(a[0], a[1]);
      o[2 * i + 1] = pack_bf16_hw(b[0], b[1]);
    }
    return __builtin_bit_cast(bf16x8_t, o);
  }
}

// Workgroup: XT x 16 rows of x against RT x 16 of the parts * rank rows of an
// adapter's A, each wave 64 of K at a time. v_mfma_f32_16x16x32_bf16 with A's
// rows as its rows and x's as its columns: a lane ends up with four
// consecutive ranks of one row.
template <int RT, int XT, bool FP8>
__global__ __launch_bounds__(kShrinkWaves * 64) void lora_shrink_kernel(LoraArgs a) {
  constexpr int kXRows = 16 * XT;
  __shared__ __align__(16) f32x4_t part[kShrinkWaves][RT * XT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x * kXRows, pr = a.parts * a.rank;
  const int r0 = blockIdx.y * 16 * RT;
  const int mine = m0 + lane < a.M && lane < kXRows ? a.adapter[m0 + lane] : -1;
  unsigned long long todo = __ballot(mine >= 0 && mine < a.adapters);
  const uint8_t* xb = static_cast<const uint8_t*>(a.x);
  const int units = a.K / 64;
  for (int idx = 0; todo != 0ull; ++idx) {
    const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__ballot(mine == id);
    if (idx % static_cast<int>(gridDim.z) != static_cast<int>(blockIdx.z)) continue;
    const uint16_t* ab = a.A + static_cast<size_t>(id) * pr * a.K;
    f32x4_t acc[RT][XT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < XT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int u = wave; u < units; u += kShrinkWaves) {
      u32x4_t xr[XT][2], ar[RT][2];
#pragma unroll
      for (int j = 0; j < XT; ++j) {
        const size_t m = static_cast<size_t>(min(m0 + 16 * j + n, a.M - 1));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const size_t at = m * a.ldx + 64 * u + 32 * s + 8 * g;
          if constexpr (FP8) {
            const u32x2_t v = *reinterpret_cast<const u32x2_t*>(xb + at);
            xr[j][s] = u32x4_t{v.x, v.y, 0u, 0u};
          } else {
            xr[j][s] = *reinterpret_cast<const u32x4_t*>(xb + 2 * at);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const uint16_t* src = ab + static_cast<size_t>(min(r0 + 16 * i + n, pr - 1)) * a.K + 64 * u + 8 * g;
#pragma unroll
        for (int s = 0; s < 2; ++s) ar[i][s] = *reinterpret_cast<const u32x4_t*>(src + 32 * s);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < XT; ++j) {
          const bf16x8_t xf = x_frag<FP8>(xr[j][s]);
#pragma unroll
          for (int i = 0; i < RT; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ar[i][s]), xf,
                                                                acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < XT; ++j) part[wave][i * XT + j][lane] = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < RT * XT * 64; e += kShrinkWaves * 64) {
      const int tile = e >> 6, l = e & 63;
      f32x4_t v = part[0][tile][l];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) v += part[w][tile][l];
      const int m = m0 + 16 * (tile % XT) + (l & 15), r = r0 + 16 * (tile / XT) + 4 * (l >> 4);
      if (m < a.M && r < pr && a.adapter[m] == id) {
        if constexpr (FP8) v *= *a.xs;
        const u32x2_t hw = {pack_bf16_hw(v[0], v[1]), pack_bf16_hw(v[2], v[3])};
        float lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float hi = (i & 1) ? hi_bf16(hw[i >> 1]) : lo_bf16(hw[i >> 1]);
          lo[i] = fabsf(hi) < INFINITY ? v[i] - hi : 0.0f;  // infinities and NaN stay in the first term
        }
        const size_t at = static_cast<size_t>(m) * pr + r;
        *reinterpret_cast<u32x2_t*>(a.t_hi + at) = hw;
        *reinterpret_cast<u32x2_t*>(a.t_lo + at) = u32x2_t{pack_bf16_hw(lo[0], lo[1]), pack_bf16_hw(lo[2], lo[3])};
      }
    }
    __syncthreads();
  }
}

// Wave: 64 output columns of 16-row tiles. B's rows (columns of y) are the
// MFMA rows, t's rows its columns; MFMA row 4 g + i of product q is column
// 16 g + 4 q + i, so that a lane's 16 values are consecutive columns of one row.
template <int KS, bool F32>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a, int tiles_per_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int c0 = (blockIdx.x * 4 + wave) * 64;
  if (c0 >= a.N) return;
  const int part = (c0 >= a.seg1) + (c0 >= a.seg2), pr = a.parts * a.rank;
  const int tile0 = blockIdx.y * tiles_per_wave;
  const int tile1 = min(tile0 + tiles_per_wave, (a.M + 15) / 16);
  const int lc = c0 + 16 * g;  // this lane's 16 columns
  bf16x8_t bf[4][KS];
  int held = -1;
  float f = 0.0f;
  for (int tile = tile0; tile < tile1; ++tile) {
    const int m = tile * 16 + n;
    int mine = m < a.M ? a.adapter[m] : -1;
    if (mine < 0 || mine >= a.adapters) mine = -1;
    unsigned long long todo = __ballot(mine >= 0) & 0xffffull;
    // Rows without an adapter: the base as it is, by the first slot.
    if (blockIdx.z == 0 && m < a.M && mine < 0 && !a.keep) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (lc + 8 * q >= a.N) continue;
        const size_t bi = static_cast<size_t>(m) * a.ldb + lc + 8 * q, yi = static_cast<size_t>(m) * a.ldy + lc + 8 * q;
        const u32x4_t z = {0u, 0u, 0u, 0u};
        if constexpr (F32) {
          const float* b = static_cast<const float*>(a.base);
          float* y = static_cast<float*>(a.y);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<u32x4_t*>(y + yi + 4 * i) = b == nullptr ? z : *reinterpret_cast<const u32x4_t*>(b + bi + 4 * i);
        } else {
          const uint16_t* b = static_cast<const uint16_t*>(a.base);
          *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.y) + yi) =
              b == nullptr ? z : *reinterpret_cast<const u32x4_t*>(b + bi);
        }
      }
    }
    for (int idx = 0; todo != 0ull; ++idx) {
      const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == id);
      if (idx % static_cast<int>(gridDim.z) != static_cast<int>(blockIdx.z)) continue;
      const bool live = mine == id;
      if (id != held) {
        held = id;
        f = a.mult * a.alpha[id];
        const uint16_t* bb = a.B + static_cast<size_t>(id) * a.N * a.rank;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = min(c0 + 16 * (n >> 2) + 4 * q + (n & 3), a.N - 1);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int r = 32 * s + 8 * g;
            const u32x4_t v = *reinterpret_cast<const u32x4_t*>(bb + static_cast<size_t>(c) * a.rank + (r < a.rank ? r : 0));
            bf[q][s] = __builtin_bit_cast(bf16x8_t, r < a.rank ? v : u32x4_t{0u, 0u, 0u, 0u});
          }
        }
      }
      // A row of another adapter (or none) has no t of this one: row of a live lane instead.
      bf16x8_t th[KS], tl[KS];
      const size_t trow = (static_cast<size_t>(live ? m : 0)) * pr + static_cast<size_t>(part) * a.rank;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int r = 32 * s + 8 * g;
        const bool on = live && r < a.rank;
        const size_t at = on ? trow + r : 0;
        const u32x4_t vh = *reinterpret_cast<const u32x4_t*>(a.t_hi + at);
        const u32x4_t vl = *reinterpret_cast<const u32x4_t*>(a.t_lo + at);
        th[s] = __builtin_bit_cast(bf16x8_t, on ? vh : u32x4_t{0u, 0u, 0u, 0u});
        tl[s] = __builtin_bit_cast(bf16x8_t, on ? vl : u32x4_t{0u, 0u, 0u, 0u});
      }
      float bv[16];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bool on = live && lc + 8 * q < a.N && a.base != nullptr;
        const size_t bi = static_cast<size_t>(m) * a.ldb + lc + 8 * q;
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (on) v = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(a.base) + bi + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) bv[8 * q + 4 * i + e] = v[e];
          }
        } else {
          V8 v{{0u, 0u, 0u, 0u}};
          if (on) v = ld8(static_cast<const uint16_t*>(a.base) + bi);
#pragma unroll
          for (int e = 0; e < 8; ++e) bv[8 * q + e] = v8_get(v, e);
        }
      }
      f32x4_t acc[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        acc[q] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[q][s], tl[s], acc[q], 0, 0, 0);
          acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[q][s], th[s], acc[q], 0, 0, 0);
        }
      }
      if (!live) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (lc + 8 * q >= a.N) continue;
        const size_t yi = static_cast<size_t>(m) * a.ldy + lc + 8 * q;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = bv[8 * q + e] + f * acc[2 * q + (e >> 2)][e & 3];
        if constexpr (F32) {
          float* y = static_cast<float*>(a.y) + yi;
          *reinterpret_cast<f32x4_t*>(y) = f32x4_t{o[0], o[1], o[2], o[3]};
          *reinterpret_cast<f32x4_t*>(y + 4) = f32x4_t{o[4], o[5], o[6], o[7]};
        } else {
          *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.y) + yi) =
              u32x4_t{pack_bf16_hw(o[0], o[1]), pack_bf16_hw(o[2], o[3]), pack_bf16_hw(o[4], o[5]), pack_bf16_hw(o[6], o[7])};
        }
      }
    }
  }
}

template <int RT, int XT>
void launch_shrink(const LoraArgs& a, bool fp8, int slots, hipStream_t st) {
  const dim3 grid((a.M + 16 * XT - 1) / (16 * XT), (a.parts * a.rank + 16 * RT - 1) / (16 * RT), slots);
  if (fp8) hipLaunchKernelGGL((lora_shrink_kernel<RT, XT, true>), grid, kShrinkWaves * 64, 0, st, a);
  else hipLaunchKernelGGL((lora_shrink_kernel<RT, XT, false>), grid, kShrinkWaves * 64, 0, st, a);
}

template <int KS>
void launch_expand(const LoraArgs& a, bool f32, int per, int slots, hipStream_t st) {
  const dim3 grid((a.N + 255) / 256, ((a.M + 15) / 16 + per - 1) / per, slots);
  if (f32) hipLaunchKernelGGL((lora_expand_kernel<KS, true>), grid, 256, 0, st, a, per);
  else hipLaunchKernelGGL((lora_expand_kernel<KS, false>), grid, 256, 0, st, a, per);
}

int parts_of(int N, int seg1, int seg2) { return seg1 >= N ? 1 : seg2 >= N ? 2 : 3; }

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" {

size_t granite4_lora_work_bytes(int M, int N, int K, int rank, int seg1, int seg2) {
  (void)K;
  if (M <= 0 || N <= 0 || rank <= 0) return 0;
  return static_cast<size_t>(M) * parts_of(N, seg1, seg2) * rank * 4;
}

int granite4_lora_add(int out, const void* X, int x_bits, int ldx, const float* d_x_scale,
                      const uint16_t* A, const uint16_t* B, const float* d_alpha, int adapters,
                      int rank, const int* d_row_adapter, int M, int N, int K, int seg1, int seg2,
                      const void* base, int ldb, float mult, void* y, int ldy, void* work) {
  const bool fp8 = x_bits == 8;
  if ((out != GRANITE4_GEMM_BF16 && out != GRANITE4_GEMM_F32) || (x_bits != 16 && !fp8) ||
      X == nullptr || (fp8 && d_x_scale == nullptr) || A == nullptr || B == nullptr ||
      d_alpha == nullptr || d_row_adapter == nullptr || y == nullptr || work == nullptr ||
      adapters < 1 || rank < 8 || rank > kMaxRank || rank % 8 != 0 || M < 1 || N < 8 ||
      N % 8 != 0 || K < 64 || K % 64 != 0 || ldx < K || ldx % (fp8 ? 16 : 8) != 0 || ldy < N ||
      ldy % 8 != 0 || (base != nullptr && (ldb < N || ldb % 8 != 0)) ||
      (base == y && ldb != ldy) || seg1 < 1 || seg2 < seg1 ||
      (seg1 < N && seg1 % 64 != 0) || (seg2 < N && seg2 % 64 != 0) || !std::isfinite(mult) ||
      !aligned(X, 16) || !aligned(A, 16) || !aligned(B, 16) || !aligned(base, 16) ||
      !aligned(y, 16) || !aligned(work, 16) || M > 16 * 65535) {
    std::fprintf(stderr, "granite4: granite4_lora_add: invalid arguments\n");
    return -1;
  }
  LoraArgs a{};
  a.x = X;
  a.ldx = ldx;
  a.xs = d_x_scale;
  a.A = A;
  a.B = B;
  a.alpha = d_alpha;
  a.adapter = d_row_adapter;
  a.adapters = adapters;
  a.rank = rank;
  a.parts = parts_of(N, seg1, seg2);
  a.M = M;
  a.N = N;
  a.K = K;
  a.seg1 = seg1;
  a.seg2 = seg2;
  a.base = base;
  a.ldb = ldb;
  a.mult = mult;
  a.y = y;
  a.ldy = ldy;
  a.keep = base == y;
  a.t_hi = static_cast<uint16_t*>(work);
  a.t_lo = a.t_hi + static_cast<size_t>(M) * a.parts * rank;
  const hipStream_t st = stream();
  const int pr = a.parts * rank;
  // One tile's distinct adapters over workgroups of their own where rows are few.
  const int slots = M <= 64 ? std::min({16, M, adapters}) : 1;
  if (M <= 64) launch_shrink<1, 1>(a, fp8, slots, st);
  else if (pr <= 16) launch_shrink<1, 2>(a, fp8, 1, st);
  else if (pr <= 32) launch_shrink<2, 2>(a, fp8, 1, st);
  else launch_shrink<4, 2>(a, fp8, 1, st);
  const int per = M <= 256 ? 1 : 4;
  const bool f32 = out == GRANITE4_GEMM_F32;
  if (rank <= 32) launch_expand<1>(a, f32, per, slots, st);
  else if (rank <= 64) launch_expand<2>(a, f32, per, slots, st);
  else launch_expand<4>(a, f32, per, slots, st);
  return launch_status("granite4_lora_add");
}

}  // extern "C"
