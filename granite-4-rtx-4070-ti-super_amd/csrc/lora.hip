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
// Two launches. lora_shrink_kernel: t, the rank-side product over K, which the
// waves of a workgroup share and several workgroups where rows are few, joined
// in LDS and by the last of them (f32 sums in a fixed order).
// lora_expand_kernel: 64 output columns per wave over the rank, the base added
// in f32 and rounded once. Between them t is a sum of bf16 terms, of two (2^-17
// of it is lost) for a bf16 output and of three (2^-25) for an f32 one: as one
// bf16 it would lose 2^-9, and the further products cost nothing beside the loads.
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
constexpr int kMaxShares = 8;  // of K: the shrink's join has that many loads

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
  // t as a sum of bf16 terms, each as the expand's fragments: [16-row tile][part]
  // [32-rank step][lane][8], lane n + 16 g having row n's ranks 8 g ..
  uint16_t* t;
  size_t t_pitch;         // between terms
  int terms;
  int splits;             // shares of K
  float* part;            // [splits][M][parts * rank]: their sums, where there are several
  unsigned* arrived;      // workgroups done, per row tile, rank group and slot; 0 between calls
};

// Eight x elements as bf16 (e4m3 values are bf16 values).
__device__ __forceinline__ u32x4_t fp8x8_bf16(const u32x2_t& r) {
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(r[i]), false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(r[i]), true);
    o[2 * i] = pack_bf16_hw(a[0], a[1]);
    o[2 * i + 1] = pack_bf16_hw(b[0], b[1]);
  }
  return o;
}

// Partials and counts pass between workgroups of any XCD: device scope.
__device__ __forceinline__ void st_dev(float* p, const f32x4_t& v) {
  unsigned long long* q = reinterpret_cast<unsigned long long*>(p);
  const unsigned long long a = __float_as_uint(v[0]) | (static_cast<unsigned long long>(__float_as_uint(v[1])) << 32);
  const unsigned long long b = __float_as_uint(v[2]) | (static_cast<unsigned long long>(__float_as_uint(v[3])) << 32);
  __hip_atomic_store(q, a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(q + 1, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4_t ld_dev(const float* p) {
  unsigned long long* q = reinterpret_cast<unsigned long long*>(const_cast<float*>(p));
  const unsigned long long a = __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const unsigned long long b = __hip_atomic_load(q + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return f32x4_t{__uint_as_float(static_cast<unsigned>(a)), __uint_as_float(static_cast<unsigned>(a >> 32)),
                 __uint_as_float(static_cast<unsigned>(b)), __uint_as_float(static_cast<unsigned>(b >> 32))};
}

// 32-rank steps of the expand's products: the forms it is compiled for.
__host__ __device__ constexpr int rank_steps(int rank) { return rank <= 32 ? 1 : rank <= 64 ? 2 : 4; }

// Four ranks of row m as bf16 terms.
template <bool FP8>
__device__ __forceinline__ void store_t(const LoraArgs& a, int m, int r, f32x4_t v) {
  if constexpr (FP8) v *= *a.xs;
  const int part = r / a.rank, rr = r - part * a.rank, steps = rank_steps(a.rank);
  uint16_t* dst = a.t + ((static_cast<size_t>(m >> 4) * a.parts + part) * steps + (rr >> 5)) * 512 +
                  8 * ((m & 15) + 16 * ((rr >> 3) & 3)) + (rr & 7);
  for (int k = 0; k < a.terms; ++k, dst += a.t_pitch) {
    const u32x2_t hw = {pack_bf16_hw(v[0], v[1]), pack_bf16_hw(v[2], v[3])};
    *reinterpret_cast<u32x2_t*>(dst) = hw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float hi = (i & 1) ? hi_bf16(hw[i >> 1]) : lo_bf16(hw[i >> 1]);
      v[i] = fabsf(hi) < INFINITY ? v[i] - hi : 0.0f;  // infinities and NaN stay in the first term
    }
  }
}

// Workgroup: XT x 16 rows of x against RT x 16 of the parts * rank rows of an
// adapter's A, over one of a.splits shares of K; its waves take 64 of K in turn.
// v_mfma_f32_16x16x32_bf16 with A's rows as its rows and x's as its columns: a
// lane ends up with four consecutive ranks of one row.
//
// A fragment read straight from memory is 16 bytes of each of 16 rows per
// quarter of a wave, 16 cache lines for 256 bytes, at which the CU's cache gives
// a quarter of its rate (8192 rows of 12800, rank 64: 94 us). Eight lanes take a
// whole 128-byte line of a row here, and a wave turns its tiles through 2 KB each
// of LDS (16-byte chunk c of row r in slot c ^ (r mod 8): 8 lanes read 128 bytes
// of different banks). DS operations of a wave execute in order, so the tiles of
// the next 64 follow without a wait.
template <int RT, int XT, bool FP8>
__global__ __launch_bounds__(kShrinkWaves * 64) __attribute__((amdgpu_waves_per_eu(RT * XT > 8 ? 2 : 4)))
void lora_shrink_kernel(LoraArgs a) {
  constexpr int kXRows = 16 * XT;
  constexpr int kDeep = RT + XT <= 3 ? 2 : 1;  // units in flight while one is multiplied
  union Lds {
    u32x4_t tile[kShrinkWaves][RT + XT][128];
    f32x4_t part[kShrinkWaves][RT * XT][64];
  };
  __shared__ Lds lds;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x * kXRows, pr = a.parts * a.rank;
  const int rg = blockIdx.y / a.splits, ks = blockIdx.y % a.splits, r0 = rg * 16 * RT;
  const int mine = m0 + lane < a.M && lane < kXRows ? a.adapter[m0 + lane] : -1;
  unsigned long long todo = __ballot(mine >= 0 && mine < a.adapters), done = 0ull;
  const uint8_t* xb = static_cast<const uint8_t*>(a.x);
  const int units = a.K / 64, u_end = units * (ks + 1) / a.splits, u_first = units * ks / a.splits + wave;
  const int lr = lane >> 3, lc = lane & 7;  // loads: row (and row + 8) and 16-byte chunk of a tile
  u32x4_t* const put = &lds.tile[wave][0][8 * lr + (lc ^ lr)];
  const u32x4_t* const get = &lds.tile[wave][0][8 * n];
  // e4m3 rows are 64 bytes: four lanes to a row, each with two chunks of bf16.
  const int fr = lane >> 2, fc = 2 * (lane & 3);
  u32x4_t* const put8 = &lds.tile[wave][0][8 * fr];
  size_t xrow[XT][FP8 ? 1 : 2];
#pragma unroll
  for (int j = 0; j < XT; ++j) {
    if constexpr (FP8) {
      xrow[j][0] = static_cast<size_t>(min(m0 + 16 * j + fr, a.M - 1)) * a.ldx + 16 * (lane & 3);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) xrow[j][e] = static_cast<size_t>(min(m0 + 16 * j + 8 * e + lr, a.M - 1)) * a.ldx + 8 * lc;
    }
  }
  for (int idx = 0; todo != 0ull; ++idx) {
    const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const unsigned long long same = __ballot(mine == id);
    todo &= ~same;
    if (idx % static_cast<int>(gridDim.z) != static_cast<int>(blockIdx.z)) continue;
    done |= same;
    // 16-row tiles of x that have a row of this adapter: a tile on the border of two
    // sessions multiplies each part with its own adapter's A only.
    unsigned need = 0u;
#pragma unroll
    for (int j = 0; j < XT; ++j) need |= static_cast<unsigned>(((same >> (16 * j)) & 0xffffull) != 0ull) << j;
    const auto needs = [&](int j) { return XT == 1 || ((need >> j) & 1u) != 0u; };
    const uint16_t* ab = a.A + static_cast<size_t>(id) * pr * a.K + 8 * lc;
    f32x4_t acc[RT][XT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < XT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4_t xr[kDeep][XT][FP8 ? 1 : 2], ar[kDeep][RT][2];
    const auto load = [&](int d, int u) {  // a unit past the end loads the last one again
      const int k = 64 * min(u, u_end - 1);
#pragma unroll
      for (int j = 0; j < XT; ++j) {
        if (!needs(j)) continue;
#pragma unroll
        for (int e = 0; e < (FP8 ? 1 : 2); ++e)
          xr[d][j][e] = *reinterpret_cast<const u32x4_t*>(xb + (FP8 ? 1 : 2) * (xrow[j][e] + k));
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          ar[d][i][e] = *reinterpret_cast<const u32x4_t*>(ab + static_cast<size_t>(min(r0 + 16 * i + 8 * e + lr, pr - 1)) * a.K + k);
    };
#pragma unroll
    for (int d = 0; d < kDeep; ++d) load(d, u_first + d * kShrinkWaves);
    for (int u0 = u_first; u0 < u_end; u0 += kDeep * kShrinkWaves) {
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const int u = u0 + d * kShrinkWaves;
        if (u >= u_end) break;
#pragma unroll
        for (int j = 0; j < XT; ++j) {
          if (!needs(j)) continue;
          if constexpr (FP8) {
            put8[128 * j + (fc ^ (fr & 7))] = fp8x8_bf16(u32x2_t{xr[d][j][0].x, xr[d][j][0].y});
            put8[128 * j + ((fc + 1) ^ (fr & 7))] = fp8x8_bf16(u32x2_t{xr[d][j][0].z, xr[d][j][0].w});
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) put[128 * j + 64 * e] = xr[d][j][e];
          }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) put[128 * (XT + i) + 64 * e] = ar[d][i][e];
        if (u + kDeep * kShrinkWaves < u_end) load(d, u + kDeep * kShrinkWaves);
        asm volatile("" ::: "memory");  // the reads stay behind the writes
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int slot = (4 * s + g) ^ (n & 7);
          bf16x8_t xf[XT];
#pragma unroll
          for (int j = 0; j < XT; ++j)
            if (needs(j)) xf[j] = __builtin_bit_cast(bf16x8_t, get[128 * j + slot]);
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            const bf16x8_t af = __builtin_bit_cast(bf16x8_t, get[128 * (XT + i) + slot]);
#pragma unroll
            for (int j = 0; j < XT; ++j)
              if (needs(j)) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, xf[j], acc[i][j], 0, 0, 0);
          }
        }
        asm volatile("" ::: "memory");  // and the next writes behind the reads
      }
    }
    __syncthreads();  // the tiles are read: their place takes the sums
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < XT; ++j) lds.part[wave][i * XT + j][lane] = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < RT * XT * 64; e += kShrinkWaves * 64) {
      const int tile = e >> 6, l = e & 63, at = 16 * (tile % XT) + (l & 15);
      f32x4_t v = lds.part[0][tile][l];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) v += lds.part[w][tile][l];
      const int r = r0 + 16 * (tile / XT) + 4 * (l >> 4);
      if (((same >> at) & 1ull) == 0ull || r >= pr) continue;
      if (a.splits == 1) store_t<FP8>(a, m0 + at, r, v);
      else st_dev(a.part + (static_cast<size_t>(ks) * a.M + m0 + at) * pr + r, v);
    }
    __syncthreads();
  }
  if (a.splits == 1 || done == 0ull) return;
  // The last of the shares' workgroups adds them up, in their order; none waits.
  __shared__ unsigned s_arrived;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  unsigned* count = a.arrived + (static_cast<size_t>(blockIdx.x) * (gridDim.y / a.splits) + rg) * gridDim.z + blockIdx.z;
  if (threadIdx.x == 0) s_arrived = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_arrived != static_cast<unsigned>(a.splits) - 1u) return;
  if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int e = threadIdx.x; e < RT * XT * 64; e += kShrinkWaves * 64) {
    const int at = e & (kXRows - 1), r = r0 + 4 * (e / kXRows);
    if (((done >> at) & 1ull) == 0ull || r >= pr) continue;
    const float* src = a.part + static_cast<size_t>(m0 + at) * pr + r;
    f32x4_t p[kMaxShares];  // two, four or all eight loads under way at once
    const auto load = [&](int k) { p[k] = ld_dev(src + static_cast<size_t>(min(k, a.splits - 1)) * a.M * pr); };
    load(0), load(1);
    if (XT == 1 || a.splits > 2) load(2), load(3);
    if (XT == 1 || a.splits > 4) load(4), load(5), load(6), load(7);
    f32x4_t v = p[0];
#pragma unroll
    for (int k = 1; k < kMaxShares; ++k)
      if (k < a.splits) v += p[k];
    store_t<FP8>(a, m0 + at, r, v);
  }
}

// Wave: 64 output columns of 16-row tiles. B's rows (columns of y) are the
// MFMA rows, t's rows its columns, so a lane gets 4 columns of a row per product.
// The tile turns through LDS (rows 272 bytes apart: 8 lanes' 16-byte writes to
// different banks) to be added to the base and written as whole 128- or 256-byte
// row pieces by consecutive lanes: straight from the product's lanes a quarter of
// a wave has 16 bytes of each of 16 rows (8192 rows, 4096 columns, rank 64: 59 us).
template <int KS, bool F32>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a, int tiles_per_wave) {
  constexpr int kTerms = F32 ? 3 : 2;
  constexpr int kVecs = F32 ? 4 : 2;            // 16-byte vectors a lane has of the tile
  constexpr int kLanes = F32 ? 16 : 8;          // lanes to a row
  constexpr int kPer = 64 / kLanes, kBytes = F32 ? 4 : 2;
  constexpr int kPitch = 68;
  __shared__ __align__(16) float turn[4][16 * kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int c0 = (blockIdx.x * 4 + wave) * 64;
  if (c0 >= a.N) return;
  const int part = (c0 >= a.seg1) + (c0 >= a.seg2);
  const int tile0 = blockIdx.y * tiles_per_wave;
  const int tile1 = min(tile0 + tiles_per_wave, (a.M + 15) / 16);
  const int r_l = lane / kLanes, c_l = c0 + kPer * (lane % kLanes);  // vector v: row r_l + v 64 / kLanes
  const bool in = c_l < a.N;
  const uint8_t* base = static_cast<const uint8_t*>(a.base);
  uint8_t* y = static_cast<uint8_t*>(a.y);
  float* const out = turn[wave];
  bf16x8_t bf[4][KS], t[KS][kTerms];
  u32x4_t bv[kVecs];
  int held = -1;
  float f = 0.0f;
  for (int tile = tile0; tile < tile1; ++tile) {
    const int m0 = tile * 16;
    int mine = m0 + n < a.M ? a.adapter[m0 + n] : -1;
    // The rows' base, those of `which`.
    const auto load_base = [&](unsigned which) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int r = r_l + v * (64 / kLanes);
        bv[v] = u32x4_t{0u, 0u, 0u, 0u};
        if (((which >> r) & 1u) != 0u && m0 + r < a.M && in && base != nullptr)
          bv[v] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(base + kBytes * (static_cast<size_t>(m0 + r) * a.ldb + c_l)));
      }
    };
    const bool slots = gridDim.z > 1;  // few rows, an adapter a workgroup: its own rows only
    if (!slots) load_base(0xffffu);
    // t: a row without an adapter has none; what is read there stays in the row's
    // own column of the product and is not written.
    const uint16_t* tf = a.t + (static_cast<size_t>(tile) * a.parts + part) * KS * 512 + 8 * lane;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int k = 0; k < kTerms; ++k) {
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(tf + k * a.t_pitch + 512 * s);
        t[s][k] = __builtin_bit_cast(bf16x8_t, 32 * s + 8 * g < a.rank ? v : u32x4_t{0u, 0u, 0u, 0u});
      }
    if (mine < 0 || mine >= a.adapters) mine = -1;
    const auto write = [&](int v, const u32x4_t& x) {
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(y + kBytes * (static_cast<size_t>(m0 + r_l + v * (64 / kLanes)) * a.ldy + c_l)));
    };
    unsigned todo = static_cast<unsigned>(__ballot(mine >= 0)) & 0xffffu;
    // Rows without an adapter: the base as it is, by the first slot.
    if (blockIdx.z == 0 && todo != 0xffffu && !a.keep) {
      if (slots) load_base(~todo);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int r = r_l + v * (64 / kLanes);
        if (((todo >> r) & 1u) == 0u && m0 + r < a.M && in) write(v, bv[v]);
      }
    }
    for (int idx = 0; todo != 0u; ++idx) {
      const int id = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
      const unsigned same = static_cast<unsigned>(__ballot(mine == id)) & 0xffffu;
      todo &= ~same;
      if (idx % static_cast<int>(gridDim.z) != static_cast<int>(blockIdx.z)) continue;
      if (slots) load_base(same);
      if (id != held) {
        held = id;
        f = a.mult * a.alpha[id];
        const uint16_t* bb = a.B + static_cast<size_t>(id) * a.N * a.rank;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = min(c0 + 16 * q + n, a.N - 1);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int r = 32 * s + 8 * g;
            const u32x4_t v = *reinterpret_cast<const u32x4_t*>(bb + static_cast<size_t>(c) * a.rank + (r < a.rank ? r : 0));
            bf[q][s] = __builtin_bit_cast(bf16x8_t, r < a.rank ? v : u32x4_t{0u, 0u, 0u, 0u});
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = kTerms - 1; k >= 0; --k)  // the smallest first
#pragma unroll
          for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[q][s], t[s][k], acc, 0, 0, 0);
        *reinterpret_cast<f32x4_t*>(out + n * kPitch + 16 * q + 4 * g) = acc;
      }
      asm volatile("" ::: "memory");  // a wave's DS operations execute in order
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int r = r_l + v * (64 / kLanes);
        const f32x4_t p = *reinterpret_cast<const f32x4_t*>(out + r * kPitch + kPer * (lane % kLanes));
        u32x4_t x;
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __float_as_uint(__uint_as_float(bv[v][e]) + f * p[e]);
        } else {
          const f32x4_t p2 = *reinterpret_cast<const f32x4_t*>(out + r * kPitch + kPer * (lane % kLanes) + 4);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            x[w] = pack_bf16_hw(lo_bf16(bv[v][w]) + f * p[2 * w], hi_bf16(bv[v][w]) + f * p[2 * w + 1]);
            x[2 + w] = pack_bf16_hw(lo_bf16(bv[v][2 + w]) + f * p2[2 * w], hi_bf16(bv[v][2 + w]) + f * p2[2 * w + 1]);
          }
        }
        if (((same >> r) & 1u) != 0u && in) write(v, x);
      }
      asm volatile("" ::: "memory");
    }
  }
}

// How a call's shrink is cut: 16-row tiles, rank tiles of a workgroup, slots, shares of K.
struct Shrink {
  int rt, xt, slots, splits;
  long long groups;  // (row tiles) x (rank groups) x slots
};
Shrink shrink_plan(int M, int K, int pr, int adapters) {
  Shrink p;
  p.xt = M <= 64 ? 1 : M >= 4096 && pr > 32 ? 4 : 2;
  p.rt = M <= 64 || pr <= 16 ? 1 : pr <= 32 ? 2 : 4;
  // One tile's distinct adapters over workgroups of their own where rows are few.
  p.slots = M <= 64 ? std::min({16, M, adapters}) : 1;
  p.groups = static_cast<long long>((M + 16 * p.xt - 1) / (16 * p.xt)) * ((pr + 16 * p.rt - 1) / (16 * p.rt)) * p.slots;
  const int units = K / (64 * kShrinkWaves);  // of 64, a wave's, in one share
  if (M <= 64) {  // 1024 workgroups where K gives them, every wave two units
    p.splits = static_cast<int>(std::max<long long>(1, std::min<long long>({kMaxShares, 1024 / p.groups, units / 2})));
    return p;
  }
  // Workgroups run in rounds of what the CUs hold, one each of the forms with four
  // rank tiles (registers) and two of the others. A workgroup's time is its share's
  // units and, about three units of each wave, its start, joins in LDS and sums to
  // memory: the number of shares that makes the least of rounds times that. us a call
  // with 1024 workgroups wherever K gives them and with the rule: 8192 x 12800 rank 64, 128 groups, 8 and 2 shares 124 and 105; 4096 rows
  // 78 and 66 (8, 4); 8192 x 4096, ranks 3 x 16, 89 and 68 (8, 2); 2048 rows, 3 x 32, 44 and 31.
  p.splits = 1;
  const long long held = p.rt == 4 ? kCUs : 2 * kCUs;
  long long least = LLONG_MAX;
  for (int s = 1; s <= std::min(kMaxShares, units) && (s == 1 || s * p.groups <= 1024); ++s) {
    const long long time = (s * p.groups + held - 1) / held * (K / 64 / s + 3 * kShrinkWaves);
    if (time < least) least = time, p.splits = s;
  }
  return p;
}
// The counts' place at the start of every workspace, whatever the call: shares
// are several only where groups are at most 512.
constexpr size_t kArrivedBytes = 512 * sizeof(unsigned);

template <int RT, int XT>
void launch_shrink(const LoraArgs& a, bool fp8, int slots, hipStream_t st) {
  const dim3 grid((a.M + 16 * XT - 1) / (16 * XT), (a.parts * a.rank + 16 * RT - 1) / (16 * RT) * a.splits, slots);
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

size_t t_elements(int M, int parts, int rank) {
  return static_cast<size_t>((M + 15) / 16) * parts * rank_steps(rank) * 512;
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" {

size_t granite4_lora_work_bytes(int M, int N, int K, int rank, int seg1, int seg2) {
  if (M <= 0 || N <= 0 || K <= 0 || rank <= 0) return 0;
  // Counts, the terms of t, the shares' sums (of the call with the most adapters).
  const int parts = parts_of(N, seg1, seg2), pr = parts * rank;
  size_t most = 0;
  for (int adapters = 1; adapters <= 16; ++adapters) {
    const Shrink p = shrink_plan(M, K, pr, adapters);
    const size_t part = p.splits > 1 ? static_cast<size_t>(M) * pr * p.splits * sizeof(float) : 0;
    most = std::max(most, kArrivedBytes + part + 3 * sizeof(uint16_t) * t_elements(M, parts, rank));
  }
  return most;
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
  const Shrink plan = shrink_plan(M, K, a.parts * rank, adapters);
  a.splits = plan.splits;
  a.arrived = static_cast<unsigned*>(work);
  a.t_pitch = t_elements(M, a.parts, rank);
  a.part = reinterpret_cast<float*>(static_cast<char*>(work) + kArrivedBytes);
  a.t = reinterpret_cast<uint16_t*>(a.part + (a.splits > 1 ? static_cast<size_t>(a.splits) * M * a.parts * rank : 0));
  a.terms = out == GRANITE4_GEMM_F32 ? 3 : 2;
  const hipStream_t st = stream();
  const int slots = plan.slots;
  if (plan.xt == 1) launch_shrink<1, 1>(a, fp8, slots, st);
  else if (plan.rt == 1) launch_shrink<1, 2>(a, fp8, 1, st);
  else if (plan.rt == 2) launch_shrink<2, 2>(a, fp8, 1, st);
  else if (plan.xt == 2) launch_shrink<4, 2>(a, fp8, 1, st);
  else launch_shrink<4, 4>(a, fp8, 1, st);
  // Row tiles of a wave: one where its columns of B are small beside the tile (rank
  // 16: 1001 x 25600 f32 50 us against 55 with six), else as many, up to eight, as
  // leave every CU four workgroups (rank 64, 8192 x 4096: 105 us the call with
  // eight, 112 with four, 121 with one).
  const long long wgs = static_cast<long long>((M + 15) / 16) * ((N + 255) / 256);
  const int per = rank <= 32 ? 1 : static_cast<int>(std::clamp<long long>(wgs / (4 * kCUs), 1, 8));
  const bool f32 = out == GRANITE4_GEMM_F32;
  const int steps = rank_steps(rank);
  if (steps == 1) launch_expand<1>(a, f32, per, slots, st);
  else if (steps == 2) launch_expand<2>(a, f32, per, slots, st);
  else launch_expand<4>(a, f32, per, slots, st);
  return launch_status("granite4_lora_add");
}

}  // extern "C"
