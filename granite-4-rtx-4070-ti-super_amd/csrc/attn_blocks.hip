// attn_blocks.hip - attention of query rows over the blocks listed for them.
//
// granite4_attn_blocks: row r at position p, KV head h and its four query
// heads attend to the positions <= p of the blocks that granite4_block_select
// (or the caller) listed for (r, h):
//   out = sum_t softmax_t(scale q . k_t) v_t
// over the listed positions t only, for every format of the pool.
//
// A list is a sequence of `block`-position slots; 64 consecutive slots make a
// tile, so a tile holds 4, 2, 1 or half a block and its keys lie wherever the
// page table puts them. One wave takes a tile with 16 MFMA columns, of which
// the four heads fill 4: rows share no lists, so there is nothing to put into
// the others, and a tile's bytes take longer than its products.
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, K rows through a stage of LDS (KStage)
//   O^T += V^T P^T  V through a row-major LDS tile, read transposed as the dense
//                   decode attention (attn.hip) does.
// The running maximum and sum
// and the logits stay in f32 (base 2, scale log2(e) folded into one factor); p
// is rounded to bf16 for the value product, after its row's V scale.
// Codes go into the products as they are: a scale group of K is one to four of
// the 32-channel products, whose sum it scales, and p takes the V scale of each
// group before its rounding, so no element of the cache is rounded again.
// The four waves of a workgroup join in LDS, the workgroups of a row (splits,
// where rows alone do not fill the chip) through memory, in the last of them.
#include "attn_kv.h"
#include "attn_rows.h"
#include "g4_common.h"
#include "g4_wave.h"
#include "granite4_layerops.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

namespace g4 {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxSplits = 32;

struct BlocksArgs {
  const uint16_t* q;   // [rows][Hq][128]
  const uint8_t* k;    // [Hk][stride][K row bytes]
  const uint8_t* v;
  const float* ksc;    // [Hk][stride][128 / group]
  const float* vsc;
  float scale2;        // scale * log2(e)
  int Hk, stride, first, rows;  // this launch's rows: first .. rows - 1
  RowSet at;
  const int32_t* sel;  // [rows][Hk][top_k]
  int top_k, log_block, splits;
  unsigned* arrived;   // [rows][Hk] workgroups of the row that are done; 0 between calls
  float2* part_ml;     // [rows][Hq][splits]
  float* part_o;       // [rows][Hq][splits][128]
  uint16_t* out;       // [rows][Hq][128]
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// K rows of 16 keys on their way from memory (16-byte chunks, consecutive lanes
// along a row) to fragments (lane n + 16 g: key n's channels 32 s + 8 g ..):
// through a stage of LDS that a wave has to itself. Straight from memory a
// quarter of a wave takes 16 bytes of each of 16 rows, 16 cache lines for 256
// bytes, and the CU's cache gives a quarter of its rate. The chunks of row r are
// exchanged (by r, r mod 8, r / 2 mod 4; K5 rows of 80 bytes need none), so that
// reads meet different banks.
template <int BITS>
struct KStage {
  static constexpr int kRow = k_row_bytes(BITS), kChunks = kRow / 16;  // per key: 16, 8, 4 or 5
  static constexpr int kLoads = (16 * kChunks + 63) / 64;
  static constexpr int kBytes = 16 * kRow;
  static __device__ __forceinline__ int slot(int key, int c) {
    if constexpr (BITS == 16) return c ^ key;
    else if constexpr (BITS == 8) return c ^ (key & 7);
    else if constexpr (BITS == 4) return c ^ ((key >> 1) & 3);
    else return c;
  }
  // Load i of the 16 keys from `first` on; row_of(key): its arena row (any, where it has none).
  template <class F>
  static __device__ __forceinline__ u32x4_t load(const uint8_t* kbase, int first, int i, F row_of) {
    const int id = i * 64 + (threadIdx.x & 63), key = min(id / kChunks, 15), c = id % kChunks;
    return *reinterpret_cast<const u32x4_t*>(kbase + static_cast<size_t>(row_of(first + key)) * kRow + 16 * c);
  }
  static __device__ __forceinline__ void put(uint8_t* stage, int i, const u32x4_t& v) {
    const int id = i * 64 + (threadIdx.x & 63), key = id / kChunks, c = id % kChunks;
    if (16 * kChunks % 64 == 0 || key < 16) *reinterpret_cast<u32x4_t*>(stage + key * kRow + 16 * slot(key, c)) = v;
  }
  // load_k_raw's form of key n, channels 32 s + 8 g ..
  static __device__ __forceinline__ u32x4_t get(const uint8_t* stage, int n, int s, int g) {
    const uint8_t* row = stage + n * kRow;
    u32x4_t r = {0u, 0u, 0u, 0u};
    if constexpr (BITS == 16) {
      r = *reinterpret_cast<const u32x4_t*>(row + 16 * slot(n, 4 * s + g));
    } else if constexpr (BITS == 8) {
      const u32x2_t v = *reinterpret_cast<const u32x2_t*>(row + 16 * slot(n, 2 * s + (g >> 1)) + 8 * (g & 1));
      r.x = v.x;
      r.y = v.y;
    } else {
      r.x = *reinterpret_cast<const uint32_t*>(row + 16 * slot(n, s) + 4 * g);
      if constexpr (BITS == 5) r.y = row[kHd / 2 + 4 * s + g];
    }
    return r;
  }
};

// Orders a wave's DS operations for the compiler; the hardware executes them in order.
__device__ __forceinline__ void ds_in_order() { asm volatile("" ::: "memory"); }

template <int BITS, int GROUP>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void attn_blocks_kernel(BlocksArgs a) {
  constexpr bool kQuant = BITS != 16;
  constexpr int kNgrp = kQuant ? kHd / GROUP : 1;
  constexpr int kSteps = 4 / kNgrp;  // 32-channel product steps per K scale
  constexpr int kKb = k_row_bytes(BITS), kVb = v_row_bytes(BITS);
  using KS = KStage<BITS>;
  constexpr bool kVDma = BITS == 16;  // V rows straight to LDS, without a pad
  // Per wave the V tile and the K stage; two workgroups fill a CU's 160 KB.
  constexpr int kVBytes = 2 * kTile * (kVDma ? kHd : kVPitch), kLdsWave = 20480;
  static_assert(kVBytes + KS::kBytes <= kLdsWave, "a wave's LDS");
  __shared__ __align__(16) uint8_t lds[kWaves][kLdsWave];
  static_assert(2 * kNgrp * sizeof(float) <= (kVPitch - kHd) * sizeof(uint16_t), "scales in the pad");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint16_t* vl = reinterpret_cast<uint16_t*>(lds[wave]);
  uint8_t* const stage = lds[wave] + kVBytes;
  float* const vlf = reinterpret_cast<float*>(vl);
  auto ksc_at = [&](int key, int gi) -> float& { return vlf[key * (kVPitch / 2) + kHd / 2 + gi]; };
  auto vsc_at = [&](int key, int gi) -> float& { return vlf[key * (kVPitch / 2) + kHd / 2 + 4 + gi]; };
  const int g = lane >> 4, n = lane & 15;
  const int h = blockIdx.x, split = blockIdx.z;
  const int row = a.first + blockIdx.y;
  const bool live = n < kGq;
  const long long pos = row_position(a.at, row);
  const int* pt = row_table(a.at, row);
  const g4_global_i32* ptg = (const g4_global_i32*)pt;
  const g4_global_i32* selg =
      (const g4_global_i32*)(a.sel + (static_cast<size_t>(row) * a.Hk + h) * a.top_k);
  const uint8_t* kbase = a.k + static_cast<size_t>(h) * a.stride * kKb;
  const uint8_t* vbase = a.v + static_cast<size_t>(h) * a.stride * kVb;
  const float* kscb = kQuant ? a.ksc + static_cast<size_t>(h) * a.stride * kNgrp : nullptr;
  const float* vscb = kQuant ? a.vsc + static_cast<size_t>(h) * a.stride * kNgrp : nullptr;
  // Positions that may be read: up to the row's own, inside the table.
  const int end = static_cast<int>(min(max(pos + 1, 0LL), static_cast<long long>(a.stride)));
  const long long slots = static_cast<long long>(a.top_k) << a.log_block;
  const int block_mask = (1 << a.log_block) - 1;
  // Arena row of this lane's slot of tile t: -1 past the list, for an entry
  // that names no block, behind the row's position and off the arena.
  auto slot_row = [&](long long t) -> int {
    const long long s = t * kTile + lane;
    const int id = s < slots ? selg[s >> a.log_block] : -1;
    const long long p = (static_cast<long long>(id) << a.log_block) + (s & block_mask);
    const bool ok = id >= 0 && p < end;
    const int r = ok ? (pt != nullptr ? ptg[p] : static_cast<int>(p)) : -1;
    return r >= 0 && r < a.stride ? r : -1;
  };
  const long long tiles = (slots + kTile - 1) / kTile;
  const int step = a.splits * kWaves;
  long long t = split * kWaves + wave;
  int prow_next = t < tiles ? slot_row(t) : -1;
  bf16x8_t qb[4];
  {
    const uint16_t* qp = a.q + (static_cast<size_t>(row) * kGq * a.Hk + kGq * h + (n & 3)) * kHd;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(qp + 32 * s + 8 * g);
      qb[s] = __builtin_bit_cast(bf16x8_t, live ? raw : u32x4_t{0u, 0u, 0u, 0u});
    }
  }
  f32x4_t o[8];
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  for (; t < tiles; t += step) {
    const int prow = prow_next;
    const unsigned long long kvalid = __ballot(prow >= 0);
    if (t + step < tiles) prow_next = slot_row(t + step);
    if (kvalid == 0ull) continue;
    // K and the scales first, then V, which lands while the logits are made.
    u32x4_t kraw[4][KS::kLoads];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < KS::kLoads; ++i)
        kraw[mb][i] = KS::load(kbase, 16 * mb, i, [&](int key) { return max(__shfl(prow, key), 0); });
    float ksr[kNgrp], vsr[kNgrp];
    if constexpr (kQuant) {
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        const size_t si = static_cast<size_t>(prow >= 0 ? prow : 0) * kNgrp + gi;
        ksr[gi] = kscb[si];
        vsr[gi] = vscb[si];
      }
    }
    u32x4_t vraw[VStage<BITS>::kSteps];
    if constexpr (kVDma) v_dma_bf16(vbase, prow, vl);
    else v_load<BITS>(vbase, prow, vraw);
    if constexpr (kQuant) {
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        ksc_at(lane, gi) = prow >= 0 ? ksr[gi] : 0.0f;
        vsc_at(lane, gi) = prow >= 0 ? vsr[gi] : 0.0f;
      }
    }
    // Keys 16 mb + 4 g + i of column n.
    float sv[4][4];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
      for (int i = 0; i < KS::kLoads; ++i) KS::put(stage, i, kraw[mb][i]);
      ds_in_order();
      bf16x8_t ka[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ka[s] = k_raw_bf16<BITS>(KS::get(stage, n, s, g));
      ds_in_order();
      // q . codes of each scale group, then its scale
      f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[kSteps * gi + s], qb[kSteps * gi + s], acc, 0, 0, 0);
        if constexpr (!kQuant) {
          x = acc;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = fmaf(acc[i], ksc_at(16 * mb + 4 * g + i, gi), x[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * mb + 4 * g + i;
        sv[mb][i] = live && ((kvalid >> key) & 1ull) ? a.scale2 * x[i] : -INFINITY;
      }
    }
    float mx = m;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sv[mb][i]);
    mx = col_max4(mx);
    // A column without a finite maximum yet keeps m = -inf, p = 0.
    const float alpha = mx == -INFINITY ? 1.0f : exp2_hw(m - mx);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) o[nb] *= alpha;
    float e[4][4];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[mb][i] = sv[mb][i] == -INFINITY ? 0.0f : exp2_hw(sv[mb][i] - m);
        l += e[mb][i];
      }
    if constexpr (kVDma) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      v_fix_bf16(vl, kvalid);
    } else {
      v_store<BITS>(vraw, vl, kvalid);
    }
    ds_in_order();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8_t pb[kNgrp];
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        float pv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int mb = 2 * s + (j >> 2), i = j & 3;
          pv[j] = e[mb][i] * (kQuant ? vsc_at(16 * mb + 4 * g + i, gi) : 1.0f);
        }
        pb[gi] = as_bf16x8(pack_bf16_hw(pv[0], pv[1]), pack_bf16_hw(pv[2], pv[3]), pack_bf16_hw(pv[4], pv[5]),
                           pack_bf16_hw(pv[6], pv[7]));
      }
      const int kk = n >> 2, dd = 4 * (n & 3);
      const int vrow = 32 * s + 4 * g + kk;
      const uint16_t* r1 = vl + vrow * (kVDma ? kHd : kVPitch) + dd;
      const uint16_t* r2 = r1 + 16 * (kVDma ? kHd : kVPitch);
      const int vt = vrow & 7;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        const int co = kVDma ? 16 * (nb ^ vt) : 16 * nb;
        const u32x2_t lo = lds_read_tr(r1 + co);
        const u32x2_t hi = lds_read_tr(r2 + co);
        o[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(lo.x, lo.y, hi.x, hi.y), pb[kQuant ? (16 * nb) / GROUP : 0],
                                                        o[nb], 0, 0, 0);
      }
    }
    wave_lds_sync();  // this tile's LDS reads are done before the next tile's writes
  }
  l = col_sum4(l);
  // The workgroup's waves joined: [wave][4 heads][128] and their (m, l).
  __syncthreads();
  float* mo = reinterpret_cast<float*>(&lds[0][0]);
  float* mml = mo + kWaves * kGq * kHd;
  if (live) {
#pragma unroll
    for (int nb = 0; nb < 8; ++nb)
      *reinterpret_cast<f32x4_t*>(mo + (wave * kGq + n) * kHd + 16 * nb + 4 * g) = o[nb];
    if (g == 0) {
      mml[(wave * kGq + n) * 2] = m;
      mml[(wave * kGq + n) * 2 + 1] = l;
    }
  }
  __syncthreads();
  // Wave w joins head w: lane c holds dims 2 c, 2 c + 1.
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mml[(w * kGq + wave) * 2]);
  float L = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = mml[(w * kGq + wave) * 2];
    const float wt = mw == -INFINITY ? 0.0f : exp2_hw(mw - M);
    const float2 ow = *reinterpret_cast<const float2*>(mo + (w * kGq + wave) * kHd + 2 * lane);
    L += mml[(w * kGq + wave) * 2 + 1] * wt;
    a0 += ow.x * wt;
    a1 += ow.y * wt;
  }
  const size_t rh = static_cast<size_t>(row) * kGq * a.Hk + kGq * h + wave;
  if (a.splits == 1) {
    // A row without a key gets zeros.
    const float inv = M == -INFINITY ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint32_t*>(a.out + rh * kHd + 2 * lane) = pack_bf16_hw(a0 * inv, a1 * inv);
    return;
  }
  const size_t at = rh * a.splits + split;
  if (lane == 0) st_dev_u64(a.part_ml + at, f2_bits(M, L));
  st_dev_u64(a.part_o + at * kHd + 2 * lane, f2_bits(a0, a1));
  // The last of the row's workgroups to arrive joins them all: none waits. The
  // join runs over the splits in order, whichever workgroup does it.
  unsigned& s_arrived = *reinterpret_cast<unsigned*>(&lds[kWaves - 1][0]);  // past the joined sums
  static_assert(sizeof(float) * kWaves * kGq * (kHd + 2) <= (kWaves - 1) * kLdsWave, "room for the count");
  wait_stores();
  __syncthreads();
  unsigned* count = a.arrived + static_cast<size_t>(row) * a.Hk + h;
  if (threadIdx.x == 0) s_arrived = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_arrived != static_cast<unsigned>(a.splits) - 1u) return;
  if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const float2* pml = a.part_ml + rh * a.splits;
  const float* po = a.part_o + rh * a.splits * kHd + 2 * lane;
  // Lane s (mod 32) has split s's maximum and sum; eight splits' sums load at once.
  static_assert(kMaxSplits <= 32, "a lane per split");
  const unsigned long long mlb = ld_dev_u64(pml + min(lane & 31, a.splits - 1));
  const float ms = __uint_as_float(static_cast<unsigned>(mlb)), ls = __uint_as_float(static_cast<unsigned>(mlb >> 32));
  const float Mall = wave_max(ms);  // repeated lanes change no maximum
  const float ws = ms == -INFINITY ? 0.0f : exp2_hw(ms - Mall);
  L = a0 = a1 = 0.0f;
#pragma unroll 1
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    unsigned long long ov[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) ov[j] = ld_dev_u64(po + static_cast<size_t>(min(s0 + j, a.splits - 1)) * kHd);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (s0 + j < a.splits) {
        const float wt = readlane_f32(ws, s0 + j);
        L += readlane_f32(ls, s0 + j) * wt;
        a0 += __uint_as_float(static_cast<unsigned>(ov[j])) * wt;
        a1 += __uint_as_float(static_cast<unsigned>(ov[j] >> 32)) * wt;
      }
    }
  }
  const float inv = Mall == -INFINITY ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint32_t*>(a.out + rh * kHd + 2 * lane) = pack_bf16_hw(a0 * inv, a1 * inv);
}

// Workgroups per (row, KV head): enough to give every CU two, each of its
// waves at least one tile.
int blocks_splits(int rows, int Hk, int top_k, int block) {
  const long long tiles = (static_cast<long long>(top_k) * block + kTile - 1) / kTile;
  const long long most = std::min<long long>(kMaxSplits, (tiles + kWaves - 1) / kWaves);
  const long long want = (2 * kCUs + static_cast<long long>(rows) * Hk - 1) / (static_cast<long long>(rows) * Hk);
  return static_cast<int>(std::max<long long>(1, std::min(most, want)));
}

template <int BITS>
void launch_blocks(const BlocksArgs& a, int group, dim3 grid, hipStream_t st) {
  if constexpr (BITS == 16) {
    hipLaunchKernelGGL((attn_blocks_kernel<16, kHd>), grid, kWaves * 64, 0, st, a);
  } else {
    if (group == 32) hipLaunchKernelGGL((attn_blocks_kernel<BITS, 32>), grid, kWaves * 64, 0, st, a);
    else if (group == 64) hipLaunchKernelGGL((attn_blocks_kernel<BITS, 64>), grid, kWaves * 64, 0, st, a);
    else hipLaunchKernelGGL((attn_blocks_kernel<BITS, kHd>), grid, kWaves * 64, 0, st, a);
  }
}

// The counts' place at the start of every scratch, whatever the call: splits are
// several only below 512 (row, KV head) pairs.
constexpr size_t kArrivedBytes = 2 * kCUs * sizeof(unsigned);

constexpr int kSlab = 65535;  // rows of one launch (grid.y)

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" {

size_t granite4_attn_blocks_scratch_bytes(int Hq, int rows, int top_k, int block) {
  if (Hq <= 0 || Hq % kGq != 0 || rows <= 0 || top_k <= 0 || block <= 0) return 0;
  const int splits = blocks_splits(rows, Hq / kGq, top_k, block);
  return splits == 1 ? 0
                     : kArrivedBytes +
                           static_cast<size_t>(rows) * Hq * splits * (sizeof(float2) + kHd * sizeof(float));
}

int granite4_attn_blocks(const uint16_t* q, int rows, int Hq, int Hk, int d, float scale,
                         const void* cache_k, const void* cache_v, const float* k_scale,
                         const float* v_scale, int bits, int group, int stride, int kv_base,
                         const int* d_pos, const int* d_pt, const int* row_pos,
                         const int* const* row_pt, const int32_t* sel, int top_k, int block,
                         void* scratch, uint16_t* out) {
  BlocksArgs a{};
  a.at = RowSet{kv_base, d_pos, d_pt, row_pos, row_pt};
  if (q == nullptr || cache_k == nullptr || cache_v == nullptr || sel == nullptr ||
      out == nullptr || !std::isfinite(scale) || d != kHd || Hk <= 0 || Hq != kGq * Hk ||
      !block_ok(block, stride) || !row_set_ok(a.at, rows, stride) || top_k < 1 ||
      !aligned(q, 16) || !aligned(cache_k, 16) || !aligned(cache_v, 16) || !aligned(scratch, 16) ||
      !aligned(out, 4) || (bits != 16 && bits != 8 && bits != 4 && bits != 5) ||
      (bits != 16 && (k_scale == nullptr || v_scale == nullptr ||
                      (group != 32 && group != 64 && group != kHd))) ||
      (scratch == nullptr && granite4_attn_blocks_scratch_bytes(Hq, rows, top_k, block) > 0)) {
    std::fprintf(stderr, "granite4: granite4_attn_blocks: invalid arguments\n");
    return -1;
  }
  a.k = static_cast<const uint8_t*>(cache_k);
  a.v = static_cast<const uint8_t*>(cache_v);
  a.ksc = k_scale;
  a.vsc = v_scale;
  a.scale2 = scale * kLog2E;
  a.Hk = Hk;
  a.stride = stride;
  a.top_k = top_k;
  a.log_block = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  a.splits = blocks_splits(rows, Hk, top_k, block);  // 1 from 64 rows of 8 KV heads on
  const hipStream_t st = stream();
  a.q = q;
  a.sel = sel;
  a.out = out;
  if (a.splits > 1) {  // below 512 (row, KV head) pairs: one launch
    a.arrived = static_cast<unsigned*>(scratch);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + kArrivedBytes);
    a.part_o = reinterpret_cast<float*>(a.part_ml + static_cast<size_t>(rows) * Hq * a.splits);
  }
  for (int r0 = 0; r0 < rows; r0 += std::min(kSlab, rows - r0)) {
    a.first = r0;
    a.rows = r0 + std::min(kSlab, rows - r0);
    const dim3 grid(Hk, a.rows - r0, a.splits);
    switch (bits) {
      case 16: launch_blocks<16>(a, group, grid, st); break;
      case 8: launch_blocks<8>(a, group, grid, st); break;
      case 4: launch_blocks<4>(a, group, grid, st); break;
      default: launch_blocks<5>(a, group, grid, st); break;
    }
  }
  return launch_status("granite4_attn_blocks");
}

}  // extern "C"
