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
// the four heads fill 4: a tile's bytes take longer than its products.
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, K rows through a stage of LDS (KStage)
//   O^T += V^T P^T  V through a row-major LDS tile, read transposed as the dense
//                   decode attention (attn.hip) does.
// Q stands in the columns four times, so that each lane gets all logits of its head's
// 64 keys four times over and keeps a fourth: the softmax is done once, not on 12
// idle columns too, and p goes to the head's first column by three lane rotations.
// The running maximum and sum and the logits stay in f32 (base 2, scale log2(e) folded into one factor); p
// is rounded to bf16 for the value product, after its row's V scale.
// Codes go into the products as they are: a scale group of K is one to four of
// the 32-channel products, whose sum it scales, and p takes the V scale of each
// group before its rounding, so no element of the cache is rounded again.
// Forms, by the rows there are (own_rows, merge_rows): a workgroup a row, whose four
// waves join in LDS and whose workgroups (splits, where rows alone do not fill the
// chip) join through memory, in the last of them; a wave a row; and for bf16 a wave
// over one to four rows (attn_blocks_merged_kernel). 8 KV heads, times a call:
//   1 row, 32 blocks of 64 of int8       7.6 us (host 5.9): the launch, list, table, K, V, join in turn
//   16 rows, 64 blocks of 32 of K5 / 32  16.9 us: codes into products, scales; with K's
//                                        codes converted to bf16 19.6, with the next
//                                        tile loaded only when this is done 17.3
//   511 rows, 32 of 640 blocks of 64     bf16 229 us, int8 222, K5 / 32 284
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
    const int lane = threadIdx.x & 63, c = (i * 64 + lane) % kChunks;
    const int key = 64 % kChunks == 0 ? 64 / kChunks * i + lane / kChunks : min((i * 64 + lane) / kChunks, 15);
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

// K codes of 4 and 5 bits go into the products without a conversion: n in [0, 2^b)
// set into the mantissa of 16 (32 for K5) is the bf16 16 + n (32 + n) exactly, two
// of them per shift and and-or. The code is n - 8 (n - 16), so the sums start at
// -24 (-48) times the sum of q. A pair is elements e and e + 4 of eight, and q is
// exchanged the same way. V's codes are converted: a sum that cancels 24 times the
// sum of p would lose what a dim of small codes is made of.
template <int BITS>
constexpr bool kPaired = BITS == 4 || BITS == 5;
constexpr uint16_t kMinus24 = 0xC1C0, kMinus48 = 0xC240;  // bf16

__device__ __forceinline__ uint32_t nibble_pair(uint32_t x, int e, int at) {  // nibbles e and e + 4 at bits at, 16 + at
  const uint32_t y = 4 * e >= at ? x >> (4 * e - at) : x << (at - 4 * e);
  return y & (0x000F000Fu << at);
}
__device__ __forceinline__ bf16x8_t paired4(uint32_t x) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = nibble_pair(x, e, 3) | 0x41804180u;
  return as_bf16x8(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ bf16x8_t paired5(uint32_t x, uint32_t high) {
  // high bit i to bits 6 + i and 18 + i, so that e and e + 4 are at 6 + e and 22 + e
  const uint32_t t = __umul24(high, (1u << 6) | (1u << 18));
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = nibble_pair(x, e, 2) | 0x42004200u | ((t >> e) & 0x00400040u);
  return as_bf16x8(w[0], w[1], w[2], w[3]);
}
template <int BITS>
__device__ __forceinline__ bf16x8_t k_frag(const u32x4_t& r) {
  if constexpr (BITS == 4) return paired4(r.x);
  else if constexpr (BITS == 5) return paired5(r.x, r.y);
  else return k_raw_bf16<BITS>(r);
}
// q's eight elements in that order.
__device__ __forceinline__ u32x4_t pair_order(const u32x4_t& w) {
  return u32x4_t{(w.x & 0xffffu) | (w.z << 16), (w.x >> 16) | (w.z & 0xffff0000u), (w.y & 0xffffu) | (w.w << 16),
                 (w.y >> 16) | (w.w & 0xffff0000u)};
}
__device__ __forceinline__ bf16x8_t bf16_all(uint16_t v) {
  const uint32_t w = v * 0x10001u;
  return as_bf16x8(w, w, w, w);
}
// x of the lane N columns on (mod 16) among 16 columns.
template <int N>
__device__ __forceinline__ unsigned column_on(unsigned x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x120 + 16 - N, 0xf, 0xf, true);  // row_ror
}
template <int N>
__device__ __forceinline__ float column_on_f32(float x) {
  return __uint_as_float(column_on<N>(__float_as_uint(x)));
}

template <int BITS, int GROUP, bool OWN>
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
  const int row = a.first + (OWN ? blockIdx.y * kWaves + wave : blockIdx.y);
  if (OWN && row >= a.rows) return;
  const int j = n >> 2;  // of 64 keys this column's sixteen
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
  // This lane's list entry of tile t, and the arena row it makes: -1 past the list,
  // for an entry that names no block, behind the row's position and off the arena.
  auto entry = [&](long long t) -> int {
    const long long s = t * kTile + lane;
    return s < slots ? selg[s >> a.log_block] : -1;
  };
  auto slot_row = [&](long long t, int id) -> int {
    const long long p = (static_cast<long long>(id) << a.log_block) + ((t * kTile + lane) & block_mask);
    const bool ok = id >= 0 && p < end;
    const int r = ok ? (pt != nullptr ? ptg[p] : static_cast<int>(p)) : -1;
    return r >= 0 && r < a.stride ? r : -1;
  };
  const long long tiles = (slots + kTile - 1) / kTile;
  const int step = OWN ? 1 : a.splits * kWaves;
  long long t = OWN ? 0 : split * kWaves + wave;
  // The list is read two tiles ahead, the table one, K, V and scales of codes (a
  // quarter of the registers that bf16 takes) as soon as a tile has used its own.
  int prow = slot_row(t, entry(t)), id_next = entry(t + step);
  bf16x8_t qb[4];
  {
    const uint16_t* qp = a.q + (static_cast<size_t>(row) * kGq * a.Hk + kGq * h + (n & 3)) * kHd;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(qp + 32 * s + 8 * g);
      qb[s] = __builtin_bit_cast(bf16x8_t, kPaired<BITS> ? pair_order(raw) : raw);
    }
  }
  f32x4_t kinit[kNgrp];  // paired codes: -off times the sum of q
#pragma unroll
  for (int gi = 0; gi < kNgrp; ++gi) {
    kinit[gi] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (kPaired<BITS>) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        kinit[gi] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_all(BITS == 5 ? kMinus48 : kMinus24),
                                                            qb[kSteps * gi + s], kinit[gi], 0, 0, 0);
    }
  }
  f32x4_t o[8];
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  u32x4_t kraw[4][KS::kLoads], vraw[VStage<BITS>::kSteps];
  float ksr[kNgrp], vsr[kNgrp];
  auto load_k = [&](int of) {
    const int at = max(of, 0);
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < KS::kLoads; ++i)
        kraw[mb][i] = KS::load(kbase, 16 * mb, i, [&](int key) { return __shfl(at, key); });
    if constexpr (kQuant) {
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        ksr[gi] = kscb[static_cast<size_t>(at) * kNgrp + gi];
        vsr[gi] = vscb[static_cast<size_t>(at) * kNgrp + gi];
      }
    }
  };
  auto skip_empty = [&]() {
    while (t < tiles && __ballot(prow >= 0) == 0ull) {
      t += step;
      prow = slot_row(t, kQuant ? id_next : entry(t));
      if (kQuant) id_next = entry(t + step);
    }
  };
  skip_empty();
  if (kQuant && t < tiles) {
    load_k(prow);
    if constexpr (kQuant) v_load<BITS>(vbase, prow, vraw);
  }
  while (t < tiles) {
    const unsigned long long kvalid = __ballot(prow >= 0);
    const int mine = prow;
    if constexpr (!kQuant) {
      t += step;
      prow = slot_row(t, entry(t));
      load_k(mine);
      v_dma_bf16(vbase, mine, vl);
    } else {
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        ksc_at(lane, gi) = prow >= 0 ? ksr[gi] : 0.0f;
        vsc_at(lane, gi) = prow >= 0 ? vsr[gi] : 0.0f;
      }
      t += step;
      prow = slot_row(t, id_next);
      id_next = entry(t + step);
    }
    // q . codes of each scale group: of the 64 keys that every column of a head
    // gets, this one keeps 16 j + 4 g + i.
    float x[kNgrp][4];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
      for (int i = 0; i < KS::kLoads; ++i) KS::put(stage, i, kraw[mb][i]);
      ds_in_order();
      bf16x8_t ka[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ka[s] = k_frag<BITS>(KS::get(stage, n, s, g));
      ds_in_order();
#pragma unroll
      for (int gi = 0; gi < kNgrp; ++gi) {
        f32x4_t acc = kinit[gi];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[kSteps * gi + s], qb[kSteps * gi + s], acc, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[gi][i] = mb == 0 || j == mb ? acc[i] : x[gi][i];
      }
    }
    skip_empty();
    if (kQuant && t < tiles) load_k(prow);
    const int key0 = 16 * j + 4 * g;
    const unsigned seen = static_cast<unsigned>(kvalid >> key0);
    float e[4];
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y = x[0][i];
      if constexpr (kQuant) {
        y = 0.0f;
#pragma unroll
        for (int gi = 0; gi < kNgrp; ++gi) y = fmaf(x[gi][i], ksc_at(key0 + i, gi), y);
      }
      e[i] = ((seen >> i) & 1u) != 0u ? a.scale2 * y : -INFINITY;
      mx = fmaxf(mx, e[i]);
    }
    mx = col_max4(mx);
    mx = fmaxf(mx, column_on_f32<8>(mx));
    mx = fmaxf(mx, column_on_f32<4>(mx));
    // Without a finite maximum yet every p is 0: exp2(-inf), not of -inf - -inf.
    const float base = mx == -INFINITY ? 0.0f : mx;
    const float alpha = exp2_hw(m - base);
    m = mx;
    l *= alpha;
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nb] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = exp2_hw(e[i] - base);
      l += e[i];
    }
    if constexpr (kVDma) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      v_fix_bf16(vl, kvalid);
    } else {
      // A key without a row needs no zeros: its p and scale are 0, every code is finite.
      v_store<BITS>(vraw, vl, ~0ull);
      if (t < tiles) v_load<BITS>(vbase, prow, vraw);
    }
    ds_in_order();
    // p times the V scale of each group, and from the columns 4, 8 and 12 on what
    // a head's first column needs of the keys 16 .. 63 (the other columns' products
    // are not read).
    bf16x8_t pb[2][kNgrp];
#pragma unroll
    for (int gi = 0; gi < kNgrp; ++gi) {
      float pv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = kQuant ? e[i] * vsc_at(key0 + i, gi) : e[i];
      const unsigned p0 = pack_bf16_hw(pv[0], pv[1]), p1 = pack_bf16_hw(pv[2], pv[3]);
      pb[0][gi] = as_bf16x8(p0, p1, column_on<4>(p0), column_on<4>(p1));
      pb[1][gi] = as_bf16x8(column_on<8>(p0), column_on<8>(p1), column_on<12>(p0), column_on<12>(p1));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
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
        o[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(lo.x, lo.y, hi.x, hi.y), pb[s][kQuant ? (16 * nb) / GROUP : 0],
                                                        o[nb], 0, 0, 0);
      }
    }
    wave_lds_sync();  // this tile's LDS reads are done before the next tile's writes
  }
  l = col_sum4(l);
  l += column_on_f32<8>(l);
  l += column_on_f32<4>(l);
  // o[nb]'s dims: 16 nb + od, od + 1, od + on, od + on + 1.
  const int od = 4 * g;
  constexpr int on = 2;
  if constexpr (OWN) {  // a row without a key gets zeros
    if (live) {
      const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
      uint16_t* dst = a.out + (static_cast<size_t>(row) * kGq * a.Hk + kGq * h + n) * kHd + od;
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        *reinterpret_cast<uint32_t*>(dst + 16 * nb) = pack_bf16_hw(o[nb][0] * inv, o[nb][1] * inv);
        *reinterpret_cast<uint32_t*>(dst + 16 * nb + on) = pack_bf16_hw(o[nb][2] * inv, o[nb][3] * inv);
      }
    }
    return;
  }
  // The workgroup's waves joined: [wave][4 heads][128] and their (m, l).
  __syncthreads();
  float* mo = reinterpret_cast<float*>(&lds[0][0]);
  float* mml = mo + kWaves * kGq * kHd;
  if (live) {
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      float* dst = mo + (wave * kGq + n) * kHd + 16 * nb + od;
      *reinterpret_cast<float2*>(dst) = float2{o[nb][0], o[nb][1]};
      *reinterpret_cast<float2*>(dst + on) = float2{o[nb][2], o[nb][3]};
    }
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

// ---------------------------------------------------------------------------
// Many rows of one sequence over a bf16 cache: a wave takes up to four consecutive
// rows of a KV head, a row in four of the 16 columns, and goes through their lists
// together, next the lowest block that any of them has next. Rows that list the same
// block read it once, and the waves of a head (an XCD's, for 8 KV heads) move along
// the sequence together, so that a block that one has read is still in the XCD's
// cache when the others come to it. 511 rows, 32 of 640 blocks of 64 at random, 8 KV
// heads, 4.3 GB asked for: a workgroup a row 378 us (two of five lines come from the
// XCD's cache), a wave a row 282 (three of five), two rows a wave 229; 1000 rows, four a
// wave: 785, 585, 385. With all blocks in that cache 160; the loads alone 234 (a wave
// a row) and 140. K of the next tile is under way while this one's p and products
// are made, V while its logits are: loads through buffer descriptors, since behind a
// global_load_lds the compiler has every load waited for.
// ---------------------------------------------------------------------------
constexpr int kMergeRows = 4;
constexpr int kMergeStride = 1 << 24;  // arena rows whose bytes a 32-bit offset reaches

// A head's bf16 rows.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_buffer(const uint8_t* p, int stride) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, static_cast<int>(static_cast<unsigned>(stride) * 256u),
                                           0x00020000);
}

__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void attn_blocks_merged_kernel(BlocksArgs a, int per_wave) {
  using KS = KStage<16>;
  constexpr int kVBytes = 2 * kTile * kHd;
  __shared__ __align__(16) uint8_t lds[kWaves][kVBytes + KS::kBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint16_t* vl = reinterpret_cast<uint16_t*>(lds[wave]);
  uint8_t* const stage = lds[wave] + kVBytes;
  const int g = lane >> 4, n = lane & 15, c = n >> 2;
  const int h = blockIdx.x;
  const int row0 = a.first + (blockIdx.y * kWaves + wave) * per_wave;
  const int nr = min(per_wave, a.rows - row0);
  if (nr <= 0) return;
  const int* pt = a.at.d_pt;  // one sequence
  const g4_global_i32* ptg = (const g4_global_i32*)pt;
  const uint8_t* kbase = a.k + static_cast<size_t>(h) * a.stride * k_row_bytes(16);
  const uint8_t* vbase = a.v + static_cast<size_t>(h) * a.stride * v_row_bytes(16);
  // Positions that each row may read, up to its own.
  int end[kMergeRows];
#pragma unroll
  for (int r = 0; r < kMergeRows; ++r) {
    const long long pos = row_position(a.at, row0 + min(r, nr - 1));
    end[r] = __builtin_amdgcn_readfirstlane(static_cast<int>(min(max(pos + 1, 0LL), static_cast<long long>(a.stride))));
  }
  // 64 entries of each list in the lanes, those not taken yet that the row sees in
  // `left`, the place of the first in `at`; `id`: the row's next block.
  int ids[kMergeRows], from[kMergeRows], id[kMergeRows];
  unsigned long long left[kMergeRows];
  auto advance = [&](int r) {
    const g4_global_i32* lst = (const g4_global_i32*)(a.sel + (static_cast<size_t>(row0 + r) * a.Hk + h) * a.top_k);
    while (left[r] == 0ull && from[r] < a.top_k) {
      ids[r] = from[r] + lane < a.top_k ? lst[from[r] + lane] : -1;
      left[r] = __ballot(ids[r] >= 0 && (static_cast<long long>(ids[r]) << a.log_block) < end[r]);
      from[r] += 64;
    }
    id[r] = left[r] == 0ull ? INT_MAX : __builtin_amdgcn_readlane(ids[r], __builtin_ctzll(left[r]));
    left[r] &= left[r] - 1;
  };
#pragma unroll
  for (int r = 0; r < kMergeRows; ++r) {
    left[r] = 0ull;
    from[r] = r < nr ? 0 : a.top_k;
    ids[r] = -1;
    advance(r);
  }
  // The block after the one in hand: the rows that take it (together only where each
  // sees all of it: what a row does not see must not be a factor of its 0), its first
  // position, where what they see ends, and this lane's table entry.
  int who = 0, pos0 = 0, part = 0, most = 0, prow = -1;
  const int parts = 1 << (a.log_block - 6);
  auto next_tile = [&]() {
    if (who != 0 && ++part < parts && pos0 + kTile < most) {
      pos0 += kTile;
    } else {
      part = 0;
      const int b = min(min(id[0], id[1]), min(id[2], id[3]));
      who = most = 0;
      if (b == INT_MAX) return;
      pos0 = b << a.log_block;
      const int past = min(pos0 + (1 << a.log_block), a.stride);
#pragma unroll
      for (int r = 0; r < kMergeRows; ++r)
        if (id[r] == b && (who == 0 || (most == past && end[r] >= past))) {
          who |= 1 << r;
          most = min(end[r], past);
          advance(r);
        }
    }
    const int p = pos0 + lane;
    prow = p < most ? (pt != nullptr ? ptg[p] : p) : -1;
  };
  // This lane's arena row of a tile, and the tile's first where all 64 lie side by side
  // (-1 where not): looked at when the table's load has landed.
  int crow = -1, cbase = -1;
  unsigned long long kvalid = 0ull;
  auto take_rows = [&]() {
    crow = prow >= 0 && prow < a.stride ? prow : -1;
    kvalid = __ballot(crow >= 0);
    cbase = __builtin_amdgcn_readfirstlane(crow);
    if (cbase < 0 || cbase > a.stride - kTile || __ballot(crow >= 0 && crow != cbase + lane) != 0ull) cbase = -1;
  };
  bf16x8_t qb[4];
  {
    const uint16_t* qp = a.q + (static_cast<size_t>(row0 + min(c, nr - 1)) * kGq * a.Hk + kGq * h + (n & 3)) * kHd;
#pragma unroll
    for (int s = 0; s < 4; ++s) qb[s] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(qp + 32 * s + 8 * g));
  }
  f32x4_t o[8];
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  // Lane: chunk lane % 16 of key 4 i + lane / 16.
  const __amdgpu_buffer_rsrc_t kbuf = head_buffer(kbase, a.stride), vbuf = head_buffer(vbase, a.stride);
  u32x4_t kraw[16];
  // Bytes of the arena rows whose pieces this lane loads, keys 4 i + g.
  unsigned at[16];
  auto load_k = [&]() {
    if (cbase >= 0) {
      const unsigned first = (cbase + g) * 256u;
#pragma unroll
      for (int i = 0; i < 16; ++i) at[i] = first + 1024u * i;
    } else {
      const int r = max(crow, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) at[i] = __shfl(r, 4 * i + g) * 256u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) kraw[i] = __builtin_amdgcn_raw_buffer_load_b128(kbuf, at[i] + 16 * n, 0, 0);
  };
  // V, as v_dma_bf16 but by instructions that the compiler counts one by one.
  auto load_v = [&]() {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vbuf, (lds_ptr_t)(lds[wave] + 1024 * i), 16,
                                               at[i] + 16 * (n ^ v_swz(4 * i + g)), 0, 0, 0);
  };
  next_tile();
  take_rows();
  if (who != 0) load_k();
  while (who != 0) {
    const int cwho = who, cpos = pos0;
    const unsigned long long keys = kvalid;
    next_tile();
    ds_in_order();
    load_v();  // lands while the logits are made
    ds_in_order();
    // Keys 16 mb + 4 g + i of column n, where its row lists the block (and then sees
    // every key that was loaded).
    const bool takes = ((cwho >> c) & 1) != 0;
    const unsigned long long seen = takes ? keys >> (4 * g) : 0ull;
    float e[4][4];
    float mx = m;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
      for (int i = 0; i < KS::kLoads; ++i) KS::put(stage, i, kraw[4 * mb + i]);
      ds_in_order();
      f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k_raw_bf16<16>(KS::get(stage, n, s, g)), qb[s], acc, 0, 0, 0);
      ds_in_order();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[mb][i] = ((seen >> (16 * mb + i)) & 1ull) != 0ull ? a.scale2 * acc[i] : -INFINITY;
        mx = fmaxf(mx, e[mb][i]);
      }
    }
    ds_in_order();
    take_rows();
    load_k();  // sixteen loads, of the next tile (of row 0 after the last)
    ds_in_order();
    mx = col_max4(mx);
    // Without a finite maximum yet every p is 0: exp2(-inf), not of -inf - -inf.
    const float base = mx == -INFINITY ? 0.0f : mx;
    const float alpha = exp2_hw(m - base);
    m = mx;
    l *= alpha;
    if (__any(takes && alpha != 1.0f)) {  // the others' is 1, or 0 with sums of 0
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) o[nb] *= alpha;
    }
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[mb][i] = exp2_hw(e[mb][i] - base);
        l += e[mb][i];
      }
    // V has landed; the next tile's K need not.
    asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    v_fix_bf16(vl, keys);
    ds_in_order();
    bf16x8_t pb[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
      pb[s] = as_bf16x8(pack_bf16_hw(e[2 * s][0], e[2 * s][1]), pack_bf16_hw(e[2 * s][2], e[2 * s][3]),
                        pack_bf16_hw(e[2 * s + 1][0], e[2 * s + 1][1]), pack_bf16_hw(e[2 * s + 1][2], e[2 * s + 1][3]));
    const int vr = 4 * g + (n >> 2), vt = vr & 7;
    const uint16_t* v0 = vl + vr * kHd + 4 * (n & 3);
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      f32x4_t x = o[nb];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x2_t lo = lds_read_tr(v0 + 32 * s * kHd + 16 * (nb ^ vt));
        const u32x2_t hi = lds_read_tr(v0 + (32 * s + 16) * kHd + 16 * (nb ^ vt));
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(lo.x, lo.y, hi.x, hi.y), pb[s], x, 0, 0, 0);
      }
      // A row that does not list the block stays: 0 times V is NaN where V is not finite.
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nb][i] = takes ? x[i] : o[nb][i];
    }
    wave_lds_sync();  // this tile's LDS reads are done before the next tile's writes
  }
  l = col_sum4(l);
  if (c >= nr) return;
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;  // a row without a key gets zeros
  uint16_t* dst = a.out + (static_cast<size_t>(row0 + c) * kGq * a.Hk + kGq * h + (n & 3)) * kHd + 4 * g;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) {
    *reinterpret_cast<uint32_t*>(dst + 16 * nb) = pack_bf16_hw(o[nb][0] * inv, o[nb][1] * inv);
    *reinterpret_cast<uint32_t*>(dst + 16 * nb + 2) = pack_bf16_hw(o[nb][2] * inv, o[nb][3] * inv);
  }
}

// Workgroups per (row, KV head): enough to give every CU two, each of its
// waves at least one tile.
int blocks_splits(int rows, int Hk, int top_k, int block) {
  const long long tiles = (static_cast<long long>(top_k) * block + kTile - 1) / kTile;
  const long long most = std::min<long long>(kMaxSplits, (tiles + kWaves - 1) / kWaves);
  const long long want = (2 * kCUs + static_cast<long long>(rows) * Hk - 1) / (static_cast<long long>(rows) * Hk);
  return static_cast<int>(std::max<long long>(1, std::min(most, want)));
}

template <int BITS, int GROUP>
void launch_form(const BlocksArgs& a, bool own, hipStream_t st) {
  const int n = a.rows - a.first;
  if (own) {
    hipLaunchKernelGGL((attn_blocks_kernel<BITS, GROUP, true>), dim3(a.Hk, (n + kWaves - 1) / kWaves), kWaves * 64, 0, st, a);
  } else {
    hipLaunchKernelGGL((attn_blocks_kernel<BITS, GROUP, false>), dim3(a.Hk, n, a.splits), kWaves * 64, 0, st, a);
  }
}

template <int BITS>
void launch_blocks(const BlocksArgs& a, int group, bool own, hipStream_t st) {
  if constexpr (BITS == 16) {
    launch_form<16, kHd>(a, own, st);
  } else {
    if (group == 32) launch_form<BITS, 32>(a, own, st);
    else if (group == 64) launch_form<BITS, 64>(a, own, st);
    else launch_form<BITS, kHd>(a, own, st);
  }
}

constexpr long long kWaveSlots = 8 * kCUs;  // two workgroups of four waves a CU

// A wave for each (row, KV head), rather than a workgroup. bf16, which memory bounds:
// from three quarters of the chip's waves on (512 rows of 4 blocks of 16, 8 KV heads: 20
// against 41 us). Codes, which the waves' work bounds: where the last round of waves is
// nearly full (511 rows, 8 KV heads, 32 blocks of 64: int8 220 against 232 us, K5 in
// groups of 32 284 against 294; 300 rows of those 220 against 183).
bool own_rows(long long pairs, int bits) {
  if (bits == 16) return 4 * pairs >= 3 * kWaveSlots;
  const long long slots = (pairs + kWaveSlots - 1) / kWaveSlots * kWaveSlots;
  return 16 * (slots - pairs) <= pairs;
}
// Rows of a wave of the merged form, 0 where it is not taken: as many as make one
// round of waves. A round takes the time of its tiles one after another, so it is the
// faster form from half the chip's waves on (32 of 640 blocks of 64, 8 KV heads: 128
// rows 80 against 91 us with a workgroup a row, 96 rows 80 against 72, 64 rows 79 against 45).
int merge_rows(long long pairs) {
  if (2 * pairs < kWaveSlots) return 0;
  return static_cast<int>(std::min<long long>(kMergeRows, (pairs + kWaveSlots - 1) / kWaveSlots));
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
  a.splits = blocks_splits(rows, Hk, top_k, block);  // 1 from 512 (row, KV head) pairs on
  const hipStream_t st = stream();
  a.q = q;
  a.sel = sel;
  a.out = out;
  if (a.splits > 1) {  // below 512 (row, KV head) pairs: one launch
    a.arrived = static_cast<unsigned*>(scratch);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + kArrivedBytes);
    a.part_o = reinterpret_cast<float*>(a.part_ml + static_cast<size_t>(rows) * Hq * a.splits);
  }
  const long long pairs = static_cast<long long>(rows) * Hk;
  const bool own = own_rows(pairs, bits);
  const int merge =
      bits == 16 && block >= kTile && row_pt == nullptr && stride < kMergeStride ? merge_rows(pairs) : 0;
  for (int r0 = 0; r0 < rows; r0 += std::min(kSlab, rows - r0)) {
    a.first = r0;
    a.rows = r0 + std::min(kSlab, rows - r0);
    if (merge > 0) {
      const int waves = (a.rows - r0 + merge - 1) / merge;
      hipLaunchKernelGGL(attn_blocks_merged_kernel, dim3(Hk, (waves + kWaves - 1) / kWaves), kWaves * 64, 0, st, a,
                         merge);
      continue;
    }
    switch (bits) {
      case 16: launch_blocks<16>(a, group, own, st); break;
      case 8: launch_blocks<8>(a, group, own, st); break;
      case 4: launch_blocks<4>(a, group, own, st); break;
      default: launch_blocks<5>(a, group, own, st); break;
    }
  }
  return launch_status("granite4_attn_blocks");
}

}  // extern "C"
