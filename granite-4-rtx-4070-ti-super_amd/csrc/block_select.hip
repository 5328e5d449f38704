// block_select.hip - which blocks of a long context a query row attends to.
//
// granite4_kv_ranges     per completed block of `block` positions and KV head,
//                        the smallest and largest cached value of each of the
//                        128 channels, as 8-bit codes under one scale.
// granite4_block_select  per query row and KV head, the blocks whose ranges
//                        allow the largest product with the row's queries.
//
// For a key k inside a block, q . k <= sum_d max(q_d lo_d, q_d hi_d), so that
// sum ranks the blocks by the best key each may hold. With 8-bit codes on both
// sides it is a sum of 256 integer products,
//   sum_d min(qc_d, 0) lo_d + max(qc_d, 0) hi_d,
// a matrix product of integers: exact in any order, below 2^24, so that its f32
// value and the two scalings after it do not depend on how the work is split.
// A row's list is therefore the same alone, in a batch and in a prompt's chunk.
#include "attn_kv.h"
#include "attn_rows.h"
#include "g4_common.h"
#include "g4_math.h"
#include "g4_wave.h"
#include "granite4_layerops.h"

#include <algorithm>
#include <climits>
#include <cstdio>

namespace g4 {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Ranges.
// ---------------------------------------------------------------------------

struct RangeArgs {
  const uint8_t* k;   // [Hk][stride][K row bytes]
  const float* ksc;   // [Hk][stride][128 / group]
  int Hk, stride, units;
  int rows;           // positions of the call (one sequence)
  RowSet at;
  int8_t* ranges;     // [Hk][stride / block][2][128]: lowest, highest
  float* rscale;      // [Hk][stride / block]
};

__device__ __forceinline__ float col_min4(float x) { return -col_max4(-x); }

// One wave per (unit, KV head): 16 lanes cover a key's 128 channels (8 each),
// four keys at a time, every load of the block in flight before the first use.
// A unit is a block of the call's positions, or (row_pos) a row, whose block
// counts where the row's position is its last. The table, the keys and the reduction
// wait for one another, and that is its time: 500 rows of bf16 in blocks of 32 with 8
// KV heads 4.6 us, 8192 rows of K5 in groups of 32 in blocks of 64 7.8 (unpacking).
template <int BITS, int GROUP, int BLOCK>
__global__ __launch_bounds__(256) void kv_ranges_kernel(RangeArgs a) {
  constexpr int kKb = k_row_bytes(BITS);
  constexpr int kNgrp = BITS == 16 ? 1 : kHd / GROUP;
  constexpr int kIt = BLOCK / 4;
  const int lane = threadIdx.x & 63;
  const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (w >= static_cast<long long>(a.units) * a.Hk) return;
  const int unit = static_cast<int>(w % a.units), h = static_cast<int>(w / a.units);
  long long first, end;  // the call's positions of this unit
  const int* pt;
  if (a.at.row_pos != nullptr) {
    first = a.at.row_pos[unit];
    end = first + 1;
    pt = a.at.row_pt[unit];
    if (first < 0 || end % BLOCK != 0) return;
  } else {
    first = row_position(a.at, 0);
    end = first + a.rows;
    pt = a.at.d_pt;
  }
  const long long b = first / BLOCK + (a.at.row_pos != nullptr ? 0 : unit);
  const long long p0 = b * BLOCK;
  if (first < 0 || p0 + BLOCK > end || p0 + BLOCK > a.stride) return;  // not completed here
  const g4_global_i32* ptg = (const g4_global_i32*)pt;
  int prow[(BLOCK + 63) / 64];
#pragma unroll
  for (int i = 0; i < (BLOCK + 63) / 64; ++i) {
    const long long p = p0 + 64 * i + lane % (BLOCK < 64 ? BLOCK : 64);
    const int r = pt != nullptr ? ptg[p] : static_cast<int>(p);
    prow[i] = r >= 0 && r < a.stride ? r : -1;
  }
  // The block's place: the arena block that its first position begins.
  const int row0 = __shfl(prow[0], 0);
  if (row0 < 0 || row0 % BLOCK != 0) return;
  const int c = lane & 15, sub = lane >> 4;
  const uint8_t* kbase = a.k + static_cast<size_t>(h) * a.stride * kKb;
  const float* sbase = BITS == 16 ? nullptr : a.ksc + static_cast<size_t>(h) * a.stride * kNgrp;
  u32x4_t raw[kIt];
  float sc[BITS == 16 ? 1 : kIt];
  bool ok[kIt];
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    const int r = __shfl(prow[(4 * i) / 64], (4 * i + sub) & 63);
    ok[i] = r >= 0;
    const size_t rr = static_cast<size_t>(r >= 0 ? r : row0);
    raw[i] = load_k_raw<BITS>(kbase + rr * kKb, 8 * c);
    if constexpr (BITS != 16) sc[i] = sbase[rr * kNgrp + (8 * c) / GROUP];
  }
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    float f[8];
    if constexpr (BITS == 16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (e & 1) ? hi_bf16(raw[i][e >> 1]) : lo_bf16(raw[i][e >> 1]);
    } else {
      k_raw_f32<BITS>(raw[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= sc[i];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // a NaN value is passed over
      lo[e] = fminf(lo[e], ok[i] ? f[e] : INFINITY);
      hi[e] = fmaxf(hi[e], ok[i] ? f[e] : -INFINITY);
    }
  }
  float am = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = col_min4(lo[e]);
    hi[e] = col_max4(hi[e]);
    am = fmaxf(am, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
  }
  am = group_max<16>(am);
  const float s = am / 127.0f, inv = 1.0f / s;
  const size_t slot = static_cast<size_t>(h) * (a.stride / BLOCK) + row0 / BLOCK;
  if (sub < 2) {
    uint32_t out[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      out[e >> 2] |= (static_cast<uint32_t>(kv_code_inv(sub == 0 ? lo[e] : hi[e], s, inv, 127)) & 0xffu)
                     << (8 * (e & 3));
    *reinterpret_cast<u32x2_t*>(a.ranges + slot * 256 + 128 * sub + 8 * c) = u32x2_t{out[0], out[1]};
  }
  if (lane == 0) a.rscale[slot] = s;
}

template <int BITS, int GROUP>
void launch_ranges_block(const RangeArgs& a, int block, unsigned grid, hipStream_t st) {
  switch (block) {
    case 16: hipLaunchKernelGGL((kv_ranges_kernel<BITS, GROUP, 16>), grid, 256, 0, st, a); break;
    case 32: hipLaunchKernelGGL((kv_ranges_kernel<BITS, GROUP, 32>), grid, 256, 0, st, a); break;
    case 64: hipLaunchKernelGGL((kv_ranges_kernel<BITS, GROUP, 64>), grid, 256, 0, st, a); break;
    default: hipLaunchKernelGGL((kv_ranges_kernel<BITS, GROUP, 128>), grid, 256, 0, st, a); break;
  }
}
template <int BITS>
void launch_ranges(const RangeArgs& a, int group, int block, unsigned grid, hipStream_t st) {
  if constexpr (BITS == 16) {
    launch_ranges_block<16, kHd>(a, block, grid, st);
  } else {
    if (group == 32) launch_ranges_block<BITS, 32>(a, block, grid, st);
    else if (group == 64) launch_ranges_block<BITS, 64>(a, block, grid, st);
    else launch_ranges_block<BITS, kHd>(a, block, grid, st);
  }
}

// ---------------------------------------------------------------------------
// Scores and selection.
// ---------------------------------------------------------------------------

struct SelectArgs {
  const uint16_t* q;     // [rows][Hq][128]
  const int8_t* ranges;  // [Hk][stride / block][2][128]
  const float* rscale;   // [Hk][stride / block]
  int rows, Hk, stride, log_block, max_len;
  int r0, nrows;         // the rows of this launch
  RowSet at;
  int top_k, sink, recent;
  int nbp;               // keys per (row, KV head): blocks of max_len, padded to 64
  uint32_t* keys;        // [nrows][Hk][nbp]
  int32_t* sel;          // [rows][Hk][top_k]
};

// Keys order as unsigned integers: 0 for a block that cannot be listed, then
// the scores (-0 as 0, NaN lowest), then the blocks that are always listed.
constexpr uint32_t kKept = 0xffffffffu;
__device__ __forceinline__ uint32_t score_key(float f) {
  const int u = __float_as_int(fmaxf(f, -INFINITY) + 0.0f);
  return static_cast<uint32_t>(u ^ ((u >> 31) | INT_MIN));
}

// Blocks that row r sees: those up to its own position's, in [0, max_len).
__device__ __forceinline__ int row_blocks(const SelectArgs& a, int r) {
  const long long p = min(row_position(a.at, r), static_cast<long long>(a.max_len) - 1);
  return p < 0 ? 0 : static_cast<int>(p >> a.log_block) + 1;
}

// The scoring of up to ROWS rows of one KV head (ROWS x 4 query columns, 16 to a
// matrix product) by a workgroup of W waves.
//
// Query codes are made once per workgroup, 16 lanes to a column, into LDS; a
// wave then takes 64 blocks at a time: their table entries, one per lane, their
// 256-byte code rows, 16 lanes to a row, through LDS as B of v_mfma_i32_16x16x64_i8
// (K = 256: the lowest, then the highest codes), and A = the queries' negative,
// then their positive codes: a lane gets the four heads of one row at one
// block, and takes their maximum without another. put(rr, b, key) receives a key.
template <int W, int ROWS>
struct Scorer {
  static constexpr int kTiles = (ROWS * 4 + 15) / 16;  // 16-column tiles
  static constexpr int kCols = ROWS * 4;
  static constexpr int kLoads = 2;  // 16-block tiles in flight (4: 0.5 us more for one row, spills)
  // One more 16-byte unit per column, so that 16 columns' reads spread over the banks.
  static constexpr int kPitch = 9;
  static constexpr int kHold = kTiles <= 2 ? kTiles : 1;  // tiles whose query codes stay in registers
  struct Shared {
    i32x4_t code[kCols * kPitch];
    __align__(16) float scale[kCols];
  };
  struct QFrag {
    i32x4_t neg[2], pos[2];
  };

  __device__ __forceinline__ static QFrag q_frag(const Shared& sh, int c) {
    const int lane = threadIdx.x & 63, col = 16 * c + (lane & 15), g = lane >> 4;
    QFrag f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const i32x4_t x = col < kCols ? sh.code[col * kPitch + 4 * s + g] : i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // 0xff in the bytes below zero
        const int neg = static_cast<int>(((static_cast<uint32_t>(x[w]) >> 7) & 0x01010101u) * 0xffu);
        f.neg[s][w] = x[w] & neg;
        f.pos[s][w] = x[w] & ~neg;
      }
    }
    return f;
  }

  __device__ static void quantise(Shared& sh, const SelectArgs& a, int h, int row0, int nr) {
    const int l16 = threadIdx.x & 15;
    for (int col = threadIdx.x >> 4; col < kCols; col += W * 4) {
      const int row = row0 + min(col >> 2, nr - 1);
      const V8 x = ld8(a.q + (static_cast<size_t>(row) * 4 * a.Hk + 4 * h + (col & 3)) * kHd + 8 * l16);
      float am = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(v8_get(x, e)));
      am = group_max<16>(am);
      const float s = am / 127.0f;
      uint32_t w[2] = {0u, 0u};
      const float inv = 1.0f / s;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e >> 2] |= (static_cast<uint32_t>(kv_code_inv(v8_get(x, e), s, inv, 127)) & 0xffu) << (8 * (e & 3));
      reinterpret_cast<u32x2_t*>(sh.code + col * kPitch)[l16] = u32x2_t{w[0], w[1]};
      if (l16 == 0) sh.scale[col] = s;
    }
  }

  // Table entries of the blocks b0 + lane, clamped to the blocks the rows see.
  __device__ static int entry(const SelectArgs& a, const int* pt, int b0, int most) {
    const g4_global_i32* ptg = (const g4_global_i32*)pt;
    const int b = min(b0 + static_cast<int>(threadIdx.x & 63), most - 1);
    return pt != nullptr ? ptg[static_cast<size_t>(b) << a.log_block] : b << a.log_block;
  }

  // 64 blocks from b0 on, kLoads 16-block tiles' rows in flight at a time.
  template <bool PLAIN, class Put>
  __device__ __forceinline__ static void unit(const Shared& sh, const SelectArgs& a, int nr, size_t hb, int ab, float sb,
                                              int b0, int row0, i32x4_t* turn,
                                              const QFrag (&held)[kHold], Put put) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll 1
    for (int t0 = 0; t0 < 4; t0 += kLoads) {
      i32x4_t ka[kLoads][4];
#pragma unroll
      for (int t = 0; t < kLoads; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ka[t][j] = *reinterpret_cast<const i32x4_t*>(a.ranges + (hb + __shfl(ab, 16 * (t0 + t) + 4 * j + g)) * 256 + 16 * n);
      // Each tile through LDS into fragments: row r's 16-byte chunk c in slot c ^ r.
#pragma unroll
      for (int t = 0; t < kLoads; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) turn[16 * (4 * j + g) + (n ^ (4 * j + g))] = ka[t][j];
        asm volatile("" ::: "memory");  // a wave's DS operations execute in order
#pragma unroll
        for (int s = 0; s < 4; ++s) ka[t][s] = turn[16 * n + ((4 * s + g) ^ n)];
        asm volatile("" ::: "memory");
      }
      float sbt[kLoads];
#pragma unroll
      for (int t = 0; t < kLoads; ++t) sbt[t] = __shfl(sb, 16 * (t0 + t) + n);
#pragma unroll 2
      for (int c = 0; c < kTiles; ++c) {
        const QFrag q = kHold == kTiles ? held[c < kHold ? c : 0] : q_frag(sh, c);
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          i32x4_t acc = {0, 0, 0, 0};
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.neg[0], ka[t][0], acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.neg[1], ka[t][1], acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.pos[0], ka[t][2], acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.pos[1], ka[t][3], acc, 0, 0, 0);
          const f32x4_t sq = *reinterpret_cast<const f32x4_t*>(sh.scale + 4 * min(4 * c + g, ROWS - 1));
          // The four heads of row 4 c + g at block n of the tile; a NaN is passed over.
          float f = (static_cast<float>(acc[0]) * sbt[t]) * sq[0];
#pragma unroll
          for (int i = 1; i < 4; ++i) f = fmaxf(f, (static_cast<float>(acc[i]) * sbt[t]) * sq[i]);
          uint32_t key = score_key(f);
          const int bb = b0 + 16 * (t0 + t) + n;
          if constexpr (!PLAIN) {
            const int rr = 4 * c + g, have = rr < nr ? row_blocks(a, row0 + rr) : 0;
            const bool kept = bb < a.sink || bb >= have - a.recent;
            key = bb < have && sbt[t] != -1.0f ? (kept ? kKept : key) : 0u;
          }
          if (4 * c + g < (PLAIN ? ROWS : nr)) put(4 * c + g, bb, key);
        }
      }
    }
  }

  template <class Put>
  __device__ __forceinline__ static void score(const Shared& sh, const SelectArgs& a, int h, int row0, int nr, int most,
                               const int* pt, int first, int b0, int step, i32x4_t* turn, Put put) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const size_t hb = static_cast<size_t>(h) * (a.stride >> a.log_block);
    const int have_least = row_blocks(a, row0);
    QFrag held[kHold];
#pragma unroll
    for (int c = 0; c < kHold; ++c) {
      if constexpr (kHold == kTiles) held[c] = q_frag(sh, c);
    }
    for (; b0 < most; b0 += step) {
      // Arena block of context block b0 + lane: -1 where the table has none.
      const bool there = first >= 0 && first < a.stride && (first & ((1 << a.log_block) - 1)) == 0;
      const int ab = there ? first >> a.log_block : 0;
      // The block's scale, -1 (no scale is negative) for one without ranges.
      const float sb_mem = a.rscale[hb + ab];
      const int next = b0 + step < most ? entry(a, pt, b0 + step, most) : -1;
      const float sb = there ? sb_mem : -1.0f;
      // Where every block of the unit is scored for every row, no key looks at more.
      const bool plain = nr == ROWS && b0 >= a.sink && b0 + 64 <= have_least - a.recent && __all(there);
      if (plain) unit<true>(sh, a, nr, hb, ab, sb, b0, row0, turn, held, put);
      else unit<false>(sh, a, nr, hb, ab, sb, b0, row0, turn, held, put);
      first = next;
    }
  }
};

// Rows of one launch share a table where they are one sequence's.
__device__ __forceinline__ int most_blocks(const SelectArgs& a, int row0, int nr) {
  return row_blocks(a, row0 + nr - 1);  // the last row sees the most
}

__device__ __forceinline__ uint32_t readlane_u32(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
  x = max(x, dpp_u32<kDppQuadXor1>(x));
  x = max(x, dpp_u32<kDppQuadXor2>(x));
  x = max(x, dpp_u32<kDppHalfMirror>(x));
  x = max(x, dpp_u32<kDppMirror>(x));
  return max(max(readlane_u32(x, 0), readlane_u32(x, 16)), max(readlane_u32(x, 32), readlane_u32(x, 48)));
}
// Sum over the lanes up to and with this one: shifts within rows of 16 (a lane
// shifted in from outside its row gives 0), then the rows before it.
constexpr int kDppShr1 = 0x111, kDppShr2 = 0x112, kDppShr4 = 0x114, kDppShr8 = 0x118;
template <int CTRL>
__device__ __forceinline__ int dpp_shr(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ int wave_prefix(int x) {
  x += dpp_shr<kDppShr1>(x);
  x += dpp_shr<kDppShr2>(x);
  x += dpp_shr<kDppShr4>(x);
  x += dpp_shr<kDppShr8>(x);
  const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = __builtin_amdgcn_readlane(x, 31),
            r2 = __builtin_amdgcn_readlane(x, 47), row = (threadIdx.x & 63) >> 4;
  return x + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}
__device__ __forceinline__ int lanes_below(unsigned long long m) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(m >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(m), 0u));
}

// From a histogram of the keys lo + (bin << shift): the bin that holds the
// want-th largest becomes the range (lo; want: the place within it). True where
// that settles which keys are listed: those >= limit, of the equal ones the first `left`.
__device__ __forceinline__ bool next_range(const int* hist, int shift, int& want, uint32_t& lo, uint32_t& limit,
                                           int& left) {
  // Lane l: bins 255 - 4 l down; the keys above them, from the lanes before it.
  const int lane = threadIdx.x & 63;
  const i32x4_t h4 = *reinterpret_cast<const i32x4_t*>(hist + 252 - 4 * lane);
  const int mine = h4[0] + h4[1] + h4[2] + h4[3];
  const int upto = wave_prefix(mine);
  const int who = __builtin_ctzll(__ballot(upto >= want));
  int above = __builtin_amdgcn_readlane(upto - mine, who);
  int bin = 252 - 4 * who, count = __builtin_amdgcn_readlane(h4[0], who);
#pragma unroll
  for (int e = 3; e > 0; --e) {  // from the lane's highest bin
    const int x = __builtin_amdgcn_readlane(h4[e], who);
    if (above + x >= want) {
      bin += e;
      count = x;
      break;
    }
    above += x;
  }
  want -= above;
  lo += static_cast<uint32_t>(bin) << shift;
  limit = lo;
  if (count == want) return true;
  if (shift == 0) left = want;
  return shift == 0;
}

// Writes the listed ones of a wave's four keys per lane (blocks i .. i + 3) behind
// the `done` before them; equals: keys equal to the limit so far.
__device__ __forceinline__ void emit(const u32x4_t& k, int i, uint32_t limit, int left, int& done, int& equals,
                                     int32_t* out) {
  int eq_before = equals;
  unsigned long long eq[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    eq[e] = __ballot(k[e] == limit);
    eq_before += lanes_below(eq[e]);
  }
  bool take[4];
  int at = done;
  unsigned long long m[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    take[e] = k[e] > limit || (k[e] == limit && eq_before < left);
    eq_before += k[e] == limit;
    m[e] = __ballot(take[e]);
    at += lanes_below(m[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (take[e]) out[at++] = i + e;
    done += __popcll(m[e]);
    equals += __popcll(eq[e]);
  }
}

// One wave lists the blocks of the top_k largest of n keys in LDS, equal keys by
// the lower number. The limit between listed and not is found by histograms of
// 256 bins over the range of the keys in question: the bin that holds the
// top_k-th key becomes the next range, until all of a bin's keys are wanted or
// its keys are equal (four rounds at most; some hundred scores of one sign take two).
// HELD > 0: n <= 256 HELD, the keys stay in registers between the rounds.
template <int HELD>
__device__ __forceinline__ void pick_blocks(const uint32_t* keys, int n, int top_k, int* hist, int32_t* out) {
  const int lane = threadIdx.x & 63, chunks = HELD > 0 ? HELD : (n + 255) / 256;
  // Four keys per lane and chunk; those behind the row's blocks do not count.
  auto load = [&](int c) {
    const int i = 256 * c + 4 * lane;
    u32x4_t k = i < n ? *reinterpret_cast<const u32x4_t*>(keys + i) : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = i + e < n ? k[e] : 0u;
    return k;
  };
  u32x4_t mem[HELD > 0 ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int c = 0; c < HELD; ++c) mem[c] = load(c);
  }
  auto four = [&](int c) {
    if constexpr (HELD > 0) return mem[c];
    else return load(c);
  };
  uint32_t top = 0u, low_inv = 0u;  // largest key, complement of the smallest, of the scored ones
  int kept = 0, scored = 0;
#pragma unroll HELD > 0 ? HELD : 2
  for (int c = 0; c < chunks; ++c) {
    const u32x4_t k = four(c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_kept = k[e] == kKept, is_scored = !is_kept && k[e] != 0u;
      kept += __popcll(__ballot(is_kept));
      scored += __popcll(__ballot(is_scored));
      top = max(top, is_scored ? k[e] : 0u);
      low_inv = max(low_inv, is_scored ? ~k[e] : 0u);
    }
  }
  // Keys >= limit are listed, of those equal to it the first `left`.
  uint32_t limit = 1u;
  int left = INT_MAX, want = top_k - kept;  // want: of the keys in [lo, hi]
  if (scored > want) {
    uint32_t hi = wave_max_u32(top), lo = ~wave_max_u32(low_inv);
    limit = hi + 1u;
    while (want > 0) {
      const int shift = hi == lo ? 0 : max(0, 24 - __builtin_clz(hi - lo));
      *reinterpret_cast<i32x4_t*>(hist + 4 * lane) = i32x4_t{0, 0, 0, 0};
      wave_lds_sync();
#pragma unroll HELD > 0 ? HELD : 2
      for (int c = 0; c < chunks; ++c) {
        const u32x4_t k = four(c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k[e] - lo <= hi - lo) atomicAdd(&hist[(k[e] - lo) >> shift], 1);
      }
      wave_lds_sync();
      if (next_range(hist, shift, want, lo, limit, left)) break;
      hi = min(hi, lo + (1u << shift) - 1u);
      wave_lds_sync();  // the bins are read
    }
  }
  int done = 0, equals = 0;
#pragma unroll HELD > 0 ? HELD : 1
  for (int c = 0; c < chunks; ++c) {
    emit(four(c), 256 * c + 4 * lane, limit, left, done, equals, out);
  }
  for (int i = done + lane; i < top_k; i += 64) out[i] = -1;
}

// The same for one row by all W waves of a workgroup, wave w the keys [256 HELD
// w, ...): shared histograms (one per round, cleared here), and counts passed
// on in LDS.
template <int W, int HELD>
struct WidePick {
  int hist[4][256];
  uint32_t top[W], low_inv[W];
  int kept[W], scored[W], equals[W], taken[W];

  __device__ __forceinline__ void run(const uint32_t* keys, int n, int top_k, int32_t* out) {
    static_assert(W == 16, "a lane of each row of 16 per wave");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, base = 256 * HELD * wave;
    u32x4_t k[HELD];
#pragma unroll
    for (int c = 0; c < HELD; ++c) {
      const int i = base + 256 * c + 4 * lane;
      k[c] = i < n ? *reinterpret_cast<const u32x4_t*>(keys + i) : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 4; ++e) k[c][e] = i + e < n ? k[c][e] : 0u;
    }
    reinterpret_cast<int*>(hist)[threadIdx.x] = 0;
    {
      uint32_t t = 0u, l = 0u;
      int nk = 0, ns = 0;
#pragma unroll
      for (int c = 0; c < HELD; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool is_kept = k[c][e] == kKept, is_scored = !is_kept && k[c][e] != 0u;
          nk += __popcll(__ballot(is_kept));
          ns += __popcll(__ballot(is_scored));
          t = max(t, is_scored ? k[c][e] : 0u);
          l = max(l, is_scored ? ~k[c][e] : 0u);
        }
      t = wave_max_u32(t);
      l = wave_max_u32(l);
      if (lane == 0) {
        top[wave] = t;
        low_inv[wave] = l;
        kept[wave] = nk;
        scored[wave] = ns;
      }
    }
    __syncthreads();
    // Every wave adds up the others' counts: lane i (mod 16) has wave i's.
    const int l16 = lane & 15;
    int want = top_k - __builtin_amdgcn_readlane(wave_prefix(lane < W ? kept[l16] : 0), 63);
    const int all = __builtin_amdgcn_readlane(wave_prefix(lane < W ? scored[l16] : 0), 63);
    uint32_t limit = 1u;
    int left = INT_MAX;
    if (all > want) {
      uint32_t hi = wave_max_u32(top[l16]), lo = ~wave_max_u32(low_inv[l16]);
      limit = hi + 1u;
#pragma unroll 1
      for (int round = 0; want > 0; ++round) {
        const int shift = hi == lo ? 0 : max(0, 24 - __builtin_clz(hi - lo));
#pragma unroll
        for (int c = 0; c < HELD; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[c][e] - lo <= hi - lo) atomicAdd(&hist[round][(k[c][e] - lo) >> shift], 1);
        __syncthreads();
        if (next_range(hist[round], shift, want, lo, limit, left)) break;
        hi = min(hi, lo + (1u << shift) - 1u);
      }
    }
    int same = 0, more = 0;
#pragma unroll
    for (int c = 0; c < HELD; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        same += __popcll(__ballot(k[c][e] == limit));
        more += __popcll(__ballot(k[c][e] > limit));
      }
    if (lane == 0) {
      equals[wave] = same;
      taken[wave] = more;
    }
    __syncthreads();
    // Before this wave: equals, of which the first `left` are taken, and larger keys.
    const int eq = wave_prefix(lane < W ? equals[l16] : 0), mo = wave_prefix(lane < W ? taken[l16] : 0);
    const int eq_before = wave > 0 ? __builtin_amdgcn_readlane(eq, max(wave - 1, 0)) : 0;
    const int mo_before = wave > 0 ? __builtin_amdgcn_readlane(mo, max(wave - 1, 0)) : 0;
    const int total = __builtin_amdgcn_readlane(mo, 63) + min(__builtin_amdgcn_readlane(eq, 63), left);
    int done = mo_before + min(eq_before, left), equal = eq_before;
#pragma unroll
    for (int c = 0; c < HELD; ++c) emit(k[c], base + 256 * c + 4 * lane, limit, left, done, equal, out);
    for (int i = total + threadIdx.x; i < top_k; i += W * 64) out[i] = -1;
  }
};

// One workgroup per (ROWS rows, KV head): scores into LDS, then one wave per
// row (all waves for one row) lists its blocks. KEYS: keys of a row that fit.
// 8 KV heads, blocks of 64, 32 listed: one row among 470 blocks 8.1 us a call (table,
// ranges, scores, limit and list in turn), 1000 rows among 900 31.7 (8000 limits and
// lists by one wave each, and the scores' f32 steps); 16 sessions, blocks of 32, 64 of
// up to 2031 listed, 13 to 15 (the longest session's blocks by one CU per KV head).
template <int W, int ROWS, int KEYS>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(4))) void block_select_kernel(SelectArgs a) {
  using S = Scorer<W, ROWS>;
  // The query codes' place serves the histograms once every score is made.
  __shared__ union {
    typename S::Shared sh;
    __align__(16) int hist[ROWS < W ? ROWS : W][256];
    __align__(16) WidePick<16, KEYS / 4096 + (KEYS < 4096)> wide;
  } u;
  __shared__ __align__(16) uint32_t keys[ROWS][KEYS];
  __shared__ i32x4_t turn[W][256];
  const int wave = threadIdx.x >> 6;
  const int h = blockIdx.x, row0 = blockIdx.y * ROWS, nr = min(ROWS, a.rows - row0);
  const int most = most_blocks(a, row0, nr);
  const int* pt = row_table(a.at, row0);
  const int first = wave * 64 < most ? S::entry(a, pt, wave * 64, most) : -1;
  S::quantise(u.sh, a, h, row0, nr);
  __syncthreads();
  S::score(u.sh, a, h, row0, nr, most, pt, first, wave * 64, W * 64, turn[wave],
           [&](int rr, int b, uint32_t k) { keys[rr][b] = k; });
  __syncthreads();
  if constexpr (ROWS == 1) {
    // A row's keys in one wave's registers, where they fit, settle before sixteen
    // waves have agreed: 470 blocks 9.0 us the call (10.0), 2000 blocks 22.9 (20.1).
    if (row_blocks(a, row0) > 1024)
      u.wide.run(keys[0], row_blocks(a, row0), a.top_k, a.sel + (static_cast<size_t>(row0) * a.Hk + h) * a.top_k);
    else if (wave == 0)
      pick_blocks<4>(keys[0], row_blocks(a, row0), a.top_k, u.hist[0], a.sel + (static_cast<size_t>(row0) * a.Hk + h) * a.top_k);
    return;
  }
  for (int rr = wave; rr < nr; rr += W) {
    const int n = row_blocks(a, row0 + rr);
    int32_t* out = a.sel + (static_cast<size_t>(row0 + rr) * a.Hk + h) * a.top_k;
    if (KEYS <= 1024 || n <= 1024) pick_blocks<4>(keys[rr], n, a.top_k, u.hist[wave], out);
    else pick_blocks<0>(keys[rr], n, a.top_k, u.hist[wave], out);
  }
}

// The same scores to memory, for contexts whose keys LDS does not hold: a
// workgroup has 256 blocks of up to four rows.
__global__ __launch_bounds__(256) void block_score_kernel(SelectArgs a) {
  using S = Scorer<4, 4>;
  __shared__ S::Shared sh;
  __shared__ i32x4_t turn[4][256];
  const int per = a.at.row_pos != nullptr ? 1 : 4;
  const int lr0 = blockIdx.x * per, nr = min(per, a.nrows - lr0), row0 = a.r0 + lr0;
  const int h = blockIdx.y, b0 = (blockIdx.z * 4 + (threadIdx.x >> 6)) * 64;
  const int most = most_blocks(a, row0, nr);
  if (static_cast<int>(blockIdx.z) * 256 >= most) return;
  const int* pt = row_table(a.at, row0);
  const int first = b0 < most ? S::entry(a, pt, b0, most) : -1;
  S::quantise(sh, a, h, row0, nr);
  __syncthreads();
  uint32_t* dst = a.keys + (static_cast<size_t>(lr0) * a.Hk + h) * a.nbp;
  S::score(sh, a, h, row0, nr, min(most, b0 + 1), pt, first, b0, 64, turn[threadIdx.x >> 6], [&](int rr, int b, uint32_t k) {
    dst[static_cast<size_t>(rr) * a.Hk * a.nbp + b] = k;
  });
}

// Sum of v over the threads before this one, and over all (256 threads).
__device__ __forceinline__ int block_scan(int v, int* s_w, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous scan's reads are done
  if (lane == 63) s_w[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < wave) before += s_w[i];
    total += s_w[i];
  }
  return before + x - v;
}

// One workgroup per (row, KV head), keys in memory: the top_k-th largest by four
// 8-bit digits, then the blocks above it and the first of its equals, in order.
__global__ __launch_bounds__(256) void block_pick_kernel(SelectArgs a) {
  __shared__ int s_hist[256];
  __shared__ int s_w[4];
  __shared__ int s_digit, s_left;
  const int tid = threadIdx.x;
  const int lr = blockIdx.x, h = blockIdx.y, row = a.r0 + lr;
  const int n = row_blocks(a, row);
  const uint32_t* keys = a.keys + (static_cast<size_t>(lr) * a.Hk + h) * a.nbp;
  int32_t* out = a.sel + (static_cast<size_t>(row) * a.Hk + h) * a.top_k;
  uint32_t limit = 1;  // keys >= limit are listed, the first `left` of those equal to it
  int left = INT_MAX;
  int valid = 0;
  for (int i = tid; i < n; i += 256) valid += keys[i] != 0u;
  int total;
  block_scan(valid, s_w, total);
  if (total > a.top_k) {
    left = a.top_k;
    uint32_t prefix = 0u, mask = 0u;
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += 256) {
        const uint32_t k = keys[i];
        if ((k & mask) == prefix && k != 0u) atomicAdd(&s_hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      // Digits from the highest: thread t looks at digit 255 - t.
      const int mine = s_hist[255 - tid];
      const int above = block_scan(mine, s_w, total);
      if (above < left && above + mine >= left) {
        s_digit = 255 - tid;
        s_left = left - above;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(s_digit) << shift;
      mask |= 255u << shift;
      left = s_left;
      __syncthreads();
    }
    limit = prefix;
  }
  // Thread t takes the blocks [t per, (t + 1) per).
  const int per = (n + 255) / 256, i0 = min(tid * per, n), i1 = min(i0 + per, n);
  int same = 0, above = 0;
  for (int i = i0; i < i1; ++i) {
    same += keys[i] == limit;
    above += keys[i] > limit;
  }
  int dummy, count;
  const int same_before = block_scan(same, s_w, dummy);
  int take = min(max(left - same_before, 0), same);
  int at = block_scan(above + take, s_w, count);
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i];
    if (k > limit || (k == limit && take-- > 0)) out[at++] = i;
  }
  for (int i = count + tid; i < a.top_k; i += 256) out[i] = -1;
}

// The most keys of a row that the one-launch form holds in LDS.
constexpr int kLdsKeys = 16384;

template <int W, int ROWS, int KEYS>
void launch_select(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((block_select_kernel<W, ROWS, KEYS>), dim3(a.Hk, (a.rows + ROWS - 1) / ROWS), W * 64, 0, st, a);
}

int padded_blocks(int max_len, int block) { return ((max_len + block - 1) / block + 63) / 64 * 64; }

// Whether LDS holds a row's keys and the rows fit a grid: scores then take no work.
bool one_launch(int rows, int nbp) { return nbp <= kLdsKeys && rows <= 65535; }

// Rows whose keys one launch holds: at most 64 MB of them, so that they are
// read back from the caches.
int slab_rows(int rows, int Hk, int nbp) {
  const size_t per = static_cast<size_t>(Hk) * nbp * sizeof(uint32_t);
  const size_t fit = (static_cast<size_t>(64) << 20) / per;
  return static_cast<int>(std::min<size_t>(rows, std::max<size_t>(16, fit / 4 * 4)));
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" {

int granite4_kv_ranges(const void* cache_k, const float* k_scale, int bits, int group, int Hk,
                       int d, int stride, int block, int base_pos, int rows, const int* d_pos,
                       const int* d_pt, const int* row_pos, const int* const* row_pt,
                       int8_t* ranges, float* range_scale) {
  RangeArgs a{};
  a.at = RowSet{base_pos, d_pos, d_pt, row_pos, row_pt};
  if (cache_k == nullptr || ranges == nullptr || range_scale == nullptr || Hk <= 0 || d != kHd ||
      !block_ok(block, stride) || !row_set_ok(a.at, rows, stride) || !aligned(cache_k, 16) ||
      !aligned(ranges, 16) || (bits != 16 && bits != 8 && bits != 4 && bits != 5) ||
      (bits != 16 && (k_scale == nullptr || (group != 32 && group != 64 && group != kHd)))) {
    std::fprintf(stderr, "granite4: granite4_kv_ranges: invalid arguments\n");
    return -1;
  }
  a.k = static_cast<const uint8_t*>(cache_k);
  a.ksc = k_scale;
  a.Hk = Hk;
  a.stride = stride;
  a.rows = rows;
  // Blocks the positions may end in; where the first position is known here,
  // those they do (the others return at once).
  const long long base = base_pos;
  const long long units = row_pos != nullptr ? rows
                          : d_pos != nullptr ? std::min<long long>(rows / block + 1, stride / block)
                                             : (base + rows) / block - base / block;
  if (units == 0) return 0;
  a.units = static_cast<int>(units);
  a.ranges = ranges;
  a.rscale = range_scale;
  const long long wgs = (units * Hk + 3) / 4;
  if (wgs > INT_MAX) {
    std::fprintf(stderr, "granite4: granite4_kv_ranges: invalid arguments\n");
    return -1;
  }
  const unsigned grid = static_cast<unsigned>(wgs);
  const hipStream_t st = stream();
  switch (bits) {
    case 16: launch_ranges<16>(a, group, block, grid, st); break;
    case 8: launch_ranges<8>(a, group, block, grid, st); break;
    case 4: launch_ranges<4>(a, group, block, grid, st); break;
    default: launch_ranges<5>(a, group, block, grid, st); break;
  }
  return launch_status("granite4_kv_ranges");
}

size_t granite4_block_select_work_bytes(int rows, int Hk, int max_len, int block) {
  if (rows <= 0 || Hk <= 0 || max_len <= 0 || max_len > INT_MAX - 128 * 64 || block <= 0) return 0;
  const int nbp = padded_blocks(max_len, block);
  if (one_launch(rows, nbp)) return 0;
  return static_cast<size_t>(slab_rows(rows, Hk, nbp)) * Hk * nbp * sizeof(uint32_t);
}

int granite4_block_select(const uint16_t* q, int rows, int Hq, int Hk, int d,
                          const int8_t* ranges, const float* range_scale, int stride, int block,
                          int kv_base, const int* d_pos, const int* d_pt, const int* row_pos,
                          const int* const* row_pt, int max_len, int top_k, int sink, int recent,
                          void* work, int32_t* sel) {
  SelectArgs a{};
  a.at = RowSet{kv_base, d_pos, d_pt, row_pos, row_pt};
  const int ml = max_len > 0 ? max_len : stride;
  if (q == nullptr || ranges == nullptr || range_scale == nullptr ||
      sel == nullptr || d != kHd || Hk <= 0 || Hk > 65535 || Hq != kGq * Hk ||
      !block_ok(block, stride) || max_len < 0 || ml > stride || !row_set_ok(a.at, rows, ml) ||
      top_k < 1 || sink < 0 || recent < 1 || recent > top_k || sink > top_k - recent ||
      ml / block > 65535 * 256 - 64 || !aligned(q, 16) || !aligned(ranges, 16) ||
      !aligned(work, 16) || (work == nullptr && !one_launch(rows, padded_blocks(ml, block)))) {
    std::fprintf(stderr, "granite4: granite4_block_select: invalid arguments\n");
    return -1;
  }
  a.q = q;
  a.ranges = ranges;
  a.rscale = range_scale;
  a.rows = rows;
  a.Hk = Hk;
  a.stride = stride;
  a.log_block = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  a.max_len = ml;
  a.top_k = top_k;
  a.sink = sink;
  a.recent = recent;
  a.nbp = padded_blocks(ml, block);
  a.keys = static_cast<uint32_t*>(work);
  a.sel = sel;
  const hipStream_t st = stream();
  const bool one_seq = row_pos == nullptr;
  if (one_launch(rows, a.nbp)) {
    if (one_seq && rows > 1 && a.nbp <= 1024) launch_select<8, 8, 1024>(a, st);
    else if (one_seq && rows > 1 && a.nbp <= 4096) launch_select<16, 4, 4096>(a, st);
    else if (a.nbp <= 4096) launch_select<16, 1, 4096>(a, st);
    else launch_select<16, 1, kLdsKeys>(a, st);
    return launch_status("granite4_block_select");
  }
  const int slab = slab_rows(rows, Hk, a.nbp), per = row_pos != nullptr ? 1 : 4;
  for (a.r0 = 0; a.r0 < rows; a.r0 += slab) {
    a.nrows = std::min(slab, rows - a.r0);
    hipLaunchKernelGGL(block_score_kernel, dim3((a.nrows + per - 1) / per, Hk, (a.nbp + 255) / 256),
                       256, 0, st, a);
    hipLaunchKernelGGL(block_pick_kernel, dim3(a.nrows, Hk), 256, 0, st, a);
  }
  return launch_status("granite4_block_select");
}

}  // extern "C"
