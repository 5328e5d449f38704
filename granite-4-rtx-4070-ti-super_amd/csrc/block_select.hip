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
// counts where the row's position is its last.
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
  int rows, Hk, stride, block, max_len;
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
  if (!(f == f)) f = -INFINITY;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) != 0u ? ~u : (u | 0x80000000u);
}

// Blocks that row r sees: those up to its own position's, in [0, max_len).
__device__ __forceinline__ int row_blocks(const SelectArgs& a, int r) {
  const long long p = min(row_position(a.at, r), static_cast<long long>(a.max_len) - 1);
  return p < 0 ? 0 : static_cast<int>(p / a.block) + 1;
}

// One wave: 64 blocks of one KV head against up to four rows of one sequence
// (16 query columns: 4 rows x 4 heads; a row with its own table is alone).
// D[block][column] by v_mfma_i32_16x16x64_i8 over K = 256: A = a block's 128
// lowest, then 128 highest codes, straight from memory; B = the column's
// negative codes, then its positive ones.
__global__ __launch_bounds__(256) void block_score_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int per = a.at.row_pos != nullptr ? 1 : 4;
  const int lr0 = blockIdx.x * per;  // within the launch
  const int nr = min(per, a.nrows - lr0);
  const int h = blockIdx.y, b0 = (blockIdx.z * 4 + (threadIdx.x >> 6)) * 64;
  const int rr = n >> 2;
  const bool live = rr < nr;
  const int row = a.r0 + lr0 + (live ? rr : 0);
  const int have = live ? row_blocks(a, row) : 0;
  const int have_max = row_blocks(a, a.r0 + lr0 + nr - 1);  // the last row sees the most
  if (b0 >= have_max) return;
  const int* pt = row_table(a.at, a.r0 + lr0);
  const g4_global_i32* ptg = (const g4_global_i32*)pt;
  // Arena block of context block b0 + lane: -1 where the table has none.
  const int b = min(b0 + lane, have_max - 1);
  const int first = pt != nullptr ? ptg[static_cast<size_t>(b) * a.block] : b * a.block;
  const int ab = first >= 0 && first < a.stride && first % a.block == 0 ? first / a.block : -1;
  const size_t hb = static_cast<size_t>(h) * (a.stride / a.block);
  i32x4_t ka[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int j = __shfl(ab, 16 * t + n);
    const int8_t* src = a.ranges + (hb + (j >= 0 ? j : 0)) * 256 + 16 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) ka[t][s] = *reinterpret_cast<const i32x4_t*>(src + 64 * s);
  }
  const float sb = a.rscale[hb + (ab >= 0 ? ab : 0)];
  // The column's codes: dims 64 s + 16 g .. + 15, under amax / 127.
  i32x4_t qn[2], qp[2];
  float sq;
  {
    const uint16_t* qr = a.q + (static_cast<size_t>(row) * 4 * a.Hk + 4 * h + (n & 3)) * kHd + 16 * g;
    V8 x[4];
    float am = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ld8(qr + 64 * (i >> 1) + 8 * (i & 1));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(v8_get(x[i], e)));
    am = col_max4(am);
    sq = am / 127.0f;
    const float inv = 1.0f / sq;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t neg = 0u, pos = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int code = live ? kv_code_inv(v8_get(x[2 * s + (w >> 1)], 4 * (w & 1) + e), sq, inv, 127) : 0;
          neg |= (static_cast<uint32_t>(min(code, 0)) & 0xffu) << (8 * e);
          pos |= (static_cast<uint32_t>(max(code, 0)) & 0xffu) << (8 * e);
        }
        qn[s][w] = static_cast<int>(neg);
        qp[s][w] = static_cast<int>(pos);
      }
  }
  uint32_t* dst = a.keys + (static_cast<size_t>(lr0 + rr) * a.Hk + h) * a.nbp + b0 + 4 * g;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    i32x4_t acc = {0, 0, 0, 0};
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[t][0], qn[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[t][1], qn[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[t][2], qp[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[t][3], qp[1], acc, 0, 0, 0);
    u32x4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 16 * t + 4 * g + i, bb = b0 + at;
      const int place = __shfl(ab, at);  // by every lane: a lane outside a branch gives nothing
      float f = (static_cast<float>(acc[i]) * __shfl(sb, at)) * sq;
      f = fmaxf(f, dpp_f32<kDppQuadXor1>(f));  // over the four heads (fmaxf passes a NaN over)
      f = fmaxf(f, dpp_f32<kDppQuadXor2>(f));
      const bool kept = bb < a.sink || bb >= have - a.recent;
      const bool can = bb < have && place >= 0;
      out[i] = can ? (kept ? kKept : score_key(f)) : 0u;
    }
    if (live && (n & 3) == 0) *reinterpret_cast<u32x4_t*>(dst + 16 * t) = out;
  }
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

// One workgroup per (row, KV head): the top_k-th largest key by four 8-bit
// digits, then the blocks above it and the first of its equals, in order.
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

int padded_blocks(int max_len, int block) { return ((max_len + block - 1) / block + 63) / 64 * 64; }

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
  if (q == nullptr || ranges == nullptr || range_scale == nullptr || work == nullptr ||
      sel == nullptr || d != kHd || Hk <= 0 || Hk > 65535 || Hq != kGq * Hk ||
      !block_ok(block, stride) || max_len < 0 || ml > stride || !row_set_ok(a.at, rows, ml) ||
      top_k < 1 || sink < 0 || recent < 1 || recent > top_k || sink > top_k - recent ||
      ml / block > 65535 * 256 - 64 || !aligned(q, 16) || !aligned(ranges, 16) ||
      !aligned(work, 16)) {
    std::fprintf(stderr, "granite4: granite4_block_select: invalid arguments\n");
    return -1;
  }
  a.q = q;
  a.ranges = ranges;
  a.rscale = range_scale;
  a.rows = rows;
  a.Hk = Hk;
  a.stride = stride;
  a.block = block;
  a.max_len = ml;
  a.top_k = top_k;
  a.sink = sink;
  a.recent = recent;
  a.nbp = padded_blocks(ml, block);
  a.keys = static_cast<uint32_t*>(work);
  a.sel = sel;
  const hipStream_t st = stream();
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
