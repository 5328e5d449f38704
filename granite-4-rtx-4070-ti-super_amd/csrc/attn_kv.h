// attn_kv.h - reading the paged KV pool for the attention kernels (attn.hip,
// attn_blocks.hip): raw bytes of cached rows to bf16 MFMA operands (values or
// integer codes, or values dequantised per scale group), V tiles into LDS for
// transposed reads, and reductions over the lanes of one query column.
#ifndef G4_ATTN_KV_H
#define G4_ATTN_KV_H

#include "g4_common.h"
#include "g4_hw.h"
#include "g4_math.h"

#include <cmath>

namespace g4 {
namespace {

constexpr int kTile = 64;
constexpr int kHd = 128;         // head dim
constexpr int kGq = 4;           // query heads per KV head
constexpr int kVPitch = kHd + 16;  // LDS V row pitch (bf16): 288 B, rows 8 banks apart

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
// The page tables are device (global) memory; typed so, their loads are
// global_load (vmcnt only) rather than flat (which LDS waits would include).
typedef __attribute__((address_space(1))) const int g4_global_i32;

// Four bf16 of a row-major LDS tile, transposed across each 16-lane group
// (ds_read_b64_tr_b16): lane i of a group receives element i % 4 of the
// 8-byte vectors addressed by lanes i / 4, 4 + i / 4, 8 + i / 4, 12 + i / 4.
__device__ __forceinline__ u32x2_t lds_read_tr(const uint16_t* p) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p)));
}

__device__ __forceinline__ bf16x8_t as_bf16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const u32x4_t u = {a, b, c, d};
  return __builtin_bit_cast(bf16x8_t, u);
}

// Maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (the four lanes of one
// query column), by row swaps within the vector unit: __shfl_xor goes through
// the LDS, two dependent round trips per tile.
__device__ __forceinline__ float col_max4(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum4(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

constexpr float kLog2E = 1.44269504088896341f;

// Exact bf16 pair of two small integers (|x| <= 127).
__device__ __forceinline__ uint32_t int_pair_bf16(int a, int b) {
  return pack_bf16_hw(static_cast<float>(a), static_cast<float>(b));
}
// The int4 codes at bits [b, b + 4) and [b + 4, b + 8) of x, as their
// values code - 8, in bf16: the code xor 8 read as a signed 4-bit field is
// code - 8, so each value is one sign-extending field extract (xs = x ^
// 0x88888888, once per word) instead of an extract and a subtraction.
__device__ __forceinline__ int sfield4(uint32_t xs, int b) {
  return static_cast<int>(xs << (28 - b)) >> 28;
}
__device__ __forceinline__ uint32_t int4_pair_bf16(uint32_t xs, int b) {
  return int_pair_bf16(sfield4(xs, b), sfield4(xs, b + 4));
}

// Row bytes of the K / V caches per format.
__host__ __device__ constexpr int k_row_bytes(int bits) {
  return bits == 16 ? 2 * kHd : bits == 8 ? kHd : bits == 4 ? kHd / 2 : kHd / 2 + kHd / 8;
}
__host__ __device__ constexpr int v_row_bytes(int bits) {
  return bits == 16 ? 2 * kHd : bits == 8 ? kHd : kHd / 2;
}

// Raw bytes of eight K elements (dims c .. c + 7, c a multiple of 8) of one
// cached row: bf16 16 B, int8 8 B, int4 4 B, K5 4 nibble bytes + the high-bit
// plane byte. Loading and converting are separate so that a tile's K and V
// loads are all in flight before any of them is used.
template <int BITS>
__device__ __forceinline__ u32x4_t load_k_raw(const uint8_t* row, int c) {
  u32x4_t r = {0u, 0u, 0u, 0u};
  if constexpr (BITS == 16) {
    r = *reinterpret_cast<const u32x4_t*>(row + 2 * c);
  } else if constexpr (BITS == 8) {
    const u32x2_t u = *reinterpret_cast<const u32x2_t*>(row + c);
    r.x = u.x;
    r.y = u.y;
  } else {
    r.x = *reinterpret_cast<const uint32_t*>(row + c / 2);
    if constexpr (BITS == 5) r.y = row[kHd / 2 + c / 8];
  }
  return r;
}

// The eight K elements as bf16: the value (bf16 cache) or the integer code.
template <int BITS>
__device__ __forceinline__ bf16x8_t k_raw_bf16(const u32x4_t& r) {
  if constexpr (BITS == 16) {
    return __builtin_bit_cast(bf16x8_t, r);
  } else if constexpr (BITS == 8) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = e < 2 ? r.x : r.y;
      const int sh = 16 * (e & 1);
      w[e] = int_pair_bf16(static_cast<int8_t>(x >> sh), static_cast<int8_t>(x >> (sh + 8)));
    }
    return as_bf16x8(w[0], w[1], w[2], w[3]);
  } else if constexpr (BITS == 4) {
    const uint32_t xs = r.x ^ 0x88888888u;
    return as_bf16x8(int4_pair_bf16(xs, 0), int4_pair_bf16(xs, 8), int4_pair_bf16(xs, 16),
                     int4_pair_bf16(xs, 24));
  } else {
    // K5: the eight 5-bit codes assembled bytewise, four at a time: the low
    // nibbles (dims c + 2 e) and the high nibbles (c + 2 e + 1) masked out of
    // x, and the high-bit plane's bits 2 e (+ 1) moved to bit 4 of byte e by
    // one 24-bit multiply (bit 2 e of t times 2^4 + 2^10 + 2^16 + 2^22 lands
    // on 8 e + 4; the other products miss bits 4, 12, 20 and 28 and carry
    // into none of them). Each byte then converts to f32 in one instruction
    // (v_cvt_f32_ubyte*) and value = code - 16 exactly.
    static_assert(BITS == 5, "k_raw_bf16: bf16, int8, int4 or K5");
    constexpr uint32_t kSpread = (1u << 4) | (1u << 10) | (1u << 16) | (1u << 22);
    const uint32_t lo = (r.x & 0x0F0F0F0Fu) | (__umul24(r.y & 0x55u, kSpread) & 0x10101010u);
    const uint32_t hi = ((r.x >> 4) & 0x0F0F0F0Fu) | (__umul24((r.y >> 1) & 0x55u, kSpread) & 0x10101010u);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = pack_bf16_hw(static_cast<float>((lo >> (8 * e)) & 0xFFu) - 16.0f,
                          static_cast<float>((hi >> (8 * e)) & 0xFFu) - 16.0f);
    return as_bf16x8(w[0], w[1], w[2], w[3]);
  }
}

// Scale groups smaller than a row (32 or 64: this build's extension; the
// reference keeps one scale per row): the attention reads each element
// dequantised, bf16(code * scale_g), and then runs the bf16 path (logits
// bf16(scale * q . k), unscaled bf16 probabilities). One scale per row keeps
// the reference's form: codes in the products, the row's scales on the dot
// and on p.
template <int BITS, int GROUP>
constexpr bool kv_deq() { return BITS != 16 && GROUP < kHd; }

// The eight K elements of a quantised row as f32 codes.
template <int BITS>
__device__ __forceinline__ void k_raw_f32(const u32x4_t& r, float (&f)[8]) {
  if constexpr (BITS == 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? r.x : r.y) >> (8 * (e & 3))));
  } else if constexpr (BITS == 4) {
    const uint32_t xs = r.x ^ 0x88888888u;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(sfield4(xs, 4 * e));
  } else {
    static_assert(BITS == 5, "k_raw_f32: int8, int4 or K5");
    constexpr uint32_t kSpread = (1u << 4) | (1u << 10) | (1u << 16) | (1u << 22);
    const uint32_t lo = (r.x & 0x0F0F0F0Fu) | (__umul24(r.y & 0x55u, kSpread) & 0x10101010u);
    const uint32_t hi = ((r.x >> 4) & 0x0F0F0F0Fu) | (__umul24((r.y >> 1) & 0x55u, kSpread) & 0x10101010u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = static_cast<float>((lo >> (8 * e)) & 0xFFu) - 16.0f;
      f[2 * e + 1] = static_cast<float>((hi >> (8 * e)) & 0xFFu) - 16.0f;
    }
  }
}
// Unsigned codes held one per byte of lo (dims 2 e) and hi (dims 2 e + 1),
// dequantised as bf16((code - bias) * s): fma(code, s, -bias * s) is the same
// f32 (code * s - bias * s is exactly (code - bias) * s, and both round it
// once; bias * s is exact), one instruction instead of a subtraction and a
// multiply.
__device__ __forceinline__ bf16x8_t bytes_deq(uint32_t lo, uint32_t hi, float s, float nbs) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = pack_bf16_hw(fmaf(static_cast<float>((lo >> (8 * e)) & 0xFFu), s, nbs),
                        fmaf(static_cast<float>((hi >> (8 * e)) & 0xFFu), s, nbs));
  return as_bf16x8(w[0], w[1], w[2], w[3]);
}

// ... dequantised with the elements' group scale: bf16(code * s).
template <int BITS>
__device__ __forceinline__ bf16x8_t k_raw_deq(const u32x4_t& r, float s) {
  if constexpr (BITS == 5) {
    constexpr uint32_t kSpread = (1u << 4) | (1u << 10) | (1u << 16) | (1u << 22);
    const uint32_t lo = (r.x & 0x0F0F0F0Fu) | (__umul24(r.y & 0x55u, kSpread) & 0x10101010u);
    const uint32_t hi = ((r.x >> 4) & 0x0F0F0F0Fu) | (__umul24((r.y >> 1) & 0x55u, kSpread) & 0x10101010u);
    return bytes_deq(lo, hi, s, -16.0f * s);
  } else if constexpr (BITS == 4) {
    return bytes_deq(r.x & 0x0F0F0F0Fu, (r.x >> 4) & 0x0F0F0F0Fu, s, -8.0f * s);
  } else {
    float f[8];
    k_raw_f32<BITS>(r, f);
    return as_bf16x8(pack_bf16_hw(f[0] * s, f[1] * s), pack_bf16_hw(f[2] * s, f[3] * s),
                     pack_bf16_hw(f[4] * s, f[5] * s), pack_bf16_hw(f[6] * s, f[7] * s));
  }
}
// One 16-byte V chunk (int8: 16 values, int4: 32), dequantised with scale s,
// as bf16 pairs w[0 .. 8 or 16).
template <int BITS>
__device__ __forceinline__ void v_chunk_deq(const u32x4_t& u, float s, uint32_t (&w)[BITS == 8 ? 8 : 16]) {
  if constexpr (BITS == 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = u[e >> 1];
      const int sh = 16 * (e & 1);
      w[e] = pack_bf16_hw(static_cast<float>(static_cast<int8_t>(x >> sh)) * s,
                          static_cast<float>(static_cast<int8_t>(x >> (sh + 8))) * s);
    }
  } else {
    // bf16((code - 8) * s) per nibble, the low nibble of byte b first
    const float nbs = -8.0f * s;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t lo = u[q] & 0x0F0F0F0Fu, hi = (u[q] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        w[4 * q + b] = pack_bf16_hw(fmaf(static_cast<float>((lo >> (8 * b)) & 0xFFu), s, nbs),
                                    fmaf(static_cast<float>((hi >> (8 * b)) & 0xFFu), s, nbs));
    }
  }
}

// V staging: each step moves one 16-byte chunk per lane of the tile's rows
// (bf16: 4 keys x 16 chunks per step, 16 steps; int8: 8 keys x 8 chunks, 8
// steps; int4: 16 keys x 4 chunks, 4 steps) from the pool into a row-major
// LDS tile, as bf16 values / integer codes; keys without an arena row read 0.
template <int BITS>
struct VStage {
  static constexpr int kSteps = BITS == 16 ? 16 : BITS == 8 ? 8 : 4;
  static constexpr int kChunks = 64 / (kTile / kSteps);  // chunks per row
  static constexpr int kRowB = BITS == 16 ? 256 : BITS == 8 ? 128 : 64;
};

template <int BITS>
__device__ __forceinline__ void v_load(const uint8_t* vbase, int prow,
                                       u32x4_t (&raw)[VStage<BITS>::kSteps]) {
  using VS = VStage<BITS>;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < VS::kSteps; ++i) {
    const int key = i * (64 / VS::kChunks) + lane / VS::kChunks, c = lane % VS::kChunks;
    const int pr = __shfl(prow, key);
    // Unconditional (row 0 for keys without a row); v_store zeroes those.
    raw[i] = *reinterpret_cast<const u32x4_t*>(vbase + static_cast<size_t>(pr >= 0 ? pr : 0) * VS::kRowB + 16 * c);
  }
}

// bf16 V tiles go from global memory straight to LDS (global_load_lds, 16
// bytes per lane): no registers hold them, so the bf16 kernel fits two waves
// per SIMD. The tile is 64 rows of 256 bytes without padding; the 16-byte
// chunk c of row r sits at chunk c ^ 2 (r & 7), so that the transposed reads
// of 16 consecutive rows (32 bytes each) spread over all 64 banks (two
// passes, as with the padded layout). Load i writes rows 4 i .. 4 i + 3.
typedef __attribute__((address_space(3))) void* lds_ptr_t;
__device__ __forceinline__ int v_swz(int row) { return 2 * (row & 7); }
__device__ __forceinline__ void v_dma_bf16(const uint8_t* vbase, int prow, uint16_t* vl) {
  const int lane = threadIdx.x & 63;
  uint8_t* dst = reinterpret_cast<uint8_t*>(vl);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = 4 * i + (lane >> 4), c = (lane & 15) ^ v_swz(row);
    const int pr = __shfl(prow, row);
    // Unconditional (row 0 for keys without a row); v_fix_bf16 zeroes those.
    __builtin_amdgcn_global_load_lds(vbase + static_cast<size_t>(pr >= 0 ? pr : 0) * 256 + 16 * c,
                                     (lds_ptr_t)(dst + 1024 * i), 16, 0, 0);
  }
}
// After the loads have landed: rows without an arena row become 0.
__device__ __forceinline__ void v_fix_bf16(uint16_t* vl, unsigned long long valid) {
  if (valid == ~0ull) return;
  const int lane = threadIdx.x & 63;
  uint8_t* dst = reinterpret_cast<uint8_t*>(vl);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = 4 * i + (lane >> 4);
    if (!((valid >> row) & 1ull))
      *reinterpret_cast<u32x4_t*>(dst + 1024 * i + 16 * lane) = u32x4_t{0u, 0u, 0u, 0u};
  }
}

// v_store for scale groups smaller than a row: each chunk dequantised with
// its key's group scale, scale_of(key, group) (keys without a row: 0).
template <int BITS, int GROUP, typename F>
__device__ __forceinline__ void v_store_deq(const u32x4_t (&raw)[VStage<BITS>::kSteps], uint16_t* vl,
                                            unsigned long long valid, F scale_of) {
  using VS = VStage<BITS>;
  static_assert(BITS == 8 || BITS == 4 || BITS == 5, "quantised V");
  constexpr int kDims = kHd / VS::kChunks;  // dims per chunk (16 or 32), within one group
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < VS::kSteps; ++i) {
    const int key = i * (64 / VS::kChunks) + lane / VS::kChunks, c = lane % VS::kChunks;
    const float sc = ((valid >> key) & 1ull) ? scale_of(key, (kDims * c) / GROUP) : 0.0f;
    uint32_t w[BITS == 8 ? 8 : 16];
    v_chunk_deq<BITS>(raw[i], sc, w);
    uint16_t* dst = vl + key * kVPitch + kDims * c;
#pragma unroll
    for (int e = 0; e < kDims / 8; ++e)
      *reinterpret_cast<u32x4_t*>(dst + 8 * e) = u32x4_t{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
    __builtin_amdgcn_sched_barrier(0);  // one step's values live at a time
  }
}

// valid: bit k set when key k of the tile has an arena row (others store 0).
template <int BITS>
__device__ __forceinline__ void v_store(const u32x4_t (&raw)[VStage<BITS>::kSteps], uint16_t* vl,
                                        unsigned long long valid) {
  using VS = VStage<BITS>;
  const int lane = threadIdx.x & 63;
  const uint32_t z = BITS == 16 || BITS == 8 ? 0u : 0x88888888u;  // int4 code 8 = value 0
#pragma unroll
  for (int i = 0; i < VS::kSteps; ++i) {
    const int key = i * (64 / VS::kChunks) + lane / VS::kChunks, c = lane % VS::kChunks;
    const u32x4_t u = ((valid >> key) & 1ull) ? raw[i] : u32x4_t{z, z, z, z};
    if constexpr (BITS == 16) {
      *reinterpret_cast<u32x4_t*>(vl + key * kVPitch + 8 * c) = u;
    } else if constexpr (BITS == 8) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t x = u[e >> 1];
        const int sh = 16 * (e & 1);
        w[e] = int_pair_bf16(static_cast<int8_t>(x >> sh), static_cast<int8_t>(x >> (sh + 8)));
      }
      uint16_t* dst = vl + key * kVPitch + 16 * c;
      *reinterpret_cast<u32x4_t*>(dst) = u32x4_t{w[0], w[1], w[2], w[3]};
      *reinterpret_cast<u32x4_t*>(dst + 8) = u32x4_t{w[4], w[5], w[6], w[7]};
    } else {
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t x = u[e >> 2];
        const int b = 8 * (e & 3);
        w[e] = int4_pair_bf16(x ^ 0x88888888u, b);
      }
      uint16_t* dst = vl + key * kVPitch + 32 * c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<u32x4_t*>(dst + 8 * e) = u32x4_t{w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]};
    }
  }
}

// Completes this wave's LDS writes before other lanes of the wave read them
// (each wave owns its LDS tile, so no workgroup barrier is needed).
__device__ __forceinline__ void wave_lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Partials and arrival tags are written and read at device scope (sc1 on
// gfx950): the workgroup that combines may run on another XCD, whose L2
// holds none of the writer's lines, and a tag must not be seen before the
// partial it announces.
__device__ __forceinline__ void st_dev_u64(void* p, unsigned long long v) {
  __hip_atomic_store(static_cast<unsigned long long*>(p), v, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long ld_dev_u64(const void* p) {
  return __hip_atomic_load(static_cast<unsigned long long*>(const_cast<void*>(p)), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long f2_bits(float x, float y) {
  return static_cast<unsigned long long>(__float_as_uint(x)) |
         (static_cast<unsigned long long>(__float_as_uint(y)) << 32);
}
__device__ __forceinline__ void wait_stores() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace
}  // namespace g4

#endif  // G4_ATTN_KV_H
