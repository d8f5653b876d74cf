// Building blocks of the tiled attention kernels (attention.hip, bias_attention.hip): LDS images of [token][64 x bf16] rows with one
// bank swizzle, MFMA fragments read from them, and the way a swapped-layout accumulator becomes an operand or leaves as rows.
#pragma once
#include "common.h"

namespace {

constexpr int HD = 64;              // head dim
constexpr int ROWB = HD * 2;        // LDS row bytes

__device__ __forceinline__ int rot3(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

// byte offset of 16-B chunk c of `row` inside an image
__device__ __forceinline__ int img_off(int row, int c) { return row * ROWB + ((c ^ rot3(row)) << 4); }

__device__ __forceinline__ bf16x8 lds_row_frag(const char* img, int row, int c) {
  return *reinterpret_cast<const bf16x8*>(img + img_off(row, c));
}

// transposed fragment for a 32x32x16 A operand: rows row0..row0+3 and row0+8..row0+11 (this lane addresses
// row0 + (t>>2)), columns col0 + 4*(t&3) .. +3 where t = lane & 15
__device__ __forceinline__ bf16x8 lds_tr_frag(const char* img, int row0, int col) {
  const int r = row0;
  const int o0 = r * ROWB + (((col >> 3) ^ rot3(r)) << 4) + ((col & 7) << 1);
  const int r8 = r + 8;
  const int o1 = r8 * ROWB + (((col >> 3) ^ rot3(r8)) << 4) + ((col & 7) << 1);
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(img + o0));
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(img + o1));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// registers 8s..8s+7 of a 32x32 fp32 accumulator -> bf16 B-operand fragment of k-step s
__device__ __forceinline__ bf16x8 acc_to_frag(const f32x16& a, int s) {
  union { uint32_t u[4]; bf16x8 v; } r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.u[j] = pack_bf16x2(a[8 * s + 2 * j], a[8 * s + 2 * j + 1]);
  return r.v;
}

// One row of a swapped-layout output tile pair (lane = (row, half); acc[eb] registers 4g .. 4g+3 = columns 32*eb + 8*g + 4*half ..)
// scaled, rounded to bf16 and stored as 16-byte pieces: the two lanes of a row trade 8-byte pieces first (merge_row_halves,
// common.h; 8-byte stores made the epilogues store-issue-bound: attention backward 146 -> 139 us at DeiT-B's layer).  Columns
// >= hd are skipped (hd is a multiple of 16).  Both lanes of a row must be active.
__device__ __forceinline__ void store_row_tile(bf16_t* row, const f32x16 (&acc)[2], int half, int hd, float sc) {
#pragma unroll
  for (int eb = 0; eb < 2; ++eb)
#pragma unroll
    for (int g4 = 0; g4 < 4; g4 += 2) {
      const int e0 = 32 * eb + 8 * g4;
      if (e0 < hd)
        *reinterpret_cast<uint4*>(row + e0 + 8 * half) = merge_row_halves(
            make_uint2(pack_bf16x2(acc[eb][4 * g4] * sc, acc[eb][4 * g4 + 1] * sc), pack_bf16x2(acc[eb][4 * g4 + 2] * sc, acc[eb][4 * g4 + 3] * sc)),
            make_uint2(pack_bf16x2(acc[eb][4 * g4 + 4] * sc, acc[eb][4 * g4 + 5] * sc), pack_bf16x2(acc[eb][4 * g4 + 6] * sc, acc[eb][4 * g4 + 7] * sc)));
    }
}

__device__ __forceinline__ bf16x8 load_row_frag_global(const bf16_t* base, size_t row, int ld, int col, bool valid) {
  bf16x8 z = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
  if (valid) z = *reinterpret_cast<const bf16x8*>(base + row * ld + col);
  return z;
}

}  // namespace
