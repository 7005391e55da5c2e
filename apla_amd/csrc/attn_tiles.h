// LDS tile layout and MFMA operand fragments shared by the attention kernels (attention.hip, attn_mod.hip): 64-column 16-bit tiles, products
// on v_mfma_f32_32x32x16 with the reduction axis on the lane's registers.
#pragma once
#include "common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// 64-column bf16 tile (128-byte rows), 16-byte chunk index XOR f(row): conflict-free for ds_read_b128 row fragments
// (32 rows x one chunk) and for ds_read_b64_tr_b16 blocks (4 rows x 64 bytes per half-wave).
__device__ __forceinline__ int tile_off(int row, int chunk) {
  const int f = (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  return row * 128 + ((chunk ^ f) << 4);
}

// Row fragment (A operand, 32 rows x 16 k): lane l holds tile[row0 + (l&31)][16*ks + 8*(l>>5) + 0..7]
__device__ __forceinline__ bf16x8 row_frag(const char* lds, int row0, int ks, int lane) {
  return *(const bf16x8*)(lds + tile_off(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}

// Transposed fragment (A operand = tile^T, 32 "columns of the tile" x 16 "rows of the tile"):
// element j of lane l = tile[rbase + 8*(j>>2) + 4*(l>>5) + (j&3)][c0 + (l&31)], matching the k-order in which a 32x32 f32
// accumulator is consumed as the other operand (see cdna guide: accumulator tile as next MFMA operand).
__device__ __forceinline__ bf16x8 tr_frag(const char* lds, int rbase, int c0, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int col = c0 + 16 * (g & 1) + 4 * (i & 3);  // this lane's address: 4 consecutive columns of one row
  const int r = rbase + 4 * (g >> 1) + (i >> 2);
  const int a0 = tile_off(r, col >> 3) + ((col & 4) << 1);
  const int a1 = tile_off(r + 8, col >> 3) + ((col & 4) << 1);
  bf16x4 lo = DS_READ_TR16_B64_H16(lds + a0);
  bf16x4 hi = DS_READ_TR16_B64_H16(lds + a1);
  bf16x8 out;
  out[0] = lo[0]; out[1] = lo[1]; out[2] = lo[2]; out[3] = lo[3];
  out[4] = hi[0]; out[5] = hi[1]; out[6] = hi[2]; out[7] = hi[3];
  return out;
}

__device__ __forceinline__ bf16x8 acc_to_operand(const f32x16& a, int s) {
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = (bf16)a[8 * s + j];
  return o;
}

// row index (within a 32-row tile) of accumulator register `reg` for lane half h
__device__ __forceinline__ int acc_row(int reg, int h) { return (reg & 3) + 8 * (reg >> 2) + 4 * h; }

// Register fragment straight from global (B operand with the matrix row on the lane):
// lane l holds M[row][16*ks + 8*(l>>5) + 0..7] for ks = 0..3
__device__ __forceinline__ void load_row_frags(bf16x8 (&f)[4], const bf16* rowptr, int lane) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) f[ks] = *(const bf16x8*)(rowptr + 16 * ks + 8 * (lane >> 5));
}

// Store a transposed accumulator pair (acc[dt][reg] = X[d = 32dt + acc_row(reg,h)][row on lane]) as bf16 to a row-major
// [rows, 64] slice: 8-byte pieces of 4 consecutive d.
__device__ __forceinline__ void store_acc_T(const f32x16 (&acc)[2], bf16* rowptr, int h, float mul) {
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x4 v = pack4(acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul, acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul);
      *(bf16x4*)(rowptr + 32 * dt + 8 * g + 4 * h) = v;
    }
}

}  // namespace
