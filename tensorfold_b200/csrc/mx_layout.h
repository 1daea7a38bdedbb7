// Layout of microscaled 4-bit operands (e2m1 codes, one power-of-two scale byte per 32 inputs) as the block-scaled tensor-core
// instruction wants them in shared memory, shared by the kernels and the host-side layout test.
//
// An operand is R rows (R a multiple of 8) of K inputs, K a multiple of 32 padded to whole steps of 64 (one MMA).  Stages of 256
// inputs are outermost, so that any run of rows that starts at a multiple of 128 is, for each stage, one run of codes and one of
// scales in memory: a bulk copy each, straight into the tile the MMA reads.
//
//     full stage   codes [R / 8][8 rows x 128 bytes], 16-byte pieces of a row permuted as the 128-byte swizzle does it
//                  scales [ceil(R / 128)][2][32][16 bytes]: for 128 inputs, byte 4 j + b of line i is row 32 j + i, block b
//     last stage   (K % 256 left: t steps of 64) codes [t][R / 8][8 rows x 32 bytes], 32-byte swizzle
//                  scales [ceil(R / 128)][ceil(t / 2)][32][16 bytes]
//
// A weight is super-blocks of 128 rows, each an operand of its own (R = 128), one after another: a block of threads streams its
// columns' bytes as they lie, and nothing is padded but K to 64 and N to 128.
#pragma once

#include <stdint.h>

#if defined(__CUDACC__)
#define TF_MX_HD __host__ __device__ __forceinline__
#else
#define TF_MX_HD inline
#endif

namespace tf {

constexpr int MX_BLOCK = 32;                     // inputs of a scale
constexpr int MX_STEP = 64;                      // inputs of one MMA
constexpr int MX_STAGE = 256;                    // inputs of a stage: one 128-byte swizzle line of codes a row
constexpr int MX_SB = 128;                       // rows of a super-block
constexpr int MX_SCALES = 1024;                  // scale bytes of a full stage per 128 rows
constexpr int MX_UNIT = MX_SB * 128 + MX_SCALES; // bytes of a full stage of a super-block
constexpr int MX_LONGEST = 0x7FFFFFFF - 255;     // of rows, columns or inputs: rounding up to tiles and stages stays an int

TF_MX_HD constexpr bool mx_sizes(int n, int k) { return n >= 1 && n <= MX_LONGEST && k >= MX_BLOCK && k <= MX_LONGEST && k % MX_BLOCK == 0; }
TF_MX_HD constexpr int mx_steps(int k) { return (k + MX_STEP - 1) / MX_STEP; }
TF_MX_HD constexpr int mx_stages(int steps) { return (steps + 3) / 4; }
TF_MX_HD constexpr int mx_scale_blocks(int rows) { return (rows + MX_SB - 1) / MX_SB; }
TF_MX_HD constexpr int64_t mx_stage_bytes(int rows) { return static_cast<int64_t>(rows) * 128 + mx_scale_blocks(rows) * MX_SCALES; }
TF_MX_HD constexpr int mx_tail_scales(int tail) { return (tail + 1) / 2 * 512; }       // per 128 rows
TF_MX_HD constexpr int64_t mx_operand_bytes(int rows, int steps) {
  return steps / 4 * mx_stage_bytes(rows) +
         (steps % 4 ? static_cast<int64_t>(rows) * 32 * (steps % 4) + mx_scale_blocks(rows) * mx_tail_scales(steps % 4) : 0);
}

// Byte offset of the 16 bytes that hold block `b` (32 codes) of row `r`.
TF_MX_HD int64_t mx_code_offset(int rows, int steps, int r, int b) {
  const int u = b >> 3, full = steps >> 2;
  if (u < full) return u * mx_stage_bytes(rows) + (r >> 3) * 1024 + (r & 7) * 128 + (((b & 7) ^ (r & 7)) << 4);
  const int j = (b & 7) >> 1;
  return full * mx_stage_bytes(rows) + static_cast<int64_t>(j) * rows * 32 + (r >> 3) * 256 + (r & 7) * 32 + (((b & 1) ^ ((r >> 2) & 1)) << 4);
}

// Byte offset of the scale of block `b` of row `r`; the four scales of blocks 4 i .. 4 i + 3 are neighbours.
TF_MX_HD int64_t mx_scale_offset(int rows, int steps, int r, int b) {
  const int u = b >> 3, full = steps >> 2, tail = steps & 3;
  const int line = (r & 31) * 16 + ((r & 127) >> 5) * 4 + (b & 3), half = (b & 7) >> 2;
  if (u < full) return u * mx_stage_bytes(rows) + static_cast<int64_t>(rows) * 128 + (r >> 7) * MX_SCALES + half * 512 + line;
  return full * mx_stage_bytes(rows) + static_cast<int64_t>(rows) * 32 * tail + (r >> 7) * mx_tail_scales(tail) + half * 512 + line;
}

// Stored row of packed row `r` where two projections are interleaved in tiles of 16 rows: (r, second) of the pair.
TF_MX_HD int mx_pair_row(int r) { return (r >> 5) * 16 + (r & 15); }
TF_MX_HD bool mx_pair_second(int r) { return (r & 16) != 0; }

}  // namespace tf
