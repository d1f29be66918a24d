// What the 8-bit kernels (fp8_kernels.hip) and their bindings share.
#pragma once

#include <cstdint>

#define EDL_FP8_BLOCK 128

// element types of the tensors around the 8-bit products
#define EDL_T_F32 0
#define EDL_T_BF16 1
#define EDL_T_F16 2

#define EDL_ACT_NONE 0
#define EDL_ACT_RELU 1
#define EDL_ACT_SIGMOID 2

// a workgroup's share of a product: 64 x 128, 128 x 128 or 256 x 256
#define EDL_TILE_RING 0
#define EDL_TILE_128 1
#define EDL_TILE_256 2

struct edl_fp8_quant {
  const void* x;  // [R, C], rows ld apart
  int64_t ld, R, C;
  int type;
  bool wide;   // 16-byte loads of 8 neighbours are aligned
  bool tile;   // a scale for 128 x 128, else for 128 neighbours
  bool deriv;  // x is a gradient behind an activation; see act
  int act;
  uint8_t* rows;        // [R, rows_ld], blocks along C; may be null
  uint8_t* rows_scale;  // [rows_ld / 128, rows_rp]
  int64_t rows_ld, rows_rp;
  uint8_t* cols;        // [C, cols_ld], blocks along R; may be null
  uint8_t* cols_scale;  // [cols_ld / 128, cols_rp]
  int64_t cols_ld, cols_rp;
  const uint8_t* mask;  // relu: a bit for each output, rows mask_ld bytes apart
  int64_t mask_ld;
  const void* y;  // sigmoid: the output, rows y_ld apart
  int64_t y_ld;
  bool y_wide;
  float* sums;  // [row tiles, C]: each tile's column sums; may be null
};

struct edl_fp8_gemm {
  const uint8_t *a, *b;    // [M, ld], [N, ld]
  const uint8_t *sa, *sb;  // [ld / 128, a_rp], [ld / 128, b_rp]
  int64_t M, N, ld, a_rp, b_rp;
  const void* bias;  // [N] or null
  int bias_type;
  int act;
  void* c;  // [M, N], contiguous
  int c_type;
  bool c_wide;    // 16-byte stores of 16 neighbours are aligned
  bool wide;      // sums in 32 bits: c is of 32 bits, or there is a mask
  uint8_t* mask;  // relu: bits of c > 0, rows mask_ld bytes apart; may be null
  int64_t mask_ld;
  int tile;     // EDL_TILE_*
  int splits;   // over the contraction
  float* part;  // [splits, M, part_ld] where splits > 1
  int64_t part_ld;  // N rounded up to 16
};

// what follows one or two products: see edl_fp8_gemm_run
struct edl_fp8_finish {
  edl_fp8_gemm g[2];
  int64_t join_blocks[2];
  const float* sums;  // [tiles, C]; may be null
  int64_t tiles, C;
  void* out;  // [C]
  int out_type;
};
