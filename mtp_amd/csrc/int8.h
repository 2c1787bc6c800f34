// The int8 products' kernels as the entry points see them.
#pragma once

#include "common.h"

// a rows [rows][K] with a scale each; b [N][K] with a scale per channel, of one expert or of all
// of them, N * K bytes apart. Output row r of a tile comes from a's row row_src[r] / src_div (r
// without row_src).
struct Int8Args {
  const int8_t* a;
  const float* a_scale;
  const int32_t* row_src;
  int src_div;
  uint32_t a_bytes;
  const int8_t* b0;       // SiLU products: gate
  const int8_t* b1;       // SiLU products: up
  const float* s0;
  const float* s1;
  const i32x4* tiles;     // {expert, first row, rows, 0}; NULL: consecutive rows of one matrix
  int m_tiles;            // entries of the tile table (behind them: how many are in use), or the
                          // row blocks of one matrix
  int M, N, K;
  void* out;              // [M][N]
  const void* bias;       // [N] or NULL
};

// Quantise rows of the dtype to int8 with a scale each.
hipError_t launch_quantize(const void* x, int T, int K, int dtype, int8_t* q, float* scale,
                           hipStream_t s);
// The kernel of a product and its rows per tile (the bm of an expert table).
enum { kInt8Stream = 0, kInt8Ring = 1, kInt8Tile = 2 };
struct Int8Plan {
  int kind, bm;
};
Int8Plan int8_experts_plan(int64_t slots, int E);
Int8Plan int8_matrix_plan(int64_t M, int64_t N);
hipError_t launch_int8_product(const Int8Args& a, Int8Plan plan, bool silu, int dtype,
                               hipStream_t s);
