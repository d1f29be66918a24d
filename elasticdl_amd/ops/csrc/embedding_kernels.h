// What the embedding kernels (embedding_kernels.hip) and their bindings share.
#pragma once

#include <cstdint>

// element types
#define EDL_T_F32 0
#define EDL_T_BF16 1
#define EDL_T_F16 2

#define EDL_BAG_SUM 0
#define EDL_BAG_MEAN 1
#define EDL_BAG_SQRTN 2

struct edl_bag {
  const void* table;  // [V, D], rows ld apart
  int64_t ld, V;
  int D, type;
  int vec;          // elements of an aligned load; D is a multiple of it
  const void* ids;  // [B, L] of int32 or int64, below 0: no token
  bool ids64;
  int64_t B;
  int L;
  const void* weights;  // [B, L] or null
  int w_type;
  int combiner;
  float scale;
  void* out;    // forward: [B, D] of the table's type
  float* coef;  // [B]: scale / norm; forward writes it where it is not null
  const void* dy;  // backward: [B, D]
  float* dw;       // [B, L]
};

struct edl_segments {
  // [N], sorted by key, then by pos; on borders of 16 bytes, with room to
  // read up to a multiple of 8
  const uint32_t *keys, *pos;
  int64_t N;
  int chunk;       // tokens that a group of lanes takes: a multiple of 8
  uint32_t limit;  // keys from here on are no rows
  const void* src;  // [*, D] contiguous: row pos / L
  int D, type, vec, L;
  float scale;
  const float* coef;  // by row of src, or null
  const void* weights;  // by pos, or null
  int w_type;
  void* out;  // [limit, D] of src's type: row keys[i]
  // where the small sort was: each run's first token, how many runs there
  // are, and their rows (null: the run's own number); keys is not used
  const uint32_t *starts, *runs, *rows;
  // else a workspace: a row of sums for each chunk's open beginning and end
  float* part;                // [chunks, 2, D]
  uint32_t *head, *tail;      // [chunks]: their keys
};

#define EDL_RANGE_PARTS 256
#define EDL_SORT_TILE 4096
#define EDL_SORT_BINS 2048  // most of a pass
#define EDL_SORT_SMALL 8192
#define EDL_SORT_FAR (192 * 1024)
