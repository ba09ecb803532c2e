// Arguments of the rotary kernel that writes the cache, and of the kernel that moves its pages.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ss {

struct RopeArgs {
  const uint16_t* q;  // [rows][heads][dim]; strides in elements, dimensions contiguous
  const uint16_t* k;  // [rows][kv_heads][dim]
  const uint16_t* v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  uint16_t* out;             // [rows][heads][dim]
  const int32_t* positions;  // [axes][rows], axes pos_stride apart
  int64_t pos_stride;
  const double* inv_freq;  // [rot / 2]
  const int32_t* axis;     // [rot / 2] or null (axis 0)
  uint16_t* k_pages;       // [n_pages][kv_heads][page][dim]
  uint16_t* v_pages;       // [n_pages][kv_heads][dim][page]
  const int32_t* cu;
  const int32_t* kv_len;
  const int32_t* table;
  int* err;
  int64_t n_pages;
  int rows, seqs, max_rows, heads, kv_heads, dim, rot, axes, page_shift, width, adjacent;
  float factor;
  int tiles;        // groups of 8 positions of one sequence
  int head_groups;  // workgroups that share the heads of a tile
  uint8_t* scales;  // [n_pages][kv_heads][2][page] exponents: the pages then hold e4m3 numbers; or null
};
hipError_t launch_rope_append(const RopeArgs& a, bool fp16, hipStream_t st);

struct MoveArgs {
  uint8_t* k;  // [layers][n_pages][page_bytes]
  uint8_t* v;
  const int32_t* src;
  const int32_t* dst;
  int32_t* table;  // entries equal to a src become its dst; or null
  int* err;
  int64_t n_pages, page_bytes, entries;
  int layers, n;
  unsigned copy_blocks, table_blocks;
  uint8_t* scales;  // [layers][n_pages][scale_bytes] that move with the pages; or null
  int64_t scale_bytes;
  unsigned scale_blocks;
};
hipError_t launch_move_pages(MoveArgs a, hipStream_t st);

}  // namespace ss
