// Arguments of the kernels around a tree of drafted tokens: its masks, its acceptance and the move of the accepted branch.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ss {

constexpr int kTreeRows = 64;  // rows of one sequence's tree: the bits of a mask

struct TreeMaskArgs {
  const int32_t* parents;  // [rows], among the sequence's rows; the first row's is not read
  const int32_t* cu;       // [seqs + 1]
  const int32_t* kv_len;   // [seqs], or null (then positions is)
  uint64_t* masks;         // [rows]
  int32_t* positions;      // [rows] or null
  int* err;
  int rows, seqs, max_rows;
};
hipError_t launch_tree_masks(const TreeMaskArgs& a, hipStream_t st);

struct TreeAcceptArgs {
  const float* target;     // [rows][vocab]
  const int32_t* tokens;   // [rows]
  const int32_t* parents;  // [rows]
  const int32_t* cu;       // [seqs + 1]
  int32_t* out;            // [seqs][4 + 2 max_rows]
  uint64_t* part;          // [rows][splits]
  int* err;
  int rows, seqs, max_rows, vocab, splits, span;
};
hipError_t launch_tree_accept(const TreeAcceptArgs& a, hipStream_t st);

struct KeepArgs {
  uint8_t* k;  // [layers][n_pages][kv_heads][page][dim], elements of `size` bytes
  uint8_t* v;  // [layers][n_pages][kv_heads][dim][page]
  uint8_t* scales;  // [layers][n_pages][kv_heads][2][page] or null
  const int32_t* cu;
  const int32_t* kv_len;
  const int32_t* table;  // [seqs][width]
  const int32_t* took;   // [seqs][4 + 2 max_rows]
  int* err;
  int64_t n_pages;
  int layers, seqs, rows, max_rows, kv_heads, dim, page_shift, width, size;
  int blocks;  // workgroups of a sequence (set by the launch)
};
hipError_t launch_keep_rows(KeepArgs a, hipStream_t st);

}  // namespace ss
