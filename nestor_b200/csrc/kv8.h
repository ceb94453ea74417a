// Argument blocks of the 8-bit key/value cache entry points (mirrored by ctypes structures in ops/cuda_decode.py).
#pragma once
#include <cuda_runtime.h>

typedef struct {
  void* codes[2];     // keys, values: [L, H, nb, U, 512] bytes
  float* scale[2];    // [L, H, nb]
  void* open[2];      // originals of the youngest two blocks [L, H, 2, 64, D]
  int* status;        // device status word
  int L, H, nb, D, U;
  int code;           // 0 int8, 1 e4m3
  int type;           // of `open` and of appended rows: 0 bf16, 1 fp16, 2 fp32
} nb_kv8_cache;

typedef struct {
  const void* src[2];         // appended rows: element (row, head, d) at row * row_stride + head * head_stride + d
  long row_stride[2], head_stride[2];
  void* dst[2];               // rows read back: [rows, H, D] contiguous
  const int* seg;             // [L + 1] row bounds
  const int* start;           // [L] first entry of each list
  int rows, max_rows;
} nb_kv8_rows;

typedef struct {
  const void* q;
  void* out;
  long q_row, q_head, o_row, o_head;
  const int* seg;             // [L + 1]
  const int* len;             // [L] entries of each list, the new rows' among them
  int rows, max_rows, group;  // group: query heads that share a key head
  int q_type;                 // of q and out: 0 bf16, 1 fp16, 2 fp32
  int zero_tail;
  float scale_log2;           // softmax scale * log2(e)
} nb_kv8_attn;
