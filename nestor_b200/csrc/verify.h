// Argument block of nb_verify_draft (mirrored by a ctypes structure in ops/cuda_decode.py).
#pragma once
#include <cuda_runtime.h>

typedef struct {
  const void* p;            // [B, n + 1, V] target probabilities, rows contiguous
  const void* q;            // [B, n, V] draft probabilities or null
  const void* tokens;       // [B, n] drafted tokens
  const float* u;           // [B, n]
  const float* w;           // [B]
  const int* len;           // [B] drafted tokens of each sequence, or null (n each)
  int* accepted;            // [B]
  int* token;               // [B]
  long p_batch, p_row, q_batch, q_row;
  int B, n, V;
  int type;                 // of p and q: 0 bf16, 1 fp16, 2 fp32
  int tokens_64;
} nb_verify_args;
