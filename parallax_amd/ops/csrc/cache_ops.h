// Arguments of the kernels that cache_ops.cpp calls.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

struct HeadNormStore {
  uint16_t* out;  // [T, Hq, D]
  const uint16_t *q, *k, *v, *q_w, *k_w;
  void *k_cache, *v_cache;  // [NB, Hk, BS, D], [NB, Hk, D, BS]
  const int* positions;
  const float* cos_sin;  // [P, rot]
  const int64_t* slots;
  int T, Hq, Hk, D, rot, BS, P;
  int64_t num_slots;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides
  float eps, inv_k, inv_v;
};

struct SharedPrefix {
  uint16_t* out;           // [B, Hq, D]
  const uint16_t* q;       // [B, Hq, D] rows at q_stride
  const uint8_t *k, *v;    // [NB, Hk, BS, D], [NB, Hk, D, BS], bf16 | fp8
  const int *tables, *lens, *group, *prefix;  // [B, max_blocks], [B], [B], [N]
  const float* sinks;      // [Hq] or null
  int B, N, Hq, Hk, D, shift, max_blocks, num_pages;
  int64_t q_stride;
  float scale, v_scale, softcap;  // scale: with that of an fp8 cache's keys
  int window;
  int runs;      // workgroups of a key/value head
  float* p_acc;  // [p_parts, Hk, SP_ITEMS, D]: part run, or run + item tile
  float* p_ml;   // [p_parts, Hk, SP_ITEMS, 2] maxima in units of log2, sums
  int4* p_info;  // [B, Hq]: first part, parts, place in them; rows of a group only
  float* s_acc;  // [s_parts, Hq, D]: part wave + row
  float* s_ml;   // [s_parts, Hq, 2]
  int2* s_info;  // [B]: first and last wave; rows with tokens behind a prefix only
  int* has;      // [B]: 1: of a prefix, + 2: behind one
};
