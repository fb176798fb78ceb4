// What the attention kernels over the cache held in 8 bits share.
#pragma once

#include "rb_common.cuh"

RB_EXPORT int rb_cache8_block(int page_size);      // cache8.cu

struct Params8 {
  const __nv_bfloat16* q;     // [T, H, D]
  __nv_bfloat16* out;         // [T, H * D]
  RbPagedLayer cache;
  const float* k_scale;       // [page][kv head][blocks of a page]
  const float* v_scale;
  int block;
  const int* tok_pos;
  const int* tok_slot;
  int H;
  float scale;
  int window, keep;
  const float* sinks;
  float softcap;
};
