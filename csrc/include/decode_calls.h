// Arguments of the decoding operators' launchers (csrc/kernels/rotary.cu, kv_cache.cu, cache_attention.cu, verify_draft.cu) as records of
// 8-byte fields, filled in by csrc/torch/decode_calls.cpp. Launchers and that module are built apart from one another: the build gives both
// a number for this file's text, and the module refuses a library that has another one.
#pragma once
#include <stdint.h>

#ifndef TB_DECODE_LAYOUT   // torsh_b200/_build.py gives it; a file that is compiled by hand has none to compare
#define TB_DECODE_LAYOUT 0
#endif

struct RotaryCall {
  const void *q, *k;
  void *yq, *yk;
  const long* pos;
  const double* freqs;
  long tokens, hq, hk, D, R, ldq, lhq, ldk, lhk, half, inverse, dtype;
  double magnitude;
};

struct KvCall {
  void* x[2];
  long strides[6];
  void* pages[2];
  float* scales[2];
  const int* table;
  long table_ld;
  const int *start, *counts;
  long B, T, H, D, page, pages_per_seq, num_pages, kind, dtype;
};

struct CacheAttnCall {
  const void* q;
  long qb, qt, qh;
  const void *k_pages, *v_pages;
  const float *k_scales, *v_scales;
  const int* table;
  long table_ld;
  const int *start, *counts;
  const uint8_t* mask;
  long mask_b, mask_t;
  void *out, *ws;
  long B, T, Hq, Hkv, D, page, pages_per_seq, num_pages, max_len, kind;
  int* status;
  double scale;
  mutable long kernels;   // out: what has been launched
};

struct VerifyCall {
  const void *probs, *draft;
  long pb, pt, db, dt;
  const long *tokens, *parents;
  long parents_ld;
  const float* uniforms;
  const int* counts;
  long* out;                    // accepted [B], next token [B], path [B, T]
  long B, T, V, dtype;
};
