// Paged KV cache: what its kernels (paged_prologue.hip, paged_attn.hip) and its entry points
// (paged_api.hip) share.
//
// A pool holds, per layer, n_pages pages of `page` slots (a power of two, 32 to 256):
//   K   [page][kv_head][slot][D]
//   V   [page][kv_head][slot / 32][4 panels][D][8]   (the transposed 32-slot tiles of bg_common.h)
//   Ks, Vs (q8) [page][kv_head][slot][D / 32] f32
// so one page of one layer is laid out as a KvCache layer of `page` slots is, and the row stores of
// bg_qkrow.h / bg_store.h write it through a LayerView of that page.
#pragma once

#include "bg_kernels.h"
#include "bg_paged_plan.h"

namespace bg {

// What a captured launch reads of the batch instead of its arguments, so that a batch set again between
// replays is the one the replay runs.
struct PagedHeader {
  int n_units, n_merges, n_tokens, n_v_single, n_v_group;
  int n_many, n_mid, n_merge_few;  // units of 128 rows (the first) and of 32; merges of few partials (the first)
  float* ws_o;      // [part][head][D] unnormalized output of a partial
  float2* ws_ml;    // [part][head] its (m, l), m in base 2
};

// The batch as the kernels see it: device arrays at fixed addresses, written by one upload a set.
struct PagedBatchView {
  const PagedHeader* hdr;
  const PagedUnit* units;
  const PagedTok* toks;
  const PagedMerge* merges;
  const int* pages;
  const int* dst;        // [tokens] page * page size + slot
  const int* pos;        // [axes][pos_stride] rotary positions
  const int* v_single;
  const int* v_group;
  int pos_stride;
  int page_shift;
  int H, G;
  // the set counts and their choices; all zero for a launch under capture, which reads hdr
  int n_units, n_many, n_mid, n_merges, n_merge_few, n_tokens, n_v_single, n_v_group;
  int stream_few;        // the few-row units' pages are read once, and too many to stay in a cache
  int captured;
};

struct PagedAppendArgs {
  const float* q; int q_stride;
  const float* k; const float* v;
  const float* q_gamma; const float* k_gamma; float eps;
  const float* cos_tab; const float* sin_tab; int rot_dim;
  int axes;                 // 1: every pair by axis 0
  uint32_t pair_axis[8];    // 2 bits a rotary pair
  float* q_out;
  int num_cus;
};
hipError_t launch_paged_prologue(const LayerView& pool, const PagedBatchView& b, const PagedAppendArgs& a, hipStream_t st);

struct PagedAttnArgs {
  const float* q;
  float scale;
  const float* gate; int gate_stride;
  float* out;
  int num_cus;
};
hipError_t launch_paged_attention(const LayerView& pool, const PagedBatchView& b, const PagedAttnArgs& a, hipStream_t st);

// copies n16 16-byte words from pinned host memory to each of up to 9 device arrays (one launch a set)
struct PagedUpload {
  const void* src[9];
  void* dst[9];
  unsigned n16[9];
};
hipError_t launch_paged_upload(const PagedUpload& u, hipStream_t st);

}  // namespace bg
