// Linear attention with a decay for each head: what its kernels (linear_prologue.hip, linear_attn.hip,
// linear_chunk.hip) and its entry points (linear_api.hip) share, and those of the 4-bit projections (gemv4.hip).
//
// Per layer, slot and value head one f32 matrix [v_dim][k_dim] (the state, transposed: a row holds what one
// value dim has gathered over the key dims), and per layer and slot the convolution's last inputs,
// [conv_width - 1][channels], channels = q heads | k heads | v heads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bg {

constexpr int kLinChunk = 64;     // rows of a unit
// Sequences of at least this many new rows are done in chunks of 64, shorter ones row by row. With 32 heads of 128 x 128
// one sequence of the delta rule takes 5.7 + 0.86 us a row so and 24 us as a chunk (4 sequences 6.1 + 0.92 and 36, 64 of
// them 50 + 5.5 and 350: they meet at 22, 33 and 54 rows), one of the sum rule 5.9 + 0.66 and 17.6 (64: 50 + 4.8 and 254: at
// 18 and 42). A batch does not know the rule: a number between.
constexpr int kLinChunkFrom = 28;
// Most bytes of chunk operands at a time. Of one sequence: what the scan reads should still be in the 256 MiB behind the
// L2s that the preparation wrote it to, beside the rows themselves (8192 rows of 48 heads, 4.7 MB a chunk: 64 MiB 751 us,
// 96 706, 112 684, 128 651, 144 651, 160 626, 176 628, 208 684, 256 684). Of several: a pass should hold many sequences,
// whose scans run side by side (2048 rows of 32 heads: two sequences 160 MiB 285 us, 384 225; four 570 and 441; eight 970
// and 966).
constexpr size_t kLinCached = (size_t)160 << 20, kLinSpace = (size_t)384 << 20;

// a row's decay as hi + lo: the rounding of one float would add up over the rows of a constant decay
__device__ inline void fade_of(float g, float& hi, float& lo) {
  const double e = exp((double)g);
  hi = (float)e;
  lo = hi < __builtin_inff() ? (float)(e - (double)hi) : 0.0f;
}

// A sequence of the batch: its new rows are rows row0 .. row0 + rows - 1 of the call's tensors; its state is
// read from slot src (-1: zeros) and left in slot dst.
struct LinSeq {
  int row0, rows, src, dst;
  int unit0, n_units;             // its units: runs of 64 rows, in order
  int pad[2];
};
struct LinUnit {
  int seq, row0, n, chunk;        // rows row0 .. row0 + n - 1, the chunk-th 64 of sequence `seq`
};
// What a captured launch reads of the batch instead of its arguments, so that a batch set again between
// replays is the one the replay runs.
struct LinHeader {
  int n_seqs, n_tokens, n_units;
  int n_chunked, n_chunk_units;   // the first ones
  int pad;
  char* ws;                       // operands of `window` chunks
};

// The batch as the kernels see it: device arrays at fixed addresses, written by one upload a set. The counts
// are upper bounds for a launch under capture, whose kernels compare with hdr.
struct LinBatchView {
  const LinHeader* hdr;
  const LinSeq* seqs;
  const LinUnit* units;
  int n_seqs, n_tokens, n_units;
  int longest;                    // rows of the longest sequence as the batch is set (not a bound)
  int most;                       // of the longest one that is not chunked, at most
  int n_chunked, n_chunk_units;
  int window;                     // chunks that the workspace holds
  char* ws;                       // NULL under capture: hdr's
};

// One layer of the caller's state.
struct LinLayer {
  float* state;                   // [slot][v_head][DV][DK]
  float* conv;                    // [slot][taps - 1][channels]
  int k_heads, v_heads, DK, DV, taps, channels;
};

struct LinPrologueArgs {
  const float* qkv;               // [rows][channels]
  const float* w;                 // [channels][taps]
  const float* a; const float* b; int ab_stride;
  const float* a_log; const float* dt_bias;
  float *q, *k, *v, *g, *beta;
};
hipError_t launch_linear_prologue(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs& a, hipStream_t st);

struct LinAttnArgs {
  const float *q, *k, *v;
  const float* g; int g_stride;   // 0: one decay a head
  const float* beta;              // NULL: a plain sum
  float scale;
  const float* gate; const float* norm; float eps;
  float* out;
};
hipError_t launch_linear_rows(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st);

hipError_t launch_linear_chunks(const LinLayer& L, const LinBatchView& b, const LinAttnArgs& a, hipStream_t st);
size_t linear_unit_bytes(int DK, int k_heads, int v_heads);  // a chunk's operands in the workspace

// gemv4.hip: 4-bit projections. Code k of row n is bits 4 (k % 8) .. of codes[n][k / 8]; a weight is
// (code - 8) * scale, or code * scale + min where mins is given, one scale (and min) per `group` weights.
struct Gemv4Args {
  const float* x; int M, K;
  const uint32_t* codes; const void* scales; const void* mins;
  int scale_f16, group;
  int N0, N1, N2;
  float *out0, *out1, *out2;
  const float* resid;
  char* room;  // of gemv4_room bytes: x prepared for more than four rows
};
size_t gemv4_room(int M, int K);
hipError_t launch_gemv4(const Gemv4Args& a, hipStream_t st);

}  // namespace bg
