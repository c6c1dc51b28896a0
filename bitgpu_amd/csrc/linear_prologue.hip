// The linear-attention layer's prologue: causal depthwise convolution + SiLU over the projected q | k | v
// channels of a batch's new rows, q and k normalized per head, the decays and write strengths, in one launch.
//
//   y_c[t] = silu(sum_j w_c[j] x_c[t - taps + 1 + j])     x before a sequence's first row: its kept inputs
//   q, k heads  y / sqrt(sum y^2 + 1e-6)                  v heads  y
//   g = -exp(a_log) softplus(a + dt_bias), beta = sigmoid(b)
//
// Bound by memory: every input row is read and every output row written once. A group of D / 4 lanes owns a
// head's channels, four a lane, and walks a run of up to 4 rows whose inputs (and the taps - 1 before them)
// are all loaded before the first is used. The lanes that hold a sequence's first run also read its kept
// inputs and, behind that, store the new ones: the sequence's other runs never look at them, so one slot may
// be both source and destination.
#include "bg_common.h"
#include "bg_linear.h"

namespace bg {

constexpr int kRun = 4;
constexpr float kUnitEps = 1e-6f;  // under the root of the q / k norm

typedef float f4 __attribute__((ext_vector_type(4)));

__device__ inline float silu(float y) { return y / (1.0f + expf(-y)); }

// A run of rows r0 .. of unit u for channels ch .. ch + 3 (a lane's): out points at the head's dims of the
// sequence's global row 0, rows `stride` values apart.
template <int D, int TAPS, bool UNIT>
__device__ __forceinline__ void conv_run(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs& a, const LinUnit& u,
                                         int r0, int ch, float* out, int stride) {
  constexpr int P = TAPS - 1;
  const int n = min(kRun, u.n - r0), C = L.channels;
  const int before = kLinChunk * u.chunk + r0;  // rows of the sequence before this run
  f4 x[P + kRun];
  const float* row = a.qkv + (size_t)(u.row0 + r0) * C + ch;
  const LinSeq s = b.seqs[u.seq];
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int t = before - P + i;
    x[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (t >= 0) x[i] = *(const f4*)(row + (ptrdiff_t)(i - P) * C);
    else if (s.src >= 0) x[i] = *(const f4*)(L.conv + ((size_t)s.src * P + (t + P)) * C + ch);
  }
#pragma unroll
  for (int i = 0; i < kRun; i++) x[P + i] = i < n ? *(const f4*)(row + (size_t)i * C) : f4{0.0f, 0.0f, 0.0f, 0.0f};
  float w[4][TAPS];
#pragma unroll
  for (int c = 0; c < 4; c++)
#pragma unroll
    for (int j = 0; j < TAPS; j++) w[c][j] = a.w[(size_t)(ch + c) * TAPS + j];
  if (before == 0) {  // the sequence's kept inputs: its last P rows, older kept ones where it has fewer
#pragma unroll
    for (int j = 0; j < P; j++) {
      const int t = s.rows - P + j;
      f4 keep = x[0];
#pragma unroll
      for (int i = 0; i < P; i++)
        if (t + P == i) keep = x[i];
      if (t >= 0) keep = *(const f4*)(a.qkv + (size_t)(s.row0 + t) * C + ch);
      *(f4*)(L.conv + ((size_t)s.dst * P + j) * C + ch) = keep;
    }
  }
#pragma unroll
  for (int i = 0; i < kRun; i++) {
    if (i >= n) break;
    f4 y;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      float t = w[c][0] * x[i][c];
#pragma unroll
      for (int j = 1; j < TAPS; j++) t = fmaf(w[c][j], x[i + j][c], t);
      y[c] = silu(t);
    }
    if constexpr (UNIT) {
      const float ss = group_sum<D / 4>(fmaf(y[0], y[0], fmaf(y[1], y[1], fmaf(y[2], y[2], y[3] * y[3]))));
      const float inv = 1.0f / sqrtf(ss + kUnitEps);
#pragma unroll
      for (int c = 0; c < 4; c++) y[c] *= inv;
    }
    *(f4*)(out + (size_t)(u.row0 + r0 + i) * stride) = y;
  }
}

// blockIdx.x: a unit; blockIdx.y: blocks of q and k heads, of v heads, then one of the gates. WIDE: a block is
// one head and its lane groups are a unit's runs (512 threads: all 16 at head dims of 128); otherwise its groups are heads
// and each walks all runs, which is for sequences of one run. 10,240 channels, one sequence of 1, 8, 64 rows 3.7, 4.5, 7.7 us
// wide, 3.8, 6.3, 31 not (there with runs of 8); 32 sequences of 1, 4, 8, 16 rows 6.0, 10.0, 11.3, 15.2 wide, 4.8, 7.5,
// 11.1, 16.1 not. Of 4,096 rows 81 us, 4.2 TB/s (runs of 8 and 256 threads 85, runs of 2 106).
template <int DK, int DV, int TAPS, bool WIDE>
__global__ __launch_bounds__(WIDE ? 512 : 256) void linear_prologue_kernel(LinLayer L, LinBatchView b, LinPrologueArgs a, int qk_blocks, int v_blocks) {
  constexpr int THREADS = WIDE ? 512 : 256;
  if ((int)blockIdx.x >= b.hdr->n_units) return;
  const LinUnit u = b.units[blockIdx.x];
  const int y = blockIdx.y;
  if (y < qk_blocks) {
    constexpr int LG = DK / 4, GROUPS = THREADS / LG;
    const int grp = threadIdx.x / LG, c = 4 * (threadIdx.x % LG);
    const int head = WIDE ? y : y * GROUPS + grp;
    if (head >= 2 * L.k_heads) return;
    const bool isq = head < L.k_heads;
    const int h = isq ? head : head - L.k_heads;
    for (int r0 = WIDE ? kRun * grp : 0; r0 < u.n; r0 += WIDE ? kRun * GROUPS : kRun)
      conv_run<DK, TAPS, true>(L, b, a, u, r0, head * DK + c, (isq ? a.q : a.k) + h * DK + c, L.k_heads * DK);
  } else if (y < qk_blocks + v_blocks) {
    constexpr int LG = DV / 4, GROUPS = THREADS / LG;
    const int grp = threadIdx.x / LG, c = 4 * (threadIdx.x % LG);
    const int head = WIDE ? y - qk_blocks : (y - qk_blocks) * GROUPS + grp;
    if (head >= L.v_heads) return;
    for (int r0 = WIDE ? kRun * grp : 0; r0 < u.n; r0 += WIDE ? kRun * GROUPS : kRun)
      conv_run<DV, TAPS, false>(L, b, a, u, r0, 2 * L.k_heads * DK + head * DV + c, a.v + head * DV + c, L.v_heads * DV);
  } else {
    for (int i = threadIdx.x; i < u.n * L.v_heads; i += THREADS) {
      const int r = u.row0 + i / L.v_heads, h = i % L.v_heads;
      const size_t at = (size_t)r * a.ab_stride + h, to = (size_t)r * L.v_heads + h;
      if (a.g) {
        const float t = a.a[at] + a.dt_bias[h];
        a.g[to] = -expf(a.a_log[h]) * (fmaxf(t, 0.0f) + log1pf(expf(-fabsf(t))));
      }
      if (a.beta) a.beta[to] = 1.0f / (1.0f + expf(-a.b[at]));
    }
  }
}

template <int DK, int DV, int TAPS>
static hipError_t launch_t(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs& a, hipStream_t st) {
  const int gates = a.g || a.beta;
  if (b.longest > kRun) {
    const int qk = 2 * L.k_heads, v = L.v_heads;
    hipLaunchKernelGGL((linear_prologue_kernel<DK, DV, TAPS, true>), dim3(b.n_units, qk + v + gates), dim3(512), 0, st, L, b, a, qk, v);
  } else {
    const int per_k = 1024 / DK, per_v = 1024 / DV;
    const int qk = (2 * L.k_heads + per_k - 1) / per_k, v = (L.v_heads + per_v - 1) / per_v;
    hipLaunchKernelGGL((linear_prologue_kernel<DK, DV, TAPS, false>), dim3(b.n_units, qk + v + gates), dim3(256), 0, st, L, b, a, qk, v);
  }
  return hipGetLastError();
}

template <int DK, int DV>
static hipError_t launch_d(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs& a, hipStream_t st) {
  if (L.taps == 2) return launch_t<DK, DV, 2>(L, b, a, st);
  if (L.taps == 3) return launch_t<DK, DV, 3>(L, b, a, st);
  return launch_t<DK, DV, 4>(L, b, a, st);
}

hipError_t launch_linear_prologue(const LinLayer& L, const LinBatchView& b, const LinPrologueArgs& a, hipStream_t st) {
  if (L.DK == 64) return L.DV == 64 ? launch_d<64, 64>(L, b, a, st) : launch_d<64, 128>(L, b, a, st);
  return L.DV == 64 ? launch_d<128, 64>(L, b, a, st) : launch_d<128, 128>(L, b, a, st);
}

}  // namespace bg
