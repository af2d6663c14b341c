// Cross-entropy epilogues of the logits product (csrc/gemm/gemm_sm100.cu) and what the two files share.
//
// An epilogue thread owns one row of a 256-column tile of z = x w^T in tensor memory, so the row statistics of the tile
// need no exchange between threads: the maximum m and s = sum exp(z - m), kept online over chunks of 32 columns.
// The gradient epilogue replaces z by (exp(z - m) / s - [column = label]) * dloss with the row's m and s over the whole
// vocabulary.  z itself is never written.  m and s are kept apart: lse = m + log s in fp32 would be off by up to
// |lse| 2^-24, which a token that the model is sure of (p near 1) carries into p - 1.
//
// exp(z - m) is ex2.approx of (z - m) log2(e) with the difference taken first: folding m log2(e) into one multiply-add
// would round that product once for the whole row, a common factor of up to |m| 2^-24 on every term of the sum.
#pragma once
#include "../include/common.cuh"

namespace emb {

struct CeArgs {
  const int64_t* labels;  // [T] vocabulary ids
  long long col0;         // vocabulary id of column 0
  long long vocab;        // ids in [0, vocab) other than `ignore` count; all other rows have loss and gradient 0
  long long ignore;
  float2* part;           // statistics: [column tiles, T] (m, s)
  float* target;          // statistics: [T] logit of the label, written where the label is one of the columns
  const float* top;       // gradient: [T] maximum and sum of exponentials of the whole vocabulary
  const float* sum;
  const float* dloss;     // gradient: [T]
  int low_row;            // gradient: 0, or the row that keeps what rounding to bf16 took from row 0, and so on
};

struct CeRow {
  float top, scale, g;  // scale = g / sum
  long long label;  // column of the label, or outside the columns
};

__device__ __forceinline__ bool ce_counts(const CeArgs& ce, int64_t label) {
  return label >= 0 && label < ce.vocab && label != ce.ignore;
}

__device__ __forceinline__ float ce_exp(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
  return y;
}

// Statistics of the 256 accumulator columns at `taddr` (columns n0.. of N) for this thread's row.
__device__ __forceinline__ void ce_stats_tile(const CeArgs& ce, uint32_t taddr, int n0, int N, int row, int rows, int tile) {
  const bool ok = row < rows;
  const int64_t label = ok ? ce.labels[row] : -1;
  const long long off = label - ce.col0 - n0;
  const int at = ok && ce_counts(ce, label) && off >= 0 && off < 256 ? (int)off : -1;  // column inside the tile
  float m = -INFINITY, s = 0.f;
  const int chunks = min(8, (N - n0 + 31) / 32);
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr + c * 32));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    const int n = N - n0 - c * 32;
    if (n < 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j >= n) r[j] = 0xff800000u;  // -inf: columns past the vocabulary
    }
    const int here = at - c * 32;
    if (__any_sync(0xffffffffu, here >= 0 && here < 32)) {  // (rare, and one branch for the warp)
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) z = j == here ? __uint_as_float(r[j]) : z;
      if (here >= 0 && here < 32) ce.target[row] = z;
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(r[j]));
    const float base = top == -INFINITY ? 0.f : top;  // a row of -inf so far keeps the sum 0
    float a[4] = {s * ce_exp(m - base), 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 32; ++j) a[j & 3] += ce_exp(__uint_as_float(r[j]) - base);
    s = (a[0] + a[1]) + (a[2] + a[3]);
    m = top;
  }
  if (ok) ce.part[(size_t)tile * rows + row] = make_float2(m, s);
}

__device__ __forceinline__ CeRow ce_load_row(const CeArgs& ce, int row, int rows) {
  CeRow r{0.f, 0.f, 0.f, -1};
  if (row < rows) {
    const int64_t label = ce.labels[row];
    if (ce_counts(ce, label)) {
      r.top = ce.top[row];
      r.g = ce.dloss[row];
      r.scale = __fdividef(r.g, ce.sum[row]);
      r.label = label - ce.col0;
    }
  }
  return r;
}

// 32 accumulators of columns col0.. -> the gradient of the logits; called by whole warps.  A row without a label gives 0 whatever z holds.
__device__ __forceinline__ void ce_grad_chunk(const CeRow& row, uint32_t* z, int col0) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    z[j] = row.g == 0.f ? 0u : __float_as_uint(ce_exp(__uint_as_float(z[j]) - row.top) * row.scale);
  const long long off = row.label - col0;
  const int here = off >= 0 && off < 32 ? (int)off : -1;
  // a label is rarely among these columns: one test for the warp, then selections (a branch for each lane and column
  // tripled the epilogue: 18 -> 61 us at 250 x 32001 x 512)
  if (__any_sync(0xffffffffu, here >= 0)) {
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = j == here ? __float_as_uint(__uint_as_float(z[j]) - row.g) : z[j];
  }
}

void linear_ce_gemm(const at::Tensor& x, const at::Tensor& w, const CeArgs& ce, bool grad, const at::Tensor& out);
void gemm_split_k(const at::Tensor& a, const at::Tensor& b, bool trans_a, const at::Tensor& parts);
at::Tensor gemm_tc(at::Tensor a, at::Tensor b, bool trans_a, bool trans_b, c10::optional<at::Tensor> out, bool accumulate,
                   int64_t variant);

}  // namespace emb
