// Linear cross entropy: loss_t = log sum_v exp(z_tv) - z_t,label(t) with z = x w^T, without keeping z [T, V].
//
// forward:  one product whose epilogue (linear_ce.cuh) leaves (max, sum exp) for each row and 256 columns, and the
//           label's logit; a join over the column tiles.  2 T V H operations, and T V / 32 bytes of statistics in place
//           of 2 T V of logits.
// backward, per piece [v0, v1) of the vocabulary, with P = (softmax(z) - onehot) dloss of that piece only:
//           product again with the gradient epilogue -> P (bf16);   dx += P w[v0:v1] (fp32);   dw[v0:v1] (+)= P^T x.
//           6 T V H operations: 2 more than with kept logits.
// 8192 x 129024 x 4096: forward 5.2 ms (1654 TFLOP/s before the power limit), a whole step 25.8 ms, 8 T V H at 1343
// TFLOP/s (the library's sustained rate: 1358); 4096 x 32000 x 4096: 3.23 ms; 250 x 32001 x 512: 76 us.
//
// P is rounded to bf16 because the tensor cores multiply bf16; everything summed over V or T is summed in fp32.  The
// roundings of P add up like the terms that they belong to, so however many tokens there are dx and dw are off by about
// the square root of two of what rounding the result alone costs (relative error 0.0024 against 0.00166 at 129 to 8000
// tokens and 1000 to 32000 words; the output layer with kept bf16 logits: 0.0024 to 0.0026).  Up to 128 rows P is kept as two
// bf16 rows, P and its rounding error, and the error is that of the result alone: the epilogue of the single-SM product, a
// tile of 128 rows, writes both, and reading w bounds the backward (weights of 129024 x 4096, 65 / 128 rows: 790 to 870 / 840
// to 960 us by run; with one row each 730 / 730 to 810).  With more rows the tensor cores bound it, and 10 T V H instead of 6 would cost in proportion.
#include "linear_ce.cuh"

#include <c10/cuda/CUDAGuard.h>

namespace emb {
namespace {

// Joins the tiles' statistics of a row: 32 rows a CTA, 32 slices of the tiles, in a fixed order.
//
// The label's logit is taken again as an fp32 dot product of x's row and w's.  Tensor cores cut their sums off towards
// zero at every step of K (3.8e-6 of a logit at K = 4096, the library's product alike), which the loss of a token with a
// large logit shows; with the label's own term exchanged in the sum and in the difference the loss of such a token
// depends on the exact value, and the rest of the sum on small logits (4096 tokens of which some are certain: relative
// error of the losses 1.9e-6 -> 0.75e-6).  `out_sum` stays the sum that the gradient's logits belong to.
__global__ void __launch_bounds__(1024) ce_join_kernel(CeArgs ce, const __nv_bfloat16* __restrict__ x, int64_t ldx,
                                                       const __nv_bfloat16* __restrict__ w, int64_t ldw, int H, int T,
                                                       int tiles, int V, bool raw, float* __restrict__ out,
                                                       float* __restrict__ out_top, float* __restrict__ out_sum,
                                                       float* __restrict__ out_loss_sum) {
  __shared__ float sm[32][33], ss[32][33];
  grid_dependency();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  if (row < T) {
#pragma unroll 4
    for (int i = slice; i < tiles; i += 32) {
      const float2 v = ce.part[(size_t)i * T + row];
      const float top = fmaxf(m, v.x), base = top == -INFINITY ? 0.f : top;
      s = s * __expf(m - base) + v.y * __expf(v.x - base);
      m = top;
    }
  }
  sm[slice][lane] = m;
  ss[slice][lane] = s;
  // warp `slice` finishes row t
  const int t = blockIdx.x * 32 + slice;
  int64_t label = -1;
  if (t < T) label = ce.labels[t];
  const bool own = t < T && ce_counts(ce, label) && label >= ce.col0 && label < ce.col0 + V;
  float dot = 0.f;
  if (own) {
    const uint4* a = reinterpret_cast<const uint4*>(x + t * ldx);
    const uint4* b = reinterpret_cast<const uint4*>(w + (label - ce.col0) * ldw);
#pragma unroll 4
    for (int i = lane; i < H / 8; i += 32) {
      float f[8], g[8];
      unpack8(a[i], f);
      unpack8(b[i], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot += f[j] * g[j];
    }
  }
  dot = warp_sum(dot);
  __syncthreads();
  if (t >= T) return;
  m = sm[lane][slice];
  s = ss[lane][slice];
  const float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  s = warp_sum(s * __expf(m - base));
  if (lane != 0) return;
  out_top[t] = top;
  out_sum[t] = s;
  float z = s;
  if (own) {
    float rest = s - __expf(ce.target[t] - top);
    if (rest < 0.f) rest = 0.f;  // (a NaN stays: fmaxf would drop it, and with it a diverged weight from every loss)
    z = rest + __expf(dot - top);
  }
  // a rank's share of the vocabulary leaves the label's logit and the sum that belongs to it, for the caller to join
  if (raw) out_loss_sum[t] = z;
  out[t] = !own ? 0.f : raw ? dot : logf(z) + (top - dot);
}

// Sum over the n fp32 parts, `stride` vectors apart, in order; with `low` each part holds a second summand that many vectors
// further on.  Rounded into the dense bf16 `out`, or added to `accum` with `width` vectors in a row and `ld` elements between
// rows.
__global__ void parts_sum_kernel(const float4* __restrict__ parts, int n, int64_t stride, int64_t low, int64_t vecs,
                                 __nv_bfloat16* __restrict__ out, float* __restrict__ accum, int width, int64_t ld) {
  grid_dependency();
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < vecs; i += (int64_t)gridDim.x * blockDim.x) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < n; ++p) {
      const float4 v = parts[p * stride + i];
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
      if (low) {
        const float4 u = parts[p * stride + low + i];
        a.x += u.x;
        a.y += u.y;
        a.z += u.z;
        a.w += u.w;
      }
    }
    if (accum) {
      float* dst = accum + i / width * ld + i % width * 4;
      dst[0] += a.x;
      dst[1] += a.y;
      dst[2] += a.z;
      dst[3] += a.w;
    } else {
      __nv_bfloat162 h[2] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w)};
      reinterpret_cast<uint2*>(out)[i] = *reinterpret_cast<uint2*>(h);
    }
  }
}

// Joins parts [n, >= rows, H] into `rows` rows of dst (dense bf16, or fp32 that is added to).
void sum_parts(const at::Tensor& parts, int64_t n, bool low, int64_t rows, const at::Tensor& dst) {
  const int64_t H = parts.size(2), vecs = rows * H / 4;
  const int grid = (int)std::min<int64_t>((vecs + 255) / 256, (int64_t)num_sms() * 8);
  const bool add = dst.scalar_type() == at::kFloat;
  launch_early(parts_sum_kernel, grid, 256, 0, reinterpret_cast<const float4*>(parts.data_ptr()), (int)n,
               parts.size(1) * H / 4, low ? vecs : 0, vecs,
               add ? nullptr : reinterpret_cast<__nv_bfloat16*>(dst.data_ptr()), add ? dst.data_ptr<float>() : nullptr,
               (int)(H / 4), dst.stride(0));
  EMB_LAUNCH_CHECK();
  count_launch();
}

// How a product of few output tiles cuts its K: `shares` so that every SM (up to 128 rows, a 128 x 256 tile each) or pair
// (256 x 256 tiles) gets one tile of at least 512 of K; 1: not at all.  `pad`: rows of a part.
struct Split {
  bool pair;
  int64_t tiles, slots, pad;
  Split(int64_t rows, int64_t cols) {
    pair = rows > 128;
    tiles = (pair ? (rows + 255) / 256 : 1) * ((cols + 255) / 256);
    slots = pair ? num_sms() / 2 : num_sms();
    pad = pair ? (rows + 255) / 256 * 256 : rows;
  }
  int64_t shares(int64_t k) const { return std::max<int64_t>(1, std::min(slots / tiles, k / 512)); }
};

void check_ce(const at::Tensor& x, const at::Tensor& w, const at::Tensor& labels) {
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.size(1) % 8 == 0 && x.size(1) > 0 &&
                        w.size(0) > 0, "x must be [T, H] and w [V, H] with H a multiple of 8");
  TORCH_CHECK_VALUE(x.scalar_type() == w.scalar_type(), "x and w must have the same type");
  TORCH_CHECK_VALUE(labels.scalar_type() == at::kLong && labels.dim() == 1 && labels.size(0) == x.size(0),
                    "labels must be int64 [T]");
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && labels.is_cuda() && x.device() == w.device() && x.device() == labels.device(),
              "x, w and labels must be on one CUDA device");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "x and w must be bf16");
  TORCH_CHECK(labels.is_contiguous(), "labels must be contiguous");
  TORCH_CHECK(x.size(0) < (1ll << 31) - 256 && w.size(0) < (1ll << 31) - 256, "too many rows");
}

// A 2-D operand that the tensor maps can take (16-byte rows), copied otherwise.
at::Tensor tma_rows(const at::Tensor& t) {
  const bool ok = t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : at::empty(t.sizes(), t.options()).copy_(t);
}

// t.narrow(dim, at, n), without the view where that is all of t
at::Tensor share(const at::Tensor& t, int64_t dim, int64_t at, int64_t n) {
  return n == t.size(dim) ? t : t.narrow(dim, at, n);
}

CeArgs ce_args(const at::Tensor& labels, int64_t col0, int64_t vocab, int64_t ignore) {
  CeArgs ce{};
  ce.labels = labels.data_ptr<int64_t>();
  ce.col0 = col0;
  ce.vocab = vocab;
  ce.ignore = ignore;
  return ce;
}

// Columns of a piece of the vocabulary in the backward pass: as many as keep its bf16 gradient within 256 MiB, 256 at least (backward of
// 8192 x 129024 x 4096 with pieces of 2048 / 8192 / 16384 / 32768 / 65536 columns: 24.5 / 22.1 / 21.4 / 22.1 / 21.9 ms).
constexpr int64_t kPieceBytes = 256ll << 20;
constexpr int kBands = 16;  // gemm_tc: choose the kernel by size and walk the tiles in bands

}  // namespace

// {loss [T], max [T], sum exp(z - max) [T]} for a whole vocabulary; with `raw`, {label's logit (0 where another rank holds
// it), max, sum, sum with the label's logit exchanged} of the columns [col0, col0 + V) that this rank holds of `vocab`.
std::vector<at::Tensor> linear_ce_fwd(at::Tensor x, at::Tensor w, at::Tensor labels, int64_t col0, int64_t vocab,
                                      int64_t ignore, bool raw) {
  check_ce(x, w, labels);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), V = w.size(0);
  TORCH_CHECK(V > 0 && col0 >= 0 && col0 + V <= vocab && (raw || V == vocab), "columns outside the vocabulary");
  // each has memory of its own: a caller may change the loss in place while the statistics are kept
  std::vector<at::Tensor> out;
  for (int i = 0; i < (raw ? 4 : 3); ++i) out.push_back(new_empty({T}, x, at::kFloat));
  if (T == 0) return out;
  const int64_t tiles = (V + 255) / 256;
  auto part = new_empty({tiles * T * 2 + T}, x, at::kFloat);  // and the labels' logits
  CeArgs ce = ce_args(labels, col0, vocab, ignore);
  ce.part = reinterpret_cast<float2*>(part.data_ptr<float>());
  ce.target = part.data_ptr<float>() + tiles * T * 2;
  auto xr = tma_rows(x), wr = tma_rows(w);
  linear_ce_gemm(xr, wr, ce, false, at::Tensor());
  launch_early(
      ce_join_kernel, (int)((T + 31) / 32), 1024, 0, ce, reinterpret_cast<const __nv_bfloat16*>(xr.data_ptr()), xr.stride(0),
      reinterpret_cast<const __nv_bfloat16*>(wr.data_ptr()), wr.stride(0), (int)x.size(1), (int)T, (int)tiles, (int)V, raw,
      out[0].data_ptr<float>(), out[1].data_ptr<float>(), out[2].data_ptr<float>(), raw ? out[3].data_ptr<float>() : nullptr);
  EMB_LAUNCH_CHECK();
  count_launch();
  return out;
}

// {dx [T, H] bf16, dw [V, H] bf16}, each undefined where it is not wanted; with `dw_accum` (fp32 [V, H]) the weight
// gradient is added there.  `piece`: columns of a piece (0: as many as fit the workspace).
std::vector<at::Tensor> linear_ce_bwd(at::Tensor dloss, at::Tensor x, at::Tensor w, at::Tensor labels, at::Tensor top,
                                      at::Tensor sum, int64_t col0, int64_t vocab, int64_t ignore, bool want_dx,
                                      bool want_dw, c10::optional<at::Tensor> dw_accum, int64_t piece) {
  check_ce(x, w, labels);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), V = w.size(0), H = x.size(1);
  for (const auto& t : {top, sum})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == T && t.device() == x.device(),
                "the statistics of the forward pass must be fp32 [T]");
  auto g = dloss.to(at::kFloat).contiguous();
  TORCH_CHECK(g.numel() == T && g.device() == x.device(), "dloss must be [T]");
  at::Tensor dx, dw;
  if (dw_accum.has_value()) {
    TORCH_CHECK(dw_accum->scalar_type() == at::kFloat && dw_accum->dim() == 2 && dw_accum->size(0) == V &&
                    dw_accum->size(1) == H && dw_accum->stride(1) == 1 && dw_accum->device() == x.device(),
                "the weight gradient accumulator must be fp32 [V, H]");
  } else if (want_dw) {
    dw = new_empty({V, H}, x, at::kBFloat16);
  }
  if (want_dx) dx = new_empty({T, H}, x, at::kBFloat16);
  if (T == 0) {
    if (dw.defined()) dw.zero_();
    return {dx, dw};
  }
  auto xr = tma_rows(x), wr = tma_rows(w);
  const int64_t rows = T <= 128 ? 2 * T : T;  // of P
  const int64_t whole = (V + 255) / 256 * 256;
  if (piece <= 0) piece = kPieceBytes / (2 * rows);
  piece = std::min(whole, std::max<int64_t>(256, piece / 256 * 256));
  const int64_t pieces = (V + piece - 1) / piece;
  auto P = new_empty({rows, piece}, x, at::kBFloat16);
  const bool wants_w = want_dw || dw_accum.has_value();
  auto xs = rows > T && wants_w ? at::cat({xr, xr}) : xr;
  CeArgs ce = ce_args(labels, col0, vocab, ignore);
  ce.top = top.data_ptr<float>();
  ce.sum = sum.data_ptr<float>();
  ce.low_row = rows > T ? (int)T : 0;
  ce.dloss = g.data_ptr<float>();
  // dx of few rows and dw of few words have few output tiles and a long sum: it is split, fp32 parts joined in order
  // (dx of 512 x 129024 x 4096: 572 -> 436 us, dw of 8192 x 1000 x 512: 82 -> 26 us against whole sums on single SMs).
  // The parts of a product fill the SMs once (a 128 x 256 tile each) and are joined before the next product.
  const Split sx(rows, H), sw(std::min(piece, V), H);
  const bool split = want_dx && (rows > T || (sx.pair ? sx.tiles : sx.tiles * 2) <= sx.slots);
  const bool split_w = wants_w && pieces == 1 && sw.shares(xs.size(0)) > 1;
  at::Tensor total;  // dx over several pieces
  if (want_dx && pieces > 1) {
    total = new_empty({1, T, H}, x, at::kFloat);
    if (split) total.zero_();
  }
  for (int64_t i = 0; i < pieces; ++i) {
    const int64_t v0 = i * piece, n = std::min(piece, V - v0);
    const auto Pi = share(P, 1, 0, n), wi = share(wr, 0, v0, n);
    ce.col0 = col0 + v0;
    linear_ce_gemm(xr, wi, ce, true, Pi);
    if (want_dx) {
      if (split) {
        const auto px = new_empty({sx.shares(n), sx.pad, H}, x, at::kFloat);
        gemm_split_k(Pi, wi, false, px);
        sum_parts(px, px.size(0), rows > T, T, pieces > 1 ? total[0] : dx);
      } else {
        gemm_tc(Pi, wi, false, false, pieces > 1 ? total[0] : dx, i > 0, kBands);
      }
    }
    if (split_w) {
      const auto pw = new_empty({sw.shares(xs.size(0)), sw.pad, H}, x, at::kFloat);
      gemm_split_k(Pi, xs, true, pw);
      sum_parts(pw, pw.size(0), false, V, dw_accum.has_value() ? *dw_accum : dw);
    } else if (dw_accum.has_value()) {
      gemm_tc(Pi, xs, true, false, share(*dw_accum, 0, v0, n), true, kBands);
    } else if (want_dw) {
      gemm_tc(Pi, xs, true, false, share(dw, 0, v0, n), false, kBands);
    }
  }
  if (total.defined()) sum_parts(total, 1, false, T, dx);
  return {dx, dw};
}

}  // namespace emb
