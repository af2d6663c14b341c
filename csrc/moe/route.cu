// Router of the mixture of experts in its general form: softmax or sigmoid scores, a selection bias, expert groups,
// top-k and renormalised, scaled weights; with the load statistics and the gradient.  For a token's logits l [E]:
//
//   s_e = exp(l_e - max) / sum exp(l - max)   or   1 / (1 + exp(-l_e))                       fp32
//   c_e = s_e + bias_e; -inf where l_e = -inf (a masked expert comes after every other expert of the kept groups).
//         without a bias and with all groups kept the choice goes by l itself, which is the same order and keeps
//         apart logits whose scores round to the same value
//   groups: the E / G neighbours of a group; its value is the sum of its `gbest` largest c (of those not masked; a
//         group with none comes last); the experts of the `topg` best groups stay
//   e_1..e_k = the k largest c in falling order; equal ones (groups too) by the lower index
//   w_j = scaling s_{e_j} / D,  D = sum_j s_{e_j} + 1e-20 (renormalised) or 1
//   counts_e = tokens that chose e;  score_sum_e = sum over tokens of p_e, p = s (softmax) or s / (sum s + 1e-20)
//
// A row whose logits are all -inf has scores and weights 0 and takes the lowest experts.  A NaN logit counts as
// masked in the selection (so every index stays in range) and makes the row's softmax scores NaN.
//
// The scores use expf and IEEE division, and the softmax sum is held in 64 bits, so s, c and with them the choice
// are the same for every order of summation: ranks, batch splits and the host implementation agree on them.
//
// Gradient, with u_j = s_{e_j} / D, a_e = scaling dw_j at e = e_j (0 elsewhere), q_e = dscore_e:
//   ds_e = (a_e - [e chosen, renormalised] sum_j a_j u_j) / D
//   softmax: dl_e = s_e (ds_e + q_e - sum_f s_f (ds_f + q_f))
//   sigmoid: dl_e = s_e (1 - s_e) (ds_e + (q_e - sum_f q_f p_f) / (sum s + 1e-20))
//
// One warp per token, lane i holding experts [i EPL, (i + 1) EPL): the logits are read once, everything else stays in
// registers, and a round of the selection is one redux over order-preserving integer keys.  The statistics are
// kept per lane over the warp's tokens, joined over the warps of a CTA and then over the CTAs in a fixed order.
#include "../include/common.cuh"

#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

namespace emb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kTiny = 1e-20f;
constexpr int kRouteWarps = 8;
constexpr int kMaxExperts = 512, kMaxTopk = 32, kMaxGroups = 32;

struct RouteParams {
  const void* logits;
  long long ld;  // elements between rows
  const float* bias;
  int T, E, k, groups, topg, gbest;
  float scaling;
  int sigmoid, renorm;
  // forward
  float* weights;
  int* experts;
  float* part;  // [blocks, E] partial score sums, followed by
  int* cpart;   // [blocks, E] partial counts
  // backward
  const float* dweights;
  const float* dscore;
  const int* chosen;
  void* dlogits;
};

template <typename T>
__device__ __forceinline__ float load_f(const T* p) { return (float)*p; }

__device__ __forceinline__ float quot(float a, float b) { return __fdiv_rn(a, b); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Unsigned keys in the order of the floats (-0 = +0); 1: masked or NaN; 0 is left for experts out of the running.
__device__ __forceinline__ unsigned order_key(float c) {
  const unsigned u = __float_as_uint(c + 0.0f);
  const unsigned o = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
  return c > -INFINITY ? o : 1u;
}

// The lane's scores s[j] of its EPL experts.  Returns what the sigmoid divides its normalised scores by.
template <int EPL>
__device__ __forceinline__ float scores(const float* l, float* s, int sigmoid) {
  if (sigmoid) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      s[j] = quot(1.f, 1.f + expf(-l[j]));
      t += s[j];
    }
    return warp_sum(t) + kTiny;
  }
  float mx = l[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) mx = fmaxf(mx, l[j]);
  mx = warp_max(mx);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    s[j] = l[j] == -INFINITY ? 0.f : expf(l[j] - mx);
    sum += (double)s[j];
  }
  const float z = (float)warp_sum_d(sum);
  const float d = z == 0.f ? 1.f : z;  // an all-masked row
#pragma unroll
  for (int j = 0; j < EPL; ++j) s[j] = quot(s[j], d);
  return 1.f;
}

template <typename T, int EPL>
__device__ __forceinline__ void load_row(const RouteParams& p, int t, int lane, float* l) {
  const T* row = reinterpret_cast<const T*>(p.logits) + (long long)t * p.ld;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    l[j] = e < p.E ? load_f(row + e) : -INFINITY;
  }
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32) route_fwd_kernel(RouteParams p) {
  extern __shared__ float s_mem[];  // [warps, E] score sums; [E] counts; [warps, E] choice values (groups)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* s_cnt = reinterpret_cast<int*>(s_mem + kRouteWarps * p.E);
  float* s_c = reinterpret_cast<float*>(s_cnt + p.E) + warp * p.E;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) s_cnt[e] = 0;
  __syncthreads();
  float bias[EPL], acc[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    bias[j] = p.bias && e < p.E ? p.bias[e] : 0.f;
    acc[j] = 0.f;
  }
  const bool by_group = p.groups > p.topg, by_logit = !p.bias && !by_group;
  for (int t = blockIdx.x * kRouteWarps + warp; t < p.T; t += gridDim.x * kRouteWarps) {
    float l[EPL], s[EPL];
    unsigned key[EPL];
    load_row<T, EPL>(p, t, lane, l);
    const float norm = scores<EPL>(l, s, p.sigmoid);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane * EPL + j;
      if (e < p.E) acc[j] += p.sigmoid ? quot(s[j], norm) : s[j];
      const float c = by_logit ? l[j] : l[j] > -INFINITY ? s[j] + bias[j] : -INFINITY;
      key[j] = e < p.E ? order_key(c) : 0u;
      if (by_group && e < p.E) s_c[e] = c;
    }
    if (by_group) {
      __syncwarp();
      // lane g values group g: its gbest largest, one after the other in falling order
      unsigned gkey = 0u;
      const int per = p.E / p.groups;
      if (lane < p.groups) {
        const float* c = s_c + lane * per;
        float sum = 0.f, last = INFINITY;
        int seen = 0, used = 0;  // values equal to `last` already taken
        for (int m = 0; m < p.gbest; ++m) {
          float best = -INFINITY;
          int ties = 0;
          for (int i = 0; i < per; ++i) {
            const float v = c[i];
            if (v == last) ++ties;
            if (v < last && v > best) best = v;
          }
          if (used < ties) best = last;  // another copy of the value taken before
          used = best == last ? used + 1 : 1;
          last = best;
          if (!(best > -INFINITY)) break;
          sum = seen ? sum + best : best;
          ++seen;
        }
        gkey = seen ? order_key(sum) : 1u;
      }
      unsigned kept = 0u;
      for (int m = 0; m < p.topg; ++m) {
        const unsigned top = __reduce_max_sync(kFull, gkey);
        const int g = __ffs(__ballot_sync(kFull, gkey == top)) - 1;
        kept |= 1u << g;
        if (lane == g) gkey = 0u;
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        if (e < p.E && !((kept >> (e / per)) & 1u)) key[j] = 0u;
      }
      __syncwarp();
    }
    float w = 0.f;
    int mine = 0;
    for (int r = 0; r < p.k; ++r) {
      unsigned best = key[0];
#pragma unroll
      for (int j = 1; j < EPL; ++j) best = max(best, key[j]);
      const unsigned top = __reduce_max_sync(kFull, best);
      const int src = __ffs(__ballot_sync(kFull, best == top)) - 1;
      float sv = 0.f;
      int at = 0;
      if (lane == src) {
        bool open = true;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          if (open && key[j] == top) {
            sv = s[j];
            at = j;
            key[j] = 0u;
            open = false;
          }
        }
      }
      sv = __shfl_sync(kFull, sv, src);
      at = src * EPL + __shfl_sync(kFull, at, src);
      if (lane == r) {
        w = sv;
        mine = at;
      }
    }
    if (p.renorm) w = quot(w, warp_sum(w) + kTiny);
    if (lane < p.k) {
      p.weights[(long long)t * p.k + lane] = w * p.scaling;
      p.experts[(long long)t * p.k + lane] = mine;
      atomicAdd(&s_cnt[mine], 1);  // whole numbers: any order gives the same counts
    }
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    if (e < p.E) s_mem[warp * p.E + e] = acc[j];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kRouteWarps; ++q) v += s_mem[q * p.E + e];
    p.part[(long long)blockIdx.x * p.E + e] = v;
    p.cpart[(long long)blockIdx.x * p.E + e] = s_cnt[e];
  }
}

// score_sum and counts from the CTAs' partials: 32 experts a CTA, 32 slices of the partials, joined by a fixed tree.
__global__ void __launch_bounds__(1024) route_join_kernel(const float* __restrict__ part, const int* __restrict__ cpart,
                                                          int blocks, int E, float* __restrict__ score_sum,
                                                          int* __restrict__ counts) {
  __shared__ float sh[32][33];
  __shared__ int shc[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  int c = 0;
  if (e < E) {
    for (int b = slice; b < blocks; b += 32) {
      v += part[(long long)b * E + e];
      c += cpart[(long long)b * E + e];
    }
  }
  sh[slice][lane] = v;
  shc[slice][lane] = c;
  __syncthreads();
  v = warp_sum(sh[lane][slice]);
  c = __reduce_add_sync(kFull, shc[lane][slice]);
  const int o = blockIdx.x * 32 + slice;
  if (lane == 0 && o < E) {
    score_sum[o] = v;
    counts[o] = c;
  }
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32) route_bwd_kernel(RouteParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float q[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    q[j] = p.dscore && e < p.E ? p.dscore[e] : 0.f;
  }
  for (int t = blockIdx.x * kRouteWarps + warp; t < p.T; t += gridDim.x * kRouteWarps) {
    float l[EPL], s[EPL], ds[EPL];
    load_row<T, EPL>(p, t, lane, l);
    float a = 0.f;
    int e_r = -1;
    if (lane < p.k) {
      a = p.dweights ? p.dweights[(long long)t * p.k + lane] * p.scaling : 0.f;
      e_r = p.chosen[(long long)t * p.k + lane];
    }
    const float norm = scores<EPL>(l, s, p.sigmoid);
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] = 0.f;
    float den = 1.f, dot = 0.f;
    if (p.renorm) {
      float sel = 0.f, prod = 0.f;  // sums over this lane's chosen experts
      for (int r = 0; r < p.k; ++r) {
        const int at = __shfl_sync(kFull, e_r, r) - lane * EPL;
        const float ar = __shfl_sync(kFull, a, r);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          if (at == j) {
            sel += s[j];
            prod += ar * s[j];
          }
        }
      }
      den = warp_sum(sel) + kTiny;
      dot = quot(warp_sum(prod), den);
    }
    for (int r = 0; r < p.k; ++r) {
      const int at = __shfl_sync(kFull, e_r, r) - lane * EPL;
      const float ar = __shfl_sync(kFull, a, r);
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (at == j) ds[j] = quot(ar - dot, den);
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (p.sigmoid) {
        sum += q[j] * s[j];
      } else {
        ds[j] += q[j];
        sum += s[j] * ds[j];
      }
    }
    sum = warp_sum(sum);
    if (p.sigmoid) sum = quot(sum, norm);
    T* out = reinterpret_cast<T*>(p.dlogits) + (long long)t * p.E;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane * EPL + j;
      float d;
      if (p.sigmoid) {
        const float x = expf(-fabsf(l[j]));  // s (1 - s) = x / (1 + x)^2, without the difference
        d = quot(x, (1.f + x) * (1.f + x)) * (ds[j] + quot(q[j] - sum, norm));
      } else {
        d = s[j] * (ds[j] - sum);
      }
      if (e < p.E) out[e] = (T)d;
    }
  }
}

void check_route(const at::Tensor& logits, int64_t k, int64_t groups, int64_t topg, const c10::optional<at::Tensor>& bias) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be a CUDA tensor [tokens, experts]");
  const int64_t E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= kMaxExperts, "1 to ", kMaxExperts, " experts are supported");
  TORCH_CHECK(k >= 1 && k <= E && k <= kMaxTopk, "k must be in 1..min(experts, ", kMaxTopk, ")");
  TORCH_CHECK(groups >= 1 && groups <= kMaxGroups && E % groups == 0, "experts must divide into at most ", kMaxGroups,
              " groups");
  TORCH_CHECK(topg >= 1 && topg <= groups && topg * (E / groups) >= k, "the kept groups must hold k experts");
  TORCH_CHECK(logits.size(0) < (1ll << 31) - (1 << 20), "too many tokens in one call");
  if (bias.has_value())
    TORCH_CHECK(bias->is_cuda() && bias->device() == logits.device() && bias->scalar_type() == at::kFloat &&
                    bias->dim() == 1 && bias->size(0) == E && bias->is_contiguous(),
                "bias must be a contiguous fp32 [experts] tensor on the device of logits");
}

RouteParams route_params(const at::Tensor& logits, int64_t k, bool sigmoid, int64_t groups, int64_t topg, bool renorm,
                         double scaling) {
  RouteParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.T = (int)logits.size(0);
  p.E = (int)logits.size(1);
  p.k = (int)k;
  p.groups = (int)groups;
  p.topg = (int)topg;
  p.gbest = (int)std::min<int64_t>(std::max<int64_t>(1, k / topg), p.E / groups);
  p.scaling = (float)scaling;
  p.sigmoid = sigmoid;
  p.renorm = renorm;
  return p;
}

template <typename F>
void by_shape(at::ScalarType t, int E, F f) {
  auto per = [&](auto v) {
    const int epl = (E + 31) / 32;
    if (epl <= 1) f(v, std::integral_constant<int, 1>{});
    else if (epl <= 2) f(v, std::integral_constant<int, 2>{});
    else if (epl <= 4) f(v, std::integral_constant<int, 4>{});
    else if (epl <= 8) f(v, std::integral_constant<int, 8>{});
    else f(v, std::integral_constant<int, 16>{});
  };
  if (t == at::kFloat) per(float{});
  else if (t == at::kBFloat16) per(__nv_bfloat16{});
  else if (t == at::kHalf) per(__half{});
  else TORCH_CHECK(false, "logits must be fp32, bf16 or fp16");
}

at::Tensor row_contiguous(const at::Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous(); }

}  // namespace

// {weights [T, k] fp32, experts [T, k] int32, score_sum [E] fp32, counts [E] int32}
std::vector<at::Tensor> moe_route_fwd(at::Tensor logits, int64_t k, bool sigmoid, c10::optional<at::Tensor> bias,
                                      int64_t groups, int64_t topg, bool renorm, double scaling) {
  check_route(logits, k, groups, topg, bias);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto x = row_contiguous(logits);
  RouteParams p = route_params(x, k, sigmoid, groups, topg, renorm, scaling);
  auto f32 = x.options().dtype(at::kFloat), i32 = x.options().dtype(at::kInt);
  auto weights = at::empty({p.T, k}, f32), experts = at::empty({p.T, k}, i32);
  if (p.T == 0) return {weights, experts, at::zeros({p.E}, f32), at::zeros({p.E}, i32)};
  auto score_sum = at::empty({p.E}, f32), counts = at::empty({p.E}, i32);
  const int grid = std::min((p.T + kRouteWarps - 1) / kRouteWarps, num_sms() * 4);
  auto part = at::empty({2, grid, p.E}, f32);
  p.bias = bias.has_value() ? bias->data_ptr<float>() : nullptr;
  p.weights = weights.data_ptr<float>();
  p.experts = experts.data_ptr<int>();
  p.part = part.data_ptr<float>();
  p.cpart = reinterpret_cast<int*>(p.part + (long long)grid * p.E);
  const int smem = (kRouteWarps * p.E * (groups > topg ? 2 : 1) + p.E) * 4;
  by_shape(x.scalar_type(), p.E, [&](auto v, auto epl) {
    route_fwd_kernel<decltype(v), epl><<<grid, kRouteWarps * 32, smem, cur_stream()>>>(p);
  });
  route_join_kernel<<<(p.E + 31) / 32, 1024, 0, cur_stream()>>>(p.part, p.cpart, grid, p.E, score_sum.data_ptr<float>(),
                                                                counts.data_ptr<int>());
  EMB_LAUNCH_CHECK();
  count_launch(2);
  return {weights, experts, score_sum, counts};
}

at::Tensor moe_route_bwd(at::Tensor logits, at::Tensor experts, c10::optional<at::Tensor> dweights,
                         c10::optional<at::Tensor> dscore, bool sigmoid, bool renorm, double scaling) {
  const int64_t k = experts.size(1);
  check_route(logits, k, 1, 1, c10::nullopt);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto x = row_contiguous(logits);
  RouteParams p = route_params(x, k, sigmoid, 1, 1, renorm, scaling);
  auto dl = at::empty({p.T, p.E}, x.options());
  if (p.T == 0) return dl;
  TORCH_CHECK(experts.scalar_type() == at::kInt && experts.is_contiguous() && experts.size(0) == p.T,
              "experts must be the int32 tensor of the forward pass");
  at::Tensor dw, dq;
  if (dweights.has_value()) {
    TORCH_CHECK(dweights->sizes() == experts.sizes(), "dweights must be [tokens, k]");
    dw = dweights->to(at::kFloat).contiguous();
    p.dweights = dw.data_ptr<float>();
  }
  if (dscore.has_value()) {
    TORCH_CHECK(dscore->numel() == p.E, "dscore must be [experts]");
    dq = dscore->to(at::kFloat).contiguous();
    p.dscore = dq.data_ptr<float>();
  }
  p.chosen = experts.data_ptr<int>();
  p.dlogits = dl.data_ptr();
  const int grid = std::min((p.T + kRouteWarps - 1) / kRouteWarps, num_sms() * 8);
  by_shape(x.scalar_type(), p.E, [&](auto v, auto epl) {
    route_bwd_kernel<decltype(v), epl><<<grid, kRouteWarps * 32, 0, cur_stream()>>>(p);
  });
  EMB_LAUNCH_CHECK();
  count_launch();
  return dl;
}

}  // namespace emb
