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
// are the same for every order of summation: ranks and batch splits agree on them bit for bit.  The host form takes the
// same steps with the host's exp and adds three or more values of a group in an order of its own, so it can choose
// otherwise between values that are apart by a few units in the last place.
//
// Gradient, with u_j = s_{e_j} / D, a_e = scaling dw_j at e = e_j (0 elsewhere), q_e = dscore_e:
//   ds_e = (a_e - [e chosen, renormalised] sum_j a_j u_j) / D
//   softmax: dl_e = s_e (ds_e + q_e - sum_f s_f (ds_f + q_f))
//   sigmoid: dl_e = s_e (1 - s_e) (ds_e + (q_e - sum_f q_f p_f) / (sum s + 1e-20))
//
// One warp per token, lane i holding experts [i EPL, (i + 1) EPL): the logits are read once and the scores stay in
// registers.  The kernels have few bytes and many instructions for a token, so these are what is kept low: each lane
// sorts its keys (integers in the order of the choice) once, a round of the selection is then one redux over the lanes'
// first keys, and the chosen indices and scores are looked up afterwards by k lanes at once through shared memory.  The
// statistics are kept per lane over the warp's tokens and joined over the warps and the CTAs in a fixed order.
// 32768 tokens, 256 experts, k = 8, 4 of 8 groups, fp32: forward 42 us with the join (1049 instructions a token at 0.69 of
// the issue slots; its bytes alone: 5 us), backward 21 us (441; 10 us).
#include "../include/common.cuh"

#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

namespace emb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kTiny = 1e-20f;
constexpr int kRouteWarps = 16;
constexpr int kMaxExperts = 512, kMaxTopk = 32, kMaxGroups = 32;
// The most shared memory that a forward asks for: 16 experts a lane (keys and scores of 512), counts, and the rows of 32
// groups of up to 16 experts at a stride of 33 words.
constexpr int kRouteSmem = (2 * kRouteWarps * 32 * 16 + kMaxExperts + kRouteWarps * kMaxGroups * 33) * 4;

struct RouteParams {
  const void* logits;
  long long ld;  // elements between rows
  const float* bias;
  int T, E, k, groups, topg, gbest;
  int gwidth;   // lanes that hold a group, if groups are whole lanes of a power of two and gbest <= 2; else 0, and
  int glanes;   // lanes that value a group from shared memory
  int gstride;  // words between groups in shared memory: the lanes of all groups hit different banks
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

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// The lane's EPL logits of a row, -inf past the last expert.  VEC: experts fill whole lanes and rows are aligned, so a
// lane reads and writes its share in one piece.
template <typename T, int EPL, bool VEC>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, float* l) {
  if constexpr (VEC) {
    if (lane * EPL < E) {
      const Pack<T, EPL> v = reinterpret_cast<const Pack<T, EPL>*>(row)[lane];
#pragma unroll
      for (int j = 0; j < EPL; ++j) l[j] = (float)v.v[j];
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) l[j] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane * EPL + j;
      l[j] = e < E ? (float)row[e] : -INFINITY;
    }
  }
}

// Maximum of the row and the 64-bit sum of its exponentials, rounded to fp32 (1 for an all-masked row); s = exponentials.
template <int EPL>
__device__ __forceinline__ void softmax_parts(const float* l, float* s, float& mx, float& z) {
  mx = l[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) mx = fmaxf(mx, l[j]);
  mx = warp_max(mx);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    s[j] = l[j] == -INFINITY ? 0.f : expf(l[j] - mx);
    sum += (double)s[j];
  }
  z = (float)warp_sum_d(sum);
  if (z == 0.f) z = 1.f;
}

// Falling order by a merge-exchange network (compile-time indices, so the keys stay in registers).
template <int N>
__device__ __forceinline__ void sort_keys(unsigned* k) {
#pragma unroll
  for (int p = 1; p < N; p *= 2) {
#pragma unroll
    for (int q = p; q >= 1; q /= 2) {
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q) {
#pragma unroll
        for (int i = 0; i < q; ++i) {
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const unsigned a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
        }
      }
    }
  }
}

template <typename T, int EPL, bool VEC>
__global__ void __launch_bounds__(kRouteWarps * 32, EPL <= 8 ? 2 : 1) route_fwd_kernel(RouteParams p) {
  // [warps, 32 EPL] keys, [warps, 32 EPL] scores (after the last token: score sums), [E] counts, [warps, groups, gstride]
  extern __shared__ __align__(16) unsigned s_mem[];
  constexpr int ROW = 32 * EPL;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned* s_key = s_mem + warp * ROW;
  float* s_val = reinterpret_cast<float*>(s_mem + kRouteWarps * ROW) + warp * ROW;
  int* s_cnt = reinterpret_cast<int*>(s_mem + 2 * kRouteWarps * ROW);
  float* s_grp = reinterpret_cast<float*>(s_cnt + p.E) + warp * p.groups * p.gstride;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) s_cnt[e] = 0;
  grid_dependency();
  __syncthreads();
  const bool by_group = p.groups > p.topg, by_logit = !p.bias && !by_group;
  const int per = p.E / p.groups;
  float bias[EPL], acc[EPL], next[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    bias[j] = p.bias && e < p.E ? p.bias[e] : 0.f;
    acc[j] = 0.f;
  }
  const T* logits = reinterpret_cast<const T*>(p.logits);
  const int step = gridDim.x * kRouteWarps;
  int t = blockIdx.x * kRouteWarps + warp;
  if (t < p.T) load_row<T, EPL, VEC>(logits + (long long)t * p.ld, p.E, lane, next);
  for (; t < p.T; t += step) {
    float s[EPL];
    unsigned key[EPL];
    float b1 = -INFINITY, b2 = -INFINITY;  // the lane's two largest choice values (groups of whole lanes)
    {
      float l[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) l[j] = next[j];
      if (t < p.T - step) load_row<T, EPL, VEC>(logits + (long long)(t + step) * p.ld, p.E, lane, next);
      if (p.sigmoid) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          s[j] = __frcp_rn(1.f + expf(-l[j]));
          sum += s[j];
        }
        const float inv = __fdividef(1.f, warp_sum(sum) + kTiny);
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] += s[j] * inv;
      } else {
        float mx, z;
        softmax_parts<EPL>(l, s, mx, z);
        const float inv = quot(1.f, z);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          s[j] = by_logit ? s[j] * inv : quot(s[j], z);
          acc[j] += s[j];
        }
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        const float c = by_logit ? l[j] : l[j] > -INFINITY ? s[j] + bias[j] : -INFINITY;
        key[j] = e < p.E ? order_key(c) : 0u;
        if (by_group) {
          if (p.gwidth) {
            b2 = fmaxf(b2, fminf(b1, c == c ? c : -INFINITY));  // (NaN is passed over)
            b1 = fmaxf(b1, c);
          } else if (e < p.E) {
            s_grp[e / per * p.gstride + e % per] = c;
          }
        }
      }
    }
    if (by_group && p.gwidth) {
      // the experts of a group are those of gwidth neighbouring lanes
      for (int o = 1; o < p.gwidth; o <<= 1) {
        const float o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
        b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
        b1 = fmaxf(b1, o1);
      }
      unsigned gkey = lane * EPL < p.E && lane % p.gwidth == 0
                          ? order_key(p.gbest == 2 && b2 > -INFINITY ? b1 + b2 : b1) : 0u;
      unsigned kept = 0u;  // first lanes of the groups
      for (int m = 0; m < p.topg; ++m) {
        const unsigned top = __reduce_max_sync(kFull, gkey);
        const unsigned at = __ballot_sync(kFull, gkey == top);
        kept |= at & -at;
        if (kept >> lane & 1u) gkey = 0u;
      }
      if (!((kept >> (lane & ~(p.gwidth - 1))) & 1u)) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = 0u;
      }
    } else if (by_group) {
      __syncwarp();
      // p.glanes lanes value a group, each from every glanes-th of its experts
      const int g = lane / p.glanes, part = lane % p.glanes;
      unsigned gkey = 0u;
      float sum = 0.f;
      bool any = false;
      const float* c = s_grp + (g < p.groups ? g : 0) * p.gstride;
      if (p.gbest <= 2) {
        for (int i = part; i < per; i += p.glanes) {
          const float v = c[i];
          b2 = fmaxf(b2, fminf(b1, v == v ? v : -INFINITY));
          b1 = fmaxf(b1, v);
        }
        for (int o = 1; o < p.glanes; o <<= 1) {
          const float o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
          b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
          b1 = fmaxf(b1, o1);
        }
        any = b1 > -INFINITY;
        sum = p.gbest == 2 && b2 > -INFINITY ? b1 + b2 : b1;
      } else {
        // one after the other in falling order; equal values are told apart by their place
        float last = INFINITY;
        int last_i = -1;
        for (int m = 0; m < p.gbest; ++m) {
          float best = -INFINITY;
          int best_i = 0x7fffffff;
          for (int i = part; i < per; i += p.glanes) {
            const float v = c[i];
            const bool open = v < last || (v == last && i > last_i);
            if (open && v > best) {
              best = v;
              best_i = i;
            }
          }
          for (int o = 1; o < p.glanes; o <<= 1) {
            const float ov = __shfl_xor_sync(kFull, best, o);
            const int oi = __shfl_xor_sync(kFull, best_i, o);
            if (ov > best || (ov == best && oi < best_i)) {
              best = ov;
              best_i = oi;
            }
          }
          if (best > -INFINITY) {
            sum = any ? sum + best : best;
            any = true;
          }
          last = best;
          last_i = best_i;
        }
      }
      if (g < p.groups && part == 0) gkey = any ? order_key(sum) : 1u;
      unsigned kept = 0u;
      for (int m = 0; m < p.topg; ++m) {
        const unsigned top = __reduce_max_sync(kFull, gkey);
        const int at = __ffs(__ballot_sync(kFull, gkey == top)) - 1;
        kept |= 1u << (at / p.glanes);
        if (lane == at) gkey = 0u;
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        if (e < p.E && !((kept >> (e / per)) & 1u)) key[j] = 0u;
      }
    }
    // keys and scores for the look-up of the chosen, then the lane's keys in falling order: a round takes the largest
    // of the lanes' first keys, and the lane that holds it moves up
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      s_key[lane * EPL + j] = key[j];
      s_val[lane * EPL + j] = s[j];
    }
    sort_keys<EPL>(key);
    unsigned my_key = 0u, last = 0u;
    int my_src = 0, skip = 0, from = -1, copies = 0;
    for (int r = 0; r < p.k; ++r) {
      const unsigned top = __reduce_max_sync(kFull, key[0]);
      const int src = __ffs(__ballot_sync(kFull, key[0] == top)) - 1;
      copies = top == last && src == from ? copies + 1 : 0;  // equal keys of a lane come one after the other
      last = top;
      from = src;
      if (lane == r) {
        my_key = top;
        my_src = src;
        skip = copies;
      }
      if (lane == src) {
#pragma unroll
        for (int j = 0; j + 1 < EPL; ++j) key[j] = key[j + 1];
        key[EPL - 1] = 0u;
      }
    }
    __syncwarp();
    // lane r finds its expert: in lane my_src's share, the copy of my_key after those that earlier rounds took
    int mine = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (s_key[my_src * EPL + j] == my_key) {
        if (skip == 0) mine = my_src * EPL + j;
        --skip;
      }
    }
    float w = lane < p.k ? s_val[mine] : 0.f;
    if (p.renorm) w = quot(w, warp_sum(w) + kTiny);
    if (lane < p.k) {
      p.weights[(long long)t * p.k + lane] = w * p.scaling;
      p.experts[(long long)t * p.k + lane] = mine;
      atomicAdd(&s_cnt[mine], 1);  // whole numbers: any order gives the same counts
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) s_val[lane * EPL + j] = acc[j];
  __syncthreads();
  const float* sums = reinterpret_cast<const float*>(s_mem + kRouteWarps * ROW);
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kRouteWarps; ++q) v += sums[q * ROW + e];
    p.part[(long long)blockIdx.x * p.E + e] = v;
    p.cpart[(long long)blockIdx.x * p.E + e] = s_cnt[e];
  }
}

// score_sum and counts from the CTAs' partials: 8 experts a CTA and 128 slices of the partials, so that a thread has two
// or three loads to wait for at once; slices are joined by a fixed tree.
__global__ void __launch_bounds__(1024) route_join_kernel(const float* __restrict__ part, const int* __restrict__ cpart,
                                                          int blocks, int E, float* __restrict__ score_sum,
                                                          int* __restrict__ counts) {
  __shared__ float sh[32][9];
  __shared__ int shc[32][9];
  grid_dependency();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 8 + (lane & 7);
  float v = 0.f;
  int c = 0;
  if (e < E) {
#pragma unroll 4
    for (int b = threadIdx.x >> 3; b < blocks; b += 128) {
      v += part[(long long)b * E + e];
      c += cpart[(long long)b * E + e];
    }
  }
  v += __shfl_xor_sync(kFull, v, 8);
  c += __shfl_xor_sync(kFull, c, 8);
  v += __shfl_xor_sync(kFull, v, 16);
  c += __shfl_xor_sync(kFull, c, 16);
  if (lane < 8) {
    sh[warp][lane] = v;
    shc[warp][lane] = c;
  }
  __syncthreads();
  if (warp >= 8) return;
  v = warp_sum(sh[lane][warp]);
  c = __reduce_add_sync(kFull, shc[lane][warp]);
  const int o = blockIdx.x * 8 + warp;
  if (lane == 0 && o < E) {
    score_sum[o] = v;
    counts[o] = c;
  }
}

template <typename T, int EPL, bool VEC>
__global__ void __launch_bounds__(kRouteWarps * 32) route_bwd_kernel(RouteParams p) {
  __shared__ __align__(16) float s_ds[kRouteWarps][32 * EPL];  // ds of the chosen experts, 0 elsewhere
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* row = s_ds[warp];
  grid_dependency();
  float q[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    q[j] = p.dscore && e < p.E ? p.dscore[e] : 0.f;
    row[e] = 0.f;
  }
  __syncwarp();
  // lane r has the r-th chosen expert: its gradient and its score.  The next token's inputs are fetched ahead.
  float next[EPL], next_a = 0.f;
  int next_e = 0;
  auto fetch = [&](int t) {
    load_row<T, EPL, VEC>(reinterpret_cast<const T*>(p.logits) + (long long)t * p.ld, p.E, lane, next);
    if (lane < p.k) {
      next_e = p.chosen[(long long)t * p.k + lane];
      if (p.dweights) next_a = p.dweights[(long long)t * p.k + lane];
    }
  };
  const int step = gridDim.x * kRouteWarps;
  int t = blockIdx.x * kRouteWarps + warp;
  if (t < p.T) fetch(t);
  for (; t < p.T; t += step) {
    float l[EPL], s[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) l[j] = next[j];
    const float a = next_a * p.scaling;
    const int er = next_e;
    const float lr = lane < p.k ? (float)(reinterpret_cast<const T*>(p.logits) + (long long)t * p.ld)[er] : -INFINITY;
    if (t < p.T - step) fetch(t + step);
    float sr = 0.f;
    float norm = 1.f, dsum = 0.f;  // dsum: s (1 - s) for the sigmoid is kept in l
    if (p.sigmoid) {
      float total = 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const float x = expf(-fabsf(l[j])), y = __fdividef(1.f, 1.f + x);
        s[j] = l[j] >= 0.f ? y : x * y;
        l[j] = x * y * y;  // s (1 - s), without the difference
        total += s[j];
        dsum += q[j] * s[j];
      }
      norm = quot(1.f, warp_sum(total) + kTiny);
      dsum = warp_sum(dsum) * norm;
      sr = __frcp_rn(1.f + expf(-lr));
    } else {
      float mx, z;
      softmax_parts<EPL>(l, s, mx, z);
      const float inv = quot(1.f, z);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        s[j] *= inv;
        dsum += q[j] * s[j];
      }
      sr = lr == -INFINITY ? 0.f : expf(lr - mx) * inv;
    }
    float ds = a;
    if (p.renorm) {
      const float den = quot(1.f, warp_sum(lane < p.k ? sr : 0.f) + kTiny);
      ds = (a - warp_sum(a * sr) * den) * den;
    }
    if (lane < p.k) {
      row[er] = ds;
      if (!p.sigmoid) dsum += sr * ds;
    }
    if (!p.sigmoid) dsum = warp_sum(dsum);
    __syncwarp();
    Pack<T, EPL> out;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float d = row[lane * EPL + j];
      out.v[j] = (T)(p.sigmoid ? l[j] * (d + (q[j] - dsum) * norm) : s[j] * (d + q[j] - dsum));
    }
    __syncwarp();
    if (lane < p.k) row[er] = 0.f;
    T* dst = reinterpret_cast<T*>(p.dlogits) + (long long)t * p.E;
    if constexpr (VEC) {
      if (lane * EPL < p.E) reinterpret_cast<Pack<T, EPL>*>(dst)[lane] = out;
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (lane * EPL + j < p.E) dst[lane * EPL + j] = out.v[j];
    }
    __syncwarp();
  }
}

void check_route(const at::Tensor& logits, int64_t k, int64_t groups, int64_t topg, const c10::optional<at::Tensor>& bias) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [tokens, experts]");
  const int64_t E = logits.size(1);
  TORCH_CHECK_VALUE(E >= 1 && E <= kMaxExperts, "1 to ", kMaxExperts, " experts are supported");
  TORCH_CHECK_VALUE(k >= 1 && k <= E && k <= kMaxTopk, "k must be in 1..min(experts, ", kMaxTopk, ")");
  TORCH_CHECK_VALUE(groups >= 1 && groups <= kMaxGroups && E % groups == 0, "experts must divide into at most ", kMaxGroups,
                    " groups");
  TORCH_CHECK_VALUE(topg >= 1 && topg <= groups && topg * (E / groups) >= k, "the kept groups must hold k experts");
  TORCH_CHECK(logits.size(0) < (1ll << 31) - (1 << 20), "too many tokens in one call");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == E, "bias must be fp32 [experts]");
    TORCH_CHECK(bias->is_cuda() && bias->device() == logits.device() && bias->is_contiguous(),
                "bias must be contiguous and on the device of logits");
  }
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
  p.glanes = 1;
  while (p.glanes * 2 * p.groups <= 32) p.glanes *= 2;
  const int per = p.E / p.groups;
  p.gstride = per + ((p.glanes - per) % 32 + 32) % 32;
  p.scaling = (float)scaling;
  p.sigmoid = sigmoid;
  p.renorm = renorm;
  return p;
}

// Experts of a lane: the smallest power of two that gives 32 lanes all experts.
int lane_share(int E) {
  int n = 1;
  while (32 * n < E) n *= 2;
  return n;
}

// Calls f(type, experts per lane, whole aligned shares) for the shape.
template <typename F>
void by_shape(const at::Tensor& x, F f) {
  const int E = (int)x.size(1);
  auto per = [&](auto v, auto epl) {
    constexpr int N = decltype(epl)::value;
    const int bytes = std::min<int>(16, N * (int)sizeof(v));
    const bool vec = N > 1 && E % N == 0 && (x.stride(0) * sizeof(v)) % bytes == 0 && (uintptr_t)x.data_ptr() % bytes == 0 &&
                     ((int64_t)E * sizeof(v)) % bytes == 0;
    if (vec) f(v, epl, std::true_type{});
    else f(v, epl, std::false_type{});
  };
  auto share = [&](auto v) {
    switch (lane_share(E)) {
      case 1: return per(v, std::integral_constant<int, 1>{});
      case 2: return per(v, std::integral_constant<int, 2>{});
      case 4: return per(v, std::integral_constant<int, 4>{});
      case 8: return per(v, std::integral_constant<int, 8>{});
      default: return per(v, std::integral_constant<int, 16>{});
    }
  };
  const auto t = x.scalar_type();
  if (t == at::kFloat) share(float{});
  else if (t == at::kBFloat16) share(__nv_bfloat16{});
  else if (t == at::kHalf) share(__half{});
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
  auto weights = new_empty({p.T, k}, x, at::kFloat), experts = new_empty({p.T, k}, x, at::kInt);
  if (p.T == 0)
    return {weights, experts, at::zeros({p.E}, weights.options()), at::zeros({p.E}, experts.options())};
  auto score_sum = new_empty({p.E}, x, at::kFloat), counts = new_empty({p.E}, x, at::kInt);
  const int epl = lane_share(p.E), width = p.E / p.groups / epl;
  p.gwidth = p.gbest <= 2 && (p.E / p.groups) % epl == 0 && (width & (width - 1)) == 0 ? width : 0;
  // (twice the resident CTAs would give a second, partial wave)
  const int grid = std::min((p.T + kRouteWarps - 1) / kRouteWarps, num_sms() * (epl <= 8 ? 2 : 1));
  p.bias = bias.has_value() ? bias->data_ptr<float>() : nullptr;
  p.weights = weights.data_ptr<float>();
  p.experts = experts.data_ptr<int>();
  at::Tensor part;
  if (grid == 1) {  // one CTA sees every token: its sums are the result
    p.part = score_sum.data_ptr<float>();
    p.cpart = counts.data_ptr<int>();
  } else {
    part = new_empty({2, grid, p.E}, x, at::kFloat);
    p.part = part.data_ptr<float>();
    p.cpart = reinterpret_cast<int*>(p.part + (long long)grid * p.E);
  }
  by_shape(x, [&](auto v, auto epl, auto vec) {
    constexpr int N = decltype(epl)::value;
    const int smem = (2 * kRouteWarps * 32 * N + p.E +
                      (groups > topg && !p.gwidth ? kRouteWarps * p.groups * p.gstride : 0)) * 4;
    auto kern = route_fwd_kernel<decltype(v), N, decltype(vec)::value>;
    if (smem > 48 * 1024) {
      static bool done[kMaxDevices] = {};  // the limit belongs to the device's context
      int dev = 0;
      EMB_CUDA_CHECK(cudaGetDevice(&dev));
      if (!done[dev]) EMB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRouteSmem));
      done[dev] = true;
    }
    launch_early(kern, grid, kRouteWarps * 32, smem, p);
  });
  EMB_LAUNCH_CHECK();
  if (grid > 1)
    launch_early(route_join_kernel, (p.E + 7) / 8, 1024, 0, p.part, p.cpart, grid, p.E, score_sum.data_ptr<float>(),
                 counts.data_ptr<int>());
  EMB_LAUNCH_CHECK();
  count_launch(grid > 1 ? 2 : 1);
  return {weights, experts, score_sum, counts};
}

at::Tensor moe_route_bwd(at::Tensor logits, at::Tensor experts, c10::optional<at::Tensor> dweights,
                         c10::optional<at::Tensor> dscore, bool sigmoid, bool renorm, double scaling) {
  const int64_t k = experts.size(1);
  check_route(logits, k, 1, 1, c10::nullopt);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto x = row_contiguous(logits);
  RouteParams p = route_params(x, k, sigmoid, 1, 1, renorm, scaling);
  auto dl = new_empty({p.T, p.E}, x, x.scalar_type());
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
  const int grid = std::min((p.T + kRouteWarps - 1) / kRouteWarps, num_sms() * 4);
  by_shape(x, [&](auto v, auto epl, auto vec) {
    launch_early(route_bwd_kernel<decltype(v), decltype(epl)::value, decltype(vec)::value>, grid, kRouteWarps * 32, 0, p);
  });
  EMB_LAUNCH_CHECK();
  count_launch();
  return dl;
}

}  // namespace emb
