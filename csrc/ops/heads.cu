// Rotary positions on the fused QKV layout, with or without an RMSNorm of every query and key head in the same
// pass.  qkv is [s, b, G, S, d]; of the S slots of a group the first nq are query heads, the next nk key heads,
// the rest (values) pass through.  With x one head, c / n the token's cosines and sines (r/2 of them, r <= d):
//
//   xh = x * rstd,  rstd = 1 / sqrt(mean(x^2) + eps)        (norm; otherwise xh w = x)
//   y  = R(xh w),   R turns the pairs (i, i + r/2) (halves) or (2i, 2i + 1) (interleaved), i < r/2:
//                   y_1 = x_1 c - x_2 n,  y_2 = x_2 c + x_1 n;  channels >= r pass
//   backward, g = R^T(dy):  dw = sum over heads of g xh,   dx = rstd (g w - xh mean(g w xh))
//
// All sums are fp32; results are rounded once, to the type of qkv.  dw is summed in a fixed order: registers, the
// lanes of a warp, the warps of a CTA, then the CTAs' partials, so it does not change from run to run.
//
// A head is held by LPH lanes, each with pairs of two VEC-channel vectors chosen so that both halves of every
// rotated pair sit in one lane: vectors (p, p + r/2/VEC) for halves, (2p, 2p + 1) for interleaved.  In both
// layouts pair p then uses cosines [VEC p, VEC p + VEC) and no rotation needs a shuffle; only the norm's mean does.
// VEC = 8 (16-byte accesses for 16-bit types) needs d % 8 == 0, r % 16 == 0 and aligned rows; every other shape
// (odd quarters of a head, unaligned views) takes VEC = 1, which touches the same sectors with narrower accesses.
#include "../include/common.cuh"

#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

namespace emb {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// VEC consecutive channels as fp32
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (VEC == 8) {
    constexpr int N = (int)sizeof(T) / 2;  // 16-byte words
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f<T>(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f<T>(p[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  if constexpr (VEC == 8) {
    constexpr int N = (int)sizeof(T) / 2;
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_f<T>(f[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = from_f<T>(f[i]);
  }
}

struct HeadParams {
  const void* x;       // qkv (forward, and the norm's backward)
  const void* dy;      // backward
  void* out;           // y or dx, contiguous
  const float* cosv;   // [s, r/2] or [s, b, r/2]
  const float* sinv;
  const void* w[2];    // norm weights of query and key heads
  float* part;         // backward: [blocks of classes 0 and 1, d] partial weight gradients
  long long xs, xb, ds, db;  // strides of x and dy over s and b, in elements
  long long tok_elems;       // G * S * d
  long long ts, tb;          // strides of the tables over s and b
  int B, S, G, d, r;
  float eps;
  long long tokens;
  int n[3];            // heads of each class in a group: query, key, other
  int block0[3];       // first block of each class
};

// Offset of pair `pair`'s first and second vector inside a head, and whether it turns.
template <int VEC, bool INTER>
__device__ __forceinline__ void pair_at(int pair, int r, int& a, int& b, bool& turn) {
  if constexpr (INTER) {
    a = 2 * pair * VEC;
    b = a + VEC;
    turn = a < r;
  } else {
    const int hv = r / (2 * VEC);
    turn = pair < hv;
    a = turn ? pair * VEC : r + 2 * (pair - hv) * VEC;
    b = turn ? (pair + hv) * VEC : a + VEC;
  }
}

template <int VEC, bool INTER>
__device__ __forceinline__ void rotate(float* a, float* b, const float* c, const float* n, bool inverse) {
  if constexpr (VEC == 1 || !INTER) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float s = inverse ? -n[j] : n[j], u = a[j], v = b[j];
      a[j] = u * c[j] - v * s;
      b[j] = v * c[j] + u * s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      float s = inverse ? -n[j] : n[j], u = a[2 * j], v = a[2 * j + 1];
      a[2 * j] = u * c[j] - v * s;
      a[2 * j + 1] = v * c[j] + u * s;
      s = inverse ? -n[VEC / 2 + j] : n[VEC / 2 + j], u = b[2 * j], v = b[2 * j + 1];
      b[2 * j] = u * c[VEC / 2 + j] - v * s;
      b[2 * j + 1] = v * c[VEC / 2 + j] + u * s;
    }
  }
}

template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kHeadThreads = 256;

// One launch does all heads; the blocks are split between the classes (query, key, passing) in proportion to
// their work, so that a block meets one weight vector and a lane always the same channels of it.
template <typename T, int VEC, int LPH, int PPL, bool INTER, bool NORM, bool BWD>
__global__ void __launch_bounds__(kHeadThreads) heads_kernel(HeadParams p) {
  const int cls = blockIdx.x >= p.block0[2] ? 2 : blockIdx.x >= p.block0[1] ? 1 : 0;
  const int blk = blockIdx.x - p.block0[cls];
  const int blocks = (cls == 2 ? gridDim.x : p.block0[cls + 1]) - p.block0[cls];
  constexpr int HPW = 32 / LPH;  // heads a warp holds at once
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPH;
  const int n = p.n[cls], cnt = n * p.G, first = cls == 0 ? 0 : cls == 1 ? p.n[0] : p.n[0] + p.n[1];
  // (the host bounds the heads of a call below 2^31; element offsets are 64-bit)
  const unsigned total = (unsigned)(p.tokens * cnt), step = (unsigned)blocks * (kHeadThreads / 32) * HPW;
  const T* xin = reinterpret_cast<const T*>(p.x);
  const T* din = reinterpret_cast<const T*>(p.dy);
  T* out = reinterpret_cast<T*>(p.out);

  int oa[PPL], ob[PPL];
  bool turn[PPL], has_a[PPL], has_b[PPL];
#pragma unroll
  for (int i = 0; i < PPL; ++i) {
    const int pair = l + i * LPH;
    pair_at<VEC, INTER>(pair, p.r, oa[i], ob[i], turn[i]);
    has_a[i] = oa[i] < p.d;
    has_b[i] = ob[i] < p.d;
    turn[i] = turn[i] && cls < 2;
  }
  float wa[PPL][VEC], wb[PPL][VEC], ga[PPL][VEC], gb[PPL][VEC];
  if (NORM) {
    const T* w = reinterpret_cast<const T*>(cls < 2 ? p.w[cls] : nullptr);
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) wa[i][j] = wb[i][j] = ga[i][j] = gb[i][j] = 0.f;
      if (cls < 2 && has_a[i]) load_vec<T, VEC>(w + oa[i], wa[i]);
      if (cls < 2 && has_b[i]) load_vec<T, VEC>(w + ob[i], wb[i]);
    }
  }
  // every lane of a warp runs the same number of rounds (the means shuffle); lanes past the end hold zeros
  for (unsigned h0 = ((unsigned)blk * (kHeadThreads / 32) + warp) * HPW; h0 < total; h0 += step) {
    const unsigned h = h0 + lane / LPH;
    const bool live = h < total;
    const unsigned tok = live ? h / (unsigned)cnt : 0u, head = live ? h - tok * cnt : 0u;
    const unsigned si = tok / (unsigned)p.B, bi = tok - si * p.B;
    const unsigned g = head / (unsigned)n, slot = first + head - g * n;
    const long long in_tok = ((long long)g * p.S + slot) * p.d;
    const T* px = xin + si * p.xs + bi * p.xb + in_tok;
    const T* pd = din + si * p.ds + bi * p.db + in_tok;
    T* po = out + (long long)tok * p.tok_elems + in_tok;
    const long long tab = si * p.ts + bi * p.tb;
    float a[PPL][VEC], b[PPL][VEC], xa[PPL][VEC], xb[PPL][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[i][j] = b[i][j] = xa[i][j] = xb[i][j] = 0.f;
      if (live && has_a[i]) load_vec<T, VEC>((BWD ? pd : px) + oa[i], a[i]);
      if (live && has_b[i]) load_vec<T, VEC>((BWD ? pd : px) + ob[i], b[i]);
      if (NORM && BWD && cls < 2) {
        if (live && has_a[i]) load_vec<T, VEC>(px + oa[i], xa[i]);
        if (live && has_b[i]) load_vec<T, VEC>(px + ob[i], xb[i]);
      }
    }
    float cs[PPL][VEC], sn[PPL][VEC];
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
      if (live && turn[i]) {
        load_vec<float, VEC>(p.cosv + tab + (l + i * LPH) * VEC, cs[i]);
        load_vec<float, VEC>(p.sinv + tab + (l + i * LPH) * VEC, sn[i]);
      }
    }
    if (NORM && cls < 2) {
#pragma unroll
      for (int i = 0; i < PPL; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = BWD ? xa[i][j] : a[i][j], v = BWD ? xb[i][j] : b[i][j];
          ss += u * u + v * v;
        }
      }
      const float rstd = rsqrtf(group_sum<LPH>(ss) / p.d + p.eps);
      if (!BWD) {
#pragma unroll
        for (int i = 0; i < PPL; ++i) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            a[i][j] *= rstd * wa[i][j];
            b[i][j] *= rstd * wb[i][j];
          }
          if (live && turn[i]) rotate<VEC, INTER>(a[i], b[i], cs[i], sn[i], false);
        }
      } else {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < PPL; ++i) {
          if (live && turn[i]) rotate<VEC, INTER>(a[i], b[i], cs[i], sn[i], true);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            xa[i][j] *= rstd;
            xb[i][j] *= rstd;
            ga[i][j] += a[i][j] * xa[i][j];
            gb[i][j] += b[i][j] * xb[i][j];
            a[i][j] *= wa[i][j];
            b[i][j] *= wb[i][j];
            dot += a[i][j] * xa[i][j] + b[i][j] * xb[i][j];
          }
        }
        const float m = group_sum<LPH>(dot) / p.d;
#pragma unroll
        for (int i = 0; i < PPL; ++i) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            a[i][j] = rstd * (a[i][j] - xa[i][j] * m);
            b[i][j] = rstd * (b[i][j] - xb[i][j] * m);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < PPL; ++i)
        if (live && turn[i]) rotate<VEC, INTER>(a[i], b[i], cs[i], sn[i], BWD);
    }
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
      if (live && has_a[i]) store_vec<T, VEC>(po + oa[i], a[i]);
      if (live && has_b[i]) store_vec<T, VEC>(po + ob[i], b[i]);
    }
  }
  if constexpr (NORM && BWD) {
    if (cls == 2) return;
    // this block's sum for each channel: over the warp's heads, then over the warps in order
    extern __shared__ float s_dw[];  // [warps, d]
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
          ga[i][j] += __shfl_xor_sync(0xffffffffu, ga[i][j], o);
          gb[i][j] += __shfl_xor_sync(0xffffffffu, gb[i][j], o);
        }
        if (lane < LPH && has_a[i]) s_dw[warp * p.d + oa[i] + j] = ga[i][j];
        if (lane < LPH && has_b[i]) s_dw[warp * p.d + ob[i] + j] = gb[i][j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += kHeadThreads) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kHeadThreads / 32; ++q) v += s_dw[q * p.d + c];
      p.part[(long long)blockIdx.x * p.d + c] = v;
    }
  }
}

// dw[cls][c] (+)= sum over the class's blocks of part[block][c]: 32 channels a CTA, 32 slices of the blocks, each
// slice summed in order and the slices joined by a fixed tree.
template <typename T>
__global__ void __launch_bounds__(1024) heads_join_kernel(const float* __restrict__ part, int d, int nb0, int nb1,
                                                          T* dw0, T* dw1, float* acc0, float* acc1) {
  __shared__ float sh[32][33];
  const int cls = blockIdx.y, b0 = cls ? nb0 : 0, b1 = cls ? nb0 + nb1 : nb0;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < d)
    for (int b = b0 + slice; b < b1; b += 32) v += part[(long long)b * d + c];
  sh[slice][lane] = v;
  __syncthreads();
  v = warp_sum(sh[lane][slice]);  // slices of channel blockIdx.x * 32 + slice
  const int ch = blockIdx.x * 32 + slice;
  if (lane == 0 && ch < d) {
    float* acc = cls ? acc1 : acc0;
    if (acc) {
      acc[ch] += v;
    } else {
      (cls ? dw1 : dw0)[ch] = from_f<T>(v);
    }
  }
}

template <typename T, int VEC, int LPH, int PPL, bool INTER, bool NORM, bool BWD>
void launch_heads(const HeadParams& p, int grid) {
  const int smem = NORM && BWD ? (kHeadThreads / 32) * p.d * (int)sizeof(float) : 0;
  heads_kernel<T, VEC, LPH, PPL, INTER, NORM, BWD><<<grid, kHeadThreads, smem, cur_stream()>>>(p);
}

template <typename T, int VEC, int LPH, int PPL>
void pick_mode(const HeadParams& p, int grid, bool inter, bool norm, bool bwd) {
  if (inter) {
    if (norm) bwd ? launch_heads<T, VEC, LPH, PPL, true, true, true>(p, grid)
                  : launch_heads<T, VEC, LPH, PPL, true, true, false>(p, grid);
    else bwd ? launch_heads<T, VEC, LPH, PPL, true, false, true>(p, grid)
             : launch_heads<T, VEC, LPH, PPL, true, false, false>(p, grid);
  } else {
    if (norm) bwd ? launch_heads<T, VEC, LPH, PPL, false, true, true>(p, grid)
                  : launch_heads<T, VEC, LPH, PPL, false, true, false>(p, grid);
    else bwd ? launch_heads<T, VEC, LPH, PPL, false, false, true>(p, grid)
             : launch_heads<T, VEC, LPH, PPL, false, false, false>(p, grid);
  }
}

// Lanes per head: the pairs of a head rounded up to a power of two, so that the mean's shuffles stay inside it.
int lanes_per_head(int d, int vec) {
  const int pairs = (d / vec + 1) / 2;
  int l = 1;
  while (l < pairs && l < 32) l *= 2;
  return l;
}

template <typename T>
void pick_shape(const HeadParams& p, int grid, bool vec, bool inter, bool norm, bool bwd) {
  if (vec) {
    switch (lanes_per_head(p.d, 8)) {
      case 1: case 2: case 4: return pick_mode<T, 8, 4, 1>(p, grid, inter, norm, bwd);
      case 8: return pick_mode<T, 8, 8, 1>(p, grid, inter, norm, bwd);
      case 16: return pick_mode<T, 8, 16, 1>(p, grid, inter, norm, bwd);
      default: return pick_mode<T, 8, 32, 1>(p, grid, inter, norm, bwd);
    }
  }
  if (p.d <= 128) return pick_mode<T, 1, 32, 2>(p, grid, inter, norm, bwd);
  return pick_mode<T, 1, 32, 8>(p, grid, inter, norm, bwd);
}

void check_table(const at::Tensor& t, const at::Tensor& qkv, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == qkv.device() && t.scalar_type() == at::kFloat, name,
              " must be an fp32 tensor on the device of qkv");
  TORCH_CHECK(t.dim() == 2 || t.dim() == 3, name, " must be [s, r/2] or [s, b, r/2]");
  TORCH_CHECK(t.size(0) == qkv.size(0) && (t.dim() == 2 || t.size(1) == qkv.size(1)), name,
              " must have a row for every position of qkv");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// qkv as [s, b, (G S d contiguous)]: a view with other strides over s and b is read in place
at::Tensor inner_contiguous(const at::Tensor& t) {
  const int64_t S = t.size(3), d = t.size(4), G = t.size(2);
  const bool ok = (d == 1 || t.stride(4) == 1) && (S == 1 || t.stride(3) == d) && (G == 1 || t.stride(2) == S * d);
  return ok ? t : t.contiguous();
}

// Fills the parameters that forward and backward share; returns whether rows allow 8-channel vectors.
bool set_up(HeadParams& p, const at::Tensor& t, const at::Tensor& cosv, const at::Tensor& sinv, int64_t nq, int64_t nk) {
  TORCH_CHECK(t.dim() == 5, "qkv must be [s, b, G, slots, d]");
  const int64_t s = t.size(0), b = t.size(1), G = t.size(2), S = t.size(3), d = t.size(4);
  TORCH_CHECK(nq >= 0 && nk >= 0 && nq + nk <= S, "more query and key heads than slots in a group");
  check_table(cosv, t, "cos");
  check_table(sinv, t, "sin");
  TORCH_CHECK(cosv.sizes() == sinv.sizes(), "cos and sin must have the same shape");
  const int64_t r = 2 * cosv.size(-1);
  TORCH_CHECK(d <= 512 && d % 2 == 0 && r <= d, "head size must be even, at most 512, and hold the turned channels");
  TORCH_CHECK(s * b * G * S < (1ll << 30), "too many heads in one call");
  p.cosv = cosv.data_ptr<float>();
  p.sinv = sinv.data_ptr<float>();
  p.tok_elems = G * S * d;
  p.ts = cosv.dim() == 3 ? b * (r / 2) : r / 2;
  p.tb = cosv.dim() == 3 ? r / 2 : 0;
  p.B = (int)b;
  p.S = (int)S;
  p.G = (int)G;
  p.d = (int)d;
  p.r = (int)r;
  p.tokens = s * b;
  p.n[0] = (int)nq;
  p.n[1] = (int)nk;
  p.n[2] = (int)(S - nq - nk);
  return d % 8 == 0 && r % 16 == 0 && (uintptr_t)p.cosv % 16 == 0 && (uintptr_t)p.sinv % 16 == 0;
}

bool rows_aligned(const at::Tensor& t) {
  const int64_t e = 16 / t.element_size();
  return (uintptr_t)t.data_ptr() % 16 == 0 && t.stride(0) % e == 0 && t.stride(1) % e == 0;
}

// Splits the grid between the classes by the heads of each; returns the grid.
int split_grid(HeadParams& p, bool vec, int waves) {
  const int hpw = vec ? 32 / std::max(4, lanes_per_head(p.d, 8)) : 1;
  const long long per_block = (long long)hpw * (kHeadThreads / 32);
  const long long all = p.tokens * p.G * p.S;
  const long long cap = (long long)num_sms() * waves;
  int at = 0;
  for (int c = 0; c < 3; ++c) {
    p.block0[c] = at;
    const long long heads = p.tokens * p.G * p.n[c];
    const long long want = (heads + per_block - 1) / per_block;
    const long long share = std::max<long long>(1, cap * heads / std::max<long long>(1, all));
    at += heads ? (int)std::min(want, share) : 0;
  }
  return at;
}

template <typename F>
void by_type(at::ScalarType t, F f) {
  if (t == at::kBFloat16) f(__nv_bfloat16{});
  else if (t == at::kHalf) f(__half{});
  else if (t == at::kFloat) f(float{});
  else TORCH_CHECK(false, "qkv must be bf16, fp16 or fp32");
}

constexpr int kHeadWaves = 8;

void check_weights(const c10::optional<at::Tensor>& w, const at::Tensor& t, const char* name) {
  TORCH_CHECK(w.has_value() && w->is_cuda() && w->device() == t.device() && w->scalar_type() == t.scalar_type() &&
                  w->dim() == 1 && w->size(0) == t.size(4) && w->is_contiguous(),
              name, " must be a contiguous [d] tensor of qkv's type and device");
}

}  // namespace

at::Tensor heads_fwd(at::Tensor qkv, at::Tensor cosv, at::Tensor sinv, int64_t nq, int64_t nk, bool interleaved,
                     c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk, double eps) {
  TORCH_CHECK(qkv.is_cuda(), "qkv must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(qkv.device());
  HeadParams p{};
  const bool norm = wq.has_value();
  bool vec = set_up(p, qkv, cosv, sinv, nq, nk);
  auto x = inner_contiguous(qkv);
  if (norm) {
    check_weights(wq, x, "q_weight");
    check_weights(wk, x, "k_weight");
    p.w[0] = wq->data_ptr();
    p.w[1] = wk->data_ptr();
    vec = vec && (uintptr_t)p.w[0] % 16 == 0 && (uintptr_t)p.w[1] % 16 == 0;
  }
  auto out = at::empty(x.sizes(), x.options());
  if (out.numel() == 0) return out;
  p.x = x.data_ptr();
  p.xs = x.stride(0);
  p.xb = x.stride(1);
  p.out = out.data_ptr();
  p.eps = (float)eps;
  vec = vec && rows_aligned(x);
  const int grid = split_grid(p, vec, kHeadWaves);
  by_type(x.scalar_type(), [&](auto t) { pick_shape<decltype(t)>(p, grid, vec, interleaved, norm, false); });
  EMB_LAUNCH_CHECK();
  count_launch();
  return out;
}

// Returns {dx} or, with norm weights, {dx, dwq, dwk}; a weight gradient goes into its fp32 accumulator where one
// is given (the returned tensor is then undefined), else into a new tensor of the weight's type.
std::vector<at::Tensor> heads_bwd(at::Tensor dy, c10::optional<at::Tensor> qkv, at::Tensor cosv, at::Tensor sinv,
                                  int64_t nq, int64_t nk, bool interleaved, c10::optional<at::Tensor> wq,
                                  c10::optional<at::Tensor> wk, double eps, c10::optional<at::Tensor> dwq_accum,
                                  c10::optional<at::Tensor> dwk_accum) {
  TORCH_CHECK(dy.is_cuda(), "dy must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(dy.device());
  HeadParams p{};
  const bool norm = wq.has_value();
  bool vec = set_up(p, dy, cosv, sinv, nq, nk);
  auto g = inner_contiguous(dy);
  at::Tensor x;
  if (norm) {
    TORCH_CHECK(qkv.has_value() && qkv->sizes() == dy.sizes() && qkv->scalar_type() == dy.scalar_type() &&
                    qkv->device() == dy.device(), "dy must have the shape, type and device of qkv");
    x = inner_contiguous(*qkv);
    check_weights(wq, x, "q_weight");
    check_weights(wk, x, "k_weight");
    p.w[0] = wq->data_ptr();
    p.w[1] = wk->data_ptr();
    p.x = x.data_ptr();
    p.xs = x.stride(0);
    p.xb = x.stride(1);
    vec = vec && rows_aligned(x) && (uintptr_t)p.w[0] % 16 == 0 && (uintptr_t)p.w[1] % 16 == 0;
  }
  auto dx = at::empty(g.sizes(), g.options());
  std::vector<at::Tensor> res{dx};
  float* acc[2] = {nullptr, nullptr};
  void* dw[2] = {nullptr, nullptr};
  if (norm) {
    int i = 0;
    for (auto* a : {&dwq_accum, &dwk_accum}) {
      if (a->has_value()) {
        TORCH_CHECK((*a)->is_cuda() && (*a)->scalar_type() == at::kFloat && (*a)->is_contiguous() &&
                        (*a)->numel() == p.d, "a weight gradient accumulator must be a contiguous fp32 [d] tensor");
        acc[i] = (*a)->data_ptr<float>();
        res.emplace_back();
      } else {
        res.push_back(at::empty({p.d}, g.options()));
        dw[i] = res.back().data_ptr();
      }
      ++i;
    }
  }
  if (dx.numel() == 0) {
    for (int i = 0; norm && i < 2; ++i)
      if (dw[i]) res[1 + i].zero_();
    return res;
  }
  p.dy = g.data_ptr();
  p.ds = g.stride(0);
  p.db = g.stride(1);
  p.out = dx.data_ptr();
  p.eps = (float)eps;
  vec = vec && rows_aligned(g);
  const int grid = split_grid(p, vec, kHeadWaves);
  at::Tensor part;
  const int nb0 = p.block0[1], nb1 = p.block0[2] - p.block0[1];
  if (norm) {
    part = at::empty({nb0 + nb1, p.d}, g.options().dtype(at::kFloat));
    p.part = part.data_ptr<float>();
  }
  by_type(g.scalar_type(), [&](auto t) {
    using T = decltype(t);
    pick_shape<T>(p, grid, vec, interleaved, norm, true);
    if (norm) {
      heads_join_kernel<T><<<dim3((p.d + 31) / 32, 2), 1024, 0, cur_stream()>>>(
          p.part, p.d, nb0, nb1, (T*)dw[0], (T*)dw[1], acc[0], acc[1]);
    }
  });
  EMB_LAUNCH_CHECK();
  count_launch(norm ? 2 : 1);
  return res;
}

}  // namespace emb
