// Rotary positions on the fused QKV layout, with or without an RMSNorm of every query and key head in the same
// pass.  qkv is [s, b, G, S, d]; of the S slots of a group the first nq are query heads, the next nk key heads,
// the rest (values) pass through.  With x one head, c / n the token's cosines and sines (r/2 of them, r <= d):
//
//   xh = x * rstd,  rstd = 1 / sqrt(mean(x^2) + eps)        (norm; otherwise xh w = x)
//   y  = R(xh w),   R turns the pairs (i, i + r/2) (halves) or (2i, 2i + 1) (interleaved), i < r/2:
//                   y_1 = x_1 c - x_2 n,  y_2 = x_2 c + x_1 n;  channels >= r pass
//   backward, g = R^T(dy):  dw = sum over heads of g xh,   dx = rstd (g w - xh mean(g w xh))
//
// Two kernels: a direct one, which holds its heads in registers (small calls, views, turns that do not fill vectors), and a
// streamed one for the rest, both bound by memory.  Of a copy's rate at 8192 x 4 tokens, 8 x (4 + 2) heads of 128, bf16: norm
// forward 128 us (0.97), norm backward 190 us (0.92 of the bytes' floor); rotation alone at 8192 x 2 tokens 65.6 us (0.94).
//
// All sums are fp32; results are rounded once, to the type of qkv.  dw is summed in a fixed order: registers, the
// lanes of a warp, the warps of a CTA, then the CTAs' partials, so it does not change from run to run.
//
// In the direct kernel a head is held by LPH lanes, each with pairs of two VEC-channel vectors chosen so that both halves of every
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
// their work, so that a block meets one weight vector and a lane always the same channels of it.  Bound by latency at the
// sizes that it is for: 64 tokens of 8 single heads of 64 take 2.4 us forward and 4.8 us backward with its join.
template <typename T, int VEC, int LPH, int PPL, bool INTER, bool NORM, bool BWD>
__global__ void __launch_bounds__(kHeadThreads) heads_kernel(HeadParams p) {
  grid_dependency();
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

// ------------------------------------------------------------------------------------------ streamed kernel
// The same operator for dense tensors.  Memory bound, so the data must not wait for registers: every warp streams
// tiles of 2 or 4 KB of consecutive heads through a ring of its own in shared memory (cp.async.bulk, an mbarrier a
// stage), turns them in place and sends them out with a bulk store.  Values pass without an instruction.  No warp waits
// for another; the loads of the next stages are in flight while a tile is worked on.
// Of one tensor, or each of two (dy and x).  Tiles of 4 KB take the rotation of 8192 x 2 x 48 x 128 from 69.7 to 65.6 us
// (a copy of it: 61.5); with two tensors they would leave one CTA an SM.
constexpr int tile_bytes(bool two) { return two ? 2048 : 4096; }
constexpr int kStreamWarps = 8;
constexpr unsigned kWaitPolls = 1u << 24;  // seconds of polling before a wait gives up

struct FastDiv {  // n / d for n < 2^30
  unsigned mul, shift, d;
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};
FastDiv fast_div(unsigned d) {
  unsigned s = 0;
  while ((1ull << s) < d) ++s;
  return {(unsigned)((((1ull << s) - d) << 32) / d + 1), s, d};
}

struct StreamParams {
  const void* x;
  const void* dy;
  void* out;
  const float* cosv;
  const float* sinv;
  const void* w[2];
  float* part;  // [blocks, 2, d]
  int* err;
  FastDiv per_token, slots, turned, rows;  // heads of a token, of a group, turned ones of a group; tokens of a table row
  int whole;  // tiles are whole groups
  int d, r, nq, nk;
  unsigned heads, tile_heads, tiles, per_row;  // per_row: consecutive heads that share a row of the tables
  float eps, inv_d;
};

__device__ __forceinline__ unsigned smem_at(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// ONCE: the rotation alone does not read its input again (evicted from L2 first); the norm does, in its backward.
// (Rotation of 8192 x 2 x 48 x 128, calls back to back: 70.5 -> 68.2 us.)
template <bool ONCE>
__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, uint64_t* bar) {
  if constexpr (ONCE) {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_at(dst)),
        "l"(src), "r"(bytes), "r"(smem_at(bar)), "l"(policy)
        : "memory");
  } else {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_at(dst)),
                 "l"(src), "r"(bytes), "r"(smem_at(bar))
                 : "memory");
  }
}
__device__ __forceinline__ bool bulk_wait(uint64_t* bar, unsigned parity) {
  for (unsigned i = 0; i < kWaitPolls; ++i) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_at(bar)), "r"(parity)
                 : "memory");
    if (ok) return true;
  }
  return false;
}

// Two fp32 in one 64-bit register, for the packed arithmetic of sm_100 (one instruction for both).
typedef unsigned long long f2;
__device__ __forceinline__ f2 f2_of(float a, float b) {
  f2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 f2_to(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
  f2 v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

// 8 channels as 4 pairs
template <typename T>
__device__ __forceinline__ void load8(const T* p, f2* v) {
  if constexpr (sizeof(T) == 4) {
    const ulonglong2* q = reinterpret_cast<const ulonglong2*>(p);
    const ulonglong2 u0 = q[0], u1 = q[1];
    v[0] = u0.x;
    v[1] = u0.y;
    v[2] = u1.x;
    v[3] = u1.y;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[i] = f2_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[i] = f2_of(f.x, f.y);
      }
    }
  }
}
// 4 channels as 2 pairs
template <typename T>
__device__ __forceinline__ void load4(const T* p, f2* v) {
  if constexpr (sizeof(T) == 4) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p);
    v[0] = u.x;
    v[1] = u.y;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const unsigned w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[i] = f2_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[i] = f2_of(f.x, f.y);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ unsigned pack2(f2 v) {
  const float2 f = f2_to(v);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const unsigned*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const unsigned*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const f2* v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0], v[1]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0]), pack2<T>(v[1]));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const f2* v) {
  if constexpr (sizeof(T) == 4) {
    ulonglong2* q = reinterpret_cast<ulonglong2*>(p);
    q[0] = make_ulonglong2(v[0], v[1]);
    q[1] = make_ulonglong2(v[2], v[3]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0]), pack2<T>(v[1]), pack2<T>(v[2]), pack2<T>(v[3]));
  }
}

// 4 cosines and sines from column `col` of a row of the tables
__device__ __forceinline__ void load_turn(const StreamParams& p, unsigned row, int col, f2* c, f2* s) {
  const size_t at = (size_t)row * (p.r / 2) + col;
  const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p.cosv + at), v = *reinterpret_cast<const ulonglong2*>(p.sinv + at);
  c[0] = u.x;
  c[1] = u.y;
  s[0] = v.x;
  s[1] = v.y;
}

// What a lane holds of its head: four quarters of 4 channels, q[i] in all.  Halves: quarter i turns with quarter i + 2 if
// turn[i], by cosines [8 lane + 4 i, ..).  Interleaved: pairs lie inside a quarter; quarters 0 and 1 turn if turn[0], 2 and 3
// if turn[1].  UNIT 8: quarters 0 and 1, and 2 and 3, are one aligned vector of 8 channels; UNIT 4 serves halves of r = 8 mod
// 16 channels, where a vector of 8 would meet its partner at an offset of 4.
struct Held {
  int at[4];
  bool has[4], turn[2];
};
template <int UNIT, bool INTER>
__device__ __forceinline__ Held held_by(int lane, int d, int r) {
  Held h;
  if constexpr (UNIT == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pair = 2 * lane + i;
      h.turn[i] = pair < r / 8;
      h.at[i] = h.turn[i] ? 4 * pair : r + 8 * (pair - r / 8);
      h.at[i + 2] = h.turn[i] ? 4 * pair + r / 2 : h.at[i] + 4;
      h.has[i] = h.has[i + 2] = pair < d / 8;
    }
  } else {
    const int pairs = (d / 8 + 1) / 2;  // lanes past them hold nothing
    int a, b;
    if constexpr (INTER) {  // neighbouring lanes take neighbouring vectors (no bank conflicts)
      a = lane * 8;
      b = a + pairs * 8;
      h.turn[0] = a < r;
      h.turn[1] = b < r;
    } else {
      const int hv = r / 16;
      h.turn[0] = h.turn[1] = lane < hv;
      a = lane < hv ? lane * 8 : r + 2 * (lane - hv) * 8;
      b = lane < hv ? (lane + hv) * 8 : a + 8;
    }
    h.has[0] = h.has[1] = lane < pairs && a < d;
    h.has[2] = h.has[3] = lane < pairs && b < d;
    h.at[0] = a;
    h.at[1] = a + 4;
    h.at[2] = b;
    h.at[3] = b + 4;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) h.turn[i] = h.turn[i] && h.has[INTER ? 2 * i : i];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (!h.has[i]) h.at[i] = 0;
  return h;
}

// A lane works on 16 channels of a head in packed fp32 and keeps the cosines and sines while it meets heads of one token
// (for the norm's backward a warp takes consecutive tiles, so that this is often); the norm weights sit in shared memory
// as fp32, [class][quarter][lane] so that a lane's four 16-byte reads are free of bank conflicts.  What keeps the
// kernel from the memory's rate otherwise is the number of instructions: 4 heads of 128 channels have about 350 issue
// slots forward and 500 backward at the rate of a plain copy; they take 196 and 308 instructions (394 and 611 in scalar
// arithmetic, which made this kernel slower than the direct one).
template <typename T, int LPH, int STAGES, int UNIT, bool INTER, bool NORM, bool BWD>
__global__ void __launch_bounds__(kStreamWarps * 32, 2) heads_stream_kernel(StreamParams p) {
  constexpr int HPW = 32 / LPH;
  constexpr int BUFS = NORM && BWD ? 2 : 1;  // dy (or x), and x
  // Tiles a warp takes in a row: the norm's backward, short of issue slots, so meets heads of one token in a row and loads its
  // cosines and sines less often (backward of 8192 x 4 / 8192 tokens, runs of 2 / 4 / 8 / 16 tiles: 202 / 194 / 190 / 192 and
  // 59.1 / 58.0 / 57.1 / 57.1 us; one run for all of a warp's tiles 200 to 209 and 56.0).
  constexpr unsigned RUN = NORM && BWD ? 8 : 1;
  constexpr int kTileBytes = tile_bytes(NORM && BWD);
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ uint64_t s_bar[kStreamWarps][STAGES];
  __shared__ __align__(16) float s_w[NORM ? 2 : 1][4][LPH][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPH, sub = lane / LPH;
  uint8_t* ring = s_ring + warp * (STAGES * BUFS * kTileBytes);
  uint64_t* bar = s_bar[warp];
  const unsigned head_bytes = p.d * (unsigned)sizeof(T);
  // The warps walk the tensor together, each taking RUN consecutive tiles at a time, and share what is left evenly.
  const unsigned me = blockIdx.x * kStreamWarps + warp, warps = gridDim.x * kStreamWarps;
  const unsigned whole = p.tiles / (warps * RUN), rest = p.tiles - whole * warps * RUN;
  const unsigned rest0 = (unsigned)((unsigned long long)rest * me / warps);
  const unsigned mine = whole * RUN + (unsigned)((unsigned long long)rest * (me + 1) / warps) - rest0;
  auto tile_of = [&](unsigned it) -> unsigned {
    return it < whole * RUN ? (it / RUN * warps + me) * RUN + it % RUN : whole * warps * RUN + rest0 + it - whole * RUN;
  };
  const char* src0 = reinterpret_cast<const char*>(BWD ? p.dy : p.x);
  const char* src1 = reinterpret_cast<const char*>(p.x);

  const Held held = held_by<UNIT, INTER>(l, p.d, p.r);
  const bool full = LPH * 16 == p.d;  // every lane holds four quarters

  auto load = [&](unsigned tile, int st) {  // lane 0
    const unsigned h0 = tile * p.tile_heads, n = min(p.tile_heads, p.heads - h0), bytes = n * head_bytes;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(bar + st)), "r"(bytes * BUFS)
                 : "memory");
    bulk_load<!NORM>(ring + st * BUFS * kTileBytes, src0 + (size_t)h0 * head_bytes, bytes, bar + st);
    if (BUFS == 2) bulk_load<!NORM>(ring + (st * BUFS + 1) * kTileBytes, src1 + (size_t)h0 * head_bytes, bytes, bar + st);
  };

  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_at(bar + i)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  grid_dependency();
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      if (i < mine) load(tile_of(i), i);
  }
  f2 gw[NORM && BWD ? 2 : 1][8];
  if constexpr (NORM) {
    if (threadIdx.x < 2 * LPH) {  // thread (class, l) lays out that lane's weights
      const int c = threadIdx.x / LPH, q = threadIdx.x % LPH;
      const Held his = held_by<UNIT, INTER>(q, p.d, p.r);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        s_w[c][j / 4][q][j & 3] =
            his.has[j / 4] ? to_f<T>(reinterpret_cast<const T*>(p.w[c])[his.at[j / 4] + (j & 3)]) : 0.f;
    }
#pragma unroll
    for (int c = 0; c < (BWD ? 2 : 1); ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) gw[c][j] = 0ull;
    __syncthreads();
  } else {
    __syncwarp();
  }

  unsigned from = 0x80000000u;  // first head of the table row in cs / sn (none yet)
  f2 cs[4], sn[4];
  for (unsigned it = 0; it < mine; ++it) {
    const unsigned tile = tile_of(it);
    const int st = it % STAGES;
    if (!bulk_wait(bar + st, (it / STAGES) & 1)) {
      // a copy that does not arrive: report it, and leave after a bounded wait for the copies in flight
      if (lane == 0) atomicExch(p.err, 1);
      for (int i = 0; i < STAGES; ++i) bulk_wait(bar + i, ((it + i) / STAGES) & 1);
      break;
    }
    uint8_t* buf = ring + st * BUFS * kTileBytes;
    const unsigned h0 = tile * p.tile_heads, n = min(p.tile_heads, p.heads - h0);
    const unsigned work = p.whole ? p.slots.div(n) * (unsigned)(p.nq + p.nk) : n;
#pragma unroll 1
    for (unsigned i0 = 0; i0 < work; i0 += HPW) {
      // tiles of whole groups: the i-th query or key head.  Else the i-th head; values are then read and worked on like
      // any other but neither counted nor written, as are the lanes past the end
      unsigned i = i0 + sub, slot;
      bool live = i < work;
      if (!live) i = 0;
      if (p.whole) {
        const unsigned g = p.turned.div(i);
        slot = i - g * p.turned.d;
        i = g * p.slots.d + slot;
      } else {
        slot = h0 + i - p.slots.div(h0 + i) * p.slots.d;
        live = live && slot < (unsigned)(p.nq + p.nk);
      }
      const unsigned h = h0 + i;
      const bool is_k = slot >= (unsigned)p.nq;
      T* head = reinterpret_cast<T*>(buf + i * head_bytes);
      if (live && h - from >= p.per_row) {  // another row of the tables than the lane's last head had
        const unsigned row = p.rows.div(p.per_token.div(h));
        from = row * p.per_row;
        if constexpr (INTER) {
          if (held.turn[0]) load_turn(p, row, held.at[0] / 2, cs, sn);
          if (held.turn[1]) load_turn(p, row, held.at[2] / 2, cs + 2, sn + 2);
        } else {
          if (held.turn[0]) load_turn(p, row, held.at[0], cs, sn);
          if (held.turn[1]) load_turn(p, row, held.at[1], cs + 2, sn + 2);
        }
      }
      f2 a[8], x[8];
      if constexpr (UNIT == 8) {
        load8<T>(head + held.at[0], a);
        load8<T>(head + held.at[2], a + 4);
        if constexpr (NORM && BWD) {
          load8<T>(head + held.at[0] + kTileBytes / sizeof(T), x);
          load8<T>(head + held.at[2] + kTileBytes / sizeof(T), x + 4);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          load4<T>(head + held.at[q], a + 2 * q);
          if constexpr (NORM && BWD) load4<T>(head + held.at[q] + kTileBytes / sizeof(T), x + 2 * q);
        }
      }
      if (!full) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!held.has[j / 2]) {
            a[j] = 0ull;
            if (NORM && BWD) x[j] = 0ull;
          }
        }
      }
      auto turn = [&](f2* v) {
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (held.turn[j / 4]) {
              const float2 c = f2_to(cs[j / 2]), s = f2_to(sn[j / 2]), u = f2_to(v[j]);
              const float cj = j & 1 ? c.y : c.x, sj = j & 1 ? s.y : s.x;
              v[j] = BWD ? f2_of(u.x * cj + u.y * sj, u.y * cj - u.x * sj) : f2_of(u.x * cj - u.y * sj, u.y * cj + u.x * sj);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!held.turn[j / 2]) continue;
            const f2 u = v[j], w = v[4 + j], neg = f2_mul(sn[j], f2_of(-1.f, -1.f));
            v[j] = f2_fma(w, BWD ? sn[j] : neg, f2_mul(u, cs[j]));
            v[4 + j] = f2_fma(u, BWD ? neg : sn[j], f2_mul(w, cs[j]));
          }
        }
      };
      if constexpr (NORM) {
        const f2* y = BWD ? x : a;
        f2 ss = 0ull;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = f2_fma(y[j], y[j], ss);
        const float2 s2 = f2_to(ss);
        const float rstd = rsqrtf(group_sum<LPH>(s2.x + s2.y) * p.inv_d + p.eps);
        const f2 r2 = f2_of(rstd, rstd);
        const float* wl = &s_w[is_k ? 1 : 0][0][l][0];
        f2 w[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(wl + q * LPH * 4);
          w[2 * q] = u.x;
          w[2 * q + 1] = u.y;
        }
        if constexpr (!BWD) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = f2_mul(f2_mul(a[j], r2), w[j]);
          turn(a);
        } else {
          // with b = g rstd:  dw += b x,  dx = b w - x rstd^2 mean(b w x)
          turn(a);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = f2_mul(a[j], r2);
          if (live) {
            if (is_k) {
#pragma unroll
              for (int j = 0; j < 8; ++j) gw[1][j] = f2_fma(a[j], x[j], gw[1][j]);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) gw[0][j] = f2_fma(a[j], x[j], gw[0][j]);
            }
          }
          f2 dot = 0ull;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            a[j] = f2_mul(a[j], w[j]);
            dot = f2_fma(a[j], x[j], dot);
          }
          const float2 d2 = f2_to(dot);
          const float m = group_sum<LPH>(d2.x + d2.y) * (-p.inv_d * rstd * rstd);
          const f2 m2 = f2_of(m, m);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = f2_fma(x[j], m2, a[j]);
        }
      } else {
        turn(a);
      }
      if constexpr (UNIT == 8) {
        if (live && held.has[0]) store8<T>(head + held.at[0], a);
        if (live && held.has[2]) store8<T>(head + held.at[2], a + 4);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (live && held.has[q]) store4<T>(head + held.at[q], a + 2 * q);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                       reinterpret_cast<char*>(p.out) + (size_t)h0 * head_bytes),
                   "r"(smem_at(buf)), "r"(n * head_bytes)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the stage of the tile before this one is free once its store has read it
      if (it > 0 && it + STAGES - 1 < mine) {
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        load(tile_of(it + STAGES - 1), (it - 1) % STAGES);
      }
    }
    __syncwarp();
  }
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  if constexpr (NORM && BWD) {
    __syncthreads();  // every ring is done with: [warps, 2, d] sums of the weight gradients take its place
    float* s_dw = reinterpret_cast<float*>(s_ring);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float2 v = f2_to(gw[c][j]);
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
          v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
          v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
        const int ch = held.at[j / 2] + 2 * (j & 1);
        if (sub == 0 && held.has[j / 2]) *reinterpret_cast<float2*>(&s_dw[(warp * 2 + c) * p.d + ch]) = v;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += kStreamWarps * 32) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kStreamWarps; ++q) v += s_dw[q * 2 * p.d + i];
      p.part[(size_t)blockIdx.x * 2 * p.d + i] = v;
    }
  }
}

// dw[cls][c] (+)= sum over the class's blocks of part[block][c]: 8 channels a CTA and 128 slices of the blocks, so that a
// thread has two or three loads to wait for at once; slices are joined by a fixed tree.
template <typename T>
__global__ void __launch_bounds__(1024) heads_join_kernel(const float* __restrict__ part, int d, int nb0, int nb1, int both,
                                                          int first, T* dw0, T* dw1, float* acc0, float* acc1) {
  __shared__ float sh[32][9];
  grid_dependency();
  // rows of `part`: those of class 0 and then those of class 1, or (`both`) the two of each block side by side
  const int cls = first + blockIdx.y, by = both ? 2 : 1;
  const int b0 = both ? 0 : cls ? nb0 : 0, b1 = both ? nb0 : cls ? nb0 + nb1 : nb0, shift = both ? cls : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 8 + (lane & 7);
  float v = 0.f;
  if (c < d) {
#pragma unroll 4
    for (int b = b0 + (threadIdx.x >> 3); b < b1; b += 128) v += part[((long long)b * by + shift) * d + c];
  }
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (lane < 8) sh[warp][lane] = v;
  __syncthreads();
  if (warp >= 8) return;
  v = warp_sum(sh[lane][warp]);
  const int ch = blockIdx.x * 8 + warp;
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
  launch_early(heads_kernel<T, VEC, LPH, PPL, INTER, NORM, BWD>, grid, kHeadThreads, smem, p);
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
  TORCH_CHECK_VALUE(t.dim() == 2 || t.dim() == 3, name, " must be [s, r/2] or [s, b, r/2]");
  TORCH_CHECK_VALUE(t.size(0) == qkv.size(0) && (t.dim() == 2 || t.size(1) == qkv.size(1)), name,
                    " must have a row for every position of qkv");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// qkv as [s, b, (G S d contiguous)]: a view with other strides over s and b is read in place
at::Tensor inner_contiguous(const at::Tensor& t) {
  const int64_t S = t.size(3), d = t.size(4), G = t.size(2);
  const bool ok = (d == 1 || t.stride(4) == 1) && (S == 1 || t.stride(3) == d) && (G == 1 || t.stride(2) == S * d);
  return ok ? t : t.contiguous();
}

// Whether rows allow 8-channel vectors, in the direct and in the streamed kernel.
struct Access {
  bool direct, stream;
  void need(bool ok) {
    direct = direct && ok;
    stream = stream && ok;
  }
};

// Fills the parameters that forward and backward share.
Access set_up(HeadParams& p, const at::Tensor& t, const at::Tensor& cosv, const at::Tensor& sinv, int64_t nq, int64_t nk) {
  TORCH_CHECK_VALUE(t.dim() == 5, "qkv must be [s, b, groups, slots, d]");
  const int64_t s = t.size(0), b = t.size(1), G = t.size(2), S = t.size(3), d = t.size(4);
  TORCH_CHECK_VALUE(nq >= 0 && nk >= 0 && nq + nk <= S, "more query and key heads than slots in a group");
  check_table(cosv, t, "cos");
  check_table(sinv, t, "sin");
  TORCH_CHECK_VALUE(cosv.sizes() == sinv.sizes(), "cos and sin must have the same shape");
  const int64_t r = 2 * cosv.size(-1);
  TORCH_CHECK_VALUE(d <= 512 && d % 2 == 0 && r <= d, "head size must be even, at most 512, and hold the turned channels");
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
  const bool ok = d % 8 == 0 && (uintptr_t)p.cosv % 16 == 0 && (uintptr_t)p.sinv % 16 == 0;
  return {ok && r % 16 == 0, ok && r % 8 == 0};
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

template <typename T, int LPH, int UNIT, bool INTER, bool NORM, bool BWD>
void launch_stream(const StreamParams& p, int grid) {
  constexpr int kStages = 3;
  constexpr int kSmem = kStreamWarps * kStages * tile_bytes(NORM && BWD) * (NORM && BWD ? 2 : 1);
  auto kern = heads_stream_kernel<T, LPH, kStages, UNIT, INTER, NORM, BWD>;
  static bool done[kMaxDevices] = {};  // the shared-memory limit belongs to the device's context
  int dev = 0;
  EMB_CUDA_CHECK(cudaGetDevice(&dev));
  if (!done[dev]) {
    EMB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    done[dev] = true;
  }
  launch_early(kern, grid, kStreamWarps * 32, kSmem, p);
}

template <typename T, int LPH, int UNIT, bool INTER>
void pick_stream_mode(const StreamParams& p, int grid, bool norm, bool bwd) {
  if (norm) bwd ? launch_stream<T, LPH, UNIT, INTER, true, true>(p, grid) : launch_stream<T, LPH, UNIT, INTER, true, false>(p, grid);
  else bwd ? launch_stream<T, LPH, UNIT, INTER, false, true>(p, grid) : launch_stream<T, LPH, UNIT, INTER, false, false>(p, grid);
}

template <typename T, int LPH>
void pick_stream_unit(const StreamParams& p, int grid, bool inter, bool norm, bool bwd) {
  if (inter) pick_stream_mode<T, LPH, 8, true>(p, grid, norm, bwd);
  else if (p.r % 16 == 0) pick_stream_mode<T, LPH, 8, false>(p, grid, norm, bwd);
  else pick_stream_mode<T, LPH, 4, false>(p, grid, norm, bwd);
}

template <typename T>
void pick_stream(const StreamParams& p, int grid, bool inter, bool norm, bool bwd) {
  switch (lanes_per_head(p.d, 8)) {
    case 1: case 2: case 4: return pick_stream_unit<T, 4>(p, grid, inter, norm, bwd);
    case 8: return pick_stream_unit<T, 8>(p, grid, inter, norm, bwd);
    case 16: return pick_stream_unit<T, 16>(p, grid, inter, norm, bwd);
    default: return pick_stream_unit<T, 32>(p, grid, inter, norm, bwd);
  }
}

// Dense tensors with 16-byte rows are streamed from a number of heads up, below which the rings' start costs more than the
// loads that they hide.  Direct / streamed in us, groups of 4 + 2 whole heads of 64 / 128 / 256 / 512 channels, calls back to back:
//   norm forward   24576 heads  bf16 3.0/3.8  4.4/5.0    7.2/7.4    10.9/10.4   fp32 3.7/4.6  5.9/5.6    9.3/8.7    16.7/17.6
//                  49152             4.5/4.6  7.1/7.3   11.6/10.8   25.1/21.8        5.5/5.5  9.6/8.4   17.2/17.6   34.4/34.5
//                  98304             7.2/6.7 11.5/10.5  27.1/22.2   54.2/39.1        9.0/8.2 17.3/17.0  35.4/34.8   66.5/69.8
//   norm backward  12288             5.2/6.4  7.3/6.8   10.1/9.2    16.6/12.2        5.3/6.6  7.5/8.1   10.6/11.0   18.5/16.2
//                  24576             7.1/7.1  9.7/9.0   15.7/11.8   25.8/17.9        7.2/7.9 10.5/10.3  16.7/15.5   32.9/30.8
//                  49152             9.6/9.2 14.8/11.6  24.8/17.5   56.1/33.4       10.4/10.1 16.2/14.7  32.2/30.5   55.2/55.0
// The rotation alone crosses where the forward does.  Larger calls gain more in 16 bits (196608 heads of 128: 26.9/21.6 and
// 56.1/32.8) and nothing or less in fp32 (of 512: 131.5/140.6 and 190.7/216.4).  They are streamed at any size where
// r = 8 mod 16, which the direct kernel would take by single channels.
bool streams(const HeadParams& p, Access a, const at::Tensor& t, const at::Tensor& other) {
  const long long heads = p.tokens * p.G * p.S, from = other.defined() ? 24576 : 49152;  // (other: the norm's backward)
  return (a.direct ? heads >= from : a.stream) && t.is_contiguous() &&
         (!other.defined() || other.is_contiguous());
}

StreamParams stream_params(const HeadParams& p, int esize, bool two) {
  StreamParams q{};
  q.x = p.x;
  q.dy = p.dy;
  q.out = p.out;
  q.cosv = p.cosv;
  q.sinv = p.sinv;
  q.w[0] = p.w[0];
  q.w[1] = p.w[1];
  q.err = device_err_flag(kErrHeads);
  q.per_token = fast_div((unsigned)(p.G * p.S));
  q.slots = fast_div((unsigned)p.S);
  q.rows = fast_div(p.tb ? 1u : (unsigned)p.B);
  q.per_row = (unsigned)(p.G * p.S) * q.rows.d;
  q.d = p.d;
  q.r = p.r;
  q.nq = p.n[0];
  q.nk = p.n[1];
  q.eps = p.eps;
  q.inv_d = 1.f / (float)p.d;
  q.heads = (unsigned)(p.tokens * p.G * p.S);
  const unsigned hpw = 32u / std::max(4, lanes_per_head(p.d, 8));
  // A tile: as many heads as fit, or whole groups where that takes fewer rounds a head (values then cost none)
  const unsigned fit = tile_bytes(two) / (unsigned)(p.d * esize), turned = (unsigned)(p.n[0] + p.n[1]);
  q.turned = fast_div(std::max(1u, turned));
  q.tile_heads = std::max(hpw, fit / hpw * hpw);
  double best = 0.95 / hpw;
  for (unsigned g = 1; turned > 0 && g * p.S <= fit; ++g) {
    const double rounds = (double)((g * turned + hpw - 1) / hpw) / (g * p.S);
    if (rounds <= best) {
      best = rounds;
      q.whole = 1;
      q.tile_heads = g * p.S;
    }
  }
  q.tiles = (q.heads + q.tile_heads - 1) / q.tile_heads;
  return q;
}

int stream_grid(const StreamParams& q, int ctas_per_sm) {
  return (int)std::min<long long>((q.tiles + kStreamWarps - 1) / kStreamWarps, (long long)num_sms() * ctas_per_sm);
}

template <typename F>
void by_type(at::ScalarType t, F f) {
  if (t == at::kBFloat16) f(__nv_bfloat16{});
  else if (t == at::kHalf) f(__half{});
  else if (t == at::kFloat) f(float{});
  else TORCH_CHECK(false, "qkv must be bf16, fp16 or fp32");
}

constexpr int kHeadWaves = 8;  // blocks an SM of the direct kernel, at most

void check_weights(const c10::optional<at::Tensor>& w, const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(w.has_value() && w->scalar_type() == t.scalar_type() && w->dim() == 1 && w->size(0) == t.size(4), name,
                    " must be [d] of qkv's type");
  TORCH_CHECK(w->is_cuda() && w->device() == t.device() && w->is_contiguous(), name,
              " must be contiguous and on the device of qkv");
}

}  // namespace

at::Tensor heads_fwd(at::Tensor qkv, at::Tensor cosv, at::Tensor sinv, int64_t nq, int64_t nk, bool interleaved,
                     c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk, double eps) {
  TORCH_CHECK(qkv.is_cuda(), "qkv must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(qkv.device());
  HeadParams p{};
  const bool norm = wq.has_value();
  Access vec = set_up(p, qkv, cosv, sinv, nq, nk);
  auto x = inner_contiguous(qkv);
  if (norm) {
    check_weights(wq, x, "q_weight");
    check_weights(wk, x, "k_weight");
    p.w[0] = wq->data_ptr();
    p.w[1] = wk->data_ptr();
    vec.need((uintptr_t)p.w[0] % 16 == 0 && (uintptr_t)p.w[1] % 16 == 0);
  }
  auto out = new_empty(x.sizes(), x, x.scalar_type());
  if (out.numel() == 0) return out;
  p.x = x.data_ptr();
  p.xs = x.stride(0);
  p.xb = x.stride(1);
  p.out = out.data_ptr();
  p.eps = (float)eps;
  vec.need(rows_aligned(x));
  if (streams(p, vec, x, at::Tensor())) {
    const StreamParams q = stream_params(p, (int)x.element_size(), false);
    by_type(x.scalar_type(), [&](auto t) { pick_stream<decltype(t)>(q, stream_grid(q, 2), interleaved, norm, false); });
    EMB_LAUNCH_CHECK();
    count_launch();
    return out;
  }
  const int grid = split_grid(p, vec.direct, kHeadWaves);
  by_type(x.scalar_type(), [&](auto t) { pick_shape<decltype(t)>(p, grid, vec.direct, interleaved, norm, false); });
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
  Access vec = set_up(p, dy, cosv, sinv, nq, nk);
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
    vec.need(rows_aligned(x) && (uintptr_t)p.w[0] % 16 == 0 && (uintptr_t)p.w[1] % 16 == 0);
  }
  auto dx = new_empty(g.sizes(), g, g.scalar_type());
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
        res.push_back(new_empty({p.d}, g, g.scalar_type()));
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
  vec.need(rows_aligned(g));
  const bool stream = streams(p, vec, g, x);
  StreamParams q{};
  if (stream) q = stream_params(p, (int)g.element_size(), norm);
  const int grid = stream ? stream_grid(q, 2) : split_grid(p, vec.direct, kHeadWaves);
  const int nb0 = stream ? grid : p.block0[1], nb1 = stream ? grid : p.block0[2] - p.block0[1];
  at::Tensor part;
  if (norm) {
    part = new_empty({nb0 + nb1, p.d}, g, at::kFloat);
    p.part = q.part = part.data_ptr<float>();
  }
  const bool same = acc[0] && acc[1] && acc[0] < acc[1] + p.d && acc[1] < acc[0] + p.d;
  const int joins = !norm ? 0 : same ? 2 : 1;
  by_type(g.scalar_type(), [&](auto t) {
    using T = decltype(t);
    if (stream) pick_stream<T>(q, grid, interleaved, norm, true);
    else pick_shape<T>(p, grid, vec.direct, interleaved, norm, true);
    if (norm) {
      // one launch for both classes, or one after the other where they add to the same words (one weight for both)
      for (int c = 0; c < joins; ++c)
        launch_early(heads_join_kernel<T>, dim3((p.d + 7) / 8, joins == 2 ? 1 : 2), 1024, 0, p.part, p.d, nb0, nb1,
                     (int)stream, c, (T*)dw[0], (T*)dw[1], acc[0], acc[1]);
    }
  });
  EMB_LAUNCH_CHECK();
  count_launch(1 + joins);
  return res;
}

int64_t heads_error_flag() {
  int v = 0;
  EMB_CUDA_CHECK(cudaMemcpy(&v, device_err_flag(kErrHeads), sizeof(int), cudaMemcpyDeviceToHost));
  return v;
}

}  // namespace emb
