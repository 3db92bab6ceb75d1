// AdamW over many tensors at once, states in 32 bits or in 8:
//
//   p <- p (1 - lr wd);  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2
//   p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// all in fp32.  The moments' products and sums are rounded one by one (no contraction), so the
// 8-bit codes do not depend on how a compiler fuses; the root and the quotient of the update are
// the MUFU unit's (2 units in the last place each, on an update that is itself a small part of p):
// with a correctly rounded quotient the 8-bit step was bound by issue, not by HBM.  The MUFU root
// takes a v below 2^-126 as 0; where eps is so small that this would show, a kernel of its own (SMALL_EPS)
// takes the rounded root: a branch in the usual one costs it 6 %.  What is coded is the correctly
// rounded root.  16-bit weights are the rounded copy of an fp32 master.
//
// The states of all tensors lie in flat buffers, each tensor beginning at a multiple of kBlock
// elements.  8 bits: a block of kBlock values of m, and of u = sqrt(v), is stored as e4m3 codes
// of value / scale with scale = max|value| / 448 in fp32.  e4m3 keeps 4 bits over 2^-9 .. 448,
// and the root doubles the range in v to 2^35; a u that is not 0 is never stored as 0, since a
// step would divide by it.
//
// Bound by HBM: 28 bytes an element (32-bit states; fp32 weights, or 16-bit with their master),
// 16 with 8-bit states.  67M bf16 weights with 32-bit states: 274 us, 6.9 TB/s; 403M with 8-bit
// states: 1126 us, 5.7 TB/s (88 % of the measured copy rate; 64 registers a thread hold two blocks of
// a warp, 32 warps an SM; with 28 warps 1180 us, with 40, which spill, 1363); there instruction issue
// (79 %) is as near its limit as HBM.
//
// One warp takes a block at a time, lane l elements 4 l .. 4 l + 3 and 128 + 4 l .. + 3, so every
// load and store of a warp is one contiguous run, 16 bytes a lane in fp32, and the block's maxima
// are warp shuffles.  One launch takes up to kMost tensors: their
// addresses travel in the kernel's parameters, so no table is copied to the device and the
// launch can be captured.  A CTA finds its tensor by a binary search over the first chunks.
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "abi.h"
#include "common.cuh"

namespace hi3d {
namespace adamw {

constexpr int kBlock = HI3D_ADAMW_BLOCK;
// Warps of a CTA: 403M bf16 weights with 8-bit states, two 1131 us, four 1126, eight 1153.
constexpr int kWarps = 4;
constexpr int kCtas8 = 8;  // CTAs an SM holds with 8-bit states (at most 64 registers)
// Elements of a CTA: a block a warp, with 8-bit states two, the second of which is loaded while the
// first is computed.  (8 bits, eight warps: one 1261 us, two 1145, three 1197, four 1208; 32 bits,
// 67M weights: one 273, two 278, four 281.)
template <bool EIGHT>
constexpr int kChunk = (EIGHT ? 2 : 1) * kWarps * kBlock;

struct Entry {
  void* p;
  const void* g;
  int64_t n;
  uint32_t at;     // offset in the flat states, in blocks
  uint32_t chunk;  // first CTA
};

template <int MOST>
struct Table {
  Entry e[MOST];
};

struct Params {
  int count;
  float* master;
  void* m;
  void* v;
  float* scale_m;
  float* scale_u;
  const float* grad_scale;  // optional
  float b1, b1c, b2, b2c, decay, step, root, eps;
};

// 4 consecutive values as they lie in memory
template <typename T>
struct Four {  // 16-bit types
  uint2 u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    f2_unpack(Cvt<T>::to_f2(u.x), v[0], v[1]);
    f2_unpack(Cvt<T>::to_f2(u.y), v[2], v[3]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(Cvt<T>::pack2(v[0], v[1]), Cvt<T>::pack2(v[2], v[3]));
  }
};
template <>
struct Four<float> {
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
struct Codes {
  uint32_t u;
  __device__ __forceinline__ void load(const uint8_t* p) { u = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const;
};

template <typename T>
__device__ __forceinline__ float one(T v) {
  return Cvt<T>::to_f(v);
}
template <>
__device__ __forceinline__ float one<float>(float v) {
  return v;
}
template <typename T>
__device__ __forceinline__ T back(float v) {
  return Cvt<T>::from_f(v);
}
template <>
__device__ __forceinline__ float back<float>(float v) {
  return v;
}

__device__ __forceinline__ void decode4(uint32_t c, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h;
    const uint16_t two = (uint16_t)(c >> (16 * i));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void Codes::get(float (&v)[4]) const { decode4(u, v); }
__device__ __forceinline__ uint32_t encode4(const float (&v)[4]) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1]), "f"(v[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3]), "f"(v[2]));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// sqrt(x) to 2 units in the last place; 0 for x below 2^-126
__device__ __forceinline__ float root_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <bool SMALL_EPS>
__device__ __forceinline__ void update(const Params& a, float gs, float& p, float g, float& m, float& v) {
  g = __fmul_rn(g, gs);
  m = __fadd_rn(__fmul_rn(m, a.b1), __fmul_rn(g, a.b1c));
  v = __fadd_rn(__fmul_rn(v, a.b2), __fmul_rn(__fmul_rn(g, g), a.b2c));
  const float den = __fadd_rn(__fmul_rn(SMALL_EPS ? __fsqrt_rn(v) : root_approx(v), a.root), a.eps);
  p = __fsub_rn(__fmul_rn(p, a.decay), __fmul_rn(__fdividef(m, den), a.step));
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// 1 / scale, or 0 where the block holds nothing that it could scale (all zero, or below 2^-111)
__device__ __forceinline__ float inverse(float scale) { return scale >= 0x1p-120f ? __frcp_rn(scale) : 0.f; }

// One block of a tensor's values as a lane holds them.
template <typename P, bool EIGHT>
struct Block {
  using State = typename std::conditional<EIGHT, uint8_t, float>::type;
  Four<P> g[2];
  Four<float> w[2];  // the fp32 weights: the tensor's own or the master's
  typename std::conditional<EIGHT, Codes, Four<float>>::type m[2], v[2];
  float sm, su;

  // i: the lane's first element in the tensor, f: in the flat states
  __device__ __forceinline__ void load(const Params& a, const P* p, const P* gr, int64_t i, int64_t f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      g[h].load(gr + i + h * 128);
      if constexpr (sizeof(P) == 4)
        w[h].load(p + i + h * 128);
      else
        w[h].load(a.master + f + h * 128);
    }
    load_state(a, f);
  }
  __device__ __forceinline__ void load_state(const Params& a, int64_t f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h].load(static_cast<const State*>(a.m) + f + h * 128);
      v[h].load(static_cast<const State*>(a.v) + f + h * 128);
    }
    if constexpr (EIGHT) sm = a.scale_m[f / kBlock], su = a.scale_u[f / kBlock];
  }
};

// New moments of four values in m and v (8 bits: v comes in as its root's codes) and weights in w.
template <bool EIGHT, bool SMALL_EPS>
__device__ __forceinline__ void update4(const Params& a, float gs, float sm, float su, const float (&g)[4],
                                        float (&w)[4], float (&m)[4], float (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (EIGHT) {
      m[k] = __fmul_rn(m[k], sm);
      const float u = __fmul_rn(v[k], su);
      v[k] = __fmul_rn(u, u);
    }
    update<SMALL_EPS>(a, gs, w[k], g[k], m[k], v[k]);
  }
}

// The states of a block whose lane holds m and v, written with their scales.  The root is taken
// again, correctly rounded: beside the middle of two codes the MUFU unit's would get the other one,
// a sixteenth of the value, once in 3 million values.
__device__ __forceinline__ void store_codes(const Params& a, int64_t f, float (&m)[2][4], float (&v)[2][4]) {
  float big_m = 0.f, big_v = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int k = 0; k < 4; ++k) big_m = fmaxf(big_m, fabsf(m[h][k])), big_v = fmaxf(big_v, v[h][k]);
  const float sm = __fmul_rn(warp_max(big_m), 1.0f / 448.0f);
  const float su = __fmul_rn(__fsqrt_rn(warp_max(big_v)), 1.0f / 448.0f);
  const float im = inverse(sm), iu = inverse(su);
  if (lane_id() == 0) a.scale_m[f / kBlock] = sm, a.scale_u[f / kBlock] = su;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int k = 0; k < 4; ++k) m[h][k] = __fmul_rn(m[h][k], im);
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + f + h * 128) = encode4(m[h]);
    float c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = __fmul_rn(__fsqrt_rn(v[h][k]), iu);
      if (v[h][k] > 0.f && iu > 0.f) c[k] = fmaxf(c[k], 0x1p-9f);
    }
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + f + h * 128) = encode4(c);
  }
}

// A whole block of an aligned tensor.
template <typename P, bool EIGHT, bool SMALL_EPS>
__device__ __forceinline__ void whole_block(const Params& a, float gs, P* p, int64_t i, int64_t f,
                                            const Block<P, EIGHT>& b) {
  float m[2][4], v[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float w[4], g[4];
    b.g[h].get(g);
    b.w[h].get(w);
    b.m[h].get(m[h]);
    b.v[h].get(v[h]);
    update4<EIGHT, SMALL_EPS>(a, gs, b.sm, b.su, g, w, m[h], v[h]);
    Four<P>::store(p + i + h * 128, w);
    if constexpr (sizeof(P) == 2) Four<float>::store(a.master + f + h * 128, w);
    if constexpr (!EIGHT) {
      Four<float>::store(static_cast<float*>(a.m) + f + h * 128, m[h]);
      Four<float>::store(static_cast<float*>(a.v) + f + h * 128, v[h]);
    }
  }
  if constexpr (EIGHT) store_codes(a, f, m, v);
}

// A tensor's ragged last block, or any of one that vectors cannot address: weights and gradients
// one by one.  The flat buffers are padded to whole blocks; the padding stays 0.
template <typename P, bool EIGHT, bool SMALL_EPS>
__device__ __noinline__ void odd_block(const Params& a, float gs, P* p, const P* gr, int64_t n, int64_t i, int64_t f) {
  Block<P, EIGHT> b;
  b.load_state(a, f);
  float m[2][4], v[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float w[4], g[4];
    const int64_t at = i + h * 128;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = at + k < n;
      g[k] = in ? one<P>(gr[at + k]) : 0.f;
      if constexpr (sizeof(P) == 4)
        w[k] = in ? one<P>(p[at + k]) : 0.f;
      else
        w[k] = a.master[f + h * 128 + k];
    }
    b.m[h].get(m[h]);
    b.v[h].get(v[h]);
    update4<EIGHT, SMALL_EPS>(a, gs, b.sm, b.su, g, w, m[h], v[h]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (at + k < n) {
        p[at + k] = back<P>(w[k]);
        if constexpr (sizeof(P) == 2) a.master[f + h * 128 + k] = w[k];
      } else {
        m[h][k] = v[h][k] = 0.f;
      }
    }
    if constexpr (!EIGHT) {
      Four<float>::store(static_cast<float*>(a.m) + f + h * 128, m[h]);
      Four<float>::store(static_cast<float*>(a.v) + f + h * 128, v[h]);
    }
  }
  if constexpr (EIGHT) store_codes(a, f, m, v);
}

template <typename P, bool EIGHT, int MOST, bool SMALL_EPS>
__global__ void __launch_bounds__(kWarps * 32, EIGHT ? kCtas8 : 1)
    adamw_kernel(const __grid_constant__ Table<MOST> table, const __grid_constant__ Params a) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.e[mid].chunk <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Entry& e = table.e[lo];
  P* p = static_cast<P*>(e.p);
  const P* g = static_cast<const P*>(e.g);
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  const bool wide = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & (4 * sizeof(P) - 1)) == 0;
  constexpr int kStep = kWarps * kBlock;
  const int64_t first = (int64_t)(blockIdx.x - e.chunk) * kChunk<EIGHT>, n = e.n;
  int64_t at = first + warp_id() * kBlock;
  const int64_t end = min(first + kChunk<EIGHT>, n);
  const int64_t fast = wide ? end - kBlock : at - 1;  // whole blocks begin up to here
  const int64_t lane4 = lane_id() * 4, flat = (int64_t)e.at * kBlock + lane4;
  if constexpr (EIGHT) {
    // the next block's values are on their way while this one is computed: its scales wait for
    // two warp maxima
    Block<P, EIGHT> b;
    if (at <= fast) b.load(a, p, g, at + lane4, flat + at);
    for (; at <= fast; at += kStep) {
      const Block<P, EIGHT> now = b;
      if (at + kStep <= fast) b.load(a, p, g, at + kStep + lane4, flat + at + kStep);
      whole_block<P, EIGHT, SMALL_EPS>(a, gs, p, at + lane4, flat + at, now);
    }
  } else {
    for (; at <= fast; at += kStep) {
      Block<P, EIGHT> b;
      b.load(a, p, g, at + lane4, flat + at);
      whole_block<P, EIGHT, SMALL_EPS>(a, gs, p, at + lane4, flat + at, b);
    }
  }
  for (; at < end; at += kStep) odd_block<P, EIGHT, SMALL_EPS>(a, gs, p, g, n, at + lane4, flat + at);
}

// Tables of two sizes: the parameters of a launch are copied with it, 2 KB for the usual handful
// of tensors, 24 KB for a model's hundreds (12 tensors of 9216: a step takes 53 us on the host, with
// the large table 56).
constexpr int kFew = 64, kMost = 768;

template <typename P, bool EIGHT, int MOST, bool SMALL_EPS>
static int launch(const hi3d_adamw_args* a, const Params& base, int from, int count, cudaStream_t st) {
  Table<MOST> t;
  Params p = base;
  p.count = 0;
  uint64_t chunks = 0;
  for (int i = from; i < from + count; ++i) {
    if (a->numels[i] == 0) continue;
    Entry& e = t.e[p.count++];
    e.p = a->params[i], e.g = a->grads[i], e.n = a->numels[i];
    e.at = (uint32_t)(a->offsets[i] / kBlock);
    e.chunk = (uint32_t)chunks;
    chunks += (uint64_t)((a->numels[i] + kChunk<EIGHT> - 1) / kChunk<EIGHT>);
    if (chunks > 0x7fffffffu) return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: too many elements");
  }
  if (p.count == 0) return HI3D_OK;
  adamw_kernel<P, EIGHT, MOST, SMALL_EPS><<<(unsigned)chunks, kWarps * 32, 0, st>>>(t, p);
  return check_launch("adamw_step");
}

template <typename P, bool EIGHT>
static int run(const hi3d_adamw_args* a, const Params& p, cudaStream_t st) {
  // whether the root of a v below 2^-126, at most 2^-63, is more than half a unit in the last place of eps
  // (eps 1e-8: not while 1 - beta2^step is above 1.4e-7)
  const bool small_eps = !(a->eps * 0x1p-25 >= p.root * 0x1p-63);
  for (int from = 0; from < a->count; from += kMost) {
    const int count = a->count - from < kMost ? a->count - from : kMost;
    const int rc = small_eps       ? launch<P, EIGHT, kMost, true>(a, p, from, count, st)
                   : count <= kFew ? launch<P, EIGHT, kFew, false>(a, p, from, count, st)
                                   : launch<P, EIGHT, kMost, false>(a, p, from, count, st);
    if (rc) return rc;
  }
  return HI3D_OK;
}

// Whether two tensors' states share a block: two CTAs would write it.
static bool overlap(const hi3d_adamw_args* a) {
  int* by_offset = static_cast<int*>(malloc(sizeof(int) * a->count));
  if (!by_offset) return true;
  int n = 0;
  for (int i = 0; i < a->count; ++i)
    if (a->numels[i] > 0) by_offset[n++] = i;
  std::sort(by_offset, by_offset + n, [a](int x, int y) { return a->offsets[x] < a->offsets[y]; });
  bool shared = false;
  for (int i = 1; i < n && !shared; ++i) {
    const int64_t blocks = (a->numels[by_offset[i - 1]] + kBlock - 1) / kBlock;
    shared = a->offsets[by_offset[i]] < a->offsets[by_offset[i - 1]] + blocks * kBlock;
  }
  free(by_offset);
  return shared;
}

}  // namespace adamw
}  // namespace hi3d

using namespace hi3d;

extern "C" int hi3d_adamw_step(const hi3d_adamw_args* a, void* stream) {
  using namespace adamw;
  if (!a || a->count < 0) return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: null arguments");
  if (a->count == 0) return HI3D_OK;
  if (!a->params || !a->grads || !a->numels || !a->offsets || !a->exp_avg || !a->exp_avg_sq)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: null pointer");
  if (a->dtype != HI3D_F16 && a->dtype != HI3D_BF16 && a->dtype != HI3D_F32)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: dtype must be f16, bf16 or f32");
  if (a->state_bits != 8 && a->state_bits != 32)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: state_bits must be 8 or 32");
  if ((a->dtype != HI3D_F32) != (a->master != nullptr))
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: 16-bit weights need a master, 32-bit ones have none");
  if ((a->state_bits == 8) != (a->scales != nullptr))
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: 8-bit states need scales, 32-bit ones have none");
  if (!aligned16(a->master) || !aligned16(a->exp_avg) || !aligned16(a->exp_avg_sq))
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: state buffers must be 16-byte aligned");
  if (a->step < 1 || !(a->beta1 >= 0 && a->beta1 < 1) || !(a->beta2 >= 0 && a->beta2 < 1) || !(a->eps >= 0) ||
      !(a->lr >= 0) || !(a->weight_decay >= 0))
    return set_error(HI3D_ERR_INVALID_ARGUMENT,
                     "adamw_step: step >= 1, betas in [0, 1), lr, eps and weight_decay not negative");
  if (a->total < 0 || a->total % kBlock || a->total / kBlock > 0xffffffffll)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: %lld state elements, not a multiple of %d",
                     (long long)a->total, kBlock);
  const int size = a->dtype == HI3D_F32 ? 4 : 2;
  int64_t end = 0;  // of the states so far, while they come in order
  bool ordered = true;
  for (int i = 0; i < a->count; ++i) {
    const int64_t n = a->numels[i], at = a->offsets[i];
    if (n < 0 || at < 0 || at % kBlock || at > a->total || n > a->total - at)
      return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: tensor %d (%lld elements at %lld) outside the states",
                       i, (long long)n, (long long)at);
    const uintptr_t p = reinterpret_cast<uintptr_t>(a->params[i]), g = reinterpret_cast<uintptr_t>(a->grads[i]);
    if (n > 0 && (!p || !g || (p | g) % size))
      return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: tensor %d: null or misaligned pointer", i);
    if (n == 0) continue;
    ordered = ordered && at >= end;
    end = at + (n + kBlock - 1) / kBlock * kBlock;
  }
  if (!ordered && overlap(a))
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "adamw_step: two tensors share state");
  Params p;
  p.count = 0;
  p.master = a->master, p.m = a->exp_avg, p.v = a->exp_avg_sq;
  p.scale_m = a->scales, p.scale_u = a->scales ? a->scales + a->total / kBlock : nullptr;
  p.grad_scale = a->grad_scale;
  p.b1 = (float)a->beta1, p.b1c = (float)(1 - a->beta1), p.b2 = (float)a->beta2, p.b2c = (float)(1 - a->beta2);
  p.decay = (float)(1 - a->lr * a->weight_decay);
  p.step = (float)(a->lr / (1 - pow(a->beta1, (double)a->step)));
  p.root = (float)pow(1 - pow(a->beta2, (double)a->step), -0.5);
  p.eps = (float)a->eps;
  cudaStream_t st = as_stream(stream);
  const bool eight = a->state_bits == 8;
  switch (a->dtype) {
    case HI3D_F32: return eight ? run<float, true>(a, p, st) : run<float, false>(a, p, st);
    case HI3D_F16: return eight ? run<__half, true>(a, p, st) : run<__half, false>(a, p, st);
    default: return eight ? run<__nv_bfloat16, true>(a, p, st) : run<__nv_bfloat16, false>(a, p, st);
  }
}
