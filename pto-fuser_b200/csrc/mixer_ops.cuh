// Shared device helpers of the operators around a recurrent token mixer (short_conv.cu,
// ssm_scan.cu, rms_norm.cu): element loads, the two activations and slot handling.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"

namespace ptof {

template <typename T>
struct Elem;
template <>
struct Elem<float> { static constexpr int code = PTOF_F32; };
template <>
struct Elem<__half> { static constexpr int code = PTOF_F16; };
template <>
struct Elem<__nv_bfloat16> { static constexpr int code = PTOF_BF16; };

// VEC elements of T as one register block: loads and stores are 16 bytes wide where the
// block is (VEC * sizeof(T) == 16; the address must then be 16-byte aligned), 32 bytes in
// two halves, 8 bytes, or element by element for VEC = 1.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> ld_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void st_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}

// e^v and 1/v to about 2 ulp (one special-function instruction each).
__device__ __forceinline__ float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fast_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 values in one 64-bit register pair, and their products and fused products in one
// instruction each.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float x, float y) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// v * sigmoid(v) = v / (1 + exp(-v)). Where exp(-v) passes 2^126 (v < -87.3) the quotient is
// zero; the true value is below |v| 2^-126 there.
__device__ __forceinline__ float silu_f32(float v) {
  return v * fast_rcp(1.f + fast_exp2(-kLog2e * v));
}

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1]. log1p(e) = e P(e) with P of
// degree 8, fitted on [0, 1] for the smallest relative error (Remez exchange): 6.4e-8 with the
// coefficients as they are rounded here, in fp32 arithmetic 1.8e-7. No step cancels, so small results (very negative v) keep their
// relative accuracy, and only the exponential needs a special-function instruction.
__device__ constexpr float kLog1p[9] = {0.99999997f,  -0.49999493f, 0.33319097f,
                                        -0.24842982f, 0.19106005f,  -0.13663240f,
                                        0.078225869f, -0.029505181f, 0.0052326787f};
__device__ __forceinline__ float softplus_f32(float v) {
  const float e = fast_exp2(-kLog2e * fabsf(v));
  float p = kLog1p[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fmaf(p, e, kLog1p[i]);
  return fmaf(p, e, fmaxf(v, 0.f));  // NaN comes through e
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The two activations on two values at once.
__device__ __forceinline__ f32x2 silu2(f32x2 v) {
  const float2 u = unpack2(mul2(v, pack2(-kLog2e, -kLog2e)));
  const float2 s = unpack2(add2(pack2(fast_exp2(u.x), fast_exp2(u.y)), pack2(1.f, 1.f)));
  return mul2(v, pack2(fast_rcp(s.x), fast_rcp(s.y)));
}
__device__ __forceinline__ f32x2 softplus2(f32x2 v) {
  const float2 w = unpack2(v);
  const float2 u = unpack2(mul2(pack2(fabsf(w.x), fabsf(w.y)), pack2(-kLog2e, -kLog2e)));
  const f32x2 e = pack2(fast_exp2(u.x), fast_exp2(u.y));
  f32x2 p = pack2(kLog1p[8], kLog1p[8]);
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fma2(p, e, pack2(kLog1p[i], kLog1p[i]));
  return fma2(p, e, pack2(fmaxf(w.x, 0.f), fmaxf(w.y, 0.f)));
}

// Copies of BYTES (4, 8 or 16, both addresses aligned to it) that land without a register. The
// clobber keeps reads of what the place held before them, in program order.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* smem, const void* gmem) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(gmem) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(gmem), "n"(BYTES) : "memory");
}

// Bounds of sequence n of a packed batch, kept inside [0, T] whatever cu holds.
__device__ __forceinline__ void seq_bounds(const int* cu, int n, int T, int& s, int& e) {
  s = min(max(cu[n], 0), T);
  e = min(max(cu[n + 1], s), T);
}

// Where rows of a single-token call share a state slot, the rows of one slot are applied
// in row order by the block that owns the first of them. For the block's row m with slot
// `slot` this says (block-wide) whether an earlier row has the slot (the block then has
// nothing to do) and whether a later one has. Every thread of the block calls it.
struct SlotUse {
  bool earlier, later;
};
__device__ __forceinline__ SlotUse slot_use(const int* slots, int M, int m, int slot) {
  bool e = false, l = false;
  for (int i = threadIdx.x; i < M; i += blockDim.x) {
    const bool same = slots[i] == slot;
    e |= same && i < m;
    l |= same && i > m;
  }
  SlotUse u{false, false};
  if (__syncthreads_or(e | l)) {  // slots are seldom shared: one barrier then
    u.earlier = __syncthreads_or(e);
    u.later = __syncthreads_or(l);
  }
  return u;
}

}  // namespace ptof
