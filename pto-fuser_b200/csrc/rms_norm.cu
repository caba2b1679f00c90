// Root-mean-square norm with the residual's addition and an optional output in 8 bits:
//   h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight
// h is summed and normed in fp32 and returned rounded to the residual's type. The 8-bit form
// returns q = y / scale in e4m3 with scale = max(amax |y| / 448, 2^-126), amax over the row or
// over each `group` columns (the last group of a row may be shorter): the floor keeps 1 / scale
// finite and gives rows of zeros the value zero.
//
// Bound by memory: x and the residual are read once, the sum, y and the scales written once.
// TPR threads hold a row in registers between the sum of squares and the output; the
// partial sums meet in shuffles and, above one warp, in shared memory. Two blocks an SM at
// least, where the registers leave room: one block of 1024 threads took 121 us for 4096 x 16384
// bf16 where two of 512 took 80. Rows of more than 2048 16-byte vectors take one of 1024 all the
// same: 4096 x 16384 fp32 177 us, where its bytes need 166.
//
// With a residual, inputs changing between calls, us (what the bytes need at the copy bandwidth
// in brackets; some of what is written last is still in L2 when a kernel ends): bf16
// 16384 x 8192 to e4m3 with a scale for 128 columns 147 (146), 4096 x 16384 84 (83). Rows that
// begin on no 16 bytes: 3001 x 5003 f16 with an fp32 residual 34 (28), kernel alone 30; 45 element
// by element. Such rows to e4m3 with a scale a group go element by element, bound by
// instructions: 4096 x 5001 takes 54 where 5000 columns take 35.
#include <cuda_fp8.h>

#include "capi_internal.h"
#include "mixer_ops.cuh"

namespace ptof {

namespace {

struct NormArgs {
  const void* x;
  const void* res;
  const void* w;
  void* y;
  void* sum;
  float* scale;
  int64_t x_rs, res_rs, y_rs, sum_rs;
  int64_t rows;
  int D, group, groups;  // columns, columns of a scale (2^shift), scales of a row
  int shift;
  int w_dtype, phase;  // phase: index of x's first element modulo 4
  float eps, inv_d;
};

constexpr float kFp8Max = 448.f;        // largest finite e4m3 value
constexpr float kTinyScale = 1.17549435e-38f;  // 2^-126

// max of three, or of two, that keeps a NaN of any side
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Codes are those of y / s rounded once, with the scale s that is returned; products with an
// approximate reciprocal give some of them the neighbouring e4m3 value. (s itself is a product with
// the rounded 1 / 448, off by one more half unit than the quotient, as torch's division of a tensor
// on the device by a number is.) With r within a unit in the last place of 1 / s, q = y r is off by
// two units at most, and adding r times the remainder y - q s of a fused product rounds to y / s
// (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990),
// or, with r not correctly rounded, to its neighbour where y / s lies within 2^-22 units of the
// middle between two values. That is two instructions a value more than the product alone:
// 16384 x 8192 to e4m3 with a scale for 128 columns takes 147 us, with the product 144, with the
// library's reciprocal and division 158. 7.4 of a million codes are not those of 64-bit
// arithmetic (the row's root, rounded), with the product 8.0.
constexpr float kLargest = 3.40282347e38f;  // largest finite fp32 value

// Scale and quotients of the values whose largest magnitude is amax.
struct Scale {
  float s, r, minus_s;
  // y / s. An infinite scale has no remainder: 0 for finite y. A quotient of zero is +0.
  __device__ __forceinline__ float quotient(float y) const {
    const float q = y * r;
    return fmaf(fmaf(q, minus_s, y), r, q);
  }
  __device__ __forceinline__ float2 quotient(f32x2 y) const {
    const f32x2 r2 = pack2(r, r), q = mul2(y, r2);
    return unpack2(fma2(fma2(q, pack2(minus_s, minus_s), y), r2, q));
  }
};
__device__ __forceinline__ Scale scale_of(float amax) {
  Scale o;
  o.s = max_nan(amax * (1.f / kFp8Max), kTinyScale);
  o.r = fast_rcp(o.s);  // s is a normal number, its reciprocal at most 2^126
  o.minus_s = o.s <= kLargest ? -o.s : 0.f;
  return o;
}

// Sum (MAX = false) or NaN-keeping maximum over the TPR threads of a row, on every thread.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int off = W / 2; off >= 1; off /= 2) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = MAX ? max_nan(v, o) : v + o;
  }
  if (TPR <= 32) return v;
  constexpr int NW = TPR / 32;
  const int warp = threadIdx.x / 32;
  __syncthreads();  // an earlier reduction's readers are done
  if (threadIdx.x % 32 == 0) red[warp] = v;
  __syncthreads();
  const int first = warp / NW * NW;
  float r = red[first];
#pragma unroll
  for (int i = 1; i < NW; ++i) r = MAX ? max_nan(r, red[first + i]) : r + red[first + i];
  return r;
}

enum { kNoQuant = 0, kQuantRow = 1, kQuantGroup = 2 };

// VEC columns, given as pairs, rounded to T.
template <typename T, int VEC>
__device__ __forceinline__ void st_pairs(T* p, const f32x2 (&v)[VEC / 2]) {
  Pack<T, VEC> o;
#pragma unroll
  for (int k = 0; k < VEC / 2; ++k) {
    const float2 u = unpack2(v[k]);
    o.v[2 * k] = from_f32<T>(u.x);
    o.v[2 * k + 1] = from_f32<T>(u.y);
  }
  st_pack<T, VEC>(p, o);
}

constexpr int threads_of(int TPR) { return TPR > 256 ? TPR : 256; }
// Blocks an SM that leave registers for `values` of a row a thread. At least two: while one
// waits for its row's sum, another reads or writes.
constexpr int blocks_of(int TPR, int values) {
  return (values <= 8 ? 1536 : values <= 24 || TPR > 256 ? 1024 : 768) / threads_of(TPR);
}

template <typename T, typename TR, int TPR, int NV, int QUANT, bool RES>
__global__ void __launch_bounds__(threads_of(TPR), TPR > 512 ? 1 : TPR > 256 ? 2 : 4) rms_norm_kernel(const NormArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int RPB = threads_of(TPR) / TPR;  // rows of a block
  __shared__ float red[32];
  const int64_t row_ = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool live = row_ < a.rows;
  const int64_t row = live ? row_ : a.rows - 1;  // barriers and shuffles need every thread
  const int tx = threadIdx.x % TPR;
  const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
  const TR* res = RES ? static_cast<const TR*>(a.res) + row * a.res_rs : nullptr;

  // the row as pairs of columns; zeros behind its end
  f32x2 h[NV][VEC / 2], ss2 = pack2(0.f, 0.f);
  {
    Pack<T, VEC> px[NV];
    Pack<TR, VEC> pr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + tx) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        px[i].v[k] = from_f32<T>(0.f);
        pr[i].v[k] = from_f32<TR>(0.f);
      }
      if (c < a.D) {
        px[i] = ld_pack<T, VEC>(x + c);
        if (RES) pr[i] = ld_pack<TR, VEC>(res + c);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < VEC; k += 2) {
        f32x2 v = pack2(to_f32<T>(px[i].v[k]), to_f32<T>(px[i].v[k + 1]));
        if (RES) v = add2(v, pack2(to_f32<TR>(pr[i].v[k]), to_f32<TR>(pr[i].v[k + 1])));
        h[i][k / 2] = v;
        ss2 = fma2(v, v, ss2);
      }
    }
  }
  if (RES) {
    TR* sum = static_cast<TR*>(a.sum) + row * a.sum_rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + tx) * VEC;
      if (live && c < a.D) st_pairs<TR, VEC>(sum + c, h[i]);
    }
  }
  const float2 sp = unpack2(ss2);
  const float ss = row_reduce<TPR, false>(sp.x + sp.y, red);
  const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
  const f32x2 r2 = pack2(r, r);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + tx) * VEC;
    if (c < a.D) {
      if (a.w_dtype == Elem<T>::code) {
        const Pack<T, VEC> w = ld_pack<T, VEC>(static_cast<const T*>(a.w) + c);
#pragma unroll
        for (int k = 0; k < VEC; k += 2)
          h[i][k / 2] = mul2(mul2(h[i][k / 2], r2), pack2(to_f32<T>(w.v[k]), to_f32<T>(w.v[k + 1])));
      } else {
        const Pack<float, VEC> w = ld_pack<float, VEC>(static_cast<const float*>(a.w) + c);
#pragma unroll
        for (int k = 0; k < VEC; k += 2)
          h[i][k / 2] = mul2(mul2(h[i][k / 2], r2), pack2(w.v[k], w.v[k + 1]));
      }
    }
    if (QUANT == kQuantRow) {
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 u = unpack2(h[i][k]);
        amax = max_nan(amax, fabsf(u.x), fabsf(u.y));
      }
    }
  }
  if (QUANT == kNoQuant) {
    T* y = static_cast<T*>(a.y) + row * a.y_rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + tx) * VEC;
      if (live && c < a.D) st_pairs<T, VEC>(y + c, h[i]);
    }
    return;
  }
  Scale by;
  if (QUANT == kQuantRow) {
    by = scale_of(row_reduce<TPR, true>(amax, red));
    if (live && tx == 0) a.scale[row] = by.s;
  }
  const int seg = a.group / VEC;  // threads of a group, a power of two up to a warp
  uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_rs;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + tx) * VEC;
    if (QUANT == kQuantGroup) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 u = unpack2(h[i][k]);
        m = max_nan(m, fabsf(u.x), fabsf(u.y));
      }
#pragma unroll
      for (int off = 1; off < 32; off *= 2)
        if (off < seg) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
      by = scale_of(m);
      if (live && c < a.D && tx % seg == 0) a.scale[row * a.groups + (c >> a.shift)] = by.s;
    }
    if (live && c < a.D) {
      Pack<uint16_t, VEC / 2> o;
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k)
        o.v[k] = __nv_cvt_float2_to_fp8x2(by.quotient(h[i][k]), __NV_SATFINITE, __NV_E4M3);
      st_pack<uint16_t, VEC / 2>(reinterpret_cast<uint16_t*>(y + c), o);
    }
  }
}


// Rows that do not begin on 16 bytes but lie alike: elements at one place of x, the residual,
// the sum and y have one index modulo 4, so vectors of 4 that are aligned in one are in all.
// A row's first vector begins `lead` columns before it. The vectors at the ends go by elements;
// every other one is loaded without a branch.
template <typename T, typename TR, int TPR, int NV, int QUANT, bool RES>
__global__ void __launch_bounds__(threads_of(TPR), blocks_of(TPR, 4 * NV)) rms_norm_shift_kernel(const NormArgs a) {
  constexpr int RPB = threads_of(TPR) / TPR;  // rows of a block
  __shared__ float red[32];
  const int64_t row_ = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool live = RPB == 1 || row_ < a.rows;
  const int64_t row = live ? row_ : a.rows - 1;  // barriers and shuffles need every thread
  const int tx = threadIdx.x % TPR, D = live ? a.D : 0;  // columns to write
  const int lead = static_cast<int>((a.phase + row * a.x_rs) & 3);
  const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
  const TR* res = RES ? static_cast<const TR*>(a.res) + row * a.res_rs : nullptr;
  TR* sum = RES ? static_cast<TR*>(a.sum) + row * a.sum_rs : nullptr;
  auto col = [&](int i) { return (i * TPR + tx) * 4 - lead; };
  auto whole = [&](int c) { return c >= 0 && c + 4 <= a.D; };
  auto in = [&](int c) { return c >= 0 && c < a.D; };

  f32x2 h[NV][2], ss2 = pack2(0.f, 0.f);
  {
    Pack<T, 4> px[NV];
    Pack<TR, 4> pr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = whole(col(i)) ? col(i) : 4 - lead;  // a row of 8 columns holds that one
      px[i] = ld_pack<T, 4>(x + c);
      if (RES) pr[i] = ld_pack<TR, 4>(res + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (!whole(c)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          px[i].v[k] = in(c + k) ? x[c + k] : from_f32<T>(0.f);
          if (RES) pr[i].v[k] = in(c + k) ? res[c + k] : from_f32<TR>(0.f);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        f32x2 v = pack2(to_f32<T>(px[i].v[k]), to_f32<T>(px[i].v[k + 1]));
        if (RES) v = add2(v, pack2(to_f32<TR>(pr[i].v[k]), to_f32<TR>(pr[i].v[k + 1])));
        h[i][k / 2] = v;
        ss2 = fma2(v, v, ss2);
      }
      if (RES && c < D) {
        if (whole(c)) {
          st_pairs<TR, 4>(sum + c, h[i]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 u = unpack2(h[i][k / 2]);
            if (in(c + k)) sum[c + k] = from_f32<TR>(k % 2 ? u.y : u.x);
          }
        }
      }
    }
  }
  const float2 sp = unpack2(ss2);
  const float ss = row_reduce<TPR, false>(sp.x + sp.y, red);
  const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
  const f32x2 r2 = pack2(r, r);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = col(i);
    if (c >= a.D) continue;
    float w[4];
    if (a.w_dtype == Elem<T>::code) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = to_f32<T>(static_cast<const T*>(a.w)[in(c + k) ? c + k : 0]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = static_cast<const float*>(a.w)[in(c + k) ? c + k : 0];
    }
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      h[i][k / 2] = mul2(mul2(h[i][k / 2], r2), pack2(w[k], w[k + 1]));
      const float2 u = unpack2(h[i][k / 2]);
      if (QUANT == kQuantRow) {
        if (in(c + k)) amax = max_nan(amax, fabsf(u.x));
        if (in(c + k + 1)) amax = max_nan(amax, fabsf(u.y));
      }
    }
  }
  Scale by;
  if (QUANT == kQuantRow) {
    by = scale_of(row_reduce<TPR, true>(amax, red));
    if (live && tx == 0) a.scale[row] = by.s;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = col(i);
    if (c >= D) continue;
    if (QUANT == kNoQuant) {
      T* y = static_cast<T*>(a.y) + row * a.y_rs;
      if (whole(c)) {
        st_pairs<T, 4>(y + c, h[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 u = unpack2(h[i][k / 2]);
          if (in(c + k)) y[c + k] = from_f32<T>(k % 2 ? u.y : u.x);
        }
      }
    } else {
      uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_rs;
      Pack<uint16_t, 2> o;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        o.v[k] = __nv_cvt_float2_to_fp8x2(by.quotient(h[i][k]), __NV_SATFINITE, __NV_E4M3);
      if (whole(c)) {
        st_pack<uint16_t, 2>(reinterpret_cast<uint16_t*>(y + c), o);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (in(c + k)) y[c + k] = static_cast<uint8_t>(o.v[k / 2] >> (8 * (k % 2)));
      }
    }
  }
}

// Any columns, strides and alignment, element by element. A warp takes 128
// columns at a time, a lane every 32nd of them, so that a group (32, 64 or 128) lies in one
// warp. NSEG > 0: each thread keeps its (at most 4 NSEG) values in registers, else a row is
// read again (from L1 and L2) by each pass.
template <typename T, typename TR, int TPR, int NSEG, int QUANT, bool RES>
__global__ void __launch_bounds__(threads_of(TPR), blocks_of(TPR, 4 * NSEG)) rms_norm_any_kernel(const NormArgs a) {
  constexpr int RPB = threads_of(TPR) / TPR;  // rows of a block
  __shared__ float red[32];
  const int64_t row_ = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool live = RPB == 1 || row_ < a.rows;
  const int64_t row = live ? row_ : a.rows - 1;  // barriers and shuffles need every thread
  const int D = live ? a.D : 0;                  // columns to write
  const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
  const TR* res = RES ? static_cast<const TR*>(a.res) + row * a.res_rs : nullptr;
  auto load = [&](int c, float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ck = min(c + 32 * k, a.D - 1);  // loads without a branch
      v[k] = to_f32<T>(x[ck]) + (RES ? to_f32<TR>(res[ck]) : 0.f);
    }
  };
  // f(first column, i) for the thread's part of every 128 columns of the row
  auto each = [&](auto&& f) {
    const int c0 = threadIdx.x % TPR / 32 * 128 + threadIdx.x % 32;
    if (NSEG) {
#pragma unroll
      for (int i = 0; i < (NSEG ? NSEG : 1); ++i) f(c0 + i * TPR * 4, i);
    } else {
      for (int c = c0; c - static_cast<int>(threadIdx.x % 32) < a.D; c += TPR * 4) f(c, 0);
    }
  };
  float h[NSEG ? NSEG : 1][4];
  float ss = 0.f;
  each([&](int c, int i) {
    load(c, h[i]);
#pragma unroll
    for (int k = 0; k < 4; ++k) ss = c + 32 * k < a.D ? fmaf(h[i][k], h[i][k], ss) : ss;
  });
  ss = row_reduce<TPR, false>(ss, red);
  const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
  auto y_of = [&](int c, float v) { return c < a.D ? v * r * ld_beta_any(a.w, a.w_dtype, c) : 0.f; };
  Scale by;
  if (QUANT == kQuantRow) {
    float amax = 0.f;
    each([&](int c, int i) {
      if (!NSEG) load(c, h[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) amax = max_nan(amax, fabsf(y_of(c + 32 * k, h[i][k])));
    });
    by = scale_of(row_reduce<TPR, true>(amax, red));
    if (live && threadIdx.x % TPR == 0) a.scale[row] = by.s;
  }
  each([&](int c, int i) {
    if (!NSEG) load(c, h[i]);
    float o[4];
    Scale of[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = y_of(c + 32 * k, h[i][k]);
      of[k] = by;
    }
    if (QUANT == kQuantGroup) {
      // the bits of numbers without a sign are in their order, with NaN above all
      unsigned b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(fabsf(o[k]));
      if (a.group >= 64) {
        b[0] = b[1] = max(b[0], b[1]);
        b[2] = b[3] = max(b[2], b[3]);
      }
      if (a.group == 128) b[0] = b[2] = max(b[0], b[2]);
      float m[4];
      m[0] = m[1] = m[2] = m[3] = __uint_as_float(__reduce_max_sync(0xffffffffu, b[0]));
      if (a.group <= 64) m[2] = m[3] = __uint_as_float(__reduce_max_sync(0xffffffffu, b[2]));
      if (a.group == 32) {
        m[1] = __uint_as_float(__reduce_max_sync(0xffffffffu, b[1]));
        m[3] = __uint_as_float(__reduce_max_sync(0xffffffffu, b[3]));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k == 0 || a.group == 32 || (k == 2 && a.group == 64)) by = scale_of(m[k]);
        of[k] = by;
        const int ck = c + 32 * k;
        if (ck < D && (ck & (a.group - 1)) == 0) a.scale[row * a.groups + (ck >> a.shift)] = by.s;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ck = c + 32 * k;
      if (ck < D) {
        if (RES) static_cast<TR*>(a.sum)[row * a.sum_rs + ck] = from_f32<TR>(h[i][k]);
        if (QUANT == kNoQuant) static_cast<T*>(a.y)[row * a.y_rs + ck] = from_f32<T>(o[k]);
        else static_cast<uint8_t*>(a.y)[row * a.y_rs + ck] =
                 __nv_cvt_float_to_fp8(of[k].quotient(o[k]), __NV_SATFINITE, __NV_E4M3);
      }
    }
  });
}

bool wide(const void* p, int bytes = 16) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

template <int TPR>
unsigned blocks_for(int64_t rows) {
  constexpr int RPB = threads_of(TPR) / TPR;
  return static_cast<unsigned>((rows + RPB - 1) / RPB);
}

template <typename T, typename TR, int TPR, int NV, bool RES>
void launch_norm_q(const NormArgs& a, int quant, cudaStream_t st) {
  const unsigned g = blocks_for<TPR>(a.rows), th = threads_of(TPR);
  if (quant == kNoQuant) rms_norm_kernel<T, TR, TPR, NV, kNoQuant, RES><<<g, th, 0, st>>>(a);
  else if (quant == kQuantRow) rms_norm_kernel<T, TR, TPR, NV, kQuantRow, RES><<<g, th, 0, st>>>(a);
  else rms_norm_kernel<T, TR, TPR, NV, kQuantGroup, RES><<<g, th, 0, st>>>(a);
}

template <typename T, typename TR, int TPR, int NSEG, bool RES>
void launch_any(const NormArgs& a, int quant, cudaStream_t st) {
  const unsigned g = blocks_for<TPR>(a.rows), th = threads_of(TPR);
  if (quant == kNoQuant) rms_norm_any_kernel<T, TR, TPR, NSEG, kNoQuant, RES><<<g, th, 0, st>>>(a);
  else if (quant == kQuantRow) rms_norm_any_kernel<T, TR, TPR, NSEG, kQuantRow, RES><<<g, th, 0, st>>>(a);
  else rms_norm_any_kernel<T, TR, TPR, NSEG, kQuantGroup, RES><<<g, th, 0, st>>>(a);
}

template <typename T, typename TR, int TPR, int NV, bool RES>
void launch_shift(const NormArgs& a, int quant, cudaStream_t st) {
  const unsigned g = blocks_for<TPR>(a.rows), th = threads_of(TPR);
  if (quant == kNoQuant) rms_norm_shift_kernel<T, TR, TPR, NV, kNoQuant, RES><<<g, th, 0, st>>>(a);
  else rms_norm_shift_kernel<T, TR, TPR, NV, kQuantRow, RES><<<g, th, 0, st>>>(a);
}

// Elements of one index modulo 4 lie on 4 elements' alignment in all of the rows.
template <typename T, typename TR, bool RES>
bool alike(NormArgs& a, int quant) {
  const int64_t i = reinterpret_cast<uintptr_t>(a.x) / sizeof(T);
  a.phase = static_cast<int>(i & 3);
  auto same = [&](const void* p, int bytes, int64_t rs) {
    const int64_t at = reinterpret_cast<uintptr_t>(p) / bytes;
    return ((at - i) & 3) == 0 && ((rs - a.x_rs) & 3) == 0;
  };
  return a.D >= 8 && quant != kQuantGroup &&
         same(a.y, quant == kNoQuant ? sizeof(T) : 1, a.y_rs) &&
         (!RES || (same(a.res, sizeof(TR), a.res_rs) && same(a.sum, sizeof(TR), a.sum_rs)));
}

template <typename T, typename TR, bool RES>
int launch_norm_t(NormArgs a, int quant, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int ybytes = quant == kNoQuant ? 16 : V;
  const bool ok = a.D % V == 0 && a.x_rs % V == 0 && wide(a.x) && wide(a.w) &&
                  (!RES || (a.res_rs % V == 0 && a.sum_rs % V == 0 && wide(a.res) && wide(a.sum))) &&
                  a.y_rs % V == 0 && wide(a.y, ybytes) && a.D <= 1024 * 4 * V;
  if (!ok && a.D + 3 <= 4 * 4096 && alike<T, TR, RES>(a, quant)) {
    const int nv = (a.D + 6) / 4;  // with up to 3 columns of lead
    if (nv <= 4 * 32) launch_shift<T, TR, 32, 4, RES>(a, quant, st);
    else if (nv <= 8 * 32) launch_shift<T, TR, 32, 8, RES>(a, quant, st);
    else if (nv <= 3 * 256) launch_shift<T, TR, 256, 3, RES>(a, quant, st);
    else if (nv <= 5 * 256) launch_shift<T, TR, 256, 5, RES>(a, quant, st);
    else if (nv <= 7 * 256) launch_shift<T, TR, 256, 7, RES>(a, quant, st);
    else if (nv <= 9 * 256) launch_shift<T, TR, 256, 9, RES>(a, quant, st);
    else if (nv <= 6 * 512) launch_shift<T, TR, 512, 6, RES>(a, quant, st);
    else launch_shift<T, TR, 512, 8, RES>(a, quant, st);
  } else if (!ok) {
    if (a.D <= 4 * 128) launch_any<T, TR, 32, 4, RES>(a, quant, st);
    else if (a.D <= 8 * 128) launch_any<T, TR, 32, 8, RES>(a, quant, st);
    else if (a.D <= 3 * 1024) launch_any<T, TR, 256, 3, RES>(a, quant, st);
    else if (a.D <= 5 * 1024) launch_any<T, TR, 256, 5, RES>(a, quant, st);
    else if (a.D <= 8 * 1024) launch_any<T, TR, 256, 8, RES>(a, quant, st);
    else launch_any<T, TR, 512, 0, RES>(a, quant, st);
  } else {
    const int nv = a.D / V;
    if (nv <= 32) launch_norm_q<T, TR, 32, 1, RES>(a, quant, st);
    else if (nv <= 128) launch_norm_q<T, TR, 32, 4, RES>(a, quant, st);
    else if (nv <= 512) launch_norm_q<T, TR, 256, 2, RES>(a, quant, st);
    else if (nv <= 1024) launch_norm_q<T, TR, 256, 4, RES>(a, quant, st);
    else if (nv <= 2048) launch_norm_q<T, TR, 512, 4, RES>(a, quant, st);
    else launch_norm_q<T, TR, 1024, 4, RES>(a, quant, st);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "add_rms_norm launch");
}

template <typename T>
int launch_norm_r(const NormArgs& a, int res_dtype, int quant, cudaStream_t st) {
  if (!a.res) return launch_norm_t<T, T, false>(a, quant, st);
  if (res_dtype == Elem<T>::code) return launch_norm_t<T, T, true>(a, quant, st);
  return launch_norm_t<T, float, true>(a, quant, st);
}

}  // namespace

int launch_add_rms_norm(const ptof_add_rms_norm_params& p, const void* x, const void* residual,
                        const void* w, void* y, void* sum, float* scale, cudaStream_t st) {
  if (p.rows == 0) return PTOF_OK;
  NormArgs a{};
  a.x = x; a.res = residual; a.w = w; a.y = y; a.sum = sum; a.scale = scale;
  a.x_rs = p.x_row_stride; a.res_rs = p.residual_row_stride;
  a.y_rs = p.y_row_stride; a.sum_rs = p.sum_row_stride;
  a.rows = p.rows; a.D = p.D;
  a.w_dtype = p.w_dtype; a.eps = p.eps; a.inv_d = 1.f / static_cast<float>(p.D);
  const int quant = !p.fp8 ? kNoQuant : p.group ? kQuantGroup : kQuantRow;
  a.group = p.group;
  while (2 << a.shift <= p.group) ++a.shift;
  a.groups = p.group ? (p.D + p.group - 1) / p.group : 1;
  if (p.dtype == PTOF_F32) return launch_norm_r<float>(a, p.residual_dtype, quant, st);
  if (p.dtype == PTOF_F16) return launch_norm_r<__half>(a, p.residual_dtype, quant, st);
  return launch_norm_r<__nv_bfloat16>(a, p.residual_dtype, quant, st);
}

}  // namespace ptof
