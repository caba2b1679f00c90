// Selective state space scan, for prompts and for single tokens. With
// dt' = softplus(dt + dt_bias) (or dt + dt_bias) and channel d of B / C group g = d G / D:
//   h[t, d, n] = exp(dt'[t, d] A[d, n]) h[t - 1, d, n] + dt'[t, d] x[t, d] B[t, g, n]
//   y[t, d]    = (sum_n C[t, g, n] h[t, d, n] + D[d] x[t, d]) * silu(z[t, d])
// All of it in fp32; y is rounded once to x's type, states stay fp32.
//
// Every (t, d, n) needs one exponential, so the prompt form is bound by the special-function
// units (16 a clock and SM), not by memory: at n = 16 a token and channel moves 8 bytes
// (bf16) and takes n + 3 of them with softplus and the gate. Counted so, at 1965 MHz, one
// sequence of 16384 tokens and 4096 channels needs 274 us (its bytes 83) and takes 735, of
// which the pass for the records is 42 %; 8 sequences of 2048 tokens and 5120 channels need 343
// and take 637 in one pass: the units (with the conversions that run there) are busy 64 % of the
// time and 60 % of the issue slots are taken, with 20 % of the warps that an SM could hold.
//
// A long axis with few channels is cut into chunks of S tokens. A first launch runs every
// chunk but the last of a sequence from a zero state and stores its final state and the sum
// of its dt' (the decay over a chunk is exp(A sum dt'), one exponential a state); the second
// joins the records before its chunk and runs it from the right state.
#include <cstring>
#include <type_traits>

#include "capi_internal.h"
#include "mixer_ops.cuh"

namespace ptof {

namespace {


struct ScanArgs {
  const void* x;
  const void* dt;
  const float* A;
  const void* B;
  const void* C;
  const float* D;
  const void* z;
  const float* bias;
  const float* init;
  const int* cu;
  void* y;
  float* fin;
  float* ws_dt;  // [slots, D] sum of dt' over the chunk
  float* ws_h;   // [slots, D, n] final state of the chunk from a zero state
  int64_t x_bs, x_ts, dt_bs, dt_ts, z_bs, z_ts, y_bs, y_ts;
  int64_t B_bs, B_ts, B_gs, C_bs, C_ts, C_gs;
  int N, T, Dch, n, G, dpg;  // sequences, tokens, channels, states, groups, channels of a group
  int softplus, fill;
  int piece;                 // copies of x, dt, z and y: 2 wide, 1 words, 0 elements
  int bc_piece;              // of B and C: 2 by 16 bytes, 1 by 4 values, 0 elements
  int S, slots, per_seq;     // chunk length (0: whole sequences), chunk slots, slots of a batch row
  int ch_blocks;             // blocks of a group's channels
};

// The chunk of slot `slot`: sequence n, its token range [s, e) and the chunk's [t0, t1).
// Packed chunks: slot cu[n] / S + n + j is chunk j of sequence n; neighbours do not overlap
// as floor(cu[n + 1] / S) + 1 - floor(cu[n] / S) >= ceil((cu[n + 1] - cu[n]) / S).
__device__ __forceinline__ bool scan_chunk(const ScanArgs& a, int slot, int& n, int& j, int& s,
                                           int& e) {
  s = 0;
  e = a.T;
  j = 0;
  n = slot;
  if (!a.cu) {
    if (a.S) {
      n = slot / a.per_seq;
      j = slot - n * a.per_seq;
    }
    return n < a.N;
  }
  if (a.S) {
    int lo = 0, hi = a.N - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (min(max(a.cu[mid], 0), a.T) / a.S + mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    n = lo;
    seq_bounds(a.cu, n, a.T, s, e);
    j = slot - (s / a.S + n);
    return j >= 0;
  }
  seq_bounds(a.cu, n, a.T, s, e);
  return true;
}

__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ f32x2 plus(f32x2 a, f32x2 b) { return add2(a, b); }

// Adds the LANES partial sums p[k] (of token k) over the lanes; lane j returns token j's sum.
template <int LANES, typename V>
__device__ __forceinline__ V transpose_sum(V (&p)[LANES], int lane) {
#pragma unroll
  for (int off = LANES / 2; off >= 1; off /= 2) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < off; ++i) {
      const V send = up ? p[i] : p[i + off];
      const V keep = up ? p[i + off] : p[i];
      p[i] = plus(keep, __shfl_xor_sync(0xffffffffu, send, off));
    }
  }
  return p[0];
}

// The sum over the lanes of a channel that transpose_sum over four tokens and the lanes behind
// them give, in the same order: what a row's result is does not depend on the rows beside it.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  constexpr int T = LANES < 4 ? LANES : 4;
#pragma unroll
  for (int off = T / 2; off >= 1; off /= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
#pragma unroll
  for (int off = T; off < LANES; off *= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// A in units of log2, kept finite (but for NaN): 0 * A is then 0, so that a step of zero
// leaves the state as it is, and 2^(dt' A) is still 0 or inf where it was.
__device__ __forceinline__ float log2_rate(float A) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(A * kLog2e), "f"(3e38f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(-3e38f));
  return r;
}

// The state after a chunk: 2^u h + r, of a record r and the decay 2^u over the chunk. Where 2^u is
// zero or infinite, though no single step's decay was, an infinite h and one of zero stay
// what they are.
__device__ __forceinline__ float join(float u, float h, float r) {
  const float e = fast_exp2(u), v = fmaf(e, h, r);
  if (v == v) return v;
  const float p = e * h;
  return (p == p || !(fabsf(u) <= 3.40282347e38f) ? p : h) + r;
}

// A warp's tile [TC tokens][CW channels] from or to global memory, in pieces of PIECE elements.
// Tokens behind the last are read as the last and not written; channels behind the block's
// are left alone.
template <typename T, int TC, int CW, int PIECE>
__device__ __forceinline__ void tile_in(T* dst, const T* src, int64_t ts, int t, int t1, int cw,
                                        int wl) {
  constexpr int ROW = CW / PIECE;
#pragma unroll
  for (int i = 0; i < (TC * ROW + 31) / 32; ++i) {
    const int idx = i * 32 + wl, r = idx / ROW, p = idx % ROW * PIECE;
    if ((TC * ROW % 32 == 0 || r < TC) && p < cw) {
      const T* g = src + min(t + r, t1 - 1) * ts + p;
      if (PIECE * sizeof(T) >= 4) copy_async<PIECE * sizeof(T)>(dst + r * CW + p, g);
      else dst[r * CW + p] = *g;
    }
  }
}
template <typename T, int TC, int CW, int PIECE>
__device__ __forceinline__ void tile_out(T* dst, const T* src, int64_t ts, int t, int t1, int cw,
                                         int wl) {
  constexpr int ROW = CW / PIECE;
#pragma unroll
  for (int i = 0; i < (TC * ROW + 31) / 32; ++i) {
    const int idx = i * 32 + wl, r = idx / ROW, p = idx % ROW * PIECE;
    if ((TC * ROW % 32 == 0 || r < TC) && p < cw && t + r < t1)
      st_pack<T, PIECE>(dst + (t + r) * ts + p, ld_pack<T, PIECE>(src + r * CW + p));
  }
}

// Two neighbouring values of T as a pair of fp32 values, and back.
template <typename T>
__device__ __forceinline__ f32x2 pair_of(const Pack<T, 2>& v) {
  return pack2(to_f32<T>(v.v[0]), to_f32<T>(v.v[1]));
}
template <typename T>
__device__ __forceinline__ void st_pair(T* p, f32x2 v) {
  const float2 u = unpack2(v);
  Pack<T, 2> o;
  o.v[0] = from_f32<T>(u.x);
  o.v[1] = from_f32<T>(u.y);
  st_pack<T, 2>(p, o);
}

// Shared memory of a block, which is one warp.
template <typename T, int LANES, int SPL, int TILE, int TL>
struct ScanSmem {
  static constexpr int CW = 64 / LANES, NP = LANES * SPL;
  T tile[2][3][TILE * CW];               // x (then y), dt, z of a tile, and of the next
  T raw[2][2][TILE * NP];                // B, C as they came
  alignas(16) float bc[2][2][TL * NP];   // B, C of a group of tokens as fp32, and of the next
  alignas(16) f32x2 d[2][TL * CW / 2][2];  // dt' and dt' x of the channel pairs, as well
};

// A warp, a block of its own so that any number of them spreads evenly over the SMs, runs
// 64 / LANES channels of one chunk of one sequence. A thread holds SPL states of two
// neighbouring channels, so that every product of the recurrence, and the activations, is
// a two-value instruction. LANES threads share a channel pair: in each group of TL tokens a
// lane prepares one (dt' and dt' x, handed over through shared memory) and finishes one
// (skip, gate, store): the partial sums of y are transposed and added over the lanes.
//
// Two streams of work are interleaved so that neither waits alone: the recurrence of one
// group, whose decays and inputs are formed ahead of the chain, and the preparation of the
// next (softplus, B and C to fp32). x, dt, z, B and C come through shared memory a tile of
// groups ahead (one asynchronous copy for many tokens, reads at constant offsets), y
// leaves through the tile of x.
//
// States with padding (PAD): theirs are zero as B and C are there, unless dt' or dt' x is infinite or
// NaN. The warp looks for that while it prepares a group and then takes the guarded pass.
template <typename T, int LANES, int SPL, int TILE, int G, bool SUMMARY, bool PAD>
__global__ void __launch_bounds__(32, SPL <= 4 ? 16 : 12) ssm_scan_kernel(const ScanArgs a) {
  constexpr int NP = LANES * SPL;            // states with padding
  constexpr int CW = 64 / LANES;             // channels of a warp
  constexpr int TL = LANES < 8 ? LANES : SPL < 8 ? 8 : 4;  // tokens of a group
  constexpr int NG = TILE / TL;              // groups of a tile
  constexpr int WIDE = CW * sizeof(T) >= 16 ? 16 / sizeof(T) : CW;  // widest copied piece
  static_assert(NG % 2 == 0 && TL % G == 0 && SPL % 2 == 0, "layout");
  extern __shared__ __align__(16) unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<ScanSmem<T, LANES, SPL, TILE, TL>*>(smem_raw);

  const int per_slot = a.ch_blocks * a.G;
  const int slot = static_cast<int>(blockIdx.x / per_slot);
  const int rest = static_cast<int>(blockIdx.x - static_cast<int64_t>(slot) * per_slot);
  const int g = rest / a.ch_blocks, cb = rest - g * a.ch_blocks;
  int n, j, s, e;
  if (!scan_chunk(a, slot, n, j, s, e)) return;
  const int64_t len = a.S ? a.S : a.T;
  const int t0 = static_cast<int>(min(static_cast<int64_t>(e), s + j * len));
  const int t1 = static_cast<int>(min(static_cast<int64_t>(e), t0 + len));
  const bool last = t1 == e;
  if (SUMMARY ? last : (j > 0 && t0 >= e)) return;

  const int wl = threadIdx.x;
  const int lane = wl % LANES, wp = wl / LANES;  // lane of the channel pair, pair of the warp
  const int tok = lane % TL;
  const int cw = min(CW, a.dpg - cb * CW);       // channels of this warp
  const bool live0 = 2 * wp < cw, live1 = 2 * wp + 1 < cw;
  const int c0 = g * a.dpg + cb * CW;
  const int64_t ca = c0 + (live0 ? 2 * wp : 0), cz = c0 + (live1 ? 2 * wp + 1 : 0);
  const int b = a.cu ? 0 : n;

  if (!SUMMARY && a.fill && a.cu && last) {
    // tokens of no sequence: before the first and after the last
    const int i = wl % CW, first = wl / CW, step = CW < 32 ? 32 / CW : 1;
    for (int k = i; k < cw; k += 32) {
      T* yc = static_cast<T*>(a.y) + c0 + k;
      if (n == 0)
        for (int64_t t = first; t < s; t += step) yc[t * a.y_ts] = from_f32<T>(0.f);
      if (n == a.N - 1)
        for (int64_t t = static_cast<int64_t>(e) + first; t < a.T; t += step)
          yc[t * a.y_ts] = from_f32<T>(0.f);
    }
  }

  f32x2 A2[SPL], h[SPL];
#pragma unroll
  for (int i = 0; i < SPL; ++i) {
    const int k = lane * SPL + i;
    A2[i] = k < a.n ? pack2(log2_rate(a.A[ca * a.n + k]), log2_rate(a.A[cz * a.n + k]))
                    : pack2(0.f, 0.f);
    h[i] = pack2(0.f, 0.f);
  }
  auto state_at = [&](const float* p, int k) { return pack2(p[ca * a.n + k], p[cz * a.n + k]); };
  if (!SUMMARY && a.init) {
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int k = lane * SPL + i;
      if (k < a.n) h[i] = state_at(a.init + static_cast<int64_t>(n) * a.Dch * a.n, k);
    }
  }
  if (!SUMMARY && j > 0) {
#pragma unroll 4
    for (int q = slot - j; q < slot; ++q) {  // the chunks before this one
      const int64_t r = static_cast<int64_t>(q) * a.Dch;
      const f32x2 sum = pack2(a.ws_dt[r + ca], a.ws_dt[r + cz]);
#pragma unroll
      for (int i = 0; i < SPL; ++i) {
        const int k = lane * SPL + i;
        const float2 u = unpack2(mul2(sum, A2[i]));
        if (k < a.n)
          h[i] = fma2(pack2(fast_exp2(u.x), fast_exp2(u.y)), h[i], state_at(a.ws_h + r * a.n, k));
      }
    }
    // A NaN, which stays through the loop, may come from a decay that is zero or infinite only over
    // a whole chunk: such states are joined again, with a test at each chunk. (The test in the
    // loop above took 777 x 512 with 64 states from 41 to 54 us.)
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int k = lane * SPL + i;
      float2 v = unpack2(h[i]);
      if (k < a.n && !(v.x == v.x && v.y == v.y)) {
        v = a.init ? unpack2(state_at(a.init + static_cast<int64_t>(n) * a.Dch * a.n, k)) : make_float2(0.f, 0.f);
#pragma unroll 1
        for (int q = slot - j; q < slot; ++q) {
          const int64_t r = static_cast<int64_t>(q) * a.Dch;
          const float2 u = unpack2(mul2(pack2(a.ws_dt[r + ca], a.ws_dt[r + cz]), A2[i]));
          const float2 w = unpack2(state_at(a.ws_h + r * a.n, k));
          v = make_float2(join(u.x, v.x, w.x), join(u.y, v.y, w.y));
        }
        h[i] = pack2(v.x, v.y);
      }
    }
  }
  const f32x2 bias = a.bias ? pack2(a.bias[ca], a.bias[cz]) : pack2(0.f, 0.f);
  const f32x2 skip = a.D ? pack2(a.D[ca], a.D[cz]) : pack2(0.f, 0.f);
  // the chunk's sum of dt': what a tile adds goes into a compensated sum (W. Kahan, Further remarks
  // on reducing truncation errors, 1965), so that its error does not grow with the chunk
  f32x2 dt_tile = pack2(0.f, 0.f), dt_sum = dt_tile, dt_rest = dt_tile;

  const T* Bp = static_cast<const T*>(a.B) + b * a.B_bs + g * a.B_gs;
  const T* Cp = static_cast<const T*>(a.C) + b * a.C_bs + g * a.C_gs;
  const T* xp = static_cast<const T*>(a.x) + b * a.x_bs + c0;
  const T* dp = static_cast<const T*>(a.dt) + b * a.dt_bs + c0;
  const T* zp = a.z && !SUMMARY ? static_cast<const T*>(a.z) + b * a.z_bs + c0 : nullptr;
  T* yp = static_cast<T*>(a.y) + b * a.y_bs + c0;

  auto copy = [&](int t, int st) {  // the inputs of the tile at t, into stage st
    T(*d)[TILE * CW] = sm.tile[st];
    if (a.piece == 2) {
      tile_in<T, TILE, CW, WIDE>(d[0], xp, a.x_ts, t, t1, cw, wl);
      tile_in<T, TILE, CW, WIDE>(d[1], dp, a.dt_ts, t, t1, cw, wl);
      if (zp) tile_in<T, TILE, CW, WIDE>(d[2], zp, a.z_ts, t, t1, cw, wl);
    } else if (a.piece == 1) {
      tile_in<T, TILE, CW, 4 / sizeof(T)>(d[0], xp, a.x_ts, t, t1, cw, wl);
      tile_in<T, TILE, CW, 4 / sizeof(T)>(d[1], dp, a.dt_ts, t, t1, cw, wl);
      if (zp) tile_in<T, TILE, CW, 4 / sizeof(T)>(d[2], zp, a.z_ts, t, t1, cw, wl);
    } else {
      tile_in<T, TILE, CW, 1>(d[0], xp, a.x_ts, t, t1, cw, wl);
      tile_in<T, TILE, CW, 1>(d[1], dp, a.dt_ts, t, t1, cw, wl);
      if (zp) tile_in<T, TILE, CW, 1>(d[2], zp, a.z_ts, t, t1, cw, wl);
    }
    T(*r)[TILE * NP] = sm.raw[st];
    constexpr int BW = 16 / sizeof(T) < NP ? 16 / sizeof(T) : 4;
    if (a.bc_piece == 2) {
      tile_in<T, TILE, NP, BW>(r[0], Bp, a.B_ts, t, t1, a.n, wl);
      if (!SUMMARY) tile_in<T, TILE, NP, BW>(r[1], Cp, a.C_ts, t, t1, a.n, wl);
    } else if (a.bc_piece == 1) {
      tile_in<T, TILE, NP, 4>(r[0], Bp, a.B_ts, t, t1, a.n, wl);
      if (!SUMMARY) tile_in<T, TILE, NP, 4>(r[1], Cp, a.C_ts, t, t1, a.n, wl);
    } else {
      tile_in<T, TILE, NP, 1>(r[0], Bp, a.B_ts, t, t1, a.n, wl);
      if (!SUMMARY) tile_in<T, TILE, NP, 1>(r[1], Cp, a.C_ts, t, t1, a.n, wl);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  if (a.n < NP) {  // zeros behind the states, where nothing is copied
    T* r = sm.raw[0][0];
    for (int i = wl; i < 4 * TILE * NP; i += 32)
      if (i % NP >= a.n) r[i] = from_f32<T>(0.f);
  }
  if (PAD && cw < CW) {  // and in the channels behind the last, so that nothing odd is found there
    T* x = sm.tile[0][0];
    for (int i = wl; i < 6 * TILE * CW; i += 32)
      if (i % CW >= cw) x[i] = from_f32<T>(0.f);
  }
  // What group `g` of the tile at t (in stage st) needs before its recurrence: dt' and dt' x
  // of this lane's token, B and C as fp32. Steps behind the chunk are zero: they leave the
  // state as it is.
  constexpr int kM = SUMMARY ? 1 : 2, kBC = (TL * NP * kM / 4 + 31) / 32;
  bool odd = false;  // PAD: the prepared group needs the guarded pass
  auto prepare = [&](int t, int st, int g) {
    const T* tx = &sm.tile[st][0][(g * TL + tok) * CW + 2 * wp];
    Pack<T, 4> raw[kBC];
#pragma unroll
    for (int i = 0; i < kBC; ++i) {
      const int idx = (i * 32 + wl) * 4;
      if (TL * NP * kM % 128 == 0 || idx < TL * NP * kM)
        raw[i] = ld_pack<T, 4>(&sm.raw[st][idx / (TL * NP)][g * TL * NP + idx % (TL * NP)]);
    }
    f32x2 d = add2(pair_of(ld_pack<T, 2>(tx + TILE * CW)), bias);
    const f32x2 xv = pair_of(ld_pack<T, 2>(tx));
    if (a.softplus) d = softplus2(d);
    ulonglong2 both;
    both.x = d;
    both.y = mul2(d, xv);
    if (t + TILE > t1 && t + g * TL + tok >= t1) both.x = both.y = pack2(0.f, 0.f);
    if (PAD) {
      const float2 zero = unpack2(mul2(add2(both.x, both.y), pack2(0.f, 0.f)));
      odd = __any_sync(0xffffffffu, !(zero.x == 0.f && zero.y == 0.f));
    }
    if (SUMMARY && lane < TL) dt_tile = add2(dt_tile, both.x);
    *reinterpret_cast<ulonglong2*>(sm.d[g % 2][tok * (CW / 2) + wp]) = both;
#pragma unroll
    for (int i = 0; i < kBC; ++i) {
      const int idx = (i * 32 + wl) * 4;
      if (TL * NP * kM % 128 == 0 || idx < TL * NP * kM) {
        Pack<float, 4> f;
#pragma unroll
        for (int u = 0; u < 4; ++u) f.v[u] = to_f32<T>(raw[i].v[u]);
        st_pack<float, 4>(&sm.bc[g % 2][0][0] + idx, f);
      }
    }
  };

  if (t0 < t1) {
    copy(t0, 0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    if (t0 + TILE < t1) copy(t0 + TILE, 1);
    prepare(t0, 0, 0);
  }
  // One group of the tile at t: its recurrence and outputs, and the preparation of the next. With
  // `guard` a state takes nothing from tokens behind the chunk, whose dt' x is zero but whose B,
  // read as the last token's, may be infinite: zero times infinity would stay in it. Kept apart
  // so that the tiles before the last go without a test inside.
  auto group = [&](auto guard, int t, int st, int g) {
    T* tx = &sm.tile[st][0][(g * TL + tok) * CW + 2 * wp];
    f32x2 part[TL], xv, zv;
    if (!SUMMARY) {
      xv = pair_of(ld_pack<T, 2>(tx));
      if (zp) zv = pair_of(ld_pack<T, 2>(tx + 2 * TILE * CW));
    }
#pragma unroll
    for (int i0 = 0; i0 < TL; i0 += G) {
      f32x2 E[G][SPL], X[G][SPL];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const ulonglong2 both = *reinterpret_cast<const ulonglong2*>(sm.d[g % 2][(i0 + i) * (CW / 2) + wp]);
        const float2 dx = unpack2(both.y);
        const Pack<float, SPL> bv = ld_pack<float, SPL>(&sm.bc[g % 2][0][(i0 + i) * NP + lane * SPL]);
#pragma unroll
        for (int k = 0; k < SPL; ++k) {
          const float2 u = unpack2(mul2(both.x, A2[k]));
          E[i][k] = pack2(fast_exp2(u.x), fast_exp2(u.y));
          X[i][k] = pack2(dx.x * bv.v[k], dx.y * bv.v[k]);
          if (guard.value) {
            if (PAD && lane * SPL + k >= a.n) E[i][k] = X[i][k] = pack2(0.f, 0.f);
            if (t + g * TL + i0 + i >= t1) X[i][k] = pack2(0.f, 0.f);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
#pragma unroll
        for (int k = 0; k < SPL; ++k) h[k] = E[i][k] = fma2(E[i][k], h[k], X[i][k]);
      }
      if (!SUMMARY) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const Pack<float, SPL> cv = ld_pack<float, SPL>(&sm.bc[g % 2][1][(i0 + i) * NP + lane * SPL]);
          float2 y2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int k = 0; k < SPL; ++k) {
            const float2 u = unpack2(E[i][k]);
            y2.x = k ? fmaf(cv.v[k], u.x, y2.x) : cv.v[k] * u.x;
            y2.y = k ? fmaf(cv.v[k], u.y, y2.y) : cv.v[k] * u.y;
          }
          part[i0 + i] = pack2(y2.x, y2.y);
        }
      }
    }
    if (g + 1 < NG) prepare(t, st, g + 1);
    else prepare(t + TILE, st ^ 1, 0);  // (behind the last tile: of no use and not used)
    if (!SUMMARY) {
      f32x2 v = transpose_sum<TL>(part, tok);
#pragma unroll
      for (int off = TL; off < LANES; off *= 2)
        v = add2(v, __shfl_xor_sync(0xffffffffu, v, off));
      if (a.D) v = fma2(skip, xv, v);  // (zero times an infinite x would stay)
      if (zp) v = mul2(v, silu2(zv));
      if (lane < TL) st_pair<T>(tx, v);  // over x, which all have read
    }
  };
  auto tile = [&](auto guard, int t, int st) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (g == NG - 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      if (PAD && !guard.value && odd) group(std::true_type{}, t, st, g);
      else group(guard, t, st, g);
    }
  };
  int st = 0;
  for (int t = t0; t < t1; t += TILE, st ^= 1) {
    if (t + TILE <= t1) tile(std::false_type{}, t, st);
    else tile(std::true_type{}, t, st);
    __syncwarp();  // y is in the tile
    if (!SUMMARY) {
      const T* ty = sm.tile[st][0];
      if (a.piece == 2) tile_out<T, TILE, CW, WIDE>(yp, ty, a.y_ts, t, t1, cw, wl);
      else if (a.piece == 1) tile_out<T, TILE, CW, 4 / sizeof(T)>(yp, ty, a.y_ts, t, t1, cw, wl);
      else tile_out<T, TILE, CW, 1>(yp, ty, a.y_ts, t, t1, cw, wl);
      __syncwarp();  // the tile is free
    }
    if (t + 2 * TILE < t1) copy(t + 2 * TILE, st);
    if (SUMMARY) {
      const f32x2 more = add2(dt_tile, dt_rest), sum = add2(dt_sum, more);
      const float2 rest = unpack2(add2(fma2(sum, pack2(-1.f, -1.f), dt_sum), more));
      dt_rest = pack2(rest.x == rest.x ? rest.x : 0.f, rest.y == rest.y ? rest.y : 0.f);  // inf - inf
      dt_sum = sum;
      dt_tile = pack2(0.f, 0.f);
    }
  }

  if (SUMMARY) {  // the lanes' parts of the sum of dt'
#pragma unroll
    for (int off = 1; off < LANES; off *= 2)
      dt_sum = add2(dt_sum, __shfl_xor_sync(0xffffffffu, dt_sum, off));
    const float2 v = unpack2(dt_sum);
    float* w = a.ws_dt + static_cast<int64_t>(slot) * a.Dch;
    if (lane == 0 && live0) w[ca] = v.x;
    if (lane == 0 && live1) w[cz] = v.y;
  }
  float* f = SUMMARY ? a.ws_h + static_cast<int64_t>(slot) * a.Dch * a.n
                     : a.fin + static_cast<int64_t>(n) * a.Dch * a.n;
  if (SUMMARY || (last && a.fin)) {
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int k = lane * SPL + i;
      const float2 v = unpack2(h[i]);
      if (live0 && k < a.n) f[ca * a.n + k] = v.x;
      if (live1 && k < a.n) f[cz * a.n + k] = v.y;
    }
  }
}

// Four neighbouring values as the words they were loaded as. They are taken apart only where
// they are used: a value that two branches could have loaded is otherwise taken apart, and so
// waited for, where the branches meet.
template <typename T>
struct Four {
  uint32_t w[sizeof(T)];
  __device__ __forceinline__ float operator[](int i) const {
    T v[4];
    memcpy(v, w, sizeof(v));
    return to_f32<T>(v[i]);
  }
};
template <typename T>
__device__ __forceinline__ Four<T> ld_four(const T* p, bool whole, int n) {  // zeros from n on
  Four<T> r;
  if (whole) {
    if (sizeof(T) == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      r.w[0] = v.x;
      r.w[1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      r.w[0] = v.x;
      r.w[1] = v.y;
      r.w[sizeof(T) - 2] = v.z;
      r.w[sizeof(T) - 1] = v.w;
    }
  } else {
    T v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = u < n ? p[u] : from_f32<T>(0.f);
    memcpy(r.w, v, sizeof(v));
  }
  return r;
}

struct ScanStepArgs {
  const void* x;
  const void* dt;
  const float* A;
  const void* B;
  const void* C;
  const float* D;
  const void* z;
  const float* bias;
  const int* slots;
  float* state;
  void* y;
  int64_t x_rs, dt_rs, z_rs, y_rs, B_rs, B_gs, C_rs, C_gs, s_ss;
  int M, S, Dch, n, dpg;
  int softplus, bc_vec;
  int ch_blocks;
};

constexpr int kScanStepThreads = 128;

// Single tokens: one row per block, LANES threads of 4 states each per channel, ITER channels a
// thread. Bound by the states' traffic (read and written once, 8 n bytes a channel): all of
// a thread's states are on their way before the first is used. As in the prompt form the
// lanes of a channel share its elementwise work, here over the ITER channels. 512 rows of
// 8192 channels and 16 states take 115 us, 0.76 of the copy bandwidth; several rows a block
// through a ring of asynchronous copies took 114.
// PAD: states that do not fill the lanes. The others' are zero as B and C are there, and are set to
// it where dt' or dt' x of any channel of the warp is infinite or NaN.
template <typename T, int LANES, int ITER, bool VEC, bool PAD>
__global__ void __launch_bounds__(kScanStepThreads, LANES < 4 ? 4 : 8) ssm_scan_step_kernel(const ScanStepArgs a) {
  constexpr int CH = kScanStepThreads / LANES;
  constexpr int TL = LANES < ITER ? LANES : ITER, PF = ITER / TL;
  const int m = static_cast<int>(blockIdx.x / a.ch_blocks);
  const int lane = threadIdx.x % LANES, tok = lane % TL;
  const int c0 = static_cast<int>(blockIdx.x % a.ch_blocks) * CH * ITER + threadIdx.x / LANES;
  const int slot = a.slots ? a.slots[m] : m;
  const bool used = slot >= 0 && slot < a.S;
  const int k0 = lane * 4;

  // what does not wait for the slot
  T rx[PF], rd[PF], rz[PF];
  Four<T> bv, cv;
  auto group_of = [&](int c) { return a.dpg == a.Dch ? 0 : min(c, a.Dch - 1) / a.dpg; };
  int g = group_of(c0);
  auto load_bc = [&](int r, int g) {
    const bool whole = a.bc_vec && k0 < a.n;  // zeros behind the states
    bv = ld_four<T>(static_cast<const T*>(a.B) + r * a.B_rs + g * a.B_gs + k0, whole, a.n - k0);
    cv = ld_four<T>(static_cast<const T*>(a.C) + r * a.C_rs + g * a.C_gs + k0, whole, a.n - k0);
  };
  auto load_row = [&](int r) {
#pragma unroll
    for (int q = 0; q < PF; ++q) {
      const int c = min(c0 + (q * TL + tok) * CH, a.Dch - 1);
      rx[q] = static_cast<const T*>(a.x)[r * a.x_rs + c];
      rd[q] = static_cast<const T*>(a.dt)[r * a.dt_rs + c];
      if (a.z) rz[q] = static_cast<const T*>(a.z)[r * a.z_rs + c];
    }
    load_bc(r, g = group_of(c0));
  };
  load_row(m);
  float bias[PF], skip[PF];
#pragma unroll
  for (int q = 0; q < PF; ++q) {
    const int c = min(c0 + (q * TL + tok) * CH, a.Dch - 1);
    bias[q] = a.bias ? a.bias[c] : 0.f;
    skip[q] = a.D ? a.D[c] : 0.f;
  }

  float4 A2[ITER], h[ITER];
  const int64_t first = static_cast<int64_t>(c0) * a.n + k0, step = static_cast<int64_t>(CH) * a.n;
  float* st = a.state + (used ? slot : 0) * a.s_ss + first;
  const float* ap = a.A + first;
  const int chans = k0 < a.n ? (a.Dch - c0 + CH - 1) / CH : 0;  // channels of this thread
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    A2[i] = h[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (used && i < chans) {
      const float* hp = st + i * step;
      const float* aq = ap + i * step;
      if (VEC) {
        h[i] = *reinterpret_cast<const float4*>(hp);
        A2[i] = *reinterpret_cast<const float4*>(aq);
      } else {
        h[i].x = hp[0];
        A2[i].x = aq[0];
        if (k0 + 1 < a.n) h[i].y = hp[1], A2[i].y = aq[1];
        if (k0 + 2 < a.n) h[i].z = hp[2], A2[i].z = aq[2];
        if (k0 + 3 < a.n) h[i].w = hp[3], A2[i].w = aq[3];
      }
    }
  }
  bool later = false;
  if (a.slots && a.M > 1) {
    const SlotUse u = slot_use(a.slots, a.M, m, slot);
    if (used && u.earlier) return;
    later = u.later;
  }
  if (!used) {  // a padding row
#pragma unroll
    for (int q = 0; q < PF; ++q) {
      const int c = c0 + (q * TL + tok) * CH;
      if (c < a.Dch && lane < TL) static_cast<T*>(a.y)[m * a.y_rs + c] = from_f32<T>(0.f);
    }
    return;
  }
  for (int r = m;;) {
    float d[PF], dx[PF], sx[PF], gate[PF], part[ITER], zero = 0.f;
#pragma unroll
    for (int q = 0; q < PF; ++q) {
      d[q] = to_f32<T>(rd[q]) + bias[q];
      if (a.softplus) d[q] = softplus_f32(d[q]);
      const float xv = to_f32<T>(rx[q]);
      dx[q] = d[q] * xv;
      if (PAD) zero = fmaf(d[q] + dx[q], 0.f, zero);
      d[q] *= kLog2e;  // exp(dt' A) = 2^(dt' log2(e) A)
      sx[q] = a.D ? skip[q] * xv : 0.f;
      gate[q] = a.z ? silu_f32(to_f32<T>(rz[q])) : 1.f;
    }
    const bool odd = PAD && __any_sync(0xffffffffu, !(zero == 0.f));
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      if (i && a.dpg != a.Dch) {
        const int gi = group_of(c0 + i * CH);
        if (gi != g) load_bc(r, g = gi);
      }
      const float di = LANES > 1 ? __shfl_sync(0xffffffffu, d[i / TL], i % TL, LANES) : d[i / TL];
      const float xi = LANES > 1 ? __shfl_sync(0xffffffffu, dx[i / TL], i % TL, LANES) : dx[i / TL];
      h[i].x = fmaf(fast_exp2(di * A2[i].x), h[i].x, xi * bv[0]);
      h[i].y = fmaf(fast_exp2(di * A2[i].y), h[i].y, xi * bv[1]);
      h[i].z = fmaf(fast_exp2(di * A2[i].z), h[i].z, xi * bv[2]);
      h[i].w = fmaf(fast_exp2(di * A2[i].w), h[i].w, xi * bv[3]);
      if (PAD && odd) {
        if (k0 >= a.n) h[i].x = 0.f;
        if (k0 + 1 >= a.n) h[i].y = 0.f;
        if (k0 + 2 >= a.n) h[i].z = 0.f;
        if (k0 + 3 >= a.n) h[i].w = 0.f;
      }
      part[i] = cv[0] * h[i].x;
      part[i] = fmaf(cv[1], h[i].y, part[i]);
      part[i] = fmaf(cv[2], h[i].z, part[i]);
      part[i] = fmaf(cv[3], h[i].w, part[i]);
    }
#pragma unroll
    for (int q = 0; q < PF; ++q) {
      float p[TL];
#pragma unroll
      for (int u = 0; u < TL; ++u) p[u] = part[q * TL + u];
      float v;
      if (ITER == 1) {
        v = lane_sum<LANES>(p[0]);
      } else {
        v = transpose_sum<TL>(p, tok);
#pragma unroll
        for (int off = TL; off < LANES; off *= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
      }
      const int c = c0 + (q * TL + tok) * CH;
      if (c < a.Dch && lane < TL)
        static_cast<T*>(a.y)[r * a.y_rs + c] = from_f32<T>((v + sx[q]) * gate[q]);
    }
    if (!later) break;
    for (++r; r < a.M && a.slots[r] != slot; ++r) {}
    if (r >= a.M) break;
    load_row(r);
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    if (i < chans) {
      float* hp = st + i * step;
      if (VEC) {
        *reinterpret_cast<float4*>(hp) = h[i];
      } else {
        hp[0] = h[i].x;
        if (k0 + 1 < a.n) hp[1] = h[i].y;
        if (k0 + 2 < a.n) hp[2] = h[i].z;
        if (k0 + 3 < a.n) hp[3] = h[i].w;
      }
    }
  }
}

// Zeros in every token of a packed call without a sequence.
template <typename T>
__global__ void __launch_bounds__(256) zero_tokens_kernel(T* y, int64_t ts, int tokens, int D) {
  const int64_t all = static_cast<int64_t>(tokens) * D, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < all; i += step)
    y[i / D * ts + i % D] = from_f32<T>(0.f);
}
template <typename T>
int launch_zero_tokens(void* y, int64_t ts, int tokens, int D, cudaStream_t st) {
  const int64_t blocks = (static_cast<int64_t>(tokens) * D + 255) / 256;
  if (blocks == 0) return PTOF_OK;
  zero_tokens_kernel<T><<<static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>(
      static_cast<T*>(y), ts, tokens, D);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "ssm_scan launch");
}

// Lanes of a channel pair, states of a lane and the chunk length for a prompt call.
struct ScanPlan {
  int lanes, spl, S, slots, per_seq;
};

// Whole sequences, or chunks at the price of a second pass without outputs? Counted in clocks:
// up to 16 warps run on an SM at a time, and with w of them a token takes a warp
// 55 + 45 SPL + 3.75 SPL w (its own latency, and what it waits for the others at the
// special-function units); a warp starts in about 3000. The two launches of a chunked call take
// 1.7 times the tokens together, 12000 to start and 100 a chunk to join the records. The
// constants were measured at n = 16 and are used for every n: with n > 16 registers leave room for
// 12 warps and shared memory for 9 (fp32, n > 32), 8 (16 bits, n > 64) or 5 (fp32, n > 64), which
// the count does not know. Measured at n = 16, bf16: one sequence of 16384 tokens and 4096 channels 2.3 ms whole, 0.74
// ms in chunks of 1024, 0.765 of 1856 and 0.87 of 2048 (14 warps an SM); 8 of 2048 tokens
// and 5120 channels 0.64 ms whole, 0.88 ms in chunks of 1024.
ScanPlan scan_plan(const ptof_ssm_scan_params& p) {
  ScanPlan q{};
  if (p.n <= 8) { q.lanes = 4; q.spl = 2; }
  else if (p.n <= 16) { q.lanes = 4; q.spl = 4; }
  else if (p.n <= 32) { q.lanes = 4; q.spl = 8; }
  else if (p.n <= 64) { q.lanes = 8; q.spl = 8; }
  else { q.lanes = 16; q.spl = 8; }
  q.slots = p.N;
  q.per_seq = 1;
  const int cw = 64 / q.lanes;
  const double blocks = static_cast<double>(p.G) * ((p.D / p.G + cw - 1) / cw);
  const double tokens = static_cast<double>(p.T) * (p.packed ? 1 : p.N);
  const double longest = p.packed && p.max_len > 0 ? p.max_len : p.T;
  const double warm = 55 + 45 * q.spl, each = 3.75 * q.spl;
  const auto clocks = [&](double len, double units) {
    const double w = units * blocks / 148, at_once = w < 16 ? w : 16;
    return (len * (warm + at_once * each) + 3000) * (w < 16 ? 1 : w / 16) + 3000;
  };
  double best = clocks(longest, p.N);
  for (int S = 64; S < longest && S <= 1 << 20; S = S < 2048 ? S + 32 : 2 * S) {
    const double chunks = p.packed ? tokens / S + 0.5 * p.N : p.N * static_cast<double>((p.T + S - 1) / S);
    if (chunks + p.N > 1 << 28) continue;  // chunk slots are counted in 32 bits
    const double cost = 1.7 * clocks(S, chunks) + 12000 + 100 * longest / S;
    if (cost < best) {
      best = cost;
      q.S = S;
    }
  }
  // still few warps: twice as many with half the states
  if (!q.S && q.lanes == 4 && q.spl == 4 && p.N * blocks < 4 * 148) {
    q.lanes = 8;
    q.spl = 2;
  }
  if (q.S) {
    q.per_seq = static_cast<int>((static_cast<int64_t>(p.T) + q.S - 1) / q.S);
    q.slots = p.packed ? p.T / q.S + p.N : p.N * q.per_seq;
  }
  return q;
}

template <typename T, int LANES, int SPL, int TILE, int G>
int launch_scan_ls(ScanArgs a, bool split, cudaStream_t st) {
  constexpr int CW = 64 / LANES;
  constexpr int TL = LANES < 8 ? LANES : SPL < 8 ? 8 : 4;
  constexpr int kSmem = sizeof(ScanSmem<T, LANES, SPL, TILE, TL>);
  a.ch_blocks = (a.dpg + CW - 1) / CW;
  // what every row start of x, dt, z, y and every block of channels is a multiple of
  auto rows = [&](int bytes) {
    const int64_t v = bytes / static_cast<int>(sizeof(T));
    const int64_t all = a.dpg | a.x_bs | a.x_ts | a.dt_bs | a.dt_ts | a.y_bs | a.y_ts |
                        (a.z ? a.z_bs | a.z_ts : 0);
    return v > 0 && all % v == 0 &&
           ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dt) |
             reinterpret_cast<uintptr_t>(a.z) | reinterpret_cast<uintptr_t>(a.y)) % bytes) == 0;
  };
  a.piece = rows(CW * sizeof(T) >= 16 ? 16 : CW * sizeof(T)) ? 2 : rows(4) ? 1 : 0;
  auto states = [&](int v) {
    return (a.n | a.B_bs | a.B_ts | a.B_gs | a.C_bs | a.C_ts | a.C_gs) % v == 0 &&
           ((reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C)) %
            (v * sizeof(T))) == 0;
  };
  a.bc_piece = states(16 / sizeof(T)) ? 2 : states(4) ? 1 : 0;
  const int64_t blocks = static_cast<int64_t>(a.slots) * a.ch_blocks * a.G;
  if (blocks == 0) return PTOF_OK;
  if (blocks > 0x7fffffffLL) return fail(PTOF_EUNSUPPORTED, "ssm_scan: too many blocks");
  const unsigned grid = static_cast<unsigned>(blocks);
  // (a padded state's value is of no use to a record)
  const auto summary = ssm_scan_kernel<T, LANES, SPL, TILE, G, true, false>;
  const auto scan = a.n == LANES * SPL ? ssm_scan_kernel<T, LANES, SPL, TILE, G, false, false>
                                       : ssm_scan_kernel<T, LANES, SPL, TILE, G, false, true>;
  static_assert(kSmem <= 48 * 1024, "no kernel attribute is set");
  if (split) summary<<<grid, 32, kSmem, st>>>(a);
  scan<<<grid, 32, kSmem, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "ssm_scan launch");
}

template <typename T>
int launch_scan_t(const ScanArgs& a, const ScanPlan& q, cudaStream_t st) {
  const bool split = q.S > 0;
  switch (q.lanes * 100 + q.spl) {
    case 402: return launch_scan_ls<T, 4, 2, 16, 4>(a, split, st);
    case 404: return launch_scan_ls<T, 4, 4, 16, 4>(a, split, st);
    case 802: return launch_scan_ls<T, 8, 2, 16, 8>(a, split, st);
    case 408: return launch_scan_ls<T, 4, 8, 16, 4>(a, split, st);
    case 808: return launch_scan_ls<T, 8, 8, 16, 4>(a, split, st);
    default: return launch_scan_ls<T, 16, 8, 16, 4>(a, split, st);
  }
}

template <typename T, int LANES, int ITER>
int launch_step_i(ScanStepArgs a, cudaStream_t st) {
  constexpr int CH = kScanStepThreads / LANES * ITER;
  a.ch_blocks = (a.Dch + CH - 1) / CH;
  const int64_t blocks = static_cast<int64_t>(a.M) * a.ch_blocks;
  if (blocks == 0) return PTOF_OK;
  if (blocks > 0x7fffffffLL) return fail(PTOF_EUNSUPPORTED, "ssm_scan_step: too many blocks");
  const unsigned grid = static_cast<unsigned>(blocks);
  const bool vec = a.n % 4 == 0 && a.s_ss % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.A)) & 15u) == 0;
  a.bc_vec = a.n % 4 == 0 && (a.B_rs | a.B_gs | a.C_rs | a.C_gs) % 4 == 0 &&
             ((reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C)) %
              (4 * sizeof(T))) == 0;
  if (!vec) ssm_scan_step_kernel<T, LANES, ITER, false, true><<<grid, kScanStepThreads, 0, st>>>(a);
  else if (a.n < 4 * LANES) ssm_scan_step_kernel<T, LANES, ITER, true, true><<<grid, kScanStepThreads, 0, st>>>(a);
  else ssm_scan_step_kernel<T, LANES, ITER, true, false><<<grid, kScanStepThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "ssm_scan_step launch");
}

// Four channels a thread where that still leaves a few blocks for every SM.
template <typename T, int LANES>
int launch_step_l(const ScanStepArgs& a, cudaStream_t st) {
  const int64_t blocks = static_cast<int64_t>(a.M) * a.Dch * LANES / (4 * kScanStepThreads);
  return blocks >= 4 * 148 ? launch_step_i<T, LANES, 4>(a, st) : launch_step_i<T, LANES, 1>(a, st);
}

template <typename T>
int launch_step_t(const ScanStepArgs& a, cudaStream_t st) {
  if (a.n <= 4) return launch_step_l<T, 1>(a, st);
  if (a.n <= 8) return launch_step_l<T, 2>(a, st);
  if (a.n <= 16) return launch_step_l<T, 4>(a, st);
  if (a.n <= 32) return launch_step_l<T, 8>(a, st);
  if (a.n <= 64) return launch_step_l<T, 16>(a, st);
  return launch_step_l<T, 32>(a, st);
}

}  // namespace

size_t ssm_scan_ws_bytes(const ptof_ssm_scan_params& p) {
  const ScanPlan q = scan_plan(p);
  if (!q.S) return 0;
  return static_cast<size_t>(q.slots) * p.D * (p.n + 1) * sizeof(float);
}

int launch_ssm_scan(const ptof_ssm_scan_params& p, const void* x, const void* dt, const float* A,
                    const void* B, const void* C, const float* D, const void* z, const float* bias,
                    const int* cu, const float* init, void* y, float* fin, void* ws,
                    cudaStream_t st) {
  if (p.N == 0) {
    if (!p.packed || !p.zero_fill) return PTOF_OK;
    if (p.dtype == PTOF_F32) return launch_zero_tokens<float>(y, p.y_token_stride, p.T, p.D, st);
    return launch_zero_tokens<__half>(y, p.y_token_stride, p.T, p.D, st);  // (bf16's zero too)
  }
  const ScanPlan q = scan_plan(p);
  ScanArgs a{};
  a.x = x; a.dt = dt; a.A = A; a.B = B; a.C = C; a.D = D; a.z = z; a.bias = bias;
  a.init = init; a.cu = cu; a.y = y; a.fin = fin;
  a.ws_h = static_cast<float*>(ws);
  a.ws_dt = a.ws_h + static_cast<size_t>(q.slots) * p.D * p.n;
  a.x_bs = p.x_batch_stride; a.x_ts = p.x_token_stride;
  a.dt_bs = p.dt_batch_stride; a.dt_ts = p.dt_token_stride;
  a.z_bs = p.z_batch_stride; a.z_ts = p.z_token_stride;
  a.y_bs = p.y_batch_stride; a.y_ts = p.y_token_stride;
  a.B_bs = p.B_batch_stride; a.B_ts = p.B_token_stride; a.B_gs = p.B_group_stride;
  a.C_bs = p.C_batch_stride; a.C_ts = p.C_token_stride; a.C_gs = p.C_group_stride;
  a.N = p.N; a.T = p.T; a.Dch = p.D; a.n = p.n; a.G = p.G; a.dpg = p.D / p.G;
  a.softplus = p.softplus; a.fill = p.zero_fill;
  a.S = q.S; a.slots = q.slots; a.per_seq = q.per_seq;
  if (p.dtype == PTOF_F32) return launch_scan_t<float>(a, q, st);
  if (p.dtype == PTOF_F16) return launch_scan_t<__half>(a, q, st);
  return launch_scan_t<__nv_bfloat16>(a, q, st);
}

int launch_ssm_scan_step(const ptof_ssm_scan_step_params& p, const void* x, const void* dt,
                         const float* A, const void* B, const void* C, const float* D,
                         const void* z, const float* bias, const int* slots, float* state, void* y,
                         cudaStream_t st) {
  ScanStepArgs a{};
  a.x = x; a.dt = dt; a.A = A; a.B = B; a.C = C; a.D = D; a.z = z; a.bias = bias;
  a.slots = slots; a.state = state; a.y = y;
  a.x_rs = p.x_row_stride; a.dt_rs = p.dt_row_stride; a.z_rs = p.z_row_stride;
  a.y_rs = p.y_row_stride;
  a.B_rs = p.B_row_stride; a.B_gs = p.B_group_stride;
  a.C_rs = p.C_row_stride; a.C_gs = p.C_group_stride;
  a.s_ss = p.state_slot_stride;
  a.M = p.M; a.S = p.slots; a.Dch = p.D; a.n = p.n; a.dpg = p.D / p.G;
  a.softplus = p.softplus;
  if (p.dtype == PTOF_F32) return launch_step_t<float>(a, st);
  if (p.dtype == PTOF_F16) return launch_step_t<__half>(a, st);
  return launch_step_t<__nv_bfloat16>(a, st);
}

}  // namespace ptof
