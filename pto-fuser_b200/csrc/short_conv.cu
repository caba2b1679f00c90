// Short causal depthwise convolution, for prompts and for single tokens:
//   y[t, d] = act(bias[d] + sum_j w[d, j] x[t - W + 1 + j, d]),  j = 0 .. W - 1,
// where inputs before a sequence's first token come from its initial state [W - 1, D]
// (zeros without one) and the state after it holds its last W - 1 inputs.
//
// Bound by memory: every input is read and every output written once, and each channel
// needs W products a token. A thread owns a few channels (one 16-byte load where rows allow) and
// a strip of tokens; the last W - 1 inputs stay in registers, so only a strip's first
// W - 1 rows are read twice (from L2: the neighbouring strip of the same block reads them
// at the same time). The rows ahead are on their way to shared memory, each thread's to a
// place of its own, so that 6 to 8 of them a thread are in flight without registers.
#include <algorithm>
#include <initializer_list>

#include "capi_internal.h"
#include "mixer_ops.cuh"

namespace ptof {

namespace {

struct ConvArgs {
  const void* x;
  const void* w;
  const void* bias;
  const int* cu;
  const void* init;
  void* y;
  void* fin;
  int64_t x_bs, x_ts, y_bs, y_ts;  // batch / token strides in elements
  int N, T, D;                     // sequences, tokens (of each, or packed), channels
  int w_dtype, w_wide, silu, fill;
  int tok;                         // tokens of a strip
  int strips;                      // strips of one batch row
  int lanes;                       // threads along the channels
  int ch_blocks;                   // blocks along the channels
  int64_t main_blocks;             // blocks before the final-state blocks
};

// A thread's channels are K vectors of VEC, `gap` channels apart: one 16-byte vector, or, where
// rows are not aligned to that, one pair or two channels that lie a warp's width apart (so that
// a warp's loads of either are neighbours). All arithmetic is on pairs of fp32 values.
template <typename T, int VEC, int K>
__device__ __forceinline__ void unpack(const Pack<T, VEC> (&p)[K], f32x2 (&f)[VEC * K / 2]) {
#pragma unroll
  for (int e = 0; e < VEC * K; e += 2)
    f[e / 2] = pack2(to_f32<T>(p[e / VEC].v[e % VEC]), to_f32<T>(p[(e + 1) / VEC].v[(e + 1) % VEC]));
}

template <typename T, int VEC, int K>
__device__ __forceinline__ void round_to(const f32x2 (&f)[VEC * K / 2], Pack<T, VEC> (&p)[K]) {
#pragma unroll
  for (int e = 0; e < VEC * K; e += 2) {
    const float2 u = unpack2(f[e / 2]);
    p[e / VEC].v[e % VEC] = from_f32<T>(u.x);
    p[(e + 1) / VEC].v[(e + 1) % VEC] = from_f32<T>(u.y);
  }
}

constexpr int kConvThreads = 128;
constexpr int kConvGroup = 2;  // rows of one asynchronous copy group
constexpr int kConvRing = 4;   // groups in flight a thread
constexpr int kConvAhead = 4;  // rows of a register buffer

// All taps of a thread's channels as pairs of channels: w[j][i] holds tap j of pair i. The taps
// of a channel are neighbours in memory; `wide` says that they begin on 16 bytes. Channels
// from D on get the taps of channel c.
template <typename TW, int VEC, int K, int W>
__device__ __forceinline__ void ld_taps(const void* wp, const void* bp, bool wide, int c, int gap, int D,
                                        f32x2 (&w)[W][VEC * K / 2], f32x2 (&bias)[VEC * K / 2]) {
  constexpr int E = VEC * K, V = 16 / sizeof(TW);  // channels, values of a load
  TW v[E * W], u[E];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int ci = c + (c + i * gap < D ? i * gap : 0);
    const TW* p = static_cast<const TW*>(wp) + static_cast<int64_t>(ci) * W;
    if (VEC * W % V == 0 && wide) {
#pragma unroll
      for (int g = 0; g < VEC * W / V; ++g) {
        const Pack<TW, V> k = ld_pack<TW, V>(p + g * V);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i * VEC * W + g * V + j] = k.v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC * W; ++j) v[i * VEC * W + j] = p[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[i * VEC + j] = bp ? static_cast<const TW*>(bp)[ci + j] : from_f32<TW>(0.f);
  }
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    bias[e / 2] = pack2(to_f32<TW>(u[e]), to_f32<TW>(u[e + 1]));
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e / 2] = pack2(to_f32<TW>(v[e * W + j]), to_f32<TW>(v[(e + 1) * W + j]));
  }
}

// Row p of sequence n (first token s): the input itself, or the initial state's row.
template <typename T, int VEC, int W>
__device__ __forceinline__ Pack<T, VEC> conv_row(const ConvArgs& a, const T* x, int n, int s, int p,
                                                 int c) {
  if (p >= s) return ld_pack<T, VEC>(x + static_cast<int64_t>(p) * a.x_ts + c);
  if (a.init)
    return ld_pack<T, VEC>(static_cast<const T*>(a.init) +
                           (static_cast<int64_t>(n) * (W - 1) + (W - 1 + p - s)) * a.D + c);
  Pack<T, VEC> z;
#pragma unroll
  for (int i = 0; i < VEC; ++i) z.v[i] = from_f32<T>(0.f);
  return z;
}

template <typename T, int VEC>
constexpr int blocks_per_sm() { return VEC * sizeof(T) == 16 ? 4 : 7; }

// 16-byte vectors come through the ring: 16384 x 12288 bf16 takes 141 to 152 us on different
// cards, 0.88 to 0.82 of the copy bandwidth. Smaller vectors come through registers, up to
// 2 kConvAhead rows ahead, and are bound by the instructions for each: 5640 x 8191 bf16 takes
// 76 us where 8192 channels take 43 (184 with one channel a thread and no rows ahead; 8 rows a
// buffer or four channels a thread, and fewer blocks for their registers, 94).
template <typename T, int VEC, int K, int W>
__global__ void __launch_bounds__(kConvThreads, blocks_per_sm<T, VEC>())
short_conv_kernel(const ConvArgs a) {
  constexpr int V2 = VEC * K / 2;  // channel pairs
  if (blockIdx.x >= a.main_blocks) {
    // final states: one vector of one of the last W - 1 inputs per thread
    const int nv = a.D / VEC;
    const int64_t i = (blockIdx.x - a.main_blocks) * kConvThreads + threadIdx.x;
    const int64_t row = i / nv;
    const int c = static_cast<int>(i - row * nv) * VEC;
    const int n = static_cast<int>(row / (W - 1)), r = static_cast<int>(row % (W - 1));
    if (n >= a.N) return;
    int s = 0, e = a.T;
    const T* x = static_cast<const T*>(a.x);
    if (a.cu) seq_bounds(a.cu, n, a.T, s, e);
    else x += n * a.x_bs;
    st_pack<T, VEC>(static_cast<T*>(a.fin) + row * a.D + c,
                    conv_row<T, VEC, W>(a, x, n, s, e - (W - 1) + r, c));
    return;
  }
  const int tb = static_cast<int>(blockIdx.x / a.ch_blocks);
  const int cb = static_cast<int>(blockIdx.x - static_cast<int64_t>(tb) * a.ch_blocks);
  const int lane = threadIdx.x % a.lanes;
  const int64_t strip = static_cast<int64_t>(tb) * (kConvThreads / a.lanes) + threadIdx.x / a.lanes;
  const int gap = a.lanes * VEC, c = cb * gap * K + lane * VEC;
  const int b = static_cast<int>(strip / a.strips);
  if (c >= a.D || b >= (a.cu ? 1 : a.N)) return;
  int t = static_cast<int>(strip - static_cast<int64_t>(b) * a.strips) * a.tok;
  const int t1 = min(t + a.tok, a.T);
  const T* x = static_cast<const T*>(a.x) + b * a.x_bs;
  T* y = static_cast<T*>(a.y) + b * a.y_bs;

  f32x2 w[W][V2], bias[V2];
  if (a.w_dtype == Elem<T>::code) ld_taps<T, VEC, K, W>(a.w, a.bias, a.w_wide, c, gap, a.D, w, bias);
  else ld_taps<float, VEC, K, W>(a.w, a.bias, a.w_wide, c, gap, a.D, w, bias);
  auto in = [&](int i) { return K == 1 || c + i * gap < a.D; };
  // a thread's own rows on their way: copied without registers, read by the same thread
  constexpr bool RING = VEC * sizeof(T) == 16;
  __shared__ __align__(16) Pack<T, VEC> ring[RING ? kConvRing * kConvGroup : 1][kConvThreads];

  while (t < t1) {
    int n = b, s = 0, e = a.T;
    if (a.cu) {
      // the last sequence that starts at or before t
      int lo = -1, hi = a.N;  // cu[lo] <= t < cu[hi + 1] with cu[-1] = -inf
      while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (a.cu[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      n = lo;
      if (n < 0 || n >= a.N) {  // tokens of no sequence
        int stop = n < 0 ? min(max(a.cu[0], t + 1), t1) : t1;
        for (; t < stop; ++t)
          if (a.fill) {
            Pack<T, VEC> z;
#pragma unroll
            for (int i = 0; i < VEC; ++i) z.v[i] = from_f32<T>(0.f);
#pragma unroll
            for (int i = 0; i < K; ++i)
              if (in(i)) st_pack<T, VEC>(y + static_cast<int64_t>(t) * a.y_ts + c + i * gap, z);
          }
        continue;
      }
      s = min(max(a.cu[n], 0), t);
      e = min(max(a.cu[n + 1], t + 1), a.T);
    }
    const int stop = min(e, t1);
    f32x2 win[W - 1][V2];  // inputs t - W + 1 .. t - 1
    auto load_window = [&]() {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        Pack<T, VEC> row[K];
#pragma unroll
        for (int i = 0; i < K; ++i)
          row[i] = conv_row<T, VEC, W>(a, x, n, s, t - (W - 1) + j, c + (in(i) ? i * gap : 0));
        unpack<T, VEC, K>(row, win[j]);
      }
    };
    auto step = [&](const Pack<T, VEC> (&row)[K], int to) {
      f32x2 cur[V2];
      unpack<T, VEC, K>(row, cur);
      Pack<T, VEC> out[K];
#pragma unroll
      for (int i = 0; i < V2; ++i) {
        f32x2 v = bias[i];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) v = fma2(w[j][i], win[j][i], v);
        v = fma2(w[W - 1][i], cur[i], v);
        if (a.silu) v = silu2(v);
        const float2 u = unpack2(v);
        out[2 * i / VEC].v[2 * i % VEC] = from_f32<T>(u.x);
        out[(2 * i + 1) / VEC].v[(2 * i + 1) % VEC] = from_f32<T>(u.y);
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
        win[W - 2][i] = cur[i];
      }
#pragma unroll
      for (int i = 0; i < K; ++i)
        if (in(i)) st_pack<T, VEC>(y + static_cast<int64_t>(to) * a.y_ts + c + i * gap, out[i]);
    };
    if (RING) {
      const T* next = x + static_cast<int64_t>(t) * a.x_ts + c;
      auto ask = [&](int group, int from) {  // the rows of one group, as far as there are any
#pragma unroll
        for (int k = 0; k < kConvGroup; ++k) {
          if (from + k < stop) copy_async<16>(&ring[group * kConvGroup + k][threadIdx.x], next);
          next += a.x_ts;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int k = 0; k < kConvRing; ++k) ask(k, t + k * kConvGroup);
      load_window();
      int group = 0;
      for (; t < stop; t += kConvGroup) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kConvRing - 1) : "memory");
        Pack<T, VEC> row[kConvGroup][K];
#pragma unroll
        for (int k = 0; k < kConvGroup; ++k) row[k][0] = ring[group * kConvGroup + k][threadIdx.x];
        if (t + kConvGroup <= stop) {
#pragma unroll
          for (int k = 0; k < kConvGroup; ++k) step(row[k], t + k);
        } else {
#pragma unroll
          for (int k = 0; k < kConvGroup; ++k)
            if (t + k < stop) step(row[k], t + k);
        }
        ask(group, t + kConvRing * kConvGroup);  // the rows there have been used
        group = group + 1 == kConvRing ? 0 : group + 1;
      }
      t = stop;
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
      // two buffers by turns: no copies between them, which would wait for the loads
      Pack<T, VEC> first[kConvAhead][K], second[kConvAhead][K];
      auto fetch = [&](Pack<T, VEC> (&rows)[kConvAhead][K], int from) {
#pragma unroll
        for (int k = 0; k < kConvAhead; ++k) {
          const T* q = x + static_cast<int64_t>(min(from + k, stop - 1)) * a.x_ts + c;
#pragma unroll
          for (int i = 0; i < K; ++i) rows[k][i] = ld_pack<T, VEC>(q + (in(i) ? i * gap : 0));
        }
      };
      auto use = [&](const Pack<T, VEC> (&rows)[kConvAhead][K], int from) {
        if (from + kConvAhead <= stop) {
#pragma unroll
          for (int k = 0; k < kConvAhead; ++k) step(rows[k], from + k);
        } else {
#pragma unroll
          for (int k = 0; k < kConvAhead; ++k)
            if (from + k < stop) step(rows[k], from + k);
        }
      };
      fetch(first, t);
      fetch(second, t + kConvAhead);
      load_window();
      for (; t < stop; t += 2 * kConvAhead) {
        use(first, t);
        fetch(first, t + 2 * kConvAhead);
        use(second, t + kConvAhead);
        fetch(second, t + 3 * kConvAhead);
      }
      t = stop;
    }
  }
}

struct ConvStepArgs {
  const void* x;
  void* state;
  const void* w;
  const void* bias;
  const int* slots;
  void* y;
  int64_t x_rs, y_rs, s_ss, s_ts;  // row strides of x and y, slot and tap strides of the state
  int M, S, D;                     // rows, slots, channels
  int w_dtype, w_wide, silu;
  int ch_blocks;
};

constexpr int kConvStepThreads = 128;

// One row and 128 threads' channels per block; the state is shifted by one in place. Bound by
// memory for many rows and by its latency for few. 512 x 12288 takes 29 us in bf16 and 38 in f32
// (its bytes need 16 and 31), without slots 23 and 33: every block looks through all the slots for
// rows that share its own, and reads the taps of its channels again. Four channels a thread in every type: with 16-byte vectors of 16-bit
// types the registers leave room for half the threads, which took 34 us.
template <typename T, int VEC, int K, int W>
__global__ void __launch_bounds__(kConvStepThreads) short_conv_step_kernel(const ConvStepArgs a) {
  constexpr int V2 = VEC * K / 2, gap = kConvStepThreads * VEC;
  const int m = static_cast<int>(blockIdx.x / a.ch_blocks);
  const int c = static_cast<int>(blockIdx.x % a.ch_blocks) * gap * K + threadIdx.x * VEC;
  const int slot = a.slots ? a.slots[m] : m;
  const bool live = c < a.D, used = slot >= 0 && slot < a.S;
  const T* x = static_cast<const T*>(a.x) + c;
  T* y = static_cast<T*>(a.y) + c;
  T* st = static_cast<T*>(a.state) + (used ? slot : 0) * a.s_ss + c;
  auto in = [&](int i) { return K == 1 || c + i * gap < a.D; };
  auto load = [&](const T* p, Pack<T, VEC> (&row)[K]) {
#pragma unroll
    for (int i = 0; i < K; ++i) row[i] = ld_pack<T, VEC>(p + (in(i) ? i * gap : 0));
  };
  auto store = [&](T* p, const Pack<T, VEC> (&row)[K]) {
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (in(i)) st_pack<T, VEC>(p + i * gap, row[i]);
  };
  Pack<T, VEC> win[W][K];
  f32x2 w[W][V2], bias[V2];
  if (used && live) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) load(st + j * a.s_ts, win[j]);
    load(x + m * a.x_rs, win[W - 1]);
    if (a.w_dtype == Elem<T>::code) ld_taps<T, VEC, K, W>(a.w, a.bias, a.w_wide, c, gap, a.D, w, bias);
    else ld_taps<float, VEC, K, W>(a.w, a.bias, a.w_wide, c, gap, a.D, w, bias);
  }
  bool later = false;
  if (a.slots && a.M > 1) {
    const SlotUse u = slot_use(a.slots, a.M, m, slot);
    if (used && u.earlier) return;
    later = u.later;
  }
  if (!live) return;
  if (!used) {  // a padding row: no state, its output is zero
    Pack<T, VEC> z[K];
#pragma unroll
    for (int i = 0; i < VEC * K; ++i) z[i / VEC].v[i % VEC] = from_f32<T>(0.f);
    store(y + m * a.y_rs, z);
    return;
  }
  for (int r = m;;) {
    f32x2 o[V2], v[W][V2];
    Pack<T, VEC> out[K];
#pragma unroll
    for (int j = 0; j < W; ++j) unpack<T, VEC, K>(win[j], v[j]);
#pragma unroll
    for (int i = 0; i < V2; ++i) {
      o[i] = bias[i];
#pragma unroll
      for (int j = 0; j < W; ++j) o[i] = fma2(w[j][i], v[j][i], o[i]);
      if (a.silu) o[i] = silu2(o[i]);
    }
    round_to<T, VEC, K>(o, out);
    store(y + r * a.y_rs, out);
    if (!later) break;
    for (++r; r < a.M && a.slots[r] != slot; ++r) {}
    if (r >= a.M) break;
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < K; ++i) win[j][i] = win[j + 1][i];
    load(x + r * a.x_rs, win[W - 1]);
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store(st + j * a.s_ts, win[j + 1]);
}

bool wide(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int VEC, int K>
int launch_conv_w(ConvArgs a, int width, cudaStream_t st) {
  const int nv = (a.D + VEC * K - 1) / (VEC * K);  // threads along the channels
  a.w_wide = wide(a.w);
  a.lanes = 32;
  while (a.lanes > 1 && a.lanes / 2 >= nv) a.lanes /= 2;
  const int per_block = kConvThreads / a.lanes;  // strips of a block
  a.ch_blocks = (nv + a.lanes - 1) / a.lanes;
  const int rows = a.cu ? 1 : a.N;
  // Strips of at most 72 tokens, as long as the fewest full waves of blocks allow: 64 tokens
  // or halves of it, whatever the waves, took 20 us for 2048 x 4096 where this takes 16.
  const int64_t wave = 148LL * blocks_per_sm<T, VEC>() * per_block, across = static_cast<int64_t>(rows) * a.ch_blocks;
  const int64_t waves = std::max<int64_t>(1, (across * ((a.T + 71) / 72) + wave - 1) / wave);
  const int64_t cuts = std::max<int64_t>(1, wave * waves / std::max<int64_t>(1, across));
  a.tok = std::max(4, static_cast<int>((a.T + cuts - 1) / cuts));
  a.strips = (a.T + a.tok - 1) / a.tok;
  const int64_t strips = static_cast<int64_t>(a.strips) * rows;
  a.main_blocks = (strips + per_block - 1) / per_block * a.ch_blocks;
  const int64_t fin = a.fin ? static_cast<int64_t>(a.N) * (width - 1) * (a.D / VEC) : 0;
  const int64_t blocks = a.main_blocks + (fin + kConvThreads - 1) / kConvThreads;
  if (blocks == 0) return PTOF_OK;
  if (blocks > 0x7fffffffLL) return fail(PTOF_EUNSUPPORTED, "short_conv: too many blocks");
  const unsigned g = static_cast<unsigned>(blocks);
  if (width == 2) short_conv_kernel<T, VEC, K, 2><<<g, kConvThreads, 0, st>>>(a);
  else if (width == 3) short_conv_kernel<T, VEC, K, 3><<<g, kConvThreads, 0, st>>>(a);
  else short_conv_kernel<T, VEC, K, 4><<<g, kConvThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "short_conv launch");
}

// Vectors of V elements fit all rows of sizes and strides `multiples` and the bases p.
bool fits(int V, int esize, std::initializer_list<int64_t> multiples, std::initializer_list<const void*> p) {
  for (int64_t m : multiples)
    if (m % V) return false;
  for (const void* q : p)
    if (reinterpret_cast<uintptr_t>(q) % (V * esize)) return false;
  return true;
}

template <typename T>
int launch_conv_t(const ConvArgs& a, int width, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto ok = [&](int v) {
    return fits(v, sizeof(T), {a.D, a.x_bs, a.x_ts, a.y_bs, a.y_ts}, {a.x, a.y, a.init, a.fin});
  };
  if (ok(V)) return launch_conv_w<T, V, 1>(a, width, st);
  return ok(2) ? launch_conv_w<T, 2, 1>(a, width, st) : launch_conv_w<T, 1, 2>(a, width, st);
}

template <typename T, int VEC, int K>
int launch_conv_step_w(ConvStepArgs a, int width, cudaStream_t st) {
  const int nv = (a.D + VEC * K - 1) / (VEC * K);
  a.w_wide = wide(a.w);
  a.ch_blocks = (nv + kConvStepThreads - 1) / kConvStepThreads;
  const int64_t blocks = static_cast<int64_t>(a.M) * a.ch_blocks;
  if (blocks == 0) return PTOF_OK;
  if (blocks > 0x7fffffffLL) return fail(PTOF_EUNSUPPORTED, "short_conv_step: too many blocks");
  const unsigned g = static_cast<unsigned>(blocks);
  if (width == 2) short_conv_step_kernel<T, VEC, K, 2><<<g, kConvStepThreads, 0, st>>>(a);
  else if (width == 3) short_conv_step_kernel<T, VEC, K, 3><<<g, kConvStepThreads, 0, st>>>(a);
  else short_conv_step_kernel<T, VEC, K, 4><<<g, kConvStepThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PTOF_OK : cuda_fail(e, "short_conv_step launch");
}

template <typename T>
int launch_conv_step_t(const ConvStepArgs& a, int width, cudaStream_t st) {
  auto ok = [&](int v) {
    return fits(v, sizeof(T), {a.D, a.x_rs, a.y_rs, a.s_ss, a.s_ts}, {a.x, a.y, a.state});
  };
  if (ok(4)) return launch_conv_step_w<T, 4, 1>(a, width, st);
  return ok(2) ? launch_conv_step_w<T, 2, 1>(a, width, st) : launch_conv_step_w<T, 1, 2>(a, width, st);
}

}  // namespace

int launch_short_conv(const ptof_short_conv_params& p, const void* x, const void* w,
                      const void* bias, const int* cu, const void* init, void* y, void* fin,
                      cudaStream_t st) {
  ConvArgs a{};
  a.x = x; a.w = w; a.bias = bias; a.cu = cu; a.init = init; a.y = y; a.fin = fin;
  a.x_bs = p.x_batch_stride; a.x_ts = p.x_token_stride;
  a.y_bs = p.y_batch_stride; a.y_ts = p.y_token_stride;
  a.N = p.N; a.T = p.T; a.D = p.D;
  a.w_dtype = p.w_dtype; a.silu = p.silu; a.fill = p.zero_fill;
  if (p.dtype == PTOF_F32) return launch_conv_t<float>(a, p.width, st);
  if (p.dtype == PTOF_F16) return launch_conv_t<__half>(a, p.width, st);
  return launch_conv_t<__nv_bfloat16>(a, p.width, st);
}

int launch_short_conv_step(const ptof_short_conv_step_params& p, const void* x, void* state,
                           const void* w, const void* bias, const int* slots, void* y,
                           cudaStream_t st) {
  ConvStepArgs a{};
  a.x = x; a.state = state; a.w = w; a.bias = bias; a.slots = slots; a.y = y;
  a.x_rs = p.x_row_stride; a.y_rs = p.y_row_stride;
  a.s_ss = p.state_slot_stride; a.s_ts = p.state_tap_stride;
  a.M = p.M; a.S = p.slots; a.D = p.D;
  a.w_dtype = p.w_dtype; a.silu = p.silu;
  if (p.dtype == PTOF_F32) return launch_conv_step_t<float>(a, p.width, st);
  if (p.dtype == PTOF_F16) return launch_conv_step_t<__half>(a, p.width, st);
  return launch_conv_step_t<__nv_bfloat16>(a, p.width, st);
}

}  // namespace ptof
