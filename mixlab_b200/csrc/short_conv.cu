// Short causal depthwise convolution on a pool of the last inputs: packed prompts, or one token of every sequence.
//     y_t = act(sum_k w[:, k] x_{t-k} + bias),  K <= 4 taps, act: none or x sigmoid(x)
// x_{t-k} in front of a sequence's first row comes from its row of the pool [slots, K-1, D] (the last K-1 inputs, oldest
// first) where the sequence goes on, and is 0 where it starts; the pool then takes the sequence's own last K-1 inputs.
//
// An HBM stream in 16-byte pieces (single elements where D or a pointer does not allow them): a thread owns C channels and
// walks down a run of rows with the last K-1 inputs in registers, four rows requested at a time.  The first K-1 rows of a
// sequence all belong to the run of its first row, so that one thread alone reads and then writes a sequence's pool entry.
//
// 32768 rows of 2048 channels in bf16, 4 taps: 52 us (269 MB: 79 % of the measured copy rate).  One token of 256 sequences of 449
// channels 5.2 us, the call on the host.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace mxb {
namespace sconv {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 128, kAhead = 4;

struct ConvP {
  int rows, S, slots, D, K, silu, run, wvec;
  const void* x;
  const float *w, *bias;
  long long wd, wk;  // strides of w in elements: channel, tap
  const int *cu, *slot;
  const unsigned char* go;
  void *state, *y;
};

template <typename IO, int C>
__device__ __forceinline__ void load_c(const IO* p, float (&e)[C]) {
  if constexpr (C == 1) {
    e[0] = to_f32(*p);
  } else if constexpr (sizeof(IO) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    e[0] = a.x; e[1] = a.y; e[2] = a.z; e[3] = a.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) { e[2 * i] = __low2float(h[i]); e[2 * i + 1] = __high2float(h[i]); }
  }
}
template <typename IO, int C>
__device__ __forceinline__ void store_c(IO* p, const float (&e)[C]) {
  if constexpr (C == 1) {
    *p = from_f32<IO>(e[0]);
  } else if constexpr (sizeof(IO) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(e[0], e[1], e[2], e[3]);
  } else {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(e[2 * i], e[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
}
// C channels of a row as they are in memory.
template <typename IO, int C>
struct Piece {
  using V = std::conditional_t<C == 1, IO, uint4>;
  V raw;
  __device__ __forceinline__ void load(const IO* p) { raw = *reinterpret_cast<const V*>(p); }
  __device__ __forceinline__ void get(float (&e)[C]) const {
    if constexpr (C == 1) e[0] = to_f32(raw);
    else load_c<IO, C>(reinterpret_cast<const IO*>(&raw), e);
  }
};
// (K is known when compiled: a tap that is not there must not meet an infinite input with a weight of 0.)
template <typename IO, int C, int K>
struct Taps {
  static constexpr int H = K > 1 ? K - 1 : 1;  // inputs that are kept
  float w[K][C], bias[C];
  int silu;
  __device__ Taps(const ConvP& p, int ch) : silu(p.silu) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      bias[c] = p.bias ? __ldg(p.bias + ch + c) : 0.f;
      if (K == 4 && p.wvec) {  // the four taps of a channel in one load
        const float4 v = __ldg(reinterpret_cast<const float4*>(p.w) + ch + c);
        w[0][c] = v.x; w[1 % K][c] = v.y; w[2 % K][c] = v.z; w[3 % K][c] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][c] = __ldg(p.w + (ch + c) * p.wd + k * p.wk);
      }
    }
  }
  // hist[j]: the input j + 1 rows in front
  __device__ void apply(const float (&x)[C], const float (&h)[H][C], float (&o)[C]) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v = fmaf(w[0][c], x[c], bias[c]);
#pragma unroll
      for (int k = 1; k < K; ++k) v = fmaf(w[k][c], h[k - 1][c], v);
      o[c] = !silu ? v : sizeof(IO) == 4 ? v / (1.f + expf(-v)) : __fdividef(v, 1.f + __expf(-v));
    }
  }
};
template <int H, int C>
__device__ __forceinline__ void push(float (&h)[H][C], const float (&x)[C]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int j = H - 1; j > 0; --j) h[j][c] = h[j - 1][c];
    h[0][c] = x[c];
  }
}
__device__ __forceinline__ int slot_of(const ConvP& p, int seq) {
  const int s = p.slot ? __ldg(p.slot + seq) : seq;
  return s >= 0 && s < p.slots ? s : -1;
}
// Pool entry of a slot: hist[j] = its row K-2-j, 0 where there is no slot or the sequence starts anew.
template <typename IO, int C, int K, int H>
__device__ __forceinline__ void load_hist(const ConvP& p, int slot, bool go, int ch, float (&h)[H][C]) {
#pragma unroll
  for (int j = 0; j < H; ++j) {
    if (slot >= 0 && go && j < K - 1) {
      load_c<IO, C>(static_cast<const IO*>(p.state) + ((size_t)slot * (K - 1) + K - 2 - j) * p.D + ch, h[j]);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) h[j][c] = 0.f;
    }
  }
}
template <typename IO, int C, int K, int H>
__device__ __forceinline__ void store_hist(const ConvP& p, int slot, int ch, const float (&h)[H][C]) {
#pragma unroll
  for (int j = 0; j < H; ++j)
    if (j < K - 1) store_c<IO, C>(static_cast<IO*>(p.state) + ((size_t)slot * (K - 1) + K - 2 - j) * p.D + ch, h[j]);
}

// grid (ceil(D / C / 128), runs)
template <typename IO, int C, int K>
__global__ void __launch_bounds__(kThreads, 4) sconv_prefill_kernel(ConvP p) {
  begin_dependent();
  using T = Taps<IO, C, K>;
  const int lane = threadIdx.x & 31, ch = (blockIdx.x * kThreads + threadIdx.x) * C;
  const int r0 = blockIdx.y * p.run, r1 = (int)min((long long)r0 + p.run, (long long)p.rows);
  auto bound = [&](int s) { return min(max(__ldg(p.cu + s), 0), p.rows); };
  // the sequence of row r0: as many as end at or in front of it
  int seq = 0;
  for (int s0 = 0; s0 < p.S; s0 += 32) {
    const int s = s0 + lane;
    const int n = __popc(__ballot_sync(0xffffffffu, s < p.S && bound(s + 1) <= r0));
    seq += n;
    if (n < 32) break;
  }
  if (ch >= p.D) return;
  const IO* __restrict__ x = static_cast<const IO*>(p.x) + ch;
  IO* __restrict__ y = static_cast<IO*>(p.y) + ch;
  const T taps(p, ch);
  float h[T::H][C];
  for (; seq < p.S; ++seq) {
    const int begin = bound(seq), end = max(bound(seq + 1), begin);
    if (begin >= r1) break;
    if (begin == end) continue;
    int t = begin, stop;
    if (begin >= r0) {  // the sequence's first row is this run's: its pool entry, and the first K - 1 rows wherever they end
      const int slot = slot_of(p, seq);
      const bool go = p.go && __ldg(p.go + seq);
      load_hist<IO, C, K>(p, slot, go, ch, h);
      if (slot >= 0) {
        float kept[T::H][C];
#pragma unroll
        for (int j = 0; j < T::H; ++j) {
          const int row = end - 1 - j;  // the input j + 1 rows in front of the end
          if (row >= begin) {
            load_c<IO, C>(x + (size_t)row * p.D, kept[j]);
          } else {
            const int old = begin - 1 - row;  // 0 .. K - 2
#pragma unroll
            for (int c = 0; c < C; ++c) kept[j][c] = old == 0 ? h[0][c] : old == 1 ? h[1 % T::H][c] : h[2 % T::H][c];
          }
        }
        store_hist<IO, C, K>(p, slot, ch, kept);
      }
      stop = min(end, max(r1, begin + K - 1));
    } else {
      t = max(r0, begin + K - 1);
      if (t >= end) continue;
      stop = min(end, r1);
#pragma unroll
      for (int j = 0; j < T::H; ++j) {
        if (j < K - 1 && t < stop) {
          load_c<IO, C>(x + (size_t)(t - 1 - j) * p.D, h[j]);
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) h[j][c] = 0.f;
        }
      }
    }
    // four rows are requested while the four before are worked on
    Piece<IO, C> next[kAhead], now[kAhead];
    auto request = [&](int at) {
#pragma unroll
      for (int r = 0; r < kAhead; ++r) next[r].load(x + (size_t)min(at + r, stop - 1) * p.D);
    };
    request(t);
    for (; t < stop; t += kAhead) {
#pragma unroll
      for (int r = 0; r < kAhead; ++r) now[r] = next[r];
      if (t + kAhead < stop) request(t + kAhead);
#pragma unroll
      for (int r = 0; r < kAhead; ++r) {
        float v[C], o[C];
        now[r].get(v);
        taps.apply(v, h, o);
        if (t + r < stop) store_c<IO, C>(y + (size_t)(t + r) * p.D, o);
        push(h, v);
      }
    }
  }
}
// grid (ceil(D / C / 128), sequences)
template <typename IO, int C, int K>
__global__ void __launch_bounds__(kThreads) sconv_step_kernel(ConvP p) {
  begin_dependent();
  using T = Taps<IO, C, K>;
  const int seq = blockIdx.y, ch = (blockIdx.x * kThreads + threadIdx.x) * C;
  const int slot = slot_of(p, seq);
  if (ch >= p.D || slot < 0) return;
  float h[T::H][C], x[C], o[C];
  load_hist<IO, C, K>(p, slot, true, ch, h);
  load_c<IO, C>(static_cast<const IO*>(p.x) + (size_t)seq * p.D + ch, x);
  const T taps(p, ch);
  taps.apply(x, h, o);
  store_c<IO, C>(static_cast<IO*>(p.y) + (size_t)seq * p.D + ch, o);
  push(h, x);
  store_hist<IO, C, K>(p, slot, ch, h);
}

template <typename IO, int C, int K>
static mxb_status launch_k(ConvP p, cudaStream_t st) {
  const unsigned cols = (p.D / C + kThreads - 1) / kThreads;
  if (p.cu) {
    // CTAs for whole rounds of what the GPU holds at once (four an SM by the kernel's registers), runs of 8 to 128 rows (rounds of
    // two or eight an SM: 57.8 and 59.3 us for 57.5)
    const size_t at_once = 148 * 4, work = (size_t)cols * p.rows, rounds = (work + at_once * 128 - 1) / (at_once * 128);
    int run = (int)std::max<size_t>(8, (work + at_once * rounds - 1) / (at_once * rounds));
    while ((p.rows + run - 1) / run > 65535) run *= 2;
    p.run = run;
    MXB_LAUNCH("sconv_prefill_kernel", st, (launch_kernel(sconv_prefill_kernel<IO, C, K>, dim3(cols, (p.rows + run - 1) / run), kThreads, 0, st, p)));
  } else {
    MXB_LAUNCH("sconv_step_kernel", st, (launch_kernel(sconv_step_kernel<IO, C, K>, dim3(cols, p.S), kThreads, 0, st, p)));
  }
  return check_launch("sconv");
}
template <typename IO, int C>
static mxb_status launch(const ConvP& p, cudaStream_t st) {
  switch (p.K) {
    case 1: return launch_k<IO, C, 1>(p, st);
    case 2: return launch_k<IO, C, 2>(p, st);
    case 3: return launch_k<IO, C, 3>(p, st);
    default: return launch_k<IO, C, 4>(p, st);
  }
}

}  // namespace sconv

// cu: packed prompts; null: one token of each of S sequences.
mxb_status short_conv(const mxb_short_conv_desc* d, const void* x, const float* w, const float* bias, const int32_t* cu,
                      const int32_t* slots, const unsigned char* go, void* state, void* y, cudaStream_t st) {
  sconv::ConvP p{d->rows, d->S, d->slots, d->D, d->K, d->activation == MXB_ACT_SILU, 0, 0, x, w, bias, d->w_stride_d, d->w_stride_k, cu, slots, go, state, y};
  p.wvec = d->K == 4 && d->w_stride_k == 1 && d->w_stride_d == 4 && reinterpret_cast<uintptr_t>(w) % 16 == 0;
  // (whole pieces 57.5 us for 32768 rows of 2048 channels, single elements, which any row allows, 99.5)
  const bool wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(state)) % 16 == 0 &&
                    d->D % (d->io_dtype == MXB_F32 ? 4 : 8) == 0;
  if (d->io_dtype == MXB_F32) return wide ? sconv::launch<float, 4>(p, st) : sconv::launch<float, 1>(p, st);
  return wide ? sconv::launch<sconv::bf16, 8>(p, st) : sconv::launch<sconv::bf16, 1>(p, st);
}

}  // namespace mxb
