// Mamba-3 recurrence, one token of every sequence on a pool of states, updated in place (the loop body of mamba3.cu):
//     phi <- phi + dt theta;  Brot, Crot = R^T(phi) B, C
//     h <- exp(dt A) (h + (1 - lam) dt Brot_prev x_prev) + lam dt Brot x;   y = <h, Crot>
// The state keeps cosine and sine of phi, and the token before as its x and its (unturned) b.
//
// The state is read once and written once, in 16-byte pieces; everything else is small.  Bound: HBM for large batches, launch
// and one chain of load -> sum -> store for small ones.  Heads, 64 channels and 128 states, bf16: 256 tokens of 32 heads 96 to
// 98 us (546 MB: 86 % of the measured copy rate), one token 6.7 us; 61 tokens of 448 channels of 16 states, float32, 8.7 us.
#include "mamba3_serve.cuh"

namespace mxb {
namespace m3s {

using bf16 = __nv_bfloat16;

// V consecutive states: 4, or 2 where N is no multiple of 4 (rows then start on 8 bytes).
template <int V>
__device__ __forceinline__ void load_states(const float* p, float (&e)[V]) {
  if constexpr (V == 4) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
    e[0] = a.x; e[1] = a.y; e[2] = a.z; e[3] = a.w;
  } else {
    const float2 a = __ldcs(reinterpret_cast<const float2*>(p));
    e[0] = a.x; e[1] = a.y;
  }
}
template <int V>
__device__ __forceinline__ void store_states(float* p, const float (&e)[V]) {
  if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(e[0], e[1], e[2], e[3]));
  else __stcs(reinterpret_cast<float2*>(p), make_float2(e[0], e[1]));
}

// Heads: a CTA per (sequence, head); LN lanes along a row of states with NV pieces of V each, 8 / NV consecutive rows a thread at a
// time.  The pieces are requested first; meanwhile two warps work out the scalars and turn b, c and the token before's b, two
// more fetch x.  b_prev has a row a head, so that the CTA which writes it is the only one that reads it.
// Four CTAs an SM (64 registers): 96 us for the 256 tokens, 101 with the three that 80 registers allow; stores that do not stream
// take 35 us more.
constexpr int kStepPieces = 8, kStepRowsMost = 8 * 256;
template <typename IO, int V, int NV>
__global__ void __launch_bounds__(256, 4) m3s_step_heads_kernel(ServeP p, int LN) {
  begin_dependent();
  constexpr int R = kStepPieces / NV;
  __shared__ __align__(16) float s_u[256], s_v[256], s_c[256];
  __shared__ float s_x[kStepRowsMost], s_xp[kStepRowsMost], s_alpha;
  const int seq = blockIdx.x / p.NH, hd = blockIdx.x % p.NH, tid = threadIdx.x, lane = tid & 31;
  const int slot = serve_slot(p, seq);
  if (slot < 0) return;
  const int ln = tid % LN, rg = tid / LN, at_once = 256 / LN * R, npad = LN * V * NV;
  const size_t chan = (size_t)hd * p.P;  // first channel of the head
  float* hp = p.h + ((size_t)slot * p.D + chan) * p.N;
  float st[R][NV][V];
  auto piece = [&](int k) { return (ln + k * LN) * V; };
  auto load = [&](int r0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = r0 + rg * R + r;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (piece(k) < p.N && row < p.P) {
          load_states<V>(hp + (size_t)row * p.N + piece(k), st[r][k]);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) st[r][k][v] = 0.f;
        }
      }
    }
  };
  load(0);
  const IO* X = static_cast<const IO*>(p.x) + (size_t)seq * p.D + chan;
  IO* XP = static_cast<IO*>(p.x_prev) + (size_t)slot * p.D + chan;
  IO* Y = static_cast<IO*>(p.y) + (size_t)seq * p.D + chan;
  auto load_x = [&](int r0, int first, int threads) {  // (one thread reads and then writes a channel's x_prev)
    for (int i = tid - first; i < min(at_once, p.P - r0); i += threads) {
      const IO x = X[r0 + i];
      s_xp[i] = to_f32(XP[r0 + i]);
      s_x[i] = to_f32(x);
      XP[r0 + i] = x;
    }
  };
  const size_t sh = (size_t)seq * p.NH + hd, ph = (size_t)slot * p.NH + hd;
  if (tid < 64) {
    // (b, c and the token before's b are requested in front of the angle: a CTA's chain of loads is what it lives for)
    const int g = hd / (p.NH / p.G);
    const IO *B = static_cast<const IO*>(p.b) + ((size_t)seq * p.G + g) * p.N, *C = static_cast<const IO*>(p.c) + ((size_t)seq * p.G + g) * p.N;
    IO* BP = static_cast<IO*>(p.b_prev) + ph * p.N;
    float2 bs[2], cs[2], bps[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * (tid + 64 * j);
      const bool in = n < p.N;
      bs[j] = in ? load_pair(B + n) : make_float2(0.f, 0.f);
      cs[j] = in ? load_pair(C + n) : make_float2(0.f, 0.f);
      bps[j] = in ? load_pair(BP + n) : make_float2(0.f, 0.f);
    }
    const float dt = m3_softplus(p.dt[sh]), lam = m3_sigmoid(p.lam[sh]), theta = p.theta[sh];
    const float look = (1.f - lam) * dt, gamma = lam * dt;
    const float2 old = p.phase[ph];
    const float2 now = m3_turned(old, m3_unit(m3_turn(dt, theta), m3_taint(dt * theta, 0.f)));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = tid + 64 * j;
      if (k >= npad / 2) break;
      const float2 u = m3_back(bs[j], now), v = m3_back(bps[j], old);
      if (2 * k < p.N) {
        BP[2 * k] = from_f32<IO>(bs[j].x);
        BP[2 * k + 1] = from_f32<IO>(bs[j].y);
      }
      reinterpret_cast<float2*>(s_u)[k] = make_float2(gamma * u.x, gamma * u.y);
      reinterpret_cast<float2*>(s_v)[k] = make_float2(look * v.x, look * v.y);
      reinterpret_cast<float2*>(s_c)[k] = m3_back(cs[j], now);
    }
    asm volatile("bar.sync 1, 64;" ::: "memory");  // (both warps have read the phase)
    if (tid == 0) {
      s_alpha = expf(-expf(p.a_log[hd]) * dt);
      p.phase[ph] = now;
    }
  } else {
    load_x(0, 64, 192);
  }
  __syncthreads();
  const float alpha = s_alpha;
  for (int r0 = 0; r0 < p.P; r0 += at_once) {
    if (r0) {
      __syncthreads();
      load(r0);
      load_x(r0, 0, 256);
      __syncthreads();
    }
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float u[V], v[V], c[V];
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const int n = (piece(k) + j) / 2;
        const float2 a = reinterpret_cast<const float2*>(s_u)[n], b = reinterpret_cast<const float2*>(s_v)[n], d = reinterpret_cast<const float2*>(s_c)[n];
        u[j] = a.x; u[j + 1] = a.y; v[j] = b.x; v[j + 1] = b.y; c[j] = d.x; c[j + 1] = d.y;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = rg * R + r, row = r0 + i;
        const float x = s_x[i], xp = s_xp[i];  // (behind the head's last channel whatever stands there: its rows go nowhere)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          st[r][k][j] = fmaf(x, u[j], alpha * fmaf(xp, v[j], st[r][k][j]));
          acc[r] = fmaf(st[r][k][j], c[j], acc[r]);
        }
        if (piece(k) < p.N && row < p.P) store_states<V>(hp + (size_t)row * p.N + piece(k), st[r][k]);
      }
    }
    if (LN == 32) {  // lane l gets row l & 7
      colsum8(acc, lane);
      const int row = r0 + rg * R + lane;
      if (lane < R && row < p.P) Y[row] = from_f32<IO>(acc[0]);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < LN)
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
      if (ln == 0)
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (r0 + rg * R + r < p.P) Y[r0 + rg * R + r] = from_f32<IO>(acc[r]);
    }
  }
}

// Channels: LN lanes a channel with V states each (V / 2 pairs), 256 / LN channels a CTA.  b_prev, which the channels of a
// group share, is written by a launch behind this one.
template <typename IO, int V>
__global__ void __launch_bounds__(256) m3s_step_channels_kernel(ServeP p, int LN, int blocks) {
  begin_dependent();
  const int seq = blockIdx.x / blocks, ln = threadIdx.x % LN, d = (blockIdx.x % blocks) * (256 / LN) + threadIdx.x / LN;
  const int slot = serve_slot(p, seq);
  if (slot < 0) return;
  const bool live = d < p.D;
  const int dd = live ? d : p.D - 1, g = dd / (p.D / p.G), passes = (p.N + LN * V - 1) / (LN * V);
  const size_t sd = (size_t)seq * p.D + dd, pd = (size_t)slot * p.D + dd;
  const float dt = m3_softplus(p.dt[sd]), lam = m3_sigmoid(p.lam[sd]);
  const float x = to_f32(static_cast<const IO*>(p.x)[sd]), xp = to_f32(static_cast<const IO*>(p.x_prev)[pd]);
  const float ex = (1.f - lam) * dt * xp, gx = lam * dt * x;
  const IO *B = static_cast<const IO*>(p.b) + ((size_t)seq * p.G + g) * p.N, *C = static_cast<const IO*>(p.c) + ((size_t)seq * p.G + g) * p.N;
  const IO* BP = static_cast<const IO*>(p.b_prev) + ((size_t)slot * p.G + g) * p.N;
  float acc = 0.f;
  for (int k = 0; k < passes; ++k) {
    const int n0 = (k * LN + ln) * V;
    if (!live || n0 >= p.N) continue;
    float h[V], a[V];
    load_states<V>(p.h + pd * p.N + n0, h);
    load_states<V>(p.a_log + (size_t)dd * p.N + n0, a);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const int kp = (n0 + i) / 2;
      const size_t at = pd * p.Kp + kp;
      const float2 old = p.phase[at];
      const float theta = p.theta[sd * p.Kp + kp];
      const float2 now = m3_turned(old, m3_unit(m3_turn(dt, theta), m3_taint(dt * theta, 0.f)));
      p.phase[at] = now;
      const float2 u = m3_back(load_pair(B + n0 + i), now), v = m3_back(load_pair(BP + n0 + i), old), c = m3_back(load_pair(C + n0 + i), now);
      h[i] = fmaf(gx, u.x, expf(-expf(a[i]) * dt) * fmaf(ex, v.x, h[i]));
      h[i + 1] = fmaf(gx, u.y, expf(-expf(a[i + 1]) * dt) * fmaf(ex, v.y, h[i + 1]));
      acc = fmaf(h[i], c.x, fmaf(h[i + 1], c.y, acc));
    }
    store_states<V>(p.h + pd * p.N + n0, h);
  }
  for (int o = LN / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (live && ln == 0) {
    static_cast<IO*>(p.y)[sd] = from_f32<IO>(acc);
    static_cast<IO*>(p.x_prev)[pd] = from_f32<IO>(x);  // (behind the shuffles: every lane has read it)
  }
}

// The last token of every sequence into the pool: x too, or only b; and the phase, where a head's slabs have left it beside the
// pool.  grid: sequences.
template <typename IO>
__global__ void __launch_bounds__(256) m3s_tails_kernel(ServeP p, int x_too) {
  begin_dependent();
  const int seq = blockIdx.x, slot = serve_slot(p, seq);
  if (slot < 0) return;
  size_t row = seq;
  if (p.cu) {
    const int a = min(max(p.cu[seq], 0), p.rows), e = min(max(p.cu[seq + 1], a), p.rows);
    if (a == e) return;
    row = (size_t)e - 1;
  }
  const int copies = p.NH ? p.NH : p.G, rep = copies / p.G;
  const IO* B = static_cast<const IO*>(p.b) + row * p.G * p.N;
  IO* BP = static_cast<IO*>(p.b_prev) + (size_t)slot * copies * p.N;
  for (int i = threadIdx.x; i < copies * p.N; i += 256) BP[i] = B[(i / p.N / rep) * p.N + i % p.N];
  if (p.phase_end)
    for (int i = threadIdx.x; i < p.NH; i += 256) p.phase[(size_t)slot * p.NH + i] = p.phase_end[(size_t)seq * p.NH + i];
  if (x_too)
    for (int i = threadIdx.x; i < p.D; i += 256) static_cast<IO*>(p.x_prev)[(size_t)slot * p.D + i] = static_cast<const IO*>(p.x)[row * p.D + i];
}

template <typename IO>
static mxb_status step(const ServeP& p, cudaStream_t st) {
  const int V = p.N % 4 ? 2 : 4;
  int LN = 1;
  if (p.NH) {
    int NV = 1;
    while (LN * V < p.N && LN < 32) LN *= 2;
    while (LN * V * NV < p.N) NV *= 2;
    const dim3 grid((unsigned)(p.S * (size_t)p.NH));
    auto launch = [&](auto kernel) { MXB_LAUNCH("m3s_step_heads_kernel", st, (launch_kernel(kernel, grid, 256, 0, st, p, LN))); };
    if (V == 4) launch(NV == 1 ? m3s_step_heads_kernel<IO, 4, 1> : m3s_step_heads_kernel<IO, 4, 2>);
    else launch(NV == 1 ? m3s_step_heads_kernel<IO, 2, 1> : NV == 2 ? m3s_step_heads_kernel<IO, 2, 2> : m3s_step_heads_kernel<IO, 2, 4>);
    return check_launch("m3s_step_heads");
  }
  while (LN * V < p.N && LN < 32) LN *= 2;
  const int blocks = (p.D + 256 / LN - 1) / (256 / LN);
  const dim3 grid((unsigned)(p.S * (size_t)blocks));
  if (V == 4) MXB_LAUNCH("m3s_step_channels_kernel", st, (launch_kernel(m3s_step_channels_kernel<IO, 4>, grid, 256, 0, st, p, LN, blocks)));
  else MXB_LAUNCH("m3s_step_channels_kernel", st, (launch_kernel(m3s_step_channels_kernel<IO, 2>, grid, 256, 0, st, p, LN, blocks)));
  const mxb_status s = check_launch("m3s_step_channels");
  return s == MXB_OK ? m3serve_tails(p, sizeof(IO) == 4, false, st) : s;
}

}  // namespace m3s

mxb_status m3serve_step(const ServeP& p, bool f32, cudaStream_t st) { return f32 ? m3s::step<float>(p, st) : m3s::step<m3s::bf16>(p, st); }
mxb_status m3serve_tails(const ServeP& p, bool f32, bool x_too, cudaStream_t st) {
  MXB_LAUNCH("m3s_tails_kernel", st,
             (launch_kernel(f32 ? m3s::m3s_tails_kernel<float> : m3s::m3s_tails_kernel<m3s::bf16>, p.S, 256, 0, st, p, x_too ? 1 : 0)));
  return check_launch("m3s_tails");
}

}  // namespace mxb
