// Mamba-3 scan of packed prompts on a pool of states, step by step: float32 and every shape, both parameter layouts (the
// recurrence and the state are mamba3_step.cu's).
//
// What is carried from step to step is G_t = h_t + (1 - lam_{t+1}) dt_{t+1} Brot_t x_t (0 for the look-ahead behind the last
// step), so that a step needs nothing of the one before:
//     h_t = alpha_t G_{t-1} + lam_t dt_t Brot_t x_t;   y_t = <h_t, Crot_t>;   G_t = alpha_t G_{t-1} + e_t Brot_t x_t
//     e_t = lam_t dt_t + (1 - lam_{t+1}) dt_{t+1}
// A walk is one chain of steps, and prompts that are few and long would leave the GPU to a few of them.  Sequences longer than
// L steps are cut into segments (walk_segment()): a first pass walks every segment but a sequence's last from a zero state,
// a second one chains what they add, H <- decay H + added, and the walk that writes y starts from the results.
//
// Head layout: decay and angle are a head's own, so turning commutes with the decay and each segment counts its angle from
// its own start; the state between two segments is the turned-on one, R(phi) h.  Channel layout: the two states of a pair
// decay at rates of their own, so angles count from the sequence's start: the first pass leaves what a segment adds as the factors
// of cosine and sine of its first angle, which the chain knows.
#include <algorithm>
#include <type_traits>

#include "mamba3_serve.cuh"
#include "packed.cuh"

namespace mxb {
namespace m3k {

using bf16 = __nv_bfloat16;
enum Mode { kOut, kEnds };

// ------------------------------------------------------------------ heads
// A CTA per (segment, head, slab of channels): LN lanes along a row of states, NV pieces of 4 states a lane, R rows a thread,
// all in registers.  16 steps at a time are made ready in shared memory: scalars by one warp, then b and c turned back and x; what
// they are made of is requested 16 steps earlier.  Bound: shared memory and the issue of instructions.  Float32, 8 heads of 64
// channels, 128 states: 16 prompts of 2048 rows 911 us, one of 16384 rows 407 us (cut in 37), one of 37 rows 24 us.
// Angles sum dt as float32 (each rounded by 2^-24 of itself, as in the scan over [B, T] batches): n steps that turn by a radian are
// off by about n 2^-24 at most.
constexpr int kW = 16;
constexpr int kRowsMost = 64;  // channels of a slab
struct HeadSmem {
  float alpha[kW], gs[kW], e[kW], gamma[kW];
  float2 unit[kW];
};
template <typename IO, int NV, int R, Mode MODE>
__global__ void __launch_bounds__(256) m3k_heads_kernel(ServeP p, int LN) {
  begin_dependent();
  extern __shared__ __align__(16) float smem[];
  __shared__ HeadSmem sc;
  __shared__ int s_turn;
  __shared__ float s_taint, s_dt;
  const int heads = p.NH * p.slabs, tid = threadIdx.x, hd = blockIdx.x % heads / p.slabs, slab = blockIdx.x % p.slabs;
  const Piece q = find_piece<MODE == kEnds ? kInner : kPieces>(p, blockIdx.x / heads, p.L);
  const int piece = q.base + q.seg;
  if (!q.ok || piece >= p.cuts) return;
  const int ln = tid % LN, rg = tid / LN, rows_at_once = 256 / LN, npad = LN * 4 * NV;
  const int per = (p.P + p.slabs - 1) / p.slabs, p0 = slab * per, np = min(per, p.P - p0);  // this CTA's channels of the head
  const size_t chan = (size_t)hd * p.P + p0;
  float *su = smem, *scv = su + kW * npad, *sx = scv + kW * npad, *sy = sx + kW * kRowsMost;
  const int slot = serve_slot(p, q.seq), g = hd / (p.NH / p.G);
  const bool from_state = MODE == kOut && q.segs == 1 && slot >= 0 && serve_goes_on(p, q.seq);
  const size_t ph = (size_t)(slot < 0 ? 0 : slot) * p.NH + hd;
  const float A = -expf(p.a_log[hd]);
  float2 start = make_float2(1.f, 0.f);
  if (MODE == kOut && q.segs > 1) start = p.start[(size_t)piece * p.NH + hd];
  else if (from_state) start = p.phase[ph];

  auto row_of = [&](int r) { return rg + r * rows_at_once; };
  auto n_of = [&](int k) { return (ln + k * LN) * 4; };
  f2 G[R][NV][2];
  const float look0 = from_state ? serve_look(p, (size_t)q.first * p.NH + hd, true) : 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int row = row_of(r), n = n_of(k) + i;
        float2 v = make_float2(0.f, 0.f);
        if (row < np && n < p.N) {
          if (MODE == kOut && q.segs > 1) {
            v = *reinterpret_cast<const float2*>(p.ends + ((size_t)piece * p.D + chan + row) * p.N + n);
          } else if (from_state) {
            v = m3_on(*reinterpret_cast<const float2*>(p.h + ((size_t)slot * p.D + chan + row) * p.N + n), start);
            const float2 b = load_pair(static_cast<const IO*>(p.b_prev) + ph * p.N + n);
            const float w = look0 * to_f32(static_cast<const IO*>(p.x_prev)[(size_t)slot * p.D + chan + row]);
            v.x = fmaf(w, b.x, v.x);
            v.y = fmaf(w, b.y, v.y);
          }
        }
        G[r][k][i / 2] = pack2(v.x, v.y);
      }
  if (tid == 0) { s_turn = 0; s_taint = 0.f; s_dt = 0.f; }
  // What 16 steps are made of, as read; requested while the 16 in front are walked.
  constexpr int XR = kW * kRowsMost / 256, NB = NV == 4 ? 8 : 4;
  struct { float dt, lam, theta, dt1, lam1, x[XR]; float2 b[NB], c[MODE == kOut ? NB : 1]; } raw;
  const int bs = tid / 16, bj = tid % 16;  // 16 threads a step
  auto request = [&](int t0) {
    if (tid < kW) {
      const int t = t0 + tid;
      const bool in = t < q.last, next = in && t + 1 < q.end;
      const size_t at = (size_t)(in ? t : q.first) * p.NH + hd;
      raw.dt = p.dt[at];
      raw.lam = p.lam[at];
      raw.theta = p.theta[at];
      raw.dt1 = next ? p.dt[at + p.NH] : -INFINITY;
      raw.lam1 = next ? p.lam[at + p.NH] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < XR; ++k) {
      const int i = tid + k * 256, s = i / kRowsMost, r = i % kRowsMost;
      raw.x[k] = r < np && t0 + s < q.last ? to_f32(static_cast<const IO*>(p.x)[(size_t)(t0 + s) * p.D + chan + r]) : 0.f;
    }
    const bool in = t0 + bs < q.last;
    const size_t row = ((size_t)(in ? t0 + bs : q.first) * p.G + g) * p.N;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int n = 2 * (bj + 16 * k);
      raw.b[k] = in && n < p.N ? load_pair(static_cast<const IO*>(p.b) + row + n) : make_float2(0.f, 0.f);
      if (MODE == kOut) raw.c[MODE == kOut ? k : 0] = in && n < p.N ? load_pair(static_cast<const IO*>(p.c) + row + n) : make_float2(0.f, 0.f);
    }
  };
  request(q.first);
  for (int t0 = q.first; t0 < q.last; t0 += kW) {
    __syncthreads();
    if (tid < 32) {  // scalars of the steps; the angle runs on from block to block
      const bool in = tid < kW && t0 + tid < q.last;
      const float dt = m3_softplus(raw.dt), lam = m3_sigmoid(raw.lam);
      const float look = (1.f - m3_sigmoid(raw.lam1)) * m3_softplus(raw.dt1);
      int turn = in ? m3_turn(dt, raw.theta) : 0;
      float taint = in ? m3_taint(dt * raw.theta, 0.f) : 0.f, sum = in ? dt : 0.f;
#pragma unroll
      for (int o = 1; o < kW; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, turn, o);
        const float b = __shfl_up_sync(0xffffffffu, taint, o), c = __shfl_up_sync(0xffffffffu, sum, o);
        if (tid >= o) { turn += a; taint += b; sum += c; }
      }
      turn += s_turn;
      taint += s_taint;
      sum += s_dt;
      __syncwarp();
      if (tid == kW - 1) { s_turn = turn; s_taint = taint; s_dt = sum; }
      if (tid < kW) {
        sc.alpha[tid] = in ? expf(A * dt) : 1.f;
        sc.gamma[tid] = in ? lam * dt : 0.f;
        sc.e[tid] = in ? lam * dt + look : 0.f;
        sc.unit[tid] = m3_unit(turn, taint);
      }
    }
#pragma unroll
    for (int k = 0; k < XR; ++k) sx[tid + k * 256] = raw.x[k];
    __syncthreads();
    {
      const float2 a = sc.unit[bs];
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const int pair = bj + 16 * k;
        if (2 * pair >= npad) break;
        reinterpret_cast<float2*>(su + bs * npad)[pair] = m3_back(raw.b[k], a);
        if (MODE == kOut) {
          const float2 b = raw.b[k], c = raw.c[MODE == kOut ? k : 0];
          dot = fmaf(b.x, c.x, fmaf(b.y, c.y, dot));  // <Brot, Crot> = <b, c>
          reinterpret_cast<float2*>(scv + bs * npad)[pair] = m3_back(c, a);
        }
      }
      if (MODE == kOut) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (bj == 0) sc.gs[bs] = sc.gamma[bs] * dot + a.x * 0.f;  // (an angle that is not finite has to reach y here too)
      }
    }
    __syncthreads();
    request(t0 + kW);
    const int steps = min(kW, q.last - t0);
    for (int s = 0; s < steps; ++s) {
      const float alpha = sc.alpha[s], e = sc.e[s];
      f2 u[NV][2], c[NV][2];
      float acc[R];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(su + s * npad + n_of(k));
        u[k][0] = a.x; u[k][1] = a.y;
        if (MODE == kOut) {
          const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(scv + s * npad + n_of(k));
          c[k][0] = b.x; c[k][1] = b.y;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = row_of(r);
        const f2 ex = dup2(row < np ? e * sx[s * kRowsMost + row] : 0.f), keep = dup2(alpha);
        f2 sum = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f2 v = mul2(keep, G[r][k][i]);
            if (MODE == kOut) sum = mad2(c[k][i], v, sum);
            G[r][k][i] = mad2(ex, u[k][i], v);
          }
        acc[r] = sum2(sum);
      }
      if (MODE == kOut) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (o < LN)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (ln == 0)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int row = row_of(r);
            if (row < np) sy[s * kRowsMost + row] = fmaf(sc.gs[s], sx[s * kRowsMost + row], acc[r]);
          }
      }
    }
    if (MODE == kOut) {
      __syncthreads();
      for (int i = tid; i < steps * np; i += 256) {
        const int s = i / np, r = i - s * np;
        static_cast<IO*>(p.y)[(size_t)(t0 + s) * p.D + chan + r] = from_f32<IO>(sy[s * kRowsMost + r]);
      }
    }
  }
  __syncthreads();
  const float2 ran = m3_unit(s_turn, s_taint);
  if (MODE == kEnds && tid == 0 && slab == 0) {
    p.turn[(size_t)piece * p.NH + hd] = s_turn;
    p.dsum[(size_t)piece * p.NH + hd] = s_dt + s_taint;
  }
  if (MODE == kOut && (q.seg != q.segs - 1 || slot < 0)) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int row = row_of(r), n = n_of(k) + i;
        if (row >= np || n >= p.N) continue;
        const float2 v = unpack2(G[r][k][i / 2]);
        if (MODE == kEnds) *reinterpret_cast<float2*>(p.ends + ((size_t)piece * p.D + chan + row) * p.N + n) = m3_on(v, ran);
        else *reinterpret_cast<float2*>(p.h + ((size_t)slot * p.D + chan + row) * p.N + n) = m3_back(v, start);
      }
  // (the slabs of a head all read its phase and b_prev; with more than one they are written behind this launch)
  if (MODE == kOut && p.slabs == 1) {
    if (tid == 0) p.phase[ph] = m3_turned(start, ran);
    serve_tail<IO>(p, q.end - 1, slot, hd, g, 256);
  } else if (MODE == kOut && tid == 0 && slab == 0) {
    p.phase_end[(size_t)q.seq * p.NH + hd] = m3_turned(start, ran);
  }
}

// What the segments of a sequence start from.  grid (sequences that can be longer than L, blocks of pairs): a thread per state
// pair of the channels walks over the segments; what kAhead segments add is requested at a time.
constexpr int kAhead = 8;
__global__ void __launch_bounds__(256) m3k_heads_chain_kernel(ServeP p, bool bf16_io) {
  begin_dependent();
  const Piece q = find_piece<kCut>(p, blockIdx.x, p.L);
  if (!q.ok || q.base + q.segs > p.cuts) return;
  const int slot = serve_slot(p, q.seq);
  const bool go = slot >= 0 && serve_goes_on(p, q.seq);
  const size_t pairs = (size_t)p.D * p.Kp;
  for (size_t i = blockIdx.y * (size_t)256 + threadIdx.x; i < pairs; i += gridDim.y * (size_t)256) {
    const int d = (int)(i / p.Kp), k = (int)(i % p.Kp), hd = d / p.P;
    float2 at = make_float2(1.f, 0.f), v = make_float2(0.f, 0.f);
    if (go) {
      const size_t ph = (size_t)slot * p.NH + hd;
      at = p.phase[ph];
      v = m3_on(reinterpret_cast<const float2*>(p.h)[((size_t)slot * p.D + d) * p.Kp + k], at);
      const float w = serve_look(p, (size_t)q.begin * p.NH + hd, true) *
                      (bf16_io ? to_f32(static_cast<const bf16*>(p.x_prev)[(size_t)slot * p.D + d]) : static_cast<const float*>(p.x_prev)[(size_t)slot * p.D + d]);
      const float2 b = bf16_io ? load_pair(static_cast<const bf16*>(p.b_prev) + ph * p.N + 2 * k) : load_pair(static_cast<const float*>(p.b_prev) + ph * p.N + 2 * k);
      v.x = fmaf(w, b.x, v.x);
      v.y = fmaf(w, b.y, v.y);
    }
    const float A = -expf(p.a_log[hd]);
    const bool first = k == 0 && d % p.P == 0;
    float2* e = reinterpret_cast<float2*>(p.ends) + ((size_t)q.base * p.D + d) * p.Kp + k;
    for (int s0 = 0; s0 < q.segs; s0 += kAhead) {
      const int n = min(kAhead, q.segs - s0), adds = min(kAhead, q.segs - 1 - s0);
      float2 add[kAhead];
      float sum[kAhead];
      int turn[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const size_t sh = (size_t)(q.base + s0 + s) * p.NH + hd;
        add[s] = s < adds ? e[s * pairs] : make_float2(0.f, 0.f);
        sum[s] = s < adds ? p.dsum[sh] : 0.f;
        turn[s] = s < adds ? p.turn[sh] : 0;
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (s >= n) break;
        e[s * pairs] = v;
        if (first) p.start[(size_t)(q.base + s0 + s) * p.NH + hd] = at;
        const float2 ran = m3_unit(turn[s], m3_taint(sum[s], 0.f)), r = m3_on(v, ran);  // (dsum carries the angle's taint)
        const float L = expf(A * sum[s]);
        v.x = fmaf(L, r.x, add[s].x);
        v.y = fmaf(L, r.y, add[s].y);
        if (first) at = m3_turned(at, ran);
      }
      e += kAhead * pairs;
    }
  }
}

// ------------------------------------------------------------------ channels
// LPC lanes a channel with PR state pairs each, 8 steps at a time: a lane works out softplus and sigmoid of its own steps and
// hands them round through shared memory; theta and the rows of b and c come by cp.async 8 steps ahead, by 16-byte pieces that a
// warp shares or each lane's own elements into its own places (no barrier of the CTA, no registers while they are under way).
//
// What bounds it is the issue of instructions, a sine, a cosine and two exponentials a state pair and step (4003 steps x 448
// channels of 16 states: 14 M of them, 62 instructions each in the first pass over what is cut, 44 us, and 80 in the second, 52
// us).  So two steps' angles go through packed polynomials, the two states of a pair are packed, and y of 8 steps is added over 8
// lanes by halving exchanges.
constexpr int kC = 8;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Cosine and sine of two angles in 2^-32 turns: the nearest half turn by integers, minimax polynomials of degree 9 and 10 on what
// is left, at most pi / 2 (fitted by least squares with Lawson's weights; with the coefficients rounded to float32 1.7e-8 and
// 5.0e-9, with the roundings of a call 2.2e-7, 4e-8 in the mean).  A nearest quarter turn would halve the roundings, and costs a
// dozen selections more.
__device__ __forceinline__ void unit2(int t0, int t1, float2& u0, float2& u1) {
  const int half0 = (t0 + 0x40000000) & 0x80000000, half1 = (t1 + 0x40000000) & 0x80000000;
  const f2 r = mul2(pack2((float)(t0 ^ half0), (float)(t1 ^ half1)), dup2(1.4629180792671596e-9f));  // 2 pi / 2^32
  const f2 r2 = mul2(r, r);
  f2 ps = dup2(2.600054585855105e-06f);
  ps = mad2(ps, r2, dup2(-0.00019806614727713168f));
  ps = mad2(ps, r2, dup2(0.008333017118275166f));
  ps = mad2(ps, r2, dup2(-0.16666656732559204f));
  ps = mad2(mul2(ps, r2), r, r);
  f2 pc = dup2(-2.6077103143506974e-07f);
  pc = mad2(pc, r2, dup2(2.4761886379565112e-05f));
  pc = mad2(pc, r2, dup2(-0.00138884037733078f));
  pc = mad2(pc, r2, dup2(0.04166664183139801f));
  pc = mad2(pc, r2, dup2(-0.5f));
  pc = mad2(pc, r2, dup2(1.f));
  const float2 s = unpack2(ps), c = unpack2(pc);
  auto by = [](float v, int half) { return __int_as_float(__float_as_int(v) ^ half); };
  u0 = make_float2(by(c.x, half0), by(s.x, half0));
  u1 = make_float2(by(c.y, half1), by(s.y, half1));
}
// m3_turn of two steps, with dt theta rounded once, as dt is.  (With this, the decays by ex2.approx and lambda by the fast
// division y of float32 prompts of 4003 rows is 3.7e-7 off in the mean; elementary operations with angles in 64 bits: 1.2e-7.  The
// nearest whole turn by adding 1.5 x 2^23: good for up to 2^22 turns a step, where a float32 is no angle any more.)
__device__ __forceinline__ void turn2(f2 p, int& t0, int& t1) {
  const f2 hi = dup2(0.15915493667125702f), t = mul2(p, hi), low = mad2(p, dup2(-6.420638243e-09f), mad2(p, dup2(-0.15915493667125702f), t));
  const f2 whole = add2(add2(t, dup2(12582912.f)), dup2(-12582912.f));
  const float2 f = unpack2(mul2(mad2(low, dup2(-1.f), mad2(whole, dup2(-1.f), t)), dup2(4294967296.f)));
  t0 = __float2int_rn(f.x);
  t1 = __float2int_rn(f.y);
}
// What the lanes have requested of 8 steps.  WHOLE: a warp's channels are of one group and their pairs fill its lanes, so that its
// rows of theta, b and c are 16-byte pieces that the warp shares; otherwise every lane requests its own elements.
template <typename IO, int PR, int LPC, Mode MODE, bool WHOLE>
struct Ahead {
  using Two = std::conditional_t<sizeof(IO) == 4, float2, uint32_t>;  // a pair of b or c
  static constexpr int kRow = PR * (WHOLE ? 4 * LPC : 128), kR = WHOLE ? LPC : 128;  // pairs of a step; of r
  float theta[kC][PR][128];
  Two b[kC][kRow], c[MODE == kOut ? kC : 1][kRow];
};
// What a step is made of, two steps side by side: dt, e x, gamma x of each; a channel's 8 steps (padded: other banks).
struct __align__(16) Two { float dt[2], ex[2], gx[2], pad[2]; };
struct __align__(16) Steps { Two two[kC / 2]; float pad[4]; };
template <int BYTES>
__device__ __forceinline__ void copy_ahead(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_ahead_16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ float2 pair_of(float2 v) { return v; }
__device__ __forceinline__ float2 pair_of(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }

template <typename IO, int PR, int LPC, Mode MODE, bool WHOLE>
__global__ void __launch_bounds__(128) m3k_channels_kernel(ServeP p) {
  begin_dependent();
  constexpr int OWN = (kC + LPC - 1) / LPC, CPB = 128 / LPC;
  const int lane = threadIdx.x & 31, sl = lane % LPC, base = lane - sl;
  const int d_raw = blockIdx.y * CPB + threadIdx.x / LPC;
  const bool live = d_raw < p.D;
  const int d = live ? d_raw : p.D - 1;
  const Piece q = find_piece<MODE == kEnds ? kInner : kPieces>(p, blockIdx.x, p.L);
  const int piece = q.base + q.seg;
  if (!q.ok || piece >= p.cuts) return;
  const int slot = serve_slot(p, q.seq), g = d / (p.D / p.G);
  const bool from_state = MODE == kOut && q.segs == 1 && slot >= 0 && serve_goes_on(p, q.seq);
  const size_t sd = (size_t)(slot < 0 ? 0 : slot) * p.D + d, row = (size_t)piece * p.D + d;
  f2 G[PR], H[MODE == kEnds ? PR : 1];  // the state; kEnds: its factors of the cosine and of the sine of the angle at the start
  float a[PR][2], taint[PR], dsum = 0.f;
  int turn[PR], kp[PR];
  bool has[PR];
#pragma unroll
  for (int r = 0; r < PR; ++r) {
    kp[r] = sl + r * LPC;
    has[r] = WHOLE || kp[r] < p.Kp;
    G[r] = 0;
    if (MODE == kEnds) H[MODE == kEnds ? r : 0] = 0;
    a[r][0] = a[r][1] = taint[r] = 0.f;
    turn[r] = 0;
    if (!has[r]) continue;
    a[r][0] = -expf(p.a_log[(size_t)d * p.N + 2 * kp[r]]) * 1.4426950408889634f;
    a[r][1] = -expf(p.a_log[(size_t)d * p.N + 2 * kp[r] + 1]) * 1.4426950408889634f;
    if (MODE == kOut && q.segs > 1) {
      const float2 v = reinterpret_cast<const float2*>(p.ends)[row * p.Kp + kp[r]];
      G[r] = pack2(v.x, v.y);
      turn[r] = p.turn[row * p.Kp + kp[r]];
      taint[r] = p.spoil[row * p.Kp + kp[r]];
    } else if (from_state) {
      const float2 unit = p.phase[sd * p.Kp + kp[r]], v = reinterpret_cast<const float2*>(p.h)[sd * p.Kp + kp[r]];
      turn[r] = serve_turn(unit);
      taint[r] = m3_taint(unit.x, m3_taint(unit.y, 0.f));
      const float2 b = m3_back(load_pair(static_cast<const IO*>(p.b_prev) + ((size_t)slot * p.G + g) * p.N + 2 * kp[r]), unit);
      const float w = serve_look(p, (size_t)q.first * p.D + d, true) * to_f32(static_cast<const IO*>(p.x_prev)[sd]);
      G[r] = pack2(fmaf(w, b.x, v.x), fmaf(w, b.y, v.y));
    }
  }
  extern __shared__ __align__(16) unsigned char raw[];
  using Block = Ahead<IO, PR, LPC, MODE, WHOLE>;
  Block* ahead = reinterpret_cast<Block*>(raw);
  Steps& made = reinterpret_cast<Steps*>(ahead + 2)[threadIdx.x / LPC];
  const int bc_at = WHOLE ? (threadIdx.x / 32) * PR * LPC + sl : threadIdx.x;  // this lane's first pair in a row of b or c
  const float* theta_at = p.theta + ((size_t)q.first * p.D + d) * p.Kp + sl;
  const IO *b_at = static_cast<const IO*>(p.b) + ((size_t)q.first * p.G + g) * p.N + 2 * sl, *c_at = static_cast<const IO*>(p.c) + ((size_t)q.first * p.G + g) * p.N + 2 * sl;
  const size_t theta_row = (size_t)p.D * p.Kp, bc_row = (size_t)p.G * p.N;
  const bool pairs = ((reinterpret_cast<uintptr_t>(p.b) | reinterpret_cast<uintptr_t>(p.c)) & (2 * sizeof(IO) - 1)) == 0;
  const size_t bc_bytes = bc_row * sizeof(IO), theta_bytes = theta_row * sizeof(float);
  // WHOLE: this lane's 16-byte pieces, the first of theta and what follows it; pieces of a step's row of b or c
  const int warp_d = min((int)(blockIdx.y * CPB + (threadIdx.x & 96) / LPC), p.D - 32 / LPC);
  const int theta_s = lane / 8 / PR, theta_r = lane / 8 % PR, theta_i = lane % 8 * 4;
  const float* theta_16 = p.theta + ((size_t)(q.first + theta_s) * p.D + warp_d) * p.Kp + theta_r * 32 + theta_i;
  constexpr int PB = 2 * LPC * PR * (int)sizeof(IO) / 16 + !WHOLE, ALL = kC * PB, PJ = (ALL + 31) / 32;
  const char *b_16[PJ], *c_16[PJ];
  if constexpr (WHOLE)
#pragma unroll
    for (int j = 0; j < PJ; ++j) {
      const int i = lane + 32 * j;
      b_16[j] = reinterpret_cast<const char*>(b_at - 2 * sl) + i / PB * bc_bytes + i % PB * 16;
      c_16[j] = reinterpret_cast<const char*>(c_at - 2 * sl) + i / PB * bc_bytes + i % PB * 16;
    }
  auto request_whole = [&](int left, Block& to, auto all) {  // of as many steps as are left, or all 8
    constexpr bool FULL = decltype(all)::value;
    float* dst = &to.theta[theta_s][theta_r][(threadIdx.x & 96) + theta_i];
#pragma unroll
    for (int j = 0; j < 2 * PR; ++j) {
      const int s = j * 4 / PR;
      const bool in = FULL || theta_s + s < left;
      copy_ahead_16(dst + s * PR * 128, in ? theta_16 + s * theta_row : p.theta, in);
    }
#pragma unroll
    for (int j = 0; j < PJ; ++j) {
      const int i = lane + 32 * j, s = i / PB, to_pair = (threadIdx.x / 32) * PR * LPC + i % PB * (8 / (int)sizeof(IO));
      if (ALL < 32 && i >= ALL) break;
      const bool in = FULL || s < left;
      copy_ahead_16(&to.b[s][to_pair], in ? b_16[j] : static_cast<const char*>(p.b), in);
      if (MODE == kOut) copy_ahead_16(&to.c[MODE == kOut ? s : 0][to_pair], in ? c_16[j] : static_cast<const char*>(p.c), in);
      b_16[j] += kC * bc_bytes;
      c_16[j] += kC * bc_bytes;
    }
    theta_16 += kC * theta_row;
  };
  auto request = [&](int t0, Block& to) {  // zeros for steps behind the last and lanes without a pair
    const int steps = min(kC, q.last - t0);
    if constexpr (WHOLE) {
      if (steps == kC) request_whole(kC, to, std::true_type{});
      else request_whole(steps, to, std::false_type{});
      asm volatile("cp.async.commit_group;" ::: "memory");
      return;
    }
    const char *th = reinterpret_cast<const char*>(theta_at), *b = reinterpret_cast<const char*>(b_at), *c = reinterpret_cast<const char*>(c_at);
    if (pairs && steps == kC) {
#pragma unroll
      for (int r = 0; r < PR; ++r) {
        if (!has[r]) continue;
        const char *th_r = th + r * LPC * sizeof(float), *b_r = b + 2 * r * LPC * sizeof(IO), *c_r = c + 2 * r * LPC * sizeof(IO);
#pragma unroll
        for (int s = 0; s < kC; ++s, th_r += theta_bytes, b_r += bc_bytes, c_r += bc_bytes) {
          copy_ahead<4>(&to.theta[s][r][threadIdx.x], th_r);
          copy_ahead<2 * sizeof(IO)>(&to.b[s][bc_at + r * Block::kR], b_r);
          if (MODE == kOut) copy_ahead<2 * sizeof(IO)>(&to.c[s][bc_at + r * Block::kR], c_r);
        }
      }
    } else {
#pragma unroll 1
      for (int s = 0; s < kC; ++s)
#pragma unroll 1
        for (int r = 0; r < PR; ++r) {
          const bool in = sl + r * LPC < p.Kp && s < steps;
          const IO *bs = reinterpret_cast<const IO*>(b + s * bc_bytes) + 2 * r * LPC, *cs = reinterpret_cast<const IO*>(c + s * bc_bytes) + 2 * r * LPC;
          IO *db = reinterpret_cast<IO*>(&to.b[s][bc_at + r * Block::kR]), *dc = reinterpret_cast<IO*>(&to.c[MODE == kOut ? s : 0][bc_at + r * Block::kR]);
          to.theta[s][r][threadIdx.x] = in ? reinterpret_cast<const float*>(th + s * theta_bytes)[r * LPC] : 0.f;
          for (int k = 0; k < 2; ++k) {
            db[k] = in ? bs[k] : from_f32<IO>(0.f);
            if (MODE == kOut) dc[k] = in ? cs[k] : from_f32<IO>(0.f);
          }
        }
    }
    theta_at += kC * theta_row;
    b_at += kC * bc_row;
    c_at += kC * bc_row;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (!WHOLE && !has[PR - 1]) {  // (a lane without a pair reads zeros)
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll 1
      for (int s = 0; s < kC; ++s)
        for (int r = 0; r < PR; ++r) {
          ahead[k].theta[s][r][threadIdx.x] = 0.f;
          ahead[k].b[s][bc_at + r * Block::kR] = {};
          if (MODE == kOut) ahead[k].c[MODE == kOut ? s : 0][bc_at + r * Block::kR] = {};
        }
  }
  // dt, lambda, x of this lane's steps of a block: as read, and what is made of them
  struct Raw { float dt[OWN], lam[OWN], x[OWN]; } next;
  struct Made { float dt[OWN], gamma[OWN], look[OWN], x[OWN]; } own;
  const float *dt_at = p.dt + (size_t)(q.first + sl) * p.D + d, *lam_at = p.lam + (size_t)(q.first + sl) * p.D + d;
  const IO* x_at = static_cast<const IO*>(p.x) + (size_t)(q.first + sl) * p.D + d;
  auto request_scalars = [&](int t0) {
#pragma unroll
    for (int o = 0; o < OWN; ++o) {  // (the step behind the segment's last counts, for its weight of that one)
      const bool in = sl + o * LPC < kC && t0 + sl + o * LPC < q.end;
      next.dt[o] = in ? dt_at[(size_t)o * LPC * p.D] : -INFINITY;
      next.lam[o] = in ? lam_at[(size_t)o * LPC * p.D] : 0.f;
      next.x[o] = in ? to_f32(x_at[(size_t)o * LPC * p.D]) : 0.f;
    }
    dt_at += (size_t)kC * p.D;
    lam_at += (size_t)kC * p.D;
    x_at += (size_t)kC * p.D;
  };
  auto make_scalars = [&](int t0) {
    Made m;
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const float dt = fmaxf(next.dt[o], 0.f) + log1pf(expf(-fabsf(next.dt[o]))), lam = __fdividef(1.f, 1.f + expf(-next.lam[o]));
      const bool in = t0 + sl + o * LPC < q.last;
      m.look[o] = (1.f - lam) * dt;
      m.dt[o] = in ? dt : 0.f;
      m.gamma[o] = in ? lam * dt : 0.f;
      m.x[o] = in ? next.x[o] : 0.f;
    }
    return m;
  };
  request(q.first, ahead[0]);
  request_scalars(q.first);
  own = make_scalars(q.first);
  request_scalars(q.first + kC);
  IO* y_at = static_cast<IO*>(p.y) + (size_t)(q.first + sl) * p.D + d;  // (of 8 lanes and more)
  int buf = 0;
  for (int t0 = q.first; t0 < q.last; t0 += kC, buf ^= 1) {
    const int steps = min(kC, q.last - t0);
    __syncwarp();  // (what the warp shares has been read)
    const Made behind = make_scalars(t0 + kC);
    if (MODE == kEnds)
#pragma unroll
      for (int o = 0; o < OWN; ++o) dsum += own.dt[o];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {  // e: lambda dt and what the step behind gives this one
      const int s = sl + o * LPC;
      const float a = __shfl_sync(0xffffffffu, own.look[o], base + (sl + 1) % LPC);
      const float b = o + 1 < OWN ? __shfl_sync(0xffffffffu, own.look[o + 1 < OWN ? o + 1 : 0], base) : __shfl_sync(0xffffffffu, behind.look[0], base);
      if (LPC > kC && sl >= kC) continue;
      Two& to = made.two[s / 2];
      to.dt[s & 1] = own.dt[o];
      to.ex[s & 1] = (own.gamma[o] + (sl + 1 < (LPC < kC ? LPC : kC) ? a : b)) * own.x[o];
      if (MODE == kOut) to.gx[s & 1] = own.gamma[o] * own.x[o];
    }
    own = behind;
    if (t0 + kC < q.last) {
      request_scalars(t0 + 2 * kC);
      request(t0 + kC, ahead[buf ^ 1]);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    const Block& now = ahead[buf];
    float ys[kC];
#pragma unroll
    for (int s = 0; s < kC; s += 2) {  // two steps' angles together
      const float4 of = *reinterpret_cast<const float4*>(&made.two[s / 2]);
      const float2 gxs = MODE == kOut ? *reinterpret_cast<const float2*>(made.two[s / 2].gx) : make_float2(0.f, 0.f);
      const float dt[2] = {of.x, of.y}, ex[2] = {of.z, of.w}, gx[2] = {gxs.x, gxs.y};
      float acc[2] = {0.f, 0.f};
#pragma unroll
      for (int r = 0; r < PR; ++r) {
        const f2 angles = mul2(pack2(dt[0], dt[1]), pack2(now.theta[s][r][threadIdx.x], now.theta[s + 1][r][threadIdx.x]));
        int t1, t2;
        turn2(angles, t1, t2);
        t1 += turn[r];
        t2 += t1;
        const float n1 = m3_taint(unpack2(angles).x, taint[r]), n2 = m3_taint(unpack2(angles).y, n1);
        float2 unit[2];
        unit2(t1, t2, unit[0], unit[1]);
        acc[0] += n1;  // (an angle that is not finite: y by hand, the state at the block's end)
        acc[1] += n2;
        turn[r] = t2;
        taint[r] = n2;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 b = pair_of(now.b[s + k][bc_at + r * Block::kR]);
          const float2 decay = unpack2(mul2(pack2(a[r][0], a[r][1]), dup2(dt[k])));
          const f2 kept = pack2(ex2(decay.x), ex2(decay.y)), v = mul2(kept, G[r]), e2 = dup2(ex[k]);
          if (MODE == kOut) {
            const float2 u2 = m3_back(b, unit[k]), c = m3_back(pair_of(now.c[MODE == kOut ? s + k : 0][bc_at + r * Block::kR]), unit[k]);
            const f2 u = pack2(u2.x, u2.y);
            const float2 h = unpack2(mad2(dup2(gx[k]), u, v));
            acc[k] = fmaf(h.x, c.x, fmaf(h.y, c.y, acc[k]));
            G[r] = mad2(e2, u, v);
          } else {
            const float2 u = m3_back(b, unit[k]);
            const int h = MODE == kEnds ? r : 0;
            const f2 w = mul2(kept, H[h]);
            G[r] = mad2(e2, pack2(u.x, u.y), v);
            H[h] = mad2(e2, pack2(u.y, -u.x), w);
          }
        }
      }
      ys[s] = acc[0];
      ys[s + 1] = acc[1];
    }
#pragma unroll
    for (int r = 0; r < PR; ++r) G[r] = add2(G[r], dup2(taint[r]));
    if (MODE == kOut) {
      if (LPC >= 8) {  // lane sl gets the sum of step sl & 7
        colsum8_step<4, 4>(ys, lane);
        colsum8_step<2, 2>(ys, lane);
        colsum8_step<1, 1>(ys, lane);
#pragma unroll
        for (int o = 8; o < LPC; o <<= 1) ys[0] += __shfl_xor_sync(0xffffffffu, ys[0], o);
        if (live && sl < steps && sl < kC) *y_at = from_f32<IO>(ys[0]);
        y_at += (size_t)kC * p.D;
      } else {
#pragma unroll
        for (int s = 0; s < kC; ++s) {
#pragma unroll
          for (int o = LPC / 2; o > 0; o >>= 1) ys[s] += __shfl_xor_sync(0xffffffffu, ys[s], o);
          if (live && sl == s % LPC && s < steps) static_cast<IO*>(p.y)[(size_t)(t0 + s) * p.D + d] = from_f32<IO>(ys[s]);
        }
      }
    }
  }
  if (MODE == kEnds) dsum = group_sum<LPC>(dsum);
  if (!live) return;
  if (MODE == kEnds && sl == 0) p.dsum[row] = dsum;
  if (MODE == kOut && (q.seg != q.segs - 1 || slot < 0)) return;
#pragma unroll
  for (int r = 0; r < PR; ++r) {
    if (!has[r]) continue;
    const float2 v = unpack2(G[r]);
    if (MODE == kEnds) {
      const size_t at = row * p.Kp + kp[r];
      reinterpret_cast<float2*>(p.ends)[at] = v;
      reinterpret_cast<float2*>(p.ends2)[at] = unpack2(H[MODE == kEnds ? r : 0]);
      p.turn[at] = turn[r];
      p.spoil[at] = taint[r];
    } else {
      reinterpret_cast<float2*>(p.h)[sd * p.Kp + kp[r]] = v;
      p.phase[sd * p.Kp + kp[r]] = m3_unit(turn[r], taint[r]);
    }
  }
}
// What the segments of a sequence start from, as m3k_heads_chain_kernel: the state and the angle.
__global__ void __launch_bounds__(256) m3k_channels_chain_kernel(ServeP p, bool bf16_io) {
  begin_dependent();
  const Piece q = find_piece<kCut>(p, blockIdx.x, p.L);
  if (!q.ok || q.base + q.segs > p.cuts) return;
  const int slot = serve_slot(p, q.seq);
  const bool go = slot >= 0 && serve_goes_on(p, q.seq);
  const size_t pairs = (size_t)p.D * p.Kp;
  for (size_t i = blockIdx.y * (size_t)256 + threadIdx.x; i < pairs; i += gridDim.y * (size_t)256) {
    const int d = (int)(i / p.Kp), k = (int)(i % p.Kp), g = d / (p.D / p.G);
    float2 v = make_float2(0.f, 0.f);
    int angle = 0;
    float taint = 0.f;
    if (go) {
      const size_t sd = (size_t)slot * p.D + d, br = ((size_t)slot * p.G + g) * p.N + 2 * k;
      const float2 unit = p.phase[sd * p.Kp + k];
      angle = serve_turn(unit);
      taint = m3_taint(unit.x, m3_taint(unit.y, 0.f));
      v = reinterpret_cast<const float2*>(p.h)[sd * p.Kp + k];
      const float w = serve_look(p, (size_t)q.begin * p.D + d, true) * (bf16_io ? to_f32(static_cast<const bf16*>(p.x_prev)[sd]) : static_cast<const float*>(p.x_prev)[sd]);
      const float2 b = m3_back(bf16_io ? load_pair(static_cast<const bf16*>(p.b_prev) + br) : load_pair(static_cast<const float*>(p.b_prev) + br), unit);
      v.x = fmaf(w, b.x, v.x);
      v.y = fmaf(w, b.y, v.y);
    }
    const float a0 = -expf(p.a_log[(size_t)d * p.N + 2 * k]), a1 = -expf(p.a_log[(size_t)d * p.N + 2 * k + 1]);
    size_t at = (size_t)q.base * pairs + i;
    for (int s0 = 0; s0 < q.segs; s0 += kAhead) {
      const int n = min(kAhead, q.segs - s0), adds = min(kAhead, q.segs - 1 - s0);
      float2 c[kAhead], s[kAhead];
      float sum[kAhead], spoil[kAhead];
      int turn[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool in = j < adds;
        c[j] = in ? reinterpret_cast<const float2*>(p.ends)[at + j * pairs] : make_float2(0.f, 0.f);
        s[j] = in ? reinterpret_cast<const float2*>(p.ends2)[at + j * pairs] : make_float2(0.f, 0.f);
        sum[j] = in ? p.dsum[(size_t)(q.base + s0 + j) * p.D + d] : 0.f;
        turn[j] = in ? p.turn[at + j * pairs] : 0;
        spoil[j] = in ? p.spoil[at + j * pairs] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (j >= n) break;
        reinterpret_cast<float2*>(p.ends)[at + j * pairs] = v;
        p.turn[at + j * pairs] = angle;
        p.spoil[at + j * pairs] = taint;
        const float2 unit = m3_unit(angle, taint);
        v.x = fmaf(expf(a0 * sum[j]), v.x, fmaf(unit.x, c[j].x, unit.y * s[j].x));
        v.y = fmaf(expf(a1 * sum[j]), v.y, fmaf(unit.x, c[j].y, unit.y * s[j].y));
        angle += turn[j];
        taint += spoil[j];
      }
      at += kAhead * pairs;
    }
  }
}

// ------------------------------------------------------------------ host
static int longer_than_L(const ServeP& p) { return std::min(p.S, (int)(p.rows / ((long long)p.L + 1))); }  // at most so many sequences
static int serve_slabs(const ServeP& p) { return (p.P + kRowsMost - 1) / kRowsMost; }
// Lanes along a row: as few as keep a row's 4 NV states (NV up to 4) in registers, for a step's sum over lanes costs a row LN's
// logarithm in exchanges, but enough that narrow heads still give all threads a row.  (Rows of 128 states over 32 lanes: 2046 us
// where 8 lanes take 931.)
struct HeadShape { int LN, NV, R, slabs; };
static HeadShape head_shape(const ServeP& p) {
  HeadShape s{4, 1, 1, 1};
  while (s.LN * 4 < p.N && (s.LN < 8 || s.LN * 16 < p.N || (256 / s.LN > p.P && s.LN < (p.N > 128 ? 16 : 32)))) s.LN *= 2;
  while (s.LN * 4 * s.NV < p.N) s.NV *= 2;
  s.slabs = (p.P + kRowsMost - 1) / kRowsMost;
  const int per = (p.P + s.slabs - 1) / s.slabs;
  while (s.R * (256 / s.LN) < per) s.R *= 2;
  return s;
}
struct ChannelShape { int PR, LPC; };
static ChannelShape channel_shape(const ServeP& p) {
  ChannelShape s{1, 1};
  while (s.LPC < p.Kp && s.LPC < 32) s.LPC *= 2;
  while (s.LPC * s.PR < p.Kp) s.PR *= 2;
  return s;
}

template <typename IO, Mode MODE>
static void heads(const ServeP& p, cudaStream_t st) {
  const HeadShape s = head_shape(p);
  const size_t smem = sizeof(float) * (2 * kW * (size_t)s.LN * 4 * s.NV + 2 * kW * kRowsMost);
  const dim3 grid((unsigned)((size_t)(MODE == kEnds ? p.rows / p.L : p.pieces) * p.NH * s.slabs));
  auto launch = [&](auto nv, auto r) {
    constexpr int NV = decltype(nv)::value, R = decltype(r)::value;
    MXB_LAUNCH(MODE == kOut ? "m3k_heads_kernel" : "m3k_heads_ends_kernel", st,
               (launch_kernel(m3k_heads_kernel<IO, NV, R, MODE>, grid, 256, smem, st, p, s.LN)));
  };
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  constexpr std::integral_constant<int, 4> four;
  auto by_r = [&](auto nv) {
    if (s.R == 1) launch(nv, one);
    else launch(nv, two);
  };
  if (s.NV == 1) by_r(one);
  else if (s.NV == 2) by_r(two);
  else if (s.R == 4) launch(four, four);
  else by_r(four);
}
template <typename IO, Mode MODE>
static mxb_status channels(const ServeP& p, cudaStream_t st) {
  const ChannelShape s = channel_shape(p);
  const dim3 grid(MODE == kEnds ? p.rows / p.L : p.pieces, (p.D + 128 / s.LPC - 1) / (128 / s.LPC));
  // (pairs that fill the lanes, warps that lie in one group, rows of whole 16-byte pieces: 97 us for 4003 rows of 448 channels of 16
  // states, where each lane fetching its own takes 127)
  const bool whole = p.Kp == s.LPC * s.PR && p.D / p.G % (32 / s.LPC) == 0 && p.N * sizeof(IO) % 16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.theta) | reinterpret_cast<uintptr_t>(p.b) | reinterpret_cast<uintptr_t>(p.c)) & 15) == 0;
  mxb_status status = MXB_OK;
  auto launch = [&](auto pr, auto lpc, auto all) {
    constexpr int PR = decltype(pr)::value, LPC = decltype(lpc)::value;
    constexpr bool WHOLE = decltype(all)::value;
    constexpr int smem = 2 * (int)sizeof(Ahead<IO, PR, LPC, MODE, WHOLE>) + 128 / LPC * (int)sizeof(Steps);
    status = MXB_ALLOW_SMEM(smem, m3k_channels_kernel<IO, PR, LPC, MODE, WHOLE>);
    if (status != MXB_OK) return;
    MXB_LAUNCH(MODE == kOut ? "m3k_channels_kernel" : "m3k_channels_ends_kernel", st,
               (launch_kernel(m3k_channels_kernel<IO, PR, LPC, MODE, WHOLE>, grid, 128, smem, st, p)));
  };
  auto by_whole = [&](auto pr, auto lpc) {
    if constexpr (2 * decltype(pr)::value * decltype(lpc)::value * sizeof(IO) % 16 == 0)
      if (whole) return launch(pr, lpc, std::true_type{});
    launch(pr, lpc, std::false_type{});
  };
  constexpr std::integral_constant<int, 1> one;
  switch (s.LPC * s.PR) {
    case 1: by_whole(one, one); break;
    case 2: by_whole(one, std::integral_constant<int, 2>{}); break;
    case 4: by_whole(one, std::integral_constant<int, 4>{}); break;
    case 8: by_whole(one, std::integral_constant<int, 8>{}); break;
    case 16: by_whole(one, std::integral_constant<int, 16>{}); break;
    case 32: by_whole(one, std::integral_constant<int, 32>{}); break;
    case 64: by_whole(std::integral_constant<int, 2>{}, std::integral_constant<int, 32>{}); break;
    default: by_whole(std::integral_constant<int, 4>{}, std::integral_constant<int, 32>{}); break;
  }
  return status;
}
template <typename IO>
static mxb_status prefill(ServeP p, bool chunks, cudaStream_t st) {
  const size_t blocks = ((size_t)p.D * p.Kp + 255) / 256;
  const int cuts = std::max(longer_than_L(p), 1);
  const dim3 chain(cuts, (unsigned)std::min<size_t>(blocks, std::max<size_t>(148 * 4 / cuts, 1)));
  const bool cut = p.ends != nullptr;
  if (p.NH) {
    p.slabs = chunks ? serve_slabs(p) : head_shape(p).slabs;
    if (chunks)
      if (const mxb_status s = m3prompt_prepare(p, st); s != MXB_OK) return s;
    if (cut) {
      if (!chunks) heads<IO, kEnds>(p, st);
      else if (const mxb_status s = m3prompt_chunks(p, true, st); s != MXB_OK) return s;
      MXB_LAUNCH("m3k_heads_chain_kernel", st, (launch_kernel(m3k_heads_chain_kernel, chain, 256, 0, st, p, sizeof(IO) == 2)));
    }
    if (!chunks) heads<IO, kOut>(p, st);
    else if (const mxb_status s = m3prompt_chunks(p, false, st); s != MXB_OK) return s;
    if (p.slabs == 1) return check_launch("m3k_prefill");
  } else {
    if (cut) {
      if (const mxb_status s = channels<IO, kEnds>(p, st); s != MXB_OK) return s;
      MXB_LAUNCH("m3k_channels_chain_kernel", st, (launch_kernel(m3k_channels_chain_kernel, chain, 256, 0, st, p, sizeof(IO) == 2)));
    }
    if (const mxb_status s = channels<IO, kOut>(p, st); s != MXB_OK) return s;
  }
  const mxb_status s = check_launch("m3k_prefill");
  return s == MXB_OK ? m3serve_tails(p, sizeof(IO) == 4, true, st) : s;
}

}  // namespace m3k

// Steps of a segment: as many segments as the CTAs that the GPU holds at once (heads), or twice that (channels: seven CTAs an SM
// by registers), and at least 64 steps each; a quarter longer where several sequences can fill the GPU side by side, since a cut
// costs a pass of its own over what lies in front of it.  (The host does not know the lengths; sequences of up to L steps are not
// cut.)  Half and twice as many segments, us: a prompt of 16381 rows of 8 heads in chunks 99 and 111 for 87; float32 599 and 480
// for 417; channels, 7 prompts of 4003 rows of 448 channels of 16 states 99 and 97 for 97, in bf16 108 and 99 for 99, one of 16384
// rows 318 and 323 for 315, 4 of 2048 rows of 256 channels of 32 states 223 and 184 for 204.  Without the quarter, heads: 16
// prompts of 32 heads, 32768 rows, 422 us for 319 (the passes after the scalars); three of 700 rows, 8 heads, float32, 85 for 103.
static int walk_segment(const ServeP& p) {
  const long long ctas = p.NH ? (long long)p.NH * m3k::serve_slabs(p) : [&] {
    const int per = 128 / m3k::channel_shape(p).LPC;
    return (long long)((p.D + per - 1) / per);
  }();
  const long long at_once = p.NH ? 148 * 2 : 148 * 16;
  long long L = (p.rows * ctas + at_once - 1) / at_once;
  if (p.S > 1) L += L / 4;
  return (int)std::min<long long>(std::max<long long>(64, (L + 63) / 64 * 64), INT32_MAX);
}
// Sets the cut and lays out the scratch (base may be null: only its size is wanted).
size_t m3walk_scratch(ServeP& p, bool f32, int flags, char* base) {
  p.L = flags & MXB_MAMBA3_SERIAL_WALK ? std::max(p.rows, 1) : walk_segment(p);
  Carver c(base);
  if (!(flags & MXB_MAMBA3_RECURRENT_KERNELS) && m3prompt_supported(p, f32)) {
    p.chunks = p.rows / 64 + std::min(p.S, p.rows);
    p.rec = c.take<float>((size_t)p.chunks * p.NH * 512);
    p.scores = c.take<float>((size_t)p.chunks * p.G * 10 * 512);
  }
  if (p.NH && m3k::serve_slabs(p) > 1) p.phase_end = c.take<float2>((size_t)p.S * p.NH);
  p.pieces = p.S;
  p.cuts = 1;
  if (p.rows <= p.L) return c.bytes();
  p.cuts += p.rows / p.L + m3k::longer_than_L(p);  // (a sequence's segments but the last are L rows each)
  p.pieces = p.rows / p.L + p.S;
  p.ends = c.take<float>((size_t)p.cuts * p.D * p.N);
  p.dsum = c.take<float>((size_t)p.cuts * (p.NH ? p.NH : p.D));
  p.turn = c.take<int>((size_t)p.cuts * (p.NH ? p.NH : (size_t)p.D * p.Kp));
  if (p.NH) p.start = c.take<float2>((size_t)p.cuts * p.NH);
  else {
    p.ends2 = c.take<float>((size_t)p.cuts * p.D * p.N);
    p.spoil = c.take<float>((size_t)p.cuts * p.D * p.Kp);
  }
  return c.bytes();
}
// The chunks on the tensor cores where they cover the call, the walks elsewhere.
mxb_status m3walk_prefill(ServeP p, bool f32, int flags, cudaStream_t st) {
  if (f32) return m3k::prefill<float>(p, false, st);
  return m3k::prefill<m3k::bf16>(p, !(flags & MXB_MAMBA3_RECURRENT_KERNELS) && m3prompt_supported(p, f32), st);
}

}  // namespace mxb
