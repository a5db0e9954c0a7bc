// Mamba-3 scan of packed bf16 prompts on a pool of states, head layout, in chunks of 64 steps on the tensor cores.
//
// With L_i the sum of the decays' logarithms from the chunk's start on, phi_i the angle from the segment's start on, and G, e_s
// as in mamba3_walk.cu (the segments and the pool are its), a chunk is
//     y_i = exp(L_i) <C_i turned back by phi_i, G> + sum_{j <= i} M_ij x_j
//     M_ij = <C_i turned back by phi_i, B_j turned back by phi_j> exp(L_i - L_j) (e_j, or lam_i dt_i where j = i)
//     G  <- exp(L_64) G + sum_j g_j (B_j turned back) (x) x_j,      g_j = exp(L_64 - L_j) e_j
// One angle turns all pairs of a head, so with J (even, odd) = (-odd, even)
//     <C_i back, v> = cos phi_i <C_i, v> + sin phi_i <C_i, J v>
// and the products of b and c, <C_i, B_j> and <C_i, J B_j>, are the same for all heads of a group.
//
// The same identity turns the state's update: with x weighted by g cos and by g sin, two products with B as it is.
//
// m3p_prepare_kernel works the scores out once (float32, from exact bf16 operands), and for every head the scalars of its steps.
// m3p_chunks_kernel takes up to 64 channels of a head through a segment, chunk after chunk, with four warps that multiply and
// four that make their operands ready (and hand them most of their registers).  The state stays in registers as the accumulators
// of its own update, 16 channels a warp; rounded to bf16 those registers are the operand of <C, G> as
// they stand, and J G is the same registers in another order.  b, c and x come by cp.async and are multiplied as they are; M, put
// together from the two scores, and the weighted x are written in the order of the registers that multiply them.  All products
// are mma.sync with bf16 operands and float32 sums: 2.2 M multiply-adds a chunk and 64 channels, of which an SM does 1024 a clock
// this way.  (Turning b and c instead halves two of the three products, but the turning, with its passes through shared memory,
// took more time than that.)
//
// Bound: shared memory.  16 prompts, 32768 rows, 32 heads of 64 channels and 128 states, half of them from states: scalars and
// scores 33 us, chunks 306 us at 70 % of the shared-memory pipe and 45 % of the tensor pipe's time, 334 us in all (the products
// alone at that rate 131, the bytes 49).  Two CTAs of eight warps an SM; one CTA of 12 or 16 warps, with the fragments of b and c
// for 32 channels a warp or products and state in warps of their own, took 359 to 374 us where this took 322.
//
// Roundings to bf16: G as operand, g x and M once each; y itself.  (In the mean y is 2.4e-3 of itself off, 1.7e-3 by its own
// rounding alone, 2.6e-3 where the state decays slowly; splitting G and M in two parts each would double the products that y is
// made of.)  The state is a float32 result of its own, so that one rounding of g x is too much where it still reaches the
// segment's end: there (decay to the end above 2^-11, above 2^-3) the remainder of the rounding is multiplied as well, and the
// remainder of that: 16 and 24 bits of g x, while b is exact.
#include <algorithm>
#include <type_traits>

#include "mamba3_serve.cuh"
#include "mma_sync.cuh"
#include "packed.cuh"

namespace mxb {
namespace m3p {

using bf16 = __nv_bfloat16;
constexpr int Q = 64, kThreads = 128, kPS = 64;  // steps of a chunk; threads of half a CTA; channels of a CTA

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
// J of a pair of bf16: (even, odd) -> (-odd, even)
__device__ __forceinline__ uint32_t turn_j(uint32_t v) { return __byte_perm(v, v, 0x1032) ^ 0x00008000u; }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <typename T>
__device__ __forceinline__ uint32_t smem_at(T& v) { return (uint32_t)__cvta_generic_to_shared(&v); }

// Byte offset of 16-byte unit u of row r in a tile of U units a row; units change places by the row, so that the eight rows of an
// ldmatrix fall on different banks.
template <int U>
__device__ __forceinline__ uint32_t at(int r, int u) { return (uint32_t)(r * U + (u ^ (r & 7))) * 16; }

// Scalars of the 64 steps of a chunk, for one head; steps behind the sequence's last weigh nothing.
struct __align__(16) Rec {
  float co[Q], si[Q];       // the angle from the chunk's start on
  float L[Q], e[Q], gam[Q]; // L in powers of two; e_j; lam dt
  float gc[Q], gs[Q];       // g_j times cosine and sine of the same angle
  int turn;                 // of the whole chunk: angle, its taint, sum of dt, L
  float taint, dsum, Lq;
  float pad[60];
};
static_assert(sizeof(Rec) == 2048, "a record is one 16-byte piece for each of 128 threads");

// The tiles of 16 x 16 scores on and below the diagonal: (0,0) (1,0) (1,1) (2,0) ...; warp w has every fourth.
constexpr int kTiles = 10;
__device__ __forceinline__ void tile_at(int tile, int& i, int& j) {
  i = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0;
  j = tile - i * (i + 1) / 2;
}

// ------------------------------------------------------------------ what the heads share, and the scalars
// grid (chunks, G + ceil(heads / 8)): the scores of a group, or the records of eight heads, two at a time.
constexpr int kRecHeads = 8;
template <int N>
__global__ void __launch_bounds__(kThreads) m3p_prepare_kernel(ServeP p) {
  begin_dependent();
  constexpr int U = N / 8;
  __shared__ uint4 tb[Q * U], tc[Q * U];
  constexpr int K2 = kRecHeads / 2;
  __shared__ float s_l[K2][4], s_r[K2][4], s_taint[K2][4], s_ds[K2][4];
  __shared__ int s_turn[K2][4];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const Piece q = find_piece<kPieces, false>(p, blockIdx.x, Q);
  if (!q.ok) return;
  if ((int)blockIdx.y < p.G) {
    const int grp = blockIdx.y;
    const bf16 *B = static_cast<const bf16*>(p.b) + (size_t)grp * p.N, *C = static_cast<const bf16*>(p.c) + (size_t)grp * p.N;
    const size_t gn = (size_t)p.G * p.N;
    const uint32_t sb = smem_at(tb), sc = smem_at(tc);
#pragma unroll
    for (int k = 0; k < Q * U / kThreads; ++k) {
      const int i = tid + k * kThreads, r = i / U, u = i % U;
      const bool in = q.first + r < q.last && u * 8 < p.N;
      const size_t off = in ? (size_t)(q.first + r) * gn + u * 8 : 0;
      cp16(sb + at<U>(r, u), B + off, in);
      cp16(sc + at<U>(r, u), C + off, in);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    float4* out = reinterpret_cast<float4*>(p.scores + ((size_t)blockIdx.x * p.G + grp) * kTiles * 512);
    for (int tile = w; tile < kTiles; tile += 4) {
      int ti, tj;
      tile_at(tile, ti, tj);
      float s1[2][4] = {}, s2[2][4] = {};
#pragma unroll
      for (int kk = 0; kk < N / 16; ++kk) {
        uint32_t a[4], b[4];
        ms::ldsm(a, sc + at<U>(16 * ti + (lane & 15), 2 * kk + (lane >> 4)));
        ms::ldsm(b, sb + at<U>(16 * tj + (lane & 7) + (lane >> 4) * 8, 2 * kk + ((lane >> 3) & 1)));
        ms::mma(s1[0], a, b[0], b[1]);
        ms::mma(s1[1], a, b[2], b[3]);
        ms::mma(s2[0], a, turn_j(b[0]), turn_j(b[1]));
        ms::mma(s2[1], a, turn_j(b[2]), turn_j(b[3]));
      }
      float4* o = out + tile * 128 + lane * 4;
      o[0] = make_float4(s1[0][0], s1[0][1], s1[0][2], s1[0][3]);
      o[1] = make_float4(s1[1][0], s1[1][1], s1[1][2], s1[1][3]);
      o[2] = make_float4(s2[0][0], s2[0][1], s2[0][2], s2[0][3]);
      o[3] = make_float4(s2[1][0], s2[1][1], s2[1][2], s2[1][3]);
    }
    return;
  }
  const int i = tid & 63, t = q.first + i, h0 = ((int)blockIdx.y - p.G) * kRecHeads;
  const bool in = t < q.last, next = in && t + 1 < q.end;
  // dt, lambda and theta of the eight heads by rows (a head by itself: a sector of 32 bytes for each of its 4), with the step behind
  constexpr int PITCH = kRecHeads + 1;
  float(*in_)[Q + 1][PITCH] = reinterpret_cast<float(*)[Q + 1][PITCH]>(tb);
  static_assert(sizeof(float) * 3 * (Q + 1) * PITCH <= sizeof(tb), "the tile of b is free here");
#pragma unroll
  for (int j = 0; j < (Q + 1) * kRecHeads; j += kThreads) {
    const int e = j + tid, r = e / kRecHeads, hd = h0 + e % kRecHeads;
    if (r > Q) break;
    const bool there = q.first + r < (r < Q ? q.last : q.end) && hd < p.NH;
    const size_t at = (size_t)(there ? q.first + r : q.first) * p.NH + min(hd, p.NH - 1);
    in_[0][r][e % kRecHeads] = there ? p.dt[at] : 0.f;
    in_[1][r][e % kRecHeads] = there ? p.lam[at] : 0.f;
    in_[2][r][e % kRecHeads] = there ? p.theta[at] : 0.f;
  }
  __syncthreads();
  // what needs no other step, of all heads before the first exchange: eight chains side by side
  float dts[K2], gammas[K2], looks[K2], taints[K2], rates[K2];
  int turns[K2];
#pragma unroll
  for (int k = 0; k < K2; ++k) {
    const int c = 2 * k + (w >> 1);
    // dt in 64 bits: an angle sums up tens of thousands of them, and their float32 roundings with it
    const double raw = in_[0][i][c], dt64 = fmax(raw, 0.0) + log1p(exp(-fabs(raw)));
    const float dt = (float)dt64, theta = in_[2][i][c];
    const double f = dt64 * theta * 0.15915494309189535;
    turns[k] = in ? (int)__double2ll_rn((f - rint(f)) * 4294967296.0) : 0;
    taints[k] = in ? m3_taint(dt * theta, 0.f) : 0.f;
    dts[k] = in ? dt : 0.f;
    gammas[k] = in ? m3_sigmoid(in_[1][i][c]) * dt : 0.f;
    looks[k] = next ? (1.f - m3_sigmoid(in_[1][i + 1][c])) * m3_softplus(in_[0][i + 1][c]) : 0.f;
    rates[k] = -expf(p.a_log[min(h0 + c, p.NH - 1)]) * 1.4426950408889634f;
  }
  // A step's decay, in powers of two.  Beyond 2^-160, which is 0 as a float32, it counts as that: what follows such a step is
  // weighed by differences of the sums from the chunk's start on, which a step of some thousands would leave few bits.
  float l[K2], r[K2], ds[K2];
#pragma unroll
  for (int k = 0; k < K2; ++k) {
    const float fall = in ? dts[k] * rates[k] : 0.f;
    l[k] = r[k] = fall < -160.f ? -160.f : fall;
    ds[k] = dts[k];
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)  // (four heads' chains of sums beside each other)
#pragma unroll
    for (int k = 0; k < K2; ++k) {
      const int b = __shfl_up_sync(0xffffffffu, turns[k], o);
      const float c = __shfl_up_sync(0xffffffffu, taints[k], o), d = __shfl_up_sync(0xffffffffu, l[k], o), e = __shfl_down_sync(0xffffffffu, r[k], o);
      ds[k] += __shfl_xor_sync(0xffffffffu, ds[k], o);
      if (lane >= o) { turns[k] += b; taints[k] += c; l[k] += d; }
      if (lane + o < 32) r[k] += e;
    }
#pragma unroll
  for (int k = 0; k < K2; ++k) {
    if (lane == 31) { s_turn[k][w] = turns[k]; s_taint[k][w] = taints[k]; s_l[k][w] = l[k]; s_ds[k][w] = ds[k]; }
    if (lane == 0) s_r[k][w] = r[k];
    const float behind = __shfl_down_sync(0xffffffffu, r[k], 1);
    r[k] = lane < 31 ? behind : 0.f;  // of the steps behind this one
  }
  __syncthreads();
  const int w0 = w & 2;
#pragma unroll
  for (int k = 0; k < K2; ++k) {
    const int hd = h0 + 2 * k + (w >> 1);
    if (hd >= p.NH) break;
    if (w & 1) { turns[k] += s_turn[k][w0]; taints[k] += s_taint[k][w0]; l[k] += s_l[k][w0]; }
    else r[k] += s_r[k][w + 1];
    Rec* rec = reinterpret_cast<Rec*>(p.rec) + (size_t)blockIdx.x * p.NH + hd;
    const float e = gammas[k] + looks[k], g = e * exp2f(r[k]);
    const float2 unit = m3_unit(turns[k], taints[k]);
    rec->co[i] = unit.x;
    rec->si[i] = unit.y;
    rec->L[i] = l[k];
    rec->e[i] = e;
    rec->gam[i] = gammas[k];
    rec->gc[i] = g * unit.x;
    rec->gs[i] = g * unit.y;
    if (i == 63) {
      rec->turn = turns[k];
      rec->taint = taints[k];
      rec->dsum = s_ds[k][w0] + s_ds[k][w0 + 1];
      rec->Lq = l[k];
    }
  }
}

// ------------------------------------------------------------------ chunks
template <int N>
struct Smem {
  uint4 x[2][Q * kPS / 8];        // [steps][channels]
  uint4 c[2][Q * N / 8], b[2][Q * N / 8];
  uint4 m[2][kTiles * 32];        // M: [tile][lane], as the registers of an A operand
  uint4 gx[4][Q / 16][2][32];     // x g cos, x g sin: [16 channels][16 steps][which][lane], likewise
  Rec rec[3];
};
// Registers: a CTA starts with 128 a thread; the warps that bring operands keep kReady of them, the others go to kMultiply.
constexpr int kStart = 128, kReady = 88, kMultiply = 168;
static_assert(kReady + kMultiply <= 2 * kStart, "what one half takes the other has to give");
// Barriers between the two halves: a chunk's b, c, x, M are there and the chunk is done with (by its parity), its weighted x is
// there, a part of that has been read.
enum { kFull = 1, kEmpty = 3, kAmong = 5, kWeighted = 6, kPart = 7 };
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// N: d_state, padded to 64 or 128.
template <int N, bool ENDS>
__global__ void __launch_bounds__(2 * kThreads, 2) m3p_chunks_kernel(ServeP p) {
  begin_dependent();
  extern __shared__ __align__(128) unsigned char raw[];
  Smem<N>& s = *reinterpret_cast<Smem<N>*>(raw);
  constexpr int U = N / 8, NT = N / 8, KK = N / 16;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) & 3, tid = threadIdx.x & (kThreads - 1);
  const int per = p.NH * p.slabs, hd = blockIdx.x % per / p.slabs, slab = blockIdx.x % p.slabs;  // (heads first)
  const Piece q = find_piece<ENDS ? kInner : kPieces>(p, blockIdx.x / per, p.L);
  const int piece = q.base + q.seg;
  if (!q.ok || piece >= p.cuts) return;
  const int chunks = (q.last - q.first + Q - 1) / Q;
  if (q.chunk + chunks > p.chunks) return;  // (lengths that add up to more than the rows)
  const int p0 = slab * kPS, np = min(kPS, p.P - p0);
  const size_t chan = (size_t)hd * p.P + p0;
  const int slot = serve_slot(p, q.seq), grp = hd / (p.NH / p.G);
  const bool goes_on = serve_goes_on(p, q.seq);
  const bool keeps = ENDS || (q.seg == q.segs - 1 && slot >= 0);  // the state at the end is somebody's
  const Rec* recs = reinterpret_cast<const Rec*>(p.rec) + (size_t)q.chunk * p.NH + hd;

  // chunks from which on one, two parts of g x are not enough: by the decay from their end to the segment's
  int from2 = chunks, from3 = chunks;
  auto find_parts = [&] {
    if (!keeps) return;
    float rem = 0.f;
    for (int k0 = chunks - 1; k0 >= 0 && !(rem <= -11.f); k0 -= 32) {
      const int k = k0 - lane;
      const float own = k >= 0 ? recs[(size_t)k * p.NH].Lq : 0.f;
      float v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float a = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += a;
      }
      const float behind = rem + v - own;
      from2 -= __popc(__ballot_sync(0xffffffffu, k >= 0 && !(behind <= -11.f)));
      from3 -= __popc(__ballot_sync(0xffffffffu, k >= 0 && !(behind <= -3.f)));
      rem += __shfl_sync(0xffffffffu, v, 31);
    }
  };

  if (threadIdx.x >= kThreads) {
    // ---------------------------------------------------------------- the warps that bring operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kReady));
    const size_t gn = (size_t)p.G * p.N;
    // A thread has unit u0 of rows r0, r0 + ROWS, ... of b and c (ux of rx, rx + XROWS, ... of x): ROWS is a multiple of 8, so
    // that its places in shared memory are a fixed distance apart.
    constexpr int ROWS = kThreads / U, PASSES = Q / ROWS, XROWS = kThreads / 8, XPASSES = Q / XROWS;
    const int r0 = tid / U, u0 = tid % U, rx = tid / 8, ux = tid % 8;
    const bool live = u0 * 8 < p.N, live_x = ux * 8 < np;
    const bf16 *X = static_cast<const bf16*>(p.x) + (size_t)(q.first + rx) * p.D + chan + (live_x ? ux * 8 : 0),
               *B = static_cast<const bf16*>(p.b) + (size_t)(q.first + r0) * gn + (size_t)grp * p.N + (live ? u0 * 8 : 0),
               *C = static_cast<const bf16*>(p.c) + (size_t)(q.first + r0) * gn + (size_t)grp * p.N + (live ? u0 * 8 : 0);
    const uint32_t dx = smem_at(s.x) + at<8>(rx, ux), db = smem_at(s.b) + at<U>(r0, u0), dc = smem_at(s.c) + at<U>(r0, u0);
    const int step = ROWS * p.G * p.N, xstep = XROWS * p.D;
    // x, b and c of the chunk that the pointers stand at: zeros behind the segment's last row and the head's last channel
    auto fetch = [&](int k) {
      const int left = q.last - q.first - k * Q;
      const uint32_t x0 = dx + (k & 1) * sizeof(s.x[0]), b0 = db + (k & 1) * sizeof(s.b[0]), c0 = dc + (k & 1) * sizeof(s.c[0]);
      if (left >= Q) {
#pragma unroll
        for (int j = 0; j < XPASSES; ++j) cp16(x0 + j * XROWS * 128, X + j * xstep, live_x);
#pragma unroll
        for (int j = 0; j < PASSES; ++j) cp16(b0 + j * ROWS * U * 16, B + j * step, live);
        if (!ENDS)
#pragma unroll
          for (int j = 0; j < PASSES; ++j) cp16(c0 + j * ROWS * U * 16, C + j * step, live);
      } else {
#pragma unroll
        for (int j = 0; j < XPASSES; ++j) {
          const bool in = rx + j * XROWS < left;
          cp16(x0 + j * XROWS * 128, in ? X + j * xstep : static_cast<const bf16*>(p.x), in && live_x);
        }
#pragma unroll
        for (int j = 0; j < PASSES; ++j) {
          const bool in = r0 + j * ROWS < left;
          cp16(b0 + j * ROWS * U * 16, in ? B + j * step : static_cast<const bf16*>(p.b), in && live);
          if (!ENDS) cp16(c0 + j * ROWS * U * 16, in ? C + j * step : static_cast<const bf16*>(p.c), in && live);
        }
      }
      X += (size_t)Q * p.D;
      B += Q * gn;
      C += Q * gn;
    };
    // M = cos(phi_i - phi_j) s1 + sin(phi_i - phi_j) s2, weighted: warp w has tile (w, w) and one or two below the diagonal
    const int i1 = w == 2 ? 2 : w == 3 ? 1 : 3, j1 = w == 0 || w == 3 ? 0 : w == 1 ? 2 : 1, i2 = w == 0 ? 3 : 2, j2 = w == 0 ? 1 : 0;
    const bool third = w < 2;
    const int tile0 = w * (w + 3) / 2, tile1 = i1 * (i1 + 1) / 2 + j1, tile2 = i2 * (i2 + 1) / 2 + j2;
    auto load_scores = [&](const float4* scores, int tile, float4 (&v)[4]) {
#pragma unroll
      for (int a = 0; a < 4; ++a) v[a] = __ldg(scores + tile * 128 + a);
    };
    auto weigh_scores = [&](const Rec& rec, uint4* m, int ti, int tj, const float4 (&v)[4], auto diagonal) {
      const int i0 = 16 * ti + lane / 4, c0 = 16 * tj + 2 * (lane % 4);
      uint32_t out[4];
#pragma unroll
      for (int low = 0; low < 2; ++low) {
        const int i = i0 + 8 * low;
        const float Li = rec.L[i], co_i = rec.co[i];
        const f2 ci = dup2(co_i), si = dup2(rec.si[i]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c = c0 + 8 * half;
          const f2 cj = *reinterpret_cast<const f2*>(&rec.co[c]), sj = *reinterpret_cast<const f2*>(&rec.si[c]), ej = *reinterpret_cast<const f2*>(&rec.e[c]);
          const float2 L = *reinterpret_cast<const float2*>(&rec.L[c]);
          const f2 a1 = low ? pack2(v[half].z, v[half].w) : pack2(v[half].x, v[half].y);
          const f2 a2 = low ? pack2(v[2 + half].z, v[2 + half].w) : pack2(v[2 + half].x, v[2 + half].y);
          // (cos_i cos_j + sin_i sin_j) s1 + (sin_i cos_j - cos_i sin_j) s2
          const f2 cosd = mad2(si, sj, mul2(ci, cj)), sind = mad2(si, cj, mul2(ci, sj ^ 0x8000000080000000ull));
          const f2 decay = mul2(pack2(ex2(Li - L.x), ex2(Li - L.y)), ej);
          float2 r = unpack2(mul2(mad2(sind, a2, mul2(cosd, a1)), decay));
          if constexpr (decltype(diagonal)::value) {
            const float2 s = unpack2(a1), g = *reinterpret_cast<const float2*>(&rec.gam[c]);
            const float tnt = co_i * 0.f;  // (an angle that is not finite has to reach the diagonal too)
            r.x = c < i ? r.x : c == i ? (s.x + tnt) * g.x : 0.f;
            r.y = c + 1 < i ? r.y : c + 1 == i ? (s.y + tnt) * g.y : 0.f;
          }
          out[2 * half + low] = pack(r.x, r.y);
        }
      }
      m[lane] = make_uint4(out[0], out[1], out[2], out[3]);
    };
    auto fetch_rec = [&](int k) { cp16(smem_at(s.rec[k % 3]) + tid * 16, reinterpret_cast<const char*>(recs + (size_t)k * p.NH) + tid * 16, true); };
    // this warp's 16 channels; part 1, 2: what rounding has left, and what rounding that has
    auto weigh_x = [&](int k, auto nth) {
      constexpr int part = decltype(nth)::value;
      const Rec& rec = s.rec[k % 3];
      const uint32_t xb = smem_at(s.x[k & 1]);
#pragma unroll
      for (int kk = 0; kk < Q / 16; ++kk) {
        uint32_t a[4], xc[4], xs[4];
        ms::ldsm_t(a, xb + at<8>(16 * kk + (lane & 7) + (lane >> 4) * 8, 2 * w + ((lane >> 3) & 1)));
        const int j = 16 * kk + 2 * (lane % 4);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {  // a[0], a[1]: steps j, j + 1; a[2], a[3]: j + 8, j + 9
          const float2 c = *reinterpret_cast<const float2*>(&rec.gc[j + 4 * i]), sn = *reinterpret_cast<const float2*>(&rec.gs[j + 4 * i]);
#pragma unroll
          for (int l = i; l < i + 2; ++l) {
            const float2 v = unpack(a[l]);
            const f2 vv = pack2(v.x, v.y);
            float2 zc = unpack2(mul2(pack2(c.x, c.y), vv)), zs = unpack2(mul2(pack2(sn.x, sn.y), vv));
            xc[l] = pack(zc.x, zc.y);
            xs[l] = pack(zs.x, zs.y);
#pragma unroll
            for (int u = 0; u < part; ++u) {
              const float2 d = unpack(xc[l]), e = unpack(xs[l]);
              zc.x -= d.x; zc.y -= d.y; zs.x -= e.x; zs.y -= e.y;
              xc[l] = pack(zc.x, zc.y);
              xs[l] = pack(zs.x, zs.y);
            }
          }
        }
        s.gx[w][kk][0][lane] = make_uint4(xc[0], xc[1], xc[2], xc[3]);
        s.gx[w][kk][1][lane] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
      }
    };
    fetch_rec(0);
    cp_commit();
    int turn = 0;  // angle in front of the chunk
    float taint = 0.f;
    for (int k = 0; k <= chunks; ++k) {
      const bool more = k < chunks;
      const float4* scores = reinterpret_cast<const float4*>(p.scores + ((size_t)(q.chunk + k) * p.G + grp) * kTiles * 512) + lane * 4;
      float4 v0[4], v1[4];
      if (!ENDS && more) {
        load_scores(scores, tile0, v0);
        load_scores(scores, tile1, v1);
      }
      if (k >= 2) bar_sync(kEmpty + (k & 1), 2 * kThreads);  // chunk k - 2 is done
      if (more) fetch(k);
      cp_commit();
      if (k + 1 < chunks) fetch_rec(k + 1);
      cp_commit();
      if (k == 0) find_parts();
      if (k >= 1) {  // the chunk that is being multiplied: its weighted x, part after part
        const int parts = k - 1 >= from3 ? 3 : k - 1 >= from2 ? 2 : 1;
        weigh_x(k - 1, std::integral_constant<int, 0>{});
        bar_arrive(kWeighted, 2 * kThreads);
        if (parts > 1) {
          bar_sync(kPart, 2 * kThreads);
          weigh_x(k - 1, std::integral_constant<int, 1>{});
          bar_arrive(kWeighted, 2 * kThreads);
        }
        if (parts > 2) {
          bar_sync(kPart, 2 * kThreads);
          weigh_x(k - 1, std::integral_constant<int, 2>{});
          bar_arrive(kWeighted, 2 * kThreads);
        }
      }
      if (!more) break;
      cp_wait<2>();  // this chunk's record
      bar_sync(kAmong, kThreads);
      Rec& rec = s.rec[k % 3];
      {  // its angles from the segment's start on
        const float2 at0 = m3_unit(turn, taint);
        const int i = tid & (Q - 1);
        float &co = tid < Q ? rec.co[i] : rec.gc[i], &si = tid < Q ? rec.si[i] : rec.gs[i];
        const float2 v = m3_on(make_float2(co, si), at0);
        co = v.x;
        si = v.y;
        turn += rec.turn;
        taint += rec.taint;
      }
      bar_sync(kAmong, kThreads);
      if (!ENDS) {
        uint4* m = s.m[k & 1];
        weigh_scores(rec, m + tile0 * 32, w, w, v0, std::true_type{});
        if (third) load_scores(scores, tile2, v0);
        weigh_scores(rec, m + tile1 * 32, i1, j1, v1, std::false_type{});
        if (third) weigh_scores(rec, m + tile2 * 32, i2, j2, v0, std::false_type{});
      }
      cp_wait<1>();  // x, b, c (the next chunk's record may be under way)
      bar_arrive(kFull + (k & 1), 2 * kThreads);
      bar_sync(kAmong, kThreads);  // (x has come for all of these warps: they weigh it next)
    }
    cp_wait<0>();
    bar_sync(kEmpty + ((chunks - 1) & 1), 2 * kThreads);
    return;
  }

  // ------------------------------------------------------------------ the warps that multiply
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMultiply));
  const bool from_state = !ENDS && q.segs == 1 && slot >= 0 && goes_on;
  const size_t ph = (size_t)(slot < 0 ? 0 : slot) * p.NH + hd;
  float2 start = make_float2(1.f, 0.f);
  if (!ENDS && q.segs > 1) start = p.start[(size_t)piece * p.NH + hd];
  else if (from_state) start = p.phase[ph];
  // h[t]: channels 16 w + lane / 4 (+ 8), states 8 t + 2 (lane % 4) + {0, 1}.  One address a row, all elements requested before
  // the first is used, and little code: a warp runs through it once.
  float h[NT][4];
  const int row0 = 16 * w + lane / 4, n0 = 2 * (lane % 4);
  const bool rows_in[2] = {row0 < np, row0 + 8 < np};
  auto load_h = [&](const float* from) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool in = rows_in[k] && 8 * t < p.N;
        const float2 v = in ? *reinterpret_cast<const float2*>(from + (size_t)8 * k * p.N + 8 * t) : make_float2(0.f, 0.f);
        h[t][2 * k] = v.x;
        h[t][2 * k + 1] = v.y;
      }
  };
  if (!ENDS && q.segs > 1) {
    load_h(p.ends + ((size_t)piece * p.D + chan + row0) * p.N + n0);
  } else if (from_state) {
    load_h(p.h + ((size_t)slot * p.D + chan + row0) * p.N + n0);
    const bf16 *b_prev = static_cast<const bf16*>(p.b_prev) + ph * p.N + n0, *x_prev = static_cast<const bf16*>(p.x_prev) + (size_t)slot * p.D + chan + row0;
    uint32_t b[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) b[t] = 8 * t < p.N ? *reinterpret_cast<const uint32_t*>(b_prev + 8 * t) : 0u;
    const float look0 = serve_look(p, (size_t)q.first * p.NH + hd, true);
    const float k0 = rows_in[0] ? look0 * to_f32(x_prev[0]) : 0.f, k1 = rows_in[1] ? look0 * to_f32(x_prev[8]) : 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float2 v = unpack(b[t]), h0 = m3_on(make_float2(h[t][0], h[t][1]), start), h1 = m3_on(make_float2(h[t][2], h[t][3]), start);
      h[t][0] = fmaf(k0, v.x, h0.x);
      h[t][1] = fmaf(k0, v.y, h0.y);
      h[t][2] = fmaf(k1, v.x, h1.x);
      h[t][3] = fmaf(k1, v.y, h1.y);
    }
  } else {
#pragma unroll
    for (int t = 0; t < NT; ++t) h[t][0] = h[t][1] = h[t][2] = h[t][3] = 0.f;
  }
  find_parts();

  int turn = 0;
  float taint = 0.f, dsum = 0.f;
  const int r16 = lane & 15, hi = lane >> 4;
  const bool whole = reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  for (int k = 0; k < chunks; ++k) {
    const int t0 = q.first + k * Q;
    const Rec& rec = s.rec[k % 3];
    const uint32_t xb = smem_at(s.x[k & 1]);
    bar_sync(kFull + (k & 1), 2 * kThreads);
    if (!ENDS) {
      const uint32_t sc = smem_at(s.c[k & 1]) + r16 * (U * 16);
      float y[4][2][4], z[4][2][4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int c = 0; c < 8; ++c) y[m][c / 4][c % 4] = z[m][c / 4][c % 4] = 0.f;
      // (operands are requested a step ahead: 33 clocks until they are there, four products of 8)
      uint32_t a[2][4];
      auto load_c = [&](int i) { ms::ldsm(a[i & 1], sc + (i % 4) * (16 * U * 16) + (((2 * (i / 4) + hi) ^ (lane & 7)) << 4)); };
      load_c(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const float *h0 = h[2 * kk], *h1 = h[2 * kk + 1];  // G and J G as operands: two tiles of 8 channels
        const uint32_t g0 = pack(h0[0], h0[1]), g1 = pack(h1[0], h1[1]), g2 = pack(h0[2], h0[3]), g3 = pack(h1[2], h1[3]);
        const uint32_t j0 = pack(-h0[1], h0[0]), j1 = pack(-h1[1], h1[0]), j2 = pack(-h0[3], h0[2]), j3 = pack(-h1[3], h1[2]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {  // (rows behind the last are zeros)
          const int i = 4 * kk + m;
          if (i + 1 < 4 * KK) load_c(i + 1);
          ms::mma(y[m][0], a[i & 1], g0, g1);
          ms::mma(y[m][1], a[i & 1], g2, g3);
          ms::mma(z[m][0], a[i & 1], j0, j1);
          ms::mma(z[m][1], a[i & 1], j2, j3);
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int i0 = 16 * m + lane / 4;
        const float f0 = ex2(rec.L[i0]), f1 = ex2(rec.L[i0 + 8]);
        const float c0 = rec.co[i0] * f0, s0 = rec.si[i0] * f0, c1 = rec.co[i0 + 8] * f1, s1 = rec.si[i0 + 8] * f1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float *a = y[m][c], *b = z[m][c];
          const float2 u = unpack2(mad2(dup2(c0), pack2(a[0], a[1]), mul2(dup2(s0), pack2(b[0], b[1])))),
                       v = unpack2(mad2(dup2(c1), pack2(a[2], a[3]), mul2(dup2(s1), pack2(b[2], b[3]))));
          a[0] = u.x; a[1] = u.y; a[2] = v.x; a[3] = v.y;
        }
      }
      // M x, below the diagonal's tiles and on them.  There, rows in front of a step meet its x with a weight of 0, which an x that
      // is not finite does not leave at 0: with one in the chunk its tiles on the diagonal are summed term by term.
      uint32_t xv[4][4];
      __nv_bfloat162 odd = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        ms::ldsm_t(xv[kk], xb + at<8>(16 * kk + r16, 2 * w + hi));
#pragma unroll
        for (int m = kk + 1; m < 4; ++m) {
          const uint4 v = s.m[k & 1][(m * (m + 1) / 2 + kk) * 32 + lane];
          const uint32_t a[4] = {v.x, v.y, v.z, v.w};
          ms::mma(y[m][0], a, xv[kk][0], xv[kk][1]);
          ms::mma(y[m][1], a, xv[kk][2], xv[kk][3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) odd = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&xv[kk][i]), __floats2bfloat162_rn(0.f, 0.f), odd);
      }
      if (!__any_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&odd) << 1 & 0xfffefffeu)) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint4 v = s.m[k & 1][m * (m + 3) / 2 * 32 + lane];
          const uint32_t a[4] = {v.x, v.y, v.z, v.w};
          ms::mma(y[m][0], a, xv[m][0], xv[m][1]);
          ms::mma(y[m][1], a, xv[m][2], xv[m][3]);
        }
      } else {
#pragma unroll 1
        for (int j = 0; j < 16; ++j)
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const bf16* row = reinterpret_cast<const bf16*>(&s.m[k & 1][m * (m + 3) / 2 * 32 + (lane & 28) + (j & 7) / 2]) + (j / 8) * 4 + (j & 1);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t v;
              asm("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(xb + at<8>(16 * m + j, 2 * w + c) + (lane & 3) * 4) : "memory");
              const float2 xj = unpack(v);
#pragma unroll
              for (int low = 0; low < 2; ++low)
                if (j <= lane / 4 + 8 * low) {
                  const float weight = __bfloat162float(row[2 * low]);
                  y[m][c][2 * low] = fmaf(weight, xj.x, y[m][c][2 * low]);
                  y[m][c][2 * low + 1] = fmaf(weight, xj.y, y[m][c][2 * low + 1]);
                }
            }
          }
      }
      // Four lanes hold a row's 2 x 8 channels in pairs, for rows 8 apart: they exchange until each has 8 channels of one row.
      const int ql = lane % 4, left = q.last - t0 - lane / 4 - 8 * (ql >> 1), ch = 16 * w + 8 * (ql & 1);
      bf16* Y = static_cast<bf16*>(p.y) + (size_t)(t0 + lane / 4 + 8 * (ql >> 1)) * p.D + chan + ch;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        // v[r]: what lane r of the four is to have: row half r / 2, channels 8 (r % 2) ...
        uint32_t v[4] = {pack(y[m][0][0], y[m][0][1]), pack(y[m][1][0], y[m][1][1]), pack(y[m][0][2], y[m][0][3]), pack(y[m][1][2], y[m][1][3])};
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(r & o)) {
              const bool up = ql & o;
              const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[r] : v[r + o], o);
              if (up) v[r] = got;
              else v[r + o] = got;
            }
        if (16 * m < left && ch < np) {
          if (whole) *reinterpret_cast<uint4*>(Y) = make_uint4(v[0], v[1], v[2], v[3]);
          else
#pragma unroll
            for (int r = 0; r < 4; ++r) reinterpret_cast<uint32_t*>(Y)[r] = v[r];
        }
        Y += (size_t)16 * p.D;
      }
    }
    {
      const f2 decay = dup2(exp2f(rec.Lq));
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          const float2 v = unpack2(mul2(decay, pack2(h[t][c], h[t][c + 1])));
          h[t][c] = v.x;
          h[t][c + 1] = v.y;
        }
    }
    // h += (g cos x) (x) b - (g sin x) (x) J b, part after part of the weighted x
    const uint32_t sb = smem_at(s.b[k & 1]) + r16 * (U * 16);
    const int parts = k >= from3 ? 3 : k >= from2 ? 2 : 1;
#pragma unroll 1
    for (int part = 0; part < parts; ++part) {
      bar_sync(kWeighted, 2 * kThreads);
      uint32_t xc[Q / 16][4], xs[Q / 16][4];
#pragma unroll
      for (int kk = 0; kk < Q / 16; ++kk) {
        const uint4 a = s.gx[w][kk][0][lane], b = s.gx[w][kk][1][lane];
        xc[kk][0] = a.x; xc[kk][1] = a.y; xc[kk][2] = a.z; xc[kk][3] = a.w;
        xs[kk][0] = b.x; xs[kk][1] = b.y; xs[kk][2] = b.z; xs[kk][3] = b.w;
      }
      if (part + 1 < parts) bar_arrive(kPart, 2 * kThreads);  // (this part is in registers: the next is made ready meanwhile)
      uint32_t b[2][4];
      auto load_b = [&](int i) { ms::ldsm_t(b[i & 1], sb + (i % 4) * (16 * U * 16) + (((2 * (i / 4) + hi) ^ (lane & 7)) << 4)); };
      load_b(0);
#pragma unroll
      for (int t = 0; t < NT / 2; ++t) {
        float v[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < Q / 16; ++kk) {
          const int i = 4 * t + kk;
          if (i + 1 < 2 * NT) load_b(i + 1);
          ms::mma(h[2 * t], xc[kk], b[i & 1][0], b[i & 1][1]);
          ms::mma(h[2 * t + 1], xc[kk], b[i & 1][2], b[i & 1][3]);
          ms::mma(v[0], xs[kk], b[i & 1][0], b[i & 1][1]);
          ms::mma(v[1], xs[kk], b[i & 1][2], b[i & 1][3]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < 4; c += 2) {
            h[2 * t + i][c] += v[i][c + 1];
            h[2 * t + i][c + 1] -= v[i][c];
          }
      }
    }
    turn += rec.turn;
    taint += rec.taint;
    dsum += rec.dsum;
    bar_arrive(kEmpty + (k & 1), 2 * kThreads);
  }

  if (ENDS && tid == 0 && slab == 0) {
    p.turn[(size_t)piece * p.NH + hd] = turn;
    p.dsum[(size_t)piece * p.NH + hd] = dsum + taint;
  }
  if (!keeps) return;
  const float2 ran = m3_unit(turn, taint), by = ENDS ? ran : make_float2(start.x, -start.y);  // (R turns on, and back by the conjugate)
  float* to = (ENDS ? p.ends + ((size_t)piece * p.D + chan + row0) * p.N : p.h + ((size_t)slot * p.D + chan + row0) * p.N) + n0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (rows_in[k] && 8 * t < p.N)
        *reinterpret_cast<float2*>(to + (size_t)8 * k * p.N + 8 * t) = m3_on(make_float2(h[t][2 * k], h[t][2 * k + 1]), by);
  // (the slabs of a head all read its phase and b_prev; with more than one they are written behind this launch)
  // (every thread has read them: barriers lie between)
  if (!ENDS && p.slabs == 1) {
    if (tid == 0) p.phase[ph] = m3_turned(start, ran);
    serve_tail<bf16>(p, q.end - 1, slot, hd, grp, kThreads);
  } else if (!ENDS && tid == 0 && slab == 0) {
    p.phase_end[(size_t)q.seq * p.NH + hd] = m3_turned(start, ran);
  }
}

// The split of the registers waits for good where the kernel starts with fewer than it counts on: looked up once.
static mxb_status registers_ok(const void* kernel) {
  cudaFuncAttributes a{};
  const cudaError_t e = cudaFuncGetAttributes(&a, kernel);
  if (e != cudaSuccess) { set_last_cuda_error((int)e); return MXB_ERR_CUDA; }
  return a.numRegs >= (kReady + kMultiply) / 2 ? MXB_OK : MXB_ERR_UNSUPPORTED;
}
template <int N>
static mxb_status launch(const ServeP& p, bool ends, cudaStream_t st) {
  const int smem = (int)sizeof(Smem<N>);
  auto go = [&](auto kernel, const char* name) {
    MXB_LAUNCH(name, st, (launch_kernel(kernel, dim3((unsigned)((size_t)(ends ? p.rows / p.L : p.pieces) * p.NH * p.slabs)), 2 * kThreads, smem, st, p)));
    return check_launch(name);
  };
  static std::atomic<bool> looked_up{false};
  if (!looked_up.load(std::memory_order_relaxed)) {
    for (const void* k : {reinterpret_cast<const void*>(m3p_chunks_kernel<N, true>), reinterpret_cast<const void*>(m3p_chunks_kernel<N, false>)})
      if (const mxb_status s = registers_ok(k); s != MXB_OK) return s;
    looked_up.store(true, std::memory_order_relaxed);
  }
  if (ends) {
    const mxb_status s = MXB_ALLOW_SMEM(smem, m3p_chunks_kernel<N, true>);
    return s == MXB_OK ? go(m3p_chunks_kernel<N, true>, "m3p_chunks_ends_kernel") : s;
  }
  const mxb_status s = MXB_ALLOW_SMEM(smem, m3p_chunks_kernel<N, false>);
  return s == MXB_OK ? go(m3p_chunks_kernel<N, false>, "m3p_chunks_kernel") : s;
}

}  // namespace m3p

// Whole 16-byte pieces of rows, a b_prev of whole pairs (read by elements, 256 short prompts take 437 us for 412), a state that
// fits the registers of four warps, and rows enough for chunks of 64 to be worth it: more than 16 in the call and more than 4 a
// sequence (the host knows their mean only).  us, chunks / walk, 128 states:
//   one prompt of 16 rows, 32 heads          14 / 14     of 24 rows 16 / 18     of 64 rows 16 / 35
//   256 prompts of 32 heads, 1 row each     410 / 288    4 rows 412 / 326       8 rows 412 / 375    16 rows 414 / 474
//   64 prompts of 8 heads, 1 row each        33 / 20     4 rows  38 / 26        8 rows  38 / 30     24 rows  39 / 48
// Tokens beside one prompt are what the line is not drawn further out for: 8 heads, 255 of them beside 512 rows (3 a sequence)
// 134 / 129, 63 beside 256 rows (5 a sequence) 46 / 71, 15 beside 128 (9 a sequence) 29 / 54.
static bool m3prompt_shape(const ServeP& p, bool f32) {
  return !f32 && p.NH > 0 && p.N % 8 == 0 && p.N <= 128 && p.P % 8 == 0 && p.rows > 16 && p.rows > 4 * (long long)p.S;
}
bool m3prompt_supported(const ServeP& p, bool f32) {
  auto al = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  return m3prompt_shape(p, f32) && al(p.x) && al(p.b) && al(p.c) && (reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.b_prev)) % 4 == 0;
}
mxb_status m3prompt_prepare(const ServeP& p, cudaStream_t st) {
  const dim3 grid(p.chunks, p.G + (p.NH + m3p::kRecHeads - 1) / m3p::kRecHeads);
  MXB_LAUNCH("m3p_prepare_kernel", st,
             (launch_kernel(p.N <= 64 ? m3p::m3p_prepare_kernel<64> : m3p::m3p_prepare_kernel<128>, grid, m3p::kThreads, 0, st, p)));
  return check_launch("m3p_prepare");
}
mxb_status m3prompt_chunks(const ServeP& p, bool ends, cudaStream_t st) {
  return p.N <= 64 ? m3p::launch<64>(p, ends, st) : m3p::launch<128>(p, ends, st);
}

}  // namespace mxb
