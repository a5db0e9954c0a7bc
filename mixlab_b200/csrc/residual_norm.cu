// The residual stream between two blocks, in one pass over its rows:
//     a = RMSNorm(y; post_norm) SiLU(z);   r' = r + scale a;   n = RMSNorm(r'; norm)
// (post_norm, z and scale may be absent), and its gradients: with k = 1 / rms(r'), t = dn norm,
//     d  = dr' + k (t - r' k^2 mean(t r'))          the gradient of r' from both its readers; dr = d
//     s  = d scale post_norm SiLU(z)
//     dy = j (s - y j^2 mean(s y)), j = 1 / rms(y)  (s itself without post_norm)
//     dz = d scale post_norm y j SiLU'(z),  dnorm = sum dn r' k,  dpost_norm = scale A,  dscale = post_norm A,
//     A = sum d y j SiLU(z) over the rows
//
// HBM streams: 8191 rows of 2048 columns, bf16 with a float32 stream, gate and scale, 42 us (235 MB: 86 % of the measured copy
// rate); every gradient of 32768 rows in bf16 218 to 229 us (1.07 GB: 72 to 75 %), 8 of them in the column sums' own launch; with
// scale alone, as behind a block's output projection, 32768 rows in bf16 85 us forwards (96 %) and 152 back (81 %); one row 6.1
// us, of which the call on the host is most.  A row is read once, held by TPR threads in 8 registers a tensor (16 or 32 for the
// widest rows), and its sums go through the lanes and, for TPR > 32, shared memory; narrow rows share a CTA.  Gradients of more
// than 4096 columns do not fit the 128 registers that 512 threads have: 0.4 KB a thread go through local memory, beyond 8192
// columns 1.2 to 1.9 KB, and rows of 8192 and 16384 columns reach 42 and 24 % of the copy rate.  Column sums of the gradients:
// every group of TPR threads walks over rows with its columns' sums in registers and leaves a partial row; a second launch adds
// those in a fixed order.  Everything is computed in float32 whatever the tensors' types.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"

namespace mxb {
namespace rnorm {

using bf16 = __nv_bfloat16;

struct NormP {
  size_t rows;
  int D;
  float eps;
  const void *resid, *y, *z;          // backward: resid is what the forward returned
  const float *norm, *post, *scale;   // post, scale may be null
  void *resid_out, *n;
  const void *d_resid, *dn;           // d_resid may be null
  void *dr, *dy, *dz;
  float* part;                        // [groups][2][D]: dnorm, A
};

// 8 consecutive columns from c0, those below D, as four packed pairs.  V says that whole pieces may be read.
__device__ __forceinline__ void unpack8(const uint4& v, f2 (&e)[4]) {  // eight bf16
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <typename T, bool V>
__device__ __forceinline__ void load8(const T* row, int c0, int D, f2 (&e)[4]) {
  if constexpr (V) {
    if (c0 < D) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 a = *reinterpret_cast<const float4*>(row + c0 + 4 * i);
          e[2 * i] = pack2(a.x, a.y);
          e[2 * i + 1] = pack2(a.z, a.w);
        }
      } else {
        unpack8(*reinterpret_cast<const uint4*>(row + c0), e);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = 0;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 2 * i;
      e[i] = pack2(c < D ? to_f32(row[c]) : 0.f, c + 1 < D ? to_f32(row[c + 1]) : 0.f);
    }
  }
}
template <typename T, bool V>
__device__ __forceinline__ void store8(T* row, int c0, int D, const f2 (&e)[4]) {
  if constexpr (V) {
    if (c0 >= D) return;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 a = unpack2(e[2 * i]), b = unpack2(e[2 * i + 1]);
        *reinterpret_cast<float4*>(row + c0 + 4 * i) = make_float4(a.x, a.y, b.x, b.y);
      }
    } else {
      uint4 v;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) { const float2 a = unpack2(e[i]); h[i] = __floats2bfloat162_rn(a.x, a.y); }
      *reinterpret_cast<uint4*>(row + c0) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(e[i]);
      const int c = c0 + 2 * i;
      if (c < D) row[c] = from_f32<T>(a.x);
      if (c + 1 < D) row[c + 1] = from_f32<T>(a.y);
    }
  }
}
// A piece of a row as it is in memory, requested ahead of its use (whole pieces only; else read when it is used).
template <typename T, bool V>
struct Ahead {
  static constexpr int W = sizeof(T) == 4 ? 2 : 1;
  uint4 raw[V ? W : 1];
  __device__ __forceinline__ void load(const T* row, int c0, int D) {
    if constexpr (V) {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = c0 < D ? reinterpret_cast<const uint4*>(row + c0)[i] : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void get(const T* row, int c0, int D, f2 (&e)[4]) const {
    if constexpr (!V) {
      load8<T, false>(row, c0, D, e);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        e[2 * i] = pack2(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y));
        e[2 * i + 1] = pack2(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w));
      }
    } else {
      unpack8(raw[0], e);
    }
  }
};
// Sums of M values over the TPR threads of a row; every thread gets them.  red: shared, M floats a warp.  All threads of the
// CTA call it.
template <int TPR, int M>
__device__ __forceinline__ void row_sum(float (&v)[M], float* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // (the last sums have been read)
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int m = 0; m < M; ++m) red[warp * M + m] = v[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[(warp / W * W + w) * M + m];
      v[m] = s;
    }
  }
}
// (bf16 tensors: the hardware's exponential and division, good to a few 2^-22 where results keep 2^-9)
template <typename IO>
__device__ __forceinline__ float sigmoid_of(float z) { return sizeof(IO) == 4 ? 1.f / (1.f + expf(-z)) : __fdividef(1.f, 1.f + __expf(-z)); }

// z -> SiLU(z) and, where wanted, its slope
template <typename IO>
__device__ __forceinline__ void gate_of(f2 z, f2& gate, f2& slope) {
  const float2 v = unpack2(z);
  const f2 sg = pack2(sigmoid_of<IO>(v.x), sigmoid_of<IO>(v.y));
  gate = mul2(z, sg);
  slope = mad2(gate, add2(dup2(1.f), sg ^ 0x8000000080000000ull), sg);
}

template <int TPR>
constexpr int kThreads = TPR > 256 ? TPR : 256;

template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>) rnorm_fwd_kernel(NormP p) {
  begin_dependent();
  __shared__ float red[kThreads<TPR> / 32];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  // the next row of each tensor is under way while one is worked on
  Ahead<RES, V> a_r[E];
  Ahead<IO, V> a_y[E], a_z[E];
  auto offset = [&](size_t r0) { return (r0 + group < p.rows ? r0 + group : r0) * p.D; };
  auto request = [&](size_t r0) {
    const size_t off = offset(r0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      a_y[e].load(static_cast<const IO*>(p.y) + off, c, p.D);
      a_r[e].load(static_cast<const RES*>(p.resid) + off, c, p.D);
      if (p.z) a_z[e].load(static_cast<const IO*>(p.z) + off, c, p.D);
    }
  };
  request((size_t)blockIdx.x * GROUPS);
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = offset(r0);
    f2 r[E][4], a[E][4];
    f2 sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      a_y[e].get(static_cast<const IO*>(p.y) + off, c, p.D, a[e]);
      a_r[e].get(static_cast<const RES*>(p.resid) + off, c, p.D, r[e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) fma2(sum, a[e][i], a[e][i]);
      if (p.z) {
        f2 z[4], gate, slope;
        a_z[e].get(static_cast<const IO*>(p.z) + off, c, p.D, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          gate_of<IO>(z[i], gate, slope);
          a[e][i] = mul2(a[e][i], gate);
        }
      }
    }
    if (r0 + (size_t)gridDim.x * GROUPS < p.rows) request(r0 + (size_t)gridDim.x * GROUPS);
    float s[1], j = 1.f;
    if (p.post) {
      s[0] = sum2(sum);
      row_sum<TPR>(s, red);
      j = rsqrtf(s[0] * inv + p.eps);
    }
    sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      f2 w[4];
      if (p.post) {
        load8<float, V>(p.post, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[e][i] = mul2(mul2(a[e][i], dup2(j)), w[i]);
      }
      if (p.scale) {
        load8<float, V>(p.scale, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[e][i] = mul2(a[e][i], w[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[e][i] = add2(r[e][i], a[e][i]);
        fma2(sum, r[e][i], r[e][i]);
      }
      if (live) store8<RES, V>(static_cast<RES*>(p.resid_out) + off, c, p.D, r[e]);
    }
    s[0] = sum2(sum);
    row_sum<TPR>(s, red);
    const float k = rsqrtf(s[0] * inv + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      f2 w[4];
      load8<float, V>(p.norm, c, p.D, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], mul2(r[e][i], dup2(k)));
      if (live) store8<IO, V>(static_cast<IO*>(p.n) + off, c, p.D, w);
    }
  }
}

template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>, TPR > 256 || E > 1 ? 1 : 2) rnorm_bwd_kernel(NormP p) {
  begin_dependent();
  __shared__ float red[kThreads<TPR> / 32 * 3];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  f2 dnorm[E][4], both[E][4];
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) dnorm[e][i] = both[e][i] = 0;
  // the next row of each tensor is under way while one is worked on (where there are registers for it)
  constexpr bool EARLY = TPR <= 256;
  Ahead<RES, V> a_r[E], a_d[E];
  Ahead<IO, V> a_g[E], a_y[E], a_z[E];
  auto offset = [&](size_t r0) { return (r0 + group < p.rows ? r0 + group : r0) * p.D; };
  auto request = [&](size_t r0) {
    const size_t off = offset(r0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      a_r[e].load(static_cast<const RES*>(p.resid) + off, c, p.D);
      a_g[e].load(static_cast<const IO*>(p.dn) + off, c, p.D);
      a_y[e].load(static_cast<const IO*>(p.y) + off, c, p.D);
      if (p.d_resid) a_d[e].load(static_cast<const RES*>(p.d_resid) + off, c, p.D);
      if (p.z) a_z[e].load(static_cast<const IO*>(p.z) + off, c, p.D);
    }
  };
  if (EARLY) request((size_t)blockIdx.x * GROUPS);
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = offset(r0);
    f2 r[E][4], y[E][4], g[E][4], d[E][4], z[E][4], s0 = 0, s1 = 0, s2 = 0;
    if (!EARLY) request(r0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      a_r[e].get(static_cast<const RES*>(p.resid) + off, c, p.D, r[e]);
      a_g[e].get(static_cast<const IO*>(p.dn) + off, c, p.D, g[e]);
      a_y[e].get(static_cast<const IO*>(p.y) + off, c, p.D, y[e]);
      if (p.d_resid) {
        a_d[e].get(static_cast<const RES*>(p.d_resid) + off, c, p.D, d[e]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[e][i] = 0;
      }
      if (p.z) a_z[e].get(static_cast<const IO*>(p.z) + off, c, p.D, z[e]);
    }
    if (EARLY && r0 + (size_t)gridDim.x * GROUPS < p.rows) request(r0 + (size_t)gridDim.x * GROUPS);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f2 w[4];
      load8<float, V>(p.norm, (lane + e * TPR) * 8, p.D, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fma2(s0, r[e][i], r[e][i]);
        fma2(s1, mul2(g[e][i], w[i]), r[e][i]);
        fma2(s2, y[e][i], y[e][i]);
      }
    }
    float s[3] = {sum2(s0), sum2(s1), sum2(s2)};
    row_sum<TPR>(s, red);
    const float k = rsqrtf(s[0] * inv + p.eps), k2 = k * k * s[1] * inv, j = p.post ? rsqrtf(s[2] * inv + p.eps) : 1.f;
    const f2 kk = dup2(k), mk2 = dup2(-k2), jj = dup2(j);
    f2 qs = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      f2 w[4], f[4];
      load8<float, V>(p.norm, c, p.D, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (live) fma2(dnorm[e][i], g[e][i], mul2(r[e][i], kk));
        d[e][i] = mad2(kk, mad2(r[e][i], mk2, mul2(g[e][i], w[i])), d[e][i]);
      }
      if (live) store8<RES, V>(static_cast<RES*>(p.dr) + off, c, p.D, d[e]);
      if (p.post) {
        load8<float, V>(p.post, c, p.D, f);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = dup2(1.f);
      }
      if (p.scale) {
        load8<float, V>(p.scale, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = mul2(f[i], w[i]);
      }
      // g <- d scale post SiLU(z): what reaches y j; on the way A and dz
      if (p.z) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f2 gate, slope;
          gate_of<IO>(z[e][i], gate, slope);
          const f2 dy = mul2(mul2(d[e][i], y[e][i]), jj);
          if (live) fma2(both[e][i], dy, gate);
          z[e][i] = mul2(slope, mul2(dy, f[i]));
          g[e][i] = mul2(mul2(d[e][i], f[i]), gate);
          fma2(qs, g[e][i], y[e][i]);
        }
        if (live) store8<IO, V>(static_cast<IO*>(p.dz) + off, c, p.D, z[e]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (live) fma2(both[e][i], mul2(d[e][i], y[e][i]), jj);
          g[e][i] = mul2(d[e][i], f[i]);
          fma2(qs, g[e][i], y[e][i]);
        }
      }
    }
    float q[1] = {sum2(qs)};
    if (p.post) row_sum<TPR>(q, red);
    const f2 mj2 = dup2(p.post ? -j * j * q[0] * inv : 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[e][i] = mul2(jj, mad2(y[e][i], mj2, g[e][i]));
      if (live) store8<IO, V>(static_cast<IO*>(p.dy) + off, (lane + e * TPR) * 8, p.D, g[e]);
    }
  }
  float* part = p.part + ((size_t)blockIdx.x * GROUPS + group) * 2 * p.D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (lane + e * TPR) * 8;
    store8<float, false>(part, c, p.D, dnorm[e]);
    store8<float, false>(part + p.D, c, p.D, both[e]);
  }
}
// Sums of the partial rows.  grid (column blocks, 1 or 2): dnorm; A, and from it dpost_norm and dscale.
struct SumP {
  const float* part;
  int rows, D;
  float *dnorm, *dpost, *dscale;
  const float *post, *scale;
};
template <bool TALL>
__global__ void __launch_bounds__(kSumThreads<TALL>) rnorm_sum_kernel(SumP p) {
  begin_dependent();
  const int c0 = blockIdx.x * kSumCols<TALL>, mine = c0 + threadIdx.x % kSumCols<TALL>;
  col_sum<TALL>(p.part + blockIdx.y * (size_t)p.D + mine, p.rows, 2 * (size_t)p.D, mine < p.D, [&](int c, float t) {
    c += c0;
    if (c >= p.D) return;
    if (blockIdx.y == 0) {
      p.dnorm[c] = t;
    } else {
      if (p.dpost) p.dpost[c] = p.scale ? t * p.scale[c] : t;
      if (p.dscale) p.dscale[c] = p.post ? t * p.post[c] : t;
    }
  });
}

// ------------------------------------------------------------------ host
static int threads_per_row(int D) {  // the smallest power of two with 8 columns a thread, 4 to 1024
  int t = 4;
  while (8 * t < D && t < 1024) t *= 2;
  return t;
}
// Threads of a row, pieces of 8 columns a thread.  The gradients hold six tensors' pieces and the columns' sums: beyond 2048 columns
// one CTA of fewer threads with more registers (16384 rows of 4096 columns in bf16 250 us, with 512 threads 326; 8192 of 8192 375,
// with 1024 threads 747), up to there two CTAs (32768 rows of 2048 218 us; with half of the threads a row 279).
struct RowShape { int tpr, e; };
static RowShape row_shape(int D, bool bwd) {
  const int t = threads_per_row(D);
  if (!bwd) return {t, D > 8192 ? 2 : 1};
  if (D <= 2048) return {t, 1};
  if (D <= 4096) return {t / 2, 2};
  return {512, D > 8192 ? 4 : 2};
}
static int groups_of(int tpr) { return tpr > 256 ? 1 : 256 / tpr; }
// CTAs: what the GPU holds at once, 4 an SM forwards and, by registers, 2 backwards (8191 rows of 2048 columns 42.6 us, 49.7 with
// half of them, 43.0 with twice as many), or one with two pieces a thread.
static int ctas(size_t rows, int D, bool bwd) {
  const RowShape s = row_shape(D, bwd);
  const int g = groups_of(s.tpr);
  const size_t want = (rows + g - 1) / g, most = std::max(148, 148 * (!bwd ? 4 : s.e == 1 ? 2 : 1) * 256 / std::max(s.tpr, 256));
  return (int)std::min(want, most);
}
template <typename F>
static void by_shape(int D, bool bwd, F&& f) {
  const RowShape s = row_shape(D, bwd);
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  if (bwd && s.e > 1) {
    switch (s.tpr) {
      case 256: f(std::integral_constant<int, 256>{}, two); break;
      default:
        if (s.e == 2) f(std::integral_constant<int, 512>{}, two);
        else f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
    }
    return;
  }
  switch (s.tpr) {
    case 4: f(std::integral_constant<int, 4>{}, one); break;
    case 8: f(std::integral_constant<int, 8>{}, one); break;
    case 16: f(std::integral_constant<int, 16>{}, one); break;
    case 32: f(std::integral_constant<int, 32>{}, one); break;
    case 64: f(std::integral_constant<int, 64>{}, one); break;
    case 128: f(std::integral_constant<int, 128>{}, one); break;
    case 256: f(std::integral_constant<int, 256>{}, one); break;
    case 512: f(std::integral_constant<int, 512>{}, one); break;
    default:
      if (s.e == 1) f(std::integral_constant<int, 1024>{}, one);
      else f(std::integral_constant<int, 1024>{}, two);
  }
}
template <typename IO, typename RES, bool V>
static mxb_status run(const NormP& p, float* const (&sums)[3], cudaStream_t st) {
  const bool bwd = p.dn != nullptr;
  const int n = ctas(p.rows, p.D, bwd);
  int parts = 0;
  by_shape(p.D, bwd, [&](auto tpr, auto e) {
    constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
    // (row_shape(): which there are)
    if constexpr (E == 1 ? TPR <= 256 : TPR <= 512)
      if (bwd) {
        parts = n * (kThreads<TPR> / TPR);
        MXB_LAUNCH("rnorm_bwd_kernel", st, (launch_kernel(rnorm_bwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
      }
    if constexpr (E == 1 || TPR > 512)
      if (!bwd) MXB_LAUNCH("rnorm_fwd_kernel", st, (launch_kernel(rnorm_fwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
  });
  if (bwd) {
    const SumP s{p.part, parts, p.D, sums[0], sums[1], sums[2], p.post, p.scale};
    const int kinds = sums[1] || sums[2] ? 2 : 1;
    auto launch = [&](auto tall) {
      constexpr bool T = decltype(tall)::value;
      MXB_LAUNCH("rnorm_sum_kernel", st, (launch_kernel(rnorm_sum_kernel<T>, dim3((p.D + kSumCols<T> - 1) / kSumCols<T>, kinds), kSumThreads<T>, 0, st, s)));
    };
    if (col_sum_tall(kinds * (size_t)p.D)) launch(std::true_type{});
    else launch(std::false_type{});
  }
  return check_launch(bwd ? "rnorm_bwd" : "rnorm_fwd");
}
template <typename IO, typename RES>
static mxb_status by_alignment(const NormP& p, float* const (&sums)[3], cudaStream_t st) {
  uintptr_t at = 0;
  for (const void* q : {p.resid, p.y, p.z, (const void*)p.norm, (const void*)p.post, (const void*)p.scale, (const void*)p.resid_out,
                        (const void*)p.n, p.d_resid, p.dn, (const void*)p.dr, (const void*)p.dy, (const void*)p.dz})
    at |= reinterpret_cast<uintptr_t>(q);
  // (whole pieces: 42.6 and 213 us for the rows above; single elements, which any row allows: 139 and 743)
  return at % 16 == 0 && p.D % 8 == 0 ? run<IO, RES, true>(p, sums, st) : run<IO, RES, false>(p, sums, st);
}
static mxb_status by_type(const mxb_residual_norm_desc* d, const NormP& p, float* const (&sums)[3], cudaStream_t st) {
  if (d->io_dtype == MXB_F32) return by_alignment<float, float>(p, sums, st);
  if (d->resid_dtype == MXB_F32) return by_alignment<bf16, float>(p, sums, st);
  return by_alignment<bf16, bf16>(p, sums, st);
}

}  // namespace rnorm

size_t residual_norm_scratch(const mxb_residual_norm_desc* d) {
  const int tpr = rnorm::row_shape(d->D, true).tpr;
  return (size_t)rnorm::ctas(d->rows, d->D, true) * rnorm::groups_of(tpr) * 2 * d->D * sizeof(float);
}
mxb_status residual_norm_fwd(const mxb_residual_norm_desc* d, const void* resid, const void* y, const float* norm, const float* post,
                             const void* z, const float* scale, void* resid_out, void* n, cudaStream_t st) {
  rnorm::NormP p{(size_t)d->rows, d->D, d->eps, resid, y, z, norm, post, scale, resid_out, n};
  return rnorm::by_type(d, p, {nullptr, nullptr, nullptr}, st);
}
mxb_status residual_norm_bwd(const mxb_residual_norm_desc* d, const void* resid, const void* y, const float* norm, const float* post,
                             const void* z, const float* scale, const void* d_resid, const void* dn, void* dr, void* dy, void* dz,
                             float* dnorm, float* dpost, float* dscale, float* part, cudaStream_t st) {
  rnorm::NormP p{(size_t)d->rows, d->D, d->eps, resid, y, z, norm, post, scale, nullptr, nullptr, d_resid, dn, dr, dy, dz, part};
  return rnorm::by_type(d, p, {dnorm, dpost, dscale}, st);
}

}  // namespace mxb
