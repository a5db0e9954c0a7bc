// The residual stream between two blocks, in one pass over its rows:
//     a = RMSNorm(y; post_norm) SiLU(z);   r' = r + scale a;   n = RMSNorm(r'; norm)
// (post_norm, z and scale may be absent), and its gradients: with k = 1 / rms(r'), t = dn norm,
//     d  = dr' + k (t - r' k^2 mean(t r'))          the gradient of r' from both its readers; dr = d
//     s  = d scale post_norm SiLU(z)
//     dy = j (s - y j^2 mean(s y)), j = 1 / rms(y)  (s itself without post_norm)
//     dz = d scale post_norm y j SiLU'(z),  dnorm = sum dn r' k,  dpost_norm = sum d scale y j SiLU(z),  dscale = sum d a
//
// HBM streams.  A row is read once, held by TPR threads in 8 (beyond 8192 columns 16) registers a tensor, and its sums go
// through the lanes and, for TPR > 32, shared memory; narrow rows share a CTA.  Column sums of the gradients: every group of
// TPR threads walks over rows with its columns' sums in registers and leaves a partial row; a second launch adds those in a
// fixed order.  Everything is computed in float32 whatever the tensors' types.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

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
  float* part;                        // [groups][3][D]
};

// 8 consecutive columns from c0, those below D: V says that whole pieces may be read.
template <typename T, bool V>
__device__ __forceinline__ void load8(const T* row, int c0, int D, float (&e)[8]) {
  if constexpr (V) {
    if (c0 < D) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 a = *reinterpret_cast<const float4*>(row + c0 + 4 * i);
          e[4 * i] = a.x; e[4 * i + 1] = a.y; e[4 * i + 2] = a.z; e[4 * i + 3] = a.w;
        }
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(row + c0);
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { e[2 * i] = __low2float(h[i]); e[2 * i + 1] = __high2float(h[i]); }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c0 + i < D ? to_f32(row[c0 + i]) : 0.f;
  }
}
template <typename T, bool V>
__device__ __forceinline__ void store8(T* row, int c0, int D, const float (&e)[8]) {
  if constexpr (V) {
    if (c0 >= D) return;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) *reinterpret_cast<float4*>(row + c0 + 4 * i) = make_float4(e[4 * i], e[4 * i + 1], e[4 * i + 2], e[4 * i + 3]);
    } else {
      uint4 v;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(e[2 * i], e[2 * i + 1]);
      *reinterpret_cast<uint4*>(row + c0) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < D) row[c0 + i] = from_f32<T>(e[i]);
  }
}
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
__device__ __forceinline__ float sigmoid_of(float z) { return 1.f / (1.f + expf(-z)); }

template <int TPR>
constexpr int kThreads = TPR > 256 ? TPR : 256;

template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>) rnorm_fwd_kernel(NormP p) {
  begin_dependent();
  __shared__ float red[kThreads<TPR> / 32];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = (live ? r0 + group : r0) * p.D;
    float r[E][8], a[E][8];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      load8<IO, V>(static_cast<const IO*>(p.y) + off, c, p.D, a[e]);
      load8<RES, V>(static_cast<const RES*>(p.resid) + off, c, p.D, r[e]);
    }
    if (p.z) {
      float s[1] = {0.f};
      float zs[E][8];
#pragma unroll
      for (int e = 0; e < E; ++e) load8<IO, V>(static_cast<const IO*>(p.z) + off, (lane + e * TPR) * 8, p.D, zs[e]);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[0] = fmaf(a[e][i], a[e][i], s[0]);
          a[e][i] *= zs[e][i] * sigmoid_of(zs[e][i]);
        }
      if (p.post) {
        row_sum<TPR>(s, red);
        const float j = rsqrtf(s[0] * inv + p.eps);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i) a[e][i] *= j;
      }
    } else if (p.post) {
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] = fmaf(a[e][i], a[e][i], s[0]);
      row_sum<TPR>(s, red);
      const float j = rsqrtf(s[0] * inv + p.eps);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) a[e][i] *= j;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      float w[8];
      if (p.post) {
        load8<float, V>(p.post, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[e][i] *= w[i];
      }
      if (p.scale) {
        load8<float, V>(p.scale, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[e][i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[e][i] += a[e][i];
        s[0] = fmaf(r[e][i], r[e][i], s[0]);
      }
      if (live) store8<RES, V>(static_cast<RES*>(p.resid_out) + off, c, p.D, r[e]);
    }
    row_sum<TPR>(s, red);
    const float k = rsqrtf(s[0] * inv + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      float w[8];
      load8<float, V>(p.norm, c, p.D, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] *= r[e][i] * k;
      if (live) store8<IO, V>(static_cast<IO*>(p.n) + off, c, p.D, w);
    }
  }
}

template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>) rnorm_bwd_kernel(NormP p) {
  begin_dependent();
  __shared__ float red[kThreads<TPR> / 32 * 3];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  float dnorm[E][8], dpost[E][8], dscale[E][8];
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < 8; ++i) dnorm[e][i] = dpost[e][i] = dscale[e][i] = 0.f;
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = (live ? r0 + group : r0) * p.D;
    float r[E][8], y[E][8], g[E][8], d[E][8], s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      load8<RES, V>(static_cast<const RES*>(p.resid) + off, c, p.D, r[e]);
      load8<IO, V>(static_cast<const IO*>(p.dn) + off, c, p.D, g[e]);
      load8<IO, V>(static_cast<const IO*>(p.y) + off, c, p.D, y[e]);
      if (p.d_resid) {
        load8<RES, V>(static_cast<const RES*>(p.d_resid) + off, c, p.D, d[e]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[e][i] = 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float w[8];
      load8<float, V>(p.norm, (lane + e * TPR) * 8, p.D, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[0] = fmaf(r[e][i], r[e][i], s[0]);
        s[1] = fmaf(g[e][i] * w[i], r[e][i], s[1]);
        s[2] = fmaf(y[e][i], y[e][i], s[2]);
      }
    }
    row_sum<TPR>(s, red);
    const float k = rsqrtf(s[0] * inv + p.eps), k2 = k * k * s[1] * inv, j = p.post ? rsqrtf(s[2] * inv + p.eps) : 1.f;
    float q[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * TPR) * 8;
      float w[8], z[8];
      load8<float, V>(p.norm, c, p.D, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (live) dnorm[e][i] = fmaf(g[e][i], r[e][i] * k, dnorm[e][i]);
        d[e][i] = fmaf(k, fmaf(-r[e][i], k2, g[e][i] * w[i]), d[e][i]);
      }
      if (live) store8<RES, V>(static_cast<RES*>(p.dr) + off, c, p.D, d[e]);
      // g <- d scale post SiLU(z): what reaches y j, and on the way the sums over the rows and dz
#pragma unroll
      for (int i = 0; i < 8; ++i) g[e][i] = d[e][i];
      float post[8], gate[8], slope[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { post[i] = 1.f; gate[i] = 1.f; slope[i] = 0.f; }
      if (p.post) load8<float, V>(p.post, c, p.D, post);
      if (p.z) {
        load8<IO, V>(static_cast<const IO*>(p.z) + off, c, p.D, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float sg = sigmoid_of(z[i]);
          gate[i] = z[i] * sg;
          slope[i] = fmaf(gate[i], 1.f - sg, sg);
        }
      }
      if (p.scale) {
        load8<float, V>(p.scale, c, p.D, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (live) dscale[e][i] = fmaf(d[e][i], y[e][i] * j * post[i] * gate[i], dscale[e][i]);
          g[e][i] *= w[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = g[e][i] * y[e][i] * j;
        if (live) dpost[e][i] = fmaf(t, gate[i], dpost[e][i]);
        slope[i] *= t * post[i];
        g[e][i] *= post[i] * gate[i];
        q[0] = fmaf(g[e][i], y[e][i], q[0]);
      }
      if (p.z && live) store8<IO, V>(static_cast<IO*>(p.dz) + off, c, p.D, slope);
    }
    if (p.post) row_sum<TPR>(q, red);
    const float j2 = p.post ? j * j * q[0] * inv : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[e][i] = j * fmaf(-y[e][i], j2, g[e][i]);
      if (live) store8<IO, V>(static_cast<IO*>(p.dy) + off, (lane + e * TPR) * 8, p.D, g[e]);
    }
  }
  float* part = p.part + ((size_t)blockIdx.x * GROUPS + group) * 3 * p.D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (lane + e * TPR) * 8;
    store8<float, false>(part, c, p.D, dnorm[e]);
    if (p.post) store8<float, false>(part + p.D, c, p.D, dpost[e]);
    if (p.scale) store8<float, false>(part + 2 * p.D, c, p.D, dscale[e]);
  }
}
// Sums of the partial rows.  grid (column blocks, 3): dnorm, dpost_norm, dscale; a null result is skipped.
struct SumP {
  const float* part;
  int rows, D;
  float* out[3];
};
template <bool TALL>
__global__ void __launch_bounds__(kSumThreads<TALL>) rnorm_sum_kernel(SumP p) {
  begin_dependent();
  float* out = p.out[blockIdx.y];
  if (!out) return;
  const int c0 = blockIdx.x * kSumCols<TALL>, mine = c0 + threadIdx.x % kSumCols<TALL>;
  col_sum<TALL>(p.part + blockIdx.y * (size_t)p.D + mine, p.rows, 3 * (size_t)p.D, mine < p.D, [&](int c, float t) {
    if (c0 + c < p.D) out[c0 + c] = t;
  });
}

// ------------------------------------------------------------------ host
static int threads_per_row(int D) {  // the smallest power of two with 8 columns a thread, 4 to 1024
  int t = 4;
  while (8 * t < D && t < 1024) t *= 2;
  return t;
}
static int groups_of(int tpr) { return tpr > 256 ? 1 : 256 / tpr; }
// CTAs: the gradients' column sums want few of them, a few a SM; the forward pass has a CTA for every group of rows.
static int ctas(size_t rows, int D, bool bwd) {
  const int tpr = threads_per_row(D), g = groups_of(tpr);
  const size_t want = (rows + g - 1) / g, most = bwd ? 148 * (tpr > 256 ? 1 : 2) : 1u << 30;
  return (int)std::min(want, most);
}
template <typename F>
static void by_shape(int D, F&& f) {
  auto call = [&](auto t) {
    if (D > 8192) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
    else f(t, std::integral_constant<int, 1>{});
  };
  switch (threads_per_row(D)) {
    case 4: call(std::integral_constant<int, 4>{}); break;
    case 8: call(std::integral_constant<int, 8>{}); break;
    case 16: call(std::integral_constant<int, 16>{}); break;
    case 32: call(std::integral_constant<int, 32>{}); break;
    case 64: call(std::integral_constant<int, 64>{}); break;
    case 128: call(std::integral_constant<int, 128>{}); break;
    case 256: call(std::integral_constant<int, 256>{}); break;
    case 512: call(std::integral_constant<int, 512>{}); break;
    default: call(std::integral_constant<int, 1024>{}); break;
  }
}
template <typename IO, typename RES, bool V>
static mxb_status run(const NormP& p, float* const (&sums)[3], cudaStream_t st) {
  const bool bwd = p.dn != nullptr;
  const int n = ctas(p.rows, p.D, bwd);
  int parts = 0;
  by_shape(p.D, [&](auto tpr, auto e) {
    constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
    if (bwd) {
      parts = n * (kThreads<TPR> / TPR);
      MXB_LAUNCH("rnorm_bwd_kernel", st, (launch_kernel(rnorm_bwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
    } else {
      MXB_LAUNCH("rnorm_fwd_kernel", st, (launch_kernel(rnorm_fwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
    }
  });
  if (bwd) {
    SumP s{p.part, parts, p.D, {sums[0], sums[1], sums[2]}};
    auto launch = [&](auto tall) {
      constexpr bool T = decltype(tall)::value;
      MXB_LAUNCH("rnorm_sum_kernel", st, (launch_kernel(rnorm_sum_kernel<T>, dim3((p.D + kSumCols<T> - 1) / kSumCols<T>, 3), kSumThreads<T>, 0, st, s)));
    };
    if (col_sum_tall(3 * (size_t)p.D)) launch(std::true_type{});
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
  return at % 16 == 0 && p.D % 8 == 0 ? run<IO, RES, true>(p, sums, st) : run<IO, RES, false>(p, sums, st);
}
static mxb_status by_type(const mxb_residual_norm_desc* d, const NormP& p, float* const (&sums)[3], cudaStream_t st) {
  if (d->io_dtype == MXB_F32) return by_alignment<float, float>(p, sums, st);
  if (d->resid_dtype == MXB_F32) return by_alignment<bf16, float>(p, sums, st);
  return by_alignment<bf16, bf16>(p, sums, st);
}

}  // namespace rnorm

size_t residual_norm_scratch(const mxb_residual_norm_desc* d) {
  const int tpr = rnorm::threads_per_row(d->D);
  return (size_t)rnorm::ctas(d->rows, d->D, true) * rnorm::groups_of(tpr) * 3 * d->D * sizeof(float);
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
