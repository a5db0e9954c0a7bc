// The layer norm over the residual stream, in one pass over its rows:
//     h = r + x (x itself where there is no stream);   m = mean h,  k = 1 / sqrt(mean (h - m)^2 + eps);   n = (h - m) k w + b
// and its gradients: with u = (h - m) k, t = dn w,
//     dh = dh' + k (t - mean t - u mean(t u)),   dw = sum dn u,   db = sum dn     over the rows
// (dh' the gradient that reaches h from its other readers).
//
// HBM streams: 32768 rows of 2048 columns in bf16 with the addition to the stream 89 us (537 MB: 92 % of the measured copy rate), their
// gradients 106 (537 MB: 78 %), 5 of them in the column sums' own launch; 4001 rows of 449 columns in float32 9.7 us; one row 5.2,
// the call on the host.  The gradients are bound by instructions and the sums across a row (62 % of the issue slots, 48 % of the
// LSU pipe): two rows under way instead of one, and sums of each warp around its own mean, joined behind one barrier instead of two,
// were no faster.  Wide rows: 2048 of 8192 columns in bf16 33 us, their gradients 39 (134 MB: 21); of 16384 columns 49 and 187 (41).  The last
// holds six arrays of 32 floats a thread in 128 registers and spills up to 2 KB of them; float32, 16384 columns: 111 and 295 (82).
//
// A row is read once and held by TPR threads in pieces of eight columns, the next row is requested while one is worked on, narrow
// rows share a CTA.  The mean is taken first and the squares of what is left after it, both from registers: no difference of two
// large sums.  Column sums: every group of TPR threads walks over rows with its columns' sums in registers and leaves a partial
// row; a second launch adds those in a fixed order.  Everything is computed in float32.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "row_pieces.cuh"

namespace mxb {
namespace lnorm {

using bf16 = __nv_bfloat16;

struct NormP {
  size_t rows;
  int D;
  float eps;
  const void *resid, *x;         // forward: resid may be null, x then is the stream; backward: x is the stream
  const float *weight, *bias;    // bias may be null
  void *stream, *n;              // stream only with resid
  const void *d_resid, *dn;      // d_resid may be null
  void* dx;
  float* part;                   // [groups][2][D]: dw, db
};

template <int TPR>
constexpr int kThreads = TPR > 256 ? TPR : 256;

// h - m in the columns that there are, zero behind them.
template <bool V>
__device__ __forceinline__ void centre(f2 (&h)[4], int base, int lane, int tpr, int D, f2 minus_m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = add2(h[i], minus_m);
    if (V) {
      if (base + lane * 8 >= D) h[i] = 0;
    } else {
      const float2 v = unpack2(h[i]);
      const int c = col_of<false>(base, lane, tpr, 2 * i);
      h[i] = pack2(c < D ? v.x : 0.f, c + tpr < D ? v.y : 0.f);
    }
  }
}
// Sums of M values over the TPR threads of a row.  One barrier: whoever calls it alternates between two places in shared memory, so
// that the barrier of one sum stands between the reads of the last and the writes of the next.
template <int TPR, int M>
__device__ __forceinline__ void row_total(float (&v)[M], float* red) {
  static_assert(M == 1 || M == 3, "");
  if constexpr (TPR <= 32) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1)
#pragma unroll
      for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  } else {
    constexpr int W = TPR / 32, N = W * M;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if constexpr (M == 1) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      if (lane == 0) red[warp] = v[0];
    } else {  // three sums in six exchanges instead of fifteen: two of them to each half of the warp, one to each quarter
      const bool up = lane & 16, odd = lane & 8;
      const float a = (up ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16);
      const float b = (up ? 0.f : v[1]) + __shfl_xor_sync(0xffffffffu, up ? v[1] : 0.f, 16);
      float s = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if ((lane & 7) == 0 && lane < 24) red[warp * 3 + (lane >> 3)] = s;
    }
    __syncthreads();
    const float* from = red + warp / W * N;
    float all[N];
    if constexpr (N % 4 == 0) {  // (a warp of the row after the other, but read in whole pieces)
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(all + i) = *reinterpret_cast<const float4*>(from + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) all[i] = from[i];
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += all[w * M + m];
      v[m] = s;
    }
  }
}

// IO: type of n and, with a stream, of x; RES: the stream's.
template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>) lnorm_fwd_kernel(NormP p) {
  begin_dependent();
  __shared__ __align__(16) float red[2][kThreads<TPR> / 32 < 4 ? 4 : kThreads<TPR> / 32];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  const RES* stream = static_cast<const RES*>(p.resid ? p.resid : p.x);
  Cols<RES, V> a_h[E];
  Cols<IO, V> a_x[E];
  auto offset = [&](size_t r0) { return (r0 + group < p.rows ? r0 + group : r0) * p.D; };
  auto request = [&](size_t r0) {
    const size_t off = offset(r0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      a_h[e].load(stream + off, c, lane, TPR, p.D);
      if (p.resid) a_x[e].load(static_cast<const IO*>(p.x) + off, c, lane, TPR, p.D);
    }
  };
  request((size_t)blockIdx.x * GROUPS);
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = offset(r0);
    f2 h[E][4], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      a_h[e].get(h[e]);
      if (p.resid) {
        f2 x[4];
        a_x[e].get(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[e][i] = add2(h[e][i], x[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = add2(sum, h[e][i]);
    }
    if (r0 + (size_t)gridDim.x * GROUPS < p.rows) request(r0 + (size_t)gridDim.x * GROUPS);
    float s[1] = {sum2(sum)};
    row_total<TPR>(s, red[0]);
    const f2 minus_m = dup2(-s[0] * inv);
    sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      if (p.resid && live) store_cols<RES, V>(static_cast<RES*>(p.stream) + off, c, lane, TPR, p.D, h[e]);
      centre<V>(h[e], c, lane, TPR, p.D, minus_m);
#pragma unroll
      for (int i = 0; i < 4; ++i) fma2(sum, h[e][i], h[e][i]);
    }
    s[0] = sum2(sum);
    row_total<TPR>(s, red[1]);
    const f2 k = dup2(rsqrtf(s[0] * inv + p.eps));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      f2 w[4], b[4] = {0, 0, 0, 0};
      load_cols<float, V>(p.weight, c, lane, TPR, p.D, w);
      if (p.bias) load_cols<float, V>(p.bias, c, lane, TPR, p.D, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = mad2(mul2(h[e][i], k), w[i], b[i]);
      if (live) store_cols<IO, V>(static_cast<IO*>(p.n) + off, c, lane, TPR, p.D, w);
    }
  }
}

template <typename IO, typename RES, int TPR, int E, bool V>
__global__ void __launch_bounds__(kThreads<TPR>, TPR > 256 || E > 1 ? 1 : V && sizeof(RES) == 2 ? 3 : 2) lnorm_bwd_kernel(NormP p) {
  begin_dependent();
  __shared__ __align__(16) float red[kThreads<TPR> / 32], red3[kThreads<TPR> / 32 * 3];
  constexpr int GROUPS = kThreads<TPR> / TPR;
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.D;
  f2 dw[E][4], db[E][4];
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[e][i] = db[e][i] = 0;
  f2 weight[4];  // (one piece of it stays in registers: read twice a row it is half of what the L1 cache delivers)
  if (E == 1) load_cols<float, V>(p.weight, 0, lane, TPR, p.D, weight);
  Cols<RES, V> a_h[E], a_d[E];
  Cols<IO, V> a_g[E];
  auto offset = [&](size_t r0) { return (r0 + group < p.rows ? r0 + group : r0) * p.D; };
  auto request = [&](size_t r0) {
    const size_t off = offset(r0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      a_h[e].load(static_cast<const RES*>(p.x) + off, c, lane, TPR, p.D);
      a_g[e].load(static_cast<const IO*>(p.dn) + off, c, lane, TPR, p.D);
      if (p.d_resid) a_d[e].load(static_cast<const RES*>(p.d_resid) + off, c, lane, TPR, p.D);
    }
  };
  request((size_t)blockIdx.x * GROUPS);
  for (size_t r0 = (size_t)blockIdx.x * GROUPS; r0 < p.rows; r0 += (size_t)gridDim.x * GROUPS) {
    const bool live = r0 + group < p.rows;
    const size_t off = offset(r0);
    f2 h[E][4], g[E][4], d[E][4], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      a_h[e].get(h[e]);
      a_g[e].get(g[e]);
      if (p.d_resid) {
        a_d[e].get(d[e]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[e][i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = add2(sum, h[e][i]);
    }
    if (r0 + (size_t)gridDim.x * GROUPS < p.rows) request(r0 + (size_t)gridDim.x * GROUPS);
    float m[1] = {sum2(sum)};
    row_total<TPR>(m, red);
    const f2 minus_m = dup2(-m[0] * inv);
    f2 s0 = 0, s1 = 0, s2 = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      centre<V>(h[e], c, lane, TPR, p.D, minus_m);
      f2 w[4];
      if constexpr (E == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = weight[i];
      } else {
        load_cols<float, V>(p.weight, c, lane, TPR, p.D, w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f2 t = mul2(g[e][i], w[i]);
        fma2(s0, h[e][i], h[e][i]);
        s1 = add2(s1, t);
        fma2(s2, t, h[e][i]);
      }
    }
    float s[3] = {sum2(s0), sum2(s1), sum2(s2)};
    row_total<TPR>(s, red3);
    const float k = rsqrtf(s[0] * inv + p.eps);
    const f2 kk = dup2(k), mt = dup2(-s[1] * inv), mtu = dup2(-k * k * s[2] * inv);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * TPR * 8;
      f2 w[4];
      if constexpr (E == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = weight[i];
      } else {
        load_cols<float, V>(p.weight, c, lane, TPR, p.D, w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (live) {
          fma2(dw[e][i], g[e][i], mul2(h[e][i], kk));
          db[e][i] = add2(db[e][i], g[e][i]);
        }
        d[e][i] = mad2(kk, mad2(h[e][i], mtu, mad2(g[e][i], w[i], mt)), d[e][i]);
      }
      if (live) store_cols<RES, V>(static_cast<RES*>(p.dx) + off, c, lane, TPR, p.D, d[e]);
    }
  }
  float* part = p.part + ((size_t)blockIdx.x * GROUPS + group) * 2 * p.D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = e * TPR * 8;
    store_cols<float, V>(part, c, lane, TPR, p.D, dw[e]);
    store_cols<float, V>(part + p.D, c, lane, TPR, p.D, db[e]);
  }
}
// Sums of the partial rows.  grid (column blocks, 2): dw, db.
template <bool TALL>
__global__ void __launch_bounds__(kSumThreads<TALL>) lnorm_sum_kernel(const float* part, int rows, int D, float* dweight, float* dbias) {
  begin_dependent();
  const int c0 = blockIdx.x * kSumCols<TALL>, mine = c0 + threadIdx.x % kSumCols<TALL>;
  col_sum<TALL>(part + blockIdx.y * (size_t)D + mine, rows, 2 * (size_t)D, mine < D, [&](int c, float t) {
    if (c0 + c < D) (blockIdx.y ? dbias : dweight)[c0 + c] = t;
  });
}

// ------------------------------------------------------------------ host
struct RowShape { int tpr, e; };
// Threads of a row, pieces of 8 columns a thread.
static RowShape row_shape(int D, bool bwd) {
  int t = 4;
  while (8 * t < D && t < 1024) t *= 2;
  if (!bwd) return {t, D > 8192 ? 2 : 1};
  if (D <= 2048) return {t, 1};
  if (D <= 4096) return {t / 2, 2};
  return {512, D > 8192 ? 4 : 2};
}
static int groups_of(int tpr) { return tpr > 256 ? 1 : 256 / tpr; }
// CTAs: what the GPU holds at once, by registers.  Forwards 4 an SM; backwards 2, or 3 where a bf16 stream comes in whole pieces (32768
// rows of 2048 columns 105 us, with two 113), or one with two pieces a thread.
static int ctas(size_t rows, int D, bool bwd, bool narrow) {
  const RowShape s = row_shape(D, bwd);
  const int g = groups_of(s.tpr), each = !bwd ? 4 : s.e > 1 ? 1 : narrow && D % 8 == 0 ? 3 : 2;
  const size_t want = (rows + g - 1) / g, most = std::max(148, 148 * each * 256 / std::max(s.tpr, 256));
  return (int)std::min(want, most);
}
template <typename F>
static void by_shape(int D, bool bwd, F&& f) {
  const RowShape s = row_shape(D, bwd);
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 2> two;
  if (bwd && s.e > 1) {
    if (s.tpr == 256) f(std::integral_constant<int, 256>{}, two);
    else if (s.e == 2) f(std::integral_constant<int, 512>{}, two);
    else f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
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
static mxb_status run(const NormP& p, float* dweight, float* dbias, cudaStream_t st) {
  const bool bwd = p.dn != nullptr;
  const int n = ctas(p.rows, p.D, bwd, sizeof(RES) == 2);
  int parts = 0;
  by_shape(p.D, bwd, [&](auto tpr, auto e) {
    constexpr int TPR = decltype(tpr)::value, E = decltype(e)::value;
    // (row_shape(): which there are)
    if constexpr (E == 1 ? TPR <= 256 : TPR <= 512)
      if (bwd) {
        parts = n * (kThreads<TPR> / TPR);
        MXB_LAUNCH("lnorm_bwd_kernel", st, (launch_kernel(lnorm_bwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
      }
    if constexpr (E == 1 || TPR > 512)
      if (!bwd) MXB_LAUNCH("lnorm_fwd_kernel", st, (launch_kernel(lnorm_fwd_kernel<IO, RES, TPR, E, V>, n, kThreads<TPR>, 0, st, p)));
  });
  if (bwd) {
    auto launch = [&](auto tall) {
      constexpr bool T = decltype(tall)::value;
      MXB_LAUNCH("lnorm_sum_kernel", st, (launch_kernel(lnorm_sum_kernel<T>, dim3((p.D + kSumCols<T> - 1) / kSumCols<T>, 2), kSumThreads<T>, 0, st,
                                                        p.part, parts, p.D, dweight, dbias)));
    };
    if (col_sum_tall(2 * (size_t)p.D)) launch(std::true_type{});
    else launch(std::false_type{});
  }
  return check_launch(bwd ? "lnorm_bwd" : "lnorm_fwd");
}
template <typename IO, typename RES>
static mxb_status by_alignment(const NormP& p, float* dweight, float* dbias, cudaStream_t st) {
  constexpr int32_t io = sizeof(IO) == 4 ? MXB_F32 : MXB_BF16, res = sizeof(RES) == 4 ? MXB_F32 : MXB_BF16;
  bool whole = whole_pieces(p.x, p.resid ? io : res, p.D) && whole_pieces(p.n, io, p.D) && whole_pieces(p.dn, io, p.D);
  for (const void* q : {p.resid, (const void*)p.stream, p.d_resid, (const void*)p.dx}) whole = whole && whole_pieces(q, res, p.D);
  for (const float* q : {p.weight, p.bias}) whole = whole && whole_pieces(q, MXB_F32, p.D);
  return whole ? run<IO, RES, true>(p, dweight, dbias, st) : run<IO, RES, false>(p, dweight, dbias, st);
}
static mxb_status by_type(const mxb_layer_norm_desc* d, const NormP& p, float* dweight, float* dbias, cudaStream_t st) {
  if (d->io_dtype == MXB_F32) return by_alignment<float, float>(p, dweight, dbias, st);
  if (d->resid_dtype == MXB_F32) return by_alignment<bf16, float>(p, dweight, dbias, st);
  return by_alignment<bf16, bf16>(p, dweight, dbias, st);
}

}  // namespace lnorm

size_t layer_norm_scratch(const mxb_layer_norm_desc* d) {
  const int tpr = lnorm::row_shape(d->D, true).tpr;
  return (size_t)lnorm::ctas(d->rows, d->D, true, d->resid_dtype == MXB_BF16) * lnorm::groups_of(tpr) * 2 * d->D * sizeof(float) + kBaseRoom;
}
mxb_status layer_norm_fwd(const mxb_layer_norm_desc* d, const void* resid, const void* x, const float* weight, const float* bias, void* stream,
                          void* n, cudaStream_t st) {
  const lnorm::NormP p{(size_t)d->rows, d->D, d->eps, resid, x, weight, bias, resid ? stream : nullptr, n};
  return lnorm::by_type(d, p, nullptr, nullptr, st);
}
mxb_status layer_norm_bwd(const mxb_layer_norm_desc* d, const void* x, const float* weight, const void* d_resid, const void* dn, void* dx,
                          float* dweight, float* dbias, void* workspace, cudaStream_t st) {
  float* part = static_cast<float*>(round_base_up(workspace));  // (written in pieces of 32 bytes)
  const lnorm::NormP p{(size_t)d->rows, d->D, d->eps, nullptr, x, weight, nullptr, nullptr, nullptr, d_resid, dn, dx, part};
  return lnorm::by_type(d, p, dweight, dbias, st);
}

}  // namespace mxb
