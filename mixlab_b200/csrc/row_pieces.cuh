// Rows of a matrix in pieces of eight columns a thread: loads, requests ahead, stores, and sums over the threads of a row.
#pragma once

#include "common.cuh"
#include "packed.cuh"

namespace mxb {

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
// Eight floats in one access (32 bytes, on 32 bytes): two of 16 would write each sector of 32 bytes in halves.
__device__ __forceinline__ void load_floats(const float* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store_floats(float* p, const f2 (&e)[4]) {
  asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(e[0]), "l"(e[1]), "l"(e[2]), "l"(e[3]) : "memory");
}
// Whether a tensor of D columns may be read and written in whole pieces: of eight floats on 32 bytes, of eight bf16 on 16.  (No tensor:
// nothing in the way.)
inline bool whole_pieces(const void* p, int32_t type, int D) { return D % 8 == 0 && reinterpret_cast<uintptr_t>(p) % (type == MXB_F32 ? 32 : 16) == 0; }

// Eight columns of a row by each of its `tpr` threads, from column `base` on.  Whole pieces (V): eight neighbours a thread.  Else
// thread `lane` takes base + lane + j tpr, so that a warp's accesses lie side by side (eight neighbours a thread in single
// elements: gradients of a layer norm of 4001 x 449 in float32 23 us).
template <bool V>
__device__ __forceinline__ int col_of(int base, int lane, int tpr, int j) { return V ? base + lane * 8 + j : base + lane + j * tpr; }
template <typename T, bool V>
__device__ __forceinline__ void load_cols(const T* row, int base, int lane, int tpr, int D, f2 (&e)[4]) {
  if constexpr (V && sizeof(T) == 4) {
    uint32_t r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (base + lane * 8 < D) load_floats(row + base + lane * 8, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
  } else if constexpr (V) {
    load8<T, true>(row, base + lane * 8, D, e);
  } else {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false>(base, lane, tpr, j);
      v[j] = c < D ? to_f32(row[c]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = pack2(v[2 * i], v[2 * i + 1]);
  }
}
template <typename T, bool V>
__device__ __forceinline__ void store_cols(T* row, int base, int lane, int tpr, int D, const f2 (&e)[4]) {
  if constexpr (V && sizeof(T) == 4) {
    if (base + lane * 8 < D) store_floats(row + base + lane * 8, e);
  } else if constexpr (V) {
    store8<T, true>(row, base + lane * 8, D, e);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(e[i]);
      const int c = col_of<false>(base, lane, tpr, 2 * i);
      if (c < D) row[c] = from_f32<T>(a.x);
      if (c + tpr < D) row[c + tpr] = from_f32<T>(a.y);
    }
  }
}
// ... as they are in memory, requested ahead of their use.
template <typename T, bool V>
struct Cols {
  static constexpr int W = V ? 2 * sizeof(T) : 1;  // words
  uint32_t raw[W];
  T one[V ? 1 : 8];
  __device__ __forceinline__ void load(const T* row, int base, int lane, int tpr, int D) {
    if constexpr (V) {
      const int c = base + lane * 8;
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = 0;
      if (c >= D) return;
      if constexpr (sizeof(T) == 4) {
        load_floats(row + c, raw);
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(row + c);
        raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = col_of<false>(base, lane, tpr, j);
        one[j] = c < D ? row[c] : from_f32<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void get(f2 (&e)[4]) const {
    if constexpr (!V) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = pack2(to_f32(one[2 * i]), to_f32(one[2 * i + 1]));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = pack2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
    } else {
      unpack8(make_uint4(raw[0], raw[1], raw[2], raw[3]), e);
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

}  // namespace mxb
