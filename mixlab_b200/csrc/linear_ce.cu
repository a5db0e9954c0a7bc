// The output head and its loss, without the logits in memory:
//     z_tv = x_t . W_v,   lse_t = log sum_v exp z_tv,   loss_t = lse_t - z_t,i_t
// and its gradients: with a_t, c_t the gradients of loss_t and lse_t,
//     g_tv = (a_t + c_t) exp(z_tv - lse_t) - a_t [v = i_t],   dx = g W,   dW = g^T x
// Tokens whose target is outside 0 .. V-1 (in the backward pass also those whose a and c are zero) have no part: a first launch
// moves the rows of the others together, so that they are neither computed nor read (they may hold anything).
//
// Products on the tensor cores, 256 x 256 a pair of CTAs, fed by TMA through a ring of shared-memory stages; accumulators in TMEM by
// turns, so that one is read while another is filled.  Forward: the accumulator is reduced to the maximum and the sum of
// exponentials of each row over the tile's columns, 8 bytes a row and tile.  Backward, in pieces of the vocabulary: z again, g in
// bf16 to a workspace of bounded size, then dx += g W and dW = g^T x from it (a second part of g, which would leave the results' own
// rounding alone, would be two products more beside three).
//
// What bounds it is the tensor pipe at the clock that the power limit leaves: 28672 tokens, 65536 words of 1024 columns 2.70 ms
// (1425 TFLOP/s; cuBLAS's product alone runs at 1402 for seconds on end); the gradients for 50001 words 7.1 to 7.4 ms (1240 to 1190),
// where g goes through HBM three times.  512 tokens, 32768 words: 36 us; by the counters, which time each launch alone and cold, the products
// take 32 - four rounds of tiles 18 of them, the first copies and the last tile's exponentials 5, 9 not taken apart - and the join 7.
// 2048 tokens, 5003 words of 448 columns in float32: 173 us for 96 of products; each of the three products waits 4 us for its first stage
// and ends with an epilogue of 3; packing is 13 of it, the shares 10 (counters).  The loss of these 56 us for 33.
// float32 tensors: every operand is split into three bf16 parts (24 bits and more), and six products of parts, those above
// 2^-24, are added up.  An accumulator in TMEM is cut, not rounded, with every product added to it, so it takes the products
// of 128 terms, small ones first, and is handed over: the sums of those are float32 in registers (2048 tokens, 5003 words of 448: gradients
// off by 7e-7, with accumulators of 2048 terms by 3.6e-6).
#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"
#include "umma_tiles.cuh"

namespace mxb {
namespace lce {

using bf16 = __nv_bfloat16;
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ tokens that count
constexpr int kCountRows = 1024;  // rows whose tokens one block counts
struct PackP {
  const void* targets;
  const void* x;
  const float *lse, *d_loss, *d_lse;  // backward; d_lse may be null
  const int32_t* counts;              // of every kCountRows rows (where there are as many)
  int32_t *live, *idx, *tgt;          // how many; their rows; their targets
  float *a, *both, *lse2;             // their gradients of loss and of both, lse (bf16: in powers of two)
  bf16* xc;                           // [parts][pad][Dp]
  void* dx;                           // backward: rows of the other tokens become zero
  float *loss, *lse_out;              // forward: likewise
  int32_t* status;
  size_t N, pad;
  int V, D, Dp, wide;                 // wide: targets of 64 bits
  int each;                           // rows of a warp of the pack kernel
  const void* w;                      // first rows of W to pack in the same launch (w_rows; 0: none)
  bf16* wc;
  size_t w_pad;
  int w_rows;
};
__device__ __forceinline__ int target_at(const void* targets, int wide, int V, size_t t) {  // -1: none
  const int64_t v = wide ? static_cast<const int64_t*>(targets)[t] : static_cast<const int32_t*>(targets)[t];
  return v >= 0 && v < V ? (int)v : -1;
}
__device__ __forceinline__ int target_of(const PackP& p, size_t t) {  // -1: none
  return target_at(p.targets, p.wide, p.V, t);
}
__device__ __forceinline__ bool counts(const PackP& p, size_t t) {
  if (target_of(p, t) < 0) return false;
  if (!p.d_loss) return true;
  return !(p.d_loss[t] == 0.f) || (p.d_lse && !(p.d_lse[t] == 0.f));
}
__device__ __forceinline__ int block_sum(int v, int32_t* red) {  // 256 threads
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += red[w];
  return s;
}
// How many of the tokens in front of t count.
__device__ __forceinline__ int counted_before(const PackP& p, size_t t, int32_t* red) {
  const size_t blocks = p.counts ? t / kCountRows : 0;
  int n = 0;
  for (size_t b = threadIdx.x; b < blocks; b += 256) n += p.counts[b];
  for (size_t i = blocks * kCountRows + threadIdx.x; i < t; i += 256) n += counts(p, i);
  return block_sum(n, red);
}
__global__ void __launch_bounds__(256) lce_count_kernel(PackP p, int32_t* out) {
  begin_dependent();
  __shared__ int32_t red[8];
  int n = 0;
  for (int k = 0; k < kCountRows / 256; ++k) {
    const size_t t = (size_t)blockIdx.x * kCountRows + k * 256 + threadIdx.x;
    n += t < p.N && counts(p, t);
  }
  n = block_sum(n, red);
  if (threadIdx.x == 0) out[blockIdx.x] = n;
}
// A value in bf16 parts, the first the nearest to it, each other the nearest to what is left.
template <int PARTS>
__device__ __forceinline__ void split(float v, bf16 (&part)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    part[k] = __float2bfloat16_rn(v);
    // (what is left of an infinity or a NaN would be a NaN)
    v = k + 1 < PARTS ? (isfinite(v) ? v - __bfloat162float(part[k]) : 0.f) : 0.f;
  }
}
// Row `from` of a matrix with D columns (null: zeros) to row `to` of its packed form, by one warp.
template <typename T>
__device__ __forceinline__ void pack_row(const T* from, bf16* to, size_t part_stride, int D, int Dp, int lane) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  const bool whole = D % 8 == 0 && (reinterpret_cast<uintptr_t>(from) & 15) == 0;  // (Dp is a multiple of 8)
  for (int c = lane * 8; c < Dp; c += 256) {
    if (PARTS == 1 && whole) {
      *reinterpret_cast<uint4*>(to + c) = from ? *reinterpret_cast<const uint4*>(from + c) : make_uint4(0, 0, 0, 0);
      continue;
    }
    float v[8];
    if (whole && from && sizeof(T) == 4) {
      const float4 lo = *reinterpret_cast<const float4*>(from + c), hi = *reinterpret_cast<const float4*>(from + c + 4);
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from && c + i < D ? to_f32(from[c + i]) : 0.f;
    }
    bf16 e[PARTS][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16 part[PARTS];
      split<PARTS>(v[i], part);
#pragma unroll
      for (int k = 0; k < PARTS; ++k) e[k][i] = part[k];
    }
#pragma unroll
    for (int k = 0; k < PARTS; ++k) *reinterpret_cast<uint4*>(to + k * part_stride + c) = *reinterpret_cast<uint4*>(e[k]);
  }
}
// Blocks of eight warps with p.each rows each; 32 blocks behind them fill up the last tile of 256 rows with zeros, those behind them
// pack rows of W.
template <typename T>
__global__ void __launch_bounds__(256) lce_pack_kernel(PackP p, int row_blocks) {
  begin_dependent();
  __shared__ int32_t red[8];
  __shared__ uint32_t counted;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x >= row_blocks) {
    if ((int)blockIdx.x >= row_blocks + 32) {
      const int r = ((int)blockIdx.x - row_blocks - 32) * 8 + warp;
      if (r < p.w_rows) pack_row<T>(static_cast<const T*>(p.w) + (size_t)r * p.D, p.wc + (size_t)r * p.Dp, p.w_pad * p.Dp, p.D, p.Dp, lane);
      return;
    }
    const int live = counted_before(p, p.N, red), k = ((int)blockIdx.x - row_blocks) * 8 + warp;
    const size_t j = (size_t)live + k;
    if (blockIdx.x == row_blocks && threadIdx.x == 0) {
      *p.live = live;
      *p.status = 0;
    }
    if (j >= ((size_t)live + 255) / 256 * 256) return;
    pack_row<T>(nullptr, p.xc + j * p.Dp, p.pad * p.Dp, p.D, p.Dp, lane);
    if (lane == 0) {
      p.tgt[j] = -1;
      if (p.d_loss) p.a[j] = p.both[j] = p.lse2[j] = 0.f;
    }
    return;
  }
  const size_t r0 = (size_t)blockIdx.x * 8 * p.each;
  if (warp == 0) {
    const uint32_t b = __ballot_sync(0xffffffffu, lane < 8 * p.each && r0 + lane < p.N && counts(p, r0 + lane));
    if (lane == 0) counted = b;
  }
  const int before = counted_before(p, r0, red);
  const uint32_t mask = counted;
  for (int k = 0; k < p.each; ++k) {
    const int i = warp * p.each + k;
    const size_t r = r0 + i;
    if (r >= p.N) return;
    if (!(mask >> i & 1u)) {
      if (p.d_loss) {
        T* to = static_cast<T*>(p.dx) + r * p.D;
        for (int c = lane; c < p.D; c += 32) to[c] = from_f32<T>(0.f);
      } else if (lane == 0) {
        p.loss[r] = p.lse_out[r] = 0.f;
      }
      continue;
    }
    const size_t j = (size_t)before + __popc(mask & ((1u << i) - 1u));
    if (lane == 0) {
      p.idx[j] = (int32_t)r;
      p.tgt[j] = target_of(p, r);
      if (p.d_loss) {
        const float a = p.d_loss[r];
        p.a[j] = a;
        p.both[j] = p.d_lse ? a + p.d_lse[r] : a;
        p.lse2[j] = sizeof(T) == 4 ? p.lse[r] : p.lse[r] * kLog2e;
      }
    }
    pack_row<T>(static_cast<const T*>(p.x) + r * p.D, p.xc + j * p.Dp, p.pad * p.Dp, p.D, p.Dp, lane);
  }
}
// Rows of a piece of W.
template <typename T>
__global__ void __launch_bounds__(256) lce_pack_weight_kernel(const T* w, bf16* to, int rows, size_t pad, int D, int Dp) {
  begin_dependent();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r < rows) pack_row<T>(w + (size_t)r * D, to + (size_t)r * Dp, pad * Dp, D, Dp, threadIdx.x & 31);
}

// ------------------------------------------------------------------ the products
enum Mode { kStats, kGrad, kDx, kDw };
// A stage of the ring: PARTS tiles of A, 128 rows a CTA, and of B, BN / 2 rows a CTA, 64 deep.  BN: columns of a tile.
template <int MODE, bool F32, int BN_>
struct Cfg {
  static constexpr int BN = BN_, PARTS = F32 ? 3 : 1, COLS = BN / 2;  // COLS: of a thread of the epilogue
  static constexpr int A = 128 * 128, B = BN / 2 * 128, STAGE = PARTS * (A + B);
  static constexpr int STAGES = !F32 ? 6 : BN == 128 ? 3 : 2;
  static constexpr bool BOXES = MODE == kDw && !F32;  // results leave in boxes of 32 rows x 64 columns a warp
  static constexpr int STAGING = BOXES ? 8 * 4096 : 0;
  static constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDx || MODE == kDw;
  static constexpr int ACCS = 512 / BN, RING = 2 * ACCS;  // accumulators in TMEM; kStats: slots for what halves of a tile exchange
  static constexpr int SMEM = 1024 + STAGES * STAGE + STAGING + 256 + (MODE == kStats ? RING * (4 * 8 + 128 * 8) : 0);
};
constexpr int kThreads = 384;  // eight warps of the epilogue, one for copies, one for products, two that fill up their warpgroup
struct GemmP {
  const int32_t* live;    // null: rows tokens, none left out
  const void* targets;    //   their targets (wide: of 64 bits)
  int32_t* flags;         //   what *status gets, by blocks
  int rows, wide;
  int32_t* status;
  int M, N, K;            // the extent that counts tokens is *live
  int b_row0;             // first row of B in its map (the vocabulary's piece)
  int group;              // tiles of M that are walked through together
  int v0, V;              // first row of the vocabulary's piece, rows in all
  bf16* g;
  size_t pad;             // rows of what is indexed by token
  int piece, blocks;      // columns of g, blocks of 128 rows of one of its parts
  float2* part;           // kStats: [tiles of the vocabulary][pad] maximum and sum
  float* hit;             //   logit of the target
  const int32_t *tgt, *idx;
  const float *a, *both, *lse2;
  float* sums;            // kDx: float32 sums of all pieces, by tiles (tile_at()), null: straight to out
  int adds;               //   to what is there
  float* shares;          // kDx, kDw: tiles of which a pair has a share of K, two a pair
  void* out;              // rows by idx (kDx) or from v0 (kDw)
  int D, whole;           // whole: out's rows may be written in pieces of 16 bytes
};
struct Maps { CUtensorMap a, b, g; };
__device__ __forceinline__ int live_of(const GemmP& p) { return p.live ? *p.live : p.rows; }
// bf16: g is kept as a multiple of the first token's gradient's mantissa (1 .. 2; 1 of a zero, an infinity or a NaN), by which dx and dW are
// multiplied before they are rounded.  Where all tokens weigh the same - a mean, a sum over some of them - what g is rounded from
// is then 2^k (p - [v = i]).  Without it the rounding of the weight itself is in every token's largest element alike: 28672 tokens that
// weigh 1 / 28672, off by 2e-3 as bf16, had gradients off by 2.3e-3, with it by 1.9e-3, of which their own rounding is 1.7e-3.
__device__ __forceinline__ float unit_of(const GemmP& p) {
  const uint32_t a = __float_as_uint(p.a[0]), v = a & 0x7fffffffu ? a : __float_as_uint(p.both[0]), e = v >> 23 & 255u;
  return e == 0u || e == 255u ? 1.f : __uint_as_float((v & 0x7fffffu) | 0x3f800000u);
}

// A wait that gives up: on its own limit, or when another role of the CTA has.
struct Wait {
  volatile int32_t* bad;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
    for (uint32_t i = 0; i < 4000000u; ++i) {
      if (tc::mbar_try_wait(bar, parity)) return true;
      if ((i & 63u) == 63u && *bad) return false;
    }
    *bad = 1;
    return false;
  }
};
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A maximum (-infinity, 0: nothing yet; +infinity, +infinity: an infinite logit) and the sum of exponentials from it, and another such
// pair.  The larger maximum's sum is not scaled, so that no infinity meets a difference of infinities or a zero.
__device__ __forceinline__ void add_sum(float2& a, float2 b) {
  const float t = fmaxf(a.x, b.x);
  a.y = a.y * (a.x == t ? 1.f : ex2((a.x - t) * kLog2e)) + b.y * (b.x == t ? 1.f : ex2((b.x - t) * kLog2e));
  a.x = t;
}

// What all roles walk through: tiles of 256 x BN, group tiles of M at a time so that both operands' tiles stay in L2.  A pair takes
// every pairs-th tile.  Where tiles stand for long sums (kDx, kDw) and the last round has fewer tiles than pairs, those are cut along K
// into equal shares for all pairs, of one or two tiles each, and left as float32 shares that lce_shares_kernel adds up in order.
// (Gradients of 28672 tokens, pieces of 8192 words: 448 and 128 tiles for 74 pairs; without the cut the last round of seven, or of
// two, runs on a few of them.)
struct Item {
  int m, n, k0, k1;
  int share;  // -1: the whole tile
};
struct Walk {
  int m_tiles, n_tiles, kblocks, tiles, whole, rest, pairs, group;
  int units, share;  // blocks of K of all tiles that are cut; a pair's
  __device__ __forceinline__ Walk(const GemmP& p, int mode, int BN, int pairs_) {
    const int live = live_of(p);
    const int M = mode == kDw ? p.M : live, K = mode == kDw ? live : p.K;
    pairs = pairs_;
    group = p.group;
    m_tiles = (M + 255) / 256;
    n_tiles = (p.N + BN - 1) / BN;
    kblocks = (K + 63) / 64;
    tiles = m_tiles * n_tiles;
    rest = mode == kStats || mode == kGrad || kblocks < 16 ? 0 : tiles % pairs;
    whole = tiles - rest;
    units = rest * kblocks;  // (2^31 at most: check_linear_ce_desc())
    const int sharers = min(pairs, units / 8);  // more than there are tiles: a share is a tile's sum at most
    share = sharers ? (units + sharers - 1) / sharers : 0;
  }
  __device__ __forceinline__ void place(int i, Item& t) const {
    const int g = i / (group * n_tiles), in = i - g * group * n_tiles, gm = min(group, m_tiles - g * group);
    t.m = g * group + in % gm;
    t.n = in / gm;
  }
  // The pair's j-th item; false: there is none.
  __device__ __forceinline__ bool item(int pair, int j, Item& t) const {
    const int64_t i = (int64_t)j * pairs + pair;
    if (i < whole) {
      place((int)i, t);
      t.k0 = 0;
      t.k1 = kblocks;
      t.share = -1;
      return true;
    }
    const int64_t from = (int64_t)pair * share, to = min(from + share, (int64_t)units);
    if (from >= units) return false;
    const int tile = (int)from / kblocks, second = j - (whole + pairs - 1 - pair) / pairs;
    const int64_t cut = (int64_t)(tile + 1) * kblocks;
    if (second > 1 || (second == 1 && to <= cut)) return false;
    place(whole + tile + second, t);
    t.k0 = second ? 0 : (int)(from - (int64_t)tile * kblocks);
    t.k1 = (int)((second ? to : min(to, cut)) - (int64_t)(tile + second) * kblocks);
    t.share = pair * 2 + second;
    return true;
  }
};
// g lies in blocks of 128 rows, in those by eight columns, 16 bytes a row: a warp of the epilogue writes whole lines straight from its
// registers, and a copy of such blocks is an operand of the products without a swizzle, with the contraction along columns (dx) or
// rows (dW).  (float32, 2048 tokens, 5003 words of 448: 52 us; rows of the matrix, 16 bytes a lane, 70.)
__device__ __forceinline__ size_t g_at(const GemmP& p, int block, int col) { return ((size_t)block * (p.piece / 8) + col / 8) * 1024; }
// Float32 tiles as the epilogue has them: element (row, c .. c + 3) of a CTA's 128 rows, 16 bytes of 32 rows side by side.
template <int BN>
__device__ __forceinline__ size_t tile_at(size_t tile, int rank, int row, int c) {
  return ((tile * 2 + rank) * (BN / 4) + c / 4) * 512 + row * 4;
}

template <typename T>
__device__ __forceinline__ void store_row(T* to, int c, int D, bool whole, const float* v) {  // 8 columns from c
  if (whole) {
    if (c >= D) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(to + c) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(to + c) = tc::pack8(v);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < D) to[c + i] = from_f32<T>(v[i]);
}

// A warp's 32 rows x COLS columns to a bf16 tensor in boxes of 64 columns, by its part of shared memory (128-byte swizzle).
template <int COLS>
__device__ __forceinline__ void leave_in_boxes(const void* map, uint8_t* box, const float (&v)[COLS], int c0, int r0, int lane) {
#pragma unroll
  for (int x = 0; x < COLS / 64; ++x) {
    if (lane == 0) tc::bulk_wait_read<0>();
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(box + lane * 128 + ((u ^ (lane & 7)) << 4)) = tc::pack8(v + x * 64 + u * 8);
    tc::fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      tc::tma_store_3d(map, tc::smem_u32(box), c0 + x * 64, r0, 0);
      tc::bulk_commit();
    }
  }
}

template <int MODE, bool F32, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) lce_gemm_kernel(const GemmP p, const __grid_constant__ Maps maps) {
  using C = Cfg<MODE, F32, BN>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (tc::smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* sm = raw + (base - tc::smem_u32(raw));
  uint8_t* staging = sm + C::STAGES * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);
  uint64_t *empty = full + C::STAGES, *acc_full = empty + C::STAGES, *acc_empty = acc_full + C::ACCS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + C::ACCS);
  volatile int32_t* bad = reinterpret_cast<volatile int32_t*>(tmem_slot + 1);
  // kStats: what the warps of a tile's second half found, for those of the first: a ring of slots by tiles, a barrier a slot and warp.
  // (When a warp writes for tile t + 2 ACCS, that tile's accumulator has been filled, so tile t + ACCS's has been read by all warps,
  // which are done with the tiles in front of it.)
  uint64_t* halves_full = reinterpret_cast<uint64_t*>(staging + C::STAGING + 256);  // [RING][4]
  float2* halves = reinterpret_cast<float2*>(halves_full + C::RING * 4);            // [RING][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(full + s, 1);
      tc::mbar_init(empty + s, 1);
    }
    for (int s = 0; s < C::ACCS; ++s) {
      tc::mbar_init(acc_full + s, 1);
      tc::mbar_init(acc_empty + s, 16);
    }
    if (MODE == kStats)
      for (int s = 0; s < C::RING * 4; ++s) tc::mbar_init(halves_full + s, 1);
    *bad = 0;
    tc::mbar_fence_init();
  }
  if (threadIdx.x == 32) {
    tc::tma_prefetch_map(&maps.a);
    tc::tma_prefetch_map(&maps.b);
  }
  if (warp == 9) {
    tc::tmem_alloc_pair(tmem_slot, 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  begin_dependent();  // (nothing but this CTA's own memory is touched before)
  const uint32_t tmem = *tmem_slot;
  const Walk walk(p, MODE, C::BN, pairs);
  Item t;
  const Wait wait{bad};
  // Blocks of K behind which an accumulator is handed over.  bf16: a cut accumulator loses up to 2^-23 of itself with every 16 terms,
  // 2^-17 over the 1024 of a loss's logits (32768 tokens, 65536 words: 2.84 ms; with 512, which halves the error, 2.91), 2^-16 over 2048
  // of a gradient's, 2^-11 over the 65536 of its sums, which a rounding to bf16 (2^-9) follows.
  constexpr int SEG = F32 ? 2 : MODE == kStats ? 16 : MODE == kGrad ? 32 : 1024;
  // Registers: the epilogue holds a row's 128 columns beside what it does with them; 256 x 232 + 128 x 40 are the 384 x 168 of the launch.
  if (warp >= 8) {
    tc::reg_dec<40>();
    if (warp == 8) {
      // ---- copies: each CTA its half of A and B, counted by the barrier of the CTA that issues the products
      if (tc::elect_one()) {
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int j = 0; ok && walk.item(pair, j, t); ++j) {
          for (int kb = t.k0; kb < t.k1; ++kb) {
            if (!(ok = wait(empty + s, phase ^ 1u))) break;
            if (rank == 0) tc::mbar_expect_tx(full + s, 2 * C::STAGE);
            const uint32_t bar = tc::in_cta(tc::smem_u32(full + s), 0);
            uint32_t to = base + s * C::STAGE;
#pragma unroll
            for (int part = 0; part < C::PARTS; ++part, to += C::A) {
              const int m0 = t.m * 256 + (int)rank * 128;
              if (MODE == kDx) tc::tma_load_4d_pair(to, &maps.a, 0, 0, kb * 8, part * p.blocks + m0 / 128, bar);
              else if (MODE == kDw) tc::tma_load_4d_pair(to, &maps.a, 0, (kb & 1) * 2, m0 / 8, part * p.blocks + kb / 2, bar);
              else tc::tma_load_3d_pair(to, &maps.a, kb * 64, m0, part, bar);
            }
#pragma unroll
            for (int part = 0; part < C::PARTS; ++part, to += C::B) {
              const int n0 = t.n * C::BN + (int)rank * (C::BN / 2);
              if (C::B_MN) {
#pragma unroll
                for (int x = 0; x < C::BN / 128; ++x) tc::tma_load_3d_pair(to + x * 8192, &maps.b, n0 + 64 * x, p.b_row0 + kb * 64, part, bar);
              } else {
                tc::tma_load_3d_pair(to, &maps.b, kb * 64, p.b_row0 + n0, part, bar);
              }
            }
            if (++s == C::STAGES) { s = 0; phase ^= 1u; }
          }
        }
      }
    } else if (warp == 9) {
      // ---- products, by one thread of the pair
      if (rank == 0 && tc::elect_one()) {
        constexpr uint32_t idesc = tc::make_idesc_bf16(256, C::BN, C::A_MN, C::B_MN);
        constexpr uint32_t a_step = MODE == kDx ? 4096 : MODE == kDw ? 256 : 32, b_step = C::B_MN ? 2048 : 32;
        int s = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int j = 0; ok && walk.item(pair, j, t); ++j) {
          const int k1 = t.k1;
          for (int ks = t.k0; ok && ks < k1; ks += SEG) {
            if (!(ok = wait(acc_empty + acc, acc_phase ^ 1u))) break;
            tc::fence_after_sync();
            const uint32_t d = tmem + acc * BN;
            const int ke = min(ks + min(SEG, k1 - ks), k1);
            for (int kb = ks; kb < ke; ++kb) {
              if (!(ok = wait(full + s, phase))) break;
              tc::fence_after_sync();
              const uint32_t sa = base + s * C::STAGE, sb = sa + C::PARTS * C::A;
              auto product = [&](int pa, int pb, bool first) {
                const uint64_t da = MODE == kDx   ? tc::make_smem_desc(sa + pa * C::A, 2048, 128, tc::kSwizzleNone)
                                    : MODE == kDw ? tc::make_smem_desc(sa + pa * C::A, 128, 1024, tc::kSwizzleNone)
                                                  : tc::make_smem_desc(sa + pa * C::A, 16, 1024, tc::kSwizzle128);
                const uint64_t db = tc::make_smem_desc(sb + pb * C::B, C::B_MN ? 8192 : 16, 1024, tc::kSwizzle128);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  tc::mma_pair(d, da + (uint64_t)((k * a_step) >> 4), db + (uint64_t)((k * b_step) >> 4), idesc, !(first && k == 0));
              };
              if (F32) {
                product(2, 0, kb == ks);
                product(0, 2, false);
                product(1, 1, false);
                product(1, 0, false);
                product(0, 1, false);
              }
              product(0, 0, !F32 && kb == ks);
              tc::mma_commit_pair(empty + s);
              if (++s == C::STAGES) { s = 0; phase ^= 1u; }
            }
            if (!ok) break;
            tc::mma_commit_pair(acc_full + acc);
            if (++acc == C::ACCS) { acc = 0; acc_phase ^= 1u; }
          }
        }
      }
    }
  } else {
    tc::reg_inc<232>();
    // ---- epilogue: a thread has a row of the CTA's 128 and half of the tile's columns
    const int half = warp >> 2, quarter = warp & 3, mine = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int live = live_of(p);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int j = 0; ok && walk.item(pair, j, t); ++j) {
      const int m = t.m, n = t.n, k0 = t.k0, k1 = t.k1;
      const int row = m * 256 + (int)rank * 128 + mine, c0 = n * C::BN + half * C::COLS;
      int target = -1;  // what the epilogue needs of its row, under way beside the products
      float both = 0.f, back = 0.f;
      if constexpr (MODE == kStats) target = p.live ? p.tgt[row] : row < live ? target_at(p.targets, p.wide, p.V, row) : -1;
      if constexpr (MODE == kGrad) {
        target = p.tgt[row];
        both = F32 ? p.both[row] : p.both[row] / unit_of(p);
        back = -p.lse2[row];
      }
      float v[C::COLS];
      if (k0 == k1 || F32)
#pragma unroll
        for (int c = 0; c < C::COLS; ++c) v[c] = 0.f;
      for (int ks = k0; ks < k1; ks += min(SEG, k1 - ks)) {
        if (!(ok = wait(acc_full + acc, acc_phase))) break;
        __syncwarp();
        tc::fence_after_sync();
        const uint32_t d = tmem + lanes + acc * BN + half * C::COLS;
        if (!F32 && ks == k0) {
#pragma unroll
          for (int c = 0; c < C::COLS; c += 32) {
            uint32_t(&r)[32] = reinterpret_cast<uint32_t(&)[32]>(v[c]);
            tc::tmem_ld_32x32b_x32(d + c, r);
          }
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < C::COLS; c += 32) {
            uint32_t sum[32];
            tc::tmem_ld_32x32b_x32(d + c, sum);
            tc::tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) v[c + x] += __uint_as_float(sum[x]);
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::in_cta(tc::smem_u32(acc_empty + acc), 0));
        if (++acc == C::ACCS) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok) break;
      if constexpr (MODE == kStats || MODE == kGrad) {
        const int here = p.V - p.v0 - c0;  // columns from c0 that are in the vocabulary
        const int at = target - p.v0 - c0;
        const bool hit = target >= 0 && at >= 0 && at < C::COLS;
        if constexpr (MODE == kStats) {
          if (here < C::COLS)
#pragma unroll
            for (int c = 0; c < C::COLS; ++c) v[c] = c < here ? v[c] : -INFINITY;
          float top = v[0];
#pragma unroll
          for (int c = 1; c < C::COLS; ++c) top = fmaxf(top, v[c]);
          // (an infinite maximum would make NaNs of the infinities: the exponentials are then 0 or infinite)
          const float back = fabsf(top) == INFINITY ? 0.f : -top * kLog2e;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int c = 0; c < C::COLS; c += 2) {
            s0 += ex2(fmaf(v[c], kLog2e, back));
            s1 += ex2(fmaf(v[c + 1], kLog2e, back));
          }
          float sum = s0 + s1;
          if (__any_sync(0xffffffffu, hit)) {
            float z = 0.f;
#pragma unroll
            for (int c = 0; c < C::COLS; ++c) z = c == at ? v[c] : z;
            if (hit && row < live) p.hit[row] = z;
          }
          const int slot = j % C::RING;
          float2* buf = halves + slot * 128;
          uint64_t* there = halves_full + slot * 4 + quarter;
          if (half == 1) {
            buf[mine] = make_float2(top, sum);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(there);
          } else {
            if (!(ok = wait(there, (uint32_t)(j / C::RING) & 1u))) break;
            const float2 o = buf[mine];
            if (row < live) {
              float2 both{top, sum};
              add_sum(both, o);
              p.part[((size_t)(p.v0 / C::BN) + n) * p.pad + row] = both;
            }
          }
        } else {
          // (float32: the logit's distance from lse first, which leaves the exponent the error of that distance alone)
#pragma unroll
          for (int c = 0; c < C::COLS; ++c) v[c] = both * ex2(F32 ? (v[c] + back) * kLog2e : fmaf(v[c], kLog2e, back));
          if (row >= live || here < C::COLS)
#pragma unroll
            for (int c = 0; c < C::COLS; ++c) v[c] = row < live && c < here ? v[c] : 0.f;
          if (__any_sync(0xffffffffu, hit)) {
            const float a = !hit ? 0.f : F32 ? p.a[row] : p.a[row] / unit_of(p);
#pragma unroll
            for (int c = 0; c < C::COLS; ++c) v[c] = c == at ? v[c] - a : v[c];
          }
          bf16* to = p.g + g_at(p, m * 2 + rank, n * C::BN + half * C::COLS) + mine * 8;
#pragma unroll
          for (int part = 0; part < C::PARTS; ++part, to += p.pad * p.piece)
#pragma unroll
            for (int c = 0; c < C::COLS; c += 8) {
              const uint4 w = tc::pack8(v + c);
              *reinterpret_cast<uint4*>(to + c * 128) = w;
              if (part + 1 == C::PARTS) continue;
              float lo[8];  // what a part leaves of a value goes to the next
              tc::unpack8(w, lo);
#pragma unroll
              for (int y = 0; y < 8; ++y) v[c + y] -= lo[y];
            }
        }
      } else if (t.share >= 0 || (MODE == kDx && p.sums)) {
        const bool add = t.share < 0 && p.adds;
        float* to = (t.share >= 0 ? p.shares : p.sums) +
                    tile_at<C::BN>(t.share >= 0 ? (size_t)t.share : (size_t)m * walk.n_tiles + n, rank, mine, half * C::COLS);
#pragma unroll
        for (int c = 0; c < C::COLS; c += 32) {
          float4 old[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) old[x] = add ? *reinterpret_cast<const float4*>(to + (c / 4 + x) * 512) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float* e = v + c + 4 * x;
            *reinterpret_cast<float4*>(to + (c / 4 + x) * 512) = make_float4(old[x].x + e[0], old[x].y + e[1], old[x].z + e[2], old[x].w + e[3]);
          }
        }
      } else {
        const float unit = F32 ? 1.f : unit_of(p);
        if (!F32)
#pragma unroll
          for (int c = 0; c < C::COLS; ++c) v[c] *= unit;
        if (C::BOXES && p.whole) {
          leave_in_boxes<C::COLS>(&maps.g, staging + warp * 4096, v, c0, p.v0 + m * 256 + (int)rank * 128 + quarter * 32, lane);
        } else if (row < (MODE == kDx ? live : p.M)) {
          using T = std::conditional_t<F32, float, bf16>;
          T* to = static_cast<T*>(p.out) + (MODE == kDx ? (size_t)p.idx[row] : (size_t)p.v0 + row) * p.D;
#pragma unroll
          for (int c = 0; c < C::COLS; c += 8) store_row<T>(to, c0 + c, p.D, p.whole, v + c);
        }
      }
    }
    if (C::BOXES && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  __syncthreads();
  if (*bad)  // a wait gave up: copies that are still under way get two milliseconds to land before this memory is given back
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  if (threadIdx.x == 0) {
    if (MODE == kStats && p.flags) p.flags[blockIdx.x] = *bad ? 11 : 0;
    else if (*bad) atomicExch(p.status, 11);
  }
  __syncwarp();
  tc::fence_before_sync();
  tc::cluster_sync();  // (neither CTA leaves while the other's products read its shared memory or arrive at its barriers)
  tc::fence_after_sync();
  if (warp == 9) tc::tmem_dealloc_pair(tmem, 512);
}

// lse and loss of each row from its tiles' maxima and sums: 32 warps take every 32nd tile, then warp 0 theirs in order.
struct JoinP {
  const float2* part;
  const float* hit;
  const int32_t *live, *idx;
  const void* targets;   // where live is null: rows in their own places
  const int32_t* flags;
  int32_t* status;
  float *loss, *lse;
  size_t pad;
  int tiles, rows, wide, V, blocks;
};
constexpr int kJoinWarps = 32;
__global__ void __launch_bounds__(32 * kJoinWarps) lce_join_kernel(JoinP p) {
  begin_dependent();
  __shared__ float2 red[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const bool in = row < (p.live ? *p.live : p.rows);
  if (!p.live && blockIdx.x == 0) {
    const int any = __syncthreads_or((int)threadIdx.x < p.blocks && p.flags[threadIdx.x]);
    if (threadIdx.x == 0) *p.status = any ? 11 : 0;
  }
  float2 all{-INFINITY, 0.f};
  if (in)
    for (int t0 = warp; t0 < p.tiles; t0 += 4 * kJoinWarps) {
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = t0 + kJoinWarps * k < p.tiles ? p.part[(size_t)(t0 + kJoinWarps * k) * p.pad + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) add_sum(all, v[k]);
    }
  red[warp][lane] = all;
  __syncthreads();
  if (warp != 0 || !in) return;
  for (int w = 1; w < min(kJoinWarps, p.tiles); ++w) add_sum(all, red[w][lane]);
  const float lse = all.x + logf(all.y);
  const bool counts = p.live || target_at(p.targets, p.wide, p.V, row) >= 0;
  const int to = p.live ? p.idx[row] : row;
  p.lse[to] = counts ? lse : 0.f;
  p.loss[to] = counts ? lse - p.hit[row] : 0.f;
}
// Tiles that were cut along K, of dx and of dW: their shares in order, up to four at a time.  grid (at most pairs - 1 tiles, 2 CTAs' rows x
// pieces of 16 columns, 2).
template <bool F32, int BN>
__global__ void __launch_bounds__(256) lce_shares_kernel(const GemmP px, const GemmP py, int pairs_x, int pairs_y) {
  using T = std::conditional_t<F32, float, bf16>;
  begin_dependent();
  const bool is_dx = blockIdx.z == 0;
  const GemmP& p = is_dx ? px : py;
  const Walk walk(p, is_dx ? kDx : kDw, BN, is_dx ? pairs_x : pairs_y);
  const int tile = blockIdx.x;
  if (tile >= walk.rest) return;
  Item t;
  walk.place(walk.whole + tile, t);
  const int rank = blockIdx.y & 1, mine = threadIdx.x & 127, c0 = (blockIdx.y >> 1) * 16 + (threadIdx.x >> 7) * 8;
  const int from = tile * walk.kblocks, pair = from / walk.share, end = (from + walk.kblocks - 1) / walk.share;
  const int first_second = pair * walk.share < from;  // (only the first pair can have begun with another tile)
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const size_t in = tile_at<BN>(0, rank, mine, c0), stride = tile_at<BN>(1, 0, 0, 0);
  for (int q = pair; q <= end; q += 4) {
    float4 e[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (q + k <= end) {
        const float* at = p.shares + in + ((size_t)(q + k) * 2 + (q + k == pair ? first_second : 0)) * stride;
        e[k][0] = *reinterpret_cast<const float4*>(at);
        e[k][1] = *reinterpret_cast<const float4*>(at + 512);
      }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (q + k <= end)
#pragma unroll
        for (int x = 0; x < 2; ++x) { v[4 * x] += e[k][x].x; v[4 * x + 1] += e[k][x].y; v[4 * x + 2] += e[k][x].z; v[4 * x + 3] += e[k][x].w; }
  }
  if (is_dx && p.sums) {
    float* e = p.sums + tile_at<BN>((size_t)t.m * walk.n_tiles + t.n, rank, mine, c0);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float4 o = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
      if (p.adds) {
        const float4 old = *reinterpret_cast<const float4*>(e + x * 512);
        o.x += old.x; o.y += old.y; o.z += old.z; o.w += old.w;
      }
      *reinterpret_cast<float4*>(e + x * 512) = o;
    }
    return;
  }
  const int row = t.m * 256 + rank * 128 + mine;
  if (row >= (is_dx ? *p.live : p.M)) return;
  if (!F32) {
    const float unit = unit_of(p);
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] *= unit;
  }
  T* out = static_cast<T*>(p.out) + (is_dx ? (size_t)p.idx[row] : (size_t)p.v0 + row) * p.D;
  store_row<T>(out, t.n * BN + c0, p.D, p.whole, v);
}
// dx from its sums by tiles, in the tensor's type.  grid (128 rows, pieces of 64 columns).
template <bool F32, int BN>
__global__ void __launch_bounds__(256) lce_finish_kernel(const GemmP p, int n_tiles) {
  using T = std::conditional_t<F32, float, bf16>;
  begin_dependent();
  __shared__ float box[128][65];
  const int m0 = blockIdx.x * 128, col = blockIdx.y * 64, live = *p.live;
  if (m0 >= live) return;
  const float* from = p.sums + tile_at<BN>((size_t)(blockIdx.x >> 1) * n_tiles + col / BN, blockIdx.x & 1, threadIdx.x & 127, col % BN);
  const float unit = F32 ? 1.f : unit_of(p);
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int c4 = x * 2 + (threadIdx.x >> 7);
    const float4 v = *reinterpret_cast<const float4*>(from + c4 * 512);
    float* to = &box[threadIdx.x & 127][c4 * 4];
    to[0] = v.x * unit; to[1] = v.y * unit; to[2] = v.z * unit; to[3] = v.w * unit;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < 128 && m0 + r < live; r += 8) {
    T* to = static_cast<T*>(p.out) + (size_t)p.idx[m0 + r] * p.D + col;
    if (p.whole) {  // two columns a lane
      if (col + 2 * lane >= p.D) continue;
      if constexpr (F32) *reinterpret_cast<float2*>(to + 2 * lane) = make_float2(box[r][2 * lane], box[r][2 * lane + 1]);
      else *reinterpret_cast<uint32_t*>(to + 2 * lane) = tc::pack_bf16(box[r][2 * lane], box[r][2 * lane + 1]);
    } else {
#pragma unroll
      for (int c = lane; c < 64; c += 32)
        if (col + c < p.D) to[c] = from_f32<T>(box[r][c]);
    }
  }
}

// ------------------------------------------------------------------ host
typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                           const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static Encode encode_fn() {
  static const Encode encode = []() -> Encode {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  return encode;
}
static bool make_map(CUtensorMap* m, const void* base, uint64_t cols, uint64_t rows, uint64_t parts, uint64_t pitch, uint64_t part_pitch,
                     uint32_t box_rows) {
  const Encode encode = encode_fn();
  const cuuint64_t dims[3] = {cols, rows, parts}, strides[2] = {pitch * 2, part_pitch * 2};
  const cuuint32_t box[3] = {64, box_rows, 1}, step[3] = {1, 1, 1};
  return encode && encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// g: boxes of 64 columns of 128 rows, or of 128 columns of 64 rows.
static bool make_g_map(CUtensorMap* m, const void* g, uint64_t piece, uint64_t blocks, bool columns) {
  const cuuint64_t dims[4] = {256, 4, piece / 8, blocks}, strides[3] = {512, 2048, piece * 256};
  const cuuint32_t box[4] = {256, columns ? 2u : 4u, columns ? 16u : 8u, 1}, step[4] = {1, 1, 1, 1};
  const Encode encode = encode_fn();
  return encode && encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(g), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kPairs = 74;
// Bytes of g that are kept at a time.
constexpr size_t kGradBytes = (size_t)640 << 20;
constexpr size_t kPackBytes = (size_t)256 << 20;

struct Plan {
  bool f32, pack_w, direct;
  int parts, Dp, piece, pieces;
  int BN, BD;             // columns of a tile: of logits, of gradients
  size_t N, pad;
  // workspace
  int32_t *status, *live, *counts, *idx, *tgt, *flags;
  float *a, *both, *lse2, *hit, *sums, *shares[2];
  float2* part;
  bf16 *xc, *wc, *g;
  size_t bytes;
};
// bwd: the backward pass.  x and weight only say whether they can be read as they are.
static Plan plan(const mxb_linear_ce_desc* d, const void* x, const void* weight, bool bwd, void* base) {
  Plan q{};
  q.f32 = d->io_dtype == MXB_F32;
  q.parts = q.f32 ? 3 : 1;
  q.BD = d->D <= 128 ? 128 : 256;
  q.Dp = (d->D + 7) / 8 * 8;
  q.N = d->rows;
  q.pad = std::max<size_t>((q.N + 255) / 256 * 256, 256);
  // (a base off 16 bytes: as many bytes of workspace are asked for whatever the pointer, so that the query needs none)
  q.pack_w = q.f32 || d->D % 8 != 0 || (reinterpret_cast<uintptr_t>(weight) & 15) != 0;
  const int64_t all = ((int64_t)d->V + 255) / 256 * 256;
  int64_t most = bwd ? (int64_t)(kGradBytes / (q.pad * q.parts * 2)) : all;
  most = std::min<int64_t>(most, (int64_t)(kPackBytes / ((size_t)q.Dp * q.parts * 2)));
  // whole rounds of dW's tiles where a piece is that large: nothing of it is cut into shares then
  const int64_t d_tiles = (d->D + q.BD - 1) / q.BD, round = kPairs / std::gcd<int64_t, int64_t>(kPairs, d_tiles);
  if (bwd && most < all && most / 256 >= round) most = most / 256 / round * round * 256;
  q.piece = (int)std::min<int64_t>(all, std::max<int64_t>(256, most / 256 * 256));
  // few tokens: a tile of 256 rows costs as much with all of them as with some (512 tokens, 32768 words of 1024: 46 us with their
  // rows moved together first, 36 without)
  q.direct = !bwd && !q.pack_w && q.N <= 1024 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (!bwd && !q.pack_w) q.piece = (int)all;
  q.pieces = (int)((d->V + (int64_t)q.piece - 1) / q.piece);
  // float32, tiles of dx and dW: narrow ones start sooner (a third of the bytes before the first product), wide ones have fewer reads
  // (2048 tokens, 5003 words of 448: gradients 159 us with narrow, 165 with wide ones on one GPU, up to 173 on others; 4096, 32000 words:
  // 1705 and 1537)
  const int64_t words = std::min<int64_t>(q.piece, d->V);
  if (q.f32 && (words + 255) / 256 * d_tiles < kPairs) q.BD = 128;
  // float32, tiles of logits: those of 128 columns take a little over half as long as those of 256 (their operands' reads bound them), which pays
  // where it saves as much of the last round
  auto rounds = [&](int64_t columns) { return ((int64_t)q.pad / 256 * ((words + columns - 1) / columns) + kPairs - 1) / kPairs; };
  q.BN = q.f32 && 115 * rounds(128) < 200 * rounds(256) ? 128 : 256;
  const int64_t m_tiles = q.pad / 256, out_tiles = (d->D + q.BD - 1) / q.BD;
  Carver c(base);
  q.status = c.take<int32_t>(64);  // (the device's error word leads the workspace)
  q.live = c.take<int32_t>(1);
  q.flags = c.take<int32_t>(2 * kPairs);
  q.counts = c.take<int32_t>(q.N / kCountRows + 1);
  q.idx = c.take<int32_t>(q.pad);
  q.tgt = c.take<int32_t>(q.pad);
  q.xc = c.take<bf16>((size_t)q.parts * q.pad * q.Dp);
  // the packed piece of W: asked for where D alone says so; a base off 16 bytes is refused instead
  if (q.f32 || d->D % 8 != 0) q.wc = c.take<bf16>((size_t)q.parts * q.piece * q.Dp);
  if (!bwd) {
    q.hit = c.take<float>(q.pad);
    q.part = c.take<float2>(((size_t)d->V + q.BN - 1) / q.BN * q.pad);
  } else {
    q.a = c.take<float>(q.pad);
    q.both = c.take<float>(q.pad);
    q.lse2 = c.take<float>(q.pad);
    q.g = c.take<bf16>((size_t)q.parts * q.pad * q.piece);
    if (q.pieces > 1) q.sums = c.take<float>((size_t)m_tiles * out_tiles * 256 * q.BD);
    for (float*& s : q.shares) s = c.take<float>((size_t)kPairs * 2 * 256 * q.BD);
  }
  q.bytes = c.bytes();
  return q;
}

// tiles, and blocks of 64 of K, at most (the tokens that count may be fewer)
template <int MODE, bool F32, int BN>
static mxb_status launch_gemm(const GemmP& p, const Maps& maps, int pairs, cudaStream_t st) {
  using C = Cfg<MODE, F32, BN>;
  if (MXB_ALLOW_SMEM(C::SMEM, lce_gemm_kernel<MODE, F32, BN>) != MXB_OK) return MXB_ERR_CUDA;
  // (warps that ask for registers which the launch did not bring would wait for good)
  static const bool fits = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, lce_gemm_kernel<MODE, F32, BN>) == cudaSuccess && a.numRegs * kThreads >= 256 * 232 + 128 * 40;
  }();
  if (!fits) return MXB_ERR_UNSUPPORTED;
  static const char* const names[] = {"lce_stats_kernel", "lce_grad_kernel", "lce_dx_kernel", "lce_dw_kernel"};
  MXB_LAUNCH(names[MODE], st, (launch_kernel(lce_gemm_kernel<MODE, F32, BN>, 2 * pairs, kThreads, C::SMEM, st, p, maps)));
  return check_launch(names[MODE]);
}
// Pairs for so many tiles, whose sums may be cut (tiles and blocks of 64 of K at most: the tokens that count may be fewer).
static int pairs_for(int64_t tiles, int64_t kblocks) {
  return (int)std::min<int64_t>(kblocks >= 16 ? std::max<int64_t>(tiles, tiles * kblocks / 8) : tiles, kPairs);
}
template <typename T>
static mxb_status pack(PackP& p, int32_t* counts, cudaStream_t st) {
  if (p.N > 4 * kCountRows) {  // (up to there every block counts for itself)
    p.counts = counts;
    MXB_LAUNCH("lce_count_kernel", st, (launch_kernel(lce_count_kernel, (unsigned)(p.N / kCountRows), 256, 0, st, p, counts)));
  }
  p.each = p.N > 148 * 32 ? 4 : 1;
  const int blocks = (int)((p.N + 8 * p.each - 1) / (8 * p.each));
  MXB_LAUNCH("lce_pack_kernel", st, (launch_kernel(lce_pack_kernel<T>, blocks + 32 + (p.w_rows + 7) / 8, 256, 0, st, p, blocks)));
  return check_launch("lce_pack_kernel");
}

template <bool F32, int BN, int BD>
static mxb_status run(const mxb_linear_ce_desc* d, const Plan& q, PackP& pk, const void* weight, void* dweight, cudaStream_t st) {
  using T = std::conditional_t<F32, float, bf16>;
  const bool bwd = pk.d_loss != nullptr;
  mxb_status s = MXB_OK;
  if (!q.direct) {
    if (q.pack_w) {
      pk.w = weight;
      pk.wc = q.wc;
      pk.w_pad = q.piece;
      pk.w_rows = (int)std::min<int64_t>(q.piece, d->V);
    }
    s = pack<T>(pk, q.counts, st);
    if (s != MXB_OK) return s;
  }
  const size_t pad = q.pad;
  const int D = d->D;
  GemmP last{};  // of the last piece's dx
  int blocks = 0;
  const int64_t m_tiles = pad / 256, d_tiles = (D + BD - 1) / BD;
  for (int piece = 0; piece < q.pieces; ++piece) {
    const int v0 = piece * q.piece, rows = (int)std::min<int64_t>(q.piece, (int64_t)d->V - v0);
    const void* w = weight;
    uint64_t w_rows = d->V, w_part = (uint64_t)d->V * D;
    int w_row0 = v0;
    if (q.pack_w) {
      if (piece > 0)
        MXB_LAUNCH("lce_pack_weight_kernel", st,
                   (launch_kernel(lce_pack_weight_kernel<T>, (unsigned)((rows + 7) / 8), 256, 0, st, static_cast<const T*>(weight) + (size_t)v0 * D,
                                  q.wc, rows, (size_t)q.piece, D, q.Dp)));
      w = q.wc;
      w_rows = rows;
      w_part = (uint64_t)q.piece * q.Dp;
      w_row0 = 0;
    }
    GemmP p{};
    p.live = q.direct ? nullptr : q.live;
    p.targets = pk.targets;
    p.wide = pk.wide;
    p.rows = (int)q.N;
    p.flags = q.direct ? q.flags : nullptr;
    p.status = q.status;
    p.g = q.g;
    p.piece = q.piece;
    p.blocks = (int)(pad / 128);
    p.tgt = q.tgt;
    p.idx = q.idx;
    p.v0 = v0;
    p.V = d->V;
    p.pad = pad;
    p.D = D;
    // as many rows of tiles as keep their x in L2 (24 MB): W is read once for all of them (28672 tokens, 65536 words of 1024: loss 2.70 ms,
    // by groups of eight 2.83)
    p.group = (int)std::min<int64_t>(64, std::max<int64_t>(8, (24 << 20) / (256 * 2 * (int64_t)q.Dp * q.parts)));
    Maps maps;
    std::memset(&maps, 0, sizeof maps);
    const bool ok = q.direct ? make_map(&maps.a, pk.x, D, q.N, 1, D, q.N * D, 128) : make_map(&maps.a, q.xc, q.Dp, pad, q.parts, q.Dp, pad * q.Dp, 128);
    if (!ok || !make_map(&maps.b, w, q.Dp, w_rows, q.parts, q.Dp, w_part, BN / 2)) return MXB_ERR_UNSUPPORTED;
    p.N = rows;
    p.K = D;
    p.b_row0 = w_row0;
    p.part = q.part;
    p.hit = q.hit;
    p.a = q.a;
    p.both = q.both;
    p.lse2 = q.lse2;
    const int64_t tiles = m_tiles * ((rows + BN - 1) / BN);
    const int pairs = (int)std::min<int64_t>(tiles, kPairs);
    s = bwd ? launch_gemm<kGrad, F32, BN>(p, maps, pairs, st) : launch_gemm<kStats, F32, BN>(p, maps, pairs, st);
    blocks = 2 * pairs;
    if (s != MXB_OK) return s;
    if (bwd) {
      // dx: sums over the piece, in the order of the pieces
      GemmP x = p;
      x.N = D;
      x.K = rows;
      x.b_row0 = w_row0;
      x.sums = q.sums;
      x.shares = q.shares[0];
      x.group = d_tiles <= 16 ? 1 : 8;  // all columns of a row of tiles side by side: its g is read once
      x.adds = piece > 0;
      x.out = pk.dx;
      x.whole = D % 8 == 0 && (reinterpret_cast<uintptr_t>(pk.dx) & 15) == 0;
      if (!make_g_map(&maps.a, q.g, q.piece, pad / 128 * q.parts, false) || !make_map(&maps.b, w, q.Dp, w_rows, q.parts, q.Dp, w_part, 64))
        return MXB_ERR_UNSUPPORTED;
      const int64_t x_tiles = m_tiles * d_tiles, x_blocks = (rows + 63) / 64, y_tiles = (int64_t)((rows + 255) / 256) * d_tiles, y_blocks = (q.N + 63) / 64;
      const int x_pairs = pairs_for(x_tiles, x_blocks), y_pairs = pairs_for(y_tiles, y_blocks);
      s = launch_gemm<kDx, F32, BD>(x, maps, x_pairs, st);
      if (s != MXB_OK) return s;
      last = x;
      // dW: sums over the tokens
      GemmP y = p;
      y.M = rows;
      y.N = D;
      y.b_row0 = 0;
      y.shares = q.shares[1];
      y.group = d_tiles <= 16 ? 1 : 8;
      y.out = dweight;
      y.whole = D % 8 == 0 && (reinterpret_cast<uintptr_t>(dweight) & 15) == 0;
      if (!make_g_map(&maps.a, q.g, q.piece, pad / 128 * q.parts, true) || !make_map(&maps.b, q.xc, q.Dp, pad, q.parts, q.Dp, pad * q.Dp, 64))
        return MXB_ERR_UNSUPPORTED;
      if (!F32 && y.whole && !make_map(&maps.g, dweight, D, d->V, 1, D, (uint64_t)d->V * D, 32)) return MXB_ERR_UNSUPPORTED;
      s = launch_gemm<kDw, F32, BD>(y, maps, y_pairs, st);
      if (s != MXB_OK) return s;
      // (how many tiles of dx there are, the device knows)
      const int64_t x_cut = x_blocks >= 16 ? std::min<int64_t>(x_tiles, x_pairs - 1) : 0, y_cut = y_blocks >= 16 ? y_tiles % y_pairs : 0;
      if (x_cut || y_cut)
        MXB_LAUNCH("lce_shares_kernel", st,
                   (launch_kernel(lce_shares_kernel<F32, BD>, dim3((unsigned)std::max(x_cut, y_cut), 2 * BD / 16, 2), 256, 0, st, x, y, x_pairs, y_pairs)));
    }
  }
  if (bwd) {
    if (q.sums)
      MXB_LAUNCH("lce_finish_kernel", st,
                 (launch_kernel(lce_finish_kernel<F32, BD>, dim3((unsigned)(pad / 128), (unsigned)((D + 63) / 64)), 256, 0, st, last, (int)d_tiles)));
    return check_launch("linear_ce_bwd");
  }
  const JoinP j{q.part, q.hit, q.direct ? nullptr : q.live, q.idx, pk.targets, q.flags, q.status, pk.loss, pk.lse_out, pad, (d->V + BN - 1) / BN, (int)q.N,
                pk.wide, d->V, blocks};
  MXB_LAUNCH("lce_join_kernel", st, (launch_kernel(lce_join_kernel, (unsigned)(pad / 32), 32 * kJoinWarps, 0, st, j)));
  return check_launch("linear_ce_fwd");
}
static mxb_status by_shape(const mxb_linear_ce_desc* d, const Plan& q, PackP& p, const void* weight, void* dweight, cudaStream_t st) {
  auto by_width = [&](auto f32, auto bn) {
    constexpr bool F = decltype(f32)::value;
    constexpr int BN = decltype(bn)::value;
    return q.BD == 128 ? run<F, BN, 128>(d, q, p, weight, dweight, st) : run<F, BN, 256>(d, q, p, weight, dweight, st);
  };
  constexpr std::integral_constant<int, 128> narrow;
  constexpr std::integral_constant<int, 256> wide;
  if (!q.f32) return by_width(std::false_type{}, wide);
  return q.BN == 128 ? by_width(std::true_type{}, narrow) : by_width(std::true_type{}, wide);
}
static PackP pack_args(const mxb_linear_ce_desc* d, const Plan& q, const void* x, const void* targets) {
  PackP p{};
  p.targets = targets;
  p.x = x;
  p.live = q.live;
  p.idx = q.idx;
  p.tgt = q.tgt;
  p.a = q.a;
  p.both = q.both;
  p.lse2 = q.lse2;
  p.xc = q.xc;
  p.status = q.status;
  p.N = q.N;
  p.pad = q.pad;
  p.V = d->V;
  p.D = d->D;
  p.Dp = q.Dp;
  p.wide = d->target_bytes == 8;
  return p;
}

}  // namespace lce

size_t linear_ce_scratch(const mxb_linear_ce_desc* d, bool bwd) { return lce::plan(d, nullptr, nullptr, bwd, nullptr).bytes; }

mxb_status linear_ce_fwd(const mxb_linear_ce_desc* d, const void* x, const void* weight, const void* targets, float* loss, float* lse,
                         void* workspace, cudaStream_t st) {
  const lce::Plan q = lce::plan(d, x, weight, false, workspace);
  lce::PackP p = lce::pack_args(d, q, x, targets);
  p.loss = loss;
  p.lse_out = lse;
  return lce::by_shape(d, q, p, weight, nullptr, st);
}
mxb_status linear_ce_bwd(const mxb_linear_ce_desc* d, const void* x, const void* weight, const void* targets, const float* lse, const float* d_loss,
                         const float* d_lse, void* dx, void* dweight, void* workspace, cudaStream_t st) {
  const lce::Plan q = lce::plan(d, x, weight, true, workspace);
  lce::PackP p = lce::pack_args(d, q, x, targets);
  p.lse = lse;
  p.d_loss = d_loss;
  p.d_lse = d_lse;
  p.dx = dx;
  return lce::by_shape(d, q, p, weight, dweight, st);
}

}  // namespace mxb
