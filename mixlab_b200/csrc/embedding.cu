// Rows of the token matrix and their gradient:
//     y_t = s W[i_t],    dW_v = s sum over the t with i_t = v of dy_t, in the order of t
// A token outside 0 .. V-1 is padding: its row of y is zero and it has no part in dW.
//
// Both are HBM streams.  32768 rows of 2048 columns, bf16 into float32: 60 us, 403 MB at the measured copy rate.  256 rows 4.6 us, of
// which the call on the host is most.  Their gradient, float32 for 65536 words: 134 us (671 MB: 76 % of the copy rate); by the counters,
// which time each launch alone and cold, the sort with zeros beside it takes 34, the sums and the other zeros 90, the join 13; 2047 rows of 448
// columns 14 us, three launches.  Tokens above 65536, sorted in launches of their own: 131072 rows of 1024 columns 148 us for 82 of bytes.
// Added to what is there, 32768 rows of 2048 of 11 thousand words: 98 us for 47 of bytes, 25 of them the sort.
//
// The gradient sorts the positions by token (stable, so that a token's positions stand in their own order and the sums do not depend
// on how blocks run), cuts the sorted list into runs of equal length, whatever the tokens' counts are, and adds up the rows of each
// run, the next batch of rows under way beside them; a token that lies in several runs leaves a partial row in each, which a last
// launch adds in the order of the runs.  Rows of words that do not occur are written by blocks of the same launch as the sums, the last
// of them beside the sort.  Sums are float32 and rounded once.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "row_pieces.cuh"
#include "tcgen05.cuh"

namespace mxb {
namespace embed {

using bf16 = __nv_bfloat16;

template <typename TOK>
__device__ __forceinline__ int token_of(const TOK* tokens, size_t t, int V) {  // V: padding
  const TOK v = tokens[t];
  return v >= 0 && v < (TOK)V ? (int)v : V;
}
// (a 32-bit token is never above what V can be)
template <>
__device__ __forceinline__ int token_of<int32_t>(const int32_t* tokens, size_t t, int V) {
  const int32_t v = tokens[t];
  return v >= 0 && v < V ? v : V;
}

// Zeros from one address to another, both multiples of two, by so many threads: whole pieces of 16 bytes, pairs of bytes in front of and
// behind them.
__device__ __forceinline__ void fill_zeros(char* begin, char* end, size_t thread, size_t threads) {
  char* from = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(begin) + 15) & ~(uintptr_t)15);
  char* to = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(end) & ~(uintptr_t)15);
  for (char* at = from + thread * 16; at < to; at += threads * 16) *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
  if (thread < 8) {
    if (begin + thread * 2 < (from < end ? from : end)) *reinterpret_cast<uint16_t*>(begin + thread * 2) = 0;
    if (to >= from && to + thread * 2 < end) *reinterpret_cast<uint16_t*>(to + thread * 2) = 0;
  }
}

// ------------------------------------------------------------------ forward
struct FwdP {
  const void* tokens;
  const void* weight;
  void* out;
  size_t N;
  int V, D;
  float scale;
};
// TPR threads a row, a group of them takes R rows at a time.
template <typename TOK, typename IN, typename OUT, int R, bool V>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(FwdP p, int tpr) {
  begin_dependent();
  const int groups = 256 / tpr, lane = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr;
  const f2 s = dup2(p.scale);
  for (size_t t0 = ((size_t)blockIdx.x * groups + group) * R; t0 < p.N; t0 += (size_t)gridDim.x * groups * R) {
    int tok[R];
#pragma unroll
    for (int r = 0; r < R; ++r) tok[r] = t0 + r < p.N ? token_of(static_cast<const TOK*>(p.tokens), t0 + r, p.V) : p.V;
    for (int c = 0; c < p.D; c += tpr * 8) {
      f2 e[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (tok[r] < p.V) {
          load_cols<IN, V>(static_cast<const IN*>(p.weight) + (size_t)tok[r] * p.D, c, lane, tpr, p.D, e[r]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[r][i] = 0;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (t0 + r >= p.N) continue;
        if (tok[r] < p.V)
#pragma unroll
          for (int i = 0; i < 4; ++i) e[r][i] = mul2(e[r][i], s);
        store_cols<OUT, V>(static_cast<OUT*>(p.out) + (t0 + r) * p.D, c, lane, tpr, p.D, e[r]);
      }
    }
  }
}

// ------------------------------------------------------------------ sorting the positions by token
// Least significant digit first, at most 10 bits a pass.  A block takes kTile consecutive entries.
constexpr int kTile = 2048, kSortThreads = 256, kWarps = kSortThreads / 32, kEach = kTile / kSortThreads, kMaxDigits = 1024;
struct SortP {
  const void* tokens;
  const int2* in;                  // tokens and their positions; null in the first pass
  int2* out;
  int32_t* hist;                   // [digits][tiles]
  uint32_t* rows;                  // the first pass sets it to zero
  int N, V, shift, digits, bits, tiles;
};
template <typename TOK>
__device__ __forceinline__ int key_at(const SortP& p, int i) {
  return p.in ? p.in[i].x : token_of(static_cast<const TOK*>(p.tokens), i, p.V);
}
// The lanes of the warp whose digits (of so many bits) are this lane's; in: which lanes have one.  (By __match_any_sync, which takes
// the longer the more digits there are, 4096 entries' ranks take 7800 cycles, so 2600.)
__device__ __forceinline__ uint32_t same_digit(int d, int bits, bool in) {
  uint32_t peers = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    if (b >= bits) break;
    const uint32_t m = __ballot_sync(0xffffffffu, d >> b & 1);
    peers &= d >> b & 1 ? m : ~m;
  }
  return peers;
}
template <typename TOK>
__global__ void __launch_bounds__(kSortThreads) embedding_count_kernel(SortP p) {
  begin_dependent();
  __shared__ int32_t count[kMaxDigits];
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) count[d] = 0;
  if (!p.in)
    for (int64_t w = (int64_t)blockIdx.x * kSortThreads + threadIdx.x; w <= p.V / 32; w += (int64_t)gridDim.x * kSortThreads) p.rows[w] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = (int64_t)blockIdx.x * kTile + k * kSortThreads + threadIdx.x;
    if (i < p.N) atomicAdd(&count[(key_at<TOK>(p, (int)i) >> p.shift) & (p.digits - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) p.hist[(size_t)d * p.tiles + blockIdx.x] = count[d];
}
// The counts become the places of each digit's first entry of each tile, without the digits in front: those are added where the
// places are used, from the row ends that this leaves in total[digit].
__global__ void __launch_bounds__(256) embedding_scan_kernel(int32_t* hist, int32_t* total, int tiles) {
  begin_dependent();
  __shared__ int32_t warps[8];
  int32_t* row = hist + (size_t)blockIdx.x * tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t before = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    const int32_t v = t < tiles ? row[t] : 0;
    int32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) warps[warp] = s;
    __syncthreads();
    int32_t base = before, all = before;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) base += warps[w];
      all += warps[w];
    }
    if (t < tiles) row[t] = base + s - v;
    before = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = before;
}
// Each entry to its place: digits in front, tiles in front, warps in front, entries in front in the warp.
template <typename TOK>
__global__ void __launch_bounds__(kSortThreads) embedding_place_kernel(SortP p, const int32_t* total) {
  begin_dependent();
  __shared__ int32_t place[kMaxDigits];
  __shared__ uint16_t mine[kWarps][kMaxDigits];
  __shared__ int32_t sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < kWarps * p.digits; d += kSortThreads) mine[d / p.digits][d % p.digits] = 0;
  // places of the digits: an exclusive sum of the totals, each thread four of them (kMaxDigits / kSortThreads)
  int32_t v[4], sum = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = threadIdx.x * 4 + k;
    v[k] = d < p.digits ? total[d] : 0;
    sum += v[k];
  }
  int32_t s = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) sums[warp] = s;
  __syncthreads();
  s -= sum;
  for (int w = 0; w < warp; ++w) s += sums[w];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = threadIdx.x * 4 + k;
    if (d < p.digits) place[d] = s + p.hist[(size_t)d * p.tiles + blockIdx.x];
    s += v[k];
  }
  // a warp takes 32 consecutive entries at a time, kEach times
  const int64_t first = (int64_t)blockIdx.x * kTile + warp * (32 * kEach) + lane;
  int key[kEach], rank[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = first + 32 * k;
    const bool in = i < p.N;
    key[k] = in ? key_at<TOK>(p, (int)i) : -1;
    const int d = in ? (key[k] >> p.shift) & (p.digits - 1) : 0;
    const uint32_t peers = same_digit(d, p.bits, in);
    rank[k] = 0;
    if (in) rank[k] = mine[warp][d] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (in && (peers >> lane) == 1u) mine[warp][d] = (uint16_t)(rank[k] + 1);  // the last of its digit in the warp
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) {
    int before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int n = mine[w][d];
      mine[w][d] = (uint16_t)before;
      before += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t i = first + 32 * k;
    if (i >= p.N) continue;
    const int d = (key[k] >> p.shift) & (p.digits - 1), to = place[d] + mine[warp][d] + rank[k];
    p.out[to] = make_int2(key[k], p.in ? p.in[i].y : (int)i);
  }
}

// A bit for each token that occurs, by its first entry in sorted order.  (By every entry, words of frequent tokens are updated so
// often that the updates, one after the other, took 20 us of 32768 tokens.)
__device__ __forceinline__ void mark_first(const int2* entry, int i, uint32_t* rows) {
  const int k = entry[i].x;
  if (i == 0 || entry[i - 1].x != k) atomicOr(rows + k / 32, 1u << (k & 31));
}
__global__ void __launch_bounds__(256) embedding_mark_kernel(const int2* entry, int N, uint32_t* rows) {
  begin_dependent();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < N) mark_first(entry, (int)i, rows);
}

// Few entries: every block reads all tokens and counts, for 32 entries, those that stand in front, eight threads an entry; its part of
// the bits that say which tokens occur likewise.  (Gradients of 2047 tokens, 257 words of
// 448 columns 13.8 us, with the sort in a cluster 15.9; of 3000, 50000 words of 1024 columns 52 and 58; of 8000, 1000 words 34 and 23.)
constexpr int kRankMost = 4096;
template <typename TOK>
__global__ void __launch_bounds__(256) embedding_rank_kernel(const void* tokens, int2* out, uint32_t* rows, int N, int V) {
  begin_dependent();
  __shared__ __align__(16) int32_t key[kRankMost];
  __shared__ uint32_t bits[256];
  const int most = (N + 31) / 32 * 32;
  for (int i = threadIdx.x; i < most; i += 256) key[i] = i < N ? token_of(static_cast<const TOK*>(tokens), i, V) : INT32_MAX;
  __syncthreads();
  const int i = blockIdx.x * 32 + threadIdx.x / 8, sub = threadIdx.x & 7;
  if (blockIdx.x * 32 < N) {
    const int k = i < N ? key[i] : -1;
    int before = 0;
    for (int j = sub * 4; j < most; j += 32) {
      const int4 o = *reinterpret_cast<const int4*>(key + j);
      before += (o.x < k || (o.x == k && j < i)) + (o.y < k || (o.y == k && j + 1 < i)) + (o.z < k || (o.z == k && j + 2 < i)) +
                (o.w < k || (o.w == k && j + 3 < i));
    }
    before += __shfl_xor_sync(0xffffffffu, before, 1);
    before += __shfl_xor_sync(0xffffffffu, before, 2);
    before += __shfl_xor_sync(0xffffffffu, before, 4);
    if (sub == 0 && i < N) out[before] = make_int2(k, i);
  }
  const int64_t words = (int64_t)V / 32 + 1;
  for (int64_t w0 = (int64_t)blockIdx.x * 256; w0 < words; w0 += (int64_t)gridDim.x * 256) {
    __syncthreads();
    bits[threadIdx.x] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < N; j += 256) {
      const int64_t w = key[j] / 32 - w0;
      if (w >= 0 && w < 256) atomicOr(&bits[w], 1u << (key[j] & 31));
    }
    __syncthreads();
    if (w0 + threadIdx.x < words) rows[w0 + threadIdx.x] = bits[threadIdx.x];
  }
}

// The whole sort in one launch for up to kClusterEntries entries: a cluster of CTAs, each with an equal share of the entries, that read
// each other's digit counts through distributed shared memory.  A CTA sorts its entries by the digit in its own memory first, so that
// it writes runs of neighbours: entries written one by one from their places in the warps were 6 to 8 thousand of 27 thousand
// cycles a pass of 32768 entries.  (Their gradient, rows of 2048 columns: 155 us with a sort of three launches a pass, so 139.)
constexpr int kClusterThreads = 1024, kClusterEach = 8, kClusterMost = 8, kClusterEntries = kClusterThreads * kClusterEach * kClusterMost;
__device__ __forceinline__ int32_t of_cta(const int32_t* p, uint32_t rank) {
  int32_t v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(tc::in_cta(tc::smem_u32(p), rank)) : "memory");
  return v;
}
struct ClusterP {
  const void* tokens;
  int2* entry[2];
  uint32_t* rows;
  int N, V, bits, passes, share, ctas;  // share: entries of a CTA; ctas: of the cluster that sorts
  char *zero_from, *zero_to;            // memory that the other clusters fill with zeros
};
__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
template <typename TOK>
__global__ void __launch_bounds__(kClusterThreads) embedding_sort_kernel(ClusterP p) {
  begin_dependent();
  if ((int)blockIdx.x >= p.ctas) {
    fill_zeros(p.zero_from, p.zero_to, (size_t)(blockIdx.x - p.ctas) * kClusterThreads + threadIdx.x, (size_t)(gridDim.x - p.ctas) * kClusterThreads);
    return;
  }
  extern __shared__ int2 local[];  // [share] entries by digit, then counts of the warps [32][digits]
  __shared__ int32_t hist[kMaxDigits], place[kMaxDigits], inside[kMaxDigits], sums[2][32];
  uint16_t* mine = reinterpret_cast<uint16_t*>(local + p.share);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << p.bits, ctas = p.ctas, rank = tc::cluster_rank();
  const int each = (p.share + kClusterThreads - 1) / kClusterThreads;  // rounds of 32 consecutive entries a warp
  const int begin = min(rank * p.share, p.N), end = min(begin + p.share, p.N), first = begin + warp * 32 * each + lane;
  for (int64_t w = (int64_t)rank * kClusterThreads + threadIdx.x; w <= p.V / 32; w += (int64_t)ctas * kClusterThreads) p.rows[w] = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const bool odd = pass & 1;
    const int2* in = odd ? p.entry[0] : p.entry[1];
    int2* out = odd ? p.entry[1] : p.entry[0];
    int2 entry[kClusterEach];
    int at[kClusterEach];
#pragma unroll
    for (int k = 0; k < kClusterEach; ++k) {
      const int i = first + 32 * k;
      entry[k] = make_int2(-1, 0);
      if (k < each && i < end) entry[k] = pass ? in[i] : make_int2(token_of(static_cast<const TOK*>(p.tokens), i, p.V), i);
    }
    for (int d = threadIdx.x; d < 16 * digits; d += kClusterThreads) reinterpret_cast<uint32_t*>(mine)[d] = 0;
    __syncthreads();
    uint16_t* own = mine + warp * digits;
#pragma unroll
    for (int k = 0; k < kClusterEach; ++k) {
      if (k >= each) break;
      const bool has = entry[k].x >= 0;
      const int d = has ? entry[k].x >> shift & digits - 1 : 0;
      const uint32_t peers = same_digit(d, p.bits, has);
      at[k] = 0;
      if (has) at[k] = own[d] + __popc(peers & ((1u << lane) - 1u));
      __syncwarp();
      if (has && (peers >> lane) == 1u) own[d] = (uint16_t)(at[k] + 1);  // the last of its digit in the warp
      __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kClusterThreads) {
      int before = 0;
#pragma unroll
      for (int w0 = 0; w0 < 32; w0 += 16) {
        int n[16];
#pragma unroll
        for (int w = 0; w < 16; ++w) n[w] = mine[(w0 + w) * digits + d];
#pragma unroll
        for (int w = 0; w < 16; ++w) {
          mine[(w0 + w) * digits + d] = (uint16_t)before;
          before += n[w];
        }
      }
      hist[d] = before;
    }
    tc::cluster_sync();
    // places of the digits: those in front (an exclusive sum over the cluster's totals) and CTAs in front; likewise in this CTA alone
    int before = 0, total = 0, here = 0;
    if ((int)threadIdx.x < digits) {
      int n[kClusterMost];
#pragma unroll
      for (int r = 0; r < kClusterMost; ++r) n[r] = r < ctas ? of_cta(hist + threadIdx.x, r) : 0;
#pragma unroll
      for (int r = 0; r < kClusterMost; ++r) {
        if (r < rank) before += n[r];
        total += n[r];
      }
      here = hist[threadIdx.x];
    }
    const int all = warp_scan(total, lane), own_all = warp_scan(here, lane);
    if (lane == 31) {
      sums[0][warp] = all;
      sums[1][warp] = own_all;
    }
    __syncthreads();
    if (warp < 2) {
      const int v = sums[warp][lane];
      sums[warp][lane] = warp_scan(v, lane) - v;
    }
    __syncthreads();
    if ((int)threadIdx.x < digits) {
      inside[threadIdx.x] = sums[1][warp] + own_all - here;
      place[threadIdx.x] = sums[0][warp] + all - total + before - inside[threadIdx.x];  // (of an entry's place in this CTA)
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kClusterEach; ++k) {
      if (k >= each || entry[k].x < 0) continue;
      const int d = entry[k].x >> shift & digits - 1;
      local[inside[d] + own[d] + at[k]] = entry[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < end - begin; i += kClusterThreads) {
      const int2 e = local[i];
      out[place[e.x >> shift & digits - 1] + i] = e;
      // (a token's entries are neighbours now in every CTA that has some)
      if (pass + 1 == p.passes) mark_first(local, i, p.rows);
    }
    tc::cluster_sync();  // (the entries are in place, the counts have been read)
  }
}

// ------------------------------------------------------------------ sums
struct SumP {
  const int2* entry;         // tokens and positions, sorted; padding (token V) stands at the end
  const uint32_t* rows;      // a bit for each row of dW: its token occurs
  const void* d_out;
  void* dweight;
  float* part;               // [runs][2][D]: 0 of a token that began before the run, 1 of one that goes on behind it
  int N, V, D, run, runs, adds;
  int zero_rows;             // rows from here on hold zeros already
  float scale;
};
template <typename OUT, bool V>
__device__ __forceinline__ void put_row(const SumP& p, int row, int c, int lane, int tpr, f2 (&acc)[4]) {
  OUT* to = static_cast<OUT*>(p.dweight) + (size_t)row * p.D;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = mul2(acc[i], dup2(p.scale));
  if (p.adds) {
    f2 old[4];
    load_cols<OUT, V>(to, c, lane, tpr, p.D, old);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = add2(old[i], acc[i]);
  }
  store_cols<OUT, V>(to, c, lane, tpr, p.D, acc);
}
// Blocks 0 .. ceil(runs / groups) - 1 add up the runs, those behind write zeros to the rows of tokens that do not occur.
constexpr int kZeroRows = 32;
template <typename IN, typename OUT, bool V>
__global__ void __launch_bounds__(256, V ? 4 : 2) embedding_bwd_kernel(SumP p, int tpr, int sum_blocks) {
  begin_dependent();
  const int groups = 256 / tpr, lane = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr;
  if ((int)blockIdx.x >= sum_blocks) {
    const int64_t word = blockIdx.x - sum_blocks, r0 = word * kZeroRows;
    const uint32_t there = p.rows[word];
    // (rows side by side in one piece, in which their own alignment has no part: 3000 tokens, 50000 words of 699 columns in bf16 43 us row
    // by row, 35 so)
    if (there == 0 && r0 + kZeroRows <= p.zero_rows) {
      char* at = static_cast<char*>(p.dweight) + (size_t)r0 * p.D * sizeof(OUT);
      fill_zeros(at, at + (size_t)kZeroRows * p.D * sizeof(OUT), threadIdx.x, 256);
      return;
    }
    f2 zero[4] = {0, 0, 0, 0};
    for (int r = group; r < kZeroRows; r += groups) {
      if (there >> r & 1u || r0 + r >= p.zero_rows) continue;
      OUT* to = static_cast<OUT*>(p.dweight) + (size_t)(r0 + r) * p.D;
      for (int c = 0; c < p.D; c += tpr * 8) store_cols<OUT, V>(to, c, lane, tpr, p.D, zero);
    }
    return;
  }
  // the runs' entries, the one in front and the one behind (-1: none)
  extern __shared__ int32_t entries[];  // [groups][run + 2] tokens, [groups][run] positions
  const int64_t begin = (int64_t)blockIdx.x * groups * p.run;
  for (int k = threadIdx.x; k < groups * (p.run + 2); k += 256) {
    const int64_t i = begin + (int64_t)(k / (p.run + 2)) * p.run + k % (p.run + 2) - 1;
    entries[k] = i >= 0 && i < p.N ? p.entry[i].x : -1;
  }
  for (int k = threadIdx.x; k < groups * p.run; k += 256) entries[groups * (p.run + 2) + k] = begin + k < p.N ? p.entry[begin + k].y : 0;
  __syncthreads();
  const int64_t run = (int64_t)blockIdx.x * groups + group, i0 = run * p.run;
  if (i0 >= p.N) return;
  const int n = (int)min((int64_t)p.run, p.N - i0);
  const int32_t *key = entries + group * (p.run + 2) + 1, *pos = entries + groups * (p.run + 2) + group * p.run;
  constexpr int R = sizeof(IN) == 4 ? 2 : 4;  // rows in a batch; the next batch is under way while one is added up
  for (int c = 0; c < p.D; c += tpr * 8) {
    f2 acc[4] = {0, 0, 0, 0};
    bool began = key[0] != key[-1];  // the token that is being added up began in this run
    Cols<IN, V> next[R];
    auto request = [&](int j0) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (j0 + j < n && key[j0 + j] < p.V) next[j].load(static_cast<const IN*>(p.d_out) + (size_t)pos[j0 + j] * p.D, c, lane, tpr, p.D);
    };
    request(0);
    for (int j0 = 0; j0 < n; j0 += R) {
      Cols<IN, V> e[R];
#pragma unroll
      for (int j = 0; j < R; ++j) e[j] = next[j];
      request(j0 + R);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int at = j0 + j;
        if (at >= n) break;
        const int k = key[at];
        if (k >= p.V) break;
        f2 row[4];
        e[j].get(row);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = add2(acc[i], row[i]);
        if (key[at + 1] == k && at + 1 < n) continue;
        // the token's last entry, or the run's
        if (began && key[at + 1] != k) put_row<OUT, V>(p, k, c, lane, tpr, acc);
        else store_cols<float, V>(p.part + ((size_t)run * 2 + (began ? 1 : 0)) * p.D, c, lane, tpr, p.D, acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = 0;
        began = true;
      }
    }
  }
}
// Tokens that lie in more than one run: the warp of the run where one begins adds up its partial rows in the order of the runs; those
// of a token in more than kLong runs are added by all warps of its block, each those of consecutive runs, then the warps' sums in
// order.  (A block's eight runs hold the beginning of one such token at most.)  grid (blocks of eight runs, pieces of 256 columns).
constexpr int kLong = 8;
template <bool V>
__device__ __forceinline__ void add_rows(const SumP& p, int from, int to, int c, int lane, f2 (&acc)[4]) {
  for (int r0 = from; r0 < to; r0 += 4) {
    Cols<float, V> e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r0 + j < to) e[j].load(p.part + (size_t)(r0 + j) * 2 * p.D, c, lane, 32, p.D);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r0 + j >= to) break;
      f2 row[4];
      e[j].get(row);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = add2(acc[i], row[i]);
    }
  }
}
template <typename OUT, bool V>
__global__ void __launch_bounds__(256) embedding_join_kernel(SumP p) {
  begin_dependent();
  __shared__ f2 sums[8][32][4];
  __shared__ int long_run, long_rows, long_tok;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, run = blockIdx.x * 8 + warp, c = blockIdx.y * 256;
  if (threadIdx.x == 0) long_run = -1;
  __syncthreads();
  const int64_t begin = (int64_t)run * p.run, end = begin + p.run;
  if (end < p.N) {
    const int tok = p.entry[end].x;
    const bool starts = tok < p.V && p.entry[end - 1].x == tok && !(run > 0 && p.entry[begin].x == tok && p.entry[begin - 1].x == tok);
    if (starts) {
      int lo = (int)end, hi = p.N;  // the first entry behind the token's
      if (end + p.run < p.N && p.entry[end + p.run].x != tok) hi = (int)end + p.run;
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (p.entry[mid].x <= tok) lo = mid + 1;
        else hi = mid;
      }
      const int n = (lo - 1) / p.run - run;  // partial rows besides the first
      if (n > kLong) {
        if (lane == 0) {
          long_run = run;
          long_rows = n;
          long_tok = tok;
        }
      } else {
        f2 acc[4];
        load_cols<float, V>(p.part + ((size_t)run * 2 + 1) * p.D, c, lane, 32, p.D, acc);
        add_rows<V>(p, run + 1, run + 1 + n, c, lane, acc);
        put_row<OUT, V>(p, tok, c, lane, 32, acc);
      }
    }
  }
  __syncthreads();
  if (long_run < 0) return;
  f2 acc[4] = {0, 0, 0, 0};
  if (warp == 0) load_cols<float, V>(p.part + ((size_t)long_run * 2 + 1) * p.D, c, lane, 32, p.D, acc);
  const int each = (long_rows + 7) / 8, from = long_run + 1 + warp * each, to = min(from + each, long_run + 1 + long_rows);
  add_rows<V>(p, from, to, c, lane, acc);
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[warp][lane][i] = acc[i];
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < 8; ++w)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = add2(acc[i], sums[w][lane][i]);
  put_row<OUT, V>(p, long_tok, c, lane, 32, acc);
}

// ------------------------------------------------------------------ host
static int threads_per_row(int D) {  // a power of two, 8 columns a thread, 4 to 256
  int t = 4;
  while (8 * t < D && t < 256) t *= 2;
  return t;
}
// Entries of a run: enough runs to give every SM eight blocks, 8 to 32 entries.
static int run_length(int64_t N, int D) {
  const int64_t groups = 256 / threads_per_row(D), want = N / (148 * 8 * groups);
  return (int)std::min<int64_t>(32, std::max<int64_t>(8, (want + 7) / 8 * 8));
}
struct Scratch {
  int2* entry[2];
  int32_t *hist, *total;
  uint32_t* rows;
  float* part;
  size_t bytes;
  int passes, bits, run, runs, tiles;
};
static Scratch carve(const mxb_embedding_desc* d, void* base) {
  Scratch s{};
  Carver c(round_base_up(base));  // (partial rows are written in pieces of 32 bytes)
  const int64_t N = d->tokens;
  int bits = 1;
  while ((int64_t)1 << bits <= d->V) ++bits;  // keys are 0 .. V
  s.passes = (bits + 9) / 10;
  s.bits = (bits + s.passes - 1) / s.passes;
  s.run = run_length(N, d->D);
  s.runs = (int)((N + s.run - 1) / s.run);
  s.tiles = (int)((N + kTile - 1) / kTile);
  for (int2*& e : s.entry) e = c.take<int2>(N);
  s.rows = c.take<uint32_t>((size_t)d->V / 32 + 1);
  s.hist = c.take<int32_t>(((size_t)1 << s.bits) * s.tiles);
  s.total = c.take<int32_t>((size_t)1 << s.bits);
  s.part = c.take<float>((size_t)s.runs * 2 * d->D);
  s.bytes = c.bytes() + kBaseRoom;
  return s;
}
template <typename F>
static void with_token(const mxb_embedding_desc* d, F&& f) {
  if (d->token_bytes == 8) f(int64_t{});
  else f(int32_t{});
}
template <typename F>
static void with_type(int32_t type, F&& f) {
  if (type == MXB_F32) f(float{});
  else f(bf16{});
}
}  // namespace embed

using namespace embed;

mxb_status embedding_fwd(const mxb_embedding_desc* d, const void* tokens, const void* weight, void* out, cudaStream_t st) {
  const FwdP p{tokens, weight, out, (size_t)d->tokens, d->V, d->D, d->scale};
  const int tpr = threads_per_row(d->D), groups = 256 / tpr;
  auto launch = [&](auto tok, auto in, auto o, auto rows, auto whole) {
    constexpr int R = decltype(rows)::value;
    const int64_t want = (d->tokens + groups * R - 1) / (groups * R);
    MXB_LAUNCH("embedding_fwd_kernel", st,
               (launch_kernel(embedding_fwd_kernel<decltype(tok), decltype(in), decltype(o), R, decltype(whole)::value>,
                              (unsigned)std::min<int64_t>(want, 148 * 8), 256, 0, st, p, tpr)));
  };
  const bool whole = whole_pieces(weight, d->io_dtype, d->D) && whole_pieces(out, d->out_dtype, d->D), many = d->tokens >= (int64_t)148 * 8 * groups;
  with_token(d, [&](auto tok) {
    with_type(d->io_dtype, [&](auto in) {
      with_type(d->out_dtype, [&](auto o) {
        auto rows = [&](auto w) {
          if (many) launch(tok, in, o, std::integral_constant<int, 4>{}, w);
          else launch(tok, in, o, std::integral_constant<int, 1>{}, w);
        };
        if (whole) rows(std::true_type{});
        else rows(std::false_type{});
      });
    });
  });
  return check_launch("embedding_fwd");
}

size_t embedding_bwd_scratch(const mxb_embedding_desc* d) { return carve(d, nullptr).bytes; }

mxb_status embedding_bwd(const mxb_embedding_desc* d, const void* tokens, const void* d_out, void* dweight, int adds, void* workspace,
                         cudaStream_t st) {
  const Scratch s = carve(d, workspace);
  int zero_rows = d->V;
  const int last = d->tokens <= kRankMost ? 0 : (s.passes - 1) & 1;  // where the sorted entries are
  if (d->tokens <= kRankMost) {
    const int64_t blocks = std::max<int64_t>((d->tokens + 31) / 32, std::min<int64_t>(148, d->V / (32 * 256) + 1));
    with_token(d, [&](auto tok) {
      MXB_LAUNCH("embedding_rank_kernel", st, (launch_kernel(embedding_rank_kernel<decltype(tok)>, (unsigned)blocks, 256, 0, st, tokens, s.entry[0], s.rows,
                                                             (int)d->tokens, d->V)));
    });
  } else if (d->tokens <= kClusterEntries) {
    // about four entries a thread
    int ctas = 1;
    while (ctas < kClusterMost && (int64_t)ctas * kClusterThreads * 4 < d->tokens) ctas *= 2;
    // The sort leaves most SMs idle: they write zeros to the last rows of dW meanwhile, those of the words that occur too - which a dW
    // smaller than that gets twice - and about as many bytes as fit beside it: 54 MB of 8192 tokens (the launch 28 us for 24 without), 117 of
    // 32768 (35 for 25), 201 of 65536 (55 for 37; all cold).  32768 rows of 2048 columns, 65536 words in float32: 138 us without, 134 with.
    const size_t row = (size_t)d->D * (d->out_dtype == MXB_F32 ? 4 : 2);
    if (!adds) zero_rows -= (int)std::min<size_t>(d->V, (((size_t)32 << 20) + (size_t)d->tokens * 2560) / row);
    char* dw = static_cast<char*>(dweight);
    const ClusterP q{tokens, {s.entry[0], s.entry[1]}, s.rows, (int)d->tokens, d->V, s.bits, s.passes, (int)((d->tokens + ctas - 1) / ctas), ctas,
                     dw + zero_rows * row, dw + d->V * row};
    mxb_status st_ = MXB_OK;
    with_token(d, [&](auto tok) {
      using TOK = decltype(tok);
      const int smem = q.share * (int)sizeof(int2) + (64 << s.bits);
      st_ = MXB_ALLOW_SMEM(kClusterThreads * kClusterEach * (int)sizeof(int2) + 64 * kMaxDigits, embedding_sort_kernel<TOK>);
      if (st_ != MXB_OK) return;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = zero_rows < d->V ? 144 / ctas * ctas : ctas;
      cfg.blockDim = kClusterThreads;
      cfg.dynamicSmemBytes = smem;
      cfg.stream = st;
      cudaLaunchAttribute attr[2] = {};
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = ctas;
      attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 2;
      MXB_LAUNCH("embedding_sort_kernel", st, (cudaLaunchKernelEx(&cfg, embedding_sort_kernel<TOK>, q)));
    });
    if (st_ != MXB_OK) return st_;
  } else {
    SortP q{tokens, nullptr, nullptr, s.hist, s.rows, (int)d->tokens, d->V, 0, 1 << s.bits, s.bits, s.tiles};
    for (int pass = 0; pass < s.passes; ++pass) {
      q.shift = pass * s.bits;
      q.out = s.entry[pass & 1];
      with_token(d, [&](auto tok) {
        using TOK = decltype(tok);
        MXB_LAUNCH("embedding_count_kernel", st, (launch_kernel(embedding_count_kernel<TOK>, s.tiles, kSortThreads, 0, st, q)));
        MXB_LAUNCH("embedding_scan_kernel", st, (launch_kernel(embedding_scan_kernel, 1 << s.bits, 256, 0, st, s.hist, s.total, s.tiles)));
        MXB_LAUNCH("embedding_place_kernel", st, (launch_kernel(embedding_place_kernel<TOK>, s.tiles, kSortThreads, 0, st, q, s.total)));
      });
      q.in = q.out;
    }
    MXB_LAUNCH("embedding_mark_kernel", st,
               (launch_kernel(embedding_mark_kernel, (unsigned)((d->tokens + 255) / 256), 256, 0, st, s.entry[last], (int)d->tokens, s.rows)));
  }
  const SumP p{s.entry[last], s.rows, d_out, dweight, s.part, (int)d->tokens, d->V, d->D, s.run, s.runs, adds, zero_rows, d->scale};
  const int tpr = threads_per_row(d->D), groups = 256 / tpr, sums = (s.runs + groups - 1) / groups;
  const int zeros = adds ? 0 : (int)(((int64_t)zero_rows + kZeroRows - 1) / kZeroRows);
  with_type(d->io_dtype, [&](auto in) {
    with_type(d->out_dtype, [&](auto o) {
      auto launch = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        MXB_LAUNCH("embedding_bwd_kernel", st,
                   (launch_kernel(embedding_bwd_kernel<decltype(in), decltype(o), W>, sums + zeros, 256, groups * (2 * s.run + 2) * sizeof(int32_t), st,
                                  p, tpr, sums)));
        if (s.runs > 1)
          MXB_LAUNCH("embedding_join_kernel", st,
                     (launch_kernel(embedding_join_kernel<decltype(o), W>, dim3((s.runs + 6) / 8, (d->D + 255) / 256), 256, 0, st, p)));
      };
      if (whole_pieces(d_out, d->io_dtype, d->D) && whole_pieces(dweight, d->out_dtype, d->D)) launch(std::true_type{});
      else launch(std::false_type{});
    });
  });
  return check_launch("embedding_bwd");
}

}  // namespace mxb
