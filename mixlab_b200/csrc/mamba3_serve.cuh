// Shared declarations of the Mamba-3 serving kernels: packed prompts and single tokens on a pool of recurrent states
// (mamba3_step.cu: one token; mamba3_walk.cu: prompts step by step, both layouts; mamba3_prompt.cu: prompts in chunks on the
// tensor cores).
#pragma once

#include "mamba3.cuh"

namespace mxb {

struct ServeP {
  int rows, S, slots;       // tokens of the call, sequences, rows of the state pool
  int D, N, G, NH, Kp, P;   // P: channels of a head (head layout)
  const void *x, *b, *c;
  const float *dt, *lam, *theta, *a_log;
  const int* cu;            // prompts: [S + 1] first rows; nullptr: one token a sequence
  const int* slot;          // [S] row of the pool, nullptr: the sequence's own number
  const unsigned char* go;  // prompts: [S] goes on from its state; nullptr: none does
  float* h;                 // [slots, D, N]
  float2* phase;            // [slots, NH] or [slots, D, Kp]: cosine and sine of the angle
  void *x_prev, *b_prev;    // [slots, D], [slots, NH or G, N]
  void* y;
  // prompts cut into segments of L steps; at most `pieces` segments, and fewer than `cuts` of sequences that have more than one
  // (what counts beyond belongs to lengths that add up to more than the rows, and is left)
  int L, pieces, cuts;
  float* ends;      // [cuts, D, N]: what a segment adds to the state, then the state that it starts from
  float* dsum;      // [cuts, NH or D]: sum of dt over the segment
  int* turn;        // [cuts, NH or D Kp]: angle of the segment in 2^-32 turns (channel layout: then the one that it starts at)
  float* ends2;     // [cuts, D, N]: what a segment adds by the sine of the angle that it starts at (channel layout)
  float* spoil;     // [cuts, D Kp]: NaN where the segment's angle is not finite, 0 elsewhere (channel layout)
  float2* start;    // [cuts, NH]: cosine and sine of the angle that the segment starts at (head layout)
  int slabs;        // head layout: CTAs that share a head's channels
  float2* phase_end;  // [S, NH]: with several slabs, the phase behind a sequence's last step (into the pool with its last row)
  // chunks on the tensor cores (mamba3_prompt.cu)
  int chunks;       // at most: ceil(length / 64) of every sequence
  float* scores;    // [chunks, G, 10 tiles, 2, 32 lanes, 8]
  float* rec;       // [chunks, NH, 512]: scalars of a chunk's steps
};

// Angles are summed as 32-bit fractions of a turn, whose additions do not round and wrap by themselves.  dt theta as such a
// fraction: the product and the division by 2 pi are carried out in two parts each, so that what is left is the rounding of dt.
__device__ __forceinline__ int m3_turn(float dt, float theta) {
  constexpr float kHi = 0.15915493667125702f, kLo = 6.420638243e-09f;  // 1 / (2 pi) in two floats
  const float p = dt * theta, pl = fmaf(dt, theta, -p);
  const float t = p * kHi, tl = fmaf(p, kHi, -t) + fmaf(p, kLo, pl * kHi);
  return __float2int_rn((t - rintf(t)) * 4294967296.f) + __float2int_rn(tl * 4294967296.f);
}
// A sum of 0 x: 0, or NaN where x is not finite - an angle that is not finite has to reach every later step.
__device__ __forceinline__ float m3_taint(float x, float sum) { return fmaf(x, 0.f, sum); }
__device__ __forceinline__ float2 m3_unit(int turn, float taint) {  // cosine, sine
  float s, c;
  sincospif((float)turn * 4.656612873077393e-10f, &s, &c);
  return make_float2(c + taint, s + taint);
}
__device__ __forceinline__ int serve_turn(float2 unit) { return __float2int_rn(atan2f(unit.y, unit.x) * 0.15915494309189535f * 4294967296.f); }
__device__ __forceinline__ float2 m3_back(float2 v, float2 a) {  // R^T: v turned back by the angle of a
  return make_float2(fmaf(a.x, v.x, a.y * v.y), fmaf(a.x, v.y, -a.y * v.x));
}
__device__ __forceinline__ float2 m3_on(float2 v, float2 a) {    // R: v turned on
  return make_float2(fmaf(a.x, v.x, -a.y * v.y), fmaf(a.x, v.y, a.y * v.x));
}
// The product of two unit vectors, of unit length again (one step of Newton's method for 1 / sqrt).
__device__ __forceinline__ float2 m3_turned(float2 u, float2 by) {
  const float2 r = m3_on(u, by);
  const float k = fmaf(-0.5f, fmaf(r.x, r.x, r.y * r.y), 1.5f);
  return make_float2(r.x * k, r.y * k);
}

// A segment of a sequence: rows [first, last) of the sequence [begin, end); `base` counts the segments of cut sequences in front of
// its own (what ends and the arrays beside it are numbered by), `chunk` is the number of its own first chunk of 64 steps.
struct Piece {
  int seq, seg, segs, base, first, last, begin, end, chunk;
  bool ok;
};
// The index-th piece: sequences one after the other, each cut every L rows; up to 32 sequences by falling length, so that the
// long ones do not start last (32 heads of 16 sequences of 440 to 4377 rows: a third off the time).  Called by whole warps, which
// look through 32 sequences at a time and add up those in front.  Whatever cu holds, rows stay inside the call's.
// kInner: the index-th of the pieces that are not their sequence's last (at most rows / L of them); kCut: the first piece of the
// index-th sequence that is cut.  SORT: false: sequences as they come (chunks are numbered so).
enum Find { kPieces, kInner, kCut };
template <Find WHAT = kPieces, bool SORT = true>
__device__ __forceinline__ Piece find_piece(const ServeP& p, int index, int L) {
  const int lane = threadIdx.x & 31;
  constexpr unsigned kAll = 0xffffffffu;
  auto scan = [&](int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kAll, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  auto wanted = [](int n) { return WHAT == kPieces ? n : WHAT == kInner ? max(n - 1, 0) : n > 1; };
  auto cut = [](int n) { return n > 1 ? n : 0; };
  Piece q{};
  int before = 0, base = 0, chunks = 0;  // wanted pieces, pieces of cut sequences, chunks in front
  for (int s0 = 0; s0 < p.S; s0 += 32) {
    const int s = s0 + lane;
    int a = 0, e = 0;
    if (s < p.S) {
      a = min(max(__ldg(p.cu + s), 0), p.rows);
      e = min(max(__ldg(p.cu + s + 1), a), p.rows);
    }
    int n = (int)(((unsigned)(e - a) + (unsigned)L - 1u) / (unsigned)L);
    const int cn = (e - a + 63) / 64, these = __reduce_add_sync(kAll, wanted(n));
    if (index >= before + these) {
      before += these;
      base += __reduce_add_sync(kAll, cut(n));
      chunks += __reduce_add_sync(kAll, cn);
      continue;
    }
    int id = s, chunk = chunks + scan(cn) - cn;
    if (SORT && p.S > 1 && p.S <= 32) {
      const int len = s < p.S ? e - a : -1;
      int rank = 0, from = 0;
#pragma unroll 8
      for (int j = 0; j < 32; ++j) {
        const int other = __shfl_sync(kAll, len, j);
        rank += other > len || (other == len && j < lane);
      }
#pragma unroll 8
      for (int j = 0; j < 32; ++j)
        if (__shfl_sync(kAll, rank, j) == lane) from = j;
      id = from;
      a = __shfl_sync(kAll, a, from);
      e = __shfl_sync(kAll, e, from);
      n = __shfl_sync(kAll, n, from);
      chunk = __shfl_sync(kAll, chunk, from);
    }
    const int cuts = scan(cut(n)), mine = scan(wanted(n));
    const int src = __ffs(__ballot_sync(kAll, before + mine > index)) - 1;
    q.seq = __shfl_sync(kAll, id, src);
    q.begin = __shfl_sync(kAll, a, src);
    q.end = __shfl_sync(kAll, e, src);
    q.segs = __shfl_sync(kAll, n, src);
    q.base = base + __shfl_sync(kAll, cuts - cut(n), src);
    q.seg = WHAT == kCut ? 0 : index - before - __shfl_sync(kAll, mine - wanted(n), src);
    q.first = q.begin + q.seg * L;
    q.last = (int)min((long long)q.first + L, (long long)q.end);
    q.chunk = __shfl_sync(kAll, chunk, src) + (q.first - q.begin) / 64;
    q.ok = true;
    return q;
  }
  return q;
}
// The sequence's row of the pool, -1 where it keeps no state.
__device__ __forceinline__ int serve_slot(const ServeP& p, int seq) {
  const int s = p.slot ? __ldg(p.slot + seq) : seq;
  return s >= 0 && s < p.slots ? s : -1;
}
__device__ __forceinline__ bool serve_goes_on(const ServeP& p, int seq) { return p.go && __ldg(p.go + seq); }

// (1 - lambda) dt of row t + 1, which weighs row t's outer product there; 0 behind the sequence's last row.
__device__ __forceinline__ float serve_look(const ServeP& p, size_t at, bool in) {
  return in ? (1.f - m3_sigmoid(__ldg(p.lam + at))) * m3_softplus(__ldg(p.dt + at)) : 0.f;
}

// Two neighbouring elements of a row (of b, c: N is even; a row may start at any element).
template <typename IO>
__device__ __forceinline__ float2 load_pair(const IO* p) { return make_float2(to_f32(p[0]), to_f32(p[1])); }

// The last row of a head into the pool: x of its channels, b of its group.  By a CTA that alone reads them.
template <typename IO>
__device__ __forceinline__ void serve_tail(const ServeP& p, int row, int slot, int hd, int g, int threads) {
  const IO *X = static_cast<const IO*>(p.x) + (size_t)row * p.D + (size_t)hd * p.P, *B = static_cast<const IO*>(p.b) + ((size_t)row * p.G + g) * p.N;
  IO *XP = static_cast<IO*>(p.x_prev) + (size_t)slot * p.D + (size_t)hd * p.P, *BP = static_cast<IO*>(p.b_prev) + ((size_t)slot * p.NH + hd) * p.N;
  for (int i = threadIdx.x; i < p.P; i += threads) XP[i] = X[i];
  for (int i = threadIdx.x; i < p.N; i += threads) BP[i] = B[i];
}

mxb_status m3serve_step(const ServeP& p, bool f32, cudaStream_t st);
bool m3prompt_supported(const ServeP& p, bool f32);
mxb_status m3prompt_prepare(const ServeP& p, cudaStream_t st);
mxb_status m3prompt_chunks(const ServeP& p, bool ends, cudaStream_t st);
size_t m3walk_scratch(ServeP& p, bool f32, int flags, char* base);
mxb_status m3walk_prefill(ServeP p, bool f32, int flags, cudaStream_t st);
mxb_status m3serve_tails(const ServeP& p, bool f32, bool x_too, cudaStream_t st);

}  // namespace mxb
