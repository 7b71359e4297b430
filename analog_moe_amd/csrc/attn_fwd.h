// Attention forward: out = softmax(scale * q k^T + mask) v in one pass over the keys, with the running maximum and sum of every
// row; a row that sees no key gives zeros.
#pragma once
#include "attn_tile.h"
#include "wave_ops.h"

namespace amoe {

// A row's scores are kept as s * c in the exponent of 2.  The maximum that is taken out of them lags behind: it follows only when
// a larger one leaves it by more than 2^kMaxLag, which after a row's first keys it hardly ever does (following at every step
// costs a multiplication of the whole output state: 8192 queries of 16 heads of 128, bf16, 311 us, so 285 us); sums in fp32 and
// bf16 operands have the range for that.  fp16 probabilities are kept 2^7 times as large, which with the lag stays below 2^16:
// what is 2^-21 of a row's largest is still a normal number, where at 1 times a long row's tail below 2^-14 would lose bits
// that its sum counts.  The sum carries the same factor and the quotient none.
constexpr float kMaxLag = 8.f;
template <typename T> inline constexpr float kProbShift = kIsF16<T> ? 7.f : 0.f;

// A row's maximum is taken out within one multiply-add, s * c - rounded(m * c), so that all terms are off by the same factor, two to
// the rounding of m * c.  The quotient does not see it, but what is joined does: terms from before the maximum moved on, and those
// of other waves and parts, have factors of their own.  Maxima further from zero than this (half a step of it: 2^-18 in fp32,
// which the scores' own rounding is as large as; 2^-15 for 16-bit types, against 2^-9 or 2^-12 of a probability's rounding) are
// subtracted before the multiplication, where the largest score's difference is exactly 0.
template <typename T> inline constexpr float kFar = sizeof(T) == 4 ? 128.f : 1024.f;
constexpr float kMaxFloat = 3.402823466e38f;

// log2 of a row's sum: m * c, finite also where the product is not, and the logarithm of the sum l of 2^(shift + (s - m) c)
template <typename T>
__device__ __forceinline__ float attn_lse(float m, float l, float c) {
  if (l == 0.f) return INFINITY;
  return fminf(fmaxf(m * c, -kMaxFloat), kMaxFloat) + (fast_log2(l) - kProbShift<T>);
}

// State of a wave's 32 queries (a lane and its partner l ^ 32 hold one): output columns, running maximum, running sum of
// this lane's keys.
template <typename T, int DP> struct AttnState {
  f32x16 o[DP / 32];
  float m, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DP / 32; t++) o[t] = f32x16_zero();
    m = -INFINITY;
    l = 0.f;
  }
};

// The scores s of NB blocks of 32 keys from key0 on become probabilities, as operands pr of the product with v; `seen` is the
// number of keys the lane's query sees (from key 0).  In 16-bit types they are rounded to the type, which is what the matrix unit takes at
// its full rate: a result is then off by 0.0023 (bf16, relative, root of the mean square) or 0.00028 (fp16), where its own last rounding
// alone is 0.0017 and 0.00021; products in fp32 have a sixteenth of the rate.
template <typename T, int DP, int NB>
__device__ __forceinline__ void attn_softmax(AttnState<T, DP>& st, f32x16 (&s)[NB], attn_frag<T> (&pr)[2 * NB], int key0, int seen,
                                             bool mask, float c) {
  const int h = lane_id() >> 5;
  float mx = st.m;
  if (mask) {
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (key0 + 32 * n + 8 * (i / 4) + 4 * h + i % 4 >= seen) s[n][i] = -INFINITY;
  }
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[n][i]);
  mx = attn_pair_max(mx);
  // what was summed so far, in units of the new maximum
  const bool follow = (mx - st.m) * c > kMaxLag;             // (the first keys: from -inf)
  if (wave_ballot(follow) != 0) {
    const float f = follow ? fast_exp2((st.m - mx) * c) : 1.f;
    st.l *= f;
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) st.o[t][i] *= f;
    st.m = follow ? mx : st.m;
  }
  const float taken = st.m == -INFINITY ? 0.f : st.m;
  float base = taken * c;
  const bool far = fabsf(base) > kFar<T>;
  if (wave_ballot(far) != 0) {
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[n][i] -= far ? taken : 0.f;
    base = far ? 0.f : base;
  }
  base = kProbShift<T> - base;
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int w = 0; w < 2; w++) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] = fast_exp2(fmaf(s[n][8 * w + j], c, base));
      pr[2 * n + w] = attn_pack<T>(e);
      // (rounded, as the product with v counts them: else the rounding of a row's largest probability stays in the quotient, and
      // with it in delta, which all but cancels that key's dP; 160 tokens, heads of 64, bf16, scores to 5000: dq 2e-2 off, so 2e-3)
      sum = attn_add_packed<T>(pr[2 * n + w], sum);
    }
  st.l += sum;
}

// What the waves of a workgroup work on, for the kernels whose lanes own queries.
struct AttnRowsOf {
  int b, hd, g, bh, w0, i, rw, kg;   // w0: the wave's first query, i: the lane's
  int length, start;
  int group_sees;     // keys that the last query of the workgroup sees
  int wave_sees;      // the last one of the wave
  int wave_all;       // the first one of the wave
  int seen;           // the lane's
};
template <class Shape>
__device__ __forceinline__ AttnRowsOf attn_rows_of(const AttnParams& p) {
  AttnRowsOf w;
  const int wave = wave_uniform(threadIdx.x >> 6);
  w.rw = wave % Shape::RW;
  w.kg = wave / Shape::RW;
  // workgroups with one head next to each other's on an XCD (ids go round the eight); the longest rows first
  const int BH = p.B * p.H;
  w.bh = (int)(blockIdx.x % (unsigned)BH);
  const int row0 = ((p.S + Shape::kRows - 1) / Shape::kRows - 1 - (int)(blockIdx.x / (unsigned)BH)) * Shape::kRows;
  w.b = w.bh / p.H;
  w.hd = w.bh - w.b * p.H;
  w.g = w.hd / p.R;
  w.length = attn_length(p, w.b);
  w.start = attn_start(p, w.b);
  const int w0 = row0 + w.rw * 32, end = p.S - 1;
  w.w0 = w0;
  w.i = w0 + (lane_id() & 31);
  const int group_last = row0 + Shape::kRows - 1, wave_last = w0 + 31;
  w.group_sees = attn_seen(p, w.length, w.start, group_last < end ? group_last : end);
  w.wave_sees = w0 <= end ? attn_seen(p, w.length, w.start, wave_last < end ? wave_last : end) : 0;
  w.wave_all = w0 <= end ? attn_seen(p, w.length, w.start, w0) : 0;
  w.seen = attn_seen(p, w.length, w.start, w.i < end ? w.i : end);
  return w;
}
// a wave's accumulators to and from LDS, 16 bytes per lane and access: slot `copy` of as many as there are
template <int DP>
__device__ __forceinline__ void attn_put_acc(f32x4* lds, int copy, const f32x16 (&acc)[DP / 32], float factor) {
  const int lane = lane_id();
#pragma unroll
  for (int t = 0; t < DP / 32; t++)
#pragma unroll
    for (int u = 0; u < 4; u++)
      lds[((copy * (DP / 32) + t) * 4 + u) * 64 + lane] =
          f32x4{acc[t][4 * u] * factor, acc[t][4 * u + 1] * factor, acc[t][4 * u + 2] * factor, acc[t][4 * u + 3] * factor};
}
template <int DP>
__device__ __forceinline__ void attn_add_acc(const f32x4* lds, int copy, f32x16 (&acc)[DP / 32], float factor) {
  const int lane = lane_id();
#pragma unroll
  for (int t = 0; t < DP / 32; t++) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const f32x4 o = lds[((copy * (DP / 32) + t) * 4 + u) * 64 + lane];
#pragma unroll
      for (int j = 0; j < 4; j++) acc[t][4 * u + j] = fmaf(o[j], factor, acc[t][4 * u + j]);
    }
    sched_fence();          // (all the reads at once do not fit the registers)
  }
}

// Many rows: a workgroup has 32 * RW queries of one head and walks the keys in tiles that go straight from memory into LDS, two
// tiles by turns with one barrier each.  Two products of 32 x 32 x d per block of 32 keys on the matrix unit, 16 exponentials and
// about 55 other vector instructions a lane between them, which are the longer part for heads of 64; operands of one wave's
// 32 queries only, as 64 would leave one wave on a SIMD with nobody to fill its waits.  8192 queries, 16 over 4 heads of 128,
// bf16, causal: 285 us, 965 TFLOP/s where a library product of 8192^3 reaches 1375; 16 x 1024, 16 heads of 64: 70 us, half
// of it the time that q, k, v and the two results take to pass through memory.
// Heads past 96 take one block of keys at a time, and with operands no more than four reads ahead three workgroups fit a CU (8192
// queries as above: two blocks and two workgroups 298 us, one and two 288, one and three 285).  Times of kernels in these files are
// means of 20 launches in a trace; the least are 5 to 15 % shorter where launches in a row bring the clock down.
template <typename T, int DP, bool EDGE, int RW>
inline constexpr bool kAttnThree = sizeof(T) == 2 && DP == 128 && !EDGE && RW == 4;
template <typename T, int DP, bool EDGE, int RW, class Shape = AttnShape<T, DP, EDGE, RW>>
__global__ __launch_bounds__(kAttnThreads, (kAttnThree<T, DP, EDGE, RW> ? 3 : Shape::kWavesPerSimd)) void attn_fwd_rows_kernel(AttnParams p) {
  using Tile = AttnTile<T, DP>;
  constexpr int KG = Shape::KG, BN = Shape::kKeys, NB = Shape::kBlocks, NK = DP / 16;
  constexpr int kElems = BN * DP, kTilesBytes = 2 * kElems * (int)sizeof(T);
  static_assert((KG - 1) * RW * DP * 32 * 4 <= kTilesBytes, "the copies are joined in the keys' tiles");
  // (arrays of their own for keys and values also where one would do: see AttnTile's reads)
  __shared__ __align__(1024) char lds_k[kTilesBytes], lds_v[kTilesBytes];
  __shared__ float lds_ml[KG][RW][2][64];
  T *const tk = reinterpret_cast<T*>(lds_k), *const tv = reinterpret_cast<T*>(lds_v);
  const int tid = threadIdx.x, lane = lane_id(), h = lane >> 5;
  const AttnRowsOf w = attn_rows_of<Shape>(p);

  const T* kb = static_cast<const T*>(p.k.p) + w.b * p.k.sb + w.g * p.k.sh;
  const T* vb = static_cast<const T*>(p.v.p) + w.b * p.v.sb + w.g * p.v.sh;
  AttnStage<T, DP, BN, kAttnThreads, EDGE> sk, sv;
  sk.init(tid, p.k.ss, p.d);
  sv.init(tid, p.v.ss, p.d);
  typename Tile::Lane at;
  const int n_tiles = (w.group_sees + BN - 1) / BN;
  if (n_tiles > 0) {
    sk.load(tid, tk, kb, p.k.ss, 0, w.group_sees, p.d, p.vec);
    sv.load(tid, tv, vb, p.v.ss, 0, w.group_sees, p.d, p.vec);
  }
  attn_frag<T> q[NK];
  attn_row_frags<T, DP, EDGE>(q, static_cast<const T*>(p.q.p) + w.b * p.q.sb + w.hd * p.q.sh, p.q.ss, w.w0, p.S, p.d, p.vec);

  AttnState<T, DP> st;
  st.clear();
  if (n_tiles > 0) {
    sk.store(tid, tk);
    sv.store(tid, tv);
  }
  for (int t = 0; t < n_tiles; t++) {
    const int cur = (t & 1) * kElems, next = kElems - cur;
    sk.finish();
    __syncthreads();       // tile t is there, and nobody reads the other one any more
    if (t + 1 < n_tiles) {
      sk.load(tid, tk + next, kb, p.k.ss, (t + 1) * BN, w.group_sees, p.d, p.vec);
      sv.load(tid, tv + next, vb, p.v.ss, (t + 1) * BN, w.group_sees, p.d, p.vec);
    }
    const int key0 = t * BN + 32 * NB * w.kg;
    if (key0 < w.wave_sees) {
      // NB * NK products for the scores, 2 * NB * DP / 32 with the probabilities
      constexpr int NS = NB * NK, NU = DP / 32;
      const typename Tile::Lane in = at.in(cur + 32 * NB * w.kg * DP);
      const auto load = [&](int e) -> attn_frag<T> {
        return e < NS ? Tile::row_frag(lds_k, in, 32 * (e % NB), e / NB) : Tile::col_frag(lds_v, in, 16 * ((e - NS) / NU), (e - NS) % NU);
      };
      AttnRun<T, NS + 2 * NB * NU, kAttnThree<T, DP, EDGE, RW> ? 4 : kAttnAhead<T>> run;
      run.begin(load);
      f32x16 s[NB];
      attn_frag<T> pr[2 * NB];
#pragma unroll
      for (int n = 0; n < NB; n++) s[n] = f32x16_zero();
      run.steps(0, NS, load, [&](int e, const attn_frag<T>& a) { s[e % NB] = attn_mma<T>(a, q[e / NB], s[e % NB]); });
      attn_softmax<T, DP, NB>(st, s, pr, key0, w.seen, key0 + 32 * NB > w.wave_all, p.c);
      run.steps(NS, NS + 2 * NB * NU, load,
                [&](int e, const attn_frag<T>& a) { st.o[(e - NS) % NU] = attn_mma<T>(a, pr[(e - NS) / NU], st.o[(e - NS) % NU]); });
    }
    if (t + 1 < n_tiles) {
      sk.store(tid, tk + next);
      sv.store(tid, tv + next);
    }
  }
  float l = attn_pair_sum(st.l);
  if constexpr (KG > 1) {
    // the copies in units of the largest maximum; the first one takes the sums
    __syncthreads();
    f32x4* join = reinterpret_cast<f32x4*>(lds_k);
    lds_ml[w.kg][w.rw][0][lane] = st.m;
    lds_ml[w.kg][w.rw][1][lane] = l;
    if (w.kg > 0) attn_put_acc<DP>(join, (w.kg - 1) * RW + w.rw, st.o, 1.f);
    __syncthreads();
    if (w.kg == 0) {
      float m = st.m;
#pragma unroll
      for (int c = 1; c < KG; c++) m = fmaxf(m, lds_ml[c][w.rw][0][lane]);
      const float own = st.m == -INFINITY ? 0.f : fast_exp2((st.m - m) * p.c);
      l *= own;
#pragma unroll
      for (int t = 0; t < DP / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) st.o[t][e] *= own;
#pragma unroll
      for (int c = 1; c < KG; c++) {
        const float mc = lds_ml[c][w.rw][0][lane], f = mc == -INFINITY ? 0.f : fast_exp2((mc - m) * p.c);
        l = fmaf(lds_ml[c][w.rw][1][lane], f, l);
        attn_add_acc<DP>(join, (c - 1) * RW + w.rw, st.o, f);
      }
      st.m = m;
    }
  }
  if (w.kg == 0) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool real = w.i < p.S;
    const int64_t row = ((int64_t)w.b * p.S + w.i) * p.H + w.hd;
    attn_store_col<T, DP, EDGE>(static_cast<T*>(p.out) + row * p.d, st.o, inv, p.d, real);
    if (p.rest) attn_store_col<T, DP, EDGE, true>(static_cast<T*>(p.rest) + row * p.d, st.o, inv, p.d, real);
    if (p.lse && real && h == 0) p.lse[(int64_t)w.bh * p.S + w.i] = attn_lse<T>(st.m, l, p.c);
  }
}

// Few rows: the copies * R * S rows that share a key head, 32 per workgroup, and one of `splits` parts of the keys they see; every
// wave takes every fourth block of 32 keys of the part.  K goes from global memory into the operands, V through a tile of the
// wave's own, both a block ahead; the waves' results are joined in LDS, and those of the parts by attn_join_kernel.  Bound by
// memory: 48 sequences over caches of 4096 to 8192, 16 over 4 heads of 128, bf16: 133 us for 604 MB (4.5 TB/s, a large copy
// reaches 5.1); one over 131071 keys, 16 over 2 heads, fp16: 24 us for 134 MB (5.6 TB/s, part of it from the cache behind the
// L2), and 5 us for the join.
//
// LDS: two halves, of two waves each.
template <int DP> inline constexpr int kAttnSplitHalf = 2 * 32 * (DP + 4) * 4;
template <typename T, int DP, bool EDGE>
__device__ __forceinline__ void attn_split_body(const AttnParams& p, int id, char* lds_lo, char* lds_hi, float (*lds_m)[32], float (*lds_l)[32]) {
  using Tile = AttnTile<T, DP>;
  constexpr int NK = DP / 16, kRowF = DP + 4;     // floats between joined rows
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6), h = lane >> 5;
  const int rows = p.copies * p.R * p.S;
  const int bg = id % (p.B * p.G);
  id /= p.B * p.G;
  const int split = id % p.splits, r0 = (id / p.splits) * 32;
  const int b = bg / p.G, g = bg - b * p.G;
  const int length = attn_length(p, b), start = attn_start(p, b);
  // row r is query r % S of the group's head r / S, those of one sequence after those of another
  const int r = r0 + (lane & 31), rr = r < rows ? r : rows - 1, hd = g * p.R + rr / p.S % p.R, i = rr % p.S;
  const int seq0 = b * p.copies;
  const int seen = attn_seen(p, length, start, i);
  // keys that any row of the tile sees: with one head's rows in order it is the last row's, else the last query's
  const int r_last = r0 + 31 < rows ? r0 + 31 : rows - 1;
  const int tile_sees = attn_seen(p, length, start, r0 / p.S == r_last / p.S ? r_last % p.S : p.S - 1);
  const int per = ((tile_sees + p.splits - 1) / p.splits + 127) / 128 * 128;
  const int64_t lo64 = (int64_t)split * per;
  const int key_lo = lo64 < tile_sees ? (int)lo64 : tile_sees, key_hi = tile_sees - key_lo < per ? tile_sees : key_lo + per;

  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.sb + g * p.k.sh;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.sb + g * p.v.sh;
  char* const lds = wave < 2 ? lds_lo : lds_hi;
  T* tile = reinterpret_cast<T*>(lds) + (wave & 1) * 32 * DP;
  attn_frag<T> q[NK], kf[NK];
  const T* qrow = static_cast<const T*>(p.q.p) + (seq0 + rr / (p.R * p.S)) * p.q.sb + hd * p.q.sh + (int64_t)i * p.q.ss;
  AttnStage<T, DP, 32, 64, EDGE, true> sv;
  sv.init(lane, p.v.ss, p.d);
  const typename Tile::Lane at = typename Tile::Lane().in((wave & 1) * 32 * DP);
  const auto fetch = [&](int key0) {
    attn_row_frags<T, DP, EDGE>(kf, kb, p.k.ss, key0, key_hi, p.d, p.vec);
    sv.load(lane, nullptr, vb, p.v.ss, key0, key_hi, p.d, p.vec);
  };
  int key0 = key_lo + 32 * wave;
  if (key0 < key_hi) fetch(key0);
#pragma unroll
  for (int kk = 0; kk < NK; kk++) q[kk] = attn_global_frag<T, EDGE>(qrow, kk, p.d, r < rows, p.vec);
  AttnState<T, DP> st;
  st.clear();
  for (; key0 < key_hi; key0 += 128) {
    f32x16 s[1] = {f32x16_zero()};
#pragma unroll
    for (int kk = 0; kk < NK; kk++) s[0] = attn_mma<T>(kf[kk], q[kk], s[0]);
    wave_sync();           // the tile's last reads are done
    sv.store(lane, tile);
    wave_sync();
    if (key0 + 128 < key_hi) fetch(key0 + 128);
    attn_frag<T> pr[2];
    attn_softmax<T, DP, 1>(st, s, pr, key0, seen < key_hi ? seen : key_hi, true, p.c);
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int u = 0; u < DP / 32; u++) st.o[u] = attn_mma<T>(Tile::col_frag(lds, at, 16 * w, u), pr[w], st.o[u]);
  }

  // the four waves' rows in units of the largest maximum
  const float l = attn_pair_sum(st.l);
  if (h == 0) {
    lds_m[wave][lane] = st.m;
    lds_l[wave][lane] = l;
  }
  __syncthreads();
  float m = lds_m[0][lane & 31];
  for (int w = 1; w < 4; w++) m = fmaxf(m, lds_m[w][lane & 31]);
  const float f = st.m == -INFINITY ? 0.f : fast_exp2((st.m - m) * p.c);
  float* mine = reinterpret_cast<float*>(lds) + ((wave & 1) * 32 + (lane & 31)) * kRowF;
#pragma unroll
  for (int t = 0; t < DP / 32; t++)
#pragma unroll
    for (int u = 0; u < 4; u++) {
      f32x4 o = {st.o[t][4 * u] * f, st.o[t][4 * u + 1] * f, st.o[t][4 * u + 2] * f, st.o[t][4 * u + 3] * f};
      *reinterpret_cast<f32x4*>(mine + 32 * t + 8 * u + 4 * h) = o;
    }
  __syncthreads();
  constexpr int kPer = 32 * DP / 4 / kAttnThreads;     // four elements each
#pragma unroll
  for (int u = 0; u < kPer; u++) {
    const int idx = tid + u * kAttnThreads, row = idx / (DP / 4), e = idx % (DP / 4) * 4;
    if (r0 + row >= rows || e >= p.d) continue;
    float mr = lds_m[0][row], lr = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = 1; w < 4; w++) mr = fmaxf(mr, lds_m[w][row]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float mw = lds_m[w][row];
      lr += lds_l[w][row] * (mw == -INFINITY ? 0.f : fast_exp2((mw - mr) * p.c));
      const f32x4 o = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(w < 2 ? lds_lo : lds_hi) + ((w & 1) * 32 + row) * kRowF + e);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += o[j];
    }
    const int head = g * p.R + (r0 + row) / p.S % p.R, query = (r0 + row) % p.S;
    const int64_t seq = seq0 + (r0 + row) / (p.R * p.S), where = (seq * p.H + head) * p.S + query;
    if (p.part_o) {
      const int64_t part = (int64_t)split * p.B * p.copies * p.H * p.S + where;
      store4<float>(p.part_o + part * ((p.d + 3) & ~3) + e, v, 4, true);
      if (e == 0) {
        p.part_ml[2 * part] = mr;
        p.part_ml[2 * part + 1] = lr;
      }
    } else {
      const float inv = lr == 0.f ? 0.f : 1.f / lr;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] *= inv;
      const int64_t to = ((seq * p.S + query) * p.H + head) * p.d + e;
      store4<T>(static_cast<T*>(p.out) + to, v, EDGE ? p.d - e : 4, !EDGE);
      if (p.rest) {
        const float rest[4] = {attn_rest<T>(v[0]), attn_rest<T>(v[1]), attn_rest<T>(v[2]), attn_rest<T>(v[3])};
        store4<T>(static_cast<T*>(p.rest) + to, rest, EDGE ? p.d - e : 4, !EDGE);
      }
      if (p.lse && e == 0) p.lse[where] = attn_lse<T>(mr, lr, p.c);
    }
  }
}

template <typename T, int DP, bool EDGE>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 4 ? 1 : 2) void attn_fwd_split_kernel(AttnParams p) {
  __shared__ __align__(16) char lds_lo[kAttnSplitHalf<DP>], lds_hi[kAttnSplitHalf<DP>];
  __shared__ float lds_m[4][32], lds_l[4][32];
  attn_split_body<T, DP, EDGE>(p, (int)blockIdx.x, lds_lo, lds_hi, lds_m, lds_l);
}

// Rows that share keys, 32 * RW of them per workgroup, and one of `splits` parts of the keys they see: as attn_fwd_rows_kernel, for
// rows of several sequences and heads, whose results are joined with those of other parts.  Keys come from memory for the first
// time here: as many tiles as LDS has room for are on their way at once.
template <typename T, int DP, bool EDGE, int RW> struct AttnParts {
  static constexpr int KG = 4 / RW, kRows = 32 * RW;
  // (two blocks of keys where one is no whole number of chunks for every thread)
  static constexpr int kBlocks = KG == 1 && sizeof(T) == 2 && DP == 96 ? 2 : 1, BN = 32 * KG * kBlocks, kTile = BN * DP * (int)sizeof(T);
  // two workgroups on a CU
  static constexpr int kMost = (36 << 10) / kTile, kStages = EDGE || kMost < 3 ? 2 : kMost < 4 ? kMost : 4;
  static constexpr int kJoin = (KG - 1) * RW * DP * 32 * 4, kBytes = kStages * kTile > kJoin ? kStages * kTile : kJoin;
};
template <typename T, int DP, bool EDGE, int RW>
__device__ __forceinline__ void attn_parts_body(const AttnParams& p, int id, char* lds_k, char* lds_v, float (*lds_ml)[2][64]) {
  using Tile = AttnTile<T, DP>;
  using Shape = AttnParts<T, DP, EDGE, RW>;
  constexpr int KG = Shape::KG, BN = Shape::BN, NB = Shape::kBlocks, NK = DP / 16, kElems = BN * DP, kStages = Shape::kStages;
  T *const tk = reinterpret_cast<T*>(lds_k), *const tv = reinterpret_cast<T*>(lds_v);
  const int tid = threadIdx.x, lane = lane_id(), h = lane >> 5, wave = wave_uniform(tid >> 6), rw = wave % RW, kg = wave / RW;
  const int rows = p.copies * p.R * p.S, blocks = (rows + Shape::kRows - 1) / Shape::kRows, BG = p.B * p.G;
  const int r0 = id % blocks * Shape::kRows;
  id /= blocks;
  const int bg = id % BG, split = id / BG, b = bg / p.G, g = bg - b * p.G;
  const int length = attn_length(p, b), start = attn_start(p, b);
  const auto sees = [&](int first, int last) {       // keys that any of these rows sees: with one head's rows in order the last one's
    last = last < rows ? last : rows - 1;
    return first >= rows ? 0 : attn_seen(p, length, start, first / p.S == last / p.S ? last % p.S : p.S - 1);
  };
  const int group_sees = sees(r0, r0 + Shape::kRows - 1);
  const int per = ((group_sees + p.splits - 1) / p.splits + BN - 1) / BN * BN;
  const int64_t lo64 = (int64_t)split * per;
  const int key_lo = lo64 < group_sees ? (int)lo64 : group_sees, key_hi = group_sees - key_lo < per ? group_sees : key_lo + per;
  const int w0 = r0 + rw * 32, w1 = w0 + 31 < rows ? w0 + 31 : rows - 1;
  const int wave_sees = sees(w0, w0 + 31), wave_all = attn_seen(p, length, start, w0 < rows && w0 / p.S == w1 / p.S ? w0 % p.S : 0);
  const int r = w0 + (lane & 31), rr = r < rows ? r : rows - 1, hd = g * p.R + rr / p.S % p.R, i = rr % p.S;
  const int64_t seq = b * p.copies + rr / (p.R * p.S);
  const int all = attn_seen(p, length, start, i), seen = all < key_hi ? all : key_hi;

  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.sb + g * p.k.sh;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.sb + g * p.v.sh;
  AttnStage<T, DP, BN, kAttnThreads, EDGE> sk, sv;
  sk.init(tid, p.k.ss, p.d);
  sv.init(tid, p.v.ss, p.d);
  typename Tile::Lane at;
  const int n_tiles = (key_hi - key_lo + BN - 1) / BN;
  // tile t on its way to its place (past the last one: nothing is read, but it counts as asked for)
  const auto ask = [&](int t) __attribute__((always_inline)) {
    const int key = key_lo + t * BN, to = t % kStages * kElems;
    sk.load(tid, tk + to, kb, p.k.ss, key < key_hi ? key : key_hi, key_hi, p.d, p.vec);
    sv.load(tid, tv + to, vb, p.v.ss, key < key_hi ? key : key_hi, key_hi, p.d, p.vec);
  };
  attn_frag<T> q[NK];
  const T* qrow = static_cast<const T*>(p.q.p) + seq * p.q.sb + hd * p.q.sh + (int64_t)i * p.q.ss;
#pragma unroll
  for (int kk = 0; kk < NK; kk++) q[kk] = attn_global_frag<T, EDGE>(qrow, kk, p.d, r < rows, p.vec);

  AttnState<T, DP> st;
  st.clear();
  if constexpr (EDGE) {
    if (n_tiles > 0) {
      ask(0);
      sk.store(tid, tk);
      sv.store(tid, tv);
    }
  } else {
#pragma unroll
    for (int t = 0; t < kStages - 1; t++) ask(t);
  }
  for (int t = 0; t < n_tiles; t++) {
    const int cur = t % kStages * kElems;
    if constexpr (EDGE) {
      __syncthreads();     // tile t is there, and nobody reads the other one any more
      if (t + 1 < n_tiles) ask(t + 1);
    } else {
      lds_dma_wait_but<(kStages - 2) * 2 * decltype(sk)::kN>();
      __syncthreads();     // tile t is there, and nobody reads the one before any more
      ask(t + kStages - 1);
    }
    const int key0 = key_lo + t * BN + 32 * NB * kg;
    if (key0 < wave_sees && key0 < key_hi) {
      constexpr int NS = NB * NK, NU = DP / 32;
      const typename Tile::Lane in = at.in(cur + 32 * NB * kg * DP);
      const auto load = [&](int e) -> attn_frag<T> {
        return e < NS ? Tile::row_frag(lds_k, in, 32 * (e % NB), e / NB) : Tile::col_frag(lds_v, in, 16 * ((e - NS) / NU), (e - NS) % NU);
      };
      AttnRun<T, NS + 2 * NB * NU> run;
      run.begin(load);
      f32x16 s[NB];
      attn_frag<T> pr[2 * NB];
#pragma unroll
      for (int n = 0; n < NB; n++) s[n] = f32x16_zero();
      run.steps(0, NS, load, [&](int e, const attn_frag<T>& a) { s[e % NB] = attn_mma<T>(a, q[e / NB], s[e % NB]); });
      attn_softmax<T, DP, NB>(st, s, pr, key0, seen, key0 + 32 * NB > wave_all || key0 + 32 * NB > key_hi, p.c);
      run.steps(NS, NS + 2 * NB * NU, load,
                [&](int e, const attn_frag<T>& a) { st.o[(e - NS) % NU] = attn_mma<T>(a, pr[(e - NS) / NU], st.o[(e - NS) % NU]); });
    }
    if constexpr (EDGE) {
      if (t + 1 < n_tiles) {
        const int next = (t + 1) % kStages * kElems;
        sk.store(tid, tk + next);
        sv.store(tid, tv + next);
      }
    }
  }
  if constexpr (!EDGE) lds_dma_wait();     // (what was asked for past the last tile)
  float l = attn_pair_sum(st.l);
  if constexpr (KG > 1) {
    // the copies in units of the largest maximum; the first one takes the sums
    __syncthreads();
    f32x4* join = reinterpret_cast<f32x4*>(lds_k);
    lds_ml[kg * RW + rw][0][lane] = st.m;
    lds_ml[kg * RW + rw][1][lane] = l;
    if (kg > 0) attn_put_acc<DP>(join, (kg - 1) * RW + rw, st.o, 1.f);
    __syncthreads();
    if (kg == 0) {
      float m = st.m;
#pragma unroll
      for (int c = 1; c < KG; c++) m = fmaxf(m, lds_ml[c * RW + rw][0][lane]);
      const float own = st.m == -INFINITY ? 0.f : fast_exp2((st.m - m) * p.c);
      l *= own;
#pragma unroll
      for (int t = 0; t < DP / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) st.o[t][e] *= own;
#pragma unroll
      for (int c = 1; c < KG; c++) {
        const float mc = lds_ml[c * RW + rw][0][lane], f = mc == -INFINITY ? 0.f : fast_exp2((mc - m) * p.c);
        l = fmaf(lds_ml[c * RW + rw][1][lane], f, l);
        attn_add_acc<DP>(join, (c - 1) * RW + rw, st.o, f);
      }
      st.m = m;
    }
  }
  if (kg == 0 && r < rows) {
    const int64_t part = (int64_t)split * p.B * p.copies * p.H * p.S + (seq * p.H + hd) * p.S + i;
    float* po = p.part_o + part * ((p.d + 3) & ~3);
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int e = 32 * t + 8 * u + 4 * h;
        if (e < p.d) *reinterpret_cast<f32x4*>(po + e) = f32x4{st.o[t][4 * u], st.o[t][4 * u + 1], st.o[t][4 * u + 2], st.o[t][4 * u + 3]};
      }
    if (h == 0) {
      p.part_ml[2 * part] = st.m;
      p.part_ml[2 * part + 1] = l;
    }
  }
}

// Parts of a prefix and of the sequences' own keys in one launch: the first kind waits for the matrix unit, the second for memory.
// RWP, RWO: rows of a workgroup of either kind (32 times this; 0: attn_split_body).  Ids go round the eight XCDs; each of them
// has its run of both kinds, next to each other what reads the same keys.  The longer ones of the prefix go first, one to a CU, and the
// others beside them (four prefixes of 8192, 64 sequences each, 32 over 8 heads of 128, bf16: 125 us, 161 where the kinds are mixed in
// proportion and the last ones of the prefix start late; 175 as two launches).
struct AttnSharedParams {
  AttnParams prefix, own;
  int n_prefix, n_own;               // workgroups
};
template <typename T, int DP, bool EDGE, int RWP, int RWO>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 4 ? 1 : 2) void attn_shared_kernel(AttnSharedParams p) {
  constexpr int kSplit = RWP == 0 || RWO == 0 ? kAttnSplitHalf<DP> : 0;
  constexpr int kPrefix = RWP ? AttnParts<T, DP, EDGE, RWP ? RWP : 4>::kBytes : 0, kOwn = RWO ? AttnParts<T, DP, EDGE, RWO ? RWO : 4>::kBytes : 0;
  constexpr int kParts = kPrefix > kOwn ? kPrefix : kOwn, kHalf = kSplit > kParts ? kSplit : kParts;
  __shared__ __align__(1024) char lds_lo[kHalf], lds_hi[kHalf];
  __shared__ float lds_ml[4][2][64];
  const auto split = [&](const AttnParams& a, int id) __attribute__((always_inline)) {
    attn_split_body<T, DP, EDGE>(a, id, lds_lo, lds_hi, reinterpret_cast<float(*)[32]>(lds_ml), reinterpret_cast<float(*)[32]>(lds_ml) + 8);
  };
  const int xcd = (int)(blockIdx.x % 8), slot = (int)(blockIdx.x / 8), each_p = (p.n_prefix + 7) / 8, each_o = (p.n_own + 7) / 8;
  if (slot < each_p) {
    const int id = xcd * each_p + slot;
    if (id >= p.n_prefix) return;
    if constexpr (RWP == 0) split(p.prefix, id);
    else attn_parts_body<T, DP, EDGE, RWP>(p.prefix, id, lds_lo, lds_hi, lds_ml);
  } else {
    const int id = xcd * each_o + slot - each_p;
    if (id >= p.n_own) return;
    if constexpr (RWO == 0) split(p.own, id);
    else attn_parts_body<T, DP, EDGE, RWO>(p.own, id, lds_lo, lds_hi, lds_ml);
  }
}

// The parts of a row joined, RW waves per row, for up to 128 of them: a lane holds two parts' maxima and sums, then two elements of the
// row.  (Parts in which a row sees nothing are zeros: a branch round them would make every read wait for the one before.)
template <typename T, int RW>
__global__ __launch_bounds__(kAttnThreads) void attn_join_rows_kernel(AttnParams p) {
  __shared__ float lds[4][2][64];
  const int64_t n = (int64_t)p.B * p.H * p.S, row0 = (int64_t)blockIdx.x * (4 / RW) + (threadIdx.x >> 6) / RW;
  const int64_t at = row0 < n ? row0 : n - 1;
  const int lane = lane_id(), pad = (p.d + 3) & ~3, wave = wave_uniform(threadIdx.x >> 6);
  float m[2], l[2], f[2];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int s = lane + 64 * u;
    m[u] = s < p.splits ? p.part_ml[2 * (s * n + at)] : -INFINITY;
    l[u] = s < p.splits ? p.part_ml[2 * (s * n + at) + 1] : 0.f;
  }
  const float top = wave_largest(fmaxf(m[0], m[1]));
#pragma unroll
  for (int u = 0; u < 2; u++) f[u] = m[u] == -INFINITY ? 0.f : fast_exp2((m[u] - top) * p.c);
  const float sum = lanes_sum(fmaf(l[1], f[1], l[0] * f[0])), inv = sum == 0.f ? 0.f : 1.f / sum;
  const int e = 2 * lane, e_in = e < p.d ? e : 0;
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int end = p.splits - 64 * u < 64 ? p.splits - 64 * u : 64;
#pragma unroll 8
    for (int s = wave % RW; s < end; s += RW) {
      const float fs = as_f32(wave_read(as_u32(f[u]), s));
      const float* po = p.part_o + ((s + 64 * u) * n + at) * pad + e_in;
      a = fmaf(po[0], fs, a);
      b = fmaf(po[1], fs, b);
    }
  }
  if constexpr (RW > 1) {
    lds[wave][0][lane] = a;
    lds[wave][1][lane] = b;
    __syncthreads();
    if (wave % RW) return;
#pragma unroll
    for (int w = 1; w < RW; w++) {
      a += lds[wave + w][0][lane];
      b += lds[wave + w][1][lane];
    }
  }
  const int64_t bh = at / p.S, i = at - bh * p.S, seq = bh / p.H, hd = bh - seq * p.H;
  T* out = static_cast<T*>(p.out) + ((seq * p.S + i) * p.H + hd) * p.d;
  if (row0 < n && e < p.d) out[e] = Elem<T>::cvt(a * inv);
  if (row0 < n && e + 1 < p.d) out[e + 1] = Elem<T>::cvt(b * inv);
}

// The parts of a row joined, a workgroup per row: sums in units of the largest maximum, eight runs of parts side by side and
// then those in order.
template <typename T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(AttnParams p) {
  __shared__ float lds_f[kAttnMaxSplits], lds_red[8];
  __shared__ __align__(16) f32x4 lds_o[8][32];
  const int64_t n = (int64_t)p.B * p.H * p.S, at = blockIdx.x;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, row_units = (p.d + 3) / 4;
  float m = -INFINITY;
  for (int s = tid; s < p.splits; s += kAttnThreads) m = fmaxf(m, p.part_ml[2 * (s * n + at)]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, wave_shfl_xor(m, x));
  if (lane == 0) lds_red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(lds_red[0], lds_red[1]), fmaxf(lds_red[2], lds_red[3]));
  float l = 0.f;
  for (int s = tid; s < p.splits; s += kAttnThreads) {
    const float ms = p.part_ml[2 * (s * n + at)];
    const float f = ms == -INFINITY ? 0.f : fast_exp2((ms - m) * p.c);
    lds_f[s] = f;
    l += p.part_ml[2 * (s * n + at) + 1] * f;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += wave_shfl_xor(l, x);
  if (lane == 0) lds_red[4 + wave] = l;
  __syncthreads();
  l = (lds_red[4] + lds_red[5]) + (lds_red[6] + lds_red[7]);
  const int unit = tid & 31, run = tid >> 5;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (unit < row_units) {
    const f32x4* po = reinterpret_cast<const f32x4*>(p.part_o) + at * row_units + unit;
#pragma unroll 8
    for (int s = run; s < p.splits; s += 8) {
      const f32x4 v = po[s * n * row_units];
      const float f = lds_f[s];
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = fmaf(v[j], f, o[j]);
    }
  }
  lds_o[run][unit] = o;
  __syncthreads();
  const int64_t bh = at / p.S, i = at - bh * p.S, b = bh / p.H, hd = bh - b * p.H;
  const int64_t to = ((b * p.S + i) * p.H + hd) * p.d;
  if (tid < p.d) {
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < 8; r++) v += lds_o[r][tid >> 2][tid & 3];
    v *= l == 0.f ? 0.f : 1.f / l;
    static_cast<T*>(p.out)[to + tid] = Elem<T>::cvt(v);
    if (p.rest) static_cast<T*>(p.rest)[to + tid] = Elem<T>::cvt(attn_rest<T>(v));
  }
  if (p.lse && tid == 0) p.lse[at] = attn_lse<T>(m, l, p.c);
}

}  // namespace amoe
