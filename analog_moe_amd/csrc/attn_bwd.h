// Attention backward, with the probabilities made again from the scores and the forward pass's log-sums:
//   P = 2^(c s - lse),  dv = P^T go,  dP = go v^T,  dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q,
// delta = sum over the head of out * go.  One kernel owns rows of dq, one owns rows of dk and dv; each makes the scores for
// itself, seven products in all where five would do, and in return nothing is added up across workgroups: no atomics, no
// partial results in memory, and the same sums in the same order every time.
#pragma once
#include "attn_fwd.h"

namespace amoe {

// fp16 probabilities as operands, 2^15 times as large: no more than 2^15, and 2^-29 is still a normal number.
template <typename T> inline constexpr float kGradShift = kIsF16<T> ? 15.f : 0.f;

// A log-sum is rounded to a float, and so are all probabilities of its row off by up to half a step of it.  Rows whose log-sum is
// further from zero than kFar get theirs from a maximum and a sum made again: P = 2^((s - top) c - norm), with the maximum taken
// out before the multiplication and norm the logarithm of the sum.  Other rows: top 0, norm lse.
__device__ __forceinline__ bool attn_is_far(float lse, float limit) { return fabsf(lse) > limit && fabsf(lse) <= kMaxFloat; }

// top and norm of a wave's far rows, whose queries q holds: the keys they see once more, from memory
template <typename T, int DP, bool EDGE>
__device__ __forceinline__ void attn_far_rows(const AttnParams& p, const attn_frag<T> (&q)[DP / 16], const T* kb, int wave_sees, int seen,
                                              bool far, float& top, float& norm) {
  const int h = lane_id() >> 5;
  float m = -INFINITY, l = 0.f;
  for (int key0 = 0; key0 < wave_sees; key0 += 32) {
    attn_frag<T> kf[DP / 16];
    attn_row_frags<T, DP, EDGE>(kf, kb, p.k.ss, key0, wave_sees, p.d, p.vec);
    f32x16 s = f32x16_zero();
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++) s = attn_mma<T>(kf[kk], q[kk], s);
    float mx = m;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      if (key0 + 8 * (i / 4) + 4 * h + i % 4 >= seen) s[i] = -INFINITY;
      mx = fmaxf(mx, s[i]);
    }
    mx = attn_pair_max(mx);
    if (mx > m) l *= fast_exp2((m - mx) * p.c);
    m = mx;
#pragma unroll
    for (int i = 0; i < 16; i++) l += fast_exp2((s[i] - m) * p.c);
  }
  l = attn_pair_sum(l);
  if (far) {
    top = m;
    norm = fast_log2(l);
  }
}

// dS as matrix operands.  fp16 has no range for it: a gradient's size is the caller's, and where many keys share a row dS is
// tiny against what it sums up to.  So every column (a lane's query or key) carries a power of two that keeps its largest
// entry within fp16; it only falls, and the sums so far fall with it.  bf16 and fp32 need none.
template <typename T, int DP> struct AttnGrad {
  f32x16 acc[DP / 32];
  float scale;                        // of acc and of what is added next
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < DP / 32; t++) acc[t] = f32x16_zero();
    scale = kIsF16<T> ? 0x1p100f : 1.f;
  }
  template <class V> __device__ __forceinline__ void fit(V& ds) {       // 16 values
    if constexpr (kIsF16<T>) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) a = fmaxf(a, fabsf(ds[i]));
      a = attn_pair_max(a);
      const bool over = a * scale > 32768.f;
      if (wave_ballot(over) != 0) {
        // 2^14 / 2^ceil(log2 a), from a's exponent
        const float fit = over ? as_f32((uint32_t)(267 - (int)(as_u32(a) >> 23)) << 23) : scale;
        const float f = fit / scale;
#pragma unroll
        for (int t = 0; t < DP / 32; t++)
#pragma unroll
          for (int i = 0; i < 16; i++) acc[t][i] *= f;
        scale = fit;
      }
#pragma unroll
      for (int i = 0; i < 16; i++) ds[i] *= scale;
    }
  }
};

// a block's 16 values of a lane as two operands
template <typename T, class V>
__device__ __forceinline__ void attn_pack_block(const V& v, attn_frag<T> (&f)[2]) {
#pragma unroll
  for (int w = 0; w < 2; w++) {
    float half[8];
#pragma unroll
    for (int j = 0; j < 8; j++) half[j] = v[8 * w + j];
    f[w] = attn_pack<T>(half);
  }
}

// dq: 32 * RW queries of one head per workgroup, keys in tiles as in the forward pass; three products per block.  Also leaves
// norm, delta and top of every row.  Bound as the forward pass is: 8192 queries, 16 over 4 heads of 128, bf16, causal: 398 us,
// 1035 TFLOP/s; 16 x 1024, 16 heads of 64: 87 us.
template <typename T, int DP, bool EDGE, int RW, class Shape = AttnShape<T, DP, EDGE, RW>>
__global__ __launch_bounds__(kAttnThreads, (Shape::kWavesPerSimd)) void attn_bwd_q_kernel(AttnParams p) {
  using Tile = AttnTile<T, DP>;
  constexpr int KG = Shape::KG, BN = Shape::kKeys, NB = Shape::kBlocks, NK = DP / 16;
  constexpr int kElems = BN * DP, kTilesBytes = 2 * kElems * (int)sizeof(T);
  static_assert((KG - 1) * RW * DP * 32 * 4 <= kTilesBytes, "the copies are joined in the keys' tiles");
  __shared__ __align__(1024) char lds_k[kTilesBytes], lds_v[kTilesBytes];
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
  attn_frag<T> q[NK], go[NK];
  const bool real = w.i < p.S;
  const int64_t row = ((int64_t)w.b * p.S + w.i) * p.H + w.hd, stat = (int64_t)w.bh * p.S + w.i;
  attn_frag<T> o[NK], rest[NK];
  const int64_t out0 = ((int64_t)w.b * p.S * p.H + w.hd) * p.d, out_stride = (int64_t)p.H * p.d;
  attn_row_frags<T, DP, EDGE>(q, static_cast<const T*>(p.q.p) + w.b * p.q.sb + w.hd * p.q.sh, p.q.ss, w.w0, p.S, p.d, p.vec);
  attn_row_frags<T, DP, EDGE>(go, static_cast<const T*>(p.go.p) + w.b * p.go.sb + w.hd * p.go.sh, p.go.ss, w.w0, p.S, p.d, p.vec);
  attn_row_frags<T, DP, EDGE>(o, static_cast<const T*>(p.o) + out0, out_stride, w.w0, p.S, p.d, p.vec);
  if constexpr (sizeof(T) == 2)
    attn_row_frags<T, DP, EDGE>(rest, static_cast<const T*>(p.rest ? p.rest : p.o) + out0, out_stride, w.w0, p.rest ? p.S : 0, p.d, p.vec);
  float delta = 0.f;
#pragma unroll
  for (int kk = 0; kk < NK; kk++) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf(o[kk].v[j], go[kk].v[j], delta);
    } else {
      float ov[8], gv[8], rv[8];
      raw_unpack<T>(o[kk], ov);
      raw_unpack<T>(go[kk], gv);
      raw_unpack<T>(rest[kk], rv);
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf(ov[j] + rv[j], gv[j], delta);
    }
  }
  delta = attn_pair_sum(delta);
  float norm = real ? p.lse[stat] : INFINITY, top = 0.f;
  const bool far = attn_is_far(norm, kFar<T>), any_far = wave_ballot(far) != 0;
  if (any_far) attn_far_rows<T, DP, EDGE>(p, q, kb, w.wave_sees, w.seen, far, top, norm);
  if (real && h == 0 && w.kg == 0) {
    const int64_t n = (int64_t)p.B * p.H * p.S;
    p.rows[stat] = norm;
    p.rows[n + stat] = delta;
    p.rows[2 * n + stat] = top;
  }

  AttnGrad<T, DP> dq;
  dq.clear();
  if (n_tiles > 0) {
    sk.store(tid, tk);
    sv.store(tid, tv);
  }
  for (int t = 0; t < n_tiles; t++) {
    const int cur = (t & 1) * kElems, next = kElems - cur;
    sk.finish();
    __syncthreads();
    if (t + 1 < n_tiles) {
      sk.load(tid, tk + next, kb, p.k.ss, (t + 1) * BN, w.group_sees, p.d, p.vec);
      sv.load(tid, tv + next, vb, p.v.ss, (t + 1) * BN, w.group_sees, p.d, p.vec);
    }
    const int key0 = t * BN + 32 * NB * w.kg;
    if (key0 < w.wave_sees) {
      const typename Tile::Lane in = at.in(cur + 32 * NB * w.kg * DP);
      const bool mask = key0 + 32 * NB > w.wave_all;
      // per 32 keys: 2 * NK products for the scores and dP by turns, 2 * DP / 32 with dS
      constexpr int NU = DP / 32, NS = 2 * NK, NF = NS + 2 * NU;
      const auto load = [&](int x) -> attn_frag<T> {
        const int n = x / NF, e = x % NF;
        return e < NS ? Tile::row_frag(e & 1 ? lds_v : lds_k, in, 32 * n, e / 2) : Tile::col_frag(lds_k, in, 32 * n + 16 * ((e - NS) / NU), (e - NS) % NU);
      };
      AttnRun<T, NB * NF, sizeof(T) == 2 && DP == 128 ? 4 : kAttnAhead<T>> run;      // (more do not fit the registers)
      run.begin(load);
#pragma unroll
      for (int n = 0; n < NB; n++) {
        f32x16 s = f32x16_zero(), dp = f32x16_zero();
        run.steps(n * NF, n * NF + NS, load, [&](int x, const attn_frag<T>& a) {
          const int e = x % NF;
          if (e & 1) dp = attn_mma<T>(a, go[e / 2], dp);
          else s = attn_mma<T>(a, q[e / 2], s);
        });
        float ds[16];
#pragma unroll
        for (int e = 0; e < 16; e++) ds[e] = fast_exp2(fmaf(s[e], p.c, -norm)) * (dp[e] - delta);
        if (mask || any_far) {
          if (any_far) {
            // (the products once more, within the branch that there is: a branch of its own before the exponentials, or scores kept
            // for this one, cost every block more)
            s = dp = f32x16_zero();
#pragma unroll
            for (int kk = 0; kk < NK; kk++) {
              s = attn_mma<T>(Tile::row_frag(lds_k, in, 32 * n, kk), q[kk], s);
              dp = attn_mma<T>(Tile::row_frag(lds_v, in, 32 * n, kk), go[kk], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) ds[e] = fast_exp2(fmaf(s[e] - top, p.c, -norm)) * (dp[e] - delta);
          }
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (key0 + 32 * n + 8 * (e / 4) + 4 * h + e % 4 >= w.seen) ds[e] = 0.f;
        }
        dq.fit(ds);
        attn_frag<T> df[2];
        attn_pack_block<T>(ds, df);
        run.steps(n * NF + NS, n * NF + NF, load, [&](int x, const attn_frag<T>& a) {
          const int e = x % NF - NS;
          dq.acc[e % NU] = attn_mma<T>(a, df[e / NU], dq.acc[e % NU]);
        });
      }
    }
    if (t + 1 < n_tiles) {
      sk.store(tid, tk + next);
      sv.store(tid, tv + next);
    }
  }
  float factor = p.scale / dq.scale;
  if constexpr (KG > 1) {
    __syncthreads();
    f32x4* join = reinterpret_cast<f32x4*>(lds_k);
    if (w.kg > 0) attn_put_acc<DP>(join, (w.kg - 1) * RW + w.rw, dq.acc, factor);
    __syncthreads();
    if (w.kg == 0) {
#pragma unroll
      for (int t = 0; t < DP / 32; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) dq.acc[t][e] *= factor;
#pragma unroll
      for (int c = 1; c < KG; c++) attn_add_acc<DP>(join, (c - 1) * RW + w.rw, dq.acc, 1.f);
      factor = 1.f;
    }
  }
  if (w.kg == 0) attn_store_col<T, DP, EDGE>(static_cast<T*>(p.dq) + row * p.d, dq.acc, factor, p.d, real);
}

// dk, dv: KW waves hold 32 keys each of one key head, k and v as operands in registers or LDS, in QW copies; the queries of all heads
// that share them pass in tiles of 32 * QW, 32 for each copy, and the copies' sums are added at the end, in order.  Every wave
// reads what the other keys' waves read; more copies make shorter loops of the same work where there are few keys, and finer
// workgroups where causal rows differ in length.  Four products per block; heads of 128 are bound by registers (two waves on a
// SIMD with every one of them used, and operands no more than three reads ahead), heads of 64 by the vector work.  8192 keys, 16
// over 4 heads of 128, bf16, causal: 653 us, 840 TFLOP/s; 16 x 1024, 16 heads of 64: 122 us.  Measured and not kept there: the
// exponentials between the products of one wave (900 us), two workgroups of four waves on a CU (1000 us), the queries from the
// other end (no difference).
template <typename T, int DP, bool EDGE, int QW_> struct AttnKvShape {
  static constexpr int KW = 2, QW = QW_, kThreads = 64 * KW * QW;
  // k and v read from LDS for every product, for the registers that makes free.  16-bit heads past 96: v only, with dk, dv and k
  // the registers are full (both do not fit LDS).  Heads of 64, two copies: both, for a third workgroup on the CU (16 x 1024, 16 heads
  // of 64, bf16: 146 us with two; with three 122 us, and as much with k in registers).  Heads of 96 have room for
  // neither third workgroup nor more reads ahead: v there or not is the same (16 x 1024, 16 heads: dq, dk and dv 324 us), both 430.
  static constexpr bool kVInLds = sizeof(T) == 2 && !EDGE && (DP == 128 || (DP == 64 && QW == 2)), kKInLds = kVInLds && DP == 64;
  static constexpr int kWavesPerSimd = sizeof(T) * DP > 256 || EDGE ? 1 : kKInLds ? 3 : 2;       // fp32 heads past 64: 512 registers a wave
  static constexpr int kAhead = kKInLds ? 4 : kVInLds ? 3 : kAttnAhead<T>;                       // (more do not fit the registers)
  // two copies have room for two workgroups on a CU or three; four are one
  static constexpr bool kFits = 128 * QW * DP * (int)sizeof(T) <= (QW == 2 && !EDGE && sizeof(T) == 2 ? 48 : 128) << 10;
};
template <typename T, int DP, bool EDGE, int QW_, class Shape = AttnKvShape<T, DP, EDGE, QW_>>
__global__ __launch_bounds__((Shape::kThreads), (Shape::kWavesPerSimd)) void attn_bwd_kv_kernel(AttnParams p) {
  using Tile = AttnTile<T, DP>;
  constexpr int KW = Shape::KW, QW = Shape::QW, NT = Shape::kThreads, BM = 32 * QW, NK = DP / 16, NU = DP / 32;
  constexpr int kTileElems = BM * DP, kTilesBytes = 2 * kTileElems * (int)sizeof(T);
  constexpr int kSumsPer = kTilesBytes / (NU * 16 * 64 * 4);       // accumulators that fit a pair of tiles
  static_assert(KW * (QW - 1) <= 2 * kSumsPer, "the copies' sums fit the tiles' room");
  __shared__ __align__(1024) char lds_q[kTilesBytes], lds_g[kTilesBytes];
  __shared__ __align__(1024) char lds_k[Shape::kKInLds ? 32 * KW * DP * (int)sizeof(T) : 16], lds_v[Shape::kVInLds ? 32 * KW * DP * (int)sizeof(T) : 16];
  // norm, delta, top.  Scores here are those of the maximum to the last bit: the same products summed in the same order, whichever
  // of q and k is the first operand
  __shared__ __align__(16) float lds_rows[3][2][BM];
  T *const tq = reinterpret_cast<T*>(lds_q), *const tg = reinterpret_cast<T*>(lds_g);
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6), kw = wave % KW, qw = wave / KW, h = lane >> 5;
  const int BG = p.B * p.G, bg = (int)(blockIdx.x % (unsigned)BG), tile = (int)(blockIdx.x / (unsigned)BG);
  const int b = bg / p.G, g = bg - b * p.G;
  const int length = attn_length(p, b), start = attn_start(p, b);
  const int group0 = tile * 32 * KW, w0 = group0 + kw * 32, key = w0 + (lane & 31);
  const bool held = key < length;
  // queries from q_first on see the first key of the group; tiles of every head in turn
  int q_first = 0;
  if (p.causal && group0 > start) q_first = group0 - start < p.S ? group0 - start : p.S;
  if (group0 >= length) q_first = p.S;
  const int tile0 = q_first / BM, per_head = (p.S + BM - 1) / BM - tile0, n_tiles = q_first < p.S ? per_head * p.R : 0;

  AttnStage<T, DP, BM, NT, EDGE> sq, sg;
  sq.init(tid, p.q.ss, p.d);
  sg.init(tid, p.go.ss, p.d);
  static_assert(3 * BM <= NT && BM % 64 == 0, "a thread for each, whole waves");
  const int part = wave_uniform(tid / BM);            // threads 0 .. BM - 1: norm, the next BM: delta, the next: top
  float stat = 0.f;
  const auto fetch = [&](int t) {
    const int hd = g * p.R + t / per_head, q0 = (tile0 + t % per_head) * BM, buf = t & 1;
    sq.load(tid, tq + buf * kTileElems, static_cast<const T*>(p.q.p) + b * p.q.sb + hd * p.q.sh, p.q.ss, q0, p.S, p.d, p.vec);
    sg.load(tid, tg + buf * kTileElems, static_cast<const T*>(p.go.p) + b * p.go.sb + hd * p.go.sh, p.go.ss, q0, p.S, p.d, p.vec);
    if (part < 3) {
      const int qi = q0 + tid % BM;
      const int64_t row = (((int64_t)part * p.B + b) * p.H + hd) * p.S + qi;
      stat = qi < p.S ? p.rows[row] : part == 0 ? INFINITY : 0.f;
    }
  };
  const auto put = [&](int buf) {
    sq.store(tid, tq + buf * kTileElems);
    sg.store(tid, tg + buf * kTileElems);
    if (part < 3) lds_rows[part][buf][tid % BM] = stat;
  };
  if (n_tiles > 0) fetch(0);
  attn_frag<T> kf[NK], vf[NK];
  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.sb + g * p.k.sh;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.sb + g * p.v.sh;
  const int wave0 = w0 < length ? w0 : 0, wave_end = w0 < length ? length : 0;
  if constexpr (!Shape::kKInLds) attn_row_frags<T, DP, EDGE>(kf, kb, p.k.ss, wave0, wave_end, p.d, p.vec);
  if constexpr (!Shape::kVInLds) attn_row_frags<T, DP, EDGE>(vf, vb, p.v.ss, wave0, wave_end, p.d, p.vec);
  if constexpr (Shape::kVInLds) {
    // (only for tiles that come after: what is on its way into LDS is waited for there, and would else outlive the workgroup)
    if (n_tiles > 0) {
      const int all0 = group0 < length ? group0 : 0, all_end = group0 < length ? length : 0;
      AttnStage<T, DP, 32 * KW, NT, EDGE> st;
      if constexpr (Shape::kKInLds) {
        st.init(tid, p.k.ss, p.d);
        st.load(tid, reinterpret_cast<T*>(lds_k), kb, p.k.ss, all0, all_end, p.d, p.vec);
      }
      st.init(tid, p.v.ss, p.d);
      st.load(tid, reinterpret_cast<T*>(lds_v), vb, p.v.ss, all0, all_end, p.d, p.vec);
    }
  }
  AttnGrad<T, DP> dk, dv;
  dk.clear();
  dv.clear();
  typename Tile::Lane at;
  if (n_tiles > 0) put(0);
  for (int t = 0; t < n_tiles; t++) {
    const int q0 = (tile0 + t % per_head) * BM + 32 * qw, buf = t & 1;
    sq.finish();
    __syncthreads();
    if (t + 1 < n_tiles) fetch(t + 1);
    // the wave's keys are seen by some query of its block, and whether by every one
    if (w0 < length && q0 < p.S && (!p.causal || start + q0 + 32 > w0)) {
      const typename Tile::Lane in = at.in(buf * kTileElems + 32 * qw * DP);
      const bool mask = w0 + 32 > length || (p.causal && start + q0 < w0 + 31);
      // 2 * NK products for the scores and dP by turns, 4 * DP / 32 with P and dS by turns; for the former are read, step by step
      // of the head, q, k if it is in LDS, go, v if it is
      constexpr int kG = Shape::kKInLds ? 2 : 1, kPer = kG + (Shape::kVInLds ? 2 : 1), NS = kPer * NK, NF = NS + 4 * NU;
      const auto load = [&](int e) -> attn_frag<T> {
        if (e < NS) {
          const int kk = e / kPer, which = e % kPer;
          if (which == 0 || which == kG) return Tile::row_frag(which ? lds_g : lds_q, in, 0, kk);
          return Tile::row_frag(which < kG ? lds_k : lds_v, at, 32 * kw, kk);
        }
        const int r = e - NS;
        return Tile::col_frag(r & 1 ? lds_q : lds_g, in, 16 * (r / (2 * NU)), r / 2 % NU);
      };
      AttnRun<T, NF, Shape::kAhead> run;
      run.begin(load);
      f32x16 s = f32x16_zero(), dp = f32x16_zero();
      attn_frag<T> rows;                            // of q or go, for the product with what is read next
      run.steps(0, NS, load, [&](int e, const attn_frag<T>& a) {
        const int kk = e / kPer, which = e % kPer;
        if (which == 0) {
          if constexpr (Shape::kKInLds) rows = a;
          else s = attn_mma<T>(a, kf[kk], s);
        } else if (which < kG) {
          s = attn_mma<T>(rows, a, s);
        } else if (which == kG) {
          if constexpr (Shape::kVInLds) rows = a;
          else dp = attn_mma<T>(a, vf[kk], dp);
        } else {
          dp = attn_mma<T>(rows, a, dp);
        }
      });
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const f32x4 norm = *reinterpret_cast<const f32x4*>(&lds_rows[0][buf][32 * qw + 8 * u + 4 * h]);
        const f32x4 del = *reinterpret_cast<const f32x4*>(&lds_rows[1][buf][32 * qw + 8 * u + 4 * h]);
        const f32x4 top = *reinterpret_cast<const f32x4*>(&lds_rows[2][buf][32 * qw + 8 * u + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int e = 4 * u + j;
          s[e] = fast_exp2(fmaf(s[e] - top[j], p.c, kGradShift<T> - norm[j]));
          dp[e] = s[e] * (dp[e] - del[j]);
        }
      }
      if (mask) {
        // queries of the block before this one do not see the key
        const int hides = held ? (p.causal ? key - start - q0 - 4 * h : -32) : 32;
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (8 * (e / 4) + e % 4 < hides) s[e] = dp[e] = 0.f;
      }
      dk.fit(dp);
      attn_frag<T> pf[2], df[2];
      attn_pack_block<T>(s, pf);
      attn_pack_block<T>(dp, df);
      run.steps(NS, NF, load, [&](int e, const attn_frag<T>& a) {
        const int r = e - NS, w = r / (2 * NU), u = r / 2 % NU;
        if (r & 1) dk.acc[u] = attn_mma<T>(a, df[w], dk.acc[u]);
        else dv.acc[u] = attn_mma<T>(a, pf[w], dv.acc[u]);
      });
    }
    if (t + 1 < n_tiles) put(buf ^ 1);
  }
  // the copies' sums, in the layout of the registers: dv, then dk
  constexpr float kUnshift = kIsF16<T> ? 0x1p-15f : 1.f;
  const int64_t row = (((int64_t)b * p.T + key) * p.G + g) * p.d;
  const auto sums = [&](int slot) { return reinterpret_cast<f32x4*>(slot < kSumsPer ? lds_q : lds_g); };
#pragma unroll
  for (int which = 0; which < 2; which++) {
    f32x16(&acc)[NU] = which ? dk.acc : dv.acc;
    const float factor = which ? p.scale * kUnshift / dk.scale : kUnshift;
    __syncthreads();
    if (qw > 0) attn_put_acc<DP>(sums((qw - 1) * KW + kw), ((qw - 1) * KW + kw) % kSumsPer, acc, factor);
    __syncthreads();
    if (qw == 0) {
#pragma unroll
      for (int t = 0; t < NU; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[t][e] *= factor;
#pragma unroll
      for (int c = 0; c < QW - 1; c++) attn_add_acc<DP>(sums(c * KW + kw), (c * KW + kw) % kSumsPer, acc, 1.f);
      attn_store_col<T, DP, EDGE>(static_cast<T*>(which ? p.dk : p.dv) + row, acc, 1.f, p.d, key < p.T);
    }
  }
}

}  // namespace amoe
