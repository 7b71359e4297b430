// Attention backward, with the probabilities made again from the scores and the forward pass's log-sums:
//   P = 2^(c s - lse),  dv = P^T go,  dP = go v^T,  dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q,
// delta = sum over the head of out * go.  One kernel owns rows of dq, one owns rows of dk and dv; each makes the scores for
// itself, seven products in all where five would do, and in return nothing is added up across workgroups: no atomics, no
// partial results in memory, and the same sums in the same order every time.
#pragma once
#include "attn_fwd.h"

namespace amoe {

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
  __device__ __forceinline__ void fit(float (&ds)[16]) {
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

// dq: 128 queries of one head per workgroup, 32 per wave, keys in tiles as in the forward pass.  Also leaves delta.
template <typename T, int DP, bool EDGE>
__global__ __launch_bounds__(kAttnThreads, sizeof(T) == 4 ? 1 : 2) void attn_bwd_q_kernel(AttnParams p) {
  using Tile = AttnTile<T, DP>;
  constexpr int BN = kAttnKeys<T>, NB = BN / 32, NK = DP / 16;
  __shared__ __align__(16) T lds_k[2][BN * DP];
  __shared__ __align__(16) T lds_v[2][BN * DP];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6), h = lane >> 5;
  const int BH = p.B * p.H, bh = (int)(blockIdx.x % (unsigned)BH), tile = (p.S + kAttnRows - 1) / kAttnRows - 1 - (int)(blockIdx.x / (unsigned)BH);
  const int b = bh / p.H, hd = bh - b * p.H, g = hd / p.R;
  const int length = attn_length(p, b), start = attn_start(p, b);
  const int w0 = tile * kAttnRows + wave * 32, i = w0 + (lane & 31);
  const int last = p.S - 1 < tile * kAttnRows + kAttnRows - 1 ? p.S - 1 : tile * kAttnRows + kAttnRows - 1;
  const int group_sees = attn_seen(p, length, start, last);
  const int wave_last = p.S - 1 < w0 + 31 ? p.S - 1 : w0 + 31;
  const int wave_sees = w0 < p.S ? attn_seen(p, length, start, wave_last) : 0;
  const int wave_all = w0 < p.S ? attn_seen(p, length, start, w0) : 0;
  const int seen = attn_seen(p, length, start, i < p.S ? i : p.S - 1);

  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.sb + g * p.k.sh;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.sb + g * p.v.sh;
  AttnStage<T, DP, BN, kAttnThreads, EDGE> sk, sv;
  sk.init(tid, p.k.ss, p.d);
  sv.init(tid, p.v.ss, p.d);
  const int n_tiles = (group_sees + BN - 1) / BN;
  if (n_tiles > 0) {
    sk.load(tid, kb, p.k.ss, 0, group_sees, p.d, p.vec);
    sv.load(tid, vb, p.v.ss, 0, group_sees, p.d, p.vec);
  }
  attn_frag<T> q[NK], go[NK];
  const int64_t row = ((int64_t)b * p.S + i) * p.H + hd;
  const T* qrow = static_cast<const T*>(p.q.p) + b * p.q.sb + hd * p.q.sh + (int64_t)i * p.q.ss;
  const T* grow = static_cast<const T*>(p.go.p) + b * p.go.sb + hd * p.go.sh + (int64_t)i * p.go.ss;
  const T* orow = static_cast<const T*>(p.o) + row * p.d;
  float delta = 0.f;
#pragma unroll
  for (int kk = 0; kk < NK; kk++) {
    q[kk] = attn_global_frag<T, EDGE>(qrow, kk, p.d, i < p.S, p.vec);
    go[kk] = attn_global_frag<T, EDGE>(grow, kk, p.d, i < p.S, p.vec);
    const attn_frag<T> o = attn_global_frag<T, EDGE>(orow, kk, p.d, i < p.S, p.vec);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf(o.v[j], go[kk].v[j], delta);
    } else {
      float ov[8], gv[8];
      raw_unpack<T>(o, ov);
      raw_unpack<T>(go[kk], gv);
#pragma unroll
      for (int j = 0; j < 8; j++) delta = fmaf(ov[j], gv[j], delta);
    }
  }
  delta = attn_pair_sum(delta);
  const float lse = i < p.S ? p.lse[(int64_t)bh * p.S + i] : INFINITY;
  if (i < p.S && h == 0) p.delta[(int64_t)bh * p.S + i] = delta;

  AttnGrad<T, DP> dq;
  dq.clear();
  if (n_tiles > 0) {
    sk.store(tid, lds_k[0]);
    sv.store(tid, lds_v[0]);
  }
  for (int t = 0; t < n_tiles; t++) {
    const int key0 = t * BN;
    __syncthreads();
    if (t + 1 < n_tiles) {
      sk.load(tid, kb, p.k.ss, key0 + BN, group_sees, p.d, p.vec);
      sv.load(tid, vb, p.v.ss, key0 + BN, group_sees, p.d, p.vec);
    }
    if (key0 < wave_sees) {
      const T *kt = lds_k[t & 1], *vt = lds_v[t & 1];
      const bool mask = key0 + BN > wave_all;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        f32x16 s = f32x16_zero(), dp = f32x16_zero();
#pragma unroll
        for (int kk = 0; kk < NK; kk++) {
          s = attn_mma<T>(Tile::row_frag(kt, 32 * n, kk), q[kk], s);
          dp = attn_mma<T>(Tile::row_frag(vt, 32 * n, kk), go[kk], dp);
        }
        float ds[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          ds[e] = fast_exp2(fmaf(s[e], p.c, -lse)) * (dp[e] - delta);
          if (mask && key0 + 32 * n + 8 * (e / 4) + 4 * h + e % 4 >= seen) ds[e] = 0.f;
        }
        dq.fit(ds);
#pragma unroll
        for (int w = 0; w < 2; w++) {
          float half[8];
#pragma unroll
          for (int j = 0; j < 8; j++) half[j] = ds[8 * w + j];
          const attn_frag<T> bf = attn_pack<T>(half);
#pragma unroll
          for (int u = 0; u < DP / 32; u++) dq.acc[u] = attn_mma<T>(Tile::col_frag(kt, 32 * n + 16 * w, u), bf, dq.acc[u]);
        }
      }
    }
    if (t + 1 < n_tiles) {
      sk.store(tid, lds_k[(t + 1) & 1]);
      sv.store(tid, lds_v[(t + 1) & 1]);
    }
  }
  if (i < p.S) attn_store_col<T, DP, EDGE>(static_cast<T*>(p.dq) + row * p.d, dq.acc, p.scale / dq.scale, p.d);
}

// dk, dv: 128 keys of one key head per workgroup, 32 per wave with their k and v as operands in registers; the queries of all
// heads that share them pass in tiles.
template <typename T, int DP, bool EDGE>
__global__ __launch_bounds__(kAttnThreads, 1) void attn_bwd_kv_kernel(AttnParams p) {
  using Tile = AttnTile<T, DP>;
  constexpr int BM = kAttnKeys<T>, NB = BM / 32, NK = DP / 16;
  __shared__ __align__(16) T lds_q[2][BM * DP];
  __shared__ __align__(16) T lds_g[2][BM * DP];
  __shared__ __align__(16) float lds_lse[2][BM], lds_delta[2][BM];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6), h = lane >> 5;
  const int BG = p.B * p.G, bg = (int)(blockIdx.x % (unsigned)BG), tile = (int)(blockIdx.x / (unsigned)BG);
  const int b = bg / p.G, g = bg - b * p.G;
  const int length = attn_length(p, b), start = attn_start(p, b);
  const int group0 = tile * kAttnRows, w0 = group0 + wave * 32, key = w0 + (lane & 31);
  const bool held = key < length;
  const T* krow = static_cast<const T*>(p.k.p) + b * p.k.sb + g * p.k.sh + (int64_t)key * p.k.ss;
  const T* vrow = static_cast<const T*>(p.v.p) + b * p.v.sb + g * p.v.sh + (int64_t)key * p.v.ss;
  attn_frag<T> kf[NK], vf[NK];
#pragma unroll
  for (int kk = 0; kk < NK; kk++) {
    kf[kk] = attn_global_frag<T, EDGE>(krow, kk, p.d, held, p.vec);
    vf[kk] = attn_global_frag<T, EDGE>(vrow, kk, p.d, held, p.vec);
  }
  // queries from q_first on see the first key of the group; tiles of every head in turn
  int q_first = 0;
  if (p.causal && group0 > start) q_first = group0 - start < p.S ? group0 - start : p.S;
  if (group0 >= length) q_first = p.S;
  const int tile0 = q_first / BM, per_head = (p.S + BM - 1) / BM - tile0, n_tiles = q_first < p.S ? per_head * p.R : 0;

  AttnStage<T, DP, BM, kAttnThreads, EDGE> sq, sg;
  sq.init(tid, p.q.ss, p.d);
  sg.init(tid, p.go.ss, p.d);
  float stat = 0.f;                                   // threads 0 .. BM - 1: lse, the next BM: delta
  const auto fetch = [&](int t) {
    const int hd = g * p.R + t / per_head, q0 = (tile0 + t % per_head) * BM;
    sq.load(tid, static_cast<const T*>(p.q.p) + b * p.q.sb + hd * p.q.sh, p.q.ss, q0, p.S, p.d, p.vec);
    sg.load(tid, static_cast<const T*>(p.go.p) + b * p.go.sb + hd * p.go.sh, p.go.ss, q0, p.S, p.d, p.vec);
    if (tid < 2 * BM) {
      const int qi = q0 + (tid < BM ? tid : tid - BM);
      const int64_t at = ((int64_t)b * p.H + hd) * p.S + qi;
      stat = qi < p.S ? (tid < BM ? p.lse[at] : p.delta[at]) : (tid < BM ? INFINITY : 0.f);
    }
  };
  const auto put = [&](int buf) {
    sq.store(tid, lds_q[buf]);
    sg.store(tid, lds_g[buf]);
    if (tid < BM) lds_lse[buf][tid] = stat;
    else if (tid < 2 * BM) lds_delta[buf][tid - BM] = stat;
  };
  AttnGrad<T, DP> dk, dv;
  dk.clear();
  dv.clear();
  if (n_tiles > 0) {
    fetch(0);
    put(0);
  }
  for (int t = 0; t < n_tiles; t++) {
    const int q0 = (tile0 + t % per_head) * BM, buf = t & 1;
    __syncthreads();
    if (t + 1 < n_tiles) fetch(t + 1);
    // the wave's keys are seen by some query of the tile, and whether by every one
    if (w0 < length && (!p.causal || start + q0 + BM > w0)) {
      const T *qt = lds_q[buf], *gt = lds_g[buf];
      const bool mask = w0 + 32 > length || (p.causal && start + q0 < w0 + 31);
#pragma unroll
      for (int n = 0; n < NB; n++) {
        f32x16 s = f32x16_zero(), dp = f32x16_zero();
#pragma unroll
        for (int kk = 0; kk < NK; kk++) {
          s = attn_mma<T>(Tile::row_frag(qt, 32 * n, kk), kf[kk], s);
          dp = attn_mma<T>(Tile::row_frag(gt, 32 * n, kk), vf[kk], dp);
        }
        float pr[16], ds[16];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const f32x4 lse = *reinterpret_cast<const f32x4*>(&lds_lse[buf][32 * n + 8 * u + 4 * h]);
          const f32x4 del = *reinterpret_cast<const f32x4*>(&lds_delta[buf][32 * n + 8 * u + 4 * h]);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int e = 4 * u + j;
            // (2^15 times P for fp16, as in the forward pass)
            pr[e] = fast_exp2(fmaf(s[e], p.c, kProbShift<T> - lse[j]));
            ds[e] = pr[e] * (dp[e] - del[j]);
            if (mask && (!held || (p.causal && key > start + q0 + 32 * n + 8 * u + 4 * h + j))) pr[e] = ds[e] = 0.f;
          }
        }
        dk.fit(ds);
#pragma unroll
        for (int w = 0; w < 2; w++) {
          float a[8], c[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            a[j] = pr[8 * w + j];
            c[j] = ds[8 * w + j];
          }
          const attn_frag<T> pf = attn_pack<T>(a), df = attn_pack<T>(c);
#pragma unroll
          for (int u = 0; u < DP / 32; u++) {
            dv.acc[u] = attn_mma<T>(Tile::col_frag(gt, 32 * n + 16 * w, u), pf, dv.acc[u]);
            dk.acc[u] = attn_mma<T>(Tile::col_frag(qt, 32 * n + 16 * w, u), df, dk.acc[u]);
          }
        }
      }
    }
    if (t + 1 < n_tiles) put(buf ^ 1);
  }
  if (key < p.T) {
    const int64_t row = (((int64_t)b * p.T + key) * p.G + g) * p.d;
    constexpr float kUnshift = kIsF16<T> ? 0x1p-15f : 1.f;
    attn_store_col<T, DP, EDGE>(static_cast<T*>(p.dv) + row, dv.acc, kUnshift, p.d);
    attn_store_col<T, DP, EDGE>(static_cast<T*>(p.dk) + row, dk.acc, p.scale * kUnshift / dk.scale, p.d);
  }
}

}  // namespace amoe
