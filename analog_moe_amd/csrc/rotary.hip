// Rotary positions: the first R elements of every head are R / 2 pairs, and pair i turns by position * turns[i].
//   (a, b) -> size * (a cos - b sin, b cos + a sin);   the rest of the head is copied.
//
// turns[i] is the fraction of a revolution per position times 2^64, so that the angle is the low 64 bits of an integer product:
// exact for any position, where 32-bit floats lose the angle of far ones.  q and k go in one launch.  Bound by memory: every
// element is read and written once, in 16-byte chunks; a token's sines and cosines are made once per workgroup, in LDS.  16 x 1024
// tokens, 32 heads of 64, bf16: 26.7 us for 134 MB (5.0 TB/s, a large copy reaches 5.1); 50001 tokens, 20 heads of 128, half of
// each turned, fp16: 116 us for 512 MB (4.4 TB/s).
#include <amoe.h>

#include "host_util.h"

namespace amoe {

struct RotaryPart {              // [B, S, heads, d] with these strides (elements)
  const void* in;
  void* out;
  int64_t in_sb, in_ss, in_sh, out_sb, out_ss, out_sh;
  int heads;
};
struct RotaryParams {
  RotaryPart part[2];
  const int64_t* turns;
  const void* pos;               // int32 / int64 with these strides, or null: pos_start + s
  int64_t pos_sb, pos_ss, pos_start;
  int pos_i64;
  int64_t tokens;                // B * S
  int S, d, R, interleaved, tokens_per_group;
  float size, sign;              // sign -1: the other way round (the gradient)
};

constexpr int kRotaryPairs = 1024;      // cosines and sines a workgroup holds

// V: elements per access, 1 or a 16-byte chunk.  A unit of work is V pairs (halves) or V / 2 pairs (interleaved; one pair for
// V == 1) of one head, or V elements behind the turned ones.
template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  __shared__ float lds_cos[kRotaryPairs], lds_sin[kRotaryPairs];
  const int tid = threadIdx.x, half = p.R / 2;
  const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_group;
  const int tokens = (int)(p.tokens - token0 < p.tokens_per_group ? p.tokens - token0 : p.tokens_per_group);
  for (int j = tid; j < tokens * half; j += 256) {
    const int t = j / half;
    const int64_t token = token0 + t, b = token / p.S, s = token - b * p.S;
    int64_t pos = p.pos_start + s;
    if (p.pos) {
      const int64_t at = b * p.pos_sb + s * p.pos_ss;
      pos = p.pos_i64 ? static_cast<const int64_t*>(p.pos)[at] : static_cast<const int32_t*>(p.pos)[at];
    }
    const uint64_t angle = (uint64_t)pos * (uint64_t)p.turns[j - t * half];
    float sn, cs;
    sincos_half_turns((float)(int32_t)(angle >> 32) * 0x1p-31f, &sn, &cs);
    lds_cos[j] = cs * p.size;
    lds_sin[j] = sn * p.size * p.sign;
  }
  __syncthreads();
  const int pair_units = p.interleaved ? (V == 1 ? half : p.R / V) : half / V;
  const int units = pair_units + (p.d - p.R) / V, heads = p.part[0].heads + p.part[1].heads;
  const int per_token = units * heads;
  struct Item {
    T* out;
    const float *cs, *sn;
    int u;
    Raw a, c;
    float x, y;
  };
  const auto fetch = [&](int j, Item& it) {
    const int t = j / per_token, hu = j - t * per_token, hd = hu / units, u = hu - hd * units;
    const int64_t token = token0 + t, b = token / p.S, s = token - b * p.S;
    const RotaryPart& part = p.part[hd < p.part[0].heads ? 0 : 1];
    const int head = hd < p.part[0].heads ? hd : hd - p.part[0].heads;
    const T* in = static_cast<const T*>(part.in) + b * part.in_sb + s * part.in_ss + head * part.in_sh;
    it.out = static_cast<T*>(part.out) + b * part.out_sb + s * part.out_ss + head * part.out_sh;
    it.cs = lds_cos + t * half;
    it.sn = lds_sin + t * half;
    it.u = u;
    if constexpr (V == 1) {
      const int ea = u >= pair_units ? p.R + u - pair_units : p.interleaved ? 2 * u : u;
      it.x = Elem<T>::load(in + ea);
      it.y = u >= pair_units ? 0.f : Elem<T>::load(in + (p.interleaved ? 2 * u + 1 : u + half));
    } else {
      const int e = u >= pair_units ? p.R + (u - pair_units) * V : u * V;
      it.a = *reinterpret_cast<const Raw*>(in + e);
      if (u < pair_units && !p.interleaved) it.c = *reinterpret_cast<const Raw*>(in + half + e);
    }
  };
  const auto finish = [&](const Item& it) {
    const int u = it.u;
    T* out = it.out;
    if constexpr (V == 1) {
      if (u >= pair_units) {
        out[p.R + u - pair_units] = Elem<T>::cvt(it.x);
        return;
      }
      out[p.interleaved ? 2 * u : u] = Elem<T>::cvt(it.x * it.cs[u] - it.y * it.sn[u]);
      out[p.interleaved ? 2 * u + 1 : u + half] = Elem<T>::cvt(it.y * it.cs[u] + it.x * it.sn[u]);
    } else if (u >= pair_units) {
      store_streaming(out + p.R + (u - pair_units) * V, it.a);
    } else if (p.interleaved) {
      float v[V];
      raw_unpack<T>(it.a, v);
#pragma unroll
      for (int i = 0; i < V / 2; i++) {
        const float a = v[2 * i], c = v[2 * i + 1], x = it.cs[u * (V / 2) + i], y = it.sn[u * (V / 2) + i];
        v[2 * i] = a * x - c * y;
        v[2 * i + 1] = c * x + a * y;
      }
      store_streaming(out + u * V, raw_pack<T>(v));
    } else {
      float a[V], c[V];
      raw_unpack<T>(it.a, a);
      raw_unpack<T>(it.c, c);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float x = it.cs[u * V + i], y = it.sn[u * V + i], first = a[i];
        a[i] = first * x - c[i] * y;
        c[i] = c[i] * x + first * y;
      }
      store_streaming(out + u * V, raw_pack<T>(a));
      store_streaming(out + half + u * V, raw_pack<T>(c));
    }
  };
  // (units are read and written by one thread each, so that outputs may be the inputs; four are on their way at once)
  constexpr int kAhead = 4;
  const int n = tokens * per_token;
  for (int j0 = tid; j0 < n; j0 += kAhead * 256) {
    Item it[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (j0 + k * 256 < n) fetch(j0 + k * 256, it[k]);
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (j0 + k * 256 < n) finish(it[k]);
  }
}

template <typename T>
int launch_rotary(const RotaryParams& p, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((p.tokens + p.tokens_per_group - 1) / p.tokens_per_group)), block(256);
  if (vec) hipLaunchKernelGGL((&rotary_kernel<T, Elem<T>::kChunk>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((&rotary_kernel<T, 1>), grid, block, 0, st, p);
  return launch_rc();
}

}  // namespace amoe

using namespace amoe;

extern "C" size_t amoe_rotary_args_bytes(void) { return sizeof(amoe_rotary_args); }

extern "C" int amoe_rotary(const amoe_rotary_args* a, void* stream) {
  if (!a) return AMOE_ENULL;
  if (a->dtype != AMOE_F32 && a->dtype != AMOE_BF16 && a->dtype != AMOE_F16) return AMOE_EINVAL;
  if (a->B < 0 || a->S < 0 || a->q_heads < 0 || a->k_heads < 0 || a->d < 1 || a->R < 2 || a->R % 2 || a->R > a->d) return AMOE_EINVAL;
  if (a->B == 0 || a->S == 0 || a->q_heads + a->k_heads == 0) return AMOE_OK;
  if (a->R / 2 > kRotaryPairs) return AMOE_EUNSUPPORTED;
  const int64_t limit = INT64_C(1) << 31;
  if (a->B >= limit || a->S >= limit || a->q_heads >= limit || a->k_heads >= limit || a->d >= limit) return AMOE_EUNSUPPORTED;
  if (a->B > limit / a->S || a->q_heads + a->k_heads > limit / 1024 / a->d) return AMOE_EUNSUPPORTED;
  if (!a->turns || (a->q_heads && (!a->q || !a->q_out)) || (a->k_heads && (!a->k || !a->k_out))) return AMOE_ENULL;
  const size_t es = esize((int)a->dtype);
  const int64_t c = 16 / (int64_t)es;
  if (!aligned(a->turns, 8) || !aligned(a->positions, a->positions_are_i64 ? 8 : 4)) return AMOE_EALIGN;
  bool vec = a->d % c == 0 && a->R % c == 0 && (a->interleaved || a->R / 2 % c == 0);
  RotaryParams p{};
  for (int i = 0; i < 2; i++) {
    const void* in = i ? a->k : a->q;
    void* out = i ? a->k_out : a->q_out;
    const int64_t* is = i ? &a->k_sb : &a->q_sb;
    const int64_t* os = i ? &a->k_out_sb : &a->q_out_sb;
    const int64_t heads = i ? a->k_heads : a->q_heads;
    const int64_t size[3] = {a->B, a->S, heads};
    int64_t st[2][3];
    p.part[i].heads = (int)heads;
    if (!heads) continue;
    if (!aligned(in, es) || !aligned(out, es)) return AMOE_EALIGN;
    vec = vec && aligned(in, 16) && aligned(out, 16);
    for (int j = 0; j < 3; j++) {
      if (is[j] < 0 || os[j] < 0) return AMOE_EINVAL;
      st[0][j] = size[j] == 1 ? 0 : is[j];
      st[1][j] = size[j] == 1 ? 0 : os[j];
      vec = vec && st[0][j] % c == 0 && st[1][j] % c == 0;
    }
    p.part[i] = {in, out, st[0][0], st[0][1], st[0][2], st[1][0], st[1][1], st[1][2], (int)heads};
  }
  p.turns = a->turns;
  p.pos = a->positions; p.pos_sb = a->pos_sb; p.pos_ss = a->pos_ss; p.pos_start = a->start; p.pos_i64 = (int)a->positions_are_i64;
  p.tokens = a->B * a->S;
  p.S = (int)a->S; p.d = (int)a->d; p.R = (int)a->R; p.interleaved = a->interleaved != 0;
  p.size = (float)a->size;
  p.sign = a->inverse ? -1.f : 1.f;
  // tokens per workgroup: about four 32-byte units per thread, as many as still give every CU four workgroups, and no more
  // than its tables hold
  int64_t n = 4 * 256 * 2 * c / ((a->q_heads + a->k_heads) * a->d);
  const int64_t spread = p.tokens / (4 * num_compute_units()), most = kRotaryPairs / (a->R / 2);
  if (n > spread) n = spread;
  if (n > most) n = most;
  p.tokens_per_group = (int)(n < 1 ? 1 : n);
  if (p.tokens / p.tokens_per_group >= INT64_C(1) << 23) return AMOE_EUNSUPPORTED;      // (threads of a launch are counted in 32 bits)
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_rotary<float>(p, vec, st)
         : a->dtype == AMOE_F16 ? launch_rotary<f16_t>(p, vec, st)
                                : launch_rotary<uint16_t>(p, vec, st);
}
