// What the attention kernels share: the arguments, the tiles in LDS, the operands of the matrix instructions.
//
// All kernels work on 32 x 32 blocks of scores whose COLUMNS belong to lanes: the forward pass and the gradient of q form
// K Q^T (a lane owns one query), the gradients of k and v form Q K^T (a lane owns one key).  Lane l then holds rows
// 8 * (i / 4) + 4 * (l / 32) + i % 4, i = 0 .. 15, of column l % 32, so that the sums of a softmax are sums over registers
// and one exchange with lane l ^ 32, and what is made of the scores is an operand of the next product where it lies: the
// contraction of that product may run over the rows in any order, so the other operand is read in the order of the registers.
#pragma once
#include "common.h"

namespace amoe {

constexpr int kAttnThreads = 256;    // 4 waves
constexpr int kAttnMaxHead = 128;    // elements of a head, at most
constexpr int kAttnMaxSplits = 1024;        // parts of the key axis
constexpr int64_t kAttnMaxRows = 1 << 28;   // queries and keys of a sequence, at most
constexpr float kLog2e = 1.4426950408889634f;

struct AttnOperand {                 // [B, rows, heads, d] with these strides (elements), the last one 1
  const void* p;
  int64_t sb, ss, sh;
};

struct AttnParams {
  AttnOperand q, k, v, go;           // go: gradient of the output
  void* out;                         // [B, S, H, d]
  const void* o;                     // the same, read by the backward pass
  void* rest;                        // [B, S, H, d]: out before its rounding less out, of the same type; written and read.  May be null
  float* lse;                        // [B, H, S]: log2 of the sum of 2^(score * c); +inf where a row sees nothing.  May be null
  float* rows;                       // 3 x [B, H, S], what dk and dv need of a row: norm and top (attn_far_rows), and between them
                                     // delta, the sum over d of out * gradient of out
  void *dq, *dk, *dv;                // [B, S, H, d], [B, T, G, d]
  const void *lengths, *starts;      // [B] int32 / int64 or null
  int lengths_i64, starts_i64;
  int B, S, T, H, G, R, d, causal;   // G key heads, R = H / G query heads share one
  int vec;                           // every operand in whole aligned 16-byte chunks with offsets that fit 32 bits
  float c;                           // scale * log2(e)
  float scale;
  int splits;                        // forward of few rows: parts of the key axis
  float *part_o, *part_ml;           // [splits][B * H * S][d rounded up to 4], [splits][B * H * S][2]
};

// keys that sequence b holds
__device__ __forceinline__ int attn_length(const AttnParams& p, int b) {
  if (!p.lengths) return p.T;
  const int64_t n = p.lengths_i64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  return (int)(n < 0 ? 0 : (n > p.T ? p.T : n));
}
// position of its first query; kept within +-2^29 (there are at most 2^28 queries and keys, so that no answer changes): sums
// with row numbers stay in 32 bits
__device__ __forceinline__ int attn_start(const AttnParams& p, int b) {
  int64_t n = (int64_t)p.T - p.S;
  if (p.starts) n = p.starts_i64 ? static_cast<const int64_t*>(p.starts)[b] : static_cast<const int32_t*>(p.starts)[b];
  constexpr int64_t lim = 1 << 29;
  return (int)(n < -lim ? -lim : (n > lim ? lim : n));
}
// keys [0, n) are what query i sees
__device__ __forceinline__ int attn_seen(const AttnParams& p, int length, int start, int i) {
  if (!p.causal) return length;
  const int n = start + i + 1;
  return n < 0 ? 0 : (n < length ? n : length);
}

// ---- operands -----------------------------------------------------------------------------------
// 16 steps of a contraction for one matrix operand: lane l holds 8 of them (which 8 depends on l / 32) of row or column
// l % 32.  16-bit types: one matrix instruction; fp32: eight, each of which takes element j of both halves of the wave.
template <typename T> struct AttnFrag { typedef u32x4 type; };
struct F32x8 { float v[8]; };
template <> struct AttnFrag<float> { typedef F32x8 type; };
template <typename T> using attn_frag = typename AttnFrag<T>::type;

template <typename T>
__device__ __forceinline__ f32x16 attn_mma(const attn_frag<T>& a, const attn_frag<T>& b, f32x16 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; j++) c = mfma_32x32x2_f32(a.v[j], b.v[j], c);
    return c;
  } else {
    return mfma_32x32x16<T>(a, b, c);
  }
}
// eight values rounded to T (nearest, ties to even): for 16-bit types the matrix unit takes nothing wider.  A probability
// or a score's gradient is off by 2^-9 (bf16) or 2^-12 (fp16) of itself at most, as much as a rounded output, and the errors
// of a sum's terms are independent of each other.
template <typename T>
__device__ __forceinline__ attn_frag<T> attn_pack(const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    F32x8 r;
#pragma unroll
    for (int j = 0; j < 8; j++) r.v[j] = v[j];
    return r;
  } else {
    return raw_pack<T>(v);
  }
}

// c plus the eight values as the matrix unit sees them, after their rounding
template <typename T>
__device__ __forceinline__ float attn_add_packed(const attn_frag<T>& f, float c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; j++) c += f.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (kIsF16<T>) {
        float a, b;                                    // (a dot product with ones as for bf16 is slower here: 38.5 us for 37.2 of the
        unpack_f16x2(f[j], a, b);                      // padded batch of 6 x 1717, heads of 80)
        c += a + b;
      } else {
        c = add_bf16x2(f[j], c);
      }
    }
  }
  return c;
}

// ---- tiles in LDS ---------------------------------------------------------------------------------
// Rows of DP elements in 16-byte chunks; chunk c of row r lies at chunk c ^ swizzle(r) of the row.  Both ways a tile is
// read touch every bank once: 16 rows at one chunk (operands whose rows are the tile's), and 4 rows at 4 adjacent chunks
// (the transposing read).  Which bits of r go where depends on how many of the 64 banks a row moves on by.
template <typename T, int DP> struct AttnTile {
  static constexpr int kRowChunks = DP * (int)sizeof(T) / 16;
  static constexpr int kChunk = 16 / (int)sizeof(T);
  static constexpr int kRowWords = DP * (int)sizeof(T) / 4;
  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (kRowWords % 64 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (kRowWords % 64 == 32) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  // element offset of chunk c of row r
  static __device__ __forceinline__ int at(int r, int c) { return (r * kRowChunks + (c ^ swizzle(r))) * kChunk; }

  // Byte offsets of a lane's reads in a tile, but for what a constant of the read adds or flips: the swizzle only sees the
  // low four bits of a row, and rows start on a power of two or 64 bytes, so that steps along the head are flipped bits.  (Kept
  // apart they would be 16 registers: in() makes them anew for every tile.)
  struct Lane {
    int row, col, first = 0;
    __device__ __forceinline__ Lane() {
      const int l = lane_id(), h = l >> 5;
      row = at(l & 31, h) * (int)sizeof(T);
      const int r = 4 * h + ((l & 15) >> 2), d = 16 * ((l >> 4) & 1) + 4 * (l & 3);
      col = (at(r, d / 8) + d % 8) * (int)sizeof(T);
    }
    // in the tile that begins at this element (a multiple of 256 bytes: no bit of it is flipped)
    __device__ __forceinline__ Lane in(int tile) const {
      Lane l = *this;
      l.row += tile * (int)sizeof(T);
      l.col += tile * (int)sizeof(T);
      l.first += tile;
      opaque(l.row);
      opaque(l.col);
      return l;
    }
  };
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  static constexpr bool kPow2 = kRowWords % 32 == 0;

  // Addresses are summed up before they meet the array of LDS that the tile lies in, and a kernel has more than one such array: the
  // compiler then knows which array a read is of, and does not make it wait for the tiles on their way into LDS.
  //
  // steps 16 * kk .. + 15 of the head axis, rows r0 + l % 32 (r0 a multiple of 16, as below)
  static __device__ __forceinline__ attn_frag<T> row_frag(const char* lds, const Lane& lane, int r0, int kk) {
    if constexpr (sizeof(T) == 4) {
      const int l = lane_id(), r = r0 + (l & 31), h = l >> 5;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(lds + 4 * (lane.first + at(r, 4 * kk + 2 * h)));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(lds + 4 * (lane.first + at(r, 4 * kk + 2 * h + 1)));
      return F32x8{{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
    } else {
      const int o = kPow2 ? lane.row ^ (kk << 5) : (lane.row ^ ((kk & 1) << 5)) + (kk >> 1) * 64;
      return *reinterpret_cast<const u32x4*>(lds + (r0 * kRowBytes + o));
    }
  }
  // rows r0 .. r0 + 15 as the steps, in the order of a score block's registers, of head elements 32 * dt + l % 32
  static __device__ __forceinline__ attn_frag<T> col_frag(const char* lds, const Lane& lane, int r0, int dt) {
    if constexpr (sizeof(T) == 4) {
      const int l = lane_id(), h = l >> 5, d = 32 * dt + (l & 31);
      F32x8 f;
#pragma unroll
      for (int j = 0; j < 8; j++)
        f.v[j] = *reinterpret_cast<const float*>(lds + 4 * (lane.first + at(r0 + 8 * (j / 4) + 4 * h + j % 4, d / 4) + d % 4));
      return f;
    } else {
      u32x2 half[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {                        // rows 4 h .. + 3, and the same 8 on
        const int o = kPow2 ? lane.col ^ (dt << 6) ^ (u << 5) : (lane.col ^ (u << 5)) + dt * 64;
        half[u] = lds_read_tr16_b64(reinterpret_cast<const uint16_t*>(lds + (r0 * kRowBytes + o + 8 * u * kRowBytes)));
      }
      return u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
    }
  }
};

// A workgroup's waves over rows and keys: RW waves have 32 queries each, in KG copies that take every KG-th block of 32 keys and
// are joined at the end.  Copies make more and shorter workgroups of the same work, for launches that would leave CUs idle, at
// the price of reading the keys for fewer rows at a time.  kBlocks blocks of keys per copy and tile: two, where the tiles and the
// registers of two blocks leave room for three workgroups on a CU: 16-bit heads up to 96.
template <typename T, int DP, bool EDGE, int RW_> struct AttnShape {
  static constexpr int RW = RW_, KG = 4 / RW, kRows = 32 * RW;
  static constexpr int kBlocks = KG == 1 && sizeof(T) == 2 && DP < 128 ? 2 : 1, kKeys = 32 * KG * kBlocks;
  static constexpr int kWavesPerSimd = sizeof(T) == 4 && (DP > 64 || EDGE) ? 1 : 2;
  // what fits the 160 KB of a CU
  static constexpr bool kFits = 4 * kKeys * DP * (int)sizeof(T) <= 128 << 10;
};

// A run of matrix products whose first operands come from LDS, with kAttnAhead of them on their way: a read takes as long as
// three or four products, and left to itself the compiler has one in flight (8192 queries, 16 over 4 heads of 128: forward 325 us
// with one ahead, 285 with four; dk and dv 728 with one, 653 with three).  Nothing is moved across a step.  fp32 products take
// eight instructions each: two ahead do.
template <typename T> inline constexpr int kAttnAhead = sizeof(T) == 4 ? 2 : 6;
template <typename T, int N, int AHEAD = kAttnAhead<T>> struct AttnRun {
  static constexpr int D = AHEAD < N ? AHEAD : N;
  attn_frag<T> f[D];
  template <class Load>
  __device__ __forceinline__ void begin(Load load) {
#pragma unroll
    for (int i = 0; i < D; i++) f[i] = load(i);
    sched_fence();
  }
  // steps lo .. hi - 1: use(i, operand i), and operand i + D is asked for
  template <class Load, class Use>
  __device__ __forceinline__ void steps(int lo, int hi, Load load, Use use) {
#pragma unroll
    for (int i = lo; i < hi; i++) {
      use(i, f[i % D]);
      if (i + D < N) f[i % D] = load(i + D);
      sched_fence();
    }
  }
};

// Rows [row0, row0 + ROWS) of one head on their way from global memory to a tile, by NT threads.  Rows at or past row_end and
// elements at or past d are zeros in the tile and are not touched in memory.  THROUGH_REGS: load() leaves them in registers and
// store() puts them into the tile; else load() sends them straight there, in the order of the tile's slots (which saves 16 to 32
// registers that the products need), to be there after finish() and a barrier.  EDGE: any strides and alignment, through registers.
template <typename T, int DP, int ROWS, int NT, bool EDGE, bool THROUGH_REGS = EDGE>
struct AttnStage {
  using Tile = AttnTile<T, DP>;
  static constexpr int kN = ROWS * Tile::kRowChunks / NT;
  static_assert(ROWS * Tile::kRowChunks % NT == 0, "whole chunks per thread");
  static_assert(!EDGE || THROUGH_REGS, "edges go through registers");
  Raw r[THROUGH_REGS ? kN : 1];
  uint32_t off[EDGE ? 1 : kN];

  __device__ __forceinline__ void init(int tid, int64_t stride, int d) {
    if constexpr (!EDGE) {
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const int idx = tid + i * NT, row = idx / Tile::kRowChunks, slot = idx % Tile::kRowChunks;
        const int ch = THROUGH_REGS ? slot : slot ^ Tile::swizzle(row);
        // (an offset past every resource: reads zero)
        off[i] = ch * Tile::kChunk < d ? (uint32_t)(row * stride * (int64_t)sizeof(T)) + (uint32_t)ch * 16u : 0xfffffff0u;
      }
    }
  }
  __device__ __forceinline__ void load(int tid, T* tile, const T* base, int64_t stride, int row0, int row_end, int d, bool vec) {
    const T* p = base + (int64_t)row0 * stride;
    const int rows = row_end - row0 < ROWS ? row_end - row0 : ROWS;
    if constexpr (EDGE) {
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const int idx = tid + i * NT, row = idx / Tile::kRowChunks, ch = idx % Tile::kRowChunks;
        r[i] = raw_zero();
        if (row < rows) r[i] = raw_load<T>(p + row * stride + ch * Tile::kChunk, d - ch * Tile::kChunk, vec);
      }
    } else {
      const uint32_t bytes = rows > 0 ? (uint32_t)((rows - 1) * stride + d) * (uint32_t)sizeof(T) : 0u;
      const BufRsrc rs = make_rsrc_sized(const_cast<T*>(rows > 0 ? p : base), bytes);
      char* to = reinterpret_cast<char*>(tile) + wave_uniform(tid >> 6) * 1024;
#pragma unroll
      for (int i = 0; i < kN; i++) {
        if constexpr (THROUGH_REGS) r[i] = buffer_load_b128(rs, off[i], 0);
        else buffer_to_lds_b128(rs, to + i * NT * 16, off[i]);
      }
    }
  }
  __device__ __forceinline__ void store(int tid, T* tile) const {
    if constexpr (THROUGH_REGS) {
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const int idx = tid + i * NT;
        *reinterpret_cast<Raw*>(tile + Tile::at(idx / Tile::kRowChunks, idx % Tile::kRowChunks)) = r[i];
      }
    }
  }
  __device__ __forceinline__ void finish() const {
    if constexpr (!THROUGH_REGS) lds_dma_wait();
  }
};

// One row's operand, steps 16 * kk .., straight from global memory; ok: the row exists.
template <typename T, bool EDGE>
__device__ __forceinline__ attn_frag<T> attn_global_frag(const T* row, int kk, int d, bool ok, bool vec) {
  const int h = lane_id() >> 5, e = 16 * kk + 8 * h;
  const bool v = EDGE ? vec : true;
  constexpr int C = Elem<T>::kChunk;
  if constexpr (sizeof(T) == 4) {
    Raw a = raw_zero(), b = raw_zero();
    if (ok && e < d) a = raw_load<T>(row + e, EDGE ? d - e : C, v);
    if (ok && e + 4 < d) b = raw_load<T>(row + e + 4, EDGE ? d - e - 4 : C, v);
    return F32x8{{as_f32(a[0]), as_f32(a[1]), as_f32(a[2]), as_f32(a[3]), as_f32(b[0]), as_f32(b[1]), as_f32(b[2]), as_f32(b[3])}};
  } else {
    Raw a = raw_zero();
    if (ok && e < d) a = raw_load<T>(row + e, EDGE ? d - e : C, v);
    return a;
  }
}

// The operands of rows row0 + l % 32, the whole head, straight from global memory; rows at or past row_end and elements past d are
// zeros.  (Without edges one resource that ends with the rows does that, and no load waits for a branch.)
template <typename T, int DP, bool EDGE>
__device__ __forceinline__ void attn_row_frags(attn_frag<T> (&f)[DP / 16], const T* base, int64_t stride, int row0, int row_end, int d, bool vec) {
  const int l = lane_id(), h = l >> 5;
  const T* p = base + (int64_t)row0 * stride;
  if constexpr (EDGE) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++)
      f[kk] = attn_global_frag<T, EDGE>(p + (l & 31) * stride, kk, d, row0 + (l & 31) < row_end, vec);
  } else {
    const int rows = row_end - row0 < 32 ? row_end - row0 : 32;
    const uint32_t bytes = rows > 0 ? (uint32_t)((rows - 1) * stride + d) * (uint32_t)sizeof(T) : 0u;
    const BufRsrc rs = make_rsrc_sized(const_cast<T*>(rows > 0 ? p : base), bytes);
    const uint32_t at = (uint32_t)((l & 31) * stride + 8 * h) * (uint32_t)sizeof(T);
    // (no more rows than there are: an offset past the end reads zero, but must not wrap round)
    const bool ok = (l & 31) < rows;
#pragma unroll
    for (int kk = 0; kk < DP / 16; kk++) {
      const uint32_t off = ok && 16 * kk + 8 * h < d ? at + 16u * kk * (uint32_t)sizeof(T) : 0xfffffff0u;
      if constexpr (sizeof(T) == 4) {
        const uint32_t off2 = ok && 16 * kk + 8 * h + 4 < d ? off + 16u : 0xfffffff0u;
        const Raw a = buffer_load_b128(rs, off, 0), b = buffer_load_b128(rs, off2, 0);
        f[kk] = F32x8{{as_f32(a[0]), as_f32(a[1]), as_f32(a[2]), as_f32(a[3]), as_f32(b[0]), as_f32(b[1]), as_f32(b[2]), as_f32(b[3])}};
      } else {
        f[kk] = buffer_load_b128(rs, off, 0);
      }
    }
  }
}

// the larger (the sum) of a lane's and its partner's in the other half of the wave
__device__ __forceinline__ float attn_pair_max(float v) {
  uint32_t a = as_u32(v), b = a;
  swap_half_waves(a, b);
  return fmaxf(as_f32(a), as_f32(b));
}
__device__ __forceinline__ float attn_pair_sum(float v) {
  uint32_t a = as_u32(v), b = a;
  swap_half_waves(a, b);
  return as_f32(a) + as_f32(b);
}

template <typename T>
__device__ __forceinline__ float attn_rest(float v) { return v - Elem<T>::to_f32(Elem<T>::cvt(v)); }

// A lane's column of a [head elements][32] product times factor, to its row in memory (ok: it has one).  It holds 4 adjacent
// elements of every 8, its partner l ^ 32 the other 4; 16-bit elements change places so that each stores 8 at a time.  The whole
// wave calls this.  REST: what the rounding to T takes away, instead.
template <typename T, int DP, bool EDGE, bool REST = false>
__device__ __forceinline__ void attn_store_col(T* row, const f32x16* acc, float factor, int d, bool ok) {
  const int h = lane_id() >> 5;
  const auto value = [&](int t, int i) {
    const float v = acc[t][i] * factor;
    return REST ? attn_rest<T>(v) : v;
  };
  if constexpr (EDGE || sizeof(T) == 4) {
    const bool vec = !EDGE || (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int e = 32 * t + 8 * g + 4 * h;
        if (!ok || e >= d) continue;
        const float v[4] = {value(t, 4 * g), value(t, 4 * g + 1), value(t, 4 * g + 2), value(t, 4 * g + 3)};
        store4<T>(row + e, v, EDGE ? d - e : 4, vec);
      }
  } else {
#pragma unroll
    for (int t = 0; t < DP / 32; t++)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        const float v[8] = {value(t, 4 * g),     value(t, 4 * g + 1), value(t, 4 * g + 2), value(t, 4 * g + 3),
                            value(t, 4 * g + 4), value(t, 4 * g + 5), value(t, 4 * g + 6), value(t, 4 * g + 7)};
        const Raw r = raw_pack<T>(v);
        uint32_t a0 = r[0], a1 = r[1], b0 = r[2], b1 = r[3];
        swap_half_waves(a0, b0);
        swap_half_waves(a1, b1);
        const int e = 32 * t + 8 * (g + h);
        if (ok && e < d) *reinterpret_cast<Raw*>(row + e) = Raw{a0, a1, b0, b1};
      }
  }
}

__device__ __forceinline__ f32x16 f32x16_zero() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; i++) z[i] = 0.f;
  return z;
}

}  // namespace amoe
