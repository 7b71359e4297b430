// The choice of a token from a row of V logits and a given number u of [0, 1).
//   weight_i = exp((x_i - max) / temperature);  tokens rank by x, the lower index first among equals
//   kept: the first top_k; of these the shortest run from the top with at least top_p of their weight; of these weights of min_p
//   or more.  Drawn: in the order of the indices, the first up to which the kept ones weigh more than u times all of them.
//
// Weights are whole multiples of 2^-44 of the largest one (made in 64 bits, by a table of 2^(j / 256) and four terms of the series
// between), so that their sums are exact and the same in any order: what is drawn depends neither on how a row is shared out
// among threads nor on the order of the atomics that count, and is the definition's wherever u, top_p and the sums do not meet to
// within 2^-44 of the largest weight.  (In fp32 a row of 10^5 logits would go to a neighbour about once in a thousand draws.)
// What weighs less than 2^-45 of the largest is never drawn.
//
// The cut that top_k and top_p make in the ranking is found without a sort: the distances from the maximum are counted (and weighed)
// in 2047 equal intervals, and only the interval with the cut is ranked.  Bound by LDS atomics and 64-bit arithmetic where rows are
// truncated, by the weights' arithmetic and memory where not.
#include <amoe.h>

#include "host_util.h"

namespace amoe {

typedef unsigned long long u64;
// (closures that are not inlined live in memory, and with them all that they refer to)
#define AMOE_INLINE __attribute__((always_inline))

struct SampleParams {
  const void* logits;                // [rows, V], ld elements apart
  const void* u;                     // [rows] fp32 or fp64
  // one for every row, or null: the number for all
  const float *temperature, *top_p, *min_p;
  const void* top_k;
  int64_t* ids;
  float* logprob;                    // may be null
  int64_t ld, rows, top_k_all;
  int V, u_f64, top_k_i64;
  float temperature_all, top_p_all, min_p_all;
};

constexpr int64_t kSampleMaxV = (1 << 20) - 1;       // (as many largest weights are less than 2^64)
constexpr int kBins = 2048;          // the last one holds what weighs nothing and is not counted
constexpr int kList = 2048;          // elements that are ranked at once
constexpr u64 kOne = 1ull << 44;
constexpr int kIndexBits = 20;

// A row of V elements: chunks of 16 bytes that begin on 4, and what is left before (one element) and behind them (less than a
// chunk), which lanes of the first wave hold one by one.  Groups of 64 chunks go to the waves in units of `per`, four units at most to
// a wave, 60 in all.  Chunks past the last one read as zeros from a resource that ends with it, so that no load waits for a branch.
template <typename T, int W> struct SampleRow {
  static constexpr int C = Elem<T>::kChunk;
  BufRsrc chunks_at;
  int head, body, tail, groups, per, units;
  float edge;                        // of the first wave's lanes: lane 0 the element before the chunks, lanes 1 .. those behind
  int edge_index;
  __device__ __forceinline__ SampleRow(const T* row, int V) {
    head = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(row) & 2) ? 1 : 0;
    body = (V - head) / C;
    tail = V - head - body * C;
    groups = (body + 63) / 64;
    const int even = (groups + W - 1) / W;
    constexpr int kMost = 4 * W < 60 ? 4 * W : 60;
    per = (groups + kMost - 1) / kMost;
    if (per < 4) per = even < 4 ? (even > 1 ? even : 1) : 4;
    units = (groups + per - 1) / per;
    chunks_at = make_rsrc_sized(const_cast<T*>(row + head), (uint32_t)body * 16u);
    const int t = threadIdx.x;
    edge_index = t == 0 ? 0 : V - tail + t - 1;
    const bool there = t == 0 ? head == 1 : t <= tail;
    edge = there ? Elem<T>::load(row + edge_index) : -INFINITY;
    edge = edge == edge ? edge : -INFINITY;
  }
  __device__ __forceinline__ int start(int j) const { return head + j * C; }
  // f(values, index of the first) for the chunks of groups [g, g_end) that are this lane's; minus infinity where there is no number
  template <class F>
  __device__ __forceinline__ void chunks(int g, int g_end, F f) const {
    constexpr int kAhead = 4;
    const int lane = lane_id();
    for (; g < g_end; g += kAhead) {
      Raw r[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) r[i] = buffer_load_b128(chunks_at, (uint32_t)((g + i) * 64 + lane) * 16u, 0);
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const int j = (g + i) * 64 + lane;
        if (g + i >= g_end) continue;
        float v[C];
        raw_unpack<T>(r[i], v);
#pragma unroll
        for (int e = 0; e < C; e++) v[e] = j < body && v[e] == v[e] ? v[e] : -INFINITY;
        f(v, start(j));
      }
    }
  }
  // every element: f(values, index of the first) on chunks, one(value, index) on single ones
  template <class F, class One>
  __device__ __forceinline__ void all(F f, One one) const {
    const int wave = wave_uniform(threadIdx.x >> 6);
    for (int u = wave; u < units; u += W) chunks(u * per, (u + 1) * per < groups ? (u + 1) * per : groups, f);
    if (threadIdx.x < 64 && edge != -INFINITY) one(edge, edge_index);
  }
};

struct SampleWeight {
  float top;
  double scale;                      // 256 log2(e) / temperature
  bool flat;                         // only the largest weigh (temperature 0, or infinite logits)
  const double* table;               // 2^(j / 256)
  __device__ __forceinline__ u64 operator()(float x) const {
    // (what is so far below that it weighs nothing, and minus infinity, whose distance may be no number)
    const double t = __builtin_fmax(((double)x - (double)top) * scale, -46.0 * 256.0);
    const double n = __builtin_rint(t), f = t - n;
    const int i = (int)n;
    constexpr double a = 0.69314718055994530942 / 256;
    const double q = f * __builtin_fma(f, __builtin_fma(f, __builtin_fma(f, a * a * a * a / 24, a * a * a / 6), a * a / 2), a);
    const double w = table[i & 255];
    // (256 + w: the last bit counts 2^-44)
    const u64 r = __builtin_bit_cast(u64, __builtin_ldexp(__builtin_fma(w, q, w), i >> 8) + 256.0) - __builtin_bit_cast(u64, 256.0);
    return flat ? (x == top ? kOne : 0) : r;
  }
};

// rank of an element as a number: the larger logit is the larger, among equals the lower index
__device__ __forceinline__ u64 sample_rank(float x, int index) {
  const uint32_t b = as_u32(x + 0.f);               // (-0 is 0)
  const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return ((u64)key << kIndexBits) | (u64)((1 << kIndexBits) - 1 - index);
}
__device__ __forceinline__ float sample_value(u64 rank) {
  const uint32_t key = (uint32_t)(rank >> kIndexBits);
  return as_f32(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ int sample_index(u64 rank) { return (1 << kIndexBits) - 1 - (int)(rank & ((1 << kIndexBits) - 1)); }

template <typename V>
__device__ __forceinline__ V wave_scan(V v) {       // sums up to and with the lane's
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const V up = wave_shfl_up(v, d);
    if (lane_id() >= d) v += up;
  }
  return v;
}

// What a workgroup shares beside the histogram.
template <int W> struct SampleShared {
  double table[256];
  u64 unit[64], group[128], wave_w[W];
  float wave_max[W], wave_min[W];
  int wave_n[W], found, listed;
  u64 found_w, found_n, cut;
};
struct SampleBins {
  uint32_t n[kBins];
  u64 w[kBins];
};
union SampleRanked {
  u64 list[kList];
  SampleBins digit;
};

// Sums of (n, w) over the threads before this one.
template <int W>
__device__ __forceinline__ void sample_scan(int& n, u64& w, SampleShared<W>& sh) {
  const int wave = threadIdx.x >> 6, lane = lane_id(), in = wave_scan(n);
  const u64 iw = wave_scan(w);
  __syncthreads();
  if (lane == 63) {
    sh.wave_n[wave] = in;
    sh.wave_w[wave] = iw;
  }
  __syncthreads();
  n = in - n;
  w = iw - w;
  for (int i = 0; i < wave; i++) {
    n += sh.wave_n[i];
    w += sh.wave_w[i];
  }
}

// The first bin up to which there are at least `target` (of what is counted, or weighed): sh.found (-1: there are fewer), and in
// found_n and found_w what is before it.
template <int NT>
__device__ __forceinline__ void sample_crossing(const SampleBins& bins, int size, bool by_weight, u64 target, SampleShared<NT / 64>& sh) {
  constexpr int P = kBins / NT;
  const int first = threadIdx.x * P;
  int n[P], before_n = 0;
  u64 w[P], before_w = 0;
#pragma unroll
  for (int i = 0; i < P; i++) {
    n[i] = first + i < size ? (int)bins.n[first + i] : 0;
    w[i] = first + i < size ? bins.w[first + i] : 0;
    before_n += n[i];
    before_w += w[i];
  }
  sample_scan<NT / 64>(before_n, before_w, sh);
  if (threadIdx.x == 0) sh.found = -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < P; i++) {
    const u64 b = by_weight ? before_w : (u64)before_n, a = b + (by_weight ? w[i] : (u64)n[i]);
    if (b < target && a >= target) {
      sh.found = first + i;
      sh.found_n = (u64)before_n;
      sh.found_w = before_w;
    }
    before_n += n[i];
    before_w += w[i];
  }
  __syncthreads();
}

// The rank at which `target` is reached within one bin of the row (n of its elements, w of weight before the bin): sh.cut, and in
// found_w the weight up to and with it.
template <typename T, int NT, class Bin>
__device__ __forceinline__ void sample_refine(const SampleRow<T, NT / 64>& row, const SampleWeight& weight, Bin bin, int b, int count,
                                              bool by_weight, u64 target, u64 before_n, u64 before_w, SampleRanked& r,
                                              SampleShared<NT / 64>& sh) {
  constexpr int W = NT / 64;
  const int tid = threadIdx.x;
  // too many to rank at once: by 11 bits of their ranks at a time
  int shift = 32 + kIndexBits;
  u64 prefix = 0;
  while (count > kList) {
    const int next = shift > 11 ? shift - 11 : 0, size = 1 << (shift - next);
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) {
      r.digit.n[i] = 0;
      r.digit.w[i] = 0;
    }
    __syncthreads();
    const auto count_one = [&](float x, int index) AMOE_INLINE {
      if (bin(x) != b) return;
      const u64 rank = sample_rank(x, index);
      if (rank >> shift != prefix) return;
      const int d = size - 1 - (int)((rank >> next) & (u64)(size - 1));
      atomicAdd(&r.digit.n[d], 1u);
      atomicAdd(&r.digit.w[d], weight(x));
    };
    row.all(
        [&](const float (&v)[SampleRow<T, W>::C], int first) AMOE_INLINE {
#pragma unroll
          for (int e = 0; e < SampleRow<T, W>::C; e++) count_one(v[e], first + e);
        },
        count_one);
    __syncthreads();
    sample_crossing<NT>(r.digit, size, by_weight, target - (by_weight ? before_w : before_n), sh);
    const int d = sh.found;
    count = (int)r.digit.n[d];
    before_n += sh.found_n;
    before_w += sh.found_w;
    prefix = (prefix << (shift - next)) | (u64)(size - 1 - d);
    shift = next;
  }
  __syncthreads();
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  const auto list_one = [&](float x, int index) AMOE_INLINE {
    if (bin(x) != b) return;
    const u64 rank = sample_rank(x, index);
    if (rank >> shift == prefix) r.list[atomicAdd(&sh.listed, 1)] = rank;
  };
  row.all(
      [&](const float (&v)[SampleRow<T, W>::C], int first) AMOE_INLINE {
#pragma unroll
        for (int e = 0; e < SampleRow<T, W>::C; e++) list_one(v[e], first + e);
      },
      list_one);
  int size = 2;
  while (size < count) size *= 2;
  for (int i = count + tid; i < size; i += NT) r.list[i] = 0;
  __syncthreads();
  // the largest first
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = tid; i < size / 2; i += NT) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const u64 a = r.list[lo], c = r.list[hi];
        if ((a < c) == ((lo & k) == 0)) {
          r.list[lo] = c;
          r.list[hi] = a;
        }
      }
      __syncthreads();
    }
  constexpr int P = kList / NT;
  u64 w[P], sum = 0;
  int none = 0;
#pragma unroll
  for (int i = 0; i < P; i++) {
    w[i] = tid * P + i < count ? weight(sample_value(r.list[tid * P + i])) : 0;
    sum += w[i];
  }
  sample_scan<W>(none, sum, sh);
#pragma unroll
  for (int i = 0; i < P; i++) {
    const int at = tid * P + i;
    const u64 b = by_weight ? before_w + sum : before_n + (u64)at, a = b + (by_weight ? w[i] : 1);
    sum += w[i];
    if (at < count && b < target && a >= target) {
      sh.cut = r.list[at];
      sh.found_w = before_w + sum;
    }
  }
  __syncthreads();
}

template <typename T, int NT, bool CUT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleParams p) {
  constexpr int W = NT / 64, C = Elem<T>::kChunk;
  __shared__ SampleShared<W> sh;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6);
  const int64_t at = blockIdx.x;
  const SampleRow<T, W> row(static_cast<const T*>(p.logits) + at * p.ld, p.V);
  const float temperature = p.temperature ? p.temperature[at] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[at] : p.top_p_all, min_p = p.min_p ? p.min_p[at] : p.min_p_all;
  const int64_t top_k = !p.top_k ? p.top_k_all : p.top_k_i64 ? static_cast<const int64_t*>(p.top_k)[at] : static_cast<const int32_t*>(p.top_k)[at];
  double u = p.u_f64 ? static_cast<const double*>(p.u)[at] : (double)static_cast<const float*>(p.u)[at];
  for (int i = tid; i < 256; i += NT) sh.table[i] = ::exp2((double)i / 256.0);

  float mx = -INFINITY, mn = INFINITY;
  const auto extremes = [&](float x, int) AMOE_INLINE {
    mx = fmaxf(mx, x);
    if (CUT) mn = fminf(mn, x == -INFINITY ? INFINITY : x);
  };
  row.all(
      [&](const float (&v)[C], int first) AMOE_INLINE {
#pragma unroll
        for (int e = 0; e < C; e++) extremes(v[e], first + e);
      },
      extremes);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    mx = fmaxf(mx, wave_shfl_xor(mx, d));
    if (CUT) mn = fminf(mn, wave_shfl_xor(mn, d));
  }
  if (lane == 0) {
    sh.wave_max[wave] = mx;
    sh.wave_min[wave] = mn;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; i++) {
    mx = fmaxf(mx, sh.wave_max[i]);
    mn = fminf(mn, sh.wave_min[i]);
  }
  if (mx == -INFINITY) {
    if (tid == 0) {
      p.ids[at] = -1;
      if (p.logprob) p.logprob[at] = -INFINITY;
    }
    return;
  }
  const bool greedy = !(temperature > 0.f);
  const SampleWeight weight{mx, greedy ? 0.0 : 256 * 1.44269504088896340736 / (double)temperature, greedy || mx == INFINITY, sh.table};
  if (greedy) u = 0.0;                               // (the first of those that weigh)

  u64 cut = 0;
  if constexpr (CUT) {
    __shared__ SampleBins hist;
    __shared__ SampleRanked ranked;
    const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.f;
    if (!greedy && (by_k || by_p)) {
      // (half the distances: they may be twice the largest float)
      const float half = 0.5f * mx, reach = fminf(fmaf(-0.5f, mn, half), 16.f * temperature);
      const float step = reach > 0.f ? fminf((kBins - 2) / reach, 3.402823466e38f) : 0.f;
      const bool flat = weight.flat;
      const auto bin = [=](float x) AMOE_INLINE {
        if (flat) return x == mx ? 0 : kBins - 1;
        return (int)fminf(fmaf(-0.5f, x, half) * step, (float)(kBins - 1));
      };
      for (int i = tid; i < kBins; i += NT) {
        hist.n[i] = 0;
        hist.w[i] = 0;
      }
      __syncthreads();
      const auto count_one = [&](float x, int) AMOE_INLINE {
        const int b = bin(x);
        if (b >= kBins - 1) return;
        atomicAdd(&hist.n[b], 1u);
        if (by_p) atomicAdd(&hist.w[b], weight(x));
      };
      row.all(
          [&](const float (&v)[C], int first) AMOE_INLINE {
#pragma unroll
            for (int e = 0; e < C; e++) count_one(v[e], first + e);
          },
          count_one);
      __syncthreads();
      u64 total = 0;
      bool cut_by_k = false;
      if (by_k) {
        sample_crossing<NT>(hist, kBins, false, (u64)top_k, sh);
        const int b = sh.found;
        if (b >= 0) {
          const u64 before_n = sh.found_n, before_w = sh.found_w;
          sample_refine<T, NT>(row, weight, bin, b, (int)hist.n[b], false, (u64)top_k, before_n, before_w, ranked, sh);
          cut_by_k = true;
          cut = sh.cut;
          total = sh.found_w;
        }
      }
      if (by_p) {
        if (!cut_by_k) {
          int n = 0;
          u64 w = 0;
          for (int i = tid; i < kBins; i += NT) w += hist.w[i];
          const u64 mine = w;
          sample_scan<W>(n, w, sh);
          __syncthreads();
          if (tid == NT - 1) sh.found_w = w + mine;
          __syncthreads();
          total = sh.found_w;
        }
        const double part = top_p > 0.f ? __builtin_ceil((double)top_p * (double)total) : 1.0;
        const u64 target = part < 1.0 ? 1 : (u64)part;
        __syncthreads();
        sample_crossing<NT>(hist, kBins, true, target, sh);
        const int b = sh.found;
        if (b >= 0) {
          const u64 before_n = sh.found_n, before_w = sh.found_w;
          sample_refine<T, NT>(row, weight, bin, b, (int)hist.n[b], true, target, before_n, before_w, ranked, sh);
          if (sh.cut > cut) cut = sh.cut;
        }
      }
    }
  }
  const float cut_x = cut ? sample_value(cut) : -INFINITY;
  const int cut_i = cut ? sample_index(cut) : p.V;
  const u64 least = min_p > 0.f ? (u64)__builtin_ceil((double)fminf(min_p, 1.f) * (double)kOne) : 0;
  // weights of a chunk's kept elements
  const auto weigh_one = [&](float x, int index) AMOE_INLINE -> u64 {
    const bool keep = (x > cut_x) | ((x == cut_x) & (index <= cut_i));
    const u64 w = weight(x);
    return keep & (w >= least) ? w : 0;
  };
  const auto weigh = [&](const float (&v)[C], int first, u64 (&w)[C]) AMOE_INLINE {
    bool any = false;
#pragma unroll
    for (int e = 0; e < C; e++) {
      any = any | (v[e] >= cut_x);
      w[e] = 0;
    }
    if (!any) return;
#pragma unroll
    for (int e = 0; e < C; e++) w[e] = weigh_one(v[e], first + e);
  };
  const auto group_sum = [&](int g, int g_end) AMOE_INLINE {
    u64 s = 0;
    row.chunks(g, g_end, [&](const float (&v)[C], int first) AMOE_INLINE {
      u64 w[C];
      weigh(v, first, w);
#pragma unroll
      for (int e = 0; e < C; e++) s += w[e];
    });
    return s;
  };
  const auto wave_total = [&](u64 s) AMOE_INLINE {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += wave_shfl_xor(s, d);
    return s;
  };
  __syncthreads();                                    // (the table, where nothing was cut)
  for (int i = wave; i < row.units; i += W) {
    const int end = (i + 1) * row.per < row.groups ? (i + 1) * row.per : row.groups;
    const u64 s = wave_total(group_sum(i * row.per, end));
    if (lane == 0) sh.unit[1 + i] = s;
  }
  // the element before the chunks and those behind them are units of their own, the first and the last
  const u64 edge_w = wave == 0 && row.edge != -INFINITY ? weigh_one(row.edge, row.edge_index) : 0;
  if (wave == 0) {
    const u64 behind = wave_total(lane == 0 ? 0 : edge_w);
    if (lane == 0) {
      sh.unit[0] = edge_w;
      sh.unit[1 + row.units] = behind;
    }
  }
  __syncthreads();
  // the unit, then the group of chunks, then the chunk, then the element at which the sum passes u times the total
  u64 mine = lane < row.units + 2 ? sh.unit[lane] : 0, run = wave_scan(mine);
  const u64 total = wave_shfl(run, 63);
  const double want = (u > 0.0 ? u : 0.0) * (double)total;
  u64 target = want < (double)total ? (u64)want : total - 1;
  if (target >= total) target = total - 1;
  const int unit = ctz64(wave_ballot(run > target)) - 1;
  target -= wave_shfl(run - mine, unit + 1);
  const bool edges = unit < 0 || unit == row.units;
  const int g0 = unit * row.per, g1 = g0 + row.per < row.groups ? g0 + row.per : row.groups;
  if (!edges) {
    for (int g = g0 + wave; g < g1; g += W) {
      const u64 s = wave_total(group_sum(g, g + 1));
      if (lane == 0) sh.group[g - g0] = s;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  int which = 0;
  float value = 0.f;
  if (edges) {
    run = wave_scan((lane == 0) == (unit < 0) ? edge_w : 0);
    if (lane != ctz64(wave_ballot(run > target))) return;
    which = row.edge_index;
    value = row.edge;
  } else {
    const u64 even = 2 * lane < g1 - g0 ? sh.group[2 * lane] : 0, odd = 2 * lane + 1 < g1 - g0 ? sh.group[2 * lane + 1] : 0;
    run = wave_scan(even + odd);
    const int pair = ctz64(wave_ballot(run > target));
    target -= wave_shfl(run - even - odd, pair);
    const u64 first_of_pair = wave_shfl(even, pair);
    const bool second = target >= first_of_pair;
    if (second) target -= first_of_pair;
    const int group = g0 + 2 * pair + (second ? 1 : 0);
    u64 w[C] = {};
    float x[C] = {};
    int start = 0;
    row.chunks(group, group + 1, [&](const float (&v)[C], int first) AMOE_INLINE {
      weigh(v, first, w);
      start = first;
#pragma unroll
      for (int e = 0; e < C; e++) x[e] = v[e];
    });
    mine = 0;
#pragma unroll
    for (int e = 0; e < C; e++) mine += w[e];
    run = wave_scan(mine);
    if (lane != ctz64(wave_ballot(run > target))) return;
    u64 sum = run - mine;
    bool found = false;
#pragma unroll
    for (int e = 0; e < C; e++) {
      sum += w[e];
      if (!found && sum > target) {
        found = true;
        which = start + e;
        value = x[e];
      }
    }
  }
  p.ids[at] = which;
  if (p.logprob) {
    const double log_total = ::log((double)total * 0x1p-44);
    p.logprob[at] = greedy ? 0.f : (float)((weight.flat ? 0.0 : ((double)value - (double)mx) / (double)temperature) - log_total);
  }
}

namespace {

template <typename T>
int launch_sample(const SampleParams& p, bool cut, hipStream_t st) {
  const dim3 grid((unsigned)p.rows);
  const bool wide = p.V > 16384 || p.rows < 2 * num_compute_units();
#define AMOE_LAUNCH(NT, CUT) hipLaunchKernelGGL((&sample_kernel<T, NT, CUT>), grid, dim3(NT), 0, st, p)
  if (wide && cut) AMOE_LAUNCH(1024, true);
  else if (wide) AMOE_LAUNCH(1024, false);
  else if (cut) AMOE_LAUNCH(256, true);
  else AMOE_LAUNCH(256, false);
#undef AMOE_LAUNCH
  return launch_rc();
}

int sample_check(const amoe_sample_args* a) {
  if (!a) return AMOE_ENULL;
  if (a->dtype != AMOE_F32 && a->dtype != AMOE_BF16 && a->dtype != AMOE_F16) return AMOE_EINVAL;
  if (a->rows < 0 || a->V < 1) return AMOE_EINVAL;
  if (!a->temperature && !(a->temperature_all >= 0 && a->temperature_all <= 3.4028234663852886e38)) return AMOE_EINVAL;
  if (!a->top_k && a->top_k_all < 0) return AMOE_EINVAL;
  if (!a->top_p && !(a->top_p_all >= 0 && a->top_p_all <= 1)) return AMOE_EINVAL;
  if (!a->min_p && !(a->min_p_all >= 0 && a->min_p_all <= 1)) return AMOE_EINVAL;
  // (threads of a launch are counted in 32 bits)
  return a->V > kSampleMaxV || a->rows >= INT64_C(1) << 22 ? AMOE_EUNSUPPORTED : AMOE_OK;
}

}  // namespace

}  // namespace amoe

using namespace amoe;

extern "C" size_t amoe_sample_args_bytes(void) { return sizeof(amoe_sample_args); }

extern "C" size_t amoe_sample_workspace(const amoe_sample_args*) { return 0; }

extern "C" int amoe_sample(const amoe_sample_args* a, void*, size_t, void* stream) {
  if (int rc = sample_check(a)) return rc;
  if (a->rows == 0) return AMOE_OK;
  if (!a->logits || !a->u || !a->ids) return AMOE_ENULL;
  if (a->rows > 1 && (a->ld < 0 || a->ld > INT64_C(1) << 40)) return AMOE_EINVAL;
  if (!aligned(a->logits, esize((int)a->dtype)) || !aligned(a->u, a->u_is_f64 ? 8 : 4) || !aligned(a->ids, 8) || !aligned(a->logprob, 4) ||
      !aligned(a->temperature, 4) || !aligned(a->top_p, 4) || !aligned(a->min_p, 4) || !aligned(a->top_k, a->top_k_is_i64 ? 8 : 4))
    return AMOE_EALIGN;
  SampleParams p{};
  p.logits = a->logits; p.ld = a->rows == 1 ? 0 : a->ld;
  p.u = a->u; p.u_f64 = a->u_is_f64 != 0;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p;
  p.top_k = a->top_k; p.top_k_i64 = a->top_k_is_i64 != 0;
  p.temperature_all = (float)a->temperature_all; p.top_p_all = (float)a->top_p_all; p.min_p_all = (float)a->min_p_all;
  p.top_k_all = a->top_k_all;
  p.ids = a->ids; p.logprob = a->logprob;
  p.rows = a->rows; p.V = (int)a->V;
  const bool cut = a->top_k || a->top_p || (a->top_k_all > 0 && a->top_k_all < a->V) || p.top_p_all < 1.f;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_sample<float>(p, cut, st)
         : a->dtype == AMOE_F16 ? launch_sample<f16_t>(p, cut, st)
                                : launch_sample<uint16_t>(p, cut, st);
}
