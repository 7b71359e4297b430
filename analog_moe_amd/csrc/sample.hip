// The choice of a token from a row of V logits and a given number u of [0, 1).
//   weight_i = exp((x_i - max) / temperature);  tokens rank by x, the lower index first among equals
//   kept: the first top_k; of these the shortest run from the top with at least top_p of their weight; of these weights of min_p
//   or more.  Drawn: in the order of the indices, the first up to which the kept ones weigh more than u times all of them.
//
// Weights are whole multiples of 2^-44 of the largest one (made in 64 bits, by a table of 2^(j / 32) and five terms of the series
// between), so that their sums are exact and the same in any order: what is drawn depends neither on how a row is shared out
// among threads nor on the order of the atomics that count.  A weight is off by up to 2^-44 of the largest and a row's sum by V times
// that: what is drawn is the definition's wherever u and top_p come no nearer to a border between tokens than this, and min_p no nearer
// to a weight than 2^-44.  (In fp32 a row of 10^5 logits would go to a neighbour about once in a thousand draws.)  What weighs less than
// 2^-45 of the largest is never drawn.
//
// The cut that top_k and top_p make in the ranking is found without a sort: tokens are counted, or weighed, by their
// distance from the largest in up to 2047 bins, and only those of the bin with the cut are ranked.
//
// Rows pass three times (their extremes, the bins, the sums), four where both cuts are made, from the caches behind the first.  Without a cut
// bound by the vector unit: 52 instructions a logit, 13 of them a weight's in 64 bits, keep it busy for 22 of 31 us (2048 rows of 8000, fp32).
// With cuts by that, by the bins' LDS atomics, of which many meet on a bank, and by waiting for both: 256 rows of 130001 fp32 logits 27 us
// for the largest alone, which is the reading, 56 with one pass of weights, 113 with top_p, 143 with top_k too (100 instructions a
// logit, 85 us, and 15 us of bank conflicts); 2048 rows of 8000 in bf16 31 and, with top_p, 72.
#include <amoe.h>

#include "host_util.h"
#include "wave_ops.h"

namespace amoe {

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
  char* work;                        // rows worked on in parts: what their launches leave for one another
  int parts;
};

constexpr int64_t kSampleMaxV = (1 << 20) - 1;       // (as many largest weights are less than 2^64)
// bins of a workgroup of NT threads, the last of which holds what is not looked at, and elements that it ranks at once
template <int NT> inline constexpr int kBins = 2 * NT;
constexpr int kUnits = 240;
constexpr int kMaxParts = 32;
constexpr int kPartList = 256;       // elements of the cut's bin that a part of a row can hand on
constexpr int kSteps = 32;           // table entries to a factor of two
constexpr int kCopies = 16;          // of the table, for 16 lanes side by side: random entries then meet on no bank
constexpr u64 kOne = 1ull << 44;
constexpr int kIndexBits = 20;

// A row of V elements: chunks of 16 bytes that begin on 4, and what is left before (one element) and behind them (less than a
// chunk), which lanes of the first wave hold one by one.  `per` groups of 64 chunks are a unit; units are counted from 1, what is
// before the chunks is unit 0 and what is behind them the last.  Chunks past the end read as zeros from a resource that ends with
// them, so that no load waits for a branch.
template <typename T, int W> struct SampleRow {
  static constexpr int C = Elem<T>::kChunk;
  BufRsrc chunks_at;
  int head, body, tail, groups, per, units, last;
  float edge;                        // of the first wave's lanes: lane 0 the element before the chunks, lanes 1 .. those behind
  int edge_index;
  __device__ __forceinline__ SampleRow(const T* row, int V) {
    head = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(row) & 2) ? 1 : 0;
    body = (V - head) / C;
    tail = V - head - body * C;
    groups = (body + 63) / 64;
    const int least = groups / (4 * W);
    per = (groups + kUnits - 1) / kUnits;
    if (per < 4) per = least >= 4 ? 4 : least > per ? least : per > 1 ? per : 1;
    units = (groups + per - 1) / per;
    last = units + 1;
    chunks_at = make_rsrc_sized(const_cast<T*>(row + head), (uint32_t)body * 16u);
    const int t = threadIdx.x;
    edge_index = t == 0 ? 0 : V - tail + t - 1;
    const bool there = t == 0 ? head == 1 : t <= tail;
    edge = there ? Elem<T>::load(row + edge_index) : -INFINITY;
    edge = edge == edge ? edge : -INFINITY;
  }
  __device__ __forceinline__ int start(int j) const { return head + j * C; }
  __device__ __forceinline__ int unit_of(int index) const {
    if (index < head) return 0;
    const int j = (index - head) / C;
    return j >= body ? last : 1 + j / 64 / per;
  }
  // f(values, index of the first, whether the chunk is in the row) for the chunks of groups [g, g_end) that are this lane's, done(unit)
  // after each unit; `low` for what is smaller, no number or not there
  template <class F, class Done>
  __device__ __forceinline__ void scan(float low, int g, int g_end, F f, Done done) const {
    constexpr int kAhead = sizeof(T) == 4 ? 8 : 4;
    const int lane = lane_id();
    int in_unit = g % per, unit = 1 + g / per;
    for (; g < g_end; g += kAhead) {
      Raw r[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) r[i] = buffer_load_b128(chunks_at, (uint32_t)((g + i) * 64 + lane) * 16u, 0);
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        if (g + i >= g_end) break;
        const int j = (g + i) * 64 + lane;
        const bool inside = j < body;
        float v[C];
        raw_unpack<T>(r[i], v);
#pragma unroll
        for (int e = 0; e < C; e++) v[e] = inside & (v[e] > low) ? v[e] : low;
        f(v, start(j), inside);
        if (++in_unit == per || g + i + 1 == g_end) {
          done(unit++);
          in_unit = 0;
        }
      }
    }
  }
  // units [first, end) of the chunks, counted from 0: a wave's lie next to each other
  template <class F, class Done>
  __device__ __forceinline__ void some(float low, int first, int end, F f, Done done) const {
    const int wave = wave_uniform(threadIdx.x >> 6), share = (end - first + W - 1) / W;
    const int u = first + wave * share, u_end = u + share < end ? u + share : end;
    if (u < u_end) scan(low, u * per, u_end * per < groups ? u_end * per : groups, f, done);
  }
  template <class F, class Done>
  __device__ __forceinline__ void all(float low, F f, Done done) const {
    some(low, 0, units, f, done);
  }
};

// The weight of an element, in multiples of 2^-44 of the largest: 2^(j / 32) from a table, e^z for the rest, |z| < 0.0109, by five
// terms of its series, which leave 2^-48.
struct SampleWeight {
  float low;                         // weighs nothing: this and what is smaller
  bool hot;                          // that is minus infinity alone: all numbers are within 66 temperatures of the largest
  double top, scale;                 // 32 log2(e) / temperature
  const double* table;               // the lane's copy of 2^(j / 32)
  __device__ __forceinline__ SampleWeight(float mx, float temperature, const double* tables) : top(mx), table(tables + (threadIdx.x & (kCopies - 1))) {
    // 33 temperatures down, and a float further (the rounding; where that is more, nothing but the largest weighs, and the scale is what
    // keeps 2^t a normal number)
    const float down = fminf(mx - 33.f * temperature, mx);
    const uint32_t b = as_u32(down);
    low = down == 0.f ? -1e-45f : as_f32(down > 0.f ? b - 1 : b + 1);
    hot = !(down > -3.402823466e38f);
    if (hot) low = -INFINITY;
    scale = kSteps * 1.44269504088896340736 / (double)temperature;
    const double most = 30000.0 / (top - (double)low);
    if (!(scale < most) && !hot) scale = most;
  }
  // of N elements, none below `low`: side by side, as each is a chain of 13 operations and a read
  template <int N>
  __device__ __forceinline__ void operator()(const float (&x)[N], u64 (&r)[N]) const {
    constexpr double kMagic = 6755399441055744.0;          // 1.5 * 2^52: whole numbers are its last bits
    constexpr double a = 0.69314718055994530942 / kSteps;
    double f[N], m[N], q[N];
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = ((double)x[e] - top) * scale;
#pragma unroll
    for (int e = 0; e < N; e++) m[e] = f[e] + kMagic;
    u64 bits[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int step = (int)(uint32_t)__builtin_bit_cast(u64, m[e]);
      bits[e] = __builtin_bit_cast(u64, table[(step & (kSteps - 1)) * kCopies]) + ((u64)(uint32_t)((step >> 5) * (1 << 20)) << 32);
    }
#pragma unroll
    for (int e = 0; e < N; e++) f[e] -= m[e] - kMagic;
#pragma unroll
    for (int e = 0; e < N; e++) q[e] = __builtin_fma(f[e], a * a * a * a * a / 120, a * a * a * a / 24);
#pragma unroll
    for (int e = 0; e < N; e++) q[e] = __builtin_fma(f[e], q[e], a * a * a / 6);
#pragma unroll
    for (int e = 0; e < N; e++) q[e] = __builtin_fma(f[e], q[e], a * a / 2);
#pragma unroll
    for (int e = 0; e < N; e++) q[e] = __builtin_fma(f[e], q[e], a);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const double w = __builtin_bit_cast(double, bits[e]);
      // (256 + w: the last bit counts 2^-44)
      r[e] = __builtin_bit_cast(u64, __builtin_fma(w * f[e], q[e], w) + 256.0) - __builtin_bit_cast(u64, 256.0);
    }
    if (hot) {
#pragma unroll
      for (int e = 0; e < N; e++) r[e] = x[e] == -INFINITY ? 0 : r[e];
    }
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const float one[1] = {x > low ? x : low};
    u64 r[1];
    (*this)(one, r);
    return r[0];
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

// What a workgroup shares beside the histogram.
template <int W> struct SampleShared {
  double table[kSteps * kCopies];
  u64 unit[kUnits + 2], group[32], wave_w[W];
  float unit_max[kUnits + 2], wave_max[W], wave_min[W];
  int wave_n[W], found, listed;
  u64 found_w, found_n, cut, rest;
};
template <int NT> struct SampleBins {
  uint32_t n[kBins<NT>];
  u64 w[kBins<NT>];
};
template <int NT> union SampleRanked {
  u64 list[kBins<NT>];
  SampleBins<NT> digit;
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
  // (those of the waves before, a lane each)
  const bool before = lane < wave;
  n = in - n + (int)wave_read((uint32_t)wave_scan(before ? sh.wave_n[lane] : 0), 63);
  w = iw - w + wave_total(before ? sh.wave_w[lane] : 0);
}

// The first bin up to which there are at least `target` (of what is counted, or weighed): sh.found (-1: there are fewer), and in
// found_n and found_w what is before it.
template <int NT>
__device__ __forceinline__ void sample_crossing(const SampleBins<NT>& bins, int size, bool by_weight, u64 target, SampleShared<NT / 64>& sh) {
  constexpr int P = 2;
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

// The list of `count` ranks, the largest first, and where `target` is reached in it (before_n elements and before_w of weight come
// before it): sh.cut, and in found_w the weight up to and with it.
template <int NT>
__device__ __forceinline__ void sample_sort(const SampleWeight& weight, int count, bool by_weight, u64 target, u64 before_n, u64 before_w,
                                            SampleRanked<NT>& r, SampleShared<NT / 64>& sh) {
  const int tid = threadIdx.x;
  int size = 2;
  while (size < count) size *= 2;
  for (int i = count + tid; i < size; i += NT) r.list[i] = 0;
  if (tid == 0) {
    sh.cut = 0;
    sh.found_w = before_w;
  }
  __syncthreads();
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
  constexpr int P = 2;
  u64 w[P], sum = 0;
  int none = 0;
#pragma unroll
  for (int i = 0; i < P; i++) {
    w[i] = tid * P + i < count ? weight(sample_value(r.list[tid * P + i])) : 0;
    sum += w[i];
  }
  sample_scan<NT / 64>(none, sum, sh);
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

// The same for one bin of the row, whatever number of elements (`count`) it has.  What is ranked is what was listed, and the digits end
// with the rank's: a row that is written to meanwhile gives some token of its own.
template <typename T, int NT, class Bin>
__device__ __forceinline__ void sample_refine(const SampleRow<T, NT / 64>& row, const SampleWeight& weight, Bin bin, int b, int count,
                                              bool by_weight, u64 target, u64 before_n, u64 before_w, SampleRanked<NT>& r,
                                              SampleShared<NT / 64>& sh) {
  constexpr int W = NT / 64, C = SampleRow<T, W>::C;
  const int tid = threadIdx.x;
  const auto none = [](int) AMOE_INLINE {};
  // too many to rank at once: by as many bits of their ranks at a time as there are bins
  constexpr int kDigit = NT == 1024 ? 11 : 9;
  static_assert(1 << kDigit == kBins<NT>, "a bin for each digit");
  int shift = 32 + kIndexBits;
  u64 prefix = 0;
  while (count > kBins<NT> && shift > 0) {
    const int next = shift > kDigit ? shift - kDigit : 0, size = 1 << (shift - next);
    __syncthreads();
    for (int i = tid; i < kBins<NT>; i += NT) {
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
        -INFINITY,
        [&](const float (&v)[C], int first, bool) AMOE_INLINE {
#pragma unroll
          for (int e = 0; e < C; e++) count_one(v[e], first + e);
        },
        none);
    if (tid < 64) count_one(row.edge, row.edge_index);
    __syncthreads();
    sample_crossing<NT>(r.digit, size, by_weight, target - (by_weight ? before_w : before_n), sh);
    const int d = sh.found < 0 ? size - 1 : sh.found;
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
    if (rank >> shift != prefix) return;
    const int n = atomicAdd(&sh.listed, 1);
    if (n < kBins<NT>) r.list[n] = rank;
  };
  row.all(
      -INFINITY,
      [&](const float (&v)[C], int first, bool) AMOE_INLINE {
#pragma unroll
        for (int e = 0; e < C; e++) list_one(v[e], first + e);
      },
      none);
  if (tid < 64) list_one(row.edge, row.edge_index);
  __syncthreads();
  sample_sort<NT>(weight, sh.listed < kBins<NT> ? sh.listed : kBins<NT>, by_weight, target, before_n, before_w, r, sh);
}

// the first lane whose sum passes; the first of all where none does, which only a row that is written to meanwhile can bring about
__device__ __forceinline__ int sample_first(bool passes) {
  const uint64_t lanes = wave_ballot(passes);
  return lanes ? ctz64(lanes) : 0;
}

// The element at which the sum of weights passes `target`, from the units' sums: weigh(value, index).  True for the thread that has
// it, one of them whatever the sums are, and its index is one of the row.  Every thread calls this.
template <typename T, int W, class Weigh>
__device__ __forceinline__ bool sample_find(const SampleRow<T, W>& row, float low, u64 target, Weigh weigh, SampleShared<W>& sh, int& index,
                                            float& value) {
  constexpr int C = SampleRow<T, W>::C, P = (kUnits + 2 + 63) / 64;
  const int lane = lane_id(), wave = wave_uniform(threadIdx.x >> 6);
  const auto none = [](int) AMOE_INLINE {};
  u64 part[P], mine = 0;
#pragma unroll
  for (int i = 0; i < P; i++) {
    part[i] = P * lane + i <= row.last ? sh.unit[P * lane + i] : 0;
    mine += part[i];
  }
  u64 run = wave_scan(mine);
  const int at = sample_first(run > target);
  run -= mine;
  int in = -1;
#pragma unroll
  for (int i = 0; i < P; i++) {
    if (in < 0 && run + part[i] > target) in = i;
    if (in < 0) run += part[i];
  }
  target -= wave_read(run, at);
  const int unit = P * at + (int)wave_read((uint32_t)(in < 0 ? 0 : in), at);
  const bool edges = unit == 0 || unit == row.last;
  const int g0 = (unit - 1) * row.per, g1 = g0 + row.per < row.groups ? g0 + row.per : row.groups;
  const auto group_sum = [&](int g, u64 (&w)[C], float (&x)[C], int& start) AMOE_INLINE {
    u64 s = 0;
    row.scan(
        low, g, g + 1,
        [&](const float (&v)[C], int first, bool) AMOE_INLINE {
#pragma unroll
          for (int e = 0; e < C; e++) {
            x[e] = v[e];
            w[e] = weigh(v[e], first + e);
            s += w[e];
          }
          start = first;
        },
        none);
    return s;
  };
  u64 w[C];
  float x[C];
  int start = 0;
  if (!edges) {
    for (int g = g0 + wave; g < g1; g += W) {
      const u64 s = wave_total(group_sum(g, w, x, start));
      if (lane == 0) sh.group[g - g0] = s;
    }
  }
  __syncthreads();
  if (wave != 0) return false;
  if (edges) {
    run = wave_scan((lane == 0) == (unit == 0) && row.edge != -INFINITY ? weigh(row.edge, row.edge_index) : 0);
    index = row.edge_index;
    value = row.edge;
    return lane == sample_first(run > target);
  }
  mine = lane < g1 - g0 ? sh.group[lane] : 0;
  run = wave_scan(mine);
  const int group = sample_first(run > target);
  target -= wave_read(run - mine, group);
  mine = group_sum(g0 + group, w, x, start);
  run = wave_scan(mine);
  const bool here = lane == sample_first(run > target);
  u64 sum = run - mine;
  bool found = false;
  index = start;
  value = x[0];
#pragma unroll
  for (int e = 0; e < C; e++) {
    sum += w[e];
    if (!found && sum > target) {
      found = true;
      index = start + e;
      value = x[e];
    }
  }
  return here;
}

// The number of [0, total) that u stands for
__device__ __forceinline__ u64 sample_target(double u, u64 total) {
  const double want = (u > 0.0 ? u : 0.0) * (double)total;
  const u64 target = want < (double)total ? (u64)want : total - 1;
  return target < total ? target : total - 1;
}

// What the launches for a row that is worked on in parts leave for one another.
struct SamplePart {
  u64 list[2][kPartList];
  float mx, mn;
  int listed[2];
};
struct SampleWork {
  SampleBins<1024> hist;             // cleared by the first launch, added to by the parts (whole numbers: in any order)
  u64 rest, unit[kUnits + 2];
  float unit_max[kUnits + 2];
  SamplePart part[1];                // as many as there are
};
__device__ __host__ inline size_t sample_work_bytes(int parts) { return sizeof(SampleWork) + (size_t)(parts - 1) * sizeof(SamplePart); }

// The launches for a row: all in one, or, of a row in parts, its extremes, its bins, the list of top_k's bin (where top_p needs its
// weight), sums and the list of the cut's bin, and the rest by one workgroup again.
enum SampleStage { kAll, kExtremes, kHistogram, kTopList, kSums, kFinish };

template <typename T, int NT, bool CUT, int STAGE>
__global__ __launch_bounds__(NT, 4) void sample_kernel(SampleParams p) {
  constexpr int W = NT / 64, C = Elem<T>::kChunk;
  constexpr bool kParted = STAGE != kAll;
  __shared__ SampleShared<W> sh;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_uniform(tid >> 6);
  const int parts = kParted && STAGE != kFinish ? p.parts : 1, part = (int)(blockIdx.x % (unsigned)parts);
  const int64_t at = blockIdx.x / (unsigned)parts;
  const SampleRow<T, W> row(static_cast<const T*>(p.logits) + at * p.ld, p.V);
  SampleWork* const work = kParted ? reinterpret_cast<SampleWork*>(p.work + at * (int64_t)sample_work_bytes(p.parts)) : nullptr;
  // this workgroup's units; the edges are the first part's
  const int first_unit = row.units * part / parts, end_unit = row.units * (part + 1) / parts;
  const bool has_edges = part == 0 && wave == 0;
  const float temperature = p.temperature ? p.temperature[at] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[at] : p.top_p_all, min_p = p.min_p ? p.min_p[at] : p.min_p_all;
  const int64_t top_k = !p.top_k ? p.top_k_all : p.top_k_i64 ? static_cast<const int64_t*>(p.top_k)[at] : static_cast<const int32_t*>(p.top_k)[at];
  const double u = p.u_f64 ? static_cast<const double*>(p.u)[at] : (double)static_cast<const float*>(p.u)[at];
  const bool greedy = !(temperature > 0.f), by_k = CUT && top_k > 0 && top_k < p.V, by_p = CUT && top_p < 1.f;
  if (STAGE != kExtremes)
    for (int i = tid; i < kSteps * kCopies; i += NT) sh.table[i] = ::exp2((double)(i / kCopies) / kSteps);

  // ---- the extremes
  float mx = -INFINITY, mn = INFINITY;
  if constexpr (STAGE == kAll || STAGE == kExtremes) {
    float unit_max = -INFINITY;
    row.some(
        -INFINITY, first_unit, end_unit,
        [&](const float (&v)[C], int, bool inside) AMOE_INLINE {
          float lo = v[0];
#pragma unroll
          for (int e = 0; e < C; e++) {
            unit_max = fmaxf(unit_max, v[e]);
            if (CUT) lo = fminf(lo, v[e]);
          }
          if (CUT) mn = inside ? fminf(mn, lo) : mn;
        },
        [&](int unit) AMOE_INLINE {
          unit_max = wave_largest(unit_max);
          if (lane == 0) {
            if constexpr (kParted) work->unit_max[unit] = unit_max;
            else sh.unit_max[unit] = unit_max;
          }
          mx = fmaxf(mx, unit_max);
          unit_max = -INFINITY;
        });
    if (has_edges) {
      const float behind = wave_largest(lane == 0 ? -INFINITY : row.edge);
      if (lane == 0) {
        float* const to = kParted ? work->unit_max : sh.unit_max;
        to[0] = row.edge;
        to[row.last] = behind;
      }
      mx = fmaxf(fmaxf(mx, behind), as_f32(wave_read(as_u32(row.edge), 0)));
      if (CUT && row.edge != -INFINITY) mn = fminf(mn, row.edge);
    }
    if (CUT) mn = -wave_largest(-mn);
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
    if constexpr (STAGE == kExtremes) {
      if constexpr (CUT) {
        for (int i = part * NT + tid; i < kBins<NT>; i += parts * NT) {
          work->hist.n[i] = 0;
          work->hist.w[i] = 0;
        }
        if (part == 0 && tid == 0) work->rest = 0;
      }
      if (tid == 0) {
        work->part[part].mx = mx;
        work->part[part].mn = mn;
      }
      return;
    }
  } else {
    // (a lane per part: one after the other they are a round trip to memory each)
    mx = wave_largest(lane < p.parts ? work->part[lane].mx : -INFINITY);
    mn = -wave_largest(lane < p.parts ? -work->part[lane].mn : -INFINITY);
    if (STAGE == kFinish)
      for (int i = tid; i <= row.last; i += NT) {
        sh.unit[i] = work->unit[i];
        sh.unit_max[i] = work->unit_max[i];
      }
    __syncthreads();
  }
  int index = 0;
  float value = 0.f;
  if (mx == -INFINITY) {
    if ((STAGE == kAll || STAGE == kFinish) && tid == 0) {
      p.ids[at] = -1;
      if (p.logprob) p.logprob[at] = -INFINITY;
    }
    return;
  }

  // ---- only those as large as the largest weigh, and all the same
  if (greedy || mx == INFINITY) {
    if (STAGE != kAll && STAGE != kFinish) return;
    const auto weigh = [&](float x, int) AMOE_INLINE { return (u64)(x == mx); };
    for (int i = 1 + wave; i < row.last; i += W) {
      u64 s = 0;
      if (sh.unit_max[i] == mx) {
        const int g = (i - 1) * row.per, end = g + row.per;
        row.scan(
            -INFINITY, g, end < row.groups ? end : row.groups,
            [&](const float (&v)[C], int, bool) AMOE_INLINE {
#pragma unroll
              for (int e = 0; e < C; e++) s += weigh(v[e], 0);
            },
            [](int) AMOE_INLINE {});
        s = wave_total(s);
      }
      if (lane == 0) sh.unit[i] = s;
    }
    if (wave == 0) {
      const u64 behind = wave_total(lane != 0 && row.edge == mx);
      if (lane == 0) {
        sh.unit[0] = row.edge == mx;
        sh.unit[row.last] = behind;
      }
    }
    __syncthreads();
    u64 kept = 1;
    if (!greedy) {
      kept = 0;
      for (int i = lane; i <= row.last; i += 64) kept += sh.unit[i];
      kept = wave_total(kept);
      if (top_k > 0 && (u64)top_k < kept) kept = (u64)top_k;
      if (top_p < 1.f) {
        const double share = top_p > 0.f ? __builtin_ceil((double)top_p * (double)kept) : 1.0;
        kept = share < 1.0 ? 1 : (u64)share;
      }
    }
    if (sample_find<T, W>(row, -INFINITY, greedy ? 0 : sample_target(u, kept), weigh, sh, index, value)) {
      p.ids[at] = index;
      if (p.logprob) p.logprob[at] = greedy ? 0.f : (float)-::log((double)kept);
    }
    return;
  }

  const SampleWeight weight(mx, temperature, sh.table);
  const u64 least = min_p > 0.f ? (u64)__builtin_ceil((double)fminf(min_p, 1.f) * (double)kOne) : 0;
  u64* const unit_to = STAGE == kSums ? work->unit : sh.unit;
  // ---- what is kept: ranks of `cut` and more
  u64 cut = 0;
  bool summed = STAGE == kFinish;
  if constexpr (CUT) {
    __shared__ SampleBins<NT> hist;
    __shared__ SampleRanked<NT> ranked;
    if (by_k || by_p) {
      if (STAGE == kTopList && !(by_k && by_p)) return;
      // Bins are equal intervals of the distance to the largest, up to where tokens occur, weigh anything and, without top_k, may be
      // kept: all that weigh less than (1 - top_p) / V are together less than what top_p may leave out.  (Half the distances: they
      // may be twice the largest float.)
      const float half = 0.5f * mx;
      float reach = fminf(fmaf(-0.5f, mn, half), 16.25f * temperature);
      if (!by_k) reach = fminf(reach, 0.3466f * temperature * (fast_log2((float)p.V) - fast_log2(1.f - fmaxf(top_p, 0.f)) + 1.f));
      const float step = reach > 0.f ? fminf((kBins<NT> - 2) / reach, 3.402823466e38f) : 0.f;
      // (What weighs nothing is in the last bin by itself: where the largest is all there is, or the distances are subnormal, its distance
      // says no such thing, and what a row is padded with would count as tokens.)
      const float low = weight.low;
      const auto bin = [=](float x) AMOE_INLINE { return x > low ? (int)fminf(fmaf(-0.5f, x, half) * step, (float)(kBins<NT> - 1)) : kBins<NT> - 1; };
      if (tid == 0) sh.rest = 0;
      if constexpr (STAGE == kAll || STAGE == kHistogram) {
        for (int i = tid; i < kBins<NT>; i += NT) {
          hist.n[i] = 0;
          hist.w[i] = 0;
        }
        __syncthreads();
        u64 rest = 0;
        const auto count = [&](const auto& v) AMOE_INLINE {
          constexpr int N = sizeof(v) / sizeof(v[0]);
          int b[N];
#pragma unroll
          for (int e = 0; e < N; e++) b[e] = bin(v[e]);
          if (by_p) {
            u64 w[N];
            weight(v, w);
#pragma unroll
            for (int e = 0; e < N; e++) {
              if (b[e] < kBins<NT> - 1) atomicAdd(&hist.w[b[e]], w[e]);
              else rest += w[e];
            }
          }
          if (by_k) {
#pragma unroll
            for (int e = 0; e < N; e++)
              if (b[e] < kBins<NT> - 1) atomicAdd(&hist.n[b[e]], 1u);
          }
        };
        row.some(
            weight.low, first_unit, end_unit, [&](const float (&v)[C], int, bool) AMOE_INLINE { count(v); }, [](int) AMOE_INLINE {});
        if (has_edges && row.edge > weight.low) {
          const float one[1] = {row.edge};
          count(one);
        }
        if (by_p) {
          rest = wave_total(rest);
          if (lane == 0 && rest) atomicAdd(&sh.rest, rest);
        }
        __syncthreads();
        if constexpr (STAGE == kHistogram) {
          for (int i = tid; i < kBins<NT> - 1; i += NT) {
            if (hist.n[i]) atomicAdd(&work->hist.n[i], hist.n[i]);
            if (hist.w[i]) atomicAdd(&work->hist.w[i], hist.w[i]);
          }
          if (tid == 0 && sh.rest) atomicAdd(&work->rest, sh.rest);
          return;
        }
      } else if constexpr (NT == 1024) {
        for (int i = tid; i < kBins<NT>; i += NT) {
          hist.n[i] = work->hist.n[i];
          hist.w[i] = work->hist.w[i];
        }
        if (tid == 0) sh.rest = work->rest;
        __syncthreads();
      }
      // the elements of bin b, from the parts' lists (l: of top_k's bin or the cut's); false if some did not fit
      const auto gather = [&](int l, int& count) AMOE_INLINE {
        const int mine = lane < p.parts ? work->part[lane].listed[l] : 0, before = wave_scan(mine) - mine;
        count = (int)wave_read((uint32_t)(before + mine), 63);
        // (as unsigned: a part of a row that is written to meanwhile may have found no bin and left no number)
        if (wave_ballot((uint32_t)mine > (uint32_t)kPartList) != 0 || count > kBins<NT>) return false;
        for (int j = wave; j < p.parts; j += W) {
          const int m = (int)wave_read((uint32_t)mine, j), to = (int)wave_read((uint32_t)before, j);
          for (int i = lane; i < m; i += 64) ranked.list[to + i] = work->part[j].list[l][i];
        }
        __syncthreads();
        return true;
      };
      u64 total = 0, target = (u64)top_k;
      int b = -1;
      if (by_k) {
        sample_crossing<NT>(hist, kBins<NT> - 1, false, target, sh);
        b = sh.found;
        if (b >= 0 && by_p && STAGE != kTopList) {
          const u64 before_n = sh.found_n, before_w = sh.found_w;
          int n = (int)hist.n[b];
          if (STAGE != kAll && gather(0, n)) sample_sort<NT>(weight, n, false, target, before_n, before_w, ranked, sh);
          else sample_refine<T, NT>(row, weight, bin, b, n, false, target, before_n, before_w, ranked, sh);
          cut = sh.cut;
          total = sh.found_w;
        }
      }
      if (by_p && STAGE != kTopList) {
        if (b < 0) {
          u64 w = 0;
          for (int i = tid; i < kBins<NT>; i += NT) w += hist.w[i];
          w = wave_total(w);
          if (lane == 0 && w) atomicAdd(&sh.rest, w);
          __syncthreads();
          total = sh.rest;
        }
        const double share = top_p > 0.f ? __builtin_ceil((double)top_p * (double)total) : 1.0;
        target = share < 1.0 ? 1 : (u64)share;
        __syncthreads();
        sample_crossing<NT>(hist, kBins<NT> - 1, true, target, sh);
        b = sh.found;
      }
      if (b >= 0) {
        // one more pass: the sums of the bins before b, and a list of b's elements
        const u64 before_n = sh.found_n, before_w = sh.found_w;
        if constexpr (STAGE != kFinish) {
          if (tid == 0) sh.listed = 0;
          __syncthreads();
          constexpr int kRoom = STAGE == kAll ? kBins<NT> : kPartList;
          u64 s = 0;
          const auto take = [&](const auto& v, int first) AMOE_INLINE -> u64 {
            constexpr int N = sizeof(v) / sizeof(v[0]);
            int in[N];
            bool any = false;
#pragma unroll
            for (int e = 0; e < N; e++) {
              in[e] = bin(v[e]);
              any = any | (STAGE == kTopList ? in[e] == b : in[e] <= b);
            }
            if (!any) return 0;
#pragma unroll
            for (int e = 0; e < N; e++)
              if (in[e] == b) {
                const int n = atomicAdd(&sh.listed, 1);
                if (n < kRoom) ranked.list[n] = sample_rank(v[e], first + e);
              }
            if (STAGE == kTopList) return 0;
            u64 w[N], sum = 0;
            weight(v, w);
#pragma unroll
            for (int e = 0; e < N; e++) sum += (in[e] < b) & (w[e] >= least) ? w[e] : 0;
            return sum;
          };
          row.some(
              weight.low, first_unit, end_unit, [&](const float (&v)[C], int first, bool) AMOE_INLINE { s += take(v, first); },
              [&](int unit) AMOE_INLINE {
                if (STAGE != kTopList) {
                  s = wave_total(s);
                  if (lane == 0) unit_to[unit] = s;
                }
                s = 0;
              });
          if (has_edges) {
            const float one[1] = {row.edge};
            const u64 w = row.edge > weight.low ? take(one, row.edge_index) : 0, behind = wave_total(lane == 0 ? 0 : w);
            if (lane == 0 && STAGE != kTopList) {
              unit_to[0] = w;
              unit_to[row.last] = behind;
            }
          }
          __syncthreads();
          if constexpr (STAGE != kAll) {
            constexpr int l = STAGE == kTopList ? 0 : 1;
            SamplePart& to = work->part[part];
            const int n = sh.listed;
            for (int i = tid; i < (n < kRoom ? n : kRoom); i += NT) to.list[l][i] = ranked.list[i];
            if (tid == 0) to.listed[l] = n;
            return;
          }
        }
        int listed = sh.listed;
        bool fit = listed <= kBins<NT>;
        if constexpr (STAGE == kFinish) fit = gather(1, listed);
        if (fit) {
          sample_sort<NT>(weight, listed, by_p, target, before_n, before_w, ranked, sh);
          cut = sh.cut;
          for (int i = tid; i < listed; i += NT) {
            const u64 rank = ranked.list[i], w = weight(sample_value(rank));
            if (rank >= cut && w >= least) atomicAdd(&sh.unit[row.unit_of(sample_index(rank))], w);
          }
          summed = true;
        } else {
          sample_refine<T, NT>(row, weight, bin, b, listed, by_p, target, before_n, before_w, ranked, sh);
          cut = sh.cut;
          summed = false;
        }
      }
    }
  }
  if (STAGE == kHistogram || STAGE == kTopList) return;
  const float cut_x = cut ? sample_value(cut) : -INFINITY;
  const int cut_i = cut ? sample_index(cut) : p.V;
  const auto weigh = [&](float x, int i) AMOE_INLINE -> u64 {
    const bool keep = (x > cut_x) | ((x == cut_x) & (i <= cut_i));
    const u64 w = weight(x);
    return keep & (w >= least) ? w : 0;
  };
  __syncthreads();                                    // (the table, where nothing was cut)
  if (!summed) {
    u64 s = 0;
    const bool every = !CUT || cut == 0;
    row.some(
        weight.low, first_unit, end_unit,
        [&](const float (&v)[C], int first, bool) AMOE_INLINE {
          u64 w[C];
          weight(v, w);
          if (least) {
#pragma unroll
            for (int e = 0; e < C; e++) w[e] = w[e] >= least ? w[e] : 0;
          }
          if (!every) {
#pragma unroll
            for (int e = 0; e < C; e++) w[e] = (v[e] > cut_x) | ((v[e] == cut_x) & (first + e <= cut_i)) ? w[e] : 0;
          }
#pragma unroll
          for (int e = 0; e < C; e++) s += w[e];
        },
        [&](int unit) AMOE_INLINE {
          s = wave_total(s);
          if (lane == 0) unit_to[unit] = s;
          s = 0;
        });
    if (has_edges) {
      const u64 w = row.edge != -INFINITY ? weigh(row.edge, row.edge_index) : 0, behind = wave_total(lane == 0 ? 0 : w);
      if (lane == 0) {
        unit_to[0] = w;
        unit_to[row.last] = behind;
      }
    }
    __syncthreads();
  }
  if (STAGE == kSums) return;
  u64 total = 0;
  for (int i = lane; i <= row.last; i += 64) total += sh.unit[i];
  total = wave_total(total);
  if (!sample_find<T, W>(row, weight.low, sample_target(u, total), weigh, sh, index, value)) return;
  p.ids[at] = index;
  if (p.logprob) p.logprob[at] = (float)(((double)value - (double)mx) / (double)temperature - ::log((double)total * 0x1p-44));
}

namespace {

// Parts that a row is worked on in, 1: all in one launch: as many as there are CUs for, of 4096 elements or more, if they are four.
// Measured (us, one launch / parts, fp32 or bf16): 8 rows of 130001 with top_p 92 / 41, without a cut 36 / 17, the largest of each
// 12 / 17; 64 of 50001 51 / 44, 21 / 17, 10 / 17 (what is launched may not depend on what the temperatures are).
int sample_parts(const amoe_sample_args* a) {
  const int64_t most = num_compute_units() / (a->rows < 1 ? 1 : a->rows), n = a->V / 4096;
  const int64_t parts = n < most ? n : most;
  return (int)(parts < 4 ? 1 : parts > kMaxParts ? kMaxParts : parts);
}

// 256 threads for short rows, and for longer ones where there are more of them than CUs; not past 32768, where too many tokens would
// share one of their bins, a quarter as many.  Measured (us, 256 / 1024 threads, top_p 0.95, bf16): 64 rows of 2000 14.5 / 15.0; 1 of 8000 21.9 / 17.7,
// 100 23.3 / 19.2, 300 26.3 / 35.7, 2048 70 / 141; 512 of 16000 41 / 48; 512 of 32000 72 / 71, 2048 193 / 274.
template <typename T, bool CUT>
int launch_sample_cut(const SampleParams& p, bool both, hipStream_t st) {
  const dim3 grid((unsigned)p.rows), parts((unsigned)(p.rows * p.parts)), block(1024);
  if (p.parts > 1) {
    hipLaunchKernelGGL((&sample_kernel<T, 1024, CUT, kExtremes>), parts, block, 0, st, p);
    if constexpr (CUT) {
      hipLaunchKernelGGL((&sample_kernel<T, 1024, true, kHistogram>), parts, block, 0, st, p);
      if (both) hipLaunchKernelGGL((&sample_kernel<T, 1024, true, kTopList>), parts, block, 0, st, p);
    }
    hipLaunchKernelGGL((&sample_kernel<T, 1024, CUT, kSums>), parts, block, 0, st, p);
    hipLaunchKernelGGL((&sample_kernel<T, 1024, CUT, kFinish>), grid, block, 0, st, p);
  } else if (p.V <= 4096 || (p.rows > num_compute_units() && p.V <= 32768)) {
    hipLaunchKernelGGL((&sample_kernel<T, 256, CUT, kAll>), grid, dim3(256), 0, st, p);
  } else {
    hipLaunchKernelGGL((&sample_kernel<T, 1024, CUT, kAll>), grid, block, 0, st, p);
  }
  return launch_rc();
}
template <typename T>
int launch_sample(const SampleParams& p, bool cut, bool both, hipStream_t st) {
  return cut ? launch_sample_cut<T, true>(p, both, st) : launch_sample_cut<T, false>(p, both, st);
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

extern "C" size_t amoe_sample_workspace(const amoe_sample_args* a) {
  if (sample_check(a) || a->rows == 0) return 0;
  const int parts = sample_parts(a);
  return parts > 1 ? (size_t)a->rows * sample_work_bytes(parts) : 0;
}

extern "C" int amoe_sample(const amoe_sample_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = sample_check(a)) return rc;
  if (a->rows == 0) return AMOE_OK;
  if (!a->logits || !a->u || !a->ids) return AMOE_ENULL;
  if (a->rows > 1 && (a->ld < 0 || a->ld > INT64_C(1) << 40)) return AMOE_EINVAL;
  if (!aligned(a->logits, esize((int)a->dtype)) || !aligned(a->u, a->u_is_f64 ? 8 : 4) || !aligned(a->ids, 8) || !aligned(a->logprob, 4) ||
      !aligned(a->temperature, 4) || !aligned(a->top_p, 4) || !aligned(a->min_p, 4) || !aligned(a->top_k, a->top_k_is_i64 ? 8 : 4))
    return AMOE_EALIGN;
  const size_t need = amoe_sample_workspace(a);
  if (need && !workspace) return AMOE_ENULL;
  if (workspace_bytes < need) return AMOE_EWORKSPACE;
  if (need && !aligned(workspace, 8)) return AMOE_EALIGN;
  SampleParams p{};
  p.work = static_cast<char*>(workspace);
  p.parts = sample_parts(a);
  p.logits = a->logits; p.ld = a->rows == 1 ? 0 : a->ld;
  p.u = a->u; p.u_f64 = a->u_is_f64 != 0;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p;
  p.top_k = a->top_k; p.top_k_i64 = a->top_k_is_i64 != 0;
  p.temperature_all = (float)a->temperature_all; p.top_p_all = (float)a->top_p_all; p.min_p_all = (float)a->min_p_all;
  p.top_k_all = a->top_k_all;
  p.ids = a->ids; p.logprob = a->logprob;
  p.rows = a->rows; p.V = (int)a->V;
  const bool by_k = a->top_k || (a->top_k_all > 0 && a->top_k_all < a->V), by_p = a->top_p || p.top_p_all < 1.f;
  const bool cut = by_k || by_p, both = by_k && by_p;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_sample<float>(p, cut, both, st)
         : a->dtype == AMOE_F16 ? launch_sample<f16_t>(p, cut, both, st)
                                : launch_sample<uint16_t>(p, cut, both, st);
}
