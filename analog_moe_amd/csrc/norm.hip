// Layer norm of rows of D elements, of a sum of two tensors if asked, and its gradients.
//   s = x + residual (rounded to the type);  h = (s - mean) * inv,  inv = 1 / sqrt(var + eps);  y = h * w + b
//   a = gy * w;  dx = gs + inv * (a - sum(a) / D - h * sum(a h) / D);  dw = sum over rows of gy h,  db = sum over rows of gy
//
// A row lies in the registers of NT threads, so that memory sees it once.  Its mean is summed first and the squares of what differs
// from it then; that sum carries the differences themselves along, whose own mean is what the rounding of the first one left (rows
// far from zero: their mean is exact only to 2^-24 of itself, which may be as large as the row's spread).  Bound by memory: 4096 rows
// of 8192 in fp32, with the sum, 92 us forward and 114 + 5 backward for 537 MB each (5.8 and 4.5 TB/s, a large copy reaches 5.1); 16384
// of 1024 in bf16 24 and 26 + 4 us for 134 MB each, a part of it from the cache behind the L2.
#include <amoe.h>

#include "host_util.h"
#include "wave_ops.h"

namespace amoe {

struct NormParams {
  const void *x, *res, *w, *b;       // [rows, D] with row strides (elements), [D] or null
  int64_t ldx, ldr;
  void *y, *sum;                     // [rows, D]; sum null: nothing is added
  float* stats;                      // [rows][3]: mean, what it is off by, inv.  May be null in the forward pass
  const void *gy, *gs;               // gradients of y and of s; gs may be null
  int64_t ldgy, ldgs;
  void *dx, *dw, *db;
  float* part;                       // [workgroups][2][D]: sums of dw and db; null: not wanted
  int64_t rows;
  int D, w_f32, parts;
  float eps;
};

constexpr int kNormStats = 3;
constexpr int64_t kNormMaxD = 32768;

// chunk c of a row that begins at p: elements past D read as zeros
template <typename T, bool VEC>
__device__ __forceinline__ Raw norm_load(const T* p, int c, int D) {
  typedef u32x4 __attribute__((aligned(4))) RawU;
  constexpr int C = Elem<T>::kChunk;
  const int n = D - c * C;
  if (n <= 0) return raw_zero();
  p += c * C;
  if constexpr (VEC) return *reinterpret_cast<const Raw*>(p);
  if (n >= C && (reinterpret_cast<uintptr_t>(p) & 3) == 0) return *reinterpret_cast<const RawU*>(p);
  return raw_load<T>(p, n, false);
}
template <typename T, bool VEC>
__device__ __forceinline__ void norm_store(T* p, int c, int D, const float (&v)[Elem<T>::kChunk]) {
  typedef u32x4 __attribute__((aligned(4))) RawU;
  constexpr int C = Elem<T>::kChunk;
  const int n = D - c * C;
  if (n <= 0) return;
  p += c * C;
  const Raw r = raw_pack<T>(v);
  if constexpr (VEC) {
    *reinterpret_cast<Raw*>(p) = r;
  } else if (n >= C && (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
    *reinterpret_cast<RawU*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < C; e++)
      if (e < n) p[e] = Elem<T>::cvt(v[e]);
  }
}
// the same chunk of a weight, of the rows' type or fp32; `none` where there is no weight
template <typename T, bool VEC>
__device__ __forceinline__ void norm_weight(const void* w, int f32, int c, int D, float none, float (&v)[Elem<T>::kChunk]) {
  constexpr int C = Elem<T>::kChunk;
  const int n = D - c * C;
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < C; e++) v[e] = none;
  } else if (sizeof(T) == 2 && f32) {
#pragma unroll
    for (int e = 0; e < C; e += 4) {
      float q[4];
      load4<float>(static_cast<const float*>(w) + c * C + e, q, n - e, VEC);
#pragma unroll
      for (int j = 0; j < 4; j++) v[e + j] = q[j];
    }
  } else {
    raw_unpack<T>(norm_load<T, VEC>(static_cast<const T*>(w), c, D), v);
  }
}

// Sums over the NT threads of a row, the same in all of them.  lds: [2][waves]; `turn` alternates from call to call, so that one
// barrier each does.
template <int NT>
__device__ __forceinline__ void norm_sum2(float& a, float& b, float (*lds)[2][16], int turn) {
  a = lanes_sum<(NT < 64 ? NT : 64)>(a);
  b = lanes_sum<(NT < 64 ? NT : 64)>(b);
  if constexpr (NT > 64) {
    constexpr int W = NT / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if (lane_id() == 0) {
      lds[turn][0][wave] = a;
      lds[turn][1][wave] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; i++) {
      a += lds[turn][0][first + i];
      b += lds[turn][1][first + i];
    }
  }
}

template <typename T, int NT, int PER, bool VEC>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_fwd_kernel(NormParams p) {
  constexpr int BT = NT < 256 ? 256 : NT, C = Elem<T>::kChunk;
  __shared__ float lds[2][2][16];
  const int t = threadIdx.x % NT;
  const int64_t row0 = (int64_t)blockIdx.x * (BT / NT) + threadIdx.x / NT;
  const bool ok = row0 < p.rows;
  const int64_t row = ok ? row0 : p.rows - 1;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float v[PER][C];
  Raw rx[PER], rr[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) rx[j] = norm_load<T, VEC>(x, t + j * NT, p.D);
  if (p.res) {
    const T* r = static_cast<const T*>(p.res) + row * p.ldr;
#pragma unroll
    for (int j = 0; j < PER; j++) rr[j] = norm_load<T, VEC>(r, t + j * NT, p.D);
#pragma unroll
    for (int j = 0; j < PER; j++) {
      float a[C], b[C];
      raw_unpack<T>(rx[j], a);
      raw_unpack<T>(rr[j], b);
#pragma unroll
      for (int e = 0; e < C; e++) a[e] += b[e];
      if (ok) norm_store<T, VEC>(static_cast<T*>(p.sum) + row * p.D, t + j * NT, p.D, a);
      rx[j] = raw_pack<T>(a);          // (rounded, as it is stored: what the backward pass reads is what was normalised)
    }
  }
  // (in units of the widest row: the sum of any finite row is finite, and the same bits otherwise)
  constexpr float kUnit = 1.f / (float)kNormMaxD;
  float sum = 0.f, sq = 0.f;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    raw_unpack<T>(rx[j], v[j]);
#pragma unroll
    for (int e = 0; e < C; e++) sum = fmaf(v[j][e], kUnit, sum);
  }
  norm_sum2<NT>(sum, sq, lds, 0);
  const float mean = sum / ((float)p.D * kUnit);
  float off = 0.f;
  sq = 0.f;
#pragma unroll
  for (int j = 0; j < PER; j++)
#pragma unroll
    for (int e = 0; e < C; e++) {
      const float d = (t + j * NT) * C + e < p.D ? v[j][e] - mean : 0.f;
      v[j][e] = d;
      off += d;
      sq = fmaf(d, d, sq);
    }
  norm_sum2<NT>(off, sq, lds, 1);
  off /= (float)p.D;
  const float var = fmaxf(fmaf(-off, off, sq / (float)p.D), 0.f), inv = 1.f / sqrtf(var + p.eps);
  if (p.stats && ok && t == 0) {
    p.stats[kNormStats * row] = mean;
    p.stats[kNormStats * row + 1] = off;
    p.stats[kNormStats * row + 2] = inv;
  }
  T* y = static_cast<T*>(p.y) + row * p.D;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    float w[C], b[C];
    norm_weight<T, VEC>(p.w, p.w_f32, t + j * NT, p.D, 1.f, w);
    norm_weight<T, VEC>(p.b, p.w_f32, t + j * NT, p.D, 0.f, b);
#pragma unroll
    for (int e = 0; e < C; e++) v[j][e] = fmaf((v[j][e] - off) * inv, w[e], b[e]);
    if (ok) norm_store<T, VEC>(y, t + j * NT, p.D, v[j]);
  }
}

// Rows go round the workgroups, and every thread keeps the sums of dw and db for its columns over all its rows; a workgroup's
// groups of threads are joined in LDS, the workgroups' sums by norm_reduce_kernel.  No atomics: the same bits every time.
template <int NT> inline constexpr int kNormBwdThreads = NT <= 256 ? 512 : NT;
template <typename T, int NT, int PER, bool VEC>
__global__ __launch_bounds__(kNormBwdThreads<NT>) void norm_bwd_kernel(NormParams p) {
  constexpr int BT = kNormBwdThreads<NT>, C = Elem<T>::kChunk, groups = BT / NT, cols = NT * PER * C;
  __shared__ float lds[2][2][16];
  __shared__ __align__(16) float lds_w[groups > 1 ? groups : 1][groups > 1 ? cols : 4];
  // Rows that all threads work on leave no registers for the weights, which come from the cache every time, and few for what comes
  // next: their sums are kept in LDS, where there is room, by the thread that has the columns, and the next row is asked for before
  // the sums of this one (2048 rows of 16384, bf16: 84 us, 3.2 TB/s).
  constexpr bool kHeld = NT <= 256 && PER <= 2, kInLds = NT == 1024 && 2 * cols * 4 <= 128 << 10, kAhead = NT == 1024 && PER <= 2;
  __shared__ __align__(16) float lds_sums[kInLds ? 2 : 1][kInLds ? cols : 4];
  const int t = threadIdx.x % NT, g = threadIdx.x / NT;
  float w[kHeld ? PER : 1][C], dw[kInLds ? 1 : PER][C], db[kInLds ? 1 : PER][C];
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if constexpr (kHeld) norm_weight<T, VEC>(p.w, p.w_f32, t + j * NT, p.D, 1.f, w[j]);
#pragma unroll
    for (int e = 0; e < C; e++) {
      dw[kInLds ? 0 : j][e] = db[kInLds ? 0 : j][e] = 0.f;
      if constexpr (kInLds) lds_sums[0][(t + j * NT) * C + e] = lds_sums[1][(t + j * NT) * C + e] = 0.f;
    }
  }
  Raw rx[PER], rg[PER], rs[PER], nx[kAhead ? PER : 1], ng[kAhead ? PER : 1], ns[kAhead ? PER : 1];
  const auto ask = [&](int64_t r0, Raw (&x)[kAhead ? PER : 1], Raw (&gy)[kAhead ? PER : 1], Raw (&gs)[kAhead ? PER : 1]) __attribute__((always_inline)) {
    const int64_t row = r0 + g < p.rows ? r0 + g : p.rows - 1;
#pragma unroll
    for (int j = 0; j < (kAhead ? PER : 1); j++) {
      x[j] = norm_load<T, VEC>(static_cast<const T*>(p.x) + row * p.ldx, t + j * NT, p.D);
      gy[j] = norm_load<T, VEC>(static_cast<const T*>(p.gy) + row * p.ldgy, t + j * NT, p.D);
      gs[j] = p.gs ? norm_load<T, VEC>(static_cast<const T*>(p.gs) + row * p.ldgs, t + j * NT, p.D) : raw_zero();
    }
  };
  if constexpr (kAhead) ask((int64_t)blockIdx.x * groups, nx, ng, ns);
  const float per_row = 1.f / (float)p.D;
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < p.rows; r0 += (int64_t)gridDim.x * groups) {
    const bool ok = r0 + g < p.rows;
    const int64_t row = ok ? r0 + g : p.rows - 1;
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < PER; j++) {
        rx[j] = nx[j];
        rg[j] = ng[j];
        rs[j] = ns[j];
      }
      if (r0 + (int64_t)gridDim.x * groups < p.rows) ask(r0 + (int64_t)gridDim.x * groups, nx, ng, ns);
    } else {
      const T* x = static_cast<const T*>(p.x) + row * p.ldx;
      const T* gy = static_cast<const T*>(p.gy) + row * p.ldgy;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        rx[j] = norm_load<T, VEC>(x, t + j * NT, p.D);
        rg[j] = ok ? norm_load<T, VEC>(gy, t + j * NT, p.D) : raw_zero();
      }
      if (p.gs) {
#pragma unroll
        for (int j = 0; j < PER; j++) rs[j] = norm_load<T, VEC>(static_cast<const T*>(p.gs) + row * p.ldgs, t + j * NT, p.D);
      }
    }
    const float mean = p.stats[kNormStats * row], off = p.stats[kNormStats * row + 1], inv = p.stats[kNormStats * row + 2];
    float h[PER][C], a[PER][C], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      raw_unpack<T>(rx[j], h[j]);
      raw_unpack<T>(rg[j], a[j]);
      float (&wj)[C] = w[kHeld ? j : 0];
      if constexpr (!kHeld) norm_weight<T, VEC>(p.w, p.w_f32, t + j * NT, p.D, 1.f, wj);
      float (&dwj)[C] = dw[kInLds ? 0 : j], (&dbj)[C] = db[kInLds ? 0 : j];
      if constexpr (kInLds) {
#pragma unroll
        for (int e = 0; e < C; e += 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&lds_sums[0][(t + j * NT) * C + e]), y = *reinterpret_cast<const f32x4*>(&lds_sums[1][(t + j * NT) * C + e]);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            dwj[e + i] = x[i];
            dbj[e + i] = y[i];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < C; e++) {
        // (columns past D: their gradients are zeros, and so is what they add, as long as h is a number)
        h[j][e] = (t + j * NT) * C + e < p.D ? ((h[j][e] - mean) - off) * inv : 0.f;
        dwj[e] = fmaf(a[j][e], h[j][e], dwj[e]);
        dbj[e] += a[j][e];
        a[j][e] *= wj[e];
        s1 += a[j][e];
        s2 = fmaf(a[j][e], h[j][e], s2);
      }
      if constexpr (kInLds) {
#pragma unroll
        for (int e = 0; e < C; e += 4) {
          *reinterpret_cast<f32x4*>(&lds_sums[0][(t + j * NT) * C + e]) = f32x4{dwj[e], dwj[e + 1], dwj[e + 2], dwj[e + 3]};
          *reinterpret_cast<f32x4*>(&lds_sums[1][(t + j * NT) * C + e]) = f32x4{dbj[e], dbj[e + 1], dbj[e + 2], dbj[e + 3]};
        }
      }
    }
    norm_sum2<NT>(s1, s2, lds, turn);
    turn ^= 1;
    s1 *= per_row;
    s2 *= per_row;
    if (ok && p.dx) {
      T* dx = static_cast<T*>(p.dx) + row * p.D;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        float s[C];
        if (p.gs) raw_unpack<T>(rs[j], s);
#pragma unroll
        for (int e = 0; e < C; e++) a[j][e] = fmaf(fmaf(-h[j][e], s2, a[j][e] - s1), inv, p.gs ? s[e] : 0.f);
        norm_store<T, VEC>(dx, t + j * NT, p.D, a[j]);
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int which = 0; which < 2; which++) {
    float* part = p.part + ((int64_t)blockIdx.x * 2 + which) * p.D;
    if constexpr (groups == 1) {
#pragma unroll
      for (int j = 0; j < PER; j++)
#pragma unroll
        for (int e = 0; e < C; e++)
          if ((t + j * NT) * C + e < p.D) {
            if constexpr (kInLds) part[(t + j * NT) * C + e] = lds_sums[which][(t + j * NT) * C + e];
            else part[(t + j * NT) * C + e] = which ? db[j][e] : dw[j][e];
          }
    } else {
      if (which) __syncthreads();
#pragma unroll
      for (int j = 0; j < PER; j++)
#pragma unroll
        for (int e = 0; e < C; e += 4) {
          const float* q = which ? &db[j][e] : &dw[j][e];
          *reinterpret_cast<f32x4*>(&lds_w[g][(t + j * NT) * C + e]) = f32x4{q[0], q[1], q[2], q[3]};
        }
      __syncthreads();
      for (int c = threadIdx.x; c < p.D; c += BT) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < groups; i++) s += lds_w[i][c];
        part[c] = s;
      }
    }
  }
}

// The workgroups' sums in order: 64 columns a workgroup, 16 runs of workgroups side by side and then those.
template <typename T>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(NormParams p) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane, n = 2 * (int64_t)p.D;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int i = run; i < p.parts; i += 16) s += p.part[i * n + c];
  }
  lds[run][lane] = s;
  __syncthreads();
  if (run == 0 && c < n) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += lds[i][lane];
    void* out = c < p.D ? p.dw : p.db;
    const int64_t at = c < p.D ? c : c - p.D;
    if (out) {
      if (p.w_f32) static_cast<float*>(out)[at] = s;
      else static_cast<T*>(out)[at] = Elem<T>::cvt(s);
    }
  }
}

namespace {

// Threads and chunks of a row: what holds it, with few idle lanes.
int norm_form(int64_t D, int chunk) {
  const int64_t n = (D + chunk - 1) / chunk;
  return n <= 16 ? 0 : n <= 64 ? 1 : n <= 128 ? 2 : n <= 256 ? 3 : n <= 512 ? 4 : n <= 1024 ? 5 : n <= 2048 ? 6 : n <= 4096 ? 7 : 8;
}
int norm_row_threads(int form) { return form == 0 ? 16 : form <= 3 ? 64 : form <= 5 ? 256 : 1024; }

#define AMOE_NORM_FORMS(LAUNCH, TYPE, VEC, FORM) \
  do {                                           \
    switch (FORM) {                              \
      case 0: LAUNCH(TYPE, 16, 1, VEC); break;   \
      case 1: LAUNCH(TYPE, 64, 1, VEC); break;   \
      case 2: LAUNCH(TYPE, 64, 2, VEC); break;   \
      case 3: LAUNCH(TYPE, 64, 4, VEC); break;   \
      case 4: LAUNCH(TYPE, 256, 2, VEC); break;  \
      case 5: LAUNCH(TYPE, 256, 4, VEC); break;  \
      case 6: LAUNCH(TYPE, 1024, 2, VEC); break; \
      case 7: LAUNCH(TYPE, 1024, 4, VEC); break; \
      default:                                   \
        if constexpr (sizeof(TYPE) == 4) LAUNCH(TYPE, 1024, 8, VEC); \
        break;                                   \
    }                                            \
  } while (0)

template <typename T>
int launch_norm_fwd(const NormParams& p, bool vec, hipStream_t st) {
  const int form = norm_form(p.D, Elem<T>::kChunk), nt = norm_row_threads(form), bt = nt < 256 ? 256 : nt;
  const dim3 grid((unsigned)((p.rows + bt / nt - 1) / (bt / nt))), block(bt);
#define AMOE_LAUNCH(TYPE, NT, PER, VEC) hipLaunchKernelGGL((&norm_fwd_kernel<TYPE, NT, PER, VEC>), grid, block, 0, st, p)
  if (vec) AMOE_NORM_FORMS(AMOE_LAUNCH, T, true, form);
  else AMOE_NORM_FORMS(AMOE_LAUNCH, T, false, form);
#undef AMOE_LAUNCH
  return launch_rc();
}

// Workgroups of the backward pass: as many as are on the CUs at once, or fewer, so that a group of threads gets four rows and a
// workgroup eight: each leaves 8 D bytes of sums, which a row's 8 D (16 bits, with the stream's gradient) are the measure of.
int64_t norm_bwd_groups(const amoe_norm_args* a) {
  const int nt = norm_row_threads(norm_form(a->D, a->dtype == AMOE_F32 ? 4 : 8)), groups = (nt <= 256 ? 512 : nt) / nt;
  const int64_t rows = groups >= 2 ? 4 * groups : 8, want = (a->rows + rows - 1) / rows, most = (nt == 1024 ? 1 : 2) * num_compute_units();
  return want < most ? want : most;
}

template <typename T>
int launch_norm_bwd(const NormParams& p, bool vec, hipStream_t st) {
  const int form = norm_form(p.D, Elem<T>::kChunk), nt = norm_row_threads(form);
  const dim3 grid((unsigned)p.parts), block(nt <= 256 ? 512 : nt);
#define AMOE_LAUNCH(TYPE, NT, PER, VEC) hipLaunchKernelGGL((&norm_bwd_kernel<TYPE, NT, PER, VEC>), grid, block, 0, st, p)
  if (vec) AMOE_NORM_FORMS(AMOE_LAUNCH, T, true, form);
  else AMOE_NORM_FORMS(AMOE_LAUNCH, T, false, form);
#undef AMOE_LAUNCH
  if (p.part) {
    const dim3 cols((unsigned)((2 * (int64_t)p.D + 63) / 64)), threads(1024);
    hipLaunchKernelGGL((&norm_reduce_kernel<T>), cols, threads, 0, st, p);
  }
  return launch_rc();
}

int norm_check(const amoe_norm_args* a) {
  if (!a) return AMOE_ENULL;
  if (a->dtype != AMOE_F32 && a->dtype != AMOE_BF16 && a->dtype != AMOE_F16) return AMOE_EINVAL;
  if (a->weight_dtype != a->dtype && a->weight_dtype != AMOE_F32) return AMOE_EINVAL;
  if (a->rows < 0 || a->D < 1 || !(a->eps >= 0) || !(a->eps <= 3e38)) return AMOE_EINVAL;
  // (threads of a launch are counted in 32 bits)
  if (a->D > kNormMaxD || a->rows >= INT64_C(1) << 31) return AMOE_EUNSUPPORTED;
  const int64_t nt = norm_row_threads(norm_form(a->D, a->dtype == AMOE_F32 ? 4 : 8));
  return a->rows * nt >= INT64_C(1) << 32 ? AMOE_EUNSUPPORTED : AMOE_OK;
}

// A tensor of rows: there, aligned to its elements; whole 16-byte chunks leave vec as it is.
int norm_rows(const void* p, int64_t ld, const amoe_norm_args* a, bool& vec) {
  const size_t es = esize((int)a->dtype);
  if (!p) return AMOE_ENULL;
  if (!aligned(p, es)) return AMOE_EALIGN;
  if (a->rows > 1 && (ld < 0 || ld > INT64_C(1) << 40)) return AMOE_EINVAL;
  vec = vec && aligned(p, 16) && (a->rows == 1 || ld * (int64_t)es % 16 == 0);
  return AMOE_OK;
}

int norm_weights(const amoe_norm_args* a, bool& vec) {
  const size_t es = esize((int)a->weight_dtype);
  if (!aligned(a->weight, es) || !aligned(a->bias, es)) return AMOE_EALIGN;
  vec = vec && aligned(a->weight, 16) && aligned(a->bias, 16) && a->D * (int64_t)esize((int)a->dtype) % 16 == 0;
  return AMOE_OK;
}

// (how far apart the one row is from the next says nothing)
NormParams norm_params(const amoe_norm_args* a) {
  NormParams p{};
  const bool one = a->rows == 1;
  p.x = a->x; p.ldx = one ? 0 : a->ldx;
  p.w = a->weight; p.b = a->bias;
  p.w_f32 = a->weight_dtype == AMOE_F32;
  p.stats = a->stats;
  p.rows = a->rows; p.D = (int)a->D;
  p.eps = (float)a->eps;
  return p;
}

}  // namespace

}  // namespace amoe

using namespace amoe;

extern "C" size_t amoe_norm_args_bytes(void) { return sizeof(amoe_norm_args); }

extern "C" int amoe_layer_norm_fwd(const amoe_norm_args* a, void* stream) {
  if (int rc = norm_check(a)) return rc;
  if (a->rows == 0) return AMOE_OK;
  bool vec = true;
  if (int rc = norm_rows(a->x, a->ldx, a, vec)) return rc;
  if (int rc = norm_rows(a->y, a->D, a, vec)) return rc;
  if (!a->residual != !a->sum) return AMOE_ENULL;
  if (a->residual) {
    if (int rc = norm_rows(a->residual, a->ldr, a, vec)) return rc;
    if (int rc = norm_rows(a->sum, a->D, a, vec)) return rc;
  }
  if (int rc = norm_weights(a, vec)) return rc;
  if (!aligned(a->stats, 4)) return AMOE_EALIGN;
  NormParams p = norm_params(a);
  p.res = a->residual; p.ldr = a->rows == 1 ? 0 : a->ldr;
  p.y = a->y; p.sum = a->sum;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_norm_fwd<float>(p, vec, st)
         : a->dtype == AMOE_F16 ? launch_norm_fwd<f16_t>(p, vec, st)
                                : launch_norm_fwd<uint16_t>(p, vec, st);
}

extern "C" size_t amoe_layer_norm_bwd_workspace(const amoe_norm_args* a) {
  if (norm_check(a) || a->rows == 0 || (!a->dweight && !a->dbias)) return 0;
  return (size_t)norm_bwd_groups(a) * 2 * (size_t)a->D * 4;
}

extern "C" int amoe_layer_norm_bwd(const amoe_norm_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = norm_check(a)) return rc;
  const size_t ws = esize((int)a->weight_dtype);
  if (!aligned(a->dweight, ws) || !aligned(a->dbias, ws)) return AMOE_EALIGN;
  if (a->rows == 0) return a->dweight || a->dbias ? AMOE_EINVAL : AMOE_OK;      // (sums of nothing are the caller's zeros)
  bool vec = true;
  if (int rc = norm_rows(a->x, a->ldx, a, vec)) return rc;
  if (int rc = norm_rows(a->gy, a->ldgy, a, vec)) return rc;
  if (a->gs) {
    if (int rc = norm_rows(a->gs, a->ldgs, a, vec)) return rc;
  }
  if (a->dx) {
    if (int rc = norm_rows(a->dx, a->D, a, vec)) return rc;
  }
  if (int rc = norm_weights(a, vec)) return rc;
  if (!a->stats) return AMOE_ENULL;
  if (!aligned(a->stats, 4)) return AMOE_EALIGN;
  const size_t need = amoe_layer_norm_bwd_workspace(a);
  if (need && !workspace) return AMOE_ENULL;
  if (workspace_bytes < need) return AMOE_EWORKSPACE;
  if (need && !aligned(workspace, 4)) return AMOE_EALIGN;
  NormParams p = norm_params(a);
  const bool one = a->rows == 1;
  p.gy = a->gy; p.ldgy = one ? 0 : a->ldgy;
  p.gs = a->gs; p.ldgs = one ? 0 : a->ldgs;
  p.dx = a->dx; p.dw = a->dweight; p.db = a->dbias;
  p.part = need ? static_cast<float*>(workspace) : nullptr;
  p.parts = (int)norm_bwd_groups(a);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_norm_bwd<float>(p, vec, st)
         : a->dtype == AMOE_F16 ? launch_norm_bwd<f16_t>(p, vec, st)
                                : launch_norm_bwd<uint16_t>(p, vec, st);
}
