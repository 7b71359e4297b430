// Entry points of attention: argument checks, the choice of the kernel, the workspace.
#include "attn_host.h"

using namespace amoe;

namespace {

int check_operand(const void* p, const int64_t* st, int64_t rows, int64_t heads, int64_t d, size_t es) {
  if (rows == 0 || heads == 0) return AMOE_OK;
  if (!p) return AMOE_ENULL;
  if (!aligned(p, es)) return AMOE_EALIGN;
  for (int i = 0; i < 3; i++)
    if (st[i] < 0 || st[i] > (INT64_C(1) << 40)) return AMOE_EINVAL;
  return d < 1 ? AMOE_EINVAL : AMOE_OK;
}

// Rows further apart than this are not addressed by 32-bit offsets (128 of them must stay below 2^31).
constexpr int64_t kAttnRowBytes = INT64_C(1) << 23;

// 1: rows start on 16 bytes; 2: and a tile's rows can be addressed by 32-bit offsets into a resource that ends with them
int operand_vec(const AttnOperand& o, int64_t rows, int64_t d, size_t es) {
  const int64_t c = 16 / (int64_t)es;
  if (!aligned(o.p, 16) || o.sb % c || o.ss % c || o.sh % c) return 0;
  if (rows > 1 && (o.ss < d || o.ss * (int64_t)es > kAttnRowBytes)) return 1;
  return 2;
}

int check_sizes(const amoe_attn_args* a) {
  if (!a) return AMOE_ENULL;
  if (a->dtype != AMOE_F32 && a->dtype != AMOE_BF16 && a->dtype != AMOE_F16) return AMOE_EINVAL;
  if (a->B < 0 || a->S < 0 || a->T < 0 || a->H < 1 || a->G < 1 || a->d < 1) return AMOE_EINVAL;
  if (a->H % a->G) return AMOE_ESHAPE;
  // (what the kernels take are the floats scale and scale * log2(e): normal ones, or masked scores meet 0 or infinity)
  if (!(a->scale >= 0x1p-126) || !(a->scale <= 0x1p127)) return AMOE_EINVAL;
  if (a->d > kAttnMaxHead || a->S > kAttnMaxRows || a->T > kAttnMaxRows) return AMOE_EUNSUPPORTED;
  // threads of a launch are counted in 32 bits: 2^24 workgroups of 256 over the queries, 2^23 of 512 over the keys
  const int64_t over = INT64_C(1) << 23;
  if (a->B > over || a->H > over || a->B * a->H > over) return AMOE_EUNSUPPORTED;
  if (a->B * a->H * ((a->S + 127) / 128) >= over || a->B * a->G * ((a->T + 63) / 64) >= over) return AMOE_EUNSUPPORTED;
  return a->H / a->G * a->S > (INT64_C(1) << 30) ? AMOE_EUNSUPPORTED : AMOE_OK;
}

// Parts of the key axis for the kernel of few rows; 0: the kernel of many rows.
//
// Up to 32 rows share one read of the keys.  More are read for 32 by 32, which pays where blocks of 32 rows would not fill half the
// CUs and every one of them would walk many keys by itself: with n of them, from 32 n keys on, and 1024.  Measured (us, many rows /
// parts; 16 over 4 heads of 128, one sequence, then of 64, four; bf16): 40 queries (n = 32) over 600 keys 11.5 / 11.2, 1024
// 15.3 / 11.8, 8192 92 / 23; 100 (64) over 1024 15.3 / 16.9, 2000 25 / 20, 8192 91 / 35; 250 (128) over 2000 25 / 28, 8192 90 / 65;
// 4 x 40 (128) over 2000 15 / 19, 8192 49 / 29; 4 x 100 (256) over 2000 16 / 28, 8192 49 / 59, 32768 182 / 200.
int attn_splits(const amoe_attn_args* a) {
  const int64_t rows = a->H / a->G * a->S, cus = num_compute_units();
  const int64_t blocks = a->B * a->H * ((a->S + 31) / 32);
  if (rows > 32 && (2 * blocks > cus || a->T < 1024 || a->T < 32 * blocks)) return 0;
  const int64_t groups = a->B * a->G * ((rows + 31) / 32);
  // parts of 512 keys or more, up to eight workgroups per CU (sequences differ in length, and the last round of workgroups
  // is then short); where that leaves CUs without work, parts of down to 128 keys for two.  One query over 131071 keys, 16 over 2
  // heads of 128: 28 us, parts of 256 31.5, of 1024 28; 8 over 4096 to 8192, 16 over 4: 25, 27.6 and 26.7; 256 over 512 to 1024:
  // 99, 100 and 87.  The smaller ones at least 256: one over 1024 keys, 16 heads of 64, 8.2 us for 7.8, over 4096 10.6 for 10.0
  const auto parts = [&](int64_t per_cu, int64_t keys) {
    const int64_t n = (per_cu * cus + groups - 1) / groups, most = (a->T + keys - 1) / keys;
    return n < most ? n : most;
  };
  int64_t n = parts(8, 512);
  const int64_t few = parts(2, 128);
  if (few > n) n = few;
  return (int)(n < 1 ? 1 : n > kAttnMaxSplits ? kAttnMaxSplits : n);
}

// (how far apart the one element of a dimension of size 1 is from the next says nothing)
AttnOperand operand(const void* p, const int64_t* st, int64_t batch, int64_t rows, int64_t heads) {
  return {p, batch == 1 ? 0 : st[0], rows == 1 ? 0 : st[1], heads == 1 ? 0 : st[2]};
}

void fill(AttnParams& p, const amoe_attn_args* a) {
  p.q = operand(a->q, &a->q_sb, a->B, a->S, a->H);
  p.k = operand(a->k, &a->k_sb, a->B, a->T, a->G);
  p.v = operand(a->v, &a->v_sb, a->B, a->T, a->G);
  p.lengths = a->lengths; p.lengths_i64 = (int)a->lengths_is_i64;
  p.starts = a->starts; p.starts_i64 = (int)a->starts_is_i64;
  p.B = (int)a->B; p.S = (int)a->S; p.T = (int)a->T; p.H = (int)a->H; p.G = (int)a->G; p.R = (int)(a->H / a->G);
  p.d = (int)a->d; p.causal = a->causal != 0;
  p.copies = 1;
  p.c = (float)(a->scale * 1.4426950408889634074);
  p.scale = (float)a->scale;
  p.lse = a->lse;
  const size_t es = esize((int)a->dtype);
  int vec = operand_vec(p.q, a->S, a->d, es);
  if (a->T > 0) {
    const int vk = operand_vec(p.k, a->T, a->d, es), vv = operand_vec(p.v, a->T, a->d, es);
    vec = vk < vec ? vk : vec;
    vec = vv < vec ? vv : vec;
  }
  p.vec = vec;
}

int check_inputs(const amoe_attn_args* a) {
  const size_t es = esize((int)a->dtype);
  if (int rc = check_operand(a->q, &a->q_sb, a->S, a->H, a->d, es)) return rc;
  if (int rc = check_operand(a->k, &a->k_sb, a->T, a->G, a->d, es)) return rc;
  if (int rc = check_operand(a->v, &a->v_sb, a->T, a->G, a->d, es)) return rc;
  if (!aligned(a->lengths, a->lengths_is_i64 ? 8 : 4) || !aligned(a->starts, a->starts_is_i64 ? 8 : 4)) return AMOE_EALIGN;
  return aligned(a->lse, 4) ? AMOE_OK : AMOE_EALIGN;
}

}  // namespace

extern "C" size_t amoe_attn_args_bytes(void) { return sizeof(amoe_attn_args); }

extern "C" size_t amoe_attention_fwd_workspace(const amoe_attn_args* a) {
  if (check_sizes(a) || a->B == 0 || a->S == 0) return 0;
  const int n = attn_splits(a);
  return n > 1 ? (size_t)n * (size_t)(a->B * a->H * a->S) * (size_t)((a->d + 3) / 4 * 4 + 2) * 4 : 0;
}

extern "C" int amoe_attention_fwd(const amoe_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_sizes(a)) return rc;
  if (a->B == 0 || a->S == 0) return AMOE_OK;
  if (int rc = check_inputs(a)) return rc;
  const size_t es = esize((int)a->dtype);
  if (!a->out) return AMOE_ENULL;
  if (!aligned(a->out, es)) return AMOE_EALIGN;
  AttnParams p{};
  fill(p, a);
  p.out = a->out;
  p.rest = a->rest;
  if (!aligned(a->rest, es)) return AMOE_EALIGN;
  if ((!aligned(a->out, 16) || !aligned(a->rest, 16)) && p.vec == 2) p.vec = 1;
  p.splits = attn_splits(a);
  if (p.splits > 1) {
    const size_t need = amoe_attention_fwd_workspace(a);
    if (!workspace) return AMOE_ENULL;
    if (workspace_bytes < need) return AMOE_EWORKSPACE;
    if (!aligned(workspace, 16)) return AMOE_EALIGN;
    // (the rows first: their 16-byte stores)
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + (size_t)p.splits * (size_t)(a->B * a->H * a->S) * (size_t)((a->d + 3) / 4 * 4);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_attn_fwd_f32(p, st)
         : a->dtype == AMOE_F16 ? launch_attn_fwd_f16(p, st)
                                : launch_attn_fwd_bf16(p, st);
}

extern "C" size_t amoe_attention_bwd_workspace(const amoe_attn_args* a) {
  if (check_sizes(a)) return 0;
  return (size_t)(a->B * a->H * a->S) * 3 * 4;
}

extern "C" int amoe_attention_bwd(const amoe_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_sizes(a)) return rc;
  if (a->B == 0 || (a->S == 0 && a->T == 0)) return AMOE_OK;
  if (int rc = check_inputs(a)) return rc;
  const size_t es = esize((int)a->dtype);
  if (int rc = check_operand(a->go, &a->go_sb, a->S, a->H, a->d, es)) return rc;
  if ((a->S > 0 && (!a->out || !a->lse || !a->dq || !workspace)) || !a->dk != !a->dv) return AMOE_ENULL;
  if (!aligned(a->out, es) || !aligned(a->rest, es) || !aligned(a->dq, es) || !aligned(a->dk, es) || !aligned(a->dv, es)) return AMOE_EALIGN;
  if (workspace_bytes < amoe_attention_bwd_workspace(a)) return AMOE_EWORKSPACE;
  if (!aligned(workspace, 4)) return AMOE_EALIGN;
  AttnParams p{};
  fill(p, a);
  p.go = operand(a->go, &a->go_sb, a->B, a->S, a->H);
  if (a->S > 0) {
    const int vg = operand_vec(p.go, a->S, a->d, es);
    p.vec = vg < p.vec ? vg : p.vec;
  }
  const bool whole = aligned(a->out, 16) && aligned(a->rest, 16) && aligned(a->dq, 16) && aligned(a->dk, 16) && aligned(a->dv, 16);
  if (!whole) p.vec = 0;
  // (rows of `out` are d elements apart: with another d their starts are not on 16 bytes)
  if ((a->d * es) % 16) p.vec = 0;
  if (a->S > 1 && a->H * a->d * (int64_t)es > kAttnRowBytes && p.vec == 2) p.vec = 1;
  p.o = a->out;
  p.rest = a->rest;
  p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  p.rows = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_attn_bwd_f32(p, st)
         : a->dtype == AMOE_F16 ? launch_attn_bwd_f16(p, st)
                                : launch_attn_bwd_bf16(p, st);
}

// ---- sequences that share a prefix ----------------------------------------------------------------
namespace {

// What is asked of one set of keys, in the terms of the other calls: the prefix's, B of which are seen by all queries of N = B / B'
// sequences each, or the sequences' own.
amoe_attn_args shared_part(const amoe_shared_attn_args* a, bool prefix) {
  amoe_attn_args s{};
  s.dtype = a->dtype; s.B = prefix ? a->prefixes : a->B; s.S = a->S; s.T = prefix ? a->P : a->T; s.H = a->H; s.G = a->G; s.d = a->d;
  s.causal = prefix ? 0 : a->causal;
  s.scale = a->scale;
  s.q = a->q; s.q_sb = a->q_sb; s.q_ss = a->q_ss; s.q_sh = a->q_sh;
  s.k = prefix ? a->prefix_k : a->k;
  s.k_sb = prefix ? a->prefix_k_sb : a->k_sb; s.k_ss = prefix ? a->prefix_k_ss : a->k_ss; s.k_sh = prefix ? a->prefix_k_sh : a->k_sh;
  s.v = prefix ? a->prefix_v : a->v;
  s.v_sb = prefix ? a->prefix_v_sb : a->v_sb; s.v_ss = prefix ? a->prefix_v_ss : a->v_ss; s.v_sh = prefix ? a->prefix_v_sh : a->v_sh;
  s.lengths = prefix ? a->prefix_lengths : a->lengths;
  s.lengths_is_i64 = prefix ? a->prefix_lengths_is_i64 : a->lengths_is_i64;
  s.starts = prefix ? nullptr : a->starts;
  s.starts_is_i64 = a->starts_is_i64;
  return s;
}

int check_shared(const amoe_shared_attn_args* a) {
  if (!a) return AMOE_ENULL;
  if (a->B < 0 || a->prefixes < 0 || a->P < 0) return AMOE_EINVAL;
  if (a->B > 0 && (a->prefixes == 0 || a->B % a->prefixes)) return AMOE_ESHAPE;
  const amoe_attn_args own = shared_part(a, false), prefix = shared_part(a, true);
  if (int rc = check_sizes(&own)) return rc;
  if (int rc = check_sizes(&prefix)) return rc;
  if (a->B == 0 || a->S == 0) return AMOE_OK;
  // threads of the join, and rows that share a key head, in 32 bits
  if (a->B * a->H >= (INT64_C(1) << 23) / a->S) return AMOE_EUNSUPPORTED;
  return a->B / a->prefixes * (a->H / a->G) * a->S > (INT64_C(1) << 30) ? AMOE_EUNSUPPORTED : AMOE_OK;
}

struct SharedPlan {
  int rw = 0, splits = 0;
};

// Waves over the rows and parts of the keys, for `rows` rows that share a key head in each of `heads` of them and T keys.  Workgroups
// of many rows: one on a CU, where it leaves room for one of few rows, which waits for memory meanwhile (64 sequences over 30001
// shared and 1024 own keys, 16 over 4 heads of 128: 46 us, with two on a CU 64; of 64: 36 and 42; four prefixes of 8192, 64 sequences
// each, 32 over 8 heads: 127 and 147), parts of 256 keys or more.  Of few rows: as attn_splits.
SharedPlan shared_plan(int64_t rows, int64_t heads, int64_t T, bool whole, size_t es) {
  SharedPlan p;
  if (T == 0) return p;
  const int64_t cus = num_compute_units();
  p.rw = rows <= 32 ? 0 : rows <= 64 && whole && es == 2 ? 2 : 4;
  const int64_t block = p.rw ? 32 * p.rw : 32, groups = heads * ((rows + block - 1) / block);
  const auto parts = [&](int64_t per_cu, int64_t keys) {
    const int64_t n = (per_cu * cus + groups - 1) / groups, most = (T + keys - 1) / keys;
    return n < most ? n : most;
  };
  int64_t n = p.rw ? parts(1, 256) : parts(8, 512);
  const int64_t few = parts(2, 128);
  if (!p.rw && few > n) n = few;
  p.splits = (int)(n < 1 ? 1 : n > kAttnMaxSplits / 2 ? kAttnMaxSplits / 2 : n);
  return p;
}

struct SharedPlans {
  SharedPlan prefix, own;
};
SharedPlans shared_plans(const amoe_shared_attn_args* a, bool whole) {
  const int64_t rows = a->H / a->G * a->S, copies = a->B / a->prefixes;
  const size_t es = esize((int)a->dtype);
  SharedPlans p{shared_plan(copies * rows, a->prefixes * a->G, a->P, whole, es), shared_plan(rows, a->B * a->G, a->T, whole, es)};
  if (p.own.rw) p.own.rw = p.prefix.rw = 4;
  return p;
}

size_t shared_bytes(const amoe_shared_attn_args* a, int parts) {
  return (size_t)parts * (size_t)(a->B * a->H * a->S) * (size_t)((a->d + 3) / 4 * 4 + 2) * 4;
}

}  // namespace

extern "C" size_t amoe_shared_attn_args_bytes(void) { return sizeof(amoe_shared_attn_args); }

extern "C" size_t amoe_attention_shared_fwd_workspace(const amoe_shared_attn_args* a) {
  if (check_shared(a) || a->B == 0 || a->S == 0) return 0;
  // (the strides decide between forms with as many parts or fewer)
  const SharedPlans x = shared_plans(a, true), y = shared_plans(a, false);
  const int m = x.prefix.splits + x.own.splits, n = y.prefix.splits + y.own.splits;
  return shared_bytes(a, m > n ? m : n);
}

extern "C" int amoe_attention_shared_fwd(const amoe_shared_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_shared(a)) return rc;
  if (a->B == 0 || a->S == 0) return AMOE_OK;
  const amoe_attn_args own = shared_part(a, false), prefix = shared_part(a, true);
  if (int rc = check_inputs(&own)) return rc;
  if (int rc = check_inputs(&prefix)) return rc;
  const size_t es = esize((int)a->dtype), need = amoe_attention_shared_fwd_workspace(a);
  if (!a->out) return AMOE_ENULL;
  if (!aligned(a->out, es)) return AMOE_EALIGN;
  if (need && !workspace) return AMOE_ENULL;
  if (workspace_bytes < need) return AMOE_EWORKSPACE;
  if (!aligned(workspace, 16)) return AMOE_EALIGN;
  AttnShared s{};
  fill(s.own, &own);
  fill(s.prefix, &prefix);
  // the queries are those of all sequences
  s.prefix.q = s.own.q;
  s.prefix.copies = (int)(a->B / a->prefixes);
  const int vec = operand_vec(s.own.q, a->S, a->d, es);
  s.prefix.vec = a->P > 0 ? operand_vec(s.prefix.k, a->P, a->d, es) : 2;
  if (a->P > 0 && operand_vec(s.prefix.v, a->P, a->d, es) < s.prefix.vec) s.prefix.vec = operand_vec(s.prefix.v, a->P, a->d, es);
  if (vec < s.prefix.vec) s.prefix.vec = vec;
  s.prefix.vec = s.own.vec = s.prefix.vec < s.own.vec ? s.prefix.vec : s.own.vec;
  const SharedPlans plans = shared_plans(a, attn_whole_chunks(s.own, es));
  s.prefix.splits = plans.prefix.splits; s.prefix_rw = plans.prefix.rw;
  s.own.splits = plans.own.splits; s.own_rw = plans.own.rw;
  const int parts = s.prefix.splits + s.own.splits;
  const size_t rows = (size_t)(a->B * a->H * a->S), pad = (size_t)((a->d + 3) / 4 * 4);
  // (the rows first: their 16-byte stores)
  s.prefix.part_o = static_cast<float*>(workspace);
  s.prefix.part_ml = s.prefix.part_o + parts * rows * pad;
  s.own.part_o = s.prefix.part_o + s.prefix.splits * rows * pad;
  s.own.part_ml = s.prefix.part_ml + s.prefix.splits * rows * 2;
  s.join = s.own;
  s.join.part_o = s.prefix.part_o;
  s.join.part_ml = s.prefix.part_ml;
  s.join.splits = parts;
  s.join.out = a->out;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a->dtype == AMOE_F32   ? launch_attn_shared_f32(s, st)
         : a->dtype == AMOE_F16 ? launch_attn_shared_f16(s, st)
                                : launch_attn_shared_bf16(s, st);
}
