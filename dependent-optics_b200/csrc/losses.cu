// losses.cu — objectives over a model's logits, each with its adjoint:
// token log-probabilities, the clipped policy loss, the preference loss and
// the distillation loss from a teacher's top logits.
//
// Every one of them takes, for a row z of V logits, x = z / tau,
// lse = log sum exp x and p = exp(x - lse), and its adjoint is a scalar per
// row times p plus a correction at a few entries:
//
//   log-probability  logp = x_a - lse               dz = g / tau ([v = a] - p)
//   policy           r = exp(logp - old), -min(r A, clip(r) A) + beta kl
//   preference       -log sigma of the difference of two sums of logp - ref
//   distillation     tau^2 KL(q || p) over K entries (and the rest as one)
//
// so one kernel serves them: a pass over the row for its maximum and sum
// (running, in fp32), the row's scalars in double by one thread (ratios and
// margins are small differences of log-probabilities), and a pass that
// writes the adjoint.
#include <cmath>
#include <string>
#include <type_traits>

#include "../../include/dop.h"
#include "kernels.cuh"
#include "tc_ptx.cuh"

namespace dop {
int set_last_error(int code, const char* msg);

namespace {

enum RowOp : int { kLogp = 0, kLogpBwd = 1, kPolicy = 2, kDistill = 3 };

constexpr int kRowThreads = 256;
constexpr int kMaxTeacherK = 1024;
constexpr int kMaxCluster = 8;
// Shared memory of a CTA's pieces: three CTAs fit an SM up to kStageBytes,
// one up to kStageBytesMost.
constexpr int64_t kStageBytes = 72 * 1024, kStageBytesMost = 200 * 1024;
constexpr double kLog2e = 1.4426950408889634;

struct RowArgs {
  const void* z;
  int64_t ld;
  void* dz;  // null: no adjoint
  int64_t ldd;
  int64_t V;
  const int64_t* tokens;
  const float* weight;  // null: 1
  double inv_tau;
  float c;       // log2(e) / tau
  int cluster;      // CTAs per row
  int stage_bytes;  // of shared memory for a CTA's pieces
  double scale;  // of the loss and the adjoint
  float* logp;
  float* logp_lo;  // null, or what logp's rounding to fp32 left out
  float* lse;
  float* row_loss;
  const float* dlogp;  // log-probability adjoint
  // policy
  const float *old_logp, *advantage, *ref_logp;
  double clip_low, clip_high, kl_coef;
  // distillation
  int K;
  const int32_t* top_index;
  const float* top_logit;
  const float* teacher_lse;
};

// Running maximum and sum of 2^(c (z - max)); a maximum of -inf (no finite
// element yet) counts as 0, so that 2^(-inf - max) stays 0.  The maximum is
// subtracted before the factor is applied: c max overflows for a row that is
// all of the type's lowest value.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m), k = base_of(m);
  return {m, a.s * tc::fast_exp2((a.m - k) * c) + b.s * tc::fast_exp2((b.m - k) * c)};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = join(v, {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)}, c);
  return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the CTA in a fixed order; every thread gets it.
__device__ double block_sum_d(double v, double* red) {
  v = warp_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < kRowThreads / 32; ++w) t += red[w];
  return t;
}

// ---- a row in shared memory
// A row is cut into 16-byte pieces at 16-byte borders of its address, so a
// row may start and end inside a piece; the cluster's CTAs hold consecutive
// runs of pieces, one CTA the whole row when it fits.  A thread copies pieces
// tid, tid + 256, ... and is the one that reads them back for the maximum and
// sum, so that pass needs no barrier.  What a piece holds beyond the row is -inf.
__device__ __forceinline__ void copy_piece(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most `n` of this thread's copy groups are under way.
__device__ __forceinline__ void copy_wait(int n) {
  switch (n) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
  }
}
__device__ __forceinline__ float2 bf16x2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// The elements of a piece as pairs.
__device__ __forceinline__ void unpack(uint4 u, float2* x, const float*) {
  x[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
  x[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ void unpack(uint4 u, float2* x, const bf16*) {
  x[0] = bf16x2(u.x);
  x[1] = bf16x2(u.y);
  x[2] = bf16x2(u.z);
  x[3] = bf16x2(u.w);
}
__device__ __forceinline__ uint32_t minus_inf_word(const float*) { return 0xff800000u; }
__device__ __forceinline__ uint32_t minus_inf_word(const bf16*) { return 0xff80ff80u; }
__device__ __forceinline__ void store_unit(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_unit(bf16* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(tc::pack_bf16(v[0], v[1]), tc::pack_bf16(v[2], v[3]),
                                            tc::pack_bf16(v[4], v[5]), tc::pack_bf16(v[6], v[7]));
}

// What the CTAs of a cluster tell one another of their part of the row.
struct alignas(16) Part {
  MaxSum rest;    // entries not listed by the teacher (all, elsewhere)
  MaxSum listed;  // listed entries, each vocabulary entry once
  float count;    // of the listed entries
};
static_assert(sizeof(Part) == 32, "a Part is written to a peer as 16 + 4 bytes");

// A cluster of `nctarank` CTAs per row.
template <RowOp OP, typename TI, typename TO>
__global__ void __launch_bounds__(kRowThreads, 3) k_vocab_row(const RowArgs a) {
  constexpr int EI = 16 / (int)sizeof(TI), EO = 16 / (int)sizeof(TO);
  constexpr int NT = kRowThreads, NW = NT / 32, U = 4;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Part s_warp[NW];
  __shared__ Part s_peer[kMaxCluster];
  __shared__ double s_red[2][NW];
  __shared__ float s_coef[4];
  __shared__ int s_twice;
  const int C = a.cluster, rank = (int)blockIdx.x % C, tid = threadIdx.x, lane = tid & 31;
  const int64_t row = blockIdx.x / C;
  const TI* z = (const TI*)a.z + row * a.ld;
  TO* dz = a.dz ? (TO*)a.dz + row * a.ldd : nullptr;
  const int V = (int)a.V;
  // this CTA's pieces [p0, p1) and elements [e_lo, e_hi)
  const int ph = (int)((uintptr_t)z & 15) / (int)sizeof(TI);
  const int64_t pieces = ((int64_t)ph + V + EI - 1) / EI;
  const int p0 = (int)(pieces * rank / C), np = (int)(pieces * (rank + 1) / C) - p0;
  const int e_org = (int)((int64_t)p0 * EI - ph);  // the row's element at image element 0
  const int e_lo = max(0, e_org), e_hi = (int)min((int64_t)V, (int64_t)e_org + (int64_t)np * EI);
  // units of 16 bytes of dz: whole ones [u0, u1), the rest of the elements ahead and behind
  const int dph = dz ? (int)((uintptr_t)dz & 15) / (int)sizeof(TO) : 0;
  const int64_t u0 = ((int64_t)dph + e_lo + EO - 1) / EO, u1 = ((int64_t)dph + e_hi) / EO;

  const float w = a.weight ? a.weight[row] : 1.f;
  const int64_t token = OP == kDistill ? -1 : a.tokens[row];
  bool skip = w == 0.f || (OP != kDistill && (token < 0 || token >= V));
  if (OP == kLogpBwd && a.dlogp[row] == 0.f) skip = true;

  // elements of the units that are not whole: f(element)
  auto ragged = [&](auto f) {
    if (u0 >= u1) {
      for (int e = e_lo + tid; e < e_hi; e += NT) f(e);
    } else {
      const int ahead = (int)(u0 * EO - dph) - e_lo, behind0 = (int)(u1 * EO - dph);
      if (tid < ahead) f(e_lo + tid);
      if (tid >= 32 && tid - 32 < e_hi - behind0) f(behind0 + tid - 32);
    }
  };
  if (skip) {
    if (dz) {
      const float zero[EO] = {};
      for (int64_t u = u0 + tid; u < u1; u += NT) store_unit(dz + (u * EO - dph), zero);
      ragged([&](int e) { st(&dz[e], 0.f); });
    }
    if (tid == 0 && rank == 0) {
      if (OP != kLogpBwd && OP != kDistill && a.logp) a.logp[row] = 0.f;
      if (OP == kLogp && a.lse) a.lse[row] = 0.f;
      if (OP == kLogp && a.logp_lo) a.logp_lo[row] = 0.f;
      if (OP == kPolicy || OP == kDistill) a.row_loss[row] = 0.f;
    }
    return;
  }
  // every CTA of the cluster has started once this barrier is through: its
  // shared memory may be written to
  if (OP != kLogpBwd && C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ---- copy this CTA's pieces
  const uint32_t img = tc::smem_u32(dyn);
  TI* image = (TI*)dyn;
  const TI* src = z + e_org;
  const int rounds = (np + U * NT - 1) / (U * NT);
  for (int r = 0; r < rounds; ++r) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = tid + (r * U + j) * NT;
      if (i >= np) continue;
      const int e = e_org + i * EI;
      if (e >= 0 && e <= V - EI) {
        copy_piece(img + i * 16, src + (int64_t)i * EI);
      } else {
        for (int k = 0; k < EI; ++k)
          image[i * EI + k] = e + k >= 0 && e + k < V ? z[e + k] : (TI)-INFINITY;
      }
    }
    copy_commit();
  }
  const float za = OP == kDistill || OP == kLogpBwd ? 0.f : ld(&z[token]);

  // ---- the teacher's entries while the copies run: q, the student's logit
  int32_t* t_idx = (int32_t*)(dyn + a.stage_bytes);
  float* t_q = (float*)(t_idx + a.K);  // q
  float* t_z = t_q + a.K;              // the student's logit
  float* t_g = t_z + a.K;              // this CTA's first ones: sum of q of the entry; else -1
  double q_sum = 0.0, q_logq = 0.0, q_rest = 0.0;
  if (OP == kDistill) {
    const float* y = a.top_logit + row * a.K;
    MaxSum t = {-INFINITY, 0.f};
    for (int k = tid; k < a.K; k += NT) {
      const int32_t i = a.top_index[row * a.K + k];
      const bool in = i >= 0 && i < V;
      const float yk = in ? y[k] : -INFINITY;
      t_idx[k] = in ? i : -1;
      t_z[k] = in ? ld(&z[i]) : 0.f;
      t_q[k] = yk;
      if (in) t = join(t, {yk, 1.f}, a.c);
    }
    if (tid == 0) s_twice = 0;
    double tl;
    if (a.teacher_lse) {
      tl = (double)a.teacher_lse[row];
    } else {
      t = warp_join(t, a.c);
      if (lane == 0) s_warp[tid >> 5].rest = t;
      __syncthreads();
      t = s_warp[0].rest;
      for (int i = 1; i < NW; ++i) t = join(t, s_warp[i].rest, a.c);
      tl = (double)base_of(t.m) * a.inv_tau + log((double)t.s);
    }
    double qs = 0.0, ql = 0.0;
    for (int k = tid; k < a.K; k += NT) {
      const double lq = (double)t_q[k] * a.inv_tau - tl;
      const double q = t_idx[k] < 0 || t_q[k] == -INFINITY ? 0.0 : exp(lq);
      t_q[k] = (float)q;
      qs += q;
      if (q > 0.0) ql += q * lq;
    }
    qs = warp_sum_d(qs);
    ql = warp_sum_d(ql);
    if (lane == 0) {
      s_red[0][tid >> 5] = qs;
      s_red[1][tid >> 5] = ql;
    }
    // ---- listed entries leave the image: -inf, and each counts once.  A word
    // of all ones marks an entry; one found marked is named twice (or was that
    // NaN), and then the entries are compared one by one.
    copy_wait(0);
    __syncthreads();
    for (int i = 0; i < NW; ++i) {
      q_sum += s_red[0][i];
      q_logq += s_red[1][i];
    }
    q_rest = a.teacher_lse ? fmax(0.0, 1.0 - q_sum) : 0.0;
    auto here = [&](int k) { return t_idx[k] >= e_lo && t_idx[k] < e_hi; };
    uint32_t* words = (uint32_t*)dyn;
    for (int k = tid; k < a.K; k += NT) {
      t_g[k] = here(k) ? t_q[k] : -1.f;
      if (!here(k)) continue;
      const uint32_t at = (uint32_t)(t_idx[k] - e_org) * sizeof(TI);
      const uint32_t ones = (sizeof(TI) == 4 ? 0xffffffffu : 0xffffu) << (8 * (at & 3));
      if ((atomicOr(&words[at >> 2], ones) & ones) == ones) s_twice = 1;
    }
    __syncthreads();
    for (int k = tid; k < a.K; k += NT) {
      if (!here(k)) continue;
      image[t_idx[k] - e_org] = (TI)-INFINITY;
      if (s_twice) {
        double g = 0.0;
        bool first = true;
        for (int j = 0; j < a.K; ++j)
          if (t_idx[j] == t_idx[k]) {
            if (j < k) first = false;
            g += (double)t_q[j];
          }
        t_g[k] = first ? (float)g : -1.f;
      }
    }
    __syncthreads();
  }

  // ---- maximum and sum
  Part part = {{-INFINITY, 0.f}, {-INFINITY, 0.f}, 0.f};
  if (OP != kLogpBwd) {
    float m = -INFINITY;
    float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);
    const float2 c2 = make_float2(a.c, a.c);
    const uint32_t none = minus_inf_word((const TI*)nullptr);
    for (int r = 0; r < rounds; ++r) {
      if (OP != kDistill) copy_wait(rounds - 1 - r);
      float2 x[U][EI / 2];
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = tid + (r * U + j) * NT;
        const uint4 u = i < np ? ((const uint4*)dyn)[i] : make_uint4(none, none, none, none);
        unpack(u, x[j], (const TI*)nullptr);
#pragma unroll
        for (int k = 0; k < EI / 2; ++k) mx = tc::fmax3(mx, x[j][k].x, x[j][k].y);
      }
      if (mx > m) {
        const float k = tc::fast_exp2((m - mx) * a.c);
        s0 = tc::fmul2(s0, make_float2(k, k));
        s1 = tc::fmul2(s1, make_float2(k, k));
        m = mx;
      }
      const float2 nb = make_float2(-base_of(m), -base_of(m));
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int k = 0; k < EI / 2; ++k) {
          const float2 t = tc::fmul2(tc::fadd2(x[j][k], nb), c2);
          const float2 e = make_float2(tc::fast_exp2(t.x), tc::fast_exp2(t.y));
          if (k & 1) s1 = tc::fadd2(s1, e);
          else s0 = tc::fadd2(s0, e);
        }
    }
    part.rest = warp_join({m, (s0.x + s0.y) + (s1.x + s1.y)}, a.c);
    if (OP == kDistill) {
      MaxSum in = {-INFINITY, 0.f};
      float n = 0.f;
      for (int k = tid; k < a.K; k += NT)
        if (!(t_g[k] < 0.f)) {
          in = join(in, {t_z[k], t_z[k] == -INFINITY ? 0.f : 1.f}, a.c);
          n += 1.f;
        }
      part.listed = warp_join(in, a.c);
      part.count = warp_sum(n);
    }
    if (lane == 0) s_warp[tid >> 5] = part;
    __syncthreads();
    auto add = [&](Part& to, const Part& p) {
      to.rest = join(to.rest, p.rest, a.c);
      if (OP == kDistill) {
        to.listed = join(to.listed, p.listed, a.c);
        to.count += p.count;
      }
    };
    part = s_warp[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) add(part, s_warp[i]);
    if (C > 1) {
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
      if (tid < C) {
        const uint32_t to = tc::mapa_shared(tc::smem_u32(&s_peer[rank]), (uint32_t)tid);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to),
                     "f"(part.rest.m), "f"(part.rest.s), "f"(part.listed.m), "f"(part.listed.s)
                     : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 16), "f"(part.count) : "memory");
      }
      tc::cluster_sync();
      part = s_peer[0];
      for (int i = 1; i < C; ++i) add(part, s_peer[i]);
    }
  }
  const MaxSum r = part.rest;

  // ---- the row's scalars: dz = c_out 2^((f z - b) c) + corrections
  float c_in = 0.f, b_in = 0.f, c_out = 0.f, hot = 0.f, b = base_of(r.m), f = 1.f, c = a.c;
  if (OP == kLogpBwd) {
    hot = (float)((double)a.dlogp[row] * a.inv_tau);
    c_out = -hot;
    f = (float)a.inv_tau;
    b = a.lse[row];
    c = (float)kLog2e;
  } else if (OP != kDistill) {
    if (tid == 0) {
      const double ls = log((double)r.s);
      const double logp = ((double)za - (double)b) * a.inv_tau - ls;
      if (rank == 0) {
        if (a.logp) a.logp[row] = (float)logp;
        if (OP == kLogp && a.logp_lo) a.logp_lo[row] = (float)(logp - (double)(float)logp);
        if (OP == kLogp && a.lse) a.lse[row] = (float)((double)b * a.inv_tau + ls);
      }
      if (OP == kPolicy) {
        const double A = a.advantage[row], ratio = exp(logp - (double)a.old_logp[row]);
        const double lo = 1.0 - a.clip_low, hi = 1.0 + a.clip_high;
        const bool clipped = (A > 0.0 && ratio > hi) || (A < 0.0 && ratio < lo);
        double l = clipped ? -(A > 0.0 ? hi : lo) * A : -ratio * A;
        double d = clipped ? 0.0 : -A * ratio;
        if (a.ref_logp) {
          const double gap = (double)a.ref_logp[row] - logp, e = expm1(gap);
          l += a.kl_coef * (e - gap);
          d -= a.kl_coef * e;
        }
        if (rank == 0) a.row_loss[row] = (float)((double)w * l);
        const double g = a.scale * (double)w * d * a.inv_tau;
        s_coef[0] = (float)g;
        s_coef[1] = (float)(-g / (double)r.s);
      }
    }
    if (OP == kLogp || !dz) return;
    __syncthreads();
    hot = s_coef[0];
    c_out = s_coef[1];
  } else {
    const MaxSum all = join(r, part.listed, a.c);
    // without an entry outside the list there is no class for the rest
    if (part.count == (float)V) q_rest = 0.0;
    const double ls = log((double)all.s), mx = (double)base_of(all.m) * a.inv_tau;
    double cross = 0.0;
    for (int k = tid; k < a.K; k += NT)
      if (t_q[k] != 0.f) cross += (double)t_q[k] * ((double)t_z[k] * a.inv_tau - mx - ls);
    if (rank == 0) {
      cross = block_sum_d(cross, s_red[0]);
      if (tid == 0) {
        double l = q_logq - cross;
        if (q_rest > 0.0)
          l += q_rest *
               (log(q_rest) - ((double)b * a.inv_tau + log((double)r.s) - mx - ls));
        a.row_loss[row] = (float)((double)w * l / (a.inv_tau * a.inv_tau));
      }
    }
    if (!dz) return;
    const double g = a.scale * (double)w / a.inv_tau;
    const double Q = q_sum + q_rest;
    c_in = (float)(g * Q / (double)all.s);
    b_in = base_of(all.m);
    // outside the list relative to the largest logit there: the student's
    // mass outside may be too small to be held relative to the row's largest
    // (none at all: an infinite loss, and entries of probability 0)
    c_out = r.s == 0.f ? 0.f
                       : (float)(g * (Q * (double)tc::fast_exp2((b - b_in) * a.c) / (double)all.s -
                                      (q_rest > 0.0 ? q_rest / (double)r.s : 0.0)));
    hot = (float)g;
  }

  // ---- the adjoint, in 16-byte units of dz; an image whose pieces do not
  // line up with them is read element by element
  if (OP == kLogpBwd) {
    copy_wait(0);
    __syncthreads();
  }
  const float2 f2 = make_float2(f, f), nb = make_float2(-b, -b), c2 = make_float2(c, c);
  auto value = [&](float x) { return c_out * tc::fast_exp2(fmaf(x, f, -b) * c); };
  const bool aligned = ((int)(u0 * EO - dph) - e_org) % EI == 0;
  auto unit = [&](int64_t u, auto lined_up) {
    const int e0 = (int)(u * EO - dph), at = e0 - e_org;
    float2 x[EO / 2];
    float v[EO];
    if constexpr (decltype(lined_up)::value) {
#pragma unroll
      for (int q = 0; q < EO / EI; ++q)
        unpack(((const uint4*)dyn)[at / EI + q], &x[q * (EI / 2)], (const TI*)nullptr);
    } else {
#pragma unroll
      for (int k = 0; k < EO / 2; ++k) x[k] = make_float2(ld(&image[at + 2 * k]), ld(&image[at + 2 * k + 1]));
    }
#pragma unroll
    for (int k = 0; k < EO / 2; ++k) {
      const float2 t = tc::fmul2(OP == kLogpBwd ? tc::ffma2(x[k], f2, nb) : tc::fadd2(x[k], nb), c2);
      v[2 * k] = c_out * tc::fast_exp2(t.x);
      v[2 * k + 1] = c_out * tc::fast_exp2(t.y);
    }
    if (OP != kDistill) {
      const int64_t d = token - e0;
      if (d >= 0 && d < EO) {
#pragma unroll
        for (int k = 0; k < EO; ++k)
          if (d == k) v[k] += hot;
      }
    }
    store_unit(dz + e0, v);
  };
  if (aligned) {
#pragma unroll 2
    for (int64_t u = u0 + tid; u < u1; u += NT) unit(u, std::true_type{});
  } else {
#pragma unroll 2
    for (int64_t u = u0 + tid; u < u1; u += NT) unit(u, std::false_type{});
  }
  ragged([&](int e) { st(&dz[e], value(ld(&image[e - e_org])) + (e == token ? hot : 0.f)); });
  if (OP == kDistill) {
    __syncthreads();
    for (int k = tid; k < a.K; k += NT)
      if (!(t_g[k] < 0.f))
        st(&dz[t_idx[k]], c_in * tc::fast_exp2((t_z[k] - b_in) * c) - hot * t_g[k]);
  }
}

// loss = scale * sum of l[0 .. n), in a fixed order.
__global__ void __launch_bounds__(1024) k_scaled_sum(const float* __restrict__ l, int64_t n,
                                                     double scale, float* __restrict__ loss) {
  __shared__ double red[32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)l[i];
  s = warp_sum_d(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 32; ++w) t += red[w];
    *loss = (float)(scale * t);
  }
}

// One CTA per pair: rows [off[2p], off[2p+1]) chosen, [off[2p+1], off[2p+2])
// rejected; the margin, the pair's loss, and each row's dlogp.  dlogp comes in
// holding what the rounding of logp to fp32 left out: a margin is a small
// difference of sums of log-probabilities, and would show it.
constexpr int kPairsPerLaunch = 128;
struct PairArgs {
  int64_t off[2 * kPairsPerLaunch + 1];
  int64_t V;
  const int64_t* tokens;
  const float *weight, *logp, *ref_logp;
  double beta, smoothing, scale;
  int normalize;
  float *pair_loss, *margin, *dlogp;
};
__global__ void __launch_bounds__(kRowThreads) k_preference_pair(const __grid_constant__ PairArgs a) {
  __shared__ double s_red[kRowThreads / 32];
  const int64_t* off = a.off + 2 * blockIdx.x;
  auto weight_of = [&](int64_t t) {
    const int64_t k = a.tokens[t];
    return k < 0 || k >= a.V ? 0.f : (a.weight ? a.weight[t] : 1.f);
  };
  double sum[2], len[2];
  for (int q = 0; q < 2; ++q) {
    double s = 0.0, n = 0.0;
    for (int64_t t = off[q] + threadIdx.x; t < off[q + 1]; t += kRowThreads) {
      const float w = weight_of(t);
      if (w == 0.f) continue;
      s += (double)w * ((double)a.logp[t] - (a.ref_logp ? (double)a.ref_logp[t] : 0.0) +
                        (double)a.dlogp[t]);
      n += (double)w;
    }
    sum[q] = block_sum_d(s, s_red);
    len[q] = a.normalize ? block_sum_d(n, s_red) : 1.0;
    if (len[q] != 0.0) sum[q] /= len[q];
  }
  const double m = a.beta * (sum[0] - sum[1]);
  // -log sigma(v) = max(-v, 0) + log(1 + exp(-|v|))
  const double tail = log1p(exp(-fabs(m)));
  const double l = (1.0 - a.smoothing) * (fmax(-m, 0.0) + tail) + a.smoothing * (fmax(m, 0.0) + tail);
  const double dm = a.smoothing / (1.0 + exp(-m)) - (1.0 - a.smoothing) / (1.0 + exp(m));
  if (threadIdx.x == 0) {
    a.pair_loss[blockIdx.x] = (float)l;
    a.margin[blockIdx.x] = (float)m;
  }
  for (int q = 0; q < 2; ++q) {
    const double g = (q ? -dm : dm) * a.beta * a.scale / (len[q] != 0.0 ? len[q] : 1.0);
    for (int64_t t = off[q] + threadIdx.x; t < off[q + 1]; t += kRowThreads) {
      const float w = weight_of(t);
      a.dlogp[t] = w == 0.f ? 0.f : (float)(g * (double)w);
    }
  }
}

// ------------------------------------------------------------------- host
template <RowOp OP>
void launch_rows(RowArgs a, int64_t rows, int prec, int grad_prec, cudaStream_t s) {
  if (rows == 0) return;
  const int64_t bytes = a.V * (prec == DOP_BF16 ? 2 : 4) + 16;
  int64_t C = ceil_div(bytes, kStageBytes);
  if (C > kMaxCluster) {
    C = kMaxCluster;
    if (ceil_div(bytes, C) > kStageBytesMost - 16)
      throw Error(DOP_E_UNSUPPORTED, "vocab (" + std::to_string(a.V) + ") is above " +
                                         std::to_string(kMaxCluster * (kStageBytesMost - 32) /
                                                        (prec == DOP_BF16 ? 2 : 4)));
  }
  if (rows * C > INT32_MAX) throw Error(DOP_E_UNSUPPORTED, "too many rows for this vocab");
  a.cluster = (int)C;
  a.stage_bytes = (int)round_up(ceil_div(bytes, C) + 16, 16);
  const size_t smem = (size_t)a.stage_bytes + (OP == kDistill ? 16 * (size_t)a.K : 0);
  auto go = [&](auto ti, auto to) {
    auto kern = k_vocab_row<OP, decltype(ti), decltype(to)>;
    DOP_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kStageBytesMost + 16 * kMaxTeacherK)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C > 1 ? 1 : 0;
    DOP_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  };
  if (prec == DOP_BF16) go(bf16{}, bf16{});
  else if (a.dz && grad_prec == DOP_BF16) go(0.f, bf16{});
  else go(0.f, 0.f);
}

int elem_bytes(int prec) { return prec == DOP_BF16 ? 2 : 4; }

// The checks every objective shares.
void check_rows(int64_t rows, int64_t vocab, int prec, const void* z, int64_t ld, double tau) {
  DOP_REQUIRE(rows >= 0 && rows <= INT32_MAX, "rows must lie in [0, 2^31)");
  DOP_REQUIRE(vocab >= 1 && vocab <= INT32_MAX, "vocab must lie in [1, 2^31)");
  DOP_REQUIRE(prec == DOP_F32 || prec == DOP_BF16, "unknown precision");
  DOP_REQUIRE(ld >= vocab, "the logits' row stride is smaller than vocab");
  DOP_REQUIRE(z || rows == 0, "null logits");
  DOP_REQUIRE((uintptr_t)z % elem_bytes(prec) == 0, "misaligned logits");
  DOP_REQUIRE(std::isfinite(tau) && tau > 0.0, "temperature must be finite and positive");
}
// dlogits: bf16 or the logits' type; either exactly the logits' memory (same
// type and stride) or apart from it.
void check_grad(int64_t rows, int64_t vocab, int prec, const void* z, int64_t ld, int grad_prec,
                const void* dz, int64_t ldd) {
  if (!dz) return;
  DOP_REQUIRE(grad_prec == DOP_F32 || grad_prec == DOP_BF16, "unknown gradient precision");
  DOP_REQUIRE(prec == DOP_F32 || grad_prec == DOP_BF16, "bf16 logits have bf16 dlogits");
  DOP_REQUIRE(ldd >= vocab, "the row stride of dlogits is smaller than vocab");
  DOP_REQUIRE((uintptr_t)dz % elem_bytes(grad_prec) == 0, "misaligned dlogits");
  if (rows == 0 || (dz == z && prec == grad_prec && ld == ldd)) return;
  const char *z0 = (const char*)z, *d0 = (const char*)dz;
  const char* z1 = z0 + ((rows - 1) * ld + vocab) * elem_bytes(prec);
  const char* d1 = d0 + ((rows - 1) * ldd + vocab) * elem_bytes(grad_prec);
  DOP_REQUIRE(z1 <= d0 || d1 <= z0,
              "dlogits overlaps the logits without being the same rows in the same type");
}

RowArgs row_args(int64_t vocab, const void* z, int64_t ld, const int64_t* tokens,
                 const float* weight, double tau) {
  RowArgs a{};
  a.z = z;
  a.ld = ld;
  a.V = vocab;
  a.tokens = tokens;
  a.weight = weight;
  a.inv_tau = 1.0 / tau;
  a.c = (float)(kLog2e / tau);
  return a;
}

void scaled_sum(const float* l, int64_t n, double scale, float* loss, cudaStream_t s) {
  k_scaled_sum<<<1, 1024, 0, s>>>(l, n, scale, loss);
  DOP_CHECK_CUDA(cudaGetLastError());
}

template <typename F>
int guarded(F&& f) {
  try {
    f();
    return DOP_OK;
  } catch (const Error& e) {
    return set_last_error(e.code, e.what());
  } catch (const std::bad_alloc&) {
    return set_last_error(DOP_E_NOMEM, "host allocation failed");
  } catch (const std::exception& e) {
    return set_last_error(DOP_E_INVALID, e.what());
  }
}
cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace
}  // namespace dop

using namespace dop;

extern "C" {

int dop_token_logp(int64_t rows, int64_t vocab, int precision, const void* logits, int64_t ld,
                   const int64_t* tokens, const float* weight, double temperature, float* logp,
                   float* lse, void* stream) {
  return guarded([&] {
    check_rows(rows, vocab, precision, logits, ld, temperature);
    DOP_REQUIRE((tokens && logp && lse) || rows == 0, "null pointer");
    RowArgs a = row_args(vocab, logits, ld, tokens, weight, temperature);
    a.logp = logp;
    a.lse = lse;
    launch_rows<kLogp>(a, rows, precision, DOP_F32, as_stream(stream));
  });
}

int dop_token_logp_backward(int64_t rows, int64_t vocab, int precision, const void* logits,
                            int64_t ld, const int64_t* tokens, const float* lse,
                            const float* dlogp, double temperature, int grad_precision,
                            void* dlogits, int64_t ldd, void* stream) {
  return guarded([&] {
    check_rows(rows, vocab, precision, logits, ld, temperature);
    DOP_REQUIRE((tokens && lse && dlogp && dlogits) || rows == 0, "null pointer");
    check_grad(rows, vocab, precision, logits, ld, grad_precision, dlogits, ldd);
    RowArgs a = row_args(vocab, logits, ld, tokens, nullptr, temperature);
    a.lse = const_cast<float*>(lse);
    a.dlogp = dlogp;
    a.dz = dlogits;
    a.ldd = ldd;
    launch_rows<kLogpBwd>(a, rows, precision, grad_precision, as_stream(stream));
  });
}

int dop_policy_loss_grad(int64_t rows, int64_t vocab, int precision, const void* logits,
                         int64_t ld, const int64_t* tokens, const float* old_logp,
                         const float* advantage, const float* ref_logp, const float* weight,
                         double temperature, double clip_low, double clip_high, double kl_coef,
                         double scale, float* loss, float* row_loss, float* logp,
                         int grad_precision, void* dlogits, int64_t ldd, void* stream) {
  return guarded([&] {
    check_rows(rows, vocab, precision, logits, ld, temperature);
    DOP_REQUIRE(loss && ((tokens && old_logp && advantage && row_loss && logp) || rows == 0),
                "null pointer");
    DOP_REQUIRE(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0 && std::isfinite(clip_high),
                "the clip must satisfy 0 <= low <= 1 and 0 <= high");
    DOP_REQUIRE(std::isfinite(kl_coef) && std::isfinite(scale), "kl_coef and scale must be finite");
    DOP_REQUIRE(kl_coef == 0.0 || ref_logp || rows == 0, "a KL term needs ref_logp");
    check_grad(rows, vocab, precision, logits, ld, grad_precision, dlogits, ldd);
    RowArgs a = row_args(vocab, logits, ld, tokens, weight, temperature);
    a.old_logp = old_logp;
    a.advantage = advantage;
    a.ref_logp = kl_coef != 0.0 ? ref_logp : nullptr;
    a.clip_low = clip_low;
    a.clip_high = clip_high;
    a.kl_coef = kl_coef;
    a.scale = scale;
    a.row_loss = row_loss;
    a.logp = logp;
    a.dz = dlogits;
    a.ldd = ldd;
    launch_rows<kPolicy>(a, rows, precision, grad_precision, as_stream(stream));
    scaled_sum(row_loss, rows, scale, loss, as_stream(stream));
  });
}

int dop_preference_loss_grad(int64_t rows, int64_t vocab, int precision, const void* logits,
                             int64_t ld, const int64_t* tokens, int64_t pairs,
                             const int64_t* seq_off, const float* ref_logp, const float* weight,
                             double temperature, double beta, double label_smoothing,
                             int length_normalize, double scale, float* loss, float* pair_loss,
                             float* margin, float* logp, float* lse, float* dlogp,
                             int grad_precision, void* dlogits, int64_t ldd, void* stream) {
  return guarded([&] {
    check_rows(rows, vocab, precision, logits, ld, temperature);
    DOP_REQUIRE(pairs >= 0, "pairs must not be negative");
    DOP_REQUIRE(loss && seq_off && ((pair_loss && margin) || pairs == 0) &&
                    ((tokens && logp && lse && dlogp) || rows == 0),
                "null pointer");
    DOP_REQUIRE(std::isfinite(beta) && std::isfinite(scale), "beta and scale must be finite");
    DOP_REQUIRE(label_smoothing >= 0.0 && label_smoothing <= 1.0,
                "label_smoothing must lie in [0, 1]");
    DOP_REQUIRE(seq_off[0] >= 0, "seq_off must start at 0 or later");
    for (int64_t i = 0; i < 2 * pairs; ++i)
      DOP_REQUIRE(seq_off[i] <= seq_off[i + 1], "seq_off must not decrease");
    DOP_REQUIRE(seq_off[2 * pairs] <= rows, "seq_off ends behind the last row");
    check_grad(rows, vocab, precision, logits, ld, grad_precision, dlogits, ldd);
    cudaStream_t s = as_stream(stream);
    const int64_t a0 = seq_off[0], a1 = seq_off[2 * pairs];
    const int zb = elem_bytes(precision);
    // rows of no sequence
    for (int64_t part = 0; part < 2; ++part) {
      const int64_t lo = part ? a1 : 0, n = (part ? rows : a0) - lo;
      if (n == 0) continue;
      for (float* p : {logp, lse, dlogp})
        DOP_CHECK_CUDA(cudaMemsetAsync(p + lo, 0, sizeof(float) * n, s));
    }
    RowArgs f = row_args(vocab, (const char*)logits + a0 * ld * zb, ld, tokens + a0,
                         weight ? weight + a0 : nullptr, temperature);
    f.logp = logp + a0;
    f.lse = lse + a0;
    f.logp_lo = dlogp + a0;
    launch_rows<kLogp>(f, a1 - a0, precision, DOP_F32, s);
    for (int64_t p0 = 0; p0 < pairs; p0 += kPairsPerLaunch) {
      const int64_t n = std::min<int64_t>(pairs - p0, kPairsPerLaunch);
      PairArgs pa{};
      for (int64_t i = 0; i <= 2 * n; ++i) pa.off[i] = seq_off[2 * p0 + i];
      pa.V = vocab;
      pa.tokens = tokens;
      pa.weight = weight;
      pa.logp = logp;
      pa.ref_logp = ref_logp;
      pa.beta = beta;
      pa.smoothing = label_smoothing;
      pa.scale = scale;
      pa.normalize = length_normalize != 0;
      pa.pair_loss = pair_loss + p0;
      pa.margin = margin + p0;
      pa.dlogp = dlogp;
      k_preference_pair<<<(unsigned)n, kRowThreads, 0, s>>>(pa);
      DOP_CHECK_CUDA(cudaGetLastError());
    }
    if (dlogits) {
      RowArgs b = row_args(vocab, logits, ld, tokens, nullptr, temperature);
      b.lse = lse;
      b.dlogp = dlogp;
      b.dz = dlogits;
      b.ldd = ldd;
      launch_rows<kLogpBwd>(b, rows, precision, grad_precision, s);
    }
    scaled_sum(pair_loss, pairs, scale, loss, s);
  });
}

int dop_distill_loss_grad(int64_t rows, int64_t vocab, int precision, const void* logits,
                          int64_t ld, int64_t top_k, const int32_t* top_index,
                          const float* top_logit, const float* teacher_lse, const float* weight,
                          double temperature, double scale, float* loss, float* row_loss,
                          int grad_precision, void* dlogits, int64_t ldd, void* stream) {
  return guarded([&] {
    check_rows(rows, vocab, precision, logits, ld, temperature);
    DOP_REQUIRE(loss && ((top_index && top_logit && row_loss) || rows == 0), "null pointer");
    DOP_REQUIRE(std::isfinite(scale), "scale must be finite");
    DOP_REQUIRE(top_k >= 1, "top_k must be at least 1");
    if (top_k > kMaxTeacherK)
      throw Error(DOP_E_UNSUPPORTED, "top_k (" + std::to_string(top_k) + ") is above " +
                                         std::to_string(kMaxTeacherK));
    check_grad(rows, vocab, precision, logits, ld, grad_precision, dlogits, ldd);
    RowArgs a = row_args(vocab, logits, ld, nullptr, weight, temperature);
    a.K = (int)top_k;
    a.top_index = top_index;
    a.top_logit = top_logit;
    a.teacher_lse = teacher_lse;
    a.scale = scale;
    a.row_loss = row_loss;
    a.dz = dlogits;
    a.ldd = ldd;
    launch_rows<kDistill>(a, rows, precision, grad_precision, as_stream(stream));
    scaled_sum(row_loss, rows, scale, loss, as_stream(stream));
  });
}

}  // extern "C"
