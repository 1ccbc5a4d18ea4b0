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
#include <cstring>
#include <mutex>
#include <set>
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
constexpr int kOnceThreads = 128, kOnceCtas = 8;
constexpr int kRing = 8;  // pieces that a thread reading a row once has under way
// Shared memory: of a CTA when three are to fit an SM (of its 228 KB, less the
// static share and what the system takes of each), and of a CTA's pieces at most.
constexpr int64_t kCtaBytes = 228 * 1024 / 3 - 2560, kStageBytesMost = 200 * 1024;
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;

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
  int64_t rows, in_lo, in_hi;  // rows outside [in_lo, in_hi) are skipped
  const float* sum_of;  // the preference loss: scale times the sum of these,
  int64_t sum_n;        // taken with the adjoint
  float* loss;
  int cluster;      // CTAs per row
  int share;        // 16-byte pieces of a row a CTA has
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

// Powers of two of a row are taken relative to its maximum m as
// 2^(c z - b) with b = rint(c m), a whole number: one fused multiply-add an
// element, no rounding of b, and sums with different b differ by exact powers
// of two.  (c is log2(e) / tau rounded to fp32, for every term of a row alike:
// a relative change of the temperature by at most 2^-24.)  b is held within
// +-1e30.  Where c m would pass that, or a row is all of the type's lowest
// value, two elements are equal or at least 2^60 apart: beyond 1e25 a row is
// far, and its powers are taken of (z - m) 2^-40, which is exact.
constexpr float kFar = 1e30f;
__device__ __forceinline__ float base_of(float m, float c) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: to a whole number without a conversion
  return fminf(fmaxf((c * m + kRound) - kRound, -kFar), kFar);
}
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > 1e25f && m != -INFINITY; }
struct Form {
  float c, b;  // 2^(c z - b)
};
__device__ __forceinline__ Form form_of(float m, float c) {
  if (is_far(m)) return {0x1p-40f, m * 0x1p-40f};
  return {c, base_of(m, c)};
}
// A maximum and the sum of 2^(c z - b) of its form; nothing: {-inf, 0}.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float warp_max_redux(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// The warp's maximum and sum; the sum of a far row is not one yet.
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
  const float m = warp_max_redux(v.m);
  return {m, warp_sum(v.s * tc::fast_exp2(base_of(v.m, c) - base_of(m, c)))};
}
// What turns a sum relative to m into one relative to `to` >= m.
__device__ __forceinline__ float rescale(float m, float to, float c) {
  if (m == to) return 1.f;
  if (is_far(m) || is_far(to)) return 0.f;
  return tc::fast_exp2(base_of(m, c) - base_of(to, c));
}
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * rescale(a.m, m, c) + b.s * rescale(b.m, m, c)};
}
// (z - m) / tau, to which log(s) is to be taken from, in double.
__device__ __forceinline__ double above(float z, float m, float c, double inv_tau) {
  if (is_far(m)) return ((double)z - (double)m) * inv_tau;
  return ((double)z * (double)c - (double)base_of(m, c)) * kLn2;
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
// N consecutive elements (N sizeof(T) is 8 or 16, and aligned to that).
__device__ __forceinline__ void store_n(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_n(bf16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(tc::pack_bf16(v[0], v[1]), tc::pack_bf16(v[2], v[3]));
}
__device__ __forceinline__ void store_n(bf16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(tc::pack_bf16(v[0], v[1]), tc::pack_bf16(v[2], v[3]),
                                            tc::pack_bf16(v[4], v[5]), tc::pack_bf16(v[6], v[7]));
}

// Bits of the filter that finds out whether a list may name an entry twice.
constexpr int kFilterBits = 32768;
// A list's arrays start at 16-byte borders.
__host__ __device__ constexpr int list_stride(int K) { return (K + 3) & ~3; }

// ln(s), to about 2^-24 of it or of 1: the exponent apart (0, subnormal, inf
// and NaN as log has them).
__device__ __forceinline__ double ln(float s) {
  if (!(s > 0x1p-126f && s < INFINITY)) return (double)logf(s);
  const int e = (__float_as_int(s) - 0x3f400000) >> 23;  // s = 2^e f, f in [0.75, 1.5)
  return (double)e * kLn2 + (double)logf(__int_as_float(__float_as_int(s) - (e << 23)));
}

// A cluster of a.cluster CTAs per row: 256 threads own the pieces, and
// distillation has a warp more for the teacher's list.
template <RowOp OP>
constexpr int kOwnersOf = OP == kLogp ? kOnceThreads : kRowThreads;
template <RowOp OP>
constexpr int kThreadsOf = kOwnersOf<OP> + (OP == kDistill ? 32 : 0);
template <RowOp OP>
constexpr int kCtasPerSM = OP == kLogp ? kOnceCtas : 3;

template <RowOp OP, typename TI, typename TO>
__device__ __forceinline__ void vocab_row(const RowArgs& a, const int64_t row, const int rank) {
  constexpr int EI = 16 / (int)sizeof(TI);
  constexpr int NT = kOwnersOf<OP>, NW = NT / 32, U = OP == kLogp ? 2 : 4;
  extern __shared__ __align__(16) uint8_t dyn[];
  // of every warp of the cluster
  __shared__ MaxSum s_rest[kMaxCluster * NW];
  __shared__ float s_again[2 * kMaxCluster * NW];
  // of every CTA: the listed entries' m, s, count; the sum of q times the logit
  __shared__ __align__(16) float4 s_listed[kMaxCluster];
  __shared__ double s_qz[kMaxCluster];
  __shared__ double s_q[3];
  __shared__ int s_twice;
  const int C = a.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool owner = OP != kDistill || tid < NT;  // of pieces
  const float w = a.weight ? a.weight[row] : 1.f;
  const int64_t token64 = OP == kDistill ? -1 : a.tokens[row];
  const float dlogp = OP == kLogpBwd ? a.dlogp[row] : 0.f;
  const float lse_in = OP == kLogpBwd ? a.lse[row] : 0.f;
  const float adv = OP == kPolicy ? a.advantage[row] : 0.f;
  const float old_logp = OP == kPolicy ? a.old_logp[row] : 0.f;
  const float ref_logp = OP == kPolicy && a.ref_logp ? a.ref_logp[row] : 0.f;

  int32_t my_idx = -1;
  float my_top = 0.f;
  if (OP == kDistill && tid < NT && tid < a.K) {
    my_idx = a.top_index[row * a.K + tid];
    my_top = a.top_logit[row * a.K + tid];
  }

  const TI* z = (const TI*)a.z + row * a.ld;
  TO* dz = a.dz ? (TO*)a.dz + row * a.ldd : nullptr;
  const int V = (int)a.V, token = (int)token64;
  // this CTA's pieces [p0, p0 + np) and elements [e_lo, e_hi)
  const int ph = (int)((uintptr_t)z & 15) / (int)sizeof(TI);
  const int pieces = (ph + V + EI - 1) / EI;
  const int p0 = min(pieces, rank * a.share), np = min(pieces, p0 + a.share) - p0;
  const int e_org = p0 * EI - ph;  // the row's element at image element 0
  const int e_lo = max(0, e_org), e_hi = max(e_lo, min(V, e_org + np * EI));
  // pieces that lie in the row altogether: [f0, f1)
  const int f0 = e_org < 0 ? 1 : 0, f1 = e_org + np * EI > V ? np - 1 : np;

  if (w == 0.f || row < a.in_lo || row >= a.in_hi || (OP != kDistill && (token64 < 0 || token64 >= V)) ||
      (OP == kLogpBwd && dlogp == 0.f)) {
    if (dz) {
      constexpr int EO = 16 / (int)sizeof(TO);
      const int dph = (int)((uintptr_t)dz & 15) / (int)sizeof(TO);
      const int u0 = (dph + e_lo + EO - 1) / EO, u1 = (dph + e_hi) / EO;  // 16-byte units
      const int ahead = u0 < u1 ? u0 * EO - dph : e_hi, behind = u0 < u1 ? u1 * EO - dph : e_hi;
      for (int u = u0 + tid; u < u1; u += kThreadsOf<OP>)
        *reinterpret_cast<uint4*>(dz + (u * EO - dph)) = make_uint4(0u, 0u, 0u, 0u);
      if (e_lo + tid < ahead) st(&dz[e_lo + tid], 0.f);
      if (behind + tid < e_hi) st(&dz[behind + tid], 0.f);
    }
    if (tid == 0 && rank == 0) {
      if (OP != kLogpBwd && OP != kDistill && a.logp) a.logp[row] = 0.f;
      if (OP == kLogp && a.lse) a.lse[row] = 0.f;
      if (OP == kLogp && a.logp_lo) a.logp_lo[row] = 0.f;
      if (OP == kPolicy || OP == kDistill) a.row_loss[row] = 0.f;
    }
    return;
  }
  constexpr bool stats = OP != kLogpBwd;  // it has lse
  // every CTA of the cluster has started once this barrier is through: its
  // shared memory may be written to
  if (stats && C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ---- copy this CTA's pieces; a thread owns pieces tid + NT k, and the
  // first `mine` of them are the row's
  // (the log-probability reads its pieces once, in a ring of kRing of them)
  constexpr bool kOnce = OP == kLogp;
  TI* image = (TI*)dyn;
  uint4* at = (uint4*)dyn + tid;  // piece k: at[k NT], in the ring at[(k % kRing) NT]
  auto place = [&](int k) { return kOnce ? (k % kRing) * NT : k * NT; };
  const int mine = owner && tid < np ? (np - tid + NT - 1) / NT : 0;
  // the first and the last piece of the row may be in part outside it
  auto edge = [&](int i) {
    TI v[EI];
#pragma unroll
    for (int k = 0; k < EI; ++k) {
      const int e = e_org + i * EI + k;
      v[k] = e >= 0 && e < V ? z[e] : (TI)-INFINITY;
    }
    uint4 u;
    memcpy(&u, v, 16);
    return u;
  };
  const uint4* src = (const uint4*)(z + e_org) + tid;
  const uint32_t dst = tc::smem_u32(at);
  auto whole = [&](int k) { return tid + k * NT >= f0 && tid + k * NT < f1; };
  auto copy_whole = [&](int k) {
    if (whole(k)) copy_piece(dst + place(k) * 16, src + k * NT);
  };
  if (owner) {
    const int n = kOnce ? min(mine, kRing) : mine;
    int k = 0;
    for (; k + U <= n; k += U) {
      if (tid + k * NT >= f0 && tid + (k + U - 1) * NT < f1) {
#pragma unroll
        for (int j = 0; j < U; ++j) copy_piece(dst + place(k + j) * 16, src + (k + j) * NT);
      } else {
        for (int j = 0; j < U; ++j) copy_whole(k + j);
      }
      copy_commit();
    }
    for (; k < n; ++k) copy_whole(k);
    copy_commit();
    // the two that a row may share with what lies beside it, while the copies run
    if (f0 == 1 && tid == 0 && n > 0) at[0] = edge(0);
    if (f1 < np && f1 >= f0 && tid == f1 % NT && f1 / NT < n) at[place(f1 / NT)] = edge(f1);
  }
  // piece k once more, after its copy (a ring may have given it up)
  auto piece = [&](int k) {
    const int i = tid + k * NT;
    return !kOnce ? at[k * NT] : i >= f0 && i < f1 ? src[k * NT] : edge(i);
  };
  const float za = OP == kDistill || OP == kLogpBwd ? 0.f : ld(&z[token]);

  // ---- the teacher's list leaves the image.  While the copies run, the
  // owners put the list into shared memory and find out whether an entry may
  // be named twice (two entries on one bit of a filter); the warp that owns
  // no pieces works out q while the others take the maximum and sum.
  const int K4 = OP == kDistill ? list_stride(a.K) : 0;
  int32_t* t_idx = (int32_t*)(dyn + a.stage_bytes);
  float* t_q = (float*)t_idx + K4;  // the teacher's logit, then q
  float* t_z = t_q + K4;            // the student's logit, of this CTA's entries
  float* t_g = t_z + K4;            // this CTA's first ones: sum of q of the entry; else -1
  if (OP == kDistill) {
    uint32_t* filter = (uint32_t*)(t_g + K4);
    if (owner) {
      for (int i = tid; i < kFilterBits / 128; i += NT) ((uint4*)filter)[i] = make_uint4(0u, 0u, 0u, 0u);
      if (tid == 0) s_twice = 0;
      asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
      for (int k = tid; k < a.K; k += NT) {
        const int32_t i = k < NT ? my_idx : a.top_index[row * a.K + k];
        const float y = k < NT ? my_top : a.top_logit[row * a.K + k];
        const bool in = i >= 0 && i < V;
        t_idx[k] = in ? i : -1;
        t_q[k] = in ? y : -INFINITY;
        if (in) {
          const uint32_t h = (uint32_t)i % kFilterBits, bit = 1u << (h & 31);
          if (atomicOr(&filter[h >> 5], bit) & bit) s_twice = 1;
        }
      }
    }
    copy_wait(0);
    __syncthreads();
    for (int k = tid; k < a.K; k += kThreadsOf<OP>) {
      const int i = t_idx[k];
      const bool here = i >= e_lo && i < e_hi;
      t_z[k] = here ? ld(&image[i - e_org]) : 0.f;
      t_g[k] = here ? 0.f : -1.f;
      if (!s_twice && here) image[i - e_org] = (TI)-INFINITY;
    }
    __syncthreads();
    if (s_twice) {
      for (int k = tid; k < a.K; k += kThreadsOf<OP>)
        if (t_g[k] == 0.f) image[t_idx[k] - e_org] = (TI)-INFINITY;
      __syncthreads();
    }
  }
  // q of the list, its sums, and which entries are a vocabulary entry's first
  auto make_q = [&] {
    MaxSum t = {-INFINITY, 0.f};
    double tl = 0.0;
    if (a.teacher_lse) {
      tl = (double)a.teacher_lse[row];
    } else {
      for (int k = lane; k < a.K; k += 32) t.m = fmaxf(t.m, t_q[k]);
      t.m = warp_max_redux(t.m);
      const Form f = form_of(t.m, a.c);
      for (int k = lane; k < a.K; k += 32) t.s += tc::fast_exp2(fmaf(t_q[k], f.c, -f.b));
      tl = ln(warp_sum(t.s));
    }
    double qs = 0.0, ql = 0.0;
    for (int k = lane; k < a.K; k += 32) {
      const float y = t_q[k];
      const double lq = (a.teacher_lse ? (double)y * a.inv_tau : above(y, t.m, a.c, a.inv_tau)) - tl;
      const float hi = (float)lq;  // q to fp32's last digits: lq rounded, the rest applied
      const float q = y == -INFINITY ? 0.f : expf(hi) * (1.f + (float)(lq - (double)hi));
      t_q[k] = q;
      if (t_g[k] == 0.f) t_g[k] = q;
      qs += (double)q;
      if (q > 0.f) ql += (double)q * lq;
    }
    qs = warp_sum_d(qs);
    ql = warp_sum_d(ql);
    __syncwarp();
    if (s_twice)
      for (int k = lane; k < a.K; k += 32) {
        const int i = t_idx[k];
        if (t_g[k] < 0.f) continue;
        double sum = 0.0;
        bool first = true;
        for (int j = 0; j < a.K; ++j)
          if (t_idx[j] == i) {
            if (j < k) first = false;
            sum += (double)t_q[j];
          }
        t_g[k] = first ? (float)sum : -1.f;
      }
    __syncwarp();
    if (lane == 0) {
      s_q[0] = qs;
      s_q[1] = ql;
      s_q[2] = a.teacher_lse ? fmax(0.0, 1.0 - qs) : 0.0;
    }
  };

  // ---- maximum and sum
  MaxSum rest = {-INFINITY, 0.f}, listed = {-INFINITY, 0.f};
  float count = 0.f;
  // v to slot `to` of every CTA of the cluster (lane r: of CTA r)
  auto tell = [&](auto* to, auto v) {
    if (C == 1) {
      if (lane == 0) *to = v;
    } else if (lane < C) {
      const uint32_t there = tc::mapa_shared(tc::smem_u32(to), (uint32_t)lane);
      uint32_t word[sizeof(v) / 4];
      memcpy(word, &v, sizeof(v));
#pragma unroll
      for (int i = 0; i < (int)sizeof(v) / 4; ++i)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + 4 * i), "r"(word[i]) : "memory");
    }
  };
  auto told = [&] {
    if (C > 1) tc::cluster_sync();
    else __syncthreads();
  };
  if constexpr (stats) {
    const uint32_t none = minus_inf_word((const TI*)nullptr);
    if (owner) {
      // the sum is taken relative to the largest of the first pieces; should
      // a later element pass that by 2^127, the sum says so and is taken
      // again relative to the maximum of all
      float m = -INFINITY;
      float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f), nb = s0;
      const float2 c2 = make_float2(a.c, a.c);
      auto largest = [&](uint4 u) {
        float2 x[EI / 2];
        unpack(u, x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i) m = tc::fmax3(m, x[i].x, x[i].y);
      };
      auto add = [&](uint4 u) {
        float2 x[EI / 2];
        unpack(u, x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i) {
          const float2 t = tc::ffma2(x[i], c2, nb);
          const float2 e = make_float2(tc::fast_exp2(t.x), tc::fast_exp2(t.y));
          if (i & 1) s1 = tc::fadd2(s1, e);
          else s0 = tc::fadd2(s0, e);
        }
      };
      auto relative_to_m = [&] { nb.x = nb.y = -base_of(m, a.c); };
      auto sum = [&] { return (s0.x + s0.y) + (s1.x + s1.y); };
      int k = 0;
      for (; k + U <= mine; k += U) {
        // group g of the copies ends with piece (g + 1) U at the latest; a
        // ring keeps kRing / U groups under way
        if (kOnce) copy_wait(mine > kRing ? kRing / U - 1 : max(0, mine / U - 1 - k / U));
        else if (OP != kDistill) copy_wait(max(0, mine / U - 1 - k / U));
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = at[place(k + j)];
        if (k == 0) {
#pragma unroll
          for (int j = 0; j < U; ++j) largest(u[j]);
          relative_to_m();
        }
#pragma unroll
        for (int j = 0; j < U; ++j) add(u[j]);
        if (kOnce && mine > kRing) {
          // (add() has used u: its place is free)
          for (int j = 0; j < U; ++j)
            if (k + kRing + j < mine) {
              copy_whole(k + kRing + j);
              if (!whole(k + kRing + j)) at[place(k + kRing + j)] = edge(tid + (k + kRing + j) * NT);
            }
          copy_commit();
        }
      }
      if (OP != kDistill) copy_wait(0);
      if (k < mine) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
          u[j] = k + j < mine ? at[place(k + j)] : make_uint4(none, none, none, none);
        if (k == 0) {
#pragma unroll
          for (int j = 0; j < U; ++j) largest(u[j]);
          relative_to_m();
        }
#pragma unroll
        for (int j = 0; j < U; ++j) add(u[j]);
      }
      if (!(sum() < INFINITY)) {
        for (k = 0; k < mine; ++k) largest(piece(k));
        relative_to_m();
        s0 = s1 = make_float2(0.f, 0.f);
        for (k = 0; k < mine; ++k) add(piece(k));
      }
      rest = warp_join({m, sum()}, a.c);
    }
    double qz = 0.0;
    if (!owner) {
      make_q();
      for (int k = lane; k < a.K; k += 32) {
        const int i = t_idx[k];
        if (i >= e_lo && i < e_hi && t_q[k] != 0.f) qz += (double)t_q[k] * (double)t_z[k];
        if (t_g[k] < 0.f) continue;
        listed.m = fmaxf(listed.m, t_z[k]);
        count += 1.f;
      }
      qz = warp_sum_d(qz);
      listed.m = warp_max_redux(listed.m);
      const Form f = form_of(listed.m, a.c);
      for (int k = lane; k < a.K; k += 32)
        if (!(t_g[k] < 0.f)) listed.s += tc::fast_exp2(fmaf(t_z[k], f.c, -f.b));
      listed.s = warp_sum(listed.s);
      count = warp_sum(count);
    }
    // every warp's to every CTA of the cluster, joined there in a fixed order
    if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (owner) {
      tell(&s_rest[rank * NW + warp], rest);
    } else {
      tell(&s_listed[rank], make_float4(listed.m, listed.s, count, 0.f));
      tell(&s_qz[rank], qz);
    }
    told();
    if (OP == kLogp && C == 1 && warp != 0) {
      // (a far row needs them all once more)
      bool far = false;
      for (int i = 0; i < NW; ++i) far = far || is_far(s_rest[i].m);
      if (!far) return;
    }
    rest = {-INFINITY, 0.f};
    if (lane < C * NW) rest = s_rest[lane];
    if (C * NW > 32 && lane + 32 < C * NW) rest = join(rest, s_rest[lane + 32], a.c);
    rest = warp_join(rest, a.c);
    if (is_far(rest.m)) {
      // the row's maximum, which is not that of the first pieces, and the sum
      // in its form: two exchanges more
      auto exchange = [&](float v, float* slots) {
        if (owner) tell(&slots[rank * NW + warp], v);
        told();
      };
      float v = -INFINITY;
      for (int k = 0; k < mine; ++k) {
        float2 x[EI / 2];
        unpack(piece(k), x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i) v = tc::fmax3(v, x[i].x, x[i].y);
      }
      exchange(warp_max_redux(v), s_again);
      v = -INFINITY;
      for (int i = lane; i < C * NW; i += 32) v = fmaxf(v, s_again[i]);
      rest.m = warp_max_redux(v);
      const Form f = form_of(rest.m, a.c);
      v = 0.f;
      for (int k = 0; k < mine; ++k) {
        float2 x[EI / 2];
        unpack(piece(k), x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i)
          v += tc::fast_exp2(fmaf(x[i].x, f.c, -f.b)) + tc::fast_exp2(fmaf(x[i].y, f.c, -f.b));
      }
      exchange(warp_sum(v), s_again + kMaxCluster * NW);
      v = 0.f;
      for (int i = lane; i < C * NW; i += 32) v += s_again[kMaxCluster * NW + i];
      rest.s = warp_sum(v);
    }
    if (OP == kDistill) {
      MaxSum one = {-INFINITY, 0.f};
      count = 0.f;
      if (lane < C) {
        one = {s_listed[lane].x, s_listed[lane].y};
        count = s_listed[lane].z;
      }
      listed.m = warp_max_redux(one.m);
      listed.s = warp_sum(one.s * rescale(one.m, listed.m, a.c));
      count = warp_sum(count);
    }
  }

  // ---- the row's scalars, by every thread: dz = c_out 2^(c z - b) +
  // corrections, in the form of the maximum outside the list
  Form f = form_of(rest.m, a.c), f_in = f;
  float c_in = 0.f, c_out = 0.f, hot = 0.f;
  if (OP == kLogp) {
    if (tid == 0 && rank == 0) {
      const double ls = log((double)rest.s), logp = above(za, rest.m, a.c, a.inv_tau) - ls;
      a.logp[row] = (float)logp;
      if (a.logp_lo) a.logp_lo[row] = (float)(logp - (double)(float)logp);
      a.lse[row] = (float)(ls - above(0.f, rest.m, a.c, a.inv_tau));
    }
    return;
  } else if (OP == kLogpBwd) {
    // 2^(c z - log2(e) lse): the whole part stays in the exponent.  An lse
    // beyond 1e25 says nothing of p: 0
    const double l2 = (double)lse_in * kLog2e;
    hot = (float)((double)dlogp * a.inv_tau);
    if (fabsf(lse_in) > 1e25f) {
      f = {0.f, 1e4f};
      c_out = -hot;
    } else {
      f = {a.c, (float)rint(l2)};
      c_out = -hot * tc::fast_exp2((float)((double)f.b - l2));
    }
  } else if (OP == kPolicy) {
    // differences of log-probabilities in double, powers of them in fp32
    const double logp = above(za, rest.m, a.c, a.inv_tau) - ln(rest.s);
    const float ratio = expf((float)(logp - (double)old_logp));
    const float lo = (float)(1.0 - a.clip_low), hi = (float)(1.0 + a.clip_high);
    const bool clipped = (adv > 0.f && ratio > hi) || (adv < 0.f && ratio < lo);
    float l = clipped ? -(adv > 0.f ? hi : lo) * adv : -ratio * adv;
    float d = clipped ? 0.f : -adv * ratio;
    if (a.ref_logp) {
      const float gap = (float)((double)ref_logp - logp), e = expm1f(gap);
      l += (float)a.kl_coef * (e - gap);
      d -= (float)a.kl_coef * e;
    }
    if (tid == 0 && rank == 0) {
      a.row_loss[row] = w * l;
      a.logp[row] = (float)logp;
    }
    hot = (float)(a.scale * a.inv_tau) * (w * d);
    c_out = -hot / rest.s;
  } else {
    const MaxSum all = join(rest, listed, a.c);
    f_in = form_of(all.m, a.c);
    // without an entry outside the list there is no class for the rest
    const float q_sum = (float)s_q[0], q_rest = count == (float)V ? 0.f : (float)s_q[2];
    hot = (float)(a.scale / a.inv_tau) * w;
    c_in = hot * (q_sum + q_rest) / all.s;
    // outside the list relative to the largest logit there: the student's
    // mass outside may be too small to be held relative to the row's largest
    // (none at all: an infinite loss, and entries of probability 0)
    c_out = rest.s == 0.f ? (all.s == 0.f ? NAN : 0.f)
                          : c_in * rescale(rest.m, all.m, a.c) -
                                (q_rest > 0.f ? hot * q_rest / rest.s : 0.f);
    if (!owner && rank == 0 && lane == 0) {
      const double qs = s_q[0], ls_all = ln(all.s), ls_rest = ln(rest.s);
      double qz = 0.0;
      for (int i = 0; i < C; ++i) qz += s_qz[i];
      // sum of q (z / tau - lse), as above() has it of one z
      const double x = is_far(all.m) ? (qz - qs * (double)all.m) * a.inv_tau
                                     : (qz * (double)a.c - qs * (double)f_in.b) * kLn2;
      double l = s_q[1] - (x - qs * ls_all);
      if (q_rest > 0.f)  // -log of the student's share outside the list
        l += (double)q_rest * ((double)logf(q_rest) + (ls_all - above(0.f, all.m, a.c, a.inv_tau)) -
                               (ls_rest - above(0.f, rest.m, a.c, a.inv_tau)));
      a.row_loss[row] = (float)((double)w * l / (a.inv_tau * a.inv_tau));
    }
  }
  if (!dz) return;

  // ---- the adjoint
  if (OP == kLogpBwd) copy_wait(0);
  const float2 c2 = make_float2(f.c, f.c), nb = make_float2(-f.b, -f.b);
  const float2 g2 = make_float2(c_out, c_out);
  auto values = [&](const float2 (&x)[EI / 2], float (&v)[EI], int e) {  // v[0] is element e's
#pragma unroll
    for (int i = 0; i < EI / 2; ++i) {
      const float2 t = tc::ffma2(x[i], c2, nb);
      const float2 d = tc::fmul2(make_float2(tc::fast_exp2(t.x), tc::fast_exp2(t.y)), g2);
      v[2 * i] = d.x;
      v[2 * i + 1] = d.y;
    }
    const unsigned to = (unsigned)(token - e);
    if (OP != kDistill && to < (unsigned)EI) {
#pragma unroll
      for (int i = 0; i < EI; ++i)
        if (to == (unsigned)i) v[i] += hot;
    }
  };
  if ((uintptr_t)(dz + e_org) % (EI * sizeof(TO)) == 0) {
    // the pieces' places in dz are aligned: every thread its own pieces
    const int k0 = tid < f0 ? 1 : 0, k1 = owner && tid < f1 ? (f1 - tid + NT - 1) / NT : 0;
#pragma unroll 2
    for (int k = k0; k < k1; ++k) {
      const int e = e_org + (tid + k * NT) * EI;
      float2 x[EI / 2];
      float v[EI];
      unpack(at[k * NT], x, (const TI*)nullptr);
      values(x, v, e);
      store_n(dz + e, v);
    }
    // the pieces in part outside the row
    auto in_part = [&](int i) {
      const int e = e_org + i * EI;
      float2 x[EI / 2];
      float v[EI];
      unpack(((const uint4*)dyn)[i], x, (const TI*)nullptr);
      values(x, v, e);
#pragma unroll
      for (int j = 0; j < EI; ++j)
        if (e + j >= 0 && e + j < V) st(&dz[e + j], v[j]);
    };
    if (f0 == 1 && tid == 0 && np > 0) in_part(0);
    if (f1 < np && f1 >= f0 && tid == f1 % NT) in_part(f1);
  } else {
    // units of dz straddle pieces: read across them
    __syncthreads();
    const int dph = (int)((uintptr_t)dz % (EI * sizeof(TO))) / (int)sizeof(TO);
    const int u0 = (dph + e_lo + EI - 1) / EI, u1 = (dph + e_hi) / EI;
#pragma unroll 2
    for (int u = u0 + tid; u < u1; u += kThreadsOf<OP>) {
      const int e = u * EI - dph;
      const TI* in = image + (e - e_org);
      float2 x[EI / 2];
      float v[EI];
#pragma unroll
      for (int i = 0; i < EI / 2; ++i) x[i] = make_float2(ld(&in[2 * i]), ld(&in[2 * i + 1]));
      values(x, v, e);
      store_n(dz + e, v);
    }
    const int ahead = u0 < u1 ? u0 * EI - dph : e_hi, behind = u0 < u1 ? u1 * EI - dph : e_hi;
    auto one = [&](int e) {
      const float d = c_out * tc::fast_exp2(fmaf(ld(&image[e - e_org]), f.c, -f.b));
      st(&dz[e], OP != kDistill && e == token ? d + hot : d);
    };
    if (e_lo + tid < ahead) one(e_lo + tid);
    if (behind + tid < e_hi) one(behind + tid);
  }
  if (OP == kDistill) {
    __syncthreads();
    for (int k = tid; k < a.K; k += kThreadsOf<OP>)
      if (!(t_g[k] < 0.f))
        st(&dz[t_idx[k]], c_in * tc::fast_exp2(fmaf(t_z[k], f_in.c, -f_in.b)) - hot * t_g[k]);
  }
}

// loss = scale * sum of l[0 .. n), in a fixed order, by NT threads.
template <int NT>
__device__ __forceinline__ void scaled_sum_of(const float* l, int64_t n, double scale, float* loss) {
  __shared__ double red[NT / 32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += NT) s += (double)l[i];
  s = warp_sum_d(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < NT / 32; ++w) t += red[w];
    *loss = (float)(scale * t);
  }
}
__global__ void __launch_bounds__(1024) k_scaled_sum(const float* l, int64_t n, double scale, float* loss) {
  scaled_sum_of<1024>(l, n, scale, loss);
}

template <RowOp OP, typename TI, typename TO>
__global__ void __launch_bounds__(kThreadsOf<OP>, kCtasPerSM<OP>) k_vocab_row(const RowArgs a) {
  if (OP == kLogpBwd) {
    // it has nothing to exchange: plain CTAs.  Last rows first: they are the
    // ones that the log-probabilities' pass has left in L2
    const unsigned C = (unsigned)a.cluster, r = blockIdx.x / C;
    if (r == a.rows) return scaled_sum_of<kRowThreads>(a.sum_of, a.sum_n, a.scale, a.loss);
    vocab_row<OP, TI, TO>(a, a.rows - 1 - r, (int)(blockIdx.x % C));
  } else {
    uint32_t row;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(row));
    vocab_row<OP, TI, TO>(a, row, (int)tc::cluster_ctarank());
  }
}

// ---- the preference loss
// A row's adjoint needs the margin of its pair, so the rows are read twice:
// for their log-probabilities, then, after the margins, for the adjoint, last
// rows first (what the first reading left in L2).
//
// A pair, by one CTA: rows [off[2p], off[2p+1]) chosen, [off[2p+1],
// off[2p+2]) rejected; the margin, the pair's loss, and each row's dlogp.
// dlogp comes in holding what the rounding of logp to fp32 left out: a margin
// is a small difference of sums of log-probabilities, and would show it.
constexpr int kPairsPerLaunch = 64;
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
  const int pair = blockIdx.x;
  const int64_t* off = a.off + 2 * pair;
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
    a.pair_loss[pair] = (float)l;
    a.margin[pair] = (float)m;
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
// Shared memory of a list of K entries and its filter.
constexpr int64_t list_bytes(int K) { return 16 * list_stride(K) + kFilterBits / 8; }
constexpr int64_t kDynamicMost = kStageBytesMost + list_bytes(kMaxTeacherK);
static_assert(kDynamicMost + 1536 <= 232448, "more shared memory than a CTA may have");
// Let a kernel use the shared memory it may need, once per device.
void allow_shared_memory(const void* kern) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = 0;
  DOP_CHECK_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (!done.count({dev, kern})) {
    DOP_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)kDynamicMost));
    done.insert({dev, kern});
  }
}

// How the rows are laid out over CTAs: as few of them per row as hold its
// 16-byte pieces when three CTAs share an SM, more of them where the rows are
// too few to occupy the SMs (down to 16 KB each), and at most kMaxCluster.
// `once`: the pieces pass through a ring and need not fit.
struct Split {
  int cluster, share;  // CTAs per row; pieces per CTA
};
Split split_of(int64_t rows, int64_t vocab, int prec, int64_t lists, bool once) {
  // the pieces that a row touches wherever it starts
  const int64_t size = prec == DOP_BF16 ? 2 : 4, pieces = ceil_div(vocab * size + 16 - size, 16);
  const int64_t fit = once ? 1 : ceil_div(16 * pieces, kCtaBytes - lists);
  const int64_t fill = std::min(ceil_div(3 * sm_count(), std::max<int64_t>(rows, 1)), ceil_div(pieces, 1024));
  const int64_t C = std::min<int64_t>(std::max(fit, fill), kMaxCluster);
  const int64_t share = ceil_div(pieces, C);
  if (!once && 16 * share > kStageBytesMost)
    throw Error(DOP_E_UNSUPPORTED, "vocab (" + std::to_string(vocab) + ") is above " +
                                       std::to_string((C * kStageBytesMost - 16) / size + 1));
  if (rows * C >= INT32_MAX) throw Error(DOP_E_UNSUPPORTED, "too many rows for this vocab");
  return {(int)C, (int)share};
}

// f(kernel's logit type, dlogits type)
template <typename F>
void by_types(int prec, int grad_prec, bool grad, F&& f) {
  if (prec == DOP_BF16) f(bf16{}, bf16{});
  else if (grad && grad_prec == DOP_BF16) f(0.f, bf16{});
  else f(0.f, 0.f);
}
template <typename A>
void launch(void (*kern)(A), const A& a, int64_t ctas, int threads, int64_t smem, int cluster,
            cudaStream_t s) {
  allow_shared_memory((const void*)kern);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  DOP_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
}

template <RowOp OP>
void launch_rows(RowArgs a, int64_t rows, int prec, int grad_prec, cudaStream_t s) {
  if (rows == 0) return;
  const int64_t lists = OP == kDistill ? list_bytes(a.K) : 0;
  const Split sp = split_of(rows, a.V, prec, lists, OP == kLogp);
  a.cluster = sp.cluster;
  a.share = sp.share;
  a.stage_bytes = 16 * (OP == kLogp ? std::min(sp.share, kRing * kOwnersOf<OP>) : sp.share);
  a.rows = rows;
  const int64_t ctas = rows * a.cluster + (a.sum_of ? 1 : 0);
  by_types(prec, grad_prec, a.dz != nullptr, [&](auto ti, auto to) {
    launch(k_vocab_row<OP, decltype(ti), decltype(to)>, a, ctas, kThreadsOf<OP>,
           a.stage_bytes + lists, OP == kLogpBwd ? 1 : a.cluster, s);
  });
}

int elem_bytes(int prec) { return prec == DOP_BF16 ? 2 : 4; }

// The checks every objective shares.
void check_rows(int64_t rows, int64_t vocab, int prec, const void* z, int64_t ld, double tau) {
  DOP_REQUIRE(rows >= 0 && rows <= INT32_MAX, "rows must lie in [0, 2^31)");
  DOP_REQUIRE(vocab >= 1 && vocab <= INT32_MAX, "vocab must lie in [1, 2^31)");
  DOP_REQUIRE(prec == DOP_F32 || prec == DOP_BF16, "unknown precision");
  split_of(rows, vocab, prec, 0, false);
  DOP_REQUIRE(ld >= vocab, "the logits' row stride is smaller than vocab");
  DOP_REQUIRE(z || rows == 0, "null logits");
  DOP_REQUIRE((uintptr_t)z % elem_bytes(prec) == 0, "misaligned logits");
  DOP_REQUIRE(tau >= 0x1p-16 && tau <= 0x1p16, "temperature must lie in [2^-16, 2^16]");
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
  a.in_lo = 0;
  a.in_hi = INT64_MAX;
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
    RowArgs f = row_args(vocab, logits, ld, tokens, weight, temperature);
    f.in_lo = seq_off[0];
    f.in_hi = seq_off[2 * pairs];
    f.logp = logp;
    f.logp_lo = dlogp;
    f.lse = lse;
    launch_rows<kLogp>(f, rows, precision, DOP_F32, s);
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
    if (!dlogits || rows == 0) return scaled_sum(pair_loss, pairs, scale, loss, s);
    RowArgs b = row_args(vocab, logits, ld, tokens, nullptr, temperature);
    b.lse = lse;
    b.dlogp = dlogp;
    b.dz = dlogits;
    b.ldd = ldd;
    b.sum_of = pair_loss;
    b.sum_n = pairs;
    b.scale = scale;
    b.loss = loss;
    launch_rows<kLogpBwd>(b, rows, precision, grad_precision, s);
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
