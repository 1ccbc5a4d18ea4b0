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

#include "../../include/dop.h"
#include "kernels.cuh"
#include "tc_ptx.cuh"

namespace dop {
int set_last_error(int code, const char* msg);

namespace {

enum RowOp : int { kLogp = 0, kLogpBwd = 1, kPolicy = 2, kDistill = 3 };

constexpr int kRowThreads = 256;
constexpr int kMaxTeacherK = 1024;
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

// One CTA per row.
template <RowOp OP, typename TI, typename TO>
__global__ void __launch_bounds__(kRowThreads) k_vocab_row(const RowArgs a) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ MaxSum s_ms[kRowThreads / 32];
  __shared__ double s_red[kRowThreads / 32];
  __shared__ float s_coef[2];
  const int64_t row = blockIdx.x;
  const TI* z = (const TI*)a.z + row * a.ld;
  TO* dz = a.dz ? (TO*)a.dz + row * a.ldd : nullptr;
  const int64_t V = a.V;
  const float w = a.weight ? a.weight[row] : 1.f;
  const int64_t token = OP == kDistill ? 0 : a.tokens[row];
  bool skip = w == 0.f || token < 0 || token >= V;
  if (OP == kLogpBwd && a.dlogp[row] == 0.f) skip = true;
  if (skip) {
    if (dz)
      for (int64_t v = threadIdx.x; v < V; v += kRowThreads) st(&dz[v], 0.f);
    if (threadIdx.x == 0) {
      if (OP != kLogpBwd && OP != kDistill && a.logp) a.logp[row] = 0.f;
      if (OP == kLogp && a.lse) a.lse[row] = 0.f;
      if (OP == kLogp && a.logp_lo) a.logp_lo[row] = 0.f;
      if (OP == kPolicy || OP == kDistill) a.row_loss[row] = 0.f;
    }
    return;
  }
  const float za = OP == kDistill ? 0.f : ld(&z[token]);

  // ---- the teacher's entries: q, the student's logit, and which are a
  // vocabulary entry's first
  int32_t* t_idx = (int32_t*)dyn;
  float* t_q = (float*)(t_idx + a.K);
  float* t_z = t_q + a.K;
  uint32_t* bits = (uint32_t*)(t_z + a.K);
  double q_sum = 0.0, q_logq = 0.0, q_rest = 0.0;
  if (OP == kDistill) {
    for (int64_t i = threadIdx.x; i < (V + 31) / 32; i += kRowThreads) bits[i] = 0;
    const float* y = a.top_logit + row * a.K;
    MaxSum t = {-INFINITY, 0.f};
    for (int k = threadIdx.x; k < a.K; k += kRowThreads) {
      const int32_t i = a.top_index[row * a.K + k];
      const bool in = i >= 0 && i < V;
      t_idx[k] = in ? i : -1;
      t_z[k] = in ? ld(&z[i]) : 0.f;
      t_q[k] = in ? y[k] : -INFINITY;
      if (in) t = join(t, {y[k], 1.f}, a.c);
    }
    t = warp_join(t, a.c);
    if ((threadIdx.x & 31) == 0) s_ms[threadIdx.x >> 5] = t;
    __syncthreads();
    t = s_ms[0];
    for (int i = 1; i < kRowThreads / 32; ++i) t = join(t, s_ms[i], a.c);
    const double tl = a.teacher_lse ? (double)a.teacher_lse[row]
                                    : (double)base_of(t.m) * a.inv_tau + log((double)t.s);
    double qs = 0.0, ql = 0.0;
    for (int k = threadIdx.x; k < a.K; k += kRowThreads) {
      const double lq = (double)t_q[k] * a.inv_tau - tl;
      const double q = t_idx[k] < 0 || t_q[k] == -INFINITY ? 0.0 : exp(lq);
      t_q[k] = (float)q;
      qs += q;
      if (q > 0.0) ql += q * lq;
      if (t_idx[k] >= 0) atomicOr(&bits[t_idx[k] >> 5], 1u << (t_idx[k] & 31));
    }
    q_sum = block_sum_d(qs, s_red);
    q_logq = block_sum_d(ql, s_red);
    q_rest = a.teacher_lse ? fmax(0.0, 1.0 - q_sum) : 0.0;
  }

  // ---- maximum and sum
  MaxSum r = {-INFINITY, 0.f};
  if (OP != kLogpBwd) {
    for (int64_t v = threadIdx.x; v < V; v += kRowThreads) {
      const float x = ld(&z[v]);
      if (OP == kDistill && (bits[v >> 5] >> (v & 31) & 1u)) continue;
      if (x > r.m) {
        r.s *= tc::fast_exp2((r.m - x) * a.c);
        r.m = x;
      }
      r.s += tc::fast_exp2((x - base_of(r.m)) * a.c);
    }
    r = warp_join(r, a.c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_ms[threadIdx.x >> 5] = r;
    __syncthreads();
    r = s_ms[0];
    for (int i = 1; i < kRowThreads / 32; ++i) r = join(r, s_ms[i], a.c);
  }

  // ---- the row's scalars: dz = c_out 2^((f z - b) c) + corrections
  float c_in = 0.f, b_in = 0.f, c_out = 0.f, hot = 0.f, b = 0.f, f = 1.f, c = a.c;
  if (OP == kLogpBwd) {
    hot = (float)((double)a.dlogp[row] * a.inv_tau);
    c_out = -hot;
    f = (float)a.inv_tau;
    b = a.lse[row];
    c = (float)kLog2e;
  } else if (OP != kDistill) {
    if (threadIdx.x == 0) {
      const double ls = log((double)r.s);
      const double logp = ((double)za - (double)base_of(r.m)) * a.inv_tau - ls;
      if (a.logp) a.logp[row] = (float)logp;
      if (OP == kLogp && a.logp_lo) a.logp_lo[row] = (float)(logp - (double)(float)logp);
      if (OP == kLogp && a.lse) a.lse[row] = (float)((double)base_of(r.m) * a.inv_tau + ls);
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
        a.row_loss[row] = (float)((double)w * l);
        const double g = a.scale * (double)w * d * a.inv_tau;
        s_coef[0] = (float)g;
        s_coef[1] = (float)(-g / (double)r.s);
      }
    }
    __syncthreads();
    hot = s_coef[0];
    c_out = s_coef[1];
  } else {
    // the listed entries join the sum: each vocabulary entry once
    MaxSum in = {-INFINITY, 0.f};
    double listed = 0.0;
    for (int k = threadIdx.x; k < a.K; k += kRowThreads) {
      bool first = t_idx[k] >= 0;
      for (int j = 0; j < k && first; ++j) first = t_idx[j] != t_idx[k];
      if (first) in = join(in, {t_z[k], t_z[k] == -INFINITY ? 0.f : 1.f}, a.c);
      if (first) listed += 1.0;
    }
    // without an entry outside the list there is no class for the rest
    if (block_sum_d(listed, s_red) == (double)V) q_rest = 0.0;
    in = warp_join(in, a.c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_ms[threadIdx.x >> 5] = in;
    __syncthreads();
    in = s_ms[0];
    for (int i = 1; i < kRowThreads / 32; ++i) in = join(in, s_ms[i], a.c);
    const MaxSum all = join(r, in, a.c);
    const double ls = log((double)all.s), mx = (double)base_of(all.m) * a.inv_tau;
    double cross = 0.0;
    for (int k = threadIdx.x; k < a.K; k += kRowThreads)
      if (t_q[k] != 0.f) cross += (double)t_q[k] * ((double)t_z[k] * a.inv_tau - mx - ls);
    cross = block_sum_d(cross, s_red);
    if (threadIdx.x == 0) {
      double l = q_logq - cross;
      if (q_rest > 0.0)
        l += q_rest * (log(q_rest) -
                       ((double)base_of(r.m) * a.inv_tau + log((double)r.s) - mx - ls));
      a.row_loss[row] = (float)((double)w * l / (a.inv_tau * a.inv_tau));
    }
    const double g = a.scale * (double)w / a.inv_tau;
    const double Q = q_sum + q_rest;
    c_in = (float)(g * Q / (double)all.s);
    b_in = base_of(all.m);
    // outside the list relative to the largest logit there: the student's
    // mass outside may be too small to be held relative to the row's largest
    // (none at all: an infinite loss, and entries of probability 0)
    c_out = r.s == 0.f ? 0.f
                       : (float)(g * (Q * (double)tc::fast_exp2((base_of(r.m) - b_in) * a.c) /
                                          (double)all.s -
                                      (q_rest > 0.0 ? q_rest / (double)r.s : 0.0)));
    hot = (float)g;
  }

  // ---- the adjoint
  if (!dz) return;
  if (OP != kLogpBwd) b = base_of(r.m);
  for (int64_t v = threadIdx.x; v < V; v += kRowThreads) {
    const float x = ld(&z[v]);
    float d = c_out * tc::fast_exp2(fmaf(x, f, -b) * c);
    if (OP == kDistill) {
      if (bits[v >> 5] >> (v & 31) & 1u) {
        double q = 0.0;
        for (int k = 0; k < a.K; ++k)
          if (t_idx[k] == v) q += t_q[k];
        d = c_in * tc::fast_exp2((x - b_in) * c) - hot * (float)q;
      }
    } else if (v == token) {
      d += hot;
    }
    st(&dz[v], d);
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
void launch_rows(const RowArgs& a, int64_t rows, int prec, int grad_prec, cudaStream_t s) {
  if (rows == 0) return;
  DOP_REQUIRE(rows <= INT32_MAX, "rows");
  const size_t smem = OP == kDistill ? 12 * (size_t)a.K + 4 * ((a.V + 31) / 32) : 0;
  auto go = [&](auto ti, auto to) {
    auto kern = k_vocab_row<OP, decltype(ti), decltype(to)>;
    if (smem > 48 * 1024)
      DOP_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kern<<<(unsigned)rows, kRowThreads, smem, s>>>(a);
    DOP_CHECK_CUDA(cudaGetLastError());
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
