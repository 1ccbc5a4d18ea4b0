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
// so one kernel serves them: a row is read once into the SM, where its sum of
// powers is taken (fp32, relative to a whole exponent, so that rescaling is
// exact), the row's scalars follow (in double but for a list's q and its
// coefficients), and the adjoint is written from what the SM kept.  What bounds it
// is the row's one read and one write; with both sides bf16 the exponentials,
// two an element at 16 a cycle and SM, come close to that.  Measured on one
// B200 (6.46 TB/s of measured copy bandwidth), of the bytes read and written
// once:
//
//   log-probabilities, 16384 x 32000 bf16, a fifth skipped          146 us  0.89
//   their adjoint, 4095 x 50001 fp32 to bf16                        207 us  0.92
//   policy loss, 8192 x 32000 fp32 to bf16, a quarter skipped       218 us  0.93
//   policy loss, 3001 x 100003 bf16 (rows on odd addresses)         255 us  0.73
//   preference loss, 16384 x 32000 bf16, three tenths skipped       410 us  0.67
//     (the margins come between two readings of the logits: 0.95 of three passes)
//   distillation from 64 logits, 32768 x 32000 bf16                 833 us  0.78
//   with a class for the rest, 128 logits, 2047 x 128000 fp32       412 us  0.79
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

// (kDistillRest: distillation with a class for the entries outside the list)
enum RowOp : int { kLogp = 0, kLogpBwd = 1, kPolicy = 2, kDistill = 3, kDistillRest = 4 };
constexpr bool has_list(RowOp op) { return op == kDistill || op == kDistillRest; }

constexpr int kMaxTeacherK = 1024;
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
constexpr int kMaxCluster = 8;
// CTAs by the pieces that they keep.  Narrow: 128 threads with up to 16 pieces
// each in shared memory (32 KB of a row), six CTAs an SM; pieces that are read
// once pass through 8 or 16 places.  Held: 256 threads, up to 18 pieces (72
// KB), three CTAs an SM.  Wide: 16 pieces more per thread in tensor memory,
// 128 KB, three CTAs an SM.  Alone: at most 40 and 64 pieces (416 KB), one CTA
// an SM.
//
// A CTA that holds tensor memory waits for the others of its cluster, so the
// CTAs that may share an SM must never ask for more than its 512 columns: 64
// KB of shared memory go with every 128 columns (three at most), and one that
// takes them all takes the shared memory that another would need.
enum Shape : int { kNarrow, kHeld, kWide, kAlone };
constexpr int owners_of(Shape s) { return s == kNarrow ? 128 : 256; }
// Columns of tensor memory.  A constant in the instruction, and kernels
// without it for the shapes that take none: CTAs of a kernel that names
// tensor memory start about half a microsecond apart on an SM.
constexpr int columns_of(Shape s) { return s == kWide ? 128 : s == kAlone ? 512 : 0; }
constexpr int kKept = 16, kHeldMost = 18, kPassing = 8, kRingMost = 40, kMovedMost = 64;
constexpr int64_t kAloneBytes = 200 * 1024;
constexpr int kPairThreads = 256;
// A warp's 512 bytes of 16-byte pieces lie on the lines of shared memory: with
// the ring 32 bytes off, behind the static variables, the policy loss of 8192 x
// 32000 fp32 takes 236 us instead of 214, the log-probability adjoint of 4095 x
// 50001 209 instead of 206; 80 bytes off, 212.
constexpr int kRingAlign = 128;

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
  // the preference loss, taken with the adjoint: loss (null: none) = scale
  // times the sum of sum_of[0 .. sum_n)
  const float* sum_of;
  int64_t sum_n;
  float* loss;
  int cluster;      // CTAs per row
  int share;         // 16-byte pieces of a row a CTA has
  int ring;          // places for pieces per thread in shared memory
  int stage_bytes;   // all of them
  int bit_words;     // of the list's bits
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
// a relative change of the temperature by at most 2^-24.)
//
// From |c m| = 2^24 on fp32 has no whole number near c m (b would miss it by
// up to half of its last digit, and the power at m itself would leave fp32);
// such a maximum is far.  The powers are then 2^(c (z - m)), from elements
// that m has been subtracted from: fp32 holds z - m to 2^-24 of it; in bf16
// two elements that differ do so by 2^15 / c at least, which leaves the
// smaller one nothing, and equal ones give 0.
constexpr float kFar = 0x1p24f;
constexpr float kBaseMost = 1e30f;  // (of a maximum of -inf)
__device__ __forceinline__ float base_of(float m, float c) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: to a whole number without a conversion
  return fminf(fmaxf((c * m + kRound) - kRound, -kBaseMost), kBaseMost);
}
__device__ __forceinline__ bool is_far(float m, float c) {  // (+inf and NaN are)
  return !(fabsf(c * m) < kFar) && m != -INFINITY;
}
struct Form {
  float c, b, m;  // 2^(c (z - m) - b)
};
__device__ __forceinline__ Form form_of(float m, float c) {
  if (is_far(m, c)) return {c, 0.f, m};
  return {c, base_of(m, c), 0.f};
}
__device__ __forceinline__ float power(float z, const Form& f) {
  return tc::fast_exp2(fmaf(z - f.m, f.c, -f.b));
}
// A maximum and a sum of powers; nothing: {-inf, 0}.  While the sums are put
// together they are relative to base_of(m) (of a far row: no sum yet); the
// row's, and those of listed entries, are of form_of(m).
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float warp_max_redux(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// What turns a sum relative to base_of(m) into one relative to that of `to` >= m.
__device__ __forceinline__ float rebase(float m, float to, float c) {
  return m == to ? 1.f : tc::fast_exp2(base_of(m, c) - base_of(to, c));
}
// The warp's maximum and sum, relative to its base.
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
  const float m = warp_max_redux(v.m);
  return {m, warp_sum(v.s * tc::fast_exp2(base_of(v.m, c) - base_of(m, c)))};
}
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * rebase(a.m, m, c) + b.s * rebase(b.m, m, c)};
}
// c z where the powers of form_of(m) are 1 (exact: 48 bits).
__device__ __forceinline__ double origin(float m, float c) {
  return is_far(m, c) ? (double)c * (double)m : (double)base_of(m, c);
}
// What turns a sum of form_of(m) into one of form_of(to), to >= m.
__device__ __forceinline__ float rescale(float m, float to, float c) {
  if (m == to) return 1.f;
  if (m == -INFINITY) return 0.f;
  if (!is_far(m, c) && !is_far(to, c)) return tc::fast_exp2(base_of(m, c) - base_of(to, c));
  return tc::fast_exp2((float)(origin(m, c) - origin(to, c)));
}
// (z - m) / tau, to which log(s) is to be taken from, in double.
__device__ __forceinline__ double above(float z, float m, float c, double inv_tau) {
  if (is_far(m, c)) return ((double)z - (double)m) * inv_tau;
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
  for (int w = 0; w < kPairThreads / 32; ++w) t += red[w];
  return t;
}

// ---- a row on the SM
// A row is cut into 16-byte pieces at 16-byte borders of its address, so a
// row may start and end inside a piece; the cluster's CTAs hold consecutive
// runs of pieces, one CTA the whole row when it fits.  Thread t owns pieces t,
// t + NT, ... of its CTA: it copies them, reads them for the maximum and sum
// and again for the adjoint, so that neither needs a barrier.  They come
// through a ring in shared memory, in groups of U pieces a thread; a group
// whose place in the ring is wanted for a later one moves to the thread's own
// lane of tensor memory, whose 256 KB double what an SM can hold of the rows
// under way.  What is kept is the bf16 logits, or of fp32 logits the powers
// of two themselves.  What a piece holds beyond the row is -inf.
__device__ __forceinline__ void copy_piece(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N of this thread's copy groups are under way.
template <int N>
__device__ __forceinline__ void copy_wait_for() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
// A piece less m (out of line: of far rows alone).
__device__ __noinline__ uint4 minus(uint4 u, float m, const float*) {
  return make_uint4(__float_as_uint(__uint_as_float(u.x) - m), __float_as_uint(__uint_as_float(u.y) - m),
                    __float_as_uint(__uint_as_float(u.z) - m), __float_as_uint(__uint_as_float(u.w) - m));
}
__device__ __noinline__ uint4 minus(uint4 u, float m, const bf16*) {
  auto word = [m](uint32_t w) {
    const float2 x = bf16x2(w);
    return tc::pack_bf16(x.x - m, x.y - m);
  };
  return make_uint4(word(u.x), word(u.y), word(u.z), word(u.w));
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

// The same where the address is only a multiple of the element: `off` is its
// remainder by the size of the N elements.
__device__ __forceinline__ void store_off(float* p, const float (&v)[4], int off) {
  if (off == 8) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    *reinterpret_cast<float2*>(p + 2) = make_float2(v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void store_off(bf16* p, const float (&v)[N], int off) {
  if (off % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      *reinterpret_cast<uint32_t*>(p + i) = tc::pack_bf16(v[i], v[i + 1]);
  } else {
    st(p, v[0]);
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2)
      *reinterpret_cast<uint32_t*>(p + i) = tc::pack_bf16(v[i], v[i + 1]);
    st(p + N - 1, v[N - 1]);
  }
}

// A list's arrays start at 16-byte borders.
__host__ __device__ constexpr int list_stride(int K) { return (K + 3) & ~3; }
// Bits of the filter that finds out whether a list may name an entry twice
// (where it need not say which entries are listed).
constexpr int kFilterBits = 8192;

// ln(s), to about 2^-24 of it or of 1: the exponent apart (0, subnormal, inf
// and NaN as log has them).
__device__ __forceinline__ double ln(float s) {
  if (!(s > 0x1p-126f && s < INFINITY)) return (double)logf(s);
  const int e = (__float_as_int(s) - 0x3f400000) >> 23;  // s = 2^e f, f in [0.75, 1.5)
  return (double)e * kLn2 + (double)logf(__int_as_float(__float_as_int(s) - (e << 23)));
}

// Pieces that are in part outside the row, and element by element: out of
// line, since the CTAs of an SM share its instruction cache.
template <typename T>
__device__ __noinline__ uint4 part_of_row(const T* z, int e, int V) {  // piece at element e
  constexpr int N = 16 / (int)sizeof(T);
  T v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = e + i >= 0 && e + i < V ? z[e + i] : (T)-INFINITY;
  uint4 u;
  memcpy(&u, v, 16);
  return u;
}
template <typename T>
__device__ __noinline__ void store_elements(T* dz, int e, int V, int n, float4 a, float4 b) {
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n && e + i >= 0 && e + i < V) st(&dz[e + i], v[i]);
}

template <int N>
__device__ __forceinline__ void alloc_columns(uint32_t slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "n"(N));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
// Two pieces to eight columns of the thread's lane, and back.
__device__ __forceinline__ void tmem_put(uint32_t at, const uint4 (&u)[2]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at),
               "r"(u[0].x), "r"(u[0].y), "r"(u[0].z), "r"(u[0].w), "r"(u[1].x), "r"(u[1].y),
               "r"(u[1].z), "r"(u[1].w)
               : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t at, uint4 (&u)[2]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0].x), "=r"(u[0].y), "=r"(u[0].z), "=r"(u[0].w), "=r"(u[1].x), "=r"(u[1].y),
        "=r"(u[1].z), "=r"(u[1].w)
      : "r"(at)
      : "memory");
}
template <int N>
__device__ __forceinline__ void free_columns(uint32_t at) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(N));
}

// The log-probability adjoint of a row whose lse fp32 does not hold well (above
// kLseMost, infinite ones too: the rounding of lse to fp32 is an error of p,
// 2^-24 of lse): from the row's own maximum and sum, by one CTA for the whole
// row, which may be written in place.  Slow, and out of line: logits in the
// thousands are rare.
constexpr float kLseMost = 4096.f;
template <typename TI, typename TO, int NT>
__device__ __noinline__ void logp_adjoint_from_row(const TI* z, TO* dz, int V, int token, float c, float hot) {
  extern __shared__ __align__(kRingAlign) uint8_t dyn[];  // (the ring, which is not in use)
  float* s_m = (float*)dyn;
  double* s_s = (double*)(dyn + 128);
  const int tid = threadIdx.x;
  float m = -INFINITY;
  for (int v = tid; v < V; v += NT) m = fmaxf(m, ld(&z[v]));
  m = warp_max_redux(m);
  if ((tid & 31) == 0) s_m[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < NT / 32; ++w) m = fmaxf(m, s_m[w]);
  const Form f = form_of(m, c);
  double s = 0.0;
  for (int v = tid; v < V; v += NT) s += (double)power(ld(&z[v]), f);
  s = warp_sum_d(s);
  if ((tid & 31) == 0) s_s[tid >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < NT / 32; ++w) s += s_s[w];
  const float c_out = (float)(-(double)hot / s);
  for (int v = tid; v < V; v += NT) st(&dz[v], c_out * power(ld(&z[v]), f) + (v == token ? hot : 0.f));
}

// A row by a cluster of a.cluster CTAs, of which NT threads own the pieces;
// distillation has a warp more for the teacher's list.
template <RowOp OP, Shape S>
constexpr int kThreadsOf = owners_of(S) + (has_list(OP) ? 32 : 0);
template <RowOp OP, Shape S>
constexpr int kCtasPerSM = S == kAlone ? 1 : S != kNarrow ? 3 : OP == kLogp ? 8 : 6;

template <RowOp OP, typename TI, typename TO, Shape S>
__device__ __forceinline__ void vocab_row(const RowArgs& a, const int64_t row, const int rank) {
  constexpr int EI = 16 / (int)sizeof(TI);
  constexpr int NT = owners_of(S), NW = NT / 32, THREADS = kThreadsOf<OP, S>;
  constexpr bool kOnce = OP == kLogp || OP == kLogpBwd;  // the pieces are read once
  constexpr bool kList = has_list(OP), tail = OP == kDistillRest;
  constexpr bool kKeepPower = sizeof(TI) == 4 && !kOnce;
  constexpr bool kTmem = !kOnce && columns_of(S) > 0;
  constexpr bool kFits = !kOnce && !kTmem;  // every piece has a place of its own
  constexpr int U = kFits && OP != kDistillRest ? 4 : 2;  // (that one, 16384 x 16001 bf16: 291 us with 4, 274 with 2)
  extern __shared__ __align__(kRingAlign) uint8_t dyn[];
  // of every warp of the cluster
  __shared__ MaxSum s_rest[kMaxCluster * NW];
  __shared__ float s_again[2 * kMaxCluster * NW];
  // of every CTA: the listed entries' m, s, count; the sum of q times the logit
  __shared__ __align__(16) float4 s_listed[kMaxCluster];
  __shared__ double s_qz[kMaxCluster];
  __shared__ double s_q[3];
  __shared__ uint32_t s_tmem;
  // bit k >> kHasShift of an owner: whether its piece k has a listed element
  // (looked at for every group, the elements' bits where it is set; 16384 x
  // 16001 bf16: 283 us without it, 274 with; 2047 x 128000 fp32: 400, 409)
  constexpr int kHasShift = S == kAlone ? 2 : 0;
  static_assert(kMovedMost + kRingMost <= 32 << 2 && 2 * kKept <= 32 && kHeldMost <= 32);
  __shared__ uint32_t s_has[tail ? NT : 1];
  const int C = a.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool owner = !kList || tid < NT;  // of pieces
  const float w = a.weight ? a.weight[row] : 1.f;
  const int64_t token64 = kList ? -1 : a.tokens[row];
  const float dlogp = OP == kLogpBwd ? a.dlogp[row] : 0.f;
  const float lse_in = OP == kLogpBwd ? a.lse[row] : 0.f;
  const float adv = OP == kPolicy ? a.advantage[row] : 0.f;
  const float old_logp = OP == kPolicy ? a.old_logp[row] : 0.f;
  const float ref_logp = OP == kPolicy && a.ref_logp ? a.ref_logp[row] : 0.f;

  int32_t my_idx = -1;
  float my_top = 0.f;
  if (kList && owner && tid < a.K) {
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
  const int e_org = p0 * EI - ph;  // the row's element where its pieces start
  const int e_lo = max(0, e_org), e_hi = max(e_lo, min(V, e_org + np * EI));
  // pieces that lie in the row altogether: [f0, f1)
  const int f0 = e_org < 0 ? 1 : 0, f1 = e_org + np * EI > V ? np - 1 : np;

  if (w == 0.f || row < a.in_lo || row >= a.in_hi || (!kList && (token64 < 0 || token64 >= V)) ||
      (OP == kLogpBwd && dlogp == 0.f)) {
    if (dz) {
      constexpr int EO = 16 / (int)sizeof(TO);
      const int dph = (int)((uintptr_t)dz & 15) / (int)sizeof(TO);
      const int u0 = (dph + e_lo + EO - 1) / EO, u1 = (dph + e_hi) / EO;  // 16-byte units
      const int ahead = u0 < u1 ? u0 * EO - dph : e_hi, behind = u0 < u1 ? u1 * EO - dph : e_hi;
      for (int u = u0 + tid; u < u1; u += THREADS)
        *reinterpret_cast<uint4*>(dz + (u * EO - dph)) = make_uint4(0u, 0u, 0u, 0u);
      if (e_lo + tid < ahead) st(&dz[e_lo + tid], 0.f);
      if (behind + tid < e_hi) st(&dz[behind + tid], 0.f);
    }
    if (tid == 0 && rank == 0) {
      if (OP != kLogpBwd && !kList && a.logp) a.logp[row] = 0.f;
      if (OP == kLogp && a.lse) a.lse[row] = 0.f;
      if (OP == kLogp && a.logp_lo) a.logp_lo[row] = 0.f;
      if (OP == kPolicy || kList) a.row_loss[row] = 0.f;
    }
    return;
  }
  if (OP == kLogpBwd && fabsf(lse_in) > kLseMost) {
    if (rank == 0)
      logp_adjoint_from_row<TI, TO, NT>(z, dz, V, token, a.c, (float)((double)dlogp * a.inv_tau));
    return;
  }
  // every CTA of the cluster has started once this barrier is through: its
  // shared memory may be written to
  if (OP != kLogpBwd && C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ---- copy the first groups of pieces
  // groups of the CTA, places for them in the ring, and those that tensor
  // memory takes over (all the same for every thread)
  const int groups = (np + NT * U - 1) / (NT * U), ring = kFits ? groups : a.ring / U;
  const int moved = dz && kTmem ? max(0, groups - ring) : 0;
  const int mine = owner && tid < np ? (np - tid + NT - 1) / NT : 0;  // pieces of this thread
  uint4* at = (uint4*)dyn + tid;  // piece j of place r: at[(r U + j) NT]
  auto edge = [&](int i) { return part_of_row(z, e_org + i * EI, V); };
  const uint4* src = (const uint4*)(z + e_org) + tid;
  const uint32_t dst = tc::smem_u32(at);
  auto whole = [&](int k) { return tid + k * NT >= f0 && tid + k * NT < f1; };
  auto copy_group = [&](int g, int r) {  // group g to place r
    if (tid + g * U * NT >= f0 && tid + (g * U + U - 1) * NT < f1) {
#pragma unroll
      for (int j = 0; j < U; ++j) copy_piece(dst + (r * U + j) * (NT * 16), src + (g * U + j) * NT);
    } else {
      for (int j = 0; j < U; ++j)
        if (whole(g * U + j)) copy_piece(dst + (r * U + j) * (NT * 16), src + (g * U + j) * NT);
    }
    copy_commit();
  };
  // the pieces of a group that are in part outside the row: at most the
  // row's first and its last
  auto copy_edges = [&](int g, int r) {
#pragma unroll 1
    for (int j = 0; j < U; ++j)
      if (g * U + j < mine && !whole(g * U + j)) at[(r * U + j) * NT] = edge(tid + (g * U + j) * NT);
  };
  const int g_head = f0 == 1 ? 0 : -1, g_tail = f1 < np ? f1 / (NT * U) : -1;
  const int first = min(groups, ring);
  if (owner) {
    for (int g = 0; g < first; ++g) copy_group(g, g);
    if (g_head >= 0 && g_head < first && tid == 0) copy_edges(g_head, g_head);
    if (g_tail >= 0 && g_tail < first && tid == f1 % NT) copy_edges(g_tail, g_tail);
  }
  if constexpr (kTmem)
    if (warp == 0) {
      __syncwarp();
      alloc_columns<columns_of(S)>(tc::smem_u32(&s_tmem));
    }
  const float za = OP == kLogp || OP == kPolicy ? ld(&z[token]) : 0.f;

  // ---- the teacher's list, by the warp that owns no pieces
  const int K4 = kList ? list_stride(a.K) : 0;
  int32_t* t_idx = (int32_t*)(dyn + a.stage_bytes);
  float* t_q = (float*)t_idx + K4;  // the teacher's logit, then q
  float* t_z = t_q + K4;            // the student's logit, of this CTA's entries
  float* t_g = t_z + K4;            // this CTA's first ones: sum of q of the entry; else -1
  // with a class for the rest, one bit per element of this CTA: whether it is
  // listed; else a filter
  uint32_t* bits = (uint32_t*)(t_g + K4);
  if (kList) {
    // its owners bring the list while their copies run, and go on; the warp
    // without pieces takes it from there
    if (owner) {
#pragma unroll 1
      for (int k = tid; k < a.K; k += NT) {
        const int32_t i = k < NT ? my_idx : a.top_index[row * a.K + k];
        const float y = k < NT ? my_top : a.top_logit[row * a.K + k];
        const bool in = i >= 0 && i < V, here = i >= e_lo && i < e_hi;
        t_idx[k] = in ? i : -1;
        t_q[k] = in ? y : -INFINITY;
        t_z[k] = here ? ld(&z[i]) : 0.f;
        t_g[k] = here ? 0.f : -1.f;
      }
      asm volatile("bar.arrive 1, %0;" ::"n"(THREADS) : "memory");
    } else {
      asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    }
  }
  auto set_bits = [&] {
#pragma unroll 1
    for (int i = lane; i < a.bit_words; i += 32) bits[i] = 0u;
    if (tail)
#pragma unroll 1
      for (int i = lane; i < NT; i += 32) s_has[i] = 0u;
    __syncwarp();
    bool twice = false;
#pragma unroll 1
    for (int k = lane; k < a.K; k += 32)
      if (!(t_g[k] < 0.f)) {
        const int i = t_idx[k];
        const uint32_t h = tail ? (uint32_t)(i - e_org) : (uint32_t)i % kFilterBits, bit = 1u << (h & 31);
        if (atomicOr(&bits[h >> 5], bit) & bit) twice = true;
        if (tail) {
          const int piece = (i - e_org) / EI;
          atomicOr(&s_has[piece % NT], 1u << (piece / NT >> kHasShift));
        }
      }
    return (bool)__any_sync(0xffffffffu, twice);
  };
  // first ones of a list that may name an entry twice get the sum of q, the
  // others -1
  auto count_once = [&] {
#pragma unroll 1
    for (int k = lane; k < a.K; k += 32) {
      const int i = t_idx[k];
      if (t_g[k] < 0.f) continue;
      double sum = 0.0;
      bool before = false;
#pragma unroll 1
      for (int j = 0; j < a.K; ++j)
        if (t_idx[j] == i) {
          if (j < k) before = true;
          sum += (double)t_q[j];
        }
      t_g[k] = before ? -1.f : (float)sum;
    }
    __syncwarp();
  };
  bool twice = false;
  if (tail && !owner) twice = set_bits();
  if (tail || kTmem) {
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
  }
  const uint32_t has = tail && owner ? s_has[tid] : 0u;
  // this thread's lane of tensor memory; the second four warps have the
  // columns behind those of the first four
  const uint32_t lane_tmem = kTmem ? s_tmem + ((uint32_t)(warp & 3) << 21) +
                                         (warp >= 4 ? (uint32_t)columns_of(S) / 2 : 0u)
                                   : 0u;
  // q of the list, its sums, and which entries are a vocabulary entry's first
  auto make_q = [&] {
    MaxSum t = {-INFINITY, 0.f};
    double tl = 0.0;
    if (tail) {
      tl = (double)a.teacher_lse[row];
    } else {
#pragma unroll 1
      for (int k = lane; k < a.K; k += 32) t.m = fmaxf(t.m, t_q[k]);
      t.m = warp_max_redux(t.m);
      const Form f = form_of(t.m, a.c);
#pragma unroll 1
      for (int k = lane; k < a.K; k += 32) t.s += power(t_q[k], f);
      tl = ln(warp_sum(t.s));
    }
    double qs = 0.0, ql = 0.0;
#pragma unroll 1
    for (int k = lane; k < a.K; k += 32) {
      const float y = t_q[k];
      const double lq = (tail ? (double)y * a.inv_tau : above(y, t.m, a.c, a.inv_tau)) - tl;
      const float hi = (float)lq;  // q to fp32's last digits: lq rounded, the rest applied
      // (below the smallest fp32 already at -104; there a masked y's rest may be infinite)
      const float q = y == -INFINITY || lq < -110.0 ? 0.f : expf(hi) * (1.f + (float)(lq - (double)hi));
      t_q[k] = q;
      if (t_g[k] == 0.f) t_g[k] = q;
      qs += (double)q;
      if (q > 0.f) ql += (double)q * lq;
    }
    qs = warp_sum_d(qs);
    ql = warp_sum_d(ql);
    __syncwarp();
    if (lane == 0) {
      s_q[0] = qs;
      s_q[1] = ql;
      s_q[2] = tail ? fmax(0.0, 1.0 - qs) : 0.0;
    }
  };

  // ---- groups of pieces
  const uint32_t none = minus_inf_word((const TI*)nullptr);
  auto in_ring = [&](int g, int r, uint4 (&u)[U]) {
    if ((g + 1) * U * NT <= np) {
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = at[(r * U + j) * NT];
    } else {
#pragma unroll
      for (int j = 0; j < U; ++j)
        u[j] = g * U + j < mine ? at[(r * U + j) * NT] : make_uint4(none, none, none, none);
    }
  };
  auto anew = [&](int g, uint4 (&u)[U]) {  // from the logits
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = g * U + j;
      u[j] = k >= mine ? make_uint4(none, none, none, none) : whole(k) ? src[k * NT] : edge(tid + k * NT);
    }
  };
  // listed elements count as -inf where the rest is a class of its own
  auto without_listed = [&](int g, uint4 (&u)[U]) {
    if constexpr (tail) {
      if (!(has >> (g * U >> kHasShift) & (kHasShift ? 1u : (1u << U) - 1))) return;
      uint32_t m[U];
  #pragma unroll
      for (int j = 0; j < U; ++j) {
        const int k = g * U + j, e = (tid + k * NT) * EI;
        m[j] = k < mine ? bits[e >> 5] >> (e & 31) & ((1u << EI) - 1) : 0u;
      }
  #pragma unroll
      for (int j = 0; j < U; ++j)
        if (m[j]) {
          uint32_t* word = &u[j].x;
  #pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t half = EI == 8 ? (m[j] >> (2 * i) & 1 ? 0xffffu : 0u) | (m[j] >> (2 * i + 1) & 1 ? 0xffff0000u : 0u)
                                          : (m[j] >> i & 1 ? 0xffffffffu : 0u);
            word[i] = (word[i] & ~half) | (none & half);
          }
        }
    }
  };
  // a group whose maximum and sum have been taken
  // (shifted: less the maximum, so that they too are not what the ring holds)
  auto keep = [&](int g, int r, const uint4 (&u)[U], bool shifted = false) {
    if (kOnce || !dz) return;
    if (g < moved) {
      if constexpr (kTmem) {
        __syncwarp();
        tmem_put(lane_tmem + (uint32_t)(g * 4 * U), u);
      }
    } else if (kKeepPower || shifted) {
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (!kFits || g * U + j < mine) at[(r * U + j) * NT] = u[j];
    }
  };
  auto kept = [&](int g, int r, uint4 (&u)[U]) {
    if constexpr (kTmem)
      if (g < moved) {
        __syncwarp();
        tmem_get(lane_tmem + (uint32_t)(g * 4 * U), u);
        return;
      }
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = at[(r * U + j) * NT];
  };
  // wait for group g's copies: `first` groups were under way at the start, and
  // one more is whenever one has been used
  // (where all are under way at the start, for all: it is less to execute)
  auto wait_group = [&](int g) {
    if (groups > ring && OP == kLogp) copy_wait_for<kPassing / U - 1>();
    else if (!kFits && groups > ring) copy_wait_for<kKept / U - 1>();
    else if (g == 0) copy_wait_for<0>();
  };
  auto refill = [&](int g, int r) {  // place r, which held group g
    if (kFits || groups <= ring) return;
    const int next = g + ring;
    if (next < groups) {
      copy_group(next, r);
      if (next == g_tail && tid == f1 % NT) copy_edges(next, r);
    } else {
      copy_commit();
    }
  };

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

  // ---- maximum and sum
  MaxSum rest = {-INFINITY, 0.f}, listed = {-INFINITY, 0.f}, all = {-INFINITY, 0.f};
  float count = 0.f;
  float my_base = 0.f;  // the b of this thread's powers
  if constexpr (OP != kLogpBwd) {
    float m = -INFINITY;
    float2 s0 = make_float2(0.f, 0.f), s1 = s0, nb = s0, c2 = make_float2(a.c, a.c);
    auto largest = [&](const uint4 (&u)[U]) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float2 x[EI / 2];
        unpack(u[j], x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i) m = tc::fmax3(m, x[i].x, x[i].y);
      }
    };
    auto add = [&](uint4 (&u)[U]) {  // fp32 logits become their powers
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float2 x[EI / 2];
        unpack(u[j], x, (const TI*)nullptr);
#pragma unroll
        for (int i = 0; i < EI / 2; ++i) {
          const float2 t = tc::ffma2(x[i], c2, nb);
          const float2 e = make_float2(tc::fast_exp2(t.x), tc::fast_exp2(t.y));
          if (i & 1) s1 = tc::fadd2(s1, e);
          else s0 = tc::fadd2(s0, e);
          x[i] = e;
        }
        if (kKeepPower)
          u[j] = make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x),
                            __float_as_uint(x[1].y));
      }
    };
    auto relative_to_m = [&] {
      my_base = base_of(m, a.c);
      nb = make_float2(-my_base, -my_base);
    };
    auto sum = [&] { return (s0.x + s0.y) + (s1.x + s1.y); };
    uint4 u[U];
    if (owner) {
      // relative to the largest of this thread's first pieces
      if (groups > 0) {
        wait_group(0);
        in_ring(0, 0, u);
        without_listed(0, u);
        largest(u);
        relative_to_m();
      }
      const int full = np / (NT * U);  // groups of which every thread has all pieces
      for (int g = 0, r = 0; g < full; ++g) {
        wait_group(g);
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = at[(r * U + j) * NT];
        without_listed(g, u);
        add(u);
        keep(g, r, u);
        refill(g, r);
        if (++r == ring) r = 0;
      }
      if (full < groups) {
        const int r = kFits ? full : full % ring;
        wait_group(full);
        in_ring(full, r, u);
        without_listed(full, u);
        add(u);
        keep(full, r, u);
      }
      // (a sum that passes its base by 2^64 is none: joined, it would meet a
      // power below 2^-126, which is 0)
      const float v = sum();
      rest = warp_join({m, v < 0x1p64f ? v : INFINITY}, a.c);
    }
    double qz = 0.0;
    if (!owner) {
      make_q();
#pragma unroll 1
      for (int k = lane; k < a.K; k += 32) {
        const int i = t_idx[k];
        if (i >= e_lo && i < e_hi && t_q[k] != 0.f) qz += (double)t_q[k] * (double)t_z[k];
      }
      qz = warp_sum_d(qz);
      if (tail) {  // the listed entries' maximum and sum
        if (twice) count_once();
#pragma unroll 1
        for (int k = lane; k < a.K; k += 32)
          if (!(t_g[k] < 0.f)) {
            listed.m = fmaxf(listed.m, t_z[k]);
            count += 1.f;
          }
        listed.m = warp_max_redux(listed.m);
        const Form f = form_of(listed.m, a.c);
#pragma unroll 1
        for (int k = lane; k < a.K; k += 32)
          if (!(t_g[k] < 0.f)) listed.s += power(t_z[k], f);
        listed.s = warp_sum(listed.s);
        count = warp_sum(count);
      }
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
    // A sum relative to first pieces is none when later elements pass them by
    // 2^64, nor is one of a far maximum; then all is taken once more, relative
    // to the maximum of the row, which is subtracted from what is kept where
    // it is far.
    auto not_one = [&](const MaxSum& v) { return is_far(v.m, a.c) || !(v.s < INFINITY); };
    if (OP == kLogp && C == 1 && warp != 0) {  // (which needs every warp)
      bool once_more = false;
      for (int i = 0; i < NW; ++i) once_more = once_more || not_one(s_rest[i]);
      if (!once_more) return;
    }
    rest = {-INFINITY, 0.f};
    for (int i = lane; i < C * NW; i += 32) rest = join(rest, s_rest[i], a.c);
    rest = warp_join(rest, a.c);
    if (not_one(rest)) {
      auto exchange = [&](float v, float* slots) {
        if (owner) tell(&slots[rank * NW + warp], v);
        told();
      };
      if (owner)
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
          anew(g, u);
          without_listed(g, u);
          largest(u);
        }
      exchange(warp_max_redux(m), s_again);
      m = -INFINITY;
      for (int i = lane; i < C * NW; i += 32) m = fmaxf(m, s_again[i]);
      rest.m = warp_max_redux(m);
      const Form f = form_of(rest.m, a.c);
      const bool far = is_far(rest.m, a.c);
      nb = make_float2(-f.b, -f.b);
      my_base = f.b;
      s0 = s1 = make_float2(0.f, 0.f);
      if (owner)
#pragma unroll 1
        for (int g = 0, r = 0; g < groups; ++g) {
          anew(g, u);
          without_listed(g, u);
          if (far)
#pragma unroll
            for (int j = 0; j < U; ++j) u[j] = minus(u[j], f.m, (const TI*)nullptr);
          add(u);
          keep(g, r, u, far);
          if (++r == ring) r = 0;
        }
      exchange(warp_sum(sum()), s_again + kMaxCluster * NW);
      float v = 0.f;
      for (int i = lane; i < C * NW; i += 32) v += s_again[kMaxCluster * NW + i];
      rest.s = warp_sum(v);
    }
    if constexpr (kTmem) tc::tmem_st_wait();
    if (tail) {  // (without a class for the rest nothing is listed apart)
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
    all = rest;
    if (tail) {
      all.m = fmaxf(rest.m, listed.m);
      all.s = rest.s * rescale(rest.m, all.m, a.c) + listed.s * rescale(listed.m, all.m, a.c);
    }
    if (kList && is_far(all.m, a.c)) {
      // the sum of q (z - m) instead, which keeps its digits
      if (!owner) {
        qz = 0.0;
#pragma unroll 1
        for (int k = lane; k < a.K; k += 32)
          if (t_idx[k] >= e_lo && t_idx[k] < e_hi && t_q[k] != 0.f)
            qz += (double)t_q[k] * ((double)t_z[k] - (double)all.m);
        qz = warp_sum_d(qz);
        tell(&s_qz[rank], qz);
      }
      told();
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
    // 2^(c z - log2(e) lse): the whole part stays in the exponent
    const double l2 = (double)lse_in * kLog2e;
    hot = (float)((double)dlogp * a.inv_tau);
    f = {a.c, (float)rint(l2), 0.f};
    c_out = -hot * tc::fast_exp2((float)((double)f.b - l2));
  } else if (OP == kPolicy) {
    // in double: a KL term is a small difference, and a ratio may be beyond
    // fp32 where the advantage is 0 or the clip holds
    const double logp = above(za, rest.m, a.c, a.inv_tau) - log((double)rest.s);
    const double A = (double)adv, ratio = exp(logp - (double)old_logp);
    const double lo = 1.0 - a.clip_low, hi = 1.0 + a.clip_high;
    const bool clipped = (A > 0.0 && ratio > hi) || (A < 0.0 && ratio < lo);
    double l = clipped ? -(A > 0.0 ? hi : lo) * A : -ratio * A;
    double d = clipped ? 0.0 : -A * ratio;
    if (a.ref_logp) {
      const double gap = (double)ref_logp - logp, e = expm1(gap);
      l += a.kl_coef * (e - gap);
      d -= a.kl_coef * e;
    }
    if (tid == 0 && rank == 0) {
      a.row_loss[row] = (float)((double)w * l);
      a.logp[row] = (float)logp;
    }
    hot = (float)(a.scale * a.inv_tau * (double)w * d);
    c_out = -hot / rest.s;
  } else {
    f_in = form_of(all.m, a.c);
    // without an entry outside the list there is no class for the rest
    const float q_sum = (float)s_q[0], q_rest = count == (float)V ? 0.f : (float)s_q[2];
    hot = (float)(a.scale / a.inv_tau) * w;
    c_in = hot * (q_sum + q_rest) / all.s;
    // outside the list relative to the largest logit there: the student's
    // mass outside may be too small to be held relative to the row's largest
    // (none at all: an infinite loss, and entries of probability 0)
    c_out = rest.s == 0.f ? (all.s > 0.f ? 0.f : NAN)
                          : c_in * rescale(rest.m, all.m, a.c) -
                                (q_rest > 0.f ? hot * q_rest / rest.s : 0.f);
    if (!owner && rank == 0 && lane == 0) {
      const double qs = s_q[0], ls_all = ln(all.s), ls_rest = ln(rest.s);
      double qz = 0.0;
#pragma unroll 1
      for (int i = 0; i < C; ++i) qz += s_qz[i];
      // sum of q (z / tau - lse), as above() has it of one z
      const bool far = is_far(all.m, a.c);
      const double x = far ? qz * a.inv_tau : (qz * (double)a.c - qs * (double)f_in.b) * kLn2;
      double l = s_q[1] - (x - qs * ls_all);
      if (q_rest > 0.f) {  // -log of the student's share outside the list
        const double apart = far && is_far(rest.m, a.c)
                                 ? ((double)all.m - (double)rest.m) * a.inv_tau
                                 : (origin(all.m, a.c) - origin(rest.m, a.c)) * kLn2;
        l += (double)q_rest * ((double)logf(q_rest) + (ls_all - ls_rest) + apart);
      }
      a.row_loss[row] = (float)((double)w * l / (a.inv_tau * a.inv_tau));
    }
    if (!owner && !tail && dz) {
      __syncwarp();
      if (set_bits()) count_once();
    }
  }
  if (!dz) {
    if constexpr (kTmem) {
      tc::tc_fence_before();
      __syncthreads();
      if (warp == 0) free_columns<columns_of(S)>(s_tmem);
    }
    return;
  }

  // ---- the adjoint
  // powers that were kept are relative to this thread's own base (each below
  // 2^64: where this factor underflows, what is lost is below 2^-62 of `hot`)
  if (kKeepPower && !is_far(rest.m, a.c)) c_out *= tc::fast_exp2(my_base - f.b);
  const float2 c2 = make_float2(f.c, f.c), nb = make_float2(-f.b, -f.b);
  const float2 g2 = make_float2(c_out, c_out);
  const int off = (int)((uintptr_t)(dz + e_org) % (EI * sizeof(TO)));  // of every piece's place in dz
  auto values = [&](uint4 u, int e, float (&v)[EI]) {  // v[0] is element e's
    float2 x[EI / 2];
    unpack(u, x, (const TI*)nullptr);
#pragma unroll
    for (int i = 0; i < EI / 2; ++i) {
      if (!kKeepPower) {
        const float2 t = tc::ffma2(x[i], c2, nb);
        x[i] = make_float2(tc::fast_exp2(t.x), tc::fast_exp2(t.y));
      }
      const float2 d = tc::fmul2(x[i], g2);
      v[2 * i] = d.x;
      v[2 * i + 1] = d.y;
    }
    const unsigned to = (unsigned)(token - e);
    if (!kList && to < (unsigned)EI) {
#pragma unroll
      for (int i = 0; i < EI; ++i)
        if (to == (unsigned)i) v[i] += hot;
    }
  };
  auto give = [&](int e, const uint4 (&u)[U]) {  // a group that lies in the row, aligned
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[EI];
      values(u[j], e + j * (NT * EI), v);
      store_n(dz + e + j * (NT * EI), v);
    }
  };
  auto give_one = [&](int k, uint4 u) {  // any piece
    const int e = e_org + (tid + k * NT) * EI;
    float v[EI];
    values(u, e, v);
    if (whole(k)) {
      if (off == 0) store_n(dz + e, v);
      else store_off(dz + e, v, off);
    } else if (k < mine) {
      store_elements(dz, e, V, EI, make_float4(v[0], v[1], v[2], v[3]),
                     make_float4(v[EI - 4], v[EI - 3], v[EI - 2], v[EI - 1]));
    }
  };
  if constexpr (kFits) {
    if (owner) {
      // groups [ga, gb) of this thread lie in the row
      const int ga = tid < f0 ? 1 : 0, last = f1 - 1 - tid - (U - 1) * NT;
      const int gb = off == 0 && last >= 0 ? last / (U * NT) + 1 : 0;
      for (int g = ga; g < gb; ++g) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = at[(g * U + j) * NT];
        give(e_org + (tid + g * U * NT) * EI, u);
      }
#pragma unroll 1
      for (int k = 0; k < mine; ++k) {
        if (k == ga * U && gb > ga) k = gb * U;
        if (k < mine) give_one(k, at[k * NT]);
      }
    }
  } else if (owner) {
    for (int g = 0, r = 0; g < groups; ++g) {
      uint4 u[U];
      if (kOnce) wait_group(g);
      kept(g, r, u);
      const int i = tid + g * U * NT;
      if (off == 0 && i >= f0 && i + (U - 1) * NT < f1) {
        give(e_org + i * EI, u);
      } else {
#pragma unroll 1
        for (int j = 0; j < U; ++j) give_one(g * U + j, j ? u[1] : u[0]);
      }
      if (kOnce) refill(g, r);
      if (++r == ring) r = 0;
    }
  }
  if (kList || kTmem) {
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
  }
  if constexpr (kTmem)
    if (warp == 0) free_columns<columns_of(S)>(s_tmem);
  if (kList)
#pragma unroll 1
    for (int k = tid; k < a.K; k += THREADS)
      if (!(t_g[k] < 0.f))
        st(&dz[t_idx[k]], c_in * power(t_z[k], f_in) - hot * t_g[k]);
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

template <RowOp OP, typename TI, typename TO, Shape S>
__global__ void __launch_bounds__(kThreadsOf<OP, S>, kCtasPerSM<OP, S>) k_vocab_row(const RowArgs a) {
  if (OP == kLogpBwd) {
    // it has nothing to exchange: plain CTAs.  Last rows first: they are the
    // ones that the log-probabilities' pass has left in L2
    const unsigned C = (unsigned)a.cluster, r = blockIdx.x / C;
    if (r == a.rows) return scaled_sum_of<owners_of(S)>(a.sum_of, a.sum_n, a.scale, a.loss);
    vocab_row<OP, TI, TO, S>(a, a.rows - 1 - r, (int)(blockIdx.x % C));
  } else {
    uint32_t row;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(row));
    vocab_row<OP, TI, TO, S>(a, row, (int)tc::cluster_ctarank());
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
__global__ void __launch_bounds__(kPairThreads) k_preference_pair(const __grid_constant__ PairArgs a) {
  __shared__ double s_red[kPairThreads / 32];
  const int pair = blockIdx.x;
  const int64_t* off = a.off + 2 * pair;
  auto weight_of = [&](int64_t t) {
    const int64_t k = a.tokens[t];
    return k < 0 || k >= a.V ? 0.f : (a.weight ? a.weight[t] : 1.f);
  };
  double sum[2], len[2];
  for (int q = 0; q < 2; ++q) {
    double s = 0.0, n = 0.0;
    for (int64_t t = off[q] + threadIdx.x; t < off[q + 1]; t += kPairThreads) {
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
    for (int64_t t = off[q] + threadIdx.x; t < off[q + 1]; t += kPairThreads) {
      const float w = weight_of(t);
      a.dlogp[t] = w == 0.f ? 0.f : (float)(g * (double)w);
    }
  }
}

// ------------------------------------------------------------------- host
// Shared memory of a list of K entries, without its bits.
constexpr int64_t list_bytes(int K) { return 16 * list_stride(K); }
constexpr int64_t kDynamicMost = 16 * owners_of(kAlone) * kRingMost + list_bytes(kMaxTeacherK) +
                                 owners_of(kAlone) * (kRingMost + kMovedMost);  // (a bit per bf16 logit)
static_assert(kDynamicMost + 2560 <= 232448, "more shared memory than a CTA may have");
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

// How the rows are laid out over CTAs.  A row whose pieces are kept goes to
// one narrow or held CTA or to as few wide ones as hold it; more of them where
// the rows are too few to occupy the SMs (down to 16 KB each).  Both sides, in
// us: narrow against held for 16384 x 16001 bf16, policy loss 209 / 269,
// distillation 250 / 340, with a rest class 274 / 371; one held CTA against two
// narrow ones for 32768 x 32000 bf16, distillation 809-827 / 861-867, and
// against a wide one, 8192 rows, 214 / 228; a wide CTA against four narrow ones
// for 8192 x 32000 fp32, policy loss 218 / 268; two wide ones against three
// held ones for 3001 x 100003 bf16, policy loss 253 / 258, and 3000 rows
// distilled with a rest class 276-281 / 400 (groups of two pieces in both).
struct Split {
  int cluster, share;  // CTAs per row; pieces per CTA
  Shape shape;
  int ring;            // places for pieces per owner
};
Split split_of(int64_t rows, int64_t vocab, int prec, bool once, int passing) {
  // the pieces that a row touches wherever it starts
  const int64_t size = prec == DOP_BF16 ? 2 : 4, pieces = ceil_div(vocab * size + 16 - size, 16);
  const int64_t narrow = kKept * owners_of(kNarrow), held = kHeldMost * owners_of(kHeld);
  const int64_t wide = 2 * kKept * owners_of(kWide);
  const int64_t fit = once ? 1 : ceil_div(pieces, pieces <= held ? held : wide);
  const int64_t fill = std::min(ceil_div(3 * sm_count(), std::max<int64_t>(rows, 1)), ceil_div(pieces, 1024));
  const int64_t C = std::min<int64_t>(std::max(fit, fill), kMaxCluster), share = ceil_div(pieces, C);
  if (rows * C >= INT32_MAX) throw Error(DOP_E_UNSUPPORTED, "too many rows for this vocab");
  if (once) return {(int)C, (int)share, kNarrow, passing};
  const Shape shape = share <= narrow ? kNarrow : share <= held ? kHeld : share <= wide ? kWide : kAlone;
  int64_t each = ceil_div(share, owners_of(shape));
  if (columns_of(shape) > 0) each = round_up(each, 2);  // in groups of 2
  if (each > kRingMost + kMovedMost)
    throw Error(DOP_E_UNSUPPORTED,
                "vocab (" + std::to_string(vocab) + ") is above " +
                    std::to_string((C * owners_of(kAlone) * 16 * (kRingMost + kMovedMost) - 16) / size + 1));
  const int most = shape == kAlone ? kRingMost : shape == kHeld ? kHeldMost : kKept;
  return {(int)C, (int)share, shape, (int)std::min<int64_t>(each, most)};
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
  constexpr bool once = OP == kLogp || OP == kLogpBwd;
  const Split sp = split_of(rows, a.V, prec, once, OP == kLogp ? kPassing : kKept);
  a.rows = rows;
  a.cluster = sp.cluster;
  a.share = sp.share;
  a.ring = sp.ring;
  a.stage_bytes = 16 * owners_of(sp.shape) * sp.ring;
  int64_t smem = a.stage_bytes;
  if (has_list(OP)) {
    const int64_t elements = (int64_t)sp.share * (prec == DOP_BF16 ? 8 : 4);
    a.bit_words = (int)ceil_div(OP == kDistillRest ? elements : (int64_t)kFilterBits, 32);
    smem += list_bytes(a.K) + 4 * a.bit_words;
  }
  if (sp.shape == kAlone) smem = std::max(smem, kAloneBytes);
  const int64_t ctas = rows * a.cluster + (OP == kLogpBwd && a.loss ? 1 : 0);  // (one for the sum)
  const int cluster = OP == kLogpBwd ? 1 : a.cluster;
  by_types(prec, grad_prec, a.dz != nullptr, [&](auto ti, auto to) {
    using TI = decltype(ti);
    using TO = decltype(to);
    auto go = [&](auto shape) {
      constexpr Shape S = decltype(shape)::value;
      launch(k_vocab_row<OP, TI, TO, S>, a, ctas, kThreadsOf<OP, S>, smem, cluster, s);
    };
    if constexpr (!once) {
      if (sp.shape == kAlone) return go(std::integral_constant<Shape, kAlone>{});
      if (sp.shape == kWide) return go(std::integral_constant<Shape, kWide>{});
      if (sp.shape == kHeld) return go(std::integral_constant<Shape, kHeld>{});
    }
    go(std::integral_constant<Shape, kNarrow>{});
  });
}

int elem_bytes(int prec) { return prec == DOP_BF16 ? 2 : 4; }

// The checks every objective shares.
void check_rows(int64_t rows, int64_t vocab, int prec, const void* z, int64_t ld, double tau) {
  DOP_REQUIRE(rows >= 0 && rows <= INT32_MAX, "rows must lie in [0, 2^31)");
  DOP_REQUIRE(vocab >= 1 && vocab <= INT32_MAX, "vocab must lie in [1, 2^31)");
  DOP_REQUIRE(prec == DOP_F32 || prec == DOP_BF16, "unknown precision");
  split_of(rows, vocab, prec, false, 0);
  DOP_REQUIRE(ld >= vocab, "the logits' row stride is smaller than vocab");
  DOP_REQUIRE(z || rows == 0, "null logits");
  DOP_REQUIRE((uintptr_t)z % elem_bytes(prec) == 0, "misaligned logits");
  DOP_REQUIRE(tau >= 0x1p-16 && tau <= 0x1p16, "temperature must lie in [2^-16, 2^16]");
}
// dlogits: bf16 or the logits' type; either exactly the logits' memory (same
// type and stride), apart from it, or between its rows.
void check_grad(int64_t rows, int64_t vocab, int prec, const void* z, int64_t ld, int grad_prec,
                const void* dz, int64_t ldd) {
  if (!dz) return;
  DOP_REQUIRE(grad_prec == DOP_F32 || grad_prec == DOP_BF16, "unknown gradient precision");
  DOP_REQUIRE(prec == DOP_F32 || grad_prec == DOP_BF16, "bf16 logits have bf16 dlogits");
  DOP_REQUIRE(ldd >= vocab, "the row stride of dlogits is smaller than vocab");
  DOP_REQUIRE((uintptr_t)dz % elem_bytes(grad_prec) == 0, "misaligned dlogits");
  if (rows == 0 || (dz == z && prec == grad_prec && (ld == ldd || rows == 1))) return;
  const int64_t size = elem_bytes(prec), gsize = elem_bytes(grad_prec);
  const uintptr_t z0 = (uintptr_t)z, d0 = (uintptr_t)dz;
  const uintptr_t z1 = z0 + ((rows - 1) * ld + vocab) * size, d1 = d0 + ((rows - 1) * ldd + vocab) * gsize;
  if (z1 <= d0 || d1 <= z0) return;
  // rows equally far apart may lie between each other: by where a row of
  // dlogits starts behind the start of a row of logits
  if (ld * size == ldd * gsize) {
    const int64_t stride = ld * size;
    const int64_t behind = d0 >= z0 ? (int64_t)((d0 - z0) % stride)
                                    : (stride - (int64_t)((z0 - d0) % stride)) % stride;
    if (behind >= vocab * size && behind + vocab * gsize <= stride) return;
  }
  DOP_REQUIRE(false, "dlogits overlaps the logits without being the same rows in the same type");
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
      k_preference_pair<<<(unsigned)n, kPairThreads, 0, s>>>(pa);
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
    (teacher_lse ? launch_rows<kDistillRest> : launch_rows<kDistill>)(a, rows, precision, grad_precision,
                                                                      as_stream(stream));
    scaled_sum(row_loss, rows, scale, loss, as_stream(stream));
  });
}

}  // extern "C"
