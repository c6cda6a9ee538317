/*!
 * Device operators over class scores for MI355X (gfx950): top logits, the distillation loss
 * with its gradient, and the verification of drafted classes.
 *
 * A row (or a sequence) belongs to a few lanes, a wave or a workgroup, by its number of classes
 * and by which of its strides is the smaller. Everything is held in 32 bits (64 for float64
 * scores); exponentials are taken to base two,
 *   exp((z - high) / T) = 2^((z - high) * s),  s = log2(e) / T,
 * of a difference that is formed first: z * s - high * s would be one operation, but high * s may
 * not be a number (masks of the type's lowest value) or be off by more than the exponent's range
 * (large scores at a small T), and is another factor wherever another maximum stands for high.
 */
#include <hip/hip_runtime.h>

#include "migbm/class_ops.h"
#include "migbm/common.h"

#include <algorithm>
#include <cfloat>
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

namespace migbm {
namespace class_ops {
namespace {

#define OPS_HIP_OK(call)                                                                 \
  do {                                                                                   \
    hipError_t _e = (call);                                                              \
    if (_e != hipSuccess)                                                                \
      ::migbm::Log::Fatal("HIP error %s at %s:%d", hipGetErrorString(_e), __FILE__,      \
                          __LINE__);                                                     \
  } while (0)

// ------------------------------------------------------------------ elements
/*! what a row of T is computed in: 64 bits for float64 scores, 32 for the others */
template <typename T> using Acc = std::conditional_t<std::is_same_v<T, double>, double, float>;
/*! the type of gradients: the framework's 32-bit gradient for float64 scores */
template <typename T> using Out = std::conditional_t<std::is_same_v<T, double>, float, T>;

template <typename A> __device__ __forceinline__ A NegInf() { return -static_cast<A>(INFINITY); }
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double Exp2(double x) { return exp2(x); }
/*!
 * 2^x to 2e-10 of itself, for sums and quotients that end in 32 bits: the exponential's series in
 * f ln 2, |f| <= 1/2, whose ninth term is at most (ln 2 / 2)^9 / 9!. 0 for -inf, NaN for NaN.
 */
__device__ __forceinline__ double ShortExp2(double x) {
  constexpr double kLn2 = 0.69314718055994530942;
  // a multiply-add whose addend is a scalar: the compiler's own form copies it to registers
  auto step = [](double p, double f, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(p), "v"(f), "s"(c));
    return r;
  };
  const double n = rint(x), f = (x - n) * kLn2;
  double p = 1.0 / 40320;
  p = step(p, f, 1.0 / 5040);
  p = step(p, f, 1.0 / 720);
  p = step(p, f, 1.0 / 120);
  p = step(p, f, 1.0 / 24);
  p = step(p, f, 1.0 / 6);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return x < -1000.0 ? 0.0 : ldexp(p, static_cast<int>(n));
}
__device__ __forceinline__ float Log2(float x) { return log2f(x); }
__device__ __forceinline__ double Log2(double x) { return log2(x); }
__device__ __forceinline__ float Fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float Max(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double Max(double a, double b) { return fmax(a, b); }

template <typename T> __device__ __forceinline__ T At(const LGBM_Array& a, int64_t at) {
  return static_cast<const T*>(a.data)[at];
}

/*! one of the small arrays (teacher, weights): its type is the same for the whole launch */
template <typename A> __device__ __forceinline__ A LoadFloat(const LGBM_Array& a, int64_t at) {
  switch (a.type) {
    case C_API_DTYPE_FLOAT64: return static_cast<A>(At<double>(a, at));
    case C_API_DTYPE_FLOAT32: return static_cast<A>(At<float>(a, at));
    case C_API_DTYPE_FLOAT16: return static_cast<A>(At<_Float16>(a, at));
    default: return static_cast<A>(static_cast<float>(At<__bf16>(a, at)));
  }
}

/*! a class id in 0..classes-1, or -1; float32 labels are whole numbers held in a float */
__device__ __forceinline__ int LoadClass(const LGBM_Array& a, int64_t at, int classes) {
  int64_t v;
  if (a.type == C_API_DTYPE_INT32) {
    v = At<int32_t>(a, at);
  } else if (a.type == C_API_DTYPE_INT64) {
    v = At<int64_t>(a, at);
  } else {
    const float f = At<float>(a, at);
    v = f >= 0.0f && f < 4e9f ? static_cast<int64_t>(f) : -1;
  }
  return v >= 0 && v < classes ? static_cast<int>(v) : -1;
}

template <typename A>
__device__ __forceinline__ void StoreFloat(const LGBM_Array& a, int64_t at, A v) {
  if (a.type == C_API_DTYPE_FLOAT64) static_cast<double*>(a.data)[at] = v;
  else static_cast<float*>(a.data)[at] = static_cast<float>(v);
}

// ------------------------------------------------------------------ keys
/*! keys order as the values do, zeros of both signs alike; 0: never chosen (NaN, -inf) */
__device__ __forceinline__ uint32_t KeyOf(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t KeyOf(double v) {
  if (!(v > -INFINITY)) return 0ull;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b >> 63 ? ~b : b | (1ull << 63);
}
/*! the value of a key that is not zero */
__device__ __forceinline__ float ValueOf(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ double ValueOf(uint64_t key) {
  return __longlong_as_double(static_cast<long long>(key >> 63 ? key & ~(1ull << 63) : ~key));
}

// ------------------------------------------------------------------ reductions
constexpr int kWave = 64;

template <typename A> __device__ __forceinline__ A WaveSum(A v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
template <typename A> __device__ __forceinline__ A WaveMax(A v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v = Max(v, __shfl_xor(v, d));
  return v;
}

/*! sums (maxima) over the workgroup, known to every thread, always in the same order.
 *  `lds` has one place a wave; it may be used again after the next barrier. */
template <int kBlock, typename A> __device__ __forceinline__ A BlockSum(A v, A* lds) {
  v = WaveSum(v);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  A s = lds[0];
#pragma unroll
  for (int i = 1; i < kBlock / kWave; ++i) s += lds[i];
  return s;
}
template <int kBlock, typename A> __device__ __forceinline__ A BlockMax(A v, A* lds) {
  v = WaveMax(v);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  A s = lds[0];
#pragma unroll
  for (int i = 1; i < kBlock / kWave; ++i) s = Max(s, lds[i]);
  return s;
}

// ------------------------------------------------------------------ distillation, any strides
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;

/*! where the student's share of the unnamed classes is below this, it is summed again
 *  against its own maximum: 2^-100 of the row's largest term is near the end of 32 bits */
template <typename A> __device__ __forceinline__ A SmallRest() { return static_cast<A>(0x1p-100); }

/*!
 * A row's teacher: the weights of its slots and of its rest, as exponents to base two against
 * the largest of them. Logits may have any common offset, and a rounding at their size is
 * another factor for each slot, so they are subtracted as they are, and in 64 bits: 32 would move
 * the probabilities by 9e-5 at logits near 1000. `largest` is the slots' largest logit,
 * `log_rest` the rest's logarithm at the temperature, -inf where there is none; `by` is
 * log2(e) / T.
 */
struct TeacherScale {
  double scale, top, shift, rest;
  __device__ __forceinline__ TeacherScale(double largest, double log_rest, double by)
      : scale(by), top(0.0), shift(0.0) {
    const bool some = largest > -INFINITY;
    if (some) top = largest;
    rest = some ? fma(-top, scale, log_rest * kLog2e) : 0.0;
    if (log_rest == -INFINITY) rest = -INFINITY;  // whatever the slots are
    else if (!(log_rest < INFINITY)) rest = NAN;  // of infinite weights none is a share
    if (rest > 0.0) {
      shift = -rest;
      rest = 0.0;
    }
  }
  template <typename S> __device__ __forceinline__ S Slot(double logit) const {
    return static_cast<S>(fma(logit - top, scale, shift));
  }
  template <typename S> __device__ __forceinline__ S Rest() const { return static_cast<S>(rest); }
};

/*!
 * p log(p / q) of a class or of the rest, whose logarithm of q is that of a score `far` below the
 * row's largest: log_pq is the logarithm of p over q without it, to base two. In 64 bits, as a
 * score of the type's lowest value is farther than 32 hold, and the loss it makes is not.
 */
__device__ __forceinline__ double Divergence(double p, double log_pq, double far,
                                             double temperature) {
  return p * (log_pq * kLn2 - far / temperature);
}

/*!
 * One workgroup a row, the row read from memory in each of its passes: maximum, sums,
 * gradients. With the teacher's slots (class c_j, logit t_j) and, where given, the
 * logarithm r of what it gives to all other classes,
 *   P = softmax(t_1 / T, .., t_k / T, r),  Q = softmax(z / T),  rho = sum of Q over the others,
 *   loss = w * (alpha T^2 (sum_j P_j log(P_j / Q_cj) + P_r log(P_r / rho))
 *               + (1 - alpha) (-log softmax(z)_y)),
 *   dloss / dz_c = w * (alpha T (Q_c - P_c) + (1 - alpha)(softmax(z)_c - [c = y])),
 *     where P_c = P_r Q_c / rho for a class without a slot,
 *   hessian_c = w * C / (C - 1) * (alpha Q_c (1 - Q_c) + (1 - alpha) p_c (1 - p_c)).
 * The slots' classes are bits in LDS, so that the sum over the others is taken directly and
 * not as a difference, which a confident student would cancel to nothing. The first slot of
 * a class counts. It serves what the kernels below do not: more than 512 classes of float64 or
 * in strides. Bound by its three passes over memory, one element a thread (8192 x 32768 bfloat16
 * gradients and loss of every second column 1039 us; of neighbours, by the rows' kernel, 233).
 */
template <typename T, int kBlock>
__global__ void __launch_bounds__(kBlock) k_distill_any(LGBM_DistillArgs a, double by) {
  using A = Acc<T>;
  extern __shared__ uint32_t mark[];
  __shared__ int s_cls[kMaxTop];
  __shared__ A s_red[6][kBlock / kWave];
  __shared__ double s_top[kBlock / kWave];
  __shared__ int s_dup;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, c = a.classes, k = a.k;
  const T* z = static_cast<const T*>(a.scores.data) + row * a.scores.stride[0];
  const int64_t zs = a.scores.stride[1];
  using O = Out<T>;
  O* grad = a.gradient.data ? static_cast<O*>(a.gradient.data) + row * a.gradient.stride[0]
                            : nullptr;
  O* hess = a.hessian.data ? static_cast<O*>(a.hessian.data) + row * a.hessian.stride[0]
                           : nullptr;
  const int64_t gs = a.gradient.stride[1], hs = a.hessian.stride[1];
  const A w = a.weight.data ? LoadFloat<A>(a.weight, row * a.weight.stride[0]) : A(1);
  const A temp = static_cast<A>(a.temperature), alpha = static_cast<A>(a.alpha);
  const A scale = static_cast<A>(by), scale1 = static_cast<A>(kLog2e);

  for (int i = tid; i < (c + 31) / 32; i += kBlock) mark[i] = 0;
  if (tid == 0) s_dup = 0;
  A high = NegInf<A>();
  bool nan = false;
  if (w != A(0)) {
    for (int i = tid; i < c; i += kBlock) {
      const A v = static_cast<A>(z[i * zs]);
      high = Max(high, v);
      nan |= v != v;
    }
  }
  high = BlockMax<kBlock>(high, s_red[0]);
  nan = __syncthreads_or(nan);
  // a row without weight, or with every class masked, has no loss and no gradient
  if (w == A(0) || (high == NegInf<A>() && !nan)) {
    if (a.loss.data && tid == 0) StoreFloat(a.loss, row * a.loss.stride[0], A(0));
    for (int i = tid; i < c; i += kBlock) {
      if (grad) grad[i * gs] = static_cast<O>(0.0f);
      if (hess) hess[i * hs] = static_cast<O>(0.0f);
    }
    return;
  }
  if (high == NegInf<A>()) high = A(0);

  // the slots, one a thread
  int cls = -1;
  if (tid < k) {
    cls = LoadClass(a.teacher_class,
                    row * a.teacher_class.stride[0] + tid * a.teacher_class.stride[1], c);
    if (cls >= 0 && (atomicOr(&mark[cls >> 5], 1u << (cls & 31)) >> (cls & 31) & 1u)) s_dup = 1;
    s_cls[tid] = cls;
  }
  __syncthreads();
  if (s_dup && tid < k) {
    for (int i = 0; i < tid; ++i)
      if (s_cls[i] == cls) cls = -1;
  }
  const double logit = cls >= 0 ? LoadFloat<double>(a.teacher_logit,
                                                    row * a.teacher_logit.stride[0] +
                                                        tid * a.teacher_logit.stride[1])
                                : NegInf<double>();
  const bool rest = a.teacher_rest.data != nullptr;
  const TeacherScale teacher(
      BlockMax<kBlock>(logit, s_top),
      rest ? LoadFloat<double>(a.teacher_rest, row * a.teacher_rest.stride[0]) : NegInf<double>(),
      by);

  // sums
  const A z_slot = cls >= 0 ? static_cast<A>(z[cls * zs]) : NegInf<A>();
  const A e_slot = cls >= 0 ? Exp2((z_slot - high) * scale) : A(0);
  A left = 0, total1 = 0;
  for (int i = tid; i < c; i += kBlock) {
    const A v = static_cast<A>(z[i * zs]);
    if (!(mark[i >> 5] >> (i & 31) & 1u)) left += Exp2((v - high) * scale);
    if (a.alpha < 1.0) total1 += Exp2((v - high) * scale1);
  }
  left = BlockSum<kBlock>(left, s_red[0]);
  const A total = left + BlockSum<kBlock>(e_slot, s_red[2]);
  if (a.alpha < 1.0) total1 = BlockSum<kBlock>(total1, s_red[3]);
  const A log_u = cls >= 0 ? teacher.template Slot<A>(logit) : NegInf<A>();
  const A log_u_rest = teacher.template Rest<A>();
  const A u = Exp2(log_u), u_rest = Exp2(log_u_rest);
  const A t_sum = BlockSum<kBlock>(u, s_red[4]) + u_rest;
  // the largest weight is one, so a sum of zero is a row without a teacher
  const bool taught = alpha > A(0) && !(t_sum == A(0));
  const A log_total = Log2(total);
  const A p = taught ? u / t_sum : A(0), share = taught ? u_rest / t_sum : A(0);
  A rest_high = high;
  bool again = rest && left < SmallRest<A>();
  if (again) {
    A own = NegInf<A>();
    for (int i = tid; i < c; i += kBlock)
      if (!(mark[i >> 5] >> (i & 31) & 1u)) own = Max(own, static_cast<A>(z[i * zs]));
    own = BlockMax<kBlock>(own, s_red[1]);
    again = own > NegInf<A>();
    if (again) {
      rest_high = own;
      left = 0;
      for (int i = tid; i < c; i += kBlock)
        if (!(mark[i >> 5] >> (i & 31) & 1u))
          left += Exp2((static_cast<A>(z[i * zs]) - own) * scale);
      left = BlockSum<kBlock>(left, s_red[5]);
    }
  }
  const int y = a.alpha < 1.0 ? LoadClass(a.label, row * a.label.stride[0], c) : -1;

  if (a.loss.data) {
    double kl = 0;
    if (cls >= 0 && !(p == A(0)))
      kl = Divergence(p, log_u - Log2(t_sum) + log_total, static_cast<double>(z_slot) - high,
                      a.temperature);
    __syncthreads();
    kl = BlockSum<kBlock>(kl, s_top);
    if (tid == 0) {
      if (rest && !(share == A(0)))
        kl += Divergence(share, log_u_rest - Log2(t_sum) - Log2(left) + log_total,
                         static_cast<double>(rest_high) - high, a.temperature);
      double v = taught ? a.alpha * a.temperature * a.temperature * kl : 0.0;
      if (y >= 0)
        v += (1.0 - a.alpha) *
             (Log2(total1) * kLn2 - (static_cast<double>(static_cast<A>(z[y * zs])) - high));
      StoreFloat(a.loss, row * a.loss.stride[0], v * w);
    }
  }
  if (!grad && !hess) return;
  const A soft = taught ? alpha : A(0), hard = y >= 0 ? static_cast<A>(1.0 - a.alpha) : A(0);
  const A inv = A(1) / total, inv1 = hard > A(0) ? A(1) / total1 : A(0);
  const A spread = rest && left > A(0) ? share / left : A(0);
  const A factor = c > 1 ? static_cast<A>(c) / static_cast<A>(c - 1) : A(1);
  // P_c of the classes without a slot is written with the row, that of a slot by its thread
  auto put = [&](int i, A v, A want, bool spread_it) {
    const A e = Exp2((v - high) * scale);
    const A q = e * inv;
    if (spread_it) want = spread * (again ? Exp2((v - rest_high) * scale) : e);
    A g = soft > A(0) ? soft * temp * (q - want) : A(0);
    A h = soft > A(0) ? soft * q * (A(1) - q) : A(0);
    if (hard > A(0)) {
      const A q1 = Exp2((v - high) * scale1) * inv1;
      g += hard * (q1 - (i == y ? A(1) : A(0)));
      h += hard * q1 * (A(1) - q1);
    }
    if (grad) grad[i * gs] = static_cast<O>(g * w);
    if (hess) hess[i * hs] = static_cast<O>(h * factor * w);
  };
  for (int i = tid; i < c; i += kBlock)
    if (!(mark[i >> 5] >> (i & 31) & 1u)) put(i, static_cast<A>(z[i * zs]), A(0), true);
  if (cls >= 0) put(cls, z_slot, p, false);
}

// ------------------------------------------------------------------ distillation, few classes
/*!
 * The threads that share a row. kAcross: a class's rows stand next to each other in memory
 * (a booster's scores), so neighbouring threads are neighbouring rows, and a row's L threads
 * are R apart; otherwise a row's threads are L neighbours. Thread l of a row holds the
 * classes e * L + l. R * L = 256. kAcross of one thread a row (kAlone) shares nothing, and its
 * classes are the same for all threads, so that their addresses are scalar arithmetic.
 */
enum TeamKind { kNeighbours, kAcross, kAlone };
template <TeamKind kKind> struct Team {
  int L, R, l, r;
  __device__ explicit Team(int lanes) {
    L = kKind == kAlone ? 1 : lanes;
    R = 256 / L;
    l = kKind == kAlone ? 0 : kKind == kAcross ? threadIdx.x / R : threadIdx.x % L;
    r = kKind == kNeighbours ? threadIdx.x / L : threadIdx.x % R;
  }
  /*! of one thread a row nothing is shared */
  __device__ void Sync() const {
    if (kKind != kAlone) __syncthreads();
  }
  /*! whether v holds for a thread that this one has to keep step with */
  __device__ bool Any(bool v) const { return kKind == kAlone ? v : __syncthreads_or(v); }
  template <typename A, typename F> __device__ A Reduce(A v, A* lds, const F& f) const {
    if (kKind == kAlone) return v;
    if (kKind == kAcross) {
      __syncthreads();
      lds[threadIdx.x] = v;
      __syncthreads();
      v = lds[r];
      for (int i = 1; i < L; ++i) v = f(v, lds[i * R + r]);
      return v;
    }
    for (int d = L / 2; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
    return v;
  }
  template <typename A> __device__ A Sum(A v, A* lds) const {
    return Reduce(v, lds, [](A a, A b) { return a + b; });
  }
  template <typename A> __device__ A Max(A v, A* lds) const {
    return Reduce(v, lds, [](A a, A b) { return class_ops::Max(a, b); });
  }
};

template <typename A>
using Word = std::conditional_t<std::is_same_v<A, double>, unsigned long long, unsigned int>;
__device__ __forceinline__ unsigned int ToBits(float v) { return __float_as_uint(v); }
__device__ __forceinline__ unsigned long long ToBits(double v) { return __double_as_longlong(v); }
__device__ __forceinline__ float FromBits(unsigned int v) { return __uint_as_float(v); }
__device__ __forceinline__ double FromBits(unsigned long long v) { return __longlong_as_double(v); }

/*! more than 32 KiB of dynamic LDS has to be asked for */
template <typename F> void AllowLds(F* kernel, size_t bytes) {
  if (bytes > 32768)
    OPS_HIP_OK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(bytes)));
}

/*!
 * Up to E * L classes: a row is read once and stays in its threads' registers. What the
 * teacher wants of each class is a table in LDS, one word a class: first the lowest slot that
 * names the class (with the sign bit set, kNone: none), then that slot's probability.
 * Everything is held as wide as the scores' statistics, 64 bits for float64 scores, whose 32-bit
 * gradients are then off by hardly more than their own rounding; in 32 bits they were off by five
 * times as much (2.8e-7 of the largest), in 82 us where this takes 96. kLoss: whether the loss is
 * among what may be asked for. Of float64 scores it has a launch of its own, as it needs the
 * exponentials in all of 64 bits, which cost a gradient 123 us. Bound by the arithmetic of 64 bits
 * beside memory: two million rows of seven float64 classes with labels, weights and hessians 96
 * us, 3.2 TB/s of what has to move.
 */
template <typename T, bool kLoss, int E, TeamKind kKind>
__global__ void __launch_bounds__(256) k_distill_tile(LGBM_DistillArgs a, double by, int lanes) {
  using A = Acc<T>;
  using S = A;
  using O = Out<T>;
  using W = Word<S>;
  constexpr W kNone = ~W{0}, kSlot = W{1} << (sizeof(W) * 8 - 1);
  extern __shared__ unsigned long long tile_lds[];
  W* want = reinterpret_cast<W*>(tile_lds);  // R * classes
  __shared__ A red_high[kKind == kAcross ? 256 : 1];
  __shared__ S red[kKind == kAcross ? 256 : 1];
  __shared__ double red_top[kKind == kAcross ? 256 : 1];
  const Team<kKind> team(lanes);
  const int c = a.classes, k = a.k, L = team.L, R = team.R;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * R;
  const int64_t row = first + team.r;
  const bool there = row < a.rows;
  // of a strided array, the place of this row: the workgroup's by scalar arithmetic
  auto at_row = [&](const LGBM_Array& v) {
    const int64_t step = v.stride[0];
    const int64_t more = step == static_cast<int>(step)
                             ? static_cast<int64_t>(team.r) * static_cast<int>(step)
                             : team.r * step;
    return first * step + more;
  };
  auto place = [&](int cls) {
    return kKind == kNeighbours ? team.r * c + cls : cls * R + team.r;
  };

  const S w = !there ? S(0) : a.weight.data ? LoadFloat<S>(a.weight, at_row(a.weight))
                                            : S(1);
  const T* x = static_cast<const T*>(a.scores.data) + at_row(a.scores);
  auto score = [&](int cls) { return static_cast<A>(x[cls * a.scores.stride[1]]); };
  A z[E];  // not kept beyond the exponentials: the few that need a score later read it again
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int cls = e * L + team.l;
    z[e] = there && cls < c ? score(cls) : NegInf<A>();
    if (cls < c) want[place(cls)] = kNone;
  }
  // whatever the row's weight is, all that is read of it is asked for here at once
  const bool rest = a.teacher_rest.data != nullptr, hard_term = a.alpha < 1.0;
  const int label = hard_term && there ? LoadClass(a.label, at_row(a.label), c) : -1;
  const double rest_read = rest && there ? LoadFloat<double>(a.teacher_rest, at_row(a.teacher_rest))
                                         : 0.0;
  team.Sync();
  const S temp = static_cast<S>(a.temperature), alpha = static_cast<S>(a.alpha);
  const A scale = static_cast<A>(by), scale1 = static_cast<A>(kLog2e);
  auto exp2_of = [](S v) {
    if constexpr (std::is_same_v<S, double> && !kLoss) return ShortExp2(v);
    else return Exp2(v);
  };
  const bool teach = w != S(0) && alpha > S(0);
  // the slots of this thread: the first few stay in registers, read before any is looked at
  constexpr int kHeld = 4;
  int held_cls[kHeld];
  double held_logit[kHeld];
  const int64_t class_row = at_row(a.teacher_class), logit_row = at_row(a.teacher_logit);
  auto load_class = [&](int j) {
    return LoadClass(a.teacher_class, class_row + j * a.teacher_class.stride[1], c);
  };
  auto load_logit = [&](int j) {
    return LoadFloat<double>(a.teacher_logit, logit_row + j * a.teacher_logit.stride[1]);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int j = team.l + i * L;
    const bool read = there && j < k;
    held_cls[i] = read ? load_class(j) : -1;
    held_logit[i] = read ? load_logit(j) : 0.0;
  }
  if (!teach) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held_cls[i] = -1;
  }
  if (w == S(0)) {
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] = NegInf<A>();
  }
  // f(slot, class, logit) of all of them
  auto all_slots = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (held_cls[i] >= 0) f(team.l + i * L, held_cls[i], held_logit[i]);
    if (!teach) return;
    for (int j = team.l + kHeld * L; j < k; j += L) {
      const int cls = load_class(j);
      if (cls >= 0) f(j, cls, load_logit(j));
    }
  };
  all_slots([&](int j, int cls, double) {
    atomicMin(&want[place(cls)], kSlot | static_cast<W>(j));
  });
  A high = NegInf<A>();
#pragma unroll
  for (int e = 0; e < E; ++e) high = Max(high, z[e]);
  high = team.Max(high, red_high);
  if (!(high > NegInf<A>())) high = A(0);
  team.Sync();

  // the teacher's distribution, in logarithms to base two
  auto for_slots = [&](auto&& f) {  // the slots that count, with their place in the table
    all_slots([&](int j, int cls, double t) {
      W* at = &want[place(cls)];
      if (*at == (kSlot | static_cast<W>(j))) f(cls, t, at);
    });
  };
  double t_top = NegInf<double>();
  for_slots([&](int, double t, W*) { t_top = Max(t_top, t); });
  const TeacherScale teacher(team.Max(t_top, red_top), rest && teach ? rest_read : NegInf<double>(),
                             by);
  S t_sum = 0;
  for_slots([&](int, double t, W*) { t_sum += exp2_of(teacher.template Slot<S>(t)); });
  const S log_u_rest = teacher.template Rest<S>(), u_rest = exp2_of(log_u_rest);
  t_sum = team.Sum(t_sum, red) + u_rest;
  // the largest weight is one, so a sum of zero is a row without a teacher
  const bool taught = teach && !(t_sum == S(0));
  const S t_inv = taught ? S(1) / t_sum : S(0);
  const S share = u_rest * t_inv;
  // the table's slots give way to their probabilities; every class has one such slot. Where the
  // loss is taken from them too, that is where the student's sums are known.
  auto put_slots = [&](auto&& f) {
    team.Sync();
    for_slots([&](int cls, double t, W* at) {
      const S log_u = teacher.template Slot<S>(t);
      const S p = taught ? exp2_of(log_u) * t_inv : S(0);
      f(cls, p, log_u);
      *at = ToBits(p) & ~kSlot;
    });
  };
  if constexpr (!kLoss) {
    put_slots([](int, S, S) {});
    team.Sync();
  }

  // the student's: the classes without a slot are summed on their own
  const bool two = hard_term && scale != scale1;
  S ez[E], e1[E], left = 0, named = 0, total1 = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int cls = e * L + team.l;
    ez[e] = exp2_of((z[e] - high) * scale);
    if (cls < c && want[place(cls)] != kNone) named += ez[e];
    else left += ez[e];
    e1[e] = two ? exp2_of((z[e] - high) * scale1) : ez[e];
    total1 += e1[e];
  }
  left = team.Sum(left, red);
  const S total = left + team.Sum(named, red);
  total1 = two ? team.Sum(total1, red) : total;
  A rest_high = high;
  const bool again = rest && w != S(0) && left < SmallRest<S>();
  if (team.Any(again)) {
    A own = NegInf<A>();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int cls = e * L + team.l;
      if (again && cls < c && want[place(cls)] == kNone) own = Max(own, score(cls));
    }
    own = team.Max(own, red_high);
    const bool able = again && own > NegInf<A>();
    S sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int cls = e * L + team.l;
      if (able && cls < c && want[place(cls)] == kNone)
        sum += exp2_of((score(cls) - own) * scale);
    }
    sum = team.Sum(sum, red);
    if (able) {
      left = sum;
      rest_high = own;
    }
  }
  const bool live = w != S(0) && !(total == S(0));  // otherwise every class is masked
  const int y = live ? label : -1;

  if constexpr (kLoss) {
    double kl = 0;
    const S log_both = Log2(total) - Log2(t_sum);
    put_slots([&](int cls, S p, S log_u) {
      if (a.loss.data && !(p == S(0)))
        kl += Divergence(p, log_u + log_both, static_cast<double>(score(cls)) - high,
                         a.temperature);
    });
    if (a.loss.data) {
      kl = team.Sum(kl, red_top);
      if (there && team.l == 0) {
        double v = 0;
        if (live) {
          if (rest && !(share == S(0)))
            kl += Divergence(share, log_u_rest - Log2(left) + log_both,
                             static_cast<double>(rest_high) - high, a.temperature);
          if (taught) v = a.alpha * a.temperature * a.temperature * kl;
          if (y >= 0)
            v += (1.0 - a.alpha) * (Log2(total1) * kLn2 - (static_cast<double>(score(y)) - high));
          v *= w;
        }
        StoreFloat(a.loss, at_row(a.loss), v);
      }
    }
    team.Sync();
  }
  if (!a.gradient.data && !a.hessian.data) return;
  const S soft = taught ? alpha : S(0), hard = y >= 0 ? static_cast<S>(1.0 - a.alpha) : S(0);
  const S inv = S(1) / total, inv1 = hard > S(0) ? S(1) / total1 : S(0);
  const S spread = rest && left > S(0) ? share / left : S(0);
  const S factor = c > 1 ? static_cast<S>(c) / static_cast<S>(c - 1) : S(1);
  const bool moved = rest_high != high;
  O* grad = static_cast<O*>(a.gradient.data) + (a.gradient.data ? at_row(a.gradient) : 0);
  O* hess = static_cast<O*>(a.hessian.data) + (a.hessian.data ? at_row(a.hessian) : 0);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int cls = e * L + team.l;
    if (!there || cls >= c) continue;
    S g = 0, h = 0;
    if (live) {
      const S q = ez[e] * inv;
      if (soft > S(0)) {
        const W bits = want[place(cls)];
        S p = FromBits(bits);
        if (bits == kNone) {
          p = S(0);
          const S e_rest = moved ? exp2_of((score(cls) - rest_high) * scale) : ez[e];
          if (spread > S(0)) p = spread * e_rest;
          else if (spread != spread) p = spread;
        }
        g = soft * temp * (q - p);
        h = soft * q * (S(1) - q);
      }
      if (hard > S(0)) {
        const S q1 = e1[e] * inv1;
        g += hard * (q1 - (cls == y ? S(1) : S(0)));
        h += hard * q1 * (S(1) - q1);
      }
    }
    if (a.gradient.data) grad[cls * a.gradient.stride[1]] = static_cast<O>(g * w);
    if (a.hessian.data) hess[cls * a.hessian.stride[1]] = static_cast<O>(h * factor * w);
  }
}

// ------------------------------------------------------------------ rows of many classes
using Words = uint32_t __attribute__((ext_vector_type(4)));

/*! sixteen bytes of a row: as many elements as they hold */
template <typename T> struct Chunk {
  static constexpr int kSize = 16 / sizeof(T);
  T v[kSize];
};

/*!
 * A row's workgroup: its threads, and the chunks that each holds in registers. kMore: a row
 * may have more than these; then up to kLdsChunks more a thread stand in LDS, as far as it
 * reaches, and what is left is read from memory in each pass.
 */
template <int kBlock, int kCached, bool kMore = false> struct RowShape {
  static constexpr int block = kBlock, cached = kCached;
  static constexpr bool more = kMore;
};
constexpr int kLdsChunks = 8;

/*!
 * A row whose classes stand next to each other, as its workgroup holds it: one chunk a thread
 * in turn, and the classes after the last whole chunk one a thread. Chunks are read at their
 * elements' alignment: the hardware splits what crosses a line. kAnew: each pass counts its chunks
 * anew, where their numbers, kept from one pass to the next, are the registers too many.
 */
template <typename T, typename Shape, bool kAnew = false> struct RowOf {
  static constexpr int kSize = Chunk<T>::kSize, kBlock = Shape::block, kCached = Shape::cached;
  using A = Acc<T>;
  const T* x;
  int chunks, tail;  // whole chunks, and the class of this thread after them (-1: none)
  int in_lds;        // chunks a thread in LDS
  Words* lds;
  A tail_value;
  Words raw[kCached];

  __device__ __forceinline__ RowOf(const T* row, int classes, Words* lds_space, int lds_chunks)
      : x(row), chunks(classes / kSize), in_lds(lds_chunks), lds(lds_space) {
    tail = chunks * kSize + static_cast<int>(threadIdx.x);
    if (tail >= classes) tail = -1;
  }
  __device__ __forceinline__ Words Read(int chunk) const {
    Words got;
    __builtin_memcpy(&got, x + static_cast<int64_t>(chunk) * kSize, sizeof(got));
    return got;
  }
  __device__ __forceinline__ void Load() {
#pragma unroll
    for (int n = 0; n < kCached; ++n) {
      const int chunk = n * kBlock + threadIdx.x;
      raw[n] = chunk < chunks ? Read(chunk) : Words{};
    }
    tail_value = tail >= 0 ? static_cast<A>(x[tail]) : A(0);
    if constexpr (Shape::more) {  // every thread reads back what it wrote itself
#pragma unroll 4
      for (int n = 0; n < in_lds; ++n) {
        const int chunk = (kCached + n) * kBlock + threadIdx.x;
        if (chunk < chunks) lds[n * kBlock + threadIdx.x] = Read(chunk);
      }
    }
  }
  template <typename F>
  static __device__ __forceinline__ void Give(const Words& words, int chunk, const F& f) {
    Chunk<T> got;
    __builtin_memcpy(&got, &words, sizeof(got));
    A v[kSize];
#pragma unroll
    for (int i = 0; i < kSize; ++i) v[i] = static_cast<A>(got.v[i]);
    f(chunk * kSize, v, words);
  }
  /*! f(first class, values) of what this thread holds, kSize or one at a time */
  template <typename F> __device__ __forceinline__ void EachHeld(const F& f) {
    int own = threadIdx.x;
    if (kAnew) asm volatile("" : "+v"(own));
#pragma unroll
    for (int n = 0; n < kCached; ++n) {
      // what a pass makes of the row is not kept for the next: the compiler would hold its
      // conversions and exponentials in registers that are not there
      asm volatile("" : "+v"(raw[n]));
      const int chunk = n * kBlock + own;
      if (chunk < chunks) Give(raw[n], chunk, f);
    }
    if constexpr (Shape::more) {
      for (int n = 0; n < in_lds; ++n) {
        const int chunk = (kCached + n) * kBlock + own;
        if (chunk < chunks) Give(lds[n * kBlock + own], chunk, f);
      }
    }
    if (tail >= 0) {
      const A v[1] = {tail_value};
      f(tail, v);
    }
  }
  /*! f(first class, values) of what this thread reads each time */
  template <typename F> __device__ __forceinline__ void EachMore(const F& f) const {
    if constexpr (Shape::more) {
#pragma unroll 4
      for (int chunk = (kCached + in_lds) * kBlock + threadIdx.x; chunk < chunks; chunk += kBlock)
        Give(Read(chunk), chunk, f);
    }
  }
  template <typename F> __device__ __forceinline__ void Each(const F& f) {
    EachHeld(f);
    EachMore(f);
  }
};

template <typename V> constexpr int kSizeOf = std::extent_v<std::remove_reference_t<V>>;

/*! kCount sums over the workgroup at once; `lds` has kCount * waves places */
template <int kBlock, int kCount, typename A>
__device__ __forceinline__ void BlockSums(A (&v)[kCount], A* lds) {
  constexpr int kWaves = kBlock / kWave;
#pragma unroll
  for (int n = 0; n < kCount; ++n) {
    v[n] = WaveSum(v[n]);
    if (threadIdx.x % kWave == 0) lds[n * kWaves + threadIdx.x / kWave] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kCount; ++n) {
    v[n] = lds[n * kWaves];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v[n] += lds[n * kWaves + i];
  }
}

/*!
 * One workgroup a row of many classes: read once, as far as its registers reach, then the
 * maximum, the sums and the gradients from there. Every thread writes its classes as if they
 * had no slot; after a barrier the slots' threads write theirs over that, which leaves the
 * write pass without a test. Bound by memory where the row fits (8192 x 32768 bfloat16 with
 * the loss 227 us, 4.7 TB/s; the loss alone of 2048 x 32768 float32 49 us, 5.5 TB/s), by
 * arithmetic that does not overlap the loads where labels have a temperature of their own (3001 x
 * 20011 float16 42 us, 2.9 TB/s, the vector units busy for 61% of it), by reading a third of the
 * row twice where it does not fit (501 x 131077 float32 142 us, 3.7 TB/s).
 */
template <typename T, typename Shape, bool kHessian>
__global__ void __launch_bounds__(Shape::block, Shape::cached >= 12 ? 4 : 1)
k_distill_row(LGBM_DistillArgs a, double by, int lds_chunks) {
  using A = Acc<T>;
  using O = Out<T>;
  using Row = RowOf<T, Shape, (Shape::block > 256)>;
  constexpr int kBlock = Shape::block, kWaves = kBlock / kWave;
  extern __shared__ Words row_lds[];  // the chunks, then the marks
  uint32_t* mark = reinterpret_cast<uint32_t*>(row_lds + lds_chunks * Shape::block);
  __shared__ int s_cls[kMaxTop];
  __shared__ A s_max[2][kWaves], s_sum[4 * kWaves], s_more[2][kWaves];
  __shared__ double s_top[kWaves];
  __shared__ int s_dup;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, c = a.classes, k = a.k;
  O* grad = a.gradient.data ? static_cast<O*>(a.gradient.data) + row * a.gradient.stride[0]
                            : nullptr;
  O* hess = kHessian ? static_cast<O*>(a.hessian.data) + row * a.hessian.stride[0] : nullptr;
  const A w = a.weight.data ? LoadFloat<A>(a.weight, row * a.weight.stride[0]) : A(1);
  auto put_zeros = [&] {
    if (a.loss.data && tid == 0) StoreFloat(a.loss, row * a.loss.stride[0], A(0));
    for (int i = tid; i < c; i += kBlock) {
      if (grad) grad[i] = static_cast<O>(0.0f);
      if (kHessian) hess[i] = static_cast<O>(0.0f);
    }
  };
  if (w == A(0)) {
    put_zeros();
    return;
  }
  Row z(static_cast<const T*>(a.scores.data) + row * a.scores.stride[0], c, row_lds, lds_chunks);
  z.Load();
  for (int i = tid; i < (c + 31) / 32; i += kBlock) mark[i] = 0;
  if (tid == 0) s_dup = 0;

  // the slots, one a thread
  const A temp = static_cast<A>(a.temperature), alpha = static_cast<A>(a.alpha);
  const A scale = static_cast<A>(by), scale1 = static_cast<A>(kLog2e);
  const bool rest = a.teacher_rest.data != nullptr, hard_term = a.alpha < 1.0;
  const bool two = hard_term && scale != scale1;  // a softmax at another temperature
  int cls = -1;
  A logit = NegInf<A>(), z_slot = NegInf<A>();
  const int64_t logit_at = row * a.teacher_logit.stride[0] + tid * a.teacher_logit.stride[1];
  if (tid < k) {
    cls = LoadClass(a.teacher_class,
                    row * a.teacher_class.stride[0] + tid * a.teacher_class.stride[1], c);
    if (cls >= 0) {
      logit = LoadFloat<A>(a.teacher_logit, logit_at);
      z_slot = static_cast<A>(z.x[cls]);
    }
    s_cls[tid] = cls;
  }
  const int64_t rest_at = row * a.teacher_rest.stride[0];
  A r = rest ? LoadFloat<A>(a.teacher_rest, rest_at) : NegInf<A>();
  const int label = hard_term ? LoadClass(a.label, row * a.label.stride[0], c) : -1;
  const A z_label = label >= 0 ? static_cast<A>(z.x[label]) : A(0);
  __syncthreads();
  if (cls >= 0 && (atomicOr(&mark[cls >> 5], 1u << (cls & 31)) >> (cls & 31) & 1u)) s_dup = 1;

  auto bits_of = [&](int base, int size) {  // those of a chunk stand in one word
    return mark[base >> 5] >> (base & 31) & ((1u << size) - 1u);
  };
  // the sums of a chunk's exponentials of the classes without a slot, and of all at T = 1
  auto add_chunk = [&](int base, const auto& v, A from, A& rest_sum, A& all_sum) {
    constexpr int kSize = kSizeOf<decltype(v)>;
    const uint32_t bits = bits_of(base, kSize);
    A e[kSize], sum = 0;
#pragma unroll
    for (int i = 0; i < kSize; ++i) e[i] = Exp2((v[i] - from) * scale);
    if (bits != 0) {
#pragma unroll
      for (int i = 0; i < kSize; ++i) e[i] = bits >> i & 1u ? A(0) : e[i];
    }
#pragma unroll
    for (int i = 0; i < kSize; ++i) sum += e[i];
    rest_sum += sum;
    if (two) {
      sum = 0;
#pragma unroll
      for (int i = 0; i < kSize; ++i) sum += Exp2((v[i] - from) * scale1);
      all_sum += sum;
    }
  };
  A high = NegInf<A>();
  z.EachHeld([&](int, const auto& v, auto...) {
#pragma unroll
    for (int i = 0; i < kSizeOf<decltype(v)>; ++i) high = Max(high, v[i]);
  });
  // what is not held is read once for both, its sums against this thread's maximum so far
  A more_high = NegInf<A>(), more_left = 0, more_total1 = 0;
  if constexpr (Shape::more) {
    __syncthreads();  // the marks
    z.EachMore([&](int base, const auto& v, auto...) {
      A top = v[0];
#pragma unroll
      for (int i = 1; i < kSizeOf<decltype(v)>; ++i) top = Max(top, v[i]);
      if (top > more_high) {
        more_left *= Exp2((more_high - top) * scale);
        if (two) more_total1 *= Exp2((more_high - top) * scale1);
        more_high = top;
      }
      add_chunk(base, v, more_high > NegInf<A>() ? more_high : A(0), more_left, more_total1);
    });
    high = Max(high, more_high);
  }
  const A own_high = more_high;
  high = WaveMax(high);
  A t_high = WaveMax(logit);
  if (tid % kWave == 0) {
    s_max[0][tid / kWave] = high;
    s_max[1][tid / kWave] = t_high;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    high = Max(high, s_max[0][i]);
    t_high = Max(t_high, s_max[1][i]);
  }
  if (s_dup) {  // the first slot of a class counts
    for (int i = 0; i < tid && tid < k; ++i)
      if (s_cls[i] == cls) cls = -1;
    if (cls < 0) logit = z_slot = NegInf<A>();
    t_high = BlockMax<kBlock>(logit, s_more[0]);
  }
  if (!(high > NegInf<A>())) high = A(0);
  // what 32 bits hold is exact in them; what they do not is read again
  double t_top = t_high, t_own = logit, t_rest = r;
  if (a.teacher_logit.type == C_API_DTYPE_FLOAT64) {
    t_own = cls >= 0 ? At<double>(a.teacher_logit, logit_at) : NegInf<double>();
    t_top = BlockMax<kBlock>(t_own, s_top);
  }
  if (rest && a.teacher_rest.type == C_API_DTYPE_FLOAT64)
    t_rest = At<double>(a.teacher_rest, rest_at);
  const TeacherScale teacher(t_top, t_rest, by);
  const A log_u = teacher.template Slot<A>(t_own), log_u_rest = teacher.template Rest<A>();

  A left = 0, total1 = 0;
  z.EachHeld([&](int base, const auto& v, auto...) {
    add_chunk(base, v, high, left, total1);
  });
  if constexpr (Shape::more) {
    if (own_high > NegInf<A>() || more_left != A(0)) {
      left += more_left * Exp2((own_high > NegInf<A>() ? own_high - high : A(0)) * scale);
      if (two)
        total1 += more_total1 * Exp2((own_high > NegInf<A>() ? own_high - high : A(0)) * scale1);
    }
  }
  A sums[4] = {left, cls >= 0 ? Exp2((z_slot - high) * scale) : A(0),
               Exp2(log_u), total1};
  const A u = sums[2];
  BlockSums<kBlock>(sums, s_sum);
  left = sums[0];
  const A total = left + sums[1];
  total1 = two ? sums[3] : total;
  if (total == A(0)) {  // every class is masked
    put_zeros();
    return;
  }
  const A u_rest = Exp2(log_u_rest);
  const A t_sum = sums[2] + u_rest;
  // the largest weight is one, so a sum of zero is a row without a teacher
  const bool taught = alpha > A(0) && !(t_sum == A(0));
  const A t_log = Log2(t_sum), log_total = Log2(total);
  const A p = taught ? u / t_sum : A(0), share = taught ? u_rest / t_sum : A(0);
  A rest_high = high;
  if (rest && left < SmallRest<A>()) {  // seldom, so from memory in a plain loop
    A own = NegInf<A>();
    for (int i = tid; i < c; i += kBlock)
      if (!bits_of(i, 1)) own = Max(own, static_cast<A>(z.x[i]));
    own = BlockMax<kBlock>(own, s_more[0]);
    if (own > NegInf<A>()) {
      rest_high = own;
      left = 0;
      for (int i = tid; i < c; i += kBlock)
        if (!bits_of(i, 1)) left += Exp2((static_cast<A>(z.x[i]) - own) * scale);
      left = BlockSum<kBlock>(left, s_more[1]);
    }
  }

  if (a.loss.data) {
    double kl = 0;
    if (tid - tid % kWave < k) {  // the waves with slots
      if (cls >= 0 && !(p == A(0)))
        kl = Divergence(p, log_u - t_log + log_total, static_cast<double>(z_slot) - high,
                        a.temperature);
      kl = WaveSum(kl);
    }
    if (tid % kWave == 0) s_top[tid / kWave] = kl;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int i = 1; i < kWaves; ++i) kl += s_top[i];
      if (rest && !(share == A(0)))
        kl += Divergence(share, log_u_rest - t_log - Log2(left) + log_total,
                         static_cast<double>(rest_high) - high, a.temperature);
      double v = taught ? a.alpha * a.temperature * a.temperature * kl : 0.0;
      if (label >= 0)
        v += (1.0 - a.alpha) * (Log2(total1) * kLn2 - (static_cast<double>(z_label) - high));
      StoreFloat(a.loss, row * a.loss.stride[0], v * w);
    }
  }
  if (!grad && !hess) return;
  const A soft = taught ? alpha : A(0), hard = label >= 0 ? static_cast<A>(1.0 - a.alpha) : A(0);
  const A inv = A(1) / total, inv1 = hard > A(0) ? A(1) / total1 : A(0);
  const A spread = rest && left > A(0) ? share / left : A(0);
  const A factor = c > 1 ? static_cast<A>(c) / static_cast<A>(c - 1) : A(1);
  // a class without a slot: its gradient is one factor of each exponential
  const bool moved = rest_high != high;
  const A each = w * soft * temp;  // 0 where there is no teacher, whose inv may be anything
  A coef = soft > A(0) ? each * (moved ? inv : inv - spread) : A(0);
  const A coef1 = hard > A(0) ? w * hard * inv1 : A(0);
  if (!two) coef += coef1;
  if (grad) {
    if (moved) {
      const A coef_rest = soft > A(0) ? -each * spread : A(0);
      z.Each([&](int base, const auto& v, auto...) {
#pragma unroll
        for (int i = 0; i < kSizeOf<decltype(v)>; ++i) {
          A g = coef * Exp2((v[i] - high) * scale);
          if (two) g = Fma(coef1, Exp2((v[i] - high) * scale1), g);
          grad[base + i] = static_cast<O>(Fma(coef_rest, Exp2((v[i] - rest_high) * scale), g));
        }
      });
    } else {
      z.Each([&](int base, const auto& v, auto...) {
        constexpr int kSize = kSizeOf<decltype(v)>;
        O g[kSize];
        if (two) {
#pragma unroll
          for (int i = 0; i < kSize; ++i)
            g[i] = static_cast<O>(Fma(coef1, Exp2((v[i] - high) * scale1),
                                      coef * Exp2((v[i] - high) * scale)));
        } else {
#pragma unroll
          for (int i = 0; i < kSize; ++i)
            g[i] = static_cast<O>(coef * Exp2((v[i] - high) * scale));
        }
        __builtin_memcpy(grad + base, &g, sizeof(g));
      });
    }
  }
  if (kHessian) {
    z.Each([&](int base, const auto& v, auto...) {
#pragma unroll
      for (int i = 0; i < kSizeOf<decltype(v)>; ++i) {
        const A q = Exp2((v[i] - high) * scale) * inv;
        A h = soft > A(0) ? soft * q * (A(1) - q) : A(0);
        if (hard > A(0)) {
          const A q1 = Exp2((v[i] - high) * scale1) * inv1;
          h += hard * q1 * (A(1) - q1);
        }
        hess[base + i] = static_cast<O>(h * factor * w);
      }
    });
  }
  if (!grad) return;
  __syncthreads();
  auto put = [&](int at, A v, A p, A from, bool spread_it) {
    const A q = Exp2((v - high) * scale) * inv;
    if (spread_it) p = spread == A(0) ? A(0) : spread * Exp2((v - from) * scale);
    A g = soft > A(0) ? soft * temp * (q - p) : A(0);
    if (hard > A(0))
      g += hard * (Exp2((v - high) * scale1) * inv1 - (at == label ? A(1) : A(0)));
    grad[at] = static_cast<O>(g * w);
  };
  if (cls >= 0) put(cls, z_slot, p, high, false);
  // the label's class, where it has no slot
  if (tid == 0 && label >= 0 && !bits_of(label, 1)) put(label, z_label, A(0), rest_high, true);
}

// ------------------------------------------------------------------ top logits, any strides
template <typename T> using Key = std::conditional_t<std::is_same_v<T, double>, uint64_t, uint32_t>;

/*!
 * The `take` largest of a digit's counts: the digit at which the count from the largest
 * digit down reaches `take`, and how many of it are still to be taken. One wave's work.
 */
__device__ __forceinline__ void PickDigit(const int* hist, int take, int* digit, int* left) {
  // lane l holds the four digits 255-4l .. 252-4l, largest first
  const int lane = threadIdx.x % kWave;
  int own[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += own[i] = hist[255 - 4 * lane - i];
  int before = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(before, d);
    if (lane >= d) before += o;
  }
  before -= sum;
  if (before < take && take <= before + sum) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < take && take <= before + own[i]) {
        *digit = 255 - 4 * lane - i;
        *left = take - before;
      }
      before += own[i];
    }
  }
}

/*!
 * One workgroup a row, in any strides and with any ties: the k-th largest key is found
 * digit by digit (eight bits a pass, counted in LDS), its equals are cut by class the same
 * way, and what is chosen is put in order by counting how many precede it. Eight to fourteen
 * passes over memory: 4096 x 50021 bfloat16, k = 64, of every second column 2507 us; of
 * neighbours, by the rows' kernel, 129. Rows of many equal scores and float64 rows of more than
 * 512 classes come here.
 */
template <typename T, int kBlock>
__device__ __forceinline__ void TopAny(const LGBM_TopLogitsArgs& a, int64_t row) {
  using A = Acc<T>;
  using K = Key<T>;
  __shared__ int hist[256];
  __shared__ int s_digit, s_left, s_count;
  __shared__ K s_key[kMaxTop];
  __shared__ int s_cls[kMaxTop];
  __shared__ A s_red[2][kBlock / kWave];
  const int tid = threadIdx.x, c = a.classes;
  const T* x = static_cast<const T*>(a.scores.data) + row * a.scores.stride[0];
  const int64_t xs = a.scores.stride[1];
  auto value = [&](int i) { return static_cast<A>(x[i * xs]); };

  int valid = 0;
  for (int i = tid; i < c; i += kBlock) valid += KeyOf(value(i)) != 0;
  if (tid == 0) s_count = 0;
  __syncthreads();
  if (valid) atomicAdd(&s_count, valid);
  __syncthreads();
  valid = s_count;
  const int take = min(a.k, valid);
  __syncthreads();
  if (tid == 0) s_count = 0;

  K edge = 0;   // the take-th largest key
  int cut = c;  // of the keys equal to it, the classes below this are chosen
  if (take > 0) {
    int left = take;
    for (int shift = sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kBlock) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < c; i += kBlock) {
        const K key = KeyOf(value(i));
        // the digits above are the edge's; the last shift is all of the key
        const bool same = shift == sizeof(K) * 8 - 8 ||
                          (key >> (shift + 8)) == (edge >> (shift + 8));
        if (key != 0 && same) atomicAdd(&hist[static_cast<int>(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < kWave) PickDigit(hist, left, &s_digit, &s_left);
      __syncthreads();
      edge |= static_cast<K>(s_digit) << shift;
      left = s_left;
    }
    // `left` of the classes whose key is the edge: the lowest, that is the largest of ~class
    int high = 0;
    for (int shift = 16; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += kBlock) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < c; i += kBlock) {
        const int turned = 0xffffff - i;
        if (KeyOf(value(i)) == edge &&
            (shift == 16 || (turned >> (shift + 8)) == (high >> (shift + 8))))
          atomicAdd(&hist[(turned >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < kWave) PickDigit(hist, left, &s_digit, &s_left);
      __syncthreads();
      high |= s_digit << shift;
      left = s_left;
    }
    cut = 0xffffff - high + 1;
  }
  __syncthreads();
  // what is chosen, and the largest and the sum of what is not
  A other = NegInf<A>();
  for (int i = tid; i < c; i += kBlock) {
    const A v = value(i);
    const K key = KeyOf(v);
    if (key == 0) continue;
    if (take > 0 && (key > edge || (key == edge && i < cut))) {
      const int at = atomicAdd(&s_count, 1);
      s_key[at] = key;
      s_cls[at] = i;
    } else {
      other = Max(other, v);
    }
  }
  __syncthreads();
  if (tid < take) {
    const K key = s_key[tid];
    const int cls = s_cls[tid];
    int rank = 0;
    for (int i = 0; i < take; ++i) rank += s_key[i] > key || (s_key[i] == key && s_cls[i] < cls);
    static_cast<int32_t*>(a.top_class.data)[row * a.top_class.stride[0] +
                                            rank * a.top_class.stride[1]] = cls;
    static_cast<T*>(a.top_logit.data)[row * a.top_logit.stride[0] + rank * a.top_logit.stride[1]] =
        x[cls * xs];
  } else if (tid < a.k) {
    static_cast<int32_t*>(a.top_class.data)[row * a.top_class.stride[0] +
                                            tid * a.top_class.stride[1]] = -1;
    static_cast<T*>(a.top_logit.data)[row * a.top_logit.stride[0] + tid * a.top_logit.stride[1]] =
        static_cast<T>(-INFINITY);
  }
  if (a.log_rest.data == nullptr) return;
  const A scale = static_cast<A>(kLog2e / a.temperature);
  other = BlockMax<kBlock>(other, s_red[0]);
  A sum = 0;
  if (other > NegInf<A>() && other < static_cast<A>(INFINITY)) {
    for (int i = tid; i < c; i += kBlock) {
      const A v = value(i);
      const K key = KeyOf(v);
      if (key != 0 && !(take > 0 && (key > edge || (key == edge && i < cut))))
        sum += Exp2((v - other) * scale);
    }
    sum = BlockSum<kBlock>(sum, s_red[1]);
  }
  if (tid == 0)
    StoreFloat(a.log_rest, row * a.log_rest.stride[0],
               sum > A(0) ? other / static_cast<A>(a.temperature) + Log2(sum) * static_cast<A>(kLn2)
                          : other);
}

template <typename T, int kBlock>
__global__ void __launch_bounds__(kBlock) k_top_any(LGBM_TopLogitsArgs a) {
  TopAny<T, kBlock>(a, blockIdx.x);
}

// ------------------------------------------------------------------ top logits, few classes
/*!
 * Up to E * L classes, in the registers of their row's threads (Team): k times the largest
 * that is left, by comparison with all others. Of equals the lowest class is met first. Bound
 * by memory for small k (1000000 x 10 float64, k = 4, 34 us, 3.9 TB/s), by the comparisons
 * for larger (400000 x 100 float32, k = 10, 144 us, the vector units busy throughout).
 */
template <typename T, int E, TeamKind kKind>
__global__ void __launch_bounds__(256) k_top_tile(LGBM_TopLogitsArgs a, int lanes) {
  using A = Acc<T>;
  __shared__ A red[256];
  __shared__ int red_cls[256];
  const Team<kKind> team(lanes);
  const int c = a.classes, L = team.L, R = team.R;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * R + team.r;
  const bool there = row < a.rows;
  A z[E];
  const T* x = static_cast<const T*>(a.scores.data) + row * a.scores.stride[0];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int cls = e * L + team.l;
    z[e] = there && cls < c ? static_cast<A>(x[cls * a.scores.stride[1]]) : NegInf<A>();
  }
  uint32_t left = ~0u;  // of this thread's classes
  int32_t* out_class = static_cast<int32_t*>(a.top_class.data) + row * a.top_class.stride[0];
  T* out_logit = static_cast<T*>(a.top_logit.data) + row * a.top_logit.stride[0];
  for (int j = 0; j < a.k; ++j) {
    A best = NegInf<A>();
    int cls = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if ((left >> e & 1u) && z[e] > best) {
        best = z[e];
        cls = e * L + team.l;
      }
    }
    auto other = [&](A v, int o) {
      if (o >= 0 && (cls < 0 || v > best || (v == best && o < cls))) {
        best = v;
        cls = o;
      }
    };
    if (kKind == kAcross) {
      __syncthreads();
      red[threadIdx.x] = best;
      red_cls[threadIdx.x] = cls;
      __syncthreads();
      for (int i = 0; i < L; ++i) other(red[i * R + team.r], red_cls[i * R + team.r]);
    } else if (kKind == kNeighbours) {
      for (int d = L / 2; d > 0; d >>= 1) {
        const A v = __shfl_xor(best, d);
        const int o = __shfl_xor(cls, d);
        other(v, o);
      }
    }
    if (cls >= 0 && (cls & (L - 1)) == team.l) left &= ~(1u << (cls / L));
    if (there && team.l == 0) {
      out_class[j * a.top_class.stride[1]] = cls;
      out_logit[j * a.top_logit.stride[1]] = static_cast<T>(best);
    }
  }
  if (a.log_rest.data == nullptr) return;
  A high = NegInf<A>();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (left >> e & 1u) high = Max(high, z[e]);
  high = team.Max(high, red);
  const A scale = static_cast<A>(kLog2e / a.temperature);
  const bool able = high > NegInf<A>() && high < static_cast<A>(INFINITY);
  A sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (able && (left >> e & 1u) && z[e] > NegInf<A>()) sum += Exp2((z[e] - high) * scale);
  sum = team.Sum(sum, red);
  if (there && team.l == 0)
    StoreFloat(a.log_rest, row * a.log_rest.stride[0],
               sum > A(0) ? high / static_cast<A>(a.temperature) + Log2(sum) * static_cast<A>(kLn2)
                          : high);
}

// ------------------------------------------------------------------ top logits, some classes
/*! a candidate as one number: the larger comes first, and of equal values the lower class */
__device__ __forceinline__ uint64_t Candidate(float v, int cls) {
  return static_cast<uint64_t>(KeyOf(v)) << 32 | ~static_cast<uint32_t>(cls);
}
/*! the same number in every lane, as a scalar */
__device__ __forceinline__ uint32_t Scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t Scalar(uint64_t v) {
  return static_cast<uint64_t>(Scalar(static_cast<uint32_t>(v >> 32))) << 32 |
         Scalar(static_cast<uint32_t>(v));
}
/*! LDS that this wave's lanes wrote is there for its other lanes */
__device__ __forceinline__ void WaveSync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kTurnedRows = 16;

/*!
 * One wave a row of up to E * 64 classes, which its lanes hold: the k-th largest by bisection
 * over the keys between the row's smallest and largest. A step compares what each lane holds
 * with the middle and counts the lanes' answers, without a word between lanes; it ends as
 * soon as the count is k. No wave waits for another. kTurned: the rows of a class stand next
 * to each other, so a workgroup turns sixteen rows in LDS first. Bound by the vector work of
 * some twenty steps and the ranking (300000 x 250 bfloat16, k = 50, 405 us, the vector units busy
 * throughout; k rounds of the largest that is left took 3024).
 */
template <typename T, int E, bool kTurned>
__global__ void __launch_bounds__(256) k_top_wave(LGBM_TopLogitsArgs a) {
  using A = Acc<T>;
  using K = Key<T>;
  constexpr bool kWide = std::is_same_v<T, double>;
  constexpr int kRows = kTurned ? kTurnedRows : 4;
  extern __shared__ unsigned long long turned_lds[];
  __shared__ uint64_t s_list[4][kMaxTop];
  __shared__ int s_cls[kWide ? 4 : 1][kMaxTop];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, c = a.classes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), a.rows - first));
  T* turned = reinterpret_cast<T*>(turned_lds);
  const int step = c | 1;  // of the turned rows: odd, so that they begin in different banks
  if constexpr (kTurned) {
    const int r = threadIdx.x % kRows;
    const T* x = static_cast<const T*>(a.scores.data) + (first + r) * a.scores.stride[0];
    if (r < rows)
#pragma unroll 4
      for (int cls = threadIdx.x / kRows; cls < c; cls += 256 / kRows)
        turned[r * step + cls] = x[cls * a.scores.stride[1]];
    __syncthreads();
  }
  const unsigned long long below = (1ull << lane) - 1;
  const A scale = static_cast<A>(kLog2e / a.temperature);
  for (int i = wave; i < rows; i += 4) {
    const int64_t row = first + i;
    const T* x = static_cast<const T*>(a.scores.data) + row * a.scores.stride[0];
    A z[E], high = NegInf<A>(), low = -NegInf<A>();
    int valid = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int cls = e * kWave + lane;
      z[e] = NegInf<A>();
      if (e * kWave < c) {
        if (cls < c)
          z[e] = kTurned ? static_cast<A>(turned[i * step + cls])
                         : static_cast<A>(x[cls * a.scores.stride[1]]);
        const bool able = z[e] > NegInf<A>();
        if (!able) z[e] = NegInf<A>();  // NaN
        valid += able;  // (a ballot of x > -inf is compiled to one that counts NaN)
        high = Max(high, z[e]);
        if (able) low = -Max(-low, -z[e]);
      }
    }
    valid = WaveSum(valid);
    const int take = min(a.k, valid);
    // the largest key that `take` scores reach
    K from = 0, to = 0;
    int reached = valid;
    if (take > 0) {
      from = Scalar(KeyOf(-WaveMax(-low)));
      to = Scalar(KeyOf(WaveMax(high)));
    }
    while (from < to && reached != take) {
      const K middle = from + (to - from + 1) / 2;
      const A at = ValueOf(middle);
      int count = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * kWave < c) count += __popcll(__ballot(z[e] >= at));
      if (count >= take) {
        from = middle;
        reached = count;
      } else {
        to = middle - 1;
      }
    }
    const A edge = take > 0 ? ValueOf(from) : -NegInf<A>();
    int spare = reached - take;  // of the scores equal to the edge, the highest classes
    if (take == 0) spare = 0;
    uint32_t chosen = 0;
    if (spare == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * kWave < c && z[e] >= edge && take > 0) chosen |= 1u << e;
    } else {
      int above = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * kWave < c) above += __popcll(__ballot(z[e] > edge));
      int need = take - above;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e * kWave >= c) continue;
        const unsigned long long equal = __ballot(z[e] == edge);
        if (z[e] > edge || (z[e] == edge && __popcll(equal & below) < need)) chosen |= 1u << e;
        need = max(0, need - static_cast<int>(__popcll(equal)));
      }
    }
    int put = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (e * kWave >= c) continue;
      const unsigned long long who = __ballot(chosen >> e & 1u);
      if (chosen >> e & 1u) {
        const int at = put + __popcll(who & below), cls = e * kWave + lane;
        if constexpr (kWide) {
          s_list[wave][at] = KeyOf(z[e]);
          s_cls[wave][at] = cls;
        } else {
          s_list[wave][at] = Candidate(z[e], cls);
        }
      }
      put += __popcll(who);
    }
    WaveSync();
    int32_t* out_class = static_cast<int32_t*>(a.top_class.data) + row * a.top_class.stride[0];
    T* out_logit = static_cast<T*>(a.top_logit.data) + row * a.top_logit.stride[0];
    for (int j = lane; j < a.k; j += kWave) {
      int rank = j, cls = -1;
      T value = static_cast<T>(-INFINITY);
      if (j < take) {
        const uint64_t own = s_list[wave][j];
        rank = 0;
        if constexpr (kWide) {
          cls = s_cls[wave][j];
#pragma unroll 4
          for (int o = 0; o < take; ++o) {
            const uint64_t other = s_list[wave][o];
            rank += other > own || (other == own && s_cls[wave][o] < cls);
          }
          value = ValueOf(own);
        } else {
          cls = static_cast<int>(~static_cast<uint32_t>(own));
#pragma unroll 4
          for (int o = 0; o < take; ++o) rank += s_list[wave][o] > own;
          value = static_cast<T>(ValueOf(static_cast<uint32_t>(own >> 32)));
        }
        // as it is: of the zeros the key does not know the sign
        if (static_cast<A>(value) == A(0)) value = x[cls * a.scores.stride[1]];
      }
      out_class[rank * a.top_class.stride[1]] = cls;
      out_logit[rank * a.top_logit.stride[1]] = value;
    }
    WaveSync();  // the list is the next row's
    if (a.log_rest.data == nullptr) continue;
    A next = NegInf<A>(), sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!(chosen >> e & 1u)) next = Max(next, z[e]);
    next = WaveMax(next);
    if (next > NegInf<A>() && next < static_cast<A>(INFINITY)) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * kWave < c && !(chosen >> e & 1u)) sum += Exp2((z[e] - next) * scale);
      sum = WaveSum(sum);
    }
    if (lane == 0)
      StoreFloat(a.log_rest, row * a.log_rest.stride[0],
                 sum > A(0)
                     ? next / static_cast<A>(a.temperature) + Log2(sum) * static_cast<A>(kLn2)
                     : next);
  }
}

// ------------------------------------------------------------------ top logits, many classes
constexpr int kTopBins = 512;         // of the threads' maxima
constexpr int kTopCandidates = 1024;  // of a row at most, or it goes the slow way
constexpr int kTopChunks = 512;       // that hold them

/*!
 * One workgroup a row. Every thread takes the maxima of four parts of what it holds: the k-th
 * largest of these 4 * kBlock values, or anything below it, has at least k scores above or
 * equal to it, and seldom many more. A histogram of the maxima gives such a value; a second
 * pass over the registers picks the scores that reach it (candidates) and sums the
 * exponentials of the others; the candidates are put in order by counting. Rows with more
 * candidates than fit, of many equal scores for instance, are done digit by digit (TopAny).
 * 4096 x 50021 bfloat16, k = 64: 126 us, of which reading and the maxima alone are 84 (4.9
 * TB/s), the second pass 17 and the ranking the rest, as the two rows that a compute unit
 * holds do not hide it.
 */
template <typename T, typename Shape>
__global__ void __launch_bounds__(Shape::block, Shape::cached >= 12 ? 4 : 1)
k_top_row(LGBM_TopLogitsArgs a, double by, int lds_chunks) {
  using A = Acc<T>;
  constexpr int kBlock = Shape::block, kWaves = kBlock / kWave;
  static_assert(std::is_same_v<A, float>, "keys of 32 bits");
  __shared__ int hist[kTopBins];
  __shared__ A s_low[kWaves], s_high[kWaves], s_sum[kWaves];
  __shared__ int s_bin, s_count, s_valid;
  __shared__ uint32_t s_edge;
  __shared__ uint64_t s_list[kTopCandidates];
  __shared__ Words s_aside[kTopChunks];
  __shared__ int s_base[kTopChunks], s_chunks;
  __shared__ A s_rest[kTopCandidates];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, k = a.k;
  extern __shared__ Words row_lds[];
  RowOf<T, Shape> z(static_cast<const T*>(a.scores.data) + row * a.scores.stride[0], a.classes,
                    row_lds, lds_chunks);
  z.Load();
  for (int i = tid; i < kTopBins; i += kBlock) hist[i] = 0;
  if (tid == 0) {
    s_count = s_valid = s_bin = s_chunks = 0;
    s_edge = ~0u;
  }
  A part[4] = {NegInf<A>(), NegInf<A>(), NegInf<A>(), NegInf<A>()};
  z.Each([&](int, const auto& v, auto...) {
#pragma unroll
    for (int i = 0; i < kSizeOf<decltype(v)>; ++i) part[i & 3] = Max(part[i & 3], v[i]);
  });
  // a quarter of them is enough where it still is four times k
  if (kBlock >= 4 * k) {
    part[0] = Max(Max(part[0], part[1]), Max(part[2], part[3]));
    part[1] = part[2] = part[3] = NegInf<A>();
  }
  A high = NegInf<A>(), low = -NegInf<A>();
  int valid = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    high = Max(high, part[i]);
    if (part[i] > NegInf<A>()) {
      low = fminf(low, part[i]);
      ++valid;
    }
  }
  high = WaveMax(high);
  low = -WaveMax(-low);
  valid = WaveSum(valid);
  __syncthreads();
  if (tid % kWave == 0) {
    s_high[tid / kWave] = high;
    s_low[tid / kWave] = low;
    atomicAdd(&s_valid, valid);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    high = Max(high, s_high[i]);
    low = fminf(low, s_low[i]);
  }
  const bool bounded = s_valid >= k;  // otherwise every score may be among the k largest
  const A range = high - low;
  if (!(range < static_cast<A>(INFINITY)) || !(high > NegInf<A>())) {
    TopAny<T, kBlock>(a, row);  // infinite scores, or none at all
    return;
  }
  // bins order as the maxima do; where rounding puts equals into one, it is for all alike
  const A per = range > A(0) ? static_cast<A>(kTopBins - 1) / range : A(0);
  auto bin_of = [&](A v) {
    return min(static_cast<int>(fminf((v - low) * per, static_cast<A>(kTopBins - 1))),
               kTopBins - 1);
  };
  if (bounded) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (part[i] > NegInf<A>()) atomicAdd(&hist[bin_of(part[i])], 1);
    __syncthreads();
    if (tid < kWave) {
      // lane l holds the bins 511 - 8 l .. 504 - 8 l, largest first
      constexpr int kEach = kTopBins / kWave;
      int own[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum += own[i] = hist[kTopBins - 1 - kEach * tid - i];
      int before = sum;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(before, d);
        if (tid >= d) before += o;
      }
      before -= sum;
      if (before < k && k <= before + sum) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (before < k && k <= before + own[i]) s_bin = kTopBins - 1 - kEach * tid - i;
          before += own[i];
        }
      }
    }
    __syncthreads();
    const int bin = s_bin;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (part[i] > NegInf<A>() && bin_of(part[i]) >= bin) atomicMin(&s_edge, KeyOf(part[i]));
    __syncthreads();
  }
  // the smallest of the maxima in the bins down to the k-th
  const A edge = bounded ? ValueOf(s_edge) : -FLT_MAX;
  const A scale = static_cast<A>(by);
  A from = bounded ? edge : A(0);  // unbounded, nothing but -inf is below the edge
  const bool rest = a.log_rest.data != nullptr;
  A sum = 0;
  // a chunk with candidates is only put aside and looked at afterwards, an element a thread:
  // most turns of a wave meet one, in one of its lanes
  auto pick = [&](int cls, A v) {
    if (!(v >= edge)) return;
    const int at = atomicAdd(&s_count, 1);
    if (at < kTopCandidates) s_list[at] = Candidate(v, cls);
  };
  z.Each([&](int base, const auto& v, auto... words) {
    constexpr int kSize = kSizeOf<decltype(v)>;
    if constexpr (sizeof...(words) == 0) {
      pick(base, v[0]);
      if (rest && v[0] < edge) sum += Exp2((v[0] - from) * scale);
    } else {
      A top = v[0];
#pragma unroll
      for (int i = 1; i < kSize; ++i) top = Max(top, v[i]);
      A e[kSize];
      if (rest) {
        // at most one, and NaN as zero: the bounds are the exponential's own modifier
#pragma unroll
        for (int i = 0; i < kSize; ++i)
          e[i] = fminf(fmaxf(Exp2((v[i] - from) * scale), 0.0f), 1.0f);
      }
      if (top >= edge) {
        const int at = atomicAdd(&s_chunks, 1);
        if (at < kTopChunks) {
          s_aside[at] = (words, ...);
          s_base[at] = base;
        }
#pragma unroll
        for (int i = 0; i < kSize; ++i) e[i] = v[i] < edge ? e[i] : A(0);
      }
      if (rest) {
        A own = 0;
#pragma unroll
        for (int i = 0; i < kSize; ++i) own += e[i];
        sum += own;
      }
    }
  });
  __syncthreads();
  if (s_chunks > kTopChunks) {
    TopAny<T, kBlock>(a, row);
    return;
  }
  {
    constexpr int kSize = Chunk<T>::kSize;
    const T* aside = reinterpret_cast<const T*>(s_aside);
    const int many = s_chunks * kSize;
    for (int i = tid; i < many; i += kBlock)
      pick(s_base[i / kSize] + i % kSize, static_cast<A>(aside[i]));
  }
  __syncthreads();
  const int n = s_count;
  if (n > kTopCandidates) {
    TopAny<T, kBlock>(a, row);
    return;
  }
  int32_t* out_class = static_cast<int32_t*>(a.top_class.data) + row * a.top_class.stride[0];
  T* out_logit = static_cast<T*>(a.top_logit.data) + row * a.top_logit.stride[0];
  // eight lanes compare one candidate with the others
  for (int i = tid / 8; i < n; i += kBlock / 8) {
    const uint64_t own = s_list[i];
    int rank = 0;
#pragma unroll 4
    for (int o = tid % 8; o < n; o += 8) rank += s_list[o] > own;
    rank += __shfl_xor(rank, 1);
    rank += __shfl_xor(rank, 2);
    rank += __shfl_xor(rank, 4);
    if (tid % 8 != 0) continue;
    const int cls = static_cast<int>(~static_cast<uint32_t>(own));
    const A v = ValueOf(static_cast<uint32_t>(own >> 32));
    if (rank < k) {
      out_class[rank * a.top_class.stride[1]] = cls;
      // as it is: of the zeros the key does not know the sign
      out_logit[rank * a.top_logit.stride[1]] = v == A(0) ? z.x[cls] : static_cast<T>(v);
    } else {
      s_rest[rank - k] = v;  // in order, so that their sum is the same every time
    }
  }
  for (int i = n + tid; i < k; i += kBlock) {
    out_class[i * a.top_class.stride[1]] = -1;
    out_logit[i * a.top_logit.stride[1]] = static_cast<T>(-INFINITY);
  }
  if (!rest) return;
  // two sums, each against a value near its own: of what is below the edge, and of the
  // candidates that were not chosen
  sum = BlockSum<kBlock>(sum, s_sum);
  if (n <= k && sum < SmallRest<A>()) {
    // far below the edge: against its own maximum; seldom, so from memory in a plain loop
    A own = NegInf<A>();
    for (int i = tid; i < a.classes; i += kBlock) {
      const A v = static_cast<A>(z.x[i]);
      if (v < edge) own = Max(own, v);
    }
    own = BlockMax<kBlock>(own, s_low);
    sum = 0;
    if (own > NegInf<A>()) {
      from = own;
      for (int i = tid; i < a.classes; i += kBlock) {
        const A v = static_cast<A>(z.x[i]);
        if (v < edge) sum += Exp2((v - from) * scale);
      }
      sum = BlockSum<kBlock>(sum, s_high);
    }
  }
  if (n > k) {
    const A next = s_rest[0];
    A more = 0;
    for (int i = tid; i < n - k; i += kBlock) more += Exp2((s_rest[i] - next) * scale);
    more = BlockSum<kBlock>(more, s_high);
    // the next candidate is not below the edge, and has a term of one in its own sum
    sum = more + (sum > A(0) ? sum * Exp2((from - next) * scale) : A(0));
    from = next;
  }
  if (tid == 0)
    StoreFloat(a.log_rest, row * a.log_rest.stride[0],
               sum > A(0) ? fma(from, by, static_cast<double>(Log2(sum))) * kLn2
                          : -static_cast<double>(INFINITY));
}

// ------------------------------------------------------------------ verification
/*! what counts as probability: NaN, infinities and negative values are none */
template <typename T> __device__ __forceinline__ double Mass(T x) {
  const double v = static_cast<double>(static_cast<Acc<T>>(x));
  return v > 0.0 && v < static_cast<double>(INFINITY) ? v : 0.0;
}

__device__ __forceinline__ double Uniform(const LGBM_Array& a, int64_t at) {
  return a.type == C_API_DTYPE_FLOAT64 ? At<double>(a, at) : static_cast<double>(At<float>(a, at));
}

/*! drafts of sequence `row`, 0..drafts */
__device__ __forceinline__ int Length(const LGBM_VerifyArgs& a, int64_t row) {
  if (a.length.data == nullptr) return a.drafts;
  const int64_t at = row * a.length.stride[0];
  const int64_t v = a.length.type == C_API_DTYPE_INT64 ? At<int64_t>(a.length, at)
                                                       : At<int32_t>(a.length, at);
  return static_cast<int>(min(max(v, int64_t{0}), static_cast<int64_t>(a.drafts)));
}

template <typename T>
__device__ __forceinline__ const T* TargetRow(const LGBM_VerifyArgs& a, int64_t row, int64_t s) {
  return static_cast<const T*>(a.target.data) + row * a.target.stride[0] + s * a.target.stride[1];
}
template <typename T>
__device__ __forceinline__ const T* DraftRow(const LGBM_VerifyArgs& a, int64_t row, int64_t s) {
  return static_cast<const T*>(a.draft_prob.data) + row * a.draft_prob.stride[0] +
         s * a.draft_prob.stride[1];
}

/*! whether draft s (class x) of the sequence stands: u q(x) < p(x), in 64 bits, where the
 *  product of 32-bit numbers is exact */
template <typename T>
__device__ __forceinline__ bool Stands(const LGBM_VerifyArgs& a, int64_t row, int s, int x) {
  if (x < 0) return false;
  const double u = Uniform(a.accept, row * a.accept.stride[0] + s * a.accept.stride[1]);
  const double p = Mass(TargetRow<T>(a, row, s)[x * a.target.stride[2]]);
  const double q = a.draft_prob.data ? Mass(DraftRow<T>(a, row, s)[x * a.draft_prob.stride[2]])
                                     : 1.0;
  return u * q < p;
}

/*! how many drafts of the sequence stand; one wave's work, known to all its lanes */
template <typename T>
__device__ __forceinline__ int Accepted(const LGBM_VerifyArgs& a, int64_t row, int length) {
  const int lane = threadIdx.x % kWave;
  for (int s0 = 0; s0 < length; s0 += kWave) {
    const int s = s0 + lane;
    bool refused = false;
    if (s < length) {
      const int x = LoadClass(a.draft_class, row * a.draft_class.stride[0] +
                                                 s * a.draft_class.stride[1], a.classes);
      refused = !Stands<T>(a, row, s, x);
    }
    const unsigned long long who = __ballot(refused);
    if (who) return s0 + __ffsll(who) - 1;
  }
  return length;
}

/*! what class c weighs in the draw of the class that follows the accepted ones */
template <typename T> struct Residual {
  const T* p;
  const T* q;        // nullptr: nothing is taken away, but for class `gone`
  int64_t ps, qs;
  int gone;
  __device__ __forceinline__ double operator()(int c) const {
    const double v = Mass(p[c * ps]);
    if (q != nullptr) return fmax(v - Mass(q[c * qs]), 0.0);
    return c == gone ? 0.0 : v;
  }
};

template <typename T>
__device__ __forceinline__ Residual<T> ResidualOf(const LGBM_VerifyArgs& a, int64_t row,
                                                  int accepted, int length) {
  Residual<T> f{TargetRow<T>(a, row, accepted), nullptr, a.target.stride[2],
                a.draft_prob.stride[2], -1};
  if (accepted < length) {
    if (a.draft_prob.data) {
      f.q = DraftRow<T>(a, row, accepted);
    } else {
      f.gone = LoadClass(a.draft_class, row * a.draft_class.stride[0] +
                                            accepted * a.draft_class.stride[1], a.classes);
    }
  }
  return f;
}

/*!
 * The first class at which the running sum of `mass` over [base, base + len) exceeds
 * `goal`; the last one with any mass where rounding keeps the sum from it, -1 where there
 * is none. The range is cut into one segment a wave, the segment that holds the goal into
 * as many again, down to one class a lane: all but the first cut read a fraction of it.
 * Whole workgroup; `sums` has one place a wave.
 */
template <int kBlock, typename F>
__device__ __forceinline__ int FindClass(const F& mass, int base, int len, double goal,
                                         double* sums) {
  constexpr int kWaves = kBlock / kWave;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  while (len > kWave) {
    const int seg = ((len + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    double own = 0;
    for (int i = wave * seg + lane; i < min(len, (wave + 1) * seg); i += kWave)
      own += mass(base + i);
    own = WaveSum(own);
    __syncthreads();
    if (lane == 0) sums[wave] = own;
    __syncthreads();
    int found = -1;
    double before = 0, reach = 0;
    for (int i = 0; i < kWaves; ++i) {
      if (!(sums[i] > 0)) continue;
      found = i;
      before = reach;
      reach += sums[i];
      if (reach > goal) break;
    }
    if (found < 0) return -1;
    goal -= before;
    base += found * seg;
    len = min(len - found * seg, seg);
  }
  const double own = lane < len ? mass(base + lane) : 0.0;
  double reach = own;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double o = __shfl_up(reach, d);
    if (lane >= d) reach += o;
  }
  const unsigned long long some = __ballot(own > 0), over = __ballot(own > 0 && reach > goal);
  if (over) return base + __ffsll(over) - 1;
  return some ? base + 63 - __clzll(some) : -1;
}

/*! writes a sequence's results; `who` and `many` are the threads that do it */
__device__ __forceinline__ void PutVerified(const LGBM_VerifyArgs& a, int64_t row, int accepted,
                                            int drawn, int who, int many) {
  int32_t* out = static_cast<int32_t*>(a.out_class.data) + row * a.out_class.stride[0];
  for (int s = who; s <= a.drafts; s += many) {
    int x = s == accepted ? drawn : -1;
    if (s < accepted)
      x = LoadClass(a.draft_class, row * a.draft_class.stride[0] + s * a.draft_class.stride[1],
                    a.classes);
    out[s * a.out_class.stride[1]] = x;
  }
  if (who == 0)
    static_cast<int32_t*>(a.out_accepted.data)[row * a.out_accepted.stride[0]] = accepted;
}

/*! one workgroup a sequence */
template <typename T, int kBlock>
__global__ void __launch_bounds__(kBlock) k_verify_any(LGBM_VerifyArgs a) {
  __shared__ double sums[kBlock / kWave];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, c = a.classes;
  const int length = Length(a, row);
  const int n = Accepted<T>(a, row, length);  // every wave finds the same
  Residual<T> mass = ResidualOf<T>(a, row, n, length);
  double total = 0;
  for (int round = 0; round < 2; ++round) {
    total = 0;
    for (int i = tid; i < c; i += kBlock) total += mass(i);
    __syncthreads();
    total = BlockSum<kBlock>(total, sums);
    if (total > 0) break;
    // nothing is left of the target: the draw is from the target itself
    mass.q = nullptr;
    mass.gone = -1;
  }
  const double goal = Uniform(a.sample, row * a.sample.stride[0]) * total;
  const int drawn = FindClass<kBlock>(mass, 0, c, goal, sums);
  PutVerified(a, row, n, drawn, tid, kBlock);
}

// ------------------------------------------------------------------ verification, few classes
constexpr int kFewEach = 4;                    // classes a lane
constexpr int kFewClasses = kWave * kFewEach;  // at most

/*!
 * `lanes` (a power of two) lanes a sequence, each with four neighbouring classes: the drafts
 * are judged one a lane, the running sums are a scan over the lanes. Bound by the latency of
 * four loads that follow from each other (length, draft, probabilities, row): 100000 sequences
 * of 3 drafts over 10 float64 classes 10 us.
 */
template <typename T>
__global__ void __launch_bounds__(256) k_verify_few(LGBM_VerifyArgs a, int lanes) {
  const int l = threadIdx.x % lanes;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
  const bool there = at < a.rows;
  const int64_t row = there ? at : a.rows - 1;  // so that every lane takes part in the shuffles
  const int length = Length(a, row);
  int n = length;
  for (int s = l; s < length; s += lanes) {
    const int x = LoadClass(a.draft_class,
                            row * a.draft_class.stride[0] + s * a.draft_class.stride[1], a.classes);
    if (!Stands<T>(a, row, s, x)) {
      n = s;
      break;
    }
  }
  for (int d = lanes / 2; d > 0; d >>= 1) n = min(n, __shfl_xor(n, d));
  Residual<T> mass = ResidualOf<T>(a, row, n, length);
  double own[kFewEach], sum, total;
  for (int round = 0; round < 2; ++round) {
    sum = 0;
#pragma unroll
    for (int i = 0; i < kFewEach; ++i) {
      const int c = l * kFewEach + i;
      own[i] = c < a.classes ? mass(c) : 0.0;
      sum += own[i];
    }
    total = sum;
    for (int d = lanes / 2; d > 0; d >>= 1) total += __shfl_xor(total, d);
    if (!(total > 0)) {  // nothing is left of the target: the draw is from the target itself
      mass.q = nullptr;
      mass.gone = -1;
    }
    if (!__any(!(total > 0))) break;
  }
  double reach = sum;
  for (int d = 1; d < lanes; d <<= 1) {
    const double o = __shfl_up(reach, d, lanes);
    if (l >= d) reach += o;
  }
  reach -= sum;
  const double goal = Uniform(a.sample, row * a.sample.stride[0]) * total;
  int first = a.classes, last = -1;
#pragma unroll
  for (int i = 0; i < kFewEach; ++i) {
    if (!(own[i] > 0)) continue;
    reach += own[i];
    last = l * kFewEach + i;
    if (reach > goal) first = min(first, last);
  }
  for (int d = lanes / 2; d > 0; d >>= 1) {
    first = min(first, __shfl_xor(first, d));
    last = max(last, __shfl_xor(last, d));
  }
  if (there) PutVerified(a, row, n, first < a.classes ? first : last, l, lanes);
}

// ------------------------------------------------------------------ verification, many classes
constexpr int kSplitBlock = 256;
constexpr int kSplitWaves = kSplitBlock / kWave;
constexpr int kMostSplits = 64;  // workgroups a sequence

/*! classes of one wave's segment: whole turns of the wave over its chunks */
template <typename T> __host__ __device__ inline int SegmentOf(int classes, int splits) {
  const int turn = kWave * Chunk<T>::kSize, waves = splits * kSplitWaves;
  return ((classes + waves - 1) / waves + turn - 1) / turn * turn;
}

/*! Mass of a value of at most 32 bits, in as many */
template <typename T> __device__ __forceinline__ float Mass32(T x) {
  const float v = fmaxf(static_cast<float>(x), 0.0f);  // NaN gives zero
  return v < INFINITY ? v : 0.0f;
}
__device__ __forceinline__ double MassOf(double x) { return Mass(x); }
__device__ __forceinline__ double MassOf(float x) { return Mass32(x); }
__device__ __forceinline__ double MassOf(_Float16 x) { return Mass32(x); }
__device__ __forceinline__ double MassOf(__bf16 x) { return Mass32(x); }

/*! the mass of classes [begin, end) of a row whose classes stand next to each other; one wave */
template <typename T>
__device__ __forceinline__ double WaveMass(const Residual<T>& f, int begin, int end) {
  constexpr int kSize = Chunk<T>::kSize;
  const int lane = threadIdx.x % kWave;
  double sum = 0;
  const int whole = begin + (end - begin) / kSize * kSize;
#pragma unroll 4
  for (int c = begin + lane * kSize; c < whole; c += kWave * kSize) {
    Chunk<T> p, q;
    __builtin_memcpy(&p, f.p + c, sizeof(p));
    if (f.q != nullptr) __builtin_memcpy(&q, f.q + c, sizeof(q));
#pragma unroll
    for (int i = 0; i < kSize; ++i) {
      double v = MassOf(p.v[i]);
      if (f.q != nullptr) v = fmax(v - MassOf(q.v[i]), 0.0);
      else if (c + i == f.gone) v = 0.0;
      sum += v;
    }
  }
  if (whole + lane < end) sum += f(whole + lane);
  return WaveSum(sum);
}

/*!
 * Each wave of `splits` workgroups a sequence sums one segment of the row that the class is
 * drawn from. Which row that is, every workgroup finds for itself: a few gathers, instead of
 * a launch before this one. The first of them writes what is known already. Bound by memory
 * for a batch (256 x 50021 bfloat16, both sides, 15 us, 3.4 TB/s), by latency for one sequence
 * (131072 float32 classes over 64 workgroups 4.4 us; one workgroup for all 230).
 */
template <typename T>
__global__ void __launch_bounds__(kSplitBlock) k_verify_sums(LGBM_VerifyArgs a) {
  const int64_t row = blockIdx.y;
  const int length = Length(a, row), n = Accepted<T>(a, row, length);
  const Residual<T> mass = ResidualOf<T>(a, row, n, length);
  const int seg = SegmentOf<T>(a.classes, gridDim.x);
  const int at = blockIdx.x * kSplitWaves + threadIdx.x / kWave;
  const int begin = min(a.classes, at * seg), end = min(a.classes, begin + seg);
  const double sum = WaveMass(mass, begin, end);
  if (threadIdx.x % kWave == 0)
    static_cast<double*>(a.workspace)[row * gridDim.x * kSplitWaves + at] = sum;
  if (blockIdx.x == 0) PutVerified(a, row, n, -1, threadIdx.x, kSplitBlock);
}

/*!
 * One workgroup a sequence: the segment that holds the goal, by the waves' sums; in it the
 * run of neighbouring classes of one thread, by a scan over the threads' sums; in that the
 * class. The row is read twice where the goal lies, and nowhere else. Latency: 4 us for one
 * sequence, 8 for 256.
 */
template <typename T>
__global__ void __launch_bounds__(kSplitBlock) k_verify_draw(LGBM_VerifyArgs a, int splits) {
  constexpr int kSize = Chunk<T>::kSize;
  __shared__ double sums[kSplitWaves];
  __shared__ double s_goal;
  __shared__ int s_base;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int segments = splits * kSplitWaves;
  static_assert(kMostSplits * kSplitWaves <= 4 * kWave, "four segments a lane");
  const double* part = static_cast<const double*>(a.workspace) + row * segments;
  const int length = Length(a, row);
  const int n = static_cast<const int32_t*>(a.out_accepted.data)[row * a.out_accepted.stride[0]];
  Residual<T> mass = ResidualOf<T>(a, row, n, length);
  const double v = Uniform(a.sample, row * a.sample.stride[0]);
  // every wave does the same with the segments' sums: lane l has those of 4 l .. 4 l + 3
  double own[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    own[i] = 4 * lane + i < segments ? part[4 * lane + i] : 0.0;
    sum += own[i];
  }
  auto wave_scan = [&](double reach) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const double o = __shfl_up(reach, d);
      if (lane >= d) reach += o;
    }
    return reach;
  };
  double reach = wave_scan(sum);
  const double total = __shfl(reach, kWave - 1);
  reach -= sum;
  int drawn;
  if (total > 0) {
    double goal = v * total;
    int found = -1, last = -1;
    double before = 0, last_before = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!(own[i] > 0)) continue;
      last = 4 * lane + i;
      last_before = reach;
      reach += own[i];
      if (found < 0 && reach > goal) {
        found = last;
        before = last_before;
      }
    }
    const unsigned long long over = __ballot(found >= 0), some = __ballot(last >= 0);
    const int who = over ? __ffsll(over) - 1 : 63 - __clzll(some);
    found = __shfl(over ? found : last, who);
    goal -= __shfl(over ? before : last_before, who);
    const int seg = SegmentOf<T>(a.classes, splits);
    const int begin = found * seg, end = min(a.classes, begin + seg);
    // this thread's run; whole chunks at first, the classes after the last of them one by one
    const int each = (seg + kSplitBlock * kSize - 1) / (kSplitBlock * kSize) * kSize;
    const int mine = min(end, begin + tid * each), stop = min(end, mine + each);
    double run = 0;
    int c = mine;
    for (; c + kSize <= stop; c += kSize) {
      Chunk<T> p, q;
      __builtin_memcpy(&p, mass.p + c, sizeof(p));
      if (mass.q != nullptr) __builtin_memcpy(&q, mass.q + c, sizeof(q));
#pragma unroll
      for (int i = 0; i < kSize; ++i) {
        double w = MassOf(p.v[i]);
        if (mass.q != nullptr) w = fmax(w - MassOf(q.v[i]), 0.0);
        else if (c + i == mass.gone) w = 0.0;
        run += w;
      }
    }
    for (; c < stop; ++c) run += mass(c);
    double upto = wave_scan(run);
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    // the first wave whose sums up to its end pass the goal, the last with any where none does
    int chosen = -1;
    double wave_before = 0, prefix = 0;
    for (int i = 0; i < kSplitWaves; ++i) {
      if (!(sums[i] > 0)) continue;
      chosen = i;
      wave_before = prefix;
      prefix += sums[i];
      if (prefix > goal) break;
    }
    upto += wave_before;
    const unsigned long long pass = __ballot(run > 0 && upto > goal), any = __ballot(run > 0);
    const int who_runs = pass ? __ffsll(pass) - 1 : 63 - __clzll(any | 1);
    const bool here = wave == chosen && lane == who_runs;
    if (here) {
      s_base = mine;
      s_goal = goal - (upto - run);
    }
    __syncthreads();
    const int base = s_base;
    drawn = FindClass<kSplitBlock>(mass, base, min(each, end - base), s_goal, sums);
  } else {  // nothing is left of the target: the draw is from the target itself
    mass.q = nullptr;
    mass.gone = -1;
    double whole = 0;
    for (int i = tid; i < a.classes; i += kSplitBlock) whole += mass(i);
    whole = BlockSum<kSplitBlock>(whole, sums);
    drawn = FindClass<kSplitBlock>(mass, 0, a.classes, v * whole, sums);
  }
  if (tid == 0)
    static_cast<int32_t*>(a.out_class.data)[row * a.out_class.stride[0] +
                                            n * a.out_class.stride[1]] = drawn;
}

// ------------------------------------------------------------------ launches
/*! the calling thread's device is `device` while this lives */
class OnDevice {
 public:
  explicit OnDevice(int device) {
    OPS_HIP_OK(hipGetDevice(&before_));
    if (device != before_) {
      OPS_HIP_OK(hipSetDevice(device));
      moved_ = true;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool moved_ = false;
};

// A launch has fewer than 2^32 threads, and a workgroup of 1024 may have a row for itself.
constexpr int64_t kRowsAtOnce = int64_t{1} << 21;

/*! an array from row `start` on */
void Advance(LGBM_Array* a, int64_t start) {
  if (a->data != nullptr)
    a->data = static_cast<char*>(a->data) + start * a->stride[0] * ElementSize(a->type);
}

/*! f(arguments of some rows) until all rows have had their turn; `arrays` are all of a call's */
template <typename Args, typename F>
void InParts(const Args& a, int64_t most, std::initializer_list<LGBM_Array Args::*> arrays, F&& f) {
  for (int64_t start = 0; start < a.rows; start += most) {
    Args part = a;
    part.rows = std::min(most, a.rows - start);
    for (auto array : arrays) Advance(&(part.*array), start);
    f(part);
  }
}

template <typename F> void ByType(int type, F&& f) {
  switch (type) {
    case C_API_DTYPE_FLOAT64: f(double{}); break;
    case C_API_DTYPE_FLOAT32: f(float{}); break;
    case C_API_DTYPE_FLOAT16: f(_Float16{}); break;
    default: f(__bf16{}); break;
  }
}

/*! the smallest power of two of threads that hold `classes` at `each` a thread */
int LanesFor(int classes, int each) {
  int lanes = 1;
  while (lanes * each < classes) lanes *= 2;
  return lanes;
}

template <typename T, bool kLoss, int E, TeamKind kKind>
void LaunchDistillTile(const LGBM_DistillArgs& a, hipStream_t s) {
  const int lanes = LanesFor(a.classes, E), rows = 256 / lanes;
  const size_t lds = sizeof(Word<Acc<T>>) * rows * a.classes;  // at most 2048 * E bytes
  auto kernel = k_distill_tile<T, kLoss, E, kKind>;
  AllowLds(kernel, lds);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((a.rows + rows - 1) / rows)), dim3(256),
                     lds, s, a, kLog2e / a.temperature, lanes);
}

template <typename T, bool kLoss>
void DistillTile(const LGBM_DistillArgs& a, bool across, hipStream_t s) {
  if (!across && a.classes <= 64) LaunchDistillTile<T, kLoss, 4, kNeighbours>(a, s);
  else if (!across) LaunchDistillTile<T, kLoss, 16, kNeighbours>(a, s);
  else if (a.classes <= 4) LaunchDistillTile<T, kLoss, 4, kAlone>(a, s);
  else if (a.classes <= 8) LaunchDistillTile<T, kLoss, 8, kAlone>(a, s);
  else if (a.classes <= 16) LaunchDistillTile<T, kLoss, 16, kAlone>(a, s);
  else if (a.classes <= 256) LaunchDistillTile<T, kLoss, 16, kAcross>(a, s);
  else LaunchDistillTile<T, kLoss, 32, kAcross>(a, s);
}

/*! whether the rows of a class stand closer together than the classes of a row */
bool ClassMajor(const LGBM_Array& scores) {
  const int64_t row_step = std::abs(scores.stride[0]);  // 0: one row for all
  return row_step != 0 && row_step < std::abs(scores.stride[1]);
}

template <typename T, int E, TeamKind kKind>
void LaunchTopTile(const LGBM_TopLogitsArgs& a, hipStream_t s) {
  const int lanes = LanesFor(a.classes, E), rows = 256 / lanes;
  hipLaunchKernelGGL((k_top_tile<T, E, kKind>),
                     dim3(static_cast<uint32_t>((a.rows + rows - 1) / rows)), dim3(256), 0, s, a,
                     lanes);
}

template <typename T, int E, bool kTurned>
void LaunchTopWave(const LGBM_TopLogitsArgs& a, hipStream_t s) {
  const int64_t rows = kTurned ? kTurnedRows : 4;
  const size_t lds = kTurned ? sizeof(T) * rows * (a.classes | 1) : 0;
  auto kernel = k_top_wave<T, E, kTurned>;
  AllowLds(kernel, lds);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((a.rows + rows - 1) / rows)), dim3(256),
                     lds, s, a);
}

/*! chunks a thread that stand in LDS, where `other` bytes of its 160 KiB have another use */
template <typename Shape> int LdsChunksOf(int chunks, size_t other) {
  if (!Shape::more) return 0;
  const int wanted = (chunks - Shape::cached * Shape::block + Shape::block - 1) / Shape::block;
  const size_t all = Shape::block <= 512 ? 80 * 1024 : 160 * 1024;  // two, or one a compute unit
  const int room = static_cast<int>((all - std::min<size_t>(other, all)) /
                                    (sizeof(Words) * Shape::block));
  return std::max(0, std::min({wanted, room, kLdsChunks}));
}

template <typename T, typename Shape>
void LaunchTopRow(const LGBM_TopLogitsArgs& a, hipStream_t s) {
  const int held = LdsChunksOf<Shape>(a.classes / Chunk<T>::kSize, 32768);
  const size_t lds = sizeof(Words) * held * Shape::block;
  auto kernel = k_top_row<T, Shape>;
  AllowLds(kernel, lds);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.rows)), dim3(Shape::block), lds, s, a,
                     kLog2e / a.temperature, held);
}

/*!
 * The workgroup of a row of `chunks` whole chunks, f(threads, chunks a thread in registers).
 * Many rows: few threads with much of the row each, so that four rows or more share a compute
 * unit and one computes while another waits for its scores. Rows that leave compute units
 * idle: as many threads as there are, so that the one row is done sooner. Rows that do not
 * fit: two share a compute unit if they are only read (1000 x 150000 bfloat16: top 64 92 us
 * against 107 of one, loss 88 against 104), but where as much is written again the part that
 * is read twice costs more than the other row hides (1500 x 131077 float32: 445 us against
 * 399).
 */
template <typename F> void ByRow(int64_t rows, int chunks, bool writes, F&& f) {
  if (chunks <= 256) f(RowShape<256, 1>{});
  else if (rows < 512 && chunks <= 4096) f(RowShape<1024, 4>{});
  else if (chunks <= 1024) f(RowShape<256, 4>{});
  else if (chunks <= 2048) f(RowShape<256, 8>{});
  else if (chunks <= 4096) f(RowShape<256, 16>{});
  else if (rows >= 512 && chunks <= 8192) f(RowShape<512, 16>{});
  else if (rows >= 512 && !writes) f(RowShape<512, 16, true>{});
  else f(RowShape<1024, 12, true>{});
}

void TopLogitsPart(const LGBM_TopLogitsArgs& a, hipStream_t s) {
  const bool across = ClassMajor(a.scores);
  ByType(a.scores.type, [&](auto t) {
    using T = decltype(t);
    if (a.classes <= 512) {
      // With k times the largest of what is left, a row's time grows with k and with the lanes
      // it takes; by bisection hardly. Row-major, the two meet where k times the lanes is about
      // 300: 400000 x 100 float32 (8 lanes) k = 10 146 us against 362, k = 50 514 against 401;
      // 300000 x 250 bfloat16 (16 lanes) k = 5 168 against 338, k = 20 402 against 381; 200000
      // x 300 float32 (32 lanes) k = 5 179 against 336, k = 20 526 against 369. Class-major,
      // where a round is two barriers and bisection has to turn the rows first, about 256, and
      // 25 rounds: float64, 8000 x 100 k = 8 20 against 29, k = 30 55 against 39; 8000 x 300
      // k = 8 36 against 43, k = 30 100 against 54; 40000 x 100 k = 8 32 against 76. A
      // wave of 1000 classes has no registers left for others beside it: 100000 x 1000
      // bfloat16, k = 100, 964 against 761 of a workgroup a row.
      const int rounds = a.k * LanesFor(a.classes, 16);
      const bool few = across ? a.k <= 25 && rounds <= 256 : rounds <= 300;
      if (!across && a.classes <= 64) LaunchTopTile<T, 4, kNeighbours>(a, s);
      else if (!across && few) LaunchTopTile<T, 16, kNeighbours>(a, s);
      else if (!across && a.classes <= 256) LaunchTopWave<T, 4, false>(a, s);
      else if (!across) LaunchTopWave<T, 8, false>(a, s);
      else if (a.classes <= 4) LaunchTopTile<T, 4, kAlone>(a, s);
      else if (a.classes <= 8) LaunchTopTile<T, 8, kAlone>(a, s);
      else if (a.classes <= 16) LaunchTopTile<T, 16, kAlone>(a, s);
      else if (few && a.classes <= 256) LaunchTopTile<T, 16, kAcross>(a, s);
      else if (few) LaunchTopTile<T, 32, kAcross>(a, s);
      else if (a.classes <= 256) LaunchTopWave<T, 4, true>(a, s);
      else LaunchTopWave<T, 8, true>(a, s);
      return;
    }
    if constexpr (!std::is_same_v<T, double>) {
      if (a.scores.stride[1] == 1) {
        ByRow(a.rows, a.classes / Chunk<T>::kSize, false, [&](auto shape) {
          LaunchTopRow<T, decltype(shape)>(a, s);
        });
        return;
      }
    }
    hipLaunchKernelGGL((k_top_any<T, 256>), dim3(static_cast<uint32_t>(a.rows)), dim3(256), 0, s,
                       a);
  });
  OPS_HIP_OK(hipGetLastError());
}

template <typename T, typename Shape>
void LaunchDistillRow(const LGBM_DistillArgs& a, hipStream_t s) {
  const size_t marks = sizeof(uint32_t) * ((a.classes + 31) / 32);
  const int held = LdsChunksOf<Shape>(a.classes / Chunk<T>::kSize, marks + 4096);
  const size_t lds = marks + sizeof(Words) * held * Shape::block;
  auto launch = [&](auto kernel) {
    AllowLds(kernel, lds);
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(a.rows)), dim3(Shape::block), lds, s, a,
                       kLog2e / a.temperature, held);
  };
  if (a.hessian.data) launch(k_distill_row<T, Shape, true>);
  else launch(k_distill_row<T, Shape, false>);
}

void TopLogitsDevice(const LGBM_TopLogitsArgs& a, int device, void* stream) {
  OnDevice on(device);
  using Args = LGBM_TopLogitsArgs;
  InParts(a, kRowsAtOnce, {&Args::scores, &Args::top_class, &Args::top_logit, &Args::log_rest},
          [&](const Args& part) { TopLogitsPart(part, static_cast<hipStream_t>(stream)); });
}

void DistillPart(const LGBM_DistillArgs& a, hipStream_t s) {
  const bool across = ClassMajor(a.scores);
  if (a.classes <= 512) {
    ByType(a.scores.type, [&](auto t) {
      using T = decltype(t);
      LGBM_DistillArgs part = a;
      if constexpr (std::is_same_v<T, double>) {
        part.gradient.data = part.hessian.data = nullptr;
        if (a.loss.data) DistillTile<double, true>(part, across, s);
        part = a;
        part.loss.data = nullptr;
      }
      if (part.loss.data || part.gradient.data || part.hessian.data)
        DistillTile<T, !std::is_same_v<T, double>>(part, across, s);
    });
    OPS_HIP_OK(hipGetLastError());
    return;
  }
  if (a.scores.stride[1] == 1 && a.scores.type != C_API_DTYPE_FLOAT64 &&
      (!a.gradient.data || a.gradient.stride[1] == 1) &&
      (!a.hessian.data || a.hessian.stride[1] == 1)) {
    ByType(a.scores.type, [&](auto t) {
      using T = decltype(t);
      if constexpr (!std::is_same_v<T, double>) {
        const bool writes = a.gradient.data || a.hessian.data;
        ByRow(a.rows, a.classes / Chunk<T>::kSize, writes, [&](auto shape) {
          LaunchDistillRow<T, decltype(shape)>(a, s);
        });
      }
    });
    OPS_HIP_OK(hipGetLastError());
    return;
  }
  const dim3 grid(static_cast<uint32_t>(a.rows));
  const size_t lds = sizeof(uint32_t) * ((a.classes + 31) / 32);
  ByType(a.scores.type, [&](auto t) {
    auto kernel = k_distill_any<decltype(t), 256>;
    AllowLds(kernel, lds);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, a, kLog2e / a.temperature);
  });
  OPS_HIP_OK(hipGetLastError());
}

void DistillDevice(const LGBM_DistillArgs& a, int device, void* stream) {
  OnDevice on(device);
  using Args = LGBM_DistillArgs;
  InParts(a, kRowsAtOnce,
          {&Args::scores, &Args::teacher_class, &Args::teacher_logit, &Args::teacher_rest,
           &Args::label, &Args::weight, &Args::loss, &Args::gradient, &Args::hessian},
          [&](const Args& part) { DistillPart(part, static_cast<hipStream_t>(stream)); });
}

constexpr int64_t kSplitRows = 32768;  // sequences of the split kernels at once

/*! workgroups a sequence, 0 where the split kernels do not apply */
int SplitsOf(const LGBM_VerifyArgs& a) {
  if (a.classes <= kFewClasses) return 0;
  if (a.target.stride[2] != 1 || (a.draft_prob.data && a.draft_prob.stride[2] != 1)) return 0;
  const int64_t wanted = (1024 + a.rows - 1) / a.rows, fitting = (a.classes + 2047) / 2048;
  return static_cast<int>(std::min<int64_t>({wanted, fitting, kMostSplits}));
}

int64_t VerifyWorkspaceDevice(const LGBM_VerifyArgs& a) {
  return std::min(a.rows, kSplitRows) * SplitsOf(a) * kSplitWaves *
         static_cast<int64_t>(sizeof(double));
}

void VerifyPart(const LGBM_VerifyArgs& a, int splits, hipStream_t s);

void VerifyDevice(const LGBM_VerifyArgs& a, int device, void* stream) {
  const int splits = SplitsOf(a);
  if (splits > 0 && (a.workspace == nullptr || a.workspace_bytes < VerifyWorkspaceDevice(a)))
    Log::Fatal("VerifyDrafts needs a workspace of %lld bytes, got %lld",
               static_cast<long long>(VerifyWorkspaceDevice(a)),
               static_cast<long long>(a.workspace ? a.workspace_bytes : 0));
  OnDevice on(device);
  using Args = LGBM_VerifyArgs;
  // parts follow each other on the stream, and use the same workspace
  InParts(a, splits > 0 ? kSplitRows : kRowsAtOnce,
          {&Args::target, &Args::draft_prob, &Args::draft_class, &Args::accept, &Args::sample,
           &Args::length, &Args::out_class, &Args::out_accepted},
          [&](const Args& part) { VerifyPart(part, splits, static_cast<hipStream_t>(stream)); });
}

void VerifyPart(const LGBM_VerifyArgs& a, int splits, hipStream_t s) {
  const uint32_t rows = static_cast<uint32_t>(a.rows);
  ByType(a.target.type, [&](auto t) {
    using T = decltype(t);
    if (a.classes <= kFewClasses) {
      const int lanes = LanesFor(a.classes, kFewEach), each = 256 / lanes;
      hipLaunchKernelGGL((k_verify_few<T>), dim3((rows + each - 1) / each), dim3(256), 0, s, a,
                         lanes);
    } else if (splits > 0) {
      hipLaunchKernelGGL((k_verify_sums<T>), dim3(splits, rows), dim3(kSplitBlock), 0, s, a);
      hipLaunchKernelGGL((k_verify_draw<T>), dim3(rows), dim3(kSplitBlock), 0, s, a, splits);
    } else {
      hipLaunchKernelGGL((k_verify_any<T, 256>), dim3(rows), dim3(256), 0, s, a);
    }
  });
  OPS_HIP_OK(hipGetLastError());
}

const DeviceOps kOps{TopLogitsDevice, DistillDevice, VerifyDevice, VerifyWorkspaceDevice};
const bool kRegistered = (g_device_ops = &kOps, true);

}  // namespace
}  // namespace class_ops
}  // namespace migbm
