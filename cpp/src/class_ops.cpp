/*! Operators over class scores: argument checks, dispatch, and the host implementation
 *  (64-bit arithmetic, one row or sequence per OpenMP iteration). */
#include "migbm/class_ops.h"

#include "migbm/common.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <limits>
#include <numeric>
#include <vector>

namespace migbm {
namespace class_ops {

const DeviceOps* g_device_ops = nullptr;

namespace {

constexpr double kInf = std::numeric_limits<double>::infinity();

float FromHalf(uint16_t h) {
  const uint32_t sign = static_cast<uint32_t>(h & 0x8000u) << 16;
  const uint32_t mag = h & 0x7fffu;
  float f;
  uint32_t bits;
  if (mag >= 0x7c00u) {
    bits = sign | 0x7f800000u | ((mag & 0x3ffu) << 13);
  } else if (mag >= 0x400u) {
    bits = sign | ((mag << 13) + (112u << 23));
  } else {
    f = static_cast<float>(mag) * 5.9604644775390625e-8f;  // 2^-24
    return sign ? -f : f;
  }
  memcpy(&f, &bits, 4);
  return f;
}

/*! nearest, ties to even */
uint16_t ToHalf(double v) {
  const float f = static_cast<float>(v);
  uint32_t b;
  memcpy(&b, &f, 4);
  const uint16_t sign = static_cast<uint16_t>((b >> 16) & 0x8000u);
  b &= 0x7fffffffu;
  if (b > 0x7f800000u) return sign | 0x7e00u;
  if (b >= 0x477ff000u) return sign | 0x7c00u;
  if (b < 0x38800000u) {  // below 2^-14: a multiple of 2^-24
    float mag;
    memcpy(&mag, &b, 4);
    return sign | static_cast<uint16_t>(std::nearbyint(mag * 16777216.0f));
  }
  const uint32_t odd = (b >> 13) & 1u;
  return sign | static_cast<uint16_t>((b - (112u << 23) + 0xfffu + odd) >> 13);
}

float FromBf16(uint16_t h) {
  const uint32_t bits = static_cast<uint32_t>(h) << 16;
  float f;
  memcpy(&f, &bits, 4);
  return f;
}

uint16_t ToBf16(double v) {
  const float f = static_cast<float>(v);
  uint32_t b;
  memcpy(&b, &f, 4);
  if ((b & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((b >> 16) | 0x40u);
  return static_cast<uint16_t>((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}

double LoadFloat(const LGBM_Array& a, int64_t at) {
  switch (a.type) {
    case C_API_DTYPE_FLOAT64: return static_cast<const double*>(a.data)[at];
    case C_API_DTYPE_FLOAT32: return static_cast<const float*>(a.data)[at];
    case C_API_DTYPE_FLOAT16: return FromHalf(static_cast<const uint16_t*>(a.data)[at]);
    case C_API_DTYPE_BFLOAT16: return FromBf16(static_cast<const uint16_t*>(a.data)[at]);
    case C_API_DTYPE_INT32: return static_cast<const int32_t*>(a.data)[at];
    default: return static_cast<double>(static_cast<const int64_t*>(a.data)[at]);
  }
}

/*! an integer, or an integer held in a floating type; what no int64 holds becomes -1 */
int64_t LoadInt(const LGBM_Array& a, int64_t at) {
  if (a.type == C_API_DTYPE_INT32) return static_cast<const int32_t*>(a.data)[at];
  if (a.type == C_API_DTYPE_INT64) return static_cast<const int64_t*>(a.data)[at];
  const double v = LoadFloat(a, at);
  return v >= 0 && v < 4e9 ? static_cast<int64_t>(v) : -1;
}

void StoreFloat(const LGBM_Array& a, int64_t at, double v) {
  switch (a.type) {
    case C_API_DTYPE_FLOAT64: static_cast<double*>(a.data)[at] = v; break;
    case C_API_DTYPE_FLOAT32: static_cast<float*>(a.data)[at] = static_cast<float>(v); break;
    case C_API_DTYPE_FLOAT16: static_cast<uint16_t*>(a.data)[at] = ToHalf(v); break;
    default: static_cast<uint16_t*>(a.data)[at] = ToBf16(v); break;
  }
}

void CopyElement(const LGBM_Array& to, int64_t i, const LGBM_Array& from, int64_t j) {
  const int64_t size = ElementSize(from.type);
  memcpy(static_cast<char*>(to.data) + i * size,
         static_cast<const char*>(from.data) + j * size, size);
}

/*! log(sum(exp(v))) of `n` values; -inf of none */
double LogSumExp(const double* v, size_t n) {
  double high = -kInf;
  for (size_t i = 0; i < n; ++i) high = std::max(high, v[i]);
  if (!(high > -kInf) || high == kInf) return high;
  double sum = 0;
  for (size_t i = 0; i < n; ++i) sum += std::exp(v[i] - high);
  return high + std::log(sum);
}

void CheckArray(const LGBM_Array& a, const char* what, bool optional, bool type_ok,
                const char* types) {
  if (a.data == nullptr) {
    if (!optional) Log::Fatal("%s is missing", what);
    return;
  }
  if (!type_ok) Log::Fatal("%s must be %s", what, types);
}

bool IsUniform(int type) {
  return type == C_API_DTYPE_FLOAT32 || type == C_API_DTYPE_FLOAT64;
}

constexpr const char* kFloats = "float64, float32, float16 or bfloat16";
constexpr const char* kInts = "int32 or int64";

void CheckClasses(int64_t rows, int classes) {
  if (rows < 0 || rows > INT32_MAX)
    Log::Fatal("the number of rows must be 0..2147483647, got %lld",
               static_cast<long long>(rows));
  if (classes < 1 || classes > kMaxClasses)
    Log::Fatal("the number of classes must be 1..%d, got %d", kMaxClasses, classes);
}

void CheckTemperature(double t) {
  // a float of its own and of its inverse, as the device computes with both
  if (!(t >= 1e-6 && t <= 1e6)) Log::Fatal("temperature must be in 1e-6..1e6, got %g", t);
}

/*! the threads of a call, and what each of them works in: made before they start, as memory that
 *  is not there ends a process that asks for it among them. kApart more elements than are used
 *  keep two threads' arrays, which stand next to each other, out of one line. */
constexpr int kApart = 32;
template <typename Scratch> std::vector<Scratch> ScratchOf(int64_t rows, const Scratch& one) {
  return std::vector<Scratch>(
      static_cast<size_t>(std::min<int64_t>(rows, omp_get_max_threads())), one);
}

// ------------------------------------------------------------------ host: top logits
struct TopScratch {
  std::vector<double> x, left;
  std::vector<int> order;
};

void TopLogitsHost(const LGBM_TopLogitsArgs& a) {
  const int c = a.classes, k = a.k;
  auto scratch = ScratchOf(a.rows, TopScratch{std::vector<double>(c + kApart),
                                              std::vector<double>(c + kApart),
                                              std::vector<int>(c + kApart)});
#pragma omp parallel num_threads(static_cast<int>(scratch.size()))
  {
    TopScratch& own = scratch[omp_get_thread_num()];
    double *const x = own.x.data(), *const left = own.left.data();
    int* const order = own.order.data();
#pragma omp for schedule(static)
    for (int64_t i = 0; i < a.rows; ++i) {
      const int64_t row = i * a.scores.stride[0];
      int n = 0;
      for (int j = 0; j < c; ++j) {
        x[j] = LoadFloat(a.scores, row + j * a.scores.stride[1]);
        if (x[j] > -kInf) order[n++] = j;  // neither -inf nor NaN
      }
      const int got = std::min(n, k);
      std::partial_sort(order, order + got, order + n,
                        [&](int p, int q) { return x[p] > x[q] || (x[p] == x[q] && p < q); });
      for (int j = 0; j < k; ++j) {
        const int64_t at = i * a.top_class.stride[0] + j * a.top_class.stride[1];
        const int64_t al = i * a.top_logit.stride[0] + j * a.top_logit.stride[1];
        static_cast<int32_t*>(a.top_class.data)[at] = j < got ? order[j] : -1;
        if (j < got) CopyElement(a.top_logit, al, a.scores, row + order[j] * a.scores.stride[1]);
        else StoreFloat(a.top_logit, al, -kInf);
      }
      if (a.log_rest.data != nullptr) {
        for (int j = got; j < n; ++j) left[j - got] = x[order[j]] / a.temperature;
        StoreFloat(a.log_rest, i * a.log_rest.stride[0], LogSumExp(left, n - got));
      }
    }
  }
}

// ------------------------------------------------------------------ host: distillation
struct DistillScratch {
  std::vector<double> z, e, e1, log_p, p;
  std::vector<int> slot, cls;
};

void DistillHost(const LGBM_DistillArgs& a) {
  const int c = a.classes, k = a.k;
  const double t = a.temperature, alpha = a.alpha;
  const double factor = c > 1 ? static_cast<double>(c) / (c - 1) : 1.0;
  const bool rest = a.teacher_rest.data != nullptr;
  const std::vector<double> wide(c + kApart), few(k + 1 + kApart);
  auto scratch = ScratchOf(a.rows, DistillScratch{wide, wide, wide, few, few,
                                                  std::vector<int>(c + kApart, -1),
                                                  std::vector<int>(k + kApart)});
#pragma omp parallel num_threads(static_cast<int>(scratch.size()))
  {
    DistillScratch& mine = scratch[omp_get_thread_num()];
    double *const z = mine.z.data(), *const e = mine.e.data(), *const e1 = mine.e1.data();
    double *const log_p = mine.log_p.data(), *const p = mine.p.data();
    int *const slot = mine.slot.data(), *const cls = mine.cls.data();
#pragma omp for schedule(static)
    for (int64_t i = 0; i < a.rows; ++i) {
      const double w = a.weight.data ? LoadFloat(a.weight, i * a.weight.stride[0]) : 1.0;
      auto put = [&](const LGBM_Array& to, int j, double v) {
        StoreFloat(to, i * to.stride[0] + j * to.stride[1], v);
      };
      double high = -kInf, total = 0, total1 = 0;
      bool live = w != 0.0;
      if (live) {
        for (int j = 0; j < c; ++j) {
          z[j] = LoadFloat(a.scores, i * a.scores.stride[0] + j * a.scores.stride[1]);
          if (z[j] > high) high = z[j];
        }
        const double base = high > -kInf ? high : 0.0;
        for (int j = 0; j < c; ++j) {
          e[j] = std::exp((z[j] - base) / t);
          e1[j] = std::exp(z[j] - base);
          total += e[j];
          total1 += e1[j];
        }
        if (total == 0.0) live = false;  // every class is masked
        high = base;
      }
      if (!live) {
        if (a.loss.data) StoreFloat(a.loss, i * a.loss.stride[0], 0.0);
        for (int j = 0; j < c; ++j) {
          if (a.gradient.data) put(a.gradient, j, 0.0);
          if (a.hessian.data) put(a.hessian, j, 0.0);
        }
        continue;
      }
      // the teacher: the first slot of a class counts
      int n = 0;
      for (int j = 0; j < k; ++j) {
        const int64_t y = LoadInt(a.teacher_class, i * a.teacher_class.stride[0] +
                                                       j * a.teacher_class.stride[1]);
        cls[j] = y >= 0 && y < c && slot[y] < 0 ? static_cast<int>(y) : -1;
        if (cls[j] < 0) continue;
        slot[y] = j;
        log_p[n++] = LoadFloat(a.teacher_logit, i * a.teacher_logit.stride[0] +
                                                    j * a.teacher_logit.stride[1]);
      }
      // against the largest logit first: over a small T a logit may be beyond 64 bits
      double top = -kInf;
      for (int j = 0; j < n; ++j) top = std::max(top, log_p[j]);
      const bool some = top > -kInf;
      if (!some) top = 0.0;
      for (int j = 0; j < n; ++j) log_p[j] = (log_p[j] - top) / t;
      const double r_read = rest ? LoadFloat(a.teacher_rest, i * a.teacher_rest.stride[0]) : -kInf;
      const double r = r_read == -kInf || !some ? r_read : r_read - top / t;
      log_p[n] = r;
      const double norm = LogSumExp(log_p, n + 1);
      bool nan = std::isnan(r) || norm == kInf;  // of infinite weights none is a share
      for (int j = 0; j < n; ++j) nan |= std::isnan(log_p[j]);
      const double lse = nan ? std::nan("") : norm;
      const bool taught = nan || norm > -kInf;
      double left = 0;
      for (int j = 0; j < c; ++j)
        if (slot[j] < 0) left += e[j];
      // where they underflow, the sum of the others is taken against their own maximum
      double log_left = std::log(left), own = high;
      if (rest && left < 1e-290) {
        own = -kInf;
        for (int j = 0; j < c; ++j)
          if (slot[j] < 0) own = std::max(own, z[j]);
        left = 0;
        for (int j = 0; j < c; ++j)
          if (slot[j] < 0 && own > -kInf) left += std::exp((z[j] - own) / t);
        log_left = left > 0 ? std::log(left) + (own - high) / t : -kInf;
      }
      double kl = 0;
      n = 0;
      for (int j = 0; j < k; ++j) {
        p[j] = 0;
        if (cls[j] < 0) continue;
        const double lp = log_p[n++] - lse;
        p[j] = std::exp(lp);
        if (!(p[j] == 0)) kl += p[j] * (lp - ((z[cls[j]] - high) / t - std::log(total)));
      }
      const double share = std::exp(r - lse);
      if (rest && !(share == 0)) kl += share * (r - lse - (log_left - std::log(total)));
      const double ratio = rest && left > 0 ? share / left : 0.0;
      const int64_t y = alpha < 1.0 ? LoadInt(a.label, i * a.label.stride[0]) : -1;
      const bool labelled = y >= 0 && y < c;
      if (a.loss.data) {
        double v = taught && alpha > 0 ? alpha * t * t * kl : 0.0;
        if (labelled) v += (1 - alpha) * (std::log(total1) - (z[y] - high));
        StoreFloat(a.loss, i * a.loss.stride[0], v * w);
      }
      if (a.gradient.data || a.hessian.data) {
        for (int j = 0; j < c; ++j) {
          double g = 0, h = 0;
          if (taught && alpha > 0) {
            const double q = e[j] / total;
            const double other = own == high ? e[j] : std::exp((z[j] - own) / t);
            g = alpha * t * (q - (slot[j] >= 0 ? p[slot[j]] : ratio == 0 ? 0.0 : ratio * other));
            h = alpha * q * (1 - q);
          }
          if (labelled) {
            const double q = e1[j] / total1;
            g += (1 - alpha) * (q - (j == y ? 1.0 : 0.0));
            h += (1 - alpha) * q * (1 - q);
          }
          if (a.gradient.data) put(a.gradient, j, g * w);
          if (a.hessian.data) put(a.hessian, j, h * factor * w);
        }
      }
      for (int j = 0; j < k; ++j)
        if (cls[j] >= 0) slot[cls[j]] = -1;
    }
  }
}

// ------------------------------------------------------------------ host: verification
/*! what counts as probability: NaN, infinities and negative values are none */
double Mass(double v) { return v > 0 && v <= DBL_MAX ? v : 0.0; }

int DrawClass(const double* mass, int classes, double total, double v) {
  const double goal = v * total;
  double reach = 0;
  int last = -1;
  for (int j = 0; j < classes; ++j) {
    if (mass[j] <= 0) continue;
    reach += mass[j];
    last = j;
    if (reach > goal) break;
  }
  return last;
}

void VerifyHost(const LGBM_VerifyArgs& a) {
  const int c = a.classes, t = a.drafts;
  auto scratch = ScratchOf(a.rows, std::vector<double>(c + kApart));
#pragma omp parallel num_threads(static_cast<int>(scratch.size()))
  {
    double* const mass = scratch[omp_get_thread_num()].data();
#pragma omp for schedule(static)
    for (int64_t i = 0; i < a.rows; ++i) {
      auto p = [&](int s, int64_t j) {
        return Mass(LoadFloat(a.target, i * a.target.stride[0] + s * a.target.stride[1] +
                                            j * a.target.stride[2]));
      };
      auto q = [&](int s, int64_t j) {
        return Mass(LoadFloat(a.draft_prob, i * a.draft_prob.stride[0] +
                                                s * a.draft_prob.stride[1] +
                                                j * a.draft_prob.stride[2]));
      };
      auto draft = [&](int s) {
        const int64_t x = LoadInt(a.draft_class, i * a.draft_class.stride[0] +
                                                     s * a.draft_class.stride[1]);
        return x >= 0 && x < c ? x : int64_t{-1};
      };
      auto out = [&](int s) -> int32_t& {
        return static_cast<int32_t*>(a.out_class.data)[i * a.out_class.stride[0] +
                                                       s * a.out_class.stride[1]];
      };
      int64_t len = t;
      if (a.length.data)
        len = std::max<int64_t>(0, std::min<int64_t>(t, LoadInt(a.length,
                                                                i * a.length.stride[0])));
      int s = 0;
      for (; s < len; ++s) {
        const int64_t x = draft(s);
        if (x < 0) break;
        const double u = LoadFloat(a.accept, i * a.accept.stride[0] + s * a.accept.stride[1]);
        if (!(u * (a.draft_prob.data ? q(s, x) : 1.0) < p(s, x))) break;
        out(s) = static_cast<int32_t>(x);
      }
      static_cast<int32_t*>(a.out_accepted.data)[i * a.out_accepted.stride[0]] = s;
      double total = 0;
      const int64_t x = s < len ? draft(s) : -1;
      for (int j = 0; j < c; ++j) {
        mass[j] = p(s, j);
        if (s < len) {
          if (a.draft_prob.data) mass[j] = std::max(0.0, mass[j] - q(s, j));
          else if (j == x) mass[j] = 0;
        }
        total += mass[j];
      }
      if (total == 0) {
        for (int j = 0; j < c; ++j) total += mass[j] = p(s, j);
      }
      out(s) = DrawClass(mass, c, total, LoadFloat(a.sample, i * a.sample.stride[0]));
      for (int j = s + 1; j <= t; ++j) out(j) = -1;
    }
  }
}

const DeviceOps& Device() {
  if (g_device_ops == nullptr) Log::Fatal("this build has no device operators");
  return *g_device_ops;
}

}  // namespace

// ------------------------------------------------------------------ checks
void Check(const LGBM_TopLogitsArgs& a) {
  CheckClasses(a.rows, a.classes);
  CheckTemperature(a.temperature);
  if (a.k < 1 || a.k > std::min(a.classes, kMaxTop))
    Log::Fatal("k must be 1..%d for %d classes, got %d", std::min(a.classes, kMaxTop), a.classes,
               a.k);
  if (a.rows == 0) return;
  CheckArray(a.scores, "scores", false, IsFloat(a.scores.type), kFloats);
  CheckArray(a.top_class, "top_class", false, a.top_class.type == C_API_DTYPE_INT32, "int32");
  CheckArray(a.top_logit, "top_logit", false, a.top_logit.type == a.scores.type,
             "of the scores' type");
  CheckArray(a.log_rest, "log_rest", true,
             a.log_rest.type == (a.scores.type == C_API_DTYPE_FLOAT64 ? C_API_DTYPE_FLOAT64
                                                                      : C_API_DTYPE_FLOAT32),
             "float64 for float64 scores, else float32");
}

void Check(const LGBM_DistillArgs& a) {
  CheckClasses(a.rows, a.classes);
  CheckTemperature(a.temperature);
  if (!(a.alpha >= 0.0 && a.alpha <= 1.0)) Log::Fatal("alpha must be in 0..1, got %g", a.alpha);
  if (a.k < 1 || a.k > kMaxTop)
    Log::Fatal("a teacher has 1..%d slots a row, got %d", kMaxTop, a.k);
  if (a.rows == 0) return;
  const int type = a.scores.type;
  const bool wide = type == C_API_DTYPE_FLOAT64;
  CheckArray(a.scores, "scores", false, IsFloat(type), kFloats);
  CheckArray(a.teacher_class, "teacher classes", false, IsInt(a.teacher_class.type), kInts);
  CheckArray(a.teacher_logit, "teacher logits", false, IsFloat(a.teacher_logit.type), kFloats);
  CheckArray(a.teacher_rest, "teacher log_rest", true, IsFloat(a.teacher_rest.type), kFloats);
  CheckArray(a.label, "labels", !(a.alpha < 1.0),
             IsInt(a.label.type) || a.label.type == C_API_DTYPE_FLOAT32,
             "int32, int64 or float32");
  CheckArray(a.weight, "weight", true, IsFloat(a.weight.type), kFloats);
  CheckArray(a.loss, "loss", true,
             a.loss.type == (wide ? C_API_DTYPE_FLOAT64 : C_API_DTYPE_FLOAT32),
             "float64 for float64 scores, else float32");
  const int out = wide ? C_API_DTYPE_FLOAT32 : type;
  const char* outs = "float32 for float64 scores, else of the scores' type";
  CheckArray(a.gradient, "gradient", true, a.gradient.type == out, outs);
  CheckArray(a.hessian, "hessian", true, a.hessian.type == out, outs);
  if (!a.loss.data && !a.gradient.data && !a.hessian.data)
    Log::Fatal("neither the loss nor the gradient nor the hessian is asked for");
}

void Check(const LGBM_VerifyArgs& a) {
  CheckClasses(a.rows, a.classes);
  if (a.drafts < 1 || a.drafts > kMaxDrafts)
    Log::Fatal("a sequence has 1..%d drafts, got %d", kMaxDrafts, a.drafts);
  if (a.rows == 0) return;
  CheckArray(a.target, "target probabilities", false, IsFloat(a.target.type), kFloats);
  CheckArray(a.draft_prob, "draft probabilities", true, a.draft_prob.type == a.target.type,
             "of the target's type");
  CheckArray(a.draft_class, "drafts", false, IsInt(a.draft_class.type), kInts);
  CheckArray(a.accept, "accept numbers", false, IsUniform(a.accept.type), "float32 or float64");
  CheckArray(a.sample, "sample numbers", false, IsUniform(a.sample.type), "float32 or float64");
  CheckArray(a.length, "lengths", true, IsInt(a.length.type), kInts);
  CheckArray(a.out_class, "out_class", false, a.out_class.type == C_API_DTYPE_INT32, "int32");
  CheckArray(a.out_accepted, "out_accepted", false, a.out_accepted.type == C_API_DTYPE_INT32,
             "int32");
}

// ------------------------------------------------------------------ dispatch
void TopLogits(const LGBM_TopLogitsArgs& a, int device, void* stream) {
  Check(a);
  if (a.rows == 0) return;
  if (device < 0) TopLogitsHost(a);
  else Device().top_logits(a, device, stream);
}

void Distill(const LGBM_DistillArgs& a, int device, void* stream) {
  Check(a);
  if (a.rows == 0) return;
  if (device < 0) DistillHost(a);
  else Device().distill(a, device, stream);
}

LGBM_DistillArgs DistillArgsOf(const Metadata& meta, data_size_t num_data, int num_class,
                               double temperature, double alpha, const double* score) {
  meta.CheckTeacher();
  LGBM_DistillArgs a{};
  a.rows = num_data;
  a.classes = num_class;
  a.k = meta.teacher_slots();
  a.temperature = temperature;
  a.alpha = alpha;
  a.scores = ArrayOf(score, C_API_DTYPE_FLOAT64, 1, num_data);
  a.teacher_class = ArrayOf(meta.teacher_class(), C_API_DTYPE_INT32, a.k, 1);
  a.teacher_logit = ArrayOf(meta.teacher_logit(), C_API_DTYPE_FLOAT32, a.k, 1);
  a.teacher_rest = ArrayOf(meta.teacher_rest(), C_API_DTYPE_FLOAT32, 1);
  a.label = ArrayOf(meta.label(), C_API_DTYPE_FLOAT32, 1);
  a.weight = ArrayOf(meta.weights(), C_API_DTYPE_FLOAT32, 1);
  return a;
}

int64_t VerifyWorkspace(const LGBM_VerifyArgs& a) {
  Check(a);
  return a.rows == 0 || g_device_ops == nullptr ? 0 : g_device_ops->verify_workspace(a);
}

void VerifyDrafts(const LGBM_VerifyArgs& a, int device, void* stream) {
  Check(a);
  if (a.rows == 0) return;
  if (device < 0) VerifyHost(a);
  else Device().verify(a, device, stream);
}

}  // namespace class_ops
}  // namespace migbm
