/*!
 * Operators over class scores and class probabilities: the top logits of a teacher,
 * the distillation loss on them with its gradient, and the verification of drafted
 * classes against a target's probabilities.
 *
 * The same arguments run on the host (OpenMP, 64-bit arithmetic) or on a HIP device; the
 * C ABI structs of c_api.h are the argument blocks of both.
 */
#ifndef MIGBM_CLASS_OPS_H_
#define MIGBM_CLASS_OPS_H_

#include "c_api.h"
#include "dataset.h"

namespace migbm {
namespace class_ops {

constexpr int kMaxTop = kMaxTeacherSlots;  //!< largest number of top logits a row may have
constexpr int kMaxClasses = 1 << 20;    //!< largest number of classes
constexpr int kMaxDrafts = 1024;        //!< largest number of drafted classes a sequence may have

inline int64_t ElementSize(int type) {
  switch (type) {
    case C_API_DTYPE_FLOAT64: case C_API_DTYPE_INT64: return 8;
    case C_API_DTYPE_FLOAT16: case C_API_DTYPE_BFLOAT16: return 2;
    default: return 4;
  }
}
inline bool IsFloat(int type) {
  return type == C_API_DTYPE_FLOAT32 || type == C_API_DTYPE_FLOAT64 ||
         type == C_API_DTYPE_FLOAT16 || type == C_API_DTYPE_BFLOAT16;
}
inline bool IsInt(int type) {
  return type == C_API_DTYPE_INT32 || type == C_API_DTYPE_INT64;
}

/*! Throws (Log::Fatal) unless the arguments are what the kernels assume. */
void Check(const LGBM_TopLogitsArgs& a);
void Check(const LGBM_DistillArgs& a);
void Check(const LGBM_VerifyArgs& a);

/*! device < 0: the host's memory; otherwise the memory of that HIP device, on `stream`. */
void TopLogits(const LGBM_TopLogitsArgs& a, int device, void* stream);
void Distill(const LGBM_DistillArgs& a, int device, void* stream);
void VerifyDrafts(const LGBM_VerifyArgs& a, int device, void* stream);
/*!
 * The distillation arguments of a dataset in the boosting engine's layout: class-major
 * float64 scores, float32 gradients, and the dataset's teacher, labels and weights in host
 * memory. The caller sets the outputs.
 */
LGBM_DistillArgs DistillArgsOf(const Metadata& meta, data_size_t num_data, int num_class,
                               double temperature, double alpha, const double* score);
inline LGBM_Array ArrayOf(const void* data, int type, int64_t s0, int64_t s1 = 0) {
  return LGBM_Array{const_cast<void*>(data), {s0, s1, 0}, type, 0};
}
/*! bytes of device scratch memory that VerifyDrafts needs (0: none) */
int64_t VerifyWorkspace(const LGBM_VerifyArgs& a);

/*! set when the device module is linked in */
struct DeviceOps {
  void (*top_logits)(const LGBM_TopLogitsArgs&, int, void*);
  void (*distill)(const LGBM_DistillArgs&, int, void*);
  void (*verify)(const LGBM_VerifyArgs&, int, void*);
  int64_t (*verify_workspace)(const LGBM_VerifyArgs&);
};
extern const DeviceOps* g_device_ops;

}  // namespace class_ops
}  // namespace migbm

#endif  // MIGBM_CLASS_OPS_H_
