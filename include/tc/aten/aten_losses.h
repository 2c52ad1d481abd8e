// Losses of a large-vocabulary head on at::Tensors: the ATen face of tcb200_linear_ce_* and tcb200_topk_distill_*.
//
//   auto r = tc::aten::linearCrossEntropy(X, W, target);              // {loss [N], lse [N]}
//   auto g = tc::aten::linearCrossEntropyBackward(X, W, target, r[1], gradLoss);   // {dX, dW}
//
// The reference's operator library ends at the layers (tc/library); these follow its ATen entry points: checks that throw,
// outputs on the device of the inputs, work on a caller's stream, no synchronisation.  The stream is ATen's current one of the
// inputs' device, or the one that the call names, which is then ATen's current stream for the length of the call: copies,
// kernels and the memory of outputs and scratch all follow its order.  Scratch memory comes from ATen's allocator, call by
// call, so calls on different streams or in different captured graphs share none.  As with every ATen operator, inputs made on
// another stream, and results read on one, need that stream's order (an event, recordStream).
#pragma once

#include <ATen/ATen.h>

#include <cmath>
#include <limits>
#include <optional>
#include <vector>

#include "tc/core/check.h"
#include "tc/core/cuda/cuda.h"
#include "tcb200.h"

// ATen's current stream through libtorch's C interface, which needs no CUDA headers (each returns 0 on success).
struct CUDAStreamGuardOpaque;
extern "C" {
int32_t aoti_torch_get_current_cuda_stream(int32_t device, void** stream);
int32_t aoti_torch_create_cuda_stream_guard(void* stream, int32_t device, CUDAStreamGuardOpaque** guard);
int32_t aoti_torch_delete_cuda_stream_guard(CUDAStreamGuardOpaque* guard);
}

namespace tc {
namespace aten {
namespace detail {

inline int32_t lossType(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return TCB200_F32;
    case at::kHalf: return TCB200_F16;
    case at::kBFloat16: return TCB200_BF16;
    default: TC_CHECK(false) << what << " must be float32, float16 or bfloat16"; return -1;
  }
}

inline void lossMatrix(const at::Tensor& t, const char* what, const at::Tensor& like) {
  TC_CHECK(t.is_cuda()) << what << " must be a CUDA tensor";
  TC_CHECK(t.get_device() == like.get_device()) << what << " is on another device";
  TC_CHECK(!t.is_neg()) << what << " is a negated view: call resolve_neg() first";
  TC_CHECK_EQ(t.dim(), 2) << what << " must have two dimensions";
  TC_CHECK(t.size(1) <= 1 || t.stride(1) == 1) << what << " must be dense along its last dimension";
  TC_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1)) << what << " has overlapping rows";
}
// Elements between rows; what a single row (or none) says does not matter.
inline int64_t lossRowStride(const at::Tensor& t) { return t.size(0) <= 1 ? std::max<int64_t>(t.size(1), 1) : t.stride(0); }

inline int32_t lossIndexBytes(const at::Tensor& t, const char* what) {
  TC_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) << what << " must be int32 or int64";
  return t.scalar_type() == at::kLong ? 8 : 4;
}

// One value a row, any stride (0: one value for all rows).
inline int64_t lossGradStride(const at::Tensor& g, int64_t n, const at::Tensor& like) {
  TC_CHECK(g.is_cuda() && g.get_device() == like.get_device()) << "the gradient of the loss is on another device";
  TC_CHECK(g.scalar_type() == at::kFloat) << "the gradient of the loss must be float32";
  TC_CHECK(g.dim() == 1 && g.size(0) == n) << "the gradient of the loss must have one value a row";
  return n <= 1 ? 0 : g.stride(0);
}

inline void lossStatus(int st, const char* what) { TC_CHECK(st == TCB200_OK) << what << ": " << tcb200_strerror(st); }

// The stream of a call, ATen's current one while this lives.
class LossStream {
 public:
  LossStream(const at::Tensor& like, const std::optional<tcb200_stream_t>& named) {
    const int32_t device = static_cast<int32_t>(like.get_device());
    void* current = nullptr;
    TC_CHECK(aoti_torch_get_current_cuda_stream(device, &current) == 0) << "no current CUDA stream";
    stream_ = static_cast<tcb200_stream_t>(current);
    if (!named) return;
    // handles that CUDA reserves for the default stream and for the calling thread's own
    const auto legacy = reinterpret_cast<tcb200_stream_t>(1), perThread = reinterpret_cast<tcb200_stream_t>(2);
    // ATen's allocator knows a stream by its handle, and this one is another stream in every thread
    TC_CHECK(*named != perThread) << "cudaStreamPerThread is not supported: pass a stream of your own";
    const tcb200_stream_t s = *named == legacy ? nullptr : *named;
    if (s == stream_) return;
    TC_CHECK(aoti_torch_create_cuda_stream_guard(s, device, &guard_) == 0) << "the stream cannot be made ATen's current one";
    stream_ = s;
  }
  ~LossStream() {
    if (guard_) aoti_torch_delete_cuda_stream_guard(guard_);
  }
  LossStream(const LossStream&) = delete;
  LossStream& operator=(const LossStream&) = delete;
  operator tcb200_stream_t() const { return stream_; }

 private:
  tcb200_stream_t stream_;
  CUDAStreamGuardOpaque* guard_ = nullptr;
};

inline tcb200_linear_ce_t linearCe(const at::Tensor& X, const at::Tensor& W, const at::Tensor& target, int64_t ignoreIndex) {
  lossMatrix(X, "X", X);
  lossMatrix(W, "W", X);
  TC_CHECK(X.scalar_type() == W.scalar_type()) << "X and W must have the same type";
  TC_CHECK_EQ(X.size(1), W.size(1)) << "X [N, D] and W [V, D] must agree in D";
  TC_CHECK(X.size(1) >= 1 && W.size(0) >= 1) << "X [N, D] and W [V, D] need D >= 1 and V >= 1";
  TC_CHECK(target.is_cuda() && target.get_device() == X.get_device()) << "target is on another device";
  TC_CHECK(target.dim() == 1 && target.size(0) == X.size(0)) << "target must have one index a row of X";
  tcb200_linear_ce_t p = {};
  p.N = X.size(0);
  p.D = X.size(1);
  p.V = W.size(0);
  p.ldx = lossRowStride(X);
  p.ldw = lossRowStride(W);
  p.ignore_index = ignoreIndex;
  p.dtype = lossType(X, "X");
  p.index_bytes = lossIndexBytes(target, "target");
  p.pack_w = p.ldw * W.element_size() % 16 != 0 || reinterpret_cast<uintptr_t>(W.data_ptr()) % 16 != 0;
  return p;
}

inline tcb200_topk_distill_t topkDistill(const at::Tensor& logits, const at::Tensor& indices, const at::Tensor& teacher,
                                         double temperature) {
  lossMatrix(logits, "logits", logits);
  lossMatrix(indices, "indices", logits);
  lossMatrix(teacher, "teacher", logits);
  TC_CHECK(indices.sizes() == teacher.sizes()) << "indices and teacher must have the same sizes";
  TC_CHECK_EQ(indices.size(0), logits.size(0)) << "indices and teacher must have one row a row of logits";
  TC_CHECK(logits.size(1) >= 1) << "logits [N, V] needs V >= 1";
  TC_CHECK(indices.size(1) >= 1 && indices.size(1) <= TCB200_TOPK_MAX) << "a row must have 1 to " << TCB200_TOPK_MAX << " entries";
  const float t = static_cast<float>(temperature);
  TC_CHECK(t > 0.f && std::isfinite(t)) << "the temperature must be positive and finite";
  TC_CHECK(std::isnormal(t * t)) << "the temperature's square must be a normal float32 number";
  tcb200_topk_distill_t p = {};
  p.N = logits.size(0);
  p.V = logits.size(1);
  p.K = indices.size(1);
  p.ld_logits = lossRowStride(logits);
  p.ld_indices = lossRowStride(indices);
  p.ld_teacher = lossRowStride(teacher);
  p.temperature = t;
  p.logits_dtype = lossType(logits, "logits");
  p.teacher_dtype = lossType(teacher, "teacher");
  p.index_bytes = lossIndexBytes(indices, "indices");
  return p;
}

}  // namespace detail

// Softmax cross entropy of z = X W^T against `target`, without keeping z: {loss [N], lse [N]}, float32.
inline std::vector<at::Tensor> linearCrossEntropy(const at::Tensor& X, const at::Tensor& W, const at::Tensor& target,
                                                  int64_t ignoreIndex = -100, std::optional<tcb200_stream_t> stream = std::nullopt) {
  const tcb200_linear_ce_t p = detail::linearCe(X, W, target, ignoreIndex);
  WithCudaDevice dev((size_t)X.get_device());
  const detail::LossStream on(X, stream);
  const at::Tensor t = target.contiguous();
  auto f32 = X.options().dtype(at::kFloat).requires_grad(false);
  at::Tensor loss = at::empty({p.N}, f32), lse = at::empty({p.N}, f32);
  int64_t bytes = 0;
  detail::lossStatus(tcb200_linear_ce_workspace(&p, &bytes, nullptr), "linearCrossEntropy");
  at::Tensor ws = at::empty({bytes}, X.options().dtype(at::kByte).requires_grad(false));
  detail::lossStatus(tcb200_linear_ce_forward(&p, X.data_ptr(), W.data_ptr(), t.data_ptr(), loss.data_ptr<float>(),
                                              lse.data_ptr<float>(), ws.data_ptr(), bytes, on, nullptr),
                     "linearCrossEntropy");
  return {loss, lse};
}

// Its gradients {dX, dW} for the gradient of the loss (one value a row); one that is not needed comes back undefined.
inline std::vector<at::Tensor> linearCrossEntropyBackward(const at::Tensor& X, const at::Tensor& W, const at::Tensor& target,
                                                          const at::Tensor& lse, const at::Tensor& gradLoss,
                                                          int64_t ignoreIndex = -100, bool needX = true, bool needW = true,
                                                          std::optional<tcb200_stream_t> stream = std::nullopt) {
  const tcb200_linear_ce_t p = detail::linearCe(X, W, target, ignoreIndex);
  TC_CHECK(lse.is_cuda() && lse.get_device() == X.get_device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
           lse.numel() == p.N) << "lse must be the second result of linearCrossEntropy";
  WithCudaDevice dev((size_t)X.get_device());
  const detail::LossStream on(X, stream);
  const at::Tensor t = target.contiguous(), g = gradLoss.resolve_neg();  // (a view that stands for its negative is copied)
  const int64_t stride = detail::lossGradStride(g, p.N, X);
  auto like = X.options().requires_grad(false);
  at::Tensor dX, dW;
  if (needX) dX = at::empty({p.N, p.D}, like);
  if (needW) dW = at::empty({p.V, p.D}, like);
  int64_t bytes = 0;
  detail::lossStatus(tcb200_linear_ce_workspace(&p, nullptr, &bytes), "linearCrossEntropyBackward");
  at::Tensor ws = at::empty({bytes}, like.dtype(at::kByte));
  detail::lossStatus(tcb200_linear_ce_backward(&p, X.data_ptr(), W.data_ptr(), t.data_ptr(), lse.data_ptr<float>(),
                                               g.data_ptr<float>(), stride, needX ? dX.data_ptr() : nullptr,
                                               needW ? dW.data_ptr() : nullptr, ws.data_ptr(), bytes, on, nullptr),
                     "linearCrossEntropyBackward");
  return {dX, dW};
}

// Distillation of `logits` [N, V] from a teacher's logits [N, K] at `indices`: {loss [N], stats [N, 3]}, float32.
inline std::vector<at::Tensor> topkDistillation(const at::Tensor& logits, const at::Tensor& indices, const at::Tensor& teacher,
                                                double temperature = 1.0, std::optional<tcb200_stream_t> stream = std::nullopt) {
  const tcb200_topk_distill_t p = detail::topkDistill(logits, indices, teacher, temperature);
  WithCudaDevice dev((size_t)logits.get_device());
  const detail::LossStream on(logits, stream);
  auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  at::Tensor loss = at::empty({p.N}, f32), stats = at::empty({p.N, 3}, f32);
  detail::lossStatus(tcb200_topk_distill_forward(&p, logits.data_ptr(), indices.data_ptr(), teacher.data_ptr(),
                                                 loss.data_ptr<float>(), stats.data_ptr<float>(), on),
                     "topkDistillation");
  return {loss, stats};
}

// Its gradient with respect to the logits.
inline at::Tensor topkDistillationBackward(const at::Tensor& logits, const at::Tensor& indices, const at::Tensor& teacher,
                                           const at::Tensor& stats, const at::Tensor& gradLoss, double temperature = 1.0,
                                           std::optional<tcb200_stream_t> stream = std::nullopt) {
  const tcb200_topk_distill_t p = detail::topkDistill(logits, indices, teacher, temperature);
  TC_CHECK(stats.is_cuda() && stats.get_device() == logits.get_device() && stats.scalar_type() == at::kFloat &&
           stats.is_contiguous() && stats.numel() == 3 * p.N) << "stats must be the second result of topkDistillation";
  WithCudaDevice dev((size_t)logits.get_device());
  const detail::LossStream on(logits, stream);
  const at::Tensor g = gradLoss.resolve_neg();
  const int64_t stride = detail::lossGradStride(g, p.N, logits);
  at::Tensor d = at::empty({p.N, p.V}, logits.options().requires_grad(false));
  detail::lossStatus(tcb200_topk_distill_backward(&p, logits.data_ptr(), indices.data_ptr(), teacher.data_ptr(),
                                                  stats.data_ptr<float>(), g.data_ptr<float>(), stride, d.data_ptr(),
                                                  on),
                     "topkDistillationBackward");
  return d;
}

}  // namespace aten
}  // namespace tc
