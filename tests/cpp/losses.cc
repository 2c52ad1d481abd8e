// tc::aten::linearCrossEntropy / topkDistillation and their backward calls from a C++ program, against ATen in 64 bits.
// Without a device: the calls refuse CPU tensors.
#include <ATen/ATen.h>

#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <string>

#include "tc/aten/aten_losses.h"

static void expect(bool ok, const char* what) {
  if (!ok) {
    std::fprintf(stderr, "FAILED: %s\n", what);
    std::exit(1);
  }
}
static double worst(const at::Tensor& a, const at::Tensor& b) { return (a.to(at::kDouble) - b).abs().max().item<double>(); }

int main() {
  int devices = 0;
  const bool gpu = tcb200_device_count(&devices) == TCB200_OK && devices > 0;
  const auto cpu = at::TensorOptions().dtype(at::kFloat);
  std::string said;
  try {
    tc::aten::linearCrossEntropy(at::zeros({2, 4}, cpu), at::zeros({3, 4}, cpu), at::zeros({2}, cpu.dtype(at::kLong)));
  } catch (const std::runtime_error& e) {
    said = e.what();
  }
  expect(said.find("X must be a CUDA tensor") != std::string::npos, "CPU tensors are refused");
  if (gpu) {
    const auto dev = cpu.device(at::kCUDA);
    const int64_t n = 70, d = 96, v = 500, k = 9;
    const at::Tensor X = at::randn({n, d}, dev), W = at::randn({v, d}, dev) / 10, g = at::rand({n}, dev);
    const at::Tensor t = at::randint(v, {n}, dev.dtype(at::kLong));
    const auto r = tc::aten::linearCrossEntropy(X, W, t);
    const auto b = tc::aten::linearCrossEntropyBackward(X, W, t, r[1], g);
    const at::Tensor logp = at::log_softmax(X.to(at::kDouble).matmul(W.to(at::kDouble).t()), 1);
    const at::Tensor dz = (logp.exp() - at::one_hot(t, v).to(at::kDouble)) * g.to(at::kDouble).unsqueeze(1);
    // values of order one, float32: well inside 2^-16
    expect(worst(r[0], -logp.gather(1, t.unsqueeze(1)).squeeze(1)) < 1.5e-5, "loss");
    expect(worst(b[0], dz.matmul(W.to(at::kDouble))) < 1.5e-5, "dX");
    expect(worst(b[1], dz.t().matmul(X.to(at::kDouble))) < 1.5e-4, "dW");  // sums of 70 values of up to 4
    const auto only = tc::aten::linearCrossEntropyBackward(X, W, t, r[1], g, -100, false, true);
    expect(!only[0].defined() && at::equal(only[1], b[1]), "dW alone");

    const at::Tensor z = at::randn({n, v}, dev), s = at::randn({n, k}, dev);
    const at::Tensor i = at::rand({n, v}, dev).argsort(int64_t{1}).slice(1, 0, k).contiguous();
    const auto q = tc::aten::topkDistillation(z, i, s, 2.0);
    const at::Tensor dl = tc::aten::topkDistillationBackward(z, i, s, q[1], g, 2.0);
    const at::Tensor lq = at::log_softmax(s.to(at::kDouble) / 2, 1), lp = at::log_softmax(z.to(at::kDouble) / 2, 1);
    expect(worst(q[0], 4 * (lq.exp() * (lq - lp.gather(1, i))).sum(1)) < 1.5e-5, "distillation loss");
    const at::Tensor spread = at::zeros_like(lp).scatter_add(1, i, lq.exp());
    expect(worst(dl, 2 * g.to(at::kDouble).unsqueeze(1) * (lp.exp() - spread)) < 1.5e-5, "dlogits");
  }
  std::printf("losses ok (gpu=%d)\n", gpu ? 1 : 0);
  return 0;
}
