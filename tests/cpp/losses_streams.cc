// The losses on a stream that the call names, another than ATen's current one: copies, kernels and the memory of outputs and scratch
// follow that stream.  Without a device: nothing to run.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
#include <vector>

#include "tc/aten/aten_losses.h"

static void expect(bool ok, const char* what) {
  if (!ok) {
    std::fprintf(stderr, "FAILED: %s\n", what);
    std::exit(1);
  }
}

struct Problem {
  at::Tensor X, W, t, g, z, i, s;
};
static Problem make(int64_t n, int64_t d, int64_t v, int64_t k) {
  const auto dev = at::TensorOptions().dtype(at::kFloat).device(at::kCUDA);
  return {at::randn({n, d}, dev).to(at::kBFloat16),
          (at::randn({v, d}, dev) / 10).to(at::kBFloat16),
          at::randint(v, {n, 2}, dev.dtype(at::kLong)).select(1, 0),  // strided: the call copies it
          at::rand({n}, dev),
          at::randn({n, v}, dev),
          at::rand({n, v}, dev).argsort(int64_t{1}).slice(1, 0, k).contiguous(),
          at::randn({n, k}, dev)};
}
using Named = std::optional<tcb200_stream_t>;
static std::vector<at::Tensor> step(const Problem& p, Named s) {
  auto r = tc::aten::linearCrossEntropy(p.X, p.W, p.t, -100, s);
  auto b = tc::aten::linearCrossEntropyBackward(p.X, p.W, p.t, r[1], p.g, -100, true, true, s);
  auto q = tc::aten::topkDistillation(p.z, p.i, p.s, 2.0, s);
  return {r[0], b[0], b[1], q[0], tc::aten::topkDistillationBackward(p.z, p.i, p.s, q[1], p.g, 2.0, s)};
}
static bool same(const std::vector<at::Tensor>& a, const std::vector<at::Tensor>& b) {
  for (size_t k = 0; k < a.size(); ++k)
    if (!at::equal(a[k], b[k])) return false;
  return true;
}
// some milliseconds of work on the current stream
static void delay(at::Tensor& a) {
  for (int k = 0; k < 20; ++k) at::mm_out(a, a.clone(), a.clone());
}

int main() {
  int devices = 0;
  const bool gpu = tcb200_device_count(&devices) == TCB200_OK && devices > 0;
  if (gpu) {
    const Problem p = make(600, 192, 3000, 12), o = make(500, 256, 2800, 9);
    const auto want = step(p, std::nullopt), other = step(o, std::nullopt);
    at::Tensor slow = at::zeros({4096, 4096}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA));
    const auto s1 = c10::cuda::getStreamFromPool(), s2 = c10::cuda::getStreamFromPool();
    const auto all = [] { expect(cudaDeviceSynchronize() == cudaSuccess, "the device"); };
    all();

    // two streams at once, neither of them current: scratch memory of their own
    for (int round = 0; round < 10; ++round) {
      const auto a = step(p, s1.stream());
      const auto b = step(o, s2.stream());
      all();
      expect(same(a, want) && same(b, other), "two streams at once");
    }
    expect(c10::cuda::getCurrentCUDAStream() == c10::cuda::getDefaultCUDAStream(), "the current stream is as it was");

    // inputs that the named stream has yet to write, and memory of the current stream that is taken and written meanwhile
    for (int round = 0; round < 3; ++round) {
      Problem late = p;
      const at::Tensor t = at::zeros({600, 2}, p.t.options());
      late.t = t.select(1, 0);
      all();
      {
        c10::cuda::CUDAStreamGuard on(s1);
        delay(slow);
        late.t.copy_(p.t);
      }
      const auto a = step(late, s1.stream());
      std::vector<at::Tensor> taken;
      for (int64_t bytes = 1 << 10; bytes <= (int64_t)64 << 20; bytes *= 2)
        for (int k = 0; k < 3; ++k) taken.push_back(at::full({bytes}, 255, p.X.options().dtype(at::kByte)));
      all();
      expect(same(a, want), "late inputs and memory of the current stream");
    }

    // no stream named: ATen's current one
    {
      Problem late = p;
      const at::Tensor t = at::zeros({600, 2}, p.t.options());
      late.t = t.select(1, 0);
      all();
      c10::cuda::CUDAStreamGuard on(s2);
      delay(slow);
      late.t.copy_(p.t);
      const auto a = step(late, std::nullopt);
      all();
      expect(same(a, want), "the current stream");
      // the default stream by its two names, while another one is current
      const auto b = step(p, Named(nullptr)), c = step(p, Named(cudaStreamLegacy));
      all();
      expect(same(b, want) && same(c, want), "the default stream by name");
      expect(c10::cuda::getCurrentCUDAStream() == s2, "the current stream is as it was");
    }
    std::string said;
    try {
      step(p, Named(cudaStreamPerThread));
    } catch (const std::runtime_error& e) {
      said = e.what();
    }
    expect(said.find("cudaStreamPerThread") != std::string::npos, "the per-thread stream is refused");
    all();
  }
  std::printf("losses on streams ok (gpu=%d)\n", gpu ? 1 : 0);
  return 0;
}
