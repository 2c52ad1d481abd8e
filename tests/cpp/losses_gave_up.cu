// The last kernel of the cross entropy's gradient behind a product whose bounded wait gave up: the status is put there by the host, no
// wait runs.  All of dX and dW is NaN then, and nothing of either otherwise.
#include <cmath>
#include <cstdio>
#include <vector>

#include "linear_ce_finish.cuh"

using namespace tcb200;

template <typename T>
static bool run(int status, bool with_dx, bool with_dw) {
  const int64_t n = 5, live = 3, d = 13, ld = 64, v = 700;
  lce::Head head{(int)live, status, 1.f, 1};
  const int place[n] = {0, -1, 1, 2, -1};
  std::vector<float> sums(pg::kTile * ld, 2.f);
  std::vector<T> dx(n * d), dw(v * d);
  for (auto& x : dw) x = T(3.f);
  lce::Rows r = {};
  float* dsums;
  T *ddx, *ddw;
  int *code, got = 0;
  cudaMalloc(&r.head, sizeof(head));
  cudaMalloc(&r.place, sizeof(place));
  cudaMalloc(&dsums, sums.size() * 4);
  cudaMalloc(&ddx, dx.size() * sizeof(T));
  cudaMalloc(&ddw, dw.size() * sizeof(T));
  cudaMalloc(&code, 4);
  cudaMemset(code, 0, 4);
  cudaMemcpy(r.head, &head, sizeof(head), cudaMemcpyHostToDevice);
  cudaMemcpy(r.place, place, sizeof(place), cudaMemcpyHostToDevice);
  cudaMemcpy(dsums, sums.data(), sums.size() * 4, cudaMemcpyHostToDevice);
  cudaMemcpy(ddw, dw.data(), dw.size() * sizeof(T), cudaMemcpyHostToDevice);
  if (launch_pdl(lce::finish_kernel<T>, dim3(2), dim3(256), 0, nullptr, r, (const float*)dsums, ld, n, d, 1.f, with_dx ? ddx : (T*)nullptr,
                 with_dw ? ddw : (T*)nullptr, v * d, code) != cudaSuccess)
    return false;
  if (cudaDeviceSynchronize() != cudaSuccess) return false;
  cudaMemcpy(dx.data(), ddx, dx.size() * sizeof(T), cudaMemcpyDeviceToHost);
  cudaMemcpy(dw.data(), ddw, dw.size() * sizeof(T), cudaMemcpyDeviceToHost);
  cudaMemcpy(&got, code, 4, cudaMemcpyDeviceToHost);
  bool ok = got == status;
  for (int64_t i = 0; with_dx && i < n * d; ++i) {
    const float x = (float)dx[i];
    ok &= status ? std::isnan(x) : x == (place[i / d] < 0 ? 0.f : 2.f);
  }
  for (int64_t i = 0; i < v * d; ++i) {
    const float x = (float)dw[i];
    ok &= status && with_dw ? std::isnan(x) : x == 3.f;
  }
  for (void* p : {(void*)r.head, (void*)r.place, (void*)dsums, (void*)ddx, (void*)ddw, (void*)code}) cudaFree(p);
  return ok;
}

int main() {
  int devices = 0;
  if (cudaGetDeviceCount(&devices) != cudaSuccess) devices = 0;
  if (devices > 0)
    for (int status : {0, 24})
      for (int which = 1; which < 4; ++which)
        if (!run<float>(status, which & 1, which & 2) || !run<__half>(status, which & 1, which & 2) || !run<__nv_bfloat16>(status, which & 1, which & 2)) {
          std::printf("FAILED: status %d, outputs %d\n", status, which);
          return 1;
        }
  std::printf("gave up ok (gpu=%d)\n", devices > 0);
  return 0;
}
