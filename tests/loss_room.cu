// The product that keeps sums of logits writes where its caller has room, and is refused where that is less than its tiles take.
#include <stdio.h>
#include <string.h>

#include "hc_gemm.cuh"

extern "C" int fake_launches();

int main() {
  for (int64_t k : {64, 1024, 1025, 4096})
    for (int64_t m : {17, 128, 257, 5000})
      for (int64_t n : {1, 100, 1000, 50257}) {
        hc::GemmCall c;
        memset(&c, 0, sizeof(c));
        c.type = 1, c.m = m, c.n = n, c.k = k, c.batch = 1;
        c.a = c.b = {reinterpret_cast<void*>(1 << 20), (k + 7) / 8 * 8, 0, true};
        c.loss.sums = reinterpret_cast<float2*>(1 << 20);
        const int before = fake_launches();
        c.loss.stretches = hc::gemm_loss_stretches(m, n, k) - 1;
        if (hc::launch_loss_sums(c, nullptr) == cudaSuccess || fake_launches() != before) return printf("%d x %d x %d: launched without room\n", (int)m, (int)n, (int)k), 1;
        ++c.loss.stretches;
        if (hc::launch_loss_sums(c, nullptr) != cudaSuccess || fake_launches() != before + 1) return printf("%d x %d x %d: not launched\n", (int)m, (int)n, (int)k), 1;
      }
  puts("ok");
}
