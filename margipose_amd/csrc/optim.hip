// SGD with momentum over every parameter of the model in ONE launch, hyper-parameters in device memory (gfx950).
//
// Replaces torch.optim.SGD(params, lr, momentum).step() of the reference's training pass (src/margipose/bin/train_3d.py:186,
// :339; the 1cycle policy of hyperparam_scheduler.py:6-42 changes lr AND momentum every batch).  Reading lr / momentum from
// device memory is what lets the whole iteration (forward, loss, backward, update) be replayed as one HIP graph while the
// schedule keeps moving: the host only refreshes three floats per step.  Arithmetic identical to torch (no dampening, no
// weight decay, no Nesterov):   buf = g (first step) | fma(momentum, buf, g) ;   p = fma(-lr, buf, p)  -- one rounding each,
// where torch's unfused path rounds the product first: the two agree to an ulp per step, not bit for bit.
#include "common.h"

namespace mpose {
namespace {

__global__ __launch_bounds__(256) void sgd_step_k(const mpose_sgd_job* __restrict__ jobs, const float* __restrict__ hyper) {
  const mpose_sgd_job j = jobs[blockIdx.y];
  const float lr = hyper[0], mom = hyper[1];
  const bool first = hyper[2] != 0.f;
  const long n4 = j.n >> 2;
  float4* p4 = reinterpret_cast<float4*>(j.p);
  const float4* g4 = reinterpret_cast<const float4*>(j.g);
  float4* b4 = reinterpret_cast<float4*>(j.buf);
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long)gridDim.x * 256) {
    const float4 g = g4[i];
    float4 b = g;
    if (!first) {
      const float4 o = b4[i];
      b.x = fmaf(mom, o.x, g.x); b.y = fmaf(mom, o.y, g.y); b.z = fmaf(mom, o.z, g.z); b.w = fmaf(mom, o.w, g.w);
    }
    b4[i] = b;
    float4 p = p4[i];
    p.x = fmaf(-lr, b.x, p.x); p.y = fmaf(-lr, b.y, p.y); p.z = fmaf(-lr, b.z, p.z); p.w = fmaf(-lr, b.w, p.w);
    p4[i] = p;
  }
  if (blockIdx.x == 0) {
    for (long i = (n4 << 2) + threadIdx.x; i < j.n; i += 256) {
      const float g = j.g[i];
      const float b = first ? g : fmaf(mom, j.buf[i], g);
      j.buf[i] = b;
      j.p[i] = fmaf(-lr, b, j.p[i]);
    }
  }
}

__global__ void set4_k(float* dst, float a, float b, float c, float d) {
  dst[0] = a; dst[1] = b; dst[2] = c; dst[3] = d;
}

}  // namespace
}  // namespace mpose

using namespace mpose;

// dst[0..3] = {a, b, c, d}: the values travel as kernel arguments (captured at enqueue time), so the host may run any number
// of steps ahead of the device without a staging buffer being overwritten under a pending copy.
extern "C" int mpose_set4(float* dst, float a, float b, float c, float d, void* stream) {
  if (!dst) return MPOSE_EINVAL;
  launch(set4_k, dim3(1), dim3(1), 0, (hipStream_t)stream, dst, a, b, c, d);
  return launch_status();
}

extern "C" int mpose_sgd_step(const mpose_sgd_job* jobs_dev, int n_jobs, int64_t max_n, const float* hyper_dev, void* stream) {
  if (n_jobs <= 0) return 0;
  if (!jobs_dev || !hyper_dev || max_n < 0) return MPOSE_EINVAL;
  long bx = (max_n / 4 + 256 * 4 - 1) / (256 * 4);
  if (bx < 1) bx = 1;
  if (bx > 64) bx = 64;
  launch(sgd_step_k, dim3(dim3((unsigned)bx, (unsigned)n_jobs)), dim3(256), 0, (hipStream_t)stream, jobs_dev, hyper_dev);
  return launch_status();
}

// ---- AdamW ----
// m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr c1 m / (sqrt(v) c2 + eps): 28 bytes per element and one pass, so
// the rate of a large copy bounds it.  The arrays' addresses travel as kernel arguments, 384 arrays a launch (a table in device
// memory would need an upload whenever a gradient moves, and could not be captured).
namespace mpose {
namespace {

constexpr int kAdamJobs = 384;
constexpr int kAdamChunk = 4096;
struct AdamArgs {
  mpose_adamw_job j[kAdamJobs];
  float h[8];
  const float* hyper_dev;
  int n;
};

__global__ __launch_bounds__(256) void adamw_step_k(AdamArgs a) {
  const mpose_adamw_job j = a.j[blockIdx.y];
  const float* hp = a.hyper_dev;
  float h[7];
#pragma unroll
  for (int i = 0; i < 7; ++i) h[i] = hp != nullptr ? hp[i] : a.h[i];
  const float lr = h[0], b1 = h[1], b2 = h[2], eps = h[3], keep = 1.f - lr * h[4], step = lr * h[5], c2 = h[6];
  auto one = [&](float& p, float g, float& m, float& v) {
    m = fmaf(b1, m, (1.f - b1) * g);
    v = fmaf(b2, v, (1.f - b2) * g * g);
    p = fmaf(p, keep, -step * m / fmaf(sqrtf(v), c2, eps));
  };
  const bool vec = (((uintptr_t)j.p | (uintptr_t)j.g | (uintptr_t)j.m | (uintptr_t)j.v) & 15) == 0;
  for (int64_t lo = (int64_t)blockIdx.x * kAdamChunk; lo < j.n; lo += (int64_t)gridDim.x * kAdamChunk) {
    const int64_t hi = lo + kAdamChunk < j.n ? lo + kAdamChunk : j.n;
    for (int q = 0; q < kAdamChunk / 1024; ++q) {
      const int64_t i = lo + q * 1024 + threadIdx.x * 4;
      if (vec && i + 4 <= hi) {
        float4 p = *reinterpret_cast<float4*>(j.p + i), m = *reinterpret_cast<float4*>(j.m + i), v = *reinterpret_cast<float4*>(j.v + i);
        const float4 g = *reinterpret_cast<const float4*>(j.g + i);
        one(p.x, g.x, m.x, v.x); one(p.y, g.y, m.y, v.y); one(p.z, g.z, m.z, v.z); one(p.w, g.w, m.w, v.w);
        *reinterpret_cast<float4*>(j.p + i) = p; *reinterpret_cast<float4*>(j.m + i) = m; *reinterpret_cast<float4*>(j.v + i) = v;
      } else {
        for (int64_t k = i; k < i + 4 && k < hi; ++k) one(j.p[k], j.g[k], j.m[k], j.v[k]);
      }
    }
  }
}

struct Eight { float v[8]; };
__global__ void set8_k(float* dst, Eight e) { if (threadIdx.x < 8) dst[threadIdx.x] = e.v[threadIdx.x]; }

}  // namespace
}  // namespace mpose

extern "C" int mpose_set8(float* dst, const float* src8, void* stream) {
  if (!dst || !src8) return MPOSE_EINVAL;
  Eight e;
  for (int i = 0; i < 8; ++i) e.v[i] = src8[i];
  launch(set8_k, dim3(1), dim3(64), 0, (hipStream_t)stream, dst, e);
  return launch_status();
}

extern "C" int mpose_adamw_step(const mpose_adamw_job* jobs, int n_jobs, const float* hyper, const float* hyper_dev, void* stream) {
  if (n_jobs < 0 || (n_jobs > 0 && !jobs) || (!hyper && !hyper_dev)) return MPOSE_EINVAL;
  if (n_jobs == 0) return 0;
  for (int i = 0; i < n_jobs; ++i) {
    const mpose_adamw_job& j = jobs[i];
    if (j.n < 0 || (j.n > 0 && (!j.p || !j.g || !j.m || !j.v))) return MPOSE_EINVAL;
    if (((uintptr_t)j.p | (uintptr_t)j.g | (uintptr_t)j.m | (uintptr_t)j.v) & 3) return MPOSE_EINVAL;
  }
  AdamArgs a{};
  for (int i = 0; i < 8; ++i) a.h[i] = hyper ? hyper[i] : 0.f;
  a.hyper_dev = hyper ? nullptr : hyper_dev;
  for (int at = 0; at < n_jobs;) {
    int64_t longest = 0;
    a.n = 0;
    while (at < n_jobs && a.n < kAdamJobs) {
      if (jobs[at].n > 0) {
        a.j[a.n++] = jobs[at];
        longest = jobs[at].n > longest ? jobs[at].n : longest;
      }
      ++at;
    }
    if (a.n == 0) return 0;              // (only arrays of no elements are left)
    int64_t bx = (longest + kAdamChunk - 1) / kAdamChunk;
    if (bx > 1024) bx = 1024;
    launch(adamw_step_k, dim3((unsigned)bx, (unsigned)a.n), dim3(256), 0, (hipStream_t)stream, a);
  }
  return launch_status();
}
