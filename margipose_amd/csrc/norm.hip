// Layer normalisation over the last axis, forward and backward (gfx950).
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd,  y = xhat w + b
//   g = dy w:  dx = rstd (g - (sum g) / D - xhat (sum g xhat) / D),   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  So a row is read once and held in registers
// (E elements of it per thread) between the two reductions and the result: one wave per row up to 1024 columns, a workgroup of 4 or 8
// waves up to 16384 (8192 backward, and where elements are loaded one by one: registers); wider rows are read again from the cache (ln_*_wide_k).  Workgroups walk over the rows with a fixed mapping of columns to
// threads, which keeps w and b -- and in the backward pass the running sums of dw and db -- in registers too: one partial row of
// sums per workgroup goes to memory, a second launch adds the partial rows in a fixed order (no atomics: the same bits every run).
#include "common.h"

namespace mpose {
namespace {

typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

constexpr int kPartRows = 512;          // most partial rows of dw / db

__device__ __forceinline__ float bf(unsigned short u) { return __uint_as_float((unsigned)u << 16); }
__device__ __forceinline__ unsigned short to_bf(float v) {      // round to nearest even; NaN stays NaN
  const unsigned b = __float_as_uint(v);
  return (v == v) ? (unsigned short)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16) : (unsigned short)0x7fc0;
}

template <int DT> __device__ __forceinline__ float get1(const void* p, int64_t i) {
  if constexpr (DT == 0) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == 1) return bf(reinterpret_cast<const unsigned short*>(p)[i]);
  else return (float)reinterpret_cast<const _Float16*>(p)[i];
}
template <int DT> __device__ __forceinline__ void put1(void* p, int64_t i, float v) {
  if constexpr (DT == 0) reinterpret_cast<float*>(p)[i] = v;
  else if constexpr (DT == 1) reinterpret_cast<unsigned short*>(p)[i] = to_bf(v);
  else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}
__device__ __forceinline__ float get_w(const void* p, int dt, int64_t i) {
  return dt == 0 ? get1<0>(p, i) : dt == 1 ? get1<1>(p, i) : get1<2>(p, i);
}

// V consecutive elements (aligned to their own size), as they are in memory -- the next row's wait in this form -- and as floats
template <int DT, int V> struct Raw { unsigned u[V == 1 ? 1 : V * (DT == 0 ? 4 : 2) / 4]; };
template <int DT, int V> __device__ __forceinline__ void fetch(Raw<DT, V>& r, const void* p, int64_t i) {
  if constexpr (V == 1) {
    if constexpr (DT == 0) r.u[0] = reinterpret_cast<const unsigned*>(p)[i];
    else r.u[0] = reinterpret_cast<const unsigned short*>(p)[i];
  } else {
    constexpr int n = V * (DT == 0 ? 4 : 2) / 4;
    const unsigned char* q = reinterpret_cast<const unsigned char*>(p) + i * (DT == 0 ? 4 : 2);
    if constexpr (n == 2) {
      const uint2 t = *reinterpret_cast<const uint2*>(q);
      r.u[0] = t.x; r.u[1] = t.y;
    } else {
#pragma unroll
      for (int k = 0; k < n / 4; ++k) {
        const uint4 t = reinterpret_cast<const uint4*>(q)[k];
        r.u[4 * k] = t.x; r.u[4 * k + 1] = t.y; r.u[4 * k + 2] = t.z; r.u[4 * k + 3] = t.w;
      }
    }
  }
}
template <int DT, int V> __device__ __forceinline__ void unpack(const Raw<DT, V>& r, float* v) {
  if constexpr (DT == 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = __uint_as_float(r.u[k]);
  } else {
#pragma unroll
    for (int k = 0; k < (V + 1) / 2; ++k) {
      if constexpr (DT == 1) {
        v[2 * k] = __uint_as_float(r.u[k] << 16);
        if constexpr (V > 1) v[2 * k + 1] = __uint_as_float(r.u[k] & 0xffff0000u);
      } else {
        _Float16 h[2];
        __builtin_memcpy(h, &r.u[k], 4);
        v[2 * k] = (float)h[0];
        if constexpr (V > 1) v[2 * k + 1] = (float)h[1];
      }
    }
  }
}
template <int DT, int V> __device__ __forceinline__ void putv(void* p, int64_t i, const float* v) {
  if constexpr (V == 1) {
    put1<DT>(p, i, v[0]);
  } else if constexpr (DT == 0) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  } else {
    unsigned u[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
      if constexpr (DT == 1) u[q] = (unsigned)to_bf(v[2 * q]) | ((unsigned)to_bf(v[2 * q + 1]) << 16);
      else {
        const _Float16 h[2] = {(_Float16)v[2 * q], (_Float16)v[2 * q + 1]};
        __builtin_memcpy(&u[q], h, 4);
      }
    }
    if constexpr (V == 4) *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p) + i) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint4*>(reinterpret_cast<unsigned short*>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

struct FwdArgs {
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  int64_t x_ld, rows;
  int cols, w_dt;
  float eps;
};
struct BwdArgs {
  const void *dy, *x, *w;
  const float *mean, *rstd;
  void* dx;
  float* part;                 // [partial row][2][cols], or NULL
  int64_t dy_ld, x_ld, rows;
  int cols, w_dt;
};

// Sums over the T threads of a row: T = 64 one wave (no barrier), else through LDS (sh: 2 x T / 64 values per buffer, two buffers in turn)
template <int T, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* sh) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (T > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sh[w * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < T / 64; ++k) s += sh[k * N + i];
      v[i] = s;
    }
  }
}

template <int DT, int T, int E, int V>
__global__ __launch_bounds__(T > 256 ? T : 256) void ln_fwd_k(FwdArgs a) {
  constexpr int RW = T == 64 ? 4 : 1;                    // rows at a time
  constexpr int NV = E / V;
  __shared__ float sh[2][T / 64];
  const int t = T == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int cols = a.cols;
  const float inv_d = 1.f / (float)cols;
  float w[E], b[E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (i * T + t) * V + e;
      w[i * V + e] = a.w != nullptr && c < cols ? get_w(a.w, a.w_dt, c) : 1.f;
      b[i * V + e] = a.b != nullptr && c < cols ? get_w(a.b, a.w_dt, c) : 0.f;
    }
  // (the next row's loads are on their way while this row is reduced and written)
  const int64_t step = (int64_t)gridDim.x * RW;
  int64_t r = (int64_t)blockIdx.x * RW + (T == 64 ? (threadIdx.x >> 6) : 0);
  Raw<DT, V> raw[NV];
  auto ask = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * T + t) * V < cols) fetch<DT, V>(raw[i], a.x, row * a.x_ld + (i * T + t) * V);
  };
  if (r < a.rows) ask(r);
  for (; r < a.rows; r += step) {
    float x[E];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * T + t) * V < cols) unpack<DT, V>(raw[i], x + i * V);
      else
#pragma unroll
        for (int e = 0; e < V; ++e) x[i * V + e] = 0.f;
    }
    if (r + step < a.rows) ask(r + step);
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] += x[i];
    row_sum<T>(s, sh[0]);
    const float mean = s[0] * inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * T + t) * V < cols)
#pragma unroll
        for (int e = 0; e < V; ++e) { const float d = x[i * V + e] - mean; s[0] = fmaf(d, d, s[0]); }
    row_sum<T>(s, sh[1]);
    const float rstd = 1.f / sqrtf(s[0] * inv_d + a.eps);
    const int64_t yo = r * cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * V;
      if (c < cols) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = fmaf((x[i * V + e] - mean) * rstd, w[i * V + e], b[i * V + e]);
        putv<DT, V>(a.y, yo + c, y);
      }
    }
    if (t == 0 && a.mean != nullptr) { a.mean[r] = mean; a.rstd[r] = rstd; }
  }
}

template <int DT, int T, int E, int V>
__global__ __launch_bounds__(T > 256 ? T : 256) void ln_bwd_k(BwdArgs a) {
  constexpr int RW = T == 64 ? 4 : 1;
  constexpr int NV = E / V;
  __shared__ float sh[2][2 * (T / 64)];
  __shared__ float acc_sh[RW > 1 ? 2 * 64 * E : 1];
  const int t = T == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int cols = a.cols;
  const float inv_d = 1.f / (float)cols;
  float w[E], dw[E], db[E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (i * T + t) * V + e;
      w[i * V + e] = a.w != nullptr && c < cols ? get_w(a.w, a.w_dt, c) : 1.f;
      dw[i * V + e] = 0.f; db[i * V + e] = 0.f;
    }
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * RW;
  int64_t r = (int64_t)blockIdx.x * RW + (T == 64 ? (threadIdx.x >> 6) : 0);
  Raw<DT, V> rx[NV], rg[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto ask = [&](int64_t row) {
    next_mean = a.mean[row]; next_rstd = a.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * V;
      if (c < cols) { fetch<DT, V>(rx[i], a.x, row * a.x_ld + c); fetch<DT, V>(rg[i], a.dy, row * a.dy_ld + c); }
    }
  };
  if (r < a.rows) ask(r);
  for (; r < a.rows; r += step, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    float x[E], g[E];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * T + t) * V < cols) { unpack<DT, V>(rx[i], x + i * V); unpack<DT, V>(rg[i], g + i * V); }
      else
#pragma unroll
        for (int e = 0; e < V; ++e) { x[i * V + e] = mean; g[i * V + e] = 0.f; }
    }
    if (r + step < a.rows) ask(r + step);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] = (x[i] - mean) * rstd;
      dw[i] = fmaf(g[i], x[i], dw[i]);
      db[i] += g[i];
      g[i] *= w[i];
      s[0] += g[i];
      s[1] = fmaf(g[i], x[i], s[1]);
    }
    if (a.dx == nullptr) continue;
    row_sum<T>(s, sh[turn]);            // (two buffers: the next row's sums may be written before every wave has read these)
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
    const int64_t yo = r * cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * V;
      if (c < cols) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = rstd * (g[i * V + e] - m0 - x[i * V + e] * m1);
        putv<DT, V>(a.dx, yo + c, y);
      }
    }
  }
  if (a.part == nullptr) return;
  if constexpr (RW > 1) {               // the four waves' sums, in the order of the waves
    for (int k = 0; k < RW; ++k) {
      if ((int)(threadIdx.x >> 6) == k)
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float* p = acc_sh + (i * 64 + t) * 2;
          p[0] = k == 0 ? dw[i] : p[0] + dw[i];
          p[1] = k == 0 ? db[i] : p[1] + db[i];
        }
      __syncthreads();
    }
    if (threadIdx.x >= 64) return;
#pragma unroll
    for (int i = 0; i < E; ++i) { dw[i] = acc_sh[(i * 64 + t) * 2]; db[i] = acc_sh[(i * 64 + t) * 2 + 1]; }
  }
  float* p = a.part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (i * T + t) * V + e;
      if (c < cols) { p[c] = dw[i * V + e]; p[cols + c] = db[i * V + e]; }
    }
}

// Rows wider than the registers hold: the row is read three times (once from memory, then from the cache).
template <int DT>
__global__ __launch_bounds__(1024) void ln_fwd_wide_k(FwdArgs a) {
  __shared__ float sh[2][16];
  const float inv_d = 1.f / (float)a.cols;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t xo = r * a.x_ld, yo = r * a.cols;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.cols; c += 1024) s[0] += get1<DT>(a.x, xo + c);
    row_sum<1024>(s, sh[0]);
    const float mean = s[0] * inv_d;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 1024) { const float d = get1<DT>(a.x, xo + c) - mean; s[0] = fmaf(d, d, s[0]); }
    row_sum<1024>(s, sh[1]);
    const float rstd = 1.f / sqrtf(s[0] * inv_d + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float w = a.w != nullptr ? get_w(a.w, a.w_dt, c) : 1.f, b = a.b != nullptr ? get_w(a.b, a.w_dt, c) : 0.f;
      put1<DT>(a.y, yo + c, fmaf((get1<DT>(a.x, xo + c) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0 && a.mean != nullptr) { a.mean[r] = mean; a.rstd[r] = rstd; }
  }
}
template <int DT>
__global__ __launch_bounds__(1024) void ln_bwd_wide_k(BwdArgs a) {
  __shared__ float sh[2][32];
  const float inv_d = 1.f / (float)a.cols;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    const int64_t xo = r * a.x_ld, go = r * a.dy_ld, yo = r * a.cols;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float g = get1<DT>(a.dy, go + c) * (a.w != nullptr ? get_w(a.w, a.w_dt, c) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, (get1<DT>(a.x, xo + c) - mean) * rstd, s[1]);
    }
    row_sum<1024>(s, sh[turn]);
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float g = get1<DT>(a.dy, go + c) * (a.w != nullptr ? get_w(a.w, a.w_dt, c) : 1.f);
      put1<DT>(a.dx, yo + c, rstd * (g - m0 - (get1<DT>(a.x, xo + c) - mean) * rstd * m1));
    }
  }
}
// ... and their sums of dw, db: 256 columns per workgroup, blockIdx.y a share of the rows
template <int DT>
__global__ __launch_bounds__(256) void ln_sums_wide_k(BwdArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  const int64_t per = (a.rows + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y, hi = lo + per < a.rows ? lo + per : a.rows;
  float dw = 0.f, db = 0.f;
  for (int64_t r = lo; r < hi; ++r) {
    const float g = get1<DT>(a.dy, r * a.dy_ld + c);
    dw = fmaf(g, (get1<DT>(a.x, r * a.x_ld + c) - a.mean[r]) * a.rstd[r], dw);
    db += g;
  }
  float* p = a.part + (int64_t)blockIdx.y * 2 * a.cols;
  p[c] = dw;
  p[a.cols + c] = db;
}

// dw, db = the partial rows' sums: 64 values per workgroup, 16 waves each a share of the rows, joined in LDS in the order of the waves
__global__ __launch_bounds__(1024) void ln_join_k(const float* __restrict__ part, int n_part, int cols, void* dw, void* db, int w_dt) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane, n = 2 * (int64_t)cols;
  float s = 0.f;
  if (i < n) {
    const int per = (n_part + 15) / 16, lo = per * wave, hi = lo + per < n_part ? lo + per : n_part;
    const float* p = part + i;
    int r = lo;
    for (; r + 8 <= hi; r += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(r + u) * n];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; r < hi; ++r) s += p[r * n];
  }
  sh[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= n) return;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += sh[k][lane];
  void* out = i < cols ? dw : db;
  const int64_t c = i < cols ? i : i - cols;
  if (out == nullptr) return;
  if (w_dt == 0) put1<0>(out, c, s);
  else if (w_dt == 1) put1<1>(out, c, s);
  else put1<2>(out, c, s);
}

constexpr int kWide = 16384;            // most columns that the register kernels hold

int size_of(int dt) { return dt == 0 ? 4 : 2; }
int part_rows(int64_t rows, int cols) {
  const int64_t at_once = cols <= 1024 ? 4 : 1, n = (rows + at_once - 1) / at_once;
  return (int)(n < kPartRows ? n : kPartRows);
}
unsigned grid_for(int64_t items, unsigned cap) { return (unsigned)(items < (int64_t)cap ? items : (int64_t)cap); }

template <int DT, int T, int E>
void fwd_t(const FwdArgs& a, bool vec, hipStream_t s) {
  constexpr int V = E < 16 / (DT == 0 ? 4 : 2) ? E : 16 / (DT == 0 ? 4 : 2);
  const dim3 grid(grid_for(T == 64 ? (a.rows + 3) / 4 : a.rows, T > 256 ? 512 : T == 256 ? 1024 : 2048)), wg(T > 256 ? T : 256);
  if (vec) launch(ln_fwd_k<DT, T, E, V>, grid, wg, 0, s, a);
  else if constexpr (E < 32) launch(ln_fwd_k<DT, T, E, 1>, grid, wg, 0, s, a);
}
template <int DT>
void fwd(const FwdArgs& a, bool vec, hipStream_t s) {
  if (a.cols <= 256) fwd_t<DT, 64, 4>(a, vec, s);
  else if (a.cols <= 512) fwd_t<DT, 64, 8>(a, vec, s);
  else if (a.cols <= 1024) fwd_t<DT, 64, 16>(a, vec, s);
  else if (a.cols <= 2048) fwd_t<DT, 256, 8>(a, vec, s);
  else if (a.cols <= 4096) fwd_t<DT, 256, 16>(a, vec, s);
  else if (a.cols <= 8192) fwd_t<DT, 512, 16>(a, vec, s);
  else if (a.cols <= kWide && vec) fwd_t<DT, 512, 32>(a, vec, s);
  else launch(ln_fwd_wide_k<DT>, dim3(grid_for(a.rows, 512)), dim3(1024), 0, s, a);
}
template <int DT, int T, int E>
void bwd_t(const BwdArgs& a, bool vec, hipStream_t s) {
  constexpr int V = E < 16 / (DT == 0 ? 4 : 2) ? E : 16 / (DT == 0 ? 4 : 2);
  const dim3 grid((unsigned)part_rows(a.rows, a.cols)), wg(T > 256 ? T : 256);
  if (vec) launch(ln_bwd_k<DT, T, E, V>, grid, wg, 0, s, a);
  else if constexpr (E < 32) launch(ln_bwd_k<DT, T, E, 1>, grid, wg, 0, s, a);
}
template <int DT>
void bwd(const BwdArgs& a, bool vec, hipStream_t s) {
  if (a.cols <= 256) bwd_t<DT, 64, 4>(a, vec, s);
  else if (a.cols <= 512) bwd_t<DT, 64, 8>(a, vec, s);
  else if (a.cols <= 1024) bwd_t<DT, 64, 16>(a, vec, s);
  else if (a.cols <= 2048) bwd_t<DT, 256, 8>(a, vec, s);
  else if (a.cols <= 4096) bwd_t<DT, 256, 16>(a, vec, s);
  else if (a.cols <= kWide / 2) bwd_t<DT, 512, 16>(a, vec, s);
  else {
    if (a.dx != nullptr) launch(ln_bwd_wide_k<DT>, dim3(grid_for(a.rows, 512)), dim3(1024), 0, s, a);
    if (a.part != nullptr) launch(ln_sums_wide_k<DT>, dim3((unsigned)((a.cols + 255) / 256), (unsigned)part_rows(a.rows, a.cols)), dim3(256), 0, s, a);
  }
}

bool bad_types(int io_dt, int w_dt) { return io_dt < 0 || io_dt > 2 || w_dt < 0 || w_dt > 2; }
// rows of p start on a boundary of 16 bytes, or of the four elements that a thread takes of rows up to 256 columns
bool rows_aligned(const void* p, int64_t ld, int cols, int dt) {
  const uintptr_t q = (cols <= 256 ? 4 : 16 / size_of(dt)) * size_of(dt) - 1;
  return (((uintptr_t)p | (uintptr_t)(ld * size_of(dt))) & q) == 0;
}

}  // namespace
}  // namespace mpose

using namespace mpose;

extern "C" int mpose_layer_norm_fwd(const void* x, int64_t x_ld, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int cols,
                                    float eps, int io_dtype, int w_dtype, void* stream) {
  if (rows < 0 || cols < 1 || x_ld < 0 || !(eps >= 0.f) || bad_types(io_dtype, w_dtype) || (mean == nullptr) != (rstd == nullptr)) return MPOSE_EINVAL;
  if (rows == 0) return 0;
  const uintptr_t own = (uintptr_t)size_of(io_dtype) - 1;
  if (!x || !y || (((uintptr_t)x | (uintptr_t)y) & own) || (((uintptr_t)w | (uintptr_t)b) & ((uintptr_t)size_of(w_dtype) - 1))) return MPOSE_EINVAL;
  const FwdArgs a{x, w, b, y, mean, rstd, x_ld, rows, cols, w_dtype, eps};
  const int v = cols <= 256 ? 4 : 16 / size_of(io_dtype);
  const bool vec = cols % v == 0 && rows_aligned(x, x_ld, cols, io_dtype) && rows_aligned(y, cols, cols, io_dtype);
  hipStream_t s = (hipStream_t)stream;
  if (io_dtype == 0) fwd<0>(a, vec, s);
  else if (io_dtype == 1) fwd<1>(a, vec, s);
  else fwd<2>(a, vec, s);
  return launch_status();
}

extern "C" int64_t mpose_layer_norm_bwd_ws_bytes(int64_t rows, int cols) {
  if (rows < 0 || cols < 1) return MPOSE_EINVAL;
  return (int64_t)part_rows(rows, cols) * 2 * cols * 4;
}

extern "C" int mpose_layer_norm_bwd(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w, const float* mean, const float* rstd, void* dx,
                                    void* dw, void* db, int64_t rows, int cols, int io_dtype, int w_dtype, void* ws, int64_t ws_bytes, void* stream) {
  if (rows < 0 || cols < 1 || x_ld < 0 || dy_ld < 0 || bad_types(io_dtype, w_dtype)) return MPOSE_EINVAL;
  const bool sums = dw != nullptr || db != nullptr;
  const uintptr_t own = (uintptr_t)size_of(io_dtype) - 1, wown = (uintptr_t)size_of(w_dtype) - 1;
  if ((((uintptr_t)w | (uintptr_t)dw | (uintptr_t)db) & wown) || (((uintptr_t)dy | (uintptr_t)x | (uintptr_t)dx) & own)) return MPOSE_EINVAL;
  if (rows > 0 && (!dy || !x || !mean || !rstd)) return MPOSE_EINVAL;
  if (sums && rows > 0 && (!ws || ((uintptr_t)ws & 3) || ws_bytes < mpose_layer_norm_bwd_ws_bytes(rows, cols))) return MPOSE_EINVAL;
  if (!sums && (rows == 0 || dx == nullptr)) return 0;
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    const BwdArgs a{dy, x, w, mean, rstd, dx, sums ? (float*)ws : nullptr, dy_ld, x_ld, rows, cols, w_dtype};
    const int v = cols <= 256 ? 4 : 16 / size_of(io_dtype);
    const bool vec = cols % v == 0 && rows_aligned(x, x_ld, cols, io_dtype) && rows_aligned(dy, dy_ld, cols, io_dtype) &&
                     (dx == nullptr || rows_aligned(dx, cols, cols, io_dtype));
    if (io_dtype == 0) bwd<0>(a, vec, s);
    else if (io_dtype == 1) bwd<1>(a, vec, s);
    else bwd<2>(a, vec, s);
  }
  if (sums) launch(ln_join_k, dim3((unsigned)((2 * (int64_t)cols + 63) / 64)), dim3(1024), 0, s, (const float*)ws, part_rows(rows, cols), cols, dw, db, w_dtype);
  return launch_status();
}
