// Newton-Schulz orthogonalisation of a set of matrices, and the Muon step built on it (gfx950).
//
// Mathematics.  X0 = G / (|G|_F + eps), the shorter axis (m) as rows, the longer (n) as columns; `steps` times
//     S = X X^T,   Q = a I + b S + c S^2,   X <- Q X
// which maps every singular value s to a s + b s^3 + c s^5.  S, Q and all products of them are polynomials in one symmetric matrix:
// they commute, they are symmetric, and the next S is Q S Q without touching X.  So the long axis is visited twice per GROUP of steps,
//     S = X X^T;   per step: Q = q(S), W = Q S, S <- W Q, P <- Q P;   X <- P X,
// and every m x m product computes only the tiles on and above the diagonal (the others are their transposes).
// In a group the rounding of S is lifted by a^2 a step where s is small, so a group is as long as a^2 to the power (length - 1) stays below
// a limit (kLift): 1 for mpose_orthogonalize's fp32 results (X on every step for the customary a = 3.4445), 12 for 16-bit results (groups of
// 2, 2, 1: their rounding hides the difference), 150 for mpose_muon_step (3, 2), whose result is a small part of a weight.  Relative error
// against float64 (plain fp32 products: 1.1e-6 at 17 x 128, 1.4e-6 at 128 x 1152): X on every step 0.9e-6 and 1.0e-6; 3, 2: 1.4e-6 and
// 3.4e-6; 2, 2, 1 on twelve 17 x 128: up to 2.2e-6.  One group of five, in a model of the arithmetic: 1e-4.  Visits of the long axis: 5, 3, 2.
//
// Arithmetic: like the convolutions (three fp16 products of two-way split operands, x * 2^k = h + l: 22 bits), but the scale
// exponents come from a bound, not from a measurement: |x_ij| <= |X|_2, and a scalar recursion bounds |X|_2, |S|_2, |Q|_2 from the
// first |X|_2 <= |G|_F / (|G|_F + eps) on (orth_scalars_k).
//
// Layout of a split matrix of R rows and K columns, "H8": [K / 8][plane h, l][R][8] fp16, R padded to the tile, K to 32 (zeros).  64 rows
// of an octet are 1 KB in a row: one LDS-DMA instruction; both operands of C = A B^T are read that way, so X is kept in both
// orientations (N: as stored, T: transposed).
#include <math.h>
#include "common.h"

namespace mpose {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_void_p;

constexpr int kMaxSteps = 24;
constexpr int kChunk = 4096;            // elements per workgroup of the momentum / norm pass
constexpr int kSetupJobs = 160;         // jobs per set-up launch (they travel as kernel arguments, 11.5 KB: 4.7 us a launch with 48 as with 160)
// Largest m whose products run as one chain in one workgroup: 128, or 192 where at least 96 matrices are larger than 128.  One chain of
// a group of three takes 81 us at m = 192 however few they are, the nine launches tile by tile 7 us each for a dozen matrices and 25 us
// each for the 205 of the default model.
constexpr int kChainMax = 192, kChainFew = 128, kChainMany = 96;
constexpr double kLift[3] = {1.0, 12.0, 150.0};     // fp32 results, 16-bit results, Muon
constexpr float kGrowth = 1024.f;       // largest singular value that a polynomial may make of one in [0, 1]

struct StepExp { int x, s, q, w, p; };  // scale exponents of X (a group's first step), S, Q, W, P

struct OrthJob {                        // device copy of one matrix's job
  const void* src;
  float* buf;
  void* dst;
  unsigned char *n[2], *t[2];           // X as stored / transposed (H8); two sets: a restart reads one and writes the other
  unsigned char *s, *w, *q[2], *p[2];   // m x m (H8)
  double* part;
  int n_part, rows, cols, m, mp, mk;    // mp: m padded as rows, mk: m padded as the K axis
  int rp, cp, rk, ck;                   // rows / cols padded the same two ways
  int wide, aligned, chained;
  float scale, in_scale;
  StepExp e[kMaxSteps];
};

struct OrthLayout {                     // byte offsets inside a job's part of the workspace
  int64_t n[2], t[2], s, w, q[2], p[2], part, total;
  int mp, mk, rp, cp, rk, ck, n_part;
};

__host__ __device__ inline int pad_to(int v, int q) { return (v + q - 1) / q * q; }

__host__ __device__ inline OrthLayout orth_layout(int rows, int cols, int pad, int n_groups) {
  OrthLayout l;
  const int m = rows < cols ? rows : cols;
  l.rp = pad_to(rows, pad); l.cp = pad_to(cols, pad); l.mp = pad_to(m, pad);
  l.rk = pad_to(rows, 32); l.ck = pad_to(cols, 32); l.mk = pad_to(m, 32);
  l.n_part = (int)(((int64_t)rows * cols + kChunk - 1) / kChunk);
  const int64_t nb = (int64_t)l.ck * l.rp * 4, tb = (int64_t)l.rk * l.cp * 4, mb = (int64_t)l.mk * l.mp * 4;
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    l.n[i] = at; if (i == 0 || n_groups > 1) at += nb;
    l.t[i] = at; if (i == 0 || n_groups > 1) at += tb;
  }
  l.s = at; at += mb;
  l.w = at; at += mb;
  for (int i = 0; i < 2; ++i) { l.q[i] = at; at += mb; l.p[i] = at; at += mb; }
  l.part = at; at += (int64_t)pad_to(l.n_part * 8, 256);
  l.total = (at + 255) / 256 * 256;
  return l;
}

// ---- set-up: job table and tile lists, written by the device from kernel arguments (no host memory outlives the call) ----
struct SetupJob {
  const void* src;
  float* buf;
  void* dst;
  unsigned char* ws;
  int rows, cols;
  float scale;
  int ew0, split0, sym0, big0, fin0;    // where the job's entries start in the lists
  int chain;                            // place in the chain list, or -1: the matrix's m x m products run tile by tile (big0)
};
struct SetupArgs {
  SetupJob j[kSetupJobs];
  OrthJob* jobs;
  int2 *ew, *split, *sym, *big, *fin;
  int* chain;
  int first, n, pad, tile_sym, tile_fin, n_groups, elem;
};

// Order of the tiles of one product: 8 x 8 blocks of tiles one after another, so that the tiles that an XCD holds at a time share their rows
// of both operands in its 4 MB of L2 (row after row, a 4096 x 4096 product fetched 1.6 GB through the fabric).
constexpr int kBlock = 8;
__device__ inline int block_place(int r, int c, int tr, int tc) {
  const int R = r / kBlock, C = c / kBlock, dr = min(kBlock, tr - R * kBlock), dc = min(kBlock, tc - C * kBlock);
  return R * kBlock * tc + C * kBlock * dr + (r - R * kBlock) * dc + (c - C * kBlock);
}
__device__ inline int upper_place(int r, int c, int t) {          // ... of the tiles on and above the diagonal
  const int R = r / kBlock, C = c / kBlock, r0 = R * kBlock, d = min(kBlock, t - r0), lr = r - r0, lc = c - C * kBlock;
  const int before = r0 * t - r0 * (r0 - 1) / 2;
  if (C == R) return before + lr * d - lr * (lr - 1) / 2 + (lc - lr);
  return before + d * (d + 1) / 2 + (C - R - 1) * d * kBlock + lr * min(kBlock, t - C * kBlock) + lc;
}

__global__ __launch_bounds__(256) void orth_setup_k(SetupArgs a) {
  const SetupJob& j = a.j[blockIdx.x];
  const int id = a.first + blockIdx.x;
  const OrthLayout l = orth_layout(j.rows, j.cols, a.pad, a.n_groups);
  if (threadIdx.x == 0) {
    OrthJob* o = a.jobs + id;
    o->src = j.src; o->buf = j.buf; o->dst = j.dst; o->scale = j.scale;
    for (int i = 0; i < 2; ++i) {
      o->n[i] = j.ws + l.n[i]; o->t[i] = j.ws + l.t[i]; o->q[i] = j.ws + l.q[i]; o->p[i] = j.ws + l.p[i];
    }
    o->s = j.ws + l.s; o->w = j.ws + l.w;
    o->part = reinterpret_cast<double*>(j.ws + l.part); o->n_part = l.n_part;
    o->rows = j.rows; o->cols = j.cols; o->m = j.rows < j.cols ? j.rows : j.cols;
    o->mp = l.mp; o->mk = l.mk; o->rp = l.rp; o->cp = l.cp; o->rk = l.rk; o->ck = l.ck;
    o->wide = j.rows <= j.cols;
    o->chained = j.chain >= 0;
    if (j.chain >= 0) a.chain[j.chain] = id;
    const uint64_t bits = (uint64_t)j.src | (uint64_t)j.buf | (uint64_t)j.dst | ((uint64_t)j.cols * (uint64_t)a.elem);
    o->aligned = (bits & (uint64_t)(4 * a.elem - 1)) == 0;        // four elements at a time: every row starts on that boundary
  }
  for (int i = threadIdx.x; i < l.n_part; i += 256) a.ew[j.ew0 + i] = make_int2(id, i);
  const int sr = (j.rows + 63) / 64, sc = (j.cols + 63) / 64;
  for (int i = threadIdx.x; i < sr * sc; i += 256) a.split[j.split0 + i] = make_int2(id, (i / sc) | ((i % sc) << 16));
  const int m = j.rows < j.cols ? j.rows : j.cols, tm = (m + a.tile_sym - 1) / a.tile_sym;
  for (int i = threadIdx.x; i < tm * tm; i += 256) {
    const int r = i / tm, c = i % tm;
    if (c < r) continue;
    const int at = upper_place(r, c, tm);
    a.sym[j.sym0 + at] = make_int2(id, r | (c << 16));
    if (j.chain < 0) a.big[j.big0 + at] = make_int2(id, r | (c << 16));
  }
  const int tr = (j.rows + a.tile_fin - 1) / a.tile_fin, tc = (j.cols + a.tile_fin - 1) / a.tile_fin;
  for (int i = threadIdx.x; i < tr * tc; i += 256) {
    const int r = i / tc, c = i % tc;
    a.fin[j.fin0 + block_place(r, c, tr, tc)] = make_int2(id, r | (c << 16));
  }
}

// ---- element access ----
template <int DT>
__device__ __forceinline__ float load1(const void* p, long i) {
  if constexpr (DT == 0) return reinterpret_cast<const float*>(p)[i];
  if constexpr (DT == 1) return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
  if constexpr (DT == 2) return (float)reinterpret_cast<const _Float16*>(p)[i];
}
template <int DT>
__device__ __forceinline__ float4 load4(const void* p, long i) {
  if constexpr (DT == 0) {
    return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
  } else if constexpr (DT == 1) {
    const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(p) + i);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  } else {
    const f16x4 v = *reinterpret_cast<const f16x4*>(reinterpret_cast<const _Float16*>(p) + i);
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
  }
}
template <int DT>
__device__ __forceinline__ void store1(void* p, long i, float v) {
  if constexpr (DT == 0) reinterpret_cast<float*>(p)[i] = v;
  if constexpr (DT == 1) {             // round to nearest even; NaN stays NaN
    const unsigned b = __float_as_uint(v);
    reinterpret_cast<unsigned short*>(p)[i] = (v == v) ? (unsigned short)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16) : (unsigned short)0x7fc0;
  }
  if constexpr (DT == 2) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

struct Hyper { float lr, momentum, first, wd; };
__device__ __forceinline__ Hyper get_hyper(const Hyper& h, const float* dev) {
  return dev != nullptr ? Hyper{dev[0], dev[1], dev[2], dev[3]} : h;
}

// what is orthogonalised at one element: the input, or (MUON) the momentum update's direction
__device__ __forceinline__ float direction(float g, float b, float mom, int nesterov) { return nesterov ? fmaf(mom, b, g) : b; }

struct PassArgs {
  const OrthJob* jobs;
  const int2* list;
  Hyper h;
  const float* hyper_dev;
  int nesterov, group;
};

// ---- pass 1: momentum update, sum of squares (float64: the squares of any finite float stay finite) ----
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void orth_norm_k(PassArgs a) {
  const int2 it = a.list[blockIdx.x];
  const OrthJob& j = a.jobs[it.x];
  const Hyper h = get_hyper(a.h, a.hyper_dev);
  const long total = (long)j.rows * j.cols, lo = (long)it.y * kChunk, hi = lo + kChunk < total ? lo + kChunk : total;
  const bool first = h.first != 0.f;
  double sum = 0.0;
  auto one = [&](float g, float& b) {
    float u = g;
    if constexpr (MUON) {
      b = first ? g : fmaf(h.momentum, b, g);
      u = direction(g, b, h.momentum, a.nesterov);
    }
    sum += (double)u * (double)u;
  };
  const bool vec = ((reinterpret_cast<uintptr_t>(j.src) & (DT == 0 ? 15 : 7)) == 0) && (!MUON || (reinterpret_cast<uintptr_t>(j.buf) & 15) == 0);
  if (vec) {
#pragma unroll
    for (int q = 0; q < kChunk / 1024; ++q) {
      const long i = lo + q * 1024 + threadIdx.x * 4;
      if (i + 4 <= hi) {
        const float4 g = load4<DT>(j.src, i);
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (MUON && !first) b = *reinterpret_cast<const float4*>(j.buf + i);
        one(g.x, b.x); one(g.y, b.y); one(g.z, b.z); one(g.w, b.w);
        if (MUON) *reinterpret_cast<float4*>(j.buf + i) = b;
      } else {
        for (long k = i; k < hi; ++k) {
          float b = (MUON && !first) ? j.buf[k] : 0.f;
          one(load1<DT>(j.src, k), b);
          if (MUON) j.buf[k] = b;
        }
      }
    }
  } else {
    for (long k = lo + threadIdx.x; k < hi; k += 256) {
      float b = (MUON && !first) ? j.buf[k] : 0.f;
      one(load1<DT>(j.src, k), b);
      if (MUON) j.buf[k] = b;
    }
  }
  __shared__ double sh[4];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) j.part[it.y] = sh[0] + sh[1] + sh[2] + sh[3];
}

struct Poly { float a, b, c; };

// largest |a + b t + c t^2| for t in [0, hi]
__host__ __device__ inline float bound_q(const Poly& k, float hi) {
  const float at_hi = fabsf(k.a + hi * (k.b + hi * k.c));
  float r = fmaxf(fabsf(k.a), at_hi);
  if (k.c != 0.f) {
    const float t = -k.b / (2.f * k.c);
    if (t > 0.f && t < hi) r = fmaxf(r, fabsf(k.a + t * (k.b + t * k.c)));
  }
  return r;
}
// largest |s (a + b s^2 + c s^4)| for s in [0, hi]: at hi or where a + 3 b t + 5 c t^2 = 0, t = s^2
__host__ __device__ inline float bound_x(const Poly& k, float hi) {
  auto f = [&](float t) { return sqrtf(t) * fabsf(k.a + t * (k.b + t * k.c)); };
  const float hi2 = hi * hi;
  float r = f(hi2);
  if (k.c != 0.f) {
    const float d = 9.f * k.b * k.b - 20.f * k.a * k.c;
    if (d >= 0.f) {
      const float root = sqrtf(d);
      const float t0 = (-3.f * k.b - root) / (10.f * k.c), t1 = (-3.f * k.b + root) / (10.f * k.c);
      if (t0 > 0.f && t0 < hi2) r = fmaxf(r, f(t0));
      if (t1 > 0.f && t1 < hi2) r = fmaxf(r, f(t1));
    }
  } else if (k.b != 0.f) {
    const float t = -k.a / (3.f * k.b);
    if (t > 0.f && t < hi2) r = fmaxf(r, f(t));
  }
  return r;
}

// scale exponent for magnitudes up to `bound`: bound * 2^k in [2^14, 2^15).  Exponents stop at 60: magnitudes below 2^-45 (a gradient
// that far below eps) lose relative precision step by step instead of overflowing the scale factors' product.
__device__ __forceinline__ int exp_of(float bound) {
  const int k = f16_scale_exp(bound * 1.01f);
  return k > 60 ? 60 : k;
}

// ---- pass 2: one workgroup per matrix: |G|_F, the input scale, every step's scale exponents ----
__global__ __launch_bounds__(256) void orth_scalars_k(OrthJob* jobs, Poly k, double eps, int steps, int group_first_mask) {
  OrthJob& j = jobs[blockIdx.x];
  __shared__ double sh[4];
  double s = 0.0;
  const int n = j.n_part;
  const double* const part = j.part;
  int at = threadIdx.x;
  for (; at + 768 < n; at += 1024) {              // four partial sums in flight
    const double v0 = part[at], v1 = part[at + 256], v2 = part[at + 512], v3 = part[at + 768];
    s += (v0 + v1) + (v2 + v3);
  }
  for (; at < n; at += 256) s += part[at];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = sh[0] + sh[1] + sh[2] + sh[3];
  const double norm = sqrt(s), den = norm + eps;
  float bx = norm > 0.0 ? (float)(norm / den) : 0.f, bp = 1.f;
  StepExp e{0, 0, 0, 0, 0};
  for (int i = 0; i < steps; ++i) {
    const float bs = bx * bx, bq = bound_q(k, bs);
    if ((group_first_mask >> i) & 1) { e.x = exp_of(bx); bp = 1.f; }
    bp *= bq;
    e.s = exp_of(bs); e.q = exp_of(bq); e.w = exp_of(bq * bs); e.p = exp_of(bp);
    j.e[i] = e;
    bx = bound_x(k, bx) * 1.00001f;
  }
  // all zeros with eps == 0: 0 / 0 stays NaN as in the formula
  j.in_scale = (float)((double)pow2f(j.e[0].x) / den);
}

__device__ __forceinline__ void split16(float x, _Float16& h, _Float16& l) {
  h = (_Float16)x;
  l = (_Float16)(x - (float)h);
}

// ---- pass 3: X0 in both orientations.  One 64 x 64 tile per workgroup, transposed through LDS. ----
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void orth_split_k(PassArgs a) {
  const int2 it = a.list[blockIdx.x];
  const OrthJob& j = a.jobs[it.x];
  const int r0 = (it.y & 0xffff) * 64, c0 = (int)((unsigned)it.y >> 16) * 64;
  const float mom = MUON ? get_hyper(a.h, a.hyper_dev).momentum : 0.f;
  const float sc = j.in_scale;
  const int rows = j.rows, cols = j.cols;
  __shared__ float tile[64][65];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = q * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r0 + r < rows) {
      const long i = (long)(r0 + r) * cols + c0 + c;
      if (j.aligned && c0 + c + 4 <= cols) {
        const float4 g = load4<DT>(j.src, i);
        v[0] = g.x; v[1] = g.y; v[2] = g.z; v[3] = g.w;
        if (MUON) {
          const float4 b = *reinterpret_cast<const float4*>(j.buf + i);
          v[0] = direction(g.x, b.x, mom, a.nesterov); v[1] = direction(g.y, b.y, mom, a.nesterov);
          v[2] = direction(g.z, b.z, mom, a.nesterov); v[3] = direction(g.w, b.w, mom, a.nesterov);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + c + e < cols) {
            v[e] = load1<DT>(j.src, i + e);
            if (MUON) v[e] = direction(v[e], j.buf[i + e], mom, a.nesterov);
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + c + e < cols) v[e] *= sc;             // (padding stays 0 whatever the scale is)
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[r][c + e] = v[e];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int row = threadIdx.x & 63, oct = q * 4 + (threadIdx.x >> 6);
    f16x8 h, l;
    if (c0 + oct * 8 < j.ck) {
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 hh, ll; split16(tile[row][oct * 8 + e], hh, ll); h[e] = hh; l[e] = ll; }
      f16x8* d = reinterpret_cast<f16x8*>(j.n[0]) + ((long)(c0 / 8 + oct) * 2 * j.rp + r0 + row);
      d[0] = h; d[j.rp] = l;
    }
    if (r0 + oct * 8 < j.rk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 hh, ll; split16(tile[oct * 8 + e][row], hh, ll); h[e] = hh; l[e] = ll; }
      f16x8* d = reinterpret_cast<f16x8*>(j.t[0]) + ((long)(r0 / 8 + oct) * 2 * j.cp + c0 + row);
      d[0] = h; d[j.cp] = l;
    }
  }
}

// ---- the products ----
// S = X X^T;  Q = q(S);  W = Q S and / or P = Q P;  S <- W Q;  X <- P X in both orientations;  the result from P X.
// (A template argument, not a run-time value: with one kernel choosing among the symmetric products at run time hipcc 7.2 left the
// output's address undefined on one of the paths.)
enum { K_GRAM = 0, K_Q = 1, K_MUL = 2, K_NEXT = 3, K_X = 4, K_OUT = 5 };

struct GemmArgs {
  const OrthJob* jobs;
  const int2* list;
  int n_tiles, n_main;                // tiles of the list; of the n_tiles (x 2) tiles of the launch, those with a workgroup each
  int split;                          // workgroups for each of the others, which leave their shares of the sum in `part`
  float* part;
  int step, step0, i, parity;         // step; the group's first step; step - step0; the group's X set
  int y0;                             // K_MUL: which of {W = Q S, P = Q P} comes first
  Poly k;
  Hyper h;
  const float* hyper_dev;
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ f32x16 mfma(const f16x8 a, const f16x8 b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Four consecutive k of one row, values v[0..3] * 2^e split into the two planes: 8 bytes each.
__device__ __forceinline__ void put4(unsigned char* base, int rp, int row, int k, const float (&v)[4]) {
  f16x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) { _Float16 hh, ll; split16(v[e], hh, ll); h[e] = hh; l[e] = ll; }
  unsigned char* d = base + (((long)(k >> 3) * 2 * rp + row) * 16 + (k & 4) * 2);
  *reinterpret_cast<f16x4*>(d) = h;
  *reinterpret_cast<f16x4*>(d + (long)rp * 16) = l;
}

// C = A B^T over H8 operands, one 64 R x 64 R tile per workgroup: 2 x 2 waves, R x R accumulator blocks of 32 x 32 per wave.
// Per k = 16: 4 R fragment reads for 3 R^2 MFMAs.  Ring of NBUF slots of k = 32, filled by LDS DMA.
// JOIN: no product, the tile's sum is that of its `split` partial sums, added in their order.
template <int R, int NBUF, int KIND, int DT, bool JOIN>
__global__ __launch_bounds__(256, NBUF * R > 4 ? 1 : 2) void orth_gemm_k(GemmArgs a) {
  constexpr int T = 64 * R;
  constexpr int kOp = 8 * T * 16, kSlot = 2 * kOp;        // bytes of one operand / both in a slot: [octet 4][plane 2][T][16 B]
  constexpr int LW = 4 * R;                               // DMA instructions per wave and slot
  constexpr int kLds = JOIN ? 4 * 32 * 33 * 4 : NBUF * kSlot;
  __shared__ __attribute__((aligned(16))) unsigned char smem[kLds];
  static_assert(4 * 32 * 33 * 4 <= kLds, "the transposing epilogue fits the ring");
  constexpr int RA = JOIN ? 1 : R;                        // accumulator blocks each way: a join takes one of its tile's R x R sets of four
  int idx, share = 0, set = 0;
  bool partial = false;
  if constexpr (JOIN) {
    idx = a.n_main + (int)blockIdx.x / (R * R);
    set = (int)blockIdx.x % (R * R);
  } else {
    // workgroup b runs on XCD b % 8 (observed placement, speed only): an XCD takes a contiguous run of the tile list
    const int per = (a.n_main + 7) >> 3, b = (int)blockIdx.x;
    if (b < per * 8) {
      idx = (b & 7) * per + (b >> 3);
      if (idx >= a.n_main) return;
    } else {
      const int q = (b - per * 8) / a.split;
      share = (b - per * 8) - q * a.split;
      idx = a.n_main + q;
      partial = true;
    }
  }
  const int second_half = idx >= a.n_tiles ? 1 : 0;
  const int2 it = a.list[idx - second_half * a.n_tiles];
  const OrthJob& j = a.jobs[it.x];
  const int i0 = (it.y & 0xffff) * T, j0 = (int)((unsigned)it.y >> 16) * T;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 31, lh = lane >> 5, wm = wave & 1, wn = wave >> 1;

  const StepExp e = j.e[a.step];
  const unsigned char *A, *B;
  unsigned char* out = nullptr;
  int arp = j.mp, brp = j.mp, kk = j.mk, ea, eb, eo = 0;
  if constexpr (KIND == K_GRAM) {
    A = B = j.wide ? j.n[a.parity] : j.t[a.parity];
    kk = j.wide ? j.ck : j.rk;
    arp = brp = j.wide ? j.rp : j.cp;
    ea = eb = e.x; eo = e.s; out = j.s;
  } else if constexpr (KIND == K_Q) {
    A = B = j.s; ea = eb = e.s; eo = e.q; out = j.q[a.i & 1];
  } else if constexpr (KIND == K_MUL) {
    const bool p = a.y0 + second_half != 0;
    unsigned char* const prev = a.i == 1 ? j.q[0] : j.p[(a.i + 1) & 1];
    unsigned char* const next = j.p[a.i & 1];
    A = j.q[a.i & 1]; ea = e.q;
    B = p ? prev : j.s;
    eb = p ? j.e[a.i > 0 ? a.step - 1 : a.step].p : e.s;
    eo = p ? e.p : e.w;
    out = p ? next : j.w;
  } else if constexpr (KIND == K_NEXT) {
    A = j.w; ea = e.w; B = j.q[a.i & 1]; eb = e.q; eo = j.e[a.step + 1].s; out = j.s;
  } else {
    const unsigned char* P = a.i == 0 && !j.chained ? j.q[0] : j.p[j.chained ? 0 : a.i & 1];
    const unsigned char* X = j.wide ? j.t[a.parity] : j.n[a.parity];
    A = j.wide ? P : X; B = j.wide ? X : P;
    arp = j.rp; brp = j.cp;
    ea = j.wide ? e.p : e.x; eb = j.wide ? e.x : e.p;
    if (KIND == K_X) eo = j.e[a.step + 1].x;
  }

  f32x16 acc[RA][RA], acx[RA][RA];      // h x h, and the two cross products (2^-11 of it: their roundings do not matter)
#pragma unroll
  for (int r = 0; r < RA; ++r)
#pragma unroll
    for (int c = 0; c < RA; ++c)
#pragma unroll
      for (int v = 0; v < 16; ++v) { acc[r][c][v] = 0.f; acx[r][c][v] = 0.f; }

  constexpr int NQ = R * R * 4;                            // float4s of a thread's share of the tile
  if constexpr (JOIN) {
    const float4* p = reinterpret_cast<const float4*>(a.part) + ((long)(idx - a.n_main) * a.split * NQ + set * 4) * 256 + tid;
#pragma unroll 4
    for (int q = 0; q < a.split; ++q) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 v = p[((long)q * NQ + g) * 256];
        acc[0][0][4 * g] += v.x; acc[0][0][4 * g + 1] += v.y; acc[0][0][4 * g + 2] += v.z; acc[0][0][4 * g + 3] += v.w;
      }
    }
  } else {
    // the slots of this workgroup: all, or its share of a tile that is split
    const int all = kk >> 5, s_lo = partial ? (int)((long)all * share / a.split) : 0, n_slots = (partial ? (int)((long)all * (share + 1) / a.split) : all) - s_lo;
    // waves 0, 1 fetch A, waves 2, 3 fetch B; each half of the operand's eight (octet, plane) slabs
    const bool isb = wave >= 2;
    const int rp = isb ? brp : arp, row0 = isb ? j0 : i0;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(isb ? B : A), 0, (int)((unsigned)kk * (unsigned)rp * 4u), 0x00020000);
    const unsigned slab = (unsigned)rp * 16u;
    unsigned char* lds0 = smem + (isb ? kOp : 0) + (wave & 1) * (kOp / 2);
    const unsigned voff = (unsigned)lane * 16u;
    auto fetch = [&](int s) {
      unsigned char* l = lds0 + (s % NBUF) * kSlot;
#pragma unroll
      for (int u = 0; u < LW; ++u) {
        const int sl = u / R, rg = u % R;
        const unsigned soff = ((unsigned)(s_lo + s) * 8u + (unsigned)((wave & 1) * 4 + sl)) * slab + (unsigned)(row0 + rg * 64) * 16u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_p)(l + u * 1024), 16, (int)voff, (int)soff, 0, 0);
      }
    };
    // The loop always reads the fragments of the next k = 16 before it multiplies the current ones: two register sets, F0 for the
    // first half of a slot, F1 for the second.  One barrier per slot, passed while F1 still has to be multiplied.
    struct Frags { f16x8 ah[R], al[R], bh[R], bl[R]; } f0, f1;
    const unsigned char* const pa = smem + (wm * 32 * R + li) * 16 + lh * 2 * T * 16;
    const unsigned char* const pb = smem + kOp + (wn * 32 * R + li) * 16 + lh * 2 * T * 16;
    auto read = [&](Frags& f, int s, int k16) {
      const int o = (s % NBUF) * kSlot + k16 * 4 * T * 16;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        f.ah[r] = *reinterpret_cast<const f16x8*>(pa + o + r * 512);
        f.bh[r] = *reinterpret_cast<const f16x8*>(pb + o + r * 512);
        f.bl[r] = *reinterpret_cast<const f16x8*>(pb + o + T * 16 + r * 512);
        f.al[r] = *reinterpret_cast<const f16x8*>(pa + o + T * 16 + r * 512);
      }
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < R; ++c) {
          acx[r][c] = mfma(f.ah[r], f.bl[c], acx[r][c]);
          acc[r][c] = mfma(f.ah[r], f.bh[c], acc[r][c]);
          acx[r][c] = mfma(f.al[r], f.bh[c], acx[r][c]);
        }
    };
    auto enter = [&](int s) {                      // slot s becomes readable, slot s - 1 writable
      if (s + NBUF - 2 < n_slots) wait_vm<LW * (NBUF - 2)>();
      else wait_vm<0>();
      __builtin_amdgcn_s_waitcnt(0xC07F);          // lgkmcnt(0): this wave's reads of slot s - 1 are in registers
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + NBUF - 1 < n_slots) fetch(s + NBUF - 1);
    };
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s)
      if (s < n_slots) fetch(s);
    if (n_slots > 0) {
      enter(0);
      read(f0, 0, 0);
    }
    for (int s = 0; s < n_slots; ++s) {
      read(f1, s, 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(f0);
      __builtin_amdgcn_sched_barrier(0);
      if (s + 1 < n_slots) {
        enter(s + 1);
        read(f0, s + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      multiply(f1);
    }
    if (partial) {
      float4* p = reinterpret_cast<float4*>(a.part) + ((long)(idx - a.n_main) * a.split + share) * NQ * 256 + tid;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < R; ++c)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[r][c][4 * g + e] + acx[r][c][4 * g + e];
            p[((r * R + c) * 4 + g) * 256] = make_float4(v[0], v[1], v[2], v[3]);
          }
      return;
    }
  }

  // Accumulator block: lane (li, lh) holds column li, rows 8 g + 4 lh + v (g, v = 0..3).
  const float da = pow2f(-ea), db = pow2f(-eb), so = pow2f(eo);
  const int ib = i0 + wm * 32 * R + (JOIN ? set / R * 32 : 0), jb = j0 + wn * 32 * R + (JOIN ? set % R * 32 : 0);
  if constexpr (KIND == K_OUT) {
    const Hyper h = get_hyper(a.h, a.hyper_dev);
    const float keep = 1.f - h.lr * h.wd, rate = h.lr * j.scale;
    const int rows = j.rows, cols = j.cols;
    typedef __attribute__((address_space(1))) float gfloat;
    gfloat* const p = (gfloat*)(float*)j.dst;
#pragma unroll
    for (int r = 0; r < RA; ++r)
#pragma unroll
      for (int c = 0; c < RA; ++c) {
        const int col = jb + c * 32 + li, row0 = ib + r * 32 + 4 * lh;
        if (col >= cols) continue;
        float old[16];
        if constexpr (DT == 3)          // (all of a block's weights are requested before the first is used)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int row = row0 + 8 * (v >> 2) + (v & 3);
            old[v] = row < rows ? p[(long)row * cols + col] : 0.f;
          }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int row = row0 + 8 * (v >> 2) + (v & 3);
          const float x = (acc[r][c][v] + acx[r][c][v]) * da * db;
          const long o = (long)row * cols + col;
          if (row < rows) {
            if constexpr (DT == 3) p[o] = fmaf(-rate, x, old[v] * keep);
            else store1<DT>(j.dst, o, x);
          }
        }
      }
    return;
  } else {
    // where the tile goes: rows of the first layout = C's columns, its K axis = C's rows; the second layout the other way round
    unsigned char* d1 = out;
    unsigned char* d2 = out;
    int rp1 = j.mp, rp2 = j.mp, lim1 = j.m, lim2 = j.m, k1 = j.mk, k2 = j.mk;
    if constexpr (KIND == K_X) {
      d1 = j.t[a.parity ^ 1]; rp1 = j.cp; lim1 = j.rows; k1 = j.rk;
      d2 = j.n[a.parity ^ 1]; rp2 = j.rp; lim2 = j.cols; k2 = j.ck;
    }
    __syncthreads();                                   // the ring becomes the transposing buffer
    float* tr = reinterpret_cast<float*>(smem) + wave * 32 * 33;
#pragma unroll
    for (int r = 0; r < RA; ++r)
#pragma unroll
      for (int c = 0; c < RA; ++c) {
        const int rb = ib + r * 32, cb = jb + c * 32;
        // A symmetric product is written once and mirrored: blocks under the diagonal are skipped, a block on it takes its own upper half
        // twice.  (Left as computed, the halves differ by their roundings, and a product with such a matrix is not S^2 but S S^T: from the
        // third step of a group on the error grew tenfold.)
        if (KIND != K_X && rb > cb) continue;
        const bool diag = KIND != K_X && rb == cb;
        float x[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = (acc[r][c][v] + acx[r][c][v]) * da * db;
        if constexpr (KIND == K_Q) {
          const int col = cb + li;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int k = rb + 8 * g + 4 * lh;
            if (k >= j.mk) continue;
            const unsigned char* sp = j.s + (((long)(k >> 3) * 2 * j.mp + col) * 16 + (k & 4) * 2);
            const f16x4 sh = *reinterpret_cast<const f16x4*>(sp), sl = *reinterpret_cast<const f16x4*>(sp + (long)j.mp * 16);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float s = ((float)sh[v] + (float)sl[v]) * da;
              x[4 * g + v] = fmaf(a.k.c, x[4 * g + v], a.k.b * s) + (k + v == col ? a.k.a : 0.f);
            }
          }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          x[v] *= so;
          tr[(8 * (v >> 2) + 4 * lh + (v & 3)) * 33 + li] = x[v];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (one wave: its LDS accesses execute in order)
        float y[16];                                            // the block's transpose: row rb + li, columns cb + 8 g + 4 lh + v
#pragma unroll
        for (int v = 0; v < 16; ++v) y[v] = tr[li * 33 + 8 * (v >> 2) + 4 * lh + (v & 3)];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int o = 8 * g + 4 * lh;
          float u[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            u[v] = diag && o + v > li ? y[4 * g + v] : x[4 * g + v];
            if (rb + o + v >= lim1) u[v] = 0.f;
          }
          if (rb + o < k1) put4(d1, rp1, cb + li, rb + o, u);
          if (diag) continue;
#pragma unroll
          for (int v = 0; v < 4; ++v) u[v] = cb + o + v < lim2 ? y[4 * g + v] : 0.f;
          if (cb + o < k2) put4(d2, rp2, rb + li, cb + o, u);
        }
      }
  }
}

// ---- the m x m products of one group as one chain, one workgroup per matrix (m <= 192) ----
// Launched product by product, a model's few hundred 192 x 192 matrices pass through the Infinity Cache at each of them (120 MB a launch: 25 us
// each, 14 launches).  Here S, then Q, sits in LDS (147 KB at m = 192) as the left operand, and a wave holds 16 columns of the right
// operand and of the result in registers: the result of one product is the right operand of the next without moving.  For that the K axis
// of a k = 32 step is permuted alike on both sides: element 4 t + v of lane quarter q is k = 32 s + 16 t + 4 q + v, which is where the
// 16 x 16 accumulators have their rows (4 q + v).  What goes to LDS is the result's transpose (8 bytes a store): with L = M^T there,
// Q = q(S^T S), W = S^T Q, P <- Q^T P and S <- Q^T W stay symmetric up to one product's rounding (no loss measured).
// P waits in memory between its products (private to the wave).  16 columns, not 32: with 32 x 32 blocks two panels of 192 rows, the
// accumulators and the fragments do not fit the 256 registers of a wave.
struct ChainArgs {
  const OrthJob* jobs;
  const int* list;
  int step0, size;
  Poly k;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int NS>                                            // NS = mk / 32: K steps of a product, half its waves and row blocks
struct Panel { f16x8 h[NS], l[NS]; };

__device__ __forceinline__ f16x4 half8(const f16x8 a, int t) { return t ? __builtin_shufflevector(a, a, 4, 5, 6, 7) : __builtin_shufflevector(a, a, 0, 1, 2, 3); }

// In LDS: [step of 32][plane][lane quarter][row][16 B]: a fragment is one ds_read_b128, a result one ds_write_b128 (with the octets of H8
// a fragment is two pieces of 8 bytes: 64 B per clock).  Three lane addresses, 48 KB apart at m = 192: every other offset is an immediate.
typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
template <int NS>
struct LdsBase { lds_byte* p[(NS + 1) / 2]; };
template <int NS>
__device__ __forceinline__ lds_f16x8* chain_at(const LdsBase<NS>& b, int s, int plane, int rb) {
  constexpr int RL = 32 * NS;
  return (lds_f16x8*)(b.p[s >> 1] + (((s & 1) * 2 + plane) * 4 * RL + rb * 16) * 16);
}
template <int NS>
__device__ __forceinline__ LdsBase<NS> chain_base(unsigned char* lds, int row, int lq) {
  LdsBase<NS> b;
#pragma unroll
  for (int k = 0; k < (NS + 1) / 2; ++k) {
    b.p[k] = (lds_byte*)lds + ((k * 16 + lq) * 32 * NS + row) * 16;
    asm volatile("" : "+v"(b.p[k]));
  }
  return b;
}

// rows 16 rb .. of L times the panel; `a`: the lane's row, octet and half
template <int NS>
__device__ __forceinline__ f32x4 chain_rows(const LdsBase<NS>& a, const Panel<NS>& b, int rb) {
  f32x4 acc = {0.f, 0.f, 0.f, 0.f}, acx = acc;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const f16x8 h = *chain_at<NS>(a, s, 0, rb), l = *chain_at<NS>(a, s, 1, rb);
    acx = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, b.l[s], acx, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, b.h[s], acc, 0, 0, 0);
    acx = __builtin_amdgcn_mfma_f32_16x16x32_f16(l, b.h[s], acx, 0, 0, 0);
  }
  asm volatile("" ::: "memory");      // (the next product over the same rows reads them again: kept from here they would spill)
  return acc + acx;
}

// two row blocks of results -> one K step of a panel (whole registers at a time: element by element the halves are kept apart)
__device__ __forceinline__ void chain_pack(const f32x4 x0, const f32x4 x1, f16x8& h, f16x8& l) {
  f16x8 hh, ll;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    _Float16 p, q;
    split16(x0[v], p, q);
    hh[v] = p; ll[v] = q;
    split16(x1[v], p, q);
    hh[4 + v] = p; ll[4 + v] = q;
  }
  u32x4 hu, lu;
  __builtin_memcpy(&hu, &hh, 16);
  __builtin_memcpy(&lu, &ll, 16);
  asm volatile("" : "+v"(hu), "+v"(lu));
  __builtin_memcpy(&h, &hu, 16);
  __builtin_memcpy(&l, &lu, 16);
}

// one K step of a panel's transpose as H8 in memory: row = the panel's column, octets = its rows
__device__ __forceinline__ void chain_store(unsigned char* base, unsigned off, unsigned ld, int s, const f16x8 h, const f16x8 l) {
  typedef __attribute__((address_space(1))) unsigned char glob_byte;
  typedef __attribute__((address_space(1))) f16x4 glob_f16x4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const unsigned o = off + (unsigned)(8 * s + 4 * t) * ld * 16u;
    *(glob_f16x4*)((glob_byte*)base + o) = half8(h, t);
    *(glob_f16x4*)((glob_byte*)base + o + ld * 16u) = half8(l, t);
  }
}

template <int NS>
__device__ __forceinline__ void chain_fill(const LdsBase<NS>& d, const Panel<NS>& b) {
#pragma unroll
  for (int s = 0; s < NS; ++s) { *chain_at<NS>(d, s, 0, 0) = b.h[s]; *chain_at<NS>(d, s, 1, 0) = b.l[s]; }
}

template <int NS>
__device__ __forceinline__ void orth_chain(const OrthJob& j, const ChainArgs& a, unsigned char* lds) {
  constexpr int RL = 32 * NS, NB = 2 * NS;                   // rows in LDS; row blocks = waves
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, lq = lane >> 4;
  const bool on = w < NB;
  const int m = j.m, mp = j.mp, col = on ? w * 16 + li : 0;
  // S into LDS, its padding cleared
  for (int i = tid; i < 8 * NS * RL; i += (int)blockDim.x) {
    const int row = i % RL, slab = i / RL;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (row < m) v = *reinterpret_cast<const u32x4*>(j.s + ((long)slab * mp + row) * 16);
    // global: [octet][plane]; the octet's halves belong to two lane quarters, as their piece t
    const int oct = slab >> 1, t = (oct >> 1) & 1, lq0 = (oct & 1) * 2;
    unsigned char* d = lds + ((((oct >> 2) * 2 + (slab & 1)) * 4 + lq0) * RL + row) * 16 + t * 8;
    *reinterpret_cast<uint2*>(d) = make_uint2(v[0], v[1]);
    *reinterpret_cast<uint2*>(d + RL * 16) = make_uint2(v[2], v[3]);
  }
  __syncthreads();
  Panel<NS> cur, out;
  if (on) {
    const LdsBase<NS> lw = chain_base<NS>(lds, col, lq);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      cur.h[s] = *chain_at<NS>(lw, s, 0, 0);
      cur.l[s] = *chain_at<NS>(lw, s, 1, 0);
    }
  }
  for (int i = 0; i < a.size; ++i) {
    const StepExp e = j.e[a.step0 + i];
    const bool last = i == a.size - 1;
    // (opaque to the compiler: it would keep the 48 comparisons and store addresses made from them in registers over the whole loop)
    int c = col - 4 * lq, ld = mp, zero = 0;
    asm volatile("" : "+v"(c), "+v"(ld), "+v"(zero));
    typedef __attribute__((address_space(1))) f16x8 glob_f16x8;
    const unsigned mine = (unsigned)(w * 2 * NS * 64 + lane + zero);
    glob_f16x8* const keep = (glob_f16x8*)(f16x8*)j.p[1] + mine;
    glob_f16x8* const park = (glob_f16x8*)(f16x8*)j.w + mine;
    const LdsBase<NS> la = chain_base<NS>(lds, li, lq);
    if (on) {                                  // out = Q
      const float ds = pow2f(-e.s), so = pow2f(e.q), a_diag = col < m ? a.k.a : 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        f32x4 x[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          x[t] = chain_rows<NS>(la, cur, 2 * s + t);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float sv = ((float)cur.h[s][4 * t + v] + (float)cur.l[s][4 * t + v]) * ds;
            x[t][v] = (fmaf(a.k.c, x[t][v] * ds * ds, a.k.b * sv) + (c == s * 32 + t * 16 + v ? a_diag : 0.f)) * so;
          }
        }
        chain_pack(x[0], x[1], out.h[s], out.l[s]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!last) {                             // cur = W = S Q
        const float dw = pow2f(-e.q) * pow2f(e.w);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const f32x4 x0 = chain_rows<NS>(la, out, 2 * s) * ds * dw, x1 = chain_rows<NS>(la, out, 2 * s + 1) * ds * dw;
          chain_pack(x0, x1, cur.h[s], cur.l[s]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (last && i == 0) {                      // a group of one step: P = Q
      if (on) {
        const unsigned off = (unsigned)((c + 4 * lq) * 16 + (lq >> 1) * 2 * ld * 16 + (lq & 1) * 8);
#pragma unroll
        for (int s = 0; s < NS; ++s) chain_store(j.p[0], off, (unsigned)ld, s, out.h[s], out.l[s]);
      }
      break;
    }
    __syncthreads();                           // every wave has read S
    if (on) {
      chain_fill<NS>(chain_base<NS>(lds, c + 4 * lq, lq), out);
      if (i == 0) {
#pragma unroll
        for (int s = 0; s < NS; ++s) { keep[(2 * s) * 64] = out.h[s]; keep[(2 * s + 1) * 64] = out.l[s]; }
      }
    }
    __syncthreads();                           // Q is whole
    constexpr bool kPark = NS > 4;             // two panels and P's results do not fit the registers there: W waits in memory too
    if (on && i > 0) {                         // P <- Q P
      if (kPark) {
#pragma unroll
        for (int s = 0; s < NS; ++s) { park[(2 * s) * 64] = cur.h[s]; park[(2 * s + 1) * 64] = cur.l[s]; }
      }
      const float dp = pow2f(-j.e[a.step0 + i - 1].p), dq = pow2f(-e.q) * pow2f(e.p);
#pragma unroll
      for (int s = 0; s < NS; ++s) { out.h[s] = keep[(2 * s) * 64]; out.l[s] = keep[(2 * s + 1) * 64]; }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        f16x8 h, l;
        const f32x4 x0 = chain_rows<NS>(la, out, 2 * s) * dp * dq, x1 = chain_rows<NS>(la, out, 2 * s + 1) * dp * dq;
        chain_pack(x0, x1, h, l);
        if (last) {
          chain_store(j.p[0], (unsigned)((c + 4 * lq) * 16 + (lq >> 1) * 2 * ld * 16 + (lq & 1) * 8), (unsigned)ld, s, h, l);
        } else {
          keep[(2 * s) * 64] = h; keep[(2 * s + 1) * 64] = l;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kPark) {
#pragma unroll
        for (int s = 0; s < NS; ++s) { cur.h[s] = park[(2 * s) * 64]; cur.l[s] = park[(2 * s + 1) * 64]; }
      }
    }
    if (last) break;
    if (on) {                                  // S <- Q W
      const float dq = pow2f(-e.q), dw = pow2f(-e.w) * pow2f(j.e[a.step0 + i + 1].s);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const f32x4 x0 = chain_rows<NS>(la, cur, 2 * s) * dq * dw, x1 = chain_rows<NS>(la, cur, 2 * s + 1) * dq * dw;
        chain_pack(x0, x1, out.h[s], out.l[s]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();                           // every wave has read Q
    if (on) { chain_fill<NS>(chain_base<NS>(lds, c + 4 * lq, lq), out); cur = out; }
    __syncthreads();
  }
}

__global__ __launch_bounds__(128 * (kChainMax / 32)) void orth_chain_k(ChainArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char chain_lds[];
  const OrthJob& j = a.jobs[a.list[blockIdx.x]];
  switch (j.mk / 32) {
    case 1: orth_chain<1>(j, a, chain_lds); break;
    case 2: orth_chain<2>(j, a, chain_lds); break;
    case 3: orth_chain<3>(j, a, chain_lds); break;
    case 4: orth_chain<4>(j, a, chain_lds); break;
    case 5: orth_chain<5>(j, a, chain_lds); break;
    default: orth_chain<6>(j, a, chain_lds); break;
  }
}

// ---- host ----
struct Groups { int n, first[kMaxSteps], size[kMaxSteps], mask; };

Groups make_groups(int steps, float a, double limit) {
  const double a2 = (double)a * a;
  int longest = 1;
  for (double lift = a2; lift <= limit && longest < steps; lift *= a2 > 1.0 ? a2 : 1.0) ++longest;
  Groups g{};
  g.n = (steps + longest - 1) / longest;
  int at = 0;
  for (int i = 0; i < g.n; ++i) {
    g.first[i] = at;
    g.size[i] = (steps - at + (g.n - i) - 1) / (g.n - i);        // as even as possible, the longer ones first
    g.mask |= 1 << at;
    at += g.size[i];
  }
  return g;
}

struct OrthPlan {
  int64_t jobs_b, ew_b, split_b, sym_b, big_b, fin_b, chain_b, head_b, total_b;
  int64_t n_ew, n_split, n_sym, n_big, n_fin;
  int n_chain[kChainMax / 32 + 1];        // chained matrices by mk / 32
  int64_t part_b;
  int k_gram, k_m, k_fin;        // mean number of K slots of a tile's product: X X^T, m x m products, P X
  int tile_sym, tile_fin, pad, chain_max;
  Groups g;
};

// How a launch of n tiles with k slots each fills the chip.  A CU holds two 128-tiles or three 64-tiles at a time; the tiles left after
// the full rounds are split along K over the idle places when that saves more than the join costs: over 32 slots of 0.3 us (a lone
// 64-tile) to 0.7 us, against 7 to 10 us.  1024 x 4096, X X^T (136 tiles, 128 slots): 44 us whole, 29 split in five and joined; at 32
// slots 13 whole, 17 split.
struct Fill { int n_main, split; };
Fill fill_for(int64_t n, int k, int tile) {
  const int64_t places = 256 * (tile == 128 ? 2 : 3), rest = n % places;
  Fill f{(int)n, 1};
  if (rest == 0) return f;
  int64_t split = places / rest;
  if (split > k / 4) split = k / 4;
  if (split > 16) split = 16;
  if (split >= 2 && k - k / split > 32) { f.n_main = (int)(n - rest); f.split = (int)split; }
  return f;
}
int64_t part_bytes(int64_t n, int k, int tile) {
  const Fill f = fill_for(n, k, tile);
  return (n - f.n_main) * f.split * (int64_t)tile * tile * 4;
}

int make_plan(const mpose_orth_job* jobs, int n_jobs, const mpose_orth_options* o, bool muon, OrthPlan& p) {
  if (n_jobs < 0 || n_jobs > 65535 || !o || (n_jobs > 0 && !jobs)) return MPOSE_EINVAL;
  if (o->steps < 1 || o->steps > kMaxSteps || o->dtype < 0 || o->dtype > 2 || !(o->eps >= 0.f) || !isfinite(o->eps)) return MPOSE_EINVAL;
  if (!isfinite(o->a) || !isfinite(o->b) || !isfinite(o->c)) return MPOSE_EINVAL;
  const Poly k{o->a, o->b, o->c};
  float bx = 1.f;
  for (int i = 0; i < o->steps; ++i) {
    if (!(bound_q(k, bx * bx) <= kGrowth)) return MPOSE_EINVAL;
    bx = bound_x(k, bx);
    if (!(bx <= kGrowth)) return MPOSE_EINVAL;
  }
  p = OrthPlan{};
  p.g = make_groups(o->steps, o->a, kLift[muon ? 2 : o->dtype == 0 ? 0 : 1]);
  // Tile sizes: 128 reads half as many operand bytes per product but wants enough tiles to fill the chip, and matrices that it does not pad by
  // more than an eighth.  4096 x 4096: symmetric products 252 us with 64, 196 with 128, P X 472 and 365; 1024 x 1024 (136 and 36 tiles): 13 and 31 us.
  int64_t area[2][2] = {}, count[2][2] = {};        // [64, 128][symmetric, P X]
  int n_between = 0;
  for (int i = 0; i < n_jobs; ++i) {
    const int rows = jobs[i].rows, cols = jobs[i].cols;
    if (rows < 1 || cols < 1 || rows > (1 << 21) || cols > (1 << 21) || (int64_t)rows * cols > (1 << 28)) return MPOSE_EINVAL;
    const int64_t m = rows < cols ? rows : cols;
    if (m > kChainFew && m <= kChainMax) ++n_between;
    for (int t = 0; t < 2; ++t) {
      const int64_t T = 64 << t, tm = (m + T - 1) / T, tf = ((rows + T - 1) / T) * ((cols + T - 1) / T);
      count[t][0] += tm * (tm + 1) / 2; count[t][1] += tf;
      area[t][0] += tm * tm * T * T; area[t][1] += tf * T * T;
    }
  }
  p.tile_sym = count[1][0] >= 384 && area[1][0] * 8 <= area[0][0] * 9 ? 128 : 64;
  p.tile_fin = count[1][1] >= 192 && area[1][1] * 8 <= area[0][1] * 9 ? 128 : 64;
  p.chain_max = n_between >= kChainMany ? kChainMax : kChainFew;
  p.pad = p.tile_sym > p.tile_fin ? p.tile_sym : p.tile_fin;
  int64_t body = 0, s_gram = 0, s_m = 0, s_fin = 0;
  for (int i = 0; i < n_jobs; ++i) {
    const int rows = jobs[i].rows, cols = jobs[i].cols;
    const OrthLayout l = orth_layout(rows, cols, p.pad, p.g.n);
    body += l.total;
    p.n_ew += l.n_part;
    p.n_split += (int64_t)((rows + 63) / 64) * ((cols + 63) / 64);
    const int m = rows < cols ? rows : cols;
    const int64_t tm = (m + p.tile_sym - 1) / p.tile_sym, ns = tm * (tm + 1) / 2;
    const int64_t nf = (int64_t)((rows + p.tile_fin - 1) / p.tile_fin) * ((cols + p.tile_fin - 1) / p.tile_fin);
    p.n_sym += ns;
    if (m <= p.chain_max) p.n_chain[l.mk / 32] += 1;
    else { p.n_big += ns; s_m += ns * (l.mk / 32); }
    p.n_fin += nf;
    s_gram += ns * ((rows < cols ? l.ck : l.rk) / 32);
    s_fin += nf * (l.mk / 32);
  }
  if (n_jobs > 0) { p.k_gram = (int)(s_gram / p.n_sym); p.k_m = p.n_big ? (int)(s_m / p.n_big) : 0; p.k_fin = (int)(s_fin / p.n_fin); }
  const int64_t parts[4] = {part_bytes(p.n_sym, p.k_gram, p.tile_sym), part_bytes(p.n_big, p.k_m, p.tile_sym), part_bytes(2 * p.n_big, p.k_m, p.tile_sym),
                            part_bytes(p.n_fin, p.k_fin, p.tile_fin)};
  for (int64_t b : parts) p.part_b = b > p.part_b ? b : p.part_b;
  if (p.n_ew > (1 << 30) || p.n_split > (1 << 30) || p.n_sym > (1 << 30) || p.n_fin > (1 << 30)) return MPOSE_EINVAL;
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  p.jobs_b = up((int64_t)n_jobs * (int64_t)sizeof(OrthJob));
  p.ew_b = up(p.n_ew * 8); p.split_b = up(p.n_split * 8); p.sym_b = up(p.n_sym * 8); p.fin_b = up(p.n_fin * 8); p.big_b = up(p.n_big * 8); p.chain_b = up((int64_t)n_jobs * 4);
  p.head_b = p.jobs_b + p.ew_b + p.split_b + p.sym_b + p.big_b + p.fin_b + p.chain_b + p.part_b;
  p.total_b = p.head_b + body;
  return 0;
}

template <int R, int NBUF, int KIND, int DT>
void gemm_tile(const GemmArgs& a, int64_t n, hipStream_t s) {
  const unsigned whole = (unsigned)((a.n_main + 7) / 8 * 8), rest = (unsigned)(n - a.n_main);
  launch(orth_gemm_k<R, NBUF, KIND, DT, false>, dim3(whole + rest * (unsigned)a.split), dim3(256), 0, s, a);
  if (rest > 0) launch(orth_gemm_k<R, NBUF, KIND, DT, true>, dim3(rest * R * R), dim3(256), 0, s, a);
}

// One product of every matrix.  k: mean number of K slots; halves: 2 when the launch makes both W and P.
template <int KIND, int DT = 0>
void gemm(GemmArgs a, int tile, int k, int halves, hipStream_t s) {
  const int64_t n = (int64_t)a.n_tiles * halves;
  const Fill f = fill_for(n, k, tile);
  a.n_main = f.n_main; a.split = f.split;
  if (tile == 128) gemm_tile<2, 2, KIND, DT>(a, n, s);
  else if (n <= 256 && f.split == 1) gemm_tile<1, 8, KIND, DT>(a, n, s);       // one tile per CU at most: a deep ring instead of neighbours
  else gemm_tile<1, 3, KIND, DT>(a, n, s);
}

int run(const mpose_orth_job* jobs, int n_jobs, const mpose_orth_options* o, bool muon, const Hyper& h, const float* hyper_dev, void* ws, int64_t ws_bytes,
        hipStream_t s) {
  OrthPlan p;
  const int rc = make_plan(jobs, n_jobs, o, muon, p);
  if (rc != 0) return rc;
  if (n_jobs == 0) return 0;
  if (!ws || ((uintptr_t)ws & 255) || ws_bytes < p.total_b) return MPOSE_EINVAL;
  const int elem = o->dtype == 0 ? 4 : 2;
  for (int i = 0; i < n_jobs; ++i) {
    if (!jobs[i].src || !jobs[i].dst || (muon && !jobs[i].buf)) return MPOSE_EINVAL;
    if (((uintptr_t)jobs[i].src | (uintptr_t)jobs[i].dst) & (uintptr_t)(elem - 1)) return MPOSE_EINVAL;
    if (muon && ((uintptr_t)jobs[i].buf & 3)) return MPOSE_EINVAL;
  }
  unsigned char* base = (unsigned char*)ws;
  SetupArgs sa{};
  sa.jobs = (OrthJob*)base; base += p.jobs_b;
  sa.ew = (int2*)base; base += p.ew_b;
  sa.split = (int2*)base; base += p.split_b;
  sa.sym = (int2*)base; base += p.sym_b;
  sa.big = (int2*)base; base += p.big_b;
  sa.chain = (int*)base; base += p.chain_b;
  sa.fin = (int2*)base; base += p.fin_b;
  float* const part = (float*)base; base += p.part_b;
  sa.pad = p.pad; sa.tile_sym = p.tile_sym; sa.tile_fin = p.tile_fin; sa.n_groups = p.g.n; sa.elem = elem;
  int ew = 0, split = 0, sym = 0, big = 0, fin = 0;
  int chain[kChainMax / 32 + 2] = {}, n_chain = 0, most = 0;      // the longest chains first
  for (int c = kChainMax / 32; c > 0; --c) {
    chain[c] = n_chain;
    n_chain += p.n_chain[c];
    if (p.n_chain[c] > 0 && most == 0) most = c;
  }
  for (int i = 0; i < n_jobs; ++i) {
    if (sa.n == 0) sa.first = i;
    SetupJob& j = sa.j[sa.n++];
    j = SetupJob{jobs[i].src, muon ? jobs[i].buf : nullptr, jobs[i].dst, base, jobs[i].rows, jobs[i].cols, jobs[i].scale, ew, split, sym, big, fin, -1};
    const OrthLayout l = orth_layout(j.rows, j.cols, p.pad, p.g.n);
    base += l.total;
    ew += l.n_part;
    split += ((j.rows + 63) / 64) * ((j.cols + 63) / 64);
    const int m = j.rows < j.cols ? j.rows : j.cols, tm = (m + p.tile_sym - 1) / p.tile_sym;
    sym += tm * (tm + 1) / 2;
    if (m <= p.chain_max) j.chain = chain[l.mk / 32]++;
    else big += tm * (tm + 1) / 2;
    fin += ((j.rows + p.tile_fin - 1) / p.tile_fin) * ((j.cols + p.tile_fin - 1) / p.tile_fin);
    if (sa.n == kSetupJobs || i == n_jobs - 1) {
      launch(orth_setup_k, dim3((unsigned)sa.n), dim3(256), 0, s, sa);
      sa.n = 0;
    }
  }
  PassArgs pa{};
  pa.jobs = sa.jobs; pa.h = h; pa.hyper_dev = hyper_dev; pa.nesterov = o->nesterov;
  const Poly k{o->a, o->b, o->c};
  pa.list = sa.ew;
  const dim3 ge((unsigned)p.n_ew), gs((unsigned)p.n_split), wg(256);
  if (muon) launch(orth_norm_k<0, true>, ge, wg, 0, s, pa);
  else if (o->dtype == 0) launch(orth_norm_k<0, false>, ge, wg, 0, s, pa);
  else if (o->dtype == 1) launch(orth_norm_k<1, false>, ge, wg, 0, s, pa);
  else launch(orth_norm_k<2, false>, ge, wg, 0, s, pa);
  launch(orth_scalars_k, dim3((unsigned)n_jobs), dim3(256), 0, s, sa.jobs, k, (double)o->eps, o->steps, p.g.mask);
  pa.list = sa.split;
  if (muon) launch(orth_split_k<0, true>, gs, wg, 0, s, pa);
  else if (o->dtype == 0) launch(orth_split_k<0, false>, gs, wg, 0, s, pa);
  else if (o->dtype == 1) launch(orth_split_k<1, false>, gs, wg, 0, s, pa);
  else launch(orth_split_k<2, false>, gs, wg, 0, s, pa);

  GemmArgs ga{};
  ga.jobs = sa.jobs; ga.k = k; ga.h = h; ga.hyper_dev = hyper_dev; ga.part = part;
  const int chain_lds = most * most * 32 * 32 * 4;
  if (n_chain > 0) {
    static bool attr_set = false;          // > 64 KiB of dynamic LDS has to be requested once per kernel
    if (!attr_set) {
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(&orth_chain_k), hipFuncAttributeMaxDynamicSharedMemorySize, kChainMax * kChainMax * 4) != hipSuccess)
        return MPOSE_EINVAL;
      attr_set = true;
    }
  }
  for (int g = 0; g < p.g.n; ++g) {
    ga.step0 = p.g.first[g]; ga.parity = g & 1;
    ga.list = sa.sym; ga.n_tiles = (int)p.n_sym;
    ga.step = ga.step0; ga.i = 0;
    gemm<K_GRAM>(ga, p.tile_sym, p.k_gram, 1, s);
    if (n_chain > 0)
      launch(orth_chain_k, dim3((unsigned)n_chain), dim3(128u * (unsigned)most), (size_t)chain_lds, s, ChainArgs{sa.jobs, sa.chain, ga.step0, p.g.size[g], k});
    ga.list = sa.big; ga.n_tiles = (int)p.n_big;
    for (int i = 0; i < p.g.size[g]; ++i) {
      ga.i = i; ga.step = ga.step0 + i;
      if (p.n_big == 0) continue;
      const bool last = i == p.g.size[g] - 1;
      gemm<K_Q>(ga, p.tile_sym, p.k_m, 1, s);
      // W = Q S unless this is the group's last step, P = Q P unless it is its first
      ga.y0 = last ? 1 : 0;
      if (!last || i > 0) gemm<K_MUL>(ga, p.tile_sym, p.k_m, (last ? 0 : 1) + (i > 0 ? 1 : 0), s);
      if (!last) gemm<K_NEXT>(ga, p.tile_sym, p.k_m, 1, s);
    }
    ga.list = sa.fin; ga.n_tiles = (int)p.n_fin;
    if (g + 1 < p.g.n) gemm<K_X>(ga, p.tile_fin, p.k_fin, 1, s);
    else if (muon) gemm<K_OUT, 3>(ga, p.tile_fin, p.k_fin, 1, s);
    else if (o->dtype == 0) gemm<K_OUT, 0>(ga, p.tile_fin, p.k_fin, 1, s);
    else if (o->dtype == 1) gemm<K_OUT, 1>(ga, p.tile_fin, p.k_fin, 1, s);
    else gemm<K_OUT, 2>(ga, p.tile_fin, p.k_fin, 1, s);
  }
  return launch_status();
}

}  // namespace
}  // namespace mpose

using namespace mpose;

extern "C" int64_t mpose_orth_ws_bytes(const mpose_orth_job* jobs, int n_jobs, const mpose_orth_options* options) {
  OrthPlan p, q;
  int rc = make_plan(jobs, n_jobs, options, false, p);
  if (rc == 0) rc = make_plan(jobs, n_jobs, options, true, q);
  if (rc != 0) return rc;
  return p.total_b > q.total_b ? p.total_b : q.total_b;
}

extern "C" int mpose_orthogonalize(const mpose_orth_job* jobs, int n_jobs, const mpose_orth_options* options, void* ws, int64_t ws_bytes, void* stream) {
  return run(jobs, n_jobs, options, false, Hyper{0.f, 0.f, 0.f, 0.f}, nullptr, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int mpose_muon_step(const mpose_orth_job* jobs, int n_jobs, const mpose_orth_options* options, const float* hyper, const float* hyper_dev, void* ws,
                               int64_t ws_bytes, void* stream) {
  if ((!hyper && !hyper_dev) || (options && options->dtype != 0)) return MPOSE_EINVAL;
  const Hyper h = hyper ? Hyper{hyper[0], hyper[1], hyper[2], hyper[3]} : Hyper{0.f, 0.f, 0.f, 0.f};
  return run(jobs, n_jobs, options, true, h, hyper ? nullptr : hyper_dev, ws, ws_bytes, (hipStream_t)stream);
}
