// Layer norm over the last axis, forward and backward (gfx950).
//
//   forward    mu = 1/D sum_j x_j,  s2 = 1/D sum_j (x_j - mu)^2,  r = (s2 + eps)^-1/2,  y_j = (x_j - mu) r gamma_j + beta_j
//   backward   h_j = (x_j - mu) r,  t_j = dy_j gamma_j,  dx_j = r (t_j - 1/D sum_k t_k - h_j 1/D sum_k t_k h_k)
//              dgamma_j = sum_rows dy_j h_j,  dbeta_j = sum_rows dy_j
//
// All arithmetic is float32 whatever the rows' type (f16 / bf16 rows are rounded once, when they are stored), but for the sums of rows too long
// for the registers, which are taken in 64 bits; the centred sum of squares is taken after the mean, not as a difference of two large
// sums.  Sums over rows are two-pass in a fixed order: n_parts partial sums of consecutive rows in the caller's workspace, then one sum
// over the parts.
#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "emx_common.h"

namespace {

using namespace emx;

constexpr int NT = 256;

// rows of D values lie `ld` elements apart; nothing is assumed of their alignment beyond the element's
struct FwdArgs {
  const void* x;
  void* y;
  const float *gamma, *beta;   // null: ones / zeros
  float *mean, *rstd;          // may be null
  long n_rows, ldx, ldy;
  int D;
  float eps;
};
struct BwdArgs {
  const void *dy, *x;
  void* dx;                    // may be null
  const float *gamma, *mean, *rstd;
  float* part;                 // [n_parts][2][D]: sums of dy h, sums of dy (null: not wanted)
  long n_rows, ld_dy, ldx, ld_dx, rows_per_part;
  int D, n_parts;
};

// the sum over groups of N lanes of a wave, in every lane (all lanes active): cross-lane moves inside rows of 16, lane swaps beyond
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));    // lane ^ 1
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));    // lane ^ 2
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));   // half mirror: quad ^ 1
  if constexpr (N > 8) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));   // mirror
  if constexpr (N > 16) v = sum_xor16(v);
  if constexpr (N > 32) v = sum_xor32(v);
  return v;
}

// the sum over the TPR threads that share a row, in each of them.  More than a wave: one slot per wave in `area`, behind ONE barrier -- the
// same area may be written again only once another barrier has been passed since it was read, so the caller has two at least and takes them in turn
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* area) {
  if constexpr (TPR <= 64) return lanes_sum<TPR>(v);
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) s += area[i];
  return s;
}
// the sum over a workgroup, in each of its threads, in 64 bits
template <int N>
__device__ __forceinline__ double block_sum64(double v, double* area /* N / 64 */) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  __syncthreads();   // (the area may still be read from the sum before)
  if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < N / 64; ++i) s += area[i];
  return s;
}

// 16 bytes of a row; the address is a multiple of the element's size only
template <typename T>
struct Lane {
  static constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T loose __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  static __device__ __forceinline__ vec load(const T* p, int left /* elements of the row from p on */) {
    if (left >= V) return *reinterpret_cast<const loose*>(p);
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : (T)0.f;
    return v;
  }
  static __device__ __forceinline__ void store(T* p, const vec v, int left) {
    if (left >= V) {
      *reinterpret_cast<loose*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) p[e] = v[e];
    }
  }
};
template <int V>
__device__ __forceinline__ void load_weights(const float* w, float other, int col, int D, float (&out)[V]) {
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    if (w != nullptr && col + 4 * q + 4 <= D) {
      const f4 v = *reinterpret_cast<const f4*>(w + col + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * q + e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * q + e] = (w != nullptr && col + 4 * q + e < D) ? w[col + 4 * q + e] : other;
    }
  }
}

// ---- rows that fit into registers: TPR threads hold a row, thread t its vectors t, t + TPR, ... (NV of them); each thread works on U
// rows at a time, whose loads are all requested before the first is used.  Bound by HBM: 1e6 x 128 f32 181 us = 5.7 TB/s (a workgroup per
// row with its sums through LDS: 969); 10007 x 1001 bf16, whose 40 MB stay in the last-level cache from call to call, 11.5 us = 3.5 TB/s, the start
// and end of so short a launch (15.5 with buffers in turn that do not); 256 x 128 3.7 us, a launch.
template <typename T, int TPR, int NV, int U>
__global__ __launch_bounds__(TPR > NT ? TPR : NT) void ln_fwd_kernel(const FwdArgs a) {
  constexpr int V = Lane<T>::V, G = (TPR > NT ? TPR : NT) / TPR;
  static_assert(TPR <= 64 || U == 1, "each of the two areas is used once: rows in turn would need them in turn");
  __shared__ float sm[2][TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.f / (float)a.D;
  const int step = TPR * V, first = t * V;
  typename Lane<T>::vec raw[U][NV];
  const long r0 = ((long)blockIdx.x * U) * G + g;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const T* x = (const T*)a.x + min(r0 + u * G, a.n_rows - 1) * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = first + i * step;
      if (col < a.D) raw[u][i] = Lane<T>::load(x + col, a.D - col);
    }
  }
  float ga[NV == 1 ? V : 1], be[NV == 1 ? V : 1];
  if constexpr (NV == 1) {
    load_weights<V>(a.gamma, 1.f, first, a.D, ga);
    load_weights<V>(a.beta, 0.f, first, a.D, be);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long r = r0 + u * G;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = a.D - (first + i * step);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[i][e] = e < left ? (float)raw[u][i][e] : 0.f;
        s += v[i][e];
      }
    }
    const float mu = row_sum<TPR>(s, sm[0]) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = a.D - (first + i * step);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[i][e] -= mu;
        s = e < left ? fmaf(v[i][e], v[i][e], s) : s;
      }
    }
    const float rs = 1.f / sqrtf(fmaf(row_sum<TPR>(s, sm[1]), inv, a.eps));
    if (r < a.n_rows) {
      T* y = (T*)a.y + r * a.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = first + i * step;
        if (col < a.D) {
          float gi[V], bi[V];
          if constexpr (NV > 1) {
            load_weights<V>(a.gamma, 1.f, col, a.D, gi);
            load_weights<V>(a.beta, 0.f, col, a.D, bi);
          }
          typename Lane<T>::vec o;
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = (T)fmaf(v[i][e] * rs, NV == 1 ? ga[NV == 1 ? e : 0] : gi[e], NV == 1 ? be[NV == 1 ? e : 0] : bi[e]);
          Lane<T>::store(y + col, o, a.D - col);
        }
      }
      if (t == 0) {
        if (a.mean) a.mean[r] = mu;
        if (a.rstd) a.rstd[r] = rs;
      }
    }
  }
}

// ---- backward, rows that fit into registers: workgroup p walks the rows of part p, G at a time, TPR threads to a row; a thread keeps the
// sums of ITS columns over the part's rows, the G groups' are added through LDS at the end.  The next rows' loads travel under this row's sums.
// Bound by HBM: 65536 x 1024 bf16 87 us = 4.6 TB/s; 2047 x 2850 f32, whose 70 MB stay in the last-level cache, 18.3 us (with the sum of the parts 20.8,
// and 25.3 with buffers in turn that do not) -- where twice and half the threads, vectors or parts are all within 5 %; 4096 x 128 f32 3.8 us.
// 16-bit rows of more than 8192 values spill fifteen registers a thread (4096 x 12288 bf16 154 us, 16384 131); with gamma read again for each row
// instead of kept the compiler spills others, and the times are the same.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > NT ? TPR : NT) void ln_bwd_kernel(const BwdArgs a) {
  constexpr int V = Lane<T>::V, NB = TPR > NT ? TPR : NT, G = NB / TPR;
  constexpr int CW = TPR * V;                                // columns of one vector of all threads of a row
  __shared__ float sm[2][2][TPR > 64 ? TPR / 64 : 1];
  __shared__ float fold[G > 1 ? G * CW : 1];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.f / (float)a.D;
  const long r0 = blockIdx.x * a.rows_per_part, r1 = min(r0 + a.rows_per_part, a.n_rows);
  float dg[NV][V], db[NV][V], gam[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_weights<V>(a.gamma, 1.f, t * V + i * CW, a.D, gam[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) dg[i][e] = db[i][e] = 0.f;
  }
  typename Lane<T>::vec rx[NV], rd[NV];
  float nmu = 0.f, nrs = 0.f;
  auto request = [&](const long row) __attribute__((always_inline)) {
    const long r = min(row, a.n_rows - 1);
    const T *x = (const T*)a.x + r * a.ldx, *dy = (const T*)a.dy + r * a.ld_dy;
    nmu = a.mean[r], nrs = a.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = t * V + i * CW;
      if (col < a.D) {
        rx[i] = Lane<T>::load(x + col, a.D - col);
        rd[i] = Lane<T>::load(dy + col, a.D - col);
      }
    }
  };
  if (r0 < r1) request(r0 + g);
  int flip = 0;
  for (long rb = r0; rb < r1; rb += G, flip ^= 1) {
    const long r = rb + g;
    const float mu = nmu, rs = nrs;
    float h[NV][V], d[NV][V];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = a.D - (t * V + i * CW);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[i][e] = e < left ? ((float)rx[i][e] - mu) * rs : 0.f;
        d[i][e] = e < left ? (float)rd[i][e] : 0.f;
      }
    }
    if (rb + G < r1) request(r + G);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (r < r1) {   // (uniform over the threads of a row; the rows behind the part's end are another part's, or none)
          dg[i][e] = fmaf(d[i][e], h[i][e], dg[i][e]);
          db[i][e] += d[i][e];
        }
        d[i][e] *= gam[i][e];
        s += d[i][e];
        q = fmaf(d[i][e], h[i][e], q);
      }
    }
    if (a.dx == nullptr) continue;
    s = row_sum<TPR>(s, sm[flip][0]) * inv;
    q = row_sum<TPR>(q, sm[flip][1]) * inv;
    if (r < r1) {
      T* dx = (T*)a.dx + r * a.ld_dx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = t * V + i * CW;
        if (col < a.D) {
          typename Lane<T>::vec o;
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = (T)(rs * (d[i][e] - fmaf(h[i][e], q, s)));
          Lane<T>::store(dx + col, o, a.D - col);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  float* out = a.part + (long)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (G > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) fold[g * CW + t * V + e] = which ? db[i][e] : dg[i][e];
        __syncthreads();
        for (int c = threadIdx.x; c < CW; c += NB) {
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < G; ++k) s += fold[k * CW + c];
          if (i * CW + c < a.D) out[(long)which * a.D + i * CW + c] = s;
        }
      } else {
        const int col = t * V + i * CW;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (col + e < a.D) out[(long)which * a.D + col + e] = which ? db[i][e] : dg[i][e];
      }
    }
  }
}

// ---- rows of any length: one workgroup per row walks it once per sum, four vectors of each thread on their way at a time.  A vector's values are
// added in 32 bits, the vectors of a thread -- up to 2^16 of them -- in 64 (in 32 the roundings of equal terms all go one way: 2^20 times
// 1.1 comes out 1 % off).  4096 x 20000 f32 forward 169-184 us = 3.6-3.9 TB/s of what has to move (the second and third walk find the row in the caches),
// backward 400-415, three walks and the sums over rows; 4096 x 12288 f32 backward 250, 16384 341; two rows of 2^24 3.4 and 6.0 ms, one CU each: fewer rows
// than CUs leave the others idle.  Eight loads in flight: within 4 % either way.
constexpr int LONG_NT = 1024, LONG_U = 4;
template <typename T, typename F>
__device__ __forceinline__ void walk(const T* x, int D, F take /* (vector, its first column, elements of the row from there on) */) {
  constexpr int V = Lane<T>::V, step = LONG_NT * V;
  for (int c0 = threadIdx.x * V; c0 < D; c0 += LONG_U * step) {
    typename Lane<T>::vec raw[LONG_U];
#pragma unroll
    for (int u = 0; u < LONG_U; ++u)
      if (c0 + u * step < D) raw[u] = Lane<T>::load(x + c0 + u * step, D - (c0 + u * step));
#pragma unroll
    for (int u = 0; u < LONG_U; ++u)
      if (c0 + u * step < D) take(raw[u], c0 + u * step, D - (c0 + u * step));
  }
}
template <typename T, typename F>
__device__ __forceinline__ void walk_two(const T* x, const T* dy, int D, F take) {
  constexpr int V = Lane<T>::V, step = LONG_NT * V;
  for (int c0 = threadIdx.x * V; c0 < D; c0 += LONG_U * step) {
    typename Lane<T>::vec rx[LONG_U], rd[LONG_U];
#pragma unroll
    for (int u = 0; u < LONG_U; ++u)
      if (c0 + u * step < D) {
        rx[u] = Lane<T>::load(x + c0 + u * step, D - (c0 + u * step));
        rd[u] = Lane<T>::load(dy + c0 + u * step, D - (c0 + u * step));
      }
#pragma unroll
    for (int u = 0; u < LONG_U; ++u)
      if (c0 + u * step < D) take(rx[u], rd[u], c0 + u * step, D - (c0 + u * step));
  }
}

template <typename T>
__global__ __launch_bounds__(LONG_NT) void ln_fwd_long_kernel(const FwdArgs a) {
  constexpr int V = Lane<T>::V;
  typedef typename Lane<T>::vec vec;
  __shared__ double sm[LONG_NT / 64];
  const double inv = 1.0 / (double)a.D;
  for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    T* y = (T*)a.y + r * a.ldy;
    double s = 0.0;
    walk<T>(x, a.D, [&](const vec v, int, int left) __attribute__((always_inline)) {
      float p = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) p += e < left ? (float)v[e] : 0.f;
      s += (double)p;
    });
    const float mu = (float)(block_sum64<LONG_NT>(s, sm) * inv);
    s = 0.0;
    walk<T>(x, a.D, [&](const vec v, int, int left) __attribute__((always_inline)) {
      float p = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float c = (float)v[e] - mu;
        p = e < left ? fmaf(c, c, p) : p;
      }
      s += (double)p;
    });
    const float rs = (float)(1.0 / sqrt(fma(block_sum64<LONG_NT>(s, sm), inv, (double)a.eps)));
    walk<T>(x, a.D, [&](const vec v, int col, int left) __attribute__((always_inline)) {
      float ga[V], be[V];
      load_weights<V>(a.gamma, 1.f, col, a.D, ga);
      load_weights<V>(a.beta, 0.f, col, a.D, be);
      vec o;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = (T)fmaf(((float)v[e] - mu) * rs, ga[e], be[e]);
      Lane<T>::store(y + col, o, left);
    });
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mu;
      if (a.rstd) a.rstd[r] = rs;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LONG_NT) void ln_bwd_long_kernel(const BwdArgs a) {
  constexpr int V = Lane<T>::V;
  typedef typename Lane<T>::vec vec;
  __shared__ double sm[LONG_NT / 64];
  const double inv = 1.0 / (double)a.D;
  for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    const T* dy = (const T*)a.dy + r * a.ld_dy;
    T* dx = (T*)a.dx + r * a.ld_dx;
    const float mu = a.mean[r], rs = a.rstd[r];
    double s64 = 0.0, q64 = 0.0;
    walk_two<T>(x, dy, a.D, [&](const vec v, const vec d, int col, int left) __attribute__((always_inline)) {
      float ga[V], p = 0.f, q = 0.f;
      load_weights<V>(a.gamma, 1.f, col, a.D, ga);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float t = e < left ? (float)d[e] * ga[e] : 0.f, h = e < left ? ((float)v[e] - mu) * rs : 0.f;
        p += t;
        q = fmaf(t, h, q);
      }
      s64 += (double)p;
      q64 += (double)q;
    });
    const float s = (float)(block_sum64<LONG_NT>(s64, sm) * inv), q = (float)(block_sum64<LONG_NT>(q64, sm) * inv);
    walk_two<T>(x, dy, a.D, [&](const vec v, const vec d, int col, int left) __attribute__((always_inline)) {
      float ga[V];
      load_weights<V>(a.gamma, 1.f, col, a.D, ga);
      vec o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = ((float)v[e] - mu) * rs;
        o[e] = (T)(rs * ((float)d[e] * ga[e] - fmaf(h, q, s)));
      }
      Lane<T>::store(dx + col, o, left);
    });
  }
}

// ---- sums over rows: workgroup (c, p) adds the rows of part p for 256 columns, a column per thread
template <typename T>
__global__ __launch_bounds__(NT) void ln_part_kernel(const BwdArgs a) {
  const long j = (long)blockIdx.x * NT + threadIdx.x;
  if (j >= a.D) return;
  const long r0 = blockIdx.y * a.rows_per_part, r1 = min(r0 + a.rows_per_part, a.n_rows);
  float dg = 0.f, db = 0.f;
  for (long r = r0; r < r1; ++r) {
    const float d = (float)((const T*)a.dy)[r * a.ld_dy + j];
    dg = fmaf(d, ((float)((const T*)a.x)[r * a.ldx + j] - a.mean[r]) * a.rstd[r], dg);
    db += d;
  }
  float* p = a.part + (long)blockIdx.y * 2 * a.D;
  p[j] = dg;
  p[a.D + j] = db;
}

// out[e] = sum over the parts of column e, for the 2 D columns (dgamma | dbeta): 32 columns and 32 shares of the parts per workgroup.
// 1024 parts of 1024 columns (8 MB): 4.2 us; 512 of 128: 2.2, a launch.
constexpr int SUM_NT = 1024;
__global__ __launch_bounds__(SUM_NT) void ln_sum_kernel(const float* __restrict__ part, int n_parts, int D, float* __restrict__ dgamma,
                                                        float* __restrict__ dbeta) {
  __shared__ float sm[32][33];
  const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long E = 2l * D;
  for (long e0 = (long)blockIdx.x * 32; e0 < E; e0 += (long)gridDim.x * 32) {   // (once, but for rows of more than 2^24 values)
    const long e = e0 + c;
    double s = 0.0;   // (up to 2048 parts)
    if (e < E) {
#pragma unroll 8
      for (int p = w; p < n_parts; p += 32) s += (double)part[(long)p * E + e];
    }
    sm[w][c] = (float)s;
    __syncthreads();
    if (w == 0 && e < E) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) v += sm[k][c];
      float* out = e < D ? dgamma : dbeta;
      if (out) out[e < D ? e : e - D] = v;
    }
    if (e0 + (long)gridDim.x * 32 < E) __syncthreads();
  }
}

// ... a column per thread, for at most 32 parts of many columns (one part of 2^24 columns: 72 us against 2260, 32 of 200000: 10.5 against 41; 32 of
// 5000 columns the other way round: 3.3 against 2.6)
constexpr int FEW_PARTS = 32, MANY_COLUMNS = 16384;
__global__ __launch_bounds__(NT) void ln_sum_few_kernel(const float* __restrict__ part, int n_parts, int D, float* __restrict__ dgamma,
                                                        float* __restrict__ dbeta) {
  const long E = 2l * D, e = (long)blockIdx.x * NT + threadIdx.x;
  float* const out = e < D ? dgamma : dbeta;
  if (e >= E || out == nullptr) return;
  double s = 0.0;
#pragma unroll 8
  for (int p = 0; p < n_parts; ++p) s += (double)part[(long)p * E + e];
  out[e < D ? e : e - D] = (float)s;
}

// The parts of a backward pass: consecutive rows each, at most 512 of them while a launch's second dimension (65535) allows it -- a thread adds
// a part's rows one after the other in 32 bits.
int parts_of(long n_rows, int D) {
  if (n_rows <= 0) return 0;
  const long cap = std::min(1024l, std::max(32l, (4l << 20) / D));
  return (int)std::min((n_rows + 7) / 8, std::max(cap, std::min((n_rows + 511) / 512, 65535l)));
}

bool known_type(int dtype) { return dtype == EMX_F32 || dtype == EMX_F16 || dtype == EMX_BF16; }
size_t size_of(int dtype) { return dtype == EMX_F32 ? 4 : 2; }

// row offsets stay far inside 64 bits
bool fits(int64_t n, int64_t ld) { return ld >= 0 && n <= ((int64_t)1 << 58) / std::max<int64_t>(ld, 1); }
bool aligned(const void* p, size_t es) { return (uintptr_t)p % es == 0; }

// Is [a, a + n rows) clear of [b, ...), or the very same rows (the in-place form)?  Clear are also different columns of rows of one stride
// (blocks of one wider buffer), whichever rows: their places modulo the stride differ.
bool disjoint_or_same(const void* a, long lda, const void* b, long ldb, long n, int D, size_t es) {
  if (a == b && lda == ldb) return true;
  const char *a0 = (const char*)a, *b0 = (const char*)b;
  const char *a1 = a0 + ((n - 1) * lda + D) * es, *b1 = b0 + ((n - 1) * ldb + D) * es;
  if (a1 <= b0 || b1 <= a0) return true;
  if (lda != ldb || lda <= 0) return false;
  const long stride = lda * (long)es, width = D * (long)es, ahead = (b0 - a0) % stride, shift = ahead < 0 ? ahead + stride : ahead;
  return shift >= width && shift + width <= stride;
}

// The memory of an operand, from its first element to its last (rows) or of n floats; none: null
struct Span {
  const char *lo, *hi;
};
Span rows_of(const void* p, long ld, long n, int D, size_t es) {
  const char* lo = (const char*)p;
  return {lo, p ? lo + ((n - 1) * ld + D) * es : lo};
}
Span vector_of(const float* p, size_t n) { return {(const char*)p, (const char*)(p ? p + n : p)}; }
// does what is written share memory with any of the others?
bool meets(Span out, std::initializer_list<Span> others) {
  for (const Span& o : others)
    if (out.lo && o.lo && out.lo < o.hi && o.lo < out.hi) return true;
  return false;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == EMX_F16) return f((_Float16)0);
  if (dtype == EMX_BF16) return f((__bf16)0);
  return f(0.f);
}

// (a launch has fewer than 2^32 threads: 2^31 at most here, the rows behind them in the next one)
template <typename T, int TPR, int NV, int U>
int start_fwd(const char* who, const FwdArgs& all, hipStream_t st) {
  constexpr int NB = TPR > NT ? TPR : NT;
  constexpr long rows = (long)(NB / TPR) * U, most = rows * ((1l << 31) / NB);
  for (long r0 = 0; r0 < all.n_rows; r0 += most) {
    FwdArgs a = all;
    a.x = (const T*)all.x + r0 * all.ldx;
    a.y = (T*)all.y + r0 * all.ldy;
    a.mean = all.mean ? all.mean + r0 : nullptr;
    a.rstd = all.rstd ? all.rstd + r0 : nullptr;
    a.n_rows = std::min(all.n_rows - r0, most);
    hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV, U>), dim3((unsigned)((a.n_rows + rows - 1) / rows)), dim3(NB), 0, st, a);
    if (const int rc = check_launch(who)) return rc;
  }
  return EMX_OK;
}
template <typename T>
int launch_fwd(const char* who, const FwdArgs& a, hipStream_t st) {
  const int nv = (a.D + Lane<T>::V - 1) / Lane<T>::V;   // 16-byte vectors of a row
  if (nv <= 8) return start_fwd<T, 8, 1, 4>(who, a, st);
  if (nv <= 16) return start_fwd<T, 16, 1, 4>(who, a, st);
  if (nv <= 32) return start_fwd<T, 32, 1, 4>(who, a, st);
  if (nv <= 64) return start_fwd<T, 64, 1, 4>(who, a, st);
  if (nv <= 128) return start_fwd<T, 64, 2, 2>(who, a, st);
  if (nv <= 256) return start_fwd<T, 64, 4, 1>(who, a, st);
  if (nv <= 512) return start_fwd<T, 256, 2, 1>(who, a, st);
  if (nv <= 1024) return start_fwd<T, 256, 4, 1>(who, a, st);
  if (nv <= 2048) return start_fwd<T, 1024, 2, 1>(who, a, st);
  if (nv <= 4096) return start_fwd<T, 1024, 4, 1>(who, a, st);
  hipLaunchKernelGGL(ln_fwd_long_kernel<T>, dim3((unsigned)std::min<long>(a.n_rows, 1 << 20)), dim3(LONG_NT), 0, st, a);
  return check_launch(who);
}
template <typename T, int TPR, int NV>
bool start_bwd(const BwdArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV>), dim3(a.n_parts), dim3(TPR > NT ? TPR : NT), 0, st, a);
  return true;
}
// false: the row is too long for the registers
template <typename T>
bool launch_bwd(const BwdArgs& a, hipStream_t st) {
  const int nv = (a.D + Lane<T>::V - 1) / Lane<T>::V;
  if (nv <= 8) return start_bwd<T, 8, 1>(a, st);
  if (nv <= 16) return start_bwd<T, 16, 1>(a, st);
  if (nv <= 32) return start_bwd<T, 32, 1>(a, st);
  if (nv <= 64) return start_bwd<T, 64, 1>(a, st);
  if (nv <= 128) return start_bwd<T, 64, 2>(a, st);
  if (nv <= 256) return start_bwd<T, 256, 1>(a, st);
  if (nv <= 512) return start_bwd<T, 256, 2>(a, st);
  if (nv <= 1024) return start_bwd<T, 512, 2>(a, st);
  if (nv <= 2048) return start_bwd<T, 1024, 2>(a, st);
  return false;
}

}  // namespace

extern "C" {

int emx_layernorm_fwd(const void* x, int dtype, int64_t n_rows, int D, int64_t ldx, const float* gamma, const float* beta, float eps, void* y,
                      int64_t ldy, float* mean, float* rstd, emx_stream_t stream) {
  const char* who = "emx_layernorm_fwd";
  EMX_REQUIRE(known_type(dtype), "%s: element type %d", who, dtype);
  EMX_REQUIRE(n_rows >= 0 && D >= 1 && D <= EMX_LAYERNORM_MAX_D, "%s: n_rows %lld, D %d", who, (long long)n_rows, D);
  EMX_REQUIRE(eps >= 0.f, "%s: eps %g", who, (double)eps);   // (refuses NaN)
  if (n_rows == 0) return EMX_OK;
  EMX_REQUIRE(aligned(gamma, 4) && aligned(beta, 4) && aligned(mean, 4) && aligned(rstd, 4), "%s: gamma, beta, mean and rstd on float boundaries", who);
  EMX_REQUIRE(!mean || mean != rstd, "%s: mean and rstd are the same vector", who);
  EMX_REQUIRE(x && y && aligned(x, size_of(dtype)) && aligned(y, size_of(dtype)), "%s: x and y are needed, on element boundaries", who);
  EMX_REQUIRE(n_rows == 1 || (fits(n_rows, ldx) && fits(n_rows, ldy) && ldy >= D), "%s: row strides %lld, %lld of %d columns", who, (long long)ldx, (long long)ldy, D);
  if (n_rows == 1) ldx = ldy = D;
  EMX_REQUIRE(disjoint_or_same(x, ldx, y, ldy, n_rows, D, size_of(dtype)), "%s: x and y overlap without being the same rows", who);
  const Span rx = rows_of(x, ldx, n_rows, D, size_of(dtype)), ry = rows_of(y, ldy, n_rows, D, size_of(dtype));
  const Span vg = vector_of(gamma, D), vb = vector_of(beta, D), vm = vector_of(mean, n_rows), vr = vector_of(rstd, n_rows);
  EMX_REQUIRE(!meets(ry, {vg, vb}) && !meets(vm, {rx, ry, vg, vb, vr}) && !meets(vr, {rx, ry, vg, vb}), "%s: what is written shares memory with another operand", who);
  const FwdArgs a{x, y, gamma, beta, mean, rstd, n_rows, ldx, ldy, D, eps};
  return by_type(dtype, [&](auto t) {
    return launch_fwd<decltype(t)>(who, a, (hipStream_t)stream);
  });
}

size_t emx_layernorm_ws_floats(int64_t n_rows, int D) { return D < 1 ? 0 : (size_t)parts_of(n_rows, D) * 2 * (size_t)D; }

int emx_layernorm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, int dtype, int64_t n_rows, int D, const float* gamma,
                      const float* mean, const float* rstd, void* dx, int64_t ld_dx, float* dgamma, float* dbeta, float* ws, size_t ws_floats,
                      emx_stream_t stream) {
  const char* who = "emx_layernorm_bwd";
  EMX_REQUIRE(known_type(dtype), "%s: element type %d", who, dtype);
  EMX_REQUIRE(n_rows >= 0 && D >= 1 && D <= EMX_LAYERNORM_MAX_D, "%s: n_rows %lld, D %d", who, (long long)n_rows, D);
  const bool sums = dgamma || dbeta;
  const size_t es = size_of(dtype);
  EMX_REQUIRE(aligned(gamma, 4) && aligned(mean, 4) && aligned(rstd, 4) && aligned(dgamma, 4) && aligned(dbeta, 4) && aligned(ws, 4),
              "%s: vectors and workspace on float boundaries", who);
  if (n_rows > 0) {
    EMX_REQUIRE(dy && x && mean && rstd && aligned(dy, es) && aligned(x, es) && aligned(dx, es), "%s: dy, x, mean and rstd are needed, on element boundaries", who);
    EMX_REQUIRE(n_rows == 1 || (fits(n_rows, ld_dy) && fits(n_rows, ldx) && (!dx || (fits(n_rows, ld_dx) && ld_dx >= D))), "%s: row strides %lld, %lld, %lld of %d columns", who,
                (long long)ld_dy, (long long)ldx, (long long)ld_dx, D);
    if (n_rows == 1) ld_dy = ldx = ld_dx = D;
    EMX_REQUIRE(!dx || (disjoint_or_same(dx, ld_dx, dy, ld_dy, n_rows, D, es) && disjoint_or_same(dx, ld_dx, x, ldx, n_rows, D, es)),
                "%s: dx overlaps dy or x without being the same rows", who);
  }
  const int parts = parts_of(n_rows, D);
  if (sums && parts > 0 && (!ws || ws_floats < emx_layernorm_ws_floats(n_rows, D)))
    return fail(EMX_EWORKSPACE, "%s: workspace of %zu floats, %zu needed", who, ws ? ws_floats : (size_t)0, emx_layernorm_ws_floats(n_rows, D));
  EMX_REQUIRE(!dgamma || dgamma != dbeta, "%s: dgamma and dbeta are the same vector", who);
  if (n_rows > 0) {
    // (dgamma and dbeta are written when everything but the parts has been read)
    const Span rdy = rows_of(dy, ld_dy, n_rows, D, es), rx = rows_of(x, ldx, n_rows, D, es), rdx = rows_of(dx, ld_dx, n_rows, D, es);
    const Span vg = vector_of(gamma, D), vm = vector_of(mean, n_rows), vr = vector_of(rstd, n_rows), part = vector_of(sums ? ws : nullptr, emx_layernorm_ws_floats(n_rows, D));
    EMX_REQUIRE(!meets(rdx, {vg, vm, vr}) && !meets(part, {rdy, rx, rdx, vg, vm, vr}), "%s: what is written shares memory with another operand", who);
    EMX_REQUIRE(!meets(vector_of(dgamma, D), {rdx, part}) && !meets(vector_of(dbeta, D), {rdx, part}), "%s: what is written shares memory with another operand", who);
  }
  EMX_REQUIRE(!meets(vector_of(dgamma, D), {vector_of(dbeta, D)}), "%s: dgamma and dbeta share memory", who);
  hipStream_t st = (hipStream_t)stream;
  if (n_rows > 0) {
    const BwdArgs a{dy, x, dx, gamma, mean, rstd, sums ? ws : nullptr, n_rows, ld_dy, ldx, ld_dx, (n_rows + parts - 1) / parts, D, parts};
    const int rc = by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (launch_bwd<T>(a, st)) return check_launch(who);
      if (sums) {   // (first: dx may lie where dy or x does)
        hipLaunchKernelGGL(ln_part_kernel<T>, dim3((D + NT - 1) / NT, parts), dim3(NT), 0, st, a);
        const int r = check_launch(who);
        if (r) return r;
      }
      if (dx) {
        hipLaunchKernelGGL(ln_bwd_long_kernel<T>, dim3((unsigned)std::min<int64_t>(n_rows, 1 << 20)), dim3(LONG_NT), 0, st, a);
        return check_launch(who);
      }
      return (int)EMX_OK;
    });
    if (rc) return rc;
  }
  if (!sums) return EMX_OK;
  if (parts <= FEW_PARTS && D >= MANY_COLUMNS) hipLaunchKernelGGL(ln_sum_few_kernel, dim3((unsigned)((2l * D + NT - 1) / NT)), dim3(NT), 0, st, ws, parts, D, dgamma, dbeta);
  else hipLaunchKernelGGL(ln_sum_kernel, dim3((unsigned)std::min((2l * D + 31) / 32, 1l << 20)), dim3(SUM_NT), 0, st, ws, parts, D, dgamma, dbeta);
  return check_launch(who);
}

}  // extern "C"
