// Layer norm over the last axis, forward and backward (gfx950).
//
//   forward    mu = 1/D sum_j x_j,  s2 = 1/D sum_j (x_j - mu)^2,  r = (s2 + eps)^-1/2,  y_j = (x_j - mu) r gamma_j + beta_j
//   backward   h_j = (x_j - mu) r,  t_j = dy_j gamma_j,  dx_j = r (t_j - 1/D sum_k t_k - h_j 1/D sum_k t_k h_k)
//              dgamma_j = sum_rows dy_j h_j,  dbeta_j = sum_rows dy_j
//
// All arithmetic is float32 whatever the rows' type (f16 / bf16 rows are rounded once, when they are stored); the centred sum of
// squares is taken after the mean, not as a difference of two large sums.  Sums over rows are two-pass in a fixed order: n_parts
// partial sums of consecutive rows in the caller's workspace, then one sum over the parts.
#include <algorithm>

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

// the sum over all threads of a block, in every thread
template <int N>
__device__ __forceinline__ float block_all_sum(float v, float* smem /* N / 64 floats */) {
  v = wave_sum(v);
  if constexpr (N > 64) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();   // (the area may still be read from the sum before)
    if (lane == 0) smem[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < N / 64; ++i) v += smem[i];
  }
  return v;
}

// ---- rows of any length: one workgroup per row, the row is walked once per sum
template <typename T>
__global__ __launch_bounds__(NT) void ln_fwd_long_kernel(const FwdArgs a) {
  __shared__ float sm[NT / 64];
  const float inv = 1.f / (float)a.D;
  for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    T* y = (T*)a.y + r * a.ldy;
    float s = 0.f;
    for (int j = threadIdx.x; j < a.D; j += NT) s += (float)x[j];
    const float mu = block_all_sum<NT>(s, sm) * inv;
    s = 0.f;
    for (int j = threadIdx.x; j < a.D; j += NT) {
      const float c = (float)x[j] - mu;
      s = fmaf(c, c, s);
    }
    const float rs = 1.f / sqrtf(fmaf(block_all_sum<NT>(s, sm), inv, a.eps));
    for (int j = threadIdx.x; j < a.D; j += NT)
      y[j] = (T)fmaf(((float)x[j] - mu) * rs, a.gamma ? a.gamma[j] : 1.f, a.beta ? a.beta[j] : 0.f);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mu;
      if (a.rstd) a.rstd[r] = rs;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void ln_bwd_long_kernel(const BwdArgs a) {
  __shared__ float sm[NT / 64];
  const float inv = 1.f / (float)a.D;
  for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const T* x = (const T*)a.x + r * a.ldx;
    const T* dy = (const T*)a.dy + r * a.ld_dy;
    T* dx = (T*)a.dx + r * a.ld_dx;
    const float mu = a.mean[r], rs = a.rstd[r];
    float s = 0.f, q = 0.f;
    for (int j = threadIdx.x; j < a.D; j += NT) {
      const float t = (float)dy[j] * (a.gamma ? a.gamma[j] : 1.f);
      s += t;
      q = fmaf(t, ((float)x[j] - mu) * rs, q);
    }
    s = block_all_sum<NT>(s, sm) * inv;
    q = block_all_sum<NT>(q, sm) * inv;
    for (int j = threadIdx.x; j < a.D; j += NT) {
      const float t = (float)dy[j] * (a.gamma ? a.gamma[j] : 1.f), h = ((float)x[j] - mu) * rs;
      dx[j] = (T)(rs * (t - fmaf(h, q, s)));
    }
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

// out[e] = sum over the parts of column e, for the 2 D columns (dgamma | dbeta)
__global__ __launch_bounds__(NT) void ln_sum_kernel(const float* __restrict__ part, int n_parts, int D, float* __restrict__ dgamma,
                                                    float* __restrict__ dbeta) {
  const long e = (long)blockIdx.x * NT + threadIdx.x;
  if (e >= 2l * D) return;
  float s = 0.f;
  for (int p = 0; p < n_parts; ++p) s += part[(long)p * 2 * D + e];
  float* out = e < D ? dgamma : dbeta;
  if (out) out[e < D ? e : e - D] = s;
}

// The parts of a backward pass: consecutive rows each.
int parts_of(long n_rows, int D) {
  if (n_rows <= 0) return 0;
  const long cap = std::min(512l, std::max(32l, (4l << 20) / D));
  return (int)std::min((n_rows + 15) / 16, cap);
}

bool known_type(int dtype) { return dtype == EMX_F32 || dtype == EMX_F16 || dtype == EMX_BF16; }
size_t size_of(int dtype) { return dtype == EMX_F32 ? 4 : 2; }

// Is [a, a + n rows) clear of [b, ...), or the very same rows (the in-place form)?
bool disjoint_or_same(const void* a, long lda, const void* b, long ldb, long n, int D, size_t es) {
  if (a == b && lda == ldb) return true;
  const char *a0 = (const char*)a, *b0 = (const char*)b;
  const char *a1 = a0 + ((n - 1) * lda + D) * es, *b1 = b0 + ((n - 1) * ldb + D) * es;
  return a1 <= b0 || b1 <= a0;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == EMX_F16) return f((_Float16)0);
  if (dtype == EMX_BF16) return f((__bf16)0);
  return f(0.f);
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
  EMX_REQUIRE(x && y, "%s: x and y are needed", who);
  EMX_REQUIRE(n_rows == 1 || (ldx >= 0 && ldy >= D), "%s: row strides %lld, %lld of %d columns", who, (long long)ldx, (long long)ldy, D);
  if (n_rows == 1) ldx = ldy = D;
  EMX_REQUIRE(disjoint_or_same(x, ldx, y, ldy, n_rows, D, size_of(dtype)), "%s: x and y overlap without being the same rows", who);
  const FwdArgs a{x, y, gamma, beta, mean, rstd, n_rows, ldx, ldy, D, eps};
  return by_type(dtype, [&](auto t) {
    hipLaunchKernelGGL(ln_fwd_long_kernel<decltype(t)>, dim3((unsigned)std::min<int64_t>(n_rows, 1 << 20)), dim3(NT), 0, (hipStream_t)stream, a);
    return check_launch(who);
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
  if (n_rows > 0) {
    EMX_REQUIRE(dy && x && mean && rstd, "%s: dy, x, mean and rstd are needed", who);
    EMX_REQUIRE(n_rows == 1 || (ld_dy >= 0 && ldx >= 0 && (!dx || ld_dx >= D)), "%s: row strides %lld, %lld, %lld of %d columns", who,
                (long long)ld_dy, (long long)ldx, (long long)ld_dx, D);
    if (n_rows == 1) ld_dy = ldx = ld_dx = D;
    EMX_REQUIRE(!dx || (disjoint_or_same(dx, ld_dx, dy, ld_dy, n_rows, D, es) && disjoint_or_same(dx, ld_dx, x, ldx, n_rows, D, es)),
                "%s: dx overlaps dy or x without being the same rows", who);
  }
  const int parts = parts_of(n_rows, D);
  if (sums && parts > 0 && (!ws || ws_floats < emx_layernorm_ws_floats(n_rows, D)))
    return fail(EMX_EWORKSPACE, "%s: workspace of %zu floats, %zu needed", who, ws ? ws_floats : (size_t)0, emx_layernorm_ws_floats(n_rows, D));
  hipStream_t st = (hipStream_t)stream;
  if (n_rows > 0) {
    const BwdArgs a{dy, x, dx, gamma, mean, rstd, sums ? ws : nullptr, n_rows, ld_dy, ldx, ld_dx, (n_rows + parts - 1) / parts, D, parts};
    const int rc = by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (sums) {   // (first: dx may lie where dy or x does)
        hipLaunchKernelGGL(ln_part_kernel<T>, dim3((D + NT - 1) / NT, parts), dim3(NT), 0, st, a);
        const int r = check_launch(who);
        if (r) return r;
      }
      if (dx) {
        hipLaunchKernelGGL(ln_bwd_long_kernel<T>, dim3((unsigned)std::min<int64_t>(n_rows, 1 << 20)), dim3(NT), 0, st, a);
        return check_launch(who);
      }
      return (int)EMX_OK;
    });
    if (rc) return rc;
  }
  if (!sums) return EMX_OK;
  hipLaunchKernelGGL(ln_sum_kernel, dim3((unsigned)((2l * D + NT - 1) / NT)), dim3(NT), 0, st, ws, parts, D, dgamma, dbeta);
  return check_launch(who);
}

}  // extern "C"
