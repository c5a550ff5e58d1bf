// Orthogonalised matrix updates (gfx950): the matrices of a flat buffer driven towards their nearest (semi-)orthogonal ones by an odd
// polynomial iteration -- matrix products only -- and the optimizer step that uses them.
//
//   X_0 = G / (|G|_F + eps)    (G transposed where it has more rows than columns, so that X is M x N with M <= N)
//   A = X X^T,  P = b A + c A^2,  X <- a X + P X       `steps` times; (a, b, c) = (3.4445, -4.7750, 2.0315)
// (K. Jordan et al., "Muon: An optimizer for hidden layers in neural networks", 2024.)
//
// A singular value s of X goes to s (a + b s^2 + c s^4): that polynomial maps [0, 1] into [0, 1.2024] and [0, 1.2024] into itself, and
// multiplies the small ones by up to 3.4, so after five steps those above ~1e-2 lie around one.  Hence the bounds every stored value
// obeys, whatever G is: |X| <= 1.21, |A| <= 1.45, |P| <= 2.81.
//
// Arithmetic (of matrices of more than 48 rows; of smaller ones: float32 and 64 bits, ns_low_kernel): as the dense layers', every float32
// product is THREE f16 matrix instructions on operands split into two f16 planes (hi = f16(v), lo = f16(v - hi): 22 bits), accumulated in
// float32.  The bounds above make a scale of 2^14 enough for X, A and P (|P| 2^14 <= 46.1e3 < 65504; what is lost below is 2^-24 2^-14 of the
// matrix' norm).  Where |G|_F is small beside eps, |X_0|_F = |G|_F / (|G|_F + eps) is too, and X is held another 2^q times as large
// (X~ = 2^q X), so that |X~| <= 1/2:  A~ = X~ X~^T = 4^q A,  P~ = b A~ + 4^-q c A~^2 = 4^q P (|P~| <= 1.2), and a X~ + 4^-q P~ X~ = 2^q X_k+1.
// q shrinks from step to step by what |X| may have grown (shift_at).  The norm is summed in 64 bits: an error of its scale is the one that
// the iteration turns into an error of every singular value.  a X joins P X behind its sum, not as a diagonal of P: the sum then rounds at the
// size of P X alone (4096 x 4096: 4.4e-6 off with it inside).
//
// Layout of an operand (X, X^T, A, P): blocks of 32 rows x 32 k; a block is two K-steps of 16, each a hi and a lo PIECE of 1 KB -- what one
// v_mfma_f32_32x32x16_f16 reads: lane l holds row l % 32, k = 8 (l / 32) .. + 7.  The accumulators of such an instruction -- lane l: column
// l % 32, rows 8 q + 4 (l / 32) + r -- are four consecutive k of an operand whose ROWS are the product's columns: a product writes its
// transpose in operand layout straight from registers.  M and N are padded to 32 with zeros, which stay zero.
#include <algorithm>
#include <climits>
#include <cstdint>
#include <new>
#include <type_traits>
#include <vector>

#include "emx_common.h"

namespace {

using namespace emx;

constexpr int NT = 256;
constexpr int MAX_TABLE = 48;                 // matrices of one launch (the table is an argument of the first: 4 KB at most)
constexpr int MAX_PARTS = 1024;               // shares of a matrix' sum of squares
constexpr float CA = 3.4445f, CB = -4.7750f, CC = 2.0315f;
constexpr float SC = 16384.f, RSC = 1.f / 16384.f;
constexpr int BLK = 4096;                     // bytes of an operand's 32 x 32 block

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// the launches whose workgroups are numbered through the matrices
enum { L_NORM = 0, L_SPLIT, L_LOW, L_GRAM, L_JOIN, L_POLY, L_FULL, L_COUNT };

struct Mat {
  long off, ld;        // first element and row stride in the flat tensors
  long ws;             // the matrix' scratch, from the workspace's begin
  int rows, cols;
  float scale;         // of the update
  int begin[L_COUNT];  // each launch's first workgroup (or tile) for this matrix
};
struct StepArgs {
  const void* g;       // gradients: flat buffer, or (slices) the parts of their sum
  void* out;           // orthogonalize: the result's flat buffer
  float *w, *mom;      // optimizer step
  long slice_stride;
  int n_slices, nesterov, steps;
  int low_steps;       // matrices of at most 128 rows: a launch per step, for all of them as one of them is longer than 128 columns
  float beta, keep, lr, eps;    // keep = 1 - lr weight_decay
};
// Everything a call is about.  The first launch gets it as an argument and leaves a copy at the workspace's begin, from which the others read it:
// an argument of this size comes from host memory at microseconds a dependent load, the copy out of the L2.
struct alignas(16) Table {
  StepArgs a;
  int n;
  Mat m[MAX_TABLE];
};
constexpr long TABLE_BYTES = 4096;
static_assert(sizeof(Table) <= 4032 && sizeof(Table) % 16 == 0, "the first launch's arguments");

// The scratch of one matrix: the shares of its sum of squares and its shift, X^T twice (read and written by a step; the second also holds the optimizer step's
// direction u at the begin) and, M > 128: X, A and P; M <= 128: the shares of A twice, 16 blocks from each workgroup.
constexpr int LOW = 4;                        // blocks: matrices of at most 128 rows stay in the LDS of a workgroup (ns_low_kernel)
constexpr int LOW_WGS = 32;                   // ... 128 columns each, or more where there are more than 32 x 128
constexpr int HEAD = MAX_PARTS * 8 + 128;     // bytes in front of the operands
struct Scratch {
  int M, N, Mb, Nb;
  bool turned;
  int* shift;          // q of X_0
  char *t0, *t1, *x, *a, *p, *parts;
  double* part;
  __host__ __device__ Scratch(int rows, int cols, char* base) {
    turned = rows > cols;
    M = turned ? cols : rows, N = turned ? rows : cols;
    Mb = (M + 31) / 32, Nb = (N + 31) / 32;
    const long xn = (long)Mb * Nb * BLK, an = low() ? (long)low_wgs() * 16 * BLK : (long)Mb * Mb * BLK;
    part = reinterpret_cast<double*>(base);
    shift = reinterpret_cast<int*>(base + MAX_PARTS * 8);
    t0 = base + HEAD, t1 = t0 + xn;
    x = t1 + xn;
    a = low() ? x : x + xn;
    p = a + an;
    parts = p + an;
  }
  __host__ __device__ bool low() const { return Mb <= LOW; }
  __host__ __device__ int strips() const { return (Nb + 3) / 4; }     // of 128 columns
  __host__ __device__ int low_wgs() const { return strips() < LOW_WGS ? strips() : LOW_WGS; }
  // A of a matrix four times as long as high and more (and 4096 at least): its sums are cut into four to eight parts, of about the length of the
  // other products.  (Two parts cost more in ns_join_kernel, 9 us, than they save: four 2048 x 512 308 us against 271.)
  __host__ __device__ int gram_parts() const {
    const int n = Nb / (Mb > 32 ? Mb : 32);
    return n < 4 ? 1 : n < 8 ? n : 8;
  }
  __host__ static size_t bytes(int rows, int cols) {
    const Scratch s(rows, cols, nullptr);
    const size_t xn = (size_t)s.Mb * s.Nb;
    const size_t an = (size_t)s.Mb * s.Mb;
    return HEAD + (s.low() ? 2 * xn + 2 * (size_t)s.low_wgs() * 16 : 3 * xn + (2 + (s.gram_parts() > 1 ? s.gram_parts() : 0)) * an) * BLK;
  }
};
// (1024 elements and more to a share: the optimizer step reads up to 32 gradient parts of each)
__host__ __device__ inline int parts_of(long n) { return (int)(n <= 1024l * MAX_PARTS ? (n + 1023) / 1024 : MAX_PARTS); }

// the matrix a workgroup (or tile) belongs to, and its number inside it: all lanes look at once
__device__ __forceinline__ int find(const Mat* m, int n, int launch, int block, int& inside) {
  int at = 0;
  if (n > 1) {
    const int lane = threadIdx.x & 63;
    const bool before = lane < n && m[lane].begin[launch] <= block;
    at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before))) - 1;
  }
  inside = block - m[at].begin[launch];
  return at;
}

// ---- 1: the sum of squares in shares; the optimizer step also forms its update's direction u here.  Four consecutive elements per
// thread at a time where the rows allow it (their length is a multiple of 4), the parts of a gradient eight at a time.  Bound by HBM: 4096 x
// 4096 f32 14.6 us = 4.6 TB/s; the optimizer step's of 21 M weights in one part 50 us, 340 MB read and written = 6.7 TB/s.
template <typename T, bool MUON, int E>
__device__ __forceinline__ double norm_share(const Mat& m, const StepArgs& a, float* u_out, unsigned e0, unsigned e1) {
  typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  typedef float fvec __attribute__((ext_vector_type(E), aligned(4)));
  const unsigned cols = m.cols;
  const bool flat = m.ld == (long)cols;
  double sum = 0.0;
#pragma unroll 2
  for (unsigned e = e0 + E * threadIdx.x; e < e1; e += E * NT) {
    long at = m.off + e;
    if (!flat) {
      const unsigned r = e / cols;
      at = m.off + r * m.ld + (e - r * cols);
    }
    float u[E];
    if constexpr (MUON) {
      const float* g = (const float*)a.g + at;
      fvec mo = *reinterpret_cast<const fvec*>(a.mom + at);
      fvec v = *reinterpret_cast<const fvec*>(g);
      // (pairs of pairs inside the eight: 32 parts one after the other are 9e-8 off, these 6e-8, as a tree over all of them)
      int k = 1;
      if (a.n_slices >= 8) {
        for (k = 0; k + 8 <= a.n_slices; k += 8) {
          fvec p[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) p[q] = k + q ? *reinterpret_cast<const fvec*>(g + (k + q) * a.slice_stride) : v;
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const float eight = ((p[0][i] + p[1][i]) + (p[2][i] + p[3][i])) + ((p[4][i] + p[5][i]) + (p[6][i] + p[7][i]));
            v[i] = k ? v[i] + eight : eight;
          }
        }
      }
      if (k < a.n_slices) {                     // the last seven at most (or all of them)
        fvec r = *reinterpret_cast<const fvec*>(g + k * a.slice_stride);
        for (++k; k < a.n_slices; ++k) {
          const fvec p = *reinterpret_cast<const fvec*>(g + k * a.slice_stride);
#pragma unroll
          for (int i = 0; i < E; ++i) r[i] += p[i];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] += r[i];
      }
      fvec o;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        mo[i] = fmaf(a.beta, mo[i], v[i]);
        o[i] = u[i] = a.nesterov ? fmaf(a.beta, mo[i], v[i]) : mo[i];
      }
      *reinterpret_cast<fvec*>(a.mom + at) = mo;
      *reinterpret_cast<fvec*>(u_out + e) = o;
    } else {
      const vec v = *reinterpret_cast<const vec*>((const T*)a.g + at);
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] = (float)v[i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) sum = fma((double)u[i], (double)u[i], sum);
  }
  return sum;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
template <typename T, bool MUON>
__global__ __launch_bounds__(NT) void ns_norm_kernel(char* ws, const Table tab) {
  __shared__ double sm[NT / 64];
  if (blockIdx.x == 0) {                        // (not read in this launch)
    const int4* const from = reinterpret_cast<const int4*>(&tab);
    for (int i = threadIdx.x; i < (int)(sizeof(Table) / 16); i += NT) reinterpret_cast<int4*>(ws)[i] = from[i];
  }
  int part;
  const StepArgs& a = tab.a;
  const Mat m = tab.m[find(tab.m, tab.n, L_NORM, blockIdx.x, part)];
  const Scratch s(m.rows, m.cols, ws + m.ws);
  const unsigned total = (unsigned)m.rows * m.cols;
  const int parts = parts_of(total);
  const unsigned chunk = ((total + parts - 1) / parts + 3) & ~3u;
  const unsigned e0 = min(part * chunk, total), e1 = min(e0 + chunk, total);
  float* const u_out = reinterpret_cast<float*>(s.t1);
  double sum = m.cols % 4 == 0 ? norm_share<T, MUON, 4>(m, a, u_out, e0, e1) : norm_share<T, MUON, 1>(m, a, u_out, e0, e1);
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) s.part[part] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}
// How X_0 is held: 2^q u / (|u|_F + eps), |X~_0|_F in 1/8 .. 1/2 (q = 0: as it is; 96 at most, |u|_F = 1e-29 eps)
struct Start {
  double inv;          // 1 / (|u|_F + eps)
  int q;
  __device__ __forceinline__ double scale() const { return ldexp(inv, 14 + q); }
};
constexpr int MAX_SHIFT = 96;
// q of X_k: a step multiplies |X| by 3.4445 = 2^1.7843 at most, and 457 / 256 = 1.7852
__device__ __forceinline__ int shift_at(int q0, int k) { return max(q0 - (457 * k + 255) / 256, 0); }
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.f, e); }
// in every thread of a workgroup of N threads
template <int N>
__device__ __forceinline__ Start start_of(const Mat& m, const Scratch& s, float eps, double* sm /* N / 64 */) {
  const int parts = parts_of((long)m.rows * m.cols);
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += N) sum += s.part[i];
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < N / 64; ++i) sum += sm[i];
  const double norm = sqrt(sum), all = norm + (double)eps;
  const auto exponent = [](double v) { return (int)((__double_as_longlong(v) >> 52) & 0x7ff); };   // (of zero: 0)
  return {1.0 / all, min(max(exponent(all) - exponent(norm) - 2, 0), MAX_SHIFT)};
}
// the matrix' shift as an earlier launch has left it: a scalar load, asked for long before its use
__device__ __forceinline__ int shift_of(const Scratch& s) {
  typedef const __attribute__((address_space(4))) int* Uniform;
  return *(Uniform)(uintptr_t)s.shift;
}

// eight values of a row as the hi and lo units of an operand
__device__ __forceinline__ void split_unit(const float (&v)[8], char* hi, char* lo) {
  unsigned x[4], y[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) split_f16_pair(v[2 * p], v[2 * p + 1], x[p], y[p]);
  *reinterpret_cast<uint4v*>(hi) = uint4v{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<uint4v*>(lo) = uint4v{y[0], y[1], y[2], y[3]};
}

// ---- 2: X_0 and its transpose as operands: a workgroup per 64 x 64 of X.  4096 x 4096 f32 35 us for 67 MB read and 134 written = 5.7 TB/s.
template <typename T, bool MUON>
__global__ __launch_bounds__(NT) void ns_split_kernel(char* ws, const int n) {
  __shared__ float tile[64][65];
  __shared__ double sm[NT / 64];
  const Table& tab = *reinterpret_cast<const Table*>(ws);
  const StepArgs& a = tab.a;
  int inside;
  const Mat m = tab.m[find(tab.m, n, L_SPLIT, blockIdx.x, inside)];
  const Scratch s(m.rows, m.cols, ws + m.ws);
  const int tid = threadIdx.x;
  const int tn = (s.Nb + 1) / 2, ti = inside / tn, tj = inside - ti * tn;
  const Start start = start_of<NT>(m, s, a.eps, sm);
  if (inside == 0 && tid == 0) *s.shift = start.q;
  const double f = start.scale();
  const float* const u_in = reinterpret_cast<const float*>(s.t1);
  // the tile as it is stored: rows (r0 ..), columns (c0 ..) of G
  const int r0 = 64 * (s.turned ? tj : ti), c0 = 64 * (s.turned ? ti : tj);
  for (int e = tid; e < 64 * 64; e += NT) {
    const int r = r0 + (e >> 6), c = c0 + (e & 63);
    float v = 0.f;
    if (r < m.rows && c < m.cols) v = MUON ? u_in[(long)r * m.cols + c] : (float)((const T*)a.g)[m.off + r * m.ld + c];
    v = (float)((double)v * f);
    tile[s.turned ? e & 63 : e >> 6][s.turned ? e >> 6 : e & 63] = v;
  }
  __syncthreads();
  // 4 blocks x 2 K-steps x 64 lanes units of X, as many of X^T
  for (int e = tid; e < 1024; e += NT) {
    const int lane = e & 63, ks = (e >> 6) & 1, bj = (e >> 7) & 1, bi = (e >> 8) & 1, tr = e >> 9;
    const int ib = 2 * ti + bi, jb = 2 * tj + bj;
    if (ib >= s.Mb || jb >= s.Nb) continue;
    const int row = lane & 31, k = 16 * ks + 8 * (lane >> 5);
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = tr ? tile[32 * bi + k + q][32 * bj + row] : tile[32 * bi + row][32 * bj + k + q];
    char* base = (tr ? s.t0 + ((long)jb * s.Mb + ib) * BLK : s.x + ((long)ib * s.Nb + jb) * BLK) + ks * 2048 + lane * 16;
    split_unit(v, base, base + 1024);
  }
}

// ---- 3: the products.  KIND 0: A = X X^T; 1: P = a I + b A + c A A^T; 2: X <- P X; 3: the last step's X, written out
enum { GRAM = 0, POLY = 1, NEXT = 2, LAST = 3 };
// A 32 x 32 block of the last X into the caller's tensors (x: row 32 ib + 8 q + 4 h + r, column 32 jb + lr, scaled by 2^28 2^shift): the update of
// w, or the result.  All of a block's reads stand in front of its writes.  A turned matrix has four consecutive elements per lane.
template <typename T, bool MUON>
__device__ __forceinline__ void write_block(const Mat& m, const StepArgs& a, const Scratch& s, f32x16 x, int shift, int ib, int jb, int lr, int h) {
  const float keep = a.keep, f = MUON ? -(a.lr * m.scale) : 1.f, unscale = RSC * RSC * pow2(-shift);
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] *= unscale;
  const int row0 = 32 * ib + 4 * h, col = 32 * jb + lr;
  typedef typename std::conditional<MUON, float, T>::type O;
  O* const base = (MUON ? (O*)a.w : (O*)a.out) + m.off;
  if (s.turned) {
    typedef O quad __attribute__((ext_vector_type(4), aligned(sizeof(O))));
    O* const p = base + (long)col * m.ld + row0;
    if (col >= s.N) return;
    quad old[4];
    if constexpr (MUON) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (row0 + 8 * q + 4 <= s.M) {
          old[q] = *reinterpret_cast<const quad*>(p + 8 * q);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) old[q][r] = row0 + 8 * q + r < s.M ? p[8 * q + r] : (O)0.f;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      quad o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = MUON ? (O)fmaf((float)old[q][r], keep, x[4 * q + r] * f) : (O)(x[4 * q + r] * f);
      if (row0 + 8 * q + 4 <= s.M) {
        *reinterpret_cast<quad*>(p + 8 * q) = o;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row0 + 8 * q + r < s.M) p[8 * q + r] = o[r];
      }
    }
  } else {
    O* const p = base + (long)row0 * m.ld + col;
    O old[16];
    if constexpr (MUON) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = 8 * (e >> 2) + (e & 3);
        if (row0 + d < s.M && col < s.N) old[e] = p[d * m.ld];
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int d = 8 * (e >> 2) + (e & 3);
      if (row0 + d < s.M && col < s.N) p[d * m.ld] = MUON ? (O)fmaf((float)old[e], keep, x[e] * f) : (O)(x[e] * f);
    }
  }
}

// ---- 3: the products, in tiles of 256 x 128 or 128 x 128 (RB = 2, 1): four waves, RB 32 x 128 each.  A wave's operand of RB 32 rows is its own
// and goes from global memory into registers (every piece is what a matrix instruction reads); the operand of 128 columns is shared through LDS.
// Per 32 k a workgroup reads 48 KB for 192 matrix instructions, its LDS traffic is 80 KB: 32 and 52 bytes a clock at their full rate.
constexpr int BT_C = 4;                       // blocks of 32 a tile has: columns; 4 RB rows
// tiles of a product, in the order they are handed out: bands of 4 tile rows, column by column inside a band
constexpr int BAND = 4;
__host__ __device__ inline long band_count(int r0, int tr, int tc, int rb, bool upper) {
  const int h = min(BAND, tr - r0);
  if (!upper) return (long)h * tc;
  const int nc = tc - rb * r0;                // columns from the diagonal on: column rb r0 + d has min(h, d / rb + 1) tiles
  if (nc >= rb * h) return rb * h * (h + 1) / 2 + (long)(nc - rb * h) * h;
  const int k = nc / rb;
  return rb * k * (k + 1) / 2 + (nc % rb) * (k + 1);
}
__host__ __device__ inline long tile_count(int tr, int tc, int rb, bool upper) {
  long n = 0;
  for (int r0 = 0; r0 < tr && (!upper || rb * r0 < tc); r0 += BAND) n += band_count(r0, tr, tc, rb, upper);
  return n;
}
__device__ __forceinline__ void tile_of(int t, int tr, int tc, int rb, bool upper, int& ti, int& tj) {
  int r0 = 0;
  for (;;) {
    const int n = (int)band_count(r0, tr, tc, rb, upper);
    if (t < n || r0 + BAND >= tr) break;
    t -= n, r0 += BAND;
  }
  const int h = min(BAND, tr - r0);
  int c0 = 0;
  if (upper) {
    c0 = rb * r0;
    for (int d = 0; d < rb * h; ++d) {
      const int n = d / rb + 1;
      if (t < n) {
        ti = r0 + t, tj = c0 + d;
        return;
      }
      t -= n;
    }
    c0 += rb * h;
  }
  tj = c0 + t / h, ti = r0 + t % h;
}

// The two planes of a 32 x 32 block as the registers hold it (x: element 4 q + r = row 8 q + 4 h + r of column lr): pairs of rows.
// (x comes out of ordinary vector instructions: split_f16_pair's assembly may not read a matrix instruction's result as it is.)
struct Planes {
  unsigned hi[8], lo[8];
  __device__ __forceinline__ explicit Planes(const f32x16& x) {
#pragma unroll
    for (int p = 0; p < 8; ++p) split_f16_pair(x[2 * p], x[2 * p + 1], hi[p], lo[p]);
  }
};
// A permuted identity that turns a block by two matrix instructions: k-slot (h, e) of K-step ks stands for the block's row
// 16 ks + 4 h + (e < 4 ? e : e + 4), which is where the accumulators of a product have it.
__device__ __forceinline__ void identity(half8 (&one)[2], int lr, int h) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int e = 0; e < 8; ++e) one[ks][e] = (_Float16)(lr == 16 * ks + 4 * h + (e < 4 ? e : e + 4) ? 1.f : 0.f);
}
// a block as an operand: its transpose as it lies in the registers ...
__device__ __forceinline__ void put_direct(char* block, const Planes& x, int lr, int h) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    char* const to = block + (q >> 1) * 2048 + ((q & 1) * 32 + lr) * 16 + h * 8;
    *reinterpret_cast<uint2*>(to) = make_uint2(x.hi[2 * q], x.hi[2 * q + 1]);
    *reinterpret_cast<uint2*>(to + 1024) = make_uint2(x.lo[2 * q], x.lo[2 * q + 1]);
  }
}
// ... and the block itself, turned by matrix instructions (their results are the planes' values: nothing is rounded)
__device__ __forceinline__ void put_turned(char* block, const Planes& x, const half8 (&one)[2], int lr, int h) {
#pragma unroll
  for (int plane = 0; plane < 2; ++plane) {
    const unsigned(&v)[8] = plane ? x.lo : x.hi;
    f32x16 d;
#pragma unroll
    for (int e = 0; e < 16; ++e) d[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      d = __builtin_amdgcn_mfma_f32_32x32x16_f16(
          __builtin_bit_cast(half8, matrix_operand(uint4v{v[4 * ks], v[4 * ks + 1], v[4 * ks + 2], v[4 * ks + 3]})), one[ks], d, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint2*>(block + (q >> 1) * 2048 + ((q & 1) * 32 + lr) * 16 + h * 8 + plane * 1024) =
          make_uint2(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(d[4 * q], d[4 * q + 1])),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(d[4 * q + 2], d[4 * q + 3])));
  }
}

// x += f (hi + lo) for the transpose of an operand's block: where put_direct puts it
__device__ __forceinline__ void add_planes(f32x16& x, const char* block, float f, int lr, int h) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const char* const at = block + (q >> 1) * 2048 + ((q & 1) * 32 + lr) * 16 + h * 8;
    const half4 hi = *reinterpret_cast<const half4*>(at), lo = *reinterpret_cast<const half4*>(at + 1024);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[4 * q + r] = fmaf(f, (float)hi[r] + (float)lo[r], x[4 * q + r]);
  }
}

// x 4^-shift; the same shift in all lanes, and most matrices' is zero
__device__ __forceinline__ void shift_down(f32x16& x, int shift) {
  if (shift == 0) return;
  const float f = pow2(-2 * shift);
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] *= f;
}

__device__ __forceinline__ float4* part_of(const Scratch& s, int part, int ib, int jb, int q, int lane) {
  return reinterpret_cast<float4*>(s.parts + (((long)part * s.Mb + ib) * s.Mb + jb) * BLK + q * 1024 + lane * 16);
}

// A block of a product where it belongs (x: element 4 q + r = row 32 ib + 8 q + 4 h + r of column 32 jb + lr, scaled by 2^28)
template <int KIND, typename T, bool MUON>
__device__ __forceinline__ void store_block(const Mat& m, const StepArgs& a, const Scratch& s, f32x16 x, int ib, int jb, int part /* of the sum; -1: all of it */,
                                            const char* t_in, char* t_out, int k /* the step */, int q0, int lr, int h) {
  if (ib >= s.Mb || jb >= (KIND <= POLY ? s.Mb : s.Nb) || (KIND <= POLY && ib > jb)) return;   // (A and P: the upper half, stored twice)
  if constexpr (KIND == GRAM) {
    if (part >= 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) *part_of(s, part, ib, jb, q, 32 * h + lr) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
      return;
    }
  }
  const int shift = shift_at(q0, k);
  if constexpr (KIND != GRAM) shift_down(x, shift);
  if constexpr (KIND >= NEXT) add_planes(x, t_in + ((long)jb * s.Mb + ib) * BLK, CA * SC, lr, h);
  if constexpr (KIND == LAST) {
    write_block<T, MUON>(m, a, s, x, shift, ib, jb, lr, h);
  } else {
    half8 one[2];
    identity(one, lr, h);
    char* const O = KIND == GRAM ? s.a : KIND == POLY ? s.p : t_out;
    const float f = KIND == NEXT ? RSC * pow2(shift_at(q0, k + 1) - shift) : RSC;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= f;
    if constexpr (KIND == POLY) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= CC;
      add_planes(x, s.a + ((long)jb * s.Mb + ib) * BLK, CB, lr, h);    // A is symmetric: its transpose
    }
    const Planes y(x);
    put_direct(O + ((long)jb * s.Mb + ib) * BLK, y, lr, h);
    if (KIND == NEXT) put_turned(s.x + ((long)ib * s.Nb + jb) * BLK, y, one, lr, h);
    else if (ib != jb) put_turned(O + ((long)ib * s.Mb + jb) * BLK, y, one, lr, h);
  }
}

// What tile `at` of a product is: its matrix, its place, and its blocks of k
template <int KIND, int RB>
struct Unit {
  Mat m;
  Scratch s;
  int parts, part, Ks, K0, Kb, ti, tj;   // (Ks: blocks of k in a row of the operands)
  __device__ __forceinline__ Unit(char* ws, int n, int at) : s(1, 1, nullptr) {
    const Table& tab = *reinterpret_cast<const Table*>(ws);
    int inside;
    m = tab.m[find(tab.m, n, KIND == GRAM ? L_GRAM : KIND == POLY ? L_POLY : L_FULL, at, inside)];
    s = Scratch(m.rows, m.cols, ws + m.ws);
    Ks = KIND == GRAM ? s.Nb : s.Mb;
    parts = KIND == GRAM ? s.gram_parts() : 1, part = inside % parts;
    K0 = part * Ks / parts, Kb = (part + 1) * Ks / parts - K0;
    tile_of(inside / parts, (s.Mb + 4 * RB - 1) / (4 * RB), ((KIND <= POLY ? s.Mb : s.Nb) + BT_C - 1) / BT_C, RB, KIND <= POLY, ti, tj);
  }
};
// The last tiles of a launch, too few to go round the CUs: each cut into `cuts` along k.  Their shares, behind the table in the workspace.
__device__ __forceinline__ float4* cut_of(char* ws, int rb, int unit, int cuts, int cut, int wave, int i, int j, int q, int lane) {
  return reinterpret_cast<float4*>(ws + TABLE_BYTES + ((((long)unit * cuts + cut) * 4 + wave) * rb * BT_C + i * BT_C + j) * BLK + q * 1024 + lane * 16);
}

template <int KIND, typename T, bool MUON, int RB>
__global__ __launch_bounds__(NT, 2) void ns_big_kernel(char* ws, const int n, const int step, const int whole, const int run, const int first_cut,
                                                       const int cuts) {
  __shared__ __align__(16) char lds[2][BT_C * BLK];
  // runs of consecutive tiles to each XCD: they share operands in its L2
  const int turn = (int)(blockIdx.x >> 3);
  int at = ((turn / run) * 8 + (int)(blockIdx.x & 7)) * run + turn % run, cut = -1;
  if ((int)blockIdx.x >= first_cut) {
    const int c = (int)blockIdx.x - first_cut;
    at = whole + c / cuts, cut = c % cuts;
  } else if (at >= whole) {
    return;
  }
  const Unit<KIND, RB> unit(ws, n, at);
  const StepArgs& a = reinterpret_cast<const Table*>(ws)->a;
  const Mat& m = unit.m;
  const Scratch& s = unit.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  char *const t_in = (step & 1) ? s.t1 : s.t0, *const t_out = (step & 1) ? s.t0 : s.t1;
  const int Jb = KIND <= POLY ? s.Mb : s.Nb, Ks = unit.Ks, parts = unit.parts, part = unit.part;
  int K0 = unit.K0, Kb = unit.Kb;                          // this workgroup's blocks of k
  if (cut >= 0) {
    K0 += cut * unit.Kb / cuts;
    Kb = (cut + 1) * unit.Kb / cuts - cut * unit.Kb / cuts;
  }
  const int ib0 = RB * (4 * unit.ti + wave), jb0 = BT_C * unit.tj;   // this wave's first blocks
  const int q0 = KIND == GRAM ? 0 : shift_of(s);
  const char* const Ub = KIND == GRAM ? s.x : KIND == POLY ? s.a : s.p;
  const char* const Vb = KIND == GRAM ? s.x : KIND == POLY ? s.a : t_in;
  // (blocks beyond the matrix are read from its last one and not stored)
  const char* U[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) U[i] = Ub + ((long)min(ib0 + i, s.Mb - 1) * Ks + K0) * BLK + lane * 16;
  const char* V = Vb + ((long)min(jb0 + wave, Jb - 1) * Ks + K0) * BLK + lane * 16;   // this wave's block of the shared operand
  f32x16 acc[RB][BT_C];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < BT_C; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  // The k loop is written in the order it is to run: a GROUP is two blocks of columns of one K-step, 6 RB matrix instructions on 2 RB
  // accumulators; the next group's reads of LDS stand in front of them (the compiler left to itself puts each read right before its use),
  // and no load is conditional (the last ones are repeated), which keeps the counts of loads in flight exact.
  half8 u[2][RB][2], v[4], w[2][2][2];           // [K-step][block][plane]; the shared operand's next block; [group parity][column block][plane]
  auto request_u = [&](const int ks, const long k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      u[ks][i][0] = *reinterpret_cast<const half8*>(U[i] + k * BLK + ks * 2048);
      u[ks][i][1] = *reinterpret_cast<const half8*>(U[i] + k * BLK + ks * 2048 + 1024);
    }
  };
  auto request_v = [&](const long k) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const half8*>(V + k * BLK + q * 1024);
  };
  auto keep_v = [&](const int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<half8*>(lds[buf] + wave * BLK + q * 1024 + lane * 16) = v[q];
  };
  auto read_w = [&](const int buf, const int g) __attribute__((always_inline)) {   // group g: K-step g >> 1, columns 2 (g & 1) ..
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int plane = 0; plane < 2; ++plane)
        w[g & 1][j][plane] = *reinterpret_cast<const half8*>(lds[buf] + (2 * (g & 1) + j) * BLK + (g >> 1) * 2048 + plane * 1024 + lane * 16);
  };
  auto multiply = [&](const int g) __attribute__((always_inline)) {
    const int ks = g >> 1, j0 = 2 * (g & 1);
#pragma unroll
    for (int pass = 0; pass < 3; ++pass)        // small products first
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < RB; ++i)
          acc[i][j0 + j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[ks][i][pass == 1], w[g & 1][j][pass == 0], acc[i][j0 + j], 0, 0, 0);
  };
  request_v(0);
  keep_v(0);
  request_v(min(1, Kb - 1));                    // (in the loop's order: the waits count loads)
  asm volatile("" ::: "memory");
  request_u(0, 0);
  asm volatile("" ::: "memory");
  request_u(1, 0);
  asm volatile("" ::: "memory");
  f32x16 sum[BT_C];
  if constexpr (RB == 1)
#pragma unroll
    for (int j = 0; j < BT_C; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[j][e] = 0.f;
  for (int k = 0; k < Kb; ++k) {
    const int buf = k & 1;
    __syncthreads();                            // the buffer is written, and the other one read to its end
    read_w(buf, 0);
    __builtin_amdgcn_sched_barrier(0);
    read_w(buf, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    keep_v(buf ^ 1);
    request_v(min(k + 2, Kb - 1));
    read_w(buf, 2);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
    request_u(0, min(k + 1, Kb - 1));           // (into the registers just used: on its way during the other K-step)
    read_w(buf, 3);
    __builtin_amdgcn_sched_barrier(0);
    multiply(2);
    __builtin_amdgcn_sched_barrier(0);
    multiply(3);
    __builtin_amdgcn_sched_barrier(0);
    request_u(1, min(k + 1, Kb - 1));
    if constexpr (RB == 1) {                    // sums in two levels, 256 k to the first (with RB = 2 there are no registers for it)
      if ((k & 7) == 7) {
#pragma unroll
        for (int j = 0; j < BT_C; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sum[j][e] += acc[0][j][e];
            acc[0][j][e] = 0.f;
          }
      }
    }
  }
  if constexpr (RB == 1) {
#pragma unroll
    for (int j = 0; j < BT_C; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[0][j][e] += sum[j][e];
  }
  if (cut >= 0) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < BT_C; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *cut_of(ws, RB, at - whole, cuts, cut, wave, i, j, q, lane) =
              make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < BT_C; ++j) store_block<KIND, T, MUON>(m, a, s, acc[i][j], ib0 + i, jb0 + j, parts > 1 ? part : -1, t_in, t_out, step, q0, lr, h);
}

// The tiles that were cut, from their shares in the shares' order: a workgroup per column of blocks
template <int KIND, typename T, bool MUON, int RB>
__global__ __launch_bounds__(NT) void ns_whole_kernel(char* ws, const int n, const int step, const int whole, const int cuts) {
  const int u = (int)blockIdx.x / BT_C, j = (int)blockIdx.x % BT_C;
  const Unit<KIND, RB> unit(ws, n, whole + u);
  const Scratch& s = unit.s;
  const int q0 = KIND == GRAM ? 0 : shift_of(s);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    f32x16 x;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
#pragma unroll 4
    for (int c = 0; c < cuts; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = *cut_of(ws, RB, u, cuts, c, wave, i, j, q, lane);
        x[4 * q] += v.x, x[4 * q + 1] += v.y, x[4 * q + 2] += v.z, x[4 * q + 3] += v.w;
      }
    store_block<KIND, T, MUON>(unit.m, reinterpret_cast<const Table*>(ws)->a, s, x, RB * (4 * unit.ti + wave) + i, BT_C * unit.tj + j,
                               unit.parts > 1 ? unit.part : -1, (step & 1) ? s.t1 : s.t0, (step & 1) ? s.t0 : s.t1, step, q0, lane & 31, lane >> 5);
  }
}

// A of a long matrix from its parts, in their order: a wave per block
__global__ __launch_bounds__(NT) void ns_join_kernel(char* ws, const int n) {
  const Table& tab = *reinterpret_cast<const Table*>(ws);
  int inside;
  const Mat m = tab.m[find(tab.m, n, L_JOIN, blockIdx.x, inside)];
  const Scratch s(m.rows, m.cols, ws + m.ws);
  const int lane = threadIdx.x & 63, block = 4 * inside + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (block >= s.Mb * s.Mb) return;
  const int ib = block / s.Mb, jb = block - ib * s.Mb;
  if (ib > jb) return;
  f32x16 x;
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
  const int parts = s.gram_parts();
#pragma unroll 4
  for (int p = 0; p < parts; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 v = *part_of(s, p, ib, jb, q, lane);
      x[4 * q] += v.x, x[4 * q + 1] += v.y, x[4 * q + 2] += v.z, x[4 * q + 3] += v.w;
    }
  store_block<GRAM, float, false>(m, tab.a, s, x, ib, jb, -1, nullptr, nullptr, 0, 0, lane & 31, lane >> 5);
}

// ---- the products in tiles of 64 x 64, for matrices that would leave most of the machine idle in larger ones: the four waves of a
// workgroup take a quarter of k each, straight from global memory (four K-steps of operands in registers: three travel under the products of
// one), and add up through LDS, a block to each wave.
template <int KIND, typename T, bool MUON>
__global__ __launch_bounds__(NT, 2) void ns_mid_kernel(char* ws, const int n, const int step, const int total, const int run, int, int) {
  __shared__ __align__(16) float4 fold[4][3][4][64];   // [block][wave but its own][q][lane]
  const int turn = (int)(blockIdx.x >> 3), at = ((turn / run) * 8 + (int)(blockIdx.x & 7)) * run + turn % run;
  if (at >= total) return;
  int inside;
  const Table& tab = *reinterpret_cast<const Table*>(ws);
  const StepArgs& a = tab.a;
  const Mat m = tab.m[find(tab.m, n, KIND == GRAM ? L_GRAM : KIND == POLY ? L_POLY : L_FULL, at, inside)];
  const Scratch s(m.rows, m.cols, ws + m.ws);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, h = lane >> 5;
  char *const t_in = (step & 1) ? s.t1 : s.t0, *const t_out = (step & 1) ? s.t0 : s.t1;
  const int Jb = KIND <= POLY ? s.Mb : s.Nb, Ks = KIND == GRAM ? s.Nb : s.Mb;
  const int parts = KIND == GRAM ? s.gram_parts() : 1, part = inside % parts;
  const int K0 = part * Ks / parts, Kb = (part + 1) * Ks / parts - K0;
  inside /= parts;
  int ti, tj;
  tile_of(inside, (s.Mb + 1) / 2, (Jb + 1) / 2, 1, KIND <= POLY, ti, tj);
  const int ib0 = 2 * ti, jb0 = 2 * tj, q0 = KIND == GRAM ? 0 : shift_of(s);
  const char* const Ub = KIND == GRAM ? s.x : KIND == POLY ? s.a : s.p;
  const char* const Vb = KIND == GRAM ? s.x : KIND == POLY ? s.a : t_in;
  // (blocks beyond the matrix are read from its last one and not stored)
  const char *U[2], *V[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    U[i] = Ub + ((long)min(ib0 + i, s.Mb - 1) * Ks + K0) * BLK + lane * 16;
    V[i] = Vb + ((long)min(jb0 + i, Jb - 1) * Ks + K0) * BLK + lane * 16;
  }
  const int k0 = 2 * (wave * Kb / 4), k1 = 2 * ((wave + 1) * Kb / 4);   // this wave's K-steps
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i >> 1][i & 1][e] = 0.f;
  half8 f[4][2][2][2];                          // [K-step % 4][operand][block][plane]
  auto request = [&](const int slot, const int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int plane = 0; plane < 2; ++plane) {
        f[slot][0][i][plane] = *reinterpret_cast<const half8*>(U[i] + k * 2048l + plane * 1024);
        f[slot][1][i][plane] = *reinterpret_cast<const half8*>(V[i] + k * 2048l + plane * 1024);
      }
  };
  const int last = max(k1, 1) - 1;
  request(0, min(k0, last));
  asm volatile("" ::: "memory");
  request(1, min(k0 + 1, last));
  asm volatile("" ::: "memory");
  request(2, min(k0 + 2, last));
  asm volatile("" ::: "memory");
  for (int k = k0; k < k1; k += 4) {
#pragma unroll
    for (int slot = 0; slot < 4; ++slot) {
      request((slot + 3) & 3, min(k + slot + 3, last));
      __builtin_amdgcn_sched_barrier(0);
      if (k + slot < k1) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass)    // small products first
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[slot][0][i][pass == 1], f[slot][1][j][pass == 0], acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // block b of the tile: wave b adds up the four waves' shares, in their order
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (b != wave)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& y = acc[b >> 1][b & 1];
        fold[b][wave - (wave > b)][q][lane] = make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      }
  __syncthreads();
  f32x16 x;
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = wave == 0 ? acc[0][0][e] : wave == 1 ? acc[0][1][e] : wave == 2 ? acc[1][0][e] : acc[1][1][e];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float4 p[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) p[i] = fold[wave][i][q][lane];
    const float4 own = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
    const float4 s0 = wave == 0 ? own : p[0], s1 = wave == 1 ? own : wave == 0 ? p[0] : p[1], s2 = wave == 2 ? own : wave == 3 ? p[2] : p[1],
                 s3 = wave == 3 ? own : p[2];
    x[4 * q] = (s0.x + s1.x) + (s2.x + s3.x);
    x[4 * q + 1] = (s0.y + s1.y) + (s2.y + s3.y);
    x[4 * q + 2] = (s0.z + s1.z) + (s2.z + s3.z);
    x[4 * q + 3] = (s0.w + s1.w) + (s2.w + s3.w);
  }
  store_block<KIND, T, MUON>(m, a, s, x, ib0 + (wave >> 1), jb0 + (wave & 1), parts > 1 ? part : -1, t_in, t_out, step, q0, lr, h);
}

// ---- matrices of at most 128 rows: a workgroup of sixteen waves holds 128 columns of X in registers, a wave one block.  The operands of the
// three products pass through two areas of LDS of 4 x 4 blocks: X, then X^T in the first, A, then P in the second.  Matrices of at
// most 128 columns go through all their steps in one launch.  Longer ones are cut into strips of 128 columns: a launch per step (then for the
// short ones too: their 40 us would stand in front of the others' steps), in which EVERY workgroup adds up the shares of A that the launch before left (in their order), forms P, takes its strip on and leaves its share of
// the next A -- one product of 128^3 and the sum more per workgroup than a division of that work would need, but 2 launches a step fewer.
// A and P are symmetric: the ten waves on and above the diagonal form them, dealt to the SIMDs by (row + column) % 4, three at most to each.
// What bounds it is the LDS (512 KB a product at 128 bytes a clock; 72 matrix instructions a wave and step are 3.8 us) and what stands
// between the barriers.  Two blocks a wave read a quarter less and are slower (two waves per SIMD: 59 us against 49 for five steps of
// 128 x 128 before the symmetry was used, four blocks a wave 88).
constexpr int LOW_NT = 1024;
constexpr int LOW_AREA = 16 * BLK;

__device__ __forceinline__ void clear(f32x16& x) {
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
}
__device__ __forceinline__ void times(f32x16& x, float f) {
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] *= f;
}
// acc += (row block u of one area) (row block v of the other)^T over nk blocks of k; u, v: this lane's 16 bytes of the first block
__device__ __forceinline__ void low_product(f32x16& acc, const char* u, const char* v, int nk) {
  half8 fu[2][2], fv[2][2];   // [K-step parity][plane]
  auto read = [&](const int ks, const int k) __attribute__((always_inline)) {
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      fu[ks][plane] = *reinterpret_cast<const half8*>(u + k * BLK + ks * 2048 + plane * 1024);
      fv[ks][plane] = *reinterpret_cast<const half8*>(v + k * BLK + ks * 2048 + plane * 1024);
    }
  };
  auto multiply = [&](const int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass)        // small products first
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fu[ks][pass == 1], fv[ks][pass == 0], acc, 0, 0, 0);
  };
  read(0, 0);
  for (int k = 0; k < nk; ++k) {
    read(1, k);
    multiply(0);
    read(0, min(k + 1, nk - 1));
    multiply(1);
  }
}

// ---- ... and of at most 16 rows, in 64 bits: A and P have so few entries that the roundings of split operands do not average out (2 x 128: 2e-6 off
// where float32 is off by 8e-7), and so few that plain arithmetic costs less than the launch.  The same strips, steps and shares as above; X travels
// from step to step as float32 rows.
constexpr int THIN = 16;
struct Thin {
  double x[THIN][129];       // (odd pitch: the 16 rows of a column of k lie in different banks)
  double a[THIN][THIN + 1], p[THIN][THIN + 1];
  double shares[LOW_NT];
};
static_assert(sizeof(Thin) <= 2 * LOW_AREA, "the low kernel's LDS");

template <typename T, bool MUON>
__device__ void thin_matrix(Thin& l, double* sm, const Mat& m, const Scratch& s, const StepArgs& a, const int wg, const int step) {
  const int tid = threadIdx.x, M = s.M, wgs = s.low_wgs(), steps = a.steps;
  const int col = tid & 127, row0 = 2 * (tid >> 7);                    // of X: two rows of a column
  const long pitch = 32l * s.Nb;
  int lg = 0;
  while ((1 << lg) < M) ++lg;
  const int entries = 1 << (2 * lg), groups = min(LOW_NT / entries, 16);   // of A; of k
  const int entry = tid & (entries - 1), group = tid >> (2 * lg), ei = entry >> lg, ej = entry & ((1 << lg) - 1);
  const bool mine = tid < entries && ei < M && ej < M;                 // this thread has an entry of A
  auto gram = [&]() {                                                  // of the strip in l.x: the entry's sum, in its thread
    double v = 0.0;
    if (group < groups && ei < M && ej < M)
      for (int k = group; k < 128; k += groups) v = fma(l.x[ei][k], l.x[ej][k], v);
    l.shares[tid] = v;
    __syncthreads();
    v = 0.0;
    if (mine)
      for (int g = 0; g < groups; ++g) v += l.shares[g * entries + entry];
    __syncthreads();
    return v;
  };
  auto poly = [&](double entry_of_a) {                                 // leaves P in l.p
    if (mine) l.a[ei][ej] = entry_of_a;
    __syncthreads();
    if (mine) {
      double v = 0.0;
      for (int k = 0; k < M; ++k) v = fma(l.a[ei][k], l.a[k][ej], v);
      l.p[ei][ej] = fma((double)CC, v, (double)CB * entry_of_a);
    }
    __syncthreads();
  };
  auto next = [&](double (&y)[2]) {                                    // a X + P X, this thread's two
#pragma unroll
    for (int r = 0; r < 2; ++r) y[r] = 0.0;
    if (row0 < M) {
      for (int k = 0; k < M; ++k) {
        const double v = l.x[k][col];
#pragma unroll
        for (int r = 0; r < 2; ++r) y[r] = fma(row0 + r < M ? l.p[row0 + r][k] : 0.0, v, y[r]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (row0 + r < M) y[r] = fma((double)CA, l.x[row0 + r][col], y[r]);
    }
    __syncthreads();
  };
  auto put = [&](const double (&y)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) l.x[row0 + r][col] = y[r];
    __syncthreads();
  };
  auto row_of = [&](char* t, int r, int st) { return reinterpret_cast<float*>(t) + (row0 + r) * pitch + 128 * st + col; };
  auto inside = [&](int r, int st) { return row0 + r < M && 128 * st + col < pitch; };
  auto write = [&](const double (&y)[2], int st) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = row0 + r, j = 128 * st + col;
      if (i < M && j < s.N) {
        const long at = m.off + (s.turned ? j * m.ld + i : i * m.ld + j);
        if constexpr (MUON) a.w[at] = fmaf(a.w[at], a.keep, -(a.lr * m.scale) * (float)y[r]);
        else ((T*)a.out)[at] = (T)(float)y[r];
      }
    }
  };
  double y[2], sum = 0.0;
  if (step == 0) {
    const double f = start_of<LOW_NT>(m, s, a.eps, sm).inv;
    for (int st = wg; st < s.strips(); st += wgs) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = row0 + r, j = 128 * st + col;
        y[r] = 0.0;
        if (i < M && j < s.N) {
          const long gr = s.turned ? j : i, gc = s.turned ? i : j;
          y[r] = f * (double)(MUON ? reinterpret_cast<const float*>(s.t1)[gr * m.cols + gc] : (float)((const T*)a.g)[m.off + gr * m.ld + gc]);
        }
        if (a.low_steps) {
          y[r] = (double)(float)y[r];
          if (inside(r, st)) *row_of(s.t0, r, st) = (float)y[r];
        }
      }
      put(y);
      sum += gram();
    }
    if (a.low_steps) {
      if (mine) reinterpret_cast<double*>(s.a + (long)wg * 16 * BLK)[entry] = sum;
      return;
    }
    for (int k = 0; k < steps; ++k) {
      poly(k == 0 ? sum : gram());
      next(y);
      put(y);
    }
    write(y, 0);
    return;
  }
  char *const shares_in = (step & 1) ? s.a : s.p, *const shares_out = (step & 1) ? s.p : s.a;
  char *const t_in = (step & 1) ? s.t0 : s.t1, *const t_out = (step & 1) ? s.t1 : s.t0;
  if (mine)
    for (int g = 0; g < wgs; ++g) sum += reinterpret_cast<const double*>(shares_in + (long)g * 16 * BLK)[entry];
  poly(sum);
  sum = 0.0;
  for (int st = wg; st < s.strips(); st += wgs) {
#pragma unroll
    for (int r = 0; r < 2; ++r) y[r] = inside(r, st) ? (double)*row_of(t_in, r, st) : 0.0;
    put(y);
    next(y);
    if (step == steps) {
      write(y, st);
      continue;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      y[r] = (double)(float)y[r];
      if (inside(r, st)) *row_of(t_out, r, st) = (float)y[r];
    }
    put(y);
    sum += gram();
  }
  if (step < steps && mine) reinterpret_cast<double*>(shares_out + (long)wg * 16 * BLK)[entry] = sum;
}

// ---- ... and of 17 to 48 rows, on float32 operands: split ones are rounded twice, and in matrices of so few rows whose singular values lie
// close together (gradients that are mostly noise) that made 1.3 times float32's error on average, 2.1 at worst; these make 0.7 times it.
// Five steps of 32 x 128 take 17.4 us (19.9 on split operands), of 48 x 128 24.4 (25.4), of 20 x 9000 73 (79), of 48 x 300 48.7 (42.6), of
// 32000 x 40 217 (197): from 33 rows on the float32 instructions bound it.  64 x 128 35.6 (25.7), and there split operands are as exact as
// float32 again.  Tiles of v_mfma_f32_16x16x4_f32 -- lane l: row l % 16 of either operand, k = l / 16; results: rows 4 (l / 16) + i, column
// l % 16.  A lane takes four consecutive k of a row at a time, one to each of four such instructions: both operands of a product have their k
// in that order.  Wave w holds the blocks (w / 8, w % 8) and (w / 8 + 2, w % 8) of the strip's 3 x 8 in registers.
constexpr int SMALL = 48;
typedef float f32x4 __attribute__((ext_vector_type(4)));
struct Small {
  float x[SMALL][132], a[SMALL][68];   // (a row is four banks behind the one above it: neither rows nor columns of 16 meet)
};
static_assert(sizeof(Small) <= 2 * LOW_AREA, "the low kernel's LDS");

template <typename T, bool MUON>
__device__ void small_matrix(Small& l, double* sm, const Mat& m, const Scratch& s, const StepArgs& a, const int wg, const int step) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, h = lane >> 4, M = s.M, nb = (M + 15) / 16, wgs = s.low_wgs(), steps = a.steps;
  const long pitch = 32l * s.Nb;
  int ib = 0, jb = wave;                                               // this wave's block of the upper half of A and P
  for (; ib < nb && jb >= nb; ++ib) jb -= nb - ib - 1;
  const bool square = ib < nb;
  const int cb = wave & 7, rb = 16 * cb < s.N ? wave >> 3 : nb;        // its blocks of X: rows rb, rb + 2 (none behind the matrix' last column)
  f32x4 y[2];                                                          // ... their values
  auto each = [&](auto take) __attribute__((always_inline)) {          // take(value, row, column of the strip)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (rb + 2 * j < nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = y[j][i];
          take(v, 16 * (rb + 2 * j) + 4 * h + i, 16 * cb + lr);
          y[j][i] = v;
        }
  };
  auto product = [&](const float* u, const float* v, int k16) __attribute__((always_inline)) {   // rows u times rows v, 16 k16 long
    f32x4 even{}, odd{};
    for (int k = 0; k < k16; ++k) {
      const f32x4 fu = *reinterpret_cast<const f32x4*>(u + 16 * k), fv = *reinterpret_cast<const f32x4*>(v + 16 * k);
      even = __builtin_amdgcn_mfma_f32_16x16x4f32(fu[0], fv[0], even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x4f32(fu[1], fv[1], odd, 0, 0, 0);
      even = __builtin_amdgcn_mfma_f32_16x16x4f32(fu[2], fv[2], even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x4f32(fu[3], fv[3], odd, 0, 0, 0);
    }
    return even + odd;
  };
  auto put = [&]() __attribute__((always_inline)) {
    each([&](float& v, int r, int c) { l.x[r][c] = v; });
    __syncthreads();
  };
  auto gram = [&](int st) __attribute__((always_inline)) {             // of the strip in l.x
    f32x4 v{};
    if (square) v = product(&l.x[16 * ib + lr][4 * h], &l.x[16 * jb + lr][4 * h], (min(s.N - 128 * st, 128) + 15) / 16);
    return v;
  };
  auto keep = [&](const f32x4 v) __attribute__((always_inline)) {      // a block of A or P, and its mirror image
    if (square) {
#pragma unroll
      for (int i = 0; i < 4; ++i) l.a[16 * ib + 4 * h + i][16 * jb + lr] = v[i];
      if (ib != jb) *reinterpret_cast<f32x4*>(&l.a[16 * jb + lr][16 * ib + 4 * h]) = v;
    }
    __syncthreads();
  };
  auto poly = [&](f32x4 v) __attribute__((always_inline)) {            // v: A.  Leaves P in l.a
    keep(v);
    f32x4 sq{};
    if (square) sq = product(&l.a[16 * ib + lr][4 * h], &l.a[16 * jb + lr][4 * h], nb);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(CC, sq[i], CB * v[i]);
    __syncthreads();
    keep(v);
  };
  auto next = [&]() __attribute__((always_inline)) {                   // y <- a X + P X
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (rb + 2 * j < nb) {
        f32x4 even{}, odd{};
        for (int k = 0; k < nb; ++k) {
          const f32x4 p = *reinterpret_cast<const f32x4*>(&l.a[16 * (rb + 2 * j) + lr][16 * k + 4 * h]);
          const float* const x = &l.x[16 * k + 4 * h][16 * cb + lr];
          even = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0], x[0], even, 0, 0, 0);
          odd = __builtin_amdgcn_mfma_f32_16x16x4f32(p[1], x[132], odd, 0, 0, 0);
          even = __builtin_amdgcn_mfma_f32_16x16x4f32(p[2], x[264], even, 0, 0, 0);
          odd = __builtin_amdgcn_mfma_f32_16x16x4f32(p[3], x[396], odd, 0, 0, 0);
        }
        y[j] = even + odd;
      }
    each([&](float& v, int r, int c) { v = fmaf(CA, l.x[r][c], v); });
    __syncthreads();
  };
  auto share = [&](char* shares, int g) { return reinterpret_cast<f32x4*>(shares + (long)g * 16 * BLK + (ib * 4 + jb) * 1024 + lane * 16); };
  auto travel = [&](char* t, int st) __attribute__((always_inline)) {  // X from step to step: float32 rows
    each([&](float& v, int r, int c) {
      if (r < M && 128 * st + c < pitch) reinterpret_cast<float*>(t)[r * pitch + 128 * st + c] = v;
    });
  };
  // a strip of the caller's matrix: a lane's four values of a block lie side by side where the matrix is turned
  typedef typename std::conditional<MUON, float, T>::type O;
  typedef O quad __attribute__((ext_vector_type(4), aligned(sizeof(O))));
  auto read = [&](const O* from, long ld, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * (rb + 2 * j) + 4 * h, c = 128 * st + 16 * cb + lr;
      y[j] = f32x4{};
      if (rb + 2 * j >= nb || c >= s.N) continue;
      if (s.turned && r + 4 <= M) {
        const quad v = *reinterpret_cast<const quad*>(from + c * ld + r);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[j][i] = (float)v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i < M) y[j][i] = (float)from[s.turned ? c * ld + r + i : (r + i) * ld + c];
      }
    }
  };
  auto write = [&](int st) __attribute__((always_inline)) {
    O* const to = (MUON ? (O*)a.w : (O*)a.out) + m.off;
    const float f = MUON ? -(a.lr * m.scale) : 1.f, keep = a.keep;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * (rb + 2 * j) + 4 * h, c = 128 * st + 16 * cb + lr;
      if (rb + 2 * j >= nb || c >= s.N) continue;
      if (s.turned && r + 4 <= M) {
        quad* const at = reinterpret_cast<quad*>(to + c * m.ld + r);
        quad o{};
        if constexpr (MUON) o = *at;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = MUON ? (O)fmaf((float)o[i], keep, f * y[j][i]) : (O)y[j][i];
        *at = o;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i < M) {
            O* const at = to + (s.turned ? c * m.ld + r + i : (r + i) * m.ld + c);
            *at = MUON ? (O)fmaf((float)*at, keep, f * y[j][i]) : (O)y[j][i];
          }
      }
    }
  };
  f32x4 sum{};
  if (step == 0) {
    const double f = start_of<LOW_NT>(m, s, a.eps, sm).inv;
    const O* const from = MUON ? reinterpret_cast<const O*>(s.t1) : (const O*)a.g + m.off;
    const long ld = MUON ? m.cols : m.ld;
    read(from, ld, wg);
    for (int st = wg; st < s.strips(); st += wgs) {
      if (st != wg) __syncthreads();                                   // (l.x may still be read for the strip before)
      each([&](float& v, int, int) { v = (float)(f * (double)v); });
      if (a.low_steps) travel(s.t0, st);
      put();
      if (st + wgs < s.strips()) read(from, ld, st + wgs);             // (on its way during the products)
      sum += gram(st);
    }
    if (a.low_steps) {
      if (square) *share(s.a, wg) = sum;
      return;
    }
    for (int k = 0; k < steps; ++k) {                                  // (one strip: y is its values still)
      poly(k == 0 ? sum : gram(0));
      next();
      if (k + 1 < steps) put();
    }
    write(0);
    return;
  }
  char *const shares_in = (step & 1) ? s.a : s.p, *const shares_out = (step & 1) ? s.p : s.a;
  char *const t_in = (step & 1) ? s.t0 : s.t1, *const t_out = (step & 1) ? s.t1 : s.t0;
  auto request = [&](int st) __attribute__((always_inline)) {
    each([&](float& v, int r, int c) { v = r < M && 128 * st + c < pitch ? reinterpret_cast<const float*>(t_in)[r * pitch + 128 * st + c] : 0.f; });
  };
  request(wg);                                                         // (on its way while the shares are added up)
  if (square)
#pragma unroll 8
    for (int g = 0; g < wgs; ++g) sum += *share(shares_in, g);
  poly(sum);
  sum = f32x4{};
  for (int st = wg; st < s.strips(); st += wgs) {
    if (st != wg) __syncthreads();
    put();
    next();
    if (step == steps) {
      write(st);
    } else {
      travel(t_out, st);
      put();
    }
    if (st + wgs < s.strips()) request(st + wgs);
    if (step < steps) sum += gram(st);
  }
  if (step < steps && square) *share(shares_out, wg) = sum;
}

template <typename T, bool MUON>
__global__ __launch_bounds__(LOW_NT) void ns_low_kernel(char* ws, const int n, const int step /* 0: X_0 and its A (or everything) */) {
  extern __shared__ __align__(16) char lds[];
  __shared__ double sm[LOW_NT / 64];
  char *const area1 = lds, *const area2 = lds + LOW_AREA;
  int wg;
  const Table& tab = *reinterpret_cast<const Table*>(ws);
  const StepArgs& a = tab.a;
  const int steps = a.steps;
  const Mat m = tab.m[find(tab.m, n, L_LOW, blockIdx.x, wg)];
  const Scratch s(m.rows, m.cols, ws + m.ws);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, h = lane >> 5, ib = wave >> 2, jb = (wave - ib) & 3;
  const int wgs = s.low_wgs(), Mb = s.Mb;
  if (s.M <= THIN) {
    thin_matrix<T, MUON>(*reinterpret_cast<Thin*>(lds), sm, m, s, a, wg, step);
    return;
  }
  if (s.M <= SMALL) {
    small_matrix<T, MUON>(*reinterpret_cast<Small*>(lds), sm, m, s, a, wg, step);
    return;
  }
  const bool rows = ib < Mb, square = ib <= jb && jb < Mb;   // this wave has a block of X; of the upper half of A and P
  const char *const u1 = area1 + ib * 4 * BLK + lane * 16, *const u2 = area2 + ib * 4 * BLK + lane * 16;
  const char *const v1 = area1 + jb * 4 * BLK + lane * 16, *const v2 = area2 + jb * 4 * BLK + lane * 16;
  half8 one[2];
  identity(one, lr, h);
  f32x16 x, av;

  auto keep_symmetric = [&](char* area, const f32x16& z) __attribute__((always_inline)) {
    const Planes y(z);
    put_direct(area + (jb * 4 + ib) * BLK, y, lr, h);
    if (ib != jb) put_turned(area + (ib * 4 + jb) * BLK, y, one, lr, h);
  };
  auto form_poly = [&](int shift) __attribute__((always_inline)) {   // av: A, area2: A (complete).  Leaves P in area2 (complete)
    const float c = CC * RSC * pow2(-2 * shift);
    f32x16 sq;
    clear(sq);
    if (square) low_product(sq, u2, v2, Mb);
    __syncthreads();
    if (square) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        av[e] = fmaf(c, sq[e], CB * av[e]);
      }
      keep_symmetric(area2, av);
    }
    __syncthreads();
  };
  auto share = [&](const char* shares, int g, int q) __attribute__((always_inline)) {
    return reinterpret_cast<float4*>(const_cast<char*>(shares) + ((long)g * 16 + ib * 4 + jb) * BLK + q * 1024 + lane * 16);
  };
  auto leave_share = [&](char* shares, const f32x16& y) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *share(shares, wg, q) = make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
  };

  if (step == 0) {
    Start start{};
    double f = 0.0;
    f32x16 gram;
    clear(gram);
    for (int st = wg; st < s.strips(); st += wgs) {
      clear(x);
      if (rows) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = 32 * ib + 8 * (e >> 2) + 4 * h + (e & 3), col = 32 * (4 * st + jb) + lr;
          if (row < s.M && col < s.N) {
            const long r = s.turned ? col : row, c = s.turned ? row : col;
            x[e] = MUON ? reinterpret_cast<const float*>(s.t1)[r * m.cols + c] : (float)((const T*)a.g)[m.off + r * m.ld + c];
          }
        }
      }
      if (st == wg) start = start_of<LOW_NT>(m, s, a.eps, sm), f = start.scale();   // (behind the first loads)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (float)((double)x[e] * f);
      if (!a.low_steps) break;                  // (one strip)
      __syncthreads();                          // (area1 may still be read for the strip before)
      if (rows) {
        const Planes y(x);
        if (4 * st + jb < s.Nb) put_direct(s.t0 + ((long)(4 * st + jb) * Mb + ib) * BLK, y, lr, h);
        put_turned(area1 + (ib * 4 + jb) * BLK, y, one, lr, h);
      }
      __syncthreads();
      if (square) low_product(gram, u1, v1, min(4, s.Nb - 4 * st));
    }
    if (a.low_steps) {
      if (square) leave_share(s.a, gram);
      if (wg == 0 && threadIdx.x == 0) *s.shift = start.q;
      return;
    }
    const int q0 = __builtin_amdgcn_readfirstlane(start.q);
    for (int k = 0; k < steps; ++k) {
      const int shift = shift_at(q0, k);
      const Planes y(x);
      if (rows) put_turned(area1 + (ib * 4 + jb) * BLK, y, one, lr, h);
      __syncthreads();
      clear(av);
      if (square) {
        low_product(av, u1, v1, s.Nb);
        times(av, RSC);
        keep_symmetric(area2, av);
      }
      __syncthreads();
      if (rows) put_direct(area1 + (jb * 4 + ib) * BLK, y, lr, h);
      form_poly(shift);
      clear(x);
      if (rows && jb < s.Nb) {
        low_product(x, u2, v1, Mb);
        shift_down(x, shift);
        add_planes(x, area1 + (jb * 4 + ib) * BLK, CA * SC, lr, h);
      }
      if (k + 1 < steps) {
        times(x, RSC * pow2(shift_at(q0, k + 1) - shift));
        __syncthreads();
      }
    }
    if (rows && jb < s.Nb) write_block<T, MUON>(m, a, s, x, shift_at(q0, steps - 1), ib, jb, lr, h);
    return;
  }

  // a step of a longer matrix
  const char *const shares = (step & 1) ? s.a : s.p, *const t_in = (step & 1) ? s.t0 : s.t1;
  char *const shares_out = (step & 1) ? s.p : s.a, *const t_out = (step & 1) ? s.t1 : s.t0;
  half8 t[4];                                   // this wave's block of the strip's X^T on its way to area1: row block ib, k-block jb
  auto request_t = [&](int st) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] = *reinterpret_cast<const half8*>(t_in + ((long)min(4 * st + ib, s.Nb - 1) * Mb + min(jb, Mb - 1)) * BLK + q * 1024 + lane * 16);
  };
  auto keep_t = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<half8*>(area1 + (ib * 4 + jb) * BLK + q * 1024 + lane * 16) = t[q];
  };
  request_t(wg);
  const int q0 = shift_of(s), shift = shift_at(q0, step - 1), shift_out = shift_at(q0, step);
  clear(av);
  if (square) {
#pragma unroll 4
    for (int g = 0; g < wgs; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = *share(shares, g, q);
        av[4 * q] += v.x, av[4 * q + 1] += v.y, av[4 * q + 2] += v.z, av[4 * q + 3] += v.w;
      }
    times(av, RSC);
    keep_symmetric(area2, av);
  }
  keep_t();
  __syncthreads();
  form_poly(shift);
  f32x16 gram;
  clear(gram);
  for (int st = wg; st < s.strips(); st += wgs) {
    if (st != wg) {
      __syncthreads();                          // (area1 may still be read for the strip before)
      request_t(st);
      keep_t();
      __syncthreads();
    }
    clear(x);
    if (rows) {
      low_product(x, u2, v1, Mb);
      shift_down(x, shift);
      add_planes(x, area1 + (jb * 4 + ib) * BLK, CA * SC, lr, h);
    }
    if (step == steps) {
      if (rows && 4 * st + jb < s.Nb) write_block<T, MUON>(m, a, s, x, shift, ib, 4 * st + jb, lr, h);
      continue;
    }
    times(x, RSC * pow2(shift_out - shift));
    __syncthreads();
    if (rows) {
      const Planes y(x);
      if (4 * st + jb < s.Nb) put_direct(t_out + ((long)(4 * st + jb) * Mb + ib) * BLK, y, lr, h);
      put_turned(area1 + (ib * 4 + jb) * BLK, y, one, lr, h);
    }
    __syncthreads();
    if (square) low_product(gram, u1, v1, min(4, s.Nb - 4 * st));
  }
  if (step < steps && square) leave_share(shares_out, gram);
}

// ---- host side
struct Span {
  int64_t a, b, ld;    // first element, behind the last one, row stride (0: one row)
  int cols;
};
int check_matrices(const char* who, const emx_matrix* mats, int n) try {
  EMX_REQUIRE(n >= 0 && (n == 0 || mats), "%s: %d matrices", who, n);
  std::vector<Span> spans;
  for (int i = 0; i < n; ++i) {
    const emx_matrix& m = mats[i];
    EMX_REQUIRE(m.rows >= 0 && m.cols >= 0 && m.offset >= 0 && m.offset <= (int64_t)1 << 50, "%s: matrix %d: %d x %d at %lld", who, i, m.rows, m.cols,
                (long long)m.offset);
    if (m.rows == 0 || m.cols == 0) continue;
    if (m.rows > EMX_MATRIX_MAX_SIDE || m.cols > EMX_MATRIX_MAX_SIDE)
      return fail(EMX_EUNSUPPORTED, "%s: matrix %d: %d x %d (at most %d a side)", who, i, m.rows, m.cols, EMX_MATRIX_MAX_SIDE);
    EMX_REQUIRE(m.rows == 1 || (m.ld >= m.cols && m.ld <= (int64_t)1 << 40), "%s: matrix %d: row stride %lld of %d columns", who, i, (long long)m.ld, m.cols);
    spans.push_back({m.offset, m.offset + (m.rows == 1 ? 0 : (m.rows - 1) * m.ld) + m.cols, m.rows == 1 ? 0 : m.ld, m.cols});
  }
  // every element is updated by ONE matrix: spans apart, or columns side by side in rows of the same length
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  for (size_t i = 0; i < spans.size(); ++i)
    for (size_t j = i + 1; j < spans.size() && spans[j].a < spans[i].b; ++j) {
      const Span &x = spans[i], &y = spans[j];
      const int64_t ld = x.ld ? x.ld : y.ld, shift = ld ? (y.a - x.a) % ld : 0;
      const bool beside = ld && (!x.ld || !y.ld || x.ld == y.ld) && shift >= x.cols && shift + y.cols <= ld;
      EMX_REQUIRE(beside, "%s: matrices at %lld and %lld overlap", who, (long long)x.a, (long long)y.a);
    }
  return EMX_OK;
} catch (const std::bad_alloc&) {
  return fail(EMX_EINVAL, "%s: no host memory for %d matrices", who, n);
}

bool empty(const emx_matrix& m) { return m.rows == 0 || m.cols == 0; }

// the elements from the first matrix' first to the last one's last
void extent(const emx_matrix* mats, int n, int64_t& lo, int64_t& hi) {
  lo = INT64_MAX, hi = 0;
  for (int i = 0; i < n; ++i)
    if (!empty(mats[i])) {
      lo = std::min(lo, mats[i].offset);
      hi = std::max(hi, mats[i].offset + (mats[i].rows == 1 ? 0 : (mats[i].rows - 1) * mats[i].ld) + mats[i].cols);
    }
}
// do elements [lo, hi) of one buffer and [lo, hi + more) of another share memory?
bool share(const void* a, const void* b, int64_t lo, int64_t hi, int64_t more, size_t es) {
  const uintptr_t a0 = (uintptr_t)a + lo * es, a1 = (uintptr_t)a + hi * es, b0 = (uintptr_t)b + lo * es, b1 = (uintptr_t)b + (hi + more) * es;
  return a0 < b1 && b0 < a1;
}

// ... elements [lo, hi) of a buffer and a workspace?
bool covers(const void* ws, size_t bytes, const void* a, int64_t lo, int64_t hi, size_t es) {
  const uintptr_t w0 = (uintptr_t)ws, a0 = (uintptr_t)a + lo * es, a1 = (uintptr_t)a + hi * es;
  return a0 < w0 + bytes && w0 < a1;
}

// hands out the workgroups (or tiles) of a launch
template <typename F>
long number(Table& t, int launch, F blocks) {
  long at = 0;
  for (int i = 0; i < t.n; ++i) {
    t.m[i].begin[launch] = (int)std::min(at, (long)INT_MAX);
    at += blocks(t.m[i], Scratch(t.m[i].rows, t.m[i].cols, nullptr));
  }
  return at;
}

// Which tiles a product runs in.  64 x 64 with k shared out over the waves below 128 tiles of 128 x 128: such a launch is bound by the time from
// one load to the next, not by its products (five steps: 1000 x 1000, 64 tiles, 196 us against 370; two 1024 x 1024, 128 tiles, 356 and
// 376; four, 256 tiles, 501 and 442).  Else 128 x 128, and 256 x 128 -- which reads a quarter less per product -- where these leave at most a
// fifth of the places of their last round empty (two to a CU; 4096 x 4096 in 512 tiles 334 us a product against 371 in 1024; six
// 1000 x 1500 in 288 tiles 82 us against 72 in 576; the upper half of 4096 x 4096 in 272 tiles 283 us against 256 in 528).
template <typename F>
int tile_size(F tiles, int launch) {
  if (tiles(launch, 1) < 128) return 0;
  const long n = tiles(launch, 2), rounds = (n + 511) / 512;
  return 5 * n >= 4 * 512 * rounds ? 2 : 1;
}

// The last tiles of a launch that has a whole round of them for the 256 CUs and at most half a round more: cut along k into as many parts as fill
// the round (16 at most, four blocks of k to each): the upper half of 4096 x 4096, 528 tiles, 255 us -> 193 + 8 in ns_whole_kernel; six 1000 x 1500, 576
// tiles, 72 -> 61 + 6.  Below 1024 k a tile is done in the time that ns_whole_kernel takes.  (Less than a round of tiles -- a CU with one runs at
// 93 % of its rate with two -- cut in two: five steps of six 1000 x 1500 742 -> 839 us.)
constexpr long CUS = 256;
int cuts_of(int size, long count, int blocks_of_k) {
  const long rest = count % CUS;
  if (size == 0 || count < CUS || rest == 0 || blocks_of_k < 32) return 1;
  return (int)std::min({CUS / rest, (long)blocks_of_k / 4, 16l});
}

// The launches of one group of matrices: at most MAX_TABLE of them from index i on.  Returns the index behind them.
struct Plan {
  long norms, splits, lows, joins;                     // workgroups
  int size[L_COUNT], cuts[L_COUNT];                    // of the products: tiles, and what the last of them are cut into
  long count[L_COUNT], whole[L_COUNT];
  bool uneven;
  size_t bytes;                                        // of the workspace
};
int plan_group(const emx_matrix* mats, int n, int i, Table& t, Plan& p) {
  t.n = 0;
  for (; i < n && t.n < MAX_TABLE; ++i)
    if (!empty(mats[i])) t.m[t.n++] = Mat{mats[i].offset, mats[i].rows == 1 ? mats[i].cols : mats[i].ld, 0, mats[i].rows, mats[i].cols, mats[i].scale, {}};
  // the long ones first: a launch ends with short tiles
  const auto length = [](const Mat& m) { return std::max(m.rows, m.cols); };
  std::stable_sort(t.m, t.m + t.n, [&](const Mat& x, const Mat& y) { return length(x) > length(y); });
  p.uneven = t.n > 0 && length(t.m[0]) != length(t.m[t.n - 1]);
  p.norms = number(t, L_NORM, [](const Mat& m, const Scratch&) { return (long)parts_of((long)m.rows * m.cols); });
  p.splits = number(t, L_SPLIT, [](const Mat&, const Scratch& s) { return s.low() ? 0 : (long)((s.Mb + 1) / 2) * ((s.Nb + 1) / 2); });
  p.lows = number(t, L_LOW, [](const Mat&, const Scratch& s) { return s.low() ? (long)s.low_wgs() : 0; });
  p.joins = number(t, L_JOIN, [](const Mat&, const Scratch& s) { return s.low() || s.gram_parts() == 1 ? 0 : ((long)s.Mb * s.Mb + 3) / 4; });
  t.a.low_steps = 0;
  // the tiles of the products, in blocks of 32: 2 x 2 (size 0), 4 x 4 (1), 8 x 4 (2)
  const auto tiles = [&](int launch, int size) {
    return number(t, launch, [&](const Mat&, const Scratch& s) {
      const int r = size == 0 ? 2 : 4 * size, c = size == 0 ? 2 : BT_C;
      const long n = s.low() ? 0 : tile_count((s.Mb + r - 1) / r, ((launch == L_FULL ? s.Nb : s.Mb) + c - 1) / c, size == 2 ? 2 : 1, launch != L_FULL);
      return launch == L_GRAM ? n * s.gram_parts() : n;
    });
  };
  size_t shares = 0;
  for (const int launch : {L_GRAM, L_POLY, L_FULL}) {
    p.size[launch] = tile_size(tiles, launch);
    p.count[launch] = p.whole[launch] = tiles(launch, p.size[launch]);
    int shortest = INT_MAX;
    for (int j = 0; j < t.n; ++j) {
      const Scratch s(t.m[j].rows, t.m[j].cols, nullptr);
      if (!s.low()) shortest = std::min(shortest, launch == L_GRAM ? s.Nb / s.gram_parts() : s.Mb);
    }
    p.cuts[launch] = cuts_of(p.size[launch], p.count[launch], shortest);
    if (p.cuts[launch] > 1) {
      p.whole[launch] = p.count[launch] / CUS * CUS;
      shares = std::max(shares, (size_t)(p.count[launch] % CUS) * p.cuts[launch] * p.size[launch] * 16 * BLK);
    }
  }
  p.bytes = TABLE_BYTES + shares;
  for (int j = 0; j < t.n; ++j) {
    const Scratch s(t.m[j].rows, t.m[j].cols, nullptr);
    if (s.low() && s.strips() > 1) t.a.low_steps = 1;
    t.m[j].ws = (long)p.bytes;
    p.bytes += Scratch::bytes(t.m[j].rows, t.m[j].cols);
  }
  return i;
}

template <typename T, bool MUON>
int run(const char* who, const emx_matrix* mats, int n, const StepArgs& a, char* ws, hipStream_t st) {
  for (int i = 0; i < n;) {
    Table t{};
    Plan p;
    t.a = a;
    i = plan_group(mats, n, i, t, p);
    if (t.n == 0) break;
    for (const long blocks : {p.norms, p.splits, p.lows, p.joins, p.count[L_GRAM], p.count[L_POLY], p.count[L_FULL]})
      EMX_REQUIRE(blocks < (1l << 24), "%s: %ld workgroups", who, blocks);
    hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)p.norms), dim3(NT), 0, st, ws, t);
    int rc = check_launch(who);
    if (rc) return rc;
    if (p.splits) {
      hipLaunchKernelGGL((ns_split_kernel<T, MUON>), dim3((unsigned)p.splits), dim3(NT), 0, st, ws, t.n);
      if ((rc = check_launch(who))) return rc;
    }
    const auto low = [&](int step) {
      if (p.lows == 0) return (int)EMX_OK;
      hipLaunchKernelGGL((ns_low_kernel<T, MUON>), dim3((unsigned)p.lows), dim3(LOW_NT), 2 * LOW_AREA, st, ws, t.n, step);
      return check_launch(who);
    };
    const auto product = [&](auto kind, int launch, int k) {
      constexpr int KIND = decltype(kind)::value;
      const long whole = p.whole[launch], rest = p.count[launch] - whole;
      const int size = p.size[launch], cuts = p.cuts[launch];
      if (whole == 0) return (int)EMX_OK;
      // consecutive tiles to an XCD: an eighth of them all, or -- where their lengths differ -- a few in turn, so that each gets long ones
      const long run = p.uneven ? 8 : (whole + 7) / 8, blocks = (whole + 8 * run - 1) / (8 * run) * 8 * run;
      const auto kernel = size == 0 ? ns_mid_kernel<KIND, T, MUON> : size == 1 ? ns_big_kernel<KIND, T, MUON, 1> : ns_big_kernel<KIND, T, MUON, 2>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks + rest * cuts)), dim3(NT), 0, st, ws, t.n, k, (int)whole, (int)run, (int)blocks, cuts);
      const int rc = check_launch(who);
      if (rc || rest == 0) return rc;
      hipLaunchKernelGGL((size == 1 ? ns_whole_kernel<KIND, T, MUON, 1> : ns_whole_kernel<KIND, T, MUON, 2>), dim3((unsigned)(rest * BT_C)), dim3(NT), 0, st, ws,
                         t.n, k, (int)whole, cuts);
      return check_launch(who);
    };
    if ((rc = low(0))) return rc;
    for (int k = 0; k < a.steps; ++k) {
      if ((rc = product(std::integral_constant<int, GRAM>{}, L_GRAM, k))) return rc;
      if (p.joins) {
        hipLaunchKernelGGL(ns_join_kernel, dim3((unsigned)p.joins), dim3(NT), 0, st, ws, t.n);
        if ((rc = check_launch(who))) return rc;
      }
      if ((rc = product(std::integral_constant<int, POLY>{}, L_POLY, k))) return rc;
      if (k + 1 < a.steps) rc = product(std::integral_constant<int, NEXT>{}, L_FULL, k);
      else rc = product(std::integral_constant<int, LAST>{}, L_FULL, k);
      if (rc || (t.a.low_steps && (rc = low(k + 1)))) return rc;
    }
  }
  return EMX_OK;
}

size_t ws_bytes_of(const emx_matrix* mats, int n) {   // (groups run one after the other, in the same scratch)
  size_t most = 16;
  for (int i = 0; i < n;) {
    Table t;
    Plan p;
    i = plan_group(mats, n, i, t, p);
    if (t.n) most = std::max(most, p.bytes);
  }
  return most;
}

int check_workspace(const char* who, const emx_matrix* mats, int n, const void* ws, size_t ws_bytes, size_t& need) {
  need = ws_bytes_of(mats, n);
  if (!ws || ws_bytes < need || ((uintptr_t)ws & 15))
    return fail(EMX_EWORKSPACE, "%s: workspace of %zu bytes at %p, %zu needed on a 16-byte boundary", who, ws_bytes, ws, need);
  return EMX_OK;
}

}  // namespace

extern "C" {

size_t emx_orthogonalize_ws_bytes(const emx_matrix* mats, int n_mats) {
  return check_matrices("emx_orthogonalize_ws_bytes", mats, n_mats) ? 0 : ws_bytes_of(mats, n_mats);
}

int emx_orthogonalize(const emx_matrix* mats, int n_mats, const void* g, void* out, int dtype, int steps, float eps, void* ws, size_t ws_bytes,
                      emx_stream_t stream) {
  const char* who = "emx_orthogonalize";
  int rc = check_matrices(who, mats, n_mats);
  if (rc) return rc;
  EMX_REQUIRE(dtype == EMX_F32 || dtype == EMX_F16 || dtype == EMX_BF16, "%s: element type %d", who, dtype);
  EMX_REQUIRE(steps >= 1 && steps <= EMX_ORTHOGONALIZE_MAX_STEPS, "%s: %d steps", who, steps);
  EMX_REQUIRE(eps > 0.f && std::isfinite(eps), "%s: eps %g", who, (double)eps);
  if (std::all_of(mats, mats + n_mats, empty)) return EMX_OK;
  const size_t es = dtype == EMX_F32 ? 4 : 2;
  EMX_REQUIRE(g && out && (uintptr_t)g % es == 0 && (uintptr_t)out % es == 0, "%s: g and out are needed, on element boundaries", who);
  int64_t lo, hi;
  extent(mats, n_mats, lo, hi);
  EMX_REQUIRE(g == out || !share(g, out, lo, hi, 0, es), "%s: g and out overlap without being the same buffer", who);
  size_t need;
  if ((rc = check_workspace(who, mats, n_mats, ws, ws_bytes, need))) return rc;
  EMX_REQUIRE(!covers(ws, need, g, lo, hi, es) && !covers(ws, need, out, lo, hi, es), "%s: the workspace lies in the matrices' memory", who);
  StepArgs a{};
  a.g = g, a.out = out, a.n_slices = 1, a.steps = steps, a.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == EMX_F16) return run<_Float16, false>(who, mats, n_mats, a, (char*)ws, st);
  if (dtype == EMX_BF16) return run<__bf16, false>(who, mats, n_mats, a, (char*)ws, st);
  return run<float, false>(who, mats, n_mats, a, (char*)ws, st);
}

int emx_muon_step(const emx_matrix* mats, int n_mats, float* w, const float* g, int n_slices, int64_t slice_stride, float* momentum, float lr,
                  float beta, int nesterov, float weight_decay, int steps, float eps, void* ws, size_t ws_bytes, emx_stream_t stream) {
  const char* who = "emx_muon_step";
  int rc = check_matrices(who, mats, n_mats);
  if (rc) return rc;
  EMX_REQUIRE(n_slices >= 1 && (n_slices == 1 || (slice_stride >= 0 && slice_stride <= ((int64_t)1 << 50) / n_slices)), "%s: %d slices, stride %lld", who, n_slices, (long long)slice_stride);
  EMX_REQUIRE(std::isfinite(lr) && beta >= 0.f && beta < 1.f && std::isfinite(weight_decay), "%s: lr %g, momentum %g, weight decay %g", who,
              (double)lr, (double)beta, (double)weight_decay);
  EMX_REQUIRE(steps >= 1 && steps <= EMX_ORTHOGONALIZE_MAX_STEPS, "%s: %d steps", who, steps);
  EMX_REQUIRE(eps > 0.f && std::isfinite(eps), "%s: eps %g", who, (double)eps);
  for (int i = 0; i < n_mats; ++i) EMX_REQUIRE(std::isfinite(mats[i].scale), "%s: matrix %d: scale %g", who, i, (double)mats[i].scale);
  if (std::all_of(mats, mats + n_mats, empty)) return EMX_OK;
  EMX_REQUIRE(w && g && momentum && ((uintptr_t)w | (uintptr_t)g | (uintptr_t)momentum) % 4 == 0, "%s: w, g and momentum are needed, on element boundaries", who);
  int64_t lo, hi;
  extent(mats, n_mats, lo, hi);
  const int64_t more = n_slices > 1 ? (n_slices - 1) * slice_stride : 0;
  EMX_REQUIRE(!share(w, momentum, lo, hi, 0, 4) && !share(w, g, lo, hi, more, 4) && !share(momentum, g, lo, hi, more, 4),
              "%s: w, g and momentum have to be three buffers", who);
  size_t need;
  if ((rc = check_workspace(who, mats, n_mats, ws, ws_bytes, need))) return rc;
  EMX_REQUIRE(!covers(ws, need, w, lo, hi, 4) && !covers(ws, need, momentum, lo, hi, 4) && !covers(ws, need, g, lo, hi + more, 4),
              "%s: the workspace lies in the matrices' memory", who);
  StepArgs a{};
  a.g = g, a.w = w, a.mom = momentum, a.slice_stride = slice_stride, a.n_slices = n_slices, a.nesterov = nesterov != 0, a.steps = steps;
  a.beta = beta, a.keep = (float)(1.0 - (double)lr * weight_decay), a.lr = lr, a.eps = eps;
  return run<float, true>(who, mats, n_mats, a, (char*)ws, (hipStream_t)stream);
}

}  // extern "C"
