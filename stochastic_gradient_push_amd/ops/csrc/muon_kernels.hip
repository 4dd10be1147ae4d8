// Orthogonalised updates for gfx950 (CDNA4): Newton-Schulz products, alone
// and as the optimiser step around them over a flat parameter buffer.
//
//   X = G / (|G|_F + eps)                      [n, m], n <= m
//   A = X X^T,  B = a I + b A + c A^2,  X = B X      (`steps` times)
//
// All products run on the matrix cores, as row-by-row products C = P Q^T of
// two operands whose rows lie along K: A = X X^T, A^2 = A A^T, and B X from
// the transpose of X, which every step stores beside X.  A and A^2 are
// symmetric: only tiles on and above the diagonal are computed, and each
// is stored twice.
//
// Precision.  A small singular value grows by the factor a in every step,
// a^5 = 485 in all with the usual coefficients, and the rounding of X, A
// and B grows with it.  Values are therefore held as two fp16 numbers,
// v = hi + lo (22 bits), and a product is hi hi + hi lo + lo hi, three
// matrix instructions with fp32 accumulation.  Where the result is 16 bits
// wide anyway the last steps, whose roundings cannot grow any more, keep hi
// alone; the host says from which step on.
//
// Scales.  fp16 has a narrow range, so X is stored times 2^e, with e from
// n m such that its entries are around 1, A times 2^11, B times 2^10; powers
// of two cost no bits.  X is kept with norm 1 rather than |G| / (|G| + eps)
// = r, which enters A as r^2 and the result as r, and 2^e follows what a
// small r lets X grow to: a gradient far below eps loses no bits.
//
// n and m are padded with zeros to whole tiles, so the products have no
// borders; zeros stay zeros in every step.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace {

typedef _Float16 half_t;
typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef half_t half4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float A_SCALE = 2048.f;
constexpr float B_SCALE = 1024.f;

// One matrix.  `start`: its first value in the source, rows * cols values
// in row order; n, m: the smaller and the larger side; np, mp: padded;
// x_off, a_off: its place in the planes of X and of A; chunk0, chunk1: its
// partial sums; e: log2 of X's scale; scale: of its update.
struct Mat {
  int64_t start, x_off, a_off;
  int rows, cols, n, m, np, mp, chunk0, chunk1;
  int e;
  float scale;
};
static_assert(sizeof(Mat) == 64, "the host packs 64 bytes");

struct Tile { int mat, tm, tn, pad; };

// Equal matrices one after another: everything from the block's number.
struct Uniform {
  Mat first;
  int batch;
  __device__ Mat mat(int i) const {
    Mat q = first;
    q.start += (int64_t)i * q.rows * q.cols;
    q.x_off += (int64_t)i * q.np * q.mp;
    q.a_off += (int64_t)i * q.np * q.np;
    const int chunks = q.chunk1;
    q.chunk0 = i * chunks;
    q.chunk1 = q.chunk0 + chunks;
    return q;
  }
  // tile `id` of nt x mt tiles in each matrix
  __device__ Tile grid_tile(int64_t id, int nt, int mt) const {
    const int64_t per = (int64_t)nt * mt;
    const int i = (int)(id / per), t = (int)(id % per);
    return {i, t / mt, t % mt, 0};
  }
  // tile `id` of the nt (nt + 1) / 2 on and above the diagonal
  __device__ Tile sym_tile(int64_t id, int nt) const {
    const int64_t per = (int64_t)nt * (nt + 1) / 2;
    const int i = (int)(id / per), t = (int)(id % per);
    int tn = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((tn + 1) * (tn + 2) / 2 <= t) ++tn;
    while (tn * (tn + 1) / 2 > t) --tn;
    return {i, t - tn * (tn + 1) / 2, tn, 0};
  }
  __device__ Tile sym(int64_t id, int T) const {
    return sym_tile(id, first.np / T);
  }
  __device__ Tile rect(int64_t id, int T) const {
    return grid_tile(id, first.np / T, first.mp / T);
  }
  __device__ Tile pack(int64_t id) const { return rect(id, 64); }
  __device__ int chunk_mat(int64_t id) const {
    return (int)(id / first.chunk1);
  }
};

// Matrices of any shapes: tables that the host has laid out.
struct Table {
  const Mat* mats;
  const Tile* syms;
  const Tile* rects;
  const Tile* packs;
  __device__ Mat mat(int i) const { return mats[i]; }
  __device__ Tile sym(int64_t id, int) const { return syms[id]; }
  __device__ Tile rect(int64_t id, int) const { return rects[id]; }
  __device__ Tile pack(int64_t id) const { return packs[id]; }
};

// Sum over a block of 256 threads, the same in each; `lds` has 4 doubles.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// ------------------------------------------------------- squared norms
// In 64 bits: squares of fp32 values leave its range, sums do not round.
constexpr int CHUNK = 8192;

template <typename T>
__global__ __launch_bounds__(256) void k_ns_sumsq(
    Uniform src, const T* __restrict__ g, double* __restrict__ partials) {
  __shared__ double lds[4];
  const int i = src.chunk_mat(blockIdx.x);
  const Mat q = src.mat(i);
  const int64_t total = (int64_t)q.rows * q.cols;
  const int64_t from = (int64_t)(blockIdx.x - q.chunk0) * CHUNK;
  const int64_t to = from + CHUNK < total ? from + CHUNK : total;
  double s = 0.0;
  for (int64_t k = from + threadIdx.x; k < to; k += 256) {
    const double v = (double)(float)g[q.start + k];
    s += v * v;
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Momentum over a flat buffer: buf = mu buf + g, and u = g + mu buf with
// Nesterov's momentum, u = buf without.  A chunk of a matrix (mat >= 0)
// leaves the sum of u^2; outside the matrices the update is applied at
// once, with weight decay in the gradient.
struct Chunk { int64_t start; int count, mat; };

template <typename T>
__global__ __launch_bounds__(256) void k_muon_momentum(
    const Chunk* __restrict__ chunks, float* __restrict__ p,
    const T* __restrict__ g, float* __restrict__ buf,
    __bf16* __restrict__ shadow, const float* __restrict__ lr_ptr, float mu,
    float wd, float rest_lr, bool nesterov, double* __restrict__ partials) {
  __shared__ double lds[4];
  const Chunk c = chunks[blockIdx.x];
  const float lr = lr_ptr[0] * rest_lr;
  double s = 0.0;
  for (int k = threadIdx.x; k < c.count; k += 256) {
    const int64_t i = c.start + k;
    float gv = (float)g[i];
    if (c.mat < 0) gv += wd * p[i];
    const float b = mu * buf[i] + gv;
    buf[i] = b;
    const float u = nesterov ? gv + mu * b : b;
    if (c.mat < 0) {
      const float v = p[i] - lr * u;
      p[i] = v;
      if (shadow != nullptr) shadow[i] = (__bf16)v;
    } else {
      s += (double)u * u;
    }
  }
  if (c.mat < 0) return;
  s = block_sum(s, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// ---------------------------------------------------------------- packing
__device__ __forceinline__ half_t hi_of(float v) { return (half_t)v; }
__device__ __forceinline__ half_t lo_of(float v, half_t hi) {
  return (half_t)(v - (float)hi);
}

// What the matrices are read from.
template <typename T>
struct Plain {
  const T* g;
  __device__ float at(int64_t i) const { return (float)g[i]; }
};
template <typename T>
struct Momentum {
  const T* g;
  const float* buf;
  float mu;
  bool nesterov;
  __device__ float at(int64_t i) const {
    return nesterov ? (float)g[i] + mu * buf[i] : buf[i];
  }
};

struct Planes { half_t *h, *l; };  // l may be null: hi alone

__device__ __forceinline__ void put(const Planes& p, int64_t i, float v) {
  const half_t h = hi_of(v);
  p.h[i] = h;
  if (p.l != nullptr) p.l[i] = lo_of(v, h);
}

// X and its transpose, 64 x 64 values a block; r[mat] = |G| / (|G| + eps).
template <class Src, class In>
__global__ __launch_bounds__(256) void k_ns_pack(
    Src src, In in, const double* __restrict__ partials, Planes x, Planes xt,
    float* __restrict__ r_out, float eps) {
  __shared__ double lds[4];
  __shared__ float tile[64][65];
  const Tile t = src.pack(blockIdx.x);
  const Mat q = src.mat(t.mat);
  double s = 0.0;
  for (int k = q.chunk0 + threadIdx.x; k < q.chunk1; k += 256)
    s += partials[k];
  const double norm = sqrt(block_sum(s, lds));
  // a matrix of zeros stays one
  const double inv = norm == 0.0 ? 0.0 : ldexp(1.0 / norm, q.e);
  if (t.tm == 0 && t.tn == 0 && threadIdx.x == 0)
    r_out[t.mat] = norm == 0.0 ? 0.f : (float)(norm / (norm + (double)eps));
  // tile[i][j] = X[64 tm + i][64 tn + j], read along the source's rows
  const bool tall = q.rows > q.cols;
  const int a0 = (tall ? t.tn : t.tm) * 64, b0 = (tall ? t.tm : t.tn) * 64;
  for (int k = threadIdx.x; k < 4096; k += 256) {
    const int a = k >> 6, b = k & 63;
    float v = 0.f;
    if (a0 + a < q.rows && b0 + b < q.cols)
      v = (float)((double)in.at(q.start + (int64_t)(a0 + a) * q.cols + b0 + b)
                  * inv);
    tile[tall ? b : a][tall ? a : b] = v;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 4096; k += 256) {
    const int a = k >> 6, b = k & 63;
    put(x, q.x_off + (int64_t)(t.tm * 64 + a) * q.mp + t.tn * 64 + b,
        tile[a][b]);
    put(xt, q.x_off + (int64_t)(t.tn * 64 + a) * q.np + t.tm * 64 + b,
        tile[b][a]);
  }
}

// --------------------------------------------------------------- products
enum { GRAM, POLY, APPLY };

struct Coef { float a, b, c, log2_growth; };

// log2 of the scale of X after `step` steps.  X of norm 1 has singular
// values of at most min(growth^step, 2 / r): the host has found the most
// that a step multiplies one with, and checked that those of r X stay below
// 2.  4 and less have room above 2^13.
__device__ __forceinline__ int x_exp(const Mat& q, float r, int step,
                                     const Coef& k) {
  const float grown = fminf((float)step * k.log2_growth, 1.f - log2f(r));
  const int shift = (int)ceilf(grown) - 2;
  return shift > 0 ? q.e - shift : q.e;
}

// Where the last product goes: a tensor, or the parameters.
template <typename T>
struct ToTensor {
  T* out;
  __device__ void put(int64_t i, float o, const Mat&) const {
    out[i] = (T)o;
  }
};
struct ToParams {
  float* p;
  __bf16* shadow;
  const float* lr_ptr;
  float wd;
  __device__ void put(int64_t i, float o, const Mat& q) const {
    const float lr = lr_ptr[0];
    const float v = p[i] * (1.f - lr * wd) - lr * q.scale * o;
    p[i] = v;
    if (shadow != nullptr) shadow[i] = (__bf16)v;
  }
};
struct ToPlanes {};  // not the last product

// C = P Q^T, one T x T tile a block, 4 waves of T/2 x T/2, K in steps of 32.
template <int T, bool SPLIT, int MODE, class Src, class Out>
__global__ __launch_bounds__(256) void k_ns_gemm(
    Src src, Planes P, Planes Q, Planes C, Planes D, Out out,
    const float* __restrict__ r, Coef k, int step) {
  constexpr int F = T / 32;            // 16 x 16 fragments a wave, a side
  constexpr int S = 40;                // a row in LDS: 32 + 8 of padding
  constexpr int V = T * 4 / 256;       // 16-byte pieces a thread, a plane
  constexpr int NP = SPLIT ? 2 : 1;    // planes
  __shared__ half_t lp[NP][T * S], lq[NP][T * S];
  const Tile t = MODE == APPLY ? src.rect(blockIdx.x, T)
                               : src.sym(blockIdx.x, T);
  const Mat q = src.mat(t.mat);
  const int K = MODE == GRAM ? q.mp : q.np;
  const int64_t p_off = (MODE == GRAM ? q.x_off : q.a_off)
                        + (int64_t)t.tm * T * K;
  const int64_t q_off = (MODE == POLY ? q.a_off : q.x_off)
                        + (int64_t)t.tn * T * K;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * (T / 2), wn = (wave & 1) * (T / 2);

  f32x4 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  for (int k0 = 0; k0 < K; k0 += 32) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int piece = threadIdx.x + v * 256;
      const int row = piece >> 2, c = (piece & 3) * 8;
      const int64_t from = (int64_t)row * K + k0 + c;
      *reinterpret_cast<half8*>(&lp[0][row * S + c]) =
          *reinterpret_cast<const half8*>(P.h + p_off + from);
      *reinterpret_cast<half8*>(&lq[0][row * S + c]) =
          *reinterpret_cast<const half8*>(Q.h + q_off + from);
      if (SPLIT) {
        *reinterpret_cast<half8*>(&lp[NP - 1][row * S + c]) =
            *reinterpret_cast<const half8*>(P.l + p_off + from);
        *reinterpret_cast<half8*>(&lq[NP - 1][row * S + c]) =
            *reinterpret_cast<const half8*>(Q.l + q_off + from);
      }
    }
    __syncthreads();
    half8 a[NP][F], b[NP][F];
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int at = (i * 16 + (lane & 15)) * S + (lane >> 4) * 8;
        a[x][i] = *reinterpret_cast<const half8*>(&lp[x][wm * S + at]);
        b[x][i] = *reinterpret_cast<const half8*>(&lq[x][wn * S + at]);
      }
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            a[0][i], b[0][j], acc[i][j], 0, 0, 0);
        if (SPLIT) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              a[0][i], b[NP - 1][j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              a[NP - 1][i], b[0][j], acc[i][j], 0, 0, 0);
        }
      }
  }

  const float rr = MODE == POLY ? 0.f : r[t.mat];
  const int e = MODE == POLY ? 0 : x_exp(q, rr, step, k);
  // what the sums are multiplied with: powers of two, and r or its square
  float f = 1.f / A_SCALE;
  if (MODE == GRAM) f = ldexpf(rr * rr, -2 * e) * A_SCALE;
  if (MODE == APPLY) {
    if constexpr (__is_same(Out, ToPlanes))
      f = ldexpf(1.f / B_SCALE, x_exp(q, rr, step + 1, k) - e);
    else
      f = ldexpf(rr / B_SCALE, -e);
  }
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = t.tm * T + wm + i * 16 + (lane >> 4) * 4 + x;
        const int col = t.tn * T + wn + j * 16 + (lane & 15);
        float v = acc[i][j][x] * f;
        if (MODE == APPLY) {
          if constexpr (__is_same(Out, ToPlanes)) {
            put(C, q.x_off + (int64_t)row * q.mp + col, v);
            put(D, q.x_off + (int64_t)col * q.np + row, v);
          } else if (row < q.n && col < q.m) {
            const int64_t at = q.rows > q.cols
                ? (int64_t)col * q.cols + row : (int64_t)row * q.cols + col;
            out.put(q.start + at, v, q);
          }
        } else {
          if (MODE == POLY) {
            const int64_t at = q.a_off + (int64_t)row * q.np + col;
            float av = (float)P.h[at];
            if (SPLIT) av += (float)P.l[at];
            v = (k.b * av + k.c * v) * (B_SCALE / A_SCALE)
                + (row == col ? k.a * B_SCALE : 0.f);
          }
          put(C, q.a_off + (int64_t)row * q.np + col, v);
          if (t.tm != t.tn) put(C, q.a_off + (int64_t)col * q.np + row, v);
        }
      }
}

// Workspace, in fp16 values: X and its transpose twice, A and B, each as
// two planes; x_total and a_total: the sizes of one plane.
struct Work {
  Planes x[2], xt[2], a, b;
};

Work split_work(void* base, int64_t x_total, int64_t a_total) {
  half_t* at = static_cast<half_t*>(base);
  Work w;
  auto take = [&](int64_t n) {
    Planes p{at, at + n};
    at += 2 * n;
    return p;
  };
  for (int i = 0; i < 2; ++i) {
    w.x[i] = take(x_total);
    w.xt[i] = take(x_total);
  }
  w.a = take(a_total);
  w.b = take(a_total);
  return w;
}

Planes planes(Planes p, bool lo) { return {p.h, lo ? p.l : nullptr}; }

template <int T, bool SPLIT, class Src, class Out>
void ns_step(Src src, const Work& w, int step, bool next_split, bool last,
             Out out, const float* r, Coef k, int64_t n_sym, int64_t n_rect,
             hipStream_t s) {
  const int now = step & 1;
  const dim3 block(256), sym((unsigned)n_sym), rect((unsigned)n_rect);
  const Planes x = w.x[now], xt = w.xt[now], none{nullptr, nullptr};
  hipLaunchKernelGGL((k_ns_gemm<T, SPLIT, GRAM, Src, ToPlanes>), sym, block,
                     0, s, src, x, x, planes(w.a, SPLIT), none, ToPlanes{},
                     r, k, step);
  hipLaunchKernelGGL((k_ns_gemm<T, SPLIT, POLY, Src, ToPlanes>), sym, block,
                     0, s, src, w.a, w.a, planes(w.b, SPLIT), none,
                     ToPlanes{}, r, k, step);
  if (last)
    hipLaunchKernelGGL((k_ns_gemm<T, SPLIT, APPLY, Src, Out>), rect, block, 0,
                       s, src, w.b, xt, none, none, out, r, k, step);
  else
    hipLaunchKernelGGL((k_ns_gemm<T, SPLIT, APPLY, Src, ToPlanes>), rect,
                       block, 0, s, src, w.b, xt,
                       planes(w.x[now ^ 1], next_split),
                       planes(w.xt[now ^ 1], next_split), ToPlanes{}, r, k,
                       step);
}

template <int T, class Src, class Out>
void ns_steps(Src src, const Work& w, int steps, int split_steps, Out out,
              const float* r, Coef k, int64_t n_sym, int64_t n_rect,
              hipStream_t s) {
  for (int i = 0; i < steps; ++i) {
    auto f = i < split_steps ? ns_step<T, true, Src, Out>
                             : ns_step<T, false, Src, Out>;
    f(src, w, i, i + 1 < split_steps, i + 1 == steps, out, r, k, n_sym,
      n_rect, s);
  }
}

template <typename T>
void newton_schulz(const T* g, T* out, const Mat& first, int batch, int tile,
                   int steps, int split_steps, Coef k, float eps, void* work,
                   double* partials, float* r, hipStream_t s) {
  const Uniform src{first, batch};
  const Work w = split_work(work, (int64_t)batch * first.np * first.mp,
                            (int64_t)batch * first.np * first.np);
  hipLaunchKernelGGL(k_ns_sumsq<T>, dim3((unsigned)(batch * first.chunk1)),
                     dim3(256), 0, s, src, g, partials);
  const int64_t packs = (int64_t)batch * (first.np / 64) * (first.mp / 64);
  hipLaunchKernelGGL((k_ns_pack<Uniform, Plain<T>>), dim3((unsigned)packs),
                     dim3(256), 0, s, src, Plain<T>{g}, partials,
                     planes(w.x[0], split_steps > 0),
                     planes(w.xt[0], split_steps > 0), r, eps);
  const int64_t nt = first.np / tile, mt = first.mp / tile;
  auto f = tile == 64 ? ns_steps<64, Uniform, ToTensor<T>>
                      : ns_steps<128, Uniform, ToTensor<T>>;
  f(src, w, steps, split_steps, ToTensor<T>{out}, r, k,
    batch * (nt * (nt + 1) / 2), batch * nt * mt, s);
}

template <typename T>
void muon_step(float* p, const T* g, float* buf, __bf16* shadow,
               const float* lr, float mu, float wd, float rest_lr,
               bool nesterov, int steps, Coef k, float eps,
               const void* tables, const int64_t* layout, void* work,
               double* partials, float* r, hipStream_t s) {
  // layout: matrices, chunks, pack tiles, sym tiles, rect tiles, size of an
  // X plane, size of an A plane, tile; the tables lie in this order
  const char* at = static_cast<const char*>(tables);
  Table src;
  src.mats = reinterpret_cast<const Mat*>(at);
  at += layout[0] * sizeof(Mat);
  const Chunk* chunks = reinterpret_cast<const Chunk*>(at);
  at += layout[1] * sizeof(Chunk);
  src.packs = reinterpret_cast<const Tile*>(at);
  at += layout[2] * sizeof(Tile);
  src.syms = reinterpret_cast<const Tile*>(at);
  at += layout[3] * sizeof(Tile);
  src.rects = reinterpret_cast<const Tile*>(at);
  if (layout[1] > 0)
    hipLaunchKernelGGL(k_muon_momentum<T>, dim3((unsigned)layout[1]),
                       dim3(256), 0, s, chunks, p, g, buf, shadow, lr, mu, wd,
                       rest_lr, nesterov, partials);
  if (layout[0] == 0) return;
  const Work w = split_work(work, layout[5], layout[6]);
  hipLaunchKernelGGL((k_ns_pack<Table, Momentum<T>>),
                     dim3((unsigned)layout[2]), dim3(256), 0, s, src,
                     Momentum<T>{g, buf, mu, nesterov}, partials, w.x[0],
                     w.xt[0], r, eps);
  auto f = layout[7] == 64 ? ns_steps<64, Table, ToParams>
                           : ns_steps<128, Table, ToParams>;
  f(src, w, steps, steps, ToParams{p, shadow, lr, wd}, r, k, layout[3],
    layout[4], s);
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16 (sgp_muon_step: of the gradients, 0 or 1).
// The host has checked shapes and sizes and laid out the tables.
extern "C" {

int sgp_ns_chunk() { return CHUNK; }

void sgp_newton_schulz(int dtype, const void* g, void* out, const void* mat,
                       int batch, int tile, int steps, int split_steps,
                       float a, float b, float c, float growth, float eps,
                       void* work, double* partials, float* r,
                       hipStream_t s) {
  const Mat& first = *static_cast<const Mat*>(mat);
  const Coef k{a, b, c, log2f(growth)};
  if (dtype == 0)
    newton_schulz(static_cast<const float*>(g), static_cast<float*>(out),
                  first, batch, tile, steps, split_steps, k, eps, work,
                  partials, r, s);
  else if (dtype == 1)
    newton_schulz(static_cast<const __bf16*>(g), static_cast<__bf16*>(out),
                  first, batch, tile, steps, split_steps, k, eps, work,
                  partials, r, s);
  else
    newton_schulz(static_cast<const half_t*>(g), static_cast<half_t*>(out),
                  first, batch, tile, steps, split_steps, k, eps, work,
                  partials, r, s);
}

void sgp_muon_step(int dtype, float* p, const void* g, float* buf,
                   void* shadow, const float* lr, float mu, float wd,
                   float rest_lr, bool nesterov, int steps, float a, float b,
                   float c, float growth, float eps, const void* tables,
                   const int64_t* layout, void* work, double* partials,
                   float* r, hipStream_t s) {
  const Coef k{a, b, c, log2f(growth)};
  __bf16* sh = static_cast<__bf16*>(shadow);
  if (dtype == 0)
    muon_step(p, static_cast<const float*>(g), buf, sh, lr, mu, wd, rest_lr,
              nesterov, steps, k, eps, tables, layout, work, partials, r, s);
  else
    muon_step(p, static_cast<const __bf16*>(g), buf, sh, lr, mu, wd, rest_lr,
              nesterov, steps, k, eps, tables, layout, work, partials, r, s);
}

}  // extern "C"
