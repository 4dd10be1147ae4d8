// Orthogonalised updates for gfx950 (CDNA4): Newton-Schulz products, alone
// and as the optimiser step around them over a flat parameter buffer.
//
//   X = G / (|G|_F + eps)                      [n, m], n <= m
//   A = X X^T,  B = a I + b A + c A^2,  X = B X      (`steps` times)
//
// Steps in groups.  For wide matrices most of the work is in X X^T and B X,
// while A, B and their products are n x n, symmetric, and commute.  So a
// group of steps computes X X^T once and goes on with A alone,
//
//   B_k = a I + b A_k + c A_k^2,  A_{k+1} = B_k (B_k A_k),
//   P_k = B_k P_{k-1},            X = P X   at the group's end.
//
// Two steps take 3 n^2 m + 5 n^3 operations like this instead of 6 n^2 m +
// 2 n^3 (symmetric results count half).  A's error grows within the group, as
// that of a recomputed A does not: groups are of two steps where the result
// is fp32 itself, of three where it is rounded to 16 bits, or is a step of
// parameters whose own rounding is larger.
//
// All products run on the matrix cores, as row-by-row products C = P Q^T of
// two operands whose rows lie along K: A = X X^T, A^2 = A A^T, and B X from
// the transpose of X, which every step stores beside X.  A and A^2 are
// symmetric: only tiles on and above the diagonal are computed, and each
// is stored twice.
//
// What bounds it.  4096 x 4096: a product of pairs runs at 1100 to 1200
// TFLOP/s of fp16 work, as a large fp16 library product does; the matrix
// pipes are busy 67% of the time at the 1.6 GHz that the power limit leaves.
// Around 1000: the 64 x 64 tiles' loads, 95 GB/s a CU (nothing but loads: 145
// from L2, 90 to 120 from behind it).  That is half of an n x n product's 11
// us; the rest is its start, the sum over four waves and two passes of stores,
// in each of 17 to 19 launches.  Below 500 the launches count, 4 us each.
//
// Precision.  A small singular value grows by the factor a in every step,
// a^5 = 485 in all with the usual coefficients, and the rounding of X, A
// and B grows with it.  Values are therefore held as two fp16 numbers,
// v = hi + lo (22 bits), and a product is hi hi + hi lo + lo hi, three
// matrix instructions with fp32 accumulation: errors are about those of
// products in fp32, mostly below (1000 x 2048 1.5e-6 against 3.4e-6, a step
// over a small network 3.9e-8 against 3.8e-8).  The last steps of
// a bf16 result, whose roundings can hardly grow any more, may keep hi alone:
// only where the caller has asked for it, and the host says from which step
// on.
//
// Scales.  fp16 has a narrow range, so X is stored times 2^e, with e from
// n m such that its entries are around 1, A times 2^11, B times 2^10; powers
// of two cost no bits.  X is kept with norm 1 rather than |G| / (|G| + eps)
// = r, which enters A as r^2 and the result as r, and 2^e follows what a
// small r lets X grow to: a gradient far below eps loses no bits.
//
// n and m are padded with zeros to multiples of 64, so the products have no
// borders; zeros stay zeros in every step.
//
// Layout.  A plane holds 32 columns of all rows, then the next 32; of these
// 16 rows at a time, as one fragment of a matrix instruction: 64 pieces of
// 8 columns, piece l for lane l, 1 KB.  A fragment is loaded from memory or
// LDS with neighbouring lanes at neighbouring places, and what a tile needs
// of its rows for 32 of K is one contiguous piece of memory.

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

// A tile of a product: rows from tm * 64, columns from tn * 64, 64 or 128
// (big) of each.
struct Tile { int mat, tm, tn, big; };

// What a block has to do, in one piece: a record after another would be a
// microsecond each at a kernel's start.
struct Task {
  Mat q;
  Tile t;
};
static_assert(sizeof(Task) == 80, "the host packs 80 bytes");

// Blocks go to the 8 XCDs in turn, each of which has an L2 of its own: the
// `n` numbers are dealt so that an XCD gets neighbours.
__device__ __forceinline__ int by_xcd(int block, int n) {
  const int xcd = block & 7, k = block >> 3, each = n >> 3, more = n & 7;
  return xcd * each + (xcd < more ? xcd : more) + k;
}

// Equal matrices one after another: everything from the block's number.
// The first n_big of a product's 128 x 128 tiles are worked on as such, the
// others as four of 64 x 64, and what an odd number of 64s leaves over too.
struct Uniform {
  Mat first;
  int batch;
  int big_sym, big_rect;
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
  // the pair tm <= tn with number t: 0 0, 0 1, 1 1, 0 2, ...
  __device__ static void triangle(int t, int& tm, int& tn) {
    tn = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((tn + 1) * (tn + 2) / 2 <= t) ++tn;
    while (tn * (tn + 1) / 2 > t) --tn;
    tm = t - tn * (tn + 1) / 2;
  }
  __device__ Tile pair(int id, int per, int mb, bool sym) const {
    Tile t;
    t.mat = id / per;
    const int k = id % per;
    if (sym) {
      triangle(k, t.tm, t.tn);
    } else {
      // down 4 rows before to the right: neighbours share both operands
      const int nb = first.np / 128, top = k / (4 * mb) * 4;
      const int rows = nb - top < 4 ? nb - top : 4, j = k - top * mb;
      t.tm = top + j % rows;
      t.tn = j / rows;
    }
    t.tm *= 2;
    t.tn *= 2;
    t.big = 1;
    return t;
  }
  __device__ Tile tile(int id, bool sym, int n_big) const {
    const int nt = first.np / 64, mt = sym ? nt : first.mp / 64;
    const int nb = nt / 2, mb = mt / 2;
    const int per = sym ? nb * (nb + 1) / 2 : nb * mb;
    if (id < n_big) return pair(by_xcd(id, n_big), per, mb, sym);
    const int fours = per * batch - n_big;
    id = by_xcd(id - n_big, (int)gridDim.x - n_big);
    if (id < 4 * fours) {
      Tile t = pair(n_big + id / 4, per, mb, sym);
      t.tm += (id >> 1) & 1;
      t.tn += id & 1;
      t.big = 0;
      return t;
    }
    id -= 4 * fours;
    // the last column of 64s, then the last row
    const int down = mt & 1 ? nt : 0;
    const int strip = down + (!sym && (nt & 1) ? 2 * mb : 0);
    const int k = id % strip;
    if (k < down) return {id / strip, k, mt - 1, 0};
    return {id / strip, nt - 1, k - down, 0};
  }
  __device__ Task task(Tile t) const { return {mat(t.mat), t}; }
  __device__ Task sym(int id) const { return task(tile(id, true, big_sym)); }
  __device__ Task rect(int id) const {
    return task(tile(id, false, big_rect));
  }
  __device__ Task pack(int id) const {
    const int mt = first.mp / 64, per = first.np / 64 * mt, k = id % per;
    return task({id / per, k / mt, k % mt, 0});
  }
  __device__ int chunk_mat(int id) const { return id / first.chunk1; }
};

// Matrices of any shapes: tables that the host has laid out.
struct Table {
  const Task* syms;
  const Task* rects;
  const Task* packs;
  __device__ Task sym(int id) const { return syms[id]; }
  __device__ Task rect(int id) const { return rects[id]; }
  __device__ Task pack(int id) const { return packs[id]; }
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

// 8 values from any element on, as floats and back.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int x = 0; x < 8; ++x) f[x] = (float)v[x];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = (T)f[x];
  *reinterpret_cast<V*>(p) = v;
}
// the first n of them, 0 behind
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float* f) {
  if (n >= 8) {
    load8(p, f);
  } else {
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = x < n ? (float)p[x] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float* f) {
  if (n >= 8) {
    store8(p, f);
  } else {
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < n) p[x] = (T)f[x];
  }
}

// ------------------------------------------------------- squared norms
// A block has a chunk, 8 values a thread.  Sums are in 64 bits: squares of
// fp32 values leave its range, and the norm's error would be X's.
constexpr int CHUNK = 2048;

template <typename T>
__global__ __launch_bounds__(256) void k_ns_sumsq(
    Uniform src, const T* __restrict__ g, double* __restrict__ partials) {
  __shared__ double lds[4];
  const Mat q = src.mat(src.chunk_mat(blockIdx.x));
  const int64_t at = (int64_t)(blockIdx.x - q.chunk0) * CHUNK
                     + threadIdx.x * 8;
  const int64_t left = (int64_t)q.rows * q.cols - at;
  float v[8];
  load8(g + q.start + at, left < 8 ? (int)left : 8, v);
  double s = 0.0;
#pragma unroll
  for (int x = 0; x < 8; ++x) s += (double)v[x] * v[x];
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
  const int64_t i = c.start + threadIdx.x * 8;
  const int n = c.count - (int)threadIdx.x * 8;
  float gv[8], bv[8], u[8];
  load8(g + i, n, gv);
  load8(buf + i, n, bv);
  if (c.mat >= 0) {
    double s = 0.0;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      bv[x] = mu * bv[x] + gv[x];
      u[x] = nesterov ? gv[x] + mu * bv[x] : bv[x];
      s += (double)u[x] * u[x];
    }
    store8(buf + i, n, bv);
    s = block_sum(s, lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
  } else {
    const float lr = lr_ptr[0] * rest_lr;
    float pv[8];
    load8(p + i, n, pv);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      gv[x] += wd * pv[x];
      bv[x] = mu * bv[x] + gv[x];
      u[x] = nesterov ? gv[x] + mu * bv[x] : bv[x];
      pv[x] -= lr * u[x];
    }
    store8(buf + i, n, bv);
    store8(p + i, n, pv);
    if (shadow != nullptr) store8(shadow + i, n, pv);
  }
}

// ---------------------------------------------------------------- packing
// v = hi + lo.  v has to be settled as an fp32 number first: where it is a
// product, the compiler may round that to fp16 for hi, and elsewhere to fp32
// and then to fp16; if the two differ, lo belongs to the other.
__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
  asm("" : "+v"(v));
  hi = (half_t)v;
  lo = (half_t)(v - (float)hi);
}

// What the matrices are read from: the first n <= 8 values from i on.
template <typename T>
struct Plain {
  const T* g;
  __device__ void read(int64_t i, int n, float* f) const {
    load8(g + i, n, f);
  }
};
template <typename T>
struct Momentum {
  const T* g;
  const float* buf;
  float mu;
  bool nesterov;
  __device__ void read(int64_t i, int n, float* f) const {
    load8(buf + i, n, f);
    if (!nesterov) return;
    float gv[8];
    load8(g + i, n, gv);
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = gv[x] + mu * f[x];
  }
};

struct Planes { half_t *h, *l; };  // l may be null: hi alone

// Where a plane of `rows` rows has (row, col).
__device__ __forceinline__ int64_t place(int row, int col, int rows) {
  return (int64_t)(col >> 5) * rows * 32 + (row >> 4) * 512
         + (col >> 3 & 3) * 128 + (row & 15) * 8 + (col & 7);
}

__device__ __forceinline__ void put8(const Planes& p, int64_t i,
                                     const float* v) {
  half8 h, l;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    half_t hi, lo;
    split(v[x], hi, lo);
    h[x] = hi;
    l[x] = lo;
  }
  *reinterpret_cast<half8*>(p.h + i) = h;
  if (p.l != nullptr) *reinterpret_cast<half8*>(p.l + i) = l;
}

// X and its transpose, 64 x 64 values a block; r[mat] = |G| / (|G| + eps).
template <class Src, class In>
__global__ __launch_bounds__(256) void k_ns_pack(
    Src src, In in, const double* __restrict__ partials, Planes x, Planes xt,
    float* __restrict__ r_out, float eps) {
  __shared__ double lds[4];
  __shared__ float tile[64][65];
  const Task task = src.pack(blockIdx.x);
  const Tile t = task.t;
  const Mat q = task.q;
  const bool tall = q.rows > q.cols;
  const int a0 = (tall ? t.tn : t.tm) * 64, b0 = (tall ? t.tm : t.tn) * 64;
  float v[2][8];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int a = (threadIdx.x >> 3) + y * 32, b = (threadIdx.x & 7) * 8;
    const int n = a0 + a < q.rows ? q.cols - b0 - b : 0;
    in.read(q.start + (int64_t)(a0 + a) * q.cols + b0 + b, n, v[y]);
  }
  double s = 0.0;
  for (int k = q.chunk0 + threadIdx.x; k < q.chunk1; k += 256)
    s += partials[k];
  const double norm = sqrt(block_sum(s, lds));
  // a matrix of zeros stays one
  const double inv = norm == 0.0 ? 0.0 : ldexp(1.0 / norm, q.e);
  if (t.tm == 0 && t.tn == 0 && threadIdx.x == 0)
    r_out[t.mat] = norm == 0.0 ? 0.f : (float)(norm / (norm + (double)eps));
  // tile[i][j] = X[64 tm + i][64 tn + j], read along the source's rows
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int a = (threadIdx.x >> 3) + y * 32, b = (threadIdx.x & 7) * 8;
    const int n = a0 + a < q.rows ? q.cols - b0 - b : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      tile[tall ? b + i : a][tall ? a : b + i] =
          i < n ? (float)((double)v[y][i] * inv) : 0.f;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 512; k += 256) {
    // 16 neighbours have the same 8 columns of 16 rows
    const int a = (k & 15) + (k >> 6 & 3) * 16;
    const int b = (k >> 8) * 32 + (k >> 4 & 3) * 8;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = tile[a][b + i];
    put8(x, q.x_off + place(t.tm * 64 + a, t.tn * 64 + b, q.np), o);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = tile[b + i][a];
    put8(xt, q.x_off + place(t.tn * 64 + a, t.tm * 64 + b, q.mp), o);
  }
}

// --------------------------------------------------------------- products
enum { GRAM, POLY, MUL, APPLY };

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

// What X X^T, of an X that is stored times 2^e, is multiplied with to be A:
// r^2 2^-2e A_SCALE.  r alone may be 1e-38 and its square 0, but r 2^-e is of
// the size that r X has at its largest.
__device__ __forceinline__ float gram_factor(float r, int e) {
  const float h = ldexpf(r, -e);
  return h * h * A_SCALE;
}

__device__ __forceinline__ void load_lds(const half_t* from, half_t* to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)from,
      (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// The operands of a product: planes and first value of P's and Q's rows.
struct Operands {
  const half_t* at[4];  // P hi, Q hi, P lo, Q lo
  int64_t next[2];      // from 32 of K to the next: of P, of Q
  int K;
};

// acc += P Q^T over 32 of K: F x F fragments from rows p_row.. of the P
// planes and q_row.. of the Q planes in LDS, one plane after another.
template <bool SPLIT, int F>
struct Fragments {
  static constexpr int NP = SPLIT ? 2 : 1;
  half8 a[NP][F], b[NP][F];
  // fragment i of plane x, as in Operands, at `row` of that plane in LDS
  __device__ __forceinline__ void read(const half_t* plane, int row, int lane,
                                       int x, int i) {
    (x & 1 ? b : a)[x >> 1][i] =
        *reinterpret_cast<const half8*>(plane + row * 32 + lane * 8);
  }
  // the same from memory
  __device__ __forceinline__ void load(const Operands& o, int kt, int lane,
                                       int x, int i) {
    half8& to = (x & 1 ? b : a)[x >> 1][i];
    to = *reinterpret_cast<const half8*>(
        o.at[x] + kt * o.next[x & 1] + i * 512 + lane * 8);
  }
  // A pair's three products apart: a matrix instruction that adds to the sum
  // of the one before it waits for that.  done(x, i): fragment i of plane x
  // is not needed any more.
  template <class Done>
  __device__ __forceinline__ void multiply(f32x4 (&acc)[F][F],
                                           Done done) const {
    auto mul = [&](int x, int y, int i, int j) {
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[x][i], b[y][j],
                                                         acc[i][j], 0, 0, 0);
    };
    if constexpr (SPLIT) {
#pragma unroll
      for (int i = 0; i < F; ++i) {
#pragma unroll
        for (int j = 0; j < F; ++j) mul(1, 0, i, j);
        done(2, i);
      }
#pragma unroll
      for (int j = 0; j < F; ++j) {
#pragma unroll
        for (int i = 0; i < F; ++i) mul(0, 0, i, j);
        done(1, j);
      }
    }
#pragma unroll
    for (int i = 0; i < F; ++i) {
#pragma unroll
      for (int j = 0; j < F; ++j) mul(0, NP - 1, i, j);
      done(0, i);
    }
#pragma unroll
    for (int j = 0; j < F; ++j) done(2 * NP - 1, j);
  }
  __device__ __forceinline__ void multiply(f32x4 (&acc)[F][F]) const {
    multiply(acc, [](int, int) {});
  }
};

// Everything but the newest N direct loads has arrived, for every wave, and
// every wave is done with what it read before.  The compiler knows of this
// wait, and adds none of its own for what was read before it.
template <int N>
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

constexpr int LDS_BYTES = 65536;  // two blocks on a CU

// 128 x 128, a wave 64 x 64 of it, 32 of K at a time through S buffers.  While
// one step is multiplied from registers, the next is read from LDS and those
// behind it are on their way from memory; reads and loads are issued between
// the products, which they would hold up in one piece (a pair's B X at 4096 x
// 4096, before the power limit slows it: 325 us instead of 341).  Two blocks
// of 64 KB on a CU: one of 128 KB with more buffers is 20% slower (all its
// waves wait at once).
template <bool SPLIT>
__device__ __forceinline__ void product128(const Operands& o, half_t* lds,
                                           f32x4 (&acc)[4][4]) {
  constexpr int NP = SPLIT ? 2 : 1, PLANE = 128 * 32;
  constexpr int S = LDS_BYTES / (2 * NP * PLANE * 2);
  constexpr int L = 4 * NP;  // direct loads of a wave for 32 of K
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto fetch_one = [&](int kt, int buf, int x, int i) {
    load_lds(o.at[x] + kt * o.next[x & 1] + (i * 4 + wave) * 512 + lane * 8,
             lds + (buf * 2 * NP + x) * PLANE + (i * 4 + wave) * 512);
  };
  auto fetch = [&](int kt, int buf) {
#pragma unroll
    for (int x = 0; x < 2 * NP; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) fetch_one(kt, buf, x, i);
  };
  auto read_one = [&](Fragments<SPLIT, 4>& f, int buf, int x, int i) {
    f.read(lds + (buf * 2 * NP + x) * PLANE,
           ((x & 1 ? wave & 1 : wave >> 1) * 4 + i) * 16, lane, x, i);
  };
  auto read = [&](Fragments<SPLIT, 4>& f, int buf) {
#pragma unroll
    for (int x = 0; x < 2 * NP; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) read_one(f, buf, x, i);
  };
  // multiplies f, and between the products reads `next` from its buffer and
  // fetches step kt to the one that f came from
  auto turn = [&](Fragments<SPLIT, 4>& f, Fragments<SPLIT, 4>& next, int from,
                  int kt, int to) {
    int n = 0;
    f.multiply(acc, [&](int, int) {
      if (n < 4 * NP) {
        __builtin_amdgcn_sched_barrier(0);
        read_one(next, from, n >> 1, (2 * n) & 3);
        read_one(next, from, n >> 1, (2 * n + 1) & 3);
        fetch_one(kt, to, n >> 1, n & 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      ++n;
    });
  };
  const int KT = o.K / 32;  // even, like S
#pragma unroll
  for (int kt = 0; kt < S; ++kt)
    if (kt < KT) fetch(kt, kt);
  Fragments<SPLIT, 4> f[2];
  if (KT >= S)
    arrive<(S - 1) * L>();
  else
    arrive<0>();
  read(f[0], 0);
  int buf = 0, kt = 0;  // f[0] has kt, and buf is where it was read from
  auto after = [&](int b) { return b + 1 == S ? 0 : b + 1; };
  for (; kt + S < KT; kt += 2) {
    arrive<(S - 2) * L>();
    const int b1 = after(buf);
    turn(f[0], f[1], b1, kt + S, buf);
    arrive<(S - 2) * L>();
    buf = after(b1);
    turn(f[1], f[0], buf, kt + 1 + S, b1);
  }
  arrive<0>();
  for (; kt < KT; kt += 2) {  // nothing left to fetch
    buf = after(buf);
    read(f[1], buf);
    f[0].multiply(acc);
    if (kt + 2 < KT) {
      buf = after(buf);
      read(f[0], buf);
    }
    f[1].multiply(acc);
  }
}

// 64 x 64, the whole of it by each wave over a part of K.  A fragment is
// 1 KB of contiguous memory, so it comes straight into registers; nothing is
// shared between the waves before the end, and LDS, which would be the
// bottleneck, stays out of it.  The next step's loads are on their way while
// one is multiplied.  The four waves' loads take longer to issue than their
// products, so a fragment is loaded anew as soon as it is not needed any
// more, between the products.  No load depends on a condition inside the
// loop, so that a wait counts exactly what was issued since.
template <bool SPLIT>
__device__ __forceinline__ void product64(const Operands& o,
                                          f32x4 (&acc)[4][4]) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = (o.K / 32 - wave + 3) / 4;  // wave, wave + 4, ...
  Fragments<SPLIT, 4> f[2];
  // in the order of their use
  auto load = [&](Fragments<SPLIT, 4>& to, int step) {
#pragma unroll
    for (int x : {2, 1, 0, 3})
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (SPLIT || x < 2) to.load(o, wave + 4 * step, lane, x, i);
  };
  auto turn = [&](Fragments<SPLIT, 4>& g, int step) {
    g.multiply(acc, [&](int x, int i) {
      __builtin_amdgcn_sched_barrier(0);
      g.load(o, wave + 4 * step, lane, x, i);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  if (steps < 1) return;
  load(f[0], 0);
  if (steps > 1) {
    load(f[1], 1);
    int i = 2;  // the next to load
    for (; i + 1 < steps; i += 2) {
      turn(f[0], i);
      turn(f[1], i + 1);
    }
    f[0].multiply(acc);
    if (i < steps) load(f[0], i);
    f[1].multiply(acc);
    if (i == steps) return;
  }
  f[0].multiply(acc);
}

// Where the last product goes, the first n <= 8 values from i on: a tensor,
// or the parameters.
template <typename T>
struct ToTensor {
  T* out;
  __device__ void put(int64_t i, const float* o, int n, const Mat&) const {
    store8(out + i, n, o);
  }
};
struct ToParams {
  float* p;
  __bf16* shadow;
  const float* lr_ptr;
  float wd;
  __device__ void put(int64_t i, const float* o, int n, const Mat& q) const {
    const float lr = lr_ptr[0], keep = 1.f - lr * wd, step = lr * q.scale;
    float v[8];
    load8(p + i, n, v);
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = v[x] * keep - step * o[x];
    store8(p + i, n, v);
    if (shadow != nullptr) store8(shadow + i, n, v);
  }
};
struct ToPlanes {};  // not the last product

// C = P Q^T for one tile, and what its product makes of it in a group of
// `group` steps that begins with step `step`:
//   GRAM   A = X X^T            stored at its place and mirrored
//   POLY   B = a I + b A + c A^2     likewise
//   MUL    B M, symmetric       likewise; the grid's second row: B M2 to D
//   APPLY  X = B X              stored, and transposed beside it; the last
//                               one goes to `out`
// Rounding, scaling and stores go through a 64-row image of the sums in LDS,
// from which 16 lanes read 8 columns of 16 rows, or 8 rows of 16 columns: with
// an odd stride both ways two lanes meet at most.
template <bool SPLIT, int MODE, class Src, class Out>
__global__ __launch_bounds__(256, 2) void k_ns_gemm(
    Src src, Planes P, Planes Q, Planes Q2, Planes C, Planes D, Out out,
    const float* __restrict__ r, Coef k, int step, int group) {
  if (MODE == MUL && blockIdx.y == 1) {
    Q = Q2;
    C = D;
  }
  __shared__ __attribute__((aligned(16))) char lds_raw[LDS_BYTES];
  half_t* lds = reinterpret_cast<half_t*>(lds_raw);
  float* image = reinterpret_cast<float*>(lds_raw);
  constexpr bool LAST = MODE == APPLY && !__is_same(Out, ToPlanes);
  const Task task = MODE == APPLY ? src.rect(blockIdx.x)
                                  : src.sym(blockIdx.x);
  const Tile t = task.t;
  const Mat q = task.q;
  if (MODE != APPLY && t.tm > t.tn) return;  // below the diagonal
  const int K = MODE == GRAM ? q.mp : q.np;
  const int q_rows = MODE == APPLY ? q.mp : q.np;
  const int64_t p_off = (MODE == GRAM ? q.x_off : q.a_off) + t.tm * 64 * 32;
  const int64_t q_off = (MODE == POLY || MODE == MUL ? q.a_off : q.x_off)
                        + t.tn * 64 * 32;
  const Operands o{{P.h + p_off, Q.h + q_off, SPLIT ? P.l + p_off : nullptr,
                    SPLIT ? Q.l + q_off : nullptr},
                   {(int64_t)q.np * 32, (int64_t)q_rows * 32}, K};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

  const float rr = MODE == GRAM || MODE == APPLY ? r[t.mat] : 0.f;

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (t.big)
    product128<SPLIT>(o, lds, acc);
  else
    product64<SPLIT>(o, acc);

  // what the sums are multiplied with: powers of two, and r or its square
  float f = MODE == MUL ? 1.f / B_SCALE : 1.f / A_SCALE;
  if (MODE == GRAM || MODE == APPLY) {
    const int e = x_exp(q, rr, step, k);
    if (MODE == GRAM)
      f = gram_factor(rr, e);
    else if (LAST)
      f = ldexpf(rr, -e) / B_SCALE;
    else
      f = ldexpf(1.f / B_SCALE, x_exp(q, rr, step + group, k) - e);
  }

  if (!t.big) {
    // the sums of all four waves: each gets a quarter of the rows
    f32x4* all = reinterpret_cast<f32x4*>(lds_raw);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        all[((wave * 4 + i) * 4 + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 v = all[(wave * 4 + j) * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w)
        v += all[((w * 4 + wave) * 4 + j) * 64 + lane];
      acc[0][j] = v;
    }
  }

  const int W = t.big ? 128 : 64, S = W + 1;
  const int row0 = t.tm * 64, col0 = t.tn * 64;
  for (int part = 0; part < W / 64; ++part) {
    // a big tile: the upper, then the lower two waves' sums; a small one:
    // every wave's quarter
    __syncthreads();
    if (!t.big || (wave >> 1) == part) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t.big || i == 0)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              image[((t.big ? i : wave) * 16 + (lane >> 4) * 4 + x) * S
                    + (t.big ? (wave & 1) * 64 : 0) + j * 16 + (lane & 15)] =
                  acc[i][j][x];
    }
    __syncthreads();
    const int rp = row0 + part * 64;  // the image's first row
    const bool mirror = MODE == APPLY ? !LAST : t.tm != t.tn;
    const bool tall = LAST && q.rows > q.cols;
    // along rows: 16 neighbours have the same 8 columns of 16 rows
    if (!tall) {
      for (int u = threadIdx.x; u < 8 * W; u += 256) {
        const int row = (u & 15) + (u >> 6 & 3) * 16;
        const int col = (u >> 8) * 32 + (u >> 4 & 3) * 8;
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = image[row * S + col + x] * f;
        if constexpr (LAST) {
          const int64_t at = q.start + (int64_t)(rp + row) * q.cols;
          if (rp + row < q.n)
            out.put(at + col0 + col, v, q.m - col0 - col, q);
        } else if constexpr (MODE == APPLY) {
          put8(C, q.x_off + place(rp + row, col0 + col, q.np), v);
        } else {
          const int64_t at = q.a_off + place(rp + row, col0 + col, q.np);
          if (MODE == POLY) {
            const half8 h = *reinterpret_cast<const half8*>(P.h + at);
            half8 l = {0, 0, 0, 0, 0, 0, 0, 0};
            if (SPLIT) l = *reinterpret_cast<const half8*>(P.l + at);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              v[x] = (k.b * ((float)h[x] + (float)l[x]) + k.c * v[x])
                     * (B_SCALE / A_SCALE);
              if (rp + row == col0 + col + x) v[x] += k.a * B_SCALE;
              if (mirror) image[row * S + col + x] = v[x];
            }
          }
          put8(C, at, v);
        }
      }
    }
    // along columns likewise: their transposed places
    if (mirror || tall) {
      if (MODE == POLY) __syncthreads();
      for (int u = threadIdx.x; u < 8 * W; u += 256) {
        const int col = (u & 15) + ((u >> 6) * 16 & (W - 1));
        const int row = (u >> (t.big ? 9 : 8)) * 32 + (u >> 4 & 3) * 8;
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x)
          v[x] = image[(row + x) * S + col] * (MODE == POLY ? 1.f : f);
        if constexpr (LAST) {
          const int64_t at = q.start + (int64_t)(col0 + col) * q.cols;
          if (col0 + col < q.m)
            out.put(at + rp + row, v, q.n - rp - row, q);
        } else if constexpr (MODE == APPLY) {
          put8(D, q.x_off + place(col0 + col, rp + row, q.mp), v);
        } else {
          put8(C, q.a_off + place(col0 + col, rp + row, q.np), v);
        }
      }
    }
  }
}

// ---------------------------------------------------------- small matrices
// n <= 64 and m <= 192: one block does all steps of a matrix, with X, its
// transpose, A and B in LDS, where 15 launches would each wait for a few
// microseconds.  The planes are those of the large products, padded to 64
// rows; a wave has 16 rows of every result.
constexpr int SMALL_N = 64, SMALL_M = 192;

// acc[j] += rows [16 wave, 16 wave + 16) of P times rows [16 j, 16 j + 16) of
// the R rows of Q, over K.
template <bool SPLIT, int R, int K>
__device__ __forceinline__ void small_product(const half_t* p, int p_plane,
                                              const half_t* q, int q_plane,
                                              int wave, int lane,
                                              f32x4* acc) {
#pragma unroll
  for (int k0 = 0; k0 < K; k0 += 32) {
    const half_t* pa = p + k0 * SMALL_N + wave * 512 + lane * 8;
    const half_t* qa = q + k0 * R + lane * 8;
    half8 a[2], b[2][R / 16];
#pragma unroll
    for (int x = 0; x < (SPLIT ? 2 : 1); ++x) {
      a[x] = *reinterpret_cast<const half8*>(pa + x * p_plane);
#pragma unroll
      for (int j = 0; j < R / 16; ++j)
        b[x][j] = *reinterpret_cast<const half8*>(qa + x * q_plane + j * 512);
    }
#pragma unroll
    for (int x = 0; x < (SPLIT ? 3 : 1); ++x)
#pragma unroll
      for (int j = 0; j < R / 16; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            a[x == 2], b[x == 1][j], acc[j], 0, 0, 0);
  }
}

// 4 values that lie together, as pairs.
__device__ __forceinline__ void put4(half_t* h, int plane, const float* v) {
  half4 hi, lo;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    half_t a, b;
    split(v[x], a, b);
    hi[x] = a;
    lo[x] = b;
  }
  *reinterpret_cast<half4*>(h) = hi;
  *reinterpret_cast<half4*>(h + plane) = lo;
}

// One step on the planes in LDS; the result in `acc`, not scaled.
template <bool SPLIT, int MP>
__device__ __forceinline__ void small_step(const half_t* x, const half_t* xt,
                                           half_t* a, half_t* b, float gram,
                                           const Coef& k, f32x4* acc) {
  constexpr int XP = SMALL_N * MP, AP = SMALL_N * SMALL_N;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r0 = wave * 16 + (lane >> 4) * 4;  // this lane's 4 rows
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // A and B are symmetric: a lane's 4 rows of a column are stored as 4
  // columns of a row, which lie together
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = zero;
  small_product<SPLIT, SMALL_N, MP>(x, XP, x, XP, wave, lane, acc);
  float av[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) av[j][i] = acc[j][i] * gram;
    put4(a + place(j * 16 + (lane & 15), r0, SMALL_N), AP, av[j]);
    acc[j] = zero;
  }
  __syncthreads();
  small_product<SPLIT, SMALL_N, SMALL_N>(a, AP, a, AP, wave, lane, acc);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = j * 16 + (lane & 15);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (k.b * av[j][i] + k.c * acc[j][i] * (1.f / A_SCALE))
             * (B_SCALE / A_SCALE) + (r0 + i == col ? k.a * B_SCALE : 0.f);
    put4(b + place(col, r0, SMALL_N), AP, v);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < MP / 16; ++j) acc[j] = zero;
  small_product<SPLIT, MP, SMALL_N>(b, AP, xt, XP, wave, lane, acc);
  __syncthreads();
}

template <typename T, int MP>
__global__ __launch_bounds__(256) void k_ns_small(
    Uniform src, const T* __restrict__ g, T* __restrict__ out, int steps,
    int split_steps, Coef k, float eps) {
  constexpr int XP = SMALL_N * MP, AP = SMALL_N * SMALL_N;
  constexpr int V = XP / 2048;  // 8 values at a time a thread
  __shared__ __attribute__((aligned(16))) half_t x[2 * XP], xt[2 * XP],
      a[2 * AP], b[2 * AP];
  const Mat q = src.mat(blockIdx.x);
  const bool tall = q.rows > q.cols;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int total = q.rows * q.cols;

  float v[V][8];
  double s = 0.0;
#pragma unroll
  for (int y = 0; y < V; ++y) {
    const int i = (y * 256 + threadIdx.x) * 8;
    load8(g + q.start + i, total - i, v[y]);
  }
#pragma unroll
  for (int i = threadIdx.x * 8; i < 2 * XP; i += 2048) {
    const half8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    *reinterpret_cast<half8*>(x + i) = zero;
    *reinterpret_cast<half8*>(xt + i) = zero;
  }
#pragma unroll
  for (int y = 0; y < V; ++y)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (double)v[y][i] * v[y][i];
  const double norm = sqrt(block_sum(s, reinterpret_cast<double*>(a)));
  const double inv = norm == 0.0 ? 0.0 : ldexp(1.0 / norm, q.e);
  const float r = norm == 0.0 ? 0.f : (float)(norm / (norm + (double)eps));
#pragma unroll
  for (int y = 0; y < V; ++y) {
    const int first = (y * 256 + threadIdx.x) * 8;
    int row = first / q.cols, col = first % q.cols;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (first + i < total) {
        const float f = (float)((double)v[y][i] * inv);
        half_t h, l;
        split(f, h, l);
        const int xr = tall ? col : row, xc = tall ? row : col;
        const int at = (int)place(xr, xc, SMALL_N), to = (int)place(xc, xr, MP);
        x[at] = h;
        x[at + XP] = l;
        xt[to] = h;
        xt[to + XP] = l;
      }
      if (++col == q.cols) {
        col = 0;
        ++row;
      }
    }
  }
  __syncthreads();

  f32x4 acc[MP / 16];
  const int r0 = wave * 16 + (lane >> 4) * 4;
  for (int step = 0; step < steps; ++step) {
    const int e = x_exp(q, r, step, k);
    const float gram = gram_factor(r, e);
    if (step < split_steps)
      small_step<true, MP>(x, xt, a, b, gram, k, acc);
    else
      small_step<false, MP>(x, xt, a, b, gram, k, acc);
    const bool last = step + 1 == steps;
    const float f = last ? ldexpf(r, -e) / B_SCALE
                         : ldexpf(1.f / B_SCALE, x_exp(q, r, step + 1, k) - e);
#pragma unroll
    for (int j = 0; j < MP / 16; ++j) {
      const int col = j * 16 + (lane & 15);
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = acc[j][i] * f;
      if (last) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r0 + i < q.n && col < q.m)
            out[q.start + (tall ? col * q.cols + r0 + i
                                : (r0 + i) * q.cols + col)] = (T)w[i];
      } else {
        put4(xt + place(col, r0, MP), XP, w);
        half_t* to = x + place(r0, col, SMALL_N);  // a row: 8 further
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          split(w[i], to[i * 8], to[i * 8 + XP]);
        }
      }
    }
    __syncthreads();
  }
}

// Workspace, in fp16 values: X and its transpose twice, A, B A, B and P
// twice, each as two planes; x_total and a_total: the sizes of one plane.  16
// bytes a padded value of X and 20 a value of A: 533 MB for ResNet-50.
struct Work {
  Planes x[2], xt[2], a, t, b, p[2];
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
    w.p[i] = take(a_total);
  }
  w.a = take(a_total);
  w.t = take(a_total);
  w.b = take(a_total);
  return w;
}

Planes planes(Planes p, bool lo) { return {p.h, lo ? p.l : nullptr}; }

// `count` steps, the first of them `step`, from X number `now` to the other,
// or to `out`.
template <bool SPLIT, class Src, class Out>
void ns_group(Src src, const Work& w, int step, int count, int now,
              bool next_split, bool last, Out out, const float* r, Coef k,
              int n_sym, int n_rect, hipStream_t s) {
  const dim3 block(256), sym(n_sym), rect(n_rect);
  const Planes x = w.x[now], xt = w.xt[now], none{nullptr, nullptr};
  auto lo = [](Planes p) { return planes(p, SPLIT); };
  // c = b m, and in the same launch d = b m2 where there is one (a step over
  // ResNet-18's matrices 356 -> 343 us, over ResNet-50's 793 -> 762)
  auto mul = [&](Planes b, Planes m, Planes c, Planes m2, Planes d) {
    hipLaunchKernelGGL((k_ns_gemm<SPLIT, MUL, Src, ToPlanes>),
                       dim3(n_sym, m2.h != nullptr ? 2 : 1), block, 0, s, src,
                       b, m, m2, lo(c), lo(d), ToPlanes{}, r, k, step, count);
  };
  hipLaunchKernelGGL((k_ns_gemm<SPLIT, GRAM, Src, ToPlanes>), sym, block, 0,
                     s, src, x, x, none, lo(w.a), none, ToPlanes{}, r, k,
                     step, count);
  for (int i = 0; i < count; ++i) {
    // the first B is P itself
    const Planes b = i == 0 ? w.p[0] : w.b;
    const Planes before = i == 0 ? none : w.p[(i - 1) & 1];
    hipLaunchKernelGGL((k_ns_gemm<SPLIT, POLY, Src, ToPlanes>), sym, block, 0,
                       s, src, w.a, w.a, none, lo(b), none, ToPlanes{}, r, k,
                       step, count);
    if (i + 1 < count) {
      mul(b, w.a, w.t, before, w.p[i & 1]);
      mul(b, w.t, w.a, none, none);
    } else if (i > 0) {
      mul(b, before, w.p[i & 1], none, none);
    }
  }
  const Planes p = w.p[(count - 1) & 1];
  if (last)
    hipLaunchKernelGGL((k_ns_gemm<SPLIT, APPLY, Src, Out>), rect, block, 0, s,
                       src, p, xt, none, none, none, out, r, k, step, count);
  else
    hipLaunchKernelGGL((k_ns_gemm<SPLIT, APPLY, Src, ToPlanes>), rect, block,
                       0, s, src, p, xt, none,
                       planes(w.x[now ^ 1], next_split),
                       planes(w.xt[now ^ 1], next_split), ToPlanes{}, r, k,
                       step, count);
}

// The first `split_steps` with pairs, in groups of up to `group`; the others
// one by one.
template <class Src, class Out>
void ns_steps(Src src, const Work& w, int steps, int split_steps, int group,
              Out out, const float* r, Coef k, int n_sym, int n_rect,
              hipStream_t s) {
  int now = 0;
  for (int i = 0; i < steps; now ^= 1) {
    const bool split = i < split_steps;
    const int left = split_steps - i;
    const int count = !split ? 1 : left < group ? left : group;
    auto f = split ? ns_group<true, Src, Out> : ns_group<false, Src, Out>;
    f(src, w, i, count, now, i + count < split_steps, i + count == steps, out,
      r, k, n_sym, n_rect, s);
    i += count;
  }
}

// Steps of a group, of at most `most`, for matrices with sum_nnm = sum of
// n^2 m and sum_nnn of n^3.  A further step in a group saves 3 n^2 m and costs
// 3 n^3, in products that fill the card less well, and a launch.  One by one
// and in groups, fp32, us:
//   128 x 1152 112, 110   256 x 512 110, 118   256 x 2304 163, 150
//   512 x 1024 148, 156   512 x 2048 175, 170   1000 x 2048 237, 235
//   1024 x 1536 218, 223   2048 x 2560 772, 781   2048 x 4096 1022, 944
//   4 of 512 x 1024 173, 169   4096 x 8192 6036, 5140
// so from m = 3 n on, and from m = 2 n on where the difference n^2 m - n^3 is
// large: 4e8 lies between one 512 x 1024 (1.3e8) and four (5.4e8).  Around the
// borders the two are within 5% of each other.
int group_of(int most, double sum_nnm, double sum_nnn) {
  const double more = sum_nnm - sum_nnn;
  return more >= 2.0 * sum_nnn || (more >= sum_nnn && more >= 4e8) ? most : 1;
}

// Of `tiles` tiles of 128 x 128, all with the same sum, how many to work on as
// such: a round is one on each of 256 CUs.  A last round of up to two thirds
// ends sooner as four times as many tiles of 64 x 64 (fp32, us, as tiles of
// 128 and of 64: the 128 of 1000 x 2048 252 and 222, 320 of 2048 x 2560 790
// and 754, 256 of 2048 x 2048 632 and 651, 253 of X X^T at 2816 x 2816 1272
// and 1377).
int64_t big_tiles(int64_t tiles) {
  const int64_t left = tiles % 256;
  return left <= 171 ? tiles - left : tiles;
}

// In a plan the sums differ, and a round of two tiles on each of 256 CUs ends
// with its longest: whole rounds of 512 only.  Of the symmetric products, where
// they last longest, none before a round and a quarter (us a step, with tiles
// of 128 and without: the 241 of ResNet-50 1015 and 793, 394 of ResNet-101 1306
// and 1147, 523 of ResNet-152 1545 and 1415; but 723 of three ResNet-50 2100
// and 2196; between 523 and 723 nothing was measured).
int64_t plan_big_tiles(int64_t tiles, bool sym) {
  return sym && tiles < 640 ? 0 : tiles - tiles % 512;
}

// Such a matrix needs no workspace.
bool is_small(int n, int m) { return n <= SMALL_N && m <= SMALL_M; }

template <typename T>
void newton_schulz(const T* g, T* out, const Mat& first, int batch, int steps,
                   int split_steps, int group, Coef k, float eps, void* work,
                   double* partials, float* r, hipStream_t s) {
  if (is_small(first.n, first.m)) {
    auto f = first.mp == 64 ? k_ns_small<T, 64>
             : first.mp == 128 ? k_ns_small<T, 128> : k_ns_small<T, 192>;
    // a launch has less than 2^32 threads
    const int most = 1 << 23;
    for (int64_t at = 0; at < batch; at += most) {
      const int now = (int)(batch - at < most ? batch - at : most);
      Uniform src{first, now, 0, 0};
      src.first.start = at * first.rows * first.cols;
      hipLaunchKernelGGL(f, dim3((unsigned)now), dim3(256), 0, s, src, g, out,
                         steps, split_steps, k, eps);
    }
    return;
  }
  const int64_t nt = first.np / 64, mt = first.mp / 64;
  const int64_t nb = nt / 2, mb = mt / 2;
  const int64_t syms = batch * (nb * (nb + 1) / 2), rects = batch * nb * mb;
  const int64_t big_sym = big_tiles(syms), big_rect = big_tiles(rects);
  const Uniform src{first, batch, (int)big_sym, (int)big_rect};
  const Work w = split_work(work, (int64_t)batch * first.np * first.mp,
                            (int64_t)batch * first.np * first.np);
  hipLaunchKernelGGL(k_ns_sumsq<T>, dim3((unsigned)(batch * first.chunk1)),
                     dim3(256), 0, s, src, g, partials);
  hipLaunchKernelGGL((k_ns_pack<Uniform, Plain<T>>),
                     dim3((unsigned)(batch * nt * mt)), dim3(256), 0, s, src,
                     Plain<T>{g}, partials, planes(w.x[0], split_steps > 0),
                     planes(w.xt[0], split_steps > 0), r, eps);
  const int64_t n_sym = big_sym + 4 * (syms - big_sym)
                        + batch * (nt & 1 ? nt : 0);
  const int64_t n_rect = big_rect + 4 * (rects - big_rect)
                         + batch * ((mt & 1 ? nt : 0)
                                    + (nt & 1 ? 2 * mb : 0));
  const double n = first.np, m = first.mp;
  ns_steps(src, w, steps, split_steps, group_of(group, n * n * m, n * n * n),
           ToTensor<T>{out}, r, k, (int)n_sym, (int)n_rect, s);
}

template <typename T>
void muon_step(float* p, const T* g, float* buf, __bf16* shadow,
               const float* lr, float mu, float wd, float rest_lr,
               bool nesterov, int steps, int group, Coef k, float eps,
               const void* tables, const int64_t* layout, void* work,
               double* partials, float* r, hipStream_t s) {
  // layout: matrices, chunks, tiles to pack, sym tiles, rect tiles, size of
  // an X plane, size of an A plane, sums of n^2 m and of n^3; the tables lie
  // in this order
  const char* at = static_cast<const char*>(tables);
  const Chunk* chunks = reinterpret_cast<const Chunk*>(at);
  Table src;
  src.packs = reinterpret_cast<const Task*>(chunks + layout[1]);
  src.syms = src.packs + layout[2];
  src.rects = src.syms + layout[3];
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
  ns_steps(src, w, steps, steps,
           group_of(group, (double)layout[7], (double)layout[8]),
           ToParams{p, shadow, lr, wd}, r, k, (int)layout[3], (int)layout[4],
           s);
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16 (sgp_muon_step: of the gradients, 0 or 1).
// The host has checked shapes and sizes and laid out the tables.
extern "C" {

int sgp_ns_chunk() { return CHUNK; }

int64_t sgp_ns_plan_big_tiles(int64_t tiles, bool sym) {
  return plan_big_tiles(tiles, sym);
}

bool sgp_ns_is_small(int n, int m) { return is_small(n, m); }

void sgp_newton_schulz(int dtype, const void* g, void* out, const void* mat,
                       int batch, int steps, int split_steps, int group,
                       float a, float b, float c, float growth, float eps,
                       void* work, double* partials, float* r,
                       hipStream_t s) {
  const Mat& first = *static_cast<const Mat*>(mat);
  const Coef k{a, b, c, log2f(growth)};
  if (dtype == 0)
    newton_schulz(static_cast<const float*>(g), static_cast<float*>(out),
                  first, batch, steps, split_steps, group, k, eps, work,
                  partials, r, s);
  else if (dtype == 1)
    newton_schulz(static_cast<const __bf16*>(g), static_cast<__bf16*>(out),
                  first, batch, steps, split_steps, group, k, eps, work,
                  partials, r, s);
  else
    newton_schulz(static_cast<const half_t*>(g), static_cast<half_t*>(out),
                  first, batch, steps, split_steps, group, k, eps, work,
                  partials, r, s);
}

void sgp_muon_step(int dtype, float* p, const void* g, float* buf,
                   void* shadow, const float* lr, float mu, float wd,
                   float rest_lr, bool nesterov, int steps, int group, float a,
                   float b, float c, float growth, float eps, const void* tables,
                   const int64_t* layout, void* work, double* partials,
                   float* r, hipStream_t s) {
  const Coef k{a, b, c, log2f(growth)};
  __bf16* sh = static_cast<__bf16*>(shadow);
  if (dtype == 0)
    muon_step(p, static_cast<const float*>(g), buf, sh, lr, mu, wd, rest_lr,
              nesterov, steps, group, k, eps, tables, layout, work, partials, r, s);
  else
    muon_step(p, static_cast<const __bf16*>(g), buf, sh, lr, mu, wd, rest_lr,
              nesterov, steps, group, k, eps, tables, layout, work, partials, r, s);
}

}  // extern "C"
