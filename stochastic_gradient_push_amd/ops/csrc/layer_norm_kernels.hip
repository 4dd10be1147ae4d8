// Layer norm over the last dimension (+residual)(+ReLU), forward and
// backward, for gfx950 (CDNA4).  bf16, fp16 or fp32 rows, fp32 arithmetic.
//
//   mean = sum(x) / C            var = sum((x - mean)^2) / C
//   hat  = (x - mean) * rstd     rstd = 1 / sqrt(var + eps)
//   y    = relu(hat * w + b + res)
//
//   g    = dy where the sum is positive, rounded to zero or not;  dres = g
//   dw   = sum_rows(g * hat)     db   = sum_rows(g)
//   dx   = rstd * (g w - mean_cols(g w) - hat * mean_cols(g w hat))
//
// The variance comes from the centred values that are still in registers,
// never from a difference of squares.
//
// Bound by memory: each row is read once per pass and written once.  100352 x
// 256 bf16 with residual and ReLU: forward 30 us (5.1 TB/s), backward 43 us
// (6.0) and 5 us for the column sums; 4096 x 16384 fp16 59 us (4.6), 101 us
// (4.0, with registers spilled) and 14 us; 8191 x 1001 fp32 16 us, 23 us and
// 9 us.  Below about 5 MB the launches count, 3 us each, and autograd's way to
// them, 50 us.

#include <hip/hip_runtime.h>

#include <cstdint>

namespace {

// N: values in 16 bytes; ZERO: the largest that rounds to 0, half of the
// type's smallest
template <typename T> struct Pack;
template <> struct Pack<__bf16> {
  static constexpr int N = 8;
  static constexpr float ZERO = 0x1p-134f;
  typedef __bf16 V __attribute__((ext_vector_type(8)));
};
template <> struct Pack<_Float16> {
  static constexpr int N = 8;
  static constexpr float ZERO = 0x1p-25f;
  typedef _Float16 V __attribute__((ext_vector_type(8)));
};
template <> struct Pack<float> {
  static constexpr int N = 4;
  static constexpr float ZERO = 0.f;
  typedef float V __attribute__((ext_vector_type(4)));
};

// 16 bytes at any element: rows of an odd width start off a 16-byte border,
// and global memory takes such an access in one instruction
template <typename T>
__device__ __forceinline__ typename Pack<T>::V ldv(const T* p) {
  typedef typename Pack<T>::V U __attribute__((aligned(sizeof(T))));
  return *reinterpret_cast<const U*>(p);
}
template <typename T>
__device__ __forceinline__ void stv(T* p, typename Pack<T>::V v) {
  typedef typename Pack<T>::V U __attribute__((aligned(sizeof(T))));
  *reinterpret_cast<U*>(p) = v;
}

// elements [c, c + N) of a row of C, 0 behind its end; as they are, or as
// floats
template <typename T>
__device__ __forceinline__ typename Pack<T>::V raw(const T* row, int c,
                                                   int C) {
  constexpr int N = Pack<T>::N;
  if (c + N <= C) return ldv(row + c);
  typename Pack<T>::V v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = c + j < C ? row[c + j] : (T)0.f;
  return v;
}
template <typename T>
__device__ __forceinline__ void load(const T* row, int c, int C, float* f) {
  const typename Pack<T>::V v = raw<T>(row, c, C);
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j) f[j] = (float)v[j];
}

template <typename T>
__device__ __forceinline__ void store(T* row, int c, int C, const float* f) {
  constexpr int N = Pack<T>::N;
  if (c + N <= C) {
    typename Pack<T>::V v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)f[j];
    stv(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j < C) row[c + j] = (T)f[j];
  }
}

// a weight vector in the rows' type or in fp32; none at all: `none`
template <typename T>
__device__ __forceinline__ void load_w(const void* w, bool w32, int c, int C,
                                       float none, float* f) {
  constexpr int N = Pack<T>::N;
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = none;
  } else if (w32) {
    const float* p = static_cast<const float*>(w);
#pragma unroll
    for (int j = 0; j < N; j += 4) load<float>(p, c + j, C, f + j);
  } else {
    load<T>(static_cast<const T*>(w), c, C, f);
  }
}

template <typename T>
__device__ __forceinline__ void put_w(void* w, bool w32, int64_t c, float f) {
  if (w32)
    static_cast<float*>(w)[c] = f;
  else
    static_cast<T*>(w)[c] = (T)f;
}

// max(z, 0); a NaN stays.  The backward pass reads y to know where z was
// positive, so a positive z that T rounds to zero becomes -0, and +0 means
// that there is no gradient.
template <typename T>
__device__ __forceinline__ float rectify(float z) {
  const float f = z > 0.f ? -0.f : 0.f;
  return !(z <= Pack<T>::ZERO) ? z : f;
}
__device__ __forceinline__ bool was_cut(float y) {
  return __float_as_uint(y) == 0;
}

// Sum of K values over the TPR threads of a row, the same in each of them.
// Up to a wave: butterflies.  Above: a block has one row, its waves meet in
// `lds` (K * TPR / 64 floats, not touched again before the next barrier).
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float* v, float* lds) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o);
  if (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) lds[k * W + wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += lds[k * W + i];
    }
  }
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

// --------------------------------------------------------------- forward
// TPR threads hold one row, VPT 16-byte vectors each, and walk over the rows
// with the weights in registers.  The next row is on its way while one is
// reduced, where a block has only one.
template <typename T, int TPR, int VPT>
__global__ __launch_bounds__(block_of(TPR)) void k_ln_fwd(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ res,
    int64_t rs, const void* __restrict__ w, const void* __restrict__ b,
    bool w32, T* __restrict__ y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, float eps, int64_t M, int C, bool relu) {
  typedef typename Pack<T>::V V;
  constexpr int N = Pack<T>::N;
  constexpr int G = block_of(TPR) / TPR;
  __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / TPR;
  constexpr bool AHEAD = TPR > 64;  // shorter rows: other waves fill in
  V next[VPT], next_res[VPT];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * TPR) * N;
      next[i] = raw<T>(x + row * xs, c, C);
      if (res != nullptr) next_res[i] = raw<T>(res + row * rs, c, C);
    }
  };
  if (AHEAD && r < M) fetch(r);
  float wv[VPT][N], bv[VPT][N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    load_w<T>(w, w32, (t + i * TPR) * N, C, 1.f, wv[i]);
    load_w<T>(b, w32, (t + i * TPR) * N, C, 0.f, bv[i]);
  }
  for (; r < M; r += step) {
    V now[VPT], now_res[VPT];
    if (!AHEAD) fetch(r);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      now[i] = next[i];
      now_res[i] = next_res[i];
    }
    if (AHEAD && r + step < M) fetch(r + step);
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) s += (float)now[i][j];
    row_sum<TPR, 1>(&s, lds);
    const float mean = s / (float)C;  // exact where the sum is
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (float)now[i][j] - mean;
        if ((t + i * TPR) * N + j < C) q += d * d;
      }
    row_sum<TPR, 1>(&q, lds);
    const float rstd = 1.f / sqrtf(q / (float)C + eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float z = ((float)now[i][j] - mean) * rstd * wv[i][j] + bv[i][j];
        if (res != nullptr) z += (float)now_res[i][j];
        f[j] = z;
      }
      if (relu)
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = rectify<T>(f[j]);
      store<T>(y + r * C, (t + i * TPR) * N, C, f);
    }
    if (mean_out != nullptr && t == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

// Rows too long for registers: one block each, read three times.  A thread
// may have 2^20 values of a row: it adds up the 4 or 8 of a vector, and the
// vectors' sums in 64 bits: one after another in 32 bits the mean of 2^26
// values of 0.1 was off by 6e-4 of itself, and of a row without a variance
// nothing else is left.  It costs nothing (4096 x 16384 fp32 147 us, both ways
// 347; 1024 x 65536 bf16 76 and 196).
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_fwd_long(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ res,
    int64_t rs, const void* __restrict__ w, const void* __restrict__ b,
    bool w32, T* __restrict__ y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, float eps, int64_t M, int C, bool relu) {
  constexpr int N = Pack<T>::N;
  __shared__ float lds[16];
  const float inv = 1.f / (float)C;
  for (int64_t r = blockIdx.x; r < M; r += gridDim.x) {
    const T* xr = x + r * xs;
    float f[N];
    double all = 0.0;
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      load<T>(xr, (int)c, C, f);
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) v += f[j];
      all += v;
    }
    float s = (float)all;
    row_sum<1024, 1>(&s, lds);
    const float mean = s / (float)C;  // exact where the sum is
    all = 0.0;
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      load<T>(xr, (int)c, C, f);
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < C) v += (f[j] - mean) * (f[j] - mean);
      all += v;
    }
    float q = (float)all;
    row_sum<1024, 1>(&q, lds);
    const float rstd = 1.f / sqrtf(q * inv + eps);
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      float wv[N], bv[N], a[N];
      load<T>(xr, (int)c, C, f);
      load_w<T>(w, w32, (int)c, C, 1.f, wv);
      load_w<T>(b, w32, (int)c, C, 0.f, bv);
      if (res != nullptr) load<T>(res + r * rs, (int)c, C, a);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float z = (f[j] - mean) * rstd * wv[j] + bv[j];
        if (res != nullptr) z += a[j];
        f[j] = z;
      }
      if (relu)
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = rectify<T>(f[j]);
      store<T>(y + r * C, (int)c, C, f);
    }
    if (mean_out != nullptr && threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

// -------------------------------------------------------------- backward
// Same split.  Each thread keeps the sums of its columns over the rows of
// its block: partials[block] = {dw[C], db[C]} in fp32, added up in a fixed
// order by k_ln_bwd_sum.
template <typename T, int TPR, int VPT, bool RELU>
__global__ __launch_bounds__(block_of(TPR)) void k_ln_bwd(
    const T* __restrict__ dy, int64_t ds, const T* __restrict__ x,
    int64_t xs, const T* __restrict__ y, const void* __restrict__ w,
    bool w32, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ dx, T* __restrict__ dres, float* __restrict__ partials,
    int64_t M, int C) {
  typedef typename Pack<T>::V V;
  constexpr int N = Pack<T>::N;
  constexpr int BT = block_of(TPR);
  constexpr int G = BT / TPR;
  constexpr int W = BT / 64;
  __shared__ float lds[TPR > 64 ? 2 * W : W * TPR * VPT * N];
  const int t = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / TPR;
  V next_x[VPT], next_g[VPT], next_y[RELU ? VPT : 1];
  float next_mu = 0.f, next_rs = 0.f;
  auto fetch = [&](int64_t row) {
    next_mu = mean[row];
    next_rs = rstd[row];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * TPR) * N;
      next_x[i] = raw<T>(x + row * xs, c, C);
      next_g[i] = raw<T>(dy + row * ds, c, C);  // g = 0 behind the end
      if (RELU) next_y[i] = raw<T>(y + row * C, c, C);
    }
  };
  if (r < M) fetch(r);
  float wv[VPT][N], sw[VPT][N], sb[VPT][N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    load_w<T>(w, w32, (t + i * TPR) * N, C, 1.f, wv[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) sw[i][j] = sb[i][j] = 0.f;
  }
  const float inv = 1.f / (float)C;
  for (; r < M; r += step) {
    V xv[VPT], gv[VPT];
    const float mu = next_mu, rs = next_rs;
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      xv[i] = next_x[i];
      gv[i] = next_g[i];
      if constexpr (RELU)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (was_cut((float)next_y[i][j])) gv[i][j] = (T)0.f;
      if (dres != nullptr) {
        const int c = (t + i * TPR) * N;
        if (c + N <= C) {
          stv(dres + r * C + c, gv[i]);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (c + j < C) dres[r * C + c + j] = gv[i][j];
        }
      }
    }
    if (r + step < M) fetch(r + step);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float g = (float)gv[i][j], h = ((float)xv[i][j] - mu) * rs;
        sw[i][j] += g * h;
        sb[i][j] += g;
        const float gw = g * wv[i][j];
        s[0] += gw;
        s[1] += gw * h;
      }
    if (dx != nullptr) {
      row_sum<TPR, 2>(s, lds);
      const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float h = ((float)xv[i][j] - mu) * rs;
          f[j] = rs * ((float)gv[i][j] * wv[i][j] - m0 - h * m1);
        }
        store<T>(dx + r * C, (t + i * TPR) * N, C, f);
      }
    }
  }
  if (partials == nullptr) return;
  float* out = partials + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float v = half ? sb[i][j] : sw[i][j];
        // the rows of a wave, then its block's waves
#pragma unroll
        for (int o = TPR; o < 64; o <<= 1) v += __shfl_xor(v, o);
        const int c = (t + i * TPR) * N + j;
        if (TPR > 64) {
          if (c < C) out[half * C + c] = v;
        } else if ((threadIdx.x & 63) < TPR) {
          lds[(threadIdx.x >> 6) * TPR * VPT * N + c] = v;
        }
      }
    if (TPR <= 64) {
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += BT) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) v += lds[k * TPR * VPT * N + c];
        out[half * C + c] = v;
      }
      __syncthreads();
    }
  }
}

// Rows too long for registers: dx of one row by one block, and the columns'
// sums by k_ln_bwd_cols.
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_bwd_long(
    const T* __restrict__ dy, int64_t ds, const T* __restrict__ x,
    int64_t xs, const T* __restrict__ y, const void* __restrict__ w,
    bool w32, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ dx, T* __restrict__ dres, int64_t M, int C) {
  constexpr int N = Pack<T>::N;
  __shared__ float lds[32];
  const float inv = 1.f / (float)C;
  for (int64_t r = blockIdx.x; r < M; r += gridDim.x) {
    const float mu = mean[r], rs = rstd[r];
    float m0 = 0.f, m1 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      double all[2] = {0.0, 0.0};  // as in k_ln_fwd_long
      for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
        float h[N], gv[N], wv[N], v[2] = {0.f, 0.f};
        load<T>(x + r * xs, (int)c, C, h);
        load<T>(dy + r * ds, (int)c, C, gv);
        load_w<T>(w, w32, (int)c, C, 1.f, wv);
        if (y != nullptr) {
          float a[N];
          load<T>(y + r * C, (int)c, C, a);
#pragma unroll
          for (int j = 0; j < N; ++j) gv[j] = was_cut(a[j]) ? 0.f : gv[j];
        }
        if (pass == 0 && dres != nullptr)
          store<T>(dres + r * C, (int)c, C, gv);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          h[j] = (h[j] - mu) * rs;
          gv[j] *= wv[j];
          v[0] += gv[j];
          v[1] += gv[j] * h[j];
          gv[j] = rs * (gv[j] - m0 - h[j] * m1);
        }
        all[0] += v[0];
        all[1] += v[1];
        if (pass == 1) store<T>(dx + r * C, (int)c, C, gv);
      }
      if (dx == nullptr) break;
      if (pass == 0) {
        float s[2] = {(float)all[0], (float)all[1]};
        row_sum<1024, 2>(s, lds);
        m0 = s[0] * inv;
        m1 = s[1] * inv;
      }
    }
  }
}

// partials[by] of 256 * N columns over the rows by, by + gridDim.y, ...
template <typename T>
__global__ __launch_bounds__(256) void k_ln_bwd_cols(
    const T* __restrict__ dy, int64_t ds, const T* __restrict__ x,
    int64_t xs, const T* __restrict__ y, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ partials, int64_t M,
    int C) {
  constexpr int N = Pack<T>::N;
  const int64_t c64 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (c64 >= C) return;
  const int c = (int)c64;
  float sw[N] = {0.f}, sb[N] = {0.f};
  for (int64_t r = blockIdx.y; r < M; r += gridDim.y) {
    const float mu = mean[r], rs = rstd[r];
    float h[N], gv[N];
    load<T>(x + r * xs, c, C, h);
    load<T>(dy + r * ds, c, C, gv);
    if (y != nullptr) {
      float a[N];
      load<T>(y + r * C, c, C, a);
#pragma unroll
      for (int j = 0; j < N; ++j) gv[j] = was_cut(a[j]) ? 0.f : gv[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      sw[j] += gv[j] * ((h[j] - mu) * rs);
      sb[j] += gv[j];
    }
  }
  float* out = partials + (int64_t)blockIdx.y * 2 * C;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (c + j < C) {
      out[c + j] = sw[j];
      out[C + c + j] = sb[j];
    }
}

// Column sums of partials [P][2C] from column c0 on: a block has 16 columns
// and `blockDim.x` / 16 threads on each, which add up in a fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_bwd_sum(
    const float* __restrict__ partials, int P, int C, int64_t c0,
    void* __restrict__ dw, void* __restrict__ db, bool w32) {
  __shared__ float lds[1024];
  const int cl = threadIdx.x & 15, k0 = threadIdx.x >> 4;
  const int K = blockDim.x >> 4;
  const int64_t c = c0 + (int64_t)blockIdx.x * 16 + cl, S = 2 * (int64_t)C;
  float v = 0.f;
  if (c < S) {
    const float* p = partials + c;
    int k = k0;
    for (; k + 7 * K < P; k += 8 * K) {  // eight on their way at once
      float a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = p[(int64_t)(k + i * K) * S];
#pragma unroll
      for (int i = 0; i < 8; ++i) v += a[i];
    }
    for (; k < P; k += K) v += p[(int64_t)k * S];
  }
  lds[threadIdx.x] = v;
  __syncthreads();
  for (int h = K / 2; h > 0; h >>= 1) {
    if (k0 < h) lds[threadIdx.x] += lds[threadIdx.x + h * 16];
    __syncthreads();
  }
  if (k0 != 0 || c >= S) return;
  v = lds[cl];
  if (c < C) {
    if (dw != nullptr) put_w<T>(dw, w32, c, v);
  } else if (db != nullptr) {
    put_w<T>(db, w32, c - C, v);
  }
}

// ---------------------------------------------------------------- launch
// The narrowest row group that holds a row in registers: short rows share
// a wave, longer ones have a wave or a block.  Two vectors a thread at most:
// with four, the backward pass has 200 registers and more.  With two it fits,
// but for 16-bit rows over 8192: 1024 threads may have 128 registers each, and
// 16 of those needed (23 with a ReLU) are spilled, 68 (80) bytes a thread.
constexpr int MAX_VECTORS = 1024 * 2;

#define LN_FOR_SHAPE(nv, CALL)                                     \
  do {                                                             \
    if ((nv) <= 8) { CALL(8, 1); }                                 \
    else if ((nv) <= 16) { CALL(16, 1); }                          \
    else if ((nv) <= 32) { CALL(32, 1); }                          \
    else if ((nv) <= 64) { CALL(64, 1); }                          \
    else if ((nv) <= 128) { CALL(64, 2); }                         \
    else if ((nv) <= 256) { CALL(256, 1); }                        \
    else if ((nv) <= 512) { CALL(256, 2); }                        \
    else if ((nv) <= 1024) { CALL(512, 2); }                       \
    else { CALL(1024, 2); }                                        \
  } while (0)

template <typename T>
int vectors(int64_t C) {
  return (int)((C + Pack<T>::N - 1) / Pack<T>::N);
}

int groups_of(int nv) {  // rows that a block of k_ln_fwd / k_ln_bwd has
  return nv <= 8 ? 32 : nv <= 16 ? 16 : nv <= 32 ? 8 : nv <= 128 ? 4 : 1;
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Blocks that the card holds at once.  A forward grid has no more: its
// blocks walk over the rows and read the weights once.
template <class K>
int64_t resident(K kernel, int threads) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &per_cu, reinterpret_cast<const void*>(kernel), threads, 0)
          != hipSuccess || per_cu < 1)
    per_cu = 1;
  return 256 * (int64_t)per_cu;
}

template <typename T>
void fwd(const void* x, int64_t xs, const void* res, int64_t rs,
         const void* w, const void* b, bool w32, void* y, float* mean,
         float* rstd, float eps, int64_t M, int C, bool relu,
         hipStream_t s) {
  const int nv = vectors<T>(C);
  const T* xp = static_cast<const T*>(x);
  const T* rp = static_cast<const T*>(res);
  T* yp = static_cast<T*>(y);
  if (nv > MAX_VECTORS) {
    const int grid = (int)(M < 512 ? M : 512);
    hipLaunchKernelGGL(k_ln_fwd_long<T>, dim3(grid), dim3(1024), 0, s, xp,
                       xs, rp, rs, w, b, w32, yp, mean, rstd, eps, M, C,
                       relu);
    return;
  }
  const int64_t rows = cdiv(M, groups_of(nv));
#define LN_FWD(TPR, VPT)                                              \
  static const int64_t most =                                         \
      resident(k_ln_fwd<T, TPR, VPT>, block_of(TPR));                 \
  hipLaunchKernelGGL((k_ln_fwd<T, TPR, VPT>),                         \
                     dim3((unsigned)(rows < most ? rows : most)),     \
                     dim3(block_of(TPR)), 0, s, xp, xs, rp, rs, w, b, \
                     w32, yp, mean, rstd, eps, M, C, relu)
  LN_FOR_SHAPE(nv, LN_FWD);
#undef LN_FWD
}

// Blocks of the backward pass, each with a row of partial sums: what the
// card holds at once, if the partial sums (16 bytes a column, written and
// read) then stay below a quarter of the rows (x, dy and dx); two a CU, one
// of 1024 threads, in any case.
template <typename T>
int partial_rows(int64_t M, int C) {
  const int nv = vectors<T>(C);
  if (nv > MAX_VECTORS) return (int)(cdiv(M, 16) < 512 ? cdiv(M, 16) : 512);
  int64_t most = 0;
#define LN_MOST(TPR, VPT)                                             \
  static const int64_t n =                                            \
      resident(k_ln_bwd<T, TPR, VPT, true>, block_of(TPR));                 \
  most = n
  LN_FOR_SHAPE(nv, LN_MOST);
#undef LN_MOST
  const int64_t least = nv > 1024 ? 256 : 512;
  const int64_t small = M * (int64_t)sizeof(T) * 3 / 64;
  if (most > small) most = small;
  if (most < least) most = least;
  const int64_t rows = cdiv(M, groups_of(nv));
  return (int)(rows < most ? rows : most);
}

template <typename T>
void bwd(const void* dy, int64_t ds, const void* x, int64_t xs,
         const void* y, const void* w, bool w32, const float* mean,
         const float* rstd, void* dx, void* dres, float* partials, int P,
         void* dw, void* db, bool g32, int64_t M, int C, hipStream_t s) {
  const int nv = vectors<T>(C);
  const T* xp = static_cast<const T*>(x);
  const T* dp = static_cast<const T*>(dy);
  const T* yp = static_cast<const T*>(y);
  T* dxp = static_cast<T*>(dx);
  T* drp = static_cast<T*>(dres);
  if (nv > MAX_VECTORS) {
    if (dx != nullptr || dres != nullptr) {
      const int grid = (int)(M < 512 ? M : 512);
      hipLaunchKernelGGL(k_ln_bwd_long<T>, dim3(grid), dim3(1024), 0, s, dp,
                         ds, xp, xs, yp, w, w32, mean, rstd, dxp, drp, M, C);
    }
    if (partials != nullptr) {
      const dim3 grid((unsigned)cdiv(C, 256 * Pack<T>::N), (unsigned)P);
      hipLaunchKernelGGL(k_ln_bwd_cols<T>, grid, dim3(256), 0, s, dp, ds, xp,
                         xs, yp, mean, rstd, partials, M, C);
    }
  } else {
#define LN_BWD(TPR, VPT)                                              \
  auto f = yp != nullptr ? k_ln_bwd<T, TPR, VPT, true>                \
                         : k_ln_bwd<T, TPR, VPT, false>;              \
  hipLaunchKernelGGL(f, dim3(P), dim3(block_of(TPR)), 0, s, dp, ds,   \
                     xp, xs, yp, w, w32, mean, rstd, dxp, drp,        \
                     partials, M, C)
    LN_FOR_SHAPE(nv, LN_BWD);
#undef LN_BWD
  }
  if (partials == nullptr) return;
  // 64 or 16 threads a column: a launch of up to 2^31 of the 2^32 threads
  // that it may have
  const int64_t S = 2 * (int64_t)C, most = (int64_t(1) << 31) / 64;
  for (int64_t c0 = 0; c0 < S; c0 += most) {
    const int64_t cols = S - c0 < most ? S - c0 : most;
    hipLaunchKernelGGL(k_ln_bwd_sum<T>, dim3((unsigned)cdiv(cols, 16)),
                       dim3(P > 64 ? 1024 : 256), 0, s, partials, P, C, c0,
                       dw, db, g32);
  }
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16.  w32 / g32: weights (their gradients) are
// fp32 rather than in the rows' type.  Any of res, w, b, mean, y, dx, dres,
// partials, dw and db may be null.  M and C are positive.  P, the backward
// grid, is what sgp_layer_norm_partials has given; partials has P rows of 2 C.
extern "C" {

void sgp_layer_norm_fwd(int dtype, const void* x, int64_t xs,
                        const void* res, int64_t rs, const void* w,
                        const void* b, bool w32, void* y, float* mean,
                        float* rstd, float eps, int64_t M, int C, bool relu,
                        hipStream_t s) {
  auto f = dtype == 0 ? fwd<float> : dtype == 1 ? fwd<__bf16> : fwd<_Float16>;
  f(x, xs, res, rs, w, b, w32, y, mean, rstd, eps, M, C, relu, s);
}

int sgp_layer_norm_partials(int dtype, int64_t M, int C) {
  return dtype == 0   ? partial_rows<float>(M, C)
         : dtype == 1 ? partial_rows<__bf16>(M, C)
                      : partial_rows<_Float16>(M, C);
}

void sgp_layer_norm_bwd(int dtype, const void* dy, int64_t ds, const void* x,
                        int64_t xs, const void* y, const void* w, bool w32,
                        const float* mean, const float* rstd, void* dx,
                        void* dres, float* partials, int P, void* dw,
                        void* db, bool g32, int64_t M, int C, hipStream_t s) {
  auto f = dtype == 0 ? bwd<float> : dtype == 1 ? bwd<__bf16> : bwd<_Float16>;
  f(dy, ds, x, xs, y, w, w32, mean, rstd, dx, dres, partials, P, dw, db, g32,
    M, C, s);
}

}  // extern "C"
