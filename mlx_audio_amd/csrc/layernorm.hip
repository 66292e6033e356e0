// Layer normalisation over the last axis, forward and backward (the norms of the transformer
// blocks behind the encoder stem; models/whisper/layers/encoder.py uses nn.LayerNorm).
//
//   forward   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) rstd w + b
//   backward  h = (x - mean) rstd, g = dy w,
//             dx = rstd (g - sum g / D - h sum (g h) / D), dw = sum over rows dy h, db = sum over rows dy
//
// Both are bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx, once
// each.  A row stays in registers between its sums and its result.  A second pass over them takes the
// differences d from the rounded mean m, and their mean c beside that of their squares: the mean is m + c
// (the error of a sum of large numbers falls out), the variance mean d^2 - c^2, and y comes from d - c, so a
// row far from zero loses nothing.  (1280 floats around 1000 +- 0.5: 2e-4 -> 2e-7; around 10000 +- 1: 1e-3.)  Rows
// up to 2048 two-byte elements (1024 ... 2048 floats) belong to one wave, so nothing waits on a
// barrier; rows up to 8192 elements to a workgroup; longer ones are read again from the caches.
// The backward's column sums are kept in registers over all rows that a wave walks, joined inside
// the workgroup in LDS, written as one partial row per workgroup and joined by a second launch in
// a fixed order, in double: no atomics, the same bits on every run.
// All sums are in float (the join, and the longer chains of rows beyond 8192 elements, in double); the one
// rounding is that of the stored result.
// Measured: forward, 96 000 x 1280 float16, 97 us a call = 5.1 TB/s; backward, 48 000 x 1280 bfloat16, 72 us =
// 5.1 TB/s, 5 of them the join (a 246 MB copy: 4.64 TB/s).  8 x 1280: 5 us, a call 13 with the host's work.
#include "column_sums.h"

namespace mia {
namespace ln {
using namespace nn;

struct Args {
  const void* x;
  const void* dy;
  long long x_stride, dy_stride;
  long long rows;
  int dim;
  const void* w;
  const void* b;
  float eps;
  float fdim;     // dim
  void* out;      // y or dx, rows of dim elements
  float* mean;    // (rows): written by the forward (or null), read by the backward
  float* rstd;
  float* partial;  // backward: (groups, 2, dim)
};

// V parameters from column i on; `other` where there are none or the row has ended
template <class W, int V>
__device__ __forceinline__ void load_params(const void* p, int i, int dim, float other, float* out) {
  constexpr int PW = kPer16<W>;
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = other;
  if (!p || i >= dim) return;
  if constexpr (PW <= V) {
#pragma unroll
    for (int j = 0; j < V; j += PW)
      if (i + j < dim) unpack<W>(load_piece(static_cast<const W*>(p) + i + j, dim - i - j), out + j);
  }
}
// sum over the LANES threads that share a row, the same value in all of them
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (LANES > 64) {
    constexpr int NW = LANES / 64;
    const int wv = threadIdx.x >> 6;
    __syncthreads();  // the last sum's readers are done
    if ((threadIdx.x & 63) == 0) red[wv] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += red[i];
  }
  return v;
}
// two sums at once
template <int LANES>
__device__ __forceinline__ void row_sums(float& v, float& w, float (*red)[2]) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o), w += __shfl_xor(w, o);
  if constexpr (LANES > 64) {
    constexpr int NW = LANES / 64;
    const int wv = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wv][0] = v, red[wv][1] = w;
    __syncthreads();
    v = w = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += red[i][0], w += red[i][1];
  }
}
// 1 / sqrt(variance + eps); c: mean difference, q: mean squared difference.  Rounding may put c^2 above q by
// its last bits where a row is constant; a NaN stays one.
__device__ __forceinline__ float inverse_spread(float c, float q, float eps) {
  const float variance = fmaf(-c, c, q);
  return 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + eps);
}
}  // namespace ln

// LANES threads per row, CH pieces of 16 bytes per thread: dim <= LANES * CH * (16 / sizeof T).
// PAST: the result goes past the caches.
template <class T, class W, int LANES, int CH, bool PAST>
__global__ __launch_bounds__(256) void ln_fwd_kernel(ln::Args p) {
  using namespace ln;
  constexpr int V = kPer16<T>, PER_WG = 256 / LANES;
  __shared__ float red[4], red2[4][2];
  const int t = threadIdx.x % LANES;
  const int dim = p.dim;
  float w[CH * V], b[CH * V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (c * LANES + t) * V;
    load_params<W, V>(p.w, i, dim, 1.0f, w + c * V);
    load_params<W, V>(p.b, i, dim, 0.0f, b + c * V);
  }
  for (long long row = (long long)blockIdx.x * PER_WG + threadIdx.x / LANES; row < p.rows;
       row += (long long)gridDim.x * PER_WG) {
    const T* __restrict__ x = static_cast<const T*>(p.x) + row * p.x_stride;
    float v[CH * V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * LANES + t) * V;
      unpack<T>(load_piece(x + i, dim - i, (p.rows - 1 - row) * p.x_stride + dim - i), v + c * V);
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < CH * V; ++j) s += v[j];
    const float mean = row_sum<LANES>(s, red) / p.fdim;  // divided: a constant row has exactly its mean
    s = 0.0f;
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = (c * LANES + t) * V + j;
        const float d = i < dim ? v[c * V + j] - mean : 0.0f;
        v[c * V + j] = d;
        s += d;
        q = fmaf(d, d, q);
      }
    row_sums<LANES>(s, q, red2);
    const float left = s / p.fdim, rstd = inverse_spread(left, q / p.fdim, p.eps);
    T* __restrict__ y = static_cast<T*>(p.out) + row * dim;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * LANES + t) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = fmaf((v[c * V + j] - left) * rstd, w[c * V + j], b[c * V + j]);
      store_piece<T, PAST>(y + i, pack<T>(o), dim - i);
    }
    if (t == 0 && p.mean) {
      p.mean[row] = mean + left;
      p.rstd[row] = rstd;
    }
  }
}

template <class T, class W, int LANES, int CH>
__global__ __launch_bounds__(256) void ln_bwd_kernel(ln::Args p) {
  using namespace ln;
  constexpr int V = kPer16<T>, PER_WG = 256 / LANES;
  constexpr int COLS = LANES * CH * V;
  __shared__ float red[4];
  __shared__ float cols[LANES == 64 ? 4 * COLS : 1];
  const int t = threadIdx.x % LANES;
  const int dim = p.dim;
  float w[CH * V], dw[CH * V], db[CH * V];
#pragma unroll
  for (int c = 0; c < CH; ++c) load_params<W, V>(p.w, (c * LANES + t) * V, dim, 1.0f, w + c * V);
#pragma unroll
  for (int j = 0; j < CH * V; ++j) dw[j] = db[j] = 0.0f;
  for (long long row = (long long)blockIdx.x * PER_WG + threadIdx.x / LANES; row < p.rows;
       row += (long long)gridDim.x * PER_WG) {
    const T* __restrict__ x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* __restrict__ dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[CH * V], g[CH * V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * LANES + t) * V;
      unpack<T>(load_piece(x + i, dim - i, (p.rows - 1 - row) * p.x_stride + dim - i), h + c * V);
      unpack<T>(load_piece(dy + i, dim - i, (p.rows - 1 - row) * p.dy_stride + dim - i), g + c * V);  // zero behind the row: no share in any sum
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < CH * V; ++j) {
      h[j] = (h[j] - mean) * rstd;
      dw[j] = fmaf(g[j], h[j], dw[j]);
      db[j] += g[j];
      g[j] *= w[j];
      s1 += g[j];
      s2 = fmaf(g[j], h[j], s2);
    }
    s1 = row_sum<LANES>(s1, red) / p.fdim;
    s2 = row_sum<LANES>(s2, red) / p.fdim;
    T* __restrict__ dx = static_cast<T*>(p.out) + row * dim;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (c * LANES + t) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = rstd * (g[c * V + j] - s1 - h[c * V + j] * s2);
      store_piece(dx + i, pack<T>(o), dim - i);
    }
  }
  if (!p.partial) return;
  float* __restrict__ out = p.partial + (long long)blockIdx.x * 2 * dim;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float* acc = half ? db : dw;
    if constexpr (LANES == 64) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) cols[(threadIdx.x >> 6) * COLS + (c * 64 + t) * V + j] = acc[c * V + j];
      __syncthreads();
      for (int i = threadIdx.x; i < dim; i += 256)
        out[half * dim + i] = (cols[i] + cols[COLS + i]) + (cols[2 * COLS + i] + cols[3 * COLS + i]);
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = (c * LANES + t) * V + j;
          if (i < dim) out[half * dim + i] = acc[c * V + j];
        }
    }
  }
}

// Rows longer than a workgroup's registers: one workgroup per row, the row read again for every sum.  A
// thread's chains, dim / 256 terms of up to 131 072, are in double.  One element a lane and load: 4000 x 10 000 float32
// 109 us, bfloat16 129 (backward 222, 157), a third and a quarter of HBM's rate.
template <class T, class W>
__global__ __launch_bounds__(256) void ln_fwd_long_kernel(ln::Args p) {
  using namespace ln;
  __shared__ float red[4], red2[4][2];
  const T* __restrict__ x = static_cast<const T*>(p.x) + (long long)blockIdx.x * p.x_stride;
  T* __restrict__ y = static_cast<T*>(p.out) + (long long)blockIdx.x * p.dim;
  double chain = 0.0, squares = 0.0;
  for (int i = threadIdx.x; i < p.dim; i += 256) chain += (double)x[i];
  const float mean = row_sum<256>((float)chain, red) / p.fdim;
  chain = 0.0;
  for (int i = threadIdx.x; i < p.dim; i += 256) {
    const double d = (double)((float)x[i] - mean);
    chain += d;
    squares = fma(d, d, squares);
  }
  float s = (float)chain, q = (float)squares;
  row_sums<256>(s, q, red2);
  const float left = s / p.fdim, rstd = inverse_spread(left, q / p.fdim, p.eps);
  for (int i = threadIdx.x; i < p.dim; i += 256) {
    const float w = p.w ? (float)static_cast<const W*>(p.w)[i] : 1.0f;
    const float b = p.b ? (float)static_cast<const W*>(p.b)[i] : 0.0f;
    y[i] = (T)fmaf(((float)x[i] - mean - left) * rstd, w, b);
  }
  if (threadIdx.x == 0 && p.mean) {
    p.mean[blockIdx.x] = mean + left;
    p.rstd[blockIdx.x] = rstd;
  }
}
template <class T, class W>
__global__ __launch_bounds__(256) void ln_bwd_long_kernel(ln::Args p) {
  using namespace ln;
  __shared__ float red[4];
  const T* __restrict__ x = static_cast<const T*>(p.x) + (long long)blockIdx.x * p.x_stride;
  const T* __restrict__ dy = static_cast<const T*>(p.dy) + (long long)blockIdx.x * p.dy_stride;
  T* __restrict__ dx = static_cast<T*>(p.out) + (long long)blockIdx.x * p.dim;
  const float mean = p.mean[blockIdx.x], rstd = p.rstd[blockIdx.x];
  double chain1 = 0.0, chain2 = 0.0;
  for (int i = threadIdx.x; i < p.dim; i += 256) {
    const float g = (float)dy[i] * (p.w ? (float)static_cast<const W*>(p.w)[i] : 1.0f);
    chain1 += (double)g;
    chain2 = fma((double)g, (double)(((float)x[i] - mean) * rstd), chain2);
  }
  const float s1 = row_sum<256>((float)chain1, red) / p.fdim;
  const float s2 = row_sum<256>((float)chain2, red) / p.fdim;
  for (int i = threadIdx.x; i < p.dim; i += 256) {
    const float g = (float)dy[i] * (p.w ? (float)static_cast<const W*>(p.w)[i] : 1.0f);
    dx[i] = (T)(rstd * (g - s1 - ((float)x[i] - mean) * rstd * s2));
  }
}
// column sums of the long rows: workgroup (x, y) adds rows y, y + gridDim.y, ... of 256 columns (up to 2^18 of
// them in one chain: in double)
template <class T>
__global__ __launch_bounds__(256) void ln_columns_kernel(ln::Args p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.dim) return;
  double dw = 0.0, db = 0.0;
  for (long long row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = (float)static_cast<const T*>(p.dy)[row * p.dy_stride + i];
    const float h = ((float)static_cast<const T*>(p.x)[row * p.x_stride + i] - p.mean[row]) * p.rstd[row];
    dw = fma((double)g, (double)h, dw);
    db += (double)g;
  }
  p.partial[((long long)blockIdx.y * 2) * p.dim + i] = (float)dw;
  p.partial[((long long)blockIdx.y * 2 + 1) * p.dim + i] = (float)db;
}

namespace ln {
constexpr int kMaxGroups = 512;   // workgroups of the backward: two per compute unit
constexpr int kLongGroups = 64;   // row groups of the long rows' column sums
constexpr int kRegisterDim = 8192;
// A forward result of this many bytes goes past the caches: what reads it next finds little of it in the
// 256 MB last-level cache anyway.  96 000 x 1280 float16 (246 MB): 114 -> 91 us, and a block of the encoder
// around it (64 clips) the same to 0.3 %; with smaller results past the caches too, such a block on 1 - 16
// clips took 2 % longer.
constexpr long long kPastCaches = 192LL << 20;

static int groups_of(long long rows, long long dim) {
  if (dim > kRegisterDim) return (int)(rows < kLongGroups ? rows : kLongGroups);
  return (int)(rows < kMaxGroups ? rows : kMaxGroups);
}

// Calls f(lanes, pieces) with the compiled shape that holds `dim` elements.
template <class T, class F>
static void with_shape(int dim, F f) {
  constexpr int V = kPer16<T>;
  using std::integral_constant;
#define MIA_LN_SHAPE(L, C) \
  if (dim <= L * C * V) return f(integral_constant<int, L>(), integral_constant<int, C>())
  MIA_LN_SHAPE(64, 1);
  MIA_LN_SHAPE(64, 2);
  MIA_LN_SHAPE(64, 3);
  MIA_LN_SHAPE(64, 4);
  if constexpr (V == 4) {
    MIA_LN_SHAPE(64, 5);
    MIA_LN_SHAPE(64, 6);
    MIA_LN_SHAPE(64, 8);
    MIA_LN_SHAPE(256, 4);
    MIA_LN_SHAPE(256, 6);
    MIA_LN_SHAPE(256, 8);
  } else {
    MIA_LN_SHAPE(256, 2);
    MIA_LN_SHAPE(256, 3);
    MIA_LN_SHAPE(256, 4);
  }
#undef MIA_LN_SHAPE
}

template <class T, class W>
static void launch_fwd(const Args& a, hipStream_t s) {
  if (a.dim > kRegisterDim) {
    hipLaunchKernelGGL((ln_fwd_long_kernel<T, W>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    return;
  }
  with_shape<T>(a.dim, [&](auto lanes, auto pieces) {
    constexpr int per = 256 / decltype(lanes)::value;
    const long long need = (a.rows + per - 1) / per;
    const unsigned grid = (unsigned)(need < 2048 ? need : 2048);  // eight workgroups per compute unit
    constexpr int L = decltype(lanes)::value, C = decltype(pieces)::value;
    if (a.rows * a.dim * (long long)sizeof(T) >= kPastCaches)
      hipLaunchKernelGGL((ln_fwd_kernel<T, W, L, C, true>), dim3(grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((ln_fwd_kernel<T, W, L, C, false>), dim3(grid), dim3(256), 0, s, a);
  });
}
template <class T, class W>
static void launch_bwd(const Args& a, int groups, hipStream_t s) {
  if (a.dim > kRegisterDim) {
    hipLaunchKernelGGL((ln_bwd_long_kernel<T, W>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    if (a.partial)
      hipLaunchKernelGGL(ln_columns_kernel<T>, dim3((unsigned)((a.dim + 255) / 256), (unsigned)groups), dim3(256), 0, s, a);
    return;
  }
  with_shape<T>(a.dim, [&](auto lanes, auto pieces) {
    hipLaunchKernelGGL((ln_bwd_kernel<T, W, decltype(lanes)::value, decltype(pieces)::value>), dim3((unsigned)groups),
                       dim3(256), 0, s, a);
  });
}

static int check(long long rows, long long dim, int dtype, const void* w, const void* b, int param_dtype) {
  MIA_REQUIRE(rows >= 0 && rows < (1LL << 31), "rows must be in 0 .. 2^31 - 1 (got %lld)", rows);
  // (a launch counts its threads in 32 bits: 64 a column in the join, 256 a long row)
  MIA_REQUIRE(dim >= 1 && dim <= (1LL << 25), "dim must be in 1 .. 2^25 (got %lld)", dim);
  MIA_REQUIRE(dim <= kRegisterDim || rows < (1LL << 24), "rows of more than %d elements: at most 2^24 - 1 (got %lld)",
              kRegisterDim, rows);
  MIA_REQUIRE(dtype_ok(dtype), "unknown dtype %d", dtype);
  MIA_REQUIRE((!w && !b) || param_dtype == dtype || param_dtype == MIA_F32,
              "parameters must be float32 or of the input's type");
  return MIA_OK;
}
}  // namespace ln
}  // namespace mia

using namespace mia;

extern "C" {

int mia_layer_norm(const void* x, int64_t rows, int64_t dim, int64_t x_stride, int dtype, const void* weight,
                   const void* bias, int param_dtype, float eps, void* y, float* mean, float* rstd, void* stream) {
  const int rc = ln::check(rows, dim, dtype, weight, bias, param_dtype);
  if (rc != MIA_OK) return rc;
  MIA_REQUIRE(eps >= 0.0f, "eps must not be negative");
  MIA_REQUIRE((mean == nullptr) == (rstd == nullptr), "mean and rstd come together");
  if (rows == 0) return MIA_OK;
  MIA_REQUIRE(x && y, "null argument");
  MIA_REQUIRE(x_stride >= 0, "rows must not run backwards");
  hipStream_t s = static_cast<hipStream_t>(stream);
  ln::Args a{x, nullptr, x_stride, 0, rows, (int)dim, weight, bias, eps, (float)dim, y, mean, rstd, nullptr};
  nn::with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (param_dtype == MIA_F32) ln::launch_fwd<T, float>(a, s);
    else ln::launch_fwd<T, T>(a, s);
    return 0;
  });
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

size_t mia_layer_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return (size_t)ln::groups_of(rows, dim) * 2 * dim * sizeof(float);
}

int mia_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                            const float* rstd, int64_t rows, int64_t dim, int dtype, const void* weight,
                            int param_dtype, void* dx, float* dweight, float* dbias, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int rc = ln::check(rows, dim, dtype, weight, nullptr, param_dtype);
  if (rc != MIA_OK) return rc;
  MIA_REQUIRE((dweight == nullptr) == (dbias == nullptr), "dweight and dbias come together");
  MIA_REQUIRE(rows == 0 || (dy && x && mean && rstd && dx), "null argument");
  MIA_REQUIRE(dy_stride >= 0 && x_stride >= 0, "rows must not run backwards");
  MIA_REQUIRE(!dweight || rows == 0 ||
                  (workspace && workspace_bytes >= mia_layer_norm_backward_workspace_bytes(rows, dim) &&
                   nn::aligned16(workspace)),
              "workspace too small or not aligned to 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int groups = rows ? ln::groups_of(rows, dim) : 0;
  if (rows) {
    ln::Args a{dy ? x : nullptr, dy, x_stride, dy_stride, rows, (int)dim, weight, nullptr, 0.0f, (float)dim, dx,
               const_cast<float*>(mean), const_cast<float*>(rstd), dweight ? static_cast<float*>(workspace) : nullptr};
    nn::with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      if (param_dtype == MIA_F32) ln::launch_bwd<T, float>(a, groups, s);
      else ln::launch_bwd<T, T>(a, groups, s);
      return 0;
    });
  }
  if (dweight) {
    const int n = (int)(2 * dim);
    hipLaunchKernelGGL(nn::join_columns_kernel, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, s,
                       static_cast<const float*>(workspace), groups, n, dweight, dbias, (int)dim);
  }
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

}  // extern "C"
