// C entry points of the linear layer (kernels: linear_kernels.h, one translation unit per element type).
#include "column_sums.h"
#include "linear_kernels.h"

namespace mia {
namespace lin {
constexpr long long kMaxSize = (1LL << 30) - 4096;  // positions along k are counted in 32 bits
constexpr long long kMaxWidth = 1LL << 26;          // and so are a launch's threads (up to 32 a column)
constexpr int kBiasGroups = 256;
// at least sixteen rows each
static int bias_groups(long long m) { return (int)((m + 15) / 16 < kBiasGroups ? (m + 15) / 16 : kBiasGroups); }

static int check(long long m, long long n, long long k, int dtype) {
  MIA_REQUIRE(m >= 0 && n >= 1 && k >= 1, "rows must be >= 0 and both widths >= 1 (got %lld rows, %lld -> %lld)", m, k, n);
  if (m > kMaxSize || n > kMaxWidth || k > kMaxWidth) {
    set_error("more than 2^30 - 4096 rows or widths beyond 2^26 are not supported");
    return MIA_ERR_UNSUPPORTED;
  }
  MIA_REQUIRE(dtype_ok(dtype), "unknown dtype %d", dtype);
  return MIA_OK;
}

}  // namespace lin
}  // namespace mia

using namespace mia;

extern "C" {

size_t mia_linear_workspace_bytes(int64_t rows, int64_t in, int64_t out, int dtype) {
  if (rows <= lin::kFewRows || in <= 0 || out <= 0 || !nn::dtype_ok(dtype)) return 0;
  return lin::split_bytes(out, rows, in, nn::dtype_size(dtype), false);
}

int mia_linear(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* bias,
               int bias_dtype, const void* residual, int64_t residual_stride, int activation, int64_t rows, int64_t in,
               int64_t out, int dtype, void* y, void* preactivation, void* workspace, size_t workspace_bytes,
               void* stream) {
  const int rc = lin::check(rows, out, in, dtype);
  if (rc != MIA_OK) return rc;
  MIA_REQUIRE(activation >= MIA_ACT_NONE && activation <= MIA_ACT_RELU, "unknown activation %d", activation);
  MIA_REQUIRE(!bias || bias_dtype == dtype || bias_dtype == MIA_F32, "bias must be float32 or of the input's type");
  MIA_REQUIRE(x_stride >= 0 && weight_stride >= 0 && residual_stride >= 0, "rows must not run backwards");
  if (rows == 0) return MIA_OK;
  MIA_REQUIRE(x && weight && y, "null argument");
  const size_t need = mia_linear_workspace_bytes(rows, in, out, dtype);
  MIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && nn::aligned16(workspace)), "workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const lin::Epilogue e{bias, bias_dtype == MIA_F32, activation, residual, residual_stride, preactivation, y};
  const int done = nn::with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return lin::Ops<T>::forward({weight, weight_stride, x, x_stride, out, rows, in}, e, workspace, s);
  });
  if (done != MIA_OK) return done;
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

size_t mia_linear_backward_workspace_bytes(int64_t rows, int64_t in, int64_t out, int dtype, int activation) {
  if (rows <= 0 || in <= 0 || out <= 0 || !nn::dtype_ok(dtype)) return 0;
  const size_t es = nn::dtype_size(dtype);
  const size_t dz = activation == MIA_ACT_NONE ? 0 : nn::align256((size_t)rows * out * es);
  const size_t bias = nn::align256((size_t)lin::bias_groups(rows) * out * sizeof(float));
  const size_t dx = lin::split_bytes(in, rows, out, es, false), dw = lin::split_bytes(in, out, rows, es, true);
  return dz + bias + (dx > dw ? dx : dw);
}

int mia_linear_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* weight,
                        int64_t weight_stride, const void* preactivation, int64_t preactivation_stride, int activation,
                        int64_t rows, int64_t in, int64_t out, int dtype, void* dx, void* dweight, float* dbias,
                        void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = lin::check(rows, out, in, dtype);
  if (rc != MIA_OK) return rc;
  MIA_REQUIRE(activation >= MIA_ACT_NONE && activation <= MIA_ACT_RELU, "unknown activation %d", activation);
  MIA_REQUIRE(dy_stride >= 0 && x_stride >= 0 && weight_stride >= 0 && preactivation_stride >= 0,
              "rows must not run backwards");
  MIA_REQUIRE(rows == 0 || dy, "null argument");
  MIA_REQUIRE(rows == 0 || activation == MIA_ACT_NONE || preactivation,
              "the backward pass of an activation needs the values before it");
  MIA_REQUIRE(rows == 0 || (!dx || weight) && (!dweight || x), "null argument");
  const size_t need = mia_linear_backward_workspace_bytes(rows, in, out, dtype, activation);
  MIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && nn::aligned16(workspace)), "workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t es = nn::dtype_size(dtype);
  unsigned char* at = static_cast<unsigned char*>(workspace);
  const int done = nn::with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* g = static_cast<const T*>(dy);
    long long g_stride = dy_stride;
    const int groups = rows ? lin::bias_groups(rows) : 0;
    float* sums = nullptr;
    if (rows) {
      T* dz = nullptr;
      if (activation != MIA_ACT_NONE) {
        dz = reinterpret_cast<T*>(at);
        at += nn::align256((size_t)rows * out * es);
      }
      sums = reinterpret_cast<float*>(at);
      at += nn::align256((size_t)groups * out * sizeof(float));
      if (dz || dbias) {
        lin::Ops<T>::dz(dy, dy_stride, dz ? preactivation : nullptr, preactivation_stride, activation, rows, out, dz,
                        dbias ? sums : nullptr, groups, s);
      }
      if (dz) g = dz, g_stride = out;
    }
    if (dbias) {
      hipLaunchKernelGGL(nn::join_columns_kernel, dim3((unsigned)((out + 31) / 32)), dim3(1024), 0, s, sums, groups,
                         (int)out, dbias, static_cast<float*>(nullptr), (int)out);
    }
    lin::Epilogue e{nullptr, 0, MIA_ACT_NONE, nullptr, 0, nullptr, nullptr};
    if (dx && rows) {
      e.out = dx;
      const int r = lin::Ops<T>::input_gradient({weight, weight_stride, g, g_stride, in, rows, out}, e, at, s);
      if (r != MIA_OK) return r;
    }
    if (dweight) {
      e.out = dweight;
      const int r = lin::Ops<T>::weight_gradient({x, x_stride, g, g_stride, in, out, rows}, e, at, s);
      if (r != MIA_OK) return r;
    }
    return MIA_OK;
  });
  if (done != MIA_OK) return done;
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

}  // extern "C"
