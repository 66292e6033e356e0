// C entry points of attention (kernels: attention_kernels.h, one translation unit per element type).
#include "attention_kernels.h"

namespace mia {
namespace att {
constexpr long long kMaxRows = 1LL << 30;

static int check(const mia_attention_desc* d) {
  MIA_REQUIRE(d, "null argument");
  MIA_REQUIRE(dtype_ok(d->dtype), "unknown dtype %d", d->dtype);
  MIA_REQUIRE(d->batch >= 0 && d->queries >= 0 && d->keys >= 0, "sizes must not be negative");
  MIA_REQUIRE(d->heads >= 1 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0,
              "heads must be a multiple of kv_heads (got %d, %d)", d->heads, d->kv_heads);
  MIA_REQUIRE(d->dim >= 1, "dim must be positive (got %d)", d->dim);
  // (exponents are taken to base 2: scale / ln 2 has to be finite as well)
  MIA_REQUIRE(d->scale > 0.0f && d->scale * kLog2e < __builtin_huge_valf(), "scale must be positive and below 2.3e38");
  for (const int64_t* s = d->stride_q; s < d->stride_q + 3; ++s) MIA_REQUIRE(*s >= 0, "strides must not be negative");
  for (const int64_t* s = d->stride_k; s < d->stride_k + 3; ++s) MIA_REQUIRE(*s >= 0, "strides must not be negative");
  for (const int64_t* s = d->stride_v; s < d->stride_v + 3; ++s) MIA_REQUIRE(*s >= 0, "strides must not be negative");
  if (d->dim > 128) {
    set_error("head dimensions beyond 128 are not supported (got %d)", d->dim);
    return MIA_ERR_UNSUPPORTED;
  }
  if (d->queries > kMaxRows || d->keys > kMaxRows || d->batch > kMaxRows || d->heads > (1 << 20) ||
      (long long)d->batch * d->heads >= (1LL << 31) || (long long)d->batch * d->heads * d->queries >= kMaxRows * 8 ||
      (long long)d->batch * d->heads * ((d->queries + 63) / 64) >= (1LL << 31) ||
      (long long)d->batch * d->heads * ((d->keys + 63) / 64) >= (1LL << 31)) {
    set_error("too many rows for one call");
    return MIA_ERR_UNSUPPORTED;
  }
  return MIA_OK;
}
static View view(const void* p, const int64_t* s) { return {p, s[0], s[1], s[2]}; }
static Args args(const mia_attention_desc* d, const void* q, const void* k, const void* v, const int* lengths) {
  Args a{};
  a.q = view(q, d->stride_q), a.k = view(k, d->stride_k), a.v = view(v, d->stride_v);
  a.lengths = lengths;
  a.batch = (int)d->batch, a.sq = (int)d->queries, a.sk = (int)d->keys;
  a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim;
  a.causal = d->causal, a.scale = d->scale;
  return a;
}
}  // namespace att
}  // namespace mia

using namespace mia;

extern "C" {

size_t mia_attention_workspace_bytes(const mia_attention_desc* d) {
  if (att::check(d) != MIA_OK || d->batch == 0 || d->queries == 0) return 0;
  const att::Plan p = att::plan_forward(d->batch, d->queries, d->keys, d->heads, d->kv_heads);
  if (p.splits == 1) return 0;
  return (size_t)p.splits * d->batch * d->heads * d->queries * (d->dim + 2) * sizeof(float);
}

int mia_attention(const mia_attention_desc* d, const void* q, const void* k, const void* v, const int32_t* key_lengths,
                  void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = att::check(d);
  if (rc != MIA_OK) return rc;
  if (d->batch == 0 || d->queries == 0) return MIA_OK;
  MIA_REQUIRE(q && out && (d->keys == 0 || (k && v)), "null argument");
  const size_t need = mia_attention_workspace_bytes(d);
  MIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && nn::aligned16(workspace)), "workspace too small");
  att::Args a = att::args(d, q, k, v, key_lengths);
  a.o0 = out, a.lse = lse, a.partial = static_cast<float*>(workspace);
  const int done = nn::with_dtype(d->dtype, [&](auto t) {
    return att::Ops<decltype(t)>::forward(a, static_cast<hipStream_t>(stream));
  });
  if (done != MIA_OK) return done;
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

size_t mia_attention_backward_workspace_bytes(const mia_attention_desc* d) {
  if (att::check(d) != MIA_OK) return 0;
  return att::gradient_bytes(d->batch, d->queries, d->keys, d->heads, d->kv_heads, d->dim, d->dtype);
}

int mia_attention_backward(const mia_attention_desc* d, const void* dout, const int64_t* stride_dout, const void* q,
                           const void* k, const void* v, const void* out, const int64_t* stride_out, const float* lse,
                           const int32_t* key_lengths, void* dq, void* dk, void* dv, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const int rc = att::check(d);
  if (rc != MIA_OK) return rc;
  MIA_REQUIRE(stride_dout && stride_out, "null argument");
  for (int i = 0; i < 3; ++i) MIA_REQUIRE(stride_dout[i] >= 0 && stride_out[i] >= 0, "strides must not be negative");
  if (d->batch == 0) return MIA_OK;
  MIA_REQUIRE(d->queries == 0 || (dout && q && out && lse && dq), "null argument");
  MIA_REQUIRE(d->keys == 0 || (k && v && dk && dv), "null argument");
  const size_t need = mia_attention_backward_workspace_bytes(d);
  MIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && nn::aligned16(workspace)), "workspace too small");
  att::Args a = att::args(d, q, k, v, key_lengths);
  a.dout = att::view(dout, stride_dout), a.out = att::view(out, stride_out);
  a.lse = const_cast<float*>(lse);
  const int done = nn::with_dtype(d->dtype, [&](auto t) {
    return att::Ops<decltype(t)>::backward(a, static_cast<float*>(workspace), dq, dk, dv, static_cast<hipStream_t>(stream));
  });
  if (done != MIA_OK) return done;
  MIA_CHECK_HIP(hipGetLastError());
  return MIA_OK;
}

}  // extern "C"
