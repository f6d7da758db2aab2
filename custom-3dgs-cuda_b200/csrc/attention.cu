// Cross attention: the C entry points, their checks, and the choice between the kernels.
//
//   S = scale q k^T,  P = softmax over the keys that length and mask leave,  O = P v,
//   lse = log sum exp S;  the gradients are in attention_backward.cu.
// A row that keeps no key has O = 0, lse = -inf and no gradient.
#include <cmath>

#include "attention.cuh"
#include "capi_internal.h"

namespace gs {

// Rows of queries (of all items and query heads) and of keys (items and key heads), at most: indexes of
// rows are 32-bit, and a tile, or a warp's next chunks, may reach this far past the last row.
static constexpr long long kMaxRows = (1ll << 31) - 1024;

// The checks that forward and backward share; "" or what is wrong.
static const char* attention_fault(const gs_attention_args& a) {
  if (a.dtype != GS_FP16 && a.dtype != GS_BF16) return "dtype must be GS_FP16 or GS_BF16";
  if (a.B < 0 || a.Lq < 0 || a.Lk < 0 || a.Hq < 0 || a.Hkv < 0) return "sizes must be non-negative";
  if (a.D < 8 || a.D > 128 || a.D % 8) return "the head size must be a multiple of 8 up to 128";
  if (a.Hkv == 0 ? a.Hq != 0 : a.Hq % a.Hkv) return "the key heads must divide the query heads";
  if (!std::isfinite(a.scale)) return "the scale must be finite";
  // two factors fit 64 bits; all three may not
  const auto many = [&](int heads, int tokens) {
    return tokens > 0 && (long long)a.B * heads > kMaxRows / tokens;
  };
  if (many(a.Hq, a.Lq) || many(a.Hkv, a.Lk)) return "more than 2^31 - 1024 rows";
  return "";
}

static const char* view_fault(const gs_token_view& v, int tokens, int heads) {
  if (tokens == 0 || heads == 0) return "";
  if (!v.data) return "null pointer";
  if (reinterpret_cast<uintptr_t>(v.data) % 16 || v.batch_stride % 8 || v.token_stride % 8 ||
      v.head_stride % 8)
    return "tensors must start on 16-byte boundaries with strides of multiples of 8 elements";
  if ((tokens > 1 && v.token_stride <= 0) || (heads > 1 && v.head_stride <= 0) || v.batch_stride < 0)
    return "strides must be positive (that of the batch may be 0)";
  return "";
}

// The workspace holds bits, sums and parts that are read 16 bytes at a time.
static const char* workspace_fault(const void* workspace, size_t bytes, size_t needed) {
  if (bytes < needed) return "workspace too small";
  if (needed && !workspace) return "null pointer";
  if (needed && reinterpret_cast<uintptr_t>(workspace) % 16)
    return "the workspace must start on a 16-byte boundary";
  return "";
}

AttentionParams attention_params(const gs_attention_args& a) {
  AttentionParams p{};
  p.B = a.B, p.Lq = a.Lq, p.Lk = a.Lk, p.Hq = a.Hq, p.Hkv = a.Hkv, p.D = a.D;
  p.scale = a.scale;
  p.q = TokenView(a.q), p.k = TokenView(a.k), p.v = TokenView(a.v), p.out = TokenView(a.out);
  p.lengths = a.lengths;
  p.mask = a.mask;
  p.mask_b = a.mask_batch_stride, p.mask_h = a.mask_head_stride, p.mask_q = a.mask_query_stride;
  p.lse = a.lse;
  return p;
}

}  // namespace gs

using namespace gs;

extern "C" size_t gs_cross_attention_workspace_size(const gs_attention_args* a) {
  if (!a || *attention_fault(*a) || a->B == 0 || a->Hq == 0 || a->Lq == 0) return 0;
  return attention_is_single(*a) ? attention_single_workspace(*a) : attention_forward_workspace(*a);
}

extern "C" int gs_cross_attention_forward(const gs_attention_args* a, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(a, "null pointer");
  const char* fault = attention_fault(*a);
  GS_REQUIRE(!*fault, fault);
  if (a->B == 0 || a->Hq == 0 || a->Lq == 0) return GS_OK;
  for (const gs_token_view* v : {&a->q, &a->out, &a->k, &a->v}) {
    const bool keys = v == &a->k || v == &a->v;
    fault = view_fault(*v, keys ? a->Lk : a->Lq, keys ? a->Hkv : a->Hq);
    GS_REQUIRE(!*fault, fault);
  }
  fault = workspace_fault(workspace, workspace_bytes, gs_cross_attention_workspace_size(a));
  GS_REQUIRE(!*fault, fault);
  return attention_is_single(*a) ? attention_single(*a, workspace, (cudaStream_t)stream)
                                 : attention_forward(*a, workspace, (cudaStream_t)stream);
  GS_API_END();
}

extern "C" size_t gs_cross_attention_backward_workspace_size(const gs_attention_args* a) {
  if (!a || *attention_fault(*a)) return 0;
  return attention_backward_workspace(*a);
}

extern "C" int gs_cross_attention_backward(const gs_attention_args* a, const gs_token_view* dout,
                                           const gs_token_view* dq, const gs_token_view* dk,
                                           const gs_token_view* dv, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(a && dout && dq && dk && dv, "null pointer");
  const char* fault = attention_fault(*a);
  GS_REQUIRE(!*fault, fault);
  const bool no_queries = a->B == 0 || a->Hq == 0 || a->Lq == 0;
  const bool no_keys = a->B == 0 || a->Hkv == 0 || a->Lk == 0;
  if (no_queries && no_keys) return GS_OK;
  for (const gs_token_view* v : {&a->q, &a->out, dout, dq}) {
    fault = view_fault(*v, no_queries ? 0 : a->Lq, a->Hq);
    GS_REQUIRE(!*fault, fault);
  }
  for (const gs_token_view* v : {&a->k, &a->v, dk, dv}) {
    fault = view_fault(*v, no_keys ? 0 : a->Lk, a->Hkv);
    GS_REQUIRE(!*fault, fault);
  }
  GS_REQUIRE(no_queries || a->lse, "the backward needs the forward's lse");
  fault = workspace_fault(workspace, workspace_bytes, gs_cross_attention_backward_workspace_size(a));
  GS_REQUIRE(!*fault, fault);
  return attention_backward(*a, *dout, *dq, *dk, *dv, workspace, (cudaStream_t)stream);
  GS_API_END();
}
