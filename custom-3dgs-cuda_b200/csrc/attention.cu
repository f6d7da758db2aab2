// Cross attention: the C entry points, and kernels with one warp for each row.
//
//   S = scale q k^T,  P = softmax over the keys that length and mask leave,  O = P v,
//   lse = log sum exp S.
// Backward: delta = rowsum(dO o O), dv = P^T dO, dS = P o (dO v^T - delta),
// dq = scale dS k, dk = scale dS^T q; the query heads that share a key head are summed.
// A row that keeps no key has O = 0, lse = -inf and no gradient.
#include <cmath>

#include "attention.cuh"
#include "capi_internal.h"

namespace gs {

constexpr int kRowWarps = 8;

// One warp: delta of a query row, then dq over its keys.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) attention_dq_row_kernel(AttentionParams p) {
  const int lane = threadIdx.x % 32;
  const long long row = (long long)blockIdx.x * kRowWarps + threadIdx.x / 32;
  if (row >= (long long)p.B * p.Hq * p.Lq) return;
  const int i = (int)(row % p.Lq), h = (int)(row / p.Lq % p.Hq), b = (int)(row / p.Lq / p.Hq);
  const int hk = h / (p.Hq / p.Hkv);
  const float lse = p.lse[row];
  const int n = lse == -INFINITY ? 0 : key_count(p, b);
  float qv[4], g[4], dq[4] = {}, delta = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 32 * k;
    const bool in = d < p.D;
    qv[k] = in ? to_f32<T>(p.q.at<T>(b, i, h)[d]) : 0.0f;
    g[k] = in ? to_f32<T>(p.dout.at<T>(b, i, h)[d]) : 0.0f;
    if (in) delta = fmaf(g[k], to_f32<T>(p.out.at<T>(b, i, h)[d]), delta);
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) delta += __shfl_xor_sync(~0u, delta, w);
  if (lane == 0) p.delta[row] = delta;
  for (int j = 0; j < n; ++j) {
    if (!keeps(p, b, h, i, j)) continue;
    const T* kr = p.k.at<T>(b, j, hk);
    const T* vr = p.v.at<T>(b, j, hk);
    float s = 0.0f, dp = 0.0f, kv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int d = lane + 32 * k;
      kv[k] = d < p.D ? to_f32<T>(kr[d]) : 0.0f;
      s = fmaf(qv[k], kv[k], s);
      dp = fmaf(g[k], d < p.D ? to_f32<T>(vr[d]) : 0.0f, dp);
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) {
      s += __shfl_xor_sync(~0u, s, w);
      dp += __shfl_xor_sync(~0u, dp, w);
    }
    const float ds = expf(s * p.scale - lse) * (dp - delta);
#pragma unroll
    for (int k = 0; k < 4; ++k) dq[k] = fmaf(ds, kv[k], dq[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 32 * k < p.D)
      p.dq.at<T>(b, i, h)[lane + 32 * k] = from_f32<T>(dq[k] * p.scale);
}

// One warp owns one key row and walks over the queries of every head that shares it.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) attention_dkv_row_kernel(AttentionParams p) {
  const int lane = threadIdx.x % 32;
  const long long row = (long long)blockIdx.x * kRowWarps + threadIdx.x / 32;
  if (row >= (long long)p.B * p.Hkv * p.Lk) return;
  const int j = (int)(row % p.Lk), hk = (int)(row / p.Lk % p.Hkv), b = (int)(row / p.Lk / p.Hkv);
  const int shared = p.Hq / p.Hkv;
  float kv[4], vv[4], dk[4] = {}, dv[4] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 32 * k;
    kv[k] = d < p.D ? to_f32<T>(p.k.at<T>(b, j, hk)[d]) : 0.0f;
    vv[k] = d < p.D ? to_f32<T>(p.v.at<T>(b, j, hk)[d]) : 0.0f;
  }
  if (j < key_count(p, b))
    for (int h = hk * shared; h < (hk + 1) * shared; ++h)
      for (int i = 0; i < p.Lq; ++i) {
        const long long at = ((long long)b * p.Hq + h) * p.Lq + i;
        const float lse = p.lse[at];
        if (lse == -INFINITY || !keeps(p, b, h, i, j)) continue;
        const T* qr = p.q.at<T>(b, i, h);
        const T* gr = p.dout.at<T>(b, i, h);
        float s = 0.0f, dp = 0.0f, qv[4], g[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int d = lane + 32 * k;
          qv[k] = d < p.D ? to_f32<T>(qr[d]) : 0.0f;
          g[k] = d < p.D ? to_f32<T>(gr[d]) : 0.0f;
          s = fmaf(qv[k], kv[k], s);
          dp = fmaf(g[k], vv[k], dp);
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) {
          s += __shfl_xor_sync(~0u, s, w);
          dp += __shfl_xor_sync(~0u, dp, w);
        }
        const float pr = expf(s * p.scale - lse);
        const float ds = pr * (dp - p.delta[at]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dk[k] = fmaf(ds, qv[k], dk[k]);
          dv[k] = fmaf(pr, g[k], dv[k]);
        }
      }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 32 * k;
    if (d < p.D) {
      p.dk.at<T>(b, j, hk)[d] = from_f32<T>(dk[k] * p.scale);
      p.dv.at<T>(b, j, hk)[d] = from_f32<T>(dv[k]);
    }
  }
}

// The checks that forward and backward share; "" or what is wrong.
static const char* attention_fault(const gs_attention_args& a) {
  if (a.dtype != GS_FP16 && a.dtype != GS_BF16) return "dtype must be GS_FP16 or GS_BF16";
  if (a.B < 0 || a.Lq < 0 || a.Lk < 0 || a.Hq < 0 || a.Hkv < 0) return "sizes must be non-negative";
  if (a.D < 8 || a.D > 128 || a.D % 8) return "the head size must be a multiple of 8 up to 128";
  if (a.Hkv == 0 ? a.Hq != 0 : a.Hq % a.Hkv) return "the key heads must divide the query heads";
  if (!std::isfinite(a.scale)) return "the scale must be finite";
  if ((long long)a.B * a.Hq * a.Lq >= (1ll << 31) || (long long)a.B * a.Hkv * a.Lk >= (1ll << 31))
    return "more than 2^31 rows";
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
  GS_REQUIRE(workspace_bytes >= gs_cross_attention_workspace_size(a), "workspace too small");
  GS_REQUIRE(workspace || !gs_cross_attention_workspace_size(a), "null pointer");
  return attention_is_single(*a) ? attention_single(*a, workspace, (cudaStream_t)stream)
                                 : attention_forward(*a, workspace, (cudaStream_t)stream);
  GS_API_END();
}

extern "C" size_t gs_cross_attention_backward_workspace_size(const gs_attention_args* a) {
  if (!a || *attention_fault(*a)) return 0;
  return (size_t)a->B * a->Hq * a->Lq * sizeof(float);
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
  GS_REQUIRE(workspace_bytes >= gs_cross_attention_backward_workspace_size(a),
             "workspace too small");
  GS_REQUIRE(no_queries || workspace, "null pointer");
  AttentionParams p = attention_params(*a);
  p.dout = TokenView(*dout), p.dq = TokenView(*dq), p.dk = TokenView(*dk), p.dv = TokenView(*dv);
  p.delta = static_cast<float*>(workspace);
  const cudaStream_t s = (cudaStream_t)stream;
  const auto blocks = [](long long rows) { return (unsigned)((rows + kRowWarps - 1) / kRowWarps); };
  if (!no_queries) {
    const unsigned n = blocks((long long)p.B * p.Hq * p.Lq);
    if (a->dtype == GS_FP16)
      attention_dq_row_kernel<__half><<<n, kRowWarps * 32, 0, s>>>(p);
    else
      attention_dq_row_kernel<__nv_bfloat16><<<n, kRowWarps * 32, 0, s>>>(p);
    GS_CHECK_LAUNCH();
  }
  if (!no_keys) {
    const unsigned n = blocks((long long)p.B * p.Hkv * p.Lk);
    if (a->dtype == GS_FP16)
      attention_dkv_row_kernel<__half><<<n, kRowWarps * 32, 0, s>>>(p);
    else
      attention_dkv_row_kernel<__nv_bfloat16><<<n, kRowWarps * 32, 0, s>>>(p);
    GS_CHECK_LAUNCH();
  }
  return GS_OK;
  GS_API_END();
}
