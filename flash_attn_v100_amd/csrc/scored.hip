// Attention with modified scores (tanh cap, distance bias, document and prefix
// masks): C ABI, and the fp16 instantiations of the forward kernels
// (scored_kernels.h).
#include <math.h>

#include "scored_launch.h"

namespace fa {
namespace scored {

static void forward_fp16(const ScoredParams& p, bool vec, hipStream_t st) {
  by_shape_fp16<true>(p.D, vec, p.mods, [&](auto dp, auto dc, auto rows, auto mods) {
    launch_query<half_t, dp(), dc(), rows(), 0, mods()>(p, split_query(p, false), st);
  });
}

// Checks what both directions share and fills the parameters that do not
// depend on the direction; B or N of 0 is left to the caller.
static int fill(const char* fn, ScoredParams& p, int B, int H_Q, int H_KV, int N, int D, int max_d, int causal, float softcap,
                const float* slopes, const int32_t* ids, const int32_t* prefix) {
  if (B < 0 || N < 0 || H_Q <= 0 || H_KV <= 0 || D <= 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: bad sizes (B=%d H_Q=%d H_KV=%d N=%d D=%d)", fn, B, H_Q, H_KV, N, D);
  if (H_Q < H_KV || H_Q % H_KV != 0)
    return set_error(FA_ERR_INVALID_ARG, "%s: H_Q (%d) must be a multiple of H_KV (%d)", fn, H_Q, H_KV);
  if (D > max_d) return set_error(FA_ERR_UNSUPPORTED, "%s: D=%d exceeds %d", fn, D, max_d);
  // (the range keeps the polynomial's coefficients, up to (scale / softcap)^8, in fp32's)
  if (softcap != 0.0f && !(softcap >= 1e-2f && softcap <= 1e3f))
    return set_error(FA_ERR_INVALID_ARG, "%s: softcap must be 0 (none) or lie in [0.01, 1000]", fn);
  if (prefix != nullptr && !causal)
    return set_error(FA_ERR_INVALID_ARG, "%s: prefix lengths need a causal mask", fn);
  // quarter-block workgroups of the padded units (deal)
  if ((static_cast<long long>(B) * H_Q + 8 * kXcds * (H_Q / H_KV)) * (4LL * ceil_div(N, kBlockRows)) > 0x3fffffffLL)
    return set_error(FA_ERR_UNSUPPORTED, "%s: problem too large for one launch", fn);
  p.slopes = slopes;
  p.ids = ids;
  p.prefix = prefix;
  p.mods = (softcap > 0.0f ? kCap : 0) | (slopes ? kBias : 0) | (ids ? kDocs : 0);
  p.B = B; p.H_Q = H_Q; p.H_KV = H_KV; p.N = N; p.D = D; p.G = H_Q / H_KV;
  p.causal = causal ? 1 : 0;
  p.scale = 1.0f / sqrtf(static_cast<float>(D));
  p.scale_log2 = p.scale * kLog2e;
  p.cap_in = softcap > 0.0f ? p.scale / softcap : 0.0f;
  p.cap_log2 = softcap * kLog2e;
  if (softcap > 0.0f) {
    const double in = static_cast<double>(p.scale) / softcap, in2 = in * in;
    const double series[5] = {1.0, kTanhP0, kTanhP1, kTanhP2, kTanhP3};
    double power = static_cast<double>(p.scale) * 1.4426950408889634;
    for (int i = 0; i < 5; ++i, power *= in2) p.cap_poly[i] = static_cast<float>(series[i] * power);
    p.cap_near = static_cast<float>(kTanhMax / in);
    p.cap_slope = 1.0f / (p.cap_log2 * p.cap_log2);
  }
  return FA_OK;
}

static int forward(const char* fn, bool fp32, const void* q, const void* k, const void* v, void* o, float* lse, int B, int H_Q,
                   int H_KV, int N, int D, int causal, float softcap, const float* slopes, const int32_t* ids,
                   const int32_t* prefix, void* stream) {
  ScoredParams p = {};
  if (int rc = fill(fn, p, B, H_Q, H_KV, N, D, fp32 ? 128 : 256, causal, softcap, slopes, ids, prefix)) return rc;
  if (B == 0 || N == 0) return FA_OK;
  if (!q || !k || !v || !o) return set_error(FA_ERR_INVALID_ARG, "%s: null tensor pointer", fn);
  p.q = q; p.k = k; p.v = v; p.out = o; p.lse = lse;
  const bool vec = aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (fp32) forward_fp32(p, vec, st);
  else forward_fp16(p, vec, st);
  return check_launch(fn);
}

static int backward(const char* fn, bool fp32, const void* dout, const void* q, const void* k, const void* v, const void* out,
                    const float* lse, void* dq, void* dk, void* dv, int B, int H_Q, int H_KV, int N, int D, int causal,
                    float softcap, const float* slopes, const int32_t* ids, const int32_t* prefix, void* workspace,
                    size_t workspace_bytes, void* stream) {
  ScoredParams p = {};
  if (int rc = fill(fn, p, B, H_Q, H_KV, N, D, 128, causal, softcap, slopes, ids, prefix)) return rc;
  if (B == 0 || N == 0) return FA_OK;
  if (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv)
    return set_error(FA_ERR_INVALID_ARG, "%s: null tensor pointer", fn);
  const size_t need = fa_scored_backward_workspace_size(B, H_Q, N);
  if (!workspace || workspace_bytes < need)
    return set_error(FA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", fn, need,
                     workspace ? workspace_bytes : static_cast<size_t>(0));
  p.q = q; p.k = k; p.v = v; p.o = out; p.dout = dout;
  p.out = dq; p.dk = dk; p.dv = dv;
  p.lse = const_cast<float*>(lse);
  p.delta = static_cast<float*>(workspace);
  p.row_lse = p.delta + static_cast<size_t>(B) * H_Q * N;
  const bool vec = aligned16(dout) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(dq) &&
                   aligned16(dk) && aligned16(dv);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (fp32) backward_fp32(p, vec, st);
  else backward_fp16(p, vec, st);
  return check_launch(fn);
}

}  // namespace scored
}  // namespace fa

extern "C" int fa_scored_fp16(const void* q, const void* k, const void* v, void* o, float* lse, int B, int H_Q, int H_KV, int N,
                              int D, int causal, float softcap, const float* slopes, const int32_t* doc_ids,
                              const int32_t* prefix_lens, void* stream) {
  return fa::scored::forward("fa_scored_fp16", false, q, k, v, o, lse, B, H_Q, H_KV, N, D, causal, softcap, slopes, doc_ids,
                             prefix_lens, stream);
}

extern "C" int fa_scored_fp32(const void* q, const void* k, const void* v, void* o, float* lse, int B, int H_Q, int H_KV, int N,
                              int D, int causal, float softcap, const float* slopes, const int32_t* doc_ids,
                              const int32_t* prefix_lens, void* stream) {
  return fa::scored::forward("fa_scored_fp32", true, q, k, v, o, lse, B, H_Q, H_KV, N, D, causal, softcap, slopes, doc_ids,
                             prefix_lens, stream);
}

extern "C" size_t fa_scored_backward_workspace_size(int B, int H_Q, int N) {
  if (B <= 0 || H_Q <= 0 || N <= 0) return 0;
  return 2 * static_cast<size_t>(B) * H_Q * N * sizeof(float);
}

extern "C" int fa_scored_backward_fp16(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                       const float* lse, void* dq, void* dk, void* dv, int B, int H_Q, int H_KV, int N, int D,
                                       int causal, float softcap, const float* slopes, const int32_t* doc_ids,
                                       const int32_t* prefix_lens, void* workspace, size_t workspace_bytes, void* stream) {
  return fa::scored::backward("fa_scored_backward_fp16", false, dout, q, k, v, out, lse, dq, dk, dv, B, H_Q, H_KV, N, D, causal,
                              softcap, slopes, doc_ids, prefix_lens, workspace, workspace_bytes, stream);
}

extern "C" int fa_scored_backward_fp32(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                       const float* lse, void* dq, void* dk, void* dv, int B, int H_Q, int H_KV, int N, int D,
                                       int causal, float softcap, const float* slopes, const int32_t* doc_ids,
                                       const int32_t* prefix_lens, void* workspace, size_t workspace_bytes, void* stream) {
  return fa::scored::backward("fa_scored_backward_fp32", true, dout, q, k, v, out, lse, dq, dk, dv, B, H_Q, H_KV, N, D, causal,
                              softcap, slopes, doc_ids, prefix_lens, workspace, workspace_bytes, stream);
}
