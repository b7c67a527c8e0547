// Sliding-window attention with always-visible first tokens (window_attn.cu).
#pragma once
#include <cuda_runtime.h>

namespace mdl {

// Attention of a query suffix over its own token sequence, forward and backward:
//   qkv  [B, Lk, (H + 2 G) * hd] bf16: per token H query heads | G key heads | G value heads;
//        last dimension dense, row stride ld and batch stride sb (elements, multiples of 8)
//   query heads h .. of group h / (H / G) share key head h / (H / G)
//   the queries are the last Lq tokens; with kst = kstart[b], token row p sees key j iff
//   kst <= j <= p and (p - j < window or j - kst < sinks)
//   out  [B, Lq, H * hd] bf16; rows before kst see nothing and are zero
//   out_lo like out: what rounding took off it (out + out_lo holds 16 significant bits); the
//        backward forms D = rowsum(dout * out) from both, so that the rounding of out does not
//        reach the gradient. May be null in a forward that no backward follows.
//   lse  [B, H, Lq] fp32: base-2 log-sum-exp of the scaled scores (+inf: a row that sees nothing)
// Backward: dqkv [B, Lk, (H + 2 G) * hd] bf16 contiguous, every element written; workspace
// dsum fp32 [B, H, Lq]. No atomics: results do not depend on the order of execution.
// Tokens before kst are never read, nor the queries of tokens that are not queries.
struct WindowAttnArgs {
  const void* qkv = nullptr;
  long long ld = 0, sb = 0;
  const int* kstart = nullptr;  // int32 [B]
  void* out = nullptr;
  void* out_lo = nullptr;
  float* lse = nullptr;
  const void* dout = nullptr;   // bf16 [B, Lq, H * hd] contiguous
  void* dqkv = nullptr;
  float* dsum = nullptr;
  float* partial = nullptr;     // window_attn_workspace() floats
  int B = 0, H = 0, G = 0, Lk = 0, Lq = 0, hd = 0, window = 0, sinks = 0;
  float scale = 1.f;
  int* err = nullptr;
};

// Floats of workspace that the backward needs (0 unless the sinks' tiles are cut into parts).
long long window_attn_workspace(const WindowAttnArgs& a);
cudaError_t window_attn_fwd(const WindowAttnArgs& a, cudaStream_t stream);
cudaError_t window_attn_bwd(const WindowAttnArgs& a, cudaStream_t stream);

}  // namespace mdl
