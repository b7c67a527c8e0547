// Key/value cache held in 4 bits, in pages (kv_cache.cu): written, read back, attended to.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mdl {

// The cache. Row r's token at position p lives in page table[r, p / page], slot p % page:
//   codes  [num_pages, G, 2, page, hd / 2] uint8: K (0) and V (1); element 2i of a head's row in
//          the low half of byte i, element 2i + 1 in the high half, each c + 8 for c = -7 .. 7
//   scales [num_pages, G, page, 2] bf16: one a token, head and K|V; the value is scale * c
// page is a power of two of at least 16, hd is 32 or 64.
struct KvCache {
  uint8_t* codes = nullptr;
  __nv_bfloat16* scales = nullptr;
  const int* table = nullptr;  // [R, max_pages] page of each run of `page` positions
  int* lengths = nullptr;      // [R] tokens held
  int R = 0, G = 0, hd = 0, page_shift = 0, max_pages = 0, num_pages = 0;
  int* err = nullptr;          // device error word
};

// Tokens kstart[i] .. T-1 of source row i go to positions start[i] .. of cache row rows[i]
// (append: start == nullptr, from the row's present length); its length becomes the end of
// what was written. Positions past the row's capacity are not written (MDL_ERR_CAPACITY);
// a row or page outside the cache is skipped (MDL_ERR_BAD_INDEX).
struct KvWriteArgs {
  KvCache c;
  const __nv_bfloat16* k = nullptr;  // [n, T, G * hd], last dimension dense
  const __nv_bfloat16* v = nullptr;
  long long k_sb = 0, k_st = 0, v_sb = 0, v_st = 0;  // batch and token strides (elements, multiples of 8)
  const int* rows = nullptr;    // [n] cache rows, or nullptr: row i
  const int* start = nullptr;   // [n], or nullptr: append
  const int* kstart = nullptr;  // [n] first valid token, or nullptr: 0
  int n = 0, T = 0;
};

// out_k, out_v [n, count, G * hd] = the values at positions start[i] .. of row rows[i]; zero
// past the row's length.
struct KvReadArgs {
  KvCache c;
  void* out_k = nullptr;
  void* out_v = nullptr;
  const int* rows = nullptr;
  const int* start = nullptr;  // or nullptr: 0
  int n = 0, count = 0;
  bool fp32 = false;           // else bf16
};

// Attention of a few queries a batch row over its cache row (see kv_attend in kv_cache.cu).
struct KvAttendArgs {
  KvCache c;
  const __nv_bfloat16* q = nullptr;   // [B, N, H * hd]
  const __nv_bfloat16* kn = nullptr;  // [B, N, G * hd] fresh keys, or nullptr
  const __nv_bfloat16* vn = nullptr;
  long long q_sb = 0, q_sn = 0, kn_sb = 0, kn_sn = 0, vn_sb = 0, vn_sn = 0;  // multiples of 8
  const int* rows = nullptr;          // [B] cache row of a batch row, or nullptr: row b
  __nv_bfloat16* out = nullptr;       // [B, N, H * hd]
  float* partial = nullptr;           // workspace of kv_attend_workspace() floats
  int B = 0, N = 0, H = 0, window = 0, sinks = 0;
  float scale = 1.f;
};

cudaError_t kv_write(const KvWriteArgs& a, cudaStream_t stream, int* launches);
cudaError_t kv_read(const KvReadArgs& a, cudaStream_t stream);
long long kv_attend_workspace(const KvAttendArgs& a);
cudaError_t kv_attend(const KvAttendArgs& a, cudaStream_t stream, int* launches);

}  // namespace mdl
