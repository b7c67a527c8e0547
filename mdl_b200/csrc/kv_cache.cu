// Key/value cache of 4 bits a value in pages: quantising as it is written, reading back, and
// the attention of single tokens or candidates over it. Layout: kv_cache.h.
//
// A token's row of hd values of one head (K or V) is held as x ~ s * c with
//   s = bf16(max |x| / 7),  c = clamp(rint(x / s), -7, 7)   (s = 0: c = 0)
// and a row that holds an infinity or a NaN gets s = NaN, so it reads back as NaN. bf16 is
// enough for s: the rounding moves the largest quotient from 7 to at most 7.03.
#include "kv_cache.h"

#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace mdl {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// Pairs of fp32, one instruction for two.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ int row_of(const KvCache& c, const int* rows, int i) {
  const int r = rows != nullptr ? rows[i] : i;
  if (static_cast<unsigned>(r) < static_cast<unsigned>(c.R)) return r;
  record_error(c.err, MDL_ERR_BAD_INDEX);
  return -1;
}

// Page of position p of row r (p within the capacity), or -1.
__device__ __forceinline__ int page_of(const KvCache& c, int r, int p) {
  const int pg = c.table[static_cast<long long>(r) * c.max_pages + (p >> c.page_shift)];
  if (static_cast<unsigned>(pg) < static_cast<unsigned>(c.num_pages)) return pg;
  record_error(c.err, MDL_ERR_BAD_INDEX);
  return -1;
}

// Scales of K (low half) and V (high half) of position p in page pg, as one word.
__device__ __forceinline__ long long scale_index(const KvCache& c, int pg, int g, int p) {
  return ((static_cast<long long>(pg) * c.G + g) << c.page_shift) + (p & ((1 << c.page_shift) - 1));
}

// First slot row of (page, head, K|V) in the codes, hd / 2 bytes each.
__device__ __forceinline__ long long slot_base(const KvCache& c, int pg, int g, int kv) {
  return ((static_cast<long long>(pg) * c.G + g) * 2 + kv) << c.page_shift;
}

// ============================================================================ write
// A lane holds 16 values of a row, hd / 16 lanes the row: wide loads, a maximum of one or two
// shuffles, and a store of 8 bytes. Bound by memory: 256 rows of up to 2,000 tokens, 8 heads of 32, K
// and V: 100 us, 5.7 TB/s read and written (434,000 tokens of histories of unequal length).
//
// c = rint(x / s) without a division: x / s of two bf16 numbers is either a tie (an odd
// multiple of 1/2) or at least 1/1020 away from one, and |x / s| <= 7.03 (up to 8-bit
// significands X, S: |X 2^e / S - (2k+1)/2| is a multiple of 1 / (2S), or of 1 / (4S) for the
// tie 1/2). x * (1/s) + 1.5 * 2^12 rounds to a multiple of 2^-11, which moves it by 2^-12 at
// most: ties become exact, nothing else reaches one. Adding 1.5 * 2^23 + 8 - 1.5 * 2^12 then
// rounds to whole numbers, ties to even, and leaves c + 8 in the low bits. In the same way
// top / 7 (8 bits over 7) stays 2^-12 of itself away from where bf16 rounding changes, so that a
// multiplication by 1/7 gives the same s. Scales near the subnormal range take the division.
template <int HD>
__device__ __forceinline__ uint2 quantise16(const uint4 x0, const uint4 x1, uint16_t& scale_bits) {
  const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  // |x| as 15-bit integers: ordered like the values, infinities and NaN on top
  uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
#pragma unroll
  for (int o = 1; o < HD / 16; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t top = max(m & 0xFFFFu, m >> 16);
  const float largest = __uint_as_float(top << 16);
  uint32_t word[2] = {0x88888888u, 0x88888888u};  // c = 0
  if (top >= 0x7F80u) {
    scale_bits = 0x7FFFu;  // NaN
  } else if (top >= 0x0800u) {  // 2^-111
    const __nv_bfloat16 s16 = __float2bfloat16_rn(largest * (1.f / 7.f));
    scale_bits = __bfloat16_as_ushort(s16);
    const float inv = __fdividef(1.f, __bfloat162float(s16));
    constexpr float SNAP = 6144.f, ROUND = 12582912.f + 8.f - 6144.f;  // 1.5 * 2^12, to 1.5 * 2^23 + 8
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t sum = 0;  // the exponent bits shifted in add up to a constant
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t u = w[4 * h + (i >> 1)];
        const F2 q = add2(fma2({bf16_lo(u), bf16_hi(u)}, {inv, inv}, {SNAP, SNAP}), {ROUND, ROUND});
        sum += __float_as_uint(q.x) << (4 * i);
        sum += __float_as_uint(q.y) << (4 * i + 4);
      }
      constexpr uint32_t BASE = 0x4B400000u;  // 1.5 * 2^23
      constexpr uint32_t CONST = BASE * 0x11111111u;
      word[h] = sum - CONST;
    }
  } else {
    const __nv_bfloat16 s16 = __float2bfloat16_rn(largest / 7.f);
    scale_bits = __bfloat16_as_ushort(s16);
    const float s = __bfloat162float(s16);
    if (s > 0.f) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        word[h] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t u = w[4 * h + (i >> 1)];
          const float v = (i & 1) ? bf16_hi(u) : bf16_lo(u);
          const int c = static_cast<int>(fminf(fmaxf(rintf(v / s), -7.f), 7.f));
          word[h] |= static_cast<uint32_t>(c + 8) << (4 * i);
        }
      }
    }
  }
  return make_uint2(word[0], word[1]);
}

// One block: a run of `chunk` tokens of one source row, every head, K and V. A unit = the row
// of one token and head (hd / 16 lanes). Long runs number the units token-fastest, so that a
// warp reads whole sectors of neighbouring tokens and writes one dense run of a page; single
// tokens number them head-fastest, so that a warp reads densely.
template <int HD>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(KvWriteArgs a, int chunk, int chunks) {
  constexpr int LPU = HD / 16;
  const KvCache& c = a.c;
  const int i = blockIdx.x / chunks;
  const int r = row_of(c, a.rows, i);
  if (r < 0) return;
  const int cap = c.max_pages << c.page_shift;
  const int first = a.kstart != nullptr ? min(max(a.kstart[i], 0), a.T) : 0;
  const int start = a.start != nullptr ? a.start[i] : c.lengths[r];
  if (start < 0 || start > cap) {
    if (threadIdx.x == 0) record_error(c.err, MDL_ERR_BAD_INDEX);
    return;
  }
  const int t0 = (blockIdx.x - i * chunks) * chunk, nt = min(chunk, a.T - t0);
  const bool token_fast = nt >= 32 / LPU;
  const int units = nt * c.G;
  const int sub = threadIdx.x % LPU;
  const __nv_bfloat16* kb = a.k + i * a.k_sb + sub * 16;
  const __nv_bfloat16* vb = a.v + i * a.v_sb + sub * 16;
  // unit u = slow * inner + fast, carried along
  constexpr int UNITS = kThreads / LPU;
  const int inner = token_fast ? nt : c.G, ds = UNITS / inner, df = UNITS % inner;
  int u = threadIdx.x / LPU, slow = u / inner, fast = u % inner;
  auto next = [&]() {
    u += UNITS;
    slow += ds;
    fast += df;
    if (fast >= inner) {
      fast -= inner;
      ++slow;
    }
  };
  for (int base = 0; base < units; base += UNITS, next()) {  // whole warps stay together: shuffles below
    const bool live = u < units;
    const int g = token_fast ? slow : fast, t = t0 + (token_fast ? fast : slow);
    const int at = t - first;  // behind start
    const bool in = live && at >= 0;
    uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0, v0 = k0, v1 = k0;
    int pg = -1;
    if (in) {
      const uint4* kp = reinterpret_cast<const uint4*>(kb + t * a.k_st + g * HD);
      const uint4* vp = reinterpret_cast<const uint4*>(vb + t * a.v_st + g * HD);
      k0 = kp[0];
      k1 = kp[1];
      v0 = vp[0];
      v1 = vp[1];
      // compared like this, since start + at may pass 32 bits in a long row
      if (at >= cap - start) record_error(c.err, MDL_ERR_CAPACITY);
      else pg = page_of(c, r, start + at);
    }
    uint16_t ks, vs;
    const uint2 kc = quantise16<HD>(k0, k1, ks), vc = quantise16<HD>(v0, v1, vs);
    if (pg < 0) continue;
    const int pos = start + at;
    const long long bk = slot_base(c, pg, g, 0) + (pos & ((1 << c.page_shift) - 1));
    const long long bv = bk + (1ll << c.page_shift);
    reinterpret_cast<uint2*>(c.codes)[bk * LPU + sub] = kc;
    reinterpret_cast<uint2*>(c.codes)[bv * LPU + sub] = vc;
    if (sub == 0) reinterpret_cast<uint32_t*>(c.scales)[scale_index(c, pg, g, pos)] = ks | (static_cast<uint32_t>(vs) << 16);
  }
  // only the single block of a row may write the length that its threads read above
  if (chunks == 1) {
    __syncthreads();
    if (threadIdx.x == 0) c.lengths[r] = start + min(a.T - first, cap - start);
  }
}

// Lengths after a write that took several blocks a row.
__global__ void kv_length_kernel(KvWriteArgs a) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.n) return;
  const KvCache& c = a.c;
  const int r = a.rows != nullptr ? a.rows[i] : i;
  if (static_cast<unsigned>(r) >= static_cast<unsigned>(c.R)) return;
  const int cap = c.max_pages << c.page_shift;
  const int first = a.kstart != nullptr ? min(max(a.kstart[i], 0), a.T) : 0;
  const int start = a.start != nullptr ? a.start[i] : c.lengths[r];
  if (start < 0 || start > cap) return;
  c.lengths[r] = start + min(a.T - first, cap - start);
}

// ============================================================================ codes
// Codes to bf16 pairs: (w >> 4i) & 0x000F000F | 0x4300_4300 is the exact bf16 pair
// (128 + nibble i, 128 + nibble i + 4) = 136 + c.
constexpr uint32_t kMagic = 0x43004300u;   // bf16 128, twice
constexpr uint32_t kOffset = 0x43084308u;  // bf16 136, twice

// (w & 0x000F000F) | magic in one instruction: it takes one immediate, so the magic number has to
// sit in a register (`magic`, which the compiler does not see through).
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(d) : "r"(w), "r"(magic));
  return d;
}

__device__ __forceinline__ uint32_t code_pair_signed(uint32_t w, uint32_t magic) {
  const uint32_t u = code_pair(w, magic), o = kOffset;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&o));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ============================================================================ read
// Thread = one code word (8 values) of K and of V, units by token, then head: a warp reads a dense
// run of a page. Bound by memory, the bf16 that it writes: 384 rows of up to 2,048 tokens, 8 heads of
// 32: 167 us, 6.0 TB/s read and written (182 us where each nibble was converted by itself, 222
// million conversions on a unit that does 16 a cycle).
template <int HD, bool F32>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvReadArgs a, int chunk, int chunks) {
  constexpr int LPU = HD / 8, UNITS = kThreads / LPU;  // units a pass
  const KvCache& c = a.c;
  const int i = blockIdx.x / chunks;
  const int r = row_of(c, a.rows, i);
  const int cap = c.max_pages << c.page_shift;
  const int len = r < 0 ? 0 : min(max(c.lengths[r], 0), cap);
  const int start = a.start != nullptr ? a.start[i] : 0;
  if (start < 0 && threadIdx.x == 0) record_error(c.err, MDL_ERR_BAD_INDEX);
  const int t0 = (blockIdx.x - i * chunks) * chunk, nt = min(chunk, a.count - t0);
  const int sub = threadIdx.x % LPU, u = threadIdx.x / LPU;
  const int dg = UNITS / nt, dt = UNITS % nt;
  uint32_t magic;
  asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(kMagic));
  for (int g = u / nt, t = u % nt; g < c.G;) {
    const long long pos = static_cast<long long>(start) + t0 + t;
    uint32_t w[2] = {0x88888888u, 0x88888888u}, sc = 0;
    if (pos >= 0 && pos < len) {
      const int pg = page_of(c, r, static_cast<int>(pos));
      if (pg >= 0) {
        const int slot = static_cast<int>(pos) & ((1 << c.page_shift) - 1);
        const long long b = slot_base(c, pg, g, 0) + slot;
        w[0] = reinterpret_cast<const uint32_t*>(c.codes)[b * LPU + sub];
        w[1] = reinterpret_cast<const uint32_t*>(c.codes)[(b + (1ll << c.page_shift)) * LPU + sub];
        sc = reinterpret_cast<const uint32_t*>(c.scales)[scale_index(c, pg, g, static_cast<int>(pos))];
      }
    }
    const long long off = (static_cast<long long>(i) * a.count + t0 + t) * (c.G * HD) + g * HD + sub * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint32_t p[4];  // values (j, j + 4), exact
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = code_pair_signed(w[kv] >> (4 * j), magic);
      void* out = kv ? a.out_v : a.out_k;
      if constexpr (F32) {
        const float s = kv ? bf16_hi(sc) : bf16_lo(sc);
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(out) + off);
        d[0] = make_float4(s * bf16_lo(p[0]), s * bf16_lo(p[1]), s * bf16_lo(p[2]), s * bf16_lo(p[3]));
        d[1] = make_float4(s * bf16_hi(p[0]), s * bf16_hi(p[1]), s * bf16_hi(p[2]), s * bf16_hi(p[3]));
      } else {
        const uint32_t ss = __byte_perm(sc, sc, kv ? 0x3232 : 0x1010);
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // s * c, rounded once
          const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&p[j]),
                                           *reinterpret_cast<const __nv_bfloat162*>(&ss));
          p[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + off) =
            make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                       __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
      }
    }
    g += dg;
    t += dt;
    if (t >= nt) {
      t -= nt;
      ++g;
    }
  }
}

// ============================================================================ attend
// Batch row b reads cache row rows[b] of length len. Query n sits at position len + n with
// fresh keys (kn, vn: the batch row's own tokens, not in the cache) and at len - N + n without
// (its own token is in the cache already). It sees a position j at or before its own with
// window == 0, or less than `window` back, or j < sinks.
//
// Work item = (b, key head g, block of 8 * NT query rows); query row m = n * (H / G) + a is
// query n of the a-th query head that shares g. The products run on mma.sync m16n8k16 with the
// KEYS in the M dimension: S^T[16 keys, 8 queries] = K Q^T and O^T[16 dims, 8 queries] =
// V^T P^T. A single query costs then half of what it would with the queries in M (8 columns
// instead of 16 rows are padding), and the codes, expanded in registers, are the A operand of
// both products. tcgen05 needs 128 rows (and its operands in shared memory): the few queries
// of a request do not fill that, and the kernel is bound by the expansion of the codes and
// its latency, not by the products.
//
// The codes enter as code_pair gives them, 136 + c. K uses it as it is: S = q . (136 + c) - 136 * sum(q), the
// second term being the accumulator's initial value. V subtracts 136 (one packed, exact
// operation), since the same shortcut over a long sum of keys would cancel. The scales enter
// in fp32: s_k multiplies the scores, s_v the probabilities.
//
// Bound by the latency of a step (expand, product, maximum, exponentials, product follow one another,
// with 8 to 16 warps a multiprocessor to hide it): issue slots are 56 % busy, the pipe that expands the
// codes 44 to 55 %, DRAM 4 to 40 %. 24 single tokens over 131,071 keys, 8 query heads on 2 key heads of
// 64: 119 us, 3.6 TB/s of cache; 1,024 samples of 32 candidates, 8 heads of 32, window 512 of 2,000
// keys: 165 us, 108 TFLOP/s; one token over 501 keys: 4.6 us.
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// 8 x 8 b16 transpose across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Eight bf16 (dims d .. d+7) as the pairs (d+i, d+i+4) that code_pair gives for a code word.
__device__ __forceinline__ void split_pairs(const uint4 v, uint32_t* p) {
  p[0] = __byte_perm(v.x, v.z, 0x5410);
  p[1] = __byte_perm(v.x, v.z, 0x7632);
  p[2] = __byte_perm(v.y, v.w, 0x5410);
  p[3] = __byte_perm(v.y, v.w, 0x7632);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Blocks an SM that the registers have to allow: the kernel hides its latencies with warps, up to
// where it spills much. 8 query rows a block: 32-wide heads with one warp an item, 256 rows of 2,000
// keys: five blocks 62 us, six (spilling) 67, seven 83; 64-wide ones with one warp, 4 heads: five blocks
// (8 bytes spilled) 52 us for 2,000 rows of 300 keys and 75 for 1,000 of 1,000, four (none) 53 and 74;
// with eight warps: two blocks 121 us for 24 rows of 131,071 keys and 48 for 256 of 2,000, three
// (spilling) 127 and 46.
template <int HD, int NT, int WPI>
constexpr int min_blocks() {
  return WPI == 1 ? (NT == 1 ? 5 : (NT == 2 ? 4 : 3)) : (NT == 1 ? (HD == 64 ? 2 : 3) : (NT == 2 ? 2 : 1));
}
template <int NT>
constexpr int tiles_a_step() { return NT == 1 ? 4 : 2; }
// Shared memory: the warps' rings of steps (K codes | V codes | scales), whose space the join of eight
// warps takes afterwards; behind both the rings' barriers and a word a warp. The barriers keep a place of
// their own: a barrier that lanes have waited on may still be written when the wait is over, and with the
// join's maxima there (more than 8 query rows a block of 64-wide heads) some of these were lost.
template <int HD, int NT>
constexpr int step_bytes() { return 16 * tiles_a_step<NT>() * (HD + 4); }
template <int HD>
constexpr int ring_steps() { return HD == 64 ? 2 : 3; }
template <int HD, int NT, int WPI>
constexpr int attend_data() {
  constexpr int ring = (WPI == 1 ? 4 : WPI) * ring_steps<HD>() * step_bytes<HD, NT>();
  constexpr int join = WPI == 1 ? 0 : WPI * 8 * NT * (HD + 6) * 4;
  return ring > join ? ring : join;
}
template <int HD, int NT, int WPI>
constexpr int attend_smem() {
  return attend_data<HD, NT, WPI>() + (WPI == 1 ? 4 : WPI) * (8 * ring_steps<HD>() + 4);
}

// Bulk copy into this CTA's shared memory, 16-byte aligned, counted on `bar`.
__device__ __forceinline__ void bulk_copy(uint8_t* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The rest of a wait that is not over at once; the same outcome on every lane.
__device__ __noinline__ bool ring_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, nullptr));
}

// Bit j: the 16-key tile at k0 + 16 j (below len) lies in a page outside the cache. Out of line: it
// is looked at only once a page has been found missing.
__device__ __noinline__ uint32_t missing_tiles(const KvCache& c, const int* table, int k0, int len, int tiles) {
  uint32_t gone = 0;
  for (int j = 0; j < tiles && k0 + 16 * j < len; ++j) {
    const int q = __ldg(table + ((k0 + 16 * j) >> c.page_shift));
    if (static_cast<unsigned>(q) >= static_cast<unsigned>(c.num_pages)) gone |= 1u << j;
  }
  return gone;
}

template <int HD, int NT, int WPI>
__global__ void __launch_bounds__(WPI == 1 ? 128 : 32 * WPI, min_blocks<HD, NT, WPI>())
    kv_attend_kernel(KvAttendArgs a, int qblocks, int splits) {
  constexpr int KT = tiles_a_step<NT>();  // 16-key tiles a step
  constexpr int CH = 16 * KT;
  constexpr int KW = HD / 32;           // code words of a key a lane
  constexpr int KS = HD / 16;           // k steps of the score product
  constexpr int MT = HD / 16;           // 16-dim tiles of the output
  constexpr int COLS = 8 * NT;
  const KvCache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, t = lane & 3;
  const long long items = static_cast<long long>(a.B) * c.G * qblocks;
  long long item;
  int part = 0, parts = 1, split = 0;
  if constexpr (WPI == 1) {
    item = static_cast<long long>(blockIdx.x) * 4 + warp;
    if (item >= items) return;
  } else {
    item = blockIdx.x / splits;
    split = static_cast<int>(blockIdx.x - item * splits);
    part = split * WPI + warp;
    parts = splits * WPI;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join of the splits may take its place
  }
  const int qb = static_cast<int>(item % qblocks);
  const int g = static_cast<int>(item / qblocks % c.G);
  const int b = static_cast<int>(item / qblocks / c.G);
  const int group = a.H / c.G, M = a.N * group, m0 = qb * COLS;
  const int r = row_of(c, a.rows, b);
  const int cap = c.max_pages << c.page_shift;
  const int len = r < 0 ? 0 : min(max(c.lengths[r], 0), cap);
  const bool fresh = a.kn != nullptr;
  const int base = fresh ? len : len - a.N;
  const int W = a.window, S = a.sinks;

  // ---- queries: B operand (column g8 of each tile), and sum(q) of columns 2t, 2t + 1
  uint32_t qf[NT][KS][2];
  float init[NT][4];  // a whole operand: building it for each product would cost four moves
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int m = min(m0 + nt * 8 + g8, M - 1);
    const __nv_bfloat16* src = a.q + b * a.q_sb + (m / group) * a.q_sn + (g * group + m % group) * HD + t * (HD / 4);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const uint4 v = reinterpret_cast<const uint4*>(src)[w];
      uint32_t p[4];
      split_pairs(v, p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qf[nt][2 * w + (i >> 1)][i & 1] = p[i];
        sum += bf16_lo(p[i]) + bf16_hi(p[i]);
      }
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      init[nt][e] = init[nt][e + 2] = -136.f * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
    }
  }
  const float scale2 = a.scale * 1.4426950408889634f;
  uint32_t magic;
  asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(kMagic));
  // query of columns 2t + e of a tile (only where a mask is needed)
  auto query_of = [&](int nt, int e) {
    const int m = min(m0 + nt * 8 + 2 * t + e, M - 1);
    return group == 1 ? m : m / group;
  };

  float o[MT][NT][4];
  float mx[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.f;
    mx[nt][0] = mx[nt][1] = -CUDART_INF_F;
    l[nt][0] = l[nt][1] = 0.f;
  }

  // Online softmax in base 2. The running maximum is a reference that is only moved when a
  // score passes it by more than 8 (exp2 of the excess stays below 256), so most steps need no
  // reduction over the lanes and no rescaling.
  auto raise = [&](float (&lm)[NT][2]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = lm[nt][e];
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        v = fmaxf(v, mx[nt][e]);
        const float alpha = v == -CUDART_INF_F ? 1.f : ex2(mx[nt][e] - v);
        mx[nt][e] = v;
        l[nt][e] *= alpha;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o[mt][nt][e] *= alpha;
          o[mt][nt][e + 2] *= alpha;
        }
      }
  };

  // ---- cached keys
  const int qmin = base + min(m0, M - 1) / group, qmax = base + min(m0 + COLS - 1, M - 1) / group;
  const int hi = min(len, qmax + 1);
  int cs = 0, cw = 0, total = 0;  // steps [0, cs) of the sinks, then [cw, ...) of the window
  if (hi > 0) {
    const int end = (hi + CH - 1) / CH;
    if (W > 0) {
      cw = min(max(0, qmin - W + 1) / CH, end);  // the window of late fresh tokens lies past the row
      cs = min((min(S, hi) + CH - 1) / CH, cw);
    }
    total = cs + end - cw;
  }
  auto step_key = [&](int i) { return (i < cs ? i : cw + i - cs) * CH; };
  // Row rho of a 16-key tile is key (rho >> 1 & 3) + 4 (rho & 1) + (rho & 8): the second product
  // then reads four neighbouring keys at once, without bank conflicts. The lane's rows: g8, + 8.
  const int row8 = (g8 >> 1) + 4 * (g8 & 1);
  // A ring of steps in shared memory, filled by bulk copies: enough bytes under way to cover
  // the memory latency without registers for them.
  constexpr int RING = ring_steps<HD>(), STEP = step_bytes<HD, NT>(), TILE_CODES = 16 * HD / 2;
  constexpr int BARS = attend_data<HD, NT, WPI>();
  static_assert(BARS % 8 == 0, "barriers");
  extern __shared__ __align__(128) uint8_t sm_ring[];
  constexpr int WARPS = WPI == 1 ? 4 : WPI;
  uint8_t* ring = sm_ring + warp * RING * STEP;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm_ring + BARS) + warp * RING;
  // Steps from all_lo + 1 (or up to S) to all_hi are visible to every query of the block. Once the warp
  // has met a page outside the cache, none is: every step is masked, by another look at the table. (In
  // shared memory: as a register that changes it made the kernels spill.)
  constexpr int BAD_PAGE = -0x7fffffff - 1;
  volatile int* all_hi = reinterpret_cast<volatile int*>(sm_ring + BARS + WARPS * RING * 8) + warp;
  *all_hi = min(len, qmin + 1) - CH;
  const int all_lo = W > 0 ? qmax - W : -1, all_sink = S - CH;
  if (lane == 0) {
    for (int s = 0; s < RING; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  // Page of each 16-key tile of a step, read a step before its copies are issued; one where a
  // page holds the whole step. The addresses are kept short: what a step costs besides its keys
  // is a fifth of its instructions.
  const bool one_page = (1 << c.page_shift) >= CH;
  const int slot_mask = (1 << c.page_shift) - 1;
  const int* table = c.table + static_cast<long long>(r < 0 ? 0 : r) * c.max_pages;
  const uint8_t* codes_g = c.codes + (slot_base(c, 0, g, 0) * (HD / 2));
  const uint8_t* scales_g = reinterpret_cast<const uint8_t*>(c.scales) + 4 * scale_index(c, 0, g, 0);
  const uint32_t v_off = (slot_mask + 1) * (HD / 2), sc_page = c.G << (c.page_shift + 2);
  const long long code_page = static_cast<long long>(c.G) * 2 * v_off;
  int pg[KT];
  auto page_at = [&](int k0) {
    const int q = __ldg(table + (k0 >> c.page_shift));
    if (static_cast<unsigned>(q) < static_cast<unsigned>(c.num_pages)) return q;
    record_error(c.err, MDL_ERR_BAD_INDEX);
    *all_hi = BAD_PAGE;  // page 0 is copied in its place and hidden
    return 0;
  };
  auto pages = [&](int i) {
    if (i >= total) return;
    const int k0 = step_key(i);
    pg[0] = page_at(k0);  // k0 < len
    if (!one_page) {
#pragma unroll
      for (int j = 1; j < KT; ++j) pg[j] = k0 + 16 * j < len ? page_at(k0 + 16 * j) : 0;
    }
  };
  auto fetch = [&](int i, int st) {
    if (i < total && lane == 0) {
      const int k0 = step_key(i);
      uint8_t* dst = ring + st * STEP;
      if (one_page) {
        const uint32_t slot = k0 & slot_mask;
        const uint8_t* kp = codes_g + pg[0] * code_page + slot * (HD / 2);
        mbar_arrive_expect_tx(&full[st], STEP);
        bulk_copy(dst, kp, KT * TILE_CODES, &full[st]);
        bulk_copy(dst + KT * TILE_CODES, kp + v_off, KT * TILE_CODES, &full[st]);
        bulk_copy(dst + 2 * KT * TILE_CODES, scales_g + static_cast<long long>(pg[0]) * sc_page + slot * 4, CH * 4,
                  &full[st]);
      } else {
        const int tiles = min(KT, (len - k0 + 15) / 16);  // the rest is masked, whatever lies there
        mbar_arrive_expect_tx(&full[st], tiles * (2 * TILE_CODES + 64));
        for (int j = 0; j < tiles; ++j) {
          int page = pg[0];
#pragma unroll
          for (int e = 1; e < KT; ++e) page = j == e ? pg[e] : page;
          const uint32_t slot = (k0 + 16 * j) & slot_mask;
          const uint8_t* kp = codes_g + page * code_page + slot * (HD / 2);
          bulk_copy(dst + j * TILE_CODES, kp, TILE_CODES, &full[st]);
          bulk_copy(dst + (KT + j) * TILE_CODES, kp + v_off, TILE_CODES, &full[st]);
          bulk_copy(dst + 2 * KT * TILE_CODES + 64 * j, scales_g + static_cast<long long>(page) * sc_page + slot * 4, 64,
                    &full[st]);
        }
      }
    }
    __syncwarp();
  };
#pragma unroll 1
  for (int s = 0; s < RING; ++s) {
    pages(part + s * parts);
    fetch(part + s * parts, s);
  }
  pages(part + RING * parts);
  int st = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (int i = part; i < total; i += parts) {
    const int k0 = step_key(i);
    if (!__all_sync(0xffffffffu, mbar_try_wait(&full[st], phase)) && !ring_wait(&full[st], phase, c.err)) {
      // the copies of the stages behind it land before the block may end
      for (int s = 1; s < RING && i + s * parts < total; ++s) {
        phase ^= st + 1 == RING ? 1 : 0;
        st = st + 1 == RING ? 0 : st + 1;
        ring_wait(&full[st], phase, c.err);
      }
      break;
    }
    const uint8_t* sk = ring + st * STEP;
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(sk) + row8 * (HD / 8) + t * KW;
    const uint32_t* vw = reinterpret_cast<const uint32_t*>(sk + KT * TILE_CODES) + t * (HD / 8) + (HD == 64 ? g8 : g8 >> 1);
    const uint32_t* scw = reinterpret_cast<const uint32_t*>(sk + 2 * KT * TILE_CODES) + row8;
    float x[KT][NT][4];  // scores: rows g8 (0, 1) and g8 + 8 (2, 3), columns 2t and 2t + 1
    uint32_t vs[2 * KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      uint32_t wk[2][KW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t* src = kw + (16 * j + 8 * h) * (HD / 8);
        if constexpr (KW == 2) {
          const uint2 y = *reinterpret_cast<const uint2*>(src);
          wk[h][0] = y.x;
          wk[h][1] = y.y;
        } else {
          wk[h][0] = *src;
        }
        vs[2 * j + h] = scw[16 * j + 8 * h];
      }
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t wa = wk[0][w], wb = wk[1][w];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a0 = code_pair(wa >> (8 * h), magic), a1 = code_pair(wb >> (8 * h), magic);
          const uint32_t a2 = code_pair(wa >> (8 * h + 4), magic), a3 = code_pair(wb >> (8 * h + 4), magic);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int ks = 2 * w + h;
            if (ks == 0)
              mma16816(x[j][nt], a0, a1, a2, a3, qf[nt][ks][0], qf[nt][ks][1], init[nt][0], init[nt][1], init[nt][2],
                       init[nt][3]);
            else
              mma16816(x[j][nt], a0, a1, a2, a3, qf[nt][ks][0], qf[nt][ks][1], x[j][nt][0], x[j][nt][1], x[j][nt][2],
                       x[j][nt][3]);
          }
        }
      }
      const float s0 = bf16_lo(vs[2 * j]) * scale2, s1 = bf16_lo(vs[2 * j + 1]) * scale2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const F2 a = mul2({x[j][nt][0], x[j][nt][1]}, {s0, s0}), b = mul2({x[j][nt][2], x[j][nt][3]}, {s1, s1});
        x[j][nt][0] = a.x;
        x[j][nt][1] = a.y;
        x[j][nt][2] = b.x;
        x[j][nt][3] = b.y;
      }
    }
    // every key of the step visible to every query of the block?
    const bool whole = k0 <= *all_hi && (k0 > all_lo || k0 <= all_sink);
    if (!whole) {
      const uint32_t gone = *all_hi == BAD_PAGE ? missing_tiles(c, table, k0, len, KT) : 0u;
      uint32_t reach[KT][2];  // a key is visible to the queries less than this far on
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kp = k0 + 16 * j + 8 * h + row8;
          reach[j][h] = kp >= len || (gone >> j & 1u) != 0 ? 0u : (W == 0 || kp < S ? 0x80000000u : static_cast<uint32_t>(W));
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int qp = base + query_of(nt, e);
#pragma unroll
          for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (static_cast<uint32_t>(qp - (k0 + 16 * j + 8 * h + row8)) >= reach[j][h])
                x[j][nt][2 * h + e] = -CUDART_INF_F;
        }
    }
    float lm[NT][2], over = -CUDART_INF_F;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = fmaxf(x[0][nt][e], x[0][nt][e + 2]);
#pragma unroll
        for (int j = 1; j < KT; ++j) v = max3(v, x[j][nt][e], x[j][nt][e + 2]);
        lm[nt][e] = v;
      }
      // -inf - -inf (nothing seen so far, nothing here) is a NaN, which the maximum passes over
      over = max3(over, lm[nt][0] - mx[nt][0], lm[nt][1] - mx[nt][1]);
    }
    if (__any_sync(0xffffffffu, over > 8.f)) raise(lm);
    // P (times the scale of V) as the B operand of the second product
    uint32_t pb[KT][NT][2];
    auto weigh = [&](auto masked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float use[2] = {mx[nt][0], mx[nt][1]};
        if constexpr (decltype(masked)::value) {
          if (use[0] == -CUDART_INF_F) use[0] = 0.f;
          if (use[1] == -CUDART_INF_F) use[1] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float v = bf16_hi(vs[2 * j + h]);
            const F2 y = fma2({use[0], use[1]}, {-1.f, -1.f}, {x[j][nt][2 * h], x[j][nt][2 * h + 1]});
            F2 e = {ex2(y.x), ex2(y.y)};
            const F2 sum = add2({l[nt][0], l[nt][1]}, e);
            l[nt][0] = sum.x;
            l[nt][1] = sum.y;
            e = mul2(e, {v, v});
            if constexpr (decltype(masked)::value) {  // the scale of a hidden key may be a NaN
              if (y.x == -CUDART_INF_F) e.x = 0.f;
              if (y.y == -CUDART_INF_F) e.y = 0.f;
            }
            pb[j][nt][h] = transpose8(pack_bf16(e.x, e.y));
          }
      }
    };
    if (whole) weigh(std::false_type{});
    else weigh(std::true_type{});
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      // rows 2t, 2t + 1, 2t + 8, 2t + 9 of the tile: keys t, t + 4, t + 8, t + 12
      const uint32_t va = vw[16 * j * (HD / 8)], vb = vw[(16 * j + 4) * (HD / 8)];
      const uint32_t vc = vw[(16 * j + 8) * (HD / 8)], vd = vw[(16 * j + 12) * (HD / 8)];
      uint32_t u0, u1, u2, u3;
      if constexpr (HD == 64) {
        u0 = __byte_perm(va, vb, 0x5410);
        u1 = __byte_perm(va, vb, 0x7632);
        u2 = __byte_perm(vc, vd, 0x5410);
        u3 = __byte_perm(vc, vd, 0x7632);
      } else {
        const uint32_t sel = (g8 & 1) ? 0x7632 : 0x5410;
        u0 = __byte_perm(va, vb, sel);
        u2 = __byte_perm(vc, vd, sel);
        u1 = u0 >> 4;
        u3 = u2 >> 4;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        constexpr int STEP = HD == 64 ? 4 : 8;
        const uint32_t a0 = code_pair_signed(u0 >> (STEP * mt), magic), a1 = code_pair_signed(u1 >> (STEP * mt), magic);
        const uint32_t a2 = code_pair_signed(u2 >> (STEP * mt), magic), a3 = code_pair_signed(u3 >> (STEP * mt), magic);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(o[mt][nt], a0, a1, a2, a3, pb[j][nt][0], pb[j][nt][1], o[mt][nt][0], o[mt][nt][1], o[mt][nt][2],
                   o[mt][nt][3]);
      }
    }
    __syncwarp();  // the warp has read the stage
    fetch(i + RING * parts, st);
    pages(i + (RING + 1) * parts);
    if (++st == RING) {
      st = 0;
      phase ^= 1;
    }
  }

  // ---- the batch row's own keys (bf16), tiles of 16
  if (fresh) {
    const int nmin = min(m0, M - 1) / group, nmax = min(m0 + COLS - 1, M - 1) / group;
    const int tiles = nmax / 16 + 1;
    for (int i = part; i < tiles; i += parts) {
      const int k0 = 16 * i;
      if (W > 0 && k0 + 15 <= nmin - W && len + k0 >= S) continue;
      float x[NT][4];
      const __nv_bfloat16* ka = a.kn + b * a.kn_sb + g * HD + t * (HD / 4);
      const int ra = min(k0 + g8, a.N - 1), rb = min(k0 + 8 + g8, a.N - 1);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        uint32_t pa[4], pb[4];
        split_pairs(reinterpret_cast<const uint4*>(ka + ra * a.kn_sn)[w], pa);
        split_pairs(reinterpret_cast<const uint4*>(ka + rb * a.kn_sn)[w], pb);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int ks = 2 * w + h;
            if (ks == 0)
              mma16816(x[nt], pa[0], pb[0], pa[1], pb[1], qf[nt][0][0], qf[nt][0][1], 0.f, 0.f, 0.f, 0.f);
            else
              mma16816(x[nt], pa[2 * h], pb[2 * h], pa[2 * h + 1], pb[2 * h + 1], qf[nt][ks][0], qf[nt][ks][1],
                       x[nt][0], x[nt][1], x[nt][2], x[nt][3]);
          }
      }
      float lm[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int qn[2] = {query_of(nt, 0), query_of(nt, 1)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kp = k0 + g8 + 8 * (e >> 1);
          const uint32_t reach = W == 0 || len + kp < S ? 0x80000000u : static_cast<uint32_t>(W);
          const bool vis = static_cast<uint32_t>(qn[e & 1] - kp) < reach;
          x[nt][e] = vis ? x[nt][e] * scale2 : -CUDART_INF_F;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          lm[nt][e] = fmaxf(x[nt][e], x[nt][e + 2]);
          grow |= lm[nt][e] > mx[nt][e] + 8.f;
        }
      }
      if (__any_sync(0xffffffffu, grow)) raise(lm);
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float use = mx[nt][e & 1] == -CUDART_INF_F ? 0.f : mx[nt][e & 1];
          p[e] = ex2(x[nt][e] - use);
          l[nt][e & 1] += p[e];
        }
        pb[nt][0] = transpose8(pack_bf16(p[0], p[1]));
        pb[nt][1] = transpose8(pack_bf16(p[2], p[3]));
      }
      // V^T of keys k0 + 2t, 2t+1, 2t+8, 2t+9: hd / 8 dims from g8 * hd / 8; zero past the last token
      uint32_t vv[4][HD / 16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int kr = k0 + 2 * t + (e & 1) + 8 * (e >> 1);
        const __nv_bfloat16* vp = a.vn + b * a.vn_sb + min(kr, a.N - 1) * a.vn_sn + g * HD + g8 * (HD / 8);
        if constexpr (HD == 64) {
          const uint4 y = *reinterpret_cast<const uint4*>(vp);
          vv[e][0] = y.x; vv[e][1] = y.y; vv[e][2] = y.z; vv[e][3] = y.w;
        } else {
          const uint2 y = *reinterpret_cast<const uint2*>(vp);
          vv[e][0] = y.x; vv[e][1] = y.y;
        }
        if (kr >= a.N) {
#pragma unroll
          for (int w = 0; w < HD / 16; ++w) vv[e][w] = 0;
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a0, a1, a2, a3;
        if constexpr (HD == 64) {  // rows g8: dims mt, rows g8 + 8: dims 4 + mt of the eight
          const uint32_t sel = (mt & 1) ? 0x7632 : 0x5410;
          a0 = __byte_perm(vv[0][mt >> 1], vv[1][mt >> 1], sel);
          a1 = __byte_perm(vv[0][2 + (mt >> 1)], vv[1][2 + (mt >> 1)], sel);
          a2 = __byte_perm(vv[2][mt >> 1], vv[3][mt >> 1], sel);
          a3 = __byte_perm(vv[2][2 + (mt >> 1)], vv[3][2 + (mt >> 1)], sel);
        } else {  // rows g8: dim 2 mt, rows g8 + 8: dim 2 mt + 1 of the four
          a0 = __byte_perm(vv[0][mt], vv[1][mt], 0x5410);
          a1 = __byte_perm(vv[0][mt], vv[1][mt], 0x7632);
          a2 = __byte_perm(vv[2][mt], vv[3][mt], 0x5410);
          a3 = __byte_perm(vv[2][mt], vv[3][mt], 0x7632);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1], o[mt][nt][0], o[mt][nt][1], o[mt][nt][2],
                   o[mt][nt][3]);
      }
    }
  }

  // ---- sums over the lanes that share a column
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = l[nt][e];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      l[nt][e] = v;
    }
  // lane's dims of column (nt, e): hd / 8 neighbouring ones from g8 * hd / 8
  auto dims = [&](int nt, int e, float* d) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (HD == 64) {
        d[mt] = o[mt][nt][e];
        d[4 + mt] = o[mt][nt][e + 2];
      } else {
        d[2 * mt] = o[mt][nt][e];
        d[2 * mt + 1] = o[mt][nt][e + 2];
      }
    }
  };
  auto out_row = [&](int m) {
    return a.out + (static_cast<long long>(b) * a.N + m / group) * a.H * HD + (g * group + m % group) * HD;
  };
  if constexpr (WPI == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int m = m0 + nt * 8 + 2 * t + e;
        if (m >= M) continue;
        const float inv = l[nt][e] == 0.f ? 0.f : 1.f / l[nt][e];
        float d[HD / 8];
        dims(nt, e, d);
        __nv_bfloat16* dst = out_row(m) + g8 * (HD / 8);
        if constexpr (HD == 64)
          *reinterpret_cast<uint4*>(dst) =
              make_uint4(pack_bf16(d[0] * inv, d[1] * inv), pack_bf16(d[2] * inv, d[3] * inv),
                         pack_bf16(d[4] * inv, d[5] * inv), pack_bf16(d[6] * inv, d[7] * inv));
        else
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(pack_bf16(d[0] * inv, d[1] * inv), pack_bf16(d[2] * inv, d[3] * inv));
      }
  } else {
    // join the warps: per column the common maximum, then the weighted sums
    __syncthreads();  // every warp is through with its ring
    float* sm = reinterpret_cast<float*>(sm_ring);
    float* so = sm;                              // [WPI][COLS][HD + 4]
    float* smx = sm + WPI * COLS * (HD + 4);     // [WPI][COLS]
    float* sl = smx + WPI * COLS;                // [WPI][COLS]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = nt * 8 + 2 * t + e;
        float d[HD / 8];
        dims(nt, e, d);
        float* dst = so + (warp * COLS + col) * (HD + 4) + g8 * (HD / 8);
#pragma unroll
        for (int w = 0; w < HD / 32; ++w)
          reinterpret_cast<float4*>(dst)[w] = make_float4(d[4 * w], d[4 * w + 1], d[4 * w + 2], d[4 * w + 3]);
        if (g8 == 0) {
          smx[warp * COLS + col] = mx[nt][e];
          sl[warp * COLS + col] = l[nt][e];
        }
      }
    __syncthreads();
    for (int idx = threadIdx.x; idx < COLS * (HD / 4); idx += 32 * WPI) {
      const int col = idx / (HD / 4), d4 = idx % (HD / 4);
      if (m0 + col >= M) continue;
      float top = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < WPI; ++w) top = fmaxf(top, smx[w * COLS + col]);
      const float use = top == -CUDART_INF_F ? 0.f : top;
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WPI; ++w) {
        const float f = ex2(smx[w * COLS + col] - use);
        const float4 y = *reinterpret_cast<const float4*>(so + (w * COLS + col) * (HD + 4) + 4 * d4);
        sum = fmaf(sl[w * COLS + col], f, sum);
        acc.x = fmaf(y.x, f, acc.x);
        acc.y = fmaf(y.y, f, acc.y);
        acc.z = fmaf(y.z, f, acc.z);
        acc.w = fmaf(y.w, f, acc.w);
      }
      if (splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(out_row(m0 + col) + 4 * d4) =
            make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
      } else {
        float* dst = a.partial + ((item * splits + split) * COLS + col) * (HD + 4);
        *reinterpret_cast<float4*>(dst + 4 * d4) = acc;
        if (d4 == 0) {
          dst[HD] = top;
          dst[HD + 1] = sum;
        }
      }
    }
  }
}

// Joins the splits, a warp a query row: lane s weighs split s (kMaxSplits is a warp), then hd / 4
// lanes add up 4 dims each, in groups that share the splits. It is launched while the splits are
// still being computed and waits for them in place.
constexpr int kMaxSplits = 32;

template <int HD>
__global__ void __launch_bounds__(128) kv_combine_kernel(KvAttendArgs a, int qblocks, int splits, int cols) {
  constexpr int LANES = HD / 4, GROUPS = 32 / LANES;
  const int group = a.H / a.c.G, M = a.N * group, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(a.B) * a.c.G * M) return;
  const int m = static_cast<int>(row % M);
  const long long bg = row / M;
  const int g = static_cast<int>(bg % a.c.G);
  const long long b = bg / a.c.G;
  const float* src = a.partial + ((bg * qblocks + m / cols) * splits * cols + m % cols) * (HD + 4);
  const long long step = static_cast<long long>(cols) * (HD + 4);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float top = -CUDART_INF_F, sum = 0.f;
  if (lane < splits) {
    const float2 y = *reinterpret_cast<const float2*>(src + lane * step + HD);
    top = y.x;
    sum = y.y;
  }
  const float own = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = ex2(own - (top == -CUDART_INF_F ? 0.f : top));
  sum *= f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int d4 = lane % LANES, first = lane / LANES;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s0 = 0; s0 < splits; s0 += GROUPS) {
    const int s = s0 + first;
    const float w = __shfl_sync(0xffffffffu, f, s & 31);
    if (s < splits) {
      const float4 y = *reinterpret_cast<const float4*>(src + s * step + 4 * d4);
      acc.x = fmaf(y.x, w, acc.x);
      acc.y = fmaf(y.y, w, acc.y);
      acc.z = fmaf(y.z, w, acc.z);
      acc.w = fmaf(y.w, w, acc.w);
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
  }
  if (first != 0) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat16* dst = a.out + (b * a.N + m / group) * a.H * HD + (g * group + m % group) * HD + 4 * d4;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

constexpr int kMaxDevices = 64;

int device_index() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}

int num_sms() {
  static std::atomic<int> n[kMaxDevices];
  const int dev = device_index();
  int v = n[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
    n[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

struct Plan {
  int nt, wpi, qblocks, splits;
  long long items;
};

// Query rows a block: the fewest of 8, 16 and (32-wide heads) 32 that hold an item's rows, so that
// the codes are expanded once. 512 rows of 2,000 cached tokens, 8 heads of 32: 8 queries 113 us in
// blocks of 8 (166 in 16, 254 in 32); 16 queries 167 us in 16 (207, 256); 32 queries 260 us in 32
// (400, 324). 64-wide heads stay at 16: the accumulators of 32 rows leave 8 warps a
// multiprocessor (512 candidates of 32 tokens: 168 us instead of 76).
//
// Warps an item, and blocks an item ("splits", joined by a second kernel): whatever has the lowest
// cost, in keys that a warp passes while its multiprocessor is full. An item costs as much as 80
// more keys with one warp and 400 with eight (which join in shared memory). With one warp an item
// the uneven ends count as 1.5 more items, 5 % all told; eight warps of blocks of 32 rows take 35 %
// longer (one block a multiprocessor). A multiprocessor with few warps is bound by their latency:
// it counts as if it held 10.6 warps of an item each, or 1.5 blocks of eight.
// Measured on single queries, 8 heads of 32, one warp an item | eight: 296 rows of 250 keys 12.6 |
// 24.7 us, 1,000 keys 37.0 | 41.3, 4,000 keys 127 | 119; 64 rows of 1,000 keys 22.1 | 14.5; 32
// queries a row, 512 rows of 8,000 keys 974 | 1,154. Splits 1 | 2 | 4 | 8 | 16 | 32: 1 row of
// 32,000 keys 88 | 49 | 29 | 18 | 12 | 12 us; 16 rows of 2,000 keys 10 | 10 | 12 | 16 | 21 | 31,
// of 32,000 keys 101 | 69 | 68 | 61 | 64 | 73. Over 130 such shapes the choice is 1.2 % slower than
// the best on average, and by 2 us or 5 % at most.
//
// The lengths are on the device, so that keys are counted by the capacity (or the window): rows that fill
// little of it are split like full ones. 16 rows of 500 tokens, 8 heads of 32: 9.7 us with room for 512,
// 14.9 with room for 131,072; 256 rows 19.1 and 25.4.
Plan plan_of(const KvAttendArgs& a) {
  Plan p;
  const int M = a.N * (a.H / a.c.G);
  p.nt = M <= 8 ? 1 : (M <= 16 || a.c.hd == 64 ? 2 : 4);
  p.qblocks = (M + 8 * p.nt - 1) / (8 * p.nt);
  p.items = static_cast<long long>(a.B) * a.c.G * p.qblocks;
  const long long cap = static_cast<long long>(a.c.max_pages) << a.c.page_shift;
  const double keys =
      static_cast<double>(a.window > 0 ? std::min<long long>(cap, static_cast<long long>(a.window) + a.sinks) : cap);
  const int sms = num_sms();
  p.wpi = 1;
  p.splits = 1;
  double best = std::max(10.6, 1.05 * (static_cast<double>(p.items) / sms + 1.5)) * (keys + 80);
  const double slower = p.nt == 4 ? 1.35 : 1.0;
  for (int n = 1; n <= kMaxSplits; ++n) {
    const double busiest = static_cast<double>((p.items * n + sms - 1) / sms);  // blocks of a multiprocessor
    const double cost = slower * std::max(1.5, busiest) * (keys / n + 400) + (n > 1 ? 1000 + 50 * n : 0);
    if (cost < best) {
      best = cost;
      p.wpi = 8;
      p.splits = n;
    }
  }
  return p;
}

template <int HD, int NT, int WPI>
cudaError_t launch_wpi(const KvAttendArgs& a, const Plan& p, cudaStream_t stream) {
  constexpr int smem = attend_smem<HD, NT, WPI>();
  static std::atomic<bool> ready[kMaxDevices];
  if (smem > 48 * 1024) {
    std::atomic<bool>& done = ready[device_index()];
    if (!done.load(std::memory_order_relaxed)) {
      const cudaError_t e =
          cudaFuncSetAttribute(kv_attend_kernel<HD, NT, WPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      done.store(true, std::memory_order_relaxed);
    }
  }
  const long long blocks = WPI == 1 ? (p.items + 3) / 4 : p.items * p.splits;
  kv_attend_kernel<HD, NT, WPI>
      <<<static_cast<unsigned>(blocks), WPI == 1 ? 128 : 32 * WPI, smem, stream>>>(a, p.qblocks, p.splits);
  return cudaGetLastError();
}

template <int HD, int NT>
cudaError_t launch_attend(const KvAttendArgs& a, const Plan& p, cudaStream_t stream) {
  return p.wpi == 1 ? launch_wpi<HD, NT, 1>(a, p, stream) : launch_wpi<HD, NT, 8>(a, p, stream);
}

template <int HD>
cudaError_t attend_hd(const KvAttendArgs& a, const Plan& p, cudaStream_t stream, int* launches) {
  cudaError_t e;
  if (p.nt == 1) e = launch_attend<HD, 1>(a, p, stream);
  else if (HD == 64 || p.nt == 2) e = launch_attend<HD, 2>(a, p, stream);
  else e = launch_attend<HD, HD == 64 ? 2 : 4>(a, p, stream);
  *launches += 1;
  if (e != cudaSuccess || p.splits == 1) return e;
  const long long rows = static_cast<long long>(a.B) * a.N * a.H;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kv_combine_kernel<HD>, a, p.qblocks, p.splits, 8 * p.nt);
  *launches += 1;
  return e;
}

}  // namespace

// Tokens a block of a write or a read: 64, or 16 where that leaves multiprocessors without one. 3 rows
// of 777 tokens, 4 heads of 64 (39 blocks of 64): read 8.4 us, with 16 tokens 4.4, written 9.8 and
// 7.2; 37 rows of 1,237 tokens, 3 heads of 32 (740 blocks): read 8.5, with 16 tokens 10.5, written 14.2
// and 17.4.
static int chunk_of(int rows, int tokens) {
  return static_cast<long long>(rows) * ((tokens + 63) / 64) < num_sms() ? 16 : 64;
}

cudaError_t kv_write(const KvWriteArgs& a, cudaStream_t stream, int* launches) {
  if (a.n == 0) return cudaSuccess;
  const int chunk = a.T > 64 ? chunk_of(a.n, a.T) : 64;  // one block a row sets the length by itself
  const int chunks = std::max(1, (a.T + chunk - 1) / chunk);
  if (static_cast<long long>(chunks) * a.n > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(chunks) * a.n;
  if (a.c.hd == 64)
    kv_write_kernel<64><<<grid, kThreads, 0, stream>>>(a, chunk, chunks);
  else
    kv_write_kernel<32><<<grid, kThreads, 0, stream>>>(a, chunk, chunks);
  *launches += 1;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || chunks == 1) return e;
  kv_length_kernel<<<(a.n + 127) / 128, 128, 0, stream>>>(a);
  *launches += 1;
  return cudaGetLastError();
}

cudaError_t kv_read(const KvReadArgs& a, cudaStream_t stream) {
  if (a.n == 0 || a.count == 0) return cudaSuccess;
  const int chunk = chunk_of(a.n, a.count), chunks = (a.count + chunk - 1) / chunk;
  if (static_cast<long long>(chunks) * a.n > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(chunks) * a.n;
  auto kern = a.c.hd == 64 ? (a.fp32 ? kv_read_kernel<64, true> : kv_read_kernel<64, false>)
                           : (a.fp32 ? kv_read_kernel<32, true> : kv_read_kernel<32, false>);
  kern<<<grid, kThreads, 0, stream>>>(a, chunk, chunks);
  return cudaGetLastError();
}

long long kv_attend_workspace(const KvAttendArgs& a) {
  const Plan p = plan_of(a);
  return p.splits == 1 ? 0 : p.items * p.splits * 8 * p.nt * (a.c.hd + 4);
}

cudaError_t kv_attend(const KvAttendArgs& a, cudaStream_t stream, int* launches) {
  if (a.B == 0 || a.N == 0) return cudaSuccess;
  const Plan p = plan_of(a);
  if (p.items * p.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  return a.c.hd == 64 ? attend_hd<64>(a, p, stream, launches) : attend_hd<32>(a, p, stream, launches);
}

}  // namespace mdl
