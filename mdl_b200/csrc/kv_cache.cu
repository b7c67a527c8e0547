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

// First slot row of (page, head, K|V): times hd / 2 in the codes, as it is in the scales.
__device__ __forceinline__ long long slot_base(const KvCache& c, int pg, int g, int kv) {
  return ((static_cast<long long>(pg) * c.G + g) * 2 + kv) << c.page_shift;
}

// ============================================================================ write
// Eight lanes' worth of a row: hd / 8 lanes hold a row, 8 values each.
template <int HD>
__device__ __forceinline__ uint32_t quantise8(const uint4 x, uint16_t& scale_bits) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  // |x| as 15-bit integers: ordered like the values, infinities and NaN on top
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
#pragma unroll
  for (int o = 1; o < HD / 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top >= 0x7F80u) {
    scale_bits = 0x7FFFu;  // NaN
    return 0x88888888u;    // c = 0
  }
  const __nv_bfloat16 s16 = __float2bfloat16_rn(__uint_as_float(top << 16) / 7.f);
  scale_bits = __bfloat16_as_ushort(s16);
  const float s = __bfloat162float(s16);
  if (s == 0.f) return 0x88888888u;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
    const int c = static_cast<int>(fminf(fmaxf(rintf(v / s), -7.f), 7.f));
    word |= static_cast<uint32_t>(c + 8) << (4 * i);
  }
  return word;
}

// One block: a run of `chunk` tokens of one source row, every head, K and V. A unit = the row
// of one token and head (hd / 8 lanes). Long runs number the units token-fastest, so that a
// warp reads whole 32-byte sectors of 4 or 8 tokens and writes one dense run of a page;
// single tokens number them head-fastest, so that a warp reads densely.
template <int HD>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(KvWriteArgs a, int chunk, int chunks) {
  constexpr int LPU = HD / 8;
  const KvCache& c = a.c;
  const int i = blockIdx.x / chunks;
  const int r = row_of(c, a.rows, i);
  if (r < 0) return;
  const int cap = c.max_pages << c.page_shift;
  const int first = a.kstart != nullptr ? min(max(a.kstart[i], 0), a.T) : 0;
  int start = a.start != nullptr ? a.start[i] : c.lengths[r];
  if (start < 0 || start > cap) {
    if (threadIdx.x == 0) record_error(c.err, MDL_ERR_BAD_INDEX);
    return;
  }
  const int t0 = (blockIdx.x - i * chunks) * chunk, nt = min(chunk, a.T - t0);
  const bool token_fast = nt >= 32 / LPU;
  const int units = nt * c.G;
  const int sub = threadIdx.x % LPU;
  for (int base = 0; base < units; base += kThreads / LPU) {  // whole warps stay together: shuffles below
    const int u = base + threadIdx.x / LPU;
    const bool live = u < units;
    const int g = live ? (token_fast ? u / nt : u % c.G) : 0;
    const int t = t0 + (live ? (token_fast ? u % nt : u / c.G) : 0);
    const int pos = start + t - first;
    const bool in = live && t >= first;
    uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
    if (in) {
      kx = *reinterpret_cast<const uint4*>(a.k + i * a.k_sb + t * a.k_st + g * HD + sub * 8);
      vx = *reinterpret_cast<const uint4*>(a.v + i * a.v_sb + t * a.v_st + g * HD + sub * 8);
    }
    uint16_t ks, vs;
    const uint32_t kc = quantise8<HD>(kx, ks), vc = quantise8<HD>(vx, vs);
    if (!in) continue;
    if (pos >= cap) {
      record_error(c.err, MDL_ERR_CAPACITY);
      continue;
    }
    const int pg = page_of(c, r, pos);
    if (pg < 0) continue;
    const int slot = pos & ((1 << c.page_shift) - 1);
    const long long bk = slot_base(c, pg, g, 0) + slot, bv = slot_base(c, pg, g, 1) + slot;
    reinterpret_cast<uint32_t*>(c.codes)[bk * LPU + sub] = kc;
    reinterpret_cast<uint32_t*>(c.codes)[bv * LPU + sub] = vc;
    if (sub == 0) {
      reinterpret_cast<uint16_t*>(c.scales)[bk] = ks;
      reinterpret_cast<uint16_t*>(c.scales)[bv] = vs;
    }
  }
  // only the single block of a row may write the length that its threads read above
  if (chunks == 1) {
    __syncthreads();
    if (threadIdx.x == 0) c.lengths[r] = min(start + a.T - first, cap);
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
  c.lengths[r] = min(start + a.T - first, cap);
}

// ============================================================================ read
// Thread = one code word (8 values) of K and of V.
template <int HD, bool F32>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvReadArgs a, int chunk, int chunks) {
  constexpr int LPU = HD / 8;
  const KvCache& c = a.c;
  const int i = blockIdx.x / chunks;
  const int r = row_of(c, a.rows, i);
  const int cap = c.max_pages << c.page_shift;
  const int len = r < 0 ? 0 : min(max(c.lengths[r], 0), cap);
  const int start = a.start != nullptr ? a.start[i] : 0;
  if (start < 0 && threadIdx.x == 0) record_error(c.err, MDL_ERR_BAD_INDEX);
  const int t0 = (blockIdx.x - i * chunks) * chunk, nt = min(chunk, a.count - t0);
  const int units = nt * c.G;
  const int sub = threadIdx.x % LPU;
  for (int u = threadIdx.x / LPU; u < units; u += kThreads / LPU) {
    const int g = u / nt, t = t0 + u % nt;
    const long long pos = static_cast<long long>(start) + t;
    uint32_t w[2] = {0x88888888u, 0x88888888u};
    float s[2] = {0.f, 0.f};
    if (pos >= 0 && pos < len) {
      const int pg = page_of(c, r, static_cast<int>(pos));
      if (pg >= 0) {
        const int slot = static_cast<int>(pos) & ((1 << c.page_shift) - 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const long long b = slot_base(c, pg, g, kv) + slot;
          w[kv] = reinterpret_cast<const uint32_t*>(c.codes)[b * LPU + sub];
          s[kv] = __bfloat162float(c.scales[b]);
        }
      }
    }
    const long long off = (static_cast<long long>(i) * a.count + t) * (c.G * HD) + g * HD + sub * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[kv] * static_cast<float>(static_cast<int>((w[kv] >> (4 * e)) & 15u) - 8);
      void* out = kv ? a.out_v : a.out_k;
      if constexpr (F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(out) + off);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + off) =
            make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
      }
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
// by memory, not by the products.
//
// Codes to bf16: (w >> 4i) & 0x000F000F | 0x4300_4300 is the exact bf16 pair (128 + nibble i,
// 128 + nibble i + 4) = 136 + c. K uses it as it is: S = q . (136 + c) - 136 * sum(q), the
// second term being the accumulator's initial value. V subtracts 136 (one packed, exact
// operation), since the same shortcut over a long sum of keys would cancel. The scales enter
// in fp32: s_k multiplies the scores, s_v the probabilities.
//
// Which key sits in which row of a 16-key tile is free as long as both products agree: lane
// group g8 = lane / 4 owns 2 KT neighbouring keys of a step, so a lane's scales are one load
// and its K rows neighbouring 32-byte sectors.
constexpr uint32_t kMagic = 0x43004300u;   // bf16 128, twice
constexpr uint32_t kOffset = 0x43084308u;  // bf16 136, twice

__device__ __forceinline__ uint32_t code_pair(uint32_t w) { return (w & 0x000F000Fu) | kMagic; }

__device__ __forceinline__ uint32_t code_pair_signed(uint32_t w) {
  const uint32_t u = code_pair(w), o = kOffset;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&o));
  return *reinterpret_cast<const uint32_t*>(&r);
}

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

template <int HD, int KT>
struct Step {  // a lane's share of one step of 16 * KT keys
  uint32_t k[2 * KT][HD / 32];  // its 2 KT keys, dims of lane % 4
  uint32_t v[4 * KT];           // 4 KT keys of the other product, the word of its dims
  uint32_t ks[KT], vs[KT];      // scales of its 2 KT keys (bf16 pairs)
};

template <int HD, int NT, int WPI>
__global__ void __launch_bounds__(WPI == 1 ? 128 : 32 * WPI) kv_attend_kernel(KvAttendArgs a, int qblocks, int splits) {
  constexpr int KT = NT == 4 ? 2 : 4;   // 16-key tiles a step
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
  float init[NT][2];
  int qn[NT][2];  // query index n of columns 2t, 2t + 1
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
      init[nt][e] = -136.f * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
      qn[nt][e] = min(m0 + nt * 8 + 2 * t + e, M - 1) / group;
    }
  }
  const float scale2 = a.scale * 1.4426950408889634f;

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
      cw = max(0, qmin - W + 1) / CH;
      cs = min((min(S, hi) + CH - 1) / CH, cw);
    }
    total = cs + end - cw;
  }
  auto step_key = [&](int i) { return (i < cs ? i : cw + i - cs) * CH; };
  // page of the lane's K keys and of its V keys; 0 (any valid page) past the length
  auto pages = [&](int i, int& pk, int& pv) {
    const int k0 = step_key(i);
    const int a0 = k0 + 2 * KT * g8, a1 = k0 + 4 * KT * t;
    pk = a0 < len ? max(page_of(c, r, a0), 0) : 0;
    pv = a1 < len ? max(page_of(c, r, a1), 0) : 0;
  };
  auto load = [&](int i, int pk, int pv, Step<HD, KT>& s) {
    const int mask = (1 << c.page_shift) - 1;
    const int k0 = step_key(i);
    const int slot = (k0 + 2 * KT * g8) & mask;
    const long long bk = slot_base(c, pk, g, 0) + slot;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(c.codes) + bk * (HD / 8) + t * KW;
#pragma unroll
    for (int e = 0; e < 2 * KT; ++e) {
      if constexpr (KW == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(kp + e * (HD / 8));
        s.k[e][0] = x.x;
        s.k[e][1] = x.y;
      } else {
        s.k[e][0] = kp[e * (HD / 8)];
      }
    }
    const __nv_bfloat16* sp = c.scales + bk;
    const __nv_bfloat16* sv = sp + (1 << c.page_shift);  // V follows K
    if constexpr (KT == 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(sp), y = *reinterpret_cast<const uint4*>(sv);
      s.ks[0] = x.x; s.ks[1] = x.y; s.ks[2] = x.z; s.ks[3] = x.w;
      s.vs[0] = y.x; s.vs[1] = y.y; s.vs[2] = y.z; s.vs[3] = y.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(sp), y = *reinterpret_cast<const uint2*>(sv);
      s.ks[0] = x.x; s.ks[1] = x.y;
      s.vs[0] = y.x; s.vs[1] = y.y;
    }
    const long long bv = slot_base(c, pv, g, 1) + ((k0 + 4 * KT * t) & mask);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(c.codes) + bv * (HD / 8) + (HD == 64 ? g8 : g8 >> 1);
#pragma unroll
    for (int e = 0; e < 4 * KT; ++e) s.v[e] = vp[e * (HD / 8)];
  };

  Step<HD, KT> cur;
  int pk = 0, pv = 0;
  if (part < total) {
    pages(part, pk, pv);
    load(part, pk, pv, cur);
    if (part + parts < total) pages(part + parts, pk, pv);
  }
  for (int i = part; i < total; i += parts) {
    const Step<HD, KT> s = cur;
    if (i + parts < total) {
      load(i + parts, pk, pv, cur);
      if (i + 2 * parts < total) pages(i + 2 * parts, pk, pv);
    }
    const int k0 = step_key(i);
    float x[KT][NT][4];
#pragma unroll
    for (int j = 0; j < KT; ++j) {
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t wa = s.k[2 * j][w], wb = s.k[2 * j + 1][w];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a0 = code_pair(wa >> (8 * h)), a1 = code_pair(wb >> (8 * h));
          const uint32_t a2 = code_pair(wa >> (8 * h + 4)), a3 = code_pair(wb >> (8 * h + 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int ks = 2 * w + h;
            if (ks == 0)
              mma16816(x[j][nt], a0, a1, a2, a3, qf[nt][ks][0], qf[nt][ks][1], init[nt][0], init[nt][1], init[nt][0],
                       init[nt][1]);
            else
              mma16816(x[j][nt], a0, a1, a2, a3, qf[nt][ks][0], qf[nt][ks][1], x[j][nt][0], x[j][nt][1], x[j][nt][2],
                       x[j][nt][3]);
          }
        }
      }
      const float s0 = bf16_lo(s.ks[j]) * scale2, s1 = bf16_hi(s.ks[j]) * scale2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        x[j][nt][0] *= s0;
        x[j][nt][1] *= s0;
        x[j][nt][2] *= s1;
        x[j][nt][3] *= s1;
      }
    }
    // every key of the step visible to every query of the block?
    const bool whole = k0 + CH <= min(len, qmin + 1) && (W == 0 || k0 > qmax - W || k0 + CH <= S);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kp = k0 + 2 * KT * g8 + 2 * j + (e >> 1);
            const int qp = base + qn[nt][e & 1];
            const bool vis = kp < len && kp <= qp && (W == 0 || qp - kp < W || kp < S);
            if (!vis) x[j][nt][e] = -CUDART_INF_F;
          }
    }
    float lm[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < KT; ++j) v = fmaxf(v, fmaxf(x[j][nt][e], x[j][nt][e + 2]));
        lm[nt][e] = v;
        grow |= v > mx[nt][e] + 8.f;
      }
    if (__any_sync(0xffffffffu, grow)) raise(lm);
    float use[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) use[nt][e] = mx[nt][e] == -CUDART_INF_F ? 0.f : mx[nt][e];
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      uint32_t pb[NT][2];
      const float v0 = bf16_lo(s.vs[j]), v1 = bf16_hi(s.vs[j]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = x[j][nt][e];
          p[e] = ex2(y - use[nt][e & 1]);
          l[nt][e & 1] += p[e];
          p[e] *= e < 2 ? v0 : v1;
          // the scale of a hidden key may be anything, a NaN too
          if (!whole && y == -CUDART_INF_F) p[e] = 0.f;
        }
        pb[nt][0] = transpose8(pack_bf16(p[0], p[1]));
        pb[nt][1] = transpose8(pack_bf16(p[2], p[3]));
      }
      // keys in tile rows 2t, 2t+1, 2t+8, 2t+9
      const uint32_t va = s.v[2 * j], vb = s.v[2 * KT + 2 * j], vc = s.v[2 * j + 1], vd = s.v[2 * KT + 2 * j + 1];
      if constexpr (HD == 64) {
        const uint32_t lo0 = __byte_perm(va, vb, 0x5410), hi0 = __byte_perm(va, vb, 0x7632);
        const uint32_t lo1 = __byte_perm(vc, vd, 0x5410), hi1 = __byte_perm(vc, vd, 0x7632);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint32_t a0 = code_pair_signed(lo0 >> (4 * mt)), a1 = code_pair_signed(hi0 >> (4 * mt));
          const uint32_t a2 = code_pair_signed(lo1 >> (4 * mt)), a3 = code_pair_signed(hi1 >> (4 * mt));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1], o[mt][nt][0], o[mt][nt][1], o[mt][nt][2],
                     o[mt][nt][3]);
        }
      } else {
        const uint32_t sel = (g8 & 1) ? 0x7632 : 0x5410;
        const uint32_t u0 = __byte_perm(va, vb, sel), u1 = __byte_perm(vc, vd, sel);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint32_t a0 = code_pair_signed(u0 >> (8 * mt)), a1 = code_pair_signed(u0 >> (8 * mt + 4));
          const uint32_t a2 = code_pair_signed(u1 >> (8 * mt)), a3 = code_pair_signed(u1 >> (8 * mt + 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1], o[mt][nt][0], o[mt][nt][1], o[mt][nt][2],
                     o[mt][nt][3]);
        }
      }
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
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kp = k0 + g8 + 8 * (e >> 1), n = qn[nt][e & 1];
          const bool vis = kp <= n && (W == 0 || n - kp < W || len + kp < S);
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
    extern __shared__ float sm[];
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

// Joins the splits: hd / 4 threads a query row.
template <int HD>
__global__ void __launch_bounds__(128) kv_combine_kernel(KvAttendArgs a, int qblocks, int splits, int cols) {
  const int group = a.H / a.c.G, M = a.N * group;
  const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long row = idx / (HD / 4);
  const int d4 = static_cast<int>(idx % (HD / 4));
  if (row >= static_cast<long long>(a.B) * a.c.G * M) return;
  const int m = static_cast<int>(row % M);
  const long long bg = row / M;
  const int g = static_cast<int>(bg % a.c.G);
  const long long b = bg / a.c.G;
  const float* src = a.partial + ((bg * qblocks + m / cols) * splits * cols + m % cols) * (HD + 4);
  const long long step = static_cast<long long>(cols) * (HD + 4);
  float top = -CUDART_INF_F;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, src[s * step + HD]);
  const float use = top == -CUDART_INF_F ? 0.f : top;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float f = ex2(src[s * step + HD] - use);
    const float4 y = *reinterpret_cast<const float4*>(src + s * step + 4 * d4);
    sum = fmaf(src[s * step + HD + 1], f, sum);
    acc.x = fmaf(y.x, f, acc.x);
    acc.y = fmaf(y.y, f, acc.y);
    acc.z = fmaf(y.z, f, acc.z);
    acc.w = fmaf(y.w, f, acc.w);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat16* dst = a.out + (b * a.N + m / group) * a.H * HD + (g * group + m % group) * HD + 4 * d4;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

int num_sms() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

struct Plan {
  int nt, wpi, qblocks, splits;
  long long items;
};

// Query rows a block: 8, 16 or 32. One warp an item where the items alone fill the device and
// each has few keys; else eight warps an item, and several blocks an item while the items
// leave multiprocessors idle.
Plan plan_of(const KvAttendArgs& a) {
  Plan p;
  const int M = a.N * (a.H / a.c.G);
  p.nt = M <= 8 ? 1 : (M <= 16 ? 2 : 4);
  p.qblocks = (M + 8 * p.nt - 1) / (8 * p.nt);
  p.items = static_cast<long long>(a.B) * a.c.G * p.qblocks;
  const long long cap = static_cast<long long>(a.c.max_pages) << a.c.page_shift;
  const long long keys = a.window > 0 ? std::min<long long>(cap, static_cast<long long>(a.window) + a.sinks) : cap;
  static const int sms = num_sms();
  p.wpi = (p.items >= 16LL * sms && keys <= 4096) ? 1 : 8;
  p.splits = 1;
  if (p.wpi == 8) {
    const long long want = (2LL * sms + p.items - 1) / p.items;
    const long long most = std::max<long long>(1, keys / (8 * 64));
    p.splits = static_cast<int>(std::max<long long>(1, std::min<long long>({want, most, 64})));
  }
  return p;
}

template <int HD, int NT>
cudaError_t launch_attend(const KvAttendArgs& a, const Plan& p, cudaStream_t stream) {
  if (p.wpi == 1) {
    kv_attend_kernel<HD, NT, 1><<<static_cast<unsigned>((p.items + 3) / 4), 128, 0, stream>>>(a, p.qblocks, 1);
  } else {
    constexpr int smem = 8 * 8 * NT * (HD + 6) * 4;
    if constexpr (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kv_attend_kernel<HD, NT, 8>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
    }
    kv_attend_kernel<HD, NT, 8>
        <<<static_cast<unsigned>(p.items * p.splits), 256, smem, stream>>>(a, p.qblocks, p.splits);
  }
  return cudaGetLastError();
}

template <int HD>
cudaError_t attend_hd(const KvAttendArgs& a, const Plan& p, cudaStream_t stream, int* launches) {
  cudaError_t e = p.nt == 1 ? launch_attend<HD, 1>(a, p, stream)
                            : (p.nt == 2 ? launch_attend<HD, 2>(a, p, stream) : launch_attend<HD, 4>(a, p, stream));
  *launches += 1;
  if (e != cudaSuccess || p.splits == 1) return e;
  const long long threads = static_cast<long long>(a.B) * a.N * a.H * (HD / 4);
  kv_combine_kernel<HD><<<static_cast<unsigned>((threads + 127) / 128), 128, 0, stream>>>(a, p.qblocks, p.splits,
                                                                                         8 * p.nt);
  *launches += 1;
  return cudaGetLastError();
}

}  // namespace

cudaError_t kv_write(const KvWriteArgs& a, cudaStream_t stream, int* launches) {
  if (a.n == 0) return cudaSuccess;
  constexpr int kChunk = 64;
  const int chunks = std::max(1, (a.T + kChunk - 1) / kChunk);
  if (static_cast<long long>(chunks) * a.n > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(chunks) * a.n;
  if (a.c.hd == 64)
    kv_write_kernel<64><<<grid, kThreads, 0, stream>>>(a, kChunk, chunks);
  else
    kv_write_kernel<32><<<grid, kThreads, 0, stream>>>(a, kChunk, chunks);
  *launches += 1;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || chunks == 1) return e;
  kv_length_kernel<<<(a.n + 127) / 128, 128, 0, stream>>>(a);
  *launches += 1;
  return cudaGetLastError();
}

cudaError_t kv_read(const KvReadArgs& a, cudaStream_t stream) {
  if (a.n == 0 || a.count == 0) return cudaSuccess;
  constexpr int kChunk = 64;
  const int chunks = (a.count + kChunk - 1) / kChunk;
  if (static_cast<long long>(chunks) * a.n > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(chunks) * a.n;
  auto kern = a.c.hd == 64 ? (a.fp32 ? kv_read_kernel<64, true> : kv_read_kernel<64, false>)
                           : (a.fp32 ? kv_read_kernel<32, true> : kv_read_kernel<32, false>);
  kern<<<grid, kThreads, 0, stream>>>(a, kChunk, chunks);
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
