// Sliding-window attention with always-visible first tokens (sinks) on the 5th-generation
// tensor cores. Contract: window_attn.h.
//
// Tiles are 128 token rows counted from a sample's FIRST VALID token (row kst + 128 t): padding
// is never loaded, the sinks lie in the first tile(s), and only the diagonal tile and the tile
// that the window's lower edge cuts need a mask. A query tile visits the tiles of the sinks and
// then those of its window, so the cost grows with the window and not with the history.
//
// Forward (192 threads, two persistent CTAs an SM, 256 TMEM columns each: S 128, P 64, O 64).
// Work item = sample, head, query tile.
//   warp 0     TMA: Q, and K / V tiles of 128 rows in two-stage rings
//   warp 1     MMA: S = Q K^T; O += P V with P as the A operand straight from TMEM
//   warps 2-5  softmax, thread = query row: P = exp2(S * c - m) as bf16 into TMEM. m is a
//              reference that moves only when a score passes it by more than 8 (exp2 of the
//              excess stays below 256), so O is rarely rescaled and is read once, at the end.
// S of the next tile is issued as soon as the softmax holds the present one in registers.
//
// Backward, two launches of one kernel (320 threads, one persistent CTA an SM, 512 columns):
// a stationary tile of 128 rows meets a stream of 64-row tiles,
//   S = A1 B1^T, dP = A2 B2^T, P = exp2(S * c - lse), dS = P * (dP - D),
//   queries stationary: A = Q, dO; B = K, V;  dQ += dS K;  D = rowsum(dO * O) on the way
//   keys stationary:    A = K, V;  B = Q, dO; dV += P dO, dK += dS Q  (all transposed; the query
//                       heads that share the key head follow one another)
// Two warpgroups take the stream's steps in turn, each with its own S, dP, P and dS columns, so
// that the products of one run under the exponentials of the other. Recomputing S and dP in
// both launches costs two products more than one launch that adds dQ to memory would, and needs
// no fp32 buffer, no clearing, no atomics: every sum has one owner and one order.
//
// Every wait is bounded (error word + abort flag) and every role drains what it has in flight
// before the CTA exits.
#include "window_attn.h"

#include <cudaTypedefs.h>
#include <math_constants.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"

namespace mdl {
namespace {

constexpr int TILE = 128;               // rows of a stationary tile and of a forward key tile
constexpr int HALF = 64;                // rows of a streamed tile of the backward
constexpr int TILE_BYTES = TILE * 128;  // 128-byte rows: 64 columns, the head's hd first
constexpr int HALF_BYTES = HALF * 128;
constexpr float kLog2e = 1.4426950408889634f;

constexpr int F_THREADS = 192, F_TMEM = 256;
constexpr int F_SMEM = 1024 + 5 * TILE_BYTES + 256;
constexpr int B_THREADS = 320, B_TMEM = 512;
constexpr int B_STAGES = 4;
// stationary pair [2] | streamed pair [4] | lse, D of the streamed rows [4][64] | barriers
constexpr int B_SMEM = 1024 + 4 * TILE_BYTES + 2 * B_STAGES * HALF_BYTES + B_STAGES * 2 * HALF * 4 + 256;
static_assert(2 * F_SMEM <= 227 * 1024 && B_SMEM <= 227 * 1024, "shared memory budget");

struct Params {
  __nv_bfloat16* out;
  float* lse;
  const int* kstart;
  const __nv_bfloat16* dout;
  __nv_bfloat16* dqkv;
  float* dsum;
  int B, H, G, Lk, Lq, hd, window, sinks;
  int tiles;  // work items a (sample, head): query tiles or key tiles
  float scale, scale2;
  int* err;
};

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~static_cast<uintptr_t>(1023));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 32 consecutive fp32 TMEM columns of this thread's lane, no wait.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem, bf16 pairs along K] * B[smem desc]^T.
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// K-major operand, 128-byte swizzle: 16-element K step ks inside the row.
__device__ __forceinline__ uint64_t desc_k(uint32_t base, int ks) { return make_smem_desc(base + ks * 32, 16, 1024); }
// MN-major operand (rows = K, 64 contiguous MN elements a 128-byte row): K step ks = 16 rows.
__device__ __forceinline__ uint64_t desc_mn(uint32_t base, int ks) {
  return make_smem_desc(base + ks * 2048, TILE_BYTES, 1024);
}

// A wait whose outcome is the same on every lane of the warp (.sync.aligned code follows).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  const bool ok = mbar_wait(bar, parity, err, abort_flag);
  return __all_sync(0xffffffffu, ok);
}

// Bits [l, h] (inclusive, clipped) of 32-column word w.
__device__ __forceinline__ uint32_t range_bits(int l, int h, int w) {
  const int a = max(l - 32 * w, 0), b = min(h - 32 * w, 31);
  if (a > b) return 0u;
  return (0xFFFFFFFFu >> (31 - b)) & (0xFFFFFFFFu << a);
}

// One row of hd zeros (bf16).
__device__ __forceinline__ void zero_row(__nv_bfloat16* dst, int hd) {
  for (int c = 0; c < hd / 8; ++c) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0, 0, 0, 0);
}

// ============================================================================ work items
// Positions below are relative to the sample's first valid token.
struct Item {
  int b, h, i;      // sample, head (query head, or key head), index within the pair
  int kst, len, qf; // first valid token, valid tokens, first query
  int t;            // tile
  int cs, k0, n;    // steps: cs from 0, then from k0 on; n in all (0: nothing to do)
};

__device__ __forceinline__ Item item_base(const Params& p, int w, int heads) {
  Item it;
  it.h = w % heads;
  const int rest = w / heads;
  it.b = rest % p.B;
  it.i = rest / p.B;
  it.kst = min(max(p.kstart[it.b], 0), p.Lk);
  it.len = p.Lk - it.kst;
  it.qf = max(0, p.Lk - p.Lq - it.kst);
  it.cs = it.k0 = it.n = 0;
  return it;
}

// Query tile i, counted from the last; key steps of `rows` rows.
__device__ __forceinline__ Item query_item(const Params& p, int w, int rows) {
  Item it = item_base(p, w, p.H);
  it.t = (it.len + TILE - 1) / TILE - 1 - it.i;
  if (it.t < 0 || TILE * (it.t + 1) <= it.qf) return it;
  const int end = (min(TILE * (it.t + 1), it.len) + rows - 1) / rows;
  it.k0 = max(0, max(TILE * it.t, it.qf) - p.window + 1) / rows;
  it.cs = min((min(p.sinks, it.len) + rows - 1) / rows, it.k0);
  it.n = it.cs + end - it.k0;
  return it;
}

// Key tile i (the sinks' first: every query sees it); query steps of 64 rows, per query head
// of the group.
__device__ __forceinline__ Item key_item(const Params& p, int w) {
  Item it = item_base(p, w, p.G);
  it.t = it.i;
  if (TILE * it.t >= it.len) return it;
  const int qs = max(TILE * it.t, it.qf);
  const int qe = TILE * it.t < p.sinks ? it.len : min(it.len, TILE * it.t + TILE - 1 + p.window);
  it.k0 = qs / HALF;
  it.cs = qe > qs ? (qe + HALF - 1) / HALF - it.k0 : 0;  // steps a query head
  it.n = it.cs * (p.H / p.G);
  return it;
}

// ============================================================================ forward
template <int HD>
__global__ void __launch_bounds__(F_THREADS, 2)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv,
                      const Params p, int num_items) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = align1024(smem_raw);
  uint8_t* sK = sQ + TILE_BYTES;      // [2]
  uint8_t* sV = sK + 2 * TILE_BYTES;  // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * TILE_BYTES);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;   // [2]
  uint64_t* k_empty = bars + 4;  // [2]
  uint64_t* v_full = bars + 6;   // [2]
  uint64_t* v_empty = bars + 8;  // [2]
  uint64_t* s_full = bars + 10;
  uint64_t* s_empty = bars + 11;
  uint64_t* p_full = bars + 12;
  uint64_t* pv_done = bars + 13;
  uint64_t* done = bars + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_empty, 4);
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, F_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tP = tmem + 128, tO = tmem + 192;
  auto tile_of = [](const Item& it, int j) { return j < it.cs ? j : it.k0 + j - it.cs; };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_kv);
      const int q0 = p.Lk - p.Lq;
      int items = 0, g = 0, k_issued = 0, v_issued = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
        const Item it = query_item(p, w, TILE);
        if (it.n == 0) continue;
        const int kvh = it.h / (p.H / p.G);
        if (items >= 1 && !mbar_wait(q_empty, (items - 1) & 1, p.err, abort_flag)) break;
        mbar_arrive_expect_tx(q_full, TILE_BYTES);
        tma_load_3d(sQ, &tm_q, q_full, it.h * HD, it.kst + TILE * it.t - q0, it.b);
        ++items;
        for (int j = 0; j < it.n; ++j, ++g) {
          const int st = g & 1;
          const int y = it.kst + TILE * tile_of(it, j);
          if (g >= 2 && !mbar_wait(&k_empty[st], ((g >> 1) - 1) & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&k_full[st], TILE_BYTES);
          tma_load_3d(sK + st * TILE_BYTES, &tm_kv, &k_full[st], (p.H + kvh) * HD, y, it.b);
          k_issued = g + 1;
          if (g >= 2 && !mbar_wait(&v_empty[st], ((g >> 1) - 1) & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&v_full[st], TILE_BYTES);
          tma_load_3d(sV + st * TILE_BYTES, &tm_kv, &v_full[st], (p.H + p.G + kvh) * HD, y, it.b);
          v_issued = g + 1;
        }
      }
      // every copy into this CTA's smem has landed before the CTA may exit
      if (items > 0) mbar_wait(q_full, (items - 1) & 1, nullptr, nullptr);
      for (int j = max(0, k_issued - 2); j < k_issued; ++j) mbar_wait(&k_full[j & 1], (j >> 1) & 1, nullptr, nullptr);
      for (int j = max(0, v_issued - 2); j < v_issued; ++j) mbar_wait(&v_full[j & 1], (j >> 1) & 1, nullptr, nullptr);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_bf16(TILE, TILE, false, false);
      constexpr uint32_t idesc_pv = make_idesc_bf16(TILE, 64, false, true);
      const uint32_t q_base = smem_u32(sQ), k_base = smem_u32(sK), v_base = smem_u32(sV);
      bool ok = true;
      int items = 0, g0 = 0;
      auto issue_s = [&](int g, bool last) -> bool {
        if (!mbar_wait(&k_full[g & 1], (g >> 1) & 1, p.err, abort_flag) ||
            (g > 0 && !mbar_wait(s_empty, (g - 1) & 1, p.err, abort_flag)))
          return false;
        tc_fence_after();
        const uint32_t kb = k_base + (g & 1) * TILE_BYTES;
        for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tS, desc_k(q_base, ks), desc_k(kb, ks), idesc_s, ks);
        tc_commit(&k_empty[g & 1]);
        tc_commit(s_full);
        if (last) tc_commit(q_empty);
        return true;
      };
      for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
        const Item it = query_item(p, w, TILE);
        if (it.n == 0) continue;
        if (!mbar_wait(q_full, items & 1, p.err, abort_flag) || !issue_s(g0, it.n == 1)) break;
        ++items;
        for (int j = 0; j < it.n; ++j) {
          const int g = g0 + j;
          if (j + 1 < it.n && !issue_s(g + 1, j + 2 == it.n)) {
            ok = false;
            break;
          }
          if (!mbar_wait(p_full, g & 1, p.err, abort_flag) ||
              !mbar_wait(&v_full[g & 1], (g >> 1) & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (int ks = 0; ks < 8; ++ks)
            tc_mma_bf16_ts(tO, tP + ks * 8, desc_mn(v_base + (g & 1) * TILE_BYTES, ks), idesc_pv,
                           (j > 0 || ks > 0) ? 1u : 0u);
          tc_commit(pv_done);
          tc_commit(&v_empty[g & 1]);
        }
        g0 += it.n;
      }
      // all MMAs have finished before TMEM is released
      tc_commit(done);
      mbar_wait(done, 0, nullptr, nullptr);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    bool ok = true;
    int g0 = 0;
    for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
      const Item it = query_item(p, w, TILE);
      const long long orow0 = static_cast<long long>(it.b) * p.Lq;
      float* lse = p.lse + (static_cast<long long>(it.b) * p.H + it.h) * p.Lq;
      // queries before the first valid token (a share of them per item)
      for (int q = it.i * TILE + r; q < min(p.Lq, it.kst - (p.Lk - p.Lq)); q += p.tiles * TILE) {
        zero_row(p.out + (orow0 + q) * p.H * HD + it.h * HD, HD);
        lse[q] = CUDART_INF_F;
      }
      if (it.n == 0) continue;
      const int qp = TILE * it.t + r;
      float m = -CUDART_INF_F, l = 0.f;
      for (int j = 0; j < it.n; ++j) {
        const int g = g0 + j;
        const int kt = tile_of(it, j);
        if (!warp_wait(s_full, g & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[TILE];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + lane_off + c * 32, sr + c * 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty);
        // the diagonal, and what the window's lower edge cuts of tiles that are not all sinks
        if (kt == it.t || (TILE * (it.t - kt) + TILE > p.window && TILE * (kt + 1) > p.sinks)) {
          const int d = qp - TILE * kt;  // columns up to d are not in the future
          const int lo = d - p.window + 1, sk = min(d, p.sinks - 1 - TILE * kt);
#pragma unroll
          for (int w4 = 0; w4 < 4; ++w4) {
            const uint32_t vm = range_bits(lo, d, w4) | range_bits(0, sk, w4);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!((vm >> c) & 1u)) sr[32 * w4 + c] = __float_as_uint(-CUDART_INF_F);
          }
        }
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = __uint_as_float(sr[k]);
#pragma unroll
        for (int c = 8; c < TILE; ++c) mx8[c & 7] = fmaxf(mx8[c & 7], __uint_as_float(sr[c]));
        const float mx = p.scale2 * fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                                          fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
        const bool grow = mx > m + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = fmaxf(m, mx);
          const float alpha = m_new == -CUDART_INF_F ? 1.f : ex2(m - m_new);
          m = m_new;
          l *= alpha;
          if (j > 0) {
            if (!warp_wait(pv_done, (g - 1) & 1, p.err, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t ov[32];
              tmem_ld32(tO + lane_off + c * 32, ov);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; ++d) ov[d] = __float_as_uint(__uint_as_float(ov[d]) * alpha);
              tmem_st32(tO + lane_off + c * 32, ov);
            }
          }
        }
        const float m_use = m == -CUDART_INF_F ? 0.f : m;
        float sum8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < TILE; c += 2) {
          const float e0 = ex2(fmaf(__uint_as_float(sr[c]), p.scale2, -m_use));
          const float e1 = ex2(fmaf(__uint_as_float(sr[c + 1]), p.scale2, -m_use));
          sum8[c & 7] += e0;
          sum8[(c + 1) & 7] += e1;
          sr[c / 2] = pack2(e0, e1);
        }
        l += ((sum8[0] + sum8[1]) + (sum8[2] + sum8[3])) + ((sum8[4] + sum8[5]) + (sum8[6] + sum8[7]));
        if (g > 0 && !warp_wait(pv_done, (g - 1) & 1, p.err, abort_flag)) {  // the last P was consumed
          ok = false;
          break;
        }
        tc_fence_after();
        tmem_st32(tP + lane_off, sr);
        tmem_st32(tP + lane_off + 32, sr + 32);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (!ok) break;
      g0 += it.n;
      if (!warp_wait(pv_done, (g0 - 1) & 1, p.err, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int qi = it.kst + qp - (p.Lk - p.Lq);
      const bool real = qi >= 0 && qi < p.Lq;
      const float inv = 1.f / l;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t ov[32];
        tmem_ld32(tO + lane_off + c * 32, ov);
        tmem_wait_ld();
        if (real) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + (orow0 + qi) * p.H * HD + it.h * HD + c * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dst[e] = make_uint4(pack2(__uint_as_float(ov[8 * e]) * inv, __uint_as_float(ov[8 * e + 1]) * inv),
                                pack2(__uint_as_float(ov[8 * e + 2]) * inv, __uint_as_float(ov[8 * e + 3]) * inv),
                                pack2(__uint_as_float(ov[8 * e + 4]) * inv, __uint_as_float(ov[8 * e + 5]) * inv),
                                pack2(__uint_as_float(ov[8 * e + 6]) * inv, __uint_as_float(ov[8 * e + 7]) * inv));
        }
      }
      tc_fence_before();
      if (real) lse[qi] = m + lg2(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, F_TMEM);
  }
}

// ============================================================================ backward
// KEYS: the stationary tile holds keys (dK, dV), else queries (dQ and D).
template <int HD, bool KEYS>
__global__ void __launch_bounds__(B_THREADS, 1)
    window_bwd_kernel(const __grid_constant__ CUtensorMap tm_a1, const __grid_constant__ CUtensorMap tm_a2,
                      const __grid_constant__ CUtensorMap tm_b1, const __grid_constant__ CUtensorMap tm_b2,
                      const Params p, int num_items) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sA1 = smem;                                // [2]
  uint8_t* sA2 = sA1 + 2 * TILE_BYTES;                // [2]
  uint8_t* sB1 = sA2 + 2 * TILE_BYTES;                // [4]
  uint8_t* sB2 = sB1 + B_STAGES * HALF_BYTES;         // [4]
  float* sLse = reinterpret_cast<float*>(sB2 + B_STAGES * HALF_BYTES);  // [4][64]
  float* sD = sLse + B_STAGES * HALF;                                  // [4][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sD + B_STAGES * HALF);
  uint64_t* a_full = bars;        // [2]
  uint64_t* a_empty = bars + 2;   // [2]
  uint64_t* b_full = bars + 4;    // [4]
  uint64_t* b_empty = bars + 8;   // [4]
  uint64_t* s_full = bars + 12;   // [2]
  uint64_t* s_empty = bars + 14;  // [2]
  uint64_t* p_full = bars + 16;   // [2]
  uint64_t* p_empty = bars + 18;  // [2]
  uint64_t* acc_full = bars + 20;
  uint64_t* acc_empty = bars + 21;
  uint64_t* done = bars + 22;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 4);
      mbar_init(&p_full[s], 4);
      mbar_init(&p_empty[s], 1);
    }
    for (int s = 0; s < B_STAGES; ++s) {
      mbar_init(&b_full[s], KEYS ? 33 : 1);  // TMA bytes (+ the 32 lanes that stage lse and D)
      mbar_init(&b_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 8);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, B_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // per warpgroup: S, dP (64 fp32 columns each), P, dS (32 columns of bf16 pairs); accumulators
  auto tS = [&](int s) { return tmem + s * 128; };
  auto tP = [&](int s) { return tmem + 256 + s * 64; };
  const uint32_t tAcc0 = tmem + 384, tAcc1 = tmem + 448;
  const int group = p.H / p.G, q0 = p.Lk - p.Lq;
  auto item_of = [&](int w) { return KEYS ? key_item(p, w) : query_item(p, w, HALF); };
  // first row (relative) of step j, and the query head of it
  auto step_row = [&](const Item& it, int j) {
    return KEYS ? HALF * (it.k0 + j % it.cs) : HALF * (j < it.cs ? j : it.k0 + j - it.cs);
  };
  auto step_head = [&](const Item& it, int j) { return KEYS ? it.h * group + j / it.cs : it.h; };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_a1);
      tma_prefetch_desc(&tm_a2);
      tma_prefetch_desc(&tm_b1);
      tma_prefetch_desc(&tm_b2);
    }
    int items = 0, g = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
      const Item it = item_of(w);
      if (it.n == 0) continue;
      const int sa = items & 1;
      if (!warp_wait(&a_empty[sa], ((items >> 1) + 1) & 1, p.err, abort_flag)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&a_full[sa], 2 * TILE_BYTES);
        const int y = it.kst + TILE * it.t;
        if constexpr (KEYS) {
          tma_load_3d(sA1 + sa * TILE_BYTES, &tm_a1, &a_full[sa], (p.H + it.h) * HD, y, it.b);
          tma_load_3d(sA2 + sa * TILE_BYTES, &tm_a2, &a_full[sa], (p.H + p.G + it.h) * HD, y, it.b);
        } else {
          tma_load_3d(sA1 + sa * TILE_BYTES, &tm_a1, &a_full[sa], it.h * HD, y - q0, it.b);
          tma_load_3d(sA2 + sa * TILE_BYTES, &tm_a2, &a_full[sa], it.h * HD, y - q0, it.b);
        }
      }
      ++items;
      for (int j = 0; j < it.n; ++j, ++g) {
        const int st = g % B_STAGES;
        // parity of the previous use of this stage; a fresh barrier passes parity 1 at once
        if (!warp_wait(&b_empty[st], (g / B_STAGES + 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        const int rel = step_row(it, j), y = it.kst + rel, h = step_head(it, j);
        if (lane == 0) {
          mbar_arrive_expect_tx(&b_full[st], 2 * HALF_BYTES);
          if constexpr (KEYS) {
            tma_load_3d(sB1 + st * HALF_BYTES, &tm_b1, &b_full[st], h * HD, y - q0, it.b);
            tma_load_3d(sB2 + st * HALF_BYTES, &tm_b2, &b_full[st], h * HD, y - q0, it.b);
          } else {
            const int kvh = h / group;
            tma_load_3d(sB1 + st * HALF_BYTES, &tm_b1, &b_full[st], (p.H + kvh) * HD, y, it.b);
            tma_load_3d(sB2 + st * HALF_BYTES, &tm_b2, &b_full[st], (p.H + p.G + kvh) * HD, y, it.b);
          }
        }
        if constexpr (KEYS) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = lane + 32 * e;
            const bool real = rel + c >= it.qf && rel + c < it.len;
            const long long off = (static_cast<long long>(it.b) * p.H + h) * p.Lq + (y + c - q0);
            sLse[st * HALF + c] = real ? p.lse[off] : CUDART_INF_F;
            sD[st * HALF + c] = real ? p.dsum[off] : 0.f;
          }
          mbar_arrive(&b_full[st]);
        }
      }
    }
    if (lane == 0) {
      for (int j = max(0, items - 2); j < items; ++j) mbar_wait(&a_full[j & 1], (j >> 1) & 1, nullptr, nullptr);
      for (int j = max(0, g - B_STAGES); j < g; ++j)
        mbar_wait(&b_full[j % B_STAGES], (j / B_STAGES) & 1, nullptr, nullptr);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_bf16(TILE, HALF, false, false);
      constexpr uint32_t idesc_acc = make_idesc_bf16(TILE, 64, false, true);
      int items = 0, g0 = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
        const Item it = item_of(w);
        if (it.n == 0) continue;
        const int sa = items & 1;
        const uint32_t a1 = smem_u32(sA1 + sa * TILE_BYTES), a2 = smem_u32(sA2 + sa * TILE_BYTES);
        if (!mbar_wait(&a_full[sa], (items >> 1) & 1, p.err, abort_flag)) break;
        auto issue_s = [&](int g) -> bool {
          const int st = g % B_STAGES, s = g & 1;
          if (!mbar_wait(&b_full[st], (g / B_STAGES) & 1, p.err, abort_flag) ||
              (g >= 2 && !mbar_wait(&s_empty[s], ((g >> 1) - 1) & 1, p.err, abort_flag)))
            return false;
          tc_fence_after();
          const uint32_t b1 = smem_u32(sB1 + st * HALF_BYTES), b2 = smem_u32(sB2 + st * HALF_BYTES);
          for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tS(s), desc_k(a1, ks), desc_k(b1, ks), idesc_s, ks);
          for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tS(s) + 64, desc_k(a2, ks), desc_k(b2, ks), idesc_s, ks);
          tc_commit(&s_full[s]);
          return true;
        };
        if (!issue_s(g0) || (it.n > 1 && !issue_s(g0 + 1))) break;
        for (int j = 0; j < it.n; ++j) {
          const int g = g0 + j, st = g % B_STAGES, s = g & 1;
          // S of two steps ahead goes to the columns that this step's warpgroup has emptied
          if (j + 2 < it.n && !issue_s(g + 2)) {
            ok = false;
            break;
          }
          if (!mbar_wait(&p_full[s], (g >> 1) & 1, p.err, abort_flag) ||
              (j == 0 && items >= 1 && !mbar_wait(acc_empty, (items - 1) & 1, p.err, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t b1 = smem_u32(sB1 + st * HALF_BYTES), b2 = smem_u32(sB2 + st * HALF_BYTES);
          for (int ks = 0; ks < HALF / 16; ++ks) {
            const uint32_t acc = (j > 0 || ks > 0) ? 1u : 0u;
            if constexpr (KEYS) tc_mma_bf16_ts(tAcc0, tP(s) + ks * 8, desc_mn(b2, ks), idesc_acc, acc);
            tc_mma_bf16_ts(tAcc1, tP(s) + 32 + ks * 8, desc_mn(b1, ks), idesc_acc, acc);
          }
          tc_commit(&p_empty[s]);
          tc_commit(&b_empty[st]);
        }
        if (!ok) break;
        tc_commit(acc_full);
        tc_commit(&a_empty[sa]);
        g0 += it.n;
        ++items;
      }
      tc_commit(done);
      mbar_wait(done, 0, nullptr, nullptr);
    }
  } else {
    // ------------------------------------------------------------ compute
    const int wg = (warp - 2) >> 2;  // takes the steps of its parity
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const int width = (p.H + 2 * p.G) * HD;
    bool ok = true;
    int items = 0, g0 = 0;
    for (int w = blockIdx.x; w < num_items && ok; w += gridDim.x) {
      const Item it = item_of(w);
      const long long trow0 = static_cast<long long>(it.b) * p.Lk;
      // gradients of what nobody sees or asks for (a share per item)
      if constexpr (KEYS) {
        for (int k = it.i * TILE + r; k < it.kst; k += p.tiles * TILE)
          zero_row(p.dqkv + (trow0 + k) * width + (wg == 0 ? p.H + p.G + it.h : p.H + it.h) * HD, HD);
      } else if (wg == 0) {
        for (int k = it.i * TILE + r; k < it.kst + it.qf; k += p.tiles * TILE)
          zero_row(p.dqkv + (trow0 + k) * width + it.h * HD, HD);
      }
      const int own = TILE * it.t + r;  // this thread's row
      if (it.n == 0) {
        if constexpr (KEYS) {  // valid keys without a query
          if (own < it.len)
            zero_row(p.dqkv + (trow0 + it.kst + own) * width + (wg == 0 ? p.H + p.G + it.h : p.H + it.h) * HD, HD);
        }
        continue;
      }
      float row_lse = CUDART_INF_F, row_d = 0.f;
      if constexpr (!KEYS) {
        const int qi = it.kst + own - q0;
        if (own >= it.qf && own < it.len) {
          const long long o = (static_cast<long long>(it.b) * p.Lq + qi) * p.H * HD + it.h * HD;
          float acc = 0.f;
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 ov = reinterpret_cast<const uint4*>(p.out + o)[c];
            const uint4 gv = reinterpret_cast<const uint4*>(p.dout + o)[c];
            const uint32_t a[4] = {ov.x, ov.y, ov.z, ov.w}, e[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              acc = fmaf(__uint_as_float(a[k] << 16), __uint_as_float(e[k] << 16), acc);
              acc = fmaf(__uint_as_float(a[k] & 0xFFFF0000u), __uint_as_float(e[k] & 0xFFFF0000u), acc);
            }
          }
          const long long s = (static_cast<long long>(it.b) * p.H + it.h) * p.Lq + qi;
          row_d = acc;
          row_lse = p.lse[s];
          if (wg == 0) p.dsum[s] = acc;
        }
      }
      for (int j = 0; j < it.n; ++j) {
        const int g = g0 + j;
        if ((g & 1) != wg) continue;
        const int st = g % B_STAGES;
        const int rel = step_row(it, j);
        if ((KEYS && !warp_wait(&b_full[st], (g / B_STAGES) & 1, p.err, abort_flag)) ||
            !warp_wait(&s_full[wg], (g >> 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[64], dp[64];
        tmem_ld32(tS(wg) + lane_off, s);
        tmem_ld32(tS(wg) + lane_off + 32, s + 32);
        tmem_ld32(tS(wg) + lane_off + 64, dp);
        tmem_ld32(tS(wg) + lane_off + 96, dp + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[wg]);
        // visible columns of this row: one or two intervals
        uint32_t vis[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        if constexpr (KEYS) {
          const bool whole = rel >= TILE * it.t + TILE - 1 && rel >= it.qf && rel + HALF <= it.len &&
                             (TILE * (it.t + 1) <= p.sinks || rel + HALF - TILE * it.t <= p.window);
          if (!whole) {
            const int lo = max(own, it.qf) - rel;
            const int hi = (own < p.sinks ? it.len - 1 : min(it.len - 1, own + p.window - 1)) - rel;
            vis[0] = range_bits(lo, hi, 0);
            vis[1] = range_bits(lo, hi, 1);
          }
        } else {
          const bool whole = rel + HALF - 1 <= TILE * it.t &&
                             (rel + HALF <= p.sinks || TILE * it.t + TILE - rel <= p.window);
          if (!whole) {
            const int d = own - rel;
            const int lo = d - p.window + 1, sk = min(d, p.sinks - 1 - rel);
            vis[0] = range_bits(lo, d, 0) | range_bits(0, sk, 0);
            vis[1] = range_bits(lo, d, 1) | range_bits(0, sk, 1);
          }
        }
        const float* lse = sLse + st * HALF;
        const float* dsv = sD + st * HALF;
        // P and dS take the registers of S and dP: pair c of each in word c
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          float pv[2], ds[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float lc = KEYS ? lse[c + e] : row_lse;
            const float dc = KEYS ? dsv[c + e] : row_d;
            const float x = ex2(fmaf(__uint_as_float(s[c + e]), p.scale2, -lc));
            const bool v = (vis[c >> 5] >> ((c + e) & 31)) & 1u;
            pv[e] = v ? x : 0.f;
            ds[e] = v ? x * (__uint_as_float(dp[c + e]) - dc) : 0.f;
          }
          if constexpr (KEYS) s[c / 2] = pack2(pv[0], pv[1]);
          dp[c / 2] = pack2(ds[0], ds[1]);
        }
        if (g >= 2 && !warp_wait(&p_empty[wg], ((g >> 1) - 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if constexpr (KEYS) tmem_st32(tP(wg) + lane_off, s);
        tmem_st32(tP(wg) + lane_off + 32, dp);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[wg]);
      }
      if (!ok) break;
      g0 += it.n;
      if (!warp_wait(acc_full, items & 1, p.err, abort_flag)) {
        ok = false;
        break;
      }
      ++items;
      tc_fence_after();
      // keys: dV by warpgroup 0, dK by warpgroup 1; queries: half of dQ each
      constexpr int COLS = KEYS ? HD : HD / 2;
      uint32_t gr[64];
      const uint32_t src = KEYS ? (wg == 0 ? tAcc0 : tAcc1) : tAcc1 + wg * COLS;
#pragma unroll
      for (int c = 0; c < (COLS + 31) / 32; ++c) tmem_ld32(src + lane_off + c * 32, gr + c * 32);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
      const bool store = own < it.len && (KEYS || own >= it.qf);
      if (store) {
        const float f = (KEYS && wg == 0) ? 1.f : p.scale;
        const int col = KEYS ? (wg == 0 ? p.H + p.G + it.h : p.H + it.h) * HD : it.h * HD + wg * COLS;
        uint4* dst = reinterpret_cast<uint4*>(p.dqkv + (trow0 + it.kst + own) * width + col);
#pragma unroll
        for (int c = 0; c < COLS / 8; ++c) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(gr[8 * c + e]) * f;
          dst[c] = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, B_TMEM);
  }
}

// ============================================================================ host side
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// [B, L, W] bf16, row stride ld and batch stride sb (elements); box 64 columns x `rows` rows,
// 128-byte swizzle. Rows and columns outside read as zeros.
bool encode_rows(CUtensorMap* map, const void* base, uint64_t W, uint64_t L, uint64_t B, uint64_t ld, uint64_t sb,
                 uint32_t rows) {
  thread_local bool bound = false;
  if (!bound) {
    cudaFree(nullptr);  // makes the device's primary context current on this thread
    bound = true;
  }
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {W, L, B};
  cuuint64_t strides[2] = {ld * 2, sb * 2};
  cuuint32_t box[3] = {64, rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Params make_params(const WindowAttnArgs& a, int tiles) {
  Params p;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.lse = a.lse;
  p.kstart = a.kstart;
  p.dout = static_cast<const __nv_bfloat16*>(a.dout);
  p.dqkv = static_cast<__nv_bfloat16*>(a.dqkv);
  p.dsum = a.dsum;
  p.B = a.B;
  p.H = a.H;
  p.G = a.G;
  p.Lk = a.Lk;
  p.Lq = a.Lq;
  p.hd = a.hd;
  p.window = std::min(a.window, a.Lk);  // wider ones see the same
  p.sinks = std::min(a.sinks, a.Lk);
  p.tiles = tiles;
  p.scale = a.scale;
  p.scale2 = a.scale * kLog2e;
  p.err = a.err;
  return p;
}

int num_sms() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool shapes_ok(const WindowAttnArgs& a) {
  return (a.hd == 32 || a.hd == 64) && a.B > 0 && a.H > 0 && a.G > 0 && a.H % a.G == 0 && a.Lq > 0 && a.Lq <= a.Lk &&
         a.window > 0 && a.sinks >= 0 && a.kstart != nullptr && a.qkv != nullptr && a.out != nullptr &&
         a.lse != nullptr && aligned16(a.qkv) && aligned16(a.out) && a.ld % 8 == 0 && a.sb % 8 == 0 && a.ld > 0 &&
         a.sb > 0;
}

// Raised once a kernel and device; an error is returned, not kept.
template <typename K>
cudaError_t allow_smem(K kern, int bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int HD>
cudaError_t fwd_hd(const WindowAttnArgs& a, cudaStream_t stream) {
  const Params p = make_params(a, (a.Lq + TILE - 1) / TILE + 1);
  const uint64_t W = static_cast<uint64_t>(a.H + 2 * a.G) * HD;
  const auto* base = static_cast<const __nv_bfloat16*>(a.qkv);
  CUtensorMap tq, tkv;
  if (!encode_rows(&tq, base + (a.Lk - a.Lq) * a.ld, W, a.Lq, a.B, a.ld, a.sb, TILE) ||
      !encode_rows(&tkv, base, W, a.Lk, a.B, a.ld, a.sb, TILE))
    return cudaErrorInvalidValue;
  const cudaError_t e = allow_smem(window_fwd_kernel<HD>, F_SMEM);
  if (e != cudaSuccess) return e;
  const long long items = static_cast<long long>(a.H) * a.B * p.tiles;
  if (items > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int grid = static_cast<int>(std::min<long long>(items, 2LL * num_sms()));
  window_fwd_kernel<HD><<<grid, F_THREADS, F_SMEM, stream>>>(tq, tkv, p, static_cast<int>(items));
  return cudaGetLastError();
}

template <int HD>
cudaError_t bwd_hd(const WindowAttnArgs& a, cudaStream_t stream) {
  const uint64_t W = static_cast<uint64_t>(a.H + 2 * a.G) * HD, D = static_cast<uint64_t>(a.H) * HD;
  const auto* base = static_cast<const __nv_bfloat16*>(a.qkv);
  const auto* qbase = base + (a.Lk - a.Lq) * a.ld;
  CUtensorMap q128, q64, kv128, kv64, do128, do64;
  if (!encode_rows(&q128, qbase, W, a.Lq, a.B, a.ld, a.sb, TILE) ||
      !encode_rows(&q64, qbase, W, a.Lq, a.B, a.ld, a.sb, HALF) ||
      !encode_rows(&kv128, base, W, a.Lk, a.B, a.ld, a.sb, TILE) ||
      !encode_rows(&kv64, base, W, a.Lk, a.B, a.ld, a.sb, HALF) ||
      !encode_rows(&do128, a.dout, D, a.Lq, a.B, D, D * a.Lq, TILE) ||
      !encode_rows(&do64, a.dout, D, a.Lq, a.B, D, D * a.Lq, HALF))
    return cudaErrorInvalidValue;
  cudaError_t e = allow_smem(window_bwd_kernel<HD, false>, B_SMEM);
  if (e == cudaSuccess) e = allow_smem(window_bwd_kernel<HD, true>, B_SMEM);
  if (e != cudaSuccess) return e;
  const int sms = num_sms();
  const Params pq = make_params(a, (a.Lq + TILE - 1) / TILE + 1);
  const Params pk = make_params(a, (a.Lk + TILE - 1) / TILE);
  const long long qi = static_cast<long long>(a.H) * a.B * pq.tiles, ki = static_cast<long long>(a.G) * a.B * pk.tiles;
  if (qi > 0x7fffffffLL || ki > 0x7fffffffLL) return cudaErrorInvalidValue;
  // queries first: they leave D behind
  window_bwd_kernel<HD, false><<<static_cast<int>(std::min<long long>(qi, sms)), B_THREADS, B_SMEM, stream>>>(
      q128, do128, kv64, kv64, pq, static_cast<int>(qi));
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  window_bwd_kernel<HD, true><<<static_cast<int>(std::min<long long>(ki, sms)), B_THREADS, B_SMEM, stream>>>(
      kv128, kv128, q64, do64, pk, static_cast<int>(ki));
  return cudaGetLastError();
}

}  // namespace

cudaError_t window_attn_fwd(const WindowAttnArgs& a, cudaStream_t stream) {
  if (!shapes_ok(a)) return cudaErrorInvalidValue;
  return a.hd == 64 ? fwd_hd<64>(a, stream) : fwd_hd<32>(a, stream);
}

cudaError_t window_attn_bwd(const WindowAttnArgs& a, cudaStream_t stream) {
  if (!shapes_ok(a) || a.dout == nullptr || a.dqkv == nullptr || a.dsum == nullptr || !aligned16(a.dout) ||
      !aligned16(a.dqkv))
    return cudaErrorInvalidValue;
  return a.hd == 64 ? bwd_hd<64>(a, stream) : bwd_hd<32>(a, stream);
}

}  // namespace mdl
