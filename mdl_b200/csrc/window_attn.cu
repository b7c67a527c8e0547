// Sliding-window attention with always-visible first tokens (sinks) on the 5th-generation
// tensor cores. Contract: window_attn.h.
//
// Tiles are 128 token rows counted from a sample's FIRST VALID token (row kst + 128 t): padding
// is never loaded, the sinks lie in the first tile(s), and only the diagonal tile and the tile
// that the window's lower edge cuts need a mask. A query tile visits the tiles of the sinks and
// then those of its window, so the cost grows with the window and not with the history.
//
// Forward (384 threads, two persistent CTAs an SM, each with two chains that share nothing but the
// CTA's 256 TMEM columns). Work item = sample, head, query tile; a step = 64 of its keys. A chain:
//   one warp    walks the items; TMA: Q, and K and V into two-stage rings
//   one warp    issues: S = Q K^T; O += P V with P as the A operand straight from TMEM
//   four warps  softmax, a thread a query row: P = exp2(S * c - m) as bf16 into TMEM. m is a
//               reference that moves only when a score passes it by more than 8 (exp2 of the
//               excess stays below 256), so O is rarely rescaled, and is read once.
// S of the next step, of the next item too, is issued as soon as the softmax has read the present
// one. Bound by latency and issue: a chain's steps follow one another, so four chains an SM fill
// its schedulers to a half (the ALUs to 42 %, the exponentials' unit to 31 %, the tensor pipe to
// 11 %, L2 to 42 %). Two chains an SM of 128-key steps, two warps a set of rows, were 736 us where these are
// 462, largely for the registers that the scores took then. Measured: 1,024 samples of up to 544
// tokens, 8 heads of 32, window 128 + 4: 462 us; 64 of 2,000, window 256 + 8: 150 us; 2 of 8,191, 4
// heads of 64, window 1,024 + 16: 43 us, 240 TFLOP/s.
//
// Backward, two launches of one kernel (320 threads, two persistent CTAs an SM): a stationary
// tile of 128 rows meets a stream of 64-row tiles,
//   S = A1 B1^T, dP = A2 B2^T, P = exp2(S * c - lse), dS = P * (dP - D),
//   queries stationary: A = Q, dO; B = K, V;  dQ += dS K;  D = rowsum(dO * O) on the way
//   keys stationary:    A = K, V;  B = Q, dO; dV += P dO, dK += dS Q  (all transposed; the query
//                       heads that share the key head follow one another)
// Recomputing S and dP in the second launch costs two products more than one launch that adds
// dQ to memory would, and needs no fp32 buffer, no clearing, no atomics: every sum has one
// owner and one order. Bound like the forward (schedulers 44 to 54 %, L2 33 %). Measured, queries |
// keys: 661 | 700 us on the first of the shapes above, 52 | 70 us on the last.
//
// Rounding to bf16: P and dS are the A operands of products with bf16 tiles, which tcgen05 takes
// in one type only. Each costs a product's result 0.0017 of its norm, as much as rounding the result
// itself does. dS of dQ is held as two bf16 terms (16 bits), which the queries' launch has room for.
// Sums, references, lse and D are fp32, O reaches D as out + out_lo (16 bits).
//
// Every wait is bounded (error word + abort flag) and every role drains what it has in flight
// before the CTA exits.
#include "window_attn.h"

#include <cudaTypedefs.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "common.cuh"

namespace mdl {
namespace {

constexpr int TILE = 128;               // rows of a tile
constexpr int BOX = 64;                 // rows of a TMA box, and of a step
constexpr int TILE_BYTES = TILE * 128;  // 128-byte rows: 64 columns, the head's hd first
constexpr float kLog2e = 1.4426950408889634f;

constexpr int RECS = 4;                 // item records in flight
constexpr int BOX_BYTES = BOX * 128;
constexpr int TAIL = 512;               // barriers and item records of the backward
constexpr int CHAINS = 2, F_THREADS = 384, F_TMEM = 256, F_STAGES = 2;
constexpr int F_BARS = 7 + 2 * RECS + 2 * F_STAGES;
// a chain: Q | K[2] | V[2]; then the item records and barriers of both chains
constexpr int F_CHAIN = TILE_BYTES + 2 * F_STAGES * BOX_BYTES;
constexpr int F_TAIL = 1024;
constexpr int F_SMEM = 1024 + CHAINS * F_CHAIN + F_TAIL;
constexpr int B_THREADS = 320, B_TMEM = 256, B_STAGES = 4;
// stationary pair | streamed pair [4] | lse, D of the streamed rows [4][64] (or lse of the
// stationary rows [128]) | halves of D [2][2][128] | tail
constexpr int B_SMEM = 1024 + 2 * TILE_BYTES + 2 * B_STAGES * BOX_BYTES + 2 * B_STAGES * BOX * 4 + 4 * TILE * 4 + TAIL;
static_assert(2 * (F_SMEM + 1024) <= 228 * 1024 && 2 * (B_SMEM + 1024) <= 228 * 1024, "two blocks an SM");

struct Params {
  __nv_bfloat16* out;
  __nv_bfloat16* out_lo;
  float* lse;
  const int* kstart;
  const __nv_bfloat16* dout;
  __nv_bfloat16* dqkv;
  float* dsum;
  int B, H, G, Lk, Lq, hd, window, sinks;
  int heads, tiles;  // work items = (head, sample, tile index): heads x B x tiles
  int dh, db, di;    // an item and the next of its block (forward: chain), in these digits
  // key tiles: the first `stiles` (those with sinks) come in `parts` items of `psteps` steps each,
  // whose sums go to `partial` (parts == 1: like any other tile)
  int stiles, parts, psteps;
  float* partial;
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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

// Operand descriptors are a base plus 16-byte units: 2 a K step (16 elements) of a K-major
// operand, 128 a K step (16 rows of 128 bytes) of an MN-major one with 64 columns.
__device__ __forceinline__ uint64_t desc_of(const void* base) { return make_smem_desc(smem_u32(base), 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn_of(const void* base) {
  return make_smem_desc(smem_u32(base), TILE_BYTES, 1024);
}
constexpr uint32_t K_STEP = 2, MN_STEP = 128, BOX_UNITS = BOX_BYTES / 16;

// True on one lane of a converged warp, always the same one. The compiler knows that a single
// lane runs what follows and keeps the operands of the tensor instructions in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}

// Barrier of the two warps that hold the column halves of the same 32 rows.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// A wait of the whole warp, with one outcome for all lanes (.sync.aligned code follows). The
// loop of a wait that is not over at once stays out of line: the issuing warp shares its
// scheduler with the computing ones, so that each instruction between two issues counts.
__device__ __forceinline__ bool bar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool warp_wait_held(uint32_t bar, uint32_t parity, int* err, volatile int* abort_flag) {
  const uint64_t start = globaltimer_ns();
  for (uint32_t spins = 1;; ++spins) {
    if (__all_sync(0xffffffffu, bar_try_wait(bar, parity))) return true;
    if ((spins & 255u) == 0) {
      const bool late = globaltimer_ns() - start > kWaitLimitNs;
      if (__any_sync(0xffffffffu, late || *abort_flag)) {
        if (late) record_error(err, MDL_ERR_MBAR_TIMEOUT);
        *abort_flag = 1;
        return false;
      }
    }
  }
}

__device__ __noinline__ bool warp_wait_slow(uint32_t bar, uint32_t parity, int* err, volatile int* abort_flag) {
  return warp_wait_held(bar, parity, err, abort_flag);
}

// By shared-memory address: barriers at fixed distances then take one register for all.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, bar_try_wait(bar, parity))) return true;
  return warp_wait_slow(bar, parity, err, abort_flag);
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  return warp_wait(smem_u32(bar), parity, err, abort_flag);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Pairs of fp32: one instruction for two columns.
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
__device__ __forceinline__ F2 pair_of(const uint32_t* r) { return {__uint_as_float(r[0]), __uint_as_float(r[1])}; }

// 4-byte asynchronous copy into shared memory; zero when !real (the source is not read then).
__device__ __forceinline__ void copy4(const void* dst, const float* src, bool real) {
  const int n = real ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
// Arrives on `bar` (as one of its expected arrivals) once this thread's copies have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bits [l, h] (inclusive, clipped) of 32-column word w.
__device__ __forceinline__ uint32_t range_bits(int l, int h, int w) {
  const int a = max(l - 32 * w, 0), b = min(h - 32 * w, 31);
  if (a > b) return 0u;
  return (0xFFFFFFFFu >> (31 - b)) & (0xFFFFFFFFu << a);
}

// 128 rows as two boxes of 64.
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* tm, uint64_t* bar, int x, int y, int b) {
  tma_load_3d(dst, tm, bar, x, y, b);
  tma_load_3d(dst + BOX * 128, tm, bar, x, y + BOX, b);
}

// One row of hd zeros (bf16).
__device__ __forceinline__ void zero_row(__nv_bfloat16* dst, int hd) {
  for (int c = 0; c < hd / 8; ++c) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0, 0, 0, 0);
}

// ============================================================================ work items
// Query tiles with runs of ROWS keys as their steps (forward, and backward with queries
// stationary), or key tiles (KEYS) with runs of ROWS queries of each query head of the group.
// Positions are relative to the first valid token.

struct alignas(16) Item {
  int n, t, cs, k0;       // steps (-1: no more items); tile; steps: cs from 0, then from k0 on (KEYS: cs a head, from k0)
  int qf, len, j0, part;  // first query, valid tokens; first step, and slot of the partial sums (-1: none)
  int h, b, kst, row0;    // head, sample, first valid token; query row of the tile's first row
  long long out, lse;     // elements from the start of out (of dqkv in the backward) and of lse to that row
};

// Query steps of key tile t: from k0 on, cs a query head.
__device__ __forceinline__ void key_steps(const Params& p, int t, int len, int qf, int& k0, int& cs) {
  const int qs = max(TILE * t, qf);
  const int qe = TILE * t < p.sinks ? len : min(len, TILE * t + TILE - 1 + p.window);
  k0 = qs / BOX;
  cs = qe > qs && TILE * t < len ? (qe + BOX - 1) / BOX - k0 : 0;
}

// First row of step j (key tiles: of step j of a query head).
template <bool KEYS, int ROWS>
__device__ __forceinline__ int step_row(int j, int cs, int k0) {
  return ROWS * (KEYS ? k0 + j : (j < cs ? j : k0 + j - cs));
}

// The items of a block (of one of its chains in the forward) one after another, a fixed distance apart. Only the loading warp walks them; it
// hands the others a record an item in shared memory, so that they carry neither the walk nor
// its registers (kept beside 64 scores a thread they spilled, and the spills set the pace).
// kstart of the next item is loaded an item ahead, and the digits are carried along.
template <bool KEYS, int ROWS>
struct Walk {
  Item it;
  int i;                // index within the pair (head, sample)
  int nh, nb, ni, nks;  // next item

  __device__ __forceinline__ Walk(const Params& p, int first) {
    nh = first % p.heads;
    const int rest = first / p.heads;
    nb = rest % p.B;
    ni = rest / p.B;
    nks = ni < p.tiles ? __ldg(p.kstart + nb) : 0;
  }
  // To the next item, with work or without (then n is 0); false: none left.
  __device__ __forceinline__ bool next(const Params& p) {
    if (ni >= p.tiles) return false;
    it.h = nh;
    it.b = nb;
    i = ni;
    const int ks = __reduce_max_sync(0xffffffffu, nks);  // the warp runs as one: uniform registers
    nh += p.dh;
    int carry = nh >= p.heads ? 1 : 0;
    nh -= carry ? p.heads : 0;
    nb += p.db + carry;
    carry = nb >= p.B ? 1 : 0;
    nb -= carry ? p.B : 0;
    ni += p.di + carry;
    nks = ni < p.tiles ? __ldg(p.kstart + nb) : 0;
    it.kst = min(max(ks, 0), p.Lk);
    it.len = p.Lk - it.kst;
    it.qf = max(0, p.Lk - p.Lq - it.kst);
    it.n = it.cs = it.k0 = 0;
    it.j0 = 0;
    it.part = -1;
    if constexpr (KEYS) {
      // the sinks' tiles come first: every query sees them
      const int split = p.stiles * p.parts;
      it.t = i < split ? i / p.parts : i - split + p.stiles;
      key_steps(p, it.t, it.len, it.qf, it.k0, it.cs);
      it.n = it.cs * (p.H / p.G);
      if (p.parts > 1 && i < split) {
        const int c = i - it.t * p.parts;
        it.j0 = c * p.psteps;
        it.n = max(0, min(it.n - it.j0, p.psteps));
        it.part = ((it.b * p.G + it.h) * p.stiles + it.t) * p.parts + c;
      }
    } else {
      it.t = (it.len + TILE - 1) / TILE - 1 - i;  // the last tile first
      if (it.t < 0 || TILE * (it.t + 1) <= it.qf) return true;
      it.k0 = max(0, max(TILE * it.t, it.qf) - p.window + 1) / ROWS;
      it.cs = min((min(p.sinks, it.len) + ROWS - 1) / ROWS, it.k0);
      it.n = it.cs + (min(TILE * (it.t + 1), it.len) + ROWS - 1) / ROWS - it.k0;
    }
    return true;
  }
};

// ============================================================================ forward
template <int HD>
__global__ void __launch_bounds__(F_THREADS, 2)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv,
                      const Params p) {
  // 64-wide heads: P takes the place of half of S (64 | O 64 columns), and the next scores wait for
  // the products; 32-wide ones have room beside it (S 64 | P 32 | O 32).
  constexpr bool OVER = HD == 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chain = warp < 4 ? warp >> 1 : (warp - 4) >> 2;
  uint8_t* sQ = smem + chain * F_CHAIN;
  uint8_t* sK = sQ + TILE_BYTES;              // [F_STAGES]
  uint8_t* sV = sK + F_STAGES * BOX_BYTES;    // [F_STAGES]
  Item* recs = reinterpret_cast<Item*>(smem + CHAINS * F_CHAIN) + chain * RECS;
  uint64_t* all_bars = reinterpret_cast<uint64_t*>(reinterpret_cast<Item*>(smem + CHAINS * F_CHAIN) + CHAINS * RECS);
  uint64_t* bars = all_bars + chain * F_BARS;
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* s_full = bars + 2;
  uint64_t* s_empty = bars + 3;
  uint64_t* p_full = bars + 4;
  uint64_t* pv_done = bars + 5;
  uint64_t* done = bars + 6;
  uint64_t* kv_full = bars + 7;                // [F_STAGES]
  uint64_t* kv_empty = kv_full + F_STAGES;     // [F_STAGES]
  uint64_t* rec_full = kv_empty + F_STAGES;    // [RECS]
  uint64_t* rec_empty = rec_full + RECS;       // [RECS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_bars + CHAINS * F_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(CHAINS * (RECS * sizeof(Item) + F_BARS * 8) + 8 <= F_TAIL, "records and barriers");

  if (threadIdx.x < 4 * 32 && (threadIdx.x & 63) == 0) {  // the first thread of each chain
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(s_empty, 4);
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    mbar_init(done, 1);
    for (int s = 0; s < F_STAGES; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < RECS; ++s) {
      mbar_init(&rec_full[s], 1);
      mbar_init(&rec_empty[s], 5);  // the issuing warp and the softmax warps
    }
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
  const uint32_t tS = *tmem_slot + chain * 128;
  const uint32_t tP = OVER ? tS + 32 : tS + 64, tO = OVER ? tS + 64 : tS + 96;

  if (warp < 4) {
    if ((warp & 1) == 0) {
      // ---------------------------------------------------------- walk and load
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_kv);
      }
      const int q0 = p.Lk - p.Lq;
      int items = 0, g = 0;
      bool ok = true;
      Walk<false, BOX> w(p, chain * gridDim.x + blockIdx.x);
      while (ok && w.next(p)) {
        const Item& it = w.it;
        // queries before the first valid token (a share of them per item)
        const int pad = min(p.Lq, it.kst - q0);
        for (int q = w.i * 32 + lane; q < pad; q += p.tiles * 32) {
          const long long row = static_cast<long long>(it.b) * p.Lq + q;
          zero_row(p.out + (row * p.H + it.h) * HD, HD);
          if (p.out_lo != nullptr) zero_row(p.out_lo + (row * p.H + it.h) * HD, HD);
          p.lse[(static_cast<long long>(it.b) * p.H + it.h) * p.Lq + q] = CUDART_INF_F;
        }
        if (it.n == 0) continue;
        const int slot = items % RECS;
        // parity of the previous use of a stage; a fresh barrier passes parity 1 at once
        if (!warp_wait(&rec_empty[slot], (items / RECS + 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        w.it.row0 = it.kst + TILE * it.t - q0;
        w.it.lse = (static_cast<long long>(it.b) * p.H + it.h) * p.Lq + it.row0;
        w.it.out = ((static_cast<long long>(it.b) * p.Lq + it.row0) * p.H + it.h) * HD;
        if (lane == 0) {
          recs[slot] = it;
          mbar_arrive(&rec_full[slot]);
        }
        __syncwarp();
        const int kvh = it.h / (p.H / p.G);
        if (!warp_wait(q_empty, (items + 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, TILE_BYTES);
          load_tile(sQ, &tm_q, q_full, it.h * HD, it.row0, it.b);
        }
        __syncwarp();
        ++items;
        for (int j = 0; j < it.n; ++j, ++g) {
          const int st = g % F_STAGES, y = it.kst + step_row<false, BOX>(j, it.cs, it.k0);
          if (!warp_wait(&kv_empty[st], (g / F_STAGES + 1) & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&kv_full[st], 2 * BOX_BYTES);
            tma_load_3d(sK + st * BOX_BYTES, &tm_kv, &kv_full[st], (p.H + kvh) * HD, y, it.b);
            tma_load_3d(sV + st * BOX_BYTES, &tm_kv, &kv_full[st], (p.H + p.G + kvh) * HD, y, it.b);
          }
          __syncwarp();
        }
      }
      const int slot = items % RECS;
      if (ok && warp_wait(&rec_empty[slot], (items / RECS + 1) & 1, p.err, abort_flag) && lane == 0) {
        recs[slot].n = -1;
        mbar_arrive(&rec_full[slot]);
      }
      __syncwarp();
      // every copy into this CTA's smem has landed before the CTA may exit
      if (lane == 0) {
        if (items > 0) mbar_wait(q_full, (items - 1) & 1, nullptr, nullptr);
        for (int j = max(0, g - F_STAGES); j < g; ++j)
          mbar_wait(&kv_full[j % F_STAGES], (j / F_STAGES) & 1, nullptr, nullptr);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- issue
      // The whole warp waits (uniform registers hold its counters and descriptors); one lane
      // issues. Scores run one step ahead of the products, across items.
      constexpr uint32_t idesc_s = make_idesc_bf16(TILE, BOX, false, false);
      constexpr uint32_t idesc_pv = make_idesc_bf16(TILE, HD, false, true);
      const uint64_t dQ = desc_of(sQ), dK = desc_of(sK), dV = desc_mn_of(sV);
      int a_items = 0, a_j = 0, a_n = 0, a_g = 0;  // ahead: item, step, its steps, step of the chain
      bool ok = true;
      // steps of item `i`, -1 after the last
      auto steps_of = [&](int i) -> int {
        if (!warp_wait(&rec_full[i % RECS], (i / RECS) & 1, p.err, abort_flag)) {
          ok = false;
          return -1;
        }
        return __reduce_max_sync(0xffffffffu, recs[i % RECS].n);
      };
      auto issue_s = [&]() -> bool {
        const int st = a_g % F_STAGES;
        if ((a_j == 0 && !warp_wait(q_full, a_items & 1, p.err, abort_flag)) ||
            !warp_wait(&kv_full[st], (a_g / F_STAGES) & 1, p.err, abort_flag) ||
            (!OVER && a_g > 0 && !warp_wait(s_empty, (a_g - 1) & 1, p.err, abort_flag)))
          return false;
        tc_fence_after();
        const uint64_t b = dK + st * BOX_UNITS;
        const bool last = a_j + 1 == a_n;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tS, dQ + ks * K_STEP, b + ks * K_STEP, idesc_s, ks);
          tc_commit(s_full);
          if (last) tc_commit(q_empty);
        }
        __syncwarp();
        ++a_g;
        ++a_j;
        if (last) {
          a_j = 0;
          a_n = steps_of(++a_items);
        }
        return ok;
      };
      a_n = steps_of(0);
      int n = a_n, g = 0;
      if (ok && a_n > 0) ok = issue_s();
      for (int items = 0; ok && n > 0; ++items) {
        for (int j = 0; j < n; ++j, ++g) {
          const int st = g % F_STAGES;
          if ((!OVER && a_n > 0 && !issue_s()) || !warp_wait(p_full, g & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t b = dV + st * BOX_UNITS;
          const uint32_t acc = j > 0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < BOX / 16; ++ks)
              tc_mma_bf16_ts(tO, tP + ks * 8, b + ks * MN_STEP, idesc_pv, ks > 0 ? 1u : acc);
            tc_commit(pv_done);
            tc_commit(&kv_empty[st]);
          }
          __syncwarp();
          if (OVER && a_n > 0 && !issue_s()) {  // behind the products: the tensor pipe keeps their order
            ok = false;
            break;
          }
        }
        if (!ok) break;
        n = steps_of(items + 1);
        if (elect_one()) mbar_arrive(&rec_empty[items % RECS]);
        __syncwarp();
      }
      // all MMAs have finished before TMEM is released
      if (elect_one()) {
        tc_commit(done);
        mbar_wait(done, 0, nullptr, nullptr);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax
    // Thread = query row.
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t bar = smem_u32(bars);
    constexpr uint32_t S_FULL = 16, S_EMPTY = 24, P_FULL = 32, PV_DONE = 40, REC_FULL = 56 + 16 * F_STAGES,
                       REC_EMPTY = REC_FULL + 8 * RECS;
    bool ok = true;
    int g = 0, items = 0;
    float m = 0.f, l = 0.f;  // reference and sum of the row
    // The output of item `items - 1`, while the next item's first scores are computed.
    auto write_out = [&](float ref, float sum) {
      const int slot = (items - 1) % RECS;
      const Item& it = recs[slot];
      const bool real = static_cast<unsigned>(it.row0 + r) < static_cast<unsigned>(p.Lq);
      const long long o = it.out + static_cast<long long>(r) * (p.H * HD);
      const long long ls = it.lse + r;
      __syncwarp();
      if (lane == 0) bar_arrive(bar + REC_EMPTY + 8 * slot);
      if (real) p.lse[ls] = ref + lg2(sum);
      const float inv = __fdividef(1.f, sum);
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t ov[16];
        tmem_ld16(tO + lanes + c * 16, ov);
        tmem_wait_ld();
        if (!real) continue;
        uint32_t hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __uint_as_float(ov[2 * e]) * inv, y = __uint_as_float(ov[2 * e + 1]) * inv;
          hi[e] = pack2(x, y);
          ov[e] = pack2(x - __uint_as_float(hi[e] << 16), y - __uint_as_float(hi[e] & 0xFFFF0000u));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          reinterpret_cast<uint4*>(p.out + o + c * 16)[e] =
              make_uint4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]);
          if (p.out_lo != nullptr)
            reinterpret_cast<uint4*>(p.out_lo + o + c * 16)[e] =
                make_uint4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
        }
      }
    };
    for (;; ++items) {
      const int slot = items % RECS;
      if (!warp_wait(bar + REC_FULL + 8 * slot, (items / RECS) & 1, p.err, abort_flag)) {
        ok = false;
        break;
      }
      const int4 first = *reinterpret_cast<const int4*>(&recs[slot]);
      const int n = first.x, t = first.y, cs = first.z, k0 = first.w;
      if (n < 0) break;
      if (items > 0) {
        if (!warp_wait(bar + PV_DONE, (g - 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        write_out(m, l);
      }
      for (int j = 0; j < n; ++j, ++g) {
        // Which of the step's two runs of 32 keys do these 32 queries see? None, all, or some.
        const int row = TILE * t + 32 * quarter;  // the first query
        const int key = step_row<false, BOX>(j, cs, k0);
        bool live[2], part[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int lo = key + 32 * c, hi = lo + 31;
          live[c] = lo <= row + 31 && (hi > row - p.window || lo < p.sinks);
          part[c] = hi > row || (lo <= row + 31 - p.window && hi >= p.sinks);
        }
        if (!warp_wait(bar + S_FULL, g & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // The scores pass through registers 32 at a time, the first 32 twice (for the maximum and for
        // the exponentials): all 64 would spill.
        uint32_t sr[32];
        auto load = [&](int c) {
          tmem_ld32(tS + lanes + 32 * c, sr);
          tmem_wait_ld();
          if (part[c]) {
            const int d = row + lane - key;  // keys up to d are not in the future
            const uint32_t vm = range_bits(d - p.window + 1, d, c) | range_bits(0, min(d, p.sinks - 1 - key), c);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((vm >> k) & 1u)) sr[k] = __float_as_uint(-CUDART_INF_F);
          }
        };
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!live[c]) continue;
          load(c);
          float m2[2] = {__uint_as_float(sr[0]), __uint_as_float(sr[1])};
#pragma unroll
          for (int k = 2; k < 30; k += 4) {
            m2[0] = max3(m2[0], __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
            m2[1] = max3(m2[1], __uint_as_float(sr[k + 2]), __uint_as_float(sr[k + 3]));
          }
          m2[0] = max3(m2[0], __uint_as_float(sr[30]), __uint_as_float(sr[31]));
          mx = max3(mx, m2[0], m2[1]);
        }
        mx *= p.scale2;
        if (g > 0 && !warp_wait(bar + PV_DONE, (g - 1) & 1, p.err, abort_flag)) {  // the last P was consumed
          ok = false;
          break;
        }
        tc_fence_after();
        if (j == 0) {
          m = mx;
          l = 0.f;
        } else if (__any_sync(0xffffffffu, mx > m + 8.f)) {
          const float m_new = fmaxf(m, mx);
          const float alpha = m_new == -CUDART_INF_F ? 1.f : ex2(m - m_new);
          m = m_new;
          l *= alpha;
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {  // few registers at a time: the scores are held
            uint32_t ov[8];
            tmem_ld8(tO + lanes + c * 8, ov);
            tmem_wait_ld();
#pragma unroll
            for (int d = 0; d < 8; ++d) ov[d] = __float_as_uint(__uint_as_float(ov[d]) * alpha);
            tmem_st8(tO + lanes + c * 8, ov);
          }
        }
        const float m_use = m == -CUDART_INF_F ? 0.f : m;
        const F2 sc = {-p.scale2, -p.scale2}, mm = {m_use, m_use};
        F2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int c = 1; c >= 0; --c) {
          uint32_t pk[16];
          if (c == 0) {
            if (live[0] && live[1]) load(0);
            if (!OVER) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) bar_arrive(bar + S_EMPTY);
            }
          }
          if (live[c]) {
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const F2 x = fma2(pair_of(sr + k), sc, mm);  // m - score; the sign is free in ex2
              const F2 e = {ex2(-x.x), ex2(-x.y)};
              sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], e);
              pk[k / 2] = pack2(e.x, e.y);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) pk[k] = 0u;
          }
          tmem_st16(tP + lanes + 16 * c, pk);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar + P_FULL);
      }
      if (!ok) break;
    }
    if (ok && items > 0 && warp_wait(bar + PV_DONE, (g - 1) & 1, p.err, abort_flag)) {
      tc_fence_after();
      write_out(m, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, F_TMEM);
  }
}

// ============================================================================ backward
// KEYS: the stationary tile holds keys (dK, dV), else queries (dQ and D).
template <int HD, bool KEYS>
__global__ void __launch_bounds__(B_THREADS, 2)
    window_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv,
                      const __grid_constant__ CUtensorMap tm_do, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sA1 = smem;
  uint8_t* sA2 = sA1 + TILE_BYTES;
  uint8_t* sB1 = sA2 + TILE_BYTES;               // [4]
  uint8_t* sB2 = sB1 + B_STAGES * BOX_BYTES;     // [4]
  float* sLse = reinterpret_cast<float*>(sB2 + B_STAGES * BOX_BYTES);  // [4][64], or [128]
  float* sD = sLse + B_STAGES * BOX;                                   // [4][64]
  float* sHalf = sD + B_STAGES * BOX;                                  // [2 items][2 halves][128]
  Item* recs = reinterpret_cast<Item*>(sHalf + 4 * TILE);              // [RECS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(recs + RECS);
  uint64_t* a_full = bars;
  uint64_t* a_empty = bars + 1;
  uint64_t* b_full = bars + 2;    // [4]
  uint64_t* b_empty = bars + 6;   // [4]
  uint64_t* s_full = bars + 10;
  uint64_t* s_empty = bars + 11;
  uint64_t* p_full = bars + 12;
  uint64_t* p_empty = bars + 13;
  uint64_t* acc_full = bars + 14;
  uint64_t* acc_empty = bars + 15;
  uint64_t* done = bars + 16;
  uint64_t* rec_full = bars + 17;   // [RECS]
  uint64_t* rec_empty = bars + 21;  // [RECS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 25);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(RECS * sizeof(Item) + 26 * 8 <= TAIL, "records and barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(a_full, KEYS ? 1 : 33);  // TMA bytes (+ the 32 lanes that copy lse)
    mbar_init(a_empty, KEYS ? 1 : 9);  // the last scores (+ the warps that read dO)
    for (int s = 0; s < B_STAGES; ++s) {
      mbar_init(&b_full[s], KEYS ? 33 : 1);  // TMA bytes (+ the 32 lanes that copy lse and D)
      mbar_init(&b_empty[s], 1);
    }
    for (int s = 0; s < RECS; ++s) {
      mbar_init(&rec_full[s], 1);
      mbar_init(&rec_empty[s], 9);  // the issuing warp and the computing warps
    }
    mbar_init(s_full, 1);
    mbar_init(s_empty, 8);
    mbar_init(p_full, 8);
    mbar_init(p_empty, 1);
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
  // S 64 | dP 64 | P 32 | dS 32 | accumulators hd each. With dK and dV 64 wide there is no room
  // for P and dS: each warp then puts them over the first half of its own scores, and the next
  // scores wait for the products that read them.
  constexpr bool OVER = KEYS && HD == 64;
  const uint32_t tS = tmem, tDP = tmem + 64, tP = OVER ? tS : tmem + 128, tDS = OVER ? tDP : tmem + 160;
  const uint32_t tAcc0 = tmem + (OVER ? 128 : 192), tAcc1 = KEYS ? tAcc0 + HD : tAcc0;
  constexpr uint32_t PAIR_STEP = OVER ? 32 : 16;  // columns from one half's P to the other's
  const int q0 = p.Lk - p.Lq;

  if (warp == 0) {
    // ------------------------------------------------------------ walk and load
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_kv);
      tma_prefetch_desc(&tm_do);
    }
    bool ok = true;
    Walk<KEYS, BOX> w(p, blockIdx.x);
    int items = 0, g = 0;
    const int width = (p.H + 2 * p.G) * HD;
    while (ok && w.next(p)) {
      const Item& it = w.it;
      const int ya = it.kst + TILE * it.t;
      // gradients of what nobody sees or asks for: a share, per item, of the rows before the
      // first valid token (queries: the first query), and valid keys without a query
      const long long trow0 = static_cast<long long>(it.b) * p.Lk;
      auto clear = [&](int row) {
        __nv_bfloat16* dst = p.dqkv + (trow0 + row) * width + (KEYS ? p.H + it.h : it.h) * HD;
        zero_row(dst, HD);
        if (KEYS) zero_row(dst + p.G * HD, HD);
      };
      for (int k = w.i * 32 + lane; k < it.kst + (KEYS ? 0 : it.qf); k += p.tiles * 32) clear(k);
      if (it.n == 0) {
        if (KEYS && it.part < 0)
          for (int k = ya + lane; k < min(ya + TILE, p.Lk); k += 32) clear(k);
        continue;
      }
      const int slot = items % RECS;
      // parity of the previous use of a stage; a fresh barrier passes parity 1 at once
      if (!warp_wait(&rec_empty[slot], (items / RECS + 1) & 1, p.err, abort_flag)) break;
      w.it.row0 = ya - q0;
      w.it.lse = (static_cast<long long>(it.b) * p.H + it.h) * p.Lq + it.row0;
      w.it.out = (trow0 + ya) * width + (KEYS ? p.H + it.h : it.h) * HD;
      if (lane == 0) {
        recs[slot] = it;
        mbar_arrive(&rec_full[slot]);
      }
      __syncwarp();
      if (!warp_wait(a_empty, (items + 1) & 1, p.err, abort_flag)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(a_full, 2 * TILE_BYTES);
        if constexpr (KEYS) {
          load_tile(sA1, &tm_kv, a_full, (p.H + it.h) * HD, ya, it.b);
          load_tile(sA2, &tm_kv, a_full, (p.H + p.G + it.h) * HD, ya, it.b);
        } else {
          load_tile(sA1, &tm_q, a_full, it.h * HD, ya - q0, it.b);
          load_tile(sA2, &tm_do, a_full, it.h * HD, ya - q0, it.b);
        }
      }
      __syncwarp();
      ++items;
      // lse (and D) of queries from `rel` on; rows that are no queries get zeros and are never
      // visible
      auto copy_rows = [&](float* lse, float* d, int rel, int h, uint64_t* bar) {
#pragma unroll
        for (int e = 0; e < (KEYS ? BOX : TILE) / 32; ++e) {
          const int c = lane + 32 * e;
          const bool real = rel + c >= it.qf && rel + c < it.len;
          const long long off = (static_cast<long long>(it.b) * p.H + h) * p.Lq + (real ? it.kst + rel + c - q0 : 0);
          copy4(lse + c, p.lse + off, real);
          if (KEYS) copy4(d + c, p.dsum + off, real);
        }
        copies_arrive(bar);
      };
      if constexpr (!KEYS) copy_rows(sLse, nullptr, TILE * it.t, it.h, a_full);
      const int a0 = KEYS && it.j0 > 0 ? it.j0 / it.cs : 0;
      int h = KEYS ? it.h * (p.H / p.G) + a0 : it.h;
      for (int j = 0, s = it.j0 - a0 * it.cs; j < it.n; ++j, ++s, ++g) {
        const int st = g % B_STAGES;
        if (!warp_wait(&b_empty[st], (g / B_STAGES + 1) & 1, p.err, abort_flag)) {
          ok = false;
          break;
        }
        if (KEYS && s == it.cs) {  // the next query head of the group
          s = 0;
          ++h;
        }
        const int rel = step_row<KEYS, BOX>(s, it.cs, it.k0), y = it.kst + rel;
        if (lane == 0) {
          mbar_arrive_expect_tx(&b_full[st], 2 * BOX_BYTES);
          if constexpr (KEYS) {
            tma_load_3d(sB1 + st * BOX_BYTES, &tm_q, &b_full[st], h * HD, y - q0, it.b);
            tma_load_3d(sB2 + st * BOX_BYTES, &tm_do, &b_full[st], h * HD, y - q0, it.b);
          } else {
            const int kvh = h / (p.H / p.G);
            tma_load_3d(sB1 + st * BOX_BYTES, &tm_kv, &b_full[st], (p.H + kvh) * HD, y, it.b);
            tma_load_3d(sB2 + st * BOX_BYTES, &tm_kv, &b_full[st], (p.H + p.G + kvh) * HD, y, it.b);
          }
        }
        __syncwarp();
        if constexpr (KEYS) copy_rows(sLse + st * BOX, sD + st * BOX, rel, h, &b_full[st]);
      }
    }
    const int slot = items % RECS;
    if (ok && warp_wait(&rec_empty[slot], (items / RECS + 1) & 1, p.err, abort_flag) && lane == 0) {
      recs[slot].n = -1;
      mbar_arrive(&rec_full[slot]);
    }
    __syncwarp();
    if (lane == 0) {  // every copy into this CTA's smem has landed before the CTA may exit
      if (items > 0) mbar_wait(a_full, (items - 1) & 1, nullptr, nullptr);
      for (int j = max(0, g - B_STAGES); j < g; ++j)
        mbar_wait(&b_full[j % B_STAGES], (j / B_STAGES) & 1, nullptr, nullptr);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ issue (see the forward)
    constexpr uint32_t idesc_s = make_idesc_bf16(TILE, BOX, false, false);
    constexpr uint32_t idesc_acc = make_idesc_bf16(TILE, HD, false, true);
    const uint64_t dA1 = desc_of(sA1), dA2 = desc_of(sA2), dB1 = desc_of(sB1), dB2 = desc_of(sB2);
    const uint64_t mB1 = desc_mn_of(sB1), mB2 = desc_mn_of(sB2);
    int a_items = 0, a_j = 0, a_n = 0, a_g = 0;  // ahead: item, step, its steps, step of the block
    bool ok = true;
    auto steps_of = [&](int i) -> int {
      if (!warp_wait(&rec_full[i % RECS], (i / RECS) & 1, p.err, abort_flag)) {
        ok = false;
        return -1;
      }
      return __reduce_max_sync(0xffffffffu, recs[i % RECS].n);
    };
    auto issue_s = [&]() -> bool {
      const int st = a_g % B_STAGES;
      if ((a_j == 0 && !warp_wait(a_full, a_items & 1, p.err, abort_flag)) ||
          !warp_wait(&b_full[st], (a_g / B_STAGES) & 1, p.err, abort_flag) ||
          (a_g > 0 && !warp_wait(OVER ? p_empty : s_empty, (a_g - 1) & 1, p.err, abort_flag)))
        return false;
      tc_fence_after();
      const uint64_t b1 = dB1 + st * BOX_UNITS, b2 = dB2 + st * BOX_UNITS;
      const bool last = a_j + 1 == a_n;
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tS, dA1 + ks * K_STEP, b1 + ks * K_STEP, idesc_s, ks);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) tc_mma_bf16(tDP, dA2 + ks * K_STEP, b2 + ks * K_STEP, idesc_s, ks);
        tc_commit(s_full);
        if (last) tc_commit(a_empty);
      }
      __syncwarp();
      ++a_g;
      ++a_j;
      if (last) {
        a_j = 0;
        a_n = steps_of(++a_items);
      }
      return ok;
    };
    a_n = steps_of(0);
    int n = a_n, g = 0;
    if (ok && a_n > 0) ok = issue_s();
    for (int items = 0; ok && n > 0; ++items) {
      for (int j = 0; j < n; ++j, ++g) {
        const int st = g % B_STAGES;
        // (OVER: the next scores come after this step's products)
        if ((!OVER && a_n > 0 && !issue_s()) || !warp_wait(p_full, g & 1, p.err, abort_flag) ||
            (j == 0 && items >= 1 && !warp_wait(acc_empty, (items - 1) & 1, p.err, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t b1 = mB1 + st * BOX_UNITS, b2 = mB2 + st * BOX_UNITS;
        const uint32_t acc = j > 0 ? 1u : 0u;
        const bool last = j + 1 == n;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < BOX / 16; ++ks) {
            const uint32_t off = (ks >> 1) * PAIR_STEP + (ks & 1) * 8;
            if constexpr (KEYS) tc_mma_bf16_ts(tAcc0, tP + off, b2 + ks * MN_STEP, idesc_acc, ks > 0 ? 1u : acc);
            tc_mma_bf16_ts(tAcc1, tDS + off, b1 + ks * MN_STEP, idesc_acc, ks > 0 ? 1u : acc);
            if constexpr (!KEYS) tc_mma_bf16_ts(tAcc1, tP + off, b1 + ks * MN_STEP, idesc_acc, 1u);
          }
          tc_commit(p_empty);
          tc_commit(&b_empty[st]);
          if (last) tc_commit(acc_full);
        }
        __syncwarp();
        if (OVER && a_n > 0 && !issue_s()) {
          ok = false;
          break;
        }
      }
      if (!ok) break;
      n = steps_of(items + 1);
      if (elect_one()) mbar_arrive(&rec_empty[items % RECS]);
      __syncwarp();
    }
    if (elect_one()) {
      tc_commit(done);
      mbar_wait(done, 0, nullptr, nullptr);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ compute
    // Two warps share 32 rows, 32 of the 64 columns each.
    const int half = (warp - 2) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS_own = tS + lane_off + 32 * half, tDP_own = tDP + lane_off + 32 * half;
    const uint32_t tP_own = tP + lane_off + PAIR_STEP * half, tDS_own = tDS + lane_off + PAIR_STEP * half;
    const int row_stride = (p.H + 2 * p.G) * HD;
    const uint32_t bar = smem_u32(bars);
    constexpr uint32_t A_FULL = 0, A_EMPTY = 8, B_FULL = 16, S_FULL = 80, S_EMPTY = 88, P_FULL = 96, P_EMPTY = 104,
                       ACC_FULL = 112, ACC_EMPTY = 120, REC_FULL = 136, REC_EMPTY = REC_FULL + 8 * RECS;
    bool ok = true;
    int items = 0, g = 0;
    // keys: dV or dK; queries: half of dQ
    constexpr int COLS = KEYS ? HD : HD / 2;
    const int col0 = KEYS ? 0 : half * COLS;
    const uint32_t tAcc_own = (KEYS && half == 0 ? tAcc0 : tAcc1) + lane_off + col0;
    // Gradients of item k: written once its successor's first scores are there.
    auto write_grad = [&](int k) -> bool {
      if (!warp_wait(bar + ACC_FULL, k & 1, p.err, abort_flag)) return false;
      tc_fence_after();
      const Item& it = recs[k % RECS];
      const int own = TILE * it.t + r;
      const bool store = own < it.len && (KEYS || own >= it.qf);
      __nv_bfloat16* dst = p.dqkv + it.out + r * row_stride + (KEYS && half == 0 ? p.G * HD : col0);
      const float f = (KEYS && half == 0) ? 1.f : p.scale;
      float4* sums = KEYS && it.part >= 0
                         ? reinterpret_cast<float4*>(p.partial + ((static_cast<long long>(it.part) * TILE + r) * 2 + half) * HD)
                         : nullptr;
#pragma unroll
      for (int e = 0; e < COLS / 8; ++e) {
        uint32_t gr[8], y[4];
        tmem_ld8(tAcc_own + 8 * e, gr);
        tmem_wait_ld();
        if (KEYS && sums != nullptr) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            sums[2 * e + c] = make_float4(__uint_as_float(gr[4 * c]) * f, __uint_as_float(gr[4 * c + 1]) * f,
                                          __uint_as_float(gr[4 * c + 2]) * f, __uint_as_float(gr[4 * c + 3]) * f);
          continue;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = pack2(__uint_as_float(gr[2 * c]) * f, __uint_as_float(gr[2 * c + 1]) * f);
        if (store) reinterpret_cast<uint4*>(dst)[e] = make_uint4(y[0], y[1], y[2], y[3]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        bar_arrive(bar + ACC_EMPTY);
        bar_arrive(bar + REC_EMPTY + 8 * (k % RECS));
      }
      return true;
    };
    for (;; ++items) {
      const int slot = items % RECS;
      if (!warp_wait(bar + REC_FULL + 8 * slot, (items / RECS) & 1, p.err, abort_flag)) {
        ok = false;
        break;
      }
      const Item& it = recs[slot];  // what only a mask or the item's ends need stays there
      const int4 first = *reinterpret_cast<const int4*>(&it);
      const int n = first.x, t = first.y, cs = first.z, k0 = first.w, own = TILE * t + r;
      if (n < 0) break;
      float row_lse = 0.f, row_d = 0.f;
      if constexpr (!KEYS) {
        // D of the row from dO (shared memory) and the output (16 bits: out + out_lo), half of
        // the head a warp; the output's loads are under way while the tile is waited for
        constexpr int V = HD / 16;  // 16-byte pieces of half a row
        const bool real = own >= it.qf && own < it.len;
        const long long ls = recs[slot].lse + r;  // (sample, head, query row)
        const long long o = ((static_cast<long long>(recs[slot].b) * p.Lq + recs[slot].row0 + r) * p.H + recs[slot].h) * HD +
                            half * (HD / 2);
        const uint8_t* go = sA2 + r * 128;
#pragma unroll
        for (int v = 0; v < V; v += 2) {
          uint4 hv[2], lv[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            hv[c] = lv[c] = make_uint4(0, 0, 0, 0);
            if (real) {
              hv[c] = __ldg(reinterpret_cast<const uint4*>(p.out + o) + v + c);
              lv[c] = __ldg(reinterpret_cast<const uint4*>(p.out_lo + o) + v + c);
            }
          }
          if (v == 0 && !warp_wait_held(bar + A_FULL, items & 1, p.err, abort_flag)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint4 gv = *reinterpret_cast<const uint4*>(go + ((half * V + v + c) ^ (r & 7)) * 16);
            const uint32_t e[4] = {gv.x, gv.y, gv.z, gv.w}, a[4] = {hv[c].x, hv[c].y, hv[c].z, hv[c].w},
                           z[4] = {lv[c].x, lv[c].y, lv[c].z, lv[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              row_d = fmaf(__uint_as_float(a[i] << 16) + __uint_as_float(z[i] << 16), __uint_as_float(e[i] << 16), row_d);
              row_d = fmaf(__uint_as_float(a[i] & 0xFFFF0000u) + __uint_as_float(z[i] & 0xFFFF0000u),
                           __uint_as_float(e[i] & 0xFFFF0000u), row_d);
            }
          }
        }
        if (!ok) break;
        row_lse = sLse[r];
        float* part = sHalf + (items & 1) * 2 * TILE;
        part[half * TILE + r] = row_d;
        __syncwarp();
        if (lane == 0) bar_arrive(bar + A_EMPTY);
        pair_sync(1 + quarter);
        row_d = part[r] + part[TILE + r];
        if (half == 0 && real) p.dsum[ls] = row_d;
      }
      for (int j = 0, s_ = KEYS && it.j0 > 0 ? it.j0 % cs : 0; j < n; ++j, ++s_, ++g) {
        if (KEYS && s_ == cs) s_ = 0;
        const int st = g % B_STAGES;
        const int c0 = step_row<KEYS, BOX>(s_, cs, k0) + 32 * half;  // this warp's first column
        // Which of the 32 x 32 scores of this warp are visible? None, all, or some (see the forward).
        const int r0 = TILE * t + 32 * quarter;  // its first row
        bool live, part;
        if constexpr (KEYS) {
          live = c0 + 31 >= max(r0, it.qf) && c0 < it.len && (r0 < p.sinks || c0 < r0 + 31 + p.window);
          part = c0 < r0 + 31 || c0 < it.qf || c0 + 32 > it.len || (r0 + 32 > p.sinks && c0 + 32 - r0 > p.window);
        } else {
          live = c0 <= min(r0 + 31, it.len - 1) && r0 + 31 >= it.qf && (c0 < p.sinks || c0 + 31 > r0 - p.window);
          part = c0 + 31 > r0 || r0 < it.qf || r0 + 32 > it.len || (c0 + 32 > p.sinks && r0 + 32 - c0 > p.window);
        }
        uint32_t vm = ~0u;
        if (part) {
          if constexpr (KEYS) {
            const int hi = own < p.sinks ? it.len - 1 : min(it.len - 1, own + p.window - 1);
            vm = range_bits(max(own, it.qf) - c0, hi - c0, 0);
          } else {
            const int d = own >= it.qf && own < it.len ? own - c0 : -1;
            vm = range_bits(d - p.window + 1, d, 0) | range_bits(0, min(d, p.sinks - 1 - c0), 0);
          }
        }
        if ((KEYS && !warp_wait(bar + B_FULL + 8 * st, (g / B_STAGES) & 1, p.err, abort_flag)) ||
            !warp_wait(bar + S_FULL, g & 1, p.err, abort_flag) || (j == 0 && items > 0 && !write_grad(items - 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float4* lse4 = reinterpret_cast<const float4*>(sLse + st * BOX + 32 * half);
        const float4* d4 = reinterpret_cast<const float4*>(sD + st * BOX + 32 * half);
        const F2 sc = {-p.scale2, -p.scale2}, minus = {-1.f, -1.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 16 columns at a time: few registers
          uint32_t s[16], dp[16], pk[8], dk[8];
          if (live) {
            tmem_ld16(tS_own + 16 * c, s);
            tmem_ld16(tDP_own + 16 * c, dp);
            tmem_wait_ld();
          }
          if (c == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bar + S_EMPTY);
          }
          if (live) {
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              float4 lv = make_float4(row_lse, row_lse, row_lse, row_lse), dv = make_float4(row_d, row_d, row_d, row_d);
              if constexpr (KEYS) {
                lv = lse4[4 * c + k / 4];
                dv = d4[4 * c + k / 4];
              }
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const int i = k + e;
                const F2 x = fma2(pair_of(s + i), sc, e == 0 ? F2{lv.x, lv.y} : F2{lv.z, lv.w});  // lse - score
                F2 pr = {ex2(-x.x), ex2(-x.y)};
                if (part) {
                  if (!((vm >> (16 * c + i)) & 1u)) pr.x = 0.f;
                  if (!((vm >> (16 * c + i + 1)) & 1u)) pr.y = 0.f;
                }
                const F2 ds = mul2(pr, fma2(e == 0 ? F2{dv.x, dv.y} : F2{dv.z, dv.w}, minus, pair_of(dp + i)));
                const uint32_t hi = pack2(ds.x, ds.y);
                dk[i / 2] = hi;
                if constexpr (KEYS) {
                  pk[i / 2] = pack2(pr.x, pr.y);
                } else {  // what rounding took off dS
                  const F2 lo = add2(ds, {-__uint_as_float(hi << 16), -__uint_as_float(hi & 0xFFFF0000u)});
                  pk[i / 2] = pack2(lo.x, lo.y);
                }
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) pk[k] = dk[k] = 0u;
          }
          if (c == 0) {  // the last step's P and dS were consumed
            if (g > 0 && !warp_wait_held(bar + P_EMPTY, (g - 1) & 1, p.err, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          tmem_st8(tP_own + 8 * c, pk);
          tmem_st8(tDS_own + 8 * c, dk);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar + P_FULL);
      }
      if (!ok) break;
    }
    if (ok && items > 0) write_grad(items - 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, B_TMEM);
  }
}

// dV and dK of the sinks' tiles from their parts, in the parts' order. JOIN_ROWS rows a block;
// a thread = four neighbouring elements. Bound by its launch: 8 tiles of 8 parts, 64-wide heads: 3.6 us.
constexpr int JOIN_ROWS = 8;
template <int HD>
__global__ void __launch_bounds__(128) window_join_kernel(const Params p) {
  const int tile = blockIdx.x / (TILE / JOIN_ROWS), r0 = blockIdx.x % (TILE / JOIN_ROWS) * JOIN_ROWS;
  const int t = tile % p.stiles, bg = tile / p.stiles;
  const int g = bg % p.G, b = bg / p.G;
  const int kst = min(max(p.kstart[b], 0), p.Lk), len = p.Lk - kst;
  int k0, cs;
  key_steps(p, t, len, max(0, p.Lk - p.Lq - kst), k0, cs);
  const int parts = (cs * (p.H / p.G) + p.psteps - 1) / p.psteps;
  const float4* src = reinterpret_cast<const float4*>(p.partial + static_cast<long long>(tile) * p.parts * TILE * 2 * HD);
  constexpr int ROW = 2 * (HD / 4);
  for (int i = r0 * ROW + threadIdx.x; i < (r0 + JOIN_ROWS) * ROW; i += blockDim.x) {
    const int row = TILE * t + i / ROW, kv = i / (HD / 4) & 1, c = i % (HD / 4);  // kv 0: V, 1: K
    if (row >= len) break;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c2 = 0; c2 < parts; ++c2) {
      const float4 y = src[c2 * (TILE * ROW) + i];
      sum.x += y.x;
      sum.y += y.y;
      sum.z += y.z;
      sum.w += y.w;
    }
    const long long o = (static_cast<long long>(b) * p.Lk + kst + row) * (p.H + 2 * p.G) + (kv ? p.H + g : p.H + p.G + g);
    reinterpret_cast<uint2*>(p.dqkv + o * HD)[c] = make_uint2(pack2(sum.x, sum.y), pack2(sum.z, sum.w));
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

// [B, L, W] bf16, row stride ld and batch stride sb (elements); box 64 columns x 64 rows,
// 128-byte swizzle. Rows and columns outside read as zeros.
bool encode_rows(CUtensorMap* map, const void* base, uint64_t W, uint64_t L, uint64_t B, uint64_t ld, uint64_t sb) {
  thread_local bool bound = false;
  if (!bound) {
    cudaFree(nullptr);  // makes the device's primary context current on this thread
    bound = true;
  }
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {W, L, B};
  cuuint64_t strides[2] = {ld * 2, sb * 2};
  cuuint32_t box[3] = {64, BOX, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `heads` x B x `tiles` items over a grid of `grid` blocks.
Params make_params(const WindowAttnArgs& a, int heads, int tiles, int stride) {
  Params p;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.out_lo = static_cast<__nv_bfloat16*>(a.out_lo);
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
  p.stiles = 0;
  p.parts = 1;
  p.psteps = 0;
  p.partial = a.partial;
  p.heads = heads;
  p.tiles = tiles;
  p.dh = stride % heads;
  p.db = stride / heads % a.B;
  p.di = stride / heads / a.B;
  p.scale = a.scale;
  p.scale2 = a.scale * kLog2e;
  p.err = a.err;
  return p;
}

constexpr int kMaxDevices = 64;

int device_index() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}

int num_sms(int dev) {
  static std::atomic<int> n[kMaxDevices];
  int v = n[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
    n[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool shapes_ok(const WindowAttnArgs& a) {
  return (a.hd == 32 || a.hd == 64) && a.B > 0 && a.H > 0 && a.G > 0 && a.H % a.G == 0 && a.Lq > 0 && a.Lq <= a.Lk &&
         a.window > 0 && a.sinks >= 0 && a.kstart != nullptr && a.qkv != nullptr && a.out != nullptr &&
         a.lse != nullptr && aligned16(a.qkv) && aligned16(a.out) && a.ld % 8 == 0 && a.sb % 8 == 0 && a.ld > 0 &&
         a.sb > 0;
}

// Raises a kernel's shared memory limit, once a device (an error is returned, not kept).
template <typename K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<bool>* done) {
  if (done->load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done->store(true, std::memory_order_relaxed);
  return e;
}

// How the sinks' key tiles are cut. Every query sees them, so that with few samples and a long
// history one of them is the critical path: from three quarters of a block's average load on it
// comes in parts of about half that load, joined by a second kernel. Backward of 2 samples of 8,191
// tokens, 8 query heads on 2 key heads of 64, window 128 + 4: 751 us in one piece, 116 in 33; of 8
// samples, 4 heads, window 1,024 + 16 (0.95 of the load): 563 and 497; of 16 samples of 2,000, 8
// heads of 32, window 256 + 8 (0.54 of the load): 159, and 169 in two.
struct Cut {
  int stiles = 0, parts = 1, psteps = 1;
};
Cut cut_of(const WindowAttnArgs& a) {
  Cut c;
  const long long group = a.H / a.G, ktiles = (a.Lk + TILE - 1) / TILE;
  const int window = std::min(a.window, a.Lk), sinks = std::min(a.sinks, a.Lk);
  c.stiles = (sinks + TILE - 1) / TILE;
  if (c.stiles == 0) return c;
  const long long most = (std::min(a.Lq, a.Lk) + BOX - 1) / BOX * group + group;  // steps of a sinks' tile
  const long long usual = std::min<long long>(most, ((window + TILE) / BOX + 1) * group);
  const long long total = static_cast<long long>(a.B) * a.G * (c.stiles * most + (ktiles - c.stiles) * usual);
  const long long load = total / (2LL * num_sms(device_index())) + 1;
  const long long steps = std::max<long long>(16, load / 2);
  const long long parts = (most + steps - 1) / steps;
  if (4 * most <= 3 * load || parts < 2) return c;
  c.parts = static_cast<int>(parts);
  c.psteps = static_cast<int>(steps);
  return c;
}

int grid_of(long long heads, long long samples, long long tiles, long long most) {
  return static_cast<int>(std::min(heads * samples * tiles, most));
}

template <int HD>
cudaError_t fwd_hd(const WindowAttnArgs& a, cudaStream_t stream) {
  static std::atomic<bool> ready[kMaxDevices];
  const int dev = device_index();
  const int tiles = (a.Lq + TILE - 1) / TILE + 1;
  const int grid = grid_of(a.H, a.B, tiles, 2LL * num_sms(dev));  // the second chains start where the first ones end
  const Params p = make_params(a, a.H, tiles, CHAINS * grid);
  const uint64_t W = static_cast<uint64_t>(a.H + 2 * a.G) * HD;
  const auto* base = static_cast<const __nv_bfloat16*>(a.qkv);
  CUtensorMap tq, tkv;
  if (!encode_rows(&tq, base + (a.Lk - a.Lq) * a.ld, W, a.Lq, a.B, a.ld, a.sb) ||
      !encode_rows(&tkv, base, W, a.Lk, a.B, a.ld, a.sb))
    return cudaErrorInvalidValue;
  const cudaError_t e = allow_smem(window_fwd_kernel<HD>, F_SMEM, &ready[dev]);
  if (e != cudaSuccess) return e;
  window_fwd_kernel<HD><<<grid, F_THREADS, F_SMEM, stream>>>(tq, tkv, p);
  return cudaGetLastError();
}

template <int HD>
cudaError_t bwd_hd(const WindowAttnArgs& a, cudaStream_t stream) {
  static std::atomic<bool> ready_q[kMaxDevices], ready_k[kMaxDevices];
  const int dev = device_index();
  const uint64_t W = static_cast<uint64_t>(a.H + 2 * a.G) * HD, D = static_cast<uint64_t>(a.H) * HD;
  const auto* base = static_cast<const __nv_bfloat16*>(a.qkv);
  CUtensorMap tq, tkv, tdo;
  if (!encode_rows(&tq, base + (a.Lk - a.Lq) * a.ld, W, a.Lq, a.B, a.ld, a.sb) ||
      !encode_rows(&tkv, base, W, a.Lk, a.B, a.ld, a.sb) || !encode_rows(&tdo, a.dout, D, a.Lq, a.B, D, D * a.Lq))
    return cudaErrorInvalidValue;
  cudaError_t e = allow_smem(window_bwd_kernel<HD, false>, B_SMEM, &ready_q[dev]);
  if (e == cudaSuccess) e = allow_smem(window_bwd_kernel<HD, true>, B_SMEM, &ready_k[dev]);
  if (e != cudaSuccess) return e;
  const long long most = 2LL * num_sms(dev);
  const Cut cut = cut_of(a);
  if (cut.parts > 1 && a.partial == nullptr) return cudaErrorInvalidValue;
  const int qtiles = (a.Lq + TILE - 1) / TILE + 1;
  const int ktiles = (a.Lk + TILE - 1) / TILE + cut.stiles * (cut.parts - 1);
  const int qgrid = grid_of(a.H, a.B, qtiles, most), kgrid = grid_of(a.G, a.B, ktiles, most);
  // queries first: they leave D behind
  window_bwd_kernel<HD, false><<<qgrid, B_THREADS, B_SMEM, stream>>>(tq, tkv, tdo,
                                                                           make_params(a, a.H, qtiles, qgrid));
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  Params pk = make_params(a, a.G, ktiles, kgrid);
  pk.stiles = cut.stiles;
  pk.parts = cut.parts;
  pk.psteps = cut.psteps;
  window_bwd_kernel<HD, true><<<kgrid, B_THREADS, B_SMEM, stream>>>(tq, tkv, tdo, pk);
  e = cudaGetLastError();
  if (e != cudaSuccess || cut.parts == 1) return e;
  window_join_kernel<HD><<<a.B * a.G * cut.stiles * (TILE / JOIN_ROWS), 128, 0, stream>>>(pk);
  return cudaGetLastError();
}

}  // namespace

long long window_attn_workspace(const WindowAttnArgs& a) {
  if (!shapes_ok(a)) return 0;
  const Cut c = cut_of(a);
  return c.parts == 1 ? 0 : static_cast<long long>(a.B) * a.G * c.stiles * c.parts * TILE * 2 * a.hd;
}

cudaError_t window_attn_fwd(const WindowAttnArgs& a, cudaStream_t stream) {
  if (!shapes_ok(a)) return cudaErrorInvalidValue;
  return a.hd == 64 ? fwd_hd<64>(a, stream) : fwd_hd<32>(a, stream);
}

cudaError_t window_attn_bwd(const WindowAttnArgs& a, cudaStream_t stream) {
  if (!shapes_ok(a) || a.dout == nullptr || a.dqkv == nullptr || a.dsum == nullptr || a.out_lo == nullptr ||
      !aligned16(a.dout) || !aligned16(a.dqkv) || !aligned16(a.out_lo))
    return cudaErrorInvalidValue;
  return a.hd == 64 ? bwd_hd<64>(a, stream) : bwd_hd<32>(a, stream);
}

}  // namespace mdl
