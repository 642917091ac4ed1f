// Attention of a tree of drafted tokens over a paged GQA cache (sm_100a).
//
// Sequence b holds ctx committed keys and, behind them in node order, the keys of its n tree
// nodes; the query of node i sees
//   * the context, or with a sliding window the keys t > ctx + depth[i] - window of it, and
//   * the nodes j whose bit is set in row i of the mask (its ancestors and itself; with a
//     window those of depth[j] > depth[i] - window),
//   o_i = sum_t p_it v_t,  p_it = exp(s q_i . k_t - m) / (sum_t exp(s q_i . k_t - m) [+ exp(sink - m)]).
// A row that sees nothing is zero.  Keys that a row does not see never reach its result,
// whatever bits they hold (see "masked pages").
//
// Rows: the G = Hq / Hkv heads of a KV head and the nodes form n * G query rows (row r = node
// r / G, head r % G), so one pass over the keys serves them all.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cfloat>
#include <climits>
#include <cstdint>
#include "launch.cuh"
#include "ptx.cuh"

namespace xtu {
namespace {

constexpr int TA_PAGE = 64;          // keys per cache block
constexpr float LOG2E = 1.4426950408889634f;

struct TaParams {
  const __nv_bfloat16* q;   // [T, Hq, D]
  long long q_ts;           // elements between tokens
  int q_hs;                 // elements between heads
  __nv_bfloat16* o;         // [T, Hq, DV] contiguous
  const int* q_start;       // [B + 1]
  const int* kv_len;        // [B] context + nodes
  const int* block_table;   // [B, bt_stride], bt_cols columns
  int bt_stride, bt_cols;
  const int* mask;          // [T, W]
  int W;
  const int* depth;         // [T] (window > 0 only)
  int window;
  int Hq, Hkv, G, T;
  uint32_t g_inv;           // ceil(2^32 / G): x / G for x < 2^25 (G = 1: unused)
  float scale_log2;         // softmax scale * log2(e) (fp8: times the K scale)
  float out_scale;          // fp8: the V scale, else 1
  const float* sinks;       // [Hq] or null
  int splits;
  float* ws_o;              // [splits, T, Hq, DV] normalised partials (splits > 1)
  float* ws_lse;            // [splits, T, Hq] m + log2(l), -FLT_MAX for an empty one
  const void* v_raw;        // V cache (non-finite values of masked pages)
  int num_blocks;
  int max_nodes;            // rows of the grid
  XtuStatus* status;
};

// query row -> node
__device__ __forceinline__ int ta_node(const TaParams& p, int row) {
  return p.G == 1 ? row : (int)__umulhi((uint32_t)row, p.g_inv);
}

__device__ __forceinline__ float ta_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __noinline__ bool ta_wait_on(uint64_t* bar, uint32_t parity, XtuStatus* st, uint32_t where,
                                        uint64_t limit_ns) {
  return mbar_wait(bar, parity, st, where, limit_ns);
}

// mbar_wait behind a few tries of its own: it reads the global timer after one failed try, and
// the read (hundreds of cycles) sat on the critical path of waits that were over sooner
__device__ __forceinline__ bool ta_wait(uint64_t* bar, uint32_t parity, XtuStatus* st, uint32_t where,
                                        uint64_t limit_ns = kIntraCtaWaitNs) {
#pragma unroll 1
  for (int it = 0; it < 64; ++it)
    if (mbar_try_wait(bar, parity)) return true;
  return ta_wait_on(bar, parity, st, where, limit_ns);
}

// a first look whose answer is used later: the looks of several barriers are under way together
__device__ __forceinline__ bool ta_look(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

// ---------------------------------------------------------------------------------------
// visibility
// ---------------------------------------------------------------------------------------
struct TaRow {
  const int* words;   // mask row, null: the row sees nothing
  int ctx, n;         // committed keys, nodes
  int low;            // first context key inside the window
  int deep;           // window: nodes of depth <= deep are outside (INT_MIN: none)
};

__device__ __forceinline__ TaRow ta_row(const TaParams& p, int q0, int n, int ctx, int node, bool valid) {
  TaRow r;
  r.words = valid ? p.mask + (size_t)(q0 + node) * p.W : nullptr;
  r.ctx = ctx;
  r.n = n;
  r.low = 0;
  r.deep = INT_MIN;
  if (p.window > 0 && valid) {
    const int far = min(max(__ldg(p.depth + q0 + node), 0), n - 1) - p.window;
    r.low = max(0, ctx + far + 1);
    r.deep = far;
  }
  return r;
}

// bits of keys key0 .. key0 + 31 that the row sees
// (not inlined: rare, and code that is never run costs fetches of the code that is)
__device__ __noinline__ uint32_t ta_see32(const TaParams& p, const TaRow& r, int q0, int key0) {
  if (r.words == nullptr) return 0u;
  const int off = key0 - r.ctx;              // node index of key0
  uint32_t bits = 0u;
  if (off > -32 && off < r.n) {
    const int lo = off >= 0 ? off >> 5 : -1;
    const uint32_t w0 = lo >= 0 && lo < p.W ? (uint32_t)__ldg(r.words + lo) : 0u;
    const uint32_t w1 = lo + 1 < p.W ? (uint32_t)__ldg(r.words + lo + 1) : 0u;
    const int sh = off & 31;
    bits = sh ? __funnelshift_r(w0, w1, sh) : (off >= 0 ? w0 : w1);
    const int left = r.n - off;              // nodes from key0 on
    if (left < 32) bits &= (1u << left) - 1u;
    if (r.deep >= 0) {                       // ancestors outside the window
      for (uint32_t m = bits; m; m &= m - 1) {
        const int e = __ffs(m) - 1;
        if (__ldg(p.depth + q0 + off + e) <= r.deep) bits &= ~(1u << e);
      }
    }
  }
  if (off < 0) {                             // context keys key0 .. ctx - 1
    uint32_t c = off <= -32 ? 0xffffffffu : (1u << -off) - 1u;
    const int cut = r.low - key0;
    if (cut >= 32) c = 0u;
    else if (cut > 0) c &= ~((1u << cut) - 1u);
    bits = (off <= -32 ? 0u : bits & ~((1u << -off) - 1u)) | c;
  }
  return bits;
}

__device__ __forceinline__ bool ta_sees(const TaParams& p, const TaRow& r, int q0, int key) {
  return (ta_see32(p, r, q0, key & ~31) >> (key & 31)) & 1u;
}

__device__ __forceinline__ float ta_v_at(const TaParams& p, bool f8, int DV, int page, int kh, int off, int d) {
  if (f8) {
    const uint8_t x = static_cast<const uint8_t*>(p.v_raw)[(((size_t)page * p.Hkv + kh) * DV + d) * TA_PAGE + off];
    const __half_raw h = __nv_cvt_fp8_to_halfraw(x, __NV_E4M3);
    return __half2float(__half(h));
  }
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p.v_raw)[(((size_t)page * p.Hkv + kh) * TA_PAGE + off) * DV + d]);
}

// a row's output (32-bit partial or bf16 result; its columns d0 .. d1 - 1) plus the non-finite
// values of the keys of logical page pg that it sees
__device__ __noinline__ void ta_add_bad(const TaParams& p, const TaRow& r, bool f8, int q0, int b, int kh, int pg, int DV,
                                        int d0, int d1, float* wo, __nv_bfloat16* o) {
  const int page = __ldg(p.block_table + (size_t)b * p.bt_stride + pg);
  if (page < 0 || page >= p.num_blocks) return;
#pragma unroll 1
  for (int k = 0; k < TA_PAGE; ++k) {
    if (!ta_sees(p, r, q0, pg * TA_PAGE + k)) continue;
#pragma unroll 1
    for (int d = d0; d < d1; ++d) {
      const float y = ta_v_at(p, f8, DV, page, kh, k, d);
      if (isfinite(y)) continue;
      if (wo != nullptr) wo[d] += y;
      else o[d] = __float2bfloat16(__bfloat162float(o[d]) + y);
    }
  }
}

__device__ __forceinline__ void tm_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {   // exact
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t tm_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// non-finite bf16 values of a packed pair as a mask of the halves to clear
__device__ __forceinline__ uint32_t bad_bf16x2(uint32_t w) {
  return ((w & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
}

// ---------------------------------------------------------------------------------------
// the kernel: 128-row tiles, S, P and O in tensor memory
// ---------------------------------------------------------------------------------------
// One CTA = ROWT row tiles of 128 query rows of one (sequence, kv head, kv split).  Softmax units of
// 128 threads, a thread a row, keep the tensor core busy in turn:
//   ROWT = 2  two units; unit u owns row tile u, and every K / V tile serves both
//   ROWT = 1  three units (fp8 caches: two) share the rows, one accumulator and one running maximum; unit u
//             takes the key tiles t = u (mod 3), and S runs three tiles ahead in buffers of its own
//   warp 0       TMA producer: key tiles of BN keys into a ring (ROWT = 1: one for K, which runs ahead, one for V)
//   warp 1       MMA issuer: S = Q K^T into TMEM, O += P V with P from TMEM
//   warp 2       ROWT = 2: gives the ring's slots back
//   warps 4 ..   the units: S -> registers, mask, online softmax, P (16 bit) over S's columns
//   last 4       fp8 caches: raw e4m3 tiles -> f16 operand tiles (exact)
// ROWT = 2: the issuer alternates PV_u(t), S_u(t + 1): S_u's completion (one commit) also tells unit u that
// PV_u(t) is done, so P and O need no barriers of their own and S and P share columns.  ROWT = 1: PV(t), S(t + 3)
// into the buffer that P(t) leaves; a unit that has to rescale O waits for the release of V(t - 1)'s slot.
//
// What bounds it.  ROWT = 2: a unit's way from S to the next S (TMEM load, max, 128 ex2, P, 256 + 512 cycles
// of MMA, and about 900 cycles of hand-overs) is 3300 cycles per 128-key tile while the
// other unit's runs beside it; the MMAs of both take 2048 of them.  Measured with parts left
// out: no exponentials -6 %, no softmax at all -8 %, 1/8 of the S products -27 %: the
// chain, not one pipe.  Variants that were slower: two warps a row with half a row's keys each (266
// against 227 us, 61-node case), 64-key tiles with S double-buffered (281: an N = 64 MMA costs as
// much as an N = 128 one), ex2 partly as a cubic on the FMA pipe (no change), the maximum
// taken between the exponentials (246: registers; with registers moved from the other warps no change).
// ROWT = 1 takes that chain off the way of S (two units on alternate tiles with an accumulator each: 1.2 us a
// tile against 0.85; 16 / 2 heads of 256 62.8 -> 57 us).  V of a masked tile is cleaned after the wait for S: before it,
// V's arrival cannot be told by the parity of its barrier.  In long runs the card's power limit binds:
// 1.65 of 1.97 GHz.
// 4 sequences x 14.6K keys, 96 / 8 heads of 128 (KV 240 MB, 36 us at the copy rate), a call among others:
//   60 rows a KV head   50 us (0.73 of the copy rate);  192 rows 67 to 82;  480 rows 112
//   732 rows            172 to 204 us (153 GFLOP: 0.45 to 0.53 of the GEMM rate, MMA pipe 52 % busy, XU 52 %)
//   192 rows over the fp8 cache  79 to 88 us: the same chain, and the second read of S that 128 registers
//                       force (one read with registers moved: no change); its bytes are 18 us
// 16 sequences of up to 12K keys, 16 / 2 heads of 256: 55 to 61 us (197 MB: 30 us; N = 64 products).  A CTA's start
// and end cost about 6 us, and 9 to 16 us is a call over a few pages.  Split counts: ops/tree.py.
//
// Masked pages: a tile that hides a key from some row of the CTA (the tree's own, the last, those a
// window cuts) is masked bit by bit in S, and V's non-finite values are zeroed in shared memory
// first, since 0 * NaN would reach every row; the rows that do see such a key get it at the end.
template <int D_, int DVT_, int BN_, int ROWT_, int SK_, int SV_, int NR_ = 0>
struct TtCfg {
  static constexpr int D = D_, DVT = DVT_, BN = BN_, ROWT = ROWT_;
  static constexpr int NR = NR_;                       // slots of the raw ring (fp8 caches)
  static constexpr bool F8 = NR > 0;
  // ROWT = 1: one accumulator, with one running maximum that goes from tile to tile (unit to unit), which
  // leaves tensor memory for a third S
  static constexpr bool SHARE = ROWT == 1;
  static constexpr int SK = SK_, SV = SV_;
  static constexpr int NO = SHARE ? 1 : 2;             // accumulators
  static constexpr int NSB = SHARE ? 3 : 2;            // S buffers: tile t in t % 3, or one a unit
  static constexpr int LEAD = SHARE ? 3 : 1;           // K tiles loaded before the first V: K(t + LEAD) follows V(t)
  static constexpr int RAW = BN * D;                   // bytes of an fp8 tile
  static constexpr int Q_BYTES = ROWT * 128 * D * 2;
  static constexpr int K_BYTES = BN * D * 2, V_BYTES = BN * DVT * 2;
  // ROWT = 2: one ring of SK + SV slots where a K and a V tile are the same size (K0 V0 K1 V1 ..; the count
  // may be odd); else a ring each
  static constexpr bool ONE = !SHARE && K_BYTES == V_BYTES;
  static constexpr int NS = SK + SV, RING = SK * K_BYTES + SV * V_BYTES;
  __device__ static int k_slot(int t) { return ONE ? 2 * t % NS : t % SK; }
  __device__ static int v_slot(int t) { return ONE ? (2 * t + 1) % NS : SK + t % SV; }
  __device__ static int k_turn(int t) { return ONE ? 2 * t / NS : t / SK; }          // how often the slot was filled before
  __device__ static int v_turn(int t) { return ONE ? (2 * t + 1) / NS : t / SV; }
  __device__ static int slot_at(int s) { return ONE || s < SK ? s * K_BYTES : SK * K_BYTES + (s - SK) * V_BYTES; }
  // tile t's K (V) slot is filled again before the last of nt tiles
  __device__ static bool k_again(int t, int nt) { return ONE ? 2 * t + NS < 2 * nt : t + SK < nt; }
  __device__ static bool v_again(int t, int nt) { return ONE ? 2 * t + 1 + NS < 2 * nt : t + SV < nt; }
  // the in-th tile that is loaded (of 2 * nt): K or V, and its number
  __device__ static bool order(int in, int nt, int& t) {
    const int lead = LEAD < nt ? LEAD : nt, j = in - lead, pairs = nt - lead;
    if (j < 0) { t = in; return false; }
    if (j >= 2 * pairs) { t = j - pairs; return true; }
    t = (j & 1) ? (j >> 1) + lead : j >> 1;
    return !(j & 1);
  }
  static constexpr int BARS = 2 * NS + 2 * NR + 4 + 3 * NSB;
  static constexpr int BYTES = Q_BYTES + RING + NR * RAW + BARS * 8 + 16 + (SHARE ? 1024 : 0);
  static constexpr int O_COL = NSB * BN;               // S0 S1 (S2) | O0 (O1)
  static constexpr int COLS = 512;                     // (every tiling takes more than 256)
  static constexpr int UNITS = SHARE && !F8 ? 3 : 2;   // softmax units of 128 threads
  static constexpr int THREADS = 128 + 128 * UNITS + (F8 ? 128 : 0);
  // with 128 registers a thread a unit takes 128 scores in two halves
  static constexpr bool HALVES = THREADS == 512 && BN == 128;
  static constexpr int P_COL = HALVES ? BN / 2 : 0;    // P's first column in S's
  static_assert(NSB * BN + NO * DVT <= 512, "tensor memory");
  // ROWT = 2 gives V(t)'s slot back once S of tile t + 1 stands, whose K the producer must have loaded
  // before it comes to wait for that slot
  static_assert(ROWT == 1 || (ONE ? NS / 2 : SV) >= 1, "the ring would wait for itself");
  static_assert(BYTES <= 232448, "shared memory");
  // ROWT = 1: a unit at tile t takes the release of V(t - 1)'s slot for the end of its product.  The slot's release
  // before that has to be over by then: it is tile t - 3's or older, whose product stands before S(t)
  static_assert(!SHARE || SV >= 2, "the release of a V slot would be ambiguous");
  // ROWT = 2: what was in V(t)'s slot before is K(t - 1), V(t - 2) or older, whose fill is over when a unit comes to tile t
  static_assert(SHARE || (ONE ? NS >= 3 : SV >= 2), "the fill of a V slot would be ambiguous");
  static_assert(D % 64 == 0 && DVT % 64 == 0 && BN % 64 == 0 && NS >= 3 && (!F8 || (D == DVT && BN == 128 && NR >= 2)), "tiles");
};

// 16 bytes to shared memory without a register stop; zeros when `there` is false
__device__ __forceinline__ void tt_copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// a row's running maximum with the tile that it is of, as one 64-bit word of shared memory (the parts of a vector
// access need not be seen together)
__device__ __forceinline__ void ta_row_max_to(uint64_t* at, float m, int tile) {
  asm volatile("{\n\t.reg .b64 x;\n\tmov.b64 x, {%1, %2};\n\tst.volatile.shared.b64 [%0], x;\n\t}" ::"r"(smem_u32(at)),
               "r"(__float_as_int(m)), "r"(tile)
               : "memory");
}
__device__ __forceinline__ float ta_row_max(const uint64_t* at, int tile, bool& ok) {   // waits for that tile, bounded
  int m, of, it = 0;
#pragma unroll 1
  do {
    asm volatile("{\n\t.reg .b64 x;\n\tld.volatile.shared.b64 x, [%2];\n\tmov.b64 {%0, %1}, x;\n\t}"
                 : "=r"(m), "=r"(of)
                 : "r"(smem_u32(at))
                 : "memory");
  } while (of != tile && ++it < (1 << 24));
  ok = of == tile;
  return __int_as_float(m);
}

// pairs of floats in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <bool F8>
__device__ __forceinline__ uint32_t tt_bad(uint32_t w) {   // the halves to clear of a pair in the operand tile
  return F8 ? ((w & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u)
            : bad_bf16x2(w);
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1) tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tk,
                                                                     const __grid_constant__ CUtensorMap tv,
                                                                     const __grid_constant__ TaParams p) {
  griddep_wait();
  constexpr int D = C::D, DVT = C::DVT, BN = C::BN, ROWT = C::ROWT;
  constexpr int PPT = BN / TA_PAGE;                    // pages of a key tile
  extern __shared__ __align__(1024) uint8_t tt_smem[];   // (the swizzle atoms' alignment)
  uint8_t* sQ = tt_smem;
  uint8_t* sK = sQ + C::Q_BYTES;                       // the ring
  uint8_t* raw = sK + C::RING;                         // fp8 tiles as they lie in the cache
  uint64_t* full = reinterpret_cast<uint64_t*>(raw + C::NR * C::RAW);
  uint64_t* empty = full + C::NS;
  uint64_t* r_full = empty + C::NS;                    // [NR]
  uint64_t* r_empty = r_full + C::NR;                  // [NR]
  uint64_t* q_ready = r_empty + C::NR;
  uint64_t* s_full = q_ready + 1;                      // [NSB]
  uint64_t* p_full = s_full + C::NSB;                  // [NSB][2] halves of P
  uint64_t* o_done = p_full + 2 * C::NSB;                     // [2], and one for an issuer that gives up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 3);
  int& s_bad = *reinterpret_cast<int*>(tmem_slot + 1);   // a masked tile held a non-finite value
  // SHARE: [128] the rows' running maximum, and the tile that it is of: the unit of the next tile waits for it.  (A
  // barrier and a load behind it took 500 cycles more a tile.)
  uint64_t* m_row = reinterpret_cast<uint64_t*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kh = blockIdx.y;
  // row tiles of one split lie next to each other, so that they meet the same K / V in L2
  const int rt = gridDim.x / p.splits;
  const int sp = blockIdx.x / rt, tile = blockIdx.x - sp * rt;
  const int q0 = __ldg(p.q_start + b), q1 = __ldg(p.q_start + b + 1);
  const bool inside = q0 >= 0 && q0 <= q1 && q1 <= p.T;   // rows outside the call's tensors: no tree here, and told
  const int n = inside ? q1 - q0 : 0;
  const int L = __ldg(p.kv_len + b), ctx = L - n;
  const int r0 = tile * (128 * ROWT);
  const int rows_all = min(n, p.max_nodes) * p.G;
  if (r0 >= rows_all) {                                // uniform: no such row tile here
    if (!inside && threadIdx.x == 0) report_error(p.status, XTU_ERR_BOUNDS, 247, q1);
    griddep_launch_dependents();
    return;
  }
  const int npages = min((L + TA_PAGE - 1) / TA_PAGE, p.bt_cols);
  const int ntile_all = (npages + PPT - 1) / PPT;
  const int tfirst = p.window > 0 ? max(0, ctx - p.window + 1) / BN : 0;
  const int per = (ntile_all - tfirst + p.splits - 1) / p.splits;
  const int t0 = min(ntile_all, tfirst + sp * per), t1 = min(ntile_all, t0 + per);
  const int nt = max(0, t1 - t0);
  // tiles at or past `shut` or below `open` hide keys from some rows (see the masked pages above)
  const int shut = ctx / BN;
  const int open = p.window > 0 ? (max(0, ctx + n - p.window) + BN - 1) / BN : 0;
  const bool two = ROWT == 2 && r0 + 128 < rows_all;   // unit 1 has a row tile

  if (threadIdx.x == 0) {
    // (nodes that the grid does not cover, keys that the table does not name: cut, and told)
    if (n > p.max_nodes) report_error(p.status, XTU_ERR_BOUNDS, 245, n);
    if (L > p.bt_cols * TA_PAGE) report_error(p.status, XTU_ERR_BOUNDS, 246, L);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    s_bad = 0;
    for (int i = 0; i < C::NS; ++i) { mbar_init(&full[i], C::F8 ? 4 : 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < C::NR; ++i) { mbar_init(&r_full[i], 1); mbar_init(&r_empty[i], 4); }
    mbar_init(q_ready, 4 * C::UNITS);
    for (int i = 0; i < 2; ++i) mbar_init(&o_done[i], 1);
    for (int i = 0; i < C::NSB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], ROWT == 2 && i == (two ? 1 : 0) ? 5 : 4);   // (and warp 2's)
    }
    fence_barrier_init();
  }
  if (C::SHARE && threadIdx.x >= 128 && threadIdx.x < 256) ta_row_max_to(&m_row[threadIdx.x - 128], 0.f, -1);
  if (warp == 1) tmem_alloc(tmem_slot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // dependents may start only now: one that took this SM's tensor memory first, and waits for
  // this grid, would never give it back
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one() && nt > 0) {
      const int* bt = p.block_table + (size_t)b * p.bt_stride;
      // rows of the pages of tile t (the caches' zero fill where there is no page)
      auto row_of = [&](int t, int sb) {
        const int lp = (t0 + t) * PPT + sb;
        int pg = lp < npages ? __ldg(bt + lp) : p.num_blocks;
        if (lp < npages) (void)XTU_IN_BOUNDS(pg >= 0 && pg < p.num_blocks, p.status, 244, pg);
        if (pg < 0 || pg > p.num_blocks) pg = p.num_blocks;
        return (pg * p.Hkv + kh) * TA_PAGE;
      };
      // (a V tile's pages are looked up with its K's; LEAD is 1 or 3)
      int krow[PPT], vrow[C::LEAD][PPT];
      bool ok = true;
      int in = 0, kn = 0, vn = 0;
#pragma unroll
      for (int sb = 0; sb < PPT; ++sb) krow[sb] = row_of(0, sb);
      for (; in < 2 * nt && ok; ++in) {
        int t;
        const bool isv = C::order(in, nt, t);
        int rows[PPT];
#pragma unroll
        for (int sb = 0; sb < PPT; ++sb) rows[sb] = isv ? vrow[0][sb] : krow[sb];
        if constexpr (C::F8) {   // as they lie: K [64 keys][D bytes], V [DV columns][64 keys] a page
          const int slot = in % C::NR, turn = in / C::NR;
          ok = turn == 0 || ta_wait(&r_empty[slot], (turn - 1) & 1, p.status, 150);
          if (!ok) break;
          mbar_arrive_expect_tx(&r_full[slot], C::RAW);
#pragma unroll
          for (int sb = 0; sb < PPT; ++sb)
            tma_load_2d(raw + slot * C::RAW + sb * TA_PAGE * D, isv ? &tv : &tk, &r_full[slot], 0,
                        isv ? rows[sb] / TA_PAGE * DVT : rows[sb]);
        } else {
          const int slot = isv ? C::v_slot(t) : C::k_slot(t), turn = isv ? C::v_turn(t) : C::k_turn(t);
          ok = turn == 0 || ta_wait(&empty[slot], (turn - 1) & 1, p.status, isv ? 151 : 150);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[slot], isv ? C::V_BYTES : C::K_BYTES);
          uint8_t* dst = sK + C::slot_at(slot);
#pragma unroll
          for (int sb = 0; sb < PPT; ++sb)
#pragma unroll
            for (int c = 0; c < (D > DVT ? D : DVT) / 64; ++c)
              if (c < (isv ? DVT : D) / 64)
                tma_load_2d(dst + c * (BN * 128) + sb * (TA_PAGE * 128), isv ? &tv : &tk, &full[slot], c * 64, rows[sb]);
        }
        if (isv) {
          ++vn;
#pragma unroll
          for (int k = 0; k + 1 < C::LEAD; ++k)
#pragma unroll
            for (int sb = 0; sb < PPT; ++sb) vrow[k][sb] = vrow[k + 1][sb];
        } else {   // queue the pages for V, look up the next tile's while slots get free
          const int at = C::LEAD == 1 ? 0 : kn - vn;
#pragma unroll
          for (int k = 0; k < C::LEAD; ++k)
#pragma unroll
            for (int sb = 0; sb < PPT; ++sb) vrow[k][sb] = k == at ? krow[sb] : vrow[k][sb];
          ++kn;
          if (kn < nt) {
#pragma unroll
            for (int sb = 0; sb < PPT; ++sb) krow[sb] = row_of(kn, sb);
          }
        }
      }
      // the copies in flight land (bounded) before the CTA ends, also when another warp gave up: the last fill of
      // every slot
      auto landed = [&](uint64_t* bar, int turn) { ta_wait(bar, turn & 1, nullptr, 0, 50000000ull); };
      if constexpr (C::F8) {
        for (int i = max(0, in - C::NR); i < in; ++i) landed(&r_full[i % C::NR], i / C::NR);
      } else if constexpr (C::ONE) {
        for (int i = max(0, in - C::NS); i < in; ++i) landed(&full[i % C::NS], i / C::NS);
      } else {
        for (int t = max(0, kn - C::SK); t < kn; ++t) landed(&full[C::k_slot(t)], C::k_turn(t));
        for (int t = max(0, vn - C::SV); t < vn; ++t) landed(&full[C::v_slot(t)], C::v_turn(t));
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one() && nt > 0) {
      // (fp8: f16 operands, type bits 0; V lies [column][key] and is K-major)
      constexpr uint32_t types = (1u << 7) | (1u << 10);
      constexpr uint32_t id_s = C::F8 ? idesc_bf16_f32(128, BN, 0, 0) & ~types : idesc_bf16_f32(128, BN, 0, 0);
      constexpr uint32_t id_o = C::F8 ? idesc_bf16_f32(128, DVT, 0, 0) & ~types : idesc_bf16_f32(128, DVT, 0, 1);
      bool ok = ta_wait(q_ready, 0, p.status, 152);
      auto wait_k = [&](int t) { return ta_wait(&full[C::k_slot(t)], C::k_turn(t) & 1, p.status, 153); };
      auto wait_v = [&](int t) { return ta_wait(&full[C::v_slot(t)], C::v_turn(t) & 1, p.status, 154); };
      // S = Q K^T of tile t into buffer sb (ROWT = 2: of unit sb)
      auto mma_s = [&](int sb, int t) {
        const uint64_t qd = sdesc_kmajor_sw128(smem_u32(sQ) + (ROWT == 2 ? sb * (128 * D * 2) : 0));
        const uint64_t kd = sdesc_kmajor_sw128(smem_u32(sK + C::slot_at(C::k_slot(t))));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)   // (descriptors count 16 bytes)
          mma_f16_ss(tmem + sb * BN, qd + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16,
                     kd + ((k >> 2) * (BN * 128) + (k & 3) * 32) / 16, id_s, k > 0);
        mma_commit(&s_full[sb]);
      };
      // O (of accumulator o) += P V of tile t, the two halves of the keys as P gets ready in buffer sb
      auto mma_o = [&](int o, int sb, int t, int phase) {
        const uint32_t va = smem_u32(sK + C::slot_at(C::v_slot(t)));
        const uint64_t vd = C::F8 ? sdesc_kmajor_sw128(va) : sdesc_mnmajor_sw128(va, BN * 128, 1024);
        const bool there[2] = {ta_look(&p_full[2 * sb], phase), ta_look(&p_full[2 * sb + 1], phase)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!there[h] && !ta_wait(&p_full[2 * sb + h], phase, p.status, 155)) return false;
          tc_fence_after();
#pragma unroll
          for (int e = 0; e < BN / 32; ++e) {
            const int k = (h ^ C::HALVES) * (BN / 32) + e;             // (halves: the second half of the keys first)
            mma_f16_ts(tmem + C::O_COL + o * DVT, tmem + sb * BN + C::P_COL + k * 8,
                       vd + (C::F8 ? ((k >> 2) * (DVT * 128) + (k & 3) * 32) / 16 : k * 128), id_o,
                       !(t == 0 && h == 0 && e == 0));
          }
        }
        return true;
      };
      // (a wait costs the issuer 100 cycles or more even when it is over, and the issuer's way from P to the
      // next S is on every unit's path)
      if constexpr (ROWT == 1) {
        // S three tiles ahead; PV of a tile, then S into the buffer that it leaves.  K's and V's slots go back by
        // commits of their own
        auto next_s = [&](int sb, int t) {
          tc_fence_after();
          mma_s(sb, t);
          if (C::k_again(t, nt)) mma_commit(&empty[C::k_slot(t)]);
        };
        for (int t = 0; t < min(nt, C::NSB) && ok; ++t) {
          ok = wait_k(t);
          if (ok) next_s(t, t);
        }
        int sb = 0, phase = 0;
        for (int t = 0; t < nt && ok; ++t) {
          const bool more = t + C::NSB < nt;
          uint64_t *fv = &full[C::v_slot(t)], *fk = &full[C::k_slot(t + C::NSB)];
          const uint32_t pv = C::v_turn(t) & 1, pk = C::k_turn(t + C::NSB) & 1;
          const bool v_there = ta_look(fv, pv), k_there = ta_look(fk, pk);
          ok = v_there || ta_wait(fv, pv, p.status, 154);
          ok = ok && mma_o(0, sb, t, phase);
          if (ok) mma_commit(&empty[C::v_slot(t)]);
          if (ok && more) {
            ok = k_there || ta_wait(fk, pk, p.status, 153);
            if (ok) next_s(sb, t + C::NSB);
          }
          if (++sb == C::NSB) {
            sb = 0;
            phase ^= 1;
          }
        }
        if (ok) mma_commit(&o_done[0]);
      } else {
        // the units in turn: PV of a tile, then S of the next.  The waits for K and V come before P's, and once
        // for both units
        const int units = two ? 2 : 1;
        ok = ok && wait_k(0);
        tc_fence_after();
        for (int u = 0; u < units && ok; ++u) mma_s(u, 0);
        for (int t = 0; t < nt && ok; ++t) {
#pragma unroll 1
          for (int u = 0; u < units; ++u) {
            // (fp8: K is still being widened when PV may start)
            if (u == 0) ok = wait_v(t) && (C::F8 || t + 1 >= nt || wait_k(t + 1));
            ok = ok && mma_o(u, u, t, t & 1);
            if (C::F8 && u == 0) ok = ok && (t + 1 >= nt || wait_k(t + 1));
            if (!ok) break;
            if (t + 1 < nt) mma_s(u, t + 1);
            else mma_commit(&o_done[u]);
          }
        }
      }
      // the MMAs in flight end (bounded) before the CTA gives its tensor memory back, also when a unit gave up
      uint64_t* drained = ok ? o_done + (two ? 1 : 0) : o_done + 2;
      if (!ok) {
        mbar_init(drained, 1);
        fence_barrier_init();
        mma_commit(drained);
      }
      ta_wait(drained, 0, nullptr, 0, 50000000ull);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ slots back to the producer (ROWT = 2)
    // S of a tile stands for the unit that is served last (s_full): K of that tile is done with, and V of the
    // tile before, whose PV the issuer put before that S.  (Softmax threads' arrivals cost their warp 350
    // cycles a tile.)  This warp's arrival with that unit's P lets S(t + 1) follow only once S(t) was seen here:
    // the wait is by parity, and two tiles further on it would be for a phase that never comes.  It is there
    // long before P.
    if (ROWT == 2 && elect_one()) {
      const int last = two ? 1 : 0;
      for (int t = 0; t < nt; ++t) {
        if (!ta_wait(&s_full[last], t & 1, p.status, 159)) break;
        mbar_arrive(&p_full[2 * last + 1]);
        if (C::k_again(t, nt)) mbar_arrive(&empty[C::k_slot(t)]);
        if (t > 0 && C::v_again(t - 1, nt)) mbar_arrive(&empty[C::v_slot(t - 1)]);
      }
    }
  } else if (C::F8 && warp >= 12) {
    // ------------------------------------------------------------ fp8 -> f16 (exact), swizzled operand tiles
    if constexpr (C::F8) {
      const int ct = threadIdx.x - 384;
      bool ok = true;
      for (int in = 0; in < 2 * nt && ok; ++in) {
        const int rs = in % C::NR;
        int t;
        const bool isv = C::order(in, nt, t);
        const int slot = isv ? C::v_slot(t) : C::k_slot(t), turn = isv ? C::v_turn(t) : C::k_turn(t);
        ok = ta_wait(&r_full[rs], (in / C::NR) & 1, p.status, 162) &&
             (turn == 0 || ta_wait(&empty[slot], (turn - 1) & 1, p.status, 163));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint4* from = reinterpret_cast<const uint4*>(raw + rs * C::RAW);
        uint8_t* to = sK + C::slot_at(slot);
#pragma unroll
        for (int i = ct; i < C::RAW / 16; i += 128) {
          const uint4 v = from[i];
          uint4 a, c;
          tm_e4m3(v.x, a.x, a.y);
          tm_e4m3(v.y, a.z, a.w);
          tm_e4m3(v.z, c.x, c.y);
          tm_e4m3(v.w, c.z, c.w);
          // K: row = key, 16 of its D values; V: row = column of page i / (DVT * 4), 16 of its 64 keys
          const int row = isv ? (i >> 2) % DVT : i / (D / 16), chunk = isv ? i / (DVT * 4) : i % (D / 16) / 4;
          uint8_t* line = to + chunk * ((isv ? DVT : BN) * 128) + row * 128;
          const int pc = (i & 3) * 2;
          *reinterpret_cast<uint4*>(line + ((pc ^ (row & 7)) << 4)) = a;
          *reinterpret_cast<uint4*>(line + (((pc + 1) ^ (row & 7)) << 4)) = c;
        }
        fence_proxy_async_smem();      // the MMAs read this, and the TMA refills the raw slot
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[slot]);
          mbar_arrive(&r_empty[rs]);
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax units
    const int u = (warp - 4) >> 2, qd = warp & 3;
    const int r = qd * 32 + lane;                      // row of the tile = TMEM lane
    const int rr = r0 + (ROWT == 2 ? u * 128 : 0) + r;
    // (worked out where it is needed: kept through the loop it costs registers that the scores need)
    auto row_here = [&](int x) {
      asm volatile("" : "+r"(x));
      return ta_row(p, q0, n, ctx, x < rows_all ? ta_node(p, x) : 0, x < rows_all);
    };
    {
      // Q, whole rows at a time: D / 8 lanes a row (a thread a row touched 32 lines a load: 5 us).
      // 128B-swizzled K-major chunks of [128 rows][64 columns]
      constexpr int PR = D / 8, TH = ROWT == 2 ? 128 : 128 * C::UNITS;     // pieces of a row, threads of this tile
      uint8_t* dst = sQ + (ROWT == 2 ? u * (128 * D * 2) : 0);
      const int base = r0 + (ROWT == 2 ? u * 128 : 0);
#pragma unroll 4
      for (int i = ROWT == 2 ? r : u * 128 + r; i < 128 * PR; i += TH) {
        const int row = i / PR, pc = i - row * PR, gr = base + row;
        const bool there = gr < rows_all;
        const int nd = there ? ta_node(p, gr) : 0;
        const int hd = there ? gr - nd * p.G : 0;
        uint8_t* at = dst + (pc >> 3) * (128 * 128) + row * 128 + (((pc & 7) ^ (row & 7)) << 4);
        const __nv_bfloat16* from = p.q + (long long)(q0 + nd) * p.q_ts + (long long)(kh * p.G + hd) * p.q_hs + pc * 8;
        if constexpr (C::F8) {   // rounded to f16 (bf16's 8 bits fit its 11; beyond 65504 infinite)
          uint4 v = there ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0u, 0u, 0u, 0u);
          v.x = tm_f16x2(bf16_lo(v.x), bf16_hi(v.x));
          v.y = tm_f16x2(bf16_lo(v.y), bf16_hi(v.y));
          v.z = tm_f16x2(bf16_lo(v.z), bf16_hi(v.z));
          v.w = tm_f16x2(bf16_lo(v.w), bf16_hi(v.w));
          *reinterpret_cast<uint4*>(at) = v;
        } else {
          tt_copy16(smem_u32(at), from, there);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const uint32_t lanes = (uint32_t)(qd * 32) << 16;
    const uint32_t o_t = tmem + lanes + C::O_COL + u % C::NO * DVT;
    float m = -FLT_MAX, l = 0.f;                       // running maximum (log2 units) and sum
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    const int mine = ROWT == 2 ? ((u == 0 || two) ? nt : 0) : (nt - u + C::UNITS - 1) / C::UNITS;   // this unit's tiles
    for (int i = 0; i < mine; ++i) {
      const int t = ROWT == 2 ? i : C::UNITS * i + u;
      const int at = t0 + t;                           // key tile
      const int buf = ROWT == 2 ? u : t % C::NSB, phase = (ROWT == 2 ? t : t / C::NSB) & 1;
      const uint32_t s_t = tmem + lanes + buf * BN;
      const bool msk = at >= shut || at < open;
      // V's non-finite values become zero (0 * p must stay 0 for keys that a row does not see) and join the rows
      // that do see them at the end.  The wait for V(t) is by parity, so the fill of its slot before that has to
      // be known to be over, and V(t) cannot leave before P(t)
      auto clean = [&] {
        ok = ta_wait(&full[C::v_slot(t)], C::v_turn(t) & 1, p.status, 156);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        uint4* vw = reinterpret_cast<uint4*>(sK + C::slot_at(C::v_slot(t)));
#pragma unroll 2
        for (int w = r; w < C::V_BYTES / 16; w += 128) {
          const uint4 x = vw[w];
          const uint4 bad = make_uint4(tt_bad<C::F8>(x.x), tt_bad<C::F8>(x.y), tt_bad<C::F8>(x.z), tt_bad<C::F8>(x.w));
          if (bad.x | bad.y | bad.z | bad.w) {
            s_bad = 1;
            __threadfence_block();                     // the flag before the zeros: the other unit may find only those
            vw[w] = make_uint4(x.x & ~bad.x, x.y & ~bad.y, x.z & ~bad.z, x.w & ~bad.w);
          }
        }
        fence_proxy_async_smem();
      };
      if (!C::SHARE && msk) {   // the unit has seen S(t - 1), which the issuer put after it had K(t - 1) and V(t - 2)
        clean();
        if (!ok) break;
      }
      ok = ta_wait(&s_full[buf], phase, p.status, 157);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (C::SHARE && msk) {
        // S(t) stands, so the product of tile t - 3 is over and V(t - SV)'s release (SV >= 2) is the slot's next one
        // or over; behind it the fill of V(t) is the slot's next one or over
        if (t >= C::SV) {
          ok = ta_wait(&empty[C::v_slot(t)], C::v_turn(t - C::SV) & 1, p.status, 166);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        clean();
        if (!ok) break;
      }
      // HW columns of S in registers at a time: all of them, or with 16 warps' share of the registers (fp8) a half
      constexpr int HW = C::HALVES ? BN / 2 : BN;
      uint32_t sv[HW];
      auto fetch = [&](int c0) {
#pragma unroll
        for (int c = 0; c < HW; c += 32) tmem_ld32p(s_t + c0 + c, sv + c);
        tmem_wait_ld();
        if (!msk) return;
        const TaRow row = row_here(rr);
#pragma unroll
        for (int c = 0; c < HW; c += 32) {
          const uint32_t see = ta_see32(p, row, q0, at * BN + c0 + c);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) sv[c + e] = 0xFF800000u;   // -inf
        }
      };
      float mx4[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += HW) {
        fetch(c0);
#pragma unroll
        for (int e = 0; e < HW; e += 2)
          mx4[(e >> 1) & 3] = fmax3(mx4[(e >> 1) & 3], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
      }
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      if (mx != -FLT_MAX) mx *= p.scale_log2;
      if constexpr (C::SHARE) {
        if (t > 0) {                                   // the maximum that the tile before (the other unit's) left
          const float m_now = ta_row_max(&m_row[r], t - 1, ok);
          if (!ok) report_error(p.status, XTU_ERR_MBAR_TIMEOUT, 164, t);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (m_now != m) {
            if (m != -FLT_MAX) l *= ta_ex2(m - m_now);
            m = m_now;
          }
        }
      }
      // the maximum moves only when it grows by more than 2^8: P stays below 2^8, O is rarely rescaled
      const bool raise = mx > m + 8.f;
      const float m_new = raise ? mx : m;
      const bool rescale = raise && m != -FLT_MAX && (C::SHARE ? t : i) > 0;
      if (__any_sync(0xffffffffu, rescale)) {
        const float f = rescale ? ta_ex2(m - m_new) : 1.f;
        l *= f;
        if constexpr (C::SHARE) {   // PV of the tile before is done once it gave its V slot back
          ok = ta_wait(&empty[C::v_slot(t - 1)], C::v_turn(t - 1) & 1, p.status, 165);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < DVT; c += 16) {
          uint32_t x[16];
          tmem_ld16(o_t + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
          tmem_st16(o_t + c, x);
        }
      }
      m = m_new;
      if constexpr (C::SHARE) {
        ta_row_max_to(&m_row[r], m, t);
      }
      const float neg = m == -FLT_MAX ? 0.f : -m;
      const float2 ng2 = make_float2(neg, neg);
      float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      auto weigh = [&](int c, int col) {               // registers c .. c + 31 into P's columns col ..
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(sv[c + e]), __uint_as_float(sv[c + e + 1])), sc2, ng2);
          const float2 y = make_float2(ta_ex2(x.x), ta_ex2(x.y));
          l2[(e >> 1) & 1] = add2(l2[(e >> 1) & 1], y);
          // P in 16 bits (bf16: half a step of 2^-8, f16: 2^-11); l keeps the 32-bit sum
          pk[e >> 1] = C::F8 ? tm_f16x2(y.x, y.y) : pack_bf16x2(y.x, y.y);
        }
        tmem_st16(s_t + C::P_COL + col, pk);
      };
      auto hand_over = [&](int h) {                    // half of P is ready: its product may start
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * buf + h]);
      };
      if constexpr (C::HALVES) {   // the second half is at hand; P lies over its S, so the first half's still stands
#pragma unroll
        for (int c = 0; c < HW; c += 32) weigh(c, (HW + c) / 2);
        hand_over(0);
        fetch(0);
#pragma unroll
        for (int c = 0; c < HW; c += 32) weigh(c, c / 2);
        hand_over(1);
      } else {
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          weigh(c, c / 2);
          if ((c + 32) % (BN / 2) == 0) hand_over(c / (BN / 2));
        }
      }
      l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
    }
    // ---- end: O / l
    bool have = ok && (C::SHARE ? nt : mine) > 0;
    if (have) {
      have = ta_wait(&o_done[C::SHARE ? 0 : u], 0, p.status, 158);
      have = __all_sync(0xffffffffu, have);
      tc_fence_after();
    }
    const bool valid = rr < rows_all;
    const int node = valid ? ta_node(p, rr) : 0, head = kh * p.G + (valid ? rr - node * p.G : 0), tok = q0 + node;
    float M = m;
    if constexpr (C::SHARE) {
      // one accumulator, each unit's part of the sum in its own last maximum; a unit writes half of the columns
      // (with the products done the ring is free)
      float* ml = reinterpret_cast<float*>(sK);                       // [units][m, l][128]
      asm volatile("bar.sync 1, %0;" ::"n"(128 * C::UNITS) : "memory");
      ml[u * 256 + r] = mine > 0 ? m : -FLT_MAX;
      ml[u * 256 + 128 + r] = mine > 0 ? l : 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(128 * C::UNITS) : "memory");
      for (int w = 0; w < C::UNITS; ++w) M = fmaxf(M, ml[w * 256 + r]);
      l = 0.f;
      for (int w = 0; w < C::UNITS; ++w) {
        const float mw = ml[w * 256 + r], lw = ml[w * 256 + 128 + r];
        l += mw == -FLT_MAX ? (lw != lw ? lw : 0.f) : lw * ta_ex2(mw - M);
      }
    }
    if (C::SHARE ? u < 2 : u == 0 || two) {
      if (p.sinks != nullptr && p.splits == 1 && M != -FLT_MAX && valid) l += ta_ex2(__ldg(p.sinks + head) * LOG2E - M);
      const float inv = l > 0.f || l != l ? p.out_scale / l : 0.f;
      const size_t at = ((size_t)tok * p.Hq + head) * DVT;
      float* wo = p.splits > 1 ? p.ws_o + (size_t)sp * p.T * p.Hq * DVT + at : nullptr;
#pragma unroll 1
      for (int c = C::SHARE ? u * (DVT / 2) : 0; c < (C::SHARE ? (u + 1) * (DVT / 2) : DVT); c += 32) {
        uint32_t x[32];
        if (have) {
          tmem_ld32(o_t + c, x);
          tmem_wait_ld();
        }
        if (!valid) continue;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = have ? __uint_as_float(x[e]) * inv : 0.f;
        if (wo == nullptr) {
          uint4* d4 = reinterpret_cast<uint4*>(p.o + at + c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d4[e] = make_uint4(pack_bf16x2(v[8 * e], v[8 * e + 1]), pack_bf16x2(v[8 * e + 2], v[8 * e + 3]),
                               pack_bf16x2(v[8 * e + 4], v[8 * e + 5]), pack_bf16x2(v[8 * e + 6], v[8 * e + 7]));
        } else {
          float4* d4 = reinterpret_cast<float4*>(wo + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) d4[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
        }
      }
      if (wo != nullptr && valid && (!C::SHARE || u == 0))
        p.ws_lse[((size_t)sp * p.T + tok) * p.Hq + head] =
            l > 0.f || l != l ? (M == -FLT_MAX ? 0.f : M) + __log2f(l) : -FLT_MAX;
      if (s_bad && valid) {   // rare: non-finite values of masked tiles, for the rows that see them
        const TaRow row = row_here(rr);
        for (int pg = t0 * PPT; pg < min(t1 * PPT, npages); ++pg)
          if (pg / PPT >= shut || pg / PPT < open)
            ta_add_bad(p, row, C::F8, q0, b, kh, pg, DVT, C::SHARE ? u * (DVT / 2) : 0,
                       C::SHARE ? (u + 1) * (DVT / 2) : DVT, wo, wo == nullptr ? p.o + at : nullptr);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// ---------------------------------------------------------------------------------------
// the splits' normalised partials by their log-sum-exp: one warp per (token, head).  Rows that the attention kernel
// left out (of no sequence, of one outside the tensors, nodes past max_nodes) have no partials and stay as they are:
// the lanes look through the sequences for the row's own, beside the loads of its values
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) tree_attn_merge_kernel(const float* __restrict__ ws_o,
                                                              const float* __restrict__ ws_lse, int splits,
                                                              int rows, int Hq, int DV, const int* __restrict__ q_start,
                                                              int B, int max_nodes, const float* __restrict__ sinks,
                                                              __nv_bfloat16* __restrict__ o) {
  griddep_wait();
  griddep_launch_dependents();
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (w >= rows) return;
  // the first four splits' values are fetched beside the log-sum-exps that weigh them (an empty split
  // wrote no values: what is read in their place is dropped)
  auto fetch = [&](int s0, int d, float4 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = s0 + k < splits && d < DV ? __ldg(reinterpret_cast<const float4*>(ws_o + ((size_t)(s0 + k) * rows + w) * DV + d))
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float4 v[4];
  fetch(0, lane * 4, v);
  const float sk = sinks != nullptr ? __ldg(sinks + w % Hq) * LOG2E : -FLT_MAX;
  // lane s holds split s (at most 64 splits: two per lane)
  const float a = lane < splits ? __ldg(ws_lse + (size_t)lane * rows + w) : -FLT_MAX;
  const float c = lane + 32 < splits ? __ldg(ws_lse + (size_t)(lane + 32) * rows + w) : -FLT_MAX;
  const int tok = w / Hq, T = rows / Hq;
  bool owned = false;
  for (int b = lane; b < B; b += 32) {
    const int q0 = __ldg(q_start + b), q1 = __ldg(q_start + b + 1);
    owned |= q0 >= 0 && q0 <= tok && tok < q1 && q1 <= T && tok - q0 < max_nodes;
  }
  if (!__any_sync(0xffffffffu, owned)) return;
  float M = fmaxf(a, c);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
  const bool some = __any_sync(0xffffffffu, a != -FLT_MAX || c != -FLT_MAX);   // NaN counts as some
  M = fmaxf(M, sk);
  const float wa = a == -FLT_MAX ? 0.f : ta_ex2(a - M), wc = c == -FLT_MAX ? 0.f : ta_ex2(c - M);
  float sum = wa + wc;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if (sk != -FLT_MAX) sum += ta_ex2(sk - M);
  const float inv = some ? 1.f / sum : 0.f;
  for (int d0 = 0; d0 < DV; d0 += 128) {
    const int d = d0 + lane * 4;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 4) {   // in the order of the splits, four fetched at a time
      if (d0 + s0 > 0) fetch(s0, d, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = s0 + k;
        const float ls = __shfl_sync(0xffffffffu, s < 32 ? a : c, s & 31);
        const float ws = __shfl_sync(0xffffffffu, s < 32 ? wa : wc, s & 31);
        if (s >= splits || ls == -FLT_MAX) continue;
        acc[0] += ws * v[k].x;
        acc[1] += ws * v[k].y;
        acc[2] += ws * v[k].z;
        acc[3] += ws * v[k].w;
      }
    }
    if (d >= DV) continue;
    uint2 pk;
    pk.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    pk.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(o + (size_t)w * DV + d) = pk;
  }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
typedef CUresult (*TaEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

TaEncode ta_encode() {
  static const TaEncode fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<TaEncode>(ptr)
               : nullptr;
  }();
  return fn;
}

// [rows, cols] matrix, boxes of box_rows x box_cols
int ta_map(CUtensorMap* map, CUtensorMapDataType t, int esz, const void* base, uint64_t rows, uint32_t cols,
           uint32_t box_rows, uint32_t box_cols, CUtensorMapSwizzle sw) {
  const TaEncode enc = ta_encode();
  if (!enc) return -100;
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0) return -101;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {(cuuint64_t)cols * esz};
  const cuuint32_t box[2] = {box_cols, box_rows}, es[2] = {1, 1};
  const CUresult r = enc(map, t, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -1000 - (int)r;
}

// the kernel's shared-memory limit, once per device
template <typename K>
int ta_allow(K kern, int bytes, bool (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -102;
  if (done[dev]) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return -(int)e;
  }
  done[dev] = true;
  return 0;
}

template <class C>
int tt_launch(const CUtensorMap& tk, const CUtensorMap& tv, const TaParams& p, int tiles, int B, cudaStream_t s) {
  static bool done[64] = {};
  if (const int rc = ta_allow(tree_attn_tc_kernel<C>, C::BYTES, done)) return rc;
  const cudaError_t e = launch_pdl(tree_attn_tc_kernel<C>, dim3(tiles * p.splits, p.Hkv, B),
                                   dim3(C::THREADS), C::BYTES, s, tk, tv, p);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? 1 : -(int)e;
}

// rows: of the largest tree.  row_tiles = 2: two row tiles a CTA that share their K / V tiles; 1: one, and
// twice the CTAs.  The host weighs them (ops/tree.py, both sides measured there).
template <class ONE, class TWO>
int tt_rows(const CUtensorMap& tk, const CUtensorMap& tv, const TaParams& p, int rows, int row_tiles, int B,
            cudaStream_t s) {
  if (row_tiles == 1) return tt_launch<ONE>(tk, tv, p, (rows + 127) / 128, B, s);
  return tt_launch<TWO>(tk, tv, p, (rows + 255) / 256, B, s);
}

}  // namespace
}  // namespace xtu

using namespace xtu;

extern "C" {

// q [T, Hq, D] (strides q_ts, q_hs), caches [num_blocks, Hkv, 64, D | DV] bf16, or fp8 K
// [num_blocks, Hkv, 64, D] and V [num_blocks, Hkv, DV, 64]; o [T, Hq, DV] bf16.  ws: splits *
// T * Hq * (DV + 2) floats when splits > 1 (<= 64).  q, o, ws and the caches start on 16-byte boundaries.  row_tiles: 128-row tiles of a CTA (1 or 2; heads of 256
// always 1).  Returns the launches, < 0 on error.
struct XtuTreeAttention {
  const void* q;
  long long q_ts;
  int q_hs;
  const void *k_cache, *v_cache;
  int fp8;
  void* o;
  const int *q_start, *kv_len, *block_table;
  int bt_stride, bt_cols;
  const int* mask;
  int W;
  const int* depth;
  int window, B, max_nodes, T, Hq, Hkv, D, DV, num_blocks;
  float scale, k_scale, v_scale;
  const float* sinks;
  int row_tiles, splits;
  float* ws;
  void* status;
  cudaStream_t s;
};

int xtu_tree_attention(const XtuTreeAttention* a) {
  const int B = a->B, T = a->T, Hq = a->Hq, Hkv = a->Hkv, D = a->D, DV = a->DV, splits = a->splits;
  const int row_tiles = a->row_tiles, num_blocks = a->num_blocks;
  const bool fp8 = a->fp8 != 0;
  cudaStream_t s = a->s;
  if (B <= 0 || T <= 0 || a->max_nodes <= 0) return 0;
  if (Hkv <= 0 || Hq % Hkv != 0 || B > 65535 || Hkv > 65535 || a->W <= 0) return -2;
  if (row_tiles < 1 || row_tiles > 2 || splits < 1 || splits > 64 || (splits > 1 && a->ws == nullptr)) return -3;
  if (a->window > 0 && a->depth == nullptr) return -4;
  // 16-byte accesses (the caches: ta_map)
  if (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o) | reinterpret_cast<uintptr_t>(a->ws)) & 15) != 0)
    return -5;
  TaParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_ts = a->q_ts;
  p.q_hs = a->q_hs;
  p.o = static_cast<__nv_bfloat16*>(a->o);
  p.q_start = a->q_start;
  p.kv_len = a->kv_len;
  p.block_table = a->block_table;
  p.bt_stride = a->bt_stride;
  p.bt_cols = a->bt_cols;
  p.mask = a->mask;
  p.W = a->W;
  p.depth = a->depth;
  p.window = a->window > 0 ? a->window : 0;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.T = T;
  p.g_inv = p.G > 1 ? (uint32_t)(((1ull << 32) + p.G - 1) / p.G) : 0u;
  p.scale_log2 = a->scale * LOG2E * (fp8 ? a->k_scale : 1.f);
  p.out_scale = fp8 ? a->v_scale : 1.f;
  p.sinks = a->sinks;
  p.splits = splits;
  p.ws_o = a->ws;
  p.ws_lse = a->ws ? a->ws + (size_t)splits * T * Hq * DV : nullptr;
  p.v_raw = a->v_cache;
  p.num_blocks = num_blocks;
  p.max_nodes = a->max_nodes;
  p.status = static_cast<XtuStatus*>(a->status);
  const void *k_cache = a->k_cache, *v_cache = a->v_cache;
  const uint64_t krows = (uint64_t)num_blocks * Hkv * TA_PAGE;
  CUtensorMap tk, tv;
  int rc;
  if (fp8) {
    rc = ta_map(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k_cache, krows, D, TA_PAGE, D, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc == 0)
      rc = ta_map(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, v_cache, (uint64_t)num_blocks * Hkv * DV, TA_PAGE, DV,
                  TA_PAGE, CU_TENSOR_MAP_SWIZZLE_NONE);
  } else {
    rc = ta_map(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, k_cache, krows, D, TA_PAGE, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == 0)
      rc = ta_map(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, v_cache, krows, DV, TA_PAGE, 64,
                  CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc) return rc;
  const int rows = p.max_nodes * p.G;
  int r = -6;   // head sizes not served
  if (fp8 && D == 64 && DV == 64)
    r = tt_rows<TtCfg<64, 64, 128, 1, 3, 3, 6>, TtCfg<64, 64, 128, 2, 3, 3, 6>>(tk, tv, p, rows, row_tiles, B, s);
  else if (fp8 && D == 128 && DV == 128)
    r = tt_rows<TtCfg<128, 128, 128, 1, 2, 2, 4>, TtCfg<128, 128, 128, 2, 2, 2, 2>>(tk, tv, p, rows, row_tiles, B, s);
  else if (fp8) return -6;
  else if (D == 64 && DV == 64)
    r = tt_rows<TtCfg<64, 64, 128, 1, 6, 6>, TtCfg<64, 64, 128, 2, 5, 5>>(tk, tv, p, rows, row_tiles, B, s);
  else if (D == 128 && DV == 128)
    r = tt_rows<TtCfg<128, 128, 128, 1, 3, 3>, TtCfg<128, 128, 128, 2, 3, 2>>(tk, tv, p, rows, row_tiles, B, s);
  else if (D == 192 && DV == 128)
    r = tt_rows<TtCfg<192, 128, 64, 1, 4, 4>, TtCfg<192, 128, 64, 2, 3, 3>>(tk, tv, p, rows, row_tiles, B, s);
  else if (D == 256 && DV == 256)
    r = tt_launch<TtCfg<256, 256, 64, 1, 3, 2>>(tk, tv, p, (rows + 127) / 128, B, s);
  if (r < 0 || splits == 1) return r;
  const int heads = T * Hq;
  const cudaError_t e = launch_pdl(tree_attn_merge_kernel, dim3((heads + 7) / 8), dim3(256), 0, s,
                                   (const float*)p.ws_o, (const float*)p.ws_lse, splits, heads, Hq, DV, p.q_start, B,
                                   p.max_nodes, p.sinks, p.o);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? r + 1 : -(int)e;
}

}  // extern "C"
