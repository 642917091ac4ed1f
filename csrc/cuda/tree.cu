// Tree speculation outside attention: the ancestor bit rows of a tree of drafted tokens, its
// verification against the target's probabilities, and the move of the accepted path's
// cache rows (tree attention itself is in tree_attention.cu).
//
// A sequence's tree: nodes 0 .. n-1 in rows q_start[b] .. q_start[b+1]-1, node 0 the root (the
// last emitted token), every other node with a parent of lower index.  A parent that is
// negative or not below its node stands for "none".
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <climits>
#include <cstdint>
#include "launch.cuh"
#include "ptx.cuh"

extern "C" struct XtuTreeVerify {
  const void* probs;
  long long ldp;
  const void* draft;
  long long ldq;
  int bf16, V;
  const int *tokens, *parents, *q_start;
  const float *u_accept, *u_draw;
  int B, T, P;
  int *accepted, *path, *out, *last_row;
  void* status;
  cudaStream_t s;
};

namespace xtu {
namespace {

namespace cg = cooperative_groups;

constexpr int TREE_MAX_NODES = 1024;   // nodes of one sequence: the shared arrays below

// rows of sequence b, at most `most` (a longer one is cut and reported), none when they lie outside
// the call's T rows (reported)
__device__ __forceinline__ int tree_nodes(const int* q_start, int b, int T, int most, XtuStatus* st, int site) {
  const int q0 = q_start[b], q1 = q_start[b + 1], n = q1 - q0;
  const bool inside = q0 >= 0 && q0 <= q1 && q1 <= T;
  if (!inside || n > most) report_error(st, XTU_ERR_BOUNDS, site, inside ? n : q1);
  return !inside ? 0 : n > most ? most : n;
}

// ---------------------------------------------------------------------------------------
// ancestor bits: row i gets bit j for j = i and for every ancestor j; depth = ancestors.
// grid (B, node chunks of 128).  A node's ancestors have falling indices, so one walk up the
// parents in shared memory meets the words of the row in falling order and writes each once.
// Latency bound: the walk is `depth` dependent shared-memory reads.
__global__ void __launch_bounds__(128) tree_mask_kernel(const int* __restrict__ parents,
                                                        const int* __restrict__ q_start, int T, int max_nodes, int W,
                                                        int* __restrict__ mask, int* __restrict__ depth,
                                                        XtuStatus* st) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int par[TREE_MAX_NODES];
  const int b = blockIdx.x;
  const int n = tree_nodes(q_start, b, T, max_nodes, st, 248);
  const int q0 = q_start[b];
  const int i0 = blockIdx.y * 128;
  if (i0 >= n) return;
  const int last = min(n, i0 + 128);
  for (int i = threadIdx.x; i < last; i += 128) par[i] = parents[q0 + i];
  __syncthreads();
  const int i = i0 + threadIdx.x;
  if (i >= n) return;
  int* row = mask + (size_t)(q0 + i) * W;
  int w = i >> 5, cur = i, d = 0;
  for (int z = W - 1; z > w; --z) row[z] = 0;
  uint32_t bits = 1u << (i & 31);
  for (;;) {
    const int p = par[cur];
    if (p < 0 || p >= cur) break;
    if ((p >> 5) != w) {
      row[w] = (int)bits;
      for (int z = w - 1; z > (p >> 5); --z) row[z] = 0;
      w = p >> 5;
      bits = 0;
    }
    bits |= 1u << (p & 31);
    cur = p;
    ++d;
  }
  row[w] = (int)bits;
  for (int z = w - 1; z >= 0; --z) row[z] = 0;
  depth[q0 + i] = d;
}

// ---------------------------------------------------------------------------------------
// the first node i >= from whose parent is `cur`, or -1 (whole warp)
__device__ __forceinline__ int next_child(const int* par, int n, int from, int cur) {
  const int lane = threadIdx.x & 31;
  for (int base = from & ~31; base < n; base += 32) {
    const int i = base + lane;
    const unsigned m = __ballot_sync(0xffffffffu, i >= from && i < n && par[i] == cur);
    if (m) return base + __ffs(m) - 1;
  }
  return -1;
}

// greedy acceptance: from the root, the first child (index order) whose token is the target's
// token at the current node, until none is.  One warp per sequence.
__global__ void __launch_bounds__(32) tree_verify_greedy_kernel(
    const int* __restrict__ target, const int* __restrict__ tokens, const int* __restrict__ parents,
    const int* __restrict__ q_start, int T, int P, int* __restrict__ accepted, int* __restrict__ path,
    int* __restrict__ out, int* __restrict__ last_row, XtuStatus* st) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int par[TREE_MAX_NODES], tok[TREE_MAX_NODES], tgt[TREE_MAX_NODES];
  const int b = blockIdx.x, lane = threadIdx.x;
  const int n = tree_nodes(q_start, b, T, P, st, 249);
  const int q0 = q_start[b];
  for (int i = lane; i < n; i += 32) {
    const int p = parents[q0 + i];
    par[i] = (p >= 0 && p < i) ? p : -1;
    tok[i] = tokens[q0 + i];
    tgt[i] = target[q0 + i];
  }
  __syncwarp();
  int* pb = path + (size_t)b * P;
  int* ob = out + (size_t)b * P;
  int cur = 0, a = 0;
  if (n > 0) {
    if (lane == 0) pb[0] = 0;
    for (int from = 1;;) {
      const int c = next_child(par, n, from, cur);
      if (c < 0) break;
      from = c + 1;
      if (tok[c] != tgt[cur]) continue;
      if (lane == 0) {
        ob[a] = tok[c];
        pb[a + 1] = c;
      }
      ++a;
      cur = c;
    }
    if (lane == 0) ob[a] = tgt[cur];
  }
  const int used = n > 0 ? a + 1 : 0;
  for (int i = used + lane; i < P; i += 32) pb[i] = ob[i] = -1;
  if (lane == 0) {
    accepted[b] = a;
    last_row[b] = n > 0 ? q0 + cur : -1;
  }
}

// ---------------------------------------------------------------------------------------
// acceptance by given random numbers.  At node v the weights start as w = p_v (Z = 1); its
// children are tried in index order, child c with token x:
//   point-mass drafts   accepted when u_c (1 - r) < w[x], r the probability of the rejected
//                       siblings' tokens; a rejection sets w[x] = 0
//   drawn from q_v      accepted when u_c q_v[x] Z < w[x]; a rejection sets
//                       w <- max(0, w / Z - q_v), Z <- sum w
// and a node whose children are all rejected emits the smallest t with
// w[0] + .. + w[t] > u_draw * sum w.
//
// Rows of the vocabulary are the traffic (one per sequence, two with q, a pass for every
// rejection of a drawn child), so a cluster of C CTAs shares a sequence's row: each sums a
// slice, and the sums meet in every CTA's shared memory.  The walk runs in all of them on one
// copy of the nodes (rank 0's, read through shared memory once) and on the same sums in the
// same order, so they agree on every step and meet at the same cluster barriers whatever the
// inputs hold or do meanwhile (a walk by rank 0 that told the others took a second barrier a
// pass).  Weights and sums are 64-bit: with 150K terms a 32-bit sum is off by more than many
// tokens' weight, and the drawn token would depend on the split.
// What bounds it is latency.  In cycles: three dependent loads before the walk (the sequence's bounds,
// its nodes, their probabilities) 5500, the first steps 3500; then per pass the load of the slice (the
// first at its node) 3000 to 6000, its weights 1100 with no rejection, 3000 with one and 1100 for each
// further one (64-bit arithmetic), sums and cluster barrier 2000, the walk 1700; the search for the drawn token 4000.
// One sequence, V = 151552: 16 us cold.  32 trees of 26 nodes: 31 to 39 us (by card and inputs) for the 30 MB
// that they read (5 us at the copy rate), in two waves: 18 clusters of 8 fit.
struct TvCmd {
  int op;        // 0 sum the weights, 1 draw, 2 done
  int row;       // row of probs
  int rej;       // rejected children of it so far
  int owner;     // draw: rank that holds the drawn token
  int slot;      // draw: position in the output row
  int any;       // draw: take the last positive weight (the target lies past the sum)
  double target; // draw: target less the slices before the owner's
};

constexpr int TV_THREADS = 512, TV_WARPS = TV_THREADS / 32;
// Weights of a thread in flight (bf16: whole 16-byte loads of them).  Drawn children take a pass for every
// rejection, so the registers hold the slices of p and q from pass to pass: 40 weights each are a vocabulary of
// 163840 over 8 CTAs.  Measured (32 sequences of 26 nodes, V = 151552): 30.7 us; 1024 threads with 20 each 37.3,
// 384 with 56 33.2, 256 with 80 39.8, slices that are read again 33.6.  Drafts chosen outright take one pass.
template <bool DRAFT>
struct TvCfg {
  static constexpr int HELD = DRAFT ? 40 : 16;
};
constexpr int TV_MAX_C = 8;

__device__ __forceinline__ float tv_load1(const float* p) { return __ldg(p); }
__device__ __forceinline__ float tv_load1(const __nv_bfloat16* p) { return __bfloat162float(__ldg(p)); }

// 16 bytes of a row: 4 floats or 8 bf16
__device__ __forceinline__ void tv_loadv(const float* p, float (&v)[4]) {
  const float4 x = __ldg(reinterpret_cast<const float4*>(p));
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void tv_loadv(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
  v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
  v[4] = bf16_lo(x.z); v[5] = bf16_hi(x.z); v[6] = bf16_lo(x.w); v[7] = bf16_hi(x.w);
}

struct TvShared {
  int par[TREE_MAX_NODES];
  int tok[TREE_MAX_NODES];
  float u[TREE_MAX_NODES], pt[TREE_MAX_NODES], qt[TREE_MAX_NODES];
  int rejected[TREE_MAX_NODES];       // tokens of the rejected children of the current node
  double zi[TREE_MAX_NODES];          // zi[r]: 1 / (sum of the weights after r rejections)
  double slice[2][TV_MAX_C];          // the CTAs' sums, of this pass and the one before
  int n, q0;
  double warp_sum[TV_WARPS];
  float u_draw;
  int found, best;                    // the draw: the first weight past the target, the last positive one
  TvCmd cmd;
};

// weights of N elements after `rej` rejections (drawn children), from their p and q.  The elements go
// through a rejection side by side: a loop per element was one chain of dependent 64-bit operations after
// another (12400 cycles a pass at two rejections against 2900 at one).
__device__ __forceinline__ double tv_left(double w) {   // max(w, 0) by its sign bit: 64-bit compares are slow
  const int hi = __double2hiint(w), keep = ~(hi >> 31);
  return __hiloint2double(hi & keep, __double2loint(w) & keep);
}
template <int N>
__device__ __forceinline__ void tv_weights(const float (&p)[N], const float (&q)[N], const double* zi, int rej,
                                           double (&w)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) w[e] = (double)fmaxf(p[e], 0.f);   // NaN and negative entries weigh nothing
  if (rej == 0) return;
  double d[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    d[e] = (double)fmaxf(q[e], 0.f);
    w[e] = tv_left(w[e] - d[e]);
  }
#pragma unroll 1
  for (int r = 1; r < rej; ++r) {
    const double z = zi[r];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = tv_left(w[e] * z - d[e]);
  }
}

// One warp's view of a row: `weights(i, w)` gives the VE weights from element i on (0 past the row).
// 16-byte loads where the rows allow them; where they do not (an odd vocabulary or stride) element
// loads of the same elements by the same lane: the order of the sums does not depend on it.
template <typename E, bool DRAFT>
struct TvRow {
  static constexpr int VE = 16 / sizeof(E);
  const E* p;
  const E* q;          // draft row (DRAFT and rej > 0)
  int hi, vec, rej;
  const double* zi;
  const int* rejected;

  __device__ __forceinline__ void load(int i, float (&x)[VE], float (&y)[VE]) const {
    if (vec && i < hi) {
      tv_loadv(p + i, x);
      if (DRAFT && rej > 0) tv_loadv(q + i, y);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        x[e] = i + e < hi ? tv_load1(p + i + e) : 0.f;
        if (DRAFT && rej > 0) y[e] = i + e < hi ? tv_load1(q + i + e) : 0.f;
      }
    }
  }
  __device__ __forceinline__ void weigh(int i, const float (&x)[VE], const float (&y)[VE], double (&w)[VE]) const {
    if constexpr (DRAFT) {
      tv_weights(x, y, zi, rej, w);
    } else {
      unsigned gone = 0;                     // point mass: rejected tokens among these
      for (int r = 0; r < rej; ++r) {
        const unsigned d = (unsigned)(rejected[r] - i);
        if (d < (unsigned)VE) gone |= 1u << d;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = (gone >> e) & 1u ? 0.0 : (double)fmaxf(x[e], 0.f);
    }
  }
};

__device__ __forceinline__ double tv_warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// inclusive prefix sums over the lanes
__device__ __forceinline__ double tv_warp_scan(double x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  return x;
}

// the first lane whose prefix sum passes t (or -1: none does), the last lane that holds anything (or 0) and
// what is left of t at the former.  (64-bit additions take some 40 cycles one after another: lanes, not a loop.)
__device__ __forceinline__ int tv_find(double x, double sum, double t, int& last, double& at) {
  const unsigned some = __ballot_sync(0xffffffffu, x > 0.0), past = __ballot_sync(0xffffffffu, x > 0.0 && sum > t);
  last = some ? 31 - __clz(some) : 0;
  const double before = __shfl_up_sync(0xffffffffu, sum, 1);
  const int first = past ? __ffs(past) - 1 : -1;
  at = t - __shfl_sync(0xffffffffu, before, first > 0 ? first : 0);
  if (first == 0) at = t;
  return first;
}

template <typename E, bool DRAFT>
__global__ void __launch_bounds__(TV_THREADS) tree_verify_kernel(
    const E* __restrict__ probs, long long ldp, const E* __restrict__ draft, long long ldq, int V, int vec,
    const int* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ q_start,
    const float* __restrict__ u_accept, const float* __restrict__ u_draw, int T, int P, int* __restrict__ accepted,
    int* __restrict__ path, int* __restrict__ out, int* __restrict__ last_row, XtuStatus* st) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ TvShared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.x, rank = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int VE = 16 / sizeof(E);
  // this warp's slice of the vocabulary: whole 32 x VE steps
  const int step = 32 * VE;
  constexpr int TV_BATCH = (TvCfg<DRAFT>::HELD + VE - 1) / VE;   // 16-byte loads of a lane under way at a time
  const int per = (((V + C * TV_WARPS - 1) / (C * TV_WARPS)) + step - 1) / step * step;
  const bool whole = per <= TV_BATCH * step;                     // the slice is one batch: it stays
  float x[TV_BATCH][VE], y[TV_BATCH][VE];
  int held = -1;                                                 // row whose slice x (and y, when held_q) holds
  bool held_q = false;
  const long long first = (long long)(rank * TV_WARPS + warp) * per;
  const int lo = (int)(first < V ? first : V), hi = (int)(first + per < V ? first + per : V);

  int cur = 0, from = 1, a = 0, rej = 0;     // warp 0: the walk, the same in every CTA
  double gone = 0.0;                         // point mass: probability of the rejected tokens
  double z = 1.0;                            // drawn children: sum of the weights at hand
  bool plain = false;                        // nothing was left: draw from p itself
  if (rank == 0) {
    const int nn = tree_nodes(q_start, b, T, P, st, 242), qq = q_start[b];
    if (tid == 0) {
      s.n = nn;
      s.q0 = qq;
    }
    for (int i = tid; i < nn; i += TV_THREADS) {
      const int p = parents[qq + i], t = tokens[qq + i];
      const bool ok = p >= 0 && p < i;
      s.par[i] = ok ? p : -1;
      s.tok[i] = t;
      s.u[i] = u_accept[qq + i];
      const bool in = ok && t >= 0 && t < V;   // a token outside the vocabulary is never accepted
      s.pt[i] = in ? tv_load1(probs + (long long)(qq + p) * ldp + t) : -1.f;
      s.qt[i] = DRAFT && in ? tv_load1(draft + (long long)(qq + p) * ldq + t) : 0.f;
    }
  }
  if (tid == 0) s.u_draw = u_draw[b];
  cl.sync();   // the nodes are there, and so is every CTA whose shared memory the others write to
  if (rank != 0) {
    const TvShared* r0 = cl.map_shared_rank(&s, 0);
    const int nn = r0->n;
    if (tid == 0) {
      s.n = nn;
      s.q0 = r0->q0;
      s.u_draw = r0->u_draw;
    }
    for (int i = tid; i < nn; i += TV_THREADS) {
      s.par[i] = r0->par[i];
      s.tok[i] = r0->tok[i];
      s.u[i] = r0->u[i];
      s.pt[i] = r0->pt[i];
      s.qt[i] = r0->qt[i];
    }
    __syncthreads();
  }
  const int n = s.n, q0 = s.q0;
  if (n == 0) cl.sync();   // (the others have read rank 0's shared memory before it ends)
  int* pb = path + (size_t)b * P;
  int* ob = out + (size_t)b * P;
  for (int pass = 0;; ++pass) {
    if (warp == 0) {
      const bool first = pass == 0;
      bool have_sum = !first;
      TvCmd c{};
      double tot = 0.0, part = 0.0, upto = 0.0;        // the CTAs' sums: all, this lane's, up to this lane's
      if (n == 0) {
        c.op = 2;
      } else {
        if (have_sum) {                       // the sum that was asked for
          part = lane < C ? s.slice[(pass - 1) & 1][lane] : 0.0;
          upto = tv_warp_scan(part);
          tot = __shfl_sync(0xffffffffu, upto, 31);
          z = tot > 0.0 ? tot : 1.0;
        }
        // walk on, unless the sum was that of the final weights (no child left)
        for (;;) {
          const int next = plain ? -1 : next_child(s.par, n, from, cur);
          if (next < 0) break;
          from = next + 1;
          const int x = s.tok[next];
          bool take;
          if (DRAFT) {
            const float p1[1] = {s.pt[next]}, q1[1] = {s.qt[next]};
            double w[1];
            tv_weights(p1, q1, s.zi, rej, w);
            const double q = q1[0] > 0.f ? (double)q1[0] : 0.0;
            take = p1[0] >= 0.f && (double)s.u[next] * q * (rej > 0 ? z : 1.0) < w[0];
          } else {
            bool dup = false;
            for (int r = lane; r < rej; r += 32) dup |= s.rejected[r] == x;
            dup = __any_sync(0xffffffffu, dup);
            take = !dup && s.pt[next] >= 0.f && (double)s.u[next] * (1.0 - gone) < (double)s.pt[next];
            if (!take && !dup && s.pt[next] > 0.f) gone += (double)s.pt[next];
          }
          have_sum = false;
          if (take) {
            if (lane == 0 && rank == 0) {
              ob[a] = x;
              pb[a + 1] = next;
            }
            ++a;
            cur = next;
            rej = 0;
            gone = 0.0;
            continue;
          }
          if (lane == 0) {
            s.rejected[rej] = x;
            if (DRAFT && rej > 0) s.zi[rej] = 1.0 / z;
          }
          ++rej;
          __syncwarp();
          if (DRAFT) break;                   // the next test (or the draw) needs the new sum
        }
        c.row = q0 + cur;
        c.rej = plain ? 0 : rej;
        if (have_sum && !(tot > 0.0) && !plain) {   // nothing left of p: the draw is from p itself
          plain = true;
          have_sum = false;
          c.rej = 0;
        }
        if (have_sum) {                       // the sum of the final weights is known: draw
          int last;
          double at;
          const int owner = tv_find(part, upto, (double)s.u_draw * tot, last, at);
          c.op = 1;
          c.any = owner < 0;
          c.owner = owner < 0 ? last : owner;
          c.target = at;
          c.slot = a;
        }
      }
      if (lane == 0) s.cmd = c;
    }
    __syncthreads();
    const TvCmd c = s.cmd;
    if (c.op == 2) break;
    TvRow<E, DRAFT> row;
    row.p = probs + (long long)c.row * ldp;
    row.q = DRAFT ? draft + (long long)c.row * ldq : nullptr;
    row.hi = hi;
    row.vec = vec;
    row.rej = c.rej;
    row.zi = s.zi;
    row.rejected = s.rejected;
    if (c.op == 0) {
      double sum = 0.0;
      for (int base = lo; base < hi; base += TV_BATCH * step) {
        if (held != c.row || (DRAFT && c.rej > 0 && !held_q)) {
#pragma unroll
          for (int k = 0; k < TV_BATCH; ++k)
            if (base + k * step < hi) row.load(base + k * step + lane * VE, x[k], y[k]);
        }
#pragma unroll
        for (int k = 0; k < TV_BATCH; ++k) {
          if (base + k * step >= hi) break;            // (the whole warp)
          double w[VE];
          row.weigh(base + k * step + lane * VE, x[k], y[k], w);
#pragma unroll
          for (int e = 0; e < VE; ++e) sum += w[e];
        }
      }
      if (whole) {
        held_q = c.rej > 0 || (held == c.row && held_q);
        held = c.row;
      }
      sum = tv_warp_sum(sum);
      if (lane == 0) s.warp_sum[warp] = sum;
      __syncthreads();
      if (warp == 0) {
        const double tot = tv_warp_sum(lane < TV_WARPS ? s.warp_sum[lane] : 0.0);
        if (lane < C) cl.map_shared_rank(&s, lane)->slice[pass & 1][rank] = tot;
      }
      cl.sync();
      continue;
    }
    if (rank == c.owner) {
      // the warp whose slice holds the target (warp_sum is of these weights), then the element
      int last;
      double at;
      const double ws = lane < TV_WARPS ? s.warp_sum[lane] : 0.0;
      const int mine = tv_find(ws, tv_warp_scan(ws), c.target, last, at);
      // that slice again, VE neighbouring weights a thread and a turn of the block (one load latency
      // instead of one warp's chain of them): prefix sums over the lanes, then over the warps
      const bool any = c.any || mine < 0;
      const int wsel = any ? last : mine;
      const long long sf = (long long)(rank * TV_WARPS + wsel) * per;
      const int slo = (int)(sf < V ? sf : V), shi = (int)(sf + per < V ? sf + per : V);
      row.hi = shi;
      double run = 0.0;
      for (int base = slo; base < shi; base += TV_THREADS * VE) {
        float x1[VE], y1[VE];
        double w[VE], own = 0.0;
        const int i = base + tid * VE;
        row.load(i, x1, y1);
        row.weigh(i, x1, y1, w);
        int last_pos = -1;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          own += w[e];
          if (w[e] > 0.0) last_pos = i + e;
        }
        const double cum = tv_warp_scan(own);            // lanes up to this one
        __syncthreads();                                 // (warp_sum was read above, or in the turn before)
        if (lane == 31) s.warp_sum[warp] = cum;
        if (tid == 0) s.found = INT_MAX;
        if (tid == 0 && base == slo) s.best = 0;
        __syncthreads();
        const double sums = tv_warp_scan(lane < TV_WARPS ? s.warp_sum[lane] : 0.0);
        double c2 = run + (warp > 0 ? __shfl_sync(0xffffffffu, sums, warp - 1) : 0.0) + (cum - own);
        run += __shfl_sync(0xffffffffu, sums, 31);
        int first_pos = INT_MAX;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          c2 += w[e];
          if (first_pos == INT_MAX && w[e] > 0.0 && c2 > at) first_pos = i + e;
        }
        if (!any && first_pos != INT_MAX) atomicMin(&s.found, first_pos);
        if (last_pos >= 0) atomicMax(&s.best, last_pos);
        __syncthreads();
        if (s.found != INT_MAX) break;
      }
      if (tid == 0) ob[c.slot] = slo < shi ? (s.found != INT_MAX ? s.found : s.best) : 0;
    }
    break;
  }
  if (rank == 0 && warp == 0) {
    const int used = n > 0 ? a + 1 : 0;
    if (lane == 0) {
      if (n > 0) pb[0] = 0;
      accepted[b] = a;
      last_row[b] = n > 0 ? q0 + cur : -1;
    }
    for (int i = used + lane; i < P; i += 32) pb[i] = ob[i] = -1;
  }
}

// ---------------------------------------------------------------------------------------
// the accepted path's rows behind the committed context: slot ctx + path[j] -> ctx + j
// (j = 1 .. accepted) in every layer.  A path rises (path[j] >= j), so no later source lies at
// an earlier destination: moves in the order of j, reading ahead of writing.
//
// Grid (sequence, layer, part).  Rows that lie whole in a page (K, bf16 V): a thread owns 16
// bytes of the row.  fp8 V lies transposed in its page, [column][64 keys]: parts 1 .. take 256
// columns each; the two pages around the tree come in whole (16-byte pieces, 128 bytes a
// column), a thread permutes its column in shared memory, and the pieces that a destination
// lies in go back: byte moves in global memory fetched the same sectors one dependent
// byte at a time (61 us for 46 layers x 16 sequences of 61 nodes).  A tree that reaches over a
// third page, or whose first page is not there, moves bytes.
constexpr int TC_LAYERS = 64;   // layers of one launch (their pointers travel as parameters)
constexpr int TC_MOVES = 256;   // moves of one turn
constexpr int TC_LD = 132;      // a column's two pages in shared memory (33 words: no bank conflicts)
struct TcLayers {
  void* k[TC_LAYERS];
  void* v[TC_LAYERS];
};

__global__ void __launch_bounds__(256) tree_commit_kernel(const __grid_constant__ TcLayers layers,
                                                          const int* __restrict__ path, int P,
                                                          const int* __restrict__ accepted,
                                                          const int* __restrict__ q_start,
                                                          const int* __restrict__ kv_len,
                                                          const int* __restrict__ bt, int bt_stride, int bt_cols,
                                                          int num_blocks, int Hkv, int kb, int vb, int fp8_v, int Dv) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int src[TC_MOVES], dst[TC_MOVES];   // flat cache rows (page * 64 + offset), -1: nothing to move
  __shared__ __align__(16) uint8_t cols[256 * TC_LD];
  __shared__ int reach;                          // the furthest source
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = q_start[b + 1] - q_start[b];
  const int ctx = kv_len[b] - n;
  const int acc = min(min(accepted[b], P - 1), n - 1);
  if (ctx < 0 || acc < 1) return;
  uint8_t* kc = static_cast<uint8_t*>(layers.k[blockIdx.y]);
  uint8_t* vc = static_cast<uint8_t*>(layers.v[blockIdx.y]);
  const int kch = kb >> 4, vch = vb >> 4;        // 16-byte pieces of one head's K and V row
  const int pg0 = (ctx + 1) >> 6;                // the two pages (fp8 V)
  const int part = blockIdx.z;
  for (int j0 = 1; j0 <= acc; j0 += TC_MOVES) {
    __syncthreads();
    if (tid == 0) reach = 0;
    __syncthreads();
    const int j = j0 + tid;
    int f = -1, t = -1;
    if (j <= acc) {
      const int node = path[(size_t)b * P + j];
      if (node > j && node < n) {                // node == j: already in place
        const int fs = ctx + node, ts = ctx + j;
        if ((fs >> 6) < bt_cols) {
          const int fp = bt[(size_t)b * bt_stride + (fs >> 6)], tp = bt[(size_t)b * bt_stride + (ts >> 6)];
          if (fp >= 0 && fp < num_blocks && tp >= 0 && tp < num_blocks) {
            f = fp * 64 + (fs & 63);
            t = tp * 64 + (ts & 63);
            if (part > 0) atomicMax(&reach, fs);
          }
        }
      }
    }
    src[tid] = f;
    dst[tid] = t;
    __syncthreads();
    const int cnt = min(TC_MOVES, acc - j0 + 1);
    if (part == 0) {
      const int kw = Hkv * kch, all = kw + (fp8_v ? 0 : Hkv * vch);
      for (int c = tid; c < all; c += 256) {
        uint8_t* base = c < kw ? kc : vc;
        const int ch = c < kw ? kch : vch, cc = c < kw ? c : c - kw;
        const int h = cc / ch, o = cc - h * ch;
        const size_t rb = (size_t)ch << 4;
        auto at = [&](int row) {
          return reinterpret_cast<uint4*>(base + (((size_t)(row >> 6) * Hkv + h) * 64 + (row & 63)) * rb) + o;
        };
        for (int i = 0; i < cnt; i += 4) {
          uint4 x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i + u < cnt && src[i + u] >= 0) x[u] = *at(src[i + u]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i + u < cnt && src[i + u] >= 0) *at(dst[i + u]) = x[u];
        }
      }
      continue;
    }
    const int c0 = (part - 1) * 256, nc = min(256, Hkv * Dv - c0);
    const size_t page_b = (size_t)Hkv * Dv * 64;
    if (reach == 0) continue;
    int pages[2];
    for (int g = 0; g < 2; ++g) pages[g] = pg0 + g < bt_cols ? bt[(size_t)b * bt_stride + pg0 + g] : -1;
    // a tree over a third page, or without the first (moves inside the second are left then)
    if ((reach >> 6) > pg0 + 1 || pages[0] < 0 || pages[0] >= num_blocks) {
      for (int i = 0; tid < nc && i < cnt; ++i) {
        const int f1 = src[i], t1 = dst[i];
        if (f1 < 0) continue;
        uint8_t* col = vc + (size_t)(c0 + tid) * 64;
        col[(t1 >> 6) * page_b + (t1 & 63)] = col[(f1 >> 6) * page_b + (f1 & 63)];
      }
      continue;
    }
    const bool second = (reach >> 6) > pg0;                               // (its id was checked with the move)
    const int pieces = second ? 8 : 4;
    for (int i = tid; i < nc * pieces; i += 256) {
      const int c = i / pieces, o = i - c * pieces;
      const uint4 x = *reinterpret_cast<const uint4*>(vc + pages[o >> 2] * page_b + (size_t)(c0 + c) * 64 + (o & 3) * 16);
      uint32_t* d = reinterpret_cast<uint32_t*>(cols + c * TC_LD + o * 16);
      d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
    }
    __syncthreads();
    if (tid < nc) {
      uint8_t* col = cols + tid * TC_LD;
      for (int i = 0; i < cnt; ++i) {
        const int f1 = src[i], t1 = dst[i];
        if (f1 < 0) continue;
        // (the same page twice in a table would be the caller's own two names of one slot)
        const int fo = ((f1 >> 6) == pages[0] ? 0 : 64) + (f1 & 63), to = ((t1 >> 6) == pages[0] ? 0 : 64) + (t1 & 63);
        col[to] = col[fo];
      }
    }
    __syncthreads();
    const int a0 = (ctx + j0) - pg0 * 64, a1 = (ctx + j0 + cnt - 1) - pg0 * 64;   // destinations
    for (int i = tid; i < nc * pieces; i += 256) {
      const int c = i / pieces, o = i - c * pieces;
      if (o * 16 > a1 || o * 16 + 15 < a0) continue;
      const uint32_t* d = reinterpret_cast<const uint32_t*>(cols + c * TC_LD + o * 16);
      *reinterpret_cast<uint4*>(vc + pages[o >> 2] * page_b + (size_t)(c0 + c) * 64 + (o & 3) * 16) =
          make_uint4(d[0], d[1], d[2], d[3]);
    }
  }
}

template <typename E, bool DRAFT>
int tv_launch(const XtuTreeVerify& a) {
  // CTAs per sequence: a slice of at least 4096 elements each.  18 clusters of 8 run at a time; for more
  // sequences 4 CTAs a cluster where their registers hold the slice (drawn children, 32 / 64 sequences: V =
  // 33000 34.8 / 57.3 -> 24.6 / 41.0 us, 65536 34.8 / 53.2 -> 28.7 / 41.0; 16: 26.6 -> 28.7)
  const bool many = DRAFT && a.B > 18 && a.V <= 4 * TV_THREADS * TvCfg<DRAFT>::HELD;
  const int C = a.V <= 4096 ? 1 : a.V <= 8192 ? 2 : a.V <= 16384 || many ? 4 : 8;
  constexpr int VE = 16 / sizeof(E);
  const bool vec = a.V % VE == 0 && a.ldp % VE == 0 && (reinterpret_cast<uintptr_t>(a.probs) & 15) == 0 &&
                   (!DRAFT || (a.ldq % VE == 0 && (reinterpret_cast<uintptr_t>(a.draft) & 15) == 0));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, a.B);
  cfg.blockDim = dim3(TV_THREADS);
  cfg.stream = a.s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, tree_verify_kernel<E, DRAFT>, static_cast<const E*>(a.probs), a.ldp,
                         static_cast<const E*>(a.draft), a.ldq, a.V, (int)vec, a.tokens, a.parents, a.q_start,
                         a.u_accept, a.u_draw, a.T, a.P, a.accepted, a.path, a.out, a.last_row,
                         static_cast<XtuStatus*>(a.status));
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return -(int)e;
  }
  return 1;
}

}  // namespace
}  // namespace xtu

using namespace xtu;

extern "C" {

// Each entry takes its arguments as one struct (the binding packs them: ops/_native.py).

struct XtuTreeMask {
  const int *parents, *q_start;
  int B, T, max_nodes, W;
  int *mask, *depth;
  void* status;
  cudaStream_t s;
};

// parents [T] -> mask [T, W] (W words of 32 nodes) and depth [T]; max_nodes <= 1024, W >= ceil(max_nodes / 32)
int xtu_tree_mask(const XtuTreeMask* a) {
  if (a->B <= 0 || a->max_nodes <= 0) return 0;
  if (a->max_nodes > TREE_MAX_NODES || a->W * 32 < a->max_nodes) return -2;
  const cudaError_t e = launch_pdl(tree_mask_kernel, dim3(a->B, (a->max_nodes + 127) / 128), dim3(128), 0, a->s,
                                   a->parents, a->q_start, a->T, a->max_nodes, a->W, a->mask, a->depth,
                                   static_cast<XtuStatus*>(a->status));
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? 1 : -(int)e;
}

struct XtuTreeVerifyGreedy {
  const int *target, *tokens, *parents, *q_start;
  int B, T, P;
  int *accepted, *path, *out, *last_row;
  void* status;
  cudaStream_t s;
};

// accepted [B], path [B, P], out [B, P], last_row [B]; P = the largest tree
int xtu_tree_verify_greedy(const XtuTreeVerifyGreedy* a) {
  if (a->B <= 0 || a->P <= 0) return 0;
  if (a->P > TREE_MAX_NODES) return -2;
  const cudaError_t e = launch_pdl(tree_verify_greedy_kernel, dim3(a->B), dim3(32), 0, a->s, a->target, a->tokens,
                                   a->parents, a->q_start, a->T, a->P, a->accepted, a->path, a->out, a->last_row,
                                   static_cast<XtuStatus*>(a->status));
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? 1 : -(int)e;
}

// probs [T, V] (row stride ldp elements), draft the same or null; bf16: both bf16, else fp32
int xtu_tree_verify(const XtuTreeVerify* a) {
  if (a->B <= 0 || a->P <= 0) return 0;
  if (a->P > TREE_MAX_NODES || a->V <= 0 || a->B > 65535) return -2;
  if (a->bf16) return a->draft ? tv_launch<__nv_bfloat16, true>(*a) : tv_launch<__nv_bfloat16, false>(*a);
  return a->draft ? tv_launch<float, true>(*a) : tv_launch<float, false>(*a);
}

// k_ptrs / v_ptrs: host arrays of L cache addresses, or null: layer l at k_base + l * k_step
// bytes.  kb / vb: bytes of one head's K / V row (vb 16-byte pieces; fp8_v: V is [Dv][64]
// inside a block and vb is unused).
struct XtuTreeCommit {
  const long long *k_ptrs, *v_ptrs;
  long long k_base, k_step, v_base, v_step;
  int L;
  const int* path;
  int P;
  const int *accepted, *q_start, *kv_len, *bt;
  int bt_stride, bt_cols, B, num_blocks, Hkv, kb, vb, fp8_v, Dv;
  cudaStream_t s;
};

int xtu_tree_commit(const XtuTreeCommit* a) {
  if (a->B <= 0 || a->L <= 0 || a->P <= 1) return 0;
  if (a->kb % 16 != 0 || (!a->fp8_v && a->vb % 16 != 0)) return -2;
  const int parts = a->fp8_v ? 1 + (a->Hkv * a->Dv + 255) / 256 : 1;
  int launches = 0;
  for (int l0 = 0; l0 < a->L; l0 += TC_LAYERS) {
    const int m = a->L - l0 < TC_LAYERS ? a->L - l0 : TC_LAYERS;
    TcLayers t{};
    for (int l = 0; l < m; ++l) {
      t.k[l] = reinterpret_cast<void*>(a->k_ptrs ? a->k_ptrs[l0 + l] : a->k_base + (l0 + l) * a->k_step);
      t.v[l] = reinterpret_cast<void*>(a->v_ptrs ? a->v_ptrs[l0 + l] : a->v_base + (l0 + l) * a->v_step);
    }
    const cudaError_t e = launch_pdl(tree_commit_kernel, dim3(a->B, m, parts), dim3(256), 0, a->s, t, a->path, a->P,
                                     a->accepted, a->q_start, a->kv_len, a->bt, a->bt_stride, a->bt_cols,
                                     a->num_blocks, a->Hkv, a->kb, a->vb, a->fp8_v, a->Dv);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return -(int)e;
    }
    ++launches;
  }
  return launches;
}

}  // extern "C"
