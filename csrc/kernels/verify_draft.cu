// Verification of drafted tokens against the target's probabilities, from given uniform numbers (sm_100a).
//
// Node 0 is the last confirmed token, nodes 1 .. n-1 are drafted; probs[b, i] is the target's distribution after node i.
//   chain with the draft's distributions q: node i + 1 is accepted while u_i q_i(x) < p_i(x). After the first refusal the next token
//     is drawn from max(p - q, 0), after the last node from p
//   fixed candidates, a chain or a tree: the children of a node share its number u; in index order each takes an interval of length
//     p(x) behind the one before, and the child whose interval holds u is accepted (a token that comes twice has its mass
//     once). Where none does, the next token is drawn from p without the children's tokens
// Either way the token that follows and the accepted ones are distributed as if they had been drawn from p one by one.
//
// The walk needs only p (and q) at the drafted tokens: T scalars, loaded at once. What is bound by memory is the row (or two) that
// the next token is drawn from, by inversion: a cluster of eight CTAs shares a sequence's row, a warp sums one segment and stores the
// sum into the shared memory of all eight, and the CTA whose segment holds u * total goes through that once more (out of L2).
// All sums are in 64 bits: a token next to a border of the cumulative sum is then the same whatever the order of adding.
// Measured: 64 chains of 5 drafted tokens, 128 000 in the vocabulary, fp32, two rows of 512 KB each, 66 MB: 18 us, 3.7 TB/s, the walk in
// front of the rows and the second look at the segment included; one tree of 26 nodes over 50 257: 10 us, of which the row takes a
// fraction: three loads that depend on one another, two barriers of the cluster.
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"
#include "decode_calls.h"
#include "host_util.h"

namespace tb {

namespace cg = cooperative_groups;

constexpr int VD_CLUSTER = 8;
constexpr int VD_MAX_NODES = 1024;
constexpr int VD_MAX_CHUNKS = 64;
constexpr int VD_UNROLL = 8;

struct VerifyArgs {
  const void *probs, *draft;        // [B, T, V], [B, T - 1, V] or null
  long pb, pt, db, dt;              // strides in elements
  const long* tokens;               // [B, T]
  const long* parents;              // [B or 1, T]; null: a chain
  long parents_ld;
  const float* uniforms;            // [B, T]
  const int* counts;                // [B] or null
  long *accepted, *path, *next;     // [B], [B, T], [B]
  int B, T, V;
};

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan_d(double v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
__device__ __forceinline__ double mass_of(float p, float q) {
  const double r = (double)p - (double)q;
  return r > 0.0 ? r : 0.0;   // negative and NaN: none
}

// The mass of columns [c, c + 32 * n) that a warp's lanes hold, in order: lane l has c + l, c + 32 + l, ...
struct Row {
  const void *p, *q;          // q null: nothing is taken off
  const uint32_t* out;        // bit per column from `base` on that is left out; null: none
  int base;
};
template <typename T>
__device__ __forceinline__ double mass_at(const Row& r, int c, int end) {
  if (c >= end) return 0.0;
  const float p = to_f<T>(((const T*)r.p)[c]);
  const float q = r.q ? to_f<T>(((const T*)r.q)[c]) : 0.f;
  const bool gone = r.out && ((r.out[(c - r.base) >> 5] >> ((c - r.base) & 31)) & 1u);
  return gone ? 0.0 : mass_of(p, q);
}
template <typename T>
__device__ __forceinline__ double sum_range(const Row& r, int c0, int end, int lane) {
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  for (int c = c0 + lane; c < end; c += 32 * VD_UNROLL) {
    float p[VD_UNROLL], q[VD_UNROLL];
#pragma unroll
    for (int i = 0; i < VD_UNROLL; ++i) p[i] = c + 32 * i < end ? to_f<T>(((const T*)r.p)[c + 32 * i]) : 0.f;
    if (r.q) {
#pragma unroll
      for (int i = 0; i < VD_UNROLL; ++i) q[i] = c + 32 * i < end ? to_f<T>(((const T*)r.q)[c + 32 * i]) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < VD_UNROLL; ++i) q[i] = 0.f;
    }
    if (r.out) {
#pragma unroll
      for (int i = 0; i < VD_UNROLL; ++i) {
        const int at = c + 32 * i - r.base;
        if (c + 32 * i < end && ((r.out[at >> 5] >> (at & 31)) & 1u)) p[i] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < VD_UNROLL; ++i) part[i & 3] += mass_of(p[i], q[i]);
  }
  return warp_sum_d((part[0] + part[1]) + (part[2] + part[3]));
}

// Of the masses of 32 N consecutive ranges (lane l of a warp holds m[0 .. N-1] of ranges N l ..): the range in which the running sum,
// `before` at the first, passes `target` (rounding can leave none: then the last that has any mass; -1: no mass at all), and the sum
// before it.
template <int N>
__device__ __forceinline__ void pick_range(const double (&m)[N], double target, int lane, int& hit, double& before) {
  double own = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) own += m[i];
  const double incl = warp_scan_d(own, lane);
  double at = __shfl_up_sync(0xffffffffu, incl, 1);
  at = before + (lane ? at : 0.0);
  int last = -1, over = -1;
  double b_last = 0.0, b_over = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double next = at + m[i];
    if (m[i] > 0.0) {
      last = N * lane + i;
      b_last = at;
      if (over < 0 && next > target) {
        over = last;
        b_over = at;
      }
    }
    at = next;
  }
  const unsigned some = __ballot_sync(0xffffffffu, last >= 0), past = __ballot_sync(0xffffffffu, over >= 0);
  const int src = past ? __ffs(past) - 1 : some ? 31 - __clz(some) : 0;
  hit = __shfl_sync(0xffffffffu, past ? over : last, src);
  before = __shfl_sync(0xffffffffu, past ? b_over : b_last, src);
}

template <typename T, int VD_WARPS>
__global__ void __cluster_dims__(VD_CLUSTER, 1, 1) __launch_bounds__(VD_WARPS * 32, VD_WARPS <= 8 ? 4 : 1) verify_kernel(const VerifyArgs a, int words) {
  constexpr int VD_THREADS = VD_WARPS * 32, VD_SEGMENTS = VD_CLUSTER * VD_WARPS, PER_LANE = VD_SEGMENTS / 32;
  extern __shared__ uint32_t out_bits[];                 // this CTA's columns
  __shared__ float mass[VD_MAX_NODES], dmass[VD_MAX_NODES];
  __shared__ int parent[VD_MAX_NODES], token[VD_MAX_NODES];
  __shared__ float num[VD_MAX_NODES];
  __shared__ double seg[2][VD_SEGMENTS];
  __shared__ int s_last, s_kids;
  cg::cluster_group cluster = cg::this_cluster();
  auto started = cluster.barrier_arrive();               // waited for before the first store into another CTA
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / VD_CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = min(max(a.counts ? a.counts[b] : a.T, 1), a.T);
  const T* probs = (const T*)a.probs + b * a.pb;
  const T* draft = a.draft ? (const T*)a.draft + b * a.db : nullptr;
  const long* par = a.parents ? a.parents + b * a.parents_ld : nullptr;
  const float* u = a.uniforms + (long)b * a.T;
  const float last_u = u[a.T - 1];

  for (int i = tid; i < a.T; i += VD_THREADS) {          // not up to n: its load is under way, too
    const long tk = a.tokens[(long)b * a.T + i];
    const long pr = par ? par[i] : i - 1;
    const float un = u[i];
    const bool ok = i > 0 && i < n && tk >= 0 && tk < a.V && pr >= 0 && pr < i;   // anything else is never accepted
    if (i > 0 && i < n && !ok) report_bad_index();
    parent[i] = ok ? (int)pr : -1;
    token[i] = ok ? (int)tk : -1;
    mass[i] = ok ? to_f<T>(probs[pr * a.pt + tk]) : 0.f;
    num[i] = un;
    dmass[i] = ok && draft ? to_f<T>(draft[pr * a.dt + tk]) : 0.f;
  }
  for (int i = tid; i < words; i += VD_THREADS) out_bits[i] = 0;
  __syncthreads();
  if (!draft && par) {   // a token that is drafted twice under one parent
    for (int i = tid; i < n; i += VD_THREADS) {
      bool twice = false;
      for (int j = 1; j < i; ++j) twice |= parent[j] == parent[i] && token[j] == token[i];
      if (twice) dmass[i] = 1.f;   // unused otherwise without a draft distribution: marks the mass as taken
    }
    __syncthreads();
  }
  if (warp == 0) {
    int cur = 0, took = 0;
    bool kids = false;
    long* path = rank == 0 ? a.path + (long)b * a.T : nullptr;
    if (path && lane == 0) path[0] = 0;
    while (true) {
      int step = -1;
      kids = false;
      if (draft) {
        if (cur + 1 < n) {
          kids = true;
          if (parent[cur + 1] == cur && (double)num[cur] * (double)dmass[cur + 1] < (double)mass[cur + 1]) step = cur + 1;
        }
      } else {
        double low = 0.0;
        const double x = (double)num[cur];
        for (int j0 = cur + 1; j0 < n; j0 += 32) {
          const int j = j0 + lane;
          unsigned hit = __ballot_sync(0xffffffffu, j < n && parent[j] == cur);
          kids |= hit != 0;
          while (hit) {
            const int c = j0 + __ffs(hit) - 1;
            hit &= hit - 1;
            const double m = dmass[c] != 0.f ? 0.0 : mass_of(mass[c], 0.f);
            if (step < 0 && low <= x && x < low + m) step = c;
            low += m;
          }
          if (!par) break;   // a chain: the child is the next node
        }
      }
      if (step < 0) break;
      cur = step;
      ++took;
      if (path && lane == 0) path[took] = cur;
    }
    if (path)
      for (int i = took + 1 + lane; i < a.T; i += 32) path[i] = -1;
    if (lane == 0) {
      s_last = cur;
      s_kids = kids;
      if (rank == 0) a.accepted[b] = took;
    }
  }
  __syncthreads();

  // segments: multiples of 32 columns, so that a segment's words of the bit map are its own
  const int last = s_last;
  const int len = (((a.V + VD_SEGMENTS - 1) / VD_SEGMENTS) + 31) & ~31;
  const int base = rank * VD_WARPS * len;                // may lie behind the last column
  Row row{probs + last * a.pt, draft && s_kids ? draft + last * a.dt : nullptr, nullptr, base};
  if (!draft && s_kids) {
    for (int i = tid + 1; i < n; i += VD_THREADS)
      if (parent[i] == last && token[i] >= base && token[i] < base + VD_WARPS * len)
        atomicOr(&out_bits[(token[i] - base) >> 5], 1u << ((token[i] - base) & 31));
    row.out = out_bits;
    __syncthreads();
  }
  double target = 0.0, at = 0.0;
  int hit = -1;
  for (int pass = 0; pass < 2; ++pass) {
    const int c0 = min(base + warp * len, a.V), c1 = min(c0 + len, a.V);
    const double s = sum_range<T>(row, c0, c1, lane);
    if (!pass) cluster.barrier_wait(std::move(started));
    // each pass has sums of its own: nobody's are written again while they are read
    if (lane < VD_CLUSTER) cluster.map_shared_rank(seg[pass], lane)[rank * VD_WARPS + warp] = s;
    cluster.sync();
    double m[PER_LANE], own = 0.0;                       // every warp does the same with the same numbers
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) own += m[i] = seg[pass][PER_LANE * lane + i];
    at = 0.0;
    target = (double)last_u * warp_sum_d(own);
    pick_range<PER_LANE>(m, target, lane, hit, at);
    if (hit >= 0) break;
    row.q = nullptr;                                     // the draft covers all of p: draw from p itself
    row.out = nullptr;
  }
  if (hit < 0) {
    if (rank == 0 && tid == 0) a.next[b] = -1;
    return;
  }
  if (hit / VD_WARPS != rank) return;
  // the segment in chunks of 256 columns: the warps sum them, then one takes the chunk, eight neighbouring columns to a lane
  __shared__ double chunk[VD_MAX_CHUNKS];
  const int c0 = hit * len, c1 = min(c0 + len, a.V), wide = max(256, ((len / 32 + VD_MAX_CHUNKS - 1) / VD_MAX_CHUNKS) * 32);
  const int chunks = (c1 - c0 + wide - 1) / wide;
  if (chunks > 1) {
    for (int k = warp; k < VD_MAX_CHUNKS; k += VD_WARPS) {
      const double s = k < chunks ? sum_range<T>(row, c0 + k * wide, min(c0 + (k + 1) * wide, c1), lane) : 0.0;
      if (lane == 0) chunk[k] = s;
    }
    __syncthreads();
  }
  if (warp) return;
  hit = 0;
  if (chunks > 1) {
    double m[VD_MAX_CHUNKS / 32];
#pragma unroll
    for (int i = 0; i < VD_MAX_CHUNKS / 32; ++i) m[i] = chunk[VD_MAX_CHUNKS / 32 * lane + i];
    pick_range<VD_MAX_CHUNKS / 32>(m, target, lane, hit, at);
    if (hit < 0) hit = 0;                                // not reached: the segment has mass
  }
  int found = -1;
  const int e1 = min(c0 + (hit + 1) * wide, c1);
  for (int e0 = c0 + hit * wide; e0 < e1; e0 += 256) {
    double m[8], next = at, own = 0.0;
    int col;
#pragma unroll
    for (int i = 0; i < 8; ++i) own += m[i] = mass_at<T>(row, e0 + 8 * lane + i, e1);
    next = at + warp_sum_d(own);
    pick_range<8>(m, target, lane, col, at);
    if (col >= 0) found = e0 + col;
    if (next > target) break;
    at = next;
  }
  if (lane == 0) a.next[b] = found;
}

template <typename T, int WARPS>
static int verify_sized(const VerifyArgs& a, cudaStream_t st) {
  const int segments = VD_CLUSTER * WARPS;
  const int len = (((a.V + segments - 1) / segments) + 31) & ~31;
  const int words = WARPS * len / 32;                    // a bit for each of a CTA's columns: 2 KB at V = 128 000, 64 KB at 2^22
  static std::atomic<uint64_t> done{0};
  if (int r = smem_opt_in(done, verify_kernel<T, WARPS>, 72 * 1024)) return r;
  verify_kernel<T, WARPS><<<a.B * VD_CLUSTER, WARPS * 32, words * 4, st>>>(a, words);
  TB_CUDA_CHECK(cudaGetLastError());
  return 0;
}
// Few sequences: as many threads as a CTA has, so that a row is loaded in one go. Many: CTAs of which four fit an SM.
template <typename T>
static int verify_launch(const VerifyArgs& a, cudaStream_t st) {
  return a.B * VD_CLUSTER <= sm_count() ? verify_sized<T, 32>(a, st) : verify_sized<T, 8>(a, st);
}

}  // namespace tb
using namespace tb;

int tb_set_check_word_verify(int* word) {
  TB_CUDA_CHECK(set_check_word_this_tu(word));
  return 0;
}

TB_EXPORT int tb_verify_draft(const VerifyCall* c, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  if (c->B <= 0) return 0;
  if (c->T < 1 || c->T > VD_MAX_NODES || c->V < 1) TB_FAIL(TB_E_ARG, "verify: 1 to %d nodes and at least one token in the vocabulary", VD_MAX_NODES);
  if (!c->probs || !c->tokens || !c->uniforms || !c->out) TB_FAIL(TB_E_ARG, "verify: null pointer");
  if (c->dtype != 0 && c->dtype != 1) TB_FAIL(TB_E_ARG, "verify: bf16 or fp32");
  if (c->B > 0x7fffffff / VD_CLUSTER || c->V > (1 << 22)) TB_FAIL(TB_E_TOO_LARGE, "verify: at most 2^22 tokens in the vocabulary");
  const VerifyArgs a{c->probs, c->draft, c->pb, c->pt, c->db, c->dt, c->tokens, c->parents, c->parents_ld, c->uniforms, c->counts,
                     c->out, c->out + 2 * c->B, c->out + c->B, (int)c->B, (int)c->T, (int)c->V};
  const int dtype = (int)c->dtype;
  return dtype == 0 ? verify_launch<bf16>(a, st) : verify_launch<float>(a, st);
}
