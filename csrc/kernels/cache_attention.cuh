// What the kernels of attention over a paged cache share: arguments, the deal of the work to the CTAs, decoding of 8-bit codes.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_util.h"

namespace tb {

enum : int { CA_BF16 = 0, CA_INT8 = 1, CA_E4M3 = 2 };

struct CacheAttnArgs {
  const bf16* q;               // [B, T, Hq, D] with strides in elements
  long qb, qt, qh;
  const void *k_pages, *v_pages;
  const float *k_scales, *v_scales;
  const int* table;            // [B, table_ld]
  const int* start;            // [B]: tokens in front of the new ones
  const int* counts;           // [B]: new tokens that count (null: T)
  const uint8_t* mask;         // [B or 1, T, T]: mask[t, j] != 0: token t sees new token j (null: j <= t)
  long mask_b, mask_t, table_ld;
  bf16* out;                   // [B, T, Hq, D] contiguous
  float *part_o, *part_ml;     // partial results: see slot_of()
  int* plan;                   // [0]: tiles of a CTA, [1 .. B]: tiles in front of each sequence
  int B, T, Hq, Hkv, G, page, page_tiles, page_shift, num_pages, row_tiles, grid;   // page_shift: log2 of a page's tiles, or -1
  int limit;                   // tokens of a sequence that the table can name, or fewer
  float scale_log2;
};

// Tokens that sequence b has to offer, and how many of its new ones count.
struct SeqLen {
  int start, count, len;
};
__device__ __forceinline__ SeqLen seq_len(const CacheAttnArgs& a, int b) {
  SeqLen s;
  s.start = max(__ldg(a.start + b), 0);
  s.count = a.counts ? min(max(__ldg(a.counts + b), 0), a.T) : a.T;
  s.len = s.count ? (int)min((long)s.start + s.count, (long)a.limit) : 0;
  return s;
}

// A CTA's partial results: a unit (sequence, head, row tile) that begins in front of the CTA's first tile goes to slot 2c, one that
// begins inside it and ends behind it to slot 2c + 1; whole units go straight to the output.
__device__ __forceinline__ int slot_of(int cta, bool begins_before) { return 2 * cta + (begins_before ? 0 : 1); }

// Sum of a value over the threads of a block in front of this one, and over all; scratch holds 33 ints.
template <int THREADS>
__device__ __forceinline__ int block_prefix(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  return before + incl - v;
}

// The deal: the tiles of all units in a row, `per` of them to each CTA, so that every CTA has the same share whatever the lengths.
// Returns the CTA's first sequence and the tiles in front of it. CTA 0 leaves the plan for the kernel that joins the parts.
struct Deal {
  int per, first, last;   // tiles of a CTA; this CTA's tiles are [first, last)
  int b, before;          // the sequence that tile `first` is of, and the tiles in front of that sequence
};
template <int THREADS, int TILE, int ROUND>
__device__ __forceinline__ Deal deal_tiles(const CacheAttnArgs& a, int* scratch) {
  Deal d;
  const int units = a.Hkv * a.row_tiles;
  int all = 0, keep_n = 0, keep_before = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const int n = b < a.B ? (seq_len(a, b).len + TILE - 1) / TILE * units : 0;
    int total;
    const int before = all + block_prefix<THREADS>(n, scratch, total);
    if (b0 == 0) keep_n = n, keep_before = before;
    if (blockIdx.x == 0 && b < a.B) a.plan[1 + b] = before;
    all += total;
  }
  d.per = max((all + a.grid - 1) / a.grid, 1);
  d.per = (d.per + ROUND - 1) / ROUND * ROUND;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = d.per;
  d.first = min((long)blockIdx.x * d.per, (long)all);
  d.last = min((long)d.first + d.per, (long)all);
  d.b = d.before = 0;
  if (d.first >= d.last) return d;
  __shared__ int found[2];
  all = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    int n = keep_n, before = keep_before, total = 0;
    if (a.B > THREADS) {
      n = b < a.B ? (seq_len(a, b).len + TILE - 1) / TILE * units : 0;
      before = all + block_prefix<THREADS>(n, scratch, total);
      all += total;
    }
    if (before <= d.first && d.first < before + n) found[0] = b, found[1] = before;
  }
  __syncthreads();
  d.b = found[0];
  d.before = found[1];
  return d;
}

__device__ __forceinline__ bool sees(const CacheAttnArgs& a, int b, int t, int pos, const SeqLen& s) {
  if (pos >= s.len) return false;
  const int j = pos - s.start;
  if (j < 0) return true;
  return a.mask ? a.mask[b * a.mask_b + t * a.mask_t + j] != 0 : j <= t;
}

// Two 8-bit codes (the low 16 bits of v) as two halves.
template <int KIND>
__device__ __forceinline__ uint32_t half2_of(uint32_t v) {
  uint32_t r;
  if (KIND == CA_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)v));
  } else {   // v holds the codes + 128: 0x6400 + u is the half 1024 + u
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6480)));
    r = *reinterpret_cast<const uint32_t*>(&h);
  }
  return r;
}
// Four codes as halves: r0 = (code 0, code 1), r1 = (code 2, code 3).
template <int KIND>
__device__ __forceinline__ void halves_of(uint32_t w, uint32_t& r0, uint32_t& r1) {
  if (KIND == CA_E4M3) {
    r0 = half2_of<KIND>(w);
    r1 = half2_of<KIND>(w >> 16);
  } else {
    w ^= 0x80808080u;
    r0 = half2_of<KIND>(__byte_perm(w, 0x64646464u, 0x4140));
    r1 = half2_of<KIND>(__byte_perm(w, 0x64646464u, 0x4342));
  }
}
// Codes of two tokens (words of four columns each) as halves (token 0, token 1) of each column.
template <int KIND>
__device__ __forceinline__ void pairs_of(uint32_t t0, uint32_t t1, uint32_t (&r)[4]) {
  const uint32_t lo = __byte_perm(t0, t1, 0x5140), hi = __byte_perm(t0, t1, 0x7362);
  halves_of<KIND>(lo, r[0], r[1]);
  halves_of<KIND>(hi, r[2], r[3]);
}

}  // namespace tb
