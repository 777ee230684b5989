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
  float *part_o, *part_ml;     // partial results, [slot][row][D] and [slot][row] of (maximum, sum): see slot_of()
  int4* plan;                  // of each CTA: the sequence, head and row tile, and tile that it begins with, and the tiles of a CTA (0: it has none)
  int* before;                 // the tiles in front of each sequence; null: the parts are looked for CTA by CTA
  int B, T, Hq, Hkv, G, page, page_tiles, page_shift, num_pages, row_tiles, grid;   // page_shift: log2 of a page's tiles, or -1
  int part_rows;               // rows of a slot of partial results
  int limit;                   // tokens of a sequence that the table can name, or fewer
  float scale_log2;
  int kernels;                 // launches of the call
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

// Sum of a value over the threads of a block in front of this one, and over all; scratch holds 32 ints.
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

// The deal: the tiles of all units in a row, `per` of them to each CTA, so that every CTA has the same share whatever the lengths. Where
// there are no more units than CTAs and the longest has at most WHOLE tiles more than such a share, each CTA has a unit: joining parts costs
// 2 to 4 us, as much as those tiles. Returns the CTA's first sequence and the tiles in front of it.
struct Deal {
  int per, first, last;   // tiles of a CTA (0: no unit is cut); this CTA's tiles are [first, last)
  int b, before;          // the sequence that tile `first` is of, and the tiles in front of that sequence
};
// `scratch`: 36 ints of shared memory.
template <int THREADS, int TILE, int ROUND, int WHOLE>
__device__ __forceinline__ Deal deal_tiles(const CacheAttnArgs& a, int* scratch) {
  Deal d;
  const int units = a.Hkv * a.row_tiles;
  int all = 0, keep_n = 0, keep_before = 0;
  int most = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const int nt = b < a.B ? (seq_len(a, b).len + TILE - 1) / TILE : 0, n = nt * units;
    most = max(most, nt);
    int total;
    const int before = all + block_prefix<THREADS>(n, scratch, total);
    if (b0 == 0) keep_n = n, keep_before = before;
    if (a.before && blockIdx.x == 0 && b < a.B) a.before[b] = before;
    all += total;
  }
  d.per = max((all + a.grid - 1) / a.grid, 1);
  d.per = (d.per + ROUND - 1) / ROUND * ROUND;
  if (a.before && !__syncthreads_or(most > d.per + WHOLE)) {
    // a unit for each CTA, and nothing to join; `first` and `before` count from the unit's sequence
    d.per = 0;
    d.b = blockIdx.x / units;
    d.before = 0;
    const int nt = d.b < a.B ? (seq_len(a, d.b).len + TILE - 1) / TILE : 0;
    d.first = ((int)blockIdx.x - d.b * units) * nt;
    d.last = d.first + nt;
    return d;
  }
  d.first = min((long)blockIdx.x * d.per, (long)all);
  d.last = min((long)d.first + d.per, (long)all);
  d.b = d.before = 0;
  if (d.first >= d.last) return d;
  all = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    int n = keep_n, before = keep_before, total = 0;
    if (a.B > THREADS) {
      n = b < a.B ? (seq_len(a, b).len + TILE - 1) / TILE * units : 0;
      before = all + block_prefix<THREADS>(n, scratch, total);
      all += total;
    }
    if (before <= d.first && d.first < before + n) scratch[34] = b, scratch[35] = before;
  }
  __syncthreads();
  d.b = scratch[34];
  d.before = scratch[35];
  return d;
}

// A walk over the tiles of the CTA's run: unit after unit, every STEP-th tile of each from the `offset`-th on.
struct Walk {
  int b, hr, h, nt, tile, end, left;   // hr: head and row tile; [tile, end): tiles of the unit in this CTA; left: tiles of the run from `end` on
  int head;                            // first tile of the unit in this CTA
  SeqLen s;
};
__device__ __forceinline__ void walk_unit(const CacheAttnArgs& a, Walk& w, int first_tile, int run) {
  w.head = first_tile;
  w.end = min(w.nt, first_tile + run);
  w.left = run - (w.end - first_tile);
  w.h = a.row_tiles == 1 ? w.hr : w.hr / a.row_tiles;
}
template <int TILE>
__device__ __forceinline__ void walk_begin(const CacheAttnArgs& a, Walk& w, const Deal& d, int offset) {
  w.b = d.b;
  w.s = seq_len(a, d.b);
  w.nt = (w.s.len + TILE - 1) / TILE;
  const int in = d.first - d.before;
  w.hr = in / w.nt;
  walk_unit(a, w, in - w.hr * w.nt, d.last - d.first);
  w.tile = w.head + offset;
}
// On to the next unit of the run; false: there is none.
template <int TILE>
__device__ __forceinline__ bool walk_next(const CacheAttnArgs& a, Walk& w, int offset) {
  if (w.left <= 0) return false;
  if (++w.hr == a.Hkv * a.row_tiles) {
    w.hr = 0;
    do {
      if (++w.b >= a.B) return false;
      w.s = seq_len(a, w.b);
      w.nt = (w.s.len + TILE - 1) / TILE;
    } while (w.nt == 0);
  }
  walk_unit(a, w, 0, w.left);
  w.tile = offset;
  return true;
}

// Where 16 tokens lie, tokens `pos` .. of a sequence. In two steps, so that the table's answer is not waited for where it is asked:
// the page that the table names and the place in it, later the row of the first token in the pool (-1: no page of the pool).
struct PageRef {
  int page, place;
};
__device__ __forceinline__ PageRef page_ref(const CacheAttnArgs& a, int b, int pos) {
  const int tile = pos >> 4;
  const int slot = a.page_shift >= 0 ? tile >> a.page_shift : tile / a.page_tiles;
  return {__ldg(a.table + (long)b * a.table_ld + slot), (tile - slot * a.page_tiles) * 16};
}
__device__ __forceinline__ long row_of(const CacheAttnArgs& a, const PageRef& r, int h) {
  return (unsigned)r.page < (unsigned)a.num_pages ? ((long)r.page * a.Hkv + h) * a.page + r.place : -1;
}

// The kernel that joins the parts may be set up while this one runs; it waits for this one's end before it reads anything.
__device__ __forceinline__ void release_join() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Sequences that see nothing: their rows are zeros.
template <int D, int THREADS>
__device__ __forceinline__ void zero_empty(const CacheAttnArgs& a) {
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (seq_len(a, b).len == 0)
      for (long i = threadIdx.x; i < (long)a.T * a.Hq * D / 8; i += THREADS) ((uint4*)(a.out + (long)b * a.T * a.Hq * D))[i] = make_uint4(0u, 0u, 0u, 0u);
}

__device__ __forceinline__ bool sees(const CacheAttnArgs& a, int b, int t, int pos, const SeqLen& s) {
  if (pos >= s.len) return false;
  const int j = pos - s.start;
  if (j < 0) return true;
  return a.mask ? a.mask[b * a.mask_b + t * a.mask_t + j] != 0 : j <= t;
}

// Scales of 8-bit values, v. Those from 2^122 on (pages hold none above 2^121) count as infinite. Those below 2^-92 count as none: their tokens'
// values are zeros, and the maximum of x + log2 v takes them for 2^CA_NONE, which moves it little beside scales of 2^-80 and more. The sum is
// that of P / v, P at most 2^14: in fp32's range for 2^21 tokens of the smallest scale, and for shares of 2^-18 and more beside one of 2^115.
constexpr float CA_NONE = -60.f;
__device__ __forceinline__ bool odd_scale(float v) { return (__float_as_uint(v) & 0x7fffffffu) >= 0x7c800000u; }
__device__ __forceinline__ bool no_scale(float v) { return (__float_as_uint(v) & 0x7fffffffu) < 0x11800000u; }

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

// Joins the units that the deal has cut; in cache_attention.cu.
int cache_attn_join(CacheAttnArgs& a, int D, int tile, int whole, cudaStream_t st);
// The same attention for many rows, on tcgen05; in cache_attention_sm100.cu.
int cache_attn_tc(CacheAttnArgs& a, int D, int kind, int* status, cudaStream_t st);

}  // namespace tb
