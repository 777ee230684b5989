// Attention of the newest tokens (one, or a tree of drafted ones) over a paged cache of keys and values (sm_100a), for few rows.
//
//   O[t] = sum_n P[t, n] V[n],  P = softmax(scale q_t . K[n]) over the context [0, start) and the new tokens that t's mask names
//
// The rows of one key/value head (the T tokens of its G query heads, row t G + g) share its keys. A warp takes 16 tokens at a time
// for 8 or 16 rows, the other way round: S^T = K Q^T and O^T += V^T P^T are mma.sync m16n8k16 products in which the tokens (then
// the columns of V) are the 16 and the rows the 8, so that one row costs 8 and not 16. Keys and values come out of a ring of the
// warp's own, filled by 16-byte cp.async: a page is a multiple of 16 tokens, so a tile is one contiguous piece of one page. Nothing
// but the end of a unit waits for another warp. These products are memory-bound (16 tokens of 256 bytes are 8 KB, which take 180
// clocks of the SM's share of HBM; their products take 32 clocks of the tensor pipe for 8 rows), and mma.sync takes its operands
// from registers, which is where the 8-bit codes are decoded.
//
// 8-bit codes are multiplied as halves: int8 and e4m3 are exact there, q is brought into the half's range by a power of two per row, and
// P carries the value's scale v: P = 2^(x - M + 8) v, M the largest x + log2 v that the row sees (with the power of two above v), so that halves have room
// for what counts in this row, whatever other scales there are (tokens that it does not see, or hardly attends to). The softmax's sum is
// that of P / v. P in halves has eight times the bits of bf16. Scores, maxima, sums and O are fp32.
//
// The work of all sequences is dealt to the CTAs in equal runs of tiles (deal_tiles), so ragged batches and single long sequences
// fill the GPU alike; a unit cut by the deal is joined by cache_attn_join_kernel. Short units are not cut (CA_WHOLE).
//
// Measured (a call among others, L2 cold): 64 sequences of up to 8192 tokens, 8 heads of D = 128 in e4m3, 618 MB: 112 us, 5.5 TB/s. One
// sequence of 131 072 tokens in int8, 277 MB: 61 us, 4.6 TB/s, of which 9 are two launches, the deal (a few dependent loads), the page
// table and the joining. One of 78 tokens: 5.3 us (9.1 with its units cut, 6.5 where the table could hold more).
#include "cache_attention.cuh"
#include "decode_calls.h"

namespace tb {

constexpr int CA_WARPS = 4;
constexpr int CA_THREADS = CA_WARPS * 32;
constexpr int CA_TILE = 16;   // tokens of a warp's tile
// Units stay whole while the longest has so many tiles more than a CTA's share. Measured (us, whole / cut): one sequence of 16 heads of 64,
// 77 tokens 6.3 / 9.3, 200: 7.7 / 9.2, 400 (21 tiles more) 9.8 / 9.2, 1600: 22.7 / 10.6; 16 sequences of 8 heads of 128 in e4m3, 400 tokens
// (18 more) 13.4 / 15.7, 800 (39 more) 19.1 / 18.2; 32 sequences of 16 heads of 64, 800 tokens (7 more) 22.4 / 27.2.
constexpr int CA_WHOLE = 20;

__device__ __forceinline__ uint32_t ca_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ca_copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ca_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ca_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ca_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool HALVES>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALVES)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool HALVES>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (HALVES) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// An 8 x 8 matrix of 16-bit values, two to a lane, the other way round.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// NT: blocks of 8 query rows.
template <int D, int KIND, int NT> struct CaShape {
  static constexpr bool HALVES = KIND != CA_BF16;
  static constexpr int ES = HALVES ? 1 : 2;
  static constexpr int ROW = D * ES;                       // bytes of a token
  static constexpr int CPR = ROW / 16;                     // 16-byte chunks of a token
  static constexpr int TILE_BYTES = CA_TILE * ROW;
  static constexpr int STAGE = 2 * TILE_BYTES + (HALVES ? 2 * CA_TILE * 4 : 0);
  static constexpr int STAGES = 3;
  static constexpr int OCC = TILE_BYTES == 4096 ? 2 : NT == 2 ? 3 : 4;   // CTAs of an SM
  static constexpr int MB = D / 16;                        // 16-column blocks of O
  static constexpr int BLOCKS = MB * NT;                   // of 16 columns and 8 rows: 512 bytes of floats
  static constexpr int PASS = 2 * TILE_BYTES / 512 < BLOCKS ? 2 * TILE_BYTES / 512 : BLOCKS;   // of which a stage takes so many
  static constexpr int ROWS = 8 * NT;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ML = CA_WARPS * ROWS * 2 * 4;
  static constexpr int WILD = CA_WARPS * CA_TILE * 8 * 4;  // P of a tile that has infinities or NaN among masked values
  static constexpr int SMEM = CA_WARPS * RING + ML + WILD;
};

// Where a token's 16-byte chunk lies in a tile: the exclusive-or spreads 8 tokens (keys), or tokens 0, 2, 4, 6 at neighbouring chunks
// (values), over all 32 banks.
template <int CPR>
__device__ __forceinline__ int chunk_at(int token, int chunk) {
  if (CPR == 4) return token * 64 + ((chunk ^ ((token >> 1) & 3)) << 4);
  return token * CPR * 16 + ((chunk ^ (token & 7)) << 4);
}
// Columns of O that a lane holds: block mb, i = 0 or 1. 8-bit values are read as the MB * 2 neighbouring columns of lane group g.
template <bool HALVES, int MB>
__device__ __forceinline__ int column_of(int mb, int i, int g) {
  return HALVES ? g * (2 * MB) + 2 * mb + i : mb * 16 + i * 8 + g;
}

template <bool HALVES, int MB>
__device__ __forceinline__ void put_pair(bf16* row, int mb, int g, float y0, float y1) {
  if (HALVES) *(uint32_t*)(row + column_of<true, MB>(mb, 0, g)) = pack2<false>(y0, y1);
  else row[column_of<false, MB>(mb, 0, g)] = __float2bfloat16(y0), row[column_of<false, MB>(mb, 1, g)] = __float2bfloat16(y1);
}

template <int D, int KIND, int NT>
__global__ void __launch_bounds__(CA_THREADS, (CaShape<D, KIND, NT>::OCC)) cache_attn_kernel(const CacheAttnArgs a) {
  using S = CaShape<D, KIND, NT>;
  constexpr bool HALVES = S::HALVES;
  constexpr int MB = S::MB;
  constexpr float OFFSET = HALVES ? 8.f : 0.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scratch[40];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  float* ml = (float*)(smem + CA_WARPS * S::RING);
  float* wild = (float*)(smem + CA_WARPS * S::RING + S::ML) + warp * CA_TILE * 8;
  const uint32_t ring_u = ca_smem(ring);

  const Deal deal = deal_tiles<CA_THREADS, CA_TILE, CA_WARPS, CA_WHOLE>(a, scratch);
  release_join();
  zero_empty<D, CA_THREADS>(a);
  if (deal.first >= deal.last) {
    if (threadIdx.x == 0) a.plan[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }

  // the loading side runs STAGES - 1 tiles ahead, its page number one more
  Walk ld;
  walk_begin<CA_TILE>(a, ld, deal, warp);
  bool more = true;
  PageRef next{-1, 0};
  auto seek = [&]() {
    while (more && ld.tile >= ld.end) more = walk_next<CA_TILE>(a, ld, warp);
    if (more) next = page_ref(a, ld.b, ld.tile * CA_TILE);
  };
  auto load = [&](int stage) {
    if (more) {
      const long next_row = row_of(a, next, ld.h);
      const int live = next_row < 0 ? 0 : min(ld.s.len - ld.tile * CA_TILE, CA_TILE);
      if (next_row < 0 && lane == 0 && !vacant_place(a.table + (long)ld.b * a.table_ld, next.page)) report_bad_index();
      const long row = max(next_row, 0l);
      const uint8_t* kp = (const uint8_t*)a.k_pages + row * S::ROW + lane * 16;
      const uint8_t* vp = (const uint8_t*)a.v_pages + row * S::ROW + lane * 16;
      const uint32_t dst = ring_u + stage * S::STAGE;
      if (live == CA_TILE) {
#pragma unroll
        for (int i = 0; i < S::TILE_BYTES / 512; ++i) {
          const int ch = i * 32 + lane;
          const uint32_t at = dst + chunk_at<S::CPR>(ch / S::CPR, ch % S::CPR);
          ca_copy16(at, kp + i * 512);
          ca_copy16(at + S::TILE_BYTES, vp + i * 512);
        }
      } else {   // zeros behind the end: what lies there may be anything
#pragma unroll 1
        for (int i = 0; i < S::TILE_BYTES / 512; ++i) {
          const int ch = i * 32 + lane, tok = ch / S::CPR;
          const uint32_t at = dst + chunk_at<S::CPR>(tok, ch % S::CPR);
          ca_copy16(at, kp + i * 512, tok < live);
          ca_copy16(at + S::TILE_BYTES, vp + i * 512, tok < live);
        }
      }
      if (HALVES && lane < 8) {
        const float* sc = (lane < 4 ? a.k_scales : a.v_scales) + row + (lane & 3) * 4;
        ca_copy16(dst + 2 * S::TILE_BYTES + lane * 16, sc, live > 0);
      }
      ld.tile += CA_WARPS;
      seek();
    }
    ca_commit();
  };
  seek();
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) load(i);

  Walk w;
  walk_begin<CA_TILE>(a, w, deal, warp);
  if (threadIdx.x == 0) a.plan[blockIdx.x] = make_int4(w.b, w.hr, w.head, deal.per);
  int stage = 0;

  while (true) {
    const int h = w.h, row0 = (w.hr - h * a.row_tiles) * S::ROWS;
    // Q as the second operand: lane (g, c) holds row g; 8-bit keys give lane c the D / 4 neighbouring columns from c D / 4 on
    uint32_t qf[NT][D / 16][2];
    float qs[NT][2];     // of rows 2c, 2c + 1, as the scores have them
    int tt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + n * 8 + g;
      const int t = r / a.G;
      const bool live = t < w.s.count;
      const bf16* qp = a.q + w.b * a.qb + (long)t * a.qt + (long)(h * a.G + r - t * a.G) * a.qh;
      float mine = a.scale_log2;
      if (!HALVES) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[n][kk][0] = live ? *(const uint32_t*)(qp + kk * 16 + 2 * c) : 0u;
          qf[n][kk][1] = live ? *(const uint32_t*)(qp + kk * 16 + 8 + 2 * c) : 0u;
        }
      } else {
        float big = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint2 v = live ? *(const uint2*)(qp + c * (D / 4) + kk * 4) : make_uint2(0u, 0u);
          qf[n][kk][0] = v.x;
          qf[n][kk][1] = v.y;
          big = fmaxf(big, fmaxf(fmaxf(fabsf(__uint_as_float(v.x << 16)), fabsf(__uint_as_float(v.x & 0xffff0000u))),
                                 fmaxf(fabsf(__uint_as_float(v.y << 16)), fabsf(__uint_as_float(v.y & 0xffff0000u)))));
        }
        big = quad_max(big);
        const uint32_t ex = __float_as_uint(big) >> 23;
        const bool plain = ex == 0 || ex > 253;
        const float down = plain ? 1.f : __uint_as_float((254u - ex) << 23);
        if (!plain) mine *= __uint_as_float(ex << 23);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t v = qf[n][kk][z];
            qf[n][kk][z] = pack2<true>(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xffff0000u) * down);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[n][e] = __shfl_sync(0xffffffffu, mine, (2 * c + e) * 4);
        tt[n][e] = min(__shfl_sync(0xffffffffu, t, (2 * c + e) * 4), a.T);
      }
    }

    float o[MB][NT][4], mx[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < MB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
      mx[n][0] = mx[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.f;
    }

    for (; w.tile < w.end; w.tile += CA_WARPS) {
      load(stage == 0 ? S::STAGES - 1 : stage - 1);
      ca_wait<S::STAGES - 1>();
      __syncwarp();
      const uint8_t* kt = ring + stage * S::STAGE;
      const uint8_t* vt = kt + S::TILE_BYTES;
      const int pos0 = w.tile * CA_TILE;

      // scores of tokens g (0, 1) and g + 8 (2, 3), rows 2c and 2c + 1
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
      if (!HALVES) {
        const int tok = lane & 15;
        const uint32_t ka = ca_smem(kt) + tok * S::ROW;
        const int x = (lane >> 4) ^ (tok & 7);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(ka + (((2 * kk) ^ x) << 4), kf);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<HALVES>(sc[n], kf, qf[n][kk][0], qf[n][kk][1]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < D / 64; ++q) {
          const uint4 v0 = *(const uint4*)(kt + chunk_at<S::CPR>(g, c * (D / 64) + q));
          const uint4 v1 = *(const uint4*)(kt + chunk_at<S::CPR>(g + 8, c * (D / 64) + q));
          const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            uint32_t kf[4];
            halves_of<KIND>(w0[k4], kf[0], kf[2]);
            halves_of<KIND>(w1[k4], kf[1], kf[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<HALVES>(sc[n], kf, qf[n][q * 4 + k4][0], qf[n][q * 4 + k4][1]);
          }
        }
      }

      const bool edge = pos0 + CA_TILE > min(w.s.start, w.s.len);   // new tokens in it, or the end of the sequence
      float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f}, reach[2] = {0.f, 0.f};
      if (HALVES) {
        const float* scales = (const float*)(vt + S::TILE_BYTES);
        ks[0] = scales[g], ks[1] = scales[g + 8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float v = scales[CA_TILE + g + 8 * i];
          const uint32_t ex = (__float_as_uint(v) & 0x7fffffffu) >> 23;
          vs[i] = odd_scale(v) ? __int_as_float(0x7fffffff) : no_scale(v) ? 0.f : v;
          // log2 of the power of two above v: the exponent as a float, by the bits of 2^23 + ex
          reach[i] = no_scale(v) ? CA_NONE : __uint_as_float(0x4b000000u | ex) - (8388608.f + 126.f);
        }
      }

      // the maximum that P is relative to moves only when a score is 2^6 above it: P stays below 2^6 (2^14 with the halves' offset)
      bool over = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = sc[n][e] * qs[n][e & 1];
          if (HALVES) x *= ks[e >> 1];
          if (edge && !(tt[n][e & 1] < a.T && sees(a, w.b, tt[n][e & 1], pos0 + g + (e >> 1) * 8, w.s))) x = -INFINITY;
          over |= x + reach[e >> 1] > mx[n][e & 1] + 6.f;
          sc[n][e] = x;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float top = fmaxf(sc[n][r] + reach[0], sc[n][2 + r] + reach[1]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(mx[n][r], top);
            const float f = now > mx[n][r] ? exp2f(mx[n][r] - now) : 1.f;
            mx[n][r] = now;
            sum[n][r] *= f;
#pragma unroll
            for (int j = 0; j < MB; ++j) o[j][n][r] *= f, o[j][n][2 + r] *= f;
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float ref[2] = {(mx[n][0] == -INFINITY ? 0.f : mx[n][0]) - OFFSET, (mx[n][1] == -INFINITY ? 0.f : mx[n][1]) - OFFSET};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p = exp2f(sc[n][e] - ref[e & 1]);
          sum[n][e & 1] += p;
          if (HALVES) p = sc[n][e] == -INFINITY ? 0.f : p * vs[e >> 1];
          sc[n][e] = p;
        }
        pf[n][0] = transpose8(pack2<HALVES>(sc[n][0], sc[n][1]));
        pf[n][1] = transpose8(pack2<HALVES>(sc[n][2], sc[n][3]));
      }

      // an infinity or a NaN among the new tokens' values meets rows that do not see it as 0 * inf: such a tile goes value by value
      bool odd = false;
      if (edge && KIND != CA_INT8) {
#pragma unroll 1
        for (int i = 0; i < S::TILE_BYTES / 512; ++i) {
          const uint4 v = *(const uint4*)(vt + i * 512 + lane * 16);
          const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            if (KIND == CA_BF16) odd |= (vw[k4] & 0x7f80u) == 0x7f80u || (vw[k4] & 0x7f800000u) == 0x7f800000u;
            else
#pragma unroll
              for (int z = 0; z < 32; z += 8) odd |= ((vw[k4] >> z) & 0x7fu) == 0x7fu;
          }
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      if (odd) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 4; ++e) wild[(g + 8 * (e >> 1)) * 8 + 2 * c + (e & 1)] = sc[n][e];
          __syncwarp();
#pragma unroll 1
          for (int tok = 0; tok < CA_TILE; ++tok) {
            const float p0 = wild[tok * 8 + 2 * c], p1 = wild[tok * 8 + 2 * c + 1];
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int d = column_of<HALVES, MB>(j, i, g);
                const uint8_t* at = vt + chunk_at<S::CPR>(tok, d * S::ES / 16) + (d * S::ES) % 16;
                float v;
                if (KIND == CA_BF16) v = __bfloat162float(*(const bf16*)at);
                else v = __half2float(__ushort_as_half((unsigned short)half2_of<CA_E4M3>(*at)));
                if (p0 != 0.f) o[j][n][2 * i] += p0 * v;
                if (p1 != 0.f) o[j][n][2 * i + 1] += p1 * v;
              }
          }
        }
      } else if (!HALVES) {
        const int tok = (lane & 7) + ((lane >> 4) << 3);
        const uint32_t va = ca_smem(vt) + tok * S::ROW;
        const int x = ((lane >> 3) & 1) ^ (tok & 7);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
          uint32_t vf[4];
          ldsm4_t(va + (((2 * j) ^ x) << 4), vf);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<HALVES>(o[j][n], vf, pf[n][0], pf[n][1]);
        }
      } else {
        // lane (g, c): 2 MB neighbouring columns of tokens 2c, 2c + 1, 2c + 8, 2c + 9; block j takes columns 2j and 2j + 1 of them
        uint32_t vw[4][MB / 2];
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          const int tok = 2 * c + (t4 & 1) + (t4 >> 1) * 8;
          if (D == 128) {
            const uint4 v = *(const uint4*)(vt + chunk_at<S::CPR>(tok, g));
            vw[t4][0] = v.x, vw[t4][1] = v.y, vw[t4][MB / 2 - 2] = v.z, vw[t4][MB / 2 - 1] = v.w;
          } else {
            const uint2 v = *(const uint2*)(vt + chunk_at<S::CPR>(tok, g >> 1) + (g & 1) * 8);
            vw[t4][0] = v.x, vw[t4][1] = v.y;
          }
        }
#pragma unroll
        for (int q = 0; q < MB / 2; ++q) {
          uint32_t lo[4], hi[4];
          pairs_of<KIND>(vw[0][q], vw[1][q], lo);
          pairs_of<KIND>(vw[2][q], vw[3][q], hi);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t vf[4] = {lo[2 * z], lo[2 * z + 1], hi[2 * z], hi[2 * z + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<HALVES>(o[q * 2 + z][n], vf, pf[n][0], pf[n][1]);
          }
        }
      }
      __syncwarp();
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    }

    // join the warps: rows of one maximum, then O through the stage that is free
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], x);
        if (g == 0) *(float2*)(ml + (warp * S::ROWS + n * 8 + 2 * c + r) * 2) = make_float2(mx[n][r], sum[n][r]);
      }
    const int free_stage = stage == 0 ? S::STAGES - 1 : stage - 1;
    if (lane == 0) scratch[36 + warp] = free_stage;
    __syncthreads();
    const bool whole = w.head == 0 && w.end == w.nt;
    const int slot = slot_of(blockIdx.x, w.head > 0);
    float* part = a.part_o + (long)slot * S::ROWS * D;
    float norm[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = -INFINITY, all = 0.f;
        const int row = n * 8 + 2 * c + r;
#pragma unroll
        for (int v = 0; v < CA_WARPS; ++v) top = fmaxf(top, ml[(v * S::ROWS + row) * 2]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int v = 0; v < CA_WARPS; ++v) {
          const float2 y = *(const float2*)(ml + (v * S::ROWS + row) * 2);
          all += y.y * exp2f(y.x - ref);
        }
        const float f = exp2f(mx[n][r] - ref);
#pragma unroll
        for (int j = 0; j < MB; ++j) o[j][n][r] *= f, o[j][n][2 + r] *= f;
        norm[n][r] = all > 0.f || all != all ? 1.f / all : 0.f;   // a row that sees nothing: zeros
        if (!whole && warp == 0 && g == 0) *(float2*)(a.part_ml + ((long)slot * S::ROWS + row) * 2) = make_float2(top, all);
      }
#pragma unroll
    for (int p0 = 0; p0 < S::BLOCKS; p0 += S::PASS) {
      if (p0) __syncthreads();
      float4* mine = (float4*)(ring + free_stage * S::STAGE);
#pragma unroll
      for (int i = 0; i < S::PASS; ++i) {
        const int n = (p0 + i) / MB, j = (p0 + i) % MB;
        mine[i * 32 + lane] = make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < S::PASS / CA_WARPS; ++k) {
        const int i = warp * (S::PASS / CA_WARPS) + k;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int v = 0; v < CA_WARPS; ++v) {
          const float4 z = ((const float4*)(smem + v * S::RING + scratch[36 + v] * S::STAGE))[i * 32 + lane];
          y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
        }
        const int n = (p0 + i) / MB, j = (p0 + i) % MB;
        if (!whole) {
          float* pr = part + (n * 8 + 2 * c) * D;
          if (HALVES) {
            *(float2*)(pr + column_of<HALVES, MB>(j, 0, g)) = make_float2(y.x, y.z);
            *(float2*)(pr + D + column_of<HALVES, MB>(j, 0, g)) = make_float2(y.y, y.w);
          } else {
            pr[column_of<HALVES, MB>(j, 0, g)] = y.x, pr[column_of<HALVES, MB>(j, 1, g)] = y.z;
            pr[D + column_of<HALVES, MB>(j, 0, g)] = y.y, pr[D + column_of<HALVES, MB>(j, 1, g)] = y.w;
          }
        } else {
          const float yy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            int t = 0;
            float f = 0.f;
#pragma unroll
            for (int m = 0; m < NT; ++m)
              if (m == n) t = tt[m][r], f = norm[m][r];
            if (t >= a.T) continue;
            const int row = row0 + n * 8 + 2 * c + r;
            bf16* op = a.out + (((long)w.b * a.T + t) * a.Hq + h * a.G + row - t * a.G) * D;
            const bool live = t < w.s.count;
            put_pair<HALVES, MB>(op, j, g, live ? yy[r] * f : 0.f, live ? yy[2 + r] * f : 0.f);
          }
        }
      }
    }
    __syncthreads();   // the stages and ml are free again
    if (!walk_next<CA_TILE>(a, w, warp)) break;
  }
  ca_wait<0>();
}

// Joins the parts of the units that the deal has cut. Blocks x are either units, or CTAs of the attention kernel and look at the unit that
// the CTA began with: if that is its first cut, they join it (whichever is fewer: a block that finds nothing to do still costs a launch
// of its own, and 4736 of them took 5 us). `share` warps have a row between them, and its parts.
constexpr int CJ_WARPS = 8;
template <int D>
__global__ void __launch_bounds__(CJ_WARPS * 32) cache_attn_join_kernel(const CacheAttnArgs a, int tile, int share) {
  constexpr int N = D / 32;                            // columns of a lane
  __shared__ float buf[CJ_WARPS][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int b, hr, per, first;
  if (a.before) {
    const int units = a.Hkv * a.row_tiles;
    b = blockIdx.x / units, hr = blockIdx.x - b * units;
    per = a.plan[0].w;
    if (per == 0) return;                                // no unit has been cut
  } else {
    const int4 p = a.plan[blockIdx.x];
    if (p.w == 0 || p.z == 0 || p.z > p.w) return;     // nothing; a unit's beginning; not its first cut
    b = p.x, hr = p.y, per = p.w;
    first = blockIdx.x * per - p.z;
  }
  const SeqLen s = seq_len(a, b);
  const int nt = (s.len + tile - 1) / tile;
  if (a.before) first = a.before[b] + hr * nt;
  if (nt == 0) return;                                 // zeros already
  const int c0 = first / per, c1 = (first + nt - 1) / per;
  if (c0 == c1) return;                                // whole: written already
  const int h = a.row_tiles == 1 ? hr : hr / a.row_tiles;
  const int r = blockIdx.y * (CJ_WARPS / share) + warp / share, sub = warp % share;
  const int row = (hr - h * a.row_tiles) * a.part_rows + r, t = row / a.G;
  const bool mine = r < a.part_rows && t < a.T;
  float top = -INFINITY, all = 0.f, y[N] = {};
  if (mine) {
#pragma unroll 4
    for (int k = c0 + lane; k <= c1; k += 32) {
      const float2 z = *(const float2*)(a.part_ml + ((long)slot_of(k, k > c0) * a.part_rows + r) * 2);
      const float now = fmaxf(top, z.x), ref = now == -INFINITY ? 0.f : now;
      all = all * exp2f(top - ref) + z.y * exp2f(z.x - ref);
      top = now;
    }
    const float now = warp_max(top), ref = now == -INFINITY ? 0.f : now;
    all = warp_sum(all * exp2f(top - ref));
#pragma unroll 8
    for (int k = c0 + sub; k <= c1; k += share) {
      const long at = (long)slot_of(k, k > c0) * a.part_rows + r;
      const float f = exp2f(a.part_ml[at * 2] - ref);
      const float* o = a.part_o + at * D + lane * N;
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 z = *(const float2*)(o + i);
        y[i] += z.x * f, y[i + 1] += z.y * f;
      }
    }
  }
  if (share > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[warp][lane * N + i] = y[i];
    __syncthreads();
    if (sub) return;
    for (int v = 1; v < share; ++v)
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] += buf[warp + v][lane * N + i];
  }
  if (!mine) return;
  const float norm = t < s.count && (all > 0.f || all != all) ? 1.f / all : 0.f;   // a row that sees nothing: zeros
  bf16* op = a.out + (((long)b * a.T + t) * a.Hq + h * a.G + row - t * a.G) * D + lane * N;
#pragma unroll
  for (int i = 0; i < N; i += 2) *(uint32_t*)(op + i) = t < s.count ? pack2<false>(y[i] * norm, y[i + 1] * norm) : 0u;
}

static long ca_units(const CacheAttnArgs& a) { return (long)a.B * a.Hkv * a.row_tiles; }

int cache_attn_join(CacheAttnArgs& a, int D, int tile, int whole, cudaStream_t st) {
  if (a.before && (a.limit + tile - 1) / tile <= whole) return 0;   // the table is so short that no unit can have been cut: 1 us
  a.kernels = 2;
  // one sequence cuts few units into many parts, many sequences many units into few
  const long units = ca_units(a);
  const int share = units * 8 >= a.grid ? 1 : CJ_WARPS;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its launch overlaps the attention kernel: 2 us
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.before ? units : a.grid), (unsigned)((a.part_rows * share + CJ_WARPS - 1) / CJ_WARPS));
  cfg.blockDim = dim3(CJ_WARPS * 32);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  TB_CUDA_CHECK(D == 64 ? cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<64>, a, tile, share) : cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<128>, a, tile, share));
  return 0;
}

template <int D, int KIND, int NT>
static int cache_attn_launch(CacheAttnArgs& a, cudaStream_t st) {
  using S = CaShape<D, KIND, NT>;
  static std::atomic<uint64_t> done{0};
  if (int r = smem_opt_in(done, cache_attn_kernel<D, KIND, NT>, S::SMEM)) return r;
  a.grid = S::OCC * sm_count();
  if (ca_units(a) > a.grid) a.before = nullptr;
  cache_attn_kernel<D, KIND, NT><<<a.grid, CA_THREADS, S::SMEM, st>>>(a);
  TB_CUDA_CHECK(cudaGetLastError());
  return cache_attn_join(a, D, CA_TILE, CA_WHOLE + CA_WARPS, st);
}

template <int D, int KIND>
static int cache_attn_rows(CacheAttnArgs& a, int nt, cudaStream_t st) {
  return nt == 1 ? cache_attn_launch<D, KIND, 1>(a, st) : cache_attn_launch<D, KIND, 2>(a, st);
}

template <int D>
static int cache_attn_kind(CacheAttnArgs& a, int kind, int nt, cudaStream_t st) {
  if (kind == CA_BF16) return cache_attn_rows<D, CA_BF16>(a, nt, st);
  if (kind == CA_INT8) return cache_attn_rows<D, CA_INT8>(a, nt, st);
  return cache_attn_rows<D, CA_E4M3>(a, nt, st);
}

// Blocks of 8 rows that a CTA takes.
static int ca_row_blocks(long rows) { return rows <= 8 ? 1 : 2; }
constexpr int CA_MAX_OCC = 4;
// Up to here the rows go to this file's kernel, beyond to the one on tcgen05. Both measured (us, this one / that one; B x context, eight
// heads of D = 128): 16 rows bf16 8 x 2000 22 / 34, 8 x 16000 72 / 106, int8 28 / 37 and 80 / 145; 24 rows (32 of this one's) bf16 40 / 34
// and 218 / 106, int8 42 / 37 and 212 / 145. With D = 64 and 24 rows it is 26 / 28 and 84 / 86, int8 28 / 31 and 95 / 112.
constexpr long CA_MAX_ROWS = 16;
// More rows go here too while what this kernel could read at most (every 16 rows their own keys and values, up to the table's end) is less
// than so many bytes: its launch is half as long. Measured (us, this one / that one): 27 tokens of 4 heads, two sequences of 8 int8 heads of
// 128, 77 tokens (3 MB) 10.3 / 12.6, 200 (6.5 MB) 13.3 / 13.7, 800 (24 MB) 25.5 / 20.6; 20 tokens, 16 heads of 64, bf16, 77 tokens (0.8 MB)
// 7.1 / 10.4; 64 tokens, 16 heads of 64, int8, 200 tokens (2.2 MB) 10.9 / 15.8, 800 (7.1 MB) 20.1 / 16.2.
constexpr double CA_SMALL = 5e6;
static long ca_slots(bool tc) { return 2l * (tc ? 1 : CA_MAX_OCC) * sm_count(); }
// Rows of a slot of partial results: a multiple of 4, so that what follows stays aligned.
static int ca_part_rows(long rows, bool tc) { return tc ? (int)(rows < 128 ? (rows + 3) & ~3l : 128) : 8 * ca_row_blocks(rows); }
static long ca_workspace(long rows, int D, bool tc) { return ca_slots(tc) * ca_part_rows(rows, tc) * (D * 4 + 8) + ca_slots(tc) / 2 * (16 + 4); }

}  // namespace tb
using namespace tb;

int tb_set_check_word_cache_attention_tc(int* word);
int tb_set_check_word_cache_attention(int* word) {
  TB_CUDA_CHECK(set_check_word_this_tu(word));
  return tb_set_check_word_cache_attention_tc(word);
}

// Bytes of workspace that tb_cache_attention needs for these sizes.
TB_EXPORT long tb_cache_attention_workspace(int B, int T, int Hq, int Hkv, int D) {
  if (ensure_device() || Hkv <= 0) return -1;
  const long rows = (long)T * (Hq / Hkv), few = ca_workspace(rows, D, false), many = ca_workspace(rows, D, true);
  return rows > CA_MAX_ROWS && many > few ? many : few;   // both kernels can be taken beyond CA_MAX_ROWS
}

// q [B, T, Hq, D] bf16 (strides in elements, multiples of 8; 16-byte aligned), out contiguous. ws: tb_cache_attention_workspace() bytes,
// 16-byte aligned, used by this call alone.
TB_EXPORT int tb_cache_attention(const CacheAttnCall* c, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  const long D = c->D, page = c->page, rows = c->Hkv > 0 ? c->T * (c->Hq / c->Hkv) : 0;
  const int kind = (int)c->kind;
  if (c->B <= 0 || c->T <= 0 || c->Hq <= 0) return 0;
  if (!c->q || !c->out || !c->ws || !c->k_pages || !c->v_pages || !c->table || !c->start || (kind != CA_BF16 && (!c->k_scales || !c->v_scales)))
    TB_FAIL(TB_E_ARG, "cache attention: null pointer");
  if (D != 64 && D != 128) TB_FAIL(TB_E_ARG, "cache attention: head dim 64 or 128");
  if (c->Hkv <= 0 || c->Hq % c->Hkv || c->kind < 0 || c->kind > 2) TB_FAIL(TB_E_ARG, "cache attention: query heads must be a multiple of the cache's");
  if (page <= 0 || page % CA_TILE || c->num_pages < 0 || c->pages_per_seq < 0 || c->max_len < 0) TB_FAIL(TB_E_ARG, "cache attention: pages of a multiple of %d tokens", CA_TILE);
  if (((uintptr_t)c->q | (uintptr_t)c->out | (uintptr_t)c->ws | (uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15 || c->qb % 8 || c->qt % 8 || c->qh % 8)
    TB_FAIL(TB_E_ARG, "cache attention: 16-byte aligned rows");
  if (kind != CA_BF16 && (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 15)) TB_FAIL(TB_E_ARG, "cache attention: 16-byte aligned scales");
  if (c->B > 0x7fffffff || c->Hq > 0x7fffffff || rows > 0x7fffff00l || page > 0x7fff0000l || c->num_pages > 0x7fffffff || c->pages_per_seq > 0x7fff0000l)
    TB_FAIL(TB_E_TOO_LARGE, "cache attention: too much for one call");
  CacheAttnArgs a{};
  a.q = (const bf16*)c->q, a.qb = c->qb, a.qt = c->qt, a.qh = c->qh;
  a.k_pages = c->k_pages, a.v_pages = c->v_pages, a.k_scales = c->k_scales, a.v_scales = c->v_scales;
  a.table = c->table, a.table_ld = c->table_ld, a.start = c->start, a.counts = c->counts;
  a.mask = c->mask, a.mask_b = c->mask_b, a.mask_t = c->mask_t, a.out = (bf16*)c->out;
  a.B = (int)c->B, a.T = (int)c->T, a.Hq = (int)c->Hq, a.Hkv = (int)c->Hkv, a.G = a.Hq / a.Hkv, a.page = (int)page, a.num_pages = (int)c->num_pages;
  a.scale_log2 = (float)(c->scale * 1.4426950408889634);
  const long held = c->pages_per_seq * page, limit = held < c->max_len ? held : c->max_len;
  const double most = (double)c->B * c->Hkv * ((rows + 15) / 16) * limit * D * (kind == CA_BF16 ? 4 : 2);
  const bool tc = rows > CA_MAX_ROWS && most > CA_SMALL;
  const int nt = ca_row_blocks(rows);
  const int per_tile = tc ? 128 : 8 * nt;
  a.row_tiles = (int)((rows + per_tile - 1) / per_tile);
  a.page_tiles = (int)(page / CA_TILE);
  a.page_shift = (a.page_tiles & (a.page_tiles - 1)) ? -1 : __builtin_ctz((unsigned)a.page_tiles);
  a.limit = (int)limit;
  if (limit > 0x7fff0000l || (double)(limit + CA_TILE) / CA_TILE * (double)ca_units(a) > 2e9) TB_FAIL(TB_E_TOO_LARGE, "cache attention: too much for one call");
  const long slots = ca_slots(tc);
  a.part_rows = ca_part_rows(rows, tc);
  a.part_o = (float*)c->ws;
  a.part_ml = a.part_o + slots * a.part_rows * D;
  a.plan = (int4*)(a.part_ml + slots * a.part_rows * 2);
  a.before = (int*)(a.plan + slots / 2);               // there are at most as many sequences as units, and units as CTAs, where it is used
  a.kernels = 1;
  const int rc = tc ? cache_attn_tc(a, (int)D, kind, c->status, st) : D == 64 ? cache_attn_kind<64>(a, kind, nt, st) : cache_attn_kind<128>(a, kind, nt, st);
  c->kernels = a.kernels;
  return rc;
}
