// Attention of the newest tokens (one, or a tree of drafted ones) over a paged cache of keys and values (sm_100a), for few rows.
//
//   O[t] = sum_n P[t, n] V[n],  P = softmax(scale q_t . K[n]) over the context [0, start) and the new tokens that t's mask names
//
// The rows of one key/value head (the T tokens of its G query heads, row t G + g) share its keys. A warp takes 16 tokens at a time
// for 16 or 32 rows: S and P V are mma.sync m16n8k16 products whose other operand comes out of a ring of the warp's own, filled by
// 16-byte cp.async: a page is a multiple of 16 tokens, so a tile is one contiguous piece of one page. Nothing but the end of a unit
// waits for another warp. These products are memory-bound (a token of 256 to 512 bytes meets 16 rows: 8192 to 16384 multiply-adds
// for 11 to 22 clocks of the SM's share of HBM, where the tensor pipe takes 8 to 16), and mma.sync takes operands from registers,
// which is where the 8-bit codes are decoded.
//
// 8-bit codes are multiplied as halves: int8 and e4m3 are exact there, q is brought into the half's range by a power of two per row,
// P carries the value's scale (relative to a running power of two, the largest scale so far) and an offset of 2^14 against
// underflow. P in halves has eight times the bits of bf16. Scores, maxima, sums and O are fp32.
//
// The work of all sequences is dealt to the CTAs in equal runs of tiles (deal_tiles), so ragged batches and single long sequences
// fill the GPU alike; a unit cut by the deal is joined by cache_attn_join_kernel.
#include "cache_attention.cuh"

namespace tb {

constexpr int CA_WARPS = 4;
constexpr int CA_THREADS = CA_WARPS * 32;
constexpr int CA_TILE = 16;   // tokens of a warp's tile

__device__ __forceinline__ uint32_t ca_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ca_copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
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
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <int D, int KIND, int MT> struct CaShape {
  static constexpr bool HALVES = KIND != CA_BF16;
  static constexpr int ES = HALVES ? 1 : 2;
  static constexpr int ROW = D * ES;                       // bytes of a token
  static constexpr int CPR = ROW / 16;                     // 16-byte chunks of a token
  static constexpr int TILE_BYTES = CA_TILE * ROW;
  static constexpr int STAGE = 2 * TILE_BYTES + (HALVES ? 2 * CA_TILE * 4 : 0);
  static constexpr int STAGES = HALVES ? 4 : 3;
  static constexpr int NB = D / 8;                         // 8-column blocks of O
  static constexpr int NBP = 2 * TILE_BYTES / 512;         // of which a stage holds, as floats of 16 rows
  static constexpr int ROWS = 16 * MT;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ML = CA_WARPS * ROWS * 2 * 4;
  static constexpr int WILD = CA_WARPS * 16 * CA_TILE * 4; // P of a tile that has infinities or NaN among masked values
  static constexpr int SMEM = CA_WARPS * RING + ML + WILD;
};

// Where a token's 16-byte chunk lies in a tile. Lanes of one access read tokens f(i, n) = 4 (n / 2) + 2 i + n % 2, n = 0 .. 7 (keys),
// or 4c, c = 0 .. 3 (values): the exclusive-or spreads either over all 32 banks.
template <int CPR>
__device__ __forceinline__ int chunk_at(int token, int chunk) {
  if (CPR == 4) return token * 64 + ((chunk ^ ((token >> 2) & 3)) << 4);
  return token * CPR * 16 + ((chunk ^ ((((token >> 2) << 1) | (token & 1)) & 7)) << 4);
}

// A warp's walk over its tiles of the CTA's run: unit after unit, every CA_WARPS-th tile.
struct Walk {
  int b, hr, nt, tile, end, left;   // hr: head and row tile; [tile, end): tiles of the unit in this CTA; left: tiles of the run from `end` on
  int head;                         // first tile of the unit in this CTA
  SeqLen s;
};
__device__ __forceinline__ void walk_unit(const CacheAttnArgs& a, Walk& w, int first_tile, int run) {
  w.head = first_tile;
  w.end = min(w.nt, first_tile + run);
  w.left = run - (w.end - first_tile);
}
__device__ __forceinline__ void walk_begin(const CacheAttnArgs& a, Walk& w, const Deal& d, int warp) {
  w.b = d.b;
  w.s = seq_len(a, d.b);
  w.nt = (w.s.len + CA_TILE - 1) / CA_TILE;
  const int in = d.first - d.before;
  w.hr = in / w.nt;
  walk_unit(a, w, in - w.hr * w.nt, d.last - d.first);
  w.tile = w.head + warp;
}
// On to the next unit of the run; false: there is none.
__device__ __forceinline__ bool walk_next(const CacheAttnArgs& a, Walk& w, int warp) {
  if (w.left <= 0) return false;
  if (++w.hr == a.Hkv * a.row_tiles) {
    w.hr = 0;
    do {
      if (++w.b >= a.B) return false;
      w.s = seq_len(a, w.b);
      w.nt = (w.s.len + CA_TILE - 1) / CA_TILE;
    } while (w.nt == 0);
  }
  walk_unit(a, w, 0, w.left);
  w.tile = warp;
  return true;
}

template <int D, int KIND, int MT>
__global__ void __launch_bounds__(CA_THREADS, 2) cache_attn_kernel(const CacheAttnArgs a) {
  using S = CaShape<D, KIND, MT>;
  constexpr bool HALVES = S::HALVES;
  constexpr float OFFSET = HALVES ? 14.f : 0.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scratch[40];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  float* ml = (float*)(smem + CA_WARPS * S::RING);
  float* wild = (float*)(smem + CA_WARPS * S::RING + S::ML) + warp * 16 * CA_TILE;
  const uint32_t ring_u = ca_smem(ring);

  const Deal deal = deal_tiles<CA_THREADS, CA_TILE, CA_WARPS>(a, scratch);
  if (deal.first >= deal.last) return;

  // the loading side runs STAGES - 1 tiles ahead, its page number one more
  Walk ld;
  walk_begin(a, ld, deal, warp);
  bool more = true;
  int pg = -1;
  auto seek = [&]() {
    while (more && ld.tile >= ld.end) more = walk_next(a, ld, warp);
    if (more) pg = page_of(a, ld.b, ld.tile * CA_TILE);
  };
  auto load = [&](int stage) {
    if (more) {
      const int pos = ld.tile * CA_TILE, h = ld.hr / a.row_tiles;
      const int live = pg < 0 ? 0 : min(ld.s.len - pos, CA_TILE);
      if (pg < 0 && lane == 0) report_bad_index();
      const long row = ((long)max(pg, 0) * a.Hkv + h) * a.page + pos % a.page;
      const uint8_t* kp = (const uint8_t*)a.k_pages + row * S::ROW + lane * 16;
      const uint8_t* vp = (const uint8_t*)a.v_pages + row * S::ROW + lane * 16;
      const uint32_t dst = ring_u + stage * S::STAGE;
#pragma unroll
      for (int i = 0; i < S::TILE_BYTES / 512; ++i) {
        const int ch = i * 32 + lane, tok = ch / S::CPR;
        const uint32_t at = dst + chunk_at<S::CPR>(tok, ch % S::CPR);
        ca_copy16(at, kp + i * 512, tok < live);
        ca_copy16(at + S::TILE_BYTES, vp + i * 512, tok < live);
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
  walk_begin(a, w, deal, warp);
  int stage = 0;
  // lane offsets into a tile
  const int ktok = HALVES ? 4 * (g >> 1) + (g & 1) : 4 * ((lane & 7) >> 1) + 2 * (lane >> 4) + (lane & 1);
  const int vtok = HALVES ? 4 * c : 4 * ((lane & 7) >> 1) + 2 * ((lane >> 3) & 1) + (lane & 1);

  while (true) {
    const int h = w.hr / a.row_tiles, row0 = (w.hr - h * a.row_tiles) * S::ROWS;
    uint32_t qf[MT][D / 16][4];
    float qs[MT][2];
    int tt[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + m * 16 + e * 8 + g;
        const int t = r / a.G;
        tt[m][e] = t;
        const bool live = t < w.s.count;
        const bf16* qp = a.q + w.b * a.qb + (long)t * a.qt + (long)(h * a.G + r - t * a.G) * a.qh;
        qs[m][e] = a.scale_log2;
        if (!HALVES) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            qf[m][kk][e] = live ? *(const uint32_t*)(qp + kk * 16 + 2 * c) : 0u;
            qf[m][kk][2 + e] = live ? *(const uint32_t*)(qp + kk * 16 + 8 + 2 * c) : 0u;
          }
        } else {
          float big = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint2 v = live ? *(const uint2*)(qp + c * (D / 4) + kk * 4) : make_uint2(0u, 0u);
            qf[m][kk][e] = v.x;
            qf[m][kk][2 + e] = v.y;
            big = fmaxf(big, fmaxf(fmaxf(fabsf(__uint_as_float(v.x << 16)), fabsf(__uint_as_float(v.x & 0xffff0000u))),
                                   fmaxf(fabsf(__uint_as_float(v.y << 16)), fabsf(__uint_as_float(v.y & 0xffff0000u)))));
          }
          big = quad_max(big);
          const uint32_t ex = __float_as_uint(big) >> 23;
          const bool plain = ex == 0 || ex > 253;
          const float down = plain ? 1.f : __uint_as_float((254u - ex) << 23);
          if (!plain) qs[m][e] *= __uint_as_float(ex << 23);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int z = 0; z < 4; z += 2) {
              const uint32_t v = qf[m][kk][z + e];
              qf[m][kk][z + e] = pack2<true>(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xffff0000u) * down);
            }
        }
      }

    float o[MT][S::NB][4], mx[MT][2], sum[MT][2], unit_v = 0.f;   // unit_v: the power of two that O's values are relative to
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int j = 0; j < S::NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][j][e] = 0.f;
      mx[m][0] = mx[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
    }

    for (; w.tile < w.end; w.tile += CA_WARPS) {
      load(stage == 0 ? S::STAGES - 1 : stage - 1);
      ca_wait<S::STAGES - 1>();
      __syncwarp();
      const uint8_t* kt = ring + stage * S::STAGE;
      const uint8_t* vt = kt + S::TILE_BYTES;
      const int pos0 = w.tile * CA_TILE;

      // S[i]: tokens pos0 + 4c + 2i + {0, 1}
      float sc[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][i][e] = 0.f;
      if (!HALVES) {
        const uint32_t ka = ca_smem(kt) + ktok * S::ROW;
        const int x = ((lane >> 3) & 1) ^ ((((ktok >> 2) << 1) | (ktok & 1)) & 7);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(ka + (((2 * kk) ^ x) << 4), kf);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<HALVES>(sc[m][0], qf[m][kk], kf[0], kf[1]);
            mma16816<HALVES>(sc[m][1], qf[m][kk], kf[2], kf[3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < D / 64; ++q) {
            const uint4 v = *(const uint4*)(kt + chunk_at<S::CPR>(ktok + 2 * i, c * (D / 64) + q));
            const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              uint32_t b0, b1;
              halves_of<KIND>(vw[k4], b0, b1);
#pragma unroll
              for (int m = 0; m < MT; ++m) mma16816<HALVES>(sc[m][i], qf[m][q * 4 + k4], b0, b1);
            }
          }
      }

      const bool edge = pos0 + CA_TILE > min(w.s.start, w.s.len);   // new tokens in it, or the end of the sequence
      float vs[4];
      if (HALVES) {
        const float4 kv4 = *(const float4*)(vt + S::TILE_BYTES + c * 16);
        const float4 vv4 = *(const float4*)(vt + S::TILE_BYTES + 64 + c * 16);
        const float ks[4] = {kv4.x, kv4.y, kv4.z, kv4.w};
        vs[0] = vv4.x, vs[1] = vv4.y, vs[2] = vv4.z, vs[3] = vv4.w;
        if (edge) {
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4)
            if (pos0 + 4 * c + k4 >= w.s.len) vs[k4] = 0.f;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[m][i][e] *= ks[2 * i + (e & 1)];
        const float top = quad_max(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])));
        const float up = __uint_as_float((__float_as_uint(top) + 0x7fffffu) & 0x7f800000u);
        if (up > unit_v) {
          const float f = unit_v / up;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[m][j][e] *= f;
          unit_v = up;
        }
        const float inv = unit_v > 0.f ? __uint_as_float(0x7f000000u - __float_as_uint(unit_v)) : 0.f;
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) vs[k4] *= inv;
      }

      uint32_t pf[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[m][i][e] *= qs[m][e >> 1];
            if (edge && !sees(a, w.b, min(tt[m][e >> 1], a.T - 1), pos0 + 4 * c + 2 * i + (e & 1), w.s)) sc[m][i][e] = -INFINITY;
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float top = quad_max(fmaxf(fmaxf(sc[m][0][2 * r], sc[m][0][2 * r + 1]), fmaxf(sc[m][1][2 * r], sc[m][1][2 * r + 1])));
          const float now = fmaxf(mx[m][r], top);
          if (__any_sync(0xffffffffu, now > mx[m][r])) {
            const float f = now > mx[m][r] ? exp2f(mx[m][r] - now) : 1.f;
            sum[m][r] *= f;
#pragma unroll
            for (int j = 0; j < S::NB; ++j) o[m][j][2 * r] *= f, o[m][j][2 * r + 1] *= f;
            mx[m][r] = now;
          }
          const float ref = (now == -INFINITY ? 0.f : now) - OFFSET;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float p = exp2f(sc[m][i][2 * r + e] - ref);
              sum[m][r] += p;
              if (HALVES) p = sc[m][i][2 * r + e] == -INFINITY ? 0.f : p * vs[2 * i + e];
              sc[m][i][2 * r + e] = p;
            }
        }
        pf[m][0] = pack2<HALVES>(sc[m][0][0], sc[m][0][1]);
        pf[m][1] = pack2<HALVES>(sc[m][0][2], sc[m][0][3]);
        pf[m][2] = pack2<HALVES>(sc[m][1][0], sc[m][1][1]);
        pf[m][3] = pack2<HALVES>(sc[m][1][2], sc[m][1][3]);
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
        for (int m = 0; m < MT; ++m) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) wild[(g + 8 * (e >> 1)) * CA_TILE + 4 * c + 2 * i + (e & 1)] = sc[m][i][e];
          __syncwarp();
#pragma unroll 1
          for (int tok = 0; tok < CA_TILE; ++tok) {
            const float p0 = wild[g * CA_TILE + tok], p1 = wild[(g + 8) * CA_TILE + tok];
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = HALVES ? (2 * c + e) * S::NB + j : j * 8 + 2 * c + e;
                const uint8_t* at = vt + chunk_at<S::CPR>(tok, d * S::ES / 16) + (d * S::ES) % 16;
                float v;
                if (KIND == CA_BF16) v = __bfloat162float(*(const bf16*)at);
                else {
                  const uint32_t hv = half2_of<CA_E4M3>(*at);
                  v = __half2float(__ushort_as_half((unsigned short)hv));
                }
                if (p0 != 0.f) o[m][j][e] += p0 * v;
                if (p1 != 0.f) o[m][j][2 + e] += p1 * v;
              }
          }
        }
      } else if (!HALVES) {
        const uint32_t va = ca_smem(vt) + vtok * S::ROW;
        const int x = (lane >> 4) ^ ((((vtok >> 2) << 1) | (vtok & 1)) & 7);
#pragma unroll
        for (int j = 0; j < S::NB; j += 2) {
          uint32_t vf[4];
          ldsm4_t(va + ((j ^ x) << 4), vf);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<HALVES>(o[m][j], pf[m], vf[0], vf[1]);
            mma16816<HALVES>(o[m][j + 1], pf[m], vf[2], vf[3]);
          }
        }
      } else {
        // lane (g, c): columns g NB .. g NB + NB - 1 of tokens 4c .. 4c + 3; block j takes column j of each g
        uint32_t vw[4][S::NB / 4];
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          if (D == 128) {
            const uint4 v = *(const uint4*)(vt + chunk_at<S::CPR>(vtok + t4, g));
            vw[t4][0] = v.x, vw[t4][1] = v.y, vw[t4][S::NB / 4 - 2] = v.z, vw[t4][S::NB / 4 - 1] = v.w;
          } else {
            const uint2 v = *(const uint2*)(vt + chunk_at<S::CPR>(vtok + t4, g >> 1) + (g & 1) * 8);
            vw[t4][0] = v.x, vw[t4][1] = v.y;
          }
        }
#pragma unroll
        for (int q = 0; q < S::NB / 4; ++q) {
          uint32_t b0[4], b1[4];
          pairs_of<KIND>(vw[0][q], vw[1][q], b0);
          pairs_of<KIND>(vw[2][q], vw[3][q], b1);
#pragma unroll
          for (int z = 0; z < 4; ++z)
#pragma unroll
            for (int m = 0; m < MT; ++m) mma16816<HALVES>(o[m][q * 4 + z], pf[m], b0[z], b1[z]);
        }
      }
      __syncwarp();
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    }

    // join the warps: rows of one maximum, then O through the stage that is free
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sum[m][r] = quad_sum(sum[m][r]);
        if (c == 0) *(float2*)(ml + ((warp * S::ROWS) + m * 16 + r * 8 + g) * 2) = make_float2(mx[m][r], sum[m][r]);
      }
    __syncthreads();
    const bool whole = w.head == 0 && w.end == w.nt;
    const int slot = slot_of(blockIdx.x, w.head > 0);
    float* part = a.part_o + (long)slot * S::ROWS * D;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float f[2], norm[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = -INFINITY, all = 0.f;
#pragma unroll
        for (int v = 0; v < CA_WARPS; ++v) top = fmaxf(top, ml[(v * S::ROWS + m * 16 + r * 8 + g) * 2]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int v = 0; v < CA_WARPS; ++v) {
          const float2 y = *(const float2*)(ml + (v * S::ROWS + m * 16 + r * 8 + g) * 2);
          all += y.y * exp2f(y.x - ref);
        }
        f[r] = exp2f(mx[m][r] - ref) * (HALVES ? unit_v : 1.f);
        norm[r] = all > 0.f || all != all ? 1.f / all : 0.f;   // a row that sees nothing: zeros
        if (!whole && warp == 0 && c == 0)
          *(float2*)(a.part_ml + ((long)slot * S::ROWS + m * 16 + r * 8 + g) * 2) = make_float2(top, all);
      }
      const int free_stage = stage == 0 ? S::STAGES - 1 : stage - 1;
#pragma unroll
      for (int j0 = 0; j0 < S::NB; j0 += S::NBP) {
        if (m || j0) __syncthreads();
        float4* mine = (float4*)(ring + free_stage * S::STAGE);
#pragma unroll
        for (int j = 0; j < S::NBP; ++j)
          mine[j * 32 + lane] = make_float4(o[m][j0 + j][0] * f[0], o[m][j0 + j][1] * f[0], o[m][j0 + j][2] * f[1], o[m][j0 + j][3] * f[1]);
        if (lane == 0) scratch[36 + warp] = free_stage;
        __syncthreads();
#pragma unroll
        for (int jj = 0; jj < S::NBP / CA_WARPS; ++jj) {
          const int j = warp * (S::NBP / CA_WARPS) + jj;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int v = 0; v < CA_WARPS; ++v) {
            const float4 z = ((const float4*)(smem + v * S::RING + scratch[36 + v] * S::STAGE))[j * 32 + lane];
            y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
          }
          if (!whole) {
            ((float4*)part)[(m * S::NB + j0 + j) * 32 + lane] = y;
          } else {
            const float yy[4] = {y.x * norm[0], y.y * norm[0], y.z * norm[1], y.w * norm[1]};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int t = tt[m][r];
              if (t >= a.T) continue;
              const bool live = t < w.s.count;
              const int row = row0 + m * 16 + r * 8 + g;
              bf16* op = a.out + (((long)w.b * a.T + t) * a.Hq + h * a.G + row - t * a.G) * D;
              const float y0 = live ? yy[2 * r] : 0.f, y1 = live ? yy[2 * r + 1] : 0.f;
              if (!HALVES) *(uint32_t*)(op + (j0 + j) * 8 + 2 * c) = pack2<false>(y0, y1);
              else {
                op[(2 * c) * S::NB + j0 + j] = __float2bfloat16(y0);
                op[(2 * c + 1) * S::NB + j0 + j] = __float2bfloat16(y1);
              }
            }
          }
        }
      }
    }
    __syncthreads();   // the stages and ml are free again
    if (!walk_next(a, w, warp)) break;
  }
  ca_wait<0>();
}

// Joins the parts of the units that the deal has cut, and writes the rows of sequences that see nothing. Block (unit, 16 rows); its
// warps share the parts, then the columns.
constexpr int CJ_WARPS = 8;
template <int D, bool HALVES, int MT>
__global__ void __launch_bounds__(CJ_WARPS * 32) cache_attn_join_kernel(const CacheAttnArgs a) {
  constexpr int NB = D / 8, ROWS = 16 * MT, JB = 4;   // blocks of columns of a thread block
  __shared__ float4 buf[CJ_WARPS][JB][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int unit = blockIdx.x, m = blockIdx.y % MT, j0 = blockIdx.y / MT * JB;
  const int units = a.Hkv * a.row_tiles;
  const int b = unit / units, hr = unit - b * units;
  const SeqLen s = seq_len(a, b);
  const int nt = (s.len + CA_TILE - 1) / CA_TILE;
  const int per = a.plan[0], first = a.plan[1 + b] + hr * nt;
  const int c0 = nt ? first / per : 0, c1 = nt ? (first + nt - 1) / per : -1;
  if (c0 == c1) return;                                // whole: written already
  float4 y[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  float top[2] = {-INFINITY, -INFINITY}, all[2] = {0.f, 0.f};
  for (int k = c0; k <= c1; ++k)
#pragma unroll
    for (int r = 0; r < 2; ++r) top[r] = fmaxf(top[r], a.part_ml[((long)slot_of(k, k > c0) * ROWS + m * 16 + r * 8 + g) * 2]);
  const float ref[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
  for (int k = c0; k <= c1; ++k) {
    const long slot = slot_of(k, k > c0);
    float f[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 z = *(const float2*)(a.part_ml + (slot * ROWS + m * 16 + r * 8 + g) * 2);
      f[r] = exp2f(z.x - ref[r]);
      all[r] += z.y * f[r];
    }
    if ((k - c0) % CJ_WARPS == warp) {
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        const float4 z = ((const float4*)(a.part_o + slot * ROWS * D))[(m * NB + j0 + j) * 32 + lane];
        y[j].x += z.x * f[0], y[j].y += z.y * f[0], y[j].z += z.z * f[1], y[j].w += z.w * f[1];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < JB; ++j) buf[warp][j][lane] = y[j];
  __syncthreads();
  if (warp >= JB) return;
  float4 z = buf[0][warp][lane];
#pragma unroll
  for (int v = 1; v < CJ_WARPS; ++v) {
    const float4 x = buf[v][warp][lane];
    z.x += x.x, z.y += x.y, z.z += x.z, z.w += x.w;
  }
  const float zz[4] = {z.x, z.y, z.z, z.w};
  const int h = hr / a.row_tiles, row0 = (hr - h * a.row_tiles) * ROWS, j = j0 + warp;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + m * 16 + r * 8 + g, t = row / a.G;
    if (t >= a.T) continue;
    const float norm = t < s.count && (all[r] > 0.f || all[r] != all[r]) ? 1.f / all[r] : 0.f;
    const bool live = t < s.count;
    bf16* op = a.out + (((long)b * a.T + t) * a.Hq + h * a.G + row - t * a.G) * D;
    const float y0 = live ? zz[2 * r] * norm : 0.f, y1 = live ? zz[2 * r + 1] * norm : 0.f;
    if (!HALVES) *(uint32_t*)(op + j * 8 + 2 * c) = pack2<false>(y0, y1);
    else {
      op[(2 * c) * NB + j] = __float2bfloat16(y0);
      op[(2 * c + 1) * NB + j] = __float2bfloat16(y1);
    }
  }
}

template <int D, int KIND, int MT>
static int cache_attn_launch(const CacheAttnArgs& a, cudaStream_t st) {
  using S = CaShape<D, KIND, MT>;
  static std::atomic<uint64_t> done{0};
  if (int r = smem_opt_in(done, cache_attn_kernel<D, KIND, MT>, S::SMEM)) return r;
  cache_attn_kernel<D, KIND, MT><<<a.grid, CA_THREADS, S::SMEM, st>>>(a);
  TB_CUDA_CHECK(cudaGetLastError());
  const dim3 grid((unsigned)(a.B * a.Hkv * a.row_tiles), (unsigned)(MT * (S::NB / 4)));
  cache_attn_join_kernel<D, S::HALVES, MT><<<grid, CJ_WARPS * 32, 0, st>>>(a);
  TB_CUDA_CHECK(cudaGetLastError());
  return 0;
}

template <int D, int KIND>
static int cache_attn_rows(const CacheAttnArgs& a, int mt, cudaStream_t st) {
  return mt == 1 ? cache_attn_launch<D, KIND, 1>(a, st) : cache_attn_launch<D, KIND, 2>(a, st);
}

template <int D>
static int cache_attn_kind(const CacheAttnArgs& a, int kind, int mt, cudaStream_t st) {
  if (kind == CA_BF16) return cache_attn_rows<D, CA_BF16>(a, mt, st);
  if (kind == CA_INT8) return cache_attn_rows<D, CA_INT8>(a, mt, st);
  return cache_attn_rows<D, CA_E4M3>(a, mt, st);
}

static int ca_grid() { return 2 * sm_count(); }

}  // namespace tb
using namespace tb;

int tb_set_check_word_cache_attention(int* word) {
  TB_CUDA_CHECK(set_check_word_this_tu(word));
  return 0;
}

// Bytes of workspace that tb_cache_attention needs for these sizes.
TB_EXPORT long tb_cache_attention_workspace(int B, int T, int Hq, int Hkv, int D) {
  if (ensure_device() || Hkv <= 0) return -1;
  const int rows = (long)T * (Hq / Hkv) <= 16 ? 16 : 32;
  const long slots = 2l * ca_grid();
  return slots * rows * D * 4 + slots * rows * 8 + ((long)B + 1) * 4 + 256;
}

// q [B, T, Hq, D] bf16 (strides in elements, multiples of 8; 16-byte aligned), out contiguous. ws: tb_cache_attention_workspace() bytes,
// 16-byte aligned, used by this call alone.
TB_EXPORT int tb_cache_attention(const void* q, const long* q_strides, const void* k_pages, const void* v_pages, const float* k_scales,
                                 const float* v_scales, const int* table, long table_ld, const int* start, const int* counts,
                                 const uint8_t* mask, long mask_b, long mask_t, void* out, void* ws, int B, int T, int Hq, int Hkv,
                                 int D, int page, int pages_per_seq, int num_pages, int max_len, int kind, float scale, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  if (B <= 0 || T <= 0 || Hq <= 0) return 0;
  if (!q || !out || !ws || !k_pages || !v_pages || !table || !start || (kind != CA_BF16 && (!k_scales || !v_scales)))
    TB_FAIL(TB_E_ARG, "cache attention: null pointer");
  if (D != 64 && D != 128) TB_FAIL(TB_E_ARG, "cache attention: head dim 64 or 128");
  if (Hkv <= 0 || Hq % Hkv || kind < 0 || kind > 2) TB_FAIL(TB_E_ARG, "cache attention: query heads must be a multiple of the cache's");
  if (page <= 0 || page % CA_TILE || num_pages < 0 || pages_per_seq < 0 || max_len < 0) TB_FAIL(TB_E_ARG, "cache attention: pages of a multiple of %d tokens", CA_TILE);
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)ws | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15 || q_strides[0] % 8 || q_strides[1] % 8 || q_strides[2] % 8)
    TB_FAIL(TB_E_ARG, "cache attention: 16-byte aligned rows");
  if (kind != CA_BF16 && (((uintptr_t)k_scales | (uintptr_t)v_scales) & 15)) TB_FAIL(TB_E_ARG, "cache attention: 16-byte aligned scales");
  CacheAttnArgs a{};
  a.q = (const bf16*)q, a.qb = q_strides[0], a.qt = q_strides[1], a.qh = q_strides[2];
  a.k_pages = k_pages, a.v_pages = v_pages, a.k_scales = k_scales, a.v_scales = v_scales;
  a.table = table, a.table_ld = table_ld, a.start = start, a.counts = counts;
  a.mask = mask, a.mask_b = mask_b, a.mask_t = mask_t, a.out = (bf16*)out;
  a.B = B, a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.page = page, a.num_pages = num_pages;
  a.scale_log2 = scale * 1.4426950408889634f;
  const long rows = (long)T * a.G;
  const int mt = rows <= 16 ? 1 : 2;
  a.row_tiles = (int)((rows + 16 * mt - 1) / (16 * mt));
  a.grid = ca_grid();
  const long held = (long)pages_per_seq * page;
  a.limit = (int)(held < max_len ? held : max_len);
  const long tiles = ((long)a.limit + CA_TILE - 1) / CA_TILE * B * Hkv * a.row_tiles;
  if (rows > 0x7fffff00l || tiles > 0x7fff0000l || a.limit > 0x7fff0000l || (long)B * Hkv * a.row_tiles > 0x7fff0000l)
    TB_FAIL(TB_E_TOO_LARGE, "cache attention: too much for one call");
  const long slots = 2l * a.grid;
  a.part_o = (float*)ws;
  a.part_ml = a.part_o + slots * 16 * mt * D;
  a.plan = (int*)(a.part_ml + slots * 16 * mt * 2);
  return D == 64 ? cache_attn_kind<64>(a, kind, mt, st) : cache_attn_kind<128>(a, kind, mt, st);
}
