// Attention over a paged cache for many rows: trees of drafted tokens whose T * G query rows share a head's keys (sm_100a, tcgen05).
//
// Same mathematics and the same deal of the work as cache_attention.cu, with 128 rows and 128 tokens to a tile: S = Q K^T and
// O += P V are tcgen05.mma products of 128 x 128 x D and 128 x D x 128 with S, P and O in TMEM. A tile's two products take 1024 clocks of
// the tensor core and its 128 x 128 exponentials 1024 of the special-function unit, whether all rows are used or not; its keys and
// values (64 KB in bf16, 33 KB in 8 bits, D = 128) take 2800 and 1450 clocks of the SM's share of HBM. So up to 128 rows cost what
// the memory takes; mma.sync at 32 rows a CTA read every token rows / 32 times through L2 and was 2.5 to 8 times slower.
//
// Measured (a call among others, L2 cold): 8 trees of 48 tokens, 32 heads of D = 128 over 4096 tokens of bf16, 549 MB: 120 to 122 us, 4.5 TB/s. A tile
// takes 2900 clocks, what the memory takes; the rest is the start (12 000 clocks until the first S: launch, deal, page table, first
// copies) and the end of a unit (11 000 from the last P to the next unit's first S, in which the ring fills and then waits). 12 trees of 27
// tokens, 32 heads over 8, ragged up to 6000 tokens of int8, 95 MB: 81 us, 33 % of the issue slots, no pipe above 23 %: warps wait for loads and for one another (a
// tile took 4300 clocks, 10 000 warp instructions, when it was 78 us with the values' scales in their halves relative to the largest of 32
// tokens, which lost what a row sees beside a larger scale that it does not see). Measured and not kept: a logarithm for each score (87),
// seven decoding warps (81 us for 75), keys' scales in the halves (82, and a rounding more), Q a unit ahead in a second place (122 for 121, 86
// for 75).
//
// One CTA per SM, 512 threads:
//   warps 0-3, 4-7  softmax, a thread per row, even tiles for the first four warps and odd ones for the others, each with a maximum, a sum
//              and an O of its own, so that the exponentials of one tile run beside the products of the other and nothing is exchanged
//              before the unit's end, where both read both O out of TMEM. They also bring Q into shared memory (8-bit caches: as halves,
//              scaled by a power of two per row)
//   warps 8-11 keys and values: 16-byte cp.async of 16-token pieces of pages (a warp has two pieces of a tile). bf16 goes straight into the
//              128-byte-swizzled tiles; 8-bit codes into a ring of their own, from where the warp that loaded them writes halves. No
//              TMA: pages of 16 tokens would be 32 copies a tile, and what lies behind a sequence's end has to become zeros
//   warp 12    issues the products (warps 13-15: none; 512 threads take no more of the SM than 416, for 128 registers each)
// TMEM: S and P of even and of odd tiles 128 columns each (P takes the first half of the S it came from), then O of either.
//
// 8-bit scales: scores are multiplied by the key's scale in fp32, and P carries the value's, v: P = 2^(x + log2 v - M + 14), M the largest
// x + log2 v that the row sees, so that halves have room for what counts in this row, whatever other scales there are (tokens that it does
// not see, or hardly attends to). The softmax's sum is that of P / v. For 32 tokens (what a loading warp has of a tile) whose scales are within
// 2^6 of one another, M takes the largest score with the largest scale; otherwise a logarithm for each score.
#include "cache_attention.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace tb {

constexpr int CT_THREADS = 512;
constexpr int CT_TILE = 128;
// Units stay whole while the longest has so many tiles more than a CTA's share. Measured (us, whole / cut): 2 trees of 27 in int8, 8 heads of
// the cache, 200 tokens (one tile more) 16.6 / 19.9, 400 (three) 21.2 / 20.1; 16 tokens of one sequence, bf16, 300 tokens (two) 16.5 / 14.2.
constexpr int CT_WHOLE = 1;
constexpr uint32_t CT_WIDE = 6;   // so many powers of two between 32 scales of values are taken for one

template <int D, int KIND> struct CtShape {
  static constexpr bool HALVES = KIND != CA_BF16;
  static constexpr int ES = HALVES ? 1 : 2;
  static constexpr int TILE = CT_TILE * D * 2;                      // Q, K or V as the products read it
  static constexpr int KST = 2, VST = HALVES ? 2 : 4;               // keys are free after S, values after O += P V, two tiles later
  static constexpr int PIECE = 16 * D * ES;                         // 16 tokens as they lie in a page
  static constexpr int RAW = HALVES ? 2 * CT_TILE * D : 0;
  static constexpr int RAWS = HALVES ? 2 : 0;
  static constexpr int Q_OFF = 0, K_OFF = TILE, V_OFF = K_OFF + KST * TILE, RAW_OFF = V_OFF + VST * TILE;
  // per value stage: scales of keys and of values, and of each loading warp's tokens log2 of the values' largest scale, and which have odd values
  static constexpr int SIDE_OFF = RAW_OFF + RAWS * RAW, SCALES = HALVES ? 2 * CT_TILE * 4 + 16 : 0, SIDE = SCALES + 16;
  static constexpr int TOP_OFF = SIDE_OFF + VST * SIDE;             // exponent of the largest |q| of either half of a row
  static constexpr int BAR_OFF = TOP_OFF + (HALVES ? 2 * CT_TILE : 0);
  // k_full[2], k_empty[2], v_full[4], v_empty[4], s_full[2], p_full[2], pv_done[2], side_full[2], q_full
  static constexpr int NBARS = 21;
  static constexpr int ALLOC = BAR_OFF + NBARS * 8 + 8;
  static_assert(ALLOC <= 232448, "one CTA per SM");
};

__device__ __forceinline__ void ct_copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ct_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ct_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Byte offset of 8 columns (16 bytes), from column 8 * chunk on, of a row in a tile of 128-byte rows, 64 columns wide, one after the other.
__device__ __forceinline__ int ct_at(int row, int chunk) { return (chunk >> 3) * 16384 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }

template <bool HALVES>
__host__ __device__ constexpr uint32_t ct_idesc(int M, int N, int b_major) {
  return HALVES ? make_idesc_bf16(M, N, 0, b_major) & ~((1u << 7) | (1u << 10)) : make_idesc_bf16(M, N, 0, b_major);   // formats: f16 0, bf16 1
}
template <bool HALVES>
__device__ __forceinline__ uint32_t ct_pack(float lo, float hi) {
  if (!HALVES) return pack_bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Infinities and NaN among the values of new tokens are zeros in the tile (0 * inf would reach rows that do not see them): here the
// rows that do see them get them, straight from the page. `words`: the tokens; O of the tile has been added.
template <int D, int KIND>
__device__ __forceinline__ void ct_odd_values(const CacheAttnArgs& a, uint32_t to, const uint32_t (&words)[4], int b, int h, int t, bool live, int pos0, const SeqLen& s) {
#pragma unroll 1
  for (int w = 0; w < 4; ++w)
#pragma unroll 1
    for (uint32_t rest = w == 0 ? words[0] : w == 1 ? words[1] : w == 2 ? words[2] : words[3]; rest; rest &= rest - 1) {
      const int pos = pos0 + w * 32 + __ffs(rest) - 1;
      const long row = row_of(a, page_ref(a, b, pos), h);
      const bool mine = live && row >= 0 && sees(a, b, t, pos, s);
      const bool wild = KIND != CA_BF16 && row >= 0 && odd_scale(__ldg(a.v_scales + row + (pos & 15)));
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_ld16(to + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v = 0.f;
          if (row >= 0) {
            const long at = (row + (pos & 15)) * D + c + i;
            if (KIND == CA_BF16) v = __bfloat162float(((const bf16*)a.v_pages)[at]);
            else if (wild || (KIND == CA_E4M3 && (((const uint8_t*)a.v_pages)[at] & 0x7f) == 0x7f)) v = __int_as_float(0x7fffffff);
          }
          const bool odd = (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
          if (mine && odd) o[i] = __float_as_uint(__uint_as_float(o[i]) + v);
        }
        tmem_st16(to + c, o);
      }
      tmem_wait_st();
    }
}

// Which of the 128 tokens from pos0 on token t sees, a bit each. Loops stay rolled here and in all that runs once a unit: what a
// launch executes for the first time comes out of L2 instruction by instruction, and unrolled it cost 6 us.
__device__ __forceinline__ void ct_visible(const CacheAttnArgs& a, int b, int t, int pos0, const SeqLen& s, uint64_t& lo, uint64_t& hi) {
  auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; };
  const int context = min(s.start, s.len) - pos0;      // so many from the first on are context, or all of them
  lo = below(context);
  hi = below(context - 64);
  const int j0 = max(pos0 - s.start, 0), j1 = min(s.len, pos0 + CT_TILE) - s.start, at0 = s.start + j0 - pos0, n = j1 - j0;
  if (n <= 0) return;
  uint64_t nlo = 0, nhi = 0;                           // new tokens j0 .. j1 - 1
  if (!a.mask) {
    nlo = below(t + 1 - j0);
    nhi = below(t + 1 - j0 - 64);
  } else {
    // the row's bytes by aligned words: each holds a byte of the mask, so each is there
    const uint8_t* m = a.mask + b * a.mask_b + t * a.mask_t + j0;
    const int off = (int)((uintptr_t)m & 3);
    const uint32_t* p = (const uint32_t*)(m - off);
#pragma unroll 8
    for (int k = 0; k * 4 < n + off; ++k) {
      const uint32_t y = __vsetne4(__ldg(p + k), 0u);
      uint64_t four = (y & 1u) | ((y >> 7) & 2u) | ((y >> 14) & 4u) | ((y >> 21) & 8u);
      int at = 4 * k - off;
      if (at < 0) four >>= -at, at = 0;
      if (at < 64) nlo |= four << at;
      if (at > 60) nhi |= at < 64 ? four >> (64 - at) : four << (at - 64);
    }
  }
  nlo &= below(n);
  nhi &= below(n - 64);
  // to their places
  if (at0 >= 64) {
    hi |= nlo << (at0 - 64);
  } else {
    lo |= nlo << at0;
    hi |= nhi << at0 | (at0 ? nlo >> (64 - at0) : 0ull);
  }
}

template <int D, int KIND>
__global__ void __launch_bounds__(CT_THREADS, 1) cache_attn_tc_kernel(const __grid_constant__ CacheAttnArgs a, int* status) {
  using L = CtShape<D, KIND>;
  constexpr bool HALVES = L::HALVES;
  constexpr int KST = L::KST, VST = L::VST, KCH = D / 64;
  constexpr uint32_t TM_S = 0, TM_O = 256;   // + 128 for odd tiles
  constexpr float OFFSET = HALVES ? 14.f : 0.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = (uint64_t*)(smem + L::BAR_OFF);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 8, *s_full = bars + 12, *p_full = bars + 14, *pv_done = bars + 16, *side_full = bars + 18, *q_full = bars + 20;
  uint32_t* tmem_ptr = (uint32_t*)(bars + L::NBARS);
  volatile int* abort_flag = (volatile int*)(tmem_ptr + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // both on their way while the deal waits for its loads
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&side_full[i], 4);
    }
    mbar_init(q_full, 256);
    *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;  // the 128-byte swizzle needs this alignment
    if (*abort_flag && status) atomicCAS(status, 0, TB_ERR_BAD_ARG);
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  // the deal uses the (not yet used) place of Q
  const Deal deal = deal_tiles<CT_THREADS, CT_TILE, 1, CT_WHOLE>(a, (int*)smem);
  release_join();
  zero_empty<D, CT_THREADS>(a);
  if (deal.first >= deal.last) {
    if (threadIdx.x == 0) a.plan[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (warp == 12) tmem_dealloc(*tmem_ptr, 512);
    return;
  }
  Walk w;
  walk_begin<CT_TILE>(a, w, deal, 0);
  if (threadIdx.x == 0) a.plan[blockIdx.x] = make_int4(w.b, w.hr, w.head, deal.per);
  const int total = deal.last - deal.first;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;

  if (warp >= 12) {
    // ---------------------------------------------------------------- products
    if (warp == 12 && elect_one()) {
      constexpr uint32_t idesc_qk = ct_idesc<HALVES>(128, 128, 0), idesc_pv = ct_idesc<HALVES>(128, D, 1);
      const uint64_t q_d = make_smem_desc_sw128(smem_u32(smem + L::Q_OFF), 16, 1024);
      const uint64_t k_d = make_smem_desc_sw128(smem_u32(smem + L::K_OFF), 16, 1024);
      const uint64_t v_d = make_smem_desc_sw128(smem_u32(smem + L::V_OFF), 16384, 1024);
      int units = 0, v = 0;      // v: the next tile whose values are due
      Walk wv = w;
      auto values = [&]() {
        const int st = v % VST, i = v & 1;
        mbar_wait(&v_full[st], (v / VST) & 1, abort_flag, status, TB_ERR_WAIT_FULL);
        mbar_wait(&p_full[i], (v >> 1) & 1, abort_flag, status, TB_ERR_WAIT_MISC);
        tc_fence_after();
        const bool first = wv.tile < wv.head + 2;      // of this O in this unit
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ts(tmem_base + TM_O + i * 128, tmem_base + TM_S + i * 128 + k * 8, desc_at(v_d, st * L::TILE + k * 2048), idesc_pv, (!first || k) ? 1u : 0u);
        umma_commit(&pv_done[i]);
        umma_commit(&v_empty[st]);
        ++v;
        if (++wv.tile >= wv.end) walk_next<CT_TILE>(a, wv, 0);
      };
      for (int n = 0; n < total; ++n) {
        const bool first = w.tile == w.head;
        // S of tile n takes the place of S and P of tile n - 2; a unit's first S needs its Q, which comes when the last unit is done with
        while (v < (first ? n : n - 1)) values();
        if (first) mbar_wait(q_full, units++ & 1, abort_flag, status, TB_ERR_WAIT_MISC);
        const int st = n % KST, i = n & 1;
        mbar_wait(&k_full[st], (n / KST) & 1, abort_flag, status, TB_ERR_WAIT_FULL);
        if (n >= 2) mbar_wait(&pv_done[i], ((n >> 1) - 1) & 1, abort_flag, status, TB_ERR_WAIT_TMEM_EMPTY);
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < KCH; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_ss(tmem_base + TM_S + i * 128, desc_at(q_d, c * 16384 + k * 32), desc_at(k_d, st * L::TILE + c * 16384 + k * 32), idesc_qk, (c | k) ? 1u : 0u);
        umma_commit(&s_full[i]);
        umma_commit(&k_empty[st]);
        if (++w.tile >= w.end) walk_next<CT_TILE>(a, w, 0);
      }
      while (v < total) values();
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- keys and values
    const int pw = warp - 8;
    const uint32_t smem_base = smem_u32(smem);
    constexpr int N = L::PIECE / 512;             // 16-byte copies of a lane for a piece of keys or values
    // of the tile last asked for: the scales of token 32 pw + lane, the first token that is a new one (CT_TILE: none), its position and its sequence's end
    float ks = 0.f, vs = 0.f;
    int first_new = CT_TILE, tile_pos = 0, seq_end = 0;
    PageRef next[2];
    auto seek = [&]() {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pos = w.tile * CT_TILE + (pw * 2 + i) * 16;
        if (pos < w.s.len) next[i] = page_ref(a, w.b, pos);
      }
    };
    // The 16-byte piece of 32 j + lane: token of 16, and piece of it. Of 128-byte rows (8 bits, D = 128) eight neighbouring lanes have four
    // pieces of two tokens, whose halves then go to all eight 16-byte places of the 128-byte swizzle; in order they met two by two.
    auto piece_of = [&](int j, int& tok, int& q) {
      if (HALVES && D == 128) {
        tok = j * 4 + ((lane >> 4) & 1) * 2 + ((lane >> 2) & 1);
        q = (lane & 3) | ((lane >> 3) & 1) << 2;
      } else {
        const int ch = j * 32 + lane;
        tok = ch / (D * L::ES / 16);
        q = ch % (D * L::ES / 16);
      }
    };
    auto raw_at = [](int tok, int q) { return tok * D + ((D == 128 ? q ^ ((tok & 1) << 2) : q) << 4); };
    auto copy = [&](const void* pages, uint32_t dst, const long (&rows)[2], int pos0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok0 = (pw * 2 + i) * 16;
        const int live = rows[i] < 0 ? 0 : min(w.s.len - pos0 - tok0, 16);
        const uint8_t* src = (const uint8_t*)pages + max(rows[i], 0l) * (D * L::ES);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          int tok, q;
          piece_of(j, tok, q);
          ct_copy16(dst + (HALVES ? raw_at(tok0 + tok, q) : ct_at(tok0 + tok, q)), src + tok * (D * L::ES) + q * 16, tok < live);
        }
      }
      ct_commit();
    };
    auto ask = [&](int n) {
      const int pos0 = w.tile * CT_TILE;
      first_new = pos0 + CT_TILE > min(w.s.start, w.s.len) ? max(w.s.start - pos0, 0) : CT_TILE;
      tile_pos = pos0, seq_end = w.s.len;
      long rows[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool there = pos0 + (pw * 2 + i) * 16 < w.s.len;
        rows[i] = there ? row_of(a, next[i], w.h) : -1;
        if (there && rows[i] < 0 && lane == 0 && !vacant_place(a.table + (long)w.b * a.table_ld, next[i].page)) report_bad_index();
      }
      if (HALVES) {
        const int pos = pos0 + pw * 32 + lane;
        const long row = lane >= 16 ? rows[1] : rows[0];
        const bool live = row >= 0 && pos < w.s.len;
        ks = live ? __ldg(a.k_scales + row + (lane & 15)) : 0.f;
        vs = live ? __ldg(a.v_scales + row + (lane & 15)) : 0.f;
        copy(a.k_pages, smem_base + L::RAW_OFF + (n & 1) * L::RAW, rows, pos0);
        copy(a.v_pages, smem_base + L::RAW_OFF + (n & 1) * L::RAW + CT_TILE * D, rows, pos0);
      } else {
        mbar_wait(&k_empty[n % KST], ((n / KST) & 1) ^ 1, abort_flag, status, TB_ERR_WAIT_EMPTY);
        copy(a.k_pages, smem_base + L::K_OFF + (n % KST) * L::TILE, rows, pos0);
        mbar_wait(&v_empty[n % VST], ((n / VST) & 1) ^ 1, abort_flag, status, TB_ERR_WAIT_EMPTY);
        copy(a.v_pages, smem_base + L::V_OFF + (n % VST) * L::TILE, rows, pos0);
      }
      if (++w.tile >= w.end) walk_next<CT_TILE>(a, w, 0);
      if (n + 1 < total) seek();
    };
    // halves of the warp's codes of a tile
    auto convert = [&](auto is_value, const uint8_t* raw, uint8_t* dst, int first_new, uint32_t& odd) {
      constexpr bool VALUE = decltype(is_value)::value;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          int tok, q;
          piece_of(j, tok, q);
          tok += (pw * 2 + i) * 16;
          uint4 v = *(const uint4*)(raw + raw_at(tok, q));
          if (VALUE && KIND == CA_E4M3 && tok >= first_new) {
            uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t nan = __vcmpeq4(x[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              x[k] &= ~nan;
              if (nan) odd |= 1u << (tok & 31);
            }
            v = make_uint4(x[0], x[1], x[2], x[3]);
          }
          uint4 lo, hi;
          halves_of<KIND>(v.x, lo.x, lo.y);
          halves_of<KIND>(v.y, lo.z, lo.w);
          halves_of<KIND>(v.z, hi.x, hi.y);
          halves_of<KIND>(v.w, hi.z, hi.w);
          *(uint4*)(dst + ct_at(tok, 2 * q)) = lo;
          *(uint4*)(dst + ct_at(tok, 2 * q + 1)) = hi;
        }
    };
    // tile n, whose copies have arrived: its halves, its odd values; then it is the products'
    auto hand_on = [&](int n, float ks, float vs, int first_new, int last_tile, int last_len) {
      const int kst = n % KST, vst = n % VST;
      uint8_t* vt = smem + L::V_OFF + vst * L::TILE;
      uint8_t* side = smem + L::SIDE_OFF + vst * L::SIDE;
      const bool edge = first_new < CT_TILE;
      uint32_t odd = 0;
      if (HALVES) {
        const uint8_t* raw = smem + L::RAW_OFF + (n & 1) * L::RAW;
        mbar_wait(&k_empty[kst], ((n / KST) & 1) ^ 1, abort_flag, status, TB_ERR_WAIT_EMPTY);
        convert(std::false_type{}, raw, smem + L::K_OFF + kst * L::TILE, 0, odd);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[kst]);
        // a scale that is no finite number leaves none among its token's values: a new token's are for the rows that see it (ct_odd_values),
        // a context's are NaN by their scale. What lies behind the end is not seen
        const bool there = last_tile + pw * 32 + lane < last_len, infinite = there && odd_scale(vs), wild = infinite && pw * 32 + lane >= first_new;
        const bool zero = wild || (there && no_scale(vs)), plain = there && !infinite && !zero;
        if (wild) odd = 1u << lane;
        const uint32_t size = __float_as_uint(vs) & 0x7fffffffu;
        const uint32_t most = __reduce_max_sync(0xffffffffu, plain ? size : 0u), least = __reduce_min_sync(0xffffffffu, plain ? size : 0xffffffffu);
        float top = most ? log2f(__uint_as_float(most)) : CA_NONE;
        if (__any_sync(0xffffffffu, zero)) top = fmaxf(top, CA_NONE);
        if (most && (most >> 23) - (least >> 23) > CT_WIDE) top = __int_as_float(0x7fffffff);
        mbar_wait(&v_empty[vst], ((n / VST) & 1) ^ 1, abort_flag, status, TB_ERR_WAIT_EMPTY);
        ((float*)side)[pw * 32 + lane] = ks;
        ((float*)side)[CT_TILE + pw * 32 + lane] = zero ? 0.f : infinite ? __int_as_float(0x7fffffff) : vs;
        if (lane == 0) ((float*)side)[2 * CT_TILE + pw] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(&side_full[vst]);                  // the softmax does not wait for the values
        convert(std::true_type{}, raw + CT_TILE * D, vt, first_new, odd);
      } else {
        if (edge) {
#pragma unroll 1
          for (int i = 0; i < 2; ++i)
#pragma unroll 1
            for (int j = 0; j < N; ++j) {
              const int ch = j * 32 + lane, tok = (pw * 2 + i) * 16 + ch / (D / 8);
              if (tok < first_new) continue;
              uint32_t* x = (uint32_t*)(vt + ct_at(tok, ch % (D / 8)));
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t v = x[k];
                const uint32_t keep = ((v & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((v & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
                if (keep != 0xffffffffu) {
                  x[k] = v & keep;
                  odd |= 1u << (tok & 31);
                }
              }
            }
        }
      }
      if (edge) odd = __reduce_or_sync(0xffffffffu, odd);
      if (lane == 0) ((uint32_t*)(side + L::SCALES))[pw] = odd;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (!HALVES) mbar_arrive(&k_full[kst]);
        mbar_arrive(&v_full[vst]);
      }
    };
    seek();
    // Tile n is asked for before tile n - 1 is handed on; what that waits for are tiles n - 2 and older.
    for (int n = 0; n <= total; ++n) {
      const float last_ks = ks, last_vs = vs;
      const int last_new = first_new, last_pos = tile_pos, last_end = seq_end;
      if (n < total) {
        ask(n);
      } else {
        ct_commit();
        ct_commit();
      }
      if (n >= 1) {
        ct_wait<2>();
        hand_on(n - 1, last_ks, last_vs, last_new, last_pos, last_end);
      }
    }
    ct_wait<0>();
  } else {
    // ---------------------------------------------------------------- softmax: a thread per row, even or odd tiles
    const int group = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_base + TM_S + group * 128 + lane_off, tp = ts, to = tmem_base + TM_O + group * 128 + lane_off;
    float2* stat = (float2*)(smem + L::Q_OFF);       // [2][128] (R, l): the place of Q once a unit's products are done
    int n = 0;                                       // the tile of the run that comes next
    while (true) {
      const int r = (w.hr - w.h * a.row_tiles) * CT_TILE + row, t = r / a.G;
      const bool live = t < w.s.count;
      const bool busy = __any_sync(0xffffffffu, live);   // a warp whose rows are all spare only keeps the others' pace
      float f = a.scale_log2;
      {
        // each group brings half of a row's columns; 8-bit caches need the whole row's largest value first
        const bf16* qp = a.q + w.b * a.qb + (long)t * a.qt + (long)(w.h * a.G + r - t * a.G) * a.qh;
        uint4 v[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) v[i] = live ? __ldg((const uint4*)qp + group * (D / 16) + i) : make_uint4(0u, 0u, 0u, 0u);
        if (HALVES) {
          float big = 0.f;
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            big = fmaxf(big, fmaxf(fmaxf(fmaxf(fabsf(bf16_lo(v[i].x)), fabsf(bf16_hi(v[i].x))), fmaxf(fabsf(bf16_lo(v[i].y)), fabsf(bf16_hi(v[i].y)))),
                                   fmaxf(fmaxf(fabsf(bf16_lo(v[i].z)), fabsf(bf16_hi(v[i].z))), fmaxf(fabsf(bf16_lo(v[i].w)), fabsf(bf16_hi(v[i].w))))));
          uint8_t* tops = smem + L::TOP_OFF;
          tops[group * 128 + row] = (uint8_t)(__float_as_uint(big) >> 23);
          asm volatile("bar.sync 1, 256;" ::: "memory");
          const uint32_t ex = max(__float_as_uint(big) >> 23, (uint32_t)tops[(group ^ 1) * 128 + row]);
          const bool plain = ex == 0 || ex > 253;
          const float down = plain ? 1.f : __uint_as_float((254u - ex) << 23);
          if (!plain) f *= __uint_as_float(ex << 23);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            v[i].x = ct_pack<true>(bf16_lo(v[i].x) * down, bf16_hi(v[i].x) * down);
            v[i].y = ct_pack<true>(bf16_lo(v[i].y) * down, bf16_hi(v[i].y) * down);
            v[i].z = ct_pack<true>(bf16_lo(v[i].z) * down, bf16_hi(v[i].z) * down);
            v[i].w = ct_pack<true>(bf16_lo(v[i].w) * down, bf16_hi(v[i].w) * down);
          }
        }
        f = fmaxf(f, 1e-30f);   // -inf (not seen) times a factor of zero would be no number
        if (!HALVES) asm volatile("bar.sync 1, 256;" ::: "memory");   // the last unit's output has left Q's place (8 bits: the barrier above)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *(uint4*)(smem + L::Q_OFF + ct_at(row, group * (D / 16) + i)) = v[i];
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      // P = 2^(x f - m f), x the score; of 8-bit caches 2^(x f - m + OFFSET) v, m the largest x f + log2 v. l sums it without v
      float m = -INFINITY, l = 0.f;
      uint32_t odd[4] = {0u, 0u, 0u, 0u};
      int odd_pos = 0;
      bool any_tile = false;
      for (; w.tile < w.end; ++w.tile, ++n) {
        if ((n & 1) != group) continue;
        const int pos0 = w.tile * CT_TILE, st = n % VST;
        const bool edge = pos0 + CT_TILE > min(w.s.start, w.s.len);
        const uint8_t* side = smem + L::SIDE_OFF + st * L::SIDE;
        uint64_t vis_lo = 0, vis_hi = 0;
        if (edge && live) ct_visible(a, w.b, t, pos0, w.s, vis_lo, vis_hi);
        if (HALVES) mbar_wait(&side_full[st], (n / VST) & 1, abort_flag, status, TB_ERR_WAIT_FULL);
        // S of this tile; O += P V of the tile before last has finished, or its place would not have been S's
        mbar_wait(&s_full[group], (n >> 1) & 1, abort_flag, status, TB_ERR_WAIT_TMEM_FULL);
        tc_fence_after();
        float alpha = 1.f;
        bool grow = false;
        const float2 f2 = make_float2(f, f);
        // Two passes over S, 64 columns at a time: the maximum, then P over the columns that have been read
        if (busy) {
          uint32_t v[2][32];
          float now = m, also = -INFINITY;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            tmem_ld32(ts + half * 64, v[0]);
            tmem_ld32(ts + half * 64 + 32, v[1]);
            tmem_wait_ld();
            if (HALVES) {
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float4 k4 = *(const float4*)(side + ((half * 2 + c) * 32 + i) * 4);
                  const float2 x = __fmul2_rn(make_float2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), make_float2(k4.x, k4.y));
                  const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3])), make_float2(k4.z, k4.w));
                  v[c][i] = __float_as_uint(x.x), v[c][i + 1] = __float_as_uint(x.y), v[c][i + 2] = __float_as_uint(y.x), v[c][i + 3] = __float_as_uint(y.y);
                }
            }
            if (edge) {
              const uint64_t seen = half ? vis_hi : vis_lo;
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(((uint32_t)(c ? seen >> 32 : seen) >> i) & 1u)) v[c][i] = 0xff800000u;
            }
            if (HALVES || edge) {   // the second pass takes them as they are now
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                tmem_st16(ts + half * 64 + c * 32, reinterpret_cast<const uint32_t(&)[16]>(v[c][0]));
                tmem_st16(ts + half * 64 + c * 32 + 16, reinterpret_cast<const uint32_t(&)[16]>(v[c][16]));
              }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (HALVES) {
                const float top = ((const float*)side)[2 * CT_TILE + half * 2 + c];
                if ((__float_as_uint(top) & 0x7fffffffu) > 0x7f800000u) {
                  const float* scales = (const float*)side + CT_TILE + (half * 2 + c) * 32;
#pragma unroll
                  for (int i = 0; i < 32; ++i) {
                    const float s = fabsf(scales[i]);
                    now = fmaxf(now, fmaf(__uint_as_float(v[c][i]), f, s == 0.f ? CA_NONE : log2f(s)));
                  }
                  continue;
                }
                also = -INFINITY;
                float here = -INFINITY;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  here = fmaxf(here, fmaxf(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])));
                  also = fmaxf(also, fmaxf(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3])));
                }
                now = fmaxf(now, fmaf(fmaxf(here, also), f, top));
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  now = fmaxf(now, fmaxf(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])));
                  also = fmaxf(also, fmaxf(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3])));
                }
              }
            }
          }
          if (!HALVES) now = fmaxf(now, also);
          if (HALVES || edge) tmem_wait_st();
          grow = now > m;
          // O of no tile yet, or of tiles that the row saw nothing of, is zero (or not there): any finite factor does
          if (grow) {
            alpha = m == -INFINITY ? 1.f : exp2f(HALVES ? m - now : (m - now) * f);
            l *= alpha;
          }
          m = now;
          const float ref = (m == -INFINITY ? 0.f : HALVES ? m : m * f) - OFFSET;
          const float2 r2 = make_float2(-ref, -ref);
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            tmem_ld32(ts + half * 64, v[0]);
            tmem_ld32(ts + half * 64 + 32, v[1]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float2 l2 = make_float2(0.f, 0.f), l3 = l2;
              uint32_t pk[16];
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float2 s01 = make_float2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), s23 = make_float2(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3]));
                const float2 x = __ffma2_rn(s01, f2, r2), y = __ffma2_rn(s23, f2, r2);
                float2 e = make_float2(exp2f(x.x), exp2f(x.y)), g = make_float2(exp2f(y.x), exp2f(y.y));
                l2 = __fadd2_rn(l2, e);
                l3 = __fadd2_rn(l3, g);
                if (HALVES) {
                  const float4 v4 = *(const float4*)(side + (CT_TILE + (half * 2 + c) * 32 + i) * 4);
                  e = __fmul2_rn(e, make_float2(v4.x, v4.y)), g = __fmul2_rn(g, make_float2(v4.z, v4.w));
                }
                pk[i / 2] = ct_pack<HALVES>(e.x, e.y);
                pk[i / 2 + 1] = ct_pack<HALVES>(g.x, g.y);
              }
              tmem_st16(tp + (half * 2 + c) * 16, pk);
              l += (l2.x + l2.y) + (l3.x + l3.y);
            }
          }
          if (odd[0] | odd[1] | odd[2] | odd[3]) ct_odd_values<D, KIND>(a, to, odd, w.b, w.h, min(t, a.T - 1), live, odd_pos, w.s);
          if (any_tile && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
            for (int c = 0; c < D; c += 64) {
              uint32_t o[4][16];
#pragma unroll
              for (int g = 0; g < 4; ++g) tmem_ld16(to + c + g * 16, o[g]);
              tmem_wait_ld();
#pragma unroll
              for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[g][i] = __float_as_uint(__uint_as_float(o[g][i]) * alpha);
                tmem_st16(to + c + g * 16, o[g]);
              }
            }
          }
        }
        if (edge) mbar_wait(&v_full[st], (n / VST) & 1, abort_flag, status, TB_ERR_WAIT_FULL);
#pragma unroll
        for (int i = 0; i < 4; ++i) odd[i] = edge ? ((const uint32_t*)(side + L::SCALES))[i] : 0u;
        odd_pos = pos0;
        any_tile = true;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[group]);
      }
      // the unit's end: the run's tiles up to n - 1 are done with, this group's last is n - 1 or n - 2
      if (any_tile) {
        const int mine = (n - 1) & 1 ? (group ? n - 1 : n - 2) : (group ? n - 2 : n - 1);
        mbar_wait(&pv_done[group], (mine >> 1) & 1, abort_flag, status, TB_ERR_WAIT_TMEM_FULL);
        tc_fence_after();
        if (busy && (odd[0] | odd[1] | odd[2] | odd[3])) {
          ct_odd_values<D, KIND>(a, to, odd, w.b, w.h, min(t, a.T - 1), live, odd_pos, w.s);
        }
      }
      const float mine_r = HALVES || m == -INFINITY ? m : m * f;
      // all products of the unit have read Q when both groups are here
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      stat[group * 128 + row] = make_float2(mine_r, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      tc_fence_after();
      const float2 other = stat[(group ^ 1) * 128 + row];
      const float top = fmaxf(mine_r, other.x), ref = top == -INFINITY ? 0.f : top;
      const float f_mine = exp2f(mine_r - ref), f_other = exp2f(other.x - ref);
      const float all = l * f_mine + other.y * f_other;
      // a group that has had no tile, or whose tiles the row saw nothing of, has nothing in its O
      const float f0 = group ? f_other : f_mine, f1 = group ? f_mine : f_other;
      const bool has0 = (group ? other.y : l) != 0.f, has1 = (group ? l : other.y) != 0.f;
      asm volatile("bar.sync 1, 256;" ::: "memory");   // read, before the next Q overwrites it
      const bool whole = w.head == 0 && w.end == w.nt;
      const int slot = slot_of(blockIdx.x, w.head > 0);
      const float inv = all > 0.f || all != all ? 1.f / all : 0.f;   // a row that sees nothing: zeros
      const long at = (long)slot * a.part_rows + row;
      if (!whole && row < a.part_rows && group == 0) *(float2*)(a.part_ml + at * 2) = make_float2(top, all);
      // this group's half of the columns, COLS at a time: through shared memory (Q's place), so that four lanes store 64 bytes of a row
      constexpr int COLS = D / 4, BLOCKS = COLS / 16;
      const uint32_t to0 = tmem_base + TM_O + lane_off;
      float4* turn = (float4*)(smem + L::Q_OFF) + warp * 128 * BLOCKS;
#pragma unroll 1
      for (int c = group * (D / 2); c < (group + 1) * (D / 2); c += COLS) {
        if (busy) {
          uint32_t o0[BLOCKS][16], o1[BLOCKS][16];
#pragma unroll
          for (int k = 0; k < BLOCKS; ++k) {
            tmem_ld16(to0 + c + k * 16, o0[k]);
            tmem_ld16(to0 + 128 + c + k * 16, o1[k]);
          }
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int k = 0; k < BLOCKS; ++k) {
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              y[i] = (has0 ? __uint_as_float(o0[k][i]) * f0 : 0.f) + (has1 ? __uint_as_float(o1[k][i]) * f1 : 0.f);
              y[i] = live ? (whole ? y[i] * inv : y[i]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) turn[k * 128 + lane * 4 + (i ^ ((lane >> 1) & 3))] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rl = i * 8 + (lane >> 2), rr = (warp & 3) * 32 + rl, piece = lane & 3, at4 = rl * 4 + (piece ^ ((rl >> 1) & 3));
          if (!whole) {
            if (rr < a.part_rows) {
              float* part = a.part_o + ((long)slot * a.part_rows + rr) * D + c + piece * 4;
#pragma unroll
              for (int k = 0; k < BLOCKS; ++k) *(float4*)(part + k * 16) = busy ? turn[k * 128 + at4] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          } else {
            const int r2 = (w.hr - w.h * a.row_tiles) * CT_TILE + rr, t2 = r2 / a.G;
            if (t2 < a.T) {
              bf16* op = a.out + (((long)w.b * a.T + t2) * a.Hq + w.h * a.G + r2 - t2 * a.G) * D + c + piece * 4;
#pragma unroll
              for (int k = 0; k < BLOCKS; ++k) {
                const float4 z = busy ? turn[k * 128 + at4] : make_float4(0.f, 0.f, 0.f, 0.f);
                *(uint2*)(op + k * 16) = make_uint2(pack_bf16x2(z.x, z.y), pack_bf16x2(z.z, z.w));
              }
            }
          }
        }
      }
      __syncwarp();
      tc_fence_before();
      if (!walk_next<CT_TILE>(a, w, 0)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, int KIND>
static int cache_attn_tc_launch(CacheAttnArgs& a, int* status, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (int r = smem_opt_in(done, cache_attn_tc_kernel<D, KIND>, CtShape<D, KIND>::ALLOC)) return r;
  cache_attn_tc_kernel<D, KIND><<<a.grid, CT_THREADS, CtShape<D, KIND>::ALLOC, st>>>(a, status);
  TB_CUDA_CHECK(cudaGetLastError());
  return cache_attn_join(a, D, CT_TILE, CT_WHOLE + 1, st);
}

int cache_attn_tc(CacheAttnArgs& a, int D, int kind, int* status, cudaStream_t st) {
  a.grid = sm_count();
  if ((long)a.B * a.Hkv * a.row_tiles > a.grid) a.before = nullptr;
  if (D == 64) {
    if (kind == CA_BF16) return cache_attn_tc_launch<64, CA_BF16>(a, status, st);
    return kind == CA_INT8 ? cache_attn_tc_launch<64, CA_INT8>(a, status, st) : cache_attn_tc_launch<64, CA_E4M3>(a, status, st);
  }
  if (kind == CA_BF16) return cache_attn_tc_launch<128, CA_BF16>(a, status, st);
  return kind == CA_INT8 ? cache_attn_tc_launch<128, CA_INT8>(a, status, st) : cache_attn_tc_launch<128, CA_E4M3>(a, status, st);
}

}  // namespace tb

int tb_set_check_word_cache_attention_tc(int* word) {
  TB_CUDA_CHECK(tb::set_check_word_this_tu(word));
  return 0;
}
