// Rotary positions with explicit positions and a frequency table, forward and backward, q and k in one launch (sm_100a).
//
//   pair (a, b) at position p, pair index i:   y_a = m (a cos t - b sin t),  y_b = m (a sin t + b cos t),  t = p * freqs[i]
//
// over the first R of D columns; pairs are (2i, 2i+1) or (i, i + R/2), columns from R on pass through. The backward pass is
// the same map with sin negated. Position and frequency meet in 64 bits: p * f / 2pi is reduced to a fraction of a turn
// before it is rounded to fp32 (p * f rounded to fp32 first is off by 0.06 rad at p = 10^6), then sincospif.
//
// Bound by memory: x is read and y written once. The angles of a token are worked out once per block into shared memory and
// stay in a thread's registers while it walks down the heads: R/2 sine/cosine pairs for every (Hq + Hk) D elements.
#include "common.cuh"
#include "host_util.h"

namespace tb {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_PAIRS = 256;   // R <= 512
constexpr int ROT_TOKENS = 2;        // tokens of a block

struct RotaryArgs {
  const void* x[2];      // q, k: [tokens, heads, D] with strides
  void* y[2];            // contiguous
  long ld[2], lh[2];     // elements between tokens, between heads
  int heads[2];
  const long* pos;
  const double* freqs;
  long tokens;
  int D, R, splits;      // splits: blocks that share a token's heads
  float magnitude, sign;
};

__device__ __forceinline__ void rot_angles(const RotaryArgs& a, long t0, int n, float2* tab) {
  const int half = a.R >> 1;
  for (int i = threadIdx.x; i < n * half; i += ROT_THREADS) {
    const int t = i / half, p = i - t * half;
    const double turns = (double)a.pos[t0 + t] * (a.freqs[p] * 0.15915494309189533577);
    const float frac = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.f * frac, &s, &c);
    tab[t * half + p] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
}

// VEC: 16-byte vectors. A thread owns one column position of a row (item) and walks down the heads.
template <typename T, bool HALF>
__global__ void __launch_bounds__(ROT_THREADS) rotary_vec_kernel(const RotaryArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int U = HALF ? 2 : 4;      // heads in flight
  __shared__ float2 tab[ROT_TOKENS * ROT_MAX_PAIRS];
  const int half = a.R >> 1, D = a.D;
  const long t0 = (long)blockIdx.x * ROT_TOKENS;
  const int nt = (int)min((long)ROT_TOKENS, a.tokens - t0);
  // items of a head row. HALF: vectors of the first halves (with their partners), then the vectors that pass through
  const int turned = HALF ? half / N : (a.R + N - 1) / N;
  const int items = HALF ? turned + (D - a.R) / N : D / N;
  const int rows = ROT_THREADS / items;
  const int it = threadIdx.x % items, row = threadIdx.x / items;
  rot_angles(a, t0, nt, tab);
  __syncthreads();
  if (row >= rows) return;
  const int total = a.heads[0] + a.heads[1];
  const bool turn = it < turned;
  const int c0 = HALF ? (turn ? it * N : a.R + (it - turned) * N) : it * N;
  for (int t = 0; t < nt; ++t) {
    float2 cs[HALF ? N : N / 2];
    if (turn) {
#pragma unroll
      for (int j = 0; j < (HALF ? N : N / 2); ++j) {
        const int p = HALF ? c0 + j : (c0 >> 1) + j;
        cs[j] = p < half ? tab[t * half + p] : make_float2(1.f, 0.f);
      }
    }
    for (int h0 = blockIdx.y * rows + row; h0 < total; h0 += U * rows * a.splits) {
      Vec16<T> u[U], w[U];
      T* dst[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int h = h0 + i * rows * a.splits;
        if (h < total) {
          const int z = h >= a.heads[0];
          const int hh = h - (z ? a.heads[0] : 0);
          const T* src = (const T*)(z ? a.x[1] : a.x[0]) + (t0 + t) * (z ? a.ld[1] : a.ld[0]) + hh * (z ? a.lh[1] : a.lh[0]) + c0;
          dst[i] = (T*)(z ? a.y[1] : a.y[0]) + ((t0 + t) * (z ? a.heads[1] : a.heads[0]) + hh) * D + c0;
          u[i].load_nc(src);
          if (HALF && turn) w[i].load_nc(src + half);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (h0 + i * rows * a.splits < total) {
          if (turn) {
            float f[N];
            u[i].get(f);
            if (HALF) {
              float g[N];
              w[i].get(g);
#pragma unroll
              for (int j = 0; j < N; ++j) {
                const float x = f[j], y = g[j];
                f[j] = x * cs[j].x - y * cs[j].y;
                g[j] = x * cs[j].y + y * cs[j].x;
              }
              w[i].set(g);
              w[i].store(dst[i] + half);
            } else {
#pragma unroll
              for (int j = 0; j < N / 2; ++j) {
                const float x = f[2 * j], y = f[2 * j + 1];
                f[2 * j] = x * cs[j].x - y * cs[j].y;
                f[2 * j + 1] = x * cs[j].y + y * cs[j].x;
              }
            }
            u[i].set(f);
          }
          u[i].store(dst[i]);
        }
      }
    }
  }
}

// Head sizes, pairings and addresses that 16-byte vectors do not fit: one pair (or one column that passes through) at a time.
template <typename T, bool HALF>
__global__ void __launch_bounds__(ROT_THREADS) rotary_scalar_kernel(const RotaryArgs a) {
  __shared__ float2 tab[ROT_TOKENS * ROT_MAX_PAIRS];
  const int half = a.R >> 1, D = a.D;
  const long t0 = (long)blockIdx.x * ROT_TOKENS;
  const int nt = (int)min((long)ROT_TOKENS, a.tokens - t0);
  rot_angles(a, t0, nt, tab);
  __syncthreads();
  const int items = half + D - a.R, total = a.heads[0] + a.heads[1];
  for (int t = 0; t < nt; ++t)
    for (long i = (long)blockIdx.y * ROT_THREADS + threadIdx.x; i < (long)total * items; i += (long)a.splits * ROT_THREADS) {
      const int h = (int)(i / items), it = (int)(i - (long)h * items);
      const int z = h >= a.heads[0];
      const int hh = h - (z ? a.heads[0] : 0);
      const T* src = (const T*)(z ? a.x[1] : a.x[0]) + (t0 + t) * (z ? a.ld[1] : a.ld[0]) + hh * (z ? a.lh[1] : a.lh[0]);
      T* dst = (T*)(z ? a.y[1] : a.y[0]) + ((t0 + t) * (z ? a.heads[1] : a.heads[0]) + hh) * D;
      if (it < half) {
        const int ca = HALF ? it : 2 * it, cb = HALF ? it + half : 2 * it + 1;
        const float2 cs = tab[t * half + it];
        const float x = to_f<T>(src[ca]), y = to_f<T>(src[cb]);
        dst[ca] = from_f<T>(x * cs.x - y * cs.y);
        dst[cb] = from_f<T>(x * cs.y + y * cs.x);
      } else {
        const int c = a.R + it - half;
        dst[c] = src[c];
      }
    }
}

template <typename T>
static int rotary_launch(const RotaryArgs& a, bool half, bool vec, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.tokens, ROT_TOKENS), (unsigned)a.splits);
  if (vec && half) rotary_vec_kernel<T, true><<<grid, ROT_THREADS, 0, st>>>(a);
  else if (vec) rotary_vec_kernel<T, false><<<grid, ROT_THREADS, 0, st>>>(a);
  else if (half) rotary_scalar_kernel<T, true><<<grid, ROT_THREADS, 0, st>>>(a);
  else rotary_scalar_kernel<T, false><<<grid, ROT_THREADS, 0, st>>>(a);
  TB_CUDA_CHECK(cudaGetLastError());
  return 0;
}

}  // namespace tb
using namespace tb;

// q [tokens, hq, D], k [tokens, hk, D] (hk = 0: none) with strides in elements, columns contiguous; yq, yk contiguous.
struct RotaryCall {
  const void *q, *k;
  void *yq, *yk;
  const long* pos;
  const double* freqs;
  long tokens, hq, hk, D, R, ldq, lhq, ldk, lhk, half, inverse, dtype;
  double magnitude;
};
TB_EXPORT int tb_rotary(const RotaryCall* c, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  const void *q = c->q, *k = c->k;
  void *yq = c->yq, *yk = c->yk;
  const long tokens = c->tokens, ldq = c->ldq, lhq = c->lhq, ldk = c->ldk, lhk = c->lhk;
  if (tokens <= 0 || c->hq + c->hk <= 0 || c->D == 0) return 0;
  if (c->R < 0 || c->R % 2 || c->R > c->D || c->R > 2 * ROT_MAX_PAIRS) TB_FAIL(TB_E_ARG, "rotary: %ld turned columns of %ld (even, at most %d)", c->R, c->D, 2 * ROT_MAX_PAIRS);
  if (!q || !yq || (c->hk > 0 && (!k || !yk)) || !c->pos || (c->R > 0 && !c->freqs)) TB_FAIL(TB_E_ARG, "rotary: null pointer");
  if (c->hq < 0 || c->hk < 0 || c->hq + c->hk > 0x7fffffff / 2 || c->D > 0x7fffffff / 2 || tokens > 0xfffffff0l) TB_FAIL(TB_E_TOO_LARGE, "rotary: too many tokens or heads");
  if (c->dtype != 0 && c->dtype != 1) TB_FAIL(TB_E_ARG, "rotary: bf16 or fp32");
  const int hq = (int)c->hq, hk = (int)c->hk, D = (int)c->D, R = (int)c->R, dtype = (int)c->dtype;
  const bool half = c->half != 0;
  const int N = dtype == 0 ? 8 : 4;
  bool vec = D % N == 0 && D / N <= ROT_THREADS && (!half || (R / 2) % N == 0);
  const uintptr_t at = (uintptr_t)q | (uintptr_t)yq | (hk ? (uintptr_t)k | (uintptr_t)yk : 0);
  vec = vec && at % 16 == 0 && ldq % N == 0 && lhq % N == 0 && (!hk || (ldk % N == 0 && lhk % N == 0));
  RotaryArgs a{{q, k}, {yq, yk}, {ldq, ldk}, {lhq, lhk}, {hq, hk}, c->pos, c->freqs, tokens, D, R, 1, (float)c->magnitude, c->inverse ? -1.f : 1.f};
  // few tokens: several blocks share a token's heads, until each SM has two blocks or a block has one pass of its threads
  const long blocks = ceil_div(tokens, ROT_TOKENS);
  const int passes = ceil_div((long)(hq + hk) * D / (vec ? N : 2), ROT_THREADS);
  long s = 2l * sm_count() / blocks;
  a.splits = (int)(s < 1 ? 1 : s > passes ? passes : s);
  return dtype == 0 ? rotary_launch<bf16>(a, half, vec, st) : rotary_launch<float>(a, half, vec, st);
}
