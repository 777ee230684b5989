// Rotary positions with explicit positions and a frequency table, forward and backward, q and k in one launch (sm_100a).
//
//   pair (a, b) at position p, pair index i:   y_a = m (a cos t - b sin t),  y_b = m (a sin t + b cos t),  t = p * freqs[i]
//
// over the first R of D columns; pairs are (2i, 2i+1) or (i, i + R/2), columns from R on pass through. The backward pass is
// the same map with sin negated. Position and frequency meet in 64 bits: p * f / 2pi is reduced to a fraction of a turn
// before it is rounded to fp32 (p * f rounded to fp32 first is off by 0.06 rad at p = 10^6), then sincospif: the fraction's
// rounding (1e-7 radians) and that of sincospif are what fp32 rows show, 4.8e-8 of a row's size where angles in 64 bits leave 3.5e-8. Turning by what the
// fraction drops as well takes 21.4 us for 19.8 in the second case below.
//
// Bound by memory: x is read and y written once. The angles of a token are worked out once per block into shared memory:
// R/2 sine/cosine pairs for every (Hq + Hk) D elements, while the block's loads are on their way. Measured, forward and backward: 8192
// tokens of 64 heads of 128 in bf16, 537 MB: 92 us, 5.8 TB/s; 4593 tokens of 20 heads of 64 in fp32, half of each turned, 94 MB: 20 us. What is
// issued for a row counts (0.78 instructions a clock of each scheduler when it took 98): a vector turns or passes through as a whole,
// addresses are offsets from the block's first token. Sines kept in registers from row to row (a branch a row): 100; twice the rows in
// flight: 110.
#include "common.cuh"
#include "decode_calls.h"
#include "host_util.h"

namespace tb {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_PAIRS = 256;   // R <= 512
constexpr int ROT_MAX_TOKENS = 8;    // tokens of a block
constexpr int ROT_ANGLES = 1024;     // pairs of a block, over its tokens: the places of its table

struct RotaryArgs {
  const void* x[2];      // q, k: [tokens, heads, D] with strides
  void* y[2];            // contiguous
  long ld[2], lh[2];     // elements between tokens, between heads
  int heads[2];
  const long* pos;
  const double* freqs;
  long tokens;
  int D, R, per_block;   // per_block: tokens of a block
  FastDiv by_heads;
  float magnitude, sign;
};

// Cosines and sines of the block's tokens. A thread of the vector kernel needs K neighbouring pairs: pair K i + j lies at place j G + i of
// its token, so that neighbouring threads read neighbouring words (in order they met four by four in a bank).
struct RotTable {
  int K, G;
  __device__ __forceinline__ int stride() const { return K * G; }
  __device__ __forceinline__ int at(int i, int j) const { return j * G + i; }
};
__device__ __forceinline__ void rot_angles(const RotaryArgs& a, long t0, int n, const RotTable& k, float2* tab) {
  const int half = a.R >> 1;
  for (int i = threadIdx.x; i < n * half; i += ROT_THREADS) {
    const int t = i / half, p = i - t * half;
    const double turns = (double)a.pos[t0 + t] * (a.freqs[p] * 0.15915494309189533577);
    const float frac = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.f * frac, &s, &c);
    tab[t * k.stride() + k.at(p / k.K, p % k.K)] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
  }
}

// A thread owns one 16-byte column position (item) of U rows (a head of a token). Its loads are on their way while the block works the
// angles of its tokens out.
template <typename T, bool HALF>
__global__ void __launch_bounds__(ROT_THREADS, HALF ? 5 : 4) rotary_vec_kernel(const RotaryArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int U = HALF ? 2 : 4;      // rows in flight
  __shared__ float2 tab[ROT_ANGLES];
  constexpr int K = HALF ? N : N / 2;
  const int half = a.R >> 1, D = a.D;
  const RotTable place{K, half / K};
  const long t0 = (long)blockIdx.x * a.per_block;
  const int nt = (int)min((long)a.per_block, a.tokens - t0);
  // items of a head row. HALF: vectors of the first halves (with their partners), then the vectors that pass through
  const int turned = (HALF ? half : a.R) / N;
  const int items = HALF ? turned + (D - a.R) / N : D / N;
  const int rows = ROT_THREADS / items;
  const int it = threadIdx.x % items, row = threadIdx.x / items;
  const bool turn = it < turned;
  const int c0 = HALF ? (turn ? it * N : a.R + (it - turned) * N) : it * N;
  const int heads = a.heads[0] + a.heads[1], total = row < rows ? nt * heads : 0;
  // the block's first token; strides fit 32 bits here
  const T *xq = (const T*)a.x[0] + t0 * a.ld[0] + c0, *xk = (const T*)a.x[1] + t0 * a.ld[1] + c0;
  T *yq = (T*)a.y[0] + t0 * a.heads[0] * D + c0, *yk = (T*)a.y[1] + t0 * a.heads[1] * D + c0;
  const int hq = a.heads[0], hk = a.heads[1], ldq = (int)a.ld[0], ldk = (int)a.ld[1], lhq = (int)a.lh[0], lhk = (int)a.lh[1];
  bool ready = false;
  for (int first = blockIdx.y * U * rows + row; first - row < nt * heads || !ready; first += gridDim.y * U * rows) {
    Vec16<T> u[U], w[U];
    T* dst[U];
    int tok[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = first + i * rows;
      if (r < total) {
        const int t = (int)a.by_heads.div((unsigned)r), h = r - t * heads;
        const bool k = h >= hq;
        const int hh = k ? h - hq : h;
        const T* src = (k ? xk : xq) + (long)t * (k ? ldk : ldq) + (long)hh * (k ? lhk : lhq);
        dst[i] = (k ? yk : yq) + (long)(t * (k ? hk : hq) + hh) * D;
        tok[i] = t * place.stride() + it;
        u[i].load_nc(src);
        if (HALF && turn) w[i].load_nc(src + half);
      }
    }
    if (!ready) {
      rot_angles(a, t0, nt, place, tab);
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (first + i * rows < total) {
        if (turn) {
          float f[N];
          u[i].get(f);
          if (HALF) {
            float g[N];
            w[i].get(g);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float2 cs = tab[tok[i] + j * place.G];
              const float x = f[j], y = g[j];
              f[j] = x * cs.x - y * cs.y;
              g[j] = x * cs.y + y * cs.x;
            }
            w[i].set(g);
            w[i].store(dst[i] + half);
          } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
              const float2 cs = tab[tok[i] + j * place.G];
              const float x = f[2 * j], y = f[2 * j + 1];
              f[2 * j] = x * cs.x - y * cs.y;
              f[2 * j + 1] = x * cs.y + y * cs.x;
            }
          }
          u[i].set(f);
        }
        u[i].store(dst[i]);
      }
    }
  }
}

// Head sizes, pairings and addresses that 16-byte vectors do not fit: one pair (or one column that passes through) at a time.
template <typename T, bool HALF>
__global__ void __launch_bounds__(ROT_THREADS) rotary_scalar_kernel(const RotaryArgs a) {
  __shared__ float2 tab[ROT_ANGLES];
  const int half = a.R >> 1, D = a.D;
  const long t0 = (long)blockIdx.x * a.per_block;
  const int nt = (int)min((long)a.per_block, a.tokens - t0);
  rot_angles(a, t0, nt, RotTable{1, half}, tab);
  __syncthreads();
  const int items = half + D - a.R, total = a.heads[0] + a.heads[1];
  for (int t = 0; t < nt; ++t)
    for (long i = (long)blockIdx.y * ROT_THREADS + threadIdx.x; i < (long)total * items; i += (long)gridDim.y * ROT_THREADS) {
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
static int rotary_launch(RotaryArgs& a, bool half, bool vec, cudaStream_t st) {
  // A block's tokens: as many as its threads have rows in flight for, and as many more as give each thread an angle while there are 24
  // blocks for each SM, of which it holds 4 at a time. (8192 tokens of 64 heads of 128: 2 tokens 46 us; 1, whose 64 angles leave six
  // warps of eight idle, 55; 4, whose last round of blocks is half empty, 52.)
  constexpr int N = Vec16<T>::N;
  const int heads = a.heads[0] + a.heads[1];
  const int items = half ? a.R / 2 / N + (a.D - a.R) / N : a.D / N;
  const long rows = vec ? (long)(ROT_THREADS / items) * (half ? 2 : 4) : 1;
  long per = vec ? rows / heads : 1;
  if (a.R) {
    long full = ROT_THREADS / (a.R / 2);
    const long room = a.tokens / (24l * sm_count());
    full = full < room ? full : room;
    per = per > full ? per : full;
  }
  const long most = a.R ? ROT_ANGLES / (a.R / 2) : ROT_MAX_TOKENS;
  per = per < 1 ? 1 : per > ROT_MAX_TOKENS ? ROT_MAX_TOKENS : per;
  per = per > most ? most : per;
  a.per_block = (int)per;
  a.by_heads = FastDiv::of((unsigned)heads);
  // few tokens with many heads: several blocks to a token
  const long all = vec ? (per * heads + rows - 1) / rows : ceil_div((long)heads * (a.R / 2 + a.D - a.R), 8 * ROT_THREADS);
  const long want = a.tokens / per < sm_count() ? all : 1;
  const long chunks = want < 65535 ? want : 65535;
  const long blocks = (a.tokens + per - 1) / per;
  if (blocks > 0x7fffffffl) TB_FAIL(TB_E_TOO_LARGE, "rotary: too many tokens or heads");
  const dim3 grid((unsigned)blocks, (unsigned)chunks);
  if (vec && half) rotary_vec_kernel<T, true><<<grid, ROT_THREADS, 0, st>>>(a);
  else if (vec) rotary_vec_kernel<T, false><<<grid, ROT_THREADS, 0, st>>>(a);
  else if (half) rotary_scalar_kernel<T, true><<<grid, ROT_THREADS, 0, st>>>(a);
  else rotary_scalar_kernel<T, false><<<grid, ROT_THREADS, 0, st>>>(a);
  TB_CUDA_CHECK(cudaGetLastError());
  return 0;
}

}  // namespace tb
using namespace tb;

// Which text of decode_calls.h the launchers of this library have been built with.
TB_EXPORT uint64_t tb_decode_layout() { return TB_DECODE_LAYOUT; }

// q [tokens, hq, D], k [tokens, hk, D] (hk = 0: none) with strides in elements, columns contiguous; yq, yk contiguous.
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
  bool vec = D % N == 0 && D / N <= ROT_THREADS && (half ? R / 2 : R) % N == 0;   // a vector turns or passes through
  const uintptr_t at = (uintptr_t)q | (uintptr_t)yq | (hk ? (uintptr_t)k | (uintptr_t)yk : 0);
  vec = vec && at % 16 == 0 && ldq % N == 0 && lhq % N == 0 && (!hk || (ldk % N == 0 && lhk % N == 0));
  // the vector kernel has strides, and the rows of a block's tokens, in 32 bits
  const long far = 0x7fffffff;
  vec = vec && labs(ldq) <= far && labs(lhq) <= far && labs(ldk) <= far && labs(lhk) <= far && (c->hq + c->hk) * ROT_MAX_TOKENS <= far;
  RotaryArgs a{{q, k}, {yq, yk}, {ldq, ldk}, {lhq, lhk}, {hq, hk}, c->pos, c->freqs, tokens, D, R, 1, {}, (float)c->magnitude, c->inverse ? -1.f : 1.f};
  return dtype == 0 ? rotary_launch<bf16>(a, half, vec, st) : rotary_launch<float>(a, half, vec, st);
}
