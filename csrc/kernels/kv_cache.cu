// Paged cache of keys and values: quantised as it is written, read back in 16 or 32 bits (sm_100a).
//
// Pages are [num_pages, heads, page, D] in bf16, int8 or e4m3, so that the tokens of one head in one page lie together, which is
// how attention reads them. 8-bit rows (one token of one head) have one fp32 scale each, [num_pages, heads, page]:
//   int8   s = fl32(max|x| / 127), code = x / s to the nearest, halves to even
//   e4m3   s = 2^k, the least with max|x| / s <= 448: x / s is then exact, and the only rounding is that to e4m3. A scale of
//          max|x| / 448 would hold no more: e4m3 has the same three bits behind the leading one in every binade
// A row whose largest magnitude is below 2^-100 is held as zeros with scale 0; one that has an infinity or a NaN gets the scale
// NaN, so that reading it says so instead of giving numbers that never were.
//
// Bound by memory: each row is read and written once. D / 8 lanes share a row (8 elements each, the row's largest magnitude over
// shuffles); neighbouring groups take neighbouring heads of a token, which lie together on the contiguous side. Measured: 8 prompts of up
// to 2048 tokens, 32 heads of 128, bf16 into e4m3, written and read back, 694 MB: 124 to 128 us, 5.4 to 5.6 TB/s (127 with addresses in 64 bits
// throughout, where it took 124). One token of 13 sequences: 6.2 to 6.5 us, two launches of three dependent loads each (start, table, row).
#include <cuda_fp8.h>

#include "common.cuh"
#include "decode_calls.h"
#include "host_util.h"

namespace tb {

enum : int { KV_BF16 = 0, KV_INT8 = 1, KV_E4M3 = 2 };
constexpr int KV_THREADS = 256;

struct KvArgs {
  const void* x[2];            // k, v [B, T, H, D] with strides (write)
  long sb[2];                  // elements
  int st[2], sh[2];
  void* y[2];                  // k, v [B, T, H, D] contiguous (read)
  void* pages[2];
  float* scales[2];
  const int* table;            // [B, table_ld]
  const int* start;            // [B]: position of token 0 (null: 0)
  const int* counts;           // [B]: tokens that count (null: T)
  long table_ld;
  int B, T, H, page, pages_per_seq, num_pages, page_rows;   // page_rows: H * page
  FastDiv by_h, by_page;
};

// Address of a row in the pages, in rows; -1 where the position is outside the table or the table names no page of the pool, KV_VACANT
// where that is because the place has no sequence.
constexpr long KV_VACANT = -3;
__device__ __forceinline__ long kv_row(const KvArgs& a, int b, int t, int h) {
  const int first = a.start ? a.start[b] : 0;
  if (first < 0) return -1;
  const unsigned pos = (unsigned)first + (unsigned)t;
  if (pos >= 0x80000000u) return -1;
  const unsigned slot = a.by_page.div(pos);
  if (slot >= (unsigned)a.pages_per_seq) return -1;
  const int p = a.table[b * a.table_ld + slot];
  if ((unsigned)p >= (unsigned)a.num_pages) return vacant_place(a.table + b * a.table_ld, p) ? KV_VACANT : -1;
  return (long)p * a.page_rows + (int)(h * a.page + (pos - slot * (unsigned)a.page));
}

// Largest |x| of 8 elements, as the bits of a float without its sign: a NaN counts for more than an infinity, that for more than any
// number. Of bf16 two at a time.
__device__ __forceinline__ uint32_t big8(const uint4& v) {
  auto m = [](uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); };
  const uint32_t x = m(m(v.x, v.y), m(v.z, v.w));
  return max(x << 16, x & 0xffff0000u);
}
__device__ __forceinline__ uint32_t big8(const uint4& v, const uint4& w) {
  const uint32_t k = 0x7fffffffu;
  return max(max(max(v.x & k, v.y & k), max(v.z & k, v.w & k)), max(max(w.x & k, w.y & k), max(w.z & k, w.w & k)));
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// 8 elements as they lie in memory, and as floats.
template <typename T> struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg((const uint4*)p + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ uint32_t big() const {
    if constexpr (sizeof(T) == 2) return big8(v[0]);
    else return big8(v[0], v[1]);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t* w = &v[0].x;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 2) f[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
      else f[j] = __uint_as_float(w[j]);
    }
  }
};

// x / s to the nearest integer, halves to even, decided exactly: n is next to the quotient, x - n s is exact in one fma (s has
// 24 bits, n 7, and the rest is smaller than s), and s / 2 is exact. A quotient in fp32 can round onto a half that x / s is not.
__device__ __forceinline__ int kv_round(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float r = fmaf(-n, s, x), h = 0.5f * s;
  const bool odd = ((int)n & 1) != 0;
  if (r > h || (r == h && odd)) n += 1.f;
  else if (r < -h || (r == -h && odd)) n -= 1.f;
  return (int)n;
}

// Row r of a sequence: token r / H, head r % H. A thread has a few rows, a pass of the block apart, so that their loads are in flight together.
constexpr int KV_WRITE_ROWS = 2, KV_READ_ROWS = 4;

template <typename T, int KIND, int D>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const KvArgs a) {
  constexpr int G = D / 8, PER = KV_THREADS / G, R = KV_WRITE_ROWS;
  const int lane = threadIdx.x % G;
  const unsigned r0 = blockIdx.x * (PER * R) + threadIdx.x / G;
  const int b = blockIdx.y;
  const int n = a.counts ? min(a.counts[b], a.T) : a.T;
  if ((int)(blockIdx.x * (PER * R) / (unsigned)a.H) >= n) return;
  Raw8<T> x[R][2];
  long row[R];
  const T *base[2] = {(const T*)a.x[0] + b * a.sb[0] + lane * 8, (const T*)a.x[1] + b * a.sb[1] + lane * 8};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const unsigned r = r0 + i * PER;
    const int t = (int)a.by_h.div(r), h = (int)(r - (unsigned)t * a.H);
    row[i] = -1;
    if (t < n) {
#pragma unroll
      for (int z = 0; z < 2; ++z) x[i][z].load(base[z] + (long)t * a.st[z] + (long)h * a.sh[z]);
      row[i] = kv_row(a, b, t, h);
      if (row[i] == -1 && lane == 0) report_bad_index();
    } else {
#pragma unroll
      for (int z = 0; z < 2; ++z) x[i][z].clear();
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      float f[8];
      x[i][z].get(f);
      if constexpr (KIND == KV_BF16) {
        Vec16<bf16> v;
        if constexpr (sizeof(T) == 2) v.raw = x[i][z].v[0];
        else v.set(f);
        if (row[i] >= 0) v.store((bf16*)a.pages[z] + row[i] * D + lane * 8);
      } else {
        const uint32_t bits = group_max<G>(x[i][z].big());
        const float big = __uint_as_float(bits);
        const bool wild = bits >= 0x7f800000u, none = bits < 0x0d800000u;   // 2^-100
        float s, inv;
        if (KIND == KV_INT8) {
          s = __fdiv_rn(big, 127.f);
          inv = __fdiv_rn(1.f, none ? 1.f : s);
        } else {
          // big = m 2^e with m in [1, 2); 448 = 1.75 x 2^8
          const int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
          s = __int_as_float((k + 127) << 23);
          inv = __int_as_float((127 - k) << 23);
        }
        uint32_t w[2] = {0u, 0u};
        if (!none && !wild) {
          if (KIND == KV_INT8) {
            // x / s to the nearest by a sum with 1.5 x 2^23. Where the rest x - n s (exact) is a half of s, or more for the error of
            // inv, the element is decided again by kv_round
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float t = fmaf(f[j], inv, 12582912.f);
              most = fmaxf(most, fabsf(fmaf(12582912.f - t, s, f[j])));
              w[j >> 2] |= (__float_as_uint(t) & 0xffu) << (8 * (j & 3));
            }
            if (most >= 0.4999f * s) {
              w[0] = w[1] = 0u;
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j >> 2] |= ((uint32_t)kv_round(f[j], s, inv) & 0xffu) << (8 * (j & 3));
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              w[j >> 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[j] * inv, f[j + 1] * inv), __NV_SATFINITE, __NV_E4M3)
                           << (8 * (j & 3));
          }
        }
        if (row[i] >= 0) {
          *(uint2*)((uint8_t*)a.pages[z] + row[i] * D + lane * 8) = make_uint2(w[0], w[1]);
          if (lane == 0) a.scales[z][row[i]] = wild ? __int_as_float(0x7fffffff) : none ? 0.f : s;
        }
      }
    }
}

template <typename T, int KIND, int D>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const KvArgs a) {
  constexpr int G = D / 8, PER = KV_THREADS / G, R = KV_READ_ROWS;
  const int lane = threadIdx.x % G;
  const unsigned r0 = blockIdx.x * (PER * R) + threadIdx.x / G;
  const int b = blockIdx.y;
  const int n = a.counts ? a.counts[b] : a.T;
  long row[R];
  T *base[2] = {(T*)a.y[0] + (long)b * a.T * a.H * D + lane * 8, (T*)a.y[1] + (long)b * a.T * a.H * D + lane * 8};
  uint4 raw[R][2];
  float sc[R][2];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const unsigned r = r0 + i * PER;
    const int t = (int)a.by_h.div(r), h = (int)(r - (unsigned)t * a.H);
    row[i] = t < a.T && t < n ? kv_row(a, b, t, h) : -2;
    if (row[i] == -1 && lane == 0) report_bad_index();
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      raw[i][z] = make_uint4(0u, 0u, 0u, 0u);
      sc[i][z] = 0.f;
      if (row[i] >= 0) {
        if constexpr (KIND == KV_BF16) {
          raw[i][z] = __ldg((const uint4*)((const bf16*)a.pages[z] + row[i] * D + lane * 8));
        } else {
          const uint2 w = __ldg((const uint2*)((const uint8_t*)a.pages[z] + row[i] * D + lane * 8));
          raw[i][z].x = w.x, raw[i][z].y = w.y;
          sc[i][z] = __ldg(a.scales[z] + row[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const unsigned r = r0 + i * PER;
    if (r >= (unsigned)a.T * (unsigned)a.H) break;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      float f[8];
      const uint32_t ws[4] = {raw[i][z].x, raw[i][z].y, raw[i][z].z, raw[i][z].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (KIND == KV_BF16) {
          f[j] = __uint_as_float(j & 1 ? ws[j >> 1] & 0xffff0000u : ws[j >> 1] << 16);
        } else {
          const uint8_t byte = (uint8_t)(ws[j >> 2] >> (8 * (j & 3)));
          if (KIND == KV_INT8) f[j] = (float)(int8_t)byte * sc[i][z];
          else f[j] = __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3))) * sc[i][z];
        }
      }
      T* y = base[z] + (long)r * D;
      if constexpr (sizeof(T) == 2) {
        Vec16<T> v;
        v.set(f);
        v.store(y);
      } else {
        *(float4*)y = make_float4(f[0], f[1], f[2], f[3]);
        *((float4*)y + 1) = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
  }
}

template <typename T, int KIND>
static int kv_launch(const KvArgs& a, int D, bool write, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div((long)a.T * a.H, KV_THREADS / (D / 8) * (write ? KV_WRITE_ROWS : KV_READ_ROWS)), (unsigned)a.B);
  if (write) {
    if (D == 64) kv_write_kernel<T, KIND, 64><<<grid, KV_THREADS, 0, st>>>(a);
    else kv_write_kernel<T, KIND, 128><<<grid, KV_THREADS, 0, st>>>(a);
  } else {
    if (D == 64) kv_read_kernel<T, KIND, 64><<<grid, KV_THREADS, 0, st>>>(a);
    else kv_read_kernel<T, KIND, 128><<<grid, KV_THREADS, 0, st>>>(a);
  }
  TB_CUDA_CHECK(cudaGetLastError());
  return 0;
}

static int kv_check(const KvArgs& a, int D, int kind, int dtype) {
  if (D != 64 && D != 128) TB_FAIL(TB_E_ARG, "kv cache: head dim 64 or 128");
  if (kind < 0 || kind > 2 || (dtype != 0 && dtype != 1)) TB_FAIL(TB_E_ARG, "kv cache: pages in bf16, int8 or e4m3, rows in bf16 or fp32");
  for (int z = 0; z < 2; ++z)
    if (!a.pages[z] || ((uintptr_t)a.pages[z] & 15) || (kind != KV_BF16 && !a.scales[z])) TB_FAIL(TB_E_ARG, "kv cache: pages must be 16-byte aligned and 8-bit pages have scales");
  if (!a.table) TB_FAIL(TB_E_ARG, "kv cache: no page table");
  return 0;
}

template <typename T>
static int kv_dispatch(const KvArgs& a, int D, int kind, bool write, cudaStream_t st) {
  if (kind == KV_BF16) return kv_launch<T, KV_BF16>(a, D, write, st);
  if (kind == KV_INT8) return kv_launch<T, KV_INT8>(a, D, write, st);
  return kv_launch<T, KV_E4M3>(a, D, write, st);
}

}  // namespace tb
using namespace tb;

int tb_set_check_word_kv_cache(int* word) {
  TB_CUDA_CHECK(set_check_word_this_tu(word));
  return 0;
}

// write: x[0], x[1] = k, v [B, T, H, D] with strides (batch, token, head) in elements, multiples of 16 bytes; rows t >= counts[b] are left out.
// read: x[0], x[1] [B, T, H, D] contiguous, written; rows t >= counts[b], and rows that no page holds, are zeros.
static int kv_call(const KvCall* c, bool write, cudaStream_t st) {
  if (c->B <= 0 || c->T <= 0) return 0;
  if (c->B > 65535 || c->H <= 0 || c->T > 0x7fffff00l || c->H > 0x7fffff00l || c->T * c->H > 0x7fffff00l)
    TB_FAIL(TB_E_TOO_LARGE, "kv cache: at most 65535 sequences and 2^31 rows a sequence in one call");
  if (c->page <= 0 || c->page > 0x7fffff00l || c->page * c->H > 0x7fffff00l || c->num_pages < 0 || c->num_pages > 0x7fffffff || c->pages_per_seq < 0 || c->pages_per_seq > 0x7fffffff)
    TB_FAIL(TB_E_ARG, "kv cache: bad sizes");
  KvArgs a{};
  for (int z = 0; z < 2; ++z) {
    if (write) a.x[z] = c->x[z], a.sb[z] = c->strides[3 * z], a.st[z] = (int)c->strides[3 * z + 1], a.sh[z] = (int)c->strides[3 * z + 2];
    else a.y[z] = c->x[z];
    a.pages[z] = c->pages[z], a.scales[z] = c->scales[z];
  }
  a.table = c->table, a.start = c->start, a.counts = c->counts, a.table_ld = c->table_ld;
  a.B = (int)c->B, a.T = (int)c->T, a.H = (int)c->H, a.page = (int)c->page, a.pages_per_seq = (int)c->pages_per_seq, a.num_pages = (int)c->num_pages;
  a.page_rows = a.page * a.H;
  a.by_h = FastDiv::of((unsigned)a.H), a.by_page = FastDiv::of((unsigned)a.page);
  const int D = (int)c->D, kind = (int)c->kind, dtype = (int)c->dtype;
  if (int r = kv_check(a, D, kind, dtype)) return r;
  if (!c->x[0] || !c->x[1] || (((uintptr_t)c->x[0] | (uintptr_t)c->x[1]) & 15)) TB_FAIL(TB_E_ARG, "kv cache: rows must be 16-byte aligned");
  const int N = dtype == 0 ? 8 : 4;
  for (int i = 0; write && i < 6; ++i)
    if (c->strides[i] % N || (i % 3 && labs(c->strides[i]) > 0x7fffffffl)) TB_FAIL(TB_E_ARG, "kv cache: strides must be multiples of 16 bytes, those of tokens and heads below 2^31");
  return dtype == 0 ? kv_dispatch<bf16>(a, D, kind, write, st) : kv_dispatch<float>(a, D, kind, write, st);
}
TB_EXPORT int tb_kv_write(const KvCall* c, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  return kv_call(c, true, st);
}
TB_EXPORT int tb_kv_read(const KvCall* c, cudaStream_t st) {
  TB_ENSURE_DEVICE();
  return kv_call(c, false, st);
}
