// A key/value cache in 4 bits: rows written and read back, and attention of the newest tokens over
// every cached key.
//
// Format.  A row of D channels (64 or 128) is D/2 code bytes and, per group of 32 channels, a bf16
// scale s and minimum m: value = m + s c, c in 0..15.  m is rounded down and s up, so that all values of
// the group lie in [m, m + 15 s] and no code has to be clamped.
#include <type_traits>

#include "async_copy.cuh"
#include "sva_common.cuh"
#include "sva_internal.h"

namespace sva {

constexpr int kGroup = 32;
constexpr int kTileKeys = 64;  // keys of one pipeline stage; page_rows is a multiple of it

struct Kv4 {
  int64_t n_pages, page_rows;
  int n_kv, shift;  // page_rows == 1 << shift with a page table
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  const int32_t* table;
  int64_t table_stride, table_cols;

  // Row index (over [page][row] of kv head h) of position l of sequence b, or -1.
  __device__ __forceinline__ int64_t row(int b, int h, int64_t l) const {
    int64_t page = b, r = l;
    if (l < 0) return -1;
    if (table) {
      const int64_t col = l >> shift;
      if (col >= table_cols) return -1;
      page = __ldg(table + b * table_stride + col);
      r = l & (page_rows - 1);
    }
    if (page < 0 || page >= n_pages || r >= page_rows) return -1;
    return (page * n_kv + h) * page_rows + r;
  }
};

// ---------------------------------------------------------------------------------------
// rows in and out
// ---------------------------------------------------------------------------------------
// HBM bound: D * size + D/2 + D/8 bytes a row, if a channel takes few instructions.  Writing, a thread has 16 channels (two
// threads a group: one shuffle joins their extremes, and what is worked out once a group is shared by 16
// channels); channels go two to an fp32x2 instruction, and numbers become integers by adding 3 * 2^22 (a conversion
// instruction runs at a quarter of the rate).  Reading, a thread has the 8 channels of one code word.  Measured: 8 x 32768 rows of 3 heads
// of 64 channels, bf16, keys and values: 76 us written (3.5 TB/s), 56 us read (4.7 TB/s); fp32: 116 us (4.0 TB/s) and 113 us.  The write is
// bound by latency: with 5.5 warps a scheduler 55 % of the cycles issue (14 instructions a channel), and of the 9.9 cycles
// that a warp takes for an instruction it waits 4.1 for the loads and 1.7 for the instruction before.

constexpr int kWriteChannels = 16;

// A thread's 16 channels as they stand in memory.
template <typename T>
struct Raw {
  static constexpr int kVecs = kWriteChannels * sizeof(T) / 16;
  uint4 v[kVecs];
};

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, Raw<T>& r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kVecs; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return;
  }
  uint32_t* w = reinterpret_cast<uint32_t*>(r.v);
#pragma unroll
  for (int i = 0; i < Raw<T>::kVecs * 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(p[i]);
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p) + 2 * i;
      w[i] = u[0] | static_cast<uint32_t>(u[1]) << 16;
    }
  }
}

// Extremes of the 16 channels; NaN in both where a channel is NaN.
template <typename T>
__device__ __forceinline__ void extremes(const Raw<T>& r, float& low, float& high) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
  if constexpr (sizeof(T) == 4) {
    float odd = 0.f;
    low = high = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 0; i < kWriteChannels; ++i) {
      const float x = __uint_as_float(w[i]);
      low = fminf(low, x);
      high = fmaxf(high, x);
      odd = fmaf(x, 0.f, odd);  // NaN for a NaN (or an infinity, which is refused all the same)
    }
    low += odd;
    high += odd;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* e = reinterpret_cast<const T2*>(r.v);
    T2 a = e[0], b = e[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      a = __hmin2_nan(a, e[i]);
      b = __hmax2_nan(b, e[i]);
    }
    low = to_f32<T>(__hmin_nan(a.x, a.y));
    high = to_f32<T>(__hmax_nan(b.x, b.y));
  }
}

template <typename T>
__device__ __forceinline__ float element(const Raw<T>& r, int i) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(w[i]);
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(__ushort_as_half((unsigned short)(w[i >> 1] >> (16 * (i & 1)))));
  else
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
}

// Two differences x - m, not below 0, rounded to odd: the one towards zero, and where that is not exact its last bit set.  A half
// step (c + 1/2) s has at most 13 bits and a difference near it 24, so such a difference is a half step only where the exact one is.
__device__ __forceinline__ uint64_t sub2_odd(uint64_t x, uint64_t minus_m) {
  uint64_t zero, up;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(zero) : "l"(x), "l"(minus_m));
  asm("add.rp.f32x2 %0, %1, %2;" : "=l"(up) : "l"(x), "l"(minus_m));
  return zero | (up & 0x0000000100000001ull);
}

// The nearest code where the group's scale is far from the ends of the fp32 range.  The quotient d * inv is corrected by its
// remainder, so that it is the exact quotient of d rounded once: one that is a half k + 1/2 comes out as exactly that and no other
// does (the next differences' quotients are more than half a unit away), and adding 3 * 2^22 rounds it to even.
template <typename T>
__device__ __forceinline__ uint64_t codes16(const Raw<T>& r, float m, float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  uint32_t w[2] = {0u, 0u};
  const uint64_t m2 = pack2(-m, -m), s2 = pack2(-s, -s), i2 = pack2(inv, inv);
  const uint64_t round2 = pack2(12582912.f, 12582912.f);
#pragma unroll
  for (int i = 0; i < kWriteChannels; i += 2) {
    const uint64_t d = sub2_odd(pack2(element<T>(r, i), element<T>(r, i + 1)), m2);
    uint64_t q = mul2(d, i2);
    q = fma2(fma2(q, s2, d), i2, q);
    q = add2(q, round2);
    float lo, hi;
    unpack2(q, lo, hi);
    // the code is the low bits; each comes in at the top
    w[i >> 3] = __funnelshift_r(w[i >> 3], __float_as_uint(lo), 4);
    w[i >> 3] = __funnelshift_r(w[i >> 3], __float_as_uint(hi), 4);
  }
  return static_cast<uint64_t>(w[1]) << 32 | w[0];
}

// The same in 64 bits, for scales near the ends of the range.
template <typename T>
__device__ __forceinline__ uint64_t codes16_wide(const Raw<T>& r, float m, float s) {
  uint64_t w = 0;
#pragma unroll 1
  for (int i = 0; i < kWriteChannels; ++i) {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < kWriteChannels; ++j) x = j == i ? element<T>(r, j) : x;
    // rounded to odd, as above
    const double zero = __dsub_rz(x, m), up = __dsub_ru(x, m);
    const double d = __longlong_as_double(__double_as_longlong(zero) | (__double_as_longlong(up) & 1ll));
    const double c = rint(d / s);
    w |= static_cast<uint64_t>(fmin(fmax(c, 0.0), 15.0)) << (4 * i);
  }
  return w;
}

struct Kv4WriteParams {
  Kv4 c;
  const void* x[2];
  int64_t seq_stride[2], head_stride[2], row_stride[2];
  bool vec[2];
  int n_seqs;
  int64_t n_tokens;
  const int64_t* start;
  const int64_t* cu;
};

constexpr int kWriteRows = 8;   // rows that a thread takes one after another
constexpr int kWriteAhead = 2;  // of which so many are on their way while one is worked on

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4WriteParams p) {
  constexpr int kLanes = D / kWriteChannels, kRows = 256 / kLanes;
  const bool second = blockIdx.z != 0;
  const int h = blockIdx.y % p.c.n_kv, lane = threadIdx.x % kLanes, b0 = blockIdx.y / p.c.n_kv;
  const int64_t row_stride = second ? p.row_stride[1] : p.row_stride[0];
  const bool vec = second ? p.vec[1] : p.vec[0];
  const T* base = reinterpret_cast<const T*>(second ? p.x[1] : p.x[0]) + h * (second ? p.head_stride[1] : p.head_stride[0]) +
                  lane * kWriteChannels;
  uint64_t* codes = reinterpret_cast<uint64_t*>(second ? p.c.v_codes : p.c.k_codes) + lane;
  uint32_t* params = (second ? p.c.v_params : p.c.k_params) + (lane >> 1);
  const int64_t t0 = (int64_t)blockIdx.x * (kRows * kWriteRows) + threadIdx.x / kLanes;
  int64_t at0 = 0;  // position of token 0
  if (!p.cu) {
    base += b0 * (second ? p.seq_stride[1] : p.seq_stride[0]);
    at0 = __ldg(p.start + b0);
  }
  Raw<T> x[kWriteAhead + 1];
  int64_t row[kWriteAhead + 1];
  auto fetch = [&](int i, Raw<T>& r, int64_t& to) {
    const int64_t t = t0 + i * kRows;
    to = -1;
    r = Raw<T>{};
    if (i >= kWriteRows || t >= p.n_tokens) return;
    int b = b0;
    int64_t l = at0 + t;
    if (p.cu) {
      // the last sequence that begins at or before t
      int lo = 0, hi = p.n_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid) <= t) lo = mid; else hi = mid;
      }
      b = lo;
      if (__ldg(p.cu + b) > t || __ldg(p.cu + b + 1) <= t) return;
      l = __ldg(p.start + b) + t - __ldg(p.cu + b);
    }
    load16<T>(base + t * row_stride, vec, r);
    to = p.c.row(b, h, l);
  };
#pragma unroll
  for (int i = 0; i < kWriteAhead; ++i) fetch(i, x[i], row[i]);
#pragma unroll
  for (int i = 0; i < kWriteRows; ++i) {
    const int now = i % (kWriteAhead + 1), next = (i + kWriteAhead) % (kWriteAhead + 1);
    fetch(i + kWriteAhead, x[next], row[next]);
    float low, high;
    extremes<T>(x[now], low, high);
    const float low1 = __shfl_xor_sync(0xFFFFFFFFu, low, 1), high1 = __shfl_xor_sync(0xFFFFFFFFu, high, 1);
    const bool nan = low != low || low1 != low1;
    low = fminf(low, low1);
    high = fmaxf(high, high1);
    // rounded down to bf16: the upper half of the bits, one further from zero below it
    const uint32_t bits = __float_as_uint(low);
    const uint32_t mb = (bits + (static_cast<uint32_t>(static_cast<int>(bits) >> 31) & 0xFFFFu)) & 0xFFFF0000u;
    const float m = __uint_as_float(mb);
    // (high - m) / 15 rounded up to bf16: a number at or just below it, and the next one if 15 of those fall short
    const float d = __fsub_ru(high, m);
    uint32_t sb = (__float_as_uint(d * 0.06666659f) + 0xFFFFu) & 0xFFFF0000u;
    if (15.f * __uint_as_float(sb) < d) sb += 0x10000u;
    const float s = __uint_as_float(sb);
    const bool bad = nan || !(fabsf(m) <= 3.4e38f) || !(s <= 3.4e38f);
    uint64_t w = 0;
    if (s > 1e-30f && s < 1e30f) {
      w = codes16<T>(x[now], m, s);
    } else if (s > 0.f) {
      w = codes16_wide<T>(x[now], m, s);
    }
    if (row[now] >= 0) {
      codes[row[now] * kLanes] = bad ? 0ull : w;
      if ((lane & 1) == 0) params[row[now] * (D / kGroup)] = bad ? 0x7FFF7FFFu : mb | sb >> 16;
    }
  }
}

struct Kv4ReadParams {
  Kv4 c;
  void* out[2];
  int64_t n_tokens;
  const int64_t* start;
};

// (a & b) | c in one instruction (the compiler takes two where b and c are constants).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

constexpr int kReadUnroll = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  const bool second = blockIdx.z != 0;
  const int h = blockIdx.y % p.c.n_kv, b = blockIdx.y / p.c.n_kv, lane = threadIdx.x % kLanes;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(second ? p.c.v_codes : p.c.k_codes);
  const uint32_t* params = second ? p.c.v_params : p.c.k_params;
  const int64_t t0 = (int64_t)blockIdx.x * (kRows * kReadUnroll) + threadIdx.x / kLanes;
  const int64_t start = __ldg(p.start + b);
  uint32_t w[kReadUnroll], sm[kReadUnroll];
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    const int64_t t = t0 + u * kRows;
    w[u] = sm[u] = 0;
    if (t >= p.n_tokens) continue;
    const int64_t row = p.c.row(b, h, start + t);
    if (row < 0) continue;
    w[u] = __ldg(codes + row * kLanes + lane);
    sm[u] = __ldg(params + row * (D / kGroup) + (lane >> 2));
  }
  T* out = reinterpret_cast<T*>(second ? p.out[1] : p.out[0]) + (int64_t)blockIdx.y * p.n_tokens * D + lane * 8;
#pragma unroll
  for (int u = 0; u < kReadUnroll; ++u) {
    const int64_t t = t0 + u * kRows;
    if (t >= p.n_tokens) continue;
    const float s = __uint_as_float(sm[u] << 16), m = __uint_as_float(sm[u] & 0xFFFF0000u);
    const uint64_t s2 = pack2(s, s), m2 = pack2(m, m);
    const uint64_t off = pack2(-128.f, -128.f);
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // bf16 pair 128 + code, as two fp32 numbers
      const uint32_t v = and_or(w[u] >> (4 * i), 0x000F000Fu, 0x43004300u);
      const uint64_t c = add2(pack2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)), off);
      unpack2(fma2(c, s2, m2), y[i], y[i + 4]);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + t * D);
    if constexpr (sizeof(T) == 4) {
      dst[0] = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
      dst[1] = make_uint4(__float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7]));
    } else {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value)
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(y[2 * i + 1]), "f"(y[2 * i]));
        else
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(y[2 * i + 1]), "f"(y[2 * i]));
      }
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// ---------------------------------------------------------------------------------------
// attention over the cache
// ---------------------------------------------------------------------------------------
// One CTA takes a chunk of the keys of one (sequence, kv head) and up to 16 query columns (tokens x heads of the
// group); each of its warps streams its own 64-key tiles through its own ring of bulk copies (no CTA barrier in the
// loop) and keeps its own running maximum and sum per column.
//
// Mathematics.  With centred codes c - 8 (exact in 16 bits) and centre z = m + 8 s of a key's group g,
//   q.k     = sum_g s_g (q_g . (c_g - 8)) + z_g sum(q_g)
//   sum p v = sum_g [ (p s_g) . (c_g - 8) ] + sum_keys p z_g
// so the tensor cores multiply whole numbers and the scales act on fp32 accumulators.  Roundings: none of 16-bit queries (but
// see the query fragments); p s to fp16 for 16-bit queries, 2^-11 of it (bf16, 2^-8, would show in fp16 outputs), kept in
// range by a running unit for each channel group; fp32 queries and their p s in three bf16 parts, 2^-24 or better.
//
// Layout.  mma.m16n8k16 with the cache as the 16-row operand and the columns as N: keys x channels for
// the scores, channels x keys for the output, because a decode step has few columns (heads of a
// group), for which a 128-row tcgen05 tile would be empty.  Slot r of a 16-key tile is physical key
// slot_key(r), which makes the value loads of a warp fall into 32 different banks.
//
// Measured (device): 8 x 32768 keys, 9 / 3 heads of 64, bf16: 23.8 us = 2.6 TB/s of the cache's 63 MB; 64 ragged sequences of
// 1.69 M keys in pages of 256: 134 us = 3.9 TB/s.  Bound by latency: with 3.3 warps a scheduler (128 registers a thread) 55 % of the active cycles
// issue, and of the 6.0 cycles that a warp takes for an instruction it waits 1.2 for the one before and 1.0 for memory.

constexpr int kDecWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4DecParams {
  Kv4 c;
  const void* q;
  int64_t q_seq, q_head, q_row;
  void* out;
  int64_t o_seq, o_head, o_row;
  const int64_t* seq_lens;
  int64_t max_len;
  float scale_log2;
  int n_heads, n_tokens, groups, n_cols, col_tiles;
  int n_chunks;
  int64_t chunk_keys;
  float* lse;
  float* weights;
  int64_t w_seq, w_head;
  float* part_ml;  // [problem][chunk][8 NT][2]
  float* part_o;   // [problem][chunk][8 NT][D]
  float* logits;   // [sequence][kv head][column][logit_stride]
  int64_t logit_stride;
  int* status;
};

__device__ __forceinline__ int64_t seq_len_of(const Kv4DecParams& p, int b) {
  int64_t n = p.max_len;
  if (p.seq_lens) {
    n = __ldg(p.seq_lens + b);
    n = n < 0 ? 0 : (n > p.max_len ? p.max_len : n);
  }
  return n;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

__device__ __forceinline__ void mma_bf16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^x by the hardware's approximation (2 units of 2^-23 relative; results below 2^-126 become 0, which a
// softmax weight beside a weight of 1 cannot show).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Two codes in the low bits of both halves of v -> bf16 pair of code - 8: 0x4300 is 128 with the code
// as its lowest mantissa bits, 0x4308 is 136.
__device__ __forceinline__ uint32_t codes_bf16(uint32_t v) {
  const uint32_t x = and_or(v, 0x000F000Fu, 0x43004300u);
  const __nv_bfloat162 d = __hsub2(reinterpret_cast<const __nv_bfloat162&>(x),
                                   __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
  return reinterpret_cast<const uint32_t&>(d);
}

__device__ __forceinline__ int slot_key(int r) { return (r & 8) + ((r & 7) >> 1) + 4 * (r & 1); }

__device__ __forceinline__ void mma_f16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two codes around 8 in fp16 from the low (high) halves of both halves of v: 0x6400 is 1024 with the code in its lowest (16 times
// the code in its next) mantissa bits; 1032, 1/16 and -72.
__device__ __forceinline__ uint32_t codes_f16_lo(uint32_t v) {
  const uint32_t x = and_or(v, 0x000F000Fu, 0x64006400u);
  const __half2 d = __hsub2(reinterpret_cast<const __half2&>(x), __half2half2(__ushort_as_half(0x6408)));
  return reinterpret_cast<const uint32_t&>(d);
}
__device__ __forceinline__ uint32_t codes_f16_hi(uint32_t v) {
  const uint32_t x = and_or(v, 0x00F000F0u, 0x64006400u);
  const __half2 d = __hfma2(reinterpret_cast<const __half2&>(x), __half2half2(__ushort_as_half(0x2C00)),
                            __half2half2(__ushort_as_half(0xD480)));
  return reinterpret_cast<const uint32_t&>(d);
}

// A word's eight codes around 8 as the pairs (i, i + 4), i = 0..3, of a score operand: in fp16 for 16-bit queries, where two of
// the four pairs need no shift (9 instructions a word), in bf16 for fp32 queries, whose three bf16 parts keep every bit.  (Read
// as e4m3 bytes the codes would be exact as they stand, 2^-9 times the code, but mma.sync on bytes compiles to conversions here:
// 224 registers instead of 99.)
template <bool kWide>
__device__ __forceinline__ void code_fragments(uint32_t w, uint32_t r[4]) {
  if constexpr (!kWide) {
    r[0] = codes_f16_lo(w);
    r[1] = codes_f16_hi(w);
    r[2] = codes_f16_lo(w >> 8);
    r[3] = codes_f16_hi(w >> 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = codes_bf16(w >> (4 * i));
  }
}

// KP: key tiles that share the 8 columns of an accumulator.  With at most 4 query columns, columns 0-3 take one 16-key
// tile and 4-7 the next (each with the other's query columns zero), so that no lane's softmax work is for nothing.
template <typename T, int D, int NT, int KP>
struct DecShape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kParts = kWide ? 3 : 1;  // operands that q, and p s, are split into: bf16, or one of fp16
  static constexpr int kGroups = D / kGroup;
  static constexpr int kTileBytes = kTileKeys * (D / 2 + D / 8) * 2;
  static constexpr int kStages = 2;
  static constexpr int kCols = KP == 2 ? 4 : 8 * NT;
  static constexpr int kSmem = kDecWarps * kStages * kTileBytes + 128;
};

template <int N>
__device__ __forceinline__ void load_params(const unsigned char* at, uint32_t (&v)[N]) {
  if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    v[0] = x.x, v[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(at);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  }
}

template <typename T, int D, int NT, int KP, bool kLogits>
__global__ void __launch_bounds__(kDecWarps * 32) kv4_decode_kernel(const Kv4DecParams p) {
  using S = DecShape<T, D, NT, KP>;
  static_assert(KP == 1 || NT == 1, "shared accumulators hold one column tile");
  constexpr int kG = S::kGroups, kStages = S::kStages, kSlots = 4 / KP;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ct = blockIdx.y % p.col_tiles, h = blockIdx.y / p.col_tiles, b = blockIdx.z;
  const int chunk = blockIdx.x;
  const int col0 = ct * S::kCols;
  pdl_launch_dependents();
  const int64_t len = seq_len_of(p, b);
  const int64_t key0 = chunk * p.chunk_keys, key1 = min(len, key0 + p.chunk_keys);
  if (key0 >= len && chunk > 0) return;  // the join reads ceil(len / chunk_keys) chunks (at least one)

  // the first key (counted from key0) of a channel group whose value is not finite and which some columns may not see
  __shared__ int hidden[kDecWarps][kG];
  if (lane < kG) hidden[warp][lane] = 0x7FFFFFFF;
  unsigned char* ring = smem + 128 + warp * (kStages * S::kTileBytes);
  const uint32_t bar0 = smem_u32(smem) + warp * (8 * kStages);
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(bar0 + 8 * s, 1);
    mbar_fence_init();
  }
  __syncwarp();

  const int n_tiles = key1 > key0 ? (int)((key1 - key0 + kTileKeys - 1) / kTileKeys) : 0;
  const int my_tiles = n_tiles > warp ? (n_tiles - warp + kDecWarps - 1) / kDecWarps : 0;
  // lane i holds the row index of this warp's tile 32 k + i; -1: not in the cache
  auto rows_of = [&](int it0) -> int64_t {
    const int i = it0 + lane;
    return i < my_tiles ? p.c.row(b, h, key0 + (int64_t)(warp + i * kDecWarps) * kTileKeys) : -1;
  };
  int64_t rows_cur = rows_of(0), rows_next = my_tiles > 32 ? rows_of(32) : -1;
  constexpr uint32_t kC = kTileKeys * D / 2, kP = kTileKeys * D / 8;  // bytes of a tile's codes and parameters
  // lanes 0-3 copy one of a tile's four arrays each: where it starts, and its offset in a stage
  const unsigned char* from = lane == 0 ? p.c.k_codes : lane == 1 ? reinterpret_cast<const unsigned char*>(p.c.k_params)
                              : lane == 2 ? p.c.v_codes : reinterpret_cast<const unsigned char*>(p.c.v_params);
  const uint32_t row_bytes = lane & 1 ? D / 8 : D / 2, bytes = row_bytes * kTileKeys;
  const uint32_t to = smem_u32(ring) + (lane & 1 ? kC : 0u) + (lane & 2 ? kC + kP : 0u);
  auto issue = [&](int it, int base) {  // copies of tile it into stage it % kStages; base: first tile of rows_cur
    const int64_t r = it < base + 32 ? __shfl_sync(0xFFFFFFFFu, rows_cur, it - base)
                                     : __shfl_sync(0xFFFFFFFFu, rows_next, it - base - 32);
    const int s = it % kStages;
    const uint32_t bar = bar0 + 8 * s;
    if (r < 0) {
      if (lane == 0) mbar_arrive(bar);
      return;
    }
    if (lane == 0) mbar_expect_tx(bar, S::kTileBytes);
    __syncwarp();
    if (lane < 4) bulk_load(to + s * S::kTileBytes, from + r * row_bytes, bytes, bar);
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (s < my_tiles) issue(s, 0);

  // query fragments: the lane's column (g, or g % 4), channels 32 G + 8 t .. + 7
  uint32_t qf[kG][S::kParts][KP][NT][4];
  float qsum[kG][NT][2], scale[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = col0 + (KP == 2 ? (g & 3) : 8 * n + g);
    const bool live = col < p.n_cols;
    const int tok = p.n_tokens == 1 ? 0 : col / p.groups, head = h * p.groups + col - tok * p.groups;
    const T* src = reinterpret_cast<const T*>(p.q) + b * p.q_seq + (int64_t)head * p.q_head + (int64_t)tok * p.q_row;
    float x[kG][8], big = 0.f, unit = 1.f;
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
#pragma unroll
    for (int gr = 0; gr < kG; ++gr) {
      uint4 raw[sizeof(T) / 2] = {};
      const T* at = src + gr * kGroup + 8 * t;
      if (live && vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
      } else if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(raw)[i] = at[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[gr][i] = to_f32<T>(reinterpret_cast<const T*>(raw)[i]);
    }
#pragma unroll
    for (int gr = 0; gr < kG; ++gr)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p.scale_log2 < 0.f) x[gr][i] = -x[gr][i];  // the scale below is then positive
        big = fmaxf(big, fabsf(x[gr][i]));
      }
    if constexpr (!S::kWide) {
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      // the power of two that brings the column's largest element to [2^14, 2^15): exact in fp16, but for what lies 2^-28 below
      // the largest, which is off by at most 2^-39 of it
      const uint32_t e = min(max(__float_as_uint(big) >> 23, 15u), 253u);
      const float factor = __uint_as_float((268u - e) << 23);
      unit = __uint_as_float((e - 14u) << 23);
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[gr][i] *= factor;
    }
    // this lane accumulates columns 2t and 2t + 1 (mod 4).  A factor of 0 would make NaN of a masked -inf; the smallest normal
    // number makes 0 of every score just as well.
    const int c = KP == 2 ? 2 * (t & 1) : 2 * t;
    const float to_log2 = fabsf(p.scale_log2);
    scale[n][0] = fmaxf(to_log2 * __shfl_sync(0xFFFFFFFFu, unit, c * 4), 1.2e-38f);
    scale[n][1] = fmaxf(to_log2 * __shfl_sync(0xFFFFFFFFu, unit, (c + 1) * 4), 1.2e-38f);
#pragma unroll
    for (int gr = 0; gr < kG; ++gr) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[gr][i];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      qsum[gr][n][0] = __shfl_sync(0xFFFFFFFFu, sum, c * 4);
      qsum[gr][n][1] = __shfl_sync(0xFFFFFFFFu, sum, (c + 1) * 4);
#pragma unroll
      for (int part = 0; part < S::kParts; ++part) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = S::kWide ? pack_bf16(x[gr][i], x[gr][i + 4]) : pack_f16(x[gr][i], x[gr][i + 4]);
          x[gr][i] -= bf16_lo(v[i]);
          x[gr][i + 4] -= bf16_hi(v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < KP; ++k) qf[gr][part][k][n][i] = KP == 1 || (g >> 2) == k ? v[i] : 0u;
      }
    }
  }
  int limit[NT][2];  // keys that the lane's columns see, counted from key0
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = col0 + (KP == 2 ? 2 * (t & 1) : 8 * n + 2 * t) + j;
      const int64_t seen = len - p.n_tokens + (p.n_tokens == 1 ? 0 : col / p.groups) + 1 - key0;
      limit[n][j] = col < p.n_cols ? (int)min(max(seen, (int64_t)0), p.chunk_keys) : 0;
    }
  // keys that every column sees, and that any sees
  const int seen_all = (int)min(max(len - p.n_tokens + 1 - key0, (int64_t)0), p.chunk_keys);
  const int seen_any = (int)(key1 - key0);

  // m_run: the largest scaled score so far; weights are taken relative to it.  fp16 weights times scales: a channel group's scales,
  // and its accumulators, are in units of 2^-15 of a power of two above the largest of its scales of V so far (the same for the
  // warp's columns), so that no product passes 2^15, and those down to 2^-29 of the largest keep all their bits whatever the
  // scales of the other groups.  Scales below 2^-100 raise no unit (nor does 0: its products are 0 in any).
  float m_run[NT][2], l_run[NT][2], zsum[kG][NT][2], acc[kG][2][NT][4];
  constexpr uint32_t kLeast = 27;  // biased exponent of 2^-100
  float per_unit[kG];              // 1 / unit; a power of two
#pragma unroll
  for (int gr = 0; gr < kG; ++gr) per_unit[gr] = __uint_as_float((269u - kLeast) << 23);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) m_run[n][j] = -INFINITY, l_run[n][j] = 0.f;
#pragma unroll
  for (int gr = 0; gr < kG; ++gr)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      zsum[gr][n][0] = zsum[gr][n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[gr][0][n][i] = acc[gr][1][n][i] = 0.f;
    }

  bool failed = false;
  int failed_at = 0, base = 0;
  const int key_a = slot_key(g);                       // the lane's first key of a 16-key tile; the other is 8 behind
  const int own = KP == 2 ? (t >> 1) * 16 + key_a : key_a;  // of a slot, for the lane's accumulator columns
  const uint32_t byte0 = 0x4400u + 0x2222u * (g & 1), byte1 = byte0 + 0x1111u;
  for (int it = 0; it < my_tiles; ++it) {
    if (it == base + 32) {
      base += 32;
      rows_cur = rows_next;
      rows_next = rows_of(base + 32);
    }
    const int s = it % kStages;
    // by vote: what follows is for whole warps
    if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar0 + 8 * s, (it / kStages) & 1))) {
      failed = true;
      failed_at = it;
      break;
    }
    const bool there = __shfl_sync(0xFFFFFFFFu, rows_cur, it - base) >= 0;
    const int l0 = (warp + it * kDecWarps) * kTileKeys;  // first key of the tile, counted from key0
    unsigned char* kc = ring + s * S::kTileBytes;
    unsigned char* kp = kc + kC;
    unsigned char* vc = kp + kP;
    unsigned char* vp = vc + kC;
    const bool whole = there && l0 + kTileKeys <= seen_all;
    if (!whole) {
      // Parameters of keys that no column sees can be anything: make their values finite.  Of keys that only some see, those that
      // are not finite become 0 too (0 times NaN is NaN) and make NaN of the columns that do see them at the end.
      const int from = there ? max(0, min(kTileKeys, seen_any - l0)) : 0;
      for (int e = max(0, min(from, seen_all - l0)) * kG + lane; e < kTileKeys * kG; e += 32) {
        uint32_t* w = reinterpret_cast<uint32_t*>(vp) + e;
        if (e >= from * kG) {
          *w = 0u;
        } else if ((*w & 0x7F80u) == 0x7F80u || (*w & 0x7F800000u) == 0x7F800000u) {
          *w = 0u;
          atomicMin(&hidden[warp][e % kG], l0 + e / kG);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }

    // scores of 64 keys
    float sc[kSlots][NT][4];
#pragma unroll
    for (int sl = 0; sl < kSlots; ++sl) {
      const int k0 = sl * 16 * KP;
      uint32_t pa[kG], pb[kG];
      load_params<kG>(kp + (k0 + own) * (D / 8), pa);
      load_params<kG>(kp + (k0 + own + 8) * (D / 8), pb);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[sl][n][i] = 0.f;
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        float c[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          const unsigned char* word = kc + (k0 + 16 * k + key_a) * (D / 2) + 16 * gr + 4 * t;
          uint32_t fa[4], fb[4];
          code_fragments<S::kWide>(*reinterpret_cast<const uint32_t*>(word), fa);
          code_fragments<S::kWide>(*reinterpret_cast<const uint32_t*>(word + 8 * (D / 2)), fb);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int part = 0; part < S::kParts; ++part) {
              const uint32_t* q = qf[gr][part][k][n];
              const uint32_t a0[4] = {fa[0], fb[0], fa[1], fb[1]}, a1[4] = {fa[2], fb[2], fa[3], fb[3]};
              if constexpr (S::kWide) {
                mma_bf16(c[n], a0, q[0], q[1]);
                mma_bf16(c[n], a1, q[2], q[3]);
              } else {
                mma_f16(c[n], a0, q[0], q[1]);
                mma_f16(c[n], a1, q[2], q[3]);
              }
            }
        }
        const float sa = bf16_lo(pa[gr]), sb = bf16_lo(pb[gr]);
        const float za = fmaf(8.f, sa, bf16_hi(pa[gr])), zb = fmaf(8.f, sb, bf16_hi(pb[gr]));
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[sl][n][i] = fmaf(i < 2 ? sa : sb, c[n][i], fmaf(i < 2 ? za : zb, qsum[gr][n][i & 1], sc[sl][n][i]));
      }
    }
    // a scale of V above the bound?  (NaN groups do not count: they make their own channels NaN)
    bool raised = false;
    float rescale[kG];  // old unit / new one
    if constexpr (!S::kWide) {
      auto bound = [&](int gr) { return (269u - (__float_as_uint(per_unit[gr]) >> 23)) << 7; };  // bf16 bits of 2^15 units
      uint32_t most[kG] = {};
#pragma unroll
      for (int i = 0; i < kG / 2; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(vp + 16 * (lane + 32 * i));
        const uint32_t x[4] = {w.x & 0xFFFFu, w.y & 0xFFFFu, w.z & 0xFFFFu, w.w & 0xFFFFu};
#pragma unroll
        for (int j = 0; j < 4; ++j) most[j % kG] = max(most[j % kG], x[j]);
      }
      bool above = false;
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) above |= most[gr] > bound(gr);
      if (__any_sync(0xFFFFFFFFu, above)) {
        uint32_t mine = 0;  // of group lane % kG
        for (int e = lane; e < kTileKeys * kG; e += 32) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(vp)[e] & 0xFFFFu;
          mine = max(mine, w < 0x7F80u ? w : 0u);
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, lane % kG == gr ? mine : 0u);
          rescale[gr] = 1.f;
          if (top > bound(gr)) {
            const float next = __uint_as_float((268u - (top >> 7)) << 23);
            rescale[gr] = next / per_unit[gr];
            per_unit[gr] = next;
            raised = true;
          }
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int sl = 0; sl < kSlots; ++sl)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int l = l0 + sl * 16 * KP + own + (i < 2 ? 0 : 8);
            if (!there || l >= limit[n][i & 1]) sc[sl][n][i] = -INFINITY;
          }
      asm volatile("");  // a branch and not a select per score
    }
    // running maximum
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int sl = 0; sl < kSlots; ++sl)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int l = l0 + sl * 16 * KP + own + (i < 2 ? 0 : 8);
          top[i & 1] = fmaxf(top[i & 1], sc[sl][n][i]);
          if constexpr (kLogits) {
            const int col = col0 + (KP == 2 ? 2 * (t & 1) : 8 * n + 2 * t) + (i & 1);
            if (col < p.n_cols && l < seen_any)
              p.logits[(((int64_t)b * p.c.n_kv + h) * p.n_cols + col) * p.logit_stride + key0 + l] =
                  sc[sl][n][i] * scale[n][i & 1];
          }
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = KP == 2 ? 2 : 4; o < 32; o <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xFFFFFFFFu, top[j], o));
        top[j] *= scale[n][j];
      }
      if (__any_sync(0xFFFFFFFFu, raised || top[0] > m_run[n][0] || top[1] > m_run[n][1])) {
        float alpha[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float m_new = fmaxf(m_run[n][j], top[j]);
          alpha[j] = m_new == -INFINITY ? 0.f : ex2(m_run[n][j] - m_new);
          m_run[n][j] = m_new;
          l_run[n][j] *= alpha[j];
        }
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          zsum[gr][n][0] *= alpha[0];
          zsum[gr][n][1] *= alpha[1];
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[gr][i >> 2][n][i & 3] *= raised ? alpha[i & 1] * rescale[gr] : alpha[i & 1];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float use[2] = {m_run[n][0] == -INFINITY ? 0.f : m_run[n][0], m_run[n][1] == -INFINITY ? 0.f : m_run[n][1]};
#pragma unroll
      for (int sl = 0; sl < kSlots; ++sl)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = ex2(fmaf(sc[sl][n][i], scale[n][i & 1], -use[i & 1]));
          sc[sl][n][i] = v;
          l_run[n][i & 1] += v;
        }
    }
    // output: channels x keys
#pragma unroll
    for (int sl = 0; sl < kSlots; ++sl) {
      const int k0 = sl * 16 * KP;
      uint32_t pa[kG], pb[kG];
      load_params<kG>(vp + (k0 + own) * (D / 8), pa);
      load_params<kG>(vp + (k0 + own + 8) * (D / 8), pb);
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        const float sa = bf16_lo(pa[gr]), sb = bf16_lo(pb[gr]);
        const float za = fmaf(8.f, sa, bf16_hi(pa[gr])), zb = fmaf(8.f, sb, bf16_hi(pb[gr]));
        const float ua = S::kWide ? sa : sa * per_unit[gr], ub = S::kWide ? sb : sb * per_unit[gr];
        uint32_t bp[NT][S::kParts][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float ps[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ps[i] = sc[sl][n][i] * (i < 2 ? ua : ub);
            zsum[gr][n][i & 1] = fmaf(sc[sl][n][i], i < 2 ? za : zb, zsum[gr][n][i & 1]);
          }
#pragma unroll
          for (int part = 0; part < S::kParts; ++part) {
            const uint32_t p0 = S::kWide ? pack_bf16(ps[0], ps[1]) : pack_f16(ps[0], ps[1]);
            const uint32_t p1 = S::kWide ? pack_bf16(ps[2], ps[3]) : pack_f16(ps[2], ps[3]);
            bp[n][part][0] = transpose8x8(p0);
            bp[n][part][1] = transpose8x8(p1);
            if (part + 1 < S::kParts) {
              ps[0] -= bf16_lo(p0);
              ps[1] -= bf16_hi(p0);
              ps[2] -= bf16_lo(p1);
              ps[3] -= bf16_hi(p1);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          uint32_t a[2][4];
          const unsigned char* word = vc + (k0 + 16 * k + t) * (D / 2) + 16 * gr + 4 * (g >> 1);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(word + (8 * half) * (D / 2));
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(word + (8 * half + 4) * (D / 2));
            const uint32_t x0 = __byte_perm(w0, w1, byte0), x1 = __byte_perm(w0, w1, byte1);
            a[0][2 * half] = S::kWide ? codes_bf16(x0) : codes_f16_lo(x0);
            a[0][2 * half + 1] = S::kWide ? codes_bf16(x0 >> 4) : codes_f16_hi(x0);
            a[1][2 * half] = S::kWide ? codes_bf16(x1) : codes_f16_lo(x1);
            a[1][2 * half + 1] = S::kWide ? codes_bf16(x1 >> 4) : codes_f16_hi(x1);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int part = 0; part < S::kParts; ++part) {
              const bool mine = KP == 1 || (g >> 2) == k;
              const uint32_t b0 = mine ? bp[n][part][0] : 0u, b1 = mine ? bp[n][part][1] : 0u;
              if constexpr (S::kWide) {
                mma_bf16(acc[gr][0][n], a[0], b0, b1);
                mma_bf16(acc[gr][1][n], a[1], b0, b1);
              } else {
                mma_f16(acc[gr][0][n], a[0], b0, b1);
                mma_f16(acc[gr][1][n], a[1], b0, b1);
              }
            }
        }
      }
    }
    __syncwarp();
    if (it + kStages < my_tiles) issue(it + kStages, base);
  }
  if (failed) {
    // the copies still in flight must land before this CTA's shared memory goes to another
    for (int it = failed_at; it < min(failed_at + kStages, my_tiles); ++it)
      mbar_wait(bar0 + 8 * (it % kStages), (it / kStages) & 1);
    if (lane == 0 && p.status) atomicExch(p.status, SVA_ERR_TIMEOUT);
#pragma unroll
    for (int n = 0; n < NT; ++n) l_run[n][0] = l_run[n][1] = NAN;
  }
  // the four warps' states meet in shared memory; every copy issued has been waited for unless a wait
  // failed, and then the ring is not reused
  __shared__ float w_m[kDecWarps][S::kCols], w_l[kDecWarps][S::kCols];
  const bool any_failed = __syncthreads_or(failed);
  float* w_o = reinterpret_cast<float*>(smem + 128);  // [warp][column][D]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = KP == 2 ? 2 : 4; o < 32; o <<= 1) {
        l_run[n][j] += __shfl_xor_sync(0xFFFFFFFFu, l_run[n][j], o);
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) zsum[gr][n][j] += __shfl_xor_sync(0xFFFFFFFFu, zsum[gr][n][j], o);
      }
      const int c = (KP == 2 ? 2 * (t & 1) : 8 * n + 2 * t) + j;
      if (g == 0 && (KP == 1 || t < 2)) {
        w_m[warp][c] = m_run[n][j];
        w_l[warp][c] = l_run[n][j];
      }
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        float o[4] = {acc[gr][0][n][j], acc[gr][0][n][2 + j], acc[gr][1][n][j], acc[gr][1][n][2 + j]};
        if constexpr (KP == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] += __shfl_xor_sync(0xFFFFFFFFu, o[i], 2);
        }
        if constexpr (!S::kWide) {
          const float unit = __uint_as_float((254u << 23) - __float_as_uint(per_unit[gr]));
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] *= unit;
        }
        const float z = limit[n][j] > hidden[warp][gr] ? NAN : zsum[gr][n][j];
        if (!any_failed && (KP == 1 || t < 2))
          *reinterpret_cast<float4*>(w_o + (warp * S::kCols + c) * D + kGroup * gr + 4 * g) =
              make_float4(o[0] + z, o[1] + z, o[2] + z, o[3] + z);
      }
    }
  __syncthreads();
  const bool last = p.n_chunks == 1;
  const int64_t problem = ((int64_t)b * p.c.n_kv + h) * p.col_tiles + ct;
  for (int e = threadIdx.x; e < S::kCols * D; e += blockDim.x) {
    const int c = e / D, d = e % D, col = col0 + c;
    if (col >= p.n_cols) break;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, w_m[w][c]);
    const float use = top == -INFINITY ? 0.f : top;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float f = ex2(w_m[w][c] - use);
      l = fmaf(f, w_l[w][c], l);
      o = any_failed ? NAN : fmaf(f, w_o[(w * S::kCols + c) * D + d], o);
    }
    if (last) {
      const int tok = p.n_tokens == 1 ? 0 : col / p.groups, head = h * p.groups + col - tok * p.groups;
      const bool none = top == -INFINITY && l == 0.f;
      reinterpret_cast<T*>(p.out)[b * p.o_seq + (int64_t)head * p.o_head + (int64_t)tok * p.o_row + d] =
          from_f32<T>(none ? 0.f : o / l);
      if (p.lse && d == 0)
        p.lse[((int64_t)b * p.n_heads + head) * p.n_tokens + tok] = none ? -INFINITY : (use + log2f(l)) / kLog2e;
    } else {
      p.part_o[((problem * p.n_chunks + chunk) * S::kCols + c) * D + d] = o;
    }
    if (d == 0 && (!last || kLogits)) {
      float* ml = p.part_ml + ((problem * p.n_chunks + chunk) * S::kCols + c) * 2;
      ml[0] = top;
      ml[1] = l;
    }
  }
}

// Joins the chunks of one (sequence, kv head, column): blockIdx.x < n_cols; the blocks behind add the
// softmax weights of 1024 keys each.  Every warp reads the chunks' maxima and sums for itself.
constexpr int kJoinThreads = 256;

template <typename T, int D, int COLS>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(const Kv4DecParams p) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t len = seq_len_of(p, b);
  const int chunks = max((int)((len + p.chunk_keys - 1) / p.chunk_keys), 1);
  const int tid = threadIdx.x, lane = tid & 31;
  const int join_blocks = p.n_chunks > 1 ? p.n_cols : 0;
  const int64_t l0 = (int64_t)((int)blockIdx.x - join_blocks) * 1024;
  __shared__ float part[kJoinThreads];
  // by every block: the next kernel of the stream starts when these have ended, and the decode kernel must have by then
  pdl_wait();
  if (l0 >= len && (int)blockIdx.x >= join_blocks) return;
  auto stats = [&](int col, float* top_out, float* l_out) {  // maximum and sum of a column over its chunks
    const int64_t problem = ((int64_t)b * p.c.n_kv + h) * p.col_tiles + col / COLS;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + problem * p.n_chunks * COLS + col % COLS;
    float top = -INFINITY, l = 0.f;
    for (int c = lane; c < chunks; c += 32) {
      const float2 x = ml[(int64_t)c * COLS];
      const float m_new = fmaxf(top, x.x), use = m_new == -INFINITY ? 0.f : m_new;
      l = fmaf(l, ex2(top - use), x.y * ex2(x.x - use));
      top = m_new;
    }
    const float all = warp_max(top);
    *l_out = warp_sum(l * ex2(top - (all == -INFINITY ? 0.f : all)));
    *top_out = all;
  };
  if ((int)blockIdx.x < join_blocks) {
    const int col = blockIdx.x;
    float top, l;
    stats(col, &top, &l);
    const float use = top == -INFINITY ? 0.f : top;
    const int64_t problem = ((int64_t)b * p.c.n_kv + h) * p.col_tiles + col / COLS;
    const int64_t first = problem * p.n_chunks * COLS + col % COLS;
    const int d = tid % D;
    float o = 0.f;
#pragma unroll 8
    for (int c = tid / D; c < chunks; c += kJoinThreads / D) {
      const int64_t at = first + (int64_t)c * COLS;
      o = fmaf(ex2(p.part_ml[at * 2] - use), p.part_o[at * D + d], o);
    }
    part[tid] = o;
    __syncthreads();
    if (tid < D) {
#pragma unroll
      for (int i = 1; i < kJoinThreads / D; ++i) o += part[tid + i * D];
      const int tok = p.n_tokens == 1 ? 0 : col / p.groups, head = h * p.groups + col - tok * p.groups;
      const bool none = top == -INFINITY && l == 0.f;
      reinterpret_cast<T*>(p.out)[b * p.o_seq + (int64_t)head * p.o_head + (int64_t)tok * p.o_row + tid] =
          from_f32<T>(none ? 0.f : o / l);
      if (p.lse && tid == 0)
        p.lse[((int64_t)b * p.n_heads + head) * p.n_tokens + tok] = none ? -INFINITY : (use + log2f(l)) / kLog2e;
    }
    return;
  }
  constexpr int kEach = 1024 / kJoinThreads;
  float sum[kEach] = {};
  for (int col = 0; col < p.n_cols; ++col) {
    float x[kEach];
    const float* row = p.logits + (((int64_t)b * p.c.n_kv + h) * p.n_cols + col) * p.logit_stride;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int64_t key = l0 + j * kJoinThreads + tid;
      x[j] = key < len ? row[key] : -INFINITY;
    }
    float top, l;
    stats(col, &top, &l);
    if (top == -INFINITY && l == 0.f) continue;
    const float inv = 1.f / l;
#pragma unroll
    for (int j = 0; j < kEach; ++j) sum[j] = fmaf(ex2(x[j] - top), inv, sum[j]);
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t key = l0 + j * kJoinThreads + tid;
    if (key < len) p.weights[b * p.w_seq + h * p.w_head + key] += sum[j];
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
static int check_cache(const sva_kv4_cache* c, int n_seqs, Kv4* out) {
  if (!c) return set_error(SVA_ERR_SHAPE, "the cache is null");
  if (c->head_dim != 64 && c->head_dim != 128) return set_error(SVA_ERR_SHAPE, "a 4-bit cache takes head_dim 64 or 128");
  if (c->n_kv_heads <= 0 || c->n_pages <= 0 || c->page_rows <= 0 || c->page_rows % kTileKeys || c->page_rows > (1ll << 31))
    return set_error(SVA_ERR_SHAPE, "the cache needs pages of a multiple of 64 rows");
  if (!c->k_codes || !c->k_params || !c->v_codes || !c->v_params) return set_error(SVA_ERR_SHAPE, "a cache pointer is null");
  const void* ptrs[4] = {c->k_codes, c->k_params, c->v_codes, c->v_params};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16) return set_error(SVA_ERR_ALIGN, "the cache must be 16-byte aligned");
  if (n_seqs <= 0 || n_seqs > 65535) return set_error(SVA_ERR_SHAPE, "n_seqs must be in 1..65535");
  int shift = 0;
  if (c->page_table) {
    while ((1ll << shift) < c->page_rows) ++shift;
    if ((1ll << shift) != c->page_rows) return set_error(SVA_ERR_SHAPE, "with a page table page_rows must be a power of two");
    if (c->page_table_cols <= 0 || c->page_table_stride < 0) return set_error(SVA_ERR_SHAPE, "bad page table sizes");
  } else if (c->n_pages < n_seqs) {
    return set_error(SVA_ERR_SHAPE, "the cache has fewer pages than there are sequences, and no page table");
  }
  *out = Kv4{c->n_pages, c->page_rows, c->n_kv_heads, shift, static_cast<uint8_t*>(c->k_codes),
             static_cast<uint32_t*>(c->k_params), static_cast<uint8_t*>(c->v_codes), static_cast<uint32_t*>(c->v_params),
             c->page_table, c->page_table_stride, c->page_table_cols};
  return SVA_OK;
}

static int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SVA_OK : set_error(SVA_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T>
static int launch_write(const Kv4WriteParams& p, int D, bool packed, cudaStream_t st) {
  const int64_t rows = kWriteRows * (256 / (D / kWriteChannels));
  const int64_t blocks = (p.n_tokens + rows - 1) / rows;
  const int64_t ys = (int64_t)p.c.n_kv * (packed ? 1 : p.n_seqs);
  if (blocks > 0x7FFFFFFFll || ys > 65535) return set_error(SVA_ERR_SHAPE, "too many rows, or sequences times kv heads");
  const dim3 grid((unsigned)blocks, (unsigned)ys, 2);
  if (D == 64)
    kv4_write_kernel<T, 64><<<grid, 256, 0, st>>>(p);
  else
    kv4_write_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  return launched();
}

template <typename T>
static int launch_read(const Kv4ReadParams& p, int D, int n_seqs, cudaStream_t st) {
  const int64_t rows = kReadUnroll * (256 / (D / 8));
  const int64_t blocks = (p.n_tokens + rows - 1) / rows;
  const int64_t ys = (int64_t)p.c.n_kv * n_seqs;
  if (blocks > 0x7FFFFFFFll || ys > 65535) return set_error(SVA_ERR_SHAPE, "too many rows, or sequences times kv heads");
  const dim3 grid((unsigned)blocks, (unsigned)ys, 2);
  if (D == 64)
    kv4_read_kernel<T, 64><<<grid, 256, 0, st>>>(p);
  else
    kv4_read_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  return launched();
}

struct DecPlan {
  int cols, col_tiles, n_cols, chunks;
  int64_t chunk_keys, logit_stride;
  size_t ml, o, logits, total;  // byte offsets into the workspace, and its size
};

static int plan_decode(const sva_kv4_cache* c, const sva_kv4_decode_args* a, Kv4* cache, DecPlan* plan) {
  if (!a) return set_error(SVA_ERR_SHAPE, "the arguments are null");
  int rc = check_cache(c, a->n_seqs, cache);
  if (rc != SVA_OK) return rc;
  if (a->n_heads <= 0 || a->n_heads % c->n_kv_heads) return set_error(SVA_ERR_SHAPE, "n_heads must be a multiple of the cache's kv heads");
  if (a->n_tokens <= 0) return set_error(SVA_ERR_SHAPE, "n_tokens must be positive");
  const int64_t capacity = c->page_table ? c->page_table_cols * c->page_rows : c->page_rows;
  if (a->max_len < 0 || a->max_len > capacity || a->max_len >= (1ll << 31))
    return set_error(SVA_ERR_SHAPE, "max_len must be within the cache's capacity and below 2^31");
  if (a->dtype < 0 || a->dtype > 2) return set_error(SVA_ERR_DTYPE, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  const int64_t n_cols = (int64_t)(a->n_heads / c->n_kv_heads) * a->n_tokens;
  // 4 columns where they suffice (two key tiles then share an accumulator), 16 where there are more than 8 (one pass
  // over the cache instead of two); fp32 queries take 8, their three parts fill the registers
  plan->cols = a->dtype == SVA_DTYPE_F32 ? 8 : (n_cols <= 4 ? 4 : (n_cols <= 8 ? 8 : 16));
  const int64_t tiles = (n_cols + plan->cols - 1) / plan->cols;
  if (n_cols > (1 << 20) || tiles * c->n_kv_heads > 65535) return set_error(SVA_ERR_SHAPE, "too many tokens times heads");
  plan->n_cols = (int)n_cols;
  plan->col_tiles = (int)tiles;
  const int64_t problems = (int64_t)a->n_seqs * c->n_kv_heads * plan->col_tiles;
  const int64_t slots = 148 * 4;  // CTAs that fit the GPU at once
  const int64_t tiles_k = std::max<int64_t>(1, (a->max_len + kTileKeys - 1) / kTileKeys);
  int64_t chunks = std::max<int64_t>(1, slots / problems);
  // at least 4 tiles a CTA (one a warp); at most 64 where lengths may differ, so that long sequences spread (64 ragged sequences of
  // 4096 to 131072 keys: 133 us with 48 or 64, 139 with 32, 146 with 128); one sequence fills the GPU in one wave of equal
  // chunks (a million keys: 90 us against 105 with chunks of 64 tiles)
  int64_t per = (tiles_k + chunks - 1) / chunks;
  per = std::max<int64_t>(per, kDecWarps);
  if (a->seq_lens && a->n_seqs > 1) per = std::min<int64_t>(per, 64);
  per = (per + kDecWarps - 1) / kDecWarps * kDecWarps;
  chunks = (tiles_k + per - 1) / per;
  plan->chunks = (int)chunks;
  plan->chunk_keys = per * kTileKeys;
  plan->logit_stride = a->max_len;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const bool parts = chunks > 1;
  plan->ml = 0;
  size_t at = (parts || a->weights) ? up((size_t)problems * chunks * plan->cols * 2 * 4) : 0;
  plan->o = at;
  if (parts) at += up((size_t)problems * chunks * plan->cols * c->head_dim * 4);
  plan->logits = at;
  if (a->weights) at += up((size_t)a->n_seqs * c->n_kv_heads * n_cols * a->max_len * 4);
  plan->total = at;
  return SVA_OK;
}

template <typename T, int D, int NT, int KP>
static int launch_decode(Kv4DecParams& p, int n_seqs, cudaStream_t st) {
  using S = DecShape<T, D, NT, KP>;
  const dim3 grid(p.n_chunks, p.c.n_kv * p.col_tiles, n_seqs);
  auto* kern = p.weights ? kv4_decode_kernel<T, D, NT, KP, true> : kv4_decode_kernel<T, D, NT, KP, false>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), S::kSmem);
  if (rc != SVA_OK) return rc;
  kern<<<grid, kDecWarps * 32, S::kSmem, st>>>(p);
  rc = launched();
  if (rc != SVA_OK) return rc;
  const int64_t wblocks = p.weights ? (p.max_len + 1023) / 1024 : 0;
  const int64_t jblocks = (p.n_chunks > 1 ? p.n_cols : 0) + wblocks;
  if (jblocks == 0) return SVA_OK;
  // launched while the decode kernel drains; it waits there for the decode kernel's memory
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)jblocks, p.c.n_kv, n_seqs);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, D, S::kCols>, p);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? SVA_OK : set_error(SVA_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T, int D>
static int decode_cols(Kv4DecParams& p, int cols, int n_seqs, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (cols == 4) return launch_decode<T, D, 1, 2>(p, n_seqs, st);
    if (cols == 16) return launch_decode<T, D, 2, 1>(p, n_seqs, st);
  }
  return launch_decode<T, D, 1, 1>(p, n_seqs, st);
}

template <typename T>
static int decode_dims(Kv4DecParams& p, int D, int cols, int n_seqs, cudaStream_t st) {
  return D == 64 ? decode_cols<T, 64>(p, cols, n_seqs, st) : decode_cols<T, 128>(p, cols, n_seqs, st);
}

}  // namespace sva

using namespace sva;

extern "C" int sva_kv4_write(const sva_kv4_cache* cache, const void* keys, int64_t k_seq_stride, int64_t k_head_stride,
                             int64_t k_row_stride, const void* values, int64_t v_seq_stride, int64_t v_head_stride,
                             int64_t v_row_stride, int32_t dtype, int32_t n_seqs, int64_t n_tokens,
                             const int64_t* start, const int64_t* cu_seqlens, void* stream) {
  Kv4WriteParams p{};
  int rc = check_cache(cache, n_seqs, &p.c);
  if (rc != SVA_OK) return rc;
  if (n_tokens < 0) return set_error(SVA_ERR_SHAPE, "n_tokens must not be negative");
  if (dtype < 0 || dtype > 2) return set_error(SVA_ERR_DTYPE, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  if (n_tokens == 0) return SVA_OK;
  if (!keys || !values || !start) return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  const int64_t strides[2][3] = {{k_seq_stride, k_head_stride, k_row_stride}, {v_seq_stride, v_head_stride, v_row_stride}};
  const void* ptr[2] = {keys, values};
  const int size = dtype == SVA_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    p.x[i] = ptr[i];
    p.seq_stride[i] = cu_seqlens ? 0 : strides[i][0];
    p.head_stride[i] = strides[i][1];
    p.row_stride[i] = strides[i][2];
    p.vec[i] = reinterpret_cast<uintptr_t>(ptr[i]) % 16 == 0 && p.seq_stride[i] * size % 16 == 0 &&
               p.head_stride[i] * size % 16 == 0 && p.row_stride[i] * size % 16 == 0;
  }
  p.n_seqs = n_seqs;
  p.n_tokens = n_tokens;
  p.start = start;
  p.cu = cu_seqlens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool packed = cu_seqlens != nullptr;
  switch (dtype) {
    case SVA_DTYPE_F32: return launch_write<float>(p, cache->head_dim, packed, st);
    case SVA_DTYPE_BF16: return launch_write<__nv_bfloat16>(p, cache->head_dim, packed, st);
    default: return launch_write<__half>(p, cache->head_dim, packed, st);
  }
}

extern "C" int sva_kv4_read(const sva_kv4_cache* cache, void* keys_out, void* values_out, int32_t dtype, int32_t n_seqs,
                            int64_t n_tokens, const int64_t* start, void* stream) {
  Kv4ReadParams p{};
  int rc = check_cache(cache, n_seqs, &p.c);
  if (rc != SVA_OK) return rc;
  if (n_tokens < 0) return set_error(SVA_ERR_SHAPE, "n_tokens must not be negative");
  if (dtype < 0 || dtype > 2) return set_error(SVA_ERR_DTYPE, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  if (n_tokens == 0) return SVA_OK;
  if (!keys_out || !values_out || !start) return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  if (reinterpret_cast<uintptr_t>(keys_out) % 16 || reinterpret_cast<uintptr_t>(values_out) % 16)
    return set_error(SVA_ERR_ALIGN, "the outputs must be 16-byte aligned");
  p.out[0] = keys_out;
  p.out[1] = values_out;
  p.n_tokens = n_tokens;
  p.start = start;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SVA_DTYPE_F32: return launch_read<float>(p, cache->head_dim, n_seqs, st);
    case SVA_DTYPE_BF16: return launch_read<__nv_bfloat16>(p, cache->head_dim, n_seqs, st);
    default: return launch_read<__half>(p, cache->head_dim, n_seqs, st);
  }
}

extern "C" size_t sva_kv4_decode_workspace_size(const sva_kv4_cache* cache, const sva_kv4_decode_args* args) {
  Kv4 c;
  DecPlan plan;
  return plan_decode(cache, args, &c, &plan) == SVA_OK ? plan.total : 0;
}

extern "C" int sva_kv4_decode(const sva_kv4_cache* cache, const sva_kv4_decode_args* a, void* workspace,
                              size_t workspace_bytes, void* stream) {
  Kv4DecParams p{};
  DecPlan plan;
  int rc = plan_decode(cache, a, &p.c, &plan);
  if (rc != SVA_OK) return rc;
  if (!a->query || !a->out) return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  if (plan.total > 0 && (!workspace || workspace_bytes < plan.total)) return set_error(SVA_ERR_WORKSPACE, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return set_error(SVA_ERR_ALIGN, "the workspace must be 16-byte aligned");
  p.q = a->query;
  p.q_seq = a->q_seq_stride, p.q_head = a->q_head_stride, p.q_row = a->q_row_stride;
  p.out = a->out;
  p.o_seq = a->out_seq_stride, p.o_head = a->out_head_stride, p.o_row = a->out_row_stride;
  p.seq_lens = a->seq_lens;
  p.max_len = a->max_len;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.n_heads = a->n_heads, p.n_tokens = a->n_tokens, p.groups = a->n_heads / cache->n_kv_heads;
  p.n_cols = plan.n_cols, p.col_tiles = plan.col_tiles, p.n_chunks = plan.chunks, p.chunk_keys = plan.chunk_keys;
  p.lse = a->lse;
  p.weights = a->weights;
  p.w_seq = a->weights_seq_stride, p.w_head = a->weights_head_stride;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.part_ml = reinterpret_cast<float*>(ws + plan.ml);
  p.part_o = reinterpret_cast<float*>(ws + plan.o);
  p.logits = reinterpret_cast<float*>(ws + plan.logits);
  p.logit_stride = plan.logit_stride;
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case SVA_DTYPE_F32: return decode_dims<float>(p, cache->head_dim, plan.cols, a->n_seqs, st);
    case SVA_DTYPE_BF16: return decode_dims<__nv_bfloat16>(p, cache->head_dim, plan.cols, a->n_seqs, st);
    default: return decode_dims<__half>(p, cache->head_dim, plan.cols, a->n_seqs, st);
  }
}
