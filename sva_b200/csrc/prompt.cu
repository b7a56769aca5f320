// Causal attention over whole prompts, packed without padding, with grouped heads.
#include <cuda.h>

#include <type_traits>

#include "async_copy.cuh"
#include "sva_common.cuh"
#include "sva_internal.h"

namespace sva {

struct PromptParams {
  int n_seqs, n_heads, n_kv, groups, head_dim, causal;
  float scale_log2;
  int64_t n_rows, n_keys;
  const void* q;
  int64_t q_row, q_head;
  const void* k;
  int64_t k_row, k_head;
  const void* v;
  int64_t v_row, v_head;
  const int64_t* cu;
  const int64_t* cu_k;
  void* out;
  int64_t o_row, o_head;
  float* lse;
  int* status;
};

struct Sequence {
  int64_t q0, k0;    // first rows
  int len_q, len_k;  // rows
};

__device__ __forceinline__ Sequence sequence_of(const PromptParams& p, int b) {
  auto bound = [](int64_t x, int64_t low, int64_t high) { return x < low ? low : (x > high ? high : x); };
  Sequence s;
  s.q0 = bound(__ldg(p.cu + b), 0, p.n_rows);
  s.len_q = (int)(bound(__ldg(p.cu + b + 1), s.q0, p.n_rows) - s.q0);
  s.k0 = bound(__ldg(p.cu_k + b), 0, p.n_keys);
  s.len_k = (int)(bound(__ldg(p.cu_k + b + 1), s.k0, p.n_keys) - s.k0);
  return s;
}

// The sequence and the tile in it of tile number `slot`, counting ceil(len_q / rows) tiles for each
// sequence in turn; false when there are fewer tiles.  A whole warp calls it.
__device__ __forceinline__ bool find_tile(const PromptParams& p, int64_t slot, int rows, int* seq, int* tile) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < p.n_seqs; b0 += 32) {
    int n = 0;
    if (b0 + lane < p.n_seqs) n = (sequence_of(p, b0 + lane).len_q + rows - 1) / rows;
    const int incl = warp_incl_scan(n);
    const int total = __shfl_sync(0xFFFFFFFFu, incl, 31);
    if (slot < total) {
      const uint32_t m = __ballot_sync(0xFFFFFFFFu, slot < incl);
      const int j = __ffs(m) - 1;
      *seq = b0 + j;
      *tile = (int)slot - __shfl_sync(0xFFFFFFFFu, incl - n, j);
      return true;
    }
    slot -= total;
  }
  return false;
}

// ---------------------------------------------------------------------------------------
// fp32 on the CUDA cores: every type, head size and stride
// ---------------------------------------------------------------------------------------
// One CTA takes 64 queries of one head and walks the keys in tiles of 64 with a running maximum and
// sum per row; a thread owns 4 rows x 4 keys of the scores and 4 rows x D / 16 channels of the output.
// Bound by instruction issue (73 % of the cycles), of which FMAs are less than half: the output loop loads its 4 weights and
// D / 64 vectors and tests a limit a row for every 16 D / 64 of them.  8192 tokens of 9 / 3 heads of 64 take 3.1 ms (25 TFLOP/s, a
// third of the fp32 rate).
constexpr int kSimtRows = 64;

template <typename T, int DP>
__global__ void __launch_bounds__(256) prompt_simt_kernel(const PromptParams p) {
  constexpr int kPitch = DP + 4, kSPitch = kSimtRows + 4;
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;
  float* sk = sq + kSimtRows * kPitch;
  float* sv = sk + kSimtRows * kPitch;
  float* sp = sv + kSimtRows * kPitch;  // [row][key]
  __shared__ int where[3];
  const int tid = threadIdx.x, tr = tid / 16, tc = tid % 16;
  const int h = blockIdx.y, kvh = h / p.groups, D = p.head_dim;
  if (tid < 32) {
    int b = 0, tile = 0;
    const bool any = find_tile(p, blockIdx.x, kSimtRows, &b, &tile);
    if (tid == 0) where[0] = any, where[1] = b, where[2] = tile;
  }
  __syncthreads();
  if (!where[0]) return;
  const Sequence s = sequence_of(p, where[1]);
  const int r0 = where[2] * kSimtRows, rows = min(kSimtRows, s.len_q - r0);
  const T* q = reinterpret_cast<const T*>(p.q) + (s.q0 + r0) * p.q_row + h * p.q_head;
  const T* k = reinterpret_cast<const T*>(p.k) + s.k0 * p.k_row + kvh * p.k_head;
  const T* v = reinterpret_cast<const T*>(p.v) + s.k0 * p.v_row + kvh * p.v_head;
  for (int e = tid; e < kSimtRows * DP; e += 256) {
    const int r = e / DP, d = e % DP;
    sq[r * kPitch + d] = (r < rows && d < D) ? to_f32<T>(q[r * p.q_row + d]) : 0.f;
  }
  int lim[4];  // keys that each of the thread's rows sees
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + tr * 4 + i;
    lim[i] = p.causal ? max(0, min(s.len_k, r + s.len_k - s.len_q + 1)) : s.len_k;
  }
  const int last = p.causal ? max(0, min(s.len_k, r0 + rows + s.len_k - s.len_q)) : s.len_k;
  float m[4], l[4], o[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) o[i][c] = 0.f;
  }
  for (int k0 = 0; k0 < last; k0 += kSimtRows) {
    __syncthreads();
    const int n = min(kSimtRows, last - k0);
    for (int e = tid; e < kSimtRows * DP; e += 256) {
      const int r = e / DP, d = e % DP;
      const bool in = r < n && d < D;
      sk[r * kPitch + d] = in ? to_f32<T>(k[(int64_t)(k0 + r) * p.k_row + d]) : 0.f;
      sv[r * kPitch + d] = in ? to_f32<T>(v[(int64_t)(k0 + r) * p.v_row + d]) : 0.f;
    }
    __syncthreads();
    float x[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 a[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sq + (tr * 4 + i) * kPitch + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const float4*>(sk + (tc + 16 * j) * kPitch + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[i][j] = fmaf(a[i].x, c[j].x, fmaf(a[i].y, c[j].y, fmaf(a[i].z, c[j].z, fmaf(a[i].w, c[j].w, x[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i][j] = k0 + tc + 16 * j < lim[i] ? x[i][j] * p.scale_log2 : -INFINITY;
        top = fmaxf(top, x[i][j]);
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
      const float m_new = fmaxf(m[i], top), use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[i] - use);
      m[i] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(x[i][j] - use);
        sum += e;
        sp[(tr * 4 + i) * kSPitch + tc + 16 * j] = e;
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
      l[i] = fmaf(l[i], alpha, sum);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) o[i][c] *= alpha;
    }
    __syncwarp();  // a row's 16 threads are one half-warp
    for (int j = 0; j < n; ++j) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = sp[(tr * 4 + i) * kSPitch + j];
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 y = *reinterpret_cast<const float4*>(sv + j * kPitch + c * 64 + tc * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (k0 + j >= lim[i]) continue;  // a value that the row may not see can be anything
          o[i][4 * c] = fmaf(w[i], y.x, o[i][4 * c]);
          o[i][4 * c + 1] = fmaf(w[i], y.y, o[i][4 * c + 1]);
          o[i][4 * c + 2] = fmaf(w[i], y.z, o[i][4 * c + 2]);
          o[i][4 * c + 3] = fmaf(w[i], y.w, o[i][4 * c + 3]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = tr * 4 + i;
    if (r >= rows) continue;
    const bool none = lim[i] == 0;
    const float inv = none ? 0.f : 1.f / l[i];
    T* dst = reinterpret_cast<T*>(p.out) + (s.q0 + r0 + r) * p.o_row + h * p.o_head;
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c * 64 + tc * 4 + e < D) dst[c * 64 + tc * 4 + e] = from_f32<T>(none ? 0.f : o[i][4 * c + e] * inv);
    if (p.lse && tc == 0)
      p.lse[h * p.n_rows + s.q0 + r0 + r] = none ? -INFINITY : (m[i] + log2f(l[i])) * 0.6931471805599453f;
  }
}

// ---------------------------------------------------------------------------------------
// bf16 and fp16 on the tensor cores
// ---------------------------------------------------------------------------------------
// One CTA takes two tiles A and B of 128 rows, a row being one (token, head of the group) pair: with G heads a
// group a tile is 128 / G tokens, so that every head of a group shares the K and V tiles and few tokens
// fill a tile.  Roles: warps 0-3 and 4-7 the softmax of A and of B (a thread owns a row), warp 8 the copies,
// warp 9 the MMAs, warps 10 and 11 the value rows that some row may not see.
//   S = Q K^T   128 x 128 x D, both operands in shared memory, S in tensor memory (fp32)
//   P = exp2(scale log2e S - m) as 16-bit numbers in tensor memory: beside S (D = 64), or over it (D = 128)
//   O += P V    128 x D x 128, P in tensor memory
// While one tile is in its softmax the tensor cores work for the other.  The maximum m that P is relative to
// moves only when a row's maximum grew by more than 2^8, so O is rescaled rarely.  fp16 weights are 2^7 larger (at most 2^15): those
// down to 2^-21 of the row's maximum keep all their bits.
// Measured (device): 8192 tokens, 9 / 3 heads of 64, bf16: 120 us = 644 TFLOP/s of the causal half; 2 x 61 tokens behind 30011
// keys, 16 / 2 heads of 128: 53 us.  With 64 channels the exponential unit (16 a cycle and SM, 1024 cycles a tile and block
// against 512 of MMAs) is the busiest and about 76 % so in the loop, a block of both tiles taking about 2700 cycles; issue is not what
// bounds it (36 % of the active cycles).
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;  // weights are 2^kLift times exp2(scale log2e S - m)
constexpr int kTcRows = 128;   // rows of a tile, keys of a block
constexpr int kTcThreads = 384;

template <int DP>
struct TcShape {
  static constexpr int kHalves = DP / 64;                       // 64-channel halves: 128-byte swizzled rows
  static constexpr int kTileBytes = kTcRows * 128 * kHalves;    // one Q, K or V tile
  static constexpr int kStages = DP == 64 ? 3 : 2;
  static constexpr int kSmem = 1024 + kTileBytes * (2 + 2 * kStages);
  // Tensor memory (512 columns): S of A and B, O of A and B.  With 64 channels there is room for P beside S: the next
  // block's S is then worked out while this block is in its softmax, and no warp waits for the tensor cores.  With 128, P
  // takes the place of S.
  static constexpr bool kApart = DP == 64;
  __host__ __device__ static constexpr uint32_t s_col(int x) { return 128u * x; }
  __host__ __device__ static constexpr uint32_t o_col(int x) { return 256u + DP * x; }
  __host__ __device__ static constexpr uint32_t p_col(int x) { return kApart ? 384u + 64u * x : 128u * x; }
};

struct TcBars {
  uint64_t q_full[2], s_full[2], s_read[2], p_full[2], pv_done[2];
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3], v_go[3], v_clean[3];
  uint64_t mma_end;
};

// Bounded wait of a whole warp: true where every lane saw the phase complete.  Lanes that decided apart would part ways before
// instructions that take the whole warp.
__device__ __forceinline__ bool warp_wait(const uint64_t& bar, int turn, volatile int* failed) {
  return __all_sync(0xFFFFFFFFu, mbar_wait_or(smem_u32(&bar), turn & 1, failed)) != 0;
}

struct PromptTcParams {
  PromptParams p;
  CUtensorMap q, k, v;
  int tokens;     // tokens of a tile: 128 / groups
  int n_slots;    // CTA slots: at least the number of tile pairs
  int splits;     // CTAs that share a tile pair's keys
  float* part_o;  // [slot][kv head][split][256][DP]
  float* part_ml; // [slot][kv head][split][256][2]
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The largest of three, one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Key blocks [first, end) of a tile in one split.
__device__ __forceinline__ void split_range(int blocks, int splits, int split, int* first, int* end) {
  const int per = (blocks + splits - 1) / splits;
  *first = min(blocks, split * per);
  *end = min(blocks, *first + per);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTcThreads, 1) prompt_tc_kernel(const __grid_constant__ PromptTcParams tp) {
  using S = TcShape<DP>;
  const PromptParams& p = tp.p;
  extern __shared__ unsigned char smem_raw[];
  __shared__ TcBars bars;
  __shared__ uint32_t tmem_base;
  __shared__ int failed_flag, any_bad;
  __shared__ int bad_from[3][DP];  // the first NaN, inf and -inf of a channel that some row may not see
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // heaviest tiles first: later tiles of a sequence see more keys
  const int id = blockIdx.x;
  const int split = id % tp.splits, h = id / tp.splits % p.n_kv, slot = tp.n_slots - 1 - id / tp.splits / p.n_kv;
  int b, pair;
  if (!find_tile(p, slot, 2 * tp.tokens, &b, &pair)) return;
  const Sequence s = sequence_of(p, b);
  const int tok0 = pair * 2 * tp.tokens;
  auto limit_of = [&](int tok) {  // keys that a token sees
    return p.causal ? max(0, min(s.len_k, tok + s.len_k - s.len_q + 1)) : s.len_k;
  };
  int blocks[2], first = 0, end = 0, stop[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int last = min(s.len_q, tok0 + (x + 1) * tp.tokens) - 1;
    blocks[x] = last >= tok0 + x * tp.tokens ? (limit_of(last) + kTcRows - 1) / kTcRows : 0;
  }
  split_range(max(blocks[0], blocks[1]), tp.splits, split, &first, &end);
#pragma unroll
  for (int x = 0; x < 2; ++x) stop[x] = min(blocks[x], end);  // tile x works on blocks [first, stop[x])
  const int masked = limit_of(tok0) / kTcRows;                // blocks from here on hold keys that some row may not see
  // v_go and v_clean count the masked blocks of a stage alone
  auto clean_turn = [&](int j) { return (j - max(first, masked)) / S::kStages; };

  unsigned char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* sq = base;
  unsigned char* sk = sq + 2 * S::kTileBytes;
  unsigned char* sv = sk + S::kStages * S::kTileBytes;
  volatile int* failed = &failed_flag;

  if (tid == 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&bars.q_full[x]), 1);
      mbar_init(smem_u32(&bars.s_full[x]), 1);
      mbar_init(smem_u32(&bars.s_read[x]), 128);
      mbar_init(smem_u32(&bars.p_full[x]), 128);
      mbar_init(smem_u32(&bars.pv_done[x]), 1);
    }
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(smem_u32(&bars.k_full[i]), 1);
      mbar_init(smem_u32(&bars.k_empty[i]), 1);
      mbar_init(smem_u32(&bars.v_full[i]), 1);
      mbar_init(smem_u32(&bars.v_empty[i]), 1);
      mbar_init(smem_u32(&bars.v_go[i]), 1);
      mbar_init(smem_u32(&bars.v_clean[i]), 2);
    }
    mbar_init(smem_u32(&bars.mma_end), 1);
    mbar_fence_init();
    failed_flag = 0;
    any_bad = 0;
  }
  for (int d = tid; d < 3 * DP; d += kTcThreads) (&bad_from[0][0])[d] = 0x7FFFFFFF;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  // the copies that lane 0 of warp 8 has issued: of both K and V below block `issued`, and of K for that block
  int issued = first;
  bool k_issued = false;

  // registers from the last four warps to the softmax: 2 x 200 + 96 of the 3 x 168 that the CTA was launched with
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
  if (warp == 8) {
    // ---- copies ----
    if (lane == 0) {
      const uint32_t q_bytes = 128u * S::kHalves * (uint32_t)(tp.tokens * p.groups);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (stop[x] <= first) continue;
        const uint32_t bar = smem_u32(&bars.q_full[x]);
        mbar_expect_tx(bar, q_bytes);
#pragma unroll
        for (int c = 0; c < S::kHalves; ++c)
          tma_load_4d(smem_u32(sq + x * S::kTileBytes + c * kTcRows * 128), &tp.q, 64 * c, 0, h,
                      (int)(s.q0 + tok0 + x * tp.tokens), bar);
      }
      bool ok = true;
      for (int j = first; j < end && ok; ++j) {
        const int n = j - first, st = n % S::kStages, turn = n / S::kStages;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t empty = smem_u32(kv ? &bars.v_empty[st] : &bars.k_empty[st]);
          const uint32_t full = smem_u32(kv ? &bars.v_full[st] : &bars.k_full[st]);
          if (ok && turn > 0) ok = mbar_wait_or(empty, (turn - 1) & 1, failed);
          if (!ok) break;
          mbar_expect_tx(full, S::kTileBytes);
#pragma unroll
          for (int c = 0; c < S::kHalves; ++c)
            tma_load_3d(smem_u32((kv ? sv : sk) + st * S::kTileBytes + c * kTcRows * 128), kv ? &tp.v : &tp.k, 64 * c, h,
                        (int)(s.k0 + (int64_t)j * kTcRows), full);
          k_issued = kv == 0;
          if (kv) issued = j + 1;
          if (kv && j >= masked) mbar_arrive(smem_u32(&bars.v_go[st]));
        }
      }
    }
  } else if (warp == 9) {
    // ---- MMAs ----
    {
      // a warp-wide maximum is what the compiler knows to be uniform
      auto uniform = [](int v) { return __reduce_max_sync(0xFFFFFFFFu, v); };
      const uint32_t one = elect_one(), tm = (uint32_t)uniform((int)tmem);
      const int count = uniform(end - first), dirty = uniform(max(0, masked - first));
      const int counts[2] = {uniform(stop[0] - first), uniform(stop[1] - first)};
      auto wait = [&](const uint64_t& bar, int turn) { return warp_wait(bar, turn, failed); };
      constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
      constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((kTcRows / 8) << 17) | ((kTcRows / 16) << 24);
      constexpr uint32_t kIdescO =
          (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((DP / 8) << 17) | ((kTcRows / 16) << 24);
      auto scores = [&](int x, int st) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk / 4) * kTcRows * 128 + (kk % 4) * 32;
          tc_mma_ss(tm + S::s_col(x), tc_desc(smem_u32(sq + x * S::kTileBytes) + off, 16),
                    tc_desc(smem_u32(sk + st * S::kTileBytes) + off, 16), kIdescS, kk > 0, one);
        }
        tc_commit(smem_u32(&bars.s_full[x]), one);
      };
      bool ok = true;
      if (count > 0) ok = wait(bars.k_full[0], 0);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (!ok || counts[x] <= 0) continue;
        ok = wait(bars.q_full[x], 0);
        if (ok) scores(x, 0);
      }
      if (ok && count > 0) tc_commit(smem_u32(&bars.k_empty[0]), one);
      for (int n = 0; n < count && ok; ++n) {
        const int st = n % S::kStages, turn = n / S::kStages;
        const int n1 = n + 1, st1 = n1 % S::kStages, turn1 = n1 / S::kStages;
        bool k_ready = false;
        auto next_scores = [&](int x) {
          if (!ok || n + 1 >= counts[x]) return;
          if (!k_ready) ok = wait(bars.k_full[st1], turn1);
          k_ready = true;
          if (ok) scores(x, st1);
        };
        if constexpr (S::kApart) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!ok || n + 1 >= counts[x]) continue;
            ok = wait(bars.s_read[x], n);
            tc_fence_after();
            next_scores(x);
          }
          if (ok && n + 1 < count) tc_commit(smem_u32(&bars.k_empty[st1]), one);
        }
        if (ok) ok = wait(bars.v_full[st], turn);
        // blocks with keys that some row may not see: wait for their value rows to be cleaned
        if (ok && n >= dirty) ok = wait(bars.v_clean[st], (n - dirty) / S::kStages);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok || n >= counts[x]) continue;
          ok = wait(bars.p_full[x], n);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kTcRows / 16; ++kk)
            tc_mma_ts(tm + S::o_col(x), tm + S::p_col(x) + 8 * kk,
                      tc_desc(smem_u32(sv + st * S::kTileBytes) + kk * 2048, kTcRows * 128), kIdescO, n > 0 || kk > 0, one);
          if (S::kApart || n + 1 >= counts[x]) tc_commit(smem_u32(&bars.pv_done[x]), one);
          if constexpr (!S::kApart) next_scores(x);
        }
        if (!ok) break;
        tc_commit(smem_u32(&bars.v_empty[st]), one);
        if (!S::kApart && n + 1 < count) tc_commit(smem_u32(&bars.k_empty[st1]), one);
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---- value rows that some row may not see ----
    // 0 times a non-finite value is NaN, so such values become 0 here.  Rows behind the sequence belong to no
    // one; a non-finite value of the sequence itself is added to its channel at the end in the rows that do see it.
    for (int j = max(first, masked); j < end; ++j) {
      const int n = j - first, st = n % S::kStages, turn = n / S::kStages;
      // the copy of this very block is under way (v_full's phase could be any before that), then complete
      if (!warp_wait(bars.v_go[st], clean_turn(j), failed)) break;
      if (!warp_wait(bars.v_full[st], turn, failed)) break;
      const int from = max(0, limit_of(tok0) - j * kTcRows), valid = s.len_k - j * kTcRows;
      unsigned char* tile = sv + st * S::kTileBytes;
      for (int e = (from * 8) + (warp - 10) * 32 + lane; e < kTcRows * 8; e += 64) {
        const int r = e >> 3, chunk = e & 7;
#pragma unroll
        for (int c = 0; c < S::kHalves; ++c) {
          uint4* at = reinterpret_cast<uint4*>(tile + c * kTcRows * 128 + r * 128 + chunk * 16);
          if (r >= valid) {
            *at = make_uint4(0u, 0u, 0u, 0u);
            continue;
          }
          constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
          uint4 v = *at;
          uint32_t* w = reinterpret_cast<uint32_t*>(&v);
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            bad |= (w[i] & kExp) == kExp || (w[i] & (kExp << 16)) == (kExp << 16);
          if (!bad) continue;
          const int d0 = c * 64 + ((chunk ^ (r & 7)) * 8);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t m = 0xFFFFu << (16 * (i & 1));
            if ((w[i >> 1] & (kExp << (16 * (i & 1)))) == (kExp << (16 * (i & 1)))) {
              const uint32_t u = w[i >> 1] >> (16 * (i & 1)) & 0xFFFFu;
              w[i >> 1] &= ~m;
              atomicMin(&bad_from[(u & 0x7FFFu) != kExp ? 0 : 1 + (u >> 15)][d0 + i], j * kTcRows + r);
            }
          }
          any_bad = 1;
          *at = v;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars.v_clean[st]));
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- softmax: a thread owns a row ----
    const int x = warp >> 2, row = (warp & 3) * 32 + lane;
    const int tok = tok0 + x * tp.tokens + row / p.groups;
    const bool live = row < tp.tokens * p.groups && tok < s.len_q;
    const int limit = live ? limit_of(tok) : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + S::s_col(x) + lanes, to = tmem + S::o_col(x) + lanes, tpr = tmem + S::p_col(x) + lanes;
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = first; j < stop[x]; ++j) {
      const int n = j - first;
      if (!warp_wait(bars.s_full[x], n, failed)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t v[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc_ld32(ts + 32 * c, v + 32 * c);
      tc_wait_ld();
      tc_pin<128>(v);
      if constexpr (S::kApart) {
        tc_fence_before();
        mbar_arrive(smem_u32(&bars.s_read[x]));
      }
      float* f = reinterpret_cast<float*>(v);
      if (j >= masked) {
        const int seen = limit - j * kTcRows;
#pragma unroll
        for (int i = 0; i < 128; ++i) f[i] = i < seen ? f[i] : -INFINITY;
      }
      float top[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) top[i] = f[i];
#pragma unroll
      for (int i = 4; i < 124; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = max3(top[k], f[i + 2 * k], f[i + 2 * k + 1]);
      top[0] = max3(top[0], f[124], f[125]);
      top[1] = max3(top[1], f[126], f[127]);
      const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]) * p.scale_log2;
      const bool grew = mx > m + 8.f;
      // O and P are free once the block before has been added.  (P in the place of S: that S is complete says so.)
      if (S::kApart && n > 0) {
        if (!warp_wait(bars.pv_done[x], n - 1, failed)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      if (__any_sync(0xFFFFFFFFu, grew)) {
        const float m_new = grew ? mx : m;
        const float alpha = grew ? ex2(m - m_new) : 1.f;  // 0 from -inf
        m = m_new;
        l *= alpha;
        if (n > 0) {
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tc_ld32(to + 32 * c, o);
            tc_wait_ld();
            tc_pin<32>(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tc_st32(to + 32 * c, o);
          }
        }
      }
      const float use = m == -INFINITY ? 0.f : m - kLift<T>;
      const uint64_t minus2 = pack2(-use, -use);
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float e0, e1;
          unpack2(fma2(pack2(f[32 * c + 2 * i], f[32 * c + 2 * i + 1]), scale2, minus2), e0, e1);
          e0 = ex2(e0);
          e1 = ex2(e1);
          sum[i & 1] = add2(sum[i & 1], pack2(e0, e1));
          w[i] = pack16<T>(e0, e1);
        }
        tc_st16(tpr + 16 * c, w);
      }
      float s0, s1;
      unpack2(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&bars.p_full[x]));
    }
    const bool any = stop[x] > first;
    if (ok && any) ok = warp_wait(bars.pv_done[x], S::kApart ? stop[x] - first - 1 : 0, failed);
    tc_fence_after();
    const int head = h * p.groups + row % p.groups;
    const int64_t qrow = s.q0 + tok;
    if (!ok && p.status) atomicExch(p.status, SVA_ERR_TIMEOUT);
    const float use = m == -INFINITY ? 0.f : m - kLift<T>;  // what the weights are relative to
    const bool whole = tp.splits == 1;
    const bool none = limit == 0;
    const float inv = none ? 0.f : 1.f / l;
    float* po = nullptr;
    if (!whole) {
      const int64_t at = (((int64_t)slot * p.n_kv + h) * tp.splits + split) * 256 + x * 128 + row;
      po = tp.part_o + at * DP;
      tp.part_ml[2 * at] = m - kLift<T>;
      tp.part_ml[2 * at + 1] = ok ? l : NAN;
    } else if (live && p.lse) {
      p.lse[head * p.n_rows + qrow] = none ? -INFINITY : (use + log2f(l)) * 0.6931471805599453f;
    }
    T* dst = reinterpret_cast<T*>(p.out) + qrow * p.o_row + head * p.o_head;
    const bool vec = p.head_dim % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.out) | (p.o_row * sizeof(T)) | (p.o_head * sizeof(T))) & 15) == 0;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      uint32_t o[32];
      if (any && ok) {
        tc_ld32(to + 32 * c, o);
        tc_wait_ld();
        tc_pin<32>(o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = ok ? 0u : 0x7FC00000u;
      }
      if (any_bad) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float y = __uint_as_float(o[i]);
          if (limit > bad_from[0][32 * c + i]) y = NAN;
          if (limit > bad_from[1][32 * c + i]) y += INFINITY;
          if (limit > bad_from[2][32 * c + i]) y -= INFINITY;
          o[i] = __float_as_uint(y);
        }
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<uint4*>(po + 32 * c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        continue;
      }
      if (!live) continue;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        w[i] = none ? 0u : pack16<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
      if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (32 * c + 8 * i < p.head_dim)
            reinterpret_cast<uint4*>(dst + 32 * c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const unsigned short u = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
          if (32 * c + i < p.head_dim) reinterpret_cast<unsigned short*>(dst)[32 * c + i] = u;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*failed) {
    // Some role gave up: what is in flight lands, and every MMA issued ends, before the shared and the tensor memory go to
    // another CTA.  (Else the others have waited for all of it.)
    if (warp == 8 && lane == 0) {
      for (int x = 0; x < 2; ++x)
        if (stop[x] > first) mbar_wait(smem_u32(&bars.q_full[x]), 0);
      for (int j = max(first, issued - S::kStages); j < min(end, issued + 1); ++j) {
        const int n = j - first, st = n % S::kStages, turn = n / S::kStages;
        if (j < issued || k_issued) mbar_wait(smem_u32(&bars.k_full[st]), turn & 1);
        if (j < issued) mbar_wait(smem_u32(&bars.v_full[st]), turn & 1);
      }
    } else if (warp == 9) {
      tc_commit(smem_u32(&bars.mma_end), elect_one());
      mbar_wait(smem_u32(&bars.mma_end), 0);
    }
  }
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the splits of a tile pair: a warp a row.
template <typename T, int DP>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ PromptTcParams tp) {
  const PromptParams& p = tp.p;
  const int lane = threadIdx.x & 31;
  const int slot = blockIdx.x, h = blockIdx.y;
  int b, pair;
  if (!find_tile(p, slot, 2 * tp.tokens, &b, &pair)) return;
  const Sequence s = sequence_of(p, b);
  const int tok0 = pair * 2 * tp.tokens;
  const int i = blockIdx.z * 8 + (threadIdx.x >> 5);
  const int x = i >> 7, row = i & 127, tok = tok0 + x * tp.tokens + row / p.groups;
  if (row >= tp.tokens * p.groups || tok >= s.len_q) return;
  const int64_t at = ((int64_t)slot * p.n_kv + h) * tp.splits * 256 + i;
  float m = -INFINITY;
  for (int k = 0; k < tp.splits; ++k) m = fmaxf(m, tp.part_ml[2 * (at + k * 256)]);
  const float use = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[DP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) o[c] = 0.f;
  for (int k = 0; k < tp.splits; ++k) {
    const int64_t a = at + k * 256;
    const float f = ex2(tp.part_ml[2 * a] - use);
    l = fmaf(f, tp.part_ml[2 * a + 1], l);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) o[c] = fmaf(f, tp.part_o[a * DP + c * 32 + lane], o[c]);
  }
  const int limit = p.causal ? max(0, min(s.len_k, tok + s.len_k - s.len_q + 1)) : s.len_k;
  const int head = h * p.groups + row % p.groups;
  const int64_t qrow = s.q0 + tok;
  T* dst = reinterpret_cast<T*>(p.out) + qrow * p.o_row + head * p.o_head;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
    if (c * 32 + lane < p.head_dim) dst[c * 32 + lane] = from_f32<T>(limit == 0 ? 0.f : o[c] / l);
  if (p.lse && lane == 0)
    p.lse[head * p.n_rows + qrow] = limit == 0 ? -INFINITY : (use + log2f(l)) * 0.6931471805599453f;
}

static int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SVA_OK : set_error(SVA_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T, int DP>
static int launch_simt(const PromptParams& p, cudaStream_t st) {
  const int smem = (3 * kSimtRows * (DP + 4) + kSimtRows * (kSimtRows + 4)) * 4;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(prompt_simt_kernel<T, DP>), smem);
  if (rc != SVA_OK) return rc;
  const int64_t tiles = p.n_rows / kSimtRows + p.n_seqs;
  prompt_simt_kernel<T, DP><<<dim3((unsigned)tiles, p.n_heads), 256, smem, st>>>(p);
  return launched();
}

template <typename T>
static int simt_dims(const PromptParams& p, cudaStream_t st) {
  if (p.head_dim <= 64) return launch_simt<T, 64>(p, st);
  if (p.head_dim <= 128) return launch_simt<T, 128>(p, st);
  return launch_simt<T, 256>(p, st);
}

// ---------------------------------------------------------------------------------------
// host side of the tensor-core path
// ---------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// A tensor map over 16-bit rows; dimensions of one element may have any stride.
static bool encode(CUtensorMap* map, int dtype, int rank, const void* ptr, const int64_t* dims, const int64_t* strides,
                   const uint32_t* box) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  cuuint64_t d[4], st[3];
  cuuint32_t bx[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i], bx[i] = box[i];
  for (int i = 1; i < rank; ++i) st[i - 1] = dims[i] == 1 ? 16 * ((cuuint64_t)dims[0] * 2 / 16 + 1) : (cuuint64_t)strides[i - 1] * 2;
  return fn(map, dtype == SVA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
            const_cast<void*>(ptr), d, st, bx, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tensor-core path takes 16-bit rows of a multiple of 8 channels up to 128, at most 128 heads a group, a
// positive scale, and pointers and strides that the tensor copies can address (multiples of 16 bytes; no
// broadcast dimension).
static bool tc_fits(const sva_prompt_args* a) {
  if (a->dtype == SVA_DTYPE_F32 || a->head_dim % 8 || a->head_dim > 128 || a->n_heads / a->n_kv_heads > kTcRows) return false;
  if (!(a->softmax_scale > 0.f) || !(a->softmax_scale < 1e30f) || a->n_key_rows == 0) return false;
  const void* ptrs[3] = {a->query, a->keys, a->values};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16) return false;
  const int64_t row[3] = {a->q_row_stride, a->k_row_stride, a->v_row_stride};
  const int64_t head[3] = {a->q_head_stride, a->k_head_stride, a->v_head_stride};
  for (int i = 0; i < 3; ++i) {
    const int64_t rows = i ? a->n_key_rows : a->n_rows, heads = i ? a->n_kv_heads : a->n_heads;
    if (rows > 1 && (row[i] <= 0 || row[i] % 8 || row[i] >= (1ll << 38))) return false;
    if (heads > 1 && (head[i] <= 0 || head[i] % 8 || head[i] >= (1ll << 32))) return false;
  }
  return true;
}

struct TcPlan {
  int dp, tokens, slots, splits;
  size_t ml, total;
};

static TcPlan plan_tc(const sva_prompt_args* a) {
  TcPlan t{};
  t.dp = a->head_dim <= 64 ? 64 : 128;
  t.tokens = kTcRows / (a->n_heads / a->n_kv_heads);
  t.slots = (int)(a->n_rows / (2 * t.tokens) + a->n_seqs);
  // Few tiles: their keys are shared out, at least 4 blocks of 128 to a CTA (by the mean length; the lengths are
  // on the device)
  const int64_t ctas = (int64_t)t.slots * a->n_kv_heads;
  const int64_t blocks = (a->n_key_rows / std::max(1, a->n_seqs) + kTcRows - 1) / kTcRows;
  t.splits = (int)std::max<int64_t>(1, std::min<int64_t>(148 / ctas, blocks / 4));
  if (t.splits > 1) {
    const size_t rows = (size_t)ctas * t.splits * 256;
    t.ml = rows * t.dp * 4;
    t.total = t.ml + rows * 2 * 4;
  }
  return t;
}

template <typename T, int DP>
static int launch_tc(const PromptTcParams& tp, cudaStream_t st) {
  using S = TcShape<DP>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(prompt_tc_kernel<T, DP>), S::kSmem);
  if (rc != SVA_OK) return rc;
  const int64_t ctas = (int64_t)tp.n_slots * tp.p.n_kv * tp.splits;
  if (ctas > 0x7FFFFFFFll) return set_error(SVA_ERR_SHAPE, "too many tiles");
  prompt_tc_kernel<T, DP><<<(unsigned)ctas, kTcThreads, S::kSmem, st>>>(tp);
  rc = launched();
  if (rc != SVA_OK || tp.splits == 1) return rc;
  prompt_join_kernel<T, DP><<<dim3(tp.n_slots, tp.p.n_kv, 32), 256, 0, st>>>(tp);
  return launched();
}

static int check_prompt(const sva_prompt_args* a) {
  if (!a) return set_error(SVA_ERR_SHAPE, "the arguments are null");
  if (a->n_heads <= 0 || a->n_kv_heads <= 0 || a->n_heads % a->n_kv_heads || a->n_heads > 65535)
    return set_error(SVA_ERR_SHAPE, "n_heads must be a multiple of n_kv_heads, at most 65535");
  if (a->head_dim <= 0 || a->head_dim > kMaxHeadDim) return set_error(SVA_ERR_SHAPE, "head_dim must be in 1..256");
  if (a->n_seqs < 0 || a->n_rows < 0 || a->n_key_rows < 0 || a->n_rows >= (1ll << 31) || a->n_key_rows >= (1ll << 31) ||
      a->n_seqs > (1 << 24))
    return set_error(SVA_ERR_SHAPE, "row counts must be below 2^31, and n_seqs at most 2^24");
  if (a->dtype < 0 || a->dtype > 2) return set_error(SVA_ERR_DTYPE, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  return SVA_OK;
}

}  // namespace sva

using namespace sva;

extern "C" size_t sva_prompt_attention_workspace_size(const sva_prompt_args* a) {
  if (check_prompt(a) != SVA_OK || a->n_seqs == 0 || a->n_rows == 0 || !tc_fits(a)) return 0;
  return plan_tc(a).total;
}

extern "C" int sva_prompt_attention(const sva_prompt_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_prompt(a);
  if (rc != SVA_OK) return rc;
  if (a->n_seqs == 0 || a->n_rows == 0) return SVA_OK;
  if (!a->query || !a->out || !a->cu_seqlens || (a->n_key_rows > 0 && (!a->keys || !a->values)))
    return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  const PromptParams p{a->n_seqs, a->n_heads, a->n_kv_heads, a->n_heads / a->n_kv_heads, a->head_dim, a->causal,
                       a->softmax_scale * 1.4426950408889634f, a->n_rows, a->n_key_rows, a->query, a->q_row_stride,
                       a->q_head_stride, a->keys, a->k_row_stride, a->k_head_stride, a->values, a->v_row_stride,
                       a->v_head_stride, a->cu_seqlens, a->cu_seqlens_k ? a->cu_seqlens_k : a->cu_seqlens, a->out,
                       a->out_row_stride, a->out_head_stride, a->lse, a->status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tc_fits(a)) {
    const TcPlan plan = plan_tc(a);
    if (plan.total > 0 && (!workspace || workspace_bytes < plan.total)) return set_error(SVA_ERR_WORKSPACE, "workspace too small");
    PromptTcParams tp{};
    tp.p = p;
    const int64_t qd[4] = {a->head_dim, p.groups, a->n_kv_heads, a->n_rows};
    const int64_t qs[3] = {a->q_head_stride, a->q_head_stride * p.groups, a->q_row_stride};
    const uint32_t qb[4] = {64, (uint32_t)p.groups, 1, (uint32_t)plan.tokens};
    const int64_t kd[3] = {a->head_dim, a->n_kv_heads, a->n_key_rows};
    const int64_t ks[2] = {a->k_head_stride, a->k_row_stride}, vs[2] = {a->v_head_stride, a->v_row_stride};
    const uint32_t kb[3] = {64, 1, kTcRows};
    if (encode(&tp.q, a->dtype, 4, a->query, qd, qs, qb) && encode(&tp.k, a->dtype, 3, a->keys, kd, ks, kb) &&
        encode(&tp.v, a->dtype, 3, a->values, kd, vs, kb)) {
      tp.tokens = plan.tokens;
      tp.n_slots = plan.slots;
      tp.splits = plan.splits;
      tp.part_o = static_cast<float*>(workspace);
      tp.part_ml = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + plan.ml);
      if (a->dtype == SVA_DTYPE_BF16)
        return plan.dp == 64 ? launch_tc<__nv_bfloat16, 64>(tp, st) : launch_tc<__nv_bfloat16, 128>(tp, st);
      return plan.dp == 64 ? launch_tc<__half, 64>(tp, st) : launch_tc<__half, 128>(tp, st);
    }
  }
  switch (a->dtype) {
    case SVA_DTYPE_F32: return simt_dims<float>(p, st);
    case SVA_DTYPE_BF16: return simt_dims<__nv_bfloat16>(p, st);
    default: return simt_dims<__half>(p, st);
  }
}
