// Causal attention over whole prompts, packed without padding, with grouped heads.
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
// Bound by fp32 issue: 4 D flops a (query, key) pair at 2 x 128 lanes a cycle and SM.
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
  if (check_prompt(a) != SVA_OK) return 0;
  return 0;
}

extern "C" int sva_prompt_attention(const sva_prompt_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_prompt(a);
  if (rc != SVA_OK) return rc;
  (void)workspace;
  (void)workspace_bytes;
  if (a->n_seqs == 0 || a->n_rows == 0) return SVA_OK;
  if (!a->query || !a->out || !a->cu_seqlens || (a->n_key_rows > 0 && (!a->keys || !a->values)))
    return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  const PromptParams p{a->n_seqs, a->n_heads, a->n_kv_heads, a->n_heads / a->n_kv_heads, a->head_dim, a->causal,
                       a->softmax_scale * 1.4426950408889634f, a->n_rows, a->n_key_rows, a->query, a->q_row_stride,
                       a->q_head_stride, a->keys, a->k_row_stride, a->k_head_stride, a->values, a->v_row_stride,
                       a->v_head_stride, a->cu_seqlens, a->cu_seqlens_k ? a->cu_seqlens_k : a->cu_seqlens, a->out,
                       a->out_row_stride, a->out_head_stride, a->lse, a->status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case SVA_DTYPE_F32: return simt_dims<float>(p, st);
    case SVA_DTYPE_BF16: return simt_dims<__nv_bfloat16>(p, st);
    default: return simt_dims<__half>(p, st);
  }
}
