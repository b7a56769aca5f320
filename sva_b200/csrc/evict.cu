// Eviction from a cache by accumulated attention weight: which rows stay, and moving them together.
#include "sva_common.cuh"
#include "sva_internal.h"

namespace sva {

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;         // 11 bits of the ordered key a pass: 3 passes cover 32 bits
constexpr int kMoveThreads = 256;
constexpr int kMoveSmem = 96 * 1024;

struct EvictParams {
  int n_seqs, n_kv, n_arrays;
  int64_t max_len, keep, recent;
  const int64_t* seq_lens;
  const float* weights;
  int64_t w_seq, w_head;
  float* dst_weights;
  int64_t dw_seq, dw_head, dw_width;
  int64_t src_pages, src_rows, dst_pages, dst_rows;
  const int32_t* src_table;
  int64_t src_table_stride, src_table_cols;
  const int32_t* dst_table;
  int64_t dst_table_stride, dst_table_cols;
  int32_t* kept;
  int64_t* lens_out;
  int32_t* counts;  // rows that stay, per problem
  sva_evict_array arrays[SVA_EVICT_MAX_ARRAYS];
};

// The weights' order as unsigned numbers, NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0xFFFFFFFFu : ordered_key(w); }

constexpr int kSelKeys = 49152;  // ordered keys held in shared memory: up to so many old rows are read once

// One CTA per (sequence, kv head).  Radix select of the need-th largest weight among the old rows, then one pass in index
// order: rows above it stay, and of the rows equal to it the first ones.  A warp owns a stretch of the rows, so that the
// order needs one scan over the warps and ballots within them.  Latency bound: 25 us for 128 problems of 9001 to 16385
// rows.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p, int room) {
  extern __shared__ __align__(16) uint32_t keys[];  // [room]
  __shared__ int hist[kBins];
  __shared__ int scratch[kSelThreads / 32 + 1];
  __shared__ int warp_above[kSelThreads / 32], warp_equal[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int problem = blockIdx.x, b = problem / p.n_kv, h = problem % p.n_kv;
  pdl_launch_dependents();
  int64_t n = __ldg(p.seq_lens + b);
  n = n < 0 ? 0 : (n > p.max_len ? p.max_len : n);
  int32_t* kept = p.kept + (int64_t)problem * p.keep;
  const int stay = (int)(n < p.keep ? n : p.keep);
  if (tid == 0) p.counts[problem] = stay;
  for (int64_t j = stay + tid; j < p.keep; j += kSelThreads) kept[j] = -1;
  if (n <= p.keep) {
    for (int j = tid; j < stay; j += kSelThreads) kept[j] = j;
    return;
  }
  const int old = (int)(n - p.recent);
  int need = (int)(p.keep - p.recent);
  for (int j = tid; j < (int)p.recent; j += kSelThreads) kept[need + j] = old + j;
  if (need == 0) return;
  const float* w = p.weights + b * p.w_seq + h * p.w_head;

  // this warp's rows: first + 32 i + lane, i < steps
  const int steps = (old + kSelThreads - 1) / kSelThreads;
  const int64_t first = (int64_t)warp * steps * 32 + lane;
  const bool held = old <= room;
  if (held) {
#pragma unroll 4
    for (int r = tid; r < old; r += kSelThreads) keys[r] = weight_key(__ldg(w + r));
    __syncthreads();
  }
  // f(key, row, whether there is such a row) for the lane's rows in order, by the whole warp together
  auto each = [&](auto&& f) {
#pragma unroll 2
    for (int i = 0; i < steps; ++i) {
      const int64_t r = first + 32 * (int64_t)i;
      const bool there = r < old;
      f(there ? (held ? keys[r] : weight_key(__ldg(w + r))) : 0u, (int)r, there);
    }
  };

  uint32_t prefix = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), above = pass == 1 ? 21 : 10;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    each([&](uint32_t k, int, bool there) {
      if (there && (pass == 0 || (k >> above) == prefix)) atomicAdd(&hist[(k >> shift) & mask], 1);
    });
    __syncthreads();
    // bins from the top: thread i owns bins 2047 - 2i and 2046 - 2i
    const int hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
    int total;
    const int before = block_excl_scan(hi + lo, scratch, &total);
    if (before < need && need <= before + hi) {
      s_prefix = (prefix << (pass == 2 ? 10 : 11)) | (uint32_t)(kBins - 1 - 2 * tid);
      s_need = need - before;
    } else if (before + hi < need && need <= before + hi + lo) {
      s_prefix = (prefix << (pass == 2 ? 10 : 11)) | (uint32_t)(kBins - 2 - 2 * tid);
      s_need = need - before - hi;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    __syncthreads();
  }
  // `prefix` is the need-th largest key; `need` of the rows equal to it stay
  int above = 0, equal = 0;
  each([&](uint32_t k, int, bool there) {
    above += __popc(__ballot_sync(0xFFFFFFFFu, there && k > prefix));
    equal += __popc(__ballot_sync(0xFFFFFFFFu, there && k == prefix));
  });
  if (lane == 0) warp_above[warp] = above, warp_equal[warp] = equal;
  __syncthreads();
  // rows above and equal to it in the warps before this one
  const int wa = warp_incl_scan(warp_above[lane]), we = warp_incl_scan(warp_equal[lane]);
  int at_above = __shfl_sync(0xFFFFFFFFu, wa - warp_above[lane], warp);
  int at_equal = __shfl_sync(0xFFFFFFFFu, we - warp_equal[lane], warp);
  const uint32_t before = (1u << lane) - 1u;
  each([&](uint32_t k, int row, bool there) {
    const bool is_above = there && k > prefix, is_equal = there && k == prefix;
    const uint32_t ma = __ballot_sync(0xFFFFFFFFu, is_above), me = __ballot_sync(0xFFFFFFFFu, is_equal);
    const int a = at_above + __popc(ma & before), e = at_equal + __popc(me & before);
    if (is_above || (is_equal && e < need)) kept[a + min(e, need)] = row;
    at_above += __popc(ma);
    at_equal += __popc(me);
  });
}

__device__ __forceinline__ int64_t page_row(const int32_t* table, int64_t stride, int64_t cols, int64_t pages,
                                            int64_t rows, int b, int64_t l, int64_t* r) {
  int64_t page = b;
  *r = l;
  if (table) {
    const int64_t c = l / rows;
    if (c >= cols) return -1;
    page = __ldg(table + b * stride + c);
    *r = l - c * rows;
  }
  return (page < 0 || page >= pages || *r >= rows) ? -1 : page;
}

template <typename V>
__device__ __forceinline__ void move_rows(const EvictParams& p, const sva_evict_array& a, const int32_t* kept, int b,
                                          int h, int j0, int j1, bool in_place, unsigned char* smem) {
  const int units = (int)(a.row_bytes / sizeof(V));
  auto src_of = [&](int j) -> const V* {
    int64_t r;
    const int64_t page = page_row(p.src_table, p.src_table_stride, p.src_table_cols, p.src_pages, p.src_rows, b, kept[j], &r);
    if (page < 0) return nullptr;
    return reinterpret_cast<const V*>(static_cast<const unsigned char*>(a.src) + page * a.src_page_stride +
                                      h * a.src_head_stride + r * a.row_bytes);
  };
  auto dst_of = [&](int j) -> V* {
    int64_t r;
    const int64_t page = page_row(p.dst_table, p.dst_table_stride, p.dst_table_cols, p.dst_pages, p.dst_rows, b, j, &r);
    if (page < 0) return nullptr;
    return reinterpret_cast<V*>(static_cast<unsigned char*>(a.dst) + page * a.dst_page_stride + h * a.dst_head_stride +
                                r * a.row_bytes);
  };
  V* buf = reinterpret_cast<V*>(smem);
  const int total = (j1 - j0) * units;
  if (!in_place && units <= kMoveThreads && !p.src_table && !p.dst_table) {
    // a thread has its place in the row, and takes four rows at a time
    const int per = kMoveThreads / units, u = threadIdx.x % units;
    if (threadIdx.x >= per * units || b >= p.src_pages || b >= p.dst_pages) return;
    const unsigned char* s = static_cast<const unsigned char*>(a.src) + b * a.src_page_stride + h * a.src_head_stride + u * sizeof(V);
    unsigned char* d = static_cast<unsigned char*>(a.dst) + b * a.dst_page_stride + h * a.dst_head_stride + u * sizeof(V);
    for (int j = j0 + threadIdx.x / units; j < j1; j += 4 * per) {
      V v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i * per < j1) v[i] = *reinterpret_cast<const V*>(s + (int64_t)kept[j + i * per] * a.row_bytes);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i * per < j1) *reinterpret_cast<V*>(d + (int64_t)(j + i * per) * a.row_bytes) = v[i];
    }
    return;
  }
  if (!in_place) {
    for (int e = threadIdx.x; e < total; e += kMoveThreads) {
      const int j = j0 + e / units, u = e % units;
      const V* s = src_of(j);
      V* d = dst_of(j);
      if (d) d[u] = s ? s[u] : V{};
    }
    return;
  }
  for (int e = threadIdx.x; e < total; e += kMoveThreads) {
    const V* s = src_of(j0 + e / units);
    buf[e] = s ? s[e % units] : V{};
  }
  __syncthreads();
  for (int e = threadIdx.x; e < total; e += kMoveThreads) {
    V* d = dst_of(j0 + e / units);
    if (d) d[e % units] = buf[e];
  }
  __syncthreads();
}

// blockIdx.y: the row arrays, then the weights.  Rows move to lower or equal positions, and row j of the
// result comes from a row >= j: in place, a CTA that owns a whole (array, sequence, head) may take the
// rows in chunks, reading a chunk before it writes it.  HBM bound: 16 x 8 heads, 4096 rows of 2 x 256 bytes each: 99 us = 5.5 TB/s.
__global__ void __launch_bounds__(kMoveThreads, 8) evict_move_kernel(const EvictParams p, int rows_per_block, bool in_place,
                                                                  bool weights_in_place) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int problem = blockIdx.z, b = problem / p.n_kv, h = problem % p.n_kv;
  const int which = blockIdx.y;
  pdl_wait();
  const int stay = p.counts[problem];
  const int32_t* kept = p.kept + (int64_t)problem * p.keep;
  if (which == p.n_arrays) {
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) p.lens_out[b] = stay;
    const float* src = p.weights + b * p.w_seq + h * p.w_head;
    float* dst = p.dst_weights + b * p.dw_seq + h * p.dw_head;
    if (!weights_in_place) {
      for (int64_t j = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; j < p.dw_width; j += (int64_t)gridDim.x * kMoveThreads)
        dst[j] = j < stay ? src[kept[j]] : 0.f;
      return;
    }
    if (blockIdx.x != 0) return;
    float* buf = reinterpret_cast<float*>(smem);
    constexpr int kChunk = kMoveSmem / 4;
    for (int j0 = 0; j0 < stay; j0 += kChunk) {
      const int c = min(kChunk, stay - j0);
      for (int j = threadIdx.x; j < c; j += kMoveThreads) buf[j] = src[kept[j0 + j]];
      __syncthreads();
      for (int j = threadIdx.x; j < c; j += kMoveThreads) dst[j0 + j] = buf[j];
      __syncthreads();
    }
    for (int64_t j = stay + threadIdx.x; j < p.dw_width; j += kMoveThreads) dst[j] = 0.f;
    return;
  }
  if (stay == 0 || (in_place && kept[stay - 1] == stay - 1)) return;  // every row is where it stays
  const sva_evict_array& a = p.arrays[which];
  int64_t bits = a.row_bytes | a.src_page_stride | a.src_head_stride | a.dst_page_stride | a.dst_head_stride |
                 (int64_t)reinterpret_cast<uintptr_t>(a.src) | (int64_t)reinterpret_cast<uintptr_t>(a.dst);
  int j0 = in_place ? 0 : blockIdx.x * rows_per_block;
  const int step = in_place ? max(1, (int)(kMoveSmem / a.row_bytes)) : rows_per_block;
  const int end = in_place ? stay : min(stay, j0 + rows_per_block);
  for (; j0 < end; j0 += step) {
    const int j1 = min(end, j0 + step);
    if ((bits & 15) == 0)
      move_rows<uint4>(p, a, kept, b, h, j0, j1, in_place, smem);
    else if ((bits & 7) == 0)
      move_rows<uint2>(p, a, kept, b, h, j0, j1, in_place, smem);
    else if ((bits & 3) == 0)
      move_rows<uint32_t>(p, a, kept, b, h, j0, j1, in_place, smem);
    else
      move_rows<uint16_t>(p, a, kept, b, h, j0, j1, in_place, smem);
  }
}

static int check_evict(const sva_evict_args* a) {
  if (!a) return set_error(SVA_ERR_SHAPE, "the arguments are null");
  if (a->n_seqs <= 0 || a->n_kv_heads <= 0 || (int64_t)a->n_seqs * a->n_kv_heads > 65535)
    return set_error(SVA_ERR_SHAPE, "n_seqs times n_kv_heads must be in 1..65535");
  if (a->n_arrays < 0 || a->n_arrays > SVA_EVICT_MAX_ARRAYS) return set_error(SVA_ERR_SHAPE, "at most 8 row arrays");
  if (a->max_len < 0 || a->max_len >= (1ll << 31)) return set_error(SVA_ERR_SHAPE, "max_len must be below 2^31");
  if (a->keep < 0 || a->keep >= (1ll << 31)) return set_error(SVA_ERR_SHAPE, "keep must be in 0..2^31 - 1");
  if (a->recent < 0 || a->recent > a->keep) return set_error(SVA_ERR_SHAPE, "recent must be in 0..keep");
  if (a->n_arrays > 0) {
    if (a->src_pages <= 0 || a->src_page_rows <= 0 || a->dst_pages <= 0 || a->dst_page_rows <= 0)
      return set_error(SVA_ERR_SHAPE, "bad page sizes");
    const int64_t src_cap = a->src_table ? a->src_table_cols * a->src_page_rows : a->src_page_rows;
    const int64_t dst_cap = a->dst_table ? a->dst_table_cols * a->dst_page_rows : a->dst_page_rows;
    if (a->max_len > src_cap) return set_error(SVA_ERR_SHAPE, "max_len exceeds the source rows of a sequence");
    if ((a->keep < a->max_len ? a->keep : a->max_len) > dst_cap)
      return set_error(SVA_ERR_SHAPE, "the destination has fewer rows a sequence than stay");
    if ((!a->src_table && a->src_pages < a->n_seqs) || (!a->dst_table && a->dst_pages < a->n_seqs))
      return set_error(SVA_ERR_SHAPE, "an array has fewer pages than there are sequences, and no page table");
  }
  return SVA_OK;
}

}  // namespace sva

using namespace sva;

extern "C" size_t sva_cache_evict_workspace_size(const sva_evict_args* a) {
  return check_evict(a) == SVA_OK ? (size_t)a->n_seqs * a->n_kv_heads * 4 : 0;
}

extern "C" int sva_cache_evict(const sva_evict_args* a, const sva_evict_array* arrays, void* workspace,
                               size_t workspace_bytes, void* stream) {
  int rc = check_evict(a);
  if (rc != SVA_OK) return rc;
  if (!a->seq_lens || !a->weights || !a->dst_weights || !a->lens_out || (a->keep > 0 && !a->kept_out) ||
      (a->n_arrays > 0 && !arrays))
    return set_error(SVA_ERR_SHAPE, "a required pointer is null");
  const bool w_in_place = a->weights == a->dst_weights;
  if (w_in_place && (a->weights_seq_stride != a->dst_weights_seq_stride || a->weights_head_stride != a->dst_weights_head_stride))
    return set_error(SVA_ERR_SHAPE, "weights in place must keep their strides");
  if (a->dst_weights_width < (a->keep < a->max_len ? a->keep : a->max_len))
    return set_error(SVA_ERR_SHAPE, "the destination weights are narrower than the rows that stay");
  const size_t need = sva_cache_evict_workspace_size(a);
  if (!workspace || workspace_bytes < need) return set_error(SVA_ERR_WORKSPACE, "workspace too small");
  EvictParams p{a->n_seqs, a->n_kv_heads, a->n_arrays, a->max_len, a->keep, a->recent, a->seq_lens, a->weights,
                a->weights_seq_stride, a->weights_head_stride, a->dst_weights, a->dst_weights_seq_stride,
                a->dst_weights_head_stride, a->dst_weights_width, a->src_pages, a->src_page_rows, a->dst_pages,
                a->dst_page_rows, a->src_table, a->src_table_stride, a->src_table_cols, a->dst_table,
                a->dst_table_stride, a->dst_table_cols, a->kept_out, a->lens_out, static_cast<int32_t*>(workspace), {}};
  for (int i = 0; i < a->n_arrays; ++i) {
    const sva_evict_array& r = arrays[i];
    if (!r.src || !r.dst) return set_error(SVA_ERR_SHAPE, "a row array is null");
    if (r.row_bytes <= 0 || r.row_bytes % 2 || r.row_bytes > kMoveSmem)
      return set_error(SVA_ERR_SHAPE, "row_bytes must be even and at most 96 KiB");
    if ((reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst) | (uintptr_t)r.src_page_stride |
         (uintptr_t)r.src_head_stride | (uintptr_t)r.dst_page_stride | (uintptr_t)r.dst_head_stride) & 1)
      return set_error(SVA_ERR_ALIGN, "row arrays must be 2-byte aligned");
    if (a->in_place && r.src != r.dst) return set_error(SVA_ERR_SHAPE, "in place, src and dst must be the same array");
    if (!a->in_place && r.src == r.dst) return set_error(SVA_ERR_SHAPE, "src equals dst but in_place is not set");
    p.arrays[i] = r;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int problems = a->n_seqs * a->n_kv_heads;
  const int room = (int)std::min<int64_t>(a->max_len, kSelKeys);
  rc = ensure_smem_attr(reinterpret_cast<const void*>(evict_select_kernel), kSelKeys * 4);
  if (rc != SVA_OK) return rc;
  evict_select_kernel<<<problems, kSelThreads, room * 4, st>>>(p, room);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(SVA_ERR_CUDA, cudaGetErrorString(e));
  const bool in_place = a->in_place != 0;
  const int smem = in_place || w_in_place ? kMoveSmem : 0;
  rc = ensure_smem_attr(reinterpret_cast<const void*>(evict_move_kernel), kMoveSmem);
  if (rc != SVA_OK) return rc;
  const int rows_per_block = 64;
  const int64_t most = a->keep < a->max_len ? a->keep : a->max_len;
  const int64_t xs = in_place ? 1 : std::max<int64_t>(1, (most + rows_per_block - 1) / rows_per_block);
  // launched while the selection drains; it waits there for the selection's memory
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)xs, a->n_arrays + 1, problems);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, evict_move_kernel, p, rows_per_block, in_place, w_in_place);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? SVA_OK : set_error(SVA_ERR_CUDA, cudaGetErrorString(e));
}
