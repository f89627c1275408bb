// The paged KV cache's bookkeeping and writes:
//   page tables of a step (pages granted from a free stack, sequence lengths, query offsets,
//   positions, slots) from the requests' lengths; release of a request's pages;
//   per-head RMS norm + rotary embedding of a fused QKV output with the K/V write.
// A slot is page * page_size + offset; a slot of -1 stands for a token without a place.
#include <mutex>
#include <string>

#include "lm_common.cuh"

namespace lm {
namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableCtas = 8;  // one cluster, so that its barrier orders reads before writes
constexpr int kMaxRequests = 4096;
constexpr int kPerThread = kMaxRequests / kTableThreads;

struct TableParams {
  const int32_t* cached;
  const int32_t* fresh;
  int32_t* tables;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* free_count_out;
  int32_t* seq_lens;
  int32_t* cu_q;
  int32_t* positions;
  int64_t* slots;
  int32_t* err;
  int64_t table_stride, max_tokens;
  int num_requests, page_size, max_pages, free_capacity;
};

// Exclusive prefix sums of two values per thread over the block; the totals come back too.
// 64-bit: bad lengths may not wrap around before they are noticed.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t& total_a,
                                            int64_t& total_b, int64_t (*s_warp)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia += ua;
      ib += ub;
    }
  }
  if (lane == 31) {
    s_warp[warp][0] = ia;
    s_warp[warp][1] = ib;
  }
  __syncthreads();
  if (warp == 0) {
    int64_t wa = lane < warps ? s_warp[lane][0] : 0, wb = lane < warps ? s_warp[lane][1] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ua = __shfl_up_sync(0xffffffffu, wa, o), ub = __shfl_up_sync(0xffffffffu, wb, o);
      if (lane >= o) {
        wa += ua;
        wb += ub;
      }
    }
    s_warp[lane][0] = wa;
    s_warp[lane][1] = wb;
  }
  __syncthreads();
  total_a = s_warp[warps - 1][0];
  total_b = s_warp[warps - 1][1];
  a = ia - a + (warp ? s_warp[warp - 1][0] : 0);
  b = ib - b + (warp ? s_warp[warp - 1][1] : 0);
}

// Every CTA scans all requests (they fit one pass of its threads) and writes its share of the
// tables and of the tokens. All reads of arrays that the call may overwrite in place (cached
// lengths, the free count) come before the cluster's barrier, all writes to them after it.
__global__ void __launch_bounds__(kTableThreads) page_tables_kernel(const TableParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int32_t s_mem[];
  __shared__ int64_t s_warp[32][2];
  __shared__ int s_used;
  if (threadIdx.x == 0) s_used = 0;
  const int B = p.num_requests, page = p.page_size;
  int32_t* s_cu = s_mem;               // [B + 1] first token of each request
  int32_t* s_page = s_cu + B + 1;      // [B] pages granted before it, or -1: none for it
  int32_t* s_cached = s_page + B;      // [B]
  const int per = (B + kTableThreads - 1) / kTableThreads;
  int free_count = *p.free_count;
  if (free_count < 0 || free_count > p.free_capacity) {
    if (threadIdx.x == 0) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    free_count = min(max(free_count, 0), p.free_capacity);
  }
  int need[kPerThread], fresh[kPerThread], cached[kPerThread];
  int64_t sum_need = 0, sum_fresh = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * per + i;
    need[i] = fresh[i] = cached[i] = 0;
    if (i >= per || b >= B) continue;
    cached[i] = p.cached[b];
    fresh[i] = p.fresh[b];
    const int64_t limit = static_cast<int64_t>(p.max_pages) * page;
    bool bad = false;
    if (cached[i] < 0 || cached[i] > limit) {
      bad = true;
      cached[i] = 0;
    }
    if (fresh[i] < 0 || fresh[i] > p.max_tokens) {
      bad = true;
      fresh[i] = 0;
    }
    if (bad) {
      record_error(p.err, LM_DEVERR_BAD_LENGTH);
      need[i] = -1;
    } else if (static_cast<int64_t>(cached[i]) + fresh[i] > limit) {
      record_error(p.err, LM_DEVERR_NO_PAGES);
      need[i] = -1;
    } else {
      need[i] = (cached[i] + fresh[i] + page - 1) / page - (cached[i] + page - 1) / page;
    }
    sum_need += max(need[i], 0);
    sum_fresh += fresh[i];
  }
  int64_t at_need = sum_need, at_fresh = sum_fresh, total_need, total_fresh;
  block_scan2(at_need, at_fresh, total_need, total_fresh, s_warp);
  int granted = 0;  // pages up to and including this thread's last request that got its pages
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * per + i;
    if (i >= per || b >= B) continue;
    s_cu[b] = static_cast<int32_t>(min(at_fresh, p.max_tokens));
    s_cached[b] = cached[i];
    bool ok = need[i] >= 0;
    if (ok && need[i] > 0 && at_need + need[i] > free_count) {
      record_error(p.err, LM_DEVERR_NO_PAGES);
      ok = false;
    }
    // a request that needs no page may stand past the stack's end: it reads none
    s_page[b] = ok ? static_cast<int32_t>(min(at_need, static_cast<int64_t>(free_count))) : -1;
    if (ok && need[i] > 0) granted = static_cast<int>(at_need) + need[i];
    at_need += max(need[i], 0);
    at_fresh += fresh[i];
  }
  if (threadIdx.x == 0) {
    s_cu[B] = static_cast<int32_t>(min(total_fresh, p.max_tokens));
    if (total_fresh > p.max_tokens) record_error(p.err, LM_DEVERR_BAD_LENGTH);
  }
  // The largest grant ends the pages taken: requests are granted in order, and once one does not
  // fit, every later one that needs a page does not either.
  if (granted > 0) atomicMax(&s_used, granted);
  __syncthreads();
  if (gridDim.x > 1) cluster_sync_all();
  const int tid = blockIdx.x * kTableThreads + threadIdx.x;
  const int stride = gridDim.x * kTableThreads;
  if (tid == 0) *p.free_count_out = free_count - s_used;
  for (int b = tid; b <= B; b += stride) {
    p.cu_q[b] = s_cu[b];
    if (b == B) break;
    const int c = s_cached[b], n = s_page[b] >= 0 ? s_cu[b + 1] - s_cu[b] : 0;
    p.seq_lens[b] = c + n;
  }
  // new table entries: a warp per request
  const int lane = threadIdx.x & 31;
  for (int b = tid >> 5; b < B; b += stride >> 5) {
    if (s_page[b] < 0) continue;
    const int c = s_cached[b], n = s_cu[b + 1] - s_cu[b];
    const int have = (c + page - 1) / page, total = (c + n + page - 1) / page;
    for (int i = have + lane; i < total; i += 32)
      p.tables[b * p.table_stride + i] = p.free_pages[free_count - 1 - (s_page[b] + i - have)];
  }
  for (int64_t t = tid; t < p.max_tokens; t += stride) {
    int pos = 0;
    int64_t slot = -1;
    if (t < total_fresh) {
      int lo = 0, hi = B;  // last request that starts at or before t and is not empty
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int c = s_cached[lo];
      pos = c + static_cast<int>(t) - s_cu[lo];
      if (s_page[lo] >= 0) {
        const int have = (c + page - 1) / page, i = pos / page;
        // pages already held are read from the table, granted ones from the stack (another CTA
        // may be writing their table entries)
        const int pg = i < have ? p.tables[lo * p.table_stride + i]
                                : p.free_pages[free_count - 1 - (s_page[lo] + i - have)];
        slot = pg < 0 ? -1 : static_cast<int64_t>(pg) * page + pos - i * page;
        if (pg < 0) record_error(p.err, LM_DEVERR_BAD_PAGE);
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// One block: the pages of the listed rows go back onto the free stack in row order.
__global__ void __launch_bounds__(256)
    release_pages_kernel(const int32_t* __restrict__ rows, int num_rows, int32_t* cached,
                         int num_requests, int page_size, int32_t* tables, int64_t table_stride,
                         int max_pages, int32_t* free_pages, int free_capacity,
                         int32_t* free_count, int32_t* err) {
  pdl_wait();
  pdl_trigger();
  int count = *free_count;
  if (count < 0 || count > free_capacity) {
    if (threadIdx.x == 0) record_error(err, LM_DEVERR_BAD_LENGTH);
    return;
  }
  for (int i = 0; i < num_rows; ++i) {
    const int b = rows[i];
    if (b < 0 || b >= num_requests || cached[b] < 0 ||
        cached[b] > static_cast<int64_t>(max_pages) * page_size) {
      if (threadIdx.x == 0) record_error(err, LM_DEVERR_BAD_LENGTH);
      continue;  // the same decision in every thread: nothing of the row changes
    }
    const int n = (cached[b] + page_size - 1) / page_size;
    if (n > free_capacity - count) {
      if (threadIdx.x == 0) record_error(err, LM_DEVERR_BAD_LENGTH);
      continue;
    }
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
      free_pages[count + j] = tables[b * table_stride + j];
      tables[b * table_stride + j] = -1;
    }
    count += n;
    __syncthreads();  // every thread has read cached[b]; a row listed twice is empty then
    if (threadIdx.x == 0) cached[b] = 0;
    __syncthreads();
  }
  if (threadIdx.x == 0) *free_count = count;
}

// ---------------------------------------------------------------------------- rope + write
constexpr int kRopeWarps = 8;

struct RopeParams {
  const uint16_t* qkv;
  const int32_t* positions;
  const int64_t* slots;
  const float* cos_sin;  // [max_pos, rot_dim]: cosines, then sines
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  uint16_t* q_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int32_t* err;
  int64_t qkv_stride, q_token_stride, q_head_stride;
  int64_t k_page_stride, k_token_stride, k_head_stride;
  int64_t v_page_stride, v_token_stride, v_head_stride;
  int64_t num_tokens, num_slots;
  float eps;
  int q_heads, kv_heads, rot_dim, max_pos, page_size, interleaved;
};

// A warp per (token, head); the head's fp32 values pass through shared memory so that a lane
// reads its rotation partner.
template <int D>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_write_kernel(const RopeParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int PER = D / 32;
  __shared__ float s_head[kRopeWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.q_heads + 2 * p.kv_heads;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRopeWarps + warp;
  if (unit >= p.num_tokens * heads) return;
  const int64_t t = unit / heads;
  const int h = static_cast<int>(unit % heads);
  const uint16_t* src = p.qkv + t * p.qkv_stride + static_cast<int64_t>(h) * D;
  float z[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) z[i] = bf16_bits_to_f32(src[lane + 32 * i]);
  const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
  uint16_t* dst;
  if (is_q) {
    dst = p.q_out + t * p.q_token_stride + h * p.q_head_stride;
  } else {
    const int64_t slot = p.slots[t];
    if (slot < 0) return;  // a padding token: nothing to store
    if (slot >= p.num_slots) {
      if (lane == 0) record_error(p.err, LM_DEVERR_BAD_PAGE);
      return;
    }
    const int64_t page = slot / p.page_size, off = slot % p.page_size;
    if (is_v)
      dst = p.v_cache + page * p.v_page_stride + off * p.v_token_stride +
            (h - p.q_heads - p.kv_heads) * p.v_head_stride;
    else
      dst = p.k_cache + page * p.k_page_stride + off * p.k_token_stride +
            (h - p.q_heads) * p.k_head_stride;
  }
  if (!is_v) {
    const uint16_t* w = is_q ? p.q_weight : p.k_weight;
    if (w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) ss += z[i] * z[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss / D + p.eps);
#pragma unroll
      for (int i = 0; i < PER; ++i) z[i] *= r * bf16_bits_to_f32(w[lane + 32 * i]);
    }
    int pos = p.positions[t];
    if (pos < 0 || pos >= p.max_pos) {
      if (lane == 0) record_error(p.err, LM_DEVERR_BAD_POSITION);
      pos = 0;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s_head[warp][lane + 32 * i] = z[i];
    __syncwarp();
    const int R = p.rot_dim, half = R / 2;
    const float* cs = p.cos_sin + static_cast<int64_t>(pos) * R;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = lane + 32 * i;
      if (c >= R) continue;
      const int f = p.interleaved ? c >> 1 : (c < half ? c : c - half);
      const bool first = p.interleaved ? (c & 1) == 0 : c < half;
      const float other = s_head[warp][p.interleaved ? c ^ 1 : (first ? c + half : c - half)];
      const float cosv = cs[f], sinv = cs[half + f];
      z[i] = first ? z[i] * cosv - other * sinv : z[i] * cosv + other * sinv;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) dst[lane + 32 * i] = f32_to_bf16_bits(z[i]);
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_build_page_tables(const int32_t* cached_lens, const int32_t* new_lens,
                                    int32_t num_requests, int32_t page_size,
                                    int32_t* block_tables, int64_t table_stride,
                                    int32_t max_pages, const int32_t* free_pages,
                                    int32_t free_capacity, const int32_t* free_count,
                                    int32_t* free_count_out, int32_t* seq_lens, int32_t* cu_q,
                                    int32_t* positions, int64_t* slot_mapping, int64_t max_tokens,
                                    int32_t* err_word, void* stream) {
  if (num_requests < 0 || num_requests > kMaxRequests)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_build_page_tables: at most 4096 requests");
  if (page_size <= 0 || max_pages <= 0 || table_stride < max_pages || free_capacity < 0 ||
      max_tokens < 0 || max_tokens > 0x7fffffff ||
      static_cast<int64_t>(max_pages) * page_size > 0x7fffffff)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_build_page_tables: bad sizes");
  if (num_requests > 0 && (cached_lens == nullptr || new_lens == nullptr ||
                           block_tables == nullptr || seq_lens == nullptr))
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_build_page_tables: null pointer");
  if (cu_q == nullptr || free_count == nullptr || free_count_out == nullptr ||
      (free_capacity > 0 && free_pages == nullptr) ||
      (max_tokens > 0 && (positions == nullptr || slot_mapping == nullptr)))
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_build_page_tables: null pointer");
  const TableParams p{cached_lens, new_lens, block_tables, free_pages, free_count, free_count_out,
                      seq_lens, cu_q, positions, slot_mapping, err_word, table_stride, max_tokens,
                      num_requests, page_size, max_pages, free_capacity};
  const size_t smem = (3 * static_cast<size_t>(num_requests) + 1) * 4;
  if (smem > 48 * 1024) {
    const int rc = check_cuda(cudaFuncSetAttribute(page_tables_kernel,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (3 * kMaxRequests + 1) * 4),
                              "lm_build_page_tables: smem attribute");
    if (rc) return rc;
  }
  const int ctas = max_tokens <= 2 * kTableThreads && num_requests <= kTableThreads ? 1 : kTableCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kTableThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, page_tables_kernel, p), "lm_build_page_tables");
}

extern "C" int lm_release_pages(const int32_t* rows, int32_t num_rows, int32_t* cached_lens,
                                int32_t num_requests, int32_t page_size, int32_t* block_tables,
                                int64_t table_stride, int32_t max_pages, int32_t* free_pages,
                                int32_t free_capacity, int32_t* free_count, int32_t* err_word,
                                void* stream) {
  if (num_rows < 0 || num_requests <= 0 || page_size <= 0 || max_pages <= 0 ||
      table_stride < max_pages || free_capacity < 0 ||
      static_cast<int64_t>(max_pages) * page_size > 0x7fffffff)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_release_pages: bad sizes");
  if (num_rows == 0) return LM_OK;
  if (rows == nullptr || cached_lens == nullptr || block_tables == nullptr ||
      free_pages == nullptr || free_count == nullptr)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_release_pages: null pointer");
  return check_cuda(
      launch_dependent(release_pages_kernel, dim3(1), dim3(256), 0,
                       static_cast<cudaStream_t>(stream), rows, num_rows, cached_lens, num_requests,
                       page_size, block_tables, table_stride, max_pages, free_pages, free_capacity,
                       free_count, err_word),
      "lm_release_pages");
}

extern "C" int lm_rope_cache_write(
    const uint16_t* qkv, int64_t qkv_stride, const int32_t* positions, const int64_t* slot_mapping,
    int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const float* cos_sin, int32_t max_positions, int32_t rot_dim, int32_t interleaved,
    const uint16_t* q_norm_weight, const uint16_t* k_norm_weight, float eps, uint16_t* q_out,
    int64_t q_token_stride, int64_t q_head_stride, uint16_t* k_cache, int64_t k_page_stride,
    int64_t k_token_stride, int64_t k_head_stride, uint16_t* v_cache, int64_t v_page_stride,
    int64_t v_token_stride, int64_t v_head_stride, int64_t num_pages, int32_t page_size,
    int32_t* err_word, void* stream) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_tokens < 0 || num_pages < 0 || page_size <= 0 ||
      max_positions <= 0)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_rope_cache_write: bad sizes");
  if (head_dim != 64 && head_dim != 128)
    return fail(LM_ERR_UNSUPPORTED, "lm_rope_cache_write: head_dim must be 64 or 128");
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_rope_cache_write: rot_dim must be even and at most head_dim");
  if (num_tokens == 0) return LM_OK;
  if (qkv == nullptr || positions == nullptr || slot_mapping == nullptr || q_out == nullptr ||
      k_cache == nullptr || v_cache == nullptr || (rot_dim > 0 && cos_sin == nullptr))
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_rope_cache_write: null pointer");
  const int64_t strides = qkv_stride | q_token_stride | q_head_stride | k_page_stride |
                          k_token_stride | k_head_stride | v_page_stride | v_token_stride |
                          v_head_stride;
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
        reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) != 0 ||
      (strides & 7) != 0)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_rope_cache_write: bases must be 16-byte aligned and strides multiples of 8 elements");
  const int heads = num_q_heads + 2 * num_kv_heads;
  const RopeParams p{qkv, positions, slot_mapping, cos_sin, q_norm_weight, k_norm_weight, q_out,
                     k_cache, v_cache, err_word, qkv_stride, q_token_stride, q_head_stride,
                     k_page_stride, k_token_stride, k_head_stride, v_page_stride, v_token_stride,
                     v_head_stride, num_tokens, num_pages * page_size, eps, num_q_heads,
                     num_kv_heads, rot_dim, max_positions, page_size, interleaved};
  const int64_t blocks = (num_tokens * heads + kRopeWarps - 1) / kRopeWarps;
  if (blocks > 0x7fffffff)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_rope_cache_write: too many tokens");
  auto kernel = head_dim == 64 ? rope_write_kernel<64> : rope_write_kernel<128>;
  return check_cuda(launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)),
                                     dim3(kRopeWarps * 32), 0, static_cast<cudaStream_t>(stream), p),
                    "lm_rope_cache_write");
}
