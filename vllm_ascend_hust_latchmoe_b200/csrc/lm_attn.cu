// Attention of a step's new tokens over the paged cache:
//   out = softmax(q k^T * scale over the keys that the row sees) v,   lse = max + ln(sum)
// A row at position p sees key j when j <= p and (window == 0 or j > p - window); a row that sees
// nothing gives zeros and an lse of -inf. One pass over the keys with the running maximum and sum
// (fp32, in the log2 domain).
//
// This kernel takes 16-row tiles: single tokens and small chunks, where reading K and V is the
// cost. The 8 warps of a CTA read 16 keys each of a 128-key block and keep their own running
// results, so the key loop has no CTA barrier: every warp has its own 3-deep cp.async ring. Warps
// are merged in shared memory at the end of a segment, segments of an item that several CTAs
// share through the workspace, by the CTA that arrives last, in the order of the keys.
#include <mutex>
#include <string>

#include "lm_attn.cuh"

namespace lm {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTileRows = 16;
constexpr int kSlice = 16;               // keys per warp and stage
constexpr int kBlock = kWarps * kSlice;  // keys per unit
constexpr int kStages = 3;

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D>
struct RowsSmem {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTile = kSlice * kRowBytes;       // K or V of one warp stage
  static constexpr int kStage = 2 * kTile;
  static constexpr int kRing = kWarps * kStages * kStage;
  // merge area over the ring: O [kWarps][16][D] fp32, then m and l [kWarps][16][2]
  static constexpr int kMerge = kWarps * kTileRows * D * 4 + kWarps * kTileRows * 2 * 4;
  static constexpr int kBytes = kRing > kMerge ? kRing : kMerge;
};

// 16-byte chunk c of row r, XOR-swizzled so that 8 rows of one chunk column hit 8 bank groups.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return static_cast<uint32_t>(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_rows_kernel(const AttnParams p) {
  using S = RowsSmem<D>;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int32_t s_warp[kWarps];
  __shared__ int s_last;
  int32_t* s_prefix = reinterpret_cast<int32_t*>(smem + S::kBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c2 = (lane & 3) * 2;

  attn_prefix<kTileRows, kBlock, kThreads>(p, s_prefix, s_warp);
  const int total = s_prefix[p.num_requests];
  const int per = (total + gridDim.x - 1) / gridDim.x;
  int w = blockIdx.x * per;
  const int w_end = min(total, w + per);
  AttnCursor at{};
  if (w < w_end) at = attn_seek<kTileRows, kBlock>(p, s_prefix, w);

  unsigned char* ring = smem + warp * kStages * S::kStage;
  const uint32_t ring_addr = smem_u32(ring);

  while (w < w_end) {
    const AttnSegment s = attn_segment<kTileRows, kBlock>(p, at, w, w_end);
    const int rows = at.req.qlen * p.group;
    const int row_base = at.tile * kTileRows;
    const int cached = at.req.seq - at.req.qlen;
    const int n_slices = s.blk1 - s.blk0;  // one slice of this warp per block
    const int32_t* table = p.tables + at.b * p.table_stride;
    const uint16_t* kh = p.k + at.head * p.k_head_stride;
    const uint16_t* vh = p.v + at.head * p.v_head_stride;
    int pages = 0, page_first = 0;  // lane i: the page of slice page_first + i

    auto load = [&](int i) {  // slice i of this warp into stage i % kStages
      if (i < n_slices) {
        if (i % 32 == 0) {
          const int tok = (s.blk0 + i + lane) * kBlock + warp * kSlice;
          pages = -1;
          if (i + lane < n_slices && tok < s.hi && tok + kSlice > s.lo) {
            pages = table[tok / p.page_size];
            if (pages < 0 || pages >= p.num_pages) {
              record_error(p.err, LM_DEVERR_BAD_PAGE);
              pages = -1;
            }
          }
          page_first = i;
        }
        const int page = __shfl_sync(0xffffffffu, pages, i - page_first);
        const int tok0 = (s.blk0 + i) * kBlock + warp * kSlice;
        const int in_page = tok0 % p.page_size;
        const uint16_t* ks = kh + page * p.k_page_stride;
        const uint16_t* vs = vh + page * p.v_page_stride;
        unsigned char* st = ring + (i % kStages) * S::kStage;
        constexpr int kChunks = D / 8;             // 16-byte chunks per row
        constexpr int kIters = kSlice * kChunks / 32;
#pragma unroll
        for (int j = 0; j < kIters; ++j) {
          const int r = (j * 32 + lane) / kChunks, c = (j * 32 + lane) % kChunks;
          // keys outside the tile's range are zeros: what the cache holds there may be anything
          const uint32_t n = page >= 0 && tok0 + r >= s.lo && tok0 + r < s.hi ? 16u : 0u;
          const int64_t tk = in_page + r;
          cp_async_16(st + swz<D>(r, c), n ? ks + tk * p.k_token_stride + c * 8 : p.k, n);
          cp_async_16(st + S::kTile + swz<D>(r, c), n ? vs + tk * p.v_token_stride + c * 8 : p.v, n);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) load(i);

    // Q fragments: rows g and g + 8 of the tile
    const int r0 = row_base + g, r1 = r0 + 8;
    const int t0 = r0 / p.group, t1 = r1 / p.group;
    uint32_t qf[D / 16][4];
    {
      const bool ok0 = r0 < rows, ok1 = r1 < rows;
      const uint16_t* q0 = p.q + (at.req.q0 + t0) * p.q_token_stride +
                           (at.head * p.group + r0 % p.group) * p.q_head_stride;
      const uint16_t* q1 = p.q + (at.req.q0 + t1) * p.q_token_stride +
                           (at.head * p.group + r1 % p.group) * p.q_head_stride;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][0] = ok0 ? *reinterpret_cast<const uint32_t*>(q0 + k * 16 + c2) : 0u;
        qf[k][1] = ok1 ? *reinterpret_cast<const uint32_t*>(q1 + k * 16 + c2) : 0u;
        qf[k][2] = ok0 ? *reinterpret_cast<const uint32_t*>(q0 + k * 16 + c2 + 8) : 0u;
        qf[k][3] = ok1 ? *reinterpret_cast<const uint32_t*>(q1 + k * 16 + c2 + 8) : 0u;
      }
    }
    // keys (j > low, j <= high) that the two rows see
    const int high0 = r0 < rows ? min(cached + t0, s.hi - 1) : -1;
    const int high1 = r1 < rows ? min(cached + t1, s.hi - 1) : -1;
    const int low0 = p.window > 0 ? cached + t0 - p.window : -1;
    const int low1 = p.window > 0 ? cached + t1 - p.window : -1;

    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int i = 0; i < n_slices; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();
      load(i + kStages - 1);  // its stage was read in the last iteration, before the syncwarp
      const uint32_t st = ring_addr + (i % kStages) * S::kStage;
      float sc[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];  // keys 0-7: k halves 0, 1; keys 8-15: k halves 0, 1
        ldmatrix_x4(b, st + swz<D>((lane & 7) + ((lane & 16) >> 1), 2 * k + ((lane >> 3) & 1)));
        mma_bf16(sc[0], qf[k], b[0], b[1]);
        mma_bf16(sc[1], qf[k], b[2], b[3]);
      }
      const int j0 = (s.blk0 + i) * kBlock + warp * kSlice + c2;
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + n * 8 + e;
          sc[n][e] = j <= high0 && j > low0 ? sc[n][e] * p.scale_log2 : -INFINITY;
          sc[n][2 + e] = j <= high1 && j > low1 ? sc[n][2 + e] * p.scale_log2 : -INFINITY;
          mx0 = fmaxf(mx0, sc[n][e]);
          mx1 = fmaxf(mx1, sc[n][2 + e]);
        }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
      }
      if (__any_sync(0xffffffffu, mx0 > m0 || mx1 > m1)) {
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        const float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - n0);
        const float f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] *= f0;
          o[n][1] *= f0;
          o[n][2] *= f1;
          o[n][3] *= f1;
        }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t pa[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e0 = exp2f(sc[n][0] - b0), e1 = exp2f(sc[n][1] - b0);
        const float e2 = exp2f(sc[n][2] - b1), e3 = exp2f(sc[n][3] - b1);
        l0 += e0 + e1;
        l1 += e2 + e3;
        pa[2 * n] = pack_bf16x2(e0, e1);
        pa[2 * n + 1] = pack_bf16x2(e2, e3);
      }
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b[4];  // d columns 16 n .. +7: keys 0-7, 8-15; columns +8: the same
        ldmatrix_x4_trans(b, st + S::kTile + swz<D>(lane & 15, 2 * n + (lane >> 4)));
        mma_bf16(o[2 * n], pa, b[0], b[1]);
        mma_bf16(o[2 * n + 1], pa, b[2], b[3]);
      }
      __syncwarp();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    __syncthreads();  // every warp is done with its ring: the merge area lies over it

    float* s_o = reinterpret_cast<float*>(smem);
    float* s_ml = s_o + kWarps * kTileRows * D;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      float* d0 = s_o + (warp * kTileRows + g) * D + n * 8 + c2;
      *reinterpret_cast<float2*>(d0) = make_float2(o[n][0], o[n][1]);
      *reinterpret_cast<float2*>(d0 + 8 * D) = make_float2(o[n][2], o[n][3]);
    }
    if ((lane & 3) == 0) {
      s_ml[(warp * kTileRows + g) * 2] = m0;
      s_ml[(warp * kTileRows + g) * 2 + 1] = l0;
      s_ml[(warp * kTileRows + g + 8) * 2] = m1;
      s_ml[(warp * kTileRows + g + 8) * 2 + 1] = l1;
    }
    __syncthreads();

    // 16 threads per row, D / 16 columns each
    const int r = threadIdx.x >> 4, col = (threadIdx.x & 15) * (D / 16);
    float m = -INFINITY, l = 0.f, acc[D / 16];
#pragma unroll
    for (int k = 0; k < kWarps; ++k) m = fmaxf(m, s_ml[(k * kTileRows + r) * 2]);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) acc[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float mk = s_ml[(k * kTileRows + r) * 2];
      const float f = mk == -INFINITY ? 0.f : exp2f(mk - m);
      l += f * s_ml[(k * kTileRows + r) * 2 + 1];
      const float* src = s_o + (k * kTileRows + r) * D + col;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] += f * src[e];
    }

    bool final = s.whole;
    if (!s.whole) {
      const int cs = s.start / per, ce = (s.end - 1) / per;
      const int me = blockIdx.x;
      const int64_t slot = 2 * static_cast<int64_t>(me) + (me == cs ? 1 : 0);
      float* po = p.partial_o + (slot * kTileRows + r) * D + col;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) po[e] = acc[e];
      if ((threadIdx.x & 15) == 0) {
        p.partial_ml[(slot * kTileRows + r) * 2] = m;
        p.partial_ml[(slot * kTileRows + r) * 2 + 1] = l;
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        s_last = atomicAdd(p.counters + cs, 1) == ce - cs;
        if (s_last) p.counters[cs] = 0;  // every other CTA of the item has arrived
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        final = true;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) acc[e] = 0.f;
        for (int c = cs; c <= ce; ++c) {
          const int64_t sl = 2 * static_cast<int64_t>(c) + (c == cs ? 1 : 0);
          const float mk = p.partial_ml[(sl * kTileRows + r) * 2];
          const float lk = p.partial_ml[(sl * kTileRows + r) * 2 + 1];
          const float mn = fmaxf(m, mk);
          const float fa = m == -INFINITY ? 0.f : exp2f(m - mn);
          const float fb = mk == -INFINITY ? 0.f : exp2f(mk - mn);
          const float* src = p.partial_o + (sl * kTileRows + r) * D + col;
          l = l * fa + lk * fb;
#pragma unroll
          for (int e = 0; e < D / 16; ++e) acc[e] = acc[e] * fa + src[e] * fb;
          m = mn;
        }
      }
    }
    if (final && row_base + r < rows) {
      const int tok = at.req.q0 + (row_base + r) / p.group;
      const int head = at.head * p.group + (row_base + r) % p.group;
      const float inv = l != 0.f ? 1.f / l : 0.f;
      uint16_t* dst = p.out + tok * p.out_token_stride + head * p.out_head_stride + col;
      uint32_t packed[D / 32];
#pragma unroll
      for (int e = 0; e < D / 32; ++e) packed[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      if constexpr (D == 128)
        *reinterpret_cast<uint4*>(dst) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      else
        *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
      if (p.lse != nullptr && (threadIdx.x & 15) == 0)
        p.lse[static_cast<int64_t>(tok) * p.q_heads + head] =
            l != 0.f ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
    }
    w += s.units;
    if (w < w_end) attn_advance<kTileRows>(p, at);
    __syncthreads();  // the merge area is free for the next segment's loads
  }
}

int attn_ctas() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 148;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = n < kAttnMaxCtas ? n : kAttnMaxCtas;
  }
  return cached[dev];
}

// The workspace: counters, then the partial sums and accumulators of 2 partials per CTA.
struct Workspace {
  static constexpr int64_t kCounterBytes = 2 * kAttnMaxCtas * 4;
  static int64_t ml_bytes() { return static_cast<int64_t>(2) * attn_ctas() * kAttnMaxPartialRows * 8; }
  static int64_t o_bytes() {
    return static_cast<int64_t>(2) * attn_ctas() * kAttnMaxPartialRows * 128 * 4;
  }
  static int64_t bytes() { return kCounterBytes + ml_bytes() + o_bytes(); }
};

template <int D>
int launch_rows(const AttnParams& p, cudaStream_t s) {
  const size_t smem = RowsSmem<D>::kBytes + (static_cast<size_t>(p.num_requests) + 1) * 4;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: device index >= 64");
  if (!done[dev]) {
    const int rc = check_cuda(
        cudaFuncSetAttribute(paged_attn_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             RowsSmem<D>::kBytes + (kAttnMaxRequests + 1) * 4),
        "lm_paged_attention: smem attribute");
    if (rc) return rc;
    done[dev] = true;
  }
  return check_cuda(launch_dependent(paged_attn_rows_kernel<D>, dim3(attn_ctas()), dim3(kThreads),
                                     smem, s, p),
                    "lm_paged_attention");
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int64_t lm_paged_attention_workspace_bytes(void) { return Workspace::bytes(); }

extern "C" int lm_paged_attention(
    const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const uint16_t* k_cache,
    int64_t k_page_stride, int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v_cache,
    int64_t v_page_stride, int64_t v_token_stride, int64_t v_head_stride, int64_t num_pages,
    int32_t page_size, const int32_t* block_tables, int64_t table_stride, int32_t max_pages,
    const int32_t* seq_lens, const int32_t* cu_q, int32_t num_requests, int64_t num_tokens,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_q_len, float scale,
    int32_t window, uint16_t* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
    void* workspace, int64_t workspace_bytes, int32_t* err_word, void* stream) {
  if (head_dim != 64 && head_dim != 128)
    return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: head_dim must be 64 or 128");
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_paged_attention: num_q_heads must be a multiple of num_kv_heads");
  if (page_size <= 0 || page_size % 16 != 0)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_paged_attention: page_size must be a multiple of 16");
  if (num_requests < 0 || num_requests > kAttnMaxRequests || num_tokens < 0 ||
      num_tokens * num_q_heads > 0x7fffffff || num_pages < 0 || num_pages > 0x7fffffff ||
      max_pages <= 0 || table_stride < max_pages || max_q_len < 0 || window < 0 ||
      static_cast<int64_t>(max_pages) * page_size > 0x7fffffff - 128)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_paged_attention: bad sizes (at most 4096 requests)");
  if (num_requests == 0 || num_tokens == 0) return LM_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_tables == nullptr ||
      seq_lens == nullptr || cu_q == nullptr || out == nullptr || workspace == nullptr)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_paged_attention: null pointer");
  if (workspace_bytes < Workspace::bytes())
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_paged_attention: the workspace is smaller than lm_paged_attention_workspace_bytes()");
  const int64_t strides = q_token_stride | q_head_stride | k_page_stride | k_token_stride |
                          k_head_stride | v_page_stride | v_token_stride | v_head_stride |
                          out_token_stride | out_head_stride;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
        reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) != 0 || (strides & 7) != 0)
    return fail(LM_ERR_INVALID_ARGUMENT,
                "lm_paged_attention: bases must be 16-byte aligned and strides multiples of 8 elements");
  AttnParams p{};
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.out = out;
  p.lse = lse;
  p.tables = block_tables;
  p.seq_lens = seq_lens;
  p.cu_q = cu_q;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.counters = reinterpret_cast<int32_t*>(ws);
  p.partial_ml = reinterpret_cast<float*>(ws + Workspace::kCounterBytes);
  p.partial_o = reinterpret_cast<float*>(ws + Workspace::kCounterBytes + Workspace::ml_bytes());
  p.err = err_word;
  p.q_token_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.out_token_stride = out_token_stride;
  p.out_head_stride = out_head_stride;
  p.k_page_stride = k_page_stride;
  p.k_token_stride = k_token_stride;
  p.k_head_stride = k_head_stride;
  p.v_page_stride = v_page_stride;
  p.v_token_stride = v_token_stride;
  p.v_head_stride = v_head_stride;
  p.table_stride = table_stride;
  p.num_tokens = num_tokens;
  p.num_requests = num_requests;
  p.q_heads = num_q_heads;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.page_size = page_size;
  p.num_pages = static_cast<int>(num_pages);
  p.max_pages = max_pages;
  p.window = window;
  p.scale_log2 = scale * 1.44269504088896341f;
  p.min_rows = 1;
  p.max_rows = 0x7fffffff;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Requests of up to 16 rows per kv head read K and V for one small tile: the row kernel. More
  // rows go to the tensor-core kernel. With what the host knows, one launch is often enough.
  const bool any_long = static_cast<int64_t>(max_q_len) * p.group > kTileRows;
  const bool any_short = p.group <= kTileRows && num_requests > 1;
  if (any_long) {
    if (any_short) p.min_rows = kTileRows + 1;
    const int rc = attn_launch_umma(p, head_dim, attn_ctas(), s);
    if (rc || !any_short) return rc;
    p.min_rows = 1;
    p.max_rows = kTileRows;
  }
  return head_dim == 64 ? launch_rows<64>(p, s) : launch_rows<128>(p, s);
}
