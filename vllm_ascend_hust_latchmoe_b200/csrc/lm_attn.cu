// Attention of a step's new tokens over the paged cache:
//   out = softmax(q k^T * scale over the keys that the row sees) v,   lse = max + ln(sum)
// A row at position p sees key j when j <= p and (window == 0 or j > p - window); a row that sees
// nothing gives zeros and an lse of -inf. One pass over the keys with the running maximum and sum
// (fp32, in the log2 domain).
//
// This kernel takes 16-row tiles: single tokens and small chunks, where reading K and V is the
// cost. Two loader warps stream 128-key blocks of K and of V by TMA (a box per page, or per 128 keys
// of a larger one) into a ring of three 64 KB stages and run ahead into the CTA's next segments, so
// that the stream does not stop where a segment ends. Of a block each of 8 consumer warps takes 16
// keys and keeps its own running results; they are merged in shared memory (over the stage that
// they read last) at the end of a segment. Segments of an item that several CTAs share are merged
// through the workspace, by the CTA that arrives last, in the order of the keys.
#include <algorithm>
#include <atomic>

#include "lm_attn.cuh"
#include "lm_attn_ring.cuh"
#include "lm_tmap.cuh"

namespace lm {
namespace {

constexpr int kWarps = 8;       // consumers
constexpr int kConsumerThreads = kWarps * 32;
constexpr int kThreads = (kWarps + 3) * 32;  // and a loader each for K, V and Q
constexpr int kTileRows = 16;
constexpr int kSlice = 16;  // keys per warp and block
constexpr int kBlock = kAttnBlock;
// What an item costs beside its blocks, in blocks (its queries, its merge, a pipeline that runs dry):
// 512 single tokens over 1 .. 1000 keys each, 40 query heads on 8, 282 us at 0, 220 at 1, 204 at 2,
// 208 at 3 (189 since items became cheaper); 64 over 1 .. 2000 keys, 32 heads on 4, 46, 37, 37 and
// 38 us. The price: few short items spread over fewer CTAs (4 tokens over 1000 keys 10.8 -> 11.8 us).
constexpr int kItem = 2;
static_assert(kBlock == kWarps * kSlice, "a slice of every block per warp");

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
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kHalf = kBlock * 128;         // 128 keys of 64 values
  static constexpr int kTile = kHalf * (D / 64);     // K or V of a block
  static constexpr int kStage = 2 * kTile;           // also 8 warps' 16 rows of D fp32
  static constexpr int kRing = kStages * kStage;
  static constexpr int kQ = kTileRows * D * 2;
  static constexpr int kBytes = kRing + 2 * kQ + 1024;
};

struct RowsCtrl {
  uint64_t full[8], empty[8];
  uint64_t q_full[2], q_empty[2];
  float ml[kWarps][kTileRows][2];
  int abort_flag;
  int last;
};

// 16-byte chunk c of key row r of a K or V tile, as TMA's 128-byte swizzle lays it.
template <int D>
__device__ __forceinline__ uint32_t kv_at(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * RowsSmem<D>::kHalf + r * 128 + (((c ^ r) & 7) << 4));
}

// The same of a row of Q, [16][D].
template <int D>
__device__ __forceinline__ uint32_t q_at(int r, int c) {
  return static_cast<uint32_t>(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

__device__ __forceinline__ void consumer_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kConsumerThreads) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_rows_kernel(const __grid_constant__ AttnLaunch up) {
  using S = RowsSmem<D>;
  const AttnParams& p = up.a;
  constexpr int kChunks = D / 8;  // 16-byte chunks per row
  extern __shared__ unsigned char smem_raw[];
  __shared__ int32_t s_warp[kThreads / 32];
  __shared__ RowsCtrl c;
  __shared__ int s_longest;
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem + S::kRing;
  int32_t* s_prefix = reinterpret_cast<int32_t*>(s_q + 2 * S::kQ);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&c.full[i], 2);
      mbar_init(&c.empty[i], kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.q_full[i], 32);
      mbar_init(&c.q_empty[i], kWarps);
    }
    c.abort_flag = 0;
    s_longest = 0;
    fence_mbarrier_init();
  }
  __syncthreads();  // the barriers and s_longest are set
  if (warp == kWarps && lane == 0) {
    tma_prefetch_desc(&up.maps.k);
    tma_prefetch_desc(&up.maps.v);
  }
  // Beside the tensor-core kernel of the same call, which touches other rows and another workspace:
  // this one starts when all of that one's CTAs have started, so all earlier kernels are complete,
  // and takes the SMs that it leaves. It waits for it at its end, so that whoever waits for this
  // kernel has waited for both.
  if (!up.beside) pdl_wait();
  pdl_trigger();
  int per, w, w_end;
  AttnCursor at;
  if (!attn_locate<kTileRows, kBlock, kItem, kThreads, false>(p, s_prefix, s_warp, &s_longest, per, w, w_end,
                                                              at)) {
    pdl_wait();  // the whole CTA
    return;
  }
  volatile int* abort_flag = &c.abort_flag;

  if (warp < kWarps + 2 && warp >= kWarps) {
    const bool is_v = warp == kWarps + 1;
    attn_load_kv<D, kTileRows, kItem, S::kStages>(up, is_v, at, w, w_end, smem + (is_v ? S::kTile : 0), S::kStage,
                                                  0, 1, c.full, c.empty, abort_flag);
    pdl_wait();
    return;
  }
  if (warp > kWarps) {
    // ------------------------------------------------------------------------ queries
    AttnQueryTurn turn;
    while (attn_has<kItem>(at, w, w_end)) {
      const AttnSegment s = attn_segment<kTileRows, kBlock, kItem>(p, at, w, w_end);
      if (turn.has_keys(s.blk0, s.blk1)) {
        const int buf = turn.buffer();
        if (!warp_wait(&c.q_empty[buf], turn.empty_parity(), p.err, abort_flag)) break;
        const int rows = at.req.qlen * p.group;
        unsigned char* dst = s_q + buf * S::kQ;
#pragma unroll
        for (int j = 0; j < kTileRows * kChunks / 32; ++j) {
          const int r = (j * 32 + lane) / kChunks, ch = (j * 32 + lane) % kChunks;
          const int row = at.tile * kTileRows + r;
          const int t = p.by_group(row), head = at.head * p.group + row - t * p.group;
          const uint16_t* src = p.q + (at.req.q0 + t) * p.q_token_stride + head * p.q_head_stride + ch * 8;
          cp_async_16(dst + q_at<D>(r, ch), row < rows ? src : p.q, row < rows ? 16u : 0u);
        }
        cp_async_arrive_noinc(&c.q_full[buf]);
        turn.next();
      }
      w += s.units;
      if (w >= w_end) break;
      attn_advance<kTileRows>(p, at);
    }
    cp_async_wait_all();  // nothing in flight into shared memory when the warp leaves
    pdl_wait();
    return;
  }

  // -------------------------------------------------------------------------- consumers
  // A wait that gave up is recorded and stops the loaders; the consumers go on to the end over
  // whatever their stages hold (every later wait returns at once), so that their barriers match.
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  int seq = 0;
  AttnQueryTurn turn;
  while (attn_has<kItem>(at, w, w_end)) {
    const AttnSegment s = attn_segment<kTileRows, kBlock, kItem>(p, at, w, w_end);
    const int rows = at.req.qlen * p.group;
    const int row_base = at.tile * kTileRows;
    const int cached = at.req.seq - at.req.qlen;
    const int n_slices = s.blk1 - s.blk0;  // one slice of this warp per block

    uint32_t qf[D / 16][4];
    if (turn.has_keys(s.blk0, s.blk1)) {
      const int buf = turn.buffer();
      mbar_wait_bounded(&c.q_full[buf], turn.full_parity(), p.err, abort_flag);
      const uint32_t qa = smem_u32(s_q + buf * S::kQ);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)  // rows 0-7, 8-15, then the same 8 columns on
        ldmatrix_x4(qf[k], qa + q_at<D>(lane & 15, 2 * k + (lane >> 4)));
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.q_empty[buf]);
      turn.next();
    }

    // keys (j > low, j <= high) that rows g and g + 8 of the tile see
    const int r0 = row_base + g, r1 = r0 + 8;
    const int t0 = p.by_group(r0), t1 = p.by_group(r1);
    const int high0 = r0 < rows ? cached + t0 : -1;
    const int high1 = r1 < rows ? cached + t1 : -1;
    const int low0 = attn_hidden(p, cached + t0), low1 = attn_hidden(p, cached + t1);

    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int i = 0; i < n_slices; ++i, ++seq) {
      const int stage = seq % S::kStages;
      mbar_wait_bounded(&c.full[stage], static_cast<uint32_t>(seq / S::kStages) & 1u, p.err, abort_flag);
      unsigned char* tile = smem + stage * S::kStage;
      const uint32_t kt = smem_u32(tile), vt = kt + S::kTile;
      const int tok0 = (s.blk0 + i) * kBlock + warp * kSlice;
      if (tok0 < s.lo || tok0 + kSlice > s.hi) {
        // V rows outside the tile's range: what the cache holds there may be anything, and a weight
        // of zero does not undo an infinity
        __syncwarp();
        for (int x = lane; x < kSlice * kChunks; x += 32) {
          const int r = x / kChunks;
          if (tok0 + r < s.lo || tok0 + r >= s.hi)
            *reinterpret_cast<uint4*>(tile + S::kTile + kv_at<D>(warp * kSlice + r, x % kChunks)) =
                make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();  // ahead of the copy that fills the stage again
        __syncwarp();
      }
      float sc[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];  // keys 0-7: k halves 0, 1; keys 8-15: k halves 0, 1
        ldmatrix_x4(b, kt + kv_at<D>(warp * kSlice + (lane & 7) + ((lane & 16) >> 1), 2 * k + ((lane >> 3) & 1)));
        mma_bf16(sc[0], qf[k], b[0], b[1]);
        mma_bf16(sc[1], qf[k], b[2], b[3]);
      }
      const int j0 = tok0 + c2;
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
        const float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0);
        const float f1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
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
        const float e0 = ex2(sc[n][0] - b0), e1 = ex2(sc[n][1] - b0);
        const float e2 = ex2(sc[n][2] - b1), e3 = ex2(sc[n][3] - b1);
        l0 += e0 + e1;
        l1 += e2 + e3;
        pa[2 * n] = pack_bf16x2(e0, e1);
        pa[2 * n + 1] = pack_bf16x2(e2, e3);
      }
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b[4];  // d columns 16 n .. +7: keys 0-7, 8-15; columns +8: the same
        ldmatrix_x4_trans(b, vt + kv_at<D>(warp * kSlice + (lane & 15), 2 * n + (lane >> 4)));
        mma_bf16(o[2 * n], pa, b[0], b[1]);
        mma_bf16(o[2 * n + 1], pa, b[2], b[3]);
      }
      __syncwarp();
      // the last stage of the segment is kept: the results go there
      if (lane == 0 && i + 1 < n_slices) mbar_arrive(&c.empty[stage]);
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    const int last_stage = (seq + S::kStages - 1) % S::kStages;
    float* results = reinterpret_cast<float*>(smem + last_stage * S::kStage);  // [kWarps][16][D]
    consumer_sync();  // every warp is done with the segment's last block
    if (n_slices > 0) {
      float* dst = results + warp * kTileRows * D;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        // columns in blocks of 8, swapped by row: 8 rows of one block would share their banks
        *reinterpret_cast<float2*>(dst + g * D + (n ^ g) * 8 + c2) = make_float2(o[n][0], o[n][1]);
        *reinterpret_cast<float2*>(dst + (g + 8) * D + (n ^ g) * 8 + c2) = make_float2(o[n][2], o[n][3]);
      }
      fence_async_shared();
    }
    if ((lane & 3) == 0) {
      c.ml[warp][g][0] = m0;
      c.ml[warp][g][1] = l0;
      c.ml[warp][g + 8][0] = m1;
      c.ml[warp][g + 8][1] = l1;
    }
    consumer_sync();

    // 16 threads per row, D / 16 columns each
    constexpr int kCols = D / 16;
    const int r = threadIdx.x >> 4, col = (threadIdx.x & 15) * kCols;
    const bool live = row_base + r < rows;
    float m = -INFINITY, l = 0.f, acc[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) acc[e] = 0.f;
    if (n_slices > 0) {
#pragma unroll
      for (int k = 0; k < kWarps; ++k) m = fmaxf(m, c.ml[k][r][0]);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float mk = c.ml[k][r][0];
        const float f = mk == -INFINITY ? 0.f : ex2(mk - m);
        l += f * c.ml[k][r][1];
        const float* src = results + (k * kTileRows + r) * D + (((col >> 3) ^ (r & 7)) * 8 + (col & 7));
#pragma unroll
        for (int e = 0; e < kCols; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(src + e);
          acc[e] += f * v.x;
          acc[e + 1] += f * v.y;
          acc[e + 2] += f * v.z;
          acc[e + 3] += f * v.w;
        }
      }
    }
    consumer_sync();  // the stages and ml have been read
    if (n_slices > 0 && lane == 0) mbar_arrive(&c.empty[last_stage]);

    bool final = s.whole;
    if (!s.whole) {
      int cs, ce;
      attn_holders<kItem>(s, per, cs, ce);
      const int me = blockIdx.x;
      const int64_t slot = 2 * static_cast<int64_t>(me) + (me == cs ? 1 : 0);
      if (live) {
        float* po = p.partial_o + (slot * kTileRows + r) * D + col;
#pragma unroll
        for (int e = 0; e < kCols; e += 4)
          *reinterpret_cast<float4*>(po + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        if ((threadIdx.x & 15) == 0)
          *reinterpret_cast<float2*>(p.partial_ml + (slot * kTileRows + r) * 2) = make_float2(m, l);
      }
      consumer_sync();
      if (threadIdx.x == 0) c.last = attn_arrive(p.counters + cs, ce - cs + 1);
      consumer_sync();
      final = c.last != 0;
      if (final && live) {
        // the common maximum first (a row's 16 threads share the partials), so that the sums'
        // loads do not wait for one another
        auto slot_of = [&](int k) { return (2 * static_cast<int64_t>(k) + (k == cs ? 1 : 0)) * kTileRows + r; };
        auto ml_of = [&](int k) {
          return __ldcg(reinterpret_cast<const float2*>(p.partial_ml + slot_of(k) * 2));
        };
        const unsigned group = 0xffffu << (lane & 16);
        m = -INFINITY;
        for (int k = cs + (threadIdx.x & 15); k <= ce; k += 16) m = fmaxf(m, ml_of(k).x);
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor_sync(group, m, x));
        l = 0.f;
#pragma unroll
        for (int e = 0; e < kCols; ++e) acc[e] = 0.f;
#pragma unroll 8
        for (int k = cs; k <= ce; ++k) {
          const float2 ml = ml_of(k);
          const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
          const float* src = p.partial_o + slot_of(k) * D + col;
          l += f * ml.y;
#pragma unroll
          for (int e = 0; e < kCols; e += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src + e));
            acc[e] += f * v.x;
            acc[e + 1] += f * v.y;
            acc[e + 2] += f * v.z;
            acc[e + 3] += f * v.w;
          }
        }
      }
    }
    if (final && live) {
      const int t = p.by_group(row_base + r);
      const int tok = at.req.q0 + t;
      const int head = at.head * p.group + row_base + r - t * p.group;
      const float inv = l != 0.f ? 1.f / l : 0.f;
      uint16_t* dst = p.out + tok * p.out_token_stride + head * p.out_head_stride + col;
      uint32_t packed[kCols / 2];
#pragma unroll
      for (int e = 0; e < kCols / 2; ++e)
        packed[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      if constexpr (D == 128)
        *reinterpret_cast<uint4*>(dst) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      else
        *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
      if (p.lse != nullptr && (threadIdx.x & 15) == 0)
        p.lse[static_cast<int64_t>(tok) * p.q_heads + head] =
            l != 0.f ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
    }
    w += s.units;
    if (w >= w_end) break;
    attn_advance<kTileRows>(p, at);
  }
  pdl_wait();
}

int attn_ctas() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    n = 148;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    n = n < kAttnMaxCtas ? n : kAttnMaxCtas;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// The workspace: for either kernel its counters, and the sums and accumulators of 2 partial results
// per CTA (256 rows of the tensor-core kernel, 16 of the other).
struct Workspace {
  static int64_t counters() { return 2 * kAttnMaxCtas * 4; }
  static int64_t ml(int rows) { return static_cast<int64_t>(2) * attn_ctas() * rows * 8; }
  static int64_t o(int rows) { return static_cast<int64_t>(2) * attn_ctas() * rows * 128 * 4; }
  static int64_t part(int rows) { return counters() + ml(rows) + o(rows); }
  static int64_t bytes() { return part(kAttnMaxPartialRows) + part(kTileRows); }
  static void place(AttnParams* p, unsigned char* at, int rows) {
    p->counters = reinterpret_cast<int32_t*>(at);
    p->partial_ml = reinterpret_cast<float*>(at + counters());
    p->partial_o = reinterpret_cast<float*>(at + counters() + ml(rows));
  }
};

// The cache as (values, then tokens and heads by growing stride, pages); boxes of box_rows tokens of
// one head x 64 values.
int cache_map(CUtensorMap* out, const void* base, const AttnParams& a, int head_dim, int64_t page_stride,
              int64_t token_stride, int64_t head_stride, int box_rows, bool heads_first) {
  // a dimension of one has no stride of its own
  if (a.kv_heads == 1) head_stride = head_dim;
  if (a.num_pages == 1) page_stride = std::max(token_stride, head_stride);
  const int h = heads_first ? 1 : 2, t = 3 - h;
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4] = {64, 1, 1, 1};
  dims[0] = static_cast<cuuint64_t>(head_dim);
  dims[h] = static_cast<cuuint64_t>(a.kv_heads);
  dims[t] = static_cast<cuuint64_t>(a.page_size);
  dims[3] = static_cast<cuuint64_t>(a.num_pages);
  strides[h - 1] = static_cast<cuuint64_t>(head_stride) * 2;
  strides[t - 1] = static_cast<cuuint64_t>(token_stride) * 2;
  strides[2] = static_cast<cuuint64_t>(page_stride) * 2;
  box[t] = static_cast<cuuint32_t>(box_rows);
  return encode_bf16_map(out, 4, base, dims, strides, box);
}

template <int D>
int launch_rows(const AttnParams& a, const AttnMaps& maps, bool beside, cudaStream_t s) {
  AttnLaunch p;
  p.a = a;
  p.maps = maps;
  p.negate_q = 0;
  p.beside = beside;
  const size_t smem = RowsSmem<D>::kBytes + (static_cast<size_t>(a.num_requests) + 1) * 4;
  static std::atomic<bool> done[64];  // two threads may both set the attribute, to the same value
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: device index >= 64");
  if (!done[dev].load(std::memory_order_acquire)) {
    const int rc = check_cuda(
        cudaFuncSetAttribute(paged_attn_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             RowsSmem<D>::kBytes + (kAttnMaxRequests + 1) * 4),
        "lm_paged_attention: smem attribute");
    if (rc) return rc;
    done[dev].store(true, std::memory_order_release);
  }
  return check_cuda(launch_dependent(paged_attn_rows_kernel<D>, dim3(attn_ctas()), dim3(kThreads),
                                     smem, s, p),
                    "lm_paged_attention");
}

}  // namespace
}  // namespace lm

namespace lm {

int attn_make_maps(const AttnParams& a, int head_dim, AttnMaps* maps) {
  maps->box_rows = 16;
  while (maps->box_rows < kAttnBlock && a.page_size % (2 * maps->box_rows) == 0) maps->box_rows *= 2;
  const bool heads_first = a.k_head_stride <= a.k_token_stride && a.v_head_stride <= a.v_token_stride;
  maps->heads_first = heads_first;
  const int rc = cache_map(&maps->k, a.k, a, head_dim, a.k_page_stride, a.k_token_stride, a.k_head_stride,
                           maps->box_rows, heads_first);
  return rc ? rc
            : cache_map(&maps->v, a.v, a, head_dim, a.v_page_stride, a.v_token_stride, a.v_head_stride,
                        maps->box_rows, heads_first);
}

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
      num_tokens > 0x7fffffff || num_tokens * num_q_heads > 0x7fffffff - kAttnMaxPartialRows || num_pages < 0 || num_pages > 0x7fffffff ||
      max_pages <= 0 || table_stride < max_pages || max_q_len < 0 || window < 0 ||
      static_cast<int64_t>(max_pages) * page_size > 0x7fffffff - 128)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_paged_attention: bad sizes (at most 4096 requests)");
  if (num_requests == 0 || num_tokens == 0) return LM_OK;
  if (num_pages == 0) return fail(LM_ERR_INVALID_ARGUMENT, "lm_paged_attention: an empty cache");
  {  // the launches count their units (row tiles x key blocks and 3 at most for each) in 32 bits
    const bool small = static_cast<int64_t>(max_q_len) * (num_q_heads / num_kv_heads) <= kTileRows;
    const int64_t tiles = num_tokens * num_q_heads / (small ? kTileRows : 2 * 128) +
                          static_cast<int64_t>(num_requests) * num_kv_heads;
    const int64_t blocks = (static_cast<int64_t>(max_pages) * page_size + kBlock - 1) / kBlock + 1 + 3;
    if (tiles > (kAttnMaxUnits - 1) / blocks)
      return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: too much work for one call");
  }
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
  p.by_group = attn_div(p.group);
  p.page_size = page_size;
  p.by_page = attn_div(page_size);
  p.num_pages = static_cast<int>(num_pages);
  p.max_pages = max_pages;
  p.window = window;
  p.scale_log2 = scale * 1.44269504088896341f;
  p.min_rows = 1;
  p.max_rows = 0x7fffffff;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Requests of up to 16 rows per kv head read K and V for one small tile: the row kernel. More
  // rows go to the tensor-core kernel. A call with both kinds makes both launches, unless its short
  // requests can only be a little work (by the block table's width, all of them single tokens): the
  // tensor-core kernel takes 1.9 us for a block of keys and the row kernel 1.4, but a second launch
  // costs 3 to 6 us (a 512-token chunk beside 7 single tokens over 4000 keys, 32 heads on 4: 36 us in
  // one launch and 42 in two, beside 15 of them 42 and 45). The lengths are on the device and the width is
  // what the host knows, so a call with much wider tables than its requests fill takes two launches.
  const bool any_long = static_cast<int64_t>(max_q_len) * p.group > kTileRows;
  const int64_t short_units = static_cast<int64_t>(num_requests) * num_kv_heads *
                              ((static_cast<int64_t>(max_pages) * page_size + kBlock - 1) / kBlock);
  const bool any_short = p.group <= kTileRows && num_requests > 1 &&
                         short_units > 16 * static_cast<int64_t>(attn_ctas());
  AttnMaps maps;
  int rc = attn_make_maps(p, head_dim, &maps);
  if (rc) return rc;
  if (any_long) {
    Workspace::place(&p, ws, kAttnMaxPartialRows);
    if (any_short) p.min_rows = kTileRows + 1;
    rc = attn_launch_umma(p, maps, head_dim, attn_ctas(), s);
    if (rc || !any_short) return rc;
    p.min_rows = 1;
    p.max_rows = kTileRows;
  }
  Workspace::place(&p, ws + Workspace::part(kAttnMaxPartialRows), kTileRows);
  return head_dim == 64 ? launch_rows<64>(p, maps, any_long, s) : launch_rows<128>(p, maps, any_long, s);
}
