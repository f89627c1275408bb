// Attention over the paged cache for requests with many query rows: the tensor-core kernel.
//
// A CTA works on tiles of 256 rows of one (request, kv head), as two streams of 128 rows, against
// blocks of 128 keys. S = Q K^T and O += P V are tcgen05 MMAs (fp32 accumulators in TMEM: S and O
// of both streams fill its 512 columns); P is written back over S's columns as bf16 and read from
// TMEM as the A operand. One warp issues the MMAs, in the order PV(0), S(0), PV(1), S(1), so the
// tensor pipe works on one stream while the other stream's 128 softmax threads (a row each) turn
// S into P. One warp loads K and V by TMA, a box per cache page (or per 128 keys of a larger one),
// into a ring of 32 KB tiles; pages that are out of range are boxes past the cache's end, which
// TMA fills with zeros, and the MMA warp zeroes the V rows past a sequence's end inside a page.
//
// A row's reference maximum moves (and O is rescaled) only when a block's maximum exceeds it by
// more than 2^8: exp2 of the difference then stays within fp32 and bf16 range, and the division by
// the sum at the end takes the reference out again.
#include "lm_attn.cuh"

namespace lm {
namespace {

constexpr int kRowsPerStream = 128;
constexpr int kTile = 2 * kRowsPerStream;
constexpr int kBlk = kAttnBlock;
constexpr int kThreads = 384;
constexpr float kRescaleAbove = 8.f;  // log2

template <int D>
struct UmmaCfg {
  static constexpr int kHalf = kBlk * 128;              // 128 rows of 64 values, 128B-swizzled
  static constexpr int kTileBytes = kHalf * (D / 64);   // a K, V or Q tile
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTileBytes + 1024;
};

struct Ctrl {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_ready[2], s_full[2], p_ready[2], o_full[2];
  uint32_t tmem_base;
  int abort_flag;
  int last[2];
};

// D[tmem] (+)= A[tmem] x B[smem desc], bf16 inputs, fp32 accumulate.
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of a tile whose rows are the K dimension (128 B of 64 N values each, 128B swizzle):
// atoms of 8 rows follow each other at 1024 B (SBO), the next 64 N values are at `n_stride` (LBO).
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t n_stride) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(n_stride >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Barrier among the 128 threads of one stream (ids 1 and 2; 0 is __syncthreads).
__device__ __forceinline__ void stream_sync(int stream) {
  if (stream == 0)
    asm volatile("bar.sync 1, 128;" ::: "memory");
  else
    asm volatile("bar.sync 2, 128;" ::: "memory");
}

// Blocks [begin, end) of a segment that rows of stream `st` see, and whether it has rows at all.
struct StreamRange {
  int begin, end;
  bool active;
};

__device__ __forceinline__ StreamRange stream_range(const AttnParams& p, const AttnCursor& c,
                                                    const AttnSegment& s, int st) {
  StreamRange r;
  const int tile = 2 * c.tile + st;
  r.active = tile * kRowsPerStream < c.req.qlen * p.group;
  r.begin = r.end = s.blk0;
  if (r.active) {
    int lo, hi;
    attn_tile_keys<kRowsPerStream>(p, c.req, tile, lo, hi);
    if (hi > lo) {
      r.begin = max(s.blk0, lo / kBlk);
      r.end = max(r.begin, min(s.blk1, (hi + kBlk - 1) / kBlk));
    }
  }
  return r;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_umma_kernel(const __grid_constant__ AttnLaunch up) {
  using C = UmmaCfg<D>;
  const AttnParams& p = up.a;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Ctrl c;
  __shared__ int32_t s_warp[kThreads / 32];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem;                       // [2][kTileBytes]
  unsigned char* s_kv = smem + 2 * C::kTileBytes;  // [kStages][kTileBytes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&c.kv_full[i], 1);
      mbar_init(&c.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.q_ready[i], kRowsPerStream);
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.p_ready[i], kRowsPerStream);
      mbar_init(&c.o_full[i], 1);
    }
    c.abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&up.maps.k);
    tma_prefetch_desc(&up.maps.v);
  }
  pdl_wait();
  pdl_trigger();
  // the prefix lies where Q goes later
  int32_t* s_prefix = reinterpret_cast<int32_t*>(s_q);
  attn_prefix<kTile, kBlk, kThreads>(p, s_prefix, s_warp);
  const int total = s_prefix[p.num_requests];
  const int per = (total + gridDim.x - 1) / gridDim.x;
  const int w0 = blockIdx.x * per;
  const int w_end = min(total, w0 + per);
  if (w0 >= w_end) return;  // the whole CTA; nothing is allocated yet
  AttnCursor at = attn_seek<kTile, kBlk>(p, s_prefix, w0);
  if (warp == 8) {
    tmem_alloc(&c.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem_base;
  volatile int* abort_flag = &c.abort_flag;

  // 256 softmax threads of 216 registers and 128 others of 72: the 384 x 168 of the launch
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 9) {
    // ---------------------------------------------------------------------- K / V loader
    attn_load_kv<D, kTile, C::kStages, 2>(up, at, w0, w_end, s_kv, C::kTileBytes, c.kv_full, c.kv_empty,
                                          abort_flag);
  } else if (warp == 8) {
    // ---------------------------------------------------------------------- MMA issuer
    const uint32_t idesc_s = idesc_bf16_f32(kRowsPerStream, kBlk);
    const uint32_t idesc_o = idesc_bf16_f32(kRowsPerStream, D) | (1u << 16);  // B is N-major
    const uint32_t q_addr = smem_u32(s_q), kv_addr = smem_u32(s_kv);
    uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    int seq = 0;  // K tiles of block n: 2 n, V tiles: 2 n + 1
    bool ok = true;
    for (int w = w0; w < w_end && ok;) {
      const AttnSegment s = attn_segment<kTile, kBlk>(p, at, w, w_end);
      const StreamRange r0 = stream_range(p, at, s, 0), r1 = stream_range(p, at, s, 1);
#pragma unroll 1
      for (int st = 0; st < 2 && ok; ++st) {
        const StreamRange& r = st ? r1 : r0;
        if (r.end > r.begin) {
          ok = warp_wait(&c.q_ready[st], q_phase[st], p.err, abort_flag);
          q_phase[st] ^= 1u;
        }
      }
      for (int blk = s.blk0 - 1; blk < s.blk1 && ok && s.blk1 > s.blk0; ++blk) {
        // S of block blk + 1, P V of block blk
        const int ks = (seq + 2) % C::kStages, vs = (seq + 1) % C::kStages;
        const bool has_k = blk + 1 < s.blk1, has_v = blk >= s.blk0;
        const int k_seq = has_v ? seq + 2 : seq, v_seq = seq + 1;
        const int k_stage = has_v ? ks : seq % C::kStages;
        if (has_k)
          ok = warp_wait(&c.kv_full[k_stage], static_cast<uint32_t>(k_seq / C::kStages) & 1u,
                                 p.err, abort_flag);
        if (has_v && ok) {
          ok = warp_wait(&c.kv_full[vs], static_cast<uint32_t>(v_seq / C::kStages) & 1u, p.err,
                                 abort_flag);
          // V rows of keys outside the tile's range, in a page that is partly inside
          const int r_lo = s.lo - blk * kBlk, r_hi = s.hi - blk * kBlk;
          if (ok && (r_lo > 0 || r_hi < kBlk)) {
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (int i = lane; i < kBlk * (D / 8); i += 32) {
              const int row = i / (D / 8), ch = i % (D / 8);
              if (row < r_lo || row >= r_hi)
                *reinterpret_cast<uint4*>(s_kv + vs * C::kTileBytes + (ch / 8) * C::kHalf + row * 128 +
                                          (ch % 8) * 16) = zero;
            }
            fence_async_shared();
            __syncwarp();
          }
        }
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int st = 0; st < 2; ++st) {
          const StreamRange& r = st ? r1 : r0;
          const uint32_t t_s = tmem + st * 256, t_o = t_s + 128;
          if (blk >= r.begin && blk < r.end) {
            if (!warp_wait(&c.p_ready[st], p_phase[st], p.err, abort_flag)) {
              ok = false;
              break;
            }
            p_phase[st] ^= 1u;
            tc_fence_after();
            if (lane == 0) {
              const uint32_t v = kv_addr + vs * C::kTileBytes;
#pragma unroll
              for (int k = 0; k < kBlk / 16; ++k)
                umma_bf16_ts(t_o, t_s + k * 8, sdesc_mn_sw128(v + k * 2048, C::kHalf), idesc_o,
                             (blk > r.begin || k > 0) ? 1u : 0u);
              if (blk == r.end - 1) umma_commit(&c.o_full[st]);
            }
            __syncwarp();
          }
          if (blk + 1 >= r.begin && blk + 1 < r.end) {
            if (lane == 0) {
              const uint32_t q = q_addr + st * C::kTileBytes, k0 = kv_addr + k_stage * C::kTileBytes;
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k / 4) * C::kHalf + (k % 4) * 32;
                umma_bf16(t_s, sdesc_k_sw128(q + off), sdesc_k_sw128(k0 + off), idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit(&c.s_full[st]);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        if (lane == 0) {
          if (has_v) umma_commit(&c.kv_empty[vs]);
          if (has_k) umma_commit(&c.kv_empty[k_stage]);
        }
        __syncwarp();
        if (has_v) seq += 2;
      }
      w += s.units;
      if (w < w_end) attn_advance<kTile>(p, at);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------------------------------------------------------------- softmax: a row per thread
    const int st = warp >> 2, row = threadIdx.x & 127;
    const uint32_t t_s = tmem + st * 256 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_o = t_s + 128;
    uint32_t s_phase = 0, o_phase = 0;
    // A wait that gave up is recorded and stops the loader and the MMA warp; the rows go on to the
    // end over whatever TMEM holds (every later wait returns at once), so that barriers match.
    for (int w = w0; w < w_end;) {
      const AttnSegment s = attn_segment<kTile, kBlk>(p, at, w, w_end);
      const StreamRange r = stream_range(p, at, s, st);
      if (r.active) {
        const int rows = at.req.qlen * p.group, cached = at.req.seq - at.req.qlen;
        const int fr = at.tile * kTile + st * kRowsPerStream + row;  // flattened row
        const bool live = fr < rows;
        const int t = fr / p.group, head = at.head * p.group + fr % p.group;
        if (r.end > r.begin) {
          const uint16_t* src = p.q + (at.req.q0 + t) * p.q_token_stride + head * p.q_head_stride;
          const uint32_t flip = up.negate_q ? 0x80008000u : 0u;
#pragma unroll
          for (int ch = 0; ch < D / 8; ++ch) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live) {
              v = *reinterpret_cast<const uint4*>(src + ch * 8);
              v.x ^= flip;
              v.y ^= flip;
              v.z ^= flip;
              v.w ^= flip;
            }
            *reinterpret_cast<uint4*>(s_q + st * C::kTileBytes + (ch / 8) * C::kHalf + row * 128 +
                                      (((ch % 8) ^ (row & 7)) << 4)) = v;
          }
          fence_async_shared();
          mbar_arrive(&c.q_ready[st]);
        }
        // keys (j > low, j <= high) of this row, and of the stream's first and last row
        const int high = live ? cached + t : -1;
        const int low = p.window > 0 ? cached + t - p.window : -1;
        const int f_row = at.tile * kTile + st * kRowsPerStream;
        const int high_min = cached + f_row / p.group;
        const int low_max =
            p.window > 0 ? cached + (min(f_row + kRowsPerStream, rows) - 1) / p.group - p.window : -1;
        float m = -INFINITY, l = 0.f;
        for (int blk = r.begin; blk < r.end; ++blk) {
          mbar_wait_bounded(&c.s_full[st], s_phase, p.err, abort_flag);
          s_phase ^= 1u;
          tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_s + i * 32, x[i]);
          tmem_ld_wait();
          const int j0 = blk * kBlk;
          if (j0 + kBlk - 1 > high_min || j0 <= low_max) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int j = j0 + i * 32 + e;
                if (j > high || j <= low) x[i][e] = 0xff800000u;
              }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(x[i][e]));
          mx *= p.scale_log2;
          const bool move = mx > m + kRescaleAbove || (m == -INFINITY && mx > m);
          if (__any_sync(0xffffffffu, move)) {
            const float nm = move ? mx : m;
            const float f = move ? (m == -INFINITY ? 0.f : ex2(m - nm)) : 1.f;
            m = nm;
            l *= f;
            if (blk > r.begin) {
#pragma unroll 1
              for (int i = 0; i < D / 32; ++i) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(t_o + i * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st_32x32b_x32(t_o + i * 32, o);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : -m;
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float a = ex2(fmaf(__uint_as_float(x[i][2 * e]), p.scale_log2, base));
              const float b = ex2(fmaf(__uint_as_float(x[i][2 * e + 1]), p.scale_log2, base));
              sum0 += a;
              sum1 += b;
              packed[e] = pack_bf16x2(a, b);
            }
            tmem_st_32x32b_x16(t_s + i * 16, packed);
          }
          l += sum0 + sum1;
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&c.p_ready[st]);
        }
        if (r.end > r.begin) {
          mbar_wait_bounded(&c.o_full[st], o_phase, p.err, abort_flag);
          o_phase ^= 1u;
          tc_fence_after();
        }
        bool final = s.whole;
        int cs = 0, ce = -1;
        if (!s.whole) {
          cs = s.start / per;
          ce = (s.end - 1) / per;
          const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (blockIdx.x == cs ? 1 : 0);
          // [D][256 rows]: the threads of a warp store neighbouring rows
          float* po = p.partial_o + slot * (kTile * D) + st * kRowsPerStream + row;
          if (r.end > r.begin) {
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + i * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) po[(i * 32 + e) * kTile] = __uint_as_float(o[e]);
            }
          }
          float* pml = p.partial_ml + (slot * kTile + st * kRowsPerStream + row) * 2;
          pml[0] = m;
          pml[1] = l;  // 0: nothing seen, and perhaps no accumulator written
          __threadfence();
          stream_sync(st);
          if (row == 0) {
            int32_t* counter = p.counters + 2 * cs + st;
            c.last[st] = atomicAdd(counter, 1) == ce - cs;
            if (c.last[st]) *counter = 0;  // every other CTA of the item has arrived
          }
          stream_sync(st);
          final = c.last[st] != 0;
          if (final) __threadfence();
        }
        if (final) {
          uint16_t* dst = p.out + (at.req.q0 + t) * p.out_token_stride + head * p.out_head_stride;
          if (s.whole) {
            const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              uint32_t o[32];
              if (r.end > r.begin) {
                tmem_ld_32x32b_x32(t_o + i * 32, o);
                tmem_ld_wait();
              }
              if (live) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  uint32_t q[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    q[e] = l != 0.f ? pack_bf16x2(__uint_as_float(o[v * 8 + 2 * e]) * inv,
                                                 __uint_as_float(o[v * 8 + 2 * e + 1]) * inv)
                                   : 0u;
                  *reinterpret_cast<uint4*>(dst + i * 32 + v * 8) = make_uint4(q[0], q[1], q[2], q[3]);
                }
              }
            }
          } else {
            // partials of CTAs cs .. ce, in the order of the keys
            m = -INFINITY;
            l = 0.f;
            for (int k = cs; k <= ce; ++k) {
              const int64_t slot = 2 * static_cast<int64_t>(k) + (k == cs ? 1 : 0);
              const float* pml = p.partial_ml + (slot * kTile + st * kRowsPerStream + row) * 2;
              if (pml[1] != 0.f) m = fmaxf(m, pml[0]);
            }
            for (int k = cs; k <= ce; ++k) {
              const int64_t slot = 2 * static_cast<int64_t>(k) + (k == cs ? 1 : 0);
              const float* pml = p.partial_ml + (slot * kTile + st * kRowsPerStream + row) * 2;
              if (pml[1] != 0.f) l += pml[1] * ex2(pml[0] - m);
            }
            const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll 1
            for (int i = 0; i < D / 8; ++i) {
              float acc[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[e] = 0.f;
              for (int k = cs; k <= ce; ++k) {
                const int64_t slot = 2 * static_cast<int64_t>(k) + (k == cs ? 1 : 0);
                const float* pml = p.partial_ml + (slot * kTile + st * kRowsPerStream + row) * 2;
                if (pml[1] != 0.f) {
                  const float f = ex2(pml[0] - m);
                  const float* po = p.partial_o + slot * (kTile * D) + st * kRowsPerStream + row;
#pragma unroll
                  for (int e = 0; e < 8; ++e) acc[e] += f * po[(i * 8 + e) * kTile];
                }
              }
              if (live)
                *reinterpret_cast<uint4*>(dst + i * 8) =
                    make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                               pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
            }
          }
          if (live && p.lse != nullptr)
            p.lse[static_cast<int64_t>(at.req.q0 + t) * p.q_heads + head] =
                l != 0.f ? (m + log2f(l)) * 0.693147180559945309f : -INFINITY;
        }
        tc_fence_before();  // O is read before the next segment's P V overwrites it
      }
      w += s.units;
      if (w < w_end) attn_advance<kTile>(p, at);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
int launch(const AttnLaunch& p, int ctas, cudaStream_t s) {
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: device index >= 64");
  if (!done[dev]) {
    const int rc = check_cuda(cudaFuncSetAttribute(paged_attn_umma_kernel<D>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   UmmaCfg<D>::kSmem),
                              "lm_paged_attention: smem attribute");
    if (rc) return rc;
    done[dev] = true;
  }
  return check_cuda(launch_dependent(paged_attn_umma_kernel<D>, dim3(ctas), dim3(kThreads),
                                     UmmaCfg<D>::kSmem, s, p),
                    "lm_paged_attention");
}

}  // namespace

int attn_launch_umma(const AttnParams& a, const AttnMaps& maps, int head_dim, int ctas, cudaStream_t s) {
  AttnLaunch p;
  p.a = a;
  p.maps = maps;
  // Q's sign takes a negative scale's, so that a row's largest S has its largest weight; with a
  // scale of 0 the masked scores (-inf) still have to vanish.
  p.negate_q = a.scale_log2 < 0.f;
  if (p.negate_q) p.a.scale_log2 = -a.scale_log2;
  if (a.scale_log2 == 0.f) p.a.scale_log2 = 1e-30f;
  return head_dim == 64 ? launch<64>(p, ctas, s) : launch<128>(p, ctas, s);
}

}  // namespace lm
