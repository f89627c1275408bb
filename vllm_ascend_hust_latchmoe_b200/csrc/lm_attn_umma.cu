// Attention over the paged cache for requests with many query rows: the tensor-core kernel.
//
// A CTA works on tiles of 256 rows of one (request, kv head), as two streams of 128 rows, against
// blocks of 128 keys. S = Q K^T and O += P V are tcgen05 MMAs (fp32 accumulators in TMEM: S and O
// of both streams fill its 512 columns); P is written back over S's columns as bf16 and read from
// TMEM as the A operand. A warp per stream issues its MMAs, P V of one block and then S of the next,
// so the tensor pipe works on one stream while the other stream's 128 softmax threads (a row each)
// turn S into P. Two warps load K and V by TMA, a box per cache page (or per 128 keys of a larger
// one), in turn into a ring of 32 KB tiles; pages that are out of range are boxes past the cache's end,
// which TMA fills with zeros, and the MMA warps zero the V rows past a sequence's end inside a page.
//
// The weights are rounded to bf16 as the MMA's operand (the error of an output then has sqrt(2) times
// the rms of its own rounding); their sum takes them unrounded.
//
// Measured: a 4096-token chunk over 16384 keys, 32 / 4 heads of 128: 731 to 760 us in short graph
// replays (1265 to 1316 TFLOP/s, 74 to 77 % of the burst GEMM rate), 850 to 875 us in stretches of seconds
// under the power cap (1100 to 1130 TFLOP/s, 77 to 80 % of the sustained rate). With heads of 64: 588 to
// 603 us, 800 TFLOP/s; at 16 exponentials a clock and SM its 1.9e9 of them take some 420 us, its MMAs
// 283 us at the burst rate. With heads of 128, a block pair takes some 3500 cycles: 2300 from S to P
// (read 160, maximum 400, exponentials 2 x 740) and 1200 from P to the next S, against 2048 of MMAs.
// Tried without gain: part of the exponentials on the FMA pipe (782 - 852 us for 1/8 to 1/2 of them),
// the first exponentials beside the maximum (884 us), the next item's Q begun ahead of its
// predecessor's last softmax (3 % slower), results exchanged between lanes for wider stores (a prompt
// of 4096 tokens -3 %, eight of 1024 +5 %), MMAs issued from a lane-0 branch (1011 us: 84 to
// 128 cycles an instruction against 70 with elect.sync and operands that the compiler sees uniform).
//
// A row's reference maximum moves (and O is rescaled) only when a block's maximum exceeds it by a
// factor of more than 2^24: weights, sums and O keep their relative precision (fp32 and bf16 have 8
// exponent bits), 2^100 of range is left for V and the number of keys, and the division by the sum
// at the end takes the reference out again. A move costs its stream some 700 cycles, and with a
// bound of 2^8 sharp heads moved one of 128 rows in most blocks.
#include <atomic>

#include "lm_attn.cuh"

namespace lm {
namespace {

constexpr int kRowsPerStream = 128;
constexpr int kTile = 2 * kRowsPerStream;
constexpr int kBlk = kAttnBlock;
// What an item costs beside its blocks, in blocks (its queries, masks and results; 7,000 to 9,000
// cycles against 3,100 for a block): a prompt of 4096 tokens, 64 query heads on 4, 469 us at 0, 318
// at 2, 277 at 3, 264 at 4, 272 at 6; 8 requests of 1 to 1000 new tokens over 3000 54.5, 51.6, 51.0,
// 52.1 and 53.4 us.
constexpr int kItem = 3;
constexpr int kThreads = 384;
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;  // per thread: 256 x 216 + 128 x 72 = 384 x 168
constexpr float kRescaleAbove = 24.f;  // log2

template <int D>
struct UmmaCfg {
  static constexpr int kHalf = kBlk * 128;              // 128 rows of 64 values, 128B-swizzled
  static constexpr int kTileBytes = kHalf * (D / 64);   // a K, V or Q tile
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTileBytes + 1024;
  // With D = 64 a stream's 256 TMEM columns hold S (128), O (64) and P (64) side by side, so S of the
  // next block is made while this block's weights are; with D = 128 P lies over S and S waits for P V.
  static constexpr bool kOwnP = D == 64;
  static constexpr int kColP = kOwnP ? 192 : 0;
};

struct Ctrl {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_ready[2], s_full[2], s_read[2], p_half[2], p_ready[2], o_full[2], turn[2];
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

// One thread of a converged warp. (Operands that the compiler can see are the same in the whole warp
// keep an MMA's issue short: see uniform().)
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

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

// Two floats in one register pair: the FMA pipe does both in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
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
  __shared__ int s_longest;
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* s_q = smem;                       // [2][kTileBytes]
  unsigned char* s_kv = smem + 2 * C::kTileBytes;  // [kStages][kTileBytes]
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&c.kv_full[i], 1);
      mbar_init(&c.kv_empty[i], 2);  // both streams'
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.q_ready[i], kRowsPerStream);
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.s_read[i], kRowsPerStream);
      mbar_init(&c.p_half[i], kRowsPerStream);
      mbar_init(&c.p_ready[i], kRowsPerStream);
      mbar_init(&c.o_full[i], 1);
      mbar_init(&c.turn[i], 1);
    }
    c.abort_flag = 0;
    s_longest = 0;
    fence_mbarrier_init();
  }
  __syncthreads();  // the barriers and s_longest are set
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&up.maps.k);
    tma_prefetch_desc(&up.maps.v);
  }
  pdl_wait();
  pdl_trigger();
  // the prefix lies where Q goes later
  int32_t* s_prefix = reinterpret_cast<int32_t*>(s_q);
  // A few long items are not cut into more pieces than pay: a block takes 1.9 us, another piece to
  // merge about as much, so n blocks are best cut into sqrt(n) pieces (16 items of 17 blocks: 42 us in
  // pieces of 4, 57 us in pieces of 2). Short items are not joined in a CTA for that.
  int per, w0, w_end;
  AttnCursor at;
  if (!attn_locate<kTile, kBlk, kItem, kThreads, true>(p, s_prefix, s_warp, &s_longest, per, w0, w_end, at))
    return;  // the whole CTA; nothing is allocated yet
  if (warp == 8) {
    tmem_alloc(&c.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(c.tmem_base);
  volatile int* abort_flag = &c.abort_flag;

  // the softmax threads' registers come from the other warps
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9 || warp == 11) {
      // ---------------------------------------------------------------------- K and V loaders
      attn_load_kv<D, kTile, kItem, C::kStages>(up, warp == 11, at, w0, w_end, s_kv, C::kTileBytes,
                                                warp == 11 ? 1 : 0, 2, c.kv_full, c.kv_empty, abort_flag);
    } else {
      // ---------------------------------------------------------------------- MMA issuers, one a stream
      const int st = warp == 8 ? 0 : 1;
      const uint32_t idesc_s = idesc_bf16_f32(kRowsPerStream, kBlk);
      const uint32_t idesc_o = idesc_bf16_f32(kRowsPerStream, D) | (1u << 16);  // B is N-major
      const uint32_t kv_addr = uniform(smem_u32(s_kv));
      const uint64_t q_desc = sdesc_k_sw128(uniform(smem_u32(s_q)) + st * C::kTileBytes);
      const uint32_t t_s = tmem + st * 256, t_o = t_s + 128;
      uint32_t q_phase = 0, p_phase = 0, kv_phase = 0;
      uint32_t turn_phase = st == 0 ? 1u : 0u;  // stream 0 begins
      int stage = 0;  // of the next tile, in the loader's order: K, V, K, V, ...
      bool ok = true;
      auto next_stage = [&]() {
        if (++stage == C::kStages) {
          stage = 0;
          kv_phase ^= 1u;
        }
      };
      auto release = [&](int tile, bool used) {  // after this stream's MMAs, if it had any
        if (elect_one()) {
          if (used)
            umma_commit(&c.kv_empty[tile]);
          else
            mbar_arrive(&c.kv_empty[tile]);
        }
        __syncwarp();
      };
      auto issue_s = [&](int tile) {
        const uint64_t k_desc = sdesc_k_sw128(uniform(kv_addr + tile * C::kTileBytes));
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = ((k / 4) * C::kHalf + (k % 4) * 32) >> 4;
            umma_bf16(t_s, q_desc + off, k_desc + off, idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&c.s_full[st]);
        }
        __syncwarp();
      };
      for (int w = w0; attn_has<kItem>(at, w, w_end) && ok;) {
        const AttnSegment s = attn_segment<kTile, kBlk, kItem>(p, at, w, w_end);
        const StreamRange r = stream_range(p, at, s, st);
        if (r.end > r.begin) {
          ok = warp_wait(&c.q_ready[st], q_phase, p.err, abort_flag);
          q_phase ^= 1u;
        }
        if (s.blk0 < s.blk1 && ok) {  // S of the first block
          ok = warp_wait(&c.kv_full[stage], kv_phase, p.err, abort_flag);
          if (!ok) break;
          const bool mine = s.blk0 == r.begin && r.end > r.begin;
          if (mine) issue_s(stage);
          release(stage, mine);
          next_stage();
        }
        for (int blk = s.blk0; blk < s.blk1; ++blk) {  // P V of blk, S of blk + 1
          const bool mine = blk >= r.begin && blk < r.end;
          const int v_tile = stage;
          const uint32_t v_phase = kv_phase;
          next_stage();
          if (blk + 1 < s.blk1) {
            ok = warp_wait(&c.kv_full[stage], kv_phase, p.err, abort_flag);  // K arrives after V
            if (!ok) break;
          }
          const bool next = blk + 1 >= r.begin && blk + 1 < r.end;
          if constexpr (C::kOwnP) {  // S of the next block as soon as this one's has been read
            if (mine) ok = warp_wait(&c.s_read[st], p_phase, p.err, abort_flag);
            if (!ok) break;
            if (next) issue_s(stage);
            if (blk + 1 < s.blk1) release(stage, next);
          }
          ok = warp_wait(&c.kv_full[v_tile], v_phase, p.err, abort_flag);
          if (!ok) break;
          // The streams take turns, so that one's softmax runs beside the other's MMAs; left alone they
          // fall into step, and exponentials and MMAs wait for their own kind (4096-token chunk over
          // 16384 keys: 1027 against 909 us when it was tried, and 681 against 588 us with D = 64).
          ok = warp_wait(&c.turn[st], turn_phase, p.err, abort_flag);
          if (!ok) break;
          turn_phase ^= 1u;
          if (mine) {
            // V rows of keys outside the tile's range, in a page that is partly inside (both streams
            // write the same zeros)
            const int r_lo = max(0, s.lo - blk * kBlk), r_hi = min(kBlk, s.hi - blk * kBlk);
            if (r_lo > 0 || r_hi < kBlk) {
              const uint4 zero = make_uint4(0, 0, 0, 0);
              for (int i = lane; i < (kBlk - (r_hi - r_lo)) * (D / 8); i += 32) {
                const int n = i / (D / 8), ch = i % (D / 8);
                const int row = n < r_lo ? n : n - r_lo + r_hi;
                *reinterpret_cast<uint4*>(s_kv + v_tile * C::kTileBytes + (ch / 8) * C::kHalf + row * 128 +
                                          (ch % 8) * 16) = zero;
              }
              fence_async_shared();
              __syncwarp();
            }
            const uint64_t v_desc = sdesc_mn_sw128(uniform(kv_addr + v_tile * C::kTileBytes), C::kHalf);
            const uint32_t accumulate = uniform(blk > r.begin ? 1u : 0u);
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              ok = ok && warp_wait(part ? &c.p_ready[st] : &c.p_half[st], p_phase, p.err, abort_flag);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int k = part * kBlk / 32; k < (part + 1) * kBlk / 32; ++k)
                  umma_bf16_ts(t_o, t_s + C::kColP + k * 8, v_desc + k * (2048 >> 4), idesc_o, k > 0 ? 1u : accumulate);
                if (part == 1 && (C::kOwnP || blk == r.end - 1)) umma_commit(&c.o_full[st]);
              }
              __syncwarp();
            }
            if (!ok) break;
            p_phase ^= 1u;
          }
          if (!C::kOwnP && next) issue_s(stage);
          if (elect_one()) mbar_arrive(&c.turn[1 - st]);
          release(v_tile, mine);
          if (blk + 1 < s.blk1) {
            if (!C::kOwnP) release(stage, next);
            next_stage();
          }
        }
        w += s.units;
        if (w >= w_end) break;
        attn_advance<kTile>(p, at);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------------------------------------------------------------- softmax: a row per thread
    const int st = warp >> 2, row = threadIdx.x & 127;
    const uint32_t t_s = tmem + st * 256 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_o = t_s + 128;
    uint32_t s_phase = 0, o_phase = 0;
    // A wait that gave up is recorded and stops the loader and the MMA warp; the rows go on to the
    // end over whatever TMEM holds (every later wait returns at once), so that barriers match.
    // This warp's 32 rows of a segment's Q into shared memory, D / 8 lanes to a row, whose place in
    // memory comes from the lane that the row belongs to. Asynchronous copies, all in flight
    // together; rows past the last are zeros.
    auto load_q = [&](const AttnCursor& q_at) {
      constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // per copy
      const int fr = q_at.tile * kTile + st * kRowsPerStream + row;
      const int t = p.by_group(fr), head = q_at.head * p.group + fr - t * p.group;
      const bool live = fr < q_at.req.qlen * p.group;
      const int64_t off = live ? (q_at.req.q0 + t) * p.q_token_stride + head * p.q_head_stride : -1;
      const int ch = lane % kLanes, first = (warp & 3) * 32 + lane / kLanes;
      unsigned char* dst = s_q + st * C::kTileBytes + (ch / 8) * C::kHalf + first * 128;
      const uint16_t* src = p.q + ch * 8;
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int64_t from = __shfl_sync(0xffffffffu, off, i * kRows + lane / kLanes);
        cp_async_16(dst + i * kRows * 128 + (((ch % 8) ^ ((first + i * kRows) & 7)) << 4),
                    from >= 0 ? src + from : p.q, from >= 0 ? 16u : 0u);
      }
      cp_async_wait_all();
      if (up.negate_q) {  // each lane over what it copied
#pragma unroll 1
        for (int i = 0; i < 32 / kRows; ++i) {
          uint4* v = reinterpret_cast<uint4*>(dst + i * kRows * 128 +
                                              (((ch % 8) ^ ((first + i * kRows) & 7)) << 4));
          *v = make_uint4(v->x ^ 0x80008000u, v->y ^ 0x80008000u, v->z ^ 0x80008000u, v->w ^ 0x80008000u);
        }
      }
      fence_async_shared();
      mbar_arrive(&c.q_ready[st]);
    };
    AttnSegment s = attn_segment<kTile, kBlk, kItem>(p, at, w0, w_end);
    StreamRange r = stream_range(p, at, s, st);
    if (r.end > r.begin) load_q(at);
    bool more = true;
    for (int w = w0; more;) {
      const int rows = at.req.qlen * p.group, cached = at.req.seq - at.req.qlen;
      const int fr = at.tile * kTile + st * kRowsPerStream + row;  // flattened row
      const bool live = fr < rows;
      const int t = p.by_group(fr), head = at.head * p.group + fr - t * p.group;
      float m = -INFINITY, l = 0.f;
      if (r.active) {
        // keys (j > low, j <= high) of this row, and those that all of the warp's rows see
        const int high = live ? cached + t : -1;
        const int low = attn_hidden(p, cached + t);
        const int f_row = at.tile * kTile + st * kRowsPerStream + (row & ~31);
        const int high_min = cached + p.by_group(f_row);
        const int low_max = attn_hidden(p, cached + p.by_group(min(f_row + 32, rows) - 1));
        for (int blk = r.begin; blk < r.end; ++blk) {
          mbar_wait_bounded(&c.s_full[st], s_phase, p.err, abort_flag);
          s_phase ^= 1u;
          tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_s + i * 32, x[i]);
          tmem_ld_wait();
          if constexpr (C::kOwnP) {
            tc_fence_before();
            mbar_arrive(&c.s_read[st]);
          }
          const int j0 = blk * kBlk;
          // 32 keys at a time, so that a block on the diagonal is not all compared (8 prompts of 1024
          // tokens, 64 heads on 4: 248 -> 232 us; a window of 512 keys, 4 requests of 2000 new tokens over
          // 2000, 32 heads on 4 of 128: 151 -> 140 us, floor 39)
          if (j0 + kBlk - 1 > high_min || j0 <= low_max) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int first = j0 + i * 32;
              if (first + 31 > high_min) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (e > high - first) x[i][e] = 0xff800000u;
              }
              if (first <= low_max) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (e <= low - first) x[i][e] = 0xff800000u;
              }
            }
          }
          float top[4];  // four chains: one would be 128 dependent steps
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            top[i] = fmaxf(__uint_as_float(x[i][0]), __uint_as_float(x[i][1]));
#pragma unroll
            for (int e = 2; e < 32; e += 2)
              top[i] = max3(top[i], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
          }
          const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
          const bool move = mx > m + kRescaleAbove || (m == -INFINITY && mx > m);
          if constexpr (C::kOwnP) {
            if (blk > r.begin) {  // P V of the last block: O is whole, P may be written again
              mbar_wait_bounded(&c.o_full[st], o_phase, p.err, abort_flag);
              o_phase ^= 1u;
              tc_fence_after();
            }
          }
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
          const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(base, base);
          uint64_t sum2 = pair(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float a, b;
              unpair(fma2(pair(__uint_as_float(x[i][2 * e]), __uint_as_float(x[i][2 * e + 1])), scale2, base2), a, b);
              a = ex2(a);
              b = ex2(b);
              sum2 = add2(sum2, pair(a, b));
              packed[e] = pack_bf16x2(a, b);
            }
            tmem_st_32x32b_x16(t_s + C::kColP + i * 16, packed);
            if (i == 1) {  // P V may begin with the first half of the keys
              tmem_st_wait();
              tc_fence_before();
              mbar_arrive(&c.p_half[st]);
            }
          }
          float sum0, sum1;
          unpair(sum2, sum0, sum1);
          l += sum0 + sum1;
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&c.p_ready[st]);
        }
      }
      // The next segment's Q goes in before this one's results come out: S of this segment's last
      // block is there, so its Q has been read.
      const AttnCursor done = at;
      const AttnSegment ds = s;
      const StreamRange dr = r;
      w += s.units;
      more = w < w_end;
      if (more) {
        attn_advance<kTile>(p, at);
        more = attn_has<kItem>(at, w, w_end);
      }
      if (more) {
        s = attn_segment<kTile, kBlk, kItem>(p, at, w, w_end);
        r = stream_range(p, at, s, st);
        if (r.end > r.begin) load_q(at);
      }
      if (!dr.active) continue;
      const bool has_o = dr.end > dr.begin;
      if (has_o) {
        mbar_wait_bounded(&c.o_full[st], o_phase, p.err, abort_flag);
        o_phase ^= 1u;
        tc_fence_after();
      }
      bool final = ds.whole;
      float total = l, scale = 1.f;
      float o[D];
#pragma unroll
      for (int i = 0; i < D; ++i) o[i] = 0.f;
      auto read_o = [&]() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_o + i * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[i * 32 + e] = __uint_as_float(v[e]);
        }
      };
      if (has_o) read_o();
      if (!ds.whole) {
        int cs, ce;
        attn_holders<kItem>(ds, per, cs, ce);
        const int me = blockIdx.x;
        // partial results lie as [D / 4][256 rows][4]: a warp's 16-byte pieces are neighbours
        auto slot_of = [&](int k) { return 2 * static_cast<int64_t>(k) + (k == cs ? 1 : 0); };
        auto o_of = [&](int k) {
          return reinterpret_cast<float4*>(p.partial_o + slot_of(k) * (kTile * D)) + st * kRowsPerStream + row;
        };
        auto ml_of = [&](int k) {
          return reinterpret_cast<float2*>(p.partial_ml) + slot_of(k) * kTile + st * kRowsPerStream + row;
        };
        if (has_o && live) {
          float4* po = o_of(me);
#pragma unroll
          for (int i = 0; i < D / 4; ++i)
            po[i * kTile] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        *ml_of(me) = make_float2(m, l);  // a sum of 0: nothing seen, and perhaps no accumulator written
        stream_sync(st);
        if (row == 0) c.last[st] = attn_arrive(p.counters + 2 * cs + st, ce - cs + 1);
        stream_sync(st);
        final = c.last[st] != 0;
        if (final && live) {
          // partials of CTAs cs .. ce, in the order of the keys whoever arrives last
          m = -INFINITY;
#pragma unroll 4
          for (int k = cs; k <= ce; ++k) {
            const float2 ml = __ldcg(ml_of(k));
            if (ml.y != 0.f) m = fmaxf(m, ml.x);
          }
          total = 0.f;
#pragma unroll
          for (int i = 0; i < D; ++i) o[i] = 0.f;
          for (int k = cs; k <= ce; ++k) {
            const float2 ml = __ldcg(ml_of(k));
            if (ml.y == 0.f) continue;
            const float f = ex2(ml.x - m);
            total += f * ml.y;
            const float4* po = o_of(k);
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
              const float4 v = __ldcg(po + i * kTile);
              o[4 * i] += f * v.x;
              o[4 * i + 1] += f * v.y;
              o[4 * i + 2] += f * v.z;
              o[4 * i + 3] += f * v.w;
            }
          }
        }
      }
      if (final && live) {
        uint16_t* dst = p.out + (done.req.q0 + t) * p.out_token_stride + head * p.out_head_stride;
        scale = total != 0.f ? 1.f / total : 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          uint32_t q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            q[e] = total != 0.f ? pack_bf16x2(o[8 * i + 2 * e] * scale, o[8 * i + 2 * e + 1] * scale) : 0u;
          *reinterpret_cast<uint4*>(dst + i * 8) = make_uint4(q[0], q[1], q[2], q[3]);
        }
        if (p.lse != nullptr)
          p.lse[static_cast<int64_t>(done.req.q0 + t) * p.q_heads + head] =
              total != 0.f ? (m + log2f(total)) * 0.693147180559945309f : -INFINITY;
      }
      tc_fence_before();  // O is read before the next segment's P V overwrites it
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
  static std::atomic<bool> done[64];  // two threads may both set the attribute, to the same value
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: device index >= 64");
  if (!done[dev].load(std::memory_order_acquire)) {
    // setmaxnreg hands out the registers that the CTA was launched with, and waits for ones that it
    // does not have
    cudaFuncAttributes attr;
    int rc = check_cuda(cudaFuncGetAttributes(&attr, paged_attn_umma_kernel<D>), "lm_paged_attention: attributes");
    if (!rc && attr.numRegs * kThreads < kSoftmaxRegs * 256 + kOtherRegs * 128)
      rc = fail(LM_ERR_UNSUPPORTED, "lm_paged_attention: built with too few registers for its register split");
    if (!rc)
      rc = check_cuda(cudaFuncSetAttribute(paged_attn_umma_kernel<D>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, UmmaCfg<D>::kSmem),
                      "lm_paged_attention: smem attribute");
    if (rc) return rc;
    done[dev].store(true, std::memory_order_release);
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
  p.beside = 0;
  // Q's sign takes a negative scale's, so that a row's largest S has its largest weight; with a
  // scale of 0 the masked scores (-inf) still have to vanish.
  p.negate_q = a.scale_log2 < 0.f;
  if (p.negate_q) p.a.scale_log2 = -a.scale_log2;
  if (a.scale_log2 == 0.f) p.a.scale_log2 = 1e-30f;
  return head_dim == 64 ? launch<64>(p, ctas, s) : launch<128>(p, ctas, s);
}

}  // namespace lm
