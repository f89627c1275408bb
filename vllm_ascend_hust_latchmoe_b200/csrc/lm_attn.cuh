// What the two attention kernels over the paged cache share: their parameters, the split of the
// work over the CTAs, and the merge of partial results.
//
// Rows: a request's queries of one kv head are flattened to (token, query head of the group)
// rows, so a row tile fills up whatever the number of query heads per kv head. An item is
// (request, kv head, row tile); its cost is ITEM units, for what it takes whatever its length, and
// one for each kv block that its rows see. All items' units are laid end to end and every CTA takes
// the same number of them, wherever that cuts an item ("per" units each): the load is even whatever
// the requests' lengths, and one long sequence spreads over the whole GPU. A boundary among an
// item's ITEM first units leaves all of the item to the CTA behind it. A CTA leaves at most two
// partial results: one of the item that it continues and one of the item that it starts and does
// not finish.
#pragma once

#include <cuda.h>

#include "lm_common.cuh"

namespace lm {

constexpr int kAttnMaxRequests = 4096;
constexpr int kAttnMaxCtas = 512;      // counters in the workspace
constexpr int kAttnMaxPartialRows = 256;
constexpr int kAttnMaxUnits = 0x7fff0000;  // of a launch; the rest of 32 bits is for a CTA's share past them

// Sum of two counts of units, at most kAttnMaxUnits. One request's units fit (the host has seen to it), and
// those of query ranges that follow each other do as well, but ranges on the device may overlap.
__device__ __forceinline__ int attn_add(int a, int b) {
  return static_cast<int>(min(static_cast<uint32_t>(a) + static_cast<uint32_t>(b),
                              static_cast<uint32_t>(kAttnMaxUnits)));
}

// n / d for 0 <= n < 2^31 as a product and a shift: mul = ceil(2^shift / d) with shift = 31 +
// ceil(log2 d) is above 2^shift / d by less than 2^(shift - 31) / d, which n is too small to show.
// (Divisions by numbers that come as arguments took 15 % of an item of one block.)
struct AttnDiv {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};

inline AttnDiv attn_div(int d) {
  AttnDiv r{0, 31};
  while ((int64_t{1} << (r.shift - 31)) < d) ++r.shift;
  r.mul = static_cast<uint32_t>(((uint64_t{1} << r.shift) + d - 1) / d);
  return r;
}

struct AttnParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* lse;  // [T, Hq] or null
  const int32_t* tables;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  int32_t* counters;   // [2 * kAttnMaxCtas], zero between launches
  float* partial_o;    // [2 * ctas][rows * D]
  float* partial_ml;   // [2 * ctas][rows][2]: running maximum (log2 domain) and sum
  int32_t* err;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int64_t k_page_stride, k_token_stride, k_head_stride;
  int64_t v_page_stride, v_token_stride, v_head_stride;
  int64_t table_stride;
  int64_t num_tokens;
  int num_requests, q_heads, kv_heads, group, page_size, num_pages, max_pages, window;
  AttnDiv by_group, by_page;
  int min_rows, max_rows;  // requests with this many rows per kv head are this launch's
  float scale_log2;        // softmax scale * log2(e)
};

struct AttnRequest {
  int q0, qlen, seq;
};

// The request's query range and length, held inside their buffers.
__device__ __forceinline__ AttnRequest attn_request(const AttnParams& p, int b, bool report) {
  AttnRequest r;
  r.q0 = p.cu_q[b];
  const int q1 = p.cu_q[b + 1];
  r.qlen = q1 - r.q0;
  r.seq = p.seq_lens[b];
  if (r.q0 < 0 || q1 < r.q0 || q1 > p.num_tokens) {
    if (report) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    r.q0 = r.qlen = 0;
  }
  const int64_t limit = static_cast<int64_t>(p.max_pages) * p.page_size;
  if (r.seq < 0 || r.seq > limit) {
    if (report) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    r.seq = r.seq < 0 ? 0 : static_cast<int>(limit);
  }
  return r;
}

// The last key that a window hides from a row at position `pos`, -1 for none. (Rows before every key have
// negative positions, see nothing and may name any key here; a window of up to 2^31 - 1 must not wrap.)
__device__ __forceinline__ int attn_hidden(const AttnParams& p, int pos) {
  return p.window > 0 ? max(pos, 0) - p.window : -1;
}

// Keys that some row of tile `tile` sees: [lo, hi).
template <int TILE_ROWS>
__device__ __forceinline__ void attn_tile_keys(const AttnParams& p, const AttnRequest& r, int tile,
                                               int& lo, int& hi) {
  const int rows = r.qlen * p.group;
  const int first = p.by_group(tile * TILE_ROWS);
  const int last = p.by_group(min((tile + 1) * TILE_ROWS, rows) - 1);
  const int cached = r.seq - r.qlen;  // negative: the first queries stand before every key
  hi = max(0, cached + last + 1);
  lo = min(hi, max(0, attn_hidden(p, cached + first) + 1));
}

template <int BLOCK>
__device__ __forceinline__ int attn_blocks(int lo, int hi) {
  // an item without keys still costs a unit: its rows have to be written
  return hi > lo ? (hi + BLOCK - 1) / BLOCK - lo / BLOCK : 1;
}

// Row tiles per kv head that this launch makes of a request.
template <int TILE_ROWS>
__device__ __forceinline__ int attn_tiles(const AttnParams& p, const AttnRequest& r) {
  const int rows = r.qlen * p.group;
  return rows >= p.min_rows && rows <= p.max_rows ? (rows + TILE_ROWS - 1) / TILE_ROWS : 0;
}

// Units of a lane's request per kv head, and the most blocks of its items; the lanes of the warp
// share the tiles of a request that has several. All lanes call it (tiles 0: no request).
template <int TILE_ROWS, int BLOCK, int ITEM>
__device__ __forceinline__ int attn_cost(const AttnParams& p, const AttnRequest& r, int tiles, int& longest) {
  int cost = 0;
  if (tiles == 1) {
    int lo, hi;
    attn_tile_keys<TILE_ROWS>(p, r, 0, lo, hi);
    cost = attn_blocks<BLOCK>(lo, hi);
    longest = max(longest, cost);
    cost += ITEM;
  }
  for (unsigned many = __ballot_sync(0xffffffffu, tiles > 1); many != 0; many &= many - 1) {
    const int src = __ffs(many) - 1;
    AttnRequest o;
    o.q0 = 0;
    o.qlen = __shfl_sync(0xffffffffu, r.qlen, src);
    o.seq = __shfl_sync(0xffffffffu, r.seq, src);
    const int n = __shfl_sync(0xffffffffu, tiles, src);
    int part = 0;
    for (int t = threadIdx.x & 31; t < n; t += 32) {
      int lo, hi;
      attn_tile_keys<TILE_ROWS>(p, o, t, lo, hi);
      const int n_blocks = attn_blocks<BLOCK>(lo, hi);
      part += n_blocks + ITEM;
      longest = max(longest, n_blocks);
    }
    part = __reduce_add_sync(0xffffffffu, part);
    if ((threadIdx.x & 31) == src) cost = part;
  }
  return cost;
}

// Exclusive prefix of the requests' costs in s_prefix[0 .. B], and the longest item's blocks (into
// *s_longest, zeroed by the caller ahead of a barrier). Called by all NT threads, a request each.
template <int TILE_ROWS, int BLOCK, int ITEM, int NT>
__device__ __forceinline__ void attn_prefix(const AttnParams& p, int32_t* s_prefix, int32_t* s_warp,
                                            int* s_longest) {
  const int B = p.num_requests;
  const int per = (B + NT - 1) / NT;
  const int b0 = threadIdx.x * per, b1 = min(B, b0 + per);
  int sum = 0, longest = 0;
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    AttnRequest r{0, 0, 0};
    int tiles = 0;
    if (b < b1) {
      r = attn_request(p, b, blockIdx.x == 0);
      tiles = attn_tiles<TILE_ROWS>(p, r);
    }
    const int cost = attn_cost<TILE_ROWS, BLOCK, ITEM>(p, r, tiles, longest);
    if (b < b1) s_prefix[b + 1] = cost * p.kv_heads;
    sum = attn_add(sum, cost * p.kv_heads);
  }
  int incl = sum;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl = attn_add(incl, u);
  }
  if (lane == 31) s_warp[warp] = incl;
  atomicMax(s_longest, longest);
  __syncthreads();
  int base = incl - sum;
  for (int w = 0; w < warp; ++w) base = attn_add(base, s_warp[w]);
  for (int b = b0; b < b1; ++b) {
    base = attn_add(base, s_prefix[b + 1]);
    s_prefix[b + 1] = base;
  }
  if (threadIdx.x == 0) s_prefix[0] = 0;
  __syncthreads();
}

// Where a CTA stands in the launch's units: item (b, head, tile), `off` of its units already passed.
struct AttnCursor {
  AttnRequest req;
  int b, head, tile, tiles, off;
};

// Whether some of the cursor's blocks lie before w_end (a boundary ahead of an item's first block
// leaves the item to the next CTA).
template <int ITEM>
__device__ __forceinline__ bool attn_has(const AttnCursor& c, int w, int w_end) {
  return w_end - w + c.off > ITEM;
}

// Sets the head and tile of a cursor whose `off` counts from its request's first unit; every warp
// computes it alike.
template <int TILE_ROWS, int BLOCK, int ITEM>
__device__ __forceinline__ void attn_enter(const AttnParams& p, AttnCursor& c, int request_units) {
  const int per_head = request_units / p.kv_heads;
  c.head = c.off / per_head;
  c.off -= c.head * per_head;
  // the tile that unit `off` of the head falls into: a lane per tile, 32 tiles at a time
  for (c.tile = 0; c.tiles > 1;) {
    const int lane = threadIdx.x & 31, t = c.tile + lane;
    int lo, hi, n = 0;
    if (t < c.tiles) {
      attn_tile_keys<TILE_ROWS>(p, c.req, t, lo, hi);
      n = attn_blocks<BLOCK>(lo, hi) + ITEM;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, t < c.tiles && incl > c.off);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      c.off -= __shfl_sync(0xffffffffu, incl - n, at);
      c.tile += at;
      break;
    }
    c.off -= __shfl_sync(0xffffffffu, incl, 31);
    c.tile += 32;
  }
}

// This CTA's units [w, w_end) of the launch's `total`, `per` to a CTA, and the cursor at w; false where
// it has none. FEW: items longer than 8 blocks are cut into sqrt(n) pieces at most. Up to 32 requests
// every warp works it out for itself, a request a lane; more go through shared memory (0.2 to 0.7 us
// more: 16 single tokens over 1000 keys 16.4 against 15.8 us).
template <int TILE_ROWS, int BLOCK, int ITEM, int NT, bool FEW>
__device__ __forceinline__ bool attn_locate(const AttnParams& p, int32_t* s_prefix, int32_t* s_warp,
                                            int* s_longest, int& per, int& w, int& w_end, AttnCursor& c) {
  const int B = p.num_requests, lane = threadIdx.x & 31;
  int total, longest = 0, incl = 0, units = 0, tiles = 0;
  AttnRequest r{0, 0, 0};
  if (B <= 32) {
    if (lane < B) {
      r = attn_request(p, lane, blockIdx.x == 0 && threadIdx.x < 32);
      tiles = attn_tiles<TILE_ROWS>(p, r);
    }
    units = attn_cost<TILE_ROWS, BLOCK, ITEM>(p, r, tiles, longest) * p.kv_heads;
    longest = __reduce_max_sync(0xffffffffu, longest);
    incl = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = attn_add(incl, u);
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
  } else {
    attn_prefix<TILE_ROWS, BLOCK, ITEM, NT>(p, s_prefix, s_warp, s_longest);
    total = s_prefix[B];
    longest = *s_longest;
  }
  if (total == kAttnMaxUnits) {  // more than can be told apart: nothing is computed
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    return false;
  }
  const int fewest = FEW && longest > 8 ? static_cast<int>(sqrtf(static_cast<float>(longest))) : 1;
  per = max(fewest, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  w = blockIdx.x * per;
  w_end = min(total, w + per);
  if (w >= w_end) return false;
  if (B <= 32) {
    c.b = __ffs(__ballot_sync(0xffffffffu, incl > w)) - 1;  // the first request that ends past w
    c.req.q0 = __shfl_sync(0xffffffffu, r.q0, c.b);
    c.req.qlen = __shfl_sync(0xffffffffu, r.qlen, c.b);
    c.req.seq = __shfl_sync(0xffffffffu, r.seq, c.b);
    c.tiles = __shfl_sync(0xffffffffu, tiles, c.b);
    units = __shfl_sync(0xffffffffu, units, c.b);
    c.off = w - (__shfl_sync(0xffffffffu, incl, c.b) - units);
  } else {
    int lo_b = 0, hi_b = B;
    while (hi_b - lo_b > 1) {  // the last request that starts at or before w; costless ones end there
      const int mid = (lo_b + hi_b) >> 1;
      if (s_prefix[mid] <= w) lo_b = mid; else hi_b = mid;
    }
    c.b = lo_b;
    c.req = attn_request(p, lo_b, false);
    c.tiles = attn_tiles<TILE_ROWS>(p, c.req);
    c.off = w - s_prefix[lo_b];
    units = s_prefix[lo_b + 1] - s_prefix[lo_b];
  }
  attn_enter<TILE_ROWS, BLOCK, ITEM>(p, c, units);
  if (c.off <= ITEM) {  // the boundary falls ahead of the item's first block: it is this CTA's from there
    w -= c.off;
    c.off = 0;
  }
  return attn_has<ITEM>(c, w, w_end);
}

// To the next item; only called when there is one.
template <int TILE_ROWS>
__device__ __forceinline__ void attn_advance(const AttnParams& p, AttnCursor& c) {
  c.off = 0;
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.head < p.kv_heads) return;
  c.head = 0;
  do {
    ++c.b;
    c.req = attn_request(p, c.b, false);
    c.tiles = attn_tiles<TILE_ROWS>(p, c.req);
  } while (c.tiles == 0 && c.b + 1 < p.num_requests);
}

// A CTA's piece of the cursor's item: kv blocks [blk0, blk1) of those that hold keys [lo, hi).
struct AttnSegment {
  int lo, hi;      // keys of the whole tile
  int blk0, blk1;  // absolute kv block numbers of this segment
  int start, end;  // the item's units [start, end) in the launch's order
  int units;       // of this segment
  bool whole;
};

template <int TILE_ROWS, int BLOCK, int ITEM>
__device__ __forceinline__ AttnSegment attn_segment(const AttnParams& p, const AttnCursor& c, int w,
                                                    int w_end) {
  AttnSegment s;
  attn_tile_keys<TILE_ROWS>(p, c.req, c.tile, s.lo, s.hi);
  const int n = attn_blocks<BLOCK>(s.lo, s.hi);
  s.start = w - c.off;
  s.end = s.start + ITEM + n;
  s.units = min(s.end, w_end) - w;
  const int b0 = max(c.off - ITEM, 0), b1 = c.off + s.units - ITEM;
  s.whole = b0 == 0 && b1 == n;
  s.blk0 = s.lo / BLOCK + b0;
  s.blk1 = s.hi > s.lo ? s.lo / BLOCK + b1 : s.blk0;
  return s;
}

// The first and last CTA that hold blocks of a segment's item.
template <int ITEM>
__device__ __forceinline__ void attn_holders(const AttnSegment& s, int per, int& first, int& last) {
  first = (s.start + ITEM) / per;
  last = (s.end - 1) / per;
}

// 2^x. Weights below 2^-126 of a row's largest are flushed: they are far below its rounding (exp2f, which
// keeps them, cost 1 % of decode steps of few keys).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A bounded wait of a whole warp, with one answer for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int32_t* err,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, err, abort_flag));
}

// One thread says that its CTA (or stream) has stored its partial result, and whether it was the last
// of `pieces` to do so; the last one resets the counter. Between two barriers of the threads that
// store and merge: this thread's fences order their stores before the count, and the others' partial
// results before the merge.
__device__ __forceinline__ bool attn_arrive(int32_t* counter, int pieces) {
  __threadfence();
  const bool last = atomicAdd(counter, 1) == pieces - 1;
  if (last) *counter = 0;  // every other CTA of the item has arrived
  __threadfence();
  return last;
}

// The cache as TMA sees it: K and V by boxes of box_rows tokens (a divisor of the page size, at
// most a block) of one head x 64 values, 128-byte swizzled.
constexpr int kAttnBlock = 128;  // keys per block

struct AttnMaps {
  CUtensorMap k, v;
  int box_rows;
  int heads_first;  // dimensions (values, heads, tokens, pages), else (values, tokens, heads, pages)
};

struct AttnLaunch {
  AttnMaps maps;
  AttnParams a;
  int negate_q;
  int beside;  // the kernel launched just before is the other half of the same call
};

int attn_make_maps(const AttnParams& a, int head_dim, AttnMaps* maps);

__device__ __forceinline__ void tma_load_4d(void* dst, const void* desc, uint64_t* bar, int32_t x,
                                            int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(desc), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// A loader warp of either kernel: the segments' blocks of K or of V, in order, as tiles of 128 keys
// ([D / 64] halves of 128 rows x 128 bytes). Its n-th tile is number first + n * step of a ring
// with STAGES places, `stage_bytes` apart. Page ids are read a block ahead. Keys outside the
// segment's item come from boxes past the cache's end, which TMA fills with zeros; inside a box
// that is partly in range, the cache's own contents arrive. One warp for both would not do: with
// pages of 16 keys (boxes of 2 KB) a warp issues 34 GB/s.
template <int D, int TILE_ROWS, int ITEM, int STAGES>
__device__ __forceinline__ void attn_load_kv(const AttnLaunch& up, bool is_v, AttnCursor at, int w,
                                             int w_end, unsigned char* ring, int stage_bytes, int first,
                                             int step, uint64_t* full, uint64_t* empty,
                                             volatile int* abort_flag) {
  constexpr int kHalf = kAttnBlock * 128, kTileBytes = kHalf * (D / 64);
  const AttnParams& p = up.a;
  const int lane = threadIdx.x & 31;
  const int boxes = kAttnBlock / up.maps.box_rows;  // per 64 values
  const int n_loads = boxes * (D / 64);             // one lane each, at most 16
  const int box = lane % boxes, half = lane / boxes;
  const CUtensorMap* map = is_v ? &up.maps.v : &up.maps.k;
  int stage = first % STAGES, passes = 0, tiles = 0;
  bool ok = true;
  while (attn_has<ITEM>(at, w, w_end) && ok) {
    const AttnSegment s = attn_segment<TILE_ROWS, kAttnBlock, ITEM>(p, at, w, w_end);
    const int32_t* table = p.tables + at.b * p.table_stride;
    auto page_of = [&](int blk) {  // the page of this lane's box, num_pages where there is none
      const int tok = blk * kAttnBlock + box * up.maps.box_rows;
      if (lane >= n_loads || tok >= s.hi || tok + up.maps.box_rows <= s.lo) return p.num_pages;
      const int pg = table[p.by_page(tok)];
      if (pg < 0 || pg >= p.num_pages) {
        record_error(p.err, LM_DEVERR_BAD_PAGE);
        return p.num_pages;
      }
      return pg;
    };
    int page = s.blk0 < s.blk1 ? page_of(s.blk0) : 0;
    for (int blk = s.blk0; blk < s.blk1 && ok; ++blk) {
      const int page_next = blk + 1 < s.blk1 ? page_of(blk + 1) : 0;
      const int tok = blk * kAttnBlock + box * up.maps.box_rows;
      const int y = tok - p.by_page(tok) * p.page_size;
      ok = warp_wait(&empty[stage], (passes & 1u) ^ 1u, p.err, abort_flag);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], kTileBytes);
      __syncwarp();
      if (lane < n_loads)
        tma_load_4d(ring + stage * stage_bytes + half * kHalf + box * up.maps.box_rows * 128, map,
                    &full[stage], half * 64, up.maps.heads_first ? at.head : y,
                    up.maps.heads_first ? y : at.head, page);
      __syncwarp();
      ++tiles;
      stage += step;
      if (stage >= STAGES) {
        stage -= STAGES;
        ++passes;
      }
      page = page_next;
    }
    w += s.units;
    if (w >= w_end) break;
    attn_advance<TILE_ROWS>(p, at);
  }
  // Every stage used is released before the CTA may leave (no copy or commit is in flight then); of
  // two warps that fill the ring in turn, the one that ends last sees the last pass of each stage.
  const int total = tiles * step;
  for (int st = 0; st < STAGES && st < total; ++st) {
    const uint32_t par = static_cast<uint32_t>((total - 1 - st) / STAGES) & 1u;
    const long long t0 = clock64();
    while (!mbar_try_wait(&empty[st], par) && clock64() - t0 < LM_SPIN_LIMIT_CYCLES) {
      if (*abort_flag && clock64() - t0 > 200000) break;
    }
  }
}

// The tensor-core launch of lm_paged_attention (lm_attn_umma.cu).
int attn_launch_umma(const AttnParams& a, const AttnMaps& maps, int head_dim, int ctas, cudaStream_t s);

}  // namespace lm
