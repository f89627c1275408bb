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
constexpr size_t kTableStatic = 1024;  // at least page_tables_kernel's static shared memory (516 bytes)

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
  int wide;  // positions and slots take 16-byte stores
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

// Pages of `tokens` tokens; unsigned, as the sum may pass 2^31 where a page is about as long.
__device__ __forceinline__ int pages_of(int tokens, int page) {
  return static_cast<int>((static_cast<uint32_t>(tokens) + static_cast<uint32_t>(page) - 1u) /
                          static_cast<uint32_t>(page));
}

// The last of n ascending values that is at most x (values[0] is).
__device__ __forceinline__ int last_at_most(const int32_t* values, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (values[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Positions and slots of N neighbouring tokens a thread, from the requests' first tokens (s_cu), pages
// granted before them (s_page) and cached lengths (inverted: no place for the new tokens).
template <int N>
__device__ __forceinline__ void place_tokens(const TableParams& p, const int32_t* s_cu, const int32_t* s_page,
                                             const int32_t* s_cached, int free_count, int tid, int stride) {
  const int B = p.num_requests, page = p.page_size, total = s_cu[B];
  for (int64_t t0 = static_cast<int64_t>(tid) * N; t0 < p.max_tokens; t0 += static_cast<int64_t>(stride) * N) {
    int pos[N];
    long long slot[N];
    // the last request that starts at or before t0: the one that t0 belongs to
    int lo = t0 < total ? last_at_most(s_cu, B, t0) : 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t t = t0 + e;
      pos[e] = 0;
      slot[e] = -1;
      if (t >= total) continue;
      while (t >= s_cu[lo + 1]) ++lo;
      const int kept = s_cached[lo], c = kept < 0 ? ~kept : kept;
      pos[e] = c + static_cast<int>(t) - s_cu[lo];
      if (kept < 0) continue;
      const int have = pages_of(c, page);  // unsigned like the next line, which shares its divisor's set-up
      const int i = static_cast<int>(static_cast<uint32_t>(pos[e]) / static_cast<uint32_t>(page));
      // pages already held are read from the table, granted ones from the stack (another CTA may be
      // writing their table entries)
      const int id = i < have ? p.tables[lo * p.table_stride + i]
                              : p.free_pages[free_count - 1 - (s_page[lo] + i - have)];
      if (id >= 0)
        slot[e] = static_cast<long long>(id) * page + (pos[e] - i * page);
      else
        record_error(p.err, LM_DEVERR_BAD_PAGE);
    }
    if (N == 4 && p.wide && t0 + N <= p.max_tokens) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1 % N], pos[2 % N], pos[3 % N]);
      reinterpret_cast<longlong2*>(p.slots + t0)[0] = make_longlong2(slot[0], slot[1 % N]);
      reinterpret_cast<longlong2*>(p.slots + t0)[1] = make_longlong2(slot[2 % N], slot[3 % N]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (t0 + e >= p.max_tokens) break;
        p.positions[t0 + e] = pos[e];
        p.slots[t0 + e] = slot[e];
      }
    }
  }
}

// Every CTA scans all requests (they fit one pass of its threads) and writes its share of the
// tables and of the tokens. All reads of arrays that the call may overwrite in place (cached
// lengths, the free count) come before the cluster's barrier, all writes to them after it.
// Latency-bound: 4.2 us a call for 64 requests with a token each, 8.8 us for 1021 requests with 30,000
// tokens (replayed from a graph; 20.6 us when a request's pages were one warp's).
__global__ void __launch_bounds__(kTableThreads) page_tables_kernel(const TableParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int32_t s_mem[];
  __shared__ int64_t s_warp[32][2];
  __shared__ int s_used;
  if (threadIdx.x == 0) s_used = 0;
  const int B = p.num_requests, page = p.page_size;
  int32_t* s_cu = s_mem;               // [B + 1] first token of each request
  int32_t* s_page = s_cu + B + 1;      // [B] pages needed before it
  int32_t* s_cached = s_page + B;      // [B] cached length; inverted where the request gets no place
  const int per = (B + kTableThreads - 1) / kTableThreads;
  int free_count = *p.free_count;
  if (free_count < 0 || free_count > p.free_capacity) {
    if (threadIdx.x == 0) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    free_count = min(max(free_count, 0), p.free_capacity);
  }
  const int64_t limit = static_cast<int64_t>(p.max_pages) * page;
  // pages that n tokens behind c cached ones need, or why they get none
  constexpr int kBadLength = -1, kNoRoom = -2;
  auto pages_for = [&](int c, int n) {
    return static_cast<int64_t>(c) + n > limit ? kNoRoom : pages_of(c + n, page) - pages_of(c, page);
  };
  int need[kPerThread], fresh[kPerThread], cached[kPerThread];
  int64_t sum_need = 0, sum_fresh = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * per + i;
    need[i] = fresh[i] = cached[i] = 0;
    if (i >= per || b >= B) continue;
    cached[i] = p.cached[b];
    fresh[i] = p.fresh[b];
    bool bad = false;
    if (cached[i] < 0 || cached[i] > limit) {
      bad = true;
      cached[i] = 0;
    }
    if (fresh[i] < 0 || fresh[i] > p.max_tokens) {
      bad = true;
      fresh[i] = 0;
    }
    if (bad) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    need[i] = bad ? kBadLength : pages_for(cached[i], fresh[i]);
    sum_need += max(need[i], 0);
    sum_fresh += fresh[i];
  }
  int64_t at_need = sum_need, at_fresh = sum_fresh, total_need, total_fresh;
  block_scan2(at_need, at_fresh, total_need, total_fresh, s_warp);
  if (total_fresh > p.max_tokens) {  // the tokens are cut, and pages are for those that are left
    if (threadIdx.x == 0) record_error(p.err, LM_DEVERR_BAD_LENGTH);
    int64_t first = at_fresh;
    sum_need = sum_fresh = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int left = static_cast<int>(max(p.max_tokens - first, int64_t{0}));
      first += fresh[i];
      fresh[i] = min(fresh[i], left);
      if (need[i] != kBadLength) need[i] = pages_for(cached[i], fresh[i]);
      sum_need += max(need[i], 0);
      sum_fresh += fresh[i];
    }
    at_need = sum_need;
    at_fresh = sum_fresh;
    __syncthreads();  // s_warp has been read
    block_scan2(at_need, at_fresh, total_need, total_fresh, s_warp);
  }
  int granted = 0;  // pages up to and including this thread's last request that got its pages
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * per + i;
    if (i >= per || b >= B) continue;
    s_cu[b] = static_cast<int32_t>(at_fresh);
    bool ok = need[i] >= 0;
    if (need[i] == kNoRoom || (need[i] > 0 && at_need + need[i] > free_count)) {
      record_error(p.err, LM_DEVERR_NO_PAGES);
      ok = false;
    }
    s_page[b] = static_cast<int32_t>(min(at_need, static_cast<int64_t>(0x7fffffff)));
    s_cached[b] = ok ? cached[i] : ~cached[i];
    if (ok && need[i] > 0) granted = static_cast<int>(at_need) + need[i];
    at_need += max(need[i], 0);
    at_fresh += fresh[i];
  }
  if (threadIdx.x == 0) s_cu[B] = static_cast<int32_t>(total_fresh);
  // The largest grant ends the pages taken: requests are granted in order, and once one does not
  // fit, every later one that needs a page does not either.
  if (granted > 0) atomicMax(&s_used, granted);
  __syncthreads();
  // this CTA has read what the call may overwrite; the wait comes right before that is written
  if (gridDim.x > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  const int tid = blockIdx.x * kTableThreads + threadIdx.x;
  const int stride = gridDim.x * kTableThreads;
  // new table entries: a thread per granted page
  for (int j = tid; j < s_used; j += stride) {
    const int b = last_at_most(s_page, B, j);
    const int have = pages_of(s_cached[b], page);
    p.tables[b * p.table_stride + have + j - s_page[b]] = p.free_pages[free_count - 1 - j];
  }
  // tokens: one a thread while that is enough, else 4 neighbours, with one search and their reads
  // in flight together
  if (p.max_tokens <= stride)
    place_tokens<1>(p, s_cu, s_page, s_cached, free_count, tid, stride);
  else
    place_tokens<4>(p, s_cu, s_page, s_cached, free_count, tid, stride);
  __syncwarp();
  if (gridDim.x > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (tid == 0) *p.free_count_out = free_count - s_used;
  for (int b = tid; b <= B; b += stride) {
    p.cu_q[b] = s_cu[b];
    if (b == B) break;
    const int kept = s_cached[b];
    p.seq_lens[b] = kept < 0 ? ~kept : kept + s_cu[b + 1] - s_cu[b];
  }
}

// One block: the pages of the listed rows go back onto the free stack in row order. Entries below 0 hold
// no page (it was given back before, as behind a sliding window) and are passed over; where a row's
// entries are more than the stack has room for, its pages are counted first, so that a row whose pages do
// not fit stays as it is. The rows follow one another, each a chain of dependent reads: 6 to 7 us a call
// for one row of 80 pages, 14 us for 16 such rows, 320 to 335 us for 512 (265 to 279 us when entries were
// pushed unchecked).
constexpr int kReleaseThreads = 256;

__global__ void __launch_bounds__(kReleaseThreads)
    release_pages_kernel(const int32_t* __restrict__ rows, int num_rows, int32_t* cached,
                         int num_requests, int page_size, int32_t* tables, int64_t table_stride,
                         int max_pages, int32_t* free_pages, int free_capacity,
                         int32_t* free_count, int32_t* err) {
  pdl_wait();
  pdl_trigger();
  __shared__ int s_held[kReleaseThreads / 32];  // pages of each warp's entries
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    const int n = pages_of(cached[b], page_size);
    int32_t* row = tables + b * table_stride;
    if (n > free_capacity - count) {
      int pages = 0;
      for (int j0 = 0; j0 < n; j0 += kReleaseThreads) {
        const int j = j0 + static_cast<int>(threadIdx.x);
        pages += __syncthreads_count(j < n && row[j] >= 0);
      }
      if (pages > free_capacity - count) {
        if (threadIdx.x == 0) record_error(err, LM_DEVERR_BAD_LENGTH);
        continue;
      }
    }
    for (int j0 = 0; j0 < n; j0 += kReleaseThreads) {
      const int j = j0 + static_cast<int>(threadIdx.x);
      const int id = j < n ? row[j] : -1;
      int at = count + static_cast<int>(threadIdx.x), pages = min(n - j0, kReleaseThreads);
      // the barrier also has every thread's read of cached[b] behind it
      if (!__syncthreads_and(j >= n || id >= 0)) {
        const unsigned held = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) s_held[warp] = __popc(held);
        __syncthreads();
        at = count + __popc(held & ((1u << lane) - 1u));
        pages = 0;
        for (int w = 0; w < kReleaseThreads / 32; ++w) {
          if (w < warp) at += s_held[w];
          pages += s_held[w];
        }
      }
      count += pages;
      if (id >= 0) free_pages[at] = id;
      if (j < n) row[j] = -1;
    }
    if (n > 0 && threadIdx.x == 0) cached[b] = 0;
    __syncthreads();  // a row listed twice is empty then
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

// Where the head h of token t goes: its row of q_out or of the cache, null for nowhere.
__device__ __forceinline__ uint16_t* rope_target(const RopeParams& p, int64_t t, int h, int64_t slot,
                                                 int64_t page, int64_t off) {
  if (h < p.q_heads) return p.q_out + t * p.q_token_stride + h * p.q_head_stride;
  if (slot < 0) return nullptr;
  h -= p.q_heads;
  if (h < p.kv_heads)
    return p.k_cache + page * p.k_page_stride + off * p.k_token_stride + h * p.k_head_stride;
  return p.v_cache + page * p.v_page_stride + off * p.v_token_stride +
         (h - p.kv_heads) * p.v_head_stride;
}

// The token's slot, -1 where nothing is stored.
__device__ __forceinline__ int64_t rope_slot(const RopeParams& p, int64_t slot) {
  if (slot < p.num_slots) return slot;
  record_error(p.err, LM_DEVERR_BAD_PAGE);
  return -1;
}

__device__ __forceinline__ int rope_position(const RopeParams& p, int pos) {
  if (pos >= 0 && pos < p.max_pos) return pos;
  record_error(p.err, LM_DEVERR_BAD_POSITION);
  return 0;
}

// A warp takes up to kRopeUnroll x (32 / (D / 8)) heads of one kind (q, k or v) of one token, 8
// values of a head per lane, so that the token's rotation and the norm's weight are read and
// multiplied once (out = r * (z * (w cos) + z' * (w' sin)) for a value z and its partner z') and all
// heads' loads are in flight together. A lane's partners are its own neighbours (interleaved) or
// the 8 values of the lane half / 8 away, which come by shuffle as the bf16 pairs they are. Needs
// 8 | rot_dim, and 16 | rot_dim for pairs half a rotation apart. Measured at 4096 tokens x 40 heads
// of 128 with norms: 18.2 to 18.6 us (4.6 TB/s, 72 % of the copy rate). Neither limit is reached: issue
// slots are 67 % busy (a version with 213 instructions per 32 lanes took 26.6 us, one with 156 21.5 us)
// and DRAM moves 2.5 TB/s, since most writes stay in L2. The blocks are uneven: 1536 of them at 4 an SM
// make 2.6 waves, and one of queries does eight times the work of one of K or V.
// With one group of heads a warp, 2 or 8 heads in flight per lane measured 24.7 and 21.7 us in the
// place of 21.5, more registers or more blocks per SM 23.7 and 26.7 us; the next group's loads ahead of
// this one's arithmetic spill (20.6 us). 16 tokens take 3.2 us.
constexpr int kRopeUnroll = 4;

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  unpack_bf16x2(v.x, f[0], f[1]);
  unpack_bf16x2(v.y, f[2], f[3]);
  unpack_bf16x2(v.z, f[4], f[5]);
  unpack_bf16x2(v.w, f[6], f[7]);
}

template <int D>
__host__ __device__ constexpr int rope_heads_per_warp() {
  return kRopeUnroll * 32 / (D / 8);
}

// Q chunks that a warp takes one after the other, with the rotation and weight in registers. Many
// tokens fill the GPU anyway; few tokens wait for one warp's chain. With 4 against 1, in us:
//   tokens                  64          1024          1536          2048          3000          4096
//   64/4 heads of 128   6.8, 3.2     13.5, 11.4   15.5, 15.5   16.9, 19.5   25.1, 26.8   30.0, 35.0
//   32/4 heads of 128   6.8, 3.2     10.2, 7.2    13.0, 9.9    13.6, 12.9   15.9, 17.0   18.6, 21.6
//   16/2 heads of 128   4.7, 3.2      5.7, 4.7     6.4, 5.2     7.9, 7.0    10.3, 10.8   12.9, 13.9
//   32/8 heads of 64    4.2, 3.1      5.7, 4.7     6.7, 5.7     8.6, 8.3    10.5, 11.3   13.4, 14.4
// They cross between 1536 and 3000 tokens, the earlier the more query heads there are.
constexpr int kRopeLoops = 4;
constexpr int64_t kRopeManyTokens = 2048;

template <int D, int LOOPS>
__global__ void __launch_bounds__(kRopeWarps * 32, 4) rope_write_kernel(const RopeParams p) {
  constexpr int LANES = D / 8, HEADS = 32 / LANES, PER_WARP = rope_heads_per_warp<D>();
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRopeWarps + (threadIdx.x >> 5);
  const int q_chunks = (p.q_heads + PER_WARP * LOOPS - 1) / (PER_WARP * LOOPS);
  const int k_chunks = (p.kv_heads + PER_WARP - 1) / PER_WARP;
  pdl_wait();
  pdl_trigger();
  if (t >= p.num_tokens) return;
  int chunk = blockIdx.y;
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;
  chunk -= kind == 0 ? 0 : kind == 1 ? q_chunks : q_chunks + k_chunks;
  const int heads = kind == 0 ? p.q_heads : p.kv_heads;  // of this kind
  const int first_head = kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.kv_heads;
  if (kind == 0) chunk *= LOOPS;
  int h0 = chunk * PER_WARP + lane / LANES;
  const int c0 = (lane % LANES) * 8;  // this lane's values of a head

  // the position first: the cosines' addresses wait for it while the heads arrive
  const int position = p.positions[t];
  const int64_t target = p.slots[t];
  uint4 raw[kRopeUnroll];
  const uint16_t* src = p.qkv + t * p.qkv_stride + (first_head + h0) * D + c0;
#pragma unroll
  for (int u = 0; u < kRopeUnroll; ++u) {
    raw[u] = make_uint4(0, 0, 0, 0);
    if (h0 + u * HEADS < heads) raw[u] = *reinterpret_cast<const uint4*>(src + u * HEADS * D);
  }

  uint16_t* dst = nullptr;
  int64_t head_stride = p.q_head_stride;
  if (kind == 0) {
    dst = p.q_out + t * p.q_token_stride;
  } else {
    const int64_t slot = rope_slot(p, target);
    if (slot < 0) return;  // the whole warp
    int64_t page, off;
    if (p.num_slots <= 0x7fffffff) {  // a 32-bit division is a fifth of a 64-bit one
      const uint32_t s = static_cast<uint32_t>(slot), n = static_cast<uint32_t>(p.page_size);
      page = s / n;
      off = s % n;
    } else {
      page = slot / p.page_size;
      off = slot % p.page_size;
    }
    dst = kind == 1 ? p.k_cache + page * p.k_page_stride + off * p.k_token_stride
                    : p.v_cache + page * p.v_page_stride + off * p.v_token_stride;
    head_stride = kind == 1 ? p.k_head_stride : p.v_head_stride;
  }
  dst += h0 * head_stride + c0;
  head_stride *= HEADS;

  if (kind == 2) {
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u)
      if (h0 + u * HEADS < heads) *reinterpret_cast<uint4*>(dst + u * head_stride) = raw[u];
    return;
  }
  const uint16_t* weight = kind == 0 ? p.q_weight : p.k_weight;
  const int R = p.rot_dim, half = R / 2;
  const bool turns = c0 < R;
  int partner = lane;
  float a[8], b[8];  // factors of a value and of its partner
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = 1.f, b[e] = 0.f;
  if (turns) {
    const float* cs = p.cos_sin + static_cast<int64_t>(rope_position(p, position)) * R;
    if (p.interleaved) {
      const float4 c = *reinterpret_cast<const float4*>(cs + c0 / 2);
      const float4 s = *reinterpret_cast<const float4*>(cs + half + c0 / 2);
      a[0] = a[1] = c.x, a[2] = a[3] = c.y, a[4] = a[5] = c.z, a[6] = a[7] = c.w;
      b[0] = -s.x, b[1] = s.x, b[2] = -s.y, b[3] = s.y, b[4] = -s.z, b[5] = s.z, b[6] = -s.w, b[7] = s.w;
    } else {
      const bool first = c0 < half;
      partner = lane + (first ? half / 8 : -half / 8);
      const float* at = cs + (first ? c0 : c0 - half);
      const float sign = first ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 c = *reinterpret_cast<const float4*>(at + 4 * i);
        const float4 s = *reinterpret_cast<const float4*>(at + half + 4 * i);
        a[4 * i] = c.x, a[4 * i + 1] = c.y, a[4 * i + 2] = c.z, a[4 * i + 3] = c.w;
        b[4 * i] = sign * s.x, b[4 * i + 1] = sign * s.y, b[4 * i + 2] = sign * s.z, b[4 * i + 3] = sign * s.w;
      }
    }
  }
  if (weight != nullptr) {
    const int c1 = p.interleaved ? c0 : c0 + (partner - lane) * 8;
    float w0[8], w1[8];
    unpack8(*reinterpret_cast<const uint4*>(weight + c0), w0);
    unpack8(*reinterpret_cast<const uint4*>(weight + c1), w1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] *= w0[e];
      b[e] *= p.interleaved ? w1[e ^ 1] : w1[e];
    }
  }

  for (int left = kind == 0 ? LOOPS : 1;;) {
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u) {
      if (chunk * PER_WARP + u * HEADS >= heads) break;  // the same in the whole warp
      float z[8], other[8];
      unpack8(raw[u], z);
      float r = 1.f;
      if (weight != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += z[e] * z[e];
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(ss * (1.f / D) + p.eps);
      }
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) other[e] = z[e ^ 1];
      } else {
        uint4 o;
        o.x = __shfl_sync(0xffffffffu, raw[u].x, partner);
        o.y = __shfl_sync(0xffffffffu, raw[u].y, partner);
        o.z = __shfl_sync(0xffffffffu, raw[u].z, partner);
        o.w = __shfl_sync(0xffffffffu, raw[u].w, partner);
        unpack8(o, other);
      }
      // outside the rotation a value passes as it is: an infinity times a factor of 0 would not
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float turned = turns ? fmaf(other[e], b[e], z[e] * a[e]) : z[e] * a[e];
        z[e] = weight != nullptr ? r * turned : turned;
      }
      if (h0 + u * HEADS < heads)
        *reinterpret_cast<uint4*>(dst + u * head_stride) =
            make_uint4(pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]), pack_bf16x2(z[4], z[5]),
                       pack_bf16x2(z[6], z[7]));
    }
    if (LOOPS == 1 || --left == 0 || ++chunk * PER_WARP >= heads) return;
    h0 += PER_WARP;
    src += PER_WARP * D;
    dst += kRopeUnroll * head_stride;
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u)
      if (h0 + u * HEADS < heads) raw[u] = *reinterpret_cast<const uint4*>(src + u * HEADS * D);
  }
}

// Any even rot_dim: a warp per (token, head); the head's fp32 values pass through shared memory so
// that a lane reads its rotation partner. 2-byte accesses, and the token's rotation and a 64-bit division
// again for every head: 47 us at 4096 tokens x 40 heads of 128 with rot_dim 30, 56 us with 120, where
// the other kernel takes 18.5 us. For sizes that models rarely have.
template <int D>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_write_any_kernel(const RopeParams p) {
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
  const int64_t slot = is_q ? 0 : rope_slot(p, p.slots[t]);
  uint16_t* dst = rope_target(p, t, h, slot, slot / p.page_size, slot % p.page_size);
  if (dst == nullptr) return;
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
    const int pos = rope_position(p, p.positions[t]);
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
                      num_requests, page_size, max_pages, free_capacity,
                      ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slot_mapping)) & 15) == 0};
  const size_t smem = (3 * static_cast<size_t>(num_requests) + 1) * 4;
  // Without the opt-in static and dynamic shared memory together have 48 KB.
  if (smem + kTableStatic > 48 * 1024) {
    const int rc = check_cuda(cudaFuncSetAttribute(page_tables_kernel,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (3 * kMaxRequests + 1) * 4),
                              "lm_build_page_tables: smem attribute");
    if (rc) return rc;
  }
  const int ctas = max_tokens <= 4 * kTableThreads && num_requests <= kTableThreads ? 1 : kTableCtas;
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
      launch_dependent(release_pages_kernel, dim3(1), dim3(kReleaseThreads), 0,
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
  // Pieces of 8 values where the rotation is made of them, else (an odd rot_dim, a table or weights
  // that no 16-byte load fits) a warp per head: 18.5 against 47 to 56 us at 4096 tokens x 40 heads of 128.
  const bool wide = rot_dim % (interleaved ? 8 : 16) == 0 &&
                    ((reinterpret_cast<uintptr_t>(cos_sin) | reinterpret_cast<uintptr_t>(q_norm_weight) |
                      reinterpret_cast<uintptr_t>(k_norm_weight)) & 15) == 0;
  const int per_warp = head_dim == 64 ? rope_heads_per_warp<64>() : rope_heads_per_warp<128>();
  const int loops = num_tokens >= kRopeManyTokens && num_q_heads > per_warp ? kRopeLoops : 1;
  const int chunks = wide ? (num_q_heads + per_warp * loops - 1) / (per_warp * loops) +
                                2 * ((num_kv_heads + per_warp - 1) / per_warp)
                          : 1;
  const int64_t units = wide ? num_tokens : num_tokens * heads;
  const int64_t blocks = (units + kRopeWarps - 1) / kRopeWarps;
  if (blocks > 0x7fffffff || chunks > 65535)
    return fail(LM_ERR_INVALID_ARGUMENT, "lm_rope_cache_write: too many tokens or heads");
  auto kernel = head_dim == 64 ? rope_write_any_kernel<64> : rope_write_any_kernel<128>;
  if (wide && loops == 1) kernel = head_dim == 64 ? rope_write_kernel<64, 1> : rope_write_kernel<128, 1>;
  if (wide && loops > 1)
    kernel = head_dim == 64 ? rope_write_kernel<64, kRopeLoops> : rope_write_kernel<128, kRopeLoops>;
  return check_cuda(launch_dependent(kernel, dim3(static_cast<unsigned>(blocks), chunks),
                                     dim3(kRopeWarps * 32), 0, static_cast<cudaStream_t>(stream), p),
                    "lm_rope_cache_write");
}
