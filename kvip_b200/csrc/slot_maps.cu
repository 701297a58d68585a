// Block tables and slot maps of a step from the requests' lengths (include/kvip_b200.h: KvipSlotMapsArgs).
//
// Two prefix sums over the requests (packed tokens, new blocks) decide everything, and they are small: every CTA makes
// both in shared memory, then writes its own share of the packed tokens, of the table rows and of the layout. No CTA
// needs another's result: a token on a page that this very launch appends takes the block from the free list, not from
// the table. Bound by latency: the lengths, one scan, one page entry, the stores (64 requests x 4 tokens 5.2 us in a graph, 1000 requests and
// 131072 packed tokens 6.8 us, of which a launch is about 2).
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kMapThreads = 256;
constexpr uint32_t kMapBatch = 1024;              // requests per launch
constexpr uint32_t kPerThread = kMapBatch / kMapThreads;
constexpr uint32_t kTokensPerThread = 4;

__global__ void __launch_bounds__(kMapThreads) slot_map_rows(const __grid_constant__ KvipSlotMapsArgs a) {
  __shared__ uint32_t s_start[kMapBatch + 1], s_off[kMapBatch], s_fresh[kMapBatch];
  __shared__ int32_t s_length[kMapBatch], s_held[kMapBatch];
  __shared__ uint8_t s_placed[kMapBatch];
  __shared__ uint64_t s_warp[kMapThreads / 32u];
  __shared__ uint32_t s_taken;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;

  // requests tid * kPerThread + i: consecutive per thread, so one scan of the threads' sums orders them all
  int32_t length[kPerThread], count[kPerThread], held[kPerThread];
#pragma unroll
  for (uint32_t i = 0; i < kPerThread; ++i) {
    const uint32_t b = tid * kPerThread + i;
    const bool live = b < a.batch;
    length[i] = live ? a.lengths[b] : 0;
    count[i] = live ? a.counts[b] : 0;
    held[i] = live ? a.held[b] : 0;
  }
  const int32_t head = a.head[0];
  const int64_t available = head < 0 ? 0 : static_cast<int64_t>(a.blocks) - head;
  const int64_t room = static_cast<int64_t>(a.pages) * a.block;   // fits 31 bits
  int32_t bad = 0;
  uint32_t fresh[kPerThread];
  uint64_t sum = 0;                     // tokens in the low half, new blocks in the high one
#pragma unroll
  for (uint32_t i = 0; i < kPerThread; ++i) {
    fresh[i] = 0;
    const int64_t end = static_cast<int64_t>(length[i]) + count[i];
    if (length[i] < 0 || count[i] < 0 || held[i] < 0 || held[i] > static_cast<int64_t>(a.pages) || end > room ||
        (a.layout && count[i] > static_cast<int32_t>(a.queries))) {
      bad |= static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
      count[i] = 0;
    } else if (count[i] > 0) {
      const uint32_t need = (static_cast<uint32_t>(end) - 1u) / a.block + 1u;
      if (need > static_cast<uint32_t>(held[i])) fresh[i] = need - static_cast<uint32_t>(held[i]);
    }
    sum += static_cast<uint32_t>(count[i]) | (static_cast<uint64_t>(fresh[i]) << 32);
  }
  uint64_t scan = sum;
#pragma unroll
  for (uint32_t d = 1; d < 32u; d <<= 1) {
    const uint64_t other = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += other;
  }
  if (lane == 31u) s_warp[warp] = scan;
  if (tid == 0) s_taken = 0;
  __syncthreads();
  uint64_t before = scan - sum, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kMapThreads / 32u; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  uint32_t start = static_cast<uint32_t>(before), off = static_cast<uint32_t>(before >> 32);
  const uint32_t total_tokens = static_cast<uint32_t>(all);
  // entries used: the requests up to the first one that the list cannot serve
  uint32_t served = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPerThread; ++i) {
    const uint32_t b = tid * kPerThread + i;
    const bool placed = fresh[i] == 0u || static_cast<int64_t>(off) + fresh[i] <= available;
    if (!placed) bad |= static_cast<int32_t>(KVIP_ERR_NO_SLOT);
    else if (fresh[i]) served = off + fresh[i];
    if (b < a.batch) {
      s_start[b] = start; s_off[b] = off; s_fresh[b] = placed ? fresh[i] : 0u; s_length[b] = length[i]; s_held[b] = held[i];
      s_placed[b] = placed ? 1u : 0u;
      if (blockIdx.x == 0) {
        a.starts[b] = static_cast<int32_t>(min(start, a.tokens));
        a.ends[b] = length[i] + (placed ? count[i] : 0);
        a.held_after[b] = held[i] + (placed ? static_cast<int32_t>(fresh[i]) : 0);
      }
    }
    start += static_cast<uint32_t>(count[i]);
    off += fresh[i];
  }
  if (blockIdx.x == 0) {
    served = __reduce_max_sync(0xffffffffu, served);
    if (lane == 0 && served) atomicMax(&s_taken, served);
    if (total_tokens > a.tokens) bad |= static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
    if (bad) atomicOr(a.status, bad);
  }
  if (tid == 0) s_start[a.batch] = total_tokens;
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.taken[0] = static_cast<int32_t>(s_taken);
    a.starts[a.batch] = static_cast<int32_t>(min(total_tokens, a.tokens));
  }

  // the appended entries of the table rows: requests in turn over the CTAs, a thread each; long appendages by the whole warp
  for (uint32_t b0 = 0; b0 < a.batch; b0 += gridDim.x * kMapThreads) {
    const uint32_t b = b0 + tid * gridDim.x + blockIdx.x;
    const uint32_t mine = b < a.batch ? s_fresh[b] : 0u;
    auto append = [&](uint32_t r, uint32_t p) {
      a.table[static_cast<uint64_t>(r) * a.pages + static_cast<uint32_t>(s_held[r]) + p] = a.free_blocks[static_cast<uint32_t>(head) + s_off[r] + p];
    };
    if (mine <= 2u)
      for (uint32_t p = 0; p < mine; ++p) append(b, p);
    uint32_t todo = __ballot_sync(0xffffffffu, mine > 2u);
    while (todo) {
      const uint32_t from = static_cast<uint32_t>(__ffs(static_cast<int>(todo))) - 1u;
      const uint32_t r = __shfl_sync(0xffffffffu, b, from), n = __shfl_sync(0xffffffffu, mine, from);
      todo &= todo - 1u;
      for (uint32_t p = lane; p < n; p += 32u) append(r, p);
    }
  }

  // packed tokens: four consecutive ones per thread, one search for the first
  bool hole = false;
  for (uint32_t t0 = (blockIdx.x * kMapThreads + tid) * kTokensPerThread; t0 < a.tokens;
       t0 += gridDim.x * kMapThreads * kTokensPerThread) {
    uint32_t lo = 0, hi = a.batch;   // largest b with s_start[b] <= t0
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) >> 1;
      if (s_start[mid] <= t0) lo = mid; else hi = mid;
    }
    uint32_t b = lo;
#pragma unroll
    for (uint32_t i = 0; i < kTokensPerThread; ++i) {
      const uint32_t t = t0 + i;
      if (t >= a.tokens) break;
      int64_t position = -1, slot = -1;
      int32_t request = -1;
      if (t < total_tokens) {
        while (s_start[b + 1] <= t) ++b;
        request = static_cast<int32_t>(b);
        if (s_placed[b]) {
          const uint32_t p = static_cast<uint32_t>(s_length[b]) + (t - s_start[b]);   // below pages * block
          const uint32_t page = p / a.block, held_b = static_cast<uint32_t>(s_held[b]);
          const int32_t block = page < held_b ? a.table[static_cast<uint64_t>(b) * a.pages + page]
                                              : a.free_blocks[head + s_off[b] + (page - held_b)];
          position = p;
          if (block >= 0) slot = static_cast<int64_t>(block) * a.block + (p - page * a.block);
          else hole = true;
        }
      }
      a.positions[t] = position;
      a.slot_mapping[t] = slot;
      a.requests[t] = request;
    }
  }

  if (hole) atomicOr(a.status, static_cast<int32_t>(KVIP_ERR_NO_SLOT));

  if (a.layout) {   // rows GATHER, QUERY_VALID, UNPACK, OUTPUT_VALID of the query slots: packed tokens behind the last output row are not there
    const uint32_t slots = a.batch * a.queries, kept = min(total_tokens, a.tokens);
    for (uint32_t s = blockIdx.x * kMapThreads + tid; s < slots; s += gridDim.x * kMapThreads) {
      const uint32_t b = s / a.queries, q = s - b * a.queries;
      const bool live = q < s_start[b + 1] - s_start[b] && s_start[b] + q < kept;
      a.layout[s] = live ? static_cast<int64_t>(s_start[b] + q) : 0;
      a.layout[slots + s] = live ? 1 : 0;
      int64_t from = 0;
      if (s < kept) {
        uint32_t lo = 0, hi = a.batch;
        while (hi - lo > 1u) {
          const uint32_t mid = (lo + hi) >> 1;
          if (s_start[mid] <= s) lo = mid; else hi = mid;
        }
        while (s_start[lo + 1] <= s) ++lo;
        from = static_cast<int64_t>(lo) * a.queries + (s - s_start[lo]);
      }
      a.layout[2 * slots + s] = from;
      a.layout[3 * slots + s] = s < kept ? 1 : 0;
    }
  }
}

// The end of a planned step, one CTA: as many loads as a plan, no scan (as single torch operations 16 launches).
__global__ void __launch_bounds__(kMapThreads) commit_rows(const KvipCommitTablesArgs a) {
  bool bad = false;
  for (uint32_t b = threadIdx.x; b < a.batch; b += kMapThreads) {
    const int32_t length = a.lengths[b], kept = a.kept[b], room = min(a.ends[b] - length, a.starts[b + 1] - a.starts[b]);
    bad |= kept > room;
    const int32_t after = length + max(0, min(kept, room));
    a.lengths[b] = after;
    a.ends[b] = after;
    a.held[b] = a.held_after[b];
  }
  if (threadIdx.x == 0) {
    a.head[0] += a.taken[0];
    a.taken[0] = 0;
  }
  if (bad) atomicOr(a.status, static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE));
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_b200_slot_maps(const KvipSlotMapsArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->lengths && a->counts && a->held && a->free_blocks && a->head && a->table && a->positions &&
                   a->slot_mapping && a->requests && a->starts && a->ends && a->held_after && a->taken && a->status,
               "slot_maps: null pointer");
  KVIP_REQUIRE(a->batch >= 1 && a->batch <= kMapBatch, "slot_maps: batch must be in 1..1024");
  KVIP_REQUIRE(a->block >= 1 && a->pages >= 1 && static_cast<uint64_t>(a->pages) * a->block <= 0x7fffffffull,
               "slot_maps: pages * block must fit int32");
  // the packed numbering is kept in 32 bits
  KVIP_REQUIRE(static_cast<uint64_t>(a->batch) * a->pages * a->block <= 0xffffffffull && a->tokens >= 1 && a->tokens <= 0x7fffffffu,
               "slot_maps: batch * pages * block must fit 32 bits, tokens 31");
  KVIP_REQUIRE(a->blocks <= 0x7fffffffu, "slot_maps: too many blocks");
  KVIP_REQUIRE(!a->layout || (a->queries >= 1 && a->queries <= KVIP_MAX_QUERIES), "slot_maps: 1..4 query slots per request");
  const uint32_t share = kMapThreads * kTokensPerThread;
  uint32_t grid = (a->tokens + share - 1) / share;
  if (grid > device_sm_count()) grid = device_sm_count();
  slot_map_rows<<<grid, kMapThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  count_launch();
  return check_launch("slot_map_rows");
}

extern "C" uint32_t kvip_b200_commit_tables(const KvipCommitTablesArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->kept && a->starts && a->held_after && a->lengths && a->held && a->ends && a->head && a->taken && a->status,
               "commit_tables: null pointer");
  KVIP_REQUIRE(a->batch >= 1 && a->batch <= kMapBatch, "commit_tables: batch must be in 1..1024");
  commit_rows<<<1, kMapThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  count_launch();
  return check_launch("commit_rows");
}
