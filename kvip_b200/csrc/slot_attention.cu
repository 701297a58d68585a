// Attention of packed query tokens over selected pool rows and drafted rows (include/kvip_b200.h: KvipAttentionArgs).
//
//   out[t,h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale' q.k_j - ref),   v_j = the first 512 elements of k_j
//
// A CTA takes one share of the rows of one (token, group of at most 64 heads) and turns the products round so that the
// gathered rows are always the M operand and the heads the N operand:
//
//   S^T [64 rows x heads]   = K [64 x 576] . Q^T            (one accumulator lane per row, one column per head)
//   O^T [512 x heads]      += V^T [512 x 64] . P^T [64 x heads]   (four accumulators of 128 value elements)
//
// Both read the same tile in shared memory: a row is nine 128-byte pieces, each piece a column of the 128-byte swizzle
// atom, K-major for the first product (elements along K) and M-major for the second (elements along M, rows along K).
// So every row is fetched once, 512 accumulator columns of a [heads x 512] output become 4 x heads <= 256, and small head
// counts cost small N. Rows as lanes also make the softmax cheap: p is scaled by a reference `ref` per head that only has
// to be near the running maximum, so a tile needs no reduction over rows unless some score leaves ref + 8 (fp16: 15; then the
// maximum is taken, and the accumulators and sums are rescaled); sums of p stay per thread until the end.
//
// p is rounded to the rows' type for the second product (half a step, as the output is; fp16 ranges see Reference); its sum is taken before the
// rounding, in fp32, because the log-sum is an output too.
//
// Bound, at 64 heads per CTA, by the loop of the two stages that shared memory holds beside the queries: a tile's rows need 3200
// clocks to land while the other tile's products run (1253 for the copies alone), 1170 more until its scores are complete, 1140 for
// the softmax and 760 until the value product lets go: 6270 clocks for two tiles. The tensor pipe is busy in about 56 % of a CTA's cycles. At
// 16 heads by HBM. Measured on one B200: 64 tokens x 128 heads x 2048 rows 64.5 us (36.5 GFLOP, 169 MB once), 128 tokens x 16 heads
// 60.8 us (5.0 TB/s of rows), one token x 128 heads 13.7 us.
#include <atomic>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kWidth = KVIP_ATTENTION_WIDTH, kValue = KVIP_ATTENTION_VALUE;
constexpr uint32_t kTile = 64;                          // rows per tile
constexpr uint32_t kPieces = kWidth / 64;               // 128-byte pieces per row
constexpr uint32_t kPieceBytes = kTile * 128;           // one piece of every row of a tile
constexpr uint32_t kStageBytes = kPieces * kPieceBytes; // 73,728
constexpr uint32_t kStages = 2;
constexpr uint32_t kGroupHeads = 64;
constexpr uint32_t kParts = 4;                          // a stage is filled, read and released in four groups of pieces: two for each block
                                                        // of 128 value elements, and with the last the piece behind the value
__host__ __device__ constexpr uint32_t part_end(uint32_t part) { return part + 1 == kParts ? kPieces : 2 * part + 2; }
// Softmax: four warps per 16 heads. Behind them four loaders and an issuer for each product.
constexpr uint32_t kLoaderWarps = 4, kRole = 128, kSideHeads = 16;
constexpr uint32_t kMaxSplits = 8;                      // CTAs of a cluster
template <uint32_t kN> struct Warps {
  static constexpr uint32_t kSides = kN / kSideHeads, kLoader = 4 * kSides, kScore = kLoader + kLoaderWarps, kValue = kScore + 1;
  static constexpr uint32_t kThreads = 32 * (kValue + 1);
};
constexpr uint32_t kOutRow = kValue * 2 + 16;           // bytes of an output row while it is laid out: four banks further than the last
// Weights lie at most 2^kSlack above the reference, and it moves to 2^kLift below the maximum. fp16 has 24 powers of two below 1 and 15
// above: the largest weight of a head stays between 2^10 and 2^15, so weights keep all their bits down to 2^-24 of the largest, and what 2^20
// rows beneath lose is 2^-15 of the result at most. With both as for bf16, whose exponents reach 2^-126, rows 2^-25 of the largest were lost.
template <typename T> struct Reference { static constexpr float kSlack = 8.f, kLift = 0.f; };
template <> struct Reference<__half> { static constexpr float kSlack = 15.f, kLift = 10.f; };
constexpr float kLowest = -3.402823466e38f;             // the reference before any row: finite, so that a score of -inf weighs 2^(-inf) = 0
constexpr uint32_t kDefaultWaitKilocycles = 2000000u;   // about one second of SM clock
constexpr uint32_t kPromptKilocycles = 100000u;         // limits up to 50 ms

// What token t may read.
struct Rows {
  uint32_t base, limit;       // first pool row of the owner and how many it has (0: none may be read)
  uint32_t draft, drafted;    // first drafted row of the request, and how many of them bound those the token sees
  uint64_t seen;
  int32_t bad, request;
};
struct Control {                                        // behind the tiles in shared memory
  uint64_t full[kStages][kParts], empty[kStages][kParts], scored[2], taken[2], weighted, query_full;
  uint32_t valid[kStages][kLoaderWarps];                // row 16 i + b of the tile is there: bit b of word i
  float reduce[4][kGroupHeads];
  float factor[kGroupHeads], top[kGroupHeads];
  Rows rows;
  uint32_t tmem, abort_flag, last[32];                  // per warp
};

template <uint32_t kN> struct Layout {
  static constexpr uint32_t kQuery = kStages * kStageBytes;
  static constexpr uint32_t kWeights = kQuery + kPieces * kN * 128;
  static constexpr uint32_t kControl = kWeights + kTile * 128;
  static constexpr uint32_t kBytes = kControl + sizeof(Control);
};
static_assert(Layout<kGroupHeads>::kBytes <= 227 * 1024, "shared memory");

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A try sleeps until the phase ends or some time that the hardware sets is over, far more than a thousand clocks; a test does not.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}
struct Waits {
  volatile uint32_t* abort_flag;   // set by the first wait of the CTA that gives up; read by all the others
  long long limit;                 // SM clock cycles a wait may take
  bool prompt;                     // a limit near the length of a try's sleep: poll
};
__device__ __forceinline__ bool mbar_done(uint32_t bar, uint32_t parity, const Waits& w) { return w.prompt ? mbar_test(bar, parity) : mbar_try(bar, parity); }
__device__ __forceinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, const Waits& w) {
  const long long start = clock64();
  do {                                 // the clock is read behind every try
    if (mbar_done(bar, parity, w)) return true;
    if (*w.abort_flag) return false;
  } while (clock64() - start <= w.limit);
  *w.abort_flag = 1u;
  return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Waits& w) {
  return mbar_done(bar, parity, w) || mbar_wait_slow(bar, parity, w);
}
// Barrier of `kThreads` threads that also tells all of them whether any has `flag`.
template <uint32_t kThreads = kRole> __device__ __forceinline__ bool role_any(uint32_t id, bool flag) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"(flag ? 1u : 0u), "r"(id), "n"(kThreads) : "memory");
  return any != 0u;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u) : "memory");
}
// Shared-memory operand in 128-byte swizzle, 8-row groups 1024 bytes apart; `pieces` is the distance between 64-element
// columns of an M-major operand (unused by K-major ones).
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t pieces) {
  return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(pieces >> 4) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 16 lanes x 16 fp32 columns: a thread holds rows lane/4 (v[4j], v[4j + 1]) and lane/4 + 8 (v[4j + 2], v[4j + 3]), columns
// 8j + 2 (lane%4) + {0, 1}.
__device__ __forceinline__ void tmem_ld_blocks(uint32_t address, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(address) : "memory");
}
// 32 lanes x 8 fp32 columns: a thread holds its lane's row.
__device__ __forceinline__ void tmem_ld_rows(uint32_t address, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(address) : "memory");
}
__device__ __forceinline__ void tmem_st_rows(uint32_t address, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tmem_ld_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes into shared memory, zeros where `present` is false.
__device__ __forceinline__ void copy16(uint32_t to, uint64_t from, bool present) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(present ? 16u : 0u) : "memory");
}
// Arrives at the barrier when this thread's copies so far have landed.
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void load_query(uint32_t to, const CUtensorMap* map, uint32_t x, uint32_t head, uint32_t token, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(bar) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t address, uint32_t rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
  return there;
}
__device__ __forceinline__ float load_remote(uint32_t address) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(address) : "memory");
  return x;
}
__device__ __forceinline__ float4 load_remote4(uint32_t address) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(address) : "memory");
  return x;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader != 0u;
}
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float x, float y);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float x, float y) {
  __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float x, float y) {
  __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ Rows rows_of(const KvipAttentionArgs& a, uint32_t t) {
  const int32_t request = a.requests ? a.requests[t] : static_cast<int32_t>(t / a.queries);
  Rows r{0u, a.output_stride, 0u, 0u, 0ull, 0, request};
  if (request < 0) return r;   // padding
  const uint64_t mask = a.draft && a.ancestors ? static_cast<uint64_t>(a.ancestors[t]) : 0ull;
  if (static_cast<uint32_t>(request) >= a.batch) {
    r.limit = 0;
    r.bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
    return r;
  }
  const int32_t owner = a.row_owners ? a.row_owners[request] : request;
  const int64_t first = a.draft ? a.starts[request] : 0, behind = a.draft ? a.starts[request + 1] : 0;
  const uint64_t base = static_cast<uint64_t>(static_cast<uint32_t>(owner)) * a.output_stride;
  if (owner < 0 || base + a.output_stride > a.pool_rows) {
    r.limit = 0;
    r.bad = static_cast<int32_t>(KVIP_ERR_SOURCE);
  } else {
    r.base = static_cast<uint32_t>(base);
  }
  if (a.draft) {
    const int64_t own = static_cast<int64_t>(t) - first;
    if (first < 0 || behind < first || behind > static_cast<int64_t>(a.tokens)) {
      r.bad |= static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
    } else {
      const uint32_t nodes = static_cast<uint32_t>(min(static_cast<int64_t>(64), behind - first));
      if (behind - first > 64) r.bad |= static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);   // what lies behind the 64th is not seen
      r.draft = static_cast<uint32_t>(first);
      r.seen = a.ancestors ? mask : (own < 0 ? 0ull : own >= 63 ? ~0ull : (2ull << own) - 1ull);
      if (nodes < 64u) r.seen &= (1ull << nodes) - 1ull;
      r.drafted = r.seen ? 64u - static_cast<uint32_t>(__clzll(static_cast<long long>(r.seen))) : 0u;
    }
  }
  return r;
}

template <typename T, uint32_t kN>
__global__ void __launch_bounds__(Warps<kN>::kThreads, 1)
attend_tiles(const __grid_constant__ CUtensorMap query_map, const __grid_constant__ KvipAttentionArgs a, const uint32_t group_heads,
             const uint32_t splits_log, const uint32_t first_token, const uint32_t behind_token) {
  constexpr uint32_t kSides = Warps<kN>::kSides, kFirstLoaderWarp = Warps<kN>::kLoader, kScoreWarp = Warps<kN>::kScore, kValueWarp = Warps<kN>::kValue;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  Control& c = *reinterpret_cast<Control*>(smem + Layout<kN>::kControl);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t splits = 1u << splits_log, split = blockIdx.x & (splits - 1u), group = blockIdx.x >> splits_log, t = first_token + blockIdx.z * gridDim.y + blockIdx.y;
  if (t >= behind_token) return;                 // behind the last token: whole clusters
  const uint32_t head0 = group * group_heads, heads = min(group_heads, a.heads - head0);
  const int32_t* list = a.slots + static_cast<uint64_t>(t) * a.entries;
  const bool vectors = (a.entries & 3u) == 0u && (reinterpret_cast<uintptr_t>(a.slots) & 15u) == 0u;
  auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
  uint32_t last = 0;
  if (warp == kScoreWarp) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&query_map)) : "memory");
      for (uint32_t s = 0; s < kStages; ++s)
        for (uint32_t part = 0; part < kParts; ++part) { mbar_init(bar(c.full[s][part]), 32 * kLoaderWarps + (part ? 0 : kLoaderWarps)); mbar_init(bar(c.empty[s][part]), 1); }
      for (uint32_t s = 0; s < 2; ++s) { mbar_init(bar(c.scored[s]), 1); mbar_init(bar(c.taken[s]), 4 * kSides); }
      mbar_init(bar(c.weighted), 4 * kSides); mbar_init(bar(c.query_full), 1);
      c.abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      fence_async();
      expect_bytes(bar(c.query_full), kPieces * kN * 128u);   // waited for in any case: by this warp
      for (uint32_t piece = 0; piece < kPieces; ++piece)
        load_query(base + Layout<kN>::kQuery + piece * (kN * 128u), &query_map, piece * 64u, head0, t, bar(c.query_full));
    }
    __syncwarp();
    // all of tensor memory: one CTA per SM
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&c.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == kValueWarp) {
    if (lane == 0) c.rows = rows_of(a, t);         // a chain of loads, beside the others' walk along the list
  } else if (vectors) {
    // lists end in -1 where a context is short: the last entry in use bounds the tiles
    for (uint32_t k = tid; k < a.entries / 4u; k += 32u * kScoreWarp) {
      const int4 e = __ldg(reinterpret_cast<const int4*>(list) + k);
      if ((e.x & e.y & e.z & e.w) >= 0) last = 4u * k + (e.w >= 0 ? 4u : e.z >= 0 ? 3u : e.y >= 0 ? 2u : 1u);
    }
  } else {
    for (uint32_t k = tid; k < a.entries; k += 32u * kScoreWarp)
      if (list[k] >= 0) last = k + 1u;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) c.last[warp] = last;
  fence_before();
  __syncthreads();
  fence_after();
  const Rows rows = c.rows;
  last = __reduce_max_sync(0xffffffffu, lane < kScoreWarp ? c.last[lane] : 0u);
  const uint32_t tmem = c.tmem;
  // tiles of the list, then one of the drafted rows
  const uint32_t listed = rows.limit ? last : 0u, list_tiles = (listed + kTile - 1) / kTile, tiles = list_tiles + (rows.drafted ? 1u : 0u);
  // A list may be far shorter than its entries. Up to three tiles are one CTA's: joining shares takes as long as two more of them.
  const uint32_t shares_log = tiles <= 3u ? 0u : splits_log, shares = 1u << shares_log;
  const bool idle = rows.request < 0 || split >= shares;
  const uint32_t first = idle ? 0u : tiles * split >> shares_log, count = idle ? 0u : (tiles * (split + 1u) >> shares_log) - first;
  const Waits waits{&c.abort_flag, static_cast<long long>(a.wait_kilocycles ? a.wait_kilocycles : kDefaultWaitKilocycles) << 10,
                    a.wait_kilocycles - 1u < kPromptKilocycles};
  constexpr uint32_t kScores = 0, kOut = 2 * kN;   // tensor-memory columns: two score tiles, four value blocks
  auto none = [&](uint32_t s) { return (c.valid[s][0] | c.valid[s][1] | c.valid[s][2] | c.valid[s][3]) == 0u; };

  if (warp >= kFirstLoaderWarp && warp < kScoreWarp) {
    // ================= loaders: each copies 16 rows of every tile =================
    // A lane copies 16 bytes of one of four rows, so that an instruction takes whole 128-byte lines and fills all banks of
    // four swizzled rows. Measured alone: 1253 clocks a tile from L2 on all SMs, 6.2 TB/s from HBM (tensor-map gathers of four rows: 1466
    // and 6.1; they also hold the products back more, 67.6 against 66.5 us for 64 tokens x 128 heads).
    const uint32_t loader = warp - kFirstLoaderWarp;
    int32_t bad = warp == kFirstLoaderWarp && lane == 0 ? rows.bad : 0;
    const uint64_t pool = reinterpret_cast<uint64_t>(a.pool), pool_row = pool + static_cast<uint64_t>(rows.base) * (kWidth * 2u);
    const uint64_t draft_bytes = static_cast<uint64_t>(a.draft_token) * 2u;
    const uint64_t draft_row = reinterpret_cast<uint64_t>(a.draft) + rows.draft * draft_bytes;
    auto entry_of = [&](uint32_t n) -> int32_t {     // list entry of row 16 loader + lane of tile n, -1 behind the list
      const uint32_t k = (first + n) * kTile + loader * 16u + lane;
      return lane < 16u && n < count && k < listed ? __ldg(list + k) : -1;
    };
    const uint32_t unit = lane & 7u, to = base + (loader * 16u + (lane >> 3)) * 128u;
    int32_t next = entry_of(0);
    for (uint32_t n = 0; n < count; ++n) {
      const uint32_t g = n & 1u, phase = ((n >> 1) & 1u) ^ 1u;
      const int32_t slot = next;
      next = entry_of(n + 1u);                       // lands while this tile is copied
      uint64_t source = 0;                           // of row 16 loader + lane
      if (first + n < list_tiles) {
        if (slot >= 0) {
          if (static_cast<uint32_t>(slot) < rows.limit) source = pool_row + static_cast<uint64_t>(static_cast<uint32_t>(slot)) * (kWidth * 2u);
          else bad |= static_cast<int32_t>(KVIP_ERR_SOURCE);
        }
      } else if (lane < 16u && ((rows.seen >> (loader * 16u + lane)) & 1ull)) {
        source = draft_row + (loader * 16u + lane) * draft_bytes;
      }
      const uint32_t present = __ballot_sync(0xffffffffu, source != 0);
      uint64_t from[4];
      bool there[4];
#pragma unroll
      for (uint32_t q = 0; q < 4u; ++q) {
        const uint64_t row = __shfl_sync(0xffffffffu, source, q * 4u + (lane >> 3));
        there[q] = row != 0;
        from[q] = (there[q] ? row : pool) + unit * 16u;
      }
      bool alive = true;
#pragma unroll
      for (uint32_t part = 0; part < kParts; ++part) {
        alive = __all_sync(0xffffffffu, mbar_wait(bar(c.empty[g][part]), phase, waits));
        if (!alive) break;
        if (part == 0 && lane == 0) {                // every reader of the mask of tile n - 2 has done with it
          c.valid[g][loader] = present;
          mbar_arrive(bar(c.full[g][0]));
        }
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) {
          const uint32_t row = loader * 16u + q * 4u + (lane >> 3);
#pragma unroll
          for (uint32_t piece = 2u * part; piece < part_end(part); ++piece)
            copy16(to + g * kStageBytes + piece * kPieceBytes + q * 512u + ((unit ^ (row & 7u)) << 4), from[q] + piece * 128u, there[q]);
        }
        arrive_after_copies(bar(c.full[g][part]));
      }
      if (!alive) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bad) atomicOr(a.status, bad);
  } else if (warp >= kScoreWarp) {
    // ================= issuers: the warp walks together, one elected thread issues =================
    constexpr uint32_t kFormat = __is_same(T, __nv_bfloat16) ? 1u : 0u;
    constexpr uint32_t kBase = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((kN >> 3) << 17);
    constexpr uint32_t kScoreDesc = kBase | ((64u >> 4) << 24);
    constexpr uint32_t kValueDesc = kBase | (1u << 15) | (1u << 16) | ((128u >> 4) << 24);   // both operands M/N-major
    const bool leader = elect_one();
    auto wait = [&](const uint64_t& b, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar(b), phase, waits)); };
    if (warp == kScoreWarp) {                // S^T of tile n, part by part as they come
      bool alive = wait(c.query_full, 0);
      for (uint32_t n = 0; alive && n < count; ++n) {
        const uint32_t s = n & 1u, phase = (n >> 1) & 1u;
        if (!wait(c.taken[s], phase ^ 1u)) break;   // the scores of tile n - 2 have been read
        const uint32_t d = tmem + kScores + s * kN;
        const uint64_t da = operand(base + s * kStageBytes, 16u), db = operand(base + Layout<kN>::kQuery, 16u);
#pragma unroll
        for (uint32_t part = 0; part < kParts; ++part) {
          alive = alive && wait(c.full[s][part], phase);
          if (!alive) break;
          fence_after();
          if (leader) {
            fence_async();                   // the rows were written by ordinary copies
            if (!none(s)) {
#pragma unroll
              for (uint32_t piece = 2u * part; piece < part_end(part); ++piece) {
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
                  mma(d, da + (piece * (kPieceBytes >> 4) + 2u * k), db + (piece * (kN * 8u) + 2u * k), kScoreDesc, (piece | k) != 0u);
              }
            }
            if (part == kParts - 1u) commit(bar(c.scored[s]));
          }
          __syncwarp();
        }
      }
    } else {                                 // O^T += V^T P^T of tile n
      bool written = false;
      for (uint32_t n = 0; n < count; ++n) {
        const uint32_t s = n & 1u;
        if (!wait(c.weighted, n & 1u)) break;
        fence_after();
        const bool empty = none(s);
        const uint64_t da = operand(base + s * kStageBytes, kPieceBytes), db = operand(base + Layout<kN>::kWeights, 16u);
        if (leader) {
#pragma unroll
          for (uint32_t m = 0; m < 4; ++m) {
            if (!empty) {
#pragma unroll
              for (uint32_t k = 0; k < kTile / 16u; ++k)
                mma(tmem + kOut + m * kN, da + (2u * m * (kPieceBytes >> 4) + k * 128u), db + k * 128u, kValueDesc, written || k != 0u);
            }
            commit(bar(c.empty[s][m]));
          }
        }
        __syncwarp();
        written = written || !empty;
      }
    }
  } else {
    // ================= softmax: rows 16 w + lane / 4 and + 8 of every tile, 16 heads =================
    constexpr uint32_t kBlocks = 2;          // blocks of eight heads; a thread holds two heads of each, for two rows
    const uint32_t side = warp >> 2, w = warp & 3u, head_at = side * kSideHeads;
    float ref[2 * kBlocks], sum[2 * kBlocks];
#pragma unroll
    for (uint32_t j = 0; j < 2 * kBlocks; ++j) { ref[j] = kLowest; sum[j] = 0.f; }
    const float scale = a.scale * 1.4426950408889634f;
    const uint32_t quad = (w * 32u) << 16;
    const uint32_t row0 = w * 16u + (lane >> 2);
    bool dead = false, written = false;
    for (uint32_t n = 0; n < count; ++n) {
      const uint32_t s = n & 1u, phase = (n >> 1) & 1u;
      bool ok = !dead && mbar_wait(bar(c.scored[s]), phase, waits) && mbar_wait(bar(c.full[s][0]), phase, waits);
      ok = __all_sync(0xffffffffu, ok);
      const bool empty = ok && none(s);        // the same for all that could wait: the mask belongs to the tile
      const uint32_t word = c.valid[s][w] >> (lane >> 2);
      const bool has0 = word & 1u, has1 = (word >> 8) & 1u;
      uint32_t v[4 * kBlocks];
      if (ok) {
        if (!empty) {
          fence_after();
          tmem_ld_blocks(tmem + quad + kScores + s * kN + head_at, v);
          tmem_ld_done();
          fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(c.taken[s]));
      }
      // scores in units of log2; one too far above its reference makes the whole side take the maximum
      float x[4 * kBlocks];
      bool above = false;
#pragma unroll
      for (uint32_t j = 0; j < 4 * kBlocks; ++j) {
        const bool has = ok && ((j & 2u) ? has1 : has0);
        x[j] = has ? __uint_as_float(v[j]) * scale : -INFINITY;
        above |= x[j] - ref[(j >> 2) * 2u + (j & 1u)] > Reference<T>::kSlack;
      }
      // Weights against the reference as it stands: on their way while the warps agree that it may stand.
      float e[4 * kBlocks];
#pragma unroll
      for (uint32_t j = 0; j < 4 * kBlocks; ++j) e[j] = exp2_fast(x[j] - ref[(j >> 2) * 2u + (j & 1u)]);
      // the product of the tile before has read its weights, and every tile before is in the accumulators
      if (n && ok) ok = mbar_wait(bar(c.empty[(n - 1u) & 1u][kParts - 1u]), ((n - 1u) >> 1) & 1u, waits);
      // an empty tile is voted on too: a warp whose wait ran out does not know that it is one
      if (role_any(1u + side, above || !ok)) {
        if (role_any(1u + side, !ok)) { dead = true; break; }
#pragma unroll
        for (uint32_t j = 0; j < 2 * kBlocks; ++j) {
          const uint32_t at = (j >> 1) * 4u + (j & 1u);
          float top = fmaxf(x[at], x[at + 2]);
#pragma unroll
          for (uint32_t o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (lane < 4) c.reduce[w][head_at + (j >> 1) * 8u + lane * 2u + (j & 1u)] = top;
        }
        role_any(1u + side, false);
#pragma unroll
        for (uint32_t j = 0; j < 2 * kBlocks; ++j) {
          const uint32_t h = head_at + (j >> 1) * 8u + (lane & 3u) * 2u + (j & 1u);
          const float top = fmaxf(fmaxf(c.reduce[0][h], c.reduce[1][h]), fmaxf(c.reduce[2][h], c.reduce[3][h]));
          const float next = fmaxf(ref[j], top - Reference<T>::kLift);
          const float factor = next == ref[j] ? 1.f : exp2_fast(ref[j] - next);   // 0 the first time
          ref[j] = next;
          sum[j] *= factor;
          if (w == 0 && lane < 4) c.factor[h] = factor;
        }
        role_any(1u + side, false);
        if (written) {                         // the accumulators hold the tiles before this one
          fence_after();
          for (uint32_t m = 0; m < 4; ++m) {
#pragma unroll
            for (uint32_t h = head_at; h < head_at + kSideHeads; h += 8) {
              uint32_t o[8];
              tmem_ld_rows(tmem + quad + kOut + m * kN + h, o);
              tmem_ld_done();
#pragma unroll
              for (uint32_t i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c.factor[h + i]);
              tmem_st_rows(tmem + quad + kOut + m * kN + h, o);
            }
          }
          tmem_st_done();
        }
#pragma unroll
        for (uint32_t j = 0; j < 4 * kBlocks; ++j) e[j] = exp2_fast(x[j] - ref[(j >> 2) * 2u + (j & 1u)]);
      }
      if (empty) {
        if (lane == 0) mbar_arrive(bar(c.weighted));
        continue;
      }
      uint32_t p[2 * kBlocks];                 // weights of a row, two heads in a word: row 0 then row 1
#pragma unroll
      for (uint32_t j = 0; j < kBlocks; ++j) {
        sum[2 * j] += e[4 * j] + e[4 * j + 2];
        sum[2 * j + 1] += e[4 * j + 1] + e[4 * j + 3];
        p[2 * j] = pack_pair<T>(e[4 * j], e[4 * j + 1]);
        p[2 * j + 1] = pack_pair<T>(e[4 * j + 2], e[4 * j + 3]);
      }
      const uint32_t to = base + Layout<kN>::kWeights + row0 * 128u + (lane & 3u) * 4u;
#pragma unroll
      for (uint32_t j = 0; j < kBlocks; ++j) {
        const uint32_t at = to + (((side * kBlocks + j) ^ (row0 & 7u)) << 4);   // row0 + 8 has the same swizzle
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(p[2 * j]) : "memory");
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 1024u), "r"(p[2 * j + 1]) : "memory");
      }
      fence_async();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(c.weighted));
      written = true;
    }
    // sums over the rows of all tiles
#pragma unroll
    for (uint32_t j = 0; j < 2 * kBlocks; ++j) {
      const uint32_t h = head_at + (j >> 1) * 8u + (lane & 3u) * 2u + (j & 1u);
      float total = sum[j];
#pragma unroll
      for (uint32_t o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      if (lane < 4) {
        c.reduce[w][h] = total;
        if (w == 0) c.top[h] = ref[j];
      }
    }
    if (!written && w == 0 && lane < 4)
      for (uint32_t j = 0; j < 2 * kBlocks; ++j) c.top[head_at + (j >> 1) * 8u + lane * 2u + (j & 1u)] = -INFINITY;
    if (count && !dead && !mbar_wait(bar(c.empty[(count - 1u) & 1u][kParts - 1u]), ((count - 1u) >> 1) & 1u, waits)) dead = true;
    dead = role_any<kSides * kRole>(kSides + 1u, dead);
    if (dead || idle) {
      written = false;                       // a share that cannot be trusted counts as empty; the status says so
      if (tid < kN) c.top[tid] = -INFINITY;
    }
    fence_after();
    if (tid < heads) {
      const float total = (c.reduce[0][tid] + c.reduce[1][tid]) + (c.reduce[2][tid] + c.reduce[3][tid]);
      if (shares > 1) c.factor[tid] = written ? total : 0.f;   // no rows: no mass; scores of NaN have a mass of NaN
      else c.factor[tid] = written && total != 0.f ? 1.f / total : 0.f;   // scores of -inf have no mass either
      if (shares == 1 && !idle && !dead)
        a.lse[static_cast<uint64_t>(t) * a.heads + head0 + tid] = written ? (c.top[tid] + log2f(total)) * 0.6931471805599453f : -INFINITY;
    }
    // The output is laid out in the stages (all products have read them). Accumulators have value elements as rows and heads as
    // columns: 8 x 8 blocks are transposed on their way into shared memory, and whole rows leave by copies. A share that
    // will be joined stays here as it is, in fp32 and undivided.
    if (shares == 1) {
      role_any<kSides * kRole>(kSides + 1u, false);
      if (!idle && !dead) {
        // addresses of stored rows: lanes 0-7 give the heads of a block for value elements 0-7, 8-15 for 8-15, 16-31 the next block's
        const uint32_t store = base + ((lane & 7u) + (lane >> 4) * 8u) * kOutRow + ((lane >> 3) & 1u) * 16u;
        for (uint32_t block = side; block < 4u; block += kSides) {
#pragma unroll
          for (uint32_t half = 0; half < 2; ++half) {
            uint32_t o[kN / 2];
            if (written) {
#pragma unroll
              for (uint32_t h = 0; h < kN; h += 16) tmem_ld_blocks(tmem + quad + (half << 20) + kOut + block * kN + h, o + h / 2);
              tmem_ld_done();
            }
            const uint32_t element = block * 128u + w * 32u + half * 16u;
#pragma unroll
            for (uint32_t j = 0; j < kN / 8u; j += 2) {
              uint32_t q[4];
#pragma unroll
              for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t* e = o + 4 * (j + i);
                const float2 f = *reinterpret_cast<const float2*>(&c.factor[8u * (j + i) + 2u * (lane & 3u)]);
                q[2 * i] = written ? pack_pair<T>(__uint_as_float(e[0]) * f.x, __uint_as_float(e[1]) * f.y) : 0u;
                q[2 * i + 1] = written ? pack_pair<T>(__uint_as_float(e[2]) * f.x, __uint_as_float(e[3]) * f.y) : 0u;
              }
              asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                           ::"r"(store + j * 8u * kOutRow + element * 2u), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
            }
          }
        }
      }
      fence_async();
      role_any<kSides * kRole>(kSides + 1u, false);
      if (tid < heads && !idle && !dead) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                     ::"l"(static_cast<T*>(a.out) + (static_cast<uint64_t>(t) * a.heads + head0 + tid) * kValue), "r"(base + tid * kOutRow), "r"(kValue * 2u)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      }
    } else if (written) {
      for (uint32_t block = side; block < 4u; block += kSides) {
        const uint32_t element = block * 128u + w * 32u + lane;
#pragma unroll
        for (uint32_t h0 = 0; h0 < kN; h0 += 16) {
          uint32_t o[16];
          tmem_ld_rows(tmem + quad + kOut + block * kN + h0, o);
          tmem_ld_rows(tmem + quad + kOut + block * kN + h0 + 8u, o + 8);
          tmem_ld_done();
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) reinterpret_cast<float*>(smem)[(h0 + i) * kValue + element] = __uint_as_float(o[i]);
        }
      }
    }
    fence_before();
  }

  // ---- shares of one unit, a CTA each: every CTA joins the heads rank, rank + splits, .. out of all of them -------------
  //   out = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(reference of share s - the largest)
  if (shares > 1) {
    cluster_barrier();
    if (rows.request >= 0) {
      for (uint32_t item = warp; ; item += Warps<kN>::kThreads / 32u) {   // half a row per warp
        const uint32_t h = split + (item >> 1) * shares, element = (item & 1u) * 256u + lane * 4u;
        if (h >= heads) break;
        float tops[kMaxSplits], top = -INFINITY;
#pragma unroll
        for (uint32_t s = 0; s < kMaxSplits; ++s) {
          tops[s] = load_remote(remote(smem_u32(&c.top[h]), min(s, shares - 1u)));
          if (s >= shares) tops[s] = -INFINITY;
        }
#pragma unroll
        for (uint32_t s = 0; s < kMaxSplits; ++s) top = fmaxf(top, tops[s]);
        float total = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t s0 = 0; s0 < kMaxSplits; s0 += 4) {                  // four shares' numbers on their way at a time
          if (s0 >= shares) break;
          float4 low[4], high[4];
          float sums[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t s = min(s0 + i, shares - 1u), from = remote(base + (h * kValue + element) * 4u, s);
            sums[i] = load_remote(remote(smem_u32(&c.factor[h]), s));
            low[i] = load_remote4(from);
            high[i] = load_remote4(from + 512u);
          }
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            if (s0 + i >= shares || sums[i] == 0.f) continue;             // no such share, or an empty one: it has written nothing
            const float weight = exp2_fast(tops[s0 + i] - top);
            total = fmaf(weight, sums[i], total);
            y[0] = fmaf(weight, low[i].x, y[0]); y[1] = fmaf(weight, low[i].y, y[1]); y[2] = fmaf(weight, low[i].z, y[2]); y[3] = fmaf(weight, low[i].w, y[3]);
            y[4] = fmaf(weight, high[i].x, y[4]); y[5] = fmaf(weight, high[i].y, y[5]); y[6] = fmaf(weight, high[i].z, y[6]); y[7] = fmaf(weight, high[i].w, y[7]);
          }
        }
        const float inverse = total == 0.f ? 0.f : 1.f / total;
        const uint64_t row = static_cast<uint64_t>(t) * a.heads + head0 + h;
        T* out = static_cast<T*>(a.out) + row * kValue + element;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_pair<T>(y[0] * inverse, y[1] * inverse), pack_pair<T>(y[2] * inverse, y[3] * inverse));
        *reinterpret_cast<uint2*>(out + 128) = make_uint2(pack_pair<T>(y[4] * inverse, y[5] * inverse), pack_pair<T>(y[6] * inverse, y[7] * inverse));
        if (!(item & 1u) && lane == 0) a.lse[row] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
      }
    }
    cluster_barrier();                       // nobody leaves while its share is being read
  }

  // ---- teardown ----------------------------------------------------------------------------
  __syncthreads();
  if (c.abort_flag) {
    if (tid == 0) atomicOr(a.status, static_cast<int32_t>(KVIP_ERR_PIPELINE));
    for (int i = 0; i < 64; ++i) __nanosleep(2000);   // copies and products in flight end before their memory is released
    __syncthreads();
  }
  if (warp == kScoreWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* symbol = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &symbol, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      symbol = nullptr;
    return reinterpret_cast<EncodeTiledFn>(symbol);
  }();
  return fn;
}
// Queries [tokens, heads, 576] of two-byte elements, boxes of 64 elements x box_heads in 128-byte swizzle; strides in elements.
bool encode_queries(CUtensorMap* map, bool bf16, const void* base, uint64_t heads, uint64_t tokens, int64_t head, int64_t token, uint32_t box_heads) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t sizes[3] = {kWidth, heads, tokens};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2u, static_cast<cuuint64_t>(token) * 2u};
  const cuuint32_t box[3] = {64, box_heads, 1}, step[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), sizes, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, uint32_t kN>
uint32_t configure(cudaLaunchConfig_t& config, cudaLaunchAttribute& cluster, KernelSlot slot, dim3 ctas, uint32_t splits, cudaStream_t stream) {
  if (uint32_t bad = raise_dynamic_smem(slot, reinterpret_cast<const void*>(attend_tiles<T, kN>), static_cast<int>(Layout<kN>::kBytes),
                                        "slot_attention attribute"))
    return bad;
  config = cudaLaunchConfig_t{};
  config.gridDim = ctas;
  config.blockDim = dim3(Warps<kN>::kThreads);
  config.dynamicSmemBytes = Layout<kN>::kBytes;
  config.stream = stream;
  cluster = cudaLaunchAttribute{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = splits;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  return 0;
}

struct Cut { uint32_t groups, group_heads, splits; uint64_t clocks; };

template <typename T, uint32_t kN>
uint32_t launch_tiles(const KvipAttentionArgs& a, KernelSlot slot, const Cut& cut, uint32_t from, uint32_t to, cudaStream_t stream) {
  const bool bf16 = __is_same(T, __nv_bfloat16);
  CUtensorMap query_map;
  // strides of a dimension of size one do not matter, but the encoder looks at them
  const int64_t head = a.heads > 1 ? a.query_head : kWidth, token = a.tokens > 1 ? a.query_token : a.heads * kWidth;
  if (!encode_queries(&query_map, bf16, a.query, a.heads, a.tokens, head, token, kN)) {
    set_error("slot_attention: the strides do not fit a tensor map");
    return KVIP_BAD_ARGUMENT;
  }
  // tokens in y and z, shares as a power of two: the kernel finds its place without a division (one token 14.1 -> 13.8 us)
  const uint32_t tokens = to - from, y = tokens < 32768u ? tokens : 32768u, splits_log = cut.splits == 8u ? 3u : cut.splits / 2u;
  cudaLaunchConfig_t config;
  cudaLaunchAttribute cluster;
  if (uint32_t bad = configure<T, kN>(config, cluster, slot, dim3(cut.groups * cut.splits, y, (tokens + y - 1u) / y), cut.splits, stream)) return bad;
  cudaLaunchKernelEx(&config, attend_tiles<T, kN>, query_map, a, cut.group_heads, splits_log, from, to);
  count_launch();
  return check_launch("attend_tiles");
}

// Clusters of `splits` CTAs that run at once on the current device (one CTA per SM; a cluster stays within a part of the GPU, so
// large ones leave SMs idle). Asked once per device.
uint32_t resident_clusters(uint32_t splits) {
  static std::atomic<uint32_t> known[64][4];
  const uint32_t at = splits == 1u ? 0u : splits == 2u ? 1u : splits == 4u ? 2u : 3u;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) device = -1;
  if (device >= 0) {
    const uint32_t n = known[device][at].load(std::memory_order_relaxed);
    if (n) return n;
  }
  cudaLaunchConfig_t config;
  cudaLaunchAttribute cluster;
  int n = 0;
  if (configure<__nv_bfloat16, 64>(config, cluster, static_cast<KernelSlot>(kSlotAttentionBf16 + 3), dim3(splits), splits, nullptr) ||
      cudaOccupancyMaxActiveClusters(&n, attend_tiles<__nv_bfloat16, 64>, &config) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return device_sm_count() * 3u / (4u * splits) + 1u;
  }
  if (device >= 0) known[device][at].store(static_cast<uint32_t>(n), std::memory_order_relaxed);
  return static_cast<uint32_t>(n);
}

// How a call is cut: heads per CTA (all up to 64, or fewer, which read the rows more often) and CTAs that share the rows of a
// token. Few tokens are cut finely, because the SMs would stand idle; each cut costs the rows' copies once more or the joining of
// the shares. Counted in clocks of full lists: a tile of 64 rows takes 2350 + 7 per head, a CTA 12700 + 228 per head before its
// first and behind its last tile (fitted to an earlier form of the kernel; the order still holds: 1 token x 128 heads x 2048 slots in
// 16 heads x 8 CTAs 14.2 us, 16 x 4 18.5, 16 x 2 28.8, 32 x 8 15.7, 64 x 8 20.6; 16 tokens 64 x 4 27.3 against 64 x 2 40.2; 64 tokens 64 x 1
// 65.0 against 64 x 2 84.6).
uint64_t clocks_of(uint32_t tiles, uint32_t group_heads, uint32_t splits) {
  return static_cast<uint64_t>((tiles + splits - 1) / splits) * (2350u + 7u * group_heads) + 12700u + 228u * group_heads;
}
Cut cut_of(const KvipAttentionArgs& a, uint32_t tokens, uint32_t tiles) {
  Cut best{0, 0, 0, ~0ull};
  for (uint32_t width = kGroupHeads; width >= 16; width /= 2) {
    const uint32_t groups = (a.heads + width - 1) / width, group_heads = (a.heads + groups - 1) / groups;
    if (width < kGroupHeads && groups == (a.heads + 2 * width - 1) / (2 * width)) continue;   // the wider cut again
    const uint64_t units = static_cast<uint64_t>(tokens) * groups;
    for (uint32_t splits = 1; splits <= kMaxSplits; splits *= 2) {
      if (a.splits ? a.splits != splits : splits > 1 && splits > tiles) continue;
      const uint64_t waves = (units + resident_clusters(splits) - 1) / resident_clusters(splits);
      const uint64_t clocks = waves * clocks_of(tiles, group_heads, splits);
      if (clocks < best.clocks) best = {groups, group_heads, splits, clocks};
    }
  }
  return best;
}

template <typename T>
uint32_t launch_part(const KvipAttentionArgs& a, uint32_t first_slot, const Cut& cut, uint32_t from, uint32_t to, cudaStream_t stream) {
  const KernelSlot slot = static_cast<KernelSlot>(first_slot + (cut.group_heads + 15u) / 16u - 1u);
  if (cut.group_heads <= 16) return launch_tiles<T, 16>(a, slot, cut, from, to, stream);
  if (cut.group_heads <= 32) return launch_tiles<T, 32>(a, slot, cut, from, to, stream);
  if (cut.group_heads <= 48) return launch_tiles<T, 48>(a, slot, cut, from, to, stream);
  return launch_tiles<T, 64>(a, slot, cut, from, to, stream);
}

// Tokens that fill the SMs a whole number of times go as they are; what is left behind them is a call of few tokens and is cut like
// one, in a launch of its own, where that is shorter by more than a launch (2048 slots: 76 tokens x 128
// heads 123 -> 84 us, 100 tokens 125 -> 108, 160 tokens 186 -> 155, 150 x 64 heads 129 -> 89, 160 x 16 heads 103 -> 82).
constexpr uint64_t kLaunchClocks = 5000;
template <typename T>
uint32_t launch_attention(const KvipAttentionArgs& a, uint32_t first_slot, cudaStream_t stream) {
  if (a.tokens > (1u << 30)) { set_error("slot_attention: too many tokens in one call"); return KVIP_BAD_ARGUMENT; }
  const uint32_t tiles = (a.entries + kTile - 1) / kTile + (a.draft ? 1u : 0u);
  const Cut whole = cut_of(a, a.tokens, tiles);
  const uint32_t groups = (a.heads + kGroupHeads - 1) / kGroupHeads, group_heads = (a.heads + groups - 1) / groups;
  const uint32_t wave = resident_clusters(1) / groups, rest = wave ? a.tokens % wave : 0u;
  if (!a.splits && rest && rest < a.tokens) {
    const Cut full{groups, group_heads, 1, a.tokens / wave * clocks_of(tiles, group_heads, 1)}, tail = cut_of(a, rest, tiles);
    if (full.clocks + tail.clocks + kLaunchClocks < whole.clocks) {
      if (uint32_t bad = launch_part<T>(a, first_slot, full, 0, a.tokens - rest, stream)) return bad;
      return launch_part<T>(a, first_slot, tail, a.tokens - rest, a.tokens, stream);
    }
  }
  return launch_part<T>(a, first_slot, whole, 0, a.tokens, stream);
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_b200_slot_attention(const KvipAttentionArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->query && a->pool && a->slots && a->out && a->lse && a->status, "slot_attention: null pointer");
  KVIP_REQUIRE(a->tokens >= 1 && a->heads >= 1 && a->heads <= 128 && a->entries >= 1 && a->entries <= (1u << 20),
               "slot_attention: tokens, 1..128 heads, 1..2^20 entries");
  KVIP_REQUIRE(a->batch >= 1 && (a->requests || (a->queries >= 1 && static_cast<uint64_t>(a->batch) * a->queries >= a->tokens)),
               "slot_attention: requests of the tokens");
  KVIP_REQUIRE(a->output_stride >= 1 && a->output_stride <= a->pool_rows && a->pool_rows <= 0x7fffffffull, "slot_attention: pool geometry");
  KVIP_REQUIRE(!a->draft || a->starts, "slot_attention: drafted rows need the requests' starts");
  KVIP_REQUIRE(a->dtype <= KVIP_FLOAT_FP16, "slot_attention: bf16 or fp16");
  KVIP_REQUIRE(((reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->pool) | reinterpret_cast<uintptr_t>(a->out) |
                 reinterpret_cast<uintptr_t>(a->draft)) & 15u) == 0 && ((a->query_token | a->query_head | a->draft_token) & 7) == 0,
               "slot_attention: 16-byte aligned rows");
  KVIP_REQUIRE(a->splits <= kMaxSplits && (a->splits & (a->splits - 1u)) == 0, "slot_attention: 0, 1, 2, 4 or 8 shares");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == KVIP_FLOAT_BF16 ? launch_attention<__nv_bfloat16>(*a, kSlotAttentionBf16, s) : launch_attention<__half>(*a, kSlotAttentionFp16, s);
}
