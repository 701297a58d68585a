// Attention of packed query tokens over selected pool rows and drafted rows (include/kvip_b200.h: KvipAttentionArgs).
//
// One warp per (token, head), one pass over the token's rows with the running maximum and sum of the softmax. A lane
// holds 18 query elements (16 of the value part, 2 of the rest) and 16 accumulators.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kWidth = KVIP_ATTENTION_WIDTH, kValue = KVIP_ATTENTION_VALUE;

__device__ __forceinline__ float2 pair_to_float(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ uint32_t pair_from_float(float x, float y, __nv_bfloat16) {
  __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair_from_float(float x, float y, __half) {
  __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T>
__global__ void __launch_bounds__(128) attend_rows(const KvipAttentionArgs a) {
  const uint32_t lane = threadIdx.x & 31u, t = blockIdx.x, h = blockIdx.y * 4u + (threadIdx.x >> 5);
  if (h >= a.heads) return;
  const int32_t request = a.requests ? a.requests[t] : static_cast<int32_t>(t / a.queries);
  if (request < 0) return;
  int32_t bad = 0;
  uint64_t base = 0;
  uint32_t drafted = 0, limit = a.output_stride;
  int64_t first = 0;
  uint64_t seen = 0;
  if (static_cast<uint32_t>(request) >= a.batch) {
    bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
    limit = 0;
  } else {
    const int32_t owner = a.row_owners ? a.row_owners[request] : request;
    base = static_cast<uint64_t>(static_cast<uint32_t>(owner)) * a.output_stride;
    if (owner < 0 || base + a.output_stride > a.pool_rows) { bad = static_cast<int32_t>(KVIP_ERR_SOURCE); limit = 0; }
    if (a.draft) {
      first = a.starts[request];
      const int64_t behind = a.starts[request + 1];
      if (first < 0 || behind < first || behind > static_cast<int64_t>(a.tokens)) bad |= static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
      else drafted = static_cast<uint32_t>(min(static_cast<int64_t>(64), behind - first));
      const int64_t own = static_cast<int64_t>(t) - first;
      seen = a.ancestors ? static_cast<uint64_t>(a.ancestors[t])
                         : (own < 0 ? 0ull : own >= 63 ? ~0ull : (2ull << own) - 1ull);
    }
  }
  const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.query) + t * a.query_token + h * a.query_head);
  float2 qv[9], acc[8];
#pragma unroll
  for (uint32_t i = 0; i < 9; ++i) {
    qv[i] = pair_to_float(q[i * 32u + lane], T());
    qv[i].x *= a.scale; qv[i].y *= a.scale;
  }
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) acc[i] = make_float2(0.f, 0.f);
  float top = -INFINITY, total = 0.f;
  const int32_t* list = a.slots + static_cast<uint64_t>(t) * a.entries;
  for (uint32_t k = 0; k < a.entries + drafted; ++k) {
    const T* row;
    if (k < a.entries) {
      const int32_t slot = list[k];
      if (slot < 0) continue;
      if (static_cast<uint32_t>(slot) >= limit) { bad |= static_cast<int32_t>(KVIP_ERR_SOURCE); continue; }
      row = static_cast<const T*>(a.pool) + (base + static_cast<uint32_t>(slot)) * kWidth;
    } else {
      const uint32_t j = k - a.entries;
      if (!((seen >> j) & 1ull)) continue;
      row = static_cast<const T*>(a.draft) + (first + j) * a.draft_token;
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(row);
    float2 v[9];
    float dot = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < 9; ++i) {
      v[i] = pair_to_float(w[i * 32u + lane], T());
      dot = fmaf(qv[i].x, v[i].x, dot);
      dot = fmaf(qv[i].y, v[i].y, dot);
    }
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float next = fmaxf(top, dot);
    const float shrink = expf(top - next), p = expf(dot - next);
    top = next;
    total = total * shrink + p;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      acc[i].x = acc[i].x * shrink + p * v[i].x;
      acc[i].y = acc[i].y * shrink + p * v[i].y;
    }
  }
  const uint64_t out_row = static_cast<uint64_t>(t) * a.heads + h;
  uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + out_row * kValue);
  const float inverse = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) out[i * 32u + lane] = pair_from_float(acc[i].x * inverse, acc[i].y * inverse, T());
  if (lane == 0) {
    a.lse[out_row] = total == 0.f ? -INFINITY : top + logf(total);
    if (bad) atomicOr(a.status, bad);
  }
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_b200_slot_attention(const KvipAttentionArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->query && a->pool && a->slots && a->out && a->lse && a->status, "slot_attention: null pointer");
  KVIP_REQUIRE(a->tokens >= 1 && a->heads >= 1 && a->heads <= 128 && a->entries >= 1, "slot_attention: tokens, 1..128 heads, entries");
  KVIP_REQUIRE(a->batch >= 1 && (a->requests || (a->queries >= 1 && static_cast<uint64_t>(a->batch) * a->queries >= a->tokens)),
               "slot_attention: requests of the tokens");
  KVIP_REQUIRE(a->output_stride >= 1 && a->output_stride <= a->pool_rows, "slot_attention: pool geometry");
  KVIP_REQUIRE(!a->draft || a->starts, "slot_attention: drafted rows need the requests' starts");
  KVIP_REQUIRE(a->dtype <= KVIP_FLOAT_FP16, "slot_attention: bf16 or fp16");
  KVIP_REQUIRE(((reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->pool) | reinterpret_cast<uintptr_t>(a->out) |
                 reinterpret_cast<uintptr_t>(a->draft)) & 15u) == 0 && ((a->query_token | a->query_head | a->draft_token) & 7) == 0,
               "slot_attention: 16-byte aligned rows");
  KVIP_REQUIRE(a->splits <= 1 || (a->partial && a->partial_stats &&
                                  static_cast<uint64_t>(a->splits) * a->tokens * a->heads <= a->partial_rows),
               "slot_attention: the workspace does not hold the shares");
  const dim3 grid(a->tokens, (a->heads + 3u) / 4u);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == KVIP_FLOAT_BF16) attend_rows<__nv_bfloat16><<<grid, 128, 0, s>>>(*a);
  else attend_rows<__half><<<grid, 128, 0, s>>>(*a);
  count_launch();
  return check_launch("attend_rows");
}
