// Verification of drafted tokens (include/kvip_b200.h: KvipVerifyArgs).
//
// A request's walk down its tree needs single probabilities (gathered up front, all nodes at once), and a pass over the
// vocabulary only where a drafted token is rejected or the walk ends: the sum of what is left, and then the place where
// the running sum passes sample * sum. One CTA per request in this form; sums are fp64 and their order is fixed.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr uint32_t kMaxNodes = 64;

template <typename T> __device__ __forceinline__ double probability(T v);
template <> __device__ __forceinline__ double probability(float v) { return v > 0.f ? static_cast<double>(v) : 0.0; }
template <> __device__ __forceinline__ double probability(__nv_bfloat16 v) { return probability(__bfloat162float(v)); }
template <> __device__ __forceinline__ double probability(__half v) { return probability(__half2float(v)); }

// What is left of probability p after the rejections so far: r = max(r - Z_i q, 0) for each of them.
__device__ __forceinline__ double remaining(double p, double q, const double* mass, uint32_t rejected) {
  for (uint32_t i = 0; i < rejected; ++i) p = fmax(__dsub_rn(p, __dmul_rn(mass[i], q)), 0.0);
  return p;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_walk(const KvipVerifyArgs a) {
  __shared__ double s_p[kMaxNodes], s_q[kMaxNodes], s_mass[kMaxNodes + 1], s_part[kVerifyWarps];
  __shared__ int64_t s_token[kMaxNodes], s_lost[kMaxNodes];
  __shared__ int32_t s_parent[kMaxNodes];
  __shared__ float s_accept[kMaxNodes];
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  int64_t* out_tokens = a.out_tokens + static_cast<uint64_t>(b) * (a.depth + 1u);
  int32_t* out_nodes = a.out_nodes + static_cast<uint64_t>(b) * (a.depth + 1u);
  const int64_t first = a.starts[b], behind = a.starts[b + 1];
  uint32_t n = 0;
  int32_t bad = 0;
  if (first >= 0 && behind >= first && behind <= static_cast<int64_t>(a.rows)) n = static_cast<uint32_t>(behind - first);
  else bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
  if (n > kMaxNodes) { n = kMaxNodes; bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE); }
  for (uint32_t i = tid; i <= a.depth; i += kVerifyThreads) { out_tokens[i] = -1; out_nodes[i] = -1; }
  if (n == 0) {
    if (tid == 0) {
      a.out_counts[b] = 0;
      if (bad) atomicOr(a.status, bad);
    }
    return;
  }
  const T* target = static_cast<const T*>(a.target) + first * a.target_row;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + first * a.draft_row : nullptr;
  if (tid < n) {
    int64_t token = a.tokens[first + tid];
    int32_t parent = tid ? a.parents[first + tid] : -1;
    s_accept[tid] = a.accept[first + tid];
    if (tid && (token < 0 || token >= static_cast<int64_t>(a.vocabulary) || parent < 0 || parent >= static_cast<int32_t>(tid))) {
      parent = -1;   // never reached
      token = 0;
      bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
    }
    s_token[tid] = token;
    s_parent[tid] = parent;
    if (parent >= 0) {
      s_p[tid] = probability(target[parent * a.target_row + token]);
      s_q[tid] = draft ? probability(draft[parent * a.draft_row + token]) : 1.0;
    }
  }
  bad = __syncthreads_or(bad);

  // the vocabulary in contiguous shares, one per warp
  const uint32_t V = a.vocabulary;
  const uint32_t share = ((V + kVerifyWarps - 1) / kVerifyWarps + 31u) & ~31u;
  const uint32_t from = min(V, warp * share), to = min(V, from + share);
  uint32_t node = 0, length = 0, rejected = 0;
  bool summed = false;
  auto left_at = [&](uint32_t v) -> double {
    const double p = probability(target[node * a.target_row + v]);
    if (!rejected) return p;
    if (draft) return remaining(p, probability(draft[node * a.draft_row + v]), s_mass, rejected);
    for (uint32_t i = 0; i < rejected; ++i)
      if (s_lost[i] == static_cast<int64_t>(v)) return 0.0;
    return p;
  };
  auto sum_all = [&]() -> double {
    double sum = 0.0;
    for (uint32_t v = from + lane; v < to; v += 32u) sum += left_at(v);
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) s_part[warp] = sum;
    __syncthreads();
    double total = 0.0;
    for (uint32_t w = 0; w < kVerifyWarps; ++w) total += s_part[w];
    return total;
  };
  double total = 0.0;
  for (uint32_t j = 1; j < n && length < a.depth; ++j) {
    if (s_parent[j] != static_cast<int32_t>(node)) continue;
    const double mass = rejected ? s_mass[rejected] : 1.0;
    double r = s_p[j];
    if (draft) {
      r = remaining(r, s_q[j], s_mass, rejected);
    } else {
      for (uint32_t i = 0; i < rejected; ++i)
        if (s_lost[i] == s_token[j]) r = 0.0;
    }
    if (__dmul_rn(__dmul_rn(static_cast<double>(s_accept[j]), s_q[j]), mass) < r) {
      if (tid == 0) { out_tokens[length] = s_token[j]; out_nodes[length + 1] = static_cast<int32_t>(j); }
      node = j;
      ++length;
      rejected = 0;
      summed = false;
    } else {
      __syncthreads();
      if (tid == 0) { s_mass[0] = 1.0; s_lost[rejected] = s_token[j]; }
      __syncthreads();
      ++rejected;
      total = sum_all();
      summed = true;
      if (tid == 0) s_mass[rejected] = total;
      __syncthreads();
      if (total == 0.0) { rejected = 0; summed = false; break; }
    }
  }
  if (!summed) total = sum_all();
  // the first share whose running sum passes the limit; where rounding leaves none, the last one that holds anything
  const double limit = __dmul_rn(static_cast<double>(a.sample[b]), total);
  double running = 0.0, base = 0.0;
  uint32_t chosen = 0;
  for (uint32_t w = 0; w < kVerifyWarps; ++w) {
    if (s_part[w] > 0.0) { chosen = w; base = running; }
    running += s_part[w];
    if (running > limit) break;
  }
  if (warp == chosen) {
    double before = base;
    uint32_t picked = 0;
    bool found = false;
    for (uint32_t v0 = from; v0 < to; v0 += 32u) {
      const uint32_t v = v0 + lane;
      const double mine = v < to ? left_at(v) : 0.0;
      double scan = mine;
#pragma unroll
      for (uint32_t d = 1; d < 32u; d <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += other;
      }
      const uint32_t holds = __ballot_sync(0xffffffffu, mine > 0.0);
      const uint32_t passed = __ballot_sync(0xffffffffu, mine > 0.0 && before + scan > limit);
      if (passed) { picked = v0 + static_cast<uint32_t>(__ffs(static_cast<int>(passed))) - 1u; found = true; break; }
      if (holds) picked = v0 + 31u - static_cast<uint32_t>(__clz(static_cast<int>(holds)));
      before += __shfl_sync(0xffffffffu, scan, 31);
    }
    (void)found;
    if (lane == 0) {
      out_tokens[length] = picked;
      out_nodes[0] = 0;
      a.out_counts[b] = static_cast<int32_t>(length + 1u);
      if (bad) atomicOr(a.status, bad);
    }
  }
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_b200_verify_drafts(const KvipVerifyArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->target && a->tokens && a->parents && a->starts && a->accept && a->sample && a->out_tokens &&
                   a->out_nodes && a->out_counts && a->status, "verify_drafts: null pointer");
  KVIP_REQUIRE(a->rows >= 1 && a->rows <= 0x7fffffffu, "verify_drafts: at least one row");
  KVIP_REQUIRE(a->vocabulary >= 1 && a->vocabulary <= (1u << 24), "verify_drafts: a vocabulary of 1..2^24 tokens");
  KVIP_REQUIRE(a->batch >= 1 && a->batch <= 65536u, "verify_drafts: 1..65536 requests");
  KVIP_REQUIRE(a->depth >= 1 && a->depth < kMaxNodes, "verify_drafts: a depth of 1..63");
  KVIP_REQUIRE(a->dtype <= KVIP_FLOAT_FP32, "verify_drafts: unknown type");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == KVIP_FLOAT_BF16) verify_walk<__nv_bfloat16><<<a->batch, kVerifyThreads, 0, s>>>(*a);
  else if (a->dtype == KVIP_FLOAT_FP16) verify_walk<__half><<<a->batch, kVerifyThreads, 0, s>>>(*a);
  else verify_walk<float><<<a->batch, kVerifyThreads, 0, s>>>(*a);
  count_launch();
  return check_launch("verify_walk");
}
