// Verification of drafted tokens (include/kvip_b200.h: KvipVerifyArgs).
//
// A request's walk down its tree needs single probabilities (gathered up front, all nodes at once), and a pass over the
// vocabulary only where a drafted token is rejected or the walk ends: the sum of what is left, and then the place where
// the running sum passes sample * sum. A cluster of CTAs takes one request. Every CTA makes the whole walk from the same
// numbers, so all of them take the same turns; a pass is split over the warps of the cluster in contiguous shares, whose sums
// go to every CTA through distributed shared memory, and the warp whose share holds the border looks for it. Sums are fp64 and
// their order is fixed. Bound by HBM: one target row (and one draft row behind a rejection) per pass.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kMostThreads = 1024, kMostWarps = kMostThreads / 32;
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores into the same place of another CTA's shared memory.
__device__ __forceinline__ void store_remote(const double* where, uint32_t rank, double value) {
  uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(where)), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(address), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(value) : "memory");
}

constexpr uint32_t kRun = 8;               // consecutive elements that a lane takes at a time
constexpr uint32_t kMaxCluster = 8;

// kRun probabilities from `row` on, zeros behind `count`. A row of odd length starts anywhere: the aligned vectors round the
// run are read and shifted. Each of them holds an element of the run, and memory is allocated in whole vectors.
template <typename T> __device__ __forceinline__ void load_run(const T* row, uint32_t count, double (&p)[kRun]) {
  if (count >= kRun) {
    constexpr uint32_t kVectors = kRun * sizeof(T) / 16u;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u;
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) - off);
    uint32_t w[4 * kVectors + 4];
#pragma unroll
    for (uint32_t i = 0; i < kVectors; ++i) {
      const uint4 x = __ldg(from + i);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
    if (off) {                             // the same for a whole row
      const uint4 x = __ldg(from + kVectors);
      w[4 * kVectors] = x.x; w[4 * kVectors + 1] = x.y; w[4 * kVectors + 2] = x.z; w[4 * kVectors + 3] = x.w;
      if (off & 8u) {
#pragma unroll
        for (uint32_t i = 0; i + 2 < 4 * kVectors + 4; ++i) w[i] = w[i + 2];
      }
      if (off & 4u) {
#pragma unroll
        for (uint32_t i = 0; i + 3 < 4 * kVectors + 4; ++i) w[i] = w[i + 1];
      }
      if (off & 2u) {
#pragma unroll
        for (uint32_t i = 0; i < 4 * kVectors; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) p[i] = probability(reinterpret_cast<const T*>(w)[i]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) p[i] = i < count ? probability(row[i]) : 0.0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kMostThreads, 1) verify_walk(const __grid_constant__ KvipVerifyArgs a) {
  __shared__ double s_p[kMaxNodes], s_q[kMaxNodes], s_mass[kMaxNodes + 1], s_part[2][kMaxCluster * kMostWarps];
  __shared__ int64_t s_token[kMaxNodes], s_lost[kMaxNodes];
  __shared__ int32_t s_parent[kMaxNodes];
  __shared__ float s_accept[kMaxNodes];
  const uint32_t rank = cluster_rank(), ctas = cluster_size();
  const uint32_t b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  int64_t* out_tokens = a.out_tokens + static_cast<uint64_t>(b) * (a.depth + 1u);
  int32_t* out_nodes = a.out_nodes + static_cast<uint64_t>(b) * (a.depth + 1u);
  const int64_t first = a.starts[b], behind = a.starts[b + 1];
  uint32_t n = 0;
  int32_t bad = 0;
  if (first >= 0 && behind >= first && behind <= static_cast<int64_t>(a.rows)) n = static_cast<uint32_t>(min(behind - first, static_cast<int64_t>(kMaxNodes + 1u)));
  else bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE);
  if (n > kMaxNodes) { n = kMaxNodes; bad = static_cast<int32_t>(KVIP_ERR_TOKEN_RANGE); }
  if (n == 0) {                            // the same for the whole cluster
    if (rank == 0) {
      for (uint32_t i = tid; i <= a.depth; i += blockDim.x) { out_tokens[i] = -1; out_nodes[i] = -1; }
      if (tid == 0) {
        a.out_counts[b] = 0;
        if (bad) atomicOr(a.status, bad);
      }
    }
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this CTA runs: its shared memory may be written
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
  if (tid == 0) s_mass[0] = 1.0;
  bad = __syncthreads_or(bad);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // ... and so do the others

  // the vocabulary in contiguous shares of whole runs, one per warp of the cluster
  const uint32_t V = a.vocabulary, warps = blockDim.x >> 5, shares = ctas * warps, mine = rank * warps + warp;
  const uint32_t share = ((V + shares - 1) / shares + kRun - 1u) / kRun * kRun;
  const uint32_t from = min(V, mine * share), to = min(V, from + share);
  uint32_t node = 0, length = 0, rejected = 0, pass = 0;
  // what is left of the probabilities v .. v + kRun - 1
  auto left_at = [&](uint32_t v, double (&p)[kRun]) {
    const uint32_t count = v < to ? to - v : 0u;
    const T* row = target + node * a.target_row + v;
    load_run(row, count, p);
    if (!rejected) return;
    if (draft) {
      double q[kRun];
      const T* guess = draft + node * a.draft_row + v;
      load_run(guess, count, q);
      for (uint32_t i = 0; i < rejected; ++i) {
        const double mass = s_mass[i];
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k) p[k] = fmax(__dsub_rn(p[k], __dmul_rn(mass, q[k])), 0.0);
      }
    } else {
      for (uint32_t i = 0; i < rejected; ++i) {
        const int64_t at = s_lost[i] - static_cast<int64_t>(v);
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k)
          if (at == static_cast<int64_t>(k)) p[k] = 0.0;
      }
    }
  };
  auto sum_all = [&]() -> double {         // leaves the shares' sums in s_part[pass & 1] of every CTA
    double sum = 0.0;
#pragma unroll 2
    for (uint32_t v = from + lane * kRun; v < to; v += 32u * kRun) {
      double p[kRun];
      left_at(v, p);
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) sum += p[k];
    }
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    ++pass;
    double* part = s_part[pass & 1u];
    if (lane < ctas) store_remote(&part[mine], lane, sum);
    cluster_barrier();
    double total = 0.0;
    for (uint32_t k = 0; k < shares; k += 32u) total += k + lane < shares ? part[k + lane] : 0.0;
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    return total;
  };
  bool summed = false;
  double total = 0.0;
  uint32_t path = 0;                       // lane `i` of warp 0 of the first CTA keeps accepted node i + 1 (two words: up to 63)
  uint32_t path_high = 0;
  for (uint32_t j = 1; j < n && length < a.depth; ++j) {
    if (s_parent[j] != static_cast<int32_t>(node)) continue;
    const double mass = s_mass[rejected];
    double r = s_p[j];
    if (draft) {
      r = remaining(r, s_q[j], s_mass, rejected);
    } else {
      for (uint32_t i = 0; i < rejected; ++i)
        if (s_lost[i] == s_token[j]) r = 0.0;
    }
    if (__dmul_rn(__dmul_rn(static_cast<double>(s_accept[j]), s_q[j]), mass) < r) {
      if (lane == (length & 31u)) { if (length < 32u) path = j; else path_high = j; }
      node = j;
      ++length;
      rejected = 0;
      summed = false;
    } else {
      if (tid == 0) s_lost[rejected] = s_token[j];
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
  if (rank == 0 && warp == 0) {            // what has been accepted; the drawn token's place is another warp's
    for (uint32_t i = lane; i <= a.depth; i += 32u) {
      const uint32_t at = i < 32u ? path : path_high;
      if (i != length) out_tokens[i] = i < length ? s_token[at] : -1;
      if (i < a.depth) out_nodes[i + 1u] = i < length ? static_cast<int32_t>(at) : -1;
    }
    if (lane == 0) {
      out_nodes[0] = 0;
      a.out_counts[b] = static_cast<int32_t>(length + 1u);
      if (bad) atomicOr(a.status, bad);
    }
  }
  // the first share whose running sum passes the limit; where rounding leaves none, the last one that holds anything
  const double limit = __dmul_rn(static_cast<double>(a.sample[b]), total);
  const double* part = s_part[pass & 1u];
  double base = 0.0, before_last = 0.0, running = 0.0;
  uint32_t chosen = 0;
  bool passed_any = false;
  for (uint32_t k = 0; k < shares && !passed_any; k += 32u) {
    const double own = k + lane < shares ? part[k + lane] : 0.0;
    double scan = own;
#pragma unroll
    for (uint32_t d = 1; d < 32u; d <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += other;
    }
    const uint32_t holds = __ballot_sync(0xffffffffu, own > 0.0);
    const uint32_t passed = __ballot_sync(0xffffffffu, own > 0.0 && running + scan > limit);
    const uint32_t pick = passed ? static_cast<uint32_t>(__ffs(static_cast<int>(passed))) - 1u : holds ? 31u - static_cast<uint32_t>(__clz(static_cast<int>(holds))) : 0u;
    if (passed || holds) {
      chosen = k + pick;
      before_last = running + __shfl_sync(0xffffffffu, scan - own, pick);
      base = before_last;
    }
    passed_any = passed != 0u;
    running += __shfl_sync(0xffffffffu, scan, 31);
  }
  if (mine == chosen) {
    double before = base;
    uint32_t picked = 0;
    for (uint32_t v0 = from; v0 < to; v0 += 32u * kRun) {
      const uint32_t v = v0 + lane * kRun;
      double p[kRun];
      left_at(v, p);
      double own = 0.0;
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) own += p[k];
      double scan = own;
#pragma unroll
      for (uint32_t d = 1; d < 32u; d <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += other;
      }
      // within the run: the first element whose running sum passes, else the last that holds anything
      double sum = before + (scan - own);
      uint32_t at = 0, last = 0;
      bool found = false;
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) {
        sum += p[k];
        if (p[k] > 0.0) {
          last = k;
          if (!found && sum > limit) { found = true; at = k; }
        }
      }
      const uint32_t passed = __ballot_sync(0xffffffffu, found), holds = __ballot_sync(0xffffffffu, own > 0.0);
      if (passed) {
        const uint32_t who = static_cast<uint32_t>(__ffs(static_cast<int>(passed))) - 1u;
        picked = v0 + who * kRun + __shfl_sync(0xffffffffu, at, who);
        break;
      }
      if (holds) {
        const uint32_t who = 31u - static_cast<uint32_t>(__clz(static_cast<int>(holds)));
        picked = v0 + who * kRun + __shfl_sync(0xffffffffu, last, who);
      }
      before += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0) out_tokens[length] = picked;
  }
}

template <typename T>
uint32_t launch_verify(const KvipVerifyArgs& a, cudaStream_t stream) {
  // Eight CTAs a request, of as many threads as leave all of them resident at once (a pass is a chain of latencies, and
  // requests wait for nothing but their own); fewer CTAs where the batch fills the SMs by itself.
  const uint32_t sms = device_sm_count();
  uint32_t ctas = kMaxCluster, threads = kMostThreads;
  while (ctas > 1u && a.batch * ctas > 8u * sms) ctas /= 2u;
  while (threads > 256u && a.batch * ctas > sms * (kMostThreads / threads)) threads /= 2u;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(a.batch * ctas);
  config.blockDim = dim3(threads);
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = ctas;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, verify_walk<T>, a);
  count_launch();
  return check_launch("verify_walk");
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
  if (a->dtype == KVIP_FLOAT_BF16) return launch_verify<__nv_bfloat16>(*a, s);
  if (a->dtype == KVIP_FLOAT_FP16) return launch_verify<__half>(*a, s);
  return launch_verify<float>(*a, s);
}
