// Verification of drafted tokens (include/kvip_b200.h: KvipVerifyArgs).
//
// A request's walk down its tree needs single probabilities (gathered up front, all nodes at once), and a pass over the
// vocabulary only where a drafted token is rejected or the walk ends: the sum of what is left, and then the place where
// the running sum passes sample * sum. A cluster of CTAs takes one request. Every CTA makes the whole walk from the same
// numbers, so all of them take the same turns; a pass is split over the warps of the cluster in contiguous shares, whose sums
// go to every CTA through distributed shared memory, and the warp whose share holds the border looks for it. Sums are fp64; how a row is
// shared out goes by the batch, which moves a border by the roundings of fp64 and no more. The rejections at one node need no pass of their
// own over each other's results: where r - Z q is not cut off, r = max(target - C draft, 0) with C = 1 + Z_1 + .. + Z_(k-1), and what was cut
// off stays below. So a pass costs one fp64 fma, one add and two conversions per element, however many rejections, beside shifting rows of odd
// length into place. Measured: 64 chains of 4 over 131072 tokens in fp32 18.9 us (67 MB; HBM 31 % of its peak, the rest is the latency before and
// behind the pass), one request 9.7 us (latency), 48 trees of up to 16 nodes over 100003 bf16 tokens 31.7 us (ALU pipe of the busiest SM 94 %, its
// conversions 54 %: the walk with the most rejections).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kMostThreads = 1024, kMostWarps = kMostThreads / 32;
constexpr uint32_t kMaxNodes = 64;

// A probability as it counts: what is negative or NaN is nothing.
template <typename T> __device__ __forceinline__ float clean(T v);
template <> __device__ __forceinline__ float clean(float v) { return fmaxf(v, 0.f); }
template <> __device__ __forceinline__ float clean(__nv_bfloat16 v) { return fmaxf(__bfloat162float(v), 0.f); }
template <> __device__ __forceinline__ float clean(__half v) { return fmaxf(__half2float(v), 0.f); }
template <typename T> __device__ __forceinline__ double probability(T v) { return static_cast<double>(clean(v)); }

// What is left of probability p where the masses taken so far sum up to `taken`: max(p - taken q, 0).
__device__ __forceinline__ double remaining(double p, double q, double taken) {
  const double d = __fma_rn(-taken, q, p);
  return __double2hiint(d) < 0 ? 0.0 : d;   // the sign by the integer units: the fp64 ones are the scarce ones
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

constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kRunsInARow = 4;        // of a lane, where one warp looks through a share

// A lane takes the probabilities of one 16-byte run at a time. A row of odd length starts anywhere: the two aligned vectors
// round the run are read and shifted. A vector is read only where it holds an element of the run (memory is allocated in whole
// vectors); `off` is the same for a whole row.
template <typename T> struct Run {
  static constexpr uint32_t kCount = 16u / sizeof(T);
  uint4 low, high;
};
template <typename T, bool kAligned> __device__ __forceinline__ Run<T> load_run(const T* row, uint32_t count) {
  Run<T> r;
  r.low = r.high = make_uint4(0u, 0u, 0u, 0u);
  const uint32_t off = kAligned ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u;
  const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) - off);
  if (count) r.low = __ldg(from);
  if (!kAligned && off + count * sizeof(T) > 16u) r.high = __ldg(from + 1);
  return r;
}
// The run's first word into place, zeros behind its elements: nothing stays nothing, whatever is taken from it.
template <typename T, bool kAligned> __device__ __forceinline__ void settle_run(Run<T>& r, uint32_t off, uint32_t count) {
  uint32_t w[8] = {r.low.x, r.low.y, r.low.z, r.low.w, r.high.x, r.high.y, r.high.z, r.high.w};
  if (!kAligned) {
    if (off & 8u) {
#pragma unroll
      for (uint32_t i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4u) {
#pragma unroll
      for (uint32_t i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (off & 2u) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
  }
  if (count < Run<T>::kCount) {            // the last run of the vocabulary
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t bytes = count * sizeof(T);
      w[i] = bytes >= 4u * i + 4u ? w[i] : bytes > 4u * i ? w[i] & 0xffffu : 0u;
    }
  }
  r.low = make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ float value_of(const Run<T>& r, uint32_t k) { return clean(reinterpret_cast<const T*>(&r.low)[k]); }

// What a pass has to take from the target's row.
struct Losses {
  double taken;            // drafted: sum of the masses, 0 where nothing was rejected
  const int64_t* lost;     // else the rejected tokens
  uint32_t rejected;
  bool drafted;
};
// What is left of a run at v.
template <typename T> __device__ __forceinline__ void left_of_run(const Run<T>& rp, const Run<T>& rq, uint32_t v, const Losses& l, double (&r)[Run<T>::kCount]) {
  constexpr uint32_t kRun = Run<T>::kCount;
#pragma unroll
  for (uint32_t k = 0; k < kRun; ++k) r[k] = static_cast<double>(value_of(rp, k));
  if (l.drafted) {
#pragma unroll
    for (uint32_t k = 0; k < kRun; ++k) r[k] = remaining(r[k], static_cast<double>(value_of(rq, k)), l.taken);
    return;
  }
  for (uint32_t i = 0; i < l.rejected; ++i) {
    const int64_t at = l.lost[i] - static_cast<int64_t>(v);
#pragma unroll
    for (uint32_t k = 0; k < kRun; ++k)
      if (at == static_cast<int64_t>(k)) r[k] = 0.0;
  }
}
// This lane's part of the sum between `from` and `to`; kMode 0: nothing rejected, 1: by a draft row, 2: certain tokens.
// kAtOnce runs are on their way at a time.
template <typename T, bool kAligned, uint32_t kMode>
__device__ __forceinline__ double sum_runs(const T* row, const T* guess, uint32_t from, uint32_t to, const Losses& l) {
  constexpr uint32_t kRun = Run<T>::kCount, kAtOnce = kMode == 2u ? 1u : kAligned && kRun == 4u ? 4u : 2u;
  const uint32_t off_p = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u, off_q = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(guess)) & 15u;
  double sums[2] = {0.0, 0.0};
  for (uint32_t v0 = from + (threadIdx.x & 31u) * kRun; v0 < to; v0 += 32u * kRun * kAtOnce) {
    Run<T> rp[kAtOnce], rq[kAtOnce];
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t v = v0 + u * 32u * kRun, count = v < to ? min(kRun, to - v) : 0u;
      rp[u] = load_run<T, kAligned>(row + v, count);
      if (kMode == 1u) rq[u] = load_run<T, kAligned>(guess + v, count);
    }
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t v = v0 + u * 32u * kRun, count = v < to ? min(kRun, to - v) : 0u;
      settle_run<T, kAligned>(rp[u], off_p, count);
      if constexpr (kMode == 0u) {
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k) sums[k & 1u] += static_cast<double>(value_of(rp[u], k));
      } else if constexpr (kMode == 1u) {
        settle_run<T, kAligned>(rq[u], off_q, count);
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k)
          sums[k & 1u] += remaining(static_cast<double>(value_of(rp[u], k)), static_cast<double>(value_of(rq[u], k)), l.taken);
      } else {
        double r[kRun];
        left_of_run<T>(rp[u], rp[u], v, l, r);
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k) sums[k & 1u] += r[k];
      }
    }
  }
  double sum = sums[0] + sums[1];
#pragma unroll
  for (uint32_t o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
template <typename T, bool kAligned>
__device__ __forceinline__ double sum_mode(const T* row, const T* guess, uint32_t from, uint32_t to, const Losses& l) {
  if (l.rejected == 0u) return sum_runs<T, kAligned, 0u>(row, row, from, to, l);
  if (l.drafted) return sum_runs<T, kAligned, 1u>(row, guess, from, to, l);
  return sum_runs<T, kAligned, 2u>(row, guess, from, to, l);
}
template <typename T> __device__ __forceinline__ double sum_between(const T* row, const T* guess, uint32_t from, uint32_t to, const Losses l) {
  return ((reinterpret_cast<uintptr_t>(row) | reinterpret_cast<uintptr_t>(guess)) & 15u) == 0 ? sum_mode<T, true>(row, guess, from, to, l)
                                                                                            : sum_mode<T, false>(row, guess, from, to, l);
}
// Of `count` sums in order, the first one whose running sum, from `running` on, passes the limit; where rounding leaves none,
// the last one that holds anything. `running` becomes the sum before it. A lane takes `each` sums in a row; sum k lies at
// place_of(k, each), where the lanes' reads meet no bank twice.
__device__ __forceinline__ uint32_t place_of(uint32_t k, uint32_t each) { return (k % each) * 32u + k / each; }
struct Place { double running; uint32_t chosen; };
__device__ __forceinline__ Place passing(const double* sums, uint32_t count, double limit, double running) {
  const uint32_t lane = threadIdx.x & 31u, each = (count + 31u) / 32u, first = lane * each;
  double own = 0.0;
  for (uint32_t i = 0; i < each; ++i) own += first + i < count ? sums[i * 32u + lane] : 0.0;
  double scan = own;
#pragma unroll
  for (uint32_t d = 1; d < 32u; d <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += other;
  }
  const uint32_t holds = __ballot_sync(0xffffffffu, own > 0.0), passed = __ballot_sync(0xffffffffu, own > 0.0 && running + scan > limit);
  const uint32_t pick = passed ? static_cast<uint32_t>(__ffs(static_cast<int>(passed))) - 1u : holds ? 31u - static_cast<uint32_t>(__clz(static_cast<int>(holds))) : 0u;
  Place at{running + (scan - own), first};   // this lane's, should it be the one
  double before = at.running;
  for (uint32_t i = 0; i < each; ++i) {
    const double x = first + i < count ? sums[i * 32u + lane] : 0.0;
    if (x > 0.0) { at.running = before; at.chosen = first + i; }
    before += x;
    if (x > 0.0 && before > limit) break;
  }
  at.running = __shfl_sync(0xffffffffu, at.running, pick);
  at.chosen = __shfl_sync(0xffffffffu, at.chosen, pick);
  return at;
}

template <typename T>
__global__ void __launch_bounds__(kMostThreads, 1) verify_walk(const __grid_constant__ KvipVerifyArgs a) {
  __shared__ double s_p[kMaxNodes], s_q[kMaxNodes], s_part[2][kMaxCluster * kMostWarps];
  __shared__ int64_t s_token[kMaxNodes], s_lost[kMaxNodes];
  __shared__ int32_t s_parent[kMaxNodes];
  __shared__ float s_accept[kMaxNodes];
  __shared__ Place s_border;
  const uint32_t rank = cluster_rank(), ctas = cluster_size();
  const uint32_t b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  int64_t* out_tokens = a.out_tokens + static_cast<uint64_t>(b) * (a.depth + 1u);
  int32_t* out_nodes = a.out_nodes + static_cast<uint64_t>(b) * (a.depth + 1u);
  const int64_t first = a.starts[b], behind = a.starts[b + 1];
  const double sample = static_cast<double>(a.sample[b]);
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
  bad = __syncthreads_or(bad);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // ... and so do the others

  // the vocabulary in contiguous shares of whole runs, one per warp of the cluster
  constexpr uint32_t kRun = Run<T>::kCount;
  const uint32_t V = a.vocabulary, warps = blockDim.x >> 5, shares = ctas * warps;
  const uint32_t share = ((V + shares - 1) / shares + kRun - 1u) / kRun * kRun;
  // A node's rejected tokens lie behind those of the nodes before it: a warp that is still at an earlier test finds its own untouched.
  uint32_t node = 0, length = 0, rejected = 0, lost = 0, pass = 0;
  double mass = 1.0, taken = 0.0;          // of what is left at the node, and of all before
  auto losses = [&]() { return Losses{taken, s_lost + lost, rejected, draft != nullptr}; };
  auto part_sum = [&](uint32_t from, uint32_t to) -> double {
    const T* row = target + node * a.target_row;
    return sum_between<T>(row, draft ? draft + node * a.draft_row : row, from, to, losses());
  };
  auto sum_all = [&]() -> double {         // leaves the shares' sums in s_part[pass & 1] of every CTA
    const uint32_t mine = rank * warps + warp, from = min(V, mine * share);
    const double sum = part_sum(from, min(V, from + share));
    ++pass;
    double* part = s_part[pass & 1u];
    const uint32_t each = (shares + 31u) / 32u;
    if (lane < ctas) store_remote(&part[place_of(mine, each)], lane, sum);
    __syncwarp();
    cluster_barrier();
    double total = 0.0;
    for (uint32_t i = 0; i < each; ++i) total += lane * each + i < shares ? part[i * 32u + lane] : 0.0;
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
    double r = s_p[j];
    if (draft) {
      r = remaining(r, s_q[j], taken);
    } else {
      for (uint32_t i = 0; i < rejected; ++i)
        if (s_lost[lost + i] == s_token[j]) r = 0.0;
    }
    if (__dmul_rn(__dmul_rn(static_cast<double>(s_accept[j]), s_q[j]), mass) < r) {
      if (lane == (length & 31u)) { if (length < 32u) path = j; else path_high = j; }
      node = j;
      ++length;
      lost += rejected;
      rejected = 0;
      mass = 1.0;
      taken = 0.0;
      summed = false;
    } else {
      if (tid == 0) s_lost[lost + rejected] = s_token[j];
      __syncthreads();
      ++rejected;
      taken += mass;
      mass = total = sum_all();
      summed = true;
      if (total == 0.0) { rejected = 0; taken = 0.0; summed = false; break; }
    }
  }
  if (!summed) total = sum_all();          // nothing rejected at the last node
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
  // The share that holds the border is looked through once more: a long one by all warps of its CTA, a part each; then a lane
  // takes a few runs in a row.
  const double limit = __dmul_rn(sample, total);
  if (warp == 0) {
    const Place border = passing(s_part[pass & 1u], shares, limit, 0.0);
    if (lane == 0) { s_border.running = border.running; s_border.chosen = border.chosen; }
  }
  __syncthreads();
  double running = s_border.running;
  const uint32_t chosen = s_border.chosen;
  if (chosen - rank * warps >= warps) return;   // another CTA's
  uint32_t begin = min(V, chosen * share), end = min(V, begin + share);
  if (share > 32u * kRun * kRunsInARow) {
    const uint32_t part = ((end - begin + warps - 1u) / warps + kRun - 1u) / kRun * kRun;
    double* sums = s_part[(pass & 1u) ^ 1u];   // the other CTAs have done with it, and write to it no more
    const uint32_t from = min(end, begin + warp * part);
    const double sum = part_sum(from, min(end, from + part));
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (warp) return;
    const Place inner = passing(sums, warps, limit, running);
    running = inner.running;
    begin = min(end, begin + inner.chosen * part);
    end = min(end, begin + part);
  } else if (warp) {
    return;
  }
  const T* row = target + node * a.target_row;
  const T* guess = draft ? draft + node * a.draft_row : row;
  const uint32_t off_p = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u, off_q = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(guess)) & 15u;
  const uint32_t each = ((end - begin + 31u) / 32u + kRun - 1u) / kRun * kRun;   // elements of a lane
  const uint32_t mine = min(end, begin + lane * each), behind_mine = min(end, mine + each);
  auto runs = [&](auto&& visit) {              // this lane's runs in order
    for (uint32_t v = mine; v < behind_mine; v += kRun) {
      const uint32_t count = min(kRun, behind_mine - v);
      Run<T> rp = load_run<T, false>(row + v, count), rq = load_run<T, false>(guess + v, count);
      settle_run<T, false>(rp, off_p, count);
      settle_run<T, false>(rq, off_q, count);
      double p[kRun];
      left_of_run<T>(rp, rq, v, losses(), p);
#pragma unroll
      for (uint32_t k = 0; k < kRun; ++k) visit(v + k, p[k]);
    }
  };
  double own = 0.0;
  runs([&](uint32_t, double p) { own += p; });
  double scan = own;
#pragma unroll
  for (uint32_t d = 1; d < 32u; d <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += other;
  }
  const uint32_t passed = __ballot_sync(0xffffffffu, own > 0.0 && running + scan > limit), holds = __ballot_sync(0xffffffffu, own > 0.0);
  const uint32_t who = passed ? static_cast<uint32_t>(__ffs(static_cast<int>(passed))) - 1u : holds ? 31u - static_cast<uint32_t>(__clz(static_cast<int>(holds))) : 0u;
  if (lane == who) {                           // the first element whose running sum passes, else the last that holds anything
    double so_far = running + (scan - own);
    uint32_t picked = 0;
    bool found = false;
    runs([&](uint32_t v, double p) {
      so_far += p;
      if (p > 0.0 && !found) {
        picked = v;
        found = so_far > limit;
      }
    });
    out_tokens[length] = picked;
  }
}

template <typename T>
uint32_t launch_verify(const KvipVerifyArgs& a, cudaStream_t stream) {
  // Eight CTAs a request, of as many threads as leave all of them resident at once (a pass is a chain of latencies, and
  // requests wait for nothing but their own); fewer CTAs where the batch fills the SMs by itself.
  const uint32_t sms = device_sm_count();
  uint32_t ctas = kMaxCluster, threads = kMostThreads;
  while (ctas > 1u && a.batch * ctas > 8u * sms) ctas /= 2u;
  const uint32_t resident = (a.batch * ctas + sms - 1) / sms;   // CTAs per SM
  if (resident > 1u) threads = resident >= 4u ? 256u : kMostThreads / resident / 32u * 32u;
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
