// Rotary positions, plain and fused with the FP8 quantisation of Index rows (include/kvip_b200.h: KvipRotaryArgs).
//
// Angles: turns[i] holds frequency_i / 2 pi in fp64, so position * turns[i] is the angle in whole turns; its fractional
// part (exact subtraction in fp64) goes to sincospi in fp32. A position of 2^21 keeps 32 bits behind the point that way,
// where an fp32 angle would have none. The rotation is fp32, rounded once to the row's type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "common.cuh"

namespace kvip {
namespace {

constexpr uint32_t kRotaryThreads = 256;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float2 cos_sin(int64_t position, double turn, float factor) {
  const double turns = static_cast<double>(position) * turn;
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c * factor, s * factor);
}

// One pair per thread: every type, layout, stride and width.
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotate_pairs(const KvipRotaryArgs a) {
  const uint32_t half = a.width >> 1, rows = a.heads[0] + a.heads[1];
  const uint64_t per_token = static_cast<uint64_t>(rows) * half;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRotaryThreads + threadIdx.x; i < per_token * a.tokens;
       i += static_cast<uint64_t>(gridDim.x) * kRotaryThreads) {
    const uint32_t token = static_cast<uint32_t>(i / per_token), rest = static_cast<uint32_t>(i % per_token);
    const uint32_t row = rest / half, pair = rest % half;
    const int64_t position = a.positions[token];
    if (position < 0) continue;
    const uint32_t set = row >= a.heads[0] ? 1u : 0u;
    const int64_t head = set ? row - a.heads[0] : row;
    const T* x = static_cast<const T*>(a.x[set]) + token * a.x_token[set] + head * a.x_head[set];
    T* y = static_cast<T*>(a.y[set]) + token * a.y_token[set] + head * a.y_head[set];
    const bool split = a.layout == KVIP_ROTARY_HALF;
    const uint32_t at = split ? pair : 2u * pair, other = split ? pair + half : at + 1u;
    const float2 cs = cos_sin(position, a.turns[pair], a.factor);
    const float u = to_float(x[at]), v = to_float(x[other]);
    y[at] = from_float<T>(u * cs.x - v * cs.y);
    y[other] = from_float<T>(v * cs.x + u * cs.y);
  }
}

// One row per warp: rotate, amax, quantise. Every type, layout, stride and width.
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) quantise_rows(const KvipRotaryArgs a) {
  const uint32_t lane = threadIdx.x & 31u, half = a.width >> 1;
  const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.heads[0];
  for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * (kRotaryThreads / 32u) + (threadIdx.x >> 5); r < rows;
       r += static_cast<uint64_t>(gridDim.x) * (kRotaryThreads / 32u)) {
    const uint32_t token = static_cast<uint32_t>(r / a.heads[0]), head = static_cast<uint32_t>(r % a.heads[0]);
    const int64_t position = a.positions[token];
    if (position < 0) continue;
    const T* x = static_cast<const T*>(a.x[0]) + token * a.x_token[0] + head * a.x_head[0];
    const bool split = a.layout == KVIP_ROTARY_HALF;
    float amax = 0.f, scale = 1.f, inverse = 1.f;
    for (uint32_t pass = 0; pass < 2u; ++pass) {
      uint8_t* codes = a.codes + r * a.dim;
      auto emit = [&](uint32_t at, float value) {
        if (pass == 0) amax = fmaxf(amax, fabsf(value));
        else codes[at] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(value * inverse, __NV_SATFINITE, __NV_E4M3));
      };
      for (uint32_t pair = lane; pair < half; pair += 32u) {
        const uint32_t at = split ? pair : 2u * pair, other = split ? pair + half : at + 1u;
        const float2 cs = cos_sin(position, a.turns[pair], a.factor);
        const float u = to_float(x[at]), v = to_float(x[other]);
        emit(at, u * cs.x - v * cs.y);
        emit(other, v * cs.x + u * cs.y);
      }
      for (uint32_t at = a.width + lane; at < a.dim; at += 32u) emit(at, to_float(x[at]));
      if (pass == 0) {
#pragma unroll
        for (uint32_t o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (amax > 0.f) { scale = amax / 448.f; inverse = 1.f / scale; }
        if (lane == 0) a.scales[r] = scale;
      }
    }
  }
}

template <typename T>
uint32_t launch_rotary(const KvipRotaryArgs& a, cudaStream_t stream) {
  const uint32_t most = device_sm_count() * 16u;
  if (a.codes) {
    const uint64_t blocks = (static_cast<uint64_t>(a.tokens) * a.heads[0] + 7u) / 8u;
    quantise_rows<T><<<static_cast<uint32_t>(blocks < most ? blocks : most), kRotaryThreads, 0, stream>>>(a);
  } else {
    const uint64_t items = static_cast<uint64_t>(a.tokens) * (a.heads[0] + a.heads[1]) * (a.width / 2u);
    const uint64_t blocks = (items + kRotaryThreads - 1) / kRotaryThreads;
    rotate_pairs<T><<<static_cast<uint32_t>(blocks < most ? blocks : most), kRotaryThreads, 0, stream>>>(a);
  }
  count_launch();
  return check_launch("rotary");
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_b200_rotary(const KvipRotaryArgs* a, void* stream) {
  using namespace kvip;
  KVIP_REQUIRE(a && a->positions && a->turns && a->x[0], "rotary: null pointer");
  KVIP_REQUIRE(a->codes ? a->scales != nullptr : a->y[0] != nullptr, "rotary: null output pointer");
  KVIP_REQUIRE(a->tokens >= 1 && a->heads[0] >= 1, "rotary: at least one token and one head");
  KVIP_REQUIRE(a->width >= 2 && a->width % 2 == 0 && a->width <= 1024, "rotary: the rotated width is even and at most 1024");
  KVIP_REQUIRE(a->heads[0] <= 65536 && a->heads[1] <= 65536, "rotary: at most 65536 heads");
  KVIP_REQUIRE(!a->codes || (a->dim >= a->width && a->dim <= 4096 && !a->heads[1]), "rotary: quantised rows hold the rotated width, at most 4096 elements");
  KVIP_REQUIRE(a->codes || (a->heads[1] == 0) == (a->x[1] == nullptr), "rotary: the second set needs rows and heads");
  KVIP_REQUIRE(a->codes || a->heads[1] == 0 || a->y[1], "rotary: null output pointer");
  KVIP_REQUIRE(a->layout <= KVIP_ROTARY_INTERLEAVED && a->dtype <= KVIP_FLOAT_FP32, "rotary: unknown layout or type");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == KVIP_FLOAT_BF16) return launch_rotary<__nv_bfloat16>(*a, s);
  if (a->dtype == KVIP_FLOAT_FP16) return launch_rotary<__half>(*a, s);
  return launch_rotary<float>(*a, s);
}
