// Rotary positions, plain and fused with the FP8 quantisation of Index rows (include/kvip_b200.h: KvipRotaryArgs).
//
// Angles: turns[i] holds frequency_i / 2 pi in fp64, so position * turns[i] is the angle in whole turns; its fractional
// part (exact subtraction in fp64) goes to sincospi in fp32. A position of 2^21 keeps 32 bits behind the point that way,
// where an fp32 angle would have none. The rotation is fp32, rounded once to the row's type.
//
// Bound by HBM: 8192 tokens x 129 rows of 64 inside rows of 576 take 50 us (5.4 TB/s), 16411 x 64 rows of 128 to FP8 87.6 us (4.65 TB/s,
// issue slots 68 % busy; 95 us where the power limit holds the clock down); one pair per thread instead of a unit of eight took 204 and 473.
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
    float amax = 0.f, scale = 1.f;
    for (uint32_t pass = 0; pass < 2u; ++pass) {
      uint8_t* codes = a.codes + r * a.dim;
      auto emit = [&](uint32_t at, float value) {
        if (pass == 0) amax = fmaxf(amax, fabsf(value));
        else codes[at] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(value / scale, __NV_SATFINITE, __NV_E4M3));
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
        scale = index_row_scale(amax);
        if (lane == 0) a.scales[r] = scale;
      }
    }
  }
}

// ---- the vector forms ----
// A unit is 16 elements of a row in two runs of 8 that make 8 pairs: elements 8 v .. and width/2 + 8 v .. of a rotated row
// in the half layout, 16 v .. in the interleaved one (and 16 elements that do not turn, behind `width` of a quantised row).
// A CTA takes `tile` tokens and a range of rows: the angles of its tokens once, into shared memory, then a thread per
// unit. Bound by memory: two (three) wide loads and stores a unit; the angles of a token serve all of its rows.
template <typename T> struct Unit;   // 16 elements as they lie in memory
template <> struct Unit<float> { float4 v[4]; };
template <> struct Unit<__nv_bfloat16> { uint4 v[2]; };
template <> struct Unit<__half> { uint4 v[2]; };

template <typename T> __device__ __forceinline__ Unit<T> load_unit(const T* low, const T* high) {
  Unit<T> u;
  if constexpr (sizeof(T) == 4) {
    u.v[0] = __ldcs(reinterpret_cast<const float4*>(low)); u.v[1] = __ldcs(reinterpret_cast<const float4*>(low) + 1);
    u.v[2] = __ldcs(reinterpret_cast<const float4*>(high)); u.v[3] = __ldcs(reinterpret_cast<const float4*>(high) + 1);
  } else {
    u.v[0] = __ldcs(reinterpret_cast<const uint4*>(low));
    u.v[1] = __ldcs(reinterpret_cast<const uint4*>(high));
  }
  return u;
}
template <typename T> __device__ __forceinline__ void store_unit(T* low, T* high, const Unit<T>& u) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(low), u.v[0]); __stcs(reinterpret_cast<float4*>(low) + 1, u.v[1]);
    __stcs(reinterpret_cast<float4*>(high), u.v[2]); __stcs(reinterpret_cast<float4*>(high) + 1, u.v[3]);
  } else {
    __stcs(reinterpret_cast<uint4*>(low), u.v[0]);
    __stcs(reinterpret_cast<uint4*>(high), u.v[1]);
  }
}
template <typename T> __device__ __forceinline__ void widen(const Unit<T>& u, float (&x)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) x[i] = reinterpret_cast<const float*>(&u)[i];
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) x[i] = to_float(reinterpret_cast<const T*>(&u)[i]);
  }
}
template <typename T> __device__ __forceinline__ Unit<T> narrow(const float (&x)[16]) {
  Unit<T> u;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) reinterpret_cast<T*>(&u)[i] = from_float<T>(x[i]);
  return u;
}
// Turns the eight pairs of a unit; cs[i] = (cos, sin) of pair i.
__device__ __forceinline__ void turn_unit(float (&x)[16], const float2* cs, bool split) {
#pragma unroll
  for (uint32_t i = 0; i < 8; i += 2) {
    const float4 c = *reinterpret_cast<const float4*>(cs + i);
    const uint32_t a0 = split ? i : 2u * i, b0 = split ? i + 8u : 2u * i + 1u, a1 = split ? i + 1u : 2u * i + 2u, b1 = split ? i + 9u : 2u * i + 3u;
    const float u0 = x[a0], v0 = x[b0], u1 = x[a1], v1 = x[b1];
    x[a0] = u0 * c.x - v0 * c.y; x[b0] = v0 * c.x + u0 * c.y;
    x[a1] = u1 * c.z - v1 * c.w; x[b1] = v1 * c.z + u1 * c.w;
  }
}
// FP8 codes of e[i] / scale, the quotient rounded to fp32 and then to the code. A product with the reciprocal would give codes next to a
// border wrongly; one correction by the remainder, q + (e - q scale) / scale, makes q the rounded quotient (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990). It wants remainders above the smallest numbers, so the elements of
// a row with a tiny scale are multiplied by 2^64 first. 16411 x 64 rows: 83 us with products alone, 87.6 so, 118 with
// divisions.
__device__ __forceinline__ uint32_t two_codes(float x, float y, float2 minus_scale, float2 inverse) {
  const float2 e = make_float2(x, y), q = __fmul2_rn(e, inverse);
  return __nv_cvt_float2_to_fp8x2(__ffma2_rn(__ffma2_rn(q, minus_scale, e), inverse, q), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ void codes_of(float (&e)[16], float scale, uint32_t (&packed)[4]) {
  if (scale < 0x1p-60f) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) e[i] *= 0x1p64f;
    scale *= 0x1p64f;
  }
  const float inverse = 1.f / scale, minus = scale < INFINITY ? -scale : 0.f;   // beside an infinity finite elements are 0, not a remainder of NaN
  const float2 i = make_float2(inverse, inverse), s = make_float2(minus, minus);
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) packed[j] = two_codes(e[4 * j], e[4 * j + 1], s, i) | (two_codes(e[4 * j + 2], e[4 * j + 3], s, i) << 16);
}
// (cos, sin) of `pairs` pairs of the CTA's tokens in shared memory: [tile][stride]
__device__ __forceinline__ void turn_table(const KvipRotaryArgs& a, float2* table, uint32_t first, uint32_t tile, uint32_t pairs) {
  for (uint32_t i = threadIdx.x; i < tile * pairs; i += kRotaryThreads) {
    const uint32_t k = i / pairs, pair = i - k * pairs, token = first + k;
    if (token < a.tokens) table[i] = cos_sin(a.positions[token], a.turns[pair], a.factor);
  }
  __syncthreads();
}

template <typename T, bool kSplit>
__global__ void __launch_bounds__(kRotaryThreads) rotate_units(const __grid_constant__ KvipRotaryArgs a, const uint32_t tile, const uint32_t rows_here) {
  extern __shared__ float2 table[];
  const uint32_t half = a.width >> 1, units = a.width >> 4, rows = a.heads[0] + a.heads[1];
  const uint32_t first = blockIdx.x * tile, row0 = blockIdx.y * rows_here, count = min(rows_here, rows - row0);
  turn_table(a, table, first, tile, half);
  const uint32_t per_token = count * units;
  for (uint32_t i = threadIdx.x; i < tile * per_token; i += kRotaryThreads) {
    const uint32_t k = i / per_token, rest = i - k * per_token, row = row0 + rest / units, v = rest % units, token = first + k;
    if (token >= a.tokens || a.positions[token] < 0) continue;
    const uint32_t set = row >= a.heads[0] ? 1u : 0u;
    const int64_t head = set ? row - a.heads[0] : row;
    const T* x = static_cast<const T*>(a.x[set]) + token * a.x_token[set] + head * a.x_head[set];
    T* y = static_cast<T*>(a.y[set]) + token * a.y_token[set] + head * a.y_head[set];
    const uint32_t low = kSplit ? 8u * v : 16u * v, high = kSplit ? half + low : low + 8u;
    const Unit<T> u = load_unit(x + low, x + high);
    float e[16];
    widen<T>(u, e);
    turn_unit(e, table + k * half + 8u * v, kSplit);
    store_unit(y + low, y + high, narrow<T>(e));
  }
}

// kLanes threads per row of 16 kLanes elements.
// Six CTAs per SM: without the bound the compiler takes 42 registers, which leave five (16411 x 64 rows 92.5 us instead of 87.6).
template <typename T, bool kSplit, uint32_t kLanes>
__global__ void __launch_bounds__(kRotaryThreads, 6) quantise_units(const __grid_constant__ KvipRotaryArgs a, const uint32_t tile, const uint32_t rows_here) {
  extern __shared__ float2 table[];
  const uint32_t half = a.width >> 1, turned = a.width >> 4;
  const uint32_t first = blockIdx.x * tile, row0 = blockIdx.y * rows_here, count = min(rows_here, a.heads[0] - row0);
  turn_table(a, table, first, tile, half);
  const uint32_t v = threadIdx.x % kLanes, items = tile * count;
  for (uint32_t i0 = 0; i0 < items; i0 += kRotaryThreads / kLanes) {   // whole warps stay together for the shuffles
    const uint32_t i = i0 + threadIdx.x / kLanes, k = i / count, row = row0 + (i - k * count), token = first + k;
    const bool live = i < items && token < a.tokens && a.positions[token] >= 0;
    float e[16];
    float amax = 0.f;
    const uint32_t low = kSplit && v < turned ? 8u * v : 16u * v, high = kSplit && v < turned ? half + low : low + 8u;
    if (live) {
      const T* x = static_cast<const T*>(a.x[0]) + token * a.x_token[0] + row * a.x_head[0];
      widen<T>(load_unit(x + low, x + high), e);
      if (v < turned) turn_unit(e, table + k * half + 8u * v, kSplit);
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(e[j]));
    }
#pragma unroll
    for (uint32_t o = kLanes / 2u; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) continue;
    const float scale = index_row_scale(amax);
    const uint64_t r = static_cast<uint64_t>(token) * a.heads[0] + row;
    uint32_t packed[4];
    codes_of(e, scale, packed);
    uint8_t* codes = a.codes + r * a.dim;
    __stcs(reinterpret_cast<uint2*>(codes + low), make_uint2(packed[0], packed[1]));
    __stcs(reinterpret_cast<uint2*>(codes + high), make_uint2(packed[2], packed[3]));
    if (v == 0) a.scales[r] = scale;
  }
}

// Tokens and rows per CTA: about 1024 units of work (512 and 2048 are slower: 16411 x 64 rows to FP8 took 88, 82 and 84 us
// before codes were quotients), tokens first (their angles are shared by all rows), and at least two
// CTAs per SM where there is that much work.
void shares(uint32_t tokens, uint32_t rows, uint32_t units, uint32_t half, uint32_t* tile, uint32_t* rows_here) {
  const uint32_t want = 2u * device_sm_count();
  *rows_here = rows;
  while (*rows_here > 1u && (*rows_here * units > 1024u || tokens * ((rows + *rows_here - 1) / *rows_here) < want) &&
         *rows_here * units > kRotaryThreads)
    *rows_here = (*rows_here + 1) / 2;
  *tile = 1;
  const uint32_t parts = (rows + *rows_here - 1) / *rows_here;
  while (*tile < 16u && *tile * half <= 2048u && *tile * *rows_here * units < 1024u && ((tokens + 2u * *tile - 1) / (2u * *tile)) * parts >= want) *tile *= 2u;
}

template <typename T> bool aligned_rows(const void* base, int64_t token, int64_t head) {
  constexpr uint32_t kRun = sizeof(T) == 4 ? 4u : 8u;   // elements of a 16-byte load
  return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && token % kRun == 0 && head % kRun == 0;
}

template <typename T, bool kSplit>
uint32_t launch_units(const KvipRotaryArgs& a, cudaStream_t stream) {
  uint32_t tile, rows_here;
  const uint32_t rows = a.heads[0] + a.heads[1];
  if (!a.codes) {
    shares(a.tokens, rows, a.width / 16u, a.width / 2u, &tile, &rows_here);
    const dim3 grid((a.tokens + tile - 1) / tile, (rows + rows_here - 1) / rows_here);
    rotate_units<T, kSplit><<<grid, kRotaryThreads, tile * (a.width / 2u) * sizeof(float2), stream>>>(a, tile, rows_here);
    return 0;
  }
  shares(a.tokens, rows, a.dim / 16u, a.width / 2u, &tile, &rows_here);
  const dim3 grid((a.tokens + tile - 1) / tile, (rows + rows_here - 1) / rows_here);
  const uint32_t shared = tile * (a.width / 2u) * sizeof(float2);
  switch (a.dim / 16u) {
    case 1: quantise_units<T, kSplit, 1><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
    case 2: quantise_units<T, kSplit, 2><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
    case 4: quantise_units<T, kSplit, 4><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
    case 8: quantise_units<T, kSplit, 8><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
    case 16: quantise_units<T, kSplit, 16><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
    default: quantise_units<T, kSplit, 32><<<grid, kRotaryThreads, shared, stream>>>(a, tile, rows_here); break;
  }
  return 0;
}

template <typename T>
uint32_t launch_rotary(const KvipRotaryArgs& a, cudaStream_t stream) {
  // the vector forms want rows of whole units at 16-byte boundaries; what else there is goes element by element
  bool wide = a.width % 16u == 0;
  if (a.codes) {
    const uint32_t lanes = a.dim / 16u;
    wide = wide && a.dim % 16u == 0 && lanes <= 32u && (lanes & (lanes - 1u)) == 0 && aligned_rows<T>(a.x[0], a.x_token[0], a.x_head[0]) &&
           (reinterpret_cast<uintptr_t>(a.codes) & 7u) == 0;
  } else {
    for (uint32_t set = 0; set < 2u && a.heads[set]; ++set)
      wide = wide && aligned_rows<T>(a.x[set], a.x_token[set], a.x_head[set]) && aligned_rows<T>(a.y[set], a.y_token[set], a.y_head[set]);
  }
  if (wide) {
    if (a.layout == KVIP_ROTARY_HALF) launch_units<T, true>(a, stream);
    else launch_units<T, false>(a, stream);
  } else if (a.codes) {
    const uint32_t most = device_sm_count() * 16u;
    const uint64_t blocks = (static_cast<uint64_t>(a.tokens) * a.heads[0] + 7u) / 8u;
    quantise_rows<T><<<static_cast<uint32_t>(blocks < most ? blocks : most), kRotaryThreads, 0, stream>>>(a);
  } else {
    const uint32_t most = device_sm_count() * 16u;
    const uint64_t items = static_cast<uint64_t>(a.tokens) * (a.heads[0] + a.heads[1]) * (a.width / 2u);
    const uint64_t blocks = (items + kRotaryThreads - 1) / kRotaryThreads;
    rotate_pairs<T><<<static_cast<uint32_t>(blocks < most ? blocks : most), kRotaryThreads, 0, stream>>>(a);
  }
  count_launch();
  return check_launch("rotary");
}

// Whether rows of `width` elements at these strides lie apart: each is written by one thread or another, in no order.
bool apart(uint64_t tokens, uint64_t heads, int64_t token, int64_t head, int64_t width) {
  if (tokens == 1) token = INT64_MAX;
  if (heads == 1) head = INT64_MAX;
  const int64_t near = token < head ? token : head, far = token < head ? head : token;
  const int64_t count = static_cast<int64_t>(token < head ? tokens : heads);
  return near >= width && (far == INT64_MAX || far >= near * (count - 1) + width);
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
  for (uint32_t set = 0; !a->codes && set < 2u && a->heads[set]; ++set)
    KVIP_REQUIRE(apart(a->tokens, a->heads[set], a->y_token[set], a->y_head[set], a->width), "rotary: output rows overlap");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == KVIP_FLOAT_BF16) return launch_rotary<__nv_bfloat16>(*a, s);
  if (a->dtype == KVIP_FLOAT_FP16) return launch_rotary<__half>(*a, s);
  return launch_rotary<float>(*a, s);
}
