// tl_row.hpp -- what the kernels that work on rows of activations or heads
// share: eight elements between storage and fp32, a row's sum over a workgroup.
#pragma once

#include "tl_device.hpp"

namespace tl {

constexpr int kNormThreads = 256;

// Sum over the workgroup, returned to every thread.
__device__ __forceinline__ float block_sum(float v, float* s_part) {
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
  const int wave = threadIdx.x / kWave;
  __syncthreads();                                   // s_part free from a previous use
  if (threadIdx.x % kWave == 0) s_part[wave] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < kNormThreads / kWave; ++w) t += s_part[w];
  return t;
}

// Sum over the wavefront, returned to every lane.
__device__ __forceinline__ float wave_total(float v) {
  v = row_sum(v);
  v = swap16_add(v, v);
  return swap32_add(v, v);
}

// Round to the storage type and back (identity for f32).
template <Kind K> __device__ __forceinline__ float round_to(float v);
template <> __device__ __forceinline__ float round_to<Kind::F32>(float v) { return v; }
template <> __device__ __forceinline__ float round_to<Kind::F16>(float v) { return f16_to_f32(f32_to_f16(v)); }
template <> __device__ __forceinline__ float round_to<Kind::BF16>(float v) { return bf16_to_f32(f32_to_bf16(v)); }

template <Kind K> __device__ __forceinline__ void unpack8(const u32x4& c, float (&f)[8]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint16_t b = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    f[j] = K == Kind::F16 ? f16_to_f32(b) : bf16_to_f32(b);
  }
}
template <Kind K> __device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint16_t lo = K == Kind::F16 ? f32_to_f16(f[2 * k]) : f32_to_bf16(f[2 * k]);
    const uint16_t hi = K == Kind::F16 ? f32_to_f16(f[2 * k + 1]) : f32_to_bf16(f[2 * k + 1]);
    w[k] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return u32x4{w[0], w[1], w[2], w[3]};
}

// Eight elements as loaded.
template <Kind K> struct Raw8 {
  u32x4 w[K == Kind::F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    const char* at = (const char*)p + i * KindInfo<K>::bytes;
    w[0] = load16(at);
    if constexpr (K == Kind::F32) w[1] = load16(at + 16);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (K == Kind::F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __builtin_bit_cast(float, word(w[j / 4], j % 4));
    } else {
      unpack8<K>(w[0], f);
    }
  }
};
template <Kind K>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&f)[8]) {
  char* at = (char*)p + i * KindInfo<K>::bytes;
  if constexpr (K == Kind::F32) {
    u32x4 w[2];
    __builtin_memcpy(w, f, 32);
    reinterpret_cast<u32x4*>(at)[0] = w[0];
    reinterpret_cast<u32x4*>(at)[1] = w[1];
  } else {
    *reinterpret_cast<u32x4*>(at) = pack8<K>(f);
  }
}

}  // namespace tl
