// tl_rope_axes.hip -- rotary positions with several axes on the way into the
// paged pools, and the quantising append: FP8 E4M3 codes with one scale for
// each token and head.
//
// Pair i of a head of q and of key is turned by the tables' row of the
// position that its token has on the pair's axis,
//   c, s = tables[positions[axis(i)][t]][i],
//   (a, b) -> (fmaf(a, c, -(b s)), fmaf(a, s, b c)),
// which with one axis is the rotation of tl_cache.hip.  A pool of the
// tensors' own type takes the result rounded once; an FP8 pool takes
//   scale = max|row| / 448,  code = e4m3(row / scale)
// of each row (one token of one kv head; the key as rotated, in fp32).
#include "tl_device.hpp"
#include "tl_fp8.hpp"
#include "tl_internal.hpp"

namespace tl {

namespace {

// An fp32 result as computed, before its conversion to a 2-byte type (which
// the compiler would otherwise fuse with the last fma, rounding once).
__device__ __forceinline__ float fp32_result(float r) {
  asm volatile("" : "+v"(r));
  return r;
}

// Whether token t is at a place of the tables on every axis.
__device__ __forceinline__ bool placed(const AxesAppend& a, int64_t t) {
  for (int x = 0; x < a.num_axes; ++x) {
    const int pos = a.positions[x * (int64_t)a.num_tokens + t];
    if (pos < 0 || pos >= a.max_positions) return false;
  }
  return true;
}

// Any size, stride and alignment: a wavefront per row (one head of one
// token), lane l with pairs l and l + 64 (head_size at most 256); a row of
// the value is taken as pairs too.
template <Kind K, Kind POOL>
__global__ __launch_bounds__(256) void axes_rows_kernel(AxesAppend a, int64_t row0) {
  const int lane = threadIdx.x % kWave, half = a.head_size / 2;
  const int per_token = a.num_heads + 2 * a.num_kv_heads;
  const int64_t row = row0 + (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  const int64_t t = row / per_token;
  if (t >= a.num_tokens) return;
  const int h = (int)(row - t * per_token);
  const bool is_q = h < a.num_heads, is_v = h >= a.num_heads + a.num_kv_heads;
  if (a.num_axes && !placed(a, t)) return;            // the token is left as it is
  int blk = 0, off = 0;
  if (!is_q) {
    const int32_t slot = a.slots[t];
    if (slot < 0 || slot / a.block_size >= a.num_blocks) return;
    blk = slot / a.block_size;
    off = slot % a.block_size;
  }
  const int hk = is_q ? h : is_v ? h - a.num_heads - a.num_kv_heads : h - a.num_heads;
  const void* src = is_q ? a.q : is_v ? a.value : a.key;
  const int64_t from = t * (is_q ? a.q_stride : is_v ? a.value_stride : a.key_stride) + (int64_t)hk * a.head_size;
  float x[2][2];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + kWave * j;
    if (i >= half) continue;
    const int e0 = a.style == 0 ? 2 * i : i, e1 = a.style == 0 ? 2 * i + 1 : i + half;
    const float x0 = load_scalar<K>(src, from + e0), x1 = load_scalar<K>(src, from + e1);
    x[j][0] = x0;
    x[j][1] = x1;
    if (!is_v && a.num_axes) {
      const int axis = (a.axis_of[i / 16] >> (2 * (i % 16))) & 3;
      const int64_t at = (int64_t)a.positions[axis * (int64_t)a.num_tokens + t] * half + i;
      const float c = a.cos_table[at], s = a.sin_table[at];
      x[j][0] = fp32_result(__builtin_fmaf(x0, c, -(x1 * s)));
      x[j][1] = fp32_result(__builtin_fmaf(x0, s, x1 * c));
    }
    top = max(top, max(abs_bits(x[j][0]), abs_bits(x[j][1])));
  }
  if (is_q) {
    const int64_t to = t * a.q_out_stride + (int64_t)hk * a.head_size;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = lane + kWave * j;
      if (i >= half) continue;
      store_scalar<K>(a.q_out, to + (a.style == 0 ? 2 * i : i), x[j][0]);
      store_scalar<K>(a.q_out, to + (a.style == 0 ? 2 * i + 1 : i + half), x[j][1]);
    }
    return;
  }
  char* pool = (char*)(is_v ? a.v_cache : a.k_cache);
  const int64_t head = (int64_t)blk * a.num_kv_heads + hk;
  const int64_t to = head * a.head_size * a.block_size + off;
  Fp8Scale scale = {};
  if constexpr (POOL == Kind::FP8) {
    scale = fp8_scale_of(lanes_umax<kWave>(top));
    if (lane == 0) (is_v ? a.v_scales : a.k_scales)[head * a.block_size + off] = scale.scale;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + kWave * j;
    if (i >= half) continue;
    const int64_t d0 = to + (int64_t)(a.style == 0 ? 2 * i : i) * a.block_size;
    const int64_t d1 = to + (int64_t)(a.style == 0 ? 2 * i + 1 : i + half) * a.block_size;
    if constexpr (POOL == Kind::FP8) {
      ((uint8_t*)pool)[d0] = f32_to_fp8(x[j][0] * scale.inv);
      ((uint8_t*)pool)[d1] = f32_to_fp8(x[j][1] * scale.inv);
    } else {
      store_scalar<K>(pool, d0, x[j][0]);
      store_scalar<K>(pool, d1, x[j][1]);
    }
  }
}

template <Kind K, Kind POOL>
int launch_pool(const AxesAppend& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.num_tokens * (a.num_heads + 2 * a.num_kv_heads), wgs = (rows + 3) / 4;
  constexpr int64_t kWgs = 1 << 23;                   // of a launch: fewer than 2^32 threads
  for (int64_t w = 0; w < wgs; w += kWgs)
    hipLaunchKernelGGL((axes_rows_kernel<K, POOL>), dim3((unsigned)(wgs - w < kWgs ? wgs - w : kWgs)), dim3(256), 0,
                       stream, a, 4 * w);
  return hipGetLastError() == hipSuccess ? 0 : 5;
}

}  // namespace

int launch_axes_append(const AxesAppend& a, hipStream_t stream) {
  if (a.num_tokens == 0) return 0;
  const Kind k = (Kind)a.dtype;
  if (a.kv_dtype == (int)Kind::FP8) {
    if (k == Kind::F16) return launch_pool<Kind::F16, Kind::FP8>(a, stream);
    if (k == Kind::BF16) return launch_pool<Kind::BF16, Kind::FP8>(a, stream);
    return 3;
  }
  if (k == Kind::F16) return launch_pool<Kind::F16, Kind::F16>(a, stream);
  if (k == Kind::BF16) return launch_pool<Kind::BF16, Kind::BF16>(a, stream);
  if (k == Kind::F32) return launch_pool<Kind::F32, Kind::F32>(a, stream);
  return 3;
}

}  // namespace tl
