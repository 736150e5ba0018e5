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
// Prompts go through the tiles of tl_append_tiles.hpp, steps (few rows) and
// blocks that hold no whole 16-byte chunks through axes_step_kernel; rows or
// tables that are not 16-byte aligned through axes_rows_kernel.
#include "tl_append_tiles.hpp"
#include "tl_device.hpp"
#include "tl_fp8.hpp"
#include "tl_internal.hpp"

namespace tl {

namespace {

// Any size, stride and alignment: a wavefront per row (one head of one
// token), lane l with pairs l and l + 64 (head_size at most 256); a row of
// the value is taken as pairs too.
template <Kind K, Kind POOL>
__global__ __launch_bounds__(256) void axes_rows_kernel(TileAppend a, int style, int64_t row0) {
  const int lane = threadIdx.x % kWave, half = a.head_size / 2;
  const int per_token = a.num_heads + 2 * a.num_kv_heads;
  const int64_t row = row0 + (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  const int64_t t = row / per_token;
  if (t >= a.num_tokens) return;
  const int h = (int)(row - t * per_token);
  const bool is_q = h < a.num_heads, is_v = h >= a.num_heads + a.num_kv_heads;
  if (a.num_axes && !Places(a, t).in_tables(a)) return;   // the token is left as it is
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
    const int e0 = style == 0 ? 2 * i : i, e1 = style == 0 ? 2 * i + 1 : i + half;
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
      store_scalar<K>(a.q_out, to + (style == 0 ? 2 * i : i), x[j][0]);
      store_scalar<K>(a.q_out, to + (style == 0 ? 2 * i + 1 : i + half), x[j][1]);
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
    const int64_t d0 = to + (int64_t)(style == 0 ? 2 * i : i) * a.block_size;
    const int64_t d1 = to + (int64_t)(style == 0 ? 2 * i + 1 : i + half) * a.block_size;
    if constexpr (POOL == Kind::FP8) {
      ((uint8_t*)pool)[d0] = f32_to_fp8(x[j][0] * scale.inv);
      ((uint8_t*)pool)[d1] = f32_to_fp8(x[j][1] * scale.inv);
    } else {
      store_scalar<K>(pool, d0, x[j][0]);
      store_scalar<K>(pool, d1, x[j][1]);
    }
  }
}

// Steps: a wavefront per (token, kv head) with its key and its value, and
// threads of 8 rotation pairs of a q head after them; lane l has the rotation
// pairs l and l + 64 of the key, and the value's elements in their place.
// Every load that hangs on nothing else is issued first, so a wavefront is two
// round trips to memory and its stores.
//
// The elements of a row lie a block apart and are stored alone.  Rewriting the
// aligned 16 to 64 bytes around each, as the 2-byte appends do, was measured
// and is slower here, in pools that the caches hold and in pools that they do
// not: 64 tokens, 8 kv heads, scaled FP8, blocks of 16: 3.5 us (rewritten 4.3),
// of 64 5.7 (8.1), of 256 5.1 (10.6); bf16 3.8 (4.9), 5.4 (10.0), 4.9 (10.6).
template <Kind K, Kind POOL, int ROPE>
__global__ __launch_bounds__(kWave) void axes_step_kernel(TileAppend a) {
  const int lane = threadIdx.x, half = a.head_size / 2;
  if constexpr (ROPE != kNoRope) {
    if ((int)blockIdx.x >= a.kv_wgs) {
      const unsigned units = half / 8, idx = (blockIdx.x - a.kv_wgs) * kWave + lane;   // fewer than 2^32 threads
      const int u = (int)(idx % units), h = (int)(idx / units % a.num_heads);
      const int64_t t = idx / units / a.num_heads;
      if (t >= a.num_tokens) return;
      float c[8], s[8], lo[8], hi[8];
      const Places at(a, t);
      load_unit<K, ROPE>(a.q, t * a.q_stride + h * a.head_size, u, half, lo, hi);
      if (!at.in_tables(a)) return;                           // the token is left as it is
      axes_turn(a, at, u, half, c, s);
      rotate_unit<ROPE>(lo, hi, c, s);
      store_unit<K, ROPE>(a.q_out, t * a.q_out_stride + h * a.head_size, u, half, lo, hi);
      return;
    }
  }
  const int t = blockIdx.x / a.num_kv_heads, h = blockIdx.x % a.num_kv_heads;
  Places at = {};
  if constexpr (ROPE != kNoRope) at = Places(a, t);
  const int32_t slot = a.slots[t];
  float k[2][2] = {}, v[2][2] = {};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + kWave * j;
    if (i >= half) break;
    const int e0 = rope_channel<ROPE>(i, 0, half), e1 = rope_channel<ROPE>(i, 1, half);
    const int64_t fk = t * a.key_stride + h * a.head_size, fv = t * a.value_stride + h * a.head_size;
    k[j][0] = load_scalar<K>(a.key, fk + e0);
    k[j][1] = load_scalar<K>(a.key, fk + e1);
    v[j][0] = load_scalar<K>(a.value, fv + e0);
    v[j][1] = load_scalar<K>(a.value, fv + e1);
  }
  if (ROPE != kNoRope && !at.in_tables(a)) return;
  if (slot < 0 || slot / a.block_size >= a.num_blocks) return;
  const int blk = slot / a.block_size, off = slot % a.block_size;
  const int64_t head = (int64_t)blk * a.num_kv_heads + h;
  uint32_t kt = 0, vt = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + kWave * j;
    if (i >= half) break;
    if constexpr (ROPE != kNoRope) {
      const int64_t row = (int64_t)at.on(axes_word(a, i / 16) >> (2 * (i % 16)) & 3) * half + i;
      const float c = a.cos_table[row], s = a.sin_table[row], x0 = k[j][0], x1 = k[j][1];
      k[j][0] = fp32_result(__builtin_fmaf(x0, c, -(x1 * s)));
      k[j][1] = fp32_result(__builtin_fmaf(x0, s, x1 * c));
    }
    kt = max(kt, max(abs_bits(k[j][0]), abs_bits(k[j][1])));
    vt = max(vt, max(abs_bits(v[j][0]), abs_bits(v[j][1])));
  }
  const int64_t to = head * a.head_size * a.block_size + off;
  if constexpr (POOL == Kind::FP8) {
    const Fp8Scale ks = fp8_scale_of(lanes_umax<kWave>(kt)), vs = fp8_scale_of(lanes_umax<kWave>(vt));
    if (lane == 0) {
      a.k_scales[head * a.block_size + off] = ks.scale;
      a.v_scales[head * a.block_size + off] = vs.scale;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        k[j][r] *= ks.inv;
        v[j][r] *= vs.inv;
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (lane + kWave * j >= half) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t e = to + (int64_t)rope_channel<ROPE>(lane + kWave * j, r, half) * a.block_size;
      if constexpr (POOL == Kind::FP8) {
        ((uint8_t*)a.k_cache)[e] = f32_to_fp8(k[j][r]);
        ((uint8_t*)a.v_cache)[e] = f32_to_fp8(v[j][r]);
      } else {
        store_scalar<POOL>(a.k_cache, e, k[j][r]);
        store_scalar<POOL>(a.v_cache, e, v[j][r]);
      }
    }
  }
}

// Rows of keys up to which a call is taken for a step.  us as a step and in
// tiles, one run of consecutive tokens and tokens that each lie in a block of
// their own, blocks of 64, bf16: 8/1 heads, 600 tokens 4.4 and 6.1, 5.3 and
// 6.7; 16/2, 600 5.6 and 5.5, 7.4 and 8.6; past the line 32/8, 300 6.9 and 5.9,
// 11.4 and 12.6, 600 11.0 and 7.3, 33.5 and 32.8; 32/32, 300 15.7 and 8.1.
constexpr int64_t kStepMaxRows = 2048;

template <Kind K, Kind POOL, int ROPE>
int launch_style(const TileAppend& a, int style, hipStream_t stream) {
  constexpr int E = KindInfo<POOL>::bytes, S = KindInfo<K>::bytes;
  const auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const auto whole = [](int64_t stride) { return stride * S % 16 == 0; };
  const bool rows16 = ROPE == kNoRope || a.num_heads == 0 ||
                      (al(a.q) && al(a.q_out) && whole(a.q_stride) && whole(a.q_out_stride));
  const bool tables16 = ROPE == kNoRope || (al(a.cos_table) && al(a.sin_table));
  if ((int64_t)a.num_tokens * a.num_kv_heads > kStepMaxRows && rows16 && whole(a.key_stride) && whole(a.value_stride) &&
      tile_shape<true>(a, S, E, ROPE != kNoRope))
    return launch_tiles<K, POOL, ROPE, true>(a, stream);
  if (rows16 && tables16) {
    TileAppend s = a;
    const int64_t q = ROPE == kNoRope ? 0 : (int64_t)a.num_tokens * a.num_heads * (a.head_size / 16);
    const int64_t wgs = (int64_t)a.num_tokens * a.num_kv_heads + (q + kWave - 1) / kWave;
    if (wgs < (1ll << 32) / kWave) {
      s.kv_wgs = a.num_tokens * a.num_kv_heads;
      hipLaunchKernelGGL((axes_step_kernel<K, POOL, ROPE>), dim3((unsigned)wgs), dim3(kWave), 0, stream, s);
      return hipGetLastError() == hipSuccess ? 0 : 5;
    }
  }
  const int64_t rows = (int64_t)a.num_tokens * (a.num_heads + 2 * a.num_kv_heads), wgs = (rows + 3) / 4;
  constexpr int64_t kWgs = 1 << 23;                   // of a launch: fewer than 2^32 threads
  for (int64_t w = 0; w < wgs; w += kWgs)
    hipLaunchKernelGGL((axes_rows_kernel<K, POOL>), dim3((unsigned)(wgs - w < kWgs ? wgs - w : kWgs)), dim3(256), 0,
                       stream, a, style, 4 * w);
  return hipGetLastError() == hipSuccess ? 0 : 5;
}

template <Kind K, Kind POOL>
int launch_pool(const AxesAppend& c, hipStream_t stream) {
  TileAppend a = {};
  a.q = c.q; a.q_out = c.q_out; a.key = c.key; a.value = c.value;
  a.k_cache = (char*)c.k_cache; a.v_cache = (char*)c.v_cache;
  a.k_scales = c.k_scales; a.v_scales = c.v_scales;
  a.slots = c.slots; a.positions = c.positions; a.cos_table = c.cos_table; a.sin_table = c.sin_table;
  a.num_tokens = c.num_tokens; a.num_heads = c.num_heads; a.num_kv_heads = c.num_kv_heads;
  a.head_size = c.head_size; a.block_size = c.block_size; a.num_blocks = c.num_blocks;
  a.max_positions = c.max_positions;
  a.q_stride = c.q_stride; a.q_out_stride = c.q_out_stride;
  a.key_stride = c.key_stride; a.value_stride = c.value_stride;
  a.num_axes = c.num_axes;
  for (int i = 0; i < 8; ++i) a.axis_of[i] = c.axis_of[i];
  if (c.num_axes == 0) return launch_style<K, POOL, kNoRope>(a, 0, stream);
  return c.style ? launch_style<K, POOL, 1>(a, 1, stream) : launch_style<K, POOL, 0>(a, 0, stream);
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
