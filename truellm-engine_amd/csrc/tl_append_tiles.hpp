// tl_append_tiles.hpp -- prompt-sized appends into the paged pools: tiles of
// tokens staged in LDS and stored along the slots, shared by the plain, the
// rotated and the quantising appends.
#pragma once

#include "tl_device.hpp"
#include "tl_fp8.hpp"
#include "tl_internal.hpp"
#include "tl_row.hpp"

namespace tl {

template <Kind SRC> __device__ __forceinline__ void load8(const void* p, int64_t i, float* f);
template <> __device__ __forceinline__ void load8<Kind::F16>(const void* p, int64_t i, float* f) {
  const u32x4 c = load16((const uint16_t*)p + i);
  Unpack<Kind::F16>::run(c.x, f); Unpack<Kind::F16>::run(c.y, f + 2);
  Unpack<Kind::F16>::run(c.z, f + 4); Unpack<Kind::F16>::run(c.w, f + 6);
}
template <> __device__ __forceinline__ void load8<Kind::BF16>(const void* p, int64_t i, float* f) {
  const u32x4 c = load16((const uint16_t*)p + i);
  Unpack<Kind::BF16>::run(c.x, f); Unpack<Kind::BF16>::run(c.y, f + 2);
  Unpack<Kind::BF16>::run(c.z, f + 4); Unpack<Kind::BF16>::run(c.w, f + 6);
}

// An fp32 result as computed, before its conversion to a 2-byte type: the
// compiler would otherwise fuse the last fma with the conversion
// (v_fma_mix*, one rounding), where rope_cache_kernel and the reference
// round to fp32 first.
__device__ __forceinline__ float fp32_result(float r) {
  asm volatile("" : "+v"(r));
  return r;
}

// The element's bits in the pool's type (the rounding of store_scalar).
template <Kind K> __device__ __forceinline__ uint32_t scalar_bits(float v);
template <> __device__ __forceinline__ uint32_t scalar_bits<Kind::F32>(float v) { return __float_as_uint(v); }
template <> __device__ __forceinline__ uint32_t scalar_bits<Kind::F16>(float v) { return f32_to_f16(v); }
template <> __device__ __forceinline__ uint32_t scalar_bits<Kind::BF16>(float v) { return f32_to_bf16(v); }

// Prompt-sized appends.  The element stores of reshape_copy_kernel and
// rope_cache_kernel leave one 2-byte store per (token, channel), each
// instruction over 64 lines of the pool.  Here a workgroup takes a tile of 32
// (small calls: 16 or 8) consecutive tokens of one kv head, of K or of V,
// stages their rows in LDS and writes the pool along the slots: where C = 16 / E tokens of the tile
// fill an aligned 16-byte chunk, it is one store per channel, with the lanes
// of a store over consecutive chunks of a block's rows; tokens that fill no
// chunk are stored element by element, and no slot of another token is
// written.
//
// Tokens belong to segments: consecutive tokens of the call in consecutive
// slots of one aligned group of `group` slots (at most 32: a block or a part
// of one).  A tile takes the segments that begin in it, so that a group's
// lines have one writer, and at most 32 + 31 tokens, whose slots fit a
// wavefront's lanes.
//
// Bound by HBM.  4180 tokens of 8 kv heads, 32 heads, d 128, bf16, blocks of
// 16, rotated: 28.2 us (element stores: 93.7); 4096 tokens copied without
// rotation 7.9 us (43.2), into FP8 pools 8.3 us (42.8).  Tokens that each lie
// in a block of their own (a decode batch of more than 256 sequences) are
// stored element by element as before: 512 of them copied 10.2 us (10.2),
// 1024 17.0 (17.8), in blocks of 32 slots 15.7 (14.8) and 28.2 (27.4); rotated
// 11.8 (14.3), into FP8 pools 7.1 (13.5).
struct TileAppend {
  const void* q; void* q_out;              // ROPE only
  const void* key; const void* value;
  char* k_cache; char* v_cache;
  const int32_t* slots; const int32_t* positions;
  const float* cos_table; const float* sin_table;
  int num_tokens, num_heads, num_kv_heads, head_size, block_size, num_blocks, max_positions;
  int group;                               // slots of a segment's group
  int tile;                                // tokens of a tile: 8, 16 or 32
  int kv_wgs;                              // workgroups over K and V; q's follow
  float k_mul, v_mul;                      // FP8 pools
  // AXES: the call's own strides and scales, and a position on each axis
  int64_t q_stride, q_out_stride, key_stride, value_stride;
  float* k_scales; float* v_scales;        // FP8 pools: [N, n_kv, block_size]
  int num_axes;
  uint32_t axis_of[8];                     // 2 bits for each rotation pair
};

// AXES: token t's position on each axis, all read at once (the last one again
// past num_axes), and whether every one is a row of the tables.
struct alignas(16) Places {
  int pos[4];
  Places() = default;
  __device__ __forceinline__ Places(const TileAppend& a, int64_t t) {
#pragma unroll
    for (int x = 0; x < 4; ++x) pos[x] = a.positions[min(x, a.num_axes - 1) * (int64_t)a.num_tokens + t];
  }
  __device__ __forceinline__ bool in_tables(const TileAppend& a) const {
    bool in = true;
#pragma unroll
    for (int x = 0; x < 4; ++x) in &= (unsigned)pos[x] < (unsigned)a.max_positions;   // no branch between the reads
    return in;
  }
  // (Opaque selects here and below, or the compiler makes an indexed read of a
  // copy in LDS or scratch of them.)
  __device__ __forceinline__ int on(uint32_t axis) const {
    int r = pos[0];
#pragma unroll
    for (int x = 1; x < 4; ++x) {
      r = axis == (uint32_t)x ? pos[x] : r;
      asm("" : "+v"(r));
    }
    return r;
  }
};
// The axes of pairs 16 w .. 16 w + 15, 2 bits each, by selects: an indexed
// read of the arguments is a round trip to memory before the tables' own.
__device__ __forceinline__ uint32_t axes_word(const TileAppend& a, int w) {
  uint32_t v = a.axis_of[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    v = w == i ? a.axis_of[i] : v;
    asm("" : "+v"(v));
  }
  return v;
}

constexpr int kTileTokens = 32;            // at most
constexpr int kTileThreads = 256, kTileRowPad = 8;
constexpr int kTileHeadsPerThread = 4;     // q heads of one token and rotation unit
constexpr int kNoRope = -1;

// Eight elements of a row in the pool's type, staged in LDS (8-byte aligned).
// FOUND: multiplied by the inverse of a scale found from them.
template <Kind POOL, bool FOUND = false>
__device__ __forceinline__ void stage8(char* dst, const float* x) {
  uint32_t* d = reinterpret_cast<uint32_t*>(dst);
  if constexpr (POOL == Kind::FP8 && FOUND) {
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = pack4_fp8_found(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else if constexpr (POOL == Kind::FP8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = pack4_fp8(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else if constexpr (POOL == Kind::F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = scalar_bits<POOL>(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = scalar_bits<POOL>(x[2 * i]) | scalar_bits<POOL>(x[2 * i + 1]) << 16;
  }
}

// Eight elements in fp32.
template <Kind K>
__device__ __forceinline__ void load8f(const void* p, int64_t i, float* f) {
  if constexpr (K == Kind::F32) {
    const u32x4 a = load16((const float*)p + i), b = load16((const float*)p + i + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
  } else {
    load8<K>(p, i, f);
  }
}

// Rotation unit u of a row at `base`: pairs 8 u .. 8 u + 7, their elements
// in lo (ADJACENT: the first 8 of 16 consecutive ones; HALVES: the first of
// each pair) and hi.
template <Kind K, int STYLE>
__device__ __forceinline__ void load_unit(const void* p, int64_t base, int u, int half, float* lo, float* hi) {
  load8f<K>(p, base + (STYLE == 0 ? 16 * u : 8 * u), lo);
  load8f<K>(p, base + (STYLE == 0 ? 16 * u + 8 : half + 8 * u), hi);
}
// and its store, rounded to K
template <Kind K, int STYLE>
__device__ __forceinline__ void store_unit(void* p, int64_t base, int u, int half, const float* lo, const float* hi) {
  constexpr int E = KindInfo<K>::bytes;
  alignas(16) char row[8 * E];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    stage8<K>(row, j ? hi : lo);
    const int64_t at = base + (STYLE == 0 ? 16 * u + 8 * j : j * half + 8 * u);
#pragma unroll
    for (int w = 0; w < E / 2; ++w)
      *reinterpret_cast<u32x4*>((char*)p + at * E + 16 * w) = reinterpret_cast<const u32x4*>(row)[w];
  }
}
// Channel j of rotation pair i (without a rotation, as HALVES).
template <int STYLE>
__device__ __forceinline__ int rope_channel(int i, int j, int half) {
  return STYLE == 0 ? 2 * i + j : i + j * half;
}
template <int STYLE>
__device__ __forceinline__ void rotate_unit(float* lo, float* hi, const float* c, const float* s) {
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    float& a = STYLE == 0 ? (p < 4 ? lo[2 * p] : hi[2 * p - 8]) : lo[p];
    float& b = STYLE == 0 ? (p < 4 ? lo[2 * p + 1] : hi[2 * p - 7]) : hi[p];
    const float x0 = a, x1 = b;
    a = fp32_result(__builtin_fmaf(x0, c[p], -(x1 * s[p])));
    b = fp32_result(__builtin_fmaf(x0, s[p], x1 * c[p]));
  }
}

// The tables' entries for pairs 8 u .. 8 u + 7 of a token in its places: the
// pairs of one row of them where they share an axis, else of every axis' row,
// of which each pair keeps its own (the lanes of a token's units read whole
// rows so; with a read for each pair 32.3 us for 4180 tokens of 32/8 heads with
// the pairs dealt out in turn, 29.7 so, 25.4 in runs).  The first pair's axis
// is not read again: 4000 tokens of 32/32 heads, bf16, dealt 49.3 us in place
// of 51.7 (43.8 in runs).
__device__ __forceinline__ void axes_turn(const TileAppend& a, const Places& at, int u, int half, float* c, float* s) {
  const uint32_t of = axes_word(a, u / 2) >> (16 * (u & 1)) & 0xffffu;
  int64_t row = (int64_t)at.on(of & 3) * half + 8 * u;
  load8f<Kind::F32>(a.cos_table, row, c);
  load8f<Kind::F32>(a.sin_table, row, s);
  if (of == (of & 3) * 0x5555u) return;
  for (int i = 1; i < a.num_axes; ++i) {                       // the other axes, from the first pair's on
    const uint32_t next = (of & 3) + i, x = next < (uint32_t)a.num_axes ? next : next - a.num_axes;
    float cx[8], sx[8];
    row = (int64_t)at.on(x) * half + 8 * u;
    load8f<Kind::F32>(a.cos_table, row, cx);
    load8f<Kind::F32>(a.sin_table, row, sx);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const bool mine = (of >> (2 * p) & 3) == x;
      c[p] = mine ? cx[p] : c[p];
      s[p] = mine ? sx[p] : s[p];
    }
  }
}

template <Kind K, int STYLE>
__device__ __forceinline__ void rotate_q_tile(const TileAppend& a, int wg) {
  const int half = a.head_size / 2, units = half / 8;
  const int sets = (a.num_heads + kTileHeadsPerThread - 1) / kTileHeadsPerThread;
  const int64_t idx = (int64_t)wg * kTileThreads + threadIdx.x;
  const int u = (int)(idx % units);
  const int set = (int)((idx / units) % sets);
  const int64_t t = idx / ((int64_t)units * sets);
  if (t >= a.num_tokens) return;
  const int pos = a.positions[t];
  if (pos < 0 || pos >= a.max_positions) return;                // token left as it is
  float c[8], s[8], lo[kTileHeadsPerThread][8], hi[kTileHeadsPerThread][8];
  load8f<Kind::F32>(a.cos_table, (int64_t)pos * half + 8 * u, c);
  load8f<Kind::F32>(a.sin_table, (int64_t)pos * half + 8 * u, s);
  // head set + sets i: the lanes of a wavefront on consecutive heads
#pragma unroll
  for (int i = 0; i < kTileHeadsPerThread; ++i) {
    const int h = set + i * sets;
    if (h < a.num_heads)
      load_unit<K, STYLE>(a.q, (t * a.num_heads + h) * a.head_size, u, half, lo[i], hi[i]);
  }
#pragma unroll
  for (int i = 0; i < kTileHeadsPerThread; ++i) {
    const int h = set + i * sets;
    if (h >= a.num_heads) break;
    rotate_unit<STYLE>(lo[i], hi[i], c, s);
    const int64_t base = (t * a.num_heads + h) * a.head_size;
    store_unit<K, STYLE>(a.q_out, base, u, half, lo[i], hi[i]);
  }
}

// AXES: the q heads of one token, of more where it has few.  A thread reads the
// tables' entries of one pair of one token, which all of the token's heads take
// from LDS, so that pairs whose axes differ cost one read each, not one for
// every head; the heads' first elements are on their way meanwhile.  Bound by
// HBM: 4055 tokens of 64/8 heads into scaled FP8 pools 36.4 us, 4.4 TB/s (36.9
// when it came in; with 4 tokens to a workgroup, of whose 8 units a thread 4 are
// in flight, 43.5; as rotate_q_tile, the tables read by every thread, 46.0).
inline __host__ __device__ int axes_q_tokens(int num_heads, int head_size) {
  const int fit = kTileThreads / (head_size / 2), units = num_heads * (head_size / 16);
  return max(1, min(fit, kTileThreads / units));
}
template <Kind K, int STYLE>
__device__ __forceinline__ void rotate_q_axes(const TileAppend& a, int wg) {
  __shared__ __attribute__((aligned(16))) float cs[kTileThreads], sn[kTileThreads];
  __shared__ int in_tables[kTileThreads / 8];
  const int half = a.head_size / 2, units = half / 8, tokens = axes_q_tokens(a.num_heads, a.head_size);
  const int tid = threadIdx.x, t0 = wg * tokens;
  const int mine = tid / half;                                  // token of the tile
  const bool turns = mine < tokens && t0 + mine < a.num_tokens;
  const Places at(a, turns ? t0 + mine : t0);
  // units of the tile's tokens and heads: kAhead of a thread in flight at once
  constexpr int kAhead = 2;
  const unsigned per_token = (unsigned)units * a.num_heads;
  const unsigned total = per_token * min(tokens, a.num_tokens - t0);
  Raw8<K> lo[kAhead], hi[kAhead];
  struct Unit { int u, t; int64_t h; };
  auto unit_of = [&](unsigned j) {
    const unsigned t = j / per_token, r = j - t * per_token, h = r / units;
    return Unit{(int)(r - h * units), (int)t, (int64_t)h * a.head_size};
  };
  auto load = [&](unsigned j0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const Unit x = unit_of(min(j0 + i * kTileThreads, total - 1));      // past the end: the last one again
      const int64_t from = (t0 + x.t) * a.q_stride + x.h;
      lo[i].load(a.q, from + (STYLE == 0 ? 16 * x.u : 8 * x.u));
      hi[i].load(a.q, from + (STYLE == 0 ? 16 * x.u + 8 : half + 8 * x.u));
    }
  };
  load(tid);
  if (turns) {
    const int i = tid - mine * half;
    const bool in = at.in_tables(a);
    const int64_t row = (int64_t)(in ? at.on(axes_word(a, i / 16) >> (2 * (i % 16)) & 3) : 0) * half + i;
    cs[tid] = a.cos_table[row];
    sn[tid] = a.sin_table[row];
    if (i == 0) in_tables[mine] = in;
  }
  __syncthreads();
  for (unsigned j0 = tid; j0 < total; j0 += kAhead * kTileThreads) {
    if (j0 >= kAhead * kTileThreads) load(j0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (j0 + i * kTileThreads >= total) break;
      const Unit x = unit_of(j0 + i * kTileThreads);
      if (!in_tables[x.t]) continue;                            // token left as it is
      float p[8], r[8];
      lo[i].get(p);
      hi[i].get(r);
      rotate_unit<STYLE>(p, r, cs + x.t * half + 8 * x.u, sn + x.t * half + 8 * x.u);
      store_unit<K, STYLE>(a.q_out, (t0 + x.t) * a.q_out_stride + x.h, x.u, half, p, r);
    }
  }
}

template <Kind SRC, Kind POOL, int ROPE, bool AXES = false>
__global__ __launch_bounds__(kTileThreads) void append_tiles_kernel(TileAppend a) {
  extern __shared__ __attribute__((aligned(16))) char tile_rows[];   // written 8 bytes at a time
  if constexpr (ROPE != kNoRope) {
    if ((int)blockIdx.x >= a.kv_wgs) {
      if constexpr (AXES) rotate_q_axes<SRC, ROPE>(a, blockIdx.x - a.kv_wgs);
      else rotate_q_tile<SRC, ROPE>(a, blockIdx.x - a.kv_wgs);
      return;
    }
  }
  constexpr int E = KindInfo<POOL>::bytes, C = 16 / E;
  constexpr bool SCALED = AXES && POOL == Kind::FP8;            // a scale for each row, found here
  const int h = (int)(blockIdx.x / 2) % a.num_kv_heads, t0 = (int)(blockIdx.x / 2) / a.num_kv_heads * a.tile;
  const bool is_v = blockIdx.x % 2;
  const int tid = threadIdx.x, lane = tid % kWave;

  // lane i: token t0 + i, and the token before it
  auto slot_of = [&](int t) {
    if constexpr (ROPE != kNoRope && AXES) {
      // reads that wait for nothing, of the nearest token there is
      const int near = min(max(t, 0), a.num_tokens - 1);
      const int s = a.slots[near];
      const Places at(a, near);
      return t == near && s >= 0 && s / a.block_size < a.num_blocks && at.in_tables(a) ? s : -1;
    }
    if (t < 0 || t >= a.num_tokens) return -1;
    int s = a.slots[t];
    if constexpr (ROPE != kNoRope) {
      const int p = a.positions[t];
      s = p >= 0 && p < a.max_positions ? s : -1;
    }
    return s >= 0 && s / a.block_size < a.num_blocks ? s : -1;
  };
  const int slot = slot_of(t0 + lane), before = slot_of(t0 + lane - 1);
  const bool next = slot >= 0 && before >= 0 && before + 1 == slot && slot % a.group != 0;
  const uint64_t valid = __builtin_amdgcn_ballot_w64(slot >= 0);
  const uint64_t lead = valid & ~__builtin_amdgcn_ballot_w64(next);
  const uint64_t in = (1ull << a.tile) - 1;
  if ((lead & in) == 0) return;
  const int lo = __builtin_ctzll(lead & in);
  // the tile's last segment ends before the first token past the tile that leads or is not written
  const uint64_t stop = (lead | ~valid) & ~in;
  const int hi = stop ? __builtin_ctzll(stop) : kWave;
  const uint64_t mine = valid & (~0ull << lo) & (hi < kWave ? (1ull << hi) - 1 : ~0ull);
  // chunks: C tokens of one segment from an aligned slot on
  uint64_t full = mine & __builtin_amdgcn_ballot_w64(slot % C == 0);
  const uint64_t follow = mine & ~lead;
#pragma unroll
  for (int i = 1; i < C; ++i) full &= follow >> i;
  uint64_t single = mine;
#pragma unroll
  for (int i = 0; i < C; ++i) single &= ~(full << i);

  // the tokens' rows into LDS, in the pool's type
  const int stride = a.head_size * E + kTileRowPad;
  const void* src = is_v ? a.value : a.key;
  auto row_of = [&](int i) {
    if constexpr (AXES) return (int64_t)(t0 + i) * (is_v ? a.value_stride : a.key_stride) + h * a.head_size;
    else return ((int64_t)(t0 + i) * a.num_kv_heads + h) * a.head_size;
  };
  __shared__ float scale_of[SCALED ? kWave : 1];                // of the tile's rows
  if (ROPE != kNoRope && !is_v) {
    // AXES: the tokens' places, a copy for each wavefront
    __shared__ __attribute__((aligned(16))) Places places[AXES ? kTileThreads : 1];
    Places* of_token = places + (AXES ? tid / kWave * kWave : 0);
    if constexpr (ROPE != kNoRope && AXES) {
      of_token[lane] = Places(a, min(t0 + lane, a.num_tokens - 1));
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    if constexpr (ROPE != kNoRope) {
      const int half = a.head_size / 2, units = half / 8;
      for (int j = tid; j < (hi - lo) * units; j += kTileThreads) {
        const int i = lo + j / units, u = j % units;
        if (!(mine >> i & 1)) continue;
        float c[8], s[8], x[8], y[8];
        if constexpr (AXES) {
          axes_turn(a, of_token[i], u, half, c, s);
        } else {
          const int64_t at = (int64_t)a.positions[t0 + i] * half + 8 * u;
          load8f<Kind::F32>(a.cos_table, at, c);
          load8f<Kind::F32>(a.sin_table, at, s);
        }
        load_unit<SRC, ROPE>(src, row_of(i), u, half, x, y);
        rotate_unit<ROPE>(x, y, c, s);
        if constexpr (SCALED) {
          // a row's units are 8 neighbouring lanes (head_size 128)
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, max(abs_bits(x[e]), abs_bits(y[e])));
          const Fp8Scale sc = fp8_scale_of(lanes_umax<8>(top));
          if (u == 0) scale_of[i] = sc.scale;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = fp32_result(x[e] * sc.inv);
            y[e] = fp32_result(y[e] * sc.inv);
          }
        }
        char* r = tile_rows + i * stride;
        stage8<POOL, SCALED>(r + (ROPE == 0 ? 16 * u : 8 * u) * E, x);
        stage8<POOL, SCALED>(r + (ROPE == 0 ? 16 * u + 8 : half + 8 * u) * E, y);
      }
    }
  } else if constexpr (POOL == Kind::FP8) {
    const int units = a.head_size / 8;
    const float mul = is_v ? a.v_mul : a.k_mul;
    for (int j = tid; j < (hi - lo) * units; j += kTileThreads) {
      const int i = lo + j / units, u = j % units;
      if (!(mine >> i & 1)) continue;
      float x[8], by = mul;
      load8<SRC>(src, row_of(i) + 8 * u, x);
      if constexpr (SCALED) {
        // 16 neighbouring lanes
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[e]));
        const Fp8Scale sc = fp8_scale_of(lanes_umax<16>(top));
        if (u == 0) scale_of[i] = sc.scale;
        by = sc.inv;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fp32_result(x[e] * by);
      stage8<POOL, SCALED>(tile_rows + i * stride + 8 * u, x);
    }
  } else {
    const int units = a.head_size / C;                          // 16 bytes, as they are
    for (int j = tid; j < (hi - lo) * units; j += kTileThreads) {
      const int i = lo + j / units, u = j % units;
      if (!(mine >> i & 1)) continue;
      const u32x4 w = load16((const char*)src + (row_of(i) + u * C) * E);
      uint2* r = reinterpret_cast<uint2*>(tile_rows + i * stride + 16 * u);
      r[0] = make_uint2(w.x, w.y);
      r[1] = make_uint2(w.z, w.w);
    }
  }
  __shared__ int64_t at[kWave];                                 // byte of (token, channel 0) in the pool
  __shared__ uint8_t heads_of[kWave / C];                       // first token of each chunk
  __shared__ uint8_t alone[kWave];
  if (tid < kWave) {
    const uint64_t below = (1ull << lane) - 1;
    const int blk = slot / a.block_size;
    at[lane] = (((int64_t)blk * a.num_kv_heads + h) * a.head_size * a.block_size + (slot - blk * a.block_size)) * E;
    if (full >> lane & 1) heads_of[__builtin_popcountll(full & below)] = (uint8_t)lane;
    if (single >> lane & 1) alone[__builtin_popcountll(single & below)] = (uint8_t)lane;
  }
  __syncthreads();
  if constexpr (SCALED) {
    if (tid < kWave && (mine >> lane & 1))                      // along the slots
      (is_v ? a.v_scales : a.k_scales)[((int64_t)(slot / a.block_size) * a.num_kv_heads + h) * a.block_size +
                                       slot % a.block_size] = scale_of[lane];
  }

  char* pool = is_v ? a.v_cache : a.k_cache;
  const int nf = __builtin_popcountll(full), ns = __builtin_popcountll(single);
  const int64_t channel = (int64_t)a.block_size * E;
  // item j is chunk j % nf of channel j / nf: a store's lanes run along each
  // block's rows.  The quotient by a product is exact for j nf < 65536 (at
  // most 128 channels x 15 chunks of 4-byte elements: 28800).
  const unsigned inv = nf ? 65536u / nf + 1 : 0;
  for (unsigned j = tid; j < (unsigned)(nf * a.head_size); j += kTileThreads) {
    const int c = (int)(j * inv >> 16), i = heads_of[j - c * nf];
    const char* col = tile_rows + i * stride + c * E;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < C; ++e) {
      const char* p = col + e * stride;
      const uint32_t v = E == 1 ? *(const uint8_t*)p : E == 2 ? *(const uint16_t*)p : *(const uint32_t*)p;
      w[e * E / 4] |= v << (8 * (e * E % 4));
    }
    *reinterpret_cast<u32x4*>(pool + at[i] + c * channel) = u32x4{w[0], w[1], w[2], w[3]};
  }
  for (int j = tid / kWave; j < ns; j += kTileThreads / kWave) {
    const int i = alone[j];
    const char* row = tile_rows + i * stride;
    char* d = pool + at[i];
    for (int c = lane; c < a.head_size; c += kWave) {
      if constexpr (E == 1) *(uint8_t*)(d + c * channel) = ((const uint8_t*)row)[c];
      else if constexpr (E == 2) *(uint16_t*)(d + c * channel) = ((const uint16_t*)row)[c];
      else *(uint32_t*)(d + c * channel) = ((const uint32_t*)row)[c];
    }
  }
}

// Slots of a segment's group: a block, or its largest power-of-two part of
// at most 32 slots that holds whole 16-byte chunks.
inline int tile_group(int block_size, int elem) {
  if (block_size <= kTileTokens) return block_size;
  int g = kTileTokens;
  while (block_size % g) g /= 2;
  return g * elem >= 16 ? g : 0;
}

// Workgroups over K and V in tiles of `tile` tokens, and over q.
inline int64_t tile_kv_wgs(const TileAppend& a, int tile) {
  return ((int64_t)a.num_tokens + tile - 1) / tile * a.num_kv_heads * 2;
}
template <bool AXES>
int64_t tile_q_wgs(const TileAppend& a) {
  if constexpr (AXES) {
    if (a.num_heads == 0) return 0;
    const int tokens = axes_q_tokens(a.num_heads, a.head_size);
    return ((int64_t)a.num_tokens + tokens - 1) / tokens;
  }
  const int64_t sets = (a.num_heads + kTileHeadsPerThread - 1) / kTileHeadsPerThread;
  return (a.num_tokens * sets * (a.head_size / 16) + kTileThreads - 1) / kTileThreads;
}

// Whether append_tiles_kernel takes the call: whole 16-byte chunks in a
// block, 16-byte aligned rows and tables, rows that leave LDS for several
// workgroups (63 rows of 512 bytes: 32 KiB), and fewer than 2^32 threads,
// past which a launch wraps (rows below 128 channels take more of them here
// than in the kernels that store elements).
template <bool AXES = false>
bool tile_shape(const TileAppend& a, int src_elem, int elem, bool rope) {
  auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  if (!al(a.key) || !al(a.value) || !al(a.k_cache) || !al(a.v_cache)) return false;
  if (rope && (!al(a.cos_table) || !al(a.sin_table) || !al(a.q) || !al(a.q_out))) return false;
  if (tile_kv_wgs(a, kTileTokens) + (rope ? tile_q_wgs<AXES>(a) : 0) >= (1ll << 32) / kTileThreads) return false;
  return a.block_size * elem % 16 == 0 && tile_group(a.block_size, elem) != 0 && a.head_size * elem <= 512 &&
         (int64_t)a.head_size * src_elem % 16 == 0 && a.head_size * elem % 8 == 0;
}

template <Kind SRC, Kind POOL, int ROPE, bool AXES = false>
int launch_tiles(TileAppend a, hipStream_t stream) {
  constexpr int E = KindInfo<POOL>::bytes;
  a.group = tile_group(a.block_size, E);
  // Shorter tiles where those of 32 tokens are fewer than the CUs: a tile of
  // tokens that fill no chunk is a serial 4096 stores of an element.  2 heads,
  // 257 tokens, each in a block of its own 5.6 us in tiles of 32, 4.1 of 8
  // (reshape_copy_kernel 5.0), in runs of 4 5.2 and 3.7 (4.2), consecutive 3.6
  // and 3.2 (4.1); 8 heads, 512 tokens, 10.6 in tiles of 32, 10.2 of 16 (10.2),
  // consecutive 3.8 and 3.6 (9.4).  Past the line 8 heads, 900 consecutive,
  // rotated 5.6 in tiles of 32, 7.0 of 16.
  const int64_t full = tile_kv_wgs(a, kTileTokens);
  a.tile = full <= 64 ? 8 : full <= 256 ? 16 : kTileTokens;
  a.kv_wgs = (int)tile_kv_wgs(a, a.tile);
  const unsigned grid = (unsigned)(a.kv_wgs + (ROPE != kNoRope ? tile_q_wgs<AXES>(a) : 0));
  const size_t lds = (size_t)(a.tile + a.group - 1) * (a.head_size * E + kTileRowPad);
  hipLaunchKernelGGL((append_tiles_kernel<SRC, POOL, ROPE, AXES>), dim3(grid), dim3(kTileThreads), lds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : 5;
}

}  // namespace tl
