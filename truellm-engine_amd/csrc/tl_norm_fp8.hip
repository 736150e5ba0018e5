// tl_norm_fp8.hip -- RMSNorm, and residual add + RMSNorm, with the output in
// FP8 E4M3 and its scales: what the product behind the norm takes, in one
// pass over the row.
//
//   r = x (+ res; res = T(r) in place),  inv = 1 / sqrt(sum(r^2) / H + eps)
//   y = float(T(r)) * inv * w                           (fp32, not rounded)
//   scale = max|y| / 448 over the row or over each group of channels
//   code  = e4m3(y / scale), round to nearest even
// sum(r^2) is over the unrounded fp32 r, as in the norm with a 2-byte output
// (layernorm_kernels.cu:64-94).  The scale's convention is that of
// per_token_fp8_quant_kernel (fp8_gemm.cu:80-93), which reads the rounded
// output of a norm before it; here y is rounded once, to the code.
#include "tl_device.hpp"
#include "tl_fp8.hpp"
#include "tl_internal.hpp"
#include "tl_row.hpp"

namespace tl {

namespace {

// Max over the workgroup of the bits of magnitudes, returned to every thread.
__device__ __forceinline__ uint32_t block_umax(uint32_t v, uint32_t* s_part) {
  v = lanes_umax<kWave>(v);
  __syncthreads();                                   // s_part free from a previous use
  if (threadIdx.x % kWave == 0) s_part[threadIdx.x / kWave] = v;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int w = 0; w < kNormThreads / kWave; ++w) t = max(t, s_part[w]);
  return t;
}

// Rows of up to TPR x 8 C elements, a multiple of 8, read once and held in
// registers: TPR threads on a row, C chunks of 8 elements each, every load of
// the row in flight before the first is used.  A group's channels lie on
// group / 8 neighbouring lanes, so its maximum takes 2 to 5 lane steps and no
// LDS.  Rows of at most 1024 elements take a wavefront each (TPR 64, no
// barrier), longer ones a workgroup.
//
// Bound by HBM from a few hundred rows on, by its round trips below.  4096
// rows of 8192, bf16, residual added, scales per 128 channels: 49.3 us, 4.79
// TB/s of the 4.99 a large copy reaches (rms_norm_fp8_kernel, which reads the
// row four times, 138 us).
template <Kind K, int C, int TPR>
__global__ __launch_bounds__(kNormThreads) void rms_norm_fp8_rows_kernel(NormFp8 a, int64_t row0) {
  __shared__ float s_sum[kNormThreads / kWave];
  __shared__ uint32_t s_max[kNormThreads / kWave];
  static_assert(TPR == kWave || TPR == kNormThreads, "a wavefront or a workgroup on a row");
  const int64_t row = row0 + (int64_t)blockIdx.x * (kNormThreads / TPR) + threadIdx.x / TPR;
  if (row >= a.rows) return;                          // with a workgroup on a row: none
  const int t = threadIdx.x % TPR;
  const int64_t base = row * a.hidden;
  const bool add = a.residual != nullptr;
  Raw8<K> rx[C], rr[C], rw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i0 = (c * TPR + t) * 8;
    if (i0 >= a.hidden) break;
    rx[c].load(a.x, base + i0);
    if (add) rr[c].load(a.residual, base + i0);
  }
  // the weights with the row while the registers allow, else once it is summed
  constexpr bool kEarly = C * KindInfo<K>::bytes <= 8;
  auto load_weight = [&]() {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i0 = (c * TPR + t) * 8;
      if (i0 >= a.hidden) break;
      rw[c].load(a.weight, i0);
    }
  };
  if constexpr (kEarly) load_weight();
  float v[C][8];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i0 = (c * TPR + t) * 8;
    if (i0 >= a.hidden) break;
    rx[c].get(v[c]);
    if (add) {
      float r[8];
      rr[c].get(r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float sum = v[c][j] + r[j];
        ss = __builtin_fmaf(sum, sum, ss);
        v[c][j] = round_to<K>(sum);
      }
      store8<K>(a.residual, base + i0, v[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(v[c][j], v[c][j], ss);
    }
  }
  if constexpr (!kEarly) load_weight();
  const float total = TPR == kWave ? wave_total(ss) : block_sum(ss, s_sum);
  const float inv = 1.0f / __builtin_sqrtf(total / (float)a.hidden + a.eps);
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i0 = (c * TPR + t) * 8;
    if (i0 >= a.hidden) break;
    float w[8];
    rw[c].get(w);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[c][j] = v[c][j] * inv * w[j];
      m = max(m, abs_bits(v[c][j]));
    }
    if (a.group == 0) {
      top = max(top, m);
      continue;
    }
    m = lanes_umax<4>(m);
    if (a.group >= 64) m = max(m, lane_bits<kDppHalfMirror>(m));
    if (a.group >= 128) m = max(m, lane_bits<kDppMirror>(m));
    if (a.group >= 256) m = lanes_umax_16(m);
    const Fp8Scale s = fp8_scale_of(m);
    if (i0 % a.group == 0) a.scales[row * (a.hidden / a.group) + i0 / a.group] = s.scale;
    *reinterpret_cast<uint2*>(a.out + base + i0) =
        make_uint2(pack4_fp8_found(v[c][0] * s.inv, v[c][1] * s.inv, v[c][2] * s.inv, v[c][3] * s.inv),
                   pack4_fp8_found(v[c][4] * s.inv, v[c][5] * s.inv, v[c][6] * s.inv, v[c][7] * s.inv));
  }
  if (a.group != 0) return;
  const Fp8Scale s = fp8_scale_of(TPR == kWave ? lanes_umax<kWave>(top) : block_umax(top, s_max));
  if (t == 0) a.scales[row] = s.scale;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i0 = (c * TPR + t) * 8;
    if (i0 >= a.hidden) break;
    *reinterpret_cast<uint2*>(a.out + base + i0) =
        make_uint2(pack4_fp8_found(v[c][0] * s.inv, v[c][1] * s.inv, v[c][2] * s.inv, v[c][3] * s.inv),
                   pack4_fp8_found(v[c][4] * s.inv, v[c][5] * s.inv, v[c][6] * s.inv, v[c][7] * s.inv));
  }
}

// Any size, alignment and type: a workgroup per row, an element per thread
// at a time; the groups of a row go to its wavefronts in turn.
template <Kind K>
__global__ __launch_bounds__(kNormThreads) void rms_norm_fp8_kernel(NormFp8 a, int64_t row0) {
  __shared__ float s_sum[kNormThreads / kWave];
  __shared__ uint32_t s_max[kNormThreads / kWave];
  const int64_t row = row0 + blockIdx.x, base = row * a.hidden;
  float ss = 0.f;
  for (int i = threadIdx.x; i < a.hidden; i += kNormThreads) {
    float v = load_scalar<K>(a.x, base + i);
    if (a.residual) {
      v += load_scalar<K>(a.residual, base + i);
      store_scalar<K>(a.residual, base + i, v);
    }
    ss = __builtin_fmaf(v, v, ss);
  }
  const float inv = 1.0f / __builtin_sqrtf(block_sum(ss, s_sum) / (float)a.hidden + a.eps);
  const void* src = a.residual ? a.residual : a.x;
  auto y = [&](int i) { return load_scalar<K>(src, base + i) * inv * load_scalar<K>(a.weight, i); };
  if (a.group == 0) {
    uint32_t m = 0;
    for (int i = threadIdx.x; i < a.hidden; i += kNormThreads) m = max(m, abs_bits(y(i)));
    const Fp8Scale s = fp8_scale_of(block_umax(m, s_max));
    if (threadIdx.x == 0) a.scales[row] = s.scale;
    for (int i = threadIdx.x; i < a.hidden; i += kNormThreads) a.out[base + i] = f32_to_fp8(y(i) * s.inv);
    return;
  }
  // the rows' elements that another thread of this workgroup stored above
  // are read below: visible after the barriers of block_sum
  const int lane = threadIdx.x % kWave, groups = a.hidden / a.group;
  for (int g = threadIdx.x / kWave; g < groups; g += kNormThreads / kWave) {
    uint32_t m = 0;
    for (int i = lane; i < a.group; i += kWave) m = max(m, abs_bits(y(g * a.group + i)));
    const Fp8Scale s = fp8_scale_of(lanes_umax<kWave>(m));
    if (lane == 0) a.scales[row * groups + g] = s.scale;
    for (int i = lane; i < a.group; i += kWave)
      a.out[base + g * a.group + i] = f32_to_fp8(y(g * a.group + i) * s.inv);
  }
}

// The rows of a launch, fewer than 2^32 threads: `wg_rows` of them to a workgroup.
template <class Kernel>
void launch_rows(Kernel kernel, const NormFp8& a, int wg_rows, hipStream_t stream) {
  constexpr int64_t kWgs = 1 << 23;
  for (int64_t r = 0; r < a.rows; r += kWgs * wg_rows) {
    const int64_t wgs = (a.rows - r + wg_rows - 1) / wg_rows;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wgs < kWgs ? wgs : kWgs)), dim3(kNormThreads), 0, stream, a, r);
  }
}

template <Kind K>
int launch_typed(const NormFp8& a, hipStream_t stream) {
  const auto al = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  if (a.hidden % 8 || a.hidden > 8 * 8 * kNormThreads || !al(a.x, 16) || !al(a.weight, 16) || !al(a.residual, 16) ||
      !al(a.out, 8)) {
    launch_rows(rms_norm_fp8_kernel<K>, a, 1, stream);
    return hipGetLastError() == hipSuccess ? 0 : 5;
  }
  if (a.hidden <= 8 * kWave) launch_rows(rms_norm_fp8_rows_kernel<K, 1, kWave>, a, kNormThreads / kWave, stream);
  else if (a.hidden <= 16 * kWave) launch_rows(rms_norm_fp8_rows_kernel<K, 2, kWave>, a, kNormThreads / kWave, stream);
  else {
    switch ((a.hidden + 8 * kNormThreads - 1) / (8 * kNormThreads)) {
      case 1: launch_rows(rms_norm_fp8_rows_kernel<K, 1, kNormThreads>, a, 1, stream); break;
      case 2: launch_rows(rms_norm_fp8_rows_kernel<K, 2, kNormThreads>, a, 1, stream); break;
      case 3: launch_rows(rms_norm_fp8_rows_kernel<K, 3, kNormThreads>, a, 1, stream); break;
      case 4: launch_rows(rms_norm_fp8_rows_kernel<K, 4, kNormThreads>, a, 1, stream); break;
      case 5: case 6: launch_rows(rms_norm_fp8_rows_kernel<K, 6, kNormThreads>, a, 1, stream); break;
      default: launch_rows(rms_norm_fp8_rows_kernel<K, 8, kNormThreads>, a, 1, stream); break;
    }
  }
  return hipGetLastError() == hipSuccess ? 0 : 5;
}

}  // namespace

int launch_rms_norm_fp8(const NormFp8& a, hipStream_t stream) {
  if (a.dtype == (int)Kind::F16) return launch_typed<Kind::F16>(a, stream);
  if (a.dtype == (int)Kind::BF16) return launch_typed<Kind::BF16>(a, stream);
  if (a.dtype == (int)Kind::F32) return launch_typed<Kind::F32>(a, stream);
  return 3;
}

}  // namespace tl
