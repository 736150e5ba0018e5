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

}  // namespace

int launch_rms_norm_fp8(const NormFp8& a, hipStream_t stream) {
  // rows of a launch: fewer than 2^32 threads
  constexpr int64_t kRows = 1 << 23;
  for (int64_t r = 0; r < a.rows; r += kRows) {
    const dim3 grid((unsigned)(a.rows - r < kRows ? a.rows - r : kRows));
    if (a.dtype == (int)Kind::F16)
      hipLaunchKernelGGL(rms_norm_fp8_kernel<Kind::F16>, grid, dim3(kNormThreads), 0, stream, a, r);
    else if (a.dtype == (int)Kind::BF16)
      hipLaunchKernelGGL(rms_norm_fp8_kernel<Kind::BF16>, grid, dim3(kNormThreads), 0, stream, a, r);
    else if (a.dtype == (int)Kind::F32)
      hipLaunchKernelGGL(rms_norm_fp8_kernel<Kind::F32>, grid, dim3(kNormThreads), 0, stream, a, r);
    else
      return 3;
  }
  return hipGetLastError() == hipSuccess ? 0 : 5;
}

}  // namespace tl
