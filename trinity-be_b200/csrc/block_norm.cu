// The seam between two blocks of a residual network, in one pass over the rows:
//
//   b = x                                       or  x / sqrt(mean(x^2) + post_eps) * post_gain
//   h = residual_scale * residual + gate * b        -> residual_out
//   y = h / sqrt(mean(h^2) + eps) * gain            -> out
//
// Bound by memory: x, the residual and a full gate are read once, residual_out and out written
// once.  A row is spread over kThreads lanes (32..1024) of 16 elements each (8 where the layout
// allows only one at a time); the lane keeps its part of the row in registers through both sums, so
// nothing is read twice.  Warps in flight decide: with 16-byte accesses 48 warps an SM (40 registers a
// thread, and 20 to 32 bytes of spills) take 170 us for 32768 x 4096 BF16 (1074 MB, 0.96 of the measured copy
// rate; 187 to 195 in passes issued one by one), 36 warps 184 us and 56 warps (spilling more) 205 us.  With FP32
// operands, 32 warps: 240 us for an FP32 stream (1611 MB), 279 with x in FP32 too.  All arithmetic is FP32; the two roundings are those of the
// two outputs (out is computed from the unrounded h).
#include "host_common.h"
#include "sm100_ptx.cuh"

namespace trinity_sm100 {
namespace {

constexpr int kSeamMaxCols = 1024 * 16;

struct SeamParams {
  const void* x;
  const void* residual;
  const __nv_bfloat16* gate;
  const __nv_bfloat16* gain;
  const __nv_bfloat16* post_gain;
  void* residual_out;
  __nv_bfloat16* out;
  long long rows, ld_x, ld_residual, ld_residual_out, ld_out, gate_row, gate_col;
  int cols, post_norm;
  float eps, post_eps, residual_scale;
};

// kW consecutive elements as FP32 (one 16-byte load for eight BF16 values, two for FP32), `at` elements
// behind the lane's first one.  Rows are read once and leave the caches first; gain vectors
// (kStream false) serve every row.
template <int kW, bool kF32, bool kStream = true>
__device__ __forceinline__ void load_elements(const void* base, int at, float (&v)[kW]) {
  if (kF32) {
    const float* p = static_cast<const float*>(base) + at;
    if (kW == 8) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
      const float4 b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1 % kW] = a.y; v[2 % kW] = a.z; v[3 % kW] = a.w;
      v[4 % kW] = b.x; v[5 % kW] = b.y; v[6 % kW] = b.z; v[7 % kW] = b.w;
    } else {
      v[0] = __ldcs(p);
    }
  } else {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + at;
    if (kW == 8) {
      const uint4 a = kStream ? __ldcs(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[(2 * e) % kW] = bf16_lo(w[e]);
        v[(2 * e + 1) % kW] = bf16_hi(w[e]);
      }
    } else {
      v[0] = __bfloat162float(*p);
    }
  }
}

template <int kW, bool kF32>
__device__ __forceinline__ void store_elements(void* base, int at, const float (&v)[kW]) {
  if (kF32) {
    float* p = static_cast<float*>(base) + at;
    if (kW == 8) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1 % kW], v[2 % kW], v[3 % kW]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4 % kW], v[5 % kW], v[6 % kW], v[7 % kW]);
    } else {
      p[0] = v[0];
    }
  } else {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + at;
    if (kW == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1 % kW]), pack_bf16x2(v[2 % kW], v[3 % kW]),
                                                pack_bf16x2(v[4 % kW], v[5 % kW]), pack_bf16x2(v[6 % kW], v[7 % kW]));
    else
      p[0] = __float2bfloat16(v[0]);
  }
}

template <bool kF32>
__device__ __forceinline__ const void* element_of(const void* base, long long offset) {
  return kF32 ? static_cast<const void*>(static_cast<const float*>(base) + offset)
              : static_cast<const void*>(static_cast<const __nv_bfloat16*>(base) + offset);
}

// Threads an SM is to hold, which bounds the registers of each (see above; FP32 operands need more).
template <int kW, bool kF32>
constexpr int seam_resident() { return kW == 1 ? 2048 : kF32 ? 1024 : 1536; }
// kW = 8: 16-byte accesses (every row of every operand starts on 16 bytes); kW = 1: any layout.
// kElements a lane.
template <int kThreads, int kW, int kElements, bool kXF32, bool kResF32>
__global__ void __launch_bounds__(kThreads > kRowBlock ? kThreads : kRowBlock, (kElements > 8 && kW == 1 ? 1 : seam_resident<kW, kXF32 || kResF32>() / (kThreads > kRowBlock ? kThreads : kRowBlock)))
rmsnorm_residual_kernel(const SeamParams p) {
  constexpr int kBlock = kThreads > kRowBlock ? kThreads : kRowBlock;
  constexpr int kRowsPerCta = kBlock / kThreads;
  constexpr int kN = kElements / kW;
  constexpr int kStep = kThreads * kW;     // columns between a lane's pieces
  __shared__ float scratch[kBlock / 32];
  grid_dependents_may_launch();
  grid_dependency_wait();   // the previous kernel of the stream may have produced any operand
  const int col = threadIdx.x % kThreads * kW;       // of the lane's first piece
  const long long row = static_cast<long long>(blockIdx.x) * kRowsPerCta + threadIdx.x / kThreads;
  // columns from the lane's first on; a lane without a row has none
  const int left = row < p.rows ? p.cols - col : 0;
  const long long at_row = row < p.rows ? row : 0;
  const void* x = element_of<kXF32>(p.x, at_row * p.ld_x + col);
  const void* residual = element_of<kResF32>(p.residual, at_row * p.ld_residual + col);
  float h[kN][kW], r[kN][kW];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
#pragma unroll
    for (int e = 0; e < kW; ++e) h[i][e] = r[i][e] = 0.0f;
    if (i * kStep >= p.cols) continue;       // (for all lanes: pieces behind the row cost nothing)
    if (i * kStep < left) {
      load_elements<kW, kXF32>(x, i * kStep, h[i]);
      load_elements<kW, kResF32>(residual, i * kStep, r[i]);
    }
  }
  if (p.post_norm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int e = 0; e < kW; ++e) ss = fmaf(h[i][e], h[i][e], ss);
    ss = row_reduce<kThreads, false>(ss, scratch);
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.cols) + p.post_eps);
    const __nv_bfloat16* gain = p.post_gain + col;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (i * kStep >= p.cols) continue;
      float g[kW];
#pragma unroll
      for (int e = 0; e < kW; ++e) g[e] = 1.0f;
      if (p.post_gain && i * kStep < left) load_elements<kW, false, false>(gain, i * kStep, g);
#pragma unroll
      for (int e = 0; e < kW; ++e) h[i][e] = h[i][e] * inv * g[e];
    }
  }
  float ss = 0.0f;
  const __nv_bfloat16* gate = p.gate + at_row * p.gate_row + col * p.gate_col;
  const float row_gate = p.gate && !p.gate_col ? __bfloat162float(*gate) : 1.0f;
  void* residual_out = const_cast<void*>(element_of<kResF32>(p.residual_out, at_row * p.ld_residual_out + col));
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if (i * kStep >= p.cols) continue;
    if (i * kStep < left) {
      float g[kW];
#pragma unroll
      for (int e = 0; e < kW; ++e) g[e] = row_gate;
      if (p.gate && p.gate_col) load_elements<kW, false, false>(gate, i * kStep, g);
#pragma unroll
      for (int e = 0; e < kW; ++e) {
        h[i][e] = fmaf(p.residual_scale, r[i][e], h[i][e] * g[e]);
        ss = fmaf(h[i][e], h[i][e], ss);
      }
      store_elements<kW, kResF32>(residual_out, i * kStep, h[i]);
    }
  }
  ss = row_reduce<kThreads, false>(ss, scratch);
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.cols) + p.eps);
  const __nv_bfloat16* gain = p.gain + col;
  __nv_bfloat16* out = p.out + at_row * p.ld_out + col;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if (i * kStep >= p.cols) continue;
    if (i * kStep < left) {
      float g[kW];
#pragma unroll
      for (int e = 0; e < kW; ++e) g[e] = 1.0f;
      if (p.gain) load_elements<kW, false, false>(gain, i * kStep, g);
#pragma unroll
      for (int e = 0; e < kW; ++e) g[e] *= h[i][e] * inv;
      store_elements<kW, false>(out, i * kStep, g);
    }
  }
}

template <int kThreads, int kW, int kElements>
cudaError_t launch_seam(const SeamParams& p, bool x_f32, bool res_f32, cudaStream_t stream) {
  constexpr int block = kThreads > kRowBlock ? kThreads : kRowBlock;
  const unsigned grid = unsigned((p.rows + block / kThreads - 1) / (block / kThreads));
  KernelLaunch launch(dim3(grid), dim3(block), 0, stream);
  if (x_f32)
    return res_f32 ? cudaLaunchKernelEx(&launch.config, rmsnorm_residual_kernel<kThreads, kW, kElements, true, true>, p)
                   : cudaLaunchKernelEx(&launch.config, rmsnorm_residual_kernel<kThreads, kW, kElements, true, false>, p);
  return res_f32 ? cudaLaunchKernelEx(&launch.config, rmsnorm_residual_kernel<kThreads, kW, kElements, false, true>, p)
                 : cudaLaunchKernelEx(&launch.config, rmsnorm_residual_kernel<kThreads, kW, kElements, false, false>, p);
}

template <int kW, int kElements>
cudaError_t launch_seam_width(const SeamParams& p, bool x_f32, bool res_f32, cudaStream_t stream) {
  if (p.cols <= 32 * kElements) return launch_seam<32, kW, kElements>(p, x_f32, res_f32, stream);
  if (p.cols <= 64 * kElements) return launch_seam<64, kW, kElements>(p, x_f32, res_f32, stream);
  if (p.cols <= 128 * kElements) return launch_seam<128, kW, kElements>(p, x_f32, res_f32, stream);
  if (p.cols <= 256 * kElements) return launch_seam<256, kW, kElements>(p, x_f32, res_f32, stream);
  if (p.cols <= 512 * kElements) return launch_seam<512, kW, kElements>(p, x_f32, res_f32, stream);
  return launch_seam<1024, kW, kElements>(p, x_f32, res_f32, stream);
}

}  // namespace
}  // namespace trinity_sm100

using namespace trinity_sm100;

extern "C" int trinity_sm100_rmsnorm_residual(const trinity_sm100_rmsnorm_residual_args* args, void* stream_handle) {
  if (!args) return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: null argument block");
  const trinity_sm100_rmsnorm_residual_args& a = *args;
  if (!a.x || !a.residual || !a.residual_out || !a.out)
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: null pointer");
  if (a.rows <= 0 || a.cols <= 0) return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: empty extent");
  if (a.cols > kSeamMaxCols)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "rmsnorm_residual: cols (%lld) above the %d a CTA keeps in registers",
                (long long)a.cols, kSeamMaxCols);
  if (a.rows > INT32_MAX) return fail(TRINITY_SM100_E_UNSUPPORTED, "rmsnorm_residual: too many rows");
  if (a.x_dtype != TRINITY_SM100_BF16 && a.x_dtype != TRINITY_SM100_FP32)
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: unknown dtype %d of x", a.x_dtype);
  if (a.residual_dtype != TRINITY_SM100_BF16 && a.residual_dtype != TRINITY_SM100_FP32)
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: unknown dtype %d of the residual", a.residual_dtype);
  if (a.ld_x < a.cols || a.ld_residual < a.cols || a.ld_residual_out < a.cols || a.ld_out < a.cols)
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: leading dimension smaller than the row");
  if (a.gate && (a.gate_row_stride < 0 || (a.gate_col_stride != 0 && a.gate_col_stride != 1) ||
                 (a.gate_col_stride == 1 && a.gate_row_stride != 0 && a.gate_row_stride < a.cols)))
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: gate strides (%lld, %lld)", (long long)a.gate_row_stride,
                (long long)a.gate_col_stride);
  if (a.residual_out == a.out) return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: the two outputs share memory");
  const bool x_f32 = a.x_dtype == TRINITY_SM100_FP32, res_f32 = a.residual_dtype == TRINITY_SM100_FP32;
  const size_t x_size = x_f32 ? 4 : 2, res_size = res_f32 ? 4 : 2;
  auto aligned_to = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  if (!aligned_to(a.x, x_size) || !aligned_to(a.residual, res_size) || !aligned_to(a.residual_out, res_size) ||
      !aligned_to(a.out, 2) || !aligned_to(a.gate, 2) || !aligned_to(a.gain, 2) || !aligned_to(a.post_gain, 2))
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: a pointer is not aligned to its element type");
  // an output may take the place of an input element for element, not with another pitch or type
  if ((a.residual_out == a.residual && a.ld_residual_out != a.ld_residual) ||
      (a.residual_out == a.x && (a.ld_residual_out != a.ld_x || x_f32 != res_f32)) ||
      (a.out == a.x && (a.ld_out != a.ld_x || x_f32)) || (a.out == a.residual && (a.ld_out != a.ld_residual || res_f32)))
    return fail(TRINITY_SM100_E_INVALID, "rmsnorm_residual: an output overlaps an input with another layout");
  if (int rc = require_sm100(nullptr)) return rc;
  SeamParams p;
  p.x = a.x;
  p.residual = a.residual;
  p.gate = static_cast<const __nv_bfloat16*>(a.gate);
  p.gain = static_cast<const __nv_bfloat16*>(a.gain);
  p.post_gain = static_cast<const __nv_bfloat16*>(a.post_gain);
  p.residual_out = a.residual_out;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.rows = a.rows;
  p.ld_x = a.ld_x;
  p.ld_residual = a.ld_residual;
  p.ld_residual_out = a.ld_residual_out;
  p.ld_out = a.ld_out;
  p.gate_row = a.gate_row_stride;
  p.gate_col = a.gate_col_stride;
  p.cols = int(a.cols);
  p.post_norm = a.post_norm != 0 || a.post_gain != nullptr;
  p.eps = a.eps;
  p.post_eps = a.post_eps;
  p.residual_scale = a.residual_scale;
  // 16-byte accesses where every row of every operand starts on 16 bytes; one element at a time otherwise
  const bool vectors = a.cols % 8 == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.residual_out) &&
                       aligned16(a.out) && aligned16(a.gain) && aligned16(a.post_gain) &&
                       (a.ld_x * x_size) % 16 == 0 && (a.ld_residual * res_size) % 16 == 0 &&
                       (a.ld_residual_out * res_size) % 16 == 0 && a.ld_out % 8 == 0 &&
                       (a.gate_col_stride == 0 || !a.gate || (aligned16(a.gate) && a.gate_row_stride % 8 == 0));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const cudaError_t e = vectors             ? launch_seam_width<8, 16>(p, x_f32, res_f32, stream)
                        : a.cols <= 8 * 1024 ? launch_seam_width<1, 8>(p, x_f32, res_f32, stream)
                                             : launch_seam<1024, 1, 16>(p, x_f32, res_f32, stream);
  if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "rmsnorm_residual launch: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("rmsnorm_residual");
}
