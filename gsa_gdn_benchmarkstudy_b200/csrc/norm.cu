// norm.cu — root-mean-square norm with the residual's addition, its backward
// pass, and the variant whose output is held in 8 bits (e4m3) with scales.
//
//   h = round(x + residual)            (the inputs' type; h = x without a residual)
//   r = 1 / sqrt(mean_j h_j^2 + eps),  y_j = h_j r w_j
// fp8:  s = max |y| / 448 over a row or over 128 values, y8_j = e4m3(y_j * (448 / max |y|))
// back: p = dy w,  dx = dresidual = r (p - h r^2 mean_j(p h)) + dh,  dw_j = sum_rows dy_j h_j r
//
// h is rounded once, to the inputs' type, because it is the tensor the next
// layer adds to: the norm of it equals a separate addition followed by a norm.
// Everything else (sums, r, y before its rounding, dw's partial sums) is fp32.
//
// The norm is bound by HBM: 4 * rows * width * 2 bytes in bf16 with a residual.
// A row is read once and stays in registers between its sum and its output
// (threads_per_row x NV vectors of 8 values), so nothing is read twice.
#include <cuda_fp8.h>

#include "kernels.h"

namespace gsa {
namespace {

constexpr int kVec = 8;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E> __device__ __forceinline__ E from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
__device__ __forceinline__ float round_f(float v, float) { return v; }
__device__ __forceinline__ float round_f(float v, __nv_bfloat16) { return bf16_round(v); }

// Column of value e of a thread's vector i.  Vector form: 8 neighbours, so a
// thread moves 16 bytes (bf16) at once.  Plain form (a width or an address that
// breaks the 16-byte rule): neighbours go to neighbouring threads.
template <bool VECTOR>
__device__ __forceinline__ int column(int i, int e, int t, int tpr) {
  return VECTOR ? (i * tpr + t) * kVec + e : (i * kVec + e) * tpr + t;
}

template <bool VECTOR, typename E>
__device__ __forceinline__ void load8(float (&v)[kVec], const E* row, int i, int t, int tpr,
                                      int width) {
  if constexpr (VECTOR) {
    const int c = column<true>(i, 0, t, tpr);
    if (c < width) {
      if constexpr (sizeof(E) == 2) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + c);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
      } else {
        const float4 a = *reinterpret_cast<const float4*>(row + c);
        const float4 b = *reinterpret_cast<const float4*>(row + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int c = column<false>(i, e, t, tpr);
      v[e] = c < width ? to_f(row[c]) : 0.f;
    }
  }
}

template <bool VECTOR, typename E>
__device__ __forceinline__ void store8(const float (&v)[kVec], E* row, int i, int t, int tpr,
                                       int width) {
  if constexpr (VECTOR) {
    const int c = column<true>(i, 0, t, tpr);
    if (c >= width) return;
    if constexpr (sizeof(E) == 2) {
      uint4 raw;
      raw.x = pack_bf16x2(v[0], v[1]);
      raw.y = pack_bf16x2(v[2], v[3]);
      raw.z = pack_bf16x2(v[4], v[5]);
      raw.w = pack_bf16x2(v[6], v[7]);
      *reinterpret_cast<uint4*>(row + c) = raw;
    } else {
      *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int c = column<false>(i, e, t, tpr);
      if (c < width) row[c] = from_f<E>(v[e]);
    }
  }
}

template <bool VECTOR>
__device__ __forceinline__ void store8_e4m3(const float (&v)[kVec], uint8_t* row, int i, int t,
                                            int tpr, int width) {
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lo |= uint32_t(__nv_cvt_float_to_fp8(v[e], __NV_SATFINITE, __NV_E4M3)) << (8 * e);
    hi |= uint32_t(__nv_cvt_float_to_fp8(v[e + 4], __NV_SATFINITE, __NV_E4M3)) << (8 * e);
  }
  if constexpr (VECTOR) {
    const int c = column<true>(i, 0, t, tpr);
    if (c < width) *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int c = column<false>(i, e, t, tpr);
      if (c < width) row[c] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
  }
}

__device__ __forceinline__ float fold_sum(float a, float b) { return a + b; }
// A NaN wins over every number, so that a row that holds one gets a NaN scale.
__device__ __forceinline__ float fold_max(float a, float b) { return a > b || a != a ? a : b; }

// Sum or maximum over the threads of a row (tpr a multiple of 32; rows of one
// warp need no barrier).  `slot` has room for 32 values and is not used again
// before the caller's next barrier.
template <bool MAX>
__device__ __forceinline__ float row_fold(float v, float* slot, int tpr) {
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const float o = __shfl_xor_sync(0xFFFFFFFFu, v, m);
    v = MAX ? fold_max(v, o) : fold_sum(v, o);
  }
  if (tpr == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  v = lane < nw ? slot[lane] : 0.f;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const float o = __shfl_xor_sync(0xFFFFFFFFu, v, m);
    v = MAX ? fold_max(v, o) : fold_sum(v, o);
  }
  return v;
}

enum NormOut { kNormPlain = 0, kNormRow8 = 1, kNormGroup8 = 2 };

// tpr threads share a row; a block holds blockDim.x / tpr rows (more than one
// only where a row is one warp).
template <typename E, bool VECTOR, int NV, int OUT, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_kernel(RmsNormArgs a, int tpr) {
  __shared__ float slots[2][32];
  const int t = threadIdx.x % tpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  if (row >= a.rows) return;  // whole warps only: a row of several warps is its block's one row
  const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
  const E* res = a.residual ? static_cast<const E*>(a.residual) + row * a.residual_stride : nullptr;
  float v[NV][kVec];
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<VECTOR>(v[i], x, i, t, tpr, a.width);
  if (res) {
    float r[NV][kVec];
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<VECTOR>(r[i], res, i, t, tpr, a.width);
    E* h = static_cast<E*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[i][e] = round_f(v[i][e] + r[i][e], E());
      store8<VECTOR>(v[i], h, i, t, tpr, a.width);
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) s = fmaf(v[i][e], v[i][e], s);
  s = row_fold<false>(s, slots[0], tpr);
  const float rstd = 1.0f / sqrtf(s / static_cast<float>(a.width) + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[kVec];
    if (a.weight_f32)
      load8<VECTOR>(w, static_cast<const float*>(a.weight), i, t, tpr, a.width);
    else
      load8<VECTOR>(w, static_cast<const __nv_bfloat16*>(a.weight), i, t, tpr, a.width);
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[i][e] = v[i][e] * rstd * w[e];
  }
  if constexpr (OUT == kNormPlain) {
    E* y = static_cast<E*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<VECTOR>(v[i], y, i, t, tpr, a.width);
  } else {
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride;
    float most = 0.f;
    if constexpr (OUT == kNormRow8) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) most = fold_max(fabsf(v[i][e]), most);
      most = fold_max(row_fold<true>(most, slots[1], tpr), 1e-12f);
      if (t == 0) a.scale[row] = most / 448.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (OUT == kNormGroup8) {  // 16 neighbouring lanes hold a group's 128 values
        most = 0.f;
#pragma unroll
        for (int e = 0; e < kVec; ++e) most = fold_max(fabsf(v[i][e]), most);
#pragma unroll
        for (int m = 8; m; m >>= 1) most = fold_max(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
        most = fold_max(most, 1e-12f);
        const int c = column<true>(i, 0, t, tpr);
        if (c < a.width && (t & 15) == 0) a.scale[row * (a.width >> 7) + (c >> 7)] = most / 448.0f;
      }
      const float inv = 448.0f / most;
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[i][e] *= inv;
      store8_e4m3<VECTOR>(v[i], y, i, t, tpr, a.width);
    }
  }
}

// Backward: block b takes the rows b, b + gridDim.x, ... and keeps its columns'
// share of dw in registers over all of them; the shares go to partial[b] and
// are added in block order by rms_norm_dw_kernel, so equal inputs give equal
// bits.  The next row's loads are in flight while a row's sum crosses the block.
template <typename E, bool VECTOR, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_backward_kernel(RmsNormBackwardArgs a) {
  __shared__ float slots[2][32];
  const int tpr = blockDim.x, t = threadIdx.x;
  float dw[NV][kVec] = {};
  float w[NV][kVec];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.weight_f32)
      load8<VECTOR>(w[i], static_cast<const float*>(a.weight), i, t, tpr, a.width);
    else
      load8<VECTOR>(w[i], static_cast<const __nv_bfloat16*>(a.weight), i, t, tpr, a.width);
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = a.rstd[row];
    float h[NV][kVec], dy[NV][kVec], d[NV][kVec];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load8<VECTOR>(h[i], static_cast<const E*>(a.h) + row * a.h_stride, i, t, tpr, a.width);
      load8<VECTOR>(dy[i], static_cast<const E*>(a.dy) + row * a.dy_stride, i, t, tpr, a.width);
      if (a.dh)
        load8<VECTOR>(d[i], static_cast<const E*>(a.dh) + row * a.dh_stride, i, t, tpr, a.width);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) s = fmaf(dy[i][e] * w[i][e], h[i][e], s);
    s = row_fold<false>(s, slots[turn], tpr);
    const float back = rstd * rstd * (s / static_cast<float>(a.width));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        dw[i][e] = fmaf(dy[i][e], h[i][e] * rstd, dw[i][e]);
        const float g = rstd * (dy[i][e] * w[i][e] - h[i][e] * back);
        h[i][e] = a.dh ? g + d[i][e] : g;
      }
      store8<VECTOR>(h[i], static_cast<E*>(a.dx) + row * a.dx_stride, i, t, tpr, a.width);
    }
  }
  if (a.partial) {
    float* p = a.partial + static_cast<int64_t>(blockIdx.x) * a.width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int c = column<VECTOR>(i, e, t, tpr);
        if (c < a.width) p[c] = dw[i][e];
      }
  }
}

// dw[c] = sum over blocks of partial[block][c]: 32 columns a block, 32 threads
// for each column.
template <typename W>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* partial, int blocks,
                                                           int width, W* dw) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < width)
    for (int b = threadIdx.y; b < blocks; b += 32) s += partial[static_cast<int64_t>(b) * width + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = part[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
  const int out = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && out < width) dw[out] = from_f<W>(s);
}

// Threads for a row of `width` values and vectors for each of them: one warp
// with up to 8 vectors where rows abound (no barrier, 8 loads in flight a
// thread), else as many threads as the row has vectors, at most 1024.
struct Shape {
  int tpr, nv;
};
Shape shape_of(int64_t rows, int width, bool backward) {
  const int vectors = (width + kVec - 1) / kVec;
  int tpr = 32;
  const int most = backward ? 2 : (rows >= 2048 ? 8 : 1);  // vectors a thread aims at
  while (tpr < 1024 && tpr * most < vectors) tpr *= 2;
  int nv = 1;
  while (tpr * nv < vectors) nv *= 2;
  return {tpr, nv};
}

// Blocks of up to 256 threads may use 255 registers a thread, wider ones 64:
// only rows of more than 256 * 8 * nv values take those.
template <typename E, bool VECTOR, int NV, int THREADS>
cudaError_t launch_norm_nv(const RmsNormArgs& a, int tpr, cudaStream_t stream) {
  const int rows_per_block = tpr == 32 ? 4 : 1;
  const int64_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tpr * rows_per_block);
  if (!a.scale)
    rms_norm_kernel<E, VECTOR, NV, kNormPlain, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  else if (a.group == 0)
    rms_norm_kernel<E, VECTOR, NV, kNormRow8, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  else if constexpr (VECTOR)
    rms_norm_kernel<E, true, NV, kNormGroup8, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  return cudaGetLastError();
}

template <typename E, bool VECTOR>
cudaError_t launch_norm(const RmsNormArgs& a, cudaStream_t stream) {
  const Shape s = shape_of(a.rows, a.width, false);
  if (s.tpr > 256)
    switch (s.nv) {
      case 1: return launch_norm_nv<E, VECTOR, 1, 1024>(a, s.tpr, stream);
      case 2: return launch_norm_nv<E, VECTOR, 2, 1024>(a, s.tpr, stream);
      default: return launch_norm_nv<E, VECTOR, 4, 1024>(a, s.tpr, stream);
    }
  switch (s.nv) {
    case 1: return launch_norm_nv<E, VECTOR, 1, 256>(a, s.tpr, stream);
    case 2: return launch_norm_nv<E, VECTOR, 2, 256>(a, s.tpr, stream);
    case 4: return launch_norm_nv<E, VECTOR, 4, 256>(a, s.tpr, stream);
    default: return launch_norm_nv<E, VECTOR, 8, 256>(a, s.tpr, stream);
  }
}

template <typename E, bool VECTOR>
void launch_back(const RmsNormBackwardArgs& a, const Shape& s, int blocks, cudaStream_t stream) {
  if (s.tpr <= 256)
    s.nv == 1 ? rms_norm_backward_kernel<E, VECTOR, 1, 256><<<blocks, s.tpr, 0, stream>>>(a)
              : rms_norm_backward_kernel<E, VECTOR, 2, 256><<<blocks, s.tpr, 0, stream>>>(a);
  else if (s.nv <= 2)
    rms_norm_backward_kernel<E, VECTOR, 2, 1024><<<blocks, s.tpr, 0, stream>>>(a);
  else
    rms_norm_backward_kernel<E, VECTOR, 4, 1024><<<blocks, s.tpr, 0, stream>>>(a);
}

bool vector_ok(const void* p, int64_t stride, int elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * elem) % 16 == 0;
}

}  // namespace

cudaError_t launch_rms_norm(const RmsNormArgs& a, int dtype, cudaStream_t stream) {
  const int e = dtype == GSA_DTYPE_BF16 ? 2 : 4;
  bool vec = a.width % kVec == 0 && vector_ok(a.x, a.x_stride, e) &&
             vector_ok(a.weight, 0, 1) &&
             (!a.residual || (vector_ok(a.residual, a.residual_stride, e) &&
                              vector_ok(a.h, a.h_stride, e)));
  vec = vec && (a.scale ? reinterpret_cast<uintptr_t>(a.y) % 8 == 0 && a.y_stride % 8 == 0
                        : vector_ok(a.y, a.y_stride, e));
  if (a.scale && a.group && !vec) return cudaErrorMisalignedAddress;
  if (dtype == GSA_DTYPE_BF16)
    return vec ? launch_norm<__nv_bfloat16, true>(a, stream)
               : launch_norm<__nv_bfloat16, false>(a, stream);
  return vec ? launch_norm<float, true>(a, stream) : launch_norm<float, false>(a, stream);
}

// Rows in flight: enough blocks to fill the SMs, few enough that the partial
// sums of dw stay small beside the rows.
int rms_norm_backward_blocks(int64_t rows, int width) {
  const Shape s = shape_of(rows, width, true);
  const int64_t per_sm = 1024 / s.tpr < 1 ? 1 : 1024 / s.tpr;
  const int64_t most = 148 * (per_sm > 8 ? 8 : per_sm);
  return static_cast<int>(rows < most ? rows : most);
}

cudaError_t launch_rms_norm_backward(const RmsNormBackwardArgs& a, int dtype,
                                     cudaStream_t stream) {
  const int e = dtype == GSA_DTYPE_BF16 ? 2 : 4;
  const bool vec = a.width % kVec == 0 && vector_ok(a.h, a.h_stride, e) &&
                   vector_ok(a.dy, a.dy_stride, e) && vector_ok(a.weight, 0, 1) &&
                   (!a.dh || vector_ok(a.dh, a.dh_stride, e)) && vector_ok(a.dx, a.dx_stride, e);
  const int blocks = rms_norm_backward_blocks(a.rows, a.width);
  if (blocks > 0) {
    const Shape s = shape_of(a.rows, a.width, true);
    if (dtype == GSA_DTYPE_BF16)
      vec ? launch_back<__nv_bfloat16, true>(a, s, blocks, stream)
          : launch_back<__nv_bfloat16, false>(a, s, blocks, stream);
    else
      vec ? launch_back<float, true>(a, s, blocks, stream)
          : launch_back<float, false>(a, s, blocks, stream);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
  }
  if (!a.dweight) return cudaSuccess;
  const dim3 grid((a.width + 31) / 32), block(32, 32);
  if (a.weight_f32)
    rms_norm_dw_kernel<float><<<grid, block, 0, stream>>>(a.partial, blocks, a.width,
                                                          static_cast<float*>(a.dweight));
  else
    rms_norm_dw_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(
        a.partial, blocks, a.width, static_cast<__nv_bfloat16*>(a.dweight));
  return cudaGetLastError();
}

}  // namespace gsa
