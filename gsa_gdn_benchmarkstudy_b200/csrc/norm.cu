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
// Bound by HBM: 4 * rows * width * 2 bytes in bf16 with a residual.  A row is
// read once and stays in registers between its sum and its output (tpr threads x
// NV vectors of 8 values), so nothing is read twice.  How many threads share a
// row was measured at 16384 rows of 2048 (bf16, residual; a plain copy of the
// same bytes takes 41 us): 32 threads x 8 vectors 55 us, 64 x 4 47, 128 x 2 47,
// 256 x 1 51; with an 8-bit output (36 us) 62, 47, 53, 63.  Fewer vectors a thread
// leave too few loads in flight, more of them too few warps.  Sums and products two
// values at a time bring 64 x 4 to 44 and 46.
#include <cuda_fp8.h>

#include "kernels.h"

namespace gsa {
namespace {

constexpr int kVec = 8;

template <typename E> __device__ __forceinline__ E from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
// Two values at a time: the sums and products are one instruction for both.
__device__ __forceinline__ uint64_t pair(const float (&v)[kVec], int e) {
  return f2_pack(v[e], v[e + 1]);
}
__device__ __forceinline__ uint64_t round_f(uint64_t v, float) { return v; }
__device__ __forceinline__ uint64_t round_f(uint64_t v, __nv_bfloat16) {
  const uint32_t r = pack_bf16x2(f2_lo(v), f2_hi(v));
  return f2_pack(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
}

// How a thread's vectors of 8 values lie in a row.
//   kPlain    neighbours go to neighbouring threads, one value a load;
//   kVector   8 neighbours, 16 bytes (bf16) at once;
//   kShifted  the same where rows start off the 16-byte grid (an odd width): windows
//             of 8 on the grid, the first one `shift` values before the row, so all but
//             a row's first and last still move 16 bytes at once.  All tensors of a
//             call then start off the grid alike.
// 8192 rows of 4099 in bf16 with a residual take 357 us plain and 106 shifted (41
// for the bytes).
enum Form { kPlain = 0, kVector = 1, kShifted = 2 };
// Column of value e of vector i.
template <int FORM>
__device__ __forceinline__ int column(int i, int e, int t, int tpr, int shift) {
  return FORM == kPlain ? (i * kVec + e) * tpr + t
                        : (i * tpr + t) * kVec + e - (FORM == kShifted ? shift : 0);
}
// Whether vector i lies in the row, and whole.
template <int FORM>
__device__ __forceinline__ bool whole_vector(int c, int width) {
  return FORM == kShifted ? c >= 0 && c + kVec <= width : FORM == kVector && c < width;
}

// Values between the 8-value grid and p.
template <typename E>
__host__ __device__ __forceinline__ int off_grid(const E* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) / sizeof(E)) % kVec);
}

// Eight values as they lie in memory: loads that can wait to be converted.  ONCE:
// they leave the caches early.  The backward pass gains by it (54 to 50 us, figures as
// above), the forward pass loses (45 to 51).
template <typename E>
struct Raw {
  static constexpr int kWords = kVec * sizeof(E) / 16;
  uint4 w[kWords];
};
__device__ __forceinline__ void unpack(float (&v)[kVec], const Raw<__nv_bfloat16>& r) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(float (&v)[kVec], const Raw<float>& r) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    v[4 * j] = __uint_as_float(r.w[j].x);
    v[4 * j + 1] = __uint_as_float(r.w[j].y);
    v[4 * j + 2] = __uint_as_float(r.w[j].z);
    v[4 * j + 3] = __uint_as_float(r.w[j].w);
  }
}
template <int FORM, bool ONCE, typename E>
__device__ __forceinline__ void load_raw(Raw<E>& r, const E* row, int i, int t, int tpr,
                                         int width, int shift) {
  const int c = column<FORM>(i, 0, t, tpr, shift);
  if (FORM == kVector || whole_vector<FORM>(c, width)) {
#pragma unroll
    for (int j = 0; j < Raw<E>::kWords; ++j) {
      const uint4* at = reinterpret_cast<const uint4*>(row + c) + j;
      r.w[j] = c < width ? (ONCE ? __ldcs(at) : *at) : make_uint4(0, 0, 0, 0);
    }
  } else {
    E e[kVec];
#pragma unroll
    for (int x = 0; x < kVec; ++x) e[x] = from_f<E>(0.f);
    if (c < width)
#pragma unroll
      for (int x = 0; x < kVec; ++x) {
        const int at = column<FORM>(i, x, t, tpr, shift);
        if (at >= 0 && at < width) e[x] = row[at];
      }
    memcpy(&r, e, sizeof(r));
  }
}
template <int FORM, typename E>
__device__ __forceinline__ void load8(float (&v)[kVec], const E* row, int i, int t, int tpr,
                                      int width, int shift) {
  Raw<E> r;
  load_raw<FORM, false>(r, row, i, t, tpr, width, shift);
  unpack(v, r);
}

// The weight's values for vector i.  Shifted: two vectors of a weight in bf16 on the
// grid, and the 8 values from their middle.
template <int FORM, typename A>
__device__ __forceinline__ void load_weight(float (&w)[kVec], const A& a, int i, int t, int tpr,
                                            int shift) {
  if constexpr (FORM != kShifted) {
    if (a.weight_f32)
      load8<FORM>(w, static_cast<const float*>(a.weight), i, t, tpr, a.width, 0);
    else
      load8<FORM>(w, static_cast<const __nv_bfloat16*>(a.weight), i, t, tpr, a.width, 0);
  } else {
    const int c = column<FORM>(i, 0, t, tpr, shift), from = c & ~7;
    if (!a.weight_f32 && c >= 0 && from + 2 * kVec <= a.width) {
      const uint4* at = reinterpret_cast<const uint4*>(
          static_cast<const __nv_bfloat16*>(a.weight) + from);
      const uint4 x = at[0], y = at[1];
      uint32_t r[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 6; ++j) r[j] = c & 4 ? r[j + 2] : r[j];
#pragma unroll
      for (int j = 0; j < 5; ++j) r[j] = c & 2 ? r[j + 1] : r[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t z = c & 1 ? __funnelshift_r(r[j], r[j + 1], 16) : r[j];
        w[2 * j] = __uint_as_float(z << 16);
        w[2 * j + 1] = __uint_as_float(z & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = 0.f;
      if (c < a.width)
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (c + e >= 0 && c + e < a.width)
            w[e] = a.weight_f32 ? static_cast<const float*>(a.weight)[c + e]
                                : __bfloat162float(
                                      static_cast<const __nv_bfloat16*>(a.weight)[c + e]);
    }
  }
}

template <int FORM, typename E>
__device__ __forceinline__ void store8(const float (&v)[kVec], E* row, int i, int t, int tpr,
                                       int width, int shift) {
  const int c = column<FORM>(i, 0, t, tpr, shift);
  if (whole_vector<FORM>(c, width)) {
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
  } else if (FORM != kVector && c < width) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int at = column<FORM>(i, e, t, tpr, shift);
      if (at >= 0 && at < width) row[at] = from_f<E>(v[e]);
    }
  }
}

template <int FORM>
__device__ __forceinline__ void store8_e4m3(const float (&v)[kVec], uint8_t* row, int i, int t,
                                            int tpr, int width, int shift) {
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    lo |= uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE,
                                            __NV_E4M3)) << (8 * e);
    hi |= uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(v[e + 4], v[e + 5]), __NV_SATFINITE,
                                            __NV_E4M3)) << (8 * e);
  }
  const int c = column<FORM>(i, 0, t, tpr, shift);
  if (whole_vector<FORM>(c, width)) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
  } else if (FORM != kVector && c < width) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int at = column<FORM>(i, e, t, tpr, shift);
      if (at >= 0 && at < width) row[at] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
  }
}

__device__ __forceinline__ float fold_sum(float a, float b) { return a + b; }
// A NaN wins over every number, so that a row that holds one gets a NaN scale.
__device__ __forceinline__ float fold_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum or maximum over the tpr threads of a row (8, 16, 32, or whole warps; rows
// within a warp need no barrier).  `slot` has room for 32 values and is not used
// again before the caller's next barrier.
template <bool MAX>
__device__ __forceinline__ float row_fold(float v, float* slot, int tpr) {
  for (int m = (tpr < 32 ? tpr : 32) >> 1; m; m >>= 1) {
    const float o = __shfl_xor_sync(0xFFFFFFFFu, v, m);
    v = MAX ? fold_max(v, o) : fold_sum(v, o);
  }
  if (tpr <= 32) return v;
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
// only where a row is a warp or less).
template <typename E, int FORM, int NV, int OUT, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_kernel(RmsNormArgs a, int tpr) {
  __shared__ float slots[2][32];
  const int t = threadIdx.x % tpr;
  int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  // threads past the last row shadow it, so that a warp's shuffles stay whole
  const bool live = row < a.rows;
  if (!live) row = a.rows - 1;
  const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
  const E* res = a.residual ? static_cast<const E*>(a.residual) + row * a.residual_stride : nullptr;
  const int shift = FORM == kShifted ? off_grid(x) : 0;
  float v[NV][kVec];
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<FORM>(v[i], x, i, t, tpr, a.width, shift);
  if (res) {
    float r[NV][kVec];
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<FORM>(r[i], res, i, t, tpr, a.width, shift);
    E* h = static_cast<E*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const uint64_t h2 = round_f(f2_add(pair(v[i], e), pair(r[i], e)), E());
        v[i][e] = f2_lo(h2);
        v[i][e + 1] = f2_hi(h2);
      }
      if (live) store8<FORM>(v[i], h, i, t, tpr, a.width, shift);
    }
  }
  uint64_t s2 = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < kVec; e += 2) s2 = f2_fma(pair(v[i], e), pair(v[i], e), s2);
  const float s = row_fold<false>(f2_lo(s2) + f2_hi(s2), slots[0], tpr);
  const float rstd = 1.0f / sqrtf(s / static_cast<float>(a.width) + a.eps);
  if (a.rstd && live && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[kVec];
    load_weight<FORM>(w, a, i, t, tpr, shift);
#pragma unroll
    for (int e = 0; e < kVec; e += 2) {
      const uint64_t y2 = f2_mul(f2_mul(pair(v[i], e), f2_pack(rstd, rstd)), pair(w, e));
      v[i][e] = f2_lo(y2);
      v[i][e + 1] = f2_hi(y2);
    }
  }
  if constexpr (OUT == kNormPlain) {
    E* y = static_cast<E*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (live) store8<FORM>(v[i], y, i, t, tpr, a.width, shift);
  } else {
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride;
    float most = 0.f;
    if constexpr (OUT == kNormRow8) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) most = fold_max(fabsf(v[i][e]), most);
      most = fold_max(row_fold<true>(most, slots[1], tpr), 1e-12f);
      if (live && t == 0) a.scale[row] = most / 448.0f;
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
        const int c = column<FORM>(i, 0, t, tpr, shift);
        if (live && c < a.width && (t & 15) == 0)
          a.scale[row * (a.width >> 7) + (c >> 7)] = most / 448.0f;
      }
      const float inv = 448.0f / most;
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const uint64_t y2 = f2_mul(pair(v[i], e), f2_pack(inv, inv));
        v[i][e] = f2_lo(y2);
        v[i][e + 1] = f2_hi(y2);
      }
      if (live) store8_e4m3<FORM>(v[i], y, i, t, tpr, a.width, shift);
    }
  }
}

// Backward: block b takes the rows b, b + gridDim.x, ... and keeps its columns'
// share of dw in registers over all of them; the shares go to partial[b] and
// are added in block order by rms_norm_dw_kernel, so equal inputs give equal
// bits.  The next row's loads are in flight while a row's sum crosses the block.
template <typename E, int FORM, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_backward_kernel(RmsNormBackwardArgs a) {
  __shared__ float slots[2][32];
  const int tpr = blockDim.x, t = threadIdx.x;
  // a shifted form's grid is a multiple of 8, so that a block's rows start alike
  const int shift =
      FORM == kShifted ? off_grid(static_cast<const E*>(a.h) + blockIdx.x * a.h_stride) : 0;
  float dw[NV][kVec] = {};
  float w[NV][kVec];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_weight<FORM>(w[i], a, i, t, tpr, shift);
  Raw<E> h_raw[NV], dy_raw[NV], d_raw[NV];
  float rstd_next = 0.f;
  auto fetch = [&](int64_t row) {
    rstd_next = a.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load_raw<FORM, true>(h_raw[i], static_cast<const E*>(a.h) + row * a.h_stride, i, t, tpr, a.width,
                           shift);
      load_raw<FORM, true>(dy_raw[i], static_cast<const E*>(a.dy) + row * a.dy_stride, i, t, tpr,
                           a.width, shift);
      if (a.dh)
        load_raw<FORM, true>(d_raw[i], static_cast<const E*>(a.dh) + row * a.dh_stride, i, t, tpr,
                             a.width, shift);
    }
  };
  if (blockIdx.x < a.rows) fetch(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = rstd_next;
    float h[NV][kVec], dy[NV][kVec], d[NV][kVec];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack(h[i], h_raw[i]);
      unpack(dy[i], dy_raw[i]);
      if (a.dh) unpack(d[i], d_raw[i]);
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
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
      store8<FORM>(h[i], static_cast<E*>(a.dx) + row * a.dx_stride, i, t, tpr, a.width, shift);
    }
  }
  if (a.partial) {
    float* p = a.partial + static_cast<int64_t>(blockIdx.x) * a.width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int c = column<FORM>(i, e, t, tpr, shift);
        if (c >= 0 && c < a.width) p[c] = dw[i][e];
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

// Threads for a row of `width` values and vectors for each of them (measured
// above): four vectors a thread where rows fill the SMs, one where they do not, in
// whole warps (rows of 2100: 75 us with a power of two of threads, 63 with 96);
// backwards one, and two past 2048 values; no fewer than `least` threads: 8, 16 where
// they hold a group of 128 values, 32 backwards, where a row is a block's.
struct Shape {
  int tpr, nv;
};
Shape shape_of(int64_t rows, int width, int least) {
  const int vectors = (width + kVec - 1) / kVec;
  int tpr = least;
  const int most = least == 32 ? (vectors > 256 ? 2 : 1) : (rows >= 2048 ? 4 : 1);
  while (tpr < 32 && tpr * most < vectors) tpr *= 2;
  if (tpr * most < vectors) {  // whole warps
    tpr = ((vectors + most - 1) / most + 31) / 32 * 32;
    tpr = tpr < 1024 ? tpr : 1024;
  }
  int nv = 1;
  while (tpr * nv < vectors) nv *= 2;
  return {tpr, nv};
}

// Wider blocks than 256 threads are kernels of their own.
template <typename E, int FORM, int NV, int THREADS>
cudaError_t launch_norm_nv(const RmsNormArgs& a, int tpr, cudaStream_t stream) {
  const int rows_per_block = tpr <= 32 ? 128 / tpr : 1;
  const int64_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
  const dim3 grid(static_cast<unsigned>(blocks)), block(tpr * rows_per_block);
  if (!a.scale)
    rms_norm_kernel<E, FORM, NV, kNormPlain, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  else if (a.group == 0)
    rms_norm_kernel<E, FORM, NV, kNormRow8, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  else if constexpr (FORM == kVector)
    rms_norm_kernel<E, kVector, NV, kNormGroup8, THREADS><<<grid, block, 0, stream>>>(a, tpr);
  return cudaGetLastError();
}

template <typename E, int FORM>
cudaError_t launch_norm(const RmsNormArgs& a, cudaStream_t stream) {
  const Shape s = shape_of(a.rows, a.width + (FORM == kShifted ? kVec - 1 : 0), a.group ? 16 : 8);
  if (s.tpr > 256) switch (s.nv) {
      case 1: return launch_norm_nv<E, FORM, 1, 1024>(a, s.tpr, stream);
      case 2: return launch_norm_nv<E, FORM, 2, 1024>(a, s.tpr, stream);
      default: return launch_norm_nv<E, FORM, 4, 1024>(a, s.tpr, stream);
    }
  switch (s.nv) {
    case 1: return launch_norm_nv<E, FORM, 1, 256>(a, s.tpr, stream);
    case 2: return launch_norm_nv<E, FORM, 2, 256>(a, s.tpr, stream);
    default: return launch_norm_nv<E, FORM, 4, 256>(a, s.tpr, stream);
  }
}

template <typename E, int FORM>
void launch_back(const RmsNormBackwardArgs& a, const Shape& s, int blocks, cudaStream_t stream) {
  if (s.tpr <= 256)
    s.nv == 1 ? rms_norm_backward_kernel<E, FORM, 1, 256><<<blocks, s.tpr, 0, stream>>>(a)
              : rms_norm_backward_kernel<E, FORM, 2, 256><<<blocks, s.tpr, 0, stream>>>(a);
  else if (s.tpr <= 512)  // two vectors a thread
    rms_norm_backward_kernel<E, FORM, 2, 512><<<blocks, s.tpr, 0, stream>>>(a);
  else if (s.nv <= 2)
    rms_norm_backward_kernel<E, FORM, 2, 1024><<<blocks, s.tpr, 0, stream>>>(a);
  else
    rms_norm_backward_kernel<E, FORM, 4, 1024><<<blocks, s.tpr, 0, stream>>>(a);
}

bool vector_ok(const void* p, int64_t stride, int elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * elem) % 16 == 0;
}

// Whether the rows of all tensors start off the 8-value grid alike.
struct Grid {
  int64_t rows;
  int off, step;
  bool alike = true;
  Grid(const void* p, int64_t stride, int elem, int64_t n)
      : rows(n), off(place(p, elem)), step(static_cast<int>(stride % kVec)) {}
  static int place(const void* p, int elem) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(p) / elem) % kVec);
  }
  void with(const void* p, int64_t stride, int elem) {
    alike = alike && place(p, elem) == off && (rows < 2 || stride % kVec == step);
  }
};
// The widest row's windows are 1024 threads' four vectors.
bool shifted_ok(const Grid& g, const void* weight, int width) {
  return g.alike && vector_ok(weight, 0, 1) && (width + 2 * (kVec - 1)) / kVec <= 4096;
}

template <typename E>
cudaError_t launch_form(const RmsNormArgs& a, int form, cudaStream_t stream) {
  switch (form) {
    case kVector: return launch_norm<E, kVector>(a, stream);
    case kShifted: return launch_norm<E, kShifted>(a, stream);
    default: return launch_norm<E, kPlain>(a, stream);
  }
}
template <typename E>
void launch_back_form(const RmsNormBackwardArgs& a, int form, const Shape& s, int blocks,
                      cudaStream_t stream) {
  switch (form) {
    case kVector: return launch_back<E, kVector>(a, s, blocks, stream);
    case kShifted: return launch_back<E, kShifted>(a, s, blocks, stream);
    default: return launch_back<E, kPlain>(a, s, blocks, stream);
  }
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
  Grid grid(a.x, a.x_stride, e, a.rows);
  grid.with(a.y, a.y_stride, a.scale ? 1 : e);
  if (a.residual) {
    grid.with(a.residual, a.residual_stride, e);
    grid.with(a.h, a.h_stride, e);
  }
  const int form = vec ? kVector : shifted_ok(grid, a.weight, a.width) ? kShifted : kPlain;
  return dtype == GSA_DTYPE_BF16 ? launch_form<__nv_bfloat16>(a, form, stream)
                                 : launch_form<float>(a, form, stream);
}

// 768 threads an SM, each with the next row's loads in flight: 16384 rows of 2048
// took 53 us so (50 since the inputs leave the caches early), 57 with twice as many,
// 65 with two thirds (41 us for the bytes); more blocks also mean more partial sums of
// dw.  512 threads where each holds two vectors, so that all blocks run at once: 8192
// rows of 4096 take 70 us with 768, 67 so.  Two values an instruction, as forwards,
// take 50 us, but 61 instead of 51 at 4096 rows of 8192, where registers run out.  Past
// 8192 values a row's 1024 threads have at most 64 registers each and spill (bf16 0.5 to 4
// KB a thread); in fp32 the 512 threads of rows past 4096 do too (0.2 to 0.4 KB).
int rms_norm_backward_blocks(int64_t rows, int width) {
  const Shape s = shape_of(rows, width, 32);
  const int threads = s.nv == 1 ? 768 : 512;
  const int64_t most = 148 * (threads / s.tpr < 1 ? 1 : threads / s.tpr);
  return static_cast<int>(rows < most ? rows : most);
}

cudaError_t launch_rms_norm_backward(const RmsNormBackwardArgs& a, int dtype,
                                     cudaStream_t stream) {
  const int e = dtype == GSA_DTYPE_BF16 ? 2 : 4;
  const bool vec = a.width % kVec == 0 && vector_ok(a.h, a.h_stride, e) &&
                   vector_ok(a.dy, a.dy_stride, e) && vector_ok(a.weight, 0, 1) &&
                   (!a.dh || vector_ok(a.dh, a.dh_stride, e)) && vector_ok(a.dx, a.dx_stride, e);
  Grid grid_of(a.h, a.h_stride, e, a.rows);
  grid_of.with(a.dy, a.dy_stride, e);
  grid_of.with(a.dx, a.dx_stride, e);
  if (a.dh) grid_of.with(a.dh, a.dh_stride, e);
  const int form = vec ? kVector : shifted_ok(grid_of, a.weight, a.width) ? kShifted : kPlain;
  int blocks = rms_norm_backward_blocks(a.rows, a.width);
  if (form == kShifted && blocks < a.rows) blocks = blocks / kVec * kVec;
  if (blocks > 0) {
    const Shape s = shape_of(a.rows, a.width + (form == kShifted ? kVec - 1 : 0), 32);
    if (dtype == GSA_DTYPE_BF16)
      launch_back_form<__nv_bfloat16>(a, form, s, blocks, stream);
    else
      launch_back_form<float>(a, form, s, blocks, stream);
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
