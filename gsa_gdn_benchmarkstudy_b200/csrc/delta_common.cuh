// delta_common.cuh — what the kernels of the gated delta rule share: arguments,
// the division of a batch into sequences and chunks, decays of a chunk.
//
// Per sequence and value head h (key head h / (Hv / Hk)), with state S [dk, dv]:
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),
//   o_t = scale S_t^T q_t.
// Over a chunk of 64 tokens that starts from S0, with c_i = g_1 + ... + g_i:
//   L_ij = beta_i e^{c_i - c_j} (k_i . k_j)  (i > j),   T = (I + L)^-1,
//   P_ij = scale e^{c_i - c_j} (q_i . k_j)   (i >= j),
//   N = T diag(beta) (V - diag(e^c) K S0),
//   O = scale diag(e^c) Q S0 + P N,   S1 = e^{c_64} S0 + K^T diag(e^{c_64 - c}) N.
// T and P depend on no state, so they are made for all chunks at once; the pass
// from S0 to S1 is the only sequential one.  Columns of S never meet, so it
// splits over dv as well as over sequences and heads.
#pragma once

#include "kernels.h"

namespace gsa {
namespace delta {

constexpr int kChunk = 64;

__device__ __forceinline__ float load_gate(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
              : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_gate(void* p, int64_t i, bool bf16, float v) {
  if (bf16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E>
__device__ __forceinline__ E from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// e^g is 0 in fp32 below -104, so a decay of -inf (a wiped state) is held as
// -110: the sums c_i stay finite and their differences stay numbers.
__device__ __forceinline__ float bounded_decay(float g) { return g < -110.0f ? -110.0f : g; }

// Packed batches (cu_seqlens): the table that delta_table_kernel writes.
//   seq_begin[s], seq_len[s], seq_chunk[s]  first row, rows and first chunk of
//     "sequence" s; s = N and N + 1 stand for the rows before the first and
//     behind the last sequence, which get zeros;
//   order[i]  the i-th longest "sequence" (as they come where they are more than
//     kSorted): blocks that start last are short;
//   chunk_seq[c]  the sequence of chunk c, -1 for an unused one.
struct Table {
  int* seq_begin;
  int* seq_len;
  int* seq_chunk;
  int* order;
  int* chunk_seq;
};
constexpr int kSorted = 1024;
__host__ __device__ inline Table table_at(void* base, int N) {
  int* p = static_cast<int*>(base);
  return {p, p + (N + 2), p + 2 * (N + 2), p + 3 * (N + 2), p + 4 * (N + 2)};
}
// Chunks that B * T rows in N sequences can have.
inline int64_t max_chunks(const gsa_delta_t& p) {
  if (p.cu_seqlens) return p.T / kChunk + static_cast<int64_t>(p.N) + 2;
  return static_cast<int64_t>(p.B) * ((p.T + kChunk - 1) / kChunk);
}
inline int64_t table_bytes(const gsa_delta_t& p) {
  if (!p.cu_seqlens) return 0;
  return (4 * (4 * (static_cast<int64_t>(p.N) + 2) + max_chunks(p)) + 255) / 256 * 256;
}

// A sequence: batch row, first token, tokens, first chunk; `gap`: no sequence
// but rows that belong to none.
struct Seq {
  int b, begin, len, chunk0;
  bool gap;
};
__device__ __forceinline__ Seq sequence(const gsa_delta_t& p, const Table& t, int s) {
  if (!p.cu_seqlens) return {s, 0, p.T, s * ((p.T + kChunk - 1) / kChunk), false};
  return {0, t.seq_begin[s], t.seq_len[s], t.seq_chunk[s], s >= p.N};
}
// A chunk: its sequence and its rows; valid = false for an unused one.
struct Chunk {
  int seq, b, begin, len;
  bool gap, valid;
};
__device__ __forceinline__ Chunk chunk_at(const gsa_delta_t& p, const Table& t, int c) {
  int s;
  if (p.cu_seqlens) {
    s = t.chunk_seq[c];
    if (s < 0) return {0, 0, 0, 0, false, false};
  } else {
    s = c / ((p.T + kChunk - 1) / kChunk);
  }
  const Seq q = sequence(p, t, s);
  const int off = (c - q.chunk0) * kChunk;
  const int left = q.len - off;
  return {s, q.b, q.begin + off, left < kChunk ? left : kChunk, q.gap, true};
}

// Cumulative decays c_i of a chunk by one warp (lane l: tokens 2l, 2l + 1), as
// hi + lo pairs of fp32 so that differences keep fp32's accuracy however far
// the sums have gone.  Rows past `len` repeat the last sum and have beta 0.
struct __align__(16) Decays {
  float hi[kChunk], lo[kChunk], beta[kChunk];
};
__device__ __forceinline__ void chunk_decays(const gsa_delta_t& p, const Chunk& c, int hv,
                                             Decays& d) {
  const int lane = threadIdx.x & 31;
  double g[2];
  float b[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    g[e] = 0.0;
    b[e] = 0.f;
    if (i < c.len) {
      const int64_t row = c.begin + i;
      g[e] = bounded_decay(load_gate(p.g, c.b * p.g_stride[0] + row * p.g_stride[1] + hv,
                                     p.gate_dtype == GSA_DTYPE_BF16));
      b[e] = load_gate(p.beta, c.b * p.beta_stride[0] + row * p.beta_stride[1] + hv,
                       p.gate_dtype == GSA_DTYPE_BF16);
    }
  }
  double s = g[0] + g[1];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const double o = __shfl_up_sync(0xFFFFFFFFu, s, m);
    if (lane >= m) s += o;
  }
  const double c1 = s, c0 = s - g[1];
  d.hi[2 * lane] = static_cast<float>(c0);
  d.lo[2 * lane] = static_cast<float>(c0 - static_cast<double>(static_cast<float>(c0)));
  d.hi[2 * lane + 1] = static_cast<float>(c1);
  d.lo[2 * lane + 1] = static_cast<float>(c1 - static_cast<double>(static_cast<float>(c1)));
  d.beta[2 * lane] = b[0];
  d.beta[2 * lane + 1] = b[1];
}
// e^{c_i - c_j}
__device__ __forceinline__ float decay_between(const Decays& d, int i, int j) {
  return expf((d.hi[i] - d.hi[j]) + (d.lo[i] - d.lo[j]));
}
__device__ __forceinline__ float decay_from_start(const Decays& d, int i) {
  return expf(d.hi[i] + d.lo[i]);
}

// What the sequential pass and the gradients need of a chunk's decays.
struct __align__(16) Gates {
  float grown[kChunk];  // e^{c_i}
  float beta[kChunk];
  float left[kChunk];   // e^{c_64 - c_i}
  float both[kChunk];   // beta_i e^{c_i}
  float hi[kChunk];     // c_i = hi + lo
  float lo[kChunk];
  float pad[2 * kChunk];
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}

constexpr int kLdL = kChunk + 4;
// out = sign a b for N x N blocks, R x 4 a thread, four k at a time.  LOWER_B: b is
// lower triangular, k starts at the thread's first column, which a warp's threads
// nearly share; else a is, and k ends behind its last row.
template <int N, int R, bool LOWER_B>
__device__ __forceinline__ void block_product(int t, const float* a, const float* b, float* out,
                                              float sign) {
  constexpr int kRows = N / R, kColGroups = N / 4, kApart = LOWER_B ? kRows : 1;
  const int r = LOWER_B ? t % kRows : t / kColGroups * R;
  const int c = (LOWER_B ? t / kRows : t % kColGroups) * 4;
  float x[R][4] = {};
  const int first = LOWER_B ? c : 0, last = LOWER_B ? N : r + R;
#pragma unroll 2
  for (int k = first; k < last; k += 4) {
    float4 u[R], v[4];
#pragma unroll
    for (int i = 0; i < R; ++i)
      u[i] = *reinterpret_cast<const float4*>(a + (r + i * kApart) * kLdL + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(b + (k + j) * kLdL + c);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float f = j == 0 ? u[i].x : j == 1 ? u[i].y : j == 2 ? u[i].z : u[i].w;
        x[i][0] = fmaf(f, v[j].x, x[i][0]);
        x[i][1] = fmaf(f, v[j].y, x[i][1]);
        x[i][2] = fmaf(f, v[j].z, x[i][2]);
        x[i][3] = fmaf(f, v[j].w, x[i][3]);
      }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    *reinterpret_cast<float4*>(out + (r + i * kApart) * kLdL + c) =
        make_float4(sign * x[i][0], sign * x[i][1], sign * x[i][2], sign * x[i][3]);
}

// L (strictly lower, 64 x 64, its upper right quarter free) becomes
// T = (I + L)^-1 in place, in fp32: the four 16 x 16 diagonal blocks by
// substitution, then T21 = -T22 L21 T11 twice over.  By the block's first 128 threads.
__device__ __forceinline__ void invert(float* L) {
  const int tid = threadIdx.x, warp = tid >> 5;
  const bool works = tid < 128;
  if (warp == 0 || warp == 2) {
    const int b = warp + ((tid >> 4) & 1), j = tid & 15;
    float* D = L + 16 * b * kLdL + 16 * b;
    float col[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; m += 4) {
        const float4 v = *reinterpret_cast<const float4*>(D + i * kLdL + m);
        s = fmaf(-v.x, col[m], s);
        if (m + 1 < i) s = fmaf(-v.y, col[m + 1], s);
        if (m + 2 < i) s = fmaf(-v.z, col[m + 2], s);
        if (m + 3 < i) s = fmaf(-v.w, col[m + 3], s);
      }
      col[i] = s;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) D[i * kLdL + j] = col[i];
  }
  __syncthreads();
  const int b = (tid >> 6) * 32, t = tid & 63;
  float* D = L + b * kLdL + b;
  float *X = L + 32, *Y = X + (tid >> 6) * 16 * kLdL;
  if (works) block_product<16, 1, true>(t, D + 16 * kLdL, D, Y, 1.f);
  __syncthreads();
  if (works) block_product<16, 1, false>(t, D + 16 * kLdL + 16, Y, D + 16 * kLdL, -1.f);
  __syncthreads();
  if (works) block_product<32, 2, true>(tid, L + 32 * kLdL, L, X, 1.f);
  __syncthreads();
  if (works) block_product<32, 2, false>(tid, L + 32 * kLdL + 32, X, L + 32 * kLdL, -1.f);
}

}  // namespace delta
}  // namespace gsa
