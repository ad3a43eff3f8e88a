// delta_simt.cu — the chunked gated delta rule, forward and backward, on the
// CUDA cores in fp32: fp32 inputs keep fp32's accuracy in every product, which
// the tensor cores' 16-bit operands do not give (delta_prep.cu, delta_seq.cu and delta_grad.cu serve bf16).
//
// Four kernels: `prep` makes T and P of every chunk, `chain` walks the chunks
// of a sequence forwards, `rev` walks them backwards with the state's gradient,
// `grad` turns what both left behind into gradients, chunk by chunk.  All
// products are 64 tokens high; 256 threads hold 4 rows x NJ columns each.
// Bound by shared-memory loads (4 + NJ words for 4 NJ multiply-adds).
#include "delta_common.cuh"

namespace gsa {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 32;  // state columns of a block of chain / rev
constexpr int kLdM = kChunk + 1;
constexpr int kLdC = kCols + 1;

// acc[i][j] += sum_k a(r0 + i, k) b(k, c0 + 16 j), r0 = 4 (tid / 16), c0 = tid % 16.
template <int NJ, typename A, typename B>
__device__ __forceinline__ void product(float (&acc)[4][NJ], int K, A a, B b) {
  const int r0 = (threadIdx.x >> 4) * 4, c0 = threadIdx.x & 15;
  for (int k = 0; k < K; ++k) {
    float av[4], bv[NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i) av[i] = a(r0 + i, k);
#pragma unroll
    for (int j = 0; j < NJ; ++j) bv[j] = b(k, c0 + 16 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
  }
}
template <int NJ, typename F>
__device__ __forceinline__ void each(float (&acc)[4][NJ], F f) {
  const int r0 = (threadIdx.x >> 4) * 4, c0 = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) f(r0 + i, c0 + 16 * j, acc[i][j]);
}

// 64 rows of `width` values from column col0 on into shared memory; rows past
// len and columns past `limit` are zero.
template <typename E>
__device__ __forceinline__ void load_rows(float* dst, int ld, const E* src, int64_t stride,
                                          int len, int col0, int width, int limit) {
  for (int i = threadIdx.x; i < kChunk * width; i += kThreads) {
    const int r = i / width, c = i % width;
    dst[r * ld + c] =
        (r < len && col0 + c < limit) ? to_float(src[r * stride + col0 + c]) : 0.f;
  }
}

__host__ __device__ inline int64_t tile_floats() { return 2 * kChunk * kChunk; }  // T, P

// Sections of the workspace (fp32), each with a slot for every chunk and head.
struct Saved {
  float* tiles;   // T, P
  float* news;    // N [64, dv]     (training)
  float* states;  // S0 [dk, dv]    (training)
};
struct Scratch {
  float* back;    // dY [64, dv]
  float* states;  // dS1 [dk, dv]
};
Saved saved_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  Saved s;
  s.tiles = reinterpret_cast<float*>(static_cast<char*>(ws) + table_bytes(p));
  s.news = s.tiles + n * tile_floats();
  s.states = s.news + n * kChunk * p.dv;
  return s;
}
Scratch scratch_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  Scratch s;
  s.back = static_cast<float*>(ws);
  s.states = s.back + n * kChunk * p.dv;
  return s;
}

template <typename E>
__device__ __forceinline__ const E* q_at(const gsa_delta_t& p, const Chunk& c, int hk) {
  return static_cast<const E*>(p.q) + c.b * p.q_stride[0] + c.begin * p.q_stride[1] +
         hk * p.q_stride[2];
}
template <typename E>
__device__ __forceinline__ const E* k_at(const gsa_delta_t& p, const Chunk& c, int hk) {
  return static_cast<const E*>(p.k) + c.b * p.k_stride[0] + c.begin * p.k_stride[1] +
         hk * p.k_stride[2];
}
template <typename E>
__device__ __forceinline__ const E* v_at(const gsa_delta_t& p, const Chunk& c, int hv) {
  return static_cast<const E*>(p.v) + c.b * p.v_stride[0] + c.begin * p.v_stride[1] +
         hv * p.v_stride[2];
}
// Row `begin` of a contiguous [B, T, heads, width] tensor.
__device__ __forceinline__ int64_t row_at(const gsa_delta_t& p, const Chunk& c, int heads, int h,
                                          int width) {
  return ((static_cast<int64_t>(c.b) * p.T + c.begin) * heads + h) * width;
}

template <typename E>
__global__ void __launch_bounds__(kThreads) prep_kernel(const gsa_delta_t p, Table table,
                                                        float* tiles) {
  extern __shared__ float sm[];
  const int ld = p.dk + 1;
  float* K = sm;
  float* Q = K + kChunk * ld;
  float* L = Q + kChunk * ld;
  __shared__ Decays d;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk);
  const Chunk c = chunk_at(p, table, blockIdx.x);
  if (!c.valid || c.gap) return;
  load_rows(K, ld, k_at<E>(p, c, hk), p.k_stride[1], c.len, 0, p.dk, p.dk);
  load_rows(Q, ld, q_at<E>(p, c, hk), p.q_stride[1], c.len, 0, p.dk, p.dk);
  if (threadIdx.x < 32) chunk_decays(p, c, hv, d);
  __syncthreads();
  float* T = tiles + (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * tile_floats();
  float* P = T + kChunk * kChunk;
  float kk[4][4] = {}, qk[4][4] = {};
  auto krow = [&](int k, int j) { return K[j * ld + k]; };
  product<4>(kk, p.dk, [&](int i, int k) { return K[i * ld + k]; }, krow);
  product<4>(qk, p.dk, [&](int i, int k) { return Q[i * ld + k]; }, krow);
  each(kk, [&](int i, int j, float v) {
    L[i * kLdM + j] = i > j ? d.beta[i] * decay_between(d, i, j) * v : 0.f;
  });
  each(qk, [&](int i, int j, float v) {
    P[i * kChunk + j] = i >= j ? p.scale * decay_between(d, i, j) * v : 0.f;
  });
  __syncthreads();
  // T = (I + L)^-1 by forward substitution, a column a thread
  const int j = threadIdx.x;
  if (j < kChunk) {
    float col[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      float s = i == j ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) s = fmaf(-L[i * kLdM + m], col[m], s);
      col[i] = i < j ? 0.f : s;
      T[i * kChunk + j] = col[i];
    }
  }
}

struct ChainArgs {
  Table table;
  const float* tiles;
  float* news;    // nullptr: inference
  float* states;
  void* o;
  float* final_state;
};

template <typename E>
__global__ void __launch_bounds__(kThreads) chain_kernel(const gsa_delta_t p, const ChainArgs a) {
  extern __shared__ float sm[];
  const int ld = p.dk + 1;
  float* K = sm;
  float* Q = K + kChunk * ld;
  float* T = Q + kChunk * ld;
  float* P = T + kChunk * kLdM;
  float* S = P + kChunk * kLdM;  // [dk][kLdC]
  float* Y = S + p.dk * kLdC;    // beta (V - e^c K S), [64][kLdC]
  float* N = Y + kChunk * kLdC;
  __shared__ Decays d;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk), col0 = blockIdx.z * kCols;
  const Seq s = sequence(p, a.table, blockIdx.x);
  E* out = static_cast<E*>(a.o);
  if (s.gap) {  // rows of no sequence
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(s.len) * kCols; i += kThreads) {
      const int64_t r = s.begin + i / kCols;
      const int col = col0 + static_cast<int>(i % kCols);
      if (col < p.dv) out[(r * p.Hv + hv) * p.dv + col] = from_float<E>(0.f);
    }
    return;
  }
  const int64_t state0 = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
    const int r = i / kCols, c = i % kCols;
    S[r * kLdC + c] = (p.initial_state && col0 + c < p.dv)
                          ? p.initial_state[state0 + static_cast<int64_t>(r) * p.dv + col0 + c]
                          : 0.f;
  }
  const int chunks = (s.len + kChunk - 1) / kChunk;
  for (int n = 0; n < chunks; ++n) {
    const int left = s.len - n * kChunk;
    const Chunk c = {static_cast<int>(blockIdx.x), s.b, s.begin + n * kChunk,
                     left < kChunk ? left : kChunk, false, true};
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    __syncthreads();
    load_rows(K, ld, k_at<E>(p, c, hk), p.k_stride[1], c.len, 0, p.dk, p.dk);
    load_rows(Q, ld, q_at<E>(p, c, hk), p.q_stride[1], c.len, 0, p.dk, p.dk);
    const float* tp = a.tiles + slot * tile_floats();
    load_rows(T, kLdM, tp, static_cast<int64_t>(kChunk), kChunk, 0, kChunk, kChunk);
    load_rows(P, kLdM, tp + kChunk * kChunk, static_cast<int64_t>(kChunk), kChunk, 0, kChunk,
              kChunk);
    if (threadIdx.x < 32) chunk_decays(p, c, hv, d);
    if (a.states) {
      float* st = a.states + slot * p.dk * p.dv;
      for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
        const int r = i / kCols, cc = i % kCols;
        if (col0 + cc < p.dv) st[static_cast<int64_t>(r) * p.dv + col0 + cc] = S[r * kLdC + cc];
      }
    }
    __syncthreads();
    float ks[4][2] = {}, qs[4][2] = {};
    auto srow = [&](int k, int j) { return S[k * kLdC + j]; };
    product<2>(ks, p.dk, [&](int i, int k) { return K[i * ld + k]; }, srow);
    product<2>(qs, p.dk, [&](int i, int k) { return Q[i * ld + k]; }, srow);
    const E* v = v_at<E>(p, c, hv);
    each(ks, [&](int i, int j, float x) {
      const float vv =
          (i < c.len && col0 + j < p.dv) ? to_float(v[i * p.v_stride[1] + col0 + j]) : 0.f;
      Y[i * kLdC + j] = d.beta[i] * (vv - decay_from_start(d, i) * x);
    });
    __syncthreads();
    float nn[4][2] = {};
    product<2>(nn, kChunk, [&](int i, int k) { return T[i * kLdM + k]; },
               [&](int k, int j) { return Y[k * kLdC + j]; });
    each(nn, [&](int i, int j, float x) {
      N[i * kLdC + j] = x;
      if (a.news && col0 + j < p.dv) a.news[(slot * kChunk + i) * p.dv + col0 + j] = x;
    });
    __syncthreads();
    each(qs, [&](int i, int, float& x) { x *= p.scale * decay_from_start(d, i); });
    product<2>(qs, kChunk, [&](int i, int k) { return P[i * kLdM + k]; },
               [&](int k, int j) { return N[k * kLdC + j]; });
    const int64_t o0 = row_at(p, c, p.Hv, hv, p.dv);
    each(qs, [&](int i, int j, float x) {
      if (i < c.len && col0 + j < p.dv)
        out[o0 + static_cast<int64_t>(i) * p.Hv * p.dv + col0 + j] = from_float<E>(x);
    });
    const float whole = decay_from_start(d, kChunk - 1);
    for (int r0 = 0; r0 < p.dk; r0 += kChunk) {
      float st[4][2] = {};
      product<2>(st, kChunk,
                 [&](int i, int k) { return r0 + i < p.dk ? K[k * ld + r0 + i] : 0.f; },
                 [&](int k, int j) { return decay_between(d, kChunk - 1, k) * N[k * kLdC + j]; });
      each(st, [&](int i, int j, float x) {
        if (r0 + i < p.dk)
          S[(r0 + i) * kLdC + j] = fmaf(whole, S[(r0 + i) * kLdC + j], x);
      });
    }
  }
  if (a.final_state) {
    __syncthreads();
    for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
      const int r = i / kCols, c = i % kCols;
      if (col0 + c < p.dv)
        a.final_state[state0 + static_cast<int64_t>(r) * p.dv + col0 + c] = S[r * kLdC + c];
    }
  }
}

struct RevArgs {
  Table table;
  const float* tiles;
  const void* dout;           // contiguous, may be nullptr
  const float* dfinal;        // may be nullptr
  float* back;                // dY
  float* states;              // dS1
  float* dinitial;            // may be nullptr
};

// dN = P^T dO + diag(e^{c_64 - c}) K dS1,  dY = T^T dN,
// dS0 = e^{c_64} dS1 + K^T (-diag(e^c beta) dY) + Q^T (diag(scale e^c) dO).
template <typename E>
__global__ void __launch_bounds__(kThreads) rev_kernel(const gsa_delta_t p, const RevArgs a) {
  extern __shared__ float sm[];
  const int ld = p.dk + 1;
  float* K = sm;
  float* Q = K + kChunk * ld;
  float* T = Q + kChunk * ld;
  float* P = T + kChunk * kLdM;
  float* S = P + kChunk * kLdM;
  float* X = S + p.dk * kLdC;   // dN, then -e^c beta dY
  float* D = X + kChunk * kLdC;  // dO
  __shared__ Decays d;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk), col0 = blockIdx.z * kCols;
  const Seq s = sequence(p, a.table, blockIdx.x);
  if (s.gap) return;
  const int64_t state0 = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
    const int r = i / kCols, c = i % kCols;
    S[r * kLdC + c] = (a.dfinal && col0 + c < p.dv)
                          ? a.dfinal[state0 + static_cast<int64_t>(r) * p.dv + col0 + c]
                          : 0.f;
  }
  const int chunks = (s.len + kChunk - 1) / kChunk;
  for (int n = chunks - 1; n >= 0; --n) {
    const int left = s.len - n * kChunk;
    const Chunk c = {static_cast<int>(blockIdx.x), s.b, s.begin + n * kChunk,
                     left < kChunk ? left : kChunk, false, true};
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    __syncthreads();
    load_rows(K, ld, k_at<E>(p, c, hk), p.k_stride[1], c.len, 0, p.dk, p.dk);
    load_rows(Q, ld, q_at<E>(p, c, hk), p.q_stride[1], c.len, 0, p.dk, p.dk);
    const float* tp = a.tiles + slot * tile_floats();
    load_rows(T, kLdM, tp, static_cast<int64_t>(kChunk), kChunk, 0, kChunk, kChunk);
    load_rows(P, kLdM, tp + kChunk * kChunk, static_cast<int64_t>(kChunk), kChunk, 0, kChunk,
              kChunk);
    load_rows(D, kLdC, static_cast<const E*>(a.dout) + (a.dout ? row_at(p, c, p.Hv, hv, p.dv) : 0),
              static_cast<int64_t>(p.Hv) * p.dv, a.dout ? c.len : 0, col0, kCols, p.dv);
    if (threadIdx.x < 32) chunk_decays(p, c, hv, d);
    float* st = a.states + slot * p.dk * p.dv;
    for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
      const int r = i / kCols, cc = i % kCols;
      if (col0 + cc < p.dv) st[static_cast<int64_t>(r) * p.dv + col0 + cc] = S[r * kLdC + cc];
    }
    __syncthreads();
    float dn[4][2] = {};
    product<2>(dn, p.dk, [&](int i, int k) { return K[i * ld + k]; },
               [&](int k, int j) { return S[k * kLdC + j]; });
    each(dn, [&](int i, int, float& x) { x *= decay_between(d, kChunk - 1, i); });
    product<2>(dn, kChunk, [&](int i, int k) { return P[k * kLdM + i]; },
               [&](int k, int j) { return D[k * kLdC + j]; });
    each(dn, [&](int i, int j, float x) { X[i * kLdC + j] = x; });
    __syncthreads();
    float dy[4][2] = {};
    product<2>(dy, kChunk, [&](int i, int k) { return T[k * kLdM + i]; },
               [&](int k, int j) { return X[k * kLdC + j]; });
    __syncthreads();
    each(dy, [&](int i, int j, float x) {
      if (col0 + j < p.dv) a.back[(slot * kChunk + i) * p.dv + col0 + j] = x;
      const float g = decay_from_start(d, i);
      X[i * kLdC + j] = -g * d.beta[i] * x;
      D[i * kLdC + j] *= p.scale * g;
    });
    __syncthreads();
    const float whole = decay_from_start(d, kChunk - 1);
    for (int r0 = 0; r0 < p.dk; r0 += kChunk) {
      float ds[4][2] = {};
      product<2>(ds, kChunk,
                 [&](int i, int k) { return r0 + i < p.dk ? K[k * ld + r0 + i] : 0.f; },
                 [&](int k, int j) { return X[k * kLdC + j]; });
      product<2>(ds, kChunk,
                 [&](int i, int k) { return r0 + i < p.dk ? Q[k * ld + r0 + i] : 0.f; },
                 [&](int k, int j) { return D[k * kLdC + j]; });
      each(ds, [&](int i, int j, float x) {
        if (r0 + i < p.dk)
          S[(r0 + i) * kLdC + j] = fmaf(whole, S[(r0 + i) * kLdC + j], x);
      });
    }
  }
  if (a.dinitial) {
    __syncthreads();
    for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
      const int r = i / kCols, c = i % kCols;
      if (col0 + c < p.dv)
        a.dinitial[state0 + static_cast<int64_t>(r) * p.dv + col0 + c] = S[r * kLdC + c];
    }
  }
}

struct GradArgs {
  Table table;
  const float* news;     // N
  const float* states;   // S0
  const float* back;     // dY
  const float* dstates;  // dS1
  const void* dout;
  void *dq, *dk, *dv, *dg, *dbeta;  // contiguous
};

// A chunk and key head; the value heads that share it one after the other, so
// their gradients add up in one order.  With dP = scale dO N^T and dL = -dY N^T
// (lower triangles), M = strict(dL beta D):
//   dQ = scale e^c dO S0^T + (dP D) K
//   dK = -e^c beta dY S0^T + e^{c_64 - c} N dS1^T + (dP D)^T Q + (M + M^T) K
//   dV = beta dY,  dbeta_i = dY_i.(V_i - e^{c_i} S0^T k_i) + sum_j dL_ij D_ij k_i.k_j
//   dg_t = what the decays between tokens before t and tokens from t on carry:
//          sum_{i >= t} (scale e^c q.dO S0^T - e^c beta k.dY S0^T + rows of E - columns of E)_i
//          + sum_{i < t} e^{c_64 - c_i} k_i.(N dS1^T)_i + e^{c_64} <S0, dS1>,
//   E_ij = (dP D)_ij q_i.k_j + M_ij k_i.k_j.
template <typename E>
__global__ void __launch_bounds__(kThreads) grad_kernel(const gsa_delta_t p, const GradArgs a) {
  extern __shared__ float sm[];
  const int ld = p.dk + 1;
  float* K = sm;
  float* Q = K + kChunk * ld;
  float* S0 = Q + kChunk * ld;    // [dk][kLdC]
  float* S1 = S0 + p.dk * kLdC;
  float* D = S1 + p.dk * kLdC;    // dO, [64][kLdC]
  float* N = D + kChunk * kLdC;
  float* Y = N + kChunk * kLdC;   // dY
  float* A = Y + kChunk * kLdC;   // dP D, [64][kLdM]
  float* M = A + kChunk * kLdM;
  __shared__ Decays d;
  __shared__ float rowsum[kChunk], colsum[kChunk], grow[kChunk], db[kChunk], red[kThreads / 32];
  const int hk = blockIdx.y, group = p.Hv / p.Hk, tid = threadIdx.x;
  const Chunk c = chunk_at(p, a.table, blockIdx.x);
  if (!c.valid) return;
  const int64_t qk0 = row_at(p, c, p.Hk, hk, p.dk);
  const int64_t qk_step = static_cast<int64_t>(p.Hk) * p.dk;
  const bool gate16 = p.gate_dtype == GSA_DTYPE_BF16;
  E* dq_out = static_cast<E*>(a.dq);
  E* dk_out = static_cast<E*>(a.dk);
  E* dv_out = static_cast<E*>(a.dv);
  if (c.gap) {
    for (int i = tid; i < c.len * p.dk; i += kThreads) {
      dq_out[qk0 + (i / p.dk) * qk_step + i % p.dk] = from_float<E>(0.f);
      dk_out[qk0 + (i / p.dk) * qk_step + i % p.dk] = from_float<E>(0.f);
    }
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      const int64_t v0 = row_at(p, c, p.Hv, h, p.dv), g0 = row_at(p, c, p.Hv, h, 1);
      for (int i = tid; i < c.len * p.dv; i += kThreads)
        dv_out[v0 + static_cast<int64_t>(i / p.dv) * p.Hv * p.dv + i % p.dv] = from_float<E>(0.f);
      for (int i = tid; i < c.len; i += kThreads) {
        store_gate(a.dg, g0 + static_cast<int64_t>(i) * p.Hv, gate16, 0.f);
        store_gate(a.dbeta, g0 + static_cast<int64_t>(i) * p.Hv, gate16, 0.f);
      }
    }
    return;
  }
  load_rows(K, ld, k_at<E>(p, c, hk), p.k_stride[1], c.len, 0, p.dk, p.dk);
  load_rows(Q, ld, q_at<E>(p, c, hk), p.q_stride[1], c.len, 0, p.dk, p.dk);
  float gq[4][8] = {}, gk[4][8] = {};  // dq and dk of 64 tokens x 128 channels
  const int r0 = (tid >> 4) * 4, lane16 = tid & 15;
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
    __syncthreads();
    if (tid < 32) chunk_decays(p, c, hv, d);
    if (tid < kChunk) rowsum[tid] = colsum[tid] = grow[tid] = db[tid] = 0.f;
    float to[4][8] = {}, ty[4][8] = {}, tn[4][8] = {}, dp[4][4] = {}, dl[4][4] = {};
    float yv[4] = {}, cross = 0.f;
    for (int col0 = 0; col0 < p.dv; col0 += kCols) {
      __syncthreads();
      load_rows(D, kLdC, static_cast<const E*>(a.dout) + (a.dout ? row_at(p, c, p.Hv, hv, p.dv) : 0),
                static_cast<int64_t>(p.Hv) * p.dv, a.dout ? c.len : 0, col0, kCols, p.dv);
      load_rows(N, kLdC, a.news + slot * kChunk * p.dv, static_cast<int64_t>(p.dv), kChunk, col0,
                kCols, p.dv);
      load_rows(Y, kLdC, a.back + slot * kChunk * p.dv, static_cast<int64_t>(p.dv), kChunk, col0,
                kCols, p.dv);
      for (int i = tid; i < p.dk * kCols; i += kThreads) {
        const int r = i / kCols, cc = i % kCols;
        const bool in = col0 + cc < p.dv;
        const int64_t at = slot * p.dk * p.dv + static_cast<int64_t>(r) * p.dv + col0 + cc;
        const float x = in ? a.states[at] : 0.f, y = in ? a.dstates[at] : 0.f;
        S0[r * kLdC + cc] = x;
        S1[r * kLdC + cc] = y;
        cross = fmaf(x, y, cross);
      }
      __syncthreads();
      auto s0t = [&](int k, int j) { return j < p.dk ? S0[j * kLdC + k] : 0.f; };
      auto s1t = [&](int k, int j) { return j < p.dk ? S1[j * kLdC + k] : 0.f; };
      auto nt = [&](int k, int j) { return N[j * kLdC + k]; };
      product<8>(to, kCols, [&](int i, int k) { return D[i * kLdC + k]; }, s0t);
      product<8>(ty, kCols, [&](int i, int k) { return Y[i * kLdC + k]; }, s0t);
      product<8>(tn, kCols, [&](int i, int k) { return N[i * kLdC + k]; }, s1t);
      product<4>(dp, kCols, [&](int i, int k) { return D[i * kLdC + k]; }, nt);
      product<4>(dl, kCols, [&](int i, int k) { return Y[i * kLdC + k]; }, nt);
      const E* v = v_at<E>(p, c, hv);
      const int64_t v0 = row_at(p, c, p.Hv, hv, p.dv);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int cc = lane16; cc < kCols; cc += 16)
          if (r0 + i < c.len && col0 + cc < p.dv) {
            const float y = Y[(r0 + i) * kLdC + cc];
            yv[i] = fmaf(y, to_float(v[(r0 + i) * p.v_stride[1] + col0 + cc]), yv[i]);
            dv_out[v0 + static_cast<int64_t>(r0 + i) * p.Hv * p.dv + col0 + cc] =
                from_float<E>(d.beta[r0 + i] * y);
          }
    }
    // lower triangles: A = dP D, M = -dL' beta D with dL' = dY N^T
    float kk[4][4] = {}, qk[4][4] = {};
    auto krow = [&](int k, int j) { return K[j * ld + k]; };
    product<4>(kk, p.dk, [&](int i, int k) { return K[i * ld + k]; }, krow);
    product<4>(qk, p.dk, [&](int i, int k) { return Q[i * ld + k]; }, krow);
    float er[4] = {}, ec[4] = {}, ebeta[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + i, cc = lane16 + 16 * j;
        const float w = r >= cc ? decay_between(d, r, cc) : 0.f;
        const float x = p.scale * dp[i][j] * w;
        const float l = r > cc ? -dl[i][j] * w : 0.f;
        const float m = l * d.beta[r];
        A[r * kLdM + cc] = x;
        M[r * kLdM + cc] = m;
        const float e = fmaf(x, qk[i][j], m * kk[i][j]);
        er[i] += e;
        ec[j] += e;
        ebeta[i] = fmaf(l, kk[i][j], ebeta[i]);
      }
    // column sums of E: over the 16 row groups, through shared memory in order
    for (int g = 0; g < 16; ++g) {
      if ((tid >> 4) == g)
#pragma unroll
        for (int j = 0; j < 4; ++j) colsum[lane16 + 16 * j] += ec[j];
      __syncthreads();
    }
    float whole_cross = cross;
#pragma unroll
    for (int m = 16; m; m >>= 1) whole_cross += __shfl_xor_sync(0xFFFFFFFFu, whole_cross, m);
    if ((tid & 31) == 0) red[tid >> 5] = whole_cross;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i;
      const float g = decay_from_start(d, r), left = decay_between(d, kChunk - 1, r);
      float qt = 0.f, kt = 0.f, nt = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int cc = lane16 + 16 * j;
        if (cc < p.dk) {
          qt = fmaf(Q[r * ld + cc], to[i][j], qt);
          kt = fmaf(K[r * ld + cc], ty[i][j], kt);
          nt = fmaf(K[r * ld + cc], tn[i][j], nt);
        }
        gq[i][j] = fmaf(p.scale * g, to[i][j], gq[i][j]);
        gk[i][j] += left * tn[i][j] - g * d.beta[r] * ty[i][j];
      }
      float vals[5] = {qt, kt, nt, er[i], yv[i]}, eb = ebeta[i];
#pragma unroll
      for (int m = 8; m; m >>= 1) {
#pragma unroll
        for (int x = 0; x < 5; ++x) vals[x] += __shfl_xor_sync(0xFFFFFFFFu, vals[x], m);
        eb += __shfl_xor_sync(0xFFFFFFFFu, eb, m);
      }
      if (lane16 == 0) {
        rowsum[r] = p.scale * g * vals[0] - g * d.beta[r] * vals[1] + vals[3];
        grow[r] = left * vals[2];
        db[r] = vals[4] - g * vals[1] + eb;
      }
    }
    __syncthreads();
    product<8>(gq, kChunk, [&](int i, int k) { return A[i * kLdM + k]; },
               [&](int k, int j) { return j < p.dk ? K[k * ld + j] : 0.f; });
    product<8>(gk, kChunk, [&](int i, int k) { return A[k * kLdM + i]; },
               [&](int k, int j) { return j < p.dk ? Q[k * ld + j] : 0.f; });
    product<8>(gk, kChunk, [&](int i, int k) { return M[i * kLdM + k] + M[k * kLdM + i]; },
               [&](int k, int j) { return j < p.dk ? K[k * ld + j] : 0.f; });
    if (tid < c.len) {
      float s = 0.f;
      for (int w = 0; w < kThreads / 32; ++w) s += red[w];
      s *= decay_from_start(d, kChunk - 1);
      for (int i = 0; i < tid; ++i) s += grow[i];
      for (int i = tid; i < c.len; ++i) s += rowsum[i] - colsum[i];
      const int64_t at = row_at(p, c, p.Hv, hv, 1) + static_cast<int64_t>(tid) * p.Hv;
      store_gate(a.dg, at, gate16, s);
      store_gate(a.dbeta, at, gate16, db[tid]);
    }
  }
  auto put = [&](E* out) {
    return [&, out](int i, int j, float x) {
      if (i < c.len && j < p.dk) out[qk0 + i * qk_step + j] = from_float<E>(x);
    };
  };
  each(gq, put(dq_out));
  each(gk, put(dk_out));
}

int64_t chain_smem(const gsa_delta_t& p) {
  return 4LL * (2 * kChunk * (p.dk + 1) + 2 * kChunk * kLdM + p.dk * kLdC + 2 * kChunk * kLdC);
}
int64_t prep_smem(const gsa_delta_t& p) {
  return 4LL * (2 * kChunk * (p.dk + 1) + kChunk * kLdM);
}
int64_t grad_smem(const gsa_delta_t& p) {
  return 4LL * (2 * kChunk * (p.dk + 1) + 2 * p.dk * kLdC + 3 * kChunk * kLdC + 2 * kChunk * kLdM);
}

// The limits are set for the widest head, once.
gsa_delta_t widest() {
  gsa_delta_t p = {};
  p.dk = kDeltaMaxDk;
  return p;
}

template <typename E>
cudaError_t forward(const gsa_delta_t& p, void* o, float* final_state, bool save, void* ws,
                    cudaStream_t stream) {
  const Saved s = saved_at(p, ws);
  const Table t = table_at(ws, p.N);
  cudaError_t e = allow_smem<prep_kernel<E>>(static_cast<int>(prep_smem(widest())));
  if (e == cudaSuccess) e = allow_smem<chain_kernel<E>>(static_cast<int>(chain_smem(widest())));
  if (e != cudaSuccess) return e;
  const int64_t chunks = max_chunks(p);
  if (chunks > 0)
    prep_kernel<E><<<dim3(static_cast<unsigned>(chunks), p.Hv), kThreads, prep_smem(p), stream>>>(
        p, t, s.tiles);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const ChainArgs a = {t, s.tiles, save ? s.news : nullptr, save ? s.states : nullptr, o,
                       final_state};
  chain_kernel<E><<<dim3(p.cu_seqlens ? p.N + 2 : p.N, p.Hv, (p.dv + kCols - 1) / kCols),
                    kThreads, chain_smem(p), stream>>>(p, a);
  return cudaGetLastError();
}

template <typename E>
cudaError_t backward(const gsa_delta_t& p, const DeltaGrads& g, void* saved, void* scratch,
                     cudaStream_t stream) {
  const Saved s = saved_at(p, saved);
  const Scratch r = scratch_at(p, scratch);
  const Table t = table_at(saved, p.N);
  cudaError_t e = allow_smem<rev_kernel<E>>(static_cast<int>(chain_smem(widest())));
  if (e == cudaSuccess) e = allow_smem<grad_kernel<E>>(static_cast<int>(grad_smem(widest())));
  if (e != cudaSuccess) return e;
  const RevArgs ra = {t, s.tiles, g.dout, g.dfinal, r.back, r.states, g.dinitial};
  rev_kernel<E><<<dim3(p.N, p.Hv, (p.dv + kCols - 1) / kCols), kThreads, chain_smem(p), stream>>>(
      p, ra);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const GradArgs ga = {t,      s.news, s.states, r.back, r.states, g.dout,
                       g.dq,   g.dk,   g.dv,     g.dg,   g.dbeta};
  const int64_t chunks = max_chunks(p);
  if (chunks > 0)
    grad_kernel<E><<<dim3(static_cast<unsigned>(chunks), p.Hk), kThreads, grad_smem(p), stream>>>(
        p, ga);
  return cudaGetLastError();
}

}  // namespace

int64_t simt_saved_bytes(const gsa_delta_t& p, bool save) {
  const int64_t n = max_chunks(p) * p.Hv;
  return table_bytes(p) +
         4 * n * (tile_floats() + (save ? kChunk * p.dv + static_cast<int64_t>(p.dk) * p.dv : 0));
}
int64_t simt_scratch_bytes(const gsa_delta_t& p) {
  return 4 * max_chunks(p) * p.Hv * (kChunk * p.dv + static_cast<int64_t>(p.dk) * p.dv);
}

cudaError_t simt_forward(const gsa_delta_t& p, void* o, float* final_state, bool save, void* ws,
                         cudaStream_t stream) {
  return forward<float>(p, o, final_state, save, ws, stream);
}
cudaError_t simt_backward(const gsa_delta_t& p, const DeltaGrads& g, void* saved, void* scratch,
                          cudaStream_t stream) {
  return backward<float>(p, g, saved, scratch, stream);
}

}  // namespace delta
}  // namespace gsa
