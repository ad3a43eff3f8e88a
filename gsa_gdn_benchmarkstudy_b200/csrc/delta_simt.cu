// delta_simt.cu — the chunked gated delta rule, forward and backward, on the
// CUDA cores in fp32: fp32 inputs keep fp32's accuracy in every product, which
// the tensor cores' 16-bit operands do not give (delta_prep.cu, delta_seq.cu and
// delta_grad.cu serve bf16).
//
// Four kernels: `prep` makes T and P of every chunk, `chain` walks the chunks
// of a sequence forwards, `rev` walks them backwards with the state's gradient,
// `grad` turns what both left behind into gradients, chunk by chunk.  All
// products are 64 tokens (or channels) high; 256 threads hold 4 rows x NJ columns
// each, and take four steps of the contraction at a time, so that an operand whose
// neighbours are contracted comes in 16-byte loads.  Channels are padded to 64 or
// 128 with zeros, so every leading dimension is a constant, 4 past a multiple of 8
// words: 16-byte loads of eight rows then touch every bank once.
// Bound by shared memory (4 + NJ to 4 + 4 NJ loads for 16 NJ multiply-adds) and,
// with few sequences and heads, by the length of a chunk's chain of products: 2 x 333
// tokens, 4 heads of 64 x 96, take 10 us prep, 54 chain, 55 rev, 64 grad (465 us with a
// load for every value, copies that nothing overlaps, and a column a thread of T).
#include "delta_common.cuh"

namespace gsa {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 32;  // state columns of a block of chain / rev
constexpr int kLdC = kCols + 4;
template <int DK>
constexpr int kLdK = DK + 4;

// Operands of a product sum_k a(i, k) b(k, j), rows i = r0 .. r0 + 3 and columns
// j = c0 + 16 jj of a thread, k .. k + 3 at a time.
struct RowsA {  // a(i, k) = p[i ld + k]
  const float* p;
  int ld;
  __device__ __forceinline__ void load(float (&v)[4][4], int r0, int k) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(p + (r0 + i) * ld + k);
      v[0][i] = x.x, v[1][i] = x.y, v[2][i] = x.z, v[3][i] = x.w;
    }
  }
};
struct ColsA {  // a(i, k) = p[k ld + i]
  const float* p;
  int ld;
  __device__ __forceinline__ void load(float (&v)[4][4], int r0, int k) const {
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const float4 x = *reinterpret_cast<const float4*>(p + (k + z) * ld + r0);
      v[z][0] = x.x, v[z][1] = x.y, v[z][2] = x.z, v[z][3] = x.w;
    }
  }
};
struct RowsB {  // b(k, j) = p[j ld + k]
  const float* p;
  int ld;
  template <int NJ>
  __device__ __forceinline__ void load(float (&v)[4][NJ], int k, int c0) const {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(p + (c0 + 16 * j) * ld + k);
      v[0][j] = x.x, v[1][j] = x.y, v[2][j] = x.z, v[3][j] = x.w;
    }
  }
};
struct ColsB {  // b(k, j) = p[k ld + j]
  const float* p;
  int ld;
  template <int NJ>
  __device__ __forceinline__ void load(float (&v)[4][NJ], int k, int c0) const {
#pragma unroll
    for (int z = 0; z < 4; ++z)
#pragma unroll
      for (int j = 0; j < NJ; ++j) v[z][j] = p[(k + z) * ld + c0 + 16 * j];
  }
};
__device__ __forceinline__ int row0() { return (threadIdx.x >> 4) * 4; }
__device__ __forceinline__ int col0_of() { return threadIdx.x & 15; }
template <int NJ>
__device__ __forceinline__ void multiply(float (&acc)[4][NJ], const float (&a)[4][4],
                                         const float (&b)[4][NJ]) {
#pragma unroll
  for (int z = 0; z < 4; ++z)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = fmaf(a[z][i], b[z][j], acc[i][j]);
}
// acc += a b over k = first .. last - 1 (multiples of 4).
template <int NJ, typename A, typename B>
__device__ __forceinline__ void product(float (&acc)[4][NJ], int first, int last, A a, B b) {
#pragma unroll(NJ > 2 ? 2 : 4)
  for (int k = first; k < last; k += 4) {
    float av[4][4], bv[4][NJ];
    a.load(av, row0(), k);
    b.load(bv, k, col0_of());
    multiply(acc, av, bv);
  }
}
// Two left operands with one right one.
template <int NJ, typename A, typename B>
__device__ __forceinline__ void product2(float (&acc)[4][NJ], float (&more)[4][NJ], int last, A a,
                                         A a2, B b) {
#pragma unroll(NJ > 2 ? 2 : 4)
  for (int k = 0; k < last; k += 4) {
    float av[4][4], bv[4][NJ];
    b.load(bv, k, col0_of());
    a.load(av, row0(), k);
    multiply(acc, av, bv);
    a2.load(av, row0(), k);
    multiply(more, av, bv);
  }
}
// Left operands that are lower triangles (their transposes) end with a warp's last
// row (begin with its first).
__device__ __forceinline__ int lower_end() { return (row0() & ~7) + 8; }
__device__ __forceinline__ int upper_begin() { return row0() & ~7; }
template <int NJ, typename F>
__device__ __forceinline__ void each(float (&acc)[4][NJ], F f) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) f(row0() + i, col0_of() + 16 * j, acc[i][j]);
}

__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(real ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_begin() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// 64 rows of `limit` floats at any address, zeros past len rows and up to WIDTH columns.
template <int WIDTH>
__device__ __forceinline__ void load_rows(float* dst, int ld, const float* src, int64_t stride,
                                          int len, int limit) {
  const uint32_t to = smem_u32(dst);
#pragma unroll 4
  for (int i = threadIdx.x; i < kChunk * WIDTH; i += kThreads) {
    const int r = i / WIDTH, c = i % WIDTH;
    const bool real = r < len && c < limit;
    cp4(to + 4 * (r * ld + c), real ? src + r * stride + c : src, real);
  }
}
// ROWS rows of the workspace (16-byte aligned), zeros past `rows` and `limit`.
template <int ROWS, int WIDTH>
__device__ __forceinline__ void load_tile(float* dst, int ld, const float* src, int stride,
                                          int rows, int limit) {
  const uint32_t to = smem_u32(dst);
#pragma unroll 4
  for (int i = threadIdx.x; i < ROWS * WIDTH / 4; i += kThreads) {
    const int r = i / (WIDTH / 4), c = i % (WIDTH / 4) * 4;
    const bool real = r < rows && c < limit;
    cp16(to + 4 * (r * ld + c), real ? src + static_cast<int64_t>(r) * stride + c : src, real);
  }
}

// What prep leaves for each chunk and value head.
struct Tiles {
  float t[kChunk * kChunk], p[kChunk * kChunk];
  Gates gates;
};
__device__ __forceinline__ void load_gates(Gates* dst, const Gates* src) {
  if (threadIdx.x < sizeof(Gates) / 16)
    cp16(smem_u32(dst) + 16 * threadIdx.x, reinterpret_cast<const uint4*>(src) + threadIdx.x, true);
}

// Sections of the workspace (fp32), each with a slot for every chunk and head.
struct Saved {
  Tiles* tiles;
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
  s.tiles = reinterpret_cast<Tiles*>(static_cast<char*>(ws) + table_bytes(p));
  s.news = reinterpret_cast<float*>(s.tiles + n);
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

__device__ __forceinline__ const float* rows_at(const void* base, const int64_t (&stride)[3],
                                                const Chunk& c, int h) {
  return static_cast<const float*>(base) + c.b * stride[0] + c.begin * stride[1] + h * stride[2];
}
// Row `begin` of a contiguous [B, T, heads, width] tensor.
__device__ __forceinline__ int64_t row_at(const gsa_delta_t& p, const Chunk& c, int heads, int h,
                                          int width) {
  return ((static_cast<int64_t>(c.b) * p.T + c.begin) * heads + h) * width;
}

template <int DK>
__global__ void __launch_bounds__(kThreads) prep_kernel(const gsa_delta_t p, Table table,
                                                        Tiles* tiles) {
  extern __shared__ __align__(16) float sm[];
  constexpr int ld = kLdK<DK>;
  float* K = sm;
  float* Q = K + kChunk * ld;
  float* L = Q + kChunk * ld;
  __shared__ Decays d;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk), tid = threadIdx.x;
  const Chunk c = chunk_at(p, table, blockIdx.x);
  if (!c.valid || c.gap) return;
  load_rows<DK>(K, ld, rows_at(p.k, p.k_stride, c, hk), p.k_stride[1], c.len, p.dk);
  load_rows<DK>(Q, ld, rows_at(p.q, p.q_stride, c, hk), p.q_stride[1], c.len, p.dk);
  copies_begin();
  if (tid < 32) chunk_decays(p, c, hv, d);
  copies_done();
  __syncthreads();
  Tiles* out = tiles + static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
  if (tid < kChunk) {
    const float grown = decay_from_start(d, tid);
    out->gates.grown[tid] = grown;
    out->gates.beta[tid] = d.beta[tid];
    out->gates.left[tid] = decay_between(d, kChunk - 1, tid);
    out->gates.both[tid] = d.beta[tid] * grown;
    out->gates.hi[tid] = d.hi[tid];
    out->gates.lo[tid] = d.lo[tid];
  }
  float kk[4][4] = {}, qk[4][4] = {};
  product2(kk, qk, DK, RowsA{K, ld}, RowsA{Q, ld}, RowsB{K, ld});
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = row0() + i, cc = col0_of() + 16 * j;
      const float w = r >= cc ? decay_between(d, r, cc) : 0.f;
      L[r * kLdL + cc] = r > cc ? d.beta[r] * w * kk[i][j] : 0.f;
      out->p[r * kChunk + cc] = r >= cc ? p.scale * w * qk[i][j] : 0.f;
    }
  __syncthreads();
  invert(L);
  __syncthreads();
#pragma unroll
  for (int i = tid; i < kChunk * kChunk / 4; i += kThreads) {
    const int r = i / 16, cc = i % 16 * 4;
    reinterpret_cast<float4*>(out->t)[i] = r < 32 && cc >= 32
                                               ? make_float4(0.f, 0.f, 0.f, 0.f)
                                               : *reinterpret_cast<const float4*>(L + r * kLdL + cc);
  }
}

// A chunk's operands in shared memory.  64 channels: two sets, the next chunk's
// copies run beside this one's products; 128: one.
template <int DK>
struct Set {
  float K[kChunk * kLdK<DK>], Q[kChunk * kLdK<DK>], T[kChunk * kLdL], P[kChunk * kLdL];
  float D[kChunk * kLdC];  // V, or dO
  Gates gates;
};
template <int DK>
constexpr int kSets = DK == 64 ? 2 : 1;
template <int DK>
struct WalkSmem {
  Set<DK> set[kSets<DK>];
  float S[DK * kLdC], X[kChunk * kLdC], Y[kChunk * kLdC], Z[kChunk * kLdC];
};

// `rows`: V's or dO's (nullptr: zeros), from the block's first column on.
template <int DK>
__device__ __forceinline__ void fetch(const gsa_delta_t& p, const Chunk& c, int hk,
                                      const Tiles* tiles, const float* rows, int64_t stride,
                                      int cols, Set<DK>& s) {
  load_rows<DK>(s.K, kLdK<DK>, rows_at(p.k, p.k_stride, c, hk), p.k_stride[1], c.len, p.dk);
  load_rows<DK>(s.Q, kLdK<DK>, rows_at(p.q, p.q_stride, c, hk), p.q_stride[1], c.len, p.dk);
  load_tile<kChunk, kChunk>(s.T, kLdL, tiles->t, kChunk, kChunk, kChunk);
  load_tile<kChunk, kChunk>(s.P, kLdL, tiles->p, kChunk, kChunk, kChunk);
  load_rows<kCols>(s.D, kLdC, rows ? rows : reinterpret_cast<const float*>(tiles), stride,
                   rows ? c.len : 0, cols);
  load_gates(&s.gates, &tiles->gates);
  copies_begin();
}
// The state's columns from (zeros without it) and to [dk, dv].
template <int DK>
__device__ __forceinline__ void load_state(const gsa_delta_t& p, const float* src, int col0,
                                           float* S) {
  for (int i = threadIdx.x; i < DK * kCols; i += kThreads) {
    const int r = i / kCols, c = i % kCols;
    S[r * kLdC + c] =
        src && r < p.dk && col0 + c < p.dv ? src[static_cast<int64_t>(r) * p.dv + col0 + c] : 0.f;
  }
}
template <int DK>
__device__ __forceinline__ void store_state(const gsa_delta_t& p, const float* S, int col0,
                                            float* dst) {
  for (int i = threadIdx.x; i < p.dk * kCols; i += kThreads) {
    const int r = i / kCols, c = i % kCols;
    if (col0 + c < p.dv) dst[static_cast<int64_t>(r) * p.dv + col0 + c] = S[r * kLdC + c];
  }
}

struct ChainArgs {
  Table table;
  const Tiles* tiles;
  float* news;    // nullptr: inference
  float* states;
  float* o;
  float* final_state;
};

template <int DK>
__global__ void __launch_bounds__(kThreads) chain_kernel(const gsa_delta_t p, const ChainArgs a) {
  extern __shared__ __align__(16) float sm[];
  WalkSmem<DK>& w = *reinterpret_cast<WalkSmem<DK>*>(sm);
  constexpr int ld = kLdK<DK>;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk), col0 = blockIdx.z * kCols;
  const Seq s = sequence(p, a.table, blockIdx.x);
  if (s.gap) {  // rows of no sequence
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(s.len) * kCols; i += kThreads) {
      const int64_t r = s.begin + i / kCols;
      const int col = col0 + static_cast<int>(i % kCols);
      if (col < p.dv) a.o[(r * p.Hv + hv) * p.dv + col] = 0.f;
    }
    return;
  }
  const int64_t state0 = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  auto chunk = [&](int n) {
    const int left = s.len - n * kChunk;
    return Chunk{static_cast<int>(blockIdx.x), s.b, s.begin + n * kChunk,
                 left < kChunk ? left : kChunk, false, true};
  };
  auto load = [&](int n) {
    const Chunk c = chunk(n);
    fetch<DK>(p, c, hk, a.tiles + static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv,
              rows_at(p.v, p.v_stride, c, hv) + col0, p.v_stride[1], p.dv - col0,
              w.set[n % kSets<DK>]);
  };
  if (chunks > 0) load(0);
  load_state<DK>(p, p.initial_state ? p.initial_state + state0 : nullptr, col0, w.S);
  for (int n = 0; n < chunks; ++n) {
    const Chunk c = chunk(n);
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    if (kSets<DK> == 1 && n > 0) {
      __syncthreads();
      load(n);
    }
    copies_done();
    __syncthreads();
    if (kSets<DK> == 2 && n + 1 < chunks) load(n + 1);
    const Set<DK>& m = w.set[n % kSets<DK>];
    const Gates& g = m.gates;
    if (a.states) store_state<DK>(p, w.S, col0, a.states + slot * p.dk * p.dv);
    float ks[4][2] = {}, qs[4][2] = {};
    product2(ks, qs, DK, RowsA{m.K, ld}, RowsA{m.Q, ld}, ColsB{w.S, kLdC});
    each(ks, [&](int i, int j, float x) {  // beta (V - e^c K S)
      w.Y[i * kLdC + j] = g.beta[i] * m.D[i * kLdC + j] - g.both[i] * x;
    });
    __syncthreads();
    float nn[4][2] = {};
    product(nn, 0, lower_end(), RowsA{m.T, kLdL}, ColsB{w.Y, kLdC});
    each(nn, [&](int i, int j, float x) {
      w.X[i * kLdC + j] = x;
      w.Z[i * kLdC + j] = g.left[i] * x;
      if (a.news && col0 + j < p.dv) a.news[(slot * kChunk + i) * p.dv + col0 + j] = x;
    });
    __syncthreads();
    each(qs, [&](int i, int, float& x) { x *= p.scale * g.grown[i]; });
    product(qs, 0, lower_end(), RowsA{m.P, kLdL}, ColsB{w.X, kLdC});
    const int64_t o0 = row_at(p, c, p.Hv, hv, p.dv);
    each(qs, [&](int i, int j, float x) {
      if (i < c.len && col0 + j < p.dv)
        a.o[o0 + static_cast<int64_t>(i) * p.Hv * p.dv + col0 + j] = x;
    });
    const float whole = g.grown[kChunk - 1];
#pragma unroll
    for (int r = 0; r < DK; r += kChunk) {
      float st[4][2] = {};
      product(st, 0, kChunk, ColsA{m.K + r, ld}, ColsB{w.Z, kLdC});
      each(st, [&](int i, int j, float x) {
        float& to = w.S[(r + i) * kLdC + j];
        to = fmaf(whole, to, x);
      });
    }
  }
  if (a.final_state) {
    __syncthreads();
    store_state<DK>(p, w.S, col0, a.final_state + state0);
  }
}

struct RevArgs {
  Table table;
  const Tiles* tiles;
  const float* dout;          // contiguous, may be nullptr
  const float* dfinal;        // may be nullptr
  float* back;                // dY
  float* states;              // dS1
  float* dinitial;            // may be nullptr
};

// dN = P^T dO + diag(e^{c_64 - c}) K dS1,  dY = T^T dN,
// dS0 = e^{c_64} dS1 + K^T (-diag(e^c beta) dY) + Q^T (diag(scale e^c) dO).
template <int DK>
__global__ void __launch_bounds__(kThreads) rev_kernel(const gsa_delta_t p, const RevArgs a) {
  extern __shared__ __align__(16) float sm[];
  WalkSmem<DK>& w = *reinterpret_cast<WalkSmem<DK>*>(sm);
  constexpr int ld = kLdK<DK>;
  const int hv = blockIdx.y, hk = hv / (p.Hv / p.Hk), col0 = blockIdx.z * kCols;
  const Seq s = sequence(p, a.table, blockIdx.x);
  if (s.gap) return;
  const int64_t state0 = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  auto load = [&](int n) {
    const int left = s.len - n * kChunk;
    const Chunk c = {static_cast<int>(blockIdx.x), s.b, s.begin + n * kChunk,
                     left < kChunk ? left : kChunk, false, true};
    fetch<DK>(p, c, hk, a.tiles + static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv,
              a.dout ? a.dout + row_at(p, c, p.Hv, hv, p.dv) + col0 : nullptr,
              static_cast<int64_t>(p.Hv) * p.dv, p.dv - col0, w.set[n % kSets<DK>]);
  };
  if (chunks > 0) load(chunks - 1);
  load_state<DK>(p, a.dfinal ? a.dfinal + state0 : nullptr, col0, w.S);
  for (int n = chunks - 1; n >= 0; --n) {
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    if (kSets<DK> == 1 && n < chunks - 1) {
      __syncthreads();
      load(n);
    }
    copies_done();
    __syncthreads();
    if (kSets<DK> == 2 && n > 0) load(n - 1);
    const Set<DK>& m = w.set[n % kSets<DK>];
    const Gates& g = m.gates;
    store_state<DK>(p, w.S, col0, a.states + slot * p.dk * p.dv);
    float dn[4][2] = {};
    product(dn, 0, DK, RowsA{m.K, ld}, ColsB{w.S, kLdC});
    each(dn, [&](int i, int, float& x) { x *= g.left[i]; });
    product(dn, upper_begin(), kChunk, ColsA{m.P, kLdL}, ColsB{m.D, kLdC});
    each(dn, [&](int i, int j, float x) {
      w.X[i * kLdC + j] = x;
      w.Z[i * kLdC + j] = p.scale * g.grown[i] * m.D[i * kLdC + j];
    });
    __syncthreads();
    float dy[4][2] = {};
    product(dy, upper_begin(), kChunk, ColsA{m.T, kLdL}, ColsB{w.X, kLdC});
    each(dy, [&](int i, int j, float x) {
      if (col0 + j < p.dv) a.back[(slot * kChunk + i) * p.dv + col0 + j] = x;
      w.Y[i * kLdC + j] = -g.both[i] * x;
    });
    __syncthreads();
    const float whole = g.grown[kChunk - 1];
#pragma unroll
    for (int r = 0; r < DK; r += kChunk) {
      float ds[4][2] = {};
      product(ds, 0, kChunk, ColsA{m.K + r, ld}, ColsB{w.Y, kLdC});
      product(ds, 0, kChunk, ColsA{m.Q + r, ld}, ColsB{w.Z, kLdC});
      each(ds, [&](int i, int j, float x) {
        float& to = w.S[(r + i) * kLdC + j];
        to = fmaf(whole, to, x);
      });
    }
  }
  if (a.dinitial) {
    __syncthreads();
    store_state<DK>(p, w.S, col0, a.dinitial + state0);
  }
}

struct GradArgs {
  Table table;
  const Tiles* tiles;
  const float* news;     // N
  const float* states;   // S0
  const float* back;     // dY
  const float* dstates;  // dS1
  const float* dout;     // contiguous, may be nullptr
  float *dq, *dk, *dv;   // contiguous
  void *dg, *dbeta;
};
template <int DK>
struct GradSmem {
  float K[kChunk * kLdK<DK>], Q[kChunk * kLdK<DK>];
  float S0[DK * kLdC], S1[DK * kLdC];
  float D[kChunk * kLdC], N[kChunk * kLdC], Y[kChunk * kLdC];  // dO, N, dY
  float A[kChunk * kLdL], M[kChunk * kLdL];
  Gates gates;
  float columns[kThreads / 16][kChunk];  // shares of E's column sums
  float rowsum[kChunk], grow[kChunk], db[kChunk], red[kThreads / 32];
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
template <int DK>
__global__ void __launch_bounds__(kThreads) grad_kernel(const gsa_delta_t p, const GradArgs a) {
  extern __shared__ __align__(16) float sm[];
  GradSmem<DK>& w = *reinterpret_cast<GradSmem<DK>*>(sm);
  const Gates& g = w.gates;
  constexpr int ld = kLdK<DK>, NJ = DK / 16;
  const int hk = blockIdx.y, group = p.Hv / p.Hk, tid = threadIdx.x;
  const Chunk c = chunk_at(p, a.table, blockIdx.x);
  if (!c.valid) return;
  const int64_t qk0 = row_at(p, c, p.Hk, hk, p.dk);
  const int64_t qk_step = static_cast<int64_t>(p.Hk) * p.dk;
  const bool gate16 = p.gate_dtype == GSA_DTYPE_BF16;
  if (c.gap) {
    for (int64_t i = tid; i < static_cast<int64_t>(c.len) * p.dk; i += kThreads) {
      a.dq[qk0 + (i / p.dk) * qk_step + i % p.dk] = 0.f;
      a.dk[qk0 + (i / p.dk) * qk_step + i % p.dk] = 0.f;
    }
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      const int64_t v0 = row_at(p, c, p.Hv, h, p.dv), g0 = row_at(p, c, p.Hv, h, 1);
      for (int64_t i = tid; i < static_cast<int64_t>(c.len) * p.dv; i += kThreads)
        a.dv[v0 + (i / p.dv) * p.Hv * p.dv + i % p.dv] = 0.f;
      for (int i = tid; i < c.len; i += kThreads) {
        store_gate(a.dg, g0 + static_cast<int64_t>(i) * p.Hv, gate16, 0.f);
        store_gate(a.dbeta, g0 + static_cast<int64_t>(i) * p.Hv, gate16, 0.f);
      }
    }
    return;
  }
  load_rows<DK>(w.K, ld, rows_at(p.k, p.k_stride, c, hk), p.k_stride[1], c.len, p.dk);
  load_rows<DK>(w.Q, ld, rows_at(p.q, p.q_stride, c, hk), p.q_stride[1], c.len, p.dk);
  float gq[4][NJ] = {}, gk[4][NJ] = {};
  const int r0 = row0(), c0 = col0_of();
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
    float dp[4][4] = {}, dl[4][4] = {};
    float yv[4] = {}, qt[4] = {}, kt[4] = {}, nt[4] = {}, cross = 0.f;
    for (int col0 = 0; col0 < p.dv; col0 += kCols) {
      __syncthreads();  // what lies there is read
      if (col0 == 0) load_gates(&w.gates, &a.tiles[slot].gates);
      load_rows<kCols>(
          w.D, kLdC,
          a.dout ? a.dout + row_at(p, c, p.Hv, hv, p.dv) + col0
                 : reinterpret_cast<const float*>(a.tiles),
          static_cast<int64_t>(p.Hv) * p.dv, a.dout ? c.len : 0, p.dv - col0);
      const int64_t tokens = slot * kChunk * p.dv + col0, channels = slot * p.dk * p.dv + col0;
      load_tile<kChunk, kCols>(w.N, kLdC, a.news + tokens, p.dv, kChunk, p.dv - col0);
      load_tile<kChunk, kCols>(w.Y, kLdC, a.back + tokens, p.dv, kChunk, p.dv - col0);
      load_tile<DK, kCols>(w.S0, kLdC, a.states + channels, p.dv, p.dk, p.dv - col0);
      load_tile<DK, kCols>(w.S1, kLdC, a.dstates + channels, p.dv, p.dk, p.dv - col0);
      copies_begin();
      const float* v = rows_at(p.v, p.v_stride, c, hv) + col0;
      float vv[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          vv[i][j] = r0 + i < c.len && col0 + c0 + 16 * j < p.dv
                         ? v[(r0 + i) * p.v_stride[1] + c0 + 16 * j]
                         : 0.f;
      copies_done();
      __syncthreads();
      for (int i = tid; i < DK * kCols; i += kThreads) {
        const int at = i / kCols * kLdC + i % kCols;
        cross = fmaf(w.S0[at], w.S1[at], cross);
      }
      {
        float t[4][NJ] = {};
        product(t, 0, kCols, RowsA{w.D, kLdC}, RowsB{w.S0, kLdC});
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = p.scale * g.grown[r0 + i];
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            qt[i] = fmaf(w.Q[(r0 + i) * ld + c0 + 16 * j], t[i][j], qt[i]);
            gq[i][j] = fmaf(f, t[i][j], gq[i][j]);
          }
        }
      }
      {
        float t[4][NJ] = {};
        product(t, 0, kCols, RowsA{w.Y, kLdC}, RowsB{w.S0, kLdC});
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = -g.both[r0 + i];
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            kt[i] = fmaf(w.K[(r0 + i) * ld + c0 + 16 * j], t[i][j], kt[i]);
            gk[i][j] = fmaf(f, t[i][j], gk[i][j]);
          }
        }
      }
      {
        float t[4][NJ] = {};
        product(t, 0, kCols, RowsA{w.N, kLdC}, RowsB{w.S1, kLdC});
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = g.left[r0 + i];
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            nt[i] = fmaf(w.K[(r0 + i) * ld + c0 + 16 * j], t[i][j], nt[i]);
            gk[i][j] = fmaf(f, t[i][j], gk[i][j]);
          }
        }
      }
      product2(dp, dl, kCols, RowsA{w.D, kLdC}, RowsA{w.Y, kLdC}, RowsB{w.N, kLdC});
      const int64_t v0 = row_at(p, c, p.Hv, hv, p.dv) + col0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int cc = c0 + 16 * j;
          const float y = w.Y[(r0 + i) * kLdC + cc];
          yv[i] = fmaf(y, vv[i][j], yv[i]);
          if (r0 + i < c.len && col0 + cc < p.dv)
            a.dv[v0 + static_cast<int64_t>(r0 + i) * p.Hv * p.dv + cc] = g.beta[r0 + i] * y;
        }
    }
    // lower triangles: A = dP D, M = -dL' beta D with dL' = dY N^T
    float kk[4][4] = {}, qk[4][4] = {};
    product2(kk, qk, DK, RowsA{w.K, ld}, RowsA{w.Q, ld}, RowsB{w.K, ld});
    float er[4] = {}, ec[4] = {}, ebeta[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + i, cc = c0 + 16 * j;
        const float e =
            r >= cc ? expf((g.hi[r] - g.hi[cc]) + (g.lo[r] - g.lo[cc])) : 0.f;
        const float x = r >= cc ? p.scale * dp[i][j] * e : 0.f;
        const float l = r > cc ? -dl[i][j] * e : 0.f;
        const float m = l * g.beta[r];
        w.A[r * kLdL + cc] = x;
        w.M[r * kLdL + cc] = m;
        const float both = r >= cc ? fmaf(x, qk[i][j], m * kk[i][j]) : 0.f;
        er[i] += both;
        ec[j] += both;
        ebeta[i] = r > cc ? fmaf(l, kk[i][j], ebeta[i]) : ebeta[i];
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) w.columns[tid >> 4][c0 + 16 * j] = ec[j];
#pragma unroll
    for (int m = 16; m; m >>= 1) cross += __shfl_xor_sync(0xFFFFFFFFu, cross, m);
    if ((tid & 31) == 0) w.red[tid >> 5] = cross;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i;
      float vals[6] = {qt[i], kt[i], nt[i], er[i], yv[i], ebeta[i]};
#pragma unroll
      for (int m = 8; m; m >>= 1)
#pragma unroll
        for (int x = 0; x < 6; ++x) vals[x] += __shfl_xor_sync(0xFFFFFFFFu, vals[x], m);
      if (c0 == 0) {
        w.rowsum[r] = p.scale * g.grown[r] * vals[0] - g.both[r] * vals[1] + vals[3];
        w.grow[r] = g.left[r] * vals[2];
        w.db[r] = vals[4] - g.grown[r] * vals[1] + vals[5];
      }
    }
    __syncthreads();
    product(gq, 0, lower_end(), RowsA{w.A, kLdL}, ColsB{w.K, ld});
    product(gk, upper_begin(), kChunk, ColsA{w.A, kLdL}, ColsB{w.Q, ld});
    product(gk, 0, lower_end(), RowsA{w.M, kLdL}, ColsB{w.K, ld});
    product(gk, upper_begin(), kChunk, ColsA{w.M, kLdL}, ColsB{w.K, ld});
    if (tid < kChunk) {
      float net = w.rowsum[tid];
#pragma unroll
      for (int x = 0; x < kThreads / 16; ++x) net -= w.columns[x][tid];
      w.rowsum[tid] = net;
    }
    __syncthreads();
    if (tid < c.len) {
      float s = 0.f;
#pragma unroll
      for (int x = 0; x < kThreads / 32; ++x) s += w.red[x];
      s *= g.grown[kChunk - 1];
#pragma unroll 8
      for (int i = 0; i < kChunk; ++i) {
        const float before = w.grow[i], behind = i < c.len ? w.rowsum[i] : 0.f;
        s += i < tid ? before : behind;
      }
      const int64_t at = row_at(p, c, p.Hv, hv, 1) + static_cast<int64_t>(tid) * p.Hv;
      store_gate(a.dg, at, gate16, s);
      store_gate(a.dbeta, at, gate16, w.db[tid]);
    }
  }
  auto put = [&](float* out) {
    return [&, out](int i, int j, float x) {
      if (i < c.len && j < p.dk) out[qk0 + i * qk_step + j] = x;
    };
  };
  each(gq, put(a.dq));
  each(gk, put(a.dk));
}

template <int DK>
constexpr int kPrepSmem = 4 * (2 * kChunk * kLdK<DK> + kChunk * kLdL);

template <int DK>
cudaError_t forward(const gsa_delta_t& p, void* o, float* final_state, bool save, void* ws,
                    cudaStream_t stream) {
  const Saved s = saved_at(p, ws);
  const Table t = table_at(ws, p.N);
  cudaError_t e = allow_smem<prep_kernel<DK>>(kPrepSmem<DK>);
  if (e == cudaSuccess) e = allow_smem<chain_kernel<DK>>(sizeof(WalkSmem<DK>));
  if (e != cudaSuccess) return e;
  const int64_t chunks = max_chunks(p);
  if (chunks > 0)
    prep_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hv), kThreads, kPrepSmem<DK>,
                      stream>>>(p, t, s.tiles);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const ChainArgs a = {t, s.tiles, save ? s.news : nullptr, save ? s.states : nullptr,
                       static_cast<float*>(o), final_state};
  chain_kernel<DK><<<dim3(p.cu_seqlens ? p.N + 2 : p.N, p.Hv, (p.dv + kCols - 1) / kCols),
                     kThreads, sizeof(WalkSmem<DK>), stream>>>(p, a);
  return cudaGetLastError();
}

template <int DK>
cudaError_t backward(const gsa_delta_t& p, const DeltaGrads& g, void* saved, void* scratch,
                     cudaStream_t stream) {
  const Saved s = saved_at(p, saved);
  const Scratch r = scratch_at(p, scratch);
  const Table t = table_at(saved, p.N);
  const float* dout = static_cast<const float*>(g.dout);
  cudaError_t e = allow_smem<rev_kernel<DK>>(sizeof(WalkSmem<DK>));
  if (e == cudaSuccess) e = allow_smem<grad_kernel<DK>>(sizeof(GradSmem<DK>));
  if (e != cudaSuccess) return e;
  const RevArgs ra = {t, s.tiles, dout, g.dfinal, r.back, r.states, g.dinitial};
  rev_kernel<DK><<<dim3(p.N, p.Hv, (p.dv + kCols - 1) / kCols), kThreads, sizeof(WalkSmem<DK>),
                   stream>>>(p, ra);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const GradArgs ga = {t,        s.tiles,
                       s.news,   s.states,
                       r.back,   r.states,
                       dout,     static_cast<float*>(g.dq),
                       static_cast<float*>(g.dk), static_cast<float*>(g.dv),
                       g.dg,     g.dbeta};
  const int64_t chunks = max_chunks(p);
  if (chunks > 0)
    grad_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hk), kThreads, sizeof(GradSmem<DK>),
                      stream>>>(p, ga);
  return cudaGetLastError();
}

}  // namespace

int64_t simt_saved_bytes(const gsa_delta_t& p, bool save) {
  const int64_t n = max_chunks(p) * p.Hv;
  return table_bytes(p) +
         n * (static_cast<int64_t>(sizeof(Tiles)) +
              (save ? 4 * (kChunk * p.dv + static_cast<int64_t>(p.dk) * p.dv) : 0));
}
int64_t simt_scratch_bytes(const gsa_delta_t& p) {
  return 4 * max_chunks(p) * p.Hv * (kChunk * p.dv + static_cast<int64_t>(p.dk) * p.dv);
}

cudaError_t simt_forward(const gsa_delta_t& p, void* o, float* final_state, bool save, void* ws,
                         cudaStream_t stream) {
  return p.dk <= 64 ? forward<64>(p, o, final_state, save, ws, stream)
                    : forward<128>(p, o, final_state, save, ws, stream);
}
cudaError_t simt_backward(const gsa_delta_t& p, const DeltaGrads& g, void* saved, void* scratch,
                          cudaStream_t stream) {
  return p.dk <= 64 ? backward<64>(p, g, saved, scratch, stream)
                    : backward<128>(p, g, saved, scratch, stream);
}

}  // namespace delta
}  // namespace gsa
