// delta_prep.cu — the gated delta rule for bf16 inputs: what a chunk needs apart
// from any state, T = (I + L)^-1 and P (formulas: delta_common.cuh), for all chunks
// at once, and the launches of the forward and backward pass.
//
// One block a chunk and key head makes T and P of the value heads that share the
// key head.  Its two products (64 x 64 x dk) are mma.sync: they are small, and
// their results are wanted in registers, where the decays are applied.  T and P
// leave as hi + lo pairs of bf16, laid out as the shared-memory tiles that the
// sequential pass copies whole.  Bound by latency: loads, two products, a
// triangular inverse and 34 KB of stores one after the other; four blocks an SM
// overlap theirs.
#include "delta_tc.cuh"

namespace gsa {
namespace delta {
namespace {

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Right operand, stored [n][k]: the pieces of two n-tiles (rows n0 .. n0 + 15)
// and 16 columns (piece c, c + 1 of the whole row).  r[0], r[1]: first n-tile.
__device__ __forceinline__ uint32_t at_nk(uint32_t tile, int n0, int c) {
  const int l = threadIdx.x & 31, m = l >> 3;
  const int row = n0 + 8 * (m >> 1) + (l & 7), piece = c + (m & 1);
  return tile + (piece >> 3) * kTile + sw128_offset(row, piece & 7);
}
// Left operand, stored [m][k]: rows m0 .. m0 + 15, pieces c, c + 1.
__device__ __forceinline__ uint32_t at_mk(uint32_t tile, int m0, int c) {
  const int l = threadIdx.x & 31, m = l >> 3;
  const int row = m0 + 8 * (m & 1) + (l & 7), piece = c + (m >> 1);
  return tile + (piece >> 3) * kTile + sw128_offset(row, piece & 7);
}

// ---------------------------------------------------------------- prep
constexpr int kPrepThreads = 128;
constexpr int kLdL = kChunk + 4;
constexpr int kLdX = 36;

// K and Q, whose place P's tiles and a 32 x 32 product take once their products are
// in registers; L, which becomes T in place.
constexpr int kPrepTiles = 2 * static_cast<int>(kTile) + 32 * kLdX * 4;
template <int DK>
constexpr int prep_smem() {
  return (2 * (DK / 64) * static_cast<int>(kTile) > kPrepTiles ? 2 * (DK / 64) * static_cast<int>(kTile)
                                                               : kPrepTiles) +
         kChunk * kLdL * 4 + 1024;
}

// out = sign a b for N x N blocks, R x 4 a thread, k = 0 .. N - 1.  LOWER_B: b is lower
// triangular, k starts at the thread's first column, which a warp's threads nearly
// share; else a is, and k ends at its last row.
template <int N, int R, bool LOWER_B>
__device__ __forceinline__ void block_product(int t, const float* a, const float* b, int ldb,
                                              float* out, int ldo, float sign) {
  constexpr int kRows = N / R, kColGroups = N / 4;
  const int r = (LOWER_B ? t % kRows : t / kColGroups) * R;
  const int c = (LOWER_B ? t / kRows : t % kColGroups) * 4;
  float x[R][4] = {};
  const int first = LOWER_B ? c : 0, last = LOWER_B ? N : r + R;
#pragma unroll 4
  for (int k = first; k < last; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(b + k * ldb + c);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float u = a[(r + i) * kLdL + k];
      x[i][0] = fmaf(u, v.x, x[i][0]);
      x[i][1] = fmaf(u, v.y, x[i][1]);
      x[i][2] = fmaf(u, v.z, x[i][2]);
      x[i][3] = fmaf(u, v.w, x[i][3]);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    *reinterpret_cast<float4*>(out + (r + i) * ldo + c) =
        make_float4(sign * x[i][0], sign * x[i][1], sign * x[i][2], sign * x[i][3]);
}

// L (strictly lower, 64 x 64) becomes T = (I + L)^-1 in place, in fp32: the four
// 16 x 16 diagonal blocks by substitution, then T21 = -T22 L21 T11 twice over.
// A column a thread over all 64 rows took 2.5 times as long: half the threads
// idle, 64 values of a column in registers.
__device__ __forceinline__ void invert(float* L, float* X) {
  const int tid = threadIdx.x;
  {
    const int b = (tid & 63) >> 4, j = tid & 15;
    float* D = L + 16 * b * kLdL + 16 * b;
    float col[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == j ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) s = fmaf(-D[i * kLdL + m], col[m], s);
      col[i] = s;
    }
    __syncthreads();
    if (tid < 64)
#pragma unroll
      for (int i = 0; i < 16; ++i) D[i * kLdL + j] = col[i];
  }
  __syncthreads();
  const int b = (tid >> 6) * 32, t = tid & 63;
  float* D = L + b * kLdL + b;
  float* Y = X + (tid >> 6) * 16 * kLdX;
  block_product<16, 1, true>(t, D + 16 * kLdL, D, kLdL, Y, kLdX, 1.f);
  __syncthreads();
  block_product<16, 1, false>(t, D + 16 * kLdL + 16, Y, kLdX, D + 16 * kLdL, kLdL, -1.f);
  __syncthreads();
  block_product<32, 2, true>(tid, L + 32 * kLdL, L, kLdL, X, kLdX, 1.f);
  __syncthreads();
  block_product<32, 2, false>(tid, L + 32 * kLdL + 32, X, kLdX, L + 32 * kLdL, kLdL, -1.f);
  __syncthreads();
}

template <int DK>
__global__ void __launch_bounds__(kPrepThreads, 4) prep_kernel(const gsa_delta_t p, Table table,
                                                               Block* blocks) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull);
  __shared__ Decays d;
  const int hk = blockIdx.y, group = p.Hv / p.Hk, tid = threadIdx.x, lane = tid & 31;
  const int m0 = (tid >> 5) * 16, gid = lane >> 2, tig = lane & 3;
  const Chunk c = chunk_at(p, table, blockIdx.x);
  if (!c.valid || c.gap) return;
  const uint32_t K = smem_u32(smem), Q = K + (DK / 64) * kTile;
  float* X = reinterpret_cast<float*>(smem + 2 * kTile);
  float* L = reinterpret_cast<float*>(smem + prep_smem<DK>() - 1024) - kChunk * kLdL;
  copy_rows(K, rows_at(p.k, p.k_stride, c.b, c.begin, hk), p.k_stride[1], c.len, DK, p.dk, tid,
            kPrepThreads);
  copy_rows(Q, rows_at(p.q, p.q_stride, c.b, c.begin, hk), p.q_stride[1], c.len, DK, p.dk, tid,
            kPrepThreads);
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (tid < 32) chunk_decays(p, c, hk * group, d);  // beside the copies
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float kk[8][4] = {}, qk[8][4] = {};
#pragma unroll
  for (int ks = 0; ks < DK / 16; ++ks) {
    uint32_t ka[4], qa[4];
    ldsm(ka, at_mk(K, m0, 2 * ks));
    ldsm(qa, at_mk(Q, m0, 2 * ks));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (16 * j > m0) continue;  // above the diagonal
      uint32_t b[4];
      ldsm(b, at_nk(K, 16 * j, 2 * ks));
      mma(kk[2 * j], ka, b[0], b[1]);
      mma(kk[2 * j + 1], ka, b[2], b[3]);
      mma(qk[2 * j], qa, b[0], b[1]);
      mma(qk[2 * j + 1], qa, b[2], b[3]);
    }
  }
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    __syncthreads();  // K and Q, or the last head's tiles, are read
    if (hv > hk * group) {
      if (tid < 32) chunk_decays(p, c, hv, d);
      __syncthreads();
    }
    Block* blk = blocks + static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
    if (tid < kChunk) {
      const float grown = decay_from_start(d, tid);
      blk->gates.grown[tid] = grown;
      blk->gates.beta[tid] = d.beta[tid];
      blk->gates.left[tid] = decay_between(d, kChunk - 1, tid);
      blk->gates.both[tid] = d.beta[tid] * grown;
      blk->gates.hi[tid] = d.hi[tid];
      blk->gates.lo[tid] = d.lo[tid];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = m0 + gid + 8 * e;
      const float hi_r = d.hi[r], lo_r = d.lo[r], beta_r = d.beta[r];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int cc = 8 * j + 2 * tig;
        const uint32_t at = sw128_offset(r, j) + 4 * tig;
        if (8 * j > m0 + 8) {  // above the diagonal, for the whole warp
          *reinterpret_cast<float2*>(L + r * kLdL + cc) = make_float2(0.f, 0.f);
          *reinterpret_cast<uint32_t*>(smem + at) = 0;
          *reinterpret_cast<uint32_t*>(smem + kTile + at) = 0;
          continue;
        }
        const float2 hc = *reinterpret_cast<const float2*>(d.hi + cc);
        const float2 lc = *reinterpret_cast<const float2*>(d.lo + cc);
        float l[2], x[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const float w = exp_of((hi_r - (f ? hc.y : hc.x)) + (lo_r - (f ? lc.y : lc.x)));
          l[f] = r > cc + f ? beta_r * w * kk[j][2 * e + f] : 0.f;
          x[f] = r >= cc + f ? p.scale * w * qk[j][2 * e + f] : 0.f;
        }
        *reinterpret_cast<float2*>(L + r * kLdL + cc) = make_float2(l[0], l[1]);
        uint32_t hi, lo;
        split(x[0], x[1], hi, lo);
        *reinterpret_cast<uint32_t*>(smem + at) = hi;
        *reinterpret_cast<uint32_t*>(smem + kTile + at) = lo;
      }
    }
    __syncthreads();
    {  // P leaves while T is made
      uint4* dst = reinterpret_cast<uint4*>(blk->p_hi);
      const uint4* src = reinterpret_cast<const uint4*>(smem);
#pragma unroll
      for (int i = 0; i < kPBytes / 16 / kPrepThreads; ++i)
        dst[tid + i * kPrepThreads] = src[tid + i * kPrepThreads];
    }
    invert(L, X);
#pragma unroll
    for (int i = 0; i < kChunk * 8 / kPrepThreads; ++i) {
      const int x = tid + i * kPrepThreads, r = x >> 3, piece = x & 7;
      const float4 u = *reinterpret_cast<const float4*>(L + r * kLdL + piece * 8);
      const float4 v = *reinterpret_cast<const float4*>(L + r * kLdL + piece * 8 + 4);
      uint4 hi, lo;
      split(u.x, u.y, hi.x, lo.x);
      split(u.z, u.w, hi.y, lo.y);
      split(v.x, v.y, hi.z, lo.z);
      split(v.z, v.w, hi.w, lo.w);
      *reinterpret_cast<uint4*>(blk->t_hi + sw128_offset(r, piece)) = hi;
      *reinterpret_cast<uint4*>(blk->t_lo + sw128_offset(r, piece)) = lo;
    }
  }
}

template <int DK>
cudaError_t launch_prep(const gsa_delta_t& p, const Table& t, Block* blocks, cudaStream_t stream) {
  const int64_t chunks = max_chunks(p);
  if (chunks == 0) return cudaSuccess;
  const cudaError_t e = allow_smem<prep_kernel<DK>>(prep_smem<DK>());
  if (e != cudaSuccess) return e;
  prep_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hk), kPrepThreads, prep_smem<DK>(),
                    stream>>>(p, t, blocks);
  return cudaGetLastError();
}

}  // namespace

namespace {
// The segments' floats lie behind what the backward pass reads.
int64_t cuts_offset(const gsa_delta_t& p, bool save) {
  const int64_t n = max_chunks(p) * p.Hv;
  return (table_bytes(p) + n * (static_cast<int64_t>(sizeof(Block)) +
                                (save ? 2 * (news_elems(p) + state_elems(p)) : 0)) + 15) / 16 * 16;
}
}  // namespace

int64_t bf16_saved_bytes(const gsa_delta_t& p, bool save) {
  return cuts_offset(p, save) + 4 * segment_floats(p);
}
int64_t bf16_scratch_bytes(const gsa_delta_t& p) {
  return 2 * max_chunks(p) * p.Hv * (news_elems(p) + state_elems(p));
}
cudaError_t bf16_forward(const gsa_delta_t& p, const DeltaMaps& m, void* o, float* final_state,
                         bool save, void* ws, int* err, cudaStream_t stream) {
  const Saved s = saved_at(p, ws);
  const Table t = table_at(ws, p.N);
  const cudaError_t e = p.dk <= 64 ? launch_prep<64>(p, t, s.blocks, stream)
                                   : launch_prep<128>(p, t, s.blocks, stream);
  if (e != cudaSuccess) return e;
  SeqArgs a = {};
  a.table = t;
  a.blocks = s.blocks;
  a.out = o;
  a.state0 = p.initial_state;
  a.state1 = final_state;
  a.rows = save ? s.news : nullptr;
  a.states = save ? s.states : nullptr;
  a.err = err;
  return launch_forward(
      p, m, a, reinterpret_cast<float*>(static_cast<char*>(ws) + cuts_offset(p, save)), stream);
}
cudaError_t bf16_backward(const gsa_delta_t& p, const DeltaMaps& m, const DeltaMaps& more,
                          const DeltaGrads& g, void* saved, void* scratch, int* err,
                          cudaStream_t stream) {
  const Saved s = saved_at(p, saved);
  const Scratch r = scratch_at(p, scratch);
  const Table t = table_at(saved, p.N);
  SeqArgs a = {};
  a.table = t;
  a.blocks = s.blocks;
  a.in = g.dout;
  a.out = g.dv;
  a.state0 = g.dfinal;
  a.state1 = g.dinitial;
  a.rows = r.back;
  a.states = r.states;
  a.err = err;
  const cudaError_t e = launch_backward(p, more, a, stream);
  if (e != cudaSuccess) return e;
  return launch_grad(p, m, more, g, s, r, t, err, stream);
}

}  // namespace delta
}  // namespace gsa
