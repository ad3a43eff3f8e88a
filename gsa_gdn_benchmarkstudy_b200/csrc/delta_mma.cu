// delta_mma.cu — the chunked gated delta rule for bf16 inputs on the tensor
// cores, forward and backward (formulas: delta_common.cuh).
//
// `prep`   one block a chunk and key head: T = (I + L)^-1 and P of the value
//          heads that share the key head, written as the shared-memory images
//          that the next kernels copy whole.
// `chain`  one warp a sequence, value head and 16 columns of the state: S^T
//          [16, dk] stays in the warp's accumulators over the whole sequence.
//          Every product has S^T, Y^T or N^T on its left, whose accumulator
//          layout is the left operand's layout of mma.sync, so the sequential
//          path stays in registers.  What is not on that path (the outputs, or
//          backwards dO's own terms) is a second warp's, beside it.
// `rev`    the same backwards, with the state's gradient.
// `grad`   one block a chunk and key head: the gradients that contract over dv.
//
// mma.sync and not tcgen05: the sequential path is four dependent products a
// chunk, 16 columns wide at the least, with a pass over the elements between
// each two.  In registers that pass costs its arithmetic; through TMEM it costs
// a round trip of commit, load, convert, store and fence each time.
//
// Accuracy: q, k, v are exact in bf16.  Factors computed in fp32 on the
// sequential path (S, Y, N, T, P and their gradients) enter a product as a pair
// hi + lo of bf16, 16 bits together: 2^-17 of a value, so that states keep about
// fp32's accuracy over any number of chunks.  Sums are fp32.  The parallel
// `grad` rounds its factors to bf16 once (2^-9 of a value): its results are
// rounded to bf16 anyway.
#include "delta_common.cuh"

namespace gsa {
namespace delta {
namespace {

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stsm(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                     uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void stsm_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                       uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x, y as hi + lo pairs of bf16.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  lo = pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u));
}
// Left operand of 16 columns from two neighbouring accumulator tiles.
__device__ __forceinline__ void left(const float (&a)[4], const float (&b)[4], uint32_t (&hi)[4],
                                     uint32_t (&lo)[4]) {
  split(a[0], a[1], hi[0], lo[0]);
  split(a[2], a[3], hi[1], lo[1]);
  split(b[0], b[1], hi[2], lo[2]);
  split(b[2], b[3], hi[3], lo[3]);
}

// Tiles of 64 rows x 64 columns (128 bytes), 16-byte pieces swizzled by row; a
// wider matrix is one such tile after the other.
constexpr uint32_t kTile = 64 * 128;
// Right operand, stored [n][k]: the pieces of two n-tiles (rows n0 .. n0 + 15)
// and 16 columns (piece c, c + 1 of the whole row).  r[0], r[1]: first n-tile.
__device__ __forceinline__ uint32_t at_nk(uint32_t tile, int n0, int c) {
  const int l = threadIdx.x & 31, m = l >> 3;
  const int row = n0 + 8 * (m >> 1) + (l & 7), piece = c + (m & 1);
  return tile + (piece >> 3) * kTile + sw128_offset(row, piece & 7);
}
// Right operand, stored [k][n] (for ldsm_t): rows k0 .. k0 + 15, two n-tiles
// (pieces c, c + 1).  r[0], r[1]: first n-tile.
__device__ __forceinline__ uint32_t at_kn(uint32_t tile, int k0, int c) {
  const int l = threadIdx.x & 31, m = l >> 3;
  const int row = k0 + 8 * (m & 1) + (l & 7), piece = c + (m >> 1);
  return tile + (piece >> 3) * kTile + sw128_offset(row, piece & 7);
}
// Left operand, stored [m][k]: rows m0 .. m0 + 15, pieces c, c + 1.
__device__ __forceinline__ uint32_t at_mk(uint32_t tile, int m0, int c) {
  return at_kn(tile, m0, c);
}
// Left operand, stored [k][m] (for ldsm_t): rows k0 .. k0 + 15, pieces c, c + 1.
__device__ __forceinline__ uint32_t at_km(uint32_t tile, int k0, int c) {
  return at_nk(tile, k0, c);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------- workspace
// For each chunk and value head, T and P as pairs of swizzled tiles with the
// decays that go with them: the first half is the sequential warp's, the second
// the other's.
struct __align__(16) Block {
  unsigned char t_hi[kTile], t_lo[kTile];
  float grown[kChunk];  // e^{c_i}
  float beta[kChunk];
  float left[kChunk];   // e^{c_64 - c_i}
  float pad0[kChunk];
  unsigned char p_hi[kTile], p_lo[kTile];
  float grown_p[kChunk];
  float pad1[3 * kChunk];
};
constexpr int kHalf = 2 * static_cast<int>(kTile) + 1024;
static_assert(sizeof(Block) == 2 * kHalf, "block");

__host__ __device__ inline int blocks16(int dv) { return (dv + 15) / 16; }
__host__ __device__ inline int padded_dk(int dk) { return dk <= 64 ? 64 : 128; }

struct Saved {
  Block* blocks;
  __nv_bfloat16* news;    // N:  [slot][16 columns][64][16]      (training)
  __nv_bfloat16* states;  // S0: [slot][16 columns][16][dk]      (training)
};
struct Scratch {
  __nv_bfloat16* back;    // dY, as N
  __nv_bfloat16* states;  // dS1, as S0
};
int64_t news_bytes(const gsa_delta_t& p) { return 2LL * kChunk * 16 * blocks16(p.dv); }
int64_t state_bytes(const gsa_delta_t& p) { return 2LL * 16 * blocks16(p.dv) * padded_dk(p.dk); }
Saved saved_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  char* c = static_cast<char*>(ws) + table_bytes(p);
  Saved s;
  s.blocks = reinterpret_cast<Block*>(c);
  c += n * static_cast<int64_t>(sizeof(Block));
  s.news = reinterpret_cast<__nv_bfloat16*>(c);
  s.states = reinterpret_cast<__nv_bfloat16*>(c + n * news_bytes(p));
  return s;
}
Scratch scratch_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  char* c = static_cast<char*>(ws);
  return {reinterpret_cast<__nv_bfloat16*>(c),
          reinterpret_cast<__nv_bfloat16*>(c + n * news_bytes(p))};
}

using bf16 = __nv_bfloat16;

__device__ __forceinline__ const bf16* rows_at(const void* base, const int64_t (&stride)[3], int b,
                                               int64_t row, int h) {
  return static_cast<const bf16*>(base) + b * stride[0] + row * stride[1] + h * stride[2];
}

// 64 rows of `width` (<= limit real) columns into swizzled tiles, zeros past
// `len` and `limit`; by `threads` threads from thread `t` on.
__device__ __forceinline__ void copy_rows(uint32_t dst, const bf16* src, int64_t stride, int len,
                                          int width, int limit, int t, int threads) {
  const int pieces = width >> 3;
  for (int i = t; i < kChunk * pieces; i += threads) {
    const int r = i / pieces, c = i % pieces;
    const bool real = r < len && c * 8 < limit;
    cp16(dst + (c >> 3) * kTile + sw128_offset(r, c & 7), real ? src + r * stride + c * 8 : src,
         real);
  }
}

// ---------------------------------------------------------------- prep
constexpr int kPrepThreads = 128;
constexpr int kLdL = kChunk + 4;
constexpr int kLdX = 36;

// K and Q, whose place the block's image takes once their products are in
// registers; L, which becomes T in place; a 32 x 32 product.
template <int DK>
constexpr int prep_smem() {
  return (2 * (DK / 64) * static_cast<int>(kTile) > static_cast<int>(sizeof(Block))
              ? 2 * (DK / 64) * static_cast<int>(kTile)
              : static_cast<int>(sizeof(Block))) +
         (kChunk * kLdL + 32 * kLdX) * 4 + 1024;
}

// out[r][c] = sign sum_k a[r][k] b[k][c] for a 32 x 32 block, 2 x 4 a thread.
__device__ __forceinline__ void block32(const float* a, int lda, const float* b, int ldb,
                                        float* out, int ldo, float sign) {
  const int r = (threadIdx.x >> 3) * 2, c = (threadIdx.x & 7) * 4;
  float x[2][4] = {};
#pragma unroll 8
  for (int k = 0; k < 32; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(b + k * ldb + c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float u = a[(r + i) * lda + k];
      x[i][0] = fmaf(u, v.x, x[i][0]);
      x[i][1] = fmaf(u, v.y, x[i][1]);
      x[i][2] = fmaf(u, v.z, x[i][2]);
      x[i][3] = fmaf(u, v.w, x[i][3]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<float4*>(out + (r + i) * ldo + c) =
        make_float4(sign * x[i][0], sign * x[i][1], sign * x[i][2], sign * x[i][3]);
}
// The same for the two 16 x 16 blocks of a level, 64 threads and 1 x 4 each.
__device__ __forceinline__ void block16(const float* a, int lda, const float* b, int ldb,
                                        float* out, int ldo, float sign) {
  const int t = threadIdx.x & 63, r = t >> 2, c = (t & 3) * 4;
  float x[4] = {};
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(b + k * ldb + c);
    const float u = a[r * lda + k];
    x[0] = fmaf(u, v.x, x[0]);
    x[1] = fmaf(u, v.y, x[1]);
    x[2] = fmaf(u, v.z, x[2]);
    x[3] = fmaf(u, v.w, x[3]);
  }
  *reinterpret_cast<float4*>(out + r * ldo + c) =
      make_float4(sign * x[0], sign * x[1], sign * x[2], sign * x[3]);
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
  const int b = (tid >> 6) * 32;
  float* D = L + b * kLdL + b;
  float* Y = X + (tid >> 6) * 16 * kLdX;
  block16(D + 16 * kLdL, kLdL, D, kLdL, Y, kLdX, 1.f);
  __syncthreads();
  block16(D + 16 * kLdL + 16, kLdL, Y, kLdX, D + 16 * kLdL, kLdL, -1.f);
  __syncthreads();
  block32(L + 32 * kLdL, kLdL, L, kLdL, X, kLdX, 1.f);
  __syncthreads();
  block32(L + 32 * kLdL + 32, kLdL, X, kLdX, L + 32 * kLdL, kLdL, -1.f);
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
  Block* img = reinterpret_cast<Block*>(smem);
  float* L = reinterpret_cast<float*>(smem + prep_smem<DK>() - 1024) - kChunk * kLdL - 32 * kLdX;
  float* X = L + kChunk * kLdL;
  copy_rows(K, rows_at(p.k, p.k_stride, c.b, c.begin, hk), p.k_stride[1], c.len, DK, p.dk, tid,
            kPrepThreads);
  copy_rows(Q, rows_at(p.q, p.q_stride, c.b, c.begin, hk), p.q_stride[1], c.len, DK, p.dk, tid,
            kPrepThreads);
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  if (tid < 32) chunk_decays(p, c, hk * group, d);
  __syncthreads();
  float kk[8][4] = {}, qk[8][4] = {};
#pragma unroll
  for (int ks = 0; ks < DK / 16; ++ks) {
    uint32_t ka[4], qa[4];
    ldsm(ka, at_mk(K, m0, 2 * ks));
    ldsm(qa, at_mk(Q, m0, 2 * ks));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t b[4];
      ldsm(b, at_nk(K, 16 * j, 2 * ks));
      mma(kk[2 * j], ka, b[0], b[1]);
      mma(kk[2 * j + 1], ka, b[2], b[3]);
      mma(qk[2 * j], qa, b[0], b[1]);
      mma(qk[2 * j + 1], qa, b[2], b[3]);
    }
  }
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    __syncthreads();  // K and Q, or the last head's image, are read
    if (hv > hk * group) {
      if (tid < 32) chunk_decays(p, c, hv, d);
      __syncthreads();
    }
    if (tid < kChunk) {
      img->grown[tid] = img->grown_p[tid] = decay_from_start(d, tid);
      img->beta[tid] = d.beta[tid];
      img->left[tid] = decay_between(d, kChunk - 1, tid);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = m0 + gid + 8 * e, cc = 8 * j + 2 * tig;
        float l[2] = {0.f, 0.f}, x[2] = {0.f, 0.f};
#pragma unroll
        for (int f = 0; f < 2; ++f)
          if (r >= cc + f) {
            const float w = decay_between(d, r, cc + f);
            if (r > cc + f) l[f] = d.beta[r] * w * kk[j][2 * e + f];
            x[f] = p.scale * w * qk[j][2 * e + f];
          }
        *reinterpret_cast<float2*>(L + r * kLdL + cc) = make_float2(l[0], l[1]);
        uint32_t hi, lo;
        split(x[0], x[1], hi, lo);
        const uint32_t at = sw128_offset(r, j) + 4 * tig;
        *reinterpret_cast<uint32_t*>(img->p_hi + at) = hi;
        *reinterpret_cast<uint32_t*>(img->p_lo + at) = lo;
      }
    __syncthreads();
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
      *reinterpret_cast<uint4*>(img->t_hi + sw128_offset(r, piece)) = hi;
      *reinterpret_cast<uint4*>(img->t_lo + sw128_offset(r, piece)) = lo;
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(blocks + static_cast<int64_t>(blockIdx.x) * p.Hv + hv);
    const uint4* src = reinterpret_cast<const uint4*>(img);
    for (int i = tid; i < static_cast<int>(sizeof(Block) / 16); i += kPrepThreads) dst[i] = src[i];
  }
}

// ---------------------------------------------------------------- chain and rev
// A block has W pairs of warps and one warp that copies.  Of a pair, the first
// warp walks the state, the second has what is off that path.  Two queues of
// kStages stages: A for the first warps (K, T and decays), B for the second (Q, P
// and decays); 64 x 16 values for each pair go with A (v) or with B (dO).
constexpr int kStages = 2;
template <int DK>
__host__ __device__ constexpr int tile_bytes() { return (DK / 64) * static_cast<int>(kTile); }
template <int DK>
__host__ __device__ constexpr int queue_bytes() { return tile_bytes<DK>() + kHalf; }
// What a pair shares: S^T and N^T as operands (forwards), or the second warp's
// part of dN^T and of dS^T (backwards); and the second (backwards: first) warp's
// staging area for rows that leave.
template <int DK>
__host__ __device__ constexpr int state_share() { return DK * 64; }
template <int DK>
__host__ __device__ constexpr int pair_bytes() { return state_share<DK>() + 4096; }
template <int DK>
__host__ __device__ constexpr int staging_bytes() { return 16 * (DK * 2 + 16); }
template <int DK>
__host__ __device__ constexpr int seq_smem(int W) {
  return kStages * (2 * queue_bytes<DK>() + W * 2048) +
         W * (pair_bytes<DK>() + staging_bytes<DK>()) + 1024;
}

struct SeqArgs {
  Table table;
  const Block* blocks;
  // chain: out o, state0 initial, state1 final.  rev: out dv, state0 dfinal,
  // state1 dinitial, in dO.
  const void* in;        // rev: dO, contiguous; may be nullptr
  void* out;
  const float* state0;   // may be nullptr: zeros
  float* state1;         // may be nullptr
  bf16* rows;            // N (chain, nullptr: inference) or dY
  bf16* states;          // S0 or dS1
  int* err;
};

struct SeqBars {
  uint64_t full_a[kStages], empty_a[kStages], full_b[kStages], empty_b[kStages];
  uint64_t s_full[8], s_free[8], n_full[8], n_free[8];  // by pair
  int abort;
};

template <int DK>
struct SeqSmem {
  unsigned char* base;
  int W;
  __device__ unsigned char* a(int st) const { return base + st * queue_bytes<DK>(); }
  __device__ unsigned char* b(int st) const { return base + (kStages + st) * queue_bytes<DK>(); }
  __device__ unsigned char* v(int st, int pair) const {
    return base + 2 * kStages * queue_bytes<DK>() + (st * W + pair) * 2048;
  }
  __device__ unsigned char* pair(int i) const {
    return v(kStages, 0) + i * (pair_bytes<DK>() + staging_bytes<DK>());
  }
};

__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* map, int x, int h,
                                              int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

// The copies of a sequence's chunks, by one warp.  Rows past the tensor's end
// come out of TMA as zeros; a chunk that ends before its 64th row inside a packed
// batch, where another sequence follows, takes its rows one by one.
template <int DK, bool REV>
__device__ __forceinline__ void produce(const gsa_delta_t& p, const DeltaMaps& maps,
                                        const SeqArgs& a, const Seq& s, int hv, int col0, int W,
                                        const SeqSmem<DK>& sm, SeqBars& bars) {
  const int lane = threadIdx.x & 31, hk = hv / (p.Hv / p.Hk);
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const bool have = !REV || a.in != nullptr;
  int na = 0, nb = 0;  // chunks begun of each queue
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, parity = ((n / kStages) & 1) ^ 1;
    const int at = REV ? chunks - 1 - n : n;
    const int begin = s.begin + at * kChunk, rest = s.len - at * kChunk;
    const int len = rest < kChunk ? rest : kChunk;
    const bool whole = len == kChunk || !p.cu_seqlens;
    const Block* blk = a.blocks + static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint64_t* full = q ? &bars.full_b[st] : &bars.full_a[st];
      if (!mbar_wait_warp(q ? &bars.empty_b[st] : &bars.empty_a[st], parity, a.err, &bars.abort))
        goto done;
      unsigned char* dst = q ? sm.b(st) : sm.a(st);
      const bool values = (q == 1) == REV;
      const bool tma_values = values && whole && have;
      if (lane == 0) {
        mbar_arrive_expect_tx(full, kHalf + (whole ? tile_bytes<DK>() : 0) +
                                        (tma_values ? W * 2048 : 0));
        bulk_load(dst + tile_bytes<DK>(), reinterpret_cast<const unsigned char*>(blk) + q * kHalf,
                  kHalf, full);
        if (whole)
          for (int i = 0; i < DK / 64; ++i)
            tma_load_rows(dst + i * kTile, q ? &maps.q : &maps.k, 64 * i, hk, begin, s.b, full);
        if (tma_values)
          for (int i = 0; i < W; ++i)
            tma_load_rows(sm.v(st, i), &maps.v, col0 + 16 * i, hv, begin, s.b, full);
      }
      if (!whole)
        copy_rows(smem_u32(dst),
                  q ? rows_at(p.q, p.q_stride, s.b, begin, hk)
                    : rows_at(p.k, p.k_stride, s.b, begin, hk),
                  q ? p.q_stride[1] : p.k_stride[1], len, DK, p.dk, lane, 32);
      if (values && !tma_values) {
        const int64_t stride = REV ? static_cast<int64_t>(p.Hv) * p.dv : p.v_stride[1];
        const bf16* v = REV ? static_cast<const bf16*>(a.in) +
                                  (have ? (static_cast<int64_t>(s.b) * p.T + begin) * stride +
                                              hv * p.dv
                                        : 0)
                            : rows_at(p.v, p.v_stride, s.b, begin, hv);
        for (int i = lane; i < kChunk * 2 * W; i += 32) {
          const int r = i / (2 * W), c = i % (2 * W), col = col0 + c * 8;
          const bool real = have && r < len && col < p.dv;
          cp16(smem_u32(sm.v(st, c >> 1)) + r * 32 + (c & 1) * 16,
               real ? v + r * stride + col : static_cast<const bf16*>(p.k), real);
        }
      }
      cp_arrive(full);
      if (q) ++nb; else ++na;
    }
  }
done:
  if (nb < chunks) {  // gave up: no copy of ours may outlive the block
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int i = na > kStages ? na - kStages : 0; i < na; ++i)
      mbar_wait_drain(&bars.full_a[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
    for (int i = nb > kStages ? nb - kStages : 0; i < nb; ++i)
      mbar_wait_drain(&bars.full_b[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
  }
}

__device__ __forceinline__ uint32_t at_v(uint32_t tile, int t0) {  // ldsm_t: see below
  const int l = threadIdx.x & 31, m = l >> 3;
  return tile + (t0 + 8 * (m >> 1) + (l & 7)) * 32 + (m & 1) * 16;
}
// Accumulator pieces of [16 columns, 64 tokens] from a warp's [64][16] tile:
// r[0], r[1]: tokens t0 + 2 tig (+1) of columns gid and gid + 8, r[2], r[3]: t0 + 8 on.
// The same four registers are the left operand [16 columns, tokens t0 .. t0 + 15].
__device__ __forceinline__ void load_v(uint32_t (&r)[4], uint32_t tile, int t0) {
  ldsm_t(r, at_v(tile, t0));
}
__device__ __forceinline__ float lo_of(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float hi_of(uint32_t r) { return __uint_as_float(r & 0xFFFF0000u); }

// [16 columns, 64 tokens] accumulators, times `by` (a value a token), as bf16 to
// the warp's staging area [64][16].
__device__ __forceinline__ void stage_rows(const float (&x)[8][4], uint32_t staging) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    stsm_t(at_v(staging, 8 * j), pack_bf16x2(x[j][0], x[j][1]), pack_bf16x2(x[j][2], x[j][3]),
           pack_bf16x2(x[j + 1][0], x[j + 1][1]), pack_bf16x2(x[j + 1][2], x[j + 1][3]));
  __syncwarp();
}
// ... from there to rows of a contiguous [.., Hv, dv] tensor
__device__ __forceinline__ void put_rows(const unsigned char* staging, bf16* dst, int64_t stride,
                                         int len, int col, int dv) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (lane + 32 * i) >> 1, c = (lane & 1) * 8;
    if (r < len && col + c < dv)
      *reinterpret_cast<uint4*>(dst + r * stride + c) =
          *reinterpret_cast<const uint4*>(staging + r * 32 + c * 2);
  }
}
__device__ __forceinline__ void put_block(const unsigned char* staging, bf16* dst) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<uint4*>(dst)[lane + 32 * i] =
        reinterpret_cast<const uint4*>(staging)[lane + 32 * i];
}
// S^T [16, DK] in bf16 by way of the staging area, to dst [16][DK]: columns
// 16 ks .. 16 ks + 15, as a left operand.
template <int DK>
__device__ __forceinline__ void stage_state(const uint32_t (&r)[4], int ks, uint32_t staging) {
  const int lane = threadIdx.x & 31, m = lane >> 3;
  stsm(staging + (8 * (m & 1) + (lane & 7)) * (DK * 2 + 16) + (2 * ks + (m >> 1)) * 16, r[0], r[1],
       r[2], r[3]);
}
template <int DK>
__device__ __forceinline__ void put_state(const unsigned char* staging, bf16* dst) {
  const int lane = threadIdx.x & 31;
  constexpr int kPieces = DK / 8;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16 * kPieces / 32; ++i) {
    const int x = lane + 32 * i, r = x / kPieces, c = x % kPieces;
    *reinterpret_cast<uint4*>(dst + r * DK + c * 8) =
        *reinterpret_cast<const uint4*>(staging + r * (DK * 2 + 16) + c * 16);
  }
  __syncwarp();
}
// S^T from / to a state [dk, dv] in fp32.
template <int DK, bool STORE, typename P>
__device__ __forceinline__ void move_state(float (&S)[DK / 8][4], P* state, int dk, int dv,
                                           int col) {
  const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
#pragma unroll
  for (int j = 0; j < DK / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 8 * j + 2 * tig + (e & 1), c = col + gid + 8 * (e >> 1);
      if (r < dk && c < dv) {
        if constexpr (STORE)
          state[static_cast<int64_t>(r) * dv + c] = S[j][e];
        else
          S[j][e] = state[static_cast<int64_t>(r) * dv + c];
      }
    }
}

// acc [16, 64 tokens] += S^T [16, DK] X^T, X a [64][DK] tile: columns 16 ks on.
template <int DK>
__device__ __forceinline__ void times_rows(float (&acc)[8][4], const uint32_t (&hi)[4],
                                           const uint32_t (&lo)[4], uint32_t X, int ks) {
  uint32_t b[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) ldsm(b[j], at_nk(X, 16 * j, 2 * ks));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mma(acc[2 * j], hi, b[j][0], b[j][1]);
    mma(acc[2 * j + 1], hi, b[j][2], b[j][3]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mma(acc[2 * j], lo, b[j][0], b[j][1]);
    mma(acc[2 * j + 1], lo, b[j][2], b[j][3]);
  }
}
// S^T [16, DK] += X^T [16, tokens 16 ks ..] Y, Y a [64][DK] tile.
template <int DK>
__device__ __forceinline__ void add_outer(float (&S)[DK / 8][4], const uint32_t (&hi)[4],
                                          const uint32_t (&lo)[4], uint32_t Y, int ks) {
#pragma unroll
  for (int j0 = 0; j0 < DK / 16; j0 += 4) {
    uint32_t b[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) ldsm_t(b[j], at_kn(Y, 16 * ks, 2 * (j0 + j)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mma(S[2 * (j0 + j)], hi, b[j][0], b[j][1]);
      mma(S[2 * (j0 + j) + 1], hi, b[j][2], b[j][3]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mma(S[2 * (j0 + j)], lo, b[j][0], b[j][1]);
      mma(S[2 * (j0 + j) + 1], lo, b[j][2], b[j][3]);
    }
  }
}
// acc [16, 64 tokens] += X^T [16, 64] M^T (COLUMNS: X^T M), M a lower triangle
// [64][64] held as a pair, X a pair (PAIR) or exact.  The left operands of the
// outer loop are independent of one another, the accumulators of the inner one.
template <bool COLUMNS, bool PAIR>
__device__ __forceinline__ void times_triangle(float (&acc)[8][4], const uint32_t (&hi)[4][4],
                                               const uint32_t (&lo)[4][4], uint32_t M) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    // rows: token tiles j >= ks meet the tokens of ks; columns: j <= ks
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (COLUMNS ? j > ks : j < ks) continue;
      uint32_t b[4], c[4];
      if constexpr (COLUMNS) {
        ldsm_t(b, at_kn(M, 16 * ks, 2 * j));
        ldsm_t(c, at_kn(M + kTile, 16 * ks, 2 * j));
      } else {
        ldsm(b, at_nk(M, 16 * j, 2 * ks));
        ldsm(c, at_nk(M + kTile, 16 * j, 2 * ks));
      }
      mma(acc[2 * j], hi[ks], b[0], b[1]);
      mma(acc[2 * j + 1], hi[ks], b[2], b[3]);
      if constexpr (PAIR) {
        mma(acc[2 * j], lo[ks], b[0], b[1]);
        mma(acc[2 * j + 1], lo[ks], b[2], b[3]);
      }
      mma(acc[2 * j], hi[ks], c[0], c[1]);
      mma(acc[2 * j + 1], hi[ks], c[2], c[3]);
    }
  }
}

struct Place {
  int pair, col;  // the pair's first column of the value head
  unsigned char* share;
  unsigned char* staging;
};
__device__ __forceinline__ void signal(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Chunks in order, the state's warp: N = T diag(beta) (V - diag(e^c) K S),
// S <- e^{c_64} S + K^T diag(e^{c_64 - c}) N, all transposed.
template <int DK>
__device__ __forceinline__ void chain_state(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                            int hv, const Place& w, const SeqSmem<DK>& sm,
                                            SeqBars& bars) {
  const int lane = threadIdx.x & 31, tig = lane & 3;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const int64_t head = static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
  uint4* s_share = reinterpret_cast<uint4*>(w.share);
  uint4* n_share = reinterpret_cast<uint4*>(w.share + state_share<DK>());
  float S[DK / 8][4] = {};
  if (a.state0) move_state<DK, false>(S, a.state0 + head * p.dk * p.dv, p.dk, p.dv, w.col);
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages;
    if (!mbar_wait_warp(&bars.full_a[st], (n / kStages) & 1, a.err, &bars.abort)) return;
    if (!mbar_wait_warp(&bars.s_free[w.pair], (n & 1) ^ 1, a.err, &bars.abort)) return;
    const uint32_t K = smem_u32(sm.a(st));
    const Block* blk = reinterpret_cast<const Block*>(sm.a(st) + tile_bytes<DK>());
    const uint32_t T = smem_u32(blk->t_hi), V = smem_u32(sm.v(st, w.pair));

    float R[8][4] = {};
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
      uint32_t hi[4], lo[4];
      left(S[2 * ks], S[2 * ks + 1], hi, lo);
      s_share[(2 * ks) * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      s_share[(2 * ks + 1) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      times_rows<DK>(R, hi, lo, K, ks);
    }
    signal(&bars.s_full[w.pair]);
    uint32_t yh[4][4], yl[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t v[4];
      load_v(v, V, 16 * j);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 16 * j + 8 * e + 2 * tig;
        const float2 g = *reinterpret_cast<const float2*>(blk->grown + t);
        const float2 b = *reinterpret_cast<const float2*>(blk->beta + t);
        float(&r)[4] = R[2 * j + e];
        r[0] = b.x * (lo_of(v[2 * e]) - g.x * r[0]);
        r[1] = b.y * (hi_of(v[2 * e]) - g.y * r[1]);
        r[2] = b.x * (lo_of(v[2 * e + 1]) - g.x * r[2]);
        r[3] = b.y * (hi_of(v[2 * e + 1]) - g.y * r[3]);
      }
      left(R[2 * j], R[2 * j + 1], yh[j], yl[j]);
    }
    float N[8][4] = {};
    times_triangle<false, true>(N, yh, yl, T);
    if (!mbar_wait_warp(&bars.n_free[w.pair], (n & 1) ^ 1, a.err, &bars.abort)) return;
    const float whole = blk->grown[kChunk - 1];
#pragma unroll
    for (int j = 0; j < DK / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[j][e] *= whole;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t hi[4], lo[4];
      left(N[2 * ks], N[2 * ks + 1], hi, lo);
      n_share[(2 * ks) * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      n_share[(2 * ks + 1) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    signal(&bars.n_full[w.pair]);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 g = *reinterpret_cast<const float2*>(blk->left + 16 * ks + 8 * e + 2 * tig);
#pragma unroll
        for (int f = 0; f < 4; ++f) N[2 * ks + e][f] *= f & 1 ? g.y : g.x;
      }
      uint32_t hi[4], lo[4];
      left(N[2 * ks], N[2 * ks + 1], hi, lo);
      add_outer<DK>(S, hi, lo, K, ks);
    }
    signal(&bars.empty_a[st]);
  }
  if (a.state1) move_state<DK, true>(S, a.state1 + head * p.dk * p.dv, p.dk, p.dv, w.col);
}

// ... and its companion: O = scale diag(e^c) Q S + P N, and what training keeps.
template <int DK>
__device__ __forceinline__ void chain_output(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                             int hv, const Place& w, const SeqSmem<DK>& sm,
                                             SeqBars& bars) {
  const int lane = threadIdx.x & 31, tig = lane & 3;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const uint4* s_share = reinterpret_cast<const uint4*>(w.share);
  const uint4* n_share = reinterpret_cast<const uint4*>(w.share + state_share<DK>());
  const uint32_t staging = smem_u32(w.staging);
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages;
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    if (!mbar_wait_warp(&bars.full_b[st], (n / kStages) & 1, a.err, &bars.abort)) return;
    if (!mbar_wait_warp(&bars.s_full[w.pair], n & 1, a.err, &bars.abort)) return;
    const uint32_t Q = smem_u32(sm.b(st)), P = Q + tile_bytes<DK>();
    const float* grown = reinterpret_cast<const float*>(sm.b(st) + tile_bytes<DK>() + 2 * kTile);
    float O[8][4] = {};
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
      const uint4 h = s_share[(2 * ks) * 32 + lane], l = s_share[(2 * ks + 1) * 32 + lane];
      const uint32_t hi[4] = {h.x, h.y, h.z, h.w}, lo[4] = {l.x, l.y, l.z, l.w};
      times_rows<DK>(O, hi, lo, Q, ks);
      if (a.states) stage_state<DK>(hi, ks, staging);
    }
    signal(&bars.s_free[w.pair]);
    if (a.states)
      put_state<DK>(w.staging, a.states + (slot * blocks16(p.dv) + w.col / 16) * 16 * DK);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 g = *reinterpret_cast<const float2*>(grown + 8 * j + 2 * tig);
#pragma unroll
      for (int f = 0; f < 4; ++f) O[j][f] *= p.scale * (f & 1 ? g.y : g.x);
    }
    if (!mbar_wait_warp(&bars.n_full[w.pair], n & 1, a.err, &bars.abort)) return;
    uint32_t hi[4][4], lo[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const uint4 h = n_share[(2 * ks) * 32 + lane], l = n_share[(2 * ks + 1) * 32 + lane];
      hi[ks][0] = h.x; hi[ks][1] = h.y; hi[ks][2] = h.z; hi[ks][3] = h.w;
      lo[ks][0] = l.x; lo[ks][1] = l.y; lo[ks][2] = l.z; lo[ks][3] = l.w;
    }
    signal(&bars.n_free[w.pair]);
    times_triangle<false, true>(O, hi, lo, P);
    signal(&bars.empty_b[st]);
    stage_rows(O, staging);
    put_rows(w.staging,
             static_cast<bf16*>(a.out) +
                 ((static_cast<int64_t>(s.b) * p.T + s.begin + n * kChunk) * p.Hv + hv) * p.dv +
                 w.col,
             static_cast<int64_t>(p.Hv) * p.dv, min(kChunk, s.len - n * kChunk), w.col, p.dv);
    __syncwarp();
    if (a.rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        stsm_t(at_v(staging, 16 * j), hi[j][0], hi[j][1], hi[j][2], hi[j][3]);
      __syncwarp();
      put_block(w.staging, a.rows + (slot * blocks16(p.dv) + w.col / 16) * kChunk * 16);
      __syncwarp();
    }
  }
}

// Chunks backwards, the state's warp: dN = (P^T dO) + diag(e^{c_64 - c}) K dS,
// dY = T^T dN, dV = beta dY, dS <- e^{c_64} dS - K^T diag(e^c beta) dY + (Q^T
// diag(scale e^c) dO), all transposed; the terms in brackets are the companion's.
template <int DK>
__device__ __forceinline__ void rev_state(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                          int hv, const Place& w, const SeqSmem<DK>& sm,
                                          SeqBars& bars) {
  const int lane = threadIdx.x & 31, tig = lane & 3;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const int64_t head = static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
  const float4* s_share = reinterpret_cast<const float4*>(w.share);
  const float4* n_share = reinterpret_cast<const float4*>(w.share + state_share<DK>());
  const uint32_t staging = smem_u32(w.staging);
  float S[DK / 8][4] = {};
  if (a.state0) move_state<DK, false>(S, a.state0 + head * p.dk * p.dv, p.dk, p.dv, w.col);
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, at = chunks - 1 - n;
    const int64_t slot = static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
    if (!mbar_wait_warp(&bars.full_a[st], (n / kStages) & 1, a.err, &bars.abort)) return;
    const uint32_t K = smem_u32(sm.a(st));
    const Block* blk = reinterpret_cast<const Block*>(sm.a(st) + tile_bytes<DK>());
    const uint32_t T = smem_u32(blk->t_hi);

    float N[8][4] = {};
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
      uint32_t hi[4], lo[4];
      left(S[2 * ks], S[2 * ks + 1], hi, lo);
      times_rows<DK>(N, hi, lo, K, ks);
      stage_state<DK>(hi, ks, staging);
    }
    put_state<DK>(w.staging, a.states + (slot * blocks16(p.dv) + w.col / 16) * 16 * DK);
    if (!mbar_wait_warp(&bars.n_full[w.pair], n & 1, a.err, &bars.abort)) return;
    uint32_t yh[4][4], yl[4][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 g = *reinterpret_cast<const float2*>(blk->left + 8 * j + 2 * tig);
      const float4 x = n_share[j * 32 + lane];
      N[j][0] = fmaf(g.x, N[j][0], x.x);
      N[j][1] = fmaf(g.y, N[j][1], x.y);
      N[j][2] = fmaf(g.x, N[j][2], x.z);
      N[j][3] = fmaf(g.y, N[j][3], x.w);
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) left(N[2 * ks], N[2 * ks + 1], yh[ks], yl[ks]);
    float Y[8][4] = {};
    times_triangle<true, true>(Y, yh, yl, T);
    stage_rows(Y, staging);
    put_block(w.staging, a.rows + (slot * blocks16(p.dv) + w.col / 16) * kChunk * 16);
    const float whole = blk->grown[kChunk - 1];
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
      const float4 x = s_share[j * 32 + lane];
      S[j][0] = fmaf(whole, S[j][0], x.x);
      S[j][1] = fmaf(whole, S[j][1], x.y);
      S[j][2] = fmaf(whole, S[j][2], x.z);
      S[j][3] = fmaf(whole, S[j][3], x.w);
    }
    signal(&bars.n_free[w.pair]);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      float x[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 16 * ks + 8 * e + 2 * tig;
        const float2 g = *reinterpret_cast<const float2*>(blk->grown + t);
        const float2 b = *reinterpret_cast<const float2*>(blk->beta + t);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          Y[2 * ks + e][f] *= f & 1 ? b.y : b.x;  // dV from here on
          x[e][f] = -(f & 1 ? g.y : g.x) * Y[2 * ks + e][f];
        }
      }
      uint32_t hi[4], lo[4];
      left(x[0], x[1], hi, lo);
      add_outer<DK>(S, hi, lo, K, ks);
    }
    signal(&bars.empty_a[st]);
    stage_rows(Y, staging);
    put_rows(w.staging,
             static_cast<bf16*>(a.out) +
                 ((static_cast<int64_t>(s.b) * p.T + s.begin + at * kChunk) * p.Hv + hv) * p.dv +
                 w.col,
             static_cast<int64_t>(p.Hv) * p.dv, min(kChunk, s.len - at * kChunk), w.col, p.dv);
    __syncwarp();
  }
  if (a.state1) move_state<DK, true>(S, a.state1 + head * p.dk * p.dv, p.dk, p.dv, w.col);
}

// ... and its companion, a chunk ahead: P^T dO and Q^T diag(scale e^c) dO.
template <int DK>
__device__ __forceinline__ void rev_input(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                          const Place& w, const SeqSmem<DK>& sm, SeqBars& bars) {
  const int lane = threadIdx.x & 31, tig = lane & 3;
  const int chunks = (s.len + kChunk - 1) / kChunk;
  float4* s_share = reinterpret_cast<float4*>(w.share);
  float4* n_share = reinterpret_cast<float4*>(w.share + state_share<DK>());
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages;
    if (!mbar_wait_warp(&bars.full_b[st], (n / kStages) & 1, a.err, &bars.abort)) return;
    const uint32_t Q = smem_u32(sm.b(st)), P = Q + tile_bytes<DK>();
    const float* grown = reinterpret_cast<const float*>(sm.b(st) + tile_bytes<DK>() + 2 * kTile);
    const uint32_t D = smem_u32(sm.v(st, w.pair));
    uint32_t d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) load_v(d[j], D, 16 * j);
    float N[8][4] = {}, Z[DK / 8][4] = {};
    times_triangle<true, false>(N, d, d, P);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      float z[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 g = *reinterpret_cast<const float2*>(grown + 16 * ks + 8 * e + 2 * tig);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const uint32_t r = d[ks][2 * e + (f >> 1)];
          z[e][f] = p.scale * (f & 1 ? g.y : g.x) * (f & 1 ? hi_of(r) : lo_of(r));
        }
      }
      uint32_t hi[4], lo[4];
      left(z[0], z[1], hi, lo);
      add_outer<DK>(Z, hi, lo, Q, ks);
    }
    signal(&bars.empty_b[st]);
    if (!mbar_wait_warp(&bars.n_free[w.pair], (n & 1) ^ 1, a.err, &bars.abort)) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      n_share[j * 32 + lane] = make_float4(N[j][0], N[j][1], N[j][2], N[j][3]);
#pragma unroll
    for (int j = 0; j < DK / 8; ++j)
      s_share[j * 32 + lane] = make_float4(Z[j][0], Z[j][1], Z[j][2], Z[j][3]);
    signal(&bars.n_full[w.pair]);
  }
}

// Block (sequence, value head, 16 W columns).
template <int DK, bool REV, int W>
__global__ void __launch_bounds__(32 * (2 * W + 1), 1)
    seq_kernel(const gsa_delta_t p, const __grid_constant__ DeltaMaps maps, const SeqArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const SeqSmem<DK> sm = {
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull),
      W};
  __shared__ SeqBars bars;
  const int hv = blockIdx.y, col0 = blockIdx.z * 16 * W, warp = threadIdx.x >> 5;
  const Seq s = sequence(p, a.table, blockIdx.x);
  if (s.gap) {  // rows of no sequence: zeros
    const int pieces = min(2 * W, (p.dv - col0) / 8);
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(s.len) * pieces; i += blockDim.x)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) +
                                ((s.begin + i / pieces) * p.Hv + hv) * p.dv + col0 +
                                i % pieces * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x == 0) {
    bars.abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full_a[i], 33);  // 32 copying lanes, and the bulk copies' announcement
      mbar_init(&bars.full_b[i], 33);
      mbar_init(&bars.empty_a[i], W);
      mbar_init(&bars.empty_b[i], W);
    }
    for (int i = 0; i < W; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.s_free[i], 1);
      mbar_init(&bars.n_full[i], 1);
      mbar_init(&bars.n_free[i], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == 2 * W) {
    produce<DK, REV>(p, maps, a, s, hv, col0, W, sm, bars);
    return;
  }
  const bool second = warp >= W;
  const int pair = second ? warp - W : warp;
  const Place w = {pair, col0 + 16 * pair, sm.pair(pair), sm.pair(pair) + pair_bytes<DK>()};
  if (w.col >= p.dv) {  // columns of no one: keep the stages moving
    const int chunks = (s.len + kChunk - 1) / kChunk;
    for (int n = 0; n < chunks; ++n) {
      if (!mbar_wait_warp(second ? &bars.full_b[n % kStages] : &bars.full_a[n % kStages],
                          (n / kStages) & 1, a.err, &bars.abort))
        return;
      signal(second ? &bars.empty_b[n % kStages] : &bars.empty_a[n % kStages]);
    }
    return;
  }
  if constexpr (REV) {
    if (second)
      rev_input<DK>(p, a, s, w, sm, bars);
    else
      rev_state<DK>(p, a, s, hv, w, sm, bars);
  } else {
    if (second)
      chain_output<DK>(p, a, s, hv, w, sm, bars);
    else
      chain_state<DK>(p, a, s, hv, w, sm, bars);
  }
}

// ---------------------------------------------------------------- grad
constexpr int kGradThreads = 512;

struct GradArgs {
  Table table;
  const Block* blocks;
  const bf16* news;     // N
  const bf16* states;   // S0
  const bf16* back;     // dY
  const bf16* dstates;  // dS1
  const void* dout;     // may be nullptr
  void *dq, *dk, *dv, *dg, *dbeta;
};

// Shared memory: K, Q; two stages of S0, dS1 [64 columns][DK], dO, N, dY
// [64][64 columns]; A and G; sums.
template <int DK>
__host__ __device__ constexpr int grad_stage() { return 2 * (DK / 64) * static_cast<int>(kTile) + 3 * static_cast<int>(kTile); }
template <int DK>
constexpr int grad_smem() {
  return 2 * (DK / 64) * static_cast<int>(kTile) + 2 * grad_stage<DK>() + 2 * static_cast<int>(kTile) + 1024;
}

// 16 warps: rows 16 (warp & 3) of the chunk, a quarter (warp >> 2) of the columns.
// With A = scale tril(dO N^T) D, M = strict(-dY N^T) beta D, G = M + M^T:
//   dQ = scale e^c dO S0^T + A K,
//   dK = -e^c beta dY S0^T + e^{c_64 - c} N dS1^T + A^T Q + G K,
//   dbeta, dg: as in delta_simt.cu.
template <int DK>
__global__ void __launch_bounds__(kGradThreads, 1) grad_kernel(const gsa_delta_t p,
                                                               const GradArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull);
  __shared__ Decays d;
  __shared__ float rows4[4][5][kChunk];  // by quarter: q.tO, k.tY, k.tN, rows of E, sum L'
  __shared__ float cols4[4][kChunk];     // by row tile: columns of E
  __shared__ float yv[kChunk], red[16], rowsum[kChunk], grow[kChunk];
  constexpr int NJ = DK / 32;  // n-tiles of a quarter of the channels
  const int hk = blockIdx.y, group = p.Hv / p.Hk, tid = threadIdx.x, lane = tid & 31;
  const int warp = tid >> 5, m0 = (warp & 3) * 16, quarter = warp >> 2;
  const int gid = lane >> 2, tig = lane & 3;
  const Chunk c = chunk_at(p, a.table, blockIdx.x);
  if (!c.valid) return;
  const bool gate16 = p.gate_dtype == GSA_DTYPE_BF16;
  const int64_t row0 = static_cast<int64_t>(c.b) * p.T + c.begin;
  bf16* dq_out = static_cast<bf16*>(a.dq) + (row0 * p.Hk + hk) * p.dk;
  bf16* dk_out = static_cast<bf16*>(a.dk) + (row0 * p.Hk + hk) * p.dk;
  const int64_t qk_step = static_cast<int64_t>(p.Hk) * p.dk;
  if (c.gap) {
    for (int i = tid; i < c.len * p.dk / 8; i += kGradThreads) {
      const int r = i / (p.dk / 8), cc = i % (p.dk / 8) * 8;
      *reinterpret_cast<uint4*>(dq_out + r * qk_step + cc) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(dk_out + r * qk_step + cc) = make_uint4(0, 0, 0, 0);
    }
    const int wide = group * p.dv / 8;
    for (int i = tid; i < c.len * wide; i += kGradThreads)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(a.dv) +
                                ((row0 + i / wide) * p.Hv + hk * group) * p.dv + i % wide * 8) =
          make_uint4(0, 0, 0, 0);
    for (int i = tid; i < c.len * group; i += kGradThreads) {
      const int64_t at = (row0 + i / group) * p.Hv + hk * group + i % group;
      store_gate(a.dg, at, gate16, 0.f);
      store_gate(a.dbeta, at, gate16, 0.f);
    }
    return;
  }
  const uint32_t K = smem_u32(smem), Q = K + tile_bytes<DK>();
  const uint32_t stages = Q + tile_bytes<DK>();
  const uint32_t A = stages + 2 * grad_stage<DK>(), G = A + kTile;
  unsigned char* smemA = smem + 2 * tile_bytes<DK>() + 2 * grad_stage<DK>();
  unsigned char* smemG = smemA + kTile;
  const int nb = blocks16(p.dv), parts = (nb + 3) / 4;  // 64 columns at a time

  auto fetch = [&](int it) {  // part it % parts of the group's head it / parts
    const int hv = hk * group + it / parts, b0 = it % parts * 4;
    const uint32_t S0 = stages + (it & 1) * grad_stage<DK>();
    const uint32_t S1 = S0 + tile_bytes<DK>(), D = S1 + tile_bytes<DK>();
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
    const bf16* s0 = a.states + slot * nb * 16 * DK;
    const bf16* s1 = a.dstates + slot * nb * 16 * DK;
    for (int i = tid; i < 64 * (DK / 8); i += kGradThreads) {
      const int r = i / (DK / 8), cc = i % (DK / 8);
      const bool real = b0 + r / 16 < nb;
      const int64_t at = real ? static_cast<int64_t>(b0 * 16 + r) * DK + cc * 8 : 0;
      const uint32_t to = (cc >> 3) * kTile + sw128_offset(r, cc & 7);
      cp16(S0 + to, s0 + at, real);
      cp16(S1 + to, s1 + at, real);
    }
    const bf16* news = a.news + slot * nb * kChunk * 16;
    const bf16* back = a.back + slot * nb * kChunk * 16;
    const bf16* dout = static_cast<const bf16*>(a.dout) +
                       (a.dout ? (row0 * p.Hv + hv) * p.dv : 0);
    {
      static_assert(kGradThreads == 512, "one piece a thread");
      const int b = tid >> 7, r = (tid >> 1) & 63, h = tid & 1;
      const bool real = b0 + b < nb;
      const int64_t at = real ? (static_cast<int64_t>(b0 + b) * kChunk + r) * 16 + h * 8 : 0;
      const uint32_t to = sw128_offset(r, 2 * b + h);
      cp16(D + kTile + to, news + at, real);
      cp16(D + 2 * kTile + to, back + at, real);
      const int r2 = tid >> 3, c2 = tid & 7, col = b0 * 16 + c2 * 8;
      const bool in = a.dout && r2 < c.len && col < p.dv;
      cp16(D + sw128_offset(r2, c2),
           in ? dout + static_cast<int64_t>(r2) * p.Hv * p.dv + col : news, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  copy_rows(K, rows_at(p.k, p.k_stride, c.b, c.begin, hk), p.k_stride[1], c.len, DK, p.dk, tid,
            kGradThreads);
  copy_rows(Q, rows_at(p.q, p.q_stride, c.b, c.begin, hk), p.q_stride[1], c.len, DK, p.dk, tid,
            kGradThreads);
  const int its = group * parts;
  fetch(0);
  float gq[NJ][4] = {}, gk[NJ][4] = {};
  int it = 0;
  for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
    float to[NJ][4] = {}, ty[NJ][4] = {}, tn[NJ][4] = {}, dp[2][4] = {}, dl[2][4] = {};
    float cross = 0.f, dot = 0.f;
    for (int part = 0; part < parts; ++part, ++it) {
      if (it + 1 < its) {
        fetch(it + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      if (part == 0 && warp == 0) chunk_decays(p, c, hv, d);
      __syncthreads();
      const uint32_t S0 = stages + (it & 1) * grad_stage<DK>();
      const uint32_t S1 = S0 + tile_bytes<DK>(), D = S1 + tile_bytes<DK>();
      const uint32_t N = D + kTile, Y = N + kTile;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t da[4], ya[4], na[4], b[4];
        ldsm(da, at_mk(D, m0, 2 * ks));
        ldsm(ya, at_mk(Y, m0, 2 * ks));
        ldsm(na, at_mk(N, m0, 2 * ks));
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
          ldsm_t(b, at_kn(S0, 16 * ks, quarter * NJ + j));
          mma(to[j], da, b[0], b[1]);
          mma(to[j + 1], da, b[2], b[3]);
          mma(ty[j], ya, b[0], b[1]);
          mma(ty[j + 1], ya, b[2], b[3]);
          ldsm_t(b, at_kn(S1, 16 * ks, quarter * NJ + j));
          mma(tn[j], na, b[0], b[1]);
          mma(tn[j + 1], na, b[2], b[3]);
        }
        ldsm(b, at_nk(N, 16 * quarter, 2 * ks));
        mma(dp[0], da, b[0], b[1]);
        mma(dp[1], da, b[2], b[3]);
        mma(dl[0], ya, b[0], b[1]);
        mma(dl[1], ya, b[2], b[3]);
      }
      // <S0, dS1> and dY_i . V_i, element by element
      const unsigned char* s0 = smem + 2 * tile_bytes<DK>() + (it & 1) * grad_stage<DK>();
      for (int i = tid; i < tile_bytes<DK>() / 16; i += kGradThreads) {
        const uint4 x = reinterpret_cast<const uint4*>(s0)[i];
        const uint4 y = reinterpret_cast<const uint4*>(s0 + tile_bytes<DK>())[i];
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cross = fmaf(lo_of(xs[e]), lo_of(ys[e]), cross);
          cross = fmaf(hi_of(xs[e]), hi_of(ys[e]), cross);
        }
      }
      {
        const int r = tid >> 3, col = part * 64 + (tid & 7) * 8;
        if (r < c.len && col < p.dv) {
          const uint4 x = *reinterpret_cast<const uint4*>(
              s0 + 2 * tile_bytes<DK>() + 2 * kTile + sw128_offset(r, tid & 7));
          const uint4 y = *reinterpret_cast<const uint4*>(
              rows_at(p.v, p.v_stride, c.b, c.begin + r, hv) + col);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dot = fmaf(lo_of(xs[e]), lo_of(ys[e]), dot);
            dot = fmaf(hi_of(xs[e]), hi_of(ys[e]), dot);
          }
        }
      }
      __syncthreads();  // the stage is free
    }
    // per row: 8 neighbouring lanes hold dY_i . V_i; <S0, dS1> over the block
#pragma unroll
    for (int m = 4; m; m >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, m);
    if ((lane & 7) == 0) yv[tid >> 3] = dot;
#pragma unroll
    for (int m = 16; m; m >>= 1) cross += __shfl_xor_sync(0xFFFFFFFFu, cross, m);
    if (lane == 0) red[warp] = cross;

    float kk[2][4] = {}, qk[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
      uint32_t ka[4], qa[4], b[4];
      ldsm(ka, at_mk(K, m0, 2 * ks));
      ldsm(qa, at_mk(Q, m0, 2 * ks));
      ldsm(b, at_nk(K, 16 * quarter, 2 * ks));
      mma(kk[0], ka, b[0], b[1]);
      mma(kk[1], ka, b[2], b[3]);
      mma(qk[0], qa, b[0], b[1]);
      mma(qk[1], qa, b[2], b[3]);
    }
    float er[2] = {}, eb[2] = {}, ec[2][2] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = m0 + gid + 8 * e, cc = 16 * quarter + 8 * j + 2 * tig;
        float x[2], g[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const float w = r >= cc + f ? decay_between(d, r, cc + f) : 0.f;
          x[f] = r >= cc + f ? p.scale * dp[j][2 * e + f] * w : 0.f;
          const float l = r > cc + f ? -dl[j][2 * e + f] * w : 0.f;
          g[f] = l * d.beta[r];
          const float ev = fmaf(x[f], qk[j][2 * e + f], g[f] * kk[j][2 * e + f]);
          er[e] += ev;
          ec[j][f] += ev;
          eb[e] = fmaf(l, kk[j][2 * e + f], eb[e]);
        }
        const uint32_t at = sw128_offset(r, cc >> 3) + 4 * tig;
        *reinterpret_cast<uint32_t*>(smemA + at) = pack_bf16x2(x[0], x[1]);
        // G = M + M^T: the lower triangle and its mirror; the diagonal is zero
#pragma unroll
        for (int f = 0; f < 2; ++f)
          if (r >= cc + f) {
            const bf16 v = __float2bfloat16_rn(g[f]);
            *reinterpret_cast<bf16*>(smemG + sw128_offset(r, (cc + f) >> 3) + 2 * ((cc + f) & 7)) = v;
            if (r > cc + f)
              *reinterpret_cast<bf16*>(smemG + sw128_offset(cc + f, r >> 3) + 2 * (r & 7)) = v;
          }
      }
    // column sums of E over the 8 rows a lane's neighbours hold
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
#pragma unroll
        for (int m = 4; m <= 16; m <<= 1) ec[j][f] += __shfl_xor_sync(0xFFFFFFFFu, ec[j][f], m);
        if (gid == 0) cols4[warp & 3][16 * quarter + 8 * j + 2 * tig + f] = ec[j][f];
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = m0 + gid + 8 * e;
      const float g = decay_from_start(d, r), lf = decay_between(d, kChunk - 1, r);
      const float gb = g * d.beta[r], sg = p.scale * g;
      float v[5] = {0.f, 0.f, 0.f, er[e], eb[e]};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int cc = quarter * NJ + j;  // piece of the row
        const uint32_t at = (cc >> 3) * kTile + sw128_offset(r, cc & 7) + 4 * tig;
        const uint32_t kv = *reinterpret_cast<const uint32_t*>(smem + at);
        const uint32_t qv = *reinterpret_cast<const uint32_t*>(smem + tile_bytes<DK>() + at);
        v[0] = fmaf(lo_of(qv), to[j][2 * e], fmaf(hi_of(qv), to[j][2 * e + 1], v[0]));
        v[1] = fmaf(lo_of(kv), ty[j][2 * e], fmaf(hi_of(kv), ty[j][2 * e + 1], v[1]));
        v[2] = fmaf(lo_of(kv), tn[j][2 * e], fmaf(hi_of(kv), tn[j][2 * e + 1], v[2]));
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          gq[j][2 * e + f] = fmaf(sg, to[j][2 * e + f], gq[j][2 * e + f]);
          gk[j][2 * e + f] += lf * tn[j][2 * e + f] - gb * ty[j][2 * e + f];
        }
      }
#pragma unroll
      for (int x = 0; x < 5; ++x) {
        v[x] += __shfl_xor_sync(0xFFFFFFFFu, v[x], 1);
        v[x] += __shfl_xor_sync(0xFFFFFFFFu, v[x], 2);
        if (tig == 0) rows4[quarter][x][r] = v[x];
      }
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {  // 16 tokens of the contraction
      uint32_t x[4], y[4], b[4];
      ldsm(x, at_mk(A, m0, 2 * ks));      // A rows
      ldsm(y, at_mk(G, m0, 2 * ks));      // G rows (symmetric)
      uint32_t z[4];
      ldsm_t(z, at_km(A, 16 * ks, m0 / 8));  // A columns
#pragma unroll
      for (int j = 0; j < NJ; j += 2) {
        ldsm_t(b, at_kn(K, 16 * ks, quarter * NJ + j));
        mma(gq[j], x, b[0], b[1]);
        mma(gq[j + 1], x, b[2], b[3]);
        mma(gk[j], y, b[0], b[1]);
        mma(gk[j + 1], y, b[2], b[3]);
        ldsm_t(b, at_kn(Q, 16 * ks, quarter * NJ + j));
        mma(gk[j], z, b[0], b[1]);
        mma(gk[j + 1], z, b[2], b[3]);
      }
    }
    if (tid < kChunk) {
      const int r = tid;
      float v[5];
#pragma unroll
      for (int x = 0; x < 5; ++x)
        v[x] = (rows4[0][x][r] + rows4[1][x][r]) + (rows4[2][x][r] + rows4[3][x][r]);
      const float ec_r = (cols4[0][r] + cols4[1][r]) + (cols4[2][r] + cols4[3][r]);
      const float g = decay_from_start(d, r);
      rowsum[r] = p.scale * g * v[0] - g * d.beta[r] * v[1] + v[3] - ec_r;
      grow[r] = decay_between(d, kChunk - 1, r) * v[2];
      if (r < c.len)
        store_gate(a.dbeta, (row0 + r) * p.Hv + hv, gate16, yv[r] - g * v[1] + v[4]);
    }
    __syncthreads();
    if (warp == 0) {
      // suffix sums of rowsum plus prefix sums of grow, two rows a lane
      float rs[2] = {rowsum[2 * lane], rowsum[2 * lane + 1]};
      float gs[2] = {grow[2 * lane], grow[2 * lane + 1]};
      float suffix = rs[0] + rs[1], prefix = gs[0] + gs[1];
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const float o = __shfl_down_sync(0xFFFFFFFFu, suffix, m);
        if (lane + m < 32) suffix += o;
        const float q = __shfl_up_sync(0xFFFFFFFFu, prefix, m);
        if (lane >= m) prefix += q;
      }
      float after = __shfl_down_sync(0xFFFFFFFFu, suffix, 1);
      float before = __shfl_up_sync(0xFFFFFFFFu, prefix, 1);
      if (lane == 31) after = 0.f;
      if (lane == 0) before = 0.f;
      float whole = lane < 16 ? red[lane] : 0.f;
#pragma unroll
      for (int m = 16; m; m >>= 1) whole += __shfl_xor_sync(0xFFFFFFFFu, whole, m);
      whole *= decay_from_start(d, kChunk - 1);
      const float dg0 = whole + before + (rs[0] + (rs[1] + after));
      const float dg1 = whole + (before + gs[0]) + (rs[1] + after);
      if (2 * lane < c.len) store_gate(a.dg, (row0 + 2 * lane) * p.Hv + hv, gate16, dg0);
      if (2 * lane + 1 < c.len) store_gate(a.dg, (row0 + 2 * lane + 1) * p.Hv + hv, gate16, dg1);
    }
    __syncthreads();  // d, A, G and the sums are the next head's
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = m0 + gid + 8 * e, cc = (quarter * NJ + j) * 8 + 2 * tig;
      if (r < c.len && cc < p.dk) {
        *reinterpret_cast<uint32_t*>(dq_out + r * qk_step + cc) =
            pack_bf16x2(gq[j][2 * e], gq[j][2 * e + 1]);
        *reinterpret_cast<uint32_t*>(dk_out + r * qk_step + cc) =
            pack_bf16x2(gk[j][2 * e], gk[j][2 * e + 1]);
      }
    }
}

// ---------------------------------------------------------------- launches
// Pairs of a block of chain / rev: as many as share the copies of K and Q while
// the blocks still cover the SMs.  Four pairs and the copying warp leave each
// thread 168 registers, which the state's warp needs.
int pairs_of(const gsa_delta_t& p) {
  const int64_t all = static_cast<int64_t>(p.N) * p.Hv * blocks16(p.dv);
  int w = 1;
  while (w < 4 && all / (2 * w) >= 128 && w < blocks16(p.dv)) w *= 2;
  return w;
}

template <int DK, bool REV, int W>
cudaError_t launch_seq_w(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a,
                         cudaStream_t stream) {
  cudaError_t e = allow_smem<seq_kernel<DK, REV, W>>(seq_smem<DK>(W));
  if (e != cudaSuccess) return e;
  const int seqs = p.N + (!REV && p.cu_seqlens ? 2 : 0);
  seq_kernel<DK, REV, W><<<dim3(seqs, p.Hv, (p.dv + 16 * W - 1) / (16 * W)), 32 * (2 * W + 1),
                           seq_smem<DK>(W), stream>>>(p, m, a);
  return cudaGetLastError();
}
template <int DK, bool REV>
cudaError_t launch_seq(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a,
                       cudaStream_t stream) {
  switch (pairs_of(p)) {
    case 1: return launch_seq_w<DK, REV, 1>(p, m, a, stream);
    case 2: return launch_seq_w<DK, REV, 2>(p, m, a, stream);
    default: return launch_seq_w<DK, REV, 4>(p, m, a, stream);
  }
}

template <int DK>
cudaError_t forward(const gsa_delta_t& p, const DeltaMaps& m, void* o, float* final_state, bool save, void* ws,
                    int* err, cudaStream_t stream) {
  const Saved s = saved_at(p, ws);
  const Table t = table_at(ws, p.N);
  const int64_t chunks = max_chunks(p);
  cudaError_t e = allow_smem<prep_kernel<DK>>(prep_smem<DK>());
  if (e != cudaSuccess) return e;
  if (chunks > 0)
    prep_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hk), kPrepThreads, prep_smem<DK>(),
                      stream>>>(p, t, s.blocks);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const SeqArgs a = {t,           s.blocks,  nullptr, o, p.initial_state,
                     final_state, save ? s.news : nullptr, save ? s.states : nullptr, err};
  return launch_seq<DK, false>(p, m, a, stream);
}

template <int DK>
cudaError_t backward(const gsa_delta_t& p, const DeltaMaps& m, const DeltaGrads& g, void* saved,
                     void* scratch, int* err, cudaStream_t stream) {
  const Saved s = saved_at(p, saved);
  const Scratch r = scratch_at(p, scratch);
  const Table t = table_at(saved, p.N);
  const SeqArgs a = {t, s.blocks, g.dout, g.dv, g.dfinal, g.dinitial, r.back, r.states, err};
  cudaError_t e = launch_seq<DK, true>(p, m, a, stream);
  if (e != cudaSuccess) return e;
  if ((e = allow_smem<grad_kernel<DK>>(grad_smem<DK>())) != cudaSuccess) return e;
  const GradArgs ga = {t,      s.blocks, s.news, s.states, r.back, r.states,
                       g.dout, g.dq,     g.dk,   g.dv,     g.dg,   g.dbeta};
  const int64_t chunks = max_chunks(p);
  if (chunks > 0)
    grad_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hk), kGradThreads, grad_smem<DK>(),
                      stream>>>(p, ga);
  return cudaGetLastError();
}

}  // namespace

int64_t mma_saved_bytes(const gsa_delta_t& p, bool save) {
  const int64_t n = max_chunks(p) * p.Hv;
  return table_bytes(p) + n * (static_cast<int64_t>(sizeof(Block)) +
                               (save ? news_bytes(p) + state_bytes(p) : 0));
}
int64_t mma_scratch_bytes(const gsa_delta_t& p) {
  return max_chunks(p) * p.Hv * (news_bytes(p) + state_bytes(p));
}
cudaError_t mma_forward(const gsa_delta_t& p, const DeltaMaps& m, void* o, float* final_state,
                        bool save, void* ws, int* err, cudaStream_t stream) {
  return p.dk <= 64 ? forward<64>(p, m, o, final_state, save, ws, err, stream)
                    : forward<128>(p, m, o, final_state, save, ws, err, stream);
}
cudaError_t mma_backward(const gsa_delta_t& p, const DeltaMaps& m, const DeltaGrads& g, void* saved,
                         void* scratch, int* err, cudaStream_t stream) {
  return p.dk <= 64 ? backward<64>(p, m, g, saved, scratch, err, stream)
                    : backward<128>(p, m, g, saved, scratch, err, stream);
}

}  // namespace delta
}  // namespace gsa
