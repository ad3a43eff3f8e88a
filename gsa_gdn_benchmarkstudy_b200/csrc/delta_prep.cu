// delta_prep.cu — the gated delta rule for bf16 inputs: what a chunk needs apart
// from any state, T = (I + L)^-1 and P (formulas: delta_common.cuh), for all chunks
// at once, and the launches of the forward and backward pass.
//
// One block a chunk and key head makes T and P of the value heads that share the
// key head.  [K; Q] K^T is one tcgen05 product of 128 x 64 x dk: tensor memory
// keeps it for all of them, a thread reads its row of KK^T or QK^T from there.
// T and P leave as hi + lo pairs of bf16, laid out as the shared-memory tiles that
// the sequential pass copies whole, so bulk copies store them.  Bound by latency:
// loads, the product, a triangular inverse and 34 KB of stores one after the
// other; six blocks an SM overlap theirs.  256 chunks of 16 heads of 128 channels take
// 65 us (42 for the bytes); products by mma.sync, copies and stores by the threads, four
// blocks an SM: 94.
#include "delta_tc.cuh"

namespace gsa {
namespace delta {
namespace {

// ---------------------------------------------------------------- prep
constexpr int kPrepThreads = 128;

// Shared memory: K and Q (64 columns of K, of Q, the next 64 of K, of Q); once they
// are multiplied, the gates, P's tiles and L, which becomes T in place, in fp32; the
// inner products of its inverse lie in L's upper right quarter.  T's tiles take the
// place of the gates and P.  Six blocks fit into an SM.
constexpr int kOffPTiles = sizeof(Gates), kOffL = kOffPTiles + kPBytes;
constexpr int kPrepUsed = kOffL + kChunk * kLdL * 4;
constexpr int kPrepSmem = kPrepUsed + 1024;
static_assert(kPrepUsed >= 4 * static_cast<int>(kTile), "K and Q");

struct PrepBars {
  uint64_t full, product;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void bulk_store(void* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                   reinterpret_cast<uint64_t>(dst)),
               "r"(smem_u32(smem_src)), "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until the stores of this thread have read shared memory, or have arrived.
__device__ __forceinline__ void bulk_stores_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_stores_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// 8 values as hi + lo in piece `at` of a pair of tiles.
__device__ __forceinline__ void put_pairs(unsigned char* tiles, uint32_t at, const float (&x)[8]) {
  uint4 hi, lo;
  split(x[0], x[1], hi.x, lo.x);
  split(x[2], x[3], hi.y, lo.y);
  split(x[4], x[5], hi.z, lo.z);
  split(x[6], x[7], hi.w, lo.w);
  *reinterpret_cast<uint4*>(tiles + at) = hi;
  *reinterpret_cast<uint4*>(tiles + kTile + at) = lo;
}

// Row `r` of L (of P with `is_p`), 32 columns from tensor memory at a time.
__device__ __forceinline__ void make_row(const Decays& d, uint32_t tmem, int r, bool is_p,
                                         float factor, float* L, unsigned char* P) {
  const uint64_t hi_r = f2_pack(d.hi[r], d.hi[r]), lo_r = f2_pack(d.lo[r], d.lo[r]);
  const uint64_t less = f2_pack(-1.f, -1.f), scale = f2_pack(factor, factor);
  const uint64_t log2e = f2_pack(kLog2e, kLog2e);
  const int half = r >> 5;
  for (int h = 0; h <= half; ++h) {
    uint32_t raw[32];
    tmem_ld32(tmem + 32 * h, raw);
    tc_wait_ld(raw);
    // the diagonal is in the last 32 columns: what lies behind it is dropped
    const int limit = r - 32 * h + (is_p ? 1 : 0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int c = 8 * g + i;
        const uint64_t hi_c = *reinterpret_cast<const uint64_t*>(d.hi + 32 * h + c);
        const uint64_t lo_c = *reinterpret_cast<const uint64_t*>(d.lo + 32 * h + c);
        const uint64_t e =
            f2_mul(f2_add(f2_fma(hi_c, less, hi_r), f2_fma(lo_c, less, lo_r)), log2e);
        const uint64_t w = f2_pack(fast_ex2(f2_lo(e)), fast_ex2(f2_hi(e)));
        const uint64_t y = f2_mul(
            f2_mul(w, scale), f2_pack(__uint_as_float(raw[c]), __uint_as_float(raw[c + 1])));
        x[i] = c < limit ? f2_lo(y) : 0.f;
        x[i + 1] = c + 1 < limit ? f2_hi(y) : 0.f;
      }
      if (is_p) {
        put_pairs(P, sw128_offset(r, 4 * h + g), x);
      } else {
        float4* to = reinterpret_cast<float4*>(L + r * kLdL + 32 * h + 8 * g);
        to[0] = make_float4(x[0], x[1], x[2], x[3]);
        to[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  }
  if (half == 0 && is_p)
#pragma unroll
    for (int g = 4; g < 8; ++g) {
      *reinterpret_cast<uint4*>(P + sw128_offset(r, g)) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(P + kTile + sw128_offset(r, g)) = make_uint4(0, 0, 0, 0);
    }
}

template <int DK>
__global__ void __launch_bounds__(kPrepThreads, 6)
    prep_kernel(const gsa_delta_t p, const __grid_constant__ DeltaMaps maps, Table table,
                Block* blocks, int* err) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull);
  __shared__ Decays d;
  __shared__ PrepBars bars;
  const int hk = blockIdx.y, group = p.Hv / p.Hk, tid = threadIdx.x, lane = tid & 31;
  const int warp = tid >> 5;
  const Chunk c = chunk_at(p, table, blockIdx.x);
  if (!c.valid || c.gap) return;
  // Rows past the tensor's end come out of TMA as zeros; a chunk that ends before its
  // 64th row inside a packed batch takes its rows one by one.
  const bool whole = c.len == kChunk || !p.cu_seqlens;
  if (tid == 0) {
    bars.abort = 0;
    mbar_init(&bars.full, 1);
    mbar_init(&bars.product, 1);
    fence_mbar_init();
    if (whole) {
      mbar_arrive_expect_tx(&bars.full, DK / 64 * 2 * kTile);
      for (int i = 0; i < DK / 64; ++i) {
        tma_load_rows(smem + 2 * i * kTile, &maps.k, 64 * i, hk, c.begin, c.b, &bars.full);
        tma_load_rows(smem + (2 * i + 1) * kTile, &maps.q, 64 * i, hk, c.begin, c.b, &bars.full);
      }
    }
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem, 64);
    tmem_relinquish();
  }
  if (!whole) {
    copy_rows(smem_u32(smem), rows_at(p.k, p.k_stride, c.b, c.begin, hk), p.k_stride[1], c.len, DK,
              p.dk, tid, kPrepThreads, 2 * kTile);
    copy_rows(smem_u32(smem) + kTile, rows_at(p.q, p.q_stride, c.b, c.begin, hk), p.q_stride[1],
              c.len, DK, p.dk, tid, kPrepThreads, 2 * kTile);
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 2) chunk_decays(p, c, hk * group, d);  // beside the copies
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, bars.tmem, 0);
  bool ok = true;
  if (warp == 0) {
    if (whole) ok = mbar_wait_warp(&bars.full, 0, err, &bars.abort);
    if (ok) {
      const uint32_t tile = smem_u32(smem);
#pragma unroll
      for (int ks = 0; ks < DK / 16; ++ks) {
        const uint64_t kq = desc_rows(tile, ks, 2 * kTile);
        warp_mma_ss(tmem, kq, kq, idesc_bf16_f32(128, 64, 0, 0), ks);
      }
      warp_commit(&bars.product);
    }
    // no copy and no product of ours may outlive the block
    if (!ok)
      mbar_wait_drain(&bars.full, 0, kWaitLimitCycles);
    else if (!(ok = mbar_wait_warp(&bars.product, 0, err, &bars.abort)))
      mbar_wait_drain(&bars.product, 0, kWaitLimitCycles);
  }
  ok = ok && mbar_wait_warp(&bars.product, 0, err, &bars.abort);
  if (__syncthreads_and(ok)) {
    tc_fence_after();
    float* L = reinterpret_cast<float*>(smem + kOffL);
    Gates* gates = reinterpret_cast<Gates*>(smem);
    const int row = 32 * (warp & 1) + lane;
    const uint32_t mine = tmem + (static_cast<uint32_t>(32 * warp) << 16);
    constexpr int kStorer = 96;
    for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
      if (hv > hk * group) {
        if (warp == 2) chunk_decays(p, c, hv, d);
        if (tid == kStorer) bulk_stores_read();
        __syncthreads();
      }
      Block* blk = blocks + static_cast<int64_t>(blockIdx.x) * p.Hv + hv;
      make_row(d, mine, row, warp >= 2, warp >= 2 ? p.scale : d.beta[row], L, smem + kOffPTiles);
      if ((warp & 1) == 0) {
        const int i = tid < 32 ? tid : tid - 32;
        const float grown = decay_from_start(d, i);
        gates->grown[i] = grown;
        gates->beta[i] = d.beta[i];
        gates->left[i] = decay_between(d, kChunk - 1, i);
        gates->both[i] = d.beta[i] * grown;
        gates->hi[i] = d.hi[i];
        gates->lo[i] = d.lo[i];
      }
      fence_proxy_async_smem();
      __syncthreads();
      if (tid == kStorer)  // P leaves while T is made
        bulk_store(&blk->gates, smem, static_cast<uint32_t>(sizeof(Gates)) + kPBytes);
      invert(L);
      if (tid == kStorer) bulk_stores_read();
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kChunk * 8 / kPrepThreads; ++i) {
        const int x = tid + i * kPrepThreads, r = x >> 3, piece = x & 7;
        float t[8] = {};
        if (r >= 32 || piece < 4) {
          const float4 u = *reinterpret_cast<const float4*>(L + r * kLdL + piece * 8);
          const float4 v = *reinterpret_cast<const float4*>(L + r * kLdL + piece * 8 + 4);
          t[0] = u.x, t[1] = u.y, t[2] = u.z, t[3] = u.w;
          t[4] = v.x, t[5] = v.y, t[6] = v.z, t[7] = v.w;
        }
        put_pairs(smem, sw128_offset(r, piece), t);
      }
      fence_proxy_async_smem();
      __syncthreads();
      if (tid == kStorer) bulk_store(blk->t_hi, smem, kPBytes);
    }
    if (tid == kStorer) bulk_stores_done();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 64);
  }
}

template <int DK>
cudaError_t launch_prep(const gsa_delta_t& p, const DeltaMaps& m, const Table& t, Block* blocks,
                        int* err, cudaStream_t stream) {
  const int64_t chunks = max_chunks(p);
  if (chunks == 0) return cudaSuccess;
  const cudaError_t e = allow_smem<prep_kernel<DK>>(kPrepSmem);
  if (e != cudaSuccess) return e;
  prep_kernel<DK><<<dim3(static_cast<unsigned>(chunks), p.Hk), kPrepThreads, kPrepSmem, stream>>>(
      p, m, t, blocks, err);
  return cudaGetLastError();
}

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
  const cudaError_t e = p.dk <= 64 ? launch_prep<64>(p, m, t, s.blocks, err, stream)
                                   : launch_prep<128>(p, m, t, s.blocks, err, stream);
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
