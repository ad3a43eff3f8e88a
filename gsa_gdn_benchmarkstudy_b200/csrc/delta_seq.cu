// delta_seq.cu — the sequential pass of the gated delta rule for bf16 inputs,
// forwards (states, outputs) and backwards (the state's gradient), on tcgen05.
//
// A block walks one sequence, value head and up to 128 columns of the state.
// Transposed, every product has 128 rows, one a column of the state:
//   R^T = S^T K^T,  N^T = Y^T T^T,  O^T = scale e^c (S^T Q^T) + N^T P^T,
//   S^T <- e^{c_64} S^T + (e^{c_64 - c} N)^T K,   Y = beta (V - e^c R),
// so a thread owns half of one column: its lane of tensor memory.  S^T itself
// stays in fp32 in registers; between two products the threads read an
// accumulator, do its element-wise part, and store the next left operand back to
// tensor memory, where the product takes it from: no operand made here passes
// through shared memory.  K, Q, V, T and P arrive by TMA, two chunks ahead.
//
// Left operands are pairs hi + lo of bf16 (2^-17 of a value together), q, k, v
// exact in bf16 and T, P pairs, so the state keeps about fp32's accuracy over
// any number of chunks.
//
// Bound by the chain of a chunk's three products and the passes between them,
// not by the tensor pipe nor by memory.
#include "delta_tc.cuh"

namespace gsa {
namespace delta {
namespace {

constexpr int kStages = 2;
constexpr int kComputeWarps = 8;
constexpr int kThreads = 32 * (kComputeWarps + 2);
constexpr int kCols = 128;  // state columns of a block: the lanes of tensor memory
constexpr uint32_t kTmemCols = 512;

// Tensor memory, 32-bit columns.
enum : uint32_t {
  kAcc = 0,      // what a chunk adds to S^T [128][dk]
  kShi = 128,    // S^T as a left operand (two values a column)
  kSlo = 192,
  kR = 256,      // R^T, then N^T (backwards dS^T K^T, then dY^T) [128][64]
  kYhi = 320,    // Y^T, then N^T (backwards dN^T, then -e^c beta dY^T)
  kYlo = 352,
  kDhi = 384,    // (e^{c_64 - c} N)^T (backwards (scale e^c dO)^T)
  kDlo = 416,
  kO = 448,      // O^T (backwards dO^T P)
};

template <int DK>
__host__ __device__ constexpr int tile_bytes() { return (DK / 64) * static_cast<int>(kTile); }
template <int DK>
__host__ __device__ constexpr int queue_bytes() { return tile_bytes<DK>() + kHalf; }
constexpr int kValueBytes = 2 * static_cast<int>(kTile);
template <int DK>
__host__ __device__ constexpr int seq_smem() {
  return kStages * (2 * queue_bytes<DK>() + kValueBytes) + 1024;
}

// Queue a holds K, T and decays, queue b Q, P and decays; the 64 x 128 values (v
// forwards, dO backwards) go with a forwards and with b backwards.
template <int DK>
struct Smem {
  unsigned char* base;
  __device__ unsigned char* a(int st) const { return base + st * queue_bytes<DK>(); }
  __device__ unsigned char* b(int st) const { return base + (kStages + st) * queue_bytes<DK>(); }
  __device__ unsigned char* v(int st) const {
    return base + 2 * kStages * queue_bytes<DK>() + st * kValueBytes;
  }
};

// Every barrier but the queues' completes once a chunk.
struct Bars {
  uint64_t full_a[kStages], empty_a[kStages], full_b[kStages], empty_b[kStages];
  uint64_t s_ready, r_full, y_ready, n_full, d_ready, upd_full;
  uint64_t o1_full, o1_read, o_full;  // backwards o1_full: dO^T P
  uint64_t drain;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ bool wait(uint64_t* bar, int n, const SeqArgs& a, Bars& bars) {
  if (!mbar_wait_warp(bar, n & 1, a.err, &bars.abort)) return false;
  tc_fence_after();
  return true;
}
// All of a warp's tensor-memory accesses so far come before the signal.
__device__ __forceinline__ void signal(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The copies of a sequence's chunks, by one warp.  Rows past the tensor's end
// come out of TMA as zeros; a chunk that ends before its 64th row inside a packed
// batch, where another sequence follows, takes its rows one by one.
template <int DK, bool REV>
__device__ __forceinline__ void produce(const gsa_delta_t& p, const DeltaMaps& maps,
                                        const SeqArgs& a, const Seq& s, int hv, int col0,
                                        const Smem<DK>& sm, Bars& bars) {
  const int lane = threadIdx.x & 31, hk = hv / (p.Hv / p.Hk);
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const bool have = !REV || a.in != nullptr;
  int begun[2] = {0, 0};
  bool ok = true;
  for (int n = 0; ok && n < chunks; ++n) {
    const int st = n % kStages, parity = ((n / kStages) & 1) ^ 1;
    const int at = REV ? chunks - 1 - n : n;
    const int begin = s.begin + at * kChunk, rest = s.len - at * kChunk;
    const int len = rest < kChunk ? rest : kChunk;
    const bool whole = len == kChunk || !p.cu_seqlens;
    const Block* blk = a.blocks + static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint64_t* full = q ? &bars.full_b[st] : &bars.full_a[st];
      ok = ok && mbar_wait_warp(q ? &bars.empty_b[st] : &bars.empty_a[st], parity, a.err,
                                &bars.abort);
      if (!ok) break;
      unsigned char* dst = q ? sm.b(st) : sm.a(st);
      const bool values = (q == 1) == REV;
      const bool tma_values = values && whole && have;
      bool by_hand = false;
      if (!whole) {
        copy_rows(smem_u32(dst),
                  q ? rows_at(p.q, p.q_stride, s.b, begin, hk)
                    : rows_at(p.k, p.k_stride, s.b, begin, hk),
                  q ? p.q_stride[1] : p.k_stride[1], len, DK, p.dk, lane, 32);
        by_hand = true;
      }
      if (values && !tma_values) {
        const int64_t stride = REV ? static_cast<int64_t>(p.Hv) * p.dv : p.v_stride[1];
        const bf16* v = REV ? static_cast<const bf16*>(a.in) +
                                  (have ? (static_cast<int64_t>(s.b) * p.T + begin) * stride +
                                              hv * p.dv
                                        : 0)
                            : rows_at(p.v, p.v_stride, s.b, begin, hv);
        copy_rows(smem_u32(sm.v(st)), have ? v + col0 : static_cast<const bf16*>(p.k), stride,
                  have ? len : 0, kCols, p.dv - col0, lane, 32);
        by_hand = true;
      }
      if (by_hand) {  // the products read through the asynchronous proxy
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(full, kHalf + (whole ? tile_bytes<DK>() : 0) +
                                        (tma_values ? kValueBytes : 0));
        bulk_load(dst + tile_bytes<DK>(), reinterpret_cast<const unsigned char*>(blk) + q * kHalf,
                  kHalf, full);
        if (whole)
          for (int i = 0; i < DK / 64; ++i)
            tma_load_rows(dst + i * kTile, q ? &maps.q : &maps.k, 64 * i, hk, begin, s.b, full);
        if (tma_values)
          for (int i = 0; i < 2; ++i)
            tma_load_rows(sm.v(st) + i * kTile, &maps.v, col0 + 64 * i, hv, begin, s.b, full);
      }
      ++begun[q];
    }
  }
  if (!ok) {  // gave up: no copy of ours may outlive the block
    for (int i = max(0, begun[0] - kStages); i < begun[0]; ++i)
      mbar_wait_drain(&bars.full_a[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
    for (int i = max(0, begun[1] - kStages); i < begun[1]; ++i)
      mbar_wait_drain(&bars.full_b[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
  }
}

// acc (+)= (hi + lo) B over KS steps of 16; COLS: B's rows are contracted.
template <int KS, bool COLS>
__device__ __forceinline__ void times(uint32_t acc, uint32_t hi, uint32_t lo, uint32_t tile,
                                      uint32_t idesc, bool fresh) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      tc_mma_ts(acc, (half ? lo : hi) + 8 * ks, COLS ? desc_cols(tile, ks) : desc_rows(tile, ks),
                idesc, !fresh || half || ks);
}
// acc (+)= (hi + lo) (M_hi + M_lo) without lo M_lo, M a pair of 64 x 64 tiles.
template <bool COLS>
__device__ __forceinline__ void times_pair(uint32_t acc, uint32_t hi, uint32_t lo, uint32_t tile,
                                           uint32_t idesc, bool fresh) {
  times<4, COLS>(acc, hi, lo, tile, idesc, fresh);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks)
    tc_mma_ts(acc, hi + 8 * ks, COLS ? desc_cols(tile + kTile, ks) : desc_rows(tile + kTile, ks),
              idesc, 1);
}

// One thread issues all products.
template <int DK, bool REV>
__device__ __forceinline__ void issue(const SeqArgs& a, int chunks, const Smem<DK>& sm,
                                      Bars& bars) {
  const uint32_t tm = bars.tmem;
  constexpr uint32_t kRows64 = idesc_bf16_f32(128, 64, 0, 0);
  constexpr uint32_t kCols64 = idesc_bf16_f32(128, 64, 0, 1);
  constexpr uint32_t kColsDk = idesc_bf16_f32(128, DK, 0, 1);
  constexpr uint32_t kColsCols = idesc_bf16_f32(128, 64, 1, 1);
  auto until = [&](uint64_t* bar, int parity) {
    if (!mbar_wait(bar, parity & 1, a.err, &bars.abort)) return false;
    tc_fence_after();
    return true;
  };
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages;
    const uint32_t K = smem_u32(sm.a(st)), T = K + tile_bytes<DK>();
    const uint32_t Q = smem_u32(sm.b(st)), P = Q + tile_bytes<DK>();
    if constexpr (REV) {
      if (!until(&bars.full_b[st], turn)) break;
      const uint32_t D = smem_u32(sm.v(st));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        tc_mma_ss(tm + kO, desc_cols(D, i & 3), desc_cols(P + (i >> 2) * kTile, i & 3), kColsCols,
                  i > 0);
      tc_commit(&bars.o1_full);
    }
    if (!until(&bars.full_a[st], turn) || !until(&bars.s_ready, n)) break;
    times<DK / 16, false>(tm + kR, tm + kShi, tm + kSlo, K, kRows64, true);
    tc_commit(&bars.r_full);
    if (!until(&bars.y_ready, n)) break;
    if constexpr (REV) {
      times_pair<true>(tm + kR, tm + kYhi, tm + kYlo, T, kCols64, true);
      tc_commit(&bars.n_full);
      times<4, true>(tm + kAcc, tm + kDhi, tm + kDlo, Q, kColsDk, true);
      tc_commit(&bars.empty_b[st]);
      if (!until(&bars.d_ready, n)) break;
      times<4, true>(tm + kAcc, tm + kYhi, tm + kYlo, K, kColsDk, false);
      tc_commit(&bars.upd_full);
      tc_commit(&bars.empty_a[st]);
    } else {
      times_pair<false>(tm + kR, tm + kYhi, tm + kYlo, T, kRows64, true);
      tc_commit(&bars.n_full);
      if (!until(&bars.full_b[st], turn)) break;
      times<DK / 16, false>(tm + kO, tm + kShi, tm + kSlo, Q, kRows64, true);
      tc_commit(&bars.o1_full);
      if (!until(&bars.d_ready, n)) break;
      times<4, true>(tm + kAcc, tm + kDhi, tm + kDlo, K, kColsDk, true);
      tc_commit(&bars.upd_full);
      tc_commit(&bars.empty_a[st]);
      if (!until(&bars.o1_read, n)) break;
      times_pair<false>(tm + kO, tm + kYhi, tm + kYlo, P, kRows64, false);
      tc_commit(&bars.o_full);
      tc_commit(&bars.empty_b[st]);
    }
  }
  // nothing of ours may be in flight when tensor memory is freed
  tc_commit(&bars.drain);
  mbar_wait_drain(&bars.drain, 0, kWaitLimitCycles);
}

// What a thread is: half `half` of column `col` of the value head.
struct Lane {
  int row;        // lane of tensor memory, 0 .. 127
  int half;       // which half of the channels, and of the tokens
  int col;        // column of the value head
  uint32_t tmem;  // its lane's address
};

// The state's half column, in fp32: from and to [dk, dv].
template <int DK>
__device__ __forceinline__ void load_state(float (&S)[DK / 2], const float* state,
                                           const gsa_delta_t& p, const Lane& l) {
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) {
    const int r = l.half * (DK / 2) + i;
    S[i] = (state && r < p.dk && l.col < p.dv) ? state[static_cast<int64_t>(r) * p.dv + l.col]
                                               : 0.f;
  }
}
template <int DK>
__device__ __forceinline__ void store_state(const float (&S)[DK / 2], float* state,
                                            const gsa_delta_t& p, const Lane& l) {
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) {
    const int r = l.half * (DK / 2) + i;
    if (r < p.dk && l.col < p.dv) state[static_cast<int64_t>(r) * p.dv + l.col] = S[i];
  }
}
// S <- whole S + what the last chunk added.
template <int DK>
__device__ __forceinline__ void add_update(float (&S)[DK / 2], float whole, const Lane& l) {
#pragma unroll
  for (int q = 0; q < DK / 64; ++q) {
    uint32_t r[32];
    tmem_ld32(l.tmem + kAcc + l.half * (DK / 2) + 32 * q, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) S[32 * q + i] = fmaf(whole, S[32 * q + i], __uint_as_float(r[i]));
  }
}
// S as the left operand, and (image != nullptr) its upper half kept in bf16.
template <int DK>
__device__ __forceinline__ void put_operand(const float (&S)[DK / 2], const Lane& l, bf16* image,
                                            int rows) {
#pragma unroll
  for (int q = 0; q < DK / 64; ++q) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) split(S[32 * q + 2 * i], S[32 * q + 2 * i + 1], hi[i], lo[i]);
    tmem_st16(l.tmem + kShi + l.half * (DK / 4) + 16 * q, hi);
    tmem_st16(l.tmem + kSlo + l.half * (DK / 4) + 16 * q, lo);
    if (image && l.col < rows)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(
            image + (static_cast<int64_t>(l.half * (DK / 16) + 4 * q + i) * rows + l.col) * 8) =
            make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
  }
}
// 32 tokens of a left operand (hi at `at`, lo 32 columns behind).
__device__ __forceinline__ void put_tokens(const float (&x)[32], uint32_t at, const Lane& l,
                                           uint32_t (&hi)[16]) {
  uint32_t lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) split(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
  tmem_st16(l.tmem + at + 16 * l.half, hi);
  tmem_st16(l.tmem + at + 32 + 16 * l.half, lo);
}
__device__ __forceinline__ void put_image(const uint32_t (&hi)[16], bf16* image, int rows,
                                          const Lane& l) {
  if (l.col < rows)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(image + (static_cast<int64_t>(4 * l.half + i) * rows + l.col) * 8) =
          make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
}
// This lane's value of token t in a 64 x 128 tile of values.
__device__ __forceinline__ float value_at(const unsigned char* v, int t, const Lane& l) {
  const uint32_t at = (l.row >> 6) * kTile + sw128_offset(t, (l.row & 63) >> 3) + 2 * (l.row & 7);
  return __bfloat162float(*reinterpret_cast<const bf16*>(v + at));
}
// 32 tokens of this lane to rows of a contiguous [.., Hv, dv] tensor.
__device__ __forceinline__ void put_rows(const float (&x)[32], bf16* dst, int64_t stride, int len,
                                         int dv, const Lane& l) {
  if (l.col >= dv) return;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int t = 32 * l.half + i;
    if (t < len) dst[t * stride] = __float2bfloat16_rn(x[i]);
  }
}

template <int DK>
__device__ __forceinline__ void walk(const gsa_delta_t& p, const SeqArgs& a, const Seq& s, int hv,
                                     const Lane& l, const Smem<DK>& sm, Bars& bars) {
  const int chunks = (s.len + kChunk - 1) / kChunk, rows = padded_dv(p.dv);
  const int64_t head = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  const int64_t stride = static_cast<int64_t>(p.Hv) * p.dv;
  bf16* out = static_cast<bf16*>(a.out) +
              ((static_cast<int64_t>(s.b) * p.T + s.begin) * p.Hv + hv) * p.dv + l.col;
  auto finish = [&](int n) {  // O of chunk n
    uint32_t r[32];
    tmem_ld32(l.tmem + kO + 32 * l.half, r);
    tc_wait_ld();
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
    put_rows(x, out + static_cast<int64_t>(n) * kChunk * stride, stride, s.len - n * kChunk, p.dv,
             l);
  };
  float S[DK / 2];
  load_state<DK>(S, a.state0 ? a.state0 + head : nullptr, p, l);
  float whole = 1.f;
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages;
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    if (n > 0) {
      if (!wait(&bars.upd_full, n - 1, a, bars)) return;
      add_update<DK>(S, whole, l);
    }
    put_operand<DK>(S, l, a.states ? a.states + slot * DK * rows : nullptr, rows);
    tc_wait_st();
    signal(&bars.s_ready);
    if (n > 0) {
      if (!wait(&bars.o_full, n - 1, a, bars)) return;
      finish(n - 1);
    }
    if (!wait(&bars.full_a[st], turn, a, bars)) return;
    const Block* blk = reinterpret_cast<const Block*>(sm.a(st) + tile_bytes<DK>());
    const unsigned char* v = sm.v(st);
    float y[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = value_at(v, 32 * l.half + i, l);
    if (!wait(&bars.r_full, n, a, bars)) return;
    uint32_t r[32], hi[16];
    tmem_ld32(l.tmem + kR + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 g = *reinterpret_cast<const float4*>(blk->grown + 32 * l.half + i);
      const float4 b = *reinterpret_cast<const float4*>(blk->beta + 32 * l.half + i);
      y[i] = b.x * fmaf(-g.x, __uint_as_float(r[i]), y[i]);
      y[i + 1] = b.y * fmaf(-g.y, __uint_as_float(r[i + 1]), y[i + 1]);
      y[i + 2] = b.z * fmaf(-g.z, __uint_as_float(r[i + 2]), y[i + 2]);
      y[i + 3] = b.w * fmaf(-g.w, __uint_as_float(r[i + 3]), y[i + 3]);
    }
    put_tokens(y, kYhi, l, hi);
    tc_wait_st();
    signal(&bars.y_ready);
    whole = blk->grown[kChunk - 1];
    if (!wait(&bars.n_full, n, a, bars)) return;
    tmem_ld32(l.tmem + kR + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 g = *reinterpret_cast<const float4*>(blk->left + 32 * l.half + i);
      y[i] = g.x * __uint_as_float(r[i]);
      y[i + 1] = g.y * __uint_as_float(r[i + 1]);
      y[i + 2] = g.z * __uint_as_float(r[i + 2]);
      y[i + 3] = g.w * __uint_as_float(r[i + 3]);
    }
    put_tokens(y, kDhi, l, hi);
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(r[i]);
    put_tokens(y, kYhi, l, hi);
    tc_wait_st();
    signal(&bars.d_ready);
    if (a.rows) put_image(hi, a.rows + slot * kChunk * rows, rows, l);
    signal(&bars.empty_a[st]);
    if (!wait(&bars.full_b[st], turn, a, bars)) return;
    const float* grown =
        reinterpret_cast<const float*>(sm.b(st) + tile_bytes<DK>() + 2 * kTile) + 32 * l.half;
    if (!wait(&bars.o1_full, n, a, bars)) return;
    tmem_ld32(l.tmem + kO + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 g = *reinterpret_cast<const float4*>(grown + i);
      r[i] = __float_as_uint(p.scale * g.x * __uint_as_float(r[i]));
      r[i + 1] = __float_as_uint(p.scale * g.y * __uint_as_float(r[i + 1]));
      r[i + 2] = __float_as_uint(p.scale * g.z * __uint_as_float(r[i + 2]));
      r[i + 3] = __float_as_uint(p.scale * g.w * __uint_as_float(r[i + 3]));
    }
    tmem_st32(l.tmem + kO + 32 * l.half, r);
    tc_wait_st();
    signal(&bars.o1_read);
    signal(&bars.empty_b[st]);
  }
  if (chunks > 0) {
    if (!wait(&bars.upd_full, chunks - 1, a, bars)) return;
    add_update<DK>(S, whole, l);
    if (!wait(&bars.o_full, chunks - 1, a, bars)) return;
    finish(chunks - 1);
  }
  if (a.state1) store_state<DK>(S, a.state1 + head, p, l);
}

// Backwards: dN = e^{c_64 - c} K dS + P^T dO, dY = T^T dN, dV = beta dY,
// dS <- e^{c_64} dS - K^T (e^c beta dY) + Q^T (scale e^c dO).
template <int DK>
__device__ __forceinline__ void walk_back(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                          int hv, const Lane& l, const Smem<DK>& sm, Bars& bars) {
  const int chunks = (s.len + kChunk - 1) / kChunk, rows = padded_dv(p.dv);
  const int64_t head = (static_cast<int64_t>(blockIdx.x) * p.Hv + hv) * p.dk * p.dv;
  const int64_t stride = static_cast<int64_t>(p.Hv) * p.dv;
  bf16* out = static_cast<bf16*>(a.out) +
              ((static_cast<int64_t>(s.b) * p.T + s.begin) * p.Hv + hv) * p.dv + l.col;
  float S[DK / 2];
  load_state<DK>(S, a.state0 ? a.state0 + head : nullptr, p, l);
  float whole = 1.f;
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages, at = chunks - 1 - n;
    const int64_t slot = static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
    if (n > 0) {
      if (!wait(&bars.upd_full, n - 1, a, bars)) return;
      add_update<DK>(S, whole, l);
    }
    put_operand<DK>(S, l, a.states + slot * DK * rows, rows);
    tc_wait_st();
    signal(&bars.s_ready);
    if (!wait(&bars.full_b[st], turn, a, bars)) return;
    float y[32];
    uint32_t r[32], hi[16];
    {
      const unsigned char* v = sm.v(st);
      const float* grown =
          reinterpret_cast<const float*>(sm.b(st) + tile_bytes<DK>() + 2 * kTile) + 32 * l.half;
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(grown + i);
        y[i] = p.scale * g.x * value_at(v, 32 * l.half + i, l);
        y[i + 1] = p.scale * g.y * value_at(v, 32 * l.half + i + 1, l);
        y[i + 2] = p.scale * g.z * value_at(v, 32 * l.half + i + 2, l);
        y[i + 3] = p.scale * g.w * value_at(v, 32 * l.half + i + 3, l);
      }
      put_tokens(y, kDhi, l, hi);
      signal(&bars.empty_b[st]);
    }
    if (!wait(&bars.full_a[st], turn, a, bars)) return;
    const Block* blk = reinterpret_cast<const Block*>(sm.a(st) + tile_bytes<DK>());
    if (!wait(&bars.o1_full, n, a, bars)) return;
    tmem_ld32(l.tmem + kO + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(r[i]);
    if (!wait(&bars.r_full, n, a, bars)) return;
    tmem_ld32(l.tmem + kR + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 g = *reinterpret_cast<const float4*>(blk->left + 32 * l.half + i);
      y[i] = fmaf(g.x, __uint_as_float(r[i]), y[i]);
      y[i + 1] = fmaf(g.y, __uint_as_float(r[i + 1]), y[i + 1]);
      y[i + 2] = fmaf(g.z, __uint_as_float(r[i + 2]), y[i + 2]);
      y[i + 3] = fmaf(g.w, __uint_as_float(r[i + 3]), y[i + 3]);
    }
    put_tokens(y, kYhi, l, hi);
    tc_wait_st();
    signal(&bars.y_ready);
    whole = blk->grown[kChunk - 1];
    if (!wait(&bars.n_full, n, a, bars)) return;
    tmem_ld32(l.tmem + kR + 32 * l.half, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 g = *reinterpret_cast<const float4*>(blk->grown + 32 * l.half + i);
      const float4 b = *reinterpret_cast<const float4*>(blk->beta + 32 * l.half + i);
      y[i] = -g.x * b.x * __uint_as_float(r[i]);
      y[i + 1] = -g.y * b.y * __uint_as_float(r[i + 1]);
      y[i + 2] = -g.z * b.z * __uint_as_float(r[i + 2]);
      y[i + 3] = -g.w * b.w * __uint_as_float(r[i + 3]);
    }
    put_tokens(y, kYhi, l, hi);
    tc_wait_st();
    signal(&bars.d_ready);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      hi[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    put_image(hi, a.rows + slot * kChunk * rows, rows, l);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 b = *reinterpret_cast<const float4*>(blk->beta + 32 * l.half + i);
      y[i] = b.x * __uint_as_float(r[i]);
      y[i + 1] = b.y * __uint_as_float(r[i + 1]);
      y[i + 2] = b.z * __uint_as_float(r[i + 2]);
      y[i + 3] = b.w * __uint_as_float(r[i + 3]);
    }
    signal(&bars.empty_a[st]);
    put_rows(y, out + static_cast<int64_t>(at) * kChunk * stride, stride, s.len - at * kChunk, p.dv,
             l);
  }
  if (chunks > 0) {
    if (!wait(&bars.upd_full, chunks - 1, a, bars)) return;
    add_update<DK>(S, whole, l);
  }
  if (a.state1) store_state<DK>(S, a.state1 + head, p, l);
}

template <int DK, bool REV>
__global__ void __launch_bounds__(kThreads, 1)
    seq_kernel(const gsa_delta_t p, const __grid_constant__ DeltaMaps maps, const SeqArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const Smem<DK> sm = {
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull)};
  __shared__ Bars bars;
  const int hv = blockIdx.y, col0 = blockIdx.z * kCols, warp = threadIdx.x >> 5;
  const Seq s = sequence(p, a.table, blockIdx.x);
  if (s.gap) {  // rows of no sequence: zeros
    const int pieces = min(kCols, p.dv - col0) / 8;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(s.len) * pieces; i += blockDim.x)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) +
                                ((s.begin + i / pieces) * p.Hv + hv) * p.dv + col0 +
                                i % pieces * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int chunks = (s.len + kChunk - 1) / kChunk;
  if (threadIdx.x == 0) {
    bars.abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full_a[i], 1);
      mbar_init(&bars.full_b[i], 1);
      mbar_init(&bars.empty_a[i], 1 + kComputeWarps);
      mbar_init(&bars.empty_b[i], 1 + kComputeWarps);
    }
    mbar_init(&bars.s_ready, kComputeWarps);
    mbar_init(&bars.y_ready, kComputeWarps);
    mbar_init(&bars.d_ready, kComputeWarps);
    mbar_init(&bars.o1_read, kComputeWarps);
    mbar_init(&bars.r_full, 1);
    mbar_init(&bars.n_full, 1);
    mbar_init(&bars.upd_full, 1);
    mbar_init(&bars.o1_full, 1);
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.drain, 1);
    fence_mbar_init();
  }
  if (warp == kComputeWarps) {
    tmem_alloc(&bars.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kComputeWarps + 1) {
    produce<DK, REV>(p, maps, a, s, hv, col0, sm, bars);
  } else if (warp == kComputeWarps) {
    if ((threadIdx.x & 31) == 0) issue<DK, REV>(a, chunks, sm, bars);
  } else {
    const int row = 32 * (warp & 3) + (threadIdx.x & 31);
    const Lane l = {row, warp >> 2, col0 + row,
                    bars.tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16)};
    if constexpr (REV)
      walk_back<DK>(p, a, s, hv, l, sm, bars);
    else
      walk<DK>(p, a, s, hv, l, sm, bars);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kComputeWarps) {
    tc_fence_after();
    tmem_dealloc(bars.tmem, kTmemCols);
  }
}

template <int DK, bool REV>
cudaError_t launch(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a,
                   cudaStream_t stream) {
  const cudaError_t e = allow_smem<seq_kernel<DK, REV>>(seq_smem<DK>());
  if (e != cudaSuccess) return e;
  const int seqs = p.N + (!REV && p.cu_seqlens ? 2 : 0);
  seq_kernel<DK, REV><<<dim3(seqs, p.Hv, (p.dv + kCols - 1) / kCols), kThreads, seq_smem<DK>(),
                        stream>>>(p, m, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_seq(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a, bool reverse,
                       cudaStream_t stream) {
  if (p.dk <= 64) return reverse ? launch<64, true>(p, m, a, stream) : launch<64, false>(p, m, a, stream);
  return reverse ? launch<128, true>(p, m, a, stream) : launch<128, false>(p, m, a, stream);
}

}  // namespace delta
}  // namespace gsa
