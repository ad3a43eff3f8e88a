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
// through shared memory.  Four more warps take the outputs away, off that path.  K, Q,
// V, T and P arrive by TMA, two chunks ahead.
//
// Left operands are pairs hi + lo of bf16 (2^-17 of a value together), q, k, v
// exact in bf16 and T, P pairs; the product of two lo parts is left out.  The state
// comes out within about 5e-6 of exact (2-norm) however many chunks there are, where
// operands in fp32 give 2e-7.  What the gradients need of a chunk (S0, N, backwards dS1, dY) is
// kept as the hi part alone: they round their factors to bf16 anyway.
//
// Bound by the chain of a chunk's three products and the passes between them,
// not by the tensor pipe (33% of the cycles) nor by memory (2.0 TB/s): 2.9 us a chunk
// alone on its SM, 4.1 with all SMs at work and rows and states kept.  64 heads of 4096
// tokens of 128 x 128 take 249 us forwards so, 225 backwards.
#include "delta_tc.cuh"

namespace gsa {
namespace delta {
namespace {

// kStates: only the state's path of kForward, for the first pass over segments.
enum Mode { kForward, kBackward, kStates };

constexpr int kStages = 2;
constexpr int kComputeWarps = 8;
constexpr int kRowWarps = 4;
constexpr int kIssueWarp = kComputeWarps + kRowWarps;
constexpr int kCopyWarp = kIssueWarp + 1;
constexpr int kThreads = 512;  // whole warpgroups: two warps idle
// Registers: 512 x 128 at launch = 256 x 168 (computing) + 256 x 88 (the others).
constexpr int kLaunchRegs = 128, kComputeRegs = 168, kOtherRegs = 88;
static_assert(256 * kComputeRegs + 256 * kOtherRegs <= kThreads * kLaunchRegs, "register split");
constexpr int kCols = 128;  // state columns of a block: the lanes of tensor memory
constexpr uint32_t kTmemCols = 512;

// Tensor memory, 32-bit columns; b = 0, 1 in turn by chunk.
enum : uint32_t {
  kAcc = 0,    // what a chunk adds to S^T [128][dk]
  kY = 0,      // forwards, before that: Y^T hi, lo (32 columns of two values each)
  kS = 128,    // S^T as a left operand hi, lo (64 columns of two values each);
               // backwards, once dS^T K^T is there: dN^T, then -e^c beta dY^T hi, lo
  kD = 192,    // then (e^{c_64 - c} N)^T (backwards (scale e^c dO)^T) hi, lo
  kRO = 256,   // + 128 b: R^T, then N^T (64), O^T (64); N^T as an operand in its own
               // place, for each half of the tokens hi, lo (16 each).  Backwards
               // dS^T K^T and dO^T P, then [dN T_hi | dN T_lo]^T
};

constexpr uint32_t kKq = 2 * kTile;  // K and Q: 128 rows of 64 channels
template <int DK>
__host__ __device__ constexpr int kq_bytes() { return (DK / 64) * static_cast<int>(kKq); }
constexpr int kValueBytes = 2 * static_cast<int>(kTile);
// Queue a: K and Q, T with the decays, 64 x 128 values (v, or dO); queue b: P.
template <int DK>
__host__ __device__ constexpr int a_bytes() { return kq_bytes<DK>() + kTBytes + kValueBytes; }
// ... and 64 rows of 128 outputs on their way out.
constexpr int kRowBytes = 256;
template <int DK>
__host__ __device__ constexpr int seq_smem() {
  // values are swizzled tiles: they come before T, whose decays break the 1024 bytes
  return kStages * (a_bytes<DK>() + kPBytes) + kChunk * kRowBytes + 1024;
}
template <int DK>
struct Smem {
  unsigned char* base;
  __device__ unsigned char* a(int st) const { return base + st * a_bytes<DK>(); }
  __device__ unsigned char* v(int st) const { return a(st) + kq_bytes<DK>(); }
  __device__ unsigned char* t(int st) const { return v(st) + kValueBytes; }
  __device__ unsigned char* p(int st) const {
    return base + kStages * a_bytes<DK>() + st * kPBytes;
  }
  __device__ unsigned char* out() const { return p(kStages); }
};

// Every barrier but the queues' completes once a chunk, and never twice while a
// warp still has to wait for the first of the two (a parity tells only neighbouring
// phases apart): whoever completes it has waited, since the time before, for
// something that its waiters signal later.
struct Bars {
  uint64_t full_a[kStages], empty_a[kStages], full_b[kStages], empty_b[kStages];
  uint64_t s_ready, r_full, o1_full, y_ready, n_full, d_ready, upd_full, o_full;
  uint64_t x_ready;  // forwards N is an operand, backwards dO is
  uint64_t o_read;   // the row warps are through with a chunk's accumulators
  uint64_t rows;     // ... and have written their columns of its output rows
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
template <int DK, int MODE>
__device__ __forceinline__ void produce(const gsa_delta_t& p, const DeltaMaps& maps,
                                        const SeqArgs& a, const Seq& s, int hv, int col0,
                                        bool values, const Smem<DK>& sm, Bars& bars) {
  constexpr bool REV = MODE == kBackward;
  const int lane = threadIdx.x & 31, hk = hv / (p.Hv / p.Hk);
  const int chunks = (s.len + kChunk - 1) / kChunk;
  const bool have = values && (!REV || a.in != nullptr);  // else zeros
  int begun[2] = {0, 0};
  bool ok = true;
  for (int n = 0; ok && n < chunks; ++n) {
    const int st = n % kStages, parity = ((n / kStages) & 1) ^ 1;
    const int at = REV ? chunks - 1 - n : n;
    const int begin = s.begin + at * kChunk, rest = s.len - at * kChunk;
    const int len = rest < kChunk ? rest : kChunk;
    const bool whole = len == kChunk || !p.cu_seqlens;
    const Block* blk = a.blocks + static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
    ok = mbar_wait_warp(&bars.empty_a[st], parity, a.err, &bars.abort);
    if (!ok) break;
    bool by_hand = false;
    if (!whole) {
      for (int i = 0; i < DK / 64; ++i) {
        const uint32_t to = smem_u32(sm.a(st)) + i * kKq;
        copy_rows(to, rows_at(p.k, p.k_stride, s.b, begin, hk) + 64 * i, p.k_stride[1], len, 64,
                  p.dk - 64 * i, lane, 32);
        if (MODE != kStates)
          copy_rows(to + kTile, rows_at(p.q, p.q_stride, s.b, begin, hk) + 64 * i, p.q_stride[1],
                    len, 64, p.dk - 64 * i, lane, 32);
      }
      by_hand = true;
    }
    if (values && (!whole || !have)) {
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
      uint64_t* full = &bars.full_a[st];
      constexpr int kRowsBytes = MODE == kStates ? kq_bytes<DK>() / 2 : kq_bytes<DK>();
      mbar_arrive_expect_tx(full, kTBytes + (whole ? kRowsBytes : 0) +
                                      (whole && have ? kValueBytes : 0));
      bulk_load(sm.t(st), blk, kTBytes, full);
      if (whole)
        for (int i = 0; i < DK / 64; ++i) {
          tma_load_rows(sm.a(st) + i * kKq, &maps.k, 64 * i, hk, begin, s.b, full);
          if (MODE != kStates)
            tma_load_rows(sm.a(st) + i * kKq + kTile, &maps.q, 64 * i, hk, begin, s.b, full);
        }
      if (whole && have)
        for (int i = 0; i < 2; ++i)
          tma_load_rows(sm.v(st) + i * kTile, &maps.v, col0 + 64 * i, hv, begin, s.b, full);
    }
    ++begun[0];
    if (MODE == kStates) continue;
    ok = mbar_wait_warp(&bars.empty_b[st], parity, a.err, &bars.abort);
    if (!ok) break;
    if (lane == 0) {
      mbar_arrive_expect_tx(&bars.full_b[st], kPBytes);
      bulk_load(sm.p(st), blk->p_hi, kPBytes, &bars.full_b[st]);
    }
    ++begun[1];
  }
  if (!ok) {  // gave up: no copy of ours may outlive the block
    for (int i = max(0, begun[0] - kStages); i < begun[0]; ++i)
      mbar_wait_drain(&bars.full_a[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
    for (int i = max(0, begun[1] - kStages); i < begun[1]; ++i)
      mbar_wait_drain(&bars.full_b[i % kStages], (i / kStages) & 1, kWaitLimitCycles);
  }
}

// acc (+)= left B over KS steps of 16 of the contraction; B's first step has the
// descriptor `b`, the next ones lie COLS ? 2048 : 32 bytes on (and `step` bytes
// after every fourth, where 64 columns end).
template <int KS, bool COLS>
__device__ __forceinline__ void times(uint32_t acc, uint32_t left, uint64_t b, uint32_t step,
                                      uint32_t idesc, bool fresh) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const uint32_t off = COLS ? ks * 2048 : (ks >> 2) * step + (ks & 3) * 32;
    warp_mma_ts(acc, left + 8 * ks, b + (off >> 4), idesc, !fresh || ks);
  }
}

// O^T += N^T P^T: N's halves lie apart.
__device__ __forceinline__ void times_inner(uint32_t ro, uint64_t p_rows, uint32_t idesc) {
#pragma unroll
  for (int i = 0; i < 3; ++i)  // hi P_hi, lo P_hi, hi P_lo
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
      warp_mma_ts(ro + 64, ro + 32 * (ks >> 1) + 8 * (ks & 1) + (i == 1 ? 16 : 0),
                  p_rows + (i == 2 ? kTile >> 4 : 0) + 2 * ks, idesc, 1);
}

// One warp issues all products.
template <int DK, int MODE>
__device__ __forceinline__ void issue(const SeqArgs& a, int chunks, const Smem<DK>& sm,
                                      Bars& bars) {
  const uint32_t tm = __shfl_sync(0xFFFFFFFFu, bars.tmem, 0);
  constexpr uint32_t kRows64 = idesc_bf16_f32(128, 64, 0, 0);
  constexpr uint32_t kCols64 = idesc_bf16_f32(128, 64, 0, 1);
  constexpr uint32_t kCols128 = idesc_bf16_f32(128, 128, 0, 1);
  constexpr uint32_t kColsDk = idesc_bf16_f32(128, DK, 0, 1);
  constexpr uint32_t kColsCols = idesc_bf16_f32(128, 64, 1, 1);
  constexpr uint32_t kLo = DK / 2;  // from S's hi columns to its lo columns
  // descriptors of stage 0; a stage is a_bytes (P: kPBytes) further
  const uint64_t k_rows = desc_rows(smem_u32(sm.a(0)), 0), q_rows = k_rows + (kTile >> 4);
  const uint64_t k_cols = desc_cols(smem_u32(sm.a(0)), 0, kKq), q_cols = k_cols + (kTile >> 4);
  const uint64_t v_cols = desc_cols(smem_u32(sm.v(0)), 0);
  const uint64_t t_rows = desc_rows(smem_u32(sm.t(0)), 0), t_cols = desc_cols(smem_u32(sm.t(0)), 0);
  const uint64_t p_rows = desc_rows(smem_u32(sm.p(0)), 0), p_cols = desc_cols(smem_u32(sm.p(0)), 0);
  auto inner = [&](int n) {  // forwards: the rest of O of chunk n
    if (!wait(&bars.full_b[n & 1], n >> 1, a, bars)) return false;
    times_inner(tm + kRO + 128 * (n & 1), p_rows + (n & 1) * (kPBytes >> 4), kRows64);
    warp_commit(&bars.o_full);
    warp_commit(&bars.empty_b[n & 1]);
    return true;
  };
  static_assert(kStages == 2, "two stages");
  for (int n = 0; n < chunks; ++n) {
    const int st = n & 1, turn = n >> 1;
    const uint32_t da = st * (a_bytes<DK>() >> 4), dp = st * (kPBytes >> 4);
    const uint32_t ro = tm + kRO + 128 * st;
    if (!wait(&bars.full_a[st], turn, a, bars)) break;
    if constexpr (MODE == kBackward) {
      if (!wait(&bars.full_b[st], turn, a, bars)) break;
      if (n > 0 && !wait(&bars.upd_full, n - 1, a, bars)) break;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        warp_mma_ss(ro + 64, v_cols + da + (i & 3) * 128,
                    p_cols + dp + (i >> 2) * (kTile >> 4) + (i & 3) * 128, kColsCols, i > 0);
      warp_commit(&bars.empty_b[st]);
      if (!wait(&bars.s_ready, n, a, bars)) break;
      times<DK / 16, false>(ro, tm + kS, k_rows + da, kKq, kRows64, true);
      times<DK / 16, false>(ro, tm + kS + kLo, k_rows + da, kKq, kRows64, false);
      warp_commit(&bars.r_full);
      if (!wait(&bars.y_ready, n, a, bars)) break;
      // the row warps have left the last chunk: its accumulators are the next one's, and
      // no barrier they wait for runs ahead of them by two
      if (n > 0 && !wait(&bars.o_read, n - 1, a, bars)) break;
      times<4, true>(ro, tm + kS, t_cols + da, kTile, kCols128, true);
      times<4, true>(ro, tm + kS + 32, t_cols + da, kTile, kCols64, false);
      warp_commit(&bars.n_full);
      if (!wait(&bars.x_ready, n, a, bars) || !wait(&bars.n_full, n, a, bars)) break;
      times<4, true>(tm + kAcc, tm + kD, q_cols + da, kKq, kColsDk, true);
      times<4, true>(tm + kAcc, tm + kD + 32, q_cols + da, kKq, kColsDk, false);
      if (!wait(&bars.d_ready, n, a, bars)) break;
      times<4, true>(tm + kAcc, tm + kS, k_cols + da, kKq, kColsDk, false);
      times<4, true>(tm + kAcc, tm + kS + 32, k_cols + da, kKq, kColsDk, false);
      warp_commit(&bars.upd_full);
      warp_commit(&bars.empty_a[st]);
    } else {
      if (!wait(&bars.s_ready, n, a, bars)) break;
      times<DK / 16, false>(ro, tm + kS, k_rows + da, kKq, kRows64, true);
      times<DK / 16, false>(ro, tm + kS + kLo, k_rows + da, kKq, kRows64, false);
      warp_commit(&bars.r_full);
      if constexpr (MODE == kForward) {
        // O's products fill the pipe while the threads work on R, and later on N.  They
        // are issued once R (N) has arrived: a commit waits for the products behind it too
        if (n > 1 && !wait(&bars.o_read, n - 2, a, bars)) break;
        if (!wait(&bars.r_full, n, a, bars)) break;
        times<DK / 16, false>(ro + 64, tm + kS, q_rows + da, kKq, kRows64, true);
        times<DK / 16, false>(ro + 64, tm + kS + kLo, q_rows + da, kKq, kRows64, false);
        warp_commit(&bars.o1_full);
      }
      if (!wait(&bars.y_ready, n, a, bars)) break;
      times<4, false>(ro, tm + kY, t_rows + da, kTile, kRows64, true);
      times<4, false>(ro, tm + kY + 32, t_rows + da, kTile, kRows64, false);
      times<4, false>(ro, tm + kY, t_rows + da + (kTile >> 4), kTile, kRows64, false);
      warp_commit(&bars.n_full);
      if constexpr (MODE == kForward) {
        if (!wait(&bars.n_full, n, a, bars)) break;
        if (n > 0 && !inner(n - 1)) break;
      }
      if (!wait(&bars.d_ready, n, a, bars)) break;
      times<4, true>(tm + kAcc, tm + kD, k_cols + da, kKq, kColsDk, true);
      times<4, true>(tm + kAcc, tm + kD + 32, k_cols + da, kKq, kColsDk, false);
      warp_commit(&bars.upd_full);
      warp_commit(&bars.empty_a[st]);
      if constexpr (MODE == kForward) {
        if (!wait(&bars.x_ready, n, a, bars)) break;
        if (n == chunks - 1) {
          // as in every step, o_full may complete again only once its last waiters are through
          if (n > 0 && !wait(&bars.o_read, n - 1, a, bars)) break;
          if (!inner(n)) break;
        }
      }
    }
  }
  // nothing of ours may be in flight when tensor memory is freed
  warp_commit(&bars.drain);
  mbar_wait_drain(&bars.drain, 0, kWaitLimitCycles);
  __syncwarp();
}

// What a computing thread is: half `half` of column `col` of the value head.
struct Lane {
  int row;        // lane of tensor memory, 0 .. 127
  int half;       // which half of the channels, and of the tokens
  int col;        // column of the value head
  uint32_t tmem;  // its lane's address
};

// Where a block's state comes from (zeros without `in`, or the identity) and goes to.
struct States {
  const float* in;
  float* out;
  int width;      // columns of both: dv, or dk for M
  bool identity;
};
// The state's half column, in fp32: from and to [dk, width].
template <int DK>
__device__ __forceinline__ void load_state(float (&S)[DK / 2], const States& st, int dk,
                                           const Lane& l) {
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) {
    const int r = l.half * (DK / 2) + i;
    const bool real = r < dk && l.col < st.width;
    S[i] = st.in && real ? st.in[static_cast<int64_t>(r) * st.width + l.col]
                         : (st.identity && real && r == l.col ? 1.f : 0.f);
  }
}
template <int DK>
__device__ __forceinline__ void store_state(const float (&S)[DK / 2], const States& st, int dk,
                                            const Lane& l) {
#pragma unroll
  for (int i = 0; i < DK / 2; ++i) {
    const int r = l.half * (DK / 2) + i;
    if (r < dk && l.col < st.width) st.out[static_cast<int64_t>(r) * st.width + l.col] = S[i];
  }
}
// S <- whole S + what the last chunk added.  All loads are under way before the
// first is waited for.
template <int DK>
__device__ __forceinline__ void add_update(float (&S)[DK / 2], float whole, const Lane& l) {
  uint32_t r[DK / 64][32];
#pragma unroll
  for (int q = 0; q < DK / 64; ++q) tmem_ld32(l.tmem + kAcc + l.half * (DK / 2) + 32 * q, r[q]);
#pragma unroll
  for (int q = 0; q < DK / 64; ++q) {
    tc_wait_ld(r[q]);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const uint64_t x = f2_fma(f2_pack(whole, whole), f2_pack(S[32 * q + i], S[32 * q + i + 1]),
                                f2_pack(__uint_as_float(r[q][i]), __uint_as_float(r[q][i + 1])));
      S[32 * q + i] = f2_lo(x);
      S[32 * q + i + 1] = f2_hi(x);
    }
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
    tmem_st16(l.tmem + kS + l.half * (DK / 4) + 16 * q, hi);
    tmem_st16(l.tmem + kS + DK / 2 + l.half * (DK / 4) + 16 * q, lo);
    if (image && l.col < rows)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(
            image + (static_cast<int64_t>(l.half * (DK / 16) + 4 * q + i) * rows + l.col) * 8) =
            make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
  }
}
// 32 tokens of a left operand (hi at `at`, lo 32 columns behind); hi is handed back.
__device__ __forceinline__ void put_tokens(const float (&x)[32], uint32_t at, const Lane& l,
                                           uint32_t (&hi)[16]) {
  uint32_t lo[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) split(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
  tmem_st16(at + 16 * l.half, hi);
  tmem_st16(at + 32 + 16 * l.half, lo);
}
// This lane's values of its 32 tokens from two 64 x 64 tiles, times a factor a token.
__device__ __forceinline__ void load_values(float (&x)[32], const unsigned char* v,
                                            const float* factor, float scale, const Lane& l) {
  v += (l.row >> 6) * kTile + 32 * l.half * 128 + 2 * (l.row & 7);
  const int piece = (l.row & 63) >> 3;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 f = *reinterpret_cast<const float4*>(factor + 32 * l.half + i);
    const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[i + e] = scale * fs[e] *
                 __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(
                                     v + sw128_offset(i + e, piece)))
                                 << 16);
  }
}

template <int DK, bool OUT>
__device__ __forceinline__ void walk(const gsa_delta_t& p, const SeqArgs& a, const Seq& s, int hv,
                                     const States& io, const Lane& l, const Smem<DK>& sm,
                                     Bars& bars) {
  const int chunks = (s.len + kChunk - 1) / kChunk, rows = padded_dv(p.dv);
  const int t0 = 32 * l.half;
  float S[DK / 2];
  load_state<DK>(S, io, p.dk, l);
  float whole = 1.f;
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages;
    const uint32_t ro = l.tmem + kRO + 128 * (n & 1);
    const int64_t slot = static_cast<int64_t>(s.chunk0 + n) * p.Hv + hv;
    if (n > 0) {
      if (!wait(&bars.upd_full, n - 1, a, bars)) return;
      add_update<DK>(S, whole, l);
    }
    put_operand<DK>(S, l, OUT && a.states ? a.states + slot * DK * rows : nullptr, rows);
    tc_wait_st();
    signal(&bars.s_ready);
    if (!wait(&bars.full_a[st], turn, a, bars)) return;
    const Gates* gates = reinterpret_cast<const Gates*>(sm.t(st) + 2 * kTile);
    float y[32];
    uint32_t hi[16];
    if (OUT || !io.identity) {
      load_values(y, sm.v(st), gates->beta, 1.f, l);  // beside the first product
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) y[i] = 0.f;
    }
    whole = gates->grown[kChunk - 1];
    if (!wait(&bars.r_full, n, a, bars)) return;
    {
      uint32_t r[32];
      tmem_ld32(ro + t0, r);
      tc_wait_ld(r);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {  // beta V - (beta e^c) R
        const float4 g = *reinterpret_cast<const float4*>(gates->both + t0 + i);
        y[i] = fmaf(-g.x, __uint_as_float(r[i]), y[i]);
        y[i + 1] = fmaf(-g.y, __uint_as_float(r[i + 1]), y[i + 1]);
        y[i + 2] = fmaf(-g.z, __uint_as_float(r[i + 2]), y[i + 2]);
        y[i + 3] = fmaf(-g.w, __uint_as_float(r[i + 3]), y[i + 3]);
      }
    }
    put_tokens(y, l.tmem + kY, l, hi);
    tc_wait_st();
    signal(&bars.y_ready);
    if constexpr (OUT) {  // beside the product with T: O's part from the state gets its decays
      if (!wait(&bars.o1_full, n, a, bars)) return;
      uint32_t r[32];
      tmem_ld32(ro + 64 + t0, r);
      tc_wait_ld(r);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(gates->grown + t0 + i);
        r[i] = __float_as_uint(p.scale * g.x * __uint_as_float(r[i]));
        r[i + 1] = __float_as_uint(p.scale * g.y * __uint_as_float(r[i + 1]));
        r[i + 2] = __float_as_uint(p.scale * g.z * __uint_as_float(r[i + 2]));
        r[i + 3] = __float_as_uint(p.scale * g.w * __uint_as_float(r[i + 3]));
      }
      tmem_st32(ro + 64 + t0, r);
    }
    if (!wait(&bars.n_full, n, a, bars)) return;
    {
      uint32_t r[32];
      tmem_ld32(ro + t0, r);
      tc_wait_ld(r);
#pragma unroll
      for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(r[i]);
    }
    {
      float x[32];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(gates->left + t0 + i);
        x[i] = g.x * y[i];
        x[i + 1] = g.y * y[i + 1];
        x[i + 2] = g.z * y[i + 2];
        x[i + 3] = g.w * y[i + 3];
      }
      put_tokens(x, l.tmem + kD, l, hi);
    }
    tc_wait_st();
    signal(&bars.d_ready);
    if constexpr (OUT) {  // beside the state's product
      uint32_t lo[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) split(y[2 * i], y[2 * i + 1], hi[i], lo[i]);
      tmem_st16(ro + t0, hi);
      tmem_st16(ro + t0 + 16, lo);
      tc_wait_st();
      signal(&bars.x_ready);
    }
    signal(&bars.empty_a[st]);
    if (OUT && a.rows && l.col < rows)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(a.rows + slot * kChunk * rows +
                                  (static_cast<int64_t>(4 * l.half + i) * rows + l.col) * 8) =
            make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
  }
  if (chunks > 0) {
    if (!wait(&bars.upd_full, chunks - 1, a, bars)) return;
    add_update<DK>(S, whole, l);
  }
  if (io.out) store_state<DK>(S, io, p.dk, l);
}

// Backwards: dN = e^{c_64 - c} K dS + P^T dO, dY = T^T dN, dV = beta dY,
// dS <- e^{c_64} dS - K^T (e^c beta dY) + Q^T (scale e^c dO).
template <int DK>
__device__ __forceinline__ void walk_back(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                          int hv, const States& io, const Lane& l,
                                          const Smem<DK>& sm, Bars& bars) {
  const int chunks = (s.len + kChunk - 1) / kChunk, rows = padded_dv(p.dv);
  const int t0 = 32 * l.half;
  float S[DK / 2];
  load_state<DK>(S, io, p.dk, l);
  float whole = 1.f;
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages, at = chunks - 1 - n;
    const uint32_t ro = l.tmem + kRO + 128 * (n & 1);
    const int64_t slot = static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
    if (n > 0) {
      if (!wait(&bars.upd_full, n - 1, a, bars)) return;
      add_update<DK>(S, whole, l);
    }
    put_operand<DK>(S, l, a.states + slot * DK * rows, rows);
    tc_wait_st();
    signal(&bars.s_ready);
    if (!wait(&bars.full_a[st], turn, a, bars)) return;
    const Gates* gates = reinterpret_cast<const Gates*>(sm.t(st) + 2 * kTile);
    whole = gates->grown[kChunk - 1];
    float y[32];
    uint32_t hi[16];
    if (!wait(&bars.r_full, n, a, bars)) return;
    {
      uint32_t r[32], u[32];
      tmem_ld32(ro + t0, r);
      tmem_ld32(ro + 64 + t0, u);
      tc_wait_ld(r, u);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(gates->left + t0 + i);
        y[i] = fmaf(g.x, __uint_as_float(r[i]), __uint_as_float(u[i]));
        y[i + 1] = fmaf(g.y, __uint_as_float(r[i + 1]), __uint_as_float(u[i + 1]));
        y[i + 2] = fmaf(g.z, __uint_as_float(r[i + 2]), __uint_as_float(u[i + 2]));
        y[i + 3] = fmaf(g.w, __uint_as_float(r[i + 3]), __uint_as_float(u[i + 3]));
      }
    }
    put_tokens(y, l.tmem + kS, l, hi);
    tc_wait_st();
    signal(&bars.y_ready);
    load_values(y, sm.v(st), gates->grown, p.scale, l);  // beside the product with T
    put_tokens(y, l.tmem + kD, l, hi);
    tc_wait_st();
    signal(&bars.x_ready);
    if (!wait(&bars.n_full, n, a, bars)) return;
    {
      uint32_t r[32], u[32];
      tmem_ld32(ro + t0, r);
      tmem_ld32(ro + 64 + t0, u);
      tc_wait_ld(r, u);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 g = *reinterpret_cast<const float4*>(gates->both + t0 + i);
        y[i] = -g.x * (__uint_as_float(r[i]) + __uint_as_float(u[i]));
        y[i + 1] = -g.y * (__uint_as_float(r[i + 1]) + __uint_as_float(u[i + 1]));
        y[i + 2] = -g.z * (__uint_as_float(r[i + 2]) + __uint_as_float(u[i + 2]));
        y[i + 3] = -g.w * (__uint_as_float(r[i + 3]) + __uint_as_float(u[i + 3]));
      }
    }
    put_tokens(y, l.tmem + kS, l, hi);
    tc_wait_st();
    signal(&bars.d_ready);
    signal(&bars.empty_a[st]);
  }
  if (chunks > 0) {
    if (!wait(&bars.upd_full, chunks - 1, a, bars)) return;
    add_update<DK>(S, whole, l);
  }
  if (io.out) store_state<DK>(S, io, p.dk, l);
}

// The row warps, one a quadrant of lanes: forwards O leaves; backwards dY is kept and
// dV = beta dY leaves.  Rows leave by way of shared memory, 256 bytes together.
template <int DK, bool REV>
__device__ __forceinline__ void take_rows(const gsa_delta_t& p, const SeqArgs& a, const Seq& s,
                                          int hv, int row, int col0, uint32_t tmem,
                                          const Smem<DK>& sm, Bars& bars) {
  const int chunks = (s.len + kChunk - 1) / kChunk, rows = padded_dv(p.dv), col = col0 + row;
  const int64_t stride = static_cast<int64_t>(p.Hv) * p.dv;
  bf16* out = static_cast<bf16*>(a.out) +
              ((static_cast<int64_t>(s.b) * p.T + s.begin) * p.Hv + hv) * p.dv + col0;
  unsigned char* mine = sm.out() + 2 * row;
  const int piece = (row & 15) * 8, first = row >> 4;
  for (int n = 0; n < chunks; ++n) {
    const int st = n % kStages, turn = n / kStages, at = REV ? chunks - 1 - n : n;
    const uint32_t ro = tmem + kRO + 128 * (n & 1);
    const int64_t slot = static_cast<int64_t>(s.chunk0 + at) * p.Hv + hv;
    const Gates* gates = reinterpret_cast<const Gates*>(sm.t(st) + 2 * kTile);
    if (REV && !wait(&bars.full_a[st], turn, a, bars)) return;
    if (!wait(REV ? &bars.n_full : &bars.o_full, n, a, bars)) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t r[16], u[16];
      tmem_ld16(ro + (REV ? 0 : 64) + 16 * q, r);
      if constexpr (REV) tmem_ld16(ro + 64 + 16 * q, u);
      tc_wait_ld(r, u);
      if constexpr (REV) {
        uint32_t hi[8];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(u[i]));
#pragma unroll
        for (int i = 0; i < 8; ++i)
          hi[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        if (col < rows)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(a.rows + slot * kChunk * rows +
                                      (static_cast<int64_t>(2 * q + i) * rows + col) * 8) =
                make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 b = *reinterpret_cast<const float4*>(gates->beta + 16 * q + i);
          r[i] = __float_as_uint(b.x * __uint_as_float(r[i]));
          r[i + 1] = __float_as_uint(b.y * __uint_as_float(r[i + 1]));
          r[i + 2] = __float_as_uint(b.z * __uint_as_float(r[i + 2]));
          r[i + 3] = __float_as_uint(b.w * __uint_as_float(r[i + 3]));
        }
      }
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const uint32_t x = pack_bf16x2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        *reinterpret_cast<uint16_t*>(mine + (16 * q + i) * kRowBytes) = static_cast<uint16_t>(x);
        *reinterpret_cast<uint16_t*>(mine + (16 * q + i + 1) * kRowBytes) =
            static_cast<uint16_t>(x >> 16);
      }
    }
    signal(&bars.o_read);
    if constexpr (REV) signal(&bars.empty_a[st]);
    signal(&bars.rows);
    if (!wait(&bars.rows, 2 * n, a, bars)) return;
    const int len = s.len - at * kChunk;
    if (piece < p.dv - col0)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (first + 8 * i < len)
          *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(at) * kChunk + first + 8 * i) *
                                              stride + piece) =
              *reinterpret_cast<const uint4*>(sm.out() + (first + 8 * i) * kRowBytes + 2 * piece);
    signal(&bars.rows);  // the rows are read: the next chunk's may be written
    if (!wait(&bars.rows, 2 * n + 1, a, bars)) return;
  }
}

// Block (sequence or segment, longest first, and value head; 128 columns).
template <int DK, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    seq_kernel(const gsa_delta_t p, const __grid_constant__ DeltaMaps maps, const SeqArgs a) {
  extern __shared__ unsigned char smem_raw[];
  constexpr bool REV = MODE == kBackward;
  const Smem<DK> sm = {
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull)};
  __shared__ Bars bars;
  const int hv = blockIdx.x % p.Hv, warp = threadIdx.x >> 5;
  const int segs = MODE == kStates ? a.seg.count - 1 : (REV ? 1 : a.seg.count);
  const int rank = blockIdx.x / p.Hv / segs, seg = blockIdx.x / p.Hv % segs;
  const int n = p.cu_seqlens ? a.table.order[rank] : rank;
  const int blocks_v = (p.dv + kCols - 1) / kCols;
  const bool matrix = MODE == kStates && static_cast<int>(blockIdx.y) == blocks_v;  // M, not B
  const int col0 = matrix ? 0 : blockIdx.y * kCols;
  Seq s = sequence(p, a.table, n);
  if (s.gap) {  // rows of no sequence: zeros (backwards the gradients' kernel writes them)
    if (REV) return;
    const int pieces = min(kCols, p.dv - col0) / 8;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(s.len) * pieces; i += blockDim.x)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) +
                                ((s.begin + i / pieces) * p.Hv + hv) * p.dv + col0 +
                                i % pieces * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int64_t size = static_cast<int64_t>(p.dk) * p.dv;
  const int64_t head = static_cast<int64_t>(n) * p.Hv + hv;
  States io = {a.state0 ? a.state0 + head * size : nullptr,
               a.state1 ? a.state1 + head * size : nullptr, p.dv, false};
  if (MODE != kBackward && a.seg.count > 1) {
    const int cuts = a.seg.count - 1;
    s.chunk0 += seg * a.seg.chunks;
    s.begin += seg * a.seg.chunks * kChunk;
    s.len = min(s.len - seg * a.seg.chunks * kChunk, a.seg.chunks * kChunk);
    const int64_t cut = static_cast<int64_t>(n) * cuts;
    if (MODE == kStates) {
      if (matrix && seg == 0) return;  // the first segment starts from its own state
      if (seg > 0) io.in = nullptr;
      io.out = matrix ? a.seg_m + ((cut + seg) * p.Hv + hv) * p.dk * p.dk
                      : a.seg_b + ((cut + seg) * p.Hv + hv) * size;
      io.identity = matrix;
      if (matrix) io.width = p.dk;
    } else {
      if (seg > 0) io.in = a.seg_s + ((cut + seg - 1) * p.Hv + hv) * size;
      if (seg < cuts) io.out = nullptr;
    }
  }
  const int chunks = (s.len + kChunk - 1) / kChunk;
  if (threadIdx.x == 0) {
    bars.abort = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full_a[i], 1);
      mbar_init(&bars.full_b[i], 1);
      mbar_init(&bars.empty_a[i], 1 + kComputeWarps + (REV ? kRowWarps : 0));
      mbar_init(&bars.empty_b[i], 1);
    }
    mbar_init(&bars.s_ready, kComputeWarps);
    mbar_init(&bars.y_ready, kComputeWarps);
    mbar_init(&bars.d_ready, kComputeWarps);
    mbar_init(&bars.x_ready, kComputeWarps);
    mbar_init(&bars.o_read, kRowWarps);
    mbar_init(&bars.rows, kRowWarps);
    mbar_init(&bars.r_full, 1);
    mbar_init(&bars.o1_full, 1);
    mbar_init(&bars.n_full, 1);
    mbar_init(&bars.upd_full, 1);
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.drain, 1);
    fence_mbar_init();
  }
  if (warp == kIssueWarp) {
    tmem_alloc(&bars.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int row = 32 * (warp & 3) + (threadIdx.x & 31);
  const uint32_t tmem = bars.tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
  if (warp < kComputeWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
    const Lane l = {row, warp >> 2, col0 + row, tmem};
    if constexpr (REV)
      walk_back<DK>(p, a, s, hv, io, l, sm, bars);
    else
      walk<DK, MODE == kForward>(p, a, s, hv, io, l, sm, bars);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kCopyWarp) {
      produce<DK, MODE>(p, maps, a, s, hv, col0, !matrix, sm, bars);
    } else if (warp == kIssueWarp) {
      issue<DK, MODE>(a, chunks, sm, bars);
    } else if (warp < kIssueWarp && MODE != kStates) {
      take_rows<DK, REV>(p, a, s, hv, row, col0, tmem, sm, bars);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_dealloc(bars.tmem, kTmemCols);
  }
}

// From segment to segment: S_1 = B_0, S_{i+1} = M_i S_i + B_i, in fp32.  A block has
// 16 columns of a head's state; M_{i+1} is on its way while M_i is used.  Bound by
// shared memory: 64 threads hold 8 rows x 4 columns each, and four such groups share
// the contraction (one group of 256 threads with 2 x 4: twice the loads).
constexpr int kLdCut = 132, kCutCols = 16, kCutThreads = 256;
constexpr int kCutSmem = (2 * 128 * kLdCut + 6 * 128 * kCutCols) * 4;
__global__ void __launch_bounds__(kCutThreads) cut_kernel(const gsa_delta_t p, const SeqArgs a) {
  extern __shared__ float cut_smem[];
  float* M = cut_smem;                  // [2][128][kLdCut]
  float* S = M + 2 * 128 * kLdCut;      // [2][128][kCutCols]
  float* parts = S + 2 * 128 * kCutCols;  // [4][128][kCutCols]
  const int tid = threadIdx.x, hv = blockIdx.y, col0 = blockIdx.z * kCutCols;
  const int cuts = a.seg.count - 1;
  const int64_t size = static_cast<int64_t>(p.dk) * p.dv;
  auto at = [&](int i) { return (static_cast<int64_t>(blockIdx.x) * cuts + i) * p.Hv + hv; };
  auto fetch = [&](int i) {
    const float* m = a.seg_m + at(i) * p.dk * p.dk;
    const uint32_t to = smem_u32(M + (i & 1) * 128 * kLdCut);
    const int c = (tid & 31) * 4;  // a row a warp
    if (c < p.dk)
#pragma unroll 4
      for (int r = tid >> 5; r < p.dk; r += kCutThreads / 32)
        cp16(to + (r * kLdCut + c) * 4, m + r * p.dk + c, true);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (cuts > 1) fetch(1);
  for (int x = tid; x < p.dk * kCutCols; x += kCutThreads) {
    const int r = x / kCutCols, c = x % kCutCols;
    if (col0 + c < p.dv) {
      const float v = a.seg_b[at(0) * size + static_cast<int64_t>(r) * p.dv + col0 + c];
      S[x] = v;
      a.seg_s[at(0) * size + static_cast<int64_t>(r) * p.dv + col0 + c] = v;
    } else {
      S[x] = 0.f;
    }
  }
  // sums and stores: rows r0 and r0 + 64
  const int r0 = tid >> 2, c0 = (tid & 3) * 4;
  const bool real = col0 + c0 < p.dv;
  for (int i = 1; i < cuts; ++i) {
    const int64_t at_i = at(i) * size + static_cast<int64_t>(r0) * p.dv + col0 + c0;
    float4 add[2];  // B_i, on its way while M_i is used
#pragma unroll
    for (int y = 0; y < 2; ++y)
      add[y] = real && r0 + 64 * y < p.dk
                   ? *reinterpret_cast<const float4*>(a.seg_b + at_i + 64 * y * p.dv)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    if (i + 1 < cuts) {
      fetch(i + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const int rr = (tid >> 2) & 15, part = tid >> 6;
    const float* m = M + (i & 1) * 128 * kLdCut + rr * kLdCut;
    const float* s = S + ((i & 1) ^ 1) * 128 * kCutCols + c0;
    float* next = S + (i & 1) * 128 * kCutCols;
    float acc[8][4] = {};
#pragma unroll 2
    for (int k = 4 * part; k < p.dk; k += 16) {
      float4 u[8], v[4];
#pragma unroll
      for (int y = 0; y < 8; ++y)
        u[y] = *reinterpret_cast<const float4*>(m + 16 * y * kLdCut + k);
#pragma unroll
      for (int z = 0; z < 4; ++z) v[z] = *reinterpret_cast<const float4*>(s + (k + z) * kCutCols);
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float f = z == 0 ? u[y].x : z == 1 ? u[y].y : z == 2 ? u[y].z : u[y].w;
          acc[y][0] = fmaf(f, v[z].x, acc[y][0]);
          acc[y][1] = fmaf(f, v[z].y, acc[y][1]);
          acc[y][2] = fmaf(f, v[z].z, acc[y][2]);
          acc[y][3] = fmaf(f, v[z].w, acc[y][3]);
        }
    }
#pragma unroll
    for (int y = 0; y < 8; ++y)
      *reinterpret_cast<float4*>(parts + (part * 128 + rr + 16 * y) * kCutCols + c0) =
          make_float4(acc[y][0], acc[y][1], acc[y][2], acc[y][3]);
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; ++y)
      if (r0 + 64 * y < p.dk) {
        float4 v = add[y];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 o = *reinterpret_cast<const float4*>(
              parts + (x * 128 + r0 + 64 * y) * kCutCols + c0);
          v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        if (real) *reinterpret_cast<float4*>(a.seg_s + at_i + 64 * y * p.dv) = v;
        *reinterpret_cast<float4*>(next + (r0 + 64 * y) * kCutCols + c0) = v;
      }
    __syncthreads();
  }
}

template <int DK, int MODE>
cudaError_t launch(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a,
                   cudaStream_t stream) {
  cudaError_t e = need_regs<seq_kernel<DK, MODE>>(kLaunchRegs);
  if (e != cudaSuccess) return e;
  e = allow_smem<seq_kernel<DK, MODE>>(seq_smem<DK>());
  if (e != cudaSuccess) return e;
  const int segs = MODE == kStates ? a.seg.count - 1 : (MODE == kForward ? a.seg.count : 1);
  const int seqs = p.N + (p.cu_seqlens ? 2 : 0);
  const int cols = (p.dv + kCols - 1) / kCols + (MODE == kStates ? 1 : 0);
  seq_kernel<DK, MODE>
      <<<dim3(seqs * segs * p.Hv, cols), kThreads, seq_smem<DK>(), stream>>>(p, m, a);
  return cudaGetLastError();
}

template <int DK>
cudaError_t forward(const gsa_delta_t& p, const DeltaMaps& m, const SeqArgs& a,
                    cudaStream_t stream) {
  if (a.seg.count > 1) {
    cudaError_t e = launch<DK, kStates>(p, m, a, stream);
    if (e != cudaSuccess) return e;
    if ((e = allow_smem<cut_kernel>(kCutSmem)) != cudaSuccess) return e;
    cut_kernel<<<dim3(p.N, p.Hv, (p.dv + kCutCols - 1) / kCutCols), kCutThreads, kCutSmem,
                 stream>>>(p, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  return launch<DK, kForward>(p, m, a, stream);
}

}  // namespace

// Of all cuts the one whose blocks take the least time, counted in rounds of 148
// blocks: a chunk takes 2.9 us in the full pass, and 1.4 us more where all SMs read
// at once; 2.8 us in the one for M and B (128 columns each of B and M, all segments
// but the last); a step between segments 3.2 us.  16 heads of 16384 tokens take 0.76
// ms uncut and 0.32 ms in nine segments; 64 heads of 4096 0.23 ms, and 0.24 in two.
// The times are those of 128 x 128 and stand for all dk and dv; narrower states were not
// measured.  Uncut stay packed batches, whose lengths the host does not know, and the
// backward pass.
Segments segments_of(const gsa_delta_t& p) {
  if (p.cu_seqlens || p.T < 16 * kChunk) return {1, p.T / kChunk + 1};
  const int chunks = (p.T + kChunk - 1) / kChunk;
  const int64_t cols = (p.dv + kCols - 1) / kCols, heads = static_cast<int64_t>(p.N) * p.Hv;
  auto rounds = [](int64_t blocks) { return static_cast<double>((blocks + 147) / 148); };
  Segments best = {1, chunks};
  auto full = [&](int64_t blocks) {
    return rounds(blocks) * (2.9 + 1.4 * (blocks < 148 ? blocks / 148.0 : 1.0));
  };
  double least = chunks * full(heads * cols);
  for (int n = 2; n <= 16 && heads * n < 2048; ++n) {
    const int each = (chunks + n - 1) / n, count = (chunks + each - 1) / each;
    if (each < 8) break;
    const double time = each * (2.8 * rounds(heads * (cols + 1) * (count - 1)) +
                                full(heads * cols * count)) +
                        3.2 * count + 10.0;
    if (time < least) {
      least = time;
      best = {count, each};
    }
  }
  return best;
}

cudaError_t launch_forward(const gsa_delta_t& p, const DeltaMaps& m, SeqArgs a, float* cuts,
                           cudaStream_t stream) {
  a.seg = segments_of(p);
  const int64_t n = static_cast<int64_t>(p.N) * (a.seg.count - 1) * p.Hv;
  a.seg_b = cuts;
  a.seg_s = a.seg_b + n * p.dk * p.dv;
  a.seg_m = a.seg_s + n * p.dk * p.dv;
  return p.dk <= 64 ? forward<64>(p, m, a, stream) : forward<128>(p, m, a, stream);
}
cudaError_t launch_backward(const gsa_delta_t& p, const DeltaMaps& m, SeqArgs a,
                            cudaStream_t stream) {
  a.seg = {1, 0};
  return p.dk <= 64 ? launch<64, kBackward>(p, m, a, stream)
                    : launch<128, kBackward>(p, m, a, stream);
}

}  // namespace delta
}  // namespace gsa
