// delta_tc.cuh — tcgen05 pieces of the gated delta rule's kernels: left operands
// from tensor memory, 16-column stores, and the operand descriptors of the tiles
// that its kernels keep in shared memory.
#pragma once

#include "delta_common.cuh"

namespace gsa {
namespace delta {

using bf16 = __nv_bfloat16;

// Tiles of 64 rows x 64 columns of bf16 (128 bytes a row) with 128-byte swizzle,
// as TMA writes them; a wider matrix is one such tile after the other.
constexpr uint32_t kTile = 64 * 128;

// tcgen05 operations issued by one elected lane of a whole warp.  The operands are
// then uniform to the compiler: 16 products of 128 x 64 x 16 take 650 cycles from
// the first issue to their barrier, against 970 from inside an `if (lane == 0)`,
// where every operand is moved to a uniform register on its own.
// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16 (bf16 in, fp32 accumulators).
__device__ __forceinline__ void warp_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// ... with A in shared memory.
__device__ __forceinline__ void warp_mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on `bar` when the operations that this warp's elected lane issued are done.
__device__ __forceinline__ void warp_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(
          smem_u32(bar))
      : "memory");
}
// Waits for this thread's tensor-memory loads; the registers they fill are named, so
// that no use of them moves in front of the wait.
template <typename... R>
__device__ __forceinline__ void tc_wait_ld(R&... r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  auto hold = [](auto& a) {
#pragma unroll
    for (uint32_t& x : a) asm volatile("" : "+r"(x));
  };
  (hold(r), ...);
}
// Store 16 consecutive 32-bit columns of this thread's lane (32x32b shape).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Tiles of `step` bytes for 64 columns.  Rows are the outer dimension (M or N) and
// columns contracted: columns 16 ks .. 16 ks + 15.
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int ks, uint32_t step = kTile) {
  return sdesc_sw128(tile + (ks >> 2) * step + (ks & 3) * 32, 16, 1024);
}
// Rows are contracted and columns are the outer dimension: rows 16 ks .. 16 ks + 15.
__device__ __forceinline__ uint64_t desc_cols(uint32_t tile, int ks, uint32_t step = kTile) {
  return sdesc_sw128(tile + ks * 2048, step, 1024);
}

// x, y as hi + lo pairs of bf16.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  const uint64_t rest = f2_fma((static_cast<uint64_t>(hi & 0xFFFF0000u) << 32) | (hi << 16),
                               f2_pack(-1.f, -1.f), f2_pack(x, y));
  lo = pack_bf16x2(f2_lo(rest), f2_hi(rest));
}
// e^x on the MUFU: 2^-22 of the value, and x log2(e) rounded once: 2^-24 |x|.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return fast_ex2(x * kLog2e); }
__device__ __forceinline__ float lo_of(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float hi_of(uint32_t r) { return __uint_as_float(r & 0xFFFF0000u); }

__device__ __forceinline__ const bf16* rows_at(const void* base, const int64_t (&stride)[3], int b,
                                               int64_t row, int h) {
  return static_cast<const bf16*>(base) + b * stride[0] + row * stride[1] + h * stride[2];
}
// 64 rows of `width` (<= limit real) columns into swizzled tiles, zeros past
// `len` and `limit`; by `threads` threads from thread `t` on.
__device__ __forceinline__ void copy_rows(uint32_t dst, const bf16* src, int64_t stride, int len,
                                          int width, int limit, int t, int threads,
                                          uint32_t step = kTile) {
  const int pieces = width >> 3;
  for (int i = t; i < kChunk * pieces; i += threads) {
    const int r = i / pieces, c = i % pieces;
    const bool real = r < len && c * 8 < limit;
    cp16(dst + (c >> 3) * step + sw128_offset(r, c & 7), real ? src + r * stride + c * 8 : src,
         real);
  }
}
__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* map, int x, int h,
                                              int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

// A split of registers by setmaxnreg is valid only for the count at launch that it
// was written for: with fewer, its `inc` would wait for registers that do not exist.
template <auto Kernel>
cudaError_t need_regs(int expected) {
  static std::atomic<int> regs{0};
  int r = regs.load(std::memory_order_acquire);
  if (r == 0) {
    cudaFuncAttributes f;
    const cudaError_t e = cudaFuncGetAttributes(&f, Kernel);
    if (e != cudaSuccess) return e;
    r = f.numRegs;
    regs.store(r, std::memory_order_release);
  }
  return r == expected ? cudaSuccess : cudaErrorNotSupported;
}

// ---------------------------------------------------------------- workspace
// For each chunk and value head, T and P as pairs of swizzled tiles with the
// decays that go with them.
struct __align__(16) Block {
  unsigned char t_hi[kTile], t_lo[kTile];
  Gates gates;
  unsigned char p_hi[kTile], p_lo[kTile];
};
constexpr int kTBytes = 2 * static_cast<int>(kTile + sizeof(Gates) / 2);  // T and the gates
constexpr int kPBytes = 2 * static_cast<int>(kTile);
static_assert(sizeof(Gates) == 2048 && sizeof(Block) == kTBytes + kPBytes, "block");

__host__ __device__ inline int padded_dk(int dk) { return dk <= 64 ? 64 : 128; }
// Rows of the images below: the value columns, rounded up to whole tiles.
__host__ __device__ inline int padded_dv(int dv) { return (dv + 63) / 64 * 64; }

// Kept for, or left by, the backward pass, in bf16, for each chunk and value
// head: N or dY as [8 groups of 8 tokens][padded dv][8], S0 or dS1 as
// [padded dk / 8][padded dv][8].  16 bytes are 8 neighbours of the dimension that
// is not contracted later, one column of the state after the other: what a thread
// with a column in its registers writes whole, and what tcgen05 reads unswizzled.
struct Saved {
  Block* blocks;
  bf16* news;
  bf16* states;
};
struct Scratch {
  bf16* back;
  bf16* states;
};
inline int64_t news_elems(const gsa_delta_t& p) {
  return static_cast<int64_t>(kChunk) * padded_dv(p.dv);
}
inline int64_t state_elems(const gsa_delta_t& p) {
  return static_cast<int64_t>(padded_dk(p.dk)) * padded_dv(p.dv);
}
inline Saved saved_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  char* c = static_cast<char*>(ws) + table_bytes(p);
  Saved s;
  s.blocks = reinterpret_cast<Block*>(c);
  s.news = reinterpret_cast<bf16*>(c + n * static_cast<int64_t>(sizeof(Block)));
  s.states = s.news + n * news_elems(p);
  return s;
}
inline Scratch scratch_at(const gsa_delta_t& p, void* ws) {
  const int64_t n = max_chunks(p) * p.Hv;
  bf16* b = static_cast<bf16*>(ws);
  return {b, b + n * news_elems(p)};
}

// Long sequences with few heads are cut into segments that run side by side
// (forwards).  What a segment does to a state is affine, S -> M S + B: a first pass
// finds M and B of every segment but the last, a small kernel goes through them from
// segment to segment, and a second pass runs all segments from their states.
struct Segments {
  int count;   // segments a sequence, 1: uncut
  int chunks;  // chunks a segment (the last may have fewer)
};
Segments segments_of(const gsa_delta_t& p);
inline int64_t segment_floats(const gsa_delta_t& p) {
  const int64_t cuts = static_cast<int64_t>(p.N) * (segments_of(p).count - 1) * p.Hv;
  return cuts * p.dk * (2 * static_cast<int64_t>(p.dv) + p.dk);  // B, S, M
}

// Launches of the parts (delta_seq.cu, delta_grad.cu).
struct SeqArgs {
  Table table;
  const Block* blocks;
  // forwards: out o, state0 initial, state1 final.  Backwards: out dv, state0
  // dfinal, state1 dinitial, in dO (contiguous).
  const void* in;        // backwards: may be nullptr
  void* out;
  const float* state0;   // may be nullptr: zeros
  float* state1;         // may be nullptr
  bf16* rows;            // N (forwards; nullptr: inference) or dY
  bf16* states;          // S0 or dS1
  int* err;
  Segments seg;
  float *seg_b, *seg_s, *seg_m;  // [sequence][cut][head]: B, S [dk][dv], M [dk][dk]
};
// Forwards: `cuts` holds segment_floats() floats, 16-byte aligned.
cudaError_t launch_forward(const gsa_delta_t& p, const DeltaMaps& m, SeqArgs a, float* cuts,
                           cudaStream_t stream);
cudaError_t launch_backward(const gsa_delta_t& p, const DeltaMaps& m, SeqArgs a,
                            cudaStream_t stream);
// maps: q, k, v; more.v: dO.
cudaError_t launch_grad(const gsa_delta_t& p, const DeltaMaps& maps, const DeltaMaps& more,
                        const DeltaGrads& g, const Saved& s, const Scratch& r, const Table& t,
                        int* err, cudaStream_t stream);

}  // namespace delta
}  // namespace gsa
