// delta_grad.cu — gradients of the gated delta rule that contract over the
// state's columns, chunk by chunk, on tcgen05 (bf16 inputs).
//
// The two sequential passes left S0, N (forwards) and dS1, dY (backwards) of
// every chunk.  With A = scale tril(dO N^T) D, M = -strict(dY N^T) beta D and
// D_ij = e^{c_i - c_j}:
//   dQ = scale e^c dO S0^T + A K,
//   dK = -e^c beta dY S0^T + e^{c_64 - c} N dS1^T + A^T Q + (M + M^T) K,
//   dbeta_i = dY_i.(V_i - e^{c_i} S0^T k_i) - sum_{j<i} (dY N^T)_ij D_ij k_i.k_j,
//   dg_t = what the decays between tokens before t and from t on carry:
//          sum_{i>=t} (scale e^c q.(dO S0^T) - e^c beta k.(dY S0^T) + E rows - E columns)_i
//          + sum_{i<t} e^{c_64 - c_i} k_i.(N dS1^T)_i + e^{c_64} <S0, dS1>,
//   E = A (q.k) + M (k.k), element by element.
//
// A block takes chunks and key heads in turn and the value heads that share the
// key head one after the other, so that their gradients add up in one order.  All
// products have 128 rows: channels (dO S0^T and its like, transposed: S0's image is
// the left operand), or N's and dY's tokens on top of one another.  The factors
// are bf16, rounded once, as dQ and dK are in the end (off by about 3e-3 together).  dg
// and dbeta are sums of products of the same factors, also where the gates are fp32 (about
// 2e-3 then).  About 210 KB a chunk and head of 128 x 128 come and go, the next
// head's while this one's elements are worked on: 64 heads of 4096 tokens take 285 us, 130 for the bytes.  Bound by the chain of copies,
// products and passes within a head (a block an SM: its operands take 202 KB of shared
// memory; 33% of the cycles issue, 14% multiply; 248 bytes of registers spill).
#include "delta_tc.cuh"

namespace gsa {
namespace delta {
namespace {

constexpr int kComputeWarps = 8;
constexpr int kThreads = 384;  // whole warpgroups: two warps idle
// Registers: 384 x 168 at launch = 256 x 216 (computing) + 128 x 72 (the others).
constexpr int kLaunchRegs = 168, kComputeRegs = 216, kOtherRegs = 72;
static_assert(256 * kComputeRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 512;

// Shared memory.  K, Q and K again, 64 channels at a time, so that [K; Q] and [Q;
// K] are 128 rows each; images of 128 columns (S0, dS1: channels, N and dY: tokens
// in groups of 8); dO and V as rows; A^T and M.
constexpr int kKqkBytes = 3 * static_cast<int>(kTile);  // for 64 channels
constexpr int kGroup = 128 * 16;                        // 8 channels or tokens of an image
constexpr int kOffS0 = 2 * kKqkBytes;
constexpr int kOffS1 = kOffS0 + 16 * kGroup;
constexpr int kOffN = kOffS1 + 16 * kGroup;
constexpr int kOffY = kOffN + 8 * kGroup;
constexpr int kOffD = kOffY + 8 * kGroup;
constexpr int kOffV = kOffD + 2 * static_cast<int>(kTile);
constexpr int kOffA = kOffV + 2 * static_cast<int>(kTile);
constexpr int kOffM = kOffA + static_cast<int>(kTile);
constexpr int kOffG = kOffM + static_cast<int>(kTile);  // gates, of two heads in turn
constexpr int kSmem = kOffG + 2 * static_cast<int>(sizeof(Gates)) + 1024;
// The gradients of 64 tokens leave by way of A's and M's place, 256 bytes a token.
constexpr int kRowBytes = 256;

enum : uint32_t {
  kTo = 0,     // (dO S0^T)^T [channels][tokens]
  kTy = 64,    // (dY S0^T)^T
  kTn = 128,   // (N dS1^T)^T
  kPd = 192,   // [N; dY] dO^T: rows 0 .. 63 are (dO N^T)^T; then (A K)^T
  kPn = 256,   // [N; dY] N^T: rows 64 .. 127 are dY N^T; then A^T Q + (M + M^T) K, transposed
  kPv = 320,   // [N; dY] V^T: rows 64 .. 127 are dY V^T
  kKq = 384,   // [K; Q] Q^T: rows 0 .. 63 are k_j.q_i
  kKk = 448,   // [Q; K] K^T: rows 64 .. 127 are k_i.k_j
};

struct GradArgs {
  Table table;
  const Block* blocks;
  const bf16* news;
  const bf16* states;
  const bf16* back;
  const bf16* dstates;
  const void* dout;  // contiguous; may be nullptr
  void *dq, *dk, *dv, *dg, *dbeta;
  int64_t items;     // chunks x key heads
  int* err;
};

struct Bars {
  uint64_t full_kq, empty_kq, full_h, empty_h;
  uint64_t ph1_full, ph2_ready, ph2_full, x_read, drain;
  uint64_t meet;  // the computing warps
  uint32_t tmem;
  int abort;
};

// Unswizzled image: 16 bytes are 8 neighbours of the outer dimension, the
// contracted one steps by 16 bytes; 16 of it from 16 ks on.
__device__ __forceinline__ uint64_t desc_image(uint32_t image, int ks) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>(((image + ks * 256) >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128 >> 4) << 16;
  d |= static_cast<uint64_t>(kGroup >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
// [K; Q] (or, from Q on, [Q; K]): 128 rows, channels 16 ks on contracted.
__device__ __forceinline__ uint64_t desc_kq(uint32_t tile, int ks) {
  return desc_rows(tile, ks, kKqkBytes);
}
// K^T or Q^T: channels are the rows, tokens 16 ks on contracted.
__device__ __forceinline__ uint64_t desc_kt(uint32_t tile, int ks) {
  return desc_cols(tile, ks, kKqkBytes);
}

// v[i] summed over the warp's lanes; lane l gets the sum of v[l].
__device__ __forceinline__ float fold_lanes(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int i = 0; i < m; ++i) {
      const float give = up ? v[i] : v[i + m], keep = up ? v[i + m] : v[i];
      v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, m);
    }
  }
  return v[0];
}

template <int DK>
__device__ __forceinline__ void produce(const gsa_delta_t& p, const DeltaMaps& maps,
                                        const DeltaMaps& more, const GradArgs& a,
                                        unsigned char* smem, Bars& bars) {
  const int lane = threadIdx.x & 31, group = p.Hv / p.Hk, rows = padded_dv(p.dv);
  int items = 0, loads = 0, heads = 0;
  bool ok = true;
  for (int64_t x = blockIdx.x; ok && x < a.items; x += gridDim.x) {
    const int chunk = static_cast<int>(x / p.Hk), hk = static_cast<int>(x % p.Hk);
    const Chunk c = chunk_at(p, a.table, chunk);
    if (!c.valid || c.gap) continue;
    const bool whole = c.len == kChunk || !p.cu_seqlens;
    // K and Q come behind the first head's operands, whose place is free earlier
    auto load_kq = [&] {
      if (!mbar_wait_warp(&bars.empty_kq, (items & 1) ^ 1, a.err, &bars.abort)) return false;
      if (!whole) {
        for (int i = 0; i < DK / 64; ++i) {
          const uint32_t t = smem_u32(smem) + i * kKqkBytes;
          const bf16* k = rows_at(p.k, p.k_stride, c.b, c.begin, hk) + 64 * i;
          copy_rows(t, k, p.k_stride[1], c.len, 64, p.dk - 64 * i, lane, 32);
          copy_rows(t + 2 * kTile, k, p.k_stride[1], c.len, 64, p.dk - 64 * i, lane, 32);
          copy_rows(t + kTile, rows_at(p.q, p.q_stride, c.b, c.begin, hk) + 64 * i, p.q_stride[1],
                    c.len, 64, p.dk - 64 * i, lane, 32);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.full_kq);
      } else if (lane == 0) {
        mbar_arrive_expect_tx(&bars.full_kq, DK / 64 * kKqkBytes);
        for (int i = 0; i < DK / 64; ++i) {
          unsigned char* t = smem + i * kKqkBytes;
          tma_load_rows(t, &maps.k, 64 * i, hk, c.begin, c.b, &bars.full_kq);
          tma_load_rows(t + kTile, &maps.q, 64 * i, hk, c.begin, c.b, &bars.full_kq);
          tma_load_rows(t + 2 * kTile, &maps.k, 64 * i, hk, c.begin, c.b, &bars.full_kq);
        }
      }
      ++items;
      return true;
    };
    for (int hv = hk * group; ok && hv < (hk + 1) * group; ++hv, ++heads) {
      const int64_t slot = static_cast<int64_t>(chunk) * p.Hv + hv;
      for (int col0 = 0; col0 < p.dv; col0 += 128) {
        ok = mbar_wait_warp(&bars.empty_h, (loads & 1) ^ 1, a.err, &bars.abort);
        if (!ok) break;
        const uint32_t wide = min(128, rows - col0) * 16;
        const bool tma_d = whole && a.dout != nullptr, tma_v = whole;
        if (!tma_d || !tma_v) {
          const int64_t stride = static_cast<int64_t>(p.Hv) * p.dv;
          if (!tma_d)
            copy_rows(smem_u32(smem) + kOffD,
                      a.dout ? static_cast<const bf16*>(a.dout) +
                                   (static_cast<int64_t>(c.b) * p.T + c.begin) * stride +
                                   hv * p.dv + col0
                             : static_cast<const bf16*>(p.k),
                      stride, a.dout ? c.len : 0, 128, p.dv - col0, lane, 32);
          if (!tma_v)
            copy_rows(smem_u32(smem) + kOffV,
                      rows_at(p.v, p.v_stride, c.b, c.begin, hv) + col0, p.v_stride[1], c.len, 128,
                      p.dv - col0, lane, 32);
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.full_h, (col0 ? 0 : sizeof(Gates)) +
                                                  (2 * (DK / 8) + 16) * wide +
                                                  (int(tma_d) + int(tma_v)) * 2 * kTile);
          if (col0 == 0)
            bulk_load(smem + kOffG + (heads & 1) * sizeof(Gates), &a.blocks[slot].gates,
                      sizeof(Gates), &bars.full_h);
          for (int i = 0; i < 2; ++i) {
            if (tma_d)
              tma_load_rows(smem + kOffD + i * kTile, &more.v, col0 + 64 * i, hv, c.begin, c.b,
                            &bars.full_h);
            if (tma_v)
              tma_load_rows(smem + kOffV + i * kTile, &maps.v, col0 + 64 * i, hv, c.begin, c.b,
                            &bars.full_h);
          }
        }
        __syncwarp();
        // groups of 8 channels or tokens: a copy each
        const int64_t step = static_cast<int64_t>(rows) * 8, at = static_cast<int64_t>(col0) * 8;
        if (lane < DK / 8) {
          const int64_t from = slot * DK * rows + lane * step + at;
          bulk_load(smem + kOffS0 + lane * kGroup, a.states + from, wide, &bars.full_h);
          bulk_load(smem + kOffS1 + lane * kGroup, a.dstates + from, wide, &bars.full_h);
        }
        if (lane < 8) {
          const int64_t from = slot * kChunk * rows + lane * step + at;
          bulk_load(smem + kOffN + lane * kGroup, a.news + from, wide, &bars.full_h);
          bulk_load(smem + kOffY + lane * kGroup, a.back + from, wide, &bars.full_h);
        }
        ++loads;
        __syncwarp();
        if (hv == hk * group && col0 == 0 && !(ok = load_kq())) break;
      }
    }
  }
  if (!ok) {  // gave up: no copy of ours may outlive the block
    if (items) mbar_wait_drain(&bars.full_kq, (items - 1) & 1, kWaitLimitCycles);
    if (loads) mbar_wait_drain(&bars.full_h, (loads - 1) & 1, kWaitLimitCycles);
  }
}

template <int DK>
__device__ __forceinline__ void issue(const gsa_delta_t& p, const GradArgs& a, uint32_t smem,
                                      Bars& bars) {
  const uint32_t tm = __shfl_sync(0xFFFFFFFFu, bars.tmem, 0), K = smem, Q = smem + kTile;
  const uint32_t S0 = smem + kOffS0, S1 = smem + kOffS1, N = smem + kOffN, Y = smem + kOffY;
  const uint32_t D = smem + kOffD, V = smem + kOffV, A = smem + kOffA, M = smem + kOffM;
  constexpr uint32_t kRR = idesc_bf16_f32(128, 64, 0, 0), kCR = idesc_bf16_f32(128, 64, 1, 0);
  constexpr uint32_t kCC = idesc_bf16_f32(128, 64, 1, 1);
  const int group = p.Hv / p.Hk, rows = padded_dv(p.dv);
  int items = 0, loads = 0, heads = 0;
  bool ok = true;
  auto until = [&](uint64_t* bar, int parity) {
    ok = ok && mbar_wait_warp(bar, parity & 1, a.err, &bars.abort);
    tc_fence_after();
    return ok;
  };
  for (int64_t x = blockIdx.x; ok && x < a.items; x += gridDim.x) {
    const Chunk c = chunk_at(p, a.table, static_cast<int>(x / p.Hk));
    if (!c.valid || c.gap) continue;
    for (int h = 0; ok && h < group; ++h, ++heads) {
      if (h == 0) {
        if (!until(&bars.full_kq, items)) break;
#pragma unroll
        for (int ks = 0; ks < DK / 16; ++ks) {
          warp_mma_ss(tm + kKq, desc_kq(K, ks), desc_kq(Q, ks), kRR, ks > 0);
          warp_mma_ss(tm + kKk, desc_kq(Q, ks), desc_kq(K, ks), kRR, ks > 0);
        }
      }
      if (heads > 0 && !until(&bars.x_read, heads - 1)) break;
      for (int col0 = 0; col0 < p.dv; col0 += 128, ++loads) {
        if (!until(&bars.full_h, loads)) break;
        const int steps = min(128, rows - col0) / 16;
#pragma unroll 4
        for (int ks = 0; ks < steps; ++ks) {
          const uint32_t on = col0 > 0 || ks > 0;
          const uint64_t s0 = desc_image(S0, ks), n = desc_image(N, ks);
          warp_mma_ss(tm + kTo, s0, desc_rows(D, ks), kCR, on);
          warp_mma_ss(tm + kTy, s0, desc_image(Y, ks), kCC, on);
          warp_mma_ss(tm + kTn, desc_image(S1, ks), n, kCC, on);
          warp_mma_ss(tm + kPd, n, desc_rows(D, ks), kCR, on);
          warp_mma_ss(tm + kPn, n, n, kCC, on);
          warp_mma_ss(tm + kPv, n, desc_rows(V, ks), kCR, on);
        }
        warp_commit(&bars.empty_h);
      }
      if (!ok) break;
      warp_commit(&bars.ph1_full);
      if (!until(&bars.ph2_ready, heads)) break;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        warp_mma_ss(tm + kPd, desc_kt(K, ks), desc_cols(A, ks), kCC, ks > 0);
        warp_mma_ss(tm + kPn, desc_kt(Q, ks), desc_rows(A, ks), kCR, ks > 0);
        warp_mma_ss(tm + kPn, desc_kt(K, ks), desc_cols(M, ks), kCC, 1);
        warp_mma_ss(tm + kPn, desc_kt(K, ks), desc_rows(M, ks), kCR, 1);
      }
      warp_commit(&bars.ph2_full);
      if (h == group - 1) warp_commit(&bars.empty_kq);
    }
    ++items;
  }
  warp_commit(&bars.drain);
  mbar_wait_drain(&bars.drain, 0, kWaitLimitCycles);
  __syncwarp();
}

struct Sums {  // per token; by quadrant of lanes where several warps have a part
  float qo[4][kChunk], ky[4][kChunk], kn[4][kChunk];  // q.tO, k.tY, k.tN
  float row_x[2][kChunk], col_x[2][kChunk];           // E from A: rows (by quadrant), columns (by half)
  float row_m[2][kChunk], col_m[2][kChunk];           // E from M: rows (by half), columns (by quadrant)
  float low[2][kChunk];                               // sum_j l_ij k_i.k_j (by half)
  float yv[kChunk];                                   // dY_i.V_i
  float cross[2][kComputeWarps];                      // <S0, dS1>, of two heads in turn
};

template <int DK>
__device__ __forceinline__ void compute(const gsa_delta_t& p, const GradArgs& a,
                                        unsigned char* smem, Bars& bars, Sums& sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = warp & 3, half = warp >> 2;
  const int row = 32 * quad + lane, tid = threadIdx.x, t0 = 32 * half;
  const uint32_t tm = bars.tmem + (static_cast<uint32_t>(32 * quad) << 16);
  const int group = p.Hv / p.Hk, rows = padded_dv(p.dv);
  const bool gate16 = p.gate_dtype == GSA_DTYPE_BF16;
  const int64_t qk_step = static_cast<int64_t>(p.Hk) * p.dk;
  int items = 0, loads = 0, heads = 0, meets = 0;
  auto until = [&](uint64_t* bar, int parity) {
    const bool ok = mbar_wait_warp(bar, parity & 1, a.err, &bars.abort);
    tc_fence_after();
    return ok;
  };
  auto signal = [&](uint64_t* bar) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  for (int64_t x = blockIdx.x; x < a.items; x += gridDim.x) {
    const int chunk = static_cast<int>(x / p.Hk), hk = static_cast<int>(x % p.Hk);
    const Chunk c = chunk_at(p, a.table, chunk);
    if (!c.valid) continue;
    const int64_t row0 = static_cast<int64_t>(c.b) * p.T + c.begin;
    bf16* dq_out = static_cast<bf16*>(a.dq) + (row0 * p.Hk + hk) * p.dk;
    bf16* dk_out = static_cast<bf16*>(a.dk) + (row0 * p.Hk + hk) * p.dk;
    if (c.gap) {
      for (int i = tid; i < c.len * p.dk / 8; i += 256) {
        const int r = i / (p.dk / 8), cc = i % (p.dk / 8) * 8;
        *reinterpret_cast<uint4*>(dq_out + r * qk_step + cc) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dk_out + r * qk_step + cc) = make_uint4(0, 0, 0, 0);
      }
      const int wide = group * p.dv / 8;
      for (int i = tid; i < c.len * wide; i += 256)
        *reinterpret_cast<uint4*>(static_cast<bf16*>(a.dv) +
                                  ((row0 + i / wide) * p.Hv + hk * group) * p.dv + i % wide * 8) =
            make_uint4(0, 0, 0, 0);
      for (int i = tid; i < c.len * group; i += 256) {
        const int64_t at = (row0 + i / group) * p.Hv + hk * group + i % group;
        store_gate(a.dg, at, gate16, 0.f);
        store_gate(a.dbeta, at, gate16, 0.f);
      }
      continue;
    }
    if (!until(&bars.full_kq, items++)) return;
    float gq[32], gk[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) gq[i] = gk[i] = 0.f;
    for (int hv = hk * group; hv < (hk + 1) * group; ++hv, ++heads) {
      const Gates& gates =
          *reinterpret_cast<const Gates*>(smem + kOffG + (heads & 1) * sizeof(Gates));
      // <S0, dS1>: a column and every second group of 8 channels a thread
      float cross = 0.f;
      for (int col0 = 0; col0 < p.dv; col0 += 128, ++loads) {
        if (!until(&bars.full_h, loads)) return;
        if (col0 + (tid & 127) < rows) {
          const unsigned char* at = smem + (tid >> 7) * kGroup + (tid & 127) * 16;
#pragma unroll
          for (int i = 0; i < DK / 16; ++i) {
            const uint4 u = *reinterpret_cast<const uint4*>(at + kOffS0 + 2 * i * kGroup);
            const uint4 w = *reinterpret_cast<const uint4*>(at + kOffS1 + 2 * i * kGroup);
            const uint32_t us[4] = {u.x, u.y, u.z, u.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              cross = fmaf(lo_of(us[e]), lo_of(ws[e]), cross);
              cross = fmaf(hi_of(us[e]), hi_of(ws[e]), cross);
            }
          }
        }
        signal(&bars.empty_h);
      }
#pragma unroll
      for (int m = 16; m; m >>= 1) cross += __shfl_xor_sync(0xFFFFFFFFu, cross, m);
      if (lane == 0) sum.cross[heads & 1][warp] = cross;

      if (!until(&bars.ph1_full, heads)) return;
      uint32_t r[32], u[32];
      float e[32];
      const int own = row & 63;
      const float hi0 = gates.hi[own], lo0 = gates.lo[own], beta0 = gates.beta[own];
      float own_sum = 0.f;
      if (quad < 2) {  // A^T: lanes are tokens j, columns i >= j
        tmem_ld32(tm + kPd + t0, r);
        tmem_ld32(tm + kKq + t0, u);
        tc_wait_ld(r, u);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 h = *reinterpret_cast<const float4*>(gates.hi + t0 + i);
          const float4 o = *reinterpret_cast<const float4*>(gates.lo + t0 + i);
          const float hs[4] = {h.x, h.y, h.z, h.w}, os[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float w = p.scale * exp_of((hs[f] - hi0) + (os[f] - lo0));
            const float x = t0 + i + f >= own ? w * __uint_as_float(r[i + f]) : 0.f;
            e[i + f] = t0 + i + f >= own ? x * __uint_as_float(u[i + f]) : 0.f;
            own_sum += e[i + f];
            r[i + f] = __float_as_uint(x);
          }
        }
      } else {  // M: lanes are tokens i, columns j < i
        float low = 0.f;
        tmem_ld32(tm + kPn + t0, r);
        tmem_ld32(tm + kKk + t0, u);
        tc_wait_ld(r, u);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 h = *reinterpret_cast<const float4*>(gates.hi + t0 + i);
          const float4 o = *reinterpret_cast<const float4*>(gates.lo + t0 + i);
          const float hs[4] = {h.x, h.y, h.z, h.w}, os[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const bool in = t0 + i + f < own;
            const float w = exp_of((hi0 - hs[f]) + (lo0 - os[f]));
            const float l = in ? -w * __uint_as_float(r[i + f]) : 0.f;
            const float dot = in ? __uint_as_float(u[i + f]) : 0.f;
            low = fmaf(l, dot, low);
            e[i + f] = l * beta0 * dot;
            own_sum += e[i + f];
            r[i + f] = __float_as_uint(l * beta0);
          }
        }
        sum.low[half][own] = low;
      }
      {
        unsigned char* tile = smem + (quad < 2 ? kOffA : kOffM);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int f = 0; f < 4; ++f)
            x[f] = pack_bf16x2(__uint_as_float(r[8 * i + 2 * f]),
                               __uint_as_float(r[8 * i + 2 * f + 1]));
          *reinterpret_cast<uint4*>(tile + sw128_offset(own, 4 * half + i)) =
              make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      fence_proxy_async_smem();  // A^T and M are read by the products
      signal(&bars.ph2_ready);
      const float across = fold_lanes(e);  // lane l: column t0 + l over this warp's rows
      if (quad < 2) {
        sum.col_x[half][own] = own_sum;
        sum.row_x[quad][t0 + lane] = across;
      } else {
        sum.row_m[half][own] = own_sum;
        sum.col_m[quad - 2][t0 + lane] = across;
        tmem_ld32(tm + kPv + t0, r);
        tc_wait_ld(r);
        float diag = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) diag = own == t0 + i ? __uint_as_float(r[i]) : diag;
        if ((own >> 5) == half) sum.yv[own] = diag;
      }
      // lanes are channels: what S0 and dS1 give, times q and k, over the channels; and
      // the gradients' part of it
      {
        const unsigned char* kt = smem + (row >> 6) * kKqkBytes + 2 * (row & 7);
        const int piece = (row & 63) >> 3;
        const bool real = row < DK;
        tmem_ld32(tm + kTo + t0, r);
        tc_wait_ld(r);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 g = *reinterpret_cast<const float4*>(gates.grown + t0 + i);
          const float gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float v = real ? __uint_as_float(r[i + f]) : 0.f;
            const float q = __uint_as_float(
                static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(
                    kt + kTile + sw128_offset(t0 + i + f, piece)))
                << 16);
            gq[i + f] = fmaf(p.scale * gs[f], v, gq[i + f]);
            e[i + f] = real ? v * q : 0.f;
          }
        }
        sum.qo[quad][t0 + lane] = fold_lanes(e);
        tmem_ld32(tm + kTy + t0, r);
        tmem_ld32(tm + kTn + t0, u);
        tc_wait_ld(r, u);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 g = *reinterpret_cast<const float4*>(gates.both + t0 + i);
          const float4 h = *reinterpret_cast<const float4*>(gates.left + t0 + i);
          const float gs[4] = {g.x, g.y, g.z, g.w}, hs[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float k =
                real ? __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(
                                           kt + sw128_offset(t0 + i + f, piece)))
                                       << 16)
                     : 0.f;
            const float y = real ? __uint_as_float(r[i + f]) : 0.f;
            const float n = real ? __uint_as_float(u[i + f]) : 0.f;
            gk[i + f] = fmaf(hs[f], n, fmaf(-gs[f], y, gk[i + f]));
            e[i + f] = y * k;
            u[i + f] = __float_as_uint(n * k);
          }
        }
        sum.ky[quad][t0 + lane] = fold_lanes(e);
#pragma unroll
        for (int i = 0; i < 32; ++i) e[i] = __uint_as_float(u[i]);
        sum.kn[quad][t0 + lane] = fold_lanes(e);
      }
      signal(&bars.meet);
      if (!until(&bars.meet, meets++)) return;
      if (warp == 0) {  // two neighbouring tokens a lane
        float rs[2], gs[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int t = 2 * lane + f;
          const float g = gates.grown[t];
          const float qo = (sum.qo[0][t] + sum.qo[1][t]) + (sum.qo[2][t] + sum.qo[3][t]);
          const float ky = (sum.ky[0][t] + sum.ky[1][t]) + (sum.ky[2][t] + sum.ky[3][t]);
          const float kn = (sum.kn[0][t] + sum.kn[1][t]) + (sum.kn[2][t] + sum.kn[3][t]);
          const float er = (sum.row_x[0][t] + sum.row_x[1][t]) + (sum.row_m[0][t] + sum.row_m[1][t]);
          const float ec = (sum.col_x[0][t] + sum.col_x[1][t]) + (sum.col_m[0][t] + sum.col_m[1][t]);
          rs[f] = p.scale * g * qo - gates.both[t] * ky + er - ec;
          gs[f] = gates.left[t] * kn;
          if (t < c.len)
            store_gate(a.dbeta, (row0 + t) * p.Hv + hv, gate16,
                       sum.yv[t] - g * ky + (sum.low[0][t] + sum.low[1][t]));
        }
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
        float whole = lane < kComputeWarps ? sum.cross[heads & 1][lane] : 0.f;
#pragma unroll
        for (int m = 16; m; m >>= 1) whole += __shfl_xor_sync(0xFFFFFFFFu, whole, m);
        whole *= gates.grown[kChunk - 1];
        const float dg0 = whole + before + (rs[0] + (rs[1] + after));
        const float dg1 = whole + (before + gs[0]) + (rs[1] + after);
        if (2 * lane < c.len) store_gate(a.dg, (row0 + 2 * lane) * p.Hv + hv, gate16, dg0);
        if (2 * lane + 1 < c.len)
          store_gate(a.dg, (row0 + 2 * lane + 1) * p.Hv + hv, gate16, dg1);
      }
      if (hv == (hk + 1) * group - 1) signal(&bars.empty_kq);  // q and k are read
      if (!until(&bars.ph2_full, heads)) return;
      tmem_ld32(tm + kPd + t0, r);
      tmem_ld32(tm + kPn + t0, u);
      tc_wait_ld(r, u);
      signal(&bars.x_read);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        gq[i] += __uint_as_float(r[i]);
        gk[i] += __uint_as_float(u[i]);
      }
    }
    // rows leave by way of shared memory
    unsigned char* mine = smem + kOffA + t0 * kRowBytes + 2 * row;
    const int piece = (tid & 15) * 8, first = tid >> 4;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const uint32_t x = z ? pack_bf16x2(gk[i], gk[i + 1]) : pack_bf16x2(gq[i], gq[i + 1]);
        *reinterpret_cast<uint16_t*>(mine + i * kRowBytes) = static_cast<uint16_t>(x);
        *reinterpret_cast<uint16_t*>(mine + (i + 1) * kRowBytes) = static_cast<uint16_t>(x >> 16);
      }
      signal(&bars.meet);
      if (!until(&bars.meet, meets++)) return;
      bf16* out = z ? dk_out : dq_out;
      if (piece < p.dk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (first + 16 * i < c.len)
            *reinterpret_cast<uint4*>(out + (first + 16 * i) * qk_step + piece) =
                *reinterpret_cast<const uint4*>(smem + kOffA + (first + 16 * i) * kRowBytes +
                                                2 * piece);
      signal(&bars.meet);
      if (!until(&bars.meet, meets++)) return;
    }
  }
}

// maps: q, k and v; more.v: dO.
template <int DK>
__global__ void __launch_bounds__(kThreads, 1)
    grad_kernel(const gsa_delta_t p, const __grid_constant__ DeltaMaps maps,
                const __grid_constant__ DeltaMaps more, const GradArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~1023ull);
  __shared__ Bars bars;
  __shared__ Sums sum;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    bars.abort = 0;
    mbar_init(&bars.full_kq, 1);
    mbar_init(&bars.empty_kq, 1 + kComputeWarps);
    mbar_init(&bars.full_h, 1);
    mbar_init(&bars.empty_h, 1 + kComputeWarps);
    mbar_init(&bars.ph1_full, 1);
    mbar_init(&bars.ph2_ready, kComputeWarps);
    mbar_init(&bars.ph2_full, 1);
    mbar_init(&bars.x_read, kComputeWarps);
    mbar_init(&bars.meet, kComputeWarps);
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
  if (warp < kComputeWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
    compute<DK>(p, a, smem, bars, sum);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kComputeWarps + 1)
      produce<DK>(p, maps, more, a, smem, bars);
    else if (warp == kComputeWarps)
      issue<DK>(p, a, smem_u32(smem), bars);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kComputeWarps) {
    tc_fence_after();
    tmem_dealloc(bars.tmem, kTmemCols);
  }
}

template <int DK>
cudaError_t launch(const gsa_delta_t& p, const DeltaMaps& maps, const DeltaMaps& more,
                   const GradArgs& a, cudaStream_t stream) {
  cudaError_t e = need_regs<grad_kernel<DK>>(kLaunchRegs);
  if (e != cudaSuccess) return e;
  e = allow_smem<grad_kernel<DK>>(kSmem);
  if (e != cudaSuccess) return e;
  const int blocks = static_cast<int>(a.items < 148 ? a.items : 148);
  grad_kernel<DK><<<blocks, kThreads, kSmem, stream>>>(p, maps, more, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grad(const gsa_delta_t& p, const DeltaMaps& maps, const DeltaMaps& more,
                        const DeltaGrads& g, const Saved& s, const Scratch& r, const Table& t,
                        int* err, cudaStream_t stream) {
  const GradArgs a = {t,      s.blocks, s.news, s.states, r.back, r.states,
                      g.dout, g.dq,     g.dk,   g.dv,     g.dg,   g.dbeta,
                      max_chunks(p) * p.Hk, err};
  if (a.items == 0) return cudaSuccess;
  return p.dk <= 64 ? launch<64>(p, maps, more, a, stream) : launch<128>(p, maps, more, a, stream);
}

}  // namespace delta
}  // namespace gsa
