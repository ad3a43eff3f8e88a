// delta_step.cu — the gated delta rule token by token against a pool of states
// that is updated in place (decoding), and the chunk table of packed batches.
//
// With a = e^g, the two products of a token with the state before it suffice:
//   r = a S^T k,  w = a S^T q,  u = beta (v - r),  o = scale (w + (q.k) u),
//   S <- a S + k u^T,
// so the state is read once, stays in registers over all tokens of the call,
// and is written once.  Bound by HBM: 8 * dk * dv bytes a head and sequence, and by
// how many of them are on their way: a batch of 128 rows, 117 of them with a state of
// 16 heads of 128 x 128, takes 48 us (5.1 TB/s; 38 at a plain copy's rate) with six
// blocks of 16 KB an SM (80 registers a thread, two columns an instruction) and states
// that leave the caches early, 53 with the four that 109 registers allow, 51 with
// eight, which spill.  Blocks of 64 and 128 columns took 61 and 83: more warps meet at
// each barrier.
#include "delta_common.cuh"

namespace gsa {
namespace delta {
namespace {

constexpr int kCols = 32;     // state columns of a block (one 128-byte line a row)
constexpr int kThreads = 128;  // 8 threads of 4 columns x 16 groups of rows
constexpr int kRowGroups = kThreads / 8;
constexpr int kMaxRows = kDeltaMaxDk / kRowGroups;

template <typename E>
__global__ void __launch_bounds__(kThreads, 6) delta_step_kernel(const gsa_delta_t p, float* pool,
                                                              int64_t slots,
                                                              const int32_t* indices, E* out,
                                                              int* err) {
  __shared__ uint64_t sk[kDeltaMaxDk], sq[kDeltaMaxDk];  // each value twice, for two columns
  __shared__ float part[4][2][kCols];
  __shared__ float dots[4];
  const int b = blockIdx.x, hv = blockIdx.y, col0 = blockIdx.z * kCols;
  const int hk = hv / (p.Hv / p.Hk);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int cols = (t & 7) * 4, rg = t >> 3;
  const int col = col0 + cols;
  const bool live = col < p.dv;
  const int64_t slot = indices ? indices[b] : b;
  const bool inside = slot >= 0 && slot < slots;

  uint64_t S[kMaxRows][2];  // two pairs of columns
  float* state = pool + ((inside ? slot : 0) * p.Hv + hv) * static_cast<int64_t>(p.dk) * p.dv;
#pragma unroll
  for (int i = 0; i < kMaxRows; ++i) {
    const int r = rg + i * kRowGroups;
    S[i][0] = S[i][1] = 0;
    if (inside && live && r < p.dk) {
      const ulonglong2 x = __ldcs(
          reinterpret_cast<const ulonglong2*>(state + static_cast<int64_t>(r) * p.dv + col));
      S[i][0] = x.x;
      S[i][1] = x.y;
    }
  }
  // Two rows of the batch must not share a state: the later one is refused, as
  // is an index outside the pool (-1 is an empty row): NaN out, no state
  // touched, and the device error word says so.
  int bad = !inside && slot != -1;
  if (indices && inside)
    for (int j = t; j < b; j += kThreads) bad |= indices[j] == slot;
  bad = __syncthreads_or(bad);
  if (bad || !inside) {
    if (bad && t == 0 && hv == 0 && col0 == 0) atomicExch(err, GSA_ERR_INVALID_ARG);
    const float fill = bad ? __int_as_float(0x7FC00000) : 0.f;
    for (int i = t; i < p.T * kCols; i += kThreads) {
      const int c = col0 + i % kCols;
      if (c < p.dv)
        out[((static_cast<int64_t>(b) * p.T + i / kCols) * p.Hv + hv) * p.dv + c] =
            from_float<E>(fill);
    }
    return;
  }

  const bool gate16 = p.gate_dtype == GSA_DTYPE_BF16;
  for (int tok = 0; tok < p.T; ++tok) {
    float qk = 0.f;
    for (int i = t; i < p.dk; i += kThreads) {
      const float kv = to_float(static_cast<const E*>(
          p.k)[b * p.k_stride[0] + tok * p.k_stride[1] + hk * p.k_stride[2] + i]);
      const float qv = to_float(static_cast<const E*>(
          p.q)[b * p.q_stride[0] + tok * p.q_stride[1] + hk * p.q_stride[2] + i]);
      sk[i] = f2_pack(kv, kv);
      sq[i] = f2_pack(qv, qv);
      qk = fmaf(qv, kv, qk);
    }
    const float a = expf(load_gate(p.g, b * p.g_stride[0] + tok * p.g_stride[1] + hv, gate16));
    const float beta =
        load_gate(p.beta, b * p.beta_stride[0] + tok * p.beta_stride[1] + hv, gate16);
    float v[4] = {};
    if (live) {
      const E* vp = static_cast<const E*>(p.v) + b * p.v_stride[0] + tok * p.v_stride[1] +
                    hv * p.v_stride[2] + col;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to_float(vp[e]);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) qk += __shfl_xor_sync(0xFFFFFFFFu, qk, m);
    if (lane == 0) dots[warp] = qk;
    __syncthreads();
    qk = (dots[0] + dots[1]) + (dots[2] + dots[3]);

    uint64_t r2[2] = {}, w2[2] = {};
    const uint64_t a2 = f2_pack(a, a);
#pragma unroll
    for (int i = 0; i < kMaxRows; ++i) {
      const int row = rg + i * kRowGroups;
      if (row < p.dk) {
        const uint64_t kv = sk[row], qv = sq[row];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          S[i][e] = f2_mul(S[i][e], a2);
          r2[e] = f2_fma(kv, S[i][e], r2[e]);
          w2[e] = f2_fma(qv, S[i][e], w2[e]);
        }
      }
    }
    float r[4] = {f2_lo(r2[0]), f2_hi(r2[0]), f2_lo(r2[1]), f2_hi(r2[1])};
    float w[4] = {f2_lo(w2[0]), f2_hi(w2[0]), f2_lo(w2[1]), f2_hi(w2[1])};
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // the warp's four row groups
#pragma unroll
      for (int m = 8; m <= 16; m <<= 1) {
        r[e] += __shfl_xor_sync(0xFFFFFFFFu, r[e], m);
        w[e] += __shfl_xor_sync(0xFFFFFFFFu, w[e], m);
      }
      if (lane < 8) {
        part[warp][0][cols + e] = r[e];
        part[warp][1][cols + e] = w[e];
      }
    }
    __syncthreads();
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = cols + e;
      const float rs = (part[0][0][c] + part[1][0][c]) + (part[2][0][c] + part[3][0][c]);
      const float ws = (part[0][1][c] + part[1][1][c]) + (part[2][1][c] + part[3][1][c]);
      u[e] = beta * (v[e] - rs);
      if (rg == 0 && live)
        out[((static_cast<int64_t>(b) * p.T + tok) * p.Hv + hv) * p.dv + col + e] =
            from_float<E>(p.scale * fmaf(qk, u[e], ws));
    }
    const uint64_t u2[2] = {f2_pack(u[0], u[1]), f2_pack(u[2], u[3])};
#pragma unroll
    for (int i = 0; i < kMaxRows; ++i) {
      const int row = rg + i * kRowGroups;
      if (row < p.dk) {
        const uint64_t kv = sk[row];
        S[i][0] = f2_fma(kv, u2[0], S[i][0]);
        S[i][1] = f2_fma(kv, u2[1], S[i][1]);
      }
    }
    __syncthreads();  // sk, sq, part and dots are written again by the next token
  }
#pragma unroll
  for (int i = 0; i < kMaxRows; ++i) {
    const int r = rg + i * kRowGroups;
    if (live && r < p.dk)
      __stcs(reinterpret_cast<ulonglong2*>(state + static_cast<int64_t>(r) * p.dv + col),
             make_ulonglong2(S[i][0], S[i][1]));
  }
}

// One block: sequences in order, each cut to [end of the one before, T], and
// their chunks numbered.  A cu_seqlens that decreases or leaves [0, T] is cut
// the same way and reported in the device error word.
__global__ void __launch_bounds__(1024) delta_table_kernel(const int32_t* cu, int N, int T,
                                                           int max_chunks, Table t, int* err) {
  __shared__ int warp_max[32], warp_sum[32], lens[kSorted];
  __shared__ int carry_end, carry_chunk;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(max(cu[0], 0), T);
  if (tid == 0) {
    carry_end = first;
    carry_chunk = 0;
    if (cu[0] < 0 || cu[0] > T) atomicExch(err, GSA_ERR_INVALID_ARG);
  }
  for (int c = tid; c < max_chunks; c += blockDim.x) t.chunk_seq[c] = -1;
  __syncthreads();
  for (int s0 = 0; s0 < N + 2; s0 += blockDim.x) {
    const int s = s0 + tid;
    const int start = carry_end, chunk_start = carry_chunk;
    // running maximum of the (cut) ends
    int end = start;
    if (s < N) {
      const int raw = cu[s + 1];
      if (raw < cu[s] || raw > T) atomicExch(err, GSA_ERR_INVALID_ARG);
      end = min(max(raw, 0), T);
    }
    int m = end;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, m, d);
      if (lane >= d) m = max(m, o);
    }
    if (lane == 31) warp_max[warp] = m;
    __syncthreads();
    int before = start;  // the largest end of the warps before this one
    for (int w = 0; w < warp; ++w) before = max(before, warp_max[w]);
    const int stop = max(m, before);
    int prev = __shfl_up_sync(0xFFFFFFFFu, stop, 1);
    if (lane == 0) prev = before;
    int total = before;
    for (int w = warp; w < 32; ++w) total = max(total, warp_max[w]);
    int begin = prev, len = stop - prev;
    if (s == N) { begin = 0; len = first; }
    if (s == N + 1) { begin = total; len = T - total; }
    if (s > N + 1) len = 0;
    const int chunks = (len + kChunk - 1) / kChunk;
    int n = chunks;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, n, d);
      if (lane >= d) n += o;
    }
    if (lane == 31) warp_sum[warp] = n;
    __syncthreads();
    int at = chunk_start + n - chunks, sum = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += warp_sum[w];
      sum += warp_sum[w];
    }
    if (s < N + 2) {
      t.seq_begin[s] = begin;
      t.seq_len[s] = len;
      if (s < kSorted) lens[s] = len;
      t.seq_chunk[s] = at;
      for (int c = 0; c < chunks; ++c)
        if (at + c < max_chunks) t.chunk_seq[at + c] = s;
    }
    __syncthreads();
    if (tid == 0) {
      carry_end = total;
      carry_chunk = chunk_start + sum;
    }
    __syncthreads();
  }
  for (int s = tid; s < N + 2; s += blockDim.x) {
    int rank = s;
    if (N + 2 <= kSorted) {
      rank = 0;
      const int mine = lens[s];
      for (int o = 0; o < N + 2; ++o) rank += lens[o] > mine || (lens[o] == mine && o < s);
    }
    t.order[rank] = s;
  }
}

}  // namespace

cudaError_t launch_table(const gsa_delta_t& p, void* workspace, int* err, cudaStream_t stream) {
  if (!p.cu_seqlens) return cudaSuccess;
  delta_table_kernel<<<1, 1024, 0, stream>>>(p.cu_seqlens, p.N, p.T,
                                             static_cast<int>(max_chunks(p)),
                                             table_at(workspace, p.N), err);
  return cudaGetLastError();
}

}  // namespace delta

cudaError_t launch_delta_step(const gsa_delta_t& p, float* state, int64_t slots,
                              const int32_t* indices, void* o, int* err, cudaStream_t stream) {
  const dim3 grid(p.B, p.Hv, (p.dv + delta::kCols - 1) / delta::kCols);
  if (p.dtype == GSA_DTYPE_BF16)
    delta::delta_step_kernel<__nv_bfloat16><<<grid, delta::kThreads, 0, stream>>>(
        p, state, slots, indices, static_cast<__nv_bfloat16*>(o), err);
  else
    delta::delta_step_kernel<float><<<grid, delta::kThreads, 0, stream>>>(
        p, state, slots, indices, static_cast<float*>(o), err);
  return cudaGetLastError();
}

}  // namespace gsa
