// fa_rotary.hip - norm of queries and keys for each head with the position rotation in the same
// pass, forward and backward, for gfx950 (the mathematics of a row: fa_rotary.h).
//
// Backward of a row, from g = R(p)^T dy:
//   n = x r;  u = g o w;  dx = r (u - n mean(u o n));  dw = sum over all rows of g o n
//
// Both directions move 2 bytes per value and array and compute ~10-30 flops for it, so the memory
// bounds them.  A workgroup of 256 threads takes 2048 / D tokens, one team of D / 8 lanes each, and
// `heads` heads of them one after another, so a token's table row (4 bytes a dim, twice a row's own
// bytes) is read once for all of them and kept in registers; kRowBatch heads' rows are in flight at a
// time.  Reads are whole rows of a packed projection, writes whole runs of tokens of one head.
// At B=4 H=H_kv=32 N=4096 D=128 bf16: forward 98 us, 5.5 TB/s; backward 172 us, 4.7 TB/s, with 5 for the sums of dw
// (a large copy reaches 4.9).
#include "fa_rotary.h"

#include <algorithm>

namespace fa {

template <typename E, int D, bool INTER>
__global__ __launch_bounds__(kRowThreads) void qk_fwd_kernel(QkArgs a, int q_chunks, int chunks) {
  using S = Slot<D>;
  const int chunk = blockIdx.x % chunks;
  const bool is_q = chunk < q_chunks;
  const long long at = (long long)(blockIdx.x / chunks) * S::TOKENS + threadIdx.x / S::TPR;
  const bool valid = at < a.B * a.N;
  const int t = valid ? (int)at : 0;
  const int b = t / a.N, n = t % a.N;
  const int h0 = (is_q ? chunk : chunk - q_chunks) * a.heads;
  turn_heads<E, D, INTER>(a.rot, is_q ? a.rot.q_weight : a.rot.k_weight, is_q ? a.q : a.k, is_q ? a.oq : a.ok, b, n, n,
                          h0, min(h0 + a.heads, is_q ? a.H : a.Hkv), valid);
}

// A workgroup keeps its chunk of heads and walks token blocks, `blocks` workgroups to a chunk; each
// leaves its fp32 sums of dw, reduced over its tokens through LDS, as one row of `part`.
template <typename E, int D, bool INTER>
__global__ __launch_bounds__(kRowThreads) void qk_bwd_kernel(QkArgs a, int q_chunks, int chunks) {
  using S = Slot<D>;
  const int lane = threadIdx.x & 63;
  const int d0 = (threadIdx.x % S::TPR) * 8;
  const int slot = threadIdx.x / S::TPR;
  const int chunk = blockIdx.x % chunks;
  const bool is_q = chunk < q_chunks;
  const int h0 = (is_q ? chunk : chunk - q_chunks) * a.heads;
  const int h1 = min(h0 + a.heads, is_q ? a.H : a.Hkv);
  const Rows& in = is_q ? a.q : a.k;
  const Rows& grad = is_q ? a.gq : a.gk;
  const Rows& out = is_q ? a.oq : a.ok;
  const void* wp = is_q ? a.rot.q_weight : a.rot.k_weight;
  const bool norm = wp != nullptr;
  const int tokens = a.B * a.N;

  float w[8], dw[8];
  load_weight(a.rot, wp, d0, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0.f;

  for (long long t0 = (long long)(blockIdx.x / chunks) * S::TOKENS; t0 < tokens; t0 += (long long)a.blocks * S::TOKENS) {
    const bool valid = t0 + slot < tokens;
    const int t = valid ? (int)t0 + slot : 0;
    const int b = t / a.N, n = t % a.N;
    Turn<D, INTER> turn;
    turn.load(a.rot, lane, d0, b, n, n);
    const uint16_t* src = static_cast<const uint16_t*>(in.data) + b * in.stride_b + n * in.stride_n + d0;
    const uint16_t* gsrc = static_cast<const uint16_t*>(grad.data) + b * grad.stride_b + n * grad.stride_n + d0;
    uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(out.data)) + b * out.stride_b + n * out.stride_n + d0;
    for (int h = h0; h < h1; h += kRowBatch) {
      u32x4 xw[kRowBatch], gw[kRowBatch];
#pragma unroll
      for (int i = 0; i < kRowBatch; ++i) {
        const int hi = min(h + i, h1 - 1);
        gw[i] = gload16(gsrc + hi * grad.stride_h);
        if (norm) xw[i] = gload16(src + hi * in.stride_h);
      }
#pragma unroll
      for (int i = 0; i < kRowBatch; ++i) {
        float gy[8], gp[8], g[8];
        unpack8<E>(gw[i], gy);
        unpack8<E>(turn.fetch(gw[i]), gp);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = __builtin_fmaf(gy[j], turn.c[j], -(partner_of<INTER>(gp, j) * turn.s[j]));
        const bool store = valid && h + i < h1;
        if (norm) {
          float x[8], u[8], dot = 0.f;
          unpack8<E>(xw[i], x);
          const float r = inv_rms<D>(x, a.rot.eps);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            u[j] = g[j] * w[j];
            dot = __builtin_fmaf(u[j], x[j], dot);
          }
          const float mean = team_sum<S::TPR>(dot) * (r * (1.0f / D));   // of u o n
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float nj = x[j] * r;
            if (store) dw[j] = __builtin_fmaf(g[j], nj, dw[j]);
            g[j] = r * __builtin_fmaf(-nj, mean, u[j]);
          }
        }
        if (store) gstore16(dst + (h + i) * out.stride_h, pack8<E>(g));
      }
    }
  }
  if (!norm) return;
  __shared__ float sums[S::TOKENS][D];
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[slot][d0 + i] = dw[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float x = 0.f;
    for (int i = 0; i < S::TOKENS; ++i) x += sums[i][threadIdx.x];
    a.part[((long long)chunk * a.blocks + blockIdx.x / chunks) * D + threadIdx.x] = x;
  }
}

// dw of q (blockIdx.y 0) or k (1): the rows of `part` of their chunks, 4 columns to a workgroup.
template <typename E, int D>
__global__ __launch_bounds__(kRowThreads) void qk_dw_kernel(QkArgs a, int q_chunks, int chunks) {
  const bool is_q = blockIdx.y == 0;
  const int c = blockIdx.x * 4;
  const long long first = is_q ? 0 : (long long)q_chunks * a.blocks;
  const long long rows = (long long)(is_q ? q_chunks : chunks - q_chunks) * a.blocks;
  f32x4 x = f32x4{};
#pragma unroll 4
  for (long long i = threadIdx.x; i < rows; i += kRowThreads) x += gload_f32x4(a.part + (first + i) * D + c);
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], d);
  __shared__ f32x4 sums[kRowThreads / 64];
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = x;
  __syncthreads();
  if (threadIdx.x < 4) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kRowThreads / 64; ++i) s += sums[i][threadIdx.x];
    void* const dst = is_q ? a.dwq : a.dwk;
    if (a.rot.weight_dtype == FA_F32) static_cast<float*>(dst)[c + threadIdx.x] = s;
    else static_cast<uint16_t*>(dst)[c + threadIdx.x] = (uint16_t)pack2<E>(s, s);
  }
}

namespace {

// Heads a workgroup takes: eight, fewer while the grid is under two workgroups to a CU (us at one / two / four: B=1
// H=32 H_kv=8 N=1531 D=128 with three axes 9.3 / 8.6 / 9.1, N=700 5.7 / 5.8 / 7.1, B=2 H=H_kv=16 N=1000 D=64 5.7 / 6.1 /
// 7.9: each workgroup reads its tokens' table rows again).
struct Plan {
  int heads, q_chunks, chunks;
  long long token_blocks;
};

Plan plan_of(int B, int H, int Hkv, int N, int D) {
  Plan p;
  const int tokens = kRowThreads / (D / 8);
  p.token_blocks = ((long long)B * N + tokens - 1) / tokens;
  p.heads = 8;
  auto chunks = [&](int h) { return (h + p.heads - 1) / p.heads; };
  while (p.heads > 1 && p.token_blocks * (chunks(H) + chunks(Hkv)) < 2LL * cu_count()) p.heads /= 2;
  p.q_chunks = chunks(H);
  p.chunks = p.q_chunks + chunks(Hkv);
  return p;
}

int bwd_blocks(const Plan& p) {
  return (int)std::min<long long>(p.token_blocks, std::max(1, 8 * cu_count() / p.chunks));
}

template <typename E, int D>
int launch_qk(QkArgs a, bool bwd) {
  const Plan p = plan_of(a.B, a.H, a.Hkv, a.N, D);
  a.heads = p.heads;
  a.blocks = bwd_blocks(p);
  const long long grid = bwd ? (long long)a.blocks * p.chunks : p.token_blocks * p.chunks;
  if (!grid_fits(grid, kRowThreads)) return FA_ERR_DIMS;
  const dim3 g((unsigned)grid), t(kRowThreads);
  hipStream_t st = (hipStream_t)a.stream;
  if (bwd) {
    if (a.rot.interleaved) hipLaunchKernelGGL((qk_bwd_kernel<E, D, true>), g, t, 0, st, a, p.q_chunks, p.chunks);
    else hipLaunchKernelGGL((qk_bwd_kernel<E, D, false>), g, t, 0, st, a, p.q_chunks, p.chunks);
    if (a.rot.q_weight != nullptr)
      hipLaunchKernelGGL((qk_dw_kernel<E, D>), dim3(D / 4, 2), t, 0, st, a, p.q_chunks, p.chunks);
  } else {
    if (a.rot.interleaved) hipLaunchKernelGGL((qk_fwd_kernel<E, D, true>), g, t, 0, st, a, p.q_chunks, p.chunks);
    else hipLaunchKernelGGL((qk_fwd_kernel<E, D, false>), g, t, 0, st, a, p.q_chunks, p.chunks);
  }
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int dispatch(int dtype, int D, const QkArgs& a, bool bwd) {
  if (dtype == FA_BF16) {
    if (D == 32) return launch_qk<BF16, 32>(a, bwd);
    if (D == 64) return launch_qk<BF16, 64>(a, bwd);
    return launch_qk<BF16, 128>(a, bwd);
  }
  if (D == 32) return launch_qk<F16, 32>(a, bwd);
  if (D == 64) return launch_qk<F16, 64>(a, bwd);
  return launch_qk<F16, 128>(a, bwd);
}

}  // namespace

int qk_norm_rotary(int dtype, int D, const QkArgs& a) { return dispatch(dtype, D, a, false); }

int qk_norm_rotary_bwd(int dtype, int D, const QkArgs& a) { return dispatch(dtype, D, a, true); }

size_t qk_norm_rotary_workspace(int B, int H, int Hkv, int N, int D) {
  const Plan p = plan_of(B, H, Hkv, N, D);
  return (size_t)bwd_blocks(p) * p.chunks * D * sizeof(float);
}

}  // namespace fa
