// fa_rotary.h - norm and position rotation of one row (one head of one token), the part that the
// rotary kernels (fa_rotary.hip) and the paged cache's append (fa_paged.hip) share.
//
//   y = R(p) (w o x r),  r = (mean(x^2) + eps)^(-1/2)
//
// R(p) turns pairs of the first `rotary` dims: (a, b) -> (a cos - b sin, b cos + a sin), the cosine
// and sine read from a table row of the pair's position; pair j is dims (j, j + rotary / 2), or
// (2j, 2j + 1) when interleaved; dims past `rotary` keep their normed value.
//
// A row of D values is held by a team of D / 8 lanes, 8 consecutive dims (16 bytes) each.  With
// `rotary` a multiple of 16, a lane's 8 dims lie in one half of the rotated part, so its partners
// are the 8 dims of one other lane (or its own, interleaved): y = r (x (C w) + x_partner (S w_partner)),
// with the partner's values moved as the row's packed 16-bit words, 4 moves instead of 8.
#pragma once

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {

// 8 packed 16-bit values as fp32.
template <typename E>
__device__ __forceinline__ void unpack8(const u32x4& w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f32<E>(w[i] & 0xFFFFu);
    x[2 * i + 1] = to_f32<E>(w[i] >> 16);
  }
}

template <typename E>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack2<E>(x[0], x[1]), pack2<E>(x[2], x[3]), pack2<E>(x[4], x[5]), pack2<E>(x[6], x[7])};
}

// Sum over the T lanes of a team (T = 4, 8 or 16 neighbours).
template <int T>
__device__ __forceinline__ float team_sum(float x) {
  x = quad_sum(x);
  // DPP row_half_mirror / row_mirror: lanes of one quad hold the same sum by then
  if constexpr (T >= 8) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, false));
  if constexpr (T >= 16) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xF, 0xF, false));
  return x;
}

// What a lane needs to turn the rows of one token.
template <int D, bool INTER>
struct Turn {
  float c[8], s[8];  // own value's factor; partner's factor, with its sign
  int partner;       // lane that holds the partners (interleaved: none)
  uint32_t turned;   // all ones; 0 where nothing turns, so a partner that is infinite or NaN has no say (0 times it is NaN)

  __device__ __forceinline__ static int partner_lane(const RotaryArgs& a, int lane, int d0) {
    if (INTER || d0 >= a.rotary_dim) return lane;
    const int half = a.rotary_dim / 2;
    return d0 < half ? lane + half / 8 : lane - half / 8;
  }

  // The token's entry of an axis; `base`: its position when none are given.
  __device__ __forceinline__ static long long position(const RotaryArgs& a, int axis, int b, int n, long long base) {
    if (a.positions == nullptr) return base;
    const long long at = axis * a.pos_axis_stride + (long long)b * a.pos_batch_stride + n;
    return a.positions_int64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
  }

  __device__ __forceinline__ static int axis_of(const RotaryArgs& a, int pair) {
    return (a.axes > 1 && pair >= a.section_end[0] ? 1 : 0) + (a.axes > 2 && pair >= a.section_end[1] ? 1 : 0);
  }

  // Cosines and sines of the lane's pairs, from pair0 on, at token (b, n).  A negative position leaves the row
  // unturned (padding); one past the table gives NaN.
  template <int NP>
  __device__ __forceinline__ void table_factors(const RotaryArgs& a, int pair0, int b, int n, long long base, float (&cc)[NP],
                                                float (&ss)[NP]) {
    const int half = a.rotary_dim / 2;
    const int axis = axis_of(a, pair0);
    const long long p = position(a, axis, b, n, base);
    turned = ~0u;
    if (axis == axis_of(a, pair0 + NP - 1)) {
      if (p < 0) turned = 0;
      const float* row = a.table + (p < 0 ? 0 : p >= a.table_len ? 0 : p) * a.rotary_dim + pair0;
#pragma unroll
      for (int i = 0; i < NP; i += 4) {
        const f32x4 x = gload_f32x4(row + i), y = gload_f32x4(row + half + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) cc[i + j] = x[j], ss[i + j] = y[j];
      }
      const float bad = p >= a.table_len ? __builtin_nanf("") : 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        cc[i] = p < 0 ? 1.f : cc[i] + bad;
        ss[i] = p < 0 ? 0.f : ss[i] + bad;
      }
    } else {
      // a section ends among this lane's pairs: every axis' position, then every table value
      long long q[kMaxAxes];
#pragma unroll
      for (int i = 0; i < kMaxAxes; ++i) q[i] = position(a, min(i, a.axes - 1), b, n, base);
      long long at[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int k = axis_of(a, pair0 + i);
        at[i] = k == 0 ? q[0] : k == 1 ? q[1] : q[2];
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float* row = a.table + (at[i] >= 0 && at[i] < a.table_len ? at[i] : 0) * a.rotary_dim + pair0 + i;
        cc[i] = row[0], ss[i] = row[half];
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float bad = at[i] >= a.table_len ? __builtin_nanf("") : 0.f;
        cc[i] = at[i] < 0 ? 1.f : cc[i] + bad;
        ss[i] = at[i] < 0 ? 0.f : ss[i] + bad;
      }
    }
  }

  // Factors of token (b, n) for dims d0 .. d0 + 7.
  __device__ __forceinline__ void load(const RotaryArgs& a, int lane, int d0, int b, int n, long long base) {
    partner = partner_lane(a, lane, d0);
    const int half = a.rotary_dim / 2;
    constexpr int NP = INTER ? 4 : 8;   // pairs of this lane
    float cc[NP], ss[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) cc[i] = 1.f, ss[i] = 0.f;
    turned = 0;
    if (a.table != nullptr && d0 < a.rotary_dim) table_factors(a, INTER ? d0 / 2 : (d0 < half ? d0 : d0 - half), b, n, base, cc, ss);
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[2 * i] = c[2 * i + 1] = cc[i];
        s[2 * i] = -ss[i];
        s[2 * i + 1] = ss[i];
      }
    } else {
      const float sign = d0 < half ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = cc[i], s[i] = sign * ss[i];
    }
  }

  // The partner lane's packed row (its own when interleaved: the pairs are inside the lane); zeros where nothing turns.
  __device__ __forceinline__ u32x4 fetch(const u32x4& w) const {
    u32x4 r = w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (!INTER) r[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(partner << 2, (int)w[i]);
      r[i] &= turned;
    }
    return r;
  }
};

// Partner's value of dim i out of the values that fetch() brought.
template <bool INTER>
__device__ __forceinline__ float partner_of(const float (&xp)[8], int i) {
  return INTER ? xp[i ^ 1] : xp[i];
}

// Norm weight of dims d0 .. d0 + 7 (ones without one), 16-byte aligned.
__device__ __forceinline__ void load_weight(const RotaryArgs& a, const void* w, int d0, float (&x)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 1.f;
  } else if (a.weight_dtype == FA_F32) {
    const float* const p = static_cast<const float*>(w) + d0;
    const f32x4 lo = gload_f32x4(p), hi = gload_f32x4(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
  } else {
    const u32x4 v = gload16(static_cast<const uint16_t*>(w) + d0);
    if (a.weight_dtype == FA_BF16) unpack8<BF16>(v, x);
    else unpack8<F16>(v, x);
  }
}

template <int D>
__device__ __forceinline__ float inv_rms(const float (&x)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
  return 1.0f / __builtin_sqrtf(team_sum<D / 8>(ss) * (1.0f / D) + eps);
}

// One row: x packed (and its partner's), cw = C w and sw = S w_partner of its token and tensor.  The row is
// z times the value returned.
template <typename E, int D, bool INTER>
__device__ __forceinline__ float turn_row(const u32x4& w, const u32x4& wp, const float (&cw)[8], const float (&sw)[8],
                                          bool norm, float eps, float (&z)[8]) {
  float x[8], xp[8];
  unpack8<E>(w, x);
  unpack8<E>(wp, xp);
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = __builtin_fmaf(x[i], cw[i], partner_of<INTER>(xp, i) * sw[i]);
  return norm ? inv_rms<D>(x, eps) : 1.f;
}

// The weights of a lane's dims and of their partners (in place of the partners' own order when
// interleaved: partner_of picks them).
template <bool INTER>
__device__ __forceinline__ void load_weights(const RotaryArgs& a, const void* w, int d0, float (&own)[8], float (&other)[8]) {
  const int half = a.rotary_dim / 2;
  const bool turned = a.table != nullptr && d0 < a.rotary_dim;
  load_weight(a, w, d0, own);
  load_weight(a, w, INTER || !turned ? d0 : d0 < half ? d0 + half : d0 - half, other);
}

template <int D, bool INTER>
__device__ __forceinline__ void fold_weights(const Turn<D, INTER>& t, const float (&own)[8], const float (&other)[8],
                                             float (&cw)[8], float (&sw)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cw[i] = t.c[i] * own[i];
    sw[i] = t.s[i] * partner_of<INTER>(other, i);
  }
}

constexpr int kRowThreads = 256;
constexpr int kRowBatch = 4;     // heads whose rows are in flight at a time

template <int D, int NT = kRowThreads>
struct Slot {
  static constexpr int TPR = D / 8;        // lanes per row
  static constexpr int TOKENS = NT / TPR;  // rows a workgroup of NT threads holds at once
};

// Heads h0 .. h1 - 1 of token (b, n): one team of lanes, the heads one after another, the token's
// table row and the weight folded into registers once.
template <typename E, int D, bool INTER>
__device__ __forceinline__ void turn_heads(const RotaryArgs& rot, const void* w, const Rows& in, const Rows& out, int b,
                                           int n, long long base, int h0, int h1, bool valid) {
  const int d0 = (threadIdx.x % Slot<D>::TPR) * 8;
  float own[8], other[8], cw[8], sw[8];
  load_weights<INTER>(rot, w, d0, own, other);
  Turn<D, INTER> turn;
  turn.load(rot, threadIdx.x & 63, d0, b, n, base);
  fold_weights(turn, own, other, cw, sw);
  const uint16_t* src = static_cast<const uint16_t*>(in.data) + b * in.stride_b + n * in.stride_n + d0;
  uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(out.data)) + b * out.stride_b + n * out.stride_n + d0;
  for (int h = h0; h < h1; h += kRowBatch) {
    u32x4 x[kRowBatch];
#pragma unroll
    for (int i = 0; i < kRowBatch; ++i) x[i] = gload16(src + min(h + i, h1 - 1) * in.stride_h);
#pragma unroll
    for (int i = 0; i < kRowBatch; ++i) {
      float y[8];
      const float r = turn_row<E, D, INTER>(x[i], turn.fetch(x[i]), cw, sw, w != nullptr, rot.eps, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= r;
      if (valid && h + i < h1) gstore16(dst + (h + i) * out.stride_h, pack8<E>(y));
    }
  }
}

}  // namespace fa
