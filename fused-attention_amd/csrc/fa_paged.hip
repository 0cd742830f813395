// fa_paged.hip - keys and values in pages of 8-bit values with a scale for each page and head:
// the append (norm, rotation, quantisation) and the attention over the pages, for gfx950.
#include "fa_paged.h"
#include "fa_rotary.h"

#include <algorithm>
#include <iterator>

namespace fa {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The least e with amax <= 448 2^e (448 = 1.75 2^8), kept within the scales' range.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleMin), kScaleMax);
}

// 8 values times `mul` as e4m3, to nearest even (NaN to NaN; the caller sees to it that none passes 448).
__device__ __forceinline__ u32x2 encode8(const float (&y)[8], float mul) {
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * mul, y[4 * i + 1] * mul, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * mul, y[4 * i + 3] * mul, w, true);
    r[i] = (uint32_t)w;
  }
  return r;
}

__device__ __forceinline__ void decode8(const u32x2& w, float (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    y[4 * i] = a[0], y[4 * i + 1] = a[1], y[4 * i + 2] = b[0], y[4 * i + 3] = b[1];
  }
}

// ---------------------------------------------------------------------------
// Append.  The first `items` workgroups each own one page of one sequence and K/V head, for K or for V, so
// nobody else writes its codes and scale: it holds the page's new rows in registers, reduces their largest
// value, and writes codes.  The others turn the queries (turn_heads); the pages, whose chain of waits is
// longer, go first (queries first: +3 % at B=2 H=32 H_kv=8 N=8192 D=128, +5 % at N=1).  PASSES: new rows of a page over
// the rows that the workgroup's NT threads hold at once; four at most, or the registers leave too few waves
// (128-row pages at D = 128: eight passes of 256 threads 101 us, four of 512 95; 64-row pages: four of 256 90, two
// of 512 91), and no more threads than the new rows have pieces: where few tokens are new, the start of the waves is the
// time (one token, B=64 D=128, pages of 128 rows: 512 threads 12.1 us, 64 5.6; with 32 K/V heads 32.6 and 6.8; 16-row
// pages at D = 64, B=3 N=1000: 256 threads 9.3 us, 128 7.1).  Bytes bound the large call: B=2 H=32 H_kv=8 N=8192 D=128
// in pages of 128 takes 93 us, 4.05 TB/s, some 12 of them K's norm and table rows; one token a sequence is a launch and
// the chain length, page, scale, row, code (B=64 H=32 H_kv=8: 5.4 us).
template <typename E, int D, bool INTER, int PASSES, int NT>
__global__ __launch_bounds__(NT) void append_kernel(AppendArgs a, int items, int q_chunks, int touched) {
  using S = Slot<D, NT>;
  const int slot = threadIdx.x / S::TPR;
  const int Hkv = a.cache.H_kv, ps = a.cache.page_size;
  if ((int)blockIdx.x >= items) {
    const int chunk = (blockIdx.x - items) % q_chunks;
    const long long at = (long long)((blockIdx.x - items) / q_chunks) * S::TOKENS + slot;
    const bool valid = at < a.B * a.N;
    const int t = valid ? (int)at : 0;
    const int b = t / a.N, n = t % a.N, h0 = chunk * a.heads;
    turn_heads<E, D, INTER>(a.rot, a.rot.q_weight, a.q, a.oq, b, n, (long long)past_of(a.past, b) + n, h0,
                            min(h0 + a.heads, a.H), valid);
    return;
  }
  int item = blockIdx.x;
  const int h = item % Hkv;
  item /= Hkv;
  const bool is_k = item % 2 == 0;
  item /= 2;
  const int b = item / touched;
  const int past = past_of(a.past, b), fresh = fresh_of(a.fresh, b, a.N);
  const int col = past / ps + item % touched;
  const int first = col * ps;                      // the page's first key
  if (first >= past + fresh) return;
  const int page = page_of(a.cache, b, col);
  if (page < 0) return;
  const int held = max(past - first, 0);           // rows the page holds already
  const int row0 = held, n0 = first + held - past; // the page's first new row, and its token

  const int lane = threadIdx.x & 63;
  const int d0 = (threadIdx.x % S::TPR) * 8;
  const long long ph = (long long)page * Hkv + h;
  uint8_t* const codes = static_cast<uint8_t*>(is_k ? a.cache.k : a.cache.v) + ph * ps * D + d0;
  void* const scales = is_k ? a.cache.k_scale : a.cache.v_scale;
  const int e_held = scale_of(scales, ph);
  const Rows& in = is_k ? a.k : a.v;
  const uint16_t* src = static_cast<const uint16_t*>(in.data) + b * in.stride_b + h * in.stride_h + d0;

  // A row is z r: r (the norm's 1 / rms) is one factor for the row, so the largest value takes it once, and the
  // codes take it with the scale (a power of two, so the product rounds as z r does).
  float z[PASSES][8], r[PASSES], own[8], other[8];
  float amax = 0.f;
  if (is_k) load_weights<INTER>(a.rot, a.rot.k_weight, d0, own, other);
  auto live = [&](int p) __attribute__((always_inline)) {
    return row0 + p * S::TOKENS + slot < ps && n0 + p * S::TOKENS + slot < fresh;
  };
  auto pass = [&](int p, bool all) __attribute__((always_inline)) {
    const bool mine = all || live(p);
    const int n = mine ? n0 + p * S::TOKENS + slot : 0;
    const u32x4 w = gload16(src + n * in.stride_n);
    r[p] = 1.f;
    if (is_k) {
      Turn<D, INTER> turn;
      turn.load(a.rot, lane, d0, b, n, (long long)past + n);
      float cw[8], sw[8];
      fold_weights(turn, own, other, cw, sw);
      r[p] = turn_row<E, D, INTER>(w, turn.fetch(w), cw, sw, a.rot.k_weight != nullptr, a.rot.eps, z[p]);
    } else {
      unpack8<E>(w, z[p]);
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf(z[p][i]));   // (NaN counts for nothing)
    if (mine) amax = fmaxf(amax, top * r[p]);
  };
  // (a page of which a few rows are new skips the passes without one; all new, no branch parts their loads)
  const bool all = held == 0 && first + ps <= past + fresh && ps >= S::TOKENS;
  if (all) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) pass(p, true);
  } else {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      if (row0 + p * S::TOKENS < ps && n0 + p * S::TOKENS < fresh) pass(p, false);
    }
  }
  __shared__ float tops[NT / 64];
  auto over_all = [&](float x) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) x = fmaxf(x, __shfl_xor(x, m));
    if (lane == 0) tops[threadIdx.x / 64] = x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) x = fmaxf(x, tops[i]);
    return x;
  };
  amax = over_all(amax);
  if (amax > kCodeMax * exp2i(kScaleMax)) {
    // infinities become NaN and count for nothing, finite values past the scales' range become its end
    amax = 0.f;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const float end = kCodeMax * exp2i(kScaleMax);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = z[p][i] * r[p];
        z[p][i] = __builtin_fabsf(y) < __builtin_inff() ? fminf(fmaxf(y, -end), end) : __builtin_nanf("");
        if (live(p) && __builtin_fabsf(y) < __builtin_inff()) amax = fmaxf(amax, __builtin_fabsf(z[p][i]));
      }
      r[p] = 1.f;
    }
    __syncthreads();
    amax = over_all(amax);
  }
  int e = scale_exponent(amax);
  if (held > 0) e = max(e, e_held);
  const float mul = exp2i(-e);
#pragma unroll
  for (int p = 0; p < PASSES; ++p)
    if (all || live(p)) *reinterpret_cast<u32x2*>(codes + (row0 + p * S::TOKENS + slot) * D) = encode8(z[p], r[p] * mul);
  if (held > 0 && e > e_held) {
    const float move = exp2i(e_held - e);
    constexpr int AHEAD = 8;   // rows in flight
    for (int at = slot; at < held; at += AHEAD * S::TOKENS) {
      u32x2 w[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int row = at + i * S::TOKENS;
        w[i] = *reinterpret_cast<const u32x2*>(codes + (row < held ? row : at) * D);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        float x[8];
        decode8(w[i], x);
        if (at + i * S::TOKENS < held) *reinterpret_cast<u32x2*>(codes + (at + i * S::TOKENS) * D) = encode8(x, move);
      }
    }
  }
  if (threadIdx.x == 0) static_cast<uint8_t*>(scales)[ph] = (uint8_t)(e + 127);
}

// ---------------------------------------------------------------------------
// Attention of few rows (the mathematics: fa_paged.h).
//
// Rows: the N x G queries of a K/V head (G = H / H_kv), row r = token r / G, head r % G: 16 or 32 to
// a workgroup, so each key's bytes serve all of them.  S^T = K Q^T as 16x16x32 products (16 keys x 16
// rows): a lane owns one row, and the scores are fed back as the B operand of O^T += V^T P^T.  Two
// 16-key tiles fill its 32 contraction slots; with slot (group g, j) = key 16 (j / 4) + 4 g + j % 4
// no score moves between lanes, and V is read in that order, straight from the pages' rows: a lane
// takes D / 16 dims of each of its 8 keys and pairs them up in registers.  Nothing is staged in LDS.
// Bytes bound it: 32 sequences of 5461 to 16384 keys, H=32 H_kv=8 D=128, 136.6 us with the join, 5.3 TB/s; where
// the bytes are few, the chain length, page, scale, keys and the join's launch do (8 sequences of up to 4005 keys:
// 12.9 + 4.0 us for 47 MB).
constexpr int kWaves = 4;
constexpr int kRows = 16;
constexpr int kStep = 32;   // keys per step of a wave
constexpr int kSplitStep = kWaves * kStep;

// Over the four 16-lane groups of a wave.
__device__ __forceinline__ float groups_max(float x) {
  x = halfwave_max(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
  x = halfwave_sum(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The keys of one 16-key tile of a wave: its K and V bytes in registers.
template <int D>
struct Tile {
  static constexpr int KB = D / 4;    // bytes of a K row per lane
  static constexpr int VB = D / 16;   // bytes of a V row per lane = 16-row blocks of O^T
  static constexpr int VW = VB >= 4 ? VB / 4 : 1;
  uint32_t k[KB / 4];
  uint32_t v[4][VW];

  // base: the tile's offset in the pools (uniform); lane (c, g): K row c, 16-byte pieces g of each 64;
  // V rows 4 g + i, bytes c VB
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, long long base, int c, int g) {
    const uint8_t* const k0 = kp + base;
    const uint8_t* const v0 = vp + base;
    if constexpr (D == 32) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(k0 + c * D + 8 * g);
      k[0] = w[0], k[1] = w[1];
    } else {
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(k0 + c * D + 64 * h + 16 * g);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[4 * h + j] = w[j];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* const p = v0 + (4 * g + i) * D + c * VB;
      if constexpr (VB == 8) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p);
        v[i][0] = w[0], v[i][1] = w[1];
      } else if constexpr (VB == 4) {
        v[i][0] = *reinterpret_cast<const uint32_t*>(p);
      } else {
        v[i][0] = *reinterpret_cast<const uint16_t*>(p);
      }
    }
  }
};

// Workgroups reach the XCDs in turn (wg % 8).  Where the parts of all units' keys fill the XCDs evenly, the row blocks of
// one part go to one XCD, whose L2 then reads those keys once (8 sequences of 4000 keys, 8 K/V heads, D = 128, four
// blocks of 16 rows 47.4 -> 26.8 us; two parts alone, 250 blocks: 25.9 -> 57 on two XCDs).  The parts take turns: a
// run of them to each XCD leaves those with the shorter sequences idle (32 sequences of 5461 to 16384 keys 137 -> 154).
__host__ __device__ __forceinline__ bool by_xcd(long long parts) { return parts % 8 == 0 || parts >= 64; }

// RT: 16-row blocks that a wave holds; each converted K and V operand serves all of them.
template <typename E, int D, int RT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void attend_kernel(PagedArgs a, int row_blocks) {
  typedef Tile<D> T;
  constexpr int VB = T::VB;
  constexpr int KT = D / 32;         // contraction steps over D
  constexpr int LD = D + 4;          // row of the merge buffer
  constexpr int BR = kRows * RT;     // rows of the workgroup
  const float NEG_INF = -__builtin_inff();
  __shared__ __attribute__((aligned(16))) float merge[kWaves][BR][LD];
  __shared__ float ml[kWaves][2][BR];

  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Hkv = a.cache.H_kv, ps = a.cache.page_size, G = a.H / Hkv;
  const int parts = a.B * Hkv * a.nsplit;   // of all units' keys
  int part = blockIdx.x / row_blocks, rb = row_blocks - 1 - blockIdx.x % row_blocks;   // (the most keys first)
  if (by_xcd(parts)) {   // (the grid is whole rounds of 8 parts)
    part = blockIdx.x / (8 * row_blocks) * 8 + blockIdx.x % 8, rb = row_blocks - 1 - blockIdx.x / 8 % row_blocks;
    if (part >= parts) return;
  }
  const int split = part % a.nsplit, bh = part / a.nsplit;
  const long long block = (long long)bh * row_blocks + rb;
  const int b = bh / Hkv, hk = bh % Hkv;
  const Block x = block_of(a, b, rb, G, BR);
  const int per = split_keys(x.keys, a.nsplit, kSplitStep);
  const int first = split * per, last = min(first + per, x.keys);   // keys of this workgroup
  if (split > 0 && first >= x.keys) return;                        // (the first split also writes what has no keys)

  // Q^T: column c of each block, dims of step s: 64 (s / 2) + 16 g + 8 (s % 2) (D = 32: 8 g)
  auto dim_of = [&](int s) __attribute__((always_inline)) { return D == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1); };
  u32x4 qf[RT][KT];
  int lim[RT];    // last key that this lane's rows see
  f32x4 acc[RT][VB];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int at = x.r0 + 16 * t + c, r = min(at, x.rows - 1), tok = r / G, head = hk * G + r % G;
    lim[t] = at < x.rows && tok < x.fresh ? x.past + tok : -1;
    const uint16_t* q = static_cast<const uint16_t*>(a.q.data) + b * a.q.stride_b + head * a.q.stride_h + tok * a.q.stride_n;
#pragma unroll
    for (int s = 0; s < KT; ++s) qf[t][s] = gload16(q + dim_of(s));
#pragma unroll
    for (int i = 0; i < VB; ++i) acc[t][i] = f32x4{};
    m[t] = -__FLT_MAX__, l[t] = 0.f;
  }
  const uint8_t* const kp = static_cast<const uint8_t*>(a.cache.k);
  const uint8_t* const vp = static_cast<const uint8_t*>(a.cache.v);

  // Step j of this wave: keys first + (4 j + wave) 32 + 0..31, two tiles.  Lane i keeps page and scales of
  // its wave's tile i of a run of 32 steps, so the loop below waits for no address.
  const int steps = last > first ? (last - first + kWaves * kStep - 1) / (kWaves * kStep) : 0;
  int my_page = 0, my_ve = 0, my_row = 0;
  float my_ks = 0.f;
  auto load_run = [&](int j0) __attribute__((always_inline)) {
    const int key = first + ((j0 + lane / 2) * kWaves + wave) * kStep + 16 * (lane & 1);
    int page = key < last ? page_of(a.cache, b, key / ps) : 0;
    const long long ph = (long long)max(page, 0) * Hkv + hk;
    const int ke = scale_of(a.cache.k_scale, ph), ve = scale_of(a.cache.v_scale, ph);
    my_ks = page < 0 ? __builtin_nanf("") : exp2i(ke) * a.scale_log2;   // (no page: its rows become NaN)
    my_ve = page < 0 ? 0 : ve;
    my_page = max(page, 0);
    my_row = key % ps;
  };
  auto load_tile = [&](T& t, int i) __attribute__((always_inline)) {   // tile i of the run
    const int page = __builtin_amdgcn_readlane(my_page, i), row = __builtin_amdgcn_readlane(my_row, i);
    t.load(kp, vp, (((long long)page * Hkv + hk) * ps + row) * D, c, g);
  };

  // V^T operand of dims block y: slots j = 4 u + n are keys (u, n), the lane's dim c VB + y
  auto v_operand = [&](const T (&t)[2], int y) __attribute__((always_inline)) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t lo = cvt_f16(t[w >> 1].v[2 * (w & 1)][y >> 2], (y & 2) != 0);
      const uint32_t hi = cvt_f16(t[w >> 1].v[2 * (w & 1) + 1][y >> 2], (y & 2) != 0);
      r[w] = __builtin_amdgcn_perm(hi, lo, y & 1 ? 0x07060302u : 0x05040100u);
    }
    return r;
  };
  bool nan_met = false;   // a masked step of V held a NaN

  auto compute = [&](T (&t)[2], int i, int k0) __attribute__((always_inline)) {
    f32x4 s[RT][2];
    int ve[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_ks), i + u));
      ve[u] = __builtin_amdgcn_readlane(my_ve, i + u);
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][u] = f32x4{};
#pragma unroll
      for (int n = 0; n < KT; ++n) {
        const u32x4 k = codes8<E>(t[u].k[2 * n], t[u].k[2 * n + 1]);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][u] = mfma16<E>(k, qf[r][n], s[r][u]);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < 4; ++n) s[r][u][n] = __builtin_fmaf(s[r][u][n], ks, (float)ve[u]);
    }
    if (k0 + kStep - 1 > x.lmin) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int key = k0 + 16 * u + 4 * g + n;
#pragma unroll
          for (int r = 0; r < RT; ++r)
            if (key > lim[r]) s[r][u][n] = NEG_INF;
#pragma unroll
          for (int w = 0; w < T::VW; ++w) {   // what lies behind the last key may be anything
            const uint32_t v = key >= x.keys ? 0u : t[u].v[n][w], nan = nan_bytes(v);
            t[u].v[n][w] = without_nan(v, nan);
            nan_met |= nan != 0;
          }
        }
    }
    u32x4 pf[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float mx = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                       fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
      mx = groups_max(mx);
      if (__builtin_amdgcn_ballot_w64(mx > m[r] + kLazy)) {
        const float mn = mx > m[r] + kLazy ? mx - kBelow : m[r];   // (a row's own scores alone move it)
        const float alpha = fast_exp2(m[r] - mn);
        m[r] = mn;
        l[r] *= alpha;
#pragma unroll
        for (int n = 0; n < VB; ++n) acc[r][n] *= alpha;
      }
      float p[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < 4; ++n) p[u][n] = fast_exp2(s[r][u][n] - m[r]);
        l[r] = __builtin_fmaf((p[u][0] + p[u][1]) + (p[u][2] + p[u][3]), exp2i(-ve[u]), l[r]);
      }
      pf[r] = u32x4{pack2<F16>(p[0][0], p[0][1]), pack2<F16>(p[0][2], p[0][3]), pack2<F16>(p[1][0], p[1][1]),
                    pack2<F16>(p[1][2], p[1][3])};
    }
#pragma unroll
    for (int y = 0; y < VB; ++y) {
      const u32x4 v = v_operand(t, y);
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r][y] = mfma16<F16>(v, pf[r], acc[r][y]);
    }
  };

  // The next step's bytes are on their way while a step is computed; past the last one its own
  // are read once more, never past the run.
  for (int j0 = 0; j0 < steps; j0 += 32) {
    load_run(j0);
    const int n = min(steps - j0, 32);
    T ta[2], tb[2];
    load_tile(ta[0], 0), load_tile(ta[1], 1);
    for (int j = 0; j < n; j += 2) {
      const int j1 = min(j + 1, n - 1), j2 = min(j + 2, n - 1);
      load_tile(tb[0], 2 * j1), load_tile(tb[1], 2 * j1 + 1);
      compute(ta, 2 * j, first + ((j0 + j) * kWaves + wave) * kStep);
      load_tile(ta[0], 2 * j2), load_tile(ta[1], 2 * j2 + 1);
      if (j + 1 < n) compute(tb, 2 * j + 2, first + ((j0 + j + 1) * kWaves + wave) * kStep);
    }
  }

  if (__builtin_amdgcn_ballot_w64(nan_met)) {
    for (int j = 0; j < steps; ++j) {
      const int k0 = first + (j * kWaves + wave) * kStep;
      if (k0 + kStep - 1 <= x.lmin || k0 >= last) continue;
      T t[2];
      u32x4 seen[RT];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int key = k0 + 16 * u;
        const long long page = key < last ? max(page_of(a.cache, b, key / ps), 0) : 0;
        t[u].load(kp, vp, ((page * Hkv + hk) * ps + key % ps) * D, c, g);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int w = 0; w < T::VW; ++w) t[u].v[n][w] = key + 4 * g + n < x.keys ? nan_as_one(t[u].v[n][w]) : 0u;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < RT; ++r)
            seen[r][2 * u + n] = (key + 4 * g + 2 * n <= lim[r] ? 0x3C00u : 0u) | (key + 4 * g + 2 * n + 1 <= lim[r] ? 0x3C000000u : 0u);
      }
#pragma unroll
      for (int y = 0; y < VB; ++y)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const f32x4 count = mfma16<F16>(v_operand(t, y), seen[r], f32x4{});
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (count[n] > 0.f) acc[r][y][n] = __builtin_nanf("");
        }
    }
  }

  // merge of the waves: lane (c, g) holds row c, dims 4 g VB .. + 4 VB - 1
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const float sum = groups_sum(l[r]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int y = 0; y < VB; ++y) merge[wave][16 * r + c][(4 * g + i) * VB + y] = acc[r][y][i];
    if (g == 0) ml[wave][0][16 * r + c] = m[r], ml[wave][1][16 * r + c] = sum;
  }
  __syncthreads();
  constexpr int PER = kRows * D / (64 * kWaves);   // values per thread (D = 32: 2)
  constexpr int TR = D / PER;                      // threads per row
  const int d0 = threadIdx.x % TR * PER;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = 16 * t + threadIdx.x / TR, rr = x.r0 + row;
    if (rr >= x.rows) return;
    const int ot = rr / G, oh = hk * G + rr % G;
    float M = -__FLT_MAX__, f[kWaves], L = 0.f, o[PER];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w][0][row]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      f[w] = fast_exp2(ml[w][0][row] - M);
      L = __builtin_fmaf(f[w], ml[w][1][row], L);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float z = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) z = __builtin_fmaf(f[w], merge[w][row][d0 + i], z);
      o[i] = z;
    }
    if (per < x.keys) {   // more than one split: the join divides
      float* const dst = part_row<D>(a, block, split, row, BR);
#pragma unroll
      for (int i = 0; i < PER; ++i) dst[d0 + i] = o[i];
      if (d0 == 0) dst[D] = M, dst[D + 1] = L;
      continue;
    }
    const bool live = ot < x.fresh;
    const float inv = live ? 1.0f / L : 0.f;
    uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(a.o.data)) + b * a.o.stride_b + oh * a.o.stride_h + ot * a.o.stride_n + d0;
#pragma unroll
    for (int i = 0; i < PER; i += 2)
      *reinterpret_cast<uint32_t*>(dst + i) = live ? pack2<E>(o[i] * inv, o[i + 1] * inv) : 0u;
    if (a.lse != nullptr && d0 == 0) a.lse[((long long)b * a.H + oh) * a.N + ot] = live ? M + __log2f(L) : NEG_INF;
  }
}

// Joins the splits of a row, a workgroup to a row: D / 4 threads a split, 1024 / D splits at a time.
// Rows of blocks that were not split are there already.
constexpr int kJoinThreads = 256;

template <typename E, int D>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(PagedArgs a, int row_blocks, int block_rows, int step) {
  constexpr int TR = D / 4, PAR = kJoinThreads / TR;
  __shared__ float factor[kMaxSplit];
  __shared__ __attribute__((aligned(16))) float sums[PAR][D];
  const int Hkv = a.cache.H_kv, G = a.H / Hkv, rows = a.N * G;
  const int bh = blockIdx.x / rows, rr = blockIdx.x % rows, b = bh / Hkv, hk = bh % Hkv;
  const long long block = (long long)bh * row_blocks + rr / block_rows;
  const int p = threadIdx.x / TR, d0 = threadIdx.x % TR * 4;
  const float* const src = part_row<D>(a, block, 0, rr % block_rows, block_rows);
  const int stride = block_rows * (D + 4);
  // every wave takes the maximum and the sum of all (m', l), two splits to a lane; the first keeps the factors.
  // (The loads reach all nsplit places, written or not, so that they do not wait for the lengths, which say how
  // many count.)
  const int lane = threadIdx.x & 63;
  float m[2], l[2], M = -__FLT_MAX__, L = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* const ml = src + min(lane + 64 * i, a.nsplit - 1) * stride + D;
    m[i] = ml[0], l[i] = ml[1];
  }
  constexpr int AHEAD = kMaxSplit / PAR < 8 ? kMaxSplit / PAR : 8;
  f32x4 v[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) v[i] = gload_f32x4(src + min(p + i * PAR, a.nsplit - 1) * stride + d0);
  const Block x = block_of(a, b, rr / block_rows, G, block_rows);
  const int per = split_keys(x.keys, a.nsplit, step);
  if (per >= x.keys) return;
  const int n = (x.keys + per - 1) / per;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i >= n) m[i] = -__FLT_MAX__, l[i] = 0.f;
  M = fmaxf(m[0], m[1]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) M = fmaxf(M, __shfl_xor(M, d));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = fast_exp2(m[i] - M);
    L = __builtin_fmaf(f, l[i], L);
    if (threadIdx.x < 64) factor[lane + 64 * i] = lane + 64 * i < n ? f : 0.f;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) L += __shfl_xor(L, d);
  __syncthreads();
  f32x4 o = f32x4{};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = p + i * PAR;
    const float f = s < n ? factor[s] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = s < n ? __builtin_fmaf(f, v[i][e], o[e]) : o[e];
  }
  for (int s = p + AHEAD * PAR; s < n; s += PAR) {
    const f32x4 w = gload_f32x4(src + s * stride + d0);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(factor[s], w[e], o[e]);
  }
  *reinterpret_cast<f32x4*>(&sums[p][d0]) = o;
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  float z[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PAR; ++i) {
    z[0] += sums[i][2 * threadIdx.x];
    z[1] += sums[i][2 * threadIdx.x + 1];
  }
  const int ot = rr / G, oh = hk * G + rr % G;
  const bool live = ot < x.fresh;
  const float inv = live ? 1.0f / L : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(a.o.data)) + b * a.o.stride_b + oh * a.o.stride_h + ot * a.o.stride_n;
  *reinterpret_cast<uint32_t*>(dst + 2 * threadIdx.x) = live ? pack2<E>(z[0] * inv, z[1] * inv) : 0u;
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[((long long)b * a.H + oh) * a.N + ot] = live ? M + __log2f(L) : -__builtin_inff();
}

// The same for few splits and many rows: D / 4 threads to a row, which walk its splits.
constexpr int kFewSplits = 16;

template <typename E, int D>
__global__ __launch_bounds__(kJoinThreads) void join_few_kernel(PagedArgs a, int row_blocks, int block_rows, int step) {
  constexpr int TR = D / 4;
  const int Hkv = a.cache.H_kv, G = a.H / Hkv, rows = a.N * G;
  const long long i = (long long)blockIdx.x * (kJoinThreads / TR) + threadIdx.x / TR;   // (batch, K/V head), row
  if (i >= (long long)a.B * Hkv * rows) return;
  const int bh = i / rows, rr = i % rows, b = bh / Hkv, hk = bh % Hkv;
  const float* const src = part_row<D>(a, (long long)bh * row_blocks + rr / block_rows, 0, rr % block_rows, block_rows);
  const int stride = block_rows * (D + 4), d0 = threadIdx.x % TR * 4;
  float m[kFewSplits], l[kFewSplits], M = -__FLT_MAX__, L = 0.f;
  f32x4 v[kFewSplits], o = f32x4{};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s)
    if (s < a.nsplit) {   // (written or not, as above)
      m[s] = src[s * stride + D], l[s] = src[s * stride + D + 1];
      v[s] = gload_f32x4(src + s * stride + d0);
    }
  const Block x = block_of(a, b, rr / block_rows, G, block_rows);
  const int per = split_keys(x.keys, a.nsplit, step);
  if (per >= x.keys) return;
  const int n = (x.keys + per - 1) / per;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s)
    if (s < n) M = fmaxf(M, m[s]);
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s)
    if (s < n) {
      const float f = fast_exp2(m[s] - M);
      L = __builtin_fmaf(f, l[s], L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(f, v[s][e], o[e]);
    }
  const int ot = rr / G, oh = hk * G + rr % G;
  const bool live = ot < x.fresh;
  const float inv = live ? 1.0f / L : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(a.o.data)) + b * a.o.stride_b + oh * a.o.stride_h + ot * a.o.stride_n;
  *reinterpret_cast<u32x2*>(dst + d0) =
      live ? u32x2{pack2<E>(o[0] * inv, o[1] * inv), pack2<E>(o[2] * inv, o[3] * inv)} : u32x2{};
  if (a.lse != nullptr && d0 == 0)
    a.lse[((long long)b * a.H + oh) * a.N + ot] = live ? M + __log2f(L) : -__builtin_inff();
}

// ---------------------------------------------------------------------------
namespace {

template <typename E, int D, bool INTER, int PASSES, int NT>
int launch_append(AppendArgs a) {
  typedef Slot<D, NT> S;
  const int ps = a.cache.page_size, touched = (a.N + ps - 2) / ps + 1;
  const long long items = 2LL * a.B * touched * a.cache.H_kv;
  long long q_blocks = 0;
  int q_chunks = 0;
  if (a.q.data != nullptr) {
    const long long token_blocks = ((long long)a.B * a.N + S::TOKENS - 1) / S::TOKENS;
    a.heads = 8;
    while (a.heads > 1 && token_blocks * ((a.H + a.heads - 1) / a.heads) < 2LL * cu_count()) a.heads /= 2;
    q_chunks = (a.H + a.heads - 1) / a.heads;
    q_blocks = token_blocks * q_chunks;
  }
  if (!grid_fits(items + q_blocks, NT)) return FA_ERR_DIMS;
  hipLaunchKernelGGL((append_kernel<E, D, INTER, PASSES, NT>), dim3((unsigned)(items + q_blocks)), dim3(NT), 0,
                     (hipStream_t)a.stream, a, (int)items, q_chunks, touched);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <typename E, int D>
int launch_append(const AppendArgs& a) {
#define FA_PASSES(P_, NT_) (a.rot.interleaved ? launch_append<E, D, true, P_, NT_>(a) : launch_append<E, D, false, P_, NT_>(a))
  const int at_once = std::min(a.N, a.cache.page_size) * Slot<D>::TPR;   // threads for a page's new rows at once
  if (at_once <= 64) return FA_PASSES(1, 64);
  if (at_once <= 128) return FA_PASSES(1, 128);
  if (at_once <= 256) return FA_PASSES(1, 256);
  if constexpr (D > 32)
    if (at_once > 512) {
      if constexpr (D > 64)
        if (at_once > 1024) return FA_PASSES(4, 512);
      return FA_PASSES(4, 256);
    }
  return FA_PASSES(2, 256);
#undef FA_PASSES
}

// How a call's rows and keys are cut: blocks of `rows` rows (16 and 32 to the kernel of few rows), each block's
// keys in up to nsplit parts of whole `step`s.  Only the lengths' bound (the table's width) is known here; a shorter
// sequence takes fewer parts (split_keys).
struct Cut {
  int rows, step, row_blocks, nsplit;
};

// The shape and the parts of the least cost by the times below: a workgroup's start, a step of its keys where each CU
// holds one workgroup, and on a full CU what each workgroup adds, a step and by itself; the join with its partial rows.
// For more than 16 rows they come within 15 % (rms) of the good ones among 1500 cuts of 150 calls (2 to 3000 new tokens,
// D = 32, 64 and 128), and the cut taken is 2 % slower than the best of its call on average, 22 % at most.
// Small blocks spread a short prompt over the CUs, large ones convert each key for more rows (us of blocks of 16 / 32 / 128 / 256
// rows, D = 128, one sequence, H=32 H_kv=8, no keys before: 64 new tokens 6.4 / 7.7 / 7.4 / 9.4, 512 18.2 / 14.0 / 16.7 /
// 20.5, 2048 119 / 75 / 53 / 57; two of 2048 235 / 151 / 87 / 77; blocks of 64 rows on four waves lay behind one of the
// others everywhere).  Parts fill the CUs and no more (up to 16 rows, us at 1 / 2 / 4 workgroups to a CU, 8 sequences of
// 1335 to 4005 keys, 8 K/V heads, D = 128: 17.4 / 20.7 / 26.4; one of 16000 keys 13.8 / 15.5 / 24.9), less where the keys are
// few (16 sequences of 160 keys, one K/V head, D = 32: filled 9.3, whole 5.5), and for lengths that differ up to four
// workgroups to a CU where a part keeps 4096 keys (32 sequences of 5461 to 16384 keys 140.9 / 141.9 / 135.3).
struct Shape {
  int rows, step;
  float start, one, full, each;   // us; steps at D = 128
};
constexpr Shape kShapes[] = {{16, kSplitStep, 6.f, 0.8f, 0.8f, 0.7f},
                             {32, kSplitStep, 7.f, 0.9f, 1.0f, 0.7f},
                             {128, kBlockKeys, 6.5f, 1.2f, 1.05f, 0.7f},
                             {256, kBlockKeys, 7.f, 1.8f, 1.9f, 3.0f}};
constexpr unsigned kParts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, kMaxSplit};

Cut cut_of(int B, int H, int Hkv, int N, int D, long long keys) {
  const long long rows = (long long)N * (H / Hkv), units = (long long)B * Hkv;
  const long long cus = cu_count();
  Cut c{16, kSplitStep, 1, 1};
  const long long least = rows <= 16 ? std::min<long long>({(4 * cus + units - 1) / units, keys / 4096, kMaxSplit}) : 1;
  const float seen = 1.f - 0.5f * (float)std::min<long long>(N, keys) / (float)keys;   // of the keys, by a row on average
  const float wide = (float)(D + 32) / 160.f, row_values = 2.5e-6f * (float)(units * rows) * (float)D;
  float best = 0.f;
  for (const Shape& s : kShapes) {
    if (s.rows > 16 && s.rows >= 2 * rows) break;
    const long long blocks = (rows + s.rows - 1) / s.rows;
    const unsigned most = (unsigned)std::min<long long>((keys + s.step - 1) / s.step, 1u << 30);
    bool first = true;
    for (const unsigned part : kParts) {
      const unsigned n = std::min(part, most);
      const long long wgs = units * blocks * n;
      if (n < least && n < most) continue;
      if (!first && wgs > 4 * cus) break;
      first = false;
      const float load = (float)wgs / (float)cus, steps = (float)((most + n - 1) / n) * wide;
      const float on_cu = s.rows <= 32 ? load : (float)(long long)(load + 0.999f);   // (one of the large at a time)
      const float work = std::max(steps * s.one, (steps * seen * s.full + s.each) * on_cu);
      const float us = s.start + work + (n == 1 ? 0.f : 2.5f + row_values * (float)n);
      if (best == 0.f || us < best) best = us, c = Cut{s.rows, s.step, (int)blocks, (int)n};
      if (n == most) break;
    }
  }
  return c;
}

size_t part_bytes(int B, int Hkv, const Cut& c, int D) {
  return c.nsplit <= 1 ? 0 : (size_t)B * Hkv * c.row_blocks * c.nsplit * c.rows * (D + 4) * sizeof(float);
}

template <typename E, int D>
int launch_attend(const PagedArgs& a, const Cut& c, int dtype) {
  const long long parts = (long long)a.B * a.cache.H_kv * a.nsplit;
  const long long grid = (c.rows <= 32 && by_xcd(parts) ? (parts + 7) / 8 * 8 : parts) * c.row_blocks;
  const long long joins = (long long)a.B * a.H * a.N;
  if (!grid_fits(grid, c.rows <= 32 ? 64 * kWaves : 2 * c.rows)) return FA_ERR_DIMS;
  if (a.nsplit > kFewSplits && !grid_fits(joins, kJoinThreads)) return FA_ERR_DIMS;
  hipStream_t st = (hipStream_t)a.stream;
  if (c.rows == 16) {
    hipLaunchKernelGGL((attend_kernel<E, D, 1>), dim3((unsigned)grid), dim3(64 * kWaves), 0, st, a, c.row_blocks);
  } else if (c.rows == 32) {
    hipLaunchKernelGGL((attend_kernel<E, D, 2>), dim3((unsigned)grid), dim3(64 * kWaves), 0, st, a, c.row_blocks);
  } else {
    const int status = paged_rows(dtype, a, c.row_blocks, c.rows);
    if (status != FA_OK) return status;
  }
  if (a.nsplit > kFewSplits)
    hipLaunchKernelGGL((join_kernel<E, D>), dim3((unsigned)joins), dim3(kJoinThreads), 0, st, a, c.row_blocks, c.rows, c.step);
  else if (a.nsplit > 1)
    hipLaunchKernelGGL((join_few_kernel<E, D>), dim3((unsigned)((joins + 1024 / D - 1) / (1024 / D))), dim3(kJoinThreads), 0,
                       st, a, c.row_blocks, c.rows, c.step);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int attend(int dtype, PagedArgs a, const Cut& c) {
  a.nsplit = c.nsplit;
  if (dtype == FA_BF16) {
    if (a.D == 32) return launch_attend<BF16, 32>(a, c, dtype);
    if (a.D == 64) return launch_attend<BF16, 64>(a, c, dtype);
    return launch_attend<BF16, 128>(a, c, dtype);
  }
  if (a.D == 32) return launch_attend<F16, 32>(a, c, dtype);
  if (a.D == 64) return launch_attend<F16, 64>(a, c, dtype);
  return launch_attend<F16, 128>(a, c, dtype);
}

}  // namespace

int paged_append(int dtype, const AppendArgs& a) {
  if (dtype == FA_BF16) {
    if (a.D == 32) return launch_append<BF16, 32>(a);
    if (a.D == 64) return launch_append<BF16, 64>(a);
    return launch_append<BF16, 128>(a);
  }
  if (a.D == 32) return launch_append<F16, 32>(a);
  if (a.D == 64) return launch_append<F16, 64>(a);
  return launch_append<F16, 128>(a);
}

int paged_attention(int dtype, PagedArgs a, size_t workspace_bytes) {
  const int Hkv = a.cache.H_kv;
  Cut c = cut_of(a.B, a.H, Hkv, a.N, a.D, (long long)a.cache.table_width * a.cache.page_size);
  while (c.nsplit > 1 && part_bytes(a.B, Hkv, c, a.D) > workspace_bytes) --c.nsplit;
  return attend(dtype, a, c);
}

int paged_attention_exact(int dtype, PagedArgs a, int block_rows, int parts, size_t workspace_bytes) {
  const Shape* const s = std::find_if(std::begin(kShapes), std::end(kShapes), [&](const Shape& x) { return x.rows == block_rows; });
  if (s == std::end(kShapes)) return FA_ERR_TILE;
  if (parts < 1 || parts > kMaxSplit) return FA_ERR_UNSUPPORTED;
  const long long rows = (long long)a.N * (a.H / a.cache.H_kv);
  const Cut c{block_rows, s->step, (int)((rows + block_rows - 1) / block_rows), parts};
  return part_bytes(a.B, a.cache.H_kv, c, a.D) > workspace_bytes ? FA_ERR_WORKSPACE : attend(dtype, a, c);
}

size_t paged_attention_workspace(int B, int H, int Hkv, int N, int D, long long keys) {
  return part_bytes(B, Hkv, cut_of(B, H, Hkv, N, D, keys), D);
}

}  // namespace fa
