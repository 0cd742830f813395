// fa_paged_rows.hip - attention over the paged 8-bit cache for many rows: pieces of prompts
// (the mathematics: fa_paged.h; few rows: fa_paged.hip).
//
// The matrix instructions bound it, so the codes become 16-bit values once per workgroup and not once
// per wave: a workgroup of 4 waves takes 128 rows (32 to a wave; row r = token r / G, query head r % G
// of one K/V head, so neighbouring rows share every key), walks the keys in tiles of 64, and keeps two
// tiles of K (in the queries' type) and V (fp16) in LDS.  A tile's codes come to registers while the tile
// before them is computed, are converted (2 codes an instruction) and written to LDS under the products of
// the next step, and are read in the step after it: no wave waits for them between two products.  8 waves and
// 256 rows where there are as many: each converted tile serves twice the rows.  Products, layouts and order of a
// step are those of the causal forward (fa_fwd.hip): S^T = K Q^T on 32x32x16 products with a lane owning one row,
// the scores fed back as the B operand of O^T += V^T P^T, V^T read transposed from LDS, S(j + 1) under the softmax
// of S(j).  B=2 H=32 H_kv=8, 2048 new tokens behind 6144, D=128: 418-449 us by machine,
// 1070-1150 TFLOP/s, the matrix pipes busy 56 % of the time at 1.94 GHz.  What differs:
//   * a 16-key part of a tile (the whole tile with pages of 64 keys or more) lies in one page: its K scale
//     multiplies its scores, its V scale joins their exponent, and leaves the row sums again, part by part;
//   * pages and scales of 16 tiles (64 with pages of 64 keys or more) at a time are kept one part to a lane
//     and loaded a run ahead;
//   * the diagonal starts at past_lens: tiles below it run without a mask; a value of V behind the last
//     key is stored as zero, and a NaN in a masked tile is dealt with behind the loop (fa_paged.h).
#include "fa_paged.h"

namespace fa {

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

constexpr float kRowSumLimit = 32768.f;   // 2^kLazy: no p' passes fp16's range

// PPT: parts of a tile that may lie in different pages (1: pages of 64 keys or more; else 4, of 16 keys).
template <typename E, int D, int NW, int PPT>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2)))
void rows_kernel(PagedArgs a, int row_blocks) {
  constexpr int BM = 32 * NW, BN = kBlockKeys, NB = BN / 32, NT = 64 * NW;
  constexpr int KT = D / 16;                 // MFMA k-steps over D
  constexpr int DB = D / 32;                 // 32-row blocks of O^T
  constexpr int ROWB = D * 2;                // bytes per K / V row in LDS
  constexpr int TILE = BN * ROWB;
  constexpr int CPR = ROWB / 16;             // 16-byte chunks per row
  constexpr int PCR = D / 16;                // 16-code pieces per row
  constexpr int PIECES = BN * PCR;
  constexpr int PT = (PIECES + NT - 1) / NT; // pieces per thread, K and V each
  constexpr int RUN = 64 / PPT;              // tiles whose parts fill the lanes of a wave
  constexpr int PART = BN / PPT;             // keys of a part
  const float NEG_INF = -__builtin_inff();
  // K buffers at [0, 2 TILE), V buffers at [2 TILE, 4 TILE)
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * TILE];
  __shared__ int nan_met;                    // a masked tile of V held a NaN

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const int Hkv = a.cache.H_kv, ps = a.cache.page_size, G = a.H / Hkv;
  const int page_bits = 31 - __builtin_clz(ps);   // (a power of two)

  // Workgroups reach the XCDs in turn (wg % 8): XCD x takes a contiguous range of (batch, K/V head)
  // units, so their pages stay in its L2, and of each the last rows, whose keys are the most, first.
  const int nunits = a.B * Hkv;
  const int wg = blockIdx.x, split = wg % a.nsplit, item = wg / a.nsplit;
  int unit, rb;
  if (nunits % 8 == 0 && a.nsplit == 1) {
    const int per = nunits / 8, i = item / 8;
    unit = (item % 8) * per + i / row_blocks;
    rb = row_blocks - 1 - i % row_blocks;
  } else {
    unit = item % nunits;
    rb = row_blocks - 1 - item / nunits;
  }
  const int b = unit / Hkv, hk = unit % Hkv;
  const Block x = block_of(a, b, rb, G, BM);
  const int per = split_keys(x.keys, a.nsplit, BN);
  const int first = split * per, last = min(first + per, x.keys);
  if (split > 0 && first >= x.keys) return;    // (the first split also writes what has no keys)
  const int ntiles = last > first ? (last - first + BN - 1) / BN : 0;
  // tiles that every live row sees whole
  const int jfull = min(max((x.lmin + 1 - first) / BN, 0), ntiles);

  const int rl = wave * 32 + c;                // this lane's row in the block
  const int r = min(x.r0 + rl, x.rows - 1), tok = r / G, head = hk * G + r % G;
  const bool real = x.r0 + rl < x.rows, live = real && tok < x.fresh;
  const int lim = live ? x.past + tok : x.lmin;   // the last key it sees (rows without one: as the first)

  u32x4 qf[KT];
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q.data) + b * a.q.stride_b + head * a.q.stride_h +
                        tok * a.q.stride_n + 8 * hh;
#pragma unroll
    for (int t = 0; t < KT; ++t) qf[t] = gload16(q + 16 * t);
  }

  // ---- pages and scales: lane i holds those of part i of the run of RUN tiles from run0, and of the next run
  struct Parts {
    uint32_t lo, hi;   // offset of its first row in the pools
    int ve;
    float ks;
  };
  Parts cur{}, nxt{};
  auto part_page = [&](int t0) __attribute__((always_inline)) {   // of the run that starts at tile t0
    // (parts behind the last key: its page, so no other page's scale has a say)
    return page_of(a.cache, b, min(first + t0 * BN + PART * lane, last - 1) >> page_bits);
  };
  auto part_place = [&](Parts& p, int t0, int page) __attribute__((always_inline)) {
    const int key = first + t0 * BN + PART * lane;
    const uint64_t at = ((((uint64_t)max(page, 0) * Hkv + hk) << page_bits) + (key & (ps - 1))) * D;
    p.lo = (uint32_t)at, p.hi = (uint32_t)(at >> 32);
  };
  auto part_scales = [&](Parts& p, int page) __attribute__((always_inline)) {
    const long long ph = (long long)max(page, 0) * Hkv + hk;
    const int ke = scale_of(a.cache.k_scale, ph), ve = scale_of(a.cache.v_scale, ph);
    p.ks = page < 0 ? __builtin_nanf("") : exp2i(ke) * a.scale_log2;   // (no page: its rows become NaN)
    p.ve = page < 0 ? 0 : ve;
  };
  int run0 = 0;

  // ---- staging: piece i of this thread is 16 codes of row prow + i RP of a tile.  Rows i RP apart swizzle
  // alike, and the two 16-byte halves of a converted piece lie 16 bytes apart (one bit of the offset).
  constexpr int RP = NT / PCR;               // rows that the workgroup stages at once
  const int prow = tid / PCR % BN;           // (D <= 64: some threads have no piece)
  const uint32_t goff = prow % PART * D + tid % PCR * 16;
  const int kdst = prow * ROWB + (((tid % PCR * 2) ^ ((prow * CPR / 16) & (CPR - 1))) << 4);
  const int vdst = prow * ROWB + ((tid % PCR * 32) ^ ((32 * (prow & 3)) & (ROWB - 1)));
  const bool stages = PIECES >= NT || tid < PIECES;
  auto fetch = [&](const void* pool, int t, u32x4 (&w)[PT]) __attribute__((always_inline)) {
    const bool now = t - run0 < RUN;
    const uint32_t lo = now ? cur.lo : nxt.lo, hi = now ? cur.hi : nxt.hi;
    auto part = [&](int i) __attribute__((always_inline)) {
      const int from = ((t - run0) & (RUN - 1)) * PPT + i;
      const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32 |
                          (uint32_t)__builtin_amdgcn_readlane(lo, from);
      return static_cast<const uint8_t*>(pool) + at;
    };
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      // a piece's row lies in part row / PART, the same for a whole wave (16-key parts at D = 32: for half a wave)
      if constexpr (PPT == 1) {
        w[i] = *reinterpret_cast<const u32x4*>(part(0) + goff + i * RP * D);
      } else if constexpr (D == 32) {
        const int i0 = wave * (64 / PCR) / 16 % PPT;
        const uint8_t* const p0 = part(i0);
        const uint8_t* const p1 = part(i0 + 1);
        w[i] = *reinterpret_cast<const u32x4*>((lane < 32 ? p0 : p1) + goff);
      } else {
        w[i] = *reinterpret_cast<const u32x4*>(part((wave * (64 / PCR) % BN + i * RP) / 16) + goff);
      }
    }
  };
  auto put_k = [&](const u32x4 (&w)[PT], unsigned char* buf) __attribute__((always_inline)) {
    if (!stages) return;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      lds_write16(buf, kdst + i * RP * ROWB, codes8<E>(w[i][0], w[i][1]));
      lds_write16(buf, (kdst ^ 16) + i * RP * ROWB, codes8<E>(w[i][2], w[i][3]));
    }
  };
  auto put_v = [&](u32x4 (&w)[PT], int t, unsigned char* buf, auto full) __attribute__((always_inline)) {
    if (!stages) return;
    if (!decltype(full)::value && t >= jfull) {   // a masked tile: nothing behind the last key, no NaN
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        uint32_t any = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t v = first + t * BN + prow + i * RP >= x.keys ? 0u : w[i][n], nan = nan_bytes(v);
          w[i][n] = without_nan(v, nan);
          any |= nan;
        }
        if (any != 0) nan_met = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      lds_write16(buf, vdst + i * RP * ROWB, codes8<F16>(w[i][0], w[i][1]));
      lds_write16(buf, (vdst ^ 16) + i * RP * ROWB, codes8<F16>(w[i][2], w[i][3]));
    }
  };

  // ---- per-lane LDS operand offsets (fa_fwd.hip)
  int koff[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) koff[t] = c * ROWB + (((2 * t + hh) ^ ((c * CPR / 16) & (CPR - 1))) << 4);
  int voff_even, voff_odd;
  {
    const int g16 = lane >> 4, kr = (lane >> 2) & 3, c4 = lane & 3;
    const int e = 2 * pi_swap23(16 * (g16 & 1) + 4 * c4);
    const int k1 = (ROWB >= 128) ? (kr >> 1) : 0;
    const int base = (4 * hh + kr) * ROWB + (e ^ (32 * (kr & 1)));
    voff_even = base + 64 * k1;
    voff_odd = base + 64 * (1 - k1) - 64;
  }

  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
  float mrun = -__FLT_MAX__;
  float lsum = 0.f;   // of this lane's half of the keys

  auto s_tile = [&](const unsigned char* Ks, f32x16 (&s)[NB]) __attribute__((always_inline)) {
    f32x16 y[NB] = {};
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) y[nb] = mfma32<E>(lds_read16(Ks, koff[t] + nb * 32 * ROWB), qf[t], y[nb]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = y[nb];
  };
  auto mask_tile = [&](f32x16 (&s)[NB], int k0) __attribute__((always_inline)) {
    const int t = lim - k0 - 4 * hh;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int g = 0; g < 16; ++g)
        if (32 * nb + 8 * (g >> 2) + (g & 3) > t) s[nb][g] = NEG_INF;
  };
  // scales of part i of tile t
  auto k_scale = [&](int t, int i) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(cur.ks), (t - run0) * PPT + i));
  };
  auto v_exp = [&](int t, int i) __attribute__((always_inline)) {
    return __builtin_amdgcn_readlane(cur.ve, (t - run0) * PPT + i);
  };
  auto tile_max = [&](const f32x16 (&s)[NB], int t) __attribute__((always_inline)) {
    float top = NEG_INF;
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      float mx = NEG_INF;
#pragma unroll
      for (int g = 0; g < 32 / PPT; ++g) mx = fmaxf(mx, s[(32 / PPT * i + g) / 16][(32 / PPT * i + g) % 16]);
      top = fmaxf(top, __builtin_fmaf(mx, k_scale(t, i), (float)v_exp(t, i)));
    }
    return halfwave_max(top);
  };
  auto rescale_to = [&](float mx) __attribute__((always_inline)) {
    const float mnew = mx > mrun + kLazy ? mx - kBelow : mrun;   // (a row's own scores alone move it)
    const float alpha = fast_exp2(mrun - mnew);
    mrun = mnew;
    lsum *= alpha;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[db][g] *= alpha;
  };
  // P^T of the tile against mrun; the row's sum of it (this lane's half), and in l that with the V scales
  // taken out.  Both in fp32 from p as it is: where scales lie far apart a key that counts may have a p' that
  // fp16 rounds to nothing.  (On the matrix pipe, from P as rounded, the sums would also hang on the other rows
  // of their column: its zeros hand on a NaN.)
  // (Masked: a key that the row does not see counts for nothing, also where it has no page and its scale is NaN.)
  auto exp_tile = [&](const f32x16 (&s)[NB], int t, u32x4 (&pk)[2 * NB], float& l, auto full) __attribute__((always_inline)) {
    float sum = 0.f;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < PPT; ++k) {
      const int ve = v_exp(t, k);
      const float ks = k_scale(t, k), off = (float)ve - mrun;
      float y = 0.f;
#pragma unroll
      for (int i = 2 * NB / PPT * k; i < 2 * NB / PPT * (k + 1); ++i) {
        float p[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float x = s[i / 2][8 * (i & 1) + g];
          p[g] = fast_exp2(__builtin_fmaf(x, ks, off));
          if (!decltype(full)::value && x == NEG_INF) p[g] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) pk[i][q] = pack2<F16>(p[2 * q], p[2 * q + 1]);
        y += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      }
      sum += y;
      l = __builtin_fmaf(y, exp2i(-ve), l);
    }
    return sum;
  };
  auto softmax = [&](const f32x16 (&s)[NB], int t, u32x4 (&pk)[2 * NB], auto full) __attribute__((always_inline)) {
    float l;
    const float sum = exp_tile(s, t, pk, l, full);
    if (__builtin_amdgcn_ballot_w64(!(sum <= kRowSumLimit))) {
      rescale_to(tile_max(s, t));
      exp_tile(s, t, pk, l, full);
    }
    lsum += l;
  };

  constexpr int NPV = DB * 2 * NB;
  u32x4 pvb[3];
  auto pv_read = [&](const unsigned char* Vs, int i) __attribute__((always_inline)) {
    const int db = i % DB, u = i / DB;
    const int o = ((db & 1) ? voff_odd : voff_even) + 64 * db + 16 * u * ROWB;
    return lds_read_tr16x2(Vs, o, o + 8 * ROWB);
  };
  auto pv_pre = [&](const unsigned char* Vs) __attribute__((always_inline)) {
    pvb[0] = pv_read(Vs, 0);
    pvb[1] = pv_read(Vs, 1);
  };
  auto pv_full = [&](const unsigned char* Vs, const u32x4 (&pk)[2 * NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NPV; ++i) {
      if (i + 2 < NPV) pvb[(i + 2) % 3] = pv_read(Vs, i + 2);
      acc[i % DB] = mfma32<F16>(pvb[i % 3], pk[i / DB], acc[i % DB]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto Kbuf = [&](int j) __attribute__((always_inline)) { return lds + (j & 1) * TILE; };
  auto Vbuf = [&](int j) __attribute__((always_inline)) { return lds + 2 * TILE + (j & 1) * TILE; };

  if (ntiles > 0) {
    if (tid == 0) nan_met = 0;
    int nxt_page = part_page(0);
    part_place(cur, 0, nxt_page);
    part_scales(cur, nxt_page);
    u32x4 rk[PT], rv[PT];
    __syncthreads();
    fetch(a.cache.k, 0, rk);
    fetch(a.cache.v, 0, rv);
    put_k(rk, Kbuf(0));
    put_v(rv, 0, Vbuf(0), Flag<false>{});
    if (ntiles > 1) {
      fetch(a.cache.k, 1, rk);
      put_k(rk, Kbuf(1));
    }
    __syncthreads();
    fetch(a.cache.k, 2, rk);
    fetch(a.cache.v, 1, rv);
    f32x16 sa[NB], sb[NB];
    s_tile(Kbuf(0), sa);
    if (jfull == 0) mask_tile(sa, first);
    mrun = fmaxf(tile_max(sa, 0) - kBelow, -__FLT_MAX__);

    auto body = [&](int j, const unsigned char* __restrict__ kcur, unsigned char* __restrict__ kdst_,
                    const unsigned char* __restrict__ vcur, unsigned char* __restrict__ vdst_, f32x16 (&sc)[NB],
                    f32x16 (&sn)[NB], auto full) __attribute__((always_inline)) {
      constexpr bool FULL = decltype(full)::value;
      // (past the last tile what is written is not read, and what is fetched lies in some page)
      put_k(rk, kdst_);
      put_v(rv, j + 1, vdst_, full);
      fetch(a.cache.k, j + 3, rk);
      fetch(a.cache.v, j + 2, rv);
      u32x4 pk[2 * NB];
      s_tile(kcur, sn);
      if constexpr (!FULL) mask_tile(sn, first + (j + 1) * BN);
      pv_pre(vcur);
      softmax(sc, j, pk, full);
      pv_full(vcur, pk);
    };
    auto iteration = [&](int j, f32x16 (&sc)[NB], f32x16 (&sn)[NB], auto full) __attribute__((always_inline)) {
      // a run's pages are asked for at its predecessor's start, their scales half a run later
      if (j % RUN == 0) {
        if (j > 0) cur = nxt, run0 = j;
        nxt_page = part_page(j + RUN);
        part_place(nxt, j + RUN, nxt_page);
      } else if (j % RUN == RUN / 2) {
        part_scales(nxt, nxt_page);
      }
      __syncthreads();
      body(j, Kbuf(j + 1), Kbuf(j), Vbuf(j), Vbuf(j + 1), sc, sn, full);
    };

    // tiles j with j + 2 < jfull: S(j), S(j + 1) and the V tile j + 1 unmasked
    int j = 0;
    for (; j + 2 < jfull; j += 2) {
      iteration(j, sa, sb, Flag<true>{});
      iteration(j + 1, sb, sa, Flag<true>{});
    }
    for (; j + 1 < ntiles; ++j) {
      iteration(j, sa, sb, Flag<false>{});
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sa[nb] = sb[nb];
    }
    if (j % RUN == 0 && j > 0) cur = nxt, run0 = j;
    __syncthreads();
    u32x4 pk[2 * NB];
    pv_pre(Vbuf(j));
    softmax(sa, j, pk, Flag<false>{});
    pv_full(Vbuf(j), pk);

    if (__builtin_amdgcn_readfirstlane(nan_met) != 0) {
      for (int t = jfull; t < ntiles; ++t) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          const int key = first + t * BN + prow + i * RP;
          const long long page = key < x.keys ? max(page_of(a.cache, b, key >> page_bits), 0) : 0;
          const uint8_t* const p = static_cast<const uint8_t*>(a.cache.v) + ((page * Hkv + hk) * ps + (key & (ps - 1))) * D + tid % PCR * 16;
          const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
          for (int n = 0; n < 4; ++n) rv[i][n] = key < x.keys ? nan_as_one(w[n]) : 0u;
        }
        put_v(rv, t, Vbuf(0), Flag<true>{});
        __syncthreads();
        f32x16 count[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) count[db] = f32x16{};
        const int left = lim - (first + t * BN) - 4 * hh;
#pragma unroll
        for (int u = 0; u < 2 * NB; ++u) {
          u32x4 seen;
#pragma unroll
          for (int q = 0; q < 4; ++q) {   // slots 2 q, 2 q + 1: keys 16 u + 4 hh + {0..3} and + 8
            const int k = 16 * u + 8 * (q / 2) + 2 * (q % 2);
            seen[q] = (k <= left ? 0x3C00u : 0u) | (k + 1 <= left ? 0x3C000000u : 0u);
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) count[db] = mfma32<F16>(pv_read(Vbuf(0), u * DB + db), seen, count[db]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 16; ++g)
            if (count[db][g] > 0.f) acc[db][g] = __builtin_nanf("");
      }
    }
  }

  // ---- epilogue: lane holds d = 32 db + 16 i1 + 8 hh + 0..7 of its row
  const float l = halfwave_sum(lsum);
  if (!real) return;
  if (per < x.keys) {   // more than one split: the join divides
    float* const dst = part_row<D>(a, (long long)unit * row_blocks + rb, split, rl, BM);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 16; g += 4)
        gstore_f32x4(dst + 32 * db + 16 * (g / 8) + 8 * hh + g % 8,
                     f32x4{acc[db][g], acc[db][g + 1], acc[db][g + 2], acc[db][g + 3]});
    if (hh == 0) dst[D] = mrun, dst[D + 1] = l;
    return;
  }
  const float inv = live ? 1.0f / l : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(a.o.data)) + b * a.o.stride_b + head * a.o.stride_h + tok * a.o.stride_n;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i1 = 0; i1 < 2; ++i1)
      gstore16(dst + 32 * db + 16 * i1 + 8 * hh, live ? pack8<E>(acc[db], 8 * i1, inv) : u32x4{});
  if (a.lse != nullptr && hh == 0)
    a.lse[((long long)b * a.H + head) * a.N + tok] = live ? mrun + __log2f(l) : NEG_INF;
}

namespace {

template <typename E, int D>
int launch_rows(const PagedArgs& a, int row_blocks, int block_rows) {
  const dim3 g((unsigned)((long long)a.B * a.cache.H_kv * row_blocks * a.nsplit)), t(2 * block_rows);
  hipStream_t st = (hipStream_t)a.stream;
  const bool whole = a.cache.page_size >= kBlockKeys;   // a tile in one page
  if (block_rows == 128) {
    if (whole) hipLaunchKernelGGL((rows_kernel<E, D, 4, 1>), g, t, 0, st, a, row_blocks);
    else hipLaunchKernelGGL((rows_kernel<E, D, 4, 4>), g, t, 0, st, a, row_blocks);
  } else {
    if (whole) hipLaunchKernelGGL((rows_kernel<E, D, 8, 1>), g, t, 0, st, a, row_blocks);
    else hipLaunchKernelGGL((rows_kernel<E, D, 8, 4>), g, t, 0, st, a, row_blocks);
  }
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // namespace

int paged_rows(int dtype, const PagedArgs& a, int row_blocks, int block_rows) {
  if (dtype == FA_BF16) {
    if (a.D == 32) return launch_rows<BF16, 32>(a, row_blocks, block_rows);
    if (a.D == 64) return launch_rows<BF16, 64>(a, row_blocks, block_rows);
    return launch_rows<BF16, 128>(a, row_blocks, block_rows);
  }
  if (a.D == 32) return launch_rows<F16, 32>(a, row_blocks, block_rows);
  if (a.D == 64) return launch_rows<F16, 64>(a, row_blocks, block_rows);
  return launch_rows<F16, 128>(a, row_blocks, block_rows);
}

}  // namespace fa
