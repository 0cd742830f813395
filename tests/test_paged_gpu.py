"""The 8-bit paged cache's append and the attention over it on the GPU, against the float64 oracle.

Bars: codes and scales are equal bit for bit where the values are (no norm, no rotation: V always);
with them, a value is off by half a step of e4m3 (2^-4, or 2^-10 of its scale) and by the rounding of 16
fp32 operations.  The attention: oracle.paged_oracle.attend's bound, and its own rounding to the output type.
"""

import math

import pytest
import torch

from attention.gqa.fused_gqa import fused_gqa_attention
from attention.paged.fused_paged import PagedKV, append_paged_kv, fused_paged_attention, paged_kv_cache
from attention.rotary.fused_rotary import fused_qk_norm_rotary, rotary_table
from oracle import paged_oracle as orc
from gpu_util import log

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
EPS = 1e-6
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(shape, generator=gen(seed), device="cuda")


def filled(pages, H, ps, D, seed, spread=0, low=118):
    """A cache of random values; scales 2^(low - 127) to `spread` steps more."""
    k, v = (randn(seed + i, pages, H, ps, D).mul(60).to(F8) for i in range(2))
    e = torch.randint(low, low + spread + 1, (2, pages, H), generator=gen(seed + 2), device="cuda", dtype=torch.uint8)
    return PagedKV(k, v, e[0].view(E8).contiguous(), e[1].view(E8).contiguous())


def tables(B, width, pages, seed):
    assert B * width <= pages
    return torch.randperm(pages, generator=gen(seed), device="cuda")[:B * width].view(B, width).int()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_attend(q, cache, bt, past, new=None, label=""):
    """o and lse of a call against the oracle, sequence by sequence; returns o."""
    B, H, N, D = q.shape
    o, lse = fused_paged_attention(q, cache, bt, past, new, return_lse=True)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (B, H, N)
    c = orc.Cache(*cache)
    worst = 0.0
    for b in range(B):
        n = int(new[b]) if new is not None else N
        want, want_lse, bound = orc.attend(q[b].cpu(), c, bt[b:b + 1].cpu(), int(past[b]), n)
        got, got_lse = o[b].double().cpu(), lse[b].double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), (label, b)
        tol = bound + want.abs() * HALF[q.dtype] + LEAST[q.dtype]
        ratio = torch.nan_to_num((got - want).abs() / tol.clamp_min(1e-300))
        worst = max(worst, float(ratio.max()))
        assert worst <= 1.0, (label, b, worst)
        fin = torch.isfinite(want_lse)
        assert torch.equal(fin, torch.isfinite(got_lse)), (label, b)
        # the weights' relative error bounds that of their sum: in log2, that over ln 2; and fp32's last bits
        err = (got_lse - want_lse)[fin].abs()
        assert bool((err <= 2.0 ** -9 + want_lse[fin].abs() * 2.0 ** -22).all()), (label, b, float(err.max()))
    log(f"{label} worst/bar {worst:.2f}")
    return o


# ---- attention

@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_types_and_pages(D, dt, ps):
    B, H, Hkv, width = 3, 6, 2, 3
    cache = filled(12, Hkv, ps, D, D + ps, spread=6)
    bt = tables(B, width, 12, ps)
    log(f"attend D={D} {dt} page {ps}")
    for N, past in ((1, (0, ps - 1, 3 * ps - 1)), (5, (0, ps - 2, 2 * ps + 3))):
        q = randn(N, B, H, N, D).mul(0.7).to(dt)
        check_attend(q, cache, bt, ints(*past), label=f"N={N}")


@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 5), (8, 1), (32, 1), (10, 2), (24, 8), (16, 2)])
@pytest.mark.parametrize("N", [1, 2, 7, 33, 150])
def test_attention_heads_and_rows(H, Hkv, N):
    D, ps, width = 64, 32, 16
    cache = filled(2 * width, Hkv, ps, D, H + N, spread=4)
    bt = tables(2, width, 2 * width, N)
    log(f"attend H={H} Hkv={Hkv} N={N}")
    q = randn(N + 1, 2, H, N, D).bfloat16()
    check_attend(q, cache, bt, ints(width * ps - N, 13))


@pytest.mark.parametrize("total", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 700, 1500])
def test_attention_lengths(total):
    cache = filled(100, 1, 16, 128, total, spread=3)
    bt = tables(1, 100, 100, total)
    for N in (1, 3, 7, 13, 25, 70):   # 4 to 280 rows: every size of row block
        if N <= total:
            q = randn(total + N, 1, 4, N, 128).to(torch.float16)
            check_attend(q, cache, bt, ints(total - N), label=f"total={total} N={N}")


@pytest.mark.parametrize("N", [4, 9, 18, 100])
def test_padded_batch_and_empty_sequences(N):
    cache = filled(64, 2, 16, 64, 1, spread=2)
    bt = tables(4, 16, 64, 2)
    q = randn(3, 4, 6, N, 64).bfloat16()
    new = ints(N, 0, N - 1, 1)
    o = check_attend(q, cache, bt, ints(7, 50, 0, 0), new)
    assert float(o[1].float().abs().max()) == 0 and float(o[2, :, N - 1:].float().abs().max()) == 0
    # values outside [0, N] and below 0 count as the nearer bound
    a = fused_paged_attention(q, cache, bt, ints(7, 50, -3, 0), ints(N + 9, -1, N - 1, 1))
    assert torch.equal(a, fused_paged_attention(q, cache, bt, ints(7, 50, 0, 0), new))


@pytest.mark.parametrize("N", [1, 3, 7, 14, 20, 90])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_what_lies_behind_a_rows_last_key_does_not_touch_it(dt, N):
    cache = filled(24, 1, 16, 64, 3, spread=3)
    bt = tables(2, 10, 24, 3)
    past = ints(35, 2)
    q = randn(4, 2, 4, N, 64).to(dt)
    want = fused_paged_attention(q, cache, bt, past)
    codes = [c.view(torch.uint8) for c in cache[:2]]
    for b, p in enumerate((35, 2)):
        total = p + N
        for c in codes:   # NaN behind the last key, in its page and in the next
            c[bt[b, total // 16].long(), :, total % 16:] = 0x7F
            c[bt[b, total // 16 + 1].long()] = 0xFF
    bt2 = bt.clone()
    bt2[0, (35 + N) // 16 + 1:] = -1   # and no page at all
    bt2[1, (2 + N) // 16 + 2:] = 9999
    assert torch.equal(fused_paged_attention(q, cache, bt2, past), want)
    if N > 1:
        # a NaN inside the new tokens reaches the rows that see it, in its own dim, and no other row
        last = 35 + N - 1
        codes[1][bt[0, last // 16].long(), 0, last % 16, 5] = 0x7F
        mid = 35 + N // 2
        codes[0][bt[0, mid // 16].long(), 0, mid % 16, 3] = 0xFF
        o = check_attend(q, cache, bt2, past)
        assert torch.equal(o[0, :, :N // 2], want[0, :, :N // 2]) and torch.equal(o[1], want[1])
        assert torch.isnan(o[0, :, N // 2:]).all()


@pytest.mark.parametrize("N", [1, 90])
def test_pages_that_hold_nothing_yet(N):
    """The tiles behind a row's last key read some page, whatever bytes its scale has (0: an empty cache's)."""
    cache = filled(10, 2, 16, 128, 8)
    bt = torch.arange(1, 10, device="cuda").int()[None]
    q = randn(9, 1, 4, N, 128).bfloat16()
    want = check_attend(q, cache, bt, ints(100 - N))
    for byte in (0, 254, 255):
        for t in cache[2:]:
            t.view(torch.uint8)[0] = byte
            t.view(torch.uint8)[9] = byte
        cache.k.view(torch.uint8)[0] = 0x7F
        cache.v.view(torch.uint8)[0] = 0x7F
        assert torch.equal(fused_paged_attention(q, cache, bt, ints(100 - N)), want)


@pytest.mark.parametrize("H", [1, 2, 4, 16])
def test_nan_in_a_value_reaches_its_dim_alone(H):
    cache = filled(8, 1, 16, 64, 5)
    bt = tables(1, 8, 8, 5)
    q = randn(6, 1, H, 20, 64).bfloat16()
    cache.v.view(torch.uint8)[bt[0, 1].long(), 0, 3, 7] = 0x7F     # key 19, seen by all rows
    cache.v.view(torch.uint8)[bt[0, 6].long(), 0, 4, 9] = 0xFF     # key 100, seen by tokens 10 on
    o = check_attend(q, cache, bt, ints(90))
    nan = torch.isnan(o[0])
    assert nan[:, :, 7].all() and nan[:, 10:, 9].all() and int(nan.sum()) == H * 20 + H * 10


def test_pages_the_table_does_not_name():
    cache = filled(10, 1, 16, 32, 7)
    bt = tables(3, 3, 10, 7)
    bt[0, 1], bt[1, 0] = -1, 10
    q = randn(8, 3, 2, 4, 32).half()
    o = check_attend(q, cache, bt, ints(14, 5, 10))
    nan = torch.isnan(o)
    assert not nan[0, :, :2].any() and nan[0, :, 2:].all() and nan[1].all() and not nan[2].any()
    # a length past the table: no page there either
    o = fused_paged_attention(q, cache, bt, ints(14, 5, 46))
    assert not torch.isnan(o[2, :, :2]).any() and torch.isnan(o[2, :, 2:]).all()
    o = fused_paged_attention(q, cache, bt, ints(14, 5, 2 ** 31 - 1))
    assert torch.isnan(o[2]).all()


@pytest.mark.parametrize("N", [1, 12, 30, 50, 140])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_scales_far_apart_and_zero_pages(dt, N):
    """V pages at 2^-40 beside 2^10, pages of zeros (the least scale) among them, K scales apart too."""
    ps, D = 16, 64
    cache = filled(12, 2, ps, D, 9)
    ke, ve = (s.view(torch.uint8) for s in cache[2:])
    ve[:] = torch.randint(87, 138, ve.shape, generator=gen(1), device="cuda", dtype=torch.uint8)
    ke[:] = torch.randint(87, 122, ke.shape, generator=gen(2), device="cuda", dtype=torch.uint8)
    zero = torch.tensor([1, 4, 5], device="cuda")
    cache.v.view(torch.uint8)[zero] = 0
    ve[zero] = 87
    bt = tables(1, 12, 12, 9)
    q = randn(10, 1, 4, N, D).to(dt)
    check_attend(q, cache, bt, ints(12 * ps - N))
    ke[:] = 87        # every key alike: the weights are even, zeros and tiny pages count in full
    check_attend(q, cache, bt, ints(12 * ps - N))


def test_long_flat_tail_keeps_its_weight():
    """One key 2^15 to 2^18 above 20000 equal ones, whose weights are far below its own."""
    ps, D, n = 64, 64, 20000
    cache = paged_kv_cache(320, 1, ps, D)
    cache.k.view(torch.uint8).zero_()
    cache.v.copy_(randn(1, 320, 1, ps, D).to(F8))
    cache.v.view(torch.uint8)[0, 0, 0] = 0x30
    for s in cache[2:]:
        s.view(torch.uint8).fill_(127)
    bt = torch.arange(320, device="cuda").int()[None]
    for top in (15.3, 17.7):
        q = torch.zeros(1, 1, 1, D, device="cuda", dtype=torch.bfloat16)
        q[..., 0] = 1.0
        cache.k[0, 0, 0] = 0
        cache.k[0, 0, 0, 0] = top * math.sqrt(D) * math.log(2.0)
        check_attend(q, cache, bt, ints(n - 1), label=f"tail under 2^{top}")


def test_sharp_rows_and_one_key():
    cache = filled(40, 2, 16, 128, 11, low=122)
    bt = tables(1, 40, 40, 11)
    for N in (1, 50):
        check_attend(randn(12, 1, 8, N, 128).mul(6).bfloat16(), cache, bt, ints(640 - N), label="sharp")
    q = randn(13, 1, 4, 1, 128).bfloat16()
    o = fused_paged_attention(q, cache, bt, ints(0))
    v = (cache.v.float() * torch.exp2(cache.v_scale.view(torch.uint8).float() - 127)[..., None, None])[bt[0, 0].long(), :, 0]
    assert torch.equal(o[0, :, 0], v.repeat_interleave(2, 0).bfloat16())


@pytest.mark.parametrize("N", [1, 6, 120])
def test_strides_of_the_queries(N):
    cache = filled(24, 2, 16, 64, 14)
    bt = tables(2, 12, 24, 14)
    past = ints(192 - N, 11)
    dense = randn(15, 2, 6, N, 64).bfloat16()
    want = fused_paged_attention(dense, cache, bt, past)
    by_token = dense.transpose(1, 2).contiguous().transpose(1, 2)
    o = fused_paged_attention(by_token, cache, bt, past)
    assert torch.equal(o, want) and (N == 1 or o.transpose(1, 2).is_contiguous())
    odd = torch.empty(dense.numel() + 8, device="cuda", dtype=torch.bfloat16)[3:3 + dense.numel()].view_as(dense)
    odd.copy_(dense)
    wide = torch.cat((bt, bt), 1)[:, :12]
    assert not wide.is_contiguous()
    assert torch.equal(fused_paged_attention(odd, cache, wide, past), want)
    every = torch.stack((bt, bt), 2)[..., 0]
    assert torch.equal(fused_paged_attention(dense, cache, every, past), want)


def test_heads_do_not_depend_on_their_batch_and_runs_repeat():
    cache = filled(600, 4, 16, 64, 16, spread=5)
    bt = tables(6, 100, 600, 16)
    past = ints(1599, 3, 800, 17, 1200, 64)
    q = randn(17, 6, 8, 1, 64).half()
    a, b = (fused_paged_attention(q, cache, bt, past) for _ in range(2))
    assert torch.equal(a, b)
    check_attend(q, cache, bt, past)


def test_long_cache_and_offsets_past_32_bits():
    """4.5 GiB of keys and of values: pages behind 2^32 bytes, and a table that mixes both ends."""
    ps, D, Hkv = 128, 128, 8
    pages = 36864
    raw = [torch.zeros(pages * Hkv * ps * D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, Hkv, dtype=torch.uint8, device="cuda") for _ in range(2)]
    big = PagedKV(*(r.view(pages, Hkv, ps, D).view(F8) for r in raw), *(s.view(E8) for s in scales))
    n = 300
    small = paged_kv_cache(4, Hkv, ps, D)
    bt_big, bt_small = ints(pages - 1, 5, pages - 2)[None], ints(0, 1, 2)[None]
    k, v = (randn(i, 1, Hkv, n, D).bfloat16() for i in range(2))
    table = rotary_table(n, D)
    for c, t in ((big, bt_big), (small, bt_small)):
        append_paged_kv(c, k, v, t, ints(0), table=table)
    for i in range(4):
        for a, b in zip(bt_big[0], bt_small[0]):
            assert torch.equal(big[i].view(torch.uint8)[a], small[i].view(torch.uint8)[b])
    for N in (1, 100):
        q = randn(3, 1, 16, N, D).bfloat16()
        assert torch.equal(fused_paged_attention(q, big, bt_big, ints(n - N)),
                           fused_paged_attention(q, small, bt_small, ints(n - N)))


def test_longest_context_in_use():
    """131072 keys of one sequence: a row of random scores against the formula in float64 on the GPU."""
    ps, D, n = 128, 64, 131072
    cache = filled(n // ps, 1, ps, D, 21, spread=2)
    bt = tables(1, n // ps, n // ps, 21)
    k, v = ((c.double() * torch.exp2(s.view(torch.uint8).double() - 127)[..., None, None])[bt[0].long(), 0].reshape(n, D)
            for c, s in zip(cache[:2], cache[2:]))
    for N in (1, 64):
        q = randn(22, 1, 8, N, D).half()
        o = fused_paged_attention(q, cache, bt, ints(n - N))
        s = torch.mm(q[0].double().reshape(-1, D), k.t()) / math.sqrt(D)
        row = torch.arange(N, device="cuda").repeat(8)[:, None] + n - N
        s = s.masked_fill(torch.arange(n, device="cuda")[None] > row, -math.inf)
        w = torch.softmax(s, -1)
        want, a = torch.mm(w, v), torch.mm(w, v.abs())
        terms = float(torch.mm(q[0].double().abs().reshape(-1, D), k.abs().t()).max()) / math.sqrt(D)
        rel = 2.0 ** -11 + 2.0 ** -23 * ((D + 2) * terms + 64) + 2.0 ** -24 * (n / 32 + 64)
        err = (o[0].double().reshape(-1, D) - want).abs()
        assert bool((err <= rel * a + want.abs() * 2.0 ** -11 + 2.0 ** -25).all())


# ---- append

def same_cache(cache, oracle, pages=None):
    for i in range(2):
        got, want = cache[i].float().double().cpu(), oracle.codes[i]
        assert torch.equal(torch.nan_to_num(got, nan=-999.0), torch.nan_to_num(want, nan=-999.0)), i
        assert torch.equal(cache[2 + i].view(torch.uint8).double().cpu() - 127, oracle.exp[i]), i


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_append_bit_for_bit(D, dt, ps):
    """Ragged batch over begun and fresh pages, rows growing so that held ones are moved along."""
    B, Hkv, width = 4, 3, 4
    pages = B * width + 2
    cache = filled(pages, Hkv, ps, D, D + ps, spread=5, low=105)
    bt = tables(B, width, pages, ps)
    want = orc.Cache(*cache)
    N = 2 * ps + 3
    past, new = (0, ps - 1, ps // 2, 2 * ps), (N, 0, N - 5, 1)
    k, v = (randn(i, B, Hkv, N, D).mul(torch.logspace(-3, 2, N, device="cuda")[:, None]).to(dt) for i in range(2))
    out = append_paged_kv(cache, k, v, bt, ints(*past), ints(*new))
    assert out is None
    for b in range(B):
        want.append((k[b].cpu(), v[b].cpu()), b, bt.cpu(), past[b], new[b])
    same_cache(cache, want)


@pytest.mark.parametrize("step", [1, 3, 16])
def test_append_in_steps_equals_append_at_once(step):
    """Powers of two move codes exactly: the pieces do not show, but where a value is subnormal in between."""
    B, Hkv, D, ps, n = 2, 2, 64, 32, 48
    k, v = (randn(i, B, Hkv, n, D).mul(2.0 ** (2 * randn(7 + i, B, 1, n, 1))).bfloat16() for i in range(2))
    bt = tables(B, 2, 4, 1)
    at_once, pieces = paged_kv_cache(4, Hkv, ps, D), paged_kv_cache(4, Hkv, ps, D)
    append_paged_kv(at_once, k, v, bt, ints(0, 0))
    for i in range(0, n, step):
        append_paged_kv(pieces, k[:, :, i:i + step], v[:, :, i:i + step], bt, ints(i, i))
    for i in range(2):
        assert torch.equal(at_once[2 + i].view(torch.uint8), pieces[2 + i].view(torch.uint8))
        a, b = at_once[i].float(), pieces[i].float()
        # subnormal codes (below 2^-6) step by 2^-9: rounded twice, one step
        assert bool((((a - b).abs() == 0) | ((a.abs() <= 2.0 ** -6) & ((a - b).abs() <= 2.0 ** -9))).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,D,R,ps", [(torch.float16, 64, 32, 16), (torch.bfloat16, 128, 128, 64),
                                       (torch.float16, 32, 32, 128), (torch.bfloat16, 128, 96, 32)])
def test_append_with_norm_and_rotation(dt, D, R, ps, interleaved):
    B, H, Hkv, N, width = 3, 10, 5, 45, 4 + 100 // ps
    cache = paged_kv_cache(B * width, Hkv, ps, D)
    bt = tables(B, width, B * width, 3)
    x = randn(4, B, N, H + 2 * Hkv, D).to(dt)
    q, k, v = (t.transpose(1, 2) for t in x.split((H, Hkv, Hkv), 2))
    wq, wk = ((0.4 * randn(i, D)).exp().to(dt) for i in range(2))
    past, new = (0, 19, 101), (N, 30, 1)
    table = rotary_table(101 + N, R)
    log(f"append norm rotation {dt} D={D} R={R} page {ps}")
    out = append_paged_kv(cache, k, v, bt, ints(*past), ints(*new), q, wq, wk, table, eps=EPS, interleaved=interleaved)
    pos = torch.stack([torch.arange(N, device="cuda") + p for p in past])
    want_q, want_k = fused_qk_norm_rotary(q, k, wq, wk, table, pos, None, EPS, interleaved)
    assert out.is_contiguous() and torch.equal(out, want_q)
    c = orc.Cache(*cache)
    for b in range(B):
        cos, sin = orc.angles(table.cpu(), pos[b].cpu(), R)
        y = orc.norm_rotary(k[b].cpu(), wk.cpu(), cos, sin, R, interleaved, EPS)
        slack = orc.norm_rotary_terms(k[b].cpu(), wk.cpu(), R, interleaved, EPS) * 2.0 ** -20
        total = past[b] + new[b]
        got_k, got_v = c.dense(b, bt.cpu(), total)
        for got, want, extra in ((got_k, y, slack), (got_v, v[b].double().cpu(), 0.0 * y)):
            g, w, s = got[:, past[b]:], want[:, :new[b]], extra[:, :new[b]]
            # the scale is that of the page: at most 2 amax / 448
            least = 2.0 * w.abs().amax((1, 2), keepdim=True) / 448 * 2.0 ** -10
            assert bool(((g - w).abs() <= torch.maximum(w.abs() * 2.0 ** -4, least) + s).all())
    # positions given: the same as those it takes by itself
    again = paged_kv_cache(B * width, Hkv, ps, D)
    append_paged_kv(again, k, v, bt, ints(*past), ints(*new), None, None, wk, table, pos, None, EPS, interleaved)
    for i in range(4):
        assert torch.equal(again[i].view(torch.uint8), cache[i].view(torch.uint8))


def test_append_axes():
    B, Hkv, N, D = 2, 2, 9, 64
    cache, other = paged_kv_cache(4, Hkv, 16, D), paged_kv_cache(4, Hkv, 16, D)
    bt = tables(B, 2, 4, 1)
    k, v, q = (randn(i, B, Hkv, N, D).half() for i in range(3))
    table = rotary_table(64, 64)
    pos = torch.randint(0, 64, (3, B, N), generator=gen(5), device="cuda")
    got = append_paged_kv(cache, k, v, bt, ints(3, 20), q=q, table=table, positions=pos, sections=(8, 12, 12))
    want_q, want_k = fused_qk_norm_rotary(q, k, None, None, table, pos, (8, 12, 12))
    assert torch.equal(got, want_q)
    append_paged_kv(other, want_k, v, bt, ints(3, 20))
    # want_k is rounded to 16 bits before its 8: one more half step of fp16 may move a tie
    a, b = cache.k.float(), other.k.float()
    assert float((a - b).abs().gt(a.abs() * 2.0 ** -3 + 2.0 ** -9).sum()) == 0


def test_append_leaves_the_rest_alone_and_skips_unnamed_pages():
    cache = filled(8, 2, 16, 64, 20)
    before = [c.view(torch.uint8).clone() for c in cache]
    k, v = (randn(i, 3, 2, 20, 64).bfloat16() for i in range(2))
    bt = ints(2, -1, 7, 8, 3, 5).view(3, 2)     # sequence 0: page 2, none; 1: page 7, none (8 of 8); 2: 3, 5
    append_paged_kv(cache, k, v, bt, ints(10, 12, 0), ints(20, 20, 3))
    want = orc.Cache(*[b.view(t.dtype) for b, t in zip(before, cache)])
    for b, (p, n) in enumerate(((10, 20), (12, 20), (0, 3))):
        want.append((k[b].cpu(), v[b].cpu()), b, bt.cpu(), p, n)
    same_cache(cache, want)
    for i in range(4):
        for page in (0, 1, 4, 5, 6):
            assert torch.equal(cache[i].view(torch.uint8)[page], before[i][page])
        if i < 2:   # rows behind the last new token, and rows before the first of a begun page's
            assert torch.equal(cache[i].view(torch.uint8)[3, :, 3:], before[i][3, :, 3:])
    now = [c.view(torch.uint8).clone() for c in cache]
    append_paged_kv(cache, k, v, bt, ints(40, 2 ** 31 - 1, 31), ints(20, 20, 0))    # past the table; nothing new
    assert all(torch.equal(a, c.view(torch.uint8)) for a, c in zip(now, cache))


def test_append_values_out_of_range_and_not_finite():
    k = torch.ones(1, 1, 6, 32, device="cuda", dtype=torch.bfloat16)
    k[0, 0, 1, 0], k[0, 0, 2, 1], k[0, 0, 3, 2] = math.inf, -math.inf, math.nan
    v = torch.full_like(k, 2.0 ** -70)                    # below what 2^-40 holds
    v[0, 0, 4] = 0
    cache = paged_kv_cache(2, 1, 16, 32)
    bt = ints(1, 0)[None]
    append_paged_kv(cache, k, v, bt, ints(0))
    want = orc.Cache(*paged_kv_cache(2, 1, 16, 32, device="cpu"))
    want.append((k[0].cpu(), v[0].cpu()), 0, bt.cpu(), 0, 6)
    same_cache(cache, want)
    assert int(torch.isnan(cache.k.float()).sum()) == 3 and float(cache.k_scale[1, 0].float()) == 2.0 ** -8
    assert float(cache.v.float().abs().max()) == 0 and float(cache.v_scale[1, 0].float()) == 2.0 ** -40
    k[0, 0, 0] = 1e30                                     # past 448 2^40
    append_paged_kv(cache, k, v, bt, ints(0))
    assert float(cache.k.float()[1, 0, 0].min()) == 448.0 and float(cache.k_scale[1, 0].float()) == 2.0 ** 40


def test_append_strides_and_alignment():
    B, Hkv, N, D = 2, 2, 21, 64
    bt = tables(B, 2, 4, 2)
    want = paged_kv_cache(4, Hkv, 16, D)
    k, v = (randn(i, B, Hkv, N, D).half() for i in range(2))
    append_paged_kv(want, k, v, bt, ints(0, 5))
    odd = torch.empty(k.numel() + 8, device="cuda", dtype=torch.float16)[1:1 + k.numel()].view_as(k)
    odd.copy_(k)
    forms = [(odd, v.transpose(1, 2).contiguous().transpose(1, 2)),
             (torch.cat((k, k), 3)[..., :D], torch.stack((v, v), 4)[..., 0])]
    for kk, vv in forms:
        got = paged_kv_cache(4, Hkv, 16, D)
        append_paged_kv(got, kk, vv, bt.t().contiguous().t(), torch.stack((ints(0, 5), ints(9, 9)), 1)[:, 0])
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


# ---- together

def serve(cache, xs, bt, H, Hkv, w, table, past, new=None):
    """One step of a layer: the outputs of its attention."""
    q, k, v = (t.transpose(1, 2) for t in xs.split((H, Hkv, Hkv), 2))
    q = append_paged_kv(cache, k, v, bt, past, new, q, *w, table)
    return fused_paged_attention(q, cache, bt, past, new)


def test_prompt_then_tokens_against_the_dense_attention():
    """A prompt in pieces, then single tokens: against the dense grouped attention of all tokens at
    once.  The two differ by the cache's 8 bits: each key and value by half a step, 2^-4 relative."""
    B, H, Hkv, D, n = 2, 8, 2, 128, 200
    x = randn(1, B, n, H + 2 * Hkv, D).bfloat16()
    w = [(0.2 * randn(i, D)).exp().bfloat16() for i in range(2)]
    table = rotary_table(n, D)
    cache = paged_kv_cache(16, Hkv, 32, D)
    bt = tables(B, 7, 16, 1)
    outs, at = [], 0
    for piece in (90, 7, 64, 1, 1, 1, 36):
        outs.append(serve(cache, x[:, at:at + piece], bt, H, Hkv, w, table, torch.full((B,), at, dtype=torch.int32, device="cuda")))
        at += piece
    got = torch.cat(outs, 2).float()
    q, k, v = (t.transpose(1, 2) for t in x.split((H, Hkv, Hkv), 2))
    q, k = fused_qk_norm_rotary(q, k, *w, table)
    want = fused_gqa_attention(q, k, v).float()
    rel = float((got - want).norm() / want.norm())
    log(f"serving against dense: {rel:.2e}")
    # uniform rounding errors of up to 2^-4 have a spread of 2^-4 / sqrt(3): 3.6e-2 of each value, and
    # scores of spread ~1 move by as much again
    assert rel <= 2 * 2.0 ** -4


@pytest.mark.parametrize("N", [1, 3])
def test_captured_steps(N):
    """The two calls of a step in one graph, replayed while lengths and tables change in place; a second
    graph of the same calls in between (their workspaces are their own)."""
    B, H, Hkv, D, steps = 3, 8, 2, 64, 6
    w = [(0.2 * randn(i, D)).exp() for i in range(2)]
    table = rotary_table(2000, D)
    start = ints(1000, 3, 130)
    caches = [filled(96, Hkv, 64, D, 30) for _ in range(2)]
    bt = tables(B, 32, 96, 31)
    x = torch.zeros(B, N, H + 2 * Hkv, D, device="cuda", dtype=torch.float16)
    past = start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve(filled(96, Hkv, 64, D, 30), x, bt, H, Hkv, w, table, past)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for c in (caches[0], filled(96, Hkv, 64, D, 33)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = serve(c, x, bt, H, Hkv, w, table, past)
        graphs.append((g, o, c))
    for i in range(steps):
        x.copy_(randn(40 + i, *x.shape))
        past.copy_(start + N * i)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, o, c), ref in zip(graphs, (caches[1], None)):
            if ref is not None:
                want = serve(ref, x, bt, H, Hkv, w, table, past)
                assert torch.equal(o, want), i
                assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, ref))
    assert not torch.isnan(graphs[1][1]).any()


@pytest.mark.parametrize("N", [1, 5, 20, 60, 100])
def test_c_entry_with_less_workspace(N):
    """fa_paged_attention splits the keys less with a smaller workspace, and not at all without one."""
    import ctypes
    from attention import _lib
    from test_serving_refusals import Cache, Rows
    lib = _lib.load()
    B, H, Hkv, D, ps, width = 2, 4, 2, 64, 16, 150
    cache = filled(B * width, Hkv, ps, D, 60, spread=3)
    bt = tables(B, width, B * width, 61)
    past = ints(width * ps - N, 700)
    q = randn(62, B, H, N, D).bfloat16()
    want = check_attend(q, cache, bt, past, label=f"whole workspace N={N}")
    need = lib.fa_paged_attention_workspace_size(B, H, Hkv, N, D, width * ps)
    assert need > 0
    c = Cache(*(t.data_ptr() for t in cache), bt.data_ptr(), width, width, B * width, ps, Hkv)
    rows = lambda t: ctypes.byref(Rows(t.data_ptr(), *t.stride()[:3]))  # noqa: E731
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for size in (need, need // 2, need // 7, 0):
        o = torch.full_like(q, 7.0)
        code = lib.fa_paged_attention(rows(q), ctypes.byref(c), past.data_ptr(), None, rows(o), None, B, H, N, D, 1,
                                      _lib.scale_log2(D), ws.data_ptr() if size else None, size,
                                      torch.cuda.current_stream().cuda_stream)
        assert code == _lib.FA_OK
        if size == need:
            assert torch.equal(o, want)
        # two splits of the same sums: each within its bound of the exact value, twice 2^-9 of it and the output's rounding
        assert bool(((o.float() - want.float()).abs() <= 2.0 ** -8 * 2 + 2.0 ** -7 * want.float().abs()).all())


def test_two_streams_at_once():
    cache = filled(64, 2, 16, 64, 50, spread=3)
    bt = tables(2, 32, 64, 50)
    past = ints(500, 250)
    qs = [randn(i, 2, 8, 1, 64).half() for i in range(2)]
    want = [fused_paged_attention(q, cache, bt, past) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = fused_paged_attention(qs[i], cache, bt, past)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_random_calls():
    """Drawn shapes through the whole step against the oracle."""
    g = torch.Generator().manual_seed(77)
    pick = lambda *x: x[int(torch.randint(len(x), (1,), generator=g))]  # noqa: E731
    for i in range(24):
        D, ps, dt = pick(32, 64, 128), pick(16, 32, 64, 128), pick(torch.float16, torch.bfloat16)
        Hkv, G, B, N = pick(1, 2, 3, 5), pick(1, 2, 3, 4, 8), pick(1, 2, 3), pick(1, 1, 2, 5, 17, 40, 129)
        lens = [int(torch.randint(0, 400, (1,), generator=g)) for _ in range(B)]
        new = [int(torch.randint(0, N + 1, (1,), generator=g)) for _ in range(B)]
        width = (max(lens) + N) // ps + 1
        log(f"random {i}: D={D} page={ps} {dt} Hkv={Hkv} G={G} N={N} past={lens} new={new}")
        cache = filled(B * width, Hkv, ps, D, i, spread=4)
        bt = tables(B, width, B * width, i)
        x = randn(i, B, N, (G + 2) * Hkv, D).to(dt)
        q, k, v = (t.transpose(1, 2) for t in x.split((G * Hkv, Hkv, Hkv), 2))
        q = append_paged_kv(cache, k, v, bt, ints(*lens), ints(*new), q, None, None, rotary_table(600, D))
        check_attend(q, cache, bt, ints(*lens), ints(*new), label=f"random {i}")


@pytest.mark.parametrize("N,D,ps", [(70, 64, 16), (150, 128, 32), (140, 32, 64), (300, 128, 128)])
def test_prompt_over_a_page_without_a_name(N, D, ps):
    """Rows before its first key do not see it, though their tile holds it."""
    width = (N + 20 + ps - 1) // ps
    cache = filled(width, 1, ps, D, 70)
    bt = tables(1, width, width, 71)
    bt[0, (20 + N // 2) // ps] = -1
    q = randn(72, 1, 2, N, D).bfloat16()
    o = check_attend(q, cache, bt, ints(20))
    first = max((20 + N // 2) // ps * ps - 20, 0)   # the first row that sees a key of that page
    nan = torch.isnan(o)
    assert not nan[0, :, :first].any() and nan[0, :, first:].all()


def exact_cut(rows, parts):
    """fused_paged_attention through the entry that takes one cut at every size."""
    import ctypes
    from attention import _lib
    from test_serving_refusals import Cache, Rows
    lib = _lib.load()

    def call(q, cache, bt, past, new=None, return_lse=False):
        B, H, N, D = q.shape
        Hkv, ps = cache.k.shape[1:3]
        bt, o = bt.contiguous(), torch.full_like(q, 7.0)
        lse = torch.full((B, H, N), 7.0, device="cuda")
        c = Cache(*(t.data_ptr() for t in cache), bt.data_ptr(), bt.shape[1], bt.shape[1], cache.k.shape[0], ps, Hkv)
        size = 0 if parts == 1 else B * Hkv * -(-N * (H // Hkv) // rows) * parts * rows * (D + 4) * 4
        ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        at = lambda t: ctypes.byref(Rows(t.data_ptr(), *t.stride()[:3]))  # noqa: E731
        assert lib.fa_paged_attention_exact(
            at(q), ctypes.byref(c), past.data_ptr(), new.data_ptr() if new is not None else None, at(o), lse.data_ptr(),
            B, H, N, D, int(q.dtype == torch.bfloat16), _lib.scale_log2(D), rows, parts, ws.data_ptr() if size else None,
            size, torch.cuda.current_stream().cuda_stream) == _lib.FA_OK
        return (o, lse) if return_lse else o
    return call


@pytest.mark.parametrize("parts", [1, 2, 5, 20])
@pytest.mark.parametrize("rows", [16, 32, 128, 256])
def test_every_cut_at_every_size(rows, parts, monkeypatch):
    """What the tests above hold the chosen cut to, of each block size and number of parts."""
    monkeypatch.setitem(globals(), "fused_paged_attention", exact_cut(rows, parts))
    for D in (32, 64, 128):
        for dt in (torch.float16, torch.bfloat16):
            for ps in (16, 32, 64, 128):
                test_attention_types_and_pages(D, dt, ps)
    for H, Hkv, N in ((5, 5, 33), (8, 1, 7), (24, 8, 150), (32, 1, 20)):
        test_attention_heads_and_rows(H, Hkv, N)
    for total in (1, 31, 64, 129, 257, 700, 1500):
        test_attention_lengths(total)
    for N in (4, 18, 100):
        test_padded_batch_and_empty_sequences(N)
    for N in (1, 14, 90):
        test_what_lies_behind_a_rows_last_key_does_not_touch_it(torch.bfloat16, N)
    for N in (1, 90):
        test_pages_that_hold_nothing_yet(N)
    for H in (2, 16):
        test_nan_in_a_value_reaches_its_dim_alone(H)
    test_pages_the_table_does_not_name()
    for N, D, ps in ((70, 64, 16), (150, 128, 32), (140, 32, 64), (300, 128, 128)):
        test_prompt_over_a_page_without_a_name(N, D, ps)
    for N in (1, 30, 140):
        test_scales_far_apart_and_zero_pages(torch.float16, N)
    test_long_flat_tail_keeps_its_weight()
    test_sharp_rows_and_one_key()


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 9, 40])
def test_every_row_of_a_page_moves_when_its_scale_grows(D, ps, n):
    """A page filled up to its last n rows, then n rows 2^9 as large: codes and scales as the oracle appends them."""
    n, B, Hkv = min(n, ps - 1), 2, 3
    k, v = (randn(i, B, Hkv, ps, D).bfloat16() for i in range(2))
    for t in (k, v):
        t[:, :, ps - n:] *= 512
    bt = tables(B, 1, 2, 3)
    cache, ref = paged_kv_cache(2, Hkv, ps, D), orc.Cache(*paged_kv_cache(2, Hkv, ps, D, device="cpu"))
    for at, end in ((0, ps - n), (ps - n, ps)):
        append_paged_kv(cache, k[:, :, at:end], v[:, :, at:end], bt, ints(at, at))
        for b in range(B):
            ref.append((k[b, :, at:end].cpu(), v[b, :, at:end].cpu()), b, bt.cpu(), at, end - at)
    same_cache(cache, ref)


@pytest.mark.parametrize("B,Hkv,parts", [(3, 5, 5), (13, 5, 1), (8, 1, 1), (1, 7, 9), (9, 8, 2)])
def test_parts_that_do_not_fill_the_last_round(B, Hkv, parts, monkeypatch):
    """Row blocks by part over the eight L2s: whole rounds of eight parts, and a last one that is not."""
    monkeypatch.setitem(globals(), "fused_paged_attention", exact_cut(16, parts))
    ps, width, N = 16, 40, 20
    cache = filled(B * width, Hkv, ps, 32, 80, spread=3)
    bt = tables(B, width, B * width, 81)
    past = ints(*((97 * b) % (width * ps - N) for b in range(B)))
    new = ints(*(N if b % 3 else 7 * (b % 2) for b in range(B)))
    check_attend(randn(82, B, 2 * Hkv, N, 32).half(), cache, bt, past, new)
