"""The float64 restatement behind the rotary and paged tests, pinned on the CPU."""

import math

import pytest
import torch

from oracle import paged_oracle as orc

F64 = torch.float64


def table_of(length, R):
    j = torch.arange(R // 2, dtype=F64)
    a = torch.arange(length, dtype=F64)[:, None] * 10000.0 ** (-2.0 * j / R)
    return torch.cat((a.cos(), a.sin()), 1)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_complex_product_and_scores_depend_on_distance(interleaved):
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, 16, dtype=F64, generator=g) for _ in range(2))
    t = table_of(64, 16)
    dots = []
    for a, b in ((5, 2), (33, 30), (60, 57)):
        qa = orc.rotate(q, *orc.angles(t, torch.tensor([a]), 16), 16, interleaved)
        kb = orc.rotate(k, *orc.angles(t, torch.tensor([b]), 16), 16, interleaved)
        dots.append(float((qa * kb).sum()))
    assert max(dots) - min(dots) < 1e-12
    cos, sin = orc.angles(t, torch.tensor([7]), 16)
    y = orc.rotate(q, cos, sin, 16, interleaved)
    a, b = (slice(0, 16, 2), slice(1, 16, 2)) if interleaved else (slice(0, 8), slice(8, 16))
    z = torch.complex(q[:, a], q[:, b]) * torch.complex(cos, sin)
    assert torch.allclose(y[:, a], z.real, atol=1e-14) and torch.allclose(y[:, b], z.imag, atol=1e-14)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_match_differences_and_autograd(interleaved, norm):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 8, dtype=F64, generator=g)
    w = torch.randn(8, dtype=F64, generator=g) if norm else None
    dy = torch.randn(2, 3, 8, dtype=F64, generator=g)
    cos, sin = orc.angles(table_of(9, 4), torch.tensor([3, 0, 8]), 4)
    f = lambda x, w: float((orc.norm_rotary(x, w, cos, sin, 4, interleaved, 1e-3) * dy).sum())  # noqa: E731
    dx, dw, _, _ = orc.norm_rotary_grads(x, w, dy, cos, sin, 4, interleaved, 1e-3)
    h = 1e-6
    for grad, var, call in ((dx, x, lambda v: f(v, w)), (dw, w, lambda v: f(x, v))):
        if grad is None:
            continue
        for i in range(var.numel()):
            up, down = var.clone().view(-1), var.clone().view(-1)
            up[i] += h
            down[i] -= h
            d = (call(up.view_as(var)) - call(down.view_as(var))) / (2 * h)
            assert abs(d - float(grad.reshape(-1)[i])) < 1e-8
    xr = x.clone().requires_grad_(True)
    (orc.norm_rotary(xr, w, cos, sin, 4, interleaved, 1e-3) * dy).sum().backward()
    assert torch.allclose(xr.grad, dx, atol=1e-12)


def test_e4m3_rounding_equals_torchs_cast():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    fin = codes[torch.isfinite(codes)].sort().values
    mid = (fin[1:] + fin[:-1]) / 2
    x = torch.cat((fin, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)))
    want = x.float().to(torch.float8_e4m3fn).double()
    assert torch.equal(orc.to_e4m3(x), want)
    assert float(orc.to_e4m3(torch.tensor([1e9], dtype=F64))) == 448.0
    assert torch.isnan(orc.to_e4m3(torch.tensor([math.inf, math.nan], dtype=F64))).all()


def test_scale_exponent_is_the_least_that_fits():
    for amax in (448.0, 448.0 * (1 + 2 ** -20), 1.0, 3.3, 0.0, 2.0 ** -60, 1e30):
        e = float(orc.scale_exponent(torch.tensor(amax, dtype=F64)))
        assert orc.E_MIN <= e <= orc.E_MAX
        if e < orc.E_MAX:
            assert amax <= 448 * 2.0 ** e
        if e > orc.E_MIN:
            assert amax > 448 * 2.0 ** (e - 1)


def tiny_cache(pages, heads, ps, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pages, heads, ps, D, generator=g).to(torch.float8_e4m3fn) for _ in range(2))
    e = torch.randint(122, 130, (2, pages, heads), generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return orc.Cache(k, v, e[0], e[1])


def test_attention_equals_sdpa_and_planted_mistakes_show():
    c = tiny_cache(4, 2, 16, 32)
    bt = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    q = torch.randn(4, 5, 32, dtype=F64, generator=torch.Generator().manual_seed(3))
    o, lse, bound = orc.attend(q, c, bt, 30, 5)
    k, v = c.dense(0, bt, 35)
    mask = torch.arange(35)[None, :] <= 30 + torch.arange(5)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q[None], k.repeat_interleave(2, 0)[None],
                                                            v.repeat_interleave(2, 0)[None], attn_mask=mask)[0]
    assert torch.allclose(o, want, atol=1e-12)
    s = (q @ k.repeat_interleave(2, 0).transpose(1, 2) / math.sqrt(32)).masked_fill(~mask, -math.inf)
    assert torch.allclose(lse, torch.logsumexp(s, -1) / math.log(2), atol=1e-12)
    for past in (29, 31):   # a mask one key off
        assert not bool(((orc.attend(q, c, bt, past, 5)[0] - want).abs() <= bound).all())
    off = tiny_cache(4, 2, 16, 32)
    off.exp[0][2, 1] += 1   # a scale one step off
    assert not bool(((orc.attend(q, off, bt, 30, 5)[0] - want).abs() <= bound).all())


def test_append_then_dense_returns_the_rounded_values():
    c = tiny_cache(3, 1, 16, 32)
    bt = torch.tensor([[1, 2]], dtype=torch.int32)
    x = torch.randn(1, 20, 32, dtype=F64, generator=torch.Generator().manual_seed(4))
    before = c.codes[0][0].clone()
    c.append((x, 3 * x), 0, bt, 0, 20)
    for got, want in zip(c.dense(0, bt, 20), (x, 3 * x)):
        for rows in (slice(0, 16), slice(16, 20)):   # half a step of 4 significant bits, or of the page's least one
            e = orc.scale_exponent(want[:, rows].abs().max())
            assert bool(((got - want)[:, rows].abs() <= torch.maximum(want[:, rows].abs() * 2.0 ** -4,
                                                                      torch.exp2(e - 10))).all())
    assert torch.equal(c.codes[0][0], before)
