"""Norm and rotation of queries and keys on the GPU against the float64 formula and its gradients.

Bars, from the arithmetic: an output is rounded once (half a step of its type, relative), after fp32
operations whose errors add up to less than 16 roundings (2^-20) of the absolute terms that make it; a
gradient of a weight is an fp32 sum of M rows, at most 64 + M / 16 roundings deep here, of terms with
the same 16 roundings each.  fp16 results below its normal range are off by half its least step.
"""

import pytest
import torch

from attention.gqa.fused_gqa import fused_gqa_attention_autograd
from attention.rotary.fused_rotary import fused_qk_norm_rotary, fused_qk_norm_rotary_autograd, rotary_table
from oracle import paged_oracle as orc
from gpu_util import log

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
EPS = 1e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def packed(B, H, Hkv, N, D, dt, seed):
    x = (torch.randn(B, N, H + 2 * Hkv, D, generator=gen(seed), device="cuda") * 1.5).to(dt)
    return [t.transpose(1, 2) for t in x.split((H, Hkv, Hkv), 2)]


def weights(D, wt, seed):
    return [(0.3 * torch.randn(D, generator=gen(seed + i), device="cuda")).exp().to(wt) for i in range(2)]


def near(got, want, terms, label, depth=16):
    tol = want.abs() * HALF[got.dtype] + terms * depth * 2.0 ** -24 + LEAST[got.dtype]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (label, float((err / tol).max()))


def positions_of(table, positions, sections, B, N):
    """cos, sin [B, N, R / 2] on the CPU."""
    R = table.shape[1]
    t = table.cpu()
    out = []
    for b in range(B):
        if positions is None:
            p = torch.arange(N)
        elif sections is None:
            p = (positions if positions.dim() == 1 else positions[b]).cpu()
        else:
            p = orc.pair_positions((positions if positions.dim() == 2 else positions[:, b]).cpu(), sections)
        out.append(orc.angles(t, p, R))
    return [torch.stack(x) for x in zip(*out)]


def check(q, k, wq, wk, table, positions, sections, interleaved, grads=True, label=""):
    """Both entries on one call against the oracle; returns the autograd entry's outputs."""
    B, _, N, D = q.shape
    R = table.shape[1] if table is not None else 0
    cos, sin = positions_of(table, positions, sections, B, N) if R else (None, None)
    turn = lambda c: c[:, None] if c is not None else None  # noqa: E731
    q, k = q.detach(), k.detach()
    plain = fused_qk_norm_rotary(q, k, wq, wk, table, positions, sections, EPS, interleaved)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, wq, wk)]
    out = fused_qk_norm_rotary_autograd(*leaves, table, positions, sections, EPS, interleaved)
    dys = [torch.randn(t.shape, generator=gen(9 + i), device="cuda").to(q.dtype) for i, t in enumerate(out)]
    for i, (x, w, name) in enumerate(((q, wq, "q"), (k, wk, "k"))):
        xc, wc = x.cpu(), w.cpu() if w is not None else None
        want = orc.norm_rotary(xc, wc, turn(cos), turn(sin), R, interleaved, EPS)
        terms = orc.norm_rotary_terms(xc, wc, R, interleaved, EPS)
        assert plain[i].is_contiguous() and plain[i].shape == x.shape
        near(plain[i], want, terms, f"{label} {name}")
        assert torch.equal(plain[i], out[i].detach())
    if not grads:
        return out
    got = torch.autograd.grad(out, [t for t in leaves if t is not None], dys)
    for i, (x, w, name) in enumerate(((q, wq, "q"), (k, wk, "k"))):
        xc, wc = x.cpu(), w.cpu() if w is not None else None
        dx, dw, dxa, dwa = orc.norm_rotary_grads(xc, wc, dys[i].cpu(), turn(cos), turn(sin), R, interleaved, EPS)
        near(got[i], dx, dxa, f"{label} d{name}", 24)
        if w is not None:
            rows = x.numel() // D
            near(got[2 + i], dw, dwa, f"{label} dw{name}", 16 + 64 + rows / 16)
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,R", [(32, 32), (32, 16), (64, 64), (64, 48), (64, 16), (128, 128), (128, 64), (128, 96), (128, 0)])
def test_packed_projection(D, R, dt, interleaved):
    q, k, _ = packed(2, 6, 3, 37, D, dt, D + R)
    wq, wk = weights(D, dt if D == 64 else torch.float32, R)
    log(f"rotary D={D} R={R} {dt} interleaved={interleaved}")
    check(q, k, wq, wk, rotary_table(50, R) if R else None, None, None, interleaved)


@pytest.mark.parametrize("B,H,Hkv,N", [(1, 1, 1, 1), (1, 32, 1, 1), (3, 5, 5, 17), (1, 9, 3, 333), (2, 17, 1, 64)])
def test_sizes(B, H, Hkv, N):
    q, k, _ = packed(B, H, Hkv, N, 128, torch.bfloat16, N)
    wq, wk = weights(128, torch.bfloat16, N)
    check(q, k, wq, wk, rotary_table(N, 128), None, None, False)


def test_no_norm_and_no_rotation():
    q, k, _ = packed(2, 4, 2, 20, 64, torch.float16, 1)
    wq, wk = weights(64, torch.float32, 1)
    check(q, k, None, None, rotary_table(20, 64), None, None, False)
    check(q, k, wq, wk, None, None, None, False)
    check(q, k, None, None, None, None, None, True)


@pytest.mark.parametrize("sections", [(4, 6, 6), (0, 16, 0), (3, 13), (5, 5, 6), (16,)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(sections, interleaved):
    B, N = 2, 21
    q, k, _ = packed(B, 4, 2, N, 64, torch.bfloat16, 2)
    wq, wk = weights(64, torch.float32, 2)
    table = rotary_table(100, 32)
    p = torch.randint(0, 100, (len(sections), B, N), generator=gen(3), device="cuda")
    check(q, k, wq, wk, table, p.int(), sections, interleaved)
    check(q, k, wq, wk, table, p.permute(1, 2, 0).contiguous().permute(2, 0, 1), sections, interleaved)   # int64, strided
    check(q, k, wq, wk, table, p[:, 0].contiguous(), sections, interleaved)


@pytest.mark.parametrize("it", [torch.int32, torch.int64])
def test_positions_far_negative_and_past_the_table(it):
    q, k, _ = packed(2, 4, 2, 6, 64, torch.float16, 4)
    wq, wk = weights(64, torch.float16, 4)
    table = rotary_table(70000, 64)
    p = torch.tensor([[69999, 3, 0, -1, -7, 65536], [1, 1, 2, 69000, 5, 40000]], device="cuda", dtype=it)
    out = check(q, k, wq, wk, table, p, None, False)
    unturned = fused_qk_norm_rotary(q, k, wq, wk)
    assert torch.equal(out[0].detach()[0, :, 3:5], unturned[0][0, :, 3:5])
    p[1, 2] = 70000
    a, b = fused_qk_norm_rotary(q, k, wq, wk, table, p)
    assert torch.isnan(a[1, :, 2]).all() and torch.isnan(b[1, :, 2]).all()
    keep = torch.ones(2, 6, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert torch.equal(a.transpose(1, 2)[keep], out[0].detach().transpose(1, 2)[keep])
    p[1, 2] = 2 ** 31 - 1
    assert torch.isnan(fused_qk_norm_rotary(q, k, wq, wk, table, p)[0][1, :, 2]).all()


def test_strides_alignment_and_broadcast():
    D, dt = 64, torch.bfloat16
    wq, wk = weights(D, dt, 5)
    table = rotary_table(40, D)
    base = torch.randn(3 * 4 * 20 * D + 8, generator=gen(5), device="cuda").to(dt)
    odd = base[1:1 + 3 * 4 * 20 * D].view(3, 4, 20, D)              # 2 bytes off 16
    k = torch.randn(3, 1, 20, D, generator=gen(6), device="cuda").to(dt).expand(3, 4, 20, D)   # one head broadcast
    check(odd, k, wq, wk, table, None, None, False, label="odd")
    wide = torch.randn(3, 20, 4, D + 4, generator=gen(7), device="cuda").to(dt)[..., :D].transpose(1, 2)  # row stride 68
    every = torch.randn(3, 4, 20, 2 * D, generator=gen(8), device="cuda").to(dt)[..., ::2]      # dims not contiguous
    check(wide, every, wq, wk, table, None, None, True, label="wide")
    off = torch.empty(D + 8, device="cuda", dtype=dt)[1:1 + D].copy_(wq)
    check(odd, k, off, wk, table[:, ::1], None, None, False, label="weight off 16 bytes")
    # the gradient of a broadcast input is the sum over what it was broadcast to
    one = k[:, :1].detach().clone().requires_grad_(True)
    q = odd.detach()
    _, y = fused_qk_norm_rotary_autograd(q, one.expand(3, 4, 20, D), wq, wk, table)
    dy = torch.randn(y.shape, generator=gen(9), device="cuda").to(dt)
    (g,) = torch.autograd.grad(y, one, dy)
    whole = k.detach().contiguous().requires_grad_(True)
    (each,) = torch.autograd.grad(fused_qk_norm_rotary_autograd(q, whole, wq, wk, table)[1], whole, dy)
    assert torch.equal(g, each.sum(1, keepdim=True))


def test_gradients_that_are_expanded_missing_or_of_some_inputs():
    q, k, _ = packed(2, 4, 2, 9, 64, torch.float16, 10)
    wq, wk = weights(64, torch.float32, 10)
    table = rotary_table(9, 64)
    leaf = lambda t: t.detach().requires_grad_(True)  # noqa: E731
    ql, wl = leaf(q), leaf(wk)
    a, b = fused_qk_norm_rotary_autograd(ql, k, wq, wl, table)
    (a.float().sum() + b.float().sum()).backward()          # expanded ones
    ones = [torch.ones_like(a), torch.ones_like(b)]
    full = [leaf(t) for t in (q, k, wq, wk)]
    got = torch.autograd.grad(fused_qk_norm_rotary_autograd(*full, table), full, ones)
    assert torch.equal(ql.grad, got[0]) and torch.equal(wl.grad, got[3])
    full = [leaf(t) for t in (q, k, wq, wk)]
    out = fused_qk_norm_rotary_autograd(*full, table)
    got = torch.autograd.grad(out[1], full, ones[1], allow_unused=True)   # q's output unused
    assert float(got[0].abs().max()) == 0 and float(got[2].abs().max()) == 0 and float(got[1].abs().max()) > 0
    with pytest.raises(RuntimeError):
        torch.autograd.grad(fused_qk_norm_rotary_autograd(*full, table)[0].sum(), full[0], create_graph=True)


def test_zero_rows_stay_zero_and_have_gradients():
    q = torch.zeros(1, 2, 5, 64, device="cuda", dtype=torch.bfloat16)
    k, _, _ = packed(1, 2, 2, 5, 64, torch.bfloat16, 11)
    wq, wk = weights(64, torch.float32, 11)
    out = check(q, k, wq, wk, rotary_table(5, 64), None, None, False)
    assert float(out[0].detach().abs().max()) == 0


def test_weight_gradients_are_reproducible_over_many_rows():
    B, H, Hkv, N, D = 3, 8, 2, 1111, 128
    q, k, _ = packed(B, H, Hkv, N, D, torch.bfloat16, 12)
    wq, wk = weights(D, torch.float32, 12)
    table = rotary_table(N, D)
    check(q, k, wq, wk, table, None, None, False, label="many")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    dys = [torch.randn(t.shape, generator=gen(i), device="cuda").to(q.dtype) for i, t in enumerate((q, k))]
    runs = [torch.autograd.grad(fused_qk_norm_rotary_autograd(*leaves, table), leaves, dys) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert runs[0][0].stride() == q.contiguous().transpose(1, 2).contiguous().transpose(1, 2).stride()   # by token, as q


def test_training_step_with_the_attention():
    """Norm and rotation, then the grouped attention with its backward: gradients at the projection
    against fp64 autograd of the formulas, through both ops' own roundings (relative, 2^-8 a step)."""
    B, H, Hkv, N, D = 2, 4, 2, 100, 64
    x = torch.randn(B, N, H + 2 * Hkv, D, generator=gen(13), device="cuda").bfloat16().requires_grad_(True)
    wq, wk = (w.requires_grad_(True) for w in weights(D, torch.float32, 13))
    table = rotary_table(N, D)
    dy = torch.randn(B, H, N, D, generator=gen(14), device="cuda").bfloat16()

    q, k, v = (t.transpose(1, 2) for t in x.split((H, Hkv, Hkv), 2))
    o = fused_gqa_attention_autograd(*fused_qk_norm_rotary_autograd(q, k, wq, wk, table), v)
    got = torch.autograd.grad(o, (x, wq, wk), dy)

    xd = x.detach().double().cpu().requires_grad_(True)
    wd = [w.detach().double().cpu().requires_grad_(True) for w in (wq, wk)]
    cos, sin = orc.angles(table.cpu(), torch.arange(N), D)
    q, k, v = (t.transpose(1, 2) for t in xd.split((H, Hkv, Hkv), 2))
    q, k = (orc.norm_rotary(t, w, cos, sin, D, False, EPS) for t, w in ((q, wd[0]), (k, wd[1])))
    want_o = torch.nn.functional.scaled_dot_product_attention(q, k.repeat_interleave(H // Hkv, 1),
                                                              v.repeat_interleave(H // Hkv, 1), is_causal=True)
    want = torch.autograd.grad(want_o, (xd, *wd), dy.double().cpu())
    # the chain rounds q, k, P, dS, the gradients between the ops and the results: under eight half steps
    for name, a, b in zip(("o", "dx", "dwq", "dwk"), (o.detach(), *got), (want_o.detach(), *want)):
        rel = float((a.double().cpu() - b).norm() / b.norm())
        log(f"training step {name}: {rel:.2e}")
        assert rel <= 8 * 2.0 ** -8, (name, rel)


def test_other_stream():
    q, k, _ = packed(2, 4, 2, 50, 64, torch.float16, 15)
    wq, wk = weights(64, torch.float32, 15)
    table = rotary_table(50, 64)
    want = fused_qk_norm_rotary(q, k, wq, wk, table)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = fused_qk_norm_rotary(q, k, wq, wk, table)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_forward_and_backward():
    B, H, Hkv, N, D = 2, 4, 2, 130, 128
    q, k, _ = packed(B, H, Hkv, N, D, torch.bfloat16, 16)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *weights(D, torch.float32, 16))]
    table = rotary_table(N, D)
    dys = [torch.randn(t.shape, generator=gen(i), device="cuda").to(q.dtype) for i, t in enumerate((q, k))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fused_qk_norm_rotary_autograd(*leaves, table), leaves, dys)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_qk_norm_rotary_autograd(*leaves, table)
        grads = torch.autograd.grad(out, leaves, dys)
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(q.shape, generator=gen(20 + i), device="cuda"))
            leaves[2].mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
        eager = fused_qk_norm_rotary_autograd(*fresh, table)
        want = list(eager) + list(torch.autograd.grad(eager, fresh, dys))
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(list(out) + list(grads), want))


def test_capture_is_refused_while_an_eager_graph_of_the_leaves_lives():
    q, k, _ = packed(1, 2, 1, 8, 64, torch.bfloat16, 17)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *weights(64, torch.float32, 17))]
    alive = fused_qk_norm_rotary_autograd(*leaves, rotary_table(8, 64))
    table = rotary_table(8, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still alive"):
            fused_qk_norm_rotary_autograd(*leaves, table)
        fused_qk_norm_rotary(*[t.detach() for t in leaves], table)
    graph.replay()
    torch.cuda.synchronize()
    del alive
    fused_qk_norm_rotary_autograd(*leaves, table)


@pytest.mark.parametrize("it", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_unturned_values_do_not_see_their_neighbours(it, bad):
    """Dims past the rotated ones and rows at negative positions are handed on as they are, whatever
    stands beside them, in the outputs and in the gradients."""
    B, H, Hkv, N, D, R = 2, 3, 1, 5, 64, 32
    q, k = (torch.randn(B, h, N, D, generator=gen(3), device="cuda").to(torch.bfloat16) for h in (H, Hkv))
    dq, dk = (torch.randn(t.shape, generator=gen(4), device="cuda").to(t.dtype) for t in (q, k))
    for t in (q, k, dq, dk):
        t[..., 40] = bad                     # a neighbour in an unturned pair
        t[:, :, 2, 1] = bad                  # and in the row that is not turned at all
    table = rotary_table(16, R)
    pos = torch.arange(N, device="cuda", dtype=torch.int32)
    pos[2] = -1
    leaves = [t.clone().requires_grad_(True) for t in (q, k)]
    out = fused_qk_norm_rotary_autograd(*leaves, None, None, table, pos, None, EPS, it)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    for got, want in (*zip(out, (q, k)), *zip(grads, (dq, dk))):
        for x, y in ((got[..., R:], want[..., R:]), (got[:, :, 2], want[:, :, 2])):
            assert torch.equal(torch.nan_to_num(x.detach(), nan=12345.0), torch.nan_to_num(y, nan=12345.0))
        live = [n for n in range(N) if n != 2]
        assert bool(torch.isfinite(got[:, :, live, :R]).all())
