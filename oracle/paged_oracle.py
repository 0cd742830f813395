"""float64 restatement of norm + rotation, the 8-bit paged cache and attention over it -- TEST
INFRASTRUCTURE ONLY, on the CPU, in torch float64, one sequence at a time.

tests/test_paged_oracle.py pins it: the gradients by central differences and torch autograd, the
rotation by complex multiplication and by its dependence on distances alone, the e4m3 rounding by
torch's own cast of every representable midpoint, the attention by torch SDPA in float64.
"""

import math

import torch

CODE_MAX, E_MIN, E_MAX = 448.0, -40, 40
F64 = torch.float64


def angles(table, pos, R):
    """cos, sin [N, R / 2] (float64) for positions [N] or, one position a pair, [N, R / 2]."""
    half = R // 2
    pos = pos[:, None].expand(-1, half) if pos.dim() == 1 else pos
    pair = torch.arange(half).expand_as(pos)
    at = pos.clamp(0, table.shape[0] - 1).long()
    cos, sin = table.double()[at, pair], table.double()[at, pair + half]
    cos = torch.where(pos < 0, 1.0, torch.where(pos >= table.shape[0], math.nan, cos))
    sin = torch.where(pos < 0, 0.0, torch.where(pos >= table.shape[0], math.nan, sin))
    return cos, sin


def pair_positions(positions, sections):
    """positions [axes, N], pairs per axis -> [N, R / 2]."""
    return torch.cat([positions[a][:, None].expand(-1, n) for a, n in enumerate(sections)], 1)


def rotate(x, cos, sin, R, interleaved):
    """x [..., N, D] with the pairs of its first R dims turned."""
    y = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def norm_rotary(x, w, cos, sin, R, interleaved, eps):
    """y of rows x [..., N, D] (float64); w None: no norm; R 0: no rotation."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return rotate(x, cos, sin, R, interleaved) if R else x


def norm_rotary_terms(x, w, R, interleaved, eps):
    """Sum of the absolute values of the terms that make y (cos, sin <= 1): what its fp32 rounding scales with."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return rotate(x.abs(), torch.ones(1), -torch.ones(1), R, interleaved).abs() + x.abs() if R else x.abs()


def norm_rotary_grads(x, w, dy, cos, sin, R, interleaved, eps):
    """(dx, dw summed over all leading dims, sum of |terms| of dx, of dw); w None: dw None."""
    x, dy = x.double(), dy.double()
    g = rotate(dy, cos, -sin, R, interleaved) if R else dy
    ga = rotate(dy.abs(), torch.ones(1), -torch.ones(1), R, interleaved).abs() + dy.abs() if R else dy.abs()
    if w is None:
        return g, None, ga, None
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n, u = x * r, g * w.double()
    dx = r * (u - n * (u * n).mean(-1, keepdim=True))
    ua = ga * w.double().abs()
    dxa = r * (ua + n.abs() * (ua * n.abs()).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return dx, (g * n).sum(lead), dxa, (ga * n.abs()).sum(lead)


def to_e4m3(x):
    """Nearest e4m3 value, ties to even; past 448 to 448; what is not finite to NaN."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    y = (torch.round(x / step) * step).clamp(-CODE_MAX, CODE_MAX)
    return torch.where(torch.isfinite(x), y, math.nan)


def scale_exponent(amax):
    """Least e with amax <= 448 2^e, in [E_MIN, E_MAX] (float64 in, float64 whole numbers out)."""
    e = torch.full_like(amax, float(E_MIN))
    for i in range(E_MIN + 1, E_MAX + 1):
        e = torch.where(amax > CODE_MAX * 2.0 ** (i - 1), float(i), e)
    return e


class Cache:
    """Values of a paged cache in float64: codes [P, H_kv, page, D], exponents [P, H_kv]."""

    def __init__(self, k, v, k_scale, v_scale):
        self.codes = [k.cpu().float().double(), v.cpu().float().double()]
        self.exp = [k_scale.cpu().view(torch.uint8).double() - 127, v_scale.cpu().view(torch.uint8).double() - 127]

    def page(self, block_table, b, col):
        p = int(block_table[b, col]) if col < block_table.shape[1] else -1
        return p if 0 <= p < self.codes[0].shape[0] else -1

    def append(self, rows, b, block_table, past, new):
        """rows: (k, v) [H_kv, N, D] of one sequence, already normed and turned."""
        ps = self.codes[0].shape[2]
        past, new = max(past, 0), min(max(new, 0), rows[0].shape[1])
        for col in range(past // ps, -(-(past + new) // ps) if new else 0):
            page = self.page(block_table, b, col)
            if page < 0:
                continue
            lo, hi = max(past, col * ps), min(past + new, (col + 1) * ps)
            for c, x in zip(range(2), rows):
                x = x[:, lo - past:hi - past].double()
                fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
                e = scale_exponent(fin.amax((1, 2)))
                if lo > col * ps:
                    old = self.exp[c][page]
                    e = torch.maximum(e, old)
                    held = self.codes[c][page, :, :lo - col * ps]
                    self.codes[c][page, :, :lo - col * ps] = to_e4m3(held * torch.exp2(old - e)[:, None, None])
                self.codes[c][page, :, lo - col * ps:hi - col * ps] = to_e4m3(x * torch.exp2(-e)[:, None, None])
                self.exp[c][page] = e

    def dense(self, b, block_table, length):
        """(k, v) [H_kv, length, D]; keys of a page that the table does not name are NaN."""
        ps = self.codes[0].shape[2]
        out = []
        for c in range(2):
            pages = []
            for col in range(-(-length // ps)):
                p = self.page(block_table, b, col)
                x = self.codes[c][max(p, 0)] * torch.exp2(self.exp[c][max(p, 0)])[:, None, None]
                pages.append(x if p >= 0 else torch.full_like(x, math.nan))
            out.append(torch.cat(pages, 1)[:, :length] if pages else self.codes[c][0][:, :0])
        return out


def attend(q, cache, block_table, past, new):
    """(o [H, N, D], lse [H, N] base 2, bound [H, N, D]) of one sequence in float64: q [H, N, D].

    bound: how far fp32 scores and 16-bit weights may take o from it, before its own rounding:
    with A = sum_j p_j |v_j|, each weight is off by its rounding to fp16 (2^-11), by 2 ln 2 times its score's
    error (D + 2 roundings of 2^-24 to the sum of the |q k| terms, and of the exponent itself), and acc
    and l by their sums' (a 2^-24 for each 32 keys and 64 for the joins)."""
    H, N, D = q.shape
    past, new = max(past, 0), min(max(new, 0), N)
    o, lse = torch.zeros((H, N, D), dtype=F64), torch.full((H, N), -math.inf, dtype=F64)
    bound = torch.zeros_like(o)
    if new == 0:
        return o, lse, bound
    length = past + new
    k, v = cache.dense(0, block_table, length)
    G = H // k.shape[0]
    k, v, q = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0), q[:, :new].double()
    s = q @ k.transpose(1, 2) / math.sqrt(D)
    hidden = torch.arange(length)[None, :] > past + torch.arange(new)[:, None]
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    w = p / total
    # (a masked key's weight is 0, and 0 NaN is not to reach its row)
    nan = torch.isnan(v)
    o[:, :new] = w @ torch.where(nan, 0.0, v)
    o[:, :new].masked_fill_((~hidden).double() @ nan.double() > 0, math.nan)
    lse[:, :new] = ((top + torch.log(total)) / math.log(2.0))[..., 0]
    terms = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(hidden, 0.0).amax(-1, keepdim=True) / math.sqrt(D)
    rel = 2.0 ** -11 + 2.0 * 2.0 ** -24 * ((D + 2) * terms + 64) + 2.0 ** -24 * (length / 32 + 64)
    bound[:, :new] = rel * (w @ torch.where(nan, 0.0, v).abs())
    return o, lse, bound
