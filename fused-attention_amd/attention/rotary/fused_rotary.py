"""Norm of queries and keys for each head with the position rotation in the same pass, on MI355X.

    q, k = fused_qk_norm_rotary(q, k, q_weight, k_weight, table, positions=None, sections=None,
                                eps=1e-6, interleaved=False)
    q, k = fused_qk_norm_rotary_autograd(...)         # the same with a backward

The step before fused_gqa_attention in a model (the reference has no counterpart: its inputs are
already normed and turned).  For each row x of D values (one head of one token):

    y = R(p) (w * x * r),   r = (mean(x^2) + eps)^(-1/2)

in fp32, rounded once.  R(p) turns the pairs of the first rotary_dim dims by the angles of the row's
position: pair j is dims (j, j + rotary_dim / 2), or (2j, 2j + 1) with interleaved=True.  The other
dims keep their normed value.

q: (B, H, N, D), k: (B, H_kv, N, D), float16 or bfloat16, D in {32, 64, 128}.  Any strides: the views
of a packed projection, qkv.view(B, N, heads, D).transpose(1, 2), are read as they are (rows that
are not 16-byte aligned are copied first).  The outputs are dense (B, heads, N, D), what the fused
attention reads without a copy; the gradients of q and k are laid out in memory as q and k are.

q_weight, k_weight: (D,) of q's dtype or float32, or None, both: no norm.
table: (length, rotary_dim) float32 from rotary_table(), or None: no rotation.
positions: (B, N) or (N,) int32 or int64; None: token n is at n.  With sections=(n0, n1[, n2]), which
    sum to rotary_dim / 2, positions is (axes, B, N) or (axes, N): the first n0 pairs turn with the first
    axis (time, say), the next n1 with the second (height), the last n2 with the third (width).
    A negative position leaves its row unturned (padding); one past the table gives NaN.

Gradients of the weights are fp32 sums over all rows in a fixed order.  There is no second
derivative: backward(create_graph=True) raises RuntimeError.  Under graph capture the autograd entry
raises RuntimeError while an earlier graph of the same leaves made on another stream is alive.
"""

import torch

from attention import _lib


def rotary_table(length, rotary_dim, base=10000.0, device="cuda"):
    """(length, rotary_dim) float32: the cosines of position * base^(-2j / rotary_dim), then the sines.

    Made in float64, so a position's angle is right to the last bits at any length; laid out once by
    a model and shared by its layers (64 MiB at 131072 positions of 128 dims)."""
    if rotary_dim % 2 or rotary_dim <= 0 or length < 1:
        raise ValueError(f"need length >= 1 and an even rotary_dim; got {length}, {rotary_dim}")
    j = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    p = torch.arange(length, dtype=torch.float64, device=device)
    angle = p[:, None] * torch.pow(torch.tensor(base, dtype=torch.float64, device=device), -2.0 * j / rotary_dim)
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def fused_qk_norm_rotary(q, k, q_weight=None, k_weight=None, table=None, positions=None, sections=None,
                         eps=1e-6, interleaved=False):
    return _lib.autograd().qk_norm_rotary(q, k, q_weight, k_weight, table, positions, sections, eps, interleaved)


def fused_qk_norm_rotary_autograd(q, k, q_weight=None, k_weight=None, table=None, positions=None, sections=None,
                                  eps=1e-6, interleaved=False):
    return _lib.autograd().qk_norm_rotary_autograd(q, k, q_weight, k_weight, table, positions, sections, eps,
                                                   interleaved)
