"""Serving: a paged cache of keys and values in 8 bits, and causal GQA/MQA attention over it.

    cache = paged_kv_cache(num_pages, H_kv, page_size, D)
    q = append_paged_kv(cache, k, v, block_table, past_lens, q=q, q_weight=wq, k_weight=wk, table=table)
    o = fused_paged_attention(q, cache, block_table, past_lens)

Beyond the reference, whose attention takes all queries and keys of a sequence at once.  A step of a
model's layer is the two calls above, for one new token of each sequence, a few, or a long piece of a
prompt: append_paged_kv stores the new keys and values (normed and turned as fused_qk_norm_rotary
does) and returns the queries ready for fused_paged_attention.  Kernels run asynchronously on the
current stream; both calls can be captured into a graph and replayed while block_table, past_lens and
new_lens change in place.

cache: PagedKV(k, v, k_scale, v_scale), or any four such tensors.  k, v are (num_pages, H_kv,
    page_size, D) float8_e4m3fn, page_size 16, 32, 64 or 128; the scales are (num_pages, H_kv)
    float8_e8m0fnu, one power of two for each page and head: value = k * 2^(k_scale's exponent).
block_table: (B, pages) int32, the page that holds keys [i * page_size, (i + 1) * page_size).
past_lens: (B,) int32, the tokens each sequence held before this step.
new_lens: (B,) int32, how many of the N new tokens are real (None: all); the rest is padding.

Pages that a call appends to must each stand once in one sequence's row of the table (copy a shared page
first); pages that are only read may be shared.  A page is begun anew when its first row is written.  Its scale is the least power of two that brings its
largest value into e4m3's range, 2^-40 at least and 2^40 at most; when a later token needs a larger one,
the rows already there are moved along, exactly but for values that become subnormal.  Infinities and NaN are stored
as NaN.  A token whose page the table does not name (negative, too large, or past its last column) is
not stored, and rows that see such a page in the attention become NaN.
"""

from collections import namedtuple

import torch

from attention import _lib

PagedKV = namedtuple("PagedKV", "k v k_scale v_scale")


def paged_kv_cache(num_pages, num_kv_heads, page_size, head_dim, device="cuda"):
    """An empty cache: 2 * num_pages * num_kv_heads * page_size * head_dim bytes and its scales."""
    if num_pages < 1 or num_kv_heads < 1 or page_size not in (16, 32, 64, 128) or head_dim not in (32, 64, 128):
        raise ValueError(f"need num_pages, num_kv_heads >= 1, page_size 16, 32, 64 or 128, head_dim 32, 64 or 128; "
                         f"got {num_pages}, {num_kv_heads}, {page_size}, {head_dim}")
    codes = [torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device)
             for _ in range(2)]
    scales = [torch.zeros((num_pages, num_kv_heads), dtype=torch.uint8, device=device) for _ in range(2)]
    return PagedKV(*(c.view(torch.float8_e4m3fn) for c in codes), *(s.view(torch.float8_e8m0fnu) for s in scales))


def append_paged_kv(cache, k, v, block_table, past_lens, new_lens=None, q=None, q_weight=None, k_weight=None,
                    table=None, positions=None, sections=None, eps=1e-6, interleaved=False):
    """Store k and v (B, H_kv, N, D), float16 or bfloat16, as tokens past_lens[b] .. of their sequences.

    k_weight, table, positions, sections, eps, interleaved: norm and rotation of k on the way, as in
    fused_qk_norm_rotary (positions None: token n is at past_lens[b] + n).  With q (B, H, N, D), q is
    normed (q_weight) and turned in the same launch; returns it, dense (B, H, N, D), else None."""
    return _lib.autograd().append_paged_kv(*cache, k, v, block_table, past_lens, new_lens, q, q_weight, k_weight,
                                           table, positions, sections, eps, interleaved)


def fused_paged_attention(q, cache, block_table, past_lens, new_lens=None, return_lse=False):
    """O of q (B, H, N, D): query n of sequence b sees keys 0 .. past_lens[b] + n, scale 1/sqrt(D).

    Query head h reads K/V head h // (H // H_kv).  O has q's shape, dtype and memory layout; padding gets zeros.
    With return_lse also the (B, H, N) float32 log-sum-exp in the units of the training forward
    (base 2; -inf for padding).  Keys behind a row's last one do not touch it, whatever they hold."""
    o, lse = _lib.autograd().paged_attention(q, *cache, block_table, past_lens, new_lens, return_lse)
    return (o, lse) if return_lse else o
