"""What the rotary and paged entry points refuse, checked without a GPU: the checks come before any
device is touched, and CPU tensors that pass all of them are refused as CPU tensors."""

import ctypes

import pytest
import torch

from attention import _lib
from attention.paged.fused_paged import append_paged_kv, fused_paged_attention, paged_kv_cache
from attention.rotary.fused_rotary import fused_qk_norm_rotary, fused_qk_norm_rotary_autograd, rotary_table

B, H, HKV, N, D, PS = 2, 4, 2, 5, 64, 16


def rows(heads, n=N, d=D, dt=torch.float16):
    return torch.zeros(B, heads, n, d, dtype=dt)


def rotary(**kw):
    a = dict(q=rows(H), k=rows(HKV), q_weight=torch.ones(D), k_weight=torch.ones(D),
             table=rotary_table(8, 32, device="cpu"))
    a.update(kw)
    return a


def paged(**kw):
    a = dict(cache=paged_kv_cache(6, HKV, PS, D, device="cpu"), block_table=torch.zeros(B, 3, dtype=torch.int32),
             past_lens=torch.zeros(B, dtype=torch.int32))
    a.update(kw)
    return a


ROTARY = [
    (dict(q=rows(H, dt=torch.float32)), TypeError),
    (dict(k=rows(HKV, dt=torch.bfloat16)), TypeError),
    (dict(q=rows(H, d=48), k=rows(HKV, d=48)), ValueError),
    (dict(k=rows(HKV, n=N + 1)), ValueError),
    (dict(q=rows(H)[0]), ValueError),
    (dict(q=rows(H, n=0), k=rows(HKV, n=0)), ValueError),
    (dict(k_weight=None), ValueError),
    (dict(k_weight=torch.ones(D, dtype=torch.float16)), TypeError),
    (dict(q_weight=torch.ones(D, dtype=torch.bfloat16)), TypeError),
    (dict(q_weight=torch.ones(D + 1)), ValueError),
    (dict(table=torch.zeros(8, 24)), ValueError),
    (dict(table=torch.zeros(8, 2 * D)), ValueError),
    (dict(table=torch.zeros(8, 32).double()), TypeError),
    (dict(table=torch.zeros(0, 32)), ValueError),
    (dict(table=None, positions=torch.zeros(N, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(N)), TypeError),
    (dict(positions=torch.zeros(B, N + 1, dtype=torch.int32)), ValueError),
    (dict(sections=(4, 6, 6)), ValueError),
    (dict(sections=(4, 6, 7), positions=torch.zeros(3, B, N, dtype=torch.int32)), ValueError),
    (dict(sections=(4, 4, 4, 4), positions=torch.zeros(4, B, N, dtype=torch.int32)), ValueError),
    (dict(sections=(20, -4), positions=torch.zeros(2, B, N, dtype=torch.int32)), ValueError),
    (dict(sections=(4, 6, 6), positions=torch.zeros(2, B, N, dtype=torch.int32)), ValueError),
    (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(), ValueError),   # all of it right, on the CPU
]


@pytest.mark.parametrize("entry", [fused_qk_norm_rotary, fused_qk_norm_rotary_autograd])
@pytest.mark.parametrize("i", range(len(ROTARY)))
def test_rotary_refuses(entry, i):
    kw, error = ROTARY[i]
    with pytest.raises(error) as e:
        entry(**rotary(**kw))
    assert ("GPU" in str(e.value)) == (i == len(ROTARY) - 1)


def cache_with(i, t):
    c = list(paged_kv_cache(6, HKV, PS, D, device="cpu"))
    c[i] = t
    return c


CACHES = [
    (dict(cache=cache_with(0, torch.zeros(6, HKV, PS, D, dtype=torch.uint8))), TypeError),
    (dict(cache=cache_with(2, torch.zeros(6, HKV))), TypeError),
    (dict(cache=cache_with(1, torch.zeros(6, HKV, PS, 32, dtype=torch.float8_e4m3fn))), ValueError),
    (dict(cache=cache_with(3, torch.zeros(5, HKV, dtype=torch.uint8).view(torch.float8_e8m0fnu))), ValueError),
    (dict(cache=[t.transpose(0, 1).contiguous().transpose(0, 1) for t in paged_kv_cache(6, HKV, PS, D, device="cpu")]),
     ValueError),
    (dict(cache=paged_kv_cache(6, HKV, PS, 32, device="cpu")), ValueError),
    (dict(cache=paged_kv_cache(6, 3, PS, D, device="cpu")), ValueError),
    (dict(block_table=torch.zeros(B, 3, dtype=torch.int64)), TypeError),
    (dict(block_table=torch.zeros(B + 1, 3, dtype=torch.int32)), ValueError),
    (dict(block_table=torch.zeros(B, 0, dtype=torch.int32)), ValueError),
    (dict(past_lens=torch.zeros(B, dtype=torch.int64)), TypeError),
    (dict(past_lens=torch.zeros(B, 1, dtype=torch.int32)), ValueError),
    (dict(new_lens=torch.zeros(B + 1, dtype=torch.int32)), ValueError),
    (dict(new_lens=torch.zeros(B)), TypeError),
    (dict(), ValueError),
]


@pytest.mark.parametrize("i", range(len(CACHES)))
def test_paged_calls_refuse(i):
    kw, error = CACHES[i]
    a = paged(**kw)
    with pytest.raises(error) as e:
        fused_paged_attention(rows(H), **a)
    assert ("GPU" in str(e.value)) == (i == len(CACHES) - 1)
    with pytest.raises(error) as e:
        append_paged_kv(a.pop("cache"), rows(HKV), rows(HKV), q=rows(H), **a)
    assert ("GPU" in str(e.value)) == (i == len(CACHES) - 1)


@pytest.mark.parametrize("kw,error", [
    (dict(v=rows(HKV, dt=torch.bfloat16)), TypeError),
    (dict(v=rows(HKV, n=N + 1)), ValueError),
    (dict(q=rows(H, dt=torch.bfloat16)), TypeError),
    (dict(q=rows(H, n=N + 1)), ValueError),
    (dict(q_weight=torch.ones(D)), ValueError),
    (dict(q=rows(H), k_weight=torch.ones(D)), ValueError),
    (dict(k_weight=torch.ones(D - 1)), ValueError),
    (dict(table=torch.zeros(8, 40)), ValueError),
    (dict(k=rows(1), v=rows(1)), ValueError),
])
def test_append_refuses(kw, error):
    a = paged(k=rows(HKV), v=rows(HKV))
    a.update(kw)
    with pytest.raises(error):
        append_paged_kv(**a)


def test_attention_refuses_heads_that_do_not_share():
    with pytest.raises(ValueError):
        fused_paged_attention(rows(5), **paged())


@pytest.mark.parametrize("args", [(0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 24, 64), (4, 2, 16, 96)])
def test_cache_refuses(args):
    with pytest.raises(ValueError):
        paged_kv_cache(*args, device="cpu")


@pytest.mark.parametrize("args", [(0, 32), (8, 0), (8, 31)])
def test_table_refuses(args):
    with pytest.raises(ValueError):
        rotary_table(*args, device="cpu")


# ---- the C entries: status codes before any launch

class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_longlong) for n in ("b", "h", "n")]


class Rotation(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("table", "positions", "q_weight", "k_weight")] +
                [(n, ctypes.c_longlong) for n in ("pos_axis", "pos_batch")] +
                [(n, ctypes.c_int) for n in ("table_len", "rotary_dim", "axes", "int64", "end0", "end1", "weight_dtype",
                                             "interleaved")] + [("eps", ctypes.c_float)])


class Cache(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "block_table")] +
                [("table_stride", ctypes.c_longlong)] +
                [(n, ctypes.c_int) for n in ("table_width", "num_pages", "page_size", "H_kv")])


FAKE, NULL = 0x1000, None   # never dereferenced: each case fails a check before a launch


def qk(lib, rows=None, rot=None, B=1, H=4, Hkv=2, N=8, D=64, dtype=0, bwd=False, ws=NULL, ws_bytes=0):
    r = Rows(FAKE, 512, 64, 64) if rows is None else rows
    t = Rotation(table=FAKE, table_len=8, rotary_dim=64, axes=1) if rot is None else rot
    p, q = ctypes.byref(r), ctypes.byref(t)
    if bwd:
        return lib.fa_qk_norm_rotary_bwd(p, p, p, p, p, p, FAKE, FAKE, q, B, H, Hkv, N, D, dtype, ws, ws_bytes, NULL)
    return lib.fa_qk_norm_rotary(p, p, p, p, q, B, H, Hkv, N, D, dtype, NULL)


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(B=0), _lib.FA_ERR_DIMS), (dict(N=0), _lib.FA_ERR_DIMS), (dict(Hkv=0), _lib.FA_ERR_DIMS),
    (dict(B=1 << 15, N=1 << 15, H=4), _lib.FA_ERR_DIMS), (dict(dtype=2), _lib.FA_ERR_DTYPE),
    (dict(D=96), _lib.FA_ERR_HEADDIM), (dict(rows=Rows(FAKE + 8, 512, 64, 64)), _lib.FA_ERR_LAYOUT),
    (dict(rows=Rows(FAKE, 512, 60, 64)), _lib.FA_ERR_LAYOUT), (dict(rows=Rows(NULL, 512, 64, 64)), _lib.FA_ERR_NULL),
    (dict(rot=Rotation(table=FAKE, table_len=8, rotary_dim=128, axes=1)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(table=FAKE, table_len=8, rotary_dim=24, axes=1)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(table=FAKE, table_len=0, rotary_dim=32, axes=1)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(table=FAKE, table_len=8, rotary_dim=32, axes=2)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(table=FAKE, positions=FAKE, table_len=8, rotary_dim=32, axes=4)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(table=FAKE, positions=FAKE, table_len=8, rotary_dim=32, axes=3, end0=9, end1=8)),
     _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(q_weight=FAKE)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(q_weight=FAKE, k_weight=FAKE, weight_dtype=1)), _lib.FA_ERR_ROTATION),
    (dict(rot=Rotation(q_weight=FAKE, k_weight=FAKE + 4, weight_dtype=0)), _lib.FA_ERR_ROTATION),
])
def test_rotary_entries_reject(lib, kw, code, bwd):
    assert qk(lib, bwd=bwd, **kw) == code


def test_rotary_backward_needs_its_workspace(lib):
    t = Rotation(q_weight=FAKE, k_weight=FAKE, weight_dtype=0)
    need = lib.fa_qk_norm_rotary_workspace_size(1, 4, 2, 8, 64)
    assert need > 0 and need % 256 == 0
    assert qk(lib, rot=t, bwd=True) == _lib.FA_ERR_NULL
    assert qk(lib, rot=t, bwd=True, ws=FAKE, ws_bytes=need - 1) == _lib.FA_ERR_WORKSPACE
    assert qk(lib, rot=t, bwd=True, ws=FAKE + 4, ws_bytes=need) == _lib.FA_ERR_WORKSPACE
    assert lib.fa_qk_norm_rotary_workspace_size(1, 4, 0, 8, 64) == 0


def pages(**kw):
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, block_table=FAKE, table_stride=4, table_width=4, num_pages=9,
             page_size=16, H_kv=2)
    a.update(kw)
    return Cache(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(cache=pages(page_size=48)), _lib.FA_ERR_PAGES), (dict(cache=pages(num_pages=0)), _lib.FA_ERR_PAGES),
    (dict(cache=pages(table_width=0)), _lib.FA_ERR_PAGES), (dict(cache=pages(k=FAKE + 8)), _lib.FA_ERR_PAGES),
    (dict(cache=pages(v=NULL)), _lib.FA_ERR_NULL), (dict(cache=pages(H_kv=0)), _lib.FA_ERR_PAGES),
    (dict(past=NULL), _lib.FA_ERR_NULL), (dict(N=0), _lib.FA_ERR_DIMS), (dict(dtype=3), _lib.FA_ERR_DTYPE),
    (dict(D=80), _lib.FA_ERR_HEADDIM), (dict(rows=Rows(FAKE, 512, 64, 4)), _lib.FA_ERR_LAYOUT),
])
def test_paged_entries_reject(lib, kw, code):
    r = ctypes.byref(kw.get("rows", Rows(FAKE, 512, 64, 64)))
    c = ctypes.byref(kw.get("cache", pages()))
    t = ctypes.byref(Rotation())
    past, n, d, dt = kw.get("past", FAKE), kw.get("N", 8), kw.get("D", 64), kw.get("dtype", 0)
    assert lib.fa_paged_append(r, r, r, r, c, past, NULL, t, 1, 4, n, d, dt, NULL) == code
    assert lib.fa_paged_attention(r, c, past, NULL, r, NULL, 1, 4, n, d, dt, 0.1, NULL, 0, NULL) == code


def test_paged_attention_entry_rejects_heads_and_workspaces(lib):
    r, c = ctypes.byref(Rows(FAKE, 512, 64, 64)), ctypes.byref(pages())
    call = lambda H, ws: lib.fa_paged_attention(r, c, FAKE, NULL, r, NULL, 1, H, 8, 64, 0, 0.1, ws, 64, NULL)  # noqa: E731
    assert call(3, NULL) == _lib.FA_ERR_DIMS
    assert call(4, FAKE + 4) == _lib.FA_ERR_WORKSPACE
    assert lib.fa_paged_attention_workspace_size(1, 3, 2, 8, 64, 100) == 0
    for code in (_lib.FA_ERR_LAYOUT, _lib.FA_ERR_ROTATION, _lib.FA_ERR_PAGES):
        assert lib.fa_strerror(code).decode() != "unknown status"
        with pytest.raises(ValueError):
            _lib.check(code, "x")


@pytest.mark.parametrize("rows,parts,ws,size,code", [
    (64, 1, NULL, 0, _lib.FA_ERR_TILE), (0, 1, NULL, 0, _lib.FA_ERR_TILE),
    (16, 0, NULL, 0, _lib.FA_ERR_UNSUPPORTED), (256, 129, FAKE, 1 << 40, _lib.FA_ERR_UNSUPPORTED),
    (16, 2, NULL, 0, _lib.FA_ERR_WORKSPACE), (16, 2, FAKE, 2 * 2 * 16 * 68 * 4 - 1, _lib.FA_ERR_WORKSPACE),
    (128, 3, FAKE, 2 * 3 * 128 * 68 * 4 - 1, _lib.FA_ERR_WORKSPACE), (16, 2, FAKE + 4, 1 << 40, _lib.FA_ERR_WORKSPACE),
])
def test_exact_cut_rejects(lib, rows, parts, ws, size, code):
    r, c = ctypes.byref(Rows(FAKE, 512, 64, 64)), ctypes.byref(pages())
    assert lib.fa_paged_attention_exact(r, c, FAKE, NULL, r, NULL, 1, 4, 8, 64, 0, 0.1, rows, parts, ws, size, NULL) == code
    assert lib.fa_paged_attention_exact(r, c, FAKE, NULL, r, NULL, 1, 3, 8, 64, 0, 0.1, rows, parts, ws, size, NULL) == _lib.FA_ERR_DIMS
