"""Refusals of the paged-cache operators, and their argument structures (CPU only: every
check here comes before the device is touched)."""
import ctypes as C
import re
from pathlib import Path

import pytest

from yanaiengine_b200 import abi

ROOT = Path(__file__).resolve().parents[1]
A = 1 << 20  # a 16-byte aligned address that is never read


def pages(**kw):
    p = abi.KVPages(A, A, abi.KV_E4M3, 64, 2, 2, 128)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def append_args(pages_=None, **kw):
    a = abi.KVAppendArgs(pages_ or pages(), 1, 8, 4, abi.DTYPE_F32, abi.DTYPE_BF16, 1e-5, A, 8 * 128, A, 4 * 128, A, A, A,
                         A, A)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention_args(pages_=None, **kw):
    a = abi.AttentionE4M3Args(pages_ or pages(), 1, 8, 2, 4, abi.DTYPE_BF16, 4, 0, 0, 0.0, 0.0, A, 4 * 128, A, 4 * 128, A,
                              A, A, A, 1 << 30, A)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_PAGES = [dict(data=0), dict(data=A + 8), dict(scales=0), dict(kind=3), dict(kind=-1), dict(num_blocks=0),
             dict(num_blocks=(1 << 27) + 1), dict(n_layers=0), dict(n_layers=1), dict(n_kv_heads=0), dict(n_kv_heads=3),
             dict(head_dim=96), dict(head_dim=0)]


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_pages_are_checked(bad):
    for make, fn in ((append_args, abi.lib().yk_kv_append), (attention_args, abi.lib().yk_attention_e4m3)):
        assert fn(0, None, C.byref(make(pages(**bad)))) == abi.YK_ERR_ARG, bad


@pytest.mark.parametrize("bad,status", [
    (dict(layer=2), 1), (dict(layer=-1), 1), (dict(T=-1), 1), (dict(n_heads=0), 1), (dict(n_heads=5), 1),
    (dict(src_dtype=abi.DTYPE_BF16, q_dtype=abi.DTYPE_F32), 7), (dict(src_dtype=abi.DTYPE_F16), 7), (dict(q_dtype=9), 7),
    (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(qkv=0), 1), (dict(q_out=0), 1), (dict(slots=0), 1),
    (dict(qkv=A + 4), 1), (dict(q_out=A + 8), 1), (dict(rope=A + 4), 1), (dict(q_gain=A + 4), 1), (dict(k_gain=A + 4), 1),
    (dict(qkv_stride=8 * 128 - 4), 1), (dict(qkv_stride=8 * 128 + 2), 1), (dict(q_stride=4 * 128 - 8), 1),
    (dict(q_stride=4 * 128 + 4), 1)])
def test_append_refuses(bad, status):
    assert abi.lib().yk_kv_append(0, None, C.byref(append_args(**bad))) == status, bad
    assert abi.last_error()


def test_append_refuses_cells_of_another_type():
    for kind in (abi.KV_F32, abi.KV_BF16):
        q = abi.DTYPE_BF16 if kind == abi.KV_F32 else abi.DTYPE_F32
        a = append_args(pages(kind=kind, scales=0), q_dtype=q)
        assert abi.lib().yk_kv_append(0, None, C.byref(a)) == abi.YK_ERR_ARG
        # scales belong to 8-bit cells alone
        assert abi.lib().yk_kv_append(0, None, C.byref(append_args(pages(kind=kind)))) == abi.YK_ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(layer=2), dict(T=-1), dict(B=0), dict(B=(1 << 20) + 1), dict(n_heads=3), dict(dtype=abi.DTYPE_F16),
    dict(max_blocks=0), dict(max_new=-1), dict(window=-1), dict(scale=-1.0), dict(scale=float("inf")),
    dict(cap=float("nan")), dict(cap=-2.0), dict(q=0), dict(out=0), dict(q=A + 8), dict(out=A + 4), dict(q_starts=0),
    dict(context_lens=0), dict(block_tables=0), dict(workspace=0), dict(workspace=A + 4), dict(q_stride=500),
    dict(q_stride=4 * 128 + 4), dict(out_stride=4 * 128 + 1)])
def test_attention_refuses(bad):
    assert abi.lib().yk_attention_e4m3(0, None, C.byref(attention_args(**bad))) == abi.YK_ERR_ARG, bad
    assert abi.last_error()


def test_attention_reads_8_bit_pools_only():
    for kind in (abi.KV_F32, abi.KV_BF16):
        assert abi.lib().yk_attention_e4m3(0, None, C.byref(attention_args(pages(kind=kind, scales=0)))) == abi.YK_ERR_ARG


def test_null_argument_structures():
    n = C.c_uint64()
    assert abi.lib().yk_kv_append(0, None, None) == abi.YK_ERR_ARG
    assert abi.lib().yk_attention_e4m3(0, None, None) == abi.YK_ERR_ARG
    assert abi.lib().yk_attention_e4m3_workspace(0, 128, None) == abi.YK_ERR_ARG
    assert abi.lib().yk_attention_e4m3_workspace(0, 100, C.byref(n)) == abi.YK_ERR_ARG


@pytest.mark.parametrize("name,cls", [("yk_kv_pages", abi.KVPages), ("yk_kv_append_args", abi.KVAppendArgs),
                                      ("yk_attention_e4m3_args", abi.AttentionE4M3Args)])
def test_structures_match_the_header(name, cls):
    text = (ROOT / "include" / "yk.h").read_text()
    body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body.split("{", 1)[1], flags=re.S)
    fields = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            fields += [re.sub(r"[\s*]", "", x).split()[-1] for x in
                       re.sub(r"^(const\s+)?\w+\s*\**\s*", "", decl).split(",")]
    assert fields == [f for f, _ in cls._fields_]


def test_wrapper_checks_tensors_on_the_host():
    import torch

    pool = torch.zeros(4, 2, 2, 2, 16, 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="not on cuda"):
        abi._pages(pool, torch.zeros(4, 2, 2, 2, dtype=torch.uint8), 0)
    with pytest.raises(ValueError, match="must be"):
        abi._pages(pool[:, :, :1], None, 0)
    with pytest.raises(ValueError, match="not on cuda"):
        abi.kv_append(pool, None, 0, torch.zeros(1, 256), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32), None,
                      None, None, 1e-5, None, 2)


def test_packed_arguments_match_the_structures():
    a = attention_args(layer=1, window=7, scale=0.5, cap=2.0, workspace_bytes=77)
    p = a.pages
    raw = abi._ATTENTION.pack(p.data, p.scales, p.kind, p.num_blocks, p.n_layers, p.n_kv_heads, p.head_dim, a.layer, a.T, a.B,
                              a.n_heads, a.dtype, a.max_blocks, a.max_new, a.window, a.scale, a.cap, a.q, a.q_stride, a.out,
                              a.out_stride, a.q_starts, a.context_lens, a.block_tables, a.workspace, a.workspace_bytes, a.err)
    b = abi.AttentionE4M3Args.from_buffer_copy(raw)
    assert all(getattr(a, f) == getattr(b, f) for f, _ in a._fields_[1:])
    assert all(getattr(a.pages, f) == getattr(b.pages, f) for f, _ in p._fields_)
    a = append_args(layer=1, eps=0.5)
    raw = abi._APPEND.pack(p.data, p.scales, p.kind, p.num_blocks, p.n_layers, p.n_kv_heads, p.head_dim, a.layer, a.T, a.n_heads,
                           a.src_dtype, a.q_dtype, a.eps, a.qkv, a.qkv_stride, a.q_out, a.q_stride, a.slots, a.rope, a.q_gain,
                           a.k_gain, a.err)
    b = abi.KVAppendArgs.from_buffer_copy(raw)
    assert all(getattr(a, f) == getattr(b, f) for f, _ in a._fields_[1:])
