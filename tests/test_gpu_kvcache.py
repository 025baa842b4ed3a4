"""yk_kv_append and yk_attention_e4m3 against 64-bit references (tests/kvcache_ref.py),
through the C-ABI on torch device buffers."""
import math

import numpy as np
import pytest
import torch

import kvcache_ref as ref
from yanaiengine_b200 import abi

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn


def dev():
    return torch.device("cuda", 0)


def e4m3_pool(rng, blocks, layers, G, dh, spread=2.0):
    """Random codes (no NaN) and scale bytes of unequal size."""
    g = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    x = torch.randn(blocks, layers, 2, G, 16, dh, generator=g) * 60.0
    pool = x.clamp(-448, 448).to(F8).view(torch.uint8)
    byte = (torch.randn(blocks, layers, 2, G, generator=g) * spread - 6).round() + 127
    return pool.to(dev()), byte.to(torch.uint8).to(dev())


def batch(rng, blocks, lens):
    """lens: (new, ctx) of each sequence -> starts, ctx, tables (int32, host)."""
    order = rng.permutation(blocks).tolist()
    width = max(1, max((c + 15) // 16 for _, c in lens))
    tables = np.zeros((len(lens), width), np.int32)
    starts = [0]
    for b, (n, c) in enumerate(lens):
        for i in range((c + 15) // 16):
            tables[b, i] = order.pop()
        starts.append(starts[-1] + n)
    return starts, [c for _, c in lens], tables


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev())


class Attention:
    """Inputs of one call, and the call."""

    def __init__(self, seed, H, G, dh, lens, dtype="bf16", layers=2, layer=1, pad=0, q_std=1.0, spread=2.0, spare=2):
        rng = np.random.default_rng(seed)
        self.blocks = sum((c + 15) // 16 for _, c in lens) + spare
        self.layer = layer
        self.pool, self.scales = e4m3_pool(rng, self.blocks, layers, G, dh, spread)
        self.starts, self.ctx, self.tables = batch(rng, self.blocks, lens)
        T = self.starts[-1] + pad
        g = torch.Generator().manual_seed(seed)
        self.q = (torch.randn(T, H, dh, generator=g) * q_std).to(DT[dtype]).to(dev())
        self.out = torch.full((T, H, dh), 7.0, dtype=DT[dtype], device=dev())
        self.err = torch.zeros(1, dtype=torch.int32, device=dev())
        self.ws = torch.zeros(abi.attention_e4m3_workspace(dh), dtype=torch.uint8, device=dev())
        self.max_new = max(n for n, _ in lens)

    def call(self, **kw):
        kw.setdefault("max_new", self.max_new)
        self.d = [i32(self.starts), i32(self.ctx), i32(self.tables)]
        abi.attention_e4m3(self.q, self.out, self.pool, self.scales, self.layer, *self.d, self.ws, self.err, **kw)

    def check(self, err=0, **kw):
        ref_kw = {k: v for k, v in kw.items() if k in ("window", "scale", "cap")}
        want, weight, spread, floor = ref.attention(self.q, self.pool, self.scales, self.layer, self.starts, self.ctx,
                                             self.tables, **ref_kw)
        self.call(**kw)
        torch.cuda.synchronize()
        self.compare(want, weight, spread, floor, err)

    def compare(self, want, weight, spread, floor, err=0):
        got = self.out.double().cpu()
        n = self.starts[-1]
        assert (got[n:] == 7.0).all(), "rows behind the last sequence were written"
        bound = ref.attention_bound(want[:n], weight[:n], spread[:n], floor[:n], want.shape[-1], self.out.dtype)
        off = (got[:n] - want[:n]).abs()
        assert not torch.isnan(got[:n]).any()
        worst = float((off / bound).max()) if n else 0.0
        assert worst <= 1.0, f"{worst:.3f} of the bound"
        assert int(self.err) == err


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,dh", [(4, 4, 64), (8, 2, 64), (3, 1, 128), (8, 1, 128), (24, 8, 128), (4, 2, 256), (16, 1, 256)])
def test_attention_decode_and_verify(dtype, H, G, dh):
    lens = [(1, 1), (1, 16), (1, 17), (3, 3), (6, 160), (5, 33), (1, 700), (2, 1031)]
    Attention(H * 100 + dh, H, G, dh, lens, dtype).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_attention_one_token_of_one_sequence(dtype, dh):
    for ctx in (1, 2, 15, 16, 31, 129, 2049):
        Attention(ctx, 8, 2, dh, [(1, ctx)], dtype).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,dh", [(4, 2, 64), (8, 1, 128), (6, 2, 128), (4, 2, 256)])
def test_attention_prompts(dtype, H, G, dh):
    Attention(dh, H, G, dh, [(97, 97), (130, 300), (1, 50), (33, 48), (16, 16)], dtype).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 37, 100, 5000])
def test_attention_window(dtype, window):
    Attention(window, 8, 2, 128, [(6, 400), (1, 65), (40, 90), (5, 5)], dtype).check(window=window)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_attention_cap_and_scale(dtype, dh):
    Attention(5, 8, 4, dh, [(6, 400), (1, 65), (20, 20)], dtype, q_std=2.0).check(cap=30.0, scale=0.21)
    Attention(6, 8, 4, dh, [(6, 300), (1, 65)], dtype, q_std=2.0).check(cap=5.0, window=50)


@pytest.mark.parametrize("max_new", [0, 1, 3, 1000])
def test_attention_whatever_max_new_says(max_new):
    Attention(8, 8, 2, 128, [(6, 400), (1, 65), (70, 90), (2, 2)]).check(max_new=max_new)


def test_attention_padding_and_empty_sequences():
    # a sequence without new tokens, rows behind the last sequence, an empty batch
    Attention(9, 8, 2, 128, [(0, 40), (3, 40), (0, 0), (1, 20), (0, 16)], pad=5).check()
    a = Attention(10, 8, 2, 128, [(0, 40), (0, 0)], pad=3)
    a.check()


def test_attention_positions_below_zero_give_zeros():
    a = Attention(11, 8, 2, 128, [(5, 40), (3, 40)])
    a.ctx[0] = 2  # five new tokens, two positions: the first three have no key
    a.check()
    assert (a.out[:3] == 0).all()


def test_attention_many_sequences():
    rng = np.random.default_rng(0)
    lens = [(1, int(c)) for c in rng.integers(1, 60, 700)]
    Attention(12, 2, 1, 64, lens).check()


def test_attention_one_long_sequence_among_short_ones():
    Attention(13, 4, 2, 64, [(1, 9000)] + [(1, 3)] * 200).check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_scales_far_apart(dtype):
    a = Attention(14, 8, 2, 128, [(4, 200), (1, 90)], dtype, spread=0.0)
    # V blocks from 2^-60 to 2^60; a sequence's result lies wherever its weights do
    byte = torch.arange(a.scales.numel()).reshape(a.scales.shape) * 7 % 121 + 67
    a.scales[:, :, 1] = byte.to(torch.uint8).to(dev())[:, :, 1]
    a.check()
    # scale bytes outside 67..187 read as the nearest of them
    a.scales[:, :, 1] = torch.tensor([0, 255], dtype=torch.uint8, device=dev())[torch.arange(2, device=dev())]
    a.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dh", [64, 128, 256])
def test_attention_nan_in_masked_cells(dtype, dh):
    lens = [(6, 101), (1, 33), (20, 40)]
    a = Attention(15, 8, 2, dh, lens, dtype)
    want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables, window=30)
    # cells past the context, and before every query's window
    for b, (n, c) in enumerate(lens):
        for j in list(range(c, (c + 15) // 16 * 16)) + list(range(0, max(0, c - n - 30 + 1))):
            a.pool[a.tables[b, j // 16], 1, :, :, j % 16] = 0x7F
    a.call(window=30)
    torch.cuda.synchronize()
    a.compare(*want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("which", [0, 1])
def test_attention_nan_cell_reaches_those_who_see_it(dtype, dh, which):
    """A NaN in the K or V of one new token: earlier tokens are untouched, later ones are NaN."""
    a = Attention(16, 4, 2, dh, [(8, 60), (1, 20)], dtype)
    want, weight, spread, floor = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    j = 60 - 3  # the sixth new token's cell
    a.pool[a.tables[0, j // 16], 1, which, 0, j % 16, 5] = 0xFF
    a.call()
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    clean = torch.ones_like(got, dtype=torch.bool)
    if which == 0:
        clean[5:8, :2] = False  # heads 0, 1 read KV head 0: every dimension
    else:
        clean[5:8, :2, 5] = False
    assert torch.isnan(got[~clean]).all()
    bound = ref.attention_bound(want, weight, spread, floor, dh, a.out.dtype)
    assert ((got - want).abs()[clean] <= bound[clean]).all()


def test_attention_block_outside_the_pool():
    """Its keys count as absent and the error word says so."""
    a = Attention(17, 8, 2, 128, [(1, 64), (6, 70), (1, 30)])
    want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    a.tables[0, 1], a.tables[0, 2] = a.blocks, -1
    a.call()
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    bound = ref.attention_bound(*want, 128, a.out.dtype)
    assert ((got - want[0]).abs()[1:] <= bound[1:]).all()
    assert not torch.isnan(got).any() and int(a.err) == 1


def test_attention_context_beyond_the_table():
    a = Attention(18, 8, 2, 128, [(1, 64), (6, 70)])
    want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    a.ctx[0] = 64 + 1600
    a.call()
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    bound = ref.attention_bound(*want, 128, a.out.dtype)
    assert ((got - want[0]).abs()[1:] <= bound[1:]).all()
    assert not torch.isnan(got).any() and int(a.err) == 1


def test_attention_starts_that_do_not_fit():
    """q_starts that fall or pass T: nothing outside the tensors is touched, the error word says so."""
    for starts in ([0, 4, 2, 6], [0, 2, 4, 900], [0, -5, 2, 6], [3, 1, 2, 6]):
        a = Attention(19, 8, 2, 64, [(2, 30), (2, 30), (2, 30)], pad=2)
        a.starts = starts
        a.call()
        torch.cuda.synchronize()
        assert int(a.err) == 1


def test_attention_strided_rows_and_first_layer():
    a = Attention(20, 8, 2, 128, [(6, 100), (1, 33)], layers=3, layer=0)
    wide = torch.randn(a.q.shape[0], 12, 128, device=dev()).to(torch.bfloat16)
    wide[:, :8] = a.q
    a.q = wide[:, :8]
    big = torch.full((a.q.shape[0], 10, 128), 7.0, dtype=torch.bfloat16, device=dev())
    a.out = big[:, 2:]
    a.check()
    assert (big[:, :2] == 7.0).all()


def test_attention_pool_beyond_32_bit_offsets():
    blocks, L, G, dh = 70000, 4, 4, 128  # 4.6 GB of cells
    a = Attention(21, 8, G, dh, [(1, 40), (6, 100)])
    pool = torch.empty(blocks, L, 2, G, 16, dh, dtype=torch.uint8, device=dev())
    scales = torch.empty(blocks, L, 2, G, dtype=torch.uint8, device=dev())
    moved = a.tables.copy()
    for b, (n, c) in enumerate([(1, 40), (6, 100)]):
        for i in range((c + 15) // 16):
            moved[b, i] = blocks - 1 - int(a.tables[b, i])
            pool[int(moved[b, i]), 3] = a.pool[int(a.tables[b, i]), 1]
            scales[int(moved[b, i]), 3] = a.scales[int(a.tables[b, i]), 1]
    a.pool, a.scales, a.tables, a.layer = pool, scales, moved, 3
    a.check()


def test_attention_does_not_overflow_on_large_scores():
    Attention(22, 8, 2, 128, [(6, 300), (1, 90)], q_std=200.0).check()
    Attention(23, 8, 2, 128, [(6, 300), (1, 90)], q_std=1e-6).check()


def test_attention_large_and_small_queries():
    for mag in (1e30, 1e-30):
        a = Attention(24, 4, 2, 64, [(3, 200)], "bf16")
        a.q = (a.q.float() * mag).to(torch.bfloat16)
        a.check(scale=float(0.125 / mag) if mag > 1 else 1e30)


def test_attention_captured_and_replayed_with_other_lengths():
    a = Attention(25, 8, 2, 128, [(6, 500), (2, 90), (1, 333)])
    a.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        abi.attention_e4m3(a.q, a.out, a.pool, a.scales, a.layer, *a.d, a.ws, a.err, max_new=6)
    for ctx in ([500, 90, 333], [100, 64, 3], [6, 2, 1]):
        a.ctx = ctx
        a.d[1].copy_(i32(ctx))
        a.out.fill_(7.0)
        want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
        g.replay()
        torch.cuda.synchronize()
        a.compare(*want)


def test_attention_on_another_stream_and_again_on_the_same_workspace():
    a = Attention(26, 8, 2, 128, [(6, 900), (1, 90)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            a.call()
    torch.cuda.current_stream().wait_stream(side)
    first = a.out.clone()
    a.check()
    assert torch.equal(first, a.out), "the same call twice gives the same bits"
    b = Attention(27, 8, 2, 128, [(3, 2000), (1, 5)])
    b.ws = a.ws
    b.check()


def test_attention_nothing_to_do_and_workspace_size():
    a = Attention(28, 8, 2, 128, [(0, 20)])
    assert a.q.shape[0] == 0
    a.call()
    torch.cuda.synchronize()
    b = Attention(29, 8, 2, 128, [(1, 20)])
    b.ws = b.ws[: b.ws.numel() - 16]
    with pytest.raises(abi.YKError) as e:
        b.call()
    assert e.value.status == abi.YK_ERR_ARG and (b.out == 7.0).all()


# ---------------------------------------------------------------------------
# Append.
# ---------------------------------------------------------------------------
class Append:
    def __init__(self, seed, H, G, dh, lens, src="f32", dst="bf16", cache="e4m3", norm=True, rope=True, layers=2, layer=1):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.H, self.G, self.dh, self.layer, self.cache = H, G, dh, layer, cache
        self.blocks = sum((c + 15) // 16 for _, c in lens) + 2
        if cache == "e4m3":
            self.pool, self.scales = e4m3_pool(rng, self.blocks, layers, G, dh)
        else:
            self.pool = torch.randn(self.blocks, layers, 2, G, 16, dh, generator=g).to(DT[cache]).to(dev())
            self.scales = None
        starts, ctx, tables = batch(rng, self.blocks, lens)
        pos = np.concatenate([np.arange(c - n, c) for n, c in lens]).astype(int)
        seq = np.repeat(np.arange(len(lens)), [n for n, _ in lens])
        self.slots = np.asarray([tables[b, p // 16] * 16 + p % 16 for b, p in zip(seq, pos)], np.int32)
        T = len(pos)
        self.qkv = (torch.randn(T, (H + 2 * G) * dh, generator=g) * torch.rand(T, 1, generator=g).mul(4).exp2()).to(
            DT[src]).to(dev())
        self.q = torch.full((T, H, dh), 7.0, dtype=DT[dst], device=dev())
        ang = torch.as_tensor(pos)[:, None] * 10000.0 ** (-torch.arange(0, dh, 2, dtype=torch.float64) / dh)
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous().to(dev()) if rope else None
        self.qg = (torch.rand(dh, generator=g) + 0.5).to(dev()) if norm else None
        self.kg = (torch.rand(dh, generator=g) + 0.5).to(dev()) if norm else None
        self.eps = 1e-5
        self.err = torch.zeros(1, dtype=torch.int32, device=dev())

    def call(self, lo=0, hi=None, **kw):
        hi = len(self.slots) if hi is None else hi
        self.d = i32(self.slots[lo:hi])
        abi.kv_append(self.pool, self.scales, self.layer, self.qkv[lo:hi], self.q[lo:hi], self.d,
                      self.rope[lo:hi] if self.rope is not None else None, self.qg, self.kg, self.eps, self.err, self.H, **kw)

    def wanted(self):
        """(q, k, v) in float64."""
        x = self.qkv.double().cpu().view(len(self.slots), self.H + 2 * self.G, self.dh)
        gain = (lambda t: None if t is None else t.cpu())
        rope = gain(self.rope)
        q = ref.rotated(ref.normed(x[:, :self.H], gain(self.qg), self.eps), rope)
        k = ref.rotated(ref.normed(x[:, self.H:self.H + self.G], gain(self.kg), self.eps), rope)
        return q, k, x[:, self.H + self.G:]

    def check(self, **kw):
        old_pool, old_scales = self.pool.cpu().clone(), None if self.scales is None else self.scales.cpu().clone()
        q, k, v = self.wanted()
        self.call(**kw)
        torch.cuda.synchronize()
        self.compare(q, k, v, old_pool, old_scales)

    def slack(self, x):
        """fp32 arithmetic of the norm and the rotation: a sum of dh squares in a tree (8 + 5 roundings), a root
        (2 steps), two products, then two products and a sum: below 24 roundings of 2^-24, relative to the
        pair's size (the rotation mixes the two; without it each value stands alone)."""
        if self.rope is None:
            return x.abs() * 24 * 2.0 ** -24
        pair = x.reshape(*x.shape[:-1], -1, 2).abs().sum(-1, keepdim=True).expand(*x.shape[:-1], x.shape[-1] // 2, 2)
        return pair.reshape(x.shape) * 24 * 2.0 ** -24

    def compare(self, q, k, v, old_pool, old_scales):
        live = torch.as_tensor(self.slots) >= 0
        got = self.q.double().cpu()
        half = torch.finfo(self.q.dtype).eps / 2
        assert (got[~live] == 7.0).all()
        assert ((got - q).abs()[live] <= (q.abs() * half + self.slack(q) * (1 + half) + 1e-37)[live]).all()
        assert int(self.err) == 0
        kv = torch.stack([k, v], 1)  # [T, 2, G, dh]
        tol = torch.stack([self.slack(k), torch.zeros_like(v)], 1)
        pool, want_pool = self.pool.cpu(), old_pool.clone()
        if self.cache != "e4m3":
            half = torch.finfo(pool.dtype).eps / 2
            for t, s in enumerate(self.slots):
                if s < 0:
                    continue
                cell = pool[s // 16, self.layer, :, :, s % 16].double()
                assert ((cell - kv[t]).abs() <= kv[t].abs() * half + tol[t] * (1 + half) + 1e-37).all()
                want_pool[s // 16, self.layer, :, :, s % 16] = pool[s // 16, self.layer, :, :, s % 16]
            assert torch.equal(pool, want_pool), "cells outside the new slots changed"
            return
        scales, want_scales = self.scales.cpu(), old_scales.clone()
        runs = {}
        for t, s in enumerate(self.slots):
            if s >= 0:
                runs.setdefault(int(s) // 16, []).append(t)
        for blk, rows in runs.items():
            at = [int(self.slots[t]) % 16 for t in rows]
            older = [i for i in range(max(at)) if i not in at]
            for c in range(2):
                for g in range(self.G):
                    x, dx = kv[rows, c, g], tol[rows, c, g]
                    byte = int(scales[blk, self.layer, c, g])
                    had = min(max(int(old_scales[blk, self.layer, c, g]) - 127, ref.EMIN), ref.EMAX)
                    fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
                    i = int(fin.argmax())
                    # the exponents that the fp32 largest value may ask for
                    may = {ref.cover(max(0.0, float(fin.flatten()[i] + s * dx.flatten()[i]))) for s in (-1, 0, 1)}
                    if older:
                        may = {max(had, e) for e in may}
                    assert byte - 127 in may, (byte - 127, may)
                    e = byte - 127
                    cell = pool[blk, self.layer, c, g]
                    val = cell[at].view(F8).double() * 2.0 ** e
                    bad = torch.isnan(x)
                    assert torch.equal(torch.isnan(val), bad)
                    sat = x.clamp(-448 * 2.0 ** e, 448 * 2.0 ** e)
                    # half a step: 2^-4 of the value, or of the smallest normal cell 2^-6
                    lim = torch.maximum(sat.abs(), torch.tensor(2.0 ** (e - 6))) * 2.0 ** -4 + dx * 1.07
                    assert ((val - sat).abs()[~bad] <= lim[~bad]).all()
                    if older:
                        kept = old_pool[blk, self.layer, c, g, older]
                        exact = kept.view(F8).double() * 2.0 ** had
                        assert torch.equal(cell[older], kept if e == had else ref.encode(exact, e))
                    want_pool[blk, self.layer, c, g, :max(at) + 1] = cell[:max(at) + 1]
                    want_scales[blk, self.layer, c, g] = byte
        assert torch.equal(pool, want_pool), "cells past the new ones, of another layer or block changed"
        assert torch.equal(scales, want_scales)


LENS = [(1, 1), (1, 16), (1, 17), (6, 37), (5, 5), (40, 100), (16, 32), (17, 17), (2, 18), (31, 63)]


@pytest.mark.parametrize("src,dst,cache", [("f32", "bf16", "e4m3"), ("bf16", "bf16", "e4m3"), ("f32", "f32", "e4m3"),
                                           ("f32", "bf16", "bf16"), ("bf16", "bf16", "bf16"), ("f32", "f32", "f32")])
@pytest.mark.parametrize("H,G,dh", [(4, 4, 64), (8, 2, 128), (3, 1, 256)])
def test_append(src, dst, cache, H, G, dh):
    Append(dh, H, G, dh, LENS, src, dst, cache).check()


@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("cache", ["e4m3", "bf16"])
def test_append_without_norm_or_rotation(norm, rope, cache):
    Append(3, 6, 2, 128, LENS, cache=cache, norm=norm, rope=rope).check()


def test_append_long_prompt():
    Append(4, 4, 1, 64, [(3000, 3001), (1111, 1111)]).check()


def test_append_is_repeatable():
    a = Append(5, 8, 2, 128, LENS)
    a.call()
    pool, scales, q = a.pool.clone(), a.scales.clone(), a.q.clone()
    a.call()
    assert torch.equal(pool, a.pool) and torch.equal(scales, a.scales) and torch.equal(q, a.q)


def test_append_token_by_token_then_rolled_back():
    """One token at a time: a block's scale only grows; appending at an earlier offset again keeps it."""
    a = Append(6, 4, 2, 128, [(40, 40)])
    last = None
    for t in range(40):
        old_pool, old_scales = a.pool.cpu().clone(), a.scales.cpu().clone()
        a.call(t, t + 1)
        torch.cuda.synchronize()
        b = Append.__new__(Append)
        b.__dict__.update(a.__dict__, slots=a.slots[t:t + 1], q=a.q[t:t + 1], qkv=a.qkv[t:t + 1], rope=a.rope[t:t + 1])
        b.compare(*b.wanted(), old_pool, old_scales)
        now = a.scales[int(a.slots[t]) // 16, 1].clone()
        if t % 16:
            assert (now >= last).all()
        last = now
    old_pool, old_scales = a.pool.cpu().clone(), a.scales.cpu().clone()
    a.call(35, 38)  # rolled back to 35 tokens
    torch.cuda.synchronize()
    assert (a.scales.cpu() == old_scales).all()
    # (their cells need not be the same bits: the first time they were rounded at the scale the block had then, and
    # again when it grew; now once, at the grown one)
    b.__dict__.update(slots=a.slots[35:38], q=a.q[35:38], qkv=a.qkv[35:38], rope=a.rope[35:38])
    b.compare(*b.wanted(), old_pool, old_scales)


def test_append_padding_and_slots_outside_the_pool():
    a = Append(7, 8, 2, 128, LENS)
    a.slots[[0, 5, 9]] = -1
    a.check()
    b = Append(8, 8, 2, 128, [(1, 40), (1, 20), (1, 3)])
    old, q = b.pool.clone(), b.wanted()[0]
    good = b.slots.copy()
    b.slots[1] = b.blocks * 16 + 4
    b.call()
    torch.cuda.synchronize()
    assert int(b.err) == 1
    changed = (b.pool != old).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted({int(good[0]) // 16, int(good[2]) // 16})
    assert ((b.q.double().cpu() - q).abs() <= q.abs() * 2.0 ** -8 + 1e-3).all()


def test_append_values_that_are_not_finite_zero_or_huge():
    a = Append(9, 4, 2, 128, [(6, 22), (20, 20), (1, 40)], norm=False, rope=False)
    x = a.qkv.view(27, 8, 128)
    x[1, 4, 3], x[1, 6, 9] = math.nan, math.nan
    x[2, 5, 7], x[2, 7, 8] = math.inf, -math.inf
    x[8] = 0.0
    x[10, 4:] = 1e30   # beyond 448 * 2^60: saturates
    x[26, 4:] = 0.0    # a block with an older scale and a zero token
    old_pool, old_scales = a.pool.cpu().clone(), a.scales.cpu().clone()
    q, k, v = a.wanted()
    a.call()
    torch.cuda.synchronize()
    a.compare(q, k, v, old_pool, old_scales)
    z = Append(10, 4, 2, 64, [(5, 5)], norm=False, rope=False)
    z.qkv.zero_()
    z.check()
    assert (z.scales[int(z.slots[0]) // 16, 1] == 127 + ref.EMIN).all()


def test_append_strided_rows():
    a = Append(11, 4, 2, 128, LENS, src="bf16")
    wide = torch.randn(a.qkv.shape[0], a.qkv.shape[1] + 256, device=dev()).to(torch.bfloat16)
    wide[:, 128:-128] = a.qkv
    a.qkv = wide[:, 128:-128]
    big = torch.full((a.q.shape[0], 7, 128), 7.0, dtype=torch.bfloat16, device=dev())
    a.q = big[:, 1:5]
    want = a.wanted
    a.wanted = lambda: (setattr(a, "qkv", a.qkv.contiguous()), want(), setattr(a, "qkv", wide[:, 128:-128]))[1]
    a.check()
    assert (big[:, 0] == 7.0).all() and (big[:, 5:] == 7.0).all()


def test_append_captured_and_replayed():
    a = Append(12, 8, 2, 128, [(6, 37), (5, 5), (20, 40)])
    old_pool, old_scales = a.pool.clone(), a.scales.clone()
    a.call()
    torch.cuda.synchronize()
    want = a.pool.clone(), a.scales.clone(), a.q.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        abi.kv_append(a.pool, a.scales, a.layer, a.qkv, a.q, a.d, a.rope, a.qg, a.kg, a.eps, a.err, a.H)
    a.pool.copy_(old_pool), a.scales.copy_(old_scales), a.q.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, (a.pool, a.scales, a.q)))


def test_append_pool_beyond_32_bit_offsets():
    a = Append(13, 8, 4, 128, [(1, 40), (6, 100)], layers=4, layer=3)
    blocks = 70000
    pool = torch.empty(blocks, 4, 2, 4, 16, 128, dtype=torch.uint8, device=dev())
    scales = torch.empty(blocks, 4, 2, 4, dtype=torch.uint8, device=dev())
    pool[blocks - a.blocks:], scales[blocks - a.blocks:] = a.pool, a.scales
    near = a.slots.copy()
    a.slots = near + (blocks - a.blocks) * 16
    q, k, v = a.wanted()
    old_pool, old_scales = a.pool.cpu().clone(), a.scales.cpu().clone()
    small = a.pool, a.scales
    a.pool, a.scales = pool, scales
    a.call()
    torch.cuda.synchronize()
    a.pool, a.scales, a.slots = pool[blocks - a.blocks:], scales[blocks - a.blocks:], near
    a.compare(q, k, v, old_pool, old_scales)
    del small


# ---------------------------------------------------------------------------
# The bf16 kernel for many rows (more than a tile of the other holds, by max_new): everything above again.
# ---------------------------------------------------------------------------
MANY = dict(max_new=1000)


@pytest.mark.parametrize("H,G,dh", [(4, 4, 64), (8, 2, 64), (3, 1, 128), (8, 1, 128), (24, 8, 128), (64, 2, 64)])
def test_many_rows_ragged(H, G, dh):
    Attention(H * 100 + dh, H, G, dh, [(1, 1), (1, 16), (40, 57), (3, 3), (6, 160), (5, 33), (130, 700), (2, 1031)]).check(**MANY)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 16, 37, 100, 5000])
def test_many_rows_window(dh, window):
    Attention(window, 8, 2, dh, [(6, 400), (1, 65), (40, 90), (5, 5), (70, 300)]).check(window=window, **MANY)


@pytest.mark.parametrize("dh", [64, 128])
def test_many_rows_cap_and_scale(dh):
    Attention(5, 8, 4, dh, [(6, 400), (1, 65), (40, 40)], q_std=2.0).check(cap=30.0, scale=0.21, **MANY)
    Attention(6, 8, 4, dh, [(6, 300), (1, 65), (40, 200)], q_std=2.0).check(cap=5.0, window=50, **MANY)


def test_many_rows_padding_empty_and_below_zero():
    Attention(9, 8, 2, 128, [(0, 40), (30, 40), (0, 0), (1, 20), (0, 16)], pad=5).check(**MANY)
    a = Attention(11, 8, 2, 128, [(25, 40), (3, 40)])
    a.ctx[0] = 2  # 25 new tokens, two positions: the first 23 have no key
    a.check(**MANY)
    assert (a.out[:23] == 0).all()


@pytest.mark.parametrize("many", [0, 1])
def test_more_spans_than_a_cta_lists_at_once(many):
    rng = np.random.default_rng(1)
    Attention(12, 8, 8, 64, [(1, int(c)) for c in rng.integers(1, 40, 700)]).check(max_new=1000 if many else 1)


@pytest.mark.parametrize("dh", [64, 128])
def test_many_rows_of_a_long_sequence_among_short_ones(dh):
    """Its spans are cut between CTAs; the parts are joined the same way each time."""
    a = Attention(13, 4, 2, dh, [(40, 9000)] + [(1, 3)] * 100 + [(33, 700)])
    a.check(**MANY)
    first = a.out.clone()
    a.check(**MANY)
    assert torch.equal(first, a.out)


def test_many_rows_scales_far_apart():
    a = Attention(14, 8, 2, 128, [(20, 200), (1, 90)], spread=0.0)
    byte = torch.arange(a.scales.numel()).reshape(a.scales.shape) * 7 % 121 + 67
    a.scales[:, :, 1] = byte.to(torch.uint8).to(dev())[:, :, 1]
    a.check(**MANY)
    a.scales[:, :, 1] = torch.tensor([0, 255], dtype=torch.uint8, device=dev())[torch.arange(2, device=dev())]
    a.check(**MANY)


@pytest.mark.parametrize("dh", [64, 128])
def test_many_rows_nan_in_masked_cells(dh):
    lens = [(6, 101), (1, 33), (20, 40), (17, 200)]
    a = Attention(15, 8, 2, dh, lens)
    want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables, window=30)
    for b, (n, c) in enumerate(lens):
        for j in list(range(c, (c + 15) // 16 * 16)) + list(range(0, max(0, c - n - 30 + 1))):
            a.pool[a.tables[b, j // 16], 1, :, :, j % 16] = 0x7F
    a.call(window=30, **MANY)
    torch.cuda.synchronize()
    a.compare(*want)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
def test_many_rows_nan_cell_reaches_those_who_see_it(dh, which):
    a = Attention(16, 4, 2, dh, [(28, 60), (1, 20), (9, 300)])
    want, weight, spread, floor = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    j = 60 - 3
    a.pool[a.tables[0, j // 16], 1, which, 0, j % 16, 37] = 0xFF
    a.call(**MANY)
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    clean = torch.ones_like(got, dtype=torch.bool)
    if which == 0:
        clean[25:28, :2] = False
    else:
        clean[25:28, :2, 37] = False
    assert torch.isnan(got[~clean]).all()
    bound = ref.attention_bound(want, weight, spread, floor, dh, a.out.dtype)
    assert ((got - want).abs()[clean] <= bound[clean]).all()


def test_many_rows_bad_blocks_contexts_and_starts():
    a = Attention(17, 8, 2, 128, [(1, 64), (30, 70), (1, 30)])
    want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    a.tables[0, 1], a.tables[0, 2], a.ctx[0] = a.blocks, -1, 64 + 1600
    a.call(**MANY)
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    bound = ref.attention_bound(*want, 128, a.out.dtype)
    assert ((got - want[0]).abs()[1:] <= bound[1:]).all()
    assert not torch.isnan(got).any() and int(a.err) == 1
    for starts in ([0, 40, 2, 60], [0, 2, 40, 900], [0, -5, 2, 60], [3, 1, 2, 60]):
        a = Attention(19, 8, 2, 64, [(20, 30), (20, 30), (20, 30)], pad=2)
        a.starts = starts
        a.call(**MANY)
        torch.cuda.synchronize()
        assert int(a.err) == 1


def test_many_rows_large_and_small_scores():
    for std in (200.0, 1e-6):
        Attention(22, 8, 2, 128, [(30, 300), (1, 90)], q_std=std).check(**MANY)
    for mag in (1e30, 1e-30):
        a = Attention(24, 4, 2, 64, [(30, 200)])
        a.q = (a.q.float() * mag).to(torch.bfloat16)
        a.check(scale=float(0.125 / mag) if mag > 1 else 1e30, **MANY)


def test_many_rows_captured_and_replayed_with_other_lengths():
    a = Attention(25, 8, 2, 128, [(36, 500), (2, 90), (1, 333)])
    a.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        abi.attention_e4m3(a.q, a.out, a.pool, a.scales, a.layer, *a.d, a.ws, a.err, max_new=36)
    for ctx in ([500, 90, 333], [100, 64, 3], [36, 2, 1]):
        a.ctx = ctx
        a.d[1].copy_(i32(ctx))
        a.out.fill_(7.0)
        want = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
        g.replay()
        torch.cuda.synchronize()
        a.compare(*want)


@pytest.mark.parametrize("dtype,max_new", [("bf16", 1), ("bf16", 6), ("bf16", 1000), ("f32", 6)])
@pytest.mark.parametrize("times", [1000.0, 1e5])
def test_attention_queries_with_an_element_far_above_the_rest(dtype, max_new, times):
    """One dimension of the queries is `times` the others, and zero in every key: what counts are the small ones.
    They are held to 2^-21 of their row's largest (bf16), which adds 2^-21 * max|q| * sum_d |K_jd| * scale to a score's
    error; two f16 terms (fp32) hold them to 2^-22 of themselves and 2^-38 of the largest."""
    a = Attention(27, 8, 2, 128, [(6, 300), (9, 90), (1, 40)], dtype)
    a.q[:, :, 3] = a.q[:, :, 3].sign() * times
    a.pool[:, :, 0, :, :, 3] = 0
    want, weight, spread, floor = ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables)
    k = ref.decode(a.pool[:, a.layer, 0].cpu(), a.scales[:, a.layer, 0].cpu()).abs().sum(-1).max()
    unit = 2.0 ** -21 if dtype == "bf16" else 2.0 ** -38
    extra = unit * a.q.double().cpu().abs().amax(-1) * k * 128 ** -0.5
    a.call(max_new=max_new)
    torch.cuda.synchronize()
    a.compare(want, weight, spread + extra / ((128 + 8) * 2.0 ** -23), floor)


# ---------------------------------------------------------------------------
# Calls among other work.
# ---------------------------------------------------------------------------
SHAPES = [("bf16", 1), ("bf16", 6), ("bf16", 1000), ("f32", 6)]


@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_attention_keeps_its_place_in_the_stream(dtype, max_new):
    """Launches overlap the end of the kernel before them: inputs written and results read by kernels right before and
    after a call, round after round without waiting, are those of the round."""
    a = Attention(28, 8, 2, 128, [(6, 700), (9, 90), (1, 400)], dtype)
    g = torch.Generator().manual_seed(1)
    qs = torch.randn(24, *a.q.shape, generator=g).to(a.q.dtype).to(dev())
    want = []
    for q in qs:
        a.q.copy_(q)
        a.call(max_new=max_new)
        torch.cuda.synchronize()
        want.append(a.out.clone())
    outs = torch.zeros(24, *a.q.shape, dtype=a.q.dtype, device=dev())
    torch.cuda.synchronize()
    for i in range(24):
        a.q.copy_(qs[i])
        abi.attention_e4m3(a.q, a.out, a.pool, a.scales, a.layer, *a.d, a.ws, a.err, max_new=max_new)
        outs[i].copy_(a.out)
        a.out.zero_()
    torch.cuda.synchronize()
    assert torch.equal(outs, torch.stack(want)) and int(a.err) == 0


@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_attention_twice_at_once(dtype, max_new):
    """Two streams, a workspace each."""
    calls = [Attention(29 + i, 8, 2, 128, [(6, 3000), (9, 90), (1, 400)], dtype) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    for a in calls:
        a.call(max_new=max_new)
    torch.cuda.synchronize()
    want = [a.out.clone() for a in calls]
    outs = [torch.zeros(16, *a.out.shape, dtype=a.out.dtype, device=dev()) for a in calls]
    torch.cuda.synchronize()
    for i in range(16):
        for a, st, out in zip(calls, streams, outs):
            with torch.cuda.stream(st):
                abi.attention_e4m3(a.q, out[i], a.pool, a.scales, a.layer, *a.d, a.ws, a.err, max_new=max_new)
    torch.cuda.synchronize()
    for a, w, out in zip(calls, want, outs):
        assert all(torch.equal(w, o) for o in out) and int(a.err) == 0


@pytest.mark.parametrize("cache", ["e4m3", "bf16"])
def test_append_keeps_its_place_in_the_stream(cache):
    H, G, dh, T, n = 8, 2, 128, 40, 24
    g = torch.Generator().manual_seed(2)
    e4 = cache == "e4m3"
    pool = torch.zeros(8, 1, 2, G, 16, dh, dtype=torch.uint8 if e4 else torch.bfloat16, device=dev())
    scales = torch.full((8, 1, 2, G), 67, dtype=torch.uint8, device=dev()) if e4 else None
    src = torch.randn(n, T, (H + 2 * G) * dh, generator=g).to(torch.bfloat16).to(dev())
    qkv, q = torch.zeros_like(src[0]), torch.zeros(T, H, dh, dtype=torch.bfloat16, device=dev())
    slots = torch.arange(T, dtype=torch.int32, device=dev()) + 5
    err = torch.zeros(1, dtype=torch.int32, device=dev())
    gain = torch.ones(dh, device=dev())

    def rounds(wait):
        got = torch.zeros(n, T, H, dh, dtype=torch.bfloat16, device=dev())
        cells = torch.zeros(n, *pool.shape, dtype=pool.dtype, device=dev())
        pool.zero_()
        if e4:
            scales.fill_(67)
        torch.cuda.synchronize()
        for i in range(n):
            qkv.copy_(src[i])
            abi.kv_append(pool, scales, 0, qkv, q, slots, None, gain, gain, 1e-6, err, H)
            got[i].copy_(q)
            cells[i].copy_(pool)
            qkv.zero_()
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return got, cells

    one, other = rounds(True), rounds(False)
    assert torch.equal(one[0], other[0]) and torch.equal(one[1], other[1]) and int(err) == 0


# ---------------------------------------------------------------------------
# Both, as a decoding step uses them.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_then_attend_over_a_growing_cache(dtype):
    """A prompt, then steps of 1 to 4 tokens, one of them rolled back: every step's attention equals the
    64-bit attention over what the cache then holds."""
    H, G, dh, blocks = 8, 2, 128, 40
    rng = np.random.default_rng(30)
    g = torch.Generator().manual_seed(30)
    pool = torch.zeros(blocks, 2, 2, G, 16, dh, dtype=torch.uint8, device=dev())
    scales = torch.full((blocks, 2, 2, G), 67, dtype=torch.uint8, device=dev())
    tables = rng.permutation(blocks)[:20].reshape(2, 10).astype(np.int32)
    ws = torch.zeros(abi.attention_e4m3_workspace(dh), dtype=torch.uint8, device=dev())
    err = torch.zeros(1, dtype=torch.int32, device=dev())
    gain = (torch.rand(dh, generator=g) + 0.5).to(dev())
    have = [0, 0]
    for new, drop in (((45, 30), 0), ((1, 1), 0), ((4, 4), 3), ((4, 4), 0), ((2, 3), 0), ((20, 1), 0)):
        starts, ctx = [0, new[0], sum(new)], [h + n for h, n in zip(have, new)]
        pos = np.concatenate([np.arange(h, c) for h, c in zip(have, ctx)])
        seq = np.repeat([0, 1], new)
        slots = i32([tables[b, p // 16] * 16 + p % 16 for b, p in zip(seq, pos)])
        qkv = torch.randn(sum(new), (H + 2 * G) * dh, generator=g).to(dev())
        ang = torch.as_tensor(pos)[:, None] * 1e4 ** (-torch.arange(0, dh, 2, dtype=torch.float64) / dh)
        rope = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous().to(dev())
        for layer in (0, 1):
            q = torch.empty(sum(new), H, dh, dtype=DT[dtype], device=dev())
            out = torch.empty_like(q)
            abi.kv_append(pool, scales, layer, qkv, q, slots, rope, gain, gain, 1e-6, err, H)
            abi.attention_e4m3(q, out, pool, scales, layer, i32(starts), i32(ctx), i32(tables), ws, err, max_new=max(new))
            torch.cuda.synchronize()
            want, weight, spread, floor = ref.attention(q, pool, scales, layer, starts, ctx, tables)
            bound = ref.attention_bound(want, weight, spread, floor, dh, q.dtype)
            assert ((out.double().cpu() - want).abs() <= bound).all()
            # and the cache holds what was appended, to half a step of its blocks' largest
            x = ref.rotated(ref.normed(qkv.double().cpu().view(-1, H + 2 * G, dh)[:, H:H + G], gain.cpu(), 1e-6), rope.cpu())
            for t, s in enumerate(slots.tolist()):
                val = ref.decode(pool[s // 16, layer, 0].cpu(), scales[s // 16, layer, 0].cpu())[:, s % 16]
                assert ((val - x[t]).abs() <= x[t].abs() * (2.0 ** -4 + 1e-5) + 448 * 2.0 ** -18 * x.abs().max()).all()
        have = [c - drop for c in ctx]
    assert int(err) == 0
