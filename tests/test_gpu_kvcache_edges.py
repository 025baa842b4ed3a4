"""The operators on an e4m3 paged cache at the ends of their arguments' ranges: cells and queries that are not
finite under a soft cap, positions far below zero, queries, caps and windows as large as their types hold, starts
that fall, steps that are padding for the most part.
The tolerances are kvcache_ref.attention_bound's and Append.compare's throughout."""
import math

import numpy as np
import pytest
import torch

import kvcache_ref as ref
from test_gpu_kvcache import Append, Attention

pytestmark = pytest.mark.gpu

# every kernel: bf16 tiles of 8, of 24 and of 128 rows (32 at head_dim 256), fp32 tiles of 8 and of 32 (16)
SHAPES = [("bf16", 1), ("bf16", 6), ("bf16", 1000), ("f32", 1), ("f32", 6)]


def reference(a, **kw):
    return ref.attention(a.q, a.pool, a.scales, a.layer, a.starts, a.ctx, a.tables, **kw)


def assert_rows(a, want, poisoned):
    """Elements of `poisoned` are NaN, the others right."""
    got = a.out.double().cpu()
    assert torch.isnan(got[poisoned]).all()
    bound = ref.attention_bound(*want, got.shape[-1], a.out.dtype)
    assert ((got - want[0]).abs()[~poisoned] <= bound[~poisoned]).all()
    assert int(a.err) == 0


# ---------------------------------------------------------------------------
# NaN.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("which", [0, 1])
def test_nan_cell_reaches_those_who_see_it(dtype, max_new, dh, cap, which):
    """A NaN in the K or V of a new token's cell: earlier tokens are untouched, later ones NaN, with a soft cap too."""
    a = Attention(16, 4, 2, dh, [(8, 60), (1, 20), (9, 300)], dtype)
    want = reference(a, cap=cap)
    j = 60 - 3  # the sixth new token's cell
    a.pool[a.tables[0, j // 16], 1, which, 0, j % 16, 37] = 0xFF
    a.call(max_new=max_new, cap=cap)
    torch.cuda.synchronize()
    poisoned = torch.zeros(a.out.shape, dtype=torch.bool)
    poisoned[5:8, :2, slice(None) if which == 0 else 37] = True  # heads 0, 1 read KV head 0
    assert_rows(a, want, poisoned)


@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("cap,window", [(0.0, 0), (30.0, 0), (30.0, 40)])
def test_nan_query_reaches_its_row_only(dtype, max_new, dh, cap, window):
    a = Attention(17, 4, 2, dh, [(8, 60), (1, 20), (9, 300)], dtype)
    want = reference(a, cap=cap, window=window)
    poisoned = torch.zeros(a.out.shape, dtype=torch.bool)
    for t, h, d in ((0, 0, 0), (5, 3, 63), (8, 1, 17), (13, 2, 40)):
        a.q[t, h, d] = math.nan
        poisoned[t, h] = True
    a.call(max_new=max_new, cap=cap, window=window)
    torch.cuda.synchronize()
    assert_rows(a, want, poisoned)


# ---------------------------------------------------------------------------
# Positions below zero.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_positions_far_below_zero_give_zeros(dtype, max_new):
    """Whole query tiles without a key, hundreds of positions below zero, after calls that left cells of others in
    shared memory."""
    a = Attention(31, 4, 2, 64, [(40, 3000), (400, 400)], dtype)
    a.check(max_new=max_new)
    a.ctx[1] = 2  # 400 new tokens, two positions
    a.check(max_new=max_new)
    assert (a.out[40:438] == 0).all()


@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_contexts_below_zero_give_zeros(dtype, max_new):
    """Every position of such a sequence is below zero, down to the lowest length there is."""
    a = Attention(34, 4, 2, 64, [(7, 300), (40, 40), (1, 30), (9, 90)], dtype)
    a.check(max_new=max_new)
    for low in (-1, -2 ** 30, -2 ** 31 + 39, -2 ** 31):
        a.ctx[1] = a.ctx[2] = low
        a.check(max_new=max_new)
        assert (a.out[7:48] == 0).all()


# ---------------------------------------------------------------------------
# Queries at the end of their type's range.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("mag", [6e37, 1e36, 1e33, 1e-33, 1e-35])
def test_queries_of_any_magnitude(dtype, max_new, dh, mag):
    a = Attention(24, 4, 2, dh, [(3, 200), (9, 40)], dtype)
    a.q = (a.q.double() * mag).to(a.q.dtype)
    assert torch.isfinite(a.q).all()
    a.check(scale=float(dh ** -0.5 / mag), max_new=max_new)


@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_infinite_query_reaches_its_row_only(dtype, max_new, dh, cap):
    """All its scores are infinite or NaN: so is no softmax of them.  A token without a key still gets zeros."""
    a = Attention(18, 4, 2, dh, [(8, 60), (1, 20), (9, 300), (5, 40)], dtype)
    a.ctx[3] = 2
    want = reference(a, cap=cap)
    poisoned = torch.zeros(a.out.shape, dtype=torch.bool)
    for t, h, d, x in ((0, 0, 0, math.inf), (5, 3, 63, -math.inf), (8, 1, 17, math.inf), (13, 2, 40, -math.inf)):
        a.q[t, h, d] = x
        poisoned[t, h] = True
    a.q[18, 1, 5] = math.inf
    a.call(max_new=max_new, cap=cap)
    torch.cuda.synchronize()
    assert_rows(a, want, poisoned)
    assert (a.out[18:21] == 0).all()


# ---------------------------------------------------------------------------
# Windows and caps at the end of their type's range.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 20, 2 ** 30])
def test_window_as_large_as_it_gets_masks_nothing(dtype, max_new, window):
    """... in a tile that begins below position zero too."""
    a = Attention(32, 8, 2, 128, [(40, 60), (9, 300)], dtype)
    a.ctx[0] = 17
    a.check(max_new=max_new, window=window)


@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("cap", [3.4028234e38, 1e38, 1e36, 1e-36, 1e-39])
def test_caps_of_any_size(dtype, max_new, cap):
    """A huge one changes nothing, a tiny one makes all weights equal."""
    Attention(33, 8, 2, 128, [(6, 300), (9, 40)], dtype).check(max_new=max_new, cap=cap)


# ---------------------------------------------------------------------------
# q_starts that fall.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_sequences_that_overlap_are_not_begun(dtype, max_new):
    """Starts that fall and rise again give 128 sequences the same 8192 rows, more work than 32 bits count (8 heads x
    8192 tokens x 131,072 keys each): nothing is written, the error word says so, and the next call is right."""
    a = Attention(35, 8, 8, 64, [(6, 300), (9, 40)], dtype)
    right = a.q, a.out, a.starts, a.ctx, a.tables
    T, B = 8192, 256
    a.q = torch.zeros(T, 8, 64, dtype=a.q.dtype, device=a.q.device)
    a.out = torch.full_like(a.q, 7.0)
    a.starts, a.ctx = [T * (b % 2) for b in range(B + 1)], [131072] * B
    a.tables = torch.zeros(B, 8192, dtype=torch.int32)
    a.call(max_new=max_new)
    torch.cuda.synchronize()
    assert (a.out == 7.0).all() and int(a.err) == 1
    a.err.zero_()
    a.q, a.out, a.starts, a.ctx, a.tables = right
    a.check(max_new=max_new)


@pytest.mark.parametrize("dtype,max_new", SHAPES)
def test_a_sequence_whose_starts_do_not_fit_leaves_the_others_right(dtype, max_new):
    a = Attention(36, 8, 2, 64, [(2, 30), (3, 40), (4, 50)], dtype)
    want = reference(a)
    a.starts = [0, 2, 5, 900]  # the last one ends past T
    a.call(max_new=max_new)
    torch.cuda.synchronize()
    got = a.out.double().cpu()
    bound = ref.attention_bound(*want, 64, a.out.dtype)
    assert ((got - want[0]).abs()[:5] <= bound[:5]).all()
    assert (got[5:] == 7.0).all() and int(a.err) == 1


# ---------------------------------------------------------------------------
# Append: long runs of padding.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["e4m3", "bf16"])
@pytest.mark.parametrize("gap", [1, 31, 32, 33, 255, 256, 287, 288, 289, 320, 700])
def test_append_rows_far_apart(cache, gap):
    """Padding between the rows of a block, between blocks, before the first row and behind the last one."""
    a = Append(37, 4, 2, 64, [(21, 40), (1, 16), (16, 32), (2, 5)], cache=cache)
    n, lead = len(a.slots), 40
    at = lead + np.arange(n) + gap * ((np.arange(n) + 1) // 2)  # a gap before every other row
    T = int(at[-1]) + 1 + 2 * gap
    at_d = torch.as_tensor(at).to(a.qkv.device)

    def spread(x, fill):
        y = torch.full((T, *x.shape[1:]), fill, dtype=x.dtype, device=x.device)
        y[at_d] = x
        return y

    a.qkv, a.q, a.rope = spread(a.qkv, 3.0), spread(a.q, 7.0), spread(a.rope, 1.0)
    slots = np.full(T, -1, np.int32)
    slots[at] = a.slots
    a.slots = slots
    a.check()


# ---------------------------------------------------------------------------
# Nothing at all.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_batch_without_sequences(dtype):
    a = Attention(38, 4, 2, 64, [(1, 20)], dtype)
    a.q, a.out = a.q[:0], a.out[:0]
    a.starts, a.ctx, a.tables = [0], [], np.zeros((0, 4), np.int32)
    a.call()
    b = Append(39, 4, 2, 64, [(1, 20)])
    pool = b.pool.clone()
    b.call(0, 0)
    torch.cuda.synchronize()
    assert int(a.err) == 0 and int(b.err) == 0 and torch.equal(pool, b.pool)


# ---------------------------------------------------------------------------
# Scores that fp32 holds to whole numbers or worse.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,max_new", SHAPES)
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("q_std,cap", [(1e6, 0.0), (3e7, 0.0), (1e9, 0.0), (1e14, 0.0), (1e14, 1e30), (1e9, 1e9)])
def test_huge_scores_give_means_of_values(dtype, max_new, dh, q_std, cap):
    """A result lies among the values that its query sees; where one score leads by more than the scores' error,
    spread * (dh + 8) * 2^-23 each and with a cap 2^-20 of themselves (its tanh: the series' next term is 2^-21.5 of the
    sum at most, the quotient beyond it 2^-22 where it is a quarter), it is that key's value."""
    lens = [(3, 40), (40, 300), (1, 700)]
    a = Attention(40, 4, 2, dh, lens, dtype, q_std=q_std)
    a.call(max_new=max_new, cap=cap)
    torch.cuda.synchronize()
    got, half, t = a.out.double().cpu(), torch.finfo(a.out.dtype).eps / 2, 0
    assert torch.isfinite(got).all() and int(a.err) == 0
    led = 0
    for b, (n, c) in enumerate(lens):
        ids = [int(i) for i in a.tables[b][:(c + 15) // 16]]
        kv = ref.decode(a.pool[ids, 1].cpu(), a.scales[ids, 1].cpu()).permute(1, 2, 0, 3, 4).reshape(2, 2, -1, dh)
        for i in range(n):
            for h in range(4):
                K, V = kv[0, h // 2, :c - n + i + 1], kv[1, h // 2, :c - n + i + 1]
                q, y = a.q[t, h].double().cpu(), got[t, h]
                slack = V.abs().amax(0) * (half + 2.0 ** -11) + V.abs().max() * 2.0 ** -26
                assert (y >= V.amin(0) - slack).all() and (y <= V.amax(0) + slack).all()
                x, d = K @ q * dh ** -0.5, float((K.abs() @ q.abs()).max()) * dh ** -0.5 * (dh + 8) * 2.0 ** -23
                if cap:
                    x = cap * torch.tanh(x / cap)
                top = x.topk(min(2, len(x)))
                if len(x) == 1 or top.values[0] - top.values[1] > 2 * d + (2 * float(x.abs().max()) * 2.0 ** -20 if cap else 0) + 40:
                    led += 1
                    assert ((y - V[top.indices[0]]).abs() <= slack).all()
            t += 1
    assert led > 0 or cap == 1e9
