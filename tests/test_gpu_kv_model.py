"""Models whose KV pool has 8-bit cells (yk_kv_pool_create_e4m3) and models with per-head norms of queries
and keys (yk_model_enable_qk_norm): steps against a 64-bit forward of the same weights.

The forward's keys and values are what the pool holds after the step (yk_kv_pool_read_page, both sides
read the same rounded cells); the pool's are compared to the forward's own separately.  Tolerances:
logits as elsewhere for these models, 2e-4 (fp32: order of sums) and 5e-2 (bf16 storage of activations) of the
largest; stored cells of an 8-bit pool: half a step of e4m3, 2^-4 of the value, or of its smallest step
2^-9 * 2^e, once for the value and (a geometric sum) at most as much again for the times its block's exponent grew,
with 2^e <= amax / 224; and the error of the value itself, 4 tol of the page's largest."""
import numpy as np
import pytest

from helpers import TINY, PageTables, gpu_model, step_inputs
from yanaiengine_b200 import abi

pytestmark = pytest.mark.gpu
NB = 32
TOL = {abi.DTYPE_F32: 2e-4, abi.DTYPE_BF16: 5e-2}
WIDE = dict(TINY, head_dim=128, n_heads=6, n_kv_heads=2)
CAPPED = dict(TINY, act=abi.ACT_GELU_TANH, attn_cap=50.0, final_cap=30.0, window=8, window_layer_parity=0,
              head_dim=256, n_heads=2, n_kv_heads=1, rms_eps=1e-6)


class Forward64:
    """Steps of a model in float64; K/V of layer l come from rows(l, kv, sequence)."""

    def __init__(self, model, cfg, qk_norm):
        self.cfg, L = cfg, range(cfg["n_layers"])
        get = lambda t: [model.get(t, l).astype(np.float64) for l in L]  # noqa: E731
        self.top = {t: model.get(t).astype(np.float64) for t in (abi.T_EMBED, abi.T_LM_HEAD, abi.T_FINAL_NORM)}
        ids = [abi.T_WQ, abi.T_WK, abi.T_WV, abi.T_WO, abi.T_WGATE, abi.T_WUP, abi.T_WDOWN, abi.T_NORM1, abi.T_NORM2]
        self.w = {t: get(t) for t in ids + ([abi.T_QNORM, abi.T_KNORM] if qk_norm else [])}
        self.qk_norm = qk_norm

    def rms(self, x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg["rms_eps"]) * g.reshape(-1)

    def rope(self, x, pos):
        dh = x.shape[-1]
        ang = pos[:, None] * self.cfg["rope_theta"] ** (-np.arange(0, dh, 2) / dh)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[..., 0::2], x[..., 1::2]
        return np.stack([a * c - b * s, a * s + b * c], -1).reshape(x.shape)

    def step(self, batch, rows):
        """batch of (sequence, tokens, length before) -> all logits, own K/V per layer [T, G, dh]."""
        cfg, w = self.cfg, self.w
        H, G, dh = cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"]
        pos = np.concatenate([np.arange(n, n + len(t)) for _, t, n in batch])
        h = self.top[abi.T_EMBED][np.concatenate([t for _, t, _ in batch])]
        T, own = len(h), []
        for l in range(cfg["n_layers"]):
            x = self.rms(h, w[abi.T_NORM1][l])
            q, k, v = ((x @ w[t][l].T).reshape(T, -1, dh) for t in (abi.T_WQ, abi.T_WK, abi.T_WV))
            if self.qk_norm:
                q, k = self.rms(q, w[abi.T_QNORM][l]), self.rms(k, w[abi.T_KNORM][l])
            q, k = self.rope(q, pos), self.rope(k, pos)
            own.append((k, v))
            windowed = cfg["window"] > 0 and (cfg["window_layer_parity"] < 0 or l % 2 == cfg["window_layer_parity"])
            att, t = np.empty((T, H, dh)), 0
            for sid, toks, n in batch:
                K, V = rows(l, 0, sid), rows(l, 1, sid)  # [G, positions, dh]
                for p in range(n, n + len(toks)):
                    lo = max(0, p - cfg["window"] + 1) if windowed else 0
                    for hd in range(H):
                        s = K[hd * G // H, lo:p + 1] @ q[t, hd] / np.sqrt(dh)
                        if cfg["attn_cap"] > 0:
                            s = cfg["attn_cap"] * np.tanh(s / cfg["attn_cap"])
                        e = np.exp(s - s.max())
                        att[t, hd] = e @ V[hd * G // H, lo:p + 1] / e.sum()
                    t += 1
            h = h + att.reshape(T, -1) @ w[abi.T_WO][l].T
            x = self.rms(h, w[abi.T_NORM2][l])
            gate, up = x @ w[abi.T_WGATE][l].T, x @ w[abi.T_WUP][l].T
            if cfg["act"] == abi.ACT_GELU_TANH:
                gate = 0.5 * gate * (1 + np.tanh(np.sqrt(2 / np.pi) * (gate + 0.044715 * gate ** 3)))
            else:
                gate = gate / (1 + np.exp(-gate))
            h = h + (gate * up) @ w[abi.T_WDOWN][l].T
        z = self.rms(h, self.top[abi.T_FINAL_NORM]) @ self.top[abi.T_LM_HEAD].T
        return (cfg["final_cap"] * np.tanh(z / cfg["final_cap"]) if cfg["final_cap"] > 0 else z), own


def _drive(engine, cfg, dtype, *, e4m3, qk_norm, split=False, prompt=((0, 17), (1, 40), (2, 5)), max_tokens=256,
           steps=((5, 5, 5), (1, 4, 2), (1, 1, 1)), drop=2, nb=NB):
    c = abi.make_config(**cfg, dtype=dtype, max_tokens=max_tokens, max_seqs=16)
    m = abi.Model(engine, c, seed=3, init_std=0.08 if cfg["attn_cap"] else 0.02)
    pools = [abi.KVPool(engine, c, nb, k, e4m3=e4m3) for k in
             ((abi.POOL_GLOBAL_LAYERS, abi.POOL_WINDOWED_LAYERS) if split else (abi.POOL_ALL_LAYERS,))]
    tol, rng = TOL[dtype], np.random.default_rng(1)
    windowed = lambda l: cfg["window"] > 0 and (cfg["window_layer_parity"] < 0 or l % 2 == cfg["window_layer_parity"])  # noqa: E731
    try:
        if qk_norm:
            m.enable_qk_norm()
            assert all((m.get(t, l) == 1).all() for t in (abi.T_QNORM, abi.T_KNORM) for l in range(cfg["n_layers"]))
            for l in range(cfg["n_layers"]):
                for t in (abi.T_QNORM, abi.T_KNORM):
                    m.set(t, l, rng.uniform(0.5, 2.0, cfg["head_dim"]).astype(np.float32))
            m.enable_qk_norm()  # (keeps them)
        fwd = Forward64(m, cfg, qk_norm)
        pts = [PageTables(nb) for _ in pools]
        pts[-1].free = [int(b) for b in rng.permutation(nb)]
        lens = {sid: 0 for sid, _ in prompt}

        def rows(l, kv, sid):
            i = int(split and windowed(l))
            return np.concatenate([pools[i].read_page(b, l, kv) for b in pts[i].tables[sid]], 1).astype(np.float64)

        for i, news in enumerate([[n for _, n in prompt], *steps]):
            batch = [(sid, rng.integers(0, cfg["vocab_size"], n).tolist(), lens[sid]) for (sid, _), n in zip(prompt, news)]
            toks, qs, ctx, bt = step_inputs(pts[0], batch)
            if split:
                got = m.forward_split(*pools, toks, qs, ctx, bt, step_inputs(pts[1], batch)[3], 0)
            else:
                got = m.forward(pools[0], toks, qs, ctx, bt, 0)
            g = m.logits(0, got)
            assert engine.device_error() == 0
            z, own = fwd.step(batch, rows)
            assert np.abs(g - z).max() <= tol * np.abs(z).max(), f"step {i}: {np.abs(g - z).max() / np.abs(z).max():.3e}"
            for l, kv in ((l, kv) for l in range(cfg["n_layers"]) for kv in (0, 1)):
                t = 0
                for sid, new, n in batch:
                    page = rows(l, kv, sid)[:, n:n + len(new)]
                    x = own[l][kv][t:t + len(new)].transpose(1, 0, 2)
                    t += len(new)
                    amax = max(np.abs(rows(l, kv, sid)).max(), np.abs(x).max())
                    half = 2.0 ** -4 * np.abs(x) * (1 + 2.0 ** -3) + 2.0 ** -9 * 2 * amax / 224 if e4m3 else 0.0
                    assert (np.abs(page - x) <= half + 4 * tol * np.abs(own[l][kv]).max()).all()
            for sid, new, n in batch:  # the last ones were rejected: written over by the next step
                lens[sid] = n + len(new) - (drop if len(new) > drop else 0)
    finally:
        for p in pools:
            p.close()
        m.close()


@pytest.mark.parametrize("dtype", [abi.DTYPE_F32, abi.DTYPE_BF16])
@pytest.mark.parametrize("cfg", [TINY, WIDE, CAPPED], ids=["dh64", "dh128", "dh256_window_cap"])
@pytest.mark.parametrize("e4m3,qk_norm", [(True, False), (True, True), (False, True)],
                         ids=["e4m3", "e4m3_qk_norm", "qk_norm"])
def test_steps_match_64_bit_forward(engine, dtype, cfg, e4m3, qk_norm):
    _drive(engine, cfg, dtype, e4m3=e4m3, qk_norm=qk_norm)


@pytest.mark.parametrize("dtype", [abi.DTYPE_F32, abi.DTYPE_BF16])
@pytest.mark.parametrize("e4m3", [True, False], ids=["e4m3", "qk_norm"])
def test_split_pools(engine, dtype, e4m3):
    _drive(engine, CAPPED, dtype, e4m3=e4m3, qk_norm=True, split=True)


@pytest.mark.parametrize("qk_norm", [True, False])
def test_long_prompt_without_the_folded_norm(engine, qk_norm):
    """More than 256 tokens in a step: the RMS norm is a kernel of its own."""
    _drive(engine, TINY, abi.DTYPE_BF16, e4m3=True, qk_norm=qk_norm, prompt=((0, 261), (1, 40), (2, 5)), max_tokens=320,
           steps=((1, 1, 1),))


def test_pool_memory_fill_and_refusals(engine):
    c = abi.make_config(**TINY, dtype=abi.DTYPE_BF16, max_tokens=64, max_seqs=4)
    G, dh, L = TINY["n_kv_heads"], TINY["head_dim"], TINY["n_layers"]
    pool, plain = abi.KVPool(engine, c, 5, e4m3=True), abi.KVPool(engine, c, 5)
    m = abi.Model(engine, c, seed=1)
    try:
        p = pool.pages()
        assert (p.kind, p.num_blocks, p.n_layers, p.n_kv_heads, p.head_dim) == (abi.KV_E4M3, 5, L, G, dh)
        assert p.data and p.scales
        q = plain.pages()
        assert q.kind == abi.KV_BF16 and q.data and not q.scales
        assert all((pool.read_page(b, l, kv) == 0).all() for b in range(5) for l in range(L) for kv in (0, 1))
        pool.fill_random(9, 0.5)
        a = np.stack([pool.read_page(b, l, kv) for b in range(5) for l in range(L) for kv in (0, 1)])
        # 20480 values of N(0, 0.5): the mean within 6 sigma, the deviation within 4% (sigma 0.5%, and rounding
        # by half a step adds at most 2^-8 / 3 to the variance), no two pages alike
        assert a.size == 5 * L * 2 * G * 16 * dh
        assert abs(a.mean()) < 6 * 0.5 / a.size ** 0.5 and abs(a.std() / 0.5 - 1) < 0.04
        assert len(np.unique(a.reshape(-1, 16 * dh), axis=0)) == 5 * L * 2 * G
        pool.fill_random(9, 0.5)
        assert (a[3] == pool.read_page(0, 1, 1)).all()  # the seed's values
        pool.fill_random(10, 0.5)
        assert (a[3] != pool.read_page(0, 1, 1)).any()
        for f in (lambda: m.get(abi.T_QNORM, 0), lambda: m.set(abi.T_KNORM, 0, np.ones(dh, np.float32))):
            with pytest.raises(abi.YKError, match="per-head norms"):
                f()
        m.enable_qk_norm()
        assert (m.get(abi.T_QNORM, 1) == 1).all()
        with pytest.raises(abi.YKError):
            m.get(abi.T_QNORM, L)
        compat = abi.make_config(**dict(TINY, ref_compat=1), dtype=abi.DTYPE_F32, max_tokens=64, max_seqs=4)
        with pytest.raises(abi.YKError) as ei:
            abi.KVPool(engine, compat, 4, e4m3=True)
        assert ei.value.status == 7
        old = abi.Model(engine, compat, seed=1)
        try:
            with pytest.raises(abi.YKError) as ei:
                old.enable_qk_norm()
            assert ei.value.status == 7
        finally:
            old.close()
        w = abi.make_config(**CAPPED, dtype=abi.DTYPE_BF16, max_tokens=64, max_seqs=4)
        wm = abi.Model(engine, w, seed=1)
        a, b = abi.KVPool(engine, w, 4, abi.POOL_GLOBAL_LAYERS, e4m3=True), abi.KVPool(engine, w, 4, abi.POOL_WINDOWED_LAYERS)
        try:
            one = np.zeros((1, 1), np.int32)
            with pytest.raises(abi.YKError, match="both with 8-bit cells"):
                wm.forward_split(a, b, [1], [0, 1], [1], one, one)
        finally:
            for x in (a, b, wm):
                x.close()
    finally:
        for x in (pool, plain, m):
            x.close()


def _scheduled(engine, t, tpool, d, dpool, prompts, temperature, n=24, k=4):
    s = abi.Sampler(engine, 8, k, TINY["vocab_size"])
    sch = abi.Scheduler(t, tpool, d, dpool, s, k, temperature, 3)
    try:
        for i, p in enumerate(prompts):
            sch.submit(p, max_tokens=n, stop_token=-1, seq_id=i)
        for _ in range(40 * len(prompts)):
            if sch.running() == 0 and sch.waiting() == 0:
                break
            sch.step()
        assert sch.running() == 0 and sch.waiting() == 0
        assert sch.usage() == 0.0 and sch.usage(draft=True) == 0.0
        return [sch.generated(i) for i in range(len(prompts))]
    finally:
        sch.close()
        s.close()


@pytest.mark.parametrize("dtype", [abi.DTYPE_F32, abi.DTYPE_BF16])
def test_scheduler_over_8_bit_pools(engine, dtype):
    """Speculative decoding with target, draft and prompts over 8-bit pools, per-head norms in the target: every
    emitted token of the greedy run is the model's own choice, or within the bound of it, when the run's tokens go
    through the 64-bit forward with the cells that a single prompt step stores."""
    t, _tp = gpu_model(engine, TINY, dtype, seed=1, num_blocks=1, max_tokens=256, max_seqs=8)
    d, _dp = gpu_model(engine, dict(TINY, n_layers=1), dtype, seed=2, num_blocks=1, max_tokens=256, max_seqs=8)
    tp, dp = abi.KVPool(engine, t.cfg, 64, e4m3=True), abi.KVPool(engine, d.cfg, 64, e4m3=True)
    try:
        t.enable_qk_norm()
        rng = np.random.default_rng(5)
        prompts = [rng.integers(0, 512, n).tolist() for n in (9, 31, 16)]
        sampled = _scheduled(engine, t, tp, d, dp, prompts, 0.8)
        assert all(24 <= len(g) <= 29 and all(0 <= x < 512 for x in g) for g in sampled)
        got = _scheduled(engine, t, tp, d, dp, prompts, 0.0)
        assert all(len(g) >= 24 for g in got)
        assert engine.device_error() == 0
        # a single step over everything stores each block with the exponent of its final amax, while the run's may
        # have grown under drafts that were dropped: cells differ by a step of e4m3 (2^-3) at most, an error of
        # the activations that moves the logits by far less than their own size; 0.1 of the largest is allowed
        for prompt, g in zip(prompts, got):
            toks = prompt + g[:-1]
            pages = (len(toks) + 15) // 16
            bt = np.arange(pages, dtype=np.int32)[None]
            rows = t.forward(tp, toks, [0, len(toks)], [len(toks)], bt, 0)
            z = t.logits(0, rows)[len(prompt) - 1:]
            chosen = z[np.arange(len(g)), g]
            assert (z.max(1) - chosen <= 0.1 * np.abs(z).max(1)).all()
    finally:
        for x in (tp, dp, _tp, _dp, t, d):
            x.close()
