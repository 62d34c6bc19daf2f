"""The LM on bounded caches: contexts with attn_window, attn_sinks or kv_track,
and ming_cuda_seq_evict, through the same entry points as ordinary contexts.

The reference here is a Qwen2 in 64-bit numpy that keeps every sequence's keys
(rotated once, at their first position), values and attention totals itself,
masks by window and sinks, and evicts by the rule. The library rounds to bf16
at the reference's points and these tests do not, so outputs are gated on the
noise that this rounding makes: the RMS distance of an ordinary context to the
same 64-bit model with full attention, on the same inputs, is measured beside
every run, and the bounded context has to stay within twice that (and cosine
above 0.999). Which positions stay is checked exactly, by the totals that the
context itself reports.
"""
import numpy as np
import pytest

import ming_b200 as M
import oracle as O
from ming_b200 import synth

from conftest import bf

pytestmark = pytest.mark.gpu

LAYERS, H, HEADS, KVH, HD = 2, 896, 14, 2, 64
QS = (0.002, 0.005)


@pytest.fixture(scope="module")
def weights(cuda_ok):
    return synth.lm_weights(seed=41, bits=4, layers=LAYERS, qscale=QS)


def context(W, **kw):
    base = dict(layers=LAYERS, weight_bits=4, dit_mode=M.DIT_NONE, agg_blocks=0, max_ctx=512, max_pages=256, max_batch=8,
                max_seqs=8, max_prefill=128)
    return M.Context(M.default_cfg(**{**base, **kw}), weights=W)


class Model:
    """Qwen2 in 64 bits with per-(layer, head) caches."""

    def __init__(self, W):
        d = lambda n: O.lin_dequant(W, n).astype(np.float64)  # noqa: E731
        self.layers = []
        for l in range(LAYERS):
            p = f"model.model.layers.{l}"
            self.layers.append({n: d(f"{p}.{n}") for n in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj",
                                                          "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")})
            for n in ("q", "k", "v"):
                self.layers[l][n + "b"] = bf(W[f"{p}.self_attn.{n}_proj.bias"])
        self.freq = 1e6 ** (-np.arange(32) / 32)

    def cache(self, window=0, sinks=0):
        z = lambda *s: np.zeros((LAYERS, KVH, 0) + s)  # noqa: E731
        return dict(k=z(HD), v=z(HD), tot=z(), pos=0, window=window, sinks=sinks)

    def rope(self, x, pos):
        a = pos[:, None, None] * self.freq
        lo, hi = x[..., :32], x[..., 32:]
        return np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)], -1)

    def forward(self, c, x):
        """x [L, hidden] bf16 bits -> post-norm hidden [L, hidden]; appends to the cache."""
        norm = lambda t: t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
        x = bf(x)
        L, n0 = x.shape[0], c["k"].shape[2]
        pos = c["pos"] + np.arange(L)
        slot = n0 + np.arange(L)
        j = np.arange(n0 + L)[None]
        see = j <= slot[:, None]
        if c["window"]:
            see &= (j < c["sinks"]) | (j > slot[:, None] - c["window"])
        K, V, T = [], [], []
        for l, w in enumerate(self.layers):
            y = norm(x)
            q = self.rope((y @ w["self_attn.q_proj"].T + w["qb"]).reshape(L, HEADS, HD), pos)
            k = self.rope((y @ w["self_attn.k_proj"].T + w["kb"]).reshape(L, KVH, HD), pos)
            v = (y @ w["self_attn.v_proj"].T + w["vb"]).reshape(L, KVH, HD)
            ks = np.concatenate([c["k"][l], k.transpose(1, 0, 2)], 1)
            vs = np.concatenate([c["v"][l], v.transpose(1, 0, 2)], 1)
            s = np.einsum("lhgd,hjd->hglj", q.reshape(L, KVH, 7, HD), ks) / 8
            s = np.where(see, s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o = np.einsum("hglj,hjd->lhgd", p, vs).reshape(L, HEADS * HD)
            x = x + o @ w["self_attn.o_proj"].T
            y = norm(x)
            g, u = y @ w["mlp.gate_proj"].T, y @ w["mlp.up_proj"].T
            x = x + (g / (1 + np.exp(-g)) * u) @ w["mlp.down_proj"].T
            K.append(ks), V.append(vs)
            T.append(np.concatenate([c["tot"][l], np.zeros((KVH, L))], 1) + p.sum((1, 2)))
        c["k"], c["v"], c["tot"], c["pos"] = np.stack(K), np.stack(V), np.stack(T), c["pos"] + L
        return norm(x)

    def evict(self, c, stay):
        """stay [layers][kv heads] lists of positions."""
        take = lambda t: np.stack([np.stack([t[l, h][stay[l][h]] for h in range(KVH)]) for l in range(LAYERS)])  # noqa: E731
        c["k"], c["v"], c["tot"] = take(c["k"]), take(c["v"]), take(c["tot"])


def rms(got, ref):
    return np.sqrt(((bf(got) - ref) ** 2).mean())


def gate(got, ref, plain, plain_ref):
    """The bounded context against its reference, no worse than twice an ordinary one against its own."""
    g = bf(got)
    cos = (g * ref).sum(-1) / np.linalg.norm(g, axis=-1) / np.linalg.norm(ref, axis=-1)
    noise = rms(plain, plain_ref)
    assert noise < 0.02, noise  # the gate is worth something
    assert cos.min() > 0.999 and rms(got, ref) <= 2 * noise, (cos.min(), rms(got, ref), noise)


@pytest.fixture(scope="module")
def plain(weights):
    ctx = context(weights)
    yield ctx, Model(weights)
    ctx.close()


@pytest.mark.parametrize("window,sinks,track", [(48, 4, 0), (48, 0, 1), (0, 0, 1), (1, 2, 1), (500, 4, 0)])
@pytest.mark.parametrize("prompt", [1, 61, 200])
def test_prompt_and_tokens(weights, plain, window, sinks, track, prompt):
    """A prompt (one chunk, or two: 200 rows over 128) and tokens of three
    sequences in one batch; totals where they are tracked."""
    pctx, model = plain
    ctx = context(weights, attn_window=window, attn_sinks=sinks, kv_track=track)
    lens = [prompt, max(1, prompt // 2), prompt + 3]
    x = [synth.normal_bf16(5, f"bounded.{prompt}.{i}", (n + 3, H)) for i, n in enumerate(lens)]
    cs, ps = [model.cache(window, sinks) for _ in lens], [model.cache() for _ in lens]
    seqs, pseqs = [], []
    for n, xi, c, p in zip(lens, x, cs, ps):
        seqs.append(ctx.seq_alloc()), pseqs.append(pctx.seq_alloc())
        out, _ = ctx.prefill(seqs[-1], xi[:n])
        po, _ = pctx.prefill(pseqs[-1], xi[:n])
        gate(out, model.forward(c, xi[:n]), po, model.forward(p, xi[:n]))
    for k in range(3):
        rows = np.stack([xi[n + k] for n, xi in zip(lens, x)])
        out, _ = ctx.decode(seqs, rows)
        po, _ = pctx.decode(pseqs, rows)
        ref = np.concatenate([model.forward(c, r[None]) for c, r in zip(cs, rows)])
        pref = np.concatenate([model.forward(p, r[None]) for p, r in zip(ps, rows)])
        gate(out, ref, po, pref)
    if track:
        for s, c in zip(seqs, cs):
            n = ctx.seq_len(s)
            for l in range(LAYERS):
                got = ctx.kv_totals(s, l, 0, n)
                # the totals of a position are sums of weights; bf16 noise in the
                # logits (well under 0.1 here) moves each by its share at most
                assert np.allclose(got, c["tot"][l], rtol=0.1, atol=1e-3)
                # every row's weights of seven heads sum to one
                assert abs(got.sum(-1) / (7 * n) - 1).max() < 1e-4
    for s in pseqs:
        pctx.seq_free(s)
    ctx.close()


def chosen(tot, n, keep, sinks, recent):
    mid = sorted(range(sinks, n - recent), key=lambda j: (-tot[j], j))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))


@pytest.mark.parametrize("window,track,keep,sinks,recent", [(0, 1, 64, 4, 20), (40, 1, 64, 4, 44), (60, 0, 64, 4, 60)])
def test_endless_stream(weights, plain, window, track, keep, sinks, recent):
    """A stream of 400 positions through a cache of 96 (max_ctx 256, a pool of 14
    pages for two sequences): evicted whenever it holds more than 90. Kept keys and
    values are the old ones bit for bit, freed pages are used again, rotations go on."""
    pctx, model = plain
    ctx = context(weights, attn_window=window, attn_sinks=sinks if window else 0, kv_track=track, max_ctx=256, max_pages=14)
    other = ctx.seq_alloc()  # a bystander whose cache no eviction touches
    ctx.prefill(other, synth.normal_bf16(6, "bystander", (20, H)))
    before = [ctx.kv_read(other, l, 0, 20) for l in range(LAYERS)]
    s, ps = ctx.seq_alloc(), pctx.seq_alloc()
    c, p = model.cache(window, sinks if window else 0), model.cache()
    x = synth.normal_bf16(6, f"stream.{track}.{window}", (400, H))
    at, evictions = 0, 0
    while at < 400:
        step = 30 if at < 60 else 1
        rows = x[at:at + step]
        if at < 60:
            out, _ = ctx.prefill(s, rows)
            po, _ = pctx.prefill(ps, rows)
        else:
            out, _ = ctx.decode([s], rows)
            po, _ = pctx.decode([ps], rows)
        ref, pref = model.forward(c, rows), model.forward(p, rows)
        if at % 13 == 0 or at < 100:
            gate(out, ref, po, pref)
        at += step
        n = ctx.seq_len(s)
        if n > 90:
            old = [ctx.kv_read(s, l, 0, n) for l in range(LAYERS)]
            tot = [ctx.kv_totals(s, l, 0, n) if track else np.zeros((KVH, n)) for l in range(LAYERS)]
            stay = [[chosen(tot[l][h], n, keep, sinks, recent) for h in range(KVH)] for l in range(LAYERS)]
            ctx.seq_evict(s, keep, sinks, recent)
            assert ctx.seq_len(s) == keep
            for l in range(LAYERS):
                k, v = ctx.kv_read(s, l, 0, keep)
                for h in range(KVH):
                    assert np.array_equal(k[h], old[l][0][h][stay[l][h]]) and np.array_equal(v[h], old[l][1][h][stay[l][h]])
                if track:
                    assert np.array_equal(ctx.kv_totals(s, l, 0, keep), np.stack([tot[l][h][stay[l][h]] for h in range(KVH)]))
            model.evict(c, stay)
            evictions += 1
            ctx.seq_evict(s, keep, sinks, recent)  # holds no more: nothing happens
            assert ctx.seq_len(s) == keep
    assert evictions >= 12
    for l in range(LAYERS):
        k, v = ctx.kv_read(other, l, 0, 20)
        assert np.array_equal(k, before[l][0]) and np.array_equal(v, before[l][1])
    # a second prompt after an eviction: rows at slots 64.. and positions 400..
    more = synth.normal_bf16(6, "second", (25, H))
    gate(ctx.prefill(s, more)[0], model.forward(c, more), pctx.prefill(ps, more)[0], model.forward(p, more))
    # a sequence that starts over counts from zero
    ctx.seq_truncate(s, 0)
    pctx.seq_truncate(ps, 0)
    c, p = model.cache(window, sinks if window else 0), model.cache()
    gate(ctx.prefill(s, more)[0], model.forward(c, more), pctx.prefill(ps, more)[0], model.forward(p, more))
    pctx.seq_free(ps)
    ctx.close()


def test_generate_and_written_caches(weights, plain):
    """lm_generate on a window equals the same steps one by one; totals of
    positions that kv_write restored start at zero."""
    ctx = context(weights, attn_window=30, attn_sinks=2, kv_track=1)
    a, b = ctx.seq_alloc(), ctx.seq_alloc()
    x = synth.normal_bf16(7, "gen", (50, H))
    ctx.prefill(a, x), ctx.prefill(b, x)
    outs, _ = ctx.generate([a], x[:1], 6)
    row = x[:1]
    for k in range(6):
        row, _ = ctx.decode([b], row)
        assert np.array_equal(outs[k], row)
    assert all(np.array_equal(ctx.kv_totals(a, l, 0, 56), ctx.kv_totals(b, l, 0, 56)) for l in range(LAYERS))
    s = ctx.seq_alloc()
    for l in range(LAYERS):
        k, v = ctx.kv_read(a, l, 0, 40)
        ctx.kv_write(s, l, 0, k, v)
        assert (ctx.kv_totals(s, l, 0, 40) == 0).all()
    ctx.decode([s], x[:1])
    assert abs(ctx.kv_totals(s, 0, 0, 41).sum(-1) / 7 - 1).max() < 1e-5
    ctx.close()


def test_sampling_loop_on_a_window(cuda_ok):
    """The sampling loop runs on a bounded context: a window that hides nothing
    gives the ordinary loop's first step (later ones feed on its rounding), a
    short one runs its budget; two requests share a step."""
    Wl = synth.lm_weights(seed=31, bits=4, layers=2, qscale=QS)
    Wl["stop_head.bias"] = synth.f32_to_bf16(np.array([0.0, -4.0], np.float32))
    Wf = synth.flow_weights(seed=32, blocks=2, hidden=512, ff=1024)
    Wa = synth.agg_weights(seed=33, blocks=2, hidden=512, ff=1024)
    kw = dict(layers=2, weight_bits=4, dit_mode=M.DIT_TOKEN, dit_hidden=512, dit_blocks=2, dit_heads=8, dit_ff=1024, agg_blocks=2,
              dit_max_batch=8, max_ctx=512, max_pages=256, max_batch=8, max_seqs=8)
    embeds = synth.normal_bf16(9, "loop.prompt", (40, H))
    got = {}
    for name, extra in (("plain", {}), ("wide", dict(attn_window=512, kv_track=1)), ("short", dict(attn_window=16, attn_sinks=2))):
        ctx = M.Context(M.default_cfg(**kw, **extra), weights={**Wl, **Wf, **Wa})
        p = M.sample_params(max_steps=8)
        lat, zt, st = ctx.sample_latents(embeds, params=p, seed=3, trace=True)
        assert lat.shape[0] == 8 and np.isfinite(bf(lat)).all()
        got[name] = (bf(lat), bf(zt))
        loop = M.Loop(ctx, 2, p)
        ids = [loop.submit(embeds[:n], seed=3) for n in (40, 25)]
        while loop.step()[0]:
            pass
        res = [loop.result(i) for i in ids]
        assert all(r[0].shape[0] == 8 for r in res)
        loop.close()
        ctx.close()
    cos = lambda a, b: (a * b).sum() / np.linalg.norm(a) / np.linalg.norm(b)  # noqa: E731
    assert cos(got["plain"][1][0], got["wide"][1][0]) > 0.999 and cos(got["plain"][0][0], got["wide"][0][0]) > 0.999


def test_refusals(weights, plain):
    pctx, _ = plain
    ps = pctx.seq_alloc()
    x = synth.normal_bf16(8, "refuse", (20, H))
    pctx.prefill(ps, x)
    with pytest.raises(M.MingError, match="attn_window or kv_track"):
        pctx.seq_evict(ps, 10, 0, 10)
    with pytest.raises(M.MingError, match="kv_track"):
        pctx.kv_totals(ps, 0, 0, 1)
    pctx.seq_free(ps)
    ctx = context(weights, attn_window=8)
    s = ctx.seq_alloc()
    ctx.prefill(s, x)
    with pytest.raises(M.MingError, match="allocation-free"):
        ctx.decode_noalloc([s], x[:1])
    for bad in ((10, 2, 3), (0, 0, 0), (5, 3, 3), (4, -1, 5)):
        with pytest.raises(M.MingError):
            ctx.seq_evict(s, *bad)
    with pytest.raises(M.MingError):
        ctx.seq_evict(5, 10, 0, 10)
    assert ctx.step_kernels(1) > 1
    ctx.close()
