"""Attention over caller-owned paged caches (window, sinks, a prompt's rows or
one new token), the weights it gives, and eviction by them, against the
definition in 64 bits.

Tolerances, fixed before the first run. Products of bf16 values are exact in
f32; a logit is a sum of 64 of them, off by at most 64 half steps of f32 of
the sum of magnitudes: eps_s = 2^-18 scale sum |q_d k_d| (2^-18 = 64 x 2^-24).
A weight exp(s - lse) is then off by at most a factor 1 + eps_w,
eps_w = 2 eps_s + 2^-20 (1 + |s - m|) (the exponent's own rounding, at most
2^-24 of it per step, the exponential 2^-22, the sum of weights 2^-24 per
term; a handful of steps each). An output is a weighted sum of values: its f32
part is off by (eps_w + n 2^-24) sum w |v| and its rounding by half a bf16
step, 2^-8 of its value. A prompt's weights enter the matrix product as bf16,
half a step, 2^-8, of each: 2^-8 sum w |v| more. A single token's enter as two
bf16 parts: 2^-16 of each. A weight below 2^-126, the smallest normal f32, may be
flushed to zero: an absolute error of at most 2^-126 each, which is all that is
left where a position's weights are that small.

Every position that no row may see (behind a sequence's length, in unused
pages, between sinks and window) holds NaN or infinities in K and V.
"""
import math

import pytest
import torch

import ming_b200 as M

pytestmark = pytest.mark.gpu

H16, PAGE, HD, TINY = 2.0 ** -8, 16, 64, 2.0 ** -126


@pytest.fixture(scope="module")
def ctx(cuda_ok):
    c = M.Context(M.default_cfg(layers=0, dit_mode=M.DIT_NONE, agg_blocks=0))
    yield c
    c.close()


def sees(n, r, window, sinks, device="cuda"):
    """[r, n] what the last r positions of n see."""
    p = torch.arange(n - r, n, device=device)[:, None]
    j = torch.arange(n, device=device)[None]
    s = j <= p
    return s & ((j < sinks) | (j > p - window)) if window else s


class Case:
    """A batch of sequences in a pool whose pages are dealt out in random order;
    `layout` orders the pool's dimensions; what nobody sees is poisoned."""

    def __init__(self, lens, rows, heads, kvh, window=0, sinks=0, layers=1, layer=0, layout="page", seed=0, spare=2,
                 poison=True, qpad=0, sharp=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.rows, self.heads, self.kvh, self.window, self.sinks = lens, rows, heads, kvh, window, sinks
        self.layers, self.layer, self.group = layers, layer, heads // kvh
        B, ld = len(lens), max(1, (max(lens) + PAGE - 1) // PAGE + 1)
        held = [(n + PAGE - 1) // PAGE for n in lens]
        pages = sum(held) + spare
        shape = dict(page=(pages, layers, 2, kvh, PAGE, HD), slot=(pages, layers, PAGE, 2, kvh, HD),
                     head=(kvh, layers, 2, pages, PAGE, HD))[layout]
        pool = torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)
        k, v = {"page": lambda p: (p[:, :, 0], p[:, :, 1]),
                "slot": lambda p: (p[:, :, :, 0].transpose(2, 3), p[:, :, :, 1].transpose(2, 3)),
                "head": lambda p: (p[:, :, 0].permute(2, 1, 0, 3, 4), p[:, :, 1].permute(2, 1, 0, 3, 4))}[layout](pool)
        bt = torch.full((B, ld), -7, dtype=torch.int32)  # entries past a sequence's pages are never read
        order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int(), 0
        for b, h in enumerate(held):
            bt[b, :h] = order[at:at + h]
            at += h
        if poison:
            used = torch.zeros(pages, PAGE, dtype=torch.bool, device="cuda")
            for b, n in enumerate(lens):
                if n == 0:
                    continue
                any_row = sees(n, min(n, max(1, rows[b])), window, sinks).any(0)
                j = any_row.nonzero()[:, 0].cpu()
                used[bt[b, j // PAGE].long().cuda(), (j % PAGE).cuda()] = True
            bad = (~used)[:, None, None, :, None]
            self.used = used
            k.masked_fill_(bad, math.nan)
            v.masked_fill_(bad, math.inf)
        self.k, self.v, self.bt = k, v, bt.cuda()
        self.lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        n = sum(rows)
        full = torch.randn(n + 2, heads + qpad, HD, generator=g, device="cuda").mul_(sharp).to(torch.bfloat16)
        self.q = full[:n, :heads]
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        self.start = start
        self.q_start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.cache = M.KvCache(k, v, self.bt, self.lens_t, max(lens))
        self.acc0 = torch.rand(B, layers, kvh, max(max(lens), 1) + 3, generator=g, device="cuda")

    def rows_of(self, t, b, h):
        n = self.lens[b]
        pages = self.bt[b, :(n + PAGE - 1) // PAGE].long()
        return t[pages, self.layer, h].reshape(-1, HD)[:n].double()

    def reference(self, rows=None):
        """out, its f32-part tolerance (per unit weights), lse, acc and theirs, in 64 bits."""
        rows = rows or self.rows
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)       # f32 part and the bf16 parts' magnitude apart
        mag = torch.zeros_like(out)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        lse_tol = torch.zeros_like(lse)
        acc = self.acc0.double()
        acc_tol = torch.zeros_like(acc)
        for b, n in enumerate(self.lens):
            r, at = rows[b], self.start[b]
            if n == 0 or r == 0:
                continue
            live = sees(n, r, self.window, self.sinks)
            own_from = max(0, n - r)
            for h in range(self.kvh):
                k, v = self.rows_of(self.k, b, h), self.rows_of(self.v, b, h)
                any_row = live.any(0)
                k = torch.where(any_row[:, None], k, 0)
                v = torch.where(any_row[:, None], v, 0)
                add, add_tol = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
                for i in range(h * self.group, (h + 1) * self.group):
                    q = self.q[at:at + r, i].double()
                    s = (q @ k.T / 8).masked_fill(~live, -math.inf)
                    eps_s = (2.0 ** -18 * (q.abs() @ k.abs().T) / 8).masked_fill(~live, 0)
                    z = torch.logsumexp(s, -1)
                    m = s.amax(-1, keepdim=True)
                    w = torch.exp(s - z[:, None]).nan_to_num(0.0)
                    eps_w = torch.where(live, 2 * eps_s + 2.0 ** -20 * (1 + (s - m).abs()), 0).nan_to_num(0.0)
                    vis = live.any(-1)
                    out[at:at + r, i] = w @ v
                    mag[at:at + r, i] = w @ v.abs()
                    tol[at:at + r, i] = (w * eps_w) @ v.abs() + n * 2.0 ** -24 * (w @ v.abs())
                    lse[at:at + r, i] = torch.where(vis, z, -math.inf)
                    lse_tol[at:at + r, i] = eps_s.amax(-1) + 2.0 ** -20 * (1 + z.abs().nan_to_num(0.0, posinf=0.0))
                    add += w.sum(0)
                    add_tol += (w * (eps_w + eps_s.amax(-1, keepdim=True) + 2.0 ** -20)).sum(0)
                a = acc[b, self.layer, h]
                a[own_from:n] = 0
                a[:n] += add
                acc_tol[b, self.layer, h, :n] = add_tol + (r * self.group + 1) * 2.0 ** -24 * a[:n] + r * self.group * TINY
        return out, tol, mag, lse, lse_tol, acc, acc_tol


def check(got, ref, tol, what):
    got = got.double()
    assert torch.equal(got.isfinite(), ref.isfinite()), f"{what}: finite where the definition is not, or the other way"
    d = torch.where(ref.isfinite(), (got - ref).abs(), 0)
    over = d - tol
    assert (over <= 0).all(), f"{what}: off by {d.max().item():.3g}, {over.max().item():.3g} over the bound"


def run_prefill(ctx, c, lse=True):
    out = torch.full((c.q.shape[0] + 1, c.heads, HD), 7.0, dtype=torch.bfloat16, device="cuda")
    z = torch.full((c.q.shape[0], c.heads), 5.0, device="cuda") if lse else None
    ctx.attn_prefill(c.q, c.q_start, c.cache, out[:-1], lse=z, max_rows=max(c.rows), layer=c.layer, window=c.window,
                     sinks=c.sinks, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    assert (out[-1] == 7).all()  # rows behind the last sequence
    return out[:-1], z


def check_prefill(ctx, c):
    out, lse = run_prefill(ctx, c)
    ro, tol, mag, rl, ltol, racc, atol = c.reference()
    check(out, ro, tol + 2 * H16 * mag * (1 + H16), "out")
    check(lse, rl, ltol, "lse")
    again, _ = run_prefill(ctx, c, lse=False)
    assert torch.equal(out, again)
    acc = c.acc0.clone()
    ctx.attn_weights(c.q, c.q_start, c.cache, lse, acc, max_rows=max(c.rows), layer=c.layer, window=c.window, sinks=c.sinks,
                     stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    # lse's own tolerance is part of a weight's (eps_s + 2^-20 above)
    check(acc, racc, atol, "acc")
    other = torch.ones_like(acc, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        other[b, c.layer, :, :n] = False
    assert torch.equal(acc[other], c.acc0[other])  # other layers, and entries past the lengths


def check_decode(ctx, c):
    ref = c.reference()
    for track in (False, True):
        out = torch.full_like(c.q.contiguous(), 3.0)
        acc = c.acc0.clone() if track else None
        ctx.attn_decode(c.q, c.cache, out, acc=acc, layer=c.layer, window=c.window, sinks=c.sinks,
                        stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        ctx.sync()
        ro, tol, mag, _, _, racc, atol = ref
        check(out, ro, tol + (2.0 ** -16 + 2.0 ** -20) * mag + H16 * ro.abs(), "out")
        if track:
            check(acc, racc, atol, "acc")
            other = torch.ones_like(acc, dtype=torch.bool)
            for b, n in enumerate(c.lens):
                other[b, c.layer, :, :n] = False
            assert torch.equal(acc[other], c.acc0[other])


HEADS = [(14, 2), (16, 2), (8, 8), (4, 2), (5, 1), (3, 1), (4, 1), (12, 2)]

PREFILL = [
    # lens, rows
    ([1], [1]), ([2], [1]), ([17], [17]), ([128], [128]), ([129], [129]), ([300], [7]), ([515], [130]),
    ([5, 0, 64, 33], [5, 0, 64, 1]), ([200, 77, 16], [0, 77, 16]), ([700, 31], [333, 31]),
]


@pytest.mark.parametrize("lens,rows", PREFILL)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 1), (40, 4), (100, 20), (1000, 4), (33, 200)])
def test_prefill(ctx, lens, rows, window, sinks):
    check_prefill(ctx, Case(lens, rows, 14, 2, window, sinks, seed=len(lens) + window))


@pytest.mark.parametrize("heads,kvh", HEADS)
@pytest.mark.parametrize("layout", ["page", "slot", "head"])
def test_prefill_heads_and_layouts(ctx, heads, kvh, layout):
    check_prefill(ctx, Case([170, 45], [170, 20], heads, kvh, 60, 3, layers=3, layer=2, layout=layout, qpad=2, seed=heads))


def test_prefill_long(ctx):
    check_prefill(ctx, Case([2600, 1201], [1100, 1201], 14, 2, 700, 5, seed=9))
    check_prefill(ctx, Case([2333], [2333], 14, 2, 0, 0, seed=10))
    check_prefill(ctx, Case([9000], [3], 14, 2, 0, 0, seed=11))
    check_prefill(ctx, Case([9000, 4100], [40, 18], 14, 2, 5000, 4, seed=12))


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 4)])
@pytest.mark.parametrize("lens", [[509, 287, 497, 507, 477, 233, 3, 358, 1], [130] * 40, [5] * 200, [700] * 7 + [19] * 30])
def test_prefill_many_sequences(ctx, lens, window, sinks):
    """More work than SMs: a CTA takes several items, of both full and odd tiles."""
    check_prefill(ctx, Case(lens, lens, 14, 2, window, sinks, seed=len(lens)))
    check_prefill(ctx, Case(lens, [(n + 1) // 2 for n in lens], 16, 2, window, sinks, seed=len(lens)))


@pytest.mark.parametrize("lens,rows,window,sinks", [
    ([18] * 37, [18] * 37, 0, 0), ([128] * 37, [100] * 37, 0, 0), ([256] * 8, [256] * 8, 0, 0), ([1024] * 2, [1024, 40], 0, 0),
    ([333], [333], 0, 0), ([1100], [256], 0, 0), ([509, 130, 1, 400], [509, 130, 1, 400], 128, 0), ([700, 20] * 4, [700, 20] * 4, 300, 5),
    ([2048], [1900], 0, 0),
], ids=lambda x: f"{len(x)}x{max(x)}" if isinstance(x, list) else str(x))
def test_weights_divisions(ctx, lens, rows, window, sinks):
    """Tiles of q divided over clusters of every size."""
    check_prefill(ctx, Case(lens, rows, 14, 2, window, sinks, seed=2))


def test_prefill_sharp(ctx):
    """Logits of hundreds: a row's weight sits on one or two positions and its maximum keeps rising."""
    check_prefill(ctx, Case([600], [600], 14, 2, 0, 0, sharp=60.0, seed=13))
    check_prefill(ctx, Case([600], [600], 14, 2, 90, 4, sharp=60.0, seed=14))


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (5, 2 ** 31 - 1), (700, 699), (699, 1)])
def test_windows_and_sinks_of_any_size(ctx, window, sinks):
    check_prefill(ctx, Case([700], [650], 14, 2, window, sinks, poison=False, seed=3))
    check_decode(ctx, Case([700], [1], 14, 2, window, sinks, poison=False, seed=3))


def test_keys_that_some_rows_do_not_see(ctx):
    """A NaN key reaches the rows that see it and no others; the same with an infinite one."""
    for bad in (math.nan, math.inf, -math.inf):
        c = Case([300], [300], 14, 2, 100, 4, poison=False, seed=5)
        clean, _ = run_prefill(ctx, c)
        c.k[c.bt[0, 9].long(), 0, 1, 3] = bad  # position 147, kv head 1
        out, lse = run_prefill(ctx, c)
        hit = torch.zeros(300, 14, dtype=torch.bool, device="cuda")
        hit[147:247, 7:] = True
        assert torch.equal(out[~hit], clean[~hit])
        assert out[hit].isnan().any(-1).all() if math.isnan(bad) else True
        d = Case([300], [1], 14, 2, 100, 4, poison=False, seed=5)
        want, got = torch.empty_like(d.q), torch.empty_like(d.q)
        s = torch.cuda.current_stream().cuda_stream
        ctx.attn_decode(d.q, d.cache, want, window=100, sinks=4, stream=s)
        d.k[d.bt[0, 9].long(), 0, 1, 3] = bad
        d.v[d.bt[0, 9].long(), 0, 1, 3] = bad
        ctx.attn_decode(d.q, d.cache, got, window=100, sinks=4, stream=s)
        assert torch.equal(want, got)


def test_strided_totals(ctx):
    """Totals in any strides: every second sequence of a larger buffer, heads outermost."""
    c = Case([200, 333], [200, 40], 14, 2, 50, 3, layers=2, layer=1, seed=6)
    base = torch.rand(2, 2, 5, 400, device="cuda")  # [kv head, layer, sequence, position]
    view = base.permute(2, 1, 0, 3)[1:5:2]
    view[..., :c.acc0.shape[-1]].copy_(c.acc0)
    before = base.clone()
    out, lse = run_prefill(ctx, c)
    s = torch.cuda.current_stream().cuda_stream
    ctx.attn_weights(c.q, c.q_start, c.cache, lse, view, max_rows=200, layer=1, window=50, sinks=3, stream=s)
    acc = c.acc0.clone()
    ctx.attn_weights(c.q, c.q_start, c.cache, lse, acc, max_rows=200, layer=1, window=50, sinks=3, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(view[..., :acc.shape[-1]], acc)
    changed = base != before
    assert not changed[:, 0].any() and not changed[:, :, ::2].any() and not changed[..., acc.shape[-1]:].any()


def test_prefill_more_rows_than_positions(ctx):
    """Rows at negative positions see nothing."""
    c = Case([5], [9], 14, 2)
    out, lse = run_prefill(ctx, c)
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all()
    assert out[4:].isfinite().all() and lse[4:].isfinite().all()


DECODE = [[1], [16], [17], [500], [1300], [4099], [0, 1, 5], [33, 0, 800, 129], [2053] * 9, list(range(1, 70, 3))]


@pytest.mark.parametrize("lens", DECODE, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 2), (16, 1), (100, 20), (512, 4), (5000, 4)])
def test_decode(ctx, lens, window, sinks):
    check_decode(ctx, Case(lens, [1] * len(lens), 14, 2, window, sinks, seed=len(lens)))


@pytest.mark.parametrize("heads,kvh", HEADS)
@pytest.mark.parametrize("layout", ["page", "slot", "head"])
def test_decode_heads_and_layouts(ctx, heads, kvh, layout):
    check_decode(ctx, Case([170, 45, 600], [1] * 3, heads, kvh, 90, 3, layers=3, layer=1, layout=layout, qpad=1, seed=heads))


def test_decode_long_and_sharp(ctx):
    check_decode(ctx, Case([70001], [1], 14, 2, 0, 0, seed=3))
    check_decode(ctx, Case([20000, 11], [1, 1], 14, 2, 9000, 16, seed=4))
    check_decode(ctx, Case([1000] * 3, [1] * 3, 14, 2, 0, 0, sharp=60.0, seed=5))


@pytest.mark.parametrize("lens", [[131001], [60001] * 5, [20, 60001, 0, 33, 59990]])
def test_decode_totals_of_caches_past_shared_memory(ctx, lens):
    """Logits that no CTA's shared memory holds: the keys are read a second time."""
    c = Case(lens, [1] * len(lens), 14, 2, 0, 0, seed=8, poison=False)
    check_decode(ctx, c)


@pytest.mark.parametrize("lens,kvh", [
    ([509], 2), ([130] * 3, 2), ([1000], 2), ([3000], 1), ([5000], 2), ([400, 0, 1, 399, 17, 33, 16, 250], 2), ([8200] * 2, 2),
    (list(range(150, 509, 15)), 2), ([500] + [60] * 11, 2), ([3001, 0, 17, 2500], 2), ([2000] + [31] * 11, 2), ([700] * 3, 8),
    ([120001], 1), ([120001], 2), ([50001] + list(range(9)), 2),
], ids=lambda x: f"{len(x)}x{max(x)}" if isinstance(x, list) else str(x))
def test_decode_divisions(ctx, lens, kvh):
    """Few heads and many, short caches and long: pages and dims divided over
    clusters of every size, with and without totals; groups of seven and one."""
    check_decode(ctx, Case(lens, [1] * len(lens), 7 * kvh, kvh, 0, 0, seed=len(lens), poison=max(lens) < 10000))
    if max(lens) < 10000:
        check_decode(ctx, Case(lens, [1] * len(lens), kvh, kvh, 300, 5, layout="slot", seed=1))


def test_one_row_of_a_prompt_is_a_token(ctx):
    """The two attention operators agree where they are the same thing."""
    c = Case([333, 40, 1], [1] * 3, 14, 2, 50, 4)
    a, _ = run_prefill(ctx, c)
    b = torch.empty_like(a)
    ctx.attn_decode(c.q, c.cache, b, window=50, sinks=4, stream=torch.cuda.current_stream().cuda_stream)
    _, tol, mag, *_ = c.reference()
    check(a, b.double(), 2 * tol + 4 * H16 * mag, "prefill against decode")


def test_offsets_past_32_bits(ctx):
    """Pages behind element 2^31 of the pool."""
    layers, kvh = 24, 2
    per = layers * 2 * kvh * PAGE * HD
    pages = 2 ** 31 // per + 40
    pool = torch.empty(pages, layers, 2, kvh, PAGE, HD, dtype=torch.bfloat16, device="cuda")
    c = Case([300], [40], 14, 2, 100, 4)
    bt = torch.arange(pages - 30, pages, dtype=torch.int32, device="cuda")[None]
    held = c.bt[0, :19].long()
    pool[pages - 30:pages - 11, 23, 0] = c.k[held, 0]
    pool[pages - 30:pages - 11, 23, 1] = c.v[held, 0]
    far = M.KvCache(pool[:, :, 0], pool[:, :, 1], bt, c.lens_t, 300)
    s = torch.cuda.current_stream().cuda_stream
    a, z = run_prefill(ctx, c)
    b, zb = torch.empty_like(a), torch.empty_like(z)
    ctx.attn_prefill(c.q, c.q_start, far, b, lse=zb, max_rows=40, layer=23, window=100, sinks=4, stream=s)
    assert torch.equal(a, b) and torch.equal(z, zb)
    q = c.q[-1:].contiguous()
    a, b = torch.empty_like(q), torch.empty_like(q)
    ctx.attn_decode(q, c.cache, a, window=100, sinks=4, stream=s)
    ctx.attn_decode(q, far, b, layer=23, window=100, sinks=4, stream=s)
    assert torch.equal(a, b)
    # moved within the far pages
    to = M.KvCache(pool[:, :, 0], pool[:, :, 1], bt[:, 20:], c.lens_t, 64)
    ctx.kv_evict(far, to, keep=64, sinks=4, recent=60, stream=s)
    stay = list(range(4)) + list(range(240, 300))
    k = c.k[held, 0].transpose(0, 1).reshape(kvh, -1, HD)[:, stay]
    got = pool[pages - 10:pages - 6, 23, 0].transpose(0, 1).reshape(kvh, -1, HD)
    assert torch.equal(got.view(torch.int16), k.view(torch.int16))


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def kept(acc, n, keep, sinks, recent):
    """The positions that stay, by sorting in 64 bits."""
    if n <= keep:
        return list(range(n))
    a = [-math.inf if math.isnan(x) else x + 0.0 for x in acc[:n]]
    mid = sorted(range(sinks, n - recent), key=lambda j: (-a[j], j))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + mid + list(range(n - recent, n)))


def totals(shape, kind, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn(shape, generator=g, device="cuda").mul(3).exp()
    if kind == "ties":
        a = torch.randint(0, 3, shape, generator=g, device="cuda").float()
    if kind == "same":
        a = torch.full(shape, 0.25, device="cuda")
    if kind == "odd":  # signs, zeros of both signs, infinities, NaN, subnormals
        v = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42, 3e38], device="cuda")
        a = v[torch.randint(0, 10, shape, generator=g, device="cuda")]
    return a


@pytest.mark.parametrize("lens,keep,sinks,recent", [
    ([40], 20, 4, 8), ([17], 16, 0, 0), ([777], 512, 4, 128), ([300, 0, 5, 64, 200], 64, 1, 16), ([1000], 1, 0, 0),
    ([1000], 1, 1, 0), ([1000], 1, 0, 1), ([2048, 1500], 1024, 4, 1020), ([513], 512, 256, 256), ([4100], 999, 0, 333),
    ([30], 100, 4, 50), ([9000], 8000, 16, 100),
])
@pytest.mark.parametrize("kind", ["spread", "ties", "same", "odd"])
@pytest.mark.parametrize("place", ["apart", "same"])
def test_evict(ctx, lens, keep, sinks, recent, kind, place):
    layers, kvh, B = 3, 2, len(lens)
    c = Case(lens, [1] * B, 14, kvh, layers=layers, poison=False, layout="slot" if place == "apart" else "page", seed=keep)
    acc = totals((B, layers, kvh, max(lens) + 5), kind, keep)
    k0, v0, a0 = c.k.clone(), c.v.clone(), acc.clone()
    index = torch.full((B, layers, kvh, keep), -5, dtype=torch.int32, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    if place == "apart":
        kd = (keep + PAGE - 1) // PAGE
        to_pool = torch.full((B * kd + 1, layers, 2, kvh, PAGE, HD), 9.0, dtype=torch.bfloat16, device="cuda")
        k_to, v_to = to_pool[:, :, 0], to_pool[:, :, 1]
        bt_to = torch.randperm(B * kd + 1, generator=torch.Generator().manual_seed(1)).int().cuda()[:B * kd].view(B, kd)
        acc_to = torch.full((B, layers, kvh, keep), 4.0, device="cuda")
        to = M.KvCache(k_to, v_to, bt_to, c.lens_t, keep)
        ctx.kv_evict(c.cache, to, acc, acc_to, keep=keep, sinks=sinks, recent=recent, index=index, stream=s)
        assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(acc.nan_to_num(5), a0.nan_to_num(5))
    else:
        k_to, v_to, bt_to, acc_to = c.k, c.v, c.bt, acc
        ctx.kv_evict(c.cache, acc=acc, keep=keep, sinks=sinks, recent=recent, index=index, stream=s)
    torch.cuda.synchronize()
    ctx.sync()
    touched = torch.zeros(k_to.shape[:4], dtype=torch.bool, device="cuda")  # [page, layer, head, slot]
    written = torch.zeros(acc_to.shape, dtype=torch.bool, device="cuda")
    a_host = a0.cpu().tolist()
    for b, n in enumerate(lens):
        for l in range(layers):
            for h in range(kvh):
                stay = kept(a_host[b][l][h], n, keep, sinks, recent)
                m = len(stay)
                assert index[b, l, h].tolist() == stay + [-1] * (keep - m)
                i = torch.tensor(stay, dtype=torch.long, device="cuda")
                t = torch.arange(m, device="cuda")
                src, dst = c.bt[b].long()[i // PAGE], bt_to[b].long()[t // PAGE]
                for to_, from_ in ((k_to, k0), (v_to, v0)):
                    assert torch.equal(to_[dst, l, h, t % PAGE].view(torch.int16), from_[src, l, h, i % PAGE].view(torch.int16))
                assert torch.equal(acc_to[b, l, h, :m].view(torch.int32), a0[b, l, h, i].view(torch.int32))
                touched[dst, l, h, t % PAGE] = True
                written[b, l, h, :m] = True
    # nothing else was written
    rest = (k0, v0, a0) if place == "same" else (torch.full_like(k_to, 9.0), torch.full_like(v_to, 9.0), torch.full_like(acc_to, 4.0))
    assert torch.equal(k_to[~touched].view(torch.int16), rest[0][~touched].view(torch.int16))
    assert torch.equal(v_to[~touched].view(torch.int16), rest[1][~touched].view(torch.int16))
    assert torch.equal(acc_to[~written].view(torch.int32), rest[2][~written].view(torch.int32))


@pytest.mark.parametrize("n,sinks,recent", [(4096, 0, 0), (4097, 0, 0), (4097, 1, 0), (4099, 1, 2), (4100, 1, 2), (513, 1, 0), (514, 1, 0)])
@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_evict_where_the_selection_changes(ctx, n, sinks, recent, kind):
    """As many positions to choose from as threads hold, and one more or less."""
    test_evict(ctx, [n, 17, n - 1], 401, sinks, recent, kind, "same")


@pytest.mark.parametrize("seqs,layers", [(1, 24), (2, 24), (8, 24), (5, 40)])
@pytest.mark.parametrize("place", ["apart", "same"])
def test_evict_many_heads(ctx, seqs, layers, place):
    """From few heads (several CTAs each) to many (one), against a stable sort."""
    kvh, keep, sinks, recent = 2, 300, 3, 50
    g = torch.Generator().manual_seed(seqs)
    lens = [900] + torch.randint(1, 900, (seqs - 1,), generator=g).tolist()
    c = Case(lens, [1] * seqs, 14, kvh, layers=layers, poison=False, seed=seqs)
    n = torch.tensor(lens, device="cuda")[:, None, None, None]
    acc = totals((seqs, layers, kvh, 900), "spread", seqs) * (torch.rand(seqs, layers, kvh, 900, device="cuda") > 0.3)
    j = torch.arange(900, device="cuda")
    a = torch.where((j < sinks) | (j >= n - recent), math.inf, acc)
    a = torch.where(j < n, a, -math.inf)
    best = a.argsort(dim=-1, descending=True, stable=True)[..., :keep].sort(-1).values
    best = torch.where(n <= keep, j[:keep].expand_as(best), best)
    stay = j[:keep] < n.clamp(max=keep)
    want_index = torch.where(stay, best, -1)
    b, l, h, s = stay.expand_as(best).nonzero(as_tuple=True)
    i = best[b, l, h, s]
    src = c.bt.long()[b, i // PAGE]
    wk, wv, wa = c.k[src, l, h, i % PAGE], c.v[src, l, h, i % PAGE], acc[b, l, h, i]
    index = torch.empty(seqs, layers, kvh, keep, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    if place == "same":
        k_to, v_to, bt_to, acc_to = c.k, c.v, c.bt, acc
        ctx.kv_evict(c.cache, acc=acc, keep=keep, sinks=sinks, recent=recent, index=index, stream=stream)
    else:
        kd = (keep + PAGE - 1) // PAGE
        pool = torch.zeros(seqs * kd, layers, 2, kvh, PAGE, HD, dtype=torch.bfloat16, device="cuda")
        k_to, v_to, acc_to = pool[:, :, 0], pool[:, :, 1], torch.zeros(seqs, layers, kvh, keep, device="cuda")
        bt_to = torch.arange(seqs * kd, dtype=torch.int32, device="cuda").view(seqs, kd)
        ctx.kv_evict(c.cache, M.KvCache(k_to, v_to, bt_to, c.lens_t, keep), acc, acc_to, keep=keep, sinks=sinks, recent=recent,
                     index=index, stream=stream)
    torch.cuda.synchronize()
    ctx.sync()
    dst = bt_to.long()[b, s // PAGE]
    assert torch.equal(index.long(), want_index)
    assert torch.equal(k_to[dst, l, h, s % PAGE], wk) and torch.equal(v_to[dst, l, h, s % PAGE], wv)
    assert torch.equal(acc_to[b, l, h, s], wa)


def test_evict_without_totals(ctx):
    """keep = sinks + recent needs no totals: sinks and the last positions."""
    c = Case([100, 7], [1, 1], 14, 2, layers=2, poison=False)
    k0 = c.k.clone()
    ctx.kv_evict(c.cache, keep=20, sinks=4, recent=16, stream=torch.cuda.current_stream().cuda_stream)
    stay = torch.tensor(list(range(4)) + list(range(84, 100)), device="cuda")
    t = torch.arange(20, device="cuda")
    bt = c.bt[0].long()
    assert torch.equal(c.k[bt[t // PAGE], :, :, t % PAGE], k0[bt[stay // PAGE], :, :, stay % PAGE])


# ---------------------------------------------------------------------------
# calls the documentation allows
# ---------------------------------------------------------------------------

def test_prompt_tokens_and_eviction_together(ctx):
    """A stream as a program runs it: a prompt in two chunks, tokens, eviction
    in place when the cache is over its budget, tokens on what stayed; after
    the eviction a cache equals one that holds only the kept positions."""
    kvh, heads, sinks, recent, keep = 2, 14, 2, 10, 40
    c = Case([120], [50], heads, kvh, poison=False, seed=21)
    s = torch.cuda.current_stream().cuda_stream
    acc = torch.full((1, 1, kvh, 128), math.nan, device="cuda")  # entries are set when their positions are new
    want = torch.zeros(kvh, 120, dtype=torch.float64, device="cuda")
    q = torch.randn(120, heads, HD, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.bfloat16)
    k = [c.rows_of(c.k, 0, h) for h in range(kvh)]
    for lo, hi in ((0, 61), (61, 117)):
        lens = torch.tensor([hi], dtype=torch.int32, device="cuda")
        cache = M.KvCache(c.k, c.v, c.bt, lens, 128)
        out, lse = torch.empty_like(q[lo:hi]), torch.empty(hi - lo, heads, device="cuda")
        start = torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda")
        ctx.attn_prefill(q[lo:hi], start, cache, out, lse=lse, stream=s)
        ctx.attn_weights(q[lo:hi], start, cache, lse, acc, stream=s)
    for n in (118, 119, 120):
        cache = M.KvCache(c.k, c.v, c.bt, torch.tensor([n], dtype=torch.int32, device="cuda"), 128)
        ctx.attn_decode(q[n - 1:n], cache, torch.empty_like(q[:1]), acc=acc, stream=s)
    for h in range(kvh):
        x = torch.einsum("rgd,jd->rgj", q.double().view(120, kvh, 7, HD)[:, h], k[h]) / 8
        x = x.masked_fill(~sees(120, 120, 0, 0)[:, None], -math.inf)
        want[h] = torch.softmax(x, -1).sum((0, 1))
    assert torch.allclose(acc[0, 0, :, :120].double(), want, rtol=1e-4, atol=0)
    index = torch.empty(1, 1, kvh, keep, dtype=torch.int32, device="cuda")
    vals = [c.rows_of(c.v, 0, h) for h in range(kvh)]
    ctx.kv_evict(cache, acc=acc, keep=keep, sinks=sinks, recent=recent, index=index, stream=s)
    lens = torch.tensor([keep], dtype=torch.int32, device="cuda")
    cache = M.KvCache(c.k, c.v, c.bt, lens, 128)
    out = torch.empty_like(q[:1])
    ctx.attn_decode(q[:1], cache, out, stream=s)
    for h in range(kvh):
        i = index[0, 0, h].long()
        x = q[0].double().view(kvh, 7, HD)[h] @ k[h][i].T / 8
        ref = torch.softmax(x, -1) @ vals[h][i]
        assert torch.allclose(out[0].double().view(kvh, 7, HD)[h], ref, rtol=2 * H16, atol=1e-4)
    torch.cuda.synchronize()
    ctx.sync()


def test_streams_graphs_and_repeats(ctx):
    """Two calls at once on two streams, a captured graph replayed on new
    inputs, and the context's own stream give what a call alone gives."""
    a, b = Case([900, 33], [300, 33], 14, 2, 200, 4, seed=1), Case([900, 33], [300, 33], 14, 2, 200, 4, seed=2)
    da, db = Case([4000] * 2, [1] * 2, 14, 2, seed=3), Case([4000] * 2, [1] * 2, 14, 2, seed=4)

    def both(c, d, stream):
        o, z = torch.empty(c.q.shape, dtype=torch.bfloat16, device="cuda"), torch.empty(c.q.shape[:2], device="cuda")
        acc, dacc, do = c.acc0.clone(), d.acc0.clone(), torch.empty_like(d.q.contiguous())
        ix = torch.empty(2, 1, 2, 100, dtype=torch.int32, device="cuda")

        def go(stream):
            ctx.attn_prefill(c.q, c.q_start, c.cache, o, lse=z, max_rows=300, window=200, sinks=4, stream=stream)
            ctx.attn_weights(c.q, c.q_start, c.cache, z, acc, max_rows=300, window=200, sinks=4, stream=stream)
            ctx.attn_decode(d.q, d.cache, do, acc=dacc, stream=stream)
        return go, (o, z, acc, do, dacc, ix)

    torch.cuda.synchronize()
    cur = torch.cuda.current_stream().cuda_stream
    want = []
    for c, d in ((a, da), (b, db)):
        go, outs = both(c, d, cur)
        go(cur)
        torch.cuda.synchronize()
        want.append([t.clone() for t in outs[:5]])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    runs = [both(a, da, s1), both(b, db, s2)]
    torch.cuda.synchronize()
    for (go, _), s in zip(runs, (s1, s2)):
        go(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, outs), w in zip(runs, want):
        assert all(torch.equal(x, y) for x, y in zip(outs, w))
    # the context's own stream
    go, outs = both(a, da, None)
    torch.cuda.synchronize()
    go(None)
    ctx.sync()
    assert all(torch.equal(x, y) for x, y in zip(outs, want[0]))
    # captured, then replayed after the inputs changed in place
    go, outs = both(a, da, None)
    fresh = [t.clone() for t in (outs[2], outs[4])]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1):
        go(s1.cuda_stream)
    for x, y in ((outs[2], fresh[0]), (outs[4], fresh[1])):
        x.copy_(y)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want[0]))
    a.q.copy_(b.q), a.k.copy_(b.k), a.v.copy_(b.v), a.bt.copy_(b.bt), outs[2].copy_(b.acc0)
    da.q.copy_(db.q), da.k.copy_(db.k), da.v.copy_(db.v), da.bt.copy_(db.bt), outs[4].copy_(db.acc0)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want[1]))
    ctx.sync()


def test_what_only_the_device_sees_is_reported(ctx):
    """Bad pages, lengths and row starts are read safely and reported once."""
    s = torch.cuda.current_stream().cuda_stream

    def reported(words):
        torch.cuda.synchronize()
        with pytest.raises(M.MingError, match=words):
            ctx.sync()
        ctx.sync()

    for bad in (-1, 10 ** 9, -2 ** 31):
        c = Case([100, 50], [20, 50], 14, 2, poison=False)
        c.bt[0, 3] = bad
        run = lambda: (torch.empty_like(c.q), torch.zeros(c.q.shape[:2], device="cuda"))  # noqa: E731
        o, z = run()
        ctx.attn_prefill(c.q, c.q_start, c.cache, o, lse=z, max_rows=50, stream=s)
        reported("block table")
        ctx.attn_weights(c.q, c.q_start, c.cache, z, c.acc0, max_rows=50, stream=s)
        reported("block table")
        q = c.q[:2].contiguous()
        ctx.attn_decode(q, c.cache, torch.empty_like(q), stream=s)
        reported("block table")
        ctx.kv_evict(c.cache, acc=c.acc0, keep=60, stream=s)
        reported("block table")
    for bad in (101, -1, 2 ** 31 - 1):
        c = Case([100, 50], [20, 50], 14, 2, poison=False)
        c.lens_t[1] = bad
        q = c.q[:2].contiguous()
        ctx.attn_decode(q, c.cache, torch.empty_like(q), acc=c.acc0, stream=s)
        # positions past the sequence's own pages have no table entry either: whichever came first is named
        reported("length|block table")
    for starts in ([0, 30, 10], [0, 20, 71], [-3, 20, 70], [0, 69, 70]):
        c = Case([100, 50], [20, 50], 14, 2, poison=False)
        c.q_start.copy_(torch.tensor(starts))
        o, z = torch.empty_like(c.q), torch.zeros(c.q.shape[:2], device="cuda")
        ctx.attn_prefill(c.q, c.q_start, c.cache, o, lse=z, max_rows=50, stream=s)
        reported("q_start")


def test_refusals_of_the_python_layer(ctx):
    c = Case([40], [8], 14, 2)
    o = torch.empty_like(c.q)
    bad = [
        lambda: ctx.attn_prefill(c.q.float(), c.q_start, c.cache, o),
        lambda: ctx.attn_prefill(c.q, c.q_start.long(), c.cache, o),
        lambda: ctx.attn_prefill(c.q, c.q_start[:1], c.cache, o),
        lambda: ctx.attn_prefill(c.q, c.q_start, c.cache, o[:4]),
        lambda: ctx.attn_prefill(c.q, c.q_start, c.cache, o.cpu()),
        lambda: ctx.attn_prefill(c.q[..., ::2], c.q_start, c.cache, o),
        lambda: ctx.attn_prefill(c.q, c.q_start, c.cache, o, lse=torch.empty(14, 8, device="cuda").T),
        lambda: ctx.attn_prefill(c.q, c.q_start, c.cache, o, layer=1),
        lambda: ctx.attn_prefill(c.q[:, :13], c.q_start, c.cache, o[:, :13]),
        lambda: ctx.attn_weights(c.q, c.q_start, c.cache, None, c.acc0),
        lambda: ctx.attn_weights(c.q, c.q_start, c.cache, torch.zeros(8, 14, device="cuda"), c.acc0[..., :20]),
        lambda: ctx.attn_decode(c.q, c.cache, o),
        lambda: ctx.attn_decode(c.q[:1], c.cache, o[:1], window=-1),
        lambda: ctx.kv_evict(c.cache, keep=20),
        lambda: ctx.kv_evict(c.cache, acc=c.acc0, keep=20, index=torch.zeros(1, 1, 2, 19, dtype=torch.int32, device="cuda")),
        lambda: M.KvCache(c.k, c.v, c.bt, c.lens_t, 10 ** 6),
        lambda: M.KvCache(c.k, c.v[:-1], c.bt, c.lens_t, 16),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(M.MingError):
            f()
            pytest.fail(f"call {i} was accepted")


def test_broadcast_tensors_are_refused(ctx):
    """A table whose rows are one row, results and totals that share places."""
    c = Case([40, 40], [1, 1], 14, 2)
    o = torch.empty_like(c.q)
    to = M.KvCache(c.k.clone(), c.v.clone(), c.bt, c.lens_t, 40)
    bad = [
        lambda: M.KvCache(c.k, c.v, c.bt[:1].expand(2, -1), c.lens_t, 40),
        lambda: M.KvCache(c.k, c.v, c.bt[:1, :1].expand(2, 1), c.lens_t, 16),
        lambda: M.KvCache(c.k, c.v, c.bt, c.lens_t[:1].expand(2), 40),
        lambda: ctx.attn_prefill(c.q, c.q_start, c.cache, o[:1].expand_as(o)),
        lambda: ctx.attn_decode(c.q, c.cache, o[:, :1].expand_as(o)),
        lambda: ctx.attn_decode(c.q, c.cache, o, acc=c.acc0[:1].expand_as(c.acc0)),
        lambda: ctx.attn_weights(c.q, c.q_start, c.cache, torch.zeros(2, 14, device="cuda"), c.acc0[:, :, :1].expand_as(c.acc0)),
        lambda: ctx.kv_evict(c.cache, to, c.acc0, c.acc0[:1].expand_as(c.acc0), keep=20),
        lambda: ctx.kv_evict(c.cache, None, c.acc0, c.acc0.clone(), keep=20),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(M.MingError):
            f()
            pytest.fail(f"call {i} was accepted")
    # a batch of one has nothing to step over
    M.KvCache(c.k, c.v, c.bt[:1].expand(1, -1), c.lens_t[:1], 40)


def test_nothing_to_do(ctx):
    s = torch.cuda.current_stream().cuda_stream
    c = Case([40, 9], [0, 0], 14, 2, poison=False)
    q = torch.empty(0, 14, HD, dtype=torch.bfloat16, device="cuda")
    ctx.attn_prefill(q, c.q_start, c.cache, q, stream=s)
    acc = c.acc0.clone()
    ctx.attn_weights(q, c.q_start, c.cache, torch.empty(0, 14, device="cuda"), acc, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(acc, c.acc0)
    c = Case([0, 0], [1, 1], 14, 2, poison=False)
    o = torch.full_like(c.q, 3.0)
    ctx.attn_decode(c.q, c.cache, o, acc=c.acc0, stream=s)
    torch.cuda.synchronize()
    assert (o == 0).all()
    ctx.kv_evict(c.cache, acc=c.acc0, keep=3, stream=s)
    torch.cuda.synchronize()
    ctx.sync()
