"""Attention over bounded paged K/V caches: the measured operators.

A long stream of speech tokens does not keep every position of its prompt and
of what it has said: the first few positions stay (sinks), a window of the last
ones stays, and of those between the ones that attention has used most. Four
operators do that work on a paged bf16 cache (pages of 16 positions, head
dimension 64, grouped query heads):

* ``prefill``: attention of a prompt's new rows, causal, with a window and sinks;
  outputs and each row's log-sum-exp;
* ``weights``: the attention weights that those rows gave to each cached position,
  summed over rows and the query heads of a group, added to a running total;
* ``decode``: attention of one new token per sequence, with window and sinks,
  its weights added to the same total where the cache is tracked;
* ``evict``: of each (sequence, layer, kv head) the sinks, the last positions and
  the positions of the largest total stay, moved together in order.

Row i of a sequence of ``len`` cached positions with ``n`` new rows sits at
position p = len - n + i and sees j <= p with j < sinks or j > p - window
(window 0: every j <= p).
"""
import functools
import math
import random

import torch

own = False

PAGE, HD = 16, 64
SCALE = 0.125  # 1 / sqrt(64)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a short prompt on an empty cache: the 128 positions every default request starts with
        dict(name="prefill 1x128", op="prefill", seqs=1, rows=128, cached=0, ragged=False, heads=14, kv_heads=2, window=0, sinks=0),
        # a handful of requests admitted together, prompts of odd lengths, the window of a streaming voice
        dict(name="prefill 8 ragged window", op="prefill", seqs=8, rows=509, cached=0, ragged=True, heads=14, kv_heads=2, window=256, sinks=4),
        # the second chunk of a long prompt
        dict(name="prefill chunk on 2048", op="prefill", seqs=1, rows=2048, cached=2048, ragged=False, heads=14, kv_heads=2, window=1024, sinks=4),
        # many 2048-position prompts at once, full causal attention
        dict(name="prefill 16x2048", op="prefill", seqs=16, rows=2048, cached=0, ragged=False, heads=14, kv_heads=2, window=0, sinks=0),
        # weights of a short odd prompt
        dict(name="weights 1x333", op="weights", seqs=1, rows=333, cached=0, ragged=False, heads=14, kv_heads=2, window=0, sinks=0),
        # weights of 2048-position prompts
        dict(name="weights 8x2048", op="weights", seqs=8, rows=2048, cached=0, ragged=True, heads=14, kv_heads=2, window=0, sinks=0),
        # one voice at the end of its default 512 positions: latency alone
        dict(name="decode 1x509", op="decode", seqs=1, cached=509, ragged=False, heads=14, kv_heads=2, window=0, sinks=0, track=False),
        # a batch of voices of uneven lengths on a window, tracked
        dict(name="decode 32 window track", op="decode", seqs=32, cached=2053, ragged=True, heads=14, kv_heads=2, window=512, sinks=4, track=True),
        # one very long cache: the split over its length carries it
        dict(name="decode 1x32768", op="decode", seqs=1, cached=32768, ragged=False, heads=14, kv_heads=2, window=0, sinks=0, track=False),
        # the largest batch at the default limit of positions, tracked
        dict(name="decode 64x4096 track", op="decode", seqs=64, cached=4096, ragged=False, heads=14, kv_heads=2, window=0, sinks=0, track=True),
        # one sequence of a 24-layer cache brought back under its budget
        dict(name="evict 1x777", op="evict", seqs=1, cached=777, ragged=False, layers=24, kv_heads=2, keep=512, sinks=4, recent=128),
        # a batch of long caches cut to a quarter
        dict(name="evict 16x4096", op="evict", seqs=16, cached=4096, ragged=True, layers=24, kv_heads=2, keep=1024, sinks=4, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "weights", "decode", "evict"])
    kv_heads, group = rng.choice([(2, 7), (2, 7), (2, 8), (4, 2), (8, 1), (1, 5)])
    c = dict(op=op, kv_heads=kv_heads, ragged=rng.random() < 0.6)
    if op == "evict":
        c["layers"] = rng.choice([2, 6, 24])
        c["seqs"] = _log(rng, 1, 16)
        c["cached"] = _log(rng, 100, min(4096, 2_000_000 // (c["seqs"] * c["layers"] * kv_heads)))
        c["keep"] = max(20, int(c["cached"] * rng.uniform(0.2, 0.9)))
        c["sinks"] = rng.choice([0, 1, 4, 16])
        c["recent"] = rng.randint(0, c["keep"] - c["sinks"])
        return c
    c["heads"] = kv_heads * group
    c["window"] = rng.choice([0, 0, _log(rng, 16, 2048)])
    c["sinks"] = rng.choice([0, 1, 4, 20]) if c["window"] else 0
    if op == "decode":
        c["seqs"] = _log(rng, 1, 64)
        c["cached"] = _log(rng, 16, min(32768, 8 * 64 * 4096 // (c["seqs"] * kv_heads * 4)))
        c["track"] = rng.random() < 0.5
    else:
        c["rows"] = _log(rng, 2, 2048)
        c["cached"] = rng.choice([0, 0, _log(rng, 1, 2048)])
        c["seqs"] = _log(rng, 1, 8)
    return c


def _lens(case):
    """(cached positions in all, new rows) of each sequence; the same for every seed."""
    r = random.Random("%d %d %d" % (case["seqs"], case["cached"], case.get("rows", 0)))
    new = case["op"] in ("prefill", "weights")
    lens, rows = [], []
    for b in range(case["seqs"]):
        full = not case["ragged"] or b == 0  # the first one always has the full length
        n = 0 if not new else case["rows"] if full else r.randint(1, case["rows"])
        p = case["cached"] if full else r.randint(0 if new else 1, case["cached"]) if case["cached"] else 0
        lens.append(p + n)
        rows.append(n if new else 1)
    return lens, rows


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    lens, rows = _lens(case)
    layers, kvh, B = case.get("layers", 1), case["kv_heads"], case["seqs"]
    ld = (max(lens) + PAGE - 1) // PAGE
    held = [(n + PAGE - 1) // PAGE for n in lens]
    pages = sum(held) + 3

    def pool(pages):
        # the framework's page: [layer][K|V][kv head][16 positions][64]
        return torch.zeros(pages, layers, 2, kvh, PAGE, HD, dtype=torch.bfloat16, device="cuda")

    def table(held, ld, pages):
        bt = torch.zeros(B, ld, dtype=torch.int32, device="cuda")
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        at = 0
        for b, h in enumerate(held):
            bt[b, :h] = order[at:at + h]
            at += h
        return bt

    kv = pool(pages).normal_(generator=g)
    # keys of one direction per head, more or less of it per position: a few
    # positions draw most of the attention, as they do in a trained model
    kv[:, :, 0] *= 1.5 * torch.rand(pages, layers, kvh, PAGE, 1, generator=g, device="cuda").to(torch.bfloat16)
    s = dict(case=case, k=kv[:, :, 0], v=kv[:, :, 1], bt=table(held, ld, pages),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), max_len=max(lens), max_rows=max(rows))
    if case["op"] == "evict":
        # running totals: most positions drew little, some none at all (ties), a few a lot
        acc = torch.randn(B, layers, kvh, ld * PAGE, generator=g, device="cuda").mul_(2).exp_()
        s["acc"] = acc * (torch.rand(acc.shape, generator=g, device="cuda") > 0.1)
        keep = case["keep"]
        kd = (keep + PAGE - 1) // PAGE
        to = pool(B * kd + 1)
        s["k_to"], s["v_to"], s["bt_to"] = to[:, :, 0], to[:, :, 1], table([kd] * B, kd, B * kd + 1)
        s["acc_to"] = torch.zeros(B, layers, kvh, kd * PAGE, device="cuda")
        s["index"] = torch.empty(B, layers, kvh, keep, dtype=torch.int32, device="cuda")
    else:
        n, H = sum(rows), case["heads"]
        s["q"] = torch.randn(n, H, HD, generator=g, device="cuda").mul_(1.5).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        s["lse"] = torch.empty(n, H, device="cuda")
        if case["op"] == "weights" or case.get("track"):
            s["acc"] = torch.rand(B, 1, kvh, ld * PAGE, generator=g, device="cuda")
        if case["op"] == "weights":
            # what the prefill of these rows gave
            s["lse"] = _attend(s, case)[1]
    if own:
        import sys
        if "ming-tts-serve_b200" not in sys.path:
            sys.path.insert(0, "ming-tts-serve_b200")
        import ming_b200
        s["cache"] = ming_b200.KvCache(s["k"], s["v"], s["bt"], s["lens"], s["max_len"])
        if case["op"] == "evict":
            s["cache_to"] = ming_b200.KvCache(s["k_to"], s["v_to"], s["bt_to"], s["lens"], case["keep"])
        s["ctx"] = _context()
    return s


@functools.lru_cache(None)
def _context():
    """The context a program holds for its GPU (no model: the caches are the caller's)."""
    import ming_b200
    return ming_b200.Context(ming_b200.default_cfg(layers=0, dit_mode=ming_b200.DIT_NONE, agg_blocks=0), device=0)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _rows_of(s):
    """(sequence, position) of every row, and which cached positions each sees: [rows, max_len]."""
    start, lens = s["q_start"].long(), s["lens"].long()
    r = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], r, right=True)
    pos = lens[seq] - (start[seq + 1] - r)
    return seq, pos


def _sees(pos, n, window, sinks):
    j = torch.arange(n, device="cuda")
    p = pos[..., None]
    see = j <= p
    if window:
        see = see & ((j < sinks) | (j > p - window))
    return see


def _padded(s, name):
    """K or V of every sequence, [seqs, kv heads, max_len, 64] in 32 bits."""
    j = torch.arange(s["max_len"], device="cuda")
    page = s["bt"].long()[:, j // PAGE]
    return s[name][:, 0][page, :, j % PAGE].permute(0, 2, 1, 3).float()


def _scores(s, case):
    """Softmax numerators' logits of every (sequence, kv head, group head, row): padded to
    [seqs, kv heads, group, rows, max_len], what is not seen at -inf; and the rows' places."""
    B, kvh = case["seqs"], case["kv_heads"]
    G, n = case["heads"] // kvh, s["max_len"]
    seq, pos = _rows_of(s)
    at = torch.arange(seq.numel(), device="cuda") - s["q_start"].long()[seq]
    q = torch.zeros(B, s["max_rows"], kvh, G, HD, device="cuda")
    q[seq, at] = s["q"].float().view(-1, kvh, G, HD)
    where = torch.full((B, s["max_rows"]), -1, dtype=torch.long, device="cuda")
    where[seq, at] = pos
    k = _padded(s, "k")
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, kvh, -1, HD), k.transpose(-1, -2)) * SCALE
    x = x.view(B, kvh, G, s["max_rows"], n)
    x.masked_fill_(~_sees(where, n, case["window"], case["sinks"])[:, None, None], -math.inf)
    return x, seq, at


def _attend(s, case):
    """Outputs [rows, heads, 64] and log-sum-exp [rows, heads]."""
    x, seq, at = _scores(s, case)
    B, kvh, G, R, n = x.shape
    m = x.amax(-1, keepdim=True).clamp_min(-1e30)
    x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, kvh, G * R, n), _padded(s, "v")).view(B, kvh, G, R, HD) / total.clamp_min(1e-30)
    lse = (m + total.log())[..., 0]
    take = lambda t: t.permute(0, 3, 1, 2, *range(4, t.dim()))[seq, at].flatten(1, 2)  # noqa: E731
    return take(o).to(torch.bfloat16), take(lse).contiguous()


def _weigh(s, case, lse):
    """The running totals with these rows' weights: positions the rows themselves brought start anew."""
    x, seq, at = _scores(s, case)
    B, kvh, G, R, n = x.shape
    l = torch.zeros(B, R, kvh, G, device="cuda")
    l[seq, at] = lse.view(-1, kvh, G)
    w = x.sub_(l.permute(0, 2, 3, 1)[..., None]).exp_().sum((2, 3))
    start, j = s["q_start"].long(), torch.arange(n, device="cuda")
    old = j < (s["lens"].long() - (start[1:] - start[:-1]))[:, None]
    held = j < s["lens"].long()[:, None]
    acc = s["acc"][:, 0, :, :n]
    acc.copy_(torch.where(held[:, None], torch.where(old[:, None], acc, 0) + w, acc))
    return s["acc"]


def _evict(s, case):
    n, keep = s["max_len"], case["keep"]
    lens = s["lens"].long()[:, None, None, None]
    j = torch.arange(n, device="cuda")
    a = s["acc"][..., :n]
    a = torch.where(a.isnan(), -math.inf, a)
    a = torch.where((j < case["sinks"]) | (j >= lens - case["recent"]), math.inf, a)
    a = torch.where(j < lens, a, -math.inf)
    best = a.argsort(dim=-1, descending=True, stable=True)[..., :keep]
    best = torch.where(best < lens, best, n).sort(-1).values
    if n < keep:
        best = torch.nn.functional.pad(best, (0, keep - n), value=n)
    stay = best < n
    s["index"].copy_(torch.where(stay, best, -1))
    b, l, h, t = stay.nonzero(as_tuple=True)
    i = best[stay]
    page, to = s["bt"].long()[b, i // PAGE], s["bt_to"].long()[b, t // PAGE]
    s["k_to"][to, l, h, t % PAGE] = s["k"][page, l, h, i % PAGE]
    s["v_to"][to, l, h, t % PAGE] = s["v"][page, l, h, i % PAGE]
    s["acc_to"][b, l, h, t] = s["acc"][b, l, h, i]
    return s["k_to"], s["v_to"], s["acc_to"], s["index"]


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        ctx, stream = s["ctx"], torch.cuda.current_stream().cuda_stream
        if op == "prefill":
            ctx.attn_prefill(s["q"], s["q_start"], s["cache"], s["out"], lse=s["lse"], max_rows=s["max_rows"],
                             window=c["window"], sinks=c["sinks"], stream=stream)
            return s["out"], s["lse"]
        if op == "weights":
            ctx.attn_weights(s["q"], s["q_start"], s["cache"], s["lse"], s["acc"], max_rows=s["max_rows"],
                             window=c["window"], sinks=c["sinks"], stream=stream)
            return s["acc"]
        if op == "decode":
            ctx.attn_decode(s["q"], s["cache"], s["out"], acc=s.get("acc"), window=c["window"], sinks=c["sinks"], stream=stream)
            return (s["out"], s["acc"]) if c["track"] else s["out"]
        ctx.kv_evict(s["cache"], s["cache_to"], s["acc"], s["acc_to"], keep=c["keep"], sinks=c["sinks"], recent=c["recent"],
                     index=s["index"], stream=stream)
        return s["k_to"], s["v_to"], s["acc_to"], s["index"]
    if op == "prefill":
        return _attend(s, c)
    if op == "weights":
        return _weigh(s, c, s["lse"])
    if op == "decode":
        out, lse = _attend(s, c)
        return (out, _weigh(s, c, lse)) if c["track"] else out
    return _evict(s, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _seen(case):
    """(pairs of rows and positions, positions that any row sees) over all sequences."""
    pairs = positions = 0
    W, S = case["window"], case["sinks"]
    for n, r in zip(*_lens(case)):
        first = n - r
        if W:
            # row at p: min(W, p + 1) of the window, and the sinks before it
            pairs += sum(min(W, p + 1) + min(S, max(0, p + 1 - W)) for p in range(first, n))
            lo = max(0, first - W + 1)
            positions += n - lo + min(S, lo)
        else:
            pairs += r * first + r * (r + 1) // 2
            positions += n
    return pairs, positions


def work(case):
    lens, rows = _lens(case)
    kvh = case["kv_heads"]
    if case["op"] == "evict":
        total, kept = sum(lens), sum(min(n, case["keep"]) for n in lens)
        per = case["layers"] * kvh
        return {"bytes": per * (4 * total + kept * (2 * (2 * HD * 2 + 4) + 4)), "flops": 0}
    pairs, positions = _seen(case)
    H, n = case["heads"], sum(rows)
    q = n * H * HD * 2
    if case["op"] == "weights":
        return {"bytes": q + n * H * 4 + positions * kvh * (HD * 2 + 8), "flops": 2 * HD * H * pairs}
    return {"bytes": 2 * q + (n * H * 4 if case["op"] == "prefill" else 0) +
            positions * kvh * (2 * HD * 2 + (8 if case.get("track") else 0)), "flops": 4 * HD * H * pairs}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    lens, rows = _lens(case)
    bt = s["bt"].cpu()

    def one(name, b, layer, h, n):
        pages = bt[b, :(n + PAGE - 1) // PAGE].long().cuda()
        return s[name][pages, layer, h].reshape(-1, HD)[:n]

    if case["op"] == "evict":
        for b, n in enumerate(lens):
            m = min(n, case["keep"])
            a = s["acc"][b, :, :, :n].double().cpu()
            rank = torch.arange(n)
            must = (rank < case["sinks"]) | (rank >= n - case["recent"])
            order = torch.where(must, torch.full_like(a, math.inf), a).neg().sort(dim=-1, stable=True).indices
            idx = order[..., :m].sort(-1).values
            s["index"][b] = -1
            s["index"][b, :, :, :m] = idx.cuda()
            s["acc_to"][b, :, :, :m] = a.gather(-1, idx).cuda()
            t = torch.arange(m, device="cuda")
            to = s["bt_to"][b].long()[t // PAGE]
            for layer in range(case["layers"]):
                for h in range(case["kv_heads"]):
                    i = idx[layer, h].cuda()
                    s["k_to"][to, layer, h, t % PAGE] = one("k", b, layer, h, n)[i]
                    s["v_to"][to, layer, h, t % PAGE] = one("v", b, layer, h, n)[i]
        return s["k_to"].double(), s["v_to"].double(), s["acc_to"].double(), s["index"]
    H, kvh = case["heads"], case["kv_heads"]
    G, W = H // kvh, case["window"]
    out = torch.zeros(sum(rows), H, HD, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(rows), H, dtype=torch.float64, device="cuda")
    acc = s["acc"].double() if "acc" in s else None
    at = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        p = torch.arange(n - r, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = j > p
        if W:
            hidden |= (j <= p - W) & (j >= case["sinks"])
        for h in range(kvh):
            k, v = one("k", b, 0, h, n).double(), one("v", b, 0, h, n).double()
            total = torch.zeros(n, dtype=torch.float64, device="cuda")
            for i in range(h * G, h * G + G):
                x = (s["q"][at:at + r, i].double() @ k.T) * SCALE
                x[hidden] = -math.inf
                z = torch.logsumexp(x, -1)
                lse[at:at + r, i] = z
                # the weights operator is given the rows' log-sum-exp in 32 bits
                w = torch.exp(x - (s["lse"][at:at + r, i].double() if case["op"] == "weights" else z)[:, None])
                out[at:at + r, i] = w @ v
                total += w.sum(0)
            if acc is not None:
                fresh = n - r
                acc[b, 0, h, fresh:n] = 0
                acc[b, 0, h, :n] += total
        at += r
    if case["op"] == "prefill":
        return out, lse
    if case["op"] == "weights":
        return acc
    return (out, acc) if case["track"] else out
