"""Operators for serving several requests at once, as cases that can be timed and compared.

  chunk     ``ops.prefill_attention_paged``: attention of several new tokens per row over a paged cache that holds them already
  adapters  ``ops.add_adapters``: what each request's low-rank adapter adds to the output of a projection that all requests share
With ``own`` false ``run`` computes them from elementary operations in float32.  Everything a case hands over is bfloat16, the type that
the package serves in; lengths, tables and slots are int32, as its caches keep them.
"""
import math

import torch

own = False

D, BF = 128, torch.bfloat16


def listed():
    return [
        # four drafted tokens of four short conversations on a small model: launches and latency
        dict(name="draft_few", path="chunk", rows=4, tokens=4, heads=6, kv_heads=6, low=40, high=500, page=192, window=-1, ragged=False),
        # five drafted tokens a row in a served batch of ragged length, grouped heads
        dict(name="draft_batch", path="chunk", rows=48, tokens=5, heads=16, kv_heads=4, low=1, high=4095, page=192, window=-1, ragged=False),
        # drafted tokens behind long contexts, as many key/value heads as heads
        dict(name="draft_long", path="chunk", rows=2, tokens=8, heads=12, kv_heads=12, low=32768, high=65535, page=192, window=-1, ragged=False),
        # a mixed batch: rows in the middle of their prompts beside rows with a token or none, short window, small pages
        dict(name="mixed", path="chunk", rows=24, tokens=384, heads=16, kv_heads=4, low=0, high=8192, page=48, window=1024, ragged=True),
        # eight prompts of 2048 tokens straight into pages
        dict(name="prompts", path="chunk", rows=8, tokens=2048, heads=12, kv_heads=12, low=0, high=0, page=192, window=-1, ragged=False),
        # a portion of odd length of one long document
        dict(name="portion", path="chunk", rows=1, tokens=2011, heads=16, kv_heads=4, low=60000, high=65000, page=96, window=-1, ragged=False),
        # decode step of a few requests on a small model: latency
        dict(name="step_few", path="adapters", rows=4, tokens=1, channels=768, outputs=768, rank=16, slots=8, none=0.0),
        # decode step of a served batch, every request its own adapter, some without one
        dict(name="step_batch", path="adapters", rows=64, tokens=1, channels=2048, outputs=2048, rank=16, slots=64, none=0.2),
        # the wide product of the feed-forward, a large batch of requests over fewer adapters of higher rank
        dict(name="step_wide", path="adapters", rows=256, tokens=1, channels=2048, outputs=8192, rank=64, slots=48, none=0.0),
        # drafted tokens of a batch
        dict(name="draft_adapters", path="adapters", rows=32, tokens=5, channels=1536, outputs=4608, rank=32, slots=32, none=0.1),
        # portions of prompts of odd length, back to the model's width
        dict(name="portions", path="adapters", rows=6, tokens=1531, channels=6144, outputs=1536, rank=32, slots=16, none=0.0),
        # prompts at a high rank, out to the feed-forward's width
        dict(name="prompts_wide", path="adapters", rows=8, tokens=2048, channels=2048, outputs=8192, rank=64, slots=8, none=0.1),
    ]


def draw(rng):
    def spread(low, high):
        return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    if rng.random() < 0.5:
        heads, kv_heads = rng.choice([(2, 2), (6, 6), (12, 12), (16, 4), (16, 2), (12, 4), (10, 1)])
        rows = spread(1, 64)
        tokens = spread(1, min(2048, max(1, 16384 // rows)))
        high = spread(1, min(65536, max(64, (1 << 20) // (rows * kv_heads)), max(64, (1 << 31) // (rows * tokens * heads))))
        return dict(path="chunk", rows=rows, tokens=tokens, heads=heads, kv_heads=kv_heads, low=rng.choice([0, spread(1, high)]), high=high,
                    page=rng.choice([48, 96, 192, 192, 240, 384]), window=rng.choice([-1, -1, 1024, spread(8, high + tokens)]),
                    ragged=rng.random() < 0.4)
    rows, channels, outputs = spread(1, 256), 8 * spread(32, 1024), 8 * spread(16, 1024)
    most = max(1, min(16384, (1 << 28) // (channels + 2 * outputs)) // rows)
    return dict(path="adapters", rows=rows, tokens=rng.choice([1, spread(1, most)]), channels=channels, outputs=outputs, rank=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                slots=spread(1, 64), none=rng.choice([0.0, 0.2]))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(BF)

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=gen, device="cuda", dtype=torch.int32)

    if case["path"] == "adapters":
        c = case
        state = dict(case=c, x=normal(c["rows"], c["tokens"], c["channels"]), y=normal(c["rows"], c["tokens"], c["outputs"]),
                     down=normal(c["slots"], c["rank"], c["channels"], scale=c["channels"] ** -0.5),
                     up=normal(c["slots"], c["outputs"], c["rank"], scale=0.5 * c["rank"] ** -0.5),
                     scales=torch.rand(c["slots"], generator=gen, device="cuda") + 0.5)
        state["ids"] = torch.randperm(c["rows"], generator=gen, device="cuda").to(torch.int32) % c["slots"]
        state["ids"][torch.rand(c["rows"], generator=gen, device="cuda") < c["none"]] = -1
        return state
    B, T, Hq, Hkv, page = case["rows"], case["tokens"], case["heads"], case["kv_heads"], case["page"]
    lens = whole(case["low"], case["high"], B)
    new = whole(0, T, B) if case["ragged"] else None
    # the tables have room for the longest row; a row's pages lie anywhere in the pool
    width = -(-(case["high"] + T) // page)
    pages = B * width
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(B, width)
    q = torch.randn(B, T, Hq, D, generator=gen, device="cuda")
    q = (q / q.square().mean(-1, keepdim=True).sqrt() * 1.2).to(BF)  # normed and scaled queries and keys, as the append leaves them
    k = torch.randn(pages, page, Hkv, D, generator=gen, device="cuda")
    k = (k / k.square().mean(-1, keepdim=True).sqrt() * 1.2).to(BF)
    return dict(case=case, q=q, k=k, v=normal(pages, page, Hkv, D), table=table, lens=lens, new=new)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        from nanochat_b200 import ops
        if c["path"] == "adapters":
            return ops.add_adapters(state["y"], state["x"], state["down"], state["up"], state["ids"], state["scales"])
        return ops.prefill_attention_paged(state["q"], state["k"], state["v"], state["table"], state["lens"], state["new"], c["window"])
    return _adapters(state) if c["path"] == "adapters" else _chunk(state)


def _adapters(state):
    """Adapter by adapter, over the rows of all its requests."""
    y = state["y"].float()
    ids = state["ids"].tolist()
    for s in sorted(set(ids) - {-1}):
        rows = torch.tensor([b for b, at in enumerate(ids) if at == s], device="cuda")
        low = state["x"][rows].float() @ state["down"][s].float().t()
        y[rows] += state["scales"][s] * (low @ state["up"][s].float().t())
    return y.to(BF)


def _chunk(state):
    """Row by row: its pages' keys and values in order, scores of a part of the queries, softmax, values."""
    c, q = state["case"], state["q"]
    B, T, Hq, _ = q.shape
    Hkv = c["kv_heads"]
    out = torch.zeros_like(q)
    lens = state["lens"].tolist()
    new = state["new"].tolist() if state["new"] is not None else [T] * B
    for b in range(B):
        L, n = lens[b], new[b]
        if n == 0:
            continue
        used = state["table"][b, :-(-(L + n) // c["page"])].long()
        k = state["k"][used].flatten(0, 1)[:L + n].float().permute(1, 2, 0).unsqueeze(1)
        v = state["v"][used].flatten(0, 1)[:L + n].float().transpose(0, 1).unsqueeze(1)
        key = torch.arange(L + n, device="cuda")
        step = max(1, (1 << 28) // (Hq * (L + n)))
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            part = q[b, t0:t1].float().view(t1 - t0, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
            s = (part @ k) * D ** -0.5
            at = torch.arange(L + t0, L + t1, device="cuda")[:, None]
            seen = key <= at
            if c["window"] >= 0:
                seen &= key >= at - c["window"]
            s.masked_fill_(~seen, -math.inf)
            s = (s - s.amax(-1, keepdim=True)).exp_()
            o = (s @ v) / s.sum(-1, keepdim=True)
            out[b, t0:t1] = o.permute(2, 0, 1, 3).reshape(t1 - t0, Hq, D).to(BF)
    return out


def work(case):
    """Each input that counts once and each output once; lengths at their mean."""
    c = case
    if c["path"] == "adapters":
        rows = c["rows"] * c["tokens"] * (1 - c["none"])
        used = min(c["slots"], c["rows"] * (1 - c["none"]))
        moved = rows * (c["channels"] + 2 * c["outputs"]) + 2 * (c["rows"] * c["tokens"] - rows) * c["outputs"]
        return {"bytes": 2 * moved + 2 * used * c["rank"] * (c["channels"] + c["outputs"]), "flops": 2 * rows * c["rank"] * (c["channels"] + c["outputs"])}
    L, n = (c["low"] + c["high"]) / 2, c["tokens"] / 2 if c["ragged"] else c["tokens"]
    keys, seen = L + n, L + (n + 1) / 2  # of a row; by a query of it
    if c["window"] >= 0:
        w = c["window"] + 1
        keys, seen = min(keys, w + n), min(seen, w)
    return {"bytes": c["rows"] * (4 * D * c["kv_heads"] * keys + 2 * D * c["heads"] * (n + c["tokens"])),
            "flops": 4 * D * c["rows"] * n * c["heads"] * seen}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st, f64 = prepare(case, seed), torch.float64
    if case["path"] == "adapters":
        out = []
        for b, s in enumerate(st["ids"].tolist()):
            y = st["y"][b].to(f64)
            if s >= 0:
                y = y + st["scales"][s].to(f64) * torch.einsum("tk,rk,nr->tn", st["x"][b].to(f64), st["down"][s].to(f64), st["up"][s].to(f64))
            out.append(y)
        return torch.stack(out)
    if work(case)["flops"] > 6e12:
        return None
    B, T, Hq, _ = st["q"].shape
    group, page = Hq // case["kv_heads"], case["page"]
    out = torch.zeros(B, T, Hq, D, dtype=f64, device="cuda")
    for b in range(B):
        L = int(st["lens"][b])
        n = T if st["new"] is None else int(st["new"][b])
        at = torch.arange(L, L + n, device="cuda")
        low = torch.clamp(at - case["window"], min=0) if case["window"] >= 0 else torch.zeros_like(at)
        places = torch.arange(L + n, device="cuda")
        where = st["table"][b].long()[places // page] * page + places % page
        for h in range(Hq if n else 0):
            k = st["k"].view(-1, case["kv_heads"], D)[where, h // group].to(f64)
            v = st["v"].view(-1, case["kv_heads"], D)[where, h // group].to(f64)
            for t0 in range(0, n, 512):
                t = slice(t0, min(n, t0 + 512))
                s = st["q"][b, t, h].to(f64) @ k.t() / math.sqrt(D)
                hidden = (places[None] > at[t, None]) | (places[None] < low[t, None])
                p = torch.softmax(torch.where(hidden, -math.inf, s), -1)
                out[b, t, h] = p @ v
    return out
