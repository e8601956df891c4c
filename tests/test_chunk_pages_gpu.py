"""Attention of several new tokens per row over a paged cache, against its definition in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def make(B, T, Hq, Hkv, page, lens, seed, new=None, stale=float("nan"), spare=3):
    """Queries, pools whose unused slots hold ``stale``, a table whose pages lie anywhere."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    new = torch.full((B,), T, dtype=torch.int32) if new is None else torch.tensor(new, dtype=torch.int32)
    width = max(1, -(-int((lens.clamp(min=0) + T).max()) // page))
    n_pages = B * width + spare
    table = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))[:B * width].view(B, width).to(torch.int32)
    pools = []
    for _ in range(2):
        pool = torch.full((n_pages, page, Hkv, 128), stale, device=DEV, dtype=BF)
        for b in range(B):
            n = int(lens[b].clamp(min=0) + new[b])
            row = torch.randn(n, Hkv, 128, generator=gen, device=DEV).to(BF)
            for i in range(-(-n // page)):
                part = row[i * page:(i + 1) * page]
                pool[int(table[b, i]), :part.size(0)] = part
        pools.append(pool)
    q = torch.randn(B, T, Hq, 128, generator=gen, device=DEV).to(BF)
    return q, pools[0], pools[1], table.to(DEV), lens.to(DEV), new.to(DEV)


def rows_of(pool, table, b, n):
    page = pool.size(1)
    return torch.cat([pool[int(table[b, i])] for i in range(-(-n // page))])[:n].double() if n else pool.new_zeros(0, pool.size(2), 128).double()


def definition(q, k_pool, v_pool, table, lens, new, window):
    """(output, what a relative error of the weights is multiplied by: their sum over |v|), float64."""
    B, T, Hq, _ = q.shape
    G = Hq // k_pool.size(2)
    out, size = torch.zeros(B, T, Hq, 128, dtype=torch.float64, device=DEV), torch.zeros(B, T, Hq, 128, dtype=torch.float64, device=DEV)
    for b in range(B):
        L, n = int(lens[b]), int(new[b])
        if n <= 0:
            continue
        k, v = rows_of(k_pool, table, b, L + n), rows_of(v_pool, table, b, L + n)
        at, key = torch.arange(L, L + n, device=DEV)[:, None], torch.arange(L + n, device=DEV)[None]
        seen = key <= at
        if window >= 0:
            seen &= key >= at - window
        for h in range(Hq):
            s = (q[b, :n, h].double() @ k[:, h // G].t()) / math.sqrt(128)
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            vh = v[:, h // G]
            clean = torch.where(vh.isfinite(), vh, torch.zeros_like(vh))
            out[b, :n, h], size[b, :n, h] = p @ clean, p @ clean.abs()
            for j, c in (~vh.isfinite()).nonzero().tolist():
                out[b, :n, h, c] += torch.where(seen[:, j], vh[j, c], torch.zeros((), dtype=torch.float64, device=DEV))
    return out, size


def check(got, q, k_pool, v_pool, table, lens, new, window):
    """A weight is rounded to bfloat16 (2^-8 of it), the result again; the rest is float32: scores of up to 2^5 from 128 products
    (2^5 * 2^-24 * 2 in the exponent), the exponential's 2^-22 and sums of up to 2^17 terms stay below 2^-12 of the size."""
    want, size = definition(q, k_pool, v_pool, table, lens, new, window)
    fine = want.isfinite()
    err = (got.double() - want).abs()
    room = 2.0 ** -8 * (size + want.abs()) + 2.0 ** -12 * size
    assert bool((err <= room)[fine].all()), f"{(err / room.clamp(min=1e-30))[fine].max().item():.2f} times the room"
    assert torch.equal(got.double()[~fine].nan_to_num(7e7), want[~fine].nan_to_num(7e7))


CASES = [
    # B, T, Hq, Hkv, page, lens, window, new
    (1, 1, 1, 1, 48, [0], -1, None),
    (3, 1, 6, 6, 48, [0, 47, 640], -1, [1, 1, 0]),
    (4, 4, 12, 12, 192, [0, 63, 64, 1000], -1, None),
    (5, 7, 16, 4, 48, [0, 1, 120, 577, 41], 100, [7, 0, 1, 6, 3]),
    (2, 13, 10, 1, 96, [3000, 17], -1, None),          # 130 query rows: two tiles of 12 tokens
    (2, 3, 21, 7, 144, [500, 333], 0, None),           # a window of the token alone; groups of three
    (1, 2, 128, 1, 48, [700], 64, None),               # one token to a tile
    (3, 200, 16, 4, 240, [0, 300, 1], -1, [200, 199, 2]),
    (2, 130, 4, 4, 48, [0, 5], 63, None),
    (1, 517, 2, 2, 384, [1234], 1024, None),
    (7, 129, 6, 6, 192, [0, 64, 128, 900, 191, 192, 193], -1, None),
    (2, 64, 8, 8, 192, [0, 0], -1, [64, 0]),
    (1, 5, 2, 1, 192, [33000], -1, None),
    (2, 300, 12, 4, 96, [20000, 5], 5000, None),
]


@pytest.mark.parametrize("B,T,Hq,Hkv,page,lens,window,new", CASES)
def test_matches_definition(B, T, Hq, Hkv, page, lens, window, new):
    from nanochat_b200 import ops
    args = make(B, T, Hq, Hkv, page, lens, seed=T + page, new=new)
    q, k, v, table, at, counts = args
    got = ops.prefill_attention_paged(q, k, v, table, at, counts if new is not None else None, window)
    assert ops.read_status(DEV) == 0
    check(got, *args, window)
    for b in range(B):
        assert not got[b, int(counts[b]):].any()
    again = ops.prefill_attention_paged(q, k, v, table, at, counts if new is not None else None, window)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


def test_many_rows_and_uniform_prompts():
    from nanochat_b200 import ops
    args = make(40, 300, 4, 4, 48, [0] * 40, seed=5)  # 480 tiles of like rows
    check(ops.prefill_attention_paged(*args[:5]), *args, -1)
    lens = [(37 * i) % 700 for i in range(300)]
    args = make(300, 3, 8, 2, 48, lens, seed=6, new=[i % 4 for i in range(300)])
    check(ops.prefill_attention_paged(*args), *args, -1)


@pytest.mark.parametrize("B,T,Hq,Hkv,lens,window,counts", [
    (48, 5, 16, 4, [(97 * i) % 1500 for i in range(48)], -1, False),         # equal stretches, several pieces each
    (48, 5, 16, 4, [(97 * i) % 1500 for i in range(48)], 300, True),
    (24, 96, 16, 4, [(211 * i) % 900 for i in range(24)], 128, True),        # dealt row by row
    (6, 300, 6, 6, [1000 + i for i in range(6)], -1, False),                 # dealt in the order of like rows
    (3, 70, 16, 2, [9000, 10, 4000], -1, False),                             # cut, several tiles of queries
    (2, 40, 16, 4, [8100, 8000], -1, False),
    (70, 2, 2, 2, [i for i in range(70)], -1, True),                         # a CTA to a pair
    (12, 16, 8, 8, [400] * 12, 63, False),                                   # clusters of 2
])
def test_all_ways_of_sharing_the_work(B, T, Hq, Hkv, lens, window, counts):
    from nanochat_b200 import ops
    new = [(5 * i + 3) % (T + 1) for i in range(B)] if counts else None
    args = make(B, T, Hq, Hkv, 48, lens, seed=B + T, new=new)
    got = ops.prefill_attention_paged(*args[:5], args[5] if counts else None, window)
    assert ops.read_status(DEV) == 0
    check(got, *args, window)
    again = ops.prefill_attention_paged(*args[:5], args[5] if counts else None, window)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    for b in range(B):
        assert not got[b, int(args[5][b]):].any()


@pytest.mark.parametrize("B,T,Hq,Hkv,L,window", [
    (80, 64, 16, 4, 2600, 2500),   # 640 tiles of like length
    (19, 140, 16, 16, 3000, 1500),  # 608
    (25, 60, 128, 4, 2300, 2200),  # 1500, four tokens each
    (300, 70, 8, 1, 2000, 2500),   # 1500
    (30, 330, 16, 4, 1500, 1400),  # 1320
])
def test_a_short_last_round_of_uneven_rows(B, T, Hq, Hkv, L, window):
    """Tiles of like length that fill the chip's CTAs some times over and a few more, with counts per row; rows share a pool of pages."""
    from nanochat_b200 import ops
    kinds = 5
    lens, new = [L - 64 * i for i in range(kinds)], [T, T, T - 1, T, T - 5]
    q, k, v, table, at, n = make(kinds, T, Hq, Hkv, 96, lens, seed=T, new=new)
    which = torch.arange(B, device=DEV) % kinds
    got = ops.prefill_attention_paged(q[which], k, v, table[which].contiguous(), at[which].contiguous(), n[which].contiguous(), window)
    assert ops.read_status(DEV) == 0
    want, size = definition(q, k, v, table, at, n, window)
    err = (got.double() - want[which]).abs()
    assert bool((err <= (2.0 ** -8 * (size + want.abs()) + 2.0 ** -12 * size)[which]).all())  # check()'s room
    for b in range(B):
        assert not got[b, int(n[b % kinds]):].any()
    again = ops.prefill_attention_paged(q[which], k, v, table[which].contiguous(), at[which].contiguous(), n[which].contiguous(), window)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("T,counts", [(3, True), (40, True), (40, False)])
def test_the_most_rows_of_a_launch(T, counts):
    """4096 rows that share two pages, of 8 lengths and 7 counts, in one launch; one more is refused."""
    from nanochat_b200 import ops
    B = 4096
    lens, new = [9 * (i % 8) for i in range(B)], [6 * (i % 7) * T // 40 if counts else T for i in range(B)]
    q, k, v, table, at, n = make(56, T, 4, 1, 96, lens[:56], seed=T, new=new[:56])
    pages = torch.randn(2, 96, 1, 128, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV).to(BF)
    k, v, table = pages, pages.flip(0).contiguous(), torch.tensor([[1, 0]] * B, dtype=torch.int32, device=DEV)
    kinds = torch.arange(B, device=DEV) % 56
    args = (q, k, v, table[:56], at, n)
    want, size = definition(*args, -1)
    got = ops.prefill_attention_paged(q[kinds], k, v, table, at[kinds].contiguous(), n[kinds].contiguous() if counts else None)
    assert ops.read_status(DEV) == 0
    check(got[:56], *args, -1)
    # every row's error has the room that check() gives
    err = (got.double() - want[kinds]).abs()
    assert bool((err <= (2.0 ** -8 * (size + want.abs()) + 2.0 ** -12 * size)[kinds]).all())
    with pytest.raises(RuntimeError, match="at most 4096"):
        ops.prefill_attention_paged(q[:1].expand(B + 1, -1, -1, -1), k, v, table[:1].expand(B + 1, -1).contiguous(),
                                    torch.zeros(B + 1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_only_who_sees_them(bad):
    from nanochat_b200 import ops
    B, T, Hq, Hkv, page, window = 2, 40, 4, 2, 48, 90
    q, k, v, table, lens, new = args = make(B, T, Hq, Hkv, page, [200, 30], seed=9)

    def at(pool, b, pos):
        return pool[int(table[b, pos // page]), pos % page]
    at(v, 0, 215)[1, 7] = bad      # a new token of the chunk: queries before it don't see it
    at(v, 0, 120)[0, 3] = bad      # leaves the window in the middle of the chunk
    at(v, 0, 20)[0, :] = bad       # before anybody's window
    at(v, 1, 30)[1, 64:] = bad
    check(ops.prefill_attention_paged(q, k, v, table, lens, None, window), *args, window)
    at(k, 0, 239)[:] = bad         # the last token's key: the others' outputs stay
    got = ops.prefill_attention_paged(q, k, v, table, lens, None, window)
    want, size = definition(q, k, v, table, lens, new, window)
    before = (want[0, :39].isfinite())
    assert ((got[0, :39].double() - want[0, :39]).abs() <= 2.0 ** -7 * (size[0, :39] + want[0, :39].abs()))[before].all()
    if not math.isfinite(bad) and math.isnan(bad):
        assert got[0, 39].isnan().all()


def test_rows_that_cannot_be_are_zero_and_flagged():
    from nanochat_b200 import ops
    q, k, v, table, lens, new = make(4, 6, 4, 2, 48, [10, 90, 20, 30], seed=2)
    lens[1] = table.size(1) * 48 - 5  # six tokens don't fit
    got = ops.prefill_attention_paged(q, k, v, table, lens)
    assert ops.read_status(DEV) == 1
    assert not got[1].any()
    lens[1] = 90
    check(got[[0, 2, 3]], q[[0, 2, 3]], k, v, table[[0, 2, 3]], lens[[0, 2, 3]], new[[0, 2, 3]], -1)
    lens[2] = -3
    got = ops.prefill_attention_paged(q, k, v, table, lens)
    assert ops.read_status(DEV) == 4 and not got[2].any() and got[3].any()
    lens[2] = 20
    for n, status in ((7, 1), (-1, 4)):
        new[3] = n
        got = ops.prefill_attention_paged(q, k, v, table, lens, new)
        assert ops.read_status(DEV) == status
        assert bool(got[3].any()) == (n > 0)


def test_a_page_outside_the_pool_reads_as_zeros():
    from nanochat_b200 import ops
    args = make(2, 5, 4, 4, 48, [100, 100], seed=3)
    q, k, v, table, lens, new = args
    zeroed = [p.clone() for p in (k, v)]
    for p in zeroed:
        p[int(table[1, 0])] = 0
    want = ops.prefill_attention_paged(q, *zeroed, table, lens)
    bad = table.clone()
    bad[1, 0] = k.size(0) + 4
    got = ops.prefill_attention_paged(q, k, v, bad, lens)
    assert ops.read_status(DEV) == 8
    assert torch.equal(got, want)
    bad = table.clone()
    bad[:, 0] = -1  # nobody's window reaches it
    assert torch.equal(ops.prefill_attention_paged(q, k, v, bad, lens, None, 20), ops.prefill_attention_paged(q, k, v, table, lens, None, 20))
    assert ops.read_status(DEV) == 0


def test_pools_with_wider_tokens_and_shared_pages():
    from nanochat_b200 import ops
    q, k, v, table, lens, new = make(3, 9, 4, 2, 96, [190, 150, 100], seed=4, stale=0.0)
    table[1, 0] = table[2, 0] = table[0, 0]  # a common prompt
    wide = [torch.full((k.size(0), 96, 5, 128), float("nan"), device=DEV, dtype=BF)[:, :, 1:3] for _ in range(2)]
    for w, p in zip(wide, (k, v)):
        w.copy_(p)
    got = ops.prefill_attention_paged(q, *wide, table, lens)
    assert torch.equal(got, ops.prefill_attention_paged(q, k, v, table, lens))
    check(got, q, k, v, table, lens, new, -1)
    odd = torch.empty(q.numel() + 8, device=DEV, dtype=BF)[8:].view(q.shape).copy_(q)
    strided = torch.empty(3, 9, 6, 128, device=DEV, dtype=BF)[:, :, 1:5].copy_(q)
    for same in (odd, strided):
        assert torch.equal(ops.prefill_attention_paged(same, k, v, table, lens), got)


def test_pools_of_more_than_32_bits():
    from nanochat_b200 import ops
    n_pages = (1 << 32) // (192 * 8 * 128) + 8  # elements pass 2^32
    k, v = (torch.zeros(n_pages, 192, 8, 128, device=DEV, dtype=BF) for _ in range(2))
    small = make(2, 3, 8, 8, 192, [380, 100], seed=8, stale=0.0, spare=0)
    q, ks, vs, table, lens, new = small
    k[-ks.size(0):], v[-ks.size(0):] = ks, vs
    got = ops.prefill_attention_paged(q, k, v, table + (n_pages - ks.size(0)), lens)
    assert torch.equal(got, ops.prefill_attention_paged(q, ks, vs, table, lens))


@pytest.mark.parametrize("T,Hkv", [(3, 2), (150, 1)])
def test_captured_and_replayed_with_other_lengths(T, Hkv):
    from nanochat_b200 import ops
    cases = [make(3, T, 4, Hkv, 48, lens, seed=s, new=new) for s, (lens, new) in
             enumerate([([5, 700, 90], [T, T, 1]), ([640, 0, 300], [0, T, T - 1])])]
    width = max(c[3].size(1) for c in cases)
    pages = max(c[1].size(0) for c in cases)
    hold = [torch.zeros(3, T, 4, 128, device=DEV, dtype=BF), torch.zeros(pages, 48, Hkv, 128, device=DEV, dtype=BF),
            torch.zeros(pages, 48, Hkv, 128, device=DEV, dtype=BF), torch.zeros(3, width, dtype=torch.int32, device=DEV),
            torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.prefill_attention_paged(*hold)
        side.synchronize()
        graphs = []
        for _ in range(2):  # two graphs that lie beside each other
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = ops.prefill_attention_paged(*hold)
            graphs.append((g, out))
    torch.cuda.synchronize()
    for c in cases:
        for h, t in zip(hold, c):
            h.zero_()
            h[tuple(slice(0, n) for n in t.shape)].copy_(t)
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            check(out, *c, -1)


def test_on_a_side_stream_and_in_two_threads():
    import threading
    from nanochat_b200 import ops
    args = [make(4, 5, 8, 2, 48, [900 + i, 20, 300, 0], seed=20 + i) for i in range(2)]
    want = [ops.prefill_attention_paged(*a) for a in args]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(ops.prefill_attention_paged(*args[i]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(y, want[i]) for y in got[i])


def test_refusals():
    from nanochat_b200 import ops
    q, k, v, table, lens, new = make(2, 4, 4, 2, 48, [10, 20], seed=1)
    bad = [dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[:, :, :3]), dict(k_pool=k.float()), dict(v_pool=v[:, :, :1]), dict(k_pool=k[:, :40], v_pool=v[:, :40]),
           dict(block_table=table.long()), dict(block_table=table[:1]), dict(cache_seqlens=lens.long()), dict(cache_seqlens=lens[:1]),
           dict(new_tokens=new.long()), dict(new_tokens=new[:1]), dict(new_tokens=new.cpu()), dict(cache_seqlens=lens.cpu()), dict(q=q.cpu())]
    good = dict(q=q, k_pool=k, v_pool=v, block_table=table, cache_seqlens=lens, new_tokens=new)
    for change in bad:
        with pytest.raises(RuntimeError):
            ops.prefill_attention_paged(**{**good, **change})
    wide = torch.zeros(1, 1, 129, 128, device=DEV, dtype=BF)
    with pytest.raises(RuntimeError, match="at most"):
        ops.prefill_attention_paged(wide, k[:, :, :1], v[:, :, :1], table[:1], lens[:1])
    assert ops.prefill_attention_paged(q[:, :0], k, v, table, lens).shape == (2, 0, 4, 128)
    assert ops.prefill_attention_paged(q[:0], k, v, table[:0], lens[:0]).shape == (0, 4, 4, 128)


def test_append_of_counts():
    from nanochat_b200 import ops
    from nanochat_b200.gpt import precompute_rotary_embeddings
    B, T, Hq, Hkv, page = 5, 6, 8, 2, 48
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(B, T, h, 128, generator=gen, device=DEV).to(BF) for h in (Hq, Hkv, Hkv))
    cos, sin = precompute_rotary_embeddings(4 * page, 128, device=DEV)
    lens = torch.tensor([0, 45, 47, 100, 4 * page - 2], dtype=torch.int32, device=DEV)
    new = torch.tensor([6, 0, 3, 1, 2], dtype=torch.int32, device=DEV)  # the last row is full behind its two
    table = torch.randperm(B * 4, generator=torch.Generator().manual_seed(1)).view(B, 4).to(torch.int32).to(DEV)
    pools = [torch.full((B * 4, page, Hkv, 128), 3.0, device=DEV, dtype=BF) for _ in range(2)]
    got = ops.append_rope_norm_paged(q, k, v, *pools, table, lens, cos, sin, new_tokens=new)
    assert ops.read_status(DEV) == 0
    want = [torch.full_like(p, 3.0) for p in pools]
    for b in range(B):
        n = int(new[b])
        if n:
            one = ops.append_rope_norm_paged(q[b:b + 1, :n], k[b:b + 1, :n], v[b:b + 1, :n], *want, table[b:b + 1], lens[b:b + 1], cos, sin)
            assert torch.equal(got[b, :n], one[0])
        assert not got[b, n:].any()
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    new[0], new[1] = 7, -2
    ops.append_rope_norm_paged(q, k, v, *pools, table, lens, cos, sin, new_tokens=new)
    assert ops.read_status(DEV) == 5


def caches(B, Hkv, layers, capacity, page):
    from nanochat_b200.engine import KVCache, PagedKVCache
    common = dict(batch_size=B, num_heads=Hkv, seq_len=capacity, head_dim=128, num_layers=layers, device=DEV, dtype=BF)
    return KVCache(**common), PagedKVCache(page_tokens=page, **common)


def test_kv_attention_of_chunks_in_pages_matches_dense_rows():
    from nanochat_b200 import ops
    from nanochat_b200.gpt import kv_attention, precompute_rotary_embeddings
    B, Hq, Hkv, page = 3, 8, 4, 48
    dense, paged = caches(B, Hkv, 1, 480, page)
    tables = precompute_rotary_embeddings(480, 128, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    pos = 0
    for T in (100, 3, 1, 64, 1, 7):
        q, k, v = (torch.randn(B, T, h, 128, generator=gen, device=DEV).to(BF) for h in (Hq, Hkv, Hkv))
        paged.reserve(pos + T)
        want = kv_attention(q, k, v, tables, (70, 0), dense, 0)
        got = kv_attention(q, k, v, tables, (70, 0), paged, 0)
        pos += T
        assert paged.cache_seqlens.tolist() == dense.cache_seqlens.tolist() == [pos] * B
        # two roundings of weights and of results apart: 4 * 2^-8 of at most the largest value in sight
        assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * v.float().abs().max()
        for i in range(-(-pos // page)):
            n = min(page, pos - i * page)
            for b in range(B):
                at = int(paged.block_table[b, i])
                assert torch.equal(paged.k_cache[0, at, :n], dense.k_cache[0, b, i * page:i * page + n])
                assert torch.equal(paged.v_cache[0, at, :n], dense.v_cache[0, b, i * page:i * page + n])
    assert ops.read_status(DEV) == 0


def test_kv_attention_of_counts_moves_each_row_by_its_own():
    from nanochat_b200.gpt import kv_attention, precompute_rotary_embeddings
    B, T, Hq, Hkv, page = 3, 20, 4, 2, 48
    _, paged = caches(B, Hkv, 2, 240, page)
    paged.reserve(3 * T)
    tables = precompute_rotary_embeddings(240, 128, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(2)
    tokens = [torch.randn(B, 3 * T, h, 128, generator=gen, device=DEV).to(BF) for h in (Hq, Hkv, Hkv)]
    counts = [torch.tensor(c, dtype=torch.int32, device=DEV) for c in ([20, 0, 7], [1, 20, 13], [0, 3, 20])]
    got = torch.zeros(B, 3 * T, Hq, 128, device=DEV, dtype=BF)
    for new in counts:
        at = paged.cache_seqlens.tolist()
        parts = [torch.stack([t[b, at[b]:at[b] + T] for b in range(B)]) for t in tokens]
        for layer in range(2):
            y = kv_attention(*parts, tables, (-1, 0), paged, layer, new_tokens=new)
        for b, n in enumerate(new.tolist()):
            got[b, at[b]:at[b] + n] = y[b, :n]
    lens = paged.cache_seqlens.tolist()
    assert lens == [21, 23, 40]
    dense, _ = caches(B, Hkv, 1, 240, page)
    want = kv_attention(*tokens, tables, (-1, 0), dense, 0)
    for b in range(B):
        assert (got[b, :lens[b]].float() - want[b, :lens[b]].float()).abs().max() <= 2.0 ** -6 * tokens[2].float().abs().max()
    with pytest.raises(NotImplementedError, match="paged"):
        kv_attention(*(t[:, :T] for t in tokens), tables, (-1, 0), dense, 0, new_tokens=counts[0])


def test_a_model_takes_its_prompt_into_pages():
    from nanochat_b200 import ops
    from nanochat_b200.engine import KVCache, PagedKVCache
    from nanochat_b200.gpt import GPT, GPTConfig
    torch.manual_seed(0)
    cfg = GPTConfig(sequence_len=256, vocab_size=512, n_layer=3, n_head=4, n_kv_head=2, n_embd=512)
    model = GPT(cfg).to(DEV)
    model.init_weights()
    for block in model.transformer.h:
        torch.nn.init.normal_(block.attn.c_proj.weight, std=0.05)
        torch.nn.init.normal_(block.mlp.c_proj.weight, std=0.05)
    model = model.to(BF)
    model.build_rotary()
    ids = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(1)).to(DEV)
    dense, paged = caches(2, 2, 3, 256, 48)
    paged.reserve(152)
    a, b = model.forward(ids, kv_cache=dense), model.forward(ids, kv_cache=paged)
    assert (a - b).abs().max() <= 0.05 * a.abs().max()  # bfloat16 activations over three layers
    for step in range(2):
        token = ids[:, step:step + 1]
        a, b = model.forward(token, kv_cache=dense), model.forward(token, kv_cache=paged)
        assert (a - b).abs().max() <= 0.05 * a.abs().max()
    assert ops.read_status(DEV) == 0 and paged.cache_seqlens.tolist() == [152, 152]
