"""Every tile of 64 keys counts once, however long the row: queries of zero weigh all keys they see alike, and each tile has ones in a (kv head,
channel) of its own, where the output is its share of the keys in sight."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


@pytest.mark.parametrize("B,T,Hq,Hkv,page,lens,window,new", [
    (1, 5, 6, 6, 192, [33000], -1, None),                                        # stretches of one row
    (2, 8, 12, 12, 192, [65000, 40001], -1, None),
    (9, 5, 16, 4, 96, [31000, 7, 20000, 0, 16384, 30011, 64, 63, 500], -1, None),
    (1, 700, 16, 4, 96, [30000], -1, None),                                      # several tiles of queries share keys
    (2, 300, 12, 4, 96, [20000, 5], 5000, None),
    (3, 200, 8, 4, 48, [16000, 9000, 30000], -1, [200, 3, 77]),
    (24, 96, 16, 4, 48, [(211 * i) % 8000 for i in range(24)], 1024, [(5 * i) % 97 for i in range(24)]),  # dealt
    (6, 300, 6, 6, 48, [3000 + i for i in range(6)], -1, None),
    (8, 700, 4, 4, 192, [0] * 8, -1, None),
    (4, 4, 6, 6, 192, [40, 500, 499, 64], -1, None),                             # clusters
    (12, 16, 8, 8, 48, [400] * 12, 63, None),
])
def test_every_tile_counts_once(B, T, Hq, Hkv, page, lens, window, new):
    from nanochat_b200 import ops
    width = -(-(max(lens) + T) // page)
    tiles = -(-width * page // 64)
    groups = -(-tiles // 128)  # kv head h has the tiles from 128 (h % groups) on, a channel each
    assert groups <= Hkv
    at = torch.arange(width * page, device=DEV) // 64
    heads = torch.arange(Hkv, device=DEV) % groups
    v_row = ((at[:, None, None] == heads[None, :, None] * 128 + torch.arange(128, device=DEV)).to(BF)).view(width, page, Hkv, 128)
    n_pages = B * width + 1
    table = torch.randperm(n_pages, generator=torch.Generator().manual_seed(T))[:B * width].view(B, width).to(DEV)
    k, v = (torch.full((n_pages, page, Hkv, 128), float("nan"), device=DEV, dtype=BF) for _ in range(2))
    counts = [T] * B if new is None else new
    for b in range(B):
        k[table[b]] = torch.randn(width, page, Hkv, 128, generator=torch.Generator(device=DEV).manual_seed(b), device=DEV).to(BF)
        v[table[b]] = v_row
        end = lens[b] + counts[b]  # what lies behind the row's tokens may be anything
        for i in range(end // page, width):
            v[table[b, i], max(0, end - i * page):] = float("nan")
            k[table[b, i], max(0, end - i * page):] = float("nan")
    ints = dict(dtype=torch.int32, device=DEV)
    got = ops.prefill_attention_paged(torch.zeros(B, T, Hq, 128, device=DEV, dtype=BF), k, v, table.to(torch.int32), torch.tensor(lens, **ints),
                                      None if new is None else torch.tensor(new, **ints), window)
    assert ops.read_status(DEV) == 0
    tile = (heads[:, None] * 128 + torch.arange(128, device=DEV)).repeat_interleave(Hq // Hkv, 0)[None]  # (1, Hq, 128)
    for b in range(B):
        pos = torch.arange(lens[b], lens[b] + counts[b], device=DEV)[:, None, None]
        low = (pos - window).clamp(min=0) if window >= 0 else torch.zeros_like(pos)
        seen = (torch.minimum(pos + 1, 64 * (tile + 1)) - torch.maximum(low, 64 * tile)).clamp(min=0)
        want = seen.double() / (pos + 1 - low)
        # weights of one and whole sums are exact; a reciprocal, a product and, where parts are joined, nothing else: 2^-8 for the result's rounding
        assert bool(((got[b, :counts[b]].double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -20)).all()), b
        assert not got[b, counts[b]:].any()
