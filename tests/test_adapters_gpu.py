"""Low-rank adapters of many requests beside a shared product, against the definition in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def make(B, T, K, N, R, S, seed, slots=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x, y = (torch.randn(B, T, c, generator=gen, device=DEV).to(BF) for c in (K, N))
    down = (torch.randn(S, R, K, generator=gen, device=DEV) * K ** -0.5).to(BF)
    up = torch.randn(S, N, R, generator=gen, device=DEV).to(BF)
    scales = torch.rand(S, generator=gen, device=DEV) * 2 - 0.5
    if slots is None:
        slots = torch.randint(-1, S, (B,), generator=gen, device=DEV, dtype=torch.int32)
    else:
        slots = torch.tensor(slots, dtype=torch.int32, device=DEV)
    return y, x, down, up, slots, scales


def check(got, y, x, down, up, slots, scales):
    """The result is rounded once (2^-8 of it).  Sums of at most 8192 float32 products, by 16 or more partial sums: 2^-24 * 512 of the sum of
    their sizes (2^-15); t as two bfloat16 terms 2^-16: 2^-14 of what the sizes of all factors give."""
    for b, s in enumerate(slots.tolist()):
        want, size = y[b].double(), torch.zeros_like(y[b]).double()
        if s >= 0:
            low = x[b].double() @ down[s].double().t()
            want = want + scales[s].double() * (low @ up[s].double().t())
            size = scales[s].double().abs() * ((x[b].double().abs() @ down[s].double().abs().t()) @ up[s].double().abs().t())
        else:
            assert torch.equal(got[b], y[b])
        err = (got[b].double() - want).abs()
        room = 2.0 ** -8 * want.abs() + 2.0 ** -14 * size
        assert bool((err <= room).all()), f"request {b}: {(err / room).max().item():.2f} times the room"


SIZES = [
    # B, T, K, N, R, S
    (1, 1, 8, 8, 8, 1),
    (4, 1, 768, 768, 16, 8),
    (33, 1, 1536, 4608, 32, 5),
    (300, 1, 264, 136, 8, 7),
    (70, 1, 2048, 520, 64, 1),
    (6, 5, 1000, 1288, 24, 3),
    (40, 3, 512, 512, 128, 4),
    (3, 16, 2048, 256, 40, 3),
    (5, 17, 328, 2048, 16, 2),
    (2, 100, 4096, 1536, 64, 4),
    (3, 131, 776, 1160, 128, 2),
    (1, 700, 1536, 392, 8, 1),
    (4, 513, 2048, 2048, 32, 3),
    (2, 1100, 200, 4104, 72, 9),
    # many tokens: tiles of 128
    (3, 400, 776, 1160, 128, 2),
    (30, 57, 264, 1032, 24, 4),
    (9, 129, 8, 8, 8, 3),
    (5, 256, 6144, 72, 16, 5),
    (2, 600, 1000, 2056, 48, 1),
]


@pytest.mark.parametrize("B,T,K,N,R,S", SIZES)
def test_matches_definition(B, T, K, N, R, S):
    from nanochat_b200 import ops
    args = make(B, T, K, N, R, S, seed=K + N)
    keep = [t.clone() for t in args]
    got = ops.add_adapters(*args)
    assert ops.read_status(DEV) == 0
    assert all(torch.equal(a, b) for a, b in zip(args, keep))
    check(got, *args)
    again = ops.add_adapters(*args)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    out = ops.add_adapters_(args[0], *args[1:])
    assert out is args[0] and torch.equal(out, got)


@pytest.mark.parametrize("T", [1, 2, 7, 200, 260])
@pytest.mark.parametrize("slots", [[-1] * 5, [2] * 5, [0, -1, 0, 3, -1], [3, 2, 1, 0, 3]])
def test_who_shares_an_adapter(T, slots):
    from nanochat_b200 import ops
    args = make(5, T, 256, 320, 16, 4, seed=T, slots=slots)
    check(ops.add_adapters(*args), *args)


def test_many_requests_of_one_adapter():
    from nanochat_b200 import ops
    gen = torch.Generator().manual_seed(0)
    slots = torch.where(torch.rand(700, generator=gen) < 0.6, 1, torch.randint(-1, 3, (700,), generator=gen)).tolist()
    for T in (1, 4):
        args = make(700, T, 128, 64, 8, 3, seed=T, slots=slots)
        check(ops.add_adapters(*args), *args)


@pytest.mark.parametrize("B", [33, 250, 256, 257, 600])
@pytest.mark.parametrize("S", [2, 255, 256, 300])
@pytest.mark.parametrize("T", [1, 3])
def test_all_ways_of_counting_requests(B, S, T):
    """Many requests of few slots beside slots of one request, in any order."""
    from nanochat_b200 import ops
    gen = torch.Generator().manual_seed(B + S)
    slots = torch.where(torch.rand(B, generator=gen) < 0.5, torch.randint(-1, 2, (B,), generator=gen), torch.randint(-1, S, (B,), generator=gen)).tolist()
    args = make(B, T, 72, 136, 8, S, seed=B + S, slots=slots)
    got = ops.add_adapters(*args)
    assert ops.read_status(DEV) == 0
    check(got, *args)


def test_a_row_does_not_depend_on_its_batch():
    from nanochat_b200 import ops
    y, x, down, up, slots, scales = make(20, 1, 512, 768, 16, 3, seed=1, slots=[i % 3 for i in range(20)])
    all_ = ops.add_adapters(y, x, down, up, slots, scales)
    x2 = x.clone()
    x2[3] = float("nan")
    x2[4] = float("inf")
    got = ops.add_adapters(y, x2, down, up, slots, scales)
    keep = [i for i in range(20) if i not in (3, 4)]
    assert torch.equal(got[keep], all_[keep]) and got[3].isnan().all() and not got[4].isfinite().any()
    down2, up2 = down.clone(), up.clone()
    down2[1], up2[1] = float("nan"), float("nan")
    got = ops.add_adapters(y, x, down2, up2, slots, scales)
    keep = [i for i in range(20) if i % 3 != 1]
    assert torch.equal(got[keep], all_[keep])


@pytest.mark.parametrize("T", [1, 150, 260])
def test_column_slices(T):
    from nanochat_b200 import ops
    y, x, down, up, slots, scales = args = make(4, T, 256, 384, 16, 3, seed=4, slots=[0, 2, -1, 1])
    want = ops.add_adapters(*args)
    wide = torch.full((4, T, 1024), 7.0, device=DEV, dtype=BF)
    part = wide[..., 256:640]
    part.copy_(y)
    wide_x = torch.full((4, T, 520), float("nan"), device=DEV, dtype=BF)[..., 8:264].copy_(x)
    assert ops.add_adapters_(part, wide_x, down, up, slots, scales) is part
    assert torch.equal(part, want) and (wide[..., :256] == 7).all() and (wide[..., 640:] == 7).all()
    assert torch.equal(ops.add_adapters(y.transpose(0, 1).contiguous().transpose(0, 1), x, down, up, slots, scales), want)
    odd = torch.empty(x.numel() + 4, device=DEV, dtype=BF)[4:].view(x.shape).copy_(x)
    assert torch.equal(ops.add_adapters(y, odd, down, up, slots, scales), want)
    if T > 1:
        with pytest.raises(RuntimeError, match="distance"):
            ops.add_adapters_(y.transpose(0, 1).contiguous().transpose(0, 1), x, down, up, slots, scales)
    rows = ops.add_adapters(y.view(-1, 384), x.view(-1, 256), down, up, slots, scales)
    assert torch.equal(rows.view(want.shape), want)


def test_a_slot_outside_the_bank():
    from nanochat_b200 import ops
    for T in (1, 3, 40, 300, 400):
        y, x, down, up, slots, scales = make(3, T, 64, 64, 8, 2, seed=T, slots=[0, 2, 1])
        got = ops.add_adapters(y, x, down, up, slots, scales)
        assert ops.read_status(DEV) == 16
        slots[1] = -1
        assert torch.equal(got, ops.add_adapters(y, x, down, up, slots, scales)) and torch.equal(got[1], y[1])
        assert ops.read_status(DEV) == 0


def test_refusals():
    from nanochat_b200 import ops
    y, x, down, up, slots, scales = make(3, 2, 64, 48, 8, 2, seed=0)
    good = dict(y=y, x=x, down=down, up=up, slots=slots, scales=scales)
    bad = [dict(y=y.float()), dict(x=x.float()), dict(x=x[:2]), dict(x=x[..., :32]), dict(down=down[:, :4]), dict(up=up[:1]), dict(up=up.transpose(1, 2)),
           dict(slots=slots.long()), dict(slots=slots[:2].repeat(2)), dict(scales=scales.double()), dict(scales=scales[:1]), dict(x=x.cpu()),
           dict(slots=slots.cpu()), dict(x=x[..., :60], down=down[..., :60].contiguous()), dict(y=y[..., :44], up=up[:, :44].contiguous()),
           dict(down=down[:, :4].contiguous(), up=up[..., :4].contiguous()), dict(slots=slots[:0])]
    for change in bad:
        for op in (ops.add_adapters, ops.add_adapters_):
            with pytest.raises(RuntimeError):
                op(**{**good, **change})
    wide = torch.zeros(2, 136, 64, device=DEV, dtype=BF), torch.zeros(2, 48, 136, device=DEV, dtype=BF)
    with pytest.raises(RuntimeError, match="at most 128"):
        ops.add_adapters(y, x, *wide, slots, scales)
    with pytest.raises(RuntimeError, match="backward"):
        ops.add_adapters(y, x.clone().requires_grad_(), down, up, slots, scales)
    assert ops.add_adapters(y[:0], x[:0], down, up, slots[:0], scales).shape == (0, 2, 48)
    assert ops.add_adapters(y[:, :0], x[:, :0], down, up, slots, scales).shape == (3, 0, 48)


@pytest.mark.parametrize("T", [1, 130, 260])
def test_captured_and_replayed_with_other_slots(T):
    from nanochat_b200 import ops
    first, second = make(4, T, 256, 256, 16, 3, seed=1, slots=[0, 1, 1, -1]), make(4, T, 256, 256, 16, 3, seed=2, slots=[2, -1, 0, 0])
    hold = [t.clone() for t in first]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.add_adapters(*hold)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.add_adapters(*hold)
            twice = ops.add_adapters(out, *hold[1:])
    torch.cuda.synchronize()
    for args in (second, first):
        for h, t in zip(hold, args):
            h.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.add_adapters(*args)) and torch.equal(twice, ops.add_adapters(out, *args[1:]))


def test_in_two_threads():
    import threading
    from nanochat_b200 import ops
    args = [make(6, T, 512, 512, 16, 3, seed=T) for T in (1, 200)]
    want = [ops.add_adapters(*a) for a in args]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(ops.add_adapters(*args[i]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(o, want[i]) for o in got[i])


def test_activations_of_more_than_32_bits():
    from nanochat_b200 import ops
    rows, N = 525_000, 8192  # 4.3e9 elements of y
    y = torch.zeros(rows, N, device=DEV, dtype=BF)
    _, x, down, up, _, scales = make(1, 1, 64, N, 8, 1, seed=3)
    xs = x.view(1, 64).repeat(rows, 1)
    ops.add_adapters_(y, xs, down, up, torch.zeros(1, dtype=torch.int32, device=DEV), scales)
    want = ops.add_adapters(torch.zeros(1, N, device=DEV, dtype=BF), x.view(1, 64), down, up, torch.zeros(1, dtype=torch.int32, device=DEV), scales)
    # the form for many rows may add up in another order: both within a rounding of the sum
    assert torch.allclose(y[-1].float(), want[0].float(), rtol=2.0 ** -7, atol=1e-4) and torch.equal(y[-1], y[0]) and torch.equal(y[-1], y[rows // 2])
