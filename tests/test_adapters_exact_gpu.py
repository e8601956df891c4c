"""Adapters on whole numbers, where every sum is exact: t = down x needs its second bfloat16 term, and y takes the large part of the result away.

|x|, |down| <= 8 and K <= 2048 leave |t| below 2^16 by far (24 sqrt(K) is its deviation): a bfloat16 and the rest of it, another one, hold it exactly.
|up| <= 4 and R <= 128 leave every partial sum a whole number below 2^24, exact in float32, and scales are powers of two.  So the result is the
rounding of the exact one, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def whole(gen, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=gen, device=DEV).to(BF)


@pytest.mark.parametrize("B,T,K,N,R,S", [
    (5, 1, 2048, 520, 64, 3), (33, 1, 1536, 1032, 16, 5), (4, 2, 512, 264, 128, 2), (40, 3, 256, 256, 128, 4), (3, 8, 1000, 776, 40, 2), (2, 100, 2048, 392, 64, 2),
    (3, 7, 520, 136, 96, 3), (300, 1, 264, 72, 72, 7),
    # tiles of 128 tokens
    (9, 129, 776, 1160, 128, 3), (5, 256, 2048, 264, 64, 2), (30, 57, 264, 1032, 24, 4), (2, 600, 1000, 520, 80, 1),
])
def test_both_terms_of_t_count(B, T, K, N, R, S):
    from nanochat_b200 import ops
    gen = torch.Generator(device=DEV).manual_seed(R + K)
    x, down, up = whole(gen, 8, B, T, K), whole(gen, 8, S, R, K), whole(gen, 4, S, N, R)
    scales = torch.tensor([1.0, 0.5, -2.0, 4.0, -0.25, 1.0, 2.0][:S], device=DEV)
    slots = torch.arange(B, device=DEV, dtype=torch.int32) % S
    want, one_term, y = (torch.empty(B, T, N, device=DEV, dtype=BF) for _ in range(3))
    for b in range(B):
        s = b % S
        t = x[b].double() @ down[s].double().t()
        assert t.abs().max() < 1 << 16
        more, less = (scales[s].double() * (part @ up[s].double().t()) for part in (t, t.to(BF).double()))
        y[b] = -more.to(BF) + whole(gen, 2, T, N)
        want[b], one_term[b] = ((y[b].double() + part).to(BF) for part in (more, less))
    if K > 500:
        assert not torch.equal(one_term, want), "these inputs tell one term from two"
    assert torch.equal(ops.add_adapters(y, x, down, up, slots, scales), want)
    assert torch.equal(ops.add_adapters_(y.clone(), x, down, up, slots, scales), want)
    assert ops.read_status(DEV) == 0
