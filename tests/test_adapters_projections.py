"""Adapters behind projections whose product somebody else holds: a hook, a module that hands out its input or a tensor of its own."""
import pytest
import torch

from nanochat_b200 import ops
from nanochat_b200.adapters import AdapterBank
from nanochat_b200.gpt import GPT, CastLinear, GPTConfig


class Kept(torch.nn.Module):
    """A projection of the same width that hands out a tensor it goes on holding."""

    def __init__(self, like):
        super().__init__()
        self.weight, self.kept = like.weight, None

    def forward(self, x):
        self.kept = torch.nn.functional.linear(x, self.weight)
        return self.kept


class Sub(CastLinear):
    def forward(self, x):
        self.kept = super().forward(x)
        return self.kept


def run(m, name, change, add):
    """(what others hold of the projection's product, that product, what the layer goes on with)"""
    block = m.transformer.h[0]
    owner, part = name.split(".")
    parent, held = getattr(block, owner), []
    plain = getattr(parent, part)
    hook = None
    if change == "hook":
        hook = plain.register_forward_hook(lambda module, args, out: held.append(out))
    elif change == "global hook":
        hook = torch.nn.modules.module.register_module_forward_hook(lambda module, args, out: held.append(out) if module is plain else None)
    elif change == "own forward":
        kept = Kept(plain)
        plain.forward = kept.forward
    elif change == "subclass":
        new = Sub(plain.in_features, plain.out_features, bias=False)
        new.weight = plain.weight
        setattr(parent, part, new)
    elif change == "module":
        setattr(parent, part, Kept(plain))
    module = getattr(parent, part)
    x = torch.randn(2, 3, plain.in_features)
    try:
        y = module(x)
        held = held[0] if held else kept.kept if change == "own forward" else getattr(module, "kept", None)
        want = torch.nn.functional.linear(x, plain.weight)
        return held, want, add(name, y, x, module), y
    finally:
        if hook is not None:
            hook.remove()
        plain.__dict__.pop("forward", None)
        setattr(parent, part, plain)


@pytest.mark.parametrize("change", ["plain", "hook", "global hook", "own forward", "subclass", "module"])
@pytest.mark.parametrize("name", ["attn.c_q", "mlp.c_proj"])
def test_others_keep_the_product(monkeypatch, name, change):
    monkeypatch.setattr(ops, "add_adapters", lambda y, *a: y + 1)
    monkeypatch.setattr(ops, "add_adapters_", lambda y, *a: y.add_(1))
    m = GPT(GPTConfig(sequence_len=64, vocab_size=64, n_layer=1, n_head=2, n_kv_head=1, n_embd=256))
    m.init_weights()
    with torch.no_grad():
        held, want, got, y = run(m, name, change, AdapterBank(m, 1, 8).at(0, None))
    assert torch.equal(got, want + 1)
    if change == "plain":
        assert got is y  # nobody else has it
    else:
        assert held is not None and torch.equal(held, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("fused", [True, False])
def test_hooks_of_a_model_see_products_alone(T, fused):
    from .test_adapters_model_gpu import cache_of, make
    m, _ = make()
    m.fused_glue = m.fused_qkv = fused
    ids = torch.randint(0, 512, (2, T), generator=torch.Generator().manual_seed(3)).cuda()
    want = m.forward(ids, kv_cache=cache_of("dense", 2, [0, 1]))
    m.fused_qkv = False  # (the stacked product calls no module)
    held, copies = [], []

    def see(module, args, out):
        held.append(out)
        copies.append(out.clone())
    for block in m.transformer.h:
        for name in ("attn.c_q", "attn.c_proj", "mlp.c_fc", "mlp.c_proj"):
            block.get_submodule(name).register_forward_hook(see)
    got = m.forward(ids, kv_cache=cache_of("dense", 2, [0, 1]))
    assert torch.equal(got, want)
    assert len(held) == 12 and all(torch.equal(a, b) for a, b in zip(held, copies))


def test_a_bank_goes_where_its_model_goes():
    m = GPT(GPTConfig(sequence_len=64, vocab_size=64, n_layer=2, n_head=2, n_kv_head=1, n_embd=256))
    bank = AdapterBank(m, 2, 8, projections=("attn.c_q", "mlp.c_proj"))
    down, up = torch.randn(8, 256), torch.randn(256, 8)
    bank.load(1, {"transformer.h.1.attn.c_q.down": down, "transformer.h.1.attn.c_q.up": up}, scale=0.3)
    before = bank.layers[1]["attn.c_q"][0]

    def tensors():
        return [bank.scales, *(t for layer in bank.layers for pair in layer.values() for t in pair)]
    assert m.to(torch.bfloat16) is m and m.float() is m
    assert bank.layers[1]["attn.c_q"][0] is before and bank.scales[1] == torch.tensor(0.3) and bank.scales.dtype == torch.float32  # only the model's type
    m.to("meta")
    assert len(tensors()) == 9 and all(t.is_meta and t.dtype == (torch.float32 if t is bank.scales else torch.bfloat16) for t in tensors())
    m.to_empty(device="cpu")  # nothing is left of it: empty slots
    assert all(t.device.type == "cpu" and not t.any() for t in tensors())
    m.adapters = None
    m.to("meta")
    assert not bank.scales.is_meta


@pytest.mark.gpu
def test_a_model_made_on_the_host_runs_with_its_bank_on_the_gpu():
    from .test_adapters_model_gpu import cache_of
    torch.manual_seed(1)
    m = GPT(GPTConfig(sequence_len=64, vocab_size=512, n_layer=3, n_head=4, n_kv_head=2, n_embd=512))
    m.init_weights()
    torch.nn.init.normal_(m.lm_head.weight, std=0.2)
    torch.nn.init.normal_(m.transformer.h[0].mlp.c_proj.weight, std=0.05)
    bank = AdapterBank(m, 2, 8)
    bank.load(1, {"transformer.h.0.mlp.c_proj.down": torch.randn(4, 2048) * 2048 ** -0.5, "transformer.h.0.mlp.c_proj.up": torch.randn(512, 4)})
    m.compute_dtype = torch.bfloat16
    m = m.to(device="cuda", dtype=torch.bfloat16)
    m.build_rotary()
    ids = torch.arange(12, device="cuda")[None]
    plain, got = (m.forward(ids, kv_cache=cache_of("dense", 1, slots)) for slots in (None, [1]))
    assert not torch.equal(plain, got) and got.isfinite().all()
