"""Requests with adapters of their own through a whole model: dense and paged caches, prompts, steps and the engine."""
import copy

import pytest
import torch

from nanochat_b200.adapters import PROJECTIONS, AdapterBank
from nanochat_b200.engine import Engine, KVCache, PagedKVCache
from nanochat_b200.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16
LAYERS, VOCAB = 3, 512


def make(slots=2, rank=12, projections=PROJECTIONS):
    torch.manual_seed(0)
    m = GPT(GPTConfig(sequence_len=256, vocab_size=VOCAB, n_layer=LAYERS, n_head=4, n_kv_head=2, n_embd=512)).to(DEV)
    m.init_weights()
    for block in m.transformer.h:
        torch.nn.init.normal_(block.attn.c_proj.weight, std=0.05)
        torch.nn.init.normal_(block.mlp.c_proj.weight, std=0.05)
    torch.nn.init.normal_(m.lm_head.weight, std=0.2)
    m = m.to(BF)
    m.build_rotary()
    bank = AdapterBank(m, slots, rank, projections)
    gen = torch.Generator().manual_seed(1)
    loaded = []
    for s in range(slots):
        tensors = {}
        for i, layer in enumerate(bank.layers):
            for name, (down, up) in layer.items():
                r = 5 + s
                tensors[f"transformer.h.{i}.{name}.down"] = torch.randn(r, down.size(2), generator=gen) * down.size(2) ** -0.5
                tensors[f"transformer.h.{i}.{name}.up"] = torch.randn(up.size(1), r, generator=gen) * 0.03
        bank.load(s, tensors, scale=1.0 + s)
        loaded.append((tensors, 1.0 + s))
    return m, loaded


def merged(m, tensors, scale):
    bank, m.adapters = m.adapters, None
    other = copy.deepcopy(m)
    m.adapters = bank
    with torch.no_grad():
        for name in {k.rsplit(".", 1)[0] for k in tensors}:
            w = other.get_submodule(name).weight
            w.copy_(w.float() + scale * (tensors[name + ".up"].to(DEV).to(BF).float() @ tensors[name + ".down"].to(DEV).to(BF).float()))
    return other


def cache_of(kind, rows, slots=None, tokens=128):
    common = dict(batch_size=rows, num_heads=2, seq_len=192, head_dim=128, num_layers=LAYERS, device=DEV, dtype=BF)
    cache = PagedKVCache(page_tokens=48, **common) if kind == "paged" else KVCache(**common)
    if kind == "paged":
        cache.reserve(tokens)
    if slots is not None:
        cache.adapter_slots = torch.tensor(slots, dtype=torch.int32, device=DEV)
    return cache


@pytest.mark.parametrize("kind", ["dense", "paged"])
def test_rows_run_with_their_own_adapters(kind):
    m, loaded = make()
    ids = torch.randint(0, VOCAB, (3, 50), generator=torch.Generator().manual_seed(2)).to(DEV)
    slots = [1, -1, 0]
    cache = cache_of(kind, 3, slots)
    singles = [merged(m, *loaded[s]) if s >= 0 else m for s in slots]
    alone = [cache_of("dense", 1) for _ in slots]
    for lo, hi in ((0, 40), (40, 41), (41, 45), (45, 46)):
        got = m.forward(ids[:, lo:hi], kv_cache=cache)
        for b in range(3):
            want = singles[b].forward(ids[b:b + 1, lo:hi], kv_cache=alone[b])
            # merged weights are rounded, and three layers of bfloat16 activations
            assert (got[b] - want[0]).abs().max() <= 0.08 * want.abs().max(), (b, lo)
    base = m.forward(ids[:1, :40], kv_cache=cache_of("dense", 1))
    other = m.forward(ids[:1, :40], kv_cache=cache_of("dense", 1, [1]))
    assert (base - other).abs().max() > 0.3 * base.abs().max(), "the adapters of this test do something"


def test_without_adapters_nothing_changes():
    m, _ = make()
    ids = torch.randint(0, VOCAB, (2, 20), generator=torch.Generator().manual_seed(3)).to(DEV)
    for T in (20, 1):
        a = m.forward(ids[:, :T], kv_cache=cache_of("dense", 2))
        b = m.forward(ids[:, :T], kv_cache=cache_of("dense", 2, [-1, -1]))
        assert torch.equal(a, b)


def test_the_eager_trunk_adds_the_same():
    m, _ = make()
    ids = torch.randint(0, VOCAB, (2, 20), generator=torch.Generator().manual_seed(4)).to(DEV)
    got = []
    for fused in (True, False):
        m.fused_glue = fused
        cache = cache_of("dense", 2, [0, 1])
        got.append([m.forward(ids[:, :12], kv_cache=cache), m.forward(ids[:, 12:13], kv_cache=cache)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_bank_of_some_projections():
    m, loaded = make(projections=("attn.c_q", "mlp.c_proj"))
    ids = torch.randint(0, VOCAB, (1, 30), generator=torch.Generator().manual_seed(5)).to(DEV)
    got = m.forward(ids, kv_cache=cache_of("dense", 1, [1]))
    want = merged(m, *loaded[1]).forward(ids, kv_cache=cache_of("dense", 1))
    assert (got - want).abs().max() <= 0.08 * want.abs().max()


class Tokenizer:
    def encode_special(self, s):
        return VOCAB + 1

    def get_bos_token_id(self):
        return VOCAB + 2

    def encode(self, s):
        return [1]

    def decode(self, tokens):
        return ""


@pytest.mark.parametrize("page_tokens", [None, 48])
def test_the_engine_generates_with_an_adapter(page_tokens):
    m, _ = make()
    prompt = torch.randint(0, VOCAB, (25,), generator=torch.Generator().manual_seed(6)).tolist()
    outs = []
    for adapter in (None, 0, 1):
        engine = Engine(m, Tokenizer(), page_tokens=page_tokens)
        eager = Engine(m, Tokenizer(), cuda_graph=False, page_tokens=page_tokens)
        got, _ = engine.generate_batch(prompt, num_samples=2, max_tokens=24, temperature=0.0, adapter=adapter)
        want, _ = eager.generate_batch(prompt, num_samples=2, max_tokens=24, temperature=0.0, adapter=adapter)
        assert got == want and got[0] == got[1] and len(got[0]) == 49
        outs.append(got[0])
    assert outs[0] != outs[1] != outs[2] != outs[0]
    with pytest.raises(ValueError):
        next(engine.generate(prompt, adapter=2))
