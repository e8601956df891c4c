"""Chunks of several tokens behind what a cache holds, through GPT.forward: the smear reaches across the border.  Pages go on, dense rows do what the
reference does."""
import pytest
import torch

from nanochat_b200.engine import KVCache, PagedKVCache
from nanochat_b200.gpt import GPT, GPTConfig, rms

from .cpu_backend import oracle_backend

VOCAB = 128


class Pages(KVCache):
    """Dense rows that pass for pages (the stand-in for the kernels takes dense rows)."""

    paged = True


def make(device, dtype, n_embd, heads, kv_heads):
    torch.manual_seed(3)
    m = GPT(GPTConfig(sequence_len=128, vocab_size=VOCAB, n_layer=2, n_head=heads, n_kv_head=kv_heads, n_embd=n_embd), compute_dtype=dtype)
    m.init_weights()
    s = 3 ** 0.5 * n_embd ** -0.5
    for block in m.transformer.h:
        torch.nn.init.uniform_(block.attn.c_proj.weight, -s, s)
        torch.nn.init.uniform_(block.mlp.c_proj.weight, -s, s)
    torch.nn.init.normal_(m.lm_head.weight, std=0.2)
    torch.nn.init.normal_(m.smear_gate.weight, std=0.5)
    m.smear_lambda.data.fill_(0.5)
    m = m.to(device=device, dtype=dtype)
    m.build_rotary()
    return m.eval()


def cache_of(kind, m, rows, **more):
    cfg = m.config
    return kind(batch_size=rows, num_heads=cfg.n_kv_head, seq_len=96, head_dim=cfg.n_embd // cfg.n_head, num_layers=cfg.n_layer, device=m.get_device(),
                dtype=m.compute_dtype, **more)


def in_portions(m, ids, cache, cuts):
    return torch.cat([m.forward(ids[:, lo:hi], kv_cache=cache) for lo, hi in zip((0, *cuts), (*cuts, ids.size(1)))], 1)


@pytest.mark.parametrize("cuts", [(), (16,), (5, 6, 10, 11, 18), (1, 2, 3), (19,)])
def test_portions_are_one_pass(cuts):
    m = make("cpu", torch.float32, 64, 2, 1)
    ids = torch.randint(0, VOCAB, (3, 20), generator=torch.Generator().manual_seed(1))
    with oracle_backend():
        want = m.forward(ids)
        got = in_portions(m, ids, cache_of(Pages, m, 3), cuts)
    # float32 activations through two layers, logits of at most 15
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


def test_refused_drafts_are_taken_back():
    """The lengths and the embedding of the last token that stays."""
    m = make("cpu", torch.float32, 64, 2, 1)
    ids = torch.randint(0, VOCAB, (2, 20), generator=torch.Generator().manual_seed(2))
    drafts = torch.cat([ids[:, 10:12], (ids[:, 12:14] + 1) % VOCAB], 1)  # two that stay, two that don't
    with oracle_backend():
        want = m.forward(ids)
        cache = cache_of(Pages, m, 2)
        m.forward(ids[:, :10], kv_cache=cache)
        m.forward(drafts, kv_cache=cache)
        cache.cache_seqlens.fill_(12)
        cache.prev_embedding = rms(m.transformer.wte(ids[:, 11:12]).to(m.compute_dtype))
        got = m.forward(ids[:, 12:], kv_cache=cache)
    assert (got - want[:, 12:]).abs().max() <= 1e-4 * want.abs().max()


def test_a_row_without_tokens_starts_a_sequence():
    """Whatever the smear state still holds of what was there."""
    m = make("cpu", torch.float32, 64, 2, 1)
    ids = torch.randint(0, VOCAB, (2, 20), generator=torch.Generator().manual_seed(7))
    with oracle_backend():
        want = m.forward(ids)
        cache = cache_of(Pages, m, 2)
        m.forward(torch.cat([ids[:1].flip(1)[:, :8], ids[1:, :8]]), kv_cache=cache)
        cache.cache_seqlens[0] = 0
        cache.prev_embedding = cache.prev_embedding.clone()
        cache.prev_embedding[0] = float("nan")
        got = m.forward(torch.stack([ids[0, :12], ids[1, 8:]]), kv_cache=cache)
    for a, b in ((got[0], want[0, :12]), (got[1], want[1, 8:])):
        assert (a - b).abs().max() <= 1e-4 * want.abs().max()


def test_dense_rows_do_what_the_reference_does():
    m = make("cpu", torch.float32, 64, 2, 1)
    ids = torch.randint(0, VOCAB, (1, 12), generator=torch.Generator().manual_seed(4))
    runs = []
    with oracle_backend():
        for forget in (False, True):
            cache = cache_of(KVCache, m, 1)
            m.forward(ids[:, :8], kv_cache=cache)
            if forget:
                cache.prev_embedding = None
            runs.append(m.forward(ids[:, 8:], kv_cache=cache))
    assert torch.equal(*runs)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [True, False])
def test_portions_into_pages_are_one_pass(fused):
    """bfloat16 activations over two layers leave 0.05 of the largest logit, as between dense rows and pages."""
    from nanochat_b200 import ops
    m = make("cuda", torch.bfloat16, 256, 2, 1)
    m.fused_glue = fused
    ids = torch.randint(0, VOCAB, (2, 60), generator=torch.Generator().manual_seed(5)).cuda()
    want = m.forward(ids, kv_cache=cache_of(KVCache, m, 2))
    for cuts in ((16,), (5, 6, 50), tuple(range(1, 60))):
        cache = cache_of(PagedKVCache, m, 2, page_tokens=48)
        cache.reserve(60)
        got = in_portions(m, ids, cache, cuts)
        assert (got - want).abs().max() <= 0.05 * want.abs().max(), cuts
    assert ops.read_status("cuda") == 0
