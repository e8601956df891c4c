"""The native calls for requests served together against the general Python path: same bits, None where only the general path applies."""
import pytest
import torch

from nanochat_b200 import _lib, ops

from .test_adapters_gpu import make as adapters_state
from .test_chunk_pages_gpu import make as chunk_state

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


class General:
    """Stands in for the native module and takes nothing."""

    set_workspace = staticmethod(_lib.native.set_workspace)

    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture
def general(monkeypatch):
    def run(fn, *args):
        with monkeypatch.context() as m:
            m.setattr(_lib, "native", General())
            return fn(*args)
    return run


@pytest.mark.parametrize("B,T,lens,new", [(3, 4, [5, 700, 90], [4, 0, 1]), (1, 200, [300], None)])
def test_chunks(general, B, T, lens, new):
    ops.workspace(torch.device(DEV), 1, 1, 1)
    q, k, v, table, at, counts = chunk_state(B, T, 8, 2, 48, lens, seed=1, new=new)
    for args in ((q, k, v, table, at, counts if new else None, -1), (q, k[:, :, :], v, table, at, None, 70)):
        native = _lib.native.prefill_attention_paged(*args)
        # (as bits: slots of the pools that no token has been put into hold NaN)
        assert native is not None and torch.equal(native.view(torch.int16), general(ops.prefill_attention_paged, *args).view(torch.int16))
    wide = torch.empty(B, T, 10, 128, device=DEV, dtype=BF)[:, :, :8].copy_(q)
    assert _lib.native.prefill_attention_paged(wide, k, v, table, at, None, -1) is None
    a, b = ops.prefill_attention_paged(wide, k, v, table, at), ops.prefill_attention_paged(q, k, v, table, at)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("T", [1, 5, 260])
def test_adapters(general, T):
    ops.workspace(torch.device(DEV), 1, 1, 1)
    y, x, *rest = args = adapters_state(5, T, 256, 320, 16, 4, seed=T, slots=[0, -1, 3, 3, 2])
    want = general(ops.add_adapters, *args)
    assert torch.equal(_lib.native.add_adapters(*args, False), want)
    wide = torch.full((5, T, 640), 7.0, device=DEV, dtype=BF)
    part = wide[..., 64:384].copy_(y)
    got = _lib.native.add_adapters(part, x, *rest, True)
    assert got.data_ptr() == part.data_ptr() and torch.equal(part, want) and (wide[..., :64] == 7).all() and (wide[..., 384:] == 7).all()
    if T > 1:
        turned = y.transpose(0, 1).contiguous().transpose(0, 1)
        assert _lib.native.add_adapters(turned, x, *rest, False) is None and torch.equal(ops.add_adapters(turned, x, *rest), want)


def test_what_the_library_refuses_is_refused_with_its_words():
    y, x, down, up, slots, scales = adapters_state(2, 1, 64, 64, 8, 2, seed=1)
    wide = torch.zeros(2, 136, 64, device=DEV, dtype=BF), torch.zeros(2, 64, 136, device=DEV, dtype=BF)
    assert _lib.native.add_adapters(y, x, *wide, slots, scales, False) is None
    with pytest.raises(_lib.NckvError, match="at most 128"):
        ops.add_adapters(y, x, *wide, slots, scales)
    q, k, v, table, at, _ = chunk_state(1, 1, 1, 1, 48, [3], seed=1)
    many = torch.zeros(1, 1, 129, 128, device=DEV, dtype=BF)
    assert _lib.native.prefill_attention_paged(many, k, v, table, at, None, -1) is None
    with pytest.raises(_lib.NckvError, match="at most 128"):
        ops.prefill_attention_paged(many, k, v, table, at)
