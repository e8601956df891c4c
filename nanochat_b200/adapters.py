"""Low-rank adapters of a GPT's projections: many of them resident at once, chosen per row of a cache.

    bank = AdapterBank(model, slots=16, rank=32)       # model.adapters = bank
    bank.load(3, tensors, scale=alpha / rank)          # "transformer.h.0.attn.c_q.down" (r, K), "....up" (N, r), ...
    cache.adapter_slots = torch.tensor([3, 0, -1, 3], dtype=torch.int32, device=...)
    model.forward(ids, kv_cache=cache)                 # row b: every projection's product + scale * up (down x) of its slot
    Engine(model, tokenizer).generate(tokens, adapter=3)

A row whose slot is negative, and a cache without slots, run the projections alone.
"""
import torch

from . import ops
from .gpt import gives_its_product_away

PROJECTIONS = ("attn.c_q", "attn.c_k", "attn.c_v", "attn.c_proj", "mlp.c_fc", "mlp.c_proj")
MAX_RANK = 128


class AdapterBank:
    """``slots`` adapters of up to ``rank`` for the given projections of every layer of ``model`` (bfloat16, zero at
    first); becomes ``model.adapters`` and goes to other devices with it."""

    def __init__(self, model, slots, rank, projections=PROJECTIONS):
        if slots <= 0 or not 0 < rank <= MAX_RANK:
            raise ValueError(f"a bank needs slots and a rank of 1 to {MAX_RANK}, got {slots} and {rank}")
        unknown = set(projections) - set(PROJECTIONS)
        if unknown or not projections:
            raise ValueError(f"unknown projections {sorted(unknown)}; known: {', '.join(PROJECTIONS)}")
        self.slots, self.rank, self.projections = slots, rank, tuple(projections)
        device = model.get_device()
        padded = -(-rank // 8) * 8  # the kernels take ranks in eights; the rest stays zero
        self.scales = torch.zeros(slots, dtype=torch.float32, device=device)
        self.layers = []
        for i, block in enumerate(model.transformer.h):
            layer = {}
            for name in self.projections:
                n, k = block.get_submodule(name).weight.shape
                if n % 8 or k % 8:
                    raise ValueError(f"layer {i}: {name} is {n} x {k}; adapters need multiples of 8")
                layer[name] = (torch.zeros(slots, padded, k, dtype=torch.bfloat16, device=device),
                               torch.zeros(slots, n, padded, dtype=torch.bfloat16, device=device))
            self.layers.append(layer)
        model.adapters = self

    def _check_slot(self, slot):
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} is not one of the bank's {self.slots}")

    def load(self, slot, tensors, scale=1.0):
        """Put an adapter into a slot.  ``tensors``: name of a projection + ``.down`` (r, K) and ``.up`` (N, r), r at most the
        bank's rank; projections that are not named get none.  Nothing is changed if a tensor does not fit."""
        self._check_slot(slot)
        known = {f"transformer.h.{i}.{name}" for i in range(len(self.layers)) for name in self.projections}
        named = {key.rsplit(".", 1)[0] for key in tensors}
        if named - known or any(key.rsplit(".", 1)[1] not in ("down", "up") for key in tensors):
            raise ValueError(f"no place in the bank for {sorted(named - known) or sorted(tensors)}")
        for name in named:
            down, up = tensors.get(name + ".down"), tensors.get(name + ".up")
            _, _, i, part = name.split(".", 3)
            mine = self.layers[int(i)][part]
            if down is None or up is None or down.dim() != 2 or up.dim() != 2 or down.size(0) != up.size(1) or not 0 < down.size(0) <= self.rank or \
                    down.size(1) != mine[0].size(2) or up.size(0) != mine[1].size(1):
                raise ValueError(f"{name}: down and up of a rank of at most {self.rank} are needed for {mine[1].size(1)} x {mine[0].size(2)}, got "
                                 f"{down is not None and tuple(down.shape)} and {up is not None and tuple(up.shape)}")
        self.clear(slot)
        with torch.no_grad():
            for name in named:
                down, up = tensors[name + ".down"], tensors[name + ".up"]
                _, _, i, part = name.split(".", 3)
                mine = self.layers[int(i)][part]
                mine[0][slot, :down.size(0)].copy_(down)
                mine[1][slot, :, :up.size(1)].copy_(up)
            self.scales[slot] = float(scale)

    def clear(self, slot):
        """Empty a slot: rows that name it run the projections alone."""
        self._check_slot(slot)
        with torch.no_grad():
            for layer in self.layers:
                for down, up in layer.values():
                    down[slot].zero_()
                    up[slot].zero_()
            self.scales[slot] = 0.0

    def to(self, device):
        """To the device that the model has gone to (of a bank without memory: empty slots)."""
        def move(t):
            return torch.zeros_like(t, device=device) if t.is_meta else t.to(device)
        self.scales = move(self.scales)
        for layer in self.layers:
            for name, pair in layer.items():
                layer[name] = tuple(move(t) for t in pair)
        return self

    def at(self, layer, slots):
        """What a layer does behind each of its products: ``add(name, y, x, module)`` -> y with the rows' adapters added, in place where
        nobody else holds the product y of ``module`` (None: of no module)."""
        mine = self.layers[layer]

        def add(name, y, x, module=None):
            pair = mine.get(name)
            if pair is None:
                return y
            op = ops.add_adapters_ if module is None or gives_its_product_away(module) else ops.add_adapters
            return op(y, x, *pair, slots, self.scales)
        return add
