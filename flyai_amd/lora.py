"""A bank of low-rank adapters for the stage: many requests' adapters of one model, each request naming its own.

``AdapterBank`` holds, for every layer, the matrices of ``n_adapters`` slots at the q, k, v and output projections in the
layout of ``ops.linear_lora`` (q, k and v are three segments of the fused projection, each with an A of its own), as deep as
``max_rank``.  Slots are filled and emptied between steps; ``RaggedStage(..., lora=bank)`` reads them in place."""
import ctypes as C

import torch

from . import _lib
from ._lib import check, lib

PROJECTIONS = ("q", "k", "v", "o")


class AdapterBank:
    def __init__(self, shape, n_layers, n_adapters, max_rank=16, device="cuda"):
        """shape: the stage's GptOssShape.  max_rank is rounded up to a multiple of 16, at most 128."""
        if n_adapters < 1 or n_layers < 1:
            raise ValueError("the bank needs adapters and layers")
        if not 1 <= max_rank <= 128:
            raise ValueError(f"max_rank must be in [1, 128], got {max_rank}")
        self.shape, self.n_layers, self.n_adapters = shape, n_layers, n_adapters
        self.max_rank = R = (max_rank + 15) // 16 * 16
        H, D = shape.hidden, shape.head_dim
        nq, nkv = shape.n_q_heads * D, shape.n_kv_heads * D
        self.segments = (nq, nkv, nkv)
        # projection -> (in features, out features, rows of the fused A before its own, features before its own)
        self._places = {"q": (H, nq, 0, 0), "k": (H, nkv, R, nq), "v": (H, nkv, 2 * R, nq + nkv), "o": (nq, H, 0, 0)}
        zeros = lambda *s: torch.zeros(n_layers, n_adapters, *s, dtype=torch.bfloat16, device=device)
        self.qkv_a, self.qkv_b = zeros(3 * R, H), zeros(sum(self.segments), R)
        self.o_a, self.o_b = zeros(R, nq), zeros(H, R)
        self.scale = torch.zeros(n_adapters, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(n_adapters, dtype=torch.int32, device=device)

    def _slot(self, index):
        if not 0 <= int(index) < self.n_adapters:
            raise ValueError(f"adapter {index} outside [0, {self.n_adapters})")
        return int(index)

    def load(self, index, layers, scale):
        """Fill slot ``index``.  layers: per layer a dict of "q", "k", "v", "o" -> (A [r, in], B [out, r]); a projection
        that is missing stays as it is without the adapter.  r may differ from place to place, up to max_rank; values are
        rounded to bf16; scale is alpha / r.  Nothing changes if anything does not fit.  Call between steps, on the stream that they run on."""
        i = self._slot(index)
        if len(layers) != self.n_layers:
            raise ValueError(f"the adapter has {len(layers)} layers, the bank {self.n_layers}")
        top = 0
        for l, projections in enumerate(layers):
            for name, (a, b) in projections.items():
                if name not in self._places:
                    raise ValueError(f"layer {l}: no projection {name!r} (only {', '.join(PROJECTIONS)})")
                n_in, n_out, _, _ = self._places[name]
                if not all(isinstance(t, torch.Tensor) and t.is_floating_point() and t.dim() == 2 for t in (a, b)):
                    raise ValueError(f"layer {l} {name}: A and B must be floating-point matrices")
                r = a.shape[0]
                if tuple(a.shape) != (r, n_in) or tuple(b.shape) != (n_out, r) or not 1 <= r <= self.max_rank:
                    raise ValueError(f"layer {l} {name}: A {tuple(a.shape)} and B {tuple(b.shape)} are not [r, {n_in}] and "
                                     f"[{n_out}, r] with r in [1, {self.max_rank}]")
                top = max(top, r)
        scale = float(scale)
        self.unload(i)
        for t in (self.qkv_a, self.qkv_b, self.o_a, self.o_b):
            t[:, i].zero_()
        for l, projections in enumerate(layers):
            for name, (a, b) in projections.items():
                _, n_out, row, col = self._places[name]
                ta, tb = (self.o_a, self.o_b) if name == "o" else (self.qkv_a, self.qkv_b)
                # detached: a parameter under training would draw the bank into its graph
                ta[l, i, row:row + a.shape[0]] = a.detach()
                tb[l, i, col:col + n_out, :a.shape[0]] = b.detach()
        self.scale[i] = scale
        self.ranks[i] = top

    def unload(self, index):
        """Empty a slot: sequences that name it have no adapter."""
        self.ranks[self._slot(index)] = 0

    def bind(self, stage):
        """Bind the bank to a stage (its C handle) -> the workspace, to be kept as long as the binding and the steps that use it."""
        size = int(lib().flyai_stage_lora_workspace_bytes(stage, self.max_rank))
        ws = torch.empty(size + 256, dtype=torch.uint8, device=self.scale.device)
        ptr = ws.data_ptr() + (-ws.data_ptr()) % 256
        rows = (_lib.LoraLayer * self.n_layers)(*[_lib.LoraLayer(
            self.qkv_a[l].data_ptr(), self.qkv_b[l].data_ptr(), self.o_a[l].data_ptr(), self.o_b[l].data_ptr())
            for l in range(self.n_layers)])
        desc = _lib.StageLora(self.n_adapters, self.max_rank, self.scale.data_ptr(), self.ranks.data_ptr(), rows, ptr, size)
        check(lib().flyai_stage_set_lora(stage, C.byref(desc)))
        return ws
