"""Residual feed-forward block behind an aggregation (no counterpart in the reference, whose layers end at
layers/sage.py:131-134):

    s = x + residual;  out = s + down(act(gate(norm(s))) * up(norm(s)))

norm: root mean square with a learned weight; gate, up, down: bias-free Linears.  The norm adds the
residual as it reads x, and gate, up, activation and product are one kernel (functional.rms_norm,
functional.gated_linear).

quantize_() lays the three weights out in 8 bits, one scale a channel, for inference: the norm then
writes 8 bits with a scale a row, and every product is an 8-bit one.  The 8-bit weights are those of the
call's moment: train() and load_state_dict() drop them, and so does the next call after any change of a weight
that torch counts (an optimizer's step, copy_, another Parameter in its place; a write through .data or through
a raw pointer is not counted and needs quantize_() again).  They serve calls in eval mode without gradients;
every other call takes the fp32 weights.  A graph captured while they served reads them where they lay: keep
the weights as they are, and the block in eval mode, for as long as it is replayed.

x and the residual are matrices [rows, channels].  With the fp32 weights they are fp32 too; the 8-bit weights serve
fp32, bf16 and fp16 rows.

A training step of the block can be captured into a graph.  As with any module, no eager output of the same
parameters may be alive then: torch keeps the stream of a parameter's gradient with the first of them, and
a captured backward pass cannot wait for that stream.
"""
import torch

from .. import functional as SF
from .. import ops


class GatedFeedForward(torch.nn.Module):
    def __init__(self, channels: int, hidden_channels: int, activation: str = 'silu', eps: float = 1e-6):
        super().__init__()
        ops._activation(activation)
        self.channels, self.hidden_channels = channels, hidden_channels
        self.activation, self.eps = activation, eps
        self.norm_weight = torch.nn.Parameter(torch.ones(channels))
        self.gate = torch.nn.Linear(channels, hidden_channels, bias=False)
        self.up = torch.nn.Linear(channels, hidden_channels, bias=False)
        self.down = torch.nn.Linear(hidden_channels, channels, bias=False)
        self._eight = None
        self._eight_of = None            # the weights that the 8 bits were made from, and how far torch had counted

    def reset_parameters(self):
        self._eight = self._eight_of = None
        with torch.no_grad():
            self.norm_weight.fill_(1.0)
        for layer in (self.gate, self.up, self.down):
            layer.reset_parameters()

    # ------------------------------------------------------------------ 8-bit weights
    @torch.no_grad()
    def quantize_(self):
        self._eight = tuple(ops.quantize_rows(layer.weight, padded=True) for layer in (self.gate, self.up, self.down))
        self._eight_of = self._weights_now()
        return self

    def _sources(self):
        """What the three weights are made of: the layers' own parameters, or a parametrization's."""
        m = self._modules
        found = []
        for layer in (m["gate"], m["up"], m["down"]):
            found += layer.parameters() if layer._modules else layer._parameters.values()
        return found

    def _weights_now(self):
        return [p if p is None else (p, p.data_ptr(), None if p.is_inference() else p._version) for p in self._sources()]

    def _current(self):
        """The 8-bit weights are there and still those of the weights; if not, they are dropped."""
        if self._eight is None:
            return False
        now = self._sources()
        same = len(now) == len(self._eight_of)
        for p, of in zip(now, self._eight_of):
            if p is not None and of is not None:
                was, at, count = of
                same = same and p is was and (count is None or p._version == count) and p.data_ptr() == at
            elif p is not of:
                same = False
        if not same:
            self._eight = self._eight_of = None
        return same

    def __getstate__(self):              # copies and pickles take the 8-bit weights along where they are current
        self._current()
        return dict(self.__dict__)

    def __setstate__(self, state):
        super().__setstate__(state)
        if self._eight is not None:
            self._eight_of = self._weights_now()

    def dequantize_(self):
        self._eight = self._eight_of = None
        return self

    @property
    def quantized(self):
        return self._current()

    def train(self, mode=True):
        if mode:
            self._eight = self._eight_of = None
        return super().train(mode)

    def _apply(self, fn, *args, **kwargs):      # .to() and the like: the 8-bit copies stay behind
        self._eight = self._eight_of = None
        return super()._apply(fn, *args, **kwargs)

    def _load_from_state_dict(self, *args, **kwargs):
        self._eight = self._eight_of = None
        return super()._load_from_state_dict(*args, **kwargs)

    # ------------------------------------------------------------------ forward
    def forward(self, x, residual=None):
        if not self.training and not torch.is_grad_enabled() and self._current():
            return self._serve(x, residual)
        if x.dtype != torch.float32 or self.down.weight.dtype != torch.float32:
            raise RuntimeError(f"GatedFeedForward: expected fp32 rows and weights, got {x.dtype} and {self.down.weight.dtype} "
                               "(16-bit rows are served by the 8-bit weights, see quantize_)")
        if residual is None:
            y, s = SF.rms_norm(x, self.norm_weight, eps=self.eps), x
        else:
            y, s = SF.rms_norm(x, self.norm_weight, residual, self.eps)
        h = SF.gated_linear(y, self.gate.weight, self.up.weight, self.activation)
        return s + SF.linear_concat(h, self.down.weight)

    def _serve(self, x, residual):
        (gate, gate_scale), (up, up_scale), (down, down_scale) = self._eight
        if x.dim() == 2 and x.stride(1) != 1:
            x = SF._rows(x)
        if residual is not None and residual.dim() == 2 and residual.stride(1) != 1:
            residual = SF._rows(residual)
        y, y_scale, s = ops.rms_norm_int8(x, self.norm_weight, residual, self.eps, padded=True)
        # bf16 between the two products: its rounding is a 128th of the 8-bit step that follows at the row's
        # largest values, and halves the bytes
        h = ops.int8_gated_linear(y, y_scale, gate, gate_scale, up, up_scale, self.activation, torch.bfloat16)
        h, h_scale = ops.quantize_rows(h, padded=True)
        # 16-bit rows: the product is rounded before the sum is.  Its own rounding is a small part of what 8-bit operands
        # leave of it, and an fp32 product costs 8 us of 60 (8192 rows of 256 channels, 1024 hidden)
        return ops.int8_linear(h, h_scale, down, down_scale, out_dtype=s.dtype).add_(s)

    def __repr__(self):
        return f'{self.__class__.__name__}({self.channels}, {self.hidden_channels}, activation={self.activation})'
