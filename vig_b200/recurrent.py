"""A causal block on the gated recurrence: norm -> one projection to ``[x | gate logits | output gate]`` -> recurrence -> ``h * silu(gate)`` ->
output projection, with the residual stream handed from block to block as in ``GLABlock.forward_deferred``.  ``forward`` trains it and
reads a prefix in; ``step`` serves one token at a time, with 8-bit products once ``quantize`` has been called."""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .modules import RMSNorm


class GatedRecurrence(nn.Module):
    def __init__(self, d_model, d_inner=None, gate_logit_normalizer=16.0, eps=1e-6):
        super().__init__()
        self.d_model, self.d_inner = d_model, d_inner or d_model
        self.gate_logit_normalizer = gate_logit_normalizer
        self.norm = RMSNorm(d_model, eps=eps)
        self.in_proj = nn.Linear(d_model, 3 * self.d_inner, bias=False)
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=False)
        self._in_8bit = None

    def forward(self, hidden, residual=None, state=None, output_final_state=False):
        """``hidden`` ``[B, L, d_model]`` and the residual stream (None: it begins with ``hidden``); ``state``: fp32 ``[B, d_inner]`` of the tokens
        before.  Returns ``(output, residual, final_state)``; differentiable.  A residual stream in fp32 takes 16-bit branches,
        as they come out of a block under ``torch.autocast``."""
        hidden = self._widened(hidden, residual)
        y, residual = ops.add_rmsnorm_train(hidden, self.norm.weight, residual, self.norm.eps)
        x, g, o = self.in_proj(y).chunk(3, -1)
        h, final = ops.gated_recurrence(x, g, state, output_final_state, gate_logit_normalizer=self.gate_logit_normalizer)
        return self.out_proj(h * F.silu(o)), residual, final

    @staticmethod
    def _widened(hidden, residual):
        return hidden.float() if residual is not None and residual.dtype == torch.float32 and hidden.dtype in (torch.bfloat16, torch.float16) else hidden

    @torch.no_grad()
    def quantize(self):
        """From now on ``step`` takes its input projection in 8 bits: e4m3 codes with a scale per output channel, laid out here and again at the first step
        behind a change of the weights (an optimizer's step, ``load_state_dict``, ``to``).  Weights made in inference mode have no version: they want
        another call when they change."""
        if self.d_model % 16 or 3 * self.d_inner % 16:
            raise ValueError(f"8-bit products want widths of whole 16s; got {self.d_model} and {self.d_inner}")
        self._in_8bit = None
        self._codes()
        return self

    def _apply(self, *args, **kwargs):
        # moved or cast: laid out again at the next step, even where the weights come to lie at the old place
        module = super()._apply(*args, **kwargs)
        if self._in_8bit is not None:
            self._in_8bit = (None, *self._in_8bit[1:])
        return module

    def _codes(self):
        """The codes and scales of the weights as they are: kept by their version, as the layouts of ``GatedLinearAttention``."""
        w = self.in_proj.weight
        key = (w.dtype, w.device, w.data_ptr(), None if w.is_inference() else w._version)
        if self._in_8bit is None or self._in_8bit[0] != key:
            w = w.float()
            scale = (w.abs().amax(1) / 448.0).clamp_min(torch.finfo(torch.float32).tiny)
            self._in_8bit = (key, (w / scale[:, None]).to(torch.float8_e4m3fn), scale)
        return self._in_8bit[1:]

    @torch.no_grad()
    def step(self, hidden, residual, state):
        """One token: ``hidden``, ``residual`` ``[B, d_model]`` (``residual`` may be None), ``state`` fp32 ``[B, d_inner]``, updated in place.
        Returns ``(output, residual)``."""
        hidden = self._widened(hidden, residual)
        if self._in_8bit is not None:
            w, w_scale = self._codes()
            q, scale, residual = ops.add_rmsnorm_8bit(hidden, self.norm.weight, residual, self.norm.eps, prenorm=True)
            z = torch._scaled_mm(q, w.t(), scale_a=scale, scale_b=w_scale[None], out_dtype=torch.bfloat16).to(hidden.dtype)
        else:
            y, residual = ops.add_rmsnorm_train(hidden, self.norm.weight, residual, self.norm.eps)
            z = self.in_proj(y)
        x, g, o = z.chunk(3, -1)
        h = ops.gated_recurrence_step(x, g, state, gate_logit_normalizer=self.gate_logit_normalizer)
        return self.out_proj(h * F.silu(o)), residual
