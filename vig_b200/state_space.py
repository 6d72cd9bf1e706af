"""A causal block on the selective scan: layer norm -> one projection to ``[x | gate]`` -> short causal convolution with SiLU -> a projection of what comes out to
steps and maps -> scan over the states, gated -> output projection, with the residual stream handed from block to block as in ``GatedRecurrence``.
``forward`` trains it and reads a prefix in, ``step`` serves one token at a time."""
import math

import torch
import torch.nn as nn

from . import ops


class SelectiveStateSpace(nn.Module):
    def __init__(self, d_model, d_inner=None, d_state=16, d_conv=4, dt_rank=None, eps=1e-5, dt_min=1e-3, dt_max=0.1):
        super().__init__()
        self.d_model, self.d_inner, self.d_state, self.d_conv = d_model, d_inner or 2 * d_model, d_state, d_conv
        self.dt_rank = dt_rank or max(1, math.ceil(d_model / 16))
        self.norm = nn.LayerNorm(d_model, eps=eps)
        self.in_proj = nn.Linear(d_model, 2 * self.d_inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(self.d_inner, d_conv).uniform_(-1, 1) / math.sqrt(d_conv))
        self.conv_bias = nn.Parameter(torch.zeros(self.d_inner))
        self.x_proj = nn.Linear(self.d_inner, self.dt_rank + 2 * d_state, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, self.d_inner, bias=False)
        # steps between dt_min and dt_max, evenly in their logarithm, rates 1 to d_state: memories of all lengths to begin with (Gu and Dao 2023, with the selective scan)
        step = torch.exp(torch.rand(self.d_inner) * math.log(dt_max / dt_min) + math.log(dt_min))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1, dtype=torch.float32)).repeat(self.d_inner, 1))
        self.D = nn.Parameter(torch.ones(self.d_inner))
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=False)

    @staticmethod
    def _widened(hidden, residual):
        return hidden.float() if residual is not None and residual.dtype == torch.float32 and hidden.dtype in (torch.bfloat16, torch.float16) else hidden

    def _normed(self, hidden, residual):
        return ops.add_layernorm_train(self._widened(hidden, residual), self.norm.weight, self.norm.bias, residual, self.norm.eps)

    def _steps_and_maps(self, x):
        t, B, C = self.x_proj(x).split([self.dt_rank, self.d_state, self.d_state], -1)
        return self.dt_proj(t), -torch.exp(self.A_log.float()), B, C

    def empty_state(self, batch, dtype=None, device=None):
        """The state ahead of the first token, for ``step`` and ``forward``: ``(last tokens of the convolution, states of the scan)``.  The tokens are of ``dtype`` (None: the
        weights'); in fp32 they take 16-bit ones too, as they are under ``torch.autocast``."""
        w = self.in_proj.weight
        return (torch.zeros(batch, self.d_conv - 1, self.d_inner, dtype=dtype or w.dtype, device=device or w.device),
                torch.zeros(batch, self.d_inner, self.d_state, dtype=torch.float32, device=device or w.device))

    def forward(self, hidden, residual=None, state=None, output_final_state=False, lengths=None):
        """``hidden`` ``[B, L, d_model]`` and the residual stream (None: it begins with ``hidden``); ``state``: what an earlier call returned; ``lengths``: int ``[B]``,
        tokens of each sequence that count.  Returns ``(output, residual, final_state)``; differentiable.  A residual stream in fp32 takes 16-bit branches."""
        y, residual = self._normed(hidden, residual)
        x, z = self.in_proj(y).chunk(2, -1)
        window, h = state if state is not None else (None, None)
        # (autocast: tokens in 16 bits, and of `empty_state` a window in the weights' fp32, which goes on as such)
        x, window = ops.causal_conv(self._widened(x, window), self.conv_weight, self.conv_bias, window, output_final_state, activation="silu", lengths=lengths)
        x = x.to(z.dtype)
        dt, A, B, C = self._steps_and_maps(x)
        y, h = ops.selective_scan(x, dt, A, B, C, self.D, z, self.dt_bias, h, output_final_state, lengths=lengths)
        return self.out_proj(y), residual, (window, h) if output_final_state else None

    @torch.no_grad()
    def step(self, hidden, residual, state):
        """One token: ``hidden``, ``residual`` ``[B, d_model]`` (``residual`` may be None); ``state`` is updated in place.  Returns ``(output, residual)``."""
        y, residual = self._normed(hidden, residual)
        x, z = self.in_proj(y).chunk(2, -1)
        x = ops.causal_conv_step(self._widened(x, state[0]), state[0], self.conv_weight, self.conv_bias, activation="silu").to(z.dtype)
        dt, A, B, C = self._steps_and_maps(x)
        y = ops.selective_scan_step(x, dt, A, B, C, state[1], self.D, z, self.dt_bias)
        return self.out_proj(y), residual
