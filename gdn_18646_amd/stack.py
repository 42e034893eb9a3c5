"""GDN layers on a residual stream, joined by block norms.

Between two layers the residual stream takes the layer's output (through a norm
of its own, a gate and a scale where the model has them) and the next layer takes
the stream's norm: one kernel, ``rmsnorm.block_norm``, instead of an addition and
two norms.
"""

import torch

from . import compile_kernels

__all__ = ["GDNStack"]


class GDNStack:
    """``layers`` (``GDNLayerCustom``) one after the other:

        h = x;  for each layer: h = h + residual_scale scale_i RMSNorm(layer_i(h); post_gamma_i)
        out = RMSNorm(h; final_gamma)          (h itself without final_gamma)

    post_gammas, scales: a tensor [D] or None for each layer (None: none at all).
    """

    def __init__(self, layers, final_gamma=None, post_gammas=None, scales=None, residual_scale=1.0, exts=None):
        if not layers:
            raise ValueError("a stack needs a layer")
        self.layers = list(layers)
        n = len(self.layers)
        self.post_gammas = list(post_gammas) if post_gammas is not None else [None] * n
        self.scales = list(scales) if scales is not None else [None] * n
        if len(self.post_gammas) != n or len(self.scales) != n:
            raise ValueError(f"{n} layers, {len(self.post_gammas)} post_gammas and {len(self.scales)} scales")
        if any(layer.D != self.layers[0].D for layer in self.layers):
            raise ValueError("the layers differ in D")
        self.final_gamma, self.residual_scale = final_gamma, float(residual_scale)
        self._norm = (exts if exts is not None else compile_kernels())["rmsnorm"]

    def _check_states(self, states):
        if states is not None and len(states) != len(self.layers):
            raise ValueError(f"{len(self.layers)} layers and {len(states)} states")

    def _join(self, i, y, h, gamma, **kw):
        """(h, n) after layer i."""
        h, n, _, _ = self._norm.block_norm(y, residual=h, post_gamma=self.post_gammas[i], gamma=gamma, scale=self.scales[i],
                                           residual_scale=self.residual_scale, eps=1e-6, **kw)  # the layers' own
        return h, n

    @torch.no_grad()
    def forward(self, x, mask=None, return_state=False, states=None, cu_seqlens=None):
        """x [B, T, D] bf16 -> out [B, T, D]; with ``return_state`` also a list of
        the layers' decode states.  The other arguments are the layer's, ``states``
        a state for each layer."""
        self._check_states(states)
        h, xn, new = x.contiguous(), None, []
        for i, layer in enumerate(self.layers):
            y = layer.forward(h if xn is None else None, mask=mask, return_state=return_state,
                              state=None if states is None else states[i], cu_seqlens=cu_seqlens, xn=xn)
            if return_state:
                y, state = y
                new.append(state)
            last = i + 1 == len(self.layers)
            gamma = self.final_gamma if last else self.layers[i + 1].gamma
            h, xn = self._join(i, y, h, gamma, store_h=not last or gamma is None)
        out = h if xn is None else xn
        return (out, new) if return_state else out

    def init_decode_state(self, B, device=None):
        return [layer.init_decode_state(B, device=device) for layer in self.layers]

    @torch.no_grad()
    def decode(self, x, states, inplace=False):
        """One token: x [B, 1, D] -> (out [B, 1, D], states).  The layers' own steps
        norm their inputs, so between them only the residual is joined."""
        if states is None:
            raise ValueError("decode needs a state for each layer")
        self._check_states(states)
        h, n, new = x.contiguous(), None, []
        for i, layer in enumerate(self.layers):
            y, state = layer.decode(h, states[i], inplace=inplace)
            new.append(state)
            last = i + 1 == len(self.layers)
            gamma = self.final_gamma if last else None
            h, n = self._join(i, y, h, gamma, store_h=gamma is None)
        return (h if n is None else n), (states if inplace else new)
