"""Rotary positions on gfx950: ``RotarySpec`` (which pairs turn, how fast) and ``apply_rotary``.

Pair ``i`` of a head's first ``dim`` values turns by ``position * f_i`` radians,
``f_i = base ** (-2 i / dim)``: ``(x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin)``.  The pairs are
``(i, i + dim/2)`` (``layout="half"``) or ``(2 i, 2 i + 1)`` (``"interleaved"``); values from ``dim`` on
are left as they are.  Angles are taken in fp64, so far positions lose nothing.

Scalings for contexts longer than a model was trained on (``factor`` times):

* ``{"type": "linear", "factor": s}``: every ``f_i / s``;
* ``{"type": "ntk", "factor": s}``: ``base * s ** (dim / (dim - 2))``, which leaves the fastest pair
  as it is and slows the slowest by ``s``;
* ``{"type": "yarn", "factor": s, "original": n, "beta_fast": 32, "beta_slow": 1, "magnitude": m}``:
  pairs with over ``beta_fast`` turns in ``n`` positions stay, those with under ``beta_slow`` slow
  by ``s``, a linear ramp between; cos and sin are scaled by ``m`` (default ``0.1 ln s + 1``).
"""

from __future__ import annotations

import math

import torch

from . import _native as nat

LAYOUTS = ("half", "interleaved")


class RotarySpec:
    """Frequencies, layout and magnitude of one model's rotary positions.

    Immutable; the fp64 frequencies are laid out on a device once, at the first use there.
    """

    def __init__(self, dim: int, *, base: float = 10000.0, layout: str = "half", scaling: dict | None = None):
        if dim <= 0 or dim % 2:
            raise ValueError("the rotated size must be even and positive")
        if layout not in LAYOUTS:
            raise ValueError(f"rotary layout must be one of {LAYOUTS}")
        if not base > 0 or not math.isfinite(base):
            raise ValueError("the rotary base must be positive and finite")
        self.dim, self.base, self.layout = int(dim), float(base), layout
        self.interleaved = layout == "interleaved"
        self.scaling = dict(scaling) if scaling else None
        self.magnitude = 1.0
        index = torch.arange(dim // 2, dtype=torch.float64)
        self.frequencies = self._frequencies(index)
        self.native = (self.dim, self.interleaved, self.magnitude)  # as the binding takes a spec
        self._on: dict[torch.device, torch.Tensor] = {}

    def _frequencies(self, index: torch.Tensor) -> torch.Tensor:
        plain = self.base ** (-2.0 * index / self.dim)
        if self.scaling is None:
            return plain
        given = dict(self.scaling)
        kind, factor = given.pop("type", None), float(given.pop("factor", 0.0))
        if kind not in ("linear", "ntk", "yarn"):
            raise ValueError("rotary scaling type must be linear, ntk or yarn")
        if not factor >= 1.0 or not math.isfinite(factor):
            raise ValueError("the rotary scaling factor must be at least 1")
        if kind == "yarn":
            original = float(given.pop("original", 0))
            fast, slow = float(given.pop("beta_fast", 32.0)), float(given.pop("beta_slow", 1.0))
            self.magnitude = float(given.pop("magnitude", 0.1 * math.log(factor) + 1.0))
            if not original > 0 or not fast > slow > 0:
                raise ValueError("yarn scaling needs original > 0 and beta_fast > beta_slow > 0")
            if self.base <= 1.0:
                raise ValueError("yarn scaling needs a base above 1")
        if given:
            raise ValueError(f"unknown rotary scaling entries: {sorted(given)}")
        if kind == "linear":
            return plain / factor
        if kind == "ntk":
            if self.dim <= 2:
                raise ValueError("ntk scaling needs a rotated size above 2")
            return (self.base * factor ** (self.dim / (self.dim - 2))) ** (-2.0 * index / self.dim)

        def pair_of(turns: float) -> float:  # the pair that makes so many turns in `original` positions
            return self.dim * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(self.base))

        low, high = max(0, math.floor(pair_of(fast))), min(self.dim - 1, math.ceil(pair_of(slow)))
        ramp = ((index - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return plain / factor * ramp + plain * (1.0 - ramp)

    def on(self, device: torch.device) -> torch.Tensor:
        """The fp64 frequencies on ``device``, laid out there by the first call, which a graph does not
        capture: a program that captures its steps calls this (or a step) before."""
        f = self._on.get(device)
        if f is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("rotary frequencies are not on the device yet: call spec.on(device) before the capture")
            f = self._on[device] = self.frequencies.to(device)
            torch.cuda.current_stream(device).synchronize()  # other streams may read it from now on
        return f


class _Turn(torch.autograd.Function):
    """The turn as autograd sees it: linear in x, with the inverse turn as its gradient."""

    @staticmethod
    def forward(ctx, x, positions, spec, inverse):
        # what a step's plan gave is an inference tensor, which autograd keeps no hold of
        ctx.save_for_backward(positions.clone() if positions.is_inference() else positions)
        ctx.spec, ctx.inverse = spec, inverse
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)  # the binding's own would be an inference tensor
        return nat.fast().rotary(x, positions, spec.on(x.device), spec.dim, spec.interleaved, inverse, spec.magnitude, out)

    @staticmethod
    def backward(ctx, grad):
        (positions,) = ctx.saved_tensors
        return apply_rotary(grad, positions, ctx.spec, inverse=not ctx.inverse), None, None, None


def apply_rotary(
    x: torch.Tensor, positions: torch.Tensor, spec: RotarySpec, *, inverse: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x [tokens, heads, head_dim]`` turned by ``positions [tokens]``, in x's type (products and
    sums in fp32, rounded once).

    ``x`` may be any view whose last dimension is contiguous (a slice of a fused projection).
    ``inverse=True`` turns back, which is also the gradient: with respect to x, of a loss whose
    gradient with respect to the result is given.  Where ``x`` requires a gradient autograd takes it
    so; otherwise the result is an inference tensor, as every operator's here.  ``out`` may be ``x``
    itself; it takes no gradient.
    """
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("rotary output given by out= takes no gradient, and x requires one")
        if not x.is_cuda:
            raise ValueError("QStore HIP operators require tensors on a HIP (cuda) device")
        return _Turn.apply(x, positions, spec, inverse)
    freq = spec.on(x.device) if x.is_cuda else None
    return nat.fast().rotary(x, positions, freq, spec.dim, spec.interleaved, inverse, spec.magnitude, out)
