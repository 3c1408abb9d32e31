"""Rotary position tables: the frequencies a model's configuration names, for :func:`dspark_rocm.ops.rope`.

``frequencies(dims, base, scaling)`` gives fp64 radians a position of each pair of a head's first ``dims``
values, and the factor its rotated values are multiplied with. ``scaling`` is the configuration's
``rope_scaling`` entry (``rope_type`` or ``type`` names the kind):

* none or ``default``: ``base^(-2i / dims)``;
* ``linear``: every frequency divided by ``factor`` (positions interpolated);
* ``llama3``: wavelengths over ``original_max_position_embeddings / low_freq_factor`` divided by ``factor``,
  those under ``... / high_freq_factor`` kept, in between a mean weighted by where the number of turns
  over the original length stands between the two factors;
* ``yarn``: pairs that turn more than ``beta_fast`` (32) times over the original length kept, under
  ``beta_slow`` (1) divided by ``factor``, in between weighted by the pair's index; rotated values times
  ``attention_factor`` (``0.1 ln(factor) + 1``). ``mscale``, ``mscale_all_dim`` and ``truncate`` are refused.

:func:`rotate` is the same rotation in torch ops, for tensors the kernel does not take (CPU, autograd).
"""

from __future__ import annotations

import math

import torch


def _need(scaling: dict, *names: str) -> list[float]:
    missing = [n for n in names if scaling.get(n) is None]
    if missing:
        raise ValueError(f"rope scaling {scaling}: lacks {', '.join(missing)}")
    return [float(scaling[n]) for n in names]


def frequencies(dims: int, base: float, scaling: dict | None = None, *, device=None) -> tuple[torch.Tensor, float]:
    """(fp64 [dims / 2] frequencies on ``device``, factor of the rotated values)."""
    if dims < 2 or dims % 2 or not base > 0:
        raise ValueError(f"rope: dims={dims} (even), base={base} (positive)")
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    scale = 1.0
    kind = "default" if not scaling else scaling.get("rope_type", scaling.get("type", "default"))
    if kind != "default":
        factor, = _need(scaling, "factor")
        if not factor > 0:
            raise ValueError(f"rope scaling {scaling}: factor")
    if kind == "linear":
        f = [v / factor for v in f]
    elif kind == "llama3":
        low, high, length = _need(scaling, "low_freq_factor", "high_freq_factor", "original_max_position_embeddings")
        if not high > low:
            raise ValueError(f"rope scaling {scaling}: high_freq_factor must be over low_freq_factor")
        for i, v in enumerate(f):
            turns = length * v / (2.0 * math.pi)
            kept = min(max((turns - low) / (high - low), 0.0), 1.0)
            f[i] = v * (kept + (1.0 - kept) / factor)
    elif kind == "yarn":
        length, = _need(scaling, "original_max_position_embeddings")
        if scaling.get("mscale") or scaling.get("mscale_all_dim") or not scaling.get("truncate", True):
            raise ValueError(f"rope scaling {scaling}: mscale, mscale_all_dim and truncate are not taken")
        if not (base > 1 and length > 0):
            raise ValueError(f"rope scaling {scaling}: base={base} (over 1), a positive original length")
        given = lambda name, default: float(default if scaling.get(name) is None else scaling[name])
        # the (fractional) pair that makes `turns` turns over the original length
        pair = lambda turns: dims * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        first = max(math.floor(pair(given("beta_fast", 32.0))), 0)
        last = min(math.ceil(pair(given("beta_slow", 1.0))), dims - 1)
        for i, v in enumerate(f):
            slow = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
            f[i] = v * ((1.0 - slow) + slow / factor)
        scale = given("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
    elif kind != "default":
        raise ValueError(f"rope scaling {kind!r} (default, linear, llama3 or yarn)")
    return torch.tensor(f, dtype=torch.float64, device=device), scale


def rotate(x: torch.Tensor, freqs: torch.Tensor, positions, *, interleaved: bool = False, scale: float = 1.0) -> torch.Tensor:
    """:func:`dspark_rocm.ops.rope` of one tensor [B, H, L, D] in torch ops: angles in fp64, the rotation in fp32 (in fp64
    for fp64 tensors, which the kernel does not take)."""
    L, half = x.shape[2], freqs.numel()
    if not isinstance(positions, torch.Tensor):
        positions = torch.arange(int(positions), int(positions) + L, device=x.device)
    ang = positions.expand(x.shape[0], L).to(torch.float64)[:, None, :, None] * freqs.to(x.device)
    ft = torch.float64 if x.dtype is torch.float64 else torch.float32
    c, s = (torch.cos(ang) * scale).to(ft), (torch.sin(ang) * scale).to(ft)
    r, rest = x[..., :2 * half].to(ft), x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * c - b * s, a * s + b * c
    y = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([y.to(x.dtype), rest], dim=-1)
