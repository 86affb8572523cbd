"""The 8-bit format and the operators on it in 64 bits, written from their definition."""

from __future__ import annotations

import torch

BLOCK = 128


def hold(x: torch.Tensor, tall: int = 1) -> torch.Tensor:
    """The values (float64) that the 8-bit form of x [rows, cols] stands for, blocks of tall x 128."""
    x = x.double()
    out = torch.empty_like(x)
    for r in range(0, x.size(0), tall if tall > 1 else max(x.size(0), 1)):
        for c in range(0, x.size(1), BLOCK):
            part = x[r : r + tall, c : c + BLOCK] if tall > 1 else x[:, c : c + BLOCK]
            size = torch.where(torch.isfinite(part), part.abs(), torch.zeros_like(part))
            amax = size.max().reshape(1, 1) if tall > 1 else size.max(1, keepdim=True).values
            e = torch.zeros_like(amax)
            some = amax > 0
            guess = torch.floor(torch.log2(torch.where(some, amax, torch.ones_like(amax)))) - 10  # never too large
            for _ in range(4):
                guess = torch.where(amax > 448 * torch.exp2(guess), guess + 1, guess)
            e = torch.where(some, guess.clamp(-127, 127), e)
            y = part / torch.exp2(e)
            place = torch.floor(torch.log2(torch.where(y.abs() >= 2.0**-6, y.abs(), torch.full_like(y, 2.0**-6))))
            place = torch.where(torch.isfinite(y), place, torch.zeros_like(place))
            step = torch.exp2(place - 3)
            held = torch.round(y / step) * step * torch.exp2(e)  # torch.round: halves to even
            held = torch.where(torch.isfinite(part), held, torch.full_like(held, float("nan")))
            if tall > 1:
                out[r : r + tall, c : c + BLOCK] = held
            else:
                out[:, c : c + BLOCK] = held
    return out


def hold_weight(w: torch.Tensor) -> torch.Tensor:
    if w.dim() == 2:
        return hold(w, BLOCK)
    return torch.stack([hold(e, BLOCK) for e in w])


def linear(x, w, d_out):
    """(out, d_x, d_w) of the 8-bit linear map, and for each the same sums of magnitudes."""
    hx, hw, hd, d = hold(x), hold(w, BLOCK), hold(d_out), d_out.double()
    values = (hx @ hw.T, hd @ hw, d.T @ hx)
    sizes = (hx.abs() @ hw.abs().T, hd.abs() @ hw.abs(), d.abs().T @ hx.abs())
    return values, sizes


def grouped(x, w, counts, d_out):
    """The same per expert; rows behind the last expert's give zeros."""
    E, N, K = w.shape
    values = [torch.zeros(x.size(0), N, dtype=torch.float64, device=x.device),
              torch.zeros(x.size(0), K, dtype=torch.float64, device=x.device),
              torch.zeros(E, N, K, dtype=torch.float64, device=x.device)]  # fmt: skip
    sizes = [v.clone() for v in values]
    at = 0
    for e, n in enumerate(counts):
        n = min(n, x.size(0) - at)
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        v, s = linear(x[rows], w[e], d_out[rows])
        for t, u in ((values, v), (sizes, s)):
            t[0][rows], t[1][rows], t[2][e] = u
    return values, sizes


def swiglu(gate, up, d_out):
    g, u, d = gate.double(), up.double(), d_out.double()
    out = u * g * torch.sigmoid(g)
    shape = g.shape
    g, u = hold(gate.reshape(-1, shape[-1])).reshape(shape), hold(up.reshape(-1, shape[-1])).reshape(shape)
    s = torch.sigmoid(g)
    return out, d * u * (s + g * s * (1 - s)), d * g * s


def check_product(got: torch.Tensor, want: torch.Tensor, size: torch.Tensor, terms: int) -> None:
    """One rounding to the type (half a step: eps / 2) and fp32 sums of `terms` products: every addition is off by at
    most 2^-23 of the sum of magnitudes (truncation counted in full).  Besides the bound for each element, the whole
    result is within half a step in the 2-norm, since roundings of random sign stay below their bound."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    off = (got - want).abs()[ok]
    bound = (half * want.abs() + (1 + half) * terms * 2.0**-23 * size + tiny)[ok]
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
    norm = float(want[ok].norm())
    if norm > 0:
        assert float(off.norm()) <= half * norm + tiny * off.numel() ** 0.5
