"""64-bit restatements of the serving operators (rotary positions, paged cache, the two attentions), for tests only.

Written from the operators' formulas with plain loops over sequences and heads; nothing here is used by
the package.
"""

from __future__ import annotations

import math

import torch


def rotate(x, cs, rotary_dim, interleaved, inverse=False):
    """x [rows, heads, head_dim], cs [rows, rotary_dim / 2, 2]: pairs turned as complex numbers, in float64."""
    y = x.double().clone()
    i = torch.arange(rotary_dim // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    turn = torch.complex(cs[..., 0].double(), (-1.0 if inverse else 1.0) * cs[..., 1].double())[:, None]
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def scale_exponent(x):
    """Least e in [-40, 40] with max|x| <= 448 * 2^e over the finite elements (an int)."""
    finite = x[torch.isfinite(x)].abs()
    top = float(finite.max()) if finite.numel() else 0.0
    e = -40
    while e < 40 and top > 448.0 * 2.0**e:
        e += 1
    return e


def e4m3_values():
    """The non-negative finite values of an e4m3 code, ascending (ordinal = position)."""
    out = [m * 2.0**-9 for m in range(8)]
    for e in range(1, 16):
        out += [(8 + m) * 2.0 ** (e - 10) for m in range(8) if not (e == 15 and m == 7)]
    return torch.tensor(out, dtype=torch.float64)


def e4m3(x):
    """Nearest e4m3 value, ties to the even code, saturating at 448; NaN where x is not finite."""
    grid = e4m3_values()
    a = x.double().abs().clamp(max=448.0)
    a = torch.where(torch.isfinite(x), a, 0.0)
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    pick = torch.where(grid[hi] == a, hi, pick)
    y = grid[pick] * torch.where(x < 0, -1.0, 1.0)
    return torch.where(torch.isfinite(x), y, math.nan)


def attend(q, k, v, visible, scale):
    """One head: q [rows, d], k and v [keys, d], visible bool [rows, keys], all float64.

    Returns the attention (zeros where a row sees nothing), sum_j w_j |v_j|, and the largest
    scale * sum_d |q_d k_d| of a visible key: what the error bounds of the kernels are made of.
    """
    if not visible.any():
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros(len(q), 1, dtype=q.dtype)
    s = (q @ k.T) * scale
    s = s.masked_fill(~visible, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    w = torch.where(visible, w, 0.0)
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0)
    used = visible.any(0)
    vv = torch.where(used[:, None], v, 0.0)
    size = ((q.abs() @ k.abs().T) * scale).masked_fill(~visible, 0.0).amax(-1, keepdim=True)
    return w @ vv, w @ vv.abs(), size


def visible_keys(positions, keys, window, sinks):
    """bool [rows, keys]: key j is seen from position p: j <= p and (no window, p - j < window, or j < sinks)."""
    p, j = positions[:, None], torch.arange(keys)[None, :]
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def stack(state, num_heads, num_layers, x, table=None, rotary_dim=0, interleaved=False, window=0, sinks=0):
    """A causal stack (the reference's block, models.py:727-738, with rotary positions and a window) in float64.

    x [tokens, d_model]: one sequence from position 0. Returns [tokens, d_model].
    """
    n, d = x.shape
    hd = d // num_heads
    par = {k: v.double() for k, v in state.items()}
    norm = torch.nn.functional.layer_norm
    seen = visible_keys(torch.arange(n), n, window, sinks)
    r = x.double()
    for i in range(num_layers):
        p = f"layers.{i}."

        def lin(y, name):
            return y @ par[p + name + ".weight"].T + par[p + name + ".bias"]

        y = norm(r, (d,), par[p + "norm1.weight"], par[p + "norm1.bias"], 1e-5)
        q, k, v = (lin(y, f"attention.{z}_proj").view(n, num_heads, hd) for z in "qkv")
        if table is not None:
            q, k = (rotate(z, table[:n], rotary_dim, interleaved) for z in (q, k))
        ctx = torch.stack([attend(q[:, h], k[:, h], v[:, h], seen, hd**-0.5)[0] for h in range(num_heads)], 1)
        r = r + lin(ctx.reshape(n, d), "attention.out_proj")
        y = norm(r, (d,), par[p + "norm2.weight"], par[p + "norm2.bias"], 1e-5)
        r = r + lin(torch.nn.functional.gelu(lin(y, "ffn_in")), "ffn_out")
    return norm(r, (d,), par["final_norm.weight"], par["final_norm.bias"], 1e-5)
