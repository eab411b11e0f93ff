"""The recurrent layer of test_gpu_recurrent_layer in plain torch operations, token by token, in
the type of its inputs (no test functions here)."""
from __future__ import annotations

import torch

PATHS = ("q", "k", "v", "gate", "beta", "z", "start", "stream")


def shapes(B, T, H, Hk, d, dv, D):
    """name -> shape of the leaves: inputs, then the layer's parameters in its own order."""
    return dict(x=(B, T, D), residual=(B, T, D), state=(B * H, d, dv), qk=(2 * Hk * d, D), v=(H * dv, D), z=(H * dv, D),
                small=(2 * H, D), out=(D, H * dv), norm=(D,), head_norm=(dv,))


def layer(p, unit, freq, H, Hk, cut=()):
    """(y, stream, final state) of the leaves p by name; `cut` names paths (PATHS) that pass no gradient."""
    B, T, _ = p["x"].shape
    d, dv = p["state"].shape[1:]
    through = lambda name, t: t.detach() if name in cut else t
    normed = lambda t, w, eps=1e-6: t * (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w
    stream = p["x"] + p["residual"]
    x = normed(through("stream", stream), p["norm"])
    heads = normed((x @ p["qk"].t()).view(B, T, 2 * Hk, d), unit)
    turn = torch.arange(T, dtype=freq.dtype, device=x.device)[:, None] * freq
    c, s, n = torch.cos(turn)[:, None], torch.sin(turn)[:, None], freq.numel()
    a, b = heads[..., :n], heads[..., n:2 * n]
    heads = torch.cat([a * c - b * s, a * s + b * c, heads[..., 2 * n:]], -1)
    streams = lambda t: t.transpose(1, 2).reshape(-1, T, t.shape[-1])
    q, k = (streams(t).repeat_interleave(H // Hk, 0) for t in (heads[:, :, :Hk], heads[:, :, Hk:]))
    v = streams((x @ p["v"].t()).view(B, T, H, dv))
    gate, beta = (x @ p["small"].t()).view(B, T, 2, H).permute(2, 0, 3, 1).reshape(2, B * H, T).unbind(0)
    a, beta, z = torch.sigmoid(gate + 2.0), torch.sigmoid(beta), (x @ p["z"].t()).view(B, T, H, dv)
    q, k, v, a, beta, z = (through(*t) for t in zip(PATHS, (q, k, v, a, beta, z)))
    S, outs = through("start", p["state"]), []
    for t in range(T):
        S = a[:, t, None, None] * S
        e = v[:, t] - (k[:, t, :, None] * S).sum(1)
        S = S + k[:, t, :, None] * (beta[:, t, None] * e)[:, None]
        outs.append(d ** -0.5 * (q[:, t, :, None] * S).sum(1))
    rows = torch.stack(outs, 1).view(B, H, T, dv).transpose(1, 2)
    rows = normed(rows, p["head_norm"]) * (z * torch.sigmoid(z))
    return rows.flatten(2) @ p["out"].t(), stream, S
