"""The operators a model built on the per-bucket op needs next to it, as timed cases.

  op "norm_rope"    race_norm_rope: every head's query and key rows normed (root
                    mean square over the head) and rotated by their positions,
                    from the projection's [B, T, H, d] to the op's streams
                    [B * H, T, d]; one position axis, or several (time, height,
                    width) that share the rotated pairs out between them.
  op "scan"         race_gated_scan: h_t = a_t h_{t-1} + u_t per channel, with
                    a = sigmoid(gate) or exp(gate) and u = x or (1 - a) x, from
                    a carried state; race_gated_scan_carry for single tokens.
  op "cross"        race_cross_fwd: the non-causal op of Tq queries over the Tk
                    keys of another sequence (an encoder's), of which each batch
                    entry has its own number; query heads may share key heads.
  op "cross_query"  race_cross_query: single queries of that op against a kept
                    encoder state [N, S*d + S] (race_cross_state).

A case is a dict of plain values.  `train` asks for the gradients w.r.t. every
differentiable input too.  Sizes are those of this repository's configurations
and tests (heads of 64 and 128 columns, 4 x 16 and 8 x 32 buckets, 12 heads,
577 patches) or generic ones.

With `own` false, run() computes the operators in elementary torch operations,
in 32 bits (angles in 64), rounded once at the end.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

EPS = 1e-6          # of the per-bucket normalization
NORM_EPS = 1e-6     # of the root mean square
LOGIT_SCALE = 4.0   # bucket probabilities: softmax of N(0, 1) * 4
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _race():
    return importlib.import_module("race-attention-kernel_amd")


def _norm_rope(name, B, T, Hq, Hk, d, pairs, dtype, sections="", interleaved=False, train=False):
    c = dict(op="norm_rope", B=B, T=T, Hq=Hq, Hk=Hk, d=d, pairs=pairs, dtype=dtype, sections=sections,
             interleaved=interleaved, train=train)
    return c if name is None else dict(c, name=name)


def _scan(name, N, T, D, dtype, form="sigmoid", complement=True, ragged=False, train=False):
    c = dict(op="scan", N=N, T=T, D=D, dtype=dtype, form=form, complement=complement, ragged=ragged, train=train)
    return c if name is None else dict(c, name=name)


def _cross(name, B, H, Hk, Tq, Tk, L, R, d, dtype, ragged=True, train=False, op="cross"):
    c = dict(op=op, B=B, H=H, Hk=Hk, Tq=Tq, Tk=Tk, L=L, R=R, d=d, dtype=dtype, ragged=ragged, train=train)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # One decode step of a batch of 64: far positions, key heads shared by four query heads.
        _norm_rope("norm_rope_decode_bf16", 64, 1, 32, 8, 128, 64, "bf16"),
        # The prefill of one long prompt at the same heads.
        _norm_rope("norm_rope_prefill_bf16", 1, 16384, 32, 8, 128, 64, "bf16"),
        # A training step on images or clips: three axes, fp32 rows.
        _norm_rope("norm_rope_train_f32_axes", 32, 1024, 12, 12, 64, 32, "f32", sections="8,12,12", train=True),
        # A training step on a ragged patch count; half of each head rotated, neighbours as pairs.
        _norm_rope("norm_rope_train_bf16_T577", 16, 577, 12, 12, 96, 24, "bf16", interleaved=True, train=True),
        # One decode step of a recurrent layer, 128 sequences.
        _scan("scan_decode_bf16", 128, 1, 2048, "bf16"),
        # A long prompt of few channels: the streams and length of the headline configuration.
        _scan("scan_prefill_bf16_T64k", 8, 65536, 64, "bf16"),
        # A training step of a recurrent layer at language-model scale.
        _scan("scan_train_bf16", 8, 4096, 2048, "bf16", train=True),
        # A training step on a padded batch: odd length and width, log gates, plain inputs.
        _scan("scan_train_f32_ragged", 24, 1531, 520, "f32", form="log", complement=False, ragged=True, train=True),
        # One decode step of a decoder: every stream's single query against its encoder state.
        _cross("cross_decode_bf16", 64, 12, 12, 1, 1500, 4, 16, 64, "bf16", op="cross_query"),
        # A prompt against a padded batch of encoder sequences.
        _cross("cross_prefill_bf16", 16, 12, 12, 448, 1500, 4, 16, 64, "bf16"),
        # A training step of a decoder on a padded batch, fp32 tokens.
        _cross("cross_train_f32", 32, 12, 12, 256, 1024, 4, 16, 64, "f32", train=True),
        # The same with many buckets, wide heads and key heads shared by four query heads, bf16.
        _cross("cross_train_bf16_S256", 8, 16, 4, 1024, 4096, 8, 32, 128, "bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the same ranges; the elements in all stay within those of the largest listed case."""
    op = rng.choice(["norm_rope", "norm_rope", "scan", "scan", "cross", "cross", "cross_query"])
    dtype = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.5
    if op == "norm_rope":
        d = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128, 160, 256, 33])
        Hk = rng.choice([1, 2, 4, 5, 8, 12])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        pairs = rng.choice([d // 2, d // 2, d // 4, max(1, d // 8)])
        sections = ""
        if pairs >= 3 and rng.random() < 0.5:
            a = rng.randint(1, pairs - 2)
            b = rng.randint(1, pairs - a - 1)
            sections = "%d,%d,%d" % (a, b, pairs - a - b)
        B = _log_int(rng, 1, 64)
        T = _log_int(rng, 1, (1 << 25) // (B * (Hq + Hk) * d))
        return _norm_rope(None, B, T, Hq, Hk, d, pairs, dtype, sections, rng.random() < 0.5, train)
    if op == "scan":
        N = _log_int(rng, 1, 256)
        D = rng.choice([_log_int(rng, 1, 4096), 8 * _log_int(rng, 1, 512)])
        T = rng.choice([1, 1, _log_int(rng, 2, max(2, min(65536, (1 << 25) // (N * D))))])
        return _scan(None, N, T, D, dtype, rng.choice(["sigmoid", "log"]), rng.random() < 0.5,
                     rng.random() < 0.5, train and T > 1)
    L, R = rng.choice([(4, 16), (4, 16), (2, 8), (3, 16), (8, 16), (8, 32), (1, 7), (3, 10)])
    d = rng.choice([64, 64, 128, 32, 96, 80, 50, 17])
    Hk = rng.choice([1, 2, 4, 12])
    H = Hk * rng.choice([1, 1, 2, 4])
    B = _log_int(rng, 1, 32)
    budget = (1 << 24) // (L * R + d)  # tokens of each side
    if op == "cross_query":
        return _cross(None, B, H, Hk, rng.choice([1, 1, 1, 2, 5]), rng.randint(1, 1024), L, R, d, dtype, False, False, op)
    Tq = _log_int(rng, 1, max(1, min(8192, budget // (B * H))))
    Tk = _log_int(rng, 1, max(1, min(16384, budget // (B * Hk))))
    return _cross(None, B, H, Hk, Tq, Tk, L, R, d, dtype, rng.random() < 0.6, train)


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.

def _inputs(case, seed):
    """The tensors of a case by name, on the GPU, rounded to its dtype."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def whole(lo, hi, shape, dtype=torch.int64):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").to(dtype)

    x = {}
    if op == "norm_rope":
        B, T, Hq, Hk, d, pairs = (case[n] for n in ("B", "T", "Hq", "Hk", "d", "pairs"))
        # Queries, keys and values leave one projection side by side.
        rows = normal(B, T, Hq + 2 * Hk, d).to(dt)
        x["q"], x["k"] = rows[:, :, :Hq], rows[:, :, Hq:Hq + Hk]
        x["q_weight"] = (1 + 0.1 * normal(d)).to(dt)
        x["k_weight"] = (1 + 0.1 * normal(d)).to(dt)
        theta = torch.tensor(10000.0 if T > 1 else 1e6, dtype=torch.float64, device="cuda")
        x["inv_freq"] = (theta ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)).float()
        # Token t of sequence b sits at start[b] + t: far into a long text when decoding.
        t = torch.arange(T, device="cuda")
        start = whole(0, (1 << 20) if T == 1 else 4096, (B, 1))
        if case["sections"]:
            width = max(1, int(math.isqrt(T)) // 2)  # frames of width x width
            frame = width * width
            x["positions"] = torch.stack([start + t // frame, (t % frame // width).expand(B, T),
                                          (t % width).expand(B, T)]).contiguous()
        else:
            x["positions"] = (start + t).contiguous()
        if case["train"]:
            x["dq"], x["dk"] = normal(B * Hq, T, d).to(dt), normal(B * Hk, T, d).to(dt)
    elif op == "scan":
        N, T, D = (case[n] for n in ("N", "T", "D"))
        x["x"] = normal(N, T, D).to(dt)
        gate = 1.5 * normal(N, T, D) + 3.0
        x["gate"] = (gate if case["form"] == "sigmoid" else torch.nn.functional.logsigmoid(gate)).to(dt)
        x["state"] = normal(N, D)
        if case["ragged"]:
            x["lengths"] = whole((T + 1) // 2, T, (N,), torch.int32)
        if case["train"]:
            x["dout"], x["dfinal"] = normal(N, T, D).to(dt), normal(N, D)
    else:
        B, H, Hk, Tq, Tk, L, R, d = (case[n] for n in ("B", "H", "Hk", "Tq", "Tk", "L", "R", "d"))

        def probs(N, T):
            return torch.softmax(normal(N, T, L, R) * LOGIT_SCALE, dim=-1).to(dt)

        x["q"] = probs(B * H, Tq)
        k, v = probs(B * Hk, Tk), normal(B * Hk, Tk, d).to(dt)
        if op == "cross_query":
            kf = k.float().flatten(2)
            sums = torch.matmul(kf.transpose(1, 2).contiguous(), v.float())
            x["state"] = torch.cat([sums.flatten(1), kf.sum(1)], dim=1).contiguous()
        else:
            x["k"], x["v"] = k, v
            if case["ragged"]:
                x["lengths"] = whole((Tk + 1) // 2, Tk, (B,), torch.int32)
                if B >= 4:
                    x["lengths"][1] = 0  # a slot of the batch that holds no sequence
            if case["train"]:
                x["dout"] = normal(B * H, Tq, d).to(dt)
    return x


def _sections(case):
    return tuple(int(n) for n in case["sections"].split(",")) if case["sections"] else None


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["train"]:
        leaves = {"norm_rope": ("q", "k", "q_weight", "k_weight"), "scan": ("x", "gate", "state"),
                  "cross": ("q", "k", "v")}[case["op"]]
        for n in leaves:
            x[n].requires_grad_(True)
        x["leaves"] = [x[n] for n in leaves]
    x["case"] = case
    return x


# ---------------------------------------------------------------------------
# One pass.

def run(x):
    if own:
        return _run_own(x)
    case = x["case"]
    with torch.no_grad():  # the gradients come from their formulas
        return {"norm_rope": _plain_norm_rope, "scan": _plain_scan, "cross": _plain_cross,
                "cross_query": _plain_cross_query}[case["op"]](case, x)


def _run_own(x):
    race, case = _race(), x["case"]
    op = case["op"]
    if op == "cross_query":
        return race.race_cross_query(x["q"], x["state"])
    if op == "norm_rope":
        outs = race.race_norm_rope(x["q"], x["k"], x["positions"], x["inv_freq"], q_weight=x["q_weight"],
                                   k_weight=x["k_weight"], eps=NORM_EPS, sections=_sections(case),
                                   interleaved=case["interleaved"])
        grads = (x["dq"], x["dk"]) if case["train"] else None
    elif op == "scan":
        step = race.race_gated_scan_carry if case["T"] == 1 else race.race_gated_scan
        outs = step(x["x"], x["gate"], x["state"], gate_form=case["form"], complement=case["complement"],
                    lengths=x.get("lengths"))
        grads = (x["dout"], x["dfinal"]) if case["train"] else None
    else:
        outs = (race.race_cross_fwd(x["q"], x["k"], x["v"], x.get("lengths")),)
        grads = (x["dout"],) if case["train"] else None
    if grads is None:
        return outs
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, x["leaves"], grads))


# ---------------------------------------------------------------------------
# The plain forms.

def _angles(x, case):
    """cos and sin [B, T, 1, pairs] of position times frequency: the products in 64 bits, a far
    position's angle has no digits left in 32."""
    pos, sections = x["positions"], _sections(case)
    if sections is None:
        per_pair = pos.double()[..., None]
    else:
        per_pair = torch.cat([pos[i].double()[..., None].expand(*pos[i].shape, n) for i, n in enumerate(sections)], -1)
    angle = per_pair * x["inv_freq"].double()
    return torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]


def _rotate(y, cos, sin, pairs, interleaved):
    if interleaved:
        a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, y[..., 2 * pairs:]], dim=-1)


def _to_streams(y):
    B, T, H, d = y.shape
    return y.permute(0, 2, 1, 3).reshape(B * H, T, d)


def _plain_norm_rope(case, x):
    cos, sin = _angles(x, case)
    pairs, interleaved, B = case["pairs"], case["interleaved"], case["B"]
    outs, dx, dw = [], [], []
    for n in ("q", "k"):
        rows, w = x[n].float(), x[n + "_weight"].float()
        scale = torch.rsqrt(rows.pow(2).mean(-1, keepdim=True) + NORM_EPS)
        unit = rows * scale
        outs.append(_to_streams(_rotate(unit * w, cos, sin, pairs, interleaved)).to(x[n].dtype))
        if case["train"]:
            H = rows.shape[2]
            up = x["d" + n].float().view(B, H, -1, case["d"]).permute(0, 2, 1, 3)
            up = _rotate(up, cos, -sin, pairs, interleaved)
            dw.append((up * unit).sum((0, 1, 2)).to(x[n + "_weight"].dtype))
            up = up * w
            dx.append((scale * (up - unit * (up * unit).mean(-1, keepdim=True))).to(x[n].dtype))
    return (*outs, *dx, *dw)


def _linear_scan(a, u):
    """h_t = a_t h_{t-1} + u_t over dim 1 by doubling: each step joins runs of twice the length."""
    a, u, T, s = a.clone(), u.clone(), u.shape[1], 1
    while s < T:
        u[:, s:] = u[:, s:] + a[:, s:] * u[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return u


def _plain_scan(case, x):
    dt, T = x["x"].dtype, case["T"]
    xs, gate = x["x"].float(), x["gate"].float()
    if case["form"] == "sigmoid":
        a, b, slope = torch.sigmoid(gate), torch.sigmoid(-gate), torch.sigmoid(-gate)  # slope: d log a / d gate
    else:
        a, b, slope = torch.exp(gate), -torch.expm1(gate), torch.ones_like(gate)
    if not case["complement"]:
        b = torch.ones_like(b)
    keep = None
    if "lengths" in x:
        keep = (torch.arange(T, device=xs.device) < x["lengths"][:, None])[..., None]
        a = torch.where(keep, a, 1.0)
        b = torch.where(keep, b, 0.0)
    u = torch.where(keep, b * xs, 0.0) if keep is not None else b * xs
    u[:, 0] += a[:, 0] * x["state"]
    h = _linear_scan(a, u)
    out, final = h if keep is None else torch.where(keep, h, 0.0), h[:, -1].contiguous()
    if not case["train"]:
        return out.to(dt), final
    # Not the input's own storage: the final state's gradient is added in place.
    up = torch.where(keep, x["dout"].float(), 0.0) if keep is not None else x["dout"].to(torch.float32, copy=True)
    up[:, -1] += x["dfinal"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    lam = _linear_scan(after.flip(1), up.flip(1)).flip(1)
    before = torch.cat([x["state"][:, None], h[:, :-1]], dim=1)
    dgate = lam * slope * a * (before - xs if case["complement"] else before)
    dx = lam * b
    if keep is not None:
        dgate, dx = torch.where(keep, dgate, 0.0), torch.where(keep, dx, 0.0)
    return out.to(dt), final, dx.to(dt), dgate.to(dt), a[:, 0] * lam[:, 0]


def _keys(case, x, dtype):
    """K [N, Tk, S] and V [N, Tk, d], zero past each sequence's end, and what tells."""
    k, v = x["k"].to(dtype).flatten(2), x["v"].to(dtype)
    if "lengths" not in x:
        return k, v, None
    n = x["lengths"].repeat_interleave(case["Hk"])
    keep = (torch.arange(case["Tk"], device=k.device) < n[:, None])[..., None]
    return torch.where(keep, k, 0.0), torch.where(keep, v, 0.0), keep


def _t(m):
    return m.transpose(1, 2).contiguous()


def _plain_cross(case, x):
    S, d, dt = case["L"] * case["R"], case["d"], x["q"].dtype
    k, v, keep = _keys(case, x, torch.float32)
    q = x["q"].float().reshape(k.shape[0], -1, S)  # the query heads of a key head one after another
    mass = k.sum(1) + EPS
    E = torch.matmul(_t(k), v) / mass[..., None]
    out = torch.matmul(q, E).reshape(x["q"].shape[0], -1, d).to(dt)
    if not case["train"]:
        return (out,)
    g = x["dout"].float().reshape(k.shape[0], -1, d)
    dq = torch.matmul(g, _t(E))
    dE = torch.matmul(_t(q), g)
    dB = dE / mass[..., None]
    dA = -(dE * E).sum(-1) / mass
    dk = torch.matmul(v, _t(dB)) + dA[:, None]
    dv = torch.matmul(k, dB)
    if keep is not None:
        dk, dv = torch.where(keep, dk, 0.0), torch.where(keep, dv, 0.0)
    return out, dq.reshape(x["q"].shape).to(dt), dk.reshape(x["k"].shape).to(dt), dv.to(dt)


def _plain_cross_query(case, x):
    S, d = case["L"] * case["R"], case["d"]
    n = x["state"].shape[0]
    B, A = x["state"][:, :S * d].reshape(n, S, d), x["state"][:, S * d:]
    q = x["q"].float().reshape(n, -1, S)
    return torch.matmul(q / (A[:, None] + EPS), B).reshape(x["q"].shape[0], -1, d).to(x["q"].dtype)


# ---------------------------------------------------------------------------

def work(case):
    """Each input read once and each output written once.  Scans and norms: a multiply-add counts
    two, a root, an exponential or a division one.  Padded batches hold three quarters of their rows."""
    es, op, train = (4 if case["dtype"] == "f32" else 2), case["op"], case["train"]
    if op == "norm_rope":
        B, T, d, H = case["B"], case["T"], case["d"], case["Hq"] + case["Hk"]
        rows = B * T * H * d
        axes = len(_sections(case) or (1,))
        return {"bytes": rows * es * (4 if train else 2) + 8 * axes * B * T + 4 * case["pairs"] + 2 * d * es * (2 if train else 1),
                "flops": rows * (20 if train else 7)}
    if op == "scan":
        n = case["N"] * case["T"] * case["D"]
        part = 0.75 if case["ragged"] and case["T"] > 1 else 1.0
        read, written = (3, 3) if train else (2, 1)
        return {"bytes": int(n * es * (read * part + written)) + 4 * case["N"] * case["D"] * (4 if train else 2),
                "flops": int(n * part * (18 if train else 6))}
    S, d = case["L"] * case["R"], case["d"]
    tq, tk = case["B"] * case["H"] * case["Tq"], case["B"] * case["Hk"] * case["Tk"]
    if op == "cross_query":
        return {"bytes": 4 * case["B"] * case["Hk"] * (S * d + S) + tq * es * (S + d), "flops": 2 * tq * S * d}
    part = 0.75 if case["ragged"] else 1.0
    if train:
        bytes_ = tq * es * 2 * (S + d) + tk * es * (S + d) * (part + 1)
    else:
        bytes_ = tq * es * (S + d) + tk * es * (S + d) * part
    return {"bytes": int(bytes_), "flops": int(2 * S * d * (tq + part * tk) * (3 if train else 1))}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.

def exact(case, seed):
    return {"norm_rope": _exact_norm_rope, "scan": _exact_scan, "cross": _exact_cross,
            "cross_query": _exact_cross}[case["op"]](case, _inputs(case, seed))


def _exact_norm_rope(case, x):
    d, pairs, B, T = case["d"], case["pairs"], case["B"], case["T"]
    pos = x["positions"].double()
    pos = pos if pos.dim() == 3 else pos[None]
    counts = _sections(case) or (pairs,)
    axis = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], device=pos.device)
    angle = pos[axis].permute(1, 2, 0) * x["inv_freq"].double()  # [B, T, pairs]
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]  # a pair as one complex number
    p = torch.arange(pairs, device=pos.device)
    first, second = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + pairs)
    outs, dx, dw = [], [], []
    for n in ("q", "k"):
        rows = x[n].double().transpose(1, 2)  # [B, H, T, d]
        w = x[n + "_weight"].double()
        length = torch.sqrt((rows * rows).sum(-1, keepdim=True) / d + NORM_EPS)
        y = rows / length * w

        def spin(y, turn):
            z = torch.complex(y[..., first], y[..., second]) * turn
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        outs.append(spin(y, turn).reshape(-1, T, d))
        if case["train"]:
            up = spin(x["d" + n].double().reshape(rows.shape), turn.conj())
            dw.append((up * rows / length).sum((0, 1, 2)))
            up = up * w
            g = up / length - rows * (up * rows).sum(-1, keepdim=True) / (d * length ** 3)
            dx.append(g.transpose(1, 2).contiguous())
    return (*outs, *dx, *dw)


def _exact_scan(case, x):
    N, T, D = case["N"], case["T"], case["D"]
    if T * (2 if case["train"] else 1) > 200000:
        return None
    xs, gate = x["x"].double().transpose(0, 1).contiguous(), x["gate"].double().transpose(0, 1).contiguous()
    log_a = gate if case["form"] == "log" else torch.nn.functional.logsigmoid(gate)
    a = torch.exp(log_a)
    b = -torch.expm1(log_a) if case["complement"] else torch.ones_like(a)
    pad = None
    if "lengths" in x:
        pad = (torch.arange(T, device=a.device)[:, None] >= x["lengths"])[..., None].expand_as(a)
        a, b = a.masked_fill(pad, 1.0), b.masked_fill(pad, 0.0)
    u, h = b * xs, [x["state"].double()]
    for t in range(T):
        h.append(torch.addcmul(u[t], a[t], h[-1]))
    h = torch.stack(h)
    out, final = h[1:], h[-1]
    out = (out if pad is None else out.masked_fill(pad, 0.0)).transpose(0, 1)
    if not case["train"]:
        return out, final
    g = x["dout"].double().transpose(0, 1).contiguous()
    if pad is not None:
        g = g.masked_fill(pad, 0.0)
    lam, run_ = torch.empty_like(g), x["dfinal"].double()
    for t in range(T - 1, -1, -1):
        lam[t] = run_ = g[t] + run_
        run_ = a[t] * run_
    dlog = lam * a * (h[:-1] - xs if case["complement"] else h[:-1])
    dgate = dlog if case["form"] == "log" else dlog * torch.sigmoid(-gate)
    dx = lam * b
    if pad is not None:
        dgate, dx = dgate.masked_fill(pad, 0.0), dx.masked_fill(pad, 0.0)
    return out, final, dx.transpose(0, 1), dgate.transpose(0, 1), run_


def _exact_cross(case, x):
    S, d, G = case["L"] * case["R"], case["d"], case["H"] // case["Hk"]
    q = x["q"].double().flatten(2)
    if case["op"] == "cross_query":
        A, B = x["state"][:, S * d:].double(), x["state"][:, :S * d].double().reshape(-1, S, d)
    else:
        k, v, keep = _keys(case, x, torch.float64)
        A, B = k.sum(1), torch.matmul(_t(k), v)
    r = 1.0 / (A + EPS)
    Er = (B * r[..., None]).repeat_interleave(G, dim=0)
    out = torch.matmul(q, Er)
    if case["op"] == "cross_query":
        return out
    if not case["train"]:
        return (out,)
    g = x["dout"].double()
    dq = torch.matmul(g, _t(Er))
    dE = torch.matmul(_t(q), g).reshape(-1, G, S, d).sum(1)
    dB = dE * r[..., None]
    dA = -(dE * B).sum(-1) * r * r
    dk, dv = torch.matmul(v, _t(dB)) + dA[:, None], torch.matmul(k, dB)
    if keep is not None:
        dk, dv = dk.masked_fill(~keep, 0.0), dv.masked_fill(~keep, 0.0)
    return out, dq.reshape(x["q"].shape), dk.reshape(x["k"].shape), dv
