"""The layer of the gated delta rule as timed cases: from the residual stream to
the streams of a matrix-valued recurrence and back.

  op "delta"      race_delta_rule: S_t = a_t S_{t-1} + b_t k_t (v_t - a_t S_{t-1}^T k_t)^T,
                  o_t = scale S_t^T q_t per stream, S [dk, dv], a = exp(gate) or
                  sigmoid(gate); value heads may share key heads, each batch entry
                  has its own length; race_delta_rule_carry for single tokens.
  op "add_norm"   race_add_norm: s = x + residual and s / rms(s) * weight;
                  race_add_norm_e4m3: the normed rows in 8 bits, with a scale per
                  row or per group of columns.
  op "gate_norm"  race_gate_norm: a recurrence's output streams [B * H, T, d] as
                  rows [B, T, H, d], normed and gated: x / rms(x) * weight * silu(gate).

A case is a dict of plain values.  `train` asks for the gradients w.r.t. every
differentiable input too.  Sizes are those of this repository's configurations
and tests (heads of 64 and 128 columns, batches of 8, 577 patches, 1531 tokens) or
generic ones.

With `own` false, run() computes the operators in elementary torch operations,
in 32 bits (sums of log decays in 64), rounded once at the end; the recurrence in
chunks of 64 tokens, whose maps of the state are joined by doubling.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

NORM_EPS = 1e-6   # of the root mean square
CHUNK = 64        # tokens of a chunk of the plain recurrence
LOWEST = -200.0   # log decays below this forget everything: exp is zero in 32 bits
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _race():
    return importlib.import_module("race-attention-kernel_amd")


def _delta(name, B, H, Hk, T, dk, dv, dtype, form="log", state=False, ragged=False, resets=False, train=False):
    c = dict(op="delta", B=B, H=H, Hk=Hk, T=T, dk=dk, dv=dv, dtype=dtype, form=form, state=state, ragged=ragged,
             resets=resets, train=train)
    return c if name is None else dict(c, name=name)


def _add_norm(name, rows, D, dtype, out="same", group=0, residual=True, train=False):
    c = dict(op="add_norm", rows=rows, D=D, dtype=dtype, out=out, group=group, residual=residual, train=train)
    return c if name is None else dict(c, name=name)


def _gate_norm(name, B, T, H, d, dtype, train=False):
    c = dict(op="gate_norm", B=B, T=T, H=H, d=d, dtype=dtype, train=train)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # One decode step of a batch of 64, two value heads to a key head.
        _delta("delta_decode_bf16", 64, 16, 8, 1, 128, 128, "bf16", state=True),
        # The prefill of one long prompt of packed documents: the state is dropped where one begins.
        _delta("delta_prefill_bf16_T32k", 1, 16, 8, 32768, 128, 128, "bf16", state=True, resets=True),
        # A padded batch of short prompts, logits as gates.
        _delta("delta_prefill_bf16_T577", 16, 12, 12, 577, 64, 128, "bf16", form="sigmoid", ragged=True),
        # A training step at language-model scale.
        _delta("delta_train_bf16", 8, 16, 16, 4096, 128, 128, "bf16", train=True),
        # A training step on a padded batch, from a learned state: odd length, narrow heads, fp32.
        _delta("delta_train_f32_ragged", 4, 6, 3, 1531, 64, 64, "f32", state=True, ragged=True, train=True),
        # One decode step: a layer's rows for an 8-bit projection, a scale a row.
        _add_norm("add_norm_decode_e4m3", 64, 4096, "bf16", out="e4m3"),
        # A prompt's rows for an 8-bit projection, a scale for every 128 columns.
        _add_norm("add_norm_prefill_e4m3_g128", 16384, 4096, "bf16", out="e4m3", group=128),
        # A training step of a layer's norm.
        _add_norm("add_norm_train_bf16", 32768, 2048, "bf16", train=True),
        # A training step at an odd width and row count, fp32 rows.
        _add_norm("add_norm_train_f32_odd", 9235, 1001, "f32", train=True),
        # One decode step of a batch of 64: the recurrence's output back to rows.
        _gate_norm("gate_norm_decode_bf16", 64, 1, 16, 128, "bf16"),
        # A training step at language-model scale.
        _gate_norm("gate_norm_train_bf16", 8, 4096, 16, 128, "bf16", train=True),
        # A training step on a ragged patch count, fp32.
        _gate_norm("gate_norm_train_f32_T577", 16, 577, 12, 96, "f32", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the same ranges; the elements in all stay within those of the largest listed case."""
    op = rng.choice(["delta", "delta", "delta", "add_norm", "add_norm", "gate_norm"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    train = rng.random() < 0.5
    if op == "delta":
        dk = rng.choice([64, 64, 128, 128, 32, 96, 80, 33, 16])
        dv = rng.choice([64, 64, 128, 128, 32, 96, 50, 256, 17])
        Hk = rng.choice([1, 2, 4, 6])
        H = Hk * rng.choice([1, 1, 2, 4])
        B = _log_int(rng, 1, 32)
        T = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 64, max(64, min(32768, (1 << 18) // (B * H))))])
        state = T == 1 or (rng.random() < 0.5 and not (train and dtype == "bf16"))
        return _delta(None, B, H, Hk, T, dk, dv, dtype, rng.choice(["log", "log", "sigmoid"]), state,
                      T > 1 and rng.random() < 0.4, T > 1 and rng.random() < 0.3, train and T > 1)
    if op == "add_norm":
        out = "same" if train else rng.choice(["same", "e4m3", "e4m3"])
        D = rng.choice([_log_int(rng, 16, 16384), 8 * _log_int(rng, 4, 2048), 8 * _log_int(rng, 4, 2048)])
        rows = _log_int(rng, 1, max(1, min(65536, (1 << 26) // D)))
        group = rng.choice([0, 32, 64, 128]) if out == "e4m3" and D % 8 == 0 else 0
        return _add_norm(None, rows, D, dtype, out, group, rng.random() < 0.8, train)
    d = rng.choice([64, 128, 128, 96, 256, 40, 33])
    H = rng.choice([1, 4, 12, 16, 32])
    B = _log_int(rng, 1, 64)
    T = _log_int(rng, 1, max(1, min(16384, (1 << 26) // (B * H * d))))
    return _gate_norm(None, B, T, H, d, dtype, train)


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.

def _inputs(case, seed):
    """The tensors of a case by name, on the GPU, rounded to its dtype."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op, train = DTYPES[case["dtype"]], case["op"], case["train"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def unit(*shape):
        x = normal(*shape)
        return x / x.pow(2).sum(-1, keepdim=True).sqrt()

    x = {}
    if op == "delta":
        B, H, Hk, T, dk, dv = (case[n] for n in ("B", "H", "Hk", "T", "dk", "dv"))
        x["q"], x["k"] = unit(B * Hk, T, dk).to(dt), unit(B * Hk, T, dk).to(dt)
        x["v"] = normal(B * H, T, dv).to(dt)
        # Decays from a few tokens to thousands, another for each head; strengths around a half.
        logit = normal(B * H, T) + torch.linspace(1.0, 7.0, H, device="cuda").repeat(B)[:, None]
        gate = torch.nn.functional.logsigmoid(logit) if case["form"] == "log" else logit
        if case["resets"]:
            at = torch.rand(B * H, T, generator=g, device="cuda") < 1 / 512
            gate = torch.where(at, -math.inf, gate)
        x["gate"] = gate.to(dt)
        x["beta"] = torch.sigmoid(normal(B * H, T)).to(dt)
        if case["state"]:
            x["state"] = normal(B * H, dk, dv) * (dk ** -0.5)
        if case["ragged"]:
            x["lengths"] = torch.randint((T + 1) // 2, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            if B >= 4:
                x["lengths"][1] = 0  # a slot of the batch that holds no sequence
        if train:
            x["dout"] = normal(B * H, T, dv).to(dt)
            if case["state"]:
                x["dfinal"] = normal(B * H, dk, dv) * (dk ** -0.5)
    elif op == "add_norm":
        rows, D = case["rows"], case["D"]
        x["x"] = normal(rows, D).to(dt)
        if case["residual"]:
            x["residual"] = (3 * normal(rows, D)).to(dt)
        x["weight"] = (1 + 0.1 * normal(D)).to(dt)
        if train:
            x["dy"] = normal(rows, D).to(dt)
            if case["residual"]:
                x["dsum"] = normal(rows, D).to(dt)
    else:
        B, T, H, d = (case[n] for n in ("B", "T", "H", "d"))
        x["x"] = normal(B * H, T, d).to(dt)
        x["gate"] = normal(B, T, H, d).to(dt)
        x["weight"] = (1 + 0.1 * normal(d)).to(dt)
        if train:
            x["dy"] = normal(B, T, H, d).to(dt)
    return x


LEAVES = {"delta": ("q", "k", "v", "gate", "beta", "state"), "add_norm": ("x", "residual", "weight"),
          "gate_norm": ("x", "gate", "weight")}


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["train"]:
        x["leaves"] = [x[n].requires_grad_(True) for n in LEAVES[case["op"]] if n in x]
    x["case"] = case
    return x


# ---------------------------------------------------------------------------
# One pass.

def run(x):
    if own:
        return _run_own(x)
    case = x["case"]
    with torch.no_grad():  # the gradients come from their formulas
        return {"delta": _plain_delta, "add_norm": _plain_add_norm, "gate_norm": _plain_gate_norm}[case["op"]](case, x)


def _run_own(x):
    race, case = _race(), x["case"]
    op = case["op"]
    if op == "delta":
        scale = case["dk"] ** -0.5
        step = race.race_delta_rule_carry if case["T"] == 1 else race.race_delta_rule
        outs = step(x["q"], x["k"], x["v"], x["gate"], x["beta"], x.get("state"), gate_form=case["form"], scale=scale,
                    lengths=x.get("lengths"))
        grads = (x.get("dout"), x.get("dfinal"))
        if case["train"] and "dfinal" not in x:  # nothing reads the state after the last token
            outs, grads = outs[:1], grads[:1]
    elif op == "add_norm":
        if case["out"] == "e4m3":
            y, scales, total = race.race_add_norm_e4m3(x["x"], x.get("residual"), x["weight"], eps=NORM_EPS,
                                                       group=case["group"])
            outs = (y, scales, total)
        else:
            outs = race.race_add_norm(x["x"], x.get("residual"), x["weight"], eps=NORM_EPS)
        grads = (x.get("dy"), x.get("dsum"))
        if "residual" not in x:
            outs, grads = outs[:-1], grads[:1]
    else:
        outs, grads = (race.race_gate_norm(x["x"], x["gate"], x["weight"], eps=NORM_EPS),), (x.get("dy"),)
    if not case["train"]:
        return outs
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, x["leaves"], grads))


# ---------------------------------------------------------------------------
# The plain forms.

def _t(m):
    return m.transpose(-1, -2).contiguous()


def _inverse(N):
    """(I + N)^-1 of strictly lower N [..., C, C]: blocks of twice the size from their halves'."""
    C = N.shape[-1]
    i = torch.arange(C, device=N.device)
    X, s = torch.eye(C, device=N.device, dtype=N.dtype).expand(N.shape).contiguous(), 1
    while s < C:
        between = (i[:, None] // (2 * s) == i // (2 * s)) & (i[:, None] // s != i // s)
        X, s = X - torch.matmul(torch.matmul(X, torch.where(between, N, 0.0)), X), 2 * s
    return X


def _join(M, X):
    """The maps s -> M s + X of the chunks (dim 1) after one another, by doubling: each step joins runs of twice the length."""
    s = 1
    while s < X.shape[1]:
        X = torch.cat([X[:, :s], X[:, s:] + torch.matmul(M[:, s:], X[:, :-s])], dim=1)
        if 2 * s < X.shape[1]:
            M = torch.cat([M[:, :s], torch.matmul(M[:, s:], M[:, :-s])], dim=1)
        s *= 2
    return X


def _log_decay(case, gate, dtype):
    g = gate.to(dtype)
    return torch.nn.functional.logsigmoid(g) if case["form"] == "sigmoid" else g


def _keep(case, x):
    """[N, T] truths: the tokens within each sequence; None without lengths."""
    if "lengths" not in x:
        return None
    return torch.arange(case["T"], device=x["v"].device) < x["lengths"].repeat_interleave(case["H"])[:, None]


def _plain_step(case, x):
    """One token."""
    g, dt = case["H"] // case["Hk"], x["v"].dtype
    q, k = (x[n][:, 0].float().repeat_interleave(g, 0)[..., None] for n in ("q", "k"))
    a = torch.exp(_log_decay(case, x["gate"], torch.float32))[:, :, None]
    S = a * x["state"]
    error = x["v"].float() - (k * S).sum(1, keepdim=True)
    S = S + x["beta"].float()[:, :, None] * k * error
    return (case["dk"] ** -0.5 * (q * S).sum(1, keepdim=True)).to(dt), S


def _plain_delta(case, x):
    if case["T"] == 1:
        return _plain_step(case, x)
    T, dk, dv, g, scale = case["T"], case["dk"], case["dv"], case["H"] // case["Hk"], case["dk"] ** -0.5
    dt, N, c = x["v"].dtype, x["v"].shape[0], -(-case["T"] // CHUNK)
    keep = _keep(case, x)

    def chunks(t, per=1):
        t = t.repeat_interleave(per, 0)
        if keep is not None:
            t = torch.where(keep.view(N, T, *[1] * (t.dim() - 2)), t, 0.0)
        return torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, c * CHUNK - T)).view(N, c, CHUNK, *t.shape[2:])

    q, k, v = chunks(x["q"].float(), g), chunks(x["k"].float(), g), chunks(x["v"].float())
    b = chunks(x["beta"].float())
    log_a = chunks(_log_decay(case, x["gate"], torch.float64).clamp(min=LOWEST))
    G = log_a.cumsum(-1)
    i = torch.arange(CHUNK, device=q.device)
    gam = torch.exp(torch.where(i[:, None] >= i, G[..., :, None] - G[..., None, :], -math.inf)).float()
    E, Z, last = torch.exp(G).float(), torch.exp(G[..., -1:] - G).float(), torch.exp(G[..., -1]).float()
    strict = torch.where(i[:, None] > i, gam, 0.0)
    kk, qk = torch.matmul(k, _t(k)), torch.matmul(q, _t(k))
    inv = _inverse(strict * kk * b[..., None, :])
    Ek, Zk = E[..., None] * k, Z[..., None] * k
    of_v, of_s = torch.matmul(inv, v), torch.matmul(inv, Ek)  # Y = of_v - of_s S
    bZk_t = _t(b[..., None] * Zk)
    M = last[..., None, None] * torch.eye(dk, device=q.device) - torch.matmul(bZk_t, of_s)
    X = torch.matmul(bZk_t, of_v)
    first = x["state"][:, None] if "state" in x else torch.zeros(N, 1, dk, dv, device=q.device)
    X = torch.cat([X[:, :1] + torch.matmul(M[:, :1], first), X[:, 1:]], dim=1)
    after = _join(M, X)
    S, final = torch.cat([first, after[:, :-1]], dim=1), after[:, -1]
    Y = of_v - torch.matmul(of_s, S)
    out = scale * (E[..., None] * torch.matmul(q, S) + torch.matmul(gam * qk * b[..., None, :], Y))

    def rows(t, per=1):
        t = t.reshape(N, c * CHUNK, *t.shape[3:])[:, :T]
        return t if per == 1 else t.view(N // per, per, *t.shape[1:]).sum(1)

    if not case["train"]:
        return rows(out).to(dt), final
    dout = chunks(x["dout"].float()) * scale
    dlast = x["dfinal"][:, None] if "dfinal" in x else torch.zeros(N, 1, dk, dv, device=q.device)
    inv_t = _t(inv)
    dU = torch.matmul(_t(gam * qk), dout)  # without the part from the state after the chunk
    part = torch.matmul(_t(E[..., None] * q), dout) - torch.matmul(_t(Ek), torch.matmul(inv_t, b[..., None] * dU))
    M_t, part = _t(M).flip(1), part.flip(1)
    part = torch.cat([part[:, :1] + torch.matmul(M_t[:, :1], dlast), part[:, 1:]], dim=1)
    before = _join(M_t, part).flip(1)
    dS, dstate = torch.cat([before[:, 1:], dlast], dim=1), before[:, 0]
    dU = dU + torch.matmul(Zk, dS)
    dV = torch.matmul(inv_t, b[..., None] * dU)
    P, Hm = torch.matmul(dout, _t(Y)), torch.matmul(dV, _t(Y))
    L, Xn = gam * b[..., None, :] * P, -strict * b[..., None, :] * Hm
    qs, ks, ys = torch.matmul(dout, _t(S)), torch.matmul(dV, _t(S)), torch.matmul(Y, _t(dS))
    dq = E[..., None] * qs + torch.matmul(L, k)
    dk_ = (torch.matmul(_t(L), q) + torch.matmul(Xn, k) + torch.matmul(_t(Xn), k)
           + (b * Z)[..., None] * ys - E[..., None] * ks)
    from_state = Z * (k * ys).sum(-1)
    db = (gam * qk * P).sum(-2) + from_state - (strict * kk * Hm).sum(-2)
    pairs = (L * qk + Xn * kk).double()
    dG = (E * ((q * qs).sum(-1) - (k * ks).sum(-1))).double() + pairs.sum(-1) - pairs.sum(-2) - (b * from_state)
    dG[..., -1] += (b * from_state).sum(-1) + last * (S * dS).sum((-1, -2))
    dlog = dG.flip(-1).cumsum(-1).flip(-1)
    slope = torch.sigmoid(-chunks(x["gate"].double())) if case["form"] == "sigmoid" else 1.0
    dgate = dlog * slope
    if keep is not None:
        dgate, db = (torch.where(chunks(torch.ones_like(x["beta"], dtype=t.dtype)) > 0, t, 0.0) for t in (dgate, db))
    grads = (rows(dq, g).to(dt), rows(dk_, g).to(dt), rows(dV).to(dt), rows(dgate).to(dt), rows(db).to(dt))
    if "state" in x:
        return (rows(out).to(dt), final, *grads, dstate)
    return (rows(out).to(dt), *grads)


def _plain_add_norm(case, x):
    s = x["x"].float()
    if case["residual"]:
        s = (s + x["residual"].float()).to(x["x"].dtype).float()  # the stream's own values are normed
    w = x["weight"].float()
    r = torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + NORM_EPS)
    unit = s * r
    y = unit * w
    total = (s.to(x["x"].dtype),) if case["residual"] else ()
    if case["out"] == "e4m3":
        group = case["group"] or case["D"]
        parts = torch.nn.functional.pad(y, (0, -case["D"] % group)).view(case["rows"], -1, group)
        most = parts.abs().amax(-1)
        y8 = (parts * torch.where(most > 0, E4M3_MAX / most, 0.0)[..., None]).flatten(1)[:, :case["D"]]
        return (y8.to(torch.float8_e4m3fn), most / E4M3_MAX, *total)
    y = y.to(x["x"].dtype)
    if not case["train"]:
        return (y, *total)
    up = x["dy"].float()
    dw = (up * unit).sum(0).to(x["weight"].dtype)
    up = up * w
    dx = r * (up - unit * (up * unit).mean(-1, keepdim=True))
    if case["residual"]:
        dx = (dx + x["dsum"].float()).to(x["x"].dtype)
        return (y, *total, dx, dx, dw)
    return (y, dx.to(x["x"].dtype), dw)


def _plain_gate_norm(case, x):
    B, T, H, d = (case[n] for n in ("B", "T", "H", "d"))
    dt = x["x"].dtype
    rows = x["x"].float().view(B, H, T, d).transpose(1, 2)
    z, w = x["gate"].float(), x["weight"].float()
    r = torch.rsqrt(rows.pow(2).mean(-1, keepdim=True) + NORM_EPS)
    unit, sig = rows * r, torch.sigmoid(z)
    silu = z * sig
    y = (unit * w * silu).to(dt).contiguous()
    if not case["train"]:
        return (y,)
    up = x["dy"].float()
    dw = (up * silu * unit).sum((0, 1, 2)).to(x["weight"].dtype)
    dz = (up * unit * w * sig * (1 + z * (1 - sig))).to(dt)
    up = up * silu * w
    dx = r * (up - unit * (up * unit).mean(-1, keepdim=True))
    return y, dx.transpose(1, 2).reshape(B * H, T, d).to(dt), dz, dw


# ---------------------------------------------------------------------------

def work(case):
    """Each input read once and each output written once; a multiply-add counts two.  Padded batches hold
    three quarters of their rows.  The recurrence token by token: S^T k, the outer product and S^T q."""
    es, op, train = (4 if case["dtype"] == "f32" else 2), case["op"], case["train"]
    if op == "delta":
        B, H, Hk, T, dk, dv = (case[n] for n in ("B", "H", "Hk", "T", "dk", "dv"))
        n, nk = B * H * T, B * Hk * T
        part = 0.75 if case["ragged"] else 1.0
        rows = (2 * nk * dk + n * dv + 2 * n) * es
        states = 4 * B * H * dk * dv * ((1 if case["state"] else 0) + (0 if train and not case["state"] else 1))
        out = n * dv * es
        if train:
            return {"bytes": int(part * (2 * rows + 2 * out) + rows + 2 * states), "flops": int(part * n * dk * dv * 18)}
        return {"bytes": int(part * rows + out + states), "flops": int(part * n * dk * dv * 6)}
    if op == "add_norm":
        n, D = case["rows"] * case["D"], case["D"]
        ins = 2 if case["residual"] else 1
        if case["out"] == "e4m3":
            groups = case["rows"] * (-(-D // case["group"]) if case["group"] else 1)
            return {"bytes": n * (es * (2 * ins - 1) + 1) + 4 * groups + D * es, "flops": n * 8}
        if not train:
            return {"bytes": n * es * 2 * ins + D * es, "flops": n * 5}
        # Forward x, residual -> y, sum; backward sum, dy, dsum -> one gradient for both.
        return {"bytes": n * es * (2 * ins + (4 if case["residual"] else 3)) + 3 * D * es, "flops": n * 16}
    n = case["B"] * case["T"] * case["H"] * case["d"]
    return {"bytes": n * es * (8 if train else 3) + case["d"] * es * (3 if train else 1), "flops": n * (32 if train else 10)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.

def exact(case, seed):
    return {"delta": _exact_delta, "add_norm": _exact_add_norm,
            "gate_norm": _exact_gate_norm}[case["op"]](case, _inputs(case, seed))


def _exact_delta(case, x):
    """The recurrence and its derivative token by token; the backward walks from kept states, 64 tokens apart."""
    T, dk, dv, g, train = case["T"], case["dk"], case["dv"], case["H"] // case["Hk"], case["train"]
    N, dev = case["B"] * case["H"], x["v"].device
    if T * (4 if train else 1) > 200000:
        return None

    def tokens(t, per=1):
        return t.double().repeat_interleave(per, 0).transpose(0, 1)

    q, k, v, b, gate = (tokens(x["q"], g), tokens(x["k"], g), tokens(x["v"]), tokens(x["beta"]), tokens(x["gate"]))
    scale = dk ** -0.5
    a = torch.exp(gate) if case["form"] == "log" else torch.sigmoid(gate)
    live = None
    if "lengths" in x:
        live = torch.arange(T, device=dev)[:, None] < x["lengths"].repeat_interleave(case["H"])
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
        q, k, v = (torch.where(live[..., None], t, 0.0) for t in (q, k, v))

    def step(S, t):
        aS = a[t, :, None, None] * S
        e = v[t] - torch.matmul(k[t, :, None], aS)[:, 0]
        return aS + (b[t, :, None] * k[t])[..., None] * e[:, None], e

    S = x["state"].double() if "state" in x else torch.zeros(N, dk, dv, device=dev, dtype=torch.float64)
    out, kept = torch.empty(T, N, dv, device=dev, dtype=torch.float64), []
    for t in range(T):
        if train and t % 64 == 0:
            kept.append(S)
        S, _ = step(S, t)
        out[t] = scale * torch.matmul(q[t, :, None], S)[:, 0]
    out, final = out.transpose(0, 1), S
    if not train:
        return out, final
    do = x["dout"].double().transpose(0, 1) * scale
    if live is not None:
        do = torch.where(live[..., None], do, 0.0)
    dS = x["dfinal"].double() if "dfinal" in x else torch.zeros_like(S)
    grads = [torch.empty_like(t) for t in (q, k, v, a, b)]
    for c in range(len(kept) - 1, -1, -1):
        walk, S = [], kept[c]
        for t in range(64 * c, min(T, 64 * c + 64)):
            S2, e = step(S, t)
            walk.append((t, S, e, S2))
            S = S2
        for t, S, e, S2 in reversed(walk):
            dS = dS + q[t][..., None] * do[t][:, None]
            grads[0][t] = torch.matmul(S2, do[t][..., None])[..., 0]
            de = b[t, :, None] * torch.matmul(k[t, :, None], dS)[:, 0]
            to_e = torch.matmul(dS, e[..., None])[..., 0]
            back = torch.matmul(S, de[..., None])[..., 0]
            grads[1][t] = b[t, :, None] * to_e - a[t, :, None] * back
            grads[2][t] = de
            grads[3][t] = (dS * S).sum((1, 2)) - (k[t] * back).sum(1)
            grads[4][t] = (k[t] * to_e).sum(1)
            dS = a[t, :, None, None] * (dS - k[t][..., None] * de[:, None])
    slope = a if case["form"] == "log" else a * torch.sigmoid(-gate)
    grads[3] = grads[3] * slope
    if live is not None:
        grads = [torch.where(live.view(T, N, *[1] * (t.dim() - 2)), t, 0.0) for t in grads]
    grads = [t.transpose(0, 1) for t in grads]
    grads[:2] = [t.reshape(N // g, g, T, dk).sum(1) for t in grads[:2]]
    return (out, final, *grads, dS) if "state" in x else (out, *grads)


def _exact_add_norm(case, x):
    s = x["x"].double()
    if case["residual"]:
        s = (s + x["residual"].double()).to(x["x"].dtype).double()
    w, D = x["weight"].double(), case["D"]
    length = torch.sqrt((s * s).sum(-1, keepdim=True) / D + NORM_EPS)
    y = s / length * w
    total = (s,) if case["residual"] else ()
    if case["out"] == "e4m3":
        size = case["group"] or D
        most = torch.stack([p.abs().amax(-1) for p in y.split(size, -1)], -1)
        return (None, most / E4M3_MAX, *total)
    if not case["train"]:
        return (y, *total)
    up = x["dy"].double()
    dw = (up * s / length).sum(0)
    up = up * w
    dx = up / length - s * (up * s).sum(-1, keepdim=True) / (D * length ** 3)
    if case["residual"]:
        dx = dx + x["dsum"].double()
        return (y, *total, dx, dx, dw)
    return (y, dx, dw)


def _exact_gate_norm(case, x):
    B, T, H, d = (case[n] for n in ("B", "T", "H", "d"))
    s = x["x"].double().unflatten(0, (B, H)).permute(0, 2, 1, 3)
    z, w = x["gate"].double(), x["weight"].double()
    length = torch.sqrt((s * s).sum(-1, keepdim=True) / d + NORM_EPS)
    gated = z / (1 + torch.exp(-z))
    y = s / length * w * gated
    if not case["train"]:
        return (y,)
    up = x["dy"].double()
    slope = (1 + torch.exp(-z) * (1 + z)) / (1 + torch.exp(-z)) ** 2
    dz, dw = up * s / length * w * slope, (up * gated * s / length).sum((0, 1, 2))
    up = up * gated * w
    dx = up / length - s * (up * s).sum(-1, keepdim=True) / (d * length ** 3)
    return y, dx.permute(0, 2, 1, 3).reshape(B * H, T, d), dz, dw
