"""Performance cases of the operators around the INT8 recurrence of a layer: the short causal convolution, the selective
scan (both for prompts and for single tokens), the INT8 matrix product of the projections, and the norms before and after a
block with their residual, gate and quantisation.

Where ``own`` is true a case makes the calls that a serving program makes; otherwise it computes the same in elementary
torch operations in 32 bits, rounded once at the end. ``exact`` computes it in 64 bits, the recurrences token by token.

Sizes: the 2.7B-shaped Mamba-2 layer of this repository's benchmark (d_model 2560, d_inner 5120, 80 heads of 64, d_state
128, one group: in_proj 10576 wide, xBC 5376 wide) and generic ones."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# --------------------------------------------------------------------------------------------------------- the cases
def _conv(B, T, D, W=4, dtype="bf16", pitch=0, ragged=False):
    """``pitch``: channels of the wider projection output that x is a slice of (0: dense). ``ragged``: prompts of different
    lengths, right-padded, one of them empty, each continuing a cached prefix."""
    return dict(op="conv", B=B, T=T, D=D, W=W, dtype=dtype, pitch=pitch, ragged=ragged)


def _conv_token(B, D, W=4, dtype="bf16", pitch=0):
    return dict(op="conv_token", B=B, D=D, W=W, dtype=dtype, pitch=pitch)


def _scan(B, T, D, N=16, G=1, dtype="bf16", gate=True, ragged=False):
    return dict(op="scan", B=B, T=T, D=D, N=N, G=G, dtype=dtype, gate=gate, ragged=ragged)


def _scan_token(B, D, N=16, G=1, dtype="bf16", state="f32"):
    """One decay rate per channel and state."""
    return dict(op="scan_token", B=B, D=D, N=N, G=G, dtype=dtype, state=state)


def _heads_token(B, H, P, N, G=1, dtype="bf16", state="f32"):
    """One decay rate per head: the token step next to the INT8 SSD prefill."""
    return dict(op="heads_token", B=B, H=H, P=P, N=N, G=G, dtype=dtype, state=state)


def _linear(M, K, N, dtype="bf16", form="codes"):
    """``form``: what the call starts from. "codes": rows that are INT8 already; "rows": floating-point rows, quantised row by
    row in the call; "norm": the residual add and norm ahead of the projection, whose kernel writes the codes."""
    return dict(op="linear", M=M, K=K, N=N, dtype=dtype, form=form)


def _norm(rows, D, dtype="bf16", post=False):
    """Residual add, then norm; ``post``: the block's output is normed too, before it is scaled and added."""
    return dict(op="norm", rows=rows, D=D, dtype=dtype, post=post)


def _gated(rows, D, group, gate_first=True, dtype="bf16", pitch=0):
    return dict(op="gated", rows=rows, D=D, group=group, gate_first=gate_first, dtype=dtype, pitch=pitch)


def listed():
    case = lambda name, c: {"name": name, **c}  # noqa: E731
    return [
        # decode step of 48 users: xBC is a slice of the in_proj output
        case("conv token", _conv_token(48, 5376, pitch=10576)),
        # a batch of uneven prompts that continue cached prefixes, channels off every vector width
        case("conv ragged prompts", _conv(6, 1037, 1667, W=3, dtype="f16", ragged=True)),
        # a long prefill
        case("conv long prompts", _conv(4, 16384, 5376, pitch=10576)),
        # one user's decode step, one decay rate per channel and state
        case("scan token", _scan_token(1, 5120)),
        # decode step of 64 users next to the INT8 SSD prefill
        case("scan token heads", _heads_token(64, 80, 64, 128)),
        # uneven prompts, few channels, a d_state off every vector width
        case("scan ragged prompts", _scan(7, 203, 1002, N=13, G=3, dtype="f32", ragged=True)),
        # one user's long prompt
        case("scan long prompt", _scan(1, 16384, 2048)),
        # out_proj of a decode step: latency and the weights' bytes
        case("product token", _linear(3, 5120, 2560, form="rows")),
        # in_proj of a short prompt behind its norm: no dimension fits a tile
        case("product after norm", _linear(333, 2560, 10576, dtype="f16", form="norm")),
        # in_proj of a long prefill
        case("product prompts", _linear(32768, 2560, 10576)),
        # norms around a block: its output normed, scaled, added to the residual, and the sum normed for the next block
        case("norms around a block", _norm(1021, 2561, dtype="f16", post=True)),
        # between the SSD and out_proj of a long prefill: the gate is a slice of the in_proj output
        case("gated norm", _gated(32768, 5120, 5120, pitch=10576)),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def some(*v):
        return v[rng.randrange(len(v))]

    op = some("conv", "conv_token", "scan", "scan_token", "heads_token", "linear", "norm", "gated")
    dt = some("bf16", "bf16", "f16", "f32")
    if op == "conv":
        D = size(64, 8192)
        B = size(1, 16)
        T = size(1, min(16384, 350_000_000 // (B * D)))
        return _conv(B, T, D, some(2, 3, 4, 4), dt, some(0, D + size(1, 4096)), some(False, True))
    if op == "conv_token":
        D = size(64, 8192)
        return _conv_token(size(1, 256), D, some(2, 3, 4, 4), dt, some(0, D + size(1, 4096)))
    if op in ("scan", "scan_token"):
        G = some(1, 1, 2, 4)
        D = G * size(64, 8192 // G)
        N = some(16, 16, 8, rng.randrange(1, 33))
        if op == "scan_token":
            return _scan_token(size(1, 256), D, N, G, dt, some("f32", "f32", "bf16", "f16"))
        B = size(1, 8)
        T = size(1, max(1, min(16384, 530_000_000 // (B * D * N))))
        return _scan(B, T, D, N, G, dt, some(True, True, False), some(False, True))
    if op == "heads_token":
        G = some(1, 1, 2, 8)
        H, P, N = G * size(1, 128 // G), some(32, 64, 64, 128), some(16, 64, 128, 128, 256)
        B = size(1, max(1, min(128, 42_000_000 // (H * P * N))))
        return _heads_token(B, H, P, N, G, dt, some("f32", "f32", "bf16", "f16"))
    if op == "linear":
        K, N = size(64, 8192), size(64, 16384)
        # codes of normed fp32 rows differ by steps between any two orders of the norm's sum: more than an fp32 output shows
        form = some("codes", "rows") if dt == "f32" else some("codes", "rows", "norm")
        return _linear(size(1, min(32768, 880_000_000_000 // (K * N))), K, N, dt, form)
    if op == "norm":
        D = size(64, 8192)
        return _norm(size(1, min(32768, 160_000_000 // D)), D, dt, some(False, True))
    group = some(1, 1, 2, 8)
    D = group * size(64, 8192 // group)
    return _gated(size(1, min(32768, 160_000_000 // D)), D, D // group, some(True, False), dt, some(0, D + size(1, 4096)))


# -------------------------------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _heavy(gen, t):
    """Activations with the few heavy channels that make quantisation hard: 1 % of them 20 times as large."""
    n = t.shape[-1]
    t[..., torch.randperm(n, generator=gen, device="cuda")[: max(1, n // 100)]] *= 20.0
    return t


def _slice(gen, lead, width, pitch, dtype):
    """[*lead, width]; with a pitch the first columns of a wider buffer."""
    t = _randn(gen, *lead, width, dtype=dtype)
    if not pitch:
        return t
    buf = torch.zeros(*lead, pitch, device="cuda", dtype=dtype)
    buf[..., :width] = t
    return buf[..., :width]


def _lengths(gen, B, T):
    n = torch.randint(1, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    n[0] = T
    if B > 1:
        n[-1] = 0
    return n


def _slots(gen, B):
    """A cache with room for more sequences than the batch has, the batch's in any order."""
    S = B + max(1, B // 2)
    return S, torch.randperm(S, generator=gen, device="cuda")[:B].to(torch.int32)


def _codes(t):
    """Symmetric INT8 codes and scales of the rows, the codes' rows on 16-byte boundaries."""
    n, k = t.shape
    scale = t.abs().amax(1) / 127
    buf = torch.zeros(n, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    codes = buf[:, :k]
    codes.copy_(torch.round(t / scale.unsqueeze(1)).clamp(-127, 127))
    return codes, scale


def _dt_inputs(gen, shape, heads, dtype):
    """Raw steps around a bias whose softplus is spread over 0.001 to 0.1."""
    want = torch.exp(torch.rand(heads, generator=gen, device="cuda") * math.log(100.0) + math.log(0.001))
    return _randn(gen, *shape, dtype=dtype) * 0.5, want + torch.log(-torch.expm1(-want))


def prepare(case, seed):
    c, gen = case, _gen(seed)
    op, dt = c["op"], DTYPES[c["dtype"]]
    s = dict(op=op, dtype=dt)
    if op in ("conv", "conv_token"):
        B, D, W = c["B"], c["D"], c["W"]
        s["weight"] = (torch.rand(D, W, generator=gen, device="cuda") * 2 - 1) / math.sqrt(W)
        s["bias"] = _randn(gen, D) * 0.1
        if op == "conv":
            s["x"] = _slice(gen, (B, c["T"]), D, c["pitch"], dt)
            s["lengths"] = _lengths(gen, B, c["T"]) if c["ragged"] else None
            s["initial"] = _randn(gen, B, W - 1, D, dtype=dt) if c["ragged"] else None
        else:
            s["x"] = _slice(gen, (B,), D, c["pitch"], dt)
            S, s["slots"] = _slots(gen, B)
            s["state"] = _randn(gen, S, W - 1, D, dtype=dt)
    elif op in ("scan", "scan_token"):
        B, D, N, G = c["B"], c["D"], c["N"], c["G"]
        lead = (B, c["T"]) if op == "scan" else (B,)
        s["u"] = _randn(gen, *lead, D, dtype=dt)
        s["dt"], s["bias"] = _dt_inputs(gen, (*lead, D), D, dt)
        s["A"] = -torch.arange(1, N + 1, device="cuda").float() * torch.exp(_randn(gen, D, N) * 0.1)
        s["B"], s["C"] = _randn(gen, *lead, G, N, dtype=dt), _randn(gen, *lead, G, N, dtype=dt)
        s["D"] = torch.rand(D, generator=gen, device="cuda") + 0.5
        s["z"] = _randn(gen, *lead, D, dtype=dt) if c.get("gate", True) else None
        if op == "scan":
            s["lengths"] = _lengths(gen, B, c["T"]) if c["ragged"] else None
            s["initial"] = _randn(gen, B, D, N) if c["ragged"] else None
        else:
            S, s["slots"] = _slots(gen, B)
            s["state"] = _randn(gen, S, D, N, dtype=DTYPES[c["state"]])
    elif op == "heads_token":
        B, H, P, N, G = c["B"], c["H"], c["P"], c["N"], c["G"]
        s["u"], s["z"] = _randn(gen, B, H, P, dtype=dt), _randn(gen, B, H, P, dtype=dt)
        s["dt"], s["bias"] = _dt_inputs(gen, (B, H), H, dt)
        s["A"] = -torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(16.0))
        s["B"], s["C"] = _randn(gen, B, G, N, dtype=dt), _randn(gen, B, G, N, dtype=dt)
        s["D"] = torch.rand(H, generator=gen, device="cuda") + 0.5
        S, s["slots"] = _slots(gen, B)
        s["state"] = _randn(gen, S, H, P, N, dtype=DTYPES[c["state"]])
    elif op == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        s["w"], s["w_scale"] = _codes(_randn(gen, N, K) / math.sqrt(K))
        s["bias"] = _randn(gen, N) * 0.1
        x = _heavy(gen, _randn(gen, M, K))
        if c["form"] == "codes":
            s["x"], s["x_scale"] = _codes(x)
        else:
            s["x"] = x.to(dt)
            if c["form"] == "norm":
                s["residual"] = _randn(gen, M, K, dtype=dt)
                s["norm"] = torch.rand(K, generator=gen, device="cuda") + 0.5
    elif op == "norm":
        R, D = c["rows"], c["D"]
        s["x"], s["residual"] = _heavy(gen, _randn(gen, R, D)).to(dt), _randn(gen, R, D, dtype=dt)
        s["weight"] = torch.rand(D, generator=gen, device="cuda") + 0.5
        s["post"] = torch.rand(D, generator=gen, device="cuda") + 0.5 if c["post"] else None
    else:
        R, D = c["rows"], c["D"]
        s["x"], s["gate"] = _randn(gen, R, D, dtype=dt), _slice(gen, (R,), D, c["pitch"], dt)
        s["weight"] = torch.rand(D, generator=gen, device="cuda") + 0.5
        s["group"], s["gate_first"] = c["group"], c["gate_first"]
    return s


RESIDUAL_SCALE = 0.5
EPS = 1e-5


# --------------------------------------------------------------------------------------------------- the plain forms
def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _inside(lengths, B, T):
    """[B, T]: tokens that belong to their sequence."""
    t = torch.arange(T, device="cuda")
    return torch.full((B,), T, device="cuda").unsqueeze(1) > t if lengths is None else lengths.unsqueeze(1) > t


def _plain_conv(s):
    x, w = s["x"].float(), s["weight"]
    B, T, D = x.shape
    W = w.shape[1]
    before = x.new_zeros(B, W - 1, D) if s["initial"] is None else s["initial"].float()
    line = torch.cat([before, x], 1)
    y = s["bias"] + sum(line[:, i:i + T] * w[:, i] for i in range(W))
    inside = _inside(s["lengths"], B, T)
    y = torch.where(inside.unsqueeze(-1), _silu(y), 0.0)
    at = inside.sum(1, keepdim=True) + torch.arange(W - 1, device="cuda")
    return {"y": y.to(s["dtype"]), "state": line.gather(1, at.unsqueeze(-1).expand(B, W - 1, D)).to(s["dtype"])}


def _plain_conv_token(s):
    at = s["slots"].long()
    line = torch.cat([s["state"][at], s["x"].unsqueeze(1)], 1).float()
    y = _silu(s["bias"] + (line * s["weight"].t()).sum(1))
    s["state"][at] = line[:, 1:].to(s["dtype"])
    return {"y": y.to(s["dtype"]), "state": s["state"]}


def _plain_scan(s):
    """h_t = a_t h_{t-1} + b_t over all tokens at once: after the round of width w, (a, b) of a token is the composition of
    the 2 w steps that end with it."""
    u = s["u"].float()
    B, T, D = u.shape
    G, N = s["B"].shape[2:]
    inside = _inside(s["lengths"], B, T).unsqueeze(-1)
    dt = torch.where(inside, _softplus(s["dt"].float() + s["bias"]), 0.0)
    step = torch.where(inside, dt * u, 0.0)
    Bm = torch.where(inside.unsqueeze(-1), s["B"].float(), 0.0).repeat_interleave(D // G, 2)
    a = torch.exp(dt.unsqueeze(-1) * s["A"])
    h = step.unsqueeze(-1) * Bm
    if s["initial"] is not None:
        h[:, 0] += a[:, 0] * s["initial"]
    width = 1
    while width < T:
        h = torch.cat([h[:, :width], h[:, width:] + a[:, width:] * h[:, :-width]], 1)
        a = torch.cat([a[:, :width], a[:, width:] * a[:, :-width]], 1)
        width *= 2
    last = h[:, -1].clone()
    del a, Bm
    y = torch.stack([torch.einsum("btdn,btn->btd", v, c) for v, c in zip(h.chunk(G, 2), s["C"].float().unbind(2))], 2).reshape(B, T, D)
    y = y + s["D"] * u
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return {"y": torch.where(inside, y, 0.0).to(s["dtype"]), "state": last}


def _plain_scan_token(s):
    at, u = s["slots"].long(), s["u"].float()
    Bm, Cm = ((t.float().repeat_interleave(u.shape[1] // t.shape[1], 1)) for t in (s["B"], s["C"]))
    dt = _softplus(s["dt"].float() + s["bias"])
    if s["op"] == "heads_token":
        h = s["state"][at].float() * torch.exp(dt * s["A"])[..., None, None] + (dt.unsqueeze(-1) * u).unsqueeze(-1) * Bm.unsqueeze(2)
        y = (h * Cm.unsqueeze(2)).sum(-1) + s["D"].unsqueeze(-1) * u
    else:
        h = s["state"][at].float() * torch.exp(dt.unsqueeze(-1) * s["A"]) + (dt * u).unsqueeze(-1) * Bm
        y = (h * Cm).sum(-1) + s["D"] * u
    s["state"][at] = h.to(s["state"].dtype)
    return {"y": (y * _silu(s["z"].float())).to(s["dtype"]), "state": s["state"]}


def _plain_quantise(x):
    """Codes as numbers, half away from zero, and their scale."""
    scale = x.abs().amax(1, keepdim=True) / 127
    y = x * (1 / scale)
    return torch.trunc(torch.clamp(y, -127, 127) + torch.copysign(torch.full_like(y, 0.5), y)), scale


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _plain_linear(s):
    r = None
    if "x_scale" in s:
        x, scale = s["x"].float(), s["x_scale"].unsqueeze(1)
    elif "norm" in s:
        r = s["residual"].float() + RESIDUAL_SCALE * s["x"].float()
        x, scale = _plain_quantise(_rms(r, s["norm"]))
    else:
        x, scale = _plain_quantise(s["x"].float())
    y = (torch.matmul(x, s["w"].float().t()) * scale * s["w_scale"] + s["bias"]).to(s["dtype"])
    return {"y": y} if r is None else {"y": y, "residual": r.to(s["dtype"])}


def _plain_norm(s):
    x = s["x"].float()
    r = s["residual"].float() + RESIDUAL_SCALE * (x if s["post"] is None else _rms(x, s["post"]))
    return {"y": _rms(r, s["weight"]).to(s["dtype"]), "residual": r.to(s["dtype"])}


def _plain_gated(s):
    x, gate = s["x"].float(), _silu(s["gate"].float())
    if s["gate_first"]:
        x = x * gate
    y = _rms(x.unflatten(-1, (-1, s["group"])), s["weight"].view(-1, s["group"])).flatten(-2)
    return {"y": (y if s["gate_first"] else y * gate).to(s["dtype"])}


PLAIN = {"conv": _plain_conv, "conv_token": _plain_conv_token, "scan": _plain_scan, "scan_token": _plain_scan_token,
         "heads_token": _plain_scan_token, "linear": _plain_linear, "norm": _plain_norm, "gated": _plain_gated}


# ------------------------------------------------------------------------------------------------------- the calls
def _own(s):
    from linquant_b200.kernels import layer

    op = s["op"]
    if op == "conv":
        y, state = layer.short_conv_fwd(s["x"], s["weight"], s["bias"], initial_state=s["initial"], lengths=s["lengths"],
                                        output_final_state=True)
        return {"y": y, "state": state}
    if op == "conv_token":
        return {"y": layer.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"]), "state": s["state"]}
    if op == "scan":
        y, state = layer.selective_scan_fwd(s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                            initial_state=s["initial"], lengths=s["lengths"], output_final_state=True)
        return {"y": y, "state": state}
    if op in ("scan_token", "heads_token"):
        y = layer.selective_scan_step(s["state"], s["u"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                      slots=s["slots"])
        return {"y": y, "state": s["state"]}
    if op == "linear":
        if "norm" in s:
            (codes, scale), r = layer.rms_norm_fwd(s["x"], s["norm"], residual=s["residual"], residual_scale=RESIDUAL_SCALE,
                                                   eps=EPS, quantize=True)
            return {"y": layer.int8_linear_fwd(codes, s["w"], s["w_scale"], x_scale=scale, bias=s["bias"], out_dtype=s["dtype"]),
                    "residual": r}
        return {"y": layer.int8_linear_fwd(s["x"], s["w"], s["w_scale"], x_scale=s.get("x_scale"), bias=s["bias"], out_dtype=s["dtype"])}
    if op == "norm":
        y, r = layer.rms_norm_fwd(s["x"], s["weight"], residual=s["residual"], residual_scale=RESIDUAL_SCALE,
                                  post_weight=s["post"], eps=EPS)
        return {"y": y, "residual": r}
    return {"y": layer.gated_rms_norm_fwd(s["x"], s["gate"], s["weight"], group_size=s["group"], gate_first=s["gate_first"], eps=EPS)}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, op, e = case, case["op"], SIZE[case["dtype"]]
    if op == "conv":
        n, state = c["B"] * c["T"] * c["D"], c["B"] * (c["W"] - 1) * c["D"]
        return {"bytes": e * (2 * n + (2 if c["ragged"] else 1) * state) + 4 * c["D"] * (c["W"] + 1), "flops": n * (2 * c["W"] + 4)}
    if op == "conv_token":
        n = c["B"] * c["D"]
        return {"bytes": e * n * (2 + 2 * (c["W"] - 1)) + 4 * c["D"] * (c["W"] + 1), "flops": n * (2 * c["W"] + 4)}
    if op == "scan":
        n = c["B"] * c["T"] * c["D"]
        state = 4 * c["B"] * c["D"] * c["N"] * (2 if c["ragged"] else 1)
        byte = e * (n * (4 if c["gate"] else 3) + 2 * c["B"] * c["T"] * c["G"] * c["N"]) + state + 4 * c["D"] * (c["N"] + 2)
        return {"bytes": byte, "flops": n * (7 * c["N"] + 10)}  # exponent, exp, decay, input, read-out per state
    if op == "scan_token":
        n = c["B"] * c["D"]
        byte = n * (4 * e + 2 * SIZE[c["state"]] * c["N"]) + 2 * e * c["B"] * c["G"] * c["N"] + 4 * c["D"] * (c["N"] + 2)
        return {"bytes": byte, "flops": n * (7 * c["N"] + 10)}
    if op == "heads_token":
        n = c["B"] * c["H"] * c["P"]
        byte = n * (3 * e + 2 * SIZE[c["state"]] * c["N"]) + e * c["B"] * (c["H"] + 2 * c["G"] * c["N"]) + 12 * c["H"]
        return {"bytes": byte, "flops": n * (5 * c["N"] + 10)}
    if op == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        rows = {"codes": 1, "rows": e, "norm": 3 * e}[c["form"]] * M * K + (4 * M if c["form"] == "codes" else 0)
        return {"bytes": rows + N * K + e * M * N + 8 * N, "flops": 2.0 * M * K * N}
    n = c["rows"] * c["D"]
    if op == "norm":
        return {"bytes": 4 * e * n + (8 if c["post"] else 4) * c["D"], "flops": n * (11 if c["post"] else 7)}
    return {"bytes": 3 * e * n + 4 * c["D"], "flops": n * 10}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def _sequence(b, lengths, T):
    return T if lengths is None else int(lengths[b])


def _exact_conv(s):
    x, w, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    B, T, D = x.shape
    W = w.shape[1]
    y, state = torch.zeros_like(x), x.new_zeros(B, W - 1, D)
    for b in range(B):
        n = _sequence(b, s["lengths"], T)
        line = x.new_zeros(W - 1 + n, D)
        line[W - 1:] = x[b, :n]
        if s["initial"] is not None:
            line[:W - 1] = s["initial"][b].double()
        if n:
            v = (line.unfold(0, W, 1) * w).sum(-1) + bias
            y[b, :n] = v * torch.sigmoid(v)
        state[b] = line[n:]
    return {"y": y, "state": state}


def _exact_conv_token(s):
    state, y = s["state"].double(), []
    for b, slot in enumerate(s["slots"].tolist()):
        line = torch.cat([state[slot], s["x"][b].double().unsqueeze(0)])
        v = s["bias"].double() + torch.einsum("td,dt->d", line, s["weight"].double())
        y.append(v * torch.sigmoid(v))
        state[slot] = line[1:]
    return {"y": torch.stack(y), "state": state}


def _exact_step(h, u, dt, A, Bm, Cm, D, z):
    """h [.., D, N] or [.., H, P, N]; A, Bm and Cm shaped to go with it; dt with one trailing axis fewer."""
    h = h * torch.exp(dt.unsqueeze(-1) * A) + (dt * u).unsqueeze(-1) * Bm
    y = (h * Cm).sum(-1) + D * u
    return h, y if z is None else y * z * torch.sigmoid(z)


def _exact_softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def _exact_scan(s):
    u, T, D = s["u"].double(), s["u"].shape[1], s["u"].shape[2]
    dt = _exact_softplus(s["dt"].double() + s["bias"].double())
    z = None if s["z"] is None else s["z"].double()
    A, Dv = s["A"].double(), s["D"].double()
    rep = D // s["B"].shape[2]
    h = u.new_zeros(u.shape[0], *A.shape) if s["initial"] is None else s["initial"].double()
    y = torch.zeros_like(u)
    live = torch.full((u.shape[0],), T, device="cuda") if s["lengths"] is None else s["lengths"]
    for t in range(T):
        Bm, Cm = (s[n][:, t].double().repeat_interleave(rep, 1) for n in ("B", "C"))
        h2, yt = _exact_step(h, u[:, t], dt[:, t], A, Bm, Cm, Dv, None if z is None else z[:, t])
        on = live > t
        h = torch.where(on[:, None, None], h2, h)
        y[:, t] = torch.where(on[:, None], yt, 0.0)
    return {"y": y, "state": h}


def _exact_scan_token(s):
    at, state, u = s["slots"].long(), s["state"].double(), s["u"].double()
    Bm, Cm = (s[n].double().repeat_interleave(u.shape[1] // s[n].shape[1], 1) for n in ("B", "C"))
    dt, A, D = _exact_softplus(s["dt"].double() + s["bias"].double()), s["A"].double(), s["D"].double()
    if s["op"] == "heads_token":
        dt, A, D = dt.unsqueeze(-1), A[:, None, None], D.unsqueeze(-1)
        Bm, Cm = Bm.unsqueeze(2), Cm.unsqueeze(2)
    h, y = _exact_step(state[at], u, dt, A, Bm, Cm, D, s["z"].double())
    state[at] = h
    return {"y": y, "state": state}


def _exact_codes(x):
    scale = x.abs().amax(1, keepdim=True) / 127
    v = x / scale
    return torch.sign(v) * torch.floor(v.abs() + 0.5) * scale


def _exact_norm(v, weight):
    return weight.double() * v / torch.sqrt(torch.mean(v * v, -1, keepdim=True) + EPS)


def _exact_linear(s):
    out = {}
    if "x_scale" in s:
        x = s["x"].double() * s["x_scale"].double().unsqueeze(1)
    elif "norm" in s:
        out["residual"] = s["residual"].double() + RESIDUAL_SCALE * s["x"].double()
        x = _exact_codes(_exact_norm(out["residual"], s["norm"]))
    else:
        x = _exact_codes(s["x"].double())
    out["y"] = torch.matmul(x, (s["w"].double() * s["w_scale"].double().unsqueeze(1)).t()) + s["bias"].double()
    return out


def _exact_norms(s):
    x = s["x"].double()
    r = s["residual"].double() + RESIDUAL_SCALE * (x if s["post"] is None else _exact_norm(x, s["post"]))
    return {"y": _exact_norm(r, s["weight"]), "residual": r}


def _exact_gated(s):
    x, gate = s["x"].double(), s["gate"].double() * torch.sigmoid(s["gate"].double())
    R, D = x.shape
    x = x * gate if s["gate_first"] else x
    y = _exact_norm(x.view(R, D // s["group"], s["group"]), s["weight"].view(-1, s["group"])).reshape(R, D)
    return {"y": y if s["gate_first"] else y * gate}


EXACT = {"conv": _exact_conv, "conv_token": _exact_conv_token, "scan": _exact_scan, "scan_token": _exact_scan_token,
         "heads_token": _exact_scan_token, "linear": _exact_linear, "norm": _exact_norms, "gated": _exact_gated}


def exact(case, seed):
    s = prepare(case, seed)
    return EXACT[s["op"]](s)
