"""Performance cases of the operators of a linear-attention layer that is served in floating point next to the INT8 path:
linear attention with a decay for each head (prompts and single tokens), the group norm behind it, and INT8 projections
whose requests bring low-rank adapters of their own.

Where ``own`` is true a case makes the calls that a serving program makes; otherwise it computes the same in elementary
torch operations in 32 bits (the sums of log-decays and of a group's values in 64), rounded once at the end. ``exact``
computes it in 64 bits, the recurrence token by token.

Sizes: the simple GLA configuration of this repository (4 prompts of 4096 tokens, 16 heads of 128 x 128), its 2.7B-shaped
Mamba-2 layer (d_model 2560, in_proj 10576 wide, out_proj 5120 -> 2560), and generic ones."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# --------------------------------------------------------------------------------------------------------- the cases
def _attention(B, T, H, K, V, share=1, dtype="bf16", decay="token", packed=False, ragged=False):
    """``share``: heads of v that share a head of q and k. ``decay``: "token" (one for each token and head), "head" (a
    constant for each head) or "none". ``packed``: q, k and v are slices of one projection's output. ``ragged``: prompts of
    different lengths, right-padded, one of them empty, each continuing a cached state."""
    return dict(op="attention", B=B, T=T, H=H, K=K, V=V, share=share, dtype=dtype, decay=decay, packed=packed, ragged=ragged)


def _attention_token(B, H, K, V, share=1, dtype="bf16", decay="token", state="f32"):
    return dict(op="attention_token", B=B, H=H, K=K, V=V, share=share, dtype=dtype, decay=decay, state=state)


def _group(rows, D, groups, dtype="bf16", silu=False, gate=False):
    """The norm of each token by itself, behind a mixer; ``gate``: times the SiLU of a slice of the layer's projection."""
    return dict(op="group", rows=rows, D=D, groups=groups, dtype=dtype, silu=silu, gate=gate)


def _group_tokens(B, T, D, groups, dtype="bf16", silu=True, ragged=False):
    """Statistics over all tokens of a sequence, channels last."""
    return dict(op="group_tokens", B=B, T=T, D=D, groups=groups, dtype=dtype, silu=silu, ragged=ragged)


def _adapters(M, K, N, R, L, dtype="bf16", form="codes", runs=1):
    """``form``: "codes" (rows that a norm made INT8 already) or "rows" (floating-point rows, whose codes the call makes). ``runs``:
    tokens of a request that lie next to one another."""
    return dict(op="adapters", M=M, K=K, N=N, R=R, L=L, dtype=dtype, form=form, runs=runs)


def listed():
    case = lambda name, c: {"name": name, **c}  # noqa: E731
    return [
        # one user's decode step: latency
        case("attention token", _attention_token(1, 16, 128, 128)),
        # decode step of 128 users: the states' bytes
        case("attention tokens", _attention_token(128, 16, 128, 128)),
        # one user's short prompt, no whole number of chunks
        case("attention short prompt", _attention(1, 200, 16, 128, 128)),
        # uneven prompts that continue cached states, heads off every vector width, two heads of v a head of q and k
        case("attention ragged prompts", _attention(5, 611, 6, 72, 100, share=2, dtype="f32", ragged=True)),
        # the simple GLA configuration, its operands slices of one projection
        case("attention prompts", _attention(4, 4096, 16, 128, 128, packed=True)),
        # one user's long prompt on few heads with constant decays
        case("attention long prompt", _attention(1, 32768, 8, 128, 128, dtype="f16", decay="head")),
        # behind the decode step's attention, with the gate
        case("group norm tokens", _group(48, 2048, 16, gate=True)),
        # behind a long prefill's attention, with the gate
        case("group norm prompts", _group(32768, 2048, 16, dtype="f16", gate=True)),
        # an encoder's sequences, groups off every vector width
        case("group norm over tokens", _group_tokens(6, 1499, 1026, 18, ragged=True)),
        # out_proj of a decode step, each token with its own adapter
        case("adapters tokens", _adapters(3, 5120, 2560, 16, 8, form="rows")),
        # in_proj of a mixed batch: short runs of many requests
        case("adapters mixed batch", _adapters(333, 2560, 10576, 32, 24, dtype="f16", runs=7)),
        # in_proj of a long prefill of few requests
        case("adapters prompts", _adapters(16384, 2560, 10576, 16, 5, runs=3000)),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def some(*v):
        return v[rng.randrange(len(v))]

    op = some("attention", "attention", "attention_token", "group", "group_tokens", "adapters", "adapters")
    dt = some("bf16", "bf16", "f16", "f32")
    if op in ("attention", "attention_token"):
        share = some(1, 1, 2, 4)
        H = share * size(1, 32 // share)
        K, V = (some(64, 128, 128, rng.randrange(8, 257)) for _ in range(2))
        if op == "attention_token":
            return _attention_token(size(1, max(1, min(256, 33_000_000 // (H * K * V)))), H, K, V, share, dt, some("token", "token", "head"),
                                    some("f32", "f32", "bf16", "f16"))
        B = size(1, 8)
        T = size(1, max(1, min(32768, (33_000_000 if dt == "f32" else 67_000_000) // (B * H * max(K, V)))))
        return _attention(B, T, H, K, V, share, dt, some("token", "token", "head", "none"), some(False, True), some(False, True))
    if op == "group":
        groups = some(1, 4, 8, 16, 32)
        D = groups * size(4, 8192 // groups)
        return _group(size(1, min(32768, 67_000_000 // D)), D, groups, dt, some(False, True), some(False, True))
    if op == "group_tokens":
        groups = some(1, 8, 16, 32)
        D, B = groups * size(2, 2048 // groups), size(1, 16)
        return _group_tokens(B, size(1, min(16384, 33_000_000 // (B * D))), D, groups, dt, some(False, True), some(False, True))
    K, N, R = size(64, 8192), size(64, 16384), some(8, 16, 16, 32, 64)
    M = size(1, min(16384, 440_000_000_000 // (K * N)))
    return _adapters(M, K, N, R, size(1, max(1, min(64, K // R))), dt, some("codes", "rows"), size(1, 512) if M > 64 else 1)


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


def _decay(gen, kind, lead, H):
    """Log-decays: a gate's log-sigmoid, most of it near 1; or the constant slopes of heads, 1 - 2^-5 to 1 - 2^-9."""
    if kind == "none":
        return None
    if kind == "head":
        return torch.log1p(-torch.exp2(-5 - 4 * torch.rand(H, generator=gen, device="cuda")))
    return torch.nn.functional.logsigmoid(_randn(gen, *lead, H) + 3.0)


def _qkv(gen, lead, Hk, H, K, V, packed, dtype):
    """k of about unit length, as a layer norms it."""
    if not packed:
        return _randn(gen, *lead, Hk, K, dtype=dtype), _randn(gen, *lead, Hk, K, dtype=dtype) / math.sqrt(K), _randn(gen, *lead, H, V, dtype=dtype)
    wide = torch.zeros(*lead, 2 * Hk * K + 2 * H * V, device="cuda", dtype=dtype)
    q, k, v, _ = wide.split([Hk * K, Hk * K, H * V, H * V], -1)
    q, k, v = q.unflatten(-1, (Hk, K)), k.unflatten(-1, (Hk, K)), v.unflatten(-1, (H, V))
    q.copy_(_randn(gen, *q.shape, dtype=dtype))
    k.copy_(_randn(gen, *k.shape, dtype=dtype) / math.sqrt(K))
    v.copy_(_randn(gen, *v.shape, dtype=dtype))
    return q, k, v


def _codes(t):
    """Symmetric INT8 codes and scales of the rows, the codes' rows on 16-byte boundaries."""
    n, k = t.shape
    scale = t.abs().amax(1) / 127
    buf = torch.zeros(n, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    codes = buf[:, :k]
    codes.copy_(torch.round(t / scale.unsqueeze(1)).clamp(-127, 127))
    return codes, scale


def prepare(case, seed):
    c, gen = case, _gen(seed)
    op, dt = c["op"], DTYPES[c["dtype"]]
    s = dict(op=op, dtype=dt)
    if op == "attention":
        B, T, H, K, V = (c[n] for n in "BTHKV")
        s["q"], s["k"], s["v"] = _qkv(gen, (B, T), H // c["share"], H, K, V, c["packed"], dt)
        s["g"] = _decay(gen, c["decay"], (B, T), H)
        s["lengths"] = _lengths(gen, B, T) if c["ragged"] else None
        s["initial"] = _randn(gen, B, H, K, V) if c["ragged"] else None
    elif op == "attention_token":
        B, H, K, V = (c[n] for n in "BHKV")
        s["q"], s["k"], s["v"] = _qkv(gen, (B,), H // c["share"], H, K, V, False, dt)
        s["g"] = _decay(gen, c["decay"], (B,), H)
        S, s["slots"] = _slots(gen, B)
        s["state"] = _randn(gen, S, H, K, V, dtype=DTYPES[c["state"]])
    elif op in ("group", "group_tokens"):
        D = c["D"]
        lead = (c["rows"],) if op == "group" else (c["B"], c["T"])
        s["x"] = (_randn(gen, *lead, D) * 2 + _randn(gen, D)).to(dt)  # channels with means of their own
        s["groups"], s["silu"] = c["groups"], c["silu"]
        s["weight"], s["bias"] = torch.rand(D, generator=gen, device="cuda") + 0.5, _randn(gen, D) * 0.1
        s["gate"] = s["lengths"] = None
        if c.get("gate"):
            wide = torch.zeros(*lead, 2 * D, device="cuda", dtype=dt)
            s["gate"] = wide[..., D:]
            s["gate"].copy_(_randn(gen, *lead, D, dtype=dt))
        if c.get("ragged"):
            s["lengths"] = _lengths(gen, c["B"], c["T"])
    else:
        M, K, N, R, L = (c[n] for n in "MKNRL")
        s["w"], s["w_scale"] = _codes(_randn(gen, N, K) / math.sqrt(K))
        s["bias"] = _randn(gen, N) * 0.1
        x = _heavy(gen, _randn(gen, M, K))
        if c["form"] == "codes":
            s["x"], s["x_scale"] = _codes(x)
        else:
            s["x"], s["x_scale"] = x.to(dt), None
        s["a"], s["b"] = (_randn(gen, L, R, K) / math.sqrt(K)).to(dt), (_randn(gen, L, N, R) / math.sqrt(R)).to(dt)
        s["scaling"] = torch.rand(L, generator=gen, device="cuda") * 0.5 + 0.1
        runs = -(-M // c["runs"])  # one in eight requests has no adapter
        which = torch.randint(-max(1, L // 8), L, (runs,), generator=gen, device="cuda").clamp(min=-1)
        s["adapters"] = which.repeat_interleave(c["runs"])[:M].to(torch.int32)
    return s


EPS = 1e-5
CHUNK = 64


# --------------------------------------------------------------------------------------------------- the plain forms
def _silu(x):
    return x / (1 + torch.exp(-x))


def _inside(lengths, B, T):
    """[B, T]: tokens that belong to their sequence."""
    t = torch.arange(T, device="cuda")
    return torch.full((B,), T, device="cuda").unsqueeze(1) > t if lengths is None else lengths.unsqueeze(1) > t


def _plain_attention(s):
    """Chunks of 64 tokens: inside one the products with all earlier keys, decayed; between them the states, whose carry is
    composed over all chunks at once (after the round of width w, (a, h) of a chunk is the composition of the 2 w chunks that
    end with it)."""
    B, T, H, V = s["v"].shape
    K = s["q"].shape[-1]
    NT = -(-T // CHUNK)
    inside = _inside(s["lengths"], B, T)

    def chunks(t, lead):  # [B, H, NT, CHUNK, ..], zeros behind each sequence
        t = torch.where(inside.view(B, T, *[1] * (t.dim() - 2)), t, 0)
        t = torch.cat([t, t.new_zeros(B, NT * CHUNK - T, *t.shape[2:])], 1) if NT * CHUNK > T else t
        return t.repeat_interleave(H // lead, 2).unflatten(1, (NT, CHUNK)).movedim(3, 1)

    q, k, v = (chunks(s[n].float(), s[n].shape[2]) for n in "qkv")
    g = torch.zeros(H, device="cuda") if s["g"] is None else s["g"]
    G = chunks(g.double().expand(B, T, H), H).cumsum(-1)  # [B, H, NT, CHUNK]
    below = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    weights = torch.exp(torch.where(below, G.unsqueeze(-1) - G.unsqueeze(-2), -math.inf).float())
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * weights, v)
    del weights
    h = torch.matmul((k * torch.exp(G[..., -1:] - G).float().unsqueeze(-1)).transpose(-1, -2), v)  # what a chunk adds
    a = torch.exp(G[..., -1]).float()[..., None, None]
    first = torch.zeros(B, H, K, V, device="cuda") if s["initial"] is None else s["initial"]
    h[:, :, 0] += a[:, :, 0] * first
    width = 1
    while width < NT:
        h = torch.cat([h[:, :, :width], h[:, :, width:] + a[:, :, width:] * h[:, :, :-width]], 2)
        a = torch.cat([a[:, :, :width], a[:, :, width:] * a[:, :, :-width]], 2)
        width *= 2
    entering = torch.cat([first.unsqueeze(2), h[:, :, :-1]], 2)
    o = (o + torch.exp(G).float().unsqueeze(-1) * torch.matmul(q, entering)) * K**-0.5
    o = o.movedim(1, 3).flatten(1, 2)[:, :T]
    return {"o": torch.where(inside[..., None, None], o, 0.0).to(s["dtype"]), "state": h[:, :, -1].contiguous()}


def _plain_attention_token(s):
    at, v = s["slots"].long(), s["v"].float()
    q, k = (s[n].float().repeat_interleave(v.shape[1] // s[n].shape[1], 1) for n in "qk")
    a = torch.exp(s["g"]).expand(v.shape[:2])
    h = s["state"][at].float() * a[..., None, None] + k.unsqueeze(-1) * v.unsqueeze(-2)
    s["state"][at] = h.to(s["state"].dtype)
    o = (q.unsqueeze(-1) * h).sum(-2) * q.shape[-1]**-0.5
    return {"o": o.to(s["dtype"]), "state": s["state"]}


def _plain_group(s):
    x = s["x"]
    B, D, C = x.shape[0], x.shape[-1], x.shape[-1] // s["groups"]
    x = x.double().reshape(B, -1, s["groups"], C)
    T = x.shape[1]
    inside = _inside(s["lengths"], B, T)[..., None, None]
    n = inside.sum(1, keepdim=True).clamp(min=1) * C
    x = torch.where(inside, x, 0.0)
    mean = x.sum((1, 3), keepdim=True) / n
    x = torch.where(inside, x - mean, 0.0)
    y = (x * torch.rsqrt((x * x).sum((1, 3), keepdim=True) / n + EPS)).float().reshape(s["x"].shape) * s["weight"] + s["bias"]
    if s["silu"]:
        y = _silu(y)
    if s["gate"] is not None:
        y = y * _silu(s["gate"].float())
    inside = inside.reshape(B, T, 1) if s["x"].dim() == 3 else inside.reshape(B, 1)
    return {"y": torch.where(inside, y, 0.0).to(s["dtype"])}


def _plain_quantise(x):
    """Codes as numbers, half away from zero, and their scale."""
    scale = x.abs().amax(1, keepdim=True) / 127
    y = x * (1 / scale)
    return torch.trunc(torch.clamp(y, -127, 127) + torch.copysign(torch.full_like(y, 0.5), y)), scale


def _plain_adapters(s):
    """The low-rank rows of all adapters side by side, each token's own kept: one product with all of them stacked."""
    codes, scale = _plain_quantise(s["x"].float()) if s["x_scale"] is None else (s["x"].float(), s["x_scale"].unsqueeze(1))
    x = s["x"].float() if s["x_scale"] is None else codes * scale
    L, R, K = s["a"].shape
    t = torch.matmul(x, s["a"].float().view(L * R, K).t()).view(-1, L, R)
    mine = s["adapters"].unsqueeze(1) == torch.arange(L, device="cuda")
    t = torch.where(mine.unsqueeze(-1), t * s["scaling"].view(L, 1), 0.0)
    low = torch.matmul(t.flatten(1), s["b"].float().transpose(1, 2).reshape(L * R, -1))
    y = torch.matmul(codes, s["w"].float().t()) * scale * s["w_scale"] + s["bias"] + low
    return {"y": y.to(s["dtype"])}


PLAIN = {"attention": _plain_attention, "attention_token": _plain_attention_token, "group": _plain_group, "group_tokens": _plain_group,
         "adapters": _plain_adapters}


# ------------------------------------------------------------------------------------------------------- the calls
def _own(s):
    from linquant_b200.kernels import layer

    op = s["op"]
    if op == "attention":
        o, state = layer.linear_attention_fwd(s["q"], s["k"], s["v"], s["g"], initial_state=s["initial"], lengths=s["lengths"],
                                              output_final_state=True)
        return {"o": o, "state": state}
    if op == "attention_token":
        return {"o": layer.linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["g"], slots=s["slots"]), "state": s["state"]}
    if op in ("group", "group_tokens"):
        return {"y": layer.group_norm_fwd(s["x"], s["groups"], s["weight"], s["bias"], activation="silu" if s["silu"] else None,
                                          gate=s["gate"], eps=EPS, over_tokens=op == "group_tokens", lengths=s["lengths"])}
    return {"y": layer.lora_linear_fwd(s["x"], s["w"], s["w_scale"], s["a"], s["b"], s["adapters"], scaling=s["scaling"],
                                       x_scale=s["x_scale"], bias=s["bias"], out_dtype=s["dtype"])}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, op, e = case, case["op"], SIZE[case["dtype"]]
    if op in ("attention", "attention_token"):
        n, token = c["B"] * c["H"], op == "attention_token"
        tokens = c["B"] * (1 if token else c["T"])
        decay = 4 * (tokens * c["H"] if c["decay"] == "token" else c["H"])
        rows = e * tokens * (2 * c["H"] // c["share"] * c["K"] + 2 * c["H"] * c["V"])
        state = n * c["K"] * c["V"] * (2 * SIZE[c["state"]] if token else 8 if c["ragged"] else 4)
        # decay and outer product of the state, and its read-out, token by token
        return {"bytes": rows + decay + state, "flops": tokens * c["H"] * c["K"] * c["V"] * 5.0}
    if op in ("group", "group_tokens"):
        n = (c["rows"] if op == "group" else c["B"] * c["T"]) * c["D"]
        return {"bytes": n * e * (3 if c.get("gate") else 2) + 8 * c["D"], "flops": 10.0 * n}
    M, K, N, R, L = (c[n] for n in "MKNRL")
    used = min(L, -(-M // c["runs"]))
    rows = M * K + 4 * M if c["form"] == "codes" else e * M * K
    return {"bytes": rows + N * K + e * M * N + 12 * N + e * used * R * (K + N), "flops": 2.0 * M * K * N + 2.0 * M * R * (K + N)}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_attention(s):
    B, T, H, V = s["v"].shape
    K, rep = s["q"].shape[-1], H // s["q"].shape[2]
    h = torch.zeros(B, H, K, V, device="cuda", dtype=torch.float64) if s["initial"] is None else s["initial"].double()
    o = torch.zeros(B, T, H, V, device="cuda", dtype=torch.float64)
    decay = torch.ones(B, T, H, 1, 1, device="cuda", dtype=torch.float64)
    if s["g"] is not None:
        decay = torch.exp(s["g"].double()).expand(B, T, H)[..., None, None]
    live = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"]
    on = live.unsqueeze(1) > torch.arange(T, device="cuda")
    for t in range(T):
        k, q = (s[n][:, t].double().repeat_interleave(rep, 1) for n in ("k", "q"))
        h2 = torch.addcmul(decay[:, t] * h, k.unsqueeze(-1), s["v"][:, t].double().unsqueeze(-2))
        h = h2 if s["lengths"] is None else torch.where(on[:, t, None, None, None], h2, h)
        o[:, t] = torch.matmul(q.unsqueeze(-2), h).squeeze(-2)
    return {"o": torch.where(on[..., None, None], o / math.sqrt(K), 0.0), "state": h}


def _exact_attention_token(s):
    at, state, rep = s["slots"].long(), s["state"].double(), s["v"].shape[1] // s["q"].shape[1]
    k, q = (s[n].double().repeat_interleave(rep, 1) for n in ("k", "q"))
    decay = torch.exp(s["g"].double()).expand(s["v"].shape[:2])
    h = decay[..., None, None] * state[at] + torch.einsum("bhk,bhv->bhkv", k, s["v"].double())
    state[at] = h
    return {"o": torch.einsum("bhk,bhkv->bhv", q, h) / math.sqrt(q.shape[-1]), "state": state}


def _exact_group(s):
    x, D = s["x"].double(), s["x"].shape[-1]
    per_row = x.dim() == 2
    y = torch.zeros_like(x)
    for part in range(1 if per_row else x.shape[0]):
        n = x.shape[1] if per_row or s["lengths"] is None else int(s["lengths"][part])
        v = x.unsqueeze(1) if per_row else x[part:part + 1, :n]
        v = v.unflatten(-1, (s["groups"], D // s["groups"]))
        if v.numel():
            v = (v - v.mean((1, 3), keepdim=True)) / torch.sqrt(v.var((1, 3), keepdim=True, unbiased=False) + EPS)
            v = v.flatten(-2) * s["weight"].double() + s["bias"].double()
            v = v * torch.sigmoid(v) if s["silu"] else v
            if per_row:
                y = v[:, 0]
            else:
                y[part, :n] = v[0]
    if s["gate"] is not None:
        gate = s["gate"].double()
        y = y * gate * torch.sigmoid(gate)
    return {"y": y}


def _exact_adapters(s):
    if s["x_scale"] is None:
        x = s["x"].double()
        scale = x.abs().amax(1, keepdim=True) / 127
        v = x / scale
        base = torch.sign(v) * torch.floor(v.abs() + 0.5) * scale
    else:
        x = base = s["x"].double() * s["x_scale"].double().unsqueeze(1)
    y = torch.matmul(base, (s["w"].double() * s["w_scale"].double().unsqueeze(1)).t()) + s["bias"].double()
    for i in range(s["a"].shape[0]):
        rows = (s["adapters"] == i).nonzero()[:, 0]
        if rows.numel():
            low = torch.matmul(x[rows], s["a"][i].double().t()) * s["scaling"][i].double()
            y[rows] += torch.matmul(low, s["b"][i].double().t())
    return {"y": y}


EXACT = {"attention": _exact_attention, "attention_token": _exact_attention_token, "group": _exact_group, "group_tokens": _exact_group,
         "adapters": _exact_adapters}


def exact(case, seed):
    s = prepare(case, seed)
    return EXACT[s["op"]](s)
