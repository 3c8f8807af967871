"""The work that the linear attention with decay, its form for single tokens and the gated feed-forward block are timed on.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw(rng)` another one of the same ranges, `prepare(case, seed)` what the
program holds before the call, `run(state)` one pass (the framework's operators where `own` is true, elementary torch operations where it is
not), `work(case)` the bytes and operations of a pass, `exact(case, seed)` what a pass returns, from the definition in 64 bits.

Value distributions: queries, keys, values, tokens and upstream gradients N(0, 1); log decays -dt a with dt = softplus(N(0, 1) + b), b the
inverse softplus of a step size log-uniform in [1e-3, 1e-1] per head, and a uniform in [1, 16] per head; weights N(0, 0.02); biases N(0, 0.1).
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CHUNK = 64                          # tokens whose pairs the plain form writes out
# of a drawn case: bounds that keep it below the largest listed one
MOST_ROW_ELEMENTS = 1 << 25         # (image, token, head, wider of key and value)
MOST_STATE_ELEMENTS = 1 << 25       # (sequence, head, key, value)
MOST_PRODUCTS = 12544 * 512 * 2048  # (token, channel, hidden)


# ------------------------------------------------------------------------------------------------ the cases
def _attend(train, dtype, batch, length, groups, heads, keys, values, carried):
    return {"kind": "attend", "train": train, "dtype": dtype, "batch": batch, "length": length, "groups": groups, "heads": heads,
            "keys": keys, "values": values, "carried": carried}


def _token(dtype, batch, groups, heads, keys, values):
    return {"kind": "token", "dtype": dtype, "batch": batch, "groups": groups, "heads": heads, "keys": keys, "values": values}


def _feed(train, dtype, tokens, channels, hidden, act, biases):
    return {"kind": "feed", "train": train, "dtype": dtype, "tokens": tokens, "channels": channels, "hidden": hidden, "act": act, "biases": biases}


def listed():
    return [
        # one image in the last stage of a classifier, 4 routes of 192 channels: the smallest call there is
        {"name": "attend_one_image", **_attend(False, "bf16", 1, 49, 4, 24, 64, 32, False)},
        # a batch of images in the second stage, inference in fp16, keys and queries of a route shared by its heads
        {"name": "attend_images", **_attend(False, "f16", 16, 784, 4, 24, 64, 32, False)},
        # one long prompt that continues from a state and leaves one, a length that no chunk divides
        {"name": "attend_long", **_attend(False, "bf16", 1, 16385, 16, 16, 128, 128, True)},
        # training step at the first stage of a classifier: 4 routes of 96 channels
        {"name": "attend_train_images", **_attend(True, "bf16", 16, 3136, 4, 12, 64, 32, False)},
        # training step on sequences, wide heads of their own keys
        {"name": "attend_train_heads", **_attend(True, "bf16", 2, 4096, 16, 16, 128, 128, False)},
        # training in fp32, ragged length, state carried in and out
        {"name": "attend_train_f32", **_attend(True, "f32", 4, 1001, 8, 8, 32, 64, True)},
        # one token of one sequence
        {"name": "token_one", **_token("bf16", 1, 4, 24, 64, 32)},
        # one token of each of 128 sequences
        {"name": "token_batch", **_token("bf16", 128, 16, 16, 128, 128)},
        # the block on one token
        {"name": "feed_one_token", **_feed(False, "bf16", 1, 768, 2048, "silu", False)},
        # 64 images of 14 x 14 tokens, 512 channels and four times as many hidden ones
        {"name": "feed_images", **_feed(False, "bf16", 12544, 512, 2048, "gelu", True)},
        # training step on 32 images of 14 x 14 tokens
        {"name": "feed_train", **_feed(True, "bf16", 6272, 384, 1536, "gelu", True)},
        # training in fp32, ragged number of tokens
        {"name": "feed_train_f32", **_feed(True, "f32", 1001, 192, 768, "silu", True)},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "token", "feed", "feed"))
    if kind in ("attend", "token"):
        groups = rng.choice((1, 2, 4, 4, 8, 16))
        heads = groups * rng.choice((1, 1, 2, 3, 6))
        keys, values = rng.choice((16, 32, 48, 64, 64, 96, 128, 128)), rng.choice((16, 24, 32, 64, 64, 80, 128, 128))
        if kind == "token":
            batch = _log_int(rng, 1, min(512, max(1, MOST_STATE_ELEMENTS // (heads * keys * values))))
            return _token(rng.choice(("bf16", "bf16", "f16", "f32")), batch, groups, heads, keys, values)
        train, dtype = rng.random() < 0.5, rng.choice(("bf16", "bf16", "f16", "f32"))
        wide = heads * max(keys, values) * (SIZE[dtype] // 2) * (2 if train else 1)
        length = _log_int(rng, 1, min(16384, MOST_ROW_ELEMENTS // wide))
        batch = _log_int(rng, 1, min(64, max(1, MOST_ROW_ELEMENTS // (wide * length))))
        return _attend(train, dtype, batch, length, groups, heads, keys, values, rng.random() < 0.4)
    train, dtype = rng.random() < 0.5, rng.choice(("bf16", "bf16", "f16", "f32"))
    channels = 8 * _log_int(rng, 4, 128)
    hidden = int(channels * rng.choice((2.0, 8.0 / 3.0, 4.0))) // 8 * 8
    most = MOST_PRODUCTS // (channels * hidden) // (3 if train else 1) // (8 if dtype == "f32" else 1)
    return _feed(train, dtype, _log_int(rng, 1, max(1, min(16384, most))), channels, hidden, rng.choice(("silu", "gelu")), rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(dtype)


def _log_decay(g, batch, tokens, heads):
    dt = torch.exp(torch.rand(heads, device="cuda", generator=g) * math.log(100.0) + math.log(1e-3))
    rate = 1.0 + 15.0 * torch.rand(heads, device="cuda", generator=g)
    raw = torch.randn((batch, tokens, heads), device="cuda", generator=g) + torch.log(torch.expm1(dt))
    return -F.softplus(raw) * rate


def prepare(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    if case["kind"] == "feed":
        M, C, Hd = case["tokens"], case["channels"], case["hidden"]
        t = {"x": _randn(g, (M, C), dt), "w1": _randn(g, (2 * Hd, C), dt, 0.02), "w2": _randn(g, (C, Hd), dt, 0.02)}
        if case["biases"]:
            t["b1"], t["b2"] = _randn(g, (2 * Hd,), dt, 0.1), _randn(g, (C,), dt, 0.1)
        upstream = [_randn(g, (M, C), dt)] if case["train"] else []
    else:
        B, L = case["batch"], case.get("length", 1)
        G, H, dk, dv = case["groups"], case["heads"], case["keys"], case["values"]
        t = {"q": _randn(g, (B, L, G, dk), dt), "k": _randn(g, (B, L, G, dk), dt), "v": _randn(g, (B, L, H, dv), dt),
             "log_decay": _log_decay(g, B, L, H)}
        if case["kind"] == "token":
            t = {n: x[:, 0].contiguous() for n, x in t.items()}
            t["state"] = _randn(g, (B, H, dk, dv))
            return {"case": case, "t": t, "state_out": torch.empty_like(t["state"])}
        if case["carried"]:
            t["initial_state"] = _randn(g, (B, H, dk, dv))
        upstream = []
        if case["train"]:
            upstream = [_randn(g, (B, L, H, dv), dt)] + ([_randn(g, (B, H, dk, dv))] if case["carried"] else [])
    if case["train"]:
        t = {n: x.requires_grad_() for n, x in t.items()}
    return {"case": case, "t": t, "upstream": upstream}


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_attention(q, k, v, log_decay, initial_state=None):
    """Chunks of tokens: the pairs inside a chunk written out, the states in front of the chunks by one product with the decays between them."""
    B, L, G, dk = q.shape
    H, dv = v.shape[2:]
    n = -(-L // CHUNK)
    cut = lambda x: F.pad(x, (0, 0) * (x.dim() - 2) + (0, n * CHUNK - L)).unflatten(1, (n, CHUNK)).transpose(2, 3)      # (B, n, heads, CHUNK, ..)
    q, k = (cut(x).repeat_interleave(H // G, 2) for x in (q, k))
    v, total = cut(v), torch.cumsum(cut(log_decay[..., None])[..., 0].double(), -1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    between = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~low, -math.inf)).float()
    inside = (q @ k.transpose(-1, -2) * between) @ v
    added = (k * torch.exp(total[..., -1:] - total).float()[..., None]).transpose(-1, -2) @ v                          # (B, n, H, dk, dv)
    ends = F.pad(torch.cumsum(total[..., -1], 1).transpose(1, 2), (1, 0))                                               # (B, H, n + 1)
    before = torch.ones(n + 1, n, dtype=torch.bool, device=q.device).tril(-1)
    carry = torch.exp((ends[..., :, None] - ends[..., None, 1:]).masked_fill(~before, -math.inf)).float()
    states = (carry @ added.transpose(1, 2).flatten(3)).unflatten(3, (dk, dv))                                          # (B, H, n + 1, dk, dv)
    if initial_state is not None:
        states = states + torch.exp(ends).float()[..., None, None] * initial_state[:, :, None]
    across = torch.exp(total).float()[..., None] * (q @ states[:, :, :-1].transpose(1, 2))
    o = (inside + across).transpose(2, 3).flatten(1, 2)[:, :L] * dk ** -0.5
    return o, states[:, :, -1]


def _plain_token(q, k, v, log_decay, state):
    r = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    state = torch.exp(log_decay)[..., None, None] * state + k[..., :, None] * v[..., None, :]
    return (q[..., :, None] * state).sum(-2) * q.shape[-1] ** -0.5, state


def _plain_feed(act, x, w1, w2, b1=None, b2=None):
    z = x @ w1.t()
    if b1 is not None:
        z = z + b1
    value, gate = z.chunk(2, -1)
    gate = gate * torch.sigmoid(gate) if act == "silu" else 0.5 * gate * (1.0 + torch.erf(gate * 0.5 ** 0.5))
    y = (value * gate) @ w2.t()
    return y if b2 is None else y + b2


def _plain(s):
    case, t = s["case"], s["t"]
    f = {n: x.detach().float() for n, x in t.items()}
    if case["kind"] == "token":
        o, state = _plain_token(**f)
        return o.to(DTYPES[case["dtype"]]), state
    if case["train"]:
        f = {n: x.requires_grad_() for n, x in f.items()}
    outs = [_plain_feed(case["act"], **f)] if case["kind"] == "feed" else list(_plain_attention(**f))[:2 if case["carried"] else 1]
    types = [DTYPES[case["dtype"]], torch.float32]
    if not case["train"]:
        return [x.to(d) for x, d in zip(outs, types)]
    grads = torch.autograd.grad(outs, list(f.values()), [u.float() for u in s["upstream"]])
    return [x.detach().to(d) for x, d in zip(outs, types)], {n: d.to(t[n].dtype) for n, d in zip(f, grads)}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if not own:
        return _plain(s)
    import vmamba_b200 as vb
    case, t = s["case"], s["t"]
    if case["kind"] == "token":
        return vb.linear_attention_step(**t, state_out=s["state_out"])
    if case["kind"] == "feed":
        outs = [vb.gated_mlp_fn(**t, act=case["act"])]
    elif case["carried"]:
        outs = list(vb.linear_attention_fn(**t, return_final_state=True))
    else:
        outs = [vb.linear_attention_fn(**t)]
    if not case["train"]:
        return outs
    grads = torch.autograd.grad(outs, list(t.values()), s["upstream"])
    return [x.detach() for x in outs], dict(zip(t, grads))


def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "feed":
        M, C, Hd = case["tokens"], case["channels"], case["hidden"]
        weights = 3 * C * Hd + (2 * Hd + C if case["biases"] else 0)
        if not case["train"]:
            return {"bytes": e * (2 * M * C + weights), "flops": 6 * M * C * Hd}
        return {"bytes": e * (4 * M * C + 2 * weights), "flops": 18 * M * C * Hd}
    B, L = case["batch"], case.get("length", 1)
    G, H, dk, dv = case["groups"], case["heads"], case["keys"], case["values"]
    rows = B * L * (e * (2 * G * dk + 2 * H * dv) + 4 * H)
    state = 4 * B * H * dk * dv
    flops = 4 * B * L * H * dk * dv                     # the recurrence: the state's update and its product with the query
    if case["kind"] == "token":
        return {"bytes": rows + 2 * state, "flops": flops}
    carried = 2 * state if case["carried"] else 0
    if not case["train"]:
        return {"bytes": rows + carried, "flops": flops}
    more = B * L * (e * (2 * G * dk + 2 * H * dv) + 4 * H)      # the upstream gradient, and the gradients of q, k, v and the decays
    return {"bytes": rows + more + 2 * carried, "flops": 3 * flops}


# ------------------------------------------------------------------------------------------------ definition in 64 bits
def _steps(q, k, v, g, scale, state, upstream, last):
    """Token by token.  Gradients: the state's own runs backwards; a decay's is the sum over what crosses it, which telescopes into what the
    queries behind it receive less what the keys behind it receive (64 bits bear the cancellation)."""
    L = q.shape[1]
    keep = torch.exp(g)
    o, dq = torch.empty_like(v), torch.empty_like(q)
    for t in range(L):
        state = keep[:, t, :, None, None] * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * torch.matmul(q[:, t, :, None, :], state)[..., 0, :]
        if upstream is not None:
            dq[:, t] = scale * torch.matmul(state, upstream[:, t, :, :, None])[..., 0]
    if upstream is None:
        return o, state, None
    dstate = torch.zeros_like(state) if last is None else last
    crossing = (dstate * state).sum((-1, -2))
    dk, dv, dg = torch.empty_like(k), torch.empty_like(v), torch.empty_like(g)
    for t in range(L - 1, -1, -1):
        dstate = dstate + scale * q[:, t, :, :, None] * upstream[:, t, :, None, :]
        dk[:, t] = torch.matmul(dstate, v[:, t, :, :, None])[..., 0]
        dv[:, t] = torch.matmul(k[:, t, :, None, :], dstate)[..., 0, :]
        crossing = crossing + (q[:, t] * dq[:, t]).sum(-1) - (k[:, t] * dk[:, t]).sum(-1)
        dg[:, t] = crossing
        dstate = keep[:, t, :, None, None] * dstate
    return o, state, (dq, dk, dv, dg, dstate)


def exact(case, seed):
    s = prepare(case, seed)
    t = {n: x.detach().double() for n, x in s["t"].items()}
    if case["kind"] == "feed":
        bias = lambda n: t[n] if n in t else 0.0
        half = case["hidden"]
        value = torch.einsum("mc,hc->mh", t["x"], t["w1"][:half]) + (t["b1"][:half] if "b1" in t else 0.0)
        gate = torch.einsum("mc,hc->mh", t["x"], t["w1"][half:]) + (t["b1"][half:] if "b1" in t else 0.0)
        if case["act"] == "silu":
            one = 1.0 / (1.0 + torch.exp(-gate))
            bent, slope = gate * one, one * (1.0 + gate * (1.0 - one))
        else:
            one = 0.5 * torch.erfc(-gate / math.sqrt(2.0))
            bent, slope = gate * one, one + gate * torch.exp(-0.5 * gate * gate) / math.sqrt(2.0 * math.pi)
        hidden = value * bent
        y = torch.einsum("mh,ch->mc", hidden, t["w2"]) + bias("b2")
        if not case["train"]:
            return [y]
        dy = s["upstream"][0].double()
        dh = torch.einsum("mc,ch->mh", dy, t["w2"])
        dz = torch.cat((dh * bent, dh * value * slope), 1)
        grads = {"x": dz @ t["w1"], "w1": torch.einsum("mh,mc->hc", dz, t["x"]), "w2": torch.einsum("mc,mh->ch", dy, hidden)}
        if case["biases"]:
            grads["b1"], grads["b2"] = dz.sum(0), dy.sum(0)
        return [y], grads
    token = case["kind"] == "token"
    r, scale = case["heads"] // case["groups"], 1.0 / math.sqrt(case["keys"])
    if token:
        t = {n: x if n == "state" else x[:, None] for n, x in t.items()}
    start = t.get("state", t.get("initial_state"))
    if start is None:
        start = torch.zeros((case["batch"], case["heads"], case["keys"], case["values"]), dtype=torch.float64, device="cuda")
    up = [u.double() for u in s.get("upstream", [])] + [None, None]
    wide = lambda x: x.repeat_interleave(r, 2)
    o, state, grads = _steps(wide(t["q"]), wide(t["k"]), t["v"], t["log_decay"], scale, start, up[0], up[1])
    if token:
        return o[:, 0], state
    outs = [o, state] if case["carried"] else [o]
    if not case["train"]:
        return outs
    dq, dk, dv, dg, dstart = grads
    fold = lambda x: x.unflatten(2, (case["groups"], r)).sum(3)
    found = {"q": fold(dq), "k": fold(dk), "v": dv, "log_decay": dg}
    if case["carried"]:
        found["initial_state"] = dstart
    return outs, found
