"""Linear attention with a decay for each head against its recurrence in 64 bits, token by token, and autograd through it.

Tolerances.  Every product and sum of the operator is positive when all its inputs are, so the same recurrence on absolute values gives, for each
output and gradient, the sum M of the magnitudes of its terms.  Against it count
  * the rounding of the result, half a step of its type relative to its value (none for fp32 beside the next);
  * what a kernel rounds for its matrix products: weights of pairs and states, once, half a step of the form that they take (bf16 2^-8, tf32 2^-11
    beside fp16, 2^-22 beside fp32: two tf32 pieces and the product of the second ones), for results of the inputs' type.  At most two such roundings meet in
    a term (its pair weight, or the state, which is itself a sum of products of two pieces);
  * for fp32 results two pieces: 2^-16 beside bf16, 2^-22 beside the others, at most three in a term (two states, one of them rounded again);
  * fp32 sums of up to 128 + 64 terms and exponentials of 2^-22: 2^-16 of M covers them (192 roundings of 2^-24).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FORM = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -22}
PIECES = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 2.0 ** -22}
SUMS = 2.0 ** -16
NAMES = ("q", "k", "v", "log_decay", "initial_state")


@pytest.fixture(scope="module")
def vb():
    import vmamba_b200
    return vmamba_b200


def recurrence(q, k, v, g, s0, scale):
    r = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
    S, out = s0, []
    for t in range(v.shape[1]):
        S = torch.exp(g[:, t])[..., None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(scale * (q[:, t, :, :, None] * S).sum(-2))
    return torch.stack(out, 1), S


def make(B, L, G, H, dk, dv, dtype, seed=0, decay=0.3):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)      # noqa: E731
    t = {"q": rnd(B, L, G, dk).to(dtype), "k": rnd(B, L, G, dk).to(dtype), "v": rnd(B, L, H, dv).to(dtype),
         "log_decay": -decay * torch.rand((B, L, H), generator=g) ** 4, "initial_state": rnd(B, H, dk, dv)}
    up = [rnd(B, L, H, dv).to(dtype), rnd(B, H, dk, dv)]
    return {n: x.cuda() for n, x in t.items()}, [u.cuda() for u in up]


def reference(t, up, scale, absolute=False):
    """out, state and the gradients in NAMES order, in 64 bits."""
    f = {n: (x.detach().double().abs() if absolute and n != "log_decay" else x.detach().double()).requires_grad_() for n, x in t.items()}
    o, S = recurrence(f["q"], f["k"], f["v"], f["log_decay"], f["initial_state"], scale)
    u = [x.double().abs() if absolute else x.double() for x in up]
    grads = torch.autograd.grad([o, S], [f[n] for n in NAMES], u)
    return [o.detach(), S.detach(), *grads]


def run(vb, t, up, scale=None):
    leaves = {n: x.detach().requires_grad_() for n, x in t.items()}
    o, S = vb.linear_attention_fn(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], scale, leaves["initial_state"], return_final_state=True)
    grads = torch.autograd.grad([o, S], [leaves[n] for n in NAMES], up)
    return [o.detach(), S.detach(), *grads]


def per_chunk(x):
    """(B, L, H): the sum over the 64 tokens of a token's chunk."""
    L = x.shape[1]
    n = -(-L // 64)
    s = torch.nn.functional.pad(x, (0, 0, 0, n * 64 - L)).unflatten(1, (n, 64)).sum(2)
    return s.repeat_interleave(64, 1)[:, :L]


def compare(got, ref, mag, dtype, t, scale):
    names = ("out", "final_state", *NAMES)
    r = t["v"].shape[2] // t["q"].shape[2]
    for name, x, y, m in zip(names, got, ref, mag):
        assert x.shape == y.shape, name
        if name in ("out", "q", "k", "v"):
            assert x.dtype == dtype
            tol = HALF[dtype] * y.abs() + (2 * FORM[dtype] + SUMS) * m
        else:
            assert x.dtype == torch.float32
            tol = (3 * PIECES[dtype] + SUMS) * m
            if name == "log_decay":     # sums over the pairs of a chunk cancel where they cross nothing: their fp32 roundings stay
                heads = lambda z: z.repeat_interleave(r, 2)      # noqa: E731
                q, k = heads(t["q"].double().abs()), heads(t["k"].double().abs())
                # magnitudes of q . dq and k . dk of a head are at most those of its group
                tol = tol + 2.0 ** -18 * per_chunk((q * heads(mag[2])).sum(-1) + (k * heads(mag[3])).sum(-1))
        tol = tol + 1e-30 + (2.0 ** -25 if dtype == torch.float16 and x.dtype == dtype else 0)      # half a step of fp16's smallest numbers
        err = (x.double() - y).abs()
        worst, rel = (err / tol).max().item(), (err.norm() / y.norm().clamp(min=1e-30)).item()
        print(f"{name}: {worst:.3f} of the tolerance, relative error {rel:.2e}")
        assert torch.isfinite(x).all() and worst <= 1, (name, worst)
        # The bound above is the worst case of every term.  Roundings of random data are independent: each has a root mean square of at most
        # 1 / sqrt(3) of half a step of what it rounds, and the terms' own signs are as random as the result's, so that three of them come to
        # half a step of its norm; the sums' own, of random sign too, to 2^-19.
        most = HALF[dtype] if x.dtype == dtype and dtype != torch.float32 else 2.0 ** -19 + 3 ** 0.5 * PIECES[dtype]
        assert x.numel() < 1000 or rel <= most, (name, rel)


SHAPES = [  # B, L, G, H, dk, dv
    (1, 1, 1, 1, 16, 16), (2, 2, 2, 4, 8, 24), (1, 63, 1, 2, 32, 64), (2, 64, 4, 4, 64, 32), (1, 65, 2, 6, 64, 64), (1, 200, 1, 1, 128, 128),
    (3, 130, 2, 2, 50, 37), (1, 129, 1, 3, 1, 1), (1, 70, 1, 1, 33, 128), (1, 66, 1, 2, 100, 65), (1, 1100, 1, 2, 32, 16), (1, 1025, 1, 1, 48, 80),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_recurrence(vb, shape, dtype):
    t, up = make(*shape, dtype)
    scale = shape[4] ** -0.5
    compare(run(vb, t, up), reference(t, up, scale), reference(t, up, scale, True), dtype, t, scale)


LONG = [  # B, L, G, H, dk, dv: long bf16 sequences, the kernels of the 5th-generation tensor cores
    (1, 193, 1, 1, 128, 128), (2, 257, 1, 3, 72, 128), (1, 320, 2, 2, 128, 40), (1, 519, 1, 2, 64, 64), (2, 640, 2, 4, 40, 56), (1, 831, 1, 1, 8, 72), (3, 385, 1, 2, 96, 96),
]


@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sequences(vb, shape):
    t, up = make(*shape, torch.bfloat16, decay=0.05)
    scale = shape[4] ** -0.5
    compare(run(vb, t, up), reference(t, up, scale), reference(t, up, scale, True), torch.bfloat16, t, scale)
    with torch.no_grad():                       # without the states that training keeps: chunks of twice as many tokens
        o, S = vb.linear_attention_fn(*(t[n] for n in NAMES[:4]), None, t["initial_state"], True)
    ref, mag = reference(t, up, scale), reference(t, up, scale, True)
    assert ((o - ref[0]).abs() <= HALF[torch.bfloat16] * ref[0].abs() + (2 * FORM[torch.bfloat16] + SUMS) * mag[0]).all()
    assert ((S - ref[1]).abs() <= (3 * PIECES[torch.bfloat16] + SUMS) * mag[1]).all()


def test_long_sequences_whose_rows_no_tile_reads(vb):
    """Strides of 0 and rows on any element take the walk, with the workspace of the shape."""
    B, L, H, d = 2, 300, 2, 128
    t, up = make(B, L, H, H, d, d, torch.bfloat16, decay=0.05)
    scale = d ** -0.5
    want = reference(t, up, scale), reference(t, up, scale, True)
    wide = torch.zeros(B, L, H, d + 3, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:1 + d] = t["v"]
    compare(run(vb, {**t, "v": wide[..., 1:1 + d]}, up), *want, torch.bfloat16, t, scale)
    same = {**t, "k": t["k"][:1].expand(B, L, H, d)}
    compare(run(vb, same, up), reference(same, up, scale), reference(same, up, scale, True), torch.bfloat16, same, scale)
    packed = torch.cat([t[n] for n in "qkv"], -1)
    three = {**t, "q": packed[..., :d], "k": packed[..., d:2 * d], "v": packed[..., 2 * d:]}
    compare(run(vb, three, up), *want, torch.bfloat16, t, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets(vb, dtype):
    """-inf, the type's lowest and merely large negative decays clear the state; a chunk whose decays run to thousands keeps the small ones exact."""
    t, up = make(2, 200, 2, 2, 32, 32, dtype, decay=0.01)
    g = t["log_decay"]
    g[0, 10], g[0, 64], g[1, 130, 0] = -float("inf"), -3e38, -1e4
    g[0, 100:131] = -float("inf")
    g[1, 20:40] = -float("inf")
    scale = 0.3
    ref = reference(t, up, scale)
    # autograd through exp(-inf) multiplies by zero, as the operator does
    assert all(torch.isfinite(x).all() for x in ref)
    compare(run(vb, t, up, scale), ref, reference(t, up, scale, True), dtype, t, scale)
    before = {n: x.clone() for n, x in t.items()}
    before["v"][0, :100] = 7.0                  # another story in front of a reset
    before["initial_state"][0] = 3.0
    a, b = run(vb, t, up, scale), run(vb, before, up, scale)
    assert torch.equal(a[0][0, 130:], b[0][0, 130:]) and torch.equal(a[1][0], b[1][0])
    assert (a[5][0, 10] == 0).all() and (a[5][1, 20:40] == 0).all()        # nothing crosses a reset


@pytest.mark.parametrize("layout", ["packed", "odd", "heads_first", "broadcast"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(vb, layout, dtype):
    B, L, H, d = 2, 130, 4, 32
    t, up = make(B, L, H, H, d, d, dtype)
    if layout == "packed":                       # one projection's output, rows of queries, keys and values side by side
        x = torch.cat([t[n] for n in "qkv"], -1)
        t["q"], t["k"], t["v"] = x[..., :d], x[..., d:2 * d], x[..., 2 * d:]
    elif layout == "odd":                        # rows that start on any element
        for n in "qkv":
            x = torch.zeros(B, L, H, d + 5, dtype=dtype, device="cuda")
            x[..., 3:3 + d] = t[n]
            t[n] = x[..., 3:3 + d]
        up[0] = torch.cat([up[0], up[0]], -1)[..., d - 1:2 * d - 1]
    elif layout == "heads_first":
        for n in "qkv":
            t[n] = t[n].transpose(1, 2).contiguous().transpose(1, 2)
        t["log_decay"] = t["log_decay"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
        up[0] = up[0].transpose(1, 2).contiguous().transpose(1, 2)
        t["initial_state"] = t["initial_state"].transpose(2, 3).contiguous().transpose(2, 3)
    else:                                        # the same queries for all sequences and heads, the last dimension with a stride of 0
        t["q"] = t["q"][:1, :, :1].expand(B, L, H, d)
        t["k"] = t["k"][..., :1].expand(B, L, H, d)
        up[0] = up[0][..., :1].expand(B, L, H, d)
    scale = d ** -0.5
    compare(run(vb, t, up), reference(t, up, scale), reference(t, up, scale, True), dtype, t, scale)


def test_decays_that_tokens_share(vb):
    t, up = make(3, 150, 2, 4, 16, 16, torch.float32)
    rate = -torch.tensor([0.001, 0.01, 0.1, 1.0], device="cuda")
    leaf, full = rate.clone().requires_grad_(), rate.expand(3, 150, 4).contiguous().requires_grad_()
    o1 = vb.linear_attention_fn(t["q"], t["k"], t["v"], leaf)
    o2 = vb.linear_attention_fn(t["q"], t["k"], t["v"], full)
    assert torch.equal(o1, o2)
    g1, = torch.autograd.grad(o1, leaf, up[0])
    g2, = torch.autograd.grad(o2, full, up[0])
    assert g1.shape == (4,) and torch.allclose(g1, g2.sum((0, 1)), rtol=450 * 2.0 ** -24, atol=450 * 2.0 ** -24 * g2.abs().sum((0, 1)).max().item())
    half = vb.linear_attention_fn(t["q"], t["k"], t["v"], rate.bfloat16())
    assert torch.equal(half, vb.linear_attention_fn(t["q"], t["k"], t["v"], rate.bfloat16().float()))


def test_gradients_against_differences(vb):
    """fp32; the loss is linear in q, k, v and the initial state one at a time, so that central differences of any step are exact but for
    the roundings of the two losses; in the decays a step of 2^-7 leaves the third derivative, bounded by the magnitudes at decays 2^-7 higher."""
    B, L, G, H, dk, dv = 1, 90, 1, 2, 16, 8
    t, up = make(B, L, G, H, dk, dv, torch.float32)
    got = dict(zip(("o", "S", *NAMES), run(vb, t, up)))

    def loss(x):
        o, S = vb.linear_attention_fn(x["q"], x["k"], x["v"], x["log_decay"], None, x["initial_state"], True)
        return (o.double() * up[0].double()).sum() + (S.double() * up[1].double()).sum()

    mag = reference(t, up, dk ** -0.5, True)
    size = (mag[0] * up[0].abs()).sum() + (mag[1] * up[1].abs()).sum()
    gen = torch.Generator().manual_seed(5)
    for name in NAMES:
        d = torch.randn(t[name].shape, generator=gen).sign().cuda()
        e = 2.0 ** -7 if name == "log_decay" else 0.5
        plus, minus = ({**t, name: t[name] + s * e * d} for s in (1, -1))
        diff = (loss(plus) - loss(minus)) / (2 * e)
        want = (got[name].double() * d.double()).sum()
        moved = {**t, name: t[name].abs() + e} if name != "log_decay" else {**t, name: t[name] + e}
        m2 = reference(moved, up, dk ** -0.5, True)
        noise = (SUMS + 3 * 2.0 ** -22) * ((m2[0] * up[0].abs()).sum() + (m2[1] * up[1].abs()).sum() + size) / e
        # third derivative along signs: at most the loss of magnitudes times the cube of the number of decays in a term
        curve = e * e / 6 * L ** 3 * (m2[0] * up[0].abs()).sum() if name == "log_decay" else 0.0
        print(name, diff.item(), want.item(), float(noise), float(curve))
        assert abs(diff - want) <= noise + curve


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1, 16, 16), (5, 2, 6, 64, 32), (3, 1, 2, 128, 128), (2, 3, 3, 50, 37), (1, 1, 1, 1, 1), (4, 2, 2, 128, 4)], ids=str)
def test_token_step(vb, shape, dtype):
    B, G, H, dk, dv = shape
    t, _ = make(B, 1, G, H, dk, dv, dtype, decay=2.0)
    a = [t[n][:, 0] for n in ("q", "k", "v", "log_decay")]
    scale = dk ** -0.5
    f = {n: x.double() for n, x in t.items()}
    o, S = recurrence(f["q"], f["k"], f["v"], f["log_decay"], f["initial_state"], scale)
    mo, mS = recurrence(f["q"].abs(), f["k"].abs(), f["v"].abs(), f["log_decay"], f["initial_state"].abs(), scale)
    state = t["initial_state"]
    kept = state.clone()
    y, new = vb.linear_attention_step(*a, state)
    assert y.dtype == dtype and new.dtype == torch.float32 and torch.equal(state, kept)
    # the state: one product, one sum, one exponential of 2 steps; the output: dk + 2 more roundings
    assert ((new - S).abs() <= 6 * 2.0 ** -24 * mS).all()
    assert ((y - o[:, 0]).abs() <= HALF[dtype] * o[:, 0].abs() + (dk + 8) * 2.0 ** -24 * mo[:, 0] + 2.0 ** -25).all()
    same = vb.linear_attention_step(*a, state, state_out=state)        # in place
    assert same[1].data_ptr() == state.data_ptr() and torch.equal(same[0], y) and torch.equal(state, new)
    # a cache with more in it than these heads, rows behind the last sequence as they were
    cache = torch.full((B + 2, H * dk * dv + 12), 7.0, device="cuda")
    view = cache[:B, 8:8 + H * dk * dv].view(B, H, dk, dv)
    view.copy_(kept)
    y3, _ = vb.linear_attention_step(*a, view, state_out=view)
    assert torch.equal(y3, y) and torch.equal(view, new)
    cache[:B, 8:8 + H * dk * dv] = 7.0
    assert (cache == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_then_tokens(vb, dtype):
    """A prompt through the chunked form and tokens through the recurrent one give what the whole sequence gives."""
    B, L, more, G, H, dk, dv = 2, 150, 20, 2, 4, 64, 48
    t, up = make(B, L + more, G, H, dk, dv, dtype)
    cut = lambda x, a, b: x[:, a:b]      # noqa: E731
    with torch.no_grad():
        o, S = vb.linear_attention_fn(*(cut(t[n], 0, L) for n in ("q", "k", "v", "log_decay")), initial_state=t["initial_state"], return_final_state=True)
        out = [o]
        for i in range(L, L + more):
            y, S = vb.linear_attention_step(*(t[n][:, i] for n in ("q", "k", "v", "log_decay")), S, state_out=S)
            out.append(y[:, None])
    scale = dk ** -0.5
    ref, mag = reference(t, up, scale), reference(t, up, scale, True)
    got = torch.cat(out, 1)
    assert ((got - ref[0]).abs() <= HALF[dtype] * ref[0].abs() + (2 * FORM[dtype] + SUMS) * mag[0]).all()
    assert ((S - ref[1]).abs() <= (3 * PIECES[dtype] + SUMS) * mag[1]).all()


def test_padded_batch(vb):
    """Padding with k = 0 and log_decay = 0 leaves the state as the shorter sequence has it."""
    t, _ = make(2, 100, 1, 2, 32, 32, torch.bfloat16)
    with torch.no_grad():
        t["k"][1, 70:] = 0
        t["log_decay"][1, 70:] = 0
        o, S = vb.linear_attention_fn(t["q"], t["k"], t["v"], t["log_decay"], return_final_state=True)
        o1, S1 = vb.linear_attention_fn(*(t[n][1:, :70] for n in ("q", "k", "v", "log_decay")), return_final_state=True)
    assert torch.equal(S[1], S1[0]) and torch.equal(o[1, :70], o1[0])


def test_no_tokens_and_no_sequences(vb):
    q, v, g = torch.zeros(2, 0, 1, 16, device="cuda"), torch.zeros(2, 0, 2, 8, device="cuda"), torch.zeros(2, 0, 2, device="cuda")
    s = torch.randn(2, 2, 16, 8, device="cuda", requires_grad=True)
    o, S = vb.linear_attention_fn(q.requires_grad_(), q, v, g, initial_state=s, return_final_state=True)
    assert o.shape == v.shape and torch.equal(S, s)
    gq, gs = torch.autograd.grad([o.sum() + S.sum()], [q, s])
    assert gq.shape == q.shape and (gs == 1).all()
    o, S = vb.linear_attention_fn(q.detach(), q.detach(), v, g, return_final_state=True)
    assert (S == 0).all() and S.shape == (2, 2, 16, 8)
    none = vb.linear_attention_fn(q.detach()[:0], q.detach()[:0], v[:0], g[:0])
    assert none.shape == (0, 0, 2, 8)
    y, S = vb.linear_attention_step(torch.zeros(0, 1, 16, device="cuda"), torch.zeros(0, 1, 16, device="cuda"), torch.zeros(0, 2, 8, device="cuda"),
                                    torch.zeros(0, 2, device="cuda"), torch.zeros(0, 2, 16, 8, device="cuda"))
    assert y.shape == (0, 2, 8) and S.shape == (0, 2, 16, 8)


def test_only_some_gradients(vb):
    t, up = make(1, 80, 1, 2, 32, 32, torch.bfloat16)
    full = dict(zip(("o", "S", *NAMES), run(vb, t, up)))
    v = t["v"].clone().requires_grad_()
    o, S = vb.linear_attention_fn(t["q"], t["k"], v, t["log_decay"], None, t["initial_state"], True)
    both, = torch.autograd.grad([o, S], v, up, retain_graph=True)
    assert torch.equal(both, full["v"])
    state_only, = torch.autograd.grad(S, v, up[1], retain_graph=True)
    out_only, = torch.autograd.grad(o, v, up[0])
    assert torch.allclose(state_only.double() + out_only.double(), both.double(), rtol=0, atol=3 * 2.0 ** -8 * (state_only.abs() + out_only.abs()).max().item())


def test_same_bits_every_time_and_from_other_streams(vb):
    t, up = make(2, 700, 2, 4, 64, 64, torch.bfloat16)
    first = run(vb, t, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(vb, t, up)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured(vb):
    """Prompt and token calls in a graph; two graphs replayed in turn do not share a workspace that either still needs."""
    t, _ = make(1, 1100, 1, 2, 32, 32, torch.bfloat16)
    names = ("q", "k", "v", "log_decay")

    def capture(x, state):
        g = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(g):
            o, S = vb.linear_attention_fn(*(x[n] for n in names), initial_state=state, return_final_state=True)
            y, S2 = vb.linear_attention_step(*(x[n][:, -1] for n in names), S)
        return g, (o, S, y, S2)

    with torch.no_grad():
        state = t["initial_state"]
        vb.linear_attention_fn(*(t[n] for n in names), initial_state=state, return_final_state=True)
        torch.cuda.synchronize()
        other = {n: x.clone() for n, x in t.items()}
        other["v"].mul_(2)
        g1, r1 = capture(t, state)
        g2, r2 = capture(other, state)
        for _ in range(2):
            g1.replay()
            g2.replay()
        torch.cuda.synchronize()
        for x, r in ((t, r1), (other, r2)):
            o, S = vb.linear_attention_fn(*(x[n] for n in names), initial_state=state, return_final_state=True)
            y, S2 = vb.linear_attention_step(*(x[n][:, -1] for n in names), S)
            assert all(torch.equal(a, b) for a, b in zip(r, (o, S, y, S2)))


def test_training_step_captured(vb):
    t, up = make(1, 300, 1, 2, 32, 32, torch.bfloat16)
    want = run(vb, t, up)
    torch.cuda.synchronize()
    leaves = {n: x.clone().requires_grad_() for n, x in t.items()}

    def step():
        o, S = vb.linear_attention_fn(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], None, leaves["initial_state"], True)
        return [o, S, *torch.autograd.grad([o, S], [leaves[n] for n in NAMES], up)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))


def test_autocast_region(vb):
    t, up = make(1, 100, 1, 2, 32, 32, torch.float32)
    want = run(vb, t, up)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = run(vb, t, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(vb):
    t, _ = make(1, 8, 1, 2, 16, 16, torch.bfloat16)
    q, k, v, g, s = (t[n] for n in NAMES)
    f = vb.linear_attention_fn
    for bad in (lambda: f(q, k[:, :4], v, g), lambda: f(q[0], k[0], v[0], g[0]), lambda: f(q, k, v, g[..., :1]), lambda: f(q, k, v, g, None, s[:, :1]),
                lambda: f(q.expand(1, 8, 3, 16), k.expand(1, 8, 3, 16), v, g), lambda: f(q, k, v, g.cpu()), lambda: f(q, k, v, torch.zeros(3, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: f(q, k, v.float(), g), lambda: f(q.double(), k.double(), v.double(), g), lambda: f(q, k, v, g.long())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="not supported"):
        wide = torch.zeros(1, 8, 1, 136, device="cuda")
        f(wide, wide, v.float(), g)
    step = vb.linear_attention_step
    one = [x[:, 0] for x in (q, k, v, g)]
    with pytest.raises(TypeError):
        step(*one, s.bfloat16())
    with pytest.raises(RuntimeError, match="dense"):
        step(*one, s.transpose(2, 3))
    with pytest.raises(RuntimeError, match="overlap"):
        two = torch.zeros(2 * s.numel(), device="cuda")
        step(*one, two[:s.numel()].view(s.shape), state_out=two[4:4 + s.numel()].view(s.shape))
    with pytest.raises(RuntimeError, match="no backward"):
        step(*one, s.clone().requires_grad_())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets_in_long_sequences(vb, dtype):
    t, up = make(1, 400, 1, 2, 128, 72, dtype, decay=0.01)
    g = t["log_decay"]
    g[0, 31:34], g[0, 127], g[0, 128], g[0, 200:231, 0] = -float("inf"), -3e38, -1e4, -float("inf")
    ref = reference(t, up, 0.2)
    got = run(vb, t, up, 0.2)
    compare(got, ref, reference(t, up, 0.2, True), dtype, t, 0.2)
    assert (got[5][0, 31:34] == 0).all() and (got[5][0, 127] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_memory(vb, dtype):
    """No decay: the state is a sum over all tokens, here of positive terms.  Chunks are summed apart (64 terms of two pieces, cut off: 2^-16) and added in fp32
    (512 roundings of 2^-24 at most, and as many products with a decay of one), so that the sum is as good after 32 768 tokens as after a few."""
    B, L, H, d = 1, 32768, 2, 16
    t, _ = make(B, L, H, H, d, d, dtype)
    k, v = t["k"].abs(), t["v"].abs()
    with torch.no_grad():
        _, S = vb.linear_attention_fn(t["q"], k, v, torch.zeros(H, device="cuda"), return_final_state=True)
    want = torch.einsum("blhk,blhv->bhkv", k.double(), v.double())
    assert ((S - want).abs() / want).max() <= 2.0 ** -16 + 1024 * 2.0 ** -24 / 3
    # the roundings of the additions are of random sign, those of the products fall off: a chunk's error is at most 24 steps of 2^-24 cut off
    assert (S - want).norm() <= 2.0 ** -18 * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_states_side_by_side(vb, dtype):
    """Two states of a sequence next to one another in one cache, read and written in turn: memory that interleaves without overlapping."""
    B, G, H, dk, dv = 5, 2, 4, 32, 16
    t, _ = make(B, 1, G, H, dk, dv, dtype)
    a = [t[n][:, 0] for n in ("q", "k", "v", "log_decay")]
    cache = torch.full((B, 3, H, dk, dv), 7.0, device="cuda")
    cache[:, 1] = t["initial_state"]
    y, new = vb.linear_attention_step(*a, t["initial_state"])
    for src, dst in ((1, 0), (1, 2)):
        y2, s2 = vb.linear_attention_step(*a, cache[:, src], state_out=cache[:, dst])
        assert torch.equal(y2, y) and torch.equal(cache[:, dst], new) and torch.equal(cache[:, 1], t["initial_state"]) and s2.data_ptr() == cache[:, dst].data_ptr()
    y3, _ = vb.linear_attention_step(*(x[:1] for x in a), cache[:1, 1], state_out=cache[:1, 0])
    assert torch.equal(y3, y[:1])
    size = H * dk * dv
    flat = cache.view(-1)
    view = lambda first, stride, n=B: flat.as_strided((n, H, dk, dv), (stride, dk * dv, dv, 1), first)      # noqa: E731
    for first in (size - 4, size + 4, 3 * size + 4, 5 * size - 4):     # into the state of the same sequence, or of the one behind ([4, 5) size)
        with pytest.raises(RuntimeError, match="overlap"):
            vb.linear_attention_step(*(x[:3] for x in a), view(size, 3 * size, 3), state_out=view(first, 3 * size, 3))
    two = [x[:2] for x in a]
    with pytest.raises(RuntimeError, match="overlap"):                  # strides that differ: the second state into the third's place
        vb.linear_attention_step(*two, view(0, 2 * size, 2), state_out=view(size, size, 2))
    flat[:size], flat[3 * size:4 * size] = t["initial_state"][0].flatten(), t["initial_state"][1].flatten()
    y4, s4 = vb.linear_attention_step(*two, view(0, 3 * size, 2), state_out=view(size, size, 2))
    assert torch.equal(y4, y[:2]) and torch.equal(s4, new[:2])


def test_a_state_written_in_place_is_seen_by_autograd(vb):
    """A tensor that a backward pass still needs and that a step has overwritten: refused, as for any operation in place."""
    t, _ = make(2, 1, 1, 2, 16, 16, torch.float32)
    a = [t[n][:, 0] for n in ("q", "k", "v", "log_decay")]
    leaf = torch.ones_like(t["initial_state"], requires_grad=True)
    state = t["initial_state"].clone()
    loss = (leaf * state).sum()
    before = state._version
    with torch.no_grad():
        vb.linear_attention_step(*a, state, state_out=state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.no_grad():
        before = state._version
        vb.linear_attention_step(*a, state)
    assert state._version == before
    with torch.inference_mode():                                        # tensors without versions
        own = state.clone()
        y, _ = vb.linear_attention_step(*a, own, state_out=own)
        z, _ = vb.linear_attention_step(*a, state)
    assert torch.equal(y, z)


def test_forward_mode_is_refused(vb):
    """There is no forward-mode derivative: a dual tensor raises instead of losing its tangent."""
    import torch.autograd.forward_ad as fwad
    t, _ = make(1, 5, 1, 2, 16, 16, torch.float32)
    for name in NAMES:
        with fwad.dual_level():
            x = {**t, name: fwad.make_dual(t[name], torch.ones_like(t[name]))}
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                vb.linear_attention_fn(x["q"], x["k"], x["v"], x["log_decay"], None, x["initial_state"])
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                vb.linear_attention_step(*(x[n][:, 0] for n in NAMES[:4]), x["initial_state"])
    with fwad.dual_level():
        vb.linear_attention_fn(*(t[n] for n in NAMES[:4]))              # plain tensors inside a level: as ever


def test_second_derivatives_are_refused(vb):
    """The gradients have no history of their own: asked for one, the backward pass raises instead of leaving a term out."""
    t, _ = make(1, 70, 1, 2, 16, 16, torch.float32)
    leaves = {n: x.requires_grad_() for n, x in t.items()}
    for start in (None, leaves["initial_state"]):
        o, S = vb.linear_attention_fn(*(leaves[n] for n in NAMES[:4]), None, start, True)
        loss = (o ** 2).sum() + S.sum() + (leaves["q"] ** 3).sum()
        with pytest.raises(RuntimeError, match="once differentiable"):
            torch.autograd.grad(loss, leaves["q"], create_graph=True)
        g, = torch.autograd.grad(loss, leaves["q"])
        assert g.shape == leaves["q"].shape


def test_no_tokens_and_only_a_state_to_differentiate(vb):
    q, v, g = torch.zeros(2, 0, 1, 16, device="cuda"), torch.zeros(2, 0, 2, 8, device="cuda"), torch.zeros(2, 0, 2, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.randn(2, 2, 16, 8, device="cuda", dtype=dtype, requires_grad=True)
        o = vb.linear_attention_fn(q, q, v, g, initial_state=s)
        assert o.dtype == torch.float32 and o.shape == v.shape
        ds, = torch.autograd.grad(o.sum(), s)
        assert ds.shape == s.shape and ds.dtype == dtype and (ds == 0).all()
    infinite = torch.full((2, 2, 16, 8), float("inf"), device="cuda", requires_grad=True)
    ds, = torch.autograd.grad(vb.linear_attention_fn(q, q, v, g, initial_state=infinite).sum(), infinite)
    assert (ds == 0).all()


@pytest.mark.parametrize("groups", [1, 2])
def test_is_the_selective_scan_of_heads_that_share_a_decay(vb, groups):
    """`selective_scan_fn` with B, C, u dt and A dt as keys, queries, values and log decays: the same numbers with scale 1, which is not the default."""
    B, L, H, N, P = 2, 150, 4, 16, 8
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen).cuda()      # noqa: E731
    u, k, q = rnd(B, H, P, L), rnd(B, groups, N, L), rnd(B, groups, N, L)
    dt, rate = 0.1 * torch.rand((B, H, 1, L), generator=gen).cuda(), -1.0 - torch.rand(H, generator=gen).cuda()
    y = vb.selective_scan_fn(u.flatten(1, 2), dt.expand(B, H, P, L).flatten(1, 2).contiguous(), rate[:, None, None].expand(H, P, N).flatten(0, 1).contiguous(),
                             k, q, delta_softplus=False).view(B, H, P, L).permute(0, 3, 1, 2)
    tokens = lambda x: x.permute(0, 3, 1, 2)      # noqa: E731
    v, g = tokens(u * dt), (dt[:, :, 0] * rate[:, None]).transpose(1, 2)
    o = vb.linear_attention_fn(tokens(q), tokens(k), v, g, scale=1.0)
    t = {"q": tokens(q), "k": tokens(k), "v": v, "log_decay": g, "initial_state": torch.zeros(B, H, N, P, device="cuda")}
    mag = recurrence(*(t[n].double().abs() if n != "log_decay" else t[n].double() for n in NAMES), 1.0)[0]
    # SUMS of the magnitudes for the one and the other, products of pieces
    assert ((o - y).abs() <= (2 * SUMS + 2 * FORM[torch.float32]) * mag).all()
    default = vb.linear_attention_fn(tokens(q), tokens(k), v, g)
    assert ((default * N ** 0.5 - y).abs() <= (2 * SUMS + 2 * FORM[torch.float32]) * mag).all()


FORMS = [(1, 400, 1, 2, 128, 128, torch.bfloat16), (1, 400, 1, 2, 32, 32, torch.bfloat16), (1, 150, 1, 2, 64, 64, torch.float16), (1, 150, 1, 2, 32, 64, torch.float32)]


@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_values_that_are_not_finite(vb, shape):
    """A query's: its own token.  A key's or decay's: its heads from its token on.  A value's: its own column, from the first token of its 128 on."""
    *shape, dtype = shape
    t, _ = make(*shape, dtype)
    at, tokens = 141, torch.arange(shape[1], device="cuda")
    for bad in (float("nan"), float("inf")):
        for name in NAMES[:4]:
            if name == "log_decay" and bad == float("inf"):
                continue
            x = {n: y.clone() for n, y in t.items()}
            x[name][(0, at, 0) + ((5,) if name != "log_decay" else ())] = bad
            with torch.no_grad():
                o, S = vb.linear_attention_fn(*(x[n] for n in NAMES[:4]), None, x["initial_state"], True)
            fine = torch.isfinite(o[0])                                 # (tokens, heads, columns)
            if name == "q":
                assert fine[tokens != at].all() and not fine[at].any() and torch.isfinite(S).all()
            elif name == "k":
                assert fine[tokens < at].all() and not fine[tokens >= at].any()
            elif name == "log_decay":
                assert fine[:, 1].all() and fine[tokens < at].all() and not fine[tokens >= at, 0].any() and torch.isfinite(S[0, 1]).all()
            else:
                assert fine[:, 1].all() and fine[tokens < 128].all() and not fine[tokens >= at, 0, 5].any()
                others = torch.arange(shape[5], device="cuda") != 5
                assert fine[:, 0][:, others].all() and torch.isfinite(S[0, 0][:, others]).all() and torch.isfinite(S[0, 1]).all()


@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_states_that_grow(vb, shape):
    """Positive log decays: exact as long as the weights between two tokens are numbers of fp32.  Growth by 2^30 over some tokens, decay by as much behind them."""
    *shape, dtype = shape
    t, _ = make(*shape, dtype, decay=0.02)
    g = t["log_decay"]
    for first in (3, 40, 70, 140):
        g[:, first:first + 10] += 3 * 0.6931
        g[:, first + 20:first + 30] -= 3 * 0.6931
    scale = 2.0 ** -24
    with torch.no_grad():
        o, S = vb.linear_attention_fn(*(t[n] for n in NAMES[:4]), scale, t["initial_state"], True)
    ref, mag = (recurrence(*(f(n) for n in NAMES), scale) for f in (lambda n: t[n].double(), lambda n: t[n].double() if n == "log_decay" else t[n].double().abs()))
    # beside the roundings of the head of this file: log decays of up to 3 in base 2, each off by 2^-23, in weights of up to 20 of them
    assert ((S - ref[1]).abs() <= (3 * PIECES[dtype] + SUMS + 2.0 ** -17) * mag[1]).all()
    assert ((o - ref[0]).abs() <= HALF[dtype] * ref[0].abs() + (2 * FORM[dtype] + SUMS + 2.0 ** -17) * mag[0] + (2.0 ** -25 if dtype == torch.float16 else 0)).all()


def test_long_memory_of_wide_heads(vb):
    """The sum of `test_long_memory` in the kernels of long bf16 sequences: chunks of 128 tokens, each summed apart (2 x 128 products of two pieces, cut off, 2^-16 as there),
    256 of them added in fp32."""
    B, L, H, d = 1, 32768, 2, 128
    t, _ = make(B, L, H, H, d, d, torch.bfloat16)
    k, v = t["k"].abs(), t["v"].abs()
    want = torch.einsum("blhk,blhv->bhkv", k.double(), v.double())
    for train in (False, True):                                         # chunks of 128 and of 64 tokens
        with torch.set_grad_enabled(train):
            leaf = v.clone().requires_grad_(train)
            _, S = vb.linear_attention_fn(t["q"], k, leaf, torch.zeros(H, device="cuda"), return_final_state=True)
        assert ((S.detach() - want).abs() / want).max() <= 2.0 ** -16 + 1024 * 2.0 ** -24 / 3
        assert (S.detach() - want).norm() <= 2.0 ** -17 * want.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets_behind_decays_of_almost_one(vb, dtype):
    """Log decays between -2^-25 and 0 (saturated gates), whose whole numbers and fractions are at their border, and resets among them: nothing crosses these."""
    t, up = make(1, 192, 1, 2, 32, 32, dtype)
    resets = [2, 7, 33, 64, 100, 127, 128, 190]
    for small in (-1e-9, -2.0 ** -26, -2.0 ** -24, 0.0):
        t["log_decay"].fill_(small)
        t["log_decay"][:, resets] = -float("inf")
        got = run(vb, t, up)
        compare(got, reference(t, up, 32 ** -0.5), reference(t, up, 32 ** -0.5, True), dtype, t, 32 ** -0.5)
        assert (got[5][:, resets] == 0).all(), small


# ---- fp32 results ------------------------------------------------------------------------------------------------------
PRECISE = [(4, 1001, 8, 8, 32, 64), (2, 359, 4, 4, 16, 24), (3, 300, 1, 6, 64, 80), (1, 640, 2, 2, 128, 128), (2, 200, 2, 4, 96, 128)]


def plain_decays(B, L, H):
    """Step sizes of [1e-3, 1e-1] through a softplus, rates of [1, 16]: what a scan's decays look like."""
    gen = torch.Generator().manual_seed(2)
    dt = torch.exp(torch.rand(H, generator=gen) * 4.6 - 6.9)
    raw = torch.randn((B, L, H), generator=gen) + torch.log(torch.expm1(dt))
    return (-torch.nn.functional.softplus(raw) * (1 + 15 * torch.rand(H, generator=gen))).cuda()


def relative_errors(vb, shape, dtype):
    t, up = make(*shape, dtype)
    t["log_decay"] = plain_decays(shape[0], shape[1], shape[3])
    got, ref = run(vb, t, up), reference(t, up, shape[4] ** -0.5)
    found = {n: ((x.double() - y).norm() / y.norm()).item() for n, x, y in zip(("out", "final_state", *NAMES), got, ref) if x.dtype == torch.float32}
    print(shape, dtype, {n: f"{e:.1e}" for n, e in found.items()})
    return found


@pytest.mark.parametrize("shape", PRECISE, ids=str)
def test_fp32_calls_are_as_exact_as_fp32(vb, shape):
    """Norm against norm, at most 2^-20: sums of some hundred terms of random sign, each product 2^-22 off (two tf32 pieces), each addition 2^-24 of what it adds to."""
    for name, e in relative_errors(vb, shape, torch.float32).items():
        assert e <= 2.0 ** -20, (name, e)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", PRECISE + [(30, 25, 1, 2, 32, 64)], ids=str)
def test_states_of_16_bit_calls_are_as_exact_as_fp32(vb, shape, dtype):
    """The same for the states and their gradients, fp32 results of 16-bit inputs: three pieces of bf16 (2^-25 off), two of tf32 beside fp16 (2^-23)."""
    e = relative_errors(vb, shape, dtype)
    assert e["final_state"] <= 2.0 ** -20 and e["initial_state"] <= 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", PRECISE + [(30, 25, 1, 2, 32, 64), (1, 1500, 4, 12, 64, 32)], ids=str)
def test_decay_gradients_of_16_bit_calls_are_as_exact_as_fp32(vb, shape, dtype):
    """The same for the gradients of the decays: sums of products with both states, which keep their 32 bits between the passes."""
    assert relative_errors(vb, shape, dtype)["log_decay"] <= 2.0 ** -20
