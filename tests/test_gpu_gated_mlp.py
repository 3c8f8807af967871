"""Gated feed-forward block against its formulas in 64 bits.

Tolerances count, term by term: half a step of the type for every result and for what is rounded to it on the way (the hidden map, the gradients of value and
gate); fp32 sums of n terms, n 2^-24 of the sum of magnitudes, and 2^-21 for products of pieces and the exponentials; and what an error of value or gate does behind the
activation, whose derivative is at most 1.13 and whose second derivative at most 0.8 in magnitude.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ORDER = ("x", "w1", "w2", "b1", "b2")


@pytest.fixture(scope="module")
def vb():
    import vmamba_b200
    return vmamba_b200


def make(M, C, H, O, dtype, biases=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)      # noqa: E731
    t = {"x": rnd(M, C), "w1": rnd(2 * H, C) / C ** 0.5, "w2": rnd(O, H) / H ** 0.5}
    if biases:
        t["b1"], t["b2"] = 0.3 * rnd(2 * H), rnd(O)
    return {n: v.to(dtype).cuda() for n, v in t.items()}, rnd(M, O).to(dtype).cuda()


def bent(g, act):
    """act, its derivative"""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    phi = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def reference(t, dy, act, dtype):
    """{name: (value, tolerance)}"""
    u = HALF[dtype]
    f = {n: v.detach().double() for n, v in t.items()}
    x, w1, w2, dy = f["x"], f["w1"], f["w2"], dy.double()
    (M, C), (O, H) = x.shape, w2.shape
    b1 = f.get("b1", torch.zeros(2 * H, dtype=torch.float64, device="cuda"))
    b2 = f.get("b2", torch.zeros(O, dtype=torch.float64, device="cuda"))
    s = lambda n: (n + 2) * 2.0 ** -24 + 2.0 ** -21      # noqa: E731
    v, g = (x @ w1.t() + b1).chunk(2, -1)
    ev, eg = (s(C) * (x.abs() @ w1.abs().t() + b1.abs())).chunk(2, -1)
    a, da = bent(g, act)
    ea, eda = 1.13 * eg + 2.0 ** -21 * g.abs(), 0.8 * eg + 2.0 ** -20
    if dtype != torch.float32:      # activations of 16-bit results: Phi by a polynomial (gelu off by 3.5e-5 at most, Phi by 1e-4), sigmoid by a tanh that is 2^-11 off
        if act == "gelu":
            ea, eda = ea + 3.5e-5, eda + 1e-4
        elif dtype == torch.bfloat16:
            ea, eda = ea + 2.0 ** -12 * g.abs(), eda + 2.0 ** -12 * (1 + 2 * g.abs())
    h = v * a
    eh = u * h.abs() + 1.01 * (ev * a.abs() + v.abs() * ea + ev * ea)
    y = h @ w2.t() + b2
    out = {"y": (y, eh @ w2.abs().t() + s(H) * (h.abs() @ w2.abs().t() + b2.abs()))}
    dh = dy @ w2
    edh = s(O) * (dy.abs() @ w2.abs())
    dz = torch.cat((dh * a, dh * v * da), 1)
    edz = torch.cat((edh * a.abs() + dh.abs() * ea + edh * ea,
                     edh * (v * da).abs() + dh.abs() * (ev * da.abs() + v.abs() * eda + ev * eda) + edh * (ev * 1.13 + v.abs() * eda)), 1)
    edz = 1.01 * edz + u * dz.abs()
    out["x"] = (dz @ w1, edz @ w1.abs() + s(2 * H) * (dz.abs() @ w1.abs()))
    out["w1"] = (dz.t() @ x, edz.t() @ x.abs() + s(M) * (dz.abs().t() @ x.abs()))
    out["w2"] = (dy.t() @ h, dy.abs().t() @ eh + s(M) * (dy.abs().t() @ h.abs()))
    out["b1"] = (dz.sum(0), edz.sum(0) + s(M) * dz.abs().sum(0))
    out["b2"] = (dy.sum(0), s(M) * dy.abs().sum(0))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    return {n: (r, 1.01 * e + u * r.abs() + tiny * (1 + H)) for n, (r, e) in out.items()}


def compare(got, ref, dtype):
    for n, y in got.items():
        r, tol = ref[n]
        assert y.shape == r.shape and y.dtype == dtype, n
        err = (y.double() - r).abs()
        worst, rel = (err / tol).max().item(), (err.norm() / r.norm().clamp(min=1e-30)).item()
        print(f"{n}: {worst:.3f} of the tolerance, relative error {rel:.2e}")
        assert torch.isfinite(y).all() and worst <= 1, (n, worst)
        # independent roundings: at most three on the way, each of a root mean square of half a step / sqrt(3)
        assert y.numel() < 1000 or rel <= max(HALF[dtype], 2.0 ** -18), (n, rel)


def run(vb, t, dy, act):
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    y = vb.gated_mlp_fn(**leaves, act=act)
    return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}


SHAPES = [(1, 8, 8, 8), (1, 768, 1024, 768), (3, 64, 128, 64), (7, 200, 504, 96), (16, 96, 384, 96), (17, 128, 256, 128), (33, 72, 152, 40), (64, 64, 64, 64),
          (65, 65, 33, 17), (100, 50, 30, 10), (130, 96, 256, 96), (250, 384, 1536, 384), (300, 1, 1, 1), (1000, 192, 512, 192), (2050, 128, 136, 264)]


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_formulas(vb, shape, dtype, act):
    t, dy = make(*shape, dtype)
    ref = reference(t, dy, act, dtype)
    compare(run(vb, t, dy, act), ref, dtype)
    with torch.no_grad():
        compare({"y": vb.gated_mlp_fn(**t, act=act)}, ref, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_without_biases_and_with_one(vb, dtype):
    t, dy = make(150, 64, 128, 64, dtype, biases=False)
    compare(run(vb, t, dy, "silu"), reference(t, dy, "silu", dtype), dtype)
    for name in ("b1", "b2"):
        full, _ = make(150, 64, 128, 64, dtype)
        one = {**t, name: full[name]}
        compare(run(vb, one, dy, "gelu"), reference(one, dy, "gelu", dtype), dtype)


@pytest.mark.parametrize("M", [5, 150, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_shapes(vb, dtype, M):
    t, dy = make(M, 64, 128, 64, dtype)
    want = run(vb, t, dy, "gelu")
    wide = torch.zeros(M, 80, dtype=dtype, device="cuda")
    for off in (0, 8, 3):                                          # rows apart, on any element
        wide[:, off:off + 64] = t["x"]
        got = run(vb, {**t, "x": wide[:, off:off + 64]}, dy, "gelu")
        compare(got, reference(t, dy, "gelu", dtype), dtype)
    got = run(vb, {**t, "w1": t["w1"].t().contiguous().t(), "x": t["x"].t().contiguous().t()}, dy.t().contiguous().t(), "gelu")
    assert all(torch.equal(got[n], want[n]) for n in want)
    y = vb.gated_mlp_fn(t["x"].view(1, M, 1, 64), t["w1"], t["w2"], t["b1"], t["b2"])
    assert y.shape == (1, M, 1, 64) and torch.equal(y.view(M, 64), want["y"])
    y = vb.gated_mlp_fn(t["x"][0], t["w1"], t["w2"], t["b1"], t["b2"])
    assert y.shape == (64,)
    same = t["x"][:1].expand(M, 64).detach().requires_grad_()      # one token for all rows
    y = vb.gated_mlp_fn(same, t["w1"], t["w2"], t["b1"], t["b2"])
    assert all(torch.equal(y[0], r) for r in y)
    g, = torch.autograd.grad(y, same, dy[:1].expand(M, 64))
    assert g.shape == same.shape


def test_gradients_against_differences(vb):
    """fp32, central differences along signs; the third derivative of the loss along a direction is bounded through that of the activation (3 in magnitude)."""
    t, dy = make(20, 24, 40, 16, torch.float32)
    got = run(vb, t, dy, "gelu")
    loss = lambda q: (vb.gated_mlp_fn(**q).double() * dy.double()).sum()      # noqa: E731
    gen = torch.Generator().manual_seed(3)
    f = {n: v.double() for n, v in t.items()}
    for n in t:
        d = torch.randn(t[n].shape, generator=gen).sign().cuda()
        e = 2.0 ** -9
        diff = (loss({**t, n: t[n] + e * d}) - loss({**t, n: t[n] - e * d})) / (2 * e)
        want = (got[n].double() * d.double()).sum()
        up = {k: v.abs() + (e if k == n else 0) for k, v in f.items()}
        z = up["x"] @ up["w1"].t() + up["b1"]
        zd = {"x": torch.ones_like(up["x"]) @ up["w1"].t(), "w1": up["x"].sum(1, keepdim=True).expand_as(z), "b1": torch.ones_like(z)}.get(n, torch.zeros_like(z))
        (v, g), (dv, dg) = z.chunk(2, -1), zd.chunk(2, -1)
        back = dy.abs().double() @ up["w2"]
        third = (back * (3 * v * dg ** 3 + 3 * 0.8 * dv * dg ** 2)).sum()
        noise = 64 * 2.0 ** -24 * ((dy.abs() * (((v * g) @ up["w2"].t()) + up["b2"])).sum()) / e
        print(n, diff.item(), want.item(), third.item() * e * e / 6, noise.item())
        assert abs(diff - want) <= third * e * e / 6 + noise


def test_large_and_small_gates(vb):
    """Gates far out: the activation is the gate or zero, its derivative one or zero, and nothing overflows on the way."""
    for dtype in (torch.float32, torch.bfloat16):
        for act in ("gelu", "silu"):
            x = torch.tensor([[1.0], [-1.0]], device="cuda").repeat(40, 8).to(dtype)
            w1 = torch.cat((torch.ones(16, 8), 100.0 * torch.ones(16, 8))).cuda().to(dtype).requires_grad_()
            w2 = torch.ones(8, 16, device="cuda", dtype=dtype)
            y = vb.gated_mlp_fn(x, w1, w2, act=act)
            assert (y[0::2] == 16 * 8 * 800).all() and (y[1::2] == 0).all()
            g, = torch.autograd.grad(y, w1, torch.ones_like(y))
            assert torch.isfinite(g).all()


def test_no_tokens(vb):
    t, _ = make(4, 16, 32, 8, torch.bfloat16)
    leaves = {n: v.requires_grad_() for n, v in t.items()}
    leaves["x"] = torch.zeros(2, 0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = vb.gated_mlp_fn(**leaves)
    assert y.shape == (2, 0, 8) and y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y.sum(), list(leaves.values()))
    assert all(g.shape == v.shape and (g == 0).all() for g, v in zip(grads, leaves.values()))


@pytest.mark.parametrize("M", [4, 200])
def test_only_some_gradients(vb, M):
    t, dy = make(M, 64, 128, 64, torch.bfloat16)
    want = run(vb, t, dy, "gelu")
    for n in ORDER:
        leaves = {k: v.detach() for k, v in t.items()}
        leaves[n].requires_grad_()
        y = vb.gated_mlp_fn(**leaves)
        g, = torch.autograd.grad(y, leaves[n], dy)
        assert torch.equal(g, want[n]), n
        leaves = {k: v.detach() for k, v in t.items() if k != "b1" or n == "b1"}      # a missing bias in front of the one that is asked for
        leaves[n].requires_grad_()
        g, = torch.autograd.grad(vb.gated_mlp_fn(**leaves), leaves[n], dy)
        assert g.shape == t[n].shape


@pytest.mark.parametrize("M", [3, 300])
def test_same_bits_streams_graphs_autocast(vb, M):
    t, dy = make(M, 96, 256, 96, torch.bfloat16)
    want = run(vb, t, dy, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(vb, t, dy, "gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[n], again[n]) for n in want)
    with torch.autocast("cuda", dtype=torch.float16):
        again = run(vb, t, dy, "gelu")
    assert all(torch.equal(want[n], again[n]) for n in want)
    torch.cuda.synchronize()
    graphs = []
    for k in range(2):
        x = t["x"] * (k + 1)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run(vb, {**t, "x": x}, dy, "gelu")
        graphs.append((g, x, got))
    for _ in range(2):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, x, got in graphs:
        now = run(vb, {**t, "x": x}, dy, "gelu")
        assert all(torch.equal(now[n], got[n]) for n in now)


def test_first_call_in_a_capture():
    """A process whose first call on the device is captured, for inference and for training (the backward pass runs on a thread of autograd's)."""
    import os
    import subprocess
    import sys
    code = """
import torch, vmamba_b200 as vb
mk = lambda *s: (torch.randn(s, device="cuda") / s[-1] ** 0.5).bfloat16()
x, w1, w2, q = mk(300, 64), mk(256, 64), mk(64, 128), mk(1, 600, 2, 128)
g = torch.zeros(1, 600, 2, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(graph):
    y, o = vb.gated_mlp_fn(x, w1, w2), vb.linear_attention_fn(q, q, q, g)
graph.replay()
leaves = [t.clone().requires_grad_() for t in (x, w1, w2, q)]
torch.cuda.synchronize()
train = torch.cuda.CUDAGraph()
with torch.cuda.graph(train):
    got = torch.autograd.grad(vb.gated_mlp_fn(*leaves[:3]).sum() + vb.linear_attention_fn(leaves[3], leaves[3], leaves[3], g).sum(), leaves)
train.replay()
torch.cuda.synchronize()
want = torch.autograd.grad(vb.gated_mlp_fn(*leaves[:3]).sum() + vb.linear_attention_fn(leaves[3], leaves[3], leaves[3], g).sum(), leaves)
with torch.no_grad():
    assert torch.equal(y, vb.gated_mlp_fn(x, w1, w2)) and torch.equal(o, vb.linear_attention_fn(q, q, q, g))
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_refusals(vb):
    t, _ = make(4, 16, 32, 8, torch.bfloat16)
    f = vb.gated_mlp_fn
    for bad in ({**t, "w1": t["w1"][:62]}, {**t, "w2": t["w2"][:, :30]}, {**t, "b1": t["b1"][:32]}, {**t, "b2": t["b2"][:4]}, {**t, "x": t["x"][:, :8]},
                {**t, "w1": t["w1"].cpu()}, {**t, "w1": t["w1"][0]}):
        with pytest.raises(RuntimeError):
            f(**bad)
    for bad in ({**t, "w1": t["w1"].float()}, {**t, "b2": t["b2"].float()}, {n: v.double() for n, v in t.items()}):
        with pytest.raises(TypeError):
            f(**bad)


def test_block_of_attention_and_feed_forward(vb):
    """The operators as a block runs them: queries, keys, values and decays from one projection, attention, residual, feed-forward, residual; a whole
    sequence against a prompt and single tokens, and its training step against the formulas."""
    B, L, H, d, C = 2, 100, 4, 16, 64
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()      # noqa: E731
    wi, w1, w2 = rnd(3 * C + H, C) / C ** 0.5, rnd(4 * C, C) / C ** 0.5, rnd(C, 2 * C) / C ** 0.5
    x = rnd(B, L, C)

    def split(z):
        q, k, v, r = z.split((C, C, C, H), -1)
        heads = lambda y: y.unflatten(-1, (H, d))      # noqa: E731
        return heads(q), heads(k), heads(v), -torch.nn.functional.softplus(r)

    def whole(x, wi, w1, w2, state=None):
        o, S = vb.linear_attention_fn(*split(x @ wi.t()), initial_state=state, return_final_state=True)
        x = x + o.flatten(-2)
        return x + vb.gated_mlp_fn(x, w1, w2), S

    def formulas(x, wi, w1, w2):
        q, k, v, r = split(x @ wi.t())
        S, o = torch.zeros(B, H, d, d, dtype=x.dtype, device="cuda"), []
        for t in range(L):
            S = torch.exp(r[:, t])[..., None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
            o.append(d ** -0.5 * (q[:, t, :, :, None] * S).sum(-2))
        x = x + torch.stack(o, 1).flatten(-2)
        a, b = (x @ w1.t()).chunk(2, -1)
        return x + (a * torch.nn.functional.gelu(b)) @ w2.t()

    ref_in = [t.double().requires_grad_() for t in (x, wi, w1, w2)]
    own_in = [t.clone().requires_grad_() for t in (x, wi, w1, w2)]
    up = rnd(B, L, C)
    want, (got, _) = formulas(*ref_in), whole(*own_in)
    wanted, found = torch.autograd.grad(want, ref_in, up.double()), torch.autograd.grad(got, own_in, up)
    # fp32 throughout: four products of up to 256 terms in a row, each of at most (256 + 2) 2^-24 of magnitudes that random signs leave some
    # 16 times as large as the results, and as much again behind them
    for a, b in zip((want, *wanted), (got, *found)):
        assert (a - b).norm() <= 2.0 ** -13 * a.norm()
    with torch.no_grad():
        y, S = whole(x[:, :90], wi, w1, w2)
        for t in range(90, L):
            z = x[:, t]
            o, S = vb.linear_attention_step(*split(z @ wi.t()), S, state_out=S)
            z = z + o.flatten(-2)
            z = z + vb.gated_mlp_fn(z, w1, w2)
            assert (z - want[:, t]).norm() <= 2.0 ** -13 * want[:, t].norm()


# ---- gates one by one -------------------------------------------------------------------------------------------------
# Half a step for a rounded result.  Activations: 2^-16 of the value beside 16-bit types (the fit of Phi 2^-18, exponents of up to 127 rounded in fp32 2^-17), for fp32
# CUDA's normcdff (5 steps of 2^-23), one more product and the two tf32 pieces that carry a gradient (2^-22).  What is below 2^-126 may come as zero.
RELATIVE = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -19}


def gates(act, dtype):
    far = -13.0 if act == "gelu" else -80.0
    g = torch.cat((torch.linspace(far, 13.0, 2417), torch.linspace(-10.0, -3.0, 700), torch.tensor([s * 2.0 ** -k for s in (1, -1) for k in range(14)]), torch.zeros(3)))
    return (g.to(dtype) if dtype != torch.float32 else g.bfloat16().float()).cuda()       # few bits: nothing is lost in front of the activation


def single_gates(vb, g, act, offset=0):
    """(act(g), gradient of the value, gradient of the gate) of a block that does nothing else: value 1, unit weights, an upstream gradient for one hidden channel"""
    M, dtype = g.numel(), g.dtype
    wide = torch.zeros(M, 16, dtype=dtype, device="cuda")
    x = wide[:, offset:offset + 8]
    x[:, 0], x[:, 1] = g, 1
    x.requires_grad_()
    w1, dy = torch.zeros(16, 8, dtype=dtype, device="cuda"), torch.zeros(M, 8, dtype=dtype, device="cuda")
    w1[:8, 1], w1[8:, 0], dy[:, 3] = 1, 1, 1
    y = vb.gated_mlp_fn(x, w1, torch.eye(8, dtype=dtype, device="cuda"), act=act)
    dx, = torch.autograd.grad(y, x, dy)
    assert all(torch.equal(y[:, 0], y[:, j]) for j in range(8))
    return y[:, 3].detach(), dx[:, 1], dx[:, 0]


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kernels", ["many_tokens", "few_tokens", "unaligned"])
def test_activations_elementwise(vb, kernels, dtype, act):
    g = gates(act, dtype)
    per = 13 if kernels == "few_tokens" else g.numel()
    parts = [single_gates(vb, c, act, offset=1 if kernels == "unaligned" else 0) for c in g.split(per)]
    got = [torch.cat(p).double() for p in zip(*parts)]
    z = g.double()
    a, da = bent(z, act)
    if act == "gelu":
        size = 0.5 * torch.erfc(-z / math.sqrt(2)) + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        size = torch.sigmoid(z) * (1 + z.abs() * torch.sigmoid(-z))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -119
    for name, x, want, mag in (("value", got[0], a, a.abs()), ("gradient of the value", got[1], a, a.abs()), ("gradient of the gate", got[2], da, size)):
        worst = ((x - want).abs() / (HALF[dtype] * want.abs() + RELATIVE[dtype] * mag + tiny)).max().item()
        print(f"{name}: {worst:.3f} of the tolerance")
        assert worst <= 1, (name, worst)


def test_forward_mode_is_refused(vb):
    """There is no forward-mode derivative: a dual tensor raises instead of losing its tangent."""
    import torch.autograd.forward_ad as fwad
    for M in (5, 0):
        t, _ = make(5, 16, 32, 8, torch.float32)
        t["x"] = t["x"][:M]
        for name in t:
            with fwad.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                vb.gated_mlp_fn(**{**t, name: fwad.make_dual(t[name], torch.ones_like(t[name]))})
    with fwad.dual_level():
        vb.gated_mlp_fn(**t)                                            # plain tensors inside a level: as ever


def test_second_derivatives_are_refused(vb):
    """The gradients have no history of their own: asked for one, the backward pass raises instead of leaving a term out."""
    t, _ = make(20, 16, 32, 8, torch.float32)
    leaves = {n: v.requires_grad_() for n, v in t.items()}
    loss = (vb.gated_mlp_fn(**leaves) ** 2).sum() + (leaves["x"] ** 3).sum()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.grad(loss, leaves["x"], create_graph=True)
    g, = torch.autograd.grad(loss, leaves["x"])
    assert g.shape == leaves["x"].shape


# ---- large calls -------------------------------------------------------------------------------------------------------
# Every form of the tensor-core kernels, with several tiles for each CTA where its form is ever chosen for that, ragged edges, and last rounds that leave some without
# a tile (test_gated_mlp_cpu.py holds the planner to it).
LARGE = [(2928, 16, 12720, 8), (320, 24, 18976, 8), (13232, 536, 8, 544), (17, 512, 12232, 1080), (6931, 48, 24, 2008), (5557, 264, 6344, 96), (2485, 40, 4904, 1920), (6225, 672, 16, 96)]


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large_calls(vb, shape, dtype, act):
    t, dy = make(*shape, dtype)
    ref = reference(t, dy, act, dtype)
    got = run(vb, t, dy, act)
    compare(got, ref, dtype)
    del ref
    again = run(vb, t, dy, act)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kernels", ["many_tokens", "few_tokens", "unaligned"])
def test_gates_of_any_size(vb, kernels, dtype, act):
    """Up to the type's largest: the activation is the gate or zero, its derivative one or zero."""
    top = 15 if dtype == torch.float16 else 126
    g = torch.tensor([s * 2.0 ** e for e in range(7, top + 1, 1 if top == 15 else 7) for s in (1, -1)], device="cuda").to(dtype)
    g = torch.cat((g, torch.ones(20, device="cuda", dtype=dtype)))
    per = 13 if kernels == "few_tokens" else g.numel()
    parts = [single_gates(vb, c, act, offset=1 if kernels == "unaligned" else 0) for c in g.split(per)]
    y, dv, dg = (torch.cat(p)[:-20] for p in zip(*parts))
    g = g[:-20]
    for x, yes in ((y, g), (dv, g), (dg, torch.ones_like(g))):
        assert torch.equal(x, torch.where(g > 0, yes, torch.zeros_like(yes)))
