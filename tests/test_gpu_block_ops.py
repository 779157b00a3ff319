"""GPU tests of the operators around the shard against plain forms in 64 bits.

Tolerances count roundings.  ``u`` is half a step of an output's type; the fp32 work before the one rounding is bounded by
``FP32`` times the same formula with every term replaced by its magnitude, which also covers sums that cancel: a row's
sum of up to 16384 squares is at most 32 terms per thread, 5 shuffles and 16 warps deep, a column's sum at most
2 + 19 + 8 deep per 300 rows, and the elementwise steps add fewer than 20 roundings of 2^-24 each, so 2^-18 = 64 of them
holds.  Single tensor-core steps may drop a bit more than a rounding, so the 4-bit products get 2^-17."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FP32, MMA = 2.0 ** -18, 2.0 ** -17
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
D = torch.float64
SMALLEST = {BF: 2.0 ** -134, HF: 2.0 ** -25, F: 2.0 ** -150}       # half of the smallest step near zero


@pytest.fixture(scope="module")
def op(pkg):
    return pkg.op


@pytest.fixture
def g():
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    return gen


def near(got, ref, size, c=FP32):
    """got = ref rounded once, up to c times the magnitude of what was added up."""
    assert got.shape == ref.shape
    d = (got.to(D) - ref).abs()
    ok = d <= torch.finfo(got.dtype).eps / 2 * ref.abs() * (1 + 2 * c) + 2 * c * size + SMALLEST[got.dtype]
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, worst {float((d / (size + 1e-300)).max()):.3g} of the size"


# ---------------------------------------------------------------------------- block norm


def norm_ref(x, pre, y=None, post=None, gate=None, a=1.0, eps=1e-6):
    """(s, h, rstd, magnitude of s, magnitude of h)."""
    x, w = x.to(D), pre.to(D)
    s, size, r1 = x, x.abs(), torch.zeros_like(x[:, :1])
    if y is not None:
        n = y.to(D)
        if post is not None:
            r1 = ((n * n).mean(1, keepdim=True) + eps).rsqrt()
            n = n * r1 * post.to(D)
        n = n if gate is None else n * gate.to(D)
        s, size = a * x + n, abs(a) * x.abs() + n.abs()
    r2 = ((s * s).mean(1, keepdim=True) + eps).rsqrt()
    # a rounding of s moves r2 as far as its row's relative error goes
    moved = (s.abs() * size).sum(1, keepdim=True) / ((s * s).sum(1, keepdim=True) + eps * s.shape[1])
    return s, s * r2 * w, torch.cat([r1, r2], 1), size, (size + s.abs() * moved) * r2 * w.abs()


def norm_inputs(g, T, H, t, gate="none", join=True, post=True, pad=0, shift=0, f32=False):
    rows = lambda s: (torch.randn((T, H + pad + shift), generator=g, device="cuda") * s).to(t)[:, shift:shift + H]  # noqa: E731
    vec = lambda m: (m + 0.2 * torch.randn(H, generator=g, device="cuda")).to(F if f32 else t)  # noqa: E731
    kw = dict(x=rows(1.5), pre_weight=vec(1.0))
    if join:
        kw.update(y=rows(0.7), residual_scale=0.75)
        if post:
            kw["post_weight"] = vec(0.5)
        if gate == "channel":
            kw["gate"] = vec(0.3)
        elif gate == "token":
            kw["gate"] = torch.rand((T, 3), generator=g, device="cuda").to(F if f32 else t)[:, 1:2]
        elif gate == "full":
            kw["gate"] = rows(1.0).to(F if f32 else t)
    return kw


def ref_args(kw):
    return (kw["x"], kw["pre_weight"], kw.get("y"), kw.get("post_weight"), kw.get("gate"), kw.get("residual_scale", 1.0))


NORM = [
    # T, H, type, gate, join, post, pad, shift, fp32 parameters
    (1, 7168, BF, "none", True, True, 0, 0, False),
    (2, 1, F, "none", True, True, 0, 0, False),
    (3, 1, BF, "token", False, False, 3, 0, False),
    (5, 7, HF, "channel", True, True, 0, 0, False),
    (149, 8, BF, "full", True, True, 8, 0, False),
    (9, 9, F, "full", True, False, 2, 1, False),
    (300, 128, BF, "token", True, True, 0, 0, True),
    (33, 127, HF, "full", True, True, 0, 0, True),
    (40, 1543, F, "channel", True, True, 9, 0, False),
    (40, 1544, BF, "channel", True, False, 0, 3, True),
    (301, 2048, HF, "full", True, True, 0, 0, False),
    (17, 2056, F, "none", False, False, 0, 0, False),
    (150, 7168, BF, "token", True, True, 24, 0, False),
    (150, 7168, BF, "channel", True, True, 0, 0, True),
    (20, 7168, F, "full", True, True, 0, 0, False),
    (20, 7168, HF, "none", True, False, 0, 0, False),
    (6, 8192, BF, "channel", True, True, 0, 0, False),
    (6, 8200, BF, "channel", True, True, 0, 0, False),
    (5, 8209, HF, "channel", True, True, 0, 0, False),
    (4, 16384, F, "channel", True, True, 0, 0, False),
    (4, 16384, BF, "token", True, True, 0, 0, True),
    (3, 16383, BF, "full", True, True, 0, 0, False),
    # rows that start anywhere, several per CTA, so that every stage of a ring is used again
    (1900, 1001, BF, "channel", True, True, 0, 0, False),
    (700, 4099, BF, "full", True, True, 0, 1, False),
    (650, 3001, HF, "token", True, True, 5, 1, False),
    (601, 5003, F, "channel", True, False, 2, 1, False),
    (460, 8191, BF, "none", True, True, 0, 0, False),
    (900, 2304, BF, "token", True, True, 3, 2, False),
    (1500, 770, HF, "none", False, False, 0, 0, False),
    (2500, 640, BF, "full", True, True, 0, 0, False),
    (1, 1001, BF, "channel", True, True, 0, 0, False),
    (2, 517, F, "token", True, True, 0, 3, False),
    (500, 6001, HF, "full", True, True, 3, 0, False),
    (340, 4104, BF, "channel", True, True, 5, 0, False),
    (620, 7168, BF, "full", True, False, 8, 0, False),
]


@pytest.mark.parametrize("T,H,t,gate,join,post,pad,shift,f32", NORM)
def test_block_norm(op, g, T, H, t, gate, join, post, pad, shift, f32):
    kw = norm_inputs(g, T, H, t, gate, join, post, pad, shift, f32)
    s, h, rstd = op.block_norm(**kw)
    rs, rh, rr, size_s, size_h = norm_ref(*ref_args(kw))
    if join:
        near(s, rs, size_s)
    else:
        assert s is kw["x"]
    near(h, rh, size_h)
    near(rstd, rr, rr * (1 + size_h.sum(1, keepdim=True) / rh.abs().sum(1, keepdim=True).clamp(min=1e-30)))
    again = op.block_norm(**kw)
    assert torch.equal(h, again[1]) and torch.equal(rstd, again[2])


def norm_grad_ref(gh, gs, rstd, x, pre, y=None, post=None, gate=None, a=1.0):
    """{argument: (gradient, magnitude)} from the formulas, the statistics as given."""
    gh, x, w = gh.to(D), x.to(D), pre.to(D)
    r1, r2 = rstd.to(D)[:, :1], rstd.to(D)[:, 1:]
    one = torch.ones_like(x[:, :1])
    gt = one if gate is None else gate.to(D)
    s, ms = x, x.abs()
    if y is not None:
        yh = y.to(D) * (r1 if post is not None else 1.0)
        n = yh * (post.to(D) if post is not None else 1.0)
        s, ms = a * x + gt * n, abs(a) * x.abs() + (gt * n).abs()
    sh, msh, u = s * r2, ms * r2, gh * w
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    d = r2 * (u - sh * mean(u * sh))
    md = r2 * (u.abs() + msh * mean(u.abs() * msh))
    out = {"pre_weight": ((gh * sh).sum(0), (gh.abs() * msh).sum(0))}
    if y is None:
        return {**out, "x": (d, md)}
    if gs is not None:
        d, md = d + gs.to(D), md + gs.to(D).abs()
    out["x"] = (a * d, abs(a) * md)
    if gate is not None:
        dg, mg = d * n, md * n.abs()
        along = 0 if gate.dim() == 1 else 1 if gate.shape[1] == 1 and n.shape[1] > 1 else None
        out["gate"] = (dg, mg) if along is None else (dg.sum(along).view(gate.shape), mg.sum(along).view(gate.shape))
    dn, mn = d * gt, md * gt.abs()
    if post is None:
        return {**out, "y": (dn, mn)}
    out["post_weight"] = ((dn * yh).sum(0), (mn * yh.abs()).sum(0))
    v, mv = dn * post.to(D), mn * post.to(D).abs()
    out["y"] = (r1 * (v - yh * mean(v * yh)), r1 * (mv + yh.abs() * mean(mv * yh.abs())))
    return out


@pytest.mark.parametrize("T,H,t,gate,join,post,pad,shift,f32", NORM)
def test_block_norm_backward(op, g, T, H, t, gate, join, post, pad, shift, f32):
    kw = norm_inputs(g, T, H, t, gate, join, post, pad, shift, f32)
    rstd = op.block_norm(**kw)[2]
    gh = torch.randn((T, H + pad), generator=g, device="cuda").to(t)[:, :H]
    gs = torch.randn((T, H), generator=g, device="cuda").to(t) if join and T != 20 else None
    got = op.block_norm_backward(rstd=rstd, grad_h=gh, grad_stream=gs, **kw)
    ref = norm_grad_ref(gh, gs, rstd, *ref_args(kw))
    assert {k for k, v in got.items() if v is not None} == set(ref)
    for k, (r, size) in ref.items():
        assert got[k].dtype == kw[k].dtype and got[k].shape == kw[k].shape
        near(got[k], r, size)
    again = op.block_norm_backward(rstd=rstd, grad_h=gh, grad_stream=gs, **kw)
    assert all(torch.equal(v, again[k]) for k, v in got.items() if v is not None)


def test_block_norm_backward_without_join_takes_the_stream_gradient(op, g):
    """Without y the stream is x itself: its gradient adds to dx."""
    kw = norm_inputs(g, 7, 96, F, join=False)
    _, _, rstd = op.block_norm(**kw)
    gh, gs = (torch.randn((7, 96), generator=g, device="cuda") for _ in range(2))
    d0 = op.block_norm_backward(rstd=rstd, grad_h=gh, **kw)["x"]
    d1 = op.block_norm_backward(rstd=rstd, grad_h=gh, grad_stream=gs, **kw)["x"]
    near(d1, d0.to(D) + gs.to(D), d0.abs().to(D) * 8 + gs.abs().to(D) * 8)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_block_norm_gradient_against_differences(op, g, gate):
    """The 64-bit formula that the kernel is held to is the derivative of the 64-bit forward."""
    kw = norm_inputs(g, 5, 24, F, gate)
    gh, gs = (torch.randn((5, 24), generator=g, device="cuda") for _ in range(2))
    wide = {k: v.to(D) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    ref = norm_grad_ref(gh, gs, norm_ref(*ref_args(wide))[2], *ref_args(wide))

    def value(at):
        s, h = norm_ref(*ref_args(at))[:2]
        return float((s * gs.to(D)).sum() + (h * gh.to(D)).sum())
    got = op.block_norm_backward(rstd=op.block_norm(**kw)[2], grad_h=gh, grad_stream=gs, **kw)
    for k, (r, size) in ref.items():
        v = torch.randn(r.shape, generator=g, device="cuda", dtype=D)
        e = 1e-5
        up, down = dict(wide, **{k: wide[k] + e * v}), dict(wide, **{k: wide[k] - e * v})
        diff = (value(up) - value(down)) / (2 * e)
        # differences of values near 1e2 in 64 bits over 2e-5, and a third derivative times 1e-10
        assert abs(diff - float((r * v).sum())) < 1e-6 * (1 + float((r * v).abs().sum()))
        assert abs(diff - float((got[k].to(D) * v).sum())) < 1e-4 * (1 + float((size * v.abs()).sum()))


def test_block_norm_of_no_tokens(op, g):
    kw = norm_inputs(g, 0, 64, BF, "channel")
    s, h, rstd = op.block_norm(**kw)
    assert s.shape == h.shape == (0, 64) and rstd.shape == (0, 2)
    got = op.block_norm_backward(rstd=rstd, grad_h=h, grad_stream=s, **kw)
    assert got["x"].shape == (0, 64) and all(not bool(got[k].any()) for k in ("pre_weight", "post_weight", "gate"))
    (q, scale) = op.block_norm(kw["x"].new_empty((0, 128)), kw["x"].new_ones(128), quantize=True)[1]
    assert q.shape == (0, 128) and scale.shape == (1, 0)


def test_block_norm_of_rows_of_zeros_and_large_values(op):
    x = torch.zeros((3, 256), device="cuda")
    x[1] = 1e18                                          # the mean of its squares is 1e36
    x[2, 7] = float("nan")
    w = torch.ones(256, device="cuda")
    _, h, rstd = op.block_norm(x, w)
    assert not bool(h[0].any()) and abs(float(rstd[0, 1]) - 1e3) < 1e-3
    assert float((h[1] - 1).abs().max()) < 1e-6 and bool(h[2].isnan().all())
    grads = op.block_norm_backward(x[:2], w, rstd[:2].contiguous(), torch.ones_like(x[:2]))
    assert bool(torch.isfinite(grads["x"]).all())


@pytest.mark.parametrize("T,H,t,gate", [(1, 7168, BF, "token"), (131, 7168, BF, "channel"), (37, 128, F, "none"),
                                        (5, 16384, HF, "full"), (150, 2176, BF, "token")])
def test_block_norm_quantized(op, g, T, H, t, gate):
    """e4m3 of the unrounded h with max / 448 per 128 columns: the result is within half an e4m3 step of h / scale."""
    kw = norm_inputs(g, T, H, t, gate)
    s, (q, scale), rstd = op.block_norm(**kw, quantize=True)
    plain = op.block_norm(**kw)
    assert torch.equal(s, plain[0]) and torch.equal(rstd, plain[2])
    _, rh, _, _, size = norm_ref(*ref_args(kw))
    blocks = rh.unflatten(1, (-1, 128))
    ref_scale = blocks.abs().amax(2).t() / 448
    near(scale, ref_scale, size.unflatten(1, (-1, 128)).amax(2).t() / 448)
    wide = scale.to(D).t().repeat_interleave(128, 1)
    v = rh / wide
    # half a step is 2^-4 of a value, 2^-10 below 2^-6
    assert bool(((q.to(D) - v).abs() <= torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10) + 4 * FP32 * size / wide).all())
    assert float(q.to(F).abs().max()) == 448.0


def test_block_norm_quantizes_as_the_activation_quantiser_does(op, g):
    """Rows of +-1 keep their norm factor at 1, so h is the weights with signs, exactly, and both ways to the shard's input
    see the same values: the same scales and codes."""
    for k in range(20):
        x = torch.where(torch.rand((33, 7168), generator=g, device="cuda") < 0.5, -1.0, 1.0).to(BF)
        w = torch.randn(7168, generator=g, device="cuda") * 2.0 ** torch.randint(-12, 12, (7168,), generator=g, device="cuda")
        w[::128] = 448.0 * 2.0 ** (k - 10)                 # quotients of few bits, ties of e4m3 among them
        w = w.to(BF)
        _, (q, scale), rstd = op.block_norm(x, w, eps=1e-30, quantize=True)
        assert bool((rstd[:, 1] == 1).all())
        want_q, want_scale = op.quantize_activations((x.float() * w.float()).to(BF))
        assert torch.equal(scale, want_scale)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


def test_block_norm_quantized_infinite_values(op):
    """One infinite value of h: its block has an infinite scale, zeros, and NaN in its place."""
    x = torch.ones((2, 256), device="cuda")
    w = torch.ones(256, device="cuda")
    w[3] = float("inf")
    q, scale = op.block_norm(x, w, quantize=True)[1]
    v = q.to(F)
    assert bool(scale[0].isinf().all()) and bool(v[:, 3].isnan().all()) and bool((v[:, 128:] == 448).all())
    assert not bool(v[:, :3].any()) and not bool(v[:, 4:128].any())


def test_block_norm_quantized_zero_rows(op):
    q, scale = op.block_norm(torch.zeros((2, 256), device="cuda"), torch.ones(256, device="cuda"), quantize=True)[1]
    assert not bool(q.to(F).any())
    floor = torch.full_like(scale, 1e-10, dtype=D) / 448
    near(scale, floor, floor)


def test_block_norm_quantized_near_the_largest_values(op):
    """h up to 3e38: the scale stays finite and the largest value of a block is 448 steps of it."""
    x = torch.ones((2, 256), device="cuda")
    w = torch.full((256,), 3e38, device="cuda")
    w[128:] = 1e-20
    q, scale = op.block_norm(x, w, quantize=True)[1]
    assert bool((q[:, :128].to(F) == 448).all()) and bool(torch.isfinite(scale).all())
    assert abs(float(scale[0, 0]) * 448 / 3e38 - 1) < 1e-5
    assert not bool(q[:, 128:].to(F).any())               # 1e-20 over the floor of 1e-10 / 448


# ---------------------------------------------------------------------------- balance loss


def balance_inputs(g, T, E, K, t=F, cu=None, mask=False):
    logits = (torch.randn((T, E + 3), generator=g, device="cuda") * 1.5).to(t)[:, :E]
    idx = torch.rand((T, E), generator=g, device="cuda").argsort(1)[:, :K].to(torch.int32).contiguous()
    idx = torch.where(torch.rand((T, K), generator=g, device="cuda") < 0.5, idx * 3 // 4, idx).contiguous()
    m = torch.rand(T, generator=g, device="cuda") < 0.7 if mask else None
    borders = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    return logits, idx, borders, m


def balance_ref(logits, idx, cu, mask, alpha, scoring):
    """Per sequence: (loss, counts, tokens) and the gradient's value and magnitude per unit of the loss's gradient."""
    T, E = logits.shape
    z = logits.to(D)
    logp = torch.nn.functional.logsigmoid(z) if scoring == "sigmoid" else z
    slope = torch.sigmoid(-z) if scoring == "sigmoid" else torch.ones_like(z)
    p = torch.where((z == float("-inf")).all(1, keepdim=True), 0.0, torch.softmax(logp, 1))
    borders = [0, T] if cu is None else [min(max(int(v), 0), T) for v in cu.tolist()]
    live = torch.ones(T, dtype=torch.bool, device=z.device) if mask is None else mask
    loss, counts, tokens = [], [], []
    grad, size = torch.zeros_like(z), torch.zeros_like(z)
    for lo, hi in zip(borders[:-1], borders[1:]):
        at = torch.arange(lo, hi, device=z.device)
        at = at[live[lo:hi]]
        n = at.numel()
        ids = idx[at].flatten().long()
        c = torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E)
        k = alpha * E / idx.shape[1] / max(n, 1) ** 2
        q = p[at]
        loss.append(k * (c * q.sum(0)).sum())
        counts.append(c)
        tokens.append(n)
        cc = c.to(D) - idx.shape[1] * n // E
        grad[at] = k * q * slope[at] * (cc - (cc * q).sum(1, keepdim=True))
        size[at] = abs(k) * q * slope[at] * (cc.abs() + (cc.abs() * q).sum(1, keepdim=True))
    stack = lambda v, t: torch.stack([torch.as_tensor(e, device=z.device) for e in v]).to(t) if v else torch.empty(0, dtype=t, device=z.device)  # noqa: E731
    return stack(loss, D), stack(counts, torch.int32).view(len(loss), E), stack(tokens, torch.int32), grad, size


BALANCE = [
    # T, E, K, type, borders, mask, scoring
    (1, 256, 8, F, None, False, "sigmoid"),
    (16, 256, 8, BF, None, False, "sigmoid"),
    (32, 1, 1, F, None, False, "softmax"),
    (33, 31, 3, HF, None, True, "sigmoid"),
    (1000, 256, 8, F, None, True, "sigmoid"),
    (20001, 256, 8, F, None, False, "sigmoid"),
    (20001, 64, 2, BF, [0, 7, 7, 8, 19000], True, "softmax"),
    (4099, 160, 6, F, list(range(0, 4099, 5)) + [4099], False, "softmax"),
    (777, 1000, 16, F, [0, 0, 0, 1, 32, 33, 64, 500, 500, 777, 777], False, "sigmoid"),
    (700, 1024, 40, BF, [10, 300, 650], True, "sigmoid"),
    (96, 512, 1, HF, [0, 32, 64, 96], False, "softmax"),
    (65, 33, 33, F, [0, 65, 65, 65], False, "sigmoid"),
    (3000, 8, 2, F, [-5, 1500, 9000], True, "sigmoid"),
    (300, 16, 4, F, [0] * 400 + [300], False, "sigmoid"),
    (300, 16, 4, F, [0] + [300] * 400, False, "sigmoid"),
    (50, 100, 4, F, [0], False, "sigmoid"),
]


@pytest.mark.parametrize("T,E,K,t,cu,mask,scoring", BALANCE)
def test_balance_loss(op, g, T, E, K, t, cu, mask, scoring):
    logits, idx, borders, m = balance_inputs(g, T, E, K, t, cu, mask)
    loss, counts, tokens = op.balance_loss(logits, idx, 0.3, cu_seqlens=borders, token_mask=m, scoring=scoring)
    rl, rc, rt, rg, size = balance_ref(logits, idx, borders, m, 0.3, scoring)
    assert torch.equal(counts, rc) and torch.equal(tokens, rt)
    near(loss, rl, rl.abs())
    again = op.balance_loss(logits, idx, 0.3, cu_seqlens=borders, token_mask=m, scoring=scoring)
    assert torch.equal(loss, again[0])
    gl = torch.randn(loss.shape, generator=g, device="cuda")
    got = op.balance_loss_backward(gl, logits, counts, tokens, K, 0.3, cu_seqlens=borders, token_mask=m, scoring=scoring)
    clamped = [0, T] if cu is None else [min(max(v, 0), T) for v in cu]
    scale = torch.zeros((T, 1), device="cuda", dtype=D)
    for i, (lo, hi) in enumerate(zip(clamped[:-1], clamped[1:])):
        scale[lo:hi] = gl[i].to(D)
    assert got.dtype == t
    near(got, rg * scale, size * scale.abs())


def test_balance_gradient_against_differences(op, g):
    logits, idx, cu, m = balance_inputs(g, 40, 24, 3, F, [0, 11, 11, 38], True)
    for scoring in ("sigmoid", "softmax"):
        _, counts, tokens = op.balance_loss(logits, idx, 2.0, cu_seqlens=cu, token_mask=m, scoring=scoring)
        gl = torch.rand(3, generator=g, device="cuda") + 0.5
        got = op.balance_loss_backward(gl, logits, counts, tokens, 3, 2.0, cu_seqlens=cu, token_mask=m, scoring=scoring)
        v = torch.randn(logits.shape, generator=g, device="cuda", dtype=D)
        value = lambda z: float((balance_ref(z, idx, cu, m, 2.0, scoring)[0] * gl.to(D)).sum())  # noqa: E731
        diff = (value(logits.to(D) + 1e-5 * v) - value(logits.to(D) - 1e-5 * v)) / 2e-5
        # 64-bit differences hold 1e-9 here; the gradient itself is fp32
        assert abs(diff - float((got.to(D) * v).sum())) < 1e-5


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_balance_with_masked_experts_and_rows(op, g, scoring):
    """Logits of -inf and the types' lowest value, rows without a score, NaN where the mask hides them, far logits."""
    logits, idx, _, _ = balance_inputs(g, 64, 40, 4)
    logits = logits.contiguous()
    logits[:, 5] = float("-inf")
    logits[3] = float("-inf")
    logits[4] = torch.finfo(F).min
    logits[6:9] -= 95.0                                 # sigmoid(z) leaves the normal range of fp32
    logits[9] -= 3000.0
    logits[11] += 80.0
    idx[7, 2], idx[8, 1] = -1, 40
    mask = torch.ones(64, dtype=torch.bool, device="cuda")
    mask[20:23] = False
    logits[20:23] = float("nan")
    idx[21] = 2 ** 30
    loss, counts, tokens = op.balance_loss(logits, idx, 0.5, token_mask=mask, scoring=scoring)
    rl, rc, rt, rg, size = balance_ref(logits, idx, None, mask, 0.5, scoring)
    assert torch.equal(counts, rc) and int(tokens) == 61
    near(loss, rl, rl.abs())
    got = op.balance_loss_backward(torch.ones(1, device="cuda"), logits, counts, tokens, 4, 0.5, token_mask=mask,
                                   scoring=scoring)
    rg, size = rg.nan_to_num(), size.nan_to_num()
    near(got, rg, size)
    assert not bool(got[20:23].any()) and not bool(got[3].any()) and not bool(got[5:, 5].any())


def test_balance_all_masked_and_empty(op, g):
    logits, idx, _, _ = balance_inputs(g, 10, 16, 2)
    none = torch.zeros(10, dtype=torch.bool, device="cuda")
    loss, counts, tokens = op.balance_loss(logits, idx, 0.5, token_mask=none)
    assert float(loss) == 0 and not bool(counts.any()) and int(tokens) == 0
    assert not bool(op.balance_loss_backward(loss + 1, logits, counts, tokens, 2, 0.5, token_mask=none).any())
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, counts, tokens = op.balance_loss(logits[:0], idx[:0], 0.5, cu_seqlens=cu)
    assert loss.tolist() == [0, 0, 0] and not bool(counts.any()) and tokens.tolist() == [0, 0, 0]
    assert op.balance_loss_backward(loss, logits[:0], counts, tokens, 2, 0.5, cu_seqlens=cu).shape == (0, 16)


# ---------------------------------------------------------------------------- 4-bit products


def matvec_inputs(g, R, N, K, G, t, E=0, zero=False, scale_t=None, pad=0):
    shape = (E, N) if E else (N,)
    r = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
    x = torch.randn((R, K + pad), generator=g, device="cuda").to(t)[:, :K]
    scale = (torch.randn(shape + (K // G,), generator=g, device="cuda") * 0.02).to(scale_t or t)
    return x, r(256, *shape, K // 2), scale, r(16, *shape, K // G) if zero else None


def matvec_ref(x, q, scale, zero):
    """One matrix: (product, sum of magnitudes)."""
    G = x.shape[1] // scale.shape[1]
    w = torch.empty((q.shape[0], x.shape[1]), device=x.device, dtype=D)
    w[:, 0::2], w[:, 1::2] = (q & 15).to(D), (q >> 4).to(D)
    w -= 8.0 if zero is None else zero.to(D).repeat_interleave(G, 1)
    w *= scale.to(D).repeat_interleave(G, 1)
    return x.to(D) @ w.t(), x.to(D).abs() @ w.abs().t()


MATVEC = [
    # R, N, K, G, type, zeros, scale type, padding of x, out type
    (1, 1, 32, 32, BF, False, None, 0, None),
    (1, 7, 64, 32, HF, True, None, 0, F),
    (1, 4096, 7168, 128, BF, False, None, 0, None),
    (1, 16, 7168, 64, BF, True, F, 0, F),
    (2, 17, 96, 32, BF, True, None, 8, None),
    (3, 33, 160, 32, HF, False, F, 0, None),
    (5, 4001, 7168, 64, HF, True, None, 0, None),
    (7, 100, 320, 64, BF, False, None, 0, F),
    (8, 2048, 2048, 32, BF, True, None, 16, None),
    (9, 31, 128, 128, BF, False, None, 0, None),
    (16, 7168, 2048, 128, BF, False, F, 0, None),
    (16, 250, 4096, 128, HF, True, None, 0, None),
    (17, 48, 1152, 128, BF, True, None, 0, None),
    (100, 40, 640, 64, BF, False, None, 0, None),
    (256, 19, 256, 128, HF, False, None, 0, None),
    # more columns than are staged at a time
    (16, 40, 20480, 128, BF, False, None, 0, None),
    (3, 24, 65536, 64, HF, True, None, 0, F),
    (11, 33, 19232, 32, BF, True, None, 0, None),
]


@pytest.mark.parametrize("R,N,K,G,t,zero,st,pad,ot", MATVEC)
def test_matvec(op, g, R, N, K, G, t, zero, st, pad, ot):
    x, q, scale, z = matvec_inputs(g, R, N, K, G, t, 0, zero, st, pad)
    out = op.matvec_w4(x, q, scale, z, out_dtype=ot)
    assert out.dtype == (ot or t)
    near(out, *matvec_ref(x, q, scale, z), MMA)
    assert torch.equal(out, op.matvec_w4(x, q, scale, z, out_dtype=ot))


@pytest.mark.parametrize("T,k,E,N,K,G,t,zero,per_pair,span", [
    (1, 8, 32, 256, 7168, 128, BF, False, False, 40),
    (1, 1, 3, 33, 64, 64, BF, True, True, 3),
    (16, 8, 32, 96, 2048, 128, BF, False, True, 64),
    (16, 8, 4, 50, 512, 32, HF, True, False, 5),
    (16, 16, 2, 40, 256, 64, BF, True, False, 1),          # every pair on one expert
    (13, 3, 7, 130, 384, 128, HF, False, True, 7),
    (256, 1, 5, 17, 128, 128, BF, False, True, 6),
    (16, 8, 32, 100, 1024, 128, BF, False, False, 3),      # more rows on an expert than the batch's size makes likely
    (3, 4, 2, 70, 512, 64, HF, False, False, 1),           # an expert named more than once by a row
    (9, 2, 1000, 33, 256, 32, BF, True, True, 1200),
])
def test_matvec_by_experts(op, g, T, k, E, N, K, G, t, zero, per_pair, span):
    x, q, scale, z = matvec_inputs(g, T * k if per_pair else T, N, K, G, t, E, zero)
    e = torch.randint(0, span, (T, k), generator=g, device="cuda", dtype=torch.int32)
    e = torch.where(torch.rand((T, k), generator=g, device="cuda") < 0.1, -3, e).to(torch.int32).contiguous()
    out = op.matvec_w4(x, q, scale, z, experts=e.view(-1) if per_pair else e).view(T * k, N)
    ref, size = (torch.zeros((T * k, N), device="cuda", dtype=D) for _ in range(2))
    for r, v in enumerate(e.flatten().tolist()):
        if 0 <= v < E:
            row = x[r:r + 1] if per_pair else x[r // k:r // k + 1]
            a, b = matvec_ref(row, q[v], scale[v], None if z is None else z[v])
            ref[r], size[r] = a[0], b[0]
    near(out, ref, size, MMA)
    outside = ((e < 0) | (e >= E)).flatten()
    assert not bool(out[outside].any())


@pytest.mark.parametrize("T,k,per_pair", [(1, 8, False), (1, 1, True), (16, 8, False), (16, 8, True), (256, 1, True)])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("ot", [None, F])
def test_matvec_when_no_expert_is_held(op, g, T, k, per_pair, far, ot):
    """A batch whose choices all lie on other shards, in front of this one's experts and behind them: zeros everywhere."""
    E, N, K = 4, 100, 512
    x, q, scale, z = matvec_inputs(g, T * k if per_pair else T, N, K, 64, BF, E, True)
    e = torch.randint(E, 2 ** 31 - 1 if far else E + 3, (T, k), generator=g, device="cuda", dtype=torch.int32)
    e = torch.where(torch.rand((T, k), generator=g, device="cuda") < 0.5, e, E - 1 - e).contiguous()
    assert not bool(((e >= 0) & (e < E)).any())
    out = op.matvec_w4(x, q, scale, z, experts=e.view(-1) if per_pair else e, out_dtype=ot)
    assert out.shape == ((T * k, N) if per_pair else (T, k, N)) and not bool(out.any())


def test_matvec_of_no_rows(op, g):
    x, q, scale, _ = matvec_inputs(g, 0, 5, 64, 32, BF)
    assert op.matvec_w4(x, q, scale).shape == (0, 5)
    x, q, scale, _ = matvec_inputs(g, 2, 5, 64, 32, BF, 3)
    assert op.matvec_w4(x, q, scale, experts=torch.empty((2, 0), dtype=torch.int32, device="cuda")).shape == (2, 0, 5)


@pytest.mark.parametrize("t,ot", [(BF, F), (HF, F), (BF, None), (HF, None)])
@pytest.mark.parametrize("R,N,K,G,zero,spread,E", [
    (1, 512, 7168, 128, False, 1.5, 0), (5, 301, 2048, 64, True, 0.5, 0), (16, 128, 4096, 32, True, 0.3, 0),
    (4, 96, 7168, 128, True, 0.2, 3), (16, 2001, 128, 128, False, 0.2, 0), (9, 999, 64, 64, True, 0.25, 2),
])
def test_matvec_of_weights_near_the_zero_point(op, g, R, N, K, G, zero, spread, E, t, ot):
    """Trained weights lie close around the zero point, and activations have a mean and a few large channels: sum q x and
    z sum x are then far larger than their difference, most of all where a large channel's weight is zero.  For an fp32 result q - z is exact and the error goes with sum |(q - z) x| all the same;
    for a 16-bit one it goes with sum (q + z) |x|."""
    x, q, scale, z = matvec_inputs(g, R, N, K, G, t, E, zero)
    x = (x.float() + 1.0).to(t)
    shape = ((E, N) if E else (N,)) + (K // G,)
    zf = torch.full(shape, 8.0, device="cuda") if z is None else z.float()
    v = (zf[..., None] + spread * torch.randn(shape + (G,), generator=g, device="cuda")).round().clamp(0, 15).to(torch.uint8)
    v[..., 5] = zf
    v = v.flatten(-2)
    x[:, 5::G] *= 2.0 ** 12
    q = (v[..., 0::2] | v[..., 1::2] << 4).contiguous()
    e = torch.randint(0, E, (R, 2), generator=g, device="cuda", dtype=torch.int32) if E else None
    out = op.matvec_w4(x, q, scale, z, experts=e, out_dtype=ot)

    def ref(i, x):
        at = (lambda v: v if v is None or i is None else v[i])  # noqa: E731
        r, size = matvec_ref(x, at(q), at(scale), at(z))
        if ot is None:
            both = at(v).to(D) + at(zf).to(D).repeat_interleave(G, -1)
            size = size + x.to(D).abs() @ (both * at(scale).to(D).abs().repeat_interleave(G, -1)).t()
        return r, size
    if not E:
        near(out, *ref(None, x), MMA)
        return
    for r in range(R):
        for k in range(2):
            a, b = ref(int(e[r, k]), x[r:r + 1])
            near(out[r, k], a[0], b[0], MMA)


@pytest.mark.parametrize("t,sizes", [(BF, [2.0 ** 110, 2.0 ** 63, 1.0, 2.0 ** -57, 2.0 ** -100]), (HF, [2.0 ** 10, 1.0, 2.0 ** -10, 2.0 ** -20])])
@pytest.mark.parametrize("zero", [False, True])
def test_matvec_over_the_activations_range(op, g, t, sizes, zero):
    """A row of every order of magnitude that the type has, each held to its own error."""
    for f32 in (False, True):
        x, q, scale, z = matvec_inputs(g, len(sizes), 130, 1024, 128, t, 0, zero, F if f32 else None)
        x = (x.float() * torch.tensor(sizes, device="cuda")[:, None]).to(t)
        near(op.matvec_w4(x, q, scale, z, out_dtype=F), *matvec_ref(x, q, scale, z), MMA)


@pytest.mark.parametrize("zero", [False, True])
def test_matvec_over_the_range_of_16_bit_results(op, g, zero):
    """bf16 activations just below 2^63 and around 2^-57; fp16 ones as large as the result allows and subnormal."""
    for t, sizes in ((BF, [2.0 ** 60, 2.0 ** 30, 2.0 ** -30, 2.0 ** -57]), (HF, [2.0 ** 8, 1.0, 2.0 ** -8, 2.0 ** -16])):
        x, q, scale, z = matvec_inputs(g, 4, 130, 1024, 128, t, 0, zero)
        x = (x.float() * torch.tensor(sizes, device="cuda")[:, None]).to(t)
        if t is BF:
            x[0, ::7] = 2.0 ** 63 * (1 - 2.0 ** -8)       # bf16's largest value below
        near(op.matvec_w4(x, q, scale, z), *matvec_ref(x, q, scale, z), MMA)


@pytest.mark.parametrize("R,N,K,G,t,E,k", [(1, 33, 2 ** 20, 32, BF, 0, 0), (16, 17, 2 ** 20, 128, HF, 0, 0), (9, 100, 2 ** 18 + 64, 64, BF, 0, 0),
                                           (5, 20, 2 ** 17, 32, HF, 2, 3), (2, 40, 2 ** 15 + 32, 32, BF, 0, 0)])
def test_matvec_of_long_rows(op, g, R, N, K, G, t, E, k):
    """Equal activations and weights, so that all terms have one sign and every addition rounds the same way: a thread adds
    at most 8 + 128 sums in a row, and 16 warps meet: 2^-17 of the sum with the few roundings of a group."""
    x, q, scale, _ = matvec_inputs(g, R, N, K, G, t, E)
    x = x[:, :1].abs().expand(R, K).contiguous()
    scale = scale[..., :1].expand(scale.shape).contiguous().float()
    q.fill_(13 * 17)
    e = torch.randint(0, E, (R, k), generator=g, device="cuda", dtype=torch.int32) if E else None
    out = op.matvec_w4(x, q, scale, experts=e, out_dtype=F)
    for r in range(R):
        for c in range(max(k, 1)):
            w = scale[int(e[r, c])] if E else scale
            ref = float(x[r, 0]) * 5 * K * w[:, 0].to(D)
            near(out[r, c] if E else out[r], ref, ref.abs(), MMA)


@pytest.mark.parametrize("t", [BF, HF])
def test_matvec_of_infinite_activations(op, g, t):
    """One infinite activation gives its weight's sign, and NaN where the weight is zero."""
    x, q, scale, _ = matvec_inputs(g, 2, 40, 256, 64, t)
    x[0, 9] = float("inf")
    out = op.matvec_w4(x, q, scale.abs(), out_dtype=F)
    w = (q[:, 4] >> 4).float() - 8
    assert bool(out[0][w == 0].isnan().all()) and torch.equal(out[0][w != 0], w[w != 0] * float("inf"))
    near(out[1], *(v[1] for v in matvec_ref(x, q, scale.abs(), None)), MMA)


def test_matvec_infinities_stay_in_their_row(op, g):
    x, q, scale, _ = matvec_inputs(g, 3, 20, 256, 64, BF)
    x[1, 9] = float("inf")
    out = op.matvec_w4(x, q, scale)
    ref, size = matvec_ref(x[::2], q, scale, None)
    near(out[::2].contiguous(), ref, size, MMA)
    assert not bool(torch.isfinite(out[1]).any())


# ---------------------------------------------------------------------------- together, streams, graphs


def test_a_block_as_it_is_used(op, pkg, g):
    """Join and norm -> route -> balance loss -> the shard's experts -> join, the parts fed with one another's outputs."""
    T, dev, gen = 24, torch.device("cuda", 0), pkg.gen
    tok = gen.make_tokens(T, 3, dev)
    W = gen.make_shard_weights(0, dev, experts=list(range(32)))
    kw = norm_inputs(g, T, 7168, BF, "token")
    stream, (q, scale), rstd = op.block_norm(**kw, quantize=True)
    router = (torch.randn((256, 7168), generator=g, device=dev) * 7168 ** -0.5).to(BF)
    logits = (op.block_norm(stream, kw["pre_weight"])[1] @ router.t()).float()
    idx, weight, _ = op.route(logits, tok.routing_bias, 0, 2.5)
    loss, counts, tokens = op.balance_loss(logits, idx, 1e-2)
    rl, rc, _, rg, size = balance_ref(logits, idx, None, None, 1e-2, "sigmoid")
    near(loss, rl, rl.abs())
    assert torch.equal(counts, rc) and int(counts.sum()) == 8 * T and int(tokens) == T
    near(op.balance_loss_backward(torch.ones_like(loss), logits, counts, tokens, 8, 1e-2), rg, size)
    out = op.run(logits, tok.routing_bias, q, scale, W.gemm1_weights, W.gemm1_weights_scale, W.gemm2_weights,
                 W.gemm2_weights_scale, 0, 2.5)
    assert op.kernel_status() == 0
    joined = dict(x=stream, y=out, pre_weight=kw["pre_weight"], post_weight=kw["post_weight"], residual_scale=0.75)
    s, h, rstd = op.block_norm(**joined)
    rs, rh, _, ms, mh = norm_ref(*ref_args(joined))
    near(s, rs, ms)
    near(h, rh, mh)
    # the same experts with 4-bit weights: up, SwiGLU, down, weighted sum
    e = idx[:5].contiguous()
    x5 = op.block_norm(stream[:5], kw["pre_weight"])[1]
    _, q1, s1, _ = matvec_inputs(g, 1, 64, 7168, 128, BF, 32)
    _, q2, s2, z2 = matvec_inputs(g, 1, 96, 32, 32, BF, 32, True)
    up = op.matvec_w4(x5, q1, s1, experts=e, out_dtype=F)
    act = (torch.nn.functional.silu(up[..., 32:]) * up[..., :32]).to(BF)
    down = op.matvec_w4(act.view(40, 32), q2, s2, z2, experts=e.view(-1)).view(5, 8, 96)
    for t in range(5):
        for k in range(8):
            v = int(e[t, k])
            if v >= 32:
                assert not bool(down[t, k].any())
                continue
            a, b = matvec_ref(x5[t:t + 1], q1[v], s1[v], None)
            near(up[t, k], a[0], b[0], MMA)
            a, b = matvec_ref(act[t, k:k + 1], q2[v], s2[v], z2[v])
            near(down[t, k], a[0], b[0], MMA)


def every_call(op, g, T=70):
    """One call of each entry point on fixed buffers: a function that makes them and returns all outputs."""
    kw = norm_inputs(g, T, 640, BF, "channel")
    gh = torch.randn((T, 640), generator=g, device="cuda").to(BF)
    logits, idx, cu, m = balance_inputs(g, T, 48, 4, F, [0, 3, 40, 40, T - 1], True)
    x, q, scale, z = matvec_inputs(g, 4, 70, 512, 64, BF, 6, True)
    e = torch.randint(0, 7, (4, 3), generator=g, device="cuda", dtype=torch.int32)
    gl = torch.rand(4, generator=g, device="cuda")
    inputs = [kw["x"], kw["y"], gh, logits, x]

    def call():
        s, h, rstd = op.block_norm(**kw)
        _, (q8, sc), _ = op.block_norm(**kw, quantize=True)
        grads = op.block_norm_backward(rstd=rstd, grad_h=gh, grad_stream=h, **kw)
        loss, counts, tokens = op.balance_loss(logits, idx, 0.1, cu_seqlens=cu, token_mask=m)
        gz = op.balance_loss_backward(gl, logits, counts, tokens, 4, 0.1, cu_seqlens=cu, token_mask=m)
        out = op.matvec_w4(x, q, scale, z, experts=e)
        return [s, h, rstd, q8.view(torch.uint8), sc, *grads.values(), loss, counts, tokens, gz, out]
    return call, inputs


def test_on_a_stream_of_its_own(op, g):
    call, inputs = every_call(op, g)
    ref = [t.clone() for t in call()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in inputs:
            t.mul_(1.0)                                   # what the calls have to wait for
        got = call()
        got = [t.clone() for t in got]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_waits_for_what_its_stream_has_to_do_first(op, g):
    """The inputs hold other values until a copy on the side stream, behind some milliseconds of work there, replaces them: a
    call that ran on another stream or read too early would see the other values."""
    call, inputs = every_call(op, g)
    final = [t.clone() for t in inputs]
    ref = [t.clone() for t in call()]
    other = [torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in inputs]
    for t, o in zip(inputs, other):
        t.copy_(o)
    stale = [t.clone() for t in call()]
    assert sum(not torch.equal(a, b) for a, b in zip(ref, stale)) == len(ref) - 2      # all but counts and tokens
    a = torch.randn((8192, 8192), generator=g, device="cuda").to(BF)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(8):
            torch.mm(a, a, out=b)
        for t, f in zip(inputs, final):
            t.copy_(f)
        got = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_captured_and_replayed(op, g):
    """Two graphs of the same calls, replayed in turn on new inputs, give what ordinary calls give."""
    call, inputs = every_call(op, g)
    call()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for k in range(4):
        for t in inputs:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        graphs[k % 2].replay()
        if k == 3:
            graphs[0].replay()
        torch.cuda.synchronize()
        ref = call()
        assert all(torch.equal(a, b) for a, b in zip(ref, outs[k % 2]))


def test_rows_far_into_a_long_batch(op, g):
    """Offsets beyond 2^31 elements: the last rows of a 300 000 x 7168 batch (4.3 GB a tensor in 16 bits)."""
    T, H = 300_000, 7168
    x = torch.zeros((T, H), dtype=BF, device="cuda")
    x[-2:] = torch.randn((2, H), generator=g, device="cuda").to(BF)
    w = torch.ones(H, dtype=BF, device="cuda")
    _, h, rstd = op.block_norm(x, w)
    _, rh, rr, _, mh = norm_ref(x[-2:], w)
    near(h[-2:], rh, mh)
    near(rstd[-2:], rr, rr)
    dx = op.block_norm_backward(x, w, rstd, h)["x"]
    r, size = norm_grad_ref(h[-2:], None, rstd[-2:], x[-2:], w)["x"]
    near(dx[-2:], r, size)
    assert not bool(dx[1000:1010].any())


# ---------------------------------------------------------------------------- sums over long batches


@pytest.mark.parametrize("T,H,t,gate,f32", [
    (2 ** 23 + 77, 8, F, "channel", False),       # the ring kernel, thousands of rows per CTA
    (2 ** 22 + 5, 9, F, "channel", False),        # with edges
    (2 ** 22 + 5, 8, BF, "channel", True),        # the other kernel, rows of 16 bytes
    (2 ** 22, 7, HF, "none", True),               # and element by element
    (148 * 256 + 1, 4608, F, "none", False),      # one row more than a wave of CTAs takes
])
def test_weight_gradients_of_a_long_batch(op, g, T, H, t, gate, f32):
    """Equal rows, so that all terms of a column have one sign and every addition rounds the same way.  A CTA adds at most
    256 terms in a row, an error of 256 * 2^-24 / 2 of the sum; what comes after keeps its errors; the terms themselves
    have fewer than 20 roundings: 148 * 2^-24 together, below 2 * 2^-17."""
    row = norm_inputs(g, 1, H, t, gate, f32=f32)
    rows = lambda v: v.expand(T, H).contiguous()  # noqa: E731
    rstd = torch.tensor([[1.37, 0.83]], device="cuda")
    gh, gs = (torch.randn((1, H), generator=g, device="cuda").to(t) for _ in range(2))
    ref = norm_grad_ref(gh, gs, rstd, *ref_args(row))
    got = op.block_norm_backward(rstd=rstd.expand(T, 2).contiguous(), grad_h=rows(gh), grad_stream=rows(gs),
                                 **dict(row, x=rows(row["x"]), y=rows(row["y"])))
    for k in ("pre_weight", "post_weight", "gate"):
        if got[k] is not None:
            near(got[k], ref[k][0] * T, ref[k][1] * T, 2.0 ** -17)
    near(got["x"][-1:], *ref["x"])


def test_weight_gradients_of_infinite_terms(op):
    """An infinite sum stays infinite, a NaN stays in its column."""
    x = torch.ones((40_000, 16), device="cuda")
    gh = torch.ones_like(x)
    gh[5, 1], gh[7, 2], gh[39_999, 3] = float("inf"), float("nan"), float("-inf")
    rstd = torch.ones((40_000, 2), device="cuda")
    dw = op.block_norm_backward(x, torch.ones(16, device="cuda"), rstd, gh)["pre_weight"].tolist()
    assert dw[1] == float("inf") and dw[2] != dw[2] and dw[3] == float("-inf") and dw[4:] == [40_000.0] * 12


@pytest.mark.parametrize("T,E,K,cu", [(2 ** 23 + 3, 2, 1, None), (2 ** 23 + 3, 2, 2, [5, 3_000_001, 8_000_000]), (700_001, 600, 6, None)])
def test_balance_loss_of_a_long_batch(op, g, T, E, K, cu):
    """Equal rows of logits, as above.  256 additions a warp, 32 for a CTA's warps, 148 for rows of chunks: 218 * 2^-24 of the sum
    at most, and a few roundings of the terms: below 2 * 2^-17."""
    _, idx, borders, _ = balance_inputs(g, T, E, K, F, cu)
    logits = torch.randn((1, E), generator=g, device="cuda").expand(T, E).contiguous()
    loss, counts, tokens = op.balance_loss(logits, idx, 0.3, cu_seqlens=borders)
    p = torch.sigmoid(logits[0].to(D))
    p = p / p.sum()
    for q, (lo, hi) in enumerate(zip((cu or [0, T])[:-1], (cu or [0, T])[1:])):
        c = torch.bincount(idx[lo:hi].flatten().long(), minlength=E)
        assert torch.equal(counts[q].long(), c) and int(tokens[q]) == hi - lo
        ref = 0.3 * E / K * (c.to(D) * p).sum() / (hi - lo)
        near(loss[q], ref, ref, 2.0 ** -17)
