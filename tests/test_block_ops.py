"""CPU tests of the operators around the shard: what the Python entry points and the C ABI refuse, before any device is
touched."""
import pytest
import torch

FAKE = 1 << 20          # non-null, aligned; never dereferenced on these paths


@pytest.fixture(scope="module")
def op(pkg):
    pkg.build.build()
    return pkg.op


def norm_args(T=4, H=256, t=torch.bfloat16):
    z = lambda *s: torch.zeros(s, dtype=t)  # noqa: E731
    return dict(x=z(T, H), pre_weight=z(H), y=z(T, H), post_weight=z(H), gate=z(T, 1), residual_scale=0.5)


@pytest.mark.parametrize("change, says", [
    (dict(x=torch.zeros(4, 256, dtype=torch.float64)), "x must be"),
    (dict(x=torch.zeros(256, dtype=torch.bfloat16)), "x must be"),
    (dict(x=torch.zeros(4, 16385, dtype=torch.bfloat16)), "columns"),
    (dict(x=torch.zeros(256, 4, dtype=torch.bfloat16).t()), "adjacent"),
    (dict(y=torch.zeros(3, 256, dtype=torch.bfloat16)), "y must be"),
    (dict(y=torch.zeros(4, 256)), "y must be"),
    (dict(pre_weight=torch.zeros(255, dtype=torch.bfloat16)), "pre_weight"),
    (dict(pre_weight=torch.zeros(256, dtype=torch.float16)), "pre_weight"),
    (dict(post_weight=torch.zeros(512, dtype=torch.bfloat16)[::2]), "post_weight"),
    (dict(gate=torch.zeros(4, 2, dtype=torch.bfloat16)), "gate"),
    (dict(gate=torch.zeros(4, 256, dtype=torch.float16)), "gate"),
    (dict(y=None), "belong to y"),
    (dict(eps=0.0), "eps"),
    (dict(x=torch.zeros(4, 200, dtype=torch.bfloat16), y=None, post_weight=None, gate=None, residual_scale=1.0,
          pre_weight=torch.zeros(200, dtype=torch.bfloat16), quantize=True), "multiple of 128"),
    (dict(x=torch.zeros(4, 260, dtype=torch.bfloat16)[:, 1:257], quantize=True), "aligned"),
    (dict(), "on a GPU"),
])
def test_block_norm_refusals(op, change, says):
    with pytest.raises(ValueError, match=says):
        op.block_norm(**{**norm_args(), **change})


@pytest.mark.parametrize("change, says", [
    (dict(rstd=torch.zeros(4)), "rstd"),
    (dict(grad_h=torch.zeros(4, 255, dtype=torch.bfloat16)), "grad_h"),
    (dict(grad_stream=torch.zeros(4, 256)), "grad_stream"),
    (dict(), "on a GPU"),
])
def test_block_norm_backward_refusals(op, change, says):
    good = dict(rstd=torch.zeros(4, 2), grad_h=torch.zeros(4, 256, dtype=torch.bfloat16), **norm_args())
    with pytest.raises(ValueError, match=says):
        op.block_norm_backward(**{**good, **change})


@pytest.mark.parametrize("change, says", [
    (dict(logits=torch.zeros(4, 16, dtype=torch.float64)), "logits"),
    (dict(logits=torch.zeros(4, 1025)), "columns"),
    (dict(logits=torch.zeros(16, 4).t()), "adjacent"),
    (dict(topk_idx=torch.zeros(4, 2, dtype=torch.int64)), "topk_idx"),
    (dict(topk_idx=torch.zeros(5, 2, dtype=torch.int32)), "topk_idx"),
    (dict(topk_idx=torch.zeros(4, 17, dtype=torch.int32)), "selects"),
    (dict(topk_idx=torch.zeros(4, 0, dtype=torch.int32)), "selects"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), "cu_seqlens"),
    (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), "cu_seqlens"),
    (dict(token_mask=torch.ones(3, dtype=torch.bool)), "token_mask"),
    (dict(token_mask=torch.ones(4, dtype=torch.uint8)), "token_mask"),
    (dict(scoring="relu"), "scoring"),
    (dict(), "on a GPU"),
])
def test_balance_loss_refusals(op, change, says):
    good = dict(logits=torch.zeros(4, 16), topk_idx=torch.zeros(4, 2, dtype=torch.int32), alpha=0.1)
    with pytest.raises(ValueError, match=says):
        op.balance_loss(**{**good, **change})


@pytest.mark.parametrize("change, says", [
    (dict(grad_loss=torch.zeros(2)), "grad_loss"),
    (dict(counts=torch.zeros(1, 15, dtype=torch.int32)), "counts"),
    (dict(tokens=torch.zeros(1)), "tokens"),
    (dict(top_k=0), "selects"),
    (dict(), "on a GPU"),
])
def test_balance_loss_backward_refusals(op, change, says):
    good = dict(grad_loss=torch.zeros(1), logits=torch.zeros(4, 16), counts=torch.zeros(1, 16, dtype=torch.int32),
                tokens=torch.zeros(1, dtype=torch.int32), top_k=2, alpha=0.1)
    with pytest.raises(ValueError, match=says):
        op.balance_loss_backward(**{**good, **change})


def matvec_args(R=4, N=8, K=256, G=64, E=3):
    return dict(x=torch.zeros(R, K, dtype=torch.bfloat16), qweight=torch.zeros(E, N, K // 2, dtype=torch.uint8),
                scale=torch.zeros(E, N, K // G), zero=torch.zeros(E, N, K // G, dtype=torch.uint8),
                experts=torch.zeros(R, 2, dtype=torch.int32))


@pytest.mark.parametrize("change, says", [
    (dict(x=torch.zeros(4, 256)), "x must be"),
    (dict(x=torch.zeros(4, 260, dtype=torch.bfloat16)[:, :256]), "aligned"),
    (dict(x=torch.zeros(4, 264, dtype=torch.bfloat16)[:, 1:257]), "aligned"),
    (dict(qweight=torch.zeros(8, 128, dtype=torch.uint8)), "qweight"),
    (dict(qweight=torch.zeros(3, 8, 127, dtype=torch.uint8)), "qweight"),
    (dict(qweight=torch.zeros(3, 8, 128, dtype=torch.int8)), "qweight"),
    (dict(scale=torch.zeros(3, 8, 16)), "scale"),
    (dict(scale=torch.zeros(3, 8, 3)), "scale"),
    (dict(scale=torch.zeros(3, 7, 4)), "scale"),
    (dict(scale=torch.zeros(3, 8, 4, dtype=torch.float16)), "scale"),
    (dict(zero=torch.zeros(3, 8, 2, dtype=torch.uint8)), "zero"),
    (dict(experts=torch.zeros(4, 2, dtype=torch.int64)), "experts"),
    (dict(experts=torch.zeros(5, dtype=torch.int32)), "experts"),
    (dict(experts=torch.zeros(4, 65, dtype=torch.int32)), "256"),
    (dict(qweight=torch.zeros(3, 8, 129, dtype=torch.uint8).view(-1)[8:8 + 3 * 8 * 128].view(3, 8, 128)), "aligned"),
    (dict(out_dtype=torch.float16), "out_dtype"),
    (dict(experts=None), "qweight"),
    (dict(), "on a GPU"),
])
def test_matvec_refusals(op, change, says):
    with pytest.raises(ValueError, match=says):
        op.matvec_w4(**{**matvec_args(), **change})


def test_c_entry_points_refuse_before_touching_a_device(op, pkg):
    lib, F = pkg.loader.lib, pkg.loader
    norm = [FAKE, 256, None, 0, None, 0, 0, FAKE, None, 4, 256, F.BF16, 0, 1.0, 1e-6, None, FAKE, None, FAKE, None]

    def call(fn, good, **at):
        args = list(good)
        for k, v in at.items():
            args[int(k[1:])] = v
        return fn(*args)
    f = lib.moe_fp8_block_scale_block_norm
    assert call(f, norm, _9=0) == F.OK
    for bad in (dict(_9=-1), dict(_10=0), dict(_10=16385), dict(_11=3), dict(_12=8), dict(_6=4), dict(_6=1), dict(_8=FAKE),
                dict(_14=0.0), dict(_14=float("nan")), dict(_0=None), dict(_7=None), dict(_16=None), dict(_18=None),
                dict(_2=FAKE), dict(_10=200, _17=FAKE), dict(_0=FAKE + 2, _17=FAKE), dict(_1=255, _17=FAKE)):
        assert call(f, norm, **bad) == F.EINVAL, bad
    back = [FAKE, 256, None, 0, None, 0, 0, FAKE, None, 4, 256, F.BF16, 0, 1.0, FAKE, FAKE, 256, None, 0, FAKE, None, None,
            FAKE, None, FAKE, 1 << 40, None]
    f = lib.moe_fp8_block_scale_block_norm_backward
    assert call(f, back, _9=0) == F.OK
    for bad in (dict(_9=-1), dict(_10=16385), dict(_14=None), dict(_15=None), dict(_19=None), dict(_22=None),
                dict(_24=None), dict(_24=FAKE + 4), dict(_2=FAKE), dict(_2=FAKE, _20=FAKE, _8=FAKE),
                dict(_2=FAKE, _20=FAKE, _4=FAKE, _6=1)):
        assert call(f, back, **bad) == F.EINVAL, bad
    assert call(f, back, _25=16) == F.EWORKSPACE
    assert lib.moe_fp8_block_scale_block_norm_backward_workspace_bytes(-1, 8) == 0
    loss = [FAKE, 256, F.F32, FAKE, 4, 256, 8, None, 1, None, 0, 0.1, FAKE, FAKE, FAKE, FAKE, 1 << 40, None]
    f = lib.moe_fp8_block_scale_balance_loss
    assert call(f, loss, _7=FAKE, _8=0) == F.OK
    for bad in (dict(_0=None), dict(_2=3), dict(_3=None), dict(_4=-1), dict(_5=0), dict(_5=1025), dict(_6=0), dict(_6=257),
                dict(_8=2), dict(_8=-1), dict(_10=2), dict(_12=None), dict(_15=None), dict(_15=FAKE + 1), dict(_0=FAKE + 2),
                dict(_3=FAKE + 1), dict(_7=FAKE + 2), dict(_4=(1 << 30) + 1)):
        assert call(f, loss, **bad) == F.EINVAL, bad
    assert call(f, loss, _16=16) == F.EWORKSPACE
    back = [FAKE, FAKE, 256, F.F32, FAKE, FAKE, 4, 256, 8, None, 1, None, 0, 0.1, FAKE, None]
    f = lib.moe_fp8_block_scale_balance_loss_backward
    assert call(f, back, _6=0) == F.OK
    for bad in (dict(_0=None), dict(_1=None), dict(_4=None), dict(_5=None), dict(_7=1025), dict(_14=None), dict(_12=-1)):
        assert call(f, back, **bad) == F.EINVAL, bad
    mv = [FAKE, 256, F.BF16, FAKE, FAKE, 0, None, None, 4, 1, 1, 16, 256, 128, FAKE, 0, None]
    f = lib.moe_fp8_block_scale_matvec_w4
    assert call(f, mv, _8=0) == F.OK
    for bad in (dict(_0=None), dict(_0=FAKE + 2), dict(_1=255), dict(_2=F.F32), dict(_3=None), dict(_3=FAKE + 4),
                dict(_4=None), dict(_8=257), dict(_8=-1), dict(_9=0), dict(_9=3), dict(_10=2), dict(_11=0), dict(_12=200),
                dict(_13=16), dict(_14=None), dict(_14=FAKE + 1), dict(_4=FAKE + 1), dict(_7=FAKE + 2), dict(_11=(1 << 22) + 1)):
        assert call(f, mv, **bad) == F.EINVAL, bad


def test_c_entry_points_refuse_results_that_are_not_aligned_to_their_elements(op, pkg):
    """A pointer between two elements would be a misaligned store on the device."""
    lib, F = pkg.loader.lib, pkg.loader
    for dtype, param_f32, element in ((F.F32, 0, 4), (F.BF16, 0, 2), (F.F16, 7, 4)):
        for off in range(1, element):
            def backward(kind, grads):
                return lib.moe_fp8_block_scale_block_norm_backward(
                    FAKE, 256, FAKE, 256, FAKE, 256, kind, FAKE, FAKE, 4, 256, dtype, param_f32, 1.0, FAKE, FAKE, 256, None, 0,
                    FAKE, FAKE, *[FAKE + off if k == grads else FAKE for k in ("gate", "pre", "post")], FAKE, 1 << 40, None)
            for kind in (1, 2, 3):
                for grads in ("gate", "pre", "post"):
                    assert backward(kind, grads) == F.EINVAL, (dtype, off, kind, grads)
    for off in (1, 2, 3):
        assert lib.moe_fp8_block_scale_block_norm(FAKE, 256, None, 0, None, 0, 0, FAKE, None, 4, 256, F.BF16, 0, 1.0, 1e-6,
                                                  None, FAKE, FAKE + off, FAKE, None) == F.EINVAL, off


@pytest.mark.parametrize("getters", [True, False])
@pytest.mark.parametrize("current", [0, 1])
def test_launches_on_the_tensors_device_with_its_stream(op, monkeypatch, getters, current):
    """Also where another device is current, and with a torch build that lacks the raw getters; on stand-ins for the
    device's state."""
    state = {"device": current}

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *exc):
            state["device"] = self.before

    class Stream:
        def __init__(self, dev):
            self.cuda_stream = 100 + (dev if isinstance(dev, int) else dev.index)

    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    if getters:
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"], raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    monkeypatch.setattr(torch.cuda, "device", device)
    seen = []

    def entry(*args):
        seen.append((state["device"], args))
        return 0
    op._launch(entry, torch.device("cuda", 1), 7, 8)
    assert seen == [(1, (7, 8, 101))] and state["device"] == current
    with pytest.raises(op.loader.MoeLibraryError):
        op._launch(lambda *args: op.loader.EINVAL, torch.device("cuda", 1))


@pytest.mark.parametrize("eps", [1e-60, 0.0, -1e-6, float("nan")])
def test_block_norm_refuses_an_eps_that_fp32_does_not_hold(op, eps):
    with pytest.raises(ValueError, match="eps"):
        op.block_norm(**norm_args(), eps=eps)
