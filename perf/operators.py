"""Performance cases of the operators around the shard: the block's norms, the balance loss, 4-bit matrix-vector products.

* ``norm``    -- ``op.block_norm`` and its backward: joins a block's output to the residual stream (norm, gate, residual
  scale) and norms the stream for the next block, as activations or in the shard's e4m3 + block-scale input layout;
* ``balance`` -- ``op.balance_loss`` and its backward: per-sequence balance loss and per-expert counts of a routing;
* ``matvec``  -- ``op.matvec_w4``: up to sixteen tokens times 4-bit weights with group scales, dense or by chosen experts.

``own`` says which side runs: the plain form in elementary torch operations, or the package's kernels.
"""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS, RESIDUAL_SCALE, ALPHA, BLOCK = 1e-6, 0.75, 1e-3, 128
LARGEST_T, LARGEST_H, LARGEST_E = 16384, 7168, 512


def _norm(name, way, T, H, dtype, gate="none", join=True, post=True, quantize=False, pad=0):
    return {"name": name, "op": "norm", "way": way, "T": T, "H": H, "dtype": dtype, "gate": gate, "join": join,
            "post": post, "quantize": quantize, "pad": pad}


def _balance(name, way, T, E, K, dtype="fp32", seqs=0, mask=False, scoring="sigmoid"):
    return {"name": name, "op": "balance", "way": way, "T": T, "E": E, "K": K, "dtype": dtype, "seqs": seqs,
            "mask": mask, "scoring": scoring}


def _matvec(name, T, N, K, G, dtype="bf16", zero=False, E=0, k=0, pool=0, per_pair=False):
    return {"name": name, "op": "matvec", "T": T, "N": N, "K": K, "G": G, "dtype": dtype, "zero": zero, "E": E, "k": k,
            "pool": pool, "per_pair": per_pair}


def listed():
    return [
        # one decoding token between two blocks: latency alone
        _norm("norm_t1", "forward", 1, 7168, "bf16", quantize=True),
        # a prefill chunk: join with a gate per token, norm, and the shard's quantised input in the same pass
        _norm("norm_quant_t4096", "forward", 4096, 7168, "bf16", "token", quantize=True),
        # an odd width in 32 bits with padded rows and a gate per channel (a fine-tuning run's small model)
        _norm("norm_odd_t515", "forward", 515, 1543, "fp32", "channel", pad=9),
        # a training step's gradient over a long batch
        _norm("norm_grad_t16384", "backward", 16384, 7168, "bf16", "channel"),
        # the same for a short odd batch in fp16 with a gate for every element
        _norm("norm_grad_t77", "backward", 77, 2048, "fp16", "full"),
        # the counts of one decode batch
        _balance("balance_t16", "forward", 16, 256, 8),
        # a prefill batch as one sequence
        _balance("balance_t16384", "forward", 16384, 256, 8),
        # a training batch of ragged sequences with padded tokens: the gradient for the router
        _balance("balance_grad_ragged", "backward", 8191, 256, 8, "bf16", seqs=61, mask=True),
        # many short sequences and a softmax router
        _balance("balance_short_seqs", "forward", 4099, 160, 6, "fp32", seqs=700, scoring="softmax"),
        # one token through the first product of the experts that it selected on this shard
        _matvec("matvec_up_t1", 1, 4096, 7168, 128, E=32, k=8, pool=32),
        # the second product of a decode batch, every row its own expert: most of the shard's experts are read
        _matvec("matvec_down_t16", 16, 7168, 2048, 128, E=32, k=8, pool=64, per_pair=True),
        # a dense projection of a few sequences, odd row count, small groups with zero points
        _matvec("matvec_dense_t5", 5, 4001, 7168, 64, "fp16", zero=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "balance", "matvec"))
    if kind == "norm":
        quantize = rng.random() < 0.3
        H = rng.choice((7168, BLOCK * rng.randint(1, 56) if quantize else rng.randint(64, LARGEST_H)))
        join = rng.random() < 0.8
        way = "backward" if not quantize and rng.random() < 0.5 else "forward"
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        most = LARGEST_T if dtype != "fp32" else LARGEST_T // 2
        case = _norm("", way, _log_uniform(rng, 1, most), H, dtype,
                     rng.choice(("none", "channel", "token", "full")) if join else "none", join,
                     rng.random() < 0.7 if join else False, quantize, rng.choice((0, 0, 8, 5)) if not quantize else 0)
    elif kind == "balance":
        E = rng.choice((256, rng.randint(24, LARGEST_E)))
        T = _log_uniform(rng, 1, LARGEST_T // 2)
        # a mean over a long batch has gradients below fp16's range, which a user scales or holds in another type
        way = rng.choice(("forward", "backward"))
        case = _balance("", way, T, E, min(E, rng.choice((1, 2, 6, 8))),
                        rng.choice(("fp32", "fp32", "bf16", "fp16" if way == "forward" else "bf16")),
                        rng.choice((0, _log_uniform(rng, 1, max(1, T // 2)))), rng.random() < 0.4,
                        rng.choice(("sigmoid", "softmax")))
    else:
        G = rng.choice((32, 64, 128))
        N, K = rng.randint(16, 7168), G * rng.randint(1, 7168 // G)
        if rng.random() < 0.6:
            k = rng.choice((1, 2, 8))
            case = _matvec("", rng.randint(1, 16), N, K, G, rng.choice(("bf16", "fp16")), rng.random() < 0.4, 16, k,
                           rng.choice((16, 32, 64)), rng.random() < 0.5)
        else:
            case = _matvec("", rng.randint(1, 16), N, K, G, rng.choice(("bf16", "fp16")), rng.random() < 0.4)
    del case["name"]
    return case


# ---------------------------------------------------------------------------- inputs


def _rows(g, T, H, dtype, pad, scale):
    """[T, H] values in rows of H + pad; a few channels carry most of the energy, as in a residual stream."""
    v = torch.randn((T, H + pad), generator=g, device=g.device) * scale
    v[:, ::211] *= 8.0
    return v.to(dtype)[:, :H]


def _prepare_norm(case, g):
    T, H, t = case["T"], case["H"], TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device=g.device)  # noqa: E731
    s = {"x": _rows(g, T, H, t, case["pad"], 1.5), "pre_weight": (1 + 0.1 * randn(H)).to(t),
         "y": None, "post_weight": None, "gate": None}
    if case["join"]:
        s["y"] = _rows(g, T, H, t, case["pad"], 0.4)
        if case["post"]:
            s["post_weight"] = (0.5 + 0.1 * randn(H)).to(t)
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        if shape is not None:
            s["gate"] = torch.sigmoid(randn(*shape)).to(t)
    if case["way"] == "backward":
        s["grad_h"] = _rows(g, T, H, t, case["pad"], 0.1)
        s["grad_stream"] = _rows(g, T, H, t, case["pad"], 0.1) if case["join"] else None
        s["rstd"] = _norm_parts(s, torch.float32)["rstd"]
    return s


def _bounds(case, g):
    """Sequence borders [seqs + 1] of a packed batch; the last rows may belong to no sequence, sequences may be empty."""
    T, n = case["T"], case["seqs"]
    cuts = torch.randint(0, T + 1, (n - 1,), generator=g, device=g.device).sort().values
    ends = torch.tensor([T - T // 50], device=g.device)
    return torch.cat([torch.zeros_like(ends), cuts.clamp(max=T - T // 50), ends]).to(torch.int32)


def _prepare_balance(case, g):
    T, E, K = case["T"], case["E"], case["K"]
    logits = torch.randn((T, E), generator=g, device=g.device) + 0.5 * torch.randn(E, generator=g, device=g.device)
    logits = logits.to(TYPES[case["dtype"]])
    s = {"logits": logits, "topk_idx": logits.float().topk(K, dim=1).indices.to(torch.int32), "cu": None, "mask": None}
    if case["seqs"]:
        s["cu"] = _bounds(case, g)
    if case["mask"]:
        s["mask"] = torch.rand(T, generator=g, device=g.device) < 0.9
    if case["way"] == "backward":
        seq, valid, S = _owners(s)
        chosen = torch.zeros((T, E), device=g.device).scatter_add_(1, s["topk_idx"].long(), torch.ones((T, K), device=g.device))
        s["counts"] = torch.zeros((S, E), device=g.device).index_add_(0, seq, chosen * valid[:, None]).to(torch.int32)
        s["tokens"] = torch.zeros(S, device=g.device).index_add_(0, seq, valid.float()).to(torch.int32)
        s["grad_loss"] = torch.rand(S, generator=g, device=g.device) + 0.5
    return s


def _experts(case, g):
    """[T, k] different experts of a pool, of which this shard holds the first E."""
    order = torch.rand((case["T"], case["pool"]), generator=g, device=g.device).argsort(1)[:, :case["k"]]
    return order.to(torch.int32)


def _prepare_matvec(case, g):
    T, N, K, G, E = (case[k] for k in ("T", "N", "K", "G", "E"))
    t, device = TYPES[case["dtype"]], g.device
    shape = (E, N) if E else (N,)
    s = {"experts": _experts(case, g).contiguous() if E else None}
    rows = T * case["k"] if case["per_pair"] and E else T
    if case["per_pair"] and E:
        s["experts"] = s["experts"].reshape(-1)
    s["x"] = torch.randn((rows, K), generator=g, device=device).to(t)
    s["qweight"] = torch.randint(0, 256, shape + (K // 2,), generator=g, device=device, dtype=torch.uint8)
    s["scale"] = ((torch.rand(shape + (K // G,), generator=g, device=device) + 0.5) * 0.01).to(t)
    s["zero"] = None
    if case["zero"]:
        s["zero"] = torch.randint(0, 16, shape + (K // G,), generator=g, device=device, dtype=torch.uint8)
    return s


def prepare(case, seed):
    g = torch.Generator(device=torch.device("cuda", torch.cuda.current_device()))
    g.manual_seed(seed)
    s = {"norm": _prepare_norm, "balance": _prepare_balance, "matvec": _prepare_matvec}[case["op"]](case, g)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------- plain forms


def _norm_parts(s, wide):
    """Everything the forward computes, unrounded."""
    x = s["x"].to(wide)
    r1, yhat, n = torch.zeros_like(x[:, :1]), None, None
    if s["y"] is not None:
        y = s["y"].to(wide)
        yhat = n = y
        if s["post_weight"] is not None:
            r1 = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
            yhat = y * r1
            n = yhat * s["post_weight"].to(wide)
        x = RESIDUAL_SCALE * x + (n if s["gate"] is None else s["gate"].to(wide) * n)
    r2 = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    return {"stream": x, "shat": x * r2, "yhat": yhat, "n": n, "rstd": torch.cat([r1, r2], 1)}


def _plain_norm(s):
    t, p = s["x"].dtype, _norm_parts(s, torch.float32)
    h = p["shat"] * s["pre_weight"].float()
    out = {"stream": p["stream"].to(t) if s["y"] is not None else None, "rstd": p["rstd"]}
    if s["case"]["quantize"]:
        blocks = h.unflatten(1, (-1, BLOCK))
        scale = blocks.abs().amax(2).clamp(min=1e-10) / 448.0
        q = (blocks / scale[:, :, None]).clamp(-448.0, 448.0).flatten(1).to(torch.float8_e4m3fn)
        return {**out, "h": q, "scale": scale.t().contiguous()}
    return {**out, "h": h.to(t)}


def _plain_norm_backward(s):
    t, p, r1, r2 = s["x"].dtype, _norm_parts(s, torch.float32), s["rstd"][:, :1], s["rstd"][:, 1:]
    gh = s["grad_h"].float()
    dh = gh * s["pre_weight"].float()
    d = r2 * (dh - p["shat"] * (dh * p["shat"]).mean(1, keepdim=True))
    out = {"pre_weight": (gh * p["shat"]).sum(0).to(t)}
    if s["y"] is None:
        return {**out, "x": d.to(t)}
    d = d + s["grad_stream"].float()
    out["x"] = (RESIDUAL_SCALE * d).to(t)
    dn = d
    if s["gate"] is not None:
        dg = d * p["n"]
        kind = s["case"]["gate"]
        out["gate"] = (dg.sum(0) if kind == "channel" else dg.sum(1, keepdim=True) if kind == "token" else dg).to(t)
        dn = d * s["gate"].float()
    if s["post_weight"] is None:
        return {**out, "y": dn.to(t)}
    out["post_weight"] = (dn * p["yhat"]).sum(0).to(t)
    dyhat = dn * s["post_weight"].float()
    out["y"] = (r1 * (dyhat - p["yhat"] * (dyhat * p["yhat"]).mean(1, keepdim=True))).to(t)
    return out


def _owners(s):
    """(sequence of every token, whether it counts, number of sequences)."""
    T = s["logits"].shape[0]
    seq = torch.zeros(T, dtype=torch.long, device=s["logits"].device)
    valid = torch.ones(T, dtype=torch.bool, device=seq.device) if s["mask"] is None else s["mask"]
    if s["cu"] is None:
        return seq, valid, 1
    S = s["cu"].numel() - 1
    seq = torch.searchsorted(s["cu"].long(), torch.arange(T, device=seq.device), right=True) - 1
    return seq.clamp(max=S - 1), valid & (seq < S), S


def _probabilities(s):
    """(p, its derivative's diagonal factor s (1 - s) / Z or p) in 32 bits."""
    z = s["logits"].float()
    if s["case"]["scoring"] == "softmax":
        p = torch.exp(z - z.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        return p, p
    e = 1.0 / (1.0 + torch.exp(-z))
    p = e / e.sum(1, keepdim=True)
    return p, p * (1.0 - e)


def _plain_balance(s):
    c = s["case"]
    seq, valid, S = _owners(s)
    p, _ = _probabilities(s)
    keep = valid[:, None]
    device = p.device
    chosen = torch.zeros_like(p).scatter_add_(1, s["topk_idx"].long(), torch.ones(s["topk_idx"].shape, device=device))
    counts = torch.zeros((S, c["E"]), device=device).index_add_(0, seq, torch.where(keep, chosen, 0.0))
    sums = torch.zeros((S, c["E"]), device=device).index_add_(0, seq, torch.where(keep, p, 0.0))
    tokens = torch.zeros(S, device=device).index_add_(0, seq, valid.float())
    n = tokens.clamp(min=1.0)
    loss = ALPHA * c["E"] / c["K"] * (counts / n[:, None] * (sums / n[:, None])).sum(1)
    return {"loss": loss, "counts": counts.to(torch.int32), "tokens": tokens.to(torch.int32)}


def _plain_balance_backward(s):
    c = s["case"]
    seq, valid, _ = _owners(s)
    p, slope = _probabilities(s)
    n = s["tokens"].float().clamp(min=1.0)
    f = (s["counts"].float() * (ALPHA * c["E"] / c["K"] * s["grad_loss"] / (n * n))[:, None])[seq]
    grad = slope * (f - (f * p).sum(1, keepdim=True))
    return {"logits": torch.where(valid[:, None], grad, 0.0).to(s["logits"].dtype)}


def _plain_matvec(s):
    c, q = s["case"], s["qweight"]
    w = torch.stack([q & 15, q >> 4], -1).flatten(-2).float().unflatten(-1, (-1, c["G"]))
    w = w - (8.0 if s["zero"] is None else s["zero"].float()[..., None])
    w = (w * s["scale"].float()[..., None]).flatten(-2)
    x = s["x"].float()
    if s["experts"] is None:
        return {"out": (x @ w.t()).to(s["x"].dtype)}
    every = (x @ w.flatten(0, 1).t()).unflatten(1, (c["E"], c["N"]))
    e = s["experts"].long().view(x.shape[0], -1)
    out = every.gather(1, e.clamp(max=c["E"] - 1)[:, :, None].expand(-1, -1, c["N"]))
    out = torch.where((e < c["E"])[:, :, None], out, 0.0)
    return {"out": out.view(tuple(s["experts"].shape) + (c["N"],)).to(s["x"].dtype)}


# ---------------------------------------------------------------------------- the package's calls


def _op():
    from __graft_entry__ import load_package
    return load_package().op


def _own_norm(s):
    stream, h, rstd = _op().block_norm(s["x"], s["pre_weight"], y=s["y"], post_weight=s["post_weight"], gate=s["gate"],
                                       residual_scale=RESIDUAL_SCALE, eps=EPS, quantize=s["case"]["quantize"])
    out = {"stream": stream if s["y"] is not None else None, "rstd": rstd}
    return {**out, "h": h[0], "scale": h[1]} if s["case"]["quantize"] else {**out, "h": h}


def _own_norm_backward(s):
    g = _op().block_norm_backward(s["x"], s["pre_weight"], s["rstd"], s["grad_h"], s["grad_stream"], y=s["y"],
                                  post_weight=s["post_weight"], gate=s["gate"], residual_scale=RESIDUAL_SCALE)
    return {k: v for k, v in g.items() if v is not None}


def _own_balance(s):
    c = s["case"]
    loss, counts, tokens = _op().balance_loss(s["logits"], s["topk_idx"], ALPHA, cu_seqlens=s["cu"],
                                              token_mask=s["mask"], scoring=c["scoring"])
    return {"loss": loss, "counts": counts, "tokens": tokens}


def _own_balance_backward(s):
    c = s["case"]
    return {"logits": _op().balance_loss_backward(s["grad_loss"], s["logits"], s["counts"], s["tokens"], c["K"], ALPHA,
                                                  cu_seqlens=s["cu"], token_mask=s["mask"], scoring=c["scoring"])}


def _own_matvec(s):
    return {"out": _op().matvec_w4(s["x"], s["qweight"], s["scale"], zero=s["zero"], experts=s["experts"])}


PLAIN = {"norm forward": _plain_norm, "norm backward": _plain_norm_backward, "balance forward": _plain_balance,
         "balance backward": _plain_balance_backward, "matvec": _plain_matvec}
OWN = {"norm forward": _own_norm, "norm backward": _own_norm_backward, "balance forward": _own_balance,
       "balance backward": _own_balance_backward, "matvec": _own_matvec}


def run(state):
    c = state["case"]
    kind = c["op"] if c["op"] == "matvec" else c["op"] + " " + c["way"]
    if own:
        return OWN[kind](state)
    return PLAIN[kind](state)


# ---------------------------------------------------------------------------- work and exact results


def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]]
        columns = H * (2 if case["post"] else 1)
        if case["way"] == "forward":
            rows = b * T * H * (3 if case["join"] else 1)      # x, y in; stream out
            rows += T * H + T * H // BLOCK * 4 if case["quantize"] else b * T * H
            return {"bytes": rows + b * (gate + columns) + 8 * T, "flops": T * H * (9 if case["join"] else 4)}
        rows = b * T * H * (6 if case["join"] else 3)          # x, y, two gradients in; two out
        return {"bytes": rows + 2 * b * (gate + columns) + 8 * T, "flops": T * H * (26 if case["join"] else 9)}
    if case["op"] == "balance":
        T, E = case["T"], case["E"]
        S = max(1, case["seqs"])
        side = T * (1 if case["mask"] else 0) + 4 * S + S * (4 * E + 8)
        if case["way"] == "forward":
            return {"bytes": T * (b * E + 4 * case["K"]) + side, "flops": 5 * T * E}
        return {"bytes": 2 * b * T * E + side, "flops": 10 * T * E}
    T, N, K, G, E = (case[k] for k in ("T", "N", "K", "G", "E"))
    rows, read, pairs = T, 1.0, T
    if E:
        # experts that at least one of the batch's pairs selects, and the pairs this shard has: means over eight batches
        read = pairs = 0.0
        for k in range(8):
            g = torch.Generator()
            g.manual_seed(k)
            e = _experts(case, g)
            read += e[e < E].unique().numel() / 8
            pairs += int((e < E).sum()) / 8
        rows = T * case["k"] if case["per_pair"] else T
    weights = N * K / 2 + N * (K // G) * (b + (1 if case["zero"] else 0))
    outs = T * case["k"] if E else T
    return {"bytes": read * weights + b * (rows * K + outs * N), "flops": 2 * pairs * N * K}


def _exact_norm(case, s):
    d = torch.float64
    x, w = s["x"].to(d), s["pre_weight"].to(d)
    H = x.shape[1]
    v, post, gate = x, None, 1.0
    r1 = torch.zeros(x.shape[0], dtype=d, device=x.device)
    if case["join"]:
        y = s["y"].to(d)
        gate = 1.0 if s["gate"] is None else s["gate"].to(d)
        if case["post"]:
            post = s["post_weight"].to(d)
            r1 = 1.0 / (y.square().sum(1) / H + EPS).sqrt()
            normed = y * r1[:, None] * post
        else:
            normed = y
        v = x * RESIDUAL_SCALE + normed * gate
    r2 = 1.0 / (v.square().sum(1) / H + EPS).sqrt()
    if case["way"] == "forward":
        h = v * r2[:, None] * w
        out = {"stream": v if case["join"] else None, "rstd": torch.stack([r1, r2], 1), "h": h}
        if case["quantize"]:
            top = h.abs().view(h.shape[0], H // BLOCK, BLOCK).max(2).values / 448.0
            out["scale"] = top.t()
            out["h"] = h / top.repeat_interleave(BLOCK, 1)
        return out
    # the gradients from the quotient v_i / |v|: (w g)_i / r - v_i (v . (w g)) / (H r^3), r = 1 / rstd
    a, g = s["rstd"].to(d), s["grad_h"].to(d)
    a1, a2 = a[:, 0:1], a[:, 1:2]
    wg = g * w
    D = a2 * wg - v * (a2 ** 3 / H) * (v * wg).sum(1, keepdim=True)
    out = {"pre_weight": (g * v * a2).sum(0)}
    if not case["join"]:
        return {**out, "x": D}
    D = D + s["grad_stream"].to(d)
    out["x"] = D * RESIDUAL_SCALE
    if case["gate"] != "none":
        scaled = D * (y * a1 * post if case["post"] else y)
        out["gate"] = {"channel": lambda: scaled.sum(0), "token": lambda: scaled.sum(1)[:, None], "full": lambda: scaled}[case["gate"]]()
    inner = D * gate
    if not case["post"]:
        return {**out, "y": inner}
    out["post_weight"] = (inner * y * a1).sum(0)
    u = inner * post
    out["y"] = a1 * u - y * (a1 ** 3 / H) * (y * u).sum(1, keepdim=True)
    return out


def _exact_balance(case, s):
    d = torch.float64
    T, E, K = case["T"], case["E"], case["K"]
    z = s["logits"].to(d)
    score = torch.sigmoid(z) if case["scoring"] == "sigmoid" else torch.softmax(z, 1)
    p = score / score.sum(1, keepdim=True)
    ends = [0, T] if s["cu"] is None else s["cu"].tolist()
    live = torch.ones(T, dtype=d, device=z.device) if s["mask"] is None else s["mask"].to(d)
    if case["way"] == "forward":
        loss = []
        for lo, hi in zip(ends[:-1], ends[1:]):
            n = float(live[lo:hi].sum())
            ids = s["topk_idx"][lo:hi].long()[live[lo:hi] > 0].flatten()
            f = torch.bincount(ids, minlength=E).to(d) * E / (K * max(n, 1.0))
            loss.append(ALPHA * (f * (p[lo:hi] * live[lo:hi, None]).sum(0) / max(n, 1.0)).sum())
        return {"loss": torch.stack(loss), "counts": None, "tokens": None}
    grad = torch.zeros_like(z)
    for i, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        n = max(1, int(s["tokens"][i]))
        f = s["counts"][i].to(d) * (E / (K * n))
        c = float(s["grad_loss"][i]) * ALPHA / n
        part = (f - (p[lo:hi] * f).sum(1, keepdim=True)) * p[lo:hi]
        grad[lo:hi] = c * part * (1.0 - score[lo:hi] if case["scoring"] == "sigmoid" else 1.0) * live[lo:hi, None]
    return {"logits": grad}


def _exact_matvec(case, s):
    d = torch.float64
    K, G = case["K"], case["G"]
    x, group = s["x"].to(d), torch.arange(K, device=s["x"].device) // G

    def matrix(q, scale, zero):
        w = torch.empty((q.shape[0], K), dtype=d, device=q.device)
        w[:, 0::2], w[:, 1::2] = (q % 16).to(d), (q // 16).to(d)
        return (w - (zero.to(d)[:, group] if zero is not None else 8.0)) * scale.to(d)[:, group]

    if s["experts"] is None:
        return {"out": x @ matrix(s["qweight"], s["scale"], s["zero"]).t()}
    flat = s["experts"].flatten().long()
    row = torch.arange(flat.numel(), device=flat.device) // (flat.numel() // x.shape[0])
    out = torch.zeros((flat.numel(), case["N"]), dtype=d, device=x.device)
    for e in sorted(set(flat.tolist())):
        if e < case["E"]:
            at = flat == e
            out[at] = x[row[at]] @ matrix(s["qweight"][e], s["scale"][e], None if s["zero"] is None else s["zero"][e]).t()
    return {"out": out.view(tuple(s["experts"].shape) + (case["N"],))}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "balance": _exact_balance, "matvec": _exact_matvec}[case["op"]](case, s)
