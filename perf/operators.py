"""What is measured of the attention operators: cases, their inputs, their plain forms and their exact results.

``run`` computes a case in its plain form, or, with ``own`` set, through this package's entry points
(``eeggan_amd.ops.attention``, ``ops.relative_bias``, ``optim.Adam(max_grad_norm=...)``)."""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------------ the cases
def _attention(name, dtype, B, heads, kv_heads, dk, dv, tq, tk, train, bias=0, distance=0, step=1, offset=0, mask=False):
    """``bias``: number of position buckets (0: none); ``mask``: ragged key lengths, one sample without any key."""
    case = dict(op="attention", dtype=dtype, B=B, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, tq=tq, tk=tk, train=train,
                bias=bias, distance=distance, step=step, offset=offset, mask=mask)
    return dict(case, name=name) if name else case


def _scores(name, B, heads, tq, tk, bias, distance, step, offset):
    case = dict(op="relative_bias", B=B, heads=heads, tq=tq, tk=tk, bias=bias, distance=distance, step=step, offset=offset)
    return dict(case, name=name) if name else case


def _clip(name, sizes, clipped):
    """``sizes``: the tensors' element counts, as text (a case holds plain values)."""
    case = dict(op="adam_clip", sizes=",".join(str(s) for s in sizes), clipped=clipped)
    return dict(case, name=name) if name else case


# The critic's parameter tensors at full depth (conv weights and biases of eight stages, the full-length layer, the scores).
_CRITIC = [64 * 5, 64] * 8 + [64 * 64 * 3, 64] * 9 + [128 * 64 * 3, 128, 128 * 128 * 3, 128, 256 * 128 * 3, 256] + \
    [256 * 256 * 3, 256] * 2 + [256 * 257 * 3, 256, 256 * 256 * 32, 256, 256, 1]
# A network of wide layers: 24 blocks of a wide matrix, a square one and their biases.
_WIDE = [1024 * 2048, 2048, 1024 * 1024, 1023] * 24


def listed():
    return [
        # the attention layer of a 64-channel stage of 1280 steps in training (keys pooled by four), 32 signals
        _attention("layer_train_64ch", "float32", 32, 1, 1, 8, 32, 1280, 320, True),
        # the attention layer of a 256-channel stage of 128 steps in training: short, many signals
        _attention("layer_train_256ch", "float32", 128, 1, 1, 32, 128, 128, 32, True),
        # signals made for evaluation in one large batch by a network with a 64-channel attention layer
        _attention("layer_generate_512", "float32", 512, 1, 1, 8, 32, 1280, 320, False),
        # several heads over long windows in training
        _attention("heads_train_long", "bfloat16", 8, 8, 8, 64, 64, 2048, 2048, True),
        # one new step asked of a long recording, key and value heads shared by four query heads
        _attention("one_step_long", "bfloat16", 8, 16, 4, 128, 128, 1, 16384, False),
        # ragged recordings in one batch, learned positions, shared key heads, in training
        _attention("ragged_positions_bf16", "bfloat16", 4, 6, 2, 64, 64, 1537, 1537, True, 32, 128, 1, 0, True),
        # odd sizes everywhere, pooled keys, learned positions, single precision, in training
        _attention("odd_positions_f32", "float32", 5, 4, 4, 24, 40, 1333, 333, True, 32, 256, 4, 2, True),
        # learned positions on stored scores (the penalty's path): the smallest stage
        _scores("scores_small", 4, 1, 128, 32, 16, 64, 4, 2),
        # ... the 64-channel stage of 1280 steps
        _scores("scores_layer", 32, 1, 1280, 320, 32, 256, 4, 2),
        # ... four heads over the full window
        _scores("scores_long", 16, 4, 1920, 1920, 32, 128, 1, 0),
        # the critic's optimizer step with a bounded gradient
        _clip("critic_step", _CRITIC, True),
        # the same step for a network of wide layers
        _clip("wide_step", _WIDE, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layer", "layer", "heads", "heads", "positions", "positions", "step", "scores", "clip"])
    if kind == "layer":  # the networks' attention layer: channels / 8 and / 2, keys pooled by four
        c = rng.choice([64, 64, 128, 256])
        tk = _log(rng, 8, 480)
        B = max(1, min(_log(rng, 4, 512), 210_000_000 // (4 * tk * tk)))
        return _attention(None, "float32", B, 1, 1, c // 8, c // 2, 4 * tk, tk, rng.random() < 0.7)
    if kind in ("heads", "positions"):
        kv = rng.choice([1, 2, 3, 4])
        heads = kv * rng.choice([1, 1, 2, 3])
        tq = _log(rng, 1, 2300)
        tk = tq if rng.random() < 0.5 else _log(rng, 1, 2300)
        B = max(1, min(_log(rng, 1, 32), 100_000_000 // (heads * tq * tk)))
        dk = rng.randint(4, 128) if rng.random() < 0.5 else rng.choice([16, 32, 64, 128])
        dv = dk if rng.random() < 0.6 else rng.randint(4, 128)
        dtype = rng.choice(["float32", "bfloat16"])
        if kind == "heads":
            return _attention(None, dtype, B, heads, kv, dk, dv, tq, tk, rng.random() < 0.7, mask=rng.random() < 0.3)
        return _attention(None, dtype, B, heads, kv, dk, dv, tq, tk, rng.random() < 0.7, rng.choice([8, 16, 32]),
                          rng.choice([64, 128, 200, 256]), rng.choice([1, 1, 2, 4]), rng.randint(-40, 3),
                          rng.random() < 0.5)
    if kind == "step":
        kv = rng.choice([1, 2, 4])
        d = rng.choice([32, 64, 128])
        tk = _log(rng, 64, 32768)
        B = max(1, min(_log(rng, 1, 32), 500_000 // (kv * tk)))
        return _attention(None, rng.choice(["float32", "bfloat16", "bfloat16"]), B, kv * rng.choice([1, 2, 4]), kv, d, d,
                          rng.choice([1, 1, 1, 2, 5]), tk, False, mask=rng.random() < 0.5)
    if kind == "scores":
        heads = rng.choice([1, 2, 4])
        tk, step = _log(rng, 16, 1900), rng.choice([1, 2, 4])
        tq = min(1900, tk * step + rng.randint(0, 9))
        B = max(1, min(_log(rng, 1, 64), 200_000_000 // (heads * tq * tk)))
        return _scores(None, B, heads, tq, tk, rng.choice([8, 16, 32]), rng.choice([64, 128, 200, 256]), step,
                       rng.randint(-5, 5))
    n = _log(rng, 1, 180)
    return _clip(None, [_log(rng, 1, 600_000) for _ in range(n)], rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------ their inputs
def _edges(buckets, distance):
    """Smallest distance of every bucket of one side: the first half of the buckets holds one distance each, the others
    grow geometrically up to ``distance``; whole-number arithmetic, no rounding at the borders."""
    exact = buckets // 2
    edges = list(range(exact))
    for i in range(buckets - exact):
        d = exact
        while d ** (buckets - exact) < exact ** (buckets - exact - i) * distance ** i:
            d += 1
        edges.append(d)
    return edges


def _views(sizes):
    """One buffer and a tensor of every size in it, each at a multiple of 64 elements."""
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += (n + 63) // 64 * 64
    flat = torch.zeros(end, device=DEV)
    return flat, [flat[a:a + n] for a, n in zip(starts, sizes)]


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1_000_003 * seed + 17)
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=gen)  # noqa: E731
    s = {"case": case}
    if case["op"] == "adam_clip":
        sizes = [int(n) for n in case["sizes"].split(",")]
        for name in ("p", "m", "v"):
            s[name + "_all"], s[name] = _views(sizes)
        s["g"] = [randn(n) * (0.01 * (1 + i % 5)) for i, n in enumerate(sizes)]
        for p, m, v in zip(s["p"], s["m"], s["v"]):
            p.copy_(randn(p.numel()) * 0.05)
            m.copy_(randn(p.numel()) * 0.01)
            v.copy_(randn(p.numel()).square() * 1e-4)
        s["max_norm"] = 0.5 * math.sqrt(sum(n * (0.01 * (1 + i % 5)) ** 2 for i, n in enumerate(sizes)))
        if not case["clipped"]:
            s["max_norm"] *= 8.0
        s["lr"], s["betas"], s["eps"], s["steps"] = 1e-3, (0.5, 0.99), 1e-8, 7
        return s
    B, heads, tq, tk = case["B"], case["heads"], case["tq"], case["tk"]
    if case["op"] == "relative_bias":
        s["scores"] = randn(B * heads, tk, tq)
        s["g"] = randn(B * heads, tk, tq) / math.sqrt(tk)
        s["table"] = randn(case["bias"], heads)
    else:
        dt = getattr(torch, case["dtype"])
        kv, dk, dv = case["kv_heads"], case["dk"], case["dv"]
        s["q"] = randn(B, heads * dk, tq).to(dt)
        s["k"] = randn(B, kv * dk, tk).to(dt)
        s["v"] = randn(B, kv * dv, tk).to(dt)
        s["g"] = randn(B, heads * dv, tq).to(dt) if case["train"] else None
        s["scale"] = 1.0 / math.sqrt(dk)
        s["table"] = randn(case["bias"], heads).to(dt) if case["bias"] else None
        s["mask"] = None
        if case["mask"]:  # ragged lengths; of several samples one has no keys at all, others lack some in the middle
            lengths = torch.randint(1, tk + 1, (B, 1), device=DEV, generator=gen)
            mask = torch.arange(tk, device=DEV)[None, :] < lengths
            mask &= torch.rand(B, tk, device=DEV, generator=gen) < 0.95
            if B > 1:
                mask[B // 2] = False
            s["mask"] = mask
    if case["bias"]:
        edges = _edges(case["bias"] // 2, case["distance"])
        s["edges"] = torch.tensor(edges, device=DEV)
        s["position"] = (case["step"], case["offset"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        if case["op"] == "adam_clip":
            from eeggan_amd import optim
            s["params"] = [torch.nn.Parameter(p) for p in s["p"]]
            opt = optim.Adam(s["params"], lr=s["lr"], betas=s["betas"], eps=s["eps"], max_grad_norm=s["max_norm"])
            for p, g, m, v in zip(s["params"], s["g"], s["m"], s["v"]):
                p.grad = g
                opt.state[p] = {"step": torch.full((), float(s["steps"]), device=DEV), "exp_avg": m, "exp_avg_sq": v}
            s["opt"] = opt
            return s
        from eeggan_amd import ops
        s["buckets"] = None
        if case["bias"]:
            s["buckets"] = ops.RelativeBuckets(case["bias"], case["distance"], step=case["step"], offset=case["offset"])
        if case["op"] == "relative_bias" or case["train"]:
            for name in ("q", "k", "v", "scores", "table"):
                if s.get(name) is not None:
                    s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "adam_clip":
        return _adam_own(state) if own else _adam_plain(state)
    if op == "relative_bias":
        return _scores_own(state) if own else _scores_plain(state)
    return _attention_own(state) if own else _attention_plain(state)


def _attention_own(s):
    from eeggan_amd import ops
    c = s["case"]
    kw = dict(heads=c["heads"], kv_heads=c["kv_heads"], scale=s["scale"], mask=s["mask"], bias=s["table"],
              buckets=s["buckets"])
    if not c["train"]:
        with torch.no_grad():
            return [ops.attention(s["q"], s["k"], s["v"], **kw)]
    out = ops.attention(s["q"], s["k"], s["v"], **kw)
    leaves = [s["q"], s["k"], s["v"]] + ([s["table"]] if c["bias"] else [])
    return [out.detach()] + list(torch.autograd.grad(out, leaves, s["g"]))


def _scores_own(s):
    from eeggan_amd import ops
    out = ops.relative_bias(s["scores"], s["table"], s["buckets"], heads=s["case"]["heads"])
    g_scores, g_table = torch.autograd.grad(out, [s["scores"], s["table"]], s["g"])
    return [out.detach(), g_scores, g_table]


def _adam_own(s):
    s["opt"].step()
    return [s["opt"].grad_norm, s["p_all"], s["m_all"], s["v_all"]]


def _bucket(case, edges):
    """[Tk, Tq] bucket of every (key, query) pair: keys behind the query take the first half, keys ahead the second."""
    rel = (torch.arange(case["tk"], device=DEV) * case["step"] + case["offset"])[:, None] \
        - torch.arange(case["tq"], device=DEV)[None, :]
    side = (rel.abs()[..., None] >= edges).sum(-1) - 1 if rel.numel() < 1_000_000 \
        else sum((rel.abs() >= e).to(torch.int64) for e in edges) - 1
    return side + (rel > 0) * (case["bias"] // 2)


def _bucket_sums(x, bucket, n):
    """x [H, Tk, Tq] -> [n, H]: sums over the pairs of every bucket."""
    flat, where = x.reshape(x.shape[0], -1), bucket.reshape(-1)
    return torch.stack([(flat * (where == j)).sum(1, dtype=torch.float64) for j in range(n)])


def _attention_plain(s):
    c = s["case"]
    B, H, KV, dk, dv, tq, tk = (c[n] for n in ("B", "heads", "kv_heads", "dk", "dv", "tq", "tk"))
    G, dt = H // KV, s["q"].dtype
    # columns of one key head: its G query heads, one after the other
    cols = lambda x, d: x.float().view(B, KV, G, d, tq).transpose(2, 3).reshape(B * KV, d, G * tq)  # noqa: E731
    back = lambda x, d: x.view(B, KV, d, G, tq).transpose(2, 3).reshape(B, H * d, tq).to(dt)  # noqa: E731
    q, k, v = cols(s["q"], dk), s["k"].float().view(B * KV, dk, tk), s["v"].float().view(B * KV, dv, tk)
    keep = None
    if s["mask"] is not None:
        keep = s["mask"][:, None, :, None].expand(B, KV, tk, 1).reshape(B * KV, tk, 1)
    p = torch.matmul(k.transpose(1, 2), q) * s["scale"]
    if c["bias"]:
        bucket = _bucket(c, s["edges"])
        bias = s["table"].float().t()[:, bucket]  # [H, Tk, Tq]
        p += bias.view(1, KV, G, tk, tq).transpose(2, 3).expand(B, KV, tk, G, tq).reshape(B * KV, tk, G * tq)
    if keep is not None:
        p.masked_fill_(~keep, -1e30)
    p -= p.amax(1, keepdim=True)
    p.exp_()
    p /= p.sum(1, keepdim=True)
    if keep is not None:
        p *= keep
    o = torch.matmul(v, p)
    if not c["train"]:
        return [back(o, dv)]
    g = cols(s["g"], dv)
    gv = torch.matmul(g, p.transpose(1, 2))
    ds = torch.matmul(v.transpose(1, 2), g)
    ds -= (o * g).sum(1, keepdim=True)
    ds *= p
    gq = torch.matmul(k, ds) * s["scale"]
    gk = torch.matmul(q, ds.transpose(1, 2)) * s["scale"]
    outs = [back(o, dv), back(gq, dk), gk.view(B, KV * dk, tk).to(dt), gv.view(B, KV * dv, tk).to(dt)]
    if c["bias"]:
        sums = ds.view(B, KV, tk, G, tq).sum(0).transpose(1, 2).reshape(H, tk, tq)
        outs.append(_bucket_sums(sums, bucket, c["bias"]).to(dt))
    return outs


def _scores_plain(s):
    c = s["case"]
    bucket = _bucket(c, s["edges"])
    bias = s["table"].t()[:, bucket]
    out = (s["scores"].view(c["B"], c["heads"], c["tk"], c["tq"]) + bias).view(s["scores"].shape)
    sums = s["g"].view(c["B"], c["heads"], c["tk"], c["tq"]).sum(0)
    return [out, s["g"], _bucket_sums(sums, bucket, c["bias"]).float()]


def _adam_plain(s):
    norm = torch.stack([g.double().square().sum() for g in s["g"]]).sum().sqrt()
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    s["steps"] += 1
    b1, b2 = s["betas"]
    r1, r2 = 1.0 - b1 ** s["steps"], math.sqrt(1.0 - b2 ** s["steps"])
    for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        g = g * c
        m.mul_(b1).add_(g * (1.0 - b1))
        v.mul_(b2).add_(g * g * (1.0 - b2))
        p.sub_(m * (s["lr"] / r1) / (v.sqrt() / r2 + s["eps"]))
    return [norm.float(), s["p_all"], s["m_all"], s["v_all"]]


# ------------------------------------------------------------------------------------------------------ work, exact results
def work(case):
    if case["op"] == "adam_clip":
        n = sum(int(x) for x in case["sizes"].split(","))
        return {"bytes": 28 * n, "flops": 14 * n}
    B, H, tq, tk = case["B"], case["heads"], case["tq"], case["tk"]
    n = B * H * tq * tk
    if case["op"] == "relative_bias":  # scores in, scores out; their gradient in (it is the scores' gradient as it is)
        return {"bytes": 3 * 4 * n + 8 * case["bias"] * H, "flops": 2 * n}
    size = 4 if case["dtype"] == "float32" else 2
    kv, dk, dv = case["kv_heads"], case["dk"], case["dv"]
    qs, os_, ks, vs = B * H * dk * tq, B * H * dv * tq, B * kv * dk * tk, B * kv * dv * tk
    if not case["train"]:
        return {"bytes": size * (qs + os_ + ks + vs), "flops": 2 * n * (dk + dv)}
    return {"bytes": size * (2 * qs + 2 * os_ + 2 * ks + 2 * vs), "flops": 2 * n * (dk + dv) + 2 * n * (3 * dk + 2 * dv)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "adam_clip":
        total = torch.zeros((), dtype=torch.float64, device=DEV)
        for g in s["g"]:
            total += torch.dot(g.double(), g.double())
        norm = total.sqrt()
        c = torch.minimum(torch.ones_like(norm), s["max_norm"] / (norm + 1e-6))
        t, (b1, b2) = s["steps"] + 1, s["betas"]
        g = torch.zeros(s["p_all"].numel(), dtype=torch.float64, device=DEV)
        for x, p in zip(s["g"], s["p"]):
            g[p.storage_offset():p.storage_offset() + p.numel()] = c * x.double()
        m = b1 * s["m_all"].double() + (1 - b1) * g
        v = b2 * s["v_all"].double() + (1 - b2) * g ** 2
        return [norm, s["p_all"].double() - s["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + s["eps"]), m, v]
    B, H, tq, tk = case["B"], case["heads"], case["tq"], case["tk"]
    rel = None
    if case["bias"]:
        # positions through a look-up by distance instead of comparisons
        half, edges = case["bias"] // 2, _edges(case["bias"] // 2, case["distance"])
        far = max(abs(case["step"] * (tk - 1) + case["offset"]), abs(case["offset"] - tq + 1), abs(case["offset"]),
                  abs(case["step"] * (tk - 1) + case["offset"] - tq + 1)) + 1
        lut = torch.zeros(far + 1, dtype=torch.int64)
        for j, e in enumerate(edges):
            lut[e:] = j
        lut = lut.to(DEV)
        t, k = torch.arange(tq, device=DEV), torch.arange(tk, device=DEV)
        diff = k[:, None] * case["step"] + case["offset"] - t
        rel = torch.where(diff > 0, lut[diff.abs()] + half, lut[diff.abs()])
    if case["op"] == "relative_bias":
        out = torch.empty(B * H, tk, tq, dtype=torch.float64, device=DEV)
        sums = torch.zeros(case["bias"], H, dtype=torch.float64, device=DEV)
        for i in range(B * H):
            out[i] = s["scores"][i].double() + s["table"].double()[rel, i % H]
            sums[:, i % H].index_add_(0, rel.reshape(-1), s["g"][i].double().reshape(-1))
        return [out, s["g"].double(), sums]
    kv, dk, dv, train = case["kv_heads"], case["dk"], case["dv"], case["train"]
    o = torch.zeros(B, H, dv, tq, dtype=torch.float64, device=DEV)
    gq = torch.zeros(B, H, dk, tq, dtype=torch.float64, device=DEV)
    gk = torch.zeros(B, kv, dk, tk, dtype=torch.float64, device=DEV)
    gv = torch.zeros(B, kv, dv, tk, dtype=torch.float64, device=DEV)
    gt = torch.zeros(max(case["bias"], 1), H, dtype=torch.float64, device=DEV)
    for b in range(B):
        for h in range(H):
            live = torch.arange(tk, device=DEV) if s["mask"] is None else s["mask"][b].nonzero()[:, 0]
            if live.numel() == 0:
                continue
            u = h // (H // kv)
            q = s["q"][b, h * dk:(h + 1) * dk].double()
            k = s["k"][b, u * dk:(u + 1) * dk].double()[:, live]
            v = s["v"][b, u * dv:(u + 1) * dv].double()[:, live]
            score = (q.t() @ k) * s["scale"]  # [Tq, live keys]
            if case["bias"]:
                score = score + s["table"].double()[:, h][rel[live]].t()
            p = torch.exp(score - torch.logsumexp(score, 1, keepdim=True))
            o[b, h] = v @ p.t()
            if train:
                g = s["g"][b, h * dv:(h + 1) * dv].double()
                dp = g.t() @ v
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                gv[b, u][:, live] += g @ p
                gk[b, u][:, live] += s["scale"] * (q @ ds)
                gq[b, h] = s["scale"] * (k @ ds.t())
                if case["bias"]:
                    gt[:, h].index_add_(0, rel[live].reshape(-1), ds.t().reshape(-1))
    res = [o.view(B, H * dv, tq)]
    if train:
        res += [gq.view(B, H * dk, tq), gk.view(B, kv * dk, tk), gv.view(B, kv * dv, tk)]
        if case["bias"]:
            res.append(gt)
    return res
