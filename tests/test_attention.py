"""Attention without stored maps (ops.attention), learned relative positions (ops.RelativeBuckets, ops.relative_bias):
against the formulas in float64 on the CPU, at the lengths, masks and layouts where tiles end, plus their refusals.

Tolerances, relative to the norm of the compared tensor.  u = half a step of the type.
float32 (u = 2^-24): a product of three-piece operands is off by at most ~4 u, a sum of n of them by ~sqrt(n) u more; the
scores of these inputs reach ~8, so their absolute error, which becomes the relative error of the probabilities, is below
8 (4 + sqrt(128)) u ~ 128 u; the output adds a sum over the keys.  Outputs: 256 u.  Gradients pass two more products and
the difference dP - delta: 1024 u.
bfloat16 (u = 2^-8): rounded are P (or dS) and the result, so outputs 2 u; gradients round P or dS and the result, and
delta uses 16 bits of the output: 4 u.  The sums and statistics are float32 and do not count."""
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
OUT = {torch.float32: 256, torch.bfloat16: 2}
GRAD = {torch.float32: 1024, torch.bfloat16: 4}


def rel_err(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    scale = max(float(want.norm()), 1e-30)
    return float((got - want).norm()) / scale


def positions(buckets, tq, tk):
    rel = torch.arange(tk)[:, None] * buckets.step + buckets.offset - torch.arange(tq)[None, :]
    lut = {int(r): buckets.bucket(int(r)) for r in rel.unique()}
    return rel.apply_(lut.__getitem__)


def plain(q, k, v, heads, kv, scale, mask=None, table=None, buckets=None, tap=None):
    """float64, per head; masked and barred pairs left out of the sums.  ``tap``: receives the probabilities and the
    expanded values."""
    B, tq, tk = q.shape[0], q.shape[2], k.shape[2]
    dk, dv, G = q.shape[1] // heads, v.shape[1] // kv, heads // kv
    keep = torch.ones(B, 1, tk, 1, dtype=torch.bool) if mask is None else mask[:, None, :, None]
    k = torch.where(keep[:, 0, :, 0][:, None, :], k, torch.zeros((), dtype=k.dtype))
    v = torch.where(keep[:, 0, :, 0][:, None, :], v, torch.zeros((), dtype=v.dtype))
    qh = q.view(B, heads, dk, tq)
    kh = k.view(B, kv, 1, dk, tk).expand(B, kv, G, dk, tk).reshape(B, heads, dk, tk)
    vh = v.view(B, kv, 1, dv, tk).expand(B, kv, G, dv, tk).reshape(B, heads, dv, tk)
    s = scale * kh.transpose(2, 3) @ qh
    if table is not None:
        bias = table[positions(buckets, tq, tk)].permute(2, 0, 1)
        barred = bias <= -1e30
        s = s + bias.masked_fill(barred, 0.0)
        keep = keep & ~barred
    keep = keep.expand(s.shape)
    s = s.masked_fill(~keep, -1e300)
    e = torch.exp(s - s.amax(2, keepdim=True).detach()) * keep
    z = e.sum(2, keepdim=True)
    p = e / torch.where(z > 0, z, torch.ones_like(z))
    if tap is not None:
        tap.extend((p.detach(), vh.detach()))
    return (vh @ p).reshape(B, heads * dv, tq)


def table_terms(tap, out, g):
    """What the terms of a table gradient amount to: an entry sums dS = P (dP - delta) over many pairs that cancel (every
    query's dS sum to zero), so its rounding is relative to the terms.  P's error (the query's log-sum, its scores) is
    common to a query: its terms add up; different queries' errors are independent: they add in squares.  Second number: the
same with every term's error independent (the rounding of each P to bfloat16 in the forward product, which reaches delta
and through it the query's terms in every bucket)."""
    p, vh = tap
    gh = g.view(p.shape[0], p.shape[1], vh.shape[2], -1)
    delta = (gh * out.detach().view(gh.shape)).sum(2).abs()
    terms = p * (vh.transpose(2, 3) @ gh).abs()
    return float((terms.sum(2) + delta).norm()), float(terms.norm())


def make(B, heads, kv, dk, dv, tq, tk, dtype, seed=0, table=None):
    gen = torch.Generator().manual_seed(seed * 7919 + tq * 31 + tk)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    t = [rnd(B, heads * dk, tq), rnd(B, kv * dk, tk), rnd(B, kv * dv, tk), rnd(B, heads * dv, tq)]
    if table is not None:
        t.append((rnd(table.num_buckets, heads).float() * 1.5).to(dtype))
    return t


def check(dev, q, k, v, g, heads, kv, scale=None, mask=None, table=None, buckets=None, what=""):
    from eeggan_amd import ops
    dt = q.dtype
    scale = (q.shape[1] // heads) ** -0.5 if scale is None else scale
    ins64 = [t.double().requires_grad_(True) for t in (q, k, v)] + ([table.double().requires_grad_(True)] if table is not None else [])
    tap = []
    want = plain(*ins64[:3], heads, kv, scale, mask, ins64[3] if table is not None else None, buckets, tap)
    gw = torch.autograd.grad(want, ins64, g.double())
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v)] + ([table.to(dev).requires_grad_(True)] if table is not None else [])
    m = None if mask is None else mask.to(dev)
    got = ops.attention(*ins[:3], heads=heads, kv_heads=kv, scale=scale, mask=m,
                        bias=ins[3] if table is not None else None, buckets=buckets)
    gg = torch.autograd.grad(got, ins, g.to(dev))
    with torch.no_grad():
        quiet = ops.attention(*ins[:3], heads=heads, kv_heads=kv, scale=scale, mask=m,
                              bias=ins[3] if table is not None else None, buckets=buckets)
    assert torch.equal(quiet, got), what
    assert got.dtype == dt and rel_err(got, want) <= OUT[dt] * U[dt], (what, "out", rel_err(got, want))
    for name, a, b in zip(("q", "k", "v", "table"), gg, gw):
        assert a.dtype == dt and a.shape == b.shape
        if k.shape[2] == 1 and name != "v":
            # one key: dS = P (dP - delta) is zero, as the difference of two float32 sums of n = Dv products g v, each off
            # by at most n 2^-24 sum |g v| (output + rest of a bfloat16 output: 2^-16 of it more): the gradients are
            # bounded by what such a dS multiplies, summed over the queries and shared heads
            n = v.shape[1] // kv
            ds = 2 * (n * 2.0 ** -24 + (2.0 ** -16 if dt == torch.bfloat16 else 0.0)) * float(g.double().norm() * v.double().norm())
            reach = 1.0 if name == "table" else scale * float((k if name == "q" else q).double().norm())
            assert float(a.double().norm()) <= ds * reach * (q.shape[2] * heads) ** 0.5, (what, name)
        elif float(b.norm()) == 0.0:
            assert not a.any(), (what, name)
        elif name == "table":
            # (1024 u of float32 for the terms, delta of a bfloat16 output 2^-16; then the result's own rounding)
            terms, single = table_terms(tap, want, g.double())
            bound = 1024 * 2.0 ** -24 * terms + U[dt] * float(b.norm())
            if dt == torch.bfloat16:
                bound += 2.0 ** -16 * terms + U[dt] * single
            assert float((a.cpu().double() - b).norm()) <= bound, (what, name, rel_err(a, b))
        else:
            assert rel_err(a, b) <= GRAD[dt] * U[dt], (what, name, rel_err(a, b))
    return got, gg


# ------------------------------------------------------------------------------------------------ the kernels
CLASSES = [(8, 32), (5, 17), (16, 64), (13, 50), (32, 32), (32, 128), (20, 100), (64, 64), (48, 40), (128, 128), (96, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dk,dv", CLASSES)
def test_channel_classes(dev, dk, dv, dtype):
    """Every tile class at full and at odd channel counts; lengths that end inside a tile, one column block and several."""
    for B, heads, kv, tq, tk in ((2, 1, 1, 70, 45), (1, 2, 2, 161, 130)):
        q, k, v, g = make(B, heads, kv, dk, dv, tq, tk, dtype)
        check(dev, q, k, v, g, heads, kv, what=(dk, dv, tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 2), (2, 1), (3, 33), (31, 32), (32, 31), (33, 64), (64, 65), (127, 129),
                                   (128, 128), (129, 127), (1, 515), (5, 1030), (640, 3), (513, 257)])
def test_lengths(dev, tq, tk, dtype):
    q, k, v, g = make(2, 2, 1, 24, 40, tq, tk, dtype)
    check(dev, q, k, v, g, 2, 1, what=(tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (4, 2), (6, 2), (8, 1), (3, 1)])
def test_shared_key_heads(dev, heads, kv, dtype):
    for tq, tk in ((50, 77), (1, 300), (7, 40)):
        q, k, v, g = make(2, heads, kv, 16, 24, tq, tk, dtype)
        check(dev, q, k, v, g, heads, kv, what=(tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tq", [1, 40, 150])
def test_masks(dev, tq, dtype):
    """Ragged lengths, holes, whole tiles without a key, one single key, no key at all; what masked keys hold (NaN,
    infinities, the type's largest values) never reaches a result, and their gradients are zero."""
    tk, B = 203, 6
    q, k, v, g = make(B, 2, 2, 20, 30, tq, tk, dtype, seed=3)
    mask = torch.zeros(B, tk, dtype=torch.bool)
    mask[0] = True
    mask[1, :101] = True
    mask[2, 70:71] = True
    mask[3, 64:128] = True
    mask[4, ::3] = True
    clean = check(dev, q, k, v, g, 2, 2, mask=mask, what="clean")
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).max, torch.finfo(dtype).min])
    dirt = bad[torch.arange(B * tk).view(B, 1, tk) % 5].to(dtype)
    k2, v2 = (torch.where(mask[:, None, :], t, dirt.expand_as(t)) for t in (k, v))
    dirty = check(dev, q, k2, v2, g, 2, 2, mask=mask, what="dirty")
    assert torch.equal(clean[0], dirty[0]) and all(torch.equal(a, b) for a, b in zip(clean[1], dirty[1]))
    assert not dirty[0][5].any()
    hidden = ~mask.to(dev)[:, None, :].expand(B, 40, tk)
    assert not dirty[1][1][hidden].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("conf", [dict(num_buckets=16, max_distance=40), dict(num_buckets=32, max_distance=128),
                                  dict(num_buckets=8, max_distance=64, step=4, offset=2),
                                  dict(num_buckets=10, max_distance=300, step=2, offset=-37),
                                  dict(num_buckets=12, max_distance=60, bidirectional=False),
                                  dict(num_buckets=32, max_distance=1024, step=16, offset=500)])
def test_positions(dev, conf, dtype):
    from eeggan_amd import ops
    b = ops.RelativeBuckets(**conf)
    for heads, kv, tq, tk in ((2, 2, 333, 90), (4, 2, 40, 200), (2, 1, 1, 150), (1, 1, 300, 517)):
        q, k, v, g, table = make(2, heads, kv, 16, 32, tq, tk, dtype, table=b)
        mask = torch.rand(2, tk, generator=torch.Generator().manual_seed(tk)) < 0.8
        check(dev, q, k, v, g, heads, kv, mask=mask, table=table, buckets=b, what=(conf, tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(8, 32), (32, 128), (64, 64), (128, 128)])
def test_positions_in_every_class(dev, dk, dv):
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 50, step=2, offset=3)
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, table = make(1, 3, 1, dk, dv, 270, 140, dtype, table=b)
        check(dev, q, k, v, g, 3, 1, table=table, buckets=b, what=(dk, dv, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -1e30])
def test_table_entries_that_bar_pairs(dev, value):
    """Bars the own position and everything ahead: the first query is left without a key."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40)
    q, k, v, g, table = make(2, 2, 2, 16, 16, 75, 75, torch.float32, table=b)
    table[0] = value
    table[8:] = value
    out, grads = check(dev, q, k, v, g, 2, 2, table=table, buckets=b, what=value)
    assert not out[:, :, 0].any() and not grads[0][:, :, 0].any()
    assert not grads[3][0].any() and not grads[3][8:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_layouts(dev, dtype):
    """Slices of one wider projection, odd storage offsets, time-major storage, an expanded batch, another batch order."""
    from eeggan_amd import ops
    B, heads, d, t = 3, 2, 12, 67
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(B, 3 * heads * d, t + 3, generator=gen).to(dtype).to(dev)
    q, k, v = (wide[:, i * heads * d:(i + 1) * heads * d, 1:t + 1] for i in range(3))
    ref = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), heads=heads, scale=0.3)
    forms = {"slices": (q, k, v),
             "time-major": tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)),
             "flipped batch": tuple(x.flip(0).contiguous().flip(0) for x in (q, k, v))}
    g = torch.ones((), device=dev, dtype=dtype).expand_as(ref)  # (a cotangent without strides)

    def grads(ins):
        leaves = [x.detach().requires_grad_(True) for x in ins]
        out = ops.attention(*leaves, heads=heads, scale=0.3)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, g))
    want = grads([x.contiguous() for x in (q, k, v)])
    for name, ins in forms.items():
        assert all(torch.equal(a, b) for a, b in zip(grads(ins), want)), name
    k1, v1 = k[:1].expand(B, -1, -1), v[:1].expand(B, -1, -1)
    assert torch.equal(ops.attention(q, k1, v1, heads=heads), ops.attention(q, k1.contiguous(), v1.contiguous(), heads=heads))


@pytest.mark.gpu
def test_gradients_of_expanded_inputs(dev):
    """Keys and values shared by the samples of a batch: the gradient is the sum over the samples."""
    from eeggan_amd import ops
    q, k, v, g = make(3, 2, 2, 16, 16, 40, 50, torch.float32)
    k, v = k[:1], v[:1]
    ins64 = [t.double().requires_grad_(True) for t in (q, k, v)]
    want = plain(ins64[0], ins64[1].expand(3, -1, -1), ins64[2].expand(3, -1, -1), 2, 2, 0.25)
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    got = ops.attention(ins[0], ins[1].expand(3, -1, -1), ins[2].expand(3, -1, -1), heads=2, scale=0.25)
    for a, b in zip(torch.autograd.grad(got, ins, g.to(dev)), torch.autograd.grad(want, ins64, g.double())):
        assert rel_err(a, b) <= 1024 * 2.0 ** -24


@pytest.mark.gpu
def test_one_step_over_a_long_recording(dev):
    """Few query columns and many keys: waves and workgroups split the keys; a mask that leaves whole parts empty."""
    for dtype in (torch.float32, torch.bfloat16):
        for d, kv, heads, tq, tk in ((64, 2, 8, 1, 9001), (128, 1, 3, 5, 5000), (32, 1, 1, 1, 30011)):
            q, k, v, g = make(2, heads, kv, d, d, tq, tk, dtype)
            mask = torch.zeros(2, tk, dtype=torch.bool)
            mask[0, 4000:4100] = True
            mask[1, ::2] = True
            check(dev, q, k, v, g, heads, kv, mask=mask, what=(dtype, d, tk))
            check(dev, q, k, v, g, heads, kv, what=(dtype, d, tk))


@pytest.mark.gpu
def test_large_scores(dev):
    """Scores of +-300 (probabilities of one and far below the smallest float) and rows whose maximum comes last."""
    from eeggan_amd import ops
    q, k, v, g = make(1, 1, 1, 16, 32, 96, 300, torch.float32)
    k = k * torch.linspace(0.01, 60.0, 300)
    ins64 = [t.double() for t in (q, k, v)]
    want = plain(*ins64, 1, 1, 1.0)
    got = ops.attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0)
    # scores of up to S = 600 are off by ~ 600 * 16 u: as much the probabilities, relatively
    assert rel_err(got, want) <= 600 * 16 * 2.0 ** -24
    low = ops.attention(q.to(dev), k.to(dev), v.to(dev), scale=-1.0)
    assert rel_err(low, plain(*ins64, 1, 1, -1.0)) <= 600 * 16 * 2.0 ** -24
    flat = ops.attention(q.to(dev), k.to(dev), v.to(dev), scale=0.0)
    assert rel_err(flat, v.double().mean(2, keepdim=True).expand(1, 32, 96)) <= 256 * 2.0 ** -24


@pytest.mark.gpu
def test_non_finite_inputs_stay_where_they_belong(dev):
    """A NaN in a query spoils its own column, a NaN in an attended value its own channel: nothing else."""
    from eeggan_amd import ops
    q, k, v, _ = make(2, 1, 1, 16, 32, 64, 64, torch.float32)
    ref = ops.attention(q.to(dev), k.to(dev), v.to(dev))
    q2, v2 = q.clone(), v.clone()
    q2[0, 3, 10] = float("nan")
    v2[1, 5, 20] = float("nan")
    got = ops.attention(q2.to(dev), k.to(dev), v2.to(dev))
    bad = torch.zeros_like(q[:, :1].expand(2, 32, 64), dtype=torch.bool).clone()
    bad[0, :, 10] = True
    bad[1, 5, :] = True
    assert bool(torch.isnan(got.cpu()[bad]).all()) and torch.equal(got.cpu()[~bad], ref.cpu()[~bad])


@pytest.mark.gpu
def test_equal_inputs_give_equal_bits(dev):
    from eeggan_amd import ops
    b = ops.RelativeBuckets(32, 128, step=4, offset=2)
    q, k, v, g, table = make(4, 4, 2, 16, 64, 700, 180, torch.float32, table=b)
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v, table)]

    def once():
        out = ops.attention(*ins[:3], heads=4, kv_heads=2, scale=0.25, bias=ins[3], buckets=b)
        return (out.detach(),) + torch.autograd.grad(out, ins, g.to(dev))
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """Central differences of the kernel's own forward: along a random direction the change of <out, g> is the inner
    product of the gradients with it.  h = 1/64: the cubic remainder is ~h^2 = 2.4e-4 of the value and the float32
    rounding of the two sums (~2^-24 sqrt(n) |out| |g| / 2h) below that; 2e-3 covers both."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 50, step=2, offset=1)
    q, k, v, g, table = make(2, 2, 1, 8, 16, 90, 45, torch.float32, table=b)
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v, table)]
    f = lambda xs: ops.attention(*xs[:3], heads=2, kv_heads=1, scale=0.35, bias=xs[3], buckets=b)  # noqa: E731
    grads = torch.autograd.grad(f(ins), ins, g.to(dev))
    gen = torch.Generator().manual_seed(9)
    for i in range(4):
        way = torch.randn(ins[i].shape, generator=gen).to(dev) * 0.25
        h = 1.0 / 64
        with torch.no_grad():
            up, down = ([x + (s * h * way if j == i else 0) for j, x in enumerate(ins)] for s in (1, -1))
            diff = ((f(up).double() - f(down).double()) * g.to(dev).double()).sum() / (2 * h)
        want = (grads[i].double() * way.double()).sum()
        size = float(grads[i].double().norm() * way.double().norm())
        assert abs(float(diff - want)) <= 2e-3 * size, (i, float(diff), float(want))


@pytest.mark.gpu
def test_second_derivatives(dev):
    """create_graph: the gradient of a gradient norm, with shared heads, a mask (one sample without keys) and positions."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 30, step=2, offset=1)
    q, k, v, g, table = make(3, 2, 1, 8, 12, 50, 25, torch.float32, table=b)
    mask = torch.ones(3, 25, dtype=torch.bool)
    mask[0, 10:] = False
    mask[1] = False

    def second(ins, f, g):
        out = f(ins)
        first = torch.autograd.grad(out, ins, g, create_graph=True)
        return torch.autograd.grad(sum((x ** 2).sum() for x in first), ins)
    ins64 = [t.double().requires_grad_(True) for t in (q, k, v, table)]
    want = second(ins64, lambda x: plain(*x[:3], 2, 1, 0.35, mask, x[3], b), g.double())
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v, table)]
    got = second(ins, lambda x: ops.attention(*x[:3], heads=2, kv_heads=1, scale=0.35, mask=mask.to(dev), bias=x[3], buckets=b),
                 g.to(dev))
    for a, c in zip(got, want):  # (two backward passes: twice the gradients' bound)
        assert rel_err(a, c) <= 2048 * 2.0 ** -24, rel_err(a, c)


@pytest.mark.gpu
def test_captured_and_replayed(dev):
    """Forward and backward in a captured graph, replayed on changing inputs between eager work; two graphs in turn."""
    from eeggan_amd import ops
    from eeggan_amd.graphs import capture
    b = ops.RelativeBuckets(16, 64, step=4, offset=2)
    sets = [[t.to(dev) for t in make(2, 2, 1, 8, 32, tq, tk, torch.float32, seed=i, table=b)]
            for i, (tq, tk) in enumerate(((200, 50), (1, 400)))]

    def work(s):
        ins = [s[i].detach().requires_grad_(True) for i in (0, 1, 2, 4)]
        out = ops.attention(*ins[:3], heads=2, kv_heads=1, scale=0.35, bias=ins[3], buckets=b)
        return [out.detach()] + list(torch.autograd.grad(out, ins, s[3]))
    graphs = []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with capture(graph):
            res = work(s)
        graphs.append((graph, res))
    for turn in range(4):
        for s in sets:
            for t in s:
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(turn)).to(dev))
        for graph, _ in graphs:
            graph.replay()
        for (_, res), s in zip(graphs, sets):
            assert all(torch.equal(a, c) for a, c in zip(res, work(s))), turn
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_on_another_stream(dev):
    from eeggan_amd import ops
    q, k, v, g = (t.to(dev) for t in make(2, 2, 2, 16, 32, 300, 200, torch.float32))
    ref = ops.attention(q, k, v, heads=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.attention(q, k, v, heads=2) for _ in range(5)]
    same = [ops.attention(q, k, v, heads=2) for _ in range(5)]  # (both streams at once)
    side.synchronize()
    assert all(torch.equal(o, ref) for o in outs + same)


# ------------------------------------------------------------------------------------------------ positions on scores
@pytest.mark.gpu
@pytest.mark.parametrize("conf", [dict(num_buckets=16, max_distance=40), dict(num_buckets=8, max_distance=64, step=4, offset=2),
                                  dict(num_buckets=12, max_distance=60, bidirectional=False, offset=-5),
                                  dict(num_buckets=32, max_distance=1024, step=16, offset=500)])
@pytest.mark.parametrize("B,heads,tq,tk", [(1, 1, 1, 1), (2, 3, 37, 19), (3, 2, 128, 32), (2, 1, 515, 261), (1, 2, 1027, 1030)])
def test_relative_bias(dev, conf, B, heads, tq, tk):
    """The sum is one rounding (u); the gradient is a sum in double of float32 values, rounded once: its bound counts the
    float32 sums of a tile too (64 u of the root of the sum of squares times the root of the count)."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(**conf)
    gen = torch.Generator().manual_seed(tq)
    s, g = torch.randn(B * heads, tk, tq, generator=gen), torch.randn(B * heads, tk, tq, generator=gen)
    table = torch.randn(b.num_buckets, heads, generator=gen)
    where = positions(b, tq, tk)
    td = table.double().requires_grad_(True)
    want = s.double() + td[where].permute(2, 0, 1).repeat(B, 1, 1)
    wg, = torch.autograd.grad(want, td, g.double())
    sg, tg = s.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True)
    got = ops.relative_bias(sg, tg, b, heads=heads)
    assert float((got.detach().cpu().double() - want.detach()).abs().max()) <= 2.0 ** -24 * 16
    ggs, ggt = torch.autograd.grad(got, [sg, tg], g.to(dev))
    assert torch.equal(ggs.cpu(), g)
    assert float((ggt.cpu().double() - wg).norm()) <= 64 * 2.0 ** -24 * float(g.double().norm())
    assert not ggt.cpu()[wg == 0].any()


@pytest.mark.gpu
def test_relative_bias_to_second_order(dev):
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40, step=2)
    gen = torch.Generator().manual_seed(2)
    s, table = torch.randn(4, 30, 60, generator=gen), torch.randn(16, 2, generator=gen)
    where = positions(b, 60, 30)

    def second(s, t, f, soft):
        out = (soft(f(s, t)) ** 2).sum()
        first = torch.autograd.grad(out, [s, t], create_graph=True)
        return torch.autograd.grad((first[0] ** 2).sum() + (first[1] ** 2).sum(), [s, t])
    want = second(s.double().requires_grad_(True), table.double().requires_grad_(True),
                  lambda x, t: x + t[where].permute(2, 0, 1).repeat(2, 1, 1), lambda x: torch.softmax(x, 1))
    got = second(s.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True),
                 lambda x, t: ops.relative_bias(x, t, b, heads=2), ops.softmax_dim1)
    for a, c in zip(got, want):
        assert rel_err(a, c) <= 2048 * 2.0 ** -24, rel_err(a, c)


# ------------------------------------------------------------------------------------------------ without a GPU
def test_bucket_borders():
    from eeggan_amd import ops
    for conf in (dict(), dict(num_buckets=8, max_distance=200), dict(num_buckets=12, max_distance=60, bidirectional=False),
                 dict(num_buckets=64, max_distance=1024)):
        b = ops.RelativeBuckets(**conf)
        side = b.num_buckets // 2 if b.bidirectional else b.num_buckets
        exact, grown = side // 2, side - side // 2
        assert b.edges[:exact + 1] == tuple(range(exact + 1)) and len(b.edges) == side
        for i, e in enumerate(b.edges[exact:]):
            bound = exact ** (grown - i) * b.max_distance ** i
            assert e ** grown >= bound and ((e - 1) ** grown < bound or e == b.edges[exact + i - 1] + 1)
        assert b.bucket(0) == 0 and b.bucket(-10 ** 6) == side - 1
        assert b.bucket(10 ** 6) == (b.num_buckets - 1 if b.bidirectional else 0)
        import copy
        import pickle
        for other in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
            assert other.edges == b.edges and list(other._c.edges) == list(b._c.edges) and other._ptr() != b._ptr()


@pytest.mark.parametrize("conf", [dict(num_buckets=2), dict(num_buckets=33), dict(num_buckets=130), dict(step=0), dict(step=17),
                                  dict(max_distance=8), dict(max_distance=1025), dict(num_buckets=64, max_distance=20),
                                  dict(num_buckets=65, bidirectional=False)])
def test_bucket_refusals(conf):
    from eeggan_amd import ops
    with pytest.raises(ValueError):
        ops.RelativeBuckets(**conf)


def test_no_cpu_path():
    from eeggan_amd import ops
    x = torch.zeros(1, 4, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attention(x, x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.relative_bias(x, torch.zeros(32, 1), ops.RelativeBuckets())
    with pytest.raises(ValueError):
        ops.set_attention("tiled")


def test_c_entry_points_refuse_before_any_launch():
    """Argument checks of the C ABI happen on the host: every call below names a fault and launches nothing."""
    import ctypes
    from eeggan_amd import _lib, ops
    lib = _lib.load()
    b = ops.RelativeBuckets()

    def desc(**kw):
        a = ops._AttentionDesc()
        a.q, a.k, a.v = 256, 512, 768
        a.q_batch, a.q_channel, a.k_batch, a.k_channel, a.v_batch, a.v_channel = 80, 10, 80, 10, 80, 10
        a.B, a.H, a.KV, a.Dk, a.Dv, a.Tq, a.Tk, a.scale = 1, 2, 1, 8, 8, 10, 10, 1.0
        for key, value in kw.items():
            setattr(a, key, value)
        return a
    assert lib.eeggan_attention_fwd_workspace(ctypes.byref(desc())) > 0
    edges = (ctypes.c_int * 64)(*([0, 5, 5] + [0] * 61))
    broken = ops._Buckets(6, 1, 1, 0, edges)
    far = ops._Buckets(4, 1, 1, 0, (ctypes.c_int * 64)(0, 1025))
    for kw, message in ((dict(q=None), b"null"), (dict(B=0), b"bad shape"), (dict(Tk=0), b"bad shape"), (dict(H=3, KV=2), b"share"),
                        (dict(Dk=129), b"128 channels"), (dict(Dv=200), b"128 channels"), (dict(Tq=1 << 28), b"time steps"),
                        (dict(k_channel=-1), b"negative"), (dict(q=258), b"misaligned"), (dict(bf16=1, v=769), b"misaligned"),
                        (dict(table=256), b"buckets"), (dict(table=256, buckets=ctypes.addressof(broken)), b"increase"),
                        (dict(table=256, buckets=ctypes.addressof(far)), b"1024")):
        a = desc(**kw)
        assert lib.eeggan_attention_fwd(ctypes.byref(a), 256, None, None, 256, 1 << 30, None) != 0, kw
        assert message in lib.eeggan_last_error(), (kw, lib.eeggan_last_error())
        assert lib.eeggan_attention_fwd_workspace(ctypes.byref(a)) == 0
        assert lib.eeggan_attention_bwd_workspace(ctypes.byref(a), 1) == 0
    a = desc()
    assert lib.eeggan_attention_fwd(ctypes.byref(a), 256, None, None, 256, 0, None) != 0 and b"workspace" in lib.eeggan_last_error()
    assert lib.eeggan_attention_bwd(ctypes.byref(a), 256, None, 256, 256, 256, 256, 256, 256, 256, 1 << 30, None) != 0
    assert b"without a table" in lib.eeggan_last_error()
    assert lib.eeggan_attention_bwd(ctypes.byref(a), 256, None, 256, 256, 256, 256, 256, None, 256, 0, None) != 0
    assert b"workspace" in lib.eeggan_last_error()
    a = desc(bf16=1)
    assert lib.eeggan_attention_bwd(ctypes.byref(a), 256, None, 256, 256, 256, 256, 256, None, 256, 1 << 30, None) != 0
    assert b"rest" in lib.eeggan_last_error()
    assert lib.eeggan_relative_bias(None, None, b._ptr(), 256, 1, 1, 1, 1, None) != 0
    assert lib.eeggan_relative_bias(None, 256, None, 256, 1, 1, 1, 1, None) != 0 and b"missing" in lib.eeggan_last_error()
    assert lib.eeggan_relative_bias(None, 256, b._ptr(), 256, 1, 0, 1, 1, None) != 0
    assert lib.eeggan_relative_bias_grad(256, b._ptr(), 256, 1, 1, 5, 5, 256, 0, None) != 0


@pytest.mark.gpu
def test_refusals(dev):
    from eeggan_amd import ops
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device=dev, dtype=dt)  # noqa: E731
    b = ops.RelativeBuckets()
    ok = (z(2, 8, 5), z(2, 8, 6), z(2, 4, 6))
    ops.attention(*ok, heads=2)
    for args, kw in (((ok[0], ok[1], ok[2].bfloat16()), {}), ((z(2, 8, 5, dt=torch.float16),) * 3, {}), ((ok[0][0], ok[1], ok[2]), {}),
                     ((z(2, 8, 0), ok[1], ok[2]), {}), ((ok[0], z(2, 8, 0), z(2, 4, 0)), {}), ((z(3, 8, 5), ok[1], ok[2]), {}),
                     ((ok[0], ok[1], z(2, 4, 7)), {}), (ok, dict(heads=3)), (ok, dict(heads=4, kv_heads=3)), (ok, dict(heads=0)),
                     ((z(1, 130, 4), z(1, 130, 4), z(1, 4, 4)), {}), ((ok[0], ok[1], z(2, 260, 6)), dict(heads=2)),
                     (ok, dict(mask=torch.zeros(2, 5, dtype=torch.bool, device=dev))), (ok, dict(mask=z(2, 6))),
                     (ok, dict(mask=torch.zeros(2, 6, dtype=torch.bool))), (ok, dict(bias=z(32, 1))), (ok, dict(buckets=b)),
                     (ok, dict(heads=2, bias=z(32, 1), buckets=b)), (ok, dict(bias=z(32, 1, dt=torch.bfloat16), buckets=b)),
                     (ok, dict(bias=torch.zeros(32, 1), buckets=b))):
        with pytest.raises(RuntimeError):
            ops.attention(*args, **kw)
    for args, kw in (((z(3, 4, 5), z(32, 2), b), dict(heads=2)), ((z(2, 4, 5), z(16, 2), b), dict(heads=2)), ((z(2, 4), z(32, 1), b), {}),
                     ((z(2, 4, 5, dt=torch.bfloat16), z(32, 1), b), {}), ((z(2, 0, 5), z(32, 1), b), {}), ((z(2, 4, 5), z(32, 1), None), {})):
        with pytest.raises(RuntimeError):
            ops.relative_bias(*args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(96, 96), (90, 70), (33, 65), (65, 33), (96, 97), (97, 96)])
def test_up_to_96_channels(dev, dk, dv, dtype):
    from eeggan_amd import ops
    buckets = ops.RelativeBuckets(16, 40)
    for B, heads, kv, tq, tk in ((2, 1, 1, 70, 45), (1, 2, 2, 161, 130), (3, 4, 1, 1, 70)):
        q, k, v, g = make(B, heads, kv, dk, dv, tq, tk, dtype)
        check(dev, q, k, v, g, heads, kv, what=(dk, dv, tq, tk))
    q, k, v, g, table = make(1, 2, 2, dk, dv, 140, 131, dtype, table=buckets)
    check(dev, q, k, v, g, 2, 2, table=table, buckets=buckets, what=(dk, dv, "positions"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tk", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 200)], ids=["f32", "bf16-short", "bf16"])
def test_table_gradient_sums_to_zero(dev, dtype, tk):
    """Every query's dS sum to zero, so all buckets' gradients of a head do.  What is left is rounding: delta and the dP of a
    query carry errors of random sign, each at most u of sum |dO O| or of |dP| with u = 2^-23 (float32: half a step from the
    output and half from the sums) or 2^-16 (bfloat16: the output in two parts, P in two pieces), so N queries leave about
    sqrt(N) u rms(dP): bounded by six times that.  An error that goes the same way in every query would add up to N times
    itself: 2e-9 of dP in each is past the bound here."""
    from eeggan_amd import ops
    B, heads, dk, dv, tq = 32, 2, 8, 32, 2300
    gen = torch.Generator(device=dev).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen).to(dtype)  # noqa: E731
    q, k, v, g = rnd(B, heads * dk, tq), rnd(B, heads * dk, tk), rnd(B, heads * dv, tk), rnd(B, heads * dv, tq)
    buckets = ops.RelativeBuckets(16, 64, step=16)
    table = torch.randn(16, heads, device=dev, generator=gen).requires_grad_(True)
    out = ops.attention(q, k, v, heads=heads, scale=dk ** -0.5, bias=table, buckets=buckets)
    gt, = torch.autograd.grad(out, [table], g)
    u = 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -16
    left = gt.double().sum(0).abs().max()
    bound = 6.0 * (B * tq) ** 0.5 * u * dv ** 0.5  # (rms of dP: a sum of dv products of unit variance)
    assert float(left) <= bound, (float(left), bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_saved_tensors_that_move(dev, dtype):
    """Saved-tensor hooks give the backward pass other tensors than the forward pass saved: copies from the host, results of
    a second forward pass.  Same bits as without them."""
    from eeggan_amd import ops
    from torch.utils.checkpoint import checkpoint
    buckets = ops.RelativeBuckets(16, 40)
    q, k, v, g, table = (t.to(dev) for t in make(2, 4, 2, 24, 40, 75, 66, dtype, table=buckets))
    mask = torch.arange(66, device=dev)[None, :] < torch.tensor([[66], [31]], device=dev)
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]

    def f(q, k, v, table):
        wide = torch.cat([k, q[:, :k.shape[1], :66]], 1)  # (the keys are a slice of a wider tensor that only this pass has)
        return ops.attention(2.0 * q, wide[:, :k.shape[1]], v * 0.5, heads=4, kv_heads=2, scale=0.2, mask=mask.clone(), bias=table * 1.0,
                             buckets=buckets)

    def grads(run):
        out = run()
        junk = [torch.full_like(q, float("nan")) for _ in range(8)]  # (what was freed is written over)
        got = torch.autograd.grad(out, leaves, g)
        del junk
        return [out.detach()] + list(got)

    want = grads(lambda: f(*leaves))
    with torch.autograd.graph.save_on_cpu():
        out = f(*leaves)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, g))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = grads(lambda: checkpoint(f, *leaves, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("conf", [dict(offset=1 << 30), dict(offset=-(1 << 30)), dict(offset=2 ** 32 + 5), dict(offset=0.5), dict(step=1.5)])
def test_positions_outside_their_type(conf):
    from eeggan_amd import ops
    with pytest.raises(ValueError):
        ops.RelativeBuckets(**conf)
    assert ops.RelativeBuckets(offset=(1 << 30) - 1).offset == (1 << 30) - 1


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,kv,dk,dv,tq,tk,train", [(4, 4, 2, 6, 6, 115, 115, True), (2, 2, 1, 128, 5, 257, 5, True), (3, 4, 4, 64, 64, 4, 4, True),
                                                          (2, 2, 2, 32, 96, 300, 170, True), (2, 4, 4, 32, 32, 1, 9000, False)])
def test_small_calls_in_bfloat16_round_only_their_results(dev, B, heads, kv, dk, dv, tq, tk, train):
    """Up to 16 M pairs (few columns over many keys: 1 M) P and dS keep 2^-18 of themselves, and 16 bits of the output go
    into delta.  The rounding of the result, u = 2^-8, is then nearly all of the error: as much again as rounding the exact
    result leaves, plus 2^-17 per term of sums that cancel to about a tenth of their terms: 2^-13 of the norm."""
    from eeggan_amd import ops
    q, k, v, g = make(B, heads, kv, dk, dv, tq, tk, torch.bfloat16, seed=3)
    ins = [t.double().requires_grad_(True) for t in (q, k, v)]
    want = plain(*ins, heads, kv, dk ** -0.5)
    leaves = [t.to(dev).requires_grad_(train) for t in (q, k, v)]
    got = ops.attention(*leaves, heads=heads, kv_heads=kv, scale=dk ** -0.5)
    pairs = [("out", got, want.detach())]
    if train:
        pairs += list(zip("qkv", torch.autograd.grad(got, leaves, g.to(dev)), torch.autograd.grad(want, ins, g.double())))
    for name, a, b in pairs:
        alone = rel_err(b.to(torch.bfloat16), b)
        assert rel_err(a, b) <= 1.02 * alone + 2.0 ** -13, (name, rel_err(a, b), alone)


@pytest.mark.gpu
def test_a_cache_past_four_gigabytes(dev):
    """One new step, four key heads of 128 channels over 5 million keys in bfloat16: the last heads lie past 2^32 bytes.  The
    last head against float32 products over pieces of the keys (out 2 u as above; the pieces' float32 sums do not count)."""
    from eeggan_amd import ops
    kv, d, tk, piece = 4, 128, 5_000_003, 500_000
    gen = torch.Generator(device=dev).manual_seed(9)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen, dtype=torch.bfloat16)  # noqa: E731
    q, k, v = rnd(1, kv * d, 1), rnd(1, kv * d, tk), rnd(1, kv * d, tk)
    mask = torch.ones(1, tk, dtype=torch.bool, device=dev)
    mask[0, 1_000_000:4_000_000] = False
    with torch.no_grad():
        got = ops.attention(q, k, v, heads=kv, scale=d ** -0.5, mask=mask)[0, -d:, 0].float()
    s = torch.cat([q[0, -d:, 0].float() @ k[0, -d:, x:x + piece].float() for x in range(0, tk, piece)]) * d ** -0.5
    p = torch.softmax(s.double().masked_fill(~mask[0], float("-inf")), 0).float()
    want = sum(v[0, -d:, x:x + piece].float() @ p[x:x + piece] for x in range(0, tk, piece))
    assert rel_err(got, want) <= 2 * U[torch.bfloat16]


@pytest.mark.gpu
def test_stored_scores_past_two_to_the_31(dev):
    """Maps of 48000 x 48000: entry numbers pass 2^31.  scores + table (each entry one float32 addition: exact equality) on
    rows at both ends, and the gradient of a table of ones' sum: counts of pairs, exact in double and float32 to half a step."""
    from eeggan_amd import ops
    n = 48000
    b = ops.RelativeBuckets(16, 64)
    table = torch.arange(16, device=dev, dtype=torch.float32)[:, None].requires_grad_(True)
    scores = torch.full((1, n, n), 0.5, device=dev)
    out = ops.relative_bias(scores, table, b)
    bucket = positions(b, 129, 1)[0]  # distances 0 .. -128
    for s in (0, 64, n - 1):
        row = out[0, s].detach().cpu()
        t = torch.arange(s, min(n, s + 129))
        assert torch.equal(row[t], 0.5 + bucket[:len(t)].float()), s
    gt, = torch.autograd.grad(out, [table], scores)
    dist = torch.arange(n, dtype=torch.float64)
    counts = torch.zeros(16, dtype=torch.float64)
    for d, c in ((0, n),) + tuple((int(x), n - int(x)) for x in dist[1:64]):
        counts[b.bucket(-d)] += c
        if d:
            counts[b.bucket(d)] += c
    counts[b.bucket(-64)] += float((n - dist[64:]).sum())
    counts[b.bucket(64)] += float((n - dist[64:]).sum())
    assert float(((gt[:, 0].cpu().double() - 0.5 * counts).abs() - U[torch.float32] * 0.5 * counts).max()) <= 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [(1 << 30) - 1, -(1 << 30) + 1, 5000, -5000, 131, -131])
def test_positions_far_from_the_queries(dev, offset):
    """Every pair in one bucket (or, at the ends of the list, at the border): the bias drops out of the softmax."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40, step=3, offset=offset)
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, table = (t.to(dev) for t in make(2, 2, 1, 16, 24, 70, 66, dtype, table=b))
        leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
        out = ops.attention(*leaves[:3], heads=2, kv_heads=1, scale=0.25, bias=table, buckets=b)
        got = torch.autograd.grad(out, leaves, g)
        none = ops.attention(*leaves[:3], heads=2, kv_heads=1, scale=0.25)
        want = torch.autograd.grad(none, leaves[:3], g)
        if abs(offset) > 3 * 66 + 70 + 40:
            assert rel_err(out, none) <= 2 * OUT[dtype] * U[dtype]
            for a, w in zip(got, want):
                assert rel_err(a, w) <= 2 * GRAD[dtype] * U[dtype]
            assert int((got[3] != 0).any(1).sum()) <= 1
        else:
            check(dev, *(t.detach().cpu() for t in (q, k, v, g)), 2, 1, scale=0.25, table=table.detach().cpu(), buckets=b, what=offset)


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls that run beside each other on two streams share nothing: the bits of calls that run alone."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 64)
    sets = [[t.to(dev) for t in make(2, 4, 2, 32, 32, 300 + 17 * i, 700, torch.bfloat16, seed=i, table=b)] for i in (0, 1)]
    for s in sets:
        for t in s[:3] + s[4:]:
            t.requires_grad_(True)

    def run(q, k, v, g, table):
        out = ops.attention(q, k, v, heads=4, kv_heads=2, scale=0.2, bias=table, buckets=b)
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v, table], g))

    alone = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    results = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for got in results[i]:
            assert all(torch.equal(a, w) for a, w in zip(got, alone[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 64), (24, 40), (17, 33), (33, 32), (32, 65)])
def test_up_to_32_and_64_channels(dev, dk, dv, dtype):
    from eeggan_amd import ops
    buckets = ops.RelativeBuckets(16, 40, step=2)
    for B, heads, kv, tq, tk in ((2, 1, 1, 70, 45), (1, 2, 2, 161, 130), (3, 4, 1, 1, 70)):
        q, k, v, g = make(B, heads, kv, dk, dv, tq, tk, dtype)
        check(dev, q, k, v, g, heads, kv, what=(dk, dv, tq, tk))
    q, k, v, g, table = make(1, 2, 2, dk, dv, 140, 131, dtype, table=buckets)
    check(dev, q, k, v, g, 2, 2, table=table, buckets=buckets, what=(dk, dv, "positions"))


# ------------------------------------------------------------------------- inputs that share tensors, under create_graph
def _shared(name, x, y, z):
    """(q, k, v) out of three leaves: how arguments may depend on each other."""
    return {"apart": (x, y, z), "k is v": (x, y, y), "q is k": (x, x, z), "all one": (x, x, x), "k from q": (x, 0.5 * x + y, z),
            "v from k": (x, y, 2.0 * y * z)}[name]


SHARED = ["apart", "k is v", "q is k", "all one", "k from q", "v from k"]


@pytest.mark.parametrize("name", SHARED)
def test_first_derivatives_under_create_graph_without_a_gpu(name, monkeypatch):
    """The routing of _Attention.backward, with the formulas in float64 in the place of the stored-score operators: gradients
    of first and second order, and one call of a hook on every leaf, as without the Function."""
    from eeggan_amd import ops

    class OnHost(ops._Attention):
        @staticmethod
        def forward(ctx, q, k, v, table, cfg):
            ctx.cfg = cfg
            ctx.save_for_backward(q, k, v, table, None, None, None, None)
            return plain(q, k, v, 1, 1, 0.4)
    monkeypatch.setattr(ops, "_attention_stored", lambda q, k, v, table, mask, cfg: plain(q.double(), k.double(), v.double(), 1, 1, 0.4))
    gen = torch.Generator().manual_seed(4)
    x, y, z, g = (torch.randn(2, 6, 9, generator=gen, dtype=torch.float64).requires_grad_(True) for _ in range(4))

    def both(f):
        calls = []
        hooks = [t.register_hook(lambda grad, i=i: calls.append(i)) for i, t in enumerate((x, y, z))]
        out = f(*_shared(name, x, y, z))
        first = torch.autograd.grad(out, (x, y, z), g.float().double(), create_graph=True, allow_unused=True)
        for h in hooks:
            h.remove()
        second = torch.autograd.grad(sum((t ** 3).sum() for t in first if t is not None), (x, y, z), allow_unused=True)
        return first + second, sorted(calls)
    want, want_calls = both(lambda q, k, v: plain(q, k, v, 1, 1, 0.4))
    got, calls = both(lambda q, k, v: OnHost.apply(q, k, v, None, ()))
    assert calls == want_calls
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        # (the Function passes its cotangent on in float32: 2^-24 per pass; the rest is float64)
        assert a is None or rel_err(a, b) <= 4 * 2.0 ** -24, (name, rel_err(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("name", SHARED)
def test_derivatives_of_inputs_that_share_tensors(dev, name):
    """First derivatives with and without create_graph, and second ones, against the formulas in float64 (GRAD, twice that
    for the second, as above); leaves in a table's place too."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 30)
    x, y, z, g = make(2, 2, 2, 12, 12, 40, 40, torch.float32, seed=6)
    table = torch.randn(16, 2, generator=torch.Generator().manual_seed(6))

    def all_of(leaves, g, f, kernels):
        x, y, z, t = leaves
        args = _shared(name, x, y, z)
        out = f(*args, t + x.mean() if name == "all one" else t)
        quick = torch.autograd.grad(out, leaves, g, retain_graph=True, allow_unused=True) if kernels else None
        first = torch.autograd.grad(out, leaves, g, create_graph=True, allow_unused=True)
        second = torch.autograd.grad(sum((d ** 2).sum() for d in first if d is not None), leaves, allow_unused=True)
        return quick, first, second
    ins64 = [t.double().requires_grad_(True) for t in (x, y, z, table)]
    _, want1, want2 = all_of(ins64, g.double(), lambda q, k, v, t: plain(q, k, v, 2, 2, 0.3, None, t, b), False)
    ins = [t.to(dev).requires_grad_(True) for t in (x, y, z, table)]
    quick, got1, got2 = all_of(ins, g.to(dev), lambda q, k, v, t: ops.attention(q, k, v, heads=2, scale=0.3, bias=t, buckets=b), True)
    tap = []
    args = _shared(name, *(t.detach() for t in ins64[:3]))
    out = plain(*args, 2, 2, 0.3, None, ins64[3].detach() + (ins64[0].detach().mean() if name == "all one" else 0.0), b, tap)
    terms, _ = table_terms(tap, out, g.double())  # (a table's gradient of first order: relative to its terms)
    for got, want, bound in ((quick, want1, 1024), (got1, want1, 1024), (got2, want2, 2048)):
        for i, (a, w) in enumerate(zip(got, want)):
            assert (a is None) == (w is None)
            if a is not None:
                size = float(w.detach().norm()) if i < 3 or want is want2 else max(float(w.detach().norm()), terms)
                assert float((a.detach().cpu().double() - w.detach()).norm()) <= bound * 2.0 ** -24 * size, (name, i, rel_err(a, w))


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,kv,dk,dv,tq,tk,train", [(50, 2, 2, 16, 16, 420, 420, True), (9, 8, 4, 32, 32, 1, 20000, False)])
def test_a_sample_is_rounded_alike_in_any_batch(dev, B, heads, kv, dk, dv, tq, tk, train):
    """bfloat16: how P and dS are rounded depends on a sample, not on its neighbours: calls of more than 2^24 pairs (2^20
    for few columns) in small samples keep the bound of small calls above."""
    from eeggan_amd import ops
    assert B * heads * tq * tk > (1 << 24 if tq > 1 else 1 << 20) >= heads * tq * tk
    q, k, v, g = make(B, heads, kv, dk, dv, tq, tk, torch.bfloat16, seed=8)
    leaves = [t.to(dev).requires_grad_(train) for t in (q, k, v)]
    got = ops.attention(*leaves, heads=heads, kv_heads=kv, scale=dk ** -0.5)
    grads = torch.autograd.grad(got, leaves, g.to(dev)) if train else ()
    for b in (0, B - 1):
        ins = [t[b:b + 1].double().requires_grad_(True) for t in (q, k, v)]
        want = plain(*ins, heads, kv, dk ** -0.5)
        pairs = [("out", got[b:b + 1], want.detach())]
        if train:
            pairs += list(zip("qkv", (x[b:b + 1] for x in grads), torch.autograd.grad(want, ins, g[b:b + 1].double())))
        for name, a, w in pairs:
            alone = rel_err(w.to(torch.bfloat16), w)
            assert rel_err(a, w) <= 1.02 * alone + 2.0 ** -13, (b, name, rel_err(a, w), alone)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tq", [64, 2])
def test_infinities_stay_where_they_belong(dev, tq, dtype):
    """An infinite query spoils its own column, an infinite value its own channel (as NaN or infinity): nothing else, and
    nothing of it looks like a number.  The largest values whose sums stay finite (256 Tk |v| < 2^128, and 2^120 twice in a
    score of partners 2^-120) are numbers like any others."""
    from eeggan_amd import ops
    q, k, v, _ = make(2, 1, 1, 16, 32, tq, 70, dtype)
    run = lambda q, k, v: ops.attention(q.to(dev), k.to(dev), v.to(dev), scale=0.25).cpu()  # noqa: E731
    ref = run(q, k, v)
    for inf in (float("inf"), float("-inf")):
        q2, v2 = q.clone(), v.clone()
        q2[0, 3, 1] = inf
        v2[1, 5, 20] = inf
        got = run(q2, k, v2)
        bad = torch.zeros(got.shape, dtype=torch.bool)
        bad[0, :, 1] = True
        bad[1, 5, :] = True
        assert not bool(torch.isfinite(got[bad]).any()) and torch.equal(got[~bad], ref[~bad])
    v2, k2, q2 = v.clone(), k.clone(), q.clone()
    v2[0, 3] *= 2.0 ** 110
    q2[0, 1] *= 2.0 ** 120
    k2[0, 1] *= 2.0 ** -120
    got = run(q2, k2, v2)
    want64 = plain(q.double(), k.double(), v.double(), 1, 1, 0.25)
    want64[0, 3] *= 2.0 ** 110
    for c in range(32):
        assert rel_err(got[:, c], want64[:, c]) <= OUT[dtype] * U[dtype], c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("low", [-1e4, -1e9])
@pytest.mark.parametrize("heads,kv,dk,dv,tq,tk,step,offset", [(2, 2, 8, 32, 300, 300, 1, 0), (2, 1, 64, 64, 200, 330, 1, -60), (1, 1, 16, 16, 2, 700, 1, -680),
                                                              (2, 2, 32, 32, 40, 33, 1, 0), (1, 1, 24, 40, 130, 1100, 2, -1900)])
def test_low_position_entries(dev, heads, kv, dk, dv, tq, tk, step, offset, low, dtype):
    """Entries far below the scores that bar nothing (>= -1e30), as tables are written to keep attention near: everything far
    behind, so that a row's first tiles are all low and ordinary scores follow; or (second head) all entries, which drop out
    of the softmax.  The bias is added to scores of about 8 once, relative to the row's reference: the bounds are those of
    ordinary tables."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40, step=step, offset=offset)
    q, k, v, g, table = make(2, heads, kv, dk, dv, tq, tk, dtype, seed=5, table=b)
    table[7, 0] = low  # (40 steps behind and more)
    if heads > 1:
        table[:, 1] = low
    check(dev, q, k, v, g, heads, kv, table=table, buckets=b, what=(low, tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tq,tk", [(150, 300), (3, 2000), (500, 70)])
def test_scores_that_rise_far(dev, tq, tk, dtype):
    """Scores of -3000 and, some tiles later, ordinary ones: what is left of the row is as exact as without the others."""
    n = 40 if tk < 300 else 130
    q, k, v, g = make(2, 2, 2, 16, 32, tq, tk, dtype, seed=7)
    q[:, ::16] = 8.0
    k[:, ::16, :n] = -1500.0
    k[:, ::16, n:] = 0.0
    check(dev, q, k, v, g, 2, 2, what=(tq, tk))


@pytest.mark.gpu
def test_entries_that_almost_bar_pairs(dev):
    """Entries above -1e30 bar nothing, however low: a head whose entries are all -9e29 weighs keys of equal scores alike,
    one whose entries are -1e30 has none; with and without create_graph."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40)
    q, k, v, g = (t.to(dev) for t in make(2, 2, 2, 8, 16, 50, 33, torch.float32))
    table = torch.full((16, 2), -9e29, device=dev)
    table[:, 1] = -1e30
    v.requires_grad_(True)
    for graph in (False, True):
        out = ops.attention(q, k, v, heads=2, scale=0.0, bias=table, buckets=b)
        gv, = torch.autograd.grad(out, [v], g, create_graph=graph)
        assert rel_err(gv[:, :16], (g[:, :16].double().sum(2, keepdim=True) / 33).expand(2, 16, 33)) <= 256 * 2.0 ** -24, graph
        assert not gv[:, 16:].any() and not out[:, 16:].any()


@pytest.mark.gpu
def test_the_penalty_pass_forms_no_table_gradient(dev, monkeypatch):
    """Where only the inputs' gradients are wanted (ops.input_grad_only: the gradient penalty's first pass) the sums by
    buckets are left out, as weight gradients are; the penalty's own gradients are the same with them."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40)
    gen = torch.Generator().manual_seed(3)
    s, table = (torch.randn(*shape, generator=gen).to(dev).requires_grad_(True) for shape in ((4, 30, 60), (16, 2)))
    counts, call = [], ops.call
    monkeypatch.setattr(ops, "call", lambda name, *a: (counts.append(name), call(name, *a))[1])

    def penalty():
        out = ops.softmax_dim1(ops.relative_bias(s, table, b, heads=2))
        first, = torch.autograd.grad((out ** 2).sum(), [s], create_graph=True)
        return (first ** 2).sum()
    want = torch.autograd.grad(penalty(), [s, table])
    assert counts.count("eeggan_relative_bias_grad") == 2
    counts.clear()
    with ops.input_grad_only():
        value = penalty()
    assert "eeggan_relative_bias_grad" not in counts
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(value, [s, table]), want))


@pytest.mark.gpu
@pytest.mark.parametrize("positions_too", [False, True], ids=["plain", "positions"])
@pytest.mark.parametrize("dtype,dk,dv", [(torch.bfloat16, 16, 32), (torch.bfloat16, 16, 64), (torch.bfloat16, 32, 32), (torch.bfloat16, 32, 64),
                                         (torch.bfloat16, 64, 64), (torch.float32, 8, 32), (torch.float32, 32, 32)])
@pytest.mark.parametrize("B,heads,kv,tq,tk", [(32, 8, 8, 300, 150), (128, 8, 4, 45, 70)])
def test_calls_that_fill_the_chip(dev, B, heads, kv, tq, tk, dtype, dk, dv, positions_too):
    """From 512 workgroups of 256 columns on, where a wave of the forward pass has two blocks of columns: against float64,
    with masks (one sample without keys), with query heads that share a block, with a row's first tiles far below the rest."""
    from eeggan_amd import ops
    assert B * kv * ((heads // kv * tq + 255) // 256) >= 512
    b = ops.RelativeBuckets(16, 40) if positions_too else None
    q, k, v, g, *table = make(B, heads, kv, dk, dv, tq, tk, dtype, seed=11, table=b)
    if b is not None:
        table[0][7, ::2] = -1e9
    mask = torch.rand(B, tk, generator=torch.Generator().manual_seed(1)) < 0.9
    mask[B // 2] = False
    mask[1, :100] = False
    check(dev, q, k, v, g, heads, kv, mask=mask, table=table[0] if table else None, buckets=b, what=(B, tq, tk))


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dk,dv,masked", [(8, 64, 64, False), (2, 24, 40, True)])
def test_samples_of_many_pairs_in_bfloat16(dev, kv, dk, dv, masked):
    """More than 2^24 pairs in a sample: P and dS in one piece, the bounds of which are this file's general ones."""
    heads, tq, tk = 8, 1530, 1477
    assert heads * tq * tk > 1 << 24
    q, k, v, g = make(1, heads, kv, dk, dv, tq, tk, torch.bfloat16, seed=12)
    mask = torch.rand(1, tk, generator=torch.Generator().manual_seed(2)) < 0.95 if masked else None
    check(dev, q, k, v, g, heads, kv, mask=mask, what=(kv, dk, dv))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_that_nobody_wants(dev, dtype, monkeypatch):
    """Any subset of the inputs may want gradients: the bits of the call that wants all.  Where neither keys nor values are
    among them the keys' pass does not run."""
    from eeggan_amd import ops
    b = ops.RelativeBuckets(16, 40)
    base = [t.to(dev) for t in make(2, 2, 1, 16, 24, 300, 5000, dtype, table=b)]
    g = base.pop(3)
    calls, call = [], ops.call
    monkeypatch.setattr(ops, "call", lambda name, *a: (calls.append((name, a)), call(name, *a))[1])

    def grads(which):
        ins = [t.clone().requires_grad_(i in which) for i, t in enumerate(base)]
        out = ops.attention(*ins[:3], heads=2, kv_heads=1, scale=0.25, bias=ins[3], buckets=b)
        calls.clear()
        got = dict(zip(which, torch.autograd.grad(out, [ins[i] for i in which], g)))
        (name, args), = calls
        assert name == "eeggan_attention_bwd" and (args[6] is None) == (args[7] is None) == (not {1, 2} & set(which))
        return got
    want = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (0, 1)):
        got = grads(which)
        assert all(torch.equal(got[i], want[i]) for i in which), which


def test_the_c_entry_point_takes_both_key_gradients_or_none():
    import ctypes
    from eeggan_amd import _lib, ops
    lib = _lib.load()
    a = ops._AttentionDesc()
    a.q, a.k, a.v, a.B, a.H, a.KV, a.Dk, a.Dv, a.Tq, a.Tk, a.scale = 256, 512, 768, 1, 1, 1, 8, 8, 10, 10, 1.0
    a.q_batch, a.q_channel, a.k_batch, a.k_channel, a.v_batch, a.v_channel = 80, 10, 80, 10, 80, 10
    for gk, gv in ((256, None), (None, 256)):
        assert lib.eeggan_attention_bwd(ctypes.byref(a), 256, None, 256, 256, 256, gk, gv, None, 256, 1 << 30, None) != 0
        assert b"null pointer" in lib.eeggan_last_error()
    # (neither: past this check, to the next that fails, the workspace's size)
    assert lib.eeggan_attention_bwd(ctypes.byref(a), 256, None, 256, 256, 256, None, None, None, 256, 0, None) != 0
    assert b"workspace too small" in lib.eeggan_last_error()
