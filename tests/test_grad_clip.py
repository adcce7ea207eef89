"""Global gradient norm, clipping, and the Adam step with a bounded gradient, against float64.

u = 2^-24.  The norm is a sum in double, rounded once: 2 u.  A clipped gradient is g times a rounded multiplier: 2 u of
its value.  The Adam step forms c g, two moments (three roundings each) and the update in float32: moments 8 u relative to
their terms, and the new parameter 2 u of itself plus 32 u of the step (bounded by lr |m| / ((1 - b1^t) root))."""
import functools
import math

import pytest
import torch

U = 2.0 ** -24


def tensors(sizes, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=gen) * scale * (1 + i % 3) for i, n in enumerate(sizes)]


SIZES = [[1], [3], [4, 5, 1023, 1024, 1025], [8191, 8192, 8193, 16385], [100003], [7] * 401, list(range(1, 175))]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm(dev, sizes):
    from eeggan_amd import optim
    gs = tensors(sizes)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(optim.grad_norm([g.to(dev) for g in gs])) - want) <= 2 * U * want


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-10, 1e15, 1e30])
def test_norm_of_extreme_gradients(dev, scale):
    """Squares far outside float32's range."""
    from eeggan_amd import optim
    gs = tensors([1000, 77], scale=scale)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(optim.grad_norm([g.to(dev) for g in gs])) - want) <= 2 * U * want


def parameters(dev, gs, layout=lambda g: g):
    ps = [torch.nn.Parameter(torch.zeros(g.shape, device=dev)) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = layout(g.to(dev))
    return ps


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_clip_in_place(dev, sizes, share):
    from eeggan_amd import optim
    gs = tensors(sizes)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    ps = parameters(dev, gs)
    got = optim.clip_grad_norm_(ps, share * norm)
    assert abs(float(got) - norm) <= 2 * U * norm
    c = min(1.0, share * norm / (norm + 1e-6))
    for p, g in zip(ps, gs):
        if c == 1.0:
            assert torch.equal(p.grad.cpu(), g)
        else:
            assert float((p.grad.cpu().double() - c * g.double()).abs().max()) <= 2 * U * c * float(g.abs().max())


@pytest.mark.gpu
def test_layouts_of_gradients(dev):
    """Odd storage offsets, transposed and strided gradients, one tensor held by two parameters, parameters without one."""
    from eeggan_amd import optim
    gs = tensors([36 * 5, 36 * 5, 36 * 5])
    flat = torch.empty(3 * 36 * 5 + 7, device=dev)
    views = [flat[1 + 183 * i:1 + 183 * i + 180] for i in range(3)]
    flat.fill_(77.0)
    for v, g in zip(views, gs):
        v.copy_(g.to(dev))
    ps = [torch.nn.Parameter(torch.zeros(180, device=dev)) for _ in range(4)]
    for p, v in zip(ps, views):
        p.grad = v
    twin = torch.nn.Parameter(torch.zeros(180, device=dev))
    twin.grad = views[0]
    norm = float(torch.cat([g.double() for g in gs]).norm())
    assert abs(float(optim.clip_grad_norm_(ps + [twin], 0.5 * norm)) - norm) <= 2 * U * norm
    for v, g in zip(views, gs):
        assert float((v.cpu().double() - 0.5 * g.double()).abs().max()) <= 1e-5
    used = torch.zeros_like(flat, dtype=torch.bool)
    for i in range(3):
        used[1 + 183 * i:1 + 183 * i + 180] = True
    assert bool((flat[~used] == 77.0).all())
    t = gs[0].view(36, 5).to(dev)
    p = torch.nn.Parameter(torch.zeros(5, 36, device=dev))
    p.grad = t.t()
    norm = float(gs[0].double().norm())
    optim.clip_grad_norm_(p, 0.1 * norm)
    assert abs(float(p.grad.double().norm()) - 0.1 * norm) <= 1e-5 * norm
    wide = torch.randn(5, 72, device=dev)
    p.grad = wide[:, ::2]
    want = wide[:, ::2].double().norm()
    assert abs(float(optim.clip_grad_norm_([p], 1e-3)) - float(want)) <= 2 * U * float(want)
    assert float(p.grad.norm()) <= 1.001e-3


@pytest.mark.gpu
def test_non_finite_gradients(dev):
    """As torch's: a NaN spoils everything, an infinity leaves zeros (and NaN in its own place); on request an error, with
    the gradients as they were."""
    from eeggan_amd import optim
    for bad in (float("nan"), float("inf")):
        gs = tensors([100, 50])
        gs[1][7] = bad
        ps, qs = parameters(dev, gs), parameters(dev, gs)
        torch.nn.utils.clip_grad_norm_(qs, 1.0)
        norm = optim.clip_grad_norm_(ps, 1.0)
        assert not math.isfinite(float(norm))
        for p, q in zip(ps, qs):
            assert torch.equal(torch.isnan(p.grad), torch.isnan(q.grad))
            assert torch.equal(torch.nan_to_num(p.grad), torch.nan_to_num(q.grad))
        ps = parameters(dev, gs)
        with pytest.raises(RuntimeError, match="total norm"):
            optim.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
        assert torch.equal(ps[0].grad.cpu(), gs[0])


def adam64(p, g, m, v, t, lr, b1, b2, eps):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    step = lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p - step, m, v, step


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [4, 5, 1023, 4096, 4097], [100003], [7] * 401, [3, 20000] * 70],
                         ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("share", [0.25, 4.0])
@pytest.mark.parametrize("betas", [(0.0, 0.99), (0.9, 0.999)])
def test_adam_with_a_bound(dev, sizes, share, betas):
    """Three steps; two parameter groups share one norm; gradients arrive as a sum over two ranks (grad_scale 1/2)."""
    from eeggan_amd import optim
    ps = [torch.nn.Parameter(x.to(dev)) for x in tensors(sizes, 1)]
    cut = len(ps) // 2
    groups = [dict(params=ps[:cut], lr=0.01), dict(params=ps[cut:], lr=0.02)] if cut else [dict(params=ps, lr=0.02)]
    lrs = [0.01 if i < cut else 0.02 for i in range(len(ps))]
    opt = optim.Adam(groups, betas=betas, max_grad_norm=1.0)
    opt.grad_scale = 0.5
    assert opt.grad_norm is None
    ref = [(p.detach().cpu().double(), 0.0, 0.0) for p in ps]
    for t in range(1, 4):
        gs = tensors(sizes, 10 + t)
        norm = 0.5 * math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        opt.max_grad_norm = share * norm
        for p, g in zip(ps, gs):
            p.grad = g.to(dev)
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        c = 0.5 * min(1.0, share * norm / (norm + 1e-6))
        for i, (p, g) in enumerate(zip(ps, gs)):
            assert torch.equal(p.grad.cpu(), g)  # (the gradients stay as they are)
            x, m, v, step = adam64(ref[i][0], c * g.double(), ref[i][1], ref[i][2], t, lrs[i], *betas, 1e-8)
            st = opt.state[p]
            assert float(st["step"]) == t
            got_m, got_v, got_p = st["exp_avg"].cpu().double(), st["exp_avg_sq"].cpu().double(), p.detach().cpu().double()
            terms = c * g.double().abs() + torch.as_tensor(m).abs()
            assert bool(((got_m - m).abs() <= 8 * t * U * terms + 1e-38).all())
            assert bool(((got_v - v).abs() <= 8 * t * U * v + 1e-38).all())
            # (a step is m / sqrt(v): the moments' relative errors, 8 t u of terms / |m| and half of 8 t u, reach it)
            bound = 2 * t * U * x.abs() + (32 + 16 * t) * U * (step.abs() + lrs[i] * terms / ((1 - betas[0] ** t) * (v / (1 - betas[1] ** t)).sqrt() + 1e-30))
            assert bool(((got_p - x).abs() <= bound).all()), float(((got_p - x).abs() / bound).max())
            ref[i] = (got_p, got_m, got_v)


@pytest.mark.gpu
def test_bound_that_never_acts_equals_no_bound(dev):
    """A bound far above the norm: the plain step's parameters up to the rounding of 1 - beta (float32 there, double here:
    2^-24 / 0.01 of the second moment)."""
    from eeggan_amd import optim
    sizes = [1000, 33]
    runs = []
    for bound in (None, 1e9):
        ps = [torch.nn.Parameter(x.to(dev)) for x in tensors(sizes, 1)]
        opt = optim.Adam(ps, lr=0.01, betas=(0.0, 0.99), max_grad_norm=bound)
        for t in range(3):
            for p, g in zip(ps, tensors(sizes, 5 + t)):
                p.grad = g.to(dev)
            opt.step()
        runs.append(ps)
    for a, b in zip(*runs):
        assert float((a - b).abs().max()) <= 3 * 0.01 * 100 * U * 4 + 4 * U * 5


@pytest.mark.gpu
def test_clipped_step_in_a_captured_graph(dev):
    """Replays follow the gradients that the buffers then hold; the norm is rewritten by every replay."""
    from eeggan_amd import optim
    from eeggan_amd.graphs import GraphedCall
    sizes = [5000, 12, 8193]
    gs = [g.to(dev) for g in tensors(sizes)]

    def build():
        ps = [torch.nn.Parameter(x.to(dev)) for x in tensors(sizes, 1)]
        for p, g in zip(ps, gs):
            p.grad = g
        return ps, optim.Adam(ps, lr=0.01, betas=(0.0, 0.99), max_grad_norm=2.0)
    (pa, oa), (pb, ob) = build(), build()
    call = GraphedCall(lambda: oa.step(), warmup=1)
    for _ in range(1):
        ob.step()
    for turn in range(4):
        for g in gs:
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(turn)) * (turn + 0.01))
        call()
        ob.step()
        assert torch.equal(oa.grad_norm, ob.grad_norm)
        assert all(torch.equal(a, b) for a, b in zip(pa, pb))


@pytest.mark.gpu
def test_trainers_follow_each_other_with_a_bound(dev, monkeypatch):
    """Eager, graphed, and data-parallel (bucketed: one bucket, the norm spans all gradients) trainers with a bound that
    acts in every step."""
    import torch.distributed as dist
    import test_e2e_gpu as E
    from eeggan_amd import layers, optim
    from eeggan_amd.graphs import GraphedTrainer
    from eeggan_amd.parallel import DataParallelStep
    from eeggan_amd.trainer import Trainer
    unbounded = optim.Adam
    layers.set_drop_mode("device")
    own_group = not dist.is_initialized()
    if own_group:
        dist.init_process_group("nccl", init_method="tcp://127.0.0.1:29518", rank=0, world_size=1,
                                device_id=torch.device(dev))
    try:
        free = E._two_steps(dev, Trainer, lr=0.0)
        monkeypatch.setattr(optim, "Adam", functools.partial(unbounded, max_grad_norm=0.05))
        sync = lambda: DataParallelStep(always_bucket=True)  # noqa: E731
        base = E._two_steps(dev, Trainer, lr=0.0), E._two_steps(dev, Trainer)
        graphed = E._two_steps(dev, GraphedTrainer, lr=0.0), E._two_steps(dev, GraphedTrainer)
        parallel = E._two_steps(dev, GraphedTrainer, sync, lr=0.0), E._two_steps(dev, GraphedTrainer, sync)
    finally:
        layers.set_drop_mode("numpy")
        if own_group:
            dist.destroy_process_group()
    E._same_trajectory(base, graphed, "graph replay, bounded gradients")
    E._same_trajectory(base, parallel, "data-parallel graphs, bounded gradients")
    for net in ("G.", "D."):  # beta1 = 0: the first moment is the last gradient
        m = torch.cat([v.flatten() for k, v in base[0].items() if k.startswith(net) and k.endswith(".m")])
        w = torch.cat([v.flatten() for k, v in free.items() if k.startswith(net) and k.endswith(".m")])
        assert float(w.norm()) > 0.05
        assert abs(float(m.norm()) - 0.05) < 1e-5


# ------------------------------------------------------------------------------------------------ without a GPU
def test_refusals():
    from eeggan_amd import optim
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            optim.Adam([p], max_grad_norm=bad)
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], bad)
    with pytest.raises(NotImplementedError):
        optim.clip_grad_norm_([p], 1.0, norm_type=1.0)
    with pytest.raises(RuntimeError, match="device tensors"):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="device tensors"):
        optim.grad_norm([p.grad])


def test_c_entry_points_refuse_before_any_launch():
    from eeggan_amd import _lib, optim
    lib = _lib.load()
    good = optim.build_table([(None, 256, None, None, None, 10)])
    size = lib.eeggan_grad_norm_workspace(good, 1)
    assert size >= 8 + 8
    assert lib.eeggan_grad_norm(good, 1, 1.0, 1.0, 256, 256, size - 1, None) != 0 and b"small" in lib.eeggan_last_error()
    assert lib.eeggan_grad_norm(good, 1, 1.0, 0.0, 256, 256, size, None) != 0 and b"positive" in lib.eeggan_last_error()
    assert lib.eeggan_grad_norm(good, 1, 1.0, float("nan"), 256, 256, size, None) != 0
    assert lib.eeggan_grad_norm(good, 1, 1.0, 1.0, None, 256, size, None) != 0
    assert lib.eeggan_grad_norm(good, 1, 1.0, 1.0, 256, 260, size, None) != 0 and b"misaligned" in lib.eeggan_last_error()
    assert lib.eeggan_grad_norm(good, 0, 1.0, 1.0, 256, 256, size, None) != 0
    for row in ((None, None, None, None, None, 10), (None, 256, None, None, None, 0), (None, 258, None, None, None, 5),
                (None, 256, None, None, None, 1 << 50)):
        table = optim.build_table([row])
        assert lib.eeggan_grad_norm_workspace(table, 1) == 0
        assert lib.eeggan_grad_scale(table, 1, 256, None) != 0 and lib.eeggan_last_error()
    assert lib.eeggan_grad_scale(good, 1, None, None) != 0
    assert lib.eeggan_adam_step_clipped(good, 1, 1e-3, 0.0, 0.99, 1e-8, 256, 256, 64, None) != 0
    assert b"state pointers" in lib.eeggan_last_error()
    full = optim.build_table([(256, 256, 256, 256, 256, 10)])
    assert lib.eeggan_adam_step_clipped(full, 1, 1e-3, 1.0, 0.99, 1e-8, 256, 256, 64, None) != 0
    assert lib.eeggan_adam_step_clipped(full, 1, 1e-3, 0.0, 0.99, 1e-8, 256, 256, 4, None) != 0


@pytest.mark.gpu
def test_parameters_without_elements(dev):
    """An empty tensor among the parameters has no part in the norm and no step."""
    from eeggan_amd import optim
    full, empty = torch.nn.Parameter(torch.ones(5, device=dev)), torch.nn.Parameter(torch.zeros(0, 3, device=dev))
    for p in (full, empty):
        p.grad = torch.ones_like(p)
    opt = optim.Adam([dict(params=[empty]), dict(params=[full])], lr=0.5, betas=(0.0, 0.99), max_grad_norm=0.1)
    opt.step()
    assert abs(float(opt.grad_norm) - 5 ** 0.5) < 1e-6 and float(full.detach().max()) < 1.0
    assert float(optim.clip_grad_norm_([empty], 1.0)) == 0.0


def test_copies_and_pickles_keep_the_bound():
    import copy
    import pickle
    from eeggan_amd import optim
    p = torch.nn.Parameter(torch.zeros(3))
    opt = optim.Adam([p], lr=0.25, max_grad_norm=0.75)
    opt.grad_scale = 0.5
    opt._norm = torch.ones(2)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt)), copy.copy(opt)):
        assert (other.max_grad_norm, other.grad_scale, other.grad_norm) == (0.75, 0.5, None)
        assert other.param_groups[0]["lr"] == 0.25
    assert copy.deepcopy(optim.Adam([p])).max_grad_norm is None


@pytest.mark.gpu
def test_a_copied_optimizer_steps_alike(dev):
    import copy
    from eeggan_amd import optim
    p = torch.nn.Parameter(torch.ones(700, device=dev))
    opt = optim.Adam([p], lr=0.1, betas=(0.5, 0.99), max_grad_norm=0.5)
    opt.grad_scale = 0.25
    p.grad = torch.linspace(-3, 5, 700, device=dev)
    opt.step()
    both = copy.deepcopy([p, opt])
    both[0].grad = p.grad.clone()
    opt.step()
    both[1].step()
    assert torch.equal(p, both[0]) and torch.equal(opt.grad_norm, both[1].grad_norm) and both[1].grad_norm is not None


@pytest.mark.parametrize("bound", [None, 1.0])
def test_gradients_that_do_not_fit_are_refused(bound):
    """Gradients handed to the step by hand (``p.grad`` is checked by torch): the kernel reads as many as the parameter has."""
    from eeggan_amd import optim
    p = torch.nn.Parameter(torch.zeros(5, 2))
    opt = optim.Adam([p], max_grad_norm=bound)
    for g in (torch.zeros(9), torch.zeros(10, dtype=torch.bfloat16), torch.zeros(10, device="meta")):
        with pytest.raises(RuntimeError, match="for a parameter of 10, torch.float32 on cpu"):
            opt.step(grads={p: g})
    with pytest.raises(RuntimeError, match="contiguous float32 device tensors"):
        opt.step(grads={p: torch.zeros(10)})


@pytest.mark.gpu
def test_more_elements_than_one_pass_of_the_grid(dev):
    """Past 16.8 M elements the norm's workgroups walk over several chunks: norm, clipping and the bounded step."""
    from eeggan_amd import optim
    sizes = [20_000_003, 5, 9_000_001]
    gen = torch.Generator(device=dev).manual_seed(1)
    gs = [torch.randn(n, device=dev, generator=gen) * (1 + i) for i, n in enumerate(sizes)]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(optim.grad_norm(gs)) - norm) <= 2 * U * norm
    ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    opt = optim.Adam(ps, lr=0.5, betas=(0.0, 0.99), max_grad_norm=0.25 * norm)
    opt.step()
    c = 0.25 * norm / (norm + 1e-6)
    for p, g in zip(ps, gs):
        # (the first step with beta1 = 0: m = c g, v / (1 - 0.99) = m^2, so that every element moves by lr)
        assert float((opt.state[p]["exp_avg"].double() - c * g.double()).abs().max()) <= 3 * U * c * float(g.abs().max())
        seen = g.abs() > 1e-3
        assert float((p.detach().double().abs()[seen] - 0.5).abs().max()) <= 0.5 * (64 * U + 1e-8 / (c * 1e-3))
    assert abs(float(optim.clip_grad_norm_(ps, 0.25 * norm)) - norm) <= 2 * U * norm
    for p, g in zip(ps, gs):
        assert float((p.grad.double() - c * g.double()).abs().max()) <= 2 * U * c * float(g.abs().max())
