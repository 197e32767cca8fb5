"""Norms over many tensors and clipping by the global norm.

Tolerances: squares are summed in 64 bits (their error is far below fp32's),
so a norm is off by its rounding to fp32, 2^-24, and its square root's, below
that: 2^-23. The factor has three fp32 roundings after the norm's, the product
one more: 5 * 2^-24, and half a step of the gradient's type.
"""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from photon_amd.ops.clip import clip_grad_norm_, clip_grads_, tensor_norms

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def exact(grads, max_norm=None):
    s = [math.fsum((g.detach().cpu().double() ** 2).reshape(-1).tolist()) for g in grads]
    total = math.sqrt(math.fsum(s))
    c = 1.0 if max_norm is None else min(1.0, max_norm / (total + 1e-6))
    return total, [math.sqrt(x) for x in s], [g.detach().cpu().double() * c for g in grads], c


def assert_clipped(grads, before, total, norms, max_norm):
    want_total, want_norms, want, c = exact(before, max_norm)
    assert abs(float(total) - want_total) <= 2.0**-23 * want_total + 1e-300
    assert norms.shape == (len(before),)
    for n, w in zip(norms.tolist(), want_norms):
        assert abs(n - w) <= 2.0**-23 * w + 1e-300
    for g, b, w in zip(grads, before, want):
        assert g.dtype == b.dtype
        if c == 1.0:
            assert torch.equal(g, b)
            continue
        room = (5 * 2.0**-24 + torch.finfo(g.dtype).eps / 2 * (1 + 2.0**-20)) * w.abs()
        err = (g.detach().cpu().double() - w).abs()
        assert bool((err <= room + 1e-38).all())


SHAPES = [(3, 5), (7,), (1,), (0,), (1000, 33), (2, 3, 4), (16385,), (70001,)]


def make(dev, dtypes, shapes=SHAPES, std=1.0, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(dev, dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


# -- CPU --------------------------------------------------------------------
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6])
def test_plain_path(max_norm):
    grads = make("cpu", [F32, BF16], SHAPES[:6])
    before = [g.clone() for g in grads]
    total, norms = clip_grads_(grads, max_norm)
    assert_clipped(grads, before, total, norms, max_norm)
    t2, n2 = tensor_norms(before)
    assert torch.equal(t2, total) and torch.equal(n2, norms)


def test_64_bit_gradients_stay_64_bit():
    g = torch.randn(100, dtype=torch.float64)
    want = g * float((0.5 / (g.norm() + 1e-6)))
    clip_grads_([g], 0.5)
    # the factor is rounded to fp32, the same for all: the ratios are exact
    ratio = g / want
    assert (ratio / ratio[0] - 1).abs().max() <= 2.0**-50
    assert abs(ratio[0] - 1) <= 4 * 2.0**-24


def test_refusals_and_empty():
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_([torch.ones(2)], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_([torch.ones(2)], float("nan"))
    assert float(clip_grads_([], 1.0)[0]) == 0.0
    assert float(tensor_norms([])[0]) == 0.0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0


def test_parameter_listed_twice_counts_once():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.full((4,), 3.0)
    assert float(clip_grad_norm_([p, p], 3.0)) == 6.0
    assert torch.allclose(p.grad, torch.full((4,), 1.5))


def refused_gradients_stay(dev):
    """One gradient made in inference mode: outside of it none is scaled."""
    plain = [torch.full((9,), 3.0, device=dev), torch.full((4, 6), 2.0, device=dev)[:, ::2]]
    with torch.inference_mode():
        made = torch.full((5,), 4.0, device=dev)
    grads = [plain[0], made, plain[1]]
    with pytest.raises(RuntimeError, match="gradient was made in inference mode"):
        clip_grads_(grads, 0.5)
    assert all(bool((g == x).all()) for g, x in zip(grads, (3.0, 4.0, 2.0)))
    before = [g.clone() for g in grads]
    with torch.inference_mode():
        total, norms = clip_grads_([made], 0.5)
    assert_clipped([made], before[1:2], total, norms, 0.5)


def test_refused_gradients_stay():
    refused_gradients_stay("cpu")


def forward_mode_is_refused(dev):
    """The factor depends on every gradient: a tangent scaled by it, or left
    as it is, would be wrong."""
    g, other = torch.full((5,), 2.0, device=dev), torch.full((3,), 2.0, device=dev)
    with fwAD.dual_level():
        dual = fwAD.make_dual(g, torch.ones_like(g))
        with pytest.raises(NotImplementedError, match="clip_grads: forward-mode"):
            clip_grads_([other, dual], 0.1)
    assert bool((g == 2.0).all()) and bool((other == 2.0).all())


def test_forward_mode_is_refused():
    forward_mode_is_refused("cpu")


def test_optimizer_monitor_matches_the_loop():
    from types import SimpleNamespace

    from photon_amd.train.monitors import OptimizerMonitor

    ps = [torch.nn.Parameter(torch.randn(5, 3)), torch.nn.Parameter(torch.randn(4))]
    opt = torch.optim.AdamW(ps)
    ps[0].grad, ps[1].grad = torch.randn(5, 3), torch.randn(4)
    opt.step()
    model = torch.nn.Module()
    model.a, model.b = ps
    tr = SimpleNamespace(optimizer=opt, model=model, timestamp=SimpleNamespace(batch=20))
    got = OptimizerMonitor(interval="10ba", only_global=True).batch_end(tr, 0.0)
    want_g = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
    want_m = math.sqrt(sum(float(opt.state[p]["exp_avg"].double().square().sum()) for p in ps))
    assert set(got) == {"optimizer/l2_norm_first_moment", "optimizer/l2_norm_grad"}
    assert abs(got["optimizer/l2_norm_grad"] - want_g) <= 2.0**-23 * want_g
    assert abs(got["optimizer/l2_norm_first_moment"] - want_m) <= 2.0**-23 * want_m
    each = OptimizerMonitor(only_global=False).batch_end(tr, 0.0)
    assert abs(each["optimizer/l2_norm_grad/a"] - float(ps[0].grad.norm())) <= 1e-6 * float(ps[0].grad.norm())
    assert "optimizer/l2_norm_first_moment/b" in each
    tr.timestamp.batch = 21
    assert OptimizerMonitor(interval="10ba").batch_end(tr, 0.0) == {}


def monitor_takes_any_tensor(devices):
    """Half and double gradients and moments, sparse ones, parameters on
    several devices: each norm within fp32's rounding, as a loop over them gave."""
    from types import SimpleNamespace

    from photon_amd.train.monitors import OptimizerMonitor

    g = torch.Generator().manual_seed(4)
    model, opt = torch.nn.Module(), SimpleNamespace(state={}, param_groups=[])
    dtypes = [F32, torch.float16, BF16, torch.float64]
    for i in range(9):
        p = torch.nn.Parameter(torch.randn(7, i + 1, generator=g).to(devices[i % len(devices)], dtypes[i % 4]))
        p.grad = torch.randn(7, i + 1, generator=g).to(p)
        opt.state[p] = {"exp_avg": torch.randn(7, i + 1, generator=g).to(p).t()}
        if i == 8:
            p.grad = p.grad.to_sparse()
        opt.param_groups.append({"params": [p]})
        model.register_parameter(f"p{i}", p)
    tr = SimpleNamespace(optimizer=opt, model=model, timestamp=SimpleNamespace(batch=20))
    got = OptimizerMonitor(only_global=False).batch_end(tr, 0.0)
    for key, pick in (("optimizer/l2_norm_grad", lambda p: p.grad.to_dense()),
                      ("optimizer/l2_norm_first_moment", lambda p: opt.state[p]["exp_avg"])):
        each = {n: float(pick(p).detach().double().square().sum()) for n, p in model.named_parameters()}
        for n, s in each.items():
            assert abs(got[f"{key}/{n}"] - math.sqrt(s)) <= 2.0**-23 * math.sqrt(s)
        # each norm is rounded to fp32 before its square joins the others
        want = math.sqrt(sum(each.values()))
        assert abs(got[key] - want) <= 2.0**-22 * want
    assert len(got) == 20


def test_optimizer_monitor_takes_any_tensor():
    monitor_takes_any_tensor(["cpu"])


# -- GPU --------------------------------------------------------------------
@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@gpu
@pytest.mark.parametrize("dtypes", [[F32], [BF16], [BF16, F32], [F32, F32, BF16]])
@pytest.mark.parametrize("max_norm", [0.0, 0.01, 3.0, 1e9])
def test_clip(dev, dtypes, max_norm):
    grads = make(dev, dtypes)
    before = [g.clone() for g in grads]
    total, norms = clip_grads_(grads, max_norm)
    assert_clipped(grads, before, total, norms, max_norm)


@gpu
@pytest.mark.parametrize("count", [1, 159, 160, 161, 500])
def test_many_tensors(dev, count):
    shapes = [(1 + 37 * i % 501,) for i in range(count)]
    grads = make(dev, [F32, BF16], shapes)
    before = [g.clone() for g in grads]
    total, norms = clip_grads_(grads, 0.5)
    assert_clipped(grads, before, total, norms, 0.5)


@gpu
def test_pieces_that_begin_anywhere(dev):
    """Views into one buffer, odd lengths, every alignment; the gaps between
    and behind them stay as they are."""
    for t in (F32, BF16):
        buf = torch.randn(400_000, device=dev).to(t)
        old = buf.clone()
        lens = [1, 2, 3, 5, 8, 13, 1021, 4099, 32768, 32769, 131_073]
        views, at = [], 1
        for n in lens:
            views.append(buf[at:at + n])
            at += n + 1  # one element between
        before = [v.clone() for v in views]
        total, norms = clip_grads_(views, 1.0)
        assert_clipped(views, before, total, norms, 1.0)
        mask = torch.ones(400_000, dtype=torch.bool, device=dev)
        at = 1
        for n in lens:
            mask[at:at + n] = False
            at += n + 1
        assert torch.equal(buf[mask], old[mask])


@gpu
def test_in_place_writes_are_known_to_autograd(dev):
    """A gradient that a later backward still needs is refused after it."""
    x = torch.randn(50, device=dev, requires_grad=True)
    y = x.exp()  # its result is saved for the backward
    clip_grads_([y.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@gpu
def test_strided_gradients(dev):
    a = torch.randn(64, 48, device=dev)
    b = torch.randn(33, 40, device=dev).to(BF16)
    rest_a, rest_b = a.clone(), b.clone()
    grads = [a.t(), b[:, ::2], b[:, 1::4]]  # dense and transposed, strided
    before = [g.clone() for g in grads]
    total, norms = clip_grads_(grads, 1.0)
    assert_clipped(grads, before, total, norms, 1.0)
    assert torch.equal(b[:, 3::4], rest_b[:, 3::4])
    assert not torch.equal(a, rest_a)


@gpu
def test_gpu_refused_gradients_stay(dev):
    refused_gradients_stay(dev)


@gpu
def test_gpu_forward_mode_is_refused(dev):
    forward_mode_is_refused(dev)


@gpu
def test_gpu_optimizer_monitor_takes_any_tensor(dev):
    monitor_takes_any_tensor([dev])
    monitor_takes_any_tensor(["cpu", dev])
    monitor_takes_any_tensor([dev, dev, "cpu"])


@gpu
def test_strided_gradients_that_share_memory(dev):
    """Named twice, from one element on, or out of a dense one; views that
    only lie between each other are taken (test_strided_gradients)."""
    a = torch.randn(8, 12, device=dev)
    old = a.clone()
    for bad in ([a[:, ::2], a[:, ::2]], [a[:, ::2], a[:, ::3]], [a, a[:, 1::2]], [a[2:, 3::4], a]):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grads_(bad, 0.1)
        assert torch.equal(a, old)
    parts = [a[:, 1::2], a[0, 4:5], a[:, 2:4:2]]
    before = [g.clone() for g in parts]
    total, norms = clip_grads_(parts, 0.5)
    assert_clipped(parts, before, total, norms, 0.5)


@gpu
def test_gpu_refusals(dev):
    g = torch.randn(100, device=dev)
    for bad, match in (([g, g], "share memory"), ([g[:60], g[50:]], "share memory"),
                       ([g, g.cpu()], "one GPU"), ([g.half()], "unsupported dtype"),
                       ([torch.ones(1, device=dev).expand(8)], "with itself")):
        old = g.clone()
        with pytest.raises(RuntimeError, match=match):
            clip_grads_(bad, 0.1)
        assert torch.equal(g, old)
    assert abs(float(tensor_norms([g, g])[0]) - math.sqrt(2) * float(g.double().norm())) <= 1e-5


@gpu
@pytest.mark.parametrize("std", [1e-30, 1e-22, 1e18])
def test_squares_outside_fp32(dev, std):
    grads = make(dev, [F32], std=std)
    total, norms = tensor_norms(grads)
    want, each, _, _ = exact(grads)
    assert abs(float(total) - want) <= 2.0**-23 * want
    for n, w in zip(norms.tolist(), each):
        assert abs(n - w) <= 2.0**-23 * w


@gpu
def test_not_finite(dev):
    for bad in (float("nan"), float("inf")):
        grads = make(dev, [F32, BF16])
        grads[4][500, 7] = bad
        before = [g.clone() for g in grads]
        total, norms = clip_grads_(grads, 1.0)
        assert not math.isfinite(float(total))
        assert int((~norms.isfinite()).sum()) == 1 and not math.isfinite(float(norms[4]))
        scale = torch.tensor(1.0, device=dev) / (total + 1e-6)
        for g, b in zip(grads, before):
            assert torch.equal(torch.nan_to_num(g, 7.0), torch.nan_to_num((b.float() * scale).to(b.dtype), 7.0))


@gpu
def test_same_bits_and_graph_replays(dev):
    grads = make(dev, [F32, BF16])
    src = [make(dev, [F32, BF16], std=s, seed=i) for i, s in enumerate((0.01, 2.0, 1e-4, 30.0))]
    graph = torch.cuda.CUDAGraph()
    clip_grads_(grads, 1.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        total, norms = clip_grads_(grads, 1.0)
    for s in src:
        for g, x in zip(grads, s):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = [x.clone() for x in s]
        t2, n2 = clip_grads_(eager, 1.0)
        assert torch.equal(total, t2) and torch.equal(norms, n2)
        assert all(torch.equal(a, b) for a, b in zip(grads, eager))


@gpu
def test_more_than_2_31_elements(dev):
    """A tensor whose element offsets pass 32 bits."""
    n = (1 << 31) + 4099
    g = torch.full((n,), 2.0**-10, dtype=BF16, device=dev)
    g[-1] = 8.0
    total, norms = clip_grads_([g], 4.0)
    want = math.sqrt((n - 1) * 2.0**-20 + 64.0)
    assert abs(float(total) - want) <= 2.0**-23 * want
    c = 4.0 / want
    for i in (0, 12345, (1 << 31) - 1, 1 << 31, n - 2):
        assert abs(float(g[i]) - c * 2.0**-10) <= 2.0**-8 * c * 2.0**-10
    assert abs(float(g[-1]) - 8 * c) <= 2.0**-8 * 8 * c
