"""Embedding lookup with scaling and its sorted gradient.

Tolerances: the lookup does one fp32 product and one rounding, as torch's
``(rows.float() * scale).to(dtype)`` does: equal bits. A gradient row is an
fp32 sum of m terms times the scale: m + 1 roundings of at most 2^-24 of the
sum of the magnitudes, and half a step of the table's type.
"""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from photon_amd.ops.embedding import FusedEmbedding, embedding

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def exact_grad(ids, dy, V, scale):
    """Gradient in 64 bits, the sum of magnitudes and the terms of each row."""
    ids, dy = ids.reshape(-1).cpu(), dy.reshape(-1, dy.shape[-1]).cpu().double()
    ok = (ids >= 0) & (ids < V)
    ids, dy = ids[ok].long(), dy[ok]
    g = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, ids, dy)
    mag = torch.zeros_like(g).index_add_(0, ids, dy.abs())
    return g * scale, mag * abs(scale), torch.bincount(ids, minlength=V).view(-1, 1)


def assert_grad(got, ids, dy, scale):
    want, mag, terms = exact_grad(ids, dy, got.shape[0], scale)
    room = (terms + 1) * 2.0**-24 * mag
    room = room + torch.finfo(got.dtype).eps / 2 * (want.abs() + room) + 1e-300
    err = (got.cpu().double() - want).abs()
    assert bool((err <= room).all()), float((err / room).max())


# -- CPU --------------------------------------------------------------------
@pytest.mark.parametrize("table_dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16)])
def test_plain_path(table_dtype, out_dtype):
    w = torch.randn(37, 10).to(table_dtype).requires_grad_()
    ids = torch.randint(0, 37, (3, 5))
    y = embedding(ids, w, 3.0, out_dtype)
    assert y.dtype == out_dtype
    assert torch.equal(y, (w[ids].float() * 3.0).to(out_dtype))
    dy = torch.randn(3, 5, 10).to(out_dtype)
    (g,) = torch.autograd.grad(y, w, dy)
    # torch adds these in the table's type: each addition rounds there
    want, mag, terms = exact_grad(ids, dy, 37, 3.0)
    eps = torch.finfo(table_dtype).eps / 2
    assert bool(((g.double() - want).abs() <= (terms + 2) * eps * mag + 1e-300).all())


def test_plain_path_keeps_64_bits():
    w = torch.randn(5, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([4, 0, 4])
    y = embedding(ids, w, 1.0 / 3.0)
    assert y.dtype == torch.float64 and torch.equal(y, w[ids] * (1.0 / 3.0))
    assert torch.autograd.gradcheck(lambda t: embedding(ids, t, 1.0 / 3.0), (w,))


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_plain_gradient_of_a_bf16_table_sums_in_32_bits(scale, out_dtype):
    """Whole numbers, the sums below 2^24: exact until the one rounding. A sum
    of 1000 ones that rounds to bf16 at each step stops at 256."""
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 4, (4000,), generator=g)
    ids[:1000] = 3
    dy = torch.randint(-3, 5, (4000, 6), generator=g).to(out_dtype)
    dy[ids == 3] = 1.0
    w = torch.randn(4, 6, generator=g).to(BF16).requires_grad_()
    y = embedding(ids, w, scale, out_dtype)
    assert torch.equal(y, (w[ids].float() * scale).to(out_dtype))
    (got,) = torch.autograd.grad(y, w, dy)
    want, _, _ = exact_grad(ids, dy, 4, scale)
    assert torch.equal(got, want.to(BF16)) and float(want[3, 0]) >= 1000 * scale


def test_refusals():
    w = torch.randn(4, 8)
    with pytest.raises(TypeError, match="int64 or int32"):
        embedding(torch.zeros(2), w)
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        embedding(torch.zeros(2, dtype=torch.long), w[0])
    with pytest.raises(IndexError):
        embedding(torch.tensor([4]), w)
    for kw in ({"padding_idx": 0}, {"max_norm": 1.0}, {"sparse": True},
               {"scale_grad_by_freq": True}):
        with pytest.raises(ValueError, match="FusedEmbedding"):
            FusedEmbedding(4, 8, **kw)


def test_module_matches_nn_embedding_on_cpu():
    torch.manual_seed(1)
    a = FusedEmbedding(11, 6)
    b = torch.nn.Embedding(11, 6)
    b.load_state_dict(a.state_dict())
    ids = torch.randint(0, 11, (2, 7))
    assert torch.equal(a(ids), b(ids))
    with torch.autocast("cpu", dtype=BF16):
        assert torch.equal(a(ids), b(ids).to(BF16))
    s = FusedEmbedding(11, 6, scale=2.5, impl="torch")
    s.load_state_dict(a.state_dict())
    assert torch.equal(s(ids), b(ids) * 2.5)


def module_takes_what_nn_embedding_takes(dev):
    """Transforms, forward mode, tracing, tables that are not rows of one
    buffer: the module's results are nn.Embedding's times the scale."""
    torch.manual_seed(2)
    a, b = FusedEmbedding(11, 6, scale=2.0).to(dev), torch.nn.Embedding(11, 6).to(dev)
    b.load_state_dict(a.state_dict())
    w = a.weight.detach()
    ids = torch.tensor([[3, 0, 3], [10, 7, 1]], device=dev)

    def apply(m, table):
        return torch.func.functional_call(m, {"weight": table}, (ids,))

    tables = torch.stack([w, w + 1.0])
    assert torch.equal(torch.func.vmap(lambda t: apply(a, t))(tables),
                       2.0 * torch.func.vmap(lambda t: apply(b, t))(tables))
    grad = torch.func.grad(lambda t: apply(a, t).square().sum())(w)
    assert torch.equal(grad, 4.0 * torch.func.grad(lambda t: apply(b, t).square().sum())(w))
    y, t = torch.func.jvp(lambda t: apply(a, t), (w,), (w.cos(),))
    assert torch.equal(y, 2.0 * w[ids]) and torch.equal(t, 2.0 * w.cos()[ids])
    with fwAD.dual_level():
        y, t = fwAD.unpack_dual(apply(a, fwAD.make_dual(w, w.cos())))
        assert torch.equal(y, 2.0 * w[ids]) and torch.equal(t, 2.0 * w.cos()[ids])
    other = ids.flip(0)
    assert torch.equal(torch.jit.trace(a, (ids,))(other), 2.0 * w[other])
    table = w.t().contiguous().t().requires_grad_()  # columns, not rows, in one piece
    y = apply(a, table)
    assert torch.equal(y, 2.0 * w[ids])
    assert torch.equal(torch.autograd.grad(y.square().sum(), table)[0], grad)
    assert torch.equal(a(ids), 2.0 * w[ids])


def test_module_takes_what_nn_embedding_takes():
    module_takes_what_nn_embedding_takes("cpu")


# -- GPU --------------------------------------------------------------------
@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def make(dev, n, V, D, table_dtype, out_dtype, seed=0, skew=True, id_dtype=torch.long):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn(V, D, generator=g, device=dev).to(table_dtype).requires_grad_()
    u = torch.rand(n, generator=g, device=dev)
    ids = (torch.exp(u * math.log(V)).long() - 1 if skew else (u * V).long()).clamp(0, V - 1)
    dy = torch.randn(n, D, generator=g, device=dev).to(out_dtype)
    return w, ids.to(id_dtype), dy


@gpu
@pytest.mark.parametrize("table_dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("n,V,D", [
    (1, 1, 1), (1, 300, 8), (2, 70000, 4), (31, 50, 12), (32, 50, 256),
    (33, 255, 260), (64, 256, 257), (65, 257, 7), (1000, 50368, 768),
    (1025, 65536, 64), (5000, 3, 320), (8191, 16777217, 2), (40000, 512, 100),
])
def test_lookup_and_gradient(dev, table_dtype, out_dtype, n, V, D):
    w, ids, dy = make(dev, n, V, D, table_dtype, out_dtype)
    scale = 0.37
    y = embedding(ids, w, scale, out_dtype)
    assert torch.equal(y, (w.detach()[ids].float() * scale).to(out_dtype))
    (g,) = torch.autograd.grad(y, w, dy)
    assert g.dtype == table_dtype and g.shape == w.shape
    assert_grad(g, ids, dy, scale)


@gpu
def test_many_ids_over_all_sort_blocks(dev):
    """More than 128 tiles of 1024 positions, int32 ids, one token in half of them."""
    w, ids, dy = make(dev, 200_003, 50368, 16, F32, BF16, id_dtype=torch.int32)
    ids[::2] = 4242
    y = embedding(ids, w, 1.0, BF16)
    (g,) = torch.autograd.grad(y, w, dy)
    assert_grad(g, ids, dy, 1.0)


@gpu
@pytest.mark.parametrize("table_dtype,dy_dtype", [(F32, BF16), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("n,V,D,top", [
    (200_003, 50368, 16, 0.5), (40000, 512, 100, 0.3), (1_000_003, 300, 4, 0.99),
    (65536, 50368, 768, 0.0), (16384, 70000, 40, 0.9), (270_000, 2, 1, 0.5),
    (1_100_000, 50257, 8, 1.0),
])
def test_frequent_tokens_are_summed_exactly(dev, table_dtype, dy_dtype, n, V, D, top):
    """Whole numbers up to 8 and a scale of a power of two: every fp32 sum is
    below 2^24 and exact in any order, so a partial sum that is lost or counted
    twice shows however many terms there are. A bf16 table rounds once."""
    w, ids, _ = make(dev, n, V, D, table_dtype, dy_dtype)
    g = torch.Generator(device=dev).manual_seed(n)
    ids[torch.rand(n, generator=g, device=dev) < top] = V - 1
    dy = torch.randint(-8, 9, (n, D), generator=g, device=dev).to(dy_dtype)
    (got,) = torch.autograd.grad(embedding(ids, w, 0.5, dy_dtype), w, dy)
    want, mag, _ = exact_grad(ids, dy, V, 0.5)
    assert float(mag.max()) < 2**23  # times the scale
    assert torch.equal(got.cpu(), want.to(table_dtype))


@gpu
@pytest.mark.parametrize("n", [4096, 4097, 16383, 16384, 16385])
@pytest.mark.parametrize("V", [200, 300, 70000, 20_000_000])
def test_both_sorts_over_one_to_four_passes(dev, n, V):
    """Either side of the longest lists that one workgroup sorts."""
    w, ids, dy = make(dev, n, V, 4, BF16, F32, skew=V < 70000)
    (g,) = torch.autograd.grad(embedding(ids, w, 1.0, F32), w, dy)
    assert_grad(g, ids, dy, 1.0)


@gpu
@pytest.mark.parametrize("n", [1, 32, 33, 64, 3000])
def test_one_token_everywhere(dev, n):
    w, ids, dy = make(dev, n, 1000, 768, F32, BF16)
    ids.fill_(999)
    y = embedding(ids, w, 2.0, BF16)
    (g,) = torch.autograd.grad(y, w, dy)
    assert_grad(g, ids, dy, 2.0)


@gpu
def test_ids_out_of_range(dev):
    w, ids, dy = make(dev, 100, 500, 64, F32, F32)
    ids[3], ids[50], ids[99] = -1, 500, 2**40
    y = embedding(ids, w)
    bad = torch.zeros(100, dtype=torch.bool, device=dev)
    bad[[3, 50, 99]] = True
    assert bool(y[bad].isnan().all())
    assert torch.equal(y[~bad], w.detach()[ids[~bad]])
    (g,) = torch.autograd.grad(y, w, dy)
    assert_grad(g, ids, dy, 1.0)


@gpu
def test_empty_and_shapes(dev):
    w = torch.randn(10, 16, device=dev, requires_grad=True)
    y = embedding(torch.empty(0, 3, dtype=torch.long, device=dev), w)
    assert y.shape == (0, 3, 16)
    (g,) = torch.autograd.grad(y.sum(), w)
    assert torch.equal(g, torch.zeros_like(w))
    ids = torch.randint(0, 10, (4, 3, 2), device=dev)
    assert embedding(ids.transpose(0, 2), w).shape == (2, 3, 4, 16)
    assert torch.equal(embedding(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])


@gpu
def test_strides_and_alignment(dev):
    base = torch.randn(101, 70, device=dev)
    ids = torch.randint(0, 100, (57,), device=dev)
    for w in (base[:100, :64], base[1:, 1:65], base[:100, 3:68], base.to(BF16)[:100, 2:66]):
        assert torch.equal(embedding(ids, w), w[ids])
    w = torch.randn(100, 64, device=dev, requires_grad=True)
    big = torch.randn(57, 200, device=dev)
    for dy in (big[:, 1:65], torch.randn(64, 57, device=dev).t(),
               torch.randn(57 * 64 + 1, device=dev)[1:].view(57, 64),
               torch.ones(1, 1, device=dev).expand(57, 64)):
        (g,) = torch.autograd.grad(embedding(ids, w), w, dy)
        assert_grad(g, ids, dy, 1.0)
    with pytest.raises(RuntimeError, match="contiguous"):
        embedding(ids, base.t())


@gpu
def test_gpu_module_takes_what_nn_embedding_takes(dev):
    module_takes_what_nn_embedding_takes(dev)


@gpu
def test_gpu_refusals(dev):
    w = torch.randn(10, 16, device=dev, requires_grad=True)
    ids = torch.zeros(3, dtype=torch.long, device=dev)
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        embedding(ids, w.half())
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        embedding(ids, w, 1.0, torch.float16)
    with pytest.raises(TypeError, match="int64 or int32"):
        embedding(ids.float(), w)
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        embedding(ids, w[0])
    with pytest.raises(RuntimeError, match="ids on"):
        embedding(ids.cpu(), w)
    y = embedding(ids, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.square().sum(), w, create_graph=True)


@gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, grad):
    """A tangent of the table, or of the output's gradient, is not dropped."""
    w = torch.randn(10, 16, device=dev, requires_grad=grad)
    ids = torch.tensor([3, 3, 9], device=dev)
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="embedding: forward-mode"):
            embedding(ids, fwAD.make_dual(w, torch.ones_like(w)))
        if grad:
            y = embedding(ids, w)
            dy = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="embedding: forward-mode"):
                torch.autograd.grad(y, w, dy)
    assert torch.equal(embedding(ids, w), w[ids])


@gpu
def test_same_bits_again_and_on_another_stream(dev):
    w, ids, dy = make(dev, 20000, 5000, 192, F32, BF16)

    def both():
        y = embedding(ids, w, 1.5, BF16)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

    y, g = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            y2, g2 = both()
        side.synchronize()
        assert torch.equal(y, y2) and torch.equal(g, g2)


@gpu
def test_graph_replays(dev):
    """Lookup and gradient captured together, replayed on other ids."""
    w, ids, dy = make(dev, 3000, 5000, 256, F32, BF16)

    def both():
        y = embedding(ids, w, 1.5, BF16)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = both()
    for seed in range(4):
        _, new, new_dy = make(dev, 3000, 5000, 256, F32, BF16, seed=seed, skew=bool(seed % 2))
        ids.copy_(new)
        dy.copy_(new_dy)
        graph.replay()
        torch.cuda.synchronize()
        want_y, want_g = both()
        assert torch.equal(y, want_y) and torch.equal(g, want_g)


@gpu
def test_gradient_against_differences(dev):
    w, ids, dy = make(dev, 40, 9, 3, F32, F32, skew=False)
    (g,) = torch.autograd.grad(embedding(ids, w, 0.5), w, dy)
    base = w.detach()
    for v, c in ((0, 0), (4, 2), (8, 1)):
        step = torch.zeros_like(base)
        step[v, c] = 2.0  # linear: the difference is exact up to fp32 sums
        f = [float((embedding(ids, base + s * step, 0.5).double() * dy.double()).sum()) for s in (-1, 1)]
        # 80 products of rounded lookups: each off by 2^-23 of about |w| + 2
        room = 2.0**-22 * float(dy.abs().sum()) * (float(base.abs().max()) + 2)
        assert abs((f[1] - f[0]) / 4 - float(g[v, c])) <= room


@gpu
def test_module_under_autocast(dev):
    m = FusedEmbedding(100, 64, scale=8.0).to(dev)
    ids = torch.randint(0, 100, (2, 9), device=dev)
    with torch.autocast("cuda", dtype=BF16):
        y = m(ids)
    assert torch.equal(y, (m.weight.detach()[ids] * 8.0).to(BF16))
    y.float().sum().backward()
    assert m.weight.grad.dtype == F32
    assert_grad(m.weight.grad, ids, torch.ones(2, 9, 64), 8.0)
