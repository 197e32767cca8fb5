"""Attention over a shared prefix: packed rows and single new tokens.

Tolerance of the bf16 kernels against 64 bits, element by element: the weights
are rounded to bf16 before they meet the values (2^-8 of each weight), and the
result once more (2^-8 of itself). The scores are fp32: their rounding is
below 2^-24 * (|w| + D * sum |q k| / sqrt(D)), and e^w turns that into a
relative error of each weight. With the inputs here |w| stays below 2^11 and
the sum below 2^9, so 2^-10 covers it. Together (2^-8 + 2^-9) * sum p |v| +
2^-8 * |out|.
"""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from photon_amd.ops.attention import alibi_slopes, reference_attention_fp32
from photon_amd.ops.prefix_attention import (
    prefix_attention_decode,
    prefix_attention_qkv,
    sequence_starts,
)

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def exact(qkv, prefix, H, slopes, lens):
    """(out, sum p |v|) in 64 bits, sequence by sequence."""
    P = prefix.shape[0]
    qkv, prefix = qkv.double().cpu(), prefix.double().cpu()
    d = qkv.shape[1] // (3 * H)
    new, old = qkv.view(-1, 3, H, d), prefix.view(P, 3, H, d)
    slope = slopes.double().cpu().view(H, 1, 1)
    outs, mags, at = [], [], 0
    for n in lens:
        x = new[at:at + n]
        at += n
        q = x[:, 0].transpose(0, 1)
        k = torch.cat([old[:, 1], x[:, 1]]).transpose(0, 1)
        v = torch.cat([old[:, 2], x[:, 2]]).transpose(0, 1)
        gap = torch.arange(P, P + n).view(-1, 1) - torch.arange(P + n)
        w = q @ k.transpose(1, 2) / math.sqrt(q.shape[-1]) - slope * gap
        p = torch.softmax(w.masked_fill(gap < 0, -math.inf), -1)
        outs.append((p @ v).transpose(0, 1).flatten(1))
        mags.append((p @ v.abs()).transpose(0, 1).flatten(1))
    return torch.cat(outs), torch.cat(mags)


def assert_near(got, want):
    out, mag = want
    room = (2.0**-8 + 2.0**-9) * mag + 2.0**-8 * out.abs() + 1e-30
    err = (got.double().cpu() - out).abs()
    assert bool((err <= room).all()), float((err / room).max())


def make(dev, T, P, H, D, dtype=BF16, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    qkv = torch.randn(T, 3 * H * D, generator=g).to(dev, dtype)
    prefix = torch.randn(P, 3 * H * D, generator=g).to(dev, dtype)
    return qkv, prefix, alibi_slopes(H).to(dev)


# -- CPU --------------------------------------------------------------------
def test_sequence_starts():
    assert sequence_starts([3, 0, 1, 2]).tolist() == [0, 0, 0, 3, 4, 4]
    assert sequence_starts([]).shape == (0,) and sequence_starts([0]).dtype == torch.int32
    with pytest.raises(ValueError, match="lengths"):
        sequence_starts([2, -1])


@pytest.mark.parametrize("P", [0, 1, 7])
@pytest.mark.parametrize("lens", [[1], [4], [2, 0, 5, 1]])
def test_plain_path_against_whole_sequences(P, lens):
    """The rows of each sequence are the last rows of attention over prefix +
    sequence, computed at once."""
    H, D = 3, 8
    qkv, prefix, slopes = make("cpu", sum(lens), P, H, D, torch.float64)
    got = prefix_attention_qkv(qkv, prefix, H, slopes, sequence_starts(lens))
    want, mag = exact(qkv, prefix, H, slopes, lens)
    assert bool(((got - want).abs() <= 1e-12 * mag).all())
    at = 0
    for n in lens:
        if n:
            whole = torch.cat([prefix, qkv[at:at + n]]).view(P + n, 3, H, D).permute(1, 2, 0, 3)
            ref = reference_attention_fp32(*(x[None] for x in whole), slopes)[0, :, P:]
            assert (got[at:at + n].view(n, H, D).transpose(0, 1) - ref).abs().max() < 1e-5
        at += n


def test_plain_decode_steps_match_packed_rows():
    H, D, lens = 2, 8, [5, 3, 6]
    qkv, prefix, slopes = make("cpu", sum(lens), 4, H, D, torch.float64)
    want = prefix_attention_qkv(qkv, prefix, H, slopes, sequence_starts(lens))
    cache = torch.full((3, 6, 2, H, D), float("nan"), dtype=torch.float64)
    held = torch.zeros(3, dtype=torch.int32)
    firsts = [0, 5, 8]
    for i in range(3):  # the steps that all three take
        rows = torch.tensor(firsts) + i
        got = prefix_attention_decode(qkv[rows], prefix, H, slopes, cache, held)
        assert (got - want[rows]).abs().max() < 1e-12
        held += 1
    assert cache[:, 3:].isnan().all() and torch.equal(cache[0, 2].flatten(), qkv[2, H * D:])
    with pytest.raises(IndexError, match="free slot"):
        prefix_attention_decode(qkv[:3], prefix, H, slopes, cache, held + 3)


def plain_keeps_bad_values(dev):
    """The plain path, as the kernels: what is not finite in a key or value
    reaches the rows that see it and no others."""
    H, D, lens, P = 2, 8, [3, 0, 5, 2], 4
    F64 = torch.float64
    qkv, prefix, slopes = make(dev, 10, P, H, D, F64)
    starts = sequence_starts(lens, dev)
    out, mag = (x.to(dev) for x in exact(qkv, prefix, H, slopes, lens))
    sees = torch.arange(10, device=dev).ge(5) & torch.arange(10, device=dev).lt(8)
    for bad in (math.nan, math.inf, -math.inf):
        x = qkv.clone()
        x[5, 2 * H * D + 3] = bad  # the third of the second sequence's five
        got = prefix_attention_qkv(x, prefix, H, slopes, starts, impl="torch")
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[sees, 3] = True
        assert bool(((got - out).abs() <= 1e-12 * mag)[~hit].all())
        assert bool((got[hit].isnan() if math.isnan(bad) else got[hit] == bad).all())
        x = qkv.clone()
        x[5, H * D + 3] = bad  # of its key: one head, and a weight may be zero
        got = prefix_attention_qkv(x, prefix, H, slopes, starts, impl="torch")
        hit.zero_()[sees, :D] = True
        assert bool(((got - out).abs() <= 1e-12 * mag)[~hit].all())
    x = qkv.clone()
    x[3, 2 * H * D], x[5, 2 * H * D] = math.inf, -math.inf  # NaN for who sees both
    got = prefix_attention_qkv(x, prefix, H, slopes, starts, impl="torch")[:, 0]
    assert got[3:5].eq(math.inf).all() and got[5:8].isnan().all() and got[[0, 1, 2, 8, 9]].isfinite().all()
    # single tokens: a cached value of one sequence, and a new one
    cache = torch.randn(3, 4, 2, H, D, generator=torch.Generator().manual_seed(3)).to(dev, F64)
    held = torch.tensor([2, 3, 0], dtype=torch.int32, device=dev)
    new = qkv[:3].clone()
    want = prefix_attention_decode(new, prefix, H, slopes, cache.clone(), held, impl="torch")
    cache[0, 1, 1, 1, 2] = math.inf
    new[2, 2 * H * D] = math.nan
    got = prefix_attention_decode(new, prefix, H, slopes, cache, held, impl="torch")
    assert got[0, D + 2] == math.inf and got[2, 0].isnan()
    got[0, D + 2], got[2, 0] = want[0, D + 2], want[2, 0]
    assert (got - want).abs().max() <= 1e-12


def test_plain_path_keeps_bad_values_in_their_sequence():
    plain_keeps_bad_values("cpu")


def refusals(dev):
    H, D = 2, 64
    qkv, prefix, slopes = make(dev, 5, 9, H, D)
    starts = sequence_starts([5], dev)
    cache = torch.zeros(5, 4, 2, H, D, dtype=BF16, device=dev)
    held = torch.zeros(5, dtype=torch.int32, device=dev)
    score = [
        ((qkv[:, :-1], prefix, H, slopes, starts), ValueError, "qkv must be"),
        ((qkv, prefix, 0, slopes, starts), ValueError, "qkv must be"),
        ((qkv[None], prefix, H, slopes, starts), ValueError, "qkv must be"),
        ((qkv, prefix[:, :-6], H, slopes, starts), ValueError, "prefix_qkv must be"),
        ((qkv, prefix.float(), H, slopes, starts), ValueError, "dtype and device"),
        ((qkv, prefix, H, slopes[:1], starts), ValueError, "slopes must be"),
        ((qkv, prefix, H, slopes, starts[:4]), ValueError, "starts must be"),
        ((qkv, prefix, H, slopes, starts.long()), ValueError, "starts must be"),
        ((qkv.clone().requires_grad_(), prefix, H, slopes, starts), RuntimeError, "no backward"),
    ]
    for args, kind, match in score:
        with pytest.raises(kind, match=match):
            prefix_attention_qkv(*args)
    for bad, match in ((cache[:4], "cache must be"), (cache[..., :32], "cache must be"),
                       (cache[:, :, :1], "cache must be"), (cache.float(), "dtype and device")):
        with pytest.raises(ValueError, match=match):
            prefix_attention_decode(qkv, prefix, H, slopes, bad, held)


def test_refusals():
    refusals("cpu")


def refused_cache_stays(dev):
    """A cache made in inference mode cannot be written outside of it: the
    call says so and leaves it as it is."""
    H, D = 2, 64
    qkv, prefix, slopes = make(dev, 3, 9, H, D)
    held = torch.zeros(3, dtype=torch.int32, device=dev)
    with torch.inference_mode():
        cache = torch.ones(3, 4, 2, H, D, dtype=BF16, device=dev)
    with torch.no_grad(), pytest.raises(RuntimeError, match="cache was made in inference mode"):
        prefix_attention_decode(qkv, prefix, H, slopes, cache, held)
    assert bool((cache == 1).all())
    with torch.inference_mode():
        prefix_attention_decode(qkv, prefix, H, slopes, cache, held)
    assert torch.equal(cache[:, 0], qkv[:, H * D:].view(3, 2, H, D)) and bool((cache[:, 1:] == 1).all())


def test_refused_cache_stays():
    refused_cache_stays("cpu")


# -- GPU --------------------------------------------------------------------
@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def check(dev, lens, P, H, D, seed=0):
    qkv, prefix, slopes = make(dev, sum(lens), P, H, D, seed=seed)
    got = prefix_attention_qkv(qkv, prefix, H, slopes, sequence_starts(lens, dev))
    assert got.dtype == BF16 and got.shape == (sum(lens), H * D)
    assert_near(got, exact(qkv, prefix, H, slopes, lens))


@gpu
def test_plain_path_on_a_gpu_keeps_bad_values_in_their_sequence(dev):
    plain_keeps_bad_values(dev)


@gpu
def test_gpu_refused_cache_stays(dev):
    refused_cache_stays(dev)


@gpu
@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(dev, which):
    H, D = 2, 64
    qkv, prefix, slopes = make(dev, 3, 9, H, D)
    cache, held = torch.zeros(3, 4, 2, H, D, dtype=BF16, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    with fwAD.dual_level():
        args = [qkv, prefix, slopes, cache]
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="prefix_attention_decode: forward-mode"):
            prefix_attention_decode(args[0], args[1], H, args[2], args[3], held)
        assert bool((cache == 0).all())
        if which < 3:
            with pytest.raises(NotImplementedError, match="prefix_attention_qkv: forward-mode"):
                prefix_attention_qkv(args[0], args[1], H, args[2], sequence_starts([3], dev))


@gpu
def test_gpu_refusals(dev):
    refusals(dev)
    qkv, prefix, slopes = make(dev, 5, 9, 2, 32)
    with pytest.raises(RuntimeError, match="64 or 128"):
        prefix_attention_qkv(qkv, prefix, 2, slopes, sequence_starts([5], dev))
    qkv, prefix, slopes = make(dev, 5, 9, 2, 64)
    with pytest.raises(RuntimeError, match="must be bf16"):
        prefix_attention_qkv(qkv.float(), prefix.float(), 2, slopes, sequence_starts([5], dev))
    with pytest.raises(ValueError, match="must be on"):
        prefix_attention_qkv(qkv, prefix, 2, slopes, sequence_starts([5]))
    cache = torch.zeros(5, 4, 2, 2, 65, dtype=BF16, device=dev)[..., :64]
    with pytest.raises(RuntimeError, match="aligned"):
        prefix_attention_decode(qkv, prefix, 2, slopes, cache,
                                torch.zeros(5, dtype=torch.int32, device=dev))


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [0, 1, 31, 64, 65, 127, 700])
@pytest.mark.parametrize("lens", [[1], [2, 0, 5, 1], [33], [31, 1, 2], [64], [30, 40], [65, 3, 200, 1, 1]])
def test_packed_rows(dev, D, P, lens):
    check(dev, lens, P, 3, D)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,P,H", [
    ([1] * 130, 333, 1), ([7, 100] * 20, 129, 12), ([1500], 63, 2), ([300, 700, 20], 0, 2), ([3] * 4, 4000, 1),
    # more than 128 items of 32 rows: tiles of 128 rows
    ([300, 700, 20], 0, 12), ([1] * 1000, 65, 12), ([500, 1, 0, 40], 1, 20), ([2, 3], 700, 150), ([4099], 31, 2),
    # whole rounds of workgroups, and a rest that is split
    ([90] * 50, 520, 16),
])
def test_packed_rows_larger(dev, D, lens, P, H):
    check(dev, lens, P, H, D)


@gpu
@pytest.mark.parametrize("H,D", [(64, 128), (100, 64)])
@pytest.mark.parametrize("kind", ["alibi", "steep", "flat", "rising", "a far key counts", "a far key is NaN"])
def test_far_keys_left_out(dev, H, D, kind):
    """More items than one round of workgroups over a long prefix: tiles that
    cannot count are not computed."""
    lens, P = [90] * 12 + [1, 0, 30], 2601
    qkv, prefix, slopes = make(dev, sum(lens), P, H, D, seed=H)
    if kind == "steep":
        slopes = torch.full_like(slopes, 1.0)
    elif kind == "flat":
        slopes = torch.zeros_like(slopes)
    elif kind == "rising":
        slopes = -0.1 * slopes
    elif kind == "a far key counts":  # q . k / sqrt(d) stays below 2^9
        prefix.view(P, 3, H, D)[0, 1, :, 5] = 1000.0
    elif kind == "a far key is NaN":
        prefix.view(P, 3, H, D)[70, 1, ::3, 5] = math.nan
    got = prefix_attention_qkv(qkv, prefix, H, slopes, sequence_starts(lens, dev))
    if kind == "a far key is NaN":
        bad = got.view(-1, H, D).isnan()
        assert bool(bad[:, ::3].all())
        keep = torch.arange(H) % 3 != 0
        sub = [x.view(-1, 3, H, D)[:, :, keep].flatten(1) for x in (qkv, prefix)]
        want = exact(*sub, int(keep.sum()), slopes[keep], lens)
        assert_near(got.view(-1, H, D)[:, keep].flatten(1), want)
    else:
        assert_near(got, exact(qkv, prefix, H, slopes, lens))


@gpu
def test_no_rows(dev):
    qkv, prefix, slopes = make(dev, 0, 9, 2, 64)
    assert prefix_attention_qkv(qkv, prefix, 2, slopes, sequence_starts([0, 0], dev)).shape == (0, 128)


@gpu
@pytest.mark.parametrize("H", [2, 48])
def test_strides_and_alignment(dev, H):
    D, lens, P = 64, [5, 60, 9], 100
    qkv, prefix, slopes = make(dev, 74, P, H, D)
    starts = sequence_starts(lens, dev)
    want = prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    W = 3 * H * D
    wide = torch.full((200, W + 24), float("nan"), dtype=BF16, device=dev)
    a, b = wide[:74, 8:8 + W], wide[80:180, 16:16 + W]
    a.copy_(qkv), b.copy_(prefix)
    assert torch.equal(prefix_attention_qkv(a, b, H, slopes, starts), want)
    odd = torch.empty(74 * (W + 1) + 1, dtype=BF16, device=dev)[1:].view(74, W + 1)[:, :W]
    odd.copy_(qkv)
    assert torch.equal(prefix_attention_qkv(odd, prefix.t().contiguous().t(), H, slopes, starts), want)
    one = qkv[:1].expand(74, W)
    assert torch.equal(prefix_attention_qkv(one, prefix, H, slopes, starts),
                       prefix_attention_qkv(one.contiguous(), prefix, H, slopes, starts))
    # behind the last row of either there is nothing that is read
    assert not want.isnan().any()


@gpu
@pytest.mark.parametrize("H,D", [(2, 64), (48, 64), (2, 128), (48, 128)])
def test_sequences_do_not_touch_each_other(dev, H, D):
    """Infinities and NaN of one sequence stay in it, and a later row's stay
    out of the earlier rows of its sequence."""
    lens, P = [5, 60, 9, 1], 100
    qkv, prefix, slopes = make(dev, 75, P, H, D)
    starts = sequence_starts(lens, dev)
    out, mag = exact(qkv, prefix, H, slopes, lens)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for part in (1, 2):  # a key, a value
            x = qkv.clone()
            x[40, part * H * D + 3] = bad
            got = prefix_attention_qkv(x, prefix, H, slopes, starts)
            clean = torch.ones(75, dtype=torch.bool)
            clean[40:65] = False
            assert_near(got[clean.to(dev)], (out[clean], mag[clean]))
            if part == 2:
                hit = got[40:65, 3]
                assert bool((hit.isnan() if math.isnan(bad) else hit == bad).all())
                rest = torch.ones(H * D, dtype=torch.bool)
                rest[3] = False
                assert_near(got[:, rest.to(dev)], (out[:, rest], mag[:, rest]))
            elif math.isnan(bad):
                assert got[40:65, :D].isnan().all()


@gpu
def test_not_finite_in_the_prefix(dev):
    """What every row sees reaches every row."""
    H, D, lens, P = 1, 64, [3, 40], 200
    qkv, prefix, slopes = make(dev, 43, P, H, D)
    starts = sequence_starts(lens, dev)
    for row, part, bad in ((199, 1, float("nan")), (0, 1, float("nan")), (199, 2, float("nan")), (199, 2, float("inf"))):
        x = prefix.clone()
        x[row, part * D + 5] = bad
        got = prefix_attention_qkv(qkv, x, H, slopes * 1e-3, starts)
        if part == 1:
            assert got.isnan().all()
        else:
            assert bool((got[:, 5].isnan() if math.isnan(bad) else got[:, 5] == bad).all())
            rest = torch.arange(D, device=dev) != 5
            assert got[:, rest].isfinite().all()


@gpu
@pytest.mark.parametrize("H", [1, 70])
def test_starts_out_of_range_stay_inside(dev, H):
    """Starts that no packing gives are read as the nearest that one could."""
    D, P = 64, 70
    qkv, prefix, slopes = make(dev, 40, P, H, D)
    starts = torch.full((40,), -5, dtype=torch.int32, device=dev)
    starts[20:] = 1000
    got = prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    want = exact(qkv, prefix, H, slopes, [20] + [1] * 20)
    assert_near(got, want)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,P,slots,H", [
    (1, 0, 1, 3), (1, 701, 24, 3), (3, 64, 7, 3), (33, 65, 40, 3), (70, 300, 130, 3), (2, 5, 700, 3),
    (1, 3000, 5, 1),  # more splits than are asked for early
    (400, 130, 9, 12), (130, 1, 3, 40),  # more than 128 items of 32 rows
    # a workgroup a CU each, and one more; the longest prefix that one attends
    (16, 40, 6, 16), (257, 40, 6, 1), (2, 1250, 300, 4), (2, 1251, 300, 4), (1, 2500, 2000, 2), (1, 2501, 3, 2),
])
def test_decode(dev, D, B, P, slots, H):
    """Against the packed form's definition, with NaN in every unused slot."""
    held = [(17 * i + slots - 1) % slots for i in range(B)]
    lens = [n + 1 for n in held]
    qkv, prefix, slopes = make(dev, sum(lens), P, H, D)
    out, mag = exact(qkv, prefix, H, slopes, lens)
    cache = torch.full((B, slots, 2, H, D), float("nan"), dtype=BF16, device=dev)
    ends, at = [], 0
    for b, n in enumerate(lens):
        cache[b, :n - 1] = qkv[at:at + n - 1, H * D:].view(n - 1, 2, H, D)
        at += n
        ends.append(at - 1)
    old = cache.clone()
    new = qkv[ends]
    got = prefix_attention_decode(new, prefix, H, slopes, cache, torch.tensor(held, dtype=torch.int32, device=dev))
    assert_near(got, (out[ends], mag[ends]))
    for b, n in enumerate(held):
        old[b, n] = new[b, H * D:].view(2, H, D)
    assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


@gpu
def test_decode_without_a_free_slot(dev):
    H, D = 2, 64
    qkv, prefix, slopes = make(dev, 4, 10, H, D)
    cache = torch.randn(4, 3, 2, H, D, device=dev).to(BF16)
    old = cache.clone()
    held = torch.tensor([2, 3, -1, 1 << 30], dtype=torch.int32, device=dev)
    out = prefix_attention_decode(qkv, prefix, H, slopes, cache, held)
    assert out[0].isfinite().all() and out[1:].isnan().all()
    assert torch.equal(cache[1:], old[1:]) and torch.equal(cache[0, :2], old[0, :2])


@gpu
def test_decode_strided_cache(dev):
    """One layer of a cache that holds all layers, heads before slots."""
    H, D, B, slots = 2, 64, 3, 9
    qkv, prefix, slopes = make(dev, B, 50, H, D)
    held = torch.tensor([4, 0, 8], dtype=torch.int32, device=dev)
    flat = torch.randn(B, slots, 2, H, D, device=dev).to(BF16)
    other = torch.randn(B, 2, 4, H, slots, D, device=dev).to(BF16)
    rest = other.clone()
    view = other[:, :, 1].permute(0, 3, 1, 2, 4)
    view.copy_(flat)
    want = prefix_attention_decode(qkv, prefix, H, slopes, flat, held)
    assert torch.equal(prefix_attention_decode(qkv, prefix, H, slopes, view, held), want)
    assert torch.equal(view, flat)
    assert torch.equal(other[:, :, [0, 2, 3]], rest[:, :, [0, 2, 3]])


@gpu
def test_two_graphs_and_a_side_stream(dev):
    """A scoring graph and a decoding graph, replayed in turn with eager work
    between, on new inputs; and both on a stream of their own."""
    H, D, lens, P = 3, 128, [9, 2, 30], 500
    qkv, prefix, slopes = make(dev, 41, P, H, D)
    starts = sequence_starts(lens, dev)
    new, _, _ = make(dev, 5, 0, H, D, seed=9)
    cache = torch.randn(5, 20, 2, H, D, device=dev).to(BF16)
    held = torch.tensor([0, 3, 7, 11, 2], dtype=torch.int32, device=dev)

    def score():
        return prefix_attention_qkv(qkv, prefix, H, slopes, starts)

    def decode(c):
        return prefix_attention_decode(new, prefix, H, slopes, c, held)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = score(), decode(cache)
    side.synchronize()
    assert torch.equal(a, score()) and torch.equal(b, decode(cache))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = score()
    with torch.cuda.graph(g2):
        b = decode(cache)
    for seed in range(1, 5):
        x, y, _ = make(dev, 41, P, H, D, seed=seed)
        qkv.copy_(x), prefix.copy_(y)
        eager_cache = cache.clone()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, score())
        assert torch.equal(b, decode(eager_cache)) and torch.equal(cache, eager_cache)
        held += 1


@gpu
def test_long_prefix_offsets_pass_32_bits(dev):
    """Byte offsets beyond 2^31 inside a prefix whose rows lie far apart."""
    H, D, P = 1, 64, 600
    qkv, small, slopes = make(dev, 3, P, H, D)
    wide = torch.zeros(P, 2_100_000, dtype=BF16, device=dev)
    prefix = wide[:, 64:64 + 3 * D]
    prefix.copy_(small)
    slopes = torch.full_like(slopes, 1e-3)
    got = prefix_attention_qkv(qkv, prefix, H, slopes, sequence_starts([3], dev))
    assert_near(got, exact(qkv, small, H, slopes, [3]))


@gpu
def test_many_rows_over_millions_of_keys(dev):
    """Slope 1: only the last keys count, as over a prefix of these alone; and
    one that is far and large enough to be all that counts."""
    H, D, P, near = 1, 64, 4_200_000, 1000
    lens = [64] * 1540
    g = torch.Generator(device=dev).manual_seed(5)
    prefix = torch.randn(P, 3 * D, generator=g, device=dev, dtype=BF16)
    qkv = torch.randn(sum(lens), 3 * D, generator=g, device=dev, dtype=BF16)
    slopes, starts = torch.ones(1, device=dev), sequence_starts(lens, dev)
    got = prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    assert_near(got[:192], exact(qkv[:192], prefix[-near:], H, slopes, lens[:3]))
    want = prefix_attention_qkv(qkv, prefix[-near:], H, slopes, starts)
    # both are off by what one call is allowed: weights, then the result
    room = 2 * (2.0**-8 + 2.0**-9) * 6.0 + 2.0**-7 * want.float().abs()
    assert bool(((got.float() - want.float()).abs() <= room).all())
    prefix[0, D + 5] = 2.0**30
    got = prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    hit, miss = qkv[:, 5] > 0.25, qkv[:, 5] < 0
    # one weight p counts: round(p) * v / p with |round(p) / p - 1| <= 2^-8
    # (scores of 2^28 leave p anywhere within 2^64), then the result's rounding
    v = prefix[0, 2 * D:].float()
    assert bool(((got[hit].float() - v).abs() <= (2.0**-8 + 2.0**-8 * (1 + 2.0**-8)) * v.abs()).all())
    assert bool(((got - want).float().abs() <= room)[miss].all())


@gpu
def test_graph_of_many_rows(dev):
    """The three kernels of a large call in a graph, on new inputs."""
    H, D, lens, P = 64, 128, [100] * 11, 2600
    qkv, prefix, slopes = make(dev, sum(lens), P, H, D)
    starts = sequence_starts(lens, dev)
    prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prefix_attention_qkv(qkv, prefix, H, slopes, starts)
    for i in range(1, 4):
        qkv.mul_(-1.0)
        prefix.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, prefix_attention_qkv(qkv, prefix, H, slopes, starts))
