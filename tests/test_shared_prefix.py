"""The model over a shared prefix, the ICL harness on it, and a training step
that runs lookup, gradient and clipping together before the model is scored.

Tolerances: on the CPU everything is fp32 and the two paths add the same
numbers in another order: below 100 keys * 2^-24 for a softmax, a few of those
a layer, values of unit size: 1e-4 for logits. Under autocast on the GPU each
of about 8 roundings a layer moves a hidden state by up to 2^-8 of itself;
with logits of std 0.3 (0.02 * sqrt(256) unit hidden values) that is 0.03 *
0.3 rms over two layers, and 0.1 is ten times that.
"""

import copy
import json
import math

import pytest
import torch
import torch.nn.functional as F

from photon_amd.data.convert import ByteTokenizer
from photon_amd.eval import evaluate_icl_tasks
from photon_amd.eval.icl import _continuation_stats, _greedy_generate, _shared_stats
from photon_amd.models import MPTCausalLM, MPTConfig, SharedPrefix
from photon_amd.ops.clip import clip_grad_norm_

gpu = pytest.mark.gpu


def tiny(impl="torch", d=64, heads=2, layers=2, vocab=300, **kw):
    torch.manual_seed(3)
    return MPTCausalLM(MPTConfig(d_model=d, n_heads=heads, n_layers=layers, max_seq_len=128,
                                 vocab_size=vocab, attn_impl=impl, **kw)).eval()


def assert_scores(model, prefix, seqs, tol):
    shared = SharedPrefix(model, prefix)
    got = shared.logits(shared.score(seqs)).float()
    dev, at = got.device, 0
    with torch.no_grad():
        for s in seqs:
            if not s:
                continue
            whole = model(torch.tensor([prefix + s], device=dev))["logits"][0].float()
            assert (got[at:at + len(s)] - whole[len(prefix):]).abs().max() < tol
            at += len(s)
        last = shared.logits(shared.last_hidden)[0].float()
        whole = model(torch.tensor([prefix], device=dev))["logits"][0, -1].float()
        assert (last - whole).abs().max() < tol
        # the same tokens one by one: the sequences' common number of steps
        live = [s for s in seqs if s]
        steps = min(map(len, live))
        shared.begin(len(live), steps)
        for i in range(steps):
            out = shared.logits(shared.step(torch.tensor([s[i] for s in live], device=dev))).float()
            for row, s in zip(out, live):
                ref = model(torch.tensor([prefix + s[:i + 1]], device=dev))["logits"][0, -1].float()
                assert (row - ref).abs().max() < tol
        with pytest.raises(IndexError, match="slots"):
            shared.step(torch.zeros(len(live), dtype=torch.long))


SEQS = [[5, 9, 200, 1], [7, 8], [], [1, 2, 3, 4, 5, 6, 7]]


@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_scores_match_whole_sequences(scale):
    assert_scores(tiny(emb_scale=scale), [11, 250, 3, 99, 42], SEQS, 1e-4)


def test_shared_prefix_refusals():
    m = tiny()
    for bad in ([], [[1, 2]]):
        with pytest.raises(ValueError, match="prefix_ids"):
            SharedPrefix(m, bad)
    with pytest.raises(TypeError, match="MPTCausalLM"):
        SharedPrefix(torch.nn.Sequential(m), [1])
    s = SharedPrefix(m, [1])
    with pytest.raises(RuntimeError, match="begin"):
        s.step(torch.tensor([1]))
    with pytest.raises(ValueError, match="count and slots"):
        s.begin(0, 4)
    s.begin(2, 4)
    with pytest.raises(ValueError, match="2 tokens"):
        s.step(torch.tensor([1]))
    assert s.score([[], []]).shape == (0, 64)


def test_prefix_takes_no_gradient():
    m = tiny()
    s = SharedPrefix(m, [1, 2])
    assert not s.score([[3]]).requires_grad and not s.last_hidden.requires_grad
    s.begin(1, 1)
    assert not s.step(torch.tensor([3])).requires_grad


PAIRS = [
    [("the sky is ", "blue"), ("the sky is ", "green and"), ("the sky is ", "b")],
    [("a cat sat ", "down"), ("a cow sat ", "down")],  # contexts differ
    [("xy", "z"), ("ab", "z")],  # nothing shared
    [("only one ", "here")],
    [("same ", ""), ("same ", "thing"), ("same ", "thin")],  # nothing to score
    [("", "abc"), ("", "abd")],  # no context
    [("long context " * 20, "one"), ("long context " * 20, "three")],  # cut off
]


@pytest.mark.parametrize("pairs", PAIRS)
def test_shared_stats_match_single_ones(pairs):
    m, tok = tiny(), ByteTokenizer()
    want = [_continuation_stats(m, tok, c, a, "cpu", 100) for c, a in pairs]
    got = _shared_stats(m, tok, pairs, "cpu", 100)
    for (ce, n, ok), (ce2, n2, ok2) in zip(want, got):
        assert n == n2 and ok == ok2 and abs(ce - ce2) <= 1e-4 * max(n, 1)


@pytest.mark.parametrize("stops", [[], ["a"], ["\n"]])
def test_cached_generation_matches(stops):
    m, tok = tiny(), ByteTokenizer()
    for prompt in ("tell me", "x", ""):
        if not prompt:
            continue
        a = _greedy_generate(m, tok, prompt, "cpu", 100, 9, stops)
        b = _greedy_generate(m, tok, prompt, "cpu", 100, 9, stops, share_prefix=True)
        assert a == b


def write_tasks(tmp_path):
    rows = {
        "multiple_choice": [{"query": f"question {i}", "choices": ["a", "bb", "c c"], "gold": i % 3} for i in range(4)],
        "schema": [{"context_options": ["the cat", "the dog"], "continuation": f"ran {i}", "gold": 0} for i in range(3)],
        "generation_task_with_answers": [{"context": f"who {i}", "answer": "me", "aliases": []} for i in range(2)],
        "language_modeling": [{"context": "one two", "continuation": "three"}] * 2,
    }
    tasks = []
    for kind, exs in rows.items():
        f = tmp_path / f"{kind}.jsonl"
        f.write_text("".join(json.dumps(e) + "\n" for e in exs))
        tasks.append({"label": kind, "dataset_uri": str(f), "icl_task_type": kind, "num_fewshot": [0, 2]})
    return tasks


def test_icl_tasks_score_the_same(tmp_path):
    tasks = write_tasks(tmp_path)
    a = evaluate_icl_tasks(tiny(), tasks, ByteTokenizer(), max_seq_len=128)
    b = evaluate_icl_tasks(tiny(), tasks, ByteTokenizer(), max_seq_len=128, share_prefix=True)
    assert a == b and len(a) == 12


def test_eval_path_of_centralised_training(tmp_path):
    """run_icl_eval reads icl_tasks_config.share_prefix; a wrapped model runs
    option by option."""
    from photon_amd.centralised_train import run_icl_eval

    tasks = write_tasks(tmp_path)
    got = {}
    for share in (False, True):
        cfg = {"icl_tasks_config": {"icl_tasks": tasks, "share_prefix": share}, "llm_config": {"max_seq_len": 128}}
        got[share] = run_icl_eval(cfg, tiny(vocab=512), "cpu")
    assert got[False] == got[True] and len(got[True]) >= 12

    class Wrapped(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, *a, **k):
            return self.inner(*a, **k)

    assert run_icl_eval(cfg, Wrapped(tiny(vocab=512)), "cpu") == got[False]


def test_icl_precision():
    """Autocast only where the flash kernels would refuse the weights."""
    from photon_amd.centralised_train import _icl_needs_autocast

    def needs(device="cuda", dtype=torch.float32, impl="flash", **llm):
        cfg = {"llm_config": {"model": {"attn_config": {"attn_impl": impl}}, **llm}}
        return _icl_needs_autocast(cfg, torch.nn.Linear(2, 2).to(dtype), device)

    assert needs() and needs("cuda:0", precision="amp_bf16")
    assert not (needs("cpu") or needs(dtype=torch.bfloat16) or needs(impl="torch") or needs(precision="fp32"))
    assert _icl_needs_autocast({"llm_config": {}}, torch.nn.Linear(2, 2), "cuda")


def test_no_tokens_to_generate():
    m, tok = tiny(vocab=512), ByteTokenizer()
    assert all(_greedy_generate(m, tok, "abc", "cpu", 50, 0, share_prefix=s) == "" for s in (False, True))


def inference_mode_matches(m, dev):
    """Scores and steps, inside inference mode and with a model made outside."""
    def run():
        shared = SharedPrefix(m, list(range(20)))
        shared.begin(2, 3)
        outs = [shared.score([[5, 6, 7], [8]])]
        outs += [shared.step(torch.tensor([i, i + 1], device=dev)) for i in range(3)]
        return torch.cat([shared.logits(x) for x in outs])

    with torch.no_grad():
        want = run()
    with torch.inference_mode():
        got = run()
        assert torch.equal(got, want)


def test_inference_mode():
    inference_mode_matches(tiny(), "cpu")


def test_nothing_keeps_a_graph():
    """Runs without gradients, its logits too, wherever it is called from."""
    m = tiny()
    assert m.transformer.wte.weight.requires_grad and torch.is_grad_enabled()
    shared = SharedPrefix(m, [1, 2, 3])
    shared.begin(2, 1)
    outs = [shared.last_hidden, shared.score([[4, 5], [6]]), shared.step(torch.tensor([7, 8]))]
    assert not any(t.requires_grad for x in outs for t in (x, shared.logits(x)))


def test_emb_scale_in_the_model():
    """emb_scale is read from the configuration, survives a resize, and 1.0
    leaves the model as it was."""
    from photon_amd.models.mpt import build_model, resize_vocab

    cfg = {"model": {"d_model": 64, "n_heads": 2, "n_layers": 1, "vocab_size": 50, "emb_scale": 8.0,
                     "attn_config": {"attn_impl": "torch"}}}
    torch.manual_seed(0)
    m = build_model(cfg)
    torch.manual_seed(0)
    plain = build_model({"model": {**cfg["model"], "emb_scale": 1.0}})
    assert all(torch.equal(a, b) for a, b in zip(m.parameters(), plain.parameters()))
    ids = torch.randint(0, 50, (2, 5))
    assert torch.equal(m.transformer.wte(ids), plain.transformer.wte(ids) * 8.0)
    assert torch.equal(plain.transformer.wte(ids), F.embedding(ids, plain.transformer.wte.weight))
    resize_vocab(m, 70)
    assert m.transformer.wte.scale == 8.0 and m.transformer.wte(ids).shape == (2, 5, 64)


def loud(impl, heads):
    """A model whose attention is most of what it says: queries, keys and
    values 5 times the usual, their projection 20 times.

    Two bf16 runs of it: some 24 roundings, each 0.42 * 2^-8 of the hidden
    state rms, added at random, move a logit of std 0.33 by 0.0027, two runs by
    0.0038 apart; the logits, up to 1.5, are rounded to 2^-8 in either. The
    largest of 10^4 is at 4 sigma, 0.015 + 0.008: LOGIT is twice that. A mean
    cross-entropy of one token, 3 sigma, 0.0114 + 0.0078: CE."""
    m = tiny(impl, 256, heads)
    with torch.no_grad():
        for block in m.transformer.blocks:
            block.attn.Wqkv.weight.mul_(5.0)
            block.attn.out_proj.weight.mul_(20.0)
    return m


LOGIT, CE = 0.05, 0.02
LOUD_PREFIX = [(37 * i) % 300 for i in range(90)]


@pytest.mark.parametrize("mistake", ["last key", "no bias", "one sequence"])
@pytest.mark.parametrize("heads", [4, 2])
def test_a_mistake_moves_the_loud_model(monkeypatch, heads, mistake):
    """What the GPU tests of this model allow is far below what a wrong call
    does to its logits and scores."""
    from photon_amd.models import shared_prefix
    from photon_amd.ops.prefix_attention import prefix_attention_decode, prefix_attention_qkv

    def planted(call):
        def wrong(qkv, prefix, h, slopes, *rest, impl="flash"):
            if mistake == "last key":
                prefix = prefix[:-1]
            elif mistake == "no bias":
                slopes = slopes * 0.0
            else:  # all rows of the first sequence, all slots empty
                rest = (*rest[:-1], rest[-1] * 0)
            return call(qkv, prefix, h, slopes, *rest, impl=impl)
        return wrong

    m, tok = loud("torch", heads), ByteTokenizer()

    def outputs():
        s = SharedPrefix(m, LOUD_PREFIX)
        s.begin(2, 2)
        return [s.logits(s.score(SEQS)), *(s.logits(s.step(torch.tensor([i, 7]))) for i in (5, 9))]

    want = outputs()
    ces = [_continuation_stats(m, tok, c, a, "cpu", 100) for p in PAIRS for c, a in p]
    monkeypatch.setattr(shared_prefix, "prefix_attention_qkv", planted(prefix_attention_qkv))
    monkeypatch.setattr(shared_prefix, "prefix_attention_decode", planted(prefix_attention_decode))
    for a, b in zip(want[::2], outputs()[::2]):  # scores, the second step
        assert (a - b).abs().max() > 4 * LOGIT
    if heads == 2:  # slopes of 2^-4 and 2^-8 say little in these short texts
        return
    wrong = [x for p in PAIRS for x in _shared_stats(m, tok, p, "cpu", 100)]
    assert max(abs(a[0] - b[0]) / max(a[1], 1) for a, b in zip(ces, wrong)) > 4 * CE


# -- GPU --------------------------------------------------------------------
@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@gpu
@pytest.mark.parametrize("d,heads", [(256, 4), (256, 2)])
@pytest.mark.parametrize("weights", ["autocast", "bf16"])
def test_gpu_scores_match_whole_sequences(dev, d, heads, weights):
    m = tiny("flash", d, heads).to(dev)
    prefix = [(37 * i) % 300 for i in range(90)]
    if weights == "bf16":
        assert_scores(m.to(torch.bfloat16), prefix, SEQS, 0.1)
    else:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert_scores(m, prefix, SEQS, 0.1)


@gpu
@pytest.mark.parametrize("heads", [4, 2])
@pytest.mark.parametrize("weights", ["autocast", "bf16"])
def test_gpu_scores_of_the_loud_model(dev, heads, weights):
    m, tok = loud("flash", heads).to(dev), ByteTokenizer()
    if weights == "bf16":
        m = m.to(torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=weights == "autocast"):
        assert_scores(m, LOUD_PREFIX, SEQS, LOGIT)
        for pairs in PAIRS:
            want = [_continuation_stats(m, tok, c, a, dev, 100) for c, a in pairs]
            got = _shared_stats(m, tok, pairs, dev, 100)
            mean, mean2 = ([ce / max(n, 1) for ce, n, _ in s] for s in (want, got))
            assert [n for _, n, _ in want] == [n for _, n, _ in got]
            assert all(abs(a - b) <= CE for a, b in zip(mean, mean2))
            if len(pairs) > 1 and sorted(mean)[1] - min(mean) > 2 * CE:
                assert mean.index(min(mean)) == mean2.index(min(mean2))


@gpu
def test_gpu_inference_mode(dev):
    inference_mode_matches(tiny("flash", 256, 4).to(dev, torch.bfloat16), dev)


@gpu
def test_gpu_icl_tasks(dev, tmp_path):
    m = tiny("flash", 256, 4).to(dev)
    tok = ByteTokenizer()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for pairs in PAIRS:
            want = [_continuation_stats(m, tok, c, a, dev, 100) for c, a in pairs]
            for (ce, n, _), (ce2, n2, _) in zip(want, _shared_stats(m, tok, pairs, dev, 100)):
                assert n == n2 and abs(ce - ce2) <= 0.1 * max(n, 1)
        got = evaluate_icl_tasks(m, write_tasks(tmp_path), tok, device=dev, max_seq_len=128, share_prefix=True)
    assert len(got) == 12 and all(0.0 <= v <= 1.0 for v in got.values())


@gpu
def test_train_clip_then_score(dev):
    """Two steps with the fused lookup, its gradient and clipping against the
    same with torch's lookup and a loop over the gradients, then both models
    score over a shared prefix."""
    from photon_amd.ops.optim import DecoupledAdamW

    ids = torch.randint(0, 300, (4, 64), device=dev)
    models = [tiny("flash", 256, 4, emb_scale=4.0, emb_impl=i).train().to(dev) for i in ("fused", "torch")]
    opts = [DecoupledAdamW(m.parameters(), lr=1e-3) for m in models]
    for step in range(2):
        norms = []
        for m, opt in zip(models, opts):
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16):
                m(ids, labels=ids)["loss"].backward()
            ps = list(m.parameters())
            if m.cfg.emb_impl == "fused":
                want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
                total = float(clip_grad_norm_(ps, 0.1))
                assert abs(total - want) <= 2.0**-22 * want
            else:
                total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
                for p in ps:
                    p.grad.mul_(min(1.0, 0.1 / (total + 1e-6)))
            norms.append(total)
            opt.step()
        if step == 0:
            # one forward and backward with the same roundings; the embedding's
            # gradient differs by fp32 sums of 256 terms
            assert abs(norms[0] - norms[1]) <= 1e-4 * norms[1]
            a, b = (m.transformer.wte.weight.grad for m in models)
            assert (a - b).norm() <= 1e-4 * b.norm()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = (SharedPrefix(m.eval(), list(range(50))) for m in models)
        x, y = (s.logits(s.score(SEQS)).float() for s in (a, b))
    assert x.isfinite().all() and (x - y).abs().max() < 0.1


@gpu
def test_microbatch_captured_beside_a_live_loss(dev):
    """A loss of an eager pass over the same parameters is alive while the
    microbatch is captured and replayed, and is used afterwards. Bounds as in
    the next test."""
    from photon_amd.train.graphs import GraphedMicrobatch

    def amp():
        return torch.autocast("cuda", dtype=torch.bfloat16)

    eager, graphed = (tiny("flash", 256, 4, emb_scale=2.0).train().to(dev) for _ in range(2))
    ids = torch.randint(0, 300, (2, 64), device=dev)

    def both(f, model):
        with amp():
            loss = model(ids, labels=ids)["loss"]
            f(loss)
        return loss

    live = both(lambda loss: None, graphed)
    g = GraphedMicrobatch(graphed, amp, 1.0, 2, 64, dev)
    loss = float(g.run(ids))
    both(lambda loss: loss.backward(), eager)
    held = [p.grad for p in graphed.parameters()]
    for times in (1, 2, 3):  # replayed once more each, then the live one's backward
        for a, b in zip(graphed.parameters(), eager.parameters()):
            assert (a.grad - times * b.grad).norm() <= 2.0**-8 * times * b.grad.norm()
        if times == 1:
            assert abs(float(g.run(ids)) - loss) <= 2.0**-8 * loss
        elif times == 2:
            with amp():
                live.backward()
    assert all(p.grad is h for p, h in zip(graphed.parameters(), held))
    assert abs(float(live.detach()) - loss) <= 2.0**-8 * loss


@gpu
def test_hooks_on_parameters_are_captured(dev):
    """Hooks that double a gradient, on a matrix and, behind the accumulation,
    on a vector: in every replay, as in an eager pass."""
    from photon_amd.train.graphs import GraphedMicrobatch

    def amp():
        return torch.autocast("cuda", dtype=torch.bfloat16)

    def double(p):
        p.grad.mul_(2.0)

    eager, graphed = (tiny("flash", 256, 4).train().to(dev) for _ in range(2))
    for m in (eager, graphed):
        m.transformer.blocks[0].attn.Wqkv.weight.register_hook(lambda g: g * 2.0)
        m.transformer.norm_f.weight.register_post_accumulate_grad_hook(double)
    ids = torch.randint(0, 300, (2, 64), device=dev)
    g = GraphedMicrobatch(graphed, amp, 1.0, 2, 64, dev)
    with amp():
        eager(ids, labels=ids)["loss"].backward()
    for i in range(3):
        if i:
            g._zero_grads()
        g.run(ids)
        for a, b in zip(graphed.parameters(), eager.parameters()):
            assert (a.grad - b.grad).norm() <= 2.0**-8 * b.grad.norm()


@gpu
def test_graphed_microbatch_matches_eager(dev):
    """Lookup and gradient inside the captured training microbatch. Should a
    library product choose another split in a graph, a bf16 value rounds to
    its other neighbour: 2^-7 of some values, below 2^-8 in the norm."""
    from photon_amd.train.graphs import GraphedMicrobatch

    def amp():
        return torch.autocast("cuda", dtype=torch.bfloat16)

    eager, graphed = (tiny("flash", 256, 4, emb_scale=2.0).train().to(dev) for _ in range(2))
    g = GraphedMicrobatch(graphed, amp, 1.0, 2, 64, dev)
    for i in range(4):
        ids = torch.randint(0, 300, (2, 64), device=dev)
        if i:
            g._zero_grads()
        loss = float(g.run(ids))
        eager.zero_grad()
        with amp():
            want = eager(ids, labels=ids)["loss"]
            want.backward()
        assert abs(loss - float(want.detach())) <= 2.0**-8 * loss
        for a, b in zip(graphed.parameters(), eager.parameters()):
            assert (a.grad - b.grad).norm() <= 2.0**-8 * b.grad.norm()
