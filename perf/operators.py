"""Measured cases of three operators: the embedding lookup with its gradient,
the gradient norm with clipping, and attention over a shared prefix.

``own`` False computes each in its plain form, from elementary torch operations
in 32 bits, rounded once at the end; ``own`` True makes the calls that a
program makes of photon_amd. Inputs, lengths and views are the same for both.
"""

import math

import torch

own = False

F32, BF16 = torch.float32, torch.bfloat16
DTYPES = {"float32": F32, "bfloat16": BF16}


# -- cases ------------------------------------------------------------------
def listed():
    return [
        # one decoding step of four sequences: fp32 table read under autocast
        _embed("lookup of a decoding step", 4, 768, "float32", "bfloat16", False),
        # a last, ragged microbatch of an fp32 run (no autocast), 7 rows of 1021
        _embed("lookup and gradient, ragged fp32", 7147, 1024, "float32", "float32", True),
        # microbatch 32 x 2048 of the 125M configuration under autocast
        _embed("lookup and gradient, 125m", 65536, 768, "float32", "bfloat16", True),
        # microbatch 8 x 2048 of the 7B configuration with bf16 weights
        _embed("lookup and gradient, 7b bf16", 16384, 4096, "bfloat16", "bfloat16", True),
        # a two-layer model as the smoke run trains it: many short tensors
        _clip("clip, two layers fp32", 256, 2, "float32", 0.5),
        # gradients of the 1B configuration, fp32 parameters under autocast
        _clip("clip, 1b fp32", 2048, 24, "float32", 0.25),
        # the 3B configuration with bf16 matrices and fp32 vectors, in bounds:
        # the norms are wanted, the gradients stay
        _clip("norms in bounds, 3b mixed", 2560, 32, "mixed", 2.0),
        # four short answers after a question without examples
        _score("score, short question", 12, 64, 93, 4, 2, 9),
        # four answers after a question with twenty-five examples
        _score("score, many examples", 16, 128, 1507, 4, 8, 40),
        # forty-eight questions that share their examples, near the longest
        _score("score, batch of questions", 32, 128, 3901, 48, 24, 160),
        # greedy generation of one answer
        _decode("decode, one answer", 12, 64, 701, 1, 24),
        # one token for each of many answers to a long shared prompt
        _decode("decode, many answers", 32, 128, 3967, 64, 512),
    ]


def _embed(name, n, d, table, out, grad, vocab=50368, scaled=True):
    return {"name": name, "op": "embed", "n": n, "d": d, "vocab": vocab, "table": table,
            "out": out, "grad": grad, "scaled": scaled}


def _clip(name, d, layers, types, bound):
    return {"name": name, "op": "clip", "d": d, "layers": layers, "vocab": 50368, "types": types, "bound": bound}


def _score(name, heads, d, prefix, count, shortest, longest):
    return {"name": name, "op": "score", "heads": heads, "d": d, "prefix": prefix, "count": count,
            "shortest": shortest, "longest": longest}


def _decode(name, heads, d, prefix, count, slots):
    return {"name": name, "op": "decode", "heads": heads, "d": d, "prefix": prefix, "count": count, "slots": slots}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "clip", "score", "decode"])
    if op == "embed":
        d = rng.choice([256, 320, 768, 1000, 1024, 2048, 2560, 4096])
        grad = rng.random() < 0.75
        table = rng.choice(["float32", "bfloat16"])
        out = "bfloat16" if table == "bfloat16" else rng.choice(["float32", "bfloat16"])
        c = _embed("", _log(rng, 1, 50_000_000 // d), d, table, out, grad,
                   rng.choice([512, 50257, 50368]), rng.random() < 0.5)
    elif op == "clip":
        d = rng.choice([256, 384, 512, 768, 1024, 1600, 2048])
        c = _clip("", d, _log(rng, 1, 24), rng.choice(["float32", "bfloat16", "mixed"]),
                  rng.choice([0.01, 0.25, 0.9, 4.0]))
    else:
        d = rng.choice([64, 128])
        heads = rng.choice([1, 2, 4, 8, 12, 16, 20, 32] if d == 128 else [1, 4, 12, 16, 25])
        if op == "score":
            shortest = _log(rng, 1, 24)
            c = _score("", heads, d, _log(rng, 1, 3901), _log(rng, 1, 48), shortest, shortest + _log(rng, 1, 136))
        else:
            c = _decode("", heads, d, _log(rng, 1, 3967), _log(rng, 1, 64), _log(rng, 1, 512))
    del c["name"]
    return c


def _lengths(c):
    """Lengths of the sequences after the prefix, spread over the case's range."""
    lo, hi = c["shortest"], c["longest"]
    return [lo + (7919 * i + 13) % (hi - lo + 1) for i in range(c["count"])]


def _held(c):
    """How many own keys each decoding sequence holds before the step."""
    return [(5077 * i + 5) % c["slots"] for i in range(c["count"])]


def _shapes(c):
    """The parameters of an MPT model, in order: (shape, whether a matrix)."""
    d = c["d"]
    block = [(d,), (d,), (3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return [(c["vocab"], d)] + block * c["layers"] + [(d,), (d,)]


def _grad_type(c, shape):
    if c["types"] == "mixed":
        return BF16 if len(shape) == 2 else F32
    return DTYPES[c["types"]]


def work(c):
    if c["op"] == "embed":
        t, o = DTYPES[c["table"]].itemsize, DTYPES[c["out"]].itemsize
        n, d, v = c["n"], c["d"], c["vocab"]
        b = n * 8 + min(n, v) * d * t + n * d * o
        f = n * d
        if c["grad"]:  # the output's gradient once, the whole table's gradient once
            b += n * d * o + v * d * t
            f += 2 * n * d
        return {"bytes": b, "flops": f}
    if c["op"] == "clip":
        sizes = [(math.prod(s), _grad_type(c, s).itemsize) for s in _shapes(c)]
        clips = c["bound"] < 1
        return {"bytes": sum(n * i for n, i in sizes) * (2 if clips else 1), "flops": sum(n for n, _ in sizes) * (3 if clips else 2)}
    h, d, p = c["heads"], c["d"], c["prefix"]
    if c["op"] == "score":
        lens = _lengths(c)
        t = sum(lens)
        pairs = t * p + sum(x * (x + 1) // 2 for x in lens)
        return {"bytes": 2 * h * d * (2 * p + 4 * t), "flops": 4 * h * d * pairs}
    b, own_keys = c["count"], sum(_held(c))
    return {"bytes": 2 * h * d * (2 * p + 2 * own_keys + 6 * b), "flops": 4 * h * d * (b * p + own_keys + b)}


# -- inputs -----------------------------------------------------------------
def _slopes(heads, dev):
    """ALiBi's slopes; a head count between powers of two takes every second
    one of the next power first."""
    full = 2 ** math.ceil(math.log2(heads))
    s = [2.0 ** (-8.0 * (i + 1) / full) for i in range(full)]
    s = s if full == heads else (s[1::2] + s[0::2])[:heads]
    return torch.tensor(s, dtype=F32, device=dev)


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=BF16, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=F32) * std).to(dtype)

    if c["op"] == "embed":
        n, d, v = c["n"], c["d"], c["vocab"]
        # Zipf's law over the vocabulary, the ranks spread over the ids
        rank = torch.exp(torch.rand(n, generator=g, device=dev) * math.log(v)).long().clamp_(1, v) - 1
        ids = torch.randperm(v, generator=g, device=dev)[rank]
        s = {"ids": ids, "table": normal(v, d, dtype=DTYPES[c["table"]], std=0.02).requires_grad_(c["grad"]),
             "scale": math.sqrt(d) if c["scaled"] else 1.0, "out": DTYPES[c["out"]]}
        if c["grad"]:
            s["dy"] = normal(n, d, dtype=s["out"], std=1e-3)
    elif c["op"] == "clip":
        shapes = _shapes(c)
        room = {t: sum(math.prod(s) for s in shapes if _grad_type(c, s) == t) for t in (F32, BF16)}
        flat = {t: torch.empty(k, dtype=t, device=dev) for t, k in room.items() if k}
        at, grads, square = {F32: 0, BF16: 0}, [], 0.0
        for i, shape in enumerate(shapes):
            t, k = _grad_type(c, shape), math.prod(shape)
            x = flat[t][at[t]:at[t] + k]
            std = 10.0 ** (-2 - i % 3)  # layers differ in scale
            step = 1 << 28
            for j in range(0, k, step):
                x[j:j + step] = normal(min(step, k - j), dtype=t, std=std)
            square += k * std * std
            grads.append(x.view(shape))
            at[t] += k
        # A pass leaves its gradients at the threshold. A threshold that falls by
        # 2^-12 a pass keeps every pass a clipping one where the first is.
        s = {"flat": [flat[t] for t in (F32, BF16) if t in flat], "grads": grads,
             "bound": c["bound"] * math.sqrt(square), "fall": 1 - 2.0 ** -12 if c["bound"] < 1 else 1.0}
    else:
        h, d, p = c["heads"], c["d"], c["prefix"]
        s = {"h": h, "slopes": _slopes(h, dev), "prefix": normal(p, 3 * h * d)}
        if c["op"] == "score":
            lens = torch.tensor(_lengths(c), device=dev)
            first = lens.cumsum(0) - lens
            # for each packed row, the row at which its sequence begins
            s["starts"] = torch.repeat_interleave(first, lens).to(torch.int32)
            s["qkv"] = normal(s["starts"].numel(), 3 * h * d)
        else:
            b, slots = c["count"], c["slots"]
            s["qkv"] = normal(b, 3 * h * d)
            s["cache"] = normal(b, slots, 2, h, d)
            s["held"] = torch.tensor(_held(c), dtype=torch.int32, device=dev)
    return {"op": c["op"], **s}


# -- one pass ---------------------------------------------------------------
def run(s):
    return {"embed": _run_embed, "clip": _run_clip, "score": _run_score, "decode": _run_decode}[s["op"]](s)


def _run_embed(s):
    if own:
        from photon_amd.ops.embedding import embedding

        y = embedding(s["ids"], s["table"], scale=s["scale"], out_dtype=s["out"])
        if "dy" not in s:
            return {"out": y}
        return {"out": y.detach(), "grad": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    table = s["table"].detach()
    y = {"out": (table[s["ids"]].float() * s["scale"]).to(s["out"])}
    if "dy" in s:
        grad = torch.zeros(table.shape, dtype=F32, device=table.device)
        y["grad"] = grad.index_add_(0, s["ids"], s["dy"].float()).mul_(s["scale"]).to(table.dtype)
    return y


def _run_clip(s):
    bound = s["bound"]
    s["bound"] *= s["fall"]
    if own:
        from photon_amd.ops.clip import clip_grads_

        total, norms = clip_grads_(s["grads"], bound)
    else:
        norms = torch.stack([g.float().square().sum() for g in s["grads"]]).sqrt()
        total = norms.square().sum().sqrt()
        share = (bound / (total + 1e-6)).clamp(max=1.0)
        [g.copy_(g.float() * share) for g in s["grads"]]
    return {"total": total, "norms": norms, "grads": s["flat"]}


def _split(qkv, h):
    """[rows, 3 * h * d] as q, k and v of [h, rows, d] in 32 bits."""
    return qkv.float().view(qkv.shape[0], 3, h, -1).permute(1, 2, 0, 3).unbind(0)


def _run_score(s):
    if own:
        from photon_amd.ops.prefix_attention import prefix_attention_qkv

        return {"out": prefix_attention_qkv(s["qkv"], s["prefix"], s["h"], s["slopes"], s["starts"])}
    q, k, v = _split(s["qkv"], s["h"])
    _, pk, pv = _split(s["prefix"], s["h"])
    p, t = pk.shape[1], q.shape[1]
    row = torch.arange(t, device=q.device)
    past = torch.arange(p, device=q.device)
    slope = s["slopes"].view(-1, 1, 1)
    r = 1.0 / math.sqrt(q.shape[-1])
    # a query's distance to each key of the prefix, and to the packed rows
    far = (p + row - s["starts"]).view(-1, 1) - past
    near = row.view(-1, 1) - row
    seen = (near >= 0) & (row >= s["starts"].view(-1, 1))
    a = torch.matmul(q, pk.transpose(1, 2)) * r - slope * far
    b = (torch.matmul(q, k.transpose(1, 2)) * r - slope * near).masked_fill(~seen, -math.inf)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    a, b = torch.exp(a - top), torch.exp(b - top)
    o = torch.matmul(a, pv) + torch.matmul(b, v)
    o = o / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
    return {"out": o.transpose(0, 1).reshape(t, -1).to(BF16)}


def _run_decode(s):
    if own:
        from photon_amd.ops.prefix_attention import prefix_attention_decode

        out = prefix_attention_decode(s["qkv"], s["prefix"], s["h"], s["slopes"], s["cache"], s["held"])
        return {"out": out, "cache": s["cache"]}
    h, cache, held = s["h"], s["cache"], s["held"].long()
    n, slots = cache.shape[:2]
    q, k, v = s["qkv"].view(n, 3, h, -1).unbind(1)
    each = torch.arange(n, device=q.device)
    cache[each, held] = torch.stack([k, v], 1)
    q = q.float()
    _, pk, pv = _split(s["prefix"], h)
    ck, cv = cache.float().unbind(2)  # [n, slots, h, d]
    p = pk.shape[1]
    slope = s["slopes"].view(1, -1, 1)
    r = 1.0 / math.sqrt(q.shape[-1])
    slot = torch.arange(slots, device=q.device)
    far = (p + held.view(-1, 1)) - torch.arange(p, device=q.device)
    near = (held.view(-1, 1) - slot).view(n, 1, slots)
    a = torch.matmul(q.transpose(0, 1), pk.transpose(1, 2)).transpose(0, 1) * r - slope * far.view(n, 1, p)
    b = ((q.unsqueeze(1) * ck).sum(-1).transpose(1, 2) * r - slope * near).masked_fill(near < 0, -math.inf)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    a, b = torch.exp(a - top), torch.exp(b - top)
    o = torch.matmul(a.transpose(0, 1), pv).transpose(0, 1) + (b.transpose(1, 2).unsqueeze(-1) * cv).sum(1)
    o = o / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
    return {"out": o.reshape(n, -1).to(BF16), "cache": cache}


# -- the same in 64 bits ----------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        if c["op"] == "embed":
            table = s["table"].detach()
            r = {"out": torch.index_select(table, 0, s["ids"]).double() * s["scale"]}
            if "dy" in s:
                g = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
                # sorted by id, a part at a time
                ids, order = torch.sort(s["ids"])
                for i in range(0, ids.numel(), 1 << 16):
                    part = order[i:i + (1 << 16)]
                    g.index_put_((ids[i:i + (1 << 16)],), s["dy"][part].double() * s["scale"], accumulate=True)
                r["grad"] = g
            return r
        if c["op"] == "clip":
            squares = [math.fsum(float(x.double().pow(2).sum()) for x in g.reshape(-1).split(1 << 28)) for g in s["grads"]]
            total = math.sqrt(math.fsum(squares))
            share = min(1.0, s["bound"] / (total + 1e-6))
            norms = torch.tensor([math.sqrt(x) for x in squares], dtype=torch.float64, device="cuda")
            return {"total": torch.tensor(total, dtype=torch.float64, device="cuda"), "norms": norms,
                    "grads": [f.double().mul_(share) for f in s["flat"]]}
        h, d, p = c["heads"], c["d"], c["prefix"]
        before = s["prefix"].view(p, 3, h, d)
        new = s["qkv"].view(-1, 3, h, d)
        slope = s["slopes"].double()

        def attend(q, k, v):
            """The last rows of k and v are q's own: [n, h, d] of [m, h, d]."""
            n, m = q.shape[0], k.shape[0]
            gap = (torch.arange(m - n, m, device=q.device).view(-1, 1) - torch.arange(m, device=q.device)).double()
            out = []
            for i in range(h):
                w = q[:, i].double() @ k[:, i].double().T / math.sqrt(d) - slope[i] * gap
                w = torch.softmax(torch.where(gap < 0, torch.full_like(w, -math.inf), w), -1)
                out.append(w @ v[:, i].double())
            return torch.cat(out, -1)

        if c["op"] == "score":
            outs, at = [], 0
            for n in _lengths(c):
                x = new[at:at + n]
                outs.append(attend(x[:, 0], torch.cat([before[:, 1], x[:, 1]]), torch.cat([before[:, 2], x[:, 2]])))
                at += n
            return {"out": torch.cat(outs)}
        outs, cache = [], s["cache"].clone()
        for i, n in enumerate(_held(c)):
            cache[i, n] = new[i, 1:]
            k, v = torch.cat([before[:, 1:], cache[i, :n + 1]]).unbind(1)
            outs.append(attend(new[i:i + 1, 0], k, v))
        return {"out": torch.cat(outs), "cache": None}
