"""Attention of a batch of sequences that share a long prefix, with ALiBi.

Scoring the answers to one question, or the questions that share their
examples, runs the same first P tokens again and again. Here their keys and
values are computed once (the packed Wqkv output of one pass over the prefix
is kept per layer) and every sequence attends them together with its own
tokens:

* :func:`prefix_attention_qkv` — all own tokens of all sequences, packed row
  behind row without padding;
* :func:`prefix_attention_decode` — one new token for each sequence, whose
  earlier own keys and values are in a cache of fixed slots.

Position i of a sequence's own tokens is position P + i of its text: the bias
is -slope * (P + i - j) for key j of the prefix and -slope * (i - j) for its
own key j <= i. Both run without gradients (and the kernels refuse
forward-mode tangents).

A key whose weight is below 2^-150 of the row's largest adds nothing; on a GPU
its value is then not looked at, so a NaN in it need not show. The kernels
take scores and biases up to 2^28 (their weights are differences of fp32 values,
which are whole numbers beyond 2^24).
"""

from __future__ import annotations

import math

import torch

from . import hip_ext, use_hip


def sequence_starts(lengths, device=None) -> torch.Tensor:
    """For each row of the packed own tokens the row at which its sequence
    begins (int32), from the sequences' lengths (zero is allowed)."""
    lens = torch.as_tensor(list(lengths), dtype=torch.int64)
    if lens.dim() != 1 or bool((lens < 0).any()):
        raise ValueError("sequence_starts: lengths must be whole numbers >= 0")
    first = lens.cumsum(0) - lens
    starts = torch.repeat_interleave(first, lens).to(torch.int32)
    return starts.to(device) if device is not None else starts


def _check(name, qkv, prefix_qkv, n_heads, slopes, info, info_name):
    """Of the plain path; the extension checks the same with the same words."""
    if torch.is_grad_enabled() and any(
            t.requires_grad for t in (qkv, prefix_qkv, slopes)):
        raise RuntimeError(f"{name}: no backward pass; call it under torch.no_grad()")
    if n_heads <= 0 or qkv.dim() != 2 or qkv.shape[1] % (3 * n_heads):
        raise ValueError(f"{name}: qkv must be [rows, 3 * n_heads * d], got "
                         f"{tuple(qkv.shape)} for {n_heads} heads")
    if prefix_qkv.dim() != 2 or prefix_qkv.shape[1] != qkv.shape[1]:
        raise ValueError(f"{name}: prefix_qkv must be [P, {qkv.shape[1]}], got "
                         f"{tuple(prefix_qkv.shape)}")
    if prefix_qkv.dtype != qkv.dtype or prefix_qkv.device != qkv.device:
        raise ValueError(f"{name}: prefix_qkv must have qkv's dtype and device")
    if slopes.shape != (n_heads,):
        raise ValueError(f"{name}: slopes must be [{n_heads}], got {tuple(slopes.shape)}")
    if info.dtype != torch.int32 or info.shape != (qkv.shape[0],):
        raise ValueError(f"{name}: {info_name} must be int32 [{qkv.shape[0]}], got "
                         f"{info.dtype} {tuple(info.shape)}")
    if info.device != qkv.device:
        raise ValueError(f"{name}: {info_name} must be on {qkv.device}")


def prefix_attention_qkv(
    qkv: torch.Tensor,
    prefix_qkv: torch.Tensor,
    n_heads: int,
    slopes: torch.Tensor,
    starts: torch.Tensor,
    impl: str = "flash",
) -> torch.Tensor:
    """Attention of packed rows over a shared prefix and over themselves.

    qkv: [T, 3*H*d] packed Wqkv output of the own tokens of all sequences;
    prefix_qkv: [P, 3*H*d] of the prefix (its q part is not read; P may be 0);
    starts: [T] int32 from :func:`sequence_starts`. Returns [T, H*d].

    impl="flash" on a GPU is the HIP kernel (bf16, d 64 or 128); elsewhere,
    and for impl="torch", plain torch in fp32."""
    if impl == "flash" and use_hip(qkv):
        return hip_ext().prefix_attention(qkv, prefix_qkv, n_heads, slopes, starts)
    _check("prefix_attention_qkv", qkv, prefix_qkv, n_heads, slopes, starts, "starts")
    return _plain(qkv, prefix_qkv, n_heads, slopes, starts)


def prefix_attention_decode(
    qkv: torch.Tensor,
    prefix_qkv: torch.Tensor,
    n_heads: int,
    slopes: torch.Tensor,
    cache: torch.Tensor,
    held: torch.Tensor,
    impl: str = "flash",
) -> torch.Tensor:
    """One new token for each of B sequences: its key and value go to the
    cache, its query attends the prefix, the cached own keys and itself.

    qkv: [B, 3*H*d] of the new tokens; cache: [B, slots, 2, H, d] of the
    sequences' own keys and values (layer by layer one such tensor); held:
    [B] int32, how many slots each sequence has filled. Slot ``held`` is
    written, later slots are not read; the caller counts ``held`` up once a
    step, after its last layer. Returns [B, H*d].

    A sequence without a free slot raises IndexError on the CPU; on the GPU
    its output is NaN and its cache stays."""
    if impl == "flash" and use_hip(qkv):
        return hip_ext().prefix_attention_decode(
            qkv, prefix_qkv, n_heads, slopes, cache, held)
    name = "prefix_attention_decode"
    _check(name, qkv, prefix_qkv, n_heads, slopes, held, "held")
    want = (2, n_heads, qkv.shape[1] // (3 * n_heads))
    if cache.dim() != 5 or cache.shape[0] != qkv.shape[0] or tuple(cache.shape[2:]) != want:
        raise ValueError(f"{name}: cache must be [{qkv.shape[0]}, slots, "
                         f"{', '.join(map(str, want))}], got {tuple(cache.shape)}")
    if cache.dtype != qkv.dtype or cache.device != qkv.device:
        raise ValueError(f"{name}: cache must have qkv's dtype and device")
    if cache.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError(f"{name}: the cache was made in inference mode and "
                           "cannot be written outside of it")
    B = qkv.shape[0]
    rows, slots = held.long(), cache.shape[1]
    if bool(((rows < 0) | (rows >= slots)).any()):
        raise IndexError(f"{name}: a sequence has no free slot of {slots}")
    new = qkv.reshape(B, 3, n_heads, want[2])
    cache[torch.arange(B, device=qkv.device), rows] = new[:, 1:]
    # every sequence's filled slots as packed rows; the last row is the query
    filled = torch.arange(slots, device=qkv.device) <= rows.view(-1, 1)
    kv = cache[filled]  # [T, 2, H, d]
    ends = (rows + 1).cumsum(0) - 1
    packed = torch.cat([torch.zeros_like(kv[:, :1]), kv], 1)
    packed[ends, 0] = new[:, 0]
    starts = sequence_starts((rows + 1).tolist(), qkv.device)
    return _plain(packed.flatten(1), prefix_qkv, n_heads, slopes, starts)[ends]


def _plain(qkv, prefix_qkv, n_heads, slopes, starts):
    """The definition, in fp32 (fp64 stays)."""
    T, P = qkv.shape[0], prefix_qkv.shape[0]
    wide = torch.promote_types(qkv.dtype, torch.float32)
    d = qkv.shape[1] // (3 * n_heads)
    q, k, v = qkv.to(wide).reshape(T, 3, n_heads, d).permute(1, 2, 0, 3).unbind(0)
    _, pk, pv = prefix_qkv.to(wide).reshape(P, 3, n_heads, d).permute(1, 2, 0, 3).unbind(0)
    row = torch.arange(T, device=qkv.device)
    first = starts.long()
    own = row - first
    far = (P + own).view(-1, 1) - torch.arange(P, device=qkv.device)
    near = row.view(-1, 1) - row
    seen = (near >= 0) & (row >= first.view(-1, 1))
    slope = slopes.to(qkv.device, wide).view(-1, 1, 1)
    scale = 1.0 / math.sqrt(q.shape[-1])
    w = torch.cat([
        q @ pk.transpose(1, 2) * scale - slope * far,
        (q @ k.transpose(1, 2) * scale - slope * near).masked_fill(~seen, -math.inf),
    ], -1)
    # A weight of zero does not hide an infinity or NaN: values that are not
    # finite are taken out and added for the rows that see them (a NaN as an
    # infinity of either sign). On a GPU without looking whether there are any.
    finite = v.isfinite()
    every = v.device.type == "cpu" and bool(finite.all())
    o = torch.softmax(w, -1) @ torch.cat([pv, v.where(finite, 0.0)], 1)
    if not every:
        sight = seen.to(wide)
        for sign in (math.inf, -math.inf):
            bad = (v.isnan() | (v == sign)).to(wide)
            o = torch.where(sight @ bad > 0, o + sign, o)
    return o.transpose(0, 1).reshape(T, -1).to(qkv.dtype)
