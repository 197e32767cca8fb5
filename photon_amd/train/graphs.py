"""hipGraph-captured training microbatch — streams & graphs, not a tracing
compiler (the north-star runtime design; no Triton / torch.compile).

Captures ONE fixed-shape microbatch forward+backward into a hipGraph
(torch.cuda.CUDAGraph is hipGraph on ROCm) and replays it per microbatch:
removes the per-kernel launch overhead of the ~80-kernel microbatch body.

Measured at MPT-125M/gb256/mb32: graphs 601-606k vs eager 611-616k
tokens/s, both with fp32+autocast and with bf16 master-weight mode — the
~10-16 us replay floor over 8 microbatches plus graph-pool memory effects
eat the launch-overhead win at this kernel count. Opt-in
(llm_config.use_hip_graphs); expected to pay off for smaller models or
larger grad-accum degrees.

Contract:
* input shape is fixed (microbatch_size x seq_len) — the bench/fed training
  path pads nothing and always ticks full microbatches;
* gradients ACCUMULATE into the captured .grad tensors — callers must zero
  with ``set_to_none=False`` (zero_()), never free them;
* the optimizer step and scheduler run OUTSIDE the graph (dynamic lr);
* weight VALUES may change between replays (the fed round copies new
  globals into the same parameter tensors — graph-safe).
"""

from __future__ import annotations

import torch


class GraphedMicrobatch:
    def __init__(self, model, autocast_ctx_factory, loss_div: float,
                 microbatch: int, seq_len: int, device):
        self.model = model
        self.device = device
        self.static_ids = torch.zeros(
            (microbatch, seq_len), dtype=torch.long, device=device
        )
        self.loss_div = loss_div
        self._graph = None
        self._static_loss = None
        self._autocast = autocast_ctx_factory

    def _capture(self):
        # warmup on a side stream (required before capture)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                self._zero_grads()
                with self._autocast():
                    out = self.model(self.static_ids, labels=self.static_ids)
                    loss = out["loss"] / self.loss_div
                    loss.backward()
        del out, loss
        torch.cuda.current_stream().wait_stream(s)
        self._zero_grads()
        # A live eager graph (a loss that somebody keeps) holds the parameters'
        # accumulation nodes on the stream that it ran on, and a captured
        # backward must not wait for that one. So the capture has leaves of its
        # own: other nodes over the same memory and the same gradients. But for
        # parameters with hooks, which belong to them and are captured too.
        params = {n: p for n, p in self.model.named_parameters()
                  if not (p._backward_hooks or p._post_accumulate_grad_hooks)}
        leaves = {n: torch.nn.Parameter(p.data, requires_grad=p.requires_grad)
                  for n, p in params.items()}
        for n, p in params.items():
            leaves[n].grad = p.grad
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with self._autocast():
                out = torch.func.functional_call(
                    self.model, leaves, (self.static_ids,),
                    {"labels": self.static_ids})
                loss = out["loss"] / self.loss_div
                loss.backward()
            self._static_loss = loss.detach()
        for n, p in params.items():
            if p.grad is None:
                p.grad = leaves[n].grad
        self._graph = g

    def _zero_grads(self):
        for p in self.model.parameters():
            if p.grad is not None:
                p.grad.zero_()

    def run(self, input_ids: torch.Tensor) -> torch.Tensor:
        """Replay the captured microbatch; returns the (device) loss."""
        if self._graph is None:
            self._capture()
        self.static_ids.copy_(input_ids, non_blocking=True)
        self._graph.replay()
        return self._static_loss
