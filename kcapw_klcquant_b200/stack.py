"""A stack of MoE blocks with the executor's RMSNorm and residual add between them.

The reference runs each transformer layer as attention, then
``post = rms_norm(hidden, ...)``, ``moe_out = router.route(..., post, ...)``
and ``hidden += moe_out`` (streamed_transformer_executor.py:231-275, rms_norm
at streamed_attention.py:27-28).  :class:`MoeStack` is the MoE half of that
layer loop over many layers and a whole batch of tokens at once:

    normed = rms_norm(hidden, norm[0])
    for every layer L:
        hidden = hidden + moe_L(normed)             # the combine adds the residual
        normed = rms_norm(hidden, norm[L + 1])      # ... and normalises for layer L+1

with the residual add and the next layer's norm fused into each layer's
combine kernel, so a layer is one MoE call.  With ``fuse_router`` the next
layer's router also runs in that call (the same kernels; a layer after the
first is then one experts-and-combine call on routing its predecessor already
computed).  Layers are :class:`MoeLayer` (one GPU) or
:class:`ExpertParallelMoe` with the peer-memory exchange (experts sharded over
the GPUs of a node); both are free of host synchronisation, so
:meth:`MoeStack.capture` records a whole decode step of all layers as one CUDA
graph and :meth:`MoeStack.replay` runs it.

With ``attention`` the stack runs whole layers as the executor does
(streamed_transformer_executor.py:231-275), over a :class:`PagedKvCache`:

    for every layer L:
        hidden = hidden + attention_L(rms_norm(hidden, input_norm[L]))
        hidden = hidden + moe_L(rms_norm(hidden, norm[L]))

:meth:`MoeStack.prompt` takes whole packed prompts, :meth:`MoeStack.step` one
token for every row of the cache.  Pages are taken and lengths advanced on the
device, so a captured step can be replayed token after token.
"""
from __future__ import annotations

import torch

from .moe import MoeLayer, as_bf16, rms_norm


class MoeStack:
    """MoE layers with RMSNorm weights ``norm_weights[L]`` (bf16 [H]) applied to each layer's input."""

    def __init__(self, layers: list, norm_weights: list[torch.Tensor], eps: float = 1e-5, precision: str = "bf16",
                 fuse_router: bool = False, attention: list | None = None, input_norm_weights: list[torch.Tensor] | None = None,
                 cache=None, rope: tuple[torch.Tensor, torch.Tensor] | None = None):
        if len(norm_weights) != len(layers):
            raise ValueError("one RMSNorm weight per layer")
        if attention is not None:
            if input_norm_weights is None or cache is None or rope is None:
                raise ValueError("attention needs input_norm_weights, a cache and the rotary tables")
            if len(attention) != len(layers) or len(input_norm_weights) != len(layers):
                raise ValueError("one attention layer and one input norm per layer")
            if cache.pool.shape[0] < len(layers):
                raise ValueError("the cache has fewer layers than the stack")
            width = input_norm_weights[0].numel()
            for layer, moe, norms in zip(attention, layers, zip(input_norm_weights, norm_weights)):
                layer.check_cache(cache, rope)
                moe_width = moe.hidden if isinstance(moe, MoeLayer) else moe.backend.local.hidden
                if {layer.qkv_weight.shape[1], moe_width, *(w.numel() for w in norms)} != {width}:
                    raise ValueError(f"attention, MoE layers and norms must all have {width} columns")
            if fuse_router:
                raise ValueError("fuse_router routes the next layer's input before its attention: not with attention")
        self.layers = list(layers)
        dev = self._device()
        self.norm_weights = [as_bf16(w, dev) for w in norm_weights]
        self.eps = float(eps)
        self.precision = precision
        self.fuse_router = bool(fuse_router)
        self.attention = None if attention is None else list(attention)
        self.cache = cache
        if attention is not None:
            self.input_norm_weights = [as_bf16(w, dev) for w in input_norm_weights]
            self.rope = tuple(t.to(device=dev, dtype=torch.float32).contiguous() for t in rope)
            # one token per step and row; rows that sit out: set_active
            self._add = torch.ones(cache.rows, dtype=torch.int32, device=dev)
            self._rows = torch.arange(cache.rows, dtype=torch.int32, device=dev)
        self._graph = None
        self._static_in = None
        self._static_out = None

    def _device(self) -> torch.device:
        first = self.layers[0]
        return first.device if isinstance(first, MoeLayer) else first.backend.device

    def step(self, hidden: torch.Tensor) -> torch.Tensor:
        """One pass of this rank's tokens bf16 [T, H] through every layer (with attention: one token for every row of
        the cache, T = its rows)."""
        if self.attention is not None:
            return self._decode_step(hidden)
        normed = rms_norm(hidden, self.norm_weights[0], self.eps)
        n = len(self.layers)
        idx = w = None  # routing of this layer, when the previous layer's combine computed it
        for li, layer in enumerate(self.layers):
            last = li + 1 == n
            nxt = None if last else (self.norm_weights[li + 1], self.eps)
            nrouter = None if (last or not self.fuse_router) else self.layers[li + 1]
            ep = not isinstance(layer, MoeLayer)
            if idx is None:
                if last:
                    y, _ = layer.forward(normed, precision=self.precision, residual=hidden)
                elif not ep:
                    y, rb = layer.forward(normed, precision=self.precision, residual=hidden, next_norm=nxt, next_router=nrouter)
                    normed, idx, w = rb.normed, rb.next_indices, rb.next_weights
                else:
                    y, rb, normed = layer.forward(normed, precision=self.precision, residual=hidden, next_norm=nxt,
                                                  next_router=nrouter)
                    idx, w = rb.next_indices, rb.next_weights
            elif last:
                if ep:
                    y, _ = layer.step_routed(normed, idx, w, hidden, None, None, self.precision)
                else:
                    y, _ = layer.experts_forward(normed, idx, w, precision=self.precision, residual=hidden)
            else:
                y, rb = (layer.step_routed(normed, idx, w, hidden, nxt, nrouter, self.precision) if ep
                         else layer.experts_step(normed, idx, w, hidden, nxt, nrouter, self.precision))
                normed, idx, w = rb.normed, rb.next_indices, rb.next_weights
            hidden = y
        return hidden

    def set_active(self, active: torch.Tensor) -> None:
        """Which rows of the cache take part in :meth:`step` (bool [rows]); the others' keys and lengths stay as they are
        and their outputs mean nothing.  May be changed between replays of a captured step."""
        on = active.to(device=self._add.device, dtype=torch.bool)
        if on.shape != self._add.shape:
            raise ValueError(f"active must have {self._add.numel()} elements")
        self._add.copy_(on)
        self._rows.copy_(torch.where(on, torch.arange(on.numel(), dtype=torch.int32, device=on.device), -1))

    def _layers(self, hidden: torch.Tensor, attend) -> torch.Tensor:
        """Whole layers; ``attend(layer, normed)`` is the attention of one."""
        normed = rms_norm(hidden, self.input_norm_weights[0], self.eps)
        n = len(self.layers)
        for li, layer in enumerate(self.layers):
            hidden = hidden + attend(li, normed)
            post = rms_norm(hidden, self.norm_weights[li], self.eps)
            nxt = None if li + 1 == n else (self.input_norm_weights[li + 1], self.eps)
            if nxt is None:
                hidden, _ = layer.forward(post, precision=self.precision, residual=hidden)
            elif isinstance(layer, MoeLayer):
                hidden, rb = layer.forward(post, precision=self.precision, residual=hidden, next_norm=nxt)
                normed = rb.normed
            else:
                hidden, _, normed = layer.forward(post, precision=self.precision, residual=hidden, next_norm=nxt)
        return hidden

    def _check_hidden(self, hidden: torch.Tensor) -> None:
        """Before lengths advance: a call that raises later would leave rows with lengths that have no keys."""
        width, dev = self.input_norm_weights[0].numel(), self.cache.device
        if hidden.dim() != 2 or hidden.shape[1] != width or hidden.dtype != torch.bfloat16 or hidden.device != dev:
            raise ValueError(f"hidden must be bf16 [tokens, {width}] on {dev}, got {hidden.dtype} {tuple(hidden.shape)} on {hidden.device}")

    def _decode_step(self, hidden: torch.Tensor) -> torch.Tensor:
        cache = self.cache
        self._check_hidden(hidden)
        if hidden.shape[0] != cache.rows:
            raise ValueError(f"a step takes one token for each of the cache's {cache.rows} rows")
        positions = cache.lens.clone()
        cache.reserve(self._add)
        return self._layers(hidden, lambda li, x: self.attention[li].decode(x, cache, li, self.rope, positions, self._rows))

    def prompt(self, hidden: torch.Tensor, cu_seqlens: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """Whole prompts through every layer: packed tokens bf16 [T, H], sequence b the rows ``cu_seqlens[b]:cu_seqlens[b + 1]``
        (int32 on the device), into the empty cache rows ``rows`` int32 [B], each listed once.  Returns [T, H].

        A row that holds keys already, is listed twice or does not exist keeps what it has, its sequence's outputs mean nothing,
        and ``cache.check()`` reports it, as it does when the pages do not suffice."""
        if self.attention is None:
            raise RuntimeError("the stack has no attention layers")
        self._check_hidden(hidden)
        T, dev = int(hidden.shape[0]), hidden.device
        if rows.dim() != 1 or rows.shape[0] == 0 or cu_seqlens.shape != (rows.shape[0] + 1,):
            raise ValueError("rows must not be empty and cu_seqlens have one element more")
        if rows.dtype != torch.int32 or cu_seqlens.dtype != torch.int32 or rows.device != dev or cu_seqlens.device != dev:
            raise ValueError(f"rows and cu_seqlens must be int32 on {dev}")
        # by comparison, not by index: a row that does not exist reserves nothing (and is reported), where an index would trap
        here = torch.arange(self.cache.rows, dtype=torch.int32, device=dev)[:, None] == rows
        # positions count from 0: in a row with keys they would fall on those, on pages it shares among them.  reserve reports a
        # negative growth and leaves the row; its tokens become padding
        times = here.sum(1, dtype=torch.int32)
        taken = (times > 0) & ((self.cache.lens != 0) | (times > 1))
        grow = (here * (cu_seqlens[1:] - cu_seqlens[:-1])).sum(1, dtype=torch.int32)
        self.cache.reserve(torch.where(taken, -1, grow))
        rows = torch.where((here & taken[:, None]).any(0), -1, torch.where(rows < 0, -2, rows))  # -2: reported, -1: padding
        # tokens before the first and past the last sequence are padding: row -1
        seq = torch.bucketize(torch.arange(T, dtype=torch.int32, device=dev), cu_seqlens[1:], right=True, out_int32=True)
        inside = seq < rows.shape[0]
        at = seq.clamp(max=rows.shape[0] - 1).long()
        positions = torch.arange(T, dtype=torch.int32, device=dev) - cu_seqlens[at]
        token_rows = torch.where(inside & (positions >= 0), rows[at], -1).to(torch.int32)
        return self._layers(hidden, lambda li, x: self.attention[li].prompt(x, self.cache, li, self.rope, cu_seqlens, positions,
                                                                            token_rows))

    def capture(self, example: torch.Tensor, warmup: int = 2) -> None:
        """Record :meth:`step` on a static input buffer shaped like ``example`` as a CUDA graph.

        With attention the warm-up steps need pages for ``warmup`` tokens in every active row; tables and lengths are put
        back behind them."""
        self._static_in = example.clone()
        state = None if self.attention is None else self.cache.snapshot()  # warm-up steps leave the sequences as they were
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warmup):  # workspaces sized and kernels loaded outside the capture
                self.step(self._static_in)
        torch.cuda.current_stream().wait_stream(side)
        if state is not None:
            self.cache.restore(state)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._static_out = self.step(self._static_in)
        self._graph = g

    def replay(self, hidden: torch.Tensor | None = None) -> torch.Tensor:
        """Run the captured step (after copying ``hidden`` into its input buffer); returns its output buffer."""
        if self._graph is None:
            raise RuntimeError("capture() first")
        if hidden is not None:
            self._static_in.copy_(hidden, non_blocking=True)
        self._graph.replay()
        return self._static_out

    def release(self) -> None:
        """Drop the captured graph (before the exchange handles of the layers are closed)."""
        self._graph = None
        self._static_out = None
