"""Answering from a trained feed-forward net, with weights in 4 or 8 bits.

`make_infer(net, static, state, weights="e2m1", rows="f32")` lays the live
edges of a TOPOLOGICAL net out once, grouped by destination, level by level,
with their weights in MX blocks of 32 in-edges of one unit (or "f32"). The
returned function runs the forward for a batch of any size, one sample
included: `infer(inputs)` with inputs (B, num_inputs) gives (B, num_outputs)
float32, the values the training step's forward leaves in the output units
(src/plastax/phases.py:972-1015). A unit that the forward never applies (level
0 and no input, or pruned) keeps its activation: the state's, as the streaming
step reads it, or 0 for a net with a `batch_reduction`, whose batched step
starts from rows of zeros. A ReLU keeps what is not a number, which the step's
makes 0. One kernel a level does the product, the activation and, with `rows`
an MX format, the quantisation of the level's rows for the next one; the
outputs are always float32.

The layout is a snapshot (of those activations too): later steps on `state` do
not change it.
"""

from __future__ import annotations

import dataclasses

import numpy as np
import torch

from plastax_b200 import mx
from plastax_b200.state import NetworkState, NetworkStatic, live_unit_mask
from plastax_b200.traits import Network
from plastax_b200.types import ACTIVATION, LEVEL, Propagation


@dataclasses.dataclass(frozen=True)
class _Stage:
    """One product of a level: into the rows buffer, or into the outputs."""

    conns: mx.MxConns
    activation: str
    to_outputs: bool


class InferFn:
    """A built forward (see the module's notes). It holds the layout only: a
    call allocates its rows on the current stream, so calls on different
    streams or in captured graphs do not share buffers."""

    def __init__(self, net: type[Network], static: NetworkStatic, state: NetworkState, weights: str,
                 rows: str) -> None:
        if net.propagation is Propagation.PIPELINE:
            raise ValueError("make_infer: a PIPELINE net carries recurrent state between steps; its forward is the "
                             "step itself (make_step)")
        if net.forward_pass.combine.lowered() != "sum":
            raise NotImplementedError("make_infer lowers the linear (sum) forward only")
        if static.num_shards > 1:
            raise NotImplementedError("make_infer under Scheme-A has no engine lowering (one device holds the arena)")
        for what, fmt in (("weights", weights), ("rows", rows)):
            if fmt not in (*mx.FORMATS, "f32"):
                raise ValueError(f"make_infer: unknown {what} {fmt!r}: one of f32, {', '.join(mx.FORMATS)}")
        if not static.input_ids or not static.output_ids:
            raise ValueError("make_infer: the net needs inputs and outputs")
        for what, ids in (("input", static.input_ids), ("output", static.output_ids)):
            if len(set(ids)) != len(ids):
                raise ValueError(f"make_infer: an {what} unit is listed twice")
        self.weights, self.rows = weights, rows
        self.device = dev = state.units[LEVEL.name].device
        self.num_inputs, self.num_outputs = len(static.input_ids), len(static.output_ids)
        n = static.num_units
        level = state.units[LEVEL.name].long()
        live = torch.ones(n, dtype=torch.bool, device=dev)
        if live_unit_mask(state.units) is not None:
            live &= live_unit_mask(state.units)
        is_input = torch.zeros(n, dtype=torch.bool, device=dev)
        is_input[list(static.input_ids)] = True
        is_output = torch.zeros(n, dtype=torch.bool, device=dev)
        is_output[list(static.output_ids)] = True
        src, dst, w = [], [], []
        for b in state.conns:
            f, t = b["from_id"].long(), b["to_id"].long()
            keep = (b["dead"] == 0) & (f >= 0) & (f < n) & (t >= 0) & (t < n)  # as the step's kernels take them
            f, t = f[keep], t[keep]
            # an edge that is not to a deeper level arrives after its destination's apply
            deeper = (level[t] > level[f]) & ~is_input[t]
            src.append(f[deeper]), dst.append(t[deeper]), w.append(b["weight"][keep][deeper])
        src, dst, w = torch.cat(src), torch.cat(dst), torch.cat(w)
        # the units that a level's apply writes; the others keep what they hold
        applied = live & ~is_input & (level >= 1) & (level <= len(state.conns))
        held = state.units[ACTIVATION.name].to(torch.float32)
        if net.batch_reduction is not None:
            held = torch.zeros_like(held)
        # compact rows: the inputs, the sources that no apply writes, then every other unit that is a source
        is_source = torch.zeros(n, dtype=torch.bool, device=dev)
        is_source[src] = True
        inputs = torch.tensor(static.input_ids, dtype=torch.int64, device=dev)
        still = torch.nonzero(is_source & ~is_input & ~applied).flatten()
        moving = torch.nonzero(is_source & applied).flatten()
        order = torch.cat([inputs, still, moving])
        row_of = torch.full((n,), -1, dtype=torch.int64, device=dev)
        row_of[order] = torch.arange(order.numel(), device=dev)
        self.num_rows, self.num_still = order.numel(), still.numel()
        self.input_rows, self.still_rows = row_of[inputs], row_of[still]
        self.still_values = held[still][:, None]
        outputs = torch.tensor(static.output_ids, dtype=torch.int64, device=dev)
        out_of = torch.full((n,), -1, dtype=torch.int64, device=dev)
        out_of[outputs] = torch.arange(outputs.numel(), device=dev)
        # an output that is an input answers with the input itself, one that no apply writes with what it holds
        pos = torch.full((n,), -1, dtype=torch.int64, device=dev)
        pos[inputs] = torch.arange(inputs.numel(), device=dev)
        as_input = pos[outputs]
        self.out_from_input = [(i, int(p)) for i, p in enumerate(as_input.tolist()) if p >= 0]
        self.out_still = torch.nonzero(~is_input[outputs] & ~applied[outputs]).flatten()
        self.out_still_values = held[outputs[self.out_still]][:, None]
        fp = net.forward_pass
        out_act = fp.output_activation or fp.activation
        rows_src = row_of[src].to(torch.int32)
        self.stages: list[_Stage] = []
        for lv in range(1, len(state.conns) + 1):
            here = applied & (level == lv)
            for sel, act, index, to_outputs in ((here & is_source & ~is_output, fp.activation, row_of, False),
                                                (here & is_source & is_output, out_act, row_of, False),
                                                (here & is_output, out_act, out_of, True)):
                ids = torch.nonzero(sel).flatten()
                if ids.numel() == 0:
                    continue
                conns = mx.MxConns.from_edges(rows_src, dst, w, ids.to(torch.int32), weights=weights)
                conns = dataclasses.replace(conns, units=index[ids].to(torch.int32).contiguous())
                self.stages.append(_Stage(conns, act, to_outputs))

    @property
    def num_edges(self) -> int:
        """Edges laid out (an output that is also a source has its own twice)."""
        return sum(s.conns.num_edges for s in self.stages)

    def __call__(self, inputs) -> torch.Tensor:
        dev = self.device
        if not isinstance(inputs, torch.Tensor):
            inputs = torch.from_numpy(np.ascontiguousarray(inputs, np.float32))
        if inputs.dim() != 2 or inputs.shape[1] != self.num_inputs:
            raise ValueError(f"infer: expected inputs (batch, {self.num_inputs}), got {tuple(inputs.shape)}")
        with mx._on(dev):
            x = inputs.to(dev, dtype=torch.float32)
            batch = x.shape[0]
            if self.rows == "f32":
                rows = torch.empty((self.num_rows, batch), dtype=torch.float32, device=dev)
                rows[:self.num_inputs] = x.t()
                rows[self.num_inputs:self.num_inputs + self.num_still] = self.still_values
            else:
                rows = mx.MxRows.empty(self.num_rows, batch, self.rows, dev)
                mx.mx_quantize(x.t(), self.rows, ids=self.input_rows, out=rows)
                if self.num_still:
                    mx.mx_quantize(self.still_values.expand(-1, batch), self.rows, ids=self.still_rows, out=rows)
            out = torch.zeros((self.num_outputs, batch), dtype=torch.float32, device=dev)
            for s in self.stages:
                mx.mx_product(s.conns, rows, activation=s.activation, out=out if s.to_outputs else rows)
            if self.out_still.numel():
                out.index_copy_(0, self.out_still, self.out_still_values.expand(-1, batch))
            for i, p in self.out_from_input:
                out[i] = x[:, p]
            return out.t()


def make_infer(net: type[Network], static: NetworkStatic, state: NetworkState, *, weights: str = "e2m1",
               rows: str = "f32") -> InferFn:
    """Build the forward of a trained feed-forward net for answering: `infer(inputs) -> outputs`.

    `weights`: "e2m1" (4 bits), "e4m3", "e5m2" (8 bits) or "f32"; `rows`: the
    form of the activations between levels, "f32" or an MX format."""
    return InferFn(net, static, state, weights, rows)


__all__ = ["InferFn", "make_infer"]
