"""The batched step, make_step(batch_size=B) (src/plastax/step.py:76-237).

For TOPOLOGICAL (feed-forward) nets: `StepInputs` carries (B, num_inputs)
inputs and (B, num_outputs) targets. Forward, loss and backward run per
sample against the shared connections, on unit columns laid out [N, B] (one
row of B samples per unit, csrc/batched.cu): each bucket's edges are read
once for the whole batch. The connection update is the exact batch-mean
gradient (src/plastax/phases.py:434-483). The per-sample unit columns then
reduce to the state's columns by the net's `batch_reduction`
(MeanFloatFirstRest: the batch mean of every float column), and prune and
growth run once on the reduced state, as the streaming step runs them.
`StepResult.loss` is the batch mean.

With `activation_checkpoint` ("e4m3" / "e5m2", plastax_b200/mx.py) the backward
pass and the update read the activations from 8-bit blocks that the forward's
applies leave behind; the forward and the loss stay in float32 (a ReLU keeps
what is not a number, which the plain step's makes 0). One [N, B]
float32 buffer then holds, row by row, the forward's sums, the activations
made from them in place and, once the checkpoint has them, the backward's sums
and gradients: 4 (rows) + 4 (the loss seeds) + 33/32 bytes a unit and sample
instead of 16. A row serves all of these because an edge of a TOPOLOGICAL net
goes to a deeper level and lies in the bucket of its source's level, so a
level's sums are complete before its apply. The step checks that on a state's
columns when it first sees them, and again once they were replaced or edited by
torch operations (not through `.data` or another alias: such an edit needs a
new column); the growth rule must have direction "deeper". The check reads the
host, so a step is run once on a state before it is captured, and a captured
step does not repeat it.
"""

from __future__ import annotations

import weakref

import numpy as np
import torch

from plastax_b200 import _lib
from plastax_b200 import kernels as K
from plastax_b200 import mx
from plastax_b200.state import NetworkState, NetworkStatic
from plastax_b200.step import StepFn, StepInputs, StepResult
from plastax_b200.traits import (
    DestinationThresholdPrune,
    LowestMagnitudePrune,
    MagnitudePrune,
    MSELoss,
    Network,
    SoftmaxCrossEntropyLoss,
)
from plastax_b200.types import ACTIVATION, LEVEL


class BatchedStepFn:
    """A built batched step: [N, B] unit rows plus a streaming StepFn whose
    structural phases run on the reduced state."""

    def __init__(self, net: type[Network], static: NetworkStatic, batch_size: int, device: torch.device,
                 activation_checkpoint: str | None = None) -> None:
        if activation_checkpoint is not None:
            if activation_checkpoint not in mx.CHECKPOINT_FORMATS:
                raise ValueError(f"make_step: unknown activation_checkpoint {activation_checkpoint!r}: one of "
                                 f"{', '.join(mx.CHECKPOINT_FORMATS)}")
            if net.add_conn is not None and net.add_conn.direction != "deeper":
                raise NotImplementedError("activation_checkpoint reuses a unit's row once its level is applied: the "
                                          "growth rule must have direction 'deeper'")
        if batch_size % 4 != 0 or batch_size > 1024:
            raise ValueError(f"make_step: the batched engine moves unit rows as float4: batch_size must be a "
                             f"multiple of 4 and at most 1024, got {batch_size}")
        if net.update_unit is not None or net.prune_unit is not None or net.add_unit is not None:
            raise NotImplementedError("a batched step has no unit-lifecycle lowering yet (update_unit runs per "
                                      "sample, prune_unit and add_unit on the reduced state)")
        if net.update_conn is not None and net.update_conn.kind == "upgd":
            raise NotImplementedError("a batched step has no UPGD lowering (the rule declares no exact "
                                      "per-sample / batch pair)")
        if net.forward_pass.combine.lowered() != "sum":
            raise NotImplementedError("a batched step lowers the linear (sum) forward only")
        if static.sharding is not None and static.num_shards > 1:
            raise NotImplementedError("a batched step under Scheme-A sharding has no engine lowering (its [N, B] "
                                      "partials would need a reduction per level)")
        self.net, self.static, self.dev, self.batch = net, static, device, int(batch_size)
        self.inner = StepFn(net, static, device)
        self.inner.use_mirror = False  # rows move per edge; the mirror serves the streaming sweep
        self.inner.acc_fixed = None
        self.inner.peer_reduce = False
        self.inner.ahead = False  # the structural phases run on the reduced state, in the step
        n, B = static.num_units, self.batch
        z = lambda: torch.zeros((n, B), dtype=torch.float32, device=device)  # noqa: E731
        self.acc_b = z()
        self.checkpoint = None  # the activations in 8-bit blocks; rows are then shared (see the module's notes)
        self._checked: dict[tuple[int, ...], list] = {}  # the columns that passed _check_deeper, and their versions
        bp, loss = net.backward_pass, net.loss
        if activation_checkpoint is not None:
            self.checkpoint = mx.MxRows.empty(n, B, activation_checkpoint, device, zero=True)
            self.act_b = self.acc_b
            self.grad_b = self.acc_b if bp is not None else None
        else:
            self.act_b = z()
            self.grad_b = z() if bp is not None else None
        self.seed_b = z() if loss is not None else None
        self.loss_b = torch.zeros(B, dtype=torch.float32, device=device)
        self.launches = 0
        # the [N, B] rows an update_conn reads its gradient from
        self.upd_grad_b = None
        uc = net.update_conn
        if uc is not None:
            name = uc.grad_field.name
            if bp is not None and name == bp.grad_field.name:
                self.upd_grad_b = self.grad_b
            elif loss is not None and name == loss.seed_field.name:
                self.upd_grad_b = self.seed_b
            else:
                raise NotImplementedError(f"update_conn reads {name!r}, which no batched phase writes")

    @property
    def num_levels(self) -> int:
        return len(self.static.level_capacities)

    def _rows(self, x, cols: int) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            x = torch.from_numpy(np.ascontiguousarray(x, np.float32))
        x = x.to(self.dev, dtype=torch.float32).reshape(self.batch, cols)
        return x.contiguous()

    def _prune(self, state: NetworkState) -> None:
        pc = self.net.prune_conn
        if pc is None:
            return
        if isinstance(pc, LowestMagnitudePrune):
            self.inner._prune_lowest(state, pc)
            return
        n = self.static.num_units
        for i, b in enumerate(state.conns):
            bm, bm_level = self.inner._bm(i)
            if isinstance(pc, MagnitudePrune):
                K.prune_conn(b, n, prune_kind=_lib.PRUNE_ABS_BELOW, threshold=pc.threshold, free_bitmap=bm,
                             bitmap_level=bm_level)
            elif isinstance(pc, DestinationThresholdPrune):
                K.prune_conn(b, n, prune_kind=_lib.PRUNE_ABS_BELOW_DST, unit_threshold=state.units[pc.field.name],
                             free_bitmap=bm, bitmap_level=bm_level)
            self.launches += 1

    def _check_deeper(self, state: NetworkState) -> None:
        """Every live edge lies in the bucket of its source's level, whose rows
        are final when it is swept, and goes to a deeper level (reads the host,
        once per set of columns and version of them; the framework's own growth
        and prune keep it so). Edges into inputs, which sit at level 0, do not."""
        level = state.units[LEVEL.name]
        cols = [level, *(b[k] for b in state.conns for k in ("from_id", "to_id", "dead"))]
        key = tuple(map(id, cols))
        versions = [-1 if t.is_inference() else t._version for t in cols]
        seen = self._checked.get(key)
        if seen is not None and all(ref() is t and v == now for (ref, v), t, now in zip(seen, cols, versions)):
            return
        if self.dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("activation_checkpoint: the state's edges have not been checked since they were made or "
                               "edited, and a capture cannot read them: run the step once before capturing it")
        n = self.static.num_units
        for i, b in enumerate(state.conns):
            f, t = b["from_id"].long(), b["to_id"].long()
            live = (b["dead"] == 0) & (f >= 0) & (f < n) & (t >= 0) & (t < n)  # as the kernels take them
            f, t = f[live], t[live]
            bad, moved = (level[t] <= level[f]).any(), (level[f] != i).any()
            if bool(bad):
                raise ValueError(f"activation_checkpoint: bucket {i} has an edge that does not go to a deeper level")
            if bool(moved):
                raise ValueError(f"activation_checkpoint: bucket {i} has an edge whose source is not at level {i}: "
                                 "resort the state")
        self._checked = {k: v for k, v in self._checked.items() if all(ref() is not None for ref, _ in v)}
        self._checked[key] = [(weakref.ref(t), v) for t, v in zip(cols, versions)]

    def _call_checkpointed(self, state: NetworkState, x: torch.Tensor, inputs: StepInputs) -> None:
        """The propagation and the update of a step whose backward reads the
        checkpoint; acc_b, act_b and grad_b are one buffer."""
        net, inner, units, rows, ck = self.net, self.inner, state.units, self.acc_b, self.checkpoint
        level, roles, L = units[LEVEL.name], inner.is_input, self.num_levels
        self._check_deeper(state)
        rows.zero_()
        rows.index_copy_(0, inner.input_ids, x.t())
        # level 0: the inputs' codes, and zeros for the other units there, whose rows in the checkpoint may be another
        # state's (the levels are the state's, not the step's)
        mx.mx_unit_apply(rows, ck, "identity", level=level, target_level=0, roles=roles)
        for lv in range(L):
            K.batched_forward(state.conns[lv], rows, rows)
            mx.mx_unit_apply(rows, ck, inner.fwd_act, level=level, target_level=lv + 1, roles=roles)
        self._loss(inputs)
        K.batch_mean(rows, units[ACTIVATION.name])
        bp = net.backward_pass
        if bp is not None:
            rows.zero_()
            mx.mx_unit_grad(rows, ck, inner.bwd_act, seed=self.seed_b, level=level, target_level=L, roles=roles,
                            out=rows)
            for lv in range(L - 1, 0, -1):
                K.batched_backward(state.conns[lv], rows, rows)
                mx.mx_unit_grad(rows, ck, inner.bwd_act, seed=self.seed_b, level=level, target_level=lv, roles=roles,
                                out=rows)
        if net.update_conn is not None:
            for b in state.conns:
                mx.mx_update(b, self.upd_grad_b, ck, inner.opt)
        self.launches += 2 * L + 1 + (0 if bp is None else 2 * L - 1) + (len(state.conns) if net.update_conn else 0)

    def _loss(self, inputs: StepInputs) -> None:
        """Loss, per sample; the batch mean to StepResult.loss."""
        loss = self.net.loss
        if loss is None:
            return
        if inputs.targets is None:
            raise ValueError("a network with a loss needs StepInputs.targets")
        t = self._rows(inputs.targets, len(self.static.output_ids))
        kind = _lib.LOSS_SOFTMAX_CE if isinstance(loss, SoftmaxCrossEntropyLoss) else _lib.LOSS_MSE
        if not isinstance(loss, (MSELoss, SoftmaxCrossEntropyLoss)):
            raise NotImplementedError(f"loss {type(loss).__name__} has no engine lowering")
        K.batched_loss(kind, self.inner.output_ids, self.batch, self.act_b, t, self.seed_b, self.loss_b,
                       self.inner.loss_buf)
        self.launches += 2

    def _call_plain(self, state: NetworkState, x: torch.Tensor, inputs: StepInputs) -> None:
        """The propagation and the update of a step on float32 rows."""
        net, inner, units = self.net, self.inner, state.units
        level, is_input = units[LEVEL.name], inner.is_input
        L = self.num_levels
        self.act_b.index_copy_(0, inner.input_ids, x.t().contiguous())
        # forward, level by level (src/plastax/phases.py:972-1015)
        fp = net.forward_pass
        self.acc_b.zero_()
        for lv in range(L):
            K.batched_forward(state.conns[lv], self.act_b, self.acc_b)
            K.batched_unit_apply(self.acc_b, self.act_b, mode=0, act_kind=inner.fwd_act, level=level,
                                 target_level=lv + 1, is_input=is_input)
            self.launches += 2
        self._loss(inputs)
        # backward, deepest level first (src/plastax/phases.py:1049-1104)
        bp = net.backward_pass
        if bp is not None:
            self.acc_b.zero_()
            K.batched_unit_apply(self.acc_b, self.grad_b, mode=1, act_kind=inner.bwd_act, act=self.act_b,
                                 seed=self.seed_b, level=level, target_level=L, is_input=is_input)
            for lv in range(L - 1, 0, -1):
                K.batched_backward(state.conns[lv], self.grad_b, self.acc_b)
                K.batched_unit_apply(self.acc_b, self.grad_b, mode=1, act_kind=inner.bwd_act, act=self.act_b,
                                     seed=self.seed_b, level=level, target_level=lv, is_input=is_input)
                self.launches += 2
        # the exact batch-mean connection update (src/plastax/phases.py:434-483)
        if net.update_conn is not None:
            for b in state.conns:
                K.batched_update(b, self.upd_grad_b, self.act_b, inner.opt)
                self.launches += 1
        K.batch_mean(self.act_b, units[ACTIVATION.name])

    def __call__(self, state: NetworkState, inputs: StepInputs) -> StepResult:
        net, inner, units = self.net, self.inner, state.units
        inner._bind(state)
        inner._level = units[LEVEL.name]
        x = self._rows(inputs.inputs, len(self.static.input_ids))
        if self.checkpoint is not None:
            self._call_checkpointed(state, x, inputs)
        else:
            self._call_plain(state, x, inputs)
        bp, loss = net.backward_pass, net.loss
        # per-sample unit columns -> the state's (batch_reduction)
        if bp is not None:
            K.batch_mean(self.grad_b, units[bp.grad_field.name])
        if loss is not None:
            K.batch_mean(self.seed_b, units[loss.seed_field.name])
        # structural phases once, on the reduced state
        self._prune(state)
        inner._clear_flags = False
        remainder = inner._add_conn(state)
        inner._step_end()
        state.step += 1
        grown = state.grown if state.grown is not None else torch.zeros((), dtype=torch.int32, device=self.dev)
        overflow = state.overflow if state.overflow is not None else torch.zeros((), dtype=torch.bool,
                                                                                 device=self.dev)
        return StepResult(state=state, overflow=overflow, loss=inner.loss_buf[0], growth_remainder=remainder,
                          grown=grown)


__all__ = ["BatchedStepFn"]
