"""Microscaled (MX) unit rows: 8- and 4-bit blocks, and the edge products that read them.

A batched step's unit rows are [num_units, B] float32. Here a row is held as
blocks of 32 samples, each one power-of-two scale byte (2^(byte - 127); 255 =
the block is not a number) and 32 codes: "e4m3" or "e5m2" (8 bits) or "e2m1"
(4 bits, the even sample in the low nibble). The scale is the smallest power of
two that holds the block's largest magnitude without saturating; a code is the
nearest element, ties to even.

- `mx_quantize` / `mx_dequantize`: rows of float32, bfloat16 or float16 (any
  strides) to MX rows and back.
- `mx_unit_grad`, `mx_edge_grad`: the backward pass from an 8-bit checkpoint of
  the activations (`make_step(..., batch_size=B, activation_checkpoint="e4m3")`
  runs them).
- `mx_product`: act(sum_e w[e] * x[src[e], :]) over in-edges grouped by
  destination (`MxConns`), weights and rows in MX blocks or float32
  (`make_infer` runs a trained feed-forward net with it).

Outputs that are not passed in are allocated on the current stream. Every call
runs on the tensors' device and its current stream, keeps nothing, and can be
captured into a CUDA graph.
"""

from __future__ import annotations

import contextlib
import ctypes
import dataclasses
import functools

import torch

from plastax_b200 import _lib
from plastax_b200 import kernels as K
from plastax_b200._lib import call

BLOCK = 32
FORMATS = ("e4m3", "e5m2", "e2m1")
CHECKPOINT_FORMATS = ("e4m3", "e5m2")
WEIGHT_FORMATS = (*FORMATS, "f32")
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_BATCH = 1 << 24
_MAX_UNITS = (1 << 31) - 1  # the C ABI's counts are 32-bit
_U8 = torch.uint8


def num_blocks(batch: int) -> int:
    return -(-batch // BLOCK)


def block_bytes(fmt: str) -> int:
    return 16 if fmt == "e2m1" else 32


def _format(fmt: str, allowed=FORMATS, what: str = "format") -> int:
    if fmt not in allowed:
        raise ValueError(f"unknown {what} {fmt!r}: one of {', '.join(allowed)}")
    return _lib.MX[fmt]


def _on(dev: torch.device):
    """The tensors' device as the current one."""
    if dev.type != "cuda":
        raise ValueError("engine tensors must live on a CUDA device")
    if dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


_entry = functools.cache(lambda name: getattr(_lib.lib(), name))


def _launch(dev: torch.device, name: str, *args) -> None:
    """Call an entry point on `dev` and its current stream."""
    i = dev.index
    if dev.type == "cuda" and i == torch.cuda.current_device() and i == getattr(K._bound, "device", -1):
        rc = _entry(name)(*args, K._raw_stream(i))  # the usual case, without a look-up twice
        if rc != 0:
            raise _lib.PxbError(f"{name} failed (status {rc}): {_lib.last_error()}")
        return
    with _on(dev):
        call(name, *args, K._stream())


def _tensor(t, dtype, shape, what: str, dev: torch.device | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if t.dtype is dtype and (shape is None or t.shape == shape) and t.is_contiguous() and (
            dev is None or t.device == dev):
        return t
    if t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")
    if dev is not None and t.device != dev:
        raise ValueError(f"{what}: on {t.device}, expected {dev}")
    return t


def _rows_shape(x: torch.Tensor, what: str) -> tuple[int, int]:
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"{what}: expected unit rows [num_units, batch], got shape {tuple(shape)}")
    n, b = shape
    if n > _MAX_UNITS or b > _MAX_BATCH:
        raise ValueError(f"{what}: [{n}, {b}] is past 2^31 - 1 units or {_MAX_BATCH} samples")
    return n, b


@dataclasses.dataclass(frozen=True)
class MxRows:
    """[num_units, batch] rows in MX blocks: `codes` uint8 [num_units,
    ceil(batch / 32) * 32] (e2m1: * 16), `scales` uint8 [num_units, ceil(batch / 32)]."""

    codes: torch.Tensor
    scales: torch.Tensor
    fmt: str
    batch: int

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        _format(self.fmt)
        if not 0 <= self.batch <= _MAX_BATCH:
            raise ValueError(f"MxRows: batch must be in [0, {_MAX_BATCH}], got {self.batch}")
        if isinstance(scales, torch.Tensor) and scales.dim() == 2 and scales.shape[0] > _MAX_UNITS:
            raise ValueError(f"MxRows: {scales.shape[0]} units are past 2^31 - 1")
        nb = num_blocks(self.batch)
        if isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor) and codes.dtype is _U8 and \
                scales.dtype is _U8 and scales.dim() == 2 and scales.shape[1] == nb and \
                codes.shape == (scales.shape[0], nb * block_bytes(self.fmt)) and codes.is_contiguous() and \
                scales.is_contiguous() and codes.device == scales.device and codes.data_ptr() % 16 == 0:
            return
        _tensor(self.scales, torch.uint8, None, "MxRows.scales")
        n = self.scales.shape[0] if self.scales.dim() == 2 else -1
        _tensor(self.scales, torch.uint8, (n, nb), "MxRows.scales")
        _tensor(self.codes, torch.uint8, (n, nb * block_bytes(self.fmt)), "MxRows.codes", self.scales.device)
        if self.codes.data_ptr() % 16:
            raise ValueError("MxRows.codes: must start on a 16-byte boundary")

    @property
    def num_units(self) -> int:
        return self.scales.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def empty(cls, num_units: int, batch: int, fmt: str, device, *, zero: bool = False) -> "MxRows":
        """Rows without values (`zero`: rows that read 0)."""
        _format(fmt)
        if not 0 <= batch <= _MAX_BATCH:
            raise ValueError(f"MxRows: batch must be in [0, {_MAX_BATCH}], got {batch}")
        if num_units > _MAX_UNITS:
            raise ValueError(f"MxRows: {num_units} units are past 2^31 - 1")
        new = torch.zeros if zero else torch.empty
        nb = num_blocks(batch)
        rows = object.__new__(cls)  # nothing to check in what is made here
        rows.__dict__.update(codes=new((num_units, nb * block_bytes(fmt)), dtype=torch.uint8, device=device),
                             scales=new((num_units, nb), dtype=torch.uint8, device=device), fmt=fmt, batch=batch)
        return rows


def mx_quantize(x: torch.Tensor, fmt: str, *, keep_nonzero: bool = False, ids: torch.Tensor | None = None,
                out: MxRows | None = None) -> MxRows:
    """Rows [num_units, batch] of float32, bfloat16 or float16 as MX rows.

    Any strides: a sample-major batch is passed as its transpose. With `ids`
    (int64), row i goes to row ids[i] of `out`, whose other rows stay as they
    were (ids have to differ; one out of range is skipped). `keep_nonzero`: a
    value that is not 0 never becomes 0 but takes the smallest magnitude of
    its sign, so the sign of every value survives (a ReLU's mask)."""
    n, b = _rows_shape(x, "mx_quantize: x")
    code = _format(fmt)
    if x.dtype not in _DT:
        raise TypeError(f"mx_quantize: x is {x.dtype}, expected float32, bfloat16 or float16")
    if out is None:
        if ids is not None:
            raise ValueError("mx_quantize: ids need out")
        out = object.__new__(MxRows)  # nothing to check in what is made here
        nb = num_blocks(b)
        out.__dict__.update(codes=x.new_empty((n, nb * block_bytes(fmt)), dtype=_U8),
                            scales=x.new_empty((n, nb), dtype=_U8), fmt=fmt, batch=b)
    elif out.fmt != fmt or out.batch != b or out.device != x.device or (ids is None and out.num_units != n):
        raise ValueError(f"mx_quantize: out holds {out.num_units} x {out.batch} {out.fmt} rows on {out.device}, "
                         f"expected {n} x {b} {fmt} on {x.device}")
    if ids is not None:
        _tensor(ids, torch.int64, (n,), "mx_quantize: ids", x.device)
    _launch(x.device, "pxb_mx_quantize", n, b, x.data_ptr(), _DT[x.dtype], x.stride(0), x.stride(1), code,
            1 if keep_nonzero else 0, K.ptr(ids), out.num_units, out.codes.data_ptr(), out.scales.data_ptr())
    return out


def mx_dequantize(rows: MxRows, *, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows' values [num_units, batch] in float32, bfloat16 or float16 (an
    element past the type's range reads infinite)
    (`out`: a buffer of that shape; its rows may be further apart than the batch)."""
    if out is None:
        if dtype not in _DT:
            raise TypeError(f"mx_dequantize: {dtype} is not float32, bfloat16 or float16")
        out = rows.codes.new_empty((rows.num_units, rows.batch), dtype=dtype)
    else:
        if out.dtype not in _DT:
            raise TypeError(f"mx_dequantize: out is {out.dtype}, expected float32, bfloat16 or float16")
        if tuple(out.shape) != (rows.num_units, rows.batch) or out.device != rows.device:
            raise ValueError(f"mx_dequantize: out is {tuple(out.shape)} on {out.device}, expected "
                             f"{(rows.num_units, rows.batch)} on {rows.device}")
        if out.numel() and ((out.stride(1) != 1 and rows.batch > 1) or
                            (out.stride(0) < rows.batch and rows.num_units > 1)):
            raise ValueError("mx_dequantize: out's samples must be adjacent and its rows must not overlap")
    ld = max(out.stride(0), rows.batch)
    _launch(rows.device, "pxb_mx_dequantize", rows.num_units, rows.batch, rows.codes.data_ptr(), rows.scales.data_ptr(),
            _lib.MX[rows.fmt], out.data_ptr(), _DT[out.dtype], ld)
    return out


def _masks(n: int, dev, level, roles, what: str) -> None:
    if level is not None:
        _tensor(level, torch.int32, (n,), f"{what}: level", dev)
    if roles is not None:
        _tensor(roles, torch.uint8, (n,), f"{what}: roles", dev)


def mx_unit_apply(rows: torch.Tensor, checkpoint: MxRows, activation, *, level: torch.Tensor | None = None,
                  target_level: int = 0, roles: torch.Tensor | None = None) -> None:
    """rows = activation(rows) in place for the units at `target_level` (all,
    without `level`; an input, role 1, keeps its row), and their checkpoint
    with `keep_nonzero`. `activation`: a name, or (name, the outputs' name). A
    ReLU keeps what is not a number (the float32 step's makes it 0), so a
    poisoned row does not read as a silent one."""
    n, b = _rows_shape(rows, "mx_unit_apply: rows")
    _format(checkpoint.fmt, CHECKPOINT_FORMATS, "checkpoint format")
    _tensor(rows, torch.float32, (checkpoint.num_units, checkpoint.batch), "mx_unit_apply: rows", checkpoint.device)
    _masks(n, rows.device, level, roles, "mx_unit_apply")
    _launch(rows.device, "pxb_mx_unit_apply", n, b, _lib.act_code(activation), rows.data_ptr(), K.ptr(level), target_level,
            K.ptr(roles), _lib.MX[checkpoint.fmt], checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr())


def mx_unit_grad(acc: torch.Tensor, act: MxRows, activation, *, seed: torch.Tensor | None = None,
                 level: torch.Tensor | None = None, target_level: int = 0, roles: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """(acc + seed) * activation'(act), the derivative taken from the
    checkpointed activations, for the units at `target_level` (all, without
    `level`; role 1 excepted). `out` may be `acc`; rows outside the mask are
    left as they were (0 in a new `out`)."""
    n, b = _rows_shape(acc, "mx_unit_grad: acc")
    _format(act.fmt, CHECKPOINT_FORMATS, "checkpoint format")
    shape = (act.num_units, act.batch)
    _tensor(acc, torch.float32, shape, "mx_unit_grad: acc", act.device)
    if seed is not None:
        _tensor(seed, torch.float32, shape, "mx_unit_grad: seed", act.device)
    _masks(n, acc.device, level, roles, "mx_unit_grad")
    if out is None:
        out = torch.zeros_like(acc) if level is not None or roles is not None else torch.empty_like(acc)
    else:
        _tensor(out, torch.float32, shape, "mx_unit_grad: out", act.device)
    _launch(acc.device, "pxb_mx_unit_grad", n, b, _lib.act_code(activation), acc.data_ptr(), K.ptr(seed), act.codes.data_ptr(),
            act.scales.data_ptr(), _lib.MX[act.fmt], K.ptr(level), target_level, K.ptr(roles), out.data_ptr())
    return out


def _edge_args(bucket, grad: torch.Tensor, act: MxRows, what: str) -> int:
    _format(act.fmt, CHECKPOINT_FORMATS, "checkpoint format")
    if act.batch < 1:
        raise ValueError(f"{what}: the batch is empty")
    _tensor(grad, torch.float32, (act.num_units, act.batch), f"{what}: grad", act.device)
    cap = bucket["dead"].numel()
    for name, dt in (("from_id", torch.int32), ("to_id", torch.int32), ("dead", torch.uint8)):
        _tensor(bucket[name], dt, (cap,), f"{what}: bucket column {name!r}", act.device)
    return cap


@functools.lru_cache(maxsize=256)
def edge_grad_scratch_bytes(capacity: int, batch: int, num_units: int) -> int:
    """Scratch that lets the gradient of a small net's many slots run as one
    matrix product (0 for most sizes)."""
    return _lib.query_size("pxb_mx_edge_grad_scratch_bytes", capacity, batch, num_units)


def _scratch(act: MxRows, cap: int) -> tuple[torch.Tensor | None, int]:
    size = edge_grad_scratch_bytes(cap, act.batch, act.num_units)
    return (act.codes.new_empty(size), size) if size else (None, 0)


def mx_edge_grad(bucket: K.Bucket, grad: torch.Tensor, act: MxRows, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The batch-mean gradient of every slot of a bucket,
    (sum_b grad[to, b] * act[from, b]) / B, from checkpointed activations:
    float32 [capacity], 0 for dead slots."""
    cap = _edge_args(bucket, grad, act, "mx_edge_grad")
    if out is None:
        out = grad.new_empty(cap)
    else:
        _tensor(out, torch.float32, (cap,), "mx_edge_grad: out", act.device)
    scratch, size = _scratch(act, cap)
    _launch(act.device, "pxb_mx_edge_grad", cap, bucket["from_id"].data_ptr(),
            bucket["to_id"].data_ptr(), bucket["dead"].data_ptr(),
            grad.data_ptr(), act.codes.data_ptr(), act.scales.data_ptr(), _lib.MX[act.fmt], act.batch,
            act.num_units, out.data_ptr(), None, None, None, None, None, K.ptr(scratch), size)
    return out


def mx_update(bucket: K.Bucket, grad: torch.Tensor, act: MxRows, opt: _lib.Optimizer) -> None:
    """The exact batch-mean update of a bucket (one optimizer step per live
    slot, in place) from checkpointed activations; `opt` is an optimizer
    bundle's `struct()` (not UPGD)."""
    cap = _edge_args(bucket, grad, act, "mx_update")
    for name in ("weight", "opt/m", "opt/v", "opt/t"):
        if name == "weight" or name in bucket:
            _tensor(bucket[name], torch.float32, (cap,), f"mx_update: bucket column {name!r}", act.device)
    scratch, size = _scratch(act, cap)
    _launch(act.device, "pxb_mx_edge_grad", cap, bucket["from_id"].data_ptr(),
            bucket["to_id"].data_ptr(), bucket["dead"].data_ptr(),
            grad.data_ptr(), act.codes.data_ptr(), act.scales.data_ptr(), _lib.MX[act.fmt], act.batch,
            act.num_units, None, bucket["weight"].data_ptr(), ctypes.byref(opt), K.ptr(bucket.get("opt/m")),
            K.ptr(bucket.get("opt/v")), K.ptr(bucket.get("opt/t")), K.ptr(scratch), size)


@dataclasses.dataclass(frozen=True)
class MxConns:
    """In-edges grouped by destination, with their weights laid out once.

    Edges [offsets[i], offsets[i + 1]) of `src` (int32) end in unit units[i]
    (int32; the units differ). `weights` names the weights' form: "f32"
    (`weight`, one an edge) or an MX format, in blocks of 32 consecutive
    in-edges of one destination: blocks [block_offsets[i], block_offsets[i +
    1]) of `codes` (uint8 [blocks, 32], e2m1 [blocks, 16]) and `scales` (uint8
    [blocks]). Offsets are int64. The tensors' memory is taken when the
    connections are made: values may be edited in place, but a tensor that gets
    other memory (`set_`, `.data`) needs new connections."""

    units: torch.Tensor
    offsets: torch.Tensor
    src: torch.Tensor
    weights: str
    weight: torch.Tensor | None = None
    block_offsets: torch.Tensor | None = None
    codes: torch.Tensor | None = None
    scales: torch.Tensor | None = None

    def __post_init__(self) -> None:
        fmt = _format(self.weights, WEIGHT_FORMATS, "weight format")
        units, offsets, src = self.units, self.offsets, self.src
        dev, m, e = units.device, units.numel(), src.numel()
        if m > _MAX_UNITS:
            raise ValueError(f"MxConns.units: {m} destinations are past 2^31 - 1")
        _tensor(units, torch.int32, (m,), "MxConns.units")
        _tensor(offsets, torch.int64, (m + 1,), "MxConns.offsets", dev)
        _tensor(src, torch.int32, (e,), "MxConns.src", dev)
        if self.weights == "f32":
            _tensor(self.weight, torch.float32, (e,), "MxConns.weight", dev)
            c = _lib.MxConns(m, fmt, e, 0, units.data_ptr(), offsets.data_ptr(), src.data_ptr(), self.weight.data_ptr(),
                             None, None, None)
        else:
            _tensor(self.block_offsets, torch.int64, (m + 1,), "MxConns.block_offsets", dev)
            _tensor(self.scales, _U8, None, "MxConns.scales", dev)
            blocks = self.scales.numel()
            if self.scales.dim() != 1:
                raise ValueError(f"MxConns.scales: expected shape {(blocks,)}, got {tuple(self.scales.shape)}")
            _tensor(self.codes, _U8, (blocks, block_bytes(self.weights)), "MxConns.codes", dev)
            if self.codes.data_ptr() % 16:
                raise ValueError("MxConns.codes: must start on a 16-byte boundary")
            c = _lib.MxConns(m, fmt, e, blocks, units.data_ptr(), offsets.data_ptr(), src.data_ptr(), None,
                             self.block_offsets.data_ptr(), self.codes.data_ptr(), self.scales.data_ptr())
        object.__setattr__(self, "_c", c)

    @property
    def num_edges(self) -> int:
        return self.src.numel()

    @classmethod
    def from_edges(cls, src: torch.Tensor, dst: torch.Tensor, weight: torch.Tensor, units: torch.Tensor, *,
                   weights: str = "e2m1") -> "MxConns":
        """Group the edges that end in `units` (int32, ascending) by
        destination, in their order, and lay their weights out. Edges into
        other units are left out. Setup: sorts and sizes on the device, and
        reads counts on the host."""
        _format(weights, WEIGHT_FORMATS, "weight format")
        dev, m = units.device, units.numel()
        ids = units.long()
        at = torch.searchsorted(ids, dst.long())
        inside = (at < m) & (ids[at.clamp(max=max(m - 1, 0))] == dst.long()) if m else torch.zeros_like(at, dtype=torch.bool)
        at, order = torch.sort(at[inside], stable=True)
        src, w = src[inside][order].to(torch.int32).contiguous(), weight[inside][order].to(torch.float32).contiguous()
        deg = torch.bincount(at, minlength=m)
        zero = torch.zeros(1, dtype=torch.int64, device=dev)
        offsets = torch.cat([zero, deg.cumsum(0)])
        if weights == "f32":
            return cls(units, offsets, src, weights, weight=w)
        blocks = torch.cat([zero, ((deg + BLOCK - 1) // BLOCK).cumsum(0)])
        padded = torch.zeros((int(blocks[-1].item()), BLOCK), dtype=torch.float32, device=dev)
        lane = torch.arange(at.numel(), device=dev) - offsets[at]
        padded.view(-1)[blocks[at] * BLOCK + lane] = w
        rows = mx_quantize(padded, weights)
        return cls(units, offsets, src, weights, block_offsets=blocks, codes=rows.codes, scales=rows.scales.view(-1))


def mx_product(conns: MxConns, x: torch.Tensor | MxRows, *, activation: str = "identity",
               out: torch.Tensor | MxRows | None = None) -> torch.Tensor | MxRows:
    """out[units[i], b] = activation(sum_e w[e] * x[src[e], b]), summed in
    float32; activation(0) for a destination without edges. A ReLU keeps what is
    not a number.

    x: float32 rows [num_units, batch] or MX rows. `out`: float32 rows or MX
    rows of the same batch, written at the destinations' rows only (a new
    float32 [num_units, batch], 0 elsewhere, when not given). It may be x's
    own buffer when no destination is a source. Sources and units out of
    range are skipped."""
    mx_in = isinstance(x, MxRows)
    if mx_in:
        n, b = x.num_units, x.batch
    else:
        n, b = _rows_shape(x, "mx_product: x")
        _tensor(x, torch.float32, None, "mx_product: x")
    dev = conns.units.device
    if x.device != dev:
        raise ValueError(f"mx_product: x is on {x.device}, the connections on {dev}")
    if activation not in _lib.ACT:
        raise ValueError(f"mx_product: unknown activation {activation!r}")
    if out is None:
        out = torch.zeros((n, b), dtype=torch.float32, device=dev)
    mx_out = isinstance(out, MxRows)
    if mx_out:
        if out.batch != b or out.device != dev:
            raise ValueError(f"mx_product: out holds {out.batch} samples on {out.device}, expected {b} on {dev}")
        rows = out.num_units
    else:
        rows, _ = _rows_shape(out, "mx_product: out")
        _tensor(out, torch.float32, (rows, b), "mx_product: out", dev)
    _launch(dev, "pxb_mx_product", ctypes.byref(conns._c), n, b, None if mx_in else x.data_ptr(),
            x.codes.data_ptr() if mx_in else None, x.scales.data_ptr() if mx_in else None,
            _lib.MX[x.fmt] if mx_in else _lib.MX["f32"], _lib.ACT[activation], rows,
            None if mx_out else out.data_ptr(), out.codes.data_ptr() if mx_out else None,
            out.scales.data_ptr() if mx_out else None, _lib.MX[out.fmt] if mx_out else _lib.MX["f32"])
    return out


__all__ = ["BLOCK", "CHECKPOINT_FORMATS", "FORMATS", "MxConns", "MxRows", "block_bytes", "mx_dequantize",
           "mx_edge_grad", "mx_product", "mx_quantize", "mx_unit_apply", "mx_unit_grad", "mx_update", "num_blocks"]
