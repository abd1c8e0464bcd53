"""The microscaled operators' checks of their arguments (no GPU: every refusal
comes before a kernel), and the numpy restatement against itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import plastax_b200 as px
from plastax_b200 import _lib, mx

from tests import _mx


def _rows(n=4, b=40, fmt="e4m3"):
    return px.MxRows.empty(n, b, fmt, "cpu", zero=True)


@pytest.mark.parametrize("fmt", sorted(_mx.FORMATS))
def test_restated_rounding_is_to_the_nearest_and_keeps_grid_values(fmt):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 70)) * np.exp(rng.standard_normal((6, 1)) * 8)
    codes, scales = _mx.quantize(x, fmt)
    v = _mx.values(codes, scales, fmt, 70)
    again = _mx.values(*_mx.quantize(v, fmt), fmt, 70)
    np.testing.assert_array_equal(v, again)
    assert (np.abs(v - x) <= _mx.half_step(x, np.zeros_like(x), fmt)).all()


def test_rows_refuse_wrong_shapes_and_types():
    ok = _rows()
    with pytest.raises(ValueError, match="format"):
        px.MxRows(ok.codes, ok.scales, "e3m4", 40)
    with pytest.raises(TypeError):
        px.MxRows(ok.codes.to(torch.int8), ok.scales, "e4m3", 40)
    with pytest.raises(ValueError, match="shape"):
        px.MxRows(ok.codes, ok.scales, "e4m3", 65)
    with pytest.raises(ValueError, match="shape"):
        px.MxRows(ok.codes, ok.scales, "e2m1", 40)
    with pytest.raises(ValueError, match="contiguous"):
        px.MxRows(ok.codes.t().contiguous().t(), ok.scales, "e4m3", 40)
    with pytest.raises(ValueError, match="16-byte"):
        flat = torch.zeros(4 * 64 + 1, dtype=torch.uint8)
        px.MxRows(flat[1:].view(4, 64), ok.scales, "e4m3", 40)
    with pytest.raises(ValueError, match="batch"):
        px.MxRows(ok.codes, ok.scales, "e4m3", -1)


def test_calls_refuse_host_tensors_and_mismatches():
    x = torch.zeros(4, 40)
    rows = _rows()
    bucket = {"from_id": torch.zeros(8, dtype=torch.int32), "to_id": torch.zeros(8, dtype=torch.int32),
              "dead": torch.zeros(8, dtype=torch.uint8)}
    for fn in (lambda: px.mx_quantize(x, "e4m3"), lambda: px.mx_dequantize(rows),
               lambda: px.mx_unit_grad(x, rows, "relu"), lambda: px.mx_unit_apply(x, rows, "relu"),
               lambda: px.mx_edge_grad(bucket, x, rows)):
        with pytest.raises(ValueError, match="CUDA"):
            fn()
    with pytest.raises(ValueError, match="format"):
        px.mx_quantize(x, "int8")
    with pytest.raises(TypeError):
        px.mx_quantize(x.double(), "e4m3")
    with pytest.raises(ValueError, match="unit rows"):
        px.mx_quantize(x[0], "e4m3")
    with pytest.raises(ValueError, match="ids need out"):
        px.mx_quantize(x, "e4m3", ids=torch.arange(4))
    with pytest.raises(TypeError):
        px.mx_quantize(x, "e4m3", ids=torch.arange(4, dtype=torch.int32), out=rows)
    with pytest.raises(ValueError, match="out holds"):
        px.mx_quantize(x, "e5m2", out=rows)
    with pytest.raises(ValueError, match="out holds"):
        px.mx_quantize(x[:, :39], "e4m3", out=rows)
    with pytest.raises(TypeError):
        px.mx_dequantize(rows, dtype=torch.float64)
    with pytest.raises(ValueError, match="out is"):
        px.mx_dequantize(rows, out=torch.zeros(4, 41))
    with pytest.raises(ValueError, match="adjacent"):
        px.mx_dequantize(rows, out=torch.zeros(40, 4).t())
    with pytest.raises(ValueError, match="overlap"):
        px.mx_dequantize(rows, out=torch.zeros(40).expand(4, 40))
    # a checkpoint has 8 bits
    four = _rows(fmt="e2m1")
    for fn in (lambda: px.mx_unit_grad(x, four, "relu"), lambda: px.mx_unit_apply(x, four, "relu"),
               lambda: px.mx_edge_grad(bucket, x, four)):
        with pytest.raises(ValueError, match="checkpoint format"):
            fn()
    with pytest.raises(ValueError, match="shape"):
        px.mx_unit_grad(x, rows, "relu", seed=x[:3])
    with pytest.raises(ValueError, match="shape"):
        px.mx_edge_grad(bucket, x[:, :39].contiguous(), rows)
    with pytest.raises(ValueError, match="contiguous"):
        px.mx_edge_grad(bucket, x.t().contiguous().t(), rows)
    with pytest.raises(TypeError):
        px.mx_edge_grad({**bucket, "to_id": bucket["to_id"].long()}, x, rows)
    with pytest.raises(ValueError, match="empty"):
        px.mx_edge_grad(bucket, x[:, :0], px.MxRows.empty(4, 0, "e4m3", "cpu"))


def _conns(**kw):
    args = dict(units=torch.tensor([1, 2], dtype=torch.int32), offsets=torch.tensor([0, 1, 2]),
                src=torch.zeros(2, dtype=torch.int32), weights="f32", weight=torch.ones(2))
    return px.MxConns(**{**args, **kw})


def test_conns_and_product_refuse():
    c = _conns()
    with pytest.raises(ValueError, match="weight format"):
        _conns(weights="e9")
    with pytest.raises(TypeError):
        _conns(weight=None)
    with pytest.raises(ValueError, match="shape"):
        _conns(offsets=torch.tensor([0, 1]))
    with pytest.raises(TypeError):
        _conns(offsets=torch.tensor([0, 1, 2], dtype=torch.int32))
    with pytest.raises(TypeError):
        _conns(weights="e2m1")
    with pytest.raises(ValueError, match="shape"):
        _conns(weights="e2m1", block_offsets=torch.tensor([0, 1, 2]), scales=torch.zeros(2, dtype=torch.uint8),
               codes=torch.zeros((2, 32), dtype=torch.uint8))
    with pytest.raises(ValueError, match="activation"):
        px.mx_product(c, torch.zeros(3, 4), activation="gelu")
    with pytest.raises(TypeError):
        px.mx_product(c, torch.zeros(3, 4).bfloat16())
    with pytest.raises(ValueError, match="contiguous"):
        px.mx_product(c, torch.zeros(4, 3).t())
    with pytest.raises(ValueError, match="expected shape"):
        px.mx_product(c, torch.zeros(3, 4), out=torch.zeros(3, 5))
    with pytest.raises(ValueError, match="samples"):
        px.mx_product(c, torch.zeros(3, 4), out=_rows())
    with pytest.raises(ValueError, match="CUDA"):
        px.mx_product(c, torch.zeros(3, 4))


def test_abi_refuses_before_a_launch():
    """The C ABI's own checks (no device is touched)."""
    lib = _lib.lib()

    def refuse(name, *args, text):
        assert getattr(lib, name)(*args) == 1
        assert text in _lib.last_error()

    refuse("pxb_mx_quantize", 1, 32, 64, 0, 32, 1, 7, 0, None, 1, 64, 64, None, text="format")
    refuse("pxb_mx_quantize", 1, 32, 64, 5, 32, 1, 0, 0, None, 1, 64, 64, None, text="type")
    refuse("pxb_mx_quantize", 2, 32, 64, 0, 32, 1, 0, 0, None, 1, 64, 64, None, text="do not fit")
    refuse("pxb_mx_quantize", 1, 32, None, 0, 32, 1, 0, 0, None, 1, 64, 64, None, text="NULL")
    refuse("pxb_mx_quantize", 1, 32, 64, 0, 32, 1, 0, 0, None, 1, 72, 64, None, text="16-byte")
    refuse("pxb_mx_quantize", (1 << 31) - 1, 96, 64, 0, 32, 1, 0, 0, None, (1 << 31) - 1, 64, 64, None, text="2^32")
    refuse("pxb_mx_dequantize", 1, 32, 64, 64, 0, 64, 0, 31, None, text="overlap")
    refuse("pxb_mx_unit_apply", 1, 32, 0, 64, None, 0, None, 2, 64, 64, None, text="8 bits")
    refuse("pxb_mx_unit_grad", 1, 32, 9, 64, None, 64, 64, 0, None, 0, None, 64, None, text="activation")
    refuse("pxb_mx_edge_grad", 8, 64, 64, 64, 64, 64, 64, 0, 0, 4, 64, None, None, None, None, None, None, 0,
           None, text="sizes")
    refuse("pxb_mx_edge_grad", 8, 64, 64, 64, 64, 64, 64, 0, 4, 4, None, None, None, None, None, None, None, 0,
           None, text="not both or neither")
    many = 1 << 20
    assert lib.pxb_mx_edge_grad(many, 64, 64, 64, 64, 64, 64, 0, 256, 1000, 64, None, None, None, None, None, 64, 16,
                                None) == 3 and "scratch" in _lib.last_error()
    assert mx.edge_grad_scratch_bytes(many, 256, 1000) == 1000 * 1000 * 4 + 16 * 16 // 8
    for sizes in ((many, 32, 1000), (many // 64, 256, 1000), (many, 256, 4097), (0, 1, 0)):
        assert mx.edge_grad_scratch_bytes(*sizes) == 0
    conns = _lib.MxConns(2, 3, 4, 0, 64, 64, 64, None, None, None, None)
    import ctypes

    refuse("pxb_mx_product", ctypes.byref(conns), 4, 4, 64, None, None, 3, 0, 4, 64, None, None, 3, None, text="NULL")
    empty = _lib.MxConns(2, 2, 0, 0, 64, 64, None, None, None, None, None)  # 4-bit weights, no edges, no block offsets
    refuse("pxb_mx_product", ctypes.byref(empty), 4, 4, 64, None, None, 3, 0, 4, 64, None, None, 3, None,
           text="block_offsets")
    refuse("pxb_mx_product", ctypes.byref(conns), 4, (1 << 30) + 1, 64, None, None, 3, 0, 4, 64, None, None, 3, None,
           text="sizes")
    refuse("pxb_mx_product", None, 4, 4, 64, None, None, 3, 0, 4, 64, None, None, 3, None, text="NULL")
    refuse("pxb_mx_product", ctypes.byref(conns), 4, 4, 64, None, None, 3, 4, 4, 64, None, None, 3, None,
           text="activation")


def _net(**kw):
    class Net(px.Network):
        forward_pass = px.ForwardPass("relu", output_activation="identity")
        backward_pass = px.BackwardPass("relu")
        loss = px.MSELoss()
        update_conn = px.optim.sgd(0.1)
        batch_reduction = px.MeanFloatFirstRest()
        propagation = kw.get("propagation", px.Propagation.TOPOLOGICAL)
        add_conn = kw.get("add_conn")

    return Net


def _built(net, device="cpu", **kw):
    return px.NetworkBuilder.from_edges(net, 5, [0, 1, 2, 2], [2, 2, 3, 4], weights=[1.0, 2.0, 3.0, 4.0],
                                        input_ids=(0, 1), output_ids=(3, 4), device=device, **kw)


def test_make_step_refuses_checkpoints_it_cannot_run():
    net = _net()
    static, _ = _built(net)
    with pytest.raises(ValueError, match="batched step"):
        px.make_step(net, static, activation_checkpoint="e4m3", device="cpu")
    with pytest.raises(ValueError, match="unknown activation_checkpoint"):
        px.make_step(net, static, batch_size=8, activation_checkpoint="e2m1", device="cpu")
    grown = _net(add_conn=px.ProposeAddConn(proposals_per_proposer=1, max_new_per_level=4))
    static, _ = _built(grown)
    with pytest.raises(NotImplementedError, match="deeper"):
        px.make_step(grown, static, batch_size=8, activation_checkpoint="e4m3", device="cpu")


def test_checkpointed_step_checks_edited_columns_again():
    """The check of a state's edges holds for its columns as they were: edited
    in place or replaced, they are looked at again; several states stay known."""
    net = _net()
    static, a = _built(net)
    _, b = _built(net)
    step = px.make_step(net, static, batch_size=8, device="cpu", activation_checkpoint="e4m3")
    step._check_deeper(a), step._check_deeper(b)
    known = dict(step._checked)
    step._check_deeper(a), step._check_deeper(b)
    assert step._checked == known and len(known) == 2  # nothing was read again
    a.units["level"][2] = 2  # the same state, a level edited in place: 2 -> 3 and 2 -> 4 stay on a level
    with pytest.raises(ValueError, match="deeper"):
        step._check_deeper(a)
    a.units["level"][2] = 1
    step._check_deeper(a)
    a.conns[0]["to_id"][0] = 1
    with pytest.raises(ValueError, match="deeper"):
        step._check_deeper(a)
    a.conns[0]["dead"][0] = 1
    step._check_deeper(a)
    cols = dict(b.conns[1])
    cols["to_id"] = torch.zeros_like(cols["to_id"])
    b.conns = (b.conns[0], cols)
    with pytest.raises(ValueError, match="deeper"):
        step._check_deeper(b)
    del a, b, cols
    step._check_deeper(_built(net)[1])
    assert len(step._checked) == 1  # what is gone is forgotten


def test_checkpointed_step_does_not_check_edges_out_of_range():
    """A live slot whose ids are out of range is no edge to the kernels."""
    net = _net()
    for column, bad in (("to_id", -1), ("to_id", 5), ("from_id", 5), ("from_id", -(1 << 31))):
        static, state = _built(net)
        state.conns[1][column][0] = bad
        px.make_step(net, static, batch_size=8, device="cpu", activation_checkpoint="e4m3")._check_deeper(state)


def test_checkpointed_step_refuses_sources_of_another_level():
    """Bucket i is swept when level i is final: a source that a caller moved to
    a deeper level, still below its destinations, is read too early."""
    net = _net()
    static, state = px.NetworkBuilder.from_edges(net, 6, [0, 1, 2, 5, 5], [2, 5, 5, 3, 4], input_ids=(0, 1),
                                                 output_ids=(3, 4), device="cpu")
    step = px.make_step(net, static, batch_size=8, device="cpu", activation_checkpoint="e4m3")
    step._check_deeper(state)
    state.conns[0]["from_id"][1], state.conns[0]["to_id"][1] = 2, 3  # 2 -> 3 in the inputs' bucket
    with pytest.raises(ValueError, match="not at level 0"):
        step._check_deeper(state)


def test_make_infer_refuses():
    net = _net()
    static, state = _built(net)
    with pytest.raises(ValueError, match="unknown weights"):
        px.make_infer(net, static, state, weights="int4")
    with pytest.raises(ValueError, match="unknown rows"):
        px.make_infer(net, static, state, rows="int4")
    pipe = _net(propagation=px.Propagation.PIPELINE)
    pstatic, pstate = _built(pipe)
    with pytest.raises(ValueError, match="PIPELINE"):
        px.make_infer(pipe, pstatic, pstate)


def test_infer_layout_is_compact_and_grouped():
    """The f32 layout (built without a GPU): rows for the sources only, each
    output's in-edges in slot order."""
    net = _net()
    static, state = _built(net)
    infer = px.make_infer(net, static, state, weights="f32")
    assert infer.num_rows == 3 and infer.num_still == 0 and infer.num_edges == 4
    hidden, outs = infer.stages
    assert hidden.conns.units.tolist() == [2] and hidden.conns.src.tolist() == [0, 1]
    assert hidden.conns.weight.tolist() == [1.0, 2.0] and not hidden.to_outputs
    assert outs.to_outputs and outs.activation == "identity" and outs.conns.units.tolist() == [0, 1]
    assert outs.conns.offsets.tolist() == [0, 1, 2] and outs.conns.weight.tolist() == [3.0, 4.0]
    with pytest.raises(ValueError, match="expected inputs"):
        infer(np.zeros((3, 5), np.float32))
    with pytest.raises(ValueError, match="CUDA"):
        infer(np.zeros((3, 2), np.float32))


def test_infer_lays_out_units_that_no_level_applies():
    """Sources that nothing writes have a row with what the state holds: a
    pruned unit, a level-0 unit that is no input; a batched net's are 0."""
    for batched in (False, True):
        net = _net()
        if not batched:
            net.batch_reduction = None
        static, state = px.NetworkBuilder.from_edges(net, 6, [0, 1, 2, 2, 5, 1], [2, 2, 3, 4, 3, 3], input_ids=(0, 1),
                                                     output_ids=(3, 4, 5), device="cpu")
        state.units["pruned"] = torch.tensor([0, 0, 1, 0, 0, 0], dtype=torch.uint8)
        state.units["activation"][2], state.units["activation"][5] = -0.5, 2.0
        infer = px.make_infer(net, static, state, weights="f32")
        assert infer.num_rows == 4 and infer.num_still == 2
        assert infer.still_rows.tolist() == [2, 3]  # units 2 and 5, after the inputs
        want = [0.0, 0.0] if batched else [-0.5, 2.0]
        assert infer.still_values.flatten().tolist() == want
        assert [s.conns.units.tolist() for s in infer.stages] == [[0, 1]] * 1
        assert infer.out_still.tolist() == [2] and infer.out_still_values.flatten().tolist() == want[1:]
        state.units["activation"].fill_(9.0)  # a snapshot
        assert infer.still_values.flatten().tolist() == want


def test_few_slots_of_a_long_batch_go_slot_by_slot():
    """One product of all pairs gives a tile of units one CTA for the whole
    batch: a small net's few slots are spread over the batch instead."""
    for sizes in ((4096, 16384, 64), (32768, 16384, 16), (16384, 1 << 20, 128), (4, 1 << 24, 2)):
        assert mx.edge_grad_scratch_bytes(*sizes) == 0
    assert mx.edge_grad_scratch_bytes(65536, 1024, 64) == 64 * 64 * 4 + 4


def test_infer_leaves_out_edges_out_of_range():
    """A live slot whose ids are out of range is no edge, as in the step (on a
    GPU, indexing by it would be a device assert)."""
    net = _net()
    for column, bad in (("to_id", -1), ("to_id", 5), ("from_id", 5), ("from_id", -2), ("from_id", -(1 << 31))):
        static, state = _built(net)
        state.conns[1][column][0] = bad
        infer = px.make_infer(net, static, state, weights="f32")
        assert infer.num_edges == 3 and infer.stages[-1].conns.offsets.tolist() == [0, 0, 1]


def test_counts_past_32_bits_are_refused():
    """The C ABI counts units in 32 bits: more would be cut off without a word."""
    n = (1 << 31) + 7
    big = lambda *shape, dtype=torch.uint8: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="2\\^31"):
        px.MxRows(big(n, 32), big(n, 1), "e4m3", 1)
    with pytest.raises(ValueError, match="2\\^31"):
        px.MxRows.empty(n, 1, "e2m1", "meta")
    with pytest.raises(ValueError, match="2\\^31"):
        px.mx_quantize(big(n, 1, dtype=torch.float32), "e4m3")
    with pytest.raises(ValueError, match="2\\^31"):
        px.MxConns(big(n, dtype=torch.int32), big(n + 1, dtype=torch.int64), big(5, dtype=torch.int32), "f32",
                   weight=big(5, dtype=torch.float32))
    assert px.MxRows(big(5, 32), big(5, 1), "e4m3", 1).num_units == 5


def test_block_counts():
    assert [mx.num_blocks(b) for b in (0, 1, 32, 33, 256)] == [0, 1, 1, 2, 8]
    assert mx.block_bytes("e2m1") == 16 and mx.block_bytes("e5m2") == 32
