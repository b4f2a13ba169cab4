"""CPU: rules that the 4-bit layers, the RMSNorms and the rotary positions keep at their limits."""
import contextlib
import ctypes
import decimal
import importlib
import os
import re

import pytest
import torch
import torch.nn as nn

PKG = "hunyuan3d-tools_b200"


@pytest.fixture(scope="module")
def lib(build_mod):
    return importlib.import_module(PKG + ".csrc._binding").configure(build_mod.load_library())


@pytest.fixture(scope="module")
def rotary():
    return importlib.import_module(PKG + ".rotary")


# ---- order of the kernels' first steps ------------------------------------------------------
def test_tensor_memory_is_taken_before_the_next_kernel_may_start(build_mod):
    """A dependent kernel takes its tensor memory and then waits for this grid to end; a CTA of this grid that is still
    without would wait for those columns for good.  So no function lets the next kernel start ahead of its allocation, and a
    block-wide barrier lies between the two."""
    csrc = os.path.dirname(build_mod.__file__)
    found = 0
    for name in sorted(f for f in os.listdir(csrc) if f.endswith(".cu")):
        with open(os.path.join(csrc, name)) as f:
            functions = re.split(r"^}", f.read(), flags=re.M)      # a function ends at a brace in the first column
        for body in functions:
            takes = [m.start() for m in re.finditer(r"\btmem_alloc_[12]cta\(", body)]
            starts = [m.start() for m in re.finditer(r"\bpdl_launch_dependents\(\)", body)]
            if not takes or not starts:
                continue
            found += 1
            assert min(starts) > max(takes), f"{name}: the next kernel may start before tensor memory is taken"
            assert "__syncthreads()" in body[max(takes):min(starts)], f"{name}: no barrier behind the allocation"
    assert found >= 5


# ---- angles in 60 digits, apart from the plan ------------------------------------------------
def _pi():
    """Machin: pi / 4 = 4 arctan(1 / 5) - arctan(1 / 239)."""
    with decimal.localcontext() as ctx:
        ctx.prec = 70

        def arctan_of_one_over(n):
            term = total = decimal.Decimal(1) / n
            i, sign = 1, 1
            while abs(term) > decimal.Decimal(10) ** -68:
                term, i, sign = term / (n * n), i + 2, -sign
                total += sign * term / i
            return total
        return 4 * (4 * arctan_of_one_over(5) - arctan_of_one_over(239))


def _frequencies_of_many_digits(d, base, scaling):
    base, scaling = decimal.Decimal(base), scaling or {}
    factor = decimal.Decimal(scaling.get("factor", 1))
    if scaling.get("kind") == "ntk":
        base *= ((decimal.Decimal(d) / (d - 2)) * factor.ln()).exp()
    out = []
    for i in range(d // 2):
        w = (-(decimal.Decimal(2 * i) / d) * base.ln()).exp()
        if scaling.get("kind") == "linear":
            w /= factor
        elif scaling.get("kind") == "by_parts":      # whole below 1 turn in the original length, none from 4 on
            keep = min(decimal.Decimal(1), max(decimal.Decimal(0), (scaling["original_length"] * w / (2 * _pi()) - 1) / 3))
            w = w * keep + w / factor * (1 - keep)
        out.append(w)
    return out


@pytest.mark.parametrize("d,base,scaling", [(64, 10000.0, None), (128, 500000.0, None), (96, 10000.0, {"kind": "linear", "factor": 3.0}),
                                            (64, 10000.0, {"kind": "ntk", "factor": 4.0}),
                                            (128, 10000.0, {"kind": "by_parts", "factor": 8.0, "original_length": 8192}), (2, 7.5, None)])
def test_rotary_fractions_are_the_nearest(rotary, d, base, scaling):
    """Half of the last of 64 bits, and 1e-6 of it for the 60 digits that both are made in."""
    r = rotary.RotaryPositions(d, base=base, scaling=scaling)
    with decimal.localcontext() as ctx:
        ctx.prec = 70
        exact = [w / (2 * _pi()) * 2 ** 64 for w in _frequencies_of_many_digits(d, base, scaling)]
        for t, e, w in zip(memoryview(r._turns).cast("Q"), exact, r.frequencies, strict=True):
            assert abs(t - e) <= decimal.Decimal("0.500001")
            assert w == float(e / 2 ** 64 * (2 * _pi()))


# ---- the device is asked for ------------------------------------------------------------------
@pytest.mark.parametrize("name,entries", [("rmsnorm.cu", ("rmsnorm", "dequantize_rows")), ("rotary.cu", ("apply",)), ("linear_w4.cu", ("linear",))])
def test_entry_points_ask_for_the_device_before_they_launch(build_mod, name, entries):
    """So that another GPU is answered with its own status, not with that of a launch that failed.  Read from the sources,
    as no other GPU is at hand."""
    with open(os.path.join(os.path.dirname(build_mod.__file__), name)) as f:
        functions = re.split(r"^}", f.read(), flags=re.M)
    for entry in entries:
        body, = [b for b in functions if re.search(rf"^int {entry}\(", b, flags=re.M)]
        body = body[re.search(rf"^int {entry}\(", body, flags=re.M).start():]
        assert re.search(r"= device_ok\(\);\s+if \(rc != HY3D_OK\) return rc;", body), f"{name}: {entry}"


# ---- what checkpoints and conversions bring ---------------------------------------------------
def _int4_state(qu, dtype=torch.float16, zeros=True):
    torch.manual_seed(4)
    codes = torch.randint(0, 16, (32, 128))
    zero = torch.randint(0, 16, (32, 2)) if zeros else None
    layer = qu.Int4Linear.from_codes(codes, (torch.rand(32, 2) + 0.5).to(dtype), zero, torch.zeros(32))
    return layer, {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in layer.state_dict().items()}


@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("name,value,match", [("weight_scale", 4096.0, "sixteenth"), ("weight_scale", float("inf"), "sixteenth"),
                                              ("weight_scale", float("nan"), "sixteenth"), ("weight_zero", 16, "zero point"),
                                              ("weight_zero", 255, "zero point")])
def test_int4_checkpoints_outside_the_kernels_limits_are_refused(qu, assign, name, value, match):
    layer, state = _int4_state(qu)
    fresh = qu.Int4Linear(128, 32, group_size=64, symmetric=False)
    before = {k: v.clone() for k, v in fresh.state_dict().items() if isinstance(v, torch.Tensor)}
    state[name].view(-1)[7] = value
    with pytest.raises(RuntimeError, match=match):
        fresh.load_state_dict(state, assign=assign)
    assert all(torch.equal(fresh.state_dict()[k], v) for k, v in before.items())
    fresh.load_state_dict(layer.state_dict(), assign=assign)
    assert torch.equal(fresh.dequantize_weight(), layer.dequantize_weight())


def test_int4_checkpoints_of_other_shapes_and_types(qu):
    layer, state = _int4_state(qu)
    for bad in (dict(weight_scale=state["weight_scale"][:1]), dict(weight_scale=torch.ones(2, 3, 16).half()),
                dict(weight_scale=torch.ones(2, 8, 16).half(), weight_zero=torch.zeros(2, 8, 16, dtype=torch.uint8)),
                dict(weight_zero=state["weight_zero"][:, :1]), dict(weight_zero=state["weight_zero"].int())):
        with pytest.raises(RuntimeError, match="weight_scale"):
            qu.Int4Linear(128, 32).load_state_dict({**state, **bad})
    with pytest.raises(RuntimeError, match="bias"):
        qu.Int4Linear(128, 32).load_state_dict({**state, "bias": torch.zeros(33)})
    wide = qu.Int4Linear(128, 32)            # scales that were kept in fp32 come back in the layer's type, which the kernels take
    wide.load_state_dict({**state, "weight_scale": state["weight_scale"].float()})
    assert wide.weight_scale.dtype == torch.float16 and torch.equal(wide.dequantize_weight(), layer.dequantize_weight())
    wide.float().load_state_dict({**state, "weight_scale": state["weight_scale"].float()})      # and into a layer in fp32, as it is
    assert wide.weight_scale.dtype == torch.float32 and torch.equal(wide.half().dequantize_weight(), layer.dequantize_weight())
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        qu.Int4Linear(128, 32).load_state_dict({**state, "weight_scale": torch.ones(2, 2, 16, dtype=torch.int32)}, assign=True)
    with pytest.raises(RuntimeError, match="zero point"):
        layer.load_state_dict({"weight_zero": torch.full((2, 2, 16), 16, dtype=torch.uint8)}, strict=False)


def test_int4_conversions_that_lose_scales_are_refused(qu):
    layer, _ = _int4_state(qu, torch.bfloat16)
    layer.weight_scale[1, 0, 3] = 4096.0
    kept = layer.weight_scale.clone()
    for convert in (lambda m: m.half(), lambda m: m.to(torch.float16), lambda m: nn.Sequential(m).half()):
        with pytest.raises(RuntimeError, match="sixteenth"):
            convert(layer)
        assert layer.weight_scale.dtype == torch.bfloat16 and torch.equal(layer.weight_scale, kept)
    layer.weight_scale[1, 0, 3] = 4080.0
    want = layer.dequantize_weight()
    layer.float().half()
    assert layer.weight_scale.dtype == torch.float16 and torch.equal(layer.dequantize_weight(), want)
    layer.to("meta").half()


# ---- multiview positions -----------------------------------------------------------------------
def test_multiview_positions_go_where_the_model_goes(pkg):
    un = importlib.import_module(PKG + ".unet")
    blk = un.TransformerBlock(128, 2, 128, 2)
    given = {8: 500001 + torch.arange(8), 4: torch.arange(4).int()}
    un.use_multiview_rotary(blk, given)
    blk.to(torch.bfloat16).double().type(torch.float16)      # types of weights are not types of positions
    assert [t.dtype for t in blk.attn_mv.rotary_positions.values()] == [torch.int64, torch.int32]
    assert torch.equal(blk.attn_mv.rotary_positions[8], given[8])
    nn.Sequential(blk).to("meta")
    assert all(t.device.type == "meta" for t in blk.attn_mv.rotary_positions.values())
    assert given[8].device.type == "cpu" and blk.attn1.rotary_positions is None


def test_multiview_positions_that_are_missing_or_do_not_fit(pkg):
    un = importlib.import_module(PKG + ".unet")
    blk = un.TransformerBlock(128, 2, 128, 2)
    un.use_multiview_rotary(blk, {8: torch.arange(8)})
    with pytest.raises(RuntimeError, match="12 tokens.*8"):
        blk.attn_mv(torch.zeros(1, 12, 128))
    other = nn.Sequential(un.TransformerBlock(128, 2, 128, 2), un.TransformerBlock(128, 32, 128, 2))      # heads of 64, and of 4
    for bad in ({8: torch.zeros(8, 3, dtype=torch.int64)}, {8: torch.zeros(8)}, {8: torch.zeros(8, 2, 2, dtype=torch.int64)}, {}):
        with pytest.raises(RuntimeError):
            un.use_multiview_rotary(other, bad)
        assert all(b.attn_mv.rotary is None and b.attn_mv.rotary_positions is None for b in other)


# ---- the scales' type ----------------------------------------------------------------------------
def test_int4_scales_take_the_type_that_is_asked_for(qu):
    torch.manual_seed(5)
    lin = nn.Linear(128, 128)
    for dt in (torch.float16, torch.bfloat16):
        for symmetric in (True, False):
            layer = qu.Int4Linear.from_linear(lin, 64, symmetric, dtype=dt)
            assert layer.weight_scale.dtype == dt and layer.bias.dtype == dt
            # half a step for the code, or where the range ends for the zero point; there the scale's rounding 15 times too
            step = layer.scales().float().repeat_interleave(64, 1)
            assert bool(((layer.dequantize_weight() - lin.weight).abs() <= step * (0.5 + 15 * torch.finfo(dt).eps)).all())
        net = nn.Sequential(nn.Linear(128, 128))
        qu.quantize_model_int4(net, verbose=False, dtype=dt)
        assert net[0].weight_scale.dtype == dt
    assert qu.Int4Linear.from_linear(lin).weight_scale.dtype == torch.float16
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        qu.Int4Linear.from_linear(lin, dtype=torch.float32)


# ---- modules that have run can be copied --------------------------------------------------------
def test_modules_keep_no_library_handle(qu, pkg, build_mod):
    """A model is copied and saved whole also after its first call, which loads the library."""
    import copy
    import pickle
    un = importlib.import_module(PKG + ".unet")
    x = torch.zeros(2, 64).half()
    for m in (qu.AddRMSNorm(nn.RMSNorm(64)), qu.Int8RMSNorm(nn.RMSNorm(64)), qu.Int8LayerNorm(nn.LayerNorm(64)),
              qu.Int4Linear(64, 16), un.GroupNormNHWC(32, 64)):
        with contextlib.suppress(RuntimeError):      # the library is loaded, and the CPU refused
            m(x)
        assert set(copy.deepcopy(m).state_dict()) == set(m.state_dict())
        assert type(pickle.loads(pickle.dumps(m))) is type(m)
        assert all(not isinstance(v, importlib.import_module(PKG + ".csrc._binding")._Base) for v in vars(m).values())
