"""CPU: what Int4Linear, the RMSNorms and the rotary positions do before a kernel runs -- layouts, plans, refusals."""
import ctypes
import importlib
import math

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


# ---- Int4Linear -------------------------------------------------------------------------
def test_packed_codes_are_where_the_header_says(qu):
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 16, (48, 192), generator=g, dtype=torch.uint8)
    words = qu._pack_codes(codes).view(3, 3, 32, 4, 4).to(torch.int64)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    for rb, tile, lane, word, nibble in [(0, 0, 0, 0, 0), (2, 1, 31, 3, 7), (1, 2, 13, 1, 5), (0, 2, 6, 2, 3), (2, 0, 17, 0, 4)]:
        row = rb * 16 + lane // 4 + 8 * (word & 1)
        i = 2 * nibble if nibble < 4 else 2 * (nibble - 4) + 1
        col = tile * 64 + 32 * (word >> 1) + 16 * (i >> 2) + 4 * (lane % 4) + (i & 3)
        assert int(words[rb, tile, lane, word] >> (4 * nibble) & 15) == int(codes[row, col])
    assert torch.equal(qu._unpack_codes(qu._pack_codes(codes)), codes)
    v = torch.randn(48, 5, generator=g)
    packed = qu._pack_groups(v)
    assert packed[1, 3, 2 * 5] == v[16 + 5, 3] and packed[1, 3, 2 * 5 + 1] == v[16 + 13, 3]
    assert torch.equal(qu._unpack_groups(packed), v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 192])
def test_conversion_rounds_to_the_nearest_code(qu, dtype, symmetric, group):
    torch.manual_seed(1)
    lin = nn.Linear(192, 48).to(dtype)
    lin.weight.data[3] = 0                                       # a row of zeros
    lin.weight.data[4, :group] = lin.weight.data[4, :group].abs() + 0.01   # a group of one sign
    layer = qu.Int4Linear.from_linear(lin, group, symmetric)
    assert layer.group_size == group and (layer.weight_zero is None) == symmetric
    w, s = lin.weight.data.double(), layer.scales().double().repeat_interleave(group, 1)
    err = (layer.dequantize_weight().double() - w).abs()
    # half a step, and what clamping at the ends of the codes may cost: the scale is rounded to 16 bits (relative eps / 2),
    # so the largest weight may lie 7 (15) times that beyond the last code's half step, and a zero point is off by up to half
    eps = torch.finfo(layer.weight_scale.dtype).eps
    assert bool((err <= s * ((0.5 if symmetric else 1.0) + 16 * eps)).all())
    assert bool((layer.dequantize_weight()[3] == 0).all())
    assert layer.codes().max() <= 15 and layer.scales().dtype == (dtype if dtype != torch.float32 else torch.float16)


def test_int4_from_codes_concat_geglu_and_state(qu):
    g = torch.Generator().manual_seed(2)
    def layer(n, zeros=True):
        return qu.Int4Linear.from_codes(torch.randint(0, 16, (n, 128), generator=g), torch.rand(n, 2, generator=g).half(),
                                        torch.randint(0, 16, (n, 2), generator=g) if zeros else None, torch.randn(n, generator=g))
    parts = [layer(32), layer(64)]
    cat = qu.Int4Linear.concat(parts)
    assert cat.out_features == 96 and torch.equal(cat.dequantize_weight(), torch.cat([p.dequantize_weight() for p in parts]))
    assert torch.equal(cat.bias, torch.cat([p.bias for p in parts])) and cat.bias.dtype == torch.float16
    with pytest.raises(RuntimeError):
        qu.Int4Linear.concat([parts[0], layer(32, zeros=False)])
    with pytest.raises(TypeError):
        qu.Int4Linear.concat([parts[0], nn.Linear(128, 32)])
    w, b = cat.dequantize_weight(), cat.bias.clone()
    cat.interleave_geglu_rows()
    order = torch.cat([torch.cat([torch.arange(16 * i, 16 * i + 16), torch.arange(48 + 16 * i, 64 + 16 * i)]) for i in range(3)])
    assert torch.equal(cat.dequantize_weight(), w[order]) and torch.equal(cat.bias, b[order])
    with pytest.raises(RuntimeError):
        cat.interleave_geglu_rows()
    other = qu.Int4Linear(128, 96, bias=False, dtype=torch.bfloat16, group_size=32)
    other.load_state_dict(cat.state_dict())
    assert other.epilogue == "geglu" and other.group_size == 64 and torch.equal(other.dequantize_weight(), cat.dequantize_weight())
    assert torch.equal(other.bias, cat.bias) and torch.equal(other.zeros(), cat.zeros())
    with pytest.raises(RuntimeError):
        qu.Int4Linear(128, 64).load_state_dict(cat.state_dict())
    state = {f"{p}.{k}": v for p, l in zip("ab", parts) for k, v in l.state_dict().items()}
    qu.Int4Linear.concat_state(state, "c.", ["a.", "b."])
    fresh = qu.Int4Linear(128, 96)
    fresh.load_state_dict({k[2:]: v for k, v in state.items()})
    assert torch.equal(fresh.dequantize_weight(), w)


def test_int4_refusals(qu):
    for args in [(100, 64), (64, 24), (128, 64, True, torch.float16, 48), (128, 64, True, torch.float16, 96),
                 (192, 64, True, torch.float16, 128), (128, 64, True, torch.float32), (0, 16)]:
        with pytest.raises(RuntimeError):
            qu.Int4Linear(*args)
    codes, scale = torch.zeros(16, 64, dtype=torch.uint8), torch.ones(16, 1).half()
    for bad in [(codes + 16, scale), (codes.float(), scale), (codes, scale.float()), (codes, scale[:8]),
                (codes, scale, scale), (codes, scale, torch.full((16, 1), 16)), (codes, scale, None, torch.zeros(8))]:
        with pytest.raises(RuntimeError):
            qu.Int4Linear.from_codes(*bad)
    layer = qu.Int4Linear.from_codes(codes, scale)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(torch.zeros(2, 64).half())
    with pytest.raises(RuntimeError, match="16-bit"):
        layer(qu.QuantizedActivation(codes, scale, (16, 64), torch.float16))


@pytest.mark.parametrize("dt,most", [(torch.float16, 4094.0), (torch.bfloat16, 2.1e37)])
def test_int4_scales_leave_every_weight_in_range(qu, dt, most):
    """A sixteenth of the largest number: 15 times that is finite, in a scale's own type."""
    codes = torch.full((16, 64), 15)
    zero = torch.zeros(16, 1, dtype=torch.uint8)
    layer = qu.Int4Linear.from_codes(codes, torch.full((16, 1), most).to(dt), zero)
    assert torch.isfinite(layer.dequantize_weight().to(dt)).all()
    for bad in (most * 1.02, -most * 1.02, float("inf"), float("nan")):
        scale = torch.ones(16, 1, dtype=dt)
        scale[3, 0] = bad
        with pytest.raises(RuntimeError, match="scale"):
            qu.Int4Linear.from_codes(codes, scale, zero)
    wide = nn.Linear(64, 16, bias=False).to(dt)
    with torch.no_grad():
        wide.weight[2, 5] = most * 7.5
    with pytest.raises(RuntimeError, match="scale"):
        qu.Int4Linear.from_linear(wide)


def test_int4_model_surgery(qu):
    torch.manual_seed(3)
    net = nn.Sequential(nn.Linear(128, 256), nn.Sequential(nn.Linear(256, 64), nn.Linear(256, 200)), nn.Linear(256, 256))
    stats = qu.quantize_model_int4(net, group_size=128, choose=lambda name, m: not name.startswith("2"), verbose=False)
    assert isinstance(net[0], qu.Int4Linear) and isinstance(net[2], nn.Linear) and isinstance(net[1][1], nn.Linear)
    assert stats == {"total_params": 128 * 256 + 256 * 64 + 256 * 200 + 256 * 256, "quantized_params": 128 * 256,
                     "skipped_params": 256 * 64, "num_replaced": 1, "kept_fp16": 2}


def test_time_projections_of_four_bits_stack(qu, pkg):
    un = importlib.import_module(PKG + ".unet")
    def model(seed):
        torch.manual_seed(seed)
        net = un.UNetSD21MV(block_out_channels=(128, 128), layers_per_block=1, attention_heads=(2, 2),
                            cross_attention_dim=128, attn_levels=(True, False), num_views=2)
        qu.quantize_model_int4(net, choose=lambda name, _: "time_emb_proj" in name, verbose=False)
        return net
    separate, stacked = model(1), model(2)
    old = separate.state_dict()
    assert un.fuse_time_projections(stacked) == 7 and type(stacked.time_proj_all) is qu.Int4Linear
    stacked.load_state_dict(old)
    assert torch.equal(stacked.time_proj_all.dequantize_weight(),
                       torch.cat([m.time_emb_proj.dequantize_weight() for m in separate._resnets()]))


# ---- C entry points: bad arguments, found before any device is asked ---------------------
P = 1 << 20      # an address that is aligned and never read


def test_rmsnorm_refuses_bad_arguments(lib):
    def call(x=P, ldx=64, add=None, ld_add=0, total=None, code=0, M=4, K=64, gamma=P, g=0, eps=1e-6, y=P, q=None, s=None):
        return lib.hy3d_rmsnorm(x, ldx, add, ld_add, total, code, M, K, gamma, g, eps, y, q, s, None)
    assert call(M=0) == 0 and call(M=0, x=None, y=None) == 0
    for bad in [dict(code=2), dict(g=3), dict(eps=-1.0), dict(eps=math.nan), dict(x=None), dict(y=None), dict(q=P, s=None),
                dict(add=P, ld_add=64)]:
        assert call(**bad) == 1, bad
    for bad in [dict(K=60), dict(K=0), dict(K=16392, ldx=16392), dict(M=-1), dict(ldx=56), dict(ldx=68), dict(add=P, ld_add=60, total=P),
                dict(x=P + 2), dict(gamma=P + 2), dict(y=P + 8), dict(q=P + 4, s=P), dict(add=P + 2, ld_add=64, total=P),
                dict(add=P, ld_add=64, total=P + 2)]:
        assert call(**bad) == 2, bad
    d = lambda q=P, s=P, M=4, K=64, code=0, y=P: lib.hy3d_dequantize_rows(q, s, M, K, code, y, None)
    assert d(M=0) == 0 and d(code=2) == 1 and d(q=None) == 1 and d(K=12) == 2 and d(y=P + 8) == 2 and d(M=-1) == 2


def test_linear_w4_refuses_bad_arguments(lib):
    def call(x=P, code=0, ldx=128, w=P, s=P, sc=0, z=None, group=64, b=None, bc=0, out=P, M=4, N=32, K=128, epi=0):
        return lib.hy3d_linear_w4(x, code, ldx, w, s, sc, z, group, b, bc, out, M, N, K, epi, None)
    assert call(M=0) == 0
    for bad in [dict(code=2), dict(sc=2), dict(epi=3), dict(epi=-1), dict(b=P, bc=3), dict(x=None), dict(w=None), dict(s=None), dict(out=None)]:
        assert call(**bad) == 1, bad
    for bad in [dict(K=96, ldx=96), dict(N=24), dict(N=0), dict(N=48, epi=2), dict(group=16), dict(group=96), dict(group=0), dict(group=256),
                dict(ldx=120), dict(ldx=132), dict(x=P + 8), dict(w=P + 8), dict(s=P + 2), dict(M=-1)]:
        assert call(**bad) == 2, bad


class Side(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in
                ("src_b", "src_n", "src_h", "dst_b", "dst_n", "dst_h")] + [("heads", ctypes.c_int)]


def test_rotary_refuses_bad_arguments(lib):
    turns, axis = (ctypes.c_uint64 * 256)(), (ctypes.c_uint8 * 256)()
    def call(n_sides=1, code=0, batch=1, n=4, dim=64, rot=64, src=P, heads=2, turns=turns, axis=axis):
        sides = (Side * 2)(*[Side(src, src, 512, 128, 64, 512, 128, 64, heads)] * 2)
        return lib.hy3d_rotary(sides, n_sides, code, batch, n, dim, rot, 0, None, 0, 0, 0, 0, 0, turns, axis, 1.0, 0, None)
    assert call(batch=0) == 0 and call(n=0) == 0 and call(heads=0) == 0
    for bad in [dict(n_sides=0), dict(n_sides=3), dict(code=2), dict(turns=None), dict(axis=None), dict(src=None)]:
        assert call(**bad) == 1, bad
    for bad in [dict(rot=63), dict(rot=0), dict(rot=66), dict(rot=514, dim=600), dict(dim=0), dict(n=-1), dict(src=P + 1), dict(heads=-1),
                dict(n=1 << 31)]:
        assert call(**bad) == 2, bad


# ---- rotary plans -------------------------------------------------------------------------
def test_rotary_frequencies(rotary):
    r = rotary.RotaryPositions(64, base=10000.0)
    assert r.frequencies[0] == 1.0 and math.isclose(r.frequencies[31], 10000.0 ** (-62 / 64))
    turns = memoryview(r._turns).cast("Q")
    for w, t in zip(r.frequencies, turns):
        assert abs(t / 2.0 ** 64 - w / (2 * math.pi)) <= 2.0 ** -52 * w + 2.0 ** -64      # the last unit is cut off
    lin = rotary.RotaryPositions(64, scaling={"kind": "linear", "factor": 8})
    assert all(math.isclose(a, b / 8) for a, b in zip(lin.frequencies, r.frequencies))
    ntk = rotary.RotaryPositions(64, scaling={"kind": "ntk", "factor": 8})
    assert ntk.frequencies[0] == 1.0 and math.isclose(ntk.frequencies[31], r.frequencies[31] / 8)
    parts = rotary.RotaryPositions(64, scaling={"kind": "by_parts", "factor": 8, "original_length": 4096})
    for a, b in zip(parts.frequencies, r.frequencies):
        turned = 4096 * b / (2 * math.pi)
        assert math.isclose(a, b if turned >= 4 else b / 8) if not 1 < turned < 4 else b / 8 < a < b
    grid = rotary.RotaryPositions(64, axes=(24, 20, 20))
    assert list(grid._axis) == [0] * 12 + [1] * 10 + [2] * 10 and grid.frequencies[12] == grid.frequencies[22] == 1.0
    assert rotary.RotaryPositions(2, scaling={"kind": "ntk", "factor": 2}).frequencies == [1.0]


def test_rotary_plan_and_call_refusals(rotary):
    for bad in [dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=0), dict(axes=(30, 30)), dict(axes=(33, 31)), dict(axes=()),
                dict(base=0.0), dict(base=math.inf), dict(amplitude=math.nan), dict(scaling={"kind": "cubic", "factor": 2}),
                dict(scaling={"kind": "linear"}), dict(scaling={"kind": "linear", "factor": -1}), dict(scaling={"kind": "linear", "factor": 2, "fast": 3}),
                dict(scaling={"kind": "by_parts", "factor": 2}), dict(scaling={"kind": "by_parts", "factor": 2, "original_length": 9, "slow": 4, "fast": 4})]:
        with pytest.raises(RuntimeError):
            rotary.RotaryPositions(64, **bad)
    r = rotary.RotaryPositions(64)
    for bad in [torch.zeros(1, 2, 3, 64), None, [1]]:
        with pytest.raises(RuntimeError, match="CUDA"):
            r(bad)


# ---- norms -----------------------------------------------------------------------------------
def test_norm_modules_refuse_what_they_cannot_run(qu):
    for cls in (qu.AddRMSNorm, qu.Int8RMSNorm):
        with pytest.raises(RuntimeError, match="last dimension"):
            cls(nn.RMSNorm((4, 8)))
        norm = cls(nn.RMSNorm(64))
        with pytest.raises(RuntimeError, match="CUDA"):
            norm(torch.zeros(2, 64).half())
        with pytest.raises(RuntimeError, match="CUDA"):
            norm(torch.zeros(2, 64).half(), torch.zeros(2, 64).half())
        with pytest.raises(RuntimeError, match="64 dimensions"):
            norm(torch.zeros(2, 32).half())
        assert list(norm.state_dict()) == ["weight"]


def test_row_pitches(qu, build_mod):
    rows = build_mod.load_int8_kernels()._rows
    t = torch.zeros(4, 6, 96)
    assert rows(t, "") == (24, 96) and rows(t[..., :64], "") == (24, 96) and rows(t[:, :3], "") is None
    assert rows(t[:, ::2], "") == (12, 192) and rows(t.transpose(0, 1), "") is None and rows(t[..., ::2], "") is None
    assert rows(t[:1], "") == (6, 96) and rows(t[0, 0], "") == (1, 96) and rows(t[0, 0].expand(5, 96), "") is None
    assert rows(torch.zeros(4, 36)[:, :32], "") is None         # a pitch that is not whole vectors


def test_fuse_layernorm_quant_takes_rmsnorms(qu, pkg):
    un = importlib.import_module(PKG + ".unet")
    blk = un.TransformerBlock(128, 2, 128, 2)
    blk.norm1, blk.norm2 = nn.RMSNorm(128), nn.RMSNorm(128)
    qu.quantize_model_tensorcore(blk, verbose=False)
    assert un.fuse_layernorm_quant(blk) == 4
    assert type(blk.norm1) is qu.Int8RMSNorm and type(blk.norm_mv) is qu.Int8LayerNorm


def test_multiview_rotary_is_set_where_there_are_views(pkg):
    un = importlib.import_module(PKG + ".unet")
    blk = un.TransformerBlock(128, 2, 128, 2)
    positions = {8: torch.zeros(8, 3, dtype=torch.int64)}
    assert un.use_multiview_rotary(nn.Sequential(blk, un.TransformerBlock(128, 2, 128, 1)), positions) == 1
    assert blk.attn_mv.rotary.axes == (22, 22, 20) and blk.attn1.rotary is None
    with pytest.raises(RuntimeError):
        un.use_multiview_rotary(blk, {8: torch.zeros(7, 3, dtype=torch.int64)})
    with pytest.raises(RuntimeError, match="CUDA"):
        with torch.no_grad():
            blk(torch.zeros(2, 4, 128), torch.zeros(2, 3, 128))
