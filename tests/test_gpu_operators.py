"""GPU: Int4Linear, AddRMSNorm / Int8RMSNorm and RotaryPositions against their definitions in 64 bits, and a run of them
together.  Tolerances: half a step of the output type plus the fp32 errors derived beside each."""
import importlib
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
PKG = "hunyuan3d-tools_b200"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative to the value
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}    # half a step of the subnormals


@pytest.fixture(scope="module")
def rotary():
    return importlib.import_module(PKG + ".rotary")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _within(y, ref, tol):
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((y.double() - ref).abs() - tol).max()):.3g} over"


# ---- Int4Linear -------------------------------------------------------------------------
def _int4(qu, n, k, group, zeros, bias, dtype, seed, epilogue="linear"):
    g = _gen(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(n, k // group, generator=g, device=DEV) * 0.02 + 0.001).to(dtype)
    zero = torch.randint(0, 16, (n, k // group), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    b = (torch.randn(n, generator=g, device=DEV) * 0.5).to(dtype) if bias else None
    layer = qu.Int4Linear.from_codes(codes, scale, zero, b)
    w = layer.dequantize_weight().double()      # exact: a 16-bit scale times a whole number below 16
    assert torch.equal(w, (codes.double() - (8 if zero is None else zero.double().repeat_interleave(group, 1)))
                       * scale.double().repeat_interleave(group, 1))
    if epilogue == "geglu":
        layer.interleave_geglu_rows()
    else:
        layer.epilogue = epilogue
    return layer, w, None if b is None else b.double()


def _check_int4(layer, w, b, x, y):
    """fp32 sums: K / 16 steps of a 16-deep product whose running sum may lose 2^-22 of the magnitudes it holds, a
    scaling per group, the joins of the K ranges: (K / 16 + K / 32 + 16) 2^-22 of sum |x| |w|."""
    k, dtype = w.shape[1], x.dtype
    x64 = x.double().reshape(-1, k)
    ref, mag = x64 @ w.t(), x64.abs() @ w.abs().t()
    if b is not None:
        ref, mag = ref + b, mag + b.abs()
    err = (k / 16 + k / 32 + 16) * 2.0 ** -22 * mag
    gelu = lambda v: v * torch.special.ndtr(v)      # its slope is at most 1.13; the kernel's own error 3e-7 plus a rounding
    if layer.epilogue == "gelu":
        ref, err = gelu(ref), 1.13 * err + 3e-7 + 2.0 ** -23 * ref.abs()
    elif layer.epilogue == "geglu":
        h = ref.shape[1] // 2
        v, g, ev, eg = ref[:, :h], ref[:, h:], err[:, :h], err[:, h:]
        eg = 1.13 * eg + 3e-7 + 2.0 ** -23 * g.abs()
        ref, err = v * gelu(g), ev * (gelu(g).abs() + eg) + (v.abs() + ev) * eg + 2.0 ** -23 * (v * g).abs()
    _within(y.reshape(ref.shape), ref, err + HALF[dtype] * (ref.abs() + err) + TINY[dtype])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,group,zeros,bias,epilogue", [
    (1, 64, 16, 64, False, False, "linear"), (1, 64, 32, 32, True, True, "geglu"), (1, 8192, 640, 128, False, True, "linear"),
    (2, 1280, 656, 64, True, True, "gelu"), (7, 1280, 2560, 32, True, False, "geglu"), (8, 320, 1280, 320, False, True, "linear"),
    (9, 1024, 48, 1024, True, True, "linear"), (12, 1280, 640, 64, False, True, "linear"), (16, 4096, 80, 128, False, False, "gelu"),
    (17, 640, 336, 32, True, True, "linear"), (33, 1536, 1056, 64, True, True, "geglu"), (77, 192, 272, 192, False, False, "linear"),
    (100, 704, 144, 64, True, True, "gelu"), (257, 1536, 1536, 128, False, True, "gelu"), (924, 1024, 2560, 64, False, False, "linear"),
    (1000, 2560, 32, 32, True, True, "geglu"), (129, 128, 16, 128, True, True, "linear"), (64, 5120, 160, 64, False, True, "linear")])
def test_int4_linear(qu, dtype, m, k, n, group, zeros, bias, epilogue):
    layer, w, b = _int4(qu, n, k, group, zeros, bias, dtype, m + k + n, epilogue)
    x = torch.randn(m, k, generator=_gen(m), device=DEV).to(dtype)
    y = layer(x)
    assert y.dtype == dtype and y.shape == (m, n // 2 if epilogue == "geglu" else n)
    _check_int4(layer, w, b, x, y)
    assert torch.equal(y, layer(x))                       # no order of addition is left to chance


def test_int4_leading_dimensions_strides_and_scale_types(qu):
    layer, w, b = _int4(qu, 96, 128, 64, True, True, torch.float16, 5)
    wide = torch.randn(3, 5, 256, generator=_gen(1), device=DEV).half()
    for x in (wide[..., 128:], wide[:, :, :128], wide.transpose(0, 1)[..., :128], wide[0, 0, :128], wide[:0, :, :128],
              torch.randn(1 + 15 * 128, generator=_gen(2), device=DEV).half()[1:].view(3, 5, 128)):      # off a 16-byte boundary
        y = layer(x)
        assert y.shape == (*x.shape[:-1], 96)
        if x.numel():
            _check_int4(layer, w, b, x, y)
    x = wide[..., :128].bfloat16().contiguous()            # fp16 scales and bias on bf16 activations
    _check_int4(layer, w, b, x, layer(x))
    layer.bias = layer.bias.float()
    _check_int4(layer, w, b, x, layer(x))


@pytest.mark.parametrize("k,n,group,zeros,epilogue", [(576, 176, 32, True, "linear"), (2048, 288, 64, False, "geglu"),
                                                      (32768, 48, 256, True, "gelu")])
def test_int4_every_number_of_tokens_around_the_kernels_limits(qu, k, n, group, zeros, epilogue):
    """8 tokens a pass of one kernel, 16 a column block of the other, 256 a CTA; rows of x taken out of a longer matrix."""
    layer, w, b = _int4(qu, n, k, group, zeros, True, torch.float16, k, epilogue)
    x = (torch.randn(520, k + 64, generator=_gen(n), device=DEV) * (2.0 if k < 32768 else 0.125)).half()[:, :k]
    for m in (1, 7, 8, 9, 15, 16, 17, 24, 33, 63, 64, 65, 80, 255, 256, 257, 513):
        _check_int4(layer, w, b, x[:m], layer(x[:m]))


@pytest.mark.parametrize("dtype,size,values", [(torch.float16, 2.0 ** -21, 1000.0), (torch.float16, 4094.0, 2.0 ** -9),
                                               (torch.bfloat16, 2.0 ** -126, 2.0 ** 20), (torch.bfloat16, 2.0 ** 60, 1.0)])
def test_int4_scales_at_the_ends_of_their_type(qu, dtype, size, values):
    """The two numbers of a weight are exact for subnormal scales and for the largest; activations of a size that keeps
    products and results in range."""
    g = _gen(8)
    scale = (size * (torch.rand(176, 4, generator=g, device=DEV).double() * 0.9 + 0.1)).to(dtype)
    codes = torch.randint(0, 16, (176, 256), generator=g, device=DEV)
    zero = torch.randint(0, 16, (176, 4), generator=g, device=DEV)
    layer = qu.Int4Linear.from_codes(codes, scale, zero)
    w = (codes - zero.repeat_interleave(64, 1)).double() * scale.double().repeat_interleave(64, 1)
    x = (torch.randn(100, 256, generator=g, device=DEV) * values).to(dtype)
    for m in (3, 100):
        _check_int4(layer, w, None, x[:m], layer(x[:m]))


def test_int4_scales_of_another_type_for_many_rows(qu):
    layer, w, b = _int4(qu, 112, 448, 64, True, True, torch.bfloat16, 9)
    x = torch.randn(333, 448, generator=_gen(3), device=DEV).half()
    _check_int4(layer, w, b, x, layer(x))


def test_int4_infinities_and_nans_stay_in_their_rows(qu):
    layer, w, b = _int4(qu, 64, 256, 64, False, True, torch.bfloat16, 6)
    for m in (5, 40, 300):
        x = torch.randn(m, 256, generator=_gen(m), device=DEV).bfloat16()
        x[1, 7], x[3, 100] = math.nan, math.inf
        y = layer(x)
        assert bool(y[1].isnan().all()) and not bool(y[3].isfinite().any())
        rest = [i for i in range(m) if i not in (1, 3)]
        _check_int4(layer, w, b, x[rest], y[rest])


def test_int4_refuses_on_the_gpu(qu):
    layer, _, _ = _int4(qu, 64, 128, 64, False, True, torch.bfloat16, 7)
    x = torch.randn(4, 128, device=DEV)
    with pytest.raises(RuntimeError, match="bf16"):
        layer(x)
    with pytest.raises(RuntimeError, match="input features"):
        layer(x[:, :64].bfloat16())
    with pytest.raises(RuntimeError, match="gradient"):
        layer(x.bfloat16().requires_grad_())
    with torch.no_grad():
        layer(x.bfloat16().requires_grad_())
    with pytest.raises(RuntimeError):
        qu.Int4Linear(128, 64)(x.half())                   # the layer is on the CPU
    layer.epilogue = "relu"
    with pytest.raises(RuntimeError, match="epilogue"):
        layer(x.bfloat16())


def test_int4_hooks_and_subclasses_are_called(qu):
    layer, w, b = _int4(qu, 64, 128, 64, False, True, torch.bfloat16, 8)
    x = torch.randn(4, 128, device=DEV).bfloat16()
    seen = []
    handle = layer.register_forward_hook(lambda *a: seen.append(1))
    y = layer(x)
    handle.remove()
    assert seen == [1] and torch.equal(y, layer(x))

    class Doubled(qu.Int4Linear):
        def forward(self, x):
            return 2 * super().forward(x)
    layer.__class__ = Doubled
    assert torch.equal(layer(x), 2 * y)


# ---- norms -----------------------------------------------------------------------------------
def _check_norm(x, add, weight, eps, total, y):
    """The sum is the 16-bit addition's own.  The statistics are a sum of squares, 2^-24 per addition along a chain of at
    most 50, halved by the root, then a root, a reciprocal and two products: 2^-18 of the value in all."""
    dtype, t = x.dtype, x
    if add is not None:
        t = x + add
        assert torch.equal(total, t)
    f = t.double()
    ref = f / (f.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        ref = ref * weight.double()
    tol = HALF[dtype] * (1 + 2.0 ** -18) * ref.abs() + 2.0 ** -18 * ref.abs() + TINY[dtype]
    _within(y, ref, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 40), (1, 4096), (5, 64), (257, 1536), (1000, 320), (33, 1288), (77, 2560),
                                        (2, 2568), (129, 5120), (9, 8192), (300, 10248), (7, 16384), (1, 16384)])
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm(qu, ik, dtype, rows, width, residual):
    g = _gen(rows + width)
    x = torch.randn(rows, width, generator=g, device=DEV).to(dtype) * 3
    add = torch.randn(rows, width, generator=g, device=DEV).to(dtype) if residual else None
    norm = nn.RMSNorm(width, eps=1e-6, device=DEV, dtype=dtype)
    norm.weight.data.copy_(1 + 0.2 * torch.randn(width, generator=g, device=DEV))
    half, codes = qu.AddRMSNorm(norm), qu.Int8RMSNorm(norm)
    assert half.weight is norm.weight
    total, y = half(x, add) if residual else (None, half(x))
    _check_norm(x, add, norm.weight, 1e-6, total, y)
    total8, q = codes(x, add) if residual else (None, codes(x))
    assert residual is False or torch.equal(total8, total)
    want_q, want_s = ik.fused_quantize_activation(y)
    assert torch.equal(q.q, want_q) and torch.equal(q.scale, want_s)
    assert torch.equal(q.dequantize(), (want_q.float() * want_s[:, None]).to(dtype).view(y.shape))
    # both outputs of one launch, and each row by itself: the same bits
    _, y2, q2, s2 = ik.rmsnorm(x, norm.weight, 1e-6, add, codes=True, normalised=True)
    assert torch.equal(y2, y) and torch.equal(q2, want_q) and torch.equal(s2, want_s)
    i = rows // 2
    one = half(x[i:i + 1], add[i:i + 1])[1] if residual else half(x[i:i + 1])
    assert torch.equal(one[0], y[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rmsnorm_parameters_strides_and_shapes(qu, ik, dtype):
    g = _gen(11)
    wide = torch.randn(4, 6, 3 * 320, generator=g, device=DEV).to(dtype)
    add = torch.randn(4, 6, 320, generator=g, device=DEV).to(dtype)
    norms = [nn.RMSNorm(320, eps=1e-5, elementwise_affine=False), nn.RMSNorm(320, device=DEV), nn.RMSNorm(320, device=DEV, dtype=dtype)]
    norms[1].weight.data.normal_()
    norms[2].weight = nn.Parameter(torch.randn(321, device=DEV, dtype=dtype)[1:], requires_grad=False)     # off its boundary
    for norm in norms:
        eps = norm.eps if norm.eps is not None else torch.finfo(dtype).eps
        for x in (wide[..., 320:640], wide[:, ::2, :320], wide.transpose(0, 1)[..., :320], wide[:0, :, :320],
                  wide.flatten()[1:1 + 24 * 320].view(4, 6, 320)):
            a = add[:x.shape[0], :x.shape[1]] if x.shape[0] != 6 else add.transpose(0, 1)
            total, y = qu.AddRMSNorm(norm)(x, a)
            assert y.shape == x.shape and total.shape == x.shape
            _check_norm(x, a, norm.weight, eps, total, y)
            assert torch.equal(qu.Int8RMSNorm(norm)(x, a)[1].q, ik.fused_quantize_activation(y.reshape(-1, 320))[0] if y.numel()
                               else y.reshape(-1, 320).to(torch.int8))


def test_rmsnorm_rows_that_are_not_finite_and_rows_of_zeros(qu):
    for dtype in HALF:
        x = torch.randn(6, 640, generator=_gen(3), device=DEV).to(dtype)
        x[1, 5], x[2, 600], x[4] = math.nan, -math.inf, 0
        norm = nn.RMSNorm(640, eps=1e-6, device=DEV, dtype=dtype)
        y, q = qu.AddRMSNorm(norm)(x), qu.Int8RMSNorm(norm)(x).dequantize()
        assert bool(y[1].isnan().all()) and bool(y[2, 600].isnan()) and bool((y[2, :600] == 0).all())
        assert bool(q[1:3].isnan().all()) and bool((q[4] == 0).all()) and bool((y[4] == 0).all())
        ok = [0, 3, 5]
        _check_norm(x[ok], None, norm.weight, 1e-6, None, y[ok])
        assert bool(q[ok].isfinite().all())


def test_rmsnorm_sum_in_place_of_an_input(qu, build_mod):
    """The C entry point may put the sum where x or add is, also for a block's threads behind the last row."""
    lib = importlib.import_module(PKG + ".csrc._binding").configure(build_mod.load_library())
    for rows, width in ((1, 640), (3, 5120), (37, 328)):
        x, add = (torch.randn(rows, width, generator=_gen(rows), device=DEV).half() for _ in range(2))
        add = add + 1
        y = torch.empty_like(x)
        for where in (0, 1):
            a, b = x.clone(), add.clone()
            assert lib.hy3d_rmsnorm(a.data_ptr(), width, b.data_ptr(), width, (a, b)[where].data_ptr(), 0, rows, width, None, 2, 1e-6,
                                    y.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream) == 0
            _check_norm(x, add, None, 1e-6, (a, b)[where], y)


def test_norm_refusals_on_the_gpu(qu):
    norm = qu.AddRMSNorm(nn.RMSNorm(64, device=DEV))
    x = torch.zeros(2, 64, device=DEV).half()
    for args in [(x.float(),), (x, x.bfloat16()), (x, x[:1]), (x, x.cpu()), (x[:, :60],), (x.requires_grad_(),)]:
        with pytest.raises(RuntimeError):
            norm(*args)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        qu.AddRMSNorm(nn.RMSNorm(60, device=DEV))(torch.zeros(2, 60, device=DEV).half())
    with pytest.raises(RuntimeError, match="weight"):
        qu.AddRMSNorm(nn.RMSNorm(64))(torch.zeros(2, 64, device=DEV).half())


# ---- rotary ------------------------------------------------------------------------------------
def _turned(r, t, positions, inverse=False):
    """(reference, tolerance): sine and cosine of an angle known to 2^-32 turns, converted and evaluated in fp32 (4e-7
    together), two products and a sum of them."""
    t64, amp = t.double(), r.amplitude
    p = positions if positions.dim() > 1 or len(r.axes) == 1 else positions[:, None]
    p = p[..., None] if len(r.axes) == 1 and (p.dim() < t.dim() - 1) else p
    axis = torch.tensor(list(r._axis), device=t.device)
    a = p.double()[..., axis] * torch.tensor(r.frequencies, dtype=torch.float64, device=t.device)
    a = (-a if inverse else a)[..., None, :]
    c, s = a.cos() * amp, a.sin() * amp
    h = r.rotary_dim // 2
    u, v = (t64[..., 0:2 * h:2], t64[..., 1:2 * h:2]) if r.interleaved else (t64[..., :h], t64[..., h:2 * h])
    y, z, m = u * c - v * s, v * c + u * s, (u.abs() + v.abs()) * abs(amp) * 4e-7
    ref, tol = t64.clone(), torch.zeros_like(t64)
    for dst, value, err in ((ref, (y, z), None), (tol, (m, m), None)):
        if r.interleaved:
            dst[..., 0:2 * h:2], dst[..., 1:2 * h:2] = value
        else:
            dst[..., :h], dst[..., h:2 * h] = value
    tol[..., :2 * h] += HALF[t.dtype] * (ref[..., :2 * h].abs() + tol[..., :2 * h]) + TINY[t.dtype]
    return ref, tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,n,h,hk,d,rot,axes", [
    (1, 1, 1, 1, 64, 64, 1), (8, 1, 32, 8, 128, 128, 1), (2, 77, 5, 5, 64, 64, 3), (1, 300, 20, 1, 128, 64, 1), (3, 50, 4, 2, 80, 40, 1),
    (2, 33, 3, 3, 40, 20, 2), (1, 17, 2, 1, 36, 18, 1), (1, 9, 1, 2, 7, 6, 1), (2, 5, 6, 6, 256, 256, 2), (1, 2000, 10, 10, 96, 96, 1),
    (1, 3, 2, 2, 600, 512, 1), (5, 4, 2, 0, 64, 64, 1)])
def test_rotary(rotary, dtype, interleaved, b, n, h, hk, d, rot, axes):
    g = _gen(b + n + d)
    q, k = (torch.randn(b, n, x, d, generator=g, device=DEV).to(dtype) for x in (h, hk))
    parts = [2 * (rot // 2 // axes + (1 if i < rot // 2 % axes else 0)) for i in range(axes)]
    r = rotary.RotaryPositions(d, rot, interleaved=interleaved, axes=parts, amplitude=1.25)
    positions = torch.randint(-5, 1 << 20, (b, n) if axes == 1 else (b, n, axes), generator=g, device=DEV)
    qr, kr = r(q, k, positions)
    for got, src in ((qr, q), (kr, k)):
        ref, tol = _turned(r, src, positions)
        assert got.shape == src.shape and got.is_contiguous()
        _within(got, ref, tol)
    # the same bits: 32-bit positions, q alone, in place, strided, and back within two roundings
    assert torch.equal(r(q, None, positions.int()), qr)
    stacked = torch.cat([q.flatten(2), k.flatten(2), q.flatten(2)], dim=-1)
    qs, ks = stacked[..., :h * d].view(b, n, h, d), stacked[..., h * d:(h + hk) * d].view(b, n, hk, d)
    out = r(qs, ks, positions)
    assert torch.equal(out[0], qr) and torch.equal(out[1], kr)
    same = r(qs, ks, positions, inplace=True)
    assert same[0] is qs and same[1] is ks and torch.equal(qs, qr) and torch.equal(ks, kr)
    assert torch.equal(stacked[..., (h + hk) * d:], q.flatten(2))                  # what lies behind is left alone
    ref, tol = _turned(r, q, positions, inverse=True)
    _within(r(q, None, positions, inverse=True), ref, tol)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(r(heads_first, None, positions), qr)


def test_rotary_positions_of_every_kind(rotary):
    r = rotary.RotaryPositions(64)
    q = torch.randn(2, 10, 4, 64, generator=_gen(1), device=DEV).half()
    count = torch.arange(10, device=DEV)
    want = r(q, None, count)
    assert torch.equal(r(q), want) and torch.equal(r(q, offset=7), r(q, None, count + 7))
    for p in (count[:, None], count.expand(2, 10), count.expand(2, 10)[..., None], (count * 3)[::1].int(), torch.stack([count, count], 1)[:, 0]):
        assert torch.equal(r(q, None, p), r(q, None, p.contiguous().long()))
    assert torch.equal(r(q[0], None, count), want[0]) and torch.equal(r(q[0]), want[0])
    flat, none = r(q[:, :0], q[:, :0]), r(q[:0])
    assert flat[0].shape == (2, 0, 4, 64) and none.shape == (0, 10, 4, 64)
    # far apart and exactly periodic in the 64-bit plan: a position and its wrap by 2^64 are one
    far = torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 40 + 3, -2 ** 40, 2 ** 62, -1, 5, 6], device=DEV)
    turns = [int.from_bytes(r._turns[8 * i:8 * i + 8], "little") for i in range(32)]
    angle = torch.tensor([[((int(p) * t) % 2 ** 64) / 2 ** 64 * 2 * math.pi for t in turns] for p in far.tolist()], dtype=torch.float64, device=DEV)
    u, v = q.double()[..., :32], q.double()[..., 32:]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    ref = torch.cat([u * c - v * s, v * c + u * s], -1)
    tol = torch.cat([u.abs() + v.abs()] * 2, -1) * 4e-7
    _within(r(q, None, far), ref, tol + HALF[torch.float16] * (ref.abs() + tol) + TINY[torch.float16])


def test_rotary_refusals_on_the_gpu(rotary):
    r, grid = rotary.RotaryPositions(64), rotary.RotaryPositions(64, axes=(32, 32))
    q = torch.randn(2, 6, 3, 64, device=DEV).half()
    n = torch.arange(6, device=DEV)
    bad = [(r, (q.float(),), {}), (r, (q, q.bfloat16()), {}), (r, (q, q[:1]), {}), (r, (q, q[:, :5]), {}), (r, (q[..., :32],), {}),
           (r, (q[..., ::1].transpose(2, 3),), {}), (r, (q, None, n.float()), {}), (r, (q, None, n[:5]), {}), (r, (q, None, n.cpu()), {}),
           (r, (q, None, n.expand(3, 6)), {}), (r, (q, None, n), {"offset": 2}), (grid, (q,), {}), (grid, (q, None, n), {}),
           (r, (q, q), {"inplace": True}), (r, (q[:1].expand(2, 6, 3, 64),), {"inplace": True}), (r, (q[:, :, :2], q[:, :, 1:]), {"inplace": True}),
           (r, (q.requires_grad_(),), {}), (r, (q.cpu(),), {})]
    for plan, args, kw in bad:
        with pytest.raises(RuntimeError):
            plan(*args, **kw)
    q = q.detach()
    assert r(q[:1].expand(2, 6, 3, 64)).shape == q.shape                        # out of place a broadcast input is fine
    k = torch.randn(2, 6, 1, 64, device=DEV).half()
    whole = torch.cat([q, k], 2)
    r(whole[:, :, :3], whole[:, :, 3:], n, inplace=True)                        # side by side in every token
    assert torch.equal(whole[:, :, 3:], r(k, None, n)) and torch.equal(whole[:, :, :3], r(q, None, n))
    first = whole.transpose(1, 2).contiguous()                                  # (batch, heads, tokens, 64): side by side in every sequence
    want = r(first.transpose(1, 2))
    r(first[:, :3].transpose(1, 2), first[:, 3:].transpose(1, 2), inplace=True)
    assert torch.equal(first.transpose(1, 2), want)


# ---- together ----------------------------------------------------------------------------------
class Block(nn.Module):
    """A pre-norm block as these operators make it up: int8 q / k / v with shared key heads, rotary positions turned in
    place, a 4-bit output projection and a 4-bit gated feed-forward."""

    def __init__(self, qu, rotary, dim, heads, kv_heads, dtype):
        super().__init__()
        d = dim // heads
        self.heads, self.kv_heads, self.d = heads, kv_heads, d
        def lin(k, n):
            return nn.Linear(k, n, bias=False, device=DEV, dtype=dtype)
        self.qkv = qu.Int8Linear.from_linear(lin(dim, (heads + 2 * kv_heads) * d))
        self.out = qu.Int4Linear.from_linear(lin(dim, dim))
        self.up = qu.Int4Linear.from_linear(lin(dim, 4 * dim), 32, symmetric=False).interleave_geglu_rows()
        self.down = qu.Int4Linear.from_linear(lin(2 * dim, dim), 128)
        self.norm1 = qu.Int8RMSNorm(nn.RMSNorm(dim, eps=1e-6, device=DEV, dtype=dtype))
        self.norm2 = qu.AddRMSNorm(nn.RMSNorm(dim, eps=1e-6, device=DEV, dtype=dtype))
        self.rotary = rotary.RotaryPositions(d)

    def attend(self, y, offset):
        b, n = y.shape[:2]
        h, hk, d = self.heads, self.kv_heads, self.d
        qkv = self.qkv(y).view(b, n, h + 2 * hk, d)
        q, k, v = qkv.split([h, hk, hk], dim=2)
        self.rotary(q, k, offset=offset, inplace=True)
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        o = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return o.transpose(1, 2).reshape(b, n, h * d)

    @torch.no_grad()
    def forward(self, x, h, offset=0):
        x, y = self.norm1(x, h)
        x, y = self.norm2(x, self.out(self.attend(y, offset)))
        return x, self.down(self.up(y))


def _block_reference(blk, x, h, offset):
    """The same in 64 bits on the stored weights, from the int8 codes that the first norm gave."""
    x, codes = blk.norm1(x, h)
    y = codes.q.double() * codes.scale.double()[:, None]
    w = blk.qkv.weight_int8_nk.double() * blk.qkv.weight_scale.double()[:, None]
    b, n, c = x.shape
    hh, hk, d = blk.heads, blk.kv_heads, blk.d
    q, k, v = (y @ w.t()).view(b, n, hh + 2 * hk, d).split([hh, hk, hk], dim=2)
    a = (offset + torch.arange(n, device=DEV).double())[:, None] * torch.tensor(blk.rotary.frequencies, dtype=torch.float64, device=DEV)
    cs, sn = a.cos()[:, None], a.sin()[:, None]
    turn = lambda t: torch.cat([t[..., :d // 2] * cs - t[..., d // 2:] * sn, t[..., d // 2:] * cs + t[..., :d // 2] * sn], -1)
    q, k, v = (t.transpose(1, 2) for t in (turn(q), turn(k), v))
    k, v = (t.repeat_interleave(hh // hk, dim=1) for t in (k, v))
    s = (q @ k.transpose(-1, -2) / math.sqrt(d)).masked_fill(torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1), -math.inf)
    o = (s.softmax(-1) @ v).transpose(1, 2).reshape(b, n, c)
    x = x.double() + o @ blk.out.dequantize_weight().double().t()
    f = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    up = f @ blk.up.dequantize_weight().double().t()
    up = up.unflatten(-1, (-1, 2, 16))
    act = (up[..., 0, :] * up[..., 1, :] * torch.special.ndtr(up[..., 1, :])).flatten(-2)
    return x, act @ blk.down.dequantize_weight().double().t()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,n,offset", [(1, 1, 70000), (2, 33, 0), (1, 300, 5)])
def test_a_block_of_them_together(qu, rotary, dtype, b, n, offset):
    torch.manual_seed(n)
    blk = Block(qu, rotary, 640, 10, 2, dtype)
    x, h = (torch.randn(b, n, 640, device=DEV).to(dtype) for _ in range(2))
    total, y = blk(x, h, offset)
    want_total, want = _block_reference(blk, x, h, offset)
    # 16-bit roundings of the stages in between: projection, attention's probabilities and output, residual, norm, gate and
    # down projection.  Eight of half a step each, at most 1.5 times larger through the gate: 12 half steps of the 2-norm.
    for got, ref in ((total, want_total), (y, want)):
        assert float((got.double() - ref).norm() / ref.norm()) < 12 * HALF[dtype]
    # captured, on a stream of its own, and replayed on other inputs: the eager call's bits
    xs, hs = x.clone(), h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        blk(xs, hs, offset)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = blk(xs, hs, offset)
    for seed in (1, 2):
        torch.manual_seed(seed)
        xs.normal_()
        hs.normal_()
        graph.replay()
        eager = blk(xs, hs, offset)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_two_streams_at_once_do_not_share_anything(qu, rotary):
    layer, w, b = _int4(qu, 1280, 1280, 64, True, True, torch.bfloat16, 3)
    r = rotary.RotaryPositions(64)
    xs = [torch.randn(m, 1280, device=DEV).bfloat16() for m in (3, 20, 90, 200)]
    want = [layer(x) for x in xs]
    turned = [r(x.view(-1, 20, 64)) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((layer(xs[i]), r(xs[i].view(-1, 20, 64))))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) and torch.equal(z, turned[i]) for i in range(len(xs)) for y, z in got[i])


def test_unet_with_multiview_rotary_rmsnorms_and_four_bit_projections(qu, pkg):
    """The UNet's own paths into these operators: rotary positions in the multiview attention, RMSNorms that emit codes,
    time projections of 4 bits stacked into one layer."""
    un = importlib.import_module(PKG + ".unet")
    torch.manual_seed(0)
    net = un.UNetSD21MV(block_out_channels=(128, 128), layers_per_block=1, attention_heads=(2, 2), cross_attention_dim=128,
                        attn_levels=(True, False), num_views=2)
    for blk in [m for m in net.modules() if isinstance(m, un.TransformerBlock)]:
        blk.norm_mv, blk.norm2 = nn.RMSNorm(128, eps=1e-6), nn.RMSNorm(128, eps=1e-6)
    net = net.to(DEV).bfloat16().eval()
    x, ctx, t = torch.randn(2, 4, 8, 8, device=DEV).bfloat16(), torch.randn(2, 3, 128, device=DEV).bfloat16(), torch.full((2,), 10, device=DEV)
    grids = {2 * s * s: torch.cartesian_prod(torch.arange(2), torch.arange(s), torch.arange(s)).to(DEV) for s in (8, 4)}
    with torch.no_grad():
        plain = net(x, t, ctx)
        assert un.use_multiview_rotary(net, grids) == 4
        turned = net(x, t, ctx)
        assert float((turned.float() - plain.float()).norm()) > 0
        qu.quantize_model_int4(net, choose=lambda name, _: "time_emb" in name, verbose=False)
        qu.quantize_model_tensorcore(net, verbose=False)
        un.fuse_qkv_layers(net)
        assert un.fuse_time_projections(net) == 7 and type(net.time_proj_all) is qu.Int4Linear
        loose = net(x, t, ctx)
        assert un.fuse_layernorm_quant(net) == 16
        fused = net(x, t, ctx)
    # 4- and 8-bit weights against 16-bit ones: 4-bit rounding is off by a step of max / 7 over sqrt(12), about 0.11 of a
    # normal weight, in the time path only; the int8 path adds 1 %
    assert float((loose.float() - turned.float()).norm() / turned.float().norm()) < 0.15
    assert float((fused.float() - loose.float()).norm() / loose.float().norm()) < 0.03


def test_attention_leaves_the_projections_outputs_to_their_hooks(pkg):
    """A hook on a projection keeps what the projection returned; the rotation writes to tensors of its own."""
    un = importlib.import_module(PKG + ".unet")
    attn = un.TransformerBlock(128, 2, 128, 2).attn_mv.to(DEV).bfloat16()
    attn.rotary = importlib.import_module(PKG + ".rotary").RotaryPositions(64)
    kept = []
    attn.to_q.register_forward_hook(lambda m, a, y: kept.append(y))
    x = torch.randn(1, 12, 128, generator=_gen(4), device=DEV).bfloat16()
    with torch.no_grad():
        attn(x)
        assert torch.equal(kept[0], nn.functional.linear(x, attn.to_q.weight, attn.to_q.bias))
