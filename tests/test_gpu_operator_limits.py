"""GPU: the 4-bit layers, the RMSNorms and the rotary positions at their limits, against their definitions in 64 bits."""
import decimal
import importlib
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn as nn

from test_gpu_operators import DEV, HALF, TINY, _check_int4, _check_norm, _gen, _int4, _within
from test_operator_limits_host import _frequencies_of_many_digits, _pi

pytestmark = pytest.mark.gpu
PKG = "hunyuan3d-tools_b200"


@pytest.fixture(scope="module")
def rotary():
    return importlib.import_module(PKG + ".rotary")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,group,zeros", [(5, 256, 64, 64, True), (40, 256, 64, 64, False), (70, 1024, 272, 32, True),
                                               (300, 448, 144, 448, True), (300, 2048, 128, 128, False)])
def test_int4_infinite_activations_give_what_the_definition_gives(qu, dtype, m, k, n, group, zeros):
    """For few rows and for many: an infinity keeps the weight's sign, two that cancel and a weight of zero give NaN, and the
    other rows stay as they are."""
    g = _gen(m + k)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    zero = torch.randint(0, 16, (n, k // group), generator=g, device=DEV) if zeros else None
    scale = ((torch.rand(n, k // group, generator=g, device=DEV) - 0.5) * 0.02).to(dtype)      # of both signs
    layer = qu.Int4Linear.from_codes(codes, scale, zero)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    x[0, 3], x[1, k - 1], x[2, 5], x[2, k // 2], x[3, 0], x[m - 1, 77] = math.inf, -math.inf, math.inf, math.inf, math.nan, math.inf
    y, ref = layer(x), x.double() @ layer.dequantize_weight().double().t()
    bad = ~ref.isfinite()
    assert torch.equal(~y.isfinite(), bad) and bool(ref[0].isinf().any()) and bool(ref[0].isnan().any())
    assert torch.equal(y[bad].isnan(), ref[bad].isnan())
    assert torch.equal(y[bad & ~ref.isnan()].double(), ref[bad & ~ref.isnan()])


def test_rotary_in_place_wherever_queries_and_keys_share_no_element(rotary):
    """Side by side in every token of a sequence-first tensor, in every head of an interleaved one, and in strided slices of
    those; refused where a single element is shared."""
    r, b, n, h, d = rotary.RotaryPositions(64), 3, 7, 4, 64
    g = _gen(21)

    def check(whole, q, k):
        other = torch.ones_like(whole, dtype=torch.bool)
        for t in (q, k):
            other.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(False)
        rest = whole[other].clone()
        want = r(q, k)
        got = r(q, k, inplace=True)
        assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(whole[other], rest)

    whole = torch.randn(n, b, 3 * h * d, generator=g, device=DEV).half()              # sequence first
    q, k, _ = (t.view(n, b, h, d).transpose(0, 1) for t in whole.split(h * d, dim=-1))
    check(whole, q, k)
    whole = torch.randn(n, b, (h + 2) * d, generator=g, device=DEV).half()            # the same with one key head
    check(whole, whole[..., :h * d].view(n, b, h, d).transpose(0, 1), whole[..., h * d:(h + 1) * d].view(n, b, 1, d).transpose(0, 1))
    whole = torch.randn(b, n, h, 3, d, generator=g, device=DEV).half()                # q, k and v of each head together
    check(whole, whole[..., 0, :], whole[..., 1, :])
    check(whole, whole[:, ::2, :, 2], whole[:, ::2, :, 0])
    check(whole[0], whole[0, ..., 1, :], whole[0, ..., 0, :])
    whole = torch.randn(n, b, h, 3, d, generator=g, device=DEV).half()                # and sequence first
    check(whole, whole[..., 0, :].transpose(0, 1), whole[..., 2, :].transpose(0, 1))
    whole = torch.randn(b, n, 2 * h, d, generator=g, device=DEV).half()               # heads in turn
    check(whole, whole[:, :, 0::2], whole[:, :, 1::2])
    whole = torch.randn(b, 2 * n, h, d, generator=g, device=DEV).half()               # tokens in turn
    check(whole, whole[:, 0::2], whole[:, 1::2])

    flat = torch.randn(b * n * h * d * 4, generator=g, device=DEV).half()
    size = (b, n, h, d)
    q = flat.as_strided(size, (n * h * 2 * d, h * 2 * d, 2 * d, 1), 0)
    for at in (d - 1, d + 1, 2 * d * h + d // 2, 2 * d):          # the last element; the next head's; inside a token; a head further
        k = flat.as_strided(size, q.stride(), at)
        with pytest.raises(RuntimeError, match="share memory"):
            r(q, k, inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):       # other steps: nothing is known of where they meet
        r(q, flat.as_strided(size, (n * h * 3 * d, h * 3 * d, 3 * d, 1), d), inplace=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base,scaling", [(10000.0, None), (500000.0, {"kind": "ntk", "factor": 4.0}),
                                          (10000.0, {"kind": "by_parts", "factor": 8.0, "original_length": 8192})])
def test_rotary_far_positions_against_angles_of_many_digits(rotary, interleaved, base, scaling):
    """The angles from the formula in 60 digits, not from the plan's own fractions.  Those are within 2^-65 of a turn, so an
    angle is off by position 2^-65 2 pi, on top of the 4e-7 of its evaluation in 32 bits."""
    r = rotary.RotaryPositions(64, base=base, scaling=scaling, interleaved=interleaved)
    far = [0, 1, 131071, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 36 + 1, 2 ** 40 + 3, -2 ** 40, -1, 999999]
    angle, pi = [], _pi()
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        for p in far:
            for w in _frequencies_of_many_digits(64, base, scaling):
                angle.append(float(p * w % (2 * pi)))
    angle = torch.tensor(angle, dtype=torch.float64, device=DEV).view(len(far), 1, 32)
    q = torch.randn(len(far), 4, 64, generator=_gen(31), device=DEV).half()
    got = r(q, None, torch.tensor(far, device=DEV))
    t = q.double()
    u, v = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :32], t[..., 32:])
    c, s = angle.cos(), angle.sin()
    y, z = u * c - v * s, v * c + u * s
    off = 4e-7 + torch.tensor([abs(p) * 2.0 ** -65 * 2 * math.pi for p in far], dtype=torch.float64, device=DEV)[:, None, None]
    tol = (u.abs() + v.abs()) * off
    join = (lambda a, b: torch.stack([a, b], -1).flatten(-2)) if interleaved else (lambda a, b: torch.cat([a, b], -1))
    ref, tol = join(y, z), join(tol, tol)
    _within(got, ref, tol + HALF[torch.float16] * (ref.abs() + tol) + TINY[torch.float16])


@pytest.mark.parametrize("m,k,n,group,scales", [(8 * 65535 + 9, 64, 32, 32, torch.float16), (2 * 65535 + 1, 32768, 16, 1024, torch.float16),
                                                (256 * 65535 + 300, 64, 16, 64, torch.bfloat16)])
def test_int4_more_rows_than_a_grid_has_blocks(qu, m, k, n, group, scales):
    """Scales of the activations' type and of the other: every row gets its answer, also behind the last block of a grid."""
    g = _gen(k)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    scale = (torch.rand(n, k // group, generator=g, device=DEV) * 0.02 + 0.001).to(scales)
    layer = qu.Int4Linear.from_codes(codes, scale)
    w = layer.dequantize_weight().double()
    x = torch.empty(m, k, device=DEV, dtype=torch.bfloat16)
    some = torch.randn(4096, k, generator=g, device=DEV).bfloat16()
    at = [0, m // 2 - 2048, m - 4096]
    x.zero_()
    for i in at:
        x[i:i + 4096] = some
    y = layer(x)
    assert y.shape == (m, n)
    for i in at:
        _check_int4(layer, w, None, some, y[i:i + 4096])
    assert not bool(y[4096:at[1]].any()) and not bool(y[at[1] + 4096:at[2]].any())


def test_norm_of_another_width_is_refused_with_any_weight(qu):
    """Also once the native path is loaded, where the weight does not tell the width (there is none, or it was replaced)."""
    x, wide = torch.randn(4, 64, device=DEV).half(), torch.randn(4, 128, device=DEV).half()
    for cls in (qu.AddRMSNorm, qu.Int8RMSNorm):
        for norm in (cls(nn.RMSNorm(64, eps=1e-6, elementwise_affine=False)), cls(nn.RMSNorm(64, eps=1e-6, device=DEV))):
            norm(x)                                     # loads the native path
            for weight in (None, nn.Parameter(torch.ones(128, device=DEV), requires_grad=False)):
                norm.weight = weight
                with pytest.raises(RuntimeError, match="64 dimensions"):
                    norm(wide)
                with pytest.raises(RuntimeError, match="64 dimensions"):
                    norm(wide, wide)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [False, True])
def test_norms_with_the_default_eps_or_without_weight_take_the_direct_way(qu, ik, monkeypatch, dtype, affine):
    x = torch.randn(6, 320, generator=_gen(5), device=DEV).to(dtype) * 2.0 ** -6      # small, so that eps counts
    norm = nn.RMSNorm(320, elementwise_affine=affine).to(DEV, dtype)
    half, codes = qu.AddRMSNorm(norm), qu.Int8RMSNorm(norm)
    want, want_q = half.forward(x), codes.forward(x)      # the binding's answer
    _check_norm(x, None, norm.weight, torch.finfo(dtype).eps, None, want)

    def refuse(*a, **k):
        raise AssertionError("the Python binding was called")
    monkeypatch.setattr(type(ik), "rmsnorm", refuse)
    assert torch.equal(half(x), want)
    total, y = half(x, x)
    assert torch.equal(total, x + x)
    got = codes(x)
    assert torch.equal(got.q, want_q.q) and torch.equal(got.scale, want_q.scale)


def test_tangents_and_traced_calls_are_refused(qu, rotary):
    """A forward-mode tangent would be dropped, and a trace would hold the answer as a constant."""
    layer, _, _ = _int4(qu, 64, 128, 64, False, True, torch.float16, 7)
    norm = nn.RMSNorm(128, eps=1e-6, device=DEV, dtype=torch.float16).requires_grad_(False)
    half, codes, r = qu.AddRMSNorm(norm), qu.Int8RMSNorm(norm), rotary.RotaryPositions(64)
    x, q = torch.randn(4, 128, device=DEV).half(), torch.randn(4, 2, 64, device=DEV).half()
    calls = [(layer, (x,)), (half, (x,)), (half, (x, x)), (codes, (x,)), (r, (q,)), (r, (q, q))]
    for f, args in calls:
        f(*args)
    with fwAD.dual_level():
        for f, args in calls:
            for i in range(len(args)):
                dual = [fwAD.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="gradient"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="gradient"):      # no_grad leaves tangents on
                    f(*dual)
            f(*args)
    outer = lambda f: (lambda *a: f(*a).q if f is codes else f(*a))
    for f, args in calls:
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(outer(f), args, check_trace=False)
        f(*args)
