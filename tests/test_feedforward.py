"""The gated product, its gradients and the gradients of the rc product: refusals on the CPU, results on the GPU against the
formulas in 64 bits.

Tolerances, element by element, from the arithmetic alone (u = half a step of the output type, torch.finfo(t).eps / 2):
  * a product accumulated in fp32 over K adds one partial sum per 16 elements of K; every addition is off by at most a step
    2^-23 of a sum no larger than S = sum |a||b|, so it is off by at most (K / 16 + 4) 2^-23 S;
  * act is at most 1.13-Lipschitz and act' at most 1.13 large; their evaluation in fp32 is off by at most 2^-16 relative (the
    fast exponential by 2 + 1.16 |x| steps of 2^-23, 104 for |x| = 88; erfc(g / sqrt 2) by g^2 steps of 2^-23.4 through its
    argument, 81 for |g| = 9);
  * one rounding of the output: u |value|, or half the spacing of the subnormals of fp16, 2^-25;
  * the backward pass rounds dg and du once to the operands' type before their products.
"""
import ctypes
import math

import pytest
import torch

ACTS = ("silu", "gelu", "gelu_tanh", "relu")
TYPES = (torch.float16, torch.bfloat16)


def act64(name, g):
    """act(g) and act'(g) by their definitions, in 64 bits."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        # (1 + tanh z) / 2 as 1 / (1 + exp(-2 z)): the sum cancels for z < -18, where 64 bits hold the quotient well
        p = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))
        return g * p, p + 2 * g * p * (1 - p) * c * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).double()


def half_step(t):
    return torch.finfo(t).eps / 2


def floor_of(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def summing(a, b):
    """What an fp32 accumulation of a @ b.T (both 64 bits) may be off by."""
    return (a.shape[1] / 16 + 4) * 2.0 ** -23 * (a.abs() @ b.abs().t())


def check(got, want, tol):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%d of %d off, worst %g allowed %g" % (bad.sum(), bad.numel(), off[bad].max(),
                                                                  tol[bad][off[bad].argmax()])


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def gated_inputs(m, f, k, dtype, seed=1):
    return (normal((m, k), dtype, seed), normal((f, k), dtype, seed + 1, k ** -0.5),
            normal((f, k), dtype, seed + 2, k ** -0.5))


def check_gated(a, bg, bu, act, c, gate=None, up=None):
    t = a.dtype
    x, wg, wu = a.double(), bg.double(), bu.double()
    g, u = x @ wg.t(), x @ wu.t()
    dg, du = summing(x, wg), summing(x, wu)
    v, _ = act64(act, g)
    want = v * u
    tol = (half_step(t) + 2.0 ** -16) * want.abs() + 1.13 * dg * u.abs() + v.abs() * du + 1.13 * dg * du + floor_of(t)
    check(c, want, tol)
    if gate is not None:
        check(gate, g, half_step(t) * g.abs() + 2 * dg + floor_of(t))
        check(up, u, half_step(t) * u.abs() + 2 * du + floor_of(t))


def check_gated_backward(dc, a, bg, bu, gate, up, act, da, dbg, dbu):
    t = a.dtype
    u16 = half_step(t)
    d, g, u = dc.double(), gate.double(), up.double()
    v, slope = act64(act, g)
    dg, du = d * u * slope, d * v
    # act'(g) may itself be near 0 where its terms are not: its evaluation is off relative to their size, at most 1.2
    e_g = u16 * dg.abs() + 2.0 ** -16 * 1.2 * (d * u).abs() + floor_of(t)
    e_u = u16 * du.abs() + 2.0 ** -16 * du.abs() + floor_of(t)
    x, wg, wu = a.double(), bg.double(), bu.double()
    f, m = bg.shape[0], a.shape[0]

    def tol(want, off, size, length):
        return u16 * want.abs() + (1 + u16) * off + (length / 16 + 8) * 2.0 ** -23 * size * 1.01 + floor_of(t)

    if da is not None:
        want = dg @ wg + du @ wu
        check(da, want, tol(want, e_g @ wg.abs() + e_u @ wu.abs(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * f))
    for got, dy, e in ((dbg, dg, e_g), (dbu, du, e_u)):
        if got is not None:
            want = dy.t() @ x
            check(got, want, tol(want, e.t() @ x.abs(), dy.abs().t() @ x.abs(), m))


@pytest.fixture(scope="module")
def beam(built_library):
    import beam as beam_pkg
    return beam_pkg


@pytest.fixture
def healthy(beam):
    yield
    assert beam.device_status() == (0, 0)


# ---------------------------------------------------------------------------------------------------- refusals, CPU
def _host(nbytes):
    raw = ctypes.create_string_buffer(nbytes + 64)
    return raw, (ctypes.addressof(raw) + 63) & ~63


def test_c_entries_refuse_bad_arguments(built_library):
    if torch.cuda.is_available():
        pytest.skip("host memory stands in for device pointers")
    L = ctypes.CDLL(built_library)
    vp, i, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    keep, base = _host(1 << 20)
    p = [base + (j << 16) for j in range(12)]  # ten tensors of 64 x 64 that do not overlap
    f = L.beam_gated_gemmrc
    f.argtypes = [vp, vp, vp, vp, vp, vp, i, i, i, i, i, vp]
    good = [p[0], p[1], p[2], p[3], p[4], p[5], 64, 64, 64, 0, 0, None]

    def call(fn, args, **change):
        args = list(args)
        for k, v in change.items():
            args[int(k[1:])] = v
        return fn(*args)

    assert call(f, good) == 8                                  # well formed: no device here
    assert call(f, good, _4=None, _5=None) == 8
    for j in range(4):
        assert call(f, good, **{"_%d" % j: None}) == 1
        assert call(f, good, **{"_%d" % j: p[j] + 2}) == 3     # misaligned
    assert call(f, good, _4=None) == 1                         # gate without up
    assert call(f, good, _6=0) == 1 and call(f, good, _7=-8) == 1 and call(f, good, _8=0) == 1
    assert call(f, good, _7=60) == 3 and call(f, good, _8=60) == 3
    assert call(f, good, _9=4) == 1 and call(f, good, _9=-1) == 1
    assert call(f, good, _10=1) == 1                           # only the bf16 flag
    assert call(f, good, _10=2) == 8
    assert call(f, good, _3=p[0] + 4096) == 1                  # c inside a
    assert call(f, good, _4=p[3]) == 1                         # gate on c
    assert call(f, good, _5=p[4] + 16) == 1                    # up inside gate

    need = L.beam_gated_gemmrc_backward_workspace_bytes
    need.restype, need.argtypes = sz, [i, i, i]
    assert need(64, 64, 64) == 2 * 64 * 64 * 2 and need(3, 8, 64) == 2 * 256 and need(0, 8, 8) == 0
    # 74 pairs without a device: dA of 16 rows is 4 tiles of 512 k-blocks, in the most slices that there are
    assert need(16, 16384, 1024) == 2 * 16 * 16384 * 2 + 16 * 16 * 1024 * 4
    # 8 tiles of 86 k-blocks in 7 slices and 88 tiles of 6 are 144 items, two rounds of 74 pairs
    assert need(333, 2744, 1000) == 2 * (-(-333 * 2744 * 2 // 256) * 256) + -(-7 * 333 * 1000 * 4 // 256) * 256
    f = L.beam_gated_gemmrc_backward
    f.argtypes = [vp] * 9 + [i, i, i, i, i, vp, sz, vp]
    good = p[:9] + [64, 64, 64, 1, 2, p[9], need(64, 64, 64), None]
    assert call(f, good) == 8
    assert call(f, good, _6=None, _2=None, _3=None) == 8       # no da: the weights are not needed
    assert call(f, good, _7=None, _8=None, _1=None) == 8       # no weight gradients: nor is a
    assert call(f, good, _6=None, _7=None, _8=None) == 1
    assert call(f, good, _2=None) == 1 and call(f, good, _1=None) == 1 and call(f, good, _4=None) == 1
    assert call(f, good, _14=None) == 4 and call(f, good, _15=100) == 4
    assert call(f, good, _10=4) == 3 and call(f, good, _11=12) == 3
    assert call(f, good, _6=p[1]) == 1 and call(f, good, _7=p[8]) == 1 and call(f, good, _14=p[4]) == 1
    assert call(f, good, _8=p[8] + 8) == 3

    need = L.beam_gemmrc_backward_workspace_bytes
    need.restype, need.argtypes = sz, [i, i, i]
    assert need(64, 64, 64) == 0 and need(8192, 4096, 8192) == 0 and need(64, 60, 64) == 0
    # dA is one tile of 64 k-blocks, in slices of 4; dB 16 tiles of one k-block
    assert need(64, 4096, 256) == 16 * 64 * 256 * 4
    f = L.beam_gemmrc_backward
    f.argtypes = [vp] * 5 + [i, i, i, i, vp, sz, vp]
    good = p[:5] + [64, 64, 64, 0, None, 0, None]
    assert call(f, good) == 8
    assert call(f, good, _3=None, _2=None) == 8 and call(f, good, _4=None, _1=None) == 8
    assert call(f, good, _3=None, _4=None) == 1 and call(f, good, _0=None) == 1
    assert call(f, good, _1=None) == 1 and call(f, good, _2=None) == 1
    assert call(f, good, _6=12) == 3 and call(f, good, _5=0) == 1 and call(f, good, _8=16) == 1
    assert call(f, good, _3=p[4]) == 1 and call(f, good, _4=p[0]) == 1
    assert call(f, good, _9=p[3], _10=64) == 1 and call(f, good, _9=p[9] + 4, _10=64) == 3


def test_python_refuses_cpu_tensors_and_bad_names(beam):
    a, w, c = torch.zeros(4, 16).half(), torch.zeros(8, 16).half(), torch.zeros(4, 8).half()
    with pytest.raises(ValueError, match="activation"):
        beam.gated_gemmrc(a, w, w, c, activation="tanh")
    with pytest.raises(ValueError, match="CUDA"):
        beam.gated_gemmrc(a, w, w, c)
    with pytest.raises(TypeError):
        beam.gated_gemmrc(a.float(), w, w, c)
    with pytest.raises(ValueError, match="CUDA"):
        beam.gated_gemmrc_backward(c, a, w, w, c, c, da=a)
    with pytest.raises(ValueError, match="CUDA"):
        beam.gemmrc_backward(c, a, w, da=a)


@pytest.mark.parametrize("act", ACTS)
def test_slopes_against_differences(act):
    """The slopes used as the reference below are those of the activations, by central differences."""
    g = torch.linspace(-9, 9, 2001, dtype=torch.float64) + 1e-3
    h = 1e-5
    v, slope = act64(act, g)
    diff = (act64(act, g + h)[0] - act64(act, g - h)[0]) / (2 * h)
    assert torch.allclose(slope, diff, atol=1e-8)  # h^2 / 6 x |act'''| < 1e-10, rounding 2^-53 x 9 / h = 1e-10


# ------------------------------------------------------------------------------------------------------- forward, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,f,k", [(1, 8, 8), (1, 1504, 264), (2, 8, 1000), (7, 24, 72), (8, 2368, 64), (17, 1192, 200),
                                   (64, 128, 512), (77, 5464, 136), (127, 3000, 8), (128, 1184, 64),
                                   (1, 1000, 3080), (33, 1192, 4104), (128, 2360, 2056), (100, 8, 8200)])
def test_gated_few_rows(beam, healthy, dtype, m, f, k):
    """Up to 128 rows: widths from 8 to 40 columns per tile, ragged in every direction; nothing written past c."""
    a, bg, bu = gated_inputs(m, f, k, dtype, m + f)
    guard = torch.full((m + 2, f), 3.0, dtype=dtype, device="cuda")
    beam.gated_gemmrc(a, bg, bu, guard[1:m + 1], activation=ACTS[(m + f) % 4])
    check_gated(a, bg, bu, ACTS[(m + f) % 4], guard[1:m + 1])
    assert (guard[0] == 3).all() and (guard[-1] == 3).all()


@pytest.mark.gpu
def test_gated_few_rows_several_waves(beam, healthy):
    """More columns than one wave of 128-wide tiles holds: every CTA works on two tiles, one in each accumulator."""
    a, bg, bu = gated_inputs(5, 40000, 128, torch.bfloat16, 3)
    c = torch.empty(5, 40000, dtype=a.dtype, device="cuda")
    gate, up = torch.empty_like(c), torch.empty_like(c)
    beam.gated_gemmrc(a, bg, bu, c, gate=gate, up=up)
    check_gated(a, bg, bu, "silu", c, gate, up)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,f,k", [(129, 8, 8), (256, 128, 64), (300, 1000, 456), (513, 264, 1096), (1024, 4096, 512)])
def test_gated_tiles(beam, healthy, dtype, act, m, f, k):
    a, bg, bu = gated_inputs(m, f, k, dtype, m + f)
    out = torch.full((3, m + 2, f), 3.0, dtype=dtype, device="cuda")
    c, gate, up = (out[j, 1:m + 1] for j in range(3))
    beam.gated_gemmrc(a, bg, bu, c, activation=act, gate=gate, up=up)
    check_gated(a, bg, bu, act, c, gate, up)
    assert (out[:, 0] == 3).all() and (out[:, -1] == 3).all()
    alone = torch.empty_like(c)
    beam.gated_gemmrc(a, bg, bu, alone, activation=act)
    assert torch.equal(alone, c)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_activation_far_out(beam, healthy, act):
    """Gates from the smallest to the largest magnitudes of bf16, with no NaN where the definition has none: a is a row of ones
    in one place, so g and u are single weights."""
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 9.0, -9.0, 40.0, -40.0, 88.5, -88.5, 200.0, -200.0, 1e4, -1e4,
                      1e20, -1e20, 3e38, -3e38, 0.5, -0.5, 2.0, -2.0], device="cuda").bfloat16()
    f = g.numel()
    for m in (1, 200):
        a = torch.zeros(m, 16, device="cuda").bfloat16()
        a[:, 3] = 1
        bg, bu = torch.zeros(2, f, 16, device="cuda").bfloat16()
        bg[:, 3], bu[:, 3] = g, 1
        c = torch.empty(m, f, dtype=torch.bfloat16, device="cuda")
        gate, up = torch.empty_like(c), torch.empty_like(c)
        beam.gated_gemmrc(a, bg, bu, c, activation=act, gate=gate, up=up)
        assert torch.equal(gate, g.expand(m, f)) and (up == 1).all()
        v, slope = act64(act, g.double())
        check(c, v.expand(m, f), ((2.0 ** -8 + 2.0 ** -16) * v.abs() + 2.0 ** -126).expand(m, f))
        one = torch.ones_like(c)
        dbg = torch.empty_like(bg)
        beam.gated_gemmrc_backward(one, a, bg, bu, gate, up, db_gate=dbg, activation=act)
        want = m * slope  # m equal summands, each rounded once to bf16 and added exactly up to one more rounding
        check(dbg[:, 3], want, 2.0 ** -7 * want.abs() + m * 2.0 ** -16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", (3, 200))
def test_gradients_of_gates_past_the_range(beam, healthy, dtype, act, m):
    """A gate's product far below what the type holds is kept as -infinity: act and its slope are 0 there, forward and backward, and
    no gradient becomes NaN.  Above the range the slope is 1."""
    f, k = 72, 136
    a, bg, bu = gated_inputs(m, f, k, dtype, 17)
    big = 1024.0 if dtype == torch.float16 else 2.0 ** 65
    a[1, 3], bg[:, 3] = big, 0.0
    bg[7, 3], bg[8, 3] = -big, big  # gates of row 1 near -big^2 and big^2
    bu[:, 3] = 0.0
    c, gate, up = (torch.empty(m, f, dtype=dtype, device="cuda") for _ in range(3))
    beam.gated_gemmrc(a, bg, bu, c, activation=act, gate=gate, up=up)
    assert torch.isneginf(gate[1, 7]) and torch.isposinf(gate[1, 8]) and gate.isinf().sum() == 2
    assert c[1, 7] == 0 and torch.isinf(c[1, 8])
    dc = normal((m, f), dtype, 18)
    dbg, dbu, da = torch.empty_like(bg), torch.empty_like(bu), torch.empty_like(a)
    # value and slope have their limits at -60000 and 60000 already, but for the value above
    at = torch.where(gate.isinf(), gate.clamp(min=-60000, max=60000), gate)
    v, slope = act64(act, at.double())
    assert v[1, 7] == 0 and slope[1, 7] == 0 and slope[1, 8] == 1
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, db_gate=dbg, activation=act)
    check_gated_backward(dc, a, bg, bu, at, up, act, None, dbg, None)
    dc[1, 8] = 0  # the value is infinite there, and so would be its gradients
    gate[1, 8] = 1.0
    at[1, 8] = 1.0
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, da=da, db_gate=dbg, db_up=dbu, activation=act)
    check_gated_backward(dc, a, bg, bu, at, up, act, da, dbg, dbu)
    assert all(t.isfinite().all() for t in (da, dbg, dbu))


@pytest.mark.gpu
def test_gated_passes_nan_and_infinity_on(beam, healthy):
    """A NaN in one row of a reaches that row of c and no other; an infinite product stays infinite."""
    for m in (3, 200):
        a, bg, bu = gated_inputs(m, 64, 64, torch.float16, 8)
        a[1, 5] = float("nan")
        a[2] = 60000.0
        bu.fill_(1.0)
        bg.fill_(1.0)
        c = torch.empty(m, 64, dtype=torch.float16, device="cuda")
        beam.gated_gemmrc(a, bg, bu, c, activation="silu")
        assert c[1].isnan().all() and torch.isposinf(c[2]).all()
        assert c[0].isfinite().all() and (m == 3 or c[3:].isfinite().all())


# ------------------------------------------------------------------------------------------------------ backward, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,f,k", [(1, 8, 8), (3, 72, 264), (64, 64, 64), (130, 520, 200), (257, 264, 1032),
                                   (1000, 776, 328), (17, 4104, 136), (300, 2744, 264), (2500, 64, 264)])
def test_gated_backward(beam, healthy, dtype, act, m, f, k):
    a, bg, bu = gated_inputs(m, f, k, dtype, m + f)
    gate, up, dc = normal((m, f), dtype, 5, 2.0), normal((m, f), dtype, 6), normal((m, f), dtype, 7)
    room = [torch.full((r + 2, k), 3.0, dtype=dtype, device="cuda") for r in (m, f, f)]
    da, dbg, dbu = (x[1:-1] for x in room)
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, da=da, db_gate=dbg, db_up=dbu, activation=act)
    check_gated_backward(dc, a, bg, bu, gate, up, act, da, dbg, dbu)
    for x in room:
        assert (x[0] == 3).all() and (x[-1] == 3).all()


@pytest.mark.gpu
def test_gated_backward_of_each_gradient_alone(beam, healthy):
    m, f, k = 200, 136, 264
    a, bg, bu = gated_inputs(m, f, k, torch.bfloat16, 4)
    gate, up, dc = (normal((m, f), torch.bfloat16, 5 + j) for j in range(3))
    full = {"da": torch.empty_like(a), "db_gate": torch.empty_like(bg), "db_up": torch.empty_like(bu)}
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, **full)
    for names in (("da",), ("db_gate",), ("db_up",), ("da", "db_up"), ("db_gate", "db_up")):
        part = {n: torch.empty_like(full[n]) for n in names}
        beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, **part)
        for n in names:
            assert torch.equal(part[n], full[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (5, 64, 72), (127, 136, 200), (256, 256, 256), (300, 1000, 1096),
                                   (1000, 264, 520), (2000, 48, 24), (40, 4104, 264), (3000, 264, 136)])
def test_gemmrc_backward(beam, healthy, dtype, m, n, k):
    dc, a, b = normal((m, n), dtype, 1), normal((m, k), dtype, 2), normal((n, k), dtype, 3)
    room = [torch.full((r + 2, k), 3.0, dtype=dtype, device="cuda") for r in (m, n)]
    da, db = (x[1:-1] for x in room)
    beam.gemmrc_backward(dc, a, b, da=da, db=db)
    for got, left, right in ((da, dc.double(), b.double().t()), (db, dc.double().t(), a.double().t())):
        want = left @ right.t()
        check(got, want, half_step(dtype) * want.abs() + 1.01 * summing(left, right) + floor_of(dtype))
    for x in room:
        assert (x[0] == 3).all() and (x[-1] == 3).all()
    one = torch.empty_like(a)
    beam.gemmrc_backward(dc, a, b, da=one)
    assert torch.equal(one, da)
    one = torch.empty_like(b)
    beam.gemmrc_backward(dc, a, b, db=one)
    assert torch.equal(one, db)


@pytest.mark.gpu
def test_gradient_against_differences(beam, healthy):
    """<gradient, direction> against the central difference of the loss sum(c * w) in 64 bits along that direction."""
    m, f, k = 48, 88, 104
    a, bg, bu = gated_inputs(m, f, k, torch.float16, 9)
    w = normal((m, f), torch.float16, 12)
    c = torch.empty(m, f, dtype=torch.float16, device="cuda")
    gate, up = torch.empty_like(c), torch.empty_like(c)
    for act in ("silu", "gelu", "gelu_tanh"):
        beam.gated_gemmrc(a, bg, bu, c, activation=act, gate=gate, up=up)
        grads = [torch.empty_like(t) for t in (a, bg, bu)]
        beam.gated_gemmrc_backward(w, a, bg, bu, gate, up, *grads, activation=act)

        def loss(x, y, z):
            return (act64(act, x @ y.t())[0] * (x @ z.t()) * w.double()).sum()

        at = [t.double() for t in (a, bg, bu)]
        for i in range(3):
            v = torch.randn(at[i].shape, dtype=torch.float64, device="cuda",
                            generator=torch.Generator(device="cuda").manual_seed(i))
            h = 1e-6
            hi, lo = list(at), list(at)
            hi[i], lo[i] = at[i] + h * v, at[i] - h * v
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            got = (grads[i].double() * v).sum()
            # gate, up, dg and du and the gradients are each rounded to fp16: independent relative errors of at most 2^-11 per
            # element in a sum of N terms stay below 6 x 2^-11 of the root of the sum of squares
            size = (grads[i].double() * v).square().sum().sqrt()
            assert abs(got - diff) <= 6 * 2.0 ** -11 * 6 * size, (act, i, got.item(), diff.item())


# -------------------------------------------------------------------------------------------------- a block, as it is used
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 96, 520])
def test_a_feed_forward_block_and_its_gradients(beam, healthy, rows):
    """y = (silu(x Wg^T) * (x Wu^T)) Wd^T and all its gradients by the library's calls, on a stream of their own, eagerly and as a
    graph that is replayed on other inputs, against 64-bit automatic differentiation."""
    d, f, t = 256, 712, torch.bfloat16
    x, wg, wu = gated_inputs(rows, f, d, t, 21)
    wd, dy = normal((d, f), t, 24, f ** -0.5), normal((rows, d), t, 25)
    h, gate, up, dh = (torch.empty(rows, f, dtype=t, device="cuda") for _ in range(4))
    y, dx, dwg, dwu, dwd = (torch.empty_like(v) for v in (dy, x, wg, wu, wd))

    def step():
        beam.gated_gemmrc(x, wg, wu, h, gate=gate, up=up)
        beam.gemmrc(h, wd, y)
        beam.gemmrc_backward(dy, h, wd, da=dh, db=dwd)
        beam.gated_gemmrc_backward(dh, x, wg, wu, gate, up, da=dx, db_gate=dwg, db_up=dwu)

    def compare():
        leaves = [v.double().requires_grad_() for v in (x, wg, wu, wd)]
        hh = torch.nn.functional.silu(leaves[0] @ leaves[1].t()) * (leaves[0] @ leaves[2].t())
        yy = hh @ leaves[3].t()
        yy.backward(dy.double())
        # three roundings to bf16 lie between the inputs and the furthest result, each within 2^-8 per element: in the
        # 2-norm of a whole result below 3 x 2^-8
        for got, want in [(y, yy)] + [(g, v.grad) for g, v in zip((dx, dwg, dwu, dwd), leaves)]:
            assert (got.double() - want).norm() <= 3 * 2.0 ** -8 * want.norm()

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    compare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    x.copy_(normal(x.shape, t, 31))
    dy.copy_(normal(dy.shape, t, 32))
    for v in (y, dx, dwg, dwu, dwd):
        v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    compare()


@pytest.mark.gpu
def test_two_streams_at_once(beam, healthy):
    """Calls on two streams share no scratch: both give what they give alone."""
    m, f, k = 640, 1160, 520
    sets = []
    for j in range(2):
        a, bg, bu = gated_inputs(m, f, k, torch.float16, 50 + j)
        rest = [normal((m, f), torch.float16, 60 + 3 * j + i) for i in range(3)]
        sets.append([rest[0], a, bg, bu, rest[1], rest[2]])
    alone = []
    for s in sets:
        out = [torch.empty_like(s[i]) for i in (1, 2, 3)]
        beam.gated_gemmrc_backward(*s, *out)
        alone.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[torch.empty_like(s[i]) for i in (1, 2, 3)] for s in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, st in zip(sets, outs, streams):
            with torch.cuda.stream(st):
                beam.gated_gemmrc_backward(*s, *o)
    torch.cuda.synchronize()
    for o, want in zip(outs, alone):
        assert all(torch.equal(x, y) for x, y in zip(o, want))


@pytest.mark.gpu
def test_shared_contractions_on_two_streams(beam, healthy):
    """Launches whose CTAs wait for one another, on two streams at once with single-CTA launches between them: all finish, and give
    what they give alone."""
    shapes = [(3, 512, 4096), (40, 2048, 4096), (3, 64, 512), (100, 1000, 8192)]
    sets = [gated_inputs(m, f, k, torch.bfloat16, 7 * j) for j, (m, f, k) in enumerate(shapes)]
    alone = []
    for (m, f, _), s in zip(shapes, sets):
        alone.append(torch.empty(m, f, dtype=torch.bfloat16, device="cuda"))
        beam.gated_gemmrc(*s, alone[-1])
    outs = [[torch.empty_like(c) for c in alone] for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(50):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                for j in range(len(sets)):
                    i = (j + 2 * n) % len(sets)
                    beam.gated_gemmrc(*sets[i], outs[n][i])
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(x, y) for x, y in zip(out, alone))


@pytest.mark.gpu
def test_refusals_on_the_device(beam):
    a, bg, bu = gated_inputs(4, 16, 32, torch.float16)
    c = torch.empty(4, 16, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="together"):
        beam.gated_gemmrc(a, bg, bu, c, gate=torch.empty_like(c))
    with pytest.raises(TypeError):
        beam.gated_gemmrc(a, bg, bu.bfloat16(), c)
    with pytest.raises(ValueError):
        beam.gated_gemmrc(a, bg, bu[:8], c)
    with pytest.raises(ValueError, match="contiguous"):
        beam.gated_gemmrc(a, bg, bu, torch.empty(16, 4, dtype=torch.float16, device="cuda").t())
    with pytest.raises(ValueError):                                  # c shares memory with a
        beam.gated_gemmrc(a, bg, bu, a.view(-1)[:64].view(4, 16))
    with pytest.raises(ValueError):                                  # K no multiple of 8
        beam.gated_gemmrc(a[:, :12].contiguous(), bg[:, :12].contiguous(), bu[:, :12].contiguous(), c)
    with pytest.raises(ValueError, match="at least one"):
        beam.gated_gemmrc_backward(c, a, bg, bu, c, c)
    with pytest.raises(ValueError, match="at least one"):
        beam.gemmrc_backward(c, a, bg)
    with pytest.raises(ValueError):
        beam.gemmrc_backward(c, a, bg, da=a)                         # in place


@pytest.mark.gpu
def test_two_graphs_replayed_at_once(beam, healthy):
    """Graphs captured one after the other on one stream own their scratch: replayed on two streams at the same time they give what
    they give alone."""
    made = []
    for j in range(2):
        a, bg, bu = gated_inputs(333, 1096, 520, torch.bfloat16, 70 + j)
        rest = [normal((333, 1096), torch.bfloat16, 80 + 3 * j + i) for i in range(3)]
        args = [rest[0], a, bg, bu, rest[1], rest[2]]
        outs = [torch.empty_like(t) for t in (a, bg, bu)]
        beam.gated_gemmrc_backward(*args, *outs)
        made.append((args, outs, [t.clone() for t in outs]))
    torch.cuda.synchronize()
    stream, graphs = torch.cuda.Stream(), []
    for args, outs, _ in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            beam.gated_gemmrc_backward(*args, *outs)
        graphs.append(graph)
    for _, outs, _ in made:
        for t in outs:
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, outs, want in made:
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.gpu
@pytest.mark.parametrize("m", (5, 300))
def test_views_inside_larger_tensors(beam, healthy, m):
    """Contiguous views that start 16 bytes into an allocation are taken as they are; a start that is no multiple of 16 bytes is
    refused."""
    f, k = 264, 200

    def inside(t, offset):
        room = torch.full((t.numel() + 64,), 5.0, dtype=t.dtype, device="cuda")
        view = room[offset:offset + t.numel()].view(t.shape)
        view.copy_(t)
        return room, view

    a, bg, bu = gated_inputs(m, f, k, torch.float16, 11)
    rooms = [inside(t, 8) for t in (a, bg, bu, torch.zeros(m, f, dtype=torch.float16, device="cuda"))]
    (_, va), (_, vg), (_, vu), (room, c) = rooms
    beam.gated_gemmrc(va, vg, vu, c)
    check_gated(a, bg, bu, "silu", c)
    assert (room[:8] == 5).all() and (room[8 + c.numel():] == 5).all()
    for j in range(4):
        args = [va, vg, vu, c]
        args[j] = inside(args[j], 4)[1]
        with pytest.raises(ValueError, match="alignment"):
            beam.gated_gemmrc(*args)


@pytest.mark.gpu
def test_offsets_past_two_to_the_31(beam, healthy):
    """More than 2^31 output elements: the last rows are right."""
    m, f, k = 135000, 16384, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    a, bg, bu = gated_inputs(m, f, k, torch.bfloat16, 13)
    c = torch.empty(m, f, dtype=torch.bfloat16, device="cuda")
    beam.gated_gemmrc(a, bg, bu, c, activation="relu")
    check_gated(a[-300:], bg, bu, "relu", c[-300:])
    check_gated(a[:300], bg, bu, "relu", c[:300])
    da = torch.empty_like(a)
    beam.gemmrc_backward(c, a, bg, da=da)
    left, right = c[-300:].double(), bg.double().t()
    want = left @ right.t()
    check(da[-300:], want, half_step(c.dtype) * want.abs() + 1.01 * summing(left, right))


@pytest.mark.gpu
def test_same_bits_every_time(beam, healthy):
    """Shared contractions, slices and two issuers add in a fixed order: equal bits from run to run, also while the device is busy."""
    noise = normal((4096, 4096), torch.bfloat16, 1)
    for m, f, k in ((3, 1000, 4104), (100, 2000, 2056), (300, 2744, 520)):
        a, bg, bu = gated_inputs(m, f, k, torch.bfloat16, 90)
        gate, up, dc = (normal((m, f), torch.bfloat16, 91 + j) for j in range(3))
        seen = []
        for j in range(4):
            c = torch.empty(m, f, dtype=torch.bfloat16, device="cuda")
            grads = [torch.empty_like(t) for t in (a, bg, bu)]
            if j:
                with torch.cuda.stream(torch.cuda.Stream()):
                    torch.matmul(noise, noise)
            beam.gated_gemmrc(a, bg, bu, c)
            beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, *grads)
            seen.append([c] + grads)
        torch.cuda.synchronize()
        for other in seen[1:]:
            assert all(torch.equal(x, y) for x, y in zip(seen[0], other)), (m, f, k)
