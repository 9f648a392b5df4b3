"""The feed-forward and 4-bit products at sizes for which the launchers choose each of their forms, every element against the
formulas in 64 bits (tolerances: see test_feedforward.py and test_mxfp4.py, whose checks are used).  The forms named beside the
sizes are those of a B200 with 148 SMs; on another device the sizes choose other forms and the results are checked all the same.
"""
import pytest
import torch

from test_feedforward import ACTS, check, check_gated, check_gated_backward, floor_of, gated_inputs, half_step, normal, summing
from test_mxfp4 import check_product, matrix, quantized, round64


@pytest.fixture(scope="module")
def beam(built_library):
    import beam as beam_pkg
    return beam_pkg


@pytest.fixture
def healthy(beam):
    yield
    assert beam.device_status() == (0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m,f,k", [
    (300, 2744, 520),    # pairs, 96 columns, one wave
    (900, 1600, 1160),   # ... K longer than the ring
    (2500, 4008, 200),   # ... six tiles a pair: both accumulators come round again
    (2500, 4008, 64),    # ... a single k-block: the epilogue is the slower part
    (300, 2000, 520),    # pairs, 64 columns, two issuers
    (300, 2000, 136),    # ... two k-blocks for one, one for the other
    (1200, 2800, 520),   # ... three tiles a pair
    (600, 6000, 328),    # pairs, 128 columns, two tiles a pair
    (4000, 8008, 136),   # ... fourteen
    (5, 8000, 1032),     # one CTA a tile, 56 columns, two issuers, zeros in the rows that do not exist
    (1, 16384, 1032),    # ... 112 columns, one issuer
    (100, 16000, 1032),  # ... 112 columns, 104 rows loaded
    (120, 9472, 1032),   # ... 64 columns
    (7, 40000, 1032),    # ... several tiles a CTA, K longer than the ring
    (3, 1184, 4096),     # four CTAs share a contraction, 64 columns
    (100, 1184, 4104),
    (2, 2200, 2056),     # two CTAs share a contraction
])
def test_gated(beam, healthy, dtype, m, f, k):
    a, bg, bu = gated_inputs(m, f, k, dtype, m + f)
    act = ACTS[(m + f // 8 + k // 8) % 4]
    room = torch.full((3, m + 2, f), 3.0, dtype=dtype, device="cuda")
    c, gate, up = (room[j, 1:-1] for j in range(3))
    beam.gated_gemmrc(a, bg, bu, c, activation=act, gate=gate, up=up)
    check_gated(a, bg, bu, act, c, gate, up)
    assert (room[:, 0] == 3).all() and (room[:, -1] == 3).all()
    alone = torch.empty_like(c)
    beam.gated_gemmrc(a, bg, bu, alone, activation=act)
    assert torch.equal(alone, c)


@pytest.mark.gpu
@pytest.mark.parametrize("m", (3, 300))
def test_gated_long_contraction(beam, healthy, m):
    """K as long as a feed-forward layer is wide."""
    a, bg, bu = gated_inputs(m, 264, 28672, torch.bfloat16, 5)
    c = torch.empty(m, 264, dtype=a.dtype, device="cuda")
    beam.gated_gemmrc(a, bg, bu, c, activation="gelu")
    check_gated(a, bg, bu, "gelu", c)


@pytest.mark.gpu
def test_gated_with_one_weight_for_both(beam, healthy):
    """Inputs may be one tensor: c = act(g) g."""
    for m in (5, 300):
        a, bg, _ = gated_inputs(m, 264, 136, torch.float16, 6)
        c = torch.empty(m, 264, dtype=a.dtype, device="cuda")
        beam.gated_gemmrc(a, bg, bg, c)
        check_gated(a, bg, bg, "silu", c)


@pytest.mark.gpu
def test_gated_gradients_in_several_launches(beam, healthy):
    """A list of 256 + 512 + 512 tiles goes out in two launches, the first of which ends among the tiles of a weight's gradient."""
    m, f, k, t = 4096, 8200, 4104, torch.bfloat16
    a, bg, bu = gated_inputs(m, f, k, t, 3)
    gate, up, dc = normal((m, f), t, 5, 2.0), normal((m, f), t, 6), normal((m, f), t, 7)
    grads = [torch.full_like(x, 3.0) for x in (a, bg, bu)]
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, *grads, activation="gelu_tanh")
    check_gated_backward(dc, a, bg, bu, gate, up, "gelu_tanh", *grads)
    one = torch.full_like(bu, 3.0)
    beam.gated_gemmrc_backward(dc, a, bg, bu, gate, up, db_up=one, activation="gelu_tanh")
    assert torch.equal(one, grads[2])


def check_gradients(dc, a, b, da, db):
    for got, left, right in ((da, dc.double(), b.double().t()), (db, dc.double().t(), a.double().t())):
        want = left @ right.t()
        check(got, want, half_step(a.dtype) * want.abs() + 1.01 * summing(left, right) + floor_of(a.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,n,k", [
    (torch.float16, 8192, 4104, 8200),   # several launches, cut among the tiles of da
    (torch.bfloat16, 40, 28672, 264),    # a long contraction of few tiles, sliced
    (torch.float16, 28680, 40, 264),     # ... of db
    (torch.bfloat16, 2600, 2600, 2600),  # several tiles a pair in one launch
])
def test_gradients(beam, healthy, dtype, m, n, k):
    dc, a, b = normal((m, n), dtype, 1), normal((m, k), dtype, 2), normal((n, k), dtype, 3)
    da, db = torch.full_like(a, 3.0), torch.full_like(b, 3.0)
    beam.gemmrc_backward(dc, a, b, da=da, db=db)
    check_gradients(dc, a, b, da, db)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m,n,k", [
    (4104, 5000, 96),     # pairs, 340 tiles: each accumulator is used three times, the epilogue is the slower part
    (4104, 5000, 2080),   # ... K longer than the ring
    (2600, 7688, 544),
    (100, 40008, 544),    # one CTA a tile, 128 columns, several tiles a CTA
    (7, 2048, 8224),      # four CTAs share a contraction
    (128, 4736, 4128),    # two
    (3, 520, 28672), (300, 264, 28672),
])
def test_mxfp4_product(beam, healthy, dtype, m, n, k):
    a, b = matrix(m, k, dtype, m + k), matrix(n, k, dtype, n, k ** -0.5)
    a64, b64 = round64(a)[0], round64(b)[0]
    room = torch.full((m + 2, n), 3.0, dtype=dtype, device="cuda")
    beam.mxfp4_gemmrc(*quantized(beam, a), *quantized(beam, b), room[1:-1])
    check_product(room[1:-1], a64, b64)
    assert (room[0] == 3).all() and (room[-1] == 3).all()


@pytest.mark.gpu
def test_mxfp4_product_with_itself(beam, healthy):
    """Inputs may be one matrix."""
    for rows in (40, 264):
        x = matrix(rows, 160, torch.bfloat16, rows)
        q, c = quantized(beam, x), torch.empty(rows, rows, dtype=x.dtype, device="cuda")
        beam.mxfp4_gemmrc(*q, *q, c)
        check_product(c, round64(x)[0], round64(x)[0])


@pytest.mark.gpu
def test_every_kind_of_call_on_three_streams(beam, healthy):
    """Calls whose CTAs wait for one another (pairs, shared contractions, the one-kernel split-K) and calls whose CTAs share an SM,
    on three streams at once and in different orders: all finish and give what they give alone."""
    t = torch.float16
    x, w = normal((300, 512), t, 1), normal((512, 512), t, 2, 512 ** -0.5)
    lx, lw = normal((8, 8192), t, 3), normal((64, 8192), t, 4, 8192 ** -0.5)
    dc = normal((300, 512), t, 5)
    qx, qw, ql, qlw = (quantized(beam, v) for v in (x, w, lx, lw))
    calls = [
        ((300, 512), lambda o: beam.gated_gemmrc(x, w, w, o)),
        ((3, 512), lambda o: beam.gated_gemmrc(x[:3], w, w, o)),
        ((8, 64), lambda o: beam.gated_gemmrc(lx, lw, lw, o)),
        ((300, 512), lambda o: beam.gemmrc_backward(dc, x, w, da=o)),
        ((300, 512), lambda o: beam.mxfp4_gemmrc(*qx, *qw, o)),
        ((8, 64), lambda o: beam.mxfp4_gemmrc(*ql, *qlw, o)),
        ((300, 512), lambda o: beam.gemmrc(x, w, o)),
        ((300, 512), lambda o: beam.gemmrc(x, w, o, tile_n=128, cta_pair=2, stages=4)),
        ((300, 512), lambda o: beam.gemmrc(x, w, o, tile_n=64, cta_pair=1, stages=4)),
        ((8, 64), lambda o: beam.cutlass_gemmrc_splitk(lx, lw, o, two_kernels=False)),
        ((8, 64), lambda o: beam.cutlass_gemmrc_splitk(lx, lw, o, two_kernels=True)),
        ((300, 512), lambda o: beam.mxfp4_dequantize(*qx, o)),
    ]
    alone = [torch.empty(s, dtype=t, device="cuda") for s, _ in calls]
    for (_, call), out in zip(calls, alone):
        call(out)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.zeros_like(o) for o in alone] for _ in streams]
    torch.cuda.synchronize()
    for r in range(30):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for j in range(len(calls)):
                    i = (j * (1, 5, 7)[n] + r) % len(calls)
                    calls[i][1](outs[n][i])
    torch.cuda.synchronize()
    for out in outs:
        for o, want in zip(out, alone):
            assert torch.equal(o, want)


@pytest.mark.gpu
def test_no_rows_are_refused(beam):
    """An empty batch is an error that the host raises; nothing is launched and nothing written."""
    a, bg, bu = gated_inputs(4, 16, 32, torch.float16)
    c, none = torch.full((4, 16), 3.0, dtype=torch.float16, device="cuda"), torch.empty(0, 16, dtype=torch.float16, device="cuda")
    db = torch.full_like(bg, 3.0)
    with pytest.raises(ValueError):
        beam.gated_gemmrc(a[:0], bg, bu, none)
    with pytest.raises(ValueError):
        beam.gated_gemmrc(a, bg[:0], bu[:0], c[:, :0].contiguous())
    with pytest.raises(ValueError):
        beam.gated_gemmrc_backward(none, a[:0], bg, bu, none, none, db_gate=db)
    with pytest.raises(ValueError):
        beam.gemmrc_backward(none, a[:0], bg, db=db)
    q, scales = beam.mxfp4_empty(4, 32)
    with pytest.raises(ValueError):
        beam.mxfp4_quantize(a[:0], q[:0], scales[:0])
    with pytest.raises(ValueError):
        beam.mxfp4_gemmrc(q[:0], scales[:0], q, scales, none[:, :4].contiguous())
    torch.cuda.synchronize()
    assert (db == 3).all() and (c == 3).all()
