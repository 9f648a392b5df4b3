"""MXFP4 quantisation and product: refusals on the CPU, results on the GPU against the definition in 64 bits.

Quantisation and its inverse are exact operations and one rounding: results are equal, not close.  The product adds, per 64
elements of K, products that are exact in fp32 to a partial sum; products of one step are aligned to the largest before they
are added, so a step may lose one part in 2^22 of the largest sum S = sum |a||b| twice: (K / 32 + 4) 2^-22 S, and one rounding
to the output type, torch.finfo(t).eps / 2 (or half the spacing of fp16's subnormals, 2^-25).
"""
import ctypes

import pytest
import torch

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def round64(x):
    """(the quantised values of x, the scale bytes [rows, k / 32]) by the definition, in 64 bits."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    bad = ~top.isfinite()
    _, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    e = torch.where(top == 0, torch.full_like(e, -127), e - 3).clamp(min=-127)
    unit = torch.exp2(e.double())
    v = torch.where(bad, torch.zeros_like(b), b / unit)
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    off = (v.abs().unsqueeze(-1) - table).abs()
    near = off.amin(-1, keepdim=True)
    hit = off == near                                   # two codes at a tie: the even one
    even = hit & (torch.arange(8, device=x.device) % 2 == 0)
    code = torch.where(hit.sum(-1) > 1, even.double().argmax(-1), hit.double().argmax(-1))
    q = table[code] * torch.where(torch.signbit(v), -1.0, 1.0)
    values = torch.where(bad, torch.full_like(q, float("nan")), q * unit).reshape(x.shape)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1)
    return values, scale.to(torch.uint8)


def untile(t, rows, cols):
    r, c = torch.arange(rows, device=t.device)[:, None], torch.arange(cols, device=t.device)[None]
    return t.reshape(-1)[((r // 128) * t.shape[1] + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4]


def matrix(rows, k, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=g) * scale
    return (x * torch.exp(torch.randn(1, k, device="cuda", generator=g))).to(dtype)


def quantized(beam, x):
    q, s = beam.mxfp4_empty(x.shape[0], x.shape[1], x.device)
    q.fill_(0xAA)
    s.fill_(0xFF)
    beam.mxfp4_quantize(x, q, s)
    return q, s


def check_product(c, a64, b64):
    t = c.dtype
    want = a64 @ b64.t()
    size = a64.abs() @ b64.abs().t()
    tol = torch.finfo(t).eps / 2 * want.abs() + 1.01 * (a64.shape[1] / 32 + 4) * 2.0 ** -22 * size
    tol = tol + (2.0 ** -25 if t == torch.float16 else 0)
    off = (c.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), "%d of %d off, worst %g" % (bad.sum(), bad.numel(), off[bad].max())


@pytest.fixture(scope="module")
def beam(built_library):
    import beam as beam_pkg
    return beam_pkg


@pytest.fixture
def healthy(beam):
    yield
    assert beam.device_status() == (0, 0)


# ---------------------------------------------------------------------------------------------------- CPU
def test_c_entries_refuse_bad_arguments(built_library):
    if torch.cuda.is_available():
        pytest.skip("host memory stands in for device pointers")
    L = ctypes.CDLL(built_library)
    vp, i = ctypes.c_void_p, ctypes.c_int
    raw = ctypes.create_string_buffer((1 << 19) + 64)
    base = (ctypes.addressof(raw) + 63) & ~63
    p = [base + (j << 16) for j in range(6)]
    size = L.beam_mxfp4_scales_bytes
    size.restype, size.argtypes = ctypes.c_size_t, [i, i]
    assert size(1, 32) == 512 and size(129, 160) == 4 * 512 and size(128, 128) == 512 and size(0, 32) == 0

    def call(fn, args, **change):
        args = list(args)
        for k, v in change.items():
            args[int(k[1:])] = v
        return fn(*args)

    f = L.beam_mxfp4_quantize
    f.argtypes = [vp, vp, vp, i, i, i, vp]
    good = [p[0], p[1], p[2], 16, 64, 0, None]
    assert call(f, good) == 8 and call(f, good, _5=2) == 8
    for j in range(3):
        assert call(f, good, **{"_%d" % j: None}) == 1 and call(f, good, **{"_%d" % j: p[j] + 4}) == 3
    assert call(f, good, _3=0) == 1 and call(f, good, _4=-32) == 1 and call(f, good, _4=48) == 3
    assert call(f, good, _5=1) == 1 and call(f, good, _1=p[0]) == 1 and call(f, good, _2=p[1] + 16) == 1
    f = L.beam_mxfp4_dequantize
    f.argtypes = [vp, vp, vp, i, i, i, vp]
    assert call(f, good) == 8 and call(f, good, _5=2) == 8
    assert call(f, good, _5=3) == 1 and call(f, good, _5=-1) == 1 and call(f, good, _4=40) == 3
    assert call(f, good, _2=p[0]) == 1
    f = L.beam_mxfp4_gemmrc
    f.argtypes = [vp] * 5 + [i, i, i, i, vp]
    good = p[:5] + [16, 32, 64, 0, None]
    assert call(f, good) == 8
    for j in range(5):
        assert call(f, good, **{"_%d" % j: None}) == 1 and call(f, good, **{"_%d" % j: p[j] + 8}) == 3
    assert call(f, good, _5=0) == 1 and call(f, good, _6=12) == 3 and call(f, good, _7=80) == 3
    assert call(f, good, _8=4) == 1 and call(f, good, _4=p[3]) == 1
    # more units of 128 elements than 32 bits count
    assert call(f, good, _5=1 << 30, _7=1 << 12) == 2


def test_python_refusals_and_layout(beam):
    with pytest.raises(ValueError):
        beam.mxfp4_empty(4, 48, "cpu")
    with pytest.raises(ValueError):
        beam.mxfp4_empty(0, 32, "cpu")
    q, s = beam.mxfp4_empty(130, 160, "cpu")
    assert q.shape == (130, 80) and s.shape == (2, 2, 512)
    with pytest.raises(ValueError, match="CUDA"):
        beam.mxfp4_quantize(torch.zeros(130, 160).half(), q, s)
    with pytest.raises(ValueError, match="CUDA"):
        beam.mxfp4_dequantize(q, s, torch.zeros(130, 160))
    with pytest.raises(ValueError, match="CUDA"):
        beam.mxfp4_gemmrc(q, s, q, s, torch.zeros(130, 130).half())
    with pytest.raises(TypeError):
        beam.mxfp4_tile_scales(torch.zeros(3, 3))
    flat = torch.randint(0, 255, (130, 5), dtype=torch.uint8)
    t = beam.mxfp4_tile_scales(flat)
    assert t.shape == (2, 2, 512) and torch.equal(untile(t, 130, 5), flat)
    assert int(t.long().sum()) == int(flat.long().sum())  # zeros elsewhere


# ------------------------------------------------------------------------------------------- quantisation, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 96), (127, 160), (128, 128), (130, 1056), (333, 8192)])
def test_quantize_and_back(beam, healthy, dtype, rows, k):
    x = matrix(rows, k, dtype, rows + k)
    q, s = quantized(beam, x)
    want, scale = round64(x)
    assert torch.equal(s, beam.mxfp4_tile_scales(scale))    # zeros outside the matrix among them
    for t in (dtype, torch.float32):
        y = torch.empty(rows, k, dtype=t, device="cuda")
        beam.mxfp4_dequantize(q, s, y)
        assert torch.equal(y, want.to(t)), t


@pytest.mark.gpu
def test_quantize_borders(beam, healthy):
    """Every tie and its neighbours, at every scale of bf16, both signs; all-zero blocks; the largest and smallest numbers."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5], dtype=torch.float64)
    rows = []
    for e in list(range(-133, 126, 7)) + [125]:
        v = torch.cat([ties * s for s in (1.0, 1 + 2.0 ** -7, 1 - 2.0 ** -7)]) * 2.0 ** e
        row = torch.cat([v, -v[:30], torch.tensor([4.0 * 2.0 ** e, 0.0]), torch.zeros(2)])
        rows.append(torch.cat([row, torch.zeros(96 - row.numel())]))
    x = torch.stack(rows).to(torch.bfloat16).cuda()
    x[1] = 0
    x[2, :32] = -0.0
    q, s = quantized(beam, x)
    want, scale = round64(x)
    assert torch.equal(untile(s, x.shape[0], 3), scale)
    y = torch.empty(x.shape, dtype=torch.float32, device="cuda")
    beam.mxfp4_dequantize(q, s, y)
    assert torch.equal(y.double(), want)
    b = torch.empty(x.shape, dtype=torch.bfloat16, device="cuda")
    beam.mxfp4_dequantize(q, s, b)
    assert torch.equal(b.double(), want)
    h = torch.empty(x.shape, dtype=torch.float16, device="cuda")
    beam.mxfp4_dequantize(q, s, h)
    assert torch.equal(h, y.half())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_infinities_and_nan_stay_in_their_block(beam, healthy, dtype):
    x = matrix(5, 128, dtype, 3)
    clean = x.clone()
    x[1, 40], x[3, 127], x[4, 0] = float("inf"), float("nan"), float("-inf")
    q, s = quantized(beam, x)
    y = torch.empty_like(x)
    beam.mxfp4_dequantize(q, s, y)
    bad = torch.zeros(5, 128, dtype=torch.bool, device="cuda")
    bad[1, 32:64] = bad[3, 96:] = bad[4, :32] = True
    assert torch.equal(y.isnan(), bad)
    assert torch.equal(y[~bad], round64(clean)[0].to(dtype)[~bad])
    for m in (5, 200):  # and in their row of a product
        a = x.repeat(40, 1)[:m].contiguous()
        qa, sa = quantized(beam, a)
        w = matrix(64, 128, dtype, 4)
        c = torch.empty(m, 64, dtype=dtype, device="cuda")
        beam.mxfp4_gemmrc(qa, sa, *quantized(beam, w), c)
        r = torch.arange(m, device="cuda") % 5
        lost = (r == 1) | (r == 3) | (r == 4)
        assert c[lost].isnan().all() and c[~lost].isfinite().all()


# ------------------------------------------------------------------------------------------------- product, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 4736, 256), (2, 128, 64), (7, 200, 96), (16, 1192, 160), (77, 5464, 128),
                                   (128, 4744, 1056), (128, 264, 4096), (129, 8, 32), (200, 264, 96), (256, 256, 256),
                                   (300, 1000, 1376), (513, 776, 544), (1024, 2048, 2048), (2304, 2560, 512),
                                   (5, 20008, 320), (33, 2072, 8224), (128, 4100 // 4 * 8, 4128)])
def test_product(beam, healthy, dtype, m, n, k):
    a, b = matrix(m, k, dtype, m + k), matrix(n, k, dtype, n, k ** -0.5)
    a64, b64 = round64(a)[0], round64(b)[0]
    room = torch.full((m + 2, n), 3.0, dtype=dtype, device="cuda")
    beam.mxfp4_gemmrc(*quantized(beam, a), *quantized(beam, b), room[1:-1])
    check_product(room[1:-1], a64, b64)
    assert (room[0] == 3).all() and (room[-1] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", (3, 300))
def test_every_code_and_scale_position(beam, healthy, m):
    """b is 0 except for a run of 32 elements that moves along K with the row, and every row and block has a scale of its own: a
    scale taken from another row, block or position shows."""
    k, n = 544, 320
    g = torch.Generator(device="cuda").manual_seed(5)
    qa = torch.randint(0, 256, (m, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    sa = torch.randint(110, 140, (m, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    qb = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    live = (torch.arange(k // 2, device="cuda")[None] // 16) == (torch.arange(n, device="cuda")[:, None] % (k // 32))
    qb *= live
    sb = torch.randint(110, 140, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8)

    def values(q, s):
        code = torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).long()
        v = torch.tensor(VALUES, dtype=torch.float64, device="cuda")[code & 7] * torch.where(code > 7, -1.0, 1.0)
        return v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)

    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    beam.mxfp4_gemmrc(qa, beam.mxfp4_tile_scales(sa), qb, beam.mxfp4_tile_scales(sb), c)
    check_product(c, values(qa, sa), values(qb, sb))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 200))
def test_a_feed_forward_block_in_four_bits(beam, healthy, rows):
    """x to 4 bits, a projection with 4-bit weights, the gated product in 16 bits on its result, 4 bits again and back to the
    width: eagerly and as a graph replayed on another x, equal to the steps checked one by one."""
    d, f, t = 256, 416, torch.bfloat16
    w1, w2 = matrix(d, d, t, 1, d ** -0.5), matrix(d, f, t, 2, f ** -0.5)
    wg, wu = matrix(f, d, t, 3, d ** -0.5), matrix(f, d, t, 4, d ** -0.5)
    q1, q2 = quantized(beam, w1), quantized(beam, w2)
    x, mid, h, y = matrix(rows, d, t, 5), *(torch.empty(rows, n, dtype=t, device="cuda") for n in (d, f, d))

    def step():
        qx = beam.mxfp4_empty(rows, d, x.device)
        beam.mxfp4_quantize(x, *qx)
        beam.mxfp4_gemmrc(*qx, *q1, mid)
        beam.gated_gemmrc(mid, wg, wu, h)
        qh = beam.mxfp4_empty(rows, f, x.device)
        beam.mxfp4_quantize(h, *qh)
        beam.mxfp4_gemmrc(*qh, *q2, y)

    def compare():
        check_product(mid, round64(x)[0], round64(w1)[0])
        check_product(y, round64(h)[0], round64(w2)[0])
        g, u = mid.double() @ wg.double().t(), mid.double() @ wu.double().t()
        want = torch.nn.functional.silu(g) * u
        assert (h.double() - want).norm() <= 2.0 ** -8 * want.norm()

    step()
    torch.cuda.synchronize()
    compare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x.copy_(matrix(rows, d, t, 6))
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    compare()


@pytest.mark.gpu
def test_refusals_on_the_device(beam):
    x = matrix(16, 64, torch.float16, 1)
    q, s = quantized(beam, x)
    c = torch.empty(16, 16, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError):
        beam.mxfp4_quantize(x.float(), q, s)
    with pytest.raises(ValueError):
        beam.mxfp4_quantize(x[:8], q, s)
    with pytest.raises(ValueError):
        beam.mxfp4_quantize(x, q, s.view(-1))
    with pytest.raises(TypeError):
        beam.mxfp4_dequantize(q, s, torch.empty(16, 64, dtype=torch.float64, device="cuda"))
    with pytest.raises(TypeError):
        beam.mxfp4_gemmrc(q, s, q, s, c.float())
    with pytest.raises(ValueError):
        beam.mxfp4_gemmrc(q, s, q[:, :16].contiguous(), s, c)
    with pytest.raises(ValueError):
        beam.mxfp4_gemmrc(q, s, q[:12].contiguous(), s, c[:, :12].contiguous())  # N no multiple of 8


@pytest.mark.gpu
def test_offsets_past_two_to_the_31(beam, healthy):
    """More than 2^31 elements to 4 bits and back, and a product whose second operand starts past 2^31: the last rows are right."""
    rows, k = 70000, 32768
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, s = beam.mxfp4_empty(rows, k)
    beam.mxfp4_quantize(x, q, s)
    y = torch.empty_like(x)
    beam.mxfp4_dequantize(q, s, y)
    for part in (slice(0, 200), slice(rows - 200, rows)):
        assert torch.equal(y[part], round64(x[part])[0].bfloat16())
    del y
    a = matrix(4, k, torch.bfloat16, 2)
    c = torch.empty(4, rows, dtype=torch.bfloat16, device="cuda")
    beam.mxfp4_gemmrc(*quantized(beam, a), q, s, c)
    check_product(c[:, -200:].contiguous(), round64(a)[0], round64(x[-200:])[0])


@pytest.mark.gpu
def test_bad_placement_is_refused(beam):
    x = matrix(4, 64, torch.float16, 1)
    q, s = quantized(beam, x)
    room = torch.zeros(4 * 32 + 8, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="alignment"):
        beam.mxfp4_quantize(x, room[8:136].view(4, 32), s)
    with pytest.raises(ValueError):  # scales inside q's memory
        big = torch.zeros(4096, dtype=torch.uint8, device="cuda")
        beam.mxfp4_quantize(x, big[:128].view(4, 32), big[64:576].view(1, 1, 512))
    with pytest.raises(ValueError):  # a view with gaps
        beam.mxfp4_quantize(x[::2], q[:2], s)
