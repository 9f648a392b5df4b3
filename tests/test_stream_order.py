"""Kernels that are launched as programmatic dependents and their place on the stream.

A kernel may start before the one ahead of it has finished.  What keeps results right is an order inside every kernel: it waits
for the kernel ahead (griddepcontrol.wait), and only then lets the one behind start (griddepcontrol.launch_dependents); and a
CTA that needs TMEM has it by then.  A violation is a race between kernels, so the order is read from the sources here, on
the CPU; the GPU tests run chains of calls in which a violation would show.
"""
import glob
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WAIT, RELEASE, ALLOC = "ptx::grid_dependency_wait()", "ptx::grid_launch_dependents()", "ptx::tmem_alloc<"
# Split-K kernels let the next call stream beside them on purpose; BEAM_FLAG_INPUTS_STABLE says what a caller vouches for.
SPLIT_K = {"splitk_stream_kernel", "splitk_reduce_kernel", "splitk_reduce_flat_kernel", "gemmrc_umma_kernel"}
ORDERED = ("gated_umma.cuh", "grad_umma.cuh", "mxfp4_umma.cuh", "gemmrc_dual.cuh", "gemmrc_wide.cuh")


def bare(text):
    return re.sub(r"//[^\n]*", "", text)


def kernels(path):
    """name -> body of every kernel of a file, with calls of release_next_kernel() spelled out."""
    with open(os.path.join(ROOT, "general-nvgpu-testing_b200", "csrc", "umma_common.cuh")) as f:
        common = bare(f.read())
    release = re.search(r"void release_next_kernel\(uint32_t warp\) \{(.*?)\n\}", common, re.S)
    release = release.group(1) if release else ""
    with open(path) as f:
        text = bare(f.read())
    found = {}
    for m in re.finditer(r"__global__ void __launch_bounds__\([^\n]*\)\s+(\w+)\(", text):
        start = text.index("{", m.end())
        depth, at = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        found[m.group(1)] = text[start:at].replace("release_next_kernel(warp);", release)
    return found


def sources():
    return sorted(glob.glob(os.path.join(ROOT, "general-nvgpu-testing_b200", "csrc", "*.cuh")))


def test_the_sources_are_understood():
    names = {n for p in sources() for n in kernels(p)}
    assert {"gated_umma_kernel", "gated_slope_kernel", "grad_umma_kernel", "grad_reduce_kernel", "mxfp4_quantize_kernel",
            "mxfp4_dequantize_kernel", "mxfp4_umma_kernel"} | SPLIT_K <= names


@pytest.mark.parametrize("name", ORDERED)
def test_dependents_are_released_after_the_wait_and_the_tmem(name):
    path = os.path.join(ROOT, "general-nvgpu-testing_b200", "csrc", name)
    for kernel, body in kernels(path).items():
        assert body.count(RELEASE) == 1, kernel
        release = body.index(RELEASE)
        # the same threads wait directly ahead of it
        assert body[:release].rstrip().endswith(WAIT + ";"), kernel + " lets the next kernel start before it has waited itself"
        if ALLOC in body:
            barrier = body.index("__syncthreads()", body.index(ALLOC))
            assert barrier < release, kernel + " lets the next kernel start before it has its TMEM"


def test_bounded_waits_begin_when_the_kernel_ahead_has_finished():
    with open(os.path.join(ROOT, "general-nvgpu-testing_b200", "csrc", "umma_common.cuh")) as f:
        common = bare(f.read())
    for name in ("bool bounded_wait(", "bool bounded_wait_warp("):
        body = common[common.index(name):]
        body = body[:body.index("\n}")]
        assert re.search(r"if \(t0 == 0\) " + re.escape(WAIT) + r";\s*const uint64_t now = ptx::globaltimer_ns\(\);", body), name


@pytest.mark.parametrize("name", ORDERED)
def test_no_read_only_loads(name):
    """A load through the read-only path may return what the memory held when the kernel began; its inputs may be written after that, by
    the kernel ahead."""
    with open(os.path.join(ROOT, "general-nvgpu-testing_b200", "csrc", name)) as f:
        text = bare(f.read())
    assert "__ldg(" not in text and ".nc" not in text and "__restrict__" not in text


def test_split_k_kernels_wait_before_they_release():
    """... unless the caller vouches for the inputs.  The kernel that leaves room on its SM has its TMEM by then, and the one that
    split-K shares with the plain product keeps the whole order for the latter."""
    seen = {}
    for path in sources():
        seen.update({n: b for n, b in kernels(path).items() if n in SPLIT_K and ALLOC in b})
    assert set(seen) == {"splitk_stream_kernel", "gemmrc_umma_kernel"}
    for kernel, body in seen.items():
        assert 0 <= body.find(WAIT) < body.index(RELEASE), kernel
    body = seen["splitk_stream_kernel"]
    assert body.index("__syncthreads()", body.index(ALLOC)) < body.index(RELEASE)
    body = seen["gemmrc_umma_kernel"]
    first, last = (m.start() for m in re.finditer(re.escape(RELEASE), body))
    assert body[:first].rstrip().endswith("if constexpr (is_splitk_mode(kMode))")
    assert body.index("__syncthreads()", body.index(ALLOC)) < body.index("if constexpr (kMode == kModeGemm)") < last


@pytest.fixture(scope="module")
def beam(built_library):
    import beam as beam_pkg
    return beam_pkg


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("between", ("quantize", "dequantize", "gradient", "product", "plain", "one plain kernel"))
def test_split_k_on_the_result_of_the_call_before_the_last(beam, between):
    """A gated product, a small call on other tensors, then a split-K call on the gated result that vouches for its inputs: they
    are not outputs of the call just before it."""
    m, f, k = 96, 32768, 2048
    a, bg, bu = (normal(s, torch.float16, j, c) for j, (s, c) in enumerate((((m, k), 1.0), ((f, k), k ** -0.5), ((f, k), k ** -0.5))))
    w = normal((64, f), torch.float16, 5, f ** -0.5)
    h, want_h = (torch.empty(m, f, dtype=torch.float16, device="cuda") for _ in range(2))
    c, want_c = (torch.empty(m, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    x = normal((8, 256), torch.float16, 7)
    v, dx = torch.empty_like(x), torch.empty_like(x)
    q, y = beam.mxfp4_empty(8, 256), torch.empty(8, 8, dtype=torch.float16, device="cuda")
    beam.mxfp4_quantize(x, *q)
    beam.gated_gemmrc(a, bg, bu, want_h)
    torch.cuda.synchronize()
    beam.cutlass_gemmrc_splitk(want_h, w, want_c)
    torch.cuda.synchronize()
    for _ in range(20):
        h.zero_()
        c.zero_()
        beam.gated_gemmrc(a, bg, bu, h)
        if between == "quantize":
            beam.mxfp4_quantize(x, *q)
        elif between == "dequantize":
            beam.mxfp4_dequantize(*q, v)
        elif between == "gradient":
            beam.gemmrc_backward(y, x, x, da=dx)
        elif between == "plain":
            beam.gemmrc(x, x, y)
        elif between == "one plain kernel":
            beam.cutlass_gemmrc_splitk(x, x, y, two_kernels=False)
        else:
            beam.mxfp4_gemmrc(*q, *q, y)
        beam.cutlass_gemmrc_splitk(h, w, c, inputs_stable=True)
        # the split factor differs from the plain call's, and with it the order of the sums: at most 512 partial sums per element,
        # each off by 2^-23 of sum |h w|, and the two roundings to fp16
        size = want_h.double().abs() @ w.double().abs().t()
        tol = 2.0 ** -10 * want_c.double().abs() + (f / 16 + 512) * 2.0 ** -22 * size + 2.0 ** -24
        assert ((c.double() - want_c.double()).abs() <= tol).all()
    assert beam.device_status() == (0, 0)


@pytest.mark.gpu
def test_behind_a_call_of_several_seconds(beam):
    """A product held to one pair of CTAs takes some 3 s and leaves the other SMs to the calls behind it, whose CTAs wait there.  What
    they wait for that long is not a fault: bounded waits (2 s) begin when the call ahead has finished."""
    n, k = 16384, 196608
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    a = torch.zeros(n, k, dtype=torch.float16, device="cuda")
    a[:, 5] = 2
    c = torch.empty(n, n, dtype=torch.float16, device="cuda")
    x, w = normal((200, 256), torch.float16, 1), normal((64, 256), torch.float16, 2, 1 / 16)
    xs, ws = normal((40, 4096), torch.float16, 3), normal((40, 4096), torch.float16, 4, 1 / 64)
    shapes = [(200, 64), (3, 64), (200, 64), (200, 64), (200, 256), (40, 40)]
    g = normal((200, 64), torch.float16, 6)
    calls = [lambda o: beam.gated_gemmrc(x, w, w, o), lambda o: beam.gated_gemmrc(x[:3], w, w, o), lambda o: beam.gemmrc(x, w, o),
             lambda o: beam.gemmrc(x, w, o, tile_n=128), lambda o: beam.gemmrc_backward(g, x, w, da=o),
             lambda o: beam.cutlass_gemmrc_splitk(xs, ws, o, two_kernels=False)]
    alone = [torch.zeros(s, dtype=torch.float16, device="cuda") for s in shapes]
    behind = [torch.zeros_like(t) for t in alone]
    for call, out in zip(calls, alone):
        call(out)
        torch.cuda.synchronize()
    for first in (0, 1, 2, 5):
        beam.gemmrc(a, a, c, max_ctas=2)
        for j in range(6):
            calls[(first + j) % 6](behind[(first + j) % 6])
        torch.cuda.synchronize()
        assert beam.device_status() == (0, 0)
        assert (c == 4).all()
        for out, want in zip(behind, alone):
            assert torch.equal(out, want)
            out.zero_()


@pytest.mark.gpu
def test_values_follow_their_quantisation(beam):
    """Quantise and dequantise through the same small tensors again and again: every call returns the values of the latest codes and
    scales."""
    xs = [normal((130, 160), torch.bfloat16, j, 4.0 ** (j - 4)) for j in range(8)]
    codes, alone = beam.mxfp4_empty(130, 160), []
    for x in xs:
        q = beam.mxfp4_empty(130, 160)
        beam.mxfp4_quantize(x, *q)
        torch.cuda.synchronize()
        alone.append(torch.empty(130, 160, device="cuda"))
        beam.mxfp4_dequantize(*q, alone[-1])
        torch.cuda.synchronize()
    seen = [[torch.empty_like(v) for v in alone] for _ in range(25)]
    for out in seen:
        for x, v in zip(xs, out):
            beam.mxfp4_quantize(x, *codes)
            beam.mxfp4_dequantize(*codes, v)
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for out in seen for v, want in zip(out, alone))


@pytest.mark.gpu
def test_long_chains_of_small_calls(beam):
    """Narrow gated products take little shared memory: several of a chain's CTAs fit on one SM, and each needs all of its TMEM.  The
    chain finishes, and every call sees the result of the one before."""
    d, t = 512, torch.bfloat16
    # element 0 stays 1 and is every element's gate; the others are turned by an orthogonal matrix
    gate, up = torch.zeros(2, d, d, dtype=t, device="cuda")
    gate[:, 0] = 1
    up[0, 0] = 1
    up[1:, 1:] = torch.linalg.qr(normal((d - 1, d - 1), torch.float64, 10))[0].to(t)
    x = [normal((1, d), t, 20)] + [torch.full((1, d), float("nan"), dtype=t, device="cuda") for _ in range(200)]
    x[0][0, 0] = 1
    for j in range(200):
        beam.gated_gemmrc(x[j], gate, up, x[j + 1], activation="relu")
    torch.cuda.synchronize()
    assert beam.device_status() == (0, 0)
    for j in range(200):  # each call again, alone
        c = torch.empty_like(x[0])
        beam.gated_gemmrc(x[j], gate, up, c, activation="relu")
        torch.cuda.synchronize()
        assert torch.equal(c, x[j + 1]), j
    assert x[200][0, 0] == 1 and 0.5 < x[200].float().norm() / x[0].float().norm() < 2  # nothing has died out on the way
