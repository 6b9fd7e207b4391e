"""Rotary positions: frequencies and refusals on the CPU; the sm_100a kernel
against the formula in 64 bits on the GPU."""

import math

import pytest
import torch

import flash_attention_2_lab_b200 as fa
from flash_attention_2_lab_b200 import _native

gpu = pytest.mark.gpu


def turn(x, positions, frequencies, layout, factor=1.0, inverse=False):
    """The formula in 64 bits, pair by pair as complex numbers."""
    r = 2 * frequencies.numel()
    x = x.double()
    angle = positions.double()[..., None] * frequencies * (-1 if inverse else 1)
    while angle.dim() < 3:
        angle = angle[None]
    unit = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    if layout == "interleaved":
        z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * unit
        head = torch.stack([z.real, z.imag], -1).flatten(-2)
    else:
        z = torch.complex(x[..., : r // 2], x[..., r // 2:r]) * unit
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., r:]], -1)


def bound(ref, x, dtype, factor=1.0):
    """One rounding to the result's type (half a step, or half of the smallest subnormal), and in
    32 bits: the angle's rounding (2 pi 2^-26 of a turn's half), sine and cosine (2 units of 2^-24
    each), factor, product and sum - under 12 steps of 2^-24 of the pair's size."""
    step = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    pair = x.double().abs().amax(-1, keepdim=True) * 2 * factor
    return step * ref.abs() + tiny + 12 * 2.0 ** -24 * pair * (1 + step)


# ------------------------------------------------------------------ frequencies (CPU)

def test_frequencies_plain_and_linear():
    f, factor = fa.rotary_frequencies(64, base=10000.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and factor == 1.0
    for i in (0, 7, 31):
        assert math.isclose(f[i], 10000.0 ** (-2 * i / 64), rel_tol=1e-15)
    g, _ = fa.rotary_frequencies(64, scaling="linear", factor=4.0)
    torch.testing.assert_close(g, f / 4, rtol=1e-15, atol=0)


def test_frequencies_ntk_stretches_the_lowest_pair_only():
    f, _ = fa.rotary_frequencies(64)
    g, factor = fa.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert factor == 1.0
    assert math.isclose(g[0], f[0], rel_tol=1e-15)
    assert math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12)


def test_frequencies_yarn_blends_by_turns():
    trained, factor = 4096, 4.0
    f, _ = fa.rotary_frequencies(128)
    g, mult = fa.rotary_frequencies(128, scaling="yarn", factor=factor, trained_length=trained)
    assert math.isclose(mult, 0.1 * math.log(4) + 1)
    turns = trained * f / (2 * math.pi)
    torch.testing.assert_close(g[turns > 40], f[turns > 40], rtol=1e-15, atol=0)
    torch.testing.assert_close(g[turns < 0.8], f[turns < 0.8] / factor, rtol=1e-15, atol=0)
    assert (g <= f).all() and (g >= f / factor).all()


@pytest.mark.parametrize(("kw", "message"), [
    (dict(rotary_dim=7), "rotary_dim must be even"),
    (dict(rotary_dim=0), "rotary_dim must be even"),
    (dict(rotary_dim=64, scaling="cubic"), "scaling must be one of"),
    (dict(rotary_dim=64, base=1.0), "base must be above 1"),
    (dict(rotary_dim=64, base=float("nan")), "base must be above 1"),
    (dict(rotary_dim=64, factor=0.5), "factor must be at least 1"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "rotary_dim above 2"),
    (dict(rotary_dim=64, scaling="yarn", factor=2.0), "trained_length"),
    (dict(rotary_dim=64, scaling="yarn", trained_length=4096, fast_turns=1.0, slow_turns=2.0),
     "slow_turns must be positive and below"),
])
def test_frequency_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        fa.rotary_frequencies(**kw)


# ------------------------------------------------------------------ refusals (CPU)

def _args(**change):
    a = dict(query=torch.zeros(2, 4, 5, 64, dtype=torch.float16),
             key=torch.zeros(2, 2, 5, 64, dtype=torch.float16), positions=torch.arange(5),
             frequencies=torch.ones(32, dtype=torch.float64))
    a.update(change)
    return a


@pytest.mark.parametrize(("change", "message"), [
    (dict(query=torch.zeros(4, 5, 64)), r"query must have shape \[B, H, N, D\]"),
    (dict(query=torch.zeros(2, 4, 5, 64, dtype=torch.float64)), "query must have dtype"),
    (dict(query=torch.zeros(2, 4, 64, 5, dtype=torch.float16).transpose(2, 3)), "dense rows"),
    (dict(key=torch.zeros(2, 2, 6, 64, dtype=torch.float16)), "agree in batch, tokens"),
    (dict(key=torch.zeros(2, 2, 5, 32, dtype=torch.float16)), "agree in batch, tokens"),
    (dict(key=torch.zeros(2, 2, 5, 64)), "same dtype"),
    (dict(positions=torch.arange(4)), r"positions must have shape"),
    (dict(positions=torch.zeros(5)), "positions must have dtype int32 or int64"),
    (dict(positions=torch.zeros(1, 5, dtype=torch.int32)), "positions must have shape"),
    (dict(frequencies=torch.ones(32)), "float64"),
    (dict(frequencies=torch.ones(64, dtype=torch.float64)[::2]), "contiguous"),
    (dict(frequencies=torch.ones(33, dtype=torch.float64)), "1 to D / 2"),
    (dict(frequencies=torch.ones(0, dtype=torch.float64)), "1 to D / 2"),
    (dict(), "query must be a CUDA tensor"),
])
def test_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        fa.apply_rotary(**_args(**change))


@pytest.mark.parametrize("wants_gradient", [False, True])
@pytest.mark.parametrize("side", ["query", "key"])
def test_forward_mode_is_refused(side, wants_gradient):
    """A tangent is not dropped."""
    args = _args()
    with torch.autograd.forward_ad.dual_level():
        x = args[side].clone().requires_grad_(wants_gradient)
        args[side] = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward mode"):
            fa.apply_rotary(**args)


def test_unknown_layout_refused():
    with pytest.raises(ValueError, match="layout must be one of"):
        fa.apply_rotary(**_args(), layout="thirds")


def test_c_entry_refuses_without_gpu():
    import ctypes

    lib = _native.lib()
    side = (ctypes.c_int64 * 6)(4096, 8192, 2, 128, 64, 64)  # x, y, heads, strides

    def call(query=ctypes.addressof(side), bits=64, batch=1, tokens=1, dim=64, rotary=64, dtype=0,
             positions=4096, frequencies=4096):
        return lib.fa_rotary_sm100(query, None, positions, bits, 0, 1, frequencies, batch, tokens,
                                   dim, rotary, 0, dtype, 1.0, 0, None)

    for kw, message in [(dict(query=None), "null"), (dict(bits=16), "32 or 64"),
                        (dict(batch=-1), "negative"), (dict(rotary=63), "rotary dimension"),
                        (dict(rotary=66), "rotary dimension"), (dict(dtype=7), "element type"),
                        (dict(positions=None), "null"), (dict(frequencies=None), "null"),
                        (dict(tokens=1 << 31), "too large")]:
        assert call(**kw) == -1, kw
        assert message in _native.last_error(), kw
    assert call(batch=0) == 0
    side[0] = 4097
    assert call() == -1 and "aligned" in _native.last_error()


# ------------------------------------------------------------------ values (GPU)

CASES = [  # batch, heads, kv heads, tokens, dim, rotary dim
    (1, 1, 1, 1, 64, 64),
    (3, 8, 2, 1, 64, 32),
    (2, 4, 4, 129, 64, 64),
    (1, 7, 1, 33, 128, 48),
    (2, 3, 2, 17, 80, 80),
    (1, 2, 1, 5, 66, 34),    # rows not a multiple of 16 bytes: one element at a time
    (2, 2, 2, 9, 7, 2),      # an odd head dimension
    (1, 1, 1, 3, 2, 2),
    (4, 32, 8, 200, 64, 64),
    (1, 0, 3, 4, 64, 64),    # no query heads
]


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", CASES)
def test_matches_formula(shape, dtype, layout):
    b, h, hk, n, d, r = shape
    g = torch.Generator().manual_seed(n * 100 + d)
    q = torch.randn(b, h, n, d, generator=g).to(dtype).cuda()
    k = torch.randn(b, hk, n, d, generator=g).to(dtype).cuda()
    positions = torch.randint(-5, 1 << 20, (b, n), generator=g).cuda()
    f, factor = fa.rotary_frequencies(r, scaling="yarn", factor=4.0, trained_length=4096,
                                      device="cuda")
    out = fa.apply_rotary(q, k, positions, f, layout=layout, attention_factor=factor)
    for x, y in zip((q, k), out):
        assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
        ref = turn(x, positions, f, layout, factor)
        if x.numel():
            assert ((y.double() - ref).abs() <= bound(ref, x, dtype, factor)).all()
        assert torch.equal(y[..., r:], x[..., r:])


@gpu
@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
@pytest.mark.parametrize("where", [0, (1 << 31) - 100, -(1 << 31)])
def test_far_positions_keep_their_angle(bits, where):
    x = torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    f, _ = fa.rotary_frequencies(64, device="cuda")
    positions = (torch.arange(64) + where).to(bits).cuda()
    y, none = fa.apply_rotary(x, None, positions, f)
    assert none is None
    ref = turn(x, positions, f, "half")
    # 2^31 positions: turns below 2^29 in 53 bits leave 2^-25 of a turn, 1.9e-7 rad
    assert ((y.double() - ref).abs() <= bound(ref, x, torch.float32) + 4e-7 * x.abs().amax()).all()


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides(layout):
    """Rows of a fused projection [B, N, H, D], a slice of wider heads at an odd offset, an
    expanded batch, expanded positions."""
    g = torch.Generator().manual_seed(4)
    f, _ = fa.rotary_frequencies(32, device="cuda")
    qkv = torch.randn(2, 19, 12, 64, generator=g).half().cuda()
    odd = torch.randn(2, 3, 19, 131, generator=g).half().cuda()[..., 1:65]
    same = torch.randn(1, 3, 19, 64, generator=g).half().cuda().expand(2, 3, 19, 64)
    positions = torch.arange(19).cuda()
    for q, k in ((qkv[:, :, :8].transpose(1, 2), qkv[:, :, 8:].transpose(1, 2)), (odd, same)):
        for pos in (positions, positions.expand(2, 19), positions.repeat_interleave(2)[::2]):
            for x, y in zip((q, k), fa.apply_rotary(q, k, pos, f, layout=layout)):
                ref = turn(x, positions, f, layout)
                assert ((y.double() - ref).abs() <= bound(ref, x, torch.float16)).all()


@gpu
def test_rows_of_infinities_stay_in_their_row():
    f, _ = fa.rotary_frequencies(64, device="cuda")
    x = torch.randn(1, 2, 9, 64, generator=torch.Generator().manual_seed(2)).half().cuda()
    clean, _ = fa.apply_rotary(x, None, torch.arange(9).cuda(), f)
    x[0, 1, 4] = float("nan")
    got, _ = fa.apply_rotary(x, None, torch.arange(9).cuda(), f)
    keep = torch.ones(1, 2, 9, dtype=torch.bool, device="cuda")
    keep[0, 1, 4] = False
    assert torch.equal(got[keep], clean[keep]) and got[0, 1, 4].isnan().all()


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradients(layout):
    g = torch.Generator().manual_seed(3)
    f, _ = fa.rotary_frequencies(48, device="cuda")
    positions = torch.randint(0, 9000, (2, 21), generator=g).cuda()
    q, k = (torch.randn(2, h, 21, 64, generator=g).half().cuda().requires_grad_() for h in (4, 2))
    gq, gk = (torch.randn(2, h, 21, 64, generator=g).half().cuda() for h in (4, 2))
    out = fa.apply_rotary(q, k, positions, f, layout=layout, attention_factor=1.25)
    for got, x in zip(torch.autograd.grad(out, (q, k), (gq, gk)), (gq, gk)):
        ref = turn(x, positions, f, layout, 1.25, inverse=True)
        assert ((got.double() - ref).abs() <= bound(ref, x, torch.float16, 1.25)).all()
    # one side alone; a gradient with no strides of its own; only one side wants a gradient
    out = fa.apply_rotary(q, k, positions, f, layout=layout)
    (only,) = torch.autograd.grad(out[1].sum(), k)
    one = torch.ones_like(k)
    ref = turn(one, positions, f, layout, inverse=True)
    assert ((only.double() - ref).abs() <= bound(ref, one, torch.float16)).all()
    out = fa.apply_rotary(q.detach(), k, positions, f, layout=layout)
    assert out[1].requires_grad and not out[0].requires_grad


@gpu
def test_gradients_against_differences():
    """Central differences in fp32: the map is linear, so they carry only roundings."""
    g = torch.Generator().manual_seed(5)
    f, _ = fa.rotary_frequencies(6, device="cuda")
    positions = torch.arange(3).cuda()
    x = torch.randn(1, 1, 3, 8, generator=g).cuda().requires_grad_()
    w = torch.randn(1, 1, 3, 8, generator=g).cuda()

    def value(x):
        return (fa.apply_rotary(x, None, positions, f, attention_factor=1.5)[0].double() * w).sum()

    (grad,) = torch.autograd.grad(value(x), x, create_graph=True)
    for i in range(24):
        e = torch.zeros(24).cuda()
        e[i] = 0.5
        with torch.no_grad():
            step = (value(x + e.view_as(x)) - value(x - e.view_as(x))).item()
        # 2 x 24 terms, each rounded to 2^-24 of at most 1.5 * sqrt(2) * (|x| + 1/2)
        assert abs(step - grad.flatten()[i].item()) < 2e-5
    # twice differentiable: the gradient is linear in w, its own backward turns forward
    v = torch.randn_like(grad)
    wv = w.clone().requires_grad_()
    (again,) = torch.autograd.grad(
        (fa.apply_rotary(x, None, positions, f)[0] * wv).sum(), x, create_graph=True)
    (back,) = torch.autograd.grad((again * v).sum(), wv)
    ref = turn(v, positions, f, "half")
    assert ((back.double() - ref).abs() <= bound(ref, v, torch.float32)).all()


@gpu
def test_streams_and_graph():
    f, _ = fa.rotary_frequencies(64, device="cuda")
    x = torch.randn(2, 4, 50, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    positions = torch.arange(50).cuda()
    expected, _ = fa.apply_rotary(x, None, positions, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = fa.apply_rotary(x, None, positions, f)
    side.synchronize()
    assert torch.equal(y, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z, _ = fa.apply_rotary(x, None, positions, f)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, -expected)


@gpu
def test_captured_backward():
    f, _ = fa.rotary_frequencies(64, device="cuda")
    g = torch.Generator().manual_seed(7)
    x, w = (torch.randn(2, 4, 50, 64, generator=g).half().cuda() for _ in range(2))
    positions = torch.arange(50).cuda()
    expected, _ = fa.apply_rotary(w, None, positions, f, inverse=True)
    x.requires_grad_()
    side = torch.cuda.Stream()

    def step():
        (grad,) = torch.autograd.grad(fa.apply_rotary(x, None, positions, f)[0], x, w)
        return grad

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step()
    w.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, -expected)

    # an eager graph holds the gradient node of x on the default stream
    eager, _ = fa.apply_rotary(x, None, positions, f)
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="captured backward pass"):
            step()
    (back,) = torch.autograd.grad(eager, x, w)
    assert torch.equal(back, -expected)
    del eager, back
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        grad = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, -expected)


@gpu
@pytest.mark.parametrize("layers", [1, 3])
def test_captured_backward_beside_a_graph_of_another_stream(layers):
    """An eager graph of a side stream holds the leaf's gradient node, as data-parallel wrappers do:
    that stream joins the capture."""
    f, _ = fa.rotary_frequencies(64, device="cuda")
    g = torch.Generator().manual_seed(9)
    x, w = (torch.randn(2, 4, 50, 64, generator=g).half().cuda() for _ in range(2))
    positions = torch.arange(50).cuda()
    x.requires_grad_()

    def forward():
        y = x
        for _ in range(layers):
            y = fa.apply_rotary(y, None, positions, f)[0]
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = forward()
        (want,) = torch.autograd.grad(forward(), x, w)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        (grad,) = torch.autograd.grad(forward(), x, w)
    w.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, -want)
    x.grad = None
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        forward().backward(w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, -want)
    with torch.cuda.stream(side):  # the stream is an ordinary one again, and the graph is whole
        (back,) = torch.autograd.grad(held, x, w)
    side.synchronize()
    assert torch.equal(back, -want)


@gpu
def test_captured_backward_passes_by_what_it_was_not_asked_for():
    """The gradient node of a factor belongs to an eager graph of the default stream; a captured pass
    that was asked for the other factor's gradient does not reach it."""
    f, _ = fa.rotary_frequencies(64, device="cuda")
    g = torch.Generator().manual_seed(10)
    x, y, w = (torch.randn(2, 4, 50, 64, generator=g).half().cuda() for _ in range(3))
    positions = torch.arange(50).cuda()
    want = fa.apply_rotary(w, None, positions, f, inverse=True)[0] * y
    x.requires_grad_()
    y.requires_grad_()
    held = fa.apply_rotary(y, None, positions, f)[0]
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        (grad,) = torch.autograd.grad(fa.apply_rotary(x * y, None, positions, f)[0], x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, want)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="captured backward pass"):
            torch.autograd.grad(fa.apply_rotary(x * y, None, positions, f)[0], (x, y), w)
    assert held.requires_grad


@gpu
def test_offsets_past_32_bits():
    f, _ = fa.rotary_frequencies(64, device="cuda")
    tokens = (1 << 25) + 70  # two heads of 64: more than 2^32 elements
    x = torch.empty(1, 2, tokens, 64, dtype=torch.float16, device="cuda")
    some = torch.randn(1, 2, 50, 64, generator=torch.Generator().manual_seed(8)).half().cuda()
    x[:, :, -50:] = some
    positions = torch.arange(tokens, device="cuda")
    far, _ = fa.apply_rotary(x, None, positions, f)
    near, _ = fa.apply_rotary(some, None, positions[-50:], f)
    assert torch.equal(far[:, :, -50:], near)
