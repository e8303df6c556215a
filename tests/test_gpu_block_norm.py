"""Block norm against its definition in 64 bits."""

import ctypes
import math

import pytest
import torch

import decoder_reference as ref
from cim22_b200 import abi, cim_ops, native
from cim22_b200.cim_ops import Norm, block_norm

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gate_rows(gate, rows, dim):
    g = gate.double().reshape(-1, gate.shape[-1])
    return g.repeat_interleave(rows // g.shape[0], dim=0).expand(rows, dim)


def expected(x, residual, post, pre, gate, act, scale):
    """(h, y) in 64 bits and, for the tolerances, each row's largest term."""
    rows, dim = x.shape
    h = x.double()
    if post:
        h = ref.norm(h, post.kind, post.weight, post.bias, post.eps)
    reach = h.abs().amax(-1, keepdim=True)
    if post and post.kind == "layer":
        # (v - mean) may cancel: its terms are as large as v itself.
        spread = (x.double() - x.double().mean(-1, keepdim=True)).pow(2).mean(-1, keepdim=True)
        weight = post.weight.double().abs().max() if post.weight is not None else 1.0
        reach = reach + weight * x.double().abs().amax(-1, keepdim=True) / (spread + post.eps).sqrt()
    if post and post.bias is not None:
        reach = reach + post.bias.double().abs().max()
    if gate is not None:
        g = gate_rows(gate, rows, dim)
        g = {None: g, "sigmoid": torch.sigmoid(g), "tanh": torch.tanh(g)}[act]
        h = h * g
        reach = reach * g.abs().amax(-1, keepdim=True)
    if residual is not None:
        h = h + scale * residual.double()
        reach = reach + abs(scale) * residual.double().abs().amax(-1, keepdim=True)
    y = y_reach = None
    if pre:
        y = ref.norm(h, pre.kind, pre.weight, pre.bias, pre.eps)
        centre = h - h.mean(-1, keepdim=True) if pre.kind == "layer" else h
        power = centre.pow(2).mean(-1, keepdim=True)
        weight = pre.weight.double().abs().max() if pre.weight is not None else 1.0
        bias = pre.bias.double().abs().max() if pre.bias is not None else 0.0
        y_reach = weight * reach / (power + pre.eps).sqrt() + bias + y.abs().amax(-1, keepdim=True)
    return h, y, reach, y_reach


def check(got, want, reach, dtype):
    """Half a step of the result's type, and 64 roundings of 2^-24 (a row sum
    takes at most 32 terms a thread and 10 shuffles, then a handful of
    operations) of the largest term."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 64 * 2.0 ** -24 * reach
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # subnormal steps
    off = (got.double().cpu() - want.cpu()).abs()
    assert bool((off <= tol.cpu()).all()), float((off / tol.cpu()).max())


def make(rows, dim, dtype, seed=0, stride=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn(rows, stride or dim, generator=g, device="cuda") * 2 + 0.5
    return wide.to(dtype)[:, :dim]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (2, 16), (5, 255), (1, 1000), (4, 1001),
                                      (9, 1024), (2, 4096), (1, 5119), (3, 8192), (2, 16383),
                                      (2, 16384)])
@pytest.mark.parametrize("post,pre,gate,act", [
    ("rms", "rms", "channel", None), ("layer", "layer", "full", "sigmoid"),
    (None, "layer", "row", "tanh"), ("layer", None, None, None), ("rms", "layer", "group", None)])
def test_block_norm(dtype, rows, dim, post, pre, gate, act):
    x, residual = make(rows, dim, dtype, 1), make(rows, dim, dtype, 2)
    wtype = dtype if dim % 2 else torch.float32

    def norm(kind, seed):
        w, b = make(2, dim, torch.float32, seed)
        return Norm(kind, w.to(wtype), b.to(wtype) if kind == "layer" else None, 1e-5) \
            if kind else None

    post, pre = norm(post, 3), norm(pre, 4)
    g = {None: None, "channel": lambda: make(1, dim, torch.float32, 5)[0],
         "full": lambda: make(rows, dim, dtype, 5), "row": lambda: make(rows, 1, dtype, 5),
         "group": lambda: make(rows if rows % 2 else 2, dim, dtype, 5)}[gate]
    g = g() if g else None
    h, y = block_norm(x, residual, post=post, pre=pre, gate=g, gate_activation=act,
                      residual_scale=0.75)
    wh, wy, reach, y_reach = expected(x, residual, post, pre, g, act, 0.75)
    check(h, wh, reach, dtype)
    if pre:
        check(y, wy, y_reach, dtype)
    else:
        assert y is None


def test_norm_alone_and_residual_alone():
    x = make(5, 300, torch.float32)
    h, y = block_norm(x, pre=Norm("rms"))
    assert h is None
    _, wy, _, reach = expected(x, None, None, Norm("rms"), None, None, 1.0)
    check(y, wy, reach, torch.float32)
    r = make(5, 300, torch.float32, 3)
    h, y = block_norm(x, r)
    assert y is None and torch.equal(h, x + r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,base", [(64, 0), (67, 0), (67, 3), (72, 5)])
def test_strided_rows_and_odd_bases(dtype, stride, base):
    rows, dim = 6, 61
    flat = make(1, rows * stride + 8, dtype, 7)[0]
    x = flat.as_strided((rows, dim), (stride, 1), base)
    residual = make(rows, dim, dtype, 8)
    out = torch.full((rows, dim + 3), 7.0, dtype=dtype, device="cuda")
    normed = torch.full((rows, dim + 5), 7.0, dtype=dtype, device="cuda")
    pre = Norm("layer", make(1, dim, torch.float32, 9)[0])
    block_norm(x, residual, pre=pre, out=out[:, :dim], normed=normed[:, :dim])
    wh, wy, reach, y_reach = expected(x, residual, None, pre, None, None, 1.0)
    check(out[:, :dim], wh, reach, dtype)
    check(normed[:, :dim], wy, y_reach, dtype)
    assert bool((out[:, dim:] == 7).all()) and bool((normed[:, dim:] == 7).all())


def test_in_place_over_the_residual_stream():
    x, residual = make(700, 1536, torch.bfloat16, 1), make(700, 1536, torch.bfloat16, 2)
    want = block_norm(x, residual, post=Norm("rms"), pre=Norm("rms"))
    h, y = block_norm(x, residual, post=Norm("rms"), pre=Norm("rms"), out=residual, normed=x)
    assert h is residual and y is x
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_nan_and_infinity_stay_in_their_rows():
    x = make(4, 128, torch.float32)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    _, y = block_norm(x, pre=Norm("rms"))
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2, 7]))
    assert bool(torch.isfinite(y[[0, 3]]).all())


def test_zero_rows_and_zero_values():
    x = torch.zeros(0, 64, device="cuda")
    h, y = block_norm(x, x, pre=Norm("rms"))
    assert h.shape == y.shape == (0, 64)
    _, y = block_norm(torch.zeros(2, 64, device="cuda"), pre=Norm("layer", eps=1e-6))
    assert bool((y == 0).all())


def test_many_rows_repeat_bit_for_bit():
    x, r = make(40000, 136, torch.float16, 1), make(40000, 136, torch.float16, 2)
    first = block_norm(x, r, post=Norm("layer"), pre=Norm("rms"))
    again = block_norm(x, r, post=Norm("layer"), pre=Norm("rms"))
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    wh, wy, reach, y_reach = expected(x, r, Norm("layer"), Norm("rms"), None, None, 1.0)
    check(first[0], wh, reach, torch.float16)
    check(first[1], wy, y_reach, torch.float16)


def test_batched_shape_and_group_gate():
    x = make(12, 96, torch.float32).view(3, 4, 96)
    gate = make(3, 96, torch.float32, 4)
    h, _ = block_norm(x, x, gate=gate.view(3, 96), pre=Norm("rms"))
    assert h.shape == x.shape
    assert torch.allclose(h, x + x * gate[:, None], rtol=2.0 ** -22, atol=0)


def test_captured_graph_takes_new_contents():
    x, r = make(17, 640, torch.float32, 1), make(17, 640, torch.float32, 2)
    w = make(1, 640, torch.float32, 3)[0]
    block_norm(x, r, pre=Norm("rms", w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y = block_norm(x, r, pre=Norm("rms", w))
    x.copy_(make(17, 640, torch.float32, 9))
    graph.replay()
    want = block_norm(x, r, pre=Norm("rms", w))
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_on_another_stream():
    x = make(64, 512, torch.float32)
    want = block_norm(x, x, pre=Norm("rms"))[1]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = block_norm(x, x, pre=Norm("rms"))[1]
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("call,error", [
    (lambda x: block_norm(x.cpu(), pre=Norm("rms")), TypeError),
    (lambda x: block_norm(x.double(), pre=Norm("rms")), TypeError),
    (lambda x: block_norm(x), ValueError),
    (lambda x: block_norm(x, x[:1], pre=Norm("rms")), TypeError),
    (lambda x: block_norm(x, x.half(), pre=Norm("rms")), TypeError),
    (lambda x: block_norm(x.t(), pre=Norm("rms")), TypeError),
    (lambda x: block_norm(x, pre=Norm("batch")), ValueError),
    (lambda x: block_norm(x, pre=Norm("rms", eps=-1.0)), cim_ops.CudaError),
    (lambda x: block_norm(x, pre=Norm("rms", x[0, :-1])), TypeError),
    (lambda x: block_norm(x, pre=Norm("rms", x[0].half())), TypeError),
    (lambda x: block_norm(x, pre=Norm("rms"), gate=x[:3]), ValueError),
    (lambda x: block_norm(x, pre=Norm("rms"), gate=x[0, :4]), ValueError),
    (lambda x: block_norm(x, pre=Norm("rms"), gate=x[0], gate_activation="relu"), ValueError),
    (lambda x: block_norm(x, x, normed=x), ValueError),
    (lambda x: block_norm(torch.zeros(1, 16385, device="cuda"), pre=Norm("rms")), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call(make(4, 32, torch.float32))


@pytest.mark.parametrize("dim", [64, 61])
@pytest.mark.parametrize("gate_rows", [7, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 62])
def test_a_gate_row_for_more_rows_than_there_are(dim, gate_rows):
    """The C entry takes any count of rows that share a gate row."""
    x, gate = make(7, dim, torch.float32), make(1, dim, torch.float32, 4)
    h = torch.empty_like(x)
    call = abi.BlockNorm(type=abi.FLOAT32, rows=7, dim=dim, x=x.data_ptr(), x_stride=dim,
                         residual=0, residual_stride=0, residual_scale=1.0,
                         gate=gate.data_ptr(), gate_stride=dim, gate_rows=gate_rows,
                         gate_columns=dim, gate_type=abi.FLOAT32, gate_activation=0,
                         h=h.data_ptr(), h_stride=dim, y=0, y_stride=0)
    stream = torch.cuda.current_stream().cuda_stream
    assert native.lib().cim22_cuda_block_norm(ctypes.byref(call), stream) == 0
    assert torch.equal(h, x * gate)


@pytest.mark.parametrize("shape", [(3, 4, 64), (3, 4, 1), (3, 1, 64), (3, 1, 1), (1, 1, 64),
                                   (3, 64)])
def test_gates_of_more_axes(shape):
    x, gate = make(12, 64, torch.float32).view(3, 4, 64), make(12, 64, torch.float32, 4)
    gate = gate.flatten()[:math.prod(shape)].view(shape)
    h, _ = block_norm(x, gate=gate)
    assert torch.equal(h, x * (gate[:, None] if len(shape) == 2 else gate))


@pytest.mark.parametrize("shape", [(1, 4, 64), (1, 4, 1), (4, 3, 64), (3, 4, 1, 64), (2, 6, 64)])
def test_gates_that_are_no_prefix_are_refused(shape):
    x = make(12, 64, torch.float32).view(3, 4, 64)
    with pytest.raises(ValueError, match="gate must be"):
        block_norm(x, gate=torch.ones(shape, device="cuda"))
