"""The int8 linear layers (launch_linear, launch_expert_linear, quantize_rows,
launch_route, launch_combine) against their formulas in 64 bits.

Tolerances, derived before the first run: the int32 sums are exact; what
follows takes at most eight roundings of 2^-24 on magnitudes up to
|sum| * scales + |bias| (and its exponentials are good to 2^-21), so with the
activations' slopes below 1.13 a value before its last rounding is off by less
than 2^-19 of that magnitude; the last rounding adds half a unit of the output's
type.  A code may differ from the exact one only where 127 x / a lies within
127 * 2^-22 of a half (three roundings of 2^-24 on a quotient up to 127).
"""
import ctypes
import math

import pytest
import torch

import int8_kernel_lab_amd as lab
from int8_kernel_lab_amd import _lib
from tests.conftest import say

DTYPES = {"int8": torch.int8, "bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}
HALF_UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
SMALLEST = {"bf16": 2.0 ** -130, "fp16": 2.0 ** -25, "fp32": 2.0 ** -130}
FAKE = 0x10000  # an aligned address that is never dereferenced


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def _strided(x, stride):
    """x in memory with `stride` elements between rows, NaN (or 77) between them."""
    if not stride:
        return x.contiguous()
    wide = torch.full((x.shape[0], stride), 77 if x.dtype == torch.int8 else math.nan,
                      device="cuda", dtype=x.dtype)
    wide[:, :x.shape[1]] = x
    return wide


def _ws(nbytes):
    """A workspace of exactly nbytes, poisoned."""
    return torch.full((max(nbytes, 1),), 0xA5, device="cuda", dtype=torch.uint8)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def quantized(x, stride=0):
    """(codes, scales) of quantize_rows, which has tests of its own below."""
    rows, k = x.shape
    name = {v: n for n, v in DTYPES.items()}[x.dtype]
    mem = _strided(x, stride)
    codes = torch.full((rows, k), 55, device="cuda", dtype=torch.int8)
    scales = torch.full((rows,), -1.0, device="cuda")
    lab.quantize_rows(_p(mem), name, rows, k, _p(codes), _p(scales), stride, _stream())
    return codes, scales


def _act(v, name):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def expected(codes, scales, w, ws, bias, act, gated, residual):
    """(values, magnitudes that the tolerance is taken of), in 64 bits."""
    sums = torch.matmul(codes.double(), w.double().t().contiguous())
    v = sums * scales.double()[:, None] * ws.double()
    mag = v.abs()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    if gated:
        n = v.shape[1] // 2
        a = _act(v[:, :n], act)
        mag = mag[:, :n] * v[:, n:].abs() + a.abs() * mag[:, n:]
        v = a * v[:, n:]
    else:
        v = _act(v, act)
    if residual is not None:
        v, mag = v + residual.double(), mag + residual.double().abs()
    return v, mag


def assert_close(y, ref, mag, kind):
    tol = ref.abs() * HALF_UNIT[kind] + mag * 2.0 ** -19 + SMALLEST[kind]
    got = y.double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    bad = ((got - ref).abs() > tol) & ~nan
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(),
                           got[bad][:4].tolist(), ref[bad][:4].tolist())


def run_linear(rows, k, n, x="bf16", y="bf16", act="none", gated=False, bias=False, residual=False,
               strides=(0, 0, 0), offset=0, in_place=False, seed=1, data=None):
    """One dense layer on seeded data, checked; returns its output."""
    say(f"[gpu] linear {rows}x{k}->{n} {x}->{y} {act} gated={gated} bias={bias} "
        f"residual={residual} strides={strides} offset={offset}")
    g = _gen(seed)
    wide = 2 * n if gated else n
    w = _codes(g, wide, k)
    ws = torch.exp(0.3 * _normal(g, wide)) * 2e-4
    b = _normal(g, wide) if bias else None
    r = _normal(g, rows, n).to(DTYPES[y]) if residual else None
    if x == "int8":
        values = _codes(g, rows, k)
        scales = torch.exp(0.3 * _normal(g, rows)) * 0.02
        codes, xs = values, scales
    else:
        values = (data if data is not None else 3 * _normal(g, rows, k)).to(DTYPES[x])
        codes, scales, xs = *quantized(values), None
    mem = _strided(values, strides[0])
    out_ld = strides[1] or n
    # `offset` elements before the first one: an address of its own alignment
    store = torch.full((rows * out_ld + offset + 8,), 9.0, device="cuda", dtype=DTYPES[y])
    out = store[offset:offset + rows * out_ld].view(rows, out_ld)
    res = None
    if residual:
        res = _strided(r, strides[2])
        if in_place:
            out[:, :n] = r
            res = out
    shape = lab.LinearShape(rows, k, n, x, y, act, gated, input_stride=strides[0],
                            output_stride=strides[1], residual_stride=strides[2])
    need = lab.linear_workspace_bytes(shape)
    work = _ws(need)
    lab.launch_linear(shape, _p(mem), _p(xs), _p(w), _p(ws), _p(b), _p(res), _p(out),
                      _p(work) if need else None, need, _stream())
    ref, mag = expected(codes, scales, w, ws, b, act, gated, r)
    assert_close(out[:, :n], ref, mag, y)
    # nothing beside the rows was written
    if strides[1]:
        assert (out[:, n:] == 9.0).all()
    assert (store[:offset] == 9.0).all() and (store[offset + rows * out_ld:] == 9.0).all()
    return out[:, :n].clone()


# ---- quantize_rows -----------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k,stride", [(1, 16, 0), (3, 48, 49), (17, 2000, 0), (5, 4096, 4104),
                                           (2, 16400, 0), (1025, 128, 0), (1, 131056, 0)])
def test_quantize_rows(kind, rows, k, stride):
    say(f"[gpu] quantize {rows}x{k} {kind} stride {stride}")
    x = (_normal(_gen(3), rows, k) * 5).to(DTYPES[kind])
    codes, scales = quantized(x, stride)
    d = x.double()
    top = d.abs().amax(dim=1, keepdim=True)
    exact = d * 127 / top
    assert ((scales.double() - top[:, 0] / 127).abs() <= top[:, 0] / 127 * 2.0 ** -24).all()
    off = codes.double() != torch.round(exact)
    near = (exact - torch.floor(exact) - 0.5).abs() <= 127 * 2.0 ** -22
    assert not (off & ~near).any()
    # values of few bits have their half steps exactly: those go to even
    if kind != "fp32":
        assert not (off & (exact - torch.floor(exact) == 0.5)).any()
    assert codes.abs().max() <= 127


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_quantize_rows_extremes(kind):
    dtype = DTYPES[kind]
    biggest, smallest = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros((8, 32), device="cuda", dtype=dtype)
    x[1, 5] = math.inf
    x[2, 31] = math.nan
    x[3, :] = biggest
    x[3, 1] = -biggest
    x[4, 0], x[4, 1] = smallest, -smallest  # of bf16 and fp32: below 2^-100
    x[5, :] = 1.0
    x[5, 7] = -2.0
    x[6, 3] = -0.0
    x[7, 0], x[7, 1], x[7, 2] = biggest, biggest / 2, -biggest / 4
    codes, scales = quantized(x)
    codes, scales = codes.cpu(), scales.cpu()
    for row in (0, 6):
        assert (codes[row] == 0).all() and scales[row] == 0
    for row in (1, 2):
        assert (codes[row] == 0).all() and math.isnan(scales[row])
    assert codes[3].tolist() == [127, -127] + [127] * 30
    if kind == "fp16":
        assert codes[4, :3].tolist() == [127, -127, 0]
    else:
        assert (codes[4] == 0).all() and scales[4] == 0
    assert codes[5].tolist() == [64] * 7 + [-127] + [64] * 24  # 63.5 to even
    assert codes[7, :4].tolist() == [127, 64, -32, 0]
    assert scales[7] == torch.tensor(biggest, dtype=torch.float32) / 127


# ---- dense layers ------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [
    (1, 16, 1), (1, 4096, 4096), (1, 1040, 523), (2, 128, 64), (7, 2000, 1003), (16, 512, 320),
    (17, 144, 130), (31, 1024, 36), (33, 1024, 256), (48, 2064, 999), (64, 4096, 128),
    (65, 640, 515), (100, 128, 2049), (128, 256, 128), (129, 272, 257), (255, 128, 384),
    (300, 1008, 1000), (513, 2048, 512), (1000, 112, 77), (2049, 256, 1024)])
def test_linear_sizes(rows, k, n):
    run_linear(rows, k, n, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 256, 100), (5, 1024, 64), (20, 2048, 1031), (40, 400, 96),
                                      (130, 384, 200), (700, 512, 520)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_linear_gated(rows, k, n, act):
    run_linear(rows, k, n, act=act, gated=True, bias=act != "relu", residual=act == "gelu", y="fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["int8", "bf16", "fp16", "fp32"])
@pytest.mark.parametrize("y", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [1, 9, 60, 333])
def test_linear_types(x, y, rows):
    run_linear(rows, 528, 260, x=x, y=y, act="silu", bias=True, residual=True)
    run_linear(rows, 528, 261, x=x, y=y, gated=True, residual=True)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 200])
def test_linear_activations_over_their_range(act, rows):
    # a bias that runs from -200 to 200 drives the activations to both limits
    n, k = 512, 64
    w = _codes(_gen(1), n, k)
    ws = torch.full((n,), 1e-4, device="cuda")
    b = torch.linspace(-200, 200, n, device="cuda")
    x = _codes(_gen(2), rows, k)
    xs = torch.full((rows,), 0.01, device="cuda")
    y = torch.empty((rows, n), device="cuda")
    shape = lab.LinearShape(rows, k, n, "int8", "fp32", act)
    say(f"[gpu] linear {act} over -200 .. 200, {rows} rows")
    lab.launch_linear(shape, _p(x), _p(xs), _p(w), _p(ws), _p(b), None, _p(y), None, 0, _stream())
    ref, mag = expected(x, xs, w, ws, b, act, False, None)
    assert_close(y, ref, mag, "fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 200])
def test_linear_activations_at_their_limits(act, rows):
    # sums of -0.26 .. 0.26 beside these biases round away
    n, k = 128, 16
    biases = torch.tensor([math.inf, 3e38, -3e38, 1e20, -1e20], device="cuda")
    ref = biases.clone() if act == "none" else biases.clamp(min=0)
    at = torch.arange(n, device="cuda") % 5
    w, x = _codes(_gen(1), n, k), _codes(_gen(2), rows, k)
    ws, xs = torch.full((n,), 1e-3, device="cuda"), torch.full((rows,), 1e-3, device="cuda")
    b, y = biases[at].contiguous(), torch.empty((rows, n), device="cuda")
    shape = lab.LinearShape(rows, k, n, "int8", "fp32", act)
    say(f"[gpu] linear {act} at its limits, {rows} rows")
    lab.launch_linear(shape, _p(x), _p(xs), _p(w), _p(ws), _p(b), None, _p(y), None, 0, _stream())
    ref = ref[at].expand(rows, n)
    infinite = torch.isinf(ref)
    assert torch.equal(y[infinite], ref[infinite])
    assert ((y - ref).abs() <= ref.abs() * 2.0 ** -20)[~infinite].all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 12, 77, 260])
@pytest.mark.parametrize("strides,offset", [((0, 0, 0), 1), ((0, 0, 0), 3), ((544, 300, 320), 0),
                                            ((544, 301, 303), 0), ((544, 512, 260), 2)])
def test_linear_strides_and_alignment(rows, strides, offset):
    for x in ("bf16", "int8", "fp32"):
        run_linear(rows, 528, 260, x=x, y="fp16", residual=True, strides=strides, offset=offset)
    run_linear(rows, 528, 259, x="fp16", y="bf16", residual=True, gated=True,
               strides=(545, 303, 0), offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_linear_residual_in_place(rows):
    run_linear(rows, 256, 192, residual=True, in_place=True)
    run_linear(rows, 256, 131, residual=True, in_place=True, y="fp32", gated=True)
    run_linear(rows, 256, 128, residual=True, in_place=True, strides=(0, 200, 200))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 40, 140])
def test_linear_largest_sums(rows):
    # every product at its largest: the sums reach 128 * 128 * 131056 < 2^31
    k, n = 131056, 40
    x = torch.full((rows, k), -128, device="cuda", dtype=torch.int8)
    w = torch.full((n, k), -128, device="cuda", dtype=torch.int8)
    w[1::2] = 127
    xs = torch.ones(rows, device="cuda")
    ws = torch.ones(n, device="cuda")
    y = torch.empty((rows, n), device="cuda")
    shape = lab.LinearShape(rows, k, n, "int8", "fp32")
    say(f"[gpu] largest sums, {rows} rows")
    lab.launch_linear(shape, _p(x), _p(xs), _p(w), _p(ws), None, None, _p(y), None, 0, _stream())
    row = torch.tensor([128 * 128 * k, -128 * 127 * k] * (n // 2), device="cuda").float()
    assert torch.equal(y, row.expand(rows, n))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 6, 50, 200])
def test_linear_rows_that_are_zero_or_not_finite(rows):
    x = _normal(_gen(4), rows, 320)
    x[0] = 0
    if rows > 4:
        x[2, 17] = math.inf
        x[3, 300] = math.nan
    out = run_linear(rows, 320, 100, bias=True, data=x)
    if rows > 4:
        assert torch.isnan(out[2:4]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[rows - 1]).all()


@pytest.mark.gpu
def test_linear_output_past_32_bits():
    # 2^31 output elements and more: 70000 rows of 32000 values
    rows, k, n = 70000, 32, 32000
    g = _gen(6)
    x, w = _codes(g, rows, k), _codes(g, n, k)
    xs = torch.exp(0.3 * _normal(g, rows)) * 0.02
    ws = torch.exp(0.3 * _normal(g, n)) * 0.02
    y = torch.zeros((rows, n), device="cuda", dtype=torch.bfloat16)
    shape = lab.LinearShape(rows, k, n, "int8", "bf16")
    say("[gpu] linear with 2.24e9 outputs")
    lab.launch_linear(shape, _p(x), _p(xs), _p(w), _p(ws), None, None, _p(y), None, 0, _stream())
    for at in (0, 33000, 67100, 67108, 69990):
        part = slice(at, at + 10)
        ref, mag = expected(x[part], xs[part], w, ws, None, "none", False, None)
        assert_close(y[part], ref, mag, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 48, 128])
def test_linear_is_repeatable_and_follows_its_stream(rows):
    g = _gen(7)
    k, n = 4096, 1000
    x, w = _normal(g, rows, k).to(torch.bfloat16), _codes(g, n, k)
    ws = torch.exp(0.3 * _normal(g, n)) * 2e-4
    shape = lab.LinearShape(rows, k, n)
    need = lab.linear_workspace_bytes(shape)
    work = _ws(need)
    y = torch.empty((rows, n), device="cuda", dtype=torch.bfloat16)

    def launch(inp, out):
        lab.launch_linear(shape, _p(inp), None, _p(w), _p(ws), None, None, _p(out), _p(work), need,
                          _stream())

    launch(x, y)
    torch.cuda.synchronize()
    want = y.clone()
    # on another stream, behind work of that stream that makes its input
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        twice = x.clone()
        for _ in range(20):
            twice = (twice * 2).mul_(0.5)
        launch(twice, y.zero_())
    side.synchronize()
    assert torch.equal(y, want)
    # in a graph, replayed with eager work between
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(x, y)
    for _ in range(4):
        y.zero_()
        work.fill_(0x5A)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        launch(x, y.zero_())
        torch.cuda.synchronize()
        assert torch.equal(y, want)


# ---- layers of experts --------------------------------------------------------

def route_reference(ids, experts):
    flat = ids.reshape(-1).tolist()
    order = [i for e in range(experts) for i, v in enumerate(flat) if v == e]
    offsets = [sum(0 <= v < e for v in flat) for e in range(experts + 1)]
    places = [-1] * len(flat)
    for row, i in enumerate(order):
        places[i] = row
    sources = [i // ids.shape[1] for i in order] + [-1] * (len(flat) - len(order))
    return offsets, sources, places


def routed(ids, experts):
    tokens, choices = ids.shape
    offsets = torch.full((experts + 1,), -7, device="cuda", dtype=torch.int32)
    sources = torch.full((tokens * choices,), -7, device="cuda", dtype=torch.int32)
    places = torch.full((tokens, choices), -7, device="cuda", dtype=torch.int32)
    shape = lab.RouteShape(tokens, choices, experts)
    need = lab.route_workspace_bytes(shape)
    work = _ws(need)
    lab.launch_route(shape, _p(ids), _p(offsets), _p(sources), _p(places),
                     _p(work) if need else None, need, _stream())
    return offsets, sources, places


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,choices,experts,dropped", [
    (1, 1, 1, 0), (1, 8, 64, 0), (7, 3, 5, 0), (63, 1, 2, 0.3), (64, 2, 4096, 0), (500, 4, 60, 0.2),
    (1025, 8, 128, 0), (3000, 5, 257, 0.05), (20000, 7, 33, 0.01), (9, 2, 3, 1.0), (0, 2, 3, 0)])
def test_route(tokens, choices, experts, dropped):
    say(f"[gpu] route {tokens}x{choices} of {experts}, dropped {dropped}")
    g = _gen(8)
    ids = torch.randint(0, experts, (tokens, choices), generator=g, device="cuda", dtype=torch.int32)
    gone = torch.rand((tokens, choices), generator=g, device="cuda") < dropped
    bad = torch.tensor([-1, experts, -2 ** 31, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    pick = torch.randint(0, 4, (tokens, choices), generator=g, device="cuda")
    ids = torch.where(gone, bad[pick], ids).contiguous()
    offsets, sources, places = routed(ids, experts)
    want = route_reference(ids.cpu(), experts) if tokens <= 3000 else None
    if want is None:  # the same by torch's stable sort
        flat = ids.reshape(-1).long()
        key = torch.where((flat >= 0) & (flat < experts), flat, experts)
        order = torch.argsort(key, stable=True)
        live = int((key < experts).sum())
        at = torch.empty_like(order)
        at[order] = torch.arange(order.numel(), device="cuda")
        want = ([int((key < e).sum()) for e in range(experts + 1)],
                (order // choices)[:live].tolist() + [-1] * (order.numel() - live),
                torch.where(key < experts, at, -1).tolist())
    assert offsets.tolist() == want[0]
    assert sources.tolist() == want[1]
    assert places.reshape(-1).tolist() == want[2]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,choices,experts,dropped", [
    (16383, 1, 1024, 0.05), (16384, 1, 1024, 0), (16385, 1, 257, 0.4), (4097, 4, 2, 0), (5000, 7, 1000, 1.0),
    (4100, 4, 1025, 0.1), (300000, 2, 37, 0.02)])
def test_route_around_two_launches(tokens, choices, experts, dropped):
    test_route(tokens, choices, experts, dropped)


def run_experts(counts, k, n, x="bf16", y="bf16", act="none", gated=False, bias=False, tokens=None,
                spare=0, seed=9, strides=(0, 0), offset=0):
    """Rows of `counts` per expert; gathered from `tokens` rows, or in place."""
    say(f"[gpu] experts {counts if len(counts) < 20 else len(counts)} {k}->{n} {x}->{y} {act} "
        f"gated={gated} bias={bias} tokens={tokens} spare={spare}")
    g = _gen(seed)
    experts, total = len(counts), sum(counts)
    rows = total + spare
    wide = 2 * n if gated else n
    w = _codes(g, experts, wide, k)
    ws = torch.exp(0.3 * _normal(g, experts, wide)) * 2e-4
    b = _normal(g, experts, wide) if bias else None
    offsets = torch.tensor([sum(counts[:e]) for e in range(experts + 1)], device="cuda",
                           dtype=torch.int32)
    x_rows = rows if tokens is None else tokens
    if x == "int8":
        values = _codes(g, x_rows, k)
        scales = torch.exp(0.3 * _normal(g, x_rows)) * 0.02
        codes, xs = values, scales
    else:
        values = (3 * _normal(g, x_rows, k)).to(DTYPES[x])
        codes, scales, xs = *quantized(values), None
    sources = None
    if tokens is not None:
        sources = torch.randint(0, tokens, (rows,), generator=g, device="cuda", dtype=torch.int32)
        sources[total:] = -1
    mem = _strided(values, strides[0])
    ld = strides[1] or n
    store = torch.full((rows * ld + offset + 8,), 9.0, device="cuda", dtype=DTYPES[y])
    out = store[offset:offset + rows * ld].view(rows, ld)
    shape = lab.LinearShape(x_rows, k, n, x, y, act, gated, experts=experts, routed=rows,
                            input_stride=strides[0], output_stride=strides[1])
    need = lab.linear_workspace_bytes(shape)
    work = _ws(need)
    lab.launch_expert_linear(shape, _p(mem), _p(xs), _p(w), _p(ws), _p(b), _p(offsets),
                             _p(sources), _p(out), _p(work) if need else None, need, _stream())
    at = 0
    for e, count in enumerate(counts):
        if count:
            index = torch.arange(at, at + count, device="cuda") if sources is None else \
                sources[at:at + count].long()
            ref, mag = expected(codes[index], scales[index], w[e], ws[e],
                                None if b is None else b[e], act, gated, None)
            assert_close(out[at:at + count, :n], ref, mag, y)
        at += count
    assert (out[total:] == 9.0).all() and (out[:, n:] == 9.0).all()
    assert (store[:offset] == 9.0).all() and (store[offset + rows * ld:] == 9.0).all()


COUNTS = [[1], [0, 0, 3], [5, 0, 0, 1, 0], [1] * 8, [17, 130, 0, 64, 1], [300, 2, 129, 0, 0, 33],
          [0] * 30 + [40] + [0] * 33, [3, 1, 0, 2] * 40, [1000, 7], [0, 0, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("gated", [False, True])
def test_experts_groups(counts, gated):
    run_experts(counts, 272, 200, gated=gated, act="silu", bias=True, tokens=37)
    run_experts(counts, 1024, 133, gated=gated, y="fp32", spare=21)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [
    [0, 250, 0, 1] + [0] * 80, [64, 65, 1, 63] + [0] * 90, [0] * 70 + [128, 129] + [0] * 30,
    [1] * 64 + [66, 0, 67] + [0] * 50, [0] * 99 + [300]], ids=lambda c: f"{len(c)}-{max(c)}")
@pytest.mark.parametrize("gated", [False, True])
def test_experts_few_rows_of_which_one_has_most(counts, gated):
    # at most 3 rows per expert in the mean: the few-row kernel, whose
    # workgroups share an expert's rows where there are many
    run_experts(counts, 272, 100, gated=gated, act="silu", bias=True, tokens=37)
    run_experts(counts, 1024, 33, gated=gated, y="fp32", spare=2)


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["int8", "bf16", "fp16", "fp32"])
@pytest.mark.parametrize("y", ["bf16", "fp16", "fp32"])
def test_experts_types(x, y):
    run_experts([3, 0, 70, 1], 144, 68, x=x, y=y, act="relu", bias=True, tokens=50)
    run_experts([3, 0, 70, 1], 144, 68, x=x, y=y, gated=True, act="gelu", spare=3)
    run_experts([2, 1, 0, 9], 144, 67, x=x, y=y, strides=(160, 75), offset=1)


@pytest.mark.gpu
def test_experts_of_most_experts():
    run_experts([e % 2 for e in range(4096)], 16, 24, tokens=10)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[4] * 4096, [e % 9 for e in range(2050)]], ids=["4096", "2050"])
def test_experts_of_many_experts_in_tiles(counts):
    run_experts(counts, 32, 24, tokens=100, y="fp32")
    run_experts(counts, 32, 24, tokens=100, gated=True, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [1, 3, 63, 65, 129, 255])
@pytest.mark.parametrize("rows", [40, 500, 3000])
def test_linear_last_channel_alone(odd, rows):
    # odd channel counts in every tile: the last one leaves by itself
    for y in ("bf16", "fp32"):
        run_linear(rows, 144, odd, y=y, residual=True, strides=(0, odd + 2, odd + 4))
        run_linear(rows, 144, odd, y=y, residual=True, gated=True, offset=1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,choices", [(1, 4), (3, 2), (90, 4), (5000, 4)])
def test_layer_of_experts_replays_from_a_graph(tokens, choices):
    # the chain captured once, replayed on other tokens and choices with eager
    # passes between: the same bytes as eager each time
    say(f"[gpu] graph of a layer of experts, {tokens} tokens of {choices}")
    k, n, experts, rows = 144, 80, 16, tokens * choices
    g = _gen(12)
    w1, w2 = _codes(g, experts, 2 * n, k), _codes(g, experts, k, n)
    s1 = torch.full((experts, 2 * n), 2e-3, device="cuda")
    s2 = torch.full((experts, k), 2e-3, device="cuda")
    x = torch.zeros(tokens, k, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(tokens, choices, device="cuda", dtype=torch.int32)
    weights = torch.zeros(tokens, choices, device="cuda")
    up = lab.LinearShape(tokens, k, n, "bf16", "bf16", gated=True, activation="silu", experts=experts, routed=rows)
    down = lab.LinearShape(rows, n, k, "bf16", "bf16", experts=experts, routed=rows)
    route, combine = lab.RouteShape(tokens, choices, experts), lab.CombineShape(tokens, choices, k)
    need = max(lab.linear_workspace_bytes(up), lab.linear_workspace_bytes(down),
               lab.route_workspace_bytes(route))

    def buffers():
        return dict(o=torch.zeros(experts + 1, device="cuda", dtype=torch.int32),
                    s=torch.zeros(rows, device="cuda", dtype=torch.int32),
                    p=torch.zeros(rows, device="cuda", dtype=torch.int32),
                    h=torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16),
                    z=torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16),
                    y=torch.zeros(tokens, k, device="cuda", dtype=torch.bfloat16), w=_ws(max(need, 1)))

    def run(b):
        st = _stream()
        lab.launch_route(route, _p(ids), _p(b["o"]), _p(b["s"]), _p(b["p"]), _p(b["w"]), need, st)
        lab.launch_expert_linear(up, _p(x), None, _p(w1), _p(s1), None, _p(b["o"]), _p(b["s"]), _p(b["h"]),
                                 _p(b["w"]), need, st)
        lab.launch_expert_linear(down, _p(b["h"]), None, _p(w2), _p(s2), None, _p(b["o"]), None, _p(b["z"]),
                                 _p(b["w"]), need, st)
        lab.launch_combine(combine, _p(b["z"]), _p(b["p"]), _p(weights), _p(x), _p(b["y"]), st)

    eager, captured = buffers(), buffers()
    run(captured)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(captured)
    for turn in range(4):
        x.copy_(_normal(g, tokens, k))
        ids.copy_(torch.randint(-1, experts, (tokens, choices), generator=g, device="cuda"))
        weights.copy_(_normal(g, tokens, choices))
        graph.replay()
        torch.cuda.synchronize()
        run(eager)
        torch.cuda.synchronize()
        assert torch.equal(eager["y"], captured["y"]), turn
        assert eager["y"].float().isfinite().all() and not torch.equal(eager["y"], x)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("n", [514, 515, 1024])
@pytest.mark.parametrize("rows", [700, 2500, 9000])
def test_linear_both_epilogues(rows, n, act):
    # whole and partial column tiles, with and without a last channel alone,
    # several tiles in turn to a workgroup
    run_linear(rows, 144, n, y="fp16", act=act, bias=True, residual=True, strides=(0, n + 6, n + 2))
    run_linear(rows, 144, n, act=act, gated=True, residual=n % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [130, 131, 768])
def test_experts_both_epilogues(n):
    counts = [300, 0, 5, 257, 1, 600, 256, 90]
    run_experts(counts, 144, n, tokens=400, act="silu", gated=True)
    run_experts(counts, 144, n, tokens=400, bias=True, y="fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("last", [3, 50, 300])
def test_experts_weights_past_32_bits(last):
    # 36 matrices of 2^27 bytes: the last begin past 2^32, in each kernel
    run_experts([2] + [0] * 34 + [last], 8192, 16384, tokens=20)


@pytest.mark.gpu
def test_combine_rows_past_32_bits():
    tokens, choices, n = 40000, 8, 8192  # 2.6e9 values
    say("[gpu] combine of 2.6e9 values")
    g = _gen(13)
    rows = tokens * choices
    v = torch.empty((rows, n), device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    places = torch.randperm(rows, generator=g, device="cuda").to(torch.int32).view(tokens, choices)
    weights = torch.rand((tokens, choices), generator=g, device="cuda")
    out = torch.empty((tokens, n), device="cuda", dtype=torch.bfloat16)
    lab.launch_combine(lab.CombineShape(tokens, choices, n), _p(v), _p(places), _p(weights), None,
                       _p(out), _stream())
    for part in (slice(0, 50), slice(tokens - 50, tokens)):
        terms = v[places[part].long()].double() * weights[part][..., None].double()
        assert_close(out[part], terms.sum(1), terms.abs().sum(1), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("experts,choices", [(0, 0), (8, 2)])
@pytest.mark.parametrize("tokens", [1, 37])
def test_feed_forward_example(experts, choices, tokens, capsys):
    from int8_kernel_lab_amd import feed_forward
    say(f"[gpu] feed forward, {tokens} tokens, {experts} experts")
    assert feed_forward.main(["--tokens", str(tokens), "--width", "256", "--hidden", "400",
                              "--experts", str(experts), "--choices", str(max(1, choices)),
                              "--iterations", "2"]) == 0
    assert '"relative_error"' in capsys.readouterr().out


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 90])
def test_experts_sources_outside_read_as_zeros(rows):
    say(f"[gpu] sources outside, {rows} rows")
    g = _gen(11)
    k, n = 256, 64
    x, w = _codes(g, 5, k), _codes(g, 1, n, k)
    xs, ws = torch.ones(5, device="cuda"), torch.ones((1, n), device="cuda")
    b = _normal(g, 1, n)
    sources = torch.tensor([0, -1, 5, 2 ** 31 - 1] * (rows // 4) + [4] * (rows % 4), device="cuda",
                           dtype=torch.int32)
    offsets = torch.tensor([0, rows], device="cuda", dtype=torch.int32)
    y = torch.empty((rows, n), device="cuda")
    shape = lab.LinearShape(5, k, n, "int8", "fp32", experts=1, routed=rows)
    lab.launch_expert_linear(shape, _p(x), _p(xs), _p(w), _p(ws), _p(b), _p(offsets), _p(sources),
                             _p(y), None, 0, _stream())
    ok = (sources >= 0) & (sources < 5)
    ref, mag = expected(torch.where(ok[:, None], x[sources.clamp(0, 4).long()], torch.zeros_like(x[:1])),
                        torch.ones(rows, device="cuda"), w[0], ws[0], b[0], "none", False, None)
    assert_close(y, ref, mag, "fp32")


# ---- combine --------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("x,y", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp16"),
                                 ("fp32", "fp32"), ("bf16", "fp16")])
@pytest.mark.parametrize("tokens,choices,n", [(1, 1, 1), (1, 8, 2048), (5, 3, 1003), (64, 2, 4100),
                                              (700, 6, 96), (33, 9, 7)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(x, y, tokens, choices, n, residual):
    say(f"[gpu] combine {tokens}x{choices} of {n}, {x} -> {y}, residual {residual}")
    g = _gen(12)
    rows = tokens * choices
    v = _normal(g, rows, n).to(DTYPES[x])
    places = torch.randperm(rows, generator=g, device="cuda").to(torch.int32).view(tokens, choices)
    places = torch.where(torch.rand((tokens, choices), generator=g, device="cuda") < 0.2, -1, places)
    places[tokens // 2] = -1  # a token without rows
    places[0, 0] = rows       # outside
    places = places.contiguous()
    weights = torch.rand((tokens, choices), generator=g, device="cuda")
    r = _normal(g, tokens, n).to(DTYPES[y]) if residual else None
    for in_place in ((False, True) if residual else (False,)):
        out = r.clone() if in_place else torch.full((tokens, n), 9.0, device="cuda", dtype=DTYPES[y])
        lab.launch_combine(lab.CombineShape(tokens, choices, n, x, y), _p(v), _p(places),
                           _p(weights), _p(out if in_place else r), _p(out), _stream())
        live = ((places >= 0) & (places < rows))[..., None]
        terms = torch.where(live, v[places.clamp(0, rows - 1).long()].double(), 0.0) * \
            weights[..., None].double()
        ref, mag = terms.sum(1), terms.abs().sum(1)
        if residual:
            ref, mag = ref + r.double(), mag + r.double().abs()
        assert_close(out, ref, mag, y)


@pytest.mark.gpu
def test_combine_leaves_out_what_it_does_not_read():
    # a dropped choice's row may hold anything, and so may a weight that belongs to none
    v = torch.full((4, 40), math.nan, device="cuda", dtype=torch.float16)
    v[2] = 1.5
    places = torch.tensor([[2, -1], [-1, -1]], device="cuda", dtype=torch.int32)
    weights = torch.tensor([[2.0, math.nan], [math.inf, math.nan]], device="cuda")
    out = torch.full((2, 40), 9.0, device="cuda")
    lab.launch_combine(lab.CombineShape(2, 2, 40, "fp16", "fp32"), _p(v), _p(places), _p(weights),
                       None, _p(out), _stream())
    assert (out[0] == 3.0).all() and (out[1] == 0.0).all()


# ---- refusals (no launch: these run without a GPU) --------------------------------

def _linear_rc(shape, **over):
    a = dict(input=FAKE, input_scale=None, weight=FAKE, weight_scale=FAKE, bias=None, residual=None,
             output=FAKE, workspace=FAKE, nbytes=1 << 30, stream=None)
    a.update(over)
    return _lib.lib().i8conv_launch_linear(ctypes.byref(shape.c_struct()), *a.values())


def _expert_rc(shape, **over):
    a = dict(input=FAKE, input_scale=None, weight=FAKE, weight_scale=FAKE, bias=None, offsets=FAKE,
             sources=FAKE, output=FAKE, workspace=FAKE, nbytes=1 << 30, stream=None)
    a.update(over)
    return _lib.lib().i8conv_launch_expert_linear(ctypes.byref(shape.c_struct()), *a.values())


@pytest.mark.parametrize("change,reason", [
    (dict(rows=-1), "rows"), (dict(inputs=0), "multiple of 16"), (dict(inputs=24), "multiple of 16"),
    (dict(inputs=1 << 17), "below 2^17"), (dict(outputs=0), "outputs"),
    (dict(output_type="int8"), "output"), (dict(experts=-1), "experts"),
    (dict(experts=4097, routed=1), "experts"), (dict(routed=3), "routed"),
    (dict(inputs=65536, outputs=32768), "2^31"), (dict(outputs=16384, inputs=65536, gated=True), "2^31"),
    (dict(input_stride=63), "stride"), (dict(output_stride=32), "stride"),
    (dict(residual_stride=32), "stride"), (dict(input_type="int8", input_stride=72), "multiple of 16"),
    (dict(input_type="int8", input_stride=1 << 23), "2^23")])
def test_bad_linear_shapes_are_refused(change, reason):
    shape = lab.LinearShape(**{**dict(rows=4, inputs=64, outputs=33), **change})
    assert _linear_rc(shape) == _lib.BAD_SHAPE
    assert reason in _lib.lib().i8conv_last_error().decode()
    assert lab.linear_workspace_bytes(shape) == 0


def test_bad_enums_are_refused():
    for field, value in (("input_type", 4), ("input_type", -1), ("output_type", 7),
                         ("activation", 5), ("activation", -1), ("gated", 2)):
        c = lab.LinearShape(4, 64, 32).c_struct()
        setattr(c, field, value)
        rc = _lib.lib().i8conv_launch_linear(ctypes.byref(c), *[FAKE] * 8, 1 << 30, None)
        assert rc == _lib.BAD_SHAPE, field
    for bad in (dict(input_type="int4"), dict(output_type="half"), dict(activation="tanh")):
        with pytest.raises(ValueError):
            lab.LinearShape(4, 64, 32, **bad).c_struct()


@pytest.mark.parametrize("over", [
    dict(input=None), dict(weight=None), dict(weight_scale=None), dict(output=None),
    dict(input_scale=FAKE), dict(weight=FAKE + 8), dict(input=FAKE + 1), dict(output=FAKE + 1),
    dict(residual=FAKE + 1), dict(bias=FAKE + 2), dict(weight_scale=FAKE + 2)])
def test_bad_linear_arguments_are_refused(over):
    assert _linear_rc(lab.LinearShape(4, 64, 32), **over) == _lib.BAD_ARGUMENT
    assert _lib.lib().i8conv_last_error()


def test_int8_inputs_need_their_scales():
    shape = lab.LinearShape(4, 64, 32, "int8")
    assert _linear_rc(shape) == _lib.BAD_ARGUMENT
    assert _linear_rc(shape, input_scale=FAKE, input=FAKE + 8) == _lib.BAD_ARGUMENT


def test_linear_workspace_is_asked_for():
    shape = lab.LinearShape(400, 640, 320)
    need = lab.linear_workspace_bytes(shape)
    assert need >= 400 * 640 + 4 * 400
    for over in (dict(nbytes=need - 1), dict(workspace=None), dict(workspace=FAKE + 64, nbytes=need)):
        assert _linear_rc(shape, **over) == _lib.WORKSPACE_TOO_SMALL
        assert str(need) in _lib.lib().i8conv_last_error().decode()
    with pytest.raises(lab.I8ConvError):
        lab.launch_linear(shape, FAKE, None, FAKE, FAKE, None, None, FAKE, FAKE, need - 1)


def test_experts_and_dense_layers_are_told_apart():
    assert _linear_rc(lab.LinearShape(4, 64, 32, experts=2, routed=8)) == _lib.BAD_SHAPE
    assert _expert_rc(lab.LinearShape(4, 64, 32)) == _lib.BAD_SHAPE
    layer = lab.LinearShape(4, 64, 32, experts=2, routed=8)
    assert _expert_rc(layer, sources=None) == _lib.BAD_SHAPE  # 8 rows of 4
    assert _expert_rc(layer, offsets=None) == _lib.BAD_ARGUMENT
    assert _expert_rc(layer, offsets=FAKE + 2) == _lib.BAD_ARGUMENT
    assert _expert_rc(layer, sources=FAKE + 2) == _lib.BAD_ARGUMENT
    assert _expert_rc(lab.LinearShape(1 << 20, 2048, 32, experts=2, routed=8)) == _lib.BAD_SHAPE


def test_nothing_to_do_is_no_error():
    assert _linear_rc(lab.LinearShape(0, 64, 32), input=None) == _lib.OK
    assert _expert_rc(lab.LinearShape(4, 64, 32, experts=2, routed=0), input=None) == _lib.OK
    assert _lib.lib().i8conv_quantize_rows(None, 1, 0, 64, 0, None, None, None) == _lib.OK
    c = lab.CombineShape(0, 2, 8).c_struct()
    assert _lib.lib().i8conv_launch_combine(ctypes.byref(c), *[None] * 6) == _lib.OK


@pytest.mark.parametrize("args", [
    (FAKE, 0, 4, 64, 0, FAKE, FAKE), (FAKE, 9, 4, 64, 0, FAKE, FAKE), (FAKE, 1, -1, 64, 0, FAKE, FAKE),
    (FAKE, 1, 4, 60, 0, FAKE, FAKE), (FAKE, 1, 4, 64, 63, FAKE, FAKE), (None, 1, 4, 64, 0, FAKE, FAKE),
    (FAKE, 1, 4, 64, 0, None, FAKE), (FAKE, 1, 4, 64, 0, FAKE, None), (FAKE + 1, 1, 4, 64, 0, FAKE, FAKE),
    (FAKE, 1, 4, 64, 0, FAKE + 8, FAKE), (FAKE, 1, 4, 64, 0, FAKE, FAKE + 2)])
def test_bad_quantize_arguments_are_refused(args):
    assert _lib.lib().i8conv_quantize_rows(*args, None) == _lib.BAD_ARGUMENT


def test_bad_route_and_combine_arguments_are_refused():
    def route(shape, *tensors, nbytes=1 << 30):
        return _lib.lib().i8conv_launch_route(ctypes.byref(shape.c_struct()), *tensors, nbytes, None)

    for bad in (lab.RouteShape(-1, 2, 4), lab.RouteShape(4, 0, 4), lab.RouteShape(4, 2, 0),
                lab.RouteShape(4, 2, 4097), lab.RouteShape(1 << 30, 2, 4)):
        assert route(bad, *[FAKE] * 5) == _lib.BAD_SHAPE
    good = lab.RouteShape(4, 2, 4)
    for i in range(4):
        tensors = [FAKE] * 5
        tensors[i] = None
        assert route(good, *tensors) == _lib.BAD_ARGUMENT
        tensors[i] = FAKE + 2
        assert route(good, *tensors) == _lib.BAD_ARGUMENT

    def combine(shape, *tensors):
        return _lib.lib().i8conv_launch_combine(ctypes.byref(shape.c_struct()), *tensors, None)

    for bad in (lab.CombineShape(-1, 2, 4), lab.CombineShape(4, 0, 4), lab.CombineShape(4, 2, 0),
                lab.CombineShape(4, 2, 4, "int8"), lab.CombineShape(4, 2, 4, "bf16", "int8"),
                lab.CombineShape(1 << 30, 2, 4)):
        assert combine(bad, *[FAKE] * 5) == _lib.BAD_SHAPE
    good = lab.CombineShape(4, 2, 4)
    for i, spoilt in ((0, None), (1, None), (2, None), (4, None), (0, FAKE + 1), (1, FAKE + 2),
                      (2, FAKE + 2), (3, FAKE + 1), (4, FAKE + 1)):
        tensors = [FAKE] * 5
        tensors[i] = spoilt
        assert combine(good, *tensors) == _lib.BAD_ARGUMENT, i


def test_sizes_beyond_the_limits_are_refused():
    for shape, reason in ((lab.LinearShape(1 << 29, 64, 32), "2^29"),
                          (lab.LinearShape(1 << 24, 16, 1 << 15), "2^39"),
                          (lab.LinearShape(4, 16, 1 << 24), "2^24"),
                          (lab.LinearShape(4, 64, 32, output_stride=1 << 24), "2^24")):
        assert _linear_rc(shape) == _lib.BAD_SHAPE
        assert reason in _lib.lib().i8conv_last_error().decode()
    wide = lab.CombineShape(4, 2, 1 << 24).c_struct()
    assert _lib.lib().i8conv_launch_combine(ctypes.byref(wide), *[FAKE] * 5, None) == _lib.BAD_SHAPE
    assert _lib.lib().i8conv_quantize_rows(FAKE, 1, 4, 1 << 24, 0, FAKE, FAKE, None) == _lib.BAD_ARGUMENT


def test_sizes_beyond_32_bits_are_refused():
    big = 2 ** 32 + 16  # 16 in a 32-bit field
    for shape in (lab.LinearShape(big, 16, 16), lab.LinearShape(16, big, 16),
                  lab.LinearShape(16, 16, big), lab.LinearShape(16, 16, 16, experts=1, routed=big),
                  lab.LinearShape(16, 16, 16, experts=big)):
        with pytest.raises(ValueError, match="32 bits"):
            lab.linear_workspace_bytes(shape)
    for shape in (lab.RouteShape(big, 1, 1), lab.RouteShape(1, big, 1), lab.RouteShape(1, 1, big)):
        with pytest.raises(ValueError, match="32 bits"):
            lab.route_workspace_bytes(shape)
    for shape in (lab.CombineShape(big, 1, 1), lab.CombineShape(1, big, 1),
                  lab.CombineShape(1, 1, big)):
        with pytest.raises(ValueError, match="32 bits"):
            lab.launch_combine(shape, FAKE, FAKE, FAKE, None, FAKE)
    for rows, inputs in ((big, 16), (16, big)):
        with pytest.raises(ValueError, match="32 bits"):
            lab.quantize_rows(FAKE, "bf16", rows, inputs, FAKE, FAKE)


def test_route_workspace_is_asked_for():
    shape = lab.RouteShape(40000, 8, 128)
    need = lab.route_workspace_bytes(shape)
    assert need > 0 and lab.route_workspace_bytes(lab.RouteShape(8, 8, 128)) == 0
    for workspace, nbytes in ((None, need), (FAKE, need - 1), (FAKE + 128, need)):
        rc = _lib.lib().i8conv_launch_route(ctypes.byref(shape.c_struct()), FAKE, FAKE, FAKE, FAKE,
                                            workspace, nbytes, None)
        assert rc == _lib.WORKSPACE_TOO_SMALL
        assert str(need) in _lib.lib().i8conv_last_error().decode()


def test_linear_plans_are_described():
    assert "few rows" in lab.describe_linear(lab.LinearShape(1, 4096, 4096))
    assert "quantize rows" not in lab.describe_linear(lab.LinearShape(500, 4096, 4096, "int8"))
    assert lab.describe_linear(lab.LinearShape(16384, 8192, 8192)).endswith("256 rows x 256")
    for rows in (33, 200, 1000, 5000):
        for gated in (False, True):
            for experts in (0, 64, 4096):
                shape = lab.LinearShape(rows, 1024, 1000, gated=gated, experts=experts,
                                        routed=rows * 4 if experts else 0)
                assert "?" not in lab.describe_linear(shape)
    with pytest.raises(lab.I8ConvError):
        lab.describe_linear(lab.LinearShape(4, 24, 8))
    buf = ctypes.create_string_buffer(4)
    c = lab.LinearShape(1, 64, 64).c_struct()
    assert _lib.lib().i8conv_linear_describe(ctypes.byref(c), buf, 4) == _lib.OK
    assert len(buf.value) == 3  # cut, and ended
    assert _lib.lib().i8conv_linear_describe(ctypes.byref(c), None, 4) == _lib.BAD_ARGUMENT


def test_linear_shapes_are_values():
    import pickle
    shape = lab.LinearShape(7, 64, 33, experts=4, routed=14)
    shape._c_ref()
    assert pickle.loads(pickle.dumps(shape)) == shape
    assert (shape.weight_rows, shape.ops()) == (33, 2 * 14 * 33 * 64)
    assert lab.LinearShape(7, 64, 33, gated=True).weight_rows == 66


def test_feed_forward_reference_is_the_formula():
    # the example's own numbers on the CPU: one token, one expert, by hand
    from int8_kernel_lab_amd import feed_forward
    import numpy as np
    codes, scale = feed_forward.quantize(np.array([[0.5, -1.0, 0.25, 0.0], [0, 0, 0, 0]]))
    assert codes.tolist() == [[64, -127, 32, 0], [0, 0, 0, 0]]  # 63.5 to even
    assert scale[1, 0] == 0 and scale[0, 0] == 1 / 127
