"""8-bit linear layer against a 64-bit computation from its definition.

The quantised integers have to be equal. Tolerances of the product: the scale of a row is a / 127 rounded once (2^-24),
converting the integer sum rounds once, each of the two multiplications by a scale rounds once, and both scales are
rounded: 5 * 2^-24 relative before the bias; adding the bias rounds once more (2^-24 of the result), storing to bf16
half a step (finfo.eps / 2).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
MAX_IN = 131056
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    from sparseforge_b200 import ops

    return ops


def _quantise64(x):
    x = x.double()
    a = x.abs().amax(dim=1, keepdim=True)
    q = torch.where(a > 0, 127.0 * x / torch.where(a > 0, a, torch.ones_like(a)), torch.zeros_like(x)).round()
    return q, (a / 127.0).squeeze(1)


def _exact(x, w, bias=None):
    """(y, magnitude before the bias) in 64 bits."""
    xq, xs = _quantise64(x)
    wq, ws = _quantise64(w)
    y = (xq @ wq.t()) * xs[:, None] * ws
    return (y if bias is None else y + bias.double()), y.abs()


def _check(y, want, mag, dtype):
    got = y.double()
    tol = 6 * U * mag + (U + torch.finfo(dtype).eps / 2) * want.abs() + 1e-37
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()), bad.nonzero()[:4].tolist())


def _inputs(T, k, n, dtype, bias=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 131 * T + 7 * k + n)
    x = torch.randn(T, k, device="cuda", generator=g)
    x[:, torch.randint(0, k, (max(1, k // 200),), device="cuda", generator=g)] *= 9.0
    w = torch.randn(n, k, device="cuda", generator=g) * 0.05
    b = (torch.randn(n, device="cuda", generator=g)).to(dtype) if bias else None
    return x.to(dtype), w.to(torch.bfloat16), b


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 3, 8, 15, 16, 17, 64, 255, 1000, 1003, 2048, 4096, 4104, 11008, 16384, 16391, 70001])
def test_quantised_rows(cols, dtype):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(9, cols, device="cuda", generator=g).to(DT[dtype])
    x[3] = 0.0
    x[4] *= 1e-30
    x[5] = (torch.randint(-508, 509, (cols,), device="cuda", generator=g) / 4.0).to(DT[dtype])  # ties, where max is 127
    x[5, 0] = 127.0
    x[5].clamp_(-127.0, 127.0)
    x[6, cols // 2] = 1e20
    q, s = _ops().int8_quantize_rows(x)
    want, scale = _quantise64(x)
    assert q.shape == (9, (cols + 15) // 16 * 16) and q.dtype == torch.int8
    assert torch.equal(q[:, :cols].double(), want)
    assert not q[:, cols:].any()
    assert ((s.double() - scale).abs() <= U * scale).all()
    assert float(s[3]) == 0.0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 23, 247, 248, 249, 1000, 1024, 1025, 2047, 4104, 20000, 32769])
def test_quantised_rows_at_every_alignment(cols, dtype):
    """Rows starting at every element offset from a 16-byte boundary, with guard elements around them; strided so that the
    offset changes from row to row, and in a constant one."""
    ops = _ops()
    for off in range(9):
        for ld in (cols + 3, (cols + 15) // 8 * 8):
            buf = torch.full((off + 11 * ld + 16,), 1e4, device="cuda", dtype=DT[dtype])  # a guard that is read would win the maximum
            x = torch.as_strided(buf, (11, cols), (ld, 1), off)
            x.copy_(torch.randn(11, cols, device="cuda"))
            q, s = ops.int8_quantize_rows(x)
            want, scale = _quantise64(x)
            assert torch.equal(q[:, :cols].double(), want) and not q[:, cols:].any(), (off, ld)
            assert ((s.double() - scale).abs() <= U * scale).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantised_rows_near_and_on_halves(dtype):
    """Quotients exactly half-way go to the even integer; the neighbours of such values go to their own side."""
    rows = []
    for a in (127.0, 254.0, 1.9921875, 0.49609375, 2.0 ** -100 * 127, 2.0 ** 100 * 127, 3.0, 1.4140625):
        a_t = torch.tensor(a, dtype=DT[dtype]).double()
        h = (torch.arange(0, 127, dtype=torch.float64) + 0.5) * a_t / 127.0
        near = torch.cat([h, torch.nextafter(h.float(), torch.tensor(math.inf)).double(),
                          torch.nextafter(h.float(), torch.tensor(-math.inf)).double()]).to(DT[dtype])
        near[-1] = a_t.to(DT[dtype])
        rows.append(near.clamp(max=float(a_t)))
    x = torch.stack(rows).cuda()
    x = torch.cat([x, -x])
    q, _ = _ops().int8_quantize_rows(x)
    want, _ = _quantise64(x)
    assert torch.equal(q[:, :x.shape[1]].double(), want)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("exponent", [0, -60, 100])
def test_every_bf16_quotient(exponent, sign):
    """All significands of a row's largest value against all of an element's, the element up to ten powers of two smaller: every
    quotient a bf16 row can hold that is not zero, on and beside every half. Through the quantiser and the single-row layer."""
    sig = torch.arange(128, 256, dtype=torch.float64, device="cuda")
    gaps = 2.0 ** -torch.arange(0, 11, dtype=torch.float64, device="cuda")
    x = (sig[None, :, None] * gaps).reshape(1, -1).expand(128, -1).clone()
    x = torch.where(x <= sig[:, None], x, torch.zeros_like(x))
    x = (torch.cat([sig[:, None], x], 1) * 2.0 ** (exponent - 8) * sign).bfloat16()
    ops = _ops()
    q, _ = ops.int8_quantize_rows(x)
    want, _ = _quantise64(x)
    assert torch.equal(q[:, :x.shape[1]].double(), want)
    # odd row length: the element-wise kernel
    q, _ = ops.int8_quantize_rows(x[:, :1001])
    assert torch.equal(q[:, :1001].double(), want[:, :1001])
    # weight = identity scaled by one: the layer returns the integers times the scale
    k = x.shape[1]
    eye = torch.eye(k, device="cuda", dtype=torch.int8)
    eye = torch.nn.functional.pad(eye, (0, -k % 16)) if k % 16 else eye
    one = torch.ones(k, device="cuda")
    for r in (0, 1, 63, 126, 127):
        y = ops.int8_linear(x[r:r + 1].float(), eye, one)
        assert torch.equal(torch.round(y.double() / (float(sig[r]) * 2.0 ** (exponent - 8) / 127.0)), want[r:r + 1])
        yb = ops.int8_linear(x[r:r + 1], eye, one)
        assert torch.equal(yb, y.bfloat16())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantised_rows_at_the_ends_of_the_range(dtype):
    top = torch.finfo(DT[dtype]).max
    tiny = 2.0 ** -133 if dtype == "bf16" else 2.0 ** -149
    for a in (top, top / 2, 1e37, 1e-36, 1e-37, 1e-38, 64 * tiny, 3 * tiny, tiny):
        x = (torch.linspace(-1.0, 1.0, 301, dtype=torch.float64) * a).to(DT[dtype]).cuda()[None]
        q, s = _ops().int8_quantize_rows(x)
        want, scale = _quantise64(x)
        assert torch.equal(q[:, :301].double(), want), a
        assert abs(float(s[0]) - float(scale[0])) <= U * float(scale[0]) + 2.0 ** -150


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [3, 6, 200])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_rows_with_infinities(bad, T, dtype):
    """Such a row's result is NaN throughout; the other rows are what they are without it."""
    x, w, b = _inputs(T, 100, 50, DT[dtype], bias=True)
    ops = _ops()
    wq, ws = ops.int8_quantize_rows(w)
    clean = ops.int8_linear(x, wq, ws, b)
    x[1, 99] = bad
    q, s = ops.int8_quantize_rows(x)
    assert math.isnan(float(s[1])) and not q[1].any()
    y = ops.int8_linear(x, wq, ws, b)
    assert torch.isnan(y[1]).all()
    keep = [t for t in range(T) if t != 1]
    assert torch.equal(y[keep], clean[keep])


def test_strided_rows():
    ops = _ops()
    big = torch.randn(40, 300, device="cuda").bfloat16()
    for view in (big[:, :64], big[:, 1:100], big[::2, 3:203], big[5:6, 7:]):
        q, s = ops.int8_quantize_rows(view)
        q2, s2 = ops.int8_quantize_rows(view.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)
        w = torch.randn(33, view.shape[1], device="cuda").bfloat16()
        wq, ws = ops.int8_quantize_rows(w)
        assert torch.equal(ops.int8_linear(view, wq, ws), ops.int8_linear(view.contiguous(), wq, ws))


# ------------------------------------------------------------------------------------------------ product
ROWS = [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 256, 257, 511]
SHAPES = [(16, 1), (1, 7), (100, 130), (128, 128), (256, 264), (500, 1000), (1003, 333), (2048, 96), (4096, 512)]


@pytest.mark.parametrize("dtype,bias", [("bf16", False), ("bf16", True), ("f32", True)])
@pytest.mark.parametrize("T", ROWS)
def test_linear(T, dtype, bias):
    ops = _ops()
    for k, n in SHAPES:
        x, w, b = _inputs(T, k, n, DT[dtype], bias)
        wq, ws = ops.int8_quantize_rows(w)
        y = ops.int8_linear(x, wq, ws, b)
        assert y.shape == (T, n) and y.dtype == x.dtype
        _check(y, *_exact(x, w, b), DT[dtype])
        xq, xs = ops.int8_quantize_rows(x)
        assert torch.equal(y, ops.int8_gemm(xq, xs, wq, ws, b, out_dtype=DT[dtype]))


@pytest.mark.parametrize("T,k,n", [(1, 4096, 4096), (1, 11008, 4096), (3, 4096, 11008), (16, 4096, 11008), (100, 11008, 4096),
                                   (512, 4096, 4096), (1000, 1500, 4096), (2048, 768, 2304), (4096, 4096, 1111)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_at_real_sizes(T, k, n, dtype):
    ops = _ops()
    x, w, b = _inputs(T, k, n, DT[dtype], True, seed=9)
    wq, ws = ops.int8_quantize_rows(w)
    y = ops.int8_linear(x, wq, ws, b)
    _check(y, *_exact(x, w, b), DT[dtype])
    # a row's values do not depend on the rows beside it, whichever kernel the number of rows selects
    for rows in (1, 2, 7, 40, 130, 300):
        if rows < T:
            assert torch.equal(ops.int8_linear(x[:rows], wq, ws, b), y[:rows]), rows
    assert torch.equal(ops.int8_linear(x[T - 1:], wq, ws, b), y[T - 1:])


# every tile shape and every cut of the reduction that the sizes select, ragged in all three directions: tokens x channels
# of 16, 32, 64 columns in 1, 2, 4, 8 parts, two tokens' worth of 64-token tiles, 256 x 256 tiles in 1 and 2 parts, persistent ones
PATHS = [(3, 200, 100), (9, 300, 129), (13, 1000, 4100), (16, 2100, 1000), (20, 129, 40), (29, 5000, 2000), (33, 4200, 300),
         (64, 9000, 500), (70, 4100, 4000), (130, 700, 3000), (190, 11008, 1100), (255, 4109, 1300), (256, 8300, 4111),
         (258, 8200, 700), (300, 9001, 261), (400, 11008, 2500), (513, 8193, 4001), (600, 3001, 1700), (700, 640, 6001),
         (1030, 1601, 5003), (2050, 777, 3001), (5000, 130, 300)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,k,n", PATHS)
def test_every_tile_shape(T, k, n, dtype):
    ops = _ops()
    x, w, b = _inputs(T, k, n, DT[dtype], True, seed=4)
    wq, ws = ops.int8_quantize_rows(w)
    want, mag = _exact(x, w, b)
    xq, xs = ops.int8_quantize_rows(x)
    for rep in range(3):  # parts join in whatever order they finish
        y = ops.int8_linear(x, wq, ws, b)
        _check(y, want, mag, DT[dtype])
        assert torch.equal(y, ops.int8_gemm(xq, xs, wq, ws, b, out_dtype=DT[dtype]))


@pytest.mark.parametrize("T", [1, 4, 9, 40, 300])
def test_extreme_integers(T):
    """-128 and 127 everywhere, at the largest reduction: the 32-bit sum is exact to its end."""
    ops = _ops()
    for k in (144, MAX_IN):
        xq = torch.full((T, k), -128, dtype=torch.int8, device="cuda")
        wq = torch.full((70, k), -128, dtype=torch.int8, device="cuda")
        wq[1] = 127
        wq[2, ::2] = 0
        xs = torch.full((T,), 2.0 ** -10, device="cuda")
        ws = torch.full((70,), 2.0 ** -8, device="cuda")
        y = ops.int8_gemm(xq, xs, wq, ws, out_dtype=torch.float32)
        want = torch.full((70,), 16384.0 * k, dtype=torch.float64)
        want[1] = -128.0 * 127.0 * k
        want[2] = 8192.0 * k
        want = (want * 2.0 ** -18).cuda().expand(T, 70)
        assert ((y.double() - want).abs() <= U * want.abs()).all()


def test_no_rows_and_refusals():
    ops = _ops()
    x, w, b = _inputs(4, 64, 32, torch.bfloat16, True)
    wq, ws = ops.int8_quantize_rows(w)
    assert ops.int8_linear(x[:0], wq, ws).shape == (0, 32)
    assert ops.int8_gemm(*ops.int8_quantize_rows(x[:0]), wq, ws).shape == (0, 32)
    with pytest.raises(ValueError):
        ops.int8_linear(x[:, :40], wq, ws)
    with pytest.raises(TypeError):
        ops.int8_linear(x.half(), wq, ws)
    with pytest.raises(TypeError):
        ops.int8_linear(x[0], wq, ws)
    with pytest.raises(TypeError):
        ops.int8_linear(x, wq.float(), ws)
    with pytest.raises(TypeError):
        ops.int8_linear(x, wq, ws[:-1])
    with pytest.raises(TypeError):
        ops.int8_linear(x, wq, ws, b.float())
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.int8_linear(x.t().contiguous().t(), wq, ws)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.int8_linear(x[:1].expand(4, 64), wq, ws)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.int8_linear(x, wq[:, ::2], ws)
    with pytest.raises(RuntimeError, match="overflow"):
        ops.int8_gemm(torch.zeros(1, MAX_IN + 16, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"),
                      torch.zeros(1, MAX_IN + 16, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.int8_linear(x.cpu(), wq, ws)
    buf = torch.zeros(64 * 32 + 1, dtype=torch.int8, device="cuda")[1:].view(32, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.int8_linear(x, buf, ws)


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_rows_behind_the_last_are_left_alone(T):
    from sparseforge_b200 import _lib

    ops = _ops()
    k, n = 200, 77
    x, w, _ = _inputs(T, k, n, torch.bfloat16)
    wq, ws = ops.int8_quantize_rows(w)
    want = ops.int8_linear(x, wq, ws)
    y = torch.full((T + 2, n), 5.0, device="cuda", dtype=torch.bfloat16)
    work = torch.empty(int(_lib.lib().sf_int8_linear_workspace_bytes(T, k)) or 16, dtype=torch.uint8, device="cuda")
    rc = _lib.lib().sf_int8_linear(x.data_ptr(), k, wq.data_ptr(), ws.data_ptr(), None, y[1:].data_ptr(), _lib.SF_BF16, T, k, n,
                                   work.data_ptr(), None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.equal(y[1:T + 1], want) and (y[0] == 5.0).all() and (y[T + 1] == 5.0).all()


def test_streams_and_graph_replay():
    ops = _ops()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    cases = []
    for T in (1, 7, 100, 400):
        x, w, b = _inputs(T, 1000, 520, torch.bfloat16, True, seed=T)
        wq, ws = ops.int8_quantize_rows(w)
        cases.append((x, wq, ws, b, ops.int8_linear(x, wq, ws, b)))
    torch.cuda.synchronize()
    got = []
    for rep in range(4):
        for i, (x, wq, ws, b, want) in enumerate(cases):
            with torch.cuda.stream((s1, s2)[(i + rep) % 2]):
                got.append((ops.int8_linear(x, wq, ws, b), want))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y, want in got)
    graphs = []
    for x, wq, ws, b, _ in cases:
        ops.int8_linear(x, wq, ws, b)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.int8_linear(x, wq, ws, b)
        graphs.append((g, y))
    for rep in range(3):
        for x, *_ in cases:
            x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        for i, (g, _) in enumerate(graphs):
            with torch.cuda.stream((s1, s2)[i % 2]):
                g.replay()
        torch.cuda.synchronize()
        for (x, wq, ws, b, _), (_, y) in zip(cases, graphs):
            assert torch.equal(y, ops.int8_linear(x, wq, ws, b))


@pytest.mark.parametrize("T,k,n", [(280000, 40, 8000), (270000, 8200, 33), (1, 8192, 270000), (2, 8192, 270000), (20, 8192, 270000),
                                   (64, 8192, 270000)])
def test_offsets_beyond_32_bits(T, k, n):
    """Outputs, inputs or weights of more than 2^31 bytes and elements: the last rows and channels are right."""
    ops = _ops()
    x = torch.randn(T, k, device="cuda", dtype=torch.bfloat16)
    wq = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), device="cuda", dtype=torch.int8)
    wq[:, k:] = 0
    ws = torch.rand(n, device="cuda") * 1e-2
    y = ops.int8_linear(x, wq, ws)
    q, s = _quantise64(x[-3:])
    last = slice(max(0, n - 300), n)
    raw = (q @ wq[last, :k].double().t()) * s[:, None] * ws[last].double()
    _check(y[-3:, last].contiguous(), raw, raw.abs(), torch.bfloat16)
    first = (q[:1] @ wq[:64, :k].double().t()) * s[:1, None] * ws[:64].double()
    _check(y[-3 if T > 2 else -T:, :64][:1].contiguous(), first, first.abs(), torch.bfloat16)


@pytest.mark.parametrize("T", [1, 2, 9, 40, 200, 600])
@pytest.mark.parametrize("captured", [False, True])
def test_operands_written_just_before_the_call(T, captured):
    """Inputs, weights, scales and bias that the work right ahead in the stream (a copy, a fill, a kernel, the
    quantiser, another 8-bit call) has just written are what the call uses, eagerly and in a graph with a fork."""
    ops = _ops()
    k, n = 1024, 1500
    g = torch.Generator(device="cuda").manual_seed(T)
    xs = [torch.randn(T, k, device="cuda", generator=g).bfloat16() for _ in range(4)]
    ws = [ops.int8_quantize_rows(torch.randn(n, k, device="cuda", generator=g).bfloat16()) for _ in range(3)]
    raw = [torch.randn(n, k, device="cuda", generator=g).bfloat16() for _ in range(2)]
    bs = [torch.randn(n, device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = []
    for i in range(4):
        for w in ws + [ops.int8_quantize_rows(r) for r in raw]:
            want.append(ops.int8_linear(xs[i], w[0], w[1], bs[i % 2]))
    torch.cuda.synchronize()
    x, wq, sc, b = torch.empty_like(xs[0]), torch.empty_like(ws[0][0]), torch.empty_like(ws[0][1]), torch.empty_like(bs[0])
    got = [torch.empty_like(want[0]) for _ in want]
    side = torch.cuda.Stream()

    def run():
        j = 0
        for i in range(4):
            for w in ws:
                wq.zero_()
                x.fill_(float("nan"))
                sc.copy_(w[1])
                b.copy_(bs[i % 2])
                x.copy_(xs[i])
                wq.copy_(w[0])
                got[j].copy_(ops.int8_linear(x, wq, sc, b))
                j += 1
            for r in raw:  # the weight comes from the quantiser right ahead, the input from a kernel on another stream
                now = torch.cuda.current_stream()
                side.wait_stream(now)
                with torch.cuda.stream(side):
                    torch.add(xs[i], 0.0, out=x)
                    y_side = ops.int8_linear(x, wq, sc, b)
                q, s = ops.int8_quantize_rows(r)
                now.wait_stream(side)
                got[j].copy_(ops.int8_linear(x, q, s, b))
                assert y_side.shape == got[j].shape
                j += 1

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for _ in range(3):
            for t in got:
                t.zero_()
            graph.replay()
    else:
        for _ in range(3):
            run()
    torch.cuda.synchronize()
    for a, w in zip(got, want):
        assert torch.equal(a, w)


def test_clipping_sees_gradients_written_just_before():
    """Gradients written by the call right ahead (and norms read by the one behind), over and over on one stream."""
    from sparseforge_b200 import ops

    src = [torch.randn(1 << 20, device="cuda").bfloat16() * s for s in (1e-3, 1.0, 30.0)]
    want = []
    for s in src:
        o = torch.empty_like(s)
        want.append((ops.clip_grad_norm([s], 0.5, out=[o]), o))
    g = torch.empty_like(src[0])
    for rep in range(20):
        s, (n, o) = src[rep % 3], want[rep % 3]
        g.copy_(s)
        norm = ops.clip_grad_norm([g], 0.5)
        again = ops.grad_norm([g])
        assert torch.equal(norm, n) and torch.equal(g, o) and torch.equal(again, ops.grad_norm([o]))


def test_status_words_the_device_cannot_write_are_refused():
    ops = _ops()
    x, w, _ = _inputs(4, 64, 32, torch.bfloat16)
    xq, xs = ops.int8_quantize_rows(x)
    wq, ws = ops.int8_quantize_rows(w)
    good = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (good.cpu(), good.float(), good[:0]):
        with pytest.raises((TypeError, RuntimeError)):
            ops.int8_linear(x, wq, ws, status=bad)
        with pytest.raises((TypeError, RuntimeError)):
            ops.int8_gemm(xq, xs, wq, ws, status=bad)
    assert torch.equal(ops.int8_linear(x, wq, ws, status=good), ops.int8_linear(x, wq, ws)) and not good.any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,k,n", [(1, 1000, 70), (2, 1003, 64), (3, 4096, 70), (20, 500, 130), (60, 2000, 130), (300, 640, 200),
                                   (513, 8193, 1700), (2048, 256, 1303)])
def test_rows_at_the_ends_of_the_range_through_the_product(T, k, n, dtype):
    """Finite rows of huge and of tiny values, against channels of all sizes: what fits the result's type comes out right even
    where the sum times one of the scales would not fit fp32.

    Tolerance: that of ``_check`` without its constant, and what the subnormal range adds. A scale below 2^-126 is a
    multiple of 2^-149 (half a step: 2^-150, times the sum and the other scale), and so is a result (2^-150 in fp32, before
    the bias 2^-150 again where the product alone is that small; 2^-134 in bf16)."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(7)
    dt = DT[dtype]
    x = torch.randn(T, k, device="cuda", generator=g).clamp_(-3, 3)
    x[:, 1] = x[:, 0]
    w = torch.randn(n, k, device="cuda", generator=g).clamp_(-3, 3)
    wscale = torch.tensor([1e-3, 1e-30, 1e30, 1e-38, 1e-20, 1e34, 0.0, 1.0], device="cuda")[torch.arange(n, device="cuda") % 8]
    w *= wscale[:, None]
    for j, b in ((9, 1e37), (17, 1.0)):  # channels whose sum is zero for every row
        w[j] = 0.0
        w[j, 0], w[j, 1] = b, -b
    w = w.to(dt)
    bias = torch.randn(n, device="cuda", generator=g).to(dt)
    wq, ws = ops.int8_quantize_rows(w)
    wi, wsc = _quantise64(w)
    top = torch.finfo(dt).max
    # 127 * 2^96 = 1.006e31 is where the scale reaches 2^96
    sizes = [1e36, 1e38, 1e31 / 3, 1.1e31 / 3, 1e20, 1e-37, 1e-40, 1e-20, 1e-3]
    for first in range(0, len(sizes), 1 if T < 9 else len(sizes)):
        rows = torch.tensor([sizes[(first + t) % len(sizes)] for t in range(T)], device="cuda")
        xt = (x.double() * rows.double()[:, None]).clamp(-top, top).to(dt)
        xi, xsc = _quantise64(xt)
        total = xi @ wi.t()
        product = total * xsc[:, None] * wsc
        for b in (None, bias):
            y = ops.int8_linear(xt, wq, ws, b)
            want = product if b is None else product + b.double()
            fits = (want.abs() < top * 0.99) & (product.abs() < torch.finfo(torch.float32).max * 0.99)
            tol = 6 * U * product.abs() + (U + torch.finfo(dt).eps / 2) * want.abs() + 2.0 ** -149
            tol = tol + 2.0 ** -150 * total.abs() * ((xsc < 2.0 ** -126)[:, None] * wsc + (wsc < 2.0 ** -126) * xsc[:, None])
            if dtype == "bf16":
                tol = tol + 2.0 ** -134
            bad = ~((y.double() - want).abs() <= tol) & fits
            assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
            over = want.abs() > top * 1.01
            assert torch.isinf(y[over]).all() and (torch.sign(y[over].double()) == torch.sign(want[over])).all()
            assert not torch.isnan(y).any()
            xq, xs = ops.int8_quantize_rows(xt)
            assert torch.equal(y, ops.int8_gemm(xq, xs, wq, ws, b, out_dtype=dt))


@pytest.mark.parametrize("T", [1, 2, 9, 40, 200, 600])
@pytest.mark.parametrize("captured", [False, True])
def test_values_of_a_forked_call(T, captured):
    """A call on a second stream, right behind the kernel that writes its input there, while weight, scales and bias were
    copied on the first stream ahead of the fork and the quantiser runs beside it: its values, eagerly and in a graph."""
    ops = _ops()
    k, n = 1024, 1500
    g = torch.Generator(device="cuda").manual_seed(T + 1)
    xs = [torch.randn(T, k, device="cuda", generator=g).bfloat16() for _ in range(4)]
    ws = [ops.int8_quantize_rows(torch.randn(n, k, device="cuda", generator=g).bfloat16()) for _ in range(4)]
    raw = torch.randn(n, k, device="cuda", generator=g).bfloat16()
    bs = [torch.randn(n, device="cuda", generator=g).bfloat16() for _ in range(4)]
    want = [ops.int8_linear(xs[i], *ws[i], bs[i]) for i in range(4)]
    beside = [ops.int8_linear(xs[i], *ops.int8_quantize_rows(raw), bs[i]) for i in range(4)]
    torch.cuda.synchronize()
    x, wq, sc, b = torch.empty_like(xs[0]), torch.empty_like(ws[0][0]), torch.empty_like(ws[0][1]), torch.empty_like(bs[0])
    got, got_beside = [torch.empty_like(y) for y in want], [torch.empty_like(y) for y in want]
    side = torch.cuda.Stream()

    def run():
        now = torch.cuda.current_stream()
        for i in range(4):
            x.fill_(float("nan"))
            sc.copy_(ws[i][1])
            b.copy_(bs[i])
            wq.copy_(ws[i][0])
            side.wait_stream(now)
            with torch.cuda.stream(side):
                torch.add(xs[i], 0.0, out=x)
                got[i].copy_(ops.int8_linear(x, wq, sc, b))
            q, s = ops.int8_quantize_rows(raw)
            now.wait_stream(side)
            got_beside[i].copy_(ops.int8_linear(x, q, s, b))

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(3):
        for t in got + got_beside:
            t.zero_()
        graph.replay() if captured else run()
        torch.cuda.synchronize()
        for a, w in zip(got + got_beside, want + beside):
            assert torch.equal(a, w)


@pytest.mark.parametrize("T,k,n", [(1, 256, 40), (5, 2048, 70), (60, 512, 130), (2048, 256, 1303)])
def test_scales_of_either_sign(T, k, n):
    """A caller's own scales may be negative: huge ones are no exception. Powers of two, so that only the sum is rounded."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(3)
    xq = torch.randint(-127, 128, (T, k), device="cuda", generator=g, dtype=torch.int8)
    wq = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    xs = torch.tensor([2.0 ** 110, -(2.0 ** 110), -1.0, -(2.0 ** 96), 2.0 ** 95], device="cuda")[torch.arange(T, device="cuda") % 5]
    xs[0] = -(2.0 ** 110)
    ws = torch.tensor([2.0 ** -80, -(2.0 ** -100)], device="cuda")[torch.arange(n, device="cuda") % 2]
    want = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    y = ops.int8_gemm(xq, xs, wq, ws, out_dtype=torch.float32)
    assert ((y.double() - want).abs() <= U * want.abs()).all()
