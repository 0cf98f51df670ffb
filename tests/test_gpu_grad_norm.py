"""Global gradient norm and clipping against a 64-bit computation.

Tolerances. The norm: squares of eight elements are added in fp32 with eight roundings at most (relative 8 * 2^-24 of a sum
of positive terms), everything else in fp64, the square root halves the relative error, one rounding to fp32:
4 * 2^-24 + 2^-24. Clipped values: the coefficient is rounded to fp32 (2^-24), the product once to fp32 (2^-24) and once to
the output's type (half a step), and the 64-bit coefficient differs by the norm's error before its last rounding
(4 * 2^-24): 6 * 2^-24 + finfo(type).eps / 2, rounded up below.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NORM_TOL = 6 * U


def _value_tol(dtype):
    return 7 * U + torch.finfo(dtype).eps / 2


def _ops():
    from sparseforge_b200 import ops

    return ops


def _make(sizes, dtypes, scale=1e-2, seed=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n, dt in zip(sizes, dtypes):
        buf = (torch.randn(n + offset, device="cuda", generator=g) * scale).to(dt)
        out.append(buf[offset:])
    return out


def _exact(grads, p=2.0):
    if p == math.inf:
        return max((float(g.double().abs().max()) for g in grads if g.numel()), default=0.0)
    return math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in grads))


SETS = {
    "one": ([1], ["bf16"]),
    "seven": ([7], ["f32"]),
    "mixed": ([1, 8, 9, 4096, 4097, 12345, 31, 262144], ["bf16", "f32"] * 4),
    "with_empty": ([0, 5, 0, 1000], ["f32", "bf16", "bf16", "f32"]),
    "matrix": ([1100 * 1024 + 3], ["bf16"]),
    "many": ([1 + 37 * i for i in range(500)], ["bf16", "f32"] * 250),
    "table_edge": ([16] * 449, ["f32"] * 449),
    "big": ([11008 * 4096, 4096 * 4096, 4096], ["bf16", "bf16", "f32"]),
}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _set(name, **kw):
    sizes, names = SETS[name]
    return _make(sizes, [DT[n] for n in names], **kw)


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("offset", [0, 1, 6])
@pytest.mark.parametrize("name", list(SETS))
def test_norm(name, offset, p):
    grads = _set(name, seed=3, offset=offset)
    got = _ops().grad_norm(grads, p)
    assert got.dtype == torch.float32 and got.dim() == 0
    want = _exact(grads, p)
    assert abs(float(got) - want) <= (0.0 if p == math.inf else NORM_TOL * want)
    assert torch.equal(got, _ops().grad_norm(grads, p))  # the order of the sum is fixed


@pytest.mark.parametrize("scale", [1e-42, 1e-38, 1e-30, 1e-22, 1e-3, 1e15, 1e20, 1e37])
def test_norm_keeps_the_range_of_fp32(scale):
    """Squares of 1e20 are beyond fp32, those of 1e-30 below it; 1e-42 is subnormal itself."""
    grads = [torch.tensor([scale, -scale, 0.0, scale * 0.5] * 37, device="cuda"),
             torch.full((4096,), scale / 64, device="cuda", dtype=torch.float32)]
    want = _exact(grads)
    # a subnormal result is rounded to a multiple of 2^-149
    assert abs(float(_ops().grad_norm(grads)) - want) <= NORM_TOL * want + 2.0 ** -150
    assert float(_ops().grad_norm(grads, math.inf)) == _exact(grads, math.inf)


def test_norm_mixes_magnitudes_and_zeros():
    big = torch.zeros(10000, device="cuda")
    big[1234] = 3e25
    tiny = torch.full((5000,), 1e-25, device="cuda")
    zeros = torch.zeros(1 << 16, device="cuda", dtype=torch.bfloat16)
    grads = [tiny, big, zeros]
    assert abs(float(_ops().grad_norm(grads)) - _exact(grads)) <= NORM_TOL * _exact(grads)
    assert float(_ops().grad_norm([zeros])) == 0.0
    assert float(_ops().grad_norm([zeros, tiny[:0]], math.inf)) == 0.0
    # a sum over more than fp32's 24 bits of equal terms
    ones = torch.ones(3 << 24, device="cuda", dtype=torch.bfloat16)
    assert abs(float(_ops().grad_norm([ones])) - math.sqrt(3 << 24)) <= NORM_TOL * math.sqrt(3 << 24)


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("at", [0, 4095, 12340])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_infinite_and_nan_gradients(bad, at, p):
    grads = _make([300, 12345], [torch.float32, torch.bfloat16], seed=5)
    grads[1][at] = bad
    want = [torch.empty_like(g) for g in grads]
    norm = _ops().clip_grad_norm(grads, 1.0, p, out=want)
    assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
    for g, o in zip(grads, want):
        ref = (g.float() * (math.nan if math.isnan(bad) else 0.0)).to(g.dtype)
        assert torch.equal(torch.nan_to_num(o.float(), nan=7.0), torch.nan_to_num(ref.float(), nan=7.0))


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("offset", [0, 3, 4])
@pytest.mark.parametrize("mode", ["in_place", "same", "other"])
@pytest.mark.parametrize("name", list(SETS))
def test_clip(name, mode, offset, p):
    ops = _ops()
    grads = _set(name, seed=11, offset=offset)
    raw = [g.clone() for g in grads]
    want_norm = _exact(raw, p)
    max_norm = 0.3 * want_norm
    factor = min(1.0, max_norm / (want_norm + 1e-6))
    if mode == "in_place":
        out = grads
        norm = ops.clip_grad_norm(grads, max_norm, p)
    else:
        flip = {torch.bfloat16: torch.float32, torch.float32: torch.bfloat16}
        guard = 5  # elements before and behind each output that no call may touch
        bufs = [torch.full((g.numel() + 2 * guard,), -3.0, device="cuda", dtype=g.dtype if mode == "same" else flip[g.dtype])
                for g in grads]
        out = [b[guard:b.numel() - guard] for b in bufs]
        norm = ops.clip_grad_norm(grads, max_norm, p, out=out)
        for b in bufs:
            assert (b[:guard] == -3.0).all() and (b[b.numel() - guard:] == -3.0).all()
        for g, r in zip(grads, raw):
            assert torch.equal(g, r)
    assert abs(float(norm) - want_norm) <= NORM_TOL * want_norm
    for r, o in zip(raw, out):
        ref = r.double() * factor
        # half a step of the subnormal range where the value is that small
        assert ((o.double() - ref).abs() <= _value_tol(o.dtype) * ref.abs() + 1e-40).all()


def test_clip_without_need_leaves_the_gradients_alone():
    ops = _ops()
    grads = _set("mixed", seed=2)
    raw = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, 1e9)
    assert abs(float(norm) - _exact(raw)) <= NORM_TOL * _exact(raw)
    assert all(torch.equal(g, r) for g, r in zip(grads, raw))
    out = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm(grads, math.inf, out=out)
    assert all(torch.equal(o, r) for o, r in zip(out, raw))
    ops.clip_grad_norm(grads, 0.0)
    assert all(float(g.abs().sum()) == 0.0 for g in grads)


def test_clip_by_a_norm_from_elsewhere():
    """The norm of two halves combined (as over two ranks), then each half clipped by it."""
    ops = _ops()
    a, b = _set("mixed", seed=21), _set("many", seed=22)
    want = [g.clone() for g in a + b]
    whole = ops.clip_grad_norm(want, 0.5)
    combined = torch.sqrt(ops.grad_norm(a).double() ** 2 + ops.grad_norm(b).double() ** 2).float()
    assert abs(float(combined) - float(whole)) <= 2 * NORM_TOL * float(whole)
    ops.clip_grads(a, combined, 0.5)
    ops.clip_grads(b, combined, 0.5)
    for g, w in zip(a + b, want):
        # both coefficients carry their norm's error, and a bf16 value may fall on either side of a half step
        assert ((g.double() - w.double()).abs() <= (20 * U + (2.0 ** -7 if g.dtype == torch.bfloat16 else 0)) * w.double().abs()).all()


def test_strided_but_dense_gradients_and_other_layouts():
    ops = _ops()
    base = torch.randn(64, 48, device="cuda")
    ops.clip_grad_norm([base.t()], 1.0)
    assert abs(_exact([base]) - 1.0) <= 1e-5
    for bad in (base[:, ::2], base[:1].expand(5, 48)):
        with pytest.raises(RuntimeError, match="contiguous"):
            ops.grad_norm([bad])
    with pytest.raises(ValueError, match="strides"):
        ops.clip_grad_norm([base.t()], 1.0, out=[torch.empty(48, 64, device="cuda")])


def test_refusals():
    ops = _ops()
    a = torch.randn(4096, device="cuda")
    b = torch.randn(4096, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grad_norm([a, b, a], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grad_norm([a[:100], a[50:200]], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grad_norm([a, b], 1.0, out=[b, a])
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grad_norm([a[:2048]], 1.0, out=[a.view(torch.bfloat16)[:2048]])
    with pytest.raises(RuntimeError, match="norm"):
        ops.clip_grads([a, b], a[7], 1.0)
    assert abs(float(ops.grad_norm([a, a])) - math.sqrt(2.0) * _exact([a])) <= 2 * NORM_TOL * _exact([a, a])  # reading twice is fine
    with pytest.raises(TypeError):
        ops.grad_norm([a.half()])
    with pytest.raises(TypeError):
        ops.grad_norm([torch.zeros(8, device="cuda", dtype=torch.int8)])
    with pytest.raises(NotImplementedError):
        ops.grad_norm([a], 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.clip_grad_norm([a], -1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.clip_grad_norm([a], math.nan)
    with pytest.raises(ValueError):
        ops.clip_grad_norm([a], 1.0, out=[])
    with pytest.raises(TypeError):
        ops.clip_grads([a], torch.ones((), device="cuda", dtype=torch.float64), 1.0)
    with pytest.raises((RuntimeError, ValueError)):
        ops.grad_norm([a, torch.zeros(3)])


def test_streams_and_graph_replay():
    """Two calls on two streams, and a captured call replayed on new gradients."""
    ops = _ops()
    one, two = _set("mixed", seed=31), _set("many", seed=32)
    want = _exact(one), _exact(two)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((ops.grad_norm(one), want[0]))
        with torch.cuda.stream(s2):
            got.append((ops.grad_norm(two), want[1]))
    torch.cuda.synchronize()
    for n, w in got:
        assert abs(float(n) - w) <= NORM_TOL * w
    # two graphs captured on one stream hold scratch of their own
    graphs, norms = [], []
    for grads in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grad_norm(grads, 0.25))
        graphs.append(g)
    for rep in range(3):
        fresh = [_set("mixed", seed=40 + rep), _set("many", seed=50 + rep)]
        for grads, new in zip((one, two), fresh):
            for a, b in zip(grads, new):
                a.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        for grads, new, n in zip((one, two), fresh, norms):
            assert abs(float(n) - _exact(new)) <= NORM_TOL * _exact(new)
            f = min(1.0, 0.25 / (_exact(new) + 1e-6))
            for a, b in zip(grads, new):
                ref = b.double() * f
                assert ((a.double() - ref).abs() <= _value_tol(a.dtype) * ref.abs() + 1e-40).all()


def test_utils_clip_matches_torch():
    """Same arguments, same effect as torch.nn.utils.clip_grad_norm_ on fp32 gradients."""
    from sparseforge_b200 import utils

    torch.manual_seed(0)
    make = lambda: [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (5, 1000, 77 * 64)]  # noqa: E731
    ours, theirs = make(), make()
    for a, b in zip(ours, theirs):
        a.grad = torch.randn_like(a)
        b.grad = a.grad.clone()
    ours.append(torch.nn.Parameter(torch.zeros(3, device="cuda")))  # no gradient
    n1 = utils.clip_grad_norm_(ours + ours[:1], 1.0)
    n2 = torch.nn.utils.clip_grad_norm_(theirs, 1.0)
    # torch adds up in fp32: a chain of rounded sums, here below 5000 terms in a tree
    assert abs(float(n1) - float(n2)) <= 64 * U * float(n2)
    for a, b in zip(ours, theirs):
        assert ((a.grad - b.grad).abs() <= 70 * U * b.grad.abs()).all()
    assert float(utils.clip_grad_norm_([], 1.0)) == 0.0
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p.grad = torch.tensor([1.0, math.nan, 0.0, 2.0], device="cuda")
    with pytest.raises(RuntimeError, match="non-finite"):
        utils.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    p.grad = torch.tensor([3.0, 4.0, 0.0, 0.0], device="cuda")
    assert float(utils.clip_grad_norm_(p, 10.0, norm_type=math.inf, error_if_nonfinite=True)) == 4.0


def test_clip_of_a_model_with_a_sharded_layer_in_one_process():
    from sparseforge_b200 import sharding, utils

    torch.manual_seed(1)
    model = torch.nn.Sequential(sharding.RowShardedLinear(torch.nn.Linear(16, 8)), torch.nn.LayerNorm(8)).cuda()
    for q in model.parameters():
        q.grad = torch.randn_like(q)
    raw = [q.grad.clone() for q in model.parameters()]
    norm = sharding.clip_grad_norm_(model, 0.25)
    clipped = [q.grad.clone() for q in model.parameters()]
    for q, r in zip(model.parameters(), raw):
        q.grad = r
    assert torch.equal(norm, utils.clip_grad_norm_(model.parameters(), 0.25))
    assert all(torch.equal(q.grad, c) for q, c in zip(model.parameters(), clipped))


def test_codes_of_the_c_entry_points():
    from sparseforge_b200 import _lib

    lib = _lib.lib()
    t = torch.ones(16, device="cuda")
    n = torch.zeros(1, device="cuda")
    sc = torch.zeros(int(lib.sf_grad_norm_scratch_doubles(1)), device="cuda", dtype=torch.float64)
    P, S, D = (ctypes.c_void_p * 1)(t.data_ptr()), (ctypes.c_int64 * 1)(16), (ctypes.c_int32 * 1)(0)
    st = torch.cuda.current_stream().cuda_stream
    assert lib.sf_grad_norm(P, S, D, 1, 0, n.data_ptr(), sc.data_ptr(), st) == 0
    assert float(n) == 4.0
    assert lib.sf_grad_norm(None, None, None, 0, 0, n.data_ptr(), sc.data_ptr(), st) == 0
    assert float(n) == 0.0


def test_a_tensor_of_more_than_2_to_the_31_elements():
    ops = _ops()
    n = (1 << 31) + 12345
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[::1 << 20] = 1.0
    g[-1] = 2.0
    want = math.sqrt(float(len(range(0, n, 1 << 20))) + 4.0 - (1.0 if (n - 1) % (1 << 20) == 0 else 0.0))
    norm = ops.clip_grad_norm([g], want / 4)
    assert abs(float(norm) - want) <= NORM_TOL * want
    assert float(g[-1]) == 0.5 and float(g[0]) == 0.25 and float(g[1 << 20]) == 0.25
    assert float(ops.grad_norm([g[-5:], g], math.inf)) == 0.5


@pytest.mark.parametrize("dt,odt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_every_alignment(dt, odt):
    """Gradients and outputs at every element offset from a 16-byte boundary, and lengths around the access sizes."""
    ops = _ops()
    src = torch.randn(9000, device="cuda").to(DT[dt])
    for go in range(9):
        for oo in (go, 0, 1, 3, 4, 7):
            for n in (1, 2, 7, 8, 9, 15, 17, 4096, 8200):
                g = src[go:go + n]
                buf = torch.full((n + oo + 9,), 7.0, device="cuda", dtype=DT[odt])
                o = buf[oo:oo + n]
                norm = ops.clip_grad_norm([g], 0.5, out=[o])
                w = _exact([g])
                assert abs(float(norm) - w) <= NORM_TOL * w
                ref = g.double() * min(1.0, 0.5 / (w + 1e-6))
                assert ((o.double() - ref).abs() <= _value_tol(o.dtype) * ref.abs() + 1e-40).all(), (go, oo, n)
                assert (buf[:oo] == 7.0).all() and (buf[oo + n:] == 7.0).all()


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-30, 1e-37])
@pytest.mark.parametrize("size", [3e38, 1e36, 4e37])
@pytest.mark.parametrize("dt,odt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_coefficients_below_the_normal_range(dt, odt, size, max_norm, p):
    """Gradients so large, or a limit so small, that max_norm / norm is subnormal or zero in fp32; with 5000 elements the
    L2 norm itself is beyond fp32. Outputs are the formula's, to the tolerance of any other case and a subnormal step
    (two half steps in fp32, half a step in bf16)."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(17)
    src = [(torch.rand(n, device="cuda", generator=g) * 2 - 1).mul_(size).to(DT[dt]) for n in (5000, 37, 4099)]
    want = _exact(src, p)
    factor = max_norm / (want + 1e-6)
    steps = 2.0 ** -149 + (2.0 ** -134 if odt == "bf16" else 0.0)

    def check(out):
        for s, o in zip(src, out):
            ref = s.double() * factor
            assert ((o.double() - ref).abs() <= _value_tol(o.dtype) * ref.abs() + steps).all()

    out = [torch.empty_like(s, dtype=DT[odt]) for s in src]
    norm = ops.clip_grad_norm(src, max_norm, p, out=out)
    assert float(norm) == math.inf if want > 3.5e38 else abs(float(norm) - want) <= NORM_TOL * want
    check(out)
    if want < 3.4e38:
        ops.clip_grads(src, norm, max_norm, out=out)
        check(out)
    if dt == odt:
        here = [s.clone() for s in src]
        ops.clip_grad_norm(here, max_norm, p)
        check(here)


@pytest.mark.parametrize("how", ["clip_grad_norm", "clip_grads", "utils"])
def test_a_graph_that_saved_a_clipped_gradient_is_told(how):
    """As after torch's own in-place clipping: the backward of a graph that saved the unclipped values raises instead of
    using the clipped ones. Outputs count as written, inputs that went to other buffers do not."""
    from sparseforge_b200 import utils

    ops = _ops()
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = torch.randn(100, device="cuda")
    out = torch.empty_like(p.grad)
    v = torch.ones(100, device="cuda", requires_grad=True)
    (v * p.grad).sum().backward()
    saved, kept = (v * p.grad).sum(), (v * out).sum()
    ops.clip_grad_norm([p.grad], 0.5, out=[out])
    saved.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    if how == "utils":
        utils.clip_grad_norm_([p], 0.5)
    elif how == "clip_grad_norm":
        ops.clip_grad_norm([p.grad], 0.5)
    else:
        ops.clip_grads([p.grad], ops.grad_norm([p.grad]), 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    with torch.inference_mode():  # tensors without a version counter
        g = torch.randn(10, device="cuda")
        ops.clip_grad_norm([g], 0.5)
        assert abs(_exact([g]) - 0.5) <= 1e-5
