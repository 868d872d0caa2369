"""pack8 / unpack8 / weight_grad8 / linear8 / checkpoint8 (csrc/acx_act8.hip): the format bit by bit against its definition, the weight
gradient against a float64 product of the values that the checkpoint stands for."""
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")


def definition(x):
    """q, exponent by the definition, in float64 on the host"""
    import numpy as np

    x = x.detach().double().cpu().numpy()
    M, K = x.shape
    q, e = np.zeros((M, K), np.int8), np.zeros((M, -(-K // 32)), np.uint8)
    for b in range(e.shape[1]):
        part = x[:, 32 * b:32 * b + 32]
        top = np.abs(part).max(1)
        ok = np.isfinite(top)
        n = np.full(M, -126)
        for _ in range(300):  # (the smallest exponent, found by trying)
            with np.errstate(all="ignore"):
                n = np.where(ok & (np.rint(top * 2.0 ** -n) > 127), n + 1, n)
        e[:, b] = np.where(ok, n + 127, 255)
        with np.errstate(all="ignore"):
            q[:, 32 * b:32 * b + 32] = np.where(ok[:, None], np.rint(part * 2.0 ** -n[:, None].astype(float)), 0)
    return q, e


def values(M, K, dtype, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((M, K), device="cuda", generator=g) * torch.exp(3 * torch.randn((M, 1), device="cuda", generator=g))
    return x.to(getattr(torch, dtype))


def check_format(x):
    import numpy as np
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8

    q, e = pack8(x)
    wq, we = definition(x)
    assert np.array_equal(e.cpu().numpy(), we) and np.array_equal(q.cpu().numpy(), wq)
    factor = np.repeat(np.where(we == 255, np.nan, 2.0 ** (we.astype(float) - 127)), 32, axis=1)[:, :wq.shape[1]]
    for dt in DTYPES:
        back = unpack8(q, e, getattr(torch, dt))
        want = torch.from_numpy(wq.astype(float) * factor).to(getattr(torch, dt)) if dt != "float16" else torch.from_numpy((wq * factor).astype(np.float32)).to(torch.float16)
        assert torch.equal(torch.nan_to_num(back.cpu(), 7.0), torch.nan_to_num(want, 7.0)), dt


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 7, 8, 9, 31, 32, 33, 50, 64, 72, 255, 256, 1031])
def test_format(K, dtype):
    print(K, dtype, flush=True)
    check_format(values(37, K, dtype, K))


def test_format_at_the_edges():
    """the magnitudes where the exponent changes, ties, zeros, subnormals, the largest number, infinities and NaNs"""
    import torch

    f = lambda *v: torch.tensor([list(v) + [0.0] * (32 - len(v))], device="cuda")  # noqa: E731
    tops = [127.0, 127.49999, 127.5, 127.50001, 128.0, 63.5, 63.75, 1.9921875, 1.9921874, 1.0, 0.99999994, 2.0 ** -120 * 1.5, 2.0 ** -126, 1e-40, 1e-45, 0.0, 3.4028235e38, 3.38e38,
            float("inf"), -float("inf"), float("nan")]
    check_format(torch.cat([f(t, 0.5, 1.5, 2.5, -0.5, -1.5, -t / 3 if t == t and abs(t) < 1e39 else 1.0) for t in tops]))
    check_format(torch.cat([-f(t, t / 254, -t / 254, t * 3 / 254) for t in tops[:18]]))
    check_format(torch.tensor([[1.0] * 40, [float("inf")] + [1.0] * 39, [1.0] * 39 + [float("nan")]], device="cuda"))  # the other block of a row is not touched
    check_format(torch.tensor([[65504.0, 1.0, 6e-8]], device="cuda", dtype=torch.float16))


def test_strides_axes_and_nothing():
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8

    x = values(24, 50, "float32", 1)
    wide = torch.zeros((24, 61), device="cuda")
    wide[:, 7:57] = x
    for a, b in ((wide[:, 7:57], x), (x.view(2, 3, 4, 50), x), (x.t().contiguous().t(), x)):
        q, e = pack8(a)
        assert q.shape == a.shape and torch.equal(q.view(24, 50), pack8(b)[0]) and torch.equal(e.view(24, 2), pack8(b)[1])
    q, e = pack8(x[:0])
    assert q.shape == (0, 50) and e.shape == (0, 2) and unpack8(q, e).shape == (0, 50)


def check_weight_grad(M, O, I, dtype, seed=0, strided=False):
    """Tolerance: a product of values that are exact in the matrix instruction, added up in float32: every one of the additions rounds by at
    most 2^-24 of the running sum, which is at most the sum of the magnitudes of what has been added; M terms pass through at most M
    additions, and the errors of these are independent in sign -- 8 sqrt(M) of them bounds what M can do with certainty for all practical
    purposes, never more than M.  Plus the joins (<= 300 additions)."""
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8, weight_grad8

    print(f"M {M} O {O} I {I} {dtype} strided {strided}", flush=True)
    x = values(M, I, "float32", seed)
    q, e = pack8(x)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    dy = (torch.randn((M, O), device="cuda", generator=g) * torch.exp(torch.randn((M, 1), device="cuda", generator=g))).to(getattr(torch, dtype))
    if strided:
        wide = torch.zeros((M, O + 3), device="cuda", dtype=dy.dtype)
        wide[:, 1:O + 1] = dy
        dy = wide[:, 1:O + 1]
    dw, db = weight_grad8(dy, q, e)
    xd, yd = unpack8(q, e).double(), dy.double()
    want, mag = yd.t() @ xd, yd.abs().t() @ xd.abs()
    adds = min(M, 8 * M ** 0.5) + 16
    assert dw.dtype == torch.float32 and dw.shape == (O, I) and db.shape == (O,)
    err, lim = (dw.double() - want).abs(), adds * 2.0 ** -24 * mag + 1e-37
    assert not bool((err > lim).any()), f"d weight: worst {float((err - lim).max())} beyond the tolerance"
    err, lim = (db.double() - yd.sum(0)).abs(), adds * 2.0 ** -24 * yd.abs().sum(0) + 1e-37
    assert not bool((err > lim).any()), f"d bias: worst {float((err - lim).max())} beyond the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("O,I", [(1, 1), (12, 256), (1, 256), (64, 64), (65, 63), (64, 65), (50, 72), (256, 72), (255, 257), (257, 255), (768, 256), (130, 1031), (3, 33)])
def test_weight_grad_sizes(O, I, dtype):
    check_weight_grad(777, O, I, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 63, 64, 65, 255, 256, 257, 4097, 70001])
def test_weight_grad_rows(M, dtype):
    check_weight_grad(M, 72, 50, dtype, seed=M)
    check_weight_grad(M, 300, 260, dtype, seed=M, strided=True)


def test_weight_grad_of_every_single_place():
    """one non-zero value of dy against one of x lands in its own place of dW, for places over the whole tile"""
    import torch

    from ac_solver.agents.activation8 import pack8, weight_grad8

    for O, I in ((300, 300), (40, 300), (300, 40), (40, 40)):
        M = max(O, I)
        dy, x = torch.zeros(M, O, device="cuda"), torch.zeros(M, I, device="cuda")
        n = min(O, I)
        k = torch.arange(n, device="cuda")
        o, i = (k * 7 + 3) % O, (k * 11 + 5) % I
        dy[k, o] = (k + 1).float() * 1.0009765625
        x[k, i] = 2.0
        want = torch.zeros(O, I, device="cuda")
        want.index_put_((o, i), (k + 1).float() * 2 * 1.0009765625, accumulate=True)
        assert torch.equal(weight_grad8(dy, *pack8(x))[0], want)


def test_weight_grad_of_an_expanded_gradient():
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8, weight_grad8

    q, e = pack8(values(300, 40, "float32", 9))
    row = torch.randn(1, 20, device="cuda")
    one = torch.ones((), device="cuda")
    for d in (row.expand(300, 20), one.expand(300, 20)):
        dw, db = weight_grad8(d, q, e)
        same, sb = weight_grad8(d.contiguous(), q, e)
        assert torch.equal(dw, same) and torch.equal(db, sb)
    one_row = weight_grad8(row.expand(5, 20)[:1], q[:1].contiguous(), e[:1].contiguous())[0]
    assert torch.equal(one_row, row.t() @ unpack8(q[:1], e[:1])) or float((one_row - row.t() @ unpack8(q[:1], e[:1])).abs().max()) < 1e-5


def test_weight_grad_shows_infinities_and_nans():
    """they reach the outputs that their row and column reach, and no others"""
    import torch

    from ac_solver.agents.activation8 import pack8, weight_grad8

    for dtype in DTYPES:
        x, dy = values(100, 96, "float32", 3).clamp(-100, 100), values(100, 70, dtype, 4).clamp(-100, 100)
        x[:, 5] = 1.0
        dy[7, 9] = float("inf")
        x[50, 40] = float("nan")
        dw, db = weight_grad8(dy, *pack8(x))
        assert torch.isnan(dw[:, 32:64]).all() and float(dw[9, 5]) == float("inf") and float(db[9]) == float("inf")
        rest = torch.ones(70, 96, dtype=torch.bool, device="cuda")
        rest[:, 32:64] = False
        rest[9] = False
        assert torch.isfinite(dw[rest]).all() and torch.isfinite(torch.cat((db[:9], db[10:]))).all()


def test_linear8_and_its_gradients():
    import torch

    from ac_solver.agents.activation8 import linear8, pack8, unpack8

    for dtype in DTYPES:
        dt = getattr(torch, dtype)
        x = values(500, 72, "float32", 2).clamp(-4, 4).to(dt).view(5, 100, 72).requires_grad_()
        w = (torch.randn(33, 72, device="cuda") * 0.1).requires_grad_()
        b = torch.randn(33, device="cuda").requires_grad_()
        out = linear8(x, w, b)
        assert torch.equal(out, torch.nn.functional.linear(x, w.to(dt), b.to(dt)))
        d = torch.randn(5, 100, 33, device="cuda").to(dt)
        dx, dw, db = torch.autograd.grad(out, (x, w, b), d)
        assert dx.dtype == dt and torch.equal(dx, d @ w.to(dt))
        kept = unpack8(*pack8(x)).double().view(-1, 72)
        d2 = d.double().view(-1, 33)
        assert bool(((dw.double() - d2.t() @ kept).abs() <= 500 * 2.0 ** -24 * (d2.abs().t() @ kept.abs())).all())
        assert bool(((db.double() - d2.sum(0)).abs() <= 500 * 2.0 ** -24 * d2.abs().sum(0)).all())
        with torch.no_grad():
            assert not linear8(x, w, b).requires_grad


def test_checkpoint8_restores_what_it_kept():
    """tanh keeps its output: inside the block the gradient is 1 - y^2 of the restored y, outside that of y itself; a leaf stays exact"""
    import torch

    from ac_solver.agents.activation8 import checkpoint8, pack8, unpack8

    a = torch.randn(64, 80, device="cuda", requires_grad=True)
    with checkpoint8():
        y = torch.tanh(a * 1.0)
        z = y.square()
    (g,) = torch.autograd.grad(z, a, torch.ones_like(z))
    k = unpack8(*pack8(y.detach()))
    want = 2 * k.double() * (1 - k.double() ** 2)
    assert float((g.double() - want).abs().max()) < 2.0 ** -20
    with checkpoint8():
        out = (a * a).sum()  # (a is a leaf)
    assert torch.equal(torch.autograd.grad(out, a)[0], 2 * a)
    with checkpoint8():
        out = (torch.tanh(a[:4] * 1.0) * 3).sum()  # small: as it is
    y = torch.tanh(a[:4].detach())
    assert float((torch.autograd.grad(out, a)[0][:4] - 3 * (1 - y * y)).abs().max()) < 2.0 ** -20


def test_repeated_calls_side_streams_and_graph_replays_agree():
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8, weight_grad8

    x, dy = values(5000, 72, "float32", 1), values(5000, 256, "float32", 2)

    def work():
        q, e = pack8(x)
        return (q, e, unpack8(q, e)) + weight_grad8(dy, q, e)

    first = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (3, 5, 7):
        x.copy_(values(5000, 72, "float32", seed))
        dy.copy_(values(5000, 256, "float32", seed + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work()))


def test_limits():
    import torch

    from ac_solver.agents import activation8 as A

    wide = torch.randn(2, (1 << 20) + 1, device="cuda")
    with pytest.raises(ValueError, match="2\\^20"):
        A.pack8(wide)
    x = wide.requires_grad_(True)
    with A.checkpoint8():  # rows that wide stay as they are
        out = ((x * 2.0) ** 2).sum()
    out.backward()
    assert torch.equal(x.grad, 8.0 * x.detach())  # (powers of two: nothing is rounded that was not before)
    narrow = torch.zeros(1, 1, device="cuda")
    with pytest.raises(ValueError, match="2\\^29"):
        A.weight_grad8(narrow.expand(1, 1 << 16), torch.zeros(1, 1 << 14, device="cuda", dtype=torch.int8), torch.zeros(1, 1 << 9, device="cuda", dtype=torch.uint8))


def test_more_lanes_than_a_launch_has():
    """2^30 + 9 rows of 5 values: four lanes a row and more than 2^32 of them, two launches"""
    import torch

    from ac_solver.agents import activation8 as A

    rows = (1 << 30) + 9
    x = torch.empty(rows, 5, device="cuda", dtype=torch.bfloat16)
    x.view(-1)[:] = 0
    places = torch.tensor([0, 1, (1 << 30) - 70, (1 << 30) - 65, (1 << 30) - 64, (1 << 30) - 63, 1 << 30, rows - 1], device="cuda")
    values = torch.randint(-127, 128, (len(places), 5), device="cuda").to(torch.bfloat16)
    values[:, 0] = 127  # (an exponent of 0)
    x[places] = values
    q, e = A.pack8(x)
    assert torch.equal(q[places], values.to(torch.int8)) and bool((e[places] == 127).all())
    x.fill_(1.0)
    del x
    back = A.unpack8(q, e, torch.bfloat16)
    assert torch.equal(back[places], values)
    assert int((q[:, 0] != 0).sum()) == len(places) and int((back[:, 0] != 0).sum()) == len(places)


def test_tensors_larger_than_the_caches():
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8

    x = values(70001, 1001, "float32", 5)
    q, e = pack8(x)
    back = unpack8(q, e)
    for part in (slice(0, 30000), slice(30000, 70001)):
        qh, eh = pack8(x[part])
        assert torch.equal(q[part], qh) and torch.equal(e[part], eh) and torch.equal(back[part], unpack8(qh, eh))


@pytest.mark.parametrize("M,O,I", [(2900003, 768, 32), (4300003, 12, 1024)])
def test_weight_grad_offsets_past_32_bits(M, O, I):
    """gradients (or checkpoints) of more than 2^31 values (2^32 bytes), all zero but for the first and the last 200 rows: the product of these 400 (zeros
    add nothing and round nothing; the tolerance of check_weight_grad with 400 terms)"""
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8, weight_grad8

    assert max(2 * M * O, M * I) > 1 << 32
    q = torch.zeros((M, I), device="cuda", dtype=torch.int8)
    e = torch.full((M, I // 32), 127, device="cuda", dtype=torch.uint8)
    dy = torch.zeros((M, O), device="cuda", dtype=torch.bfloat16)
    rows = torch.cat([torch.arange(200), torch.arange(M - 200, M)]).cuda()
    q[rows], e[rows] = pack8(values(400, I, "float32", 8))
    dy[rows] = torch.randn((400, O), device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(torch.bfloat16)
    dw, db = weight_grad8(dy, q, e)
    xd, yd = unpack8(q[rows], e[rows]).double(), dy[rows].double()
    adds = 8 * 400 ** 0.5 + 16 + 300
    err, lim = (dw.double() - yd.t() @ xd).abs(), adds * 2.0 ** -24 * (yd.abs().t() @ xd.abs()) + 1e-37
    assert not bool((err > lim).any())
    err, lim = (db.double() - yd.sum(0)).abs(), adds * 2.0 ** -24 * yd.abs().sum(0) + 1e-37
    assert not bool((err > lim).any())


FORMS_OF_A_LEAF = {
    "view": lambda a: a.view(5, 60, 256),
    "transpose": lambda a: a.t(),
    "slice": lambda a: a[:, 3:131],
    "select": lambda a: a.view(5, 60, 256)[2],
    "split": lambda a: a.split(128, 1)[1],
    "unbind": lambda a: a.view(2, 150, 256).unbind(0)[1],
    "expand": lambda a: a.unsqueeze(0).expand(2, 300, 256),
    "view of a view": lambda a: a.t()[:100].unsqueeze(1),
}


@pytest.mark.parametrize("form", sorted(FORMS_OF_A_LEAF))
def test_checkpoint8_keeps_views_of_leaves(form):
    """a leaf in another shape is still the leaf: the gradient is the one outside the block, bit by bit"""
    import torch

    from ac_solver.agents.activation8 import checkpoint8

    a = torch.randn(300, 256, device="cuda", requires_grad=True)
    with checkpoint8():
        out = FORMS_OF_A_LEAF[form](a).square()
    d = torch.randn_like(out)
    (got,) = torch.autograd.grad(out, a, d)
    (want,) = torch.autograd.grad(FORMS_OF_A_LEAF[form](a).square(), a, d)
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(300, 256), (3, 100, 256)])
def test_checkpoint8_around_a_plain_layer(shape):
    """torch's own linear layer keeps a transposed view of its weight: that one stays exact, its input is kept in 8 bits.  The gradient of the weight is a sum of
    300 products in float32, in whatever order the library takes: at most 300 roundings of 2^-24 of the magnitudes."""
    import torch

    from ac_solver.agents.activation8 import checkpoint8, pack8, unpack8

    torch.manual_seed(3)
    layer = torch.nn.Linear(256, 192).cuda()
    x = torch.randn(*shape, device="cuda", requires_grad=True)
    u = x * 1.0
    with checkpoint8():
        out = layer(u)
    plain = layer(u)
    d = torch.randn_like(out)
    dx, dw, db = torch.autograd.grad(out, (x, layer.weight, layer.bias), d, retain_graph=True)
    wx, ww, wb = torch.autograd.grad(plain, (x, layer.weight, layer.bias), d)
    assert torch.equal(dx, wx) and torch.equal(db, wb)
    kept, d2 = unpack8(*pack8(u.detach())).double().view(-1, 256), d.double().view(-1, 192)
    assert bool(((dw.double() - d2.t() @ kept).abs() <= 300 * 2.0 ** -24 * (d2.abs().t() @ kept.abs())).all())
    assert not torch.equal(dw, ww)  # (the input is an activation: it is in 8 bits)


def test_checkpoint8_keeps_copies_of_leaves_in_other_types():
    """a layer in bfloat16 reads a bfloat16 copy of its float32 weight, autocast makes that copy itself: the gradient of the input is the one outside the
    block, bit by bit; a clone and a contiguous transpose of a leaf are kept, too"""
    import contextlib

    import torch
    from torch.nn import functional as F

    from ac_solver.agents.activation8 import checkpoint8

    torch.manual_seed(4)
    w = torch.randn(192, 256, device="cuda", requires_grad=True)
    x = torch.randn(300, 256, device="cuda", requires_grad=True)

    def cast(block):
        with block:
            return F.linear((x * 1.0).bfloat16(), w.bfloat16())

    def cast_of_a_view(block):
        with block:
            return (x * 1.0).bfloat16() @ w.t().bfloat16()

    def autocast(block):
        with block, torch.autocast("cuda", torch.bfloat16):
            return F.linear(x * 1.0, w)

    for f in (cast, cast_of_a_view, autocast):
        got, want = f(checkpoint8()), f(contextlib.nullcontext())
        d = torch.randn_like(got)
        assert torch.equal(torch.autograd.grad(got, x, d)[0], torch.autograd.grad(want, x, d)[0]), f.__name__
    for f in (lambda: w.clone().square(), lambda: w.t().contiguous().square(), lambda: w.double().float().square()):
        with checkpoint8():
            got = f()
        d = torch.randn_like(got)
        assert torch.equal(torch.autograd.grad(got, w, d)[0], torch.autograd.grad(f(), w, d)[0])


def test_checkpoint8_keeps_one_value_a_row():
    """a column of row statistics (the reciprocal root of a norm) would take two bytes a value, and every value of its row hangs on it: kept as it is"""
    import torch

    from ac_solver.agents.activation8 import checkpoint8

    a = torch.randn(8192, 8, device="cuda", requires_grad=True)

    def f():
        return torch.rsqrt(a.square().mean(-1, keepdim=True) + 1e-6)

    with checkpoint8():
        out = f()
    d = torch.randn_like(out)
    assert out.numel() == 8192 and torch.equal(torch.autograd.grad(out, a, d)[0], torch.autograd.grad(f(), a, d)[0])


def test_finite_values_restore_to_finite_values():
    """where rounding up to the next exponent carries a block's largest value past the type's largest finite one (float16 from 65280 on, float32 and bfloat16
    from 1.9921875 * 2^127 on) it restores to that largest one: off by at most 2^-8 of it; the fifths of
    it beside it lie a quarter of q's unit from a whole number, 2^-8 of the largest again (2^-7 leaves a factor of two); infinities and NaN still restore to NaN"""
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8

    border = {"float16": [65280.0, 65376.0, 65504.0, 65248.0], "bfloat16": [3.3895313892515355e38, 3.37e38], "float32": [3.3895313892515355e38, 3.4e38, 3.4028234663852886e38, 3.3895311e38]}
    for name, tops in border.items():
        dt = getattr(torch, name)
        for width in (1, 3, 8, 32, 40):
            rows = [[s * t] + [t / 5] * (width - 1) for t in tops for s in (1.0, -1.0)]
            x = torch.tensor(rows, device="cuda", dtype=torch.float64).to(dt)
            back = unpack8(*pack8(x), dt)
            assert torch.isfinite(x).all() and torch.isfinite(back).all(), (name, width)
            err, top = (back.double() - x.double()).abs(), x.double().abs()[:, :1]
            assert bool((err[:, :32] <= 2.0 ** -7 * top).all()), (name, width)
            for other in DTYPES:
                assert torch.isfinite(unpack8(*pack8(x), getattr(torch, other))).all(), (name, other, width)
    x = torch.full((4, 40), 1.0, device="cuda")
    x[0, 3], x[1, 3], x[2, 35] = float("inf"), -float("inf"), float("nan")
    for other in DTYPES:
        bad = torch.isnan(unpack8(*pack8(x), getattr(torch, other)))
        want = torch.zeros_like(bad)
        want[0, :32], want[1, :32], want[2, 32:] = True, True, True
        assert torch.equal(bad, want)


@pytest.mark.parametrize("M", [3, 200])
def test_weight_grad_of_the_largest_finite_values(M):
    """the largest finite activations count as what they restore to in bfloat16, 1.9921875 * 2^127 (M 3: the rows that are read one by one; 200: whole
    vectors, too).  Only these rows are not zero, so a product is one term of float32: the two roundings of a term and of its sum."""
    import torch

    from ac_solver.agents.activation8 import pack8, unpack8, weight_grad8

    for dtype in DTYPES:
        for O, I in ((3, 5), (70, 40), (65, 129), (300, 260)):
            x = torch.zeros(M, I, device="cuda")
            dy = torch.zeros(M, O, device="cuda", dtype=getattr(torch, dtype))
            for row, sign in ((0, 1.0), (M - 1, -1.0)):
                x[row, row % I] = sign * 3.4028234663852886e38
            dy[0], dy[M - 1, :2] = 2.0 ** -9, 2.0 ** -10
            q, e = pack8(x)
            dw, db = weight_grad8(dy, q, e)
            kept = unpack8(q, e, torch.bfloat16).double()
            want = dy.double().t() @ kept
            assert torch.isfinite(dw).all() and float(want.abs().max()) > 1e35
            assert bool(((dw.double() - want).abs() <= 2.0 ** -23 * want.abs()).all()), (dtype, O, I)
