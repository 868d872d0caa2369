"""block_output / block_input / recurrent_step (csrc/acx_block.hip) against their definitions in float64."""
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")
EPS = 1e-6


def make(M, D, dtype, seed, layout="contiguous"):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    n = lambda *s, k=1.0, b=0.0: torch.randn(s, device="cuda", generator=g) * k + b  # noqa: E731
    x, y, gate, dx, du = (n(M, D, k=k).to(dt) for k in (2.0, 0.5, 1.0, 0.3, 0.3))
    if layout == "slices":
        p = torch.empty((M, 3 * D + 1), device="cuda", dtype=dt)
        p[:, 1:1 + D], p[:, 2 * D:3 * D] = gate, y
        gate, y = p[:, 1:1 + D], p[:, 2 * D:3 * D]
    return x, y, gate, n(D, k=0.2, b=1.0), n(D, k=0.2, b=0.5), n(D, k=0.2, b=1.0), dx, du


def definition(x, y, gate, w, scale, nw, dx, du):
    """autograd of the formula in float64"""
    import torch

    leaves = [None if t is None else t.double().detach().requires_grad_() for t in (x, y, gate, w, scale, nw)]
    x, y, gate, w, scale, nw = leaves
    rms = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)  # noqa: E731
    new = x
    if y is not None:
        p = rms(y) * w
        if gate is not None:
            p = p * gate * torch.sigmoid(gate)
        new = x + (p if scale is None else scale * p)
    u = None if nw is None else rms(new) * nw
    outs, gs = [], []
    for o, g in ((new, dx), (u, du)):
        if o is not None and g is not None and o.requires_grad:
            outs.append(o)
            gs.append(g.double())
    used = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(outs, used, gs, allow_unused=True))
    return new.detach(), None if u is None else u.detach(), [None if t is None else next(grads) for t in leaves]


def magnitudes(real, x, y, gate, w, scale, nw, dx, du):
    """(`real`: new in float64.)  For the gradients of weight, scale, next_weight: the sum over the rows of the magnitudes that went into a row's term.  A term is a product;
    two of its factors are differences and can cancel, so their error goes by what was subtracted, not by what is left:
        |new| -> |x| + |scale p|,    |d x| -> |d_new| + rx (|t| + |xn| mean |t xn|),   t = d_u next_weight, xn = new rx"""
    import torch

    x, dx, du = (None if t is None else t.double().abs() for t in (x, dx, du))
    rms = lambda v: 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)  # noqa: E731
    one = torch.ones(x.shape[1], dtype=torch.float64, device=x.device)
    s = one if scale is None else scale.double().abs()
    if y is None:
        p, a, yn, new = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), x
    else:
        yn = y.double().abs() * rms(y.double())
        a = one if gate is None else (gate.double() * torch.sigmoid(gate.double())).abs()
        p = a * yn * w.double().abs()
        new = x + s * p
    bound = torch.zeros_like(x) if dx is None else dx
    d_next = None
    if nw is not None and du is not None:
        rx = rms(real)
        t, xn = du * nw.double().abs(), new * rx
        bound = bound + rx * (t + xn * (t * xn).mean(-1, keepdim=True))
        d_next = (du * xn).sum(0)
    return (bound * s * a * yn).sum(0), (bound * p).sum(0), d_next


def assert_close(got, want, dtype, what, terms=1, sums=None):
    """one rounding to the output's type (eps / 2 of the value) plus float32 arithmetic: a chain of some forty operations with relative errors
    of at most 2^-24 each on terms no larger than the tensor's largest magnitude (which bounds the terms up to the factor `terms` where they
    cancel).  A sum over rows (`sums`: see magnitudes) adds 2^-24 of that for each of the up to 64
    roundings a term passes through: its own ~40, the additions of one lane's chain weighted by the partial sums, and the joins."""
    import torch

    eps = torch.finfo(getattr(torch, dtype)).eps / 2
    err = (got.double() - want).abs()
    tiny = torch.finfo(torch.float16).smallest_normal * eps if dtype == "float16" else 0.0
    lim = want.abs() * eps * (1 + 2 ** -7) + tiny + (64 * 2.0 ** -24 * sums if sums is not None else float(want.abs().max()) * terms * 64 * 2.0 ** -24)
    bad = err > lim
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {err.numel()} off, worst {float((err - lim).max())} beyond the tolerance"


def check(M, D, dtype, seed=0, layout="contiguous", gate=True, scale=True, nxt=True, d_new=True, d_u=True):
    import torch

    from ac_solver.agents.block_norm import block_output

    print(f"M {M} D {D} {dtype} {layout} gate {gate} scale {scale} next {nxt} grads {d_new} {d_u}", flush=True)
    x, y, g, w, s, v, dx, du = make(M, D, dtype, seed, layout)
    ops = [x, y, g if gate else None, w, s if scale else None, v if nxt else None]
    leaves = [None if t is None else t.detach().requires_grad_() for t in ops]
    new, u = block_output(*leaves, eps=EPS)
    wn, wu, wg = definition(*ops, dx if d_new else None, du if d_u else None)
    assert_close(new, wn, dtype, "new")
    assert (u is None) == (not nxt)
    if nxt:
        assert_close(u, wu, dtype, "u")
    outs = [o for o, on in ((new, d_new), (u, d_u and nxt)) if on]
    gos = [o for o, on in ((dx, d_new), (du, d_u and nxt)) if on]
    used = [t for t in leaves if t is not None]
    sums = dict(zip(("weight", "scale", "next_weight"), magnitudes(wn, *ops, dx if d_new else None, du if d_u else None)))
    got = iter(torch.autograd.grad(outs, used, gos))
    for name, leaf, want in zip(("x", "y", "gate", "weight", "scale", "next_weight"), leaves, wg):
        if leaf is None:
            continue
        g1 = next(got)
        if want is None:
            assert not bool(g1.any()), name
            continue
        if name in ("weight", "scale", "next_weight"):
            assert_close(g1, want, "float32", "d " + name, sums=sums[name])
        else:
            assert_close(g1, want, dtype, "d " + name, terms=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 7, 8, 9, 31, 32, 33, 50, 64, 65, 127, 130, 255, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 3001, 4095, 4096])
def test_widths(D, dtype):
    check(70 if D < 600 else 9, D, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 63, 1023, 1025, 5000])
def test_rows(M, dtype):
    check(M, 72, dtype)
    check(M, 256, dtype, seed=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [dict(gate=False), dict(scale=False), dict(nxt=False), dict(d_new=False), dict(d_u=False), dict(gate=False, scale=False, nxt=False)])
def test_parts_left_out(off, dtype):
    check(37, 50, dtype, **off)
    check(5, 2100, dtype, **off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [50, 255, 256])
def test_slices_of_a_projection(D, dtype):
    check(33, D, dtype, layout="slices")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 50, 256, 1500])
def test_the_norm_in_front(D, dtype):
    import torch

    from ac_solver.agents.block_norm import block_input

    x, _, _, _, _, v, _, du = make(45, D, dtype, 3)
    leaves = [x.detach().requires_grad_(), v.detach().requires_grad_()]
    u = block_input(*leaves, eps=EPS)
    _, wu, wg = definition(x, None, None, None, None, v, None, du)
    assert_close(u, wu, dtype, "u")
    got = torch.autograd.grad(u, leaves, du)
    assert_close(got[0], wg[0], dtype, "d x", terms=4)
    assert_close(got[1], wg[5], "float32", "d weight", sums=magnitudes(x.double(), x, None, None, None, None, v, None, du)[2])


def test_more_axes_no_rows_and_zero_rows():
    import torch

    from ac_solver.agents.block_norm import block_output

    x, y, g, w, s, v, dx, du = make(24, 40, "float32", 4)
    a = block_output(x, y, g, w, s, v)
    b = block_output(x.view(2, 3, 4, 40), y.view(2, 3, 4, 40), g.view(2, 3, 4, 40), w, s, v)
    assert all(torch.equal(p.view(-1), q.view(-1)) for p, q in zip(a, b)) and b[0].shape == (2, 3, 4, 40)
    leaves = [t[:0].detach().requires_grad_() for t in (x, y, g)] + [t.detach().requires_grad_() for t in (w, s, v)]
    new, u = block_output(*leaves)
    grads = torch.autograd.grad((new, u), leaves, (new.detach(), u.detach()))
    assert new.shape == (0, 40) and not any(bool(t.any()) for t in grads[3:])
    # a row of zeros: rms is 0 / sqrt(eps); its gradients are finite
    z = torch.zeros(2, 40, device="cuda")
    leaves = [t.requires_grad_() for t in (z.clone(), z.clone(), z.clone())]
    new, u = block_output(*leaves, w, s, v)
    assert not bool(new.any()) and not bool(u.any())
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad((new, u), leaves, (z + 1, z + 1)))


def test_one_bad_row_stays_alone():
    """an infinity or NaN in one row leaves the others what they were"""
    import torch

    from ac_solver.agents.block_norm import block_output

    for D in (50, 256, 3000):
        x, y, g, w, s, v, _, _ = make(9, D, "float32", 5)
        want = block_output(x, y, g, w, s, v)
        y2 = y.clone()
        y2[4, D // 2] = float("nan")
        got = block_output(x, y2, g, w, s, v)
        rows = [r for r in range(9) if r != 4]
        assert all(torch.equal(a[rows], b[rows]) for a, b in zip(got, want)) and torch.isnan(got[0][4]).all()


def test_repeated_calls_side_streams_and_graph_replays_agree():
    import torch

    from ac_solver.agents.block_norm import block_output_backward, block_output_forward

    for M, D, dtype in ((5000, 256, "bfloat16"), (300, 2050, "float32")):
        x, y, g, w, s, v, dx, du = make(M, D, dtype, 6)

        def both():
            new, u, st = block_output_forward(x, y, g, w, s, v)
            return (new, u, st) + block_output_backward(dx, du, x, y, g, w, s, v, st)

        first = both()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            again = both()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        for seed in (7, 8, 9):
            for dst, src in zip((x, y, g, w, s, v, dx, du), make(M, D, dtype, seed)):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, both()))


def step_definition(x, p, h, w, s, v, r):
    import torch

    D = x.shape[1]
    c, z, g = (t.double() for t in (p[:, :D], p[:, D:2 * D], p[:, 2 * D:]))
    h = h.double()
    if r is not None:
        h = h.masked_fill(r[:, None], 0.0)
    h = torch.sigmoid(z) * h + torch.sigmoid(-z) * c
    new, u, _ = definition(x, h, g, w, s, v, torch.zeros_like(x), None)
    return new, u, h


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(1, 1), (1, 256), (3, 50), (70, 130), (9, 1031), (3, 4096), (5000, 72), (1025, 256)])
def test_one_step(N, D, dtype):
    import torch

    from ac_solver.agents.recurrence import recurrent_step

    print(f"N {N} D {D} {dtype}", flush=True)
    x, y, g, w, s, v, dx, du = make(N, D, dtype, 10)
    p = torch.cat((y * 2, g + 2, dx), dim=1)
    gen = torch.Generator(device="cuda").manual_seed(N)
    h = torch.randn((N, D), device="cuda", generator=gen)
    r = torch.rand(N, device="cuda", generator=gen) < 0.3
    for reset, scale, nxt in ((r, s, v), (None, None, None)):
        want = step_definition(x, p, h, w, scale, nxt, reset)
        new, u, ns = recurrent_step(x, p, h, w, scale, nxt, reset=reset)
        assert_close(new, want[0], dtype, "new")
        assert_close(ns, want[2], "float32", "state")
        assert (u is None) == (nxt is None)
        if nxt is not None:
            assert_close(u, want[1], dtype, "u")
        wide = torch.zeros((N, 3 * D + 5), device="cuda", dtype=x.dtype)  # strided rows, in place
        wide[:, 3:3 + 3 * D] = p
        h2 = h.clone()
        again = recurrent_step(x, wide[:, 3:3 + 3 * D], h2, w, scale, nxt, reset=reset, next_state=h2)
        assert again[2] is h2 and torch.equal(h2, ns) and torch.equal(again[0], new)


def test_a_step_starts_episodes_from_zero_whatever_the_state():
    import torch

    from ac_solver.agents.recurrence import recurrent_step

    x, y, g, w, s, v, dx, du = make(4, 60, "float32", 12)
    p = torch.cat((y, g, dx), dim=1)
    h = torch.full((4, 60), float("nan"), device="cuda")
    new, u, ns = recurrent_step(x, p, h, w, s, v, reset=torch.ones(4, dtype=torch.bool, device="cuda"))
    want = recurrent_step(x, p, torch.zeros_like(h), w, s, v)
    assert all(torch.equal(a, b) for a, b in zip((new, u, ns), want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [2, 8, 13, 17])
def test_many_narrow_rows(D, dtype):
    check(140001, D, dtype)


def test_offsets_past_32_bits():
    """2.16e9 values a tensor: rows do not depend on each other, so the last ones have the bits they have alone; gradients only behind the last 100
    rows make the sums over the rows theirs"""
    import torch

    from ac_solver.agents.block_norm import block_output_backward, block_output_forward

    M, D, some = (1 << 21) + 5, 1030, slice(-100, None)
    x, y, g, w, s, v, dx, du = make(M, D, "bfloat16", 3, "contiguous")
    assert x.numel() > 1 << 31
    dx[:-100], du[:-100] = 0, 0
    new, u, stats = block_output_forward(x, y, g, w, s, v, EPS)
    grads = block_output_backward(dx, du, x, y, g, w, s, v, stats)
    last = [t[some] for t in (x, y, g)]
    new1, u1, stats1 = block_output_forward(*last, w, s, v, EPS)
    grads1 = block_output_backward(dx[some], du[some], *last, w, s, v, stats1)
    assert torch.equal(new[some], new1) and torch.equal(u[some], u1) and torch.equal(stats[some], stats1)
    assert all(torch.equal(a[some], b) for a, b in zip(grads[:3], grads1[:3]))
    assert not any(bool(a[:-100].any()) for a in grads[:3])
    ops = [*last, w, s, v]
    wn, _, wg = definition(*ops, dx[some], du[some])
    for name, got, want, sums in zip(("weight", "scale", "next_weight"), grads[3:], wg[3:], magnitudes(wn, *ops, dx[some], du[some])):
        assert_close(got, want, "float32", "d " + name, sums=sums)


def test_a_step_past_32_bits_of_offset():
    import torch

    from ac_solver.agents.recurrence import recurrent_step

    N, D = 2900000, 256
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((N, D), device="cuda", generator=g, dtype=torch.bfloat16)
    p = torch.randn((N, 3 * D), device="cuda", generator=g, dtype=torch.bfloat16)
    h = torch.randn((N, D), device="cuda", generator=g)
    r = torch.rand(N, device="cuda", generator=g) < 0.1
    w = torch.rand(D, device="cuda", generator=g)
    assert p.numel() > 1 << 31
    out = recurrent_step(x, p, h, w, w, w, reset=r)
    for part in (slice(0, 1000), slice(-1000, None)):
        for a, b in zip(out, recurrent_step(x[part], p[part], h[part], w, w, w, reset=r[part])):
            assert torch.equal(a[part], b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1104, 2050, 2712, 3302, 4096])
def test_wide_rows_walk_the_grid(D, dtype):
    """more rows than workgroups, of every size that a wide row takes"""
    check(3001, D, dtype)
