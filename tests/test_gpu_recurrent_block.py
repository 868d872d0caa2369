"""recurrent_block (a block of the recurrent agent over a rollout, one node of autograd) against its formulas in float64: values, and the gradients from
new, u and the last state, with everything autograd kept exact or in 8 bits."""
import pytest

from tests.test_gpu_block_norm import assert_close
from tests.test_gpu_recurrence import definition as scan_definition

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")
EPS = 1e-6
SEGMENT = 16  # steps between two states that the forward pass keeps


def block_end(x, y, g, w, s, v, stats=None, d_new=None, d_u=None):
    """new, u, the reciprocal roots of the two norms (`stats`: others to use), and by the formulas the gradients of x, y, g, w, s, v with the magnitudes that
    go into the last three: sums over the rows of products, with the terms of a difference taken one by one (they can cancel, their roundings do not)"""
    import torch

    x, y, g, w, s, v = (None if t is None else t.double() for t in (x, y, g, w, s, v))
    s = torch.ones_like(w) if s is None else s
    inverse = lambda t: 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)  # noqa: E731
    ry = inverse(y) if stats is None else stats[0]
    yn, sig = y * ry, torch.sigmoid(g)
    a, n = g * sig, yn * w
    new = x + s * a * n
    rx = inverse(new) if stats is None else stats[1]
    u = None if v is None else new * rx * v
    if d_new is None:
        return new, u, (ry, rx)
    xn, t = new * rx, (torch.zeros_like(x) if v is None else d_u.double() * v)
    dx = d_new.double() + rx * (t - xn * (t * xn).mean(-1, keepdim=True))
    dn = dx * s * a
    dy = ry * (dn * w - yn * (dn * w * yn).mean(-1, keepdim=True))
    dg = dx * s * n * (sig + a * (1 - sig))
    wide = (x.abs() + (s * a * n).abs()) * rx
    top = d_new.double().abs() + rx * (t.abs() + wide * (t.abs() * wide).mean(-1, keepdim=True))
    rows = lambda t: t.flatten(0, -2).sum(0)  # noqa: E731
    du = torch.zeros_like(x) if v is None else d_u.double()
    sums = [rows(dn * yn), rows(dx * a * n), rows(du * xn)]
    magnitudes = [rows(top * (s * a * yn).abs()), rows(top * (a * n).abs()), rows(du.abs() * wide)]
    return dx, dy, dg, sums, magnitudes


def scan_gradient(c, z, r, fronts, dh, dl):
    """gradients of c, z and the state from those of hidden and last, the states in front of every segment given"""
    import torch

    c, z = c.double(), z.double()
    f, k = torch.sigmoid(z), torch.sigmoid(-z)
    live = (~r).double().unsqueeze(-1)
    before = []
    for t in range(c.shape[0]):
        b = live[t] * (fronts[t // SEGMENT] if t % SEGMENT == 0 else h)  # noqa: F821
        before.append(b)
        h = f[t] * b + k[t] * c[t]  # noqa: F841
    X = torch.zeros_like(c[0]) if dl is None else dl.double()
    dc, dz = torch.empty_like(c), torch.empty_like(c)
    for t in range(c.shape[0] - 1, -1, -1):
        G = dh[t] + X
        dc[t], dz[t] = k[t] * G, f[t] * k[t] * (before[t] - c[t]) * G
        X = live[t] * f[t] * G
    return dc, dz, X


def check(T, N, D, dtype, scale=True, nxt=True, last_only=False, packed=False, seed=0):
    """Tolerances: values and gradients of the block's end as in its own test (assert_close there).  The gradient that it hands to the scan is rounded once to the
    activations' type and carries the same float32 errors; the scan is linear in it with coefficients of one sign, so what becomes of these errors is the
    scan's gradient of their bounds.  On top of that the scan's own: one rounding, and 64 * 2^-24 of the largest gradient."""
    import torch

    from ac_solver.agents import activation8
    from ac_solver.agents.recurrence import gated_scan_forward, recurrent_block

    print(f"T {T} N {N} D {D} {dtype} scale {scale} next {nxt} last only {last_only} packed {packed}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    normal = lambda *shape, k=1.0, b=0.0: torch.randn(shape, device="cuda", generator=gen) * k + b  # noqa: E731
    x = normal(T, N, D, k=2.0).to(dt)
    p = torch.cat((normal(T, N, D), normal(T, N, D, k=1.5, b=2.0), normal(T, N, D)), -1).to(dt)
    r = torch.rand((T, N), device="cuda", generator=gen) < 0.1
    state, w, s, v = normal(N, D), normal(D, k=0.2, b=1.0), normal(D, k=0.2, b=0.5) if scale else None, normal(D, k=0.2, b=1.0) if nxt else None
    d_new, d_u, d_last = normal(T, N, D, k=0.3).to(dt), normal(T, N, D, k=0.3).to(dt), normal(N, D, k=0.3)
    leaves = [t if t is None else t.clone().requires_grad_() for t in (x, p, state, w, s, v)]
    inner = [leaves[0] * 1.0, leaves[1] * 1.0] if packed else leaves[:2]  # (leaves are kept as they are)
    if packed:
        with activation8.checkpoint8():
            new, u, last = recurrent_block(*inner, leaves[2], *leaves[3:], reset=r, eps=EPS)
    else:
        new, u, last = recurrent_block(*inner, leaves[2], *leaves[3:], reset=r, eps=EPS)
    c, z, g = (p[..., k * D:(k + 1) * D] for k in range(3))
    hidden = gated_scan_forward(c, z, r, state)[0]  # (as the block's end reads it: rounded; tested for itself)
    states, want_last = scan_definition(c, z, r, state, torch.zeros_like(x), None)[:2]
    want_new, want_u, stats = block_end(x, hidden, g, w, s, v)
    assert_close(new, want_new, dtype, "new")
    assert_close(last, want_last, "float32", "last")
    assert (u is None) == (not nxt) and last.dtype == torch.float32
    if nxt:
        assert_close(u, want_u, dtype, "u")
    outs, gs = ([last], [d_last]) if last_only else ([new, u, last], [d_new, d_u, d_last]) if nxt else ([new, last], [d_new, d_last])
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(outs, wanted, gs))
    got = [None if t is None else next(grads) for t in leaves]
    if last_only:
        assert not got[0].any() and not got[3].any() and not any(t is not None and t.any() for t in got[4:]) and not got[1][..., 2 * D:].any()
        dh, sent = torch.zeros_like(want_new), torch.zeros_like(want_new)
    kept = (lambda t: activation8.unpack8(*activation8.pack8(t), t.dtype)) if packed else (lambda t: t)
    xk, pk, hk = kept(x), kept(p), kept(hidden)
    ck, zk, gk = (pk[..., k * D:(k + 1) * D] for k in range(3))
    eps = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * eps if dtype == "float16" else 0.0
    if not last_only:
        dx, dh, dg, sums, magnitudes = block_end(xk, hk, gk, w, s, v, stats, d_new, d_u)
        assert_close(got[0], dx, dtype, "d x", terms=4)
        assert_close(got[1][..., 2 * D:], dg, dtype, "d output gate", terms=4)
        for name, k in (("weight", 0), ("scale", 1), ("next_weight", 2)):
            if got[3 + k] is not None:
                assert_close(got[3 + k], sums[k], "float32", "d " + name, sums=magnitudes[k])
        sent = dh.abs() * eps * (1 + 2 ** -7) + tiny + float(dh.abs().max()) * 4 * 64 * 2.0 ** -24
    fronts = [state.double() if t == 0 else states[t - 1] for t in range(0, T, SEGMENT)]
    dc, dz, ds = scan_gradient(ck, zk, r, fronts, dh, d_last)
    ec, ez, es = (t.abs() for t in scan_gradient(ck, zk, r, fronts, sent, None))
    gtop = float(dc.abs().max()) + float(dh.abs().max()) * 4 + float(d_last.abs().max())
    for name, g1, want, error, top, e in (("candidate", got[1][..., :D], dc, ec, gtop, eps), ("gate", got[1][..., D:2 * D], dz, ez, 4 * gtop, eps), ("state", got[2], ds, es, gtop, 2.0 ** -24)):
        err, lim = (g1.double() - want).abs(), error + want.abs() * e * (1 + 2 ** -7) + tiny + top * 64 * 2.0 ** -24
        assert not bool((err > lim).any()), f"d {name}: worst {float((err - lim).max())} beyond the tolerance"


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("part", [dict(), dict(scale=False), dict(nxt=False), dict(scale=False, nxt=False), dict(last_only=True), dict(last_only=True, nxt=False)])
def test_values_and_gradients(part, dtype, packed):
    check(37, 5, 50, dtype, packed=packed, **part)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,D", [(1, 131, 33), (16, 9, 64), (17, 1, 257), (200, 3, 130), (2000, 1, 64), (33, 399, 150)])
def test_sizes(T, N, D, dtype, packed):
    check(T, N, D, dtype, packed=packed, seed=1)
