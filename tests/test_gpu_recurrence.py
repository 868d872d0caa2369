"""gated_scan (csrc/acx_scan.hip): the recurrence and its gradient against the definition in float64, at the lengths, widths, strides and
resets where a segment, a wave's share or a chunk of the steps ends; its refusals are in test_recurrence_cpu.py."""
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")


def inputs(T, N, D, dtype, seed, reset=True, state=True, layout="contiguous"):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def make(scale, shift=0.0):
        x = torch.randn((T, N, D), device="cuda", generator=g) * scale + shift
        return x.to(dt)

    c, z, dh = make(1.0), make(1.5, 2.0), make(0.5)
    if layout == "slices":  # slices of one projection, as the agent has them
        p = torch.empty((T, N, 3 * D + 1), device="cuda", dtype=dt)
        p[..., :D], p[..., D:2 * D] = c, z
        c, z = p[..., :D], p[..., D:2 * D]
    elif layout == "rows first":  # [rows, steps, features] in memory
        c, z, dh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (c, z, dh))
    r = (torch.rand((T, N), device="cuda", generator=g) < 0.1) if reset else None
    s = torch.randn((N, D), device="cuda", generator=g) if state else None
    dl = torch.randn((N, D), device="cuda", generator=g) * 0.5 if state else None
    return c, z, r, s, dh, dl


def definition(c, z, r, s, dh, dl):
    """hidden, last, gradients in float64, step by step"""
    import torch

    c, z, dh = c.double(), z.double(), dh.double()
    T = c.shape[0]
    f, k = torch.sigmoid(z), torch.sigmoid(-z)
    h = torch.zeros_like(c[0]) if s is None else s.double()
    hs, before = [], []
    for t in range(T):
        if r is not None:
            h = h.masked_fill(r[t, :, None], 0.0)
        before.append(h)
        h = f[t] * h + k[t] * c[t]
        hs.append(h)
    x = torch.zeros_like(c[0]) if dl is None else dl.double()
    dc, dz = [None] * T, [None] * T
    for t in range(T - 1, -1, -1):
        G = dh[t] + x
        dc[t] = k[t] * G
        dz[t] = f[t] * k[t] * (before[t] - c[t]) * G
        x = f[t] * G
        if r is not None:
            x = x.masked_fill(r[t, :, None], 0.0)
    return torch.stack(hs), h, torch.stack(dc), torch.stack(dz), x


def assert_close(got, want, dtype, what, top=None):
    """Tolerance: one rounding to the output's type, |want| eps / 2, plus the float32 arithmetic in front of it.  That arithmetic adds up at most
    sum of f^j ~ 1 / (1 - f) terms that matter, with a relative error of a few 2^-24 each, of values no larger than the largest one: 64 * 2^-24
    of the largest magnitude of the tensor covers forty operations on each of the terms that have not decayed."""
    import torch

    top = float(want.abs().max()) if top is None else top
    eps = torch.finfo(getattr(torch, dtype)).eps / 2
    err = (got.double() - want).abs()
    tiny = torch.finfo(getattr(torch, dtype)).smallest_normal * eps if dtype == "float16" else 0.0
    lim = want.abs() * eps * (1 + 2 ** -7) + top * 64 * 2.0 ** -24 + tiny
    bad = err > lim
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {err.numel()} off, worst {float((err - lim).max())} beyond the tolerance"


def check(T, N, D, dtype, seed=0, **kw):
    import torch

    from ac_solver.agents.recurrence import gated_scan

    c, z, r, s, dh, dl = inputs(T, N, D, dtype, seed, **kw)
    print(f"T {T} N {N} D {D} {dtype} {kw}", flush=True)
    leaves = [t.detach().requires_grad_() for t in ([c, z] if s is None else [c, z, s])]
    hidden, last = gated_scan(leaves[0], leaves[1], reset=r, state=leaves[2] if s is not None else None)
    assert hidden.dtype == c.dtype and last.dtype == torch.float32 and hidden.is_contiguous()
    outs, gouts = ([hidden, last], [dh, dl]) if s is not None else ([hidden], [dh])
    grads = torch.autograd.grad(outs, leaves, gouts)
    want = definition(c, z, r, s, dh, dl)
    assert_close(hidden, want[0], dtype, "hidden")
    assert_close(last, want[1], "float32", "last")
    gtop = float(want[2].abs().max()) + float(dh.abs().max()) * 4  # (G itself, before the factor 1 - f, can be larger than dc)
    assert_close(grads[0], want[2], dtype, "d candidate", gtop)
    assert_close(grads[1], want[3], dtype, "d gate", gtop * 4)
    if s is not None:
        assert_close(grads[2], want[4], "float32", "d state", gtop)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 255, 257, 600])
def test_lengths(T, dtype):
    check(T, 3, 70, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(1, 1), (1, 2), (5, 1), (3, 33), (2, 64), (1, 129), (7, 130), (2, 1031)])
def test_widths(N, D, dtype):
    check(37, N, D, dtype, reset=N % 2 == 1, state=D % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["slices", "rows first"])
@pytest.mark.parametrize("D", [50, 63])
def test_strides(D, layout, dtype):
    check(70, 9, D, dtype, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_wave_over_all_steps(dtype):
    check(50, 1030, 256, dtype)  # channels enough for W = 1 (2048 groups and more)
    check(35, 520, 130, dtype, state=False)


@pytest.mark.parametrize("T", [4096, 5003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_chunks_of_a_long_sequence(T, dtype):
    check(T, 2, 66, dtype)
    check(T, 1, 1, dtype, reset=False)


def test_resets_cut_infinities_and_nans_off():
    """what an episode left behind, infinite or NaN, does not reach the next one; gradients of the steps before are those of a cut"""
    import torch

    from ac_solver.agents.recurrence import gated_scan

    for T in (40, 4100):  # within one launch; through the composed chunks
        c, z, _, s, dh, dl = inputs(T, 2, 64, "float32", 3)
        r = torch.zeros((T, 2), dtype=torch.bool, device="cuda")
        r[T // 2] = True
        s[0], s[1] = float("inf"), float("nan")
        c[3, 0] = float("nan")
        hidden, last = gated_scan(c, z, reset=r, state=s)
        assert not torch.isfinite(hidden[0]).any()
        fresh, fresh_last = gated_scan(c[T // 2:], z[T // 2:])
        assert torch.isfinite(hidden[T // 2:]).all() and torch.isfinite(last).all()
        # (cut into other segments: other roundings)
        assert float((hidden[T // 2:] - fresh).abs().max()) < 64 * 2.0 ** -24 * float(fresh.abs().max())
        assert float((last - fresh_last).abs().max()) < 64 * 2.0 ** -24 * float(fresh.abs().max())


def test_gates_at_the_ends_of_their_range():
    """z = +-infinity, +-200, 0: f is exactly 1, 0 and 1 / 2, and 1 - f keeps its accuracy where f rounds to 1"""
    import torch

    from ac_solver.agents.recurrence import gated_scan

    z = torch.tensor([float("inf"), -float("inf"), 200.0, -200.0, 0.0, -0.0, 20.0, -20.0], device="cuda").view(1, 1, -1)
    c = torch.full_like(z, 3.0)
    s = torch.full((1, 8), 5.0, device="cuda")
    hidden, _ = gated_scan(c, z, state=s)
    want = (torch.sigmoid(z.double()) * 5 + torch.sigmoid(-z.double()) * 3)[0]
    assert float((hidden[0].double() - want).abs().max()) <= 5 * 2.0 ** -22
    hidden, _ = gated_scan(c, z)  # state 0: h = (1 - f) c alone
    want = torch.sigmoid(-z.double()) * 3
    ok = (hidden.double() - want).abs() <= want * 8 * 2.0 ** -24 + 1e-37
    assert bool(ok.all()), (hidden, want)


def test_gradient_against_differences():
    """central differences of the kernel's own forward pass in float32: step 2^-6 on values of order one leaves h^2 / 6 f''' ~ 1e-4 and
    rounding 2^-24 / 2^-6 * |sum|"""
    import torch

    from ac_solver.agents.recurrence import gated_scan

    c, z, r, s, dh, dl = inputs(20, 2, 5, "float32", 11)
    leaves = [t.detach().clone().requires_grad_() for t in (c, z, s)]

    def loss(c, z, s):
        h, last = gated_scan(c, z, reset=r, state=s)
        return (h.double() * dh.double()).sum() + (last.double() * dl.double()).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    g = torch.Generator(device="cuda").manual_seed(5)
    for k in range(3):
        for _ in range(6):
            e = torch.zeros_like(leaves[k])
            i = int(torch.randint(0, e.numel(), (1,), device="cuda", generator=g))
            e.view(-1)[i] = 2.0 ** -6
            args = [t.detach() for t in leaves]
            up, down = list(args), list(args)
            up[k], down[k] = args[k] + e, args[k] - e
            num = float((loss(*up) - loss(*down)) / 2 ** -5)
            assert abs(num - float(grads[k].view(-1)[i])) < 2e-3


def test_only_what_is_asked_for_is_differentiated():
    import torch

    from ac_solver.agents.recurrence import gated_scan

    c, z, r, s, dh, dl = inputs(18, 2, 8, "float32", 2)
    want = definition(c, z, r, s, torch.zeros_like(dh), dl)
    c2 = c.clone().requires_grad_()
    _, last = gated_scan(c2, z, reset=r, state=s)  # only the last state is used
    (g,) = torch.autograd.grad(last, [c2], dl)
    assert_close(g, want[2], "float32", "d candidate of the last state", 4.0)
    hidden, _ = gated_scan(c2, z, reset=r, state=s)
    (g,) = torch.autograd.grad(hidden.sum(), [c2])  # an expanded gradient: no strides at all
    want = definition(c, z, r, s, torch.ones_like(dh), None)
    assert_close(g, want[2], "float32", "d candidate of a sum", 40.0)
    with torch.no_grad():
        assert not gated_scan(c2, z)[0].requires_grad


def test_other_streams_and_repeated_calls_agree():
    import torch

    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    c, z, r, s, dh, dl = inputs(4100, 2, 66, "bfloat16", 8)
    first = gated_scan_forward(c, z, r, s)
    grads = gated_scan_backward(dh, dl, c, z, r, first[2])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            again = gated_scan_forward(c, z, r, s)
            g2 = gated_scan_backward(dh, dl, c, z, r, again[2])
        here = gated_scan_forward(c, z, r, s)
        side.synchronize()
        for a, b, d in zip(first + grads, again + g2, here):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(first, here))


def test_a_captured_pass_replays():
    """forward and backward captured into one graph, replayed on new inputs with eager calls between the replays"""
    import torch

    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    c, z, r, s, dh, dl = inputs(4100, 2, 66, "float32", 8)
    gated_scan_forward(c, z, r, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hidden, last, bounds = gated_scan_forward(c, z, r, s)
        grads = gated_scan_backward(dh, dl, c, z, r, bounds)
    for seed in (1, 2, 3):
        for dst, src in zip((c, z, r, s, dh, dl), inputs(4100, 2, 66, "float32", seed)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want = gated_scan_forward(c, z, r, s)
        wg = gated_scan_backward(dh, dl, c, z, r, want[2])
        for a, b in zip((hidden, last, bounds) + grads, want + wg):
            assert torch.equal(a, b)


def test_the_gradient_of_the_gradient_is_refused_not_zero():
    import torch

    from ac_solver.agents.block_norm import block_output
    from ac_solver.agents.recurrence import gated_scan, recurrent_block

    c, z, r, s, dh, dl = inputs(6, 2, 8, "float32", 2)
    leaves = [t.clone().requires_grad_() for t in (c, z)]
    w = torch.ones(8, device="cuda", requires_grad=True)
    p = torch.cat((c, z, dh), dim=-1).requires_grad_()
    for out, wrt in ((gated_scan(*leaves)[0], leaves), (block_output(leaves[0], leaves[1], None, w, w, w)[1], leaves + [w]),
                     (recurrent_block(leaves[0], p, None, w, w, w)[1], [leaves[0], p, w])):
        first = torch.autograd.grad(out.square().sum(), wrt, create_graph=True)
        assert all(g.requires_grad for g in first)
        with pytest.raises(RuntimeError):  # (the leaves are not reached at all)
            torch.autograd.grad(sum(g.sum() for g in first), wrt, retain_graph=True)
        with pytest.raises(RuntimeError, match="again"):
            sum(g.sum() for g in first).backward()


def test_two_threads_at_once():
    """calls from two host threads on streams of their own: the interpreter's lock is not held meanwhile, scratch memory is each call's own"""
    import threading

    import torch

    from ac_solver.agents.recurrence import gated_scan

    jobs = [inputs(4100, 2, 66, "float32", k) for k in range(2)]

    def run(c, z, r, s, dh, dl):
        leaves = [t.clone().requires_grad_() for t in (c, z, s)]
        h, last = gated_scan(leaves[0], leaves[1], reset=r, state=leaves[2])
        return [h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (dh, dl))]

    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = run(*jobs[k])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        bad.append(k)
        except BaseException as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_targets_of_gradients_are_checked():
    import torch

    from ac_solver.agents.block_norm import block_output_backward, block_output_forward
    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    c, z, r, s, dh, dl = inputs(6, 3, 8, "float32", 2)
    _, _, bounds = gated_scan_forward(c, z, r, s)
    one = torch.zeros(1, 3, 8, device="cuda").expand(6, 3, 8)
    with pytest.raises(ValueError, match="overlap"):
        gated_scan_backward(dh, dl, c, z, r, bounds, out=(one, torch.empty_like(c)))
    with pytest.raises(ValueError, match="contiguous last axis"):
        gated_scan_backward(dh, dl, c, z, r, bounds, out=(torch.empty_like(c), torch.empty(6, 8, 3, device="cuda").transpose(1, 2)))
    w = torch.ones(8, device="cuda")
    _, _, stats = block_output_forward(c, z, dh, w, w, w)
    with pytest.raises(ValueError, match="overlap"):
        block_output_backward(c, c, c, z, dh, w, w, w, stats, d_gate_out=one)
    wanted = gated_scan_backward(dh, dl, c, z, r, bounds)
    buffer = torch.zeros(6, 3, 25, device="cuda")
    ok = (buffer[..., :8], buffer[..., 8:16])
    for a, b in zip(gated_scan_backward(dh, dl, c, z, r, bounds, out=ok), wanted):
        assert torch.equal(a, b)
    assert torch.equal(ok[0], wanted[0]) and torch.equal(ok[1], wanted[1]) and not buffer[..., 16:].any()
    crossed = torch.empty(400, device="cuda").as_strided((6, 3, 8), (16, 16, 1))  # (steps and rows that meet)
    woven = torch.empty(400, device="cuda").as_strided((6, 3, 8), (16, 8, 1))
    for bad in (crossed, woven):
        with pytest.raises(ValueError, match="overlap"):
            gated_scan_backward(dh, dl, c, z, r, bounds, out=(torch.empty_like(c), bad))
    for bad in ((c, torch.empty_like(c)), (torch.empty_like(c), dh), (buffer[..., :8], buffer[..., 7:15]), (buffer[..., :8], buffer[..., :8])):
        with pytest.raises(ValueError, match="in the memory of another operand"):
            gated_scan_backward(dh, dl, c, z, r, bounds, out=bad)
    with pytest.raises(ValueError, match="in the memory of another operand"):
        block_output_backward(c, c, c, z, dh, w, w, w, stats, d_gate_out=dh)
    with pytest.raises(ValueError, match="bounds has the shape"):
        gated_scan_backward(dh, dl, c, z, r, bounds[1:])
    with pytest.raises(ValueError, match="stats has the shape"):
        block_output_backward(c, c, c, z, dh, w, w, w, stats[1:])


def test_tensors_of_another_device_than_the_current_one():
    """(one GPU: the current device is the tensors' own; a tensor elsewhere is refused by name)"""
    import torch

    from ac_solver.agents.recurrence import gated_scan

    c, z, r, s, dh, dl = inputs(6, 3, 8, "float32", 2)
    with pytest.raises(ValueError, match="state lives on cpu"):
        gated_scan(c, z, state=s.cpu())
    with pytest.raises(ValueError, match="gate is"):
        gated_scan(c, z.cpu())
    if torch.cuda.device_count() > 1:
        with torch.cuda.device(1):
            assert torch.equal(gated_scan(c, z, r, s)[0], gated_scan(c, z, r, s)[0])


def test_in_place_changes_of_what_autograd_kept_are_noticed():
    import torch

    from ac_solver.agents.recurrence import gated_scan

    c, z, r, s, dh, dl = inputs(6, 3, 8, "float32", 2)
    c.requires_grad_()
    z2 = z * 1.0
    h, _ = gated_scan(c, z2)
    z2.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        h.sum().backward()


def test_tensors_larger_than_the_caches():
    """over 256 MiB a tensor the accesses go past the caches: the same bits as in halves that do not"""
    import torch

    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    c, z, r, s, dh, dl = inputs(20, 13200, 257, "float32", 4)
    whole = gated_scan_forward(c, z, r, s)
    grads = gated_scan_backward(dh, dl, c, z, r, whole[2])
    for part in (slice(0, 6600), slice(6600, 13200)):
        cut = lambda t: t[:, part] if t.dim() == 3 or t.dtype == torch.bool else t[part]  # noqa: E731
        args = [cut(c), cut(z), cut(r).contiguous(), cut(s).contiguous()]
        half = gated_scan_forward(*args)
        g = gated_scan_backward(cut(dh), cut(dl).contiguous(), args[0], args[1], args[2], half[2])
        assert torch.equal(cut(whole[0]), half[0]) and torch.equal(cut(whole[1]), half[1])
        assert all(torch.equal(cut(a), b) for a, b in zip(grads, g))


def test_offsets_past_32_bits():
    """slices of a projection of 2.15e9 values; the same bits as in halves (a lane walks all steps in either)"""
    import torch

    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    T, N, D = 20, 140000, 256
    c, z, r, s, dh, dl = inputs(T, N, D, "bfloat16", 6, layout="slices")
    assert T * c.stride(0) > 1 << 31
    d_projected = torch.zeros(T, N, 3 * D, device="cuda", dtype=torch.bfloat16)
    whole = gated_scan_forward(c, z, r, s)
    grads = gated_scan_backward(dh, dl, c, z, r, whole[2], out=(d_projected[..., :D], d_projected[..., D:2 * D]))
    assert not bool(d_projected[..., 2 * D:].any())
    for part in (slice(0, 70000), slice(70000, N)):
        args = [c[:, part], z[:, part], r[:, part].contiguous(), s[part].contiguous()]
        half = gated_scan_forward(*args)
        g = gated_scan_backward(dh[:, part], dl[part].contiguous(), args[0], args[1], args[2], half[2])
        assert torch.equal(whole[0][:, part], half[0]) and torch.equal(whole[1][part], half[1])
        assert torch.equal(grads[0][:, part], g[0]) and torch.equal(grads[1][:, part], g[1]) and torch.equal(grads[2][part], g[2])


def test_steps_past_32_bits_of_offset():
    """8.4e6 steps of 280 channels, cut into chunks: the first and the last steps against the definition of 1000 of them.  What 600 steps hand on is the
    product of 600 gates: sigmoid of normal numbers around 2 with a deviation of 1.5 has a mean logarithm below -0.2 (at the mean it is -0.127, and the
    logarithm of the sigmoid is concave, with variance 2.25 taking it to about -0.25), so e^-120, far below float32's 2^-24."""
    import torch

    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    T, N, D = (1 << 23) + 3, 4, 70
    c, z, _, s, dh, dl = inputs(T, N, D, "bfloat16", 7, reset=False)
    assert c.numel() > 1 << 31
    hidden, last, bounds = gated_scan_forward(c, z, None, s)
    dc, dz, ds = gated_scan_backward(dh, dl, c, z, None, bounds)
    want = definition(c[:1000], z[:1000], None, s, dh[:1000], None)
    gtop = float(want[2].abs().max()) + float(dh[:1000].abs().max()) * 4
    assert_close(hidden[:1000], want[0], "bfloat16", "first hidden")
    assert_close(dc[:400], want[2][:400], "bfloat16", "first d candidate", gtop)
    assert_close(dz[:400], want[3][:400], "bfloat16", "first d gate", gtop * 4)
    assert_close(ds, want[4], "float32", "d state", gtop)
    want = definition(c[-1000:], z[-1000:], None, None, dh[-1000:], dl)
    assert_close(hidden[-400:], want[0][-400:], "bfloat16", "last hidden")
    assert_close(last, want[1], "float32", "last")
    assert_close(dc[-400:], want[2][-400:], "bfloat16", "last d candidate", gtop)
    assert_close(dz[-400:], want[3][-400:], "bfloat16", "last d gate", gtop * 4)


def test_forward_mode_is_refused():
    """a tangent on an operand, or on the gradient that a backward pass starts from, is not dropped silently"""
    import torch
    import torch.autograd.forward_ad as forward_ad

    from ac_solver.agents.activation8 import linear8
    from ac_solver.agents.block_norm import block_input, block_output, block_output_backward, block_output_forward
    from ac_solver.agents.recurrence import gated_scan, gated_scan_backward, gated_scan_forward, recurrent_block

    c, z, r, s, dh, dl = inputs(6, 2, 8, "float32", 2)
    w, p = torch.ones(8, device="cuda"), torch.cat((c, z, dh), dim=-1)
    calls = ((lambda t: gated_scan(t, z)[0], c), (lambda t: gated_scan(c, z, state=t)[0], s), (lambda t: block_output(c, t, z, w, w, w)[0], dh), (lambda t: block_output(c, z, dh, t)[0], w),
             (lambda t: block_input(t, w), c), (lambda t: recurrent_block(c, t, None, w)[0], p), (lambda t: linear8(t, torch.ones(3, 8, device="cuda")), c))
    for f, t in calls:
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                f(forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(NotImplementedError):
                f(forward_ad.make_dual(t.clone().requires_grad_(), torch.ones_like(t)))
        leaf = t.clone().requires_grad_()
        out = f(leaf)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            if t.dim() == 3 and out.shape[-1] == 3:  # (linear8's gradient of x is torch's own, which has a tangent: take the weight's)
                weight = torch.ones(3, 8, device="cuda", requires_grad=True)
                out, leaf = linear8(t, weight), weight
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
    _, _, bounds = gated_scan_forward(c, z, r, s)
    _, _, stats = block_output_forward(c, z, dh, w, w, w)
    for f, args, places in ((gated_scan_backward, [dh, dl, c, z, None, bounds], (0, 1, 5)), (block_output_backward, [dh, dh, c, z, dh, w, w, w, stats], (0, 1, 8))):
        for k in places:
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
                f(*args[:k], forward_ad.make_dual(args[k], torch.ones_like(args[k])), *args[k + 1:])


def test_the_states_of_a_scan_do_not_replace_each_other_in_place():
    """of the C functions (from Python the results are new tensors): the last state over the first, the first state's gradient over the last one's, whole or in part,
    where other workgroups may still have to read; buffers side by side are taken"""
    import torch

    from ac_solver import _acx
    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward

    T, N, D = 4100, 2, 66
    c, z, r, s, dh, dl = inputs(T, N, D, "float32", 8)
    hidden, last, bounds = gated_scan_forward(c, z, r, s)
    dc, dz, ds = gated_scan_backward(dh, dl, c, z, r, bounds)
    work = torch.empty(_acx.lib.acx_scan_workspace_bytes(T, N, D, _acx.F32), dtype=torch.uint8, device="cuda")
    assert work.numel()
    both = torch.zeros(2 * N * D, device="cuda")
    st = N * D, D
    stream = torch.cuda.current_stream().cuda_stream

    def forward(place):
        both[:N * D] = s.view(-1)
        return _acx.lib.acx_scan_forward(c.data_ptr(), *st, z.data_ptr(), *st, _acx.F32, r.data_ptr(), both.data_ptr(), T, N, D, torch.empty_like(hidden).data_ptr(),
                                         both.data_ptr() + 4 * place, None, work.data_ptr(), work.numel(), stream)

    def backward(place):
        both[:N * D] = dl.view(-1)
        return _acx.lib.acx_scan_backward(c.data_ptr(), *st, z.data_ptr(), *st, dh.data_ptr(), *st, _acx.F32, r.data_ptr(), bounds.data_ptr(), both.data_ptr(), T, N, D,
                                          torch.empty_like(dc).data_ptr(), *st, torch.empty_like(dz).data_ptr(), *st, both.data_ptr() + 4 * place, work.data_ptr(), work.numel(), stream)

    for call, want in ((forward, last), (backward, ds)):
        for place in (0, 1, N * D - 1):
            assert call(place) == _acx.E_INVAL and b"in place" in _acx.lib.acx_last_error()
        assert call(N * D) == _acx.OK
        torch.cuda.synchronize()
        assert torch.equal(both[N * D:].view(N, D), want)


def test_writing_into_a_callers_tensor_is_noticed_by_autograd():
    """what another function kept of a tensor that a result is then written into is not what it was: its gradient is refused, as after torch's own in-place functions"""
    import torch

    from ac_solver.agents.block_norm import block_output_backward, block_output_forward
    from ac_solver.agents.recurrence import gated_scan_backward, gated_scan_forward, recurrent_step

    c, z, r, s, dh, dl = inputs(6, 3, 8, "float32", 2)
    w, k = torch.ones(8, device="cuda"), torch.ones(8, device="cuda", requires_grad=True)
    _, _, bounds = gated_scan_forward(c, z, r, s)
    _, _, stats = block_output_forward(c, z, dh, w, w, w)
    p = torch.cat((c, z, dh), dim=-1)[0]
    memory, a, b, g = s.clone(), torch.zeros_like(c), torch.zeros_like(c), torch.zeros_like(c)
    for target, write in ((memory, lambda: recurrent_step(c[0], p, memory, w, next_state=memory)), (a, lambda: gated_scan_backward(dh, dl, c, z, r, bounds, out=(a, b))),
                          (b, lambda: gated_scan_backward(dh, dl, c, z, r, bounds, out=(a, b))), (g, lambda: block_output_backward(c, c, c, z, dh, w, w, w, stats, d_gate_out=g))):
        out = (target * k).sum()
        write()
        with pytest.raises(RuntimeError, match="inplace"):
            out.backward()
    with torch.inference_mode():  # (tensors that count no changes)
        state = s.clone()
        recurrent_step(c[0], p, state, w, next_state=state)


VARIANTS = {  # (steps, rows, features): how plan_of cuts them
    "16 waves, 5 tiles, the last one ragged": (1046, 19, 846),
    "16 waves, 3 tiles": (523, 19, 846),
    "two channels a lane, 4 waves, 4 tiles, an odd width": (201, 399, 151),
    "two channels a lane, 4 waves, 2 tiles, an even width": (128, 399, 150),
    "two channels a lane, 4 waves, rows of three lanes": (90, 9000, 5),
    "two channels a lane, one wave, an odd width": (37, 1030, 257),
    "two channels a lane, one wave, rows of two lanes": (20, 66000, 3),
    "one channel a lane, one wave, rows of one lane": (10, 9000, 1),
    "one channel a lane, chunks, rows of 7 lanes": (5003, 9, 7),
    "one channel a lane, 8 waves, 3 tiles, no chunks": (300, 40000, 1),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("variant", list(VARIANTS))
def test_every_way_of_cutting_the_work(variant, dtype):
    check(*VARIANTS[variant], dtype, seed=3)
    check(*VARIANTS[variant], dtype, seed=4, layout="slices", state=False)


def test_second_derivatives_are_refused_wherever_they_are_asked_for():
    """gradients that were taken with create_graph hang on all operands, also on those that the gradient itself was not kept for: a sum of a loss and a penalty on its
    gradient, a Hessian, or a penalty alone with operands that may be unused all raise, none leaves its second-order term out; what does not depend on
    the gradient is not in the way"""
    import torch

    from ac_solver.agents.activation8 import linear8
    from ac_solver.agents.block_norm import block_input, block_output
    from ac_solver.agents.recurrence import gated_scan, recurrent_block

    c, z, r, s, dh, dl = inputs(6, 2, 8, "float32", 2)
    w, p, m = torch.rand(8, device="cuda"), torch.cat((c, z, dh), dim=-1), torch.randn(3, 8, device="cuda")
    calls = ((lambda c, z, s: gated_scan(c, z, r, s), (c, z, s)), (lambda x, y, g, w, s, v: block_output(x, y, g, w, s, v), (c, z, dh, w, w + 1, w + 2)), (lambda x, w: (block_input(x, w),), (c, w)),
             (lambda x, p, s, w, a, v: recurrent_block(x, p, s, w, a, v), (c, p, s, w, w + 1, w + 2)), (lambda x, m, b: (linear8(x, m, b),), (c, m, torch.ones(3, device="cuda"))))
    for f, operands in calls:
        for k in range(len(operands)):
            leaves = [t.clone().requires_grad_() for t in operands]
            other = torch.ones((), device="cuda", requires_grad=True)
            outs = f(*leaves)
            loss = sum(o.square().sum() for o in outs) * other
            first = torch.autograd.grad(loss, leaves, create_graph=True)
            penalty = first[k].square().sum()
            assert all(g.requires_grad for g in first)
            for total, unused in ((penalty, True), (penalty + sum(t.square().sum() for t in leaves), False)):
                for leaf in leaves:
                    with pytest.raises(RuntimeError, match="again"):
                        torch.autograd.grad(total, [leaf], retain_graph=True, allow_unused=unused)
            with pytest.raises(RuntimeError, match="again"):
                (penalty + sum(t.square().sum() for t in leaves)).backward(retain_graph=True)
            apart = torch.ones((), device="cuda", requires_grad=True)
            assert float(torch.autograd.grad(penalty.detach() + 2 * apart, apart)[0]) == 2
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.functional.hessian(lambda t: gated_scan(t, z)[0].square().sum(), c)
