"""What the recurrent agent's operators refuse, and how: types, shapes and devices are checked on the host, before any allocation or
launch (no GPU needed)."""
import pytest
import torch

from ac_solver.agents import recurrence as R


def scan_args(T=3, N=2, D=4, dtype=torch.float32):
    return torch.zeros(T, N, D, dtype=dtype), torch.zeros(T, N, D, dtype=dtype)


def test_the_scan_refuses_what_it_cannot_read():
    c, z = scan_args()
    ok = dict(reset=torch.zeros(3, 2, dtype=torch.bool), state=torch.zeros(2, 4))
    with pytest.raises(ValueError, match="GPU"):  # everything in order but the place
        R.gated_scan(c, z, **ok)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        R.gated_scan(c.double(), z.double())
    with pytest.raises(TypeError, match="tensor"):
        R.gated_scan([1.0], z)
    with pytest.raises(ValueError, match="gate is"):
        R.gated_scan(c, z.half())
    with pytest.raises(ValueError, match="gate has the shape"):
        R.gated_scan(c, z[:2])
    with pytest.raises(ValueError, match="steps, rows, features"):
        R.gated_scan(c[0], z[0])
    with pytest.raises(ValueError, match="at least one step"):
        R.gated_scan(c[:0], z[:0])
    with pytest.raises(ValueError, match="reset has the shape"):
        R.gated_scan(c, z, reset=ok["reset"].t())
    with pytest.raises(TypeError, match="reset"):
        R.gated_scan(c, z, reset=torch.zeros(3, 2))
    with pytest.raises(TypeError, match="state"):
        R.gated_scan(c, z, state=torch.zeros(2, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="state has the shape"):
        R.gated_scan(c, z, state=torch.zeros(1, 4))


def test_the_scan_gradient_refuses_what_does_not_fit_its_forward_pass():
    c, z = scan_args()
    with pytest.raises(ValueError, match="GPU"):
        R.gated_scan_backward(c, None, c, z, None, torch.zeros(8))


def test_scan_buffer_sizes():
    from ac_solver import _acx

    assert _acx.lib.acx_scan_bounds_bytes(1, 2, 4) == 32 and _acx.lib.acx_scan_bounds_bytes(17, 2, 4) == 64 and _acx.lib.acx_scan_bounds_bytes(16, 0, 4) == 0
    assert _acx.lib.acx_scan_workspace_bytes(1, 1, 1, _acx.F32) == 0 and _acx.lib.acx_scan_workspace_bytes(1 << 16, 1, 256, _acx.BF16) > 0
    assert _acx.lib.acx_scan_workspace_bytes(32, 131072, 256, _acx.F32) == 0


def test_sizes_that_no_memory_holds_are_no_division_by_zero():
    from ac_solver import _acx

    lib, huge = _acx.lib, 1 << 62
    for T, N, D in ((1000, huge, 64), (1000, 1 << 31, 1 << 20), (huge, 64, 64), (1000, 64, huge), (-1, 4, 4), (1000, -4, 4)):
        assert lib.acx_scan_workspace_bytes(T, N, D, _acx.F32) == 0
        assert lib.acx_scan_bounds_bytes(T, N, D) == 0
    assert lib.acx_scan_workspace_bytes(1000, 4, 64, _acx.I64) == 0
    for M, D in ((huge, 64), (64, huge), (-1, 64), (64, 4097)):
        assert lib.acx_block_workspace_bytes(M, D, _acx.F32) == 0
    for M, O, I in ((1000, huge, 64), (1000, 1 << 32, 1 << 32), (1000, 64, huge), (huge, 64, 64), (1000, 1 << 16, 1 << 16), (0, 64, 64)):
        assert lib.acx_act8_workspace_bytes(M, O, I) == 0
    assert lib.acx_act8_workspace_bytes(1000, 1 << 16, 1 << 13) > 0


def test_the_block_end_refuses_what_it_cannot_read():
    from ac_solver.agents import block_norm as B

    x, w = torch.zeros(5, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        B.block_output(x, x, x, w, w, w)
    with pytest.raises(ValueError, match="GPU"):
        B.block_input(x, w)
    with pytest.raises(ValueError, match="4096"):
        B.block_input(torch.zeros(1, 4097), torch.zeros(4097))
    with pytest.raises(ValueError, match="y has the shape"):
        B.block_output(x, x[:4], x, w)
    with pytest.raises(ValueError, match="gate is"):
        B.block_output(x, x, x.half(), w)
    with pytest.raises(TypeError, match="weight"):
        B.block_output(x, x, x, w.half())
    with pytest.raises(ValueError, match="scale has the shape"):
        B.block_output(x, x, x, w, w[:3])
    with pytest.raises(TypeError, match="weight has to be a tensor"):
        B.block_output(x, x, x, None)
    with pytest.raises(ValueError, match="eps"):
        B.block_input(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        B.block_input(x, w, eps=float("nan"))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        B.block_input(x.to(torch.int8), w)


def test_a_step_refuses_what_it_cannot_read():
    x, p, h, w = torch.zeros(5, 8), torch.zeros(5, 24), torch.zeros(5, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        R.recurrent_step(x, p, h, w, w, w, reset=torch.zeros(5, dtype=torch.bool), next_state=h)
    with pytest.raises(ValueError, match="projected has the shape"):
        R.recurrent_step(x, p[:, :16], h, w)
    with pytest.raises(ValueError, match="rows, features"):
        R.recurrent_step(x[0], p, h, w)
    with pytest.raises(TypeError, match="state"):
        R.recurrent_step(x.half(), p.half(), h.half(), w)
    with pytest.raises(ValueError, match="next_state has to be contiguous"):
        R.recurrent_step(x, p, h, w, next_state=torch.zeros(8, 5).t())
    both = torch.zeros(6, 8)  # (the state itself may be the target, not a part of it, nor anything else that is read)
    for state, target, inputs in ((both[:5], both[1:], x), (h, x, x)):
        with pytest.raises(ValueError, match="next_state lies in the memory"):
            R.recurrent_step(inputs, p, state, w, next_state=target)
    with pytest.raises(TypeError, match="reset"):
        R.recurrent_step(x, p, h, w, reset=torch.zeros(5))
    with pytest.raises(ValueError, match="4096"):
        R.recurrent_step(torch.zeros(1, 4097), torch.zeros(1, 3 * 4097), torch.zeros(1, 4097), torch.zeros(4097))


def test_8_bit_checkpoints_refuse_what_they_cannot_read():
    from ac_solver.agents import activation8 as A

    x, q, e = torch.zeros(5, 40), torch.zeros(5, 40, dtype=torch.int8), torch.zeros(5, 2, dtype=torch.uint8)
    for call in (lambda: A.pack8(x), lambda: A.unpack8(q, e), lambda: A.weight_grad8(x, q, e), lambda: A.linear8(x, torch.zeros(3, 40), torch.zeros(3))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        A.pack8(x.double())
    with pytest.raises(TypeError, match="q has to be"):
        A.unpack8(x, e)
    with pytest.raises(TypeError, match="q has to be a tensor"):
        A.unpack8(None, e)
    with pytest.raises(ValueError, match="exponent has the shape"):
        A.unpack8(q, e[:, :1])
    with pytest.raises(TypeError, match="dtype"):
        A.unpack8(q, e, torch.float64)
    with pytest.raises(ValueError, match="rows in common"):
        A.weight_grad8(x[:4], q, e)
    with pytest.raises(TypeError, match="weight"):
        A.linear8(x, torch.zeros(3, 40).half())
    with pytest.raises(TypeError, match="bias"):
        A.linear8(x, torch.zeros(3, 40), torch.zeros(4))
    with pytest.raises(ValueError, match="weight"):
        A.linear8(x, torch.zeros(3, 41))
    with A.checkpoint8():  # nothing on the CPU is packed
        a = torch.randn(100, 100, requires_grad=True)
        out = torch.tanh(a * 1.0).sum()
    out.backward()
    # (values up to 1, a product and a difference on either side: four roundings of at most 2^-24)
    assert float((a.grad - (1 - torch.tanh(a.detach()) ** 2)).abs().max()) <= 2.0 ** -22


def test_arguments_of_the_recurrent_agent():
    from ac_solver.agents.args import parse_args

    a = parse_args(["--recurrent", "--recurrent-width", "64", "--recurrent-blocks", "3", "--recurrent-dtype", "bfloat16", "--checkpoint-8bit"])
    assert a.recurrent and (a.recurrent_width, a.recurrent_blocks, a.recurrent_dtype, a.checkpoint_8bit) == (64, 3, "bfloat16", True)
    d = parse_args([])
    assert not d.recurrent and not d.checkpoint_8bit
    for bad in (["--recurrent", "--fused-policy"], ["--checkpoint-8bit"], ["--recurrent", "--recurrent-dtype", "float64"]):
        with pytest.raises(AssertionError):
            parse_args(bad)


def test_the_recurrent_agent_needs_a_gpu_and_says_so():
    from types import SimpleNamespace

    from ac_solver.agents.recurrent_agent import RecurrentAgent

    spaces = SimpleNamespace(single_observation_space=SimpleNamespace(shape=(50,)), single_action_space=SimpleNamespace(n=12))
    agent = RecurrentAgent(spaces, 32, 2)
    assert sum(p.numel() for p in agent.parameters()) == 50 * 32 + 32 + 2 * (3 * 32 * 32 + 3 * 32 + 3 * 32) + 32 + 32 * 12 + 12 + 32 + 1
    with pytest.raises(ValueError, match="GPU"):
        agent.act(torch.zeros(4, 50), torch.zeros(4, dtype=torch.bool), agent.initial_state(4))
    with pytest.raises(ValueError, match="at least one"):
        RecurrentAgent(spaces, 32, 0)
    with pytest.raises(ValueError, match="4096"):
        RecurrentAgent(spaces, 4097, 1)
    with pytest.raises(ValueError, match="steps, rows, features"):
        R.recurrent_block(torch.zeros(4, 8), torch.zeros(4, 24), None, torch.ones(8))
    with pytest.raises(ValueError, match="projected has the shape"):
        R.recurrent_block(torch.zeros(2, 4, 8), torch.zeros(2, 4, 16), None, torch.ones(8))


def test_checkpoint8_holds_no_graph_that_nobody_else_holds():
    """an output that its own node keeps (tanh) goes with the last reference to it, also where no backward pass runs; second derivatives pass through"""
    import gc
    import weakref

    from ac_solver.agents.activation8 import checkpoint8

    a = torch.randn(64, 4, requires_grad=True)
    with checkpoint8():
        y = torch.tanh(a * 1.0)
    gone = weakref.ref(y)
    del y
    gc.collect()
    assert gone() is None
    with checkpoint8():
        y = torch.tanh(a * 1.0)
    (g,) = torch.autograd.grad(y.sum(), a, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), a)
    t = torch.tanh(a.detach().double())
    # 1 - t^2 and 2 t: at most eight roundings of values of at most 2
    assert float((h.double() + 2 * t * (1 - t * t)).abs().max()) <= 16 * 2.0 ** -24


def test_checkpoint8_notices_in_place_changes_of_what_it_kept_as_it_was():
    """as autograd itself does: no gradient from a tensor that has changed since"""
    from ac_solver.agents.activation8 import checkpoint8

    a, b = torch.randn(64, 4, requires_grad=True), torch.randn(64, 4)
    with checkpoint8():
        out = a * b
    b.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with checkpoint8():
        out = a * b
    d = torch.randn(64, 4)
    assert torch.equal(torch.autograd.grad(out, a, d, retain_graph=True)[0], d * b) and torch.equal(torch.autograd.grad(out, a, d)[0], d * b)


def test_forward_mode_tangents_are_refused_not_dropped():
    """an operand with a tangent, with or without a gradient of its own, in every function: the outputs would carry none, which reads as a derivative of zero
    (what the backward functions look at behind the place of the tensors needs a GPU)"""
    import torch.autograd.forward_ad as forward_ad

    from ac_solver.agents import activation8 as A
    from ac_solver.agents import block_norm as B

    c, z = scan_args()
    x, w, p, h = torch.zeros(5, 8), torch.ones(8), torch.zeros(5, 24), torch.zeros(5, 8)
    s, bounds, stats = torch.zeros(2, 4), torch.zeros(8), torch.zeros(5, 2)
    q, e = torch.zeros(5, 8, dtype=torch.int8), torch.zeros(5, 1, dtype=torch.uint8)
    calls = [(R.gated_scan, [c, z, None, s], (0, 1, 3)), (R.gated_scan_forward, [c, z, None, s], (0, 1, 3)),
             (R.gated_scan_backward, [c, s, c, z, None, bounds], (2, 3)), (B.block_output, [x, x, x, w, w, w], (0, 1, 2, 3, 4, 5)), (B.block_input, [x, w], (0, 1)),
             (B.block_output_forward, [x, x, x, w, w, w], (0, 1, 2, 3, 4, 5)), (B.block_output_backward, [x, x, x, x, x, w, w, w, stats], (2, 3, 4, 5, 6, 7)),
             (R.recurrent_block, [x[None], p[None], h, w, w, w], (0, 1, 2, 3, 4, 5)), (R.recurrent_step, [x, p, h, w, w, w], (0, 1, 2, 3, 4, 5)),
             (A.pack8, [x], (0,)), (A.weight_grad8, [x, q, e], (0,))]
    for f, args, places in calls:
        for k in places:
            for grad in (False, True):
                with forward_ad.dual_level():
                    mine = list(args)
                    mine[k] = forward_ad.make_dual(args[k].clone().requires_grad_(grad), torch.ones_like(args[k]))
                    with pytest.raises(NotImplementedError, match="forward mode"):
                        f(*mine)
        with pytest.raises(ValueError, match="GPU"):  # without a tangent only the place is wrong
            f(*args)
    with forward_ad.dual_level():  # (outside a level, or with forward mode off, there are no tangents)
        d = forward_ad.make_dual(c, torch.ones_like(c))
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="GPU"):
            R.gated_scan(d, z)


def _make(*args):
    """make in csrc/, the libraries of HIP and plain C++ code taken as up to date"""
    import os
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ac-solver_amd", "csrc")
    return subprocess.run(["make", "-C", csrc, "-o", "../lib/libacx.so", "-o", "../lib/libacx_trainer.so", *args], capture_output=True, text=True)


@pytest.mark.parametrize("where", ["", "nowhere"])
def test_the_library_builds_without_torch(tmp_path, where):
    """no torch, or one without its headers: everything but the binding is built, and make says so"""
    out = _make(f"BINDING={tmp_path}/acx_torch.so", f"BUILD={tmp_path}", f"TORCH_DIR={tmp_path / where if where else ''}")
    assert out.returncode == 0 and "not built" in out.stderr and not (tmp_path / "acx_torch.so").exists(), out.stderr


def test_the_binding_is_built_again_for_another_torch(tmp_path):
    """(the compiler is replaced by one that only makes the file)"""
    import os

    (tmp_path / "bin").mkdir()
    fake = tmp_path / "bin" / "g++"
    fake.write_text("#!/bin/sh\nwhile [ \"$1\" != -o ]; do shift; done\necho built > \"$2\"\n")
    fake.chmod(0o755)
    path = os.environ["PATH"]
    os.environ["PATH"] = f"{tmp_path / 'bin'}:{path}"
    try:
        args = (f"BINDING={tmp_path}/acx_torch.so", f"BUILD={tmp_path}/build")
        said = [_make(*args, f"TORCH_VERSION={v}") for v in ("1", "1", "2", "2", "1", "1")]
    finally:
        os.environ["PATH"] = path
    assert all(s.returncode == 0 for s in said), [s.stderr for s in said]
    assert ["acx_torch.cpp" in s.stdout for s in said] == [True, False, True, False, True, False]


def test_a_layer_whose_gradient_is_out_of_reach_is_refused_before_it_is_used():
    from ac_solver.agents.activation8 import linear8

    for outputs, inputs in (((1 << 16) + 1, 1), (1, (1 << 16) + 1)):
        w, x, b = torch.zeros(outputs, inputs), torch.zeros(2, inputs), torch.zeros(outputs)
        for weight, bias in ((w.clone().requires_grad_(), None), (w, b.clone().requires_grad_())):
            with pytest.raises(ValueError, match="65536 outputs and inputs"):
                linear8(x, weight, bias)
            with torch.no_grad(), pytest.raises(ValueError, match="GPU"):  # no gradient is wanted: only the place is wrong
                linear8(x, weight, bias)
        with pytest.raises(ValueError, match="GPU"):
            linear8(x.requires_grad_(), w, b)


def test_a_checkpoint8_block_that_could_not_be_entered_leaves_nothing_behind():
    """where saved-tensor hooks are forbidden: outside the block nothing is packed (recurrent_block asks `packing`)"""
    from ac_solver.agents import activation8 as A

    with torch.autograd.graph.disable_saved_tensors_hooks("not here"), pytest.raises(RuntimeError, match="not here"):
        with A.checkpoint8():
            pass
    assert not A.packing()
    with A.checkpoint8():
        with A.checkpoint8():
            assert A.packing()
        assert A.packing()
    assert not A.packing()


def test_what_counts_as_a_leaf_in_another_form():
    """views and copies of a leaf, and nothing that has been computed: not behind a view or a copy either, nor a function that happens to be named like one of torch's"""
    from ac_solver.agents.activation8 import _is_leaf

    class View(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2

    w = torch.randn(8, 8, requires_grad=True)
    buffer, changed, part = torch.zeros(8, 8), w.clone(), w.clone()
    buffer[0] = w[0] * 2
    changed.mul_(2)
    part[0] *= 2
    for t in (w, w.detach(), w.t(), w.view(4, 16)[None].expand(2, 4, 16), w.chunk(2)[1], w.mT, w.unbind(0)[1], w.clone(), w.bfloat16(), w.bfloat16().t(), w.t().bfloat16(), w.double().float()[1:],
              w.t().reshape(-1), buffer.detach()):
        assert _is_leaf(t)
    for t in (w * 1, (w * 1).t(), (w * 1).bfloat16(), w.bfloat16().exp().t(), torch.cat([w, w]), w[torch.tensor([1, 2])], buffer, buffer.t(), changed, changed.t(), part, part.t(), View.apply(w),
              View.apply(w).t()):
        assert not _is_leaf(t)
