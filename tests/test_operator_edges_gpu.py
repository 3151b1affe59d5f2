"""Calls at the edges of what linear attention and cache pages accept: lengths past 2^25, no tokens, remembered call forms,
derivatives that there are none of, waits that run out.  Small tolerances only where sums are involved (tests/linear_cases.py)."""
import pytest
import torch

import viby_model_b200 as V
from linear_cases import check, decays, magnitudes, make, tolerance
from oracle import linear_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("side", ["left", "right"])
def test_padding_of_more_than_2_to_the_25_tokens(side):
    """One part of the time axis whose padding, times the 64 columns of a slab, does not fit 31 bits."""
    T, D, n = (1 << 25) + 389, 8, 5
    q, k, v = (torch.full((1, T, 1, D), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(3))
    small = make(1, n, 1, 1, 1, D, D, torch.bfloat16)[:3]
    at = slice(T - n, T) if side == "left" else slice(0, n)
    for x, y in zip((q, k, v), small):
        x[:, at] = y.to(DEV)
    mask = torch.zeros(1, T, dtype=torch.bool, device=DEV)
    mask[:, at] = True
    out = torch.ones(1, T, 1, D, dtype=torch.bfloat16, device=DEV)
    g = decays(1)
    _, state = V.linear_attention_fn(q, k, v, g.to(DEV), return_final_states=True, attention_mask=mask, out=out, kernel="tc", segments=1)
    ref, ref_s = O.linear_attention(*small, g)
    M, M_s = magnitudes(*small, g)
    check(out[:, at], ref, tolerance(ref, M, torch.bfloat16, D, n, True), "out")
    check(state, ref_s, tolerance(ref_s, M_s, torch.bfloat16, D, n, True, torch.float32), "state")
    out[:, at] = 0
    assert not bool(out.view(torch.int32).any())  # +0, every one of them


@pytest.mark.parametrize("kernel", ["simt", "mma", "tc"])
def test_the_named_kernel_runs_under_compile_too(kernel):
    """Forward and backward; each kernel rounds differently, so that equal bits show which one ran."""
    q, k, v, do, s0, ds = (x.to(DEV) for x in make(1, 260, 2, 1, 2, 64, 64, torch.bfloat16))
    g = decays(2).to(DEV)

    def f(q, k, v, s0):
        return V.linear_attention_fn(q, k, v, g, None, s0, True, kernel=kernel, segments=2)

    torch._dynamo.reset()
    results = []
    for call in (f, torch.compile(f, fullgraph=True)):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, s0)]
        o, s = call(*leaves)
        before = V.last_kernel()
        results.append((o, s, *torch.autograd.grad([o, s], leaves, [do, ds])))
        assert before == f"linear_{kernel}"
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_an_unknown_kernel_is_refused_under_compile():
    q, k, v, *_ = (x.to(DEV) for x in make(1, 8, 2, 2, 2, 16, 16, torch.bfloat16))
    g = decays(2).to(DEV)
    with pytest.raises(Exception, match="unknown linear attention kernel"):
        torch.compile(lambda q: V.linear_attention_fn(q, k, v, g, kernel="best"))(q)


@pytest.mark.parametrize("kernel", [None, "simt", "mma", "tc"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [16, 160, 256])
def test_calls_without_tokens_copy_the_state(dtype, D, kernel):
    """There is nothing to make tensor maps of, so none of the kernels that take tokens by them may run."""
    q, k, v, do, s0, ds = (x.to(DEV) for x in make(2, 0, 2, 1, 2, D, D, dtype))
    g = decays(2).to(DEV)
    for initial in (s0, None):
        o, s = V.linear_attention_fn(q, k, v, g, None, initial, True, kernel=kernel, segments=2)
        assert V.last_kernel() == "linear_simt"
        assert tuple(o.shape) == (2, 0, 2, D) and torch.equal(s, s0 if initial is not None else torch.zeros_like(s0))
    for dfinal in (ds, None):
        *grads, di = V.linear_attention_bwd(q, k, v, g, do, None, s0, dfinal, kernel=kernel)
        assert V.last_kernel() == "linear_simt"
        assert all(x.shape == y.shape for x, y in zip(grads, (q, k, v)))
        assert torch.equal(di, ds if dfinal is not None else torch.zeros_like(ds))


def test_waits_of_the_tcgen05_kernel_run_out_and_report():
    """With the self-test's chunk withheld, the warps that wait for it give up, the others follow, the CTA waits for its
    products and copies in flight and frees its tensor memory: the launch returns, the count of expired waits grows, and
    the next ordinary launch is clean.  For one and two buffers of keys (heads of 160 and 64), both directions, the pass that
    finds the parts' states, rows with and without masks, and the first, second and a later chunk.  In a process of its
    own: the count stays."""
    import subprocess
    import sys

    from conftest import ROOT

    code = r"""
import ctypes as C
import torch
import viby_model_b200 as V
from viby_model_b200 import _cabi, linear_attention as la
for D, masked, runs in ((64, 0, ((1, 1), (1, 4))), (64, 1, ((2, 3),)), (160, 1, ((1, 2), (1, 4))), (160, 0, ((2, 2),))):
    g = torch.Generator().manual_seed(D)
    T, H = 900, 2
    q, k, v, do = (torch.randn(2, T, H, D, generator=g).bfloat16().cuda() for _ in range(4))
    ld = torch.tensor([-0.01, -0.3]).cuda()
    m = (torch.rand(2, T, generator=g) < 0.8).cuda() if masked else None
    for segments, chunk in runs:
        want = V.linear_attention_fn(q, k, v, ld, None, None, True, attention_mask=m, kernel="tc", segments=segments)
        grads = V.linear_attention_bwd(q, k, v, ld, do, attention_mask=m, kernel="tc", segments=segments)
        assert V.last_kernel() == "linear_tc"
        stream = torch.cuda.current_stream().cuda_stream
        before = V.tma_timeouts()
        a, keep = la._fill(q, k, v, ld, None, None, m, None, "tc", segments)
        out, state = torch.zeros_like(want[0]), torch.zeros_like(want[1])
        a.out, a.out_strides[:], a.final_state, a.final_strides[:] = out.data_ptr(), out.stride(), state.data_ptr(), state.stride()
        a.test_expire = chunk
        ws = la._workspace(a, _cabi.lib.vc1d_linear_workspace, q.device)
        assert _cabi.lib.vc1d_linear(C.byref(a), stream) == 0
        torch.cuda.synchronize()  # the launch returns: nothing hangs, nothing traps
        between = V.tma_timeouts()
        assert between > before, "the expired waits were not reported"
        b = _cabi.LinearBwdArgs()
        b.struct_size, b.segments, b.f, b.dout = C.sizeof(b), segments, a, do.data_ptr()
        b.dout_strides[:] = do.stride()
        new = [torch.zeros_like(x) for x in (q, k, v)]
        b.dq, b.dk, b.dv = (x.data_ptr() for x in new)
        b.dq_strides[:], b.dk_strides[:], b.dv_strides[:] = (x.stride() for x in new)
        ws2 = la._workspace(b, _cabi.lib.vc1d_linear_bwd_workspace, q.device)
        assert _cabi.lib.vc1d_linear_bwd(C.byref(b), stream) == 0
        torch.cuda.synchronize()
        expired = V.tma_timeouts()
        assert expired > between
        o, s = V.linear_attention_fn(q, k, v, ld, None, None, True, attention_mask=m, kernel="tc", segments=segments)
        again = V.linear_attention_bwd(q, k, v, ld, do, attention_mask=m, kernel="tc", segments=segments)
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])
        assert all(torch.equal(x, y) for x, y in zip(again[:3], grads[:3]))
        assert V.tma_timeouts() == expired, "an ordinary launch after the self-test reported expired waits"
print("EXPIRED", expired)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=str(ROOT))
    assert r.returncode == 0, r.stdout + r.stderr
    assert "EXPIRED" in r.stdout


def test_new_forms_are_remembered_after_hundreds_of_others(monkeypatch):
    """Prompts of 300 lengths and batches of 300 sizes, as a server sees them: the form that comes next is prepared once, and the
    number of those that are kept is bounded."""
    from viby_model_b200 import linear_attention as la

    q, k, v, _, s0, _ = (x.to(DEV) for x in make(1, 402, 1, 1, 1, 8, 8, torch.bfloat16))
    g = decays(1).to(DEV)
    state = s0.expand(402, -1, -1, -1).contiguous()
    for n in range(1, 301):
        V.linear_attention_fn(q[:, :n], k[:, :n], v[:, :n], g)
        V.linear_attention_update(q[0, :n], k[0, :n], v[0, :n], state[:n], g)
    checked = []
    for name in ("_check_heads", "_fill"):
        monkeypatch.setattr(la, name, lambda *a, f=getattr(la, name), name=name: (checked.append(name), f(*a))[1])
    for n in (401, 402):
        for turn in range(3):
            V.linear_attention_fn(q[:, :n], k[:, :n], v[:, :n], g)
            V.linear_attention_update(q[0, :n], k[0, :n], v[0, :n], state[:n], g)
            assert checked == (["_fill", "_check_heads", "_check_heads"] if turn == 0 else []), (n, turn)
            checked.clear()
    assert len(la._prepared("linear_args")) <= 256 and len(la._prepared("linear_update_args")) <= 256


@pytest.mark.parametrize("kernel", ["simt", "mma", "tc"])
def test_gradients_that_arrive_expanded(kernel):
    """The gradient of a sum is one value, repeated by strides of 0, which the named tensor-core kernels do not take."""
    q, k, v, *_ = (x.to(DEV) for x in make(1, 150, 2, 2, 2, 64, 64, torch.bfloat16))
    g = decays(2).to(DEV)
    grads = []
    for whole in (False, True):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        o = V.linear_attention_fn(*leaves, g, kernel=kernel)
        (o.backward(torch.ones_like(o)) if whole else o.sum().backward())
        grads.append([x.grad for x in leaves])
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    torch.compile(lambda *x: V.linear_attention_fn(*x, g, kernel=kernel).sum(), backend="aot_eager")(*leaves).backward()
    grads.append([x.grad for x in leaves])
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*grads))
