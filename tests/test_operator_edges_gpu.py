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
