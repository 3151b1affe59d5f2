"""The recurrent-state operators as a serving loop and a training step use them together: Canon convolution and linear
attention on one cache, prompts, forks, beams, requests that end, single tokens; and torch.compile."""
import types

import pytest
import torch

import viby_model_b200 as V
from linear_cases import check, decays, magnitudes, make, tolerance
from oracle import linear_oracle as O
from viby_model_b200 import canon_cache as CC

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_serving_loop_prompt_fork_beams_compact_tokens():
    B, T, H, D, rows = 4, 90, 4, 64, 8
    dt = torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    g = decays(H)
    q, k, v = (torch.randn(B, T, n, D, generator=gen).to(dt) for n in (H, 1, 1))
    x, w = torch.randn(B, T, 640, generator=gen).to(dt), torch.randn(640, 4, generator=gen).to(dt)
    lens = torch.tensor([90, 31, 64, 1])
    mask = torch.arange(T)[None] < lens[:, None]
    pool = torch.full((rows, H, D, D), float("nan"), device=DEV)
    conv = torch.full((rows, 640, 3), float("nan"), dtype=dt, device=DEV)
    cache = types.SimpleNamespace(_max_layers=1)
    CC.set_state(cache, "a", 0, conv)
    CC.free(cache, torch.arange(rows, device=DEV), also=[pool])
    assert not pool.any() and not conv.any()
    # prompts into the first rows
    V.linear_attention_fn(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), final_states_out=pool[:B], attention_mask=mask.to(DEV))
    V.causal_conv1d_fn(x.to(DEV).transpose(1, 2), w.to(DEV), attention_mask=mask.to(DEV), final_states_out=conv[:B])
    ref, Mref = O.linear_attention(q, k, v, g, mask=mask)[1], magnitudes(q, k, v, g, mask=mask)[1]
    check(pool[:B], ref, tolerance(ref, Mref, dt, D, T, True, torch.float32), "prompt states")
    ids = list(range(B)) + [None] * (rows - B)  # which prompt each row continues
    conv_ref = conv.clone()

    def moved(source):
        nonlocal conv_ref, ids
        conv_ref = conv_ref[torch.tensor(source, device=DEV)]
        ids = [ids[i] for i in source]

    # request 2 is sampled three times
    CC.fork(cache, torch.tensor([2, 2], device=DEV), torch.tensor([4, 6], device=DEV), also=[pool])
    moved([0, 1, 2, 3, 2, 5, 2, 7])
    # beams of all rows are reordered
    CC.reorder(cache, torch.tensor([3, 3, 2, 0, 6, 5, 4, 1], device=DEV), inplace=True, also=[pool])
    moved([3, 3, 2, 0, 6, 5, 4, 1])
    # rows 1, 4 and the unused one end
    live = torch.tensor([1, 0, 1, 1, 0, 0, 1, 1], dtype=torch.bool, device=DEV)
    new, count = CC.compact(cache, live, also=[pool])
    plan, new_ref, n = O.compact_plan(live.tolist())
    moved(plan)
    assert new.tolist() == new_ref and int(count) == n == 5
    assert torch.equal(conv, conv_ref)
    # tokens on the live rows; what lies behind them stays
    behind, S, M = pool[n:].clone(), ref[ids[:n]], Mref[ids[:n]]
    for step in range(3):
        tq, tk, tv, *_ = make(n, 1, H, 1, 1, D, D, dt, step)
        o = V.linear_attention_update(tq[:, 0].to(DEV), tk[:, 0].to(DEV), tv[:, 0].to(DEV), pool[:n], g.to(DEV))
        V.causal_conv1d_update(torch.randn(n, 640, generator=gen).to(dt).to(DEV), conv[:n], w.to(DEV))
        want, S = O.linear_attention(tq, tk, tv, g, initial=S)
        size, M = O.linear_attention(tq.abs(), tk.abs(), tv.abs(), g, initial=M)
        check(o, want[:, 0], tolerance(want, size, dt, D, T + 64, True)[:, 0], f"token {step}")
    check(pool[:n], S, tolerance(S, M, dt, D, T + 192, True, torch.float32), "states")
    assert torch.equal(pool[n:].view(torch.int32), behind.view(torch.int32))


def test_canon_cache_in_place_reorder_equals_the_selecting_one():
    gen = torch.Generator().manual_seed(1)
    a, b = (types.SimpleNamespace(_max_layers=3) for _ in range(2))
    shared = torch.arange(5, dtype=torch.int32, device=DEV)
    for layer in range(3):
        for pos, d in zip(CC.CANON_POSITIONS, (640, 960, 640, 3456)):
            s = torch.randn(5, d, 4, generator=gen).bfloat16().to(DEV)
            CC.set_state(a, pos, layer, s.clone())
            CC.set_state(b, pos, layer, s.clone())
        CC.set_seqlens(a, "a", layer, shared)  # one vector for all layers moves once
    idx = torch.tensor([4, 4, 0, 1, 3], device=DEV)
    held = CC.get_state(a, "d", 1)
    before = V.launch_count()
    CC.reorder(a, idx, inplace=True)
    assert V.launch_count() == before + 1 and CC.get_state(a, "d", 1) is held
    CC.reorder(b, idx)
    for (n0, l0, s0), (n1, l1, s1) in zip(CC.states(a), CC.states(b)):
        assert (n0, l0) == (n1, l1) and torch.equal(s0, s1)
    assert shared.tolist() == [4, 4, 0, 1, 3]


def test_training_step_of_a_small_mixer_and_its_gradients():
    """Canon convolution, linear attention, a projection: the loss's gradients against the same network in 64 bits."""
    torch.manual_seed(0)
    B, T, H, D = 2, 70, 2, 16
    x0, w0 = torch.randn(B, T, 3 * H * D), torch.randn(3 * H * D, 4) * 0.3
    p0 = torch.randn(H * D, 5) * 0.1
    target = torch.randn(B, T, 5)
    g = decays(H)

    def loss(x, w, p, conv, attend):
        y = conv(x, w)
        q, k, v = (t.unflatten(-1, (H, D)) for t in y.split(H * D, -1))
        return ((attend(q, k, v).flatten(2) @ p - target.to(x)) ** 2).mean()

    conv64 = lambda x, w: torch.nn.functional.conv1d(  # noqa: E731
        torch.nn.functional.pad(x.transpose(1, 2), (3, 0)), w[:, None], groups=3 * H * D).transpose(1, 2)
    ref = [t.double().requires_grad_() for t in (x0, w0, p0)]
    loss(*ref, conv64, lambda q, k, v: O.linear_attention(q, k, v, g)[0]).backward()
    got = [t.to(DEV).requires_grad_() for t in (x0, w0, p0)]
    loss(*got, lambda x, w: V.causal_conv1d_fn(x.transpose(1, 2), w).transpose(1, 2),
         lambda q, k, v: V.linear_attention_fn(q, k, v, g.to(DEV))).backward()
    for a, b in zip(got, ref):
        # fp32 throughout: some hundred roundings of 2^-24 on sums of the gradient's own size
        assert float((a.grad.cpu().double() - b.grad).norm() / b.grad.norm()) < 300 * 2.0 ** -24


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_prompt_training_and_token(backend):
    q, k, v, do, s0, ds = (t.to(DEV) for t in make(2, 70, 2, 1, 2, 32, 32, torch.bfloat16))
    g = decays(2).to(DEV)
    m = torch.arange(70, device=DEV)[None] < torch.tensor([[70], [33]], device=DEV)

    def prompt(q, k, v, s0):
        o, s = V.linear_attention_fn(q * 1.0, k, v, g, None, s0, True, attention_mask=m)
        return o * 2.0, s

    def token(q, k, v, s):
        return V.linear_attention_update(q, k, v, s, g) + 1.0

    with torch.no_grad():
        want = prompt(q, k, v, s0)
        got = torch.compile(prompt, backend=backend, fullgraph=True)(q, k, v, s0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a, b = s0.clone(), s0.clone()
        assert torch.equal(torch.compile(token, backend=backend, fullgraph=True)(q[:, 0], k[:, 0], v[:, 0], a), token(q[:, 0], k[:, 0], v[:, 0], b))
        assert torch.equal(a, b)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, s0)]
    want = torch.autograd.grad(prompt(*leaves), leaves, [do, ds])
    got = torch.autograd.grad(torch.compile(prompt, backend=backend, fullgraph=True)(*leaves), leaves, [do, ds])
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_backward_captured_while_an_eager_graph_of_the_same_leaves_lives():
    """The explicit backward call makes no use of autograd's nodes, so it is captured whatever graphs are alive."""
    q, k, v, do, s0, ds = (t.to(DEV) for t in make(1, 300, 2, 1, 1, 64, 64, torch.bfloat16))
    g = decays(2).to(DEV)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    alive = V.linear_attention_fn(*leaves, g)  # an eager graph
    want = V.linear_attention_bwd(*(x.detach() for x in leaves), g, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = V.linear_attention_bwd(*(x.detach() for x in leaves), g, do)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
    eager = torch.autograd.grad(alive, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(eager, want[:3]))


def test_writing_a_saved_state_in_place_is_noticed():
    q, k, v, do, s0, _ = (t.to(DEV) for t in make(1, 20, 2, 2, 2, 32, 32, torch.bfloat16))
    g = decays(2).to(DEV)
    x = q.clone().requires_grad_()
    o = V.linear_attention_fn(x, k, v, g, None, s0)
    V.linear_attention_update(k[:, 0], k[:, 0], v[:, 0], s0, g)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
    o = V.linear_attention_fn(x, k, v, g, None, s0)
    V.free_pages([s0], torch.tensor([0], device=DEV))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)


def test_refusals_on_the_device():
    q, k, v, do, s0, ds = (t.to(DEV) for t in make(2, 8, 2, 2, 2, 16, 16, torch.bfloat16))
    g = decays(2).to(DEV)
    bad = pytest.raises(ValueError)
    with bad:
        V.linear_attention_fn(q, k, v, g.double())
    with bad:
        V.linear_attention_fn(q, k, v, g[:1])
    with bad:
        V.linear_attention_fn(q, k, v, g.clone().requires_grad_())
    with bad:
        V.linear_attention_fn(q, k, v, g.cpu())
    with bad:
        V.linear_attention_fn(q, k.cpu(), v, g)
    with bad:
        V.linear_attention_fn(q, k, v, g, None, s0.half())
    with bad:
        V.linear_attention_fn(q, k, v, g, None, s0[:1])
    with bad:
        V.linear_attention_fn(q, k, v, g, None, s0, final_states_out=s0)  # overlaps
    with bad:
        V.linear_attention_fn(q, k, v, g, attention_mask=torch.ones(2, 7, device=DEV))
    with bad:
        V.linear_attention_fn(q, k, v, g, torch.zeros(2, 9, dtype=torch.int32, device=DEV))
    with bad:
        V.linear_attention_fn(q, k, v, g, out=q)  # overlaps an input
    with bad:
        V.linear_attention_fn(q, k, v, g, kernel="none such")
    with bad:
        V.linear_attention_fn(q[..., 1:], k[..., 1:], v, g, kernel="mma")  # not aligned
    with bad:
        V.linear_attention_fn(q.half(), k.half(), v.half(), g, kernel="tc")
    with bad:
        V.linear_attention_bwd(q, k, v, g, do.float())
    with bad:
        V.linear_attention_bwd(q, k, v, g, do, None, s0, ds[..., :4])
    with bad:
        V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], s0.expand(2, 2, 16, 16)[:1], g)
    with bad:
        V.linear_attention_update(q[:1, 0].expand(2, 2, 16), k[:, 0], v[:, 0], s0[:1].expand(2, 2, 16, 16), g)  # one state for two rows
    with bad:
        V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], s0, g, attention_mask=torch.ones(3, device=DEV))
    idx = torch.tensor([0, 1], device=DEV)
    for states in ([s0, s0], [s0, s0[:, :1]], [s0.transpose(2, 3)], [s0[:1].expand(2, 2, 16, 16)], [s0, g[:1]], [s0, torch.zeros(2)]):
        with bad:
            V.reorder_pages(states, idx)
    with bad:
        V.reorder_pages([s0], idx[:1])
    with bad:
        V.reorder_pages([s0], idx.cpu())
    with bad:
        V.copy_pages([s0], idx, idx.int())
    with bad:
        V.compact_pages([s0], torch.ones(2, device=DEV))
    with bad:
        V.reorder_pages([s0, idx], idx)  # the index is one of the states


def test_a_decay_that_wants_a_gradient_is_refused_whatever_else_wants_one():
    q, k, v, *_ = (t.to(DEV) for t in make(1, 8, 2, 2, 2, 16, 16, torch.bfloat16))
    g = decays(2).to(DEV).requires_grad_()
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(ValueError, match="no gradient"):
            V.linear_attention_fn(x, k, v, g)
    with pytest.raises(ValueError, match="no gradient"):
        V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], torch.zeros(1, 2, 16, 16, device=DEV), g)
    with torch.no_grad():
        V.linear_attention_fn(q, k, v, g)
    V.linear_attention_fn(q.clone().requires_grad_(), k, v, g.detach())


def test_repeated_calls_with_other_data_alignment_and_devices_of_the_same_signature():
    """A call's checked arguments are remembered by shapes and strides: data elsewhere, at odd addresses, in other
    dtypes of the mask, has to come out the same."""
    q, k, v, _, s0, _ = make(2, 130, 2, 2, 2, 64, 64, torch.bfloat16)
    g = decays(2).to(DEV)
    want = V.linear_attention_fn(q.to(DEV), k.to(DEV), v.to(DEV), g, None, s0.to(DEV), True, kernel="simt")
    ref, ref_s = O.linear_attention(q, k, v, decays(2), initial=s0)
    M, M_s = magnitudes(q, k, v, decays(2), s0)
    for turn in range(4):
        args = []
        for x in (q, k, v):
            buf = torch.empty(x.numel() + 8, dtype=x.dtype, device=DEV)
            at = (0, 1, 8, 3)[turn]
            buf[at: at + x.numel()] = x.reshape(-1).to(DEV)
            args.append(buf[at: at + x.numel()].view(x.shape))
        o, s = V.linear_attention_fn(*args, g, None, s0.to(DEV), True)
        check(o, ref, tolerance(ref, M, torch.bfloat16, 64, 130, True), "out")
        check(s, ref_s, tolerance(ref_s, M_s, torch.bfloat16, 64, 130, True, torch.float32), "state")
        state = s0.to(DEV)
        V.linear_attention_update(args[0][:, 0], args[1][:, 0], args[2][:, 0], state, g)
    assert want[0].shape == o.shape


def test_calls_without_tokens_are_remembered_too():
    """Empty tensors have no address.  A thread of its own starts without prepared calls, whatever ran before."""
    from concurrent.futures import ThreadPoolExecutor

    def calls():
        g = torch.full((2,), -0.1, device=DEV)
        for dtype in (torch.float32, torch.bfloat16):
            for shape in ((2, 0, 2, 16), (0, 5, 2, 16), (2, 3, 2, 16)):
                x = torch.ones(shape, device=DEV, dtype=dtype)
                for _ in range(3):
                    o, s = V.linear_attention_fn(x, x, x, g, None, None, True)
                    assert tuple(o.shape) == shape and bool(s.any()) == (x.numel() > 0)
                    assert x.numel() == 0 or bool(o.any())
                if shape[1] == 0 or shape[0] == 0:
                    s = torch.ones(shape[0], 2, 16, 16, device=DEV)
                    for _ in range(2):
                        assert torch.equal(V.linear_attention_fn(x, x, x, g, None, s, True)[1], s)
        return True

    with ThreadPoolExecutor(1) as pool:
        assert pool.submit(calls).result()
