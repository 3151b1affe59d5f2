"""Linear attention on the GPU against the recurrence in 64 bits: types, head layouts, lengths, masks, packed rows,
states, strides, gradients, streams and captured graphs.  Tolerances: tests/linear_cases.py."""
import pytest
import torch

import viby_model_b200 as V
from linear_cases import DTYPES, check, decays, grad_magnitudes, magnitudes, make, tolerance
from oracle import linear_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x):
    return None if x is None else x.to(DEV)


def forward_case(dtype, B, T, H, Hk, Hv, Dk, Dv, *, mask=None, seq=None, init=False, final=False, kind="mixed", kernel=None,
                 segments=0, seed=0, layout=None, poison=None):
    q, k, v, _, s0, _ = make(B, T, H, Hk, Hv, Dk, Dv, dtype, seed)
    g = decays(H, kind)
    if mask is not None and poison is not None:
        dead = mask == 0
        for x in (q, k, v):
            x[dead] = poison
    s0 = s0 if init else None
    dq, dk, dv = dev(q), dev(k), dev(v)
    if layout is not None:
        dq, dk, dv = layout(dq, dk, dv)
    r = V.linear_attention_fn(dq, dk, dv, dev(g), dev(seq), dev(s0), final, attention_mask=dev(mask), kernel=kernel, segments=segments)
    o, S = r if final else (r, None)
    ref_o, ref_S = O.linear_attention(q, k, v, g, mask=mask, seq_idx=seq, initial=s0)
    M_o, M_S = magnitudes(q, k, v, g, s0, mask=mask, seq_idx=seq)
    tc = kernel != "simt" and dtype != torch.float32
    assert o.dtype == dtype and tuple(o.shape) == (B, T, H, Dv)
    check(o, ref_o, tolerance(ref_o, M_o, dtype, Dk, T, tc), "out")
    if final:
        assert S.dtype == torch.float32
        check(S, ref_S, tolerance(ref_S, M_S, dtype, Dk, T, tc, torch.float32), "final state")
    return o, S


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 200])
def test_lengths(dtype, T, kernel):
    forward_case(DTYPES[dtype], 2, T, 3, 3, 3, 64, 64, init=True, final=True, kernel=kernel)


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (1, 256), (8, 8), (16, 24), (33, 17), (72, 88), (128, 128), (160, 160), (192, 64), (256, 256), (40, 200)])
def test_head_dims(dtype, Dk, Dv, kernel):
    forward_case(DTYPES[dtype], 1, 130, 2, 2, 1, Dk, Dv, init=True, final=True, kernel=kernel)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,Hv", [(1, 1, 1), (4, 1, 1), (4, 4, 1), (4, 1, 4), (6, 2, 3)])
def test_head_layouts(dtype, H, Hk, Hv):
    forward_case(DTYPES[dtype], 2, 70, H, Hk, Hv, 64, 64, final=True)


def masks(B, T):
    t = torch.arange(T)[None]
    lens = torch.tensor([T, T // 2, 1, 0])[:B, None]
    holes = torch.rand(B, T, generator=torch.Generator().manual_seed(3)) < 0.4
    holes[-1] = False
    return {"right": t < lens, "left": t >= T - lens, "holes": holes}


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["right", "left", "holes"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), "lowest"])
def test_masks_rows_without_a_token_and_poison_in_masked_places(dtype, which, poison, kernel):
    dt = DTYPES[dtype]
    value = torch.finfo(dt).min if poison == "lowest" else poison
    o, S = forward_case(dt, 4, 150, 2, 1, 2, 64, 32, mask=masks(4, 150)[which], init=True, final=True, poison=value, kernel=kernel)
    assert not o[-1].any()  # the row without a token


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.float16])
def test_mask_types(mask_dtype):
    forward_case(torch.bfloat16, 4, 90, 2, 2, 2, 64, 64, mask=masks(4, 90)["holes"].to(mask_dtype), final=True)


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[1], [64, 64], [1, 1, 1, 60, 5, 130, 3], [200], [33, 31, 64, 1, 128]])
def test_packed_rows(dtype, lengths, kernel):
    seq = V.seq_idx_from_lengths(lengths)
    forward_case(DTYPES[dtype], 1, sum(lengths), 2, 2, 2, 64, 64, seq=seq, kernel=kernel)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_rows_equal_separate_calls(dtype):
    lengths = [70, 1, 129, 64]
    q, k, v, *_ = make(1, sum(lengths), 2, 1, 2, 64, 64, DTYPES[dtype])
    g = dev(decays(2))
    whole = V.linear_attention_fn(dev(q), dev(k), dev(v), g, V.seq_idx_from_lengths(lengths, DEV))
    ref, _ = O.linear_attention(q, k, v, decays(2), seq_idx=V.seq_idx_from_lengths(lengths))
    M, _ = magnitudes(q, k, v, decays(2), seq_idx=V.seq_idx_from_lengths(lengths))
    tol = tolerance(ref, M, DTYPES[dtype], 64, sum(lengths), dtype != "f32")
    t = 0
    for n in lengths:
        part = V.linear_attention_fn(*(dev(x[:, t: t + n]) for x in (q, k, v)), g)
        check(part, whole[:, t: t + n].cpu().double(), 2 * tol[:, t: t + n], "part")
        t += n


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "one token", "fast"])
def test_decays(dtype, kind, kernel):
    forward_case(DTYPES[dtype], 2, 140, 4, 4, 4, 32, 48, init=kind != "one token", final=True, kind=kind, kernel=kernel)


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("segments", [2, 3, 64])
@pytest.mark.parametrize("case", ["plain", "mask", "packed"])
def test_split_time_axis(dtype, segments, case, kernel):
    T = 500
    kw = {}
    if case == "mask":
        kw["mask"] = masks(2, T)["holes"]
    if case == "packed":
        kw["seq"] = V.seq_idx_from_lengths([100, 27, 300, 73]).expand(2, -1).contiguous()
    else:
        kw.update(init=True, final=True)
    forward_case(DTYPES[dtype], 2, T, 2, 1, 1, 72, 80, segments=segments, kernel=kernel, **kw)


def fused(q, k, v):
    B, T = q.shape[:2]
    x = torch.cat([t.reshape(B, T, -1) for t in (q, k, v)], -1)
    parts = x.split([t.shape[2] * t.shape[3] for t in (q, k, v)], -1)
    return tuple(p.unflatten(-1, t.shape[2:]) for p, t in zip(parts, (q, k, v)))


def heads_first(q, k, v):
    return tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))


def odd_offset(q, k, v):
    out = []
    for t in (q, k, v):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        buf[1:] = t.reshape(-1)
        out.append(buf[1:].view(t.shape))
    return tuple(out)


def channels_strided(q, k, v):
    return tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v))


def time_reversed_storage(q, k, v):
    out = []
    for t in (q, k, v):
        B, T, H, D = t.shape
        buf = torch.zeros(B, T, H, 2 * D, dtype=t.dtype, device=t.device)
        buf[..., :D] = t
        out.append(buf[..., :D])
    return tuple(out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", [fused, heads_first, odd_offset, channels_strided, time_reversed_storage])
def test_strides_and_alignment(dtype, layout):
    forward_case(DTYPES[dtype], 2, 100, 4, 2, 2, 64, 64, init=True, final=True, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES)
def test_broadcast_inputs_and_their_gradients(dtype):
    dt = DTYPES[dtype]
    q, k, v, do, *_ = make(3, 80, 4, 4, 4, 32, 32, dt)
    g = decays(4)
    kb = dev(k[:1, :, :1]).requires_grad_()  # one key for all rows and heads
    o = V.linear_attention_fn(dev(q), kb.expand(3, 80, 4, 32), dev(v), dev(g))
    (gk,) = torch.autograd.grad(o, kb, dev(do))
    kk = k[:1, :, :1].expand(3, 80, 4, 32)
    _, ref, _, _ = O.grads(q, kk, v, g, do)
    _, M, _, _ = grad_magnitudes(q, kk, v, g, do)
    each = tolerance(ref, M, dt, 32, 80, dt != torch.float32)
    total = ref.sum((0, 2), keepdim=True)
    # torch sums twelve rounded gradients: each partial sum rounds once more
    tol = each.sum((0, 2), keepdim=True) + 13 * torch.finfo(dt).eps / 2 * ref.abs().sum((0, 2), keepdim=True)
    check(gk, total, tol, "gradient of the broadcast key")


@pytest.mark.parametrize("dtype", DTYPES)
def test_given_outputs(dtype):
    dt = DTYPES[dtype]
    q, k, v, _, s0, _ = make(2, 70, 2, 2, 2, 64, 48, dt)
    g = dev(decays(2))
    want_o, want_s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, dev(s0), True)
    out = torch.full((2, 2, 70, 48), 7.0, dtype=dt, device=DEV).transpose(1, 2)
    pool = torch.full((5, 2, 64, 48), 7.0, device=DEV)
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, dev(s0), final_states_out=pool[1:3], out=out)
    assert o is out and torch.equal(o, want_o) and torch.equal(pool[1:3], want_s)
    assert (pool[0] == 7).all() and (pool[3:] == 7).all()


def test_no_tokens():
    q, k, v, do, s0, ds = make(2, 0, 2, 2, 2, 16, 16, torch.bfloat16)
    g = dev(decays(2))
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, dev(s0), True)
    assert tuple(o.shape) == (2, 0, 2, 16) and torch.equal(s.cpu(), s0)
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, None, True)
    assert not s.any()
    *_, di = V.linear_attention_bwd(dev(q), dev(k), dev(v), g, dev(do), None, dev(s0), dev(ds))
    assert torch.equal(di.cpu(), ds)
    q, k, v, *_ = make(0, 5, 2, 2, 2, 16, 16, torch.bfloat16)
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, None, True)
    assert tuple(o.shape) == (0, 5, 2, 16) and tuple(s.shape) == (0, 2, 16, 16)


def test_long_prompt_in_parts_equals_the_whole():
    q, k, v, *_ = make(1, 700, 2, 2, 2, 64, 64, torch.float32)
    g = dev(decays(2, "none"))
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), g, None, None, True)
    ref, ref_s = O.linear_attention(q, k, v, decays(2, "none"))
    M, M_s = magnitudes(q, k, v, decays(2, "none"))
    state, parts = None, []
    for a, b in ((0, 1), (1, 300), (300, 301), (301, 700)):
        p, state = V.linear_attention_fn(*(dev(x[:, a:b]) for x in (q, k, v)), g, None, state, True)
        parts.append(p)
    check(torch.cat(parts, 1), ref, tolerance(ref, M, torch.float32, 64, 1000, False), "out")
    check(state, ref_s, tolerance(ref_s, M_s, torch.float32, 64, 1000, False), "state")
    check(s, ref_s, tolerance(ref_s, M_s, torch.float32, 64, 700, False), "state of the whole")


# ------------------------------------------------------------------------------------------------ gradients


def backward_case(dtype, B, T, H, Hk, Hv, Dk, Dv, *, mask=None, seq=None, init=False, final=False, kind="mixed", kernel=None,
                  segments=0, layout=None, poison=None):
    q, k, v, do, s0, ds = make(B, T, H, Hk, Hv, Dk, Dv, dtype, 1)
    g = decays(H, kind)
    if mask is not None and poison is not None:
        for x in (q, k, v, do):
            x[mask == 0] = poison
    s0, ds = s0 if init else None, ds if final else None
    leaves = list(layout(dev(q), dev(k), dev(v)) if layout else (dev(q), dev(k), dev(v)))
    leaves = [x.detach().requires_grad_() for x in leaves]
    if init:
        leaves.append(dev(s0).requires_grad_())
    r = V.linear_attention_fn(*leaves[:3], dev(g), dev(seq), leaves[3] if init else None, final, attention_mask=dev(mask),
                              kernel=kernel, segments=segments)
    outs, gouts = ([r[0], r[1]], [dev(do), dev(ds)]) if final else ([r], [dev(do)])
    got = torch.autograd.grad(outs, leaves, gouts)
    ref = O.grads(q, k, v, g, do, mask=mask, seq_idx=seq, initial=s0, dfinal=ds)
    M = grad_magnitudes(q, k, v, g, do, s0, ds, mask=mask, seq_idx=seq)
    tc = kernel != "simt" and dtype != torch.float32
    for i, name in enumerate(("dq", "dk", "dv")):
        check(got[i], ref[i], tolerance(ref[i], M[i], dtype, max(Dk, Dv) + H, T, tc), name)
    if init:
        check(got[3], ref[3], tolerance(ref[3], M[3], dtype, max(Dk, Dv), T, tc, torch.float32), "dinitial")
    return got


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 64, 65, 180])
def test_backward_lengths(dtype, T, kernel):
    backward_case(DTYPES[dtype], 2, T, 2, 2, 2, 64, 64, init=True, final=True, kernel=kernel)


@pytest.mark.parametrize("kernel", [None, "simt"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (16, 40), (72, 88), (128, 64), (160, 160), (256, 256)])
def test_backward_head_dims(dtype, Dk, Dv, kernel):
    backward_case(DTYPES[dtype], 1, 100, 2, 2, 2, Dk, Dv, kernel=kernel)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,Hv", [(4, 1, 1), (4, 4, 2), (6, 2, 3)])
def test_backward_shared_heads(dtype, H, Hk, Hv):
    backward_case(DTYPES[dtype], 2, 100, H, Hk, Hv, 64, 32, init=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["right", "left", "holes"])
def test_backward_masks(dtype, which):
    got = backward_case(DTYPES[dtype], 4, 140, 2, 1, 2, 32, 32, mask=masks(4, 140)[which], init=True, final=True, poison=float("nan"))
    assert not any(x[3].any() for x in got[:3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("segments", [0, 3])
def test_backward_packed(dtype, segments):
    backward_case(DTYPES[dtype], 1, 300, 2, 2, 2, 64, 64, seq=V.seq_idx_from_lengths([64, 1, 100, 135]), segments=segments)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "one token", "fast"])
def test_backward_decays(dtype, kind):
    backward_case(DTYPES[dtype], 1, 130, 4, 4, 4, 32, 32, kind=kind, init=kind != "one token", final=kind != "one token")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("segments", [2, 5])
def test_backward_split_time_axis(dtype, segments):
    backward_case(DTYPES[dtype], 1, 400, 2, 1, 2, 64, 72, init=True, final=True, segments=segments, mask=masks(2, 400)["holes"][:1])


@pytest.mark.parametrize("layout", [fused, heads_first, odd_offset, channels_strided])
def test_backward_strides(layout):
    backward_case(torch.bfloat16, 2, 70, 2, 2, 2, 64, 64, layout=layout)


def test_gradient_against_differences():
    """The derivative along random directions, from outputs of the fp32 kernel: central differences of a function that
    is a polynomial of degree three in the step, so that two steps give it without a truncation error."""
    torch.manual_seed(0)
    q, k, v, do, s0, ds = make(1, 90, 2, 1, 2, 24, 40, torch.float32)
    g = dev(decays(2))
    leaves = [dev(x).requires_grad_() for x in (q, k, v, s0)]
    f = lambda *x: [V.linear_attention_fn(*x[:3], g, None, x[3], True)]  # noqa: E731
    o, s = f(*leaves)[0]
    grads = torch.autograd.grad([o, s], leaves, [dev(do), dev(ds)])
    value = lambda *x: sum(float((y.double() * w.double()).sum()) for y, w in zip(f(*x)[0], (dev(do), dev(ds))))  # noqa: E731
    with torch.no_grad():
        for i, x in enumerate(leaves):
            d = torch.randn_like(x)
            slope = lambda h: (value(*[y + h * d if j == i else y for j, y in enumerate(leaves)])  # noqa: E731
                               - value(*[y - h * d if j == i else y for j, y in enumerate(leaves)])) / (2 * h)
            want = (4 * slope(0.5) - slope(1.0)) / 3
            got = float((grads[i].double() * d.double()).sum())
            size = float((grads[i].double() * d.double()).abs().sum())
            assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_only_some_inputs_need_a_gradient_and_unused_outputs():
    q, k, v, do, s0, ds = (dev(x) for x in make(1, 70, 2, 2, 2, 32, 32, torch.bfloat16))
    g = dev(decays(2))
    full = [x.clone().requires_grad_() for x in (q, k, v, s0)]
    o, s = V.linear_attention_fn(*full[:3], g, None, full[3], True)
    want = torch.autograd.grad([o, s], full, [do, ds])
    for i in range(3):
        args = [q, k, v]
        args[i] = args[i].clone().requires_grad_()
        o, s = V.linear_attention_fn(*args, g, None, s0, True)
        (got,) = torch.autograd.grad([o, s], args[i], [do, ds])
        assert torch.equal(got, want[i])
    s_leaf = s0.clone().requires_grad_()
    _, s = V.linear_attention_fn(q, k, v, g, None, s_leaf, True)
    (got,) = torch.autograd.grad(s, s_leaf, ds)  # the output itself is not used
    ref = ds * torch.exp(70 * g.double()).float().view(1, 2, 1, 1)
    assert torch.allclose(got, ref, rtol=1e-5, atol=1e-6)
    with pytest.raises(RuntimeError):
        o, _ = V.linear_attention_fn(full[0], k, v, g, None, s0, True)
        (x,) = torch.autograd.grad(o, full[0], do, create_graph=True)
        x.sum().backward()


# ------------------------------------------------------------------------------------------------ one token


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,Hv,Dk,Dv", [(1, 1, 1, 1, 1), (4, 1, 1, 160, 160), (6, 2, 3, 72, 88), (2, 2, 2, 256, 256), (2, 1, 2, 33, 17),
                                           (2, 2, 1, 128, 30)])
def test_update_tokens(dtype, H, Hk, Hv, Dk, Dv):
    dt = DTYPES[dtype]
    B, steps = 3, 5
    q, k, v, _, s0, _ = make(B, steps, H, Hk, Hv, Dk, Dv, dt)
    g = decays(H)
    state = dev(s0).clone()
    outs = [V.linear_attention_update(dev(q[:, t]), dev(k[:, t]), dev(v[:, t]), state, dev(g)) for t in range(steps)]
    ref, ref_s = O.linear_attention(q, k, v, g, initial=s0)
    M, M_s = magnitudes(q, k, v, g, s0)
    check(torch.stack(outs, 1), ref, tolerance(ref, M, dt, Dk, 64 * steps, False), "out")
    check(state, ref_s, tolerance(ref_s, M_s, dt, Dk, 64 * steps, False, torch.float32), "state")


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.int64, torch.float32, torch.bfloat16])
def test_update_leaves_idle_rows_alone(mask_dtype):
    B, H, D = 5, 2, 64
    q, k, v, _, s0, _ = make(B, 1, H, H, H, D, D, torch.bfloat16)
    m = torch.tensor([1, 0, 1, 0, 0]).to(mask_dtype)
    for x in (q, k, v):
        x[m == 0] = float("nan")
    s0[1] = float("nan")
    state = dev(s0).clone()
    o = V.linear_attention_update(dev(q[:, 0]), dev(k[:, 0]), dev(v[:, 0]), state, dev(decays(H)), attention_mask=dev(m))
    idle = m == 0
    assert torch.equal(state.cpu()[idle].view(torch.int32), s0[idle].view(torch.int32)) and not o.cpu()[idle].any()
    ref, ref_s = O.linear_attention(q[~idle], k[~idle], v[~idle], decays(H), initial=s0[~idle])
    M, M_s = magnitudes(q[~idle], k[~idle], v[~idle], decays(H), s0[~idle])
    check(o.cpu()[~idle], ref[:, 0], tolerance(ref, M, torch.bfloat16, D, 64, False)[:, 0], "out")
    check(state.cpu()[~idle], ref_s, tolerance(ref_s, M_s, torch.bfloat16, D, 64, False, torch.float32), "state")


@pytest.mark.parametrize("view", ["slice of a pool", "transposed state", "odd offset", "heads inside"])
def test_update_state_layouts(view):
    B, H, Dk, Dv = 3, 2, 64, 48
    q, k, v, _, s0, _ = make(B, 1, H, H, H, Dk, Dv, torch.float16)
    if view == "slice of a pool":
        pool = torch.full((6, H, Dk, Dv), 3.0, device=DEV)
        state = pool[2:5]
    elif view == "transposed state":
        state = torch.empty(B, H, Dv, Dk, device=DEV).transpose(2, 3)
    elif view == "odd offset":
        state = torch.empty(B * H * Dk * Dv + 1, device=DEV)[1:].view(B, H, Dk, Dv)
    else:
        state = torch.empty(B, Dk, H, Dv, device=DEV).transpose(1, 2)
    state.copy_(s0)
    qkv = torch.cat([dev(x[:, 0]).reshape(B, -1) for x in (q, k, v)], 1)
    qq, kk, vv = (p.unflatten(1, (H, -1)) for p in qkv.split([H * Dk, H * Dk, H * Dv], 1))
    out = torch.empty(H, B, Dv, dtype=torch.float16, device=DEV).transpose(0, 1)
    o = V.linear_attention_update(qq, kk, vv, state, dev(decays(H)), out=out)
    assert o is out
    ref, ref_s = O.linear_attention(q, k, v, decays(H), initial=s0)
    M, M_s = magnitudes(q, k, v, decays(H), s0)
    check(o, ref[:, 0], tolerance(ref, M, torch.float16, Dk, 64, False)[:, 0], "out")
    check(state, ref_s, tolerance(ref_s, M_s, torch.float16, Dk, 64, False, torch.float32), "state")
    if view == "slice of a pool":
        assert (pool[:2] == 3).all() and (pool[5:] == 3).all()


def test_prompt_then_tokens_equal_the_whole_prompt():
    q, k, v, *_ = make(2, 100, 4, 1, 1, 160, 160, torch.bfloat16)
    g = dev(decays(4))
    _, state = V.linear_attention_fn(*(dev(x[:, :90]) for x in (q, k, v)), g, None, None, True)
    outs = [V.linear_attention_update(*(dev(x[:, t]) for x in (q, k, v)), state, g) for t in range(90, 100)]
    ref, ref_s = O.linear_attention(q, k, v, decays(4))
    M, M_s = magnitudes(q, k, v, decays(4))
    check(torch.stack(outs, 1), ref[:, 90:], tolerance(ref, M, torch.bfloat16, 160, 1000, True)[:, 90:], "tokens")
    check(state, ref_s, tolerance(ref_s, M_s, torch.bfloat16, 160, 1000, True, torch.float32), "state")


# ------------------------------------------------------------------------------------------------ streams and graphs


def test_two_streams_at_once():
    cases = [make(1, 2000, 2, 2, 2, 64, 64, torch.bfloat16, s) for s in range(2)]
    g = dev(decays(2))
    args = [[dev(x) for x in c[:3]] for c in cases]
    want = [V.linear_attention_fn(*a, g, None, None, True) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = V.linear_attention_fn(*args[i], g, None, None, True)
    torch.cuda.synchronize()
    for (o, s), (wo, ws) in zip(got, want):
        assert torch.equal(o, wo) and torch.equal(s, ws)


def test_captured_and_replayed_prompt_training_and_tokens():
    q, k, v, do, s0, ds = (dev(x) for x in make(1, 900, 2, 1, 1, 64, 64, torch.bfloat16))
    g = dev(decays(2))
    state = s0.clone()
    V.linear_attention_bwd(q, k, v, g, do, None, s0, ds)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = V.linear_attention_fn(q, k, v, g, None, s0, True)
        grads = V.linear_attention_bwd(q, k, v, g, do, None, s0, ds)
        tok = V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], state, g)
    for seed in (1, 2):
        new = make(1, 900, 2, 1, 1, 64, 64, torch.bfloat16, seed)
        for x, y in zip((q, k, v, do, s0, ds), new):
            x.copy_(y)
        state.copy_(s0)
        graph.replay()
        torch.cuda.synchronize()
        wo, ws = V.linear_attention_fn(q, k, v, g, None, s0, True)
        assert torch.equal(o, wo) and torch.equal(s, ws)
        for a, b in zip(grads, V.linear_attention_bwd(q, k, v, g, do, None, s0, ds)):
            assert torch.equal(a, b)
        again = s0.clone()
        assert torch.equal(tok, V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], again, g)) and torch.equal(state, again)


def test_results_repeat_bit_for_bit():
    q, k, v, do, s0, ds = (dev(x) for x in make(2, 300, 4, 2, 1, 64, 64, torch.bfloat16))
    g = dev(decays(4))
    first = V.linear_attention_bwd(q, k, v, g, do, None, s0, ds)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, V.linear_attention_bwd(q, k, v, g, do, None, s0, ds)))


@pytest.mark.parametrize("dtype,kernel", [("bf16", "tc"), ("bf16", "mma"), ("f16", "mma"), ("f32", "simt")])
@pytest.mark.parametrize("which", ["right", "left", "holes"])
def test_long_masked_rows(dtype, kernel, which):
    """Many chunks: whole chunks of padding at either end, rows without a token, holes."""
    T = 900
    t = torch.arange(T)[None]
    lens = torch.tensor([[900], [517], [128], [0]])
    m = {"right": t < lens, "left": t >= T - lens, "holes": (t // 131) % 2 == torch.tensor([[0], [1], [0], [1]])}[which]
    backward_case(DTYPES[dtype], 4, T, 2, 1, 2, 64, 48, mask=m, init=True, final=True, poison=float("nan"), kernel=kernel)
    forward_case(DTYPES[dtype], 4, T, 2, 1, 2, 64, 48, mask=m, init=True, final=True, poison=float("nan"), kernel=kernel)
    forward_case(DTYPES[dtype], 4, T, 2, 1, 2, 64, 48, mask=m, init=True, final=True, kernel=kernel, segments=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(dtype):
    """Tokens far apart in memory: the last lies more than 2^32 elements behind the first."""
    dt = DTYPES[dtype]
    T, H, D, far = 300, 1, 32, 1 << 24
    q, k, v, do, *_ = make(1, T, H, H, H, D, D, dt)
    buf = torch.empty(T * far, dtype=dt, device=DEV).view(1, T, far)
    views = [buf[:, :, i * D: (i + 1) * D].unflatten(-1, (H, D)) for i in range(4)]
    for x, y in zip(views, (q, k, v)):
        x.copy_(y)
    out = torch.empty(T * far, dtype=dt, device=DEV).view(1, T, far)[:, :, :D].unflatten(-1, (H, D))
    g = decays(H)
    V.linear_attention_fn(*views[:3], dev(g), out=out)
    ref, _ = O.linear_attention(q, k, v, g)
    M, _ = magnitudes(q, k, v, g)
    check(out, ref, tolerance(ref, M, dt, D, T, dt != torch.float32), "out")


def test_update_of_states_far_apart():
    far = (1 << 31) + 64
    pool = torch.empty(3 * far, device=DEV)
    q, k, v, _, s0, _ = make(3, 1, 2, 2, 2, 32, 32, torch.bfloat16)
    state = pool.as_strided((3, 2, 32, 32), (far, 1024, 32, 1))
    state.copy_(s0)
    g = decays(2)
    o = V.linear_attention_update(dev(q[:, 0]), dev(k[:, 0]), dev(v[:, 0]), state, dev(g))
    ref, ref_s = O.linear_attention(q, k, v, g, initial=s0)
    M, M_s = magnitudes(q, k, v, g, s0)
    check(o, ref[:, 0], tolerance(ref, M, torch.bfloat16, 32, 64, False)[:, 0], "out")
    check(state, ref_s, tolerance(ref_s, M_s, torch.bfloat16, 32, 64, False, torch.float32), "state")


@pytest.mark.parametrize("dtype,kernel", [("bf16", "tc"), ("f16", "mma"), ("f32", "simt")])
def test_whole_and_partly_masked_chunks_in_every_order(dtype, kernel):
    """Rows whose chunks of 128 are whole, holed or empty, in many orders."""
    T, B = 128 * 7 + 50, 24
    g = torch.Generator().manual_seed(11)
    kind = torch.randint(0, 3, (B, 8), generator=g).repeat_interleave(128, 1)[:, :T]  # 0 whole, 1 holed, 2 empty
    m = (kind == 0) | ((kind == 1) & (torch.rand(B, T, generator=g) < 0.7))
    for segments in (0, 3):
        forward_case(DTYPES[dtype], B, T, 1, 1, 1, 32, 32, mask=m, init=True, final=True, poison=float("nan"), kernel=kernel, segments=segments)
        backward_case(DTYPES[dtype], B, T, 1, 1, 1, 32, 32, mask=m, init=True, final=True, poison=float("nan"), kernel=kernel, segments=segments)


def test_no_wait_of_a_kernel_has_run_out():
    assert V.tma_timeouts() == 0
