"""Every compiled form of the linear attention kernels over many chunks: heads of 128, 160 and 256 with masks, packed rows,
split time axes, both directions; the warp-level kernel for bf16; own scales; fp16 values far outside fp16's range; the bits
that the state keeps.  Tolerances: tests/linear_cases.py, or derived beside the test."""
import pytest
import torch

import viby_model_b200 as V
from linear_cases import DTYPES, check, decays, grad_magnitudes, magnitudes, make, tolerance
from oracle import linear_oracle as O
from test_linear_attention_gpu import backward_case, dev, forward_case

pytestmark = pytest.mark.gpu

# (type, kernel, Dk, Dv): tcgen05 with two buffers of keys and with one; warp-level with 64, 128, 160 x 80 and 256 rows
FORMS = [("bf16", "tc", 128, 128), ("bf16", "tc", 160, 160), ("bf16", "tc", 136, 72), ("bf16", "tc", 72, 160),
         ("bf16", "mma", 64, 64), ("bf16", "mma", 128, 96), ("bf16", "mma", 160, 160), ("bf16", "mma", 144, 88), ("bf16", "mma", 256, 200),
         ("f16", "mma", 128, 128), ("f16", "mma", 160, 160), ("f16", "mma", 200, 256), ("f32", "simt", 160, 100)]
T = 400  # four chunks of 128, seven of 64; the last ones are not whole


def variant_masks(B):
    t = torch.arange(T)[None]
    lens = torch.tensor([T, 259])[:B, None]
    holes = torch.rand(B, T, generator=torch.Generator().manual_seed(5)) < 0.5
    holes[:, 128:256] = True   # a whole chunk between chunks with holes
    holes[:, 384:] = False
    return {"right": t < lens, "left": t >= T - lens, "holes": holes}


@pytest.mark.parametrize("dtype,kernel,Dk,Dv", FORMS)
@pytest.mark.parametrize("which", ["none", "right", "left", "holes"])
@pytest.mark.parametrize("segments", [1, 3])
def test_prompts(dtype, kernel, Dk, Dv, which, segments):
    mask = None if which == "none" else variant_masks(2)[which]
    forward_case(DTYPES[dtype], 2, T, 2, 1, 2, Dk, Dv, mask=mask, init=True, final=True, poison=float("nan"), kernel=kernel, segments=segments)
    assert V.last_kernel() == f"linear_{kernel}"


@pytest.mark.parametrize("dtype,kernel,Dk,Dv", FORMS)
@pytest.mark.parametrize("segments", [1, 2])
def test_packed_prompts(dtype, kernel, Dk, Dv, segments):
    seq = V.seq_idx_from_lengths([100, 28, 1, 130, 127, 14])
    forward_case(DTYPES[dtype], 1, T, 2, 1, 2, Dk, Dv, seq=seq, kernel=kernel, segments=segments)


@pytest.mark.parametrize("dtype,kernel,Dk,Dv", [f for f in FORMS if f[2:] not in ((64, 64), (136, 72), (160, 100))])
@pytest.mark.parametrize("which,segments", [("none", 1), ("none", 3), ("right", 3), ("left", 1), ("holes", 1), ("holes", 3), ("packed", 1), ("packed", 3)])
def test_gradients(dtype, kernel, Dk, Dv, which, segments):
    if which == "packed":
        backward_case(DTYPES[dtype], 1, T, 2, 1, 2, Dk, Dv, seq=V.seq_idx_from_lengths([100, 28, 1, 130, 127, 14]), kernel=kernel, segments=segments)
    else:
        mask = None if which == "none" else variant_masks(2)[which][1:]
        backward_case(DTYPES[dtype], 1, T, 2, 1, 2, Dk, Dv, mask=mask, init=True, final=True, poison=float("nan"), kernel=kernel, segments=segments)


@pytest.mark.parametrize("D", [128, 160])
@pytest.mark.parametrize("what", ["heads", "rows"])
def test_broadcast_keys_of_large_heads(D, what):
    """Tensor maps have no zero strides: these bf16 calls go to the warp-level kernel by themselves."""
    def spread(q, k, v):
        return q, (k[:, :, :1].expand_as(k) if what == "heads" else k[:1].expand_as(k)), v

    B, H, n = 2, 2, 200
    q, k, v, *_ = make(B, n, H, H, H, D, D, torch.bfloat16, 0)
    kk = (k[:, :, :1] if what == "heads" else k[:1]).expand_as(k)
    g = decays(H)
    o, s = V.linear_attention_fn(*spread(dev(q), dev(k), dev(v)), dev(g), None, None, True)
    assert V.last_kernel() == "linear_mma"
    ref, ref_s = O.linear_attention(q, kk, v, g)
    M, M_s = magnitudes(q, kk, v, g)
    check(o, ref, tolerance(ref, M, torch.bfloat16, D, n, True), "out")
    check(s, ref_s, tolerance(ref_s, M_s, torch.bfloat16, D, n, True, torch.float32), "state")


@pytest.mark.parametrize("dtype,kernel", [("bf16", "tc"), ("bf16", "mma"), ("f16", "mma"), ("f32", "simt"), ("f16", None)])
def test_own_scales(dtype, kernel):
    """Values given by the caller, also 0 and negative ones, one after another on the same call form and back again."""
    dt, n, D = DTYPES[dtype], 150, 48
    q, k, v, do, s0, ds = make(2, n, 2, 1, 2, D, D, dt)
    g = decays(2)
    on = [dev(x) for x in (q, k, v, do, s0, ds)]
    seen = {}
    for scale in (None, 0.0, -0.75, 2.5, 1, None, -0.75, 0.0):
        o, s = V.linear_attention_fn(*on[:3], dev(g), None, on[4], True, scale=scale, kernel=kernel)
        grads = V.linear_attention_bwd(*on[:3], dev(g), on[3], None, on[4], on[5], scale=scale, kernel=kernel)
        state = on[4].clone()
        token = V.linear_attention_update(on[0][:, 0], on[1][:, 0], on[2][:, 0], state, dev(g), scale=scale)
        size = D ** -0.5 if scale is None else abs(scale)
        ref, ref_s = O.linear_attention(q, k, v, g, initial=s0, scale=scale)
        M, M_s = magnitudes(q, k, v, g, s0, scale=size)
        tc = kernel != "simt"
        check(o, ref, tolerance(ref, M, dt, D, n, tc), f"out, scale {scale}")
        check(s, ref_s, tolerance(ref_s, M_s, dt, D, n, tc, torch.float32), f"state, scale {scale}")
        ref_g = O.grads(q, k, v, g, do, initial=s0, dfinal=ds, scale=scale)
        M_g = grad_magnitudes(q, k, v, g, do, s0, ds, scale=size)
        for x, r, m, name in zip(grads[:3], ref_g, M_g, ("dq", "dk", "dv")):
            check(x, r, tolerance(r, m, dt, D + 2, n, tc), f"{name}, scale {scale}")
        check(grads[3], ref_g[3], tolerance(ref_g[3], M_g[3], dt, D, n, tc, torch.float32), f"dinitial, scale {scale}")
        first, _ = O.linear_attention(q[:, :1], k[:, :1], v[:, :1], g, initial=s0, scale=scale)
        M_1, _ = magnitudes(q[:, :1], k[:, :1], v[:, :1], g, s0, scale=size)
        check(token, first[:, 0], tolerance(first, M_1, dt, D, 64, False)[:, 0], f"token, scale {scale}")
        if scale == 0:
            assert not o.any() and not grads[0].any()
        if scale in seen:  # the same call again, with others in between
            assert torch.equal(o, seen[scale][0]) and torch.equal(s, seen[scale][1])
        seen[scale] = (o, s)


# powers of two on q, k, v, the initial state and the scale: states and products far outside fp16's range (its largest value is
# below 2^16, its smallest normal one 2^-14) while inputs and outputs stay inside it
RANGES = {"large state": (-8, 0, 0, 20, None), "larger state": (-14, 0, 4, 26, None), "small state": (10, -12, -10, -24, None),
          "large products": (7, 7, -9, 0, 1.0), "larger products": (10, 9, -14, 0, 0.5), "small products": (-10, -10, 12, 0, 2.0 ** -6),
          "products smaller than any": (-13, -13, 13, -60, 2.0 ** -10), "both large": (5, 9, 0, 24, 2.0 ** -21)}


@pytest.mark.parametrize("kernel", ["mma", "simt"])
@pytest.mark.parametrize("D", [64, 160])
@pytest.mark.parametrize("name", RANGES)
def test_fp16_states_and_products_outside_the_range_of_fp16(name, D, kernel):
    eq, ek, ev, es, scale = RANGES[name]
    n = 200
    q, k, v, _, s0, _ = make(1, n, 2, 2, 1, D, D, torch.float32)
    q, k, v = ((x * 2.0 ** e).half() for x, e in ((q, eq), (k, ek), (v, ev)))
    s0 = s0 * 2.0 ** es
    g = decays(2)
    ref, ref_s = O.linear_attention(q, k, v, g, initial=s0, scale=scale)
    assert float(ref.abs().max()) < 65504  # the case itself
    M, M_s = magnitudes(q, k, v, g, s0, scale=scale)
    for segments in (1, 2):
        o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), dev(g), None, dev(s0), True, scale=scale, kernel=kernel, segments=segments)
        check(o, ref, tolerance(ref, M, torch.float16, D, n, kernel == "mma"), "out")
        check(s, ref_s, tolerance(ref_s, M_s, torch.float16, D, n, kernel == "mma", torch.float32), "state")


@pytest.mark.parametrize("kernel", ["mma", "simt"])
@pytest.mark.parametrize("exps", [(-6, -10, -12, -8, 18, 19), (7, -9, -9, -5, -20, -18)])
def test_fp16_gradients_outside_the_range_of_fp16(exps, kernel):
    n, D = 150, 64
    given = make(1, n, 2, 1, 2, D, D, torch.float32)
    x = [t * 2.0 ** e for t, e in zip(given, exps)]
    q, k, v, do = (t.half() for t in x[:4])
    s0, ds = x[4:]
    g = decays(2)
    ref = O.grads(q, k, v, g, do, initial=s0, dfinal=ds)
    M = grad_magnitudes(q, k, v, g, do, s0, ds)
    assert all(float(r.abs().max()) < 65504 for r in ref[:3])
    got = V.linear_attention_bwd(dev(q), dev(k), dev(v), dev(g), dev(do), None, dev(s0), dev(ds), kernel=kernel)
    tc = kernel == "mma"
    for i, what in enumerate(("dq", "dk", "dv")):
        check(got[i], ref[i], tolerance(ref[i], M[i], torch.float16, D + 2, n, tc), what)
    check(got[3], ref[3], tolerance(ref[3], M[3], torch.float16, D, n, tc, torch.float32), "dinitial")


@pytest.mark.parametrize("dtype,kernel,D", [("bf16", "tc", 64), ("bf16", "tc", 160), ("bf16", "mma", 64), ("bf16", "mma", 160), ("bf16", "mma", 256),
                                            ("f16", "mma", 64), ("f16", "mma", 160), ("f32", "simt", 64)])
@pytest.mark.parametrize("n,segments", [(2, 1), (300, 1), (300, 2)])
def test_the_state_keeps_its_bits(dtype, kernel, D, n, segments):
    """One key that counts, then keys of zero: S = a^(n-1) k v^T.  Relative error of an element: the powers of the decay 2^-24
    for each of the chunks that carry it (five of 64 tokens at most), the weighted value or key 2^-24, and, because sums with
    zeros are exact, one truncation of 2^-22 for each of the three parts it is split into; two parts of fp16 keys leave
    2^-23: below 2^-20 in all.  Dropping the last part would leave 2^-17 of bf16 and 2^-12 of fp16 values."""
    dt = DTYPES[dtype]
    q, k, v, *_ = make(1, n, 2, 2, 2, D, D, dt, 3)
    k[:, 1:] = 0
    g = torch.tensor([-0.013, -0.0021])
    _, s = V.linear_attention_fn(dev(q), dev(k), dev(v), dev(g), None, None, True, kernel=kernel, segments=segments)
    a = torch.exp(g.double() * (n - 1)).view(1, 2, 1, 1)
    want = a * k[:, 0].double()[..., None] * v[:, 0].double()[..., None, :]
    off = ((s.cpu().double() - want).abs() / want.abs().clamp(min=1e-30)).max()
    assert float(off) < 2.0 ** -20, float(off) * 2.0 ** 20


def test_no_wait_of_a_kernel_has_run_out():
    assert V.tma_timeouts() == 0
