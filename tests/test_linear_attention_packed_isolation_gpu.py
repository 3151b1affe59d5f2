"""A bad value in one sequence of a packed row stays in that sequence, and behind the token that has it."""
import pytest
import torch

import viby_model_b200 as V
from linear_cases import DTYPES, check, decays, grad_magnitudes, magnitudes, make, tolerance
from oracle import linear_oracle as O
from test_linear_attention_gpu import dev

pytestmark = pytest.mark.gpu

FORMS = [("bf16", "tc", 64, 64), ("bf16", "tc", 160, 136), ("bf16", "mma", 64, 64), ("bf16", "mma", 160, 160), ("f16", "mma", 64, 72),
         ("f16", "mma", 256, 64), ("f32", "simt", 40, 100), ("f16", "simt", 33, 17)]
LENGTHS = [70, 30, 1, 200, 5, 94, 160]
# sequence, token in it, what is bad
PLACES = [(0, 69, "v"), (1, 0, "k"), (2, 0, "q"), (3, 140, "v"), (3, 10, "k"), (6, 0, "v"), (5, 50, "all")]
T = sum(LENGTHS)


def rows(H, Dk, Dv, dtype, places, bad):
    """Clean inputs, poisoned ones, and for each token whether its own sequence is clean up to it and from it on."""
    q, k, v, do, *_ = make(1, T, H, 1, H, Dk, Dv, dtype, 7)
    q, k, v, do = ([x, x.clone()] for x in (q, k, v, do))
    before, after = torch.ones(T, dtype=torch.bool), torch.ones(T, dtype=torch.bool)
    for sequence, token, what in places:
        first = sum(LENGTHS[:sequence])
        at, last = first + token, first + LENGTHS[sequence]
        for name, x in (("q", q), ("k", k), ("v", v), ("do", do)):
            if what in (name, "all"):
                x[1][0, at, :, ::5] = bad
        before[at:last] = False
        after[first:at + 1] = False
    return q, k, v, do, before, after


@pytest.mark.parametrize("dtype,kernel,Dk,Dv", FORMS)
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("segments", [1, 3])
def test_outputs_of_the_other_sequences(dtype, kernel, Dk, Dv, bad, segments):
    dt, H = DTYPES[dtype], 2
    g = decays(H)
    seq = V.seq_idx_from_lengths(LENGTHS)
    for places in [[p] for p in PLACES] + [PLACES]:
        q, k, v, _, before, _ = rows(H, Dk, Dv, dt, places, bad)
        o = V.linear_attention_fn(dev(q[1]), dev(k[1]), dev(v[1]), dev(g), dev(seq), kernel=kernel, segments=segments)
        ref, _ = O.linear_attention(q[0], k[0], v[0], g, seq_idx=seq)
        M, _ = magnitudes(q[0], k[0], v[0], g, seq_idx=seq)
        tol = tolerance(ref, M, dt, Dk, T, kernel != "simt")
        check(o[:, dev(before)], ref[:, before], tol[:, before], f"tokens that {places} must not reach")
        for sequence, token, what in places:  # and the token itself shows it
            at = sum(LENGTHS[:sequence]) + token
            assert not torch.isfinite(o[0, at]).all(), (sequence, token, what)


@pytest.mark.parametrize("dtype,kernel,Dk,Dv", FORMS)
@pytest.mark.parametrize("segments", [1, 2])
def test_gradients_of_the_other_sequences(dtype, kernel, Dk, Dv, segments):
    """Shared key heads: their gradients are sums over the heads that read them."""
    dt, H, bad = DTYPES[dtype], 2, float("inf")
    g = decays(H)
    seq = V.seq_idx_from_lengths(LENGTHS)
    for places in ([(3, 140, "do")], [(1, 0, "v"), (5, 50, "q")], [(0, 69, "all"), (6, 3, "k")]):
        q, k, v, do, before, after = rows(H, Dk, Dv, dt, places, bad)
        got = V.linear_attention_bwd(*(dev(x[1]) for x in (q, k, v)), dev(g), dev(do[1]), dev(seq), kernel=kernel, segments=segments)
        ref = O.grads(q[0], k[0], v[0], g, do[0], seq_idx=seq)
        M = grad_magnitudes(q[0], k[0], v[0], g, do[0], seq_idx=seq)
        for x, r, m, clean, name in zip(got, ref, M, (before, after, after), ("dq", "dk", "dv")):
            tol = tolerance(r, m, dt, max(Dk, Dv) + H, T, kernel != "simt")
            check(x[:, dev(clean)], r[:, clean], tol[:, clean], f"{name}, {places}")


@pytest.mark.parametrize("dtype,kernel", [("bf16", "tc"), ("f16", "mma"), ("f32", "simt")])
def test_layouts_and_long_sequences(dtype, kernel):
    """Outputs with strides of their own, sequences over many parts of 256 tokens behind a bad neighbour, several rows."""
    dt, H, D, lengths = DTYPES[dtype], 2, 48, [3, 1400, 97]
    n = sum(lengths)
    q, k, v, *_ = make(2, n, H, H, H, D, D, dt, 9)
    g = decays(H)
    seq = V.seq_idx_from_lengths(lengths).expand(2, -1).contiguous()
    ref, _ = O.linear_attention(q, k, v, g, seq_idx=seq)
    M, _ = magnitudes(q, k, v, g, seq_idx=seq)
    tol = tolerance(ref, M, dt, D, n, kernel != "simt")
    bad = [x.clone() for x in (q, k, v)]
    bad[2][1, 1, 0, 5] = float("inf")  # row 1, sequence 0, head 0
    for out in (None, torch.empty(2, H, D, n, dtype=dt, device="cuda").permute(0, 3, 1, 2)):
        o = V.linear_attention_fn(*(dev(x) for x in bad), dev(g), dev(seq), kernel=kernel, out=out)
        check(o[0], ref[0], tol[0], "the other row")
        check(o[1, :, 1], ref[1, :, 1], tol[1, :, 1], "the other head")
        check(o[1, 3:], ref[1, 3:], tol[1, 3:], "the sequences behind")
        check(o[1, :1], ref[1, :1], tol[1, :1], "the token before")
        assert not torch.isfinite(o[1, 1, 0, 5]) and not torch.isfinite(o[1, 2, 0, 5])
    clean = V.linear_attention_fn(dev(q), dev(k), dev(v), dev(g), dev(seq), kernel=kernel)
    assert torch.equal(clean[0], o[0]) and torch.equal(clean[1, :, 1], o[1, :, 1])  # untouched, bit for bit


def test_captured_and_replayed():
    q, k, v, *_ = (dev(x) for x in make(1, 300, 2, 2, 2, 64, 64, torch.bfloat16))
    g, seq = dev(decays(2)), V.seq_idx_from_lengths([100, 200], "cuda")
    V.linear_attention_fn(q, k, v, g, seq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = V.linear_attention_fn(q, k, v, g, seq)
    graph.replay()
    want = o.clone()
    v[0, 50] = float("nan")
    graph.replay()
    torch.cuda.synchronize()
    assert torch.isfinite(o[:, 100:]).all() and torch.isfinite(o[:, :50]).all() and o[0, 50:100].isnan().all()
    v[0, 50] = 0
    k[0, 50] = 0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.isfinite(o).all() and torch.equal(o[:, 128:], want[:, 128:])


@pytest.mark.parametrize("dtype,kernel,D", [("bf16", "tc", 64), ("bf16", "tc", 160), ("bf16", "mma", 128), ("f16", "mma", 64), ("f32", "simt", 40)])
@pytest.mark.parametrize("seed", range(8))
def test_random_lengths_and_places(dtype, kernel, D, seed):
    """Outputs and gradients of every token that a bad value must not reach are what they are without it (within the roundings of
    another way to compute them)."""
    dt, H = DTYPES[dtype], 2
    r = torch.Generator().manual_seed(100 + seed)
    lengths = []
    while sum(lengths) < 700:
        lengths.append(int(torch.randint(1, (6, 60, 300)[seed % 3], (1,), generator=r)))
    n = sum(lengths)
    q, k, v, do, *_ = make(1, n, H, 1, H, D, D, dt, seed)
    g = dev(decays(H))
    seq = dev(V.seq_idx_from_lengths(lengths))
    ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    args = dict(kernel=kernel, segments=1 + seed % 3)
    want = (V.linear_attention_fn(dev(q), dev(k), dev(v), g, seq, **args), *V.linear_attention_bwd(dev(q), dev(k), dev(v), g, dev(do), seq, **args)[:3])
    M = magnitudes(q, k, v, g.cpu(), seq_idx=seq.cpu())[0], *grad_magnitudes(q, k, v, g.cpu(), do, seq_idx=seq.cpu())[:3]
    before, after = torch.ones(n, dtype=torch.bool), torch.ones(n, dtype=torch.bool)
    for _ in range(int(torch.randint(1, 4, (1,), generator=r))):
        t = int(torch.randint(0, n, (1,), generator=r))
        x = (q, k, v, do)[int(torch.randint(0, 4, (1,), generator=r))]
        x[0, t, int(torch.randint(0, x.shape[2], (1,), generator=r)), int(torch.randint(0, D, (1,), generator=r))] = (float("inf"), float("nan"))[seed % 2]
        same = ids == ids[t]
        before &= ~(same & (torch.arange(n) >= t))
        after &= ~(same & (torch.arange(n) <= t))
    got = (V.linear_attention_fn(dev(q), dev(k), dev(v), g, seq, **args), *V.linear_attention_bwd(dev(q), dev(k), dev(v), g, dev(do), seq, **args)[:3])
    for x, w, m, clean, name in zip(got, want, M, (before, before, after, after), ("out", "dq", "dk", "dv")):
        w = w.cpu().double()
        tol = 2 * tolerance(w, m, dt, D + H, n, kernel != "simt")  # of either way
        check(x[:, dev(clean)], w[:, clean], tol[:, clean], f"{name}, {lengths}")


@pytest.mark.parametrize("dtype,kernel,D", [("bf16", "tc", 64), ("bf16", "mma", 64), ("f16", "mma", 160), ("f32", "simt", 40)])
@pytest.mark.parametrize("places", [[("v", 1)], [("v", 1), ("v", 700)], [("k", 2), ("q", 255), ("q", 256)], [("k", 2), ("q", 255), ("v", 300)],
                                    [("q", 255), ("v", 300)], [("q", 255), ("q", 256), ("v", 257)], [("q", 511), ("k", 512), ("v", 1020)],
                                    [("v", 1002), ("k", 1044)], [("v", 1003), ("v", 1342)], [("q", 767), ("v", 1002), ("k", 1030)]])
def test_bad_values_at_the_borders_of_parts(dtype, kernel, D, places):
    """Sequences over several parts of 256 tokens: one part repairs what a bad state did to the others, each what is its own."""
    dt, H, lengths = DTYPES[dtype], 2, [3, 1000, 40, 300]
    n = sum(lengths)
    q, k, v, *_ = make(1, n, H, H, H, D, D, dt, 11)
    g = decays(H, "none" if D == 64 else "mixed")
    seq = V.seq_idx_from_lengths(lengths)
    ref, _ = O.linear_attention(q, k, v, g, seq_idx=seq)
    M, _ = magnitudes(q, k, v, g, seq_idx=seq)
    clean = torch.ones(n, dtype=torch.bool)
    for what, at in places:
        {"q": q, "k": k, "v": v}[what][0, at, :, 3] = float("inf")
        if what == "q":
            clean[at] = False
        else:
            clean[(seq[0] == seq[0, at]) & (torch.arange(n) >= at)] = False
    for segments in (1, 2):
        o = V.linear_attention_fn(dev(q), dev(k), dev(v), dev(g), dev(seq), kernel=kernel, segments=segments)
        check(o[:, dev(clean)], ref[:, clean], tolerance(ref, M, dt, D, n, kernel != "simt")[:, clean], str(places))
