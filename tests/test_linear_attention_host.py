"""Refusals of the linear attention and cache page operators, through Python and the C ABI.  Nothing is launched; runs
without a GPU.  The oracle's own pieces are checked against each other here too."""
import ctypes as C
import types

import pytest
import torch

import viby_model_b200 as V
from oracle import linear_oracle as O
from viby_model_b200 import _cabi, canon_cache as CC


def qkv(B=1, T=4, H=2, Hk=2, Hv=2, Dk=8, Dv=8, dtype=torch.float32):
    return torch.zeros(B, T, H, Dk, dtype=dtype), torch.zeros(B, T, Hk, Dk, dtype=dtype), torch.zeros(B, T, Hv, Dv, dtype=dtype)


def refused(match, *args, **kw):
    with pytest.raises(ValueError, match=match):
        V.linear_attention_fn(*args, **kw)


def test_prompt_refusals():
    q, k, v = qkv()
    g = torch.zeros(2)
    refused("CUDA device", q, k, v, g)
    refused("4D q", q[0], k, v, g)
    refused("one dtype", q, k.half(), v, g)
    refused("unsupported dtype", q.double(), k.double(), v.double(), g)
    refused("does not match q shape", q, k[:, :3], v, g)
    refused("k dim", q, k[..., :4], v, g)
    refused("cannot share", *qkv(H=4, Hk=3), g)
    refused("1..256", *qkv(Dk=264), g)
    refused("1..256", *qkv(Dv=0), g)
    with pytest.raises(ValueError, match="cannot be combined"):
        V.linear_attention_fn(q, k, v, g, torch.zeros(1, 4, dtype=torch.int32), return_final_states=True)
    x = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="out="):
        V.linear_attention_fn(x, k, v, g, out=torch.zeros_like(v))
    with pytest.raises(ValueError, match="cannot be combined"):
        V.linear_attention_bwd(q, k, v, g, v, torch.zeros(1, 4, dtype=torch.int32), need_dinitial=True)


def test_update_refusals():
    q, k, v = (x[:, 0] for x in qkv())
    s = torch.zeros(1, 2, 8, 8)
    with pytest.raises(ValueError, match="CUDA device"):
        V.linear_attention_update(q, k, v, s, torch.zeros(2))
    with pytest.raises(ValueError, match="no gradient"):
        V.linear_attention_update(q.clone().requires_grad_(), k, v, s, torch.zeros(2))
    with pytest.raises(ValueError, match="3D q"):
        V.linear_attention_update(q[0], k, v, s, torch.zeros(2))


def test_a_scale_held_on_the_device_is_refused():
    """Its value could change between two calls of the same arguments, and it could want a gradient."""
    q, k, v = qkv()
    g, scale, state = torch.zeros(2), torch.tensor(0.5), torch.zeros(1, 2, 8, 8)
    for call in (lambda: V.linear_attention_fn(q, k, v, g, scale=scale), lambda: V.linear_attention_bwd(q, k, v, g, v, scale=scale),
                 lambda: V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], state, g, scale=scale)):
        with pytest.raises(TypeError, match="scale must be a number"):
            call()


def test_overlapping_states_of_large_tables():
    """Tables of more tensors than one launch takes are looked over as a whole, against all pairs byte by byte."""
    from viby_model_b200.cache_pages import _check_apart

    def shared(table, pages):
        seen = set()
        for base, size, stride in table:
            mine = {base + i * stride + j for i in range(pages) for j in range(size)}
            if seen & mine:
                return True
            seen |= mine
        return False

    # layers side by side in one pool, given twice, one byte too long at the front, in the middle, at the end, empty ones
    pool = [(16 * n, 16, 160) for n in range(10)]
    for table in (pool, pool[::-1], pool + [(160 * 4, 16, 16)], pool + [pool[3]], [(0, 17, 160)] + pool[1:], pool[:9] + [(144, 17, 160)],
                  pool[:4] + [(64, 17, 160)] + pool[5:], pool + [(32, 0, 160)], [(0, 16, 16), (64, 16, 16), (128, 4, 4)],
                  [(0, 16, 16), (63, 16, 16)], [(0, 400, 400), (100, 8, 8), (1600, 8, 8)]):
        if shared(table, 4):
            with pytest.raises(ValueError, match="overlap"):
                _check_apart(table, 4)
        else:
            _check_apart(table, 4)


def test_page_refusals():
    s = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="CUDA device"):
        V.PageTable([s])
    with pytest.raises(ValueError, match="first dimension"):
        V.PageTable([torch.tensor(1.0)])
    empty = V.PageTable([])
    empty.reorder(torch.zeros(0, dtype=torch.int64))
    empty.copy(torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    empty.free(torch.zeros(0, dtype=torch.int32))
    with pytest.raises(ValueError, match="no states"):
        empty.compact(torch.zeros(0, dtype=torch.bool))
    for bad in (torch.zeros(2), torch.zeros(2, 2, dtype=torch.int32), [0, 1]):
        with pytest.raises(ValueError):
            empty.free(bad)
    with pytest.raises(ValueError, match="same length"):
        empty.copy(torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_canon_cache_in_place_forms_need_the_gpu_and_leave_the_rest_alone():
    cache = types.SimpleNamespace(_max_layers=2)
    CC.set_state(cache, "a", 0, torch.arange(12.0).view(3, 2, 2))
    before = CC.get_state(cache, "a", 0)
    with pytest.raises(ValueError, match="CUDA device"):
        CC.reorder(cache, torch.tensor([2, 1, 0]), inplace=True)
    with pytest.raises(ValueError, match="inplace"):
        CC.reorder(cache, torch.tensor([2, 1, 0]), also=[torch.zeros(3)])
    for call in (lambda: CC.fork(cache, torch.tensor([0]), torch.tensor([1])), lambda: CC.free(cache, torch.tensor([0])),
                 lambda: CC.compact(cache, torch.ones(3, dtype=torch.bool))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    assert CC.get_state(cache, "a", 0) is before
    CC.reorder(cache, torch.tensor([2, 1, 0]))
    assert torch.equal(CC.get_state(cache, "a", 0), before[torch.tensor([2, 1, 0])])


# ------------------------------------------------------------------------------------------------- C ABI

FAKE = 1 << 20  # never dereferenced: the call is refused first


def linear_args(**kw):
    a = _cabi.LinearArgs()
    a.struct_size = C.sizeof(_cabi.LinearArgs)
    a.dtype = _cabi.VC1D_BF16
    a.batch, a.seqlen, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = 1, 4, 2, 2, 2, 8, 8
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


POINTERS = dict(q=FAKE, k=2 * FAKE, v=3 * FAKE, out=4 * FAKE, log_decay=5 * FAKE, q_strides=(64, 16, 8, 1), k_strides=(64, 16, 8, 1),
                v_strides=(64, 16, 8, 1), out_strides=(64, 16, 8, 1))


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), _cabi.VC1D_E_STRUCT),
    (dict(dtype=7), _cabi.VC1D_E_DTYPE),
    (dict(mask=FAKE, mask_dtype=77), _cabi.VC1D_E_DTYPE),
    (dict(batch=-1), _cabi.VC1D_E_SHAPE),
    (dict(heads_k=3), _cabi.VC1D_E_SHAPE),
    (dict(heads_v=0), _cabi.VC1D_E_SHAPE),
    (dict(kernel=9), _cabi.VC1D_E_SHAPE),
    (dict(segments=1000), _cabi.VC1D_E_SHAPE),
    (dict(dim_k=257), _cabi.VC1D_E_TOO_LARGE),
    (dict(seqlen=(1 << 30) + 1), _cabi.VC1D_E_TOO_LARGE),
    (dict(seq_idx=FAKE, final_state=FAKE), _cabi.VC1D_E_SHAPE),
    (dict(), _cabi.VC1D_E_NULL),
    ({**POINTERS, "out": FAKE + 64}, _cabi.VC1D_E_ALIAS),
    ({**POINTERS, "out_strides": (64, 16, 0, 1)}, _cabi.VC1D_E_STRIDE),
    ({**POINTERS, "initial_state": 6 * FAKE, "final_state": 6 * FAKE + 4, "initial_strides": (128, 64, 8, 1),
      "final_strides": (128, 64, 8, 1)}, _cabi.VC1D_E_ALIAS),
    ({**POINTERS, "workspace": 7 * FAKE + 4, "workspace_bytes": 1 << 20}, _cabi.VC1D_E_STRIDE),
    ({**POINTERS, "kernel": 2, "q": FAKE + 2}, _cabi.VC1D_E_STRIDE),
    ({**POINTERS, "kernel": 3, "dtype": _cabi.VC1D_F16}, _cabi.VC1D_E_STRIDE),
])
def test_linear_rejects_bad_arguments_without_launching(kw, code):
    before = _cabi.launch_count()
    assert _cabi.lib.vc1d_linear(C.byref(linear_args(**kw)), None) == code
    assert _cabi.launch_count() == before


def test_linear_empty_and_null():
    assert _cabi.lib.vc1d_linear(None, None) == _cabi.VC1D_E_NULL
    assert _cabi.lib.vc1d_linear_bwd(None, None) == _cabi.VC1D_E_NULL
    assert _cabi.lib.vc1d_linear_update(None, None) == _cabi.VC1D_E_NULL
    assert _cabi.lib.vc1d_pages(None, None) == _cabi.VC1D_E_NULL
    assert _cabi.lib.vc1d_linear(C.byref(linear_args(batch=0)), None) == _cabi.VC1D_OK
    assert _cabi.lib.vc1d_linear(C.byref(linear_args(seqlen=0, log_decay=FAKE)), None) == _cabi.VC1D_OK
    assert _cabi.lib.vc1d_linear_workspace(C.byref(linear_args(seqlen=0))) == 0
    assert _cabi.lib.vc1d_linear_workspace(C.byref(linear_args(dim_k=0))) == _cabi.VC1D_E_SHAPE


def test_linear_workspace_holds_the_states_of_the_parts():
    """(parts - 1) states and factors, 16 bytes aligned each."""
    a = linear_args(dtype=_cabi.VC1D_F32, seqlen=640, segments=4)
    want = 3 * 2 * 8 * 8 * 4 + 3 * 2 * 8
    assert _cabi.lib.vc1d_linear_workspace(C.byref(a)) == want
    a.segments = 1
    assert _cabi.lib.vc1d_linear_workspace(C.byref(a)) == 0


def test_linear_bwd_rejects_bad_arguments_without_launching():
    b = _cabi.LinearBwdArgs()
    b.struct_size = C.sizeof(_cabi.LinearBwdArgs)
    b.f = linear_args(**{k: v for k, v in POINTERS.items() if not k.startswith("out")})
    assert _cabi.lib.vc1d_linear_bwd(C.byref(b), None) == _cabi.VC1D_E_NULL
    b.dout, b.dq, b.dk, b.dv = 8 * FAKE, 9 * FAKE, 10 * FAKE, 10 * FAKE + 32
    for name in ("dout", "dq", "dk", "dv"):
        getattr(b, name + "_strides")[:] = (64, 16, 8, 1)
    assert _cabi.lib.vc1d_linear_bwd(C.byref(b), None) == _cabi.VC1D_E_ALIAS  # dk and dv
    b.dv = 11 * FAKE
    b.f.heads_k = 1  # shared heads: partial sums need a workspace
    assert _cabi.lib.vc1d_linear_bwd(C.byref(b), None) == _cabi.VC1D_E_NULL
    assert _cabi.lib.vc1d_linear_bwd_workspace(C.byref(b)) >= 4 * 4 * 2 * 8
    b.struct_size = 3
    assert _cabi.lib.vc1d_linear_bwd(C.byref(b), None) == _cabi.VC1D_E_STRUCT


def test_linear_update_rejects_bad_arguments_without_launching():
    before = _cabi.launch_count()

    def args(**kw):
        a = _cabi.LinearUpdateArgs()
        a.struct_size = C.sizeof(_cabi.LinearUpdateArgs)
        a.dtype = _cabi.VC1D_F16
        a.batch, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = 2, 2, 1, 2, 8, 8
        a.q, a.k, a.v, a.out, a.state, a.log_decay = (i * FAKE for i in range(1, 7))
        a.q_strides[:], a.k_strides[:], a.v_strides[:], a.out_strides[:] = (16, 8, 1), (8, 8, 1), (16, 8, 1), (16, 8, 1)
        a.state_strides[:] = (128, 64, 8, 1)
        for k, v in kw.items():
            if k.endswith("strides"):
                getattr(a, k)[:] = v
            else:
                setattr(a, k, v)
        return a

    for kw, code in ((dict(struct_size=1), _cabi.VC1D_E_STRUCT), (dict(dtype=9), _cabi.VC1D_E_DTYPE), (dict(heads_k=3), _cabi.VC1D_E_SHAPE),
                     (dict(dim_v=300), _cabi.VC1D_E_TOO_LARGE), (dict(state=None), _cabi.VC1D_E_NULL),
                     (dict(state_strides=(0, 64, 8, 1)), _cabi.VC1D_E_STRIDE), (dict(out=FAKE), _cabi.VC1D_E_ALIAS),
                     (dict(out=5 * FAKE), _cabi.VC1D_E_ALIAS), (dict(batch=0), _cabi.VC1D_OK)):
        assert _cabi.lib.vc1d_linear_update(C.byref(args(**kw)), None) == code, kw
    assert _cabi.launch_count() == before


def page_args(tensors, pages=4, op=_cabi.PAGES_REORDER, **kw):
    table = (_cabi.PageTensor * max(len(tensors), 1))()
    for e, (base, size, stride) in zip(table, tensors):
        e.base, e.page_bytes, e.stride_bytes = base, size, stride
    a = _cabi.PagesArgs()
    a.struct_size = C.sizeof(_cabi.PagesArgs)
    a.op, a.pages, a.n_tensors, a.index_dtype = op, pages, len(tensors), _cabi.VC1D_I32
    a.tensors = table
    a.source = 9 * FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    a._table = table
    return a


@pytest.mark.parametrize("tensors,kw,code", [
    ([(FAKE, 64, 64)], dict(struct_size=4), _cabi.VC1D_E_STRUCT),
    ([(FAKE, 64, 64)], dict(op=4), _cabi.VC1D_E_SHAPE),
    ([(FAKE, 64, 64)], dict(pages=-1), _cabi.VC1D_E_SHAPE),
    ([(FAKE, 64, 64)], dict(pages=8193), _cabi.VC1D_E_TOO_LARGE),
    ([(FAKE, 64, 64)], dict(n_tensors=129), _cabi.VC1D_E_TOO_LARGE),
    ([(FAKE, 64, 64)], dict(index_dtype=_cabi.VC1D_F32), _cabi.VC1D_E_DTYPE),
    ([(FAKE, 64, 64)], dict(source=None), _cabi.VC1D_E_NULL),
    ([(FAKE, 64, 64)], dict(op=_cabi.PAGES_COPY, n=2), _cabi.VC1D_E_NULL),
    ([(FAKE, 64, 64)], dict(op=_cabi.PAGES_COMPACT), _cabi.VC1D_E_NULL),
    ([(None, 64, 64)], {}, _cabi.VC1D_E_NULL),
    ([(FAKE, 64, 32)], {}, _cabi.VC1D_E_STRIDE),
    ([(FAKE, 64, 64), (FAKE + 128, 64, 64)], {}, _cabi.VC1D_E_ALIAS),       # page 2 of the first
    ([(FAKE, 64, 256), (FAKE + 32, 64, 256)], {}, _cabi.VC1D_E_ALIAS),      # interleaved, but overlapping
    ([(FAKE, 64, 256), (FAKE + 64, 64, 128)], {}, _cabi.VC1D_E_ALIAS),
    ([(FAKE, 64, 64)], dict(source=FAKE + 64), _cabi.VC1D_E_ALIAS),         # the index lies among the pages
    ([(FAKE, 64, 64)], dict(op=_cabi.PAGES_COPY, n=0), _cabi.VC1D_OK),
    ([(FAKE, 64, 64)], dict(pages=0), _cabi.VC1D_OK),
    ([], {}, _cabi.VC1D_OK),
])
def test_pages_reject_bad_tables_without_launching(tensors, kw, code):
    before = _cabi.launch_count()
    a = page_args(tensors, **kw)
    assert _cabi.lib.vc1d_pages(C.byref(a), None) == code
    assert _cabi.launch_count() == before


# ------------------------------------------------------------------------------------------------- the oracle


def test_oracle_recurrence_equals_the_sum_over_pairs_and_its_gradient_the_formulas():
    g = torch.Generator().manual_seed(0)
    T, Dk, Dv = 7, 3, 4
    q, k, v, do = (torch.randn(1, T, 1, d, generator=g, dtype=torch.float64) for d in (Dk, Dk, Dv, Dv))
    s0, ds = (torch.randn(1, 1, Dk, Dv, generator=g, dtype=torch.float64) for _ in range(2))
    ld = torch.tensor([-0.3])
    a, s = float(torch.exp(ld.double())), Dk ** -0.5
    lag = torch.arange(T)[:, None] - torch.arange(T)[None]
    L = torch.where(lag >= 0, a ** lag.clamp(min=0).double(), 0.0)
    n = torch.arange(1, T + 1).double()[:, None]
    Q, K, W, G = q[0, :, 0], k[0, :, 0], v[0, :, 0], do[0, :, 0]
    o, S = O.linear_attention(q, k, v, ld, initial=s0)
    assert torch.allclose(o[0, :, 0], s * ((Q @ K.T * L) @ W + a ** n * (Q @ s0[0, 0])))
    assert torch.allclose(S[0, 0], a ** T * s0[0, 0] + (K * a ** (T - n)).T @ W)
    dq, dk, dv, di = O.grads(q, k, v, ld, do, initial=s0, dfinal=ds)
    A, B = Q @ K.T * L, G @ W.T * L
    assert torch.allclose(dq[0, :, 0], s * (B @ K + a ** n * (G @ s0[0, 0].T)))
    assert torch.allclose(dk[0, :, 0], s * B.T @ Q + a ** (T - n) * (W @ ds[0, 0].T))
    assert torch.allclose(dv[0, :, 0], s * A.T @ G + a ** (T - n) * (K @ ds[0, 0]))
    assert torch.allclose(di[0, 0], a ** T * ds[0, 0] + s * (Q * a ** n).T @ G)


def test_oracle_packed_rows_and_plans():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 9, 2, 3, generator=g) for _ in range(3))
    ld = torch.tensor([-0.1, -0.7])
    whole, _ = O.linear_attention(q, k, v, ld, seq_idx=V.seq_idx_from_lengths([4, 1, 4]))
    parts = [O.linear_attention(*(x[:, a:b] for x in (q, k, v)), ld)[0] for a, b in ((0, 4), (4, 5), (5, 9))]
    assert torch.allclose(whole, torch.cat(parts, 1))
    assert O.compact_plan([False, True, False, True, True]) == ([3, 1, 4, 3, 4], [-1, 1, -1, 0, 2], 3)
    assert O.compact_plan([]) == ([], [], 0)
