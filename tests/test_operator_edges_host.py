"""Refusals at the edges of what the operators accept, through Python and the C ABI.  Nothing is launched; runs without a
GPU."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import viby_model_b200 as V
from conftest import ROOT
from test_linear_attention_host import FAKE, POINTERS, linear_args, page_args, qkv
from viby_model_b200 import _cabi


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require grad and has a data pointer: its tangent would be dropped without a word."""
    q, k, v = qkv()
    g, state, dout = torch.zeros(2), torch.zeros(1, 2, 8, 8), torch.zeros(1, 4, 2, 8)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        t = [x[:, 0] for x in (q, k, v)]
        for call in (lambda: V.linear_attention_fn(dual(q), k, v, g), lambda: V.linear_attention_fn(q, dual(k), v, g),
                     lambda: V.linear_attention_fn(q, k, dual(v), g), lambda: V.linear_attention_fn(q, k, v, dual(g)),
                     lambda: V.linear_attention_fn(q, k, v, g, None, dual(state), True),
                     lambda: V.linear_attention_fn(q, k, v, g, out=dual(dout)),
                     lambda: V.linear_attention_bwd(q, k, v, g, dual(dout)),
                     lambda: V.linear_attention_bwd(q, k, v, g, dout, None, state, dual(state)),
                     lambda: V.linear_attention_update(dual(t[0]), t[1], t[2], state, g),
                     lambda: V.linear_attention_update(*t, dual(state), g),
                     lambda: V.PageTable([state, dual(state)]), lambda: V.reorder_pages([dual(state)], torch.tensor([0]))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA device"):  # inputs without tangents: as ever
            V.linear_attention_fn(q, k, v, g)


def test_forward_mode_derivatives_of_the_convolution_are_refused():
    x, w, b, state = torch.zeros(2, 8, 5), torch.zeros(8, 4), torch.zeros(8), torch.zeros(2, 8, 4)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: V.causal_conv1d_fn(dual(x), w, b), lambda: V.causal_conv1d_fn(x, dual(w), b),
                     lambda: V.causal_conv1d_fn(x, w, b, residual=dual(x)), lambda: V.causal_conv1d_bwd(x, w, b, dual(x)),
                     lambda: V.causal_conv1d_update(dual(x[:, :, 0]), state, w, b),
                     lambda: V.causal_conv1d_update(x[:, :, 0], dual(state), w, b),
                     lambda: V.causal_conv1d_update_bwd(x[:, :, 0], state, w, b, dual(x[:, :, 0])),
                     lambda: V.causal_conv1d_update_multi([x[:, :, 0]], [dual(state)], [w], [b])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_one_page_of_overlapping_tensors_without_a_stride():
    """Strides say nothing where there is one page.  In a process of its own: a division by such a stride ends it."""
    code = ("import ctypes as C, sys; sys.path[:0] = ['tests', '.']\n"
            "from test_linear_attention_host import FAKE, page_args\n"
            "from viby_model_b200 import _cabi\n"
            "for tensors in ([(FAKE, 16, 0), (FAKE, 16, 0)], [(FAKE, 16, 0), (FAKE + 8, 16, 0)], [(FAKE, 16, -4), (FAKE, 16, -4)]):\n"
            "    assert _cabi.lib.vc1d_pages(C.byref(page_args(tensors, pages=1)), None) == _cabi.VC1D_E_ALIAS\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, env=dict(os.environ))
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


F32_STATES = dict(initial_strides=(128, 64, 8, 1), final_strides=(128, 64, 8, 1))
SIDES = [dict(mask=4 * FAKE + 16, mask_dtype=_cabi.VC1D_U8, mask_strides=(4, 1)),
         dict(mask=4 * FAKE - 24, mask_dtype=_cabi.VC1D_I64, mask_strides=(4, 1)),
         dict(seq_idx=4 * FAKE + 8, seq_strides=(4, 1)), dict(log_decay=4 * FAKE + 4), dict(log_decay=4 * FAKE - 4)]


@pytest.mark.parametrize("side", SIDES)
def test_outputs_over_masks_sequence_numbers_and_decays_are_refused(side):
    """Some CTAs would read them while others already store."""
    before = _cabi.launch_count()
    a = linear_args(**{**POINTERS, **side})  # out lies at 4 * FAKE
    assert _cabi.lib.vc1d_linear(C.byref(a), None) == _cabi.VC1D_E_ALIAS
    if "seq_idx" not in side:  # states and packed rows are not combined
        a = linear_args(**{**POINTERS, **side, "out": 6 * FAKE, "final_state": 4 * FAKE, **F32_STATES})
        assert _cabi.lib.vc1d_linear(C.byref(a), None) == _cabi.VC1D_E_ALIAS
        a = linear_args(**{**POINTERS, "seqlen": 0, "log_decay": 4 * FAKE, "final_state": 4 * FAKE, **F32_STATES})
        assert _cabi.lib.vc1d_linear(C.byref(a), None) == _cabi.VC1D_E_ALIAS
    for grad in ("dq", "dk", "dv", "dinitial"):
        if grad == "dinitial" and "seq_idx" in side:
            continue
        b = _cabi.LinearBwdArgs()
        b.struct_size = C.sizeof(_cabi.LinearBwdArgs)
        b.f = linear_args(**{**POINTERS, **side, "out": None})
        b.dout, b.dq, b.dk, b.dv = 8 * FAKE, 9 * FAKE, 10 * FAKE, 11 * FAKE
        for name in ("dout", "dq", "dk", "dv"):
            getattr(b, name + "_strides")[:] = (64, 16, 8, 1)
        b.dinitial_strides[:] = (128, 64, 8, 1)
        setattr(b, grad, 4 * FAKE)
        assert _cabi.lib.vc1d_linear_bwd(C.byref(b), None) == _cabi.VC1D_E_ALIAS, grad
    assert _cabi.launch_count() == before


@pytest.mark.parametrize("written", ["out", "state"])
@pytest.mark.parametrize("side", [dict(mask=4 * FAKE + 1, mask_dtype=_cabi.VC1D_U8, mask_stride=1),
                                  dict(mask=4 * FAKE - 8, mask_dtype=_cabi.VC1D_F32, mask_stride=2), dict(log_decay=4 * FAKE + 4)])
def test_a_token_written_over_its_mask_or_decays_is_refused(side, written):
    a = _cabi.LinearUpdateArgs()
    a.struct_size = C.sizeof(_cabi.LinearUpdateArgs)
    a.dtype = _cabi.VC1D_F16
    a.batch, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = 2, 2, 1, 2, 8, 8
    a.q, a.k, a.v, a.out, a.state, a.log_decay = FAKE, 2 * FAKE, 3 * FAKE, 5 * FAKE, 6 * FAKE, 7 * FAKE
    a.q_strides[:], a.k_strides[:], a.v_strides[:], a.out_strides[:] = (16, 8, 1), (8, 8, 1), (16, 8, 1), (16, 8, 1)
    a.state_strides[:] = (128, 64, 8, 1)
    setattr(a, written, 4 * FAKE)
    for k, v in side.items():
        setattr(a, k, v)
    before = _cabi.launch_count()
    assert _cabi.lib.vc1d_linear_update(C.byref(a), None) == _cabi.VC1D_E_ALIAS
    assert _cabi.launch_count() == before


@pytest.mark.parametrize("new_index,count", [(2 * FAKE + 3, 4 * FAKE), (2 * FAKE - 12, 4 * FAKE), (3 * FAKE, 2 * FAKE), (3 * FAKE, 2 * FAKE - 1),
                                             (3 * FAKE, 3 * FAKE + 12)])
def test_compaction_whose_results_overlap_its_input_is_refused(new_index, count):
    """One CTA writes them while the others still read which pages are live."""
    before = _cabi.launch_count()
    a = page_args([(FAKE, 64, 64)], op=_cabi.PAGES_COMPACT, live=2 * FAKE, new_index=new_index, count=count)
    assert _cabi.lib.vc1d_pages(C.byref(a), None) == _cabi.VC1D_E_ALIAS
    a.n_tensors = 0
    assert _cabi.lib.vc1d_pages(C.byref(a), None) == _cabi.VC1D_E_ALIAS
    assert _cabi.launch_count() == before


OVERLAPPING = [(64, 16, 4, 1), (64, 16, 8, 2), (64, 8, 8, 1), (64, 15, 8, 1), (32, 16, 8, 1), (1, 2, 8, 1)]  # [2, 4, 2, 8]
APART = [(64, 16, 8, 1), (64, 8, 32, 1), (8, 16, 64, 1), (64, 1, 32, 4), (1000, 17, 8, 1), (64, -16, 8, 1)]


@pytest.mark.parametrize("strides,ok", [(s, False) for s in OVERLAPPING] + [(s, True) for s in APART])
def test_outputs_whose_elements_share_memory_are_refused(strides, ok):
    """Windows that overlap as well as stride 0.  Where the strides are fine, the next check (the workspace's address) refuses."""
    places = {sum(i * s for i, s in zip((b, t, h, d), strides)) for b in range(2) for t in range(4) for h in range(2) for d in range(8)}
    assert (len(places) == 2 * 4 * 2 * 8) == ok
    before = _cabi.launch_count()
    a = linear_args(**{**POINTERS, "batch": 2, "out_strides": strides, "workspace": 7 * FAKE + 4, "workspace_bytes": 1 << 20})
    a.out = 4 * FAKE
    want = _cabi.VC1D_E_STRIDE
    assert _cabi.lib.vc1d_linear(C.byref(a), None) == want
    a.mask, a.mask_dtype, a.mask_strides[:] = 4 * FAKE, _cabi.VC1D_U8, (4, 1)  # found only after the strides
    assert _cabi.lib.vc1d_linear(C.byref(a), None) == (_cabi.VC1D_E_ALIAS if ok else want)
    assert _cabi.launch_count() == before


@pytest.mark.parametrize("strides,ok", [((512, 64, 8, 1), True), ((64, 128, 8, 1), True), ((512, 64, 1, 8), True), ((64, 64, 8, 1), False),
                                        ((512, 64, 4, 1), False), ((512, 60, 8, 1), False), ((100, 64, 8, 1), False)])
def test_states_whose_requests_share_memory_are_refused(strides, ok):
    a = _cabi.LinearUpdateArgs()
    a.struct_size = C.sizeof(_cabi.LinearUpdateArgs)
    a.dtype = _cabi.VC1D_F32
    a.batch, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = 2, 2, 2, 2, 8, 8
    a.q, a.k, a.v, a.out, a.state, a.log_decay = FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 4 * FAKE, 7 * FAKE  # out and state overlap
    for name in ("q", "k", "v", "out"):
        getattr(a, name + "_strides")[:] = (16, 8, 1)
    a.state_strides[:] = strides
    before = _cabi.launch_count()
    assert _cabi.lib.vc1d_linear_update(C.byref(a), None) == (_cabi.VC1D_E_ALIAS if ok else _cabi.VC1D_E_STRIDE)
    assert _cabi.launch_count() == before


@pytest.mark.parametrize("shape", [((1 << 32) + 8, 1, 1), (1, (1 << 32) + 8, 1), (1, 1, (1 << 32) + 2), ((1 << 31), 1, 1)])
def test_axes_that_do_not_fit_the_call_are_refused(shape):
    """They would be cut to 32 bits: 2^32 + 8 rows became 8, and the other outputs stayed unwritten."""
    x = torch.zeros(1, 1, 1, 1).expand(*shape, 1)
    with pytest.raises(ValueError, match="too large"):
        V.linear_attention_fn(x, x, x, torch.zeros(1).expand(shape[2]))
    with pytest.raises(ValueError, match="too large"):
        V.linear_attention_bwd(x, x, x, torch.zeros(1).expand(shape[2]), x)
    t = x.squeeze(1) if shape[1] == 1 else x.squeeze(0)
    with pytest.raises(ValueError, match="too large"):
        V.linear_attention_update(t, t, t, t.unsqueeze(-1), torch.zeros(1).expand(t.shape[1]))


def test_lists_of_too_many_pages_are_refused():
    """At most 2^30 entries: the kernel's and the call's counters are 32 bits wide."""
    long = torch.zeros(1, dtype=torch.int32).expand((1 << 32) + 5)
    for call in (lambda: V.free_pages([], long), lambda: V.copy_pages([], long, long), lambda: V.reorder_pages([], long),
                 lambda: V.free_pages([], long[: (1 << 30) + 1])):
        with pytest.raises(ValueError, match="at most"):
            call()
    before = _cabi.launch_count()
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        for op in (_cabi.PAGES_COPY, _cabi.PAGES_FREE):
            a = page_args([(FAKE, 64, 64)], op=op, n=n, dst=16 * FAKE, source=1 << 40)
            assert _cabi.lib.vc1d_pages(C.byref(a), None) == _cabi.VC1D_E_TOO_LARGE
    assert _cabi.launch_count() == before
