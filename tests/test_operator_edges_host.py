"""Refusals at the edges of what the operators accept, through Python and the C ABI.  Nothing is launched; runs without a
GPU."""
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import viby_model_b200 as V
from conftest import ROOT
from test_linear_attention_host import qkv


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
