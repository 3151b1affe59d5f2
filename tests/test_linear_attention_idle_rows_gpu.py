"""Rows without a valid token, and chunks without one, leave the state as it is, whatever it holds."""
import pytest
import torch

import viby_model_b200 as V
from linear_cases import DTYPES, decays, make
from test_linear_attention_gpu import dev

pytestmark = pytest.mark.gpu

FORMS = [("bf16", "tc", 64), ("bf16", "tc", 160), ("bf16", "mma", 64), ("bf16", "mma", 160), ("bf16", "mma", 256), ("f16", "mma", 64),
         ("f16", "mma", 160), ("f32", "simt", 64), ("bf16", "simt", 40)]


@pytest.mark.parametrize("dtype,kernel,D", FORMS)
@pytest.mark.parametrize("segments", [1, 3])
def test_states_of_rows_without_a_token(dtype, kernel, D, segments):
    """An idle slot of a pool may hold anything; another row of the same call does its work."""
    dt, n = DTYPES[dtype], 300
    q, k, v, do, s0, ds = make(4, n, 2, 2, 2, D, D, dt)
    g = decays(2)
    mask = torch.ones(4, n, dtype=torch.bool)
    mask[1:] = False
    for x in (q, k, v, do):
        x[1:] = float("nan")
    for x in (s0, ds):
        x[1, :, ::3] = float("inf")
        x[1, :, 1::3, ::2] = float("-inf")
        x[2] = float("nan")
        x[3] = torch.finfo(torch.float32).min
    o, s = V.linear_attention_fn(dev(q), dev(k), dev(v), dev(g), None, dev(s0), True, attention_mask=dev(mask), kernel=kernel, segments=segments)
    assert not o[1:].any() and torch.isfinite(o[0]).all() and torch.isfinite(s[0]).all()
    assert torch.equal(torch.nan_to_num(s[1:].cpu(), nan=12345.0), torch.nan_to_num(s0[1:], nan=12345.0))
    *grads, di = V.linear_attention_bwd(dev(q), dev(k), dev(v), dev(g), dev(do), None, dev(s0), dev(ds), attention_mask=dev(mask), kernel=kernel,
                                        segments=segments)
    assert not any(x[1:].any() for x in grads) and all(torch.isfinite(x[0]).all() for x in grads)
    assert torch.equal(torch.nan_to_num(di[1:].cpu(), nan=12345.0), torch.nan_to_num(ds[1:], nan=12345.0))
