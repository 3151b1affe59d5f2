"""Inputs and tolerances of the linear attention tests, in one place.

Every output is a sum of products; with M the sum of their magnitudes (the oracle run on absolute values):
  fp32 pipes: each of the n roundings on the way of a term costs at most 2^-24 relative to M.  A term passes at most
      dim (q.k or q.S) + 64 (inside its chunk) + 3 per chunk it is carried over + 16 (decay, scale, joins) of them.
  tensor cores: an accumulation may truncate, at most 2^-22 relative, every 8 or 16 terms; counted per term above, 2^-22.
      The I/O type's rounding, u = eps / 2, meets a term once before the second product (the product inside a chunk, or
      the state that queries read) and the output once; keys that enter the state are split so that 16 (two parts) or
      24 bits (three) of them remain: u^2 more.
  16-bit outputs: u of the output's own size on top.
"""
import torch

from oracle import linear_oracle as O

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def decays(H, kind="mixed"):
    if kind == "none":
        return torch.zeros(H)
    if kind == "one token":
        return torch.full((H,), float("-inf"))
    if kind == "fast":
        return -torch.linspace(0.5, 60.0, H)
    e = torch.linspace(3.0, 12.0, H, dtype=torch.float64) if H > 1 else torch.tensor([5.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float()


def make(B, T, H, Hk, Hv, Dk, Dv, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, T, n, d, generator=g).to(dtype) for n, d in ((H, Dk), (Hk, Dk), (Hv, Dv), (H, Dv)))
    s0, ds = (torch.randn(B, H, Dk, Dv, generator=g) * 2 for _ in range(2))
    return q, k, v, do, s0, ds


def roundings(dim, T):
    return dim + 64 + 3 * ((T + 63) // 64) + 16


def tolerance(ref, M, dtype, dim, T, tensor_cores, out_dtype=None):
    """Largest difference allowed, element by element."""
    out_dtype = dtype if out_dtype is None else out_dtype
    tol = roundings(dim, T) * (2.0 ** -22 if tensor_cores else 2.0 ** -24) * M
    if dtype != torch.float32 and out_dtype != torch.float32:
        tol = tol + unit(out_dtype) * ref.abs() * (1 + 2.0 ** -6)
        if tensor_cores:
            u = unit(dtype)
            tol = tol + (u + 4 * u * u) * M * (1 + u)
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -24  # half a step of its subnormals
    return tol + 1e-30


def check(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} vs {tuple(ref.shape)}"
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    err = (got - ref).abs()
    bad = err > tol
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {got.numel()} off; worst {float((err / tol).max()):.2f} of the tolerance, "
                                 f"error {float(err.max()):.3e}, at {tuple(int(i) for i in bad.nonzero()[0])}")


def magnitudes(q, k, v, log_decay, s0=None, **kw):
    z = lambda x: None if x is None else torch.nan_to_num(x.float(), 0.0, 0.0, 0.0).abs()  # noqa: E731
    return O.linear_attention(z(q), z(k), z(v), log_decay, initial=z(s0), **kw)


def grad_magnitudes(q, k, v, log_decay, do, s0=None, dfinal=None, **kw):
    z = lambda x: None if x is None else torch.nan_to_num(x.float(), 0.0, 0.0, 0.0).abs()  # noqa: E731
    return O.grads(z(q), z(k), z(v), log_decay, z(do), initial=z(s0), dfinal=z(dfinal), **kw)
