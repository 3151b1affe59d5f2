"""Linear attention with a fixed decay for each head: ``linear_attention_fn`` (prompts and training),
``linear_attention_bwd`` and ``linear_attention_update`` (one token), the long-range companion of the Canon
convolution with the same pair of forms (a prompt leaves a state, single tokens roll it on).

With ``a = exp(log_decay[h])``:  ``S_t = a S_{t-1} + k_t v_t^T``,  ``o_t = scale * q_t^T S_t``.

Host code only checks and marshals into the C ABI (include/vc1d.h); there is no PyTorch or CPU implementation.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _cabi
from .ops import _IO_DTYPES, _MASK_DTYPES, _TLS, _no_tangents, _require_cuda, _stream_handle


def _launch(device: torch.device, call, *args):
    """Runs a library call with ``device`` current."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return call(*args)
    return call(*args)


def _check_heads(q, k, v, lead: int, what: str):
    """Shapes of q, k, v whose last two axes are (heads, dim) after ``lead`` axes.  Returns the sizes."""
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != lead + 2:
            raise ValueError(f"Expected {lead + 2}D {name} tensor ({what}, heads, dim), got {x.dim()}D")
        if x.dtype not in _IO_DTYPES:
            raise ValueError(f"unsupported dtype {x.dtype}: expected float32, bfloat16 or float16")
        if x.dtype != q.dtype:
            raise ValueError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
        if x.shape[:lead] != q.shape[:lead]:
            raise ValueError(f"{name} shape {tuple(x.shape)} does not match q shape {tuple(q.shape)} in {what}")
    H, Dk = q.shape[lead:]
    Hk, Hv, Dv = k.shape[lead], v.shape[lead], v.shape[lead + 1]
    if max(H, *q.shape[:lead]) > 0x7fffffff:  # more than the fields of the C structs hold
        raise ValueError(f"q shape {tuple(q.shape)} is too large: at most 2^31 - 1 along an axis")
    if k.shape[lead + 1] != Dk:
        raise ValueError(f"k dim {k.shape[lead + 1]} does not match q dim {Dk}")
    if H < 1 or Hk < 1 or Hv < 1 or H % Hk != 0 or H % Hv != 0:
        raise ValueError(f"{H} heads cannot share {Hk} key and {Hv} value heads: both must divide the number of heads")
    for name, d in (("q and k", Dk), ("v", Dv)):
        if not 1 <= d <= _cabi.LINEAR_MAX_DIM:
            raise ValueError(f"head dim of {name} must be 1..{_cabi.LINEAR_MAX_DIM}, got {d}")
    return H, Hk, Hv, Dk, Dv


def _check_decay(log_decay: torch.Tensor, heads: int, device) -> torch.Tensor:
    if log_decay.dim() != 1 or log_decay.shape[0] != heads:
        raise ValueError(f"log_decay shape {tuple(log_decay.shape)} does not match the {heads} heads")
    if log_decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be float32, got {log_decay.dtype}")
    _require_cuda(log_decay, "log_decay")
    _same_device(log_decay, device, "log_decay")
    return log_decay.contiguous()


def _check_scale(scale) -> None:
    """A tensor's value is on the device, may change between two calls, and would want a gradient."""
    if isinstance(scale, torch.Tensor):
        raise TypeError("scale must be a number, got a tensor")


def _changed(*tensors) -> None:
    """Tells autograd that the tensors were written in place: a graph that saved one of them then refuses to run."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


def _signature(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _aligned(q, k, v) -> bool:
    return not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15


# Prepared argument structs by call signature (shapes, strides, dtypes, devices, options), per host thread: a repeated call
# only refreshes the pointers.  Nothing of the tensors' contents or addresses is kept.
def _prepared(kind: str) -> dict:
    cache = getattr(_TLS, kind, None)
    if cache is None:
        cache = {}
        setattr(_TLS, kind, cache)
    return cache


_MAX_FORMS = 256  # of a kind and thread


def _remember(forms: dict, key, value) -> None:
    """Keeps a prepared struct; the oldest makes room, because prompt lengths that do not come back would else fill the place
    for good."""
    if len(forms) >= _MAX_FORMS:
        del forms[next(iter(forms))]
    forms[key] = value


def _same_device(t: torch.Tensor, device, what: str) -> None:
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, q on {device}")


def _check_state(s: torch.Tensor, shape, device, what: str) -> None:
    if tuple(s.shape) != tuple(shape):
        raise ValueError(f"{what} shape {tuple(s.shape)} does not match (batch, heads, dim_k, dim_v) = {tuple(shape)}")
    if s.dtype != torch.float32:
        raise ValueError(f"{what} must be float32, got {s.dtype}")
    _require_cuda(s, what)
    _same_device(s, device, what)


def _fill(q, k, v, log_decay, seq_idx, initial_states, attention_mask, scale, kernel, segments) -> Tuple[_cabi.LinearArgs, tuple]:
    """Validates what forward and backward share and fills the struct.  Returns it with the tensors it names."""
    H, Hk, Hv, Dk, Dv = _check_heads(q, k, v, 2, "batch, seqlen")
    B, T = q.shape[:2]
    for name, x in (("q", q), ("k", k), ("v", v)):
        _require_cuda(x, name)
        _same_device(x, q.device, name)
    log_decay = _check_decay(log_decay, H, q.device)
    a = _cabi.LinearArgs()
    a.struct_size = C.sizeof(_cabi.LinearArgs)
    a.dtype = _IO_DTYPES[q.dtype]
    a.batch, a.seqlen, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = B, T, H, Hk, Hv, Dk, Dv
    if kernel not in _cabi.LINEAR_KERNEL_BY_NAME:
        raise ValueError(f"unknown linear attention kernel {kernel!r}")
    a.kernel = _cabi.LINEAR_KERNEL_BY_NAME[kernel]
    a.segments = int(segments)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = q.stride(), k.stride(), v.stride()
    a.log_decay = log_decay.data_ptr()
    a.scale = float(Dk ** -0.5 if scale is None else scale)
    if attention_mask is not None:
        m = attention_mask
        _require_cuda(m, "Attention mask")
        _same_device(m, q.device, "Attention mask")
        if m.dim() != 2:
            raise ValueError(f"Expected 2D attention mask, got {m.dim()}D")
        if tuple(m.shape) != (B, T):
            raise ValueError(f"Attention mask shape {tuple(m.shape)} does not match input shape ({B}, {T})")
        if m.dtype not in _MASK_DTYPES:
            raise ValueError(f"unsupported attention mask dtype {m.dtype}")
        a.mask = m.data_ptr()
        a.mask_dtype = _MASK_DTYPES[m.dtype]
        a.mask_strides[:] = m.stride()
    if seq_idx is not None:
        _require_cuda(seq_idx, "seq_idx")
        _same_device(seq_idx, q.device, "seq_idx")
        if tuple(seq_idx.shape) != (B, T):
            raise ValueError(f"seq_idx shape {tuple(seq_idx.shape)} does not match input shape ({B}, {T})")
        if seq_idx.dtype != torch.int32:
            seq_idx = seq_idx.to(torch.int32)
        a.seq_idx = seq_idx.data_ptr()
        a.seq_strides[:] = seq_idx.stride()
    if initial_states is not None:
        _check_state(initial_states, (B, H, Dk, Dv), q.device, "initial_states")
        a.initial_state = initial_states.data_ptr()
        a.initial_strides[:] = initial_states.stride()
    return a, (log_decay, seq_idx)


def _workspace(a, query, device) -> Optional[torch.Tensor]:
    n = _launch(device, query, C.byref(a))
    if n < 0:
        _cabi.check(int(n), "linear_attention")
    if n == 0:
        a.workspace, a.workspace_bytes = None, 0
        return None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    return ws


def _forward(q, k, v, log_decay, seq_idx, initial_states, return_final_states, final_states_out, attention_mask, scale, out,
             kernel, segments):
    want_state = bool(return_final_states) or final_states_out is not None
    plain = out is None and final_states_out is None and q.is_cuda and (seq_idx is None or seq_idx.dtype == torch.int32) \
        and log_decay.is_contiguous()
    key = None
    if plain:
        key = (_signature(q), _signature(k), _signature(v), _signature(log_decay), _signature(seq_idx),
               _signature(initial_states), _signature(attention_mask), want_state, scale, kernel, segments)
        known = _prepared("linear_args").get(key)
        if known is not None:
            a, ws_bytes = known
            return _run_prepared(a, ws_bytes, q, k, v, log_decay, seq_idx, initial_states, attention_mask, want_state)
    if seq_idx is not None and (attention_mask is not None or initial_states is not None or want_state):
        raise ValueError("seq_idx cannot be combined with attention_mask, initial_states or final states")
    a, keep = _fill(q, k, v, log_decay, seq_idx, initial_states, attention_mask, scale, kernel, segments)
    shape = (a.batch, a.seqlen, a.heads, a.dim_v)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be {shape} of q's dtype on q's device")
    a.out = out.data_ptr()
    a.out_strides[:] = out.stride()
    state = None
    if want_state:
        s_shape = (a.batch, a.heads, a.dim_k, a.dim_v)
        if final_states_out is not None:
            _check_state(final_states_out, s_shape, q.device, "final_states_out")
            state = final_states_out
        else:
            state = torch.empty(s_shape, dtype=torch.float32, device=q.device)
        a.final_state = state.data_ptr()
        a.final_strides[:] = state.stride()
    ws = _workspace(a, _cabi.lib.vc1d_linear_workspace, q.device)
    st = _launch(q.device, _cabi.lib.vc1d_linear, C.byref(a), _stream_handle(q.device))
    _cabi.check(st, "linear_attention_fn")
    _changed(out, state)
    # workspace sizes and kernels depend on the alignment of the data too: only aligned calls are remembered, for aligned calls
    if key is not None and _aligned(q, k, v):
        _remember(_prepared("linear_args"), key, (a, 0 if ws is None else ws.numel()))
    del keep, ws
    return out, state


def _run_prepared(a, ws_bytes, q, k, v, log_decay, seq_idx, initial_states, attention_mask, want_state):
    """The launch of _forward for a signature that has been checked before."""
    device = q.device
    a.q, a.k, a.v, a.log_decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr()
    if seq_idx is not None:
        a.seq_idx = seq_idx.data_ptr()
    if initial_states is not None:
        a.initial_state = initial_states.data_ptr()
    if attention_mask is not None:
        a.mask = attention_mask.data_ptr()
    out = torch.empty((a.batch, a.seqlen, a.heads, a.dim_v), dtype=q.dtype, device=device)
    a.out = out.data_ptr()
    state = None
    if want_state:
        state = torch.empty((a.batch, a.heads, a.dim_k, a.dim_v), dtype=torch.float32, device=device)
        a.final_state = state.data_ptr()
    if not _aligned(q, k, v):  # another kernel, maybe with a workspace of its own size
        ws = _workspace(a, _cabi.lib.vc1d_linear_workspace, device)
    else:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        a.workspace, a.workspace_bytes = (ws.data_ptr(), ws_bytes) if ws_bytes else (None, 0)
    st = _launch(device, _cabi.lib.vc1d_linear, C.byref(a), _stream_handle(device))
    if st != 0:
        _cabi.check(st, "linear_attention_fn")
    return out, state


def linear_attention_fn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    seq_idx: Optional[torch.Tensor] = None,
    initial_states: Optional[torch.Tensor] = None,
    return_final_states: bool = False,
    final_states_out: Optional[torch.Tensor] = None,
    *,
    attention_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    kernel: Optional[str] = None,
    segments: int = 0,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal linear attention with a decay for each head (prompts, training).

    ``S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T``;  ``o_t = scale * q_t^T S_t``;  returns ``o[batch, seqlen, heads, dim_v]``
    (and the state after the last token, fp32 ``[batch, heads, dim_k, dim_v]``).

      q ``[batch, seqlen, heads, dim_k]``, k ``[batch, seqlen, heads_k, dim_k]``, v ``[batch, seqlen, heads_v, dim_v]``: one
        dtype (float32, bfloat16, float16), any strides (parts of one fused projection too).  ``heads_k`` and ``heads_v``
        divide ``heads``; head h reads key head ``h // (heads // heads_k)``, likewise for v.  Dims 1..256.
      log_decay ``[heads]`` float32, fixed (no gradient), usually negative; 0 never forgets, ``-inf`` keeps one token.
      seq_idx ``[batch, seqlen]`` (int32): packed rows; the state starts at zero wherever the value changes, and an infinity
        or NaN of one sequence does not reach another.  Not combined with a mask or states, as in ``causal_conv1d_fn``.
      initial_states fp32 ``[batch, heads, dim_k, dim_v]``: continues a prompt.  ``return_final_states`` /
        ``final_states_out`` give the state that the next part or ``linear_attention_update`` continues from (it must not
        overlap ``initial_states``).
      attention_mask ``[batch, seqlen]`` (bool / int / float; nonzero = valid): a masked token has no effect whatever it holds,
        leaves the state as it is (no decay either) and its output is 0.
      scale: a number, ``dim_k ** -0.5`` by default.
      kernel: None, "simt", "mma" or "tc".  16-bit inputs go to the tensor cores by default, where the products inside a chunk
        and the state that queries read are rounded to 16 bits before the second product; "simt" keeps both in fp32, at the
        fp32 pipes' speed.  segments: parts of the time axis (0 = automatic).

    Differentiable in q, k, v and initial_states, through o and the final state (``linear_attention_bwd``); in reverse mode
    only, inputs with a tangent are refused.
    """
    _check_scale(scale)
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise ValueError("log_decay is fixed: it has no gradient (pass log_decay.detach())")
    if torch.compiler.is_compiling():
        if out is not None or final_states_out is not None:
            raise ValueError("out= / final_states_out= cannot be used under torch.compile")
        o, state = torch.ops.vc1d.linear_attention(q, k, v, log_decay, seq_idx, initial_states, attention_mask,
                                                   float(q.shape[-1] ** -0.5 if scale is None else scale),
                                                   bool(return_final_states), kernel or "auto", int(segments))
        return (o, state) if return_final_states else o
    _no_tangents("linear_attention_fn", q, k, v, log_decay, initial_states, out, final_states_out)
    needs_grad = torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or v.requires_grad
        or (initial_states is not None and initial_states.requires_grad)
    )
    want_state = bool(return_final_states) or final_states_out is not None
    if needs_grad:
        if out is not None or final_states_out is not None:
            raise ValueError("out= / final_states_out= cannot be used when a gradient is required")
        o, state = _LinearAttentionFunction.apply(q, k, v, log_decay, seq_idx, initial_states, want_state, attention_mask,
                                                  scale, kernel, segments)
    else:
        o, state = _forward(q, k, v, log_decay, seq_idx, initial_states, return_final_states, final_states_out,
                            attention_mask, scale, out, kernel, segments)
    return (o, state) if want_state else o


def linear_attention_bwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    dout: torch.Tensor,
    seq_idx: Optional[torch.Tensor] = None,
    initial_states: Optional[torch.Tensor] = None,
    dfinal_states: Optional[torch.Tensor] = None,
    *,
    attention_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    need_dinitial: Optional[bool] = None,
    kernel: Optional[str] = None,
    segments: int = 0,
):
    """Gradients of ``linear_attention_fn``: ``(dq, dk, dv, dinitial)`` for the gradient ``dout`` of its output and,
    where the final state was used, ``dfinal_states`` of that.  ``dinitial`` (fp32) is None unless ``need_dinitial``
    (default: when ``initial_states`` is given).  Gradients of shared key / value heads are summed over their heads."""
    _check_scale(scale)
    _no_tangents("linear_attention_bwd", q, k, v, log_decay, dout, initial_states, dfinal_states)
    if need_dinitial is None:
        need_dinitial = initial_states is not None
    if seq_idx is not None and (attention_mask is not None or initial_states is not None or dfinal_states is not None or need_dinitial):
        raise ValueError("seq_idx cannot be combined with attention_mask, initial_states or final states")
    f, keep = _fill(q, k, v, log_decay, seq_idx, initial_states, attention_mask, scale, kernel, 0)
    B, T, H, Dk, Dv = f.batch, f.seqlen, f.heads, f.dim_k, f.dim_v
    if tuple(dout.shape) != (B, T, H, Dv) or dout.dtype != q.dtype:
        raise ValueError(f"dout must be {(B, T, H, Dv)} of dtype {q.dtype}, got {tuple(dout.shape)} of {dout.dtype}")
    _require_cuda(dout, "dout")
    _same_device(dout, q.device, "dout")
    a = _cabi.LinearBwdArgs()
    a.struct_size = C.sizeof(_cabi.LinearBwdArgs)
    a.segments = int(segments)
    a.f = f
    a.dout = dout.data_ptr()
    a.dout_strides[:] = dout.stride()
    grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)]
    a.dq, a.dk, a.dv = (x.data_ptr() for x in grads)
    a.dq_strides[:], a.dk_strides[:], a.dv_strides[:] = (x.stride() for x in grads)
    if dfinal_states is not None:
        _check_state(dfinal_states, (B, H, Dk, Dv), q.device, "dfinal_states")
        a.dfinal = dfinal_states.data_ptr()
        a.dfinal_strides[:] = dfinal_states.stride()
    dinitial = None
    if need_dinitial:
        dinitial = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=q.device)
        a.dinitial = dinitial.data_ptr()
        a.dinitial_strides[:] = dinitial.stride()
    ws = _workspace(a, _cabi.lib.vc1d_linear_bwd_workspace, q.device)
    st = _launch(q.device, _cabi.lib.vc1d_linear_bwd, C.byref(a), _stream_handle(q.device))
    _cabi.check(st, "linear_attention_bwd")
    del keep, ws
    return (*grads, dinitial)


class _LinearAttentionFunction(torch.autograd.Function):
    """Autograd glue of linear_attention_fn."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, seq_idx, initial_states, want_state, attention_mask, scale, kernel, segments):
        o, state = _forward(q, k, v, log_decay, seq_idx, initial_states, want_state, None, attention_mask, scale, None,
                            kernel, segments)
        ctx.save_for_backward(q, k, v, log_decay, seq_idx, initial_states, attention_mask)
        ctx.scale, ctx.kernel, ctx.segments = scale, kernel, segments
        ctx.set_materialize_grads(False)
        if state is None:
            state = o.new_empty(0)
            ctx.mark_non_differentiable(state)
        return o, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dstate):
        q, k, v, log_decay, seq_idx, init, mask = ctx.saved_tensors
        if dout is None and dstate is None:
            return (None,) * 11
        if dout is None:
            dout = q.new_zeros(1).expand(*q.shape[:3], v.shape[3])
        if ctx.kernel not in (None, "auto"):  # the kernel that the caller named may not take every layout
            dout = dout.contiguous()
        if dstate is not None and dstate.numel() == 0 and v.shape[0] > 0:
            dstate = None  # no final state was returned
        grads = linear_attention_bwd(q, k, v, log_decay, dout, seq_idx, init, dstate, attention_mask=mask, scale=ctx.scale,
                                     need_dinitial=init is not None and ctx.needs_input_grad[5], kernel=ctx.kernel,
                                     segments=ctx.segments)
        dq, dk, dv = (g if need else None for g, need in zip(grads[:3], ctx.needs_input_grad[:3]))
        return dq, dk, dv, None, None, grads[3], None, None, None, None, None


def linear_attention_update(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    state: torch.Tensor,
    log_decay: torch.Tensor,
    *,
    attention_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One token of linear attention (decode): ``state <- exp(log_decay) state + k v^T`` **in place**, returns
    ``o = scale * q^T state`` as ``[batch, heads, dim_v]``.

    q ``[batch, heads, dim_k]``, k ``[batch, heads_k, dim_k]``, v ``[batch, heads_v, dim_v]``; state fp32
    ``[batch, heads, dim_k, dim_v]`` as ``linear_attention_fn`` returns it (a slice ``pool[:n]`` of a larger pool too).
    ``attention_mask[batch]``: rows whose value is 0 (idle slots of a captured decode step) keep their state untouched
    and get zeros.  No gradient: for one differentiable token call ``linear_attention_fn`` with ``seqlen`` 1."""
    _check_scale(scale)
    if torch.compiler.is_compiling():
        if out is not None:
            raise ValueError("out= cannot be used under torch.compile")
        return torch.ops.vc1d.linear_attention_update(q, k, v, state, log_decay, attention_mask,
                                                      float(q.shape[-1] ** -0.5 if scale is None else scale))
    return _update(q, k, v, state, log_decay, attention_mask, scale, out)


def _update(q, k, v, state, log_decay, attention_mask, scale, out):
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad
                                    or log_decay.requires_grad):
        raise ValueError("linear_attention_update has no gradient: use linear_attention_fn with seqlen 1 and initial_states")
    _no_tangents("linear_attention_update", q, k, v, state, log_decay, out)
    key = None
    if out is None and q.is_cuda and log_decay.is_contiguous():
        key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype,
               v.get_device(), state.shape, state.stride(), state.dtype, state.get_device(), log_decay.shape, log_decay.dtype,
               log_decay.get_device(), _signature(attention_mask), scale)
        a = _prepared("linear_update_args").get(key)
        if a is not None:
            out = torch.empty((a.batch, a.heads, a.dim_v), dtype=q.dtype, device=q.device)
            a.q, a.k, a.v, a.out, a.state = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), state.data_ptr()
            a.log_decay = log_decay.data_ptr()
            if attention_mask is not None:
                a.mask = attention_mask.data_ptr()
            st = _launch(q.device, _cabi.lib.vc1d_linear_update, C.byref(a), _stream_handle(q.device))
            if st != 0:
                _cabi.check(st, "linear_attention_update")
            _changed(state)
            return out
    H, Hk, Hv, Dk, Dv = _check_heads(q, k, v, 1, "batch")
    B = q.shape[0]
    for name, x in (("q", q), ("k", k), ("v", v)):
        _require_cuda(x, name)
        _same_device(x, q.device, name)
    log_decay = _check_decay(log_decay, H, q.device)
    _check_state(state, (B, H, Dk, Dv), q.device, "state")
    if out is None:
        out = torch.empty((B, H, Dv), dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (B, H, Dv) or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be {(B, H, Dv)} of q's dtype on q's device")
    a = _cabi.LinearUpdateArgs()
    a.struct_size = C.sizeof(_cabi.LinearUpdateArgs)
    a.dtype = _IO_DTYPES[q.dtype]
    a.batch, a.heads, a.heads_k, a.heads_v, a.dim_k, a.dim_v = B, H, Hk, Hv, Dk, Dv
    a.q, a.k, a.v, a.out, a.state = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), state.data_ptr()
    a.log_decay = log_decay.data_ptr()
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = q.stride(), k.stride(), v.stride()
    a.out_strides[:], a.state_strides[:] = out.stride(), state.stride()
    a.scale = float(Dk ** -0.5 if scale is None else scale)
    if attention_mask is not None:
        m = attention_mask
        _require_cuda(m, "Attention mask")
        _same_device(m, q.device, "Attention mask")
        if tuple(m.shape) != (B,):
            raise ValueError(f"Attention mask shape {tuple(m.shape)} does not match the batch ({B},)")
        if m.dtype not in _MASK_DTYPES:
            raise ValueError(f"unsupported attention mask dtype {m.dtype}")
        a.mask, a.mask_dtype, a.mask_stride = m.data_ptr(), _MASK_DTYPES[m.dtype], m.stride(0)
    st = _launch(q.device, _cabi.lib.vc1d_linear_update, C.byref(a), _stream_handle(q.device))
    _cabi.check(st, "linear_attention_update")
    _changed(state, out)
    if key is not None:
        _remember(_prepared("linear_update_args"), key, a)
    return out
