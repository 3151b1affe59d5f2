"""Cases for timing and checking the operators on the recurrent state: linear attention with a decay for each
head (prompts, training, single tokens) and the pages of a state cache (copy / fork, reorder, compact, free).

``own`` False computes every operator in a plain form out of elementary torch operations; ``own`` True makes the
calls a user of ``viby_model_b200`` makes.  Shapes: Viby's own heads (4 query heads, 1 key/value head, head_dim 160;
Canon channels 640 / 960 / 640 / 3456, 4 columns; batch 64 x 1024 tokens) and generic ones.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CANON = (640, 960, 640, 3456)  # channels of the four Canon positions


def listed():
    return [
        # one request being decoded by a model of Viby's heads: the call is all latency
        dict(name="update one request", op="update", B=1, H=4, Hk=1, Hv=1, Dk=160, Dv=160, dtype="bf16", idle=0),
        # a full decode batch; some slots of the batch are idle
        dict(name="update full batch", op="update", B=256, H=16, Hk=16, Hv=16, Dk=128, Dv=128, dtype="bf16", idle=9),
        # the prompt of one request: few heads, so the work has to be split along time
        dict(name="prompt of one request", op="fn", B=1, T=1000, H=4, Hk=1, Hv=1, Dk=160, Dv=160, dtype="bf16",
             rows="full", init=False, final=True),
        # a batch of prompts, right padded, lengths uniform in [T/8, T]
        dict(name="padded prompts", op="fn", B=32, T=1024, H=4, Hk=1, Hv=1, Dk=160, Dv=160, dtype="bf16",
             rows="right", init=False, final=True),
        # prompts of very different lengths packed end to end in one row
        dict(name="packed prompts", op="fn", B=1, T=24567, H=8, Hk=8, Hv=8, Dk=64, Dv=64, dtype="f16",
             rows="packed", init=False, final=False),
        # the next part of a long document, continued from the state of what came before
        dict(name="long prompt, continued", op="fn", B=1, T=65536, H=16, Hk=16, Hv=16, Dk=128, Dv=128, dtype="bf16",
             rows="full", init=True, final=True),
        # one layer's training step at Viby's training batch
        dict(name="training step", op="train", B=64, T=1024, H=4, Hk=1, Hv=1, Dk=160, Dv=160, dtype="bf16",
             rows="full", init=False, final=False),
        # a chunk of a longer sequence in fp32, gradients through both states, left padding, odd sizes
        dict(name="training chunk f32", op="train", B=3, T=777, H=6, Hk=2, Hv=3, Dk=72, Dv=88, dtype="f32",
             rows="left", init=True, final=True),
        # beam search over the Canon states of 12 layers, every row is replaced by its parent's
        dict(name="reorder beams", op="reorder", pages=64, layers=12, kind="canon"),
        # a request is forked into three samples; linear attention states of 18 layers
        dict(name="fork a request", op="copy", pages=8, layers=18, kind="linear", H=4, Dk=160, Dv=160, moved=3),
        # half of the requests have ended: the others move together at the front of the pool
        dict(name="compact the pool", op="compact", pages=512, layers=6, kind="linear", H=4, Dk=160, Dv=160, moved=256),
        # new requests start on cleared pages
        dict(name="clear pages", op="free", pages=96, layers=18, kind="linear", H=4, Dk=64, Dv=64, moved=17),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("update", "fn", "fn", "train", "reorder", "copy", "compact", "free"))
    if op in ("update", "fn", "train"):
        H = rng.choice((1, 2, 3, 4, 6, 8, 12, 16))
        Hk = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16) if H % h == 0])
        Hv = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16) if H % h == 0])
        Dk = rng.choice((16, 33, 64, 72, 96, 128, 160, 256))
        Dv = rng.choice((Dk, Dk, 24, 64, 100, 128, 192, 256))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        case = dict(op=op, H=H, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=dtype)
        per_token = H * max(Dk, 64) * max(Dv, 64)
        if op == "update":
            case["B"] = _log_int(rng, 1, max(1, min(512, (60 << 20) // per_token)))
            case["idle"] = rng.randrange(0, case["B"]) if case["B"] > 2 and rng.random() < 0.3 else 0
            return case
        # tokens in all: at most what costs as much as the long prompt (fn) or the training step (train)
        most = (1 << 34 if op == "fn" else 1 << 32) // per_token // (4 if dtype == "f32" else 1)
        most = min(most, 1 << 16)
        tokens = _log_int(rng, 1, most)
        rows = rng.choice(("full", "full", "right", "left", "packed"))
        B = 1 if rows == "packed" else min(tokens, rng.choice((1, 1, 2, 3, 8, 32)))
        case.update(B=B, T=max(1, tokens // B), rows=rows, init=rows != "packed" and rng.random() < 0.4,
                    final=rows != "packed" and rng.random() < 0.6)
        return case
    kind = rng.choice(("canon", "linear"))
    pages = _log_int(rng, 2, 600)
    case = dict(op=op, pages=pages, kind=kind)
    if kind == "canon":
        case["layers"] = rng.randint(1, 12)
    else:
        case.update(H=rng.choice((1, 4, 5, 8)), Dk=rng.choice((33, 64, 128, 160)), Dv=rng.choice((17, 64, 128, 160)))
        per_page = 4 * case["H"] * case["Dk"] * case["Dv"]
        case["layers"] = max(1, min(rng.randint(1, 18), (1200 << 20) // (per_page * pages)))
        if per_page * pages > 1200 << 20:
            case["pages"] = (1200 << 20) // per_page
    if op != "reorder":
        case["moved"] = rng.randint(1, max(1, case["pages"] // 2))
    return case


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _log_decay(H):
    """Decays from 1 - 2^-5 (about 32 tokens back) to 1 - 2^-12 (about 4096), as retention models fix them."""
    e = torch.linspace(5.0, 12.0, H, dtype=torch.float64) if H > 1 else torch.tensor([7.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float().cuda()


def _prepare_attention(case, g):
    B, T, H, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "T", "H", "Hk", "Hv", "Dk", "Dv"))
    dt = _DT[case["dtype"]]
    st = dict(case=case, log_decay=_log_decay(H), mask=None, seq_idx=None, init=None)
    if Dk == Dv:  # q, k, v are parts of one projection's output
        qkv = torch.randn(B, T, (H + Hk + Hv) * Dk, device="cuda", generator=g).to(dt)
        q, k, v = qkv.split([H * Dk, Hk * Dk, Hv * Dv], dim=-1)
    else:
        q, k, v = (torch.randn(B, T, n, device="cuda", generator=g).to(dt) for n in (H * Dk, Hk * Dk, Hv * Dv))
    st.update(q=q.unflatten(-1, (H, Dk)), k=k.unflatten(-1, (Hk, Dk)), v=v.unflatten(-1, (Hv, Dv)))
    if case["rows"] in ("right", "left"):
        lens = torch.randint(max(1, T // 8), T + 1, (B, 1), device="cuda", generator=g)
        t = torch.arange(T, device="cuda")[None]
        st["mask"] = t < lens if case["rows"] == "right" else t >= T - lens
    if case["rows"] == "packed":  # lengths log-uniform in [16, T / 2]
        u = torch.rand(max(1, T // 16), device="cuda", generator=g)
        ends = torch.exp(math.log(16.0) + u * math.log(max(1.0, T / 32))).long().cumsum(0)
        st["seq_idx"] = torch.searchsorted(ends, torch.arange(T, device="cuda"), right=True).int()[None]
    if case["init"]:
        st["init"] = torch.randn(B, H, Dk, Dv, device="cuda", generator=g) * 4
    if case["op"] == "train":
        st["dout"] = torch.randn(B, T, H, Dv, device="cuda", generator=g).to(dt)
        st["dfinal"] = torch.randn(B, H, Dk, Dv, device="cuda", generator=g) if case["final"] else None
    return st


def _prepare_update(case, g):
    B, H, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "H", "Hk", "Hv", "Dk", "Dv"))
    dt = _DT[case["dtype"]]
    q, k, v = (torch.randn(B, n, d, device="cuda", generator=g).to(dt) for n, d in ((H, Dk), (Hk, Dk), (Hv, Dv)))
    mask = None
    if case["idle"]:
        mask = torch.ones(B, dtype=torch.bool, device="cuda")
        mask[torch.randperm(B, device="cuda", generator=g)[: case["idle"]]] = False
    state = torch.randn(B, H, Dk, Dv, device="cuda", generator=g) * 4
    return dict(case=case, q=q, k=k, v=v, state=state, mask=mask, log_decay=_log_decay(H))


def _prepare_pages(case, g):
    N, L = case["pages"], case["layers"]
    if case["kind"] == "canon":
        pools = [torch.randn(N, d, 4, device="cuda", generator=g).bfloat16() for d in _CANON for _ in range(L)]
    else:
        pools = [torch.randn(N, case["H"], case["Dk"], case["Dv"], device="cuda", generator=g) for _ in range(L)]
    st = dict(case=case, pools=pools)
    order = torch.randperm(N, device="cuda", generator=g).int()
    if case["op"] == "reorder":  # what beam search gives: some rows twice, some not at all
        st["source"] = torch.randint(0, N, (N,), device="cuda", generator=g, dtype=torch.int32)
    elif case["op"] == "copy":  # the first page of `order` is forked, or several are copied
        parents = order[:1].repeat(case["moved"]) if case["moved"] < 4 else order[-case["moved"]:]
        st.update(src=parents.contiguous(), dst=order[1: 1 + case["moved"]].contiguous() if case["moved"] < 4
                  else order[: case["moved"]].contiguous())
        if st["dst"].numel() < st["src"].numel():
            st["src"] = st["src"][: st["dst"].numel()].contiguous()
    elif case["op"] == "compact":  # `moved` requests have ended
        live = torch.ones(N, dtype=torch.bool, device="cuda")
        live[order[: case["moved"]].long()] = False
        st["live"] = live
    else:
        st["pages"] = order[: case["moved"]].contiguous()
    return st


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "update":
        return _prepare_update(case, g)
    if case["op"] in ("fn", "train"):
        return _prepare_attention(case, g)
    return _prepare_pages(case, g)


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------


def _counts(st, T, B):
    """valid [B,T], n [B,T] = valid tokens up to and with t, run [B,T] = number of the packed sequence."""
    q = st["q"]
    valid = st["mask"] if st["mask"] is not None else torch.ones(B, T, dtype=torch.bool, device=q.device)
    n = valid.long().cumsum(1)
    run = torch.zeros(B, T, dtype=torch.long, device=q.device)
    if st["seq_idx"] is not None:
        run[:, 1:] = (st["seq_idx"][:, 1:] != st["seq_idx"][:, :-1]).long().cumsum(1)
    return valid, n, run


def _plain_attention(st, q, k, v, init):
    """The chunked form in fp32, all chunks at once: products inside a chunk, the states of all chunks, and the
    chunks' states joined by a matrix of decays between chunks.  Decays in 64 bits, rounded once."""
    case = st["case"]
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    C = 128
    NC = -(-T // C)
    pad = NC * C - T
    valid, n, run = _counts(st, T, B)
    f = torch.nn.functional.pad
    valid = f(valid, (0, pad)).view(B, 1, NC, C)
    n = torch.cat([n, n[:, -1:].expand(B, pad)], 1).view(B, 1, NC, C).double()
    run = torch.cat([run, run[:, -1:].expand(B, pad)], 1).view(B, 1, NC, C)
    chunks = lambda x: f(x.repeat_interleave(H // x.shape[2], 2).permute(0, 2, 1, 3), (0, 0, 0, pad)).reshape(  # noqa: E731
        B, H, NC, C, x.shape[-1]).masked_fill(~valid[..., None], 0.0)
    q, k, v = chunks(q), chunks(k), chunks(v)
    g = st["log_decay"].double().view(1, H, 1, 1)
    n_end, run_end = n[..., -1], run[..., -1]  # [B,1,NC]
    n_before = torch.cat([torch.zeros_like(n_end[..., :1]), n_end[..., :-1]], -1)
    run_before = torch.cat([torch.zeros_like(run_end[..., :1]), run_end[..., :-1]], -1)
    # inside the chunks
    lag = n[..., :, None] - n[..., None, :]
    ok = (run[..., :, None] == run[..., None, :]) & torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp(g[..., None] * lag.clamp_min(0)).masked_fill(~ok, 0.0).float()
    out = ((q @ k.transpose(-1, -2)) * decay) @ v
    # the states that the chunks add, and those that they start from
    w = torch.exp(g * (n_end[..., None] - n)).masked_fill(run != run_end[..., None], 0.0).float()
    added = (k * w[..., None]).transpose(-1, -2) @ v  # [B,H,NC,Dk,Dv]
    before = n_before[..., :, None] - n_end[..., None, :]
    joins = (run_before[..., :, None] == run_end[..., None, :]) & torch.ones(
        NC, NC, dtype=torch.bool, device=q.device).tril(-1)
    m = torch.exp(g * before.clamp_min(0)).masked_fill(~joins, 0.0).float()
    start = (m @ added.reshape(B, H, NC, Dk * Dv)).view(B, H, NC, Dk, Dv)
    if init is not None:
        start = start + torch.exp(g[..., None] * n_before[..., None, None]).float() * init[:, :, None]
    carry = torch.exp(g * (n - n_before[..., None])).masked_fill(run != run_before[..., None], 0.0).float()
    out = (out + (q @ start) * carry[..., None]) * (Dk ** -0.5)
    out = out.masked_fill(~valid[..., None], 0.0).reshape(B, H, NC * C, Dv)[:, :, :T].transpose(1, 2)
    final = None
    if case["final"]:
        final = torch.exp(g * (n_end[..., -1] - n_before[..., -1])[..., None, None]).float() * start[:, :, -1] + added[:, :, -1]
    return out, final


def _plain_fn(st):
    out, final = _plain_attention(st, st["q"].float(), st["k"].float(), st["v"].float(), st["init"])
    return [out.to(st["q"].dtype)] + ([final] if final is not None else [])


def _plain_train(st):
    leaves = [st[n].float().requires_grad_() for n in ("q", "k", "v")]
    if st["init"] is not None:
        leaves.append(st["init"].clone().requires_grad_())
    out, final = _plain_attention(st, *leaves[:3], leaves[3] if st["init"] is not None else None)
    outs, grads = [out], [st["dout"].float()]
    if final is not None:
        outs, grads = [out, final], [grads[0], st["dfinal"]]
    grads = torch.autograd.grad(outs, leaves, grads)
    dt = st["q"].dtype
    return [out.detach().to(dt)] + ([final.detach()] if final is not None else []) + [
        x.to(dt) for x in grads[:3]] + list(grads[3:])


def _plain_update(st):
    H, Dk = st["q"].shape[1:]
    q, k, v = (st[n].float().repeat_interleave(H // st[n].shape[1], 1) for n in ("q", "k", "v"))
    a = torch.exp(st["log_decay"].double()).float().view(1, H, 1, 1)
    new = st["state"] * a + k[..., :, None] * v[..., None, :]
    out = (q[..., :, None] * new).sum(-2) * (Dk ** -0.5)
    if st["mask"] is not None:
        new = torch.where(st["mask"].view(-1, 1, 1, 1), new, st["state"])
        out = out.masked_fill(~st["mask"].view(-1, 1, 1), 0.0)
    st["state"].copy_(new)
    return [out.to(st["q"].dtype), st["state"]]


def _compact_maps(live):
    """source [N]: the page that page i takes over (i itself where it stays); new_index [N]: where page i is
    afterwards (-1: nowhere); count [1].  The holes below the count take, in order, the live pages behind it."""
    N = live.numel()
    at = torch.arange(N, device=live.device)
    count = live.sum()
    hole, tail = ~live & (at < count), live & (at >= count)
    holes = torch.where(hole, at, N).sort().values
    tails = torch.where(tail, at, N).sort().values
    source = torch.where(hole, tails[(hole.cumsum(0) - 1).clamp_min(0)], at)
    new_index = torch.where(tail, holes[(tail.cumsum(0) - 1).clamp_min(0)], torch.where(live, at, -1))
    return source, new_index.int(), count.int().view(1)


def _plain_pages(st):
    op, pools = st["case"]["op"], st["pools"]
    if op == "reorder":
        [t.copy_(t[st["source"].long()]) for t in pools]
    elif op == "copy":
        [t.index_copy_(0, st["dst"].long(), t[st["src"].long()]) for t in pools]
    elif op == "free":
        [t.index_fill_(0, st["pages"].long(), 0.0) for t in pools]
    else:
        source, new_index, count = _compact_maps(st["live"])
        [t.copy_(t[source]) for t in pools]
        return list(pools) + [new_index, count]
    return list(pools)


# ---------------------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------------------


def _own(st):
    import viby_model_b200 as V

    case = st["case"]
    op = case["op"]
    if op == "update":
        out = V.linear_attention_update(st["q"], st["k"], st["v"], st["state"], st["log_decay"], attention_mask=st["mask"])
        return [out, st["state"]]
    if op == "fn":
        r = V.linear_attention_fn(st["q"], st["k"], st["v"], st["log_decay"], st["seq_idx"], st["init"], case["final"],
                                  attention_mask=st["mask"])
        return list(r) if case["final"] else [r]
    if op == "train":
        leaves = [st[n].detach().requires_grad_() for n in ("q", "k", "v")]
        if st["init"] is not None:
            leaves.append(st["init"].detach().requires_grad_())
        r = V.linear_attention_fn(*leaves[:3], st["log_decay"], st["seq_idx"], leaves[3] if len(leaves) > 3 else None,
                                  case["final"], attention_mask=st["mask"])
        outs = list(r) if case["final"] else [r]
        grads = torch.autograd.grad(outs, leaves, [st["dout"], st["dfinal"]][: len(outs)])
        return [x.detach() for x in outs] + list(grads)
    if op == "reorder":
        V.reorder_pages(st["pools"], st["source"])
    elif op == "copy":
        V.copy_pages(st["pools"], st["src"], st["dst"])
    elif op == "free":
        V.free_pages(st["pools"], st["pages"])
    else:
        new_index, count = V.compact_pages(st["pools"], st["live"])
        return list(st["pools"]) + [new_index, count]
    return list(st["pools"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "update":
        return _plain_update(state)
    if op == "fn":
        return _plain_fn(state)
    if op == "train":
        return _plain_train(state)
    return _plain_pages(state)


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("reorder", "copy", "compact", "free"):
        per_page = case["layers"] * (4 * 2 * sum(_CANON) if case["kind"] == "canon" else 4 * case["H"] * case["Dk"] * case["Dv"])
        N = case["pages"]
        if op == "reorder":  # N draws of N rows: about 1 - 1/e of them are read, and all but one in N written
            return dict(bytes=per_page * (N * (1 - math.exp(-1)) + N - 1) + 4 * N, flops=0)
        m = min(case["moved"], N)
        if op == "copy":
            one = case["moved"] < 4  # one page is read for all its forks
            m = min(m, N - 1) if one else m
            return dict(bytes=per_page * (m + (1 if one else m)) + 8 * m, flops=0)
        if op == "free":
            return dict(bytes=per_page * m + 4 * m, flops=0)
        return dict(bytes=2 * per_page * m * (N - m) / N + N + 4 * N + 4, flops=0)  # holes below the count, on average
    B, H, Hk, Hv, Dk, Dv = (case[n] for n in ("B", "H", "Hk", "Hv", "Dk", "Dv"))
    es = 4 if case["dtype"] == "f32" else 2
    states = 4 * B * H * Dk * Dv
    token = es * (H * Dk + Hk * Dk + Hv * Dv + H * Dv)
    if op == "update":
        busy = (B - case["idle"]) / B
        return dict(bytes=busy * (2 * states + B * token), flops=busy * 5 * B * H * Dk * Dv)
    share = 1.0 if case["rows"] in ("full", "packed") else 9 / 16  # of the tokens that are valid, on average
    tokens = B * case["T"] * share
    n = tokens * token + (B * case["T"] if share < 1 else 0) + (4 * case["T"] if case["rows"] == "packed" else 0)
    n += states * (case["init"] + case["final"])
    if op == "fn":
        return dict(bytes=n, flops=4 * tokens * H * Dk * Dv)
    n += tokens * es * (H * Dv + H * Dk + Hk * Dk + Hv * Dv) + states * (case["init"] + case["final"])
    return dict(bytes=n, flops=12 * tokens * H * Dk * Dv)


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------


def _exact_attention(st):
    """Token against token, from o_i = s (a^{n_i} q_i S_0 + sum_{j<=i} a^{n_i-n_j} (q_i.k_j) v_j) and its derivatives,
    for one row and head at a time, in blocks of queries."""
    case = st["case"]
    B, T, H, Dk = st["q"].shape
    Dv = st["v"].shape[-1]
    dev, scale, train = st["q"].device, Dk ** -0.5, case["op"] == "train"
    out = torch.zeros(B, T, H, Dv, dtype=torch.float64, device=dev)
    final = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=dev)
    dq, dk, dv = (torch.zeros(st[n].shape, dtype=torch.float64, device=dev) for n in ("q", "k", "v"))
    dinit = torch.zeros_like(final)
    for b in range(B):
        keep = st["mask"][b].nonzero().view(-1) if st["mask"] is not None else torch.arange(T, device=dev)
        ids = st["seq_idx"][b][keep] if st["seq_idx"] is not None else torch.zeros(keep.numel(), dtype=torch.int32, device=dev)
        n = torch.arange(1, keep.numel() + 1, device=dev, dtype=torch.float64)
        for h in range(H):
            hk, hv = h // (H // case["Hk"]), h // (H // case["Hv"])
            g = float(st["log_decay"][h].double())
            q, k, v = st["q"][b, keep, h].double(), st["k"][b, keep, hk].double(), st["v"][b, keep, hv].double()
            s0 = st["init"][b, h].double() if st["init"] is not None else None
            do = st["dout"][b, keep, h].double() if train else None
            o, gq = torch.zeros(len(n), Dv, dtype=torch.float64, device=dev), torch.zeros_like(q)
            gk, gv = torch.zeros_like(k), torch.zeros_like(v)
            for i in range(0, len(n), 2048):
                e = min(len(n), i + 2048)
                lag = n[i:e, None] - n[None, :e]
                d = torch.where((lag >= 0) & (ids[i:e, None] == ids[None, :e]), torch.exp(g * lag.clamp(min=0)), 0.0) * scale
                p = (q[i:e] @ k[:e].T) * d
                o[i:e] = p @ v[:e]
                if train:
                    dp = (do[i:e] @ v[:e].T) * d
                    gq[i:e] = dp @ k[:e]
                    gk[:e] += dp.T @ q[i:e]
                    gv[:e] += p.T @ do[i:e]
            from_start = torch.exp(g * n)[:, None]
            to_end = torch.exp(g * (len(n) - n))[:, None]
            if s0 is not None:
                o += from_start * (q @ s0) * scale
                final[b, h] = math.exp(g * len(n)) * s0
            final[b, h] += (k * to_end).T @ v
            out[b, keep, h] = o
            if train:
                if s0 is not None:
                    gq += from_start * (do @ s0.T) * scale
                    dinit[b, h] = (q * from_start).T @ do * scale
                if st["dfinal"] is not None:
                    ds = st["dfinal"][b, h].double()
                    gk += to_end * (v @ ds.T)
                    gv += to_end * (k @ ds)
                    dinit[b, h] += math.exp(g * len(n)) * ds
                dq[b, keep, h] = gq
                dk[b, keep, hk] += gk
                dv[b, keep, hv] += gv
    r = [out] + ([final] if case["final"] else [])
    if train:
        r += [dq, dk, dv] + ([dinit] if case["init"] else [])
    return r


def _exact_update(st):
    case = st["case"]
    H, Dk = case["H"], case["Dk"]
    out, new = torch.zeros(case["B"], H, case["Dv"], dtype=torch.float64, device="cuda"), st["state"].double()
    busy = st["mask"].nonzero().view(-1) if st["mask"] is not None else torch.arange(case["B"], device="cuda")
    for h in range(H):
        k, v = st["k"][busy, h // (H // case["Hk"])].double(), st["v"][busy, h // (H // case["Hv"])].double()
        s = math.exp(float(st["log_decay"][h].double())) * new[busy, h] + torch.einsum("bi,bj->bij", k, v)
        new[busy, h] = s
        out[busy, h] = torch.einsum("bi,bij->bj", st["q"][busy, h].double(), s) * Dk ** -0.5
    return [out, new]


def _exact_pages(st):
    """Page by page on the host's lists."""
    op, pools, N = st["case"]["op"], st["pools"], st["case"]["pages"]
    source, zero, more = list(range(N)), [], []
    if op == "reorder":
        source = st["source"].tolist()
    elif op == "copy":
        for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
            source[d] = s
    elif op == "free":
        zero = st["pages"].tolist()
    else:
        live = st["live"].tolist()
        count = sum(live)
        where = [i if x else -1 for i, x in enumerate(live)]
        behind = [i for i in range(count, N) if live[i]]
        for hole, page in zip([i for i in range(count) if not live[i]], behind):
            source[hole], where[page] = page, hole
        more = [torch.tensor(where, dtype=torch.int32), torch.tensor([count], dtype=torch.int32)]
    r = []
    for t in pools:
        x = torch.stack([t[i] for i in source]).double()
        for i in zero:
            x[i] = 0
        r.append(x)
    return r + more


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "update":
        return _exact_update(st)
    if case["op"] in ("fn", "train"):
        return _exact_attention(st)
    return _exact_pages(st)
