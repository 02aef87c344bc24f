"""Cases of the selective-scan operators: the short causal convolution, the
selective state-space scan (both for training and for packed serving batches
with cache-slot state) and the packed batch's metadata.

`run` computes a case in its plain form (elementary torch operations, fp32),
or, with `own` set, through the framework's public entry points. `exact` is the
operators' definition in fp64, written separately: the recurrence step by step
and gradients by automatic differentiation.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _csv(values):
    return ",".join(str(int(v)) for v in values)


def listed():
    return [
        # a decode step of 256 running requests, some idle: slots of the new
        # tokens in the paged cache, new blocks taken where a block is full
        {"name": "metadata decode", "kind": "metadata", "requests": 256, "tokens": 256, "longest": 1,
         "context": 32768, "block": 16},
        # a large mixed step (chunked prefill beside decodes)
        {"name": "metadata mixed", "kind": "metadata", "requests": 1024, "tokens": 8192, "longest": 512,
         "context": 32768, "block": 64},
        # one training step of the convolution over packed documents, the
        # convolution benchmark's channel count
        {"name": "conv train bf16", "kind": "conv_train", "lens": "4096,311,2048,1,4096,1733,77,3000,1022",
         "channels": 4096, "width": 4, "type": "bf16", "bias": True, "silu": True},
        # odd channel count and kernel size, no activation
        {"name": "conv train fp32 odd", "kind": "conv_train", "lens": "1024,2,1001,750", "channels": 1000, "width": 3,
         "type": "fp32", "bias": False, "silu": False},
        # chunked prefill: eight requests, some continuing from the cache
        {"name": "conv prefill", "kind": "conv_serve", "lens": "128,97,1,256,33,200,151,32", "channels": 4096,
         "width": 4, "type": "bf16", "padding": 0, "tail": 0},
        # decode: 256 requests of one token, 26 of them padding
        {"name": "conv decode", "kind": "conv_serve", "lens": _csv([1] * 256), "channels": 4096, "width": 4,
         "type": "bf16", "padding": 26, "tail": 0},
        # one training step of the scan over packed documents: the largest call
        {"name": "scan train bf16", "kind": "scan_train", "lens": "4096,311,2048,1,4096,1733,77,3000,1022",
         "channels": 4096, "states": 16, "groups": 1, "type": "bf16", "gate": True},
        # odd sizes: channels, states and groups that fill no vector
        {"name": "scan train fp32 odd", "kind": "scan_train", "lens": "700,1,513,317", "channels": 1000,
         "states": 12, "groups": 2, "type": "fp32", "gate": False},
        # chunked prefill: eight requests, some continuing from the cache
        {"name": "scan prefill", "kind": "scan_serve", "lens": "128,97,1,256,33,200,151,32", "channels": 4096,
         "states": 16, "groups": 1, "type": "bf16", "padding": 0, "tail": 0},
        # one long prompt alone, a wide state in groups, padded rows behind it
        {"name": "scan prompt long", "kind": "scan_serve", "lens": "8000", "channels": 2048, "states": 64,
         "groups": 8, "type": "fp16", "padding": 0, "tail": 192},
        # decode: 256 requests of one token, 26 of them padding
        {"name": "scan decode", "kind": "scan_serve", "lens": _csv([1] * 256), "channels": 4096, "states": 16,
         "groups": 1, "type": "bf16", "padding": 26, "tail": 0},
        # a few requests decoding: latency is all that counts
        {"name": "scan decode few", "kind": "scan_serve", "lens": "1,1,1,1", "channels": 2048, "states": 16,
         "groups": 1, "type": "bf16", "padding": 0, "tail": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lengths(rng, total, most):
    """Between 1 and `most` sequence lengths that add up to `total`."""
    n = min(_log_int(rng, 1, most), total)
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["metadata", "conv_train", "conv_serve", "scan_train", "scan_train", "scan_serve",
                       "scan_serve"])
    if kind == "metadata":
        longest = rng.choice([1, 4, 64, 512])
        requests = _log_int(rng, 1, 1024)
        return {"kind": kind, "requests": requests, "tokens": min(requests * longest, 16384) + rng.randint(0, 64),
                "longest": longest, "context": _log_int(rng, 64, 32768), "block": rng.choice([16, 32, 64, 100])}
    kinds = ["bf16", "fp16", "fp32"]
    channels = rng.choice([_log_int(rng, 64, 4096), 8 * _log_int(rng, 8, 512), 2048, 4096])
    if kind.endswith("train"):
        lens = _lengths(rng, _log_int(rng, 64, 16384), 64)
        case = {"kind": kind, "lens": _csv(lens), "channels": channels, "type": rng.choice(kinds)}
    else:
        if rng.random() < 0.4:
            lens = [1] * _log_int(rng, 1, 256)
        else:
            lens = _lengths(rng, _log_int(rng, 16, 8192), 64)
        case = {"kind": kind, "lens": _csv(lens), "channels": channels, "type": rng.choice(kinds),
                "padding": rng.randint(0, len(lens) // 8), "tail": rng.choice([0, rng.randint(1, 64)])}
    if kind.startswith("conv"):
        case["width"] = rng.choice([2, 3, 4, 4, 4, 7])
        if kind == "conv_train":
            case["bias"] = rng.random() < 0.7
            case["silu"] = rng.random() < 0.8
        return case
    tokens = sum(lens)
    states = rng.choice([8, 12, 16, 16, 16, 32, 64, 128])
    while states > 16 and tokens * channels * states > 16384 * 4096 * 16:
        states //= 2
    case["states"] = states
    case["groups"] = rng.choice([1, 1, 2, 8])
    case["channels"] = max(1, channels // case["groups"]) * case["groups"]
    if kind == "scan_train":
        case["gate"] = rng.random() < 0.7
    return case


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _requests(case, g, rows):
    """Request metadata of a packed batch: offsets, cache slots (padding
    requests have slot -1), which requests continue from their slot."""
    lens = _lens(case)
    n = len(lens)
    host = np.random.RandomState(rows)
    order = host.permutation(rows)[:n].astype(np.int32)
    if case["padding"]:
        order[host.permutation(n)[:case["padding"]]] = -1
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    init = (torch.rand(n, generator=g, device=DEV) < 0.8).to(torch.int8)
    return starts, torch.from_numpy(order).to(DEV), init


def _scan_inputs(case, g, tokens):
    """Inputs as a state-space layer has them: steps softplus(delta + bias)
    between 1e-3 and 1e-1, decay rates -1 .. -N."""
    dt, d, n, f = TYPES[case["type"]], case["channels"], case["states"], case["groups"]
    step = torch.exp(torch.rand(d, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
    return {
        "u": _randn(g, tokens, d, dtype=dt), "delta": _randn(g, tokens, d, dtype=dt, scale=0.5),
        "A": -torch.arange(1, n + 1, device=DEV, dtype=torch.float32) * torch.exp(_randn(g, d, n, scale=0.1)),
        "B": _randn(g, tokens, f, n, dtype=dt), "C": _randn(g, tokens, f, n, dtype=dt),
        "skip": 1 + _randn(g, d, scale=0.1), "gate": _randn(g, tokens, d, dtype=dt),
        "delta_bias": step + torch.log(-torch.expm1(-step)),
    }


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"kind": kind}
    if kind == "metadata":
        n, longest = case["requests"], case["longest"]
        query = torch.randint(0 if n > 1 else 1, longest + 1, (n,), generator=g, device=DEV)
        if longest == 1:
            query = (torch.rand(n, generator=g, device=DEV) < 0.95).long()
        room = torch.cumsum(query, 0) <= case["tokens"]
        s["query_lens"] = torch.where(room, query, torch.zeros_like(query)).to(torch.int32)
        s["context_lens"] = torch.randint(0, case["context"] + 1, (n,), generator=g, device=DEV, dtype=torch.int32)
        s["block"], s["tokens"] = case["block"], case["tokens"]
        width = -(-(case["context"] + longest) // case["block"])
        pool = torch.randperm(n * width + case["tokens"] + n, generator=g, device=DEV).to(torch.int32)
        s["block_tables"] = pool[:n * width].view(n, width).contiguous()
        s["free_blocks"] = pool[n * width:].contiguous()
        return s
    dt, d, lens = TYPES[case["type"]], case["channels"], _lens(case)
    tokens = s["tokens"] = sum(lens)
    s["longest"] = max(lens)
    if kind == "conv_train":
        w = case["width"]
        s["x"] = _randn(g, 1, tokens, d, dtype=dt).requires_grad_()
        s["weight"] = _randn(g, w, d, dtype=dt, scale=w ** -0.5).requires_grad_()
        s["bias"] = _randn(g, d, dtype=dt, scale=0.5).requires_grad_() if case["bias"] else None
        s["activation"] = "silu" if case["silu"] else None
        s["dout"] = _randn(g, 1, tokens, d, dtype=dt)
        s["cu_seqlens"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    elif kind == "conv_serve":
        w, rows = case["width"], len(lens) + 4
        s["x"] = _randn(g, tokens + case["tail"], d, dtype=dt)
        s["weight"] = _randn(g, w, d, dtype=dt, scale=w ** -0.5)
        s["bias"] = _randn(g, d, dtype=dt, scale=0.5)
        s["activation"] = "silu"
        s["state"] = _randn(g, rows, d, w - 1, dtype=dt)
        s["starts"], s["slots"], s["init"] = _requests(case, g, rows)
        s["out"] = torch.zeros_like(s["x"])
    elif kind == "scan_train":
        s.update(_scan_inputs(case, g, tokens))
        for k in ("u", "delta", "gate"):
            s[k] = s[k][None]
        if not case["gate"]:
            s["gate"] = None
        s["leaves"] = [k for k in ("u", "delta", "A", "B", "C", "skip", "gate", "delta_bias") if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_()
        s["dout"] = _randn(g, 1, tokens, d, dtype=dt)
        s["cu_seqlens"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    else:
        rows = len(lens) + 4
        s.update(_scan_inputs(case, g, tokens + case["tail"]))
        s["state"] = _randn(g, rows, d, case["states"], scale=0.3)
        s["starts"], s["slots"], s["init"] = _requests(case, g, rows)
        s["out"] = torch.zeros_like(s["u"])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _owner(starts, tokens):
    """(request of each token, its position there), for tokens below starts[-1]."""
    t = torch.arange(tokens, device=DEV)
    req = torch.searchsorted(starts.long(), t, right=True) - 1
    return req, t - starts.long()[req]


def _plain_metadata(s):
    bs, tokens = s["block"], s["tokens"]
    query, context = s["query_lens"].long(), s["context_lens"].long()
    table, free = s["block_tables"], s["free_blocks"]
    starts = torch.cat([query.new_zeros(1), torch.cumsum(query, 0)])
    have, need = (context + bs - 1) // bs, (context + query + bs - 1) // bs
    first = torch.cumsum(need - have, 0) - (need - have)
    # the request's new blocks, in request order, from the front of the free list
    col = torch.arange(table.shape[1], device=DEV)
    new = (col >= have[:, None]) & (col < need[:, None])
    pick = (first - have)[:, None] + col
    table.copy_(torch.where(new, free[pick.clamp(0, free.numel() - 1)], table))
    t = torch.arange(tokens, device=DEV)
    live = t < starts[-1]
    req = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=query.numel() - 1)
    pos = context[req] + t - starts[req]
    slot = table[req, torch.where(live, pos // bs, 0)].long() * bs + pos % bs
    return {"starts": starts.to(torch.int32), "has_initial": (context > 0).to(torch.int8),
            "seq_idx": torch.where(live, req, -1).to(torch.int32), "positions": torch.where(live, pos, 0),
            "slot_map": torch.where(live, slot, -1), "blocks_used": (need - have).sum().to(torch.int32).view(1),
            "block_tables": table}


def _taps(x, req, pos, width, history=None):
    """[T, W, D] inputs of every tap; before a sequence's first token zeros or
    `history` [requests, W - 1, D]."""
    t = torch.arange(x.shape[0], device=DEV)[:, None]
    back = torch.arange(width - 1, -1, -1, device=DEV)
    inside = pos[:, None] >= back
    taps = torch.where(inside[..., None], x[(t - back).clamp(min=0)], 0)
    if history is not None and width > 1:
        old = history[req[:, None], (pos[:, None] - back + width - 1).clamp(0, width - 2)]
        taps = torch.where(inside[..., None], taps, old)
    return taps


def _plain_conv_train(s):
    x, w, dout = s["x"][0].detach().float(), s["weight"].detach().float(), s["dout"][0].float()
    width, (tokens, _) = w.shape[0], x.shape
    req, pos = _owner(s["cu_seqlens"], tokens)
    taps = _taps(x, req, pos, width)
    pre = (taps * w).sum(1)
    if s["bias"] is not None:
        pre = pre + s["bias"].detach().float()
    if s["activation"]:
        sig = torch.sigmoid(pre)
        out, dpre = pre * sig, dout * sig * (1 + pre * (1 - sig))
    else:
        out, dpre = pre, dout
    # dx[t] = sum_j w[W-1-j] dpre[t+j] over the later tokens t+j of the sequence
    t = torch.arange(tokens, device=DEV)[:, None]
    ahead = torch.arange(width - 1, -1, -1, device=DEV)
    left = s["cu_seqlens"].long()[req + 1][:, None] - t
    later = torch.where((ahead < left)[..., None], dpre[(t + ahead).clamp(max=tokens - 1)], 0)
    dt = s["x"].dtype
    got = {"out": out.to(dt)[None], "dx": (later * w).sum(1).to(dt)[None],
           "dweight": (taps * dpre[:, None]).sum(0).to(dt)}
    if s["bias"] is not None:
        got["dbias"] = dpre.sum(0).to(dt)
    return got


def _store(state, slots, new):
    """state[slots[i]] = new[i] for the requests that have a slot."""
    rows = state.shape[0]
    owner = torch.full((rows + 1,), -1, dtype=torch.long, device=DEV)
    owner[torch.where(slots >= 0, slots, rows)] = torch.arange(slots.numel(), device=DEV)
    state.copy_(torch.where((owner[:rows] >= 0)[:, None, None], new[owner[:rows].clamp(min=0)], state))


def _plain_conv_serve(s):
    x, w, state = s["x"].float(), s["weight"].float(), s["state"]
    width, starts = w.shape[0], s["starts"].long()
    tokens, slots = x.shape[0], s["slots"].long()
    inside = torch.arange(tokens, device=DEV) < starts[-1]
    req, pos = _owner(s["starts"], tokens)
    req = req.clamp(max=slots.numel() - 1)
    held = (slots >= 0) & (s["init"] != 0)
    history = torch.where(held[:, None, None], state[slots.clamp(min=0)], 0).transpose(1, 2)
    pre = (_taps(x, req, pos, width, history.float()) * w).sum(1) + s["bias"].float()
    s["out"].copy_(torch.where(inside[:, None], (pre * torch.sigmoid(pre)).to(s["out"].dtype), s["out"]))
    if width > 1:
        # the last W - 1 inputs of (old state, the request's tokens)
        n = (starts[1:] - starts[:-1])[:, None]
        at = n + torch.arange(width - 1, device=DEV)
        rows = (starts[:-1, None] + at - (width - 1)).clamp(0, tokens - 1)
        old = torch.gather(history, 1, at.clamp(max=width - 2)[..., None].expand(-1, -1, x.shape[1]))
        _store(state, slots, torch.where((at >= width - 1)[..., None], s["x"][rows], old).transpose(1, 2))
    return {"out": s["out"], "state": state}


def _doubling_scan(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, by doubling."""
    k = 1
    while k < longest:
        b = torch.cat([b[:k], torch.addcmul(b[k:], a[k:], b[:-k])])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _steps(s, rows):
    """(delta, its derivative by the raw step) in fp32."""
    raw = s["delta"].detach().reshape(rows, -1).float() + s["delta_bias"].detach()
    return torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))), torch.sigmoid(raw)


def _by_channel(v, channels):
    """[T, F, N] -> [T, D, N]: channel d belongs to group d * F // D."""
    return v.detach().float().repeat_interleave(channels // v.shape[1], dim=1)


def _plain_scan_train(s):
    u, dout = s["u"][0].detach().float(), s["dout"][0].float()
    tokens, d = u.shape
    A, skip, f = s["A"].detach(), s["skip"].detach(), s["B"].shape[1]
    req, pos = _owner(s["cu_seqlens"], tokens)
    first = (pos == 0)[:, None, None]
    delta, slope = _steps(s, tokens)
    B, C = _by_channel(s["B"], d), _by_channel(s["C"], d)
    a = torch.exp(delta[..., None] * A)
    h = _doubling_scan(torch.where(first, 0, a), (delta * u)[..., None] * B, s["longest"])
    y = (h * C).sum(-1) + skip * u
    got = {"out": y}
    dy = dout
    if s["gate"] is not None:
        z = s["gate"][0].detach().float()
        sig = torch.sigmoid(z)
        got["out"], dy = y * z * sig, dout * z * sig
        got["dgate"] = dout * y * sig * (1 + z * (1 - sig))
    # adjoint of the state: g[t] = C[t] dy[t] + a[t+1] g[t+1] inside a sequence
    ahead = torch.cat([torch.where(first, 0, a)[1:], torch.zeros_like(a[:1])])
    g = _doubling_scan(ahead.flip(0), (C * dy[..., None]).flip(0), s["longest"]).flip(0)
    del ahead
    got["dC"] = (h * dy[..., None]).view(tokens, f, d // f, -1).sum(2)
    got["dB"] = (g * (delta * u)[..., None]).view(tokens, f, d // f, -1).sum(2)
    kept = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    kept = torch.where(first, 0, kept) * a * g  # a[t] h[t-1] g[t]
    gB = (g * B).sum(-1)
    ddelta = ((kept * A).sum(-1) + gB * u) * slope
    got["dA"] = (kept * delta[..., None]).sum(0)
    got["du"] = dy * skip + delta * gB
    got["ddelta"], got["ddelta_bias"], got["dskip"] = ddelta, ddelta.sum(0), (dy * u).sum(0)
    dt = s["u"].dtype
    whole = ("dA", "dskip", "ddelta_bias")
    per_token = ("out", "du", "ddelta", "dgate")
    return {k: v if k in whole else v.to(dt)[None] if k in per_token else v.to(dt) for k, v in got.items()}


def _plain_scan_serve(s):
    rows, d = s["u"].shape
    u, starts, slots, state = s["u"].float(), s["starts"].long(), s["slots"].long(), s["state"]
    tokens = s["tokens"]
    req, pos = _owner(s["starts"], tokens)
    first = (pos == 0)[:, None, None]
    delta = _steps(s, rows)[0]
    a = torch.exp(delta[:tokens, :, None] * s["A"])
    b = (delta * u)[:tokens, :, None] * _by_channel(s["B"], d)[:tokens]
    held = (slots >= 0) & (s["init"] != 0)
    before = torch.where(held[:, None, None], state[slots.clamp(min=0)], 0)
    b = torch.where(first, b + a * before[req], b)
    h = _doubling_scan(torch.where(first, 0, a), b, s["longest"])
    y = (h * _by_channel(s["C"], d)[:tokens]).sum(-1) + s["skip"] * u[:tokens]
    z = s["gate"][:tokens].float()
    s["out"][:tokens] = (y * z * torch.sigmoid(z)).to(s["out"].dtype)
    _store(state, slots, h[starts[1:] - 1])
    return {"out": s["out"], "state": state}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    s, kind = state, state["kind"]
    if own:
        import greta_plugin_b200 as greta

        if kind == "metadata":
            m = greta.packed_batch_metadata(s["query_lens"], s["context_lens"], s["tokens"],
                                            block_tables=s["block_tables"], block_size=s["block"],
                                            free_blocks=s["free_blocks"])
            return {"starts": m.starts, "has_initial": m.has_initial, "seq_idx": m.seq_idx,
                    "positions": m.positions, "slot_map": m.slot_map, "blocks_used": m.blocks_used,
                    "block_tables": s["block_tables"]}
        if kind == "conv_train":
            out = greta.causal_conv1d(s["x"], s["weight"], s["bias"], cu_seqlens=s["cu_seqlens"],
                                      activation=s["activation"])
            keys = [k for k in ("x", "weight", "bias") if s[k] is not None]
            grads = torch.autograd.grad(out, [s[k] for k in keys], s["dout"])
            return {"out": out, **{"d" + k: v for k, v in zip(keys, grads)}}
        if kind == "conv_serve":
            greta.packed_causal_conv1d(s["x"], s["weight"], s["bias"], s["state"], s["starts"], s["slots"],
                                       s["init"], activation=s["activation"], out=s["out"])
            return {"out": s["out"], "state": s["state"]}
        if kind == "scan_train":
            out = greta.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], skip=s["skip"], gate=s["gate"],
                                       delta_bias=s["delta_bias"], delta_softplus=True, cu_seqlens=s["cu_seqlens"])
            grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["dout"])
            return {"out": out, **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
        greta.packed_selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["skip"], s["gate"],
                                    s["delta_bias"], s["state"], s["starts"], s["slots"], s["init"],
                                    delta_softplus=True, out=s["out"])
        return {"out": s["out"], "state": s["state"]}
    with torch.no_grad():
        return {"metadata": _plain_metadata, "conv_train": _plain_conv_train, "conv_serve": _plain_conv_serve,
                "scan_train": _plain_scan_train, "scan_serve": _plain_scan_serve}[kind](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "metadata":
        n, tokens = case["requests"], case["tokens"]
        # lengths in; offsets, flags and per-token numbers out; a table entry read per token
        return {"bytes": 8 * n + 5 * n + tokens * (4 + 8 + 8 + 4), "flops": 10 * tokens + 10 * n}
    es, d, lens = BYTES[case["type"]], case["channels"], _lens(case)
    tokens = sum(lens)
    live = len(lens) - case.get("padding", 0)
    if kind == "conv_train":
        w = case["width"]
        # x, out forward; x, dout, dx backward
        return {"bytes": es * (5 * tokens * d + 4 * w * d), "flops": tokens * d * (6 * w + 20)}
    if kind == "conv_serve":
        w = case["width"]
        return {"bytes": es * (2 * tokens * d + (w + 1) * d + 2 * live * d * (w - 1)),
                "flops": tokens * d * (2 * w + 5)}
    n, f = case["states"], case["groups"]
    if kind == "scan_train":
        rows = 3 if case["gate"] else 2  # u, delta, gate
        fwd = es * tokens * (d * (rows + 1) + 2 * f * n) + 4 * d * (n + 2)
        bwd = es * tokens * (d * (2 * rows + 1) + 4 * f * n) + 8 * d * (n + 2)
        # per state: decay, input, state and output forward; states again, their
        # adjoints and five sums backward
        return {"bytes": fwd + bwd, "flops": tokens * d * (24 * n + 50)}
    return {"bytes": es * tokens * (4 * d + 2 * f * n) + 4 * d * (n + 2) + 8 * live * d * n,
            "flops": tokens * d * (7 * n + 25)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_conv(x, w, bias, silu, lens, history):
    """Sequence by sequence on [W - 1 + n, D] rows."""
    width, outs, at = w.shape[0], [], 0
    for i, n in enumerate(lens):
        rows = torch.cat([history[i], x[at:at + n]])
        pre = sum(rows[k:k + n] * w[k] for k in range(width))
        if bias is not None:
            pre = pre + bias
        outs.append(pre / (1 + torch.exp(-pre)) if silu else pre)
        at += n
    return torch.cat(outs)


def _exact_recurrence(u, raw, A, B, C, skip, gate, before, lens):
    """The recurrence step by step over [sequences, channels, states], the
    sequences sorted by falling length so that the running ones come first.
    B, C: [T, channels or 1, N]. Returns (out [T, D], last states)."""
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    first = np.cumsum([0] + list(lens))
    begin = [int(first[i]) for i in order]
    delta = torch.nn.functional.softplus(raw, threshold=1000)
    h = before[order]
    ys, rows, final = [], [], [None] * len(lens)
    running = len(order)
    for t in range(max(lens)):
        alive = sum(1 for i in order[:running] if lens[i] > t)
        for k in range(alive, running):
            final[order[k]] = h[k]
        running = alive
        at = torch.tensor([b + t for b in begin[:running]], device=DEV)
        h = torch.exp(delta[at, :, None] * A) * h[:running] + (delta[at] * u[at])[..., None] * B[at]
        ys.append((h * C[at]).sum(-1))
        rows.append(at)
    for k in range(running):
        final[order[k]] = h[k]
    y = torch.cat(ys)[torch.argsort(torch.cat(rows))] + skip * u
    if gate is not None:
        y = y * gate / (1 + torch.exp(-gate))
    return y, torch.stack(final)


def exact(case, seed):
    kind = case["kind"]
    if kind == "metadata":
        return None
    s = prepare(case, seed)
    lens, d = _lens(case), case["channels"]
    tokens = sum(lens)
    if kind == "conv_train":
        leaves = {k: s[k].detach().double().requires_grad_() for k in ("x", "weight", "bias") if s[k] is not None}
        zero = torch.zeros(len(lens), case["width"] - 1, d, dtype=torch.float64, device=DEV)
        out = _exact_conv(leaves["x"][0], leaves["weight"], leaves.get("bias"), case["silu"], lens, zero)
        grads = torch.autograd.grad(out[None], list(leaves.values()), s["dout"].double())
        return {"out": out[None].detach(), **{"d" + k: v for k, v in zip(leaves, grads)}}
    live = s["slots"] >= 0 if "slots" in s else None
    if kind == "conv_serve":
        state, x = s["state"].double(), s["x"].double()
        out, history = s["out"].double(), torch.zeros(len(lens), case["width"] - 1, d, dtype=torch.float64, device=DEV)
        at = 0
        for i, n in enumerate(lens):
            slot = int(s["slots"][i])
            if slot >= 0 and int(s["init"][i]):
                history[i] = state[slot].t()
            if slot >= 0 and case["width"] > 1:
                state[slot] = torch.cat([history[i], x[at:at + n]])[1 - case["width"]:].t()
            at += n
        out[:tokens] = _exact_conv(x, s["weight"].double(), s["bias"].double(), True, lens, history)
        return {"out": out, "state": state}
    n, f = case["states"], case["groups"]
    per = d // f
    if kind == "scan_serve":
        if max(lens) * f * 1e-4 > 15:  # about 20 seconds
            return None
        state, out = s["state"].double(), s["out"].double()
        for j in range(f):
            c = slice(j * per, (j + 1) * per)
            v = {k: s[k][:tokens, c].double() for k in ("u", "delta", "gate")}
            before = torch.where((live & (s["init"] != 0))[:, None, None], s["state"][s["slots"].clamp(min=0), c], 0)
            out[:tokens, c], last = _exact_recurrence(
                v["u"], v["delta"] + s["delta_bias"][c].double(), s["A"][c].double(), s["B"][:, j, None].double(),
                s["C"][:, j, None].double(), s["skip"][c].double(), v["gate"], before.double(), lens)
            state[s["slots"][live].long(), c] = last[live]
        return {"out": out, "state": state}
    # blocks of channels, so that what differentiation keeps fits the card
    size = max(1, int(3e9 / (tokens * n)))
    blocks = [(j, slice(lo, min(lo + size, (j + 1) * per))) for j in range(f) for lo in range(j * per, (j + 1) * per, size)]
    if max(lens) * len(blocks) * 6e-4 > 18:  # about 20 seconds
        return None
    got = {"out": torch.empty(1, tokens, d, dtype=torch.float64, device=DEV)}
    for k in s["leaves"]:
        got["d" + k] = torch.zeros(s[k].shape, dtype=torch.float64, device=DEV)
    for j, c in blocks:
        leaf = {}
        for k in s["leaves"]:
            v = s[k].detach().double()
            leaf[k] = (v[0, :, c] if v.dim() == 3 and k in ("u", "delta", "gate") else v[:, j, None] if k in "BC"
                       else v[c]).clone().requires_grad_()
        zero = torch.zeros(len(lens), c.stop - c.start, n, dtype=torch.float64, device=DEV)
        out, _ = _exact_recurrence(leaf["u"], leaf["delta"] + leaf["delta_bias"], leaf["A"], leaf["B"], leaf["C"],
                                   leaf["skip"], leaf.get("gate"), zero, lens)
        grads = dict(zip(leaf, torch.autograd.grad(out, list(leaf.values()), s["dout"][0, :, c].double())))
        got["out"][0, :, c] = out.detach()
        for k, v in grads.items():
            if k in ("u", "delta", "gate"):
                got["d" + k][0, :, c] = v
            elif k in ("B", "C"):
                got["d" + k][:, j] += v[:, 0]
            else:
                got["d" + k][c] = v
    return got
