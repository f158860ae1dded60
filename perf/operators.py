"""Routing and 4-bit matrix-vector operators: their plain forms, inputs and cases.

Four operators that stand around one MoE layer call of the backend:

- matvec: y = W x for 1-16 tokens, W in the backend's 4-bit row formats (Q4_K: 256-weight super-blocks of eight
  scaled groups; MXFP4: 32-weight blocks with an E8M0 scale).
- route: per token the ten largest expert logits and their softmax gates, in the form frc_run_device reads; with
  balance outputs it also makes the per-expert counts, mean probabilities and the balance loss in the same pass.
- balance: those statistics for expert ids that something else chose.
- route_backward: the gradient of the gates and of the balance loss with respect to the logits.

`run` computes the plain form with elementary torch operations in 32 bits while `own` is false, and calls the library
while it is true.
"""
import math

import numpy as np
import torch

own = False

TOPK = 10
ACTIVE = 11           # ten gates and the shared expert's
Q4_K, MXFP4 = 12, 39  # row format ids of the library
FORMATS = {"q4k": Q4_K, "mxfp4": MXFP4}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases

def _matvec(name, fmt, rows, n, tokens, x, y):
    return {"name": name, "op": "matvec", "fmt": fmt, "rows": rows, "n": n, "tokens": tokens, "x": x, "y": y}


def _routing(name, op, tokens, experts, dtype, pad=0, shared=False, masked=0, padded=False, balance=False,
             gates=True):
    """pad: extra elements between rows; masked: experts whose logits are -inf; padded: rows behind the ends of
    sequences (marked invalid, their logits undefined); balance: the statistics or their gradient are wanted;
    gates: the gates' gradient is wanted."""
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "dtype": dtype, "pad": pad,
            "shared": shared, "masked": masked, "padded": padded, "balance": balance, "gates": gates}


def listed():
    return [
        # the router of a decode step: 512 experts and the shared expert's gate, one token (latency)
        _matvec("matvec_router", "q4k", 513, 2048, 1, "f32", "f32"),
        # a dense projection of the same block in the other format, bf16 in and out
        _matvec("matvec_projection", "mxfp4", 4096, 2048, 1, "bf16", "bf16"),
        # a vocabulary head, one token: the largest matrix, bound by its bytes
        _matvec("matvec_head", "q4k", 131072, 2048, 1, "f32", "f32"),
        # a burst at the reference's hidden size, the plugin's largest burst
        _matvec("matvec_burst8", "q4k", 5120, 2560, 8, "f32", "f32"),
        # the largest burst over a vocabulary whose size is no multiple of anything
        _matvec("matvec_burst16", "mxfp4", 50021, 2560, 16, "bf16", "f32"),
        # one decode token: the smallest call
        _routing("route_decode", "route", 1, 512, "f32", shared=True),
        # a prefill burst, bf16 logits (many ties), a few experts switched off
        _routing("route_burst", "route", 512, 512, "bf16", pad=7, shared=True, masked=5),
        # the forward half of a router's training step over padded sequences: selection and statistics in one pass
        _routing("route_train", "route", 16384, 512, "f32", padded=True, balance=True),
        # statistics of ids chosen elsewhere: a small ragged batch, fewer experts
        _routing("balance_small", "balance", 333, 160, "bf16", balance=True),
        # and of a large batch
        _routing("balance_large", "balance", 65536, 512, "f32", balance=True),
        # the backward half: both gradients, padded sequences
        _routing("backward_train", "route_backward", 16384, 512, "f32", shared=True, padded=True, balance=True),
        # the balance loss alone, bf16 logits of a small ragged batch
        _routing("backward_small", "route_backward", 777, 200, "bf16", pad=3, balance=True, gates=False),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("matvec", "matvec", "route", "balance", "route_backward"))
    if op == "matvec":
        fmt = rng.choice(tuple(FORMATS))
        step = 256 if fmt == "q4k" else 32
        n = step * _log_uniform(rng, 256 // step, 16384 // step)
        tokens = rng.choice((1, 1, rng.randint(1, 16)))
        rows = _log_uniform(rng, 64, min(131072, 131072 * 2048 // n, 50021 * 2560 * 16 // (n * tokens)))
        c = _matvec("", fmt, rows, n, tokens, rng.choice(tuple(DTYPES)), rng.choice(tuple(DTYPES)))
    else:
        experts = rng.choice((512, rng.randint(16, 512)))
        c = _routing("", op, _log_uniform(rng, 1, 32768 if op == "route_backward" else 65536), experts, rng.choice(tuple(DTYPES)),
                     pad=rng.choice((0, 0, rng.randint(1, 31))), shared=op != "balance" and rng.random() < 0.5,
                     masked=rng.choice((0, 0, rng.randint(1, 5))), padded=rng.random() < 0.5,
                     balance=op == "balance" or rng.random() < 0.6)
        if op == "route_backward":
            c["gates"] = not c["balance"] or rng.random() < 0.7
            c["shared"] = c["shared"] and c["gates"]
    del c["name"]
    return c


# ----------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _encode_q4k(w):
    """[rows][n] weights -> Q4_K row bytes: per 32 an affine range that holds zero, 6-bit scales and minima against
    fp16 super scales."""
    rows, n = w.shape
    g = w.view(rows, n // 256, 8, 32)
    lo = g.amin(-1).clamp_max(0.0)
    hi = g.amax(-1).clamp_min(0.0)
    step = (hi - lo) / 15
    d = (step.amax(-1) / 63).half()
    dmin = (-lo.amin(-1) / 63).half()
    df, mf = d.float()[..., None], dmin.float()[..., None]
    sc = (step / df.clamp_min(1e-30)).round().clamp(0, 63)
    mi = (-lo / mf.clamp_min(1e-30)).round().clamp(0, 63)
    q = ((g + (mf * mi)[..., None]) / (df * sc)[..., None].clamp_min(1e-30)).round().clamp(0, 15).to(torch.uint8)
    sc, mi = sc.to(torch.uint8), mi.to(torch.uint8)
    out = torch.empty(rows, n // 256, 144, dtype=torch.uint8, device=w.device)
    out[..., 0:2] = d[..., None].view(torch.uint8)
    out[..., 2:4] = dmin[..., None].view(torch.uint8)
    out[..., 4:8] = sc[..., :4] | (sc[..., 4:] >> 4) << 6
    out[..., 8:12] = mi[..., :4] | (mi[..., 4:] >> 4) << 6
    out[..., 12:16] = (sc[..., 4:] & 15) | (mi[..., 4:] & 15) << 4
    out[..., 16:] = (q[:, :, 0::2] | q[:, :, 1::2] << 4).reshape(rows, n // 256, 128)
    return out.view(rows, -1)


def _encode_mxfp4(w):
    """[rows][n] weights -> MXFP4 row bytes: the exponent that fits the largest magnitude under 6, nearest E2M1."""
    rows, n = w.shape
    b = w.view(rows, n // 32, 32)
    k = (b.abs().amax(-1).clamp_min(1e-37) / 6).log2().ceil()
    r = b.abs() / torch.exp2(k)[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    code = torch.bucketize(r, edges).to(torch.uint8) | (b < 0).to(torch.uint8) << 3
    out = torch.empty(rows, n // 32, 17, dtype=torch.uint8, device=w.device)
    out[..., 0] = (k + 127).to(torch.uint8)
    out[..., 1:] = code[..., :16] | code[..., 16:] << 4
    return out.view(rows, -1)


def _matvec_inputs(case, seed):
    gen = _generator(seed)
    rows, n, tokens = case["rows"], case["n"], case["tokens"]
    encode = _encode_q4k if case["fmt"] == "q4k" else _encode_mxfp4
    parts, chunk = [], max(1, (1 << 26) // n)
    for r in range(0, rows, chunk):
        w = torch.randn(min(chunk, rows - r), n, generator=gen, device="cuda") * 0.02
        parts.append(encode(w))
    # normed activations; a few channels stand out, as they do in trained models
    x = torch.randn(tokens, n, generator=gen, device="cuda")
    x[:, torch.randperm(n, generator=gen, device="cuda")[:n // 64]] *= 8
    return {"weights": torch.cat(parts), "x": x.to(DTYPES[case["x"]])}


def _choose(logits, valid):
    """The ten largest logits of every row: values descending, ties by index; a row that is not valid gets 0..9."""
    left = logits.clone()
    left[~valid] = 0
    index = torch.arange(logits.shape[1], device=logits.device)
    free = torch.ones_like(left, dtype=torch.bool)
    out = []
    for _ in range(TOPK):
        best = torch.where(free, left, -torch.inf).amax(1, keepdim=True)
        pick = torch.where(free & (left == best), index, logits.shape[1]).amin(1, keepdim=True)
        free.scatter_(1, pick, False)
        out.append(pick)
    return torch.cat(out, 1)


def _routing_inputs(case, seed):
    gen = _generator(seed)
    T, E = case["tokens"], case["experts"]
    cols = E + int(case["shared"])
    dt = DTYPES[case["dtype"]]
    buf = torch.zeros(T, cols + case["pad"], dtype=dt, device="cuda")
    # some experts are more popular than others
    popularity = torch.randn(E, generator=gen, device="cuda")
    logits = buf[:, :cols]
    logits.copy_(torch.randn(T, cols, generator=gen, device="cuda") * 1.5)
    logits[:, :E] += popularity.to(dt)
    if case["masked"]:
        logits[:, torch.randperm(E, generator=gen, device="cuda")[:case["masked"]]] = -torch.inf
    valid = torch.ones(T, dtype=torch.bool, device="cuda")
    if case["padded"]:
        # sequences of 256 positions, each filled to a length of its own; what lies behind is undefined
        lengths = torch.randint(128, 257, ((T + 255) // 256,), generator=gen, device="cuda")
        pos = torch.arange(T, device="cuda")
        valid = pos % 256 < lengths[pos // 256]
        logits[~valid] = torch.nan
    s = {"buffer": buf, "logits": logits, "valid": valid}
    if case["op"] != "route":
        chosen_by = logits[:, :E].float()
        if case["op"] == "balance":  # chosen elsewhere, by noisy logits
            chosen_by = chosen_by + 0.5 * torch.randn(T, E, generator=gen, device="cuda")
        s["expert"] = _choose(chosen_by, valid).to(torch.int16)
    if case["op"] == "route_backward":
        # gradients of a loss that is a mean over the batch, and the usual small weight of the balance loss
        s["d_gate"] = torch.randn(T, ACTIVE, generator=gen, device="cuda") / T if case["gates"] else None
        s["d_loss"] = torch.full((1,), 0.01, device="cuda")
        e = s["expert"].long()
        taken = valid[:, None] & (logits.gather(1, e) > -torch.inf)
        count = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
        count.scatter_add_(0, e.reshape(-1), taken.reshape(-1).long())
        count[E] = valid.sum()
        s["count"] = count.to(torch.int32)
    return s


def _inputs(case, seed):
    return (_matvec_inputs if case["op"] == "matvec" else _routing_inputs)(case, seed)


_ctx = None


def _context():
    """The backend context a program opens once."""
    global _ctx
    if _ctx is None:
        import fronk_b200 as fb
        _ctx = fb.Context(torch.cuda.current_device())
    return _ctx


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    import fronk_b200 as fb
    ctx = s["ctx"] = _context()
    T = case["tokens"]
    if case["op"] == "matvec":
        w = s.pop("weights")
        torch.cuda.current_stream().synchronize()
        s["matrix"] = ctx.matrix(FORMATS[case["fmt"]], case["rows"], case["n"], w.data_ptr(), w.numel())
        s["y_out"] = torch.empty(T, case["rows"], dtype=DTYPES[case["y"]], device="cuda")
        return s
    E = case["experts"]
    s["mask"] = s["valid"].to(torch.uint8) if case["padded"] else None
    if case["op"] == "route":
        s["expert_out"] = torch.empty(T, TOPK, dtype=torch.int16, device="cuda")
        s["gate_out"] = torch.empty(T, ACTIVE, device="cuda")
    if case["op"] != "route_backward" and case["balance"]:
        s["loss_out"] = torch.empty(1, device="cuda")
        s["count_out"] = torch.empty(E + 1, dtype=torch.int32, device="cuda")
        s["prob_out"] = torch.empty(E, device="cuda")
        s["workspace"] = torch.empty(fb.balance_workspace(T, E), dtype=torch.uint8, device="cuda")
        s["balance"] = fb.Balance(s["loss_out"].data_ptr(), s["count_out"].data_ptr(), s["prob_out"].data_ptr(),
                                  s["workspace"].data_ptr(), s["workspace"].numel())
    if case["op"] == "route_backward":
        s["d_out"] = torch.zeros_like(s["buffer"])
    return s


# ----------------------------------------------------------------- plain

def _decode(fmt, rows, n, raw):
    """fp32 weights of 4-bit rows."""
    if fmt == "q4k":
        b = raw.view(rows, n // 256, 144)
        d = b[..., 0:2].contiguous().view(torch.float16).float()
        dmin = b[..., 2:4].contiguous().view(torch.float16).float()
        lo, mid, hi = b[..., 4:8], b[..., 8:12], b[..., 12:16]
        sc = torch.cat([lo & 63, (hi & 15) | (lo >> 6) << 4], -1).float()
        mi = torch.cat([mid & 63, (hi >> 4) | (mid >> 6) << 4], -1).float()
        nib = b[..., 16:].reshape(rows, n // 256, 4, 1, 32)
        q = torch.cat([nib & 15, nib >> 4], 3).reshape(rows, n // 256, 8, 32).float()
        return (q * (d * sc)[..., None] - (dmin * mi)[..., None]).view(rows, n)
    b = raw.view(rows, n // 32, 17)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=raw.device)
    code = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    scale = torch.exp2(b[..., :1].float() - 127)
    return (table[code.int()] * scale).view(rows, n)


def _plain_matvec(s):
    c = s["case"]
    w = _decode(c["fmt"], c["rows"], c["n"], s["weights"])
    return (s["x"].float() @ w.t()).to(DTYPES[c["y"]])


def _softmax(l, valid):
    """Rows' softmax; zero where a row is not valid or has nothing left."""
    l = torch.where(valid[:, None], l, -torch.inf)
    m = l.amax(1, keepdim=True)
    e = torch.exp(l - torch.where(m > -torch.inf, m, 0.0))
    return e / e.sum(1, keepdim=True).clamp_min(1e-30)


def _statistics(l, expert, valid, E):
    p = _softmax(l, valid)
    n = valid.sum()
    taken = valid[:, None] & (l.gather(1, expert) > -torch.inf)
    count = torch.zeros(E + 1, dtype=torch.int64, device=l.device)
    count.scatter_add_(0, expert.reshape(-1), taken.reshape(-1).long())
    count[E] = n
    prob = p.sum(0, dtype=torch.float64) / n.clamp_min(1)
    loss = E * (count[:E] * prob).sum() / (TOPK * n.clamp_min(1))
    return loss.float().reshape(1), count.to(torch.int32), prob.float()


def _plain_route(s):
    c = s["case"]
    E, valid = c["experts"], s["valid"]
    l = s["logits"].float()
    expert = _choose(l[:, :E], valid)
    gate = torch.zeros(c["tokens"], ACTIVE, device=l.device)
    gate[:, :TOPK] = _softmax(l.gather(1, expert), valid)
    if c["shared"]:
        gate[:, TOPK] = torch.where(valid, 1 / (1 + torch.exp(-l[:, E])), 0.0)
    out = [expert.to(torch.int16), gate]
    if c["balance"]:
        out += _statistics(l[:, :E], expert, valid, E)
    return out


def _plain_balance(s):
    E = s["case"]["experts"]
    return list(_statistics(s["logits"][:, :E].float(), s["expert"].long(), s["valid"], E))


def _plain_backward(s):
    c = s["case"]
    E, valid = c["experts"], s["valid"]
    l = s["logits"].float()
    d = torch.zeros_like(l)
    if c["balance"]:
        p = _softmax(l[:, :E], valid)
        count = s["count"][:E].float()
        n = s["count"][E].float()
        scale = s["d_loss"] * E / (TOPK * n * n)
        d[:, :E] = scale * p * (count - (p * count).sum(1, keepdim=True))
    if c["gates"]:
        e = s["expert"].long()
        g = _softmax(l.gather(1, e), valid)
        dg = s["d_gate"][:, :TOPK]
        d.scatter_add_(1, e, g * (dg - (g * dg).sum(1, keepdim=True)))
        if c["shared"]:
            sg = 1 / (1 + torch.exp(-l[:, E]))
            d[:, E] = torch.where(valid, sg * (1 - sg) * s["d_gate"][:, TOPK], 0.0)
    return d.to(DTYPES[c["dtype"]])


# ------------------------------------------------------------------- run

def run(s):
    c = s["case"]
    if not own:
        return {"matvec": _plain_matvec, "route": _plain_route, "balance": _plain_balance,
                "route_backward": _plain_backward}[c["op"]](s)
    import fronk_b200 as fb
    ctx, T, stream = s["ctx"], c["tokens"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "matvec":
        y = s["y_out"]
        s["matrix"].matvec_device(T, s["x"].data_ptr(), y.data_ptr(), x_type=_type(fb, c["x"]),
                                  y_type=_type(fb, c["y"]), stream=stream)
        return y
    E, dt, logits = c["experts"], _type(fb, c["dtype"]), s["buffer"]
    valid = None if s["mask"] is None else s["mask"].data_ptr()
    flags = fb.ROUTE_SHARED if c["shared"] else 0
    if c["op"] == "route":
        ctx.route_device(T, E, logits.data_ptr(), s["expert_out"].data_ptr(), s["gate_out"].data_ptr(),
                         stride=logits.shape[1], type_=dt, valid_ptr=valid, flags=flags, balance=s.get("balance"),
                         stream=stream)
        out = [s["expert_out"], s["gate_out"]]
        return out + [s["loss_out"], s["count_out"], s["prob_out"]] if c["balance"] else out
    if c["op"] == "balance":
        ctx.balance_device(T, E, logits.data_ptr(), s["expert"].data_ptr(), s["balance"], stride=logits.shape[1],
                           type_=dt, valid_ptr=valid, stream=stream)
        return [s["loss_out"], s["count_out"], s["prob_out"]]
    ctx.route_backward_device(T, E, logits.data_ptr(), s["expert"].data_ptr(), s["d_out"].data_ptr(),
                              d_gate_ptr=s["d_gate"].data_ptr() if c["gates"] else None,
                              count_ptr=s["count"].data_ptr() if c["balance"] else None,
                              d_loss_ptr=s["d_loss"].data_ptr() if c["balance"] else None,
                              stride=logits.shape[1], d_stride=logits.shape[1], type_=dt, valid_ptr=valid,
                              flags=flags, stream=stream)
    return s["d_out"][:, :E + int(c["shared"])]


def _type(fb, name):
    return fb.BF16 if name == "bf16" else fb.F32


# ------------------------------------------------------------------ work

def work(case):
    T = case["tokens"]
    if case["op"] == "matvec":
        rows, n = case["rows"], case["n"]
        weights = rows * (n // 256 * 144 if case["fmt"] == "q4k" else n // 32 * 17)
        size = {"f32": 4, "bf16": 2}
        return {"bytes": weights + T * (n * size[case["x"]] + rows * size[case["y"]]), "flops": 2 * rows * n * T}
    E, size = case["experts"], 4 if case["dtype"] == "f32" else 2
    cols = E + int(case["shared"])
    row = T * cols * size
    ids, gates = T * TOPK * 2, T * ACTIVE * 4
    mask = T if case["padded"] else 0
    stats = 8 * E + 8
    if case["op"] == "route":
        # a compare per logit and choice is not counted: one look at each, and the softmax where it is wanted
        return {"bytes": row + mask + ids + gates + (stats if case["balance"] else 0),
                "flops": T * E * (5 if case["balance"] else 1)}
    if case["op"] == "balance":
        return {"bytes": row + mask + ids + stats, "flops": T * E * 4}
    # without the balance term only the chosen logits are read
    read = row if case["balance"] else T * (ACTIVE if case["shared"] else TOPK) * size
    return {"bytes": read + row + mask + (ids + gates if case["gates"] else 0) + (stats if case["balance"] else 0),
            "flops": T * E * (7 if case["balance"] else 1)}


# ----------------------------------------------------------------- exact

def _exact_matvec(case, s):
    rows, n = case["rows"], case["n"]
    x = s["x"].double()
    y = torch.empty(case["tokens"], rows, dtype=torch.float64, device="cuda")
    chunk = max(1, (1 << 26) // n)
    for r in range(0, rows, chunk):
        raw = s["weights"][r:r + chunk]
        k = raw.shape[0]
        w = torch.empty(k, n, dtype=torch.float64, device="cuda")
        if case["fmt"] == "q4k":
            for sb in range(n // 256):
                b = raw[:, 144 * sb:144 * sb + 144].long()
                half = (b[:, 0:4:2] | b[:, 1:4:2] << 8).to(torch.int32).to(torch.int16).view(torch.float16).double()
                for g in range(8):
                    if g < 4:
                        sc, mi = b[:, 4 + g] % 64, b[:, 8 + g] % 64
                    else:
                        sc = b[:, 8 + g] % 16 + 16 * (b[:, g] // 64)
                        mi = b[:, 8 + g] // 16 + 16 * (b[:, 4 + g] // 64)
                    byte = b[:, 16 + 32 * (g // 2):48 + 32 * (g // 2)]
                    level = byte // 16 if g % 2 else byte % 16
                    at = 256 * sb + 32 * g
                    w[:, at:at + 32] = (half[:, :1] * sc[:, None]) * level - half[:, 1:] * mi[:, None]
        else:
            for bl in range(n // 32):
                b = raw[:, 17 * bl:17 * bl + 17].long()
                code = torch.cat([b[:, 1:] % 16, b[:, 1:] // 16], 1)
                ex, man = code // 2 % 4, code % 2
                mag = torch.where(ex > 0, torch.exp2(ex.double() - 1) * (1 + man / 2), man / 2)
                sign = 1.0 - 2.0 * (code // 8)
                w[:, 32 * bl:32 * bl + 32] = sign * mag * torch.exp2(b[:, :1].double() - 127)
        y[:, r:r + k] = x @ w.t()
    return y


def _exact_routing(case, s):
    """Row by row in 64 bits on the host's arrays."""
    E, T = case["experts"], case["tokens"]
    l = s["logits"].double().cpu().numpy()
    valid = s["valid"].cpu().numpy()
    L = np.where(valid[:, None], l[:, :E], -np.inf)
    top = L.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        z = np.where(np.isneginf(top), 0.0, np.exp(L - np.where(np.isneginf(top), 0.0, top)))
    total = z.sum(1, keepdims=True)
    p = np.divide(z, total, out=np.zeros_like(z), where=total > 0)
    if case["op"] == "route":
        order = np.argsort(np.where(valid[:, None], -l[:, :E], 0.0), axis=1, kind="stable")[:, :TOPK]
    else:
        order = s["expert"].cpu().numpy().astype(np.int64)
    # the gates have a softmax of their own: a chosen logit far below the row's largest keeps its share of the ten
    lp = np.take_along_axis(L, order, 1)
    lt = lp.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        picked = np.where(np.isneginf(lt), 0.0, np.exp(lp - np.where(np.isneginf(lt), 0.0, lt)))
    share = picked.sum(1, keepdims=True)
    g = np.divide(picked, share, out=np.zeros_like(picked), where=share > 0)
    sig = np.zeros(T)
    if case["shared"]:
        sig[valid] = 1 / (1 + np.exp(-l[valid, E]))
    if case["op"] == "route_backward":
        d = np.zeros((T, E + int(case["shared"])))
        if case["balance"]:
            count = s["count"].cpu().numpy().astype(np.float64)
            n = count[E]
            factor = s["d_loss"].double().item() * E / (TOPK * n * n) if n else 0.0
            d[:, :E] = factor * p * (count[:E] - (p @ count[:E])[:, None])
        if case["gates"]:
            dg = s["d_gate"].double().cpu().numpy()
            term = g * (dg[:, :TOPK] - (g * dg[:, :TOPK]).sum(1, keepdims=True))
            np.add.at(d, (np.arange(T)[:, None], order), term)
            if case["shared"]:
                d[:, E] = sig * (1 - sig) * dg[:, TOPK]
        return torch.from_numpy(d)
    out = []
    if case["op"] == "route":
        gate = np.concatenate([g, sig[:, None]], 1)
        out = [torch.from_numpy(order.astype(np.int16)), torch.from_numpy(gate)]
    if case["balance"]:
        n = int(valid.sum())
        hit = order[valid][~np.isneginf(lp[valid])]
        count = np.append(np.bincount(hit, minlength=E), n)
        prob = p.sum(0) / max(n, 1)
        loss = E * float(count[:E] @ prob) / (TOPK * max(n, 1))
        out += [torch.tensor([loss], dtype=torch.float64), torch.from_numpy(count.astype(np.int32)),
                torch.from_numpy(prob)]
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "matvec":
        return _exact_matvec(case, s)
    return _exact_routing(case, s)
