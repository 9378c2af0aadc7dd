"""Cases of the operators for compressed weight matrices and their plain forms.

Three operators: the 4-bit form of a weight matrix with one scale per (column, row segment) and the residual that a
low-rank fit takes ("quantize"), products with that form and an optional low-rank correction ("product"), and the
distillation loss of the compressed model's logits against the original's top logits ("distill").

Matrices are column-major: an M x N matrix is a tensor (N, ld) whose row j is column j.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step through a small layer: launch latency counts
        {"name": "product-small-1", "op": "product", "dir": "T", "type": "f16", "m": 512, "n": 1024, "t": 1, "seg": 128,
         "zeros": False, "rank": 0, "pad": 0},
        # one decoding step through a square layer, with the low-rank correction that a fit of the residual gives
        {"name": "product-square-1-rank", "op": "product", "dir": "T", "type": "bf16", "m": 4096, "n": 4096, "t": 1, "seg": 128,
         "zeros": False, "rank": 64, "pad": 0},
        # one decoding step through a wide layer, zero points and short segments
        {"name": "product-wide-1-zeros", "op": "product", "dir": "T", "type": "f16", "m": 8192, "n": 16384, "t": 1, "seg": 64,
         "zeros": True, "rank": 0, "pad": 0},
        # a few sequences decoded together, odd sizes, the shortest segments
        {"name": "product-odd-9", "op": "product", "dir": "T", "type": "bf16", "m": 5001, "n": 6003, "t": 9, "seg": 32,
         "zeros": True, "rank": 24, "pad": 3},
        # single precision activations (the fits' own F32 path next to it)
        {"name": "product-single-4", "op": "product", "dir": "T", "type": "f32", "m": 4096, "n": 8192, "t": 4, "seg": 128,
         "zeros": False, "rank": 0, "pad": 0},
        # a short prompt, or the tokens of a training batch, at once
        {"name": "product-prompt-256", "op": "product", "dir": "T", "type": "bf16", "m": 4096, "n": 16384, "t": 256, "seg": 128,
         "zeros": False, "rank": 64, "pad": 0},
        # the gradient to the layer's input, a block of tokens
        {"name": "product-back-64", "op": "product", "dir": "N", "type": "f16", "m": 4096, "n": 16384, "t": 64, "seg": 64,
         "zeros": True, "rank": 32, "pad": 0},
        # a training step on a batch: loss and gradient in one call, a fifth of the tokens masked
        {"name": "distill-step-512", "op": "distill", "mode": "step", "type": "bf16", "n": 128000, "t": 512, "k": 64, "tau": 2.0,
         "tail": False, "masked": 0.2, "pad": 0},
        # loss first, gradient later with what came from above; odd vocabulary; the teacher's rest as one outcome
        {"name": "distill-two-calls-odd", "op": "distill", "mode": "two", "type": "f16", "n": 50257, "t": 301, "k": 32, "tau": 1.0,
         "tail": True, "masked": 0.0, "pad": 0},
        # a handful of tokens checked against the teacher, in single precision, small vocabulary
        {"name": "distill-loss-small", "op": "distill", "mode": "loss", "type": "f32", "n": 8192, "t": 8, "k": 16, "tau": 1.0,
         "tail": True, "masked": 0.0, "pad": 5},
        # a layer brought to 4 bits
        {"name": "quantize-square", "op": "quantize", "type": "bf16", "stype": "bf16", "m": 4096, "n": 4096, "seg": 128,
         "zeros": False, "residual": False, "pad": 0},
        # the same with zero points, and the residual that the low-rank fit takes
        {"name": "quantize-residual-odd", "op": "quantize", "type": "f32", "stype": "f16", "m": 8190, "n": 2049, "seg": 32,
         "zeros": True, "residual": True, "pad": 1},
    ]


def _spread(rng, low, high):
    """A whole number, spread over its logarithm; one in two is a multiple of 64 where there is room."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 128 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["product", "product", "product", "distill", "distill", "quantize"])
    kind = rng.choice(["f16", "bf16", "bf16", "f32"])
    if op == "product":
        while True:
            m, n, t = _spread(rng, 200, 16384), _spread(rng, 200, 32768), _spread(rng, 1, 256)
            if kind == "f32":
                t = min(t, 32)
            if m * n <= 8192 * 16384 and m * n * t <= 4096 * 16384 * 256:
                break
        return {"op": op, "dir": rng.choice(["T", "T", "N"]), "type": kind, "m": m, "n": n, "t": t,
                "seg": rng.choice([32, 64, 128, 256]), "zeros": rng.random() < 0.5,
                "rank": rng.choice([0, 0, _spread(rng, 4, 128)]), "pad": rng.choice([0, 0, 1, 8])}
    if op == "distill":
        while True:
            n, t = _spread(rng, 1000, 256000), _spread(rng, 1, 4096)
            if n * t <= 128000 * 512 and (kind != "f32" or n * t <= 64000 * 512):
                break
        return {"op": op, "mode": rng.choice(["step", "two", "loss"]), "type": kind, "n": n, "t": t, "k": _spread(rng, 1, 128),
                "tau": rng.choice([1.0, 1.0, 2.0, 4.0]), "tail": rng.random() < 0.5, "masked": rng.choice([0.0, 0.3]),
                "pad": rng.choice([0, 0, 3])}
    while True:
        m, n = _spread(rng, 200, 16384), _spread(rng, 200, 16384)
        if m * n <= 8190 * 2049:
            break
    return {"op": op, "type": kind, "stype": rng.choice(["f16", "bf16", "f32"]), "m": m, "n": n, "seg": rng.choice([32, 64, 128, 256]),
            "zeros": rng.random() < 0.5, "residual": rng.random() < 0.5, "pad": rng.choice([0, 0, 1])}


def work(case):
    e = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["op"] == "product":
        m, n, t, r = case["m"], case["n"], case["t"], case["rank"]
        groups = n * -(-m // case["seg"])
        return {"bytes": m * n // 2 + groups * (e + (1 if case["zeros"] else 0)) + (m + n) * (t + r) * e,
                "flops": 2 * m * n * t + 2 * (m + n) * r * t}
    if case["op"] == "distill":
        live = case["t"] - int(case["masked"] * case["t"])
        # "two": the logits are needed once for the loss and once more for the gradient, which comes from above in between
        reads, writes = {"step": (1, 1), "two": (2, 1), "loss": (1, 0)}[case["mode"]]
        small = case["t"] * (case["k"] * 8 + 16)
        return {"bytes": case["n"] * e * (live * reads + case["t"] * writes) + small,
                "flops": case["n"] * live * (4 * reads + 4 * writes)}
    m, n = case["m"], case["n"]
    groups = n * -(-m // case["seg"])
    s = {"f32": 4, "f16": 2, "bf16": 2}[case["stype"]]
    return {"bytes": m * n * e + m * n // 2 + groups * (s + (1 if case["zeros"] else 0)) + (4 * m * n if case["residual"] else 0),
            "flops": 6 * m * n}


# ---------------------------------------------------------------------------------------------------------
# the 4-bit form
# ---------------------------------------------------------------------------------------------------------
# A column is stored in blocks of 128 rows, 64 bytes each, of sixteen 32-bit words.  Row 32 i + 8 c + 2 p + h of the
# block (i, c, p < 4, h < 2) is the nibble p + 4 h of word 4 c + i.  Rows behind the last hold 0.
def _pack(codes):
    n, m = codes.shape
    blocks = -(-m // 128)
    full = codes.new_zeros((n, blocks * 128))
    full[:, :m] = codes
    nib = full.view(n, blocks, 4, 4, 4, 2).permute(0, 1, 3, 2, 5, 4).reshape(n, blocks * 64, 2)
    return (nib[..., 0] | (nib[..., 1] << 4)).contiguous()


def _unpack(packed, m):
    n = packed.shape[0]
    nib = torch.stack((packed & 15, packed >> 4), dim=-1).view(n, -1, 4, 4, 2, 4)
    return nib.permute(0, 1, 3, 2, 5, 4).reshape(n, -1)[:, :m]


def _groups(w, seg):
    """(N, M) -> (N, segments, seg), zeros behind the last row."""
    n, m = w.shape
    segs = -(-m // seg)
    full = w.new_zeros((n, segs * seg))
    full[:, :m] = w
    return full.view(n, segs, seg)


def _quantize(w, seg, stype, zeros):
    """Codes (N, M) uint8, scales (N, segments), zero points or None.  Quotients next to a border in 64 bits."""
    m = w.shape[1]
    g = _groups(w.float(), seg).double()
    if zeros:
        hi, lo = g.amax(2).clamp_min(0), g.amin(2).clamp_max(0)
        scale = ((hi - lo) / 15).float().to(stype)
    else:
        scale = (g.abs().amax(2) / 7).float().to(stype)
    s = scale.double()
    div = torch.where(s > 0, s, torch.ones_like(s))
    if zeros:
        z = torch.where(s > 0, torch.round(-lo / div).clamp(0, 15), torch.zeros_like(s))
        q = (torch.round(g / div[..., None]) + z[..., None]).clamp(0, 15)
    else:
        z = torch.full_like(s, 8)
        q = torch.round(g / div[..., None]).clamp(-7, 7) + 8
    q = torch.where(s[..., None] > 0, q, z[..., None])
    codes = q.to(torch.uint8).view(w.shape[0], -1)[:, :m].contiguous()
    return codes, scale, (z.to(torch.uint8) if zeros else None)


def _values(codes, scale, z, seg):
    """(N, M) in 32 bits: what the codes stand for."""
    m = codes.shape[1]
    g = _groups(codes.float(), seg)
    zero = z.float()[..., None] if z is not None else 8.0
    return ((g - zero) * scale.float()[..., None]).view(codes.shape[0], -1)[:, :m]


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def _weights(gen, n, m):
    """Weights of a trained layer: normal, columns of unequal size, one entry in a thousand larger."""
    w = torch.randn((n, m), generator=gen, device="cuda")
    w *= 0.02 * torch.exp(0.3 * torch.randn((n, 1), generator=gen, device="cuda"))
    big = torch.rand((n, m), generator=gen, device="cuda") < 1e-3
    return torch.where(big, w * 6, w)


def _padded(values, ld, kind):
    """Column-major with a leading dimension that may be larger than the column."""
    out = torch.zeros((values.shape[0], ld), dtype=kind, device="cuda")
    out[:, :values.shape[1]] = values.to(kind)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = TYPES[case["type"]]
    st = {"case": case}
    if case["op"] == "product":
        m, n, t, r, seg = case["m"], case["n"], case["t"], case["rank"], case["seg"]
        codes, st["scales"], st["zeros"] = _quantize(_weights(gen, n, m), seg, kind, case["zeros"])
        st["codes"] = _pack(codes)
        rows_in, rows_out = (m, n) if case["dir"] == "T" else (n, m)
        # activations: normal with a few large features; gradients are smaller and have none
        x = torch.randn((t, rows_in), generator=gen, device="cuda")
        if case["dir"] == "T":
            x[:, ::97] *= 8
        else:
            x *= 0.01
        st["X"] = _padded(x, rows_in + case["pad"], kind)
        st["Y"] = torch.zeros((t, rows_out + case["pad"]), dtype=kind, device="cuda")
        st["U"] = st["V"] = None
        if r:
            st["U"] = (0.01 * torch.randn((r, m), generator=gen, device="cuda")).to(kind)
            st["V"] = (torch.randn((r, n), generator=gen, device="cuda") / math.sqrt(n)).to(kind)
    elif case["op"] == "distill":
        n, t, k = case["n"], case["t"], case["k"]
        base = torch.randn((t, n), generator=gen, device="cuda") * 2
        peak = torch.randint(0, n, (t, 8), generator=gen, device="cuda")
        base.scatter_add_(1, peak, 4 + 3 * torch.rand((t, 8), generator=gen, device="cuda"))
        top, ids = torch.topk(base, k, dim=1)
        st["teacher"], st["ids"] = top.contiguous(), ids.to(torch.int32)
        if k >= 8:      # a teacher that keeps only what carries its mass: shorter lists end in -1
            keep = torch.randint(k // 2, k + 1, (t, 1), generator=gen, device="cuda")
            st["ids"][torch.arange(k, device="cuda")[None, :] >= keep] = -1
        st["lse"] = torch.logsumexp(base / case["tau"], dim=1) if case["tail"] else None
        z = base + 0.7 * torch.randn((t, n), generator=gen, device="cuda")
        st["Z"] = _padded(z, n + case["pad"], kind)
        weight = torch.rand((t,), generator=gen, device="cuda") + 0.5
        masked = int(case["masked"] * t)
        if masked:
            weight[torch.randperm(t, generator=gen, device="cuda")[:masked]] = 0
        # half-precision gradients are trained with a scaled loss: most of them would be subnormal otherwise
        st["weight"] = weight / t * (65536.0 if case["type"] == "f16" else 1.0)
        st["loss"] = torch.zeros((t,), device="cuda")
        st["stats"] = torch.zeros((t, 2), device="cuda")
        st["dZ"] = torch.zeros((t, n + case["pad"]), dtype=kind, device="cuda") if case["mode"] != "loss" else None
    else:
        m, n, seg = case["m"], case["n"], case["seg"]
        st["W"] = _padded(_weights(gen, n, m), m + case["pad"], kind)
        segs = -(-m // seg)
        st["codes"] = torch.zeros((n, -(-m // 128) * 64), dtype=torch.uint8, device="cuda")
        st["scales"] = torch.zeros((n, segs), dtype=TYPES[case["stype"]], device="cuda")
        st["zeros"] = torch.zeros((n, segs), dtype=torch.uint8, device="cuda") if case["zeros"] else None
        st["R"] = torch.zeros((n, m), device="cuda") if case["residual"] else None
    return st


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    return {"product": _plain_product, "distill": _plain_distill, "quantize": _plain_quantize}[st["case"]["op"]](st)


def _plain_product(st):
    case = st["case"]
    m, n = case["m"], case["n"]
    w = _values(_unpack(st["codes"], m), st["scales"], st["zeros"], case["seg"])          # (N, M)
    if case["dir"] == "T":
        x = st["X"][:, :m].float()
        y = x @ w.T
        first, second = st["U"], st["V"]
    else:
        x = st["X"][:, :n].float()
        y = x @ w
        first, second = st["V"], st["U"]
    if first is not None:
        y = y + (x @ first.float().T) @ second.float()
    return y.to(st["Y"].dtype)


def _plain_distill(st):
    case = st["case"]
    n, tau, weight = case["n"], case["tau"], st["weight"]
    u = st["Z"][:, :n].float() / tau
    valid = st["ids"] >= 0
    index = st["ids"].clamp_min(0).long()
    t = (st["teacher"] / tau).masked_fill(~valid, -math.inf).double()
    if case["tail"]:
        p = torch.exp(t - st["lse"].double()[:, None])
        rest = (1 - p.sum(1)).clamp_min(0)
    else:
        p = torch.exp(t - t.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        rest = torch.zeros_like(p[:, 0])
    top = u.amax(1, keepdim=True)
    e = torch.exp(u - top)
    # sums over the vocabulary and the few listed entries in 64 bits: where student and teacher nearly agree, q - p is
    # the difference of two numbers close to one
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    logq = u.gather(1, index).double() - top.double() - torch.log(total)
    # the student's mass outside the list, summed without the listed entries so that nothing cancels
    listed = torch.zeros_like(u, dtype=torch.bool)
    rows = torch.arange(u.shape[0], device=u.device)[:, None].expand_as(index)
    listed[rows[valid], index[valid]] = True
    outside = e.masked_fill(listed, 0).sum(1, dtype=torch.float64)
    log_outside = torch.log(outside) - torch.log(total[:, 0])
    loss = torch.where(valid & (p > 0), p * (torch.log(p) - logq), torch.zeros_like(p)).sum(1)
    if case["tail"]:
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_outside), torch.zeros_like(rest))
    loss = loss.float()
    live = weight != 0
    loss = torch.where(live, loss * weight, torch.zeros_like(loss))
    if case["mode"] == "loss":
        return {"loss": loss}
    mass = p.sum(1) + rest
    outer = mass - rest * total[:, 0] / outside
    d = e * (outer / total[:, 0]).float()[:, None]
    inner = torch.exp(logq) * mass[:, None]
    pairs = (rows[valid], index[valid])
    # an entry that is listed twice counts with both its probabilities
    sums = torch.zeros((u.shape[0], n), dtype=torch.float64, device=u.device).index_put_(pairs, p[valid], accumulate=True)
    d[pairs] = (inner[valid] - sums[pairs]).float()
    d = d * (weight / tau)[:, None]
    d = torch.where(live[:, None], d, torch.zeros_like(d)).to(st["Z"].dtype)
    return {"loss": loss, "dZ": d}


def _plain_quantize(st):
    case = st["case"]
    w = st["W"][:, :case["m"]]
    codes, scale, z = _quantize(w, case["seg"], TYPES[case["stype"]], case["zeros"])
    out = {"codes": _pack(codes), "scales": scale}
    if z is not None:
        out["zeros"] = z
    if case["residual"]:
        out["residual"] = w.float() - _values(codes, scale, z, case["seg"])
    return out


_handles = {}


def _handle():
    """The library's handle of the current stream: made once, as a user's program does."""
    from hyacinth_b200 import api
    stream = torch.cuda.current_stream().cuda_stream
    key = (torch.cuda.current_device(), stream)
    if key not in _handles:
        _handles[key] = api.Hyacin(stream=stream)
    return api, _handles[key]


def _run_own(st):
    api, h = _handle()
    case = st["case"]
    kinds = {"f32": api.F32, "f16": api.F16, "bf16": api.BF16}
    kind = kinds[case["type"]]
    if case["op"] == "product":
        m, n, t, r = case["m"], case["n"], case["t"], case["rank"]
        x, y, codes, scales = st["X"], st["Y"], st["codes"], st["scales"]
        h.product_w4(case["dir"], m, n, t, kind, codes, codes.shape[1], case["seg"], scales, st["zeros"], scales.shape[1],
                     x, x.shape[1], r, st["U"], m, st["V"], n, y, y.shape[1])
        return y[:, :n if case["dir"] == "T" else m]
    if case["op"] == "distill":
        n, t, k = case["n"], case["t"], case["k"]
        z, d = st["Z"], st["dZ"]
        step = d if case["mode"] == "step" else None
        h.distill_loss(kind, n, t, z, z.shape[1], k, st["ids"], st["teacher"], k, case["tau"], st["lse"], st["weight"],
                       st["loss"], st["stats"], step, step.shape[1] if step is not None else 0)
        if case["mode"] == "two":
            h.distill_grad(kind, n, t, z, z.shape[1], k, st["ids"], st["teacher"], k, case["tau"], st["lse"], st["weight"],
                           st["stats"], d, d.shape[1])
        return {"loss": st["loss"]} if d is None else {"loss": st["loss"], "dZ": d[:, :n]}
    m, n = case["m"], case["n"]
    w, codes, scales = st["W"], st["codes"], st["scales"]
    h.quantize_w4(kind, m, n, w, w.shape[1], case["seg"], kinds[case["stype"]], codes, codes.shape[1], scales, st["zeros"],
                  scales.shape[1], st["R"], m)
    out = {"codes": codes, "scales": scales}
    if st["zeros"] is not None:
        out["zeros"] = st["zeros"]
    if st["R"] is not None:
        out["residual"] = st["R"]
    return out


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"product": _exact_product, "distill": _exact_distill, "quantize": _exact_quantize}[case["op"]](case, st)


def _row_of_nibble(m):
    """For each nibble of a stored column, in storage order, the row it belongs to."""
    blocks = -(-m // 128)
    rows = []
    for word in range(16):
        c, i = word // 4, word % 4
        for nibble in range(8):
            h, p = nibble // 4, nibble % 4
            rows.append(32 * i + 8 * c + 2 * p + h)
    one = torch.tensor(rows, device="cuda")
    return (torch.arange(blocks, device="cuda")[:, None] * 128 + one[None, :]).reshape(-1)


def _exact_weights(case, st):
    """(N, M) in 64 bits, a share of the columns at a time."""
    m, n = case["m"], case["n"]
    row = _row_of_nibble(m)
    where = torch.empty_like(row)
    where[row] = torch.arange(row.numel(), device="cuda")
    where = where[:m]
    shift = ((where % 2) * 4).to(torch.uint8)
    group = torch.arange(m, device="cuda") // case["seg"]
    w = torch.empty((n, m), dtype=torch.float64, device="cuda")
    for a in range(0, n, 2048):
        b = min(n, a + 2048)
        q = ((st["codes"][a:b][:, where // 2] >> shift[None, :]) & 15).double()
        z = st["zeros"][a:b].double()[:, group] if st["zeros"] is not None else 8.0
        w[a:b] = (q - z) * st["scales"][a:b].double()[:, group]
    return w


def _exact_product(case, st):
    w = _exact_weights(case, st)
    if case["dir"] == "N":
        w = w.T
    if case["rank"]:
        u, v = st["U"].double(), st["V"].double()
        w = w + (v.T @ u if case["dir"] == "T" else u.T @ v)
    return (w @ st["X"][:, :w.shape[1]].double().T).T


def _exact_distill(case, st):
    n, t, tau = case["n"], case["t"], case["tau"]
    loss = torch.zeros((t,), dtype=torch.float64, device="cuda")
    grad = torch.zeros((t, n), dtype=torch.float64, device="cuda") if case["mode"] != "loss" else None
    for a in range(0, t, 64):
        b = min(t, a + 64)
        ids = st["ids"][a:b].long()
        ok = ids >= 0
        target = torch.zeros((b - a, n + 1), dtype=torch.float64, device="cuda")       # one column more for the padding
        mark = torch.zeros((b - a, n + 1), dtype=torch.float64, device="cuda")
        score = st["teacher"][a:b].double() / tau
        score = torch.where(ok, score, torch.full_like(score, -math.inf))
        norm = st["lse"][a:b].double() if case["tail"] else torch.logsumexp(score, 1)
        slot = torch.where(ok, ids, torch.full_like(ids, n))
        target.scatter_add_(1, slot, torch.exp(score - norm[:, None]))
        mark.scatter_(1, slot, 1.0)
        target, mark = target[:, :n], mark[:, :n] > 0
        logq = torch.log_softmax(st["Z"][a:b, :n].double() / tau, dim=1)
        value = torch.where(target > 0, target * (torch.log(target) - logq), torch.zeros_like(target)).sum(1)
        q = torch.exp(logq)
        g = q * target.sum(1, keepdim=True) - target
        if case["tail"]:
            r = (1 - target.sum(1)).clamp_min(0)
            log_rest = torch.logsumexp(logq.masked_fill(mark, -math.inf), 1)
            value = value + torch.where(r > 0, r * (torch.log(r) - log_rest), torch.zeros_like(r))
            inside = torch.where(mark, torch.zeros_like(q), torch.exp(logq - log_rest[:, None]))
            g = g + r[:, None] * (q - inside)
        w = st["weight"][a:b].double()
        loss[a:b] = value * w
        if grad is not None:
            grad[a:b] = g * (w / tau)[:, None]
    return {"loss": loss} if grad is None else {"loss": loss, "dZ": grad}


def _exact_quantize(case, st):
    m, n, seg = case["m"], case["n"], case["seg"]
    w = st["W"][:, :m].double()
    segs = -(-m // seg)
    stype = TYPES[case["stype"]]
    scale = torch.zeros((n, segs), dtype=stype, device="cuda")
    zero = torch.full((n, segs), 8, dtype=torch.int64, device="cuda")
    q = torch.zeros((n, m), dtype=torch.int64, device="cuda")
    value = torch.zeros((n, m), dtype=torch.float64, device="cuda")
    for b in range(segs):
        part = w[:, b * seg:min(m, (b + 1) * seg)]
        if case["zeros"]:
            low = torch.minimum(part.min(1).values, torch.zeros(n, dtype=torch.float64, device="cuda"))
            high = torch.maximum(part.max(1).values, torch.zeros(n, dtype=torch.float64, device="cuda"))
            span = (high - low) / 15
        else:
            span = part.abs().max(1).values / 7
        scale[:, b] = span.to(torch.float32).to(stype)
        s = scale[:, b].double()
        nonzero = s > 0
        safe = torch.where(nonzero, s, torch.ones_like(s))
        if case["zeros"]:
            zero[:, b] = torch.where(nonzero, torch.round(-low / safe).clamp(0, 15), torch.zeros_like(s)).long()
            code = torch.round(part / safe[:, None]).long() + zero[:, b:b + 1]
            code = code.clamp(0, 15)
        else:
            code = torch.round(part / safe[:, None]).long().clamp(-7, 7) + 8
        code = torch.where(nonzero[:, None], code, zero[:, b:b + 1].expand_as(code))
        q[:, b * seg:b * seg + part.shape[1]] = code
        value[:, b * seg:b * seg + part.shape[1]] = (code - zero[:, b:b + 1]).double() * s[:, None]
    row = _row_of_nibble(m)
    line = torch.cat((q, torch.zeros((n, row.numel() - m), dtype=torch.int64, device="cuda")), 1)[:, row]
    out = {"codes": (line[:, 0::2] + 16 * line[:, 1::2]).to(torch.uint8), "scales": scale}
    if case["zeros"]:
        out["zeros"] = zero.to(torch.uint8)
    if case["residual"]:
        out["residual"] = w - value
    return out
