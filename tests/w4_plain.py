"""Plain 64-bit statements of the 4-bit weight operators and the distillation loss (numpy, test infrastructure)."""
import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # of a rounding, relative
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}           # half the spacing of the subnormals


def kinds():
    import torch
    from hyacinth_b200 import api
    return {"f32": (torch.float32, api.F32), "f16": (torch.float16, api.F16), "bf16": (torch.bfloat16, api.BF16)}


def row_of_nibble():
    """Row within a block of 128 of each nibble of the block's 64 bytes, low nibble of byte 0 first."""
    rows = np.zeros(128, dtype=np.int64)
    for i in range(4):
        for c in range(4):
            for p in range(4):
                for h in range(2):
                    rows[(4 * c + i) * 8 + p + 4 * h] = 32 * i + 8 * c + 2 * p + h
    return rows


def pack(codes, ldq):
    """codes (N, M) -> bytes (N, ldq), rows behind M as 0."""
    n, m = codes.shape
    blocks = -(-m // 128)
    full = np.zeros((n, blocks * 128), dtype=np.uint8)
    full[:, :m] = codes
    nib = full.reshape(n, blocks, 128)[:, :, row_of_nibble()].reshape(n, -1)
    out = np.zeros((n, ldq), dtype=np.uint8)
    out[:, :blocks * 64] = nib[:, 0::2] | (nib[:, 1::2] << 4)
    return out


def unpack(packed, m):
    n = packed.shape[0]
    blocks = -(-m // 128)
    b = packed[:, :blocks * 64]
    nib = np.stack((b & 15, b >> 4), axis=-1).reshape(n, blocks, 128)
    out = np.zeros((n, blocks, 128), dtype=np.uint8)
    out[:, :, row_of_nibble()] = nib
    return out.reshape(n, -1)[:, :m]


def values(codes, scales, zeros, seg):
    """Wq (N, M) in 64 bits from codes (N, M), scales (N, S), zeros (N, S) or None."""
    m = codes.shape[1]
    g = np.arange(m) // seg
    z = 8.0 if zeros is None else zeros.astype(np.float64)[:, g]
    return (codes.astype(np.float64) - z) * scales.astype(np.float64)[:, g]


def round_to(x, kind):
    import torch
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(kinds()[kind][0]).to(torch.float64).numpy()


def quantize(w, seg, skind, zeros):
    """codes (N, M), scales (N, S) as float64, zero points (N, S) or None; w (N, M) float64."""
    n, m = w.shape
    segs = -(-m // seg)
    codes = np.zeros((n, m), dtype=np.uint8)
    scales = np.zeros((n, segs))
    zp = np.zeros((n, segs), dtype=np.uint8)
    for s in range(segs):
        part = w[:, s * seg:(s + 1) * seg]
        bad = ~np.isfinite(part).all(axis=1)
        clean = np.where(np.isfinite(part), part, 0.0)
        lo, hi = np.minimum(clean.min(1), 0), np.maximum(clean.max(1), 0)
        span = (hi - lo) / 15 if zeros else np.maximum(-lo, hi) / 7
        sc = round_to(np.float32(span), skind)
        sc[bad] = np.nan
        scales[:, s] = sc
        live = sc > 0
        safe = np.where(live, sc, 1.0)
        z = np.where(live, np.clip(np.rint(-lo / safe), 0, 15), 0) if zeros else np.full(n, 8.0)
        with np.errstate(invalid="ignore"):
            q = np.rint(clean / safe[:, None])
            q = np.clip(q + z[:, None], 0, 15) if zeros else np.clip(q, -7, 7) + 8
        q = np.where(live[:, None], q, z[:, None])
        codes[:, s * seg:(s + 1) * seg] = q.astype(np.uint8)
        zp[:, s] = z
    return codes, scales, (zp if zeros else None)


def distill(z, ids, teacher, tau, lse_t, weight, want_grad=True):
    """loss (T,), dZ (T, N) and a scale for dZ's errors (T, N), all in 64 bits; z (T, N), ids / teacher (T, K)."""
    t_count, n = z.shape
    loss, grad, scale = np.zeros(t_count), np.zeros((t_count, n)), np.zeros((t_count, n))
    for t in range(t_count):
        w = 1.0 if weight is None else float(weight[t])
        if w == 0:
            continue
        ok = (ids[t] >= 0) & (ids[t] < n)
        idx, score = ids[t][ok].astype(np.int64), teacher[t][ok].astype(np.float64) / tau
        with np.errstate(all="ignore"):
            if lse_t is not None:
                logp = score - float(lse_t[t])
            else:
                top = score.max() if score.size else 0.0
                logp = score - (top + np.log(np.exp(score - top).sum())) if score.size else score
            p = np.exp(logp)
            rest = max(0.0, 1.0 - p.sum()) if lse_t is not None else 0.0
            mass = p.sum() + rest
            u = z[t].astype(np.float64) / tau
            top = u.max()
            e = np.exp(u - top) if np.isfinite(top) else np.zeros(n)
            total = e.sum()
            q = e / total if total > 0 else np.zeros(n)
            out = np.ones(n, dtype=bool)
            out[idx] = False
            qr = q[out].sum()
            logq = np.where((u > -np.inf) & (total > 0), u - top - np.log(total), -np.inf)      # finite where q underflows
            live = p > 0
            kl = (p[live] * (logp[live] - logq[idx[live]])).sum()
            if rest > 0:
                kl += rest * (np.log(rest) - np.log(qr))
            loss[t] = w * kl
            target = np.zeros(n)
            np.add.at(target, idx, p)
            inside = np.where(out & (qr > 0), rest * q / qr if qr > 0 else 0.0, 0.0)
            grad[t] = w / tau * (q * mass - target - inside)
            scale[t] = abs(w) / tau * (q * mass + target + inside)
    return loss, grad, scale
