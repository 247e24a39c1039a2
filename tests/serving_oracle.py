"""Plain 64-bit implementations of the operators that serve several requests:
the shared projection with per-row adapters and drafted-token verification."""
from __future__ import annotations

import numpy as np

NONE = -(2**31)
NO_TOKEN = 0xFFFFFFFF


def rnd(v, k):
    return (v + (1 << (k - 1))) >> k


def project(x, w, slot, adapters, wide):
    """adapters: {slot: (scale, down [r][K], up [N][r])}.  The dot products are
    formed in float64, where every partial sum is a whole number below 2^53
    (at most 2^30 * 32768 = 2^45)."""
    y = np.matmul(x.astype(np.float64), w.astype(np.float64).T).astype(np.int64)
    for i in range(x.shape[0]):
        a = adapters.get(int(slot[i])) if slot is not None else None
        if a is None:
            continue
        scale, down, up = a
        t = np.matmul(down.astype(np.float64), x[i].astype(np.float64)).astype(np.int64)
        t = np.clip(rnd(t * int(scale), 24), -32768, 32767)
        y[i] += np.matmul(up.astype(np.float64), t.astype(np.float64)).astype(np.int64)
    q = np.clip(rnd(y, 4), -(2**31), 2**31 - 1)
    return q.astype(np.int32) if wide else np.clip(rnd(q, 8), -32768, 32767).astype(np.int16)


COEF = [float.fromhex(c) for c in ("0x1.5bba12p-10", "0x1.3cea88p-7", "0x1.c6b752p-5", "0x1.ebf9bcp-3", "0x1.62e42ap-1",
                                   "0x1p+0")]
LOG2E_16 = float.fromhex("0x1.715476p-16")


def weights(z, temperature):
    """Whole-number weights of one row of Q16.16 logits."""
    z = np.asarray(z).astype(np.int64)
    top = int(z.max())
    if not np.float32(temperature) > np.float32(1e-6):
        w = np.zeros(len(z), np.int64)
        if top != NONE:
            w[int(np.argmax(z))] = 1 << 31
        return w
    f32 = np.float32
    scale = f32(LOG2E_16) / f32(temperature)
    e = np.minimum((top - z).astype(f32) * scale, f32(100))
    i = np.rint(e)
    f = (i - e).astype(f32)
    g = np.full(len(z), f32(COEF[0]))
    for c in COEF[1:]:
        g = g * f + f32(c)
    assert g.dtype == np.float32
    w = np.floor(np.ldexp(g.astype(np.float64), 31 - i.astype(np.int64))).astype(np.int64)
    w[z == NONE] = 0
    return w


def shares(w):
    """Q0.40 probabilities of one row of weights."""
    total = int(w.sum())
    if total == 0:
        return np.zeros(len(w), np.int64)
    h = total.bit_length() - 32
    inverse = (1 << 62) // (total >> h)
    return (w * inverse) >> (22 + h)


def verify(target, draft, tokens, offsets, most, temperature, accept_u, sample_u):
    """(tokens [B][most + 1], accepted [B], probs [drafts][2]) as whole numbers."""
    b, vocab = len(offsets) - 1, target.shape[1]
    drafts = len(tokens)
    out = np.full((b, most + 1), NO_TOKEN, np.uint32)
    accepted = np.full(b, NO_TOKEN, np.uint32)
    probs = {}
    for r in range(b):
        at, end = int(offsets[r]), int(offsets[r + 1])
        count = end - at
        if count < 0 or end > drafts or count > most:
            continue
        n, stopped, rest = 0, False, None
        for j in range(count):
            x = int(tokens[at + j])
            p = shares(weights(target[at + r + j], temperature[r]))
            if draft is not None:
                q = shares(weights(draft[at + j], temperature[r]))
                qx = int(q[x]) if x < vocab else 0
            else:
                q = np.zeros(vocab, np.int64)
                qx = 1 << 40
                if x < vocab:
                    q[x] = qx
            px = int(p[x]) if x < vocab else 0
            probs[at + j] = (px, qx)
            if stopped:
                continue
            if int(accept_u[at + j]) * qx < px << 32:
                out[r, j] = x
                n += 1
            else:
                stopped, rest = True, np.maximum(p - q, 0)
        p = rest if stopped and rest.sum() > 0 else shares(weights(target[at + r + n], temperature[r]))
        mass = np.cumsum(p)
        point = int(sample_u[r]) * int(mass[-1]) >> 32
        out[r, n] = int(np.searchsorted(mass, point, side="right")) if mass[-1] else NO_TOKEN
        accepted[r] = n
    return out, accepted, probs
