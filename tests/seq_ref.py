"""float64 references of the many-sequence operators and the bounds of their f32 and bf16 forms.

Attention: tokens at positions pos0 + i of a sequence see positions [max(0, p + 1 - window), p] of it.
The f32 bound is attn_ref's: a score is off by at most ds = 2^-20 * scale * sum |q k| (the soft-cap adds
1e-6 of its value), which moves the output by at most 2 max(ds) * sum w |v - out|; exponentials, sums and
the quotient add 2^-19 * sum w |v|. bf16 adds the rounding of the weights for their product with V, half
a step each (2^-8 relative), and that of the output: 2^-8 * (sum w |v| + |out|), the second with the
first's error inside: 2^-8 * (1 + 2^-8).
"""
import numpy as np


def attend_f64(q, K, V, pos0, scale, cap=0.0, window=0, there=None, lim=None, bf16=False):
    """q [nq][nh][D], K, V [L][nkv][D] float64 -> (out, tol) [nq][nh][D]; there: [L] which positions have a
    row at all; lim: positions are below it. Tokens with no key give zeros."""
    nq, nh, D = q.shape
    L, nkv = K.shape[:2]
    lim = L if lim is None else lim
    out, tol = np.zeros((nq, nh, D)), np.full((nq, nh, D), 1e-7)
    there = np.ones(L, bool) if there is None else there
    for i in range(nq):
        p = pos0 + i
        if p < 0 or p >= lim:
            continue
        lo = max(0, p + 1 - window) if window else 0
        at = np.arange(lo, p + 1)[there[lo:p + 1]]
        if not at.size:
            continue
        g = nh // nkv
        for j in range(nkv):
            k, v, hs = K[at, j], V[at, j], slice(j * g, (j + 1) * g)
            s = q[i, hs] @ k.T * scale
            ds = 2.0 ** -20 * abs(scale) * (np.abs(q[i, hs]) @ np.abs(k).T)
            if cap > 0:
                s = cap * np.tanh(s / cap)
                ds = ds + 1e-6 * np.abs(s)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            o = w @ v
            mass = w @ np.abs(v)
            # sum w |v - out| <= 2 sum w |v|, and exactly where that is small enough to form
            off = np.einsum("ht,htd->hd", w, np.abs(v[None] - o[:, None])) if g * v.size <= 1 << 22 else 2 * mass
            out[i, hs] = o
            tol[i, hs] += 2 * ds.max(1, keepdims=True) * off + 2.0 ** -19 * mass
            if bf16:
                tol[i, hs] += 2.0 ** -8 * (mass + (1 + 2.0 ** -8) * np.abs(o))
    return out, tol


def plan(ctx, new, page, most, free, cursor, table, cap):
    """The step's bookkeeping, token by token."""
    table = table.copy()
    cu, length, pos, slot = [0], [], [], []
    room = cap  # tokens that the buffer has left, before pages are looked at
    at = cursor
    for s, (c, m) in enumerate(zip(ctx, new)):
        c, m = max(int(c), 0), max(int(m), 0)
        fit = min(m, max(most * page - c, 0), room)
        room -= fit
        held = -(-c // page)
        want = -(-(c + fit) // page) - held
        got = min(want, len(free) - at)
        for j in range(got):
            table[s, held + j] = free[at + j]
        at += got
        taken = min(fit, (held + got) * page - c)
        for p in range(c, c + taken):
            e = table[s, p // page]
            pos.append(p)
            slot.append(-1 if e < 0 else int(e) * page + p % page)
        cu.append(cu[-1] + taken)
        length.append(c + taken)
    pad = [-1] * (cap - cu[-1])
    left = sum(max(int(m), 0) for m in new) - cu[-1]
    return {"cu": np.array(cu, np.int32), "len": np.array(length, np.int32), "pos": np.array(pos + pad, np.int32),
            "slot": np.array(slot + pad, np.int64), "table": table, "state": np.array([at, left], np.int32)}
