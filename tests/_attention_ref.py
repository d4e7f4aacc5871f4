"""The quantised attention, the paging plan and the cache write from their definitions, in 64-bit integers (numpy), for the tests."""
import numpy as np

ONE = 1 << 14
LO, HI = -(1 << 31), (1 << 31) - 1


def exp_tables():
    from oracle.graph import exp_lut
    hi, lo, log_base = exp_lut(ONE)
    assert log_base == 9 and len(hi) == 512
    return hi, lo


def attend(q, k, v, limits, score_mul=ONE):
    """rows q [n, H, d] over keys k, v [m, KV, d]; row i sees the keys [0, limits[i]) that `there` holds"""
    hi, lo = exp_tables()
    n, H, d = q.shape
    G = H // k.shape[1]
    out = np.zeros((n, H, d), np.int64)
    with np.errstate(over="ignore"):
        for h in range(H):
            kk, vv = k[:, h // G].astype(np.int64), v[:, h // G].astype(np.int64)
            for i in range(n):
                see = limits[i]
                if np.ndim(see) == 0:
                    see = np.arange(len(kk)) < see
                if not see.any():
                    continue
                x = np.clip((kk[see] * q[i, h].astype(np.int64)[None, :]).sum(axis=1) >> 14, LO, HI)
                x = np.clip((x * score_mul) >> 14, LO, HI)
                z = np.minimum(x.max() - x, (1 << 18) - 1)
                e = (hi[z >> 9] * lo[z & 511]) >> 14
                p = (e * ((1 << 28) // e.sum())) >> 14
                out[i, h] = np.clip((p[:, None] * vv[see]).sum(axis=0) >> 14, LO, HI)
    return out.astype(np.int32)


def prompt(q, k, v, lens, score_mul=ONE, causal=True):
    out, at = np.zeros(q.shape, np.int32), 0
    for n in lens:
        s = slice(at, at + n)
        out[s] = attend(q[s], k[s], v[s], [i + 1 if causal else n for i in range(n)], score_mul)
        at += n
    return out


def mask_weighs(q, k, limits, positions, score_mul, fill, tokens):
    """whether a key behind some row's own, whose score is `fill` in a graph of `tokens` tokens, would have a weight or be the maximum there"""
    hi, lo = exp_tables()
    n, H, d = q.shape
    G = H // k.shape[1]
    for h in range(H):
        kk = k[:, h // G].astype(np.int64)
        for i in range(n):
            see = limits[i]
            if np.ndim(see) == 0:
                see = np.arange(len(kk)) < see
            if not see.any() or positions[i] + 1 >= tokens:
                continue
            with np.errstate(over="ignore"):
                x = np.clip((kk[see] * q[i, h].astype(np.int64)[None, :]).sum(axis=1) >> 14, LO, HI)
            m = int(np.clip((x * score_mul) >> 14, LO, HI).max())
            z = min(max(m - fill, 0), (1 << 18) - 1)
            if fill > m or (int(hi[z >> 9]) * int(lo[z & 511])) >> 14:
                return True
    return False


def plan(have, new, table, free, n_free, block, n_blocks, cap):
    """the step's outputs, on copies"""
    table, free = table.copy(), free.copy()
    up = lambda n: -(-n // block)  # noqa: E731
    status = 0
    for c, f in zip(have, new):
        if c < 0 or f < -1:
            status |= 8
        elif up(c + max(f, 0)) > table.shape[1]:
            status |= 2
    back = sum(up(c) for c, f in zip(have, new) if f < 0) if not status else 0
    need = sum(up(c + f) - up(c) for c, f in zip(have, new) if f >= 0) if not status else 0
    if not 0 <= n_free <= n_blocks - back:
        status |= 8
    elif need > n_free + back:
        status |= 1
    if not status & 10 and sum(max(f, 0) for f in new) > cap:
        status |= 4
    slots, positions, cu, lens, top = [], [], [0], [], n_free
    if not status:
        for i, f in enumerate(new):
            if f < 0:
                for b in range(up(have[i])):
                    free[top] = table[i, b]
                    top += 1
        for i, (c, f) in enumerate(zip(have, new)):
            lens.append(0 if f < 0 else c + f)
            for b in range(up(c), up(lens[-1])):
                top -= 1
                table[i, b] = free[top]
            for p in range(c, lens[-1]):
                slots.append(int(table[i, p // block]) * block + p % block)
                positions.append(p)
            cu.append(len(slots))
    else:
        lens, cu = list(have), [0] * (len(have) + 1)
    pad = cap - len(slots)
    return dict(table=table, free=free, n_free_out=np.array([top]), cu=np.array(cu), lens=np.array(lens), slots=np.array(slots + [-1] * pad, np.int64),
                positions=np.array(positions + [0] * pad), status=np.array([status]))
