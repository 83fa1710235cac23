"""Plain 64-bit restatements of the paged-cache operators for the tests, one request and one token at a time."""
import numpy as np

NONE = 0xFFFFFFFF


def round_bf16(x):
    """Round to nearest even on the integer bits (finite values)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) & np.uint32(0xFFFF0000)).view(np.float32)


def plan(cached, new, free, head, tables, page, capacity, parents=None, words=0):
    """(starts, slots, positions, masks, head) and the tables, as ojc_paged_plan defines them for valid inputs."""
    tables = tables.copy()
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    slots, positions = np.full(capacity, NONE, np.int64), np.zeros(capacity, np.int64)
    masks = np.zeros((capacity, words), np.uint32)
    for b, (c, n) in enumerate(zip(cached, new)):
        for p in range(-(-c // page), -(-(c + n) // page)):
            tables[b, p] = free[head]
            head += 1
        for i in range(n):
            t = starts[b] + i
            slots[t] = int(tables[b, (c + i) // page]) * page + (c + i) % page
            chain, at = [], i
            while at != NONE and at >= 0:
                chain.append(at)
                at = at - 1 if parents is None else int(parents[t - i + at])
            positions[t] = c + len(chain) - 1
            if words:
                for a in chain:
                    masks[t, a // 32] |= np.uint32(1 << (a % 32))
    return starts, slots, positions, masks, head, tables


def frequencies(rotary, base=10000.0, scaling="none", factor=1.0, original=0.0, low=1.0, high=32.0):
    i = np.arange(0, rotary, 2, dtype=np.float64)
    if scaling == "base":
        base = base * factor ** (rotary / (rotary - 2))
    f = base ** (-i / rotary)
    if scaling == "linear":
        f = f / factor
    if scaling == "by_turns":
        w = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0, 1)
        f = f * (w + (1 - w) / factor)
    return f


def rotate(x, positions, freqs, layout="half", amplitude=1.0, back=False):
    """x [N, H, D] in 64 bits; positions [N]."""
    y = np.array(x, np.float64)
    r = 2 * len(freqs)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    angle = np.asarray(positions, np.float64)[:, None] * freqs[None]
    z = (y[..., first] + 1j * y[..., second]) * (amplitude * np.exp((-1j if back else 1j) * angle))[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def attention(q, k_pages, v_pages, tables, cached, starts, masks=None, positions=None, window=None, eps_out=0.0, eps_p=0.0):
    """(out, lse, bound on |out error|, bound on |lse error|). The bounds: a score of D products in f32 is off by at most (D + 4) 2^-24 times the sum of
    their magnitudes (times the scale), e_s below; each weight by e_s (relative), the exponential's 2^-20 and eps_p where it is rounded for the second product;
    the sums of L terms by L 2^-24; the result by its own rounding eps_out. The weights' errors enter the result twice, through the numerator
    and the normaliser."""
    q, page = np.asarray(q, np.float64), k_pages.shape[1]
    n, h, d = q.shape
    hk = k_pages.shape[2]
    out, lse = np.zeros((n, h, d)), np.full((n, h), -np.inf)
    tol, lse_tol = np.zeros((n, h, d)), np.zeros((n, h))
    for b in range(len(cached)):
        c, lo, hi = int(cached[b]), int(starts[b]), int(starts[b + 1])
        at = np.arange(c + hi - lo)
        ids = np.asarray(tables[b], np.int64)[at // page] if len(at) else at
        k_all, v_all = k_pages[ids, at % page], v_pages[ids, at % page]
        for t in range(lo, hi):
            i = t - lo
            sees = np.ones(len(at), bool)
            for j in range(hi - lo):
                sees[c + j] = j <= i if masks is None else bool(masks[t, j // 32] >> np.uint32(j % 32) & 1) if j // 32 < masks.shape[1] else False
            if window is not None:
                mine = (c + np.arange(hi - lo)) if positions is None else np.asarray(positions[lo:hi], np.int64)
                sees &= np.concatenate([at[:c], mine]) > mine[i] - window
            if not sees.any():
                continue
            k, v = k_all[sees].astype(np.float64), v_all[sees].astype(np.float64)
            for head in range(h):
                kk, vv = k[:, head // (h // hk)], v[:, head // (h // hk)]
                s = kk @ q[t, head] / np.sqrt(d)
                top = s.max()
                p = np.exp(s - top)
                total = p.sum()
                lse[t, head] = top + np.log(total)
                out[t, head] = p @ vv / total
                e_s = (d + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[t, head])).max() / np.sqrt(d)
                e_w = e_s + 2.0 ** -20 + (len(s) + 8) * 2.0 ** -24
                spread = p @ np.abs(vv) / total
                tol[t, head] = (eps_out + 2.0 ** -22) * np.abs(out[t, head]) + (2 * e_w + eps_p * (1 + 2.0 ** -6)) * spread * (1 + eps_out) + 1e-30
                lse_tol[t, head] = e_w + e_s + 2.0 ** -22 * (1 + abs(lse[t, head]))
    return out, lse, tol, lse_tol
