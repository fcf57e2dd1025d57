"""The token stage's operators in 64 bits, one request / page / row at a time (include/pigeon_hip.h states them)."""
import math

import numpy as np
import torch

SCALE_FLOOR = -100


def page_advance_ref(lens, keep, add, table, free, count, P, T):
    """Lists in, lists out: (lens, table, free, count, slots, starts, status); `free` is the whole array of the stack."""
    R, W = len(lens), len(table[0])
    lens = [min(max(h, 0), W * P) for h in lens]
    keep = list(lens) if keep is None else [min(max(k, 0), h) for k, h in zip(keep, lens)]
    add = [max(a, 0) for a in add]
    table, free = [list(r) for r in table], list(free)
    pages = lambda n: -(-n // P)                                   # noqa: E731
    back = [table[r][j] for r in range(R) for j in range(pages(keep[r]), pages(lens[r]))]
    for e, page in enumerate(reversed(back)):
        free[count + e] = page
    top = count + len(back)
    slots, starts, status, end, wanted, avail = [-1] * T, [0], [], 0, 0, top
    for r in range(R):
        begin, end = end, end + add[r]
        starts.append(min(end, T))
        fits = keep[r] + add[r] <= W * P and end <= T
        want = pages(keep[r] + add[r]) - pages(keep[r]) if fits else 0
        wanted += want
        ok = fits and (want == 0 or wanted <= avail)
        status.append(0 if ok else 1)
        lens[r] = keep[r]
        if ok:
            for j in range(want):
                top -= 1
                table[r][pages(keep[r]) + j] = free[top]
            lens[r] += add[r]
            for i in range(add[r]):
                pos = keep[r] + i
                slots[begin + i] = table[r][pos // P] * P + pos % P
    return lens, table, free, top, slots, starts, status


def e4m3_round(x):
    """Nearest e4m3 value, ties to even, of finite magnitudes up to 448 (their overflow is not this function's)."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        step = np.ldexp(1.0, np.maximum(np.frexp(np.where(np.isfinite(x), x, 0.0))[1] - 1, -6) - 3)
        return np.rint(x / step) * step


def page_scale(amax):
    k = SCALE_FLOOR
    while amax > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def cache_write_ref(x, slots, pages, scale):
    """x [T, H, D], slots [T], pages [N, H, P, D] of byte values, scale [N, H]: float64 arrays -> new (pages, scale).
    Values are passed as keys are laid out; the transposition is the caller's."""
    x, pages, scale = np.asarray(x, np.float64), pages.copy(), scale.copy()
    P, t, T = pages.shape[2], 0, len(slots)
    while t < T:
        page, row = divmod(int(slots[t]), P)
        n = 1
        while t + n < T and row + n < P and slots[t + n] == slots[t] + n:
            n += 1
        if 0 <= page < len(pages):
            for h in range(x.shape[1]):
                new = x[t:t + n, h]
                s = page_scale(np.max(np.abs(new), where=np.isfinite(new), initial=0.0))
                if row > 0:
                    s = max(s, scale[page, h])
                    if scale[page, h] < s:
                        pages[page, h, :row] = e4m3_round(pages[page, h, :row] * (scale[page, h] / s))
                pages[page, h, row:row + n] = np.where(np.isfinite(new), e4m3_round(new / s), np.nan)
                scale[page, h] = s
        t += n
    return pages, scale


def cached_attention_ref(q, k_pages, v_pages, k_scale, v_scale, table, lens, starts=None, scale=None, causal=True,
                         window=0):
    """float64 result [T, Hq, D] (NaN in rows of no request), and per output the two magnitudes that error bounds need:
    sum_j p_j |v_j| and max_j |scale| * sum_d |q_d k_jd|."""
    q = q.double().cpu()
    T, Hq, D = q.shape
    N, H, P, _ = k_pages.shape
    kb, vb = k_pages.cpu().float().double(), v_pages.cpu().float().double().transpose(2, 3)
    ks, vs = k_scale.double().cpu(), v_scale.double().cpu()
    table, lens = table.cpu().tolist(), lens.cpu().tolist()
    starts = list(range(len(lens) + 1)) if starts is None else starts.cpu().tolist()
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    mag = torch.zeros(T, Hq, D, dtype=torch.float64)
    big = torch.zeros(T, Hq, 1, dtype=torch.float64)
    W = len(table[0])
    for r, L in enumerate(lens):
        L = min(max(L, 0), W * P)
        n = starts[r + 1] - starts[r]
        keys = [(table[r][p // P], p % P) for p in range(L)]
        good = torch.tensor([0 <= pg < N for pg, _ in keys], dtype=torch.bool)
        pg = torch.tensor([pg if 0 <= pg < N else 0 for pg, _ in keys], dtype=torch.long)
        rw = torch.tensor([w for _, w in keys], dtype=torch.long)
        for i in range(n):
            pos, t = L - n + i, starts[r] + i
            see = good.clone()
            j = torch.arange(L)
            if causal:
                see &= j <= pos
            if window:
                see &= j > pos - window
            if not bool(see.any()):
                out[t] = 0.0
                continue
            for h in range(Hq):
                kh = h // (Hq // H)
                k = kb[pg[see], kh, rw[see]] * ks[pg[see], kh, None]
                v = vb[pg[see], kh, rw[see]] * vs[pg[see], kh, None]
                x = (k @ q[t, h]) * scale
                p = torch.softmax(x, 0)
                out[t, h] = p @ v
                mag[t, h] = p @ v.abs()
                big[t, h] = ((k.abs() @ q[t, h].abs()) * abs(scale)).max()
    return out, mag, big


def sample_tokens_ref(logits, u, temperature, top_k, top_p, min_p):
    """One row: float64 logits, numbers -> id."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    m = x.max()
    if m == -np.inf:
        return -1
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not temperature > 0 or top_p <= 0:
        return int(order[0])
    if top_k > 0:
        order = order[:top_k]
    if m == np.inf:
        w = (x[order] == np.inf).astype(np.float64)
    else:
        w = np.exp((x[order] - m) / np.float64(temperature))
    if top_p < 1:
        c = np.cumsum(w)
        n = int(np.searchsorted(c, np.float64(top_p) * c[-1], side="left")) + 1
        order, w = order[:n], w[:n]
    kept = (w >= min_p) | (x[order] == m)
    order, w = order[kept], w[kept]
    by = np.argsort(order)
    order, c = order[by], np.cumsum(w[by])
    i = int(np.searchsorted(c, np.float64(u) * c[-1], side="right"))
    return int(order[min(i, np.flatnonzero(w[by] > 0)[-1])])
