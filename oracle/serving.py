"""Tables of a step and sampling, restated one request and one row at a time."""
from __future__ import annotations

import numpy as np


def step_tables(past, new, table, free, count, page_size, num_rows):
    """build_step_tables on the host.  table [B][max_pages], free: list as long as the stack's
    capacity; both are copied.  Returns a dict of lists."""
    table = [list(r) for r in table]
    free = list(free)
    maxp = len(table[0])
    pages = lambda n: -(-n // page_size)  # noqa: E731
    past = [max(0, p) for p in past]
    refused = False
    for b, n in enumerate(new):
        if n < 0:
            for i in range(min(pages(past[b]), maxp)):
                if count < len(free):
                    free[count] = table[b][i]
                else:
                    refused = True
                count += 1
    left, asked = count, 0  # pages on the stack; pages asked for so far
    kv, granted = [], []
    for b, n in enumerate(new):
        if n < 0:
            kv.append(0)
            granted.append(False)
            continue
        held, need = pages(past[b]), pages(past[b] + n)
        want = need - held if need <= maxp else 0
        ok = need <= maxp and (want == 0 or asked + want <= count)
        asked += want
        if ok:
            for i in range(want):
                left -= 1
                table[b][held + i] = free[left]
        else:
            refused = True
        granted.append(ok)
        kv.append(past[b] + n if ok else past[b])
    cu, seq, pos, rows = [0], [], [], []
    for b, n in enumerate(new):
        for j in range(max(n, 0)):
            p = past[b] + j
            seq.append(b)
            pos.append(p)
            rows.append(table[b][p // page_size] * page_size + p % page_size if granted[b] else -1)
        cu.append(len(rows))
    pad = num_rows - len(rows)
    return dict(kv_lens=kv, cu_tokens=cu, seq_ids=(seq + [-1] * pad)[:num_rows],
                positions=(pos + [0] * pad)[:num_rows], slot_rows=(rows + [-1] * pad)[:num_rows],
                page_table=table, free_pages=free, free_count=left, refused=refused)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, log probability), float64."""
    l = np.array(logits, dtype=np.float64)
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return -1, -np.inf
    t = float(temperature) if temperature > 0 else 1.0
    with np.errstate(invalid="ignore"):
        z = np.where(l == top, 0.0, (l - top) / t)
    w = np.exp(z)
    order = np.lexsort((np.arange(len(l)), -l))
    if not temperature > 0:
        token = int(order[0])
    else:
        if 0 < top_k < len(l):
            order = order[:top_k]
        if top_p < 1:
            c = np.concatenate([[0.0], np.cumsum(w[order])])
            n = max(1, int((c[:-1] < np.float64(top_p) * c[-1]).sum()))
            order = order[:n]
        order = np.array([i for i in order if w[i] >= min_p or l[i] == top])
        kept = np.zeros_like(w)
        kept[order] = w[order]
        c = np.cumsum(kept)
        token = int(min((c <= np.float64(u) * c[-1]).sum(), order.max()))
    return token, z[token] - np.log(w.sum())
