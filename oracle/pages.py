"""A cache of pages that several requests share, from its definitions: which page holds what, request by request, and attention over the pages in
float64.  Test infrastructure; nothing here comes from the package."""
import math

import torch

from . import long_video as L


def plan(tables, lens, new_lens, n_tokens, n_pages, page):
    """Lists of whole numbers in, (tables, lens, cu_seqlens, slots, served) out."""
    tables = [list(row) for row in tables]
    width = len(tables[0]) if tables else 0
    lens = [min(max(n, 0), width * page) for n in lens]
    held = [math.ceil(n / page) for n in lens]
    taken = {p for row, h in zip(tables, held) for p in row[:h]}
    free = [p for p in range(n_pages) if p not in taken]
    asked, cu, slots, served = 0, [0], [-1] * n_tokens, []
    for b, n in enumerate(new_lens):
        n = min(max(n, 0), n_tokens - cu[b])
        cu.append(cu[b] + n)
        need = math.ceil((lens[b] + n) / page) - held[b]
        fits = lens[b] + n <= width * page
        first = asked
        asked += need if fits else 0
        served.append(fits and (need == 0 or asked <= len(free)))
        if not served[b]:
            continue
        tables[b][held[b]:held[b] + need] = free[first:first + need]
        for i in range(n):
            j = lens[b] + i
            if 0 <= tables[b][j // page] < n_pages:
                slots[cu[b] + i] = tables[b][j // page] * page + j % page
        lens[b] += n
    return tables, lens, cu, slots, served


def gathered(pages, table, length):
    """``[length, Hk, D]``: a request's rows of the pages ``[pages, page, Hk, D]``; zeros where an entry is no page."""
    page = pages.shape[1]
    out = torch.zeros(length, *pages.shape[2:], dtype=pages.dtype, device=pages.device)
    for i in range(math.ceil(length / page)):
        p = int(table[i])
        if 0 <= p < pages.shape[0]:
            n = min(page, length - i * page)
            out[i * page:i * page + n] = pages[p, :n]
    return out


def attention(q, k_pages, v_pages, tables, lens, cu, **window):
    """(out, lse, sum of weights times |v|, largest sum |q_i k_i| scale) in float64; rows of no request get 0 and -inf."""
    T, H, D = q.shape
    out, weight = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((H, T), -math.inf, dtype=torch.float64, device=q.device)
    top = 0.0
    for b in range(len(tables)):
        lo, hi = (min(max(int(cu[b + i]), 0), T) for i in range(2))
        n = hi - lo
        length = min(max(int(lens[b]), 0), len(tables[b]) * k_pages.shape[1])
        if n <= 0:
            continue
        k, v = (gathered(x, tables[b], length)[None] for x in (k_pages, v_pages))
        o, l, w, t = L.window_attention(q[None, lo:hi], k, v, q_begin=length - n, **window)
        out[lo:hi], lse[:, lo:hi], weight[lo:hi], top = o[0], l[0], w[0], max(top, t)
    return out, lse, weight, top
