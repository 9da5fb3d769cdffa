"""The package's operators for several rollouts that share a cache of pages, as cases that can be timed and checked.

A server keeps the keys and values of many videos in one pool of pages. A step of it gives every request the pages for its new tokens,
writes their keys and values into them, and lets the new tokens attend to what their request has so far.

Kinds:

* ``plan``     pages of the new tokens, their slots and boundaries from the requests' lengths, ``pages.plan_pages``
* ``append``   keys and values into their slots, ``pages.append_pages``
* ``prepare``  QK norm and rotation of q and k by positions on several axes, keys and values into their slots, ``pages.prepare_qkv_pages``
* ``attend``   attention of each request's new tokens over its pages, ``pages.paged_attention``

``run`` computes them in elementary torch operations in fp32 where ``own`` is false, and calls the package where it is true.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda:0"

# (sections of the head dimension by axis, how elements pair) as the three models lay them out
_AXES = {
    "cogvideox": dict(dims=(16, 24, 24), pairing="interleaved", base=10000.0),
    "hunyuan": dict(dims=(16, 56, 56), pairing="interleaved", base=256.0),
    "step": dict(dims=(64, 32, 32), pairing="rotate_half", base=10000.0),
}


def listed():
    return [
        # the next token of 8 requests: nothing but latency
        dict(name="plan_token", kind="plan", B=8, new=1, chunk=1, lo=200, hi=9001, page=16, width=640, spare=100),
        # 64 rollouts get their next latent frame of 1350 tokens, some of them more than the pool has left
        dict(name="plan_frames", kind="plan", B=64, new=1350, chunk=1350, lo=1000, hi=57600, page=64, width=1024, spare=1250),
        # keys and values of three prompts in fp16
        dict(name="append_prompt", kind="append", B=3, new=77, chunk=77, Hk=12, D=64, page=16, dtype="fp16"),
        # the HunyuanVideo share of one of 8 ranks
        dict(name="append_hunyuan", kind="append", B=1, new=14882, chunk=14882, Hk=24, D=128, page=64, dtype="bf16"),
        # the next token of 8 rollouts, far into them
        dict(name="prepare_token", kind="prepare", axes="hunyuan", B=8, new=1, chunk=1, H=24, Hk=24, norm="rms", far=200000, page=64,
             dtype="bf16"),
        # the CogVideoX share, two guided samples, LayerNorm
        dict(name="prepare_cogvideox", kind="prepare", axes="cogvideox", B=2, new=2222, chunk=2222, H=48, Hk=48, norm="layer", far=0,
             page=32, dtype="bf16"),
        # a frame of each of four Step-Video rollouts
        dict(name="prepare_step", kind="prepare", axes="step", B=4, new=1802, chunk=1802, H=48, Hk=48, norm="rms", far=300, page=128,
             dtype="bf16"),
        # three short requests in fp16, a few tokens each: a speculative step of a small model
        dict(name="attend_small", kind="attend", B=3, new=4, chunk=4, lo=60, hi=700, H=8, Hk=2, D=64, page=16, left=-1, right=0, frame=1,
             sinks=0, dtype="fp16"),
        # a token of each of 8 rollouts over caches of unequal length
        dict(name="attend_token", kind="attend", B=8, new=1, chunk=1, lo=3000, hi=17776, H=24, Hk=24, D=128, page=64, left=-1, right=0,
             frame=1, sinks=0, dtype="bf16"),
        # single tokens beside a prompt of 2048 tokens that comes in a chunk, shared key heads, causal, in fp16
        dict(name="attend_mixed", kind="attend", B=16, new=1, chunk=2048, lo=500, hi=8191, H=32, Hk=8, D=128, page=16, left=-1, right=0,
             frame=1, sinks=0, dtype="fp16"),
        # CogVideoX's next latent frame of 1350 tokens for two rollouts, behind up to twelve others and 226 text tokens
        dict(name="attend_cogvideox", kind="attend", B=2, new=1350, chunk=1350, lo=9676, hi=17776, H=48, Hk=48, D=64, page=32, left=-1,
             right=0, frame=1350, sinks=226, dtype="bf16"),
        # the next frame of two HunyuanVideo rollouts over the seven frames before, the first frame stays visible
        dict(name="attend_hunyuan", kind="attend", B=2, new=3600, chunk=3600, lo=39600, hi=57600, H=24, Hk=24, D=128, page=128, left=7,
             right=0, frame=3600, sinks=3600, dtype="bf16"),
    ]


_MOST_PAIRS = 5.0e9          # of (query, key, head), heads of 128: below the largest listed case
_MOST_KEYS = 3.0e8           # elements of all requests' keys
_MOST_ROWS = 14882 * 24


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges: tokens and requests over their logarithm, any head count, page size and type."""
    kind = rng.choice(["plan", "plan", "append", "prepare", "prepare", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([16, 16, 32, 48, 64, 64, 128, 144, 256])
    B = _spread(rng, 1, 64)
    if kind == "plan":
        hi = _spread(rng, 10, 57600)
        new = min(_spread(rng, 1, 3000), 86400 // B)
        return dict(kind=kind, B=B, new=new, chunk=rng.choice([new, min(4 * new, 8000)]), lo=rng.randint(0, hi), hi=hi, page=page,
                    width=(hi + 8000) // page + rng.randint(1, 40), spare=rng.randint(1, 2 * B * (new // page + 1)))
    H = rng.choice([1, 2, 3, 4, 6, 8, 10, 12, 16, 20, 24, 30, 32, 40, 48])
    Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0])
    D = rng.choice([64, 128])
    if kind in ("append", "prepare"):
        B = min(B, 16)
        most = _MOST_ROWS // (2 if kind == "prepare" else 1) * 128 // D // (B * H)
        new = max(1, min(_spread(rng, 1, 16000), most))
        if kind == "append":
            return dict(kind=kind, B=B, new=new, chunk=new, Hk=H, D=D, page=page, dtype=dtype)
        axes = rng.choice(["cogvideox"] if D == 64 else ["hunyuan", "step"])
        return dict(kind=kind, axes=axes, B=B, new=new, chunk=new, H=H, Hk=Hk, norm=rng.choice(["rms", "layer", "none"]),
                    far=rng.choice([0, 100, 50000, 1000000]), page=page, dtype=dtype)
    while True:
        B = _spread(rng, 1, 64)
        single = rng.random() < 0.4
        new = rng.randint(1, 8) if single else _spread(rng, 9, 4000)
        chunk = rng.choice([new, _spread(rng, 100, 2500)])
        hi = _spread(rng, 40, 60000)
        lo = rng.randint(min(new, hi), hi)
        frame = 1 if single or chunk != new else rng.choice([1, 1, _spread(rng, 20, 4000)])
        reach = _spread(rng, 1, 8192) if frame == 1 else rng.randint(0, 8)
        case = dict(kind=kind, B=B, new=new, chunk=chunk, lo=lo, hi=hi, H=H, Hk=Hk, D=D, page=page, left=rng.choice([-1, -1, reach]),
                    right=rng.choice([0, 0, 0, -1]), frame=frame, sinks=rng.choice([0, 4, rng.randint(1, 300), frame]), dtype=dtype)
        if max(new, chunk) > hi or case["sinks"] > hi:
            continue
        # (the plain form scores all keys of a request: the whole rectangle has to stay affordable as well)
        square = sum(n * l for n, l in zip(_new(case), _lens(case)))
        if _pairs(case) * D <= _MOST_PAIRS * 128 and square * H <= 1.0e10 and sum(_lens(case)) * Hk * D <= _MOST_KEYS:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _new(c):
    """New tokens of each request: one has ``chunk``, the others ``new``."""
    return [c["chunk"]] + [c["new"]] * (c["B"] - 1)


def _lens(c):
    """Tokens of each request, the new ones among them (``plan``: without them): from ``lo`` to ``hi``, the first one's the most."""
    B = c["B"]
    lens = [int(c["hi"] - (c["hi"] - c["lo"]) * b / max(B - 1, 1)) for b in range(B)]
    return lens if c["kind"] == "plan" else [max(n, l) for n, l in zip(_new(c), lens)]


def _shuffled(c, seed):
    """(lens, new) in an order of the seed's."""
    order = torch.randperm(c["B"], generator=torch.Generator().manual_seed(seed)).tolist()
    lens, new = _lens(c), _new(c)
    return [lens[b] for b in order], [new[b] for b in order]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=_DEV)


def _sums(values):
    res = [0]
    for v in values:
        res.append(res[-1] + v)
    return res


def _tables(lens, page, width, spare, g):
    """(tables, pages): pages of a pool in any order, what stands behind a request's last one is left over from others."""
    held = [-(-l // page) for l in lens]
    n_pages = sum(held) + spare
    ids = torch.randperm(n_pages, generator=g, device=_DEV).to(torch.int32)
    tables = torch.randint(-1, max(n_pages, 1), (len(lens), width), generator=g, device=_DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        tables[b, :n] = ids[at:at + n]
        at += n
    return tables, n_pages


def _slots(case, tables, lens, new):
    """Slots of the new tokens of each request, the last ones of its length."""
    page, res = case["page"], []
    for b, (l, n) in enumerate(zip(lens, new)):
        j = torch.arange(l - n, l, device=_DEV)
        res.append(tables[b, j // page].long() * page + j % page)
    return torch.cat(res)


def _positions(T, far, g):
    """int32 ``[T, 3]``: tokens of frames, row by row, ``far`` frames into a rollout."""
    w = max(1, int(math.sqrt(T / 4 * 45 / 30)))
    h = max(1, T // 4 // w)
    i = torch.arange(T, device=_DEV)
    shift = torch.randint(0, 50, (1,), generator=g, device=_DEV)
    return torch.stack((i // (h * w) + far + shift, i // w % h, i % w), -1).to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    c = case
    st = {"case": c}
    if c["kind"] == "plan":
        lens, new = _shuffled(c, seed)
        st["tables"], st["n_pages"] = _tables(lens, c["page"], c["width"], c["spare"], g)
        st["lens"], st["new"], st["T"] = _ints(lens), _ints(new), sum(new)
        return st
    dtype = _DTYPES[c["dtype"]]
    if c["kind"] == "attend":
        lens, new = _shuffled(c, seed)
        H, Hk, D = c["H"], c["Hk"], c["D"]
        st["tables"], n_pages = _tables(lens, c["page"], -(-c["hi"] // c["page"]) + 3, 5, g)
        unit = lambda x: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        st["q"] = (1.5 * unit(torch.randn(sum(new), H, D, generator=g, device=_DEV))).to(dtype)
        st["k_pages"] = (1.5 * unit(torch.randn(n_pages, c["page"], Hk, D, generator=g, device=_DEV))).to(dtype)
        st["v_pages"] = torch.randn(n_pages, c["page"], Hk, D, generator=g, device=_DEV).to(dtype)
        st["lens"], st["cu"] = _ints(lens), _ints(_sums(new))
        st["host"] = (lens, new)          # what the scheduler of a server knows
        return st
    new = _new(c)
    T, Hk = sum(new), c["Hk"]
    H, D = c.get("H", 0), c["D"] if c["kind"] == "append" else sum(_AXES[c["axes"]]["dims"])
    ends = [n + int(c["page"] * 1.5) for n in new]                        # the cache already holds a page and a half of each request
    tables, n_pages = _tables(ends, c["page"], -(-max(ends) // c["page"]) + 1, 3, g)
    st["slots"] = _slots(c, tables, ends, new)
    st["k_pages"] = torch.randn(n_pages, c["page"], Hk, D, generator=g, device=_DEV).to(dtype)
    st["v_pages"] = torch.randn(n_pages, c["page"], Hk, D, generator=g, device=_DEV).to(dtype)
    # q, k and v lie side by side in the output of a fused projection
    qkv = (torch.randn(T, H + 2 * Hk, D, generator=g, device=_DEV) * 1.5).to(dtype)
    st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    if c["kind"] == "prepare":
        st["positions"] = _positions(T, c["far"], g)
        st["weights"] = [(torch.rand(D, generator=g, device=_DEV) + 0.5).to(dtype) for _ in range(2)]
        st["biases"] = [(torch.randn(D, generator=g, device=_DEV) * 0.1).to(dtype) for _ in range(2)]
        if own:
            from ditango_amd.producer import RotaryAxes
            st["axes"] = RotaryAxes(**_AXES[c["axes"]])
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)[st["case"]["kind"]](st)


def _none(x):
    return None if x < 0 else x


def _own_plan(st):
    from ditango_amd.pages import plan_pages
    c = st["case"]
    plan = plan_pages(st["tables"], st["lens"], st["new"], st["T"], n_pages=st["n_pages"], page_size=c["page"])
    return st["tables"], plan.lens, plan.cu_seqlens, plan.slots, plan.served


def _own_append(st):
    from ditango_amd.pages import append_pages
    append_pages(st["k"], st["v"], st["k_pages"], st["v_pages"], st["slots"])
    return st["k_pages"], st["v_pages"]


def _own_prepare(st):
    from ditango_amd.pages import prepare_qkv_pages
    norm = {"rms": "rms", "layer": "layer_norm", "none": None}[st["case"]["norm"]]
    weights = st["weights"] if norm else (None, None)
    biases = st["biases"] if norm == "layer_norm" else (None, None)
    q = prepare_qkv_pages(st["q"], st["k"], st["v"], st["positions"], st["axes"], st["k_pages"], st["v_pages"], st["slots"], norm=norm,
                          q_weight=weights[0], k_weight=weights[1], q_bias=biases[0], k_bias=biases[1], eps=1e-6)
    return q, st["k_pages"], st["v_pages"]


def _own_attend(st):
    from ditango_amd.pages import paged_attention
    c = st["case"]
    return paged_attention(st["q"], st["k_pages"], st["v_pages"], st["tables"], st["lens"], st["cu"], max_seqlen_q=max(c["new"], c["chunk"]),
                           left=_none(c["left"]), right=_none(c["right"]), frame=c["frame"], sinks=c["sinks"])


def _plain_plan(st):
    page, n_pages, T, tables = st["case"]["page"], st["n_pages"], st["T"], st["tables"]
    B, P = tables.shape
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=_DEV), st["new"].clamp(min=0).long().cumsum(0).clamp(max=T)))
    n = cu[1:] - cu[:-1]
    length = st["lens"].long().clamp(min=0, max=P * page)
    held = (length + page - 1) // page
    need = (length + n + page - 1) // page - held
    fits = length + n <= P * page
    # pages that no request holds, the lowest first
    entry = torch.arange(P, device=_DEV)
    taken = torch.zeros(n_pages + 1, dtype=torch.bool, device=_DEV)
    valid = (entry < held[:, None]) & (tables >= 0) & (tables < n_pages)
    taken[torch.where(valid, tables, n_pages).long()] = True
    free = ~taken[:n_pages]
    rank = free.long().cumsum(0)
    ids = torch.zeros(n_pages + 1, dtype=torch.int32, device=_DEV)
    ids[torch.where(free, rank - 1, n_pages)] = torch.arange(n_pages, dtype=torch.int32, device=_DEV)
    want = need * fits
    start = want.cumsum(0) - want
    served = fits & ((need == 0) | (start + need <= rank[-1]))
    fresh = served[:, None] & (entry >= held[:, None]) & (entry < (held + need)[:, None])
    tables.copy_(torch.where(fresh, ids[(start[:, None] + entry - held[:, None]).clamp(min=0, max=n_pages)], tables))
    row = torch.arange(T, device=_DEV)
    b = torch.searchsorted(cu[1:], row, right=True).clamp(max=B - 1)
    j = length[b] + row - cu[b]
    at = tables[b, (j // page).clamp(max=P - 1)].long()
    ok = served[b] & (row < cu[-1]) & (at >= 0) & (at < n_pages)
    slots = torch.where(ok, at * page + j % page, torch.full_like(at, -1))
    return tables, torch.where(served, length + n, length).to(torch.int32), cu.to(torch.int32), slots, served


def _plain_append(st):
    for x, pages in ((st["k"], st["k_pages"]), (st["v"], st["v_pages"])):
        pages.view(-1, *pages.shape[2:])[st["slots"]] = x
    return st["k_pages"], st["v_pages"]


def _normed(x, norm, weight, bias, eps=1e-6):
    if norm == "none":
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return x + bias if norm == "layer" else x


def _plain_prepare(st):
    c = st["case"]
    spec = _AXES[c["axes"]]
    cos, sin = [], []
    for axis, d in enumerate(spec["dims"]):
        freq = spec["base"] ** (-torch.arange(0, d, 2, dtype=torch.float64, device=_DEV) / d)
        angle = st["positions"][..., axis].double()[..., None] * freq       # (a far position times a frequency needs 64 bits)
        cos.append(angle.cos().float()[:, None])
        sin.append(angle.sin().float()[:, None])
    res = []
    for x, w, b in zip((st["q"], st["k"]), st["weights"], st["biases"]):
        x32 = _normed(x.float(), c["norm"], w.float(), b.float())
        y = torch.empty_like(x32)
        lo = 0
        for d, co, si in zip(spec["dims"], cos, sin):
            part, dst = x32[..., lo:lo + d], y[..., lo:lo + d]
            if spec["pairing"] == "interleaved":
                a, bb = part[..., 0::2], part[..., 1::2]
                dst[..., 0::2] = a * co - bb * si
                dst[..., 1::2] = bb * co + a * si
            else:
                a, bb = part[..., :d // 2], part[..., d // 2:]
                dst[..., :d // 2] = a * co - bb * si
                dst[..., d // 2:] = bb * co + a * si
            lo += d
        res.append(y.to(x.dtype))
    st["k_pages"].view(-1, *st["k_pages"].shape[2:])[st["slots"]] = res[1]
    st["v_pages"].view(-1, *st["v_pages"].shape[2:])[st["slots"]] = st["v"]
    return res[0], st["k_pages"], st["v_pages"]


def _bounds(c, pos):
    """(lo, hi): the keys [lo, hi) a query at ``pos`` sees, before the first ``sinks`` keys are added and the length is applied."""
    start = c["sinks"] + torch.div(pos - c["sinks"], c["frame"], rounding_mode="floor") * c["frame"]
    lo = torch.full_like(pos, -2 ** 40) if c["left"] < 0 else start - c["left"] * c["frame"]
    hi = torch.full_like(pos, 2 ** 40) if c["right"] < 0 else start + (c["right"] + 1) * c["frame"]
    return lo, hi


def _plain_attend(st):
    c = st["case"]
    q = st["q"]
    T, H, D = q.shape
    Hk = c["Hk"]
    G = H // Hk
    out = torch.empty_like(q)
    lse = torch.empty(H, T, dtype=torch.float32, device=_DEV)
    t0 = 0
    for b, (length, n) in enumerate(zip(*st["host"])):
        ids = st["tables"][b, :-(-length // c["page"])].long()
        kt = st["k_pages"][ids].flatten(0, 1)[:length].float().permute(1, 2, 0).contiguous()     # [Hk, D, len]
        vt = st["v_pages"][ids].flatten(0, 1)[:length].float().transpose(0, 1).contiguous()      # [Hk, len, D]
        keys = torch.arange(length, device=_DEV)
        rows = max(1, min(1024, int(4.0e8 / (H * length))))
        for s0 in range(0, n, rows):
            s1 = min(n, s0 + rows)
            m = s1 - s0
            lo, hi = _bounds(c, length - n + torch.arange(s0, s1, device=_DEV))
            seen = (keys < hi[:, None]) & ((keys < c["sinks"]) | (keys >= lo[:, None]))
            qb = q[t0 + s0:t0 + s1].float().view(m, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * m, D)
            x = torch.bmm(qb, kt).view(Hk, G, m, length) * D ** -0.5
            x = x.masked_fill_(~seen, -math.inf)
            top = x.amax(-1, keepdim=True)
            top = torch.where(top > -math.inf, top, torch.zeros_like(top))
            p = x.sub_(top).exp_()
            den = p.sum(-1, keepdim=True)
            o = torch.bmm(p.view(Hk, G * m, length), vt).view(Hk, G, m, D) / torch.where(den > 0, den, torch.ones_like(den))
            out[t0 + s0:t0 + s1] = o.permute(2, 0, 1, 3).reshape(m, H, D).to(q.dtype)
            lse[:, t0 + s0:t0 + s1] = (top + den.log()).reshape(H, m)
        t0 += n
    return out, lse


_run_own = {"plan": _own_plan, "append": _own_append, "prepare": _own_prepare, "attend": _own_attend}
_run_plain = {"plan": _plain_plan, "append": _plain_append, "prepare": _plain_prepare, "attend": _plain_attend}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _extent(c, length, n):
    """Per new token of a request, (sinks in front of its window, its window's keys [lo, hi))."""
    lo, hi = _bounds(c, length - n + torch.arange(n, dtype=torch.int64))
    hi = hi.clamp(min=0, max=length)
    lo = torch.minimum(lo.clamp(min=0), hi)
    return torch.minimum(torch.full_like(lo, c["sinks"]), lo), lo, hi


def _pairs(c):
    total = 0
    for length, n in set(zip(_lens(c), _new(c))):
        first, lo, hi = _extent(c, length, n)
        total += int((first + hi - lo).sum()) * sum((l, m) == (length, n) for l, m in zip(_lens(c), _new(c)))
    return total * c["H"]


def work(case):
    c = case
    if c["kind"] == "plan":
        T = sum(_new(c))
        held = sum(-(-l // c["page"]) for l in _lens(c))
        # lengths in and out, boundaries, a request's pages in and the new ones out, slots
        return {"bytes": 17 * c["B"] + 4 * held + 4 * (T // c["page"]) + 8 * T, "flops": held + T}
    T = sum(_new(c))
    if c["kind"] == "append":
        return {"bytes": T * (8 * c["Hk"] * c["D"] + 8), "flops": 0}
    if c["kind"] == "prepare":
        D = sum(_AXES[c["axes"]]["dims"])
        rows = T * (c["H"] + c["Hk"])
        return {"bytes": (rows + T * c["Hk"]) * D * 4 + T * 20, "flops": rows * D * (3 if c["norm"] == "none" else 8)}
    keys = 0
    for length, n in zip(_lens(c), _new(c)):
        first, lo, hi = _extent(c, length, n)
        # keys that some row sees: the windows of a run of rows follow each other without a hole
        keys += max(0, int(hi.max()) - int(lo.min())) + min(int(first.max()), int(lo.min()))
    return {"bytes": keys * c["Hk"] * c["D"] * 4 + T * c["H"] * (4 * c["D"] + 4), "flops": 4 * c["D"] * _pairs(c)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "prepare": _exact_prepare, "attend": _exact_attend}[case["kind"]](st)


def _exact_plan(st):
    """Request by request, page by page."""
    page, n_pages, T = st["case"]["page"], st["n_pages"], st["T"]
    tables, lens, new = (st[x].tolist() for x in ("tables", "lens", "new"))
    width = len(tables[0])
    lens = [min(max(l, 0), width * page) for l in lens]
    held = [-(-l // page) for l in lens]
    taken = {p for row, h in zip(tables, held) for p in row[:h]}
    free = [p for p in range(n_pages) if p not in taken]
    given, cu, slots, served = 0, [0], [-1] * T, []
    for b, n in enumerate(new):
        n = max(0, min(n, T - cu[b]))
        cu.append(cu[b] + n)
        need = -(-(lens[b] + n) // page) - held[b]
        fits = lens[b] + n <= width * page
        if fits:
            given += need
        served.append(fits and (need == 0 or given <= len(free)))
        if not served[b]:
            continue
        tables[b][held[b]:held[b] + need] = free[given - need:given]
        for i in range(n):
            p = tables[b][(lens[b] + i) // page]
            if 0 <= p < n_pages:
                slots[cu[b] + i] = p * page + (lens[b] + i) % page
        lens[b] += n
    return _ints(tables), _ints(lens), _ints(cu), _ints(slots, torch.int64), _ints(served, torch.bool)


def _exact_written(pages, slots, x):
    """The pages once row i of x is in slot i."""
    page = pages.shape[1]
    res = pages.double().clone()
    res[slots // page, slots % page] = x.double()
    return res


def _exact_append(st):
    return _exact_written(st["k_pages"], st["slots"], st["k"]), _exact_written(st["v_pages"], st["slots"], st["v"])


def _exact_prepare(st):
    c = st["case"]
    spec = _AXES[c["axes"]]
    pos = st["positions"].double()
    turned = []
    for axis, d in enumerate(spec["dims"]):
        i = torch.arange(d // 2, dtype=torch.float64, device=_DEV)
        angle = pos[..., axis, None] * torch.exp(-math.log(spec["base"]) * 2 * i / d)
        turned.append(torch.polar(torch.ones_like(angle), angle))
    res = []
    for x, w, b in zip((st["q"], st["k"]), st["weights"], st["biases"]):
        x = x.double()
        if c["norm"] == "layer":
            x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt() * w.double() + b.double()
        elif c["norm"] == "rms":
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        parts = []
        for part, t in zip(x.split(spec["dims"], -1), turned):
            d = part.shape[-1]
            z = part.unflatten(-1, (d // 2, 2)) if spec["pairing"] == "interleaved" else part.unflatten(-1, (2, d // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * t[:, None])
            parts.append((z if spec["pairing"] == "interleaved" else z.transpose(-1, -2)).flatten(-2))
        res.append(torch.cat(parts, -1))
    return res[0], _exact_written(st["k_pages"], st["slots"], res[1]), _exact_written(st["v_pages"], st["slots"], st["v"])


def _exact_attend(st):
    c = st["case"]
    q = st["q"].double()
    T, H, D = q.shape
    G = H // c["Hk"]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=_DEV)
    lse = torch.full((H, T), -math.inf, dtype=torch.float64, device=_DEV)
    t0 = 0
    for b, (length, n) in enumerate(zip(*st["host"])):
        j = torch.arange(length, device=_DEV)
        page, at = st["tables"][b][j // c["page"]].long(), j % c["page"]
        for s0 in range(0, n, 2048):
            s1 = min(n, s0 + 2048)
            p = (length - n + torch.arange(s0, s1, device=_DEV))[:, None]
            f, key_frame = (p - c["sinks"]) // c["frame"], (j - c["sinks"]) // c["frame"]
            see = torch.ones(p.shape[0], length, dtype=torch.bool, device=_DEV)
            if c["right"] >= 0:
                see &= key_frame <= f + c["right"]
            if c["left"] >= 0:
                see &= (j < c["sinks"]) | (key_frame >= f - c["left"])
            used = see.any(0).nonzero()[:, 0]
            if used.numel() == 0:
                continue
            mask = torch.zeros(see.shape, dtype=torch.float64, device=_DEV).masked_fill(~see, -math.inf)[:, used]
            for h in range(H):
                k = st["k_pages"][page[used], at[used], h // G].double()
                v = st["v_pages"][page[used], at[used], h // G].double()
                x = q[t0 + s0:t0 + s1, h] @ k.T / math.sqrt(D) + mask
                l = torch.logsumexp(x, -1)
                w = torch.exp(x - torch.where(l > -math.inf, l, torch.zeros_like(l))[:, None])
                out[t0 + s0:t0 + s1, h] = w @ v
                lse[h, t0 + s0:t0 + s1] = l
        t0 += n
    return out, lse
