"""The package's operators for long videos, as cases that can be timed and checked.

A rolled-out video goes through three of them, layer by layer: queries and keys get their norm and their rotation by the token's place
in time, height and width; a query attends to the frames around it and to the first tokens of the sequence; the states that a later
denoising step reuses are kept in 8 bits and merged from there.

Kinds:

* ``rotary``   QK norm and rotation of q and k by positions on several axes, ``producer.prepare_qk_axes``
* ``window``   attention in a window of tokens or frames, with first keys that stay visible, ``window.window_attention``
* ``store``    a state into the 8-bit cache and back out as 16-bit values, ``proCache.store_block`` / ``load_block``
* ``merge``    the merge of cached 8-bit states and fresh 16-bit ones, ``core.cache.merge_any``

``run`` computes them in elementary torch operations in fp32 where ``own`` is false, and calls the package where it is true.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
_DEV = "cuda:0"
_PEAK = {"e4m3": 448.0, "int8": 127.0}          # largest element of an 8-bit block format
_BLOCK = 32

# (sections of the head dimension by axis, how elements pair) as the three models lay them out
_AXES = {
    "cogvideox": dict(dims=(16, 24, 24), pairing="interleaved", base=10000.0),
    "hunyuan": dict(dims=(16, 56, 56), pairing="interleaved", base=256.0),
    "step": dict(dims=(64, 32, 32), pairing="rotate_half", base=10000.0),
    "step64": dict(dims=(32, 16, 16), pairing="rotate_half", base=10000.0),
}


def listed():
    return [
        # a rollout's next token of 8 samples: nothing but latency
        dict(name="rotary_token", kind="rotary", axes="hunyuan", B=8, S=1, H=24, Hk=24, norm="rms", far=200000, dtype="bf16"),
        # the CogVideoX share of one of 8 ranks, two guided samples, LayerNorm, 226 text tokens at the origin
        dict(name="rotary_cogvideox", kind="rotary", axes="cogvideox", B=2, S=2222, H=48, Hk=48, norm="layer", far=0, dtype="bf16"),
        # the HunyuanVideo share
        dict(name="rotary_hunyuan", kind="rotary", axes="hunyuan", B=1, S=14882, H=24, Hk=24, norm="rms", far=0, dtype="bf16"),
        # single tokens against caches of unequal length, a causal window of 4096 tokens and 64 sinks; the lengths live on the GPU
        dict(name="window_token", kind="window", B=4, Sq=1, Sk=9001, H=24, Hk=24, D=128, left=4095, right=0, frame=1, sinks=64,
             begin=-1, ragged=True, dtype="bf16"),
        # a preview in fp16: a token window to both sides, odd sizes
        dict(name="window_preview", kind="window", B=2, Sq=1001, Sk=1001, H=12, Hk=12, D=64, left=200, right=131, frame=1, sinks=5,
             begin=0, ragged=False, dtype="fp16"),
        # CogVideoX's 13 latent frames of 1350 tokens behind 226 text tokens that stay visible: two frames to each side, all video
        # queries of one sample
        dict(name="window_cogvideox", kind="window", B=1, Sq=17550, Sk=17776, H=48, Hk=48, D=64, left=2, right=2, frame=1350,
             sinks=226, begin=226, ragged=False, dtype="bf16"),
        # shared key heads, causal, a window of 2500 tokens: a prompt of a language model's size in fp16
        dict(name="window_shared", kind="window", B=2, Sq=5003, Sk=5003, H=32, Hk=8, D=128, left=2499, right=0, frame=1, sinks=4,
             begin=0, ragged=False, dtype="fp16"),
        # the newest four frames of a HunyuanVideo rollout over the seven frames before, the first frame stays visible
        dict(name="window_rollout", kind="window", B=1, Sq=14400, Sk=57600, H=24, Hk=24, D=128, left=7, right=0, frame=3600,
             sinks=3600, begin=43200, ragged=False, dtype="bf16"),
        # a small problem's state, kept and read back
        dict(name="store_small", kind="store", B=1, Sq=512, H=4, D=64, format="e4m3", dtype="f32"),
        # the HunyuanVideo share's
        dict(name="store_hunyuan", kind="store", B=1, Sq=14882, H=24, D=128, format="int8", dtype="bf16"),
        # a layer call's merge at the CogVideoX share: three fresh states, five cached ones
        dict(name="merge_cogvideox", kind="merge", B=1, Sq=2222, H=48, D=64, cached=5, fresh=3, format="e4m3", dtype="bf16",
             out="bf16"),
        # ... and at the HunyuanVideo share, in int8, into the fp32 result that the layer call returns by default
        dict(name="merge_hunyuan", kind="merge", B=1, Sq=14882, H=24, D=128, cached=6, fresh=2, format="int8", dtype="bf16",
             out="f32"),
    ]


_MOST_PAIRS = 3.4e9          # of (query, key, head): below the largest listed case
_MOST_ROWS = 14882 * 24


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges: tokens over their logarithm, any head count, every format and type."""
    kind = rng.choice(["rotary", "rotary", "window", "window", "window", "store", "merge", "merge"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    H = rng.choice([1, 2, 3, 4, 6, 8, 10, 12, 16, 20, 24, 30, 32, 40, 48])
    B = rng.choice([1, 1, 2, 3])
    if kind == "rotary":
        axes = rng.choice(sorted(_AXES))
        Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0])
        S = max(1, min(_spread(rng, 1, 16000), _MOST_ROWS * (1 if "64" not in axes and axes != "cogvideox" else 2) // (B * H)))
        return dict(kind=kind, axes=axes, B=B, S=S, H=H, Hk=Hk, norm=rng.choice(["rms", "layer", "none"]),
                    far=rng.choice([0, 0, 100, 50000, 1000000]), dtype=dtype)
    D = rng.choice([64, 128])
    if kind == "window":
        while True:
            Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0])
            single = rng.random() < 0.35
            Sk = _spread(rng, 40, 60000)
            Sq = rng.randint(1, 8) if single else _spread(rng, 17, 16000)
            frame = 1 if single else rng.choice([1, 1, _spread(rng, 20, 4000)])
            reach = _spread(rng, 1, 8192) if frame == 1 else rng.randint(0, 8)
            left = rng.choice([reach, reach, reach, -1])
            right = rng.choice([0, 0, reach, -1]) if not single else 0
            sinks = rng.choice([0, 4, rng.randint(1, 300), frame])
            if sinks > Sk or Sq > Sk:
                continue
            case = dict(kind=kind, B=B, Sq=Sq, Sk=Sk, H=H, Hk=Hk, D=D, left=left, right=right, frame=frame, sinks=sinks,
                        begin=-1 if single else rng.randint(0, Sk - Sq), ragged=single, dtype=dtype)
            # (the plain form scores all keys of a block of queries: the whole square has to stay affordable as well)
            if _pairs(case) * D <= _MOST_PAIRS * 128 and B * H * Sq * Sk <= 2.4e10 and B * Hk * Sk * D <= 4.0e8:
                return case
    Sq = max(1, min(_spread(rng, 1, 16000), _MOST_ROWS * 128 // D // (B * H)))
    fmt = rng.choice(["e4m3", "int8"])
    if kind == "store":
        return dict(kind=kind, B=B, Sq=Sq, H=H, D=D, format=fmt, dtype=rng.choice(["bf16", "bf16", "f32"]))
    n = rng.randint(1, 8)
    fresh = rng.randint(0, n - 1)
    return dict(kind=kind, B=B, Sq=Sq, H=H, D=D, cached=n - fresh, fresh=fresh, format=fmt, dtype=dtype, out=rng.choice([dtype, "f32"]))


# ---- inputs -------------------------------------------------------------------------------------------------------

def _positions(case, g):
    """int32 ``[B, S, 3]``: text tokens at the origin, then the frames of a clip row by row, ``far`` frames into a rollout."""
    B, S = case["B"], case["S"]
    text = S // 10 if S > 100 else 0
    n = S - text
    w = max(1, int(math.sqrt(n / 13 * 45 / 30)))
    h = max(1, n // 13 // w)
    i = torch.arange(n, device=_DEV)
    grid = torch.stack((i // (h * w) + case["far"], i // w % h, i % w), -1)
    pos = torch.cat((torch.zeros(text, 3, dtype=torch.int64, device=_DEV), grid)).expand(B, S, 3)
    shift = torch.randint(0, 50, (B, 1, 1), generator=g, device=_DEV)      # the samples of a batch are at different frames
    return (pos + shift * torch.tensor([1, 0, 0], device=_DEV)).to(torch.int32).contiguous()


def _state(case, g, dtype):
    """(out, lse) of an attention state: rows of unequal size, a few channels that stand out, a spread of log sums."""
    B, S, H, D = case["B"], case["Sq"], case["H"], case["D"]
    out = torch.randn(B, S, H, D, generator=g, device=_DEV) * torch.exp(0.5 * torch.randn(B, S, H, 1, generator=g, device=_DEV)) * 0.3
    out *= 1.0 + 6.0 * (torch.rand(1, 1, H, D, generator=g, device=_DEV) < 0.02)
    lse = 8.0 + 2.0 * torch.randn(B, H, S, generator=g, device=_DEV)
    return out.to(dtype), lse


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    st = {"case": case}
    dtype = _DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "rotary":
        D = sum(_AXES[case["axes"]]["dims"])
        B, S, H, Hk = case["B"], case["S"], case["H"], case["Hk"]
        # q, k and v lie side by side in the output of a fused projection
        qkv = (torch.randn(B, S, H + 2 * Hk, D, generator=g, device=_DEV) * 1.5).to(dtype)
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        st["positions"] = _positions(case, g)
        st["weights"] = [(torch.rand(D, generator=g, device=_DEV) + 0.5).to(dtype) for _ in range(2)]
        st["biases"] = [(torch.randn(D, generator=g, device=_DEV) * 0.1).to(dtype) for _ in range(2)]
        if own:
            from ditango_amd.producer import RotaryAxes
            st["axes"] = RotaryAxes(**_AXES[case["axes"]])
        return st
    if kind == "window":
        B, Sq, Sk, H, Hk, D = (case[x] for x in ("B", "Sq", "Sk", "H", "Hk", "D"))
        unit = lambda x: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        st["q"] = (1.5 * unit(torch.randn(B, Sq, H, D, generator=g, device=_DEV))).to(dtype)
        st["k"] = (1.5 * unit(torch.randn(B, Sk, Hk, D, generator=g, device=_DEV))).to(dtype)
        st["v"] = torch.randn(B, Sk, Hk, D, generator=g, device=_DEV).to(dtype)
        st["lens"] = None
        if case["ragged"]:
            st["lens"] = torch.randint(max(case["Sq"], Sk // 2), Sk + 1, (B,), generator=g, device=_DEV).to(torch.int32)
        return st
    if kind == "store":
        st["out"], st["lse"] = _state(case, g, dtype)
        if own:
            from ditango_amd.core.cache import proCache
            st["cache"] = proCache(isp_size=8, layer_id=1, state_format=case["format"])
        return st
    st["cached"] = [_quantized(*_state(case, g, torch.float32), case["format"]) for _ in range(case["cached"])]
    st["fresh"] = [_state(case, g, dtype) for _ in range(case["fresh"])]
    if own:
        from ditango_amd.core.cache import BlockState
        st["states"] = [BlockState(*s) for s in st["cached"]] + st["fresh"]
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)[st["case"]["kind"]](st)


def _none(x):
    return None if x < 0 else x


def _own_rotary(st):
    from ditango_amd.producer import prepare_qk_axes
    norm = {"rms": "rms", "layer": "layer_norm", "none": None}[st["case"]["norm"]]
    weights = st["weights"] if norm else (None, None)
    biases = st["biases"] if norm == "layer_norm" else (None, None)
    return prepare_qk_axes(st["q"], st["k"], st["positions"], st["axes"], norm=norm, q_weight=weights[0], k_weight=weights[1],
                           q_bias=biases[0], k_bias=biases[1], eps=1e-6)


def _own_window(st):
    from ditango_amd.window import window_attention
    c = st["case"]
    return window_attention(st["q"], st["k"], st["v"], left=_none(c["left"]), right=_none(c["right"]), frame=c["frame"],
                            sinks=c["sinks"], q_begin=_none(c["begin"]), kv_lens=st["lens"])


def _own_store(st):
    st["cache"].store_block(3, st["out"], st["lse"])
    return st["cache"].load_block(3, torch.bfloat16)


def _own_merge(st):
    from ditango_amd.core.cache import merge_any
    return merge_any(st["states"], dst_dtype=_DTYPES[st["case"]["out"]], dst_lse_bsh=True)


def _normed(x, norm, weight, bias, eps=1e-6):
    if norm == "none":
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return x + bias if norm == "layer" else x


def _plain_rotary(st):
    c = st["case"]
    spec = _AXES[c["axes"]]
    cos, sin = [], []
    for axis, d in enumerate(spec["dims"]):
        freq = spec["base"] ** (-torch.arange(0, d, 2, dtype=torch.float64, device=_DEV) / d)
        angle = st["positions"][..., axis].double()[..., None] * freq       # (a far position times a frequency needs 64 bits)
        cos.append(angle.cos().float()[:, :, None])
        sin.append(angle.sin().float()[:, :, None])
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
    return tuple(res)


def _bounds(c, pos):
    """(lo, hi): the keys [lo, hi) a query at ``pos`` sees, before the first ``sinks`` keys are added and the length is applied."""
    start = c["sinks"] + torch.div(pos - c["sinks"], c["frame"], rounding_mode="floor") * c["frame"]
    lo = torch.full_like(pos, -2 ** 40) if c["left"] < 0 else start - c["left"] * c["frame"]
    hi = torch.full_like(pos, 2 ** 40) if c["right"] < 0 else start + (c["right"] + 1) * c["frame"]
    return lo, hi


def _plain_window(st):
    c = st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    kt = k.float().permute(0, 2, 3, 1).reshape(B * Hk, D, Sk).contiguous()
    vt = v.float().permute(0, 2, 1, 3).reshape(B * Hk, Sk, D).contiguous()
    out = torch.empty(B, Sq, H, D, dtype=q.dtype, device=_DEV)
    lse = torch.empty(B, H, Sq, dtype=torch.float32, device=_DEV)
    rows = max(1, min(1024, int(4.0e8 / (B * H * Sk))))
    keys = torch.arange(Sk, device=_DEV)
    lens = torch.full((B,), Sk, device=_DEV) if st["lens"] is None else st["lens"].long()
    for s0 in range(0, Sq, rows):
        s1 = min(Sq, s0 + rows)
        n = s1 - s0
        row = torch.arange(s0, s1, device=_DEV)
        first = torch.full((B,), c["begin"], device=_DEV) if c["begin"] >= 0 else lens - Sq
        pos = first[:, None] + row                                                        # [B, n]
        lo, hi = _bounds(c, pos)
        seen = (keys < torch.minimum(hi, lens[:, None])[..., None]) & ((keys < c["sinks"]) | (keys >= lo[..., None]))   # [B, n, Sk]
        qb = q[:, s0:s1].float().reshape(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, G * n, D)
        x = torch.bmm(qb, kt).view(B, Hk, G, n, Sk) * D ** -0.5
        x = x.masked_fill_(~seen[:, None, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        m = torch.where(m > -math.inf, m, torch.zeros_like(m))
        p = x.sub_(m).exp_()
        den = p.sum(-1, keepdim=True)
        o = torch.bmm(p.view(B * Hk, G * n, Sk), vt).view(B, Hk, G, n, D) / torch.where(den > 0, den, torch.ones_like(den))
        out[:, s0:s1] = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(q.dtype)
        lse[:, :, s0:s1] = (m + den.log()).reshape(B, H, n)
    return out, lse


def _two_to(e):
    """2^e in fp32, -127 <= e <= 127, exactly (a power function may be off by a step, which moves what lies on a border)."""
    return torch.where(e < -126, 1 << 22, (e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantized(out, lse, fmt):
    """(elements, scales, lse) of a state in 8 bits: blocks of 32 along D, scale byte e + 127 with the smallest e >= -127 for which the
    block's largest magnitude is at most the format's largest element times 2^e."""
    x = out.float().unflatten(-1, (-1, _BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    exp = torch.frexp(amax / _PEAK[fmt])[1].clamp(min=-126)
    e = torch.where(amax <= _PEAK[fmt] * _two_to(exp - 1), exp - 1, exp)
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    y = x * _two_to(-e)
    elements = y.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(y).to(torch.int8)
    return elements.flatten(-2), (e + 127).to(torch.uint8).squeeze(-1), lse


def _value(elements, scales):
    x = elements.float().unflatten(-1, (-1, _BLOCK))
    return (x * _two_to(scales.to(torch.int32).unsqueeze(-1) - 127)).flatten(-2)


def _plain_store(st):
    elements, scales, lse = _quantized(st["out"], st["lse"], st["case"]["format"])
    return _value(elements, scales).to(torch.bfloat16), lse.transpose(1, 2).unsqueeze(-1).contiguous()


def _plain_merge(st):
    c = st["case"]
    states = [(_value(e, s), l) for e, s, l in st["cached"]] + [(o.float(), l) for o, l in st["fresh"]]
    m = states[0][1]
    for _, l in states[1:]:
        m = torch.maximum(m, l)
    den, acc = torch.zeros_like(m), None
    for o, l in states:
        w = (l - m).exp()
        den = den + w
        part = o * w.transpose(1, 2).unsqueeze(-1)
        acc = part if acc is None else acc + part
    out = acc / den.transpose(1, 2).unsqueeze(-1)
    return out.to(_DTYPES[c["out"]]), (m + den.log()).transpose(1, 2).unsqueeze(-1).contiguous()


_run_own = {"rotary": _own_rotary, "window": _own_window, "store": _own_store, "merge": _own_merge}
_run_plain = {"rotary": _plain_rotary, "window": _plain_window, "store": _plain_store, "merge": _plain_merge}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _extent(c, rows_of=None):
    """Per query row (of a sample whose keys are all valid), the number of keys it sees."""
    pos = (c["begin"] if c["begin"] >= 0 else c["Sk"] - c["Sq"]) + torch.arange(c["Sq"], dtype=torch.int64)
    lo, hi = _bounds(c, pos)
    hi = hi.clamp(max=c["Sk"]).clamp(min=0)
    lo = torch.minimum(lo.clamp(min=0), hi)
    first = torch.minimum(torch.full_like(lo, c["sinks"]), lo)          # sinks in front of the window
    return first, lo, hi


def _pairs(c):
    first, lo, hi = _extent(c)
    return int((first + hi - lo).sum()) * c["B"] * c["H"]


def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "f32": 4}
    if c["kind"] == "rotary":
        D = sum(_AXES[c["axes"]]["dims"])
        rows = c["B"] * c["S"] * (c["H"] + c["Hk"])
        return {"bytes": rows * D * 4 + c["B"] * c["S"] * 12, "flops": rows * D * (3 if c["norm"] == "none" else 8)}
    if c["kind"] == "window":
        first, lo, hi = _extent(c)
        # keys that some row sees: the windows of a run of rows follow each other without a hole
        keys = max(0, int(hi.max()) - int(lo.min())) + min(int(first.max()), int(lo.min()))
        kv = 2 * c["B"] * c["Hk"] * min(keys, c["Sk"]) * c["D"] * 2
        rows = c["B"] * c["Sq"] * c["H"]
        return {"bytes": kv + rows * (4 * c["D"] + 4), "flops": 4 * c["D"] * _pairs(c)}
    rows = c["B"] * c["Sq"] * c["H"]
    cached = c["D"] + c["D"] // _BLOCK + 4
    if c["kind"] == "store":   # read the state, write the slot; read the slot, write the values
        return {"bytes": rows * (size[c["dtype"]] * c["D"] + 4 + 2 * cached + 2 * c["D"] + 4), "flops": 4 * rows * c["D"]}
    n = c["cached"] + c["fresh"]
    moved = c["cached"] * cached + c["fresh"] * (2 * c["D"] + 4) + size[c["out"]] * c["D"] + 4
    return {"bytes": rows * moved, "flops": 2 * n * rows * c["D"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "window": _exact_window, "store": _exact_store, "merge": _exact_merge}[case["kind"]](st)


def _exact_rotary(st):
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
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * t[:, :, None])
            parts.append((z if spec["pairing"] == "interleaved" else z.transpose(-1, -2)).flatten(-2))
        res.append(torch.cat(parts, -1))
    return tuple(res)


def _exact_window(st):
    c = st["case"]
    q, k, v = (st[x].double() for x in "qkv")
    B, Sq, H, D = q.shape
    Sk, G = k.shape[1], H // k.shape[2]
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=_DEV)
    lse = torch.full((B, H, Sq), -math.inf, dtype=torch.float64, device=_DEV)
    j = torch.arange(Sk, device=_DEV)
    for b in range(B):
        n = Sk if st["lens"] is None else int(st["lens"][b])
        begin = c["begin"] if c["begin"] >= 0 else n - Sq
        for s0 in range(0, Sq, 2048):
            p = begin + torch.arange(s0, min(Sq, s0 + 2048), device=_DEV)[:, None]
            f = (p - c["sinks"]) // c["frame"]
            key_frame = (j - c["sinks"]) // c["frame"]
            see = j < n
            if c["right"] >= 0:
                see = see & (key_frame <= f + c["right"])
            if c["left"] >= 0:
                see = see & ((j < c["sinks"]) | (key_frame >= f - c["left"]))
            see = see.expand(p.shape[0], Sk)
            used = see.any(0).nonzero()[:, 0]
            if used.numel() == 0:
                continue
            mask = torch.zeros(see.shape, dtype=torch.float64, device=_DEV).masked_fill(~see, -math.inf)[:, used]
            for h in range(H):
                x = q[b, s0:s0 + 2048, h] @ k[b, used, h // G].T / math.sqrt(D) + mask
                l = torch.logsumexp(x, -1)
                w = torch.exp(x - torch.where(l > -math.inf, l, torch.zeros_like(l))[:, None])
                out[b, s0:s0 + 2048, h] = w @ v[b, used, h // G]
                lse[b, h, s0:s0 + 2048] = l
    return out, lse


def _exact_value(x, fmt):
    """The values that x's blocks stand for once they are kept in 8 bits."""
    x = x.double().unflatten(-1, (-1, _BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    power = lambda n: ((n.long() + 1023) << 52).view(torch.float64)
    e = torch.ceil(torch.log2((amax / _PEAK[fmt]).clamp(min=2.0 ** -127)))
    e = torch.where(amax <= _PEAK[fmt] * power(e - 1), e - 1, e)        # the logarithm's own rounding, either way
    e = torch.where(amax > _PEAK[fmt] * power(e), e + 1, e).clamp(min=-127)
    step = power(e)
    if fmt == "e4m3":                                                    # 3 bits behind the leading one, from 2^-6 down a fixed step
        mag = (x / step).abs().clamp(min=2.0 ** -6)
        step = step * power(torch.frexp(mag)[1] - 1 - 3)
    return (torch.round(x / step) * step).flatten(-2)


def _exact_store(st):
    return _exact_value(st["out"], st["case"]["format"]), st["lse"].double().transpose(1, 2).unsqueeze(-1)


def _exact_merge(st):
    outs = [e.double().unflatten(-1, (-1, _BLOCK)) * _two_to(s.to(torch.int32).unsqueeze(-1) - 127).double() for e, s, _ in st["cached"]]
    outs = [o.flatten(-2) for o in outs] + [o.double() for o, _ in st["fresh"]]
    lses = torch.stack([s[-1].double() for s in st["cached"] + st["fresh"]])
    weights = torch.softmax(lses, 0).transpose(2, 3).unsqueeze(-1)
    return sum(w * o for w, o in zip(weights, outs)), torch.logsumexp(lses, 0).transpose(1, 2).unsqueeze(-1)
