"""Timed cases of the rotary-position and differential-attention operators.

Each case names one pass through an operator as a program makes it: rotary positions over the axes of the token grid
(``ops.rope_axes_fwd`` / ``ops.rope_axes_bwd``) and differential attention (``ops.diff_attention_fwd`` /
``ops.diff_attention_bwd``), the latter for inference, for a training step (forward and every gradient) and for a few new
tokens against a cache.  With ``own`` false ``run`` computes the operators in elementary torch operations in 32 bits, with
``own`` true it calls the HIP kernels.  ``exact`` is the definition in 64 bits.

Sizes: 8 x 14 x 14 = 1568 tokens are a 16-frame 224 x 224 clip, 160 its visible tokens under the 0.9 tube mask, 6 / 3
differential heads the 768- / 384-wide encoder / decoder, 32 clips the training batch.
"""
import math

import torch

own = False

DH = 64            # width of one softmax map's queries and keys
DV = 2 * DH        # width of a head's values and outputs
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
EPS = 1e-5
BASE = 10000.0


# ---------------------------------------------------------------------------------------------------------------- cases
def _rope(name, **kw):
    c = {"name": name, "op": "rope", "B": 1, "N": 1568, "heads": 24, "dim": 64, "st": 8, "sh": 12, "sw": 12, "tokens": True,
         "far": 0, "f32": False, "interleaved": False, "back": False}
    c.update(kw)
    return c


def _diff(name, **kw):
    c = {"name": name, "op": "infer", "B": 1, "Nq": 1568, "Nk": 1568, "H": 6, "Hkv": 6, "norm": True, "causal": 0, "ragged": False,
         "lam_init": 0.5}
    c.update(kw)
    return c


def listed():
    return [
        # the visible tokens of one clip, q and k of the packed projection: the smallest call, where latency counts
        _rope("rope-visible-1", N=160),
        # a training batch of whole clips, encoder width
        _rope("rope-clips-32", B=32),
        # its gradient at decoder width, adjacent pairs rotated, part of every head left as it is
        _rope("rope-back-dec-32", B=32, heads=12, st=4, sh=10, sw=10, interleaved=True, back=True),
        # f32 rows with positions of their own, far into a long stream; an odd number of rows
        _rope("rope-stream-f32", B=3, N=4999, heads=7, tokens=False, far=1 << 22, f32=True),
        # features of one clip
        _diff("diff-clip-1"),
        # features of a batch of clips
        _diff("diff-clips-16", B=16),
        # one long clip: 128 frames
        _diff("diff-long", Nq=12544, Nk=12544),
        # training, encoder: visible tokens of a batch
        _diff("diff-train-enc", op="train", B=32, Nq=160, Nk=160),
        # training, decoder: all tokens of a batch
        _diff("diff-train-dec", op="train", B=32, H=3, Hkv=3, lam_init=0.35),
        # training, causal, shared key heads, a padded batch of odd length with an empty clip in it
        _diff("diff-train-ragged", op="train", B=8, Nq=1111, Nk=1111, H=8, Hkv=2, norm=False, causal=1, ragged=True, lam_init=0.2),
        # one new token of every stream against a long cache filled to different lengths
        _diff("diff-token-16", op="token", B=16, Nq=1, Nk=8192, H=8, Hkv=2, causal=2, ragged=True),
        # the smallest: one new token, one stream, a short cache
        _diff("diff-token-1", op="token", Nq=1, Nk=257, causal=2),
    ]


def _spread(rng, lo, hi):
    """a whole number, even over its logarithm"""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "infer", "infer", "train", "train", "token", "token"])
    if kind == "rope":
        interleaved = rng.random() < 0.5
        half = 8 * rng.randint(2, 8)                    # rotated pairs of a head
        st = rng.randint(1, half - 2)
        sh = rng.randint(1, half - st - 1)
        dim = 2 * half + 16 * rng.randint(0, 2)
        heads = rng.randint(1, 32)
        rows = min(_spread(rng, 1, 60000), 60 * 1000 * 1000 // (heads * dim))
        B = rng.choice([1, 2, 3, 4, 8])
        tokens = rng.random() < 0.5
        N = max(1, min(rows // B, 1568 if tokens else rows))
        return {"op": "rope", "B": B, "N": N, "heads": heads, "dim": dim, "st": st, "sh": sh, "sw": half - st - sh, "tokens": tokens,
                "far": 0 if tokens else _spread(rng, 16, 1 << 22), "f32": rng.random() < 0.3, "interleaved": interleaved, "back": rng.random() < 0.5}
    group = rng.choice([1, 1, 2, 4])
    Hkv = rng.choice([3, 4, 6, 8]) if group == 1 else rng.choice([2, 3])
    H = group * Hkv
    lam_init = round(rng.uniform(0.2, 0.75), 3)
    norm = rng.random() < 0.6
    if kind == "token":
        Nk = _spread(rng, 2, 16384)
        B = max(1, min(_spread(rng, 1, 32), 131072 // Nk))
        Nq = rng.choice([1, 1, 1, min(2, Nk), min(5, Nk)])
        return {"op": "token", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "norm": norm, "causal": 2, "ragged": rng.random() < 0.5, "lam_init": lam_init}
    Nk = _spread(rng, 33, 8192 if kind == "infer" else 3000)
    B = max(1, min(_spread(rng, 1, 32), int((120e6 if kind == "infer" else 60e6) / (Nk * Nk * H))))
    cross = kind == "infer" and rng.random() < 0.3      # queries of another length
    Nq = _spread(rng, 8, Nk) if cross else Nk
    return {"op": kind, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "norm": norm, "causal": 0 if cross else rng.choice([0, 0, 1]),
            "ragged": rng.random() < 0.4, "lam_init": lam_init}


def _lengths(case):
    """keys that each clip holds: all of them, or spread over 0 .. Nk (a cache: at least its new tokens)"""
    B, Nk = case["B"], case["Nk"]
    if not case["ragged"]:
        return [Nk] * B
    least = case["Nq"] if case["op"] == "token" else 0
    return [least + (Nk - least) * (b + 1) // B if b else (least if B > 1 else Nk) for b in range(B)]


def _pairs(case):
    """(query, key) pairs that see each other, over clips and heads"""
    n = 0
    for length in _lengths(case):
        if case["causal"] == 0:
            n += case["Nq"] * length
        else:
            off = 0 if case["causal"] == 1 else length - case["Nq"]
            n += sum(max(0, min(length, i + off + 1)) for i in range(case["Nq"]))
    return n * case["H"]


def work(case):
    if case["op"] == "rope":
        n = case["B"] * case["N"] * case["heads"] * case["dim"]
        place = (1 if case["tokens"] else 3) * 4 * case["B"] * case["N"]
        return {"bytes": 2 * n * (4 if case["f32"] else 2) + place, "flops": 3 * n}
    rows, kept = case["B"] * case["Nq"], sum(_lengths(case))
    q, kv = rows * case["H"] * DV * 2, kept * case["Hkv"] * DV * 2
    pairs = _pairs(case)
    # two maps of 64, one product of their difference with the 128 wide values; training: the values' gradient, the
    # difference's, and the queries' and keys' of both maps
    if case["op"] == "train":
        return {"bytes": 4 * q + 4 * kv, "flops": (4 * DH + 2 * DV + 4 * DV + 8 * DH) * pairs}
    return {"bytes": 2 * q + 2 * kv, "flops": (4 * DH + 2 * DV) * pairs}


# --------------------------------------------------------------------------------------------------------------- inputs
def _made(seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return g, lambda *shape, std=1.0, dt=BF16: (torch.randn(*shape, generator=g, device=dev) * std).to(dt)


def _positions(case, g, dev):
    """token ids on the 8 x 14 x 14 grid, ascending within a clip (what a tube mask leaves), or (time, row, column) of a stream"""
    B, N = case["B"], case["N"]
    if case["tokens"]:
        order = torch.rand(B, 1568, generator=g, device=dev).argsort(1)[:, :N].sort(1).values
        return order.to(I32).contiguous()
    first = torch.randint(0, case["far"], (B, 1), generator=g, device=dev)
    at = torch.arange(N, device=dev)[None] + first * 196
    return torch.stack([at // 196, at // 14 % 14, at % 14], -1).to(I32).reshape(B * N, 3).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g, rand = _made(seed, dev)
    s = {"case": case}
    if case["op"] == "rope":
        M, W = case["B"] * case["N"], case["heads"] * case["dim"]
        dt = F32 if case["f32"] else BF16
        packed = rand(M, W + W // 2 // 8 * 8, dt=dt)      # q | k | v of the projection; q and k are rotated
        s.update(x=packed[:, :W], at=_positions(case, g, dev), out=torch.empty(M, W, dtype=dt, device=dev),
                 freqs=_frequencies(case, dev))
        return s
    B, Nq, Nk, H, Hkv = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv"))
    if case["op"] != "token" and Nq == Nk:               # packed projection
        # a token's query resembles its own key, and the gradient that comes back leans towards its own value
        packed = rand(B * Nq, (H + 2 * Hkv) * DV)
        alike = packed[:, H * DV:].reshape(-1, 2, Hkv, 1, DV).expand(-1, -1, -1, H // Hkv, -1).reshape(-1, 2, H * DV)
        packed[:, :H * DV] = 1.375 * packed[:, :H * DV] + 0.6 * alike[:, 0]
        s.update(q=packed[:, :H * DV], k=packed[:, H * DV:(H + Hkv) * DV], v=packed[:, (H + Hkv) * DV:])
        if case["op"] == "train":
            d = torch.empty_like(packed)
            s.update(dout=rand(B * Nq, H * DV) + 0.5 * alike[:, 1], dq=d[:, :H * DV], dk=d[:, H * DV:(H + Hkv) * DV], dv=d[:, (H + Hkv) * DV:])
    else:                                                # a cache of Nk rows a clip
        s.update(q=rand(B * Nq, H * DV, std=1.5), k=rand(B * Nk, Hkv * DV), v=rand(B * Nk, Hkv * DV))
    lens = _lengths(case)
    order = torch.randperm(B, generator=g, device=dev).tolist()
    s["kv_len"] = torch.tensor([lens[i] for i in order], dtype=I32, device=dev) if case["ragged"] else None
    s["lam"] = rand(4, H, DH, std=0.1)
    s["gamma"] = (1 + rand(DV, std=0.2, dt=F32)).to(BF16) if case["norm"] else None
    s["out"] = torch.empty(B * Nq, H * DV, dtype=BF16, device=dev)
    if case["op"] == "train":
        s["saved"] = (torch.empty_like(s["out"]), torch.empty_like(s["out"]), torch.empty(2, B, H, Nq, dtype=F32, device=dev))
        s["dlam"], s["dgamma"] = torch.empty_like(s["lam"]), torch.empty_like(s["gamma"]) if case["norm"] else None
    # scratch of the kernels, kept from call to call: at most the f32 maps' sums of every split, or the gradient's rows
    s["ws"] = torch.empty(_scratch(case), dtype=F32, device=dev)
    return s


def _frequencies(case, dev):
    """turns per position of every rotated pair, an axis after the other, each with a ladder of its own (64 bits)"""
    f = [BASE ** (-i / n) / (2 * math.pi) for n in (case["st"], case["sh"], case["sw"]) for i in range(n)]
    return torch.tensor(f, dtype=F64, device=dev)


def _scratch(case):
    rows = case["B"] * case["Nq"] * case["H"]
    parts = 260 * min(64 * rows, 1 << 16)
    return max(parts, rows * (DV // 2 + 2) + (1 << 18)) if case["op"] == "train" else parts


# ------------------------------------------------------------------------------------------------------------ plain form
def _sections(case):
    return (case["st"], case["sh"], case["sw"])


def _plain_rope(s):
    case = s["case"]
    M, heads, dim = s["x"].shape[0], case["heads"], case["dim"]
    if case["tokens"]:
        at = s["at"].reshape(-1).long()
        place = torch.stack([at // 196, at // 14 % 14, at % 14], -1)
    else:
        place = s["at"]
    axis = torch.repeat_interleave(torch.arange(3, device=place.device), torch.tensor(_sections(case), device=place.device))
    turns = place.double()[:, axis] * s["freqs"]                          # angles of far positions: 64 bits
    angle = (turns - turns.floor()) * (2 * math.pi)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["back"]:
        sin = -sin
    half = axis.numel()
    x = s["x"].reshape(M, heads, dim).float()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if case["interleaved"] else (x[..., :half], x[..., half:2 * half])
    a, b = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([a, b], -1).flatten(2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * half:]], -1).reshape(M, heads * dim).to(s["x"].dtype)


def _split(t, B, heads, parts):
    """[B * N, heads * parts * w] -> [B, heads, parts, N, w]"""
    return t.reshape(B, t.shape[0] // B, heads, parts, -1).permute(0, 2, 3, 1, 4)


def _visible(case, kv_len, dev):
    """[B, 1, 1, Nq, Nk] truth values"""
    Nq, Nk = case["Nq"], case["Nk"]
    length = kv_len.long() if kv_len is not None else torch.full((case["B"],), Nk, device=dev)
    j = torch.arange(Nk, device=dev)
    last = length[:, None, None].expand(-1, Nq, 1)
    if case["causal"]:
        i = torch.arange(Nq, device=dev)[None, :, None]
        last = torch.minimum(last, i + 1 + (length[:, None, None] - Nq if case["causal"] == 2 else 0))
    return (j < last)[:, None, None]


def _plain_maps(s):
    """both softmax maps [B, H, 2, Nq, Nk], rows that see nothing all zero, and the heads' lambda"""
    case = s["case"]
    B, H, Hkv = case["B"], case["H"], case["Hkv"]
    q = _split(s["q"].float(), B, H, 2).contiguous()
    k = _split(s["k"].float(), B, Hkv, 2).repeat_interleave(H // Hkv, 1).contiguous()
    v = _split(s["v"].float(), B, Hkv, 1).repeat_interleave(H // Hkv, 1).squeeze(2).contiguous()
    see = _visible(case, s["kv_len"], q.device)
    x = (q @ k.transpose(-1, -2).contiguous()) * DH ** -0.5
    x = x.masked_fill(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    lam = s["lam"].float()
    e1, e2 = (lam[0] * lam[1]).sum(-1).exp(), (lam[2] * lam[3]).sum(-1).exp()
    return q, k, v, p, e1, e2, (e1 - e2 + case["lam_init"])[None, :, None, None]


def _plain_norm(s, o):
    if not s["case"]["norm"]:
        return o, None
    r = (o.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return o * r * s["gamma"].float() * (1 - s["case"]["lam_init"]), r


def _rows(t):
    """[B, heads, N, w] -> [B * N, heads * w] in bf16"""
    return t.transpose(1, 2).reshape(t.shape[0] * t.shape[2], -1).to(BF16)


def _plain_attention(s):
    q, k, v, p, e1, e2, lam = _plain_maps(s)
    o = (p[:, :, 0] - lam * p[:, :, 1]) @ v
    return {"out": _rows(_plain_norm(s, o)[0])}


def _plain_training(s):
    case = s["case"]
    B, H, Hkv = case["B"], case["H"], case["Hkv"]
    q, k, v, p, e1, e2, lam = _plain_maps(s)
    a = p[:, :, 0] - lam * p[:, :, 1]
    o = a @ v
    y, r = _plain_norm(s, o)
    dy = _split(s["dout"].float(), B, H, 1).squeeze(2)
    got = {"out": _rows(y)}
    if case["norm"]:
        xhat, g = o * r, dy * s["gamma"].float() * (1 - case["lam_init"])
        got["dgamma"] = (dy * xhat * (1 - case["lam_init"])).sum((0, 1, 2)).to(BF16)
        dy = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    dy = dy.contiguous()
    da = dy @ v.transpose(-1, -2).contiguous()
    dv = a.transpose(-1, -2).contiguous() @ dy
    drop = (da[:, :, None] * p).sum(-1, keepdim=True)                       # [B, H, 2, Nq, 1]
    ds = p * (da[:, :, None] - drop) * DH ** -0.5
    ds[:, :, 1] *= -lam
    dlam = -drop[:, :, 1].double().sum((0, 2, 3)).float()                   # a long sum that cancels
    dq = ds @ k
    dk = ds.transpose(-1, -2).contiguous() @ q
    share = lambda t: t.reshape(B, Hkv, H // Hkv, *t.shape[2:]).sum(2)  # noqa: E731
    joined = lambda t: _rows(t.transpose(2, 3).flatten(3))  # noqa: E731
    l = s["lam"].float()
    d1, d2 = (dlam * e1)[:, None], (-dlam * e2)[:, None]
    got.update(dq=joined(dq), dk=joined(share(dk)), dv=_rows(share(dv)), dlam=torch.stack([d1 * l[1], d1 * l[0], d2 * l[3], d2 * l[2]]).to(BF16))
    return got


# ------------------------------------------------------------------------------------------------------------------- run
def _kernel_rope(s):
    from mofo_amd import ops
    case = s["case"]
    where = {"tok_idx": s["at"], "grid": (8, 14, 14)} if case["tokens"] else {"pos": s["at"]}
    turn = ops.rope_axes_bwd if case["back"] else ops.rope_axes_fwd
    turn(s["x"], case["heads"], case["dim"], _sections(case), s["freqs"], s["out"], interleaved=case["interleaved"], **where)
    return s["out"]


def _kernel_attention(s):
    from mofo_amd import ops
    case = s["case"]
    B, H, Hkv, scale = case["B"], case["H"], case["Hkv"], DH ** -0.5
    form = {"gamma": s["gamma"], "eps": EPS, "out_scale": 1 - case["lam_init"] if case["norm"] else 1.0, "kv_len": s["kv_len"],
            "causal": case["causal"]}
    if case["op"] != "train":
        ops.diff_attention_fwd(s["q"], s["k"], s["v"], B, H, Hkv, scale, s["lam"], case["lam_init"], s["out"], ws=s["ws"], **form)
        return {"out": s["out"]}
    ops.diff_attention_fwd(s["q"], s["k"], s["v"], B, H, Hkv, scale, s["lam"], case["lam_init"], s["out"], saved=s["saved"], ws=s["ws"], **form)
    ops.diff_attention_bwd(s["q"], s["k"], s["v"], B, H, Hkv, scale, s["lam"], case["lam_init"], s["saved"], s["dout"], s["dq"], s["dk"], s["dv"],
                           s["dlam"], s["ws"], dgamma=s["dgamma"], **form)
    got = {"out": s["out"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"], "dlam": s["dlam"]}
    if case["norm"]:
        got["dgamma"] = s["dgamma"]
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return _kernel_rope(state) if op == "rope" else _kernel_attention(state)
    return _plain_rope(state) if op == "rope" else _plain_training(state) if op == "train" else _plain_attention(state)


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_rope(s):
    case = s["case"]
    M, heads, dim = s["x"].shape[0], case["heads"], case["dim"]
    at = s["at"].long()
    if case["tokens"]:
        at = at.reshape(-1)
        t = at.div(196, rounding_mode="floor")
        h = (at - 196 * t).div(14, rounding_mode="floor")
        at = torch.stack([t, h, at - 196 * t - 14 * h], -1)
    at = at.double()
    cols = [(at[:, a] * (BASE ** (-i / n) / (2 * math.pi))).remainder(1.0) * (2 * math.pi) for a, n in enumerate(_sections(case)) for i in range(n)]
    angle = torch.stack(cols, -1)
    turn = torch.polar(torch.ones_like(angle), -angle if case["back"] else angle)[:, None]
    half = angle.shape[1]
    x = s["x"].double().reshape(M, heads, dim)
    y = x.clone()
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    z = torch.complex(x[..., lo], x[..., hi]) * turn
    y[..., lo], y[..., hi] = z.real, z.imag
    return y.reshape(M, heads * dim)


def _exact_clip(case, q, k, v, length):
    """one clip, one key head and its queries: [G, Nq, 2, 64], [Nk, 2, 64], [Nk, 128] in 64 bits -> both maps' outputs [G, 2, Nq, 128]"""
    Nq, Nk = case["Nq"], case["Nk"]
    i, j = torch.arange(Nq, device=q.device)[:, None], torch.arange(Nk, device=q.device)[None]
    hide = j >= length
    if case["causal"]:
        hide = hide | (j > i + (length - Nq if case["causal"] == 2 else 0))
    full = hide.expand(Nq, Nk).all(-1)[:, None]
    x = torch.matmul(q.permute(2, 0, 1, 3).reshape(2, -1, DH), k.permute(1, 2, 0)).reshape(2, -1, Nq, Nk) / math.sqrt(DH)
    w = torch.softmax(x.masked_fill(hide, -1e300), -1).masked_fill(full, 0.0)
    return torch.matmul(w, v).transpose(0, 1)


def _exact_head(case, s, q, k, v, lam, gamma, b, h, length):
    """one clip's queries of one key head: the heads' outputs [G, Nq, 128]"""
    B, Nq, Nk, H, Hkv = (case[n] for n in ("B", "Nq", "Nk", "H", "Hkv"))
    heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
    o = _exact_clip(case, q.view(B, Nq, H, 2, DH)[b, :, heads].transpose(0, 1), k.view(B, Nk, Hkv, 2, DH)[b, :, h], v.view(B, Nk, Hkv, DV)[b, :, h],
                    length)
    weight = torch.exp((lam[0, heads] * lam[1, heads]).sum(-1)) - torch.exp((lam[2, heads] * lam[3, heads]).sum(-1)) + case["lam_init"]
    y = o[:, 0] - weight[:, None, None] * o[:, 1]
    if gamma is None:
        return y
    return y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma * (1 - case["lam_init"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    B, Nq, H, Hkv, train = case["B"], case["Nq"], case["H"], case["Hkv"], case["op"] == "train"
    G = H // Hkv
    lens = s["kv_len"].tolist() if s["kv_len"] is not None else [case["Nk"]] * B
    q, k, v, lam = (s[n].double().contiguous().requires_grad_(train) for n in ("q", "k", "v", "lam"))
    gamma = s["gamma"].double().requires_grad_(train) if case["norm"] else None
    out = torch.empty(B, Nq, H, DV, dtype=F64, device=q.device)
    for b in range(B):
        for h in range(Hkv):
            with torch.set_grad_enabled(train):
                y = _exact_head(case, s, q, k, v, lam, gamma, b, h, lens[b])
                if train:
                    (y * s["dout"].double().view(B, Nq, H, DV)[b, :, h * G:(h + 1) * G].transpose(0, 1)).sum().backward()
            out[b, :, h * G:(h + 1) * G] = y.detach().transpose(0, 1)
    got = {"out": out.reshape(B * Nq, H * DV)}
    if train:
        got.update(dq=q.grad, dk=k.grad, dv=v.grad, dlam=lam.grad)
        if case["norm"]:
            got["dgamma"] = gamma.grad
    return got
