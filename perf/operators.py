"""Measured cases of the long-context streaming operators: attention with a sliding window and a few first
tokens that stay visible (prefill, training, paged decode), rotary positions (training, and fused with the
append to a paged cache), and the copies inside a paged cache (whole pages, single tokens).

``run`` computes a case with the package's kernels where ``own`` is true, and in a plain form of elementary
torch operations in 32 bits where it is false; ``exact`` gives the 64-bit result of the definition."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_MAX_SCORES = 32 * 8192 * 8192  # scores of the largest attention case's plain form


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a short prompt on a small model: a call bound by latency, odd in length and window
        dict(name="prefill short", op="prefill", dtype="fp16", B=3, Hq=8, Hkv=2, S=77, D=64, window=32, sinks=3,
             softcap=0.0),
        # prefill of a long prompt at the grouped-query shape of the benchmark, window 1024
        dict(name="prefill long", op="prefill", dtype="bf16", B=1, Hq=32, Hkv=8, S=8192, D=128, window=1024, sinks=4,
             softcap=0.0),
        # a training step of the windowed, capped configuration of the benchmark, half its batch
        dict(name="train", op="train", dtype="bf16", B=4, Hq=16, Hkv=16, S=4096, D=128, window=1024, sinks=4,
             softcap=30.0),
        # grouped heads at head dim 64, a ragged length, sinks that end inside a tile
        dict(name="train ragged", op="train", dtype="fp16", B=2, Hq=12, Hkv=3, S=1543, D=64, window=200, sinks=17,
             softcap=0.0),
        # the framework's fp32 configuration with a window
        dict(name="train fp32", op="train", dtype="fp32", B=2, Hq=8, Hkv=8, S=1024, D=64, window=256, sinks=4,
             softcap=0.0),
        # one user's next token far into a conversation: latency
        dict(name="decode one", op="decode", dtype="bf16", R=1, Hq=32, Hkv=8, D=128, page=64, ctx_lo=20011,
             ctx_hi=20011, window=4096, sinks=4, softcap=0.0),
        # a serving batch with the context lengths of the benchmark's paged decode
        dict(name="decode batch", op="decode", dtype="bf16", R=64, Hq=32, Hkv=8, D=128, page=16, ctx_lo=512,
             ctx_hi=32768, window=4096, sinks=4, softcap=0.0),
        # many heads without grouping, pages that are no multiple of a tile, an empty context among them
        dict(name="decode odd", op="decode", dtype="fp16", R=5, Hq=20, Hkv=20, D=64, page=24, ctx_lo=0, ctx_hi=3001,
             window=1000, sinks=1, softcap=0.0),
        # queries and keys of a training step, with their gradients
        dict(name="rotary train", op="rotary", dtype="bf16", B=4, S=4096, Hq=32, Hkv=8, D=128, rot=128,
             layout="half"),
        # one new token for each of 64 requests: rotated and written into the paged cache
        dict(name="rotary append", op="append", dtype="bf16", T=64, Hq=32, Hkv=8, D=128, rot=64, page=16,
             layout="interleaved"),
        # forks of a few sequences: their last pages copied
        dict(name="pages fork", op="pages", dtype="bf16", n=16, Hkv=8, D=128, page=64),
        # 64 sequences, each compacted to its window and its first tokens
        dict(name="pages compact", op="tokens", dtype="bf16", n=64 * 4100, Hkv=8, D=128, page=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the same operators, sizes over the whole range between one token and the largest case."""
    op = rng.choice(["prefill", "prefill", "train", "train", "decode", "decode", "decode", "rotary", "append",
                     "pages", "tokens"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    hkv = rng.choice([1, 2, 3, 5, 8])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    dim = rng.choice([64, 96, 128, 128])
    if op in ("prefill", "train"):
        dtype = "fp32" if rng.random() < 0.15 else half
        s = _log_int(rng, 1, 4096 if dtype != "fp32" else 1500)
        heads = hkv * group
        cap = _MAX_SCORES // (2 if op == "prefill" else 8)
        b = max(1, min(_log_int(rng, 1, 8), cap // (heads * s * s)))
        return dict(op=op, dtype=dtype, B=b, Hq=heads, Hkv=hkv, S=s, D=dim, window=_log_int(rng, 1, 4096),
                    sinks=rng.choice([1, 2, 4, 4, 8, 37, 130]), softcap=rng.choice([0.0, 0.0, 30.0]))
    if op == "decode":
        r = _log_int(rng, 1, 64)
        lo = rng.choice([0, 1, 100, 512])
        return dict(op=op, dtype=half, R=r, Hq=hkv * group, Hkv=hkv, D=dim, page=rng.choice([16, 24, 64, 128]),
                    ctx_lo=lo, ctx_hi=lo + _log_int(rng, 1, 32000), window=_log_int(rng, 16, 4096),
                    sinks=rng.choice([1, 4, 4, 16, 70]), softcap=rng.choice([0.0, 0.0, 30.0]))
    if op == "rotary":
        return dict(op=op, dtype=rng.choice([half, half, "fp32"]), B=_log_int(rng, 1, 4), S=_log_int(rng, 1, 4096),
                    Hq=min(32, hkv * group), Hkv=hkv, D=dim, rot=rng.choice([dim, dim // 2, 20]),
                    layout=rng.choice(["half", "interleaved"]))
    if op == "append":
        return dict(op=op, dtype=half, T=_log_int(rng, 1, 8192), Hq=min(32, hkv * group), Hkv=hkv, D=dim,
                    rot=rng.choice([dim, dim // 2, 20]), page=rng.choice([16, 24, 64, 128]),
                    layout=rng.choice(["half", "interleaved"]))
    page = rng.choice([16, 24, 64, 128])
    if op == "pages":
        return dict(op=op, dtype=half, n=_log_int(rng, 1, 16384 * 16 // page), Hkv=hkv, D=dim, page=page)
    return dict(op=op, dtype=half, n=_log_int(rng, 1, 64 * 4096), Hkv=hkv, D=dim, page=page)


# -------------------------------------------------------------------------------------------- inputs
def _lens(case):
    """Context lengths, spread evenly over [ctx_lo, ctx_hi] (the seed decides their order alone)."""
    r, lo, hi = case["R"], case["ctx_lo"], case["ctx_hi"]
    return [hi] if r == 1 else [lo + (hi - lo) * i // (r - 1) for i in range(r)]


def _tables(positions, dim, base):
    """cos / sin [positions, dim / 2] fp32 of the rotary angles, built once in 64 bits."""
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float().cuda(), ang.sin().float().cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    def perm(n):
        return torch.randperm(n, generator=g, device="cuda")

    if op in ("prefill", "train"):
        # the heads of a projection's output: [B, S, H, D] storage seen as [B, H, S, D]
        b, s, d = case["B"], case["S"], case["D"]
        q, do = (randn(b, s, case["Hq"], d).transpose(1, 2) for _ in range(2))
        k, v = (randn(b, s, case["Hkv"], d).transpose(1, 2) for _ in range(2))
        return dict(case=case, q=q, k=k, v=v, do=do)
    if op == "decode":
        lens = torch.tensor(_lens(case), device="cuda")[perm(case["R"])]
        ps, w, n = case["page"], case["window"], case["sinks"]
        width = max(1, -(-case["ctx_hi"] // ps))
        first = torch.arange(width, device="cuda")[None, :] * ps  # first token of each page
        ln = lens[:, None]
        # pages that hold a first token or one of the window; the others were freed (-1 in the table)
        held = (first < ln) & ((first < n) | (first + ps > ln - w))
        pages = max(1, int(held.sum()))
        bt = torch.full(held.shape, -1, dtype=torch.int32, device="cuda")
        bt[held] = perm(pages)[: int(held.sum())].to(torch.int32)
        shape = (pages, case["Hkv"], ps, case["D"])
        return dict(case=case, q=randn(case["R"], case["Hq"], case["D"]), kp=randn(*shape), vp=randn(*shape), bt=bt,
                    lens=lens.to(torch.int32))
    if op == "rotary":
        b, s, d = case["B"], case["S"], case["D"]
        q, dq = (randn(b, s, case["Hq"], d).transpose(1, 2) for _ in range(2))
        k, dk = (randn(b, s, case["Hkv"], d).transpose(1, 2) for _ in range(2))
        cos, sin = _tables(8192, case["rot"], 10000.0)
        # each row of the batch goes on from a position of its own
        start = torch.randint(0, 8192 - s + 1, (b, 1), generator=g, device="cuda")
        pos = (start + torch.arange(s, device="cuda")[None, :]).to(torch.int32)
        return dict(case=case, q=q, k=k, dq=dq, dk=dk, cos=cos, sin=sin, pos=pos)
    if op == "append":
        t, hq, hkv, d, ps = (case[x] for x in ("T", "Hq", "Hkv", "D", "page"))
        x = randn(t, (hq + 2 * hkv) * d)  # the output of one stacked projection
        cos, sin = _tables(32768, case["rot"], 10000.0)
        pages = -(-2 * t // ps) + 1
        shape = (pages, hkv, ps, d)
        return dict(case=case, q=x[:, :hq * d].view(t, hq, d), k=x[:, hq * d:(hq + hkv) * d].view(t, hkv, d),
                    v=x[:, (hq + hkv) * d:].view(t, hkv, d), cos=cos, sin=sin,
                    pos=torch.randint(0, 32768, (t,), generator=g, device="cuda", dtype=torch.int32),
                    slots=perm(pages * ps)[:t].to(torch.int32), kp=randn(*shape), vp=randn(*shape))
    if op == "pages":
        n = case["n"]
        shape = (2 * n, case["Hkv"], case["page"], case["D"])
        order = perm(2 * n).to(torch.int32)
        return dict(case=case, kp=randn(*shape), vp=randn(*shape), src=order[:n].clone(), dst=order[n:].clone())
    # tokens: the kept ones of old pages, in runs, go to fresh pages in order
    n, ps = case["n"], case["page"]
    old, new = -(-5 * n // (4 * ps)) + 1, -(-n // ps)
    order = perm(old + new)
    kept = perm(old * ps)[:n].sort().values
    src = order[kept // ps] * ps + kept % ps
    at = torch.arange(n, device="cuda")
    dst = order[old + at // ps] * ps + at % ps
    shape = (old + new, case["Hkv"], ps, case["D"])
    return dict(case=case, kp=randn(*shape), vp=randn(*shape), src=src.to(torch.int32), dst=dst.to(torch.int32))


# ----------------------------------------------------------------------------------------- plain forms
def _visible(sq, skv, window, sinks):
    """[sq, skv]: key j of query i is in its past, and in its window or one of the first tokens."""
    i = torch.arange(sq, device="cuda")[:, None]
    j = torch.arange(skv, device="cuda")[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks))


def _plain_forward(st):
    c = st["case"]
    group = c["Hq"] // c["Hkv"]
    q = st["q"].float()
    k, v = (st[x].float().repeat_interleave(group, 1) for x in ("k", "v"))
    s = q @ k.transpose(-1, -2) * (1.0 / math.sqrt(c["D"]))
    th = None
    if c["softcap"] > 0:
        th = torch.tanh(s / c["softcap"])
        s = th * c["softcap"]
    s = s.masked_fill_(~_visible(c["S"], c["S"], c["window"], c["sinks"]), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p = p.div_(l)
    return q, k, v, th, p, p @ v, m + l.log()


def _plain_backward(st, q, k, v, th, p, o):
    c = st["case"]
    b, hkv, s, d = st["k"].shape
    do = st["do"].float()
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if th is not None:
        ds = ds.mul_(1 - th * th)
    ds = ds.mul_(1.0 / math.sqrt(d))
    dq = ds @ k
    dk = ds.transpose(-1, -2) @ q
    dk, dv = (x.view(b, hkv, c["Hq"] // hkv, s, d).sum(2) for x in (dk, dv))
    return dq, dk, dv


def _plain_decode(st):
    c = st["case"]
    r, hq, hkv, d, ps, w, n = (c[x] for x in ("R", "Hq", "Hkv", "D", "page", "window", "sinks"))
    ln = st["lens"].long()[:, None]
    # the tokens a request sees: its first ones, then its window (without those counted already)
    start = torch.maximum(ln - w, ln.clamp(max=n))
    first = torch.arange(min(n, c["ctx_hi"]), device="cuda")[None, :].expand(r, -1)
    last = start + torch.arange(min(w, c["ctx_hi"]), device="cuda")[None, :]
    tok = torch.cat([first, last], 1)
    seen = tok < ln
    tok = torch.where(seen, tok, 0)
    page = st["bt"].long().gather(1, tok // ps).clamp(min=0)
    k = st["kp"][page, :, tok % ps].float()  # [R, tokens, Hkv, D]
    v = st["vp"][page, :, tok % ps].float()
    q = st["q"].float().view(r, hkv, hq // hkv, d)
    s = torch.einsum("rhgd,rthd->rhgt", q, k) * (1.0 / math.sqrt(d))
    if c["softcap"] > 0:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    s = torch.where(seen[:, None, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = torch.einsum("rhgt,rthd->rhgd", p / torch.where(l > 0, l, 1.0), v)
    return o.reshape(r, hq, d), (m + l.log()).reshape(r, hq)


def _plain_rotate(x, cos, sin, layout, back=False):
    """x [..., D]: its first 2 * cos.shape[-1] values rotated in pairs (by the negative angle with `back`)."""
    rot = 2 * cos.shape[-1]
    y = x.float()
    head, rest = y[..., :rot], y[..., rot:]
    if layout == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
    else:
        a, b = head[..., 0::2], head[..., 1::2]
    sn = -sin if back else sin
    a, b = a * cos - b * sn, b * cos + a * sn
    head = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([head, rest], -1).to(x.dtype)


def _plain(st):
    c = st["case"]
    op = c["op"]
    if op == "prefill":
        o, lse = _plain_forward(st)[5:]
        return dict(o=o.to(st["q"].dtype), lse=lse)
    if op == "train":
        q, k, v, th, p, o, _ = _plain_forward(st)
        dq, dk, dv = _plain_backward(st, q, k, v, th, p, o)
        dt = st["q"].dtype
        return dict(o=o.to(dt), dq=dq.to(dt), dk=dk.to(dt), dv=dv.to(dt))
    if op == "decode":
        o, lse = _plain_decode(st)
        return dict(o=o.to(st["q"].dtype), lse=lse)
    if op == "rotary":
        pos = st["pos"].long()
        cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]  # [B, 1, S, rot / 2]
        out = {x: _plain_rotate(st[x], cos, sin, c["layout"]) for x in ("q", "k")}
        out.update({x: _plain_rotate(st[x], cos, sin, c["layout"], back=True) for x in ("dq", "dk")})
        return out
    if op == "append":
        pos, slots, ps = st["pos"].long(), st["slots"].long(), c["page"]
        cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]  # [T, 1, rot / 2]
        st["kp"][slots // ps, :, slots % ps] = _plain_rotate(st["k"], cos, sin, c["layout"])
        st["vp"][slots // ps, :, slots % ps] = st["v"]
        return dict(q=_plain_rotate(st["q"], cos, sin, c["layout"]), kp=st["kp"], vp=st["vp"])
    src, dst, ps = st["src"].long(), st["dst"].long(), c["page"]
    if op == "pages":
        st["kp"][dst] = st["kp"][src]
        st["vp"][dst] = st["vp"][src]
    else:
        st["kp"][dst // ps, :, dst % ps] = st["kp"][src // ps, :, src % ps]
        st["vp"][dst // ps, :, dst % ps] = st["vp"][src // ps, :, src % ps]
    return dict(kp=st["kp"], vp=st["vp"])


def run(st):
    if not own:
        with torch.no_grad():
            return _plain(st)
    import fastest_flash_attention_b200 as ffa

    c = st["case"]
    op = c["op"]
    if op == "prefill":
        o, lse = ffa.fastest_flash_attn_forward(
            st["q"], st["k"], st["v"], causal=True, sliding_window=c["window"], sink_tokens=c["sinks"],
            softcap=c["softcap"] or None, return_lse=True)
        return dict(o=o, lse=lse)
    if op == "train":
        q, k, v = (st[x].detach().requires_grad_() for x in ("q", "k", "v"))
        o = ffa.fastest_flash_attn_func(q, k, v, causal=True, sliding_window=c["window"], sink_tokens=c["sinks"],
                                        softcap=c["softcap"] or None)
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), st["do"])
        return dict(o=o, dq=dq, dk=dk, dv=dv)
    if op == "decode":
        o, lse = ffa.paged_decode(st["q"], st["kp"], st["vp"], st["bt"], st["lens"], sliding_window=c["window"],
                                  sink_tokens=c["sinks"], softcap=c["softcap"] or None, return_lse=True)
        return dict(o=o, lse=lse)
    if op == "rotary":
        q, k = (st[x].detach().requires_grad_() for x in ("q", "k"))
        qr, kr = ffa.apply_rotary(q, k, st["cos"], st["sin"], st["pos"], layout=c["layout"])
        dq, dk = torch.autograd.grad((qr, kr), (q, k), (st["dq"], st["dk"]))
        return dict(q=qr, k=kr, dq=dq, dk=dk)
    if op == "append":
        q = ffa.rotary_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["slots"], st["kp"],
                              st["vp"], layout=c["layout"])
        return dict(q=q, kp=st["kp"], vp=st["vp"])
    if op == "pages":
        ffa.copy_pages(st["kp"], st["vp"], st["src"], st["dst"])
    else:
        ffa.move_tokens(st["kp"], st["vp"], st["src"], st["dst"])
    return dict(kp=st["kp"], vp=st["vp"])


# ------------------------------------------------------------------------------------------------ work
def _pairs(s, window, sinks):
    """Visible (query, key) pairs of one head: query i sees min(i + 1, window) keys of its window, and those of
    the first `sinks` that lie before it."""
    n = 0
    for i in range(s):
        n += min(i + 1, window) + min(sinks, max(0, i + 1 - window))
    return n


def work(case):
    op, es = case["op"], _BYTES[case["dtype"]]
    if op in ("prefill", "train"):
        b, hq, hkv, s, d = (case[x] for x in ("B", "Hq", "Hkv", "S", "D"))
        qo, kv = b * hq * s * d * es, b * hkv * s * d * es
        pairs = b * hq * _pairs(s, case["window"], case["sinks"])
        if op == "prefill":  # q, k, v read, o and the statistics written; Q.K and P.V
            return dict(bytes=2 * qo + 2 * kv + 4 * b * hq * s, flops=4 * d * pairs)
        # and the gradient: dO read, dq, dk, dv written; Q.K again, dO.V, and the three gradients' products
        return dict(bytes=4 * qo + 4 * kv, flops=14 * d * pairs)
    if op == "decode":
        seen = sum(min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in _lens(case))
        hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
        return dict(bytes=2 * seen * hkv * d * es + case["R"] * hq * (2 * d * es + 4), flops=4 * seen * hq * d)
    if op == "rotary":  # q, k and the two gradients, each read and written
        values = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * case["D"]
        turned = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * case["rot"]
        return dict(bytes=4 * values * es + 4 * case["B"] * case["S"] * (case["rot"] + 1), flops=6 * turned)
    if op == "append":
        values = case["T"] * (case["Hq"] + 2 * case["Hkv"]) * case["D"]
        turned = case["T"] * (case["Hq"] + case["Hkv"]) * case["rot"]
        return dict(bytes=2 * values * es + 4 * case["T"] * (case["rot"] + 2), flops=3 * turned)
    tokens = case["n"] * (case["page"] if op == "pages" else 1)
    return dict(bytes=4 * tokens * case["Hkv"] * case["D"] * es + 8 * case["n"], flops=0)


# ----------------------------------------------------------------------------------------------- exact
def _exact_attention(st):
    """By the definition, one key/value head at a time, gradients by 64-bit automatic differentiation."""
    c = st["case"]
    train = c["op"] == "train"
    group = c["Hq"] // c["Hkv"]
    hide = ~_visible(c["S"], c["S"], c["window"], c["sinks"])
    names = ("o", "dq", "dk", "dv") if train else ("o", "lse")
    parts = {x: [] for x in names}
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            k, v = (st[x][b, h].double().requires_grad_(train) for x in ("k", "v"))
            dk, dv = torch.zeros_like(k), torch.zeros_like(v)
            for x in range(h * group, (h + 1) * group):
                q = st["q"][b, x].double().requires_grad_(train)
                s = (q / math.sqrt(c["D"])) @ k.T
                if c["softcap"] > 0:
                    s = c["softcap"] * torch.tanh(s / c["softcap"])
                s = s.masked_fill(hide, -math.inf)
                o = torch.softmax(s, -1) @ v
                parts["o"].append(o.detach())
                if train:
                    gq, gk, gv = torch.autograd.grad(o, (q, k, v), st["do"][b, x].double())
                    parts["dq"].append(gq)
                    dk += gk
                    dv += gv
                else:
                    parts["lse"].append(torch.logsumexp(s, -1, keepdim=True))
            if train:
                parts["dk"].append(dk)
                parts["dv"].append(dv)
    return {x: torch.stack(p).view(c["B"], len(p) // c["B"], c["S"], -1) for x, p in parts.items()}


def _exact_decode(st):
    c = st["case"]
    outs, lses = [], []
    for r, n in enumerate(st["lens"].tolist()):
        tok = [t for t in range(n) if t >= n - c["window"] or t < c["sinks"]]
        if not tok:
            outs.append(torch.zeros(c["Hq"], c["D"], dtype=torch.float64, device="cuda"))
            lses.append(torch.full((c["Hq"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        tok = torch.tensor(tok, device="cuda")
        page = st["bt"][r, tok // c["page"]].long()
        k, v = (st[x][page, :, tok % c["page"]].double().transpose(0, 1).repeat_interleave(c["Hq"] // c["Hkv"], 0)
                for x in ("kp", "vp"))  # [Hq, tokens, D]
        s = (k @ st["q"][r].double()[:, :, None])[..., 0] / math.sqrt(c["D"])
        if c["softcap"] > 0:
            s = c["softcap"] * torch.tanh(s / c["softcap"])
        outs.append((torch.softmax(s, -1)[:, None] @ v)[:, 0])
        lses.append(torch.logsumexp(s, -1))
    return dict(o=torch.stack(outs), lse=torch.stack(lses))


def _exact_rotate(x, cos, sin, layout, sign=1.0):
    """The pairs as complex numbers, multiplied by cos + i sin."""
    turn = torch.complex(cos.double(), sign * sin.double())
    half = turn.shape[-1]
    y = x.double().clone()
    if layout == "half":
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:2 * half:2].contiguous(), y[..., 1:2 * half:2].contiguous()) * turn
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    return y


def exact(case, seed):
    """Outputs in 64 bits; None for the copies, whose values are not computed."""
    op = case["op"]
    if op in ("pages", "tokens"):
        return None
    st = prepare(case, seed)
    if op in ("prefill", "train"):
        return _exact_attention(st)
    if op == "decode":
        return _exact_decode(st)
    if op == "rotary":
        cos, sin = (st[x][st["pos"].long()].unsqueeze(1) for x in ("cos", "sin"))
        return dict(q=_exact_rotate(st["q"], cos, sin, case["layout"]),
                    k=_exact_rotate(st["k"], cos, sin, case["layout"]),
                    dq=_exact_rotate(st["dq"], cos, sin, case["layout"], -1.0),
                    dk=_exact_rotate(st["dk"], cos, sin, case["layout"], -1.0))
    cos, sin = (st[x][st["pos"].long()].unsqueeze(1) for x in ("cos", "sin"))
    kp, vp = st["kp"].double(), st["vp"].double()
    k = _exact_rotate(st["k"], cos, sin, case["layout"])
    for t, slot in enumerate(st["slots"].tolist()):
        kp[slot // case["page"], :, slot % case["page"]] = k[t]
        vp[slot // case["page"], :, slot % case["page"]] = st["v"][t].double()
    return dict(q=_exact_rotate(st["q"], cos, sin, case["layout"]), kp=kp, vp=vp)
