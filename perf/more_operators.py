"""Measured cases of serving from a paged cache: block tables and slot maps built on the GPU from request lengths
(pages taken for new tokens, pages given back), decoding of requests that share a long prefix, and several new tokens
of each request (a chunk of a prompt, a few drafted tokens) against its pages.

``run`` computes a case with the package's kernels where ``own`` is true, and in a plain form of elementary torch
operations where it is false; ``exact`` gives the 64-bit result of the definition."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MAX_PAIRS = 32 * 2048 * 32768  # (query head, key) pairs of the largest attention case
_MAX_BYTES = 3 << 30  # keys and values of the largest case


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step's bookkeeping for a serving batch: every request gets a token, a few of them a page
        dict(name="tables step", op="assign", R=64, ctx_lo=512, ctx_hi=32768, new_lo=1, new_hi=1, page=16),
        # prompts of many lengths admitted at once: empty rows, some requests without a new token
        dict(name="tables prompts", op="assign", R=1024, ctx_lo=0, ctx_hi=700, new_lo=0, new_hi=256, page=64),
        # the requests of a batch that end with a step give their pages back
        dict(name="tables retire", op="release", R=64, ctx_lo=512, ctx_hi=32768, keep=0, page=16),
        # a large batch whose requests keep the pages of the prefix that they share
        dict(name="tables retire many", op="release", R=1021, ctx_lo=0, ctx_hi=2900, keep=96, page=24),
        # four samples of a short prompt on a small model: a call bound by latency
        dict(name="prefix few", op="prefix", dtype="fp16", R=4, groups=1, alone=0, Hq=8, Hkv=2, D=64, page=16,
             prefix_lo=200, prefix_hi=200, own_lo=1, own_hi=40, softcap=0.0),
        # a serving batch behind one system prompt, at the heads of the benchmark's paged decode
        dict(name="prefix batch", op="prefix", dtype="bf16", R=64, groups=1, alone=0, Hq=32, Hkv=8, D=128, page=16,
             prefix_lo=8192, prefix_hi=8192, own_lo=1, own_hi=1024, softcap=0.0),
        # many questions on one long document
        dict(name="prefix wide", op="prefix", dtype="bf16", R=256, groups=1, alone=0, Hq=32, Hkv=8, D=128, page=64,
             prefix_lo=32768, prefix_hi=32768, own_lo=1, own_hi=512, softcap=0.0),
        # three prefixes of odd lengths, requests without one, seven heads a group, head dim 96, a softcap
        dict(name="prefix groups", op="prefix", dtype="fp16", R=37, groups=3, alone=5, Hq=21, Hkv=3, D=96, page=24,
             prefix_lo=77, prefix_hi=4099, own_lo=0, own_hi=333, softcap=30.0),
        # a few tokens of a few short requests: a call bound by latency
        dict(name="prefill few", op="prefill", dtype="fp16", R=3, Hq=8, Hkv=2, D=64, page=16, old_lo=0, old_hi=100,
             new_lo=1, new_hi=7, softcap=0.0),
        # four drafted tokens of each request of a serving batch, verified at once
        dict(name="prefill drafts", op="prefill", dtype="bf16", R=64, Hq=32, Hkv=8, D=128, page=16, old_lo=512,
             old_hi=16384, new_lo=4, new_hi=4, softcap=0.0),
        # a chunk of a long prompt
        dict(name="prefill chunk", op="prefill", dtype="bf16", R=1, Hq=32, Hkv=8, D=128, page=64, old_lo=30720,
             old_hi=30720, new_lo=2048, new_hi=2048, softcap=0.0),
        # prompts of many lengths, some behind a cached context, heads without grouping
        dict(name="prefill ragged", op="prefill", dtype="fp16", R=9, Hq=20, Hkv=20, D=64, page=24, old_lo=0,
             old_hi=2900, new_lo=1, new_hi=1500, softcap=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the same operators, sizes over the whole range between one token and the largest case."""
    op = rng.choice(["assign", "release", "prefix", "prefix", "prefix", "prefill", "prefill", "prefill"])
    page = rng.choice([16, 24, 64, 128])
    if op == "assign":
        r = _log_int(rng, 1, 4096)
        lo = rng.choice([0, 1, 100])
        return dict(op=op, R=r, ctx_lo=lo, ctx_hi=lo + _log_int(rng, 1, min(32768, (1 << 22) // r)),
                    new_lo=rng.choice([0, 1]), new_hi=_log_int(rng, 1, max(1, (1 << 18) // r)), page=page)
    if op == "release":
        r = _log_int(rng, 1, 4096)
        return dict(op=op, R=r, ctx_lo=rng.choice([0, 1, 100]), ctx_hi=100 + _log_int(rng, 1, min(32768, (1 << 22) // r)),
                    keep=page * rng.choice([0, 0, 1, 3]), page=page)
    hkv = rng.choice([1, 2, 3, 5, 8])
    base = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), Hq=hkv * rng.choice([1, 2, 4, 4, 7, 8]), Hkv=hkv,
                D=rng.choice([64, 96, 128, 128]), page=page, softcap=rng.choice([0.0, 0.0, 30.0]))
    token = 4 * hkv * base["D"]  # bytes of a token's keys and values
    if op == "prefix":
        r = _log_int(rng, 1, 256)
        groups = min(r, rng.choice([1, 1, 2, 5]))
        prefix = _log_int(rng, 1, min(32768, _MAX_PAIRS // (base["Hq"] * r)))
        own_hi = _log_int(rng, 1, max(1, min(2048, _MAX_BYTES // (token * r))))
        alone = rng.choice([0, 0, r // 5])
        return dict(base, R=r, groups=min(groups, r - alone), alone=alone, prefix_lo=max(1, prefix // rng.choice([1, 3])),
                    prefix_hi=prefix, own_lo=rng.choice([0, 1]), own_hi=own_hi)
    r = _log_int(rng, 1, 64)
    new = _log_int(rng, 1, max(1, 2048 // r))
    old = _log_int(rng, 1, max(1, min(30000, _MAX_BYTES // (token * r), _MAX_PAIRS // (2 * base["Hq"] * r * new))))
    return dict(base, R=r, old_lo=rng.choice([0, old // 2]), old_hi=old, new_lo=rng.choice([1, new]), new_hi=new)


# -------------------------------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers, evenly over [lo, hi] (the seed decides their order alone)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _groups(case):
    """Sizes of the groups (each half the one before, the last requests alone) and their prefixes' lengths."""
    left, sizes = case["R"] - case["alone"], []
    for i in range(case["groups"]):
        last = i + 1 == case["groups"]
        size = left if last else max(1, min(left // 2, left - (case["groups"] - i - 1)))
        sizes.append(size)
        left -= size
    return sizes, _spread(case["groups"], case["prefix_lo"], case["prefix_hi"])


def _pages(n, page):
    return -(-n // page)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op, ps, r = case["op"], case["page"], case["R"]

    def mixed(values):
        return [values[i] for i in torch.randperm(len(values), generator=host).tolist()]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(_DTYPES[case["dtype"]])

    def tables(counts, width, shared=()):
        """[R, width] page ids in random order (-1 behind a request's own), and the ids left over; a request's first
        pages are those of the request that `shared` names, as (request, owner, pages)."""
        used = sum(counts) - sum(n for _, _, n in shared)
        ids = torch.randperm(used + spare, generator=host)
        first = {q: n for q, _, n in shared}
        bt = torch.full((r, width), -1, dtype=torch.int64)
        at = 0
        for i, c in enumerate(counts):
            n = c - first.get(i, 0)
            bt[i, c - n:c] = ids[at:at + n]
            at += n
        for q, owner, n in shared:
            bt[q, :n] = bt[owner, :n]
        return bt.to(torch.int32).cuda(), ids[at:], used + spare

    spare = 0
    if op in ("assign", "release"):
        lens = mixed(_spread(r, case["ctx_lo"], case["ctx_hi"]))
        new = mixed(_spread(r, case["new_lo"], case["new_hi"])) if op == "assign" else [0] * r
        counts = [_pages(n, ps) for n in lens]
        need = sum(_pages(n + m, ps) for n, m in zip(lens, new)) - sum(counts)
        spare = need + need // 4 + 7
        bt, free, total = tables(counts, max(1, max(_pages(n + m, ps) for n, m in zip(lens, new))))
        # the free pages lie in a ring that starts anywhere
        head = int(torch.randint(0, total, (1,), generator=host))
        ring = torch.full((total,), -1, dtype=torch.int64)
        ring[(head + torch.arange(len(free))) % total] = free
        st = dict(case=case, bt=bt, lens=_ints(lens), ring=ring.to(torch.int32).cuda(), state=_ints([head, len(free)]))
        if op == "assign":
            return dict(st, new=_ints(new), tokens=sum(new))
        done = torch.rand(r, generator=host) < 0.5
        done[0] = True
        return dict(st, done=done.cuda(), keep=_ints([min(case["keep"], n // ps * ps) for n in lens]))
    if op == "prefix":
        sizes, prefixes = _groups(case)
        own_lens, lens, starts, shared = mixed(_spread(r, case["own_lo"], case["own_hi"])), [], [0], []
        for size, n in zip(sizes, prefixes):
            first = len(lens)
            for i in range(size):
                lens.append(n + own_lens[len(lens)])
                if i:  # full pages are shared; a page that the prefix ends in is each request's own
                    shared.append((first + i, first, n // ps))
            starts.append(len(lens))
        lens += own_lens[len(lens):]
        bt, _, pages = tables([_pages(n, ps) for n in lens], max(1, _pages(max(lens), ps)), shared)
        kp, vp = (randn(max(pages, 1), case["Hkv"], ps, case["D"]) for _ in range(2))
        for first, end, n in zip(starts, starts[1:], prefixes):  # copies of the tokens in the prefix's last page
            if n % ps and end > first + 1:
                old, fresh = bt[first, n // ps].long(), bt[first + 1:end, n // ps].long()
                for pool in (kp, vp):
                    pool[fresh, :, :n % ps] = pool[old, :, :n % ps]
        return dict(case=case, q=randn(r, case["Hq"], case["D"]), kp=kp, vp=vp, bt=bt, lens=_ints(lens),
                    starts=_ints(starts), prefixes=_ints(prefixes), host=(lens, starts, prefixes))
    new, old = mixed(_spread(r, case["new_lo"], case["new_hi"])), mixed(_spread(r, case["old_lo"], case["old_hi"]))
    lens = [a + b for a, b in zip(old, new)]
    bt, _, pages = tables([_pages(n, ps) for n in lens], _pages(max(lens), ps))
    starts = [sum(new[:i]) for i in range(r + 1)]
    return dict(case=case, q=randn(starts[-1], case["Hq"], case["D"]), bt=bt, lens=_ints(lens), starts=_ints(starts),
                kp=randn(pages, case["Hkv"], ps, case["D"]), vp=randn(pages, case["Hkv"], ps, case["D"]),
                host=(lens, starts))


# ----------------------------------------------------------------------------------------- plain forms
def _plain_assign(st):
    ps, bt, ring = st["case"]["page"], st["bt"], st["ring"].long()
    lens, new = st["lens"].long(), st["new"].long()
    r, width = bt.shape
    old, end = -(-lens // ps), -(-(lens + new) // ps)
    need = end - old
    first = need.cumsum(0) - need
    at = torch.arange(width, device="cuda")[None, :]
    take = (st["state"][0].long() + first[:, None] + at - old[:, None]) % ring.numel()
    fresh = (at >= old[:, None]) & (at < end[:, None])
    bt.copy_(torch.where(fresh, ring[take], bt.long()))
    starts = torch.zeros(r + 1, dtype=torch.int64, device="cuda")
    starts[1:] = new.cumsum(0)
    tok = torch.arange(st["tokens"], device="cuda")
    row = torch.searchsorted(starts, tok, right=True) - 1
    pos = lens[row] + tok - starts[row]
    slots = bt[row, pos // ps].long() * ps + pos % ps
    total = need.sum()
    state = torch.stack([(st["state"][0] + total) % ring.numel(), st["state"][1] - total])
    out = dict(slots=slots, positions=pos, starts=starts, lens=lens + new, state=state)
    return dict({k: v.to(torch.int32) for k, v in out.items()}, table=bt)


def _plain_release(st):
    ps, bt, ring = st["case"]["page"], st["bt"].long(), st["ring"]
    lens, done = st["lens"].long(), st["done"]
    first, end = -(-st["keep"].long() // ps), -(-lens // ps)
    give = torch.where(done, (end - first).clamp(min=0), 0)
    upto = give.cumsum(0)
    # the i-th page given goes to the i-th place behind the ring's last free one
    i = (torch.arange(ring.numel(), device="cuda") - st["state"][0] - st["state"][1]) % ring.numel()
    row = torch.searchsorted(upto, i, right=True).clamp(max=bt.shape[0] - 1)
    at = (first[row] + i - upto[row] + give[row]).clamp(min=0, max=bt.shape[1] - 1)
    ring.copy_(torch.where(i < upto[-1], bt[row, at], ring.long()))
    state = torch.stack([st["state"][0], (st["state"][1] + upto[-1]).to(torch.int32)])
    return dict(ring=ring, lens=torch.where(done, 0, st["lens"]), state=state)


def _softmax_parts(s):
    """exp(s - max), its sum, and the maximum of the last axis; rows that see nothing give zeros and -inf."""
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    return p, p.sum(-1, keepdim=True), m


def _plain_scores(s, c):
    s = s.mul_(1.0 / math.sqrt(c["D"]))
    return torch.tanh(s / c["softcap"]).mul_(c["softcap"]) if c["softcap"] > 0 else s


def _plain_prefix(st):
    """Scores against the prefix from one product for each group, those against a request's own tokens from its own
    pages, one softmax over both."""
    c = st["case"]
    r, hq, hkv, d, ps = (c[x] for x in ("R", "Hq", "Hkv", "D", "page"))
    lens, starts, prefixes = st["host"]
    q = st["q"].float().view(r, hkv, hq // hkv, d)
    outs, lses = [], []
    bounds = list(zip(starts, starts[1:], prefixes)) + ([(starts[-1], r, 0)] if starts[-1] < r else [])
    for a, b, n in bounds:
        qg, ln = q[a:b], st["lens"][a:b].long()[:, None]
        own_max = max(lens[a:b]) - n
        tok = n + torch.arange(own_max, device="cuda")[None, :]
        seen = tok < ln
        page = st["bt"][a:b].long().gather(1, torch.where(seen, tok, 0) // ps).clamp(min=0)
        at = tok.expand_as(page) % ps
        k, v = (st[x][page, :, at].float() for x in ("kp", "vp"))  # [members, own, Hkv, D]
        s = _plain_scores(torch.einsum("rhgd,rthd->rhgt", qg, k), c).masked_fill_(~seen[:, None, None, :], -math.inf)
        if n:
            tokp = torch.arange(n, device="cuda")
            pg = st["bt"][a].long()[tokp // ps]
            kx, vx = (st[x][pg, :, tokp % ps].float() for x in ("kp", "vp"))  # [prefix, Hkv, D]
            s = torch.cat([_plain_scores(torch.einsum("rhgd,thd->rhgt", qg, kx), c), s], -1)
        if s.shape[-1] == 0:
            s = torch.full((*s.shape[:-1], 1), -math.inf, device="cuda")
            p, l, m = _softmax_parts(s)
            o = torch.zeros_like(qg)
        else:
            p, l, m = _softmax_parts(s)
            p = p.div_(torch.where(l > 0, l, 1.0))
            o = torch.einsum("rhgt,rthd->rhgd", p[..., n:], v)
            if n:
                o += torch.einsum("rhgt,thd->rhgd", p[..., :n], vx)
        outs.append(o.reshape(b - a, hq, d))
        lses.append((m + l.log()).reshape(b - a, hq))
    return dict(o=torch.cat(outs).to(st["q"].dtype), lse=torch.cat(lses))


def _plain_prefill(st):
    c = st["case"]
    hq, hkv, d, ps = (c[x] for x in ("Hq", "Hkv", "D", "page"))
    lens, starts = st["host"]
    outs, lses = [], []
    for i, n in enumerate(lens):
        new = starts[i + 1] - starts[i]
        tok = torch.arange(n, device="cuda")
        pg = st["bt"][i].long()[tok // ps]
        hide = tok[None, :] > n - new + torch.arange(new, device="cuda")[:, None]
        q = st["q"][starts[i]:starts[i + 1]].float().view(new, hkv, hq // hkv, d)
        k, v = (st[x][pg, :, tok % ps].float() for x in ("kp", "vp"))  # [n, Hkv, D]
        o = torch.empty(new, hkv, hq // hkv, d, device="cuda")
        lse = torch.empty(new, hkv, hq // hkv, device="cuda")
        for h in range(hkv):
            s = _plain_scores(torch.einsum("ngd,td->gnt", q[:, h], k[:, h]), c).masked_fill_(hide, -math.inf)
            p, l, m = _softmax_parts(s)
            o[:, h] = torch.einsum("gnt,td->ngd", p.div_(l), v[:, h])
            lse[:, h] = (m + l.log())[..., 0].transpose(0, 1)
        outs.append(o.reshape(new, hq, d))
        lses.append(lse.reshape(new, hq))
    return dict(o=torch.cat(outs).to(st["q"].dtype), lse=torch.cat(lses))


_PLAIN = dict(assign=_plain_assign, release=_plain_release, prefix=_plain_prefix, prefill=_plain_prefill)


def run(st):
    c = st["case"]
    if not own:
        with torch.no_grad():
            return _PLAIN[c["op"]](st)
    import fastest_flash_attention_b200 as ffa

    if c["op"] == "assign":
        plan = ffa.assign_slots(st["bt"], st["lens"], st["new"], st["ring"], st["state"], page_size=c["page"],
                                max_tokens=st["tokens"])
        return dict(slots=plan.slots, positions=plan.positions, starts=plan.starts, lens=plan.ctx_lens,
                    state=plan.free_state, table=st["bt"])
    if c["op"] == "release":
        lens, state = ffa.release_pages(st["bt"], st["lens"], st["done"], st["ring"], st["state"],
                                        page_size=c["page"], keep=st["keep"])
        return dict(ring=st["ring"], lens=lens, state=state)
    if c["op"] == "prefix":
        o, lse = ffa.prefix_decode(st["q"], st["kp"], st["vp"], st["bt"], st["lens"], st["starts"], st["prefixes"],
                                   softcap=c["softcap"] or None, return_lse=True, max_prefix=c["prefix_hi"],
                                   max_own=c["own_hi"])
        return dict(o=o, lse=lse)
    o, lse = ffa.paged_prefill(st["q"], st["kp"], st["vp"], st["bt"], st["lens"], st["starts"],
                               softcap=c["softcap"] or None, return_lse=True, max_ctx=max(st["host"][0]))
    return dict(o=o, lse=lse)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, r, ps = case["op"], case["R"], case["page"]
    if op in ("assign", "release"):
        lens = _spread(r, case["ctx_lo"], case["ctx_hi"])
        if op == "release":  # lengths and marks read, lengths written; about half of the pages read and written
            return dict(bytes=13 * r + 4 * sum(max(0, _pages(n, ps) - case["keep"] // ps) for n in lens), flops=0)
        tokens = sum(_spread(r, case["new_lo"], case["new_hi"]))
        # lengths read and written, starts, a slot and a position for each token, an id read and written for each page
        return dict(bytes=16 * r + 8 * tokens + 8 * (tokens // ps), flops=0)
    hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
    if op == "prefix":
        sizes, prefixes = _groups(case)
        mine = sum(_spread(r, case["own_lo"], case["own_hi"]))
        seen = mine + sum(s * n for s, n in zip(sizes, prefixes))
        return dict(bytes=4 * (mine + sum(prefixes)) * hkv * d + r * hq * (4 * d + 4), flops=4 * seen * hq * d)
    old, new = _spread(r, case["old_lo"], case["old_hi"]), _spread(r, case["new_lo"], case["new_hi"])
    mean_old = sum(old) / r  # which old context goes with which new tokens is the seed's
    pairs = sum(n * mean_old + n * (n + 1) / 2 for n in new)
    return dict(bytes=4 * (sum(old) + sum(new)) * hkv * d + sum(new) * hq * (4 * d + 4),
                flops=int(4 * pairs * hq * d))


# ----------------------------------------------------------------------------------------------- exact
def _exact_row(st, row, q, limits):
    """q [n, Hq, D] of one request over its first tokens: query i sees the first limits[i] of them."""
    c = st["case"]
    group, ps = c["Hq"] // c["Hkv"], c["page"]
    n = max(limits)
    if n == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64,
                                                                    device="cuda")
    pages = st["bt"][row, :_pages(n, ps)].long()
    hide = torch.arange(n, device="cuda")[None, :] >= torch.tensor(limits, device="cuda")[:, None]
    o, lse = torch.empty(q.shape, dtype=torch.float64, device="cuda"), []
    for h in range(c["Hkv"]):
        k, v = (st[x][pages, h].reshape(-1, c["D"])[:n].double() for x in ("kp", "vp"))
        for x in range(h * group, (h + 1) * group):
            s = q[:, x].double() @ k.T / math.sqrt(c["D"])
            if c["softcap"] > 0:
                s = c["softcap"] * torch.tanh(s / c["softcap"])
            s = s.masked_fill(hide, -math.inf)
            o[:, x] = torch.softmax(s, -1) @ v
            lse.append(torch.logsumexp(s, -1))
    return o, torch.stack(lse, 1)


def exact(case, seed):
    """Outputs in 64 bits; None for the tables, whose values are whole numbers."""
    op = case["op"]
    if op in ("assign", "release"):
        return None
    st = prepare(case, seed)
    lens, starts = st["host"][:2]
    parts = []
    for i, n in enumerate(lens):
        if op == "prefix":
            parts.append(_exact_row(st, i, st["q"][i:i + 1], [n]))
        else:
            new = starts[i + 1] - starts[i]
            parts.append(_exact_row(st, i, st["q"][starts[i]:starts[i + 1]], [n - new + 1 + j for j in range(new)]))
    return dict(o=torch.cat([p[0] for p in parts]), lse=torch.cat([p[1] for p in parts]))
