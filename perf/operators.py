"""What the operators of the 8-bit KV cache cost: WriteKv8, AttentionKv8, ScoreKv8 and EvictKv8.

Each case is one call of one operator on inputs a decoder has at that point: a cache of pages of 64
tokens whose keys and values are int8 or e4m3 codes with an f32 scale for each block of tokens and
KV head, and a batch of sequences described by device tables. With ``own`` false the operators are
computed by elementary torch operations in 32 bits, with ``own`` true by this package: `run` then enqueues on
the backend's stream, and its outputs are there once that stream (``HipBackend.sync``) or the device was waited for."""
import math

import numpy as np
import torch

own = False

PAGE = 64
FLOOR = 2.0 ** -96          # smallest scale
CODE_MAX = {"i8": 127.0, "f8": 448.0}


# ---------------------------------------------------------------- cases

def _lens(case):
    """Tokens each sequence has cached, this call's among them: from `low` to `high`, spread evenly in
    the logarithm, in an order that mixes long and short ones, none of them rounded to a page."""
    n, lo, hi = case["n_seq"], case["low"], case["high"]
    if n == 1:
        return [hi]
    out = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    step = next(k for k in (7, 5, 3, 11, 1) if math.gcd(k, n) == 1)
    return [out[(i * step) % n] for i in range(n)]


def _news(case):
    """Rows of each sequence in this call: `rows` of them, or the whole sequence where that is 0."""
    return [min(l, case["rows"]) if case["rows"] else l for l in _lens(case)]


def listed():
    return [
        # one decode step of a full batch: every sequence appends one token
        dict(name="write-step", op="write", type="i8", block=16, n_seq=64, low=100, high=2000, rows=1, n_kv=8, dim=128),
        # four prompts of different lengths written in one chunk
        dict(name="write-prompt", op="write", type="f8", block=64, n_seq=4, low=900, high=3500, rows=0, n_kv=8, dim=128),
        # one user, one token, a short conversation: latency
        dict(name="attend-one", op="attend", type="i8", block=16, n_seq=1, low=700, high=700, rows=1, n_head=32, n_kv=8,
             dim=128, softcap=0.0, window=0, slopes=False, docs=0, prefix=0),
        # a decode step of a full batch with conversations of 500 to 8000 tokens
        dict(name="attend-step", op="attend", type="i8", block=16, n_seq=64, low=500, high=8000, rows=1, n_head=32, n_kv=8,
             dim=128, softcap=0.0, window=0, slopes=False, docs=0, prefix=0),
        # two long documents being answered on: few rows over a very long axis
        dict(name="attend-far", op="attend", type="f8", block=64, n_seq=2, low=100003, high=131071, rows=1, n_head=32, n_kv=4,
             dim=128, softcap=0.0, window=0, slopes=False, docs=0, prefix=0),
        # four drafted tokens per sequence being verified in a layer with a sliding window and capped scores
        dict(name="attend-draft", op="attend", type="i8", block=32, n_seq=16, low=300, high=5000, rows=4, n_head=16, n_kv=8,
             dim=256, softcap=50.0, window=1024, slopes=False, docs=0, prefix=0),
        # a prompt of 4096 tokens
        dict(name="attend-prompt", op="attend", type="i8", block=64, n_seq=1, low=4096, high=4096, rows=0, n_head=32, n_kv=8,
             dim=128, softcap=0.0, window=0, slopes=False, docs=0, prefix=0),
        # prompts that pack several documents, with a prefix seen from everywhere in them and a bias by distance
        dict(name="attend-packed", op="attend", type="f8", block=64, n_seq=3, low=700, high=2501, rows=0, n_head=16, n_kv=16,
             dim=80, softcap=0.0, window=0, slopes=True, docs=5, prefix=100),
        # the sums of attention weights after a decode step
        dict(name="score-step", op="score", type="i8", block=16, n_seq=32, low=1000, high=8000, rows=1, n_head=32, n_kv=8,
             dim=128, softcap=0.0, window=0, slopes=False, docs=0, prefix=0, decay=1.0),
        # the same after the last chunk of a prompt
        dict(name="score-prompt", op="score", type="f8", block=64, n_seq=1, low=4001, high=4001, rows=1000, n_head=32, n_kv=4,
             dim=128, softcap=30.0, window=0, slopes=False, docs=0, prefix=0, decay=0.5),
        # a short cache that has grown over its budget by a few tokens
        dict(name="evict-little", op="evict", type="i8", block=16, n_seq=4, low=1050, high=1100, n_kv=8, dim=128, keep=1024,
             sink=4, recent=256),
        # long prompts cut down to what decoding will keep
        dict(name="evict-deep", op="evict", type="f8", block=64, n_seq=8, low=9000, high=32000, n_kv=8, dim=128, keep=4096,
             sink=16, recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write", "attend", "attend", "attend", "attend", "score", "evict"])
    n_kv = rng.choice([1, 2, 4, 8, 16])
    c = dict(op=op, type=rng.choice(["i8", "f8"]), block=rng.choice([16, 32, 64]), n_kv=n_kv,
             dim=rng.choice([64, 128, 128, 256, rng.randrange(33, 256)]))
    if op == "write":
        decode = rng.random() < 0.5
        c["n_seq"] = _log(rng, 1, 200) if decode else rng.randrange(1, 5)
        c["high"] = _log(rng, 40, 3500)
        c["low"] = max(1, int(c["high"] * rng.uniform(0.1, 1.0)))
        c["rows"] = 1 if decode else 0
        return c
    if op == "evict":
        c["n_seq"] = rng.randrange(1, 9)
        c["high"] = _log(rng, 300, 30000)
        c["low"] = max(200, int(c["high"] * rng.uniform(0.3, 1.0)))
        c["keep"] = rng.randrange(64, 4097)
        c["sink"] = rng.randrange(0, 9)
        c["recent"] = rng.randrange(0, c["keep"] // 2)
        return c
    few = rng.random() < 0.6
    c["n_head"] = n_kv * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if g * n_kv <= 48])
    if few:  # decode and drafts
        c["n_seq"], c["rows"] = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7])
        c["high"] = _log(rng, 100, 60000 // c["n_seq"] + 500)
    else:    # chunks of prompts and whole ones
        c["n_seq"] = rng.randrange(1, 4)
        c["high"] = _log(rng, 100, 3500 // c["n_seq"] + 300)
        c["rows"] = rng.choice([0, 0, c["high"] // 2 + 1])
    c["low"] = max(1, int(c["high"] * rng.uniform(0.2, 1.0)))
    c["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    c["window"] = rng.choice([0, 0, _log(rng, 30, 2000)])
    c["slopes"] = rng.random() < 0.3
    c["docs"] = rng.choice([0, 0, rng.randrange(2, 7)])
    c["prefix"] = rng.choice([0, 0, rng.randrange(1, 200)])
    if op == "score":
        c["decay"] = rng.choice([1.0, 0.5])
    return c


# ---------------------------------------------------------------- the cache's layout

def _padded(dim):
    return -(-dim // 64) * 64


def _regions(n_pages, n_kv, dim, n_slots, block):
    """Byte offset, type and shape of the parts of a cache buffer, each on a multiple of 256 bytes."""
    dp, sub = _padded(dim), PAGE // block
    parts = [("k", torch.uint8, (n_pages, n_kv, dp // 64, PAGE, 64)), ("v", torch.uint8, (n_pages, n_kv, dp, PAGE)),
             ("k_scale", torch.float32, (n_pages, n_kv, sub)), ("v_scale", torch.float32, (n_pages, n_kv, sub)),
             ("pos", torch.int32, (n_pages, n_kv, PAGE)), ("sums", torch.float32, (n_pages, n_kv, PAGE)),
             ("tail", torch.float32, (n_slots, n_kv, 2, block, dim)), ("tag", torch.int32, (n_slots, n_kv, 2, 2))]
    at, out = 0, {}
    for name, t, shape in parts:
        size = math.prod(shape) * (1 if t == torch.uint8 else 4)
        out[name] = (at, size, t, shape)
        at += -(-size // 256) * 256
    return out, at


def _views(cache, regions):
    return {n: cache[at:at + size].view(t).view(shape) for n, (at, size, t, shape) in regions.items()}


def _encode(x, scale, type_):
    y = x / scale
    return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8) if type_ == "i8" else y.to(torch.float8_e4m3fn).view(torch.uint8)


def _typed(codes, type_):
    return codes.view(torch.int8 if type_ == "i8" else torch.float8_e4m3fn)


def _decode(codes, type_):
    return _typed(codes, type_).float()


def _wide(codes):
    """Rows of key codes [..., dim] as the cache holds them: [..., columns / 64, 64], zeros behind the last."""
    return torch.nn.functional.pad(codes, (0, _padded(codes.shape[-1]) - codes.shape[-1])).unflatten(-1, (-1, 64))


# ---------------------------------------------------------------- what the caller has in hand

def _slopes(n_head, dev):
    return torch.pow(2.0, -8.0 * torch.arange(1, n_head + 1, device=dev, dtype=torch.float32) / n_head)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rand = np.random.RandomState(int(seed) % (1 << 31))
    lens = _lens(case)
    news = _news(case) if case["op"] != "evict" else [0] * len(lens)
    n_seq, n_kv, dim, block, type_ = case["n_seq"], case["n_kv"], case["dim"], case["block"], case["type"]
    max_pages = -(-max(lens) // PAGE)
    counts = [-(-l // PAGE) for l in lens]
    keep = case.get("keep", 0)
    out_pages = -(-keep // PAGE)
    n_pages = sum(counts) + 3 + (out_pages * n_seq if keep else 0)
    order = rand.permutation(n_pages)
    pages = np.full((n_seq, max_pages), -1, np.int32)
    for s, n in enumerate(counts):
        pages[s, :n], order = order[:n], order[n:]
    regions, size = _regions(n_pages, n_kv, dim, n_seq, block)
    cache = torch.zeros(size, dtype=torch.uint8, device=dev)
    view = _views(cache, regions)
    # every page holds values: those behind a sequence's end are what an earlier one left there. Channels
    # of keys differ in size, as they do in trained models
    amp = torch.exp(0.5 * torch.randn(n_kv, 1, dim, device=dev, generator=g))
    for part in ("k", "v"):
        for p in range(0, n_pages, 256):
            n = min(256, n_pages - p)
            x = torch.randn(n, n_kv, PAGE, dim, device=dev, generator=g)
            if part == "k":
                x *= amp
            amax = x.view(n, n_kv, PAGE // block, block * dim).abs().amax(-1)
            scale = (amax / CODE_MAX[type_]).clamp_min(FLOOR)
            codes = _encode(x, scale.repeat_interleave(block, -1)[..., None], type_)
            if part == "k":
                view["k"][p:p + n] = _wide(codes).transpose(2, 3)
            else:
                view["v"][p:p + n, :, :dim, :] = codes.transpose(2, 3)
            view[part + "_scale"][p:p + n] = scale
    for s, n in enumerate(counts):
        at = torch.from_numpy(pages[s, :n].astype(np.int64)).to(dev)
        view["pos"][at] = torch.arange(n * PAGE, device=dev, dtype=torch.int32).view(n, 1, PAGE).expand(n, n_kv, PAGE)
    view["sums"].copy_(torch.rand(view["sums"].shape, device=dev, generator=g) ** 4)
    m = sum(news)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)  # noqa: E731
    st = {"case": dict(case), "cache": cache, "view": view, "pages": i32(pages), "lens": i32(lens),
          "max_len": max(lens), "max_q": max(news), "m": m, "n_pages": n_pages}
    start = np.concatenate([[0], np.cumsum(news)])
    st["q_start"] = i32(start)
    pos = np.concatenate([np.arange(l - n, l) for l, n in zip(lens, news)]) if m else np.zeros(1)
    st["pos"] = i32(pos)
    if case["op"] == "write":
        st["k"] = torch.randn(m, n_kv * dim, device=dev, generator=g) * amp.expand(n_kv, 1, dim).reshape(1, -1)
        st["v"] = torch.randn(m, n_kv * dim, device=dev, generator=g)
        st["slots"] = i32(rand.permutation(n_seq))
        for s, (l, n) in enumerate(zip(lens, news)):  # the open block's rows, as earlier steps have left them
            have = (l - n) % block
            if have:
                first = (l - n) // block * block
                page, sub = int(pages[s, first // PAGE]), first % PAGE // block
                slot = int(st["slots"][s])
                raw = torch.randn(n_kv, 2, have, dim, device=dev, generator=g)
                raw[:, 0] *= amp
                view["tail"][slot, :, :, :have] = raw
                view["tag"][slot, :, :, 0] = page * (PAGE // block) + sub
                view["tag"][slot, :, :, 1] = have
    elif case["op"] in ("attend", "score"):
        n_head = case["n_head"]
        st["q"] = torch.randn(m, n_head * dim, device=dev, generator=g)
        st["scale"] = 1.0 / math.sqrt(dim)
        st["slopes"] = _slopes(n_head, dev) if case["slopes"] else None
        if case["docs"]:  # a sequence holds `docs` documents; a row sees from its own one's start on
            first = []
            for l, n in zip(lens, news):
                cuts = np.sort(rand.randint(0, l, case["docs"] - 1))
                cuts = np.concatenate([[0], cuts])
                first.append(cuts[np.searchsorted(cuts, np.arange(l - n, l), side="right") - 1])
            st["first"] = i32(np.concatenate(first))
        else:
            st["first"] = None
        st["prefix"] = i32(np.minimum(case["prefix"], np.array(lens))) if case["prefix"] else None
        st["out"] = torch.empty(m, n_head * dim, device=dev)
        st["lse"] = torch.empty(m, n_head, device=dev)
        if case["op"] == "score":
            _plain_attend(st, weights=False)
    else:
        po = np.full((n_seq, out_pages), -1, np.int32)
        for s in range(n_seq):
            po[s], order = order[:out_pages], order[out_pages:]
        st["pages_out"] = i32(po)
        st["lens_out"] = torch.zeros(n_seq, dtype=torch.int32, device=dev)
        st["kept"] = torch.zeros(n_seq, n_kv, keep, dtype=torch.int32, device=dev)
    if own:
        _handles(st)
        # the backend has a stream of its own, which does not wait for torch's: what is in hand is finished
        torch.cuda.current_stream().synchronize()
    return st


# ---------------------------------------------------------------- the plain forms

def _rows_of(st):
    """Sequence and cache slot of each row."""
    start, lens = st["q_start"].long(), st["lens"].long()
    r = torch.arange(st["m"], device=start.device)
    s = torch.searchsorted(start[1:].contiguous(), r, right=True)
    return s, lens[s] - start[s + 1] + r


def _plain_write(st):
    c, view, block, type_ = st["case"], st["view"], st["case"]["block"], st["case"]["type"]
    n_kv, dim, sub = c["n_kv"], c["dim"], PAGE // c["block"]
    seq, slot = _rows_of(st)
    start, lens, pages, slots = st["q_start"].long(), st["lens"].long(), st["pages"].long(), st["slots"].long()
    n_new = start[1:] - start[:-1]
    begin = lens - n_new
    blk = slot // block
    first_blk = begin // block
    have = begin % block
    j = torch.arange(block, device=pages.device)
    page = pages[seq, slot // PAGE]
    fpage = pages.gather(1, (first_blk * block // PAGE).clamp_max(pages.shape[1] - 1)[:, None])[:, 0]
    fsub = first_blk * block % PAGE // block
    old = j[None, :] < have[:, None]
    raw = view["tail"][slots]                                   # [n_seq, n_kv, 2, block, dim]
    last_blk = (lens - 1) // block
    for part, name in enumerate(("k", "v")):
        x = st[name].view(st["m"], n_kv, dim)
        table = torch.zeros(c["n_seq"], -(-st["max_len"] // block), n_kv, device=x.device)
        keep = torch.where(old[:, None, :, None], raw[:, :, part], torch.zeros((), device=x.device))
        table.scatter_(1, first_blk.clamp_max(table.shape[1] - 1)[:, None, None].expand(-1, 1, n_kv), keep.abs().amax((2, 3))[:, None])
        flat = (seq * table.shape[1] + blk)[:, None].expand(-1, n_kv)
        table.view(-1, n_kv).scatter_reduce_(0, flat, x.abs().amax(-1), "amax")
        scale = (table / CODE_MAX[type_]).clamp_min(FLOOR)
        mine = scale[seq, blk]
        codes = _encode(x, mine[..., None], type_)
        s_old, j_old = torch.nonzero(old, as_tuple=True)
        again = _encode(keep[s_old, :, j_old], scale[s_old, first_blk[s_old]][..., None], type_)
        at_old = fsub[s_old] * block + j_old
        if name == "k":
            view["k"][page, :, :, slot % PAGE] = _wide(codes)
            view["k"][fpage[s_old], :, :, at_old] = _wide(again)
        else:
            view["v"][page, :, :dim, slot % PAGE] = codes
            view["v"][fpage[s_old], :, :dim, at_old] = again
        view[name + "_scale"][page, :, slot % PAGE // block] = mine
        is_last = torch.nonzero(blk == last_blk[seq])[:, 0]
        view["tail"][slots[seq[is_last]], :, part, slot[is_last] % block] = x[is_last]
    view["pos"][page, :, slot % PAGE] = st["pos"][:, None].expand(-1, n_kv)
    view["sums"][page, :, slot % PAGE] = 0.0
    lpage = pages.gather(1, (last_blk * block // PAGE)[:, None])[:, 0]
    tag = torch.stack([lpage * sub + last_blk * block % PAGE // block, (lens - 1) % block + 1], -1).int()
    view["tag"][slots] = tag[:, None, None, :].expand(-1, n_kv, 2, -1)


def _gathered(st):
    """Keys, values and positions of every sequence side by side: [n_seq, n_kv, L, dim], [n_seq, n_kv, L]."""
    c, view = st["case"], st["view"]
    n = -(-st["max_len"] // PAGE)
    at = st["pages"][:, :n].long().clamp_min(0)
    rep = c["block"]
    scale = lambda x: x[at].permute(0, 2, 1, 3).repeat_interleave(rep, -1).flatten(2)[..., None]  # noqa: E731
    k = _decode(view["k"][at].permute(0, 2, 1, 4, 3, 5).flatten(-2)[..., :c["dim"]], c["type"]).flatten(2, 3) * scale(view["k_scale"])
    v = _decode(view["v"][at][..., :c["dim"], :], c["type"]).permute(0, 2, 1, 4, 3).flatten(2, 3) * scale(view["v_scale"])
    return k, v, view["pos"][at].permute(0, 2, 1, 3).flatten(2)


def _plain_attend(st, weights):
    """Attention of all sequences, padded to the longest: fills out and lse, and gives the weights on request."""
    c = st["case"]
    n_kv, dim, n_head = c["n_kv"], c["dim"], c["n_head"]
    group = n_head // n_kv
    k, v, kpos = _gathered(st)
    dev, n_seq, length = k.device, c["n_seq"], k.shape[2]
    start, lens = st["q_start"].long(), st["lens"].long()
    n_new = start[1:] - start[:-1]
    i = torch.arange(st["max_q"], device=dev)
    real = i[None] < n_new[:, None]
    row = torch.where(real, start[:-1, None] + i[None], torch.zeros((), dtype=torch.long, device=dev))
    q = st["q"].view(st["m"], n_kv, group, dim)[row].permute(0, 2, 3, 1, 4).reshape(n_seq, n_kv, -1, dim)
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
    s = s.view(n_seq, n_kv, group, st["max_q"], length)
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    qpos = st["pos"].long()[row][:, None, :, None]
    apart = qpos - kpos.long()[:, :, None, :]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(n_kv, group)[None, :, :, None, None] * apart.abs().float()[:, :, None]
    at = torch.arange(length, device=dev)
    seen = at[None, None, :] <= (lens - n_new)[:, None, None] + i[None, :, None]
    seen = seen[:, None].expand(-1, n_kv, -1, -1)
    if st["prefix"] is not None:
        seen = seen | (kpos[:, :, None, :] < st["prefix"][:, None, None, None])
    seen = seen & (at[None, None, None, :] < lens[:, None, None, None]) & real[:, None, :, None]
    if c["window"]:
        seen = seen & (apart < c["window"])
    if st["first"] is not None:
        seen = seen & (kpos[:, :, None, :] >= st["first"][row][:, None, :, None])
    s = s.masked_fill(~seen[:, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros((), device=dev)))
    total = p.sum(-1, keepdim=True)
    keep_s, keep_i = torch.nonzero(real, as_tuple=True)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(n_seq, -1, n_head)
    st["lse"].copy_(lse[keep_s, keep_i])
    if weights:
        p = torch.exp(s - st["lse"][row].view(n_seq, -1, n_kv, group).permute(0, 2, 3, 1)[..., None])
        return p.masked_fill(~seen[:, :, None], 0.0).sum((2, 3))
    out = torch.matmul(p.view(n_seq, n_kv, -1, length), v).view(n_seq, n_kv, group, -1, dim) / torch.where(total > 0, total, torch.ones((), device=dev))
    out = out.permute(0, 3, 1, 2, 4).reshape(n_seq, -1, n_head * dim)
    st["out"].copy_(out[keep_s, keep_i])
    return None


def _plain_score(st):
    c, sums = st["case"], st["view"]["sums"]
    got = _plain_attend(st, weights=True)                          # [n_seq, n_kv, L]
    at = torch.arange(got.shape[2], device=got.device)
    s, j = torch.nonzero(at[None] < st["lens"][:, None], as_tuple=True)
    page = st["pages"].long()[s, j // PAGE]
    sums[page, :, j % PAGE] = c["decay"] * sums[page, :, j % PAGE] + got[s, :, j]


def _plain_evict(st):
    c, view, block, type_ = st["case"], st["view"], st["case"]["block"], st["case"]["type"]
    n_kv, dim, keep = c["n_kv"], c["dim"], c["keep"]
    lens, pages, pages_out = st["lens"].long(), st["pages"].long(), st["pages_out"].long()
    n = -(-st["max_len"] // PAGE)
    sums = view["sums"][pages[:, :n].clamp_min(0)].permute(0, 2, 1, 3).flatten(2)
    j = torch.arange(sums.shape[2], device=sums.device)
    end = lens[:, None, None]
    must = (j < c["sink"]) | (j >= end - c["recent"])
    rank = torch.where(must, torch.full_like(sums, math.inf), sums)
    rank = torch.where(j < end, rank, torch.full_like(sums, -math.inf))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    n_out = lens.clamp_max(keep)
    i = torch.arange(keep, device=sums.device)
    pad = keep - best.shape[-1]
    best = torch.nn.functional.pad(best, (0, pad)) if pad > 0 else best
    far = sums.shape[2] + keep
    src = torch.where(i < n_out[:, None, None], best, torch.full_like(best, far)).sort(-1).values
    live = i < n_out[:, None, None]
    st["kept"].copy_(torch.where(live, src, torch.full_like(src, -1)))
    st["lens_out"].copy_(n_out)
    src = torch.where(live, src, torch.zeros_like(src))
    # the kept tokens, block by block of where they go
    nb = -(-keep // block)
    fill = nb * block - keep
    src = torch.nn.functional.pad(src, (0, fill)).view(c["n_seq"], n_kv, nb, block)
    live = torch.nn.functional.pad(live.expand(-1, n_kv, -1), (0, fill)).view(c["n_seq"], n_kv, nb, block)
    seq = torch.arange(c["n_seq"], device=src.device)[:, None, None, None]
    head = torch.arange(n_kv, device=src.device)[None, :, None, None]
    page = pages[seq, src // PAGE].clamp_min(0)
    slot = src % PAGE
    tok = torch.arange(nb * block, device=src.device).view(nb, block)
    to = pages_out[seq, (tok // PAGE)[None, None]].expand_as(src)
    lead = src[..., :1]
    whole = ((src == lead + torch.arange(block, device=src.device)) | ~live).all(-1) & (lead[..., 0] % block == 0) & live[..., 0]
    w = torch.nonzero(live, as_tuple=True)
    at = (to[w], w[1], tok[w[2], w[3]] % PAGE)
    for name in ("k", "v"):
        old = view[name + "_scale"][page, head, slot // block]
        codes = view["k"][page, head, :, slot].flatten(-2)[..., :dim] if name == "k" else view["v"][page, head, :dim, slot]
        x = _decode(codes, type_) * old[..., None]
        amax = torch.where(live[..., None], x.abs(), torch.zeros((), device=x.device)).amax((-1, -2))
        new = torch.where(whole, old[..., 0], (amax / CODE_MAX[type_]).clamp_min(FLOOR))
        fresh = torch.where(whole[..., None, None], codes, _encode(x, new[..., None, None], type_))
        if name == "k":
            view["k"][at[0], at[1], :, at[2]] = _wide(fresh[w])
        else:
            view["v"][at[0], at[1], :dim, at[2]] = fresh[w]
        view[name + "_scale"][at[0], at[1], at[2] // block] = new[..., None].expand_as(src)[w]
    for name in ("pos", "sums"):
        view[name][at] = view[name][page[w], w[1], slot[w]]


# ---------------------------------------------------------------- the framework's calls

_backend = None


def _handles(st):
    """The plan and bindings a runner keeps for this step."""
    global _backend
    import infr_amd as I
    if _backend is None:
        _backend = I.HipBackend(0)
    be, c = _backend, st["case"]
    geom = I.Kv8(n_pages=st["n_pages"], n_kv=c["n_kv"], head_dim=c["dim"], n_slots=c["n_seq"], block=c["block"],
                 dtype=I.DType.I8 if c["type"] == "i8" else I.DType.F8E4M3)
    g, binds = I.Graph(), I.Bindings()

    def bound(t, kind="input"):
        if t is None:
            return None
        dt = I.DType.F32 if t.dtype == torch.float32 else I.DType.I32 if t.dtype == torch.int32 else I.DType.I8
        tid = getattr(g, kind)(I.TensorDesc(tuple(t.shape), dt))
        binds.bind(tid, be.wrap(t.data_ptr(), t.numel() * t.element_size()))
        return tid

    cache = bound(st["cache"])
    pages, lens = bound(st["pages"]), bound(st["lens"])
    if c["op"] == "evict":
        g.push(I.EvictKv8(cache, pages, lens, bound(st["pages_out"]), bound(st["lens_out"], "output"), bound(st["kept"], "output"),
                          geom, n_seq=c["n_seq"], max_pages=st["pages"].shape[1], keep=c["keep"], sink=c["sink"], recent=c["recent"]))
    else:
        batch = I.Kv8Batch(rows=st["m"], n_seq=c["n_seq"], max_q=st["max_q"], max_pages=st["pages"].shape[1])
        pos, start = bound(st["pos"]), bound(st["q_start"])
        if c["op"] == "write":
            g.push(I.WriteKv8(bound(st["k"]), bound(st["v"]), cache, pos, pages, start, lens, bound(st["slots"]), geom, batch))
        else:
            mode = dict(n_head=c["n_head"], scale=st["scale"], softcap=c["softcap"], window=c["window"], first=bound(st["first"]),
                        prefix=bound(st["prefix"]), slopes=bound(st["slopes"]))
            if c["op"] == "attend":
                g.push(I.AttentionKv8(bound(st["q"]), cache, bound(st["out"], "output"), pos, pages, start, lens, geom, batch,
                                      lse=bound(st["lse"], "output"), **mode))
            else:
                g.push(I.ScoreKv8(bound(st["q"]), cache, bound(st["lse"]), pos, pages, start, lens, geom, batch, decay=c["decay"], **mode))
    st["plan"], st["binds"] = be.compile(g), binds


def run(state):
    c, view = state["case"], state["view"]
    op = c["op"]
    if own:
        _backend.execute(state["plan"], state["binds"])
    elif op == "write":
        _plain_write(state)
    elif op == "attend":
        _plain_attend(state, weights=False)
    elif op == "score":
        _plain_score(state)
    else:
        _plain_evict(state)
    if op == "attend":
        return {"out": state["out"], "lse": state["lse"]}
    if op == "score":
        return {"sums": view["sums"]}
    got = {"k": _typed(view["k"], c["type"]), "v": _typed(view["v"], c["type"]), "k_scale": view["k_scale"], "v_scale": view["v_scale"],
           "pos": view["pos"], "sums": view["sums"]}
    if op == "write":
        return {**got, "tail": view["tail"], "tag": view["tag"]}
    return {**got, "kept": state["kept"], "lens": state["lens_out"]}


# ---------------------------------------------------------------- what a pass has to move and compute

def _seen_pairs(case):
    """(pairs of row and key that see each other, cached tokens some row sees), over one head. The documents'
    cuts are drawn with the inputs: a row is counted as seeing back half a document's length on average."""
    pairs = tokens = 0
    for l, n in zip(_lens(case), _news(case)):
        slot = np.arange(l - n, l, dtype=np.float64)
        back = slot + 1
        if case["docs"]:
            back = np.minimum(back, l / case["docs"])
        if case["window"]:
            back = np.minimum(back, case["window"])
        ahead = np.clip(min(case["prefix"], l) - (slot + 1), 0, None) if case["prefix"] else 0.0
        pairs += float((back + ahead).sum())
        tokens += min(l, int(np.max(back)) + n - 1) if n else 0
    return pairs, tokens


def work(case):
    dim, n_kv, sub = case["dim"], case["n_kv"], case["block"]
    token = 2 * dim + 8.0 / sub                                   # codes and scales of a cached token of a head
    if case["op"] == "write":
        m = sum(_news(case))
        return {"bytes": m * n_kv * (8.0 * dim + token + 8) + 4.0 * m, "flops": 4.0 * m * n_kv * dim}
    if case["op"] == "evict":
        out = sum(min(l, case["keep"]) for l in _lens(case))
        return {"bytes": n_kv * (4.0 * sum(_lens(case)) + out * (2 * token + 16 + 4)), "flops": 4.0 * out * n_kv * dim}
    pairs, tokens = _seen_pairs(case)
    m = sum(_news(case))
    if case["op"] == "attend":
        return {"bytes": tokens * n_kv * token + m * case["n_head"] * (8.0 * dim + 4), "flops": 4.0 * dim * case["n_head"] * pairs}
    return {"bytes": n_kv * (tokens * (dim + 4.0 / sub) + 8.0 * sum(_lens(case))) + m * case["n_head"] * (4.0 * dim + 4),
            "flops": 2.0 * dim * case["n_head"] * pairs}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_tokens(st, s, h, name):
    """Sequence s's cached keys or values of KV head h, [len, dim], in 64 bits."""
    c, view = st["case"], st["view"]
    length = int(st["lens"][s])
    at = st["pages"][s, :-(-length // PAGE)].long()
    codes = view[name][at, h]
    codes = codes.transpose(1, 2).flatten(2)[..., :c["dim"]] if name == "k" else codes[:, :c["dim"]].transpose(1, 2)
    value = _decode(codes.contiguous(), c["type"]).double().reshape(-1, c["dim"])
    scale = view[name + "_scale"][at, h].double().reshape(-1)
    return (value * scale.repeat_interleave(c["block"])[:, None])[:length]


def _exact_attention(st, sums):
    c = st["case"]
    n_kv, group, dim = c["n_kv"], c["n_head"] // c["n_kv"], c["dim"]
    out = torch.zeros(st["m"], c["n_head"], dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["m"], c["n_head"], dtype=torch.float64, device="cuda")
    begin = st["q_start"].tolist()
    for s, length in enumerate(st["lens"].tolist()):
        rows = slice(begin[s], begin[s + 1])
        n = begin[s + 1] - begin[s]
        if not n:
            continue
        pos_q = st["pos"][rows].double()
        at = st["pages"][s, :-(-length // PAGE)].long()
        for h in range(n_kv):
            pos_k = st["view"]["pos"][at, h].reshape(-1)[:length].double()
            q = st["q"].view(st["m"], c["n_head"], dim)[rows, h * group:(h + 1) * group].double()
            x = (q.reshape(n * group, dim) @ _exact_tokens(st, s, h, "k").T).view(n, group, length) * st["scale"]
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            gap = pos_q[:, None] - pos_k[None]
            if st["slopes"] is not None:
                x = x - st["slopes"].double()[h * group:(h + 1) * group][None, :, None] * gap.abs()[:, None]
            blind = torch.arange(length, device="cuda")[None] > (length - n + torch.arange(n, device="cuda"))[:, None]
            if st["prefix"] is not None:
                blind &= pos_k[None] >= st["prefix"][s].double()
            if c["window"]:
                blind |= gap >= c["window"]
            if st["first"] is not None:
                blind |= pos_k[None] < st["first"][rows].double()[:, None]
            x = x.masked_fill(blind[:, None], -math.inf)
            l = torch.logsumexp(x, -1)
            p = torch.exp(x - torch.where(l == -math.inf, torch.zeros_like(l), l)[..., None])
            if sums is not None:
                # the sums are of exp(score - lse) with the lse that the operator is given
                given = st["lse"].view(st["m"], n_kv, group)[rows, h].double()
                p = torch.exp(x - given[..., None]).masked_fill(blind[:, None], 0.0)
                old = sums[at, h].reshape(-1)
                old[:length] = c["decay"] * old[:length] + p.sum((0, 1))
                sums[at, h] = old.view(-1, PAGE)
                continue
            out[rows, h * group:(h + 1) * group] = (p.reshape(n * group, length) @ _exact_tokens(st, s, h, "v")).view(n, group, dim)
            lse[rows, h * group:(h + 1) * group] = l
    return out.view(st["m"], -1), lse


def exact(case, seed):
    global own
    before, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = before
    view, op, block = st["view"], case["op"], case["block"]
    if op == "attend":
        out, lse = _exact_attention(st, None)
        return {"out": out, "lse": lse}
    if op == "score":
        sums = view["sums"].double()
        _exact_attention(st, sums)
        return {"sums": sums}
    got = {n: None for n in ("k", "v", "pos")}
    scales = {n: view[n + "_scale"].double() for n in ("k", "v")}
    sums = view["sums"].double()
    begin = st["q_start"].tolist()
    if op == "write":
        tail = view["tail"].double()
        for s, length in enumerate(st["lens"].tolist()):
            r0, n = begin[s], begin[s + 1] - begin[s]
            slot = int(st["slots"][s])
            have = (length - n) % block
            for part, name in enumerate(("k", "v")):
                new = st[name][r0:r0 + n].view(n, case["n_kv"], case["dim"]).double()
                seq = torch.cat([tail[slot, :, part, :have].transpose(0, 1), new])
                for b in range(-(-seq.shape[0] // block)):
                    at = length - n - have + b * block
                    peak = seq[b * block:(b + 1) * block].abs().amax((0, 2))
                    scales[name][int(st["pages"][s, at // PAGE]), :, at % PAGE // block] = (peak / CODE_MAX[case["type"]]).clamp_min(FLOOR)
                left = (seq.shape[0] - 1) // block * block
                tail[slot, :, part, :seq.shape[0] - left] = seq[left:].transpose(0, 1)
            at = torch.arange(length - n, length, device="cuda")
            sums[st["pages"][s, at // PAGE].long(), :, at % PAGE] = 0.0
        return {**got, "k_scale": scales["k"], "v_scale": scales["v"], "sums": sums, "tail": tail, "tag": None}
    old_sums = sums.clone()
    old = {n: scales[n].clone() for n in scales}
    for s, length in enumerate(st["lens"].tolist()):
        at = st["pages"][s, :-(-length // PAGE)].long()
        for h in range(case["n_kv"]):
            mass = old_sums[at, h].reshape(-1)[:length].cpu().numpy()
            always = np.zeros(length, bool)
            always[:case["sink"]] = True
            always[max(0, length - case["recent"]):] = True
            rest = np.flatnonzero(~always)
            rest = rest[np.argsort(-mass[rest], kind="stable")]
            free = max(0, min(case["keep"], length) - int(always.sum()))
            src = np.sort(np.concatenate([np.flatnonzero(always), rest[:free]]))
            if length <= case["keep"]:
                src = np.arange(length)
            src = torch.from_numpy(src).cuda()
            i = torch.arange(src.numel(), device="cuda")
            to = st["pages_out"][s, i // PAGE].long()
            sums[to, h, i % PAGE] = old_sums[at[src // PAGE], h, src % PAGE]
            nb = -(-src.numel() // block)
            gap = nb * block - src.numel()
            grid = torch.nn.functional.pad(src, (0, gap), value=-1).view(nb, block)
            lead = grid[:, :1]
            whole = (((grid - lead) == torch.arange(block, device="cuda")) | (grid < 0)).all(1) & (lead[:, 0] % block == 0)
            b = torch.arange(nb, device="cuda")
            for name in ("k", "v"):
                x = _exact_tokens(st, s, h, name)[src].abs().amax(1)
                peak = torch.nn.functional.pad(x, (0, gap)).view(nb, block).amax(1)
                copied = old[name][at[lead[:, 0] // PAGE], h, lead[:, 0] % PAGE // block]
                scales[name][st["pages_out"][s, b * block // PAGE].long(), h, b * block % PAGE // block] = torch.where(
                    whole, copied, (peak / CODE_MAX[case["type"]]).clamp_min(FLOOR))
    return {**got, "k_scale": scales["k"], "v_scale": scales["v"], "sums": sums, "kept": None, "lens": None}
