"""Plain 64-bit implementations of the 8-bit KV cache's operators, written token by token from their definitions
(include/infr_hip.h). Codes and scales are defined in f32 and are computed in f32 here too; everything that is summed
is summed in f64. The cache is one byte array, as the library's buffer is, so that whole buffers can be compared."""
import copy
import math

import numpy as np
import torch

PAGE = 64
CODE_MAX = {"i8": np.float32(127), "f8": np.float32(448)}


class Cache:
    def __init__(self, n_pages, n_kv, dim, n_slots, type_="i8", block=16, fill=0):
        self.n_pages, self.n_kv, self.dim, self.n_slots, self.type, self.block = n_pages, n_kv, dim, n_slots, type_, block
        dp = self.dp = -(-dim // 64) * 64
        sub = PAGE // block
        parts = [("k", np.uint8, (n_pages, n_kv, dp // 64, PAGE, 64)), ("v", np.uint8, (n_pages, n_kv, dp, PAGE)),
                 ("k_scale", np.float32, (n_pages, n_kv, sub)), ("v_scale", np.float32, (n_pages, n_kv, sub)),
                 ("pos", np.int32, (n_pages, n_kv, PAGE)), ("sums", np.float32, (n_pages, n_kv, PAGE)),
                 ("tail", np.float32, (n_slots, n_kv, 2, block, dim)), ("tag", np.int32, (n_slots, n_kv, 2, 2))]
        self.offsets, at = {}, 0
        for name, dt, shape in parts:
            self.offsets[name] = at
            at += -(-math.prod(shape) * np.dtype(dt).itemsize // 256) * 256
        self.nbytes = at
        self.buf = np.full(at, fill, np.uint8)
        for name, dt, shape in parts:
            n = math.prod(shape) * np.dtype(dt).itemsize
            setattr(self, name, self.buf[self.offsets[name]:self.offsets[name] + n].view(dt).reshape(shape))
        self.tag[...] = 0

    def clone(self):
        c = Cache(self.n_pages, self.n_kv, self.dim, self.n_slots, self.type, self.block)
        c.buf[...] = self.buf
        return c

    # -- codes --
    def decode(self, codes):
        codes = np.ascontiguousarray(codes)
        if self.type == "i8":
            return codes.view(np.int8).astype(np.float32)
        return torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()

    def quantize(self, x):
        """(scale, codes) of one block's rows x f32 [n, dim]."""
        bits = np.ascontiguousarray(x, np.float32).view(np.uint32) & 0x7FFFFFFF
        if bits.size and bits.max() >= 0x7F800000:
            return np.float32(np.nan), np.zeros(x.shape, np.uint8)
        amax = bits.max().view(np.float32) if bits.size else np.float32(0)
        scale = max(np.float32(amax * (np.float32(1) / CODE_MAX[self.type])), np.float32(2.0 ** -96))
        y = (x / scale).astype(np.float32)
        if self.type == "i8":
            return scale, np.rint(y).clip(-127, 127).astype(np.int8).view(np.uint8)
        return scale, torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()

    # -- single tokens --
    def codes(self, part, page, h, t):
        return self.k[page, h, :, t].reshape(-1)[:self.dim] if part == "k" else self.v[page, h, :self.dim, t]

    def put_codes(self, part, page, h, t, codes):
        wide = np.zeros(self.dp, np.uint8)
        wide[:self.dim] = codes
        if part == "k":
            self.k[page, h, :, t] = wide.reshape(-1, 64)
        else:
            self.v[page, h, :, t] = wide

    def scale_of(self, part):
        return self.k_scale if part == "k" else self.v_scale

    def value(self, part, page, h, t):
        with np.errstate(invalid="ignore"):
            return (self.decode(self.codes(part, page, h, t)) * self.scale_of(part)[page, h, t // self.block]).astype(np.float32)

    def values(self, part, pages, h, n):
        """Cached values of the first n tokens on these pages, f64 [n, dim]."""
        return np.stack([self.value(part, pages[t // PAGE], h, t % PAGE) for t in range(n)]).astype(np.float64) if n else np.zeros((0, self.dim))


def sequences(c, b):
    """(s, first row, rows, len, ok) of each sequence; ok as the tables and the pages needed allow."""
    out = []
    for s in range(b.n_seq):
        r0, r1, n_len = int(b.q_start[s]), int(b.q_start[s + 1]), int(b.lens[s])
        c0 = min(max(r0, 0), b.rows)
        c1 = min(max(r1, c0), b.rows)
        n = min(c1 - c0, b.max_q)
        ok = r0 == c0 and r1 == c1 and c1 - c0 <= b.max_q and n_len >= n and n_len <= b.max_pages * PAGE
        out.append((s, c0, n, n_len, ok))
    return out


class Batch:
    """The tables of a call."""
    def __init__(self, news, lens, pages, max_pages=None, pos=None, slots=None, rows=None, max_q=None):
        self.n_seq = len(news)
        self.lens = np.array(lens, np.int32)
        self.q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.q_start[-1]) if rows is None else rows
        self.max_q = max(max(news), 1) if max_q is None else max_q
        self.max_pages = max(max(len(p) for p in pages), 1) if max_pages is None else max_pages
        self.pages = np.full((self.n_seq, self.max_pages), -1, np.int32)
        for s, p in enumerate(pages):
            self.pages[s, :len(p)] = p
        if pos is None:
            pos = np.concatenate([np.arange(l - n, l) for n, l in zip(news, lens)])
        self.pos = np.zeros(self.rows, np.int32)
        self.pos[:len(pos)] = pos
        self.slots = np.arange(self.n_seq, dtype=np.int32) if slots is None else np.array(slots, np.int32)


def write(c, b, k, v):
    """WriteKv8 on the cache c; k, v f32 [rows, n_kv * dim]."""
    k, v = (np.asarray(x, np.float32).reshape(b.rows, c.n_kv, c.dim) for x in (k, v))
    sub = PAGE // c.block
    for s, r0, n, n_len, ok in sequences(c, b):
        if not ok or n == 0:
            continue
        begin, slot = n_len - n, int(b.slots[s])
        slot_ok = 0 <= slot < c.n_slots
        good = lambda page: 0 <= page < c.n_pages  # noqa: E731
        for h in range(c.n_kv):
            for part, x in (("k", k), ("v", v)):
                pi = 0 if part == "k" else 1
                new = {begin + i: x[r0 + i, h] for i in range(n)}
                rows = {}
                for blk in range(begin // c.block, (n_len - 1) // c.block + 1):
                    t0 = blk * c.block
                    page = int(b.pages[s, t0 // PAGE])
                    have = begin - t0
                    raw = (slot_ok and good(page) and c.tag[slot, h, pi, 0] == page * sub + t0 % PAGE // c.block and
                           c.tag[slot, h, pi, 1] >= have)
                    toks = range(t0, min(t0 + c.block, n_len))
                    if have > 0:
                        for t in range(t0, begin):
                            if raw:
                                rows[t] = c.tail[slot, h, pi, t - t0].copy()
                            elif good(page):
                                rows[t] = c.value(part, page, h, t % PAGE)
                    for t in toks:
                        if t >= begin:
                            rows[t] = new[t]
                    if not good(page):
                        continue
                    scale, codes = c.quantize(np.stack([rows[t] for t in toks]))
                    c.scale_of(part)[page, h, t0 % PAGE // c.block] = scale
                    for i in range(len(toks)):
                        c.put_codes(part, page, h, t0 % PAGE + i, codes[i])
                        if part == "k" and t0 + i >= begin:
                            c.pos[page, h, t0 % PAGE + i] = b.pos[r0 + t0 + i - begin]
                            c.sums[page, h, t0 % PAGE + i] = 0
                if slot_ok:
                    last = (n_len - 1) // c.block * c.block
                    page = int(b.pages[s, last // PAGE])
                    for t in range(last, n_len):
                        if t in rows:
                            c.tail[slot, h, pi, t - last] = rows[t]
                    c.tag[slot, h, pi] = (page * sub + last % PAGE // c.block if good(page) else -1, n_len - last)


class Mode:
    def __init__(self, n_head, scale=None, softcap=0.0, window=0, causal=True, first=None, prefix=None, slopes=None):
        self.n_head, self.scale, self.softcap, self.window, self.causal = n_head, scale, softcap, window, causal
        self.first, self.prefix, self.slopes = first, prefix, slopes


def pages_ok(c, b, s, n_len):
    need = b.pages[s, :-(-n_len // PAGE)]
    return bool(((need >= 0) & (need < c.n_pages)).all())


def scores(c, b, m, q, s, r0, n, n_len, head):
    """f64 scores [n, n_len], the pairs that see each other, and a bound on sum |q k| * |scale| per pair."""
    h = head // (m.n_head // c.n_kv)
    pages = b.pages[s]
    scale = float(np.float32(m.scale if m.scale is not None else 1.0 / math.sqrt(c.dim)))
    x = np.asarray(q, np.float64).reshape(b.rows, m.n_head, c.dim)[r0:r0 + n, head]
    k = c.values("k", pages, h, n_len)
    kpos = np.array([c.pos[pages[t // PAGE], h, t % PAGE] for t in range(n_len)], np.int64)
    with np.errstate(invalid="ignore"):
        sc = scale * (x @ k.T)
        size = abs(scale) * (np.abs(x) @ np.abs(k).T)
        if m.softcap:
            sc = m.softcap * np.tanh(sc / m.softcap)
    qpos = b.pos[r0:r0 + n].astype(np.int64)
    gap = qpos[:, None] - kpos[None]
    if m.slopes is not None:
        sc = sc - float(np.float32(m.slopes[head])) * np.abs(gap)
    see = np.ones((n, n_len), bool)
    if m.causal:
        see = np.arange(n_len)[None] <= (n_len - n + np.arange(n))[:, None]
        if m.prefix is not None:
            see = see | (kpos[None] < m.prefix[s])
    if m.window:
        see &= gap < m.window
    if m.first is not None:
        see &= kpos[None] >= np.asarray(m.first)[r0:r0 + n, None]
    return sc, see, size


def attention(c, b, m, q):
    """(out, lse, tol): f64 [rows, n_head * dim], [rows, n_head]; rows of no sequence are NaN in tol (unchecked).

    tol is what f32 arithmetic with 22-bit operands may be off, from the definition: a score is a sum of dim products
    (each rounding of the partial sum at most 2^-24 of it, q's split and the product 2^-21: dim * 2^-24 + 2^-21 of
    sum |q k|) and a handful of roundings of the score itself and of its exponential (2^-21 of |s|, 2^-20); the
    weights' relative error is that of their scores, doubled for the division by their sum; the sums over n tokens add
    n * 2^-24, and V's weights are split like q."""
    out = np.zeros((b.rows, m.n_head, c.dim))
    lse = np.zeros((b.rows, m.n_head))
    tol = np.full((b.rows, m.n_head, c.dim), np.nan)
    ltol = np.full((b.rows, m.n_head), np.nan)
    for s, r0, n, n_len, ok in sequences(c, b):
        if n == 0:
            continue
        rows = slice(r0, r0 + n)
        if not ok or not pages_ok(c, b, s, n_len):
            out[rows], lse[rows], tol[rows], ltol[rows] = np.nan, np.nan, 0, 0
            continue
        for head in range(m.n_head):
            sc, see, size = scores(c, b, m, q, s, r0, n, n_len, head)
            v = c.values("v", b.pages[s], head // (m.n_head // c.n_kv), n_len)
            for i in range(n):
                js = np.flatnonzero(see[i])
                if js.size == 0:
                    out[r0 + i, head], lse[r0 + i, head], tol[r0 + i, head], ltol[r0 + i, head] = 0, -np.inf, 0, 0
                    continue
                x = sc[i, js]
                top = x.max()
                p = np.exp(x - top)
                l = p.sum()
                eps = (size[i, js].max() * (c.dim * 2.0 ** -24 + 2.0 ** -21) + np.abs(x).max() * 2.0 ** -21 + 2.0 ** -20 +
                       js.size * 2.0 ** -24)
                out[r0 + i, head] = p @ v[js] / l
                lse[r0 + i, head] = top + np.log(l)
                tol[r0 + i, head] = 2 * eps * (p @ np.abs(v[js])) / l + 2.0 ** -22 * np.abs(v[js]).max()
                ltol[r0 + i, head] = 2 * eps + np.abs(lse[r0 + i, head]) * 2.0 ** -22
    return out.reshape(b.rows, -1), lse, tol.reshape(b.rows, -1), ltol


def score(c, b, m, q, lse, decay):
    """(new sums of the whole cache, tolerance), f64 [n_pages, n_kv, 64]."""
    sums, tol = c.sums.astype(np.float64), np.zeros(c.sums.shape)
    group = m.n_head // c.n_kv
    for s, r0, n, n_len, ok in sequences(c, b):
        if not ok:
            continue
        acc, err = np.zeros((c.n_kv, n_len)), np.zeros((c.n_kv, n_len))
        good = (b.pages[s] >= 0) & (b.pages[s] < c.n_pages)  # tokens on other pages have no sums
        safe = copy.copy(b)
        safe.pages = np.where((b.pages >= 0) & (b.pages < c.n_pages), b.pages, 0)
        if n:
            for head in range(m.n_head):
                sc, see, size = scores(c, safe, m, q, s, r0, n, n_len, head)
                with np.errstate(invalid="ignore"):
                    w = np.where(see, np.exp(sc - np.asarray(lse, np.float64)[r0:r0 + n, head, None]), 0)
                    eps = size * (c.dim * 2.0 ** -24 + 2.0 ** -21) + (np.abs(sc) + np.abs(lse[r0:r0 + n, head, None])) * 2.0 ** -21 + 2.0 ** -20
                    acc[head // group] += w.sum(0)
                    err[head // group] += np.where(see, w * (eps + n * group * 2.0 ** -24), 0).sum(0)
        for t in range(n_len):
            if not good[t // PAGE]:
                continue
            at = (b.pages[s, t // PAGE], slice(None), t % PAGE)
            old = decay * c.sums[at].astype(np.float64) if decay else 0.0
            sums[at] = old + acc[:, t]
            tol[at] = err[:, t] + (np.abs(old) + acc[:, t]) * 2.0 ** -22
    return sums, tol


def evict(c, b_pages, lens, pages_out, keep, sink, recent):
    """EvictKv8 on the cache c: (lens_out, kept)."""
    n_seq, max_pages = b_pages.shape
    lens_out = np.full(n_seq, -1, np.int32)
    kept = np.full((n_seq, c.n_kv, keep), -1, np.int32)
    old = c.clone()
    for s in range(n_seq):
        n_len = int(lens[s])
        if not 0 <= n_len <= max_pages * PAGE:
            continue
        n_out = min(n_len, keep)
        need = np.concatenate([b_pages[s, :-(-n_len // PAGE)], pages_out[s, :-(-n_out // PAGE)]])
        if ((need < 0) | (need >= c.n_pages)).any():
            continue
        lens_out[s] = n_out
        for h in range(c.n_kv):
            mass = np.array([old.sums[b_pages[s, t // PAGE], h, t % PAGE] for t in range(n_len)], np.float32)
            if n_len <= keep:
                src = np.arange(n_len)
            else:
                must = np.zeros(n_len, bool)
                must[:sink] = True
                must[n_len - recent:] = True
                order = [t for t in range(n_len) if not must[t]]
                order.sort(key=lambda t: (0 if np.isnan(mass[t]) else 1, 0.0 if np.isnan(mass[t]) else -mass[t], t))
                src = np.sort(np.concatenate([np.flatnonzero(must), np.array(order[:keep - sink - recent], int)]))
            kept[s, h, :n_out] = src
            for page in pages_out[s, :-(-n_out // PAGE)]:  # tails of what was on the new pages before
                tag = c.tag[:, h, :, 0]
                tag[(tag >= 0) & (tag // (PAGE // c.block) == page)] = -1
            for t0 in range(0, n_out, c.block):
                to, at = int(pages_out[s, t0 // PAGE]), t0 % PAGE
                toks = src[t0:t0 + c.block]
                whole = toks[0] % c.block == 0 and (toks == toks[0] + np.arange(len(toks))).all()
                for part in ("k", "v"):
                    if whole:
                        scale = old.scale_of(part)[b_pages[s, toks[0] // PAGE], h, toks[0] % PAGE // c.block]
                        codes = [old.codes(part, b_pages[s, t // PAGE], h, t % PAGE) for t in toks]
                    else:
                        scale, codes = c.quantize(np.stack([old.value(part, b_pages[s, t // PAGE], h, t % PAGE) for t in toks]))
                    c.scale_of(part)[to, h, at // c.block] = scale
                    for i in range(len(toks)):
                        c.put_codes(part, to, h, at + i, codes[i])
                for i, t in enumerate(toks):
                    c.pos[to, h, at + i] = old.pos[b_pages[s, t // PAGE], h, t % PAGE]
                    c.sums[to, h, at + i] = old.sums[b_pages[s, t // PAGE], h, t % PAGE]
    return lens_out, kept
