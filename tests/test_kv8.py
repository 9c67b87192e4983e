"""The operators of the 8-bit KV cache (WriteKv8, AttentionKv8, ScoreKv8, EvictKv8) against the plain 64-bit
implementations of tests/kv8_oracle.py. What is held in 8 bits, the scales, positions, tails and kept tokens are
compared bit for bit over the whole cache buffer, so that what a call must leave alone is checked too; attention and
sums against tolerances that the oracle derives from the operation counts."""
import ctypes
import math

import numpy as np
import pytest

import infr_amd as I
from infr_amd import DType, Graph, InfrError, Kv8, Kv8Batch, Linear, RmsNorm, Add, Status, TensorDesc, Bindings
from infr_amd import AttentionKv8, EvictKv8, ScoreKv8, WriteKv8, kv8_supported
from tests import kv8_oracle as orc

TYPES = {"i8": DType.I8, "f8": DType.F8E4M3}
gpu = pytest.mark.gpu


def geom_of(c):
    return Kv8(c.n_pages, c.n_kv, c.dim, c.n_slots, TYPES[c.type], c.block)


def batch_of(b):
    return Kv8Batch(b.rows, b.n_seq, b.max_q, b.max_pages)


def same(a, b):
    """Equal bytes, but for the payload of NaNs in f32 parts."""
    return np.array_equal(a, b) if a.dtype != np.float32 else np.array_equal(a, b, equal_nan=True)


def assert_same_cache(got, want):
    for n in ("k_scale", "v_scale", "k", "v", "pos", "sums", "tail", "tag"):
        g, w = getattr(got, n), getattr(want, n)
        assert same(g, w), f"{n}: {np.count_nonzero(g != w)} of {g.size} differ, first at {np.argwhere(g != w)[:3].tolist()}"


class Dev:
    """A cache and the tables of a batch on the device."""
    def __init__(self, be, c):
        self.be, self.c = be, c
        self.cache = be.upload_new(c.buf)

    def pull(self):
        got = self.c.clone()
        self.be.download(self.cache, got.buf)
        return got

    def tables(self, b):
        up = self.be.upload_new
        return dict(pos=up(b.pos), pages=up(b.pages), q_start=up(b.q_start), lens=up(b.lens))

    def write(self, b, k, v, **kw):
        t = self.tables(b)
        self.be.run_kv8(WriteKv8(self.be.upload_new(k), self.be.upload_new(v), self.cache, slots=self.be.upload_new(b.slots),
                                 geom=geom_of(self.c), batch=batch_of(b), **t, **kw))

    def mode(self, m):
        up = lambda x, t: None if x is None else self.be.upload_new(np.asarray(x, t))  # noqa: E731
        return dict(n_head=m.n_head, scale=m.scale, softcap=m.softcap, window=m.window, causal=m.causal,
                    first=up(m.first, np.int32), prefix=up(m.prefix, np.int32), slopes=up(m.slopes, np.float32))

    def attention(self, b, m, q, fill=7.0, lse=True, **kw):
        dst = self.be.upload_new(np.full((b.rows, m.n_head * self.c.dim), fill, np.float32))
        out_l = self.be.upload_new(np.full((b.rows, m.n_head), fill, np.float32))
        self.be.run_kv8(AttentionKv8(self.be.upload_new(q), self.cache, dst, geom=geom_of(self.c), batch=batch_of(b),
                                     lse=out_l if lse else None, **self.tables(b), **self.mode(m), **kw))
        return (self.be.download(dst, np.empty((b.rows, m.n_head * self.c.dim), np.float32)),
                self.be.download(out_l, np.empty((b.rows, m.n_head), np.float32)))

    def score(self, b, m, q, lse, decay=1.0, **kw):
        self.be.run_kv8(ScoreKv8(self.be.upload_new(q), self.cache, self.be.upload_new(np.asarray(lse, np.float32)),
                                 geom=geom_of(self.c), batch=batch_of(b), decay=decay, **self.tables(b), **self.mode(m), **kw))

    def evict(self, pages, lens, pages_out, keep, sink=0, recent=0):
        up = self.be.upload_new
        n_seq = pages.shape[0]
        lo, kept = self.be.alloc(n_seq * 4), self.be.alloc(n_seq * self.c.n_kv * keep * 4)
        self.be.run_kv8(EvictKv8(self.cache, up(pages), up(np.asarray(lens, np.int32)), up(pages_out), lo, kept, geom_of(self.c),
                                 n_seq=n_seq, max_pages=pages.shape[1], keep=keep, sink=sink, recent=recent))
        return (self.be.download(lo, np.empty(n_seq, np.int32)),
                self.be.download(kept, np.empty((n_seq, self.c.n_kv, keep), np.int32)))


def page_lists(rng, n_pages, counts):
    order = rng.permutation(n_pages)
    out = []
    for n in counts:
        out.append(order[:n].tolist())
        order = order[n:]
    return out, order


def rows_of(rng, b, c, spread=1.0):
    amp = np.exp(spread * rng.standard_normal(c.n_kv * c.dim))
    return ((rng.standard_normal((b.rows, c.n_kv * c.dim)) * amp).astype(np.float32),
            rng.standard_normal((b.rows, c.n_kv * c.dim)).astype(np.float32))


def filled(rng, type_="i8", block=16, n_kv=2, dim=64, lens=(100,), spare=2, pos=None, n_slots=None, fill=0xFF):
    """A cache whose sequences of these lengths were written in one go, and their pages. Bytes that nothing has
    written are `fill` (0xFF: NaN as an e4m3 code, as a scale and as a sum)."""
    counts = [-(-l // 64) for l in lens]
    c = orc.Cache(sum(counts) + spare, n_kv, dim, n_slots or len(lens), type_, block, fill)
    pages, free = page_lists(rng, c.n_pages, counts)
    b = orc.Batch(list(lens), list(lens), pages, pos=pos)
    if b.rows:
        orc.write(c, b, *rows_of(rng, b, c))
    return c, pages, free


def close(got, want, tol):
    """Within tol where it is a number; equal where the oracle is not finite."""
    checked = ~np.isnan(tol)
    finite = checked & np.isfinite(want)
    odd = checked & ~np.isfinite(want)
    assert np.array_equal(got[odd], want[odd], equal_nan=True)
    assert np.isfinite(got[finite]).all()
    over = np.abs(got[finite].astype(np.float64) - want[finite]) - tol[finite]
    assert over.size == 0 or over.max() <= 0, f"off by up to {over.max():.3g} over a tolerance of {tol[finite].mean():.3g} on average"


# ---------------------------------------------------------------- without a GPU

@pytest.mark.parametrize("dim", [1, 64, 80, 256])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_layout_is_the_documented_one(dim, block):
    c = orc.Cache(5, 3, dim, 2, "i8", block)
    lay = Kv8(5, 3, dim, 2, DType.I8, block).layout()
    assert lay["bytes"] == c.nbytes
    assert {n: lay[n] for n in c.offsets} == c.offsets


def write_op(**kw):
    g = dict(n_pages=4, n_kv=2, head_dim=64, n_slots=1, dtype=DType.I8, block=16)
    b = dict(rows=3, n_seq=1, max_q=3, max_pages=4)
    rest = {}
    for k, v in kw.items():
        (g if k in g else b if k in b else rest)[k] = v
    return WriteKv8(*[None] * 8, Kv8(**g), Kv8Batch(**b), **rest)


@pytest.mark.parametrize("kw,word", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"), (dict(block=8), "block"), (dict(block=48), "block"),
    (dict(dtype=DType.Q8_0), "dtype"), (dict(n_pages=0), "n_pages"), (dict(n_kv=0), "n_kv"), (dict(n_kv=5000), "n_kv"),
    (dict(n_slots=0), "tail slots"), (dict(rows=0), "rows"), (dict(max_q=0), "max_q"), (dict(max_q=4), "max_q"),
    (dict(n_seq=0), "n_seq"), (dict(n_seq=70000), "n_seq"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 26), "max_pages"), (dict(max_pages=65536), "max_pages"), (dict(rows=(1 << 28) + 1), "rows"),
    (dict(k_stride=127), "stride"), (dict(v_stride=1), "stride")])
def test_write_refuses(kw, word):
    assert kv8_supported(write_op()) is None
    assert word in kv8_supported(write_op(**kw))


@pytest.mark.parametrize("kind", [AttentionKv8, ScoreKv8])
@pytest.mark.parametrize("kw,word", [(dict(n_head=3), "n_head"), (dict(n_head=0), "n_head"), (dict(softcap=-1.0), "softcap"),
                                     (dict(softcap=math.nan), "softcap"), (dict(softcap=math.inf), "softcap"),
                                     (dict(scale=math.inf), "scale"), (dict(window=1 << 31), "window"),
                                     (dict(q_stride=100), "stride")])
def test_attention_and_score_refuse(kind, kw, word):
    def op(**k):
        return kind(*[None] * 7, Kv8(4, 2, 64, 1), Kv8Batch(3, 1, 3, 4), **{"n_head": 4, **k})
    assert kv8_supported(op()) is None
    assert word in kv8_supported(op(**kw))
    if kind is ScoreKv8:
        assert "decay" in kv8_supported(op(decay=math.nan))


@pytest.mark.parametrize("kind", [AttentionKv8, ScoreKv8])
@pytest.mark.parametrize("n_kv,n_head,n_seq,max_q,word", [
    (2, 4, 1, 65535 * 64, None), (2, 4, 1, 65535 * 64 + 1, "max_q"), (4096, 4096, 1024, 128, None), (4096, 4096, 1024, 129, "row tiles"),
    (4096, 4096, 1025, 1, "row tiles"), (1, 65535, 65535, 1, "row tiles"), (64, 64, 65535, 1, None)])
def test_calls_larger_than_a_launch_are_refused(kind, n_kv, n_head, n_seq, max_q, word):
    why = kv8_supported(kind(*[None] * 7, Kv8(4, n_kv, 64, 1), Kv8Batch(1 << 28, n_seq, max_q, 65535), n_head=n_head))
    assert why is None if word is None else word in why


@pytest.mark.parametrize("kw,word", [(dict(keep=0), "keep"), (dict(keep=65535 * 64 + 1), "keep"), (dict(sink=40, recent=25), "exceeds"), (dict(keep=0x7FFFFFFF), "keep"),
                                     (dict(sink=0xFFFFFFFF, recent=2), "exceeds")])
def test_evict_refuses(kw, word):
    def op(**k):
        return EvictKv8(*[None] * 6, Kv8(4, 2, 64, 1), n_seq=1, max_pages=2, **{"keep": 64, **k})
    assert kv8_supported(op()) is None
    assert word in kv8_supported(op(**kw))


def test_oracle_write_does_not_depend_on_the_pieces():
    rng = np.random.default_rng(1)
    for type_ in TYPES:
        for block in (16, 64):
            a = orc.Cache(4, 2, 24, 1, type_, block)
            b = a.clone()
            n = 150
            whole = orc.Batch([n], [n], [[2, 0, 3]])
            k, v = rows_of(rng, whole, a)
            orc.write(a, whole, k, v)
            at = 0
            for piece in (1, 1, 13, 1, 40, 7, 64, 23):
                orc.write(b, orc.Batch([piece], [at + piece], [[2, 0, 3]]), k[at:at + piece], v[at:at + piece])
                at += piece
            assert at == n
            for name in ("k", "v", "k_scale", "v_scale", "pos", "sums", "tag"):
                assert np.array_equal(getattr(a, name), getattr(b, name)), name
            step = np.abs(a.values("k", [2, 0, 3], 1, n) - k.reshape(n, 2, 24)[:, 1].astype(np.float64))
            scale = a.k_scale[[2, 0, 3], 1].reshape(-1).repeat(block)[:n, None]
            # int8: half a step; e4m3: half of 2^-3 of the value, or half the smallest step below the normal range
            assert (step <= (scale * 0.5001 if type_ == "i8" else np.maximum(np.abs(k.reshape(n, 2, 24)[:, 1]) * 2.0 ** -4, scale * 2.0 ** -10) * 1.0001)).all()


def test_oracle_attention_is_the_softmax_of_its_definition():
    rng = np.random.default_rng(2)
    c, pages, _ = filled(rng, lens=(70,), dim=16, n_kv=1)
    b = orc.Batch([3], [70], pages)
    q = rng.standard_normal((3, 2 * 16)).astype(np.float32)
    out, lse, _, _ = orc.attention(c, b, orc.Mode(2), q)
    k, v = c.values("k", pages[0], 0, 70), c.values("v", pages[0], 0, 70)
    for i in range(3):
        for h in range(2):
            s = k[:68 + i] @ q[i, h * 16:(h + 1) * 16].astype(np.float64) / 4.0
            p = np.exp(s) / np.exp(s).sum()
            assert np.allclose(out[i, h * 16:(h + 1) * 16], p @ v[:68 + i], rtol=1e-12, atol=1e-14)
            assert math.isclose(lse[i, h], math.log(np.exp(s).sum()), rel_tol=1e-12)


# ---------------------------------------------------------------- WriteKv8

@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dim", [1, 33, 64, 80, 128, 200, 256])
def test_write_in_pieces(be, type_, block, dim):
    rng = np.random.default_rng(dim * 100 + block)
    c = orc.Cache(11, 2, dim, 4, type_, block, 0xA5)
    dev = Dev(be, c)
    pages, _ = page_lists(rng, c.n_pages, [4, 3, 3])
    at = [0, 0, 0]
    for news in ([1, 100, 0], [1, 1, 1], [15, 27, 64], [0, 1, 0], [130, 0, 66], [1, 1, 1]):
        at = [a + n for a, n in zip(at, news)]
        b = orc.Batch(news, at, pages, slots=[3, 0, 2], pos=np.concatenate([np.arange(a - n, a) * 3 + 5 for a, n in zip(at, news)]))
        k, v = rows_of(rng, b, c)
        dev.write(b, k, v)
        orc.write(c, b, k, v)
        assert_same_cache(dev.pull(), c)


@gpu
@pytest.mark.parametrize("type_", TYPES)
def test_write_takes_rows_out_of_a_wider_tensor(be, type_):
    rng = np.random.default_rng(5)
    c = orc.Cache(6, 3, 40, 2, type_, 16)
    dev = Dev(be, c)
    pages, _ = page_lists(rng, 6, [2, 3])
    b = orc.Batch([70, 129], [70, 129], pages)
    wide = rng.standard_normal((b.rows, 7 * 40 + 3)).astype(np.float32)
    dev.write(b, wide, wide, k_off=5, k_stride=7 * 40 + 3, v_off=3 * 40 + 1, v_stride=7 * 40 + 3)
    flat = wide.reshape(-1)
    take = lambda off: np.stack([flat[off + r * (7 * 40 + 3):][:120] for r in range(b.rows)])  # noqa: E731
    orc.write(c, b, take(5), take(121))
    assert_same_cache(dev.pull(), c)


@gpu
@pytest.mark.parametrize("type_", TYPES)
def test_write_after_the_sequence_was_cut_back(be, type_):
    """Cut back inside the open block: the tail still holds the rows. Cut back behind it, or on other pages: the
    cached values count."""
    rng = np.random.default_rng(6)
    c = orc.Cache(8, 2, 48, 2, type_, 16)
    dev = Dev(be, c)
    pages, free = page_lists(rng, 8, [3])
    for n, n_len in ((75, 75), (1, 70), (2, 60), (30, 82), (5, 66), (1, 33)):
        b = orc.Batch([n], [n_len], pages)
        k, v = rows_of(rng, b, c)
        dev.write(b, k, v)
        orc.write(c, b, k, v)
        assert_same_cache(dev.pull(), c)
    moved = [[pages[0][0], int(free[0]), pages[0][2]]]
    b = orc.Batch([4], [70], moved, slots=[1])
    k, v = rows_of(rng, b, c)
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 0.0, 1e-40, 3e38, 2.0 ** -90])
def test_write_of_extreme_values(be, type_, value):
    rng = np.random.default_rng(7)
    c = orc.Cache(3, 2, 20, 1, type_, 16)
    dev = Dev(be, c)
    b = orc.Batch([70], [70], [[1, 2]])
    k, v = rows_of(rng, b, c)
    k[20, 3] = value
    v[17:33] = value
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)
    b = orc.Batch([1], [71], [[1, 2]])
    k, v = rows_of(rng, b, c)
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)


@gpu
@pytest.mark.parametrize("type_", TYPES)
def test_write_codes_next_to_the_rounding_borders(be, type_):
    """Values one ulp either side of, and on, the middle between two codes, for scales of any mantissa and size."""
    rng = np.random.default_rng(34)
    n, dim = 16 * 60, 256
    c = orc.Cache(n // 64, 1, dim, 1, type_, 16)
    scale = (np.exp2(rng.uniform(-60, 60, n // 16)) * np.where(rng.random(n // 16) < 0.2, 1, rng.uniform(1, 2, n // 16))).astype(np.float32)
    codes = np.arange(0, 127) if type_ == "i8" else np.unique(np.abs(np.nan_to_num(c.decode(np.arange(256, dtype=np.uint8)))))
    middle = ((codes[1:] + codes[:-1]) / 2).astype(np.float32)
    x = (rng.choice(middle, (n // 16, 16, dim)) * scale[:, None, None]).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape)).astype(np.int32).view(np.float32) * rng.choice([-1, 1], x.shape).astype(np.float32)
    x[:, rng.integers(0, 16), rng.integers(0, dim)] = scale * orc.CODE_MAX[type_]
    b = orc.Batch([n], [n], [list(range(n // 64))])
    dev = Dev(be, c)
    dev.write(b, x.reshape(n, dim), x[::-1].reshape(n, dim))
    orc.write(c, b, x.reshape(n, dim), x[::-1].reshape(n, dim))
    assert_same_cache(dev.pull(), c)


@gpu
def test_write_leaves_alone_what_wrong_tables_name(be):
    rng = np.random.default_rng(8)
    c = orc.Cache(6, 2, 32, 3, "i8", 16, 0x3C)
    dev = Dev(be, c)
    good, bad_page, big_page, too_long, short = [0, 1], [2, -1], [3, 6], [4], [5]
    b = orc.Batch([100, 100, 100, 10, 10], [100, 100, 100, 200, 4], [good, bad_page, big_page, too_long, short],
                  slots=[0, 1, 2, -1, 3])
    k, v = rows_of(rng, b, c)
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)
    for start in ([0, 400, 9, 20, 30, 40], [-3, 5, 10, 20, 30, 40], [0, 10, 20, 30, 40, 2000]):
        b.q_start[:] = start
        dev.write(b, k, v)
        orc.write(c, b, k, v)
        assert_same_cache(dev.pull(), c)


@gpu
def test_write_many_sequences(be):
    rng = np.random.default_rng(9)
    n = 150
    c = orc.Cache(2 * n, 1, 16, n, "i8", 16)
    dev = Dev(be, c)
    pages, _ = page_lists(rng, 2 * n, [2] * n)
    lens = rng.integers(0, 100, n)
    news = np.array([rng.integers(0, min(l, 9) + 1) for l in lens])
    b = orc.Batch(news.tolist(), lens.tolist(), pages, slots=rng.permutation(n))
    k, v = rows_of(rng, b, c)
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)


# ---------------------------------------------------------------- AttentionKv8

def check_attention(be, c, pages, news, lens, m, seed=0, pos=None, scale_q=1.0, **kw):
    rng = np.random.default_rng(seed)
    b = orc.Batch(news, lens, pages, pos=pos)
    q = (scale_q * rng.standard_normal((b.rows, m.n_head * c.dim))).astype(np.float32)
    out, lse = Dev(be, c).attention(b, m, q, **kw)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    close(out, want, tol)
    close(lse, want_l, ltol)
    return b, q, out, lse


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dim", [1, 40, 64, 80, 128, 192, 256])
def test_attention_single_tokens(be, type_, block, dim):
    rng = np.random.default_rng(dim + block)
    lens = (1, 63, 64, 65, 200, 17)
    c, pages, _ = filled(rng, type_, block, 2, dim, lens)
    check_attention(be, c, pages, [1] * len(lens), list(lens), orc.Mode(6), seed=dim)


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_kv,n_head", [(1, 1), (1, 16), (2, 34), (3, 3), (4, 20), (1, 7)])
def test_attention_head_groups(be, type_, n_kv, n_head):
    rng = np.random.default_rng(n_head)
    c, pages, _ = filled(rng, type_, 32, n_kv, 64, (130, 90))
    check_attention(be, c, pages, [1, 1], [130, 90], orc.Mode(n_head))
    check_attention(be, c, pages, [5, 33], [130, 90], orc.Mode(n_head))


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [24, 64, 100, 128, 176, 256])
@pytest.mark.parametrize("lens,news", [((300,), (300,)), ((129, 64, 1), (129, 64, 1)), ((260, 190), (70, 1)), ((200, 150), (0, 150))])
def test_attention_prompts(be, type_, dim, lens, news):
    rng = np.random.default_rng(dim)
    c, pages, _ = filled(rng, type_, 64, 2, dim, lens)
    check_attention(be, c, pages, list(news), list(lens), orc.Mode(4), seed=dim)


MODES = [dict(softcap=5.0), dict(window=1), dict(window=50), dict(slopes=True), dict(prefix=True), dict(first=True),
         dict(causal=False), dict(softcap=30.0, window=40, slopes=True, prefix=True, first=True), dict(causal=False, window=30, slopes=True),
         dict(scale=0.0), dict(scale=-0.3), dict(first="none"), dict(softcap=2.0, prefix=True)]


def mode_of(kw, n_head, news, lens, rng):
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = 2.0 ** -np.arange(1, n_head + 1)
    if kw.get("prefix"):
        kw["prefix"] = [l // 2 for l in lens]
    pos = np.concatenate([np.arange(l - n, l) for n, l in zip(news, lens)])
    if kw.get("first") == "none":  # every row's document begins behind it
        kw["first"] = pos + 1
    elif kw.get("first"):          # and here every third row's does
        kw["first"] = np.where(np.arange(len(pos)) % 3 == 0, pos + 1, (pos // 37) * 37)
    return orc.Mode(n_head, **kw)


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("kw", MODES, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
@pytest.mark.parametrize("news,lens", [((1, 1), (150, 70)), ((4, 3), (150, 70)), ((150, 70), (150, 70)), ((60, 70), (150, 70))])
def test_attention_modes(be, type_, kw, news, lens):
    rng = np.random.default_rng(len(kw))
    c, pages, _ = filled(rng, type_, 16, 2, 96, lens)
    check_attention(be, c, pages, list(news), list(lens), mode_of(kw, 6, news, lens, rng), seed=3)


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("kw", [{}, *MODES], ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
@pytest.mark.parametrize("dim,n_head,news,lens", [(96, 6, (150, 70), (150, 70)), (128, 4, (130, 0), (200, 3)), (200, 2, (90, 33), (90, 200))])
def test_attention_modes_in_a_batch_of_many_rows(be, type_, kw, dim, n_head, news, lens):
    """max_q and rows far above what the sequences have: such a call takes tiles of 128 rows. One sequence's cache holds
    a value that is not finite."""
    rng = np.random.default_rng(len(kw) + dim)
    rows = 512 * 128 // n_head + 1
    c, pages, _ = filled(rng, type_, 16, 2, dim, lens)
    c.v_scale[pages[0][1], 1, 0] = np.nan
    m = mode_of(kw, n_head, news, lens, rng)
    if m.first is not None:
        m.first = np.concatenate([m.first, np.zeros(rows - len(m.first), int)])
    b = orc.Batch(list(news), list(lens), pages, rows=rows, max_q=rows)
    q = rng.standard_normal((rows, n_head * dim)).astype(np.float32)
    out, lse = Dev(be, c).attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    close(out, want, tol)
    close(lse, want_l, ltol)
    assert (out[sum(news):] == 7.0).all()


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 200])
@pytest.mark.parametrize("kw", [{}, dict(softcap=30.0, window=700, slopes=True, prefix=True, first=True), dict(causal=False)], ids=str)
def test_attention_of_a_chunk_in_three_parts(be, type_, dim, kw):
    """Tiles of 128 rows whose pages are cut into parts: a bound on the rows that leaves a few workgroups to each tile."""
    rng = np.random.default_rng(dim)
    rows, news, lens = 10240, (150,), (2000,)
    c, pages, _ = filled(rng, type_, 64, 2, dim, lens)
    m = mode_of(kw, 2, news, lens, rng)
    if m.first is not None:
        m.first = np.concatenate([m.first, np.zeros(rows - len(m.first), int)])
    b = orc.Batch(list(news), list(lens), pages, rows=rows, max_q=rows, max_pages=40)
    q = rng.standard_normal((rows, 2 * dim)).astype(np.float32)
    out, lse = Dev(be, c).attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    close(out, want, tol)
    close(lse, want_l, ltol)
    assert (out[150:] == 7.0).all()


@gpu
@pytest.mark.parametrize("news", [(1,), (2,), (40,)])
def test_attention_over_positions_with_gaps(be, news):
    """As after an eviction: positions ascend with gaps, the masks and the bias go by them."""
    rng = np.random.default_rng(11)
    n_len = 180
    pos = np.cumsum(rng.integers(1, 6, n_len)).astype(np.int32)
    c, pages, _ = filled(rng, "i8", 32, 2, 64, (n_len,), pos=pos)
    for kw in (dict(window=100), dict(slopes=2.0 ** -np.arange(1, 5)), dict(prefix=[int(pos[60])]),
               dict(first=np.full(news[0], pos[100])), dict(window=300, prefix=[int(pos[150])], first=np.full(news[0], pos[20]))):
        check_attention(be, c, pages, list(news), [n_len], orc.Mode(4, **kw), pos=pos[n_len - news[0]:])


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("news", [1, 3, 64])
def test_attention_long_axis(be, type_, news):
    """Enough pages for the work on them to be split, next to a sequence that is not."""
    rng = np.random.default_rng(12)
    lens = (3001, 70)
    c, pages, _ = filled(rng, type_, 64, 1, 64, lens)
    check_attention(be, c, pages, [news, 1], list(lens), orc.Mode(4))
    check_attention(be, c, pages, [news, 1], list(lens), orc.Mode(4, window=1000, softcap=20.0))


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [130, 192, 256])
@pytest.mark.parametrize("news,lens", [((1, 1), (150, 70)), ((4, 3), (500, 129))])
def test_attention_wide_heads_and_wide_page_tables(be, type_, dim, news, lens):
    """Tables for far longer sequences than there are, as a server keeps them: waves take whole pages then."""
    rng = np.random.default_rng(dim)
    c, pages, _ = filled(rng, type_, 32, 2, dim, lens)
    for kw in [{}, dict(window=10 ** 6), *MODES]:
        m = mode_of(kw, 6, news, lens, rng)
        b = orc.Batch(list(news), list(lens), pages, max_pages=9000)
        q = rng.standard_normal((b.rows, 6 * dim)).astype(np.float32)
        out, lse = Dev(be, c).attention(b, m, q)
        want, want_l, tol, ltol = orc.attention(c, b, m, q)
        close(out, want, tol)
        close(lse, want_l, ltol)


@gpu
@pytest.mark.parametrize("news", [1, 3])
@pytest.mark.parametrize("dim,pages_whole", [(64, 8), (160, 4)])
def test_attention_windows_around_a_whole_piece(be, news, dim, pages_whole):
    """Long sequences whose windows reach as many pages as one workgroup takes, one less and one more, from every 7th slot
    of a page."""
    rng = np.random.default_rng(15)
    lens = tuple(range(940, 1010, 7))
    c, pages, _ = filled(rng, "i8", 16, 1, dim, lens)
    for window in (pages_whole * 64 - 62 - news, pages_whole * 64 - 61 - news, pages_whole * 64 - 126 - news):
        check_attention(be, c, pages, [news] * len(lens), list(lens), orc.Mode(1, window=window))


@gpu
@pytest.mark.parametrize("news", [1, 40])
def test_attention_many_sequences(be, news):
    rng = np.random.default_rng(13)
    lens = tuple(int(x) for x in rng.integers(40, 130, 150 if news == 1 else 9))
    c, pages, _ = filled(rng, "i8", 16, 1, 16, lens)
    check_attention(be, c, pages, [news] * len(lens), list(lens), orc.Mode(2))


@gpu
@pytest.mark.parametrize("news", [1, 30])
@pytest.mark.parametrize("scale_q", [1e-30, 1e-3, 1e4, 1e20])
def test_attention_sizes_of_queries(be, news, scale_q):
    """Query rows of any size: a one-hot softmax for the large ones."""
    rng = np.random.default_rng(14)
    c, pages, _ = filled(rng, "i8", 16, 1, 64, (100,))
    check_attention(be, c, pages, [news], [100], orc.Mode(3), scale_q=scale_q)


@gpu
@pytest.mark.parametrize("news", [1, 70])
def test_attention_scales_of_blocks_far_apart(be, news):
    """Keys and values whose blocks differ by many powers of two, a block of zeros among them."""
    rng = np.random.default_rng(15)
    c = orc.Cache(5, 1, 64, 1, "f8", 16)
    pages = [[4, 0, 2, 1]]
    b = orc.Batch([200], [200], pages)
    k, v = rows_of(rng, b, c)
    v *= (10.0 ** rng.integers(-6, 3, 13)).repeat(16)[:200, None].astype(np.float32)
    k *= (2.0 ** rng.integers(-8, 2, 13)).repeat(16)[:200, None].astype(np.float32)
    v[32:48] = 0
    k[64:80] = 0
    orc.write(c, b, k, v)
    check_attention(be, c, pages, [news], [200], orc.Mode(4))
    v[:] = 0
    orc.write(c, b, k, v)
    check_attention(be, c, pages, [news], [200], orc.Mode(4))


@gpu
@pytest.mark.parametrize("news", [1, 5, 90])
def test_attention_nan_reaches_only_the_rows_that_see_it(be, news):
    rng = np.random.default_rng(16)
    n_len = 150
    c, pages, _ = filled(rng, "i8", 16, 2, 32, (n_len,))
    for part, page, h, sub in (("k_scale", 0, 0, 1), ("v_scale", 1, 1, 2)):
        getattr(c, part)[pages[0][page], h, sub] = np.nan
    first = np.arange(n_len - news, n_len) // 2
    first[-1] = 120                                  # behind both blocks
    m = orc.Mode(4, first=first)
    b, q, out, _ = check_attention(be, c, pages, [news], [n_len], m)
    assert np.isfinite(out[-1]).all()
    q[0] = np.nan
    out, lse = Dev(be, c).attention(b, orc.Mode(4), q)
    assert np.isnan(out[0]).all() and np.isnan(lse[0]).all()


@gpu
@pytest.mark.parametrize("max_q", [1, 2, 64])
def test_attention_wrong_tables_are_nan_and_rows_behind_the_last_stay(be, max_q):
    rng = np.random.default_rng(17)
    c, pages, _ = filled(rng, "i8", 16, 2, 64, (100, 100, 100))
    pages = [pages[0], [pages[1][0], -1], [9999, pages[2][1]], [0], [0]]
    news = [1, 1, 1, max_q, 1]
    b = orc.Batch(news, [100, 100, 100, max_q - 1, 129], pages, rows=sum(news) + 2, max_q=max_q, max_pages=2,
                  pos=[99, 99, 99] + list(range(max_q)) + [128])
    q = rng.standard_normal((b.rows, 4 * 64)).astype(np.float32)
    m = orc.Mode(4)
    dev = Dev(be, c)
    for start in (None, [0, 1, 2, 3, 3 + max_q + 1, 3 + max_q + 2], [-5, 1, 2, 3, 3, 3]):
        if start:
            b.q_start[:] = start
        out, lse = dev.attention(b, m, q)
        want, want_l, tol, ltol = orc.attention(c, b, m, q)
        close(out, want, tol)
        close(lse, want_l, ltol)
        untouched = np.isnan(tol[:, 0])
        assert (out[untouched] == 7.0).all() and (lse[untouched] == 7.0).all()
        assert untouched[-1]


@gpu
def test_attention_reads_rows_out_of_a_wider_tensor_and_without_lse(be):
    rng = np.random.default_rng(18)
    for dim, off, extra in ((40, 3, 5), (64, 8, 16)):
        c, pages, _ = filled(rng, "i8", 16, 2, dim, (100, 70))
        for news in ([1, 1], [50, 70]):
            b = orc.Batch(news, [100, 70], pages)
            stride = 4 * dim + extra
            wide = rng.standard_normal((b.rows, stride)).astype(np.float32)
            wide = np.concatenate([wide.reshape(-1), np.zeros(off, np.float32)])
            q = np.stack([wide[off + r * stride:][:4 * dim] for r in range(b.rows)])
            m = orc.Mode(4)
            out, lse = Dev(be, c).attention(b, m, wide, q_off=off, q_stride=stride, lse=False)
            want, _, tol, _ = orc.attention(c, b, m, q)
            close(out, want, tol)
            assert (lse == 7.0).all()


@gpu
def test_attention_sequences_share_pages(be):
    rng = np.random.default_rng(19)
    c, pages, free = filled(rng, "i8", 16, 2, 64, (192,), spare=3)
    two = [pages[0], [pages[0][0], pages[0][1], int(free[0])]]
    b = orc.Batch([0, 20], [192, 148], two, slots=[0, 0])
    orc.write(c, b, *rows_of(rng, b, c))
    check_attention(be, c, two, [1, 20], [192, 148], orc.Mode(4))


@gpu
@pytest.mark.parametrize("news", [1, 100])
def test_attention_gives_the_same_bits_each_time(be, news):
    rng = np.random.default_rng(20)
    c, pages, _ = filled(rng, "f8", 64, 1, 128, (2000,))
    b = orc.Batch([news], [2000], pages)
    q = rng.standard_normal((b.rows, 8 * 128)).astype(np.float32)
    dev = Dev(be, c)
    a = dev.attention(b, orc.Mode(8), q)
    for _ in range(3):
        again = dev.attention(b, orc.Mode(8), q)
        assert np.array_equal(a[0], again[0]) and np.array_equal(a[1], again[1])


# ---------------------------------------------------------------- ScoreKv8

@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [24, 64, 128, 256])
@pytest.mark.parametrize("news,lens", [((1, 1, 1), (150, 70, 1)), ((3, 1, 1), (150, 70, 1)), ((150, 30, 0), (150, 70, 1))])
@pytest.mark.parametrize("decay", [0.0, 1.0, 0.5])
def test_score(be, type_, dim, news, lens, decay):
    rng = np.random.default_rng(dim)
    c, pages, _ = filled(rng, type_, 16, 2, dim, lens)
    for s, p in enumerate(pages):
        c.sums[p] = np.nan if decay == 0.0 else rng.random((len(p), 2, 64))
    b = orc.Batch(list(news), list(lens), pages)
    for m in (orc.Mode(4), mode_of(MODES[7], 4, news, lens, rng)):
        q = rng.standard_normal((b.rows, 4 * dim)).astype(np.float32)
        lse = orc.attention(c, b, m, q)[1].astype(np.float32)
        want, tol = orc.score(c, b, m, q, lse, decay)
        dev = Dev(be, c)
        dev.score(b, m, q, lse, decay)
        got = dev.pull()
        assert np.array_equal(got.buf[:c.offsets["sums"]], c.buf[:c.offsets["sums"]])
        for s, n in enumerate(lens):
            for t in range(n):
                at = (pages[s][t // 64], slice(None), t % 64)
                assert (np.abs(got.sums[at] - want[at]) <= tol[at]).all()
                got.sums[at] = c.sums[at]
        assert np.array_equal(got.sums.view(np.uint32), c.sums.view(np.uint32))  # slots behind the ends and other pages


@gpu
def test_score_many_heads_long_axis_and_wrong_tables(be):
    rng = np.random.default_rng(21)
    lens = (1500, 90, 90)
    c, pages, _ = filled(rng, "i8", 64, 1, 64, lens)
    c.sums[...] = 0.25
    pages[2] = [pages[2][0], 12345]
    for news in ([1, 1, 1], [9, 9, 9]):
        b = orc.Batch(news, list(lens), pages)
        m = orc.Mode(20)
        q = rng.standard_normal((b.rows, 20 * 64)).astype(np.float32)
        lse = orc.attention(c, orc.Batch(news, list(lens), [pages[0], pages[1], [0, 0]]), m, q)[1].astype(np.float32)
        want, tol = orc.score(c, b, m, q, lse, 1.0)
        dev = Dev(be, c)
        dev.score(b, m, q, lse)
        got = dev.pull().sums
        assert (np.abs(got - want) <= tol).all()


# ---------------------------------------------------------------- EvictKv8

def check_evict(be, c, pages, lens, pages_out, keep, sink, recent):
    table = np.full((len(pages), max(len(p) for p in pages)), -1, np.int32)
    for s, p in enumerate(pages):
        table[s, :len(p)] = p
    out = np.full((len(pages), -(-keep // 64)), -1, np.int32)
    for s, p in enumerate(pages_out):
        out[s, :len(p)] = p
    dev = Dev(be, c)
    lo, kept = dev.evict(table, lens, out, keep, sink, recent)
    want_lo, want_kept = orc.evict(c, table, lens, out, keep, sink, recent)
    assert lo.tolist() == want_lo.tolist()
    assert np.array_equal(kept, want_kept)
    assert_same_cache(dev.pull(), c)


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dim,keep,sink,recent", [(64, 64, 0, 0), (40, 100, 4, 30), (128, 130, 0, 130), (256, 33, 33, 0), (1, 150, 1, 1)])
def test_evict(be, type_, block, dim, keep, sink, recent):
    rng = np.random.default_rng(keep)
    lens = (300, keep, keep + 1, 20, 200, 0)
    n_out = -(-keep // 64)
    c, pages, free = filled(rng, type_, block, 2, dim, lens, spare=n_out * len(lens) + 1)
    for p in pages:
        c.sums[p] = rng.random((len(p), 2, 64)) ** 4
    out = [free[s * n_out:(s + 1) * n_out].tolist() for s in range(len(lens))]
    check_evict(be, c, pages, lens, out, keep, sink, recent)


@gpu
@pytest.mark.parametrize("type_", TYPES)
def test_evict_there_and_back_leaves_no_stale_tail(be, type_):
    """A sequence moves to other pages and back to its first ones, with other tokens, before it goes on: the tail's tag
    then names the block that is open, but its rows are not that block's. A bystander's tail stays."""
    rng = np.random.default_rng(25)
    c, pages, free = filled(rng, type_, 32, 2, 40, (75, 90), spare=4)
    old = [[int(x) for x in p] for p in pages]
    for p in pages:
        c.sums[p] = rng.random((len(p), 2, 64))
    there = [[int(free[0]), int(free[1])]]
    before = c.tag.copy()
    assert before[0, 0, 0, 0] == old[0][1] * 2 and before[0, 0, 0, 1] == 11
    check_evict(be, c, old[:1], (75,), there, 74, 2, 3)
    check_evict(be, c, there, (74,), [old[0]], 73, 2, 3)
    assert (c.tag[0, :, :, 0] == -1).all() and np.array_equal(c.tag[1], before[1])
    b = orc.Batch([1, 1], [74, 91], old, slots=[0, 1], pos=[75, 90])
    k, v = rows_of(rng, b, c)
    dev = Dev(be, c)
    dev.write(b, k, v)
    orc.write(c, b, k, v)
    assert_same_cache(dev.pull(), c)


@gpu
def test_evict_ties_zeros_and_odd_sums(be):
    rng = np.random.default_rng(23)
    lens = (500, 1500, 400)
    c, pages, free = filled(rng, "i8", 16, 3, 32, lens, spare=10)
    c.sums[...] = 0.0
    c.sums[:, 1] = rng.integers(0, 3, c.sums[:, 1].shape) * 0.5          # many ties across passes
    c.sums[pages[1], 2] = -rng.random((len(pages[1]), 64))
    c.sums[pages[2][3], 2, :8] = [np.nan, np.inf, -np.inf, -0.0, 0.0, 1e-45, -1e-45, 3e38]
    check_evict(be, c, pages, lens, [free[3 * s:3 * s + 3].tolist() for s in range(3)], 150, 3, 40)


@gpu
@pytest.mark.parametrize("n_len", [4096, 4097, 32768, 32769, 70001])
@pytest.mark.parametrize("sums", ["spread", "steps", "one"])
def test_evict_of_long_sequences(be, n_len, sums):
    """Lengths either side of what a workgroup holds at once; sums of many sizes, of few values and all equal."""
    rng = np.random.default_rng(n_len)
    n_pages = -(-n_len // 64) + 3
    c = orc.Cache(n_pages, 1, 2, 1, "i8", 16)
    order = rng.permutation(n_pages)
    c.k[...], c.v[...] = rng.integers(0, 256, c.k.shape), rng.integers(0, 256, c.v.shape)
    c.k[..., 2:] = 0
    c.v[:, :, 2:] = 0
    c.k_scale[...], c.v_scale[...] = rng.random(c.k_scale.shape) + 0.5, rng.random(c.v_scale.shape) + 0.5
    c.pos[order[:-3]] = np.arange((n_pages - 3) * 64, dtype=np.int32).reshape(-1, 1, 64)
    shape = c.sums.shape
    c.sums[...] = {"spread": np.exp(10 * rng.standard_normal(shape)), "steps": rng.integers(0, 5, shape) * 0.125, "one": np.full(shape, 0.5)}[sums]
    check_evict(be, c, [order[:-3].tolist()], [n_len], [order[-3:].tolist()], 190, 3, 60)


@gpu
def test_evict_leaves_alone_sequences_with_wrong_tables(be):
    rng = np.random.default_rng(24)
    c, pages, free = filled(rng, "i8", 16, 2, 32, (200, 200, 200, 200), spare=8)
    pages[1][2] = -1
    out = [free[2 * s:2 * s + 2].tolist() for s in range(4)]
    out[2][1] = c.n_pages
    check_evict(be, c, pages, (200, 200, 200, -7), out, 100, 0, 10)
    check_evict(be, c, pages, (200, 10 ** 6, 200, 2 ** 31 - 1), out, 100, 0, 10)


# ---------------------------------------------------------------- together, in plans

def pack(be, g, binds, arr, kind="input", dt=None):
    arr = np.ascontiguousarray(arr)
    dt = dt or (DType.F32 if arr.dtype == np.float32 else DType.I32)
    t = getattr(g, kind)(TensorDesc(arr.shape, dt))
    buf = be.upload_new(arr)
    binds.bind(t, buf)
    return t, buf


@gpu
@pytest.mark.parametrize("type_", TYPES)
def test_a_decoder_layers_steps_in_one_plan(be, type_):
    """RmsNorm -> one Linear onto q|k|v -> WriteKv8 -> AttentionKv8 -> ScoreKv8 -> output Linear -> Add: a prompt, then
    single tokens through one plan whose tables change between the replays, then an eviction and single tokens on the
    new pages. Each step equals the ops called one by one, and the cache equals the oracle's."""
    rng = np.random.default_rng(30)
    n_kv, n_head, dim, ne, keep = 2, 4, 64, 256, 96
    c = orc.Cache(12, n_kv, dim, 2, type_, 16)
    width = (n_head + 2 * n_kv) * dim
    wq, wo = I.synth_weight(DType.Q8_0, 1, width, ne, 0.05), I.synth_weight(DType.Q8_0, 2, ne, n_head * dim, 0.05)
    norm = np.ones(ne, np.float32)
    cache = be.upload_new(c.buf)
    mine = be.upload_new(c.buf)
    table = np.full((2, 4), -1, np.int32)
    table[0, :3], table[1, :4] = [7, 1, 4], [0, 9, 2, 5]

    def build(rows, news_max):
        g, binds, bufs = Graph(), Bindings(), {}
        def add(name, arr, kind="input", dt=None):
            t, bufs[name] = pack(be, g, binds, arr, kind, dt)
            return t
        x = add("x", np.zeros((rows, ne), np.float32))
        n = g.output(TensorDesc((rows, ne), DType.F32))
        qkv = g.output(TensorDesc((rows, width), DType.F32))
        att = g.output(TensorDesc((rows, n_head * dim), DType.F32))
        lse = g.output(TensorDesc((rows, n_head), DType.F32))
        o = g.output(TensorDesc((rows, ne), DType.F32))
        y = g.output(TensorDesc((rows, ne), DType.F32))
        for t, w in ((n, ne), (qkv, width), (att, n_head * dim), (lse, n_head), (o, ne), (y, ne)):
            bufs[t.id] = be.alloc(rows * w * 4)
            binds.bind(t, bufs[t.id])
        nw = add("norm", norm)
        wqt, wot = g.weight(TensorDesc((width, ne), DType.Q8_0)), g.weight(TensorDesc((ne, n_head * dim), DType.Q8_0))
        bufs["wq"], bufs["wo"] = be.upload_new(wq), be.upload_new(wo)
        binds.bind(wqt, bufs["wq"]).bind(wot, bufs["wo"])
        ct = g.input(TensorDesc((c.nbytes,), DType.I8))
        binds.bind(ct, cache)
        pos, pages = add("pos", np.zeros(rows, np.int32)), add("pages", table)
        start, lens, slots = add("start", np.zeros(3, np.int32)), add("lens", np.zeros(2, np.int32)), add("slots", np.array([1, 0], np.int32))
        geom, batch = geom_of(c), Kv8Batch(rows, 2, news_max, 4)
        g.push(RmsNorm(x, nw, n, rows, ne, 1e-6))
        g.push(Linear(n, wqt, qkv, rows, ne, width))
        g.push(WriteKv8(qkv, qkv, ct, pos, pages, start, lens, slots, geom, batch, k_off=n_head * dim, k_stride=width,
                        v_off=(n_head + n_kv) * dim, v_stride=width))
        tables = dict(pos=pos, pages=pages, q_start=start, lens=lens, geom=geom, batch=batch, n_head=n_head, q_stride=width)
        g.push(AttentionKv8(qkv, ct, att, lse=lse, **tables))
        g.push(ScoreKv8(qkv, ct, lse, decay=0.9, **tables))
        g.push(Linear(att, wot, o, rows, n_head * dim, ne))
        g.push(Add(x, o, y, rows * ne))
        return be.compile(g), binds, bufs, dict(n=n.id, qkv=qkv.id, att=att.id, lse=lse.id, y=y.id)

    def step(built, b):
        plan, binds, bufs, ids = built
        x = rng.standard_normal((b.rows, ne)).astype(np.float32)
        for name, arr in (("x", x), ("pos", b.pos), ("pages", b.pages), ("start", b.q_start), ("lens", b.lens)):
            be.upload(bufs[name], arr)
        be.execute(plan, binds)
        get = lambda i, w: be.download(bufs[ids[i]], np.empty((b.rows, w), np.float32))  # noqa: E731
        qkv, att, lse, y = get("qkv", width), get("att", n_head * dim), get("lse", n_head), get("y", ne)
        # the same ops one by one on a second cache
        t = dict(pos=bufs["pos"], pages=bufs["pages"], q_start=bufs["start"], lens=bufs["lens"], geom=geom_of(c), batch=batch_of(b))
        qb = be.upload_new(qkv)
        be.run_kv8(WriteKv8(qb, qb, mine, slots=bufs["slots"], k_off=n_head * dim, k_stride=width, v_off=(n_head + n_kv) * dim, v_stride=width, **t))
        a2, l2 = be.alloc(att.nbytes), be.alloc(lse.nbytes)
        be.run_kv8(AttentionKv8(qb, mine, a2, lse=l2, n_head=n_head, q_stride=width, **t))
        be.run_kv8(ScoreKv8(qb, mine, l2, n_head=n_head, q_stride=width, decay=0.9, **t))
        assert np.array_equal(be.download(a2, np.empty_like(att)), att)
        assert np.array_equal(be.download(l2, np.empty_like(lse)), lse)
        one, two = np.empty_like(c.buf), np.empty_like(c.buf)
        be.download(cache, one)
        be.download(mine, two)
        assert np.array_equal(one, two)
        # and the oracle, whose cache goes on from the device's sums
        m = orc.Mode(n_head)
        q = qkv[:, :n_head * dim]
        orc.write(c, b, qkv[:, n_head * dim:(n_head + n_kv) * dim], qkv[:, (n_head + n_kv) * dim:])
        want, want_l, tol, ltol = orc.attention(c, b, m, q)
        close(att, want, tol)
        close(lse, want_l, ltol)
        sums, stol = orc.score(c, b, m, q, lse, np.float32(0.9))
        got = c.clone()
        got.buf[...] = one
        assert (np.abs(got.sums - sums) <= stol).all()
        c.sums[...] = got.sums
        assert_same_cache(got, c)
        # the output Linear reads att: y - x is its result
        ob = be.alloc(y.nbytes)
        be.linear(DType.Q8_0, bufs["wo"], be.upload_new(att), ob, b.rows, n_head * dim, ne)
        assert np.array_equal(x + be.download(ob, np.empty_like(y)), y)

    lens = [70, 110]
    step(build(180, 110), orc.Batch([70, 110], lens, table.tolist(), max_pages=4, slots=[1, 0]))
    single = build(2, 1)
    for _ in range(4):
        lens = [l + 1 for l in lens]
        step(single, orc.Batch([1, 1], lens, table.tolist(), max_pages=4, slots=[1, 0]))
    out = np.array([[3, 6], [8, 10]], np.int32)
    dev = Dev(be, c)
    for buf in (cache, mine):
        dev.cache = buf
        lo, kept = dev.evict(table, lens, out, keep, 2, 20)
        assert lo.tolist() == [74, 96]
    want_lo, want_kept = orc.evict(c, table, lens, out, keep, 2, 20)
    assert np.array_equal(kept, want_kept)
    assert_same_cache(dev.pull(), c)
    table[:] = -1
    table[:, :2] = out
    at, lens = lens, [74, 96]
    for i in range(3):  # the sequences go on: lengths from the new lens, positions from the old ones
        lens = [l + 1 for l in lens]
        step(single, orc.Batch([1, 1], lens, table.tolist(), max_pages=4, slots=[1, 0], pos=[at[0] + i, at[1] + i]))


@gpu
def test_plans_that_share_the_scratch(be):
    """Two recorded plans of one backend and a direct call between them: each result stays its own."""
    rng = np.random.default_rng(31)
    c, pages, _ = filled(rng, "i8", 64, 1, 64, (2500,))
    cache = be.upload_new(c.buf)
    plans = []
    for n_head in (4, 8):
        g, binds = Graph(), Bindings()
        b = orc.Batch([1], [2500], pages)
        q = rng.standard_normal((1, n_head * 64)).astype(np.float32)
        t = {n: pack(be, g, binds, a)[0] for n, a in (("q", q), ("pos", b.pos), ("pages", b.pages), ("q_start", b.q_start), ("lens", b.lens))}
        ct, dst = g.input(TensorDesc((c.nbytes,), DType.I8)), g.output(TensorDesc((1, n_head * 64), DType.F32))
        out = be.alloc(n_head * 64 * 4)
        binds.bind(ct, cache).bind(dst, out)
        g.push(AttentionKv8(t["q"], ct, dst, t["pos"], t["pages"], t["q_start"], t["lens"], geom_of(c), batch_of(b), n_head))
        plans.append((be.compile(g), binds, out, n_head, orc.attention(c, b, orc.Mode(n_head), q)))
    for _ in range(3):
        for plan, binds, out, n_head, (want, _, tol, _) in plans:
            be.execute(plan, binds)
        check_attention(be, c, pages, [64], [2500], orc.Mode(16))
        for plan, binds, out, n_head, (want, _, tol, _) in plans:
            close(be.download(out, np.empty((1, n_head * 64), np.float32)), want, tol)
            be.upload(out, np.zeros(n_head * 64, np.float32))


@gpu
def test_two_backends_at_once(be):
    """Calls of two backends, each on its own stream and scratch, that nothing waits between."""
    rng = np.random.default_rng(35)
    other = I.HipBackend(0)
    try:
        calls = []
        for k in range(6):
            owner = (be, other)[k % 2]
            c, pages, _ = filled(rng, "i8", 16, 2, 64, (2500 + k, 70))
            b = orc.Batch([1 + k, 40], [2500 + k, 70], pages)
            m = orc.Mode(4, window=0 if k < 3 else 900)
            q = rng.standard_normal((b.rows, 256)).astype(np.float32)
            dev = Dev(owner, c)
            up = owner.upload_new
            op = AttentionKv8(up(q), dev.cache, up(np.zeros((b.rows, 256), np.float32)), geom=geom_of(c), batch=batch_of(b),
                              lse=up(np.zeros((b.rows, 4), np.float32)), **dev.tables(b), **dev.mode(m))
            calls.append((owner, op, orc.attention(c, b, m, q)))
        for _ in range(20):
            for owner, op, _ in calls:
                owner.run_kv8(op)
        for owner, op, (want, want_l, tol, ltol) in calls:
            close(owner.download(op.dst, np.empty(want.shape, np.float32)), want, tol)
            close(owner.download(op.lse, np.empty(want_l.shape, np.float32)), want_l, ltol)
    finally:
        calls = dev = op = None  # its buffers go first
        other.close()


@gpu
def test_refusals_of_operands(be):
    rng = np.random.default_rng(32)
    c, pages, _ = filled(rng, "i8", 16, 2, 64, (70,))
    b = orc.Batch([1], [70], pages)
    up = be.upload_new
    good = dict(q=up(np.zeros((1, 256), np.float32)), cache=up(c.buf), dst=be.alloc(1024), pos=up(b.pos), pages=up(b.pages),
                q_start=up(b.q_start), lens=up(b.lens), geom=geom_of(c), batch=batch_of(b), n_head=4, lse=be.alloc(16))
    be.run_kv8(AttentionKv8(**good))
    for name, word in (("q", "q is"), ("cache", "cache"), ("dst", "dst"), ("pos", "pos"), ("pages", "pages"), ("q_start", "q_start"),
                       ("lens", "lens"), ("lse", "lse")):
        small = be.alloc(good[name].len_bytes() - 4)
        with pytest.raises(InfrError) as e:
            be.run_kv8(AttentionKv8(**{**good, name: small}))
        assert e.value.status == Status.Invalid and word in e.value.msg and "too small" in e.value.msg
        if name != "lse":
            with pytest.raises(InfrError) as e:
                be.run_kv8(AttentionKv8(**{**good, name: None}))
            assert e.value.status == Status.Invalid and "unbound" in e.value.msg
    with pytest.raises(InfrError) as e:
        be.run_kv8(AttentionKv8(**{**good, "dst": good["q"]}))
    assert e.value.status == Status.Invalid and "overlaps" in e.value.msg
    with pytest.raises(InfrError) as e:
        be.run_kv8(AttentionKv8(**{**good, "lse": good["dst"]}))
    assert e.value.status == Status.Invalid and "overlap" in e.value.msg
    with pytest.raises(InfrError) as e:
        be.run_kv8(AttentionKv8(**{**good, "n_head": 3}))
    assert e.value.status == Status.Unsupported
    odd = be.wrap(good["cache"].device_addr() + 4, c.nbytes)
    with pytest.raises(InfrError) as e:
        be.run_kv8(AttentionKv8(**{**good, "cache": odd}))
    assert e.value.status == Status.Invalid and "misaligned" in e.value.msg
    lens = up(np.array([70], np.int32))
    with pytest.raises(InfrError) as e:
        be.run_kv8(EvictKv8(good["cache"], good["pages"], lens, up(np.zeros((1, 1), np.int32)), lens, be.alloc(512), geom_of(c), n_seq=1,
                            max_pages=2, keep=64))
    assert e.value.status == Status.Invalid and "overlaps" in e.value.msg
    g, binds = Graph(), Bindings()
    t = [g.input(TensorDesc((4,), DType.F32)) for _ in range(7)]
    g.push(AttentionKv8(*t, geom_of(c), batch_of(b), 4))
    plan = be.compile(g)
    for x in t:
        binds.bind(x, good["cache"])
    binds.slots[t[3].id] = None
    with pytest.raises(InfrError) as e:
        be.execute(plan, binds)
    assert e.value.status == Status.Invalid and "pos is unbound" in e.value.msg
    g = Graph()
    t = [g.input(TensorDesc((4,), DType.F32)) for _ in range(7)]
    g.push(AttentionKv8(*t, Kv8(4, 2, 300, 1), batch_of(b), 4))
    with pytest.raises(InfrError) as e:
        be.compile(g)
    assert e.value.status == Status.Unsupported and "head_dim" in e.value.msg


@gpu
def test_calls_with_another_device_current(be):
    """One device here: the entry points may not depend on which one the caller's thread has current."""
    hip = ctypes.CDLL("libamdhip64.so")
    n = ctypes.c_int()
    assert hip.hipGetDeviceCount(ctypes.byref(n)) == 0
    if n.value < 2:
        pytest.skip("one device")
    assert hip.hipSetDevice(1) == 0
    try:
        rng = np.random.default_rng(33)
        c, pages, _ = filled(rng, "i8", 16, 2, 64, (70,))
        check_attention(be, c, pages, [1], [70], orc.Mode(4))
    finally:
        hip.hipSetDevice(0)
