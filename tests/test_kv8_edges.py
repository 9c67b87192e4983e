"""The 8-bit KV cache's operators where their arithmetic could go wrong: documents that begin behind a row, value scales
and weights many powers of two apart, values next to the largest f32, caps and positions of any size. Against the plain
64-bit implementations of tests/kv8_oracle.py."""
import numpy as np
import pytest

from tests import kv8_oracle as orc
from tests.test_kv8 import TYPES, Dev, close, filled, gpu, rows_of


# forms of AttentionKv8 by the shape that a call states (four query heads, 256 compute units): least max_q, the table's width
FORMS = {"few rows": (0, None), "64 rows": (140, None), "128 rows": (512 * 64 + 1, None), "128 rows in parts": (5120, 40)}


def batch_in_form(form, news, lens, pages, pos=None):
    """A batch whose stated shape takes this form, with rows behind the last sequence's where the form needs more."""
    max_q, max_pages = FORMS[form]
    rows = max(max_q, sum(news))
    return orc.Batch(list(news), list(lens), pages, pos=pos, rows=rows, max_q=max(max_q, *news, 1), max_pages=max_pages)


def padded(a, rows, value=0):
    return np.concatenate([a, np.full(rows - len(a), value, np.asarray(a).dtype)])


# ---------------------------------------------------------------- masks

@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("kw", [dict(causal=False), dict(prefix=True), dict(causal=False, window=40), dict(prefix=True, window=70)], ids=str)
@pytest.mark.parametrize("form,news", [("few rows", 3), ("64 rows", 200), ("128 rows", 200), ("128 rows in parts", 200)])
def test_documents_that_begin_behind_every_row(be, type_, kw, form, news):
    """A row whose document begins behind it sees the document's tokens all the same, where the call is not causal or the
    tokens lie in the prefix; the sums of weights with the lse that comes out of it are those of the definition."""
    rng = np.random.default_rng(40)
    n_len = 230
    c, pages, _ = filled(rng, type_, 16, 2, 64, (n_len,))
    c.sums[...] = 0.5
    b = batch_in_form(form, (news,), (n_len,), pages)
    kw = dict(kw, first=padded(np.arange(n_len - news, n_len) + 1, b.rows))
    if kw.get("prefix"):
        kw["prefix"] = [n_len]
    m = orc.Mode(4, **kw)
    q = rng.standard_normal((b.rows, 4 * 64)).astype(np.float32)
    dev = Dev(be, c)
    out, lse = dev.attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    assert np.isfinite(want_l[:news - 1]).all() and np.isneginf(want_l[news - 1]).all()
    close(out, want, tol)
    close(lse, want_l, ltol)
    sums, stol = orc.score(c, b, m, q, lse, 1.0)
    dev.score(b, m, q, lse)
    assert (np.abs(dev.pull().sums - sums) <= stol).all()


@gpu
@pytest.mark.parametrize("form,news", [("few rows", 3), ("64 rows", 150), ("128 rows", 150), ("128 rows in parts", 150)])
@pytest.mark.parametrize("first", [-2 ** 31, -2 ** 31 + 5, -1])
def test_documents_that_begin_before_all_positions(be, form, news, first):
    """No position is negative: such a document's beginning masks nothing, also where positions have gaps."""
    rng = np.random.default_rng(41)
    n_len = 180
    pos = np.cumsum(rng.integers(1, 6, n_len)).astype(np.int32)
    c, pages, _ = filled(rng, "i8", 32, 2, 64, (n_len,), pos=pos)
    b = batch_in_form(form, (news,), (n_len,), pages, pos=pos[n_len - news:])
    q = rng.standard_normal((b.rows, 4 * 64)).astype(np.float32)
    out, lse = Dev(be, c).attention(b, orc.Mode(4, first=np.full(b.rows, first)), q)
    want, want_l, tol, ltol = orc.attention(c, b, orc.Mode(4), q)
    close(out, want, tol)
    close(lse, want_l, ltol)


# ---------------------------------------------------------------- weights

def weights_of(c, b, m, q, head):
    """(p, largest p is 1; scores; which pairs see each other; sum |q k| of each pair) of sequence 0, f64 [rows, tokens]."""
    n, n_len = int(b.q_start[1]), int(b.lens[0])
    sc, see, size = orc.scores(c, b, m, q, 0, 0, n, n_len, head)
    sc = np.where(see, sc, -np.inf)
    return np.exp(sc - sc.max(-1, keepdims=True)), sc, see, size


def relative_tolerance(c, b, m, q, head):
    """What the weighted sum of values may be off, [rows, dim], relative to the sum of |weight * value| of its column.

    A weight is off by its score's error (a sum of dim products, 2^-24 for each addition and 2^-22 for the operand and the
    products' roundings, each of |q k|; 2^-21 of the score itself, which counts in log2 units from the row's largest;
    2^-20 for the exponential and the scales' logarithm) and by 2^-22 for its two halves. Below that a product of weight and scale
    counts to 2^-33 of the row's largest. The sums over n tokens add n * 2^-24 and the quotient doubles it all."""
    p, sc, see, size = weights_of(c, b, m, q, head)
    h = head // (m.n_head // c.n_kv)
    n_len = int(b.lens[0])
    v = np.abs(c.values("v", b.pages[0], h, n_len))
    scale = np.repeat(c.v_scale[b.pages[0, :-(-n_len // 64)], h].reshape(-1).astype(np.float64), c.block)[:n_len]
    far = np.where(see, sc.max(-1, keepdims=True) - sc, 0)
    eps = size * (c.dim * 2.0 ** -24 + 2.0 ** -22) + (np.abs(np.where(see, sc, 0)) + far) * 2.0 ** -21 + 2.0 ** -20 + 2.0 ** -22
    least = (p * scale).max(-1, keepdims=True) * 2.0 ** -33 / scale  # of a weight, in units of p
    l = p.sum(-1, keepdims=True)
    return ((p * eps) @ v + (p @ v) * (p * eps).sum(-1, keepdims=True) / l + 2 * n_len * 2.0 ** -24 * (p @ v) + np.where(see, least, 0) @ v) / l


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("block,at", [(16, 0), (16, 130), (64, 0), (64, 128)])
@pytest.mark.parametrize("form,news", [("few rows", 1), ("few rows", 7), ("64 rows", 140), ("128 rows", 140), ("128 rows in parts", 140)])
def test_a_block_of_large_values_and_next_to_no_weight(be, type_, dim, block, at, form, news):
    """The weight lies on blocks whose scale is far below another visible block's: their values keep their bits."""
    if dim > 128 and form == "128 rows":
        pytest.skip("the same code as with 64 columns, on inputs of 130 MB")
    rng = np.random.default_rng(42)
    n_len = 150
    for ratio in (0, 14, 24, 30, 40, 52, 57, 64, 90):
        c = orc.Cache(5, 2, dim, 1, type_, block)
        pages = [[4, 0, 2]]
        new = orc.Batch([n_len], [n_len], pages)
        k, v = (rng.standard_normal((n_len, 2 * dim)).astype(np.float32) for _ in range(2))
        k.reshape(n_len, 2, dim)[:, :, 0] = 0
        big = slice(at, min(at + block, n_len))
        v[big] *= np.float32(2.0 ** ratio)
        k[big] = 0
        k.reshape(n_len, 2, dim)[big, :, 0] = -40
        orc.write(c, new, k, v)
        b = batch_in_form(form, (news,), (n_len,), pages)
        m = orc.Mode(4, scale=1.0, causal=False)
        q = np.zeros((b.rows, 4, dim), np.float32)
        q[..., 0] = 1
        q[:, 1::2, 1:] = 0.03 * rng.standard_normal((b.rows, 2, dim - 1))
        q = q.reshape(b.rows, -1)
        out, lse = Dev(be, c).attention(b, m, q)
        want, want_l, _, ltol = orc.attention(c, b, m, q)
        close(lse, want_l, ltol)
        for head in range(4):
            cols = slice(head * dim, (head + 1) * dim)
            off = np.abs(out[:news, cols] - want[:news, cols]) / relative_tolerance(c, b, m, q, head)
            assert off.max() <= 1, f"2^{ratio}, head {head}: {off.max():.3g} tolerances"


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("form,news", [("few rows", 1), ("few rows", 4), ("few rows", 8), ("64 rows", 64), ("128 rows", 64), ("128 rows in parts", 64)])
def test_small_weights_are_rounded_to_the_nearest(be, type_, form, news):
    """One token has all but 2^-19 of the weight and the value 0: what is left are weights near the smallest ones that
    count, in steps of 2^-24 where the largest product of weight and scale is at 2^10 or above. Each is off by half a step
    at most, and all of a row by the same."""
    rng = np.random.default_rng(43)
    c = orc.Cache(3, 2, 64, 1, type_, 64)
    pages = [[1]]
    new = orc.Batch([64], [64], pages)
    k, v = np.zeros((64, 2, 64), np.float32), np.ones((64, 2, 64), np.float32)
    k[1:, :, 0] = -1
    v[0] = 0
    orc.write(c, new, k.reshape(64, -1), v.reshape(64, -1))
    b = batch_in_form(form, (news,), (64,), pages)
    m = orc.Mode(4, scale=1.0, causal=False)
    q = np.zeros((b.rows, 4, 64), np.float32)
    q[..., 0] = rng.uniform(16, 18, (b.rows, 4))
    q = q.reshape(b.rows, -1)
    out, _ = Dev(be, c).attention(b, m, q)
    want = orc.attention(c, b, m, q)[0]
    for head in range(4):
        cols = slice(head * 64, (head + 1) * 64)
        p = weights_of(c, b, m, q, head)[0]
        # half a step of each of 63 weights, of a largest one that stands at 2^10 or above; 2^-16 covers the f32 arithmetic
        tol = 63 * 2.0 ** -35 / p.sum(-1, keepdims=True) + 2.0 ** -16 * want[:news, cols]
        off = np.abs(out[:news, cols] - want[:news, cols]) / tol
        assert off.max() <= 1, f"head {head}: {off.max():.3g} tolerances"


@gpu
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 200])
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 125])
@pytest.mark.parametrize("form,news,n_len", [("few rows", 1, 150), ("few rows", 7, 150), ("few rows", 1, 3001), ("64 rows", 140, 150), ("128 rows", 140, 150),
                                             ("128 rows in parts", 140, 1500)])
def test_values_next_to_the_largest(be, type_, dim, size, form, news, n_len):
    """Weighted means of finite values are finite."""
    rng = np.random.default_rng(44)
    c = orc.Cache(-(-n_len // 64), 1, dim, 1, type_, 16)
    pages = [rng.permutation(c.n_pages).tolist()]
    new = orc.Batch([n_len], [n_len], pages)
    k = rng.standard_normal((n_len, dim)).astype(np.float32)
    v = (rng.uniform(0.5, 1.5, (n_len, dim)) * size).astype(np.float32)
    orc.write(c, new, k, v)
    b = batch_in_form(form, (news,), (n_len,), pages)
    m = orc.Mode(4)
    q = rng.standard_normal((b.rows, 4 * dim)).astype(np.float32)
    out, lse = Dev(be, c).attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    close(out, want, tol)
    close(lse, want_l, ltol)


# ---------------------------------------------------------------- caps and positions of any size

@gpu
@pytest.mark.parametrize("softcap,scale_q", [(1e-10, 1.0), (1e-25, 1.0), (1e-37, 1.0), (1e-44, 1.0), (1e25, 1e22), (3e38, 1e30)])
@pytest.mark.parametrize("form,news", [("few rows", 3), ("64 rows", 140), ("128 rows", 140)])
def test_caps_of_any_size(be, softcap, scale_q, form, news):
    """c * tanh(s / c) is a number for every finite score and every cap, scores of 0 among them."""
    rng = np.random.default_rng(45)
    n_len = 150
    c, pages, _ = filled(rng, "i8", 16, 2, 64, (n_len,))
    c.sums[...] = 0.5
    b = batch_in_form(form, (news,), (n_len,), pages)
    m = orc.Mode(4, softcap=float(np.float32(softcap)))
    q = (scale_q * rng.standard_normal((b.rows, 4 * 64))).astype(np.float32)
    q[::2] = 0
    dev = Dev(be, c)
    out, lse = dev.attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    close(out, want, tol)
    close(lse, want_l, ltol)
    if scale_q == 1.0:  # (beyond, an lse's own rounding is more than an exponential bears)
        sums, stol = orc.score(c, b, m, q, lse, 1.0)
        dev.score(b, m, q, lse)
        assert (np.abs(dev.pull().sums - sums) <= stol).all()


@gpu
@pytest.mark.parametrize("form,news", [("few rows", 3), ("64 rows", 250), ("128 rows", 250), ("128 rows in parts", 250)])
@pytest.mark.parametrize("causal", [True, False])
def test_the_bias_by_distance_is_exact_at_far_positions(be, form, news, causal):
    """Two documents in one sequence, the second at positions from 2^27 on: distances within it are small numbers. Its rows
    see nothing of the first one, so their scores are of ordinary size, and the oracle's tolerances are."""
    rng = np.random.default_rng(46)
    n_len, cut = 250, 100
    pos = np.concatenate([np.arange(cut), 2 ** 27 + 1 + 3 * np.arange(n_len - cut)]).astype(np.int32)
    c, pages, _ = filled(rng, "i8", 16, 2, 64, (n_len,), pos=pos)
    c.sums[...] = 0.5
    b = batch_in_form(form, (news,), (n_len,), pages, pos=pos[n_len - news:])
    first = np.where(np.arange(n_len) < cut, 0, pos[cut])[n_len - news:]
    m = orc.Mode(4, slopes=2.0 ** -np.arange(1, 5), first=padded(first, b.rows), causal=causal)
    q = rng.standard_normal((b.rows, 4 * 64)).astype(np.float32)
    dev = Dev(be, c)
    out, lse = dev.attention(b, m, q)
    want, want_l, tol, ltol = orc.attention(c, b, m, q)
    assert ltol[max(0, news - (n_len - cut)):news].max() < 1e-3
    close(out, want, tol)
    close(lse, want_l, ltol)
    sums, stol = orc.score(c, b, m, q, lse, 1.0)
    dev.score(b, m, q, lse)
    assert (np.abs(dev.pull().sums - sums) <= stol).all()
