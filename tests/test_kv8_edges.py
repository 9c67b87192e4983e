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
