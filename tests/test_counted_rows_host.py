"""Argument checks of ma_linear_counted_rows before any launch (no GPU)."""
import pytest

from maester_amd import _lib

P = 0x1000


def _call(e=P, es=64, targets=P, rows=4, vocab=100, dim=64, copies=1, out=P, dtype=1):
    return _lib.lib().ma_linear_counted_rows(e, es, targets, rows, vocab, dim, -100, copies, out, dtype, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(e=None), -1, "NULL"), (dict(targets=None), -1, "NULL"), (dict(out=None), -1, "NULL"), (dict(e=P + 8), -1, "aligned"),
    (dict(out=P + 4), -1, "aligned"), (dict(rows=0), -1, "rows"), (dict(rows=1 << 26), -1, "rows"), (dict(vocab=0), -1, "vocab"),
    (dict(dim=60), -2, "dim"), (dict(dim=65544, es=65544), -2, "dim"), (dict(es=56), -1, "e_stride"), (dict(es=68), -1, "e_stride"),
    (dict(copies=0), -1, "copies"), (dict(copies=9), -1, "copies"), (dict(dtype=7), -1, "dtype")])
def test_refusals(kw, code, text):
    assert _call(**kw) == code and text in _lib.lib().ma_last_error().decode()
