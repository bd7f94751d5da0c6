"""CPU: addresses that are not multiples of their elements' size are refused
before anything is launched: on the device such an access is a fault."""
import ctypes

import pytest

import quantr
from test_serve_args import BAD_ARG, OK, P, batch, pool, ref, tables

F32, F16, BF16 = 0, 1, 30
OTHER = dict(table=2 * P, lens=2 * P, refs=2 * P)


def rows_call(name, type_, k, v, b=None, t=None):
    return getattr(quantr.lib(), name)(k, 128, v, 128, type_, ref(pool()), ref(t or tables()), ref(b or batch()), 0, None)


@pytest.mark.parametrize("name", ["quantr_kv8_append_dev", "quantr_kv8_read_dev"])
def test_rows(name):
    for type_, off in ((F32, 1), (F32, 2), (F16, 1), (BF16, 3)):
        assert rows_call(name, type_, P + off, P) == BAD_ARG
        assert rows_call(name, type_, P, P + off) == BAD_ARG
    for field in ("slot", "start"):
        assert rows_call(name, F32, P, P, b=batch(**{field: P + 2})) == BAD_ARG
    for field in ("table", "lens", "refs"):
        assert rows_call(name, F32, P, P, t=tables(**{field: P + 1})) == BAD_ARG


def attend(out=P, q=P, type_=F32, lse=None, b=None, t=None):
    return quantr.lib().quantr_kv8_attend_dev(out, 256, q, 256, type_, 4, ref(pool()), ref(t or tables()), ref(b or batch()),
                                              0, 1.0, 0, 64, lse, P, 1 << 30, None)


def test_attend():
    for type_, off in ((F32, 1), (F32, 2), (F16, 1), (BF16, 3)):
        assert attend(out=P + off, type_=type_) == BAD_ARG
        assert attend(q=P + off, type_=type_) == BAD_ARG
    assert attend(lse=P + 2) == BAD_ARG
    assert attend(b=batch(slot=P + 3)) == BAD_ARG
    assert attend(b=batch(start=P + 2)) == BAD_ARG
    assert attend(t=tables(lens=P + 2)) == BAD_ARG


def test_pages():
    L, p, t = quantr.lib(), pool(), tables()
    n = quantr.kv8_pages_workspace_bytes(p, t)
    assert L.quantr_kv8_select_dev(ref(tables(**OTHER)), ref(t), P + 2, ref(p), None) == BAD_ARG
    for field in OTHER:
        bad = tables(**dict(OTHER, **{field: 2 * P + 2}))
        assert L.quantr_kv8_select_dev(ref(bad), ref(t), P, ref(p), None) == BAD_ARG
        assert L.quantr_kv8_select_dev(ref(t), ref(bad), P, ref(p), None) == BAD_ARG
        assert L.quantr_kv8_extend_dev(ref(p), ref(bad), P, None, 2, None, P, n, None) == BAD_ARG
        assert L.quantr_kv8_compact_dev(ref(p), ref(bad), None, None, P, n, None) == BAD_ARG
    ext = L.quantr_kv8_extend_dev
    assert ext(ref(p), ref(t), P + 1, None, 2, None, P, n, None) == BAD_ARG
    assert ext(ref(p), ref(t), P, P + 2, 2, None, P, n, None) == BAD_ARG
    assert ext(ref(p), ref(t), P, None, 2, P + 3, P, n, None) == BAD_ARG
    assert ext(ref(p), ref(t), P, None, 0, None, P, n, None) == OK
    assert L.quantr_kv8_compact_dev(ref(p), ref(t), P + 2, None, P, n, None) == BAD_ARG
    assert L.quantr_kv8_compact_dev(ref(p), ref(t), None, P + 2, P, n, None) == BAD_ARG
    assert L.quantr_kv8_copy_pages_dev(ref(p), P + 2, P, 1, None) == BAD_ARG
    assert L.quantr_kv8_copy_pages_dev(ref(p), P, P + 2, 1, None) == BAD_ARG


@pytest.mark.parametrize("field", ["token", "logprob", "entropy", "lse", "top_id", "top_logprob"])
def test_logprobs(field):
    a = dict(token=P, logprob=P, entropy=P, lse=P, top_id=P, top_logprob=P)
    a[field] = P + 2
    assert quantr.lib().quantr_logprobs_dev(P, 100, F32, 2, 100, ctypes.c_float(1.0), a["token"], a["logprob"], a["entropy"],
                                            a["lse"], 5, a["top_id"], a["top_logprob"], None, 0, None) == BAD_ARG
