"""CPU: what the cache and log-probability entry points refuse, before they
touch a device (include/quantr_cuda.h, Part 3)."""
import ctypes

import pytest

import quantr

BAD_ARG, UNSUPPORTED, TOO_LARGE, WORKSPACE, OK = 3, 4, 7, 8, 0
P = 1 << 20  # an address that is never read


def pool(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, n_pages=8, n_layers=2, n_kv_heads=2, page_tokens=64, head_dim=64)
    d.update(kw)
    return quantr.Kv8Pool(**d)


def tables(**kw):
    d = dict(table=P, lens=P, refs=P, slots=4, max_pages=4)
    d.update(kw)
    return quantr.Kv8Tables(**d)


def batch(**kw):
    d = dict(slot=None, start=None, B=2, max_rows=1)
    d.update(kw)
    return quantr.Kv8Batch(**d)


def ref(x):
    return None if x is None else ctypes.byref(x)


def append(p=None, t=None, b=None, k=P, ldk=128, v=P, ldv=128, type_=0, layer=0, null=None):
    args = {"pool": p or pool(), "tables": t or tables(), "batch": b or batch()}
    if null:
        args[null] = None
    L = quantr.lib()
    return [getattr(L, f)(k, ldk, v, ldv, type_, ref(args["pool"]), ref(args["tables"]), ref(args["batch"]), layer, None)
            for f in ("quantr_kv8_append_dev", "quantr_kv8_read_dev")]


@pytest.mark.parametrize("want,kw", [
    (BAD_ARG, dict(null="pool")), (BAD_ARG, dict(null="tables")), (BAD_ARG, dict(null="batch")),
    (BAD_ARG, dict(p=pool(k=None))), (BAD_ARG, dict(p=pool(v_scale=None))), (BAD_ARG, dict(p=pool(k=P + 8))),
    (BAD_ARG, dict(p=pool(k_scale=P + 2))), (BAD_ARG, dict(p=pool(n_pages=0))), (BAD_ARG, dict(p=pool(n_layers=-1))),
    (BAD_ARG, dict(p=pool(n_kv_heads=0))), (BAD_ARG, dict(p=pool(page_tokens=16))), (BAD_ARG, dict(p=pool(page_tokens=48))),
    (BAD_ARG, dict(p=pool(head_dim=0))), (BAD_ARG, dict(p=pool(head_dim=72))), (TOO_LARGE, dict(p=pool(head_dim=144), ldk=999, ldv=999)),
    (TOO_LARGE, dict(p=pool(n_pages=1 << 30))), (BAD_ARG, dict(t=tables(table=None))), (BAD_ARG, dict(t=tables(lens=None))),
    (BAD_ARG, dict(t=tables(refs=None))), (BAD_ARG, dict(t=tables(slots=0))), (BAD_ARG, dict(t=tables(max_pages=0))),
    (BAD_ARG, dict(b=batch(B=-1))), (BAD_ARG, dict(b=batch(max_rows=-2))), (BAD_ARG, dict(layer=2)), (BAD_ARG, dict(layer=-1)),
    (UNSUPPORTED, dict(type_=8)), (UNSUPPORTED, dict(type_=2)), (BAD_ARG, dict(k=None)), (BAD_ARG, dict(v=None)),
    (BAD_ARG, dict(ldk=127)), (BAD_ARG, dict(ldv=0)), (OK, dict(b=batch(B=0))), (OK, dict(b=batch(max_rows=0), k=None)),
    (TOO_LARGE, dict(b=batch(B=1 << 20, max_rows=1 << 20))),
])
def test_append_and_read(want, kw):
    assert append(**kw) == [want, want]


def attend(p=None, t=None, b=None, out=P, ldo=256, q=P, ldq=256, type_=0, H=4, layer=0, scale=1.0, window=0, max_len=64,
           ws=P, ws_bytes=1 << 30):
    return quantr.lib().quantr_kv8_attend_dev(out, ldo, q, ldq, type_, H, ref(p or pool()), ref(t or tables()),
                                              ref(b or batch()), layer, scale, window, max_len, None, ws, ws_bytes, None)


@pytest.mark.parametrize("want,kw", [
    (BAD_ARG, dict(p=pool(page_tokens=8))), (BAD_ARG, dict(t=tables(slots=-1))), (BAD_ARG, dict(b=batch(B=-1))),
    (BAD_ARG, dict(H=0)), (BAD_ARG, dict(H=3)), (BAD_ARG, dict(window=-1)), (BAD_ARG, dict(max_len=-1)),
    (BAD_ARG, dict(scale=float("nan"))), (BAD_ARG, dict(scale=float("inf"))), (BAD_ARG, dict(out=None)),
    (BAD_ARG, dict(q=None)), (BAD_ARG, dict(ldo=255)), (BAD_ARG, dict(ldq=255)), (UNSUPPORTED, dict(type_=12)),
    (BAD_ARG, dict(layer=5)), (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(ws=P + 16)), (WORKSPACE, dict(ws_bytes=4096)),
    (TOO_LARGE, dict(b=batch(max_rows=1 << 30))), (OK, dict(b=batch(B=0))),
])
def test_attend(want, kw):
    assert attend(**kw) == want


def test_pages():
    L, p, t = quantr.lib(), pool(), tables()
    other = tables(table=2 * P, lens=2 * P, refs=2 * P)
    sel = L.quantr_kv8_select_dev
    assert sel(ref(other), ref(t), None, ref(p), None) == BAD_ARG
    assert sel(None, ref(t), P, ref(p), None) == BAD_ARG
    assert sel(ref(t), ref(t), P, ref(p), None) == BAD_ARG
    for kw in (dict(slots=3), dict(max_pages=5), dict(table=P), dict(lens=P), dict(refs=P)):
        d = dict(table=2 * P, lens=2 * P, refs=2 * P)
        d.update(kw)
        assert sel(ref(tables(**d)), ref(t), P, ref(p), None) == BAD_ARG
    assert sel(ref(other), ref(t), P, ref(pool(head_dim=8)), None) == BAD_ARG
    n = quantr.kv8_pages_workspace_bytes(p, t)
    ext = L.quantr_kv8_extend_dev
    assert ext(ref(p), ref(t), P, None, -1, None, P, n, None) == BAD_ARG
    assert ext(ref(p), ref(t), None, None, 5, None, P, n, None) == BAD_ARG
    assert ext(ref(p), ref(t), P, None, 1025, None, P, n, None) == TOO_LARGE
    assert ext(ref(p), ref(t), P, None, 2, None, P, n - 1, None) == WORKSPACE
    assert ext(ref(p), ref(t), P, None, 2, None, P + 64, n, None) == WORKSPACE
    assert ext(ref(p), ref(t), P, None, 0, None, P, n, None) == OK
    assert L.quantr_kv8_compact_dev(ref(p), ref(t), None, None, None, n, None) == WORKSPACE
    assert L.quantr_kv8_compact_dev(ref(p), ref(tables(slots=0)), None, None, P, n, None) == BAD_ARG
    cp = L.quantr_kv8_copy_pages_dev
    assert cp(ref(p), None, P, 1, None) == BAD_ARG
    assert cp(ref(p), P, P, -1, None) == BAD_ARG
    assert cp(ref(p), None, None, 0, None) == OK


def logprobs(x=P, ldl=100, type_=0, rows=2, V=100, temp=1.0, token=P, logprob=P, k=0):
    return quantr.lib().quantr_logprobs_dev(x, ldl, type_, rows, V, temp, token, logprob, None, None, k, None, None, None,
                                            0, None)


@pytest.mark.parametrize("want,kw", [
    (UNSUPPORTED, dict(type_=8)), (BAD_ARG, dict(rows=-1)), (BAD_ARG, dict(V=0)), (BAD_ARG, dict(k=-1)),
    (TOO_LARGE, dict(k=65)), (BAD_ARG, dict(ldl=99)), (BAD_ARG, dict(temp=0.0)), (BAD_ARG, dict(temp=-1.0)),
    (BAD_ARG, dict(temp=float("nan"))), (BAD_ARG, dict(temp=float("inf"))), (BAD_ARG, dict(temp=1e-42)),
    (BAD_ARG, dict(x=None)), (BAD_ARG, dict(x=P + 2)), (BAD_ARG, dict(x=P + 1, type_=30)), (BAD_ARG, dict(token=None)),
    (OK, dict(rows=0, x=None)),
])
def test_logprobs(want, kw):
    assert logprobs(**kw) == want


def test_python_raises():
    with pytest.raises(quantr.QuantrError) as e:
        quantr.kv8_append_dev(None, 0, None, 0, 0, pool(), tables(), batch(), 0)
    assert e.value.code == BAD_ARG
    with pytest.raises(quantr.QuantrError) as e:
        quantr.logprobs_dev(P, 10, 3, 1, 10, None, None, None, 0, None, None, None, 0)
    assert e.value.code == UNSUPPORTED
    assert "page" in quantr.lib().quantr_gpu_error_string(11).decode()
