"""Refusals of the generation entry points that need no GPU: sizes and types come before handles, handles before devices."""
import ctypes as C

import numpy as np
import pytest

from zillaphp_b200 import native


@pytest.fixture(scope="module")
def lib():
    return native.load()


def test_rope_table_refusals(lib):
    ok = dict(table=1, rot=64, base=10000.0, scaling=3, factor=4.0, original=4096, slow=1.0, fast=32.0)
    call = lambda **kw: lib.rope_table_dev(*{**ok, **kw}.values())  # noqa: E731
    assert call() == -1 and "handle" in native.last_error()
    for bad in (dict(rot=63), dict(rot=0), dict(rot=258), dict(rot=-2), dict(base=0.0), dict(base=-1.0), dict(base=float("nan")),
                dict(base=float("inf")), dict(scaling=4), dict(scaling=-1), dict(factor=0.0), dict(factor=float("nan")),
                dict(original=0), dict(slow=32.0), dict(fast=float("nan")), dict(fast=float("inf"))):
        assert call(**bad) == -2, bad
    assert call(scaling=0, factor=0.0) == -1          # without scaling its numbers are not looked at


def test_rope_refusals(lib):
    ok = dict(x=1, x_off=0, x_ld=512, y=2, y_off=0, y_ld=512, pos=3, table=4, type=1, rows=8, heads=4, dim=128, rot=64, inter=0, inv=0)
    call = lambda **kw: lib.rope_dev(*{**ok, **kw}.values())  # noqa: E731
    assert call() == -1
    for bad in (dict(type=3), dict(type=-1), dict(rows=-1), dict(heads=0), dict(dim=0), dict(dim=257), dict(rot=65), dict(rot=130), dict(rot=0),
                dict(x_off=1), dict(x_off=-1), dict(x_ld=511), dict(y_ld=500), dict(y_off=8), dict(inter=2), dict(inv=2), dict(inter=-1),
                dict(heads=1 << 20, x_ld=1 << 30, y_ld=1 << 30), dict(y=4), dict(y=3),
                dict(y=1, y_ld=600), dict(y=1, x_ld=1000, y_ld=1000, y_off=8)):
        assert call(**bad) == -2, bad
    assert call(y=1) == -1 and call(y=1, x_ld=1024, y_ld=1024, y_off=512) == -1       # in place, or beside it in the row


def test_kv_refusals(lib):
    for bad in ((4, 24, 2, 64, 1), (4, 8, 2, 64, 1), (4, 256, 2, 64, 1), (4, 16, 2, 96, 1), (4, 16, 2, 256, 1), (4, 16, 0, 64, 1), (0, 16, 2, 64, 1),
                (4, 16, 2, 64, 0), (4, 16, 2, 64, 3), (2 ** 30, 128, 2, 64, 1), (4, 16, 1025, 64, 1)):
        assert lib.zilla_kv_create(*bad) == -2, bad
    assert lib.zilla_kv_destroy(77) == -1 and lib.zilla_kv_k_id(77) == -1 and lib.zilla_kv_v_id(0) == -1
    assert lib.zilla_kv_append(*([77] + [1] * 22)) == -1
    assert lib.zilla_kv_attend(*([77] + [1] * 13), C.c_float(1.0), 1) == -1
    assert lib.zilla_kv_attend_work(77, 1, 1, 1, 1, 1, 1) == -1


def test_draft_verify_refusals(lib):
    ok = dict(p=1, p_ld=100, q=2, q_ld=100, draft=3, u=4, start=5, tokens=6, accepted=7, batch=2, rows=6, vocab=100)
    call = lambda **kw: lib.draft_verify_dev(*{**ok, **kw}.values())  # noqa: E731
    assert call() == -1 and call(q=0, q_ld=0) == -1
    for bad in (dict(batch=-1), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 29, p_ld=1 << 29, q_ld=1 << 29), dict(p_ld=99), dict(q_ld=99),
                dict(tokens=3), dict(accepted=5), dict(tokens=7), dict(tokens=1), dict(accepted=4)):
        assert call(**bad) == -2, bad


def test_integers_of_other_types(lib):
    """The entry points without argtypes take numpy integers through native.call and refuse anything else."""
    args = [np.int64(1), 100, 2, 100, 3, 4, 5, 6, 7, np.int32(2), 6, 100]
    assert native.call(lib.draft_verify_dev, *args) == -1
    with pytest.raises(TypeError):
        native.call(lib.draft_verify_dev, *(args[:-1] + [100.0]))
    assert set(native.PLAIN_INTS) <= set(native.SIGNATURES)


def test_arguments_of_the_plain_entry_points(lib):
    """Direct calls and calls through the Python classes refuse what is no integer, and a wrong number of arguments."""
    args = {"rope_dev": [1, 0, 512, 2, 0, 512, 3, 4, 1, 8, 4, 128, 64, 0, 0], "zilla_kv_append": [77] + [1] * 22,
            "zilla_kv_attend": [77] + [1] * 13 + [C.c_float(1.0), 1], "draft_verify_dev": [1, 100, 2, 100, 3, 4, 5, 6, 7, 2, 6, 100]}
    assert set(args) == native.PLAIN_INTS
    for name, ok in args.items():
        fn = getattr(lib, name)
        assert fn(*ok) == -1, name
        assert fn(*[np.int32(a) if isinstance(a, int) else a for a in ok]) == -1 and fn(*([True] + ok[1:])) == -1
        for few in (ok[:-1], ok + [0], []):
            with pytest.raises(TypeError):
                fn(*few)
        for at in (0, 3, len(ok) - 1):
            for bad in (None, "2", b"2", 2.0, C.c_float(2.0), C.c_int(2), [2]):
                with pytest.raises(TypeError):
                    fn(*(ok[:at] + [bad] + ok[at + 1:]))
                with pytest.raises(TypeError):
                    native.call(fn, *(ok[:at] + [bad] + ok[at + 1:]))
    for scale in (1, 0.5, np.float32(0.5), np.float64(0.5)):
        assert lib.zilla_kv_attend(*(args["zilla_kv_attend"][:14] + [scale, 1])) == -1
    for scale in (None, "1", b"1", C.c_int(1)):
        with pytest.raises(TypeError):
            lib.zilla_kv_attend(*(args["zilla_kv_attend"][:14] + [scale, 1]))
