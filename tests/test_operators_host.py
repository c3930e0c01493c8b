"""Refusals and host arithmetic of the optimizer and token entry points, through the C ABI: nothing here reaches a GPU (every
call is refused, or has nothing to do, before anything is launched)."""
import ctypes as C
import os

import pytest

import oneccl_amd.comp as c

pytestmark = pytest.mark.skipif(not os.path.exists(c.LIB_PATH), reason="libmi_ccl_comp.so not built")

BAD, OK, A = c.INVALID_ARGUMENTS, c.SUCCESS, 0x1000        # A: an address that nothing reads


def test_rows_and_workspace():
    assert c.token_rows(0, 1, 1) == 0
    assert c.token_rows(5, 2, 8) == 10
    assert c.token_rows(5, 2, 8, align=16) == 10 + 8 * 15
    assert c.token_rows(1, 2, 8, align=16) == 2 + 2 * 15          # no more experts than entries have rows to pad
    assert c.token_rows(1000, 2, 8, capacity=10) == 80
    assert c.token_rows(1000, 2, 8, align=4, capacity=10) == 80 + 8 * 3
    assert c.token_sort_workspace(2048, 2, 64) == 0
    assert c.token_sort_workspace(2049, 2, 64) > 0
    for args in ((1, 0, 1, 1, 0), (1, 1, 0, 1, 0), (1, 1, 1025, 1, 0), (1, 1, 1, 0, 0), (1 << 31, 1, 1, 1, 0), (1 << 30, 2, 1, 1, 0),
                 (1 << 22, 1, 1024, 1 << 22, 0), (1, 1, 1, 1 << 31, 0), (1, 1, 1, 1, 1 << 31)):
        with pytest.raises(c.CclError):
            c.token_rows(*args)


def test_sort_refusals():
    f = c.lib().mi_ccl_token_sort
    ok = dict(idx=c.INT32, ids=A, n=3, k=2, e=4, align=1, cap=0, pos=A, cnt=A, off=A, ws=None, wb=0)

    def call(**kw):
        d = dict(ok, **kw)
        return f(d["idx"], d["ids"], d["n"], d["k"], d["e"], d["align"], d["cap"], d["pos"], d["cnt"], d["off"], d["ws"], d["wb"], None)
    for kw in (dict(idx=c.INT8), dict(idx=c.FLOAT32), dict(ids=None), dict(ids=A + 2), dict(idx=c.INT64, ids=A + 4), dict(pos=None), dict(pos=A + 1),
               dict(cnt=None), dict(off=None), dict(off=A + 2), dict(k=0), dict(k=-1), dict(e=0), dict(e=1025), dict(align=0), dict(n=1 << 31),
               dict(n=8193, k=1), dict(n=8193, k=1, ws=A, wb=8), dict(n=8193, k=1, ws=A + 2, wb=1 << 20)):
        assert call(**kw) == BAD, kw


def test_dispatch_refusals():
    f = c.lib().mi_ccl_token_dispatch
    ok = dict(dt=c.BFLOAT16, x=A, ldx=8, n=3, k=2, h=8, pos=A, cnt=A, off=A, e=4, out=A, ldo=8, rows=6, ws=None, wb=0)

    def call(**kw):
        d = dict(ok, **kw)
        return f(d["dt"], d["x"], d["ldx"], d["n"], d["k"], d["h"], d["pos"], d["cnt"], d["off"], d["e"], d["out"], d["ldo"], d["rows"], d["ws"], d["wb"],
                 None)
    for kw in (dict(ws=A + 4, wb=1 << 20), dict(dt=c.INT8), dict(dt=c.FLOAT64), dict(x=None), dict(x=A + 1), dict(dt=c.FLOAT32, out=A + 2), dict(ldx=7), dict(ldo=7), dict(k=0),
               dict(pos=None), dict(cnt=None), dict(off=None), dict(e=0), dict(e=2000), dict(out=None), dict(rows=1 << 31), dict(n=1 << 31)):
        assert call(**kw) == BAD, kw
    for kw in (dict(n=0, x=None, pos=None), dict(h=0, x=None), dict(rows=0, out=None)):
        assert call(**kw) == OK, kw


def test_combine_refusals():
    f = c.lib().mi_ccl_token_combine
    ok = dict(dt=c.FLOAT16, y=A, ldy=8, rows=6, pos=A, w=None, n=3, k=2, h=8, out=A, ldo=8)

    def call(**kw):
        d = dict(ok, **kw)
        return f(d["dt"], d["y"], d["ldy"], d["rows"], d["pos"], d["w"], d["n"], d["k"], d["h"], d["out"], d["ldo"], None)
    for kw in (dict(dt=c.INT32), dict(y=None), dict(y=A + 1), dict(ldy=7), dict(ldo=7), dict(pos=None), dict(out=None), dict(out=A + 1), dict(k=0),
               dict(n=1 << 31), dict(rows=1 << 31), dict(w=A + 2), dict(pos=A + 2)):
        assert call(**kw) == BAD, kw
    assert call(n=0, y=None, pos=None, out=None) == OK
    assert call(h=0, y=None, out=None) == OK


def test_combine_backward_refusals():
    f = c.lib().mi_ccl_token_combine_backward
    ok = dict(dt=c.FLOAT32, g=A, ldg=8, y=A, ldy=8, rows=6, pos=A, w=A, cnt=A, off=A, e=4, n=3, k=2, h=8, gy=A, ldd=8, gw=A, ws=None)

    def call(**kw):
        d = dict(ok, **kw)
        return f(d["dt"], d["g"], d["ldg"], d["y"], d["ldy"], d["rows"], d["pos"], d["w"], d["cnt"], d["off"], d["e"], d["n"], d["k"], d["h"], d["gy"],
                 d["ldd"], d["gw"], d["ws"], 1 << 20, None)
    for kw in (dict(dt=c.INT32), dict(g=None), dict(g=A + 2), dict(ldg=7), dict(y=None), dict(ldy=7), dict(pos=None), dict(cnt=None), dict(off=None),
               dict(gy=None), dict(gy=A + 2), dict(ldd=7), dict(e=0), dict(k=0), dict(n=1 << 31), dict(rows=1 << 31), dict(gw=A + 2), dict(w=A + 1),
               dict(ws=A + 4)):
        assert call(**kw) == BAD, kw
    assert call(n=0, g=None, y=None, pos=None) == OK
    assert call(gw=None, h=0, g=None) == OK
    assert call(gw=None, rows=0, gy=None) == OK


def test_optimizer_calls_refuse_a_missing_plan():
    L = c.lib()
    o = c.AdamwOptions(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1)
    assert L.mi_ccl_fusion_norm(None, None, A, 1.0, 1.0, A, A, 1 << 20, None) == BAD
    assert L.mi_ccl_fusion_adamw(None, c.FLOAT32, A, None, A, 0, A, A, None, None, C.byref(o), None) == BAD
    assert L.mi_ccl_fusion_state_decode(None, A, A, A, c.FLOAT32, A, A, None) == BAD
    assert L.mi_ccl_fusion_state_encode(None, c.FLOAT32, A, A, A, A, A, None) == BAD
    assert L.mi_ccl_fusion_norm_workspace(None) == 0 and L.mi_ccl_fusion_plan_elements(None) == 0


# ---- what the binding asks of tensors in one pass; device -1 is host memory

def tensors():
    return pytest.importorskip("oneccl_amd._tensors", reason="not built")


def test_memory_of_a_tensor():
    import torch
    t = tensors()
    x = torch.zeros(4, 6)
    assert t.memory(x, torch.float32, 24, -1) == x.data_ptr()
    assert t.memory(torch.nn.Parameter(x), torch.float32, 0, -1) == x.data_ptr()
    assert t.memory(x[1], torch.float32, 6, -1) == x.data_ptr() + 24
    assert t.memory(torch.zeros(0), torch.float32, 0, -1) == 0
    for bad in (None, 3, [x], x.t(), x[:, 1:], x.double(), x.to("meta"), x.to_sparse(), torch.zeros(23), x.expand(2, 4, 6)):
        assert t.memory(bad, torch.float32, 24, -1) is None
    for call in ((x, "float32", 24, -1), (x, None, 24, -1), (x, torch.float32, 24, 0), (x, torch.float32, None, -1), (x, torch.float32, 1 << 70, -1),
                 (x, torch.float32, 24, 1.5), (x, torch.float32, 24), ()):
        assert t.memory(*call) is None


def test_rows_of_a_matrix():
    import torch
    t = tensors()
    x = torch.zeros(4, 6)
    assert t.rows(x, 6, torch.float32, -1) == (4, 6, x.data_ptr())
    assert t.rows(x[::2, 1:5], 4, torch.float32, -1) == (2, 12, x.data_ptr() + 4)
    assert t.rows(x[1:2], 6, torch.float32, -1) == (1, 6, x.data_ptr() + 24)
    assert t.rows(x[:0], 6, torch.float32, -1)[:2] == (0, 6)
    assert t.rows(x[:, :1], 1, torch.float32, -1) == (4, 6, x.data_ptr())
    assert t.rows(x[:, :0], 0, torch.float32, -1)[:2] == (4, 6)
    for bad, hidden in ((x, 5), (x[0], 6), (x.t(), 4), (x[:1].expand(4, 6), 6), (x[:, ::2], 3), (x.half(), 6), (x[None], 6), (None, 6), (x.to("meta"), 6)):
        got = t.rows(bad, hidden, torch.float32, -1)
        assert got is None


def test_addresses_of_tensors():
    import array
    import torch
    t = tensors()
    xs = [torch.zeros(n) for n in (3, 0, 5, 1)]
    least = array.array("q", [3, 0, 5, 1])
    for seq in (xs, tuple(xs)):
        assert array.array("Q", t.addresses(seq, torch.float32, least, -1)).tolist() == [x.data_ptr() for x in xs]
    assert t.addresses([], torch.float32, array.array("q"), -1) == b""
    for bad in (xs[:3], xs + xs[:1], [None] + xs[1:], [x.double() for x in xs], xs[::-1], iter(xs), None, xs[:3] + [3]):
        assert t.addresses(bad, torch.float32, least, -1) is None
    assert t.addresses(xs, torch.float32, least, 0) is None
    assert t.addresses(xs, torch.float32, [3, 0, 5, 1], -1) is None
    assert t.addresses(xs[:3] + [torch.zeros(4, 3).t()], torch.float32, least, -1) is None


def test_the_binding_refuses_the_same_without_the_native_pass(monkeypatch):
    import array
    import torch
    t = tensors()
    x = torch.zeros(4, 6)
    for native in (t, False):
        monkeypatch.setattr(c, "_native", native)
        assert c._memory("x", x, torch.float32, 24, -1) == x.data_ptr()
        assert c._rows("x", x, 6, torch.float32, -1) == (4, 6, x.data_ptr())
        address, table = c._table("x", [x, x[1]], torch.float32, array.array("q", [24, 6]), -1)
        assert array.array("Q", table).tolist() == [x.data_ptr(), x[1].data_ptr()]
        for call in (lambda: c._memory("x", x.t(), torch.float32, 24, -1), lambda: c._memory("x", None, torch.float32, 0, -1),
                     lambda: c._rows("x", x, 5, torch.float32, -1), lambda: c._table("x", [x, None], torch.float32, array.array("q", [1, 1]), -1),
                     lambda: c._table("x", [x], torch.float32, array.array("q", [25]), -1),
                     lambda: c._table("x", [x], torch.float16, array.array("q", [1]), -1),
                     lambda: c._table("x", [x], torch.float32, array.array("q", [1]), 0)):
            with pytest.raises(ValueError):
                call()
