"""What attn_cross refuses, and its workspace: host code, no GPU. Every refused
call names addresses that nothing reads."""
import ctypes

import pytest
import torch

import synth_hip as S
from test_kv_checks import BAD, F, I, NOT_HERE, Q4, Q8, R, mk


def attend(**over):
    a = dict(q=mk(F, 64, 8, 9, 3), k=mk(F, 64, 2, 900, 3), v=mk(F, 64, 2, 900, 3), length=mk(I, 3), count=mk(I, 3), scale=0.125,
             work=mk(F, 1 << 22), y=mk(F, 64, 8, 9, 3))
    a.update(over)
    return S.load().shp_attn_cross(R(a["q"]), R(a["k"]), R(a["v"]), R(a["length"]), R(a["count"]), a["scale"], R(a["work"]), R(a["y"]), None)


def floats(q, k):
    n = ctypes.c_int64(-7)
    st = S.load().shp_attn_cross_work(R(q), R(k), ctypes.byref(n))
    return n.value if st == S.OK else -st


def test_refusals():
    for name in ("q", "k", "v", "y"):
        assert attend(**{name: None}) == BAD, name
    for shape in ((64, 7, 9, 3), (96, 8, 9, 3), (64, 8, 9, 2)):
        assert attend(q=mk(F, *shape), y=mk(F, *shape)) == BAD, shape
    assert attend(v=mk(F, 64, 2, 899, 3)) == BAD and attend(y=mk(F, 64, 8, 8, 3)) == BAD
    assert attend(v=mk(S.TYPE_BF16, 64, 2, 900, 3)) == NOT_HERE and attend(q=mk(S.TYPE_BF16, 64, 8, 9, 3)) == NOT_HERE
    assert attend(k=mk(Q4, 64, 2, 900, 3), v=mk(Q8, 64, 2, 900, 3)) == NOT_HERE
    assert attend(y=mk(S.TYPE_F16, 64, 8, 9, 3)) == NOT_HERE
    for scale in (float("nan"), float("inf"), 3e38):
        assert attend(scale=scale) == BAD
    for name in ("length", "count"):
        assert attend(**{name: mk(I, 2)}) == BAD and attend(**{name: mk(F, 3)}) == BAD
        assert attend(**{name: mk(I, 3, at=(1 << 43) + 2)}) == NOT_HERE
    big = mk(S.TYPE_F16, 258, 2, 900, 3)
    assert attend(k=big, v=big, q=mk(F, 258, 8, 9, 3), y=mk(F, 258, 8, 9, 3)) == NOT_HERE
    for name, shape in (("q", (64, 8, 9, 3)), ("k", (64, 2, 900, 3)), ("v", (64, 2, 900, 3))):
        first = mk(F, *shape)
        assert attend(**{name: first, "y": mk(F, 64, 8, 9, 3, at=first.data)}) == NOT_HERE, name
        assert attend(**{name: first, "work": mk(F, 1 << 22, at=first.data)}) == NOT_HERE, name
    deep = mk(Q4, 64, 2, (1 << 30) + 1, 1)
    assert attend(q=mk(F, 64, 8, 1, 1), y=mk(F, 64, 8, 1, 1), k=deep, v=deep, length=None, count=None) == NOT_HERE


def test_workspace():
    q, k = mk(F, 64, 8, 9, 3), mk(F, 64, 2, 900, 3)
    need = floats(q, k)
    assert need > 0
    assert attend(work=None) == BAD and attend(work=mk(F, need - 1)) == BAD and attend(work=mk(S.TYPE_F16, need)) == BAD
    assert attend(work=mk(F, need, at=(1 << 43) + 4)) == NOT_HERE
    assert floats(q, mk(F, 64, 2, 60, 3)) == 0 and floats(mk(F, 64, 8, 30000, 3), k) == 0
    assert floats(mk(F, 64, 7, 9, 3), k) == -BAD and floats(mk(S.TYPE_F16, 64, 8, 9, 3), k) == -NOT_HERE
    assert S.load().shp_attn_cross_work(R(q), R(k), None) == BAD


def test_binding_raises(monkeypatch):
    monkeypatch.setattr(S, "_stream", lambda: 0)
    q, k = torch.zeros(1, 2, 4, 64), torch.zeros(1, 9, 2, 64)
    for call, status in ((lambda: S.attn_cross(q, k, k[:, :8]), BAD), (lambda: S.attn_cross(q[:, :, :3], k, k), BAD),
                         (lambda: S.attn_cross_work(q.half(), k), NOT_HERE), (lambda: S.attn_cross(q, k, k.half()), NOT_HERE),
                         (lambda: S.attn_cross(q, k, k, out=q), NOT_HERE)):
        with pytest.raises(S.ShpError) as e:
            call()
        assert e.value.status == status
