"""What kv_store, kv_load and attn_kv refuse, and the workspace that attn_kv
asks for: host code, no GPU. Every refused call names addresses that nothing
reads."""
import ctypes

import pytest
import torch

import synth_hip as S

UNIT = {S.TYPE_F32: 4, S.TYPE_F16: 2, S.TYPE_BF16: 2, S.TYPE_I32: 4, S.TYPE_Q8_0: 34, S.TYPE_Q4_0: 18, S.TYPE_Q5_K: 176}
BLOCK = {S.TYPE_Q8_0: 32, S.TYPE_Q4_0: 32, S.TYPE_Q5_K: 256}
_at = [1 << 44]
BAD, NOT_HERE = S.ERR_INVALID_ARG, S.ERR_UNSUPPORTED


def mk(type_, *ne, nb=None, at=None):
    t = S.ShpTensor()
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [UNIT[type_], ne[0] // BLOCK.get(type_, 1) * UNIT[type_]]
        nb += [nb[1] * ne[1], nb[1] * ne[1] * ne[2]]
    t.type, t.reserved = type_, 0
    for i in range(4):
        t.ne[i], t.nb[i] = ne[i], nb[i]
    t.data = _at[0] if at is None else at
    if at is None:
        _at[0] += (max(max(ne[i], 1) * nb[i] for i in range(4)) + 4096) // 256 * 256
    return t


def R(t):
    return None if t is None else ctypes.byref(t)


F, I, Q4, Q8 = S.TYPE_F32, S.TYPE_I32, S.TYPE_Q4_0, S.TYPE_Q8_0


def store(load=False, **over):
    a = dict(k=mk(F, 64, 2, 5, 3), v=mk(F, 64, 2, 5, 3), slot=mk(I, 3), count=mk(I, 3), kc=mk(Q4, 64, 2, 9, 3),
             vc=mk(Q4, 64, 2, 9, 3), status=mk(I, 1))
    a.update(over)
    L = S.load()
    if load:
        return L.shp_kv_load(R(a["kc"]), R(a["vc"]), R(a["slot"]), R(a["count"]), R(a["k"]), R(a["v"]), None)
    return L.shp_kv_store(R(a["k"]), R(a["v"]), R(a["slot"]), R(a["count"]), R(a["kc"]), R(a["vc"]), R(a["status"]), None)


@pytest.mark.parametrize("load", [False, True])
def test_store_and_load_refuse(load):
    for name in ("k", "v", "slot", "kc", "vc"):
        assert store(load, **{name: None}) == BAD, name
    for name in ("k", "v"):
        assert store(load, **{name: mk(F, 64, 2, 4, 3)}) == BAD           # positions differ
        assert store(load, **{name: mk(F, 0, 2, 5, 3)}) == BAD
    for k in (mk(F, 32, 2, 5, 3), mk(F, 64, 4, 5, 3), mk(F, 64, 2, 5, 2)):
        assert store(load, k=k, v=k) == BAD                              # not the cache's head_dim, heads, sequences
    assert store(load, k=mk(S.TYPE_F16, 64, 2, 5, 3)) == NOT_HERE
    for name in ("slot", "count"):
        assert store(load, **{name: mk(I, 2)}) == BAD
        assert store(load, **{name: mk(I, 3, 2)}) == BAD
        assert store(load, **{name: mk(F, 3)}) == BAD
        assert store(load, **{name: mk(I, 3, at=(1 << 43) + 2)}) == NOT_HERE
    for name in ("kc", "vc"):
        assert store(load, **{name: mk(Q4, 64, 2, 8, 3)}) == BAD          # capacities differ
        assert store(load, **{name: mk(Q8, 64, 2, 9, 3)}) == NOT_HERE     # types differ
        assert store(load, **{name: mk(Q4, 64, 2, 9, 3, at=(1 << 43) + 1)}) == NOT_HERE
        odd = mk(Q4, 64, 2, 9, 3)
        odd.nb[1] = 37
        assert store(load, **{name: odd}) == NOT_HERE
        wide = mk(Q4, 64, 2, 9, 3)
        wide.nb[0] = 20
        assert store(load, **{name: wide}) == BAD
    for bad in (mk(S.TYPE_Q5_K, 256, 2, 9, 3), mk(I, 64, 2, 9, 3), mk(Q4, 48, 2, 9, 3)):
        assert store(load, kc=bad, vc=bad) == BAD
    big = mk(S.TYPE_F16, 257, 2, 9, 3)
    assert store(load, kc=big, vc=big, k=mk(F, 257, 2, 5, 3), v=mk(F, 257, 2, 5, 3)) == NOT_HERE
    misaligned = mk(F, 64, 2, 5, 3, at=(1 << 43) + 2)
    assert store(load, k=misaligned) == NOT_HERE


def test_a_call_that_would_be_too_long_is_refused():
    n = 1 << 27
    k = mk(F, 64, 2, n, 1)
    c = mk(Q4, 64, 2, n, 1)
    assert store(k=k, v=mk(F, 64, 2, n, 1), slot=mk(I, 1), count=None, kc=c, vc=mk(Q4, 64, 2, n, 1)) == NOT_HERE
    far = mk(F, 64, 2, 5, 3, nb=[4, 256, 1 << 62, 1 << 63])
    assert store(k=far) == NOT_HERE


@pytest.mark.parametrize("load", [False, True])
def test_written_tensors_overlap_nothing(load):
    k, kc = mk(F, 64, 2, 5, 3), mk(Q4, 64, 2, 9, 3)
    assert store(load, **({"k": k, "v": k} if load else {"kc": kc, "vc": kc})) == NOT_HERE
    shifted = mk(Q4, 64, 2, 9, 3, at=kc.data + 36 * 2 * 8) if not load else mk(F, 64, 2, 5, 3, at=k.data + 512)
    assert store(load, **({"k": k, "v": shifted} if load else {"kc": kc, "vc": shifted})) == NOT_HERE
    for d in (1, 2, 3):                                                   # rows on top of each other
        t = mk(F, 64, 2, 5, 3) if load else mk(Q4, 64, 2, 9, 3)
        t.nb[d] = 0
        assert store(load, **{"k" if load else "kc": t}) == NOT_HERE, d
    slot = mk(I, 3, at=(k if load else kc).data + 4)
    assert store(load, k=k, kc=kc, slot=slot) == NOT_HERE
    if not load:
        assert store(k=k, status=mk(I, 1, at=k.data)) == NOT_HERE
        assert store(status=mk(I, 2)) == BAD and store(status=mk(F, 1)) == BAD


def attend(**over):
    a = dict(q=mk(F, 64, 8, 1, 3), kc=mk(Q4, 64, 2, 900, 3), vc=mk(Q4, 64, 2, 900, 3), length=mk(I, 3), count=mk(I, 3),
             scale=0.125, window=0, sinks=0, work=mk(F, 1 << 22), y=mk(F, 64, 8, 1, 3))
    a.update(over)
    return S.load().shp_attn_kv(R(a["q"]), R(a["kc"]), R(a["vc"]), R(a["length"]), R(a["count"]), a["scale"], a["window"],
                                a["sinks"], R(a["work"]), R(a["y"]), None)


def floats(q, kc, window=0, sinks=0):
    n = ctypes.c_int64(-7)
    st = S.load().shp_attn_kv_work(R(q), R(kc), window, sinks, ctypes.byref(n))
    return n.value if st == S.OK else -st


def test_attention_refuses():
    for name in ("q", "kc", "vc", "y"):
        assert attend(**{name: None}) == BAD, name
    assert attend(q=mk(F, 64, 7, 1, 3), y=mk(F, 64, 7, 1, 3)) == BAD      # heads no multiple of kv heads
    assert attend(q=mk(F, 96, 8, 1, 3), y=mk(F, 96, 8, 1, 3)) == BAD
    assert attend(q=mk(F, 64, 8, 1, 2), y=mk(F, 64, 8, 1, 2)) == BAD
    assert attend(y=mk(F, 64, 8, 2, 3)) == BAD
    assert attend(y=mk(S.TYPE_F16, 64, 8, 1, 3)) == NOT_HERE
    assert attend(q=mk(S.TYPE_BF16, 64, 8, 1, 3)) == NOT_HERE
    assert attend(window=-1) == BAD and attend(sinks=-1) == BAD
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert attend(scale=scale) == BAD
    for name in ("length", "count"):
        assert attend(**{name: mk(I, 2)}) == BAD
        assert attend(**{name: mk(F, 3)}) == BAD
        assert attend(**{name: mk(I, 3, at=(1 << 43) + 2)}) == NOT_HERE
    assert attend(vc=mk(Q8, 64, 2, 900, 3)) == NOT_HERE
    assert attend(vc=mk(Q4, 64, 2, 899, 3)) == BAD
    assert attend(q=mk(F, 64, 8, 1, 3, at=(1 << 43) + 2)) == NOT_HERE
    y = mk(F, 64, 8, 1, 3)
    assert attend(q=y, y=y) == NOT_HERE and attend(work=mk(F, 1 << 22, at=y.data), y=y) == NOT_HERE
    q = mk(F, 64, 8, 1, 3)
    assert attend(work=mk(F, 1 << 22, at=q.data), q=q) == NOT_HERE
    flat = mk(F, 64, 8, 1, 3)
    flat.nb[1] = 0
    assert attend(y=flat) == NOT_HERE
    rows = 1 << 27
    long_q = mk(F, 64, 8, rows, 1)
    one = mk(Q4, 64, 2, 900, 1)
    assert attend(q=long_q, y=mk(F, 64, 8, rows, 1), kc=one, vc=one, length=None, count=None) == NOT_HERE
    deep = mk(Q4, 64, 2, (1 << 30) + 1, 1)
    assert attend(q=mk(F, 64, 8, 1, 1), y=mk(F, 64, 8, 1, 1), kc=deep, vc=deep, length=None, count=None) == NOT_HERE


def test_workspace_is_checked_against_the_size_asked_for():
    q, kc = mk(F, 64, 8, 1, 3), mk(Q4, 64, 2, 900, 3)
    need = floats(q, kc)
    assert need > 0
    assert attend(work=None) == BAD
    assert attend(work=mk(F, need - 1)) == BAD
    assert attend(work=mk(S.TYPE_F16, need)) == BAD
    strided = mk(F, need, 2)
    strided.nb[1] += 4
    assert attend(work=strided) == BAD
    assert attend(work=mk(F, need, at=(1 << 43) + 4)) == NOT_HERE


def test_workspace_size():
    kc = mk(Q4, 64, 2, 900, 3)
    assert floats(mk(F, 64, 8, 1, 3), mk(Q4, 64, 2, 30, 3)) == 0           # too few rows to split
    assert floats(mk(F, 64, 8, 4000, 3), mk(Q4, 64, 2, 9000, 3)) == 0      # enough queries
    assert floats(mk(F, 64, 8, 1, 3), kc, window=10, sinks=2) == 0
    assert floats(mk(F, 64, 7, 1, 3), kc) == -BAD
    assert floats(mk(F, 64, 8, 1, 3), kc, window=-1) == -BAD
    assert floats(mk(S.TYPE_F16, 64, 8, 1, 3), kc) == -NOT_HERE
    assert S.load().shp_attn_kv_work(R(mk(F, 64, 8, 1, 3)), R(kc), 0, 0, None) == BAD


def test_binding_raises(monkeypatch):
    monkeypatch.setattr(S, "_stream", lambda: 0)
    k = torch.zeros(1, 2, 2, 64)
    c = S.Q4Tensor(torch.zeros(1, 9, 2, 36, dtype=torch.uint8), 64)
    other = S.Q8Tensor(torch.zeros(1, 9, 2, 68, dtype=torch.uint8), 64)
    slot = torch.zeros(1, dtype=torch.int32)
    for call, status in ((lambda: S.kv_store(k, k, c, other, slot), NOT_HERE),
                         (lambda: S.kv_store(k, k, c, c, slot), NOT_HERE),
                         (lambda: S.kv_load(c, other, slot, 2), NOT_HERE),
                         (lambda: S.attn_kv_work(k.half(), c), NOT_HERE),
                         (lambda: S.attn_kv(k[:, :, :1], c, c), BAD),
                         (lambda: S.attn_kv(k, c, c, window=-1), BAD)):
        with pytest.raises(S.ShpError) as e:
            call()
        assert e.value.status == status
    with pytest.raises(AssertionError):
        S.Q4Tensor(torch.zeros(9, 35, dtype=torch.uint8), 64)


def test_a_scale_past_what_f32_holds_in_powers_of_two():
    """scale log2(e) has to be finite: the kernels' exponentials are of two."""
    for scale in (3e38, -2.5e38):
        assert attend(scale=scale) == BAD
    assert attend(scale=2e38, work=None) == BAD                           # (the workspace; nothing is run)
