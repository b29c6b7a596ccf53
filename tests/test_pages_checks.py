"""What the paged KV cache's entry points refuse, and their workspaces: host code,
no GPU. Every refused call names addresses that nothing reads."""
import ctypes

import pytest
import torch

import synth_hip as S

UNIT = {S.TYPE_F32: 4, S.TYPE_F16: 2, S.TYPE_BF16: 2, S.TYPE_I32: 4, S.TYPE_I8: 1}
BAD, NOT_HERE = S.ERR_INVALID_ARG, S.ERR_UNSUPPORTED
F, I, C = S.TYPE_F32, S.TYPE_I32, S.TYPE_I8
_at = [1 << 44]


def mk(type_, *ne, nb=None, at=None):
    t = S.ShpTensor()
    ne = list(ne) + [1] * (4 - len(ne))
    if nb is None:
        nb = [UNIT[type_], ne[0] * UNIT[type_]]
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


def step(**over):
    a = dict(length=mk(I, 3), page=16, held=mk(I, 3), free=mk(I, 40), left=mk(I, 1), table=mk(I, 9, 3), work=None, status=mk(I, 1))
    a.update(over)
    return S.load().shp_kv_pages(R(a["length"]), a["page"], R(a["held"]), R(a["free"]), R(a["left"]), R(a["table"]), R(a["work"]),
                                 R(a["status"]), None)


def step_ints(table):
    n = ctypes.c_int64(-7)
    st = S.load().shp_kv_pages_work(R(table), ctypes.byref(n))
    return n.value if st == S.OK else -st


def test_tables_refuse():
    for name in ("length", "held", "free", "left", "table"):
        assert step(**{name: None}) == BAD, name
        assert step(**{name: mk(F, *([9, 3] if name == "table" else [3]))}) == BAD, name
    for name in ("length", "held", "left", "status"):
        assert step(**{name: mk(I, 2)}) == BAD, name
        assert step(**{name: mk(I, 1 if name in ("left", "status") else 3, at=(1 << 43) + 2)}) == NOT_HERE, name
    assert step(table=mk(I, 9, 2)) == BAD and step(table=mk(I, 9, 3, 2)) == BAD and step(free=mk(I, 4, 10)) == BAD
    for page in (0, -16, 8, 17, 24, 512):
        assert step(page=page) == NOT_HERE, page
    assert step(table=mk(I, (1 << 26) + 1, 3), work=mk(I, 100)) == NOT_HERE                # rows past 2^30
    assert step(free=mk(I, 1 << 27)) == NOT_HERE                                           # slots past 2^31
    n = 65536
    assert step(length=mk(I, n), held=mk(I, n), table=mk(I, 9, n), work=mk(I, 1 << 20)) == NOT_HERE
    for a in ("held", "free", "left", "table", "status"):
        for b in ("length", "held", "free", "left", "table", "status"):
            if a != b:
                shapes = dict(length=(3,), held=(3,), free=(40,), left=(1,), table=(9, 3), status=(1,))
                first = mk(I, *shapes[a])
                assert step(**{a: first, b: mk(I, *shapes[b], at=first.data)}) == NOT_HERE, (a, b)
    flat = mk(I, 9, 3, nb=[4, 32, 108, 108])
    assert step(table=flat) == NOT_HERE                                                    # rows on top of each other


def test_workspace_of_tables():
    assert step_ints(mk(I, 9, 3)) == 0 and step_ints(mk(I, 1 << 16, 1)) == 0 and step_ints(mk(I, 16, 4096)) == 0
    big = mk(I, 1 << 16, 2)
    need = step_ints(big)
    assert need > 0 and step_ints(mk(I, 1, 4097)) > 0
    two = dict(length=mk(I, 2), held=mk(I, 2), table=big)
    assert step(**two) == BAD and step(**two, work=mk(I, need - 1)) == BAD and step(**two, work=mk(F, need)) == BAD
    assert step(**two, work=mk(I, need, at=(1 << 43) + 2)) == NOT_HERE
    assert step(**two, work=mk(I, need, at=big.data + 64)) == NOT_HERE
    assert step_ints(None) == -BAD and step_ints(mk(F, 9, 3)) == -BAD
    assert S.load().shp_kv_pages_work(R(big), None) == BAD


def slots(**over):
    a = dict(table=mk(I, 9, 3), length=mk(I, 3), count=mk(I, 3), page=16, slots=mk(I, 5, 3))
    a.update(over)
    return S.load().shp_kv_slots(R(a["table"]), R(a["length"]), R(a["count"]), a["page"], R(a["slots"]), None)


def test_slots_refuse():
    for name in ("table", "length", "slots"):
        assert slots(**{name: None}) == BAD, name
    for name, shape in (("table", (9, 2)), ("length", (2,)), ("count", (2,)), ("slots", (5, 2)), ("slots", (5, 3, 2))):
        assert slots(**{name: mk(I, *shape)}) == BAD, name
    for name, shape in (("table", (9, 3)), ("length", (3,)), ("count", (3,)), ("slots", (5, 3))):
        assert slots(**{name: mk(F, *shape)}) == BAD, name
        assert slots(**{name: mk(I, *shape, at=(1 << 43) + 2)}) == NOT_HERE, name
    assert slots(page=48) == NOT_HERE
    out = mk(I, 5, 3)
    for name, shape in (("table", (9, 3)), ("length", (3,)), ("count", (3,))):
        assert slots(**{name: mk(I, *shape, at=out.data + 4)}, slots=out) == NOT_HERE, name


def rows(load=False, **over):
    a = dict(k=mk(F, 64, 2, 5, 3), v=mk(F, 64, 2, 5, 3), table=mk(I, 9, 3), length=mk(I, 3), count=mk(I, 3), kp=mk(C, 64, 32, 2, 7),
             vp=mk(C, 32, 64, 2, 7), ks=mk(F, 2, 7), vs=mk(F, 2, 7), status=mk(I, 1), slots=mk(I, 5, 3))
    a.update(over)
    L = S.load()
    if load:
        return L.shp_kv_load_pages(R(a["kp"]), R(a["vp"]), R(a["ks"]), R(a["vs"]), R(a["slots"]), R(a["k"]), R(a["v"]), None)
    return L.shp_kv_store_pages(R(a["k"]), R(a["v"]), R(a["table"]), R(a["length"]), R(a["count"]), R(a["kp"]), R(a["vp"]),
                                R(a["ks"]), R(a["vs"]), R(a["status"]), None)


# (made anew for each test: the module of the binding may have been loaded again meanwhile)
def pools():
    return (dict(kp=mk(C, 64, 32, 2, 7), vp=mk(C, 64, 32, 2, 7)),                               # V not turned
            dict(kp=mk(C, 64, 32, 2, 6)), dict(vp=mk(C, 32, 64, 3, 7)), dict(ks=mk(F, 3, 7)), dict(vs=mk(F, 2, 6)),
            dict(ks=mk(F, 2, 7, 2)), dict(kp=mk(F, 64, 32, 2, 7)), dict(kp=mk(C, 64, 32, 2, 7, nb=[2, 128, 4096, 8192])))


def far():
    return (dict(kp=mk(C, 64, 32, 2, 7, at=(1 << 43) + 8)), dict(vp=mk(C, 32, 64, 2, 7, nb=[1, 48, 4096, 8192])),
            dict(kp=mk(C, 64, 32, 2, 7, nb=[1, 64, 2056, 8192])), dict(vp=mk(C, 32, 64, 2, 7, nb=[1, 32, 2048, 4104])),
            dict(ks=mk(F, 2, 7, at=(1 << 43) + 2)), dict(vs=mk(S.TYPE_F16, 2, 7)),
            dict(kp=mk(C, 64, 48, 2, 7), vp=mk(C, 48, 64, 2, 7)), dict(kp=mk(C, 64, 8, 2, 7), vp=mk(C, 8, 64, 2, 7)),
            dict(kp=mk(C, 64, 512, 2, 7), vp=mk(C, 512, 64, 2, 7)), dict(kp=mk(C, 272, 32, 2, 7), vp=mk(C, 32, 272, 2, 7)),
            dict(kp=mk(C, 72, 32, 2, 7), vp=mk(C, 32, 72, 2, 7)),
            dict(kp=mk(C, 64, 32, 2, 1 << 26), vp=mk(C, 32, 64, 2, 1 << 26), ks=mk(F, 2, 1 << 26), vs=mk(F, 2, 1 << 26)))


@pytest.mark.parametrize("load", [False, True])
def test_store_and_load_refuse(load):
    for name in ("k", "v", "kp", "vp", "ks", "vs") + (("slots",) if load else ("table", "length")):
        assert rows(load, **{name: None}) == BAD, name
    for over in pools():
        assert rows(load, **over) == BAD, over
    for over in far():
        assert rows(load, **over) == NOT_HERE, over
    for name in ("k", "v"):
        assert rows(load, **{name: mk(F, 64, 2, 4, 3)}) == BAD
        assert rows(load, **{name: mk(F, 64, 2, 0, 3)}) == BAD
        assert rows(load, **{name: mk(F, 64, 2, 5, 3, at=(1 << 43) + 2)}) == NOT_HERE
        assert rows(load, **{name: mk(S.TYPE_BF16, 64, 2, 5, 3)}) == NOT_HERE
    for shape in ((48, 2, 5, 3), (64, 1, 5, 3), (64, 2, 5, 2)):
        assert rows(load, k=mk(F, *shape), v=mk(F, *shape)) == BAD
    if load:
        assert rows(True, slots=mk(I, 4, 3)) == BAD and rows(True, slots=mk(I, 5, 2)) == BAD and rows(True, slots=mk(F, 5, 3)) == BAD
        assert rows(True, slots=mk(I, 5, 3, at=(1 << 43) + 2)) == NOT_HERE
        return
    for name, shape in (("table", (9, 2)), ("length", (2,)), ("count", (2,)), ("status", (2,))):
        assert rows(**{name: mk(I, *shape)}) == BAD, name
    for name, shape in (("table", (9, 3)), ("length", (3,)), ("count", (3,)), ("status", (1,))):
        assert rows(**{name: mk(F, *shape)}) == BAD, name
        assert rows(**{name: mk(I, *shape, at=(1 << 43) + 2)}) == NOT_HERE, name
    long = dict(k=mk(F, 64, 2, 1 << 27, 1), v=mk(F, 64, 2, 1 << 27, 1), table=mk(I, 9), length=mk(I, 1), count=None)
    assert rows(**long) == NOT_HERE


@pytest.mark.parametrize("load", [False, True])
def test_written_tensors_overlap_nothing(load):
    shapes = dict(k=(F, 64, 2, 5, 3), v=(F, 64, 2, 5, 3), kp=(C, 64, 32, 2, 7), vp=(C, 32, 64, 2, 7), ks=(F, 2, 7), vs=(F, 2, 7),
                  table=(I, 9, 3), length=(I, 3), count=(I, 3), status=(I, 1), slots=(I, 5, 3))
    written = ("k", "v") if load else ("kp", "vp", "ks", "vs", "status")
    others = ("kp", "vp", "ks", "vs", "slots", "k", "v") if load else tuple(n for n in shapes if n != "slots")
    for a in written:
        for b in others:
            if a != b:
                first = mk(*shapes[a])
                assert rows(load, **{a: first, b: mk(*shapes[b], at=first.data)}) == NOT_HERE, (a, b)
    if not load:
        assert rows(kp=mk(C, 64, 32, 2, 7, nb=[1, 64, 0, 4096])) == NOT_HERE                # heads, pages on top of each other
        assert rows(kp=mk(C, 64, 32, 2, 7, nb=[1, 64, 2048, 2048])) == NOT_HERE
        assert rows(ks=mk(F, 2, 7, nb=[4, 4, 56, 56])) == NOT_HERE


def test_binding_raises(monkeypatch):
    monkeypatch.setattr(S, "_stream", lambda: 0)
    k = torch.zeros(1, 2, 2, 64)
    cache = S.PagedCache.empty(3, 32, 2, 64, device="cpu")
    assert cache.page == 32
    assert S.desc(cache.k).type == S.TYPE_I8 and list(S.desc(cache.v).ne) == [32, 64, 2, 3]
    turned = S.PagedCache(cache.k, cache.k, cache.k_scale, cache.v_scale)
    table, one = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call, status in ((lambda: S.kv_store_pages(k, k, turned, table, one), BAD),
                         (lambda: S.kv_store_pages(k.half(), k.half(), cache, table, one), NOT_HERE),
                         (lambda: S.kv_load_pages(cache, table.float()), BAD),
                         (lambda: S.kv_slots(table, one, 17, 4), NOT_HERE),
                         (lambda: S.kv_pages_work(k), BAD),
                         (lambda: S.kv_pages(one, 16, one, table[0], one, table), NOT_HERE)):
        with pytest.raises(S.ShpError) as e:
            call()
        assert e.value.status == status
    with pytest.raises(KeyError):
        S.desc(torch.zeros(3, dtype=torch.uint8))


def attend(**over):
    a = dict(q=mk(F, 64, 8, 1, 3), kp=mk(C, 64, 32, 2, 7), vp=mk(C, 32, 64, 2, 7), ks=mk(F, 2, 7), vs=mk(F, 2, 7), table=mk(I, 90, 3),
             length=mk(I, 3), count=mk(I, 3), scale=0.125, window=0, sinks=0, work=mk(F, 1 << 22), y=mk(F, 64, 8, 1, 3))
    a.update(over)
    return S.load().shp_attn_pages(R(a["q"]), R(a["kp"]), R(a["vp"]), R(a["ks"]), R(a["vs"]), R(a["table"]), R(a["length"]),
                                   R(a["count"]), a["scale"], a["window"], a["sinks"], R(a["work"]), R(a["y"]), None)


def floats(q, kp, table, window=0, sinks=0):
    n = ctypes.c_int64(-7)
    st = S.load().shp_attn_pages_work(R(q), R(kp), R(table), window, sinks, ctypes.byref(n))
    return n.value if st == S.OK else -st


def test_attention_refuses():
    for name in ("q", "kp", "vp", "ks", "vs", "table", "length", "y"):
        assert attend(**{name: None}) == BAD, name
    for over in pools():
        assert attend(**over) == BAD, over
    for over in far():
        assert attend(**over) == NOT_HERE or over.get("kp", mk(C, 64, 32, 2, 7)).ne[0] != 64, over
    for hd in (72, 272):
        q = mk(F, hd, 8, 1, 3)
        assert attend(q=q, y=mk(F, hd, 8, 1, 3), kp=mk(C, hd, 32, 2, 7), vp=mk(C, 32, hd, 2, 7)) == NOT_HERE
    for shape in ((64, 7, 1, 3), (96, 8, 1, 3)):
        assert attend(q=mk(F, *shape), y=mk(F, *shape)) == BAD
    assert attend(q=mk(F, 64, 8, 1, 2), y=mk(F, 64, 8, 1, 2)) == BAD                        # tables of another number of sequences
    assert attend(y=mk(F, 64, 8, 2, 3)) == BAD and attend(y=mk(S.TYPE_F16, 64, 8, 1, 3)) == NOT_HERE
    assert attend(q=mk(S.TYPE_BF16, 64, 8, 1, 3)) == NOT_HERE and attend(q=mk(F, 64, 8, 1, 3, at=(1 << 43) + 2)) == NOT_HERE
    assert attend(window=-1) == BAD and attend(sinks=-1) == BAD
    for scale in (float("nan"), float("inf"), 3e38):
        assert attend(scale=scale) == BAD
    for name, shape in (("table", (90, 2)), ("table", (90, 3, 2)), ("length", (2,)), ("count", (2,))):
        assert attend(**{name: mk(I, *shape)}) == BAD, name
    for name, shape in (("table", (90, 3)), ("length", (3,)), ("count", (3,))):
        assert attend(**{name: mk(F, *shape)}) == BAD, name
        assert attend(**{name: mk(I, *shape, at=(1 << 43) + 2)}) == NOT_HERE, name
    assert attend(table=mk(I, (1 << 25) + 1, 3)) == NOT_HERE
    for name, shape in (("q", (F, 64, 8, 1, 3)), ("kp", (C, 64, 32, 2, 7)), ("vp", (C, 32, 64, 2, 7)), ("ks", (F, 2, 7)), ("vs", (F, 2, 7)),
                        ("table", (I, 90, 3)), ("length", (I, 3)), ("count", (I, 3))):
        first = mk(*shape)
        assert attend(**{name: first, "y": mk(F, 64, 8, 1, 3, at=first.data)}) == NOT_HERE, name
        assert attend(**{name: first, "work": mk(F, 1 << 22, at=first.data)}) == NOT_HERE, name
    y = mk(F, 64, 8, 1, 3)
    assert attend(work=mk(F, 1 << 22, at=y.data), y=y) == NOT_HERE
    flat = mk(F, 64, 8, 1, 3)
    flat.nb[1] = 0
    assert attend(y=flat) == NOT_HERE


def test_workspace_of_the_attention():
    q, kp, table = mk(F, 64, 8, 1, 3), mk(C, 64, 32, 2, 7), mk(I, 90, 3)
    need = floats(q, kp, table)
    assert need > 0
    assert attend(work=None) == BAD and attend(work=mk(F, need - 1)) == BAD and attend(work=mk(S.TYPE_F16, need)) == BAD
    assert attend(work=mk(F, need, at=(1 << 43) + 4)) == NOT_HERE
    assert floats(q, kp, mk(I, 2, 3)) == 0 and floats(q, kp, table, window=30, sinks=4) == 0
    assert floats(mk(F, 64, 8, 9000, 3), kp, mk(I, 290, 3)) == 0                            # enough queries
    assert floats(mk(F, 64, 7, 1, 3), kp, table) == -BAD and floats(q, kp, mk(I, 90, 2)) == -BAD
    assert floats(q, kp, table, window=-1) == -BAD and floats(mk(S.TYPE_F16, 64, 8, 1, 3), kp, table) == -NOT_HERE
    assert S.load().shp_attn_pages_work(R(q), R(kp), R(table), 0, 0, None) == BAD
