"""Host side of the paged K/V cache: the page pool's bookkeeping against a
plain model of it, the axis map, and the refusals (checked before anything
reaches a GPU)."""
import ctypes

import numpy as np
import pytest

b2 = pytest.importorskip("b2gguf")


def pages_of(pool, seq):
    t = pool.table([seq])[0]
    n = -(-pool.length(seq) // pool.page_size)
    assert np.all(t[:n] >= 0) and np.all(t[n:] == -1)
    return t[:n].tolist()


def test_extend_fork_and_copy_on_write():
    p = b2.PagePool(8, 16, 3, 6)
    assert p.extend(0, 40) == (0, None)
    assert pages_of(p, 0) == [0, 1, 2] and p.free_pages() == 5
    p.fork(0, 1)
    assert pages_of(p, 1) == [0, 1, 2] and p.free_pages() == 5
    rc, copy = p.extend(1, 1)                      # writes into the shared, partly filled page
    assert rc == 0 and copy == (2, 3) and pages_of(p, 1) == [0, 1, 3]
    assert p.extend(0, 1) == (0, None)             # no longer shared
    p.fork(0, 2, 32)                               # a page boundary: nothing to copy
    assert p.extend(2, 5) == (0, None) and pages_of(p, 2) == [0, 1, 4]
    p.truncate(0)
    assert pages_of(p, 0) == [] and p.free_pages() == 8 - 4
    p.truncate(1)
    p.truncate(2)
    assert p.free_pages() == 8


def test_extend_refuses_without_change():
    p = b2.PagePool(3, 16, 2, 2)
    assert p.extend(0, 33)[0] == b2.NO_KV_SLOT     # past max_pages
    assert p.length(0) == 0 and p.free_pages() == 3
    assert p.extend(0, 32)[0] == 0
    assert p.extend(1, 17)[0] == b2.NO_KV_SLOT     # one page left
    assert p.extend(1, 16)[0] == 0 and p.free_pages() == 0
    p.truncate(1)
    p.fork(0, 1, 20)
    assert p.extend(1, 1) == (0, (1, 2))
    p.truncate(1, 17)
    assert p.extend(1, 16)[0] == b2.NO_KV_SLOT
    assert p.length(1) == 17


def test_keep_holds_old_pages_until_settled():
    p = b2.PagePool(10, 4, 2, 8)
    p.extend(0, 22)                                # pages 0..5
    rc, old = p.keep(0, [0, 1, 2, 3, 4, 10, 11, 20])
    assert rc == 0 and old.tolist() == [0, 1, 2, 3, 4, 5, -1, -1]
    assert pages_of(p, 0) == [0, 6] and p.length(0) == 8
    assert p.free_pages() == 3                     # 1..5 are held
    with pytest.raises(b2.B2Error):
        p.defrag()
    p.settle()
    assert p.free_pages() == 8
    rc, old = p.keep(0, np.arange(6))              # a plain truncation takes no page
    assert rc == 0 and pages_of(p, 0) == [0, 6]
    rc, old = p.keep(0, [])
    p.settle()
    assert p.length(0) == 0 and p.free_pages() == 10


def test_keep_leaves_shared_pages_to_their_other_holders():
    p = b2.PagePool(8, 4, 2, 6)
    p.extend(0, 12)
    p.fork(0, 1)
    p.keep(0, [0, 5, 6])
    p.settle()
    assert pages_of(p, 1) == [0, 1, 2] and pages_of(p, 0) == [3] and p.free_pages() == 4


def test_defrag_moves_used_pages_to_the_front():
    p = b2.PagePool(12, 4, 4, 6)
    for s in range(3):
        p.extend(s, 12)
    p.fork(2, 3, 8)
    p.truncate(0)
    p.truncate(1, 4)
    before = {s: pages_of(p, s) for s in (1, 2, 3)}
    src, dst = p.defrag()
    assert set(src) & set(dst) == set()
    move = dict(zip(src.tolist(), dst.tolist()))
    for s in (1, 2, 3):
        assert pages_of(p, s) == [move.get(x, x) for x in before[s]]
    used = {x for s in (1, 2, 3) for x in pages_of(p, s)}
    assert used == set(range(len(used))) and p.free_pages() == 12 - len(used)
    assert p.extend(0, 1)[0] == 0 and pages_of(p, 0) == [len(used)]


def test_random_walk_against_a_model():
    r = np.random.default_rng(0)
    n_pages, ps, n_seq = 40, 4, 6
    p = b2.PagePool(n_pages, ps, n_seq, 12)
    data = {i: {} for i in range(n_pages)}         # page -> slot -> token, as the device would hold it
    want = {s: [] for s in range(n_seq)}
    fresh = iter(range(10 ** 9))

    def copy(a, b):
        data[b] = dict(data[a])

    for _ in range(3000):
        s = int(r.integers(n_seq))
        op = r.integers(6)
        if op <= 1:
            n = int(r.integers(1, 9))
            rc, c = p.extend(s, n)
            if rc:
                continue
            if c:
                copy(*c)
            t = p.table([s])[0]
            for _ in range(n):
                pos = len(want[s])
                want[s].append(next(fresh))
                data[t[pos // ps]][pos % ps] = want[s][-1]
        elif op == 2:
            d = int(r.integers(n_seq))
            if d != s and not want[d]:
                n = int(r.integers(0, len(want[s]) + 1))
                p.fork(s, d, n)
                want[d] = want[s][:n]
        elif op == 3:
            n = int(r.integers(0, len(want[s]) + 1))
            p.truncate(s, n)
            want[s] = want[s][:n]
        elif op == 4:
            k = [i for i in range(len(want[s])) if r.random() < 0.7]
            rc, old = p.keep(s, k)
            if rc:
                continue
            t = p.table([s])[0]
            rows = [data[old[i // ps]][i % ps] for i in k]
            for i, v in enumerate(rows):
                data[t[i // ps]][i % ps] = v
            p.settle()
            want[s] = [want[s][i] for i in k]
        else:
            for a, b in zip(*p.defrag()):
                copy(int(a), int(b))
        for q in range(n_seq):
            t = p.table([q])[0]
            assert p.length(q) == len(want[q])
            assert [data[t[i // ps]][i % ps] for i in range(len(want[q]))] == want[q]
    held = {x for q in range(n_seq) for x in pages_of(p, q)}
    assert p.free_pages() == n_pages - len(held)


def test_pool_refusals():
    with pytest.raises(b2.B2Error):
        b2.PagePool(4, 12, 1, 1)
    with pytest.raises(b2.B2Error):
        b2.PagePool(0, 16, 1, 1)
    p = b2.PagePool(4, 16, 2, 4)
    p.extend(0, 10)
    for call in (lambda: p.extend(2, 1), lambda: p.extend(-1, 1), lambda: p.extend(0, -1), lambda: p.fork(0, 0),
                 lambda: p.fork(0, 1, 11), lambda: p.truncate(0, 11), lambda: p.truncate(0, -1),
                 lambda: p.keep(0, [3, 3]), lambda: p.keep(0, [10]), lambda: p.keep(0, [-1, 2]),
                 lambda: p.fork(1, 0, 0)):
        with pytest.raises(b2.B2Error):
            call()
    assert p.length(0) == 10 and p.free_pages() == 3


def test_rope_sections():
    assert b2.rope_sections([16, 24, 24]).tolist() == [0] * 16 + [1] * 24 + [2] * 24
    assert b2.rope_sections([2, 3, 1], True).tolist() == [0, 1, 2, 0, 1, 1]
    assert b2.rope_sections([0, 2]).tolist() == [1, 1]
    out = np.zeros(4, np.uint8)
    for sec, n in (([1, 2], 4), ([-1, 5], 4)):
        a = np.array(sec, np.int32)
        assert b2.lib.b2_rope_sections(a.ctypes.data, 2, n, 0, out.ctypes.data) == b2.ERR_INVALID
    assert b2.lib.b2_rope_sections(None, 2, 4, 0, out.ctypes.data) == b2.ERR_INVALID


def cache(**kw):
    a = dict(n_layer=2, n_pages=4, page_size=16, n_kv=2, head_dim=64, type_k=b2.F16, type_v=b2.F16, k=1 << 20, v=1 << 24)
    a.update(kw)
    return b2.PageCache(**a)


def batch(**kw):
    a = dict(q_start=1 << 12, kv_len=1 << 12, table=1 << 12, n_seq=2, max_pages=4, n_tok=2, max_q=1)
    a.update(kw)
    return b2.PageBatch(**a)


def test_cache_bytes():
    c = cache(type_k=b2.Q8_0, type_v=b2.Q4_0)
    assert c.bytes_k == 2 * 4 * 2 * 16 * 80 and c.bytes_v == 2 * 4 * 2 * 16 * 48


@pytest.mark.parametrize("bad", [dict(page_size=24), dict(page_size=4), dict(page_size=512), dict(head_dim=40), dict(head_dim=288),
                                 dict(type_k=b2.Q4_K), dict(n_pages=0), dict(n_layer=0), dict(n_kv=0)])
def test_cache_refusals(bad):
    with pytest.raises(b2.B2Error):
        cache(**bad)


def attn(c, b, n_head=4, q=1 << 12, out=1 << 12, t=b2.F32, layer=0, **kw):
    return b2.page_attn(c, layer, b, n_head, q, out, t, **kw)


@pytest.mark.parametrize("kw", [
    dict(b=dict(n_seq=0)), dict(b=dict(n_seq=1025)), dict(b=dict(max_q=3)), dict(b=dict(max_q=0)), dict(b=dict(n_tok=0)),
    dict(b=dict(max_pages=0)), dict(b=dict(max_pages=1 << 27)), dict(b=dict(table=None)), dict(c=dict(k=(1 << 20) + 8)),
    dict(c=dict(head_dim=160)), dict(a=dict(n_head=3)), dict(a=dict(t=b2.Q8_0)), dict(a=dict(layer=2)),
    dict(a=dict(layer=-1)), dict(a=dict(q=None)), dict(a=dict(out=4)), dict(a=dict(scale=float("nan"))),
    dict(a=dict(scale=float("inf")))])
def test_attn_refusals(kw):
    with pytest.raises(b2.B2Error) as e:
        attn(cache(**kw.get("c", {})), batch(**kw.get("b", {})), **kw.get("a", {}))
    assert e.value.rc in (b2.ERR_INVALID, b2.ERR_UNSUPPORTED)


@pytest.mark.parametrize("kw", [dict(rot=12), dict(rot=72), dict(rot=0), dict(style=2), dict(axes=0), dict(axes=9),
                                dict(axes=3, axis=None), dict(tx=b2.Q8_0), dict(tq=b2.Q8_0), dict(n_pos=0),
                                dict(qkv=None), dict(qkv=20), dict(layer=5)])
def test_store_refusals(kw):
    a = dict(layer=0, qkv=1 << 12, tx=b2.F32, tq=b2.F32, axes=1, axis=1 << 12, n_pos=10, rot=64, style=0)
    a.update(kw)
    with pytest.raises(b2.B2Error):
        b2.page_rope_store(cache(), a["layer"], batch(), 4, a["qkv"], a["tx"], 1 << 12, a["tq"], 1 << 12, a["axes"],
                           a["axis"], 1 << 12, a["n_pos"], a["rot"], a["style"])


@pytest.mark.parametrize("src,dst", [([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([1], [1])])
def test_copy_refusals(src, dst):
    with pytest.raises(b2.B2Error):
        b2.page_copy(cache(), src, dst)


def test_gather_refusals():
    c = cache()
    for a in ((0, 1, 1, 1, 1, 1, 4), (1, None, 1, 1, 1, 1, 4), (1, 1, None, 1, 1, 1, 4), (1, 1, 1, 1, 1, 1, 0),
              (1, 1, 1, -1, 1, 1, 4)):
        with pytest.raises(b2.B2Error):
            b2.page_gather(c, *a)
    b2.page_gather(c, 1, 16, 16, 0, 16, 16, 4)     # nothing to keep: nothing is launched
    b2.page_copy(c, [], [])
