"""The paged K/V cache on the GPU, through the C ABI: rotary positions with
several axes and the store, attention of one or many new tokens per sequence,
page copies and gathers, each against a plain numpy form in 64 bits.

Tolerances.  Attention with B2_F32: a weight's exponent is a sum of head_dim
products, each good to 2^-22 of its size (queries carry 22 bits), and
ex2.approx and the split weights add 2^-22 each; with |q·k|·scale summing to
at most ~16 that is below 1e-5 of a weight, so 2e-5 of the largest |v| for the
quotient of the weighted sums.  With B2_F16 a weight is rounded once to fp16
and so is the output: 2^-11 each of at most the largest |v|, 2^-10 together,
beside the above.  Stores, copies and gathers are exact: bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

b2 = pytest.importorskip("b2gguf")

F32, F16, Q8, Q4 = b2.F32, b2.F16, b2.Q8_0, b2.Q4_0
NP = {F32: np.float32, F16: np.float16}


def dev(a):
    return b2.DeviceBuffer.from_array(np.ascontiguousarray(a))


# ---- the cache in numpy ------------------------------------------------------------------------
def rows_of(x, t):
    """Values [..., hd] -> stored rows (uint8 [..., row bytes])."""
    hd = x.shape[-1]
    if t == F16:
        return np.ascontiguousarray(x.astype(np.float16)).view(np.uint8)
    b = x.astype(np.float32).reshape(-1, hd // 32, 32)
    out = np.zeros((b.shape[0], b2.lib.b2_kv_row_bytes(t, hd)), np.uint8)
    if t == Q8:
        amax = np.abs(b).max(-1)
        inv = np.where(amax > 0, np.float32(127) / np.where(amax > 0, amax, 1), 0).astype(np.float32)
        s = b * inv[..., None]
        codes = np.trunc(s + np.where(s >= 0, np.float32(0.5), np.float32(-0.5))).clip(-127, 127).astype(np.int8)
        d, cb = amax * np.float32(1 / 127.0), hd
        out[:, :cb] = codes.reshape(-1, hd).view(np.uint8)
    else:
        d = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)[..., 0] / np.float32(-8)
        inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, 1), 0).astype(np.float32)
        n = np.minimum(np.trunc(b * inv[..., None] + np.float32(8.5)), 15).astype(np.uint8)
        cb = hd // 2
        out[:, :cb] = (n[..., :16] | (n[..., 16:] << 4)).reshape(-1, cb)
    out[:, cb:cb + hd // 16] = d.astype(np.float16).view(np.uint8).reshape(-1, hd // 16)
    return out.reshape(*x.shape[:-1], -1)


def values_of(rows, t, hd):
    if t == F16:
        return rows.view(np.float16).astype(np.float64)
    cb = hd if t == Q8 else hd // 2
    d = np.ascontiguousarray(rows[..., cb:cb + hd // 16]).view(np.float16).astype(np.float64)
    if t == Q8:
        c = np.ascontiguousarray(rows[..., :cb]).view(np.int8).astype(np.float64)
    else:
        n = rows[..., :cb].reshape(*rows.shape[:-1], hd // 32, 16)
        c = np.concatenate([n & 15, n >> 4], -1).reshape(*rows.shape[:-1], hd).astype(np.float64) - 8
    return (c.reshape(*c.shape[:-1], hd // 32, 32) * d[..., None]).reshape(c.shape)


class Setup:
    """A pool with the pages of ragged sequences in random order, some free
    pages, every slot past a sequence's end filled with NaN patterns."""

    def __init__(self, q_len, kv_len, n_head, n_kv, hd, page, kt=F16, vt=F16, qt=F32, seed=0, n_layer=1, layer=0,
                 poison=True, extra_pages=3):
        r = np.random.default_rng(seed)
        self.__dict__.update(q_len=q_len, kv_len=kv_len, n_head=n_head, n_kv=n_kv, hd=hd, page=page, kt=kt, vt=vt,
                             qt=qt, n_layer=n_layer, layer=layer)
        need = [-(-n // page) for n in kv_len]
        self.n_pages = sum(need) + extra_pages
        self.max_pages = max(1, max(need))
        order = r.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(kv_len), self.max_pages), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (n_layer, self.n_pages, n_kv, page, hd)
        self.K = rows_of(r.standard_normal(shape, dtype=np.float32), kt)
        self.V = rows_of(r.standard_normal(shape, dtype=np.float32), vt)
        if poison:
            live = np.zeros((self.n_pages, page), bool)
            for s, n in enumerate(kv_len):
                p = np.arange(n)
                live[self.table[s, p // page], p % page] = True
            for pool in (self.K, self.V):
                pool.transpose(0, 1, 3, 2, 4)[:, ~live] = 0x7E   # fp16 0x7E7E is a NaN, as value or as scale
        self.q_start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.n_tok = int(self.q_start[-1])
        self.Q = r.standard_normal((self.n_tok, n_head, hd), dtype=np.float32).astype(NP[qt])

    def cache(self):
        self.k, self.v = dev(self.K), dev(self.V)
        return b2.PageCache(self.n_layer, self.n_pages, self.page, self.n_kv, self.hd, self.kt, self.vt, k=self.k,
                            v=self.v)

    def batch(self):
        return b2.PageBatch(self.q_start, np.array(self.kv_len, np.int32), self.table, n_tok=self.n_tok)

    def seq_values(self, s, n):
        p = np.arange(n)
        pages = self.table[s, p // self.page]
        bad = (pages < 0) | (pages >= self.n_pages)
        pages = np.where(bad, 0, pages)
        k = values_of(self.K[self.layer, pages, :, p % self.page], self.kt, self.hd)
        v = values_of(self.V[self.layer, pages, :, p % self.page], self.vt, self.hd)
        k[bad] = 0
        v[bad] = 0
        return k, v      # [n][n_kv][hd]

    def run(self, window=0, scale=None, workspace=True, stream=None):
        c, b = self.cache(), self.batch()
        q, out = dev(self.Q), dev(np.full(self.Q.shape, 77, NP[self.qt]))
        ws = None
        if workspace:
            ws = b2.page_attn_workspace(c, b, self.n_head, self.qt)
        status = dev(np.zeros(1, np.int32))
        b2.synchronize()
        b2.page_attn(c, self.layer, b, self.n_head, q, out, self.qt, scale=scale, window=window, workspace=ws,
                     status=status, stream=stream)
        b2.synchronize()
        assert status.download(np.int32)[0] == 0
        return out.download(NP[self.qt]).reshape(self.Q.shape)

    def want(self, window=0, scale=None):
        """out, and the largest |v| a row sees, in 64 bits."""
        scale = self.hd ** -0.5 if scale is None else scale
        o = np.zeros(self.Q.shape, np.float64)
        vmax = np.zeros((self.n_tok, self.n_head, 1))
        G = self.n_head // self.n_kv
        for s in range(len(self.kv_len)):
            n = self.kv_len[s]
            k, v = self.seq_values(s, n)
            for i in range(self.q_len[s]):
                p, row = n - self.q_len[s] + i, self.q_start[s] + i
                lo = max(0, p - window + 1) if window else 0
                if p < 0:
                    continue
                for h in range(self.n_head):
                    kk, vv = k[lo:p + 1, h // G], v[lo:p + 1, h // G]
                    z = kk @ self.Q[row, h].astype(np.float64) * scale
                    w = np.exp(z - z.max())
                    o[row, h] = (w / w.sum()) @ vv
                    vmax[row, h] = np.abs(vv).max()
        return o, vmax

    def check(self, **kw):
        got = self.run(**kw).astype(np.float64)
        kw.pop("workspace", None)
        kw.pop("stream", None)
        want, vmax = self.want(**kw)
        tol = 2e-5 * vmax + (2.0 ** -10 * vmax if self.qt == F16 else 0) + 1e-30
        err = np.abs(got - want)
        assert np.all(np.isfinite(got))
        assert np.all(err <= tol), f"worst {np.max(err / tol):.3g} of the tolerance"
        return got


HEADS = [(32, 8, 128), (32, 4, 64), (6, 2, 96), (4, 2, 256), (16, 16, 64), (12, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("n_head,n_kv,hd", HEADS)
def test_attn_one_token_ragged(n_head, n_kv, hd, qt):
    """Decode: lengths 1, around a page, a unit of 64 and longer ones."""
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 300]
    Setup([1] * len(kv), kv, n_head, n_kv, hd, 16, qt=qt, seed=hd + n_head).check()


@pytest.mark.parametrize("kt,vt", [(Q8, Q8), (Q4, Q4), (F16, Q8), (Q8, F16), (Q4, Q8), (F16, Q4)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_quantized_caches(kt, vt, hd, qt):
    """Single tokens and a chunk over quantized pages."""
    Setup([1, 1, 21], [5, 130, 90], 8, 2, hd, 32, kt, vt, qt, seed=kt * 7 + vt + hd).check()


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("q_len,kv_len", [
    ([5], [5]), ([3, 1, 7], [3, 200, 64]), ([64], [64]), ([65], [129]), ([130, 1, 33], [130, 77, 300]),
    ([200], [513]), ([2, 2], [2, 66])])
def test_attn_chunks(q_len, kv_len, qt):
    Setup(q_len, kv_len, 8, 2, 128, 16, qt=qt, seed=sum(kv_len)).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("q_len", [1, 40])
def test_attn_page_sizes(page, q_len):
    Setup([q_len, q_len], [q_len + 70, q_len + 257], 4, 2, 64, page, qt=F16, seed=page).check()


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200])
@pytest.mark.parametrize("q_len", [1, 37])
def test_attn_window(window, q_len, qt):
    Setup([q_len, q_len, q_len], [q_len, 150, 400], 8, 2, 64, 16, qt=qt, seed=window).check(window=window)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("q_max", [1, 9, 120])
def test_attn_many_sequences_mixed(q_max, qt):
    """Many ragged sequences, some without new tokens or positions."""
    r = np.random.default_rng(q_max)
    q = [int(x) for x in r.integers(0, q_max + 1, 70)]
    kv = [n + int(x) for n, x in zip(q, r.integers(0, 150, 70))]
    q[3], kv[3], q[69], kv[69] = 0, 0, 0, 12
    q[0] = max(q[0], 1)
    kv[0] = max(kv[0], q[0])
    Setup(q, kv, 8, 4, 64, 16, qt=qt, seed=5).check()


@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_long_context_split(qt):
    """One sequence's positions over every SM, and a deep scale change along them."""
    s = Setup([1, 3], [9001, 4097], 8, 2, 128, 64, qt=qt, seed=9)
    s.check()
    s.check(scale=0.9)
    s.check(scale=-0.2)
    s.check(scale=0.0)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attn_scale_signs(hd, qt):
    s = Setup([1, 90], [200, 300], 8, 2, hd, 16, qt=qt, seed=6)
    for scale in (-0.3, 0.0, 1.0):
        s.check(scale=scale)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("q_len", [4, 70])
def test_attn_rows_without_positions(q_len, qt):
    """More new tokens than positions: the first ones see nothing and get zeros."""
    s = Setup([q_len, 1, q_len], [q_len - 3, 0, 0], 8, 2, 64, 16, qt=qt, seed=3)
    got = s.check()
    assert np.all(got[:3] == 0) and np.all(got[q_len:] == 0)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q8)])
@pytest.mark.parametrize("q_len,window", [(6, 0), (6, 3), (150, 0), (150, 20), (1, 5)])
def test_attn_nonfinite_values_stay_with_rows_that_see_them(q_len, window, kt, vt, hd, qt):
    """Infinite and NaN K and V at positions that only some rows see."""
    n = q_len + 100
    s = Setup([q_len], [n], 8, 2, hd, 16, kt, vt, qt, seed=1)
    bad = {n - 1: 0x7C00, n - 2: 0x7E00} if q_len > 1 else {}
    if window:
        bad[0] = 0x7E00
        bad[n - q_len - window] = 0xFC00      # just before the first row's window
    for p, bits in bad.items():
        page, slot = s.table[0, p // 16], p % 16
        for pool, t in ((s.K, kt), (s.V, vt)):
            at = 0 if t == F16 else hd          # a value, or the first block's scale
            pool[0, page, :, slot, at:at + 2] = np.frombuffer(np.uint16(bits).tobytes(), np.uint8)
    got = s.run(window=window).astype(np.float64)
    clean = Setup([q_len], [n], 8, 2, hd, 16, kt, vt, qt, seed=1)
    want, vmax = clean.want(window=window)
    rows = np.arange(n - q_len, n)              # positions of the rows
    sees = np.zeros(q_len, bool)
    for p in bad:
        sees |= (p <= rows) & ((rows - p < window) if window else True)
    assert (~sees).any()
    tol = 2e-5 * vmax + (2.0 ** -10 * vmax if qt == F16 else 0)
    assert np.all(np.abs(got - want)[~sees] <= tol[~sees])
    if sees.any():
        assert np.all(~np.isfinite(got[sees]).all(-1))


def test_attn_table_entries_outside_the_pool_read_as_zeros():
    s = Setup([1, 20], [100, 130], 8, 2, 128, 16, qt=F32, seed=2)
    s.table[0, 2], s.table[1, 0] = -5, s.n_pages + 7
    s.check()


def test_attn_malformed_lengths_stay_in_bounds():
    """Lengths past the table are clamped into it."""
    s = Setup([2, 1], [40, 33], 4, 2, 64, 16, seed=2)
    c = s.cache()
    b = b2.PageBatch(s.q_start, np.array([10 ** 9, -4], np.int32), s.table, n_tok=s.n_tok)
    out = dev(np.full(s.Q.shape, 77, np.float32))
    b2.page_attn(c, 0, b, 4, dev(s.Q), out, F32)
    b2.synchronize()
    got = out.download(np.float32).reshape(s.Q.shape)
    assert np.all(got[2] == 0)                 # no positions
    assert not np.any(got == 77)


def test_attn_layer_workspace_stream_and_graph():
    """Another layer of the pool; NULL and given workspace; another stream and
    a replayed capture that follows the lengths on the device: the same bits."""
    s = Setup([1, 1, 4], [500, 33, 90], 8, 2, 128, 16, qt=F16, seed=4, n_layer=3, layer=2)
    a = s.check()
    assert np.array_equal(a, s.run(workspace=False).astype(np.float64))
    st = b2.Stream()
    assert np.array_equal(a, s.run(stream=st.h).astype(np.float64))
    c, b = s.cache(), s.batch()
    q, out = dev(s.Q), dev(np.zeros(s.Q.shape, np.float16))
    ws = b2.page_attn_workspace(c, b, 8, F16)
    b2.page_attn(c, 2, b, 8, q, out, F16, workspace=ws, stream=st.h)
    st.synchronize()
    g = b2.Graph(st, lambda h: b2.page_attn(c, 2, b, 8, q, out, F16, workspace=ws, stream=h))
    s.kv_len = [480, 20, 70]
    b.kv_len.upload(np.array(s.kv_len, np.int32))
    g.launch()
    st.synchronize()
    want, vmax = s.want()
    got = out.download(np.float16).reshape(s.Q.shape).astype(np.float64)
    assert np.all(np.abs(got - want) <= (2e-5 + 2.0 ** -10) * vmax)


def test_attn_same_bits_every_time():
    s = Setup([1, 50, 1], [3000, 2000, 17], 8, 2, 128, 32, qt=F32, seed=8)
    a = s.run()
    for _ in range(3):
        assert np.array_equal(a, s.run())


# ---- rotary positions and the store --------------------------------------------------------------
def rotate(x, cs, style):
    """x [n][heads][hd] fp32, cs [n][rot/2][2] fp32 -> the same, every product and sum rounded to fp32."""
    rot = cs.shape[1] * 2
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if style else (x[..., 0:rot:2], x[..., 1:rot:2])
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    y0, y1 = a * c - b * n, a * n + b * c
    out = x.copy()
    if style:
        out[..., :rot // 2], out[..., rot // 2:rot] = y0, y1
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = y0, y1
    return out


@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q8), (Q4, Q4), (Q8, F16), (Q4, Q8)])
@pytest.mark.parametrize("n_head,n_kv,hd,rot", [(32, 8, 128, 128), (6, 2, 96, 48), (4, 4, 64, 32), (2, 1, 256, 256),
                                                (3, 3, 32, 8)])
@pytest.mark.parametrize("axes,style,interleave", [(1, 0, 0), (3, 1, 0), (3, 0, 1), (2, 1, 1)])
@pytest.mark.parametrize("tx,tq", [(F32, F32), (F16, F16)])
def test_store_bit_exact(kt, vt, n_head, n_kv, hd, rot, axes, style, interleave, tx, tq):
    q_len, kv_len, page, n_pos = [1, 0, 19, 3], [40, 7, 19, 33], 16, 500
    s = Setup(q_len, kv_len, n_head, n_kv, hd, page, kt, vt, tq, seed=rot, n_layer=2, layer=1, poison=False)
    r = np.random.default_rng(1)
    x = r.standard_normal((s.n_tok, n_head + 2 * n_kv, hd), dtype=np.float32).astype(NP[tx])
    x[0, n_head + n_kv] = 0                    # an all-zero block
    pos = r.integers(0, n_pos, (axes, s.n_tok)).astype(np.int32)
    half = rot // 2
    sec = [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    axis = b2.rope_sections(sec, bool(interleave))
    assert [int((axis == a).sum()) for a in range(axes)] == sec
    table = b2.rope_table(10000.0, rot, 0, n_pos)
    cs = table.reshape(n_pos, half, 2)[pos[axis].T, np.arange(half)]
    c, q = s.cache(), dev(np.full((s.n_tok, n_head, hd), 77, NP[tq]))
    b2.page_rope_store(c, 1, s.batch(), n_head, dev(x), tx, q, tq, dev(pos), axes, dev(axis), dev(table), n_pos, rot,
                       style)
    b2.synchronize()
    x32 = x.astype(np.float32)
    y = rotate(x32[:, :n_head + n_kv], cs, style)
    assert np.array_equal(q.download(NP[tq]).reshape(s.n_tok, n_head, hd).view(np.uint8),
                          np.ascontiguousarray(y[:, :n_head].astype(NP[tq])).view(np.uint8))
    K, V = s.K.copy(), s.V.copy()
    for b in range(len(kv_len)):
        for i in range(q_len[b]):
            p, row = kv_len[b] - q_len[b] + i, s.q_start[b] + i
            for pool, t, val in ((K, kt, y[row, n_head:]), (V, vt, x32[row, n_head + n_kv:])):
                new = rows_of(val, t)
                n = 2 * hd if t == F16 else (hd if t == Q8 else hd // 2) + hd // 16     # padding is left alone
                pool[1, s.table[b, p // page], :, p % page, :n] = new[:, :n]
    assert np.array_equal(s.k.download(np.uint8).reshape(K.shape), K)
    assert np.array_equal(s.v.download(np.uint8).reshape(V.shape), V)


def test_store_matches_the_contiguous_caches_store():
    """One axis, fp32, adjacent pairs: the bits of b2_rope_kv_store_typed."""
    n_head, n_kv, hd, n = 8, 2, 64, 37
    for t in (F16, Q8, Q4):
        s = Setup([n], [n], n_head, n_kv, hd, 64, t, t, F32, poison=False, extra_pages=0)
        r = np.random.default_rng(3)
        x = dev(r.standard_normal((n, n_head + 2 * n_kv, hd), dtype=np.float32))
        table, pos = dev(b2.rope_table(10000.0, hd, 0, 64)), dev(np.arange(n, dtype=np.int32))
        c, q = s.cache(), b2.DeviceBuffer(n * n_head * hd * 4)
        b2.page_rope_store(c, 0, s.batch(), n_head, x, F32, q, F32, pos, 1, None, table, 64, hd)
        q2, k2, v2 = b2.DeviceBuffer(q.nbytes), dev(s.K), dev(s.V)     # one page of 64 is [n_kv][cap = 64]
        b2.check(b2.lib.b2_rope_kv_store_typed(x.ptr, n, 1, n_head, n_kv, hd, pos.ptr, dev(np.zeros(n, np.int32)).ptr,
                                               table.ptr, q2.ptr, k2.ptr, t, v2.ptr, t, 64, None))
        b2.synchronize()
        for a, b in ((q, q2), (s.k, k2), (s.v, v2)):
            assert np.array_equal(a.download(np.uint8), b.download(np.uint8))


def test_store_tokens_without_a_place():
    """Rotary positions outside the table, a missing page, more tokens than
    positions, rows past the last sequence: zero q rows (the last: untouched),
    nothing stored."""
    s = Setup([2, 3, 2], [2, 2, 2], 4, 2, 64, 16, qt=F32, poison=False)
    s.table[2, 0] = -1
    n = s.n_tok
    x = np.random.default_rng(0).standard_normal((n + 2, 8, 64), dtype=np.float32)
    pos = np.array([0, 99, 0, 1, 2, 3, 4, 5, 6], np.int32)      # token 1 outside a table of 50
    c, q = s.cache(), dev(np.full((n + 2, 4, 64), 77, np.float32))
    b = b2.PageBatch(s.q_start, np.array(s.kv_len, np.int32), s.table, n_tok=n + 2, max_q=3)
    b2.page_rope_store(c, 0, b, 4, dev(x), F32, q, F32, dev(pos), 1, None, dev(b2.rope_table(1e4, 64, 0, 50)), 50, 64)
    b2.synchronize()
    got = q.download(np.float32).reshape(n + 2, 4, 64)
    zero = [1, 2, 5, 6]      # table, position -1, no page
    assert np.all(got[zero] == 0) and np.all(got[[0, 3, 4]] != 77) and np.all(got[n:] == 77)
    k = s.k.download(np.uint8).reshape(s.K.shape)
    touched = {(int(s.table[0, 0]), 0), (int(s.table[1, 0]), 0), (int(s.table[1, 0]), 1)}
    for page in range(s.n_pages):
        for slot in range(16):
            assert ((page, slot) in touched) != np.array_equal(k[0, page, :, slot], s.K[0, page, :, slot])


# ---- pages -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q4)])
@pytest.mark.parametrize("n_copy", [1, 7, 300])
def test_copy(kt, vt, n_copy):
    s = Setup([1], [1], 2, 2, 96, 8, kt, vt, n_layer=3, poison=False, extra_pages=2 * n_copy + 5)
    order = np.random.default_rng(n_copy).permutation(s.n_pages).astype(np.int32)
    src, dst = order[:n_copy].copy(), order[n_copy:2 * n_copy].copy()
    if n_copy > 2:
        src[1] = src[0]                          # one page copied twice
    c = s.cache()
    b2.page_copy(c, src, dst)
    b2.synchronize()
    for pool, d in ((s.K, s.k), (s.V, s.v)):
        want = pool.copy()
        want[:, dst] = pool[:, src]
        assert np.array_equal(d.download(np.uint8).reshape(pool.shape), want)


@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q4)])
@pytest.mark.parametrize("page", [8, 16, 64])
def test_gather(kt, vt, page):
    """Kept positions move to fresh pages in every layer; a list of none, of
    one, of all; pages that stay are not touched."""
    r = np.random.default_rng(page)
    kv = [77, 5, 130, 64, 1]
    s = Setup([1] * 5, kv, 2, 2, 64, page, kt, vt, n_layer=2, poison=False, extra_pages=300)
    keeps = [np.sort(r.choice(77, 40, False)), np.arange(0), np.concatenate([np.arange(70), np.arange(100, 130)]),
             np.arange(64), np.arange(1)]
    used = set(s.table[s.table >= 0].tolist())
    free = [p for p in range(s.n_pages) if p not in used]
    new = np.full_like(s.table, -1)
    for i, k in enumerate(keeps):
        n = -(-len(k) // page)
        stay = (70 // page if i == 2 else n if i == 3 else 0)
        new[i, :stay] = s.table[i, :stay]
        for x in range(stay, n):
            new[i, x] = free.pop()
    start = np.concatenate([[0], np.cumsum([len(k) for k in keeps])]).astype(np.int32)
    c = s.cache()
    keep = np.concatenate(keeps).astype(np.int32)
    b2.page_gather(c, 5, dev(start), dev(keep), keep.size, dev(s.table), dev(new), s.max_pages)
    b2.synchronize()
    for pool, d in ((s.K, s.k), (s.V, s.v)):
        want = pool.copy()
        for i, k in enumerate(keeps):
            for to, p in enumerate(k):
                want[:, new[i, to // page], :, to % page] = pool[:, s.table[i, p // page], :, p % page]
        assert np.array_equal(d.download(np.uint8).reshape(pool.shape), want)


def test_gather_skips_positions_outside_the_tables():
    s = Setup([1], [20], 2, 2, 64, 16, poison=False)
    new = np.array([[s.table[0, 0] ^ 0, -1]], np.int32)
    free = [p for p in range(s.n_pages) if p not in s.table[0]]
    new[0, 0] = free[0]
    c = s.cache()
    b2.page_gather(c, 1, dev(np.array([0, 3], np.int32)), dev(np.array([-1, 19, 5000], np.int32)), 3, dev(s.table),
                   dev(new), 2)
    b2.synchronize()
    want = s.K.copy()
    want[:, free[0], :, 1] = s.K[:, s.table[0, 1], :, 3]
    assert np.array_equal(s.k.download(np.uint8).reshape(want.shape), want)


# ---- together -----------------------------------------------------------------------------------------
def test_example_conversations():
    """examples/paged_chat.py: a forked conversation decoded token by token
    gives the hidden states of the same tokens fed alone in one piece.  The
    two differ by the order of fp32 sums and by Q8_0 codes of activations that
    such differences move across a rounding boundary (one code is 1/127 of a
    block's largest value, in one of 512 products)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_chat.py")
    spec = importlib.util.spec_from_file_location("paged_chat", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for users, steps in ((2, 3), (4, 20)):
        difference, size = mod.main(n_users=users, steps=steps, seed=users)
        assert difference < 2e-2 * size


@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_nonfinite_values_in_whole_tiles(qt):
    """As above, with enough sequences that tiles are finished by one CTA."""
    n_seq, q_len, n = 24, 70, 90
    s = Setup([q_len] * n_seq, [n] * n_seq, 16, 4, 64, 16, qt=qt, seed=2)
    for i in range(n_seq):
        p = n - 1 - (i % 40)
        s.V[0, s.table[i, p // 16], :, p % 16, 6:8] = np.frombuffer(np.uint16(0x7C00 if i % 2 else 0x7E00).tobytes(), np.uint8)
    got = s.run().astype(np.float64).reshape(n_seq, q_len, 16, 64)
    clean = Setup([q_len] * n_seq, [n] * n_seq, 16, 4, 64, 16, qt=qt, seed=2)
    want, vmax = (x.reshape(n_seq, q_len, 16, -1) for x in clean.want())
    tol = 2e-5 * vmax + (2.0 ** -10 * vmax if qt == F16 else 0)
    for i in range(n_seq):
        first = q_len - 1 - (i % 40)          # the first row that sees the value, in dim 3
        assert np.all(~np.isfinite(got[i, first:, :, 3]))
        got[i, first:, :, 3] = want[i, first:, :, 3]
    assert np.all(np.abs(got - want) <= tol)


def test_attn_fp32_accuracy_does_not_fall_with_length():
    """A chunk's fp32 sums over many positions, held to 4e-6 of the result in
    the 2-norm: a score's products keep 22 bits of q (2^-23 each, of terms that
    add like a random walk) and sums of at most 48 steps of 16 that the tensor
    pipe cuts at 2^-24 each, 48 · 2^-24 = 2.9e-6 if every cut fell alike."""
    for n in (2000, 12000):
        s = Setup([24], [n], 4, 1, 128, 64, qt=F32, seed=n)
        got = s.run().astype(np.float64)
        want, _ = s.want()
        assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)
