"""Page attention in every form that a call can take, held to 64 bits: shares
of many tiles and units, caches of every type, values of every size.

Tolerances.  Of a row element by element as in test_gpu_pages.py.  In the
2-norm with B2_F32: a score's 22 bits of q and its sum's 2^-24 a step of the
tensor pipe, a weight's ex2.approx and its two parts at 2^-22 each, and sums of
V that the pipe cuts at 2^-24 a step between additions with rounding, at most
48 steps: below 4e-6 together.  With B2_F16 a weight and the result are rounded
to 2^-11 each, 2^-11/sqrt(3) in the 2-norm, so 2^-11 holds both, beside
2^-25 a value where results are subnormal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

b2 = pytest.importorskip("b2gguf")
from tests.test_gpu_pages import F16, F32, NP, Q4, Q8, Setup, rows_of  # noqa: E402


def shared(n_seq, n, n_head, n_kv, hd, page, kt, vt, qt, seed, q_len=1, k=None, v=None):
    """n_seq sequences over the same pages of n positions: much work over a
    small pool.  k, v: the pool's values from unit normal ones."""
    s = Setup([q_len], [n], n_head, n_kv, hd, page, kt, vt, qt, seed=seed, poison=False)
    r = np.random.default_rng(seed + 1)
    shape = (1, s.n_pages, n_kv, page, hd)
    if k is not None:
        s.K = rows_of(k(r.standard_normal(shape, dtype=np.float32)).astype(np.float32), kt)
    if v is not None:
        s.V = rows_of(v(r.standard_normal(shape, dtype=np.float32)).astype(np.float32), vt)
    s.q_len, s.kv_len = [q_len] * n_seq, [n] * n_seq
    s.table = np.repeat(s.table, n_seq, 0)
    s.q_start = (q_len * np.arange(n_seq + 1)).astype(np.int32)
    s.n_tok = int(s.q_start[-1])
    s.Q = r.standard_normal((s.n_tok, n_head, hd), dtype=np.float32).astype(NP[qt])
    return s


def sampled(s, got, n_rows, seed=0, window=0, scale=None):
    """Some (token, head) rows of the result, the same in 64 bits, and the largest |v| each sees."""
    r = np.random.default_rng(seed)
    scale = s.hd ** -0.5 if scale is None else scale
    G, kv, a, b, top = s.n_head // s.n_kv, {}, [], [], []
    for x in np.sort(r.choice(s.n_tok * s.n_head, min(n_rows, s.n_tok * s.n_head), False)):
        row, h = divmod(int(x), s.n_head)
        q = int(np.searchsorted(s.q_start, row, side="right")) - 1
        key = (s.table[q].tobytes(), s.kv_len[q])
        if key not in kv:
            kv = {key: s.seq_values(q, s.kv_len[q])}
        k, v = kv[key]
        p = s.kv_len[q] - s.q_len[q] + row - s.q_start[q]
        lo = max(0, p - window + 1) if window else 0
        a.append(got[row, h].astype(np.float64))
        if p < 0:
            b.append(np.zeros(s.hd))
            top.append(0.0)
            continue
        z = k[lo:p + 1, h // G] @ s.Q[row, h].astype(np.float64) * scale
        w = np.exp(z - z.max())
        b.append((w / w.sum()) @ v[lo:p + 1, h // G])
        top.append(np.abs(v[lo:p + 1, h // G]).max())
    return np.array(a), np.array(b), np.array(top)[:, None]


def check_sampled(s, n_rows=300, **kw):
    got = s.run(**kw)
    assert np.all(np.isfinite(got.astype(np.float32)))
    kw.pop("workspace", None)
    kw.pop("stream", None)
    a, w, top = sampled(s, got, n_rows, **kw)
    tol = 2e-5 * top + (2.0 ** -10 * top if s.qt == F16 else 0) + 1e-30
    assert np.all(np.abs(a - w) <= tol), f"worst {np.max(np.abs(a - w) / tol):.3g} of the tolerance"
    return got


# ---- shares of many units and tiles: every stage of the rings is used again ----------------------
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("n_head,n_kv,hd,q_len,n_seq", [
    (16, 8, 64, 1, 500), (8, 8, 128, 1, 300), (96, 8, 64, 1, 400),     # warps along the positions: two parts, and (fp16) one
    (8, 4, 96, 9, 150), (4, 4, 256, 17, 90)])                          # warps along the rows
def test_attn_stages_used_again_after_masked_units(n_head, n_kv, hd, q_len, n_seq, qt):
    """Many ragged tiles a CTA over fp16 pages: every tile ends inside a unit
    or within a causal edge, whose V is changed in shared memory, and the next
    tiles' copies take the same stages."""
    r = np.random.default_rng(hd)
    kv = [int(x) for x in r.integers(q_len, 260, n_seq)]
    check_sampled(Setup([q_len] * n_seq, kv, n_head, n_kv, hd, 16, qt=qt, seed=hd + q_len), 400)


# ---- values of every size ------------------------------------------------------------------------
FORMS = {"tokens": (1, 8, 4), "tokens of 12 heads": (1, 12, 1), "chunk": (40, 4, 2)}   # new tokens, heads, kv heads


def check_norm(s, blocks=1, n_rows=200, **kw):
    """The 2-norm's bound, for every run of hd / blocks values on its own."""
    got = s.run(**kw)
    a, w, _ = sampled(s, got, n_rows, **kw)
    for x, y in zip(np.split(a, blocks, 1), np.split(w, blocks, 1)):
        tol = 4e-6 * np.linalg.norm(y) if s.qt == F32 else 2.0 ** -11 * np.linalg.norm(y) + 2.0 ** -25 * y.size ** 0.5
        err = np.linalg.norm(x - y)
        assert err <= tol, f"{err / np.linalg.norm(y):.3g} of the result, {err / tol:.3g} of the tolerance"


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("t", [Q8, Q4])
@pytest.mark.parametrize("size", [1, 1e-2, 1e-3, 1e-4, 300])
def test_attn_quantized_values_of_any_size(form, qt, t, size):
    q_len, n_head, n_kv = FORMS[form]
    check_norm(shared(3, 1500, n_head, n_kv, 128, 32, t, t, qt, 11, q_len, v=lambda x: size * x))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [Q8, Q4])
def test_attn_quantized_values_of_mixed_size(form, t):
    """Blocks of one row whose sizes differ: each is good on its own."""
    q_len, n_head, n_kv = FORMS[form]
    f = np.repeat(np.array([1, 1e-3, 30, 1e-2], np.float32), 32)
    check_norm(shared(3, 1500, n_head, n_kv, 128, 32, t, t, F32, 12, q_len, v=lambda x: f * x), blocks=4)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [Q8, Q4])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("grow", [1, -1])
def test_attn_quantized_values_growing_along_the_positions(form, t, hd, grow):
    """The largest block scale rises (or falls) by six decades along a sequence, and some blocks are zero."""
    q_len, n_head, n_kv = FORMS[form]
    s = shared(300, 900, n_head, n_kv, hd, 16, t, t, F32, 16, q_len)
    p = np.arange(900)
    size = 10.0 ** (grow * (p - 450) / 150)
    size[100:170] = 0
    v = np.random.default_rng(1).standard_normal((900, n_kv, hd)) * size[:, None, None]
    s.V[0, s.table[0, p // 16], :, p % 16] = rows_of(v.astype(np.float32), t)
    check_norm(s)


@pytest.mark.parametrize("form,hd", [("tokens", 64), ("tokens", 128), ("chunk", 64), ("chunk", 128), ("chunk", 96)])
@pytest.mark.parametrize("qt,size", [(F32, 1e-4), (F32, 1e-3), (F32, 1), (F32, 1.4e4), (F32, 1e6), (F16, 1e-3), (F16, 1.4e4)])
@pytest.mark.parametrize("kt", [F16, Q8])
def test_attn_queries_of_any_size(form, hd, qt, size, kt):
    """Scores of unit size from small queries and large keys and the reverse;
    products of large ones pass fp16's range."""
    q_len, n_head, n_kv = FORMS[form]
    s = shared(3, 700, n_head, n_kv, hd, 16, kt, kt, qt, 13, q_len, k=lambda x: x / (size * hd ** 0.5))
    s.Q = s.Q.astype(np.float32) * np.float32(size)
    s.Q = (s.Q if qt == F32 else np.clip(s.Q, -65504, 65504)).astype(NP[qt])
    check_norm(s, scale=1.0)
    check_norm(s, scale=-1.0)


@pytest.mark.parametrize("form,hd", [("tokens", 64), ("tokens", 128), ("chunk", 64), ("chunk", 128), ("chunk", 96)])
def test_attn_rows_of_mixed_size(form, hd):
    """Rows of one call between 1e-20 and 1e20 and all-zero ones: none disturbs
    another.  Scores of the large ones only tell the largest key."""
    q_len, n_head, n_kv = FORMS[form]
    s = shared(3, 400, n_head, n_kv, hd, 16, F16, F16, F32, 14, q_len)
    size = 10.0 ** np.array([0, -20, 20, 1, -3, -38])[np.arange(s.n_tok * n_head) % 6].reshape(s.n_tok, n_head, 1)
    s.Q = (s.Q * size).astype(np.float32)
    s.Q[0, 0] = 0
    check_sampled(s)
    check_sampled(s, scale=0.0)


@pytest.mark.parametrize("form,hd", [("tokens", 128), ("chunk", 64), ("chunk", 128), ("chunk", 96)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_attn_nonfinite_queries_stay_in_their_rows(form, hd, bad):
    q_len, n_head, n_kv = FORMS[form]
    s = shared(3, 400, n_head, n_kv, hd, 16, F16, F16, F32, 14, q_len)
    clean = s.run()
    s.Q[1::2, 1, 5] = bad
    got = s.run()
    assert np.all(np.isnan(got[1::2, 1]))
    got[1::2, 1] = clean[1::2, 1]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("form,hd", [("tokens", 64), ("tokens of 12 heads", 128), ("chunk", 64), ("chunk", 128), ("chunk", 96)])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_scores_of_any_size(form, hd, qt):
    """Scores past 2^24, whose rounding alone is more than an exponent may be
    off by: each row takes the value of its largest key."""
    q_len, n_head, n_kv = FORMS[form]
    for size in (1e2, 1e4, 6e4):
        s = shared(3, 700, n_head, n_kv, hd, 16, F16, F16, qt, 17, q_len, k=lambda x: np.clip(x * size, -65504, 65504))
        s.Q = np.clip(s.Q.astype(np.float32) * size, -65504, 65504).astype(NP[qt])
        check_sampled(s, scale=1.0)
        check_sampled(s, scale=-1.0)


@pytest.mark.parametrize("form,hd", [("tokens", 64), ("tokens of 12 heads", 128), ("chunk", 64), ("chunk", 128), ("chunk", 96)])
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("vt", [F16, Q8])
def test_attn_weights_add_up_at_any_score(form, hd, qt, vt):
    """Scores around 2^18 to 2^44, many within a few units of the last place of
    the largest: all values are one number, so every result is."""
    q_len, n_head, n_kv = FORMS[form]
    for size in (1.0, 2.0 ** -10):
        s = shared(3, 700, n_head, n_kv, hd, 16, F16, vt, qt, 18, q_len, k=lambda x: 1 - (x > 1) * 2.0 ** -11,
                   v=lambda x: 0 * x + size)
        s.Q = np.abs(s.Q.astype(np.float32) * 100 + 1000).astype(NP[qt])
        v = s.seq_values(0, 700)[1]
        assert np.all(v == v[0, 0, 0])
        for e in range(18, 45):
            for sign in (1, -1):
                got = s.run(scale=sign * 2.0 ** e / (1000 * hd)).astype(np.float64) / v[0, 0, 0]
                assert np.all(np.abs(got - 1) <= (2e-5 if qt == F32 else 2.0 ** -10)), (e, sign)


# ---- long shares ---------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [F16, Q8, Q4])
@pytest.mark.parametrize("hd,page,n_seq,n", [(64, 256, 70, 32768), (128, 64, 70, 32768), (96, 16, 70, 9000), (256, 8, 90, 9000)])
def test_attn_tokens_fp32_accuracy_does_not_fall_with_a_ctas_share(t, hd, page, n_seq, n):
    """A CTA adds over hundreds of units of one tile; values of one sign, so that cuts of a sum add up."""
    check_norm(shared(n_seq, n, 8, 8, hd, page, t, t, F32, 14, v=lambda x: 1 + x), n_rows=60)


@pytest.mark.parametrize("t,hd", [(F16, 64), (F16, 128), (F16, 96), (Q8, 64), (Q4, 128)])
def test_attn_chunks_fp32_accuracy_does_not_fall_with_a_ctas_share(t, hd):
    """The same with many rows: tiles of 16384 positions, two and more a CTA."""
    check_norm(shared(50, 16384, 32, 8, hd, 64, t, t, F32, 14, 30, v=lambda x: 1 + x), n_rows=60)


# ---- windows -------------------------------------------------------------------------------------
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("q_len,hd", [(4, 64), (70, 64), (70, 128), (40, 96)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 4096])
def test_attn_windows_past_every_position(q_len, hd, window, qt):
    """A window that hides nothing, with more new tokens than positions: the
    first ones' positions lie below zero."""
    s = Setup([q_len, 1, q_len], [q_len - 3, 0, q_len + 200], 8, 2, hd, 16, qt=qt, seed=3)
    got = s.check(window=window)
    assert np.all(got[:3] == 0)
    assert np.array_equal(got, s.run().astype(np.float64))


# ---- values that are not finite -------------------------------------------------------------------
@pytest.mark.parametrize("bits", [0x7C00, 0x7E00])
@pytest.mark.parametrize("q_len,hd,kt,qt", [(1, 64, F16, F32), (1, 128, F16, F16), (1, 128, Q8, F32), (40, 64, F16, F32),
                                            (40, 128, F16, F16), (40, 128, Q8, F16), (40, 96, F16, F32)])
def test_attn_infinite_value_of_a_low_score(q_len, hd, kt, qt, bits):
    """An infinite or NaN value whose weight is some e^-500, in another part of
    a split tile than the large weights, still reaches every row that sees it."""
    n, at = 6000, 10
    s = Setup([q_len], [n], 4, 2, hd, 16, kt, kt, qt, seed=15)
    p = np.arange(n)
    k = np.random.default_rng(0).standard_normal((1, s.n_pages, 2, 16, hd), dtype=np.float32)
    k[0, s.table[0, p // 16], :, p % 16] = np.where(p < n // 2, -20, 20)[:, None, None]
    s.K = rows_of(k, kt)
    s.Q = (np.abs(s.Q) + 1).astype(NP[qt])
    clean, _ = s.want()
    first = 0 if kt == F16 else hd           # a value, or the first block's scale
    s.V[0, s.table[0, at // 16], :, at % 16, first:first + 2] = [0, bits >> 8]
    got = s.run().astype(np.float64)
    touched = 1 if kt == F16 else 32
    assert np.all(~np.isfinite(got[..., :touched]).all(-1))
    tol = 1e-4 if qt == F32 else 4e-3        # the rest is as it was (|v| below 5)
    assert np.all(np.abs(got - clean)[..., touched:] <= tol)


# ---- the workspace -------------------------------------------------------------------------------
def test_workspace_is_zero_when_it_is_handed_out(monkeypatch):
    """For calls on any stream: streams of their own do not wait for the
    default one, which may be busy."""
    s = Setup([1], [100], 8, 2, 64, 16)
    c, b = s.cache(), s.batch()
    n = b2.page_attn_workspace_bytes(c, b, 8, F32)
    big, ws = b2.DeviceBuffer(8 << 30), b2.DeviceBuffer(n)
    host, st = b2.PinnedArray((n,), np.uint8), b2.Stream()
    b2.check(b2.lib.b2_memset(ws.ptr, 0xFF, n, None))
    b2.synchronize()
    for _ in range(20):                        # some 20 ms of work
        b2.check(b2.lib.b2_memset(big.ptr, 1, big.nbytes, None))
    with monkeypatch.context() as m:
        m.setattr(b2, "DeviceBuffer", lambda size: ws)
        assert b2.page_attn_workspace(c, b, 8, F32) is ws
    b2.check(b2.lib.b2_memcpy_d2h(host.p, ws.ptr, n, st.h))
    st.synchronize()
    got = host.array.copy()
    b2.synchronize()
    assert not got.any()


# ---- malformed batches ---------------------------------------------------------------------------
@pytest.mark.parametrize("qt,kt", [(F16, F16), (F32, F16), (F32, Q8)])
def test_attn_overlapping_sequences_that_pass_all_counts(qt, kt):
    """512 sequences that claim all of 65536 tokens each: more work units than
    32 bits count.  The call does nothing, and the workspace stays fit."""
    n, n_seq, n_kv, hd = 1 << 16, 1024, 8, 64
    c = b2.PageCache(1, 4, 256, n_kv, hd, kt, kt)
    start = np.where(np.arange(n_seq + 1) % 2, n, 0).astype(np.int32)
    start[-1] = n
    b = b2.PageBatch(start, np.full(n_seq, 1 << 20, np.int32), np.full((n_seq, 4096), -1, np.int32), n_tok=n, max_q=n)
    q, out = b2.DeviceBuffer(n * n_kv * hd * 4), b2.DeviceBuffer(n * n_kv * hd * 4)
    b2.check(b2.lib.b2_memset(out.ptr, 77, out.nbytes, None))
    ws = b2.page_attn_workspace(c, b, n_kv, qt)
    b2.page_attn(c, 0, b, n_kv, q, out, qt, workspace=ws)
    b2.synchronize()
    assert np.all(out.download(np.uint8) == 77)
    s = Setup([70, 3], [200, 300], 8, 2, 64, 16, kt, kt, qt, seed=1)
    c, b = s.cache(), s.batch()
    x, y = b2.DeviceBuffer.from_array(s.Q), b2.DeviceBuffer(s.Q.nbytes)
    assert b2.page_attn_workspace_bytes(c, b, 8, qt) <= ws.nbytes
    b2.page_attn(c, 0, b, 8, x, y, qt, workspace=ws)
    b2.synchronize()
    assert np.array_equal(y.download(NP[qt]).reshape(s.Q.shape), s.run())


# ---- every form over every cache -----------------------------------------------------------------
TYPES = [(a, b) for a in (F16, Q8, Q4) for b in (F16, Q8, Q4)]


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("n_head,n_kv", [(4, 4), (16, 2), (12, 1), (16, 1)])
def test_attn_single_tokens_over_every_cache(kt, vt, hd, qt, n_head, n_kv):
    """Steps of single tokens only: 1, 8, 12 and 16 rows a kv head."""
    kv = [1, 31, 33, 64, 130, 700]
    Setup([1] * len(kv), kv, n_head, n_kv, hd, 32, kt, vt, qt, seed=kt * 7 + vt + hd + n_head).check()


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_single_tokens_many_units_and_tiles(kt, vt, hd, qt):
    """At least 8 tiles and 60 units a CTA; fp16 queries with 12 heads a kv head and with one."""
    n_head = 96 if qt == F16 and hd <= 128 else 8
    check_sampled(shared(450 if hd < 256 else 150, 460, n_head, 8, hd, 16, kt, vt, qt, hd + kt, 1), 200)


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_chunks_many_units_and_tiles(kt, vt, hd, qt):
    """At least 6 tiles and 40 units a CTA in either kernel for many rows."""
    over_tc = kt == vt == F16 and hd in (64, 128)
    q_len, n_seq = (150, 80) if over_tc else (50, 180)
    check_sampled(shared(n_seq, 900, 16, 8, hd, 64, kt, vt, qt, hd + vt, q_len), 200)


@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q8), (Q4, Q8)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("window", [0, 100])
def test_attn_ragged_chunks_many_tiles(kt, vt, hd, qt, window):
    """Tiles of every length in one share, most of them short."""
    r = np.random.default_rng(hd + window)
    q = [int(x) for x in r.integers(0, 200, 90)]
    kv = [n + int(x) for n, x in zip(q, r.integers(0, 700, 90))]
    q[5], kv[5], kv[7] = 40, 10, 0
    check_sampled(Setup(q, kv, 16, 8, hd, 16, kt, vt, qt, seed=7), 300, window=window)


@pytest.mark.parametrize("page", [8, 128, 256])
@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q8), (Q4, Q4), (F16, Q4), (Q8, F16)])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("hd", [96, 256])
def test_attn_page_sizes_over_every_cache(page, kt, vt, q_len, hd):
    Setup([q_len, q_len], [q_len + 70, q_len + 257], 4, 2, hd, page, kt, vt, F32, seed=page).check()


@pytest.mark.parametrize("kt,vt", [(Q8, Q8), (Q4, Q4), (F16, Q8), (Q4, F16)])
@pytest.mark.parametrize("hd,n_head,n_kv,page", [(64, 8, 2, 8), (128, 4, 1, 32), (128, 6, 2, 256), (64, 5, 5, 128)])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_quantized_chunks(kt, vt, hd, n_head, n_kv, page, qt):
    Setup([130, 1, 0, 45, 3], [130, 257, 12, 300, 3], n_head, n_kv, hd, page, kt, vt, qt, seed=hd + page).check()


@pytest.mark.parametrize("window", [1, 50, 300])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("q_len", [[140, 64, 1], [1, 1, 1]])
@pytest.mark.parametrize("kt,vt", [(Q8, Q4), (Q4, Q4)])
def test_attn_quantized_windows(window, page, q_len, kt, vt):
    Setup(q_len, [700, 64, 513], 4, 2, 64, page, kt, vt, qt=F32, seed=window).check(window=window)


@pytest.mark.parametrize("q_len", [[128, 150, 30], [1, 150, 1], [1, 1, 1]])
@pytest.mark.parametrize("kt,vt", [(Q8, Q8), (Q4, F16), (F16, Q4)])
@pytest.mark.parametrize("qt", [F32, F16])
def test_attn_quantized_layer_table_and_workspace(q_len, kt, vt, qt):
    """Another layer, table entries outside the pool, more new tokens than
    positions, a workspace that holds anything past its counters."""
    s = Setup(q_len, [200, 140, 90], 4, 2, 128, 16, kt, vt, qt, seed=9, n_layer=3, layer=1)
    s.table[0, 3], s.table[2, 0] = -7, s.n_pages + 1
    a = s.check()
    assert np.array_equal(a, s.run(workspace=False).astype(np.float64))
    c, b = s.cache(), s.batch()
    ws = b2.page_attn_workspace(c, b, s.n_head, qt)
    x = np.full(ws.nbytes, 0x7E, np.uint8)
    x[:1 << 16] = 0                            # the counters
    ws.upload(x)
    q, out = b2.DeviceBuffer.from_array(s.Q), b2.DeviceBuffer(s.Q.nbytes)
    for _ in range(2):
        b2.page_attn(c, s.layer, b, s.n_head, q, out, qt, workspace=ws)
    b2.synchronize()
    assert np.array_equal(out.download(NP[qt]).reshape(s.Q.shape).astype(np.float64), a)


@pytest.mark.parametrize("bits", [0x7C00, 0xFC00, 0x7E00])
@pytest.mark.parametrize("t", [Q8, Q4])
@pytest.mark.parametrize("q_len,window", [(140, 0), (9, 0), (9, 5), (1, 0), (1, 20)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attn_nonfinite_scales(bits, t, q_len, window, hd):
    """Infinite and NaN block scales reach the rows that see them and no others."""
    n = 200
    at = n - 5 if q_len > 5 else n - 40
    s = Setup([q_len], [n], 4, 2, hd, 16, t, t, F32, seed=3)
    want, vmax = s.want(window=window)
    code = hd if t == Q8 else hd // 2
    for pool in (s.K, s.V):
        pool[0, s.table[0, at // 16], :, at % 16, code:code + 2] = np.frombuffer(np.uint16(bits).tobytes(), np.uint8)
    got = s.run(window=window).astype(np.float64)
    p = np.arange(n - q_len, n)
    sees = (p >= at) & ((p - at < window) if window else True)
    assert np.all(~np.isfinite(got[sees]).all(-1))
    assert np.all(np.abs(got - want)[~sees] <= 2e-5 * vmax[~sees])


@pytest.mark.parametrize("axes", [4, 5, 8])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 32)])
def test_store_of_many_axes(axes, style, hd, rot):
    """Bit for bit, as with fewer axes; and an axis past the last stores nothing."""
    from tests.test_gpu_pages import dev, rotate
    n_head, n_kv, n, n_pos, half = 4, 2, 29, 300, rot // 2
    s = Setup([n], [40], n_head, n_kv, hd, 16, qt=F32, seed=axes, poison=False)
    r = np.random.default_rng(axes)
    x = r.standard_normal((n, n_head + 2 * n_kv, hd), dtype=np.float32)
    pos = r.integers(0, n_pos, (axes, n)).astype(np.int32)
    axis = r.integers(0, axes, half).astype(np.uint8)
    table = b2.rope_table(10000.0, rot, 0, n_pos)
    for broken in (False, True):
        if broken:
            axis[half // 2] = axes
        c, q = s.cache(), dev(np.full((n, n_head, hd), 77, np.float32))
        b2.page_rope_store(c, 0, s.batch(), n_head, dev(x), F32, q, F32, dev(pos), axes, dev(axis), dev(table), n_pos, rot,
                           style)
        b2.synchronize()
        got, K = q.download(np.float32).reshape(n, n_head, hd), s.K.copy()
        if broken:
            assert not got.any()
        else:
            y = rotate(x[:, :n_head + n_kv], table.reshape(n_pos, half, 2)[pos[axis].T, np.arange(half)], style)
            assert np.array_equal(got, y[:, :n_head])
            p = 40 - n + np.arange(n)
            K[0, s.table[0, p // 16], :, p % 16] = rows_of(y[:, n_head:], F16)
        assert np.array_equal(s.k.download(np.uint8).reshape(K.shape), K)
