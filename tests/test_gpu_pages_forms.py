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
