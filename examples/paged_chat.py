"""Conversations over one paged K/V cache: a small decoder of attention layers (random weights) that

1. feeds a shared prompt with a picture in it, in two chunks (rotary positions with three axes);
2. forks it for several users, whose first own token makes a copy of the shared, partly filled page;
3. decodes all users in one batch, step by step;
4. drops the middle of one user's conversation and gathers what is kept into fresh pages;
5. frees a user, moves the pages that are left to the front of the pool, and decodes on.

Run it from the repository's root on a machine with a B200:  python examples/paged_chat.py
"""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "arkantos-ai-stack-suite_b200"))
import b2gguf as b2  # noqa: E402


class PagedDecoder:
    """Attention layers with Q8_0 weights over a paged cache; every sequence
    of a step brings one token or many."""

    def __init__(self, n_layer=2, n_embd=512, n_head=8, n_kv=2, head_dim=64, n_pages=96, page_size=16, n_seq=8,
                 max_pages=32, type_kv=b2.F16, n_pos=4096, seed=0):
        self.n_layer, self.n_embd, self.n_head, self.n_kv, self.hd = n_layer, n_embd, n_head, n_kv, head_dim
        rows = (n_head + 2 * n_kv) * head_dim

        def weights(i, n, k):
            w = b2.synth_normal(seed + i, n * k, std=k ** -0.5).reshape(n, k)
            return b2.QMatrix(b2.Q8_0, b2.quantize_weights(b2.Q8_0, w), n, k)

        self.wqkv = [weights(2 * i, rows, n_embd) for i in range(n_layer)]
        self.wo = [weights(2 * i + 1, n_embd, n_head * head_dim) for i in range(n_layer)]
        self.norm = b2.DeviceBuffer.from_array(np.ones(n_embd, np.float32))
        self.rope = b2.DeviceBuffer.from_array(b2.rope_table(10000.0, head_dim, 0, n_pos))
        self.n_pos = n_pos
        half = head_dim // 2       # time, height and width share the pairs 1 : 1.5 : 1.5
        third = 3 * half // 8
        self.axis = b2.DeviceBuffer.from_array(b2.rope_sections([half - 2 * third, third, third]))
        self.cache = b2.PageCache(n_layer, n_pages, page_size, n_kv, head_dim, type_kv, type_kv)
        self.pool = b2.PagePool(n_pages, page_size, n_seq, max_pages)
        self.workspace = None

    def extend(self, seq, n):
        """Room for n positions; the copy a shared page needs before it is written."""
        rc, copy = self.pool.extend(seq, n)
        if rc:
            raise RuntimeError("the pool has no pages left")
        if copy:
            b2.page_copy(self.cache, [copy[0]], [copy[1]])

    def step(self, seqs, embeds, positions):
        """embeds[i] [n][n_embd] and positions[i] [3][n] of the new tokens of
        sequence seqs[i]; the hidden states of all of them [n_tok][n_embd]."""
        lengths = [len(e) for e in embeds]
        for s, n in zip(seqs, lengths):
            self.extend(s, n)
        batch = self.pool.batch(seqs, lengths)
        n_tok = sum(lengths)
        x = b2.DeviceBuffer.from_array(np.concatenate(embeds).astype(np.float32))
        pos = b2.DeviceBuffer.from_array(np.concatenate(positions, axis=1).astype(np.int32))
        h, y = b2.DeviceBuffer(x.nbytes), b2.DeviceBuffer(x.nbytes)
        qkv = b2.DeviceBuffer(n_tok * self.wqkv[0].n_rows * 4)
        q, o = (b2.DeviceBuffer(n_tok * self.n_head * self.hd * 4) for _ in range(2))
        need = b2.page_attn_workspace_bytes(self.cache, batch, self.n_head, b2.F32)
        if self.workspace is None or self.workspace.nbytes < need:
            self.workspace = b2.page_attn_workspace(self.cache, batch, self.n_head, b2.F32)
        delta = None
        for i in range(self.n_layer):
            b2.check(b2.lib.b2_rmsnorm(x.ptr, delta.ptr if delta else None, self.norm.ptr, h.ptr, n_tok, self.n_embd,
                                       1e-5, None), "rmsnorm")
            self.project(self.wqkv[i], h, n_tok, qkv)
            b2.page_rope_store(self.cache, i, batch, self.n_head, qkv, b2.F32, q, b2.F32, pos, 3, self.axis, self.rope,
                               self.n_pos, self.hd, b2.ROPE_HALVES)
            b2.page_attn(self.cache, i, batch, self.n_head, q, o, b2.F32, workspace=self.workspace)
            self.project(self.wo[i], o, n_tok, y)
            delta = y
        b2.check(b2.lib.b2_rmsnorm(x.ptr, delta.ptr, self.norm.ptr, h.ptr, n_tok, self.n_embd, 1e-5, None), "rmsnorm")
        return h.download(np.float32).reshape(n_tok, self.n_embd)

    @staticmethod
    def project(w, x, n_tok, y):
        (w.gemv_device if n_tok <= 8 else w.gemm_device)(x, n_tok, y)

    def keep(self, seq, positions):
        """Drops all but the given positions of a sequence."""
        rc, old = self.pool.keep(seq, positions)
        if rc:
            raise RuntimeError("the pool has no pages left")
        keep = np.ascontiguousarray(positions, np.int32)
        start = b2.DeviceBuffer.from_array(np.array([0, keep.size], np.int32))
        lists = [b2.DeviceBuffer.from_array(a) for a in (keep, old, self.pool.table([seq])[0])]
        b2.page_gather(self.cache, 1, start, lists[0], keep.size, lists[1], lists[2], self.pool.max_pages)
        self.pool.settle()
        b2.synchronize()       # the lists live until the gather has run

    def defrag(self):
        src, dst = self.pool.defrag()
        b2.page_copy(self.cache, src, dst)
        return len(src)


def text(first, n):
    """Positions of n text tokens: all axes run together."""
    return np.tile(np.arange(first, first + n), (3, 1))


def picture(first, height, width):
    """Positions of a picture's tokens: one moment, rows and columns."""
    r, c = np.divmod(np.arange(height * width), width)
    return np.stack([np.full(height * width, first), first + r, first + c])


def main(n_users=3, steps=12, seed=0):
    rng = np.random.default_rng(seed)
    m = PagedDecoder(seed=seed)

    def tokens(n):
        return rng.standard_normal((n, m.n_embd)).astype(np.float32)

    # the shared prompt: 21 text tokens, a picture of 6 x 8, 20 more of text
    prompt = tokens(21 + 48 + 20)
    where = np.concatenate([text(0, 21), picture(21, 6, 8), text(29, 20)], axis=1)
    m.step([0], [prompt[:50]], [where[:, :50]])
    m.step([0], [prompt[50:]], [where[:, 50:]])
    free = m.pool.free_pages()
    users = list(range(n_users))
    for u in users[1:]:
        m.pool.fork(0, u)
    assert m.pool.free_pages() == free                      # the prompt is held once
    said = {u: [] for u in users}
    heard = {u: [] for u in users}

    def decode(seqs, n):
        for _ in range(n):
            new = [tokens(1) for _ in seqs]
            at = [text(49 + len(said[u]), 1) for u in seqs]
            for u, t in zip(seqs, new):
                said[u].append(t)
            for u, row in zip(seqs, m.step(seqs, new, at)):
                heard[u].append(row)

    decode(users, steps)
    # the same conversation without sharing, in one piece: the same hidden states
    last = users[-1]
    alone = n_users
    whole = np.concatenate([prompt] + said[last])
    again = m.step([alone], [whole], [np.concatenate([where, text(49, steps)], axis=1)])
    worst = float(np.abs(again[-steps:] - np.stack(heard[last])).max())
    print(f"{n_users} users over one prompt of {len(prompt)} tokens: {steps} steps each, "
          f"{m.pool.n_pages - m.pool.free_pages()} pages in use, forked against alone {worst:.1e}")
    m.pool.truncate(alone)
    # user 0 drops the picture; another user leaves
    length = m.pool.length(0)
    m.keep(0, list(range(21)) + list(range(69, length)))
    m.pool.truncate(1)
    before = m.step([0], [tokens(1)], [text(80, 1)])
    m.pool.truncate(0, m.pool.length(0) - 1)
    moved = m.defrag()
    used = m.pool.n_pages - m.pool.free_pages()
    decode([u for u in users if u != 1], 2)
    print(f"picture dropped: {length} -> {m.pool.length(0) - 2} positions; {moved} pages moved, {used} in use")
    return worst, float(np.abs(before).max())


if __name__ == "__main__":
    difference, size = main()
    assert difference < 1e-3 * size
