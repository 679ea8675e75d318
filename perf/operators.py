"""The paged K/V cache operators, as they are measured.

Four operators of one decoder layer over a cache whose positions live in fixed-size pages:

* ``store``: rotary positions with one or several axes (time, height, width) applied to the q and k heads of
  fused q|k|v rows; q handed on, k and v written to the pages of their sequences;
* ``attn``: causal (optionally windowed) attention of each sequence's newest tokens, one or many, over the pages
  of that sequence;
* ``copy``: whole pages copied in every layer (a forked sequence's first write to a shared page, or pages moved
  down so that the used ones are a prefix of the pool);
* ``gather``: kept positions of sequences gathered into fresh pages in every layer (positions dropped from the
  middle of a conversation).

Sequence s has its new tokens at rows q_start[s] .. q_start[s + 1] of the token arrays; they are the last ones of
its kv_len[s] positions.  Position p of a sequence is slot p % page of page table[s][p // page].
"""
import math

import torch

own = False

F32, F16, Q4_0, Q8_0 = 0, 1, 2, 8          # ggml type ids, as the framework uses them
NAMES = {"f32": F32, "f16": F16, "q4_0": Q4_0, "q8_0": Q8_0}
TORCH = {"f32": torch.float32, "f16": torch.float16}


# ---- cases ----------------------------------------------------------------------------------------------------
def listed():
    b8 = {"n_head": 32, "n_kv": 8, "hd": 128}      # the 8B model's heads
    b1 = {"n_head": 32, "n_kv": 4, "hd": 64}       # the 1.1B model's heads
    return [
        # one user, one token: every layer of every step waits for this call
        {"name": "attn_one_token", "op": "attn", **b1, "page": 16, "q": "f32", "k": "f16", "v": "f16", "window": 0,
         "n_seq": 1, "q_min": 1, "q_max": 1, "kv_min": 517, "kv_max": 517},
        # a served batch in its decode steps, conversations of different lengths
        {"name": "attn_decode_batch", "op": "attn", **b8, "page": 64, "q": "f16", "k": "f16", "v": "f16", "window": 0,
         "n_seq": 8, "q_min": 1, "q_max": 1, "kv_min": 700, "kv_max": 2057},
        # long conversations over the 8-bit cache, the default cache type of the host program
        {"name": "attn_decode_q8_0", "op": "attn", **b8, "page": 32, "q": "f32", "k": "q8_0", "v": "q8_0",
         "window": 0, "n_seq": 16, "q_min": 1, "q_max": 1, "kv_min": 4001, "kv_max": 4096},
        # the next piece of a long prompt that is fed in chunks
        {"name": "attn_chunk", "op": "attn", **b8, "page": 32, "q": "f16", "k": "f16", "v": "f16", "window": 0,
         "n_seq": 1, "q_min": 512, "q_max": 512, "kv_min": 4096, "kv_max": 4096},
        # prompts of 8 users at once, ragged
        {"name": "attn_prompts", "op": "attn", **b8, "page": 64, "q": "f16", "k": "f16", "v": "f16", "window": 0,
         "n_seq": 8, "q_min": 1500, "q_max": 2048, "kv_min": 0, "kv_max": 0},
        # one step of a server that mixes decoding sequences with short chunks, in the framework's fp32 activations
        {"name": "attn_mixed_f32", "op": "attn", **b8, "page": 64, "q": "f32", "k": "f16", "v": "f16", "window": 0,
         "n_seq": 16, "q_min": 1, "q_max": 129, "kv_min": 300, "kv_max": 2049},
        # a decode step of 8 text sequences: one position axis
        {"name": "store_decode", "op": "store", **b8, "page": 64, "x": "f32", "q": "f32", "axes": 1, "style": 0,
         "rot": 128, "n_seq": 8, "q_min": 1, "q_max": 1, "kv_min": 700, "kv_max": 2057, "n_pos": 4096},
        # prompts with images: three position axes, rotation of half-split pairs, queries for the tensor cores
        {"name": "store_images", "op": "store", **b8, "page": 64, "x": "f32", "q": "f16", "axes": 3, "style": 1,
         "rot": 128, "n_seq": 8, "q_min": 1500, "q_max": 2048, "kv_min": 0, "kv_max": 0, "n_pos": 4096},
        # a forked conversation writes to its shared last page
        {"name": "copy_on_write", "op": "copy", "n_layer": 22, "n_kv": 4, "hd": 64, "page": 16, "n_pages": 64,
         "n_copy": 1},
        # scattered pages moved to the front of the pool
        {"name": "copy_defrag", "op": "copy", "n_layer": 32, "n_kv": 8, "hd": 128, "page": 32, "n_pages": 96,
         "n_copy": 40},
        # one conversation drops a quarter of its middle
        {"name": "gather_one", "op": "gather", "n_layer": 22, "n_kv": 4, "hd": 64, "page": 16, "n_seq": 1,
         "kv_min": 517, "kv_max": 517, "drop": 0.25},
        # four long ones do, in the 8B model's cache
        {"name": "gather_four", "op": "gather", "n_layer": 32, "n_kv": 8, "hd": 128, "page": 32, "n_seq": 4,
         "kv_min": 900, "kv_max": 1024, "drop": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = [(32, 8, 128), (32, 4, 64), (16, 16, 128), (24, 8, 128), (64, 8, 128), (8, 8, 64), (32, 8, 96),
             (16, 8, 256)]
    top = work(next(c for c in listed() if c["name"] == "attn_prompts"))
    while True:
        op = rng.choice(["attn", "attn", "attn", "store", "copy", "gather"])
        n_head, n_kv, hd = rng.choice(heads)
        c = {"op": op, "n_kv": n_kv, "hd": hd, "page": rng.choice([16, 16, 32, 64, 128])}
        if op in ("attn", "store"):
            c.update(n_head=n_head, n_seq=_log(rng, 1, 32), q=rng.choice(["f32", "f16"]))
            kind = rng.choice(["decode", "chunk", "prompt", "mixed"])
            lo = _log(rng, 16, 4096)
            c.update(kv_min=max(1, int(lo * rng.uniform(0.3, 1.0))), kv_max=lo)
            q = _log(rng, 2, 2048)
            c.update({"decode": {"q_min": 1, "q_max": 1}, "chunk": {"q_min": max(1, q // 2), "q_max": q},
                      "prompt": {"q_min": max(1, q // 2), "q_max": q, "kv_min": 0, "kv_max": 0},
                      "mixed": {"q_min": 1, "q_max": min(q, 256)}}[kind])
        if op == "attn":
            k, v = rng.choice([("f16", "f16"), ("f16", "f16"), ("q8_0", "q8_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0"),
                               ("f16", "q8_0")])
            c.update(k=k, v=v, window=rng.choice([0, 0, 0, _log(rng, 8, 2048)]))
            # the plain form's padded scores stay within a few gigabytes
            pad = c["n_seq"] * n_head * c["q_max"] * (c["q_max"] + c["kv_max"])
            if pad > 1.2e9:
                continue
        elif op == "store":
            c.update(x=rng.choice(["f32", "f16"]), axes=rng.choice([1, 2, 3]), style=rng.choice([0, 1]),
                     rot=rng.choice([hd, hd, hd // 2]), n_pos=8192)
        elif op == "copy":
            c.update(n_layer=rng.randint(2, 32), n_pages=rng.choice([32, 64, 96]), n_copy=_log(rng, 1, 16))
        else:
            c.update(n_layer=rng.randint(2, 32), n_seq=rng.randint(1, 4), drop=round(rng.uniform(0.05, 0.6), 2))
            hi = _log(rng, 16, 1024)
            c.update(kv_min=max(2, hi // 2), kv_max=max(2, hi))
        if op in ("copy", "gather") and work(c)["bytes"] > 3e8:
            continue
        if op in ("attn", "store") and _store_bytes(c) > 6e8:
            continue
        if op == "attn" and (work(c)["flops"] > top["flops"] or work(c)["bytes"] > 2e9):
            continue
        return c


# ---- sizes ----------------------------------------------------------------------------------------------------
def _row_bytes(t, hd):
    """A cache row of one head at one position: fp16 values, or codes, the fp16 scales of 32-value blocks, padding."""
    return {F16: 2 * hd, Q8_0: hd + 16, Q4_0: hd // 2 + 16}[t]


def _lengths(case, salt=17):
    """New tokens and positions of every sequence: spread evenly over the case's ranges, the same for every seed."""
    n = case["n_seq"]
    spread = [((i * 7 + salt) % n) / max(1, n - 1) for i in range(n)]
    q = [round(case["q_min"] + f * (case["q_max"] - case["q_min"])) for f in spread]
    if case["q_min"] == 1 < case["q_max"] and case["kv_max"]:      # mixed steps: three of four sequences decode
        q = [x if i % 4 == 0 else 1 for i, x in enumerate(q)]
        q[0] = case["q_max"]
    back = [round(case["kv_min"] + f * (case["kv_max"] - case["kv_min"])) for f in reversed(spread)]
    return q, [max(a, b) for a, b in zip(q, back)]


def _store_bytes(case):
    q, kv = _lengths(case)
    return (sum(q) * (case["n_head"] + 2 * case["n_kv"]) + sum(kv) * 2 * case["n_kv"]) * case["hd"] * 4


def work(case):
    if case["op"] == "copy":
        return {"bytes": 2 * 2 * case["n_copy"] * case["n_layer"] * case["n_kv"] * case["page"] * 2 * case["hd"],
                "flops": 0}
    if case["op"] == "gather":
        kept = sum(len(_kept(n, case["drop"])) for n in _gather_lengths(case))
        return {"bytes": 2 * 2 * kept * case["n_layer"] * case["n_kv"] * 2 * case["hd"] + 4 * kept, "flops": 0}
    q, kv = _lengths(case)
    n_tok, hd = sum(q), case["hd"]
    if case["op"] == "store":
        rows = case["n_head"] + 2 * case["n_kv"]
        size = {"f32": 4, "f16": 2}
        return {"bytes": n_tok * (rows * hd * size[case["x"]] + case["n_head"] * hd * size[case["q"]] +
                                  2 * case["n_kv"] * 2 * hd + case["rot"] * 4 + case["axes"] * 4),
                "flops": 3 * n_tok * (case["n_head"] + case["n_kv"]) * case["rot"]}
    w, pairs, read = case["window"], 0, 0
    for a, b in zip(q, kv):
        first = b - a                                               # position of the first new token
        seen = [min(p + 1, w) if w else p + 1 for p in range(first, b)]
        pairs += sum(seen)
        read += b - (max(0, first - w + 1) if w else 0)
    rb = _row_bytes(NAMES[case["k"]], hd) + _row_bytes(NAMES[case["v"]], hd)
    return {"bytes": read * case["n_kv"] * rb + 2 * n_tok * case["n_head"] * hd * (4 if case["q"] == "f32" else 2),
            "flops": 4 * pairs * case["n_head"] * hd}


# ---- inputs ---------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantize(x, t):
    """Rows x [..., hd] as the cache holds them: fp16, or uint8 rows of codes and block scales."""
    if t == F16:
        return x.to(torch.float16)
    hd = x.shape[-1]
    b = x.reshape(-1, hd // 32, 32)
    if t == Q8_0:
        d = b.abs().amax(-1) / 127.0
        codes = torch.round(b / d.clamp_min(1e-30)[..., None]).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        d = torch.gather(b, -1, b.abs().argmax(-1, keepdim=True))[..., 0] / -8.0
        n = (b / torch.where(d == 0, torch.ones_like(d), d)[..., None] + 8.5).floor().clamp(0, 15).to(torch.uint8)
        codes = n[..., :16] | (n[..., 16:] << 4)
    out = torch.zeros(b.shape[0], _row_bytes(t, hd), dtype=torch.uint8, device="cuda")
    cb = hd if t == Q8_0 else hd // 2
    out[:, :cb] = codes.reshape(b.shape[0], cb)
    out[:, cb:cb + hd // 16] = d.to(torch.float16).view(torch.uint8).reshape(b.shape[0], hd // 16)
    return out.reshape(*x.shape[:-1], -1)


def _tables(g, kv, page, slack=2):
    """Page tables over a pool with a few free pages, in random order, and the pool's size."""
    need = [max(1, -(-n // page)) for n in kv]
    n_pages = sum(need) + slack
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    max_pages = max(need)
    start = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)[:, None]
    col = torch.arange(max_pages, device="cuda")[None, :]
    used = col < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[(start + col).clamp_max(n_pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    return table.contiguous(), n_pages


def _batch(g, case):
    q, kv = _lengths(case)
    table, n_pages = _tables(g, kv, case["page"])
    return {"q_start": _int32([sum(q[:i]) for i in range(len(q) + 1)]), "kv_len": _int32(kv), "table": table,
            "n_tok": sum(q), "max_q": max(q), "n_pages": n_pages}


def _kept(n, drop):
    """The positions that stay when a share of the middle of n is dropped: a kept head (1/16) and the newest ones."""
    head = n // 16
    cut = min(n - 1 - head, round(n * drop))
    return list(range(head)) + list(range(head + cut, n))


def _gather_lengths(case):
    n = case["n_seq"]
    return [round(case["kv_min"] + (i / max(1, n - 1)) * (case["kv_max"] - case["kv_min"])) for i in range(n)]


def _rope_table(n_pos, n_rot):
    i = torch.arange(n_rot // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * (500000.0 ** (-2.0 * i / n_rot))[None, :]
    return torch.stack([a.cos(), a.sin()], -1).reshape(n_pos, n_rot).to(torch.float32)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] in ("attn", "store"):
        s.update(_batch(g, case))
        shape = (1, s["n_pages"], s["n_kv"], s["page"], s["hd"])
        if case["op"] == "attn":
            s["K"], s["V"] = _quantize(randn(*shape), NAMES[s["k"]]), _quantize(randn(*shape), NAMES[s["v"]])
            s["Q"] = (1.5 * randn(s["n_tok"], s["n_head"], s["hd"])).to(TORCH[s["q"]])
            s["out"] = torch.empty_like(s["Q"])
            s["scale"] = 1.0 / math.sqrt(s["hd"])
        else:
            s["K"], s["V"] = randn(*shape).half(), randn(*shape).half()
            s["X"] = randn(s["n_tok"], s["n_head"] + 2 * s["n_kv"], s["hd"]).to(TORCH[s["x"]])
            s["out"] = torch.empty(s["n_tok"], s["n_head"], s["hd"], dtype=TORCH[s["q"]], device="cuda")
            s["rope"] = _rope_table(s["n_pos"], s["rot"])
            # positions of a prompt with images: time moves slowly, height and width run within a picture
            i = torch.arange(s["n_tok"], device="cuda")
            t = i % (s["n_pos"] // 2)
            pos = torch.stack([t, t // 3 + (i // 24) % 24, t // 3 + i % 24])[:s["axes"]] + int(
                torch.randint(0, 64, (1,), generator=g, device="cuda"))
            s["pos"] = pos.to(torch.int32).contiguous()
            half = s["rot"] // 2                       # sections of 1/4, 3/8, 3/8 of the pairs, as for 16, 24, 24 of 64
            cut = {1: [half], 2: [half // 2], 3: [half // 4, half // 4 + 3 * half // 8]}[s["axes"]]
            pair = torch.arange(half, device="cuda")
            s["axis"] = sum((pair >= c).to(torch.uint8) for c in cut).clamp_max(s["axes"] - 1).to(torch.uint8)
    elif case["op"] == "copy":
        shape = (s["n_layer"], s["n_pages"], s["n_kv"], s["page"], s["hd"])
        s["K"], s["V"] = randn(*shape).half(), randn(*shape).half()
        order = torch.randperm(s["n_pages"], generator=g, device="cuda")[:2 * s["n_copy"]].cpu()
        s["src"], s["dst"] = order[:s["n_copy"]].int().numpy(), order[s["n_copy"]:].int().numpy()
        s["src_dev"], s["dst_dev"] = order[:s["n_copy"]].cuda(), order[s["n_copy"]:].cuda()
    else:
        kv = _gather_lengths(case)
        kept = [_kept(n, s["drop"]) for n in kv]
        both, s["n_pages"] = _tables(g, kv + [len(k) for k in kept], s["page"])
        s["src_table"], s["dst_table"] = both[:len(kv)].contiguous(), both[len(kv):].contiguous()
        shape = (s["n_layer"], s["n_pages"], s["n_kv"], s["page"], s["hd"])
        s["K"], s["V"] = randn(*shape).half(), randn(*shape).half()
        s["keep"] = _int32([p for k in kept for p in k])
        s["keep_start"] = _int32([sum(len(k) for k in kept[:i]) for i in range(len(kept) + 1)])
        s["n_tok"] = len(s["keep"])
    if own:
        _handles(s)
    return s


# ---- the framework's operators --------------------------------------------------------------------------------
def _b2():
    import os
    import sys
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arkantos-ai-stack-suite_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import b2gguf
    return b2gguf


def _handles(s):
    """What a program keeps beside its tensors: the cache's and the step's descriptors and the attention's workspace."""
    b2 = _b2()
    s["b2"] = b2
    s["cache"] = b2.PageCache(s["K"].shape[0], s["n_pages"], s["page"], s["n_kv"], s["hd"], NAMES[s.get("k", "f16")],
                              NAMES[s.get("v", "f16")], k=s["K"].data_ptr(), v=s["V"].data_ptr())
    if s["op"] in ("attn", "store"):
        s["batch"] = b2.PageBatch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(),
                                  n_seq=s["n_seq"], max_pages=s["table"].shape[1], n_tok=s["n_tok"], max_q=s["max_q"])
    if s["op"] == "attn":
        size = b2.page_attn_workspace_bytes(s["cache"], s["batch"], s["n_head"], NAMES[s["q"]])
        s["workspace"] = b2.DeviceBuffer(size)
        s["workspace"].zero()


def _run_own(s):
    b2, stream = s["b2"], torch.cuda.current_stream().cuda_stream
    if s["op"] == "attn":
        b2.page_attn(s["cache"], 0, s["batch"], s["n_head"], s["Q"].data_ptr(), s["out"].data_ptr(), NAMES[s["q"]],
                     scale=s["scale"], window=s["window"], workspace=s["workspace"], stream=stream)
        return s["out"]
    if s["op"] == "store":
        b2.page_rope_store(s["cache"], 0, s["batch"], s["n_head"], s["X"].data_ptr(), NAMES[s["x"]],
                           s["out"].data_ptr(), NAMES[s["q"]], s["pos"].data_ptr(), s["axes"], s["axis"].data_ptr(),
                           s["rope"].data_ptr(), s["n_pos"], s["rot"], s["style"], stream=stream)
        return s["out"], s["K"], s["V"]
    if s["op"] == "copy":
        b2.page_copy(s["cache"], s["src"], s["dst"], stream=stream)
    else:
        b2.page_gather(s["cache"], s["n_seq"], s["keep_start"].data_ptr(), s["keep"].data_ptr(), s["n_tok"],
                       s["src_table"].data_ptr(), s["dst_table"].data_ptr(), s["src_table"].shape[1], stream=stream)
    return s["K"], s["V"]


# ---- the plain form -------------------------------------------------------------------------------------------
def _values(rows, t, hd):
    """Cache rows as fp32 values."""
    if t == F16:
        return rows.float()
    cb = hd if t == Q8_0 else hd // 2
    d = rows[..., cb:cb + hd // 16].contiguous().view(torch.float16).float()
    if t == Q8_0:
        c = rows[..., :cb].contiguous().view(torch.int8).float()
    else:
        n = rows[..., :cb].reshape(*rows.shape[:-1], hd // 32, 16)
        c = torch.cat([n & 15, n >> 4], -1).reshape(*rows.shape[:-1], hd).float() - 8.0
    return (c.reshape(*c.shape[:-1], hd // 32, 32) * d[..., None]).reshape(*c.shape)


def _tokens(s):
    """Sequence and position of every token."""
    i = torch.arange(s["n_tok"], device="cuda")
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:].contiguous(), i, right=True)
    return seq, i - start[seq + 1] + s["kv_len"].long()[seq]


def _attn_plain(s):
    hd, n_kv, n_seq, group = s["hd"], s["n_kv"], s["n_seq"], s["n_head"] // s["n_kv"]
    table, kv = s["table"].long(), s["kv_len"].long()
    t = torch.arange(table.shape[1] * s["page"], device="cuda")

    def rows(pool, kind):     # [n_seq][n_kv][positions][hd]
        return _values(pool[0][table], kind, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, t.numel(), hd)

    start = s["q_start"].long()
    length = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device="cuda")
    tok = (start[:-1, None] + i[None, :]).clamp_max(s["n_tok"] - 1)
    p = (kv - length)[:, None] + i[None, :]                                   # [n_seq][max_q]
    see = (t <= p[..., None]) & (t < kv[:, None, None])
    if s["window"]:
        see = see & (t > p[..., None] - s["window"])
    q = s["Q"].float()[tok].reshape(n_seq, s["max_q"], n_kv, group, hd).permute(0, 2, 3, 1, 4)
    k, v = rows(s["K"], NAMES[s["k"]]), rows(s["V"], NAMES[s["v"]])
    e = torch.matmul(q.reshape(n_seq, n_kv, -1, hd), k.transpose(-1, -2)).reshape(n_seq, n_kv, group, s["max_q"], -1)
    e = (e * s["scale"]).masked_fill_(~see[:, None, None], -math.inf)
    top = e.amax(-1, keepdim=True)
    e = e.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(n_seq, n_kv, -1, t.numel()), v).reshape(n_seq, n_kv, group, s["max_q"], hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4)
    seq, pos = _tokens(s)
    return o.reshape(n_seq, s["max_q"], s["n_head"], hd)[seq, pos - (kv - length)[seq]].to(s["Q"].dtype)


def _rotate(x, s, table):
    """The first `rot` values of every head rotated, pair j by the angle of its axis' position."""
    half = s["rot"] // 2
    j = torch.arange(half, device="cuda")
    cs = table.reshape(s["n_pos"], half, 2)[s["pos"].long()[s["axis"].long()].T, j]      # [n_tok][half][2]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    r, rest = x[..., :s["rot"]], x[..., s["rot"]:]
    a, b = (r[..., :half], r[..., half:]) if s["style"] else (r[..., 0::2], r[..., 1::2])
    y = torch.cat([a * c - b * n, a * n + b * c], -1) if s["style"] else \
        torch.stack([a * c - b * n, a * n + b * c], -1).reshape(r.shape)
    return torch.cat([y, rest], -1)


def _store_plain(s):
    h, n = s["n_head"], s["n_kv"]
    seq, p = _tokens(s)
    x = s["X"].float()
    page, slot = s["table"].long()[seq, p // s["page"]], p % s["page"]
    s["K"][0, page, :, slot] = _rotate(x[:, h:h + n], s, s["rope"]).half()
    s["V"][0, page, :, slot] = x[:, h + n:].half()
    return _rotate(x[:, :h], s, s["rope"]).to(TORCH[s["q"]]), s["K"], s["V"]


def _copy_plain(s):
    s["K"][:, s["dst_dev"]] = s["K"][:, s["src_dev"]]
    s["V"][:, s["dst_dev"]] = s["V"][:, s["src_dev"]]
    return s["K"], s["V"]


def _gather_plain(s):
    i = torch.arange(s["n_tok"], device="cuda")
    start, keep = s["keep_start"].long(), s["keep"].long()
    seq = torch.searchsorted(start[1:].contiguous(), i, right=True)
    to = i - start[seq]
    src, dst = s["src_table"].long()[seq, keep // s["page"]], s["dst_table"].long()[seq, to // s["page"]]
    s["K"][:, dst, :, to % s["page"]] = s["K"][:, src, :, keep % s["page"]]
    s["V"][:, dst, :, to % s["page"]] = s["V"][:, src, :, keep % s["page"]]
    return s["K"], s["V"]


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _attn_plain, "store": _store_plain, "copy": _copy_plain, "gather": _gather_plain}[state["op"]](state)


# ---- in 64 bits -----------------------------------------------------------------------------------------------
def _cache_row_64(rows, t, hd):
    """One sequence's rows as doubles, value by value from the storage's definition."""
    if t == F16:
        return rows.double()
    j = torch.arange(hd, device="cuda")
    if t == Q8_0:
        code = rows[..., :hd].view(torch.int8).double()
        at = hd + 2 * (j // 32)
    else:
        byte = rows[..., (j // 32) * 16 + j % 16].int()
        code = torch.where(j % 32 < 16, byte & 15, byte >> 4).double() - 8
        at = hd // 2 + 2 * (j // 32)
    scale = torch.stack([rows[..., at], rows[..., at + 1]], -1).contiguous().view(torch.float16)[..., 0].double()
    return code * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        K, V = s["K"].double(), s["V"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            K[:, b], V[:, b] = s["K"][:, a].double(), s["V"][:, a].double()
        return K, V
    if case["op"] == "gather":
        K, V, page, first = s["K"].double(), s["V"].double(), s["page"], s["keep_start"].tolist()
        old, new, keep = s["src_table"].tolist(), s["dst_table"].tolist(), s["keep"].tolist()
        for b in range(s["n_seq"]):
            for i, p in enumerate(keep[first[b]:first[b + 1]]):
                for to, pool in ((K, s["K"]), (V, s["V"])):
                    to[:, new[b][i // page], :, i % page] = pool[:, old[b][p // page], :, p % page].double()
        return K, V
    start, kv, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].long()
    if case["op"] == "store":
        x, h, n = s["X"].double(), s["n_head"], s["n_kv"]
        K, V = s["K"].double(), s["V"].double()
        j = torch.arange(s["rot"] // 2, device="cuda")
        # the table is an input: its rounded values are the angles' cosines and sines here
        c = s["rope"].double()[:, 0::2][s["pos"].long()[s["axis"].long()], j[:, None]].T[:, None]
        d = s["rope"].double()[:, 1::2][s["pos"].long()[s["axis"].long()], j[:, None]].T[:, None]
        i0, i1 = (j, j + s["rot"] // 2) if s["style"] else (2 * j, 2 * j + 1)
        y = x.clone()
        y[:, :h + n, i0] = x[:, :h + n, i0] * c - x[:, :h + n, i1] * d
        y[:, :h + n, i1] = x[:, :h + n, i0] * d + x[:, :h + n, i1] * c
        for b in range(s["n_seq"]):
            a, e = start[b], start[b + 1]
            p = torch.arange(kv[b] - (e - a), kv[b], device="cuda")
            K[0, table[b, p // s["page"]], :, p % s["page"]] = y[a:e, h:h + n]
            V[0, table[b, p // s["page"]], :, p % s["page"]] = y[a:e, h + n:]
        return y[:, :h], K, V
    out = torch.zeros(s["Q"].shape, dtype=torch.float64, device="cuda")
    group = s["n_head"] // s["n_kv"]
    for b in range(s["n_seq"]):
        a, e = start[b], start[b + 1]
        t = torch.arange(kv[b], device="cuda")
        p = torch.arange(kv[b] - (e - a), kv[b], device="cuda")[:, None]
        hide = t[None] > p
        if s["window"]:
            hide |= p - t[None] >= s["window"]
        pages, slots = table[b, t // s["page"]], t % s["page"]
        for m in range(s["n_kv"]):
            k = _cache_row_64(s["K"][0, pages, m, slots], NAMES[s["k"]], s["hd"])
            v = _cache_row_64(s["V"][0, pages, m, slots], NAMES[s["v"]], s["hd"])
            for u in range(m * group, (m + 1) * group):
                z = (s["Q"][a:e, u].double() @ k.T * s["scale"]).masked_fill(hide, -math.inf)
                out[a:e, u] = torch.softmax(z, -1) @ v
    return out
