"""The dense attention block of a serving step, operator by operator: a projection's result with the low-rank adapters of
many requests added to it, keys and values rotated into a paged cache, and attention of one new token over that cache.

A case is a dict of plain values; `kind` says which operator it goes through:
  append    ops.kv_rope_append   new rows (prompts or single tokens) -> cache slots, rotated; queries rotated beside them
  attend    ops.paged_decode     one new token a sequence over its slots
  adapters  ops.adapter_add      out = y + scale[i] (x A[i]) B[i], i = the adapter of the row's request

Where `own` is false, `run` computes the same in elementary torch operations.
"""
import math
from types import SimpleNamespace

import torch

own = False  # whether run() makes the package's calls

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def _append(batch, heads, kv_heads, new, ctx, dtype, cache="same", page=16, head_dim=128, rot_dim=0, layout="half",
            offset=0):
    """new, ctx: (lowest, highest) number of new rows and of rows already there, per sequence; cache "same" holds the rows'
    type, "int8" bytes with one f16 scale per row; page: slots of a page; offset: added to the positions (up to)."""
    return dict(kind="append", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot_dim=rot_dim or head_dim,
                layout=layout, dtype=dtype, cache=cache, new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                page=page, offset=offset)


def _attend(batch, heads, kv_heads, length, dtype, cache="same", page=16, head_dim=128, window=0, lse=False):
    return dict(kind="attend", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, cache=cache,
                len_lo=length[0], len_hi=length[1], page=page, window=window, lse=lse)


def _adapters(batch, rows, n_in, n_out, rank, count, dtype, idle=0.0):
    """rows: (lowest, highest) rows of a request; count: adapters in memory, of which each request names one; idle: the
    share of requests without one."""
    return dict(kind="adapters", batch=batch, rows_lo=rows[0], rows_hi=rows[1], n_in=n_in, n_out=n_out, rank=rank,
                count=count, dtype=dtype, idle=idle)


def listed():
    return [
        # one user's next token, 7B shape (latency)
        dict(name="append_7b_b1", **_append(1, 32, 32, (1, 1), (2048, 2048), "f16")),
        # a server's step with grouped heads, in bf16
        dict(name="append_gqa_b64", **_append(64, 32, 8, (1, 1), (100, 500), "bf16")),
        # image prompts of different lengths, 13B shape
        dict(name="append_13b_prompts", **_append(8, 40, 40, (700, 2880), (0, 0), "f16", page=64)),
        # the next chunk of long prompts into a cache of bytes, far positions
        dict(name="append_chunk_int8", **_append(3, 32, 8, (1500, 2048), (0, 100), "bf16", cache="int8", page=64,
                                                 offset=100000)),
        # one user's chat turn, 7B shape (latency)
        dict(name="attend_7b_b1_s2048", **_attend(1, 32, 32, (2048, 2048), "f16")),
        # a server's batch, 13B shape, every head with keys of its own
        dict(name="attend_13b_b16_s4096", **_attend(16, 40, 40, (4096, 4096), "f16", page=64)),
        # grouped heads, prompts of very different lengths
        dict(name="attend_gqa_b32_ragged8k", **_attend(32, 32, 8, (300, 8192), "bf16", lse=True)),
        # long contexts in a cache of bytes
        dict(name="attend_gqa_b8_int8_32k", **_attend(8, 32, 8, (9000, 32768), "bf16", cache="int8", page=64)),
        # a sliding window, small heads
        dict(name="attend_window_b48_d64", **_attend(48, 32, 8, (20, 12000), "f16", head_dim=64, window=4096, lse=True)),
        # a few requests' adapters at the attention's output projection
        dict(name="adapters_b4", **_adapters(4, (1, 1), 4096, 4096, 16, 8, "f16")),
        # a server's step at the joined projection of queries, keys and values
        dict(name="adapters_b64_qkv", **_adapters(64, (1, 1), 5120, 15360, 32, 48, "bf16", idle=0.1)),
        # prompts at the gate's projection
        dict(name="adapters_prompts", **_adapters(5, (300, 2048), 4096, 11008, 64, 8, "f16")),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "adapters"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv = rng.choice([(32, 32), (40, 40), (32, 8), (32, 4), (8, 1), (40, 8), (28, 4), (16, 1), (48, 2), (8, 8)])
    if kind == "append":
        head_dim = rng.choice([64, 96, 128, 128, 128, 256])
        step = rng.random() < 0.5
        batch = _log_int(rng, 1, 128) if step else _log_int(rng, 1, 12)
        hi = 1 if step else _log_int(rng, 2, max(2, min(4096, 20_000_000 // (batch * (heads + 2 * kv) * head_dim // 8))))
        ctx = _log_int(rng, 1, 600)
        return _append(batch, heads, kv, (rng.choice([1, hi, max(1, hi // 3)]), hi), (rng.choice([0, ctx]), ctx), dtype,
                       rng.choice(["same", "same", "int8"]), rng.choice([1, 16, 64, 256]), head_dim,
                       rng.choice([0, 0, 0, head_dim // 2]), rng.choice(["half", "half", "interleaved"]),
                       rng.choice([0, 0, 5000, 120000]))
    if kind == "attend":
        head_dim = rng.choice([64, 96, 128, 128, 128, 256])
        hi = _log_int(rng, 1, 60000)
        batch = _log_int(rng, 1, max(1, min(128, 290_000_000 // (hi * max(kv, heads // 3) * head_dim))))
        return _attend(batch, heads, kv, (rng.choice([hi, max(1, hi // 3), 1]), hi), dtype, rng.choice(["same", "same", "int8"]),
                       rng.choice([1, 16, 64, 256]), head_dim, rng.choice([0, 0, 0, _log_int(rng, 1, 5000)]), rng.random() < 0.5)
    n_in, n_out = rng.choice([(4096, 4096), (4096, 11008), (11008, 4096), (5120, 5120), (5120, 15360), (1000, 2040), (4096, 8192)])
    rank = rng.choice([4, 8, 16, 16, 32, 64, 100, 128])
    step = rng.random() < 0.6
    batch = _log_int(rng, 1, 128) if step else _log_int(rng, 1, 12)
    hi = 1 if step else _log_int(rng, 2, max(2, min(2048, 90_000_000 // (batch * (n_in + 2 * n_out)))))
    count = rng.choice([n for n in (1, 4, 16, 40) if step or n * rank <= 512])
    return _adapters(batch, (rng.choice([hi, max(1, hi // 4)]), hi), n_in, n_out, rank, count, dtype,
                     rng.choice([0.0, 0.0, 0.3]))


# ------------------------------------------------------------------ inputs

def _counts(lo, hi, n, seed=None):
    """n whole numbers in [lo, hi], the highest among them; a seed puts them in another order, their sum stays."""
    c = torch.randint(lo, hi + 1, (n,), generator=torch.Generator().manual_seed(lo * 7919 + hi))
    c[0] = hi
    return c if seed is None else c[torch.randperm(n, generator=torch.Generator().manual_seed(seed * 7919 + 3))]


def _table(width, batch, page, seed):
    """Token slots handed out page by page in a shuffled order: ([batch, width] table, number of slots)."""
    per = (width + page - 1) // page
    perm = torch.randperm(batch * per, generator=torch.Generator().manual_seed(seed * 31 + 5))
    table = (perm[:, None] * page + torch.arange(page)[None, :]).reshape(batch, per * page)[:, :width]
    return table.to(torch.int32).contiguous().to(DEV), batch * per * page


def _state(lens, table):
    """What a server keeps of its batch: lengths, and the rows of the page table that its sequences have."""
    n = len(lens)
    return SimpleNamespace(batch_size=n, max_len_in_batch=int(lens.max()), b_seq_len=lens.to(torch.int32).to(DEV),
                           b_req_idx=torch.arange(n, dtype=torch.int32, device=DEV),
                           req_manager=SimpleNamespace(req_to_token_indexs=table))


def _starts(counts):
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to(DEV)


def _quantize(x):
    """Per row: scale = max|x| / 127 as f16 (1 for a zero row), int8 against the stored scale."""
    amax = x.abs().amax(dim=-1)
    scale = torch.where(amax == 0, torch.ones_like(amax), amax / 127.0).half()
    return torch.clamp(torch.round(x / scale.float().unsqueeze(-1)), -128, 127).to(torch.int8), scale


def _rows(gen, slots, heads, dim, dtype, cache):
    """A cache's rows [slots, heads, dim] (and scales [slots, heads] or None) with values in every slot."""
    if cache != "int8":
        return torch.randn(slots, heads, dim, generator=gen, device=DEV, dtype=dtype), None
    store = torch.empty(slots, heads, dim, dtype=torch.int8, device=DEV)
    scale = torch.empty(slots, heads, dtype=torch.float16, device=DEV)
    for at in range(0, slots, 65536):  # (in pieces: a long cache in f32 would not fit three times over)
        piece = slice(at, min(slots, at + 65536))
        store[piece], scale[piece] = _quantize(torch.randn(piece.stop - at, heads, dim, generator=gen, device=DEV))
    return store, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    st = {"case": case}

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    if case["kind"] == "append":
        B, H, K, D = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim"))
        new, ctx = _counts(case["new_lo"], case["new_hi"], B, seed), _counts(case["ctx_lo"], case["ctx_hi"], B, seed + 1)
        table, slots = _table(case["new_hi"] + case["ctx_hi"], B, case["page"], seed)
        st["state"] = _state(ctx, table)
        st["cu_new"] = None if case["new_hi"] == 1 else _starts(new)
        n = int(new.sum())
        # the column slices of one joined projection
        qkv = randn(n, (H + 2 * K) * D)
        st["q"] = qkv[:, :H * D].unflatten(1, (H, D))
        st["k"] = qkv[:, H * D:(H + K) * D].unflatten(1, (K, D))
        st["v"] = qkv[:, (H + K) * D:].unflatten(1, (K, D))
        st["inv_freq"] = (10000.0 ** (-torch.arange(0, case["rot_dim"], 2, dtype=torch.float64) / case["rot_dim"])).float().to(DEV)
        g = torch.Generator().manual_seed(seed * 13 + 1)
        st["pos_offset"] = torch.randint(0, case["offset"] + 1, (B,), generator=g, dtype=torch.int32).to(DEV) if case["offset"] else None
        st["ck"], st["ks"] = _rows(gen, slots, K, D, dtype, case["cache"])
        st["cv"], st["vs"] = _rows(gen, slots, K, D, dtype, case["cache"])
    elif case["kind"] == "attend":
        B, H, K, D = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim"))
        table, slots = _table(case["len_hi"], B, case["page"], seed)
        st["state"] = _state(_counts(case["len_lo"], case["len_hi"], B, seed), table)
        st["q"] = randn(B, H, D)
        st["ck"], st["ks"] = _rows(gen, slots, K, D, dtype, case["cache"])
        st["cv"], st["vs"] = _rows(gen, slots, K, D, dtype, case["cache"])
    else:
        B, n_in, n_out, r = (case[k] for k in ("batch", "n_in", "n_out", "rank"))
        rows = _counts(case["rows_lo"], case["rows_hi"], B, seed)
        st["cu_new"] = None if case["rows_hi"] == 1 else _starts(rows)
        n = int(rows.sum())
        st["x"], st["y"] = randn(n, n_in), randn(n, n_out)
        # a trained adapter's first factor keeps the spread of its initialisation, the second one has grown from zero
        st["a"] = randn(case["count"], n_in, r, scale=1 / math.sqrt(n_in))
        st["b"] = randn(case["count"], r, n_out, scale=0.3 / math.sqrt(r))
        g = torch.Generator().manual_seed(seed * 17 + 2)
        pick = torch.randint(0, case["count"], (B,), generator=g, dtype=torch.int32)
        idle = torch.rand(B, generator=g) < case["idle"]
        idle[0] = False
        st["adapter"] = torch.where(idle, torch.full_like(pick, -1), pick).to(DEV)
        st["scale"] = (torch.rand(case["count"], generator=g) + 0.5).to(DEV)
    return st


# ------------------------------------------------------------------ the plain forms

def _sequence_of(cu, n):
    """Which sequence each of the n packed rows belongs to, and the row's place in it."""
    row = torch.arange(n, device=DEV)
    b = torch.searchsorted(cu[1:].long(), row, right=True)
    return b, row - cu.long()[b]


def _rotate(x, cos, sin, rot, layout):
    """x [n, heads, D] in f32, cos and sin [n, 1, rot / 2]: the first rot dims rotated in pairs."""
    y = x.float()
    if layout == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], dim=-1)


def _store(cache, scale, slot, rows):
    if scale is None:
        cache[slot] = rows.to(cache.dtype)
    else:
        cache[slot], scale[slot] = _quantize(rows)


def _plain_append(st):
    case, s = st["case"], st["state"]
    n = st["q"].shape[0]
    if st["cu_new"] is None:
        b, i = torch.arange(n, device=DEV), 0
    else:
        b, i = _sequence_of(st["cu_new"], n)
    at = s.b_seq_len.long()[b] + i
    slot = s.req_manager.req_to_token_indexs[s.b_req_idx.long()[b], at].long()
    place = at if st["pos_offset"] is None else at + st["pos_offset"].long()[b]
    angle = place.double()[:, None, None] * st["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    rot = case["rot_dim"]
    q = _rotate(st["q"], cos, sin, rot, case["layout"]).to(st["q"].dtype)
    _store(st["ck"], st["ks"], slot, _rotate(st["k"], cos, sin, rot, case["layout"]))
    _store(st["cv"], st["vs"], slot, st["v"].float())
    return q


def _plain_attend(st):
    case, s = st["case"], st["state"]
    q = st["q"].float()
    B, H, D = q.shape
    S, K = case["len_hi"], case["kv_heads"]
    table = s.req_manager.req_to_token_indexs[s.b_req_idx.long(), :S].long()
    lens = s.b_seq_len.long()[:, None]
    place = torch.arange(S, device=DEV)[None, :]
    seen = place < lens
    if case["window"]:
        seen = seen & (place >= lens - case["window"])
    k = st["ck"][table].float()  # [B, S, K, D]
    if st["ks"] is not None:
        k = k * st["ks"][table].float().unsqueeze(-1)
    z = torch.einsum("bkgd,bskd->bkgs", q.view(B, K, H // K, D), k) / math.sqrt(D)
    del k
    z = z.masked_fill(~seen[:, None, None, :], -math.inf)
    top = z.amax(dim=-1, keepdim=True)
    w = (z - top).exp()
    total = w.sum(dim=-1, keepdim=True)
    v = st["cv"][table].float()
    if st["vs"] is not None:
        v = v * st["vs"][table].float().unsqueeze(-1)
    o = torch.einsum("bkgs,bskd->bkgd", w, v) / total
    return o.reshape(B, H, D).to(st["q"].dtype), (top + total.log()).reshape(B, H)


def _plain_adapters(st):
    x, a, b = st["x"].float(), st["a"].float(), st["b"].float()
    n, (count, n_in, r), n_out = x.shape[0], a.shape, b.shape[2]
    of_row = st["adapter"].long()
    if st["cu_new"] is not None:
        of_row = of_row[_sequence_of(st["cu_new"], n)[0]]
    # every adapter's product, all but the row's own one set to zero
    h = (x @ a.permute(1, 0, 2).reshape(n_in, count * r)).view(n, count, r)
    mine = of_row[:, None] == torch.arange(count, device=DEV)[None, :]
    h = h * torch.where(mine, st["scale"][None, :], torch.zeros((), device=DEV)).unsqueeze(-1)
    return (st["y"].float() + h.view(n, count * r) @ b.reshape(count * r, n_out)).to(st["y"].dtype)


def _ops():
    from wsvd_b200 import ops

    return ops


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "append":
        if own:
            q = _ops().kv_rope_append(st["k"], st["v"], st["state"], st["ck"], st["cv"], st["inv_freq"], cache_k_scale=st["ks"],
                                      cache_v_scale=st["vs"], q=st["q"], cu_new=st["cu_new"], pos_offset=st["pos_offset"],
                                      rope_layout=case["layout"])
        else:
            q = _plain_append(st)
        if st["ks"] is None:
            return {"q": q, "k": st["ck"], "v": st["cv"]}
        # the values that the bytes stand for
        return {"q": q, "k": st["ck"] * st["ks"].unsqueeze(-1), "v": st["cv"] * st["vs"].unsqueeze(-1), "ks": st["ks"], "vs": st["vs"]}
    if kind == "attend":
        if own:
            got = _ops().paged_decode(st["q"], st["state"], st["ck"], st["cv"], st["ks"], st["vs"], window=case["window"],
                                      return_lse=case["lse"])
            return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}
        out, lse = _plain_attend(st)
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    if own:
        return _ops().adapter_add(st["y"], st["x"], st["a"], st["b"], st["adapter"], scale=st["scale"], cu_new=st["cu_new"])
    return _plain_adapters(st)


# ------------------------------------------------------------------ what a pass cannot do without

def _distinct(case):
    """Expected number of different adapters that the requests name."""
    n = 1 + (case["batch"] - 1) * (1 - case["idle"])
    return case["count"] * (1 - (1 - 1 / case["count"]) ** n)


def work(case):
    if case["kind"] == "adapters":
        rows = int(_counts(case["rows_lo"], case["rows_hi"], case["batch"]).sum())
        n_in, n_out, r = case["n_in"], case["n_out"], case["rank"]
        busy = rows * (1 - case["idle"])
        return {"bytes": 2 * (_distinct(case) * r * (n_in + n_out) + busy * n_in + 2 * rows * n_out), "flops": 2 * busy * r * (n_in + n_out)}
    B, H, K, D = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim"))
    held = D + 2 if case["cache"] == "int8" else 2 * D  # bytes of a cached row
    if case["kind"] == "append":
        rows = int(_counts(case["new_lo"], case["new_hi"], B).sum())
        return {"bytes": rows * (2 * (2 * H + 2 * K) * D + 2 * K * held + 4), "flops": rows * (H + K) * 3 * case["rot_dim"]}
    lens = _counts(case["len_lo"], case["len_hi"], B)
    tokens = int((lens.clamp(max=case["window"]) if case["window"] else lens).sum())
    return {"bytes": tokens * (2 * K * held + 4) + 4 * B * H * D, "flops": 4 * tokens * H * D}


# ------------------------------------------------------------------ the same in 64 bits

def _turn64(x, place, inv_freq, rot, layout):
    """Each pair of x [heads, n, D] as a complex number times e^(i angle)."""
    ang = torch.outer(place.double(), inv_freq.double())
    turn = torch.complex(ang.cos(), ang.sin())
    x = x.double()
    head = x[..., :rot]
    pairs = torch.stack([head[..., :rot // 2], head[..., rot // 2:]], -1) if layout == "half" else head.unflatten(-1, (-1, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = torch.cat([z[..., 0], z[..., 1]], -1) if layout == "half" else z.flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _held64(rows):
    """What an int8 cache holds of rows in 64 bits, and the scales."""
    amax = rows.abs().amax(dim=-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 127, torch.ones_like(amax)).half().double()
    return (rows / scale).round().clamp(-128, 127) * scale, scale.squeeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        s, B = st["state"], case["batch"]
        n = st["q"].shape[0]
        cu = list(range(n + 1)) if st["cu_new"] is None else st["cu_new"].tolist()
        q = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
        out = {"q": q}
        for name, cache, scale in (("k", st["ck"], st["ks"]), ("v", st["cv"], st["vs"])):
            out[name] = cache.double() if scale is None else cache.double() * scale.double()[..., None]
            if scale is not None:
                out[name + "s"] = scale.double()
        for b in range(B):
            rows = slice(cu[b], cu[b + 1])
            at = int(s.b_seq_len[b]) + torch.arange(cu[b + 1] - cu[b], device=DEV)
            slot = s.req_manager.req_to_token_indexs[b].long()[at]
            place = at + (0 if st["pos_offset"] is None else int(st["pos_offset"][b]))

            def turn(x):
                return _turn64(x[rows].transpose(0, 1), place, st["inv_freq"], case["rot_dim"], case["layout"]).transpose(0, 1)

            q[rows] = turn(st["q"])
            for name, x in (("k", turn(st["k"])), ("v", st["v"][rows].double())):
                if st["ks"] is None:
                    out[name][slot] = x
                else:
                    out[name][slot], out[name + "s"][slot] = _held64(x)
        return out
    if case["kind"] == "attend":
        s, K, D = st["state"], case["kv_heads"], case["head_dim"]
        out, lse = [], []
        for b, n in enumerate(s.b_seq_len.tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            slot = s.req_manager.req_to_token_indexs[b, first:n].long()
            k, v = st["ck"][slot].double(), st["cv"][slot].double()
            if st["ks"] is not None:
                k, v = k * st["ks"][slot].double()[..., None], v * st["vs"][slot].double()[..., None]
            z = st["q"][b].double().view(K, -1, D) @ k.permute(1, 2, 0) / math.sqrt(D)
            out.append((torch.softmax(z, dim=-1) @ v.transpose(0, 1)).reshape(-1, D))
            lse.append(torch.logsumexp(z, dim=-1).reshape(-1))
        return {"out": torch.stack(out), "lse": torch.stack(lse)} if case["lse"] else {"out": torch.stack(out)}
    n = st["x"].shape[0]
    cu = list(range(n + 1)) if st["cu_new"] is None else st["cu_new"].tolist()
    out = st["y"].double()
    for b, i in enumerate(st["adapter"].tolist()):
        if i >= 0:
            rows = slice(cu[b], cu[b + 1])
            out[rows] += float(st["scale"][i]) * ((st["x"][rows].double() @ st["a"][i].double()) @ st["b"][i].double())
    return out
