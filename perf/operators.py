"""Cases that time the serving operators: the paged cache's append with its position
rotation, attention over packed prompts with grouped heads, and attention of single new
tokens over the paged cache.

A case is a dict of plain values.  Lengths follow from the case alone (`mix` seeds them);
values, page order and histories' contents follow from the seed.  `own` selects the
framework's kernels; without it `run` computes the same results from elementary torch
operations in f32, rounded once at the end.
"""
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_PREFIX = 5           # camera + register tokens of a frame, which carry no rotation
_FRAME = 1374         # tokens of a 518 x 518 frame: 37 x 37 patches + the prefix
_SPARE_PAGES = 7      # pages of the pool that belong to no sequence
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        from headshot_b200.engine import GpuContext

        _ctx = GpuContext(torch.cuda.current_device())
    return _ctx


# ------------------------------------------------------------------ cases --


def _append(name, dtype, heads, kv_heads, dim, page, seqs, shortest, longest, history, rope, mix):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "seqs": seqs, "shortest": shortest, "longest": longest, "history": history, "rope": rope,
            "mix": mix}


def _prompt(name, dtype, heads, kv_heads, dim, seqs, shortest, longest, history, causal, mix):
    return {"name": name, "op": "prompt", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "seqs": seqs, "shortest": shortest, "longest": longest, "history": history, "causal": causal, "mix": mix}


def _token(name, dtype, heads, kv_heads, dim, page, seqs, shortest, longest, mix):
    return {"name": name, "op": "token", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "seqs": seqs, "shortest": shortest, "longest": longest, "mix": mix}


def listed():
    return [
        # One stream generating: its newest token goes into the cache.  Launch latency.
        _append("append_one_token", "bf16", 32, 8, 128, 16, 1, 1, 1, 4096, "text", 1),
        # A batch of camera streams, one new token each, frame positions.
        _append("append_batch", "f16", 16, 16, 64, 32, 96, 1, 1, 2000, "frames", 2),
        # Prompts of very different lengths admitted together, some onto a history.
        _append("append_prompts", "bf16", 32, 8, 128, 64, 24, 1, 2501, 700, "text", 3),
        # One very long prompt filling an empty cache.
        _append("append_long_prompt", "bf16", 32, 8, 128, 64, 1, 32768, 32768, 0, "text", 4),
        # The shortest prompt that is still a prompt: latency.
        _prompt("prompt_short", "f16", 16, 16, 64, 1, 17, 17, 0, True, 5),
        # Images of different sizes in one call, every token of an image with every other.
        _prompt("prompt_images", "f16", 16, 16, 64, 12, 261, 1374, 0, False, 6),
        # Prompts packed without padding, some behind keys that are there already.
        _prompt("prompt_packed", "bf16", 32, 8, 128, 20, 5, 4001, 900, True, 7),
        # A long document, grouped heads.
        _prompt("prompt_long", "bf16", 32, 8, 128, 1, 16384, 16384, 0, True, 8),
        # 32 frames of 1374 tokens as one causal stream.
        _prompt("prompt_stream", "bf16", 16, 16, 64, 1, 43968, 43968, 0, True, 9),
        # One stream's next token over a long cache: work only when the cache is split.
        _token("token_one", "bf16", 32, 8, 128, 16, 1, 8191, 8191, 10),
        # A serving batch, from sequences just begun to long ones.
        _token("token_batch", "bf16", 32, 8, 128, 64, 128, 1, 16001, 11),
        # 200 frames of 1374 tokens in the cache of a single stream, ungrouped heads.
        _token("token_stream", "f16", 16, 16, 64, 128, 1, 274800, 274800, 12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_SHAPES = [(16, 16, 64), (16, 4, 64), (32, 8, 64), (8, 1, 64), (20, 4, 64), (12, 4, 64), (16, 16, 128), (32, 8, 128),
           (28, 4, 128), (40, 8, 128), (8, 8, 128), (16, 1, 128)]
_PAGES = [8, 16, 24, 32, 64, 100, 128, 256]


def draw(rng):
    op = rng.choice(["append", "prompt", "token"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv_heads, dim = rng.choice(_SHAPES)
    mix = rng.randrange(1 << 30)
    if op == "append":
        total = _log_int(rng, 1, 24000)
        seqs = _log_int(rng, 1, min(total, 200))
        longest = max(1, total // seqs)
        rope = rng.choice(["text", "frames"]) if dim == 64 else "text"
        c = _append("", dtype, heads, kv_heads, dim, rng.choice(_PAGES), seqs, max(1, longest // rng.choice([1, 5, 40])),
                    longest, rng.choice([0, _log_int(rng, 1, 1500)]), rope, mix)
    elif op == "prompt":
        longest = _log_int(rng, 1, 12000)
        seqs = _log_int(rng, 1, max(1, min(64, 12000 // longest)))
        c = _prompt("", dtype, heads, kv_heads, dim, seqs, max(1, longest // rng.choice([1, 5, 40])), longest,
                    rng.choice([0, 0, _log_int(rng, 1, 2000)]), rng.random() < 0.75, mix)
    else:
        keys = (1 << 30) // (4 * kv_heads * dim)  # the cache stays within about 1 GB
        seqs = _log_int(rng, 1, 160)
        longest = _log_int(rng, 1, max(1, keys // seqs))
        c = _token("", dtype, heads, kv_heads, dim, rng.choice(_PAGES), seqs,
                   max(1, longest // rng.choice([1, 10, 1000])), longest, mix)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, tokens before them) of each sequence."""
    rng = random.Random(case["mix"])
    new = [_log_int(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    new[-1] = case["longest"]
    if len(new) > 1:
        new[0] = case["shortest"]
    h = case.get("history", 0)
    old = [_log_int(rng, 1, h + 1) - 1 if h else 0 for _ in new]
    if h:
        old[-1] = h
    return new, old


def work(case):
    new, old = _lengths(case)
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    n = sum(new)
    if case["op"] == "append":
        rows = len({r for a, b in zip(new, old) for r in _table_rows(case, b, a)})
        return {"bytes": 2 * d * n * (2 * hq + 2 * hk + 3 * hk) + rows * d * 8, "flops": n * d * 3 * (hq + hk)}
    if case["op"] == "prompt":
        keys = n + sum(old)
        pairs = sum(a * b + a * (a + 1) // 2 if case["causal"] else a * (a + b) for a, b in zip(new, old))
        return {"bytes": 2 * d * (2 * n * hq + 2 * keys * hk), "flops": 4 * d * hq * pairs}
    return {"bytes": 2 * d * (2 * n * hk + 2 * case["seqs"] * hq), "flops": 4 * d * hq * n}


# ----------------------------------------------------------------- inputs --


def _table_rows(case, start, count):
    """Rotation-table rows of positions [start, start + count), without the prefix tokens."""
    if case["rope"] == "text":
        return range(start, start + count)
    rows = ((p % _FRAME) - _PREFIX for p in range(start, start + min(count, _FRAME)))
    return (r for r in rows if r >= 0)


def _tables(case, rows, dev):
    d = case["dim"]
    if case["rope"] == "text":
        # base 10000, angle of pair i at position p: p / 10000^(2i/d)
        pos = torch.arange(rows, dtype=torch.float64, device=dev)
        freq = 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=dev) * 2 / d)
        a = pos[:, None] * freq
    else:
        # patch centres of a 37 x 37 grid in [-1, 1], base 100, rows in the first half of the pairs
        c = (torch.arange(37, dtype=torch.float64, device=dev) + 0.5) / 37 * 2 - 1
        freq = 2 * math.pi / 100.0 ** (torch.arange(d // 4, dtype=torch.float64, device=dev) * 4 / d)
        ah = (c[:, None] * freq)[:, None, :].expand(37, 37, d // 4)
        aw = (c[:, None] * freq)[None, :, :].expand(37, 37, d // 4)
        a = torch.cat([ah, aw], -1).reshape(37 * 37, d // 2)
    a = torch.cat([a, a], -1)
    return a.sin().float().contiguous(), a.cos().float().contiguous()


def _offsets(counts, dev):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device=dev)


def _pages(lens, page, gen, dev):
    """A block table whose pages lie in a random order of the pool; unused entries are -1."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + _SPARE_PAGES
    order = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pool


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=dt)

    new, old = _lengths(case)
    n = sum(new)
    st = {"case": case, "new": new, "old": old}
    if case["op"] == "prompt":
        st["q"] = normal(n, hq, d)
        st["k"], st["v"] = normal(n + sum(old), hk, d), normal(n + sum(old), hk, d)
        st["cu_q"] = _offsets(new, dev)
        st["cu_k"] = _offsets([a + b for a, b in zip(new, old)], dev) if sum(old) else None
        return st
    lens = [a + b for a, b in zip(new, old)]
    table, pool = _pages(lens, case["page"], gen, dev)
    st["table"] = table
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["k_cache"], st["v_cache"] = (normal(pool, hk, case["page"], d) for _ in range(2))
    if case["op"] == "append":
        # q, k and v side by side in one row a token, as one projection writes them
        rows = normal(n, hq + 2 * hk, d)
        st["q"], st["k"], st["v"] = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        st["q_out"], st["k_out"] = torch.empty_like(st["q"]).contiguous(), torch.empty_like(st["k"]).contiguous()
        st["cu"] = None if case["longest"] == 1 else _offsets(new, dev)
        st["sin"], st["cos"] = _tables(case, max(lens), dev)
    else:
        st["q"] = normal(case["seqs"], hq, d)
        if own:
            st["workspace"] = _context().paged_workspace()
    return st


# ------------------------------------------------------------- plain forms --


def _token_map(st):
    """(sequence, position) of every new token."""
    dev = st["k"].device
    new = torch.tensor(st["new"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(st["new"]), device=dev), new)
    first = torch.cumsum(new, 0) - new
    i = torch.arange(sum(st["new"]), device=dev) - first[seq]
    return seq, i + torch.tensor(st["old"], device=dev)[seq]


def _rotate(x, sin, cos, rot):
    h = x.shape[-1] // 2
    y = x * cos[:, None] + torch.cat([-x[..., h:], x[..., :h]], -1) * sin[:, None]
    return torch.where(rot[:, None, None], y, x)


def _append_plain(st):
    case, page = st["case"], st["case"]["page"]
    seq, pos = _token_map(st)
    row = pos if case["rope"] == "text" else pos % _FRAME - _PREFIX
    rot, row = row >= 0, row.clamp_min(0)
    sin, cos = st["sin"][row], st["cos"][row]
    dt = st["k"].dtype
    st["q_out"].copy_(_rotate(st["q"].float(), sin, cos, rot).to(dt))
    st["k_out"].copy_(_rotate(st["k"].float(), sin, cos, rot).to(dt))
    at, off = st["table"][seq, pos // page].long(), pos % page
    st["k_cache"][at, :, off] = st["k_out"]
    st["v_cache"][at, :, off] = st["v"]
    return {"q": st["q_out"], "k": st["k_out"], "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _prompt_plain(st):
    case = st["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty_like(st["q"])
    q0 = k0 = 0
    for a, b in zip(st["new"], st["old"]):
        keys = a + b
        k = st["k"][k0:k0 + keys].float().permute(1, 2, 0)
        v = st["v"][k0:k0 + keys].float().transpose(0, 1)
        j = torch.arange(keys, device=k.device)
        step = max(16, (1 << 28) // (hq * keys))
        for i0 in range(0, a, step):
            m = min(step, a - i0)
            q = st["q"][q0 + i0:q0 + i0 + m].float().reshape(m, hk, hq // hk, d).permute(1, 2, 0, 3)
            s = torch.matmul(q.reshape(hk, -1, d), k).div_(math.sqrt(d)).view(hk, hq // hk, m, keys)
            if case["causal"]:
                i = torch.arange(i0, i0 + m, device=k.device)
                s.masked_fill_(j > (i + b)[:, None], -math.inf)
            s = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
            o = torch.matmul(s.view(hk, -1, keys), v).view(hk, hq // hk, m, d) / s.sum(-1, keepdim=True)
            out[q0 + i0:q0 + i0 + m] = o.permute(2, 0, 1, 3).reshape(m, hq, d).to(out.dtype)
        q0, k0 = q0 + a, k0 + keys
    return out


def _token_plain(st):
    case, page = st["case"], st["case"]["page"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty_like(st["q"])
    for s, n in enumerate(st["new"]):
        at = st["table"][s, :-(-n // page)].long()
        k = st["k_cache"][at].float().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        v = st["v_cache"][at].float().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        q = st["q"][s].float().view(hk, hq // hk, d)
        p = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(d)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[s] = o.reshape(hq, d).to(out.dtype)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _append_plain, "prompt": _prompt_plain, "token": _token_plain}[op](state)
    ctx = _context()
    if op == "prompt":
        return ctx.attention_varlen(state["q"], state["k"], state["v"], state["cu_q"], cu_k=state["cu_k"],
                                    causal=state["case"]["causal"])
    from headshot_b200.engine import PagedKv, Rope

    cache = PagedKv(state["k_cache"], state["v_cache"], state["table"])
    if op == "token":
        return ctx.attention_paged(state["q"], cache, state["lens"], workspace=state["workspace"])
    rope = Rope(state["sin"], state["cos"], 0) if state["case"]["rope"] == "text" else \
        Rope(state["sin"], state["cos"], _PREFIX, _FRAME)
    q = ctx.kv_append(cache, state["k"], state["v"], state["lens"], cu_new=state["cu"], rope=rope, q=state["q"],
                      q_out=state["q_out"], k_out=state["k_out"])
    return {"q": q, "k": state["k_out"], "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


# ---------------------------------------------------------- 64-bit results --


def exact(case, seed):
    st = prepare(case, seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    g = hq // hk
    if case["op"] == "append":
        res = {"q": st["q"].double(), "k": st["k"].double(), "k_cache": st["k_cache"].double(),
               "v_cache": st["v_cache"].double()}
        sin, cos, table = st["sin"].double(), st["cos"].double(), st["table"].cpu()
        t = 0
        for s, (a, b) in enumerate(zip(st["new"], st["old"])):
            p = torch.arange(b, b + a, device=sin.device)
            row = p if case["rope"] == "text" else p % _FRAME - _PREFIX
            on = row >= 0
            for x in (res["q"], res["k"]):
                lo, hi = x[t:t + a, :, :d // 2].clone(), x[t:t + a, :, d // 2:].clone()
                c, w = cos[row[on]][:, None], sin[row[on]][:, None]
                new_lo = lo[on] * c[..., :d // 2] - hi[on] * w[..., :d // 2]
                new_hi = hi[on] * c[..., d // 2:] + lo[on] * w[..., d // 2:]
                lo[on], hi[on] = new_lo, new_hi
                x[t:t + a] = torch.cat([lo, hi], -1)
            done = 0
            while done < a:  # one stretch of a page at a time
                at, off = divmod(b + done, case["page"])
                m = min(a - done, case["page"] - off)
                pg = int(table[s, at])
                res["k_cache"][pg, :, off:off + m] = res["k"][t + done:t + done + m].transpose(0, 1)
                res["v_cache"][pg, :, off:off + m] = st["v"][t + done:t + done + m].double().transpose(0, 1)
                done += m
            t += a
        return res
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    if case["op"] == "prompt":
        q0 = k0 = 0
        for a, b in zip(st["new"], st["old"]):
            keys = a + b
            for h in range(hq):
                k = st["k"][k0:k0 + keys, h // g].double()
                v = st["v"][k0:k0 + keys, h // g].double()
                step = max(1, (1 << 27) // keys)
                for i0 in range(0, a, step):
                    i1 = min(a, i0 + step)
                    top = b + i1 if case["causal"] else keys
                    s = st["q"][q0 + i0:q0 + i1, h].double() @ k[:top].T
                    s *= d ** -0.5
                    if case["causal"]:
                        s += torch.triu(torch.full_like(s, -math.inf), diagonal=b + i0 + 1)
                    out[q0 + i0:q0 + i1, h] = torch.softmax(s, -1) @ v[:top]
            q0, k0 = q0 + a, k0 + keys
        return out
    for s, n in enumerate(st["new"]):
        p = torch.arange(n, device=out.device)
        at, off = st["table"][s][p // case["page"]].long(), p % case["page"]
        for h in range(hk):
            k, v = st["k_cache"][at, h, off].double(), st["v_cache"][at, h, off].double()
            w = torch.softmax(st["q"][s, h * g:(h + 1) * g].double() @ k.T * d ** -0.5, -1)
            out[s, h * g:(h + 1) * g] = w @ v
    return out
