"""The workloads of the serving-step operators: block tables and slot maps, the 8-bit key / value cache (append, read
back, attention) and the gated delta rule.

Each operator has a plain form here in elementary torch operations (32-bit arithmetic, one rounding at the end) and the
call a user makes of ``tinystrata_b200``; ``own`` selects which of the two ``run`` takes.  ``exact`` states the same
results in 64 bits, token by token or request by request.
"""
import math
import random

import torch

own = False

BLOCK = 64            # tokens of a chunk of the plain gated delta rule
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a small decode batch: eight requests, one token each; the launch is all the cost
        dict(name="tables, 8 requests", kind="tables", requests=8, context=4000, new=1, prompts=0, block=16, lens=1),
        # a busy server's step: a thousand requests, one in sixteen of them a new prompt, some finished
        dict(name="tables, 1000 requests", kind="tables", requests=1000, context=32000, new=1, prompts=900, block=16,
             lens=2),
        # the new token of 48 decoding requests, into blocks that already hold tokens
        dict(name="append, 48 tokens", kind="append", requests=48, context=2000, new=1, heads=2, dim=256, block=16,
             dtype="bf16", lens=3),
        # prompts of 16,000 tokens in all, in the framework's own activation type
        dict(name="append, 8 prompts", kind="append", requests=8, context=0, new=2003, heads=8, dim=128, block=32,
             dtype="fp32", lens=4),
        # one user, a short conversation: latency
        dict(name="attention, 1 x 700", kind="attention", requests=1, context=700, queries=1, q_heads=16, heads=2,
             dim=256, block=16, window=0, dtype="bf16", lens=0),
        # a decode batch of uneven lengths up to 8192, some requests checking two or three drafted tokens
        dict(name="attention, 64 x 8192", kind="attention", requests=64, context=8192, queries=3, q_heads=32, heads=8,
             dim=128, block=16, window=0, dtype="bf16", lens=5),
        # two users with very long documents, queries in the framework's own activation type
        dict(name="attention, 2 x 131072", kind="attention", requests=2, context=131072, queries=1, q_heads=16,
             heads=2, dim=256, block=64, window=0, dtype="fp32", lens=0),
        # a chunk of a prompt over what is cached already
        dict(name="attention, prompt 2048", kind="attention", requests=1, context=8192, queries=2048, q_heads=16,
             heads=2, dim=256, block=16, window=0, dtype="bf16", lens=0),
        # one decoding user: one token through the recurrence
        dict(name="delta, 1 token", kind="delta", requests=1, tokens=1, k_heads=16, v_heads=32, dim=128,
             dtype="fp32", lens=0),
        # a decode batch: the states' traffic is the cost
        dict(name="delta, 128 x 1", kind="delta", requests=128, tokens=1, k_heads=16, v_heads=32, dim=128,
             dtype="bf16", lens=0),
        # prompts of uneven lengths in one packed batch
        dict(name="delta, 8 prompts", kind="delta", requests=8, tokens=1024, k_heads=16, v_heads=32, dim=128,
             dtype="fp32", lens=6),
        # one long prompt: the chunks follow one another
        dict(name="delta, prompt 8192", kind="delta", requests=1, tokens=8192, k_heads=16, v_heads=32, dim=128,
             dtype="bf16", lens=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "delta", "delta"])
    lens = rng.randrange(1, 1 << 30)
    dtype = rng.choice(list(DTYPES))
    block = rng.choice([16, 32, 64])
    if kind == "tables":
        return dict(kind=kind, requests=_log(rng, 1, 1000), context=_log(rng, 16, 32000), new=rng.randint(1, 4),
                    prompts=rng.choice([0, _log(rng, 1, 900)]), block=block, lens=lens)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, requests=_log(rng, 1, 256), context=_log(rng, 1, 4000), new=rng.randint(1, 4),
                        heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]), block=block, dtype=dtype,
                        lens=lens)
        return dict(kind=kind, requests=rng.randint(1, 8), context=rng.choice([0, _log(rng, 1, 500)]),
                    new=_log(rng, 5, 2000), heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), block=block,
                    dtype=dtype, lens=lens)
    if kind == "attention":
        heads, group, dim = rng.choice([(1, 8, 128), (2, 8, 256), (8, 4, 64), (4, 4, 128), (2, 6, 128), (8, 1, 64),
                                        (4, 2, 256), (3, 5, 64)])
        window = rng.choice([0, 0, _log(rng, 16, 2048)])
        if rng.random() < 0.3:
            q = _log(rng, 16, 1024)
            return dict(kind=kind, requests=rng.randint(1, 2), context=q + _log(rng, 1, 3000), queries=q,
                        q_heads=heads * group, heads=heads, dim=dim, block=block, window=window, dtype=dtype, lens=lens)
        requests = _log(rng, 1, 64)
        most = min(131072, (64 * 8192 * 8 * 128) // (2 * requests * heads * dim))
        return dict(kind=kind, requests=requests, context=_log(rng, 1, most), queries=rng.randint(1, 4),
                    q_heads=heads * group, heads=heads, dim=dim, block=block, window=window, dtype=dtype, lens=lens)
    k_heads, v_heads = rng.choice([(16, 32), (8, 8), (4, 16), (16, 16), (2, 6)])
    dim = rng.choice([64, 128, 128])
    if rng.random() < 0.5:
        return dict(kind=kind, requests=_log(rng, 1, 128), tokens=rng.choice([1, 1, 2, 4]), k_heads=k_heads,
                    v_heads=v_heads, dim=dim, dtype=dtype, lens=0)
    requests = _log(rng, 1, 16)
    return dict(kind=kind, requests=requests, tokens=_log(rng, 16, 4096 // requests), k_heads=k_heads,
                v_heads=v_heads, dim=dim, dtype=dtype, lens=rng.choice([0, lens]))


def lengths(case):
    """The requests' lengths, from the case alone: (cached before the step, new in it); for attention (cached with
    the step's own tokens, queries)."""
    rng = random.Random(case["lens"])
    n = case["requests"]
    if case["kind"] == "delta":
        t = case["tokens"]
        if not case["lens"]:
            return [0] * n, [t] * n
        return [0] * n, [t] + [_log(rng, 1, t) for _ in range(n - 1)]
    if case["kind"] == "attention":
        q = case["queries"]
        if not case["lens"]:
            return [case["context"]] * n, [q] * n
        new = [rng.randint(1, q) if q < 16 else q for _ in range(n)]
        c = case["context"]
        return [max(v, c if i == 0 else rng.randint(1, c)) for i, v in enumerate(new)], new
    if case["kind"] == "append":
        return [rng.randint(0, case["context"]) for _ in range(n)], [case["new"]] * n
    old, new = [], []
    for i in range(n):
        if case["prompts"] and i % 16 == 0:
            old.append(0)
            new.append(_log(rng, 1, case["prompts"]))
        else:
            old.append(rng.randint(1, case["context"]))
            new.append(case["new"])
    return old, new


def blocks_of(n, block):
    return (n + block - 1) // block


def seen(length, queries, window):
    """Pairs of queries and the keys they see."""
    total = 0
    for i in range(queries):
        p = length - queries + i + 1
        total += min(p, window) if window else p
    return total


def work(case):
    old, new = lengths(case)
    n, total = case["requests"], sum(new)
    if case["kind"] == "tables":
        done = [i for i in range(n) if _finished(case, i)]
        moved = sum(blocks_of(old[i], case["block"]) for i in done)
        taken = sum(blocks_of(a + b, case["block"]) - blocks_of(a, case["block"]) for a, b in zip(old, new))
        # lengths, new tokens and marks in; lengths and bounds out; blocks from and to the free list; the slots
        return {"bytes": 9 * n + 8 * n + 8 * (moved + taken) + 8 * total, "flops": 0}
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["kind"] == "append":
        row = case["heads"] * case["dim"] * 2
        kept = sum(a % case["block"] for a in old)
        scales = 8 * case["heads"] * sum(blocks_of(a + b, case["block"]) - a // case["block"] for a, b in zip(old, new))
        pool = sum(blocks_of(a + b, case["block"]) - a // case["block"] for a, b in zip(old, new)) * case["block"]
        # the new rows in, their codes and the partial blocks' codes out, and the whole read back as 32-bit values
        return {"bytes": total * row * (size + 1) + 2 * kept * row + scales + pool * row * 5, "flops": 0}
    if case["kind"] == "attention":
        dim, hq, hk, w = case["dim"], case["q_heads"], case["heads"], case["window"]
        keys = sum(min(a, b + w - 1) if w else a for a, b in zip(old, new))
        blocks = sum(blocks_of(a, case["block"]) for a in old)
        pairs = sum(seen(a, b, w) for a, b in zip(old, new))
        return {"bytes": 2 * keys * hk * dim + 8 * blocks * hk + 4 * blocks + 2 * total * hq * dim * size,
                "flops": 4 * pairs * hq * dim}
    dim, hk, hv = case["dim"], case["k_heads"], case["v_heads"]
    state = n * hv * dim * dim * 4
    return {"bytes": 2 * state + total * (2 * hk + 2 * hv) * dim * size + total * hv * 8,
            "flops": 6 * total * hv * dim * dim}


def _finished(case, i):
    return not (case["prompts"] and i % 16 == 0) and i % 9 == 4


# ---------------------------------------------------------------------------------------------------------- prepare
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _int(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


def _codes(shape, g, dev):
    """Codes of roughly normal values with a few large ones, as a block's largest value sets its scale."""
    out = torch.empty(shape, dtype=torch.int8, device=dev)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.randn(part.shape, device=dev, generator=g).mul_(36).round_().clamp_(-127, 127))
    return out


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    old, new = lengths(case)
    n, total = case["requests"], sum(new)
    s = dict(case=case)
    if case["kind"] == "tables":
        bs = case["block"]
        width = blocks_of(max(a + b for a, b in zip(old, new)), bs) + 1
        used = [0 if not a else blocks_of(a, bs) for a in old]
        need = sum(blocks_of(a + b, bs) - u for a, b, u in zip(old, new, used))
        pool = sum(used) + need + 37
        perm = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
        count = _int(used, dev, torch.int64)
        first = torch.cumsum(count, 0) - count
        col = torch.arange(width, device=dev)
        inside = col < count[:, None]
        s["table"] = torch.where(inside, perm[(first[:, None] + col).clamp(max=pool - 1)], -1).to(torch.int32)
        held = sum(used)
        s["free_room"] = torch.full((pool + 1,), -1, dtype=torch.int32, device=dev)   # one more than the blocks
        s["free_room"][:pool - held] = perm[held:]
        s["n_free"] = _int([pool - held], dev)
        s["lens"] = _int(old, dev)
        done = [_finished(case, i) for i in range(n)]
        s["new"] = _int([0 if d else b for d, b in zip(done, new)], dev)
        s["done"] = _int(done, dev, torch.uint8)
        s["room"] = total + 5         # the slots' buffer: a little more than the step's tokens
        return s
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "append":
        h, d, bs = case["heads"], case["dim"], case["block"]
        touched = [blocks_of(a + b, bs) - a // bs for a, b in zip(old, new)]
        nb = sum(touched)
        order = torch.randperm(nb, device=dev, generator=g)
        at, slots = 0, []
        for a, b, t in zip(old, new, touched):
            p = torch.arange(a % bs, a % bs + b, device=dev)
            slots.append(order[at + p // bs] * bs + p % bs)
            at += t
        s["slots"] = torch.cat(slots).to(torch.int64)
        s["every"] = torch.arange(nb * bs, device=dev, dtype=torch.int64)
        for x in "kv":
            s[x + "_codes"] = _codes((nb, h, bs, d), g, dev)
            s[x + "_scale"] = torch.rand((nb, h), device=dev, generator=g).mul_(0.02).add_(0.005)
            gain = torch.exp(torch.randn((1, h, d), device=dev, generator=g) * 0.5)
            s[x] = (torch.randn((total, h, d), device=dev, generator=g) * gain).to(dt)
    elif case["kind"] == "attention":
        h, d, bs = case["heads"], case["dim"], case["block"]
        count = [blocks_of(a, bs) for a in old]
        nb, width = sum(count) + 3, max(count)
        order = torch.randperm(nb, device=dev, generator=g).to(torch.int32)
        cnt = _int(count, dev, torch.int64)
        col = torch.arange(width, device=dev)
        first = torch.cumsum(cnt, 0) - cnt
        s["table"] = torch.where(col < cnt[:, None], order[(first[:, None] + col).clamp(max=nb - 1)], -1).to(torch.int32)
        s["lens"] = _int(old, dev)
        s["cu"] = _int([sum(new[:i]) for i in range(n + 1)], dev)
        s["max_queries"] = max(new)
        for x in "kv":
            s[x + "_codes"] = _codes((nb, h, bs, d), g, dev)
            s[x + "_scale"] = torch.rand((nb, h), device=dev, generator=g).mul_(0.02).add_(0.015)
        s["q"] = (torch.randn((total, case["q_heads"], d), device=dev, generator=g) * 1.5).to(dt)
    else:
        hk, hv, d = case["k_heads"], case["v_heads"], case["dim"]
        unit = torch.nn.functional.normalize
        s["q"] = unit(torch.randn((total, hk, d), device=dev, generator=g), dim=-1).to(dt)
        s["k"] = unit(torch.randn((total, hk, d), device=dev, generator=g), dim=-1).to(dt)
        s["v"] = torch.randn((total, hv, d), device=dev, generator=g).to(dt)
        rate = torch.exp(torch.rand((1, hv), device=dev, generator=g) * 5 - 5)          # heads that keep long and short
        s["g"] = -rate * torch.nn.functional.softplus(torch.randn((total, hv), device=dev, generator=g))
        s["beta"] = torch.sigmoid(torch.randn((total, hv), device=dev, generator=g))
        s["state"] = torch.randn((n, hv, d, d), device=dev, generator=g) * 0.1
        s["after"] = torch.empty_like(s["state"])
        s["cu"] = _int([sum(new[:i]) for i in range(n + 1)], dev)
        s["max_tokens"] = max(new)
        s["scale"] = d ** -0.5
        return s
    if own:
        import tinystrata_b200 as T
        s["cache"] = T.KV8Cache(k=s["k_codes"], v=s["v_codes"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"tables": plain_tables, "append": plain_append, "attention": plain_attention,
                "delta": plain_delta}[kind](s)
    import tinystrata_b200 as T
    if kind == "tables":
        free = s["free_room"][:-1]
        p = T.block_tables(s["lens"], s["new"], s["table"], free, s["n_free"], s["case"]["block"], s["room"], done=s["done"])
        return dict(lens=p.lens, bounds=p.cu, slots=p.slots, n_free=p.n_free, free=free, table=s["table"])
    if kind == "append":
        T.kv8_append(s["cache"], s["k"], s["v"], s["slots"])
        k, v = T.kv8_read(s["cache"], s["every"])
        return dict(k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "attention":
        return T.kv8_attention(s["cache"], s["q"], s["table"], s["lens"], cu_q=s["cu"], max_q=s["max_queries"],
                               window=s["case"]["window"])
    o, after = T.gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], cu_seqlens=s["cu"],
                             max_len=s["max_tokens"], scale=s["scale"], state_out=s["after"])
    return dict(o=o, state=after)


def plain_tables(s):
    bs, table, room = s["case"]["block"], s["table"], s["free_room"]
    lens, width, cap = s["lens"].long(), s["table"].shape[1], room.numel() - 1
    col = torch.arange(width, device=table.device)
    gone = torch.where(s["done"] != 0, (lens + bs - 1) // bs, 0)
    first = s["n_free"] + torch.cumsum(gone, 0) - gone
    to = torch.where(col < gone[:, None], first[:, None] + col, cap)
    room[to.view(-1)] = table.view(-1)                        # what is not given back goes to the place past the end
    n_free = s["n_free"] + gone.sum()
    lens = torch.where(s["done"] != 0, 0, lens)
    new = s["new"].long().clamp(min=0)
    before, after = (lens + bs - 1) // bs, (lens + new + bs - 1) // bs
    fits = after <= width
    need = torch.where(fits, after - before, 0)
    taken = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (taken <= n_free))
    at = n_free - 1 - ((taken - need)[:, None] + col - before[:, None])
    put = ok[:, None] & (col >= before[:, None]) & (col < after[:, None])
    table.copy_(torch.where(put, room[at.clamp(0, cap - 1)], table))
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    t = torch.arange(s["room"], device=table.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = r < len(lens)
    r = r.clamp(max=len(lens) - 1)
    pos = lens[r] + t - cu[r]
    slot = table[r, (pos // bs).clamp(max=width - 1)].long() * bs + pos % bs
    slots = torch.where(live & ok[r], slot, -1)
    left = n_free - torch.where(ok, need, 0).sum()
    return dict(lens=torch.where(ok, lens + new, lens).int(), bounds=cu.int(), slots=slots, n_free=left.int(),
                free=room[:-1], table=table)


def plain_append(s):
    bs = s["case"]["block"]
    blk, off = s["slots"] // bs, s["slots"] % bs
    out = {}
    for x in "kv":
        codes, scale, rows = s[x + "_codes"], s[x + "_scale"], s[x].float()
        nb, h = scale.shape
        peak = torch.zeros_like(scale).scatter_reduce(0, blk[:, None].expand(-1, h), rows.abs().amax(-1), "amax")
        start = torch.full((nb,), bs, device=blk.device).scatter_reduce(0, blk, off, "amin")
        touched = (start < bs)[:, None]
        was = torch.where((start > 0)[:, None] | ~touched, scale, 0.0)
        now = torch.where(touched, torch.maximum(was, peak / torch.full_like(peak, 127.0)), was)   # a true division
        ratio = torch.where(now > 0, was / now, 0.0)
        old = (torch.arange(bs, device=blk.device) < start[:, None]) & touched
        again = torch.round(codes.float() * ratio[:, :, None, None]).to(torch.int8)
        codes.copy_(torch.where(old[:, None, :, None], again, codes))
        by = now[blk][:, :, None]
        new = torch.where(by > 0, torch.round(rows / by).clamp(-127, 127), 0.0).to(torch.int8)
        codes[blk, :, off] = new
        scale.copy_(now)
        e = s["every"]
        out[x] = codes[e // bs, :, e % bs].float() * scale[e // bs][:, :, None]
        out[x + "_scale"] = scale
    return out


def plain_attention(s):
    c = s["case"]
    bs, hq, h, d = c["block"], c["q_heads"], c["heads"], c["dim"]
    table, lens, cu, q = s["table"].long(), s["lens"].long(), s["cu"].long(), s["q"]
    n, width, most = len(lens), table.shape[1], s["max_queries"]
    keys = width * bs
    at = table.clamp(min=0)
    k = (s["k_codes"][at].float() * s["k_scale"][at][..., None, None]).transpose(1, 2).reshape(n, h, keys, d)
    count = cu[1:] - cu[:-1]
    i = torch.arange(most, device=q.device)
    rows = (cu[:-1, None] + i).clamp(max=len(q) - 1)
    qp = q[rows].float().view(n, most, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(n, h, hq // h * most, d)
    x = (qp @ k.transpose(-1, -2)).mul_(d ** -0.5)
    del k
    j = torch.arange(keys, device=q.device)
    pos = lens[:, None] - count[:, None] + i
    see = (j <= pos[..., None]) & (i < count[:, None])[..., None]
    if c["window"]:
        see &= j > pos[..., None] - c["window"]
    x = x.view(n, h, hq // h, most, keys).masked_fill_(~see[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3.0e38)).exp_()
    total = x.sum(-1, keepdim=True)
    v = (s["v_codes"][at].float() * s["v_scale"][at][..., None, None]).transpose(1, 2).reshape(n, h, keys, d)
    o = (x.view(n, h, hq // h * most, keys) @ v).view(n, h, hq // h, most, d) / total.clamp(min=1e-30)
    t = torch.arange(len(q), device=q.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, hq, d)[r, t - cu[r]].to(q.dtype)


def plain_delta(s):
    q, k, v, g, beta, cu = s["q"], s["k"], s["v"], s["g"], s["beta"], s["cu"].long()
    n, most, hk, hv, d = len(cu) - 1, s["max_tokens"], q.shape[1], v.shape[1], q.shape[2]
    i = torch.arange(most, device=q.device)
    live = i < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + i).clamp(max=len(q) - 1)
    pad = lambda x: torch.where(live.view(n, most, *[1] * (x.dim() - 1)), x[rows].float(), 0.0)  # noqa: E731
    heads = lambda x: pad(x).repeat_interleave(hv // hk, 2).transpose(1, 2)  # noqa: E731
    q, k, v = heads(q) * s["scale"], heads(k), pad(v).transpose(1, 2)
    g, beta = pad(g).transpose(1, 2), pad(beta).transpose(1, 2)
    state = s["state"]
    if most < 16:
        out = []
        for t in range(most):                              # the recurrence itself
            state = state * g[:, :, t].exp()[..., None, None]
            u = beta[:, :, t, None] * (v[:, :, t] - (k[:, :, t, None] @ state)[:, :, 0])
            state = state + k[:, :, t, :, None] * u[:, :, None]
            out.append((q[:, :, t, None] @ state)[:, :, 0])
        o = torch.stack(out, 2)
    else:
        m = -most % BLOCK
        fill = lambda x: torch.nn.functional.pad(x, (0, 0, 0, m)).view(n, hv, -1, BLOCK, x.shape[-1])  # noqa: E731
        q, k, v, beta = fill(q), fill(k), fill(v), fill(beta[..., None])
        gc = fill(g[..., None]).cumsum(3)
        low = torch.ones(BLOCK, BLOCK, dtype=torch.bool, device=q.device).tril()
        fall = torch.where(low, (gc - gc.transpose(-1, -2)).clamp(max=0), -math.inf).exp()
        a = beta * (k @ k.transpose(-1, -2)) * fall.tril(-1)
        inv = torch.eye(BLOCK, device=q.device).expand_as(a).contiguous()
        for r in range(1, BLOCK):                          # the rows of (1 + a)^-1, one after the other
            inv[..., r, :r] = -(a[..., r, None, :r] @ inv[..., :r, :r])[..., 0, :]
        mix = inv * beta.transpose(-1, -2)
        att = (q @ k.transpose(-1, -2)) * fall
        end = gc[..., -1:, :]
        out = []
        for t in range(q.shape[2]):                        # the chunks follow one another through the state
            w = mix[:, :, t] @ (v[:, :, t] - gc[:, :, t].exp() * (k[:, :, t] @ state))
            out.append(gc[:, :, t].exp() * (q[:, :, t] @ state) + att[:, :, t] @ w)
            state = end[:, :, t].exp() * state + (k[:, :, t] * (end[:, :, t] - gc[:, :, t]).exp()).transpose(-1, -2) @ w
        o = torch.cat(out, 2)
    t = torch.arange(len(s["q"]), device=q.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    s["after"].copy_(state)
    return dict(o=o.transpose(1, 2)[r, t - cu[r]].to(s["v"].dtype), state=s["after"])


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    if case["kind"] == "tables":
        return None            # whole numbers: equal or wrong
    s = prepare(case, seed)
    old, new = lengths(case)
    at = [sum(new[:i]) for i in range(len(new) + 1)]
    if case["kind"] == "append":
        return None if len(s["slots"]) > 3000 else exact_append(s, case)
    if case["kind"] == "attention":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        hq, h, d, bs = case["q_heads"], case["heads"], case["dim"], case["block"]
        for r, (length, queries) in enumerate(zip(old, new)):
            b = s["table"][r, :blocks_of(length, bs)].long()
            q = s["q"][at[r]:at[r + 1]].double()
            for head in range(h):
                k, v = ((s[x + "_codes"][b, head].double() * s[x + "_scale"][b, head].double()[:, None, None])
                        .reshape(-1, d)[:length] for x in "kv")
                for first in range(0, queries, 256):
                    part = q[first:first + 256, head * (hq // h):(head + 1) * (hq // h)]
                    x = torch.einsum("igd,jd->igj", part, k) / math.sqrt(d)
                    p = length - queries + first + torch.arange(len(part), device=q.device)[:, None, None]
                    j = torch.arange(length, device=q.device)
                    hidden = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
                    x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                    out[at[r] + first:at[r] + first + len(part), head * (hq // h):(head + 1) * (hq // h)] = \
                        torch.einsum("igj,jd->igd", x, v)
        return out
    rep = case["v_heads"] // case["k_heads"]
    n, most = case["requests"], max(new)
    o = torch.empty(s["v"].shape, dtype=torch.float64, device=s["v"].device)
    state = s["state"].double()
    cu = s["cu"].long()
    for t in range(most):                                  # the recurrence, every request at once
        alive = [r for r in range(n) if new[r] > t]
        rows = cu[:-1][alive] + t
        q, k = (s[x][rows].double().repeat_interleave(rep, 1) for x in "qk")
        now = state[alive] if len(alive) < n else state
        now = now * s["g"][rows].double().exp()[..., None, None]
        u = s["beta"][rows].double()[..., None] * (s["v"][rows].double() - torch.einsum("rhk,rhkv->rhv", k, now))
        now = now + torch.einsum("rhk,rhv->rhkv", k, u)
        o[rows] = torch.einsum("rhk,rhkv->rhv", q, now) * case["dim"] ** -0.5
        if len(alive) < n:
            state[alive] = now
        else:
            state = now
    return dict(o=o, state=state)


def exact_append(s, case):
    """Block by block, as a reader of the definition would do it by hand; codes by the same 32-bit divisions, since a
    value half way between two codes has no other definition."""
    import numpy as np
    bs, f = case["block"], np.float32
    slots = s["slots"].cpu().numpy()
    out = {}
    for x in "kv":
        codes, scale = s[x + "_codes"].cpu().numpy(), s[x + "_scale"].cpu().numpy()
        rows = s[x].float().cpu().numpy()
        values = np.zeros((codes.shape[0] * bs, codes.shape[1], codes.shape[3]))
        for b in np.unique(slots // bs):
            mine = np.nonzero(slots // bs == b)[0]
            first = int((slots[mine] % bs).min())
            for h in range(codes.shape[1]):
                was = scale[b, h] if first else f(0)
                now = max(was, f(np.abs(rows[mine, h]).max() / f(127)))
                codes[b, h, :first] = np.rint(codes[b, h, :first].astype(f) * (was / now if now else f(0)))
                for t in mine:
                    codes[b, h, slots[t] % bs] = np.rint(rows[t, h] / now) if now else 0
                scale[b, h] = now
        values = codes.astype(np.float64) * scale.astype(np.float64)[:, :, None, None]
        out[x] = values.transpose(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])
        out[x + "_scale"] = scale.astype(np.float64)
    return out
