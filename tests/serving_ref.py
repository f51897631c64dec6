"""Plain statements of the serving-step operators (block tables, the 8-bit cache, attention over it, the gated delta
rule), value by value in 64 bits where they compute, for the tests."""
import math

import numpy as np
import torch


def blocks_of(n, bs):
    return -(-n // bs)


def block_tables(lens, new, table, free, n_free, bs, cap, done=None):
    """Python integers in the order of the definition; table and free are copies that come back changed."""
    R, W = len(lens), table.shape[1]
    table, stack = table.copy(), [int(x) for x in free[:n_free]]
    free = free.copy()
    done = [0] * R if done is None else done
    for r in range(R):
        if done[r]:
            stack += [int(x) for x in table[r, :min(blocks_of(max(lens[r], 0), bs), W)]]
    free[:len(stack)] = stack
    have, taken, granted, out_lens, slots, cu = len(stack), 0, 0, [], [], [0]
    for r in range(R):
        n, a = max(lens[r], 0), max(new[r], 0)
        has, after = blocks_of(n, bs), blocks_of(n + a, bs)
        fits = after <= W and not done[r]
        need = after - has if fits else 0
        taken += need
        ok = fits and (need == 0 or taken <= have)
        if ok:
            for j in range(need):
                table[r, has + j] = stack[have - 1 - (taken - need + j)]
        out_lens.append(0 if done[r] else n + a if ok else n)
        for i in range(a):
            p = n + i
            slots.append(int(table[r, p // bs]) * bs + p % bs if ok else -1)
        cu.append(cu[-1] + a)
        if taken <= have:
            granted = taken
    slots = (slots + [-1] * cap)[:cap]
    return dict(lens=out_lens, cu=cu, slots=slots, n_free=have - granted, table=table, free=free)


def append(codes, scale, rows, slots, bs):
    """codes int8 [NB, H, bs, D] and scale fp32 [NB, H] (numpy, changed in place), rows fp32 [T, H, D]; one run (tokens of
    one call in one block) after the other, with the 32-bit divisions of the definition."""
    f = np.float32
    rows = np.nan_to_num(rows, nan=0.0, posinf=f(3.3895314e38), neginf=f(-3.3895314e38)).astype(f)
    NB = codes.shape[0]
    t = 0
    while t < len(slots):
        s = int(slots[t])
        n = 1
        if 0 <= s < NB * bs:
            while t + n < len(slots) and int(slots[t + n]) == s + n and (s + n) % bs:
                n += 1
            b, off = s // bs, s % bs
            for h in range(codes.shape[1]):
                was = scale[b, h] if off else f(0)
                now = f(max(was, f(np.abs(rows[t:t + n, h]).max() / f(127))))
                if off and now != was:
                    codes[b, h, :off] = np.rint(codes[b, h, :off].astype(f) * f(was / now))
                with np.errstate(over="ignore"):
                    codes[b, h, off:off + n] = np.clip(np.rint(rows[t:t + n, h] / now), -127, 127) if now > 0 else 0
                scale[b, h] = now
        t += n


def attention(k_codes, v_codes, ks, vs, q, table, lens, cu, scale, window):
    """fp64 outputs and sum p |v| (the size of what each output sums).  Block ids outside the cache hide their keys."""
    NB, H, bs, D = k_codes.shape
    T, Hq, _ = q.shape
    G = Hq // H
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for r in range(len(lens)):
        n, L = cu[r + 1] - cu[r], min(int(lens[r]), table.shape[1] * bs)
        if n <= 0 or L <= 0:
            continue
        ids = table[r, :blocks_of(L, bs)].long()
        good = (ids >= 0) & (ids < NB)
        ids = ids.clamp(0, NB - 1)
        j = torch.arange(L, device=q.device)
        pos = L - n + torch.arange(n, device=q.device)
        see = (j <= pos[:, None]) & good.repeat_interleave(bs)[:L]
        if window:
            see &= j > pos[:, None] - window
        for h in range(H):
            k = (k_codes[ids, h].double() * ks[ids, h].double()[:, None, None]).reshape(-1, D)[:L]
            v = (v_codes[ids, h].double() * vs[ids, h].double()[:, None, None]).reshape(-1, D)[:L]
            for i in range(G):
                x = (q[cu[r]:cu[r + 1], h * G + i].double() @ k.T) * scale
                x = x.masked_fill(~see, -math.inf)
                p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
                z = p.sum(-1, keepdim=True)
                p = torch.where(z > 0, p / z.clamp(min=1e-300), torch.zeros_like(p))
                out[cu[r]:cu[r + 1], h * G + i] = p @ v
                mag[cu[r]:cu[r + 1], h * G + i] = p @ v.abs()
    return out, mag


def gated_delta(q, k, v, g, beta, state, cu, idx=None, scale=None, qk_norm=False, eps=1e-6):
    """fp64 recurrence over the sequences; returns outputs and the states after."""
    T, Hk, Dk = q.shape
    Hv, Dv = v.shape[1:]
    rep = Hv // Hk
    scale = Dk ** -0.5 if scale is None else scale
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if qk_norm:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    out = torch.zeros((T, Hv, Dv), dtype=torch.float64, device=q.device)
    after = state.double().clone()
    for b in range(len(cu) - 1):
        i = b if idx is None else idx[b]
        S = state[i].double() if i >= 0 else torch.zeros(state.shape[1:], dtype=torch.float64, device=q.device)
        for t in range(cu[b], cu[b + 1]):
            S = S * torch.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - torch.einsum("hk,hkv->hv", k[t], S))
            S = S + k[t][:, :, None] * u[:, None]
            out[t] = scale * torch.einsum("hk,hkv->hv", q[t], S)
        if i >= 0:
            after[i] = S
    return out, after
