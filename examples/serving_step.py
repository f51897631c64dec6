"""A small hybrid decoder served step by step: paged 8-bit attention layers and gated delta rule layers between MoE layers.

Every layer is a mixer (three of four the gated delta rule, the fourth attention over the paged 8-bit cache) and a MoE block
of the Qwen configuration with fewer experts.  A step takes the packed tokens of all requests (prompts and single tokens
together), and its mixers, caches and block tables run without a word of the lengths on the host.

    python -m examples.serving_step [--layers 4] [--requests 16] [--prompt 200] [--steps 32]

Weights are random and position embeddings, convolutions and sampling are left out: it shows the calls and their order.
"""
from __future__ import annotations

import argparse

import torch

import tinystrata_b200 as T
from tinystrata_b200 import synth
from tinystrata_b200.layer import PrefillLayer

Q_HEADS, KV_HEADS, HEAD_DIM = 16, 2, 256          # attention
K_HEADS, V_HEADS, RULE_DIM = 16, 32, 128          # gated delta rule
FEW = 16                                          # tokens a step up to which the MoE block takes the decode path


def rms(x, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


class HybridDecoder:
    """The model and the state of its requests: row r of ``table``, ``lens`` and every layer's ``states`` is request r."""

    def __init__(self, n_layers=4, requests=16, max_tokens=4096, pool_blocks=1024, block_size=16, max_len=4096,
                 n_expert=32, device="cuda", seed=0):
        self.cfg = dict(synth.QWEN, n_expert=n_expert)
        H, self.requests, self.block_size = self.cfg["n_embd"], requests, block_size
        w = synth.device_layers(self.cfg, n_layers, seed, device)
        gen = torch.Generator(device=device).manual_seed(seed + 1)

        def dense(n, m):
            return (torch.randn((n, m), generator=gen, device=device) * n ** -0.5).bfloat16()

        self.layers = []
        for i in range(n_layers):
            layer = dict(moe=T.MoELayer(self.cfg, w["blobs"][i], w["routers"][i], w["sh_blobs"][i], max_tokens=FEW),
                         prompt=PrefillLayer(self.cfg, w["blobs"][i], w["routers"][i], w["sh_blobs"][i], max_tokens=max_tokens))
            if i % 4 == 3:
                layer.update(cache=T.KV8Cache(pool_blocks, KV_HEADS, HEAD_DIM, block_size, device=device),
                             inp=dense(H, (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM), out=dense(Q_HEADS * HEAD_DIM, H))
            else:
                layer.update(states=torch.zeros((requests, V_HEADS, RULE_DIM, RULE_DIM), device=device),
                             inp=dense(H, (2 * K_HEADS + V_HEADS) * RULE_DIM), gates=dense(H, 2 * V_HEADS),
                             out=dense(V_HEADS * RULE_DIM, H))
            self.layers.append(layer)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.table = torch.full((requests, (max_len + block_size - 1) // block_size), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pool_blocks, dtype=torch.int32, device=device)
        self.n_free = torch.full((1,), pool_blocks, dtype=torch.int32, device=device)
        self.order = torch.arange(requests, dtype=torch.int32, device=device)

    def attend(self, layer, h, plan, longest):
        """[T, H] -> [T, Q_HEADS * HEAD_DIM]: the tokens into the cache, then attention over it."""
        x = (h @ layer["inp"]).view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM)
        q, k, v = x.split((Q_HEADS, KV_HEADS, KV_HEADS), 1)                 # strided views: no copies
        T.kv8_append(layer["cache"], k, v, plan.slots)
        return T.kv8_attention(layer["cache"], q, self.table, plan.lens, cu_q=plan.cu, max_q=longest).flatten(1)

    def recur(self, layer, h, plan, longest, idx):
        """[T, H] -> [T, V_HEADS * RULE_DIM]: the tokens through the requests' states."""
        x = (h @ layer["inp"]).view(-1, 2 * K_HEADS + V_HEADS, RULE_DIM)
        q, k, v = x.split((K_HEADS, K_HEADS, V_HEADS), 1)
        g, beta = (h @ layer["gates"]).float().split(V_HEADS, 1)
        out, _ = T.gated_delta(q, k, v, -torch.nn.functional.softplus(g), torch.sigmoid(beta), layer["states"],
                               cu_seqlens=plan.cu, max_len=longest, state_idx=idx, qk_norm=True)
        return out.flatten(1)

    @torch.no_grad()
    def step(self, x, n_new, longest, done=None):
        """One step of all requests.  x fp32 [tokens, H], request after request; n_new int32 [requests] on the device;
        longest: at least the most tokens of one request; done uint8 [requests] ends requests, whose rows start anew.
        Returns (hidden states, BlockPlan); a request that found no blocks keeps its caches and states as they were."""
        plan = T.block_tables(self.lens, n_new, self.table, self.free, self.n_free, self.block_size, x.shape[0], done)
        kept = self.lens if done is None else torch.where(done != 0, 0, self.lens)
        idx = torch.where(plan.lens > kept, self.order, -1)                 # -1: not served, its state is not touched
        self.lens, self.n_free = plan.lens, plan.n_free
        x = x.clone()
        h = torch.empty_like(x)
        hq = torch.empty((x.shape[0], x.shape[1] // 32 * 36), dtype=torch.uint8, device=x.device)
        for layer in self.layers:
            mixed = rms(x).bfloat16()
            if "cache" in layer:
                mixed = self.attend(layer, mixed, plan, longest)
            else:
                if done is not None:
                    layer["states"].masked_fill_((done != 0).view(-1, 1, 1, 1), 0.0)
                mixed = self.recur(layer, mixed, plan, longest, idx)
            x += (mixed @ layer["out"]).float()
            T.rms_norm_q8_1(x, h, hq)
            if x.shape[0] <= FEW:
                layer["moe"].forward(x, h, hq)
            else:
                layer["prompt"].forward(x, h)
        return x, plan


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args(argv)
    if not torch.cuda.is_available():
        raise SystemExit("serving_step: a B200 is needed (there is no CPU path)")
    block = 16
    need = a.requests * ((a.prompt + a.steps + block - 1) // block)
    m = HybridDecoder(a.layers, a.requests, max_tokens=max(a.requests * a.prompt, FEW), pool_blocks=need + 4,
                      max_len=a.prompt + a.steps)
    H = m.cfg["n_embd"]

    def timed(x, counts, longest):
        ev = [torch.cuda.Event(enable_timing=True) for _ in "ab"]
        ev[0].record()
        out, _ = m.step(x, counts, longest)
        ev[1].record()
        ev[1].synchronize()
        return out, ev[0].elapsed_time(ev[1])

    x = torch.randn((a.requests * a.prompt, H), device="cuda")
    out, ms = timed(x, torch.full((a.requests,), a.prompt, dtype=torch.int32, device="cuda"), a.prompt)
    print(f"prompts: {x.shape[0]} tokens in {ms:.2f} ms (the first step, with its set-up)")
    one = torch.ones(a.requests, dtype=torch.int32, device="cuda")
    x = out.view(a.requests, a.prompt, H)[:, -1].contiguous()
    times = []
    for _ in range(a.steps):
        x, ms = timed(x, one, 1)
        x = rms(x)
        times.append(ms)
    times.sort()
    print(f"decode: {a.requests} requests, {a.layers} layers: {times[len(times) // 2]:.3f} ms a step (median of {a.steps}); "
          f"lengths {m.lens.min().item()} to {m.lens.max().item()}, {m.n_free.item()} blocks left")
    if not torch.isfinite(x).all() or T.device_error():
        raise SystemExit("serving_step: the outputs are not finite")


if __name__ == "__main__":
    main()
