"""One attention layer over the quantised paged cache, as a server runs it: prompts of different lengths together, then
one token of every sequence per step, then a sequence taken out of the cache.

    python examples/quantised_cache.py [--v-bits 4] [--steps 8]

Prints, for the prompts and for every step, how far the layer's output is from plain attention in 64 bits over the keys
and values before they were quantised."""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from chonklm_b200.kv_cache import QuantKvCache  # noqa: E402

HEADS, KV_HEADS, HEAD_DIM, BLOCK = 16, 8, 128, 16


def plain_attention(q, k, v):
    """64 bits: q [n, heads, hd], the last n tokens of k, v [len, kv_heads, hd]."""
    n, length = q.shape[0], k.shape[0]
    k, v = (t.double().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
    s = torch.einsum("nhd,phd->hnp", q.double(), k) / math.sqrt(HEAD_DIM)
    p = torch.arange(length, device=q.device)
    s = s.masked_fill(p > torch.arange(length - n, length, device=q.device)[:, None], -math.inf)
    return torch.einsum("hnp,phd->nhd", torch.softmax(s, -1), v)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--v-bits", type=int, default=8, choices=(8, 4))
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    prompts = [37, 512, 5, 260]
    most = max(prompts) + a.steps
    # every sequence's blocks up to its longest, handed out once
    per = (most + BLOCK - 1) // BLOCK
    table = torch.randperm(per * len(prompts), device="cuda").to(torch.int32).view(len(prompts), per)
    cache = QuantKvCache(HEADS, KV_HEADS, HEAD_DIM, n_blocks=table.numel(), block=BLOCK, v_bits=a.v_bits)
    inv_freq = (1e6 ** (-torch.arange(0, HEAD_DIM, 2, device="cuda", dtype=torch.float64) / HEAD_DIM)).float()
    weights = [1 + 0.1 * torch.randn(HEAD_DIM, device="cuda") for _ in range(2)]
    held = [([], []) for _ in prompts]           # plain keys and values of each sequence
    worst = 0.0

    def store(new):
        """Project (here: draw) q, k, v of new[i] tokens of each sequence; q as attention wants it."""
        seq = torch.repeat_interleave(torch.arange(len(prompts)), torch.tensor(new)).to("cuda", torch.int32)
        pos = torch.cat([torch.arange(sum(t.shape[0] for t in held[i][0]), sum(t.shape[0] for t in held[i][0]) + n)
                         for i, n in enumerate(new)]).to("cuda", torch.int32)
        qkv = torch.randn(sum(new), HEADS + 2 * KV_HEADS, HEAD_DIM, device="cuda", dtype=torch.bfloat16)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q = cache.store(q, k, v, seq, pos, table, inv_freq=inv_freq, q_norm=weights[0], k_norm=weights[1])
        kf = k.double() / torch.sqrt((k.double() ** 2).mean(-1, keepdim=True) + 1e-6) * weights[1].double()
        ang = (pos.double()[:, None] * inv_freq.double())[:, None]
        x, y = kf.chunk(2, -1)
        kf = torch.cat((x * ang.cos() - y * ang.sin(), x * ang.sin() + y * ang.cos()), -1)
        for i, (kk, vv) in enumerate(zip(kf.split(new), v.split(new))):
            held[i][0].append(kk)
            held[i][1].append(vv)
        return q

    def error(out, q, new):
        off = norm = 0.0
        for i, (o, qq) in enumerate(zip(out.split(new), q.split(new))):
            want = plain_attention(qq, torch.cat(held[i][0]), torch.cat(held[i][1]))
            off, norm = off + (o.double() - want).square().sum().item(), norm + want.square().sum().item()
        return math.sqrt(off / norm)

    q = store(prompts)
    cu = torch.tensor([0] + prompts).cumsum(0).to("cuda", torch.int32)
    length = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    out = cache.attend_prompt(q, cu, length, table)
    worst = error(out, q, prompts)
    print(f"prompts of {prompts} tokens: {worst:.4f} of the output's norm off")
    for step in range(a.steps):
        q = store([1] * len(prompts))
        length += 1
        out = cache.attend(q, length, table)
        e = error(out, q, [1] * len(prompts))
        worst = max(worst, e)
        print(f"step {step}: {e:.4f}")
    cache.check()
    n = int(length[1])
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    k, v = cache.load(torch.full_like(pos, 1), pos, table)
    off = ((k.double() - torch.cat(held[1][0])).norm() / torch.cat(held[1][0]).norm()).item()
    print(f"sequence 1 out of the cache: {tuple(k.shape)} keys, {off:.4f} of their norm off; {cache.nbytes} bytes of pages")
    return worst


if __name__ == "__main__":
    main()
