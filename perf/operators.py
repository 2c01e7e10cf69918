"""The quantised paged key-value cache: its operators as cases to be timed and compared.

Four operators work on one layer of a paged cache whose keys take 8 bits and whose values take 8 or 4 bits, one scale of
16 bits for each 32 values of a head:

  write    q and k of new tokens normed per head (or not) and rotated, q returned, k and v quantised into their pages
  read     cached keys and values of given (sequence, position) pairs, as the 16-bit values they stand for
  token    attention of one new token per sequence over its cached positions
  prompt   causal attention of several new tokens per sequence over its cached positions, sequences of different lengths together

`own` chooses between the plain form (elementary torch operations in 32 bits) and chonklm_b200.kv_cache.
"""
import math
import random

import torch

own = False

GROUP = 32          # values that share a scale
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases

def _case(op, heads, kv_heads, head_dim, **kw):
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": 16, "v_bits": 8, "dtype": "f16",
         "window": 0, "norm": False, "interleaved": False, "seqs": 1, "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 0}
    c.update(kw)
    return c


def listed():
    small, mid, wide = (9, 3, 64), (16, 8, 128), (4, 1, 256)   # the head layouts of this repository's configurations
    return [
        # the smallest call: the one new token of one sequence, written and read back
        _case("write", *small, name="write one token", old_lo=57, old_hi=57),
        # one step of the batched decode: 256 sequences, a token each, 32-bit projections
        _case("write", *small, name="write a decode step of 256", seqs=256, old_lo=128, old_hi=383, dtype="f32"),
        # prompts of several sequences at once, with per-head norms; the largest write
        _case("write", *mid, name="write ragged prompts", seqs=7, new_lo=333, new_hi=4091, norm=True, dtype="bf16", v_bits=4),
        # sequences taken out of the cache (to move them elsewhere); the largest read
        _case("read", *mid, name="read four sequences", seqs=4, new_lo=9001, new_hi=16001, dtype="bf16", v_bits=4, block=32),
        # one short conversation: latency
        _case("token", *small, name="token, one short", old_lo=130, old_hi=130),
        # the batched decode workload: many short sequences
        _case("token", *small, name="token, 256 short", seqs=256, old_lo=128, old_hi=383),
        # wide heads, one kv head, a sliding window
        _case("token", *wide, name="token, window of 512", seqs=24, old_lo=90, old_hi=2040, window=512, dtype="bf16", block=64),
        # one long document: the length has to be split over the machine
        _case("token", *mid, name="token, one long", old_lo=32747, old_hi=32747, dtype="bf16"),
        # a serving batch at long contexts, four query heads to a kv head: the most bytes
        _case("token", 32, 8, 128, name="token, 64 long", seqs=64, old_lo=1021, old_hi=8190, v_bits=4, dtype="bf16", block=32),
        # a follow-up question on a cached conversation
        _case("prompt", *small, name="prompt, short follow-up", new_lo=37, new_hi=37, old_lo=203, old_hi=203),
        # fresh prompts of different lengths: the most arithmetic
        _case("prompt", *mid, name="prompt, ragged fresh", seqs=3, new_lo=701, new_hi=4093, dtype="bf16"),
        # chunks on top of cached prefixes, wide heads, a sliding window
        _case("prompt", *wide, name="prompt, chunks, window", seqs=6, new_lo=65, new_hi=1501, old_lo=0, old_hi=700, window=512, v_bits=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "token", "token", "prompt", "prompt"])
    heads, kv, hd = rng.choice([(9, 3, 64), (16, 8, 128), (4, 1, 256), (32, 8, 128), (8, 8, 64), (14, 2, 64), (10, 2, 128), (12, 1, 128), (6, 3, 256)])
    kw = {"block": rng.choice([16, 32, 64, 128]), "v_bits": rng.choice([8, 4]), "dtype": rng.choice(["f16", "bf16"]),
          "window": rng.choice([0, 0, _log(rng, 17, 2000)])}
    per = kv * hd / 1024.0                    # a position's size against the middle layout's
    if op in ("write", "read"):
        total = _log(rng, 1, (16000 if op == "write" else 48000) / max(per, heads * hd / 2048.0))
        kw["seqs"] = min(total, _log(rng, 1, 64))
        each = max(1, total // kw["seqs"])
        kw["new_lo"], kw["new_hi"] = max(1, each // 2), each
        kw["old_lo"], kw["old_hi"] = (0, 0) if op == "read" else (0, _log(rng, 1, 3000))
        kw["norm"], kw["interleaved"], kw["window"] = rng.random() < 0.5, rng.random() < 0.3, 0
        if op == "write" and rng.random() < 0.3:
            kw["dtype"] = "f32"
    elif op == "token":
        total = _log(rng, 20, 250000 / per)   # cached positions of all sequences
        kw["seqs"] = max(1, min(_log(rng, 1, 256), total // 8))
        each = max(1, min(60000, total // kw["seqs"]))
        kw["old_lo"], kw["old_hi"] = each // 3, each
    else:
        each = _log(rng, 2, 2000)
        kw["seqs"] = max(1, min(_log(rng, 1, 24), 3000 // each))
        kw["new_lo"], kw["new_hi"] = max(1, each // 3), each
        old = _log(rng, 1, 1500)
        kw["old_lo"], kw["old_hi"] = rng.choice([(0, 0), (0, old), (old // 2, old)])
    return _case(op, heads, kv, hd, **kw)


def _lens(case):
    """[(cached before, new)] of each sequence: spread over the case's range, in no order; the longest is there."""
    r = random.Random("%(seqs)d %(new_lo)d %(new_hi)d %(old_lo)d %(old_hi)d" % case)
    got = [(r.randint(case["old_lo"], case["old_hi"]), r.randint(case["new_lo"], case["new_hi"])) for _ in range(case["seqs"])]
    got[r.randrange(len(got))] = (case["old_hi"], case["new_hi"])
    return got


# ---------------------------------------------------------------------------
# inputs

def _inputs(case, seed):
    """Everything that the case's pass reads, as torch tensors: values before they are quantised."""
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    H, K, hd, block, dt = case["heads"], case["kv_heads"], case["head_dim"], case["block"], DTYPES[case["dtype"]]
    lens = _lens(case)
    S = len(lens)
    new = torch.tensor([n for _, n in lens])
    end = torch.tensor([o + n for o, n in lens])
    need = (end + block - 1) // block
    n_blocks, most = int(need.sum()) + 3, int(need.max())
    # pages are handed out in no order, as after sequences have come and gone
    pages = torch.randperm(n_blocks, device=dev, generator=g)[: int(need.sum())].to(torch.int32)
    table = torch.zeros(S, most, dtype=torch.int32, device=dev)
    table[(torch.arange(most)[None] < need[:, None]).to(dev)] = pages
    T = int(new.sum())
    start = torch.cumsum(new, 0) - new
    seq = torch.repeat_interleave(torch.arange(S), new)
    pos = torch.arange(T) - start[seq] + (end - new)[seq]
    x = {"n_blocks": n_blocks, "table": table, "end": end.to(dev, torch.int32), "seq": seq.to(dev, torch.int32), "pos": pos.to(dev, torch.int32),
         "cu": torch.cat([start, torch.tensor([T])]).to(dev, torch.int32), "longest_new": int(new.max()), "scale": 1.0 / math.sqrt(hd)}

    def values(n):   # some channels of a head are much larger than the rest, as keys' are
        v = torch.randn(n, K, hd, device=dev, generator=g, dtype=torch.float32)
        big = 1.0 + 5.0 * (torch.rand(K, hd, device=dev, generator=g) > 0.96)
        return v.mul_(big)

    if case["op"] == "write":   # one projection's output: q, k and v of a token side by side
        qkv = torch.randn(T, (H + 2 * K) * hd, device=dev, generator=g)
        qkv[:, H * hd: (H + K) * hd] *= 1.0 + 5.0 * (torch.rand(K * hd, device=dev, generator=g) > 0.96)
        x["qkv"] = qkv.to(dt)
        x["inv_freq"] = (10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)).float()
        if case["norm"]:
            x["q_norm"], x["k_norm"] = (1.0 + 0.2 * torch.randn(hd, device=dev, generator=g) for _ in range(2))
    else:
        # the cache's content: keys and values of every position up to each sequence's end
        n = int(end.sum())
        x["all_seq"] = torch.repeat_interleave(torch.arange(S), end)
        first = torch.cumsum(end, 0) - end
        x["all_pos"] = (torch.arange(n) - first[x["all_seq"]]).to(dev, torch.int32)
        x["all_seq"] = x["all_seq"].to(dev, torch.int32)
        x["k"], x["v"] = values(n).half(), values(n).half()
        if case["op"] != "read":
            x["q"] = (torch.randn(T, H, hd, device=dev, generator=g) * 1.5).to(dt)
    return x


def _rows(x, seq, pos, block):
    """The cache row (page and place in it) of each token."""
    return x["table"][seq.long(), (pos // block).long()].long() * block + (pos % block).long()


def prepare(case, seed):
    x = _inputs(case, seed)
    H, K, hd, block = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    st = {"case": case, "x": x}
    if own:
        from chonklm_b200.kv_cache import QuantKvCache
        st["cache"] = QuantKvCache(H, K, hd, n_blocks=x["n_blocks"], block=block, v_bits=case["v_bits"])
        if case["op"] != "write":
            st["cache"].store(None, x.pop("k"), x.pop("v"), x["all_seq"], x["all_pos"], x["table"])
    else:
        n = x["n_blocks"] * block
        st["kc"], st["vc"] = (torch.zeros(n, K, hd, dtype=torch.int8, device="cuda") for _ in range(2))
        st["ks"], st["vs"] = (torch.zeros(n, K, hd // GROUP, dtype=torch.float16, device="cuda") for _ in range(2))
        if case["op"] != "write":
            at = _rows(x, x["all_seq"], x["all_pos"], block)
            st["kc"][at], st["ks"][at] = _quantise(x.pop("k").float(), 8)
            st["vc"][at], st["vs"][at] = _quantise(x.pop("v").float(), case["v_bits"])
    if case["op"] == "write":
        q, k, v = x["qkv"].split([H * hd, K * hd, K * hd], dim=1)
        st["q"], st["k"], st["v"] = q.unflatten(1, (H, hd)), k.unflatten(1, (K, hd)), v.unflatten(1, (K, hd))
    return st


# ---------------------------------------------------------------------------
# the plain form

def _quantise(x, bits):
    g = x.unflatten(-1, (-1, GROUP))
    if bits == 8:
        d, lo, hi = g.abs().amax(-1) / 127, -127, 127
    else:
        up, down = g.amax(-1), g.amin(-1)
        d, lo, hi = torch.where(up >= -down, up, down) / -8, -8, 7
    d = d.half()
    inv = torch.where(d == 0, 0.0, 1.0 / d.float())
    return torch.round(g * inv[..., None]).clamp(lo, hi).to(torch.int8).flatten(-2), d


def _values(codes, scales):
    return (codes.unflatten(-1, (-1, GROUP)).float() * scales.float()[..., None]).flatten(-2)


def _norm_rotate(x, w, angle, interleaved):
    x = x.float()
    if w is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) * w
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    a, b = a * c - b * s, a * s + b * c
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_write(st):
    case, x = st["case"], st["x"]
    angle = x["pos"][:, None].float() * x["inv_freq"]
    q = _norm_rotate(st["q"], x.get("q_norm"), angle, case["interleaved"])
    k = _norm_rotate(st["k"], x.get("k_norm"), angle, case["interleaved"])
    at = _rows(x, x["seq"], x["pos"], case["block"])
    st["kc"][at], st["ks"][at] = _quantise(k, 8)
    st["vc"][at], st["vs"][at] = _quantise(st["v"].float(), case["v_bits"])
    k, v = _plain_read(st, at, torch.float16)
    return q.to(torch.float16 if case["dtype"] == "f32" else DTYPES[case["dtype"]]), k, v


def _plain_read(st, at, dt):
    return _values(st["kc"][at], st["ks"][at]).to(dt), _values(st["vc"][at], st["vs"][at]).to(dt)


def _plain_attention(st):
    """q of each sequence padded to the longest; the sequence's pages gathered; products, a softmax under the mask, products."""
    case, x = st["case"], st["x"]
    H, K, hd, block = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    S, most = x["table"].shape
    G, n = H // K, x["longest_new"]
    at = (x["table"].long()[..., None] * block + torch.arange(block, device="cuda")).flatten(1)
    k = _values(st["kc"][at], st["ks"][at]).transpose(1, 2)                      # S, K, positions, hd
    place = x["seq"].long() * n + (torch.arange(len(x["seq"]), device="cuda") - x["cu"].long()[x["seq"].long()])
    q = torch.zeros(S * n, H, hd, device="cuda")
    q[place] = x["q"].float()
    q = q.view(S, n, K, G, hd).permute(0, 2, 3, 1, 4).reshape(S, K, G * n, hd)
    s = ((q @ k.transpose(2, 3)) * x["scale"]).view(S, K, G, n, -1)
    del k
    own_pos = torch.full((S * n,), -1, device="cuda", dtype=torch.long)
    own_pos[place] = x["pos"].long()
    own_pos = own_pos.view(S, n, 1)
    j = torch.arange(at.shape[1], device="cuda")
    seen = j <= own_pos
    if case["window"]:
        seen &= j > own_pos - case["window"]
    seen = seen[:, None, None]
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    v = _values(st["vc"][at], st["vs"][at]).transpose(1, 2)
    o = (e.view(S, K, G * n, -1) @ v).view(S, K, G, n, hd) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(S * n, H, hd)[place].to(x["q"].dtype)


def run(st):
    case, x = st["case"], st["x"]
    if not own:
        if case["op"] == "write":
            return _plain_write(st)
        if case["op"] == "read":
            return _plain_read(st, _rows(x, x["all_seq"], x["all_pos"], case["block"]), DTYPES[case["dtype"]])
        return _plain_attention(st)
    cache = st["cache"]
    if case["op"] == "write":
        q = cache.store(st["q"], st["k"], st["v"], x["seq"], x["pos"], x["table"], inv_freq=x["inv_freq"], q_norm=x.get("q_norm"),
                        k_norm=x.get("k_norm"), eps=1e-6, interleaved=case["interleaved"])
        return (q, *cache.load(x["seq"], x["pos"], x["table"], dtype=torch.float16))
    if case["op"] == "read":
        return cache.load(x["all_seq"], x["all_pos"], x["table"], dtype=DTYPES[case["dtype"]])
    if case["op"] == "token":
        return cache.attend(x["q"], x["end"], x["table"], scale=x["scale"], window=case["window"])
    return cache.attend_prompt(x["q"], x["cu"], x["end"], x["table"], scale=x["scale"], window=case["window"])


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits

def _seen(lens, window):
    """Positions that the new tokens see (summed), and cached positions that any of them sees."""
    pairs = rows = 0
    for old, n in lens:
        if window:
            full = max(0, min(n, old + n - window))          # tokens whose window is cut off
            short = n - full                                 # tokens that see all before them
            pairs += full * window + short * (old + 1) + short * (short - 1) // 2
            rows += min(old + n, window + n - 1)
        else:
            pairs += n * (old + 1) + n * (n - 1) // 2
            rows += old + n
    return pairs, rows


def work(case):
    H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
    row = K * (hd + hd * case["v_bits"] // 8 + 2 * 2 * hd // GROUP)       # a cached position: codes and scales
    lens = _lens(case)
    T = sum(n for _, n in lens)
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "write":   # projections in, q out, the rows written, and what they stand for read back
        return {"bytes": T * ((H + 2 * K) * hd * size + H * hd * 2 + 2 * row + 2 * K * hd * 2), "flops": T * (12 * (H + K) * hd + 6 * K * hd)}
    if case["op"] == "read":
        n = sum(o + k for o, k in lens)
        return {"bytes": n * (row + 2 * K * hd * size), "flops": n * 2 * K * hd}
    pairs, rows = _seen(lens, case["window"])
    return {"bytes": rows * row + T * 2 * H * hd * size, "flops": 4 * pairs * H * hd}


def _exact_stored(x, bits):
    """x (64 bits) after the cache: scale and codes by their definition."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    big = g.gather(-1, g.abs().argmax(-1, keepdim=True))
    d = (big.abs() / 127 if bits == 8 else big / -8).half().double()
    lim = (-127, 127) if bits == 8 else (-8, 7)
    c = torch.where(d == 0, torch.zeros_like(g), (g / torch.where(d == 0, torch.ones_like(d), d)).round().clamp(*lim))
    return (c * d).reshape(x.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        y = x["qkv"].double().view(-1, H + 2 * K, hd)
        out = []
        for part, w in ((y[:, :H], x.get("q_norm")), (y[:, H: H + K], x.get("k_norm"))):
            if w is not None:
                part = part * w.double() / (part.square().sum(-1, keepdim=True) / hd + 1e-6).sqrt()
            turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), x["pos"].double()[:, None] * x["inv_freq"].double())[:, None]
            if case["interleaved"]:
                part = torch.view_as_real(torch.view_as_complex(part.reshape(*part.shape[:-1], hd // 2, 2).contiguous()) * turn).flatten(-2)
            else:
                z = torch.complex(part[..., : hd // 2].contiguous(), part[..., hd // 2:].contiguous()) * turn
                part = torch.cat((z.real, z.imag), -1)
            out.append(part)
        return out[0], _exact_stored(out[1], 8), _exact_stored(y[:, H + K:], case["v_bits"])
    k, v = _exact_stored(x["k"].double(), 8), _exact_stored(x["v"].double(), case["v_bits"])
    if case["op"] == "read":
        return k, v
    pairs, _ = _seen(_lens(case), 0)
    if pairs * H * hd > 4e11:
        return None
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    at = row = 0
    for old, n in _lens(case):
        ks, vs = k[at: at + old + n], v[at: at + old + n]
        j = torch.arange(old + n, device="cuda")
        p = old + torch.arange(n, device="cuda")[:, None]
        hide = (j > p) | (j <= p - case["window"] if case["window"] else torch.zeros_like(j > p))
        for h in range(H):
            s = (x["q"][row: row + n, h].double() @ ks[:, h * K // H].T) * x["scale"]
            out[row: row + n, h] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ vs[:, h * K // H]
        at, row = at + old + n, row + n
    return out
