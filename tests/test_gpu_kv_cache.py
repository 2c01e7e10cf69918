"""The quantised paged key-value cache (chonklm_b200/kv_cache.py) against plain
implementations in 64 bits, at the sizes and masks where it can go wrong."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
LAYOUTS = [(9, 3, 64), (16, 8, 128), (4, 1, 256), (24, 2, 64), (10, 1, 128), (16, 1, 256), (3, 3, 128)]
EPS = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}   # half a step of the type, relative


def _cache(heads, kv, hd, n_blocks=64, block=16, v_bits=8):
    from chonklm_b200.kv_cache import QuantKvCache
    return QuantKvCache(heads, kv, hd, n_blocks=n_blocks, block=block, v_bits=v_bits)


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def _tables(lens, block, gen, extra=2):
    """Block table of sequences of the given lengths, blocks in no order; (table, blocks in all)."""
    need = [(n + block - 1) // block for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen).tolist()
    table = torch.full((len(lens), max(max(need), 1)), -7, dtype=torch.int32)   # entries past the end are never read
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), total


def _tokens(lens, start=None):
    seq = [i for i, n in enumerate(lens) for _ in range(n)]
    pos = [p + (start[i] if start else 0) for i, n in enumerate(lens) for p in range(n)]
    return _i32(seq), _i32(pos)


# ---------------------------------------------------------------------------
# write and read back

def _stored64(x, bits):
    """What the cache holds for x [..., hd] (float32 values as float64): the definition, its scale rounded to 16 bits and
    x times the 32-bit reciprocal of the scale rounded to the code."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(g).max(-1)
    if bits == 8:
        d = (top.astype(np.float32) / np.float32(127))
        lo, hi = -127, 127
    else:
        m = np.where(g.max(-1) >= -g.min(-1), g.max(-1), g.min(-1))
        d = m.astype(np.float32) / np.float32(-8)
        lo, hi = -8, 7
    d = d.astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d.astype(np.float32)).astype(np.float32)
    code = np.clip(np.rint(g.astype(np.float32) * inv[..., None]), lo, hi)
    return (code.astype(np.float64) * d.astype(np.float64)[..., None]).reshape(x.shape), np.abs(d.astype(np.float64))


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("layout", LAYOUTS[:4])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_stored_values_are_the_definition(layout, dtype, v_bits):
    """Without norm and rotation nothing but the quantisation happens: what is read back has to be its definition to the
    bit, zero groups, tiny groups and ties of the largest magnitude among them."""
    H, K, hd = layout
    g = torch.Generator().manual_seed(5)
    lens = [1, 37, 16]
    block = 32
    table, nb = _tables(lens, block, g)
    seq, pos = _tokens(lens)
    n = len(seq)
    k, v = (torch.randn(n, K, hd, generator=g) * torch.exp(torch.randn(n, K, 1, generator=g)) for _ in range(2))
    for t in (k, v):
        t[0, 0, :32] = 0.0                       # a zero group
        t[1, 0, :32] *= 1e-9                     # a scale that rounds to zero
        t[2, 0, 5], t[2, 0, 9] = 3.5, -3.5       # a tie of the largest magnitude
        t[3, 0, 32:64] *= 1e-5                   # a scale below the normal range
    k, v = k.to(dtype).cuda(), v.to(dtype).cuda()
    c = _cache(H, K, hd, nb, block, v_bits)
    assert c.store(None, k, v, seq, pos, table) is None
    c.check()
    kk, vv = c.load(seq, pos, table, dtype=F32)
    for got, x, bits in ((kk, k, 8), (vv, v, v_bits)):
        want, _ = _stored64(x.double().cpu().numpy(), bits)
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want.astype(np.float32).astype(np.float64))
    for dt in (F16, BF16):                       # the 16-bit forms are those values rounded once
        k16, v16 = c.load(seq, pos, table, dtype=dt)
        assert torch.equal(k16, kk.to(dt)) and torch.equal(v16, vv.to(dt))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_norm_rotation_and_quantised_keys(layout, interleaved, norm):
    """q out and the stored keys against the formulas in 64 bits.  The angle is the 32-bit product pos * inv_freq, as
    everywhere in the engine.  q: half a step of its type, and 2e-6 of the row's largest value for the 32-bit arithmetic
    (norm, sine, two products).  A stored key is within half a scale step of its value, plus that arithmetic and the
    clipped end (127 steps of a scale rounded to 11 bits)."""
    H, K, hd = layout
    g = torch.Generator().manual_seed(11)
    lens, start = [1, 45, 17], [1999, 0, 250]
    block = 64
    table, nb = _tables([a + b for a, b in zip(lens, start)], block, g)
    seq, pos = _tokens(lens, start)
    n = len(seq)
    for dtype in (F32, F16, BF16):
        q, k, v = (torch.randn(n, h, hd, generator=g).to(dtype) for h in (H, K, K))
        qw, kw = (1 + 0.3 * torch.randn(hd, generator=g) for _ in range(2))
        f = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float()
        c = _cache(H, K, hd, nb, block)
        out = c.store(q.cuda(), k.cuda(), v.cuda(), seq, pos, table, inv_freq=f.cuda(), q_norm=qw.cuda() if norm else None,
                      k_norm=kw.cuda() if norm else None, eps=1e-5, interleaved=interleaved)
        kk, _ = c.load(seq, pos, table, dtype=F32)
        c.check()
        a = (pos.cpu().float()[:, None] * f).double()[:, None]

        def turn(x, w):
            x = x.double()
            if norm:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()
            if interleaved:
                x0, x1 = x[..., 0::2], x[..., 1::2]
                return torch.stack((x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()), -1).flatten(-2)
            x0, x1 = x.chunk(2, -1)
            return torch.cat((x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()), -1)

        wq, wk = turn(q, qw), turn(k, kw)
        assert out.dtype is (F16 if dtype is F32 else dtype)
        tol = EPS[out.dtype] * wq.abs() + 2e-6 * wq.abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert ((out.double().cpu() - wq).abs() <= tol).all()
        top = wk.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
        tol = (top / 254 * (1 + 2.0 ** -10) + top * (2.0 ** -11 + 2e-6)).expand(-1, -1, -1, 32).flatten(-2)
        assert ((kk.double().cpu() - wk).abs() <= tol).all()


def test_strides_alignment_and_padding():
    """Rows of a fused projection, a head-major tensor, rows off the vector alignment, padding tokens, an output given by
    the caller, a stream of the caller's: the same bits as plain contiguous rows on the current stream."""
    H, K, hd, n, block = 6, 2, 128, 19, 16
    g = torch.Generator().manual_seed(3)
    table, nb = _tables([n], block, g)
    seq, pos = _tokens([n])
    q, k, v = (torch.randn(n, h, hd, generator=g).half().cuda() for h in (H, K, K))
    f = torch.rand(hd // 2, generator=g).cuda()
    ref = _cache(H, K, hd, nb, block)
    want = ref.store(q, k, v, seq, pos, table, inv_freq=f)
    kw, vw = ref.load(seq, pos, table)

    def same(q2, k2, v2, seq2=seq, out=None, stream=None):
        c = _cache(H, K, hd, nb, block)
        got = c.store(q2, k2, v2, seq2, pos, table, inv_freq=f, out=out, stream=stream)
        lo = tuple(torch.full((K, n, hd), 9.0, device="cuda", dtype=F16).transpose(0, 1) for _ in range(2))   # head-major
        k3, v3 = c.load(seq2, pos, table, out=lo, stream=stream)
        c.check(stream)
        return got, k3, v3

    fused = torch.zeros(n, (H + 2 * K) * hd + 1, dtype=F16, device="cuda")
    for off in (0, 1):   # off 1: rows and strides off every vector alignment
        part = fused[:, off: off + (H + 2 * K) * hd].unflatten(1, (H + 2 * K, hd))
        part[:, :H], part[:, H: H + K], part[:, H + K:] = q, k, v
        got, k3, v3 = same(part[:, :H], part[:, H: H + K], part[:, H + K:])
        assert torch.equal(got, want) and torch.equal(k3, kw) and torch.equal(v3, vw)
    odd = torch.zeros(H * n * hd + 1, dtype=F16, device="cuda")[1:].view(H, n, hd).transpose(0, 1)
    got, k3, v3 = same(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, out=odd)
    assert got is odd and torch.equal(odd, want) and torch.equal(k3, kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, k3, v3 = same(q, k, v, stream=s.cuda_stream, out=torch.empty_like(q))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(k3, kw) and torch.equal(v3, vw)
    pad = seq.clone()
    pad[4] = -1
    got, k3, v3 = same(q, k, v, seq2=pad)
    live = torch.arange(n, device="cuda") != 4
    assert torch.equal(got, want) and torch.equal(k3[live], kw[live]) and not k3[4].any() and not v3[4].any()


def test_not_finite_groups_read_as_nan():
    K, hd = 2, 64
    k = torch.randn(3, K, hd).cuda()
    k[0, 0, 3], k[1, 1, 40] = float("nan"), float("-inf")
    for bits in (8, 4):
        c = _cache(2, K, hd, 4, 16, bits)
        seq, pos = _tokens([3])
        table = _i32([[2]])
        c.store(None, k, k, seq, pos, table)
        for got in c.load(seq, pos, table):
            bad = torch.isnan(got)
            want = torch.zeros_like(bad)
            want[0, 0, :32] = want[1, 1, 32:] = True
            assert torch.equal(bad, want)


# ---------------------------------------------------------------------------
# attention

def _ref_attention(q, k, v, lens, news, scale, window):
    """64 bits: (out, sum p|v|, largest sum |q||k| scale) of each query row.  k, v: per sequence [len, K, hd]."""
    outs, mags, tops, row = [], [], [], 0
    for i, (length, n) in enumerate(zip(lens, news)):
        qi = q[row: row + n].double()
        row += n
        ki, vi = k[i].double(), v[i].double()
        G = qi.shape[1] // ki.shape[1] if length else 1
        for t in range(n):
            end = length - n + t + 1
            lo = max(0, end - window) if window else 0
            if end <= lo:
                outs.append(torch.zeros_like(qi[t])); mags.append(torch.zeros_like(qi[t]))
                tops.append(torch.zeros(qi.shape[1], 1, dtype=torch.float64, device=q.device))
                continue
            kk, vv = (x[lo:end].repeat_interleave(G, 1) for x in (ki, vi))
            s = torch.einsum("hd,phd->hp", qi[t], kk) * scale
            p = torch.softmax(s, -1)
            outs.append(torch.einsum("hp,phd->hd", p, vv))
            mags.append(torch.einsum("hp,phd->hd", p, vv.abs()))
            tops.append((torch.einsum("hd,phd->hp", qi[t].abs(), kk.abs()) * abs(scale)).amax(-1, keepdim=True))
    return torch.stack(outs), torch.stack(mags), torch.stack(tops)


def _close(got, want, mag, top, key_step):
    """Operands in 16 bits, sums in 32.  The probability and the value are each rounded once to 11 bits, the output to
    its type; a score is off by key_step (0 where the key codes enter the product as they are, half an fp16 step where
    code * scale is rounded) and 2^-20 of the magnitudes it sums, which moves every probability by at most that factor."""
    ds = (key_step + 2.0 ** -20) * top
    tol = (2 * 2.0 ** -11 + 2 * ds) * mag + EPS[got.dtype] * want.abs() + 1e-6
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off - tol).max()


def _filled(H, K, hd, lens, block, v_bits, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    table, nb = _tables(lens, block, g)
    seq, pos = _tokens(lens)
    c = _cache(H, K, hd, nb, block, v_bits)
    k, v = (torch.randn(len(seq), K, hd, generator=g).mul_(gain).cuda() for _ in range(2))
    c.store(None, k, v, seq, pos, table)
    kk, vv = c.load(seq, pos, table, dtype=F32)   # attention reads these, so quantisation is no error of its own
    return c, table, kk.split(lens), vv.split(lens), g


TOKEN_LENS = [[1], [0], [15], [16], [17], [5, 0, 33, 1, 250], [1000], [128, 127, 129, 0, 0, 7], [4097], list(range(0, 300))]


@pytest.mark.parametrize("window", [0, 1, 16, 50])
@pytest.mark.parametrize("lens", TOKEN_LENS, ids=[str(len(x)) + "x" + str(max(x)) for x in TOKEN_LENS])
def test_token_attention_lengths(lens, window):
    H, K, hd, block = 6, 2, 64, 32
    c, table, k, v, g = _filled(H, K, hd, lens, block, 8, seed=len(lens))
    q = torch.randn(len(lens), H, hd, generator=g).mul_(2).half().cuda()
    got = c.attend(q, _i32(lens), table, window=window)
    c.check()
    want, mag, top = _ref_attention(q, k, v, lens, [1] * len(lens), 1 / math.sqrt(hd), window)
    _close(got, want, mag, top, 0)
    for i, n in enumerate(lens):
        if n == 0:
            assert not got[i].any()
    assert torch.equal(got, c.attend(q, _i32(lens), table, window=window))   # no order of atomics in the result


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_token_attention_layouts(layout, block, dtype, v_bits):
    H, K, hd = layout
    lens = [70, 301, 2, 555]
    c, table, k, v, g = _filled(H, K, hd, lens, block, v_bits, seed=1)
    big = torch.randn(H, len(lens), hd, generator=g).mul_(3).to(dtype).cuda().transpose(0, 1)   # head-major
    out = torch.full((len(lens), H + 2, hd), 7.0, dtype=dtype, device="cuda")
    got = c.attend(big, _i32(lens), table, scale=0.11, window=333, out=out[:, 1: H + 1])
    c.check()
    want, mag, top = _ref_attention(big, k, v, lens, [1] * len(lens), 0.11, 333)
    _close(got, want, mag, top, 0)
    assert (out[:, 0] == 7).all() and (out[:, -1] == 7).all()


def test_token_attention_rows_of_the_table():
    """`seq` names the table's row of each query; the same row may be read twice."""
    lens = [40, 333, 90]
    c, table, k, v, g = _filled(4, 2, 128, lens, 16, 8)
    order = [2, 0, 2, 1, 1]
    q = torch.randn(5, 4, 128, generator=g).half().cuda()
    ln = [90, 40, 33, 333, 100]                  # shorter than what is cached: only the first positions
    got = c.attend(q, _i32(ln), table, seq=_i32(order))
    c.check()
    want, mag, top = _ref_attention(q, [k[i][:n] for i, n in zip(order, ln)], [v[i][:n] for i, n in zip(order, ln)], ln,
                                    [1] * 5, 1 / math.sqrt(128), 0)
    _close(got, want, mag, top, 0)


@pytest.mark.parametrize("window", [0, 40, 1600])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256), (24, 1, 128)])
def test_token_attention_by_list(layout, window):
    """Block tables too wide for a CTA per unit: ragged lengths, empty queries among them, cut into shares and joined; as
    many queries as two launches take, by table row and by `seq`."""
    H, K, hd = layout
    lens = [1500, 0, 3, 700, 0, 0, 64, 1100, 1, 2100]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=21)
    q = torch.randn(len(lens), H, hd, generator=g).mul_(2).half().cuda()
    got = c.attend(q, _i32(lens), table, window=window)
    want, mag, top = _ref_attention(q, k, v, lens, [1] * len(lens), 1 / math.sqrt(hd), window)
    _close(got, want, mag, top, 0)
    assert torch.equal(got, c.attend(q, _i32(lens), table, window=window))
    n = 1100
    order = torch.arange(n) % len(lens)
    many = c.attend(q[order.cuda()].contiguous(), _i32(torch.tensor(lens)[order]), table, window=window, seq=_i32(order))
    wide = c.attend(q[order.cuda()].contiguous(), _i32(torch.tensor(lens)[order]), table[order.cuda()].contiguous(), window=window)
    c.check()
    assert torch.equal(many, wide)
    _close(many[-20:], *(t[order[-20:].cuda()] for t in (want, mag, top)), 0)   # the second launch's, shared out otherwise


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_token_attention_of_wide_tables(layout, window, v_bits):
    """The same lengths under tables of several widths: few and many CTAs a unit, and shares of a list (the widest, where
    no window bounds what can be visible).  Entries past a sequence's end are never read."""
    H, K, hd = layout
    lens = [1500, 0, 3, 700, 64, 1, 2100]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, v_bits, seed=22)
    q = torch.randn(len(lens), H, hd, generator=g).mul_(2).half().cuda()
    want, mag, top = _ref_attention(q, k, v, lens, [1] * len(lens), 1 / math.sqrt(hd), window)
    for blocks in (table.shape[1], 300, 600, 1100):
        wide = torch.full((len(lens), blocks), -7, dtype=torch.int32, device="cuda")
        wide[:, : table.shape[1]] = table
        got = c.attend(q, _i32(lens), wide, window=window)
        c.check()
        _close(got, want, mag, top, 0)
        assert torch.equal(got, c.attend(q, _i32(lens), wide, window=window))


PROMPTS = [([1], [1]), ([5], [5]), ([127], [127]), ([129], [129]), ([300], [43]), ([513], [513]),
           ([64, 1, 257, 40, 700], [64, 1, 130, 3, 65]), ([33, 20], [0, 20]), ([16] * 40, [7] * 40)]


@pytest.mark.parametrize("window", [0, 1, 70])
@pytest.mark.parametrize("case", PROMPTS, ids=[str(max(a)) + "-" + str(sum(b)) for a, b in PROMPTS])
@pytest.mark.parametrize("layout", [(9, 3, 64), (16, 8, 128), (4, 1, 256), (5, 1, 128)])
def test_prompt_attention(layout, case, window):
    H, K, hd = layout
    lens, news = case
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=2)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).to(BF16 if hd == 128 else F16).cuda()
    cu = _i32(np.concatenate([[0], np.cumsum(news)]))
    got = c.attend_prompt(q, cu, _i32(lens), table, window=window)
    c.check()
    want, mag, top = _ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), window)
    _close(got, want, mag, top, 2.0 ** -11)
    assert torch.equal(got, c.attend_prompt(q, cu, _i32(lens), table, window=window))


@pytest.mark.parametrize("window", [0, 900])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
def test_prompt_attention_over_a_long_cache(layout, window):
    """Few rows on long caches: the positions are split over CTAs and joined; rows and sequences that see nothing, and
    parts of a split that nothing of a tile falls into."""
    H, K, hd = layout
    lens, news = [3000, 17, 0, 1500, 5], [33, 17, 2, 1, 9]
    c, table, k, v, g = _filled(H, K, hd, lens, 32, 8, seed=6)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).half().cuda()
    cu = _i32(np.concatenate([[0], np.cumsum(news)]))
    got = c.attend_prompt(q, cu, _i32(lens), table, window=window)
    c.check()
    want, mag, top = _ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), window)
    _close(got, want, mag, top, 2.0 ** -11)
    assert torch.equal(got, c.attend_prompt(q, cu, _i32(lens), table, window=window))


def test_prompt_attention_of_more_sequences_than_a_launch_takes():
    H, K, hd, S = 4, 2, 64, 1090
    lens = [1 + i % 37 for i in range(S)]
    news = [min(n, 1 + i % 5) for i, n in enumerate(lens)]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=12)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).half().cuda()
    cu = np.concatenate([[0], np.cumsum(news)])
    got = c.attend_prompt(q, _i32(cu), _i32(lens), table)
    c.check()
    for part in (slice(0, 40), slice(1010, S)):
        rows = slice(int(cu[part.start]), int(cu[part.stop]))
        want, mag, top = _ref_attention(q[rows], k[part], v[part], lens[part], news[part], 1 / math.sqrt(hd), 0)
        _close(got[rows], want, mag, top, 2.0 ** -11)


@pytest.mark.parametrize("n", [1, 64, 65, 128, 129, 192])
@pytest.mark.parametrize("layout", [(6, 3, 64), (16, 8, 128), (4, 1, 256)])
def test_prompt_attention_of_many_short_sequences(layout, n):
    """A few position tiles a CTA, on every SM at once and many times over: the roles of a CTA hand over from the first
    tile to the last without a long run in between, and every pass gives the same bits."""
    H, K, hd = layout
    lens = [n] * 120
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=n)
    q = torch.randn(sum(lens), H, hd, generator=g).mul_(2).half().cuda()
    cu, ln = _i32(np.arange(121) * n), _i32(lens)
    first = c.attend_prompt(q, cu, ln, table)
    c.check()
    want, mag, top = _ref_attention(q[: 2 * n], k[:2], v[:2], lens[:2], lens[:2], 1 / math.sqrt(hd), 0)
    _close(first[: 2 * n], want, mag, top, 2.0 ** -11)
    for _ in range(200):
        again = c.attend_prompt(q, cu, ln, table)
    c.check()
    assert torch.equal(first, again)


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_prompt_attention_layouts(layout, block, v_bits):
    H, K, hd = layout
    lens, news = [150, 290], [150, 77]
    c, table, k, v, g = _filled(H, K, hd, lens, block, v_bits, seed=4)
    q = torch.randn(H, sum(news), hd, generator=g).mul_(2).half().cuda().transpose(0, 1)
    got = c.attend_prompt(q, _i32([0, 150, 227]), _i32(lens), table, window=100)
    c.check()
    want, mag, top = _ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), 100)
    _close(got, want, mag, top, 2.0 ** -11)


def test_prompt_rows_before_the_sequence_are_empty():
    """More query rows than cached positions: the first rows have no position to see and are zero, as are rows of a
    sequence without any."""
    c, table, k, v, g = _filled(4, 2, 64, [3, 20], 16, 8)
    q = torch.randn(5 + 4, 4, 64, generator=g).half().cuda()
    got = c.attend_prompt(q, _i32([0, 5, 9]), _i32([3, 0]), table)
    c.check()
    want, mag, top = _ref_attention(q, [k[0], k[1][:0]], [v[0], v[1][:0]], [3, 0], [5, 4], 0.125, 0)
    _close(got, want, mag, top, 2.0 ** -11)
    assert not got[:2].any() and not got[5:].any() and got[2:5].any()


@pytest.mark.parametrize("prompt", [False, True])
def test_masked_places_never_reach_the_result(prompt):
    """NaN and infinite groups in positions past the length or before the window, in blocks and tiles that are read."""
    H, K, hd, n = 4, 2, 64, 77
    for v_bits in (8, 4):
        c, table, k, v, g = _filled(H, K, hd, [96], 32, v_bits)
        bad = torch.full((96, K, hd), float("nan"), device="cuda")
        at = [p for p in range(96) if p >= n or p < n - 40]
        c.store(None, bad[: len(at)], bad[: len(at)], _i32([0] * len(at)), _i32(at), table)
        if prompt:
            q = torch.randn(1, H, hd, generator=g).half().cuda()
            got = c.attend_prompt(q, _i32([0, 1]), _i32([n]), table, window=40)
        else:
            q = torch.randn(1, H, hd, generator=g).half().cuda()
            got = c.attend(q, _i32([n]), table, window=40)
        want, mag, top = _ref_attention(q, [k[0][:n]], [v[0][:n]], [n], [1], 0.125, 40)
        _close(got, want, mag, top, 2.0 ** -11)
        c.store(None, bad[:1], bad[:1], _i32([0]), _i32([n - 1]), table)   # a visible one does
        assert torch.isnan(c.attend(q, _i32([n]), table, window=40)).all()


def test_large_scores_and_repeated_maxima():
    """Scores far apart (a softmax of one position), rising along the sequence (the maximum grows in every tile), and all
    alike (a mean over the positions)."""
    H, K, hd, n = 2, 1, 128, 600
    g = torch.Generator().manual_seed(9)
    table, nb = _tables([n], 16, g)
    seq, pos = _tokens([n])
    v = torch.randn(n, K, hd, generator=g).cuda()
    base = torch.randn(1, K, hd, generator=g)
    for gain in (torch.arange(n)[:, None, None] / 20.0, -torch.arange(n)[:, None, None] / 20.0, torch.ones(n, 1, 1)):
        c = _cache(H, K, hd, nb, 16)
        c.store(None, (base * gain).cuda(), v, seq, pos, table)
        kk, vv = c.load(seq, pos, table, dtype=F32)
        q = base.expand(1, H, hd).half().cuda()
        for got in (c.attend(q, _i32([n]), table), c.attend_prompt(q, _i32([0, 1]), _i32([n]), table)):
            want, mag, top = _ref_attention(q, [kk], [vv], [n], [1], 1 / math.sqrt(hd), 0)
            _close(got, want, mag, top, 2.0 ** -11)


def test_offsets_past_32_bits():
    """A pool of more than 4 GB whose last blocks are used."""
    H, K, hd, block = 8, 8, 128, 128
    nb = (9 << 30) // 2 // (block * K * (2 * hd + 4 * hd // 32))
    c = _cache(H, K, hd, nb, block)
    assert c.nbytes > 1 << 32
    lens = [200]
    table = _i32([[nb - 1, nb - 2]])
    seq, pos = _tokens(lens)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(200, K, hd, generator=g).cuda() for _ in range(2))
    c.store(None, k, v, seq, pos, table)
    kk, vv = c.load(seq, pos, table, dtype=F32)
    q = torch.randn(3, H, hd, generator=g).half().cuda()
    got = c.attend(q[:1], _i32(lens), table)
    gotp = c.attend_prompt(q, _i32([0, 3]), _i32(lens), table)
    c.check()
    assert (kk - k).abs().max() < 0.04
    _close(got, *_ref_attention(q[:1], [kk], [vv], lens, [1], 1 / math.sqrt(hd), 0), 0)
    _close(gotp, *_ref_attention(q, [kk], [vv], lens, [3], 1 / math.sqrt(hd), 0), 2.0 ** -11)


def test_nothing_to_do():
    c = _cache(4, 2, 64, 4)
    e = _i32([])
    table = torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    z = torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    q = torch.zeros(0, 4, 64, dtype=F16, device="cuda")
    assert c.store(q, z, z, e, e, table).shape == q.shape
    assert c.load(e, e, table)[0].shape == z.shape
    assert c.attend(q, e, table).shape == q.shape
    assert c.attend_prompt(q, _i32([0]), e, table).shape == q.shape
    c.check()


def test_captured_in_a_graph():
    """A decode step of the cache (write, attention) captured once and replayed on new inputs and lengths."""
    H, K, hd, block = 4, 2, 64, 16
    lens = [5, 90]
    c, table, k, v, g = _filled(H, K, hd, [96, 96], block, 8)
    q, kn, vn = (torch.randn(2, h, hd, generator=g).half().cuda() for h in (H, K, K))
    seq, pos, length = _i32([0, 1]), _i32([4, 89]), _i32(lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(c.store(q, kn, vn, seq, pos, table), length, table)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend(c.store(q, kn, vn, seq, pos, table), length, table)
    for step in range(3):
        q.copy_(torch.randn(2, H, hd, generator=g))
        pos.add_(1)
        length.add_(1)
        graph.replay()
        want = c.attend(q, length, table)
        assert torch.equal(out, want)
    c.check()


# ---------------------------------------------------------------------------
# refusals

def test_refuses_geometry():
    from chonklm_b200 import _lib
    for args, word in [((4, 2, 96, 4), "head_dim"), ((5, 2, 64, 4), "heads"), ((0, 0, 64, 4), "heads"), ((4, 2, 64, 0), "blocks")]:
        with pytest.raises(_lib.CkError, match=word):
            _cache(*args)
    with pytest.raises(_lib.CkError, match="positions"):
        _cache(4, 2, 64, 4, 24)
    with pytest.raises(_lib.CkError, match="bits"):
        _cache(4, 2, 64, 4, 16, 5)
    with pytest.raises(_lib.CkError):
        _cache(64, 64, 256, 1 << 24, 128)        # more than the device has


def test_refuses_arguments():
    from chonklm_b200 import _lib
    c = _cache(4, 2, 64, 4)
    table = _i32([[0, 1]])
    one, q = _i32([1]), torch.zeros(1, 4, 64, dtype=F16, device="cuda")
    k = torch.zeros(1, 2, 64, dtype=F16, device="cuda")
    bad = [lambda: c.attend(q.float(), one, table), lambda: c.attend(q[:, :3], one, table), lambda: c.attend(q.cpu(), one, table),
           lambda: c.attend(q, one.long(), table), lambda: c.attend(q, one, table.long()),
           lambda: c.attend(torch.zeros(1, 4, 128, dtype=F16, device="cuda")[..., ::2], one, table),
           lambda: c.attend(q, _i32([1, 2]), table), lambda: c.attend_prompt(q, _i32([]), _i32([]), table),
           lambda: c.store(q, k, k, one, one, table, inv_freq=torch.zeros(64, device="cuda")),
           lambda: c.store(q, k, k.double(), one, one, table), lambda: c.store(None, k, k, one, one, table, out=q),
           lambda: c.store(q, k, k, one, one, table, q_norm=torch.zeros(64)),
           lambda: c.load(one, one, table, dtype=torch.float64)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    two = torch.zeros(2, 4, 64, dtype=F16, device="cuda")
    for f, word in [(lambda: c.attend(q, one, table, window=-1), "window"), (lambda: c.attend(q, one, table, scale=float("nan")), "scale"),
                    (lambda: c.attend(two, _i32([1, 1]), table), "rows of the block table"),
                    (lambda: c.attend_prompt(two, _i32([0, 1, 2]), _i32([1, 1]), table), "rows of the block table"),
                    (lambda: c.attend(q, one, table, out=q[:, :1].expand(1, 4, 64)), "overlap"),
                    (lambda: c.store(q, k, k, one, one, table, q_norm=torch.zeros(64, device="cuda"), eps=-1.0), "eps")]:
        with pytest.raises(_lib.CkError, match=word):
            f()
    c.check()


def test_device_reports_what_is_out_of_range():
    """Places that do not exist are skipped, reported once by check(), and nothing else changes."""
    from chonklm_b200 import _lib
    c = _cache(4, 2, 64, 4)
    table = _i32([[0, 1], [9, 2]])
    k = torch.randn(1, 2, 64).half().cuda()
    q = torch.randn(2, 4, 64).half().cuda()
    for seq, pos, word in [(5, 0, "sequence"), (0, 32, "position"), (0, -3, "position"), (1, 0, "pool")]:
        c.store(None, k, k, _i32([seq]), _i32([pos]), table)
        with pytest.raises(_lib.CkError, match=word):
            c.check()
        got = c.load(_i32([seq]), _i32([pos]), table)
        assert not got[0].any()
        with pytest.raises(_lib.CkError, match=word):
            c.check()
    c.store(None, k, k, _i32([0]), _i32([0]), table)
    c.check()
    for ln, word in [([1, 33], "length"), ([1, 3], "pool")]:
        for f in (lambda: c.attend(q, _i32(ln), table), lambda: c.attend_prompt(q, _i32([0, 1, 2]), _i32(ln), table)):
            got = f()
            with pytest.raises(_lib.CkError, match=word):
                c.check()
            assert torch.isfinite(got[0]).all() and not got[1].any()
    c.attend(q[:1], _i32([1]), table, seq=_i32([7]))
    with pytest.raises(_lib.CkError, match="sequence"):
        c.check()


# Independent rounding to 8 bits: a step of 1/127 of a group's largest value (2.2 of 32 normal values, on average) is an
# error of 0.005 of a value's size at 8 bits, 0.08 at 4; averaged by the attention it stays below twice that.
@pytest.mark.parametrize("v_bits,tol", [(8, 0.01), (4, 0.16)])
def test_example_runs_all_operators_together(v_bits, tol, capsys):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import quantised_cache
    assert quantised_cache.main(["--v-bits", str(v_bits), "--steps", "4"]) < tol
    assert "out of the cache" in capsys.readouterr().out
