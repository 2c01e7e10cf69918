"""The quantised paged key-value cache at its edges: streams, windows without
end, tables with gaps, rows of no sequence, scores of every size."""
import math

import numpy as np
import pytest
import torch

from conftest import tiny_model
from test_gpu_kv_cache import BF16, EPS, F16, F32, _cache, _close, _filled, _i32, _ref_attention, _tables, _tokens

pytestmark = pytest.mark.gpu


def _cu(news):
    return _i32(np.concatenate([[0], np.cumsum(news)]))


def test_default_outputs_belong_to_the_given_stream():
    """A call on a stream of the caller's makes its outputs there: memory that work still pending on the current stream
    writes is not handed out."""
    H, K, hd, lens = 6, 2, 128, [40, 33]
    c, table, _, _, g = _filled(H, K, hd, lens, 16, 8)
    seq, pos = _tokens(lens)
    q = torch.randn(sum(lens), H, hd, generator=g).half().cuda()
    k, v = (torch.randn(sum(lens), K, hd, generator=g).half().cuda() for _ in range(2))
    s = torch.cuda.Stream()
    calls = [lambda st: (c.store(q, k, v, seq, pos, table, stream=st),), lambda st: c.load(seq, pos, table, stream=st),
             lambda st: (c.attend(q[: len(lens)], _len, table, stream=st),),
             lambda st: (c.attend_prompt(q, _row, _len, table, stream=st),)]
    _len, _row = _i32(lens), _cu(lens)
    for call in calls:
        want = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        spare = [torch.empty_like(t) for t in want for _ in range(4)]
        torch.cuda._sleep(20_000_000)            # some 10 ms, then the current stream writes its memory
        for t in spare:
            t.fill_(7.0)
        del t, spare                             # back to the allocator, the writes still pending
        got = call(s.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for t in got:
            t.record_stream(torch.cuda.current_stream())
    c.check()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 20])
def test_a_window_wider_than_any_sequence_is_none(window):
    """Rows that lie before their sequence among them."""
    for H, K, hd in ((4, 2, 64), (4, 1, 256)):
        c, table, k, v, g = _filled(H, K, hd, [3, 20], 16, 8)
        q = torch.randn(9 + 4, H, hd, generator=g).half().cuda()
        cu, ln = _cu([9, 4]), _i32([3, 20])
        got = c.attend_prompt(q, cu, ln, table, window=window)
        assert torch.equal(got, c.attend_prompt(q, cu, ln, table))
        want, mag, top = _ref_attention(q, k, v, [3, 20], [9, 4], 1 / math.sqrt(hd), 0)
        _close(got, want, mag, top, 2.0 ** -11)
        assert torch.equal(c.attend(q[:2], ln, table, window=window), c.attend(q[:2], ln, table))
        c.check()


@pytest.mark.parametrize("queries", [80, 1])
@pytest.mark.parametrize("lowest", [60, 100])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_small_probabilities_beside_a_large_one(hd, lowest, queries):
    """131072 positions some 20 to 26 octaves (lowest 100: 25 to 26) below the first one's, whose value is zero: the
    output is what the small probabilities add up to.  Key codes, scales (2^-3) and q are chosen so that code * scale and
    the scores are exact.  A probability is rounded to 11 bits, or to half a step of the smallest fp16 numbers: 2^-25,
    kept times 2^8, of the reference maximum, which may lie 2^7 above the largest probability; so 2^-33 each, in the
    outputs' sum and in the sum that divides it.  80 queries of one sequence are not split over its positions, 1 is."""
    n, block = 131072, 128
    g = torch.Generator().manual_seed(hd + lowest)
    k = torch.zeros(n, 1, hd)
    k[:, 0, 1::32] = 127 / 8                     # each group's largest value: scale 1 / 8, where q is zero
    k[:, 0, 0] = -torch.randint(lowest, 108, (n,), generator=g) / 8
    k[0, 0, 0] = 100 / 8
    v = 0.5 + 0.5 * torch.rand(n, 1, hd, generator=g)
    v[0] = 0
    table, nb = _tables([n], block, g)
    seq, pos = _tokens([n])
    c = _cache(1, 1, hd, nb, block)
    c.store(None, k.cuda(), v.cuda(), seq, pos, table)
    kk, vv = c.load(seq, pos, table, dtype=F32)
    assert torch.equal(kk.cpu(), k)
    q = torch.zeros(queries, 1, hd, dtype=F16, device="cuda")
    q[:, 0, 0] = 1
    scale = float(np.float32(math.log(2)))       # a score is its exponent of two
    want, mag, top = _ref_attention(q[:1], [kk], [vv], [n], [1], scale, 0)
    table = table.expand(queries, -1).contiguous()
    ln = _i32([n] * queries)
    for got in (c.attend_prompt(q, _cu([1] * queries), ln, table, scale=scale), c.attend(q, ln, table, scale=scale)):
        tol = (2 * 2.0 ** -11 + 2 * 2.0 ** -20 * top) * mag + 2 * n * 2.0 ** -33 * vv.abs().max().item() + EPS[F16] * want.abs()
        assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()
    c.check()


def _far_apart(hd, gain):
    """A cache of 200 positions and a bf16 query whose scores are so large, and so far from each other (2^-9 of the
    magnitudes they sum, which 16-bit operands cannot turn round), that the softmax is one position's."""
    n = 200
    g = torch.Generator().manual_seed(hd)
    table, nb = _tables([n], 16, g)
    seq, pos = _tokens([n])
    k, v = (torch.randn(n, 1, hd, generator=g).mul_(0.01).cuda() for _ in range(2))
    c = _cache(2, 1, hd, nb, 16)
    c.store(None, k, v, seq, pos, table)
    kk, vv = c.load(seq, pos, table, dtype=F32)
    q = (torch.randn(1, 2, hd, generator=g) * gain).to(BF16).cuda()
    s = torch.einsum("nhd,pkd->hp", q.double(), kk.double())
    first, second = s.topk(2).values.unbind(1)
    size = torch.einsum("nhd,pkd->hp", q.double().abs(), kk.double().abs()).amax(1)
    assert ((first - second) > 2.0 ** -9 * size).all() and ((first - second) * 0.05 > 64).all()
    return c, table, q, _i32([n]), vv[s.argmax(1), 0].double()[None]


def _one_value(got, want):
    """A value rounded to 11 bits as an operand, then to the output's type."""
    assert ((got.double() - want).abs() <= (EPS[BF16] + 2.0 ** -10) * want.abs() + 1e-6).all()


GAINS = [2.0 ** 24, 2.0 ** 40, 2.0 ** 100, 2.0 ** 114, 2.0 ** 124]


@pytest.mark.parametrize("gain", GAINS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_very_large_queries_of_one_token(hd, gain):
    c, table, q, ln, want = _far_apart(hd, gain)
    _one_value(c.attend(q, ln, table, scale=0.05), want)
    wide = torch.zeros(1, 40000, dtype=torch.int32, device="cuda")       # by list
    wide[:, : table.shape[1]] = table
    _one_value(c.attend(q, ln, wide, scale=0.05), want)
    c.check()


@pytest.mark.parametrize("gain", GAINS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_very_large_queries_in_prompts(hd, gain):
    """With a row that lies before the sequence beside the live one, and with the positions split over CTAs (a table wide
    enough for it)."""
    c, table, q, ln, want = _far_apart(hd, gain)
    _one_value(c.attend_prompt(q, _i32([0, 1]), ln, table, scale=0.05), want)
    wide = torch.zeros(1, 40000, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    _one_value(c.attend_prompt(q, _i32([0, 1]), ln, wide, scale=0.05), want)
    many = q.expand(201, -1, -1).contiguous()
    got = c.attend_prompt(many, _i32([0, 201]), ln, table, scale=0.05)
    assert not got[0].any()
    _one_value(got[-1:], want)
    assert torch.isfinite(got).all()
    c.check()


@pytest.mark.parametrize("gain", [2.0 ** 10, 2.0 ** 20] + GAINS)
def test_equal_scores_of_any_size_weigh_alike(gain):
    n, hd = 300, 128
    g = torch.Generator().manual_seed(1)
    table, nb = _tables([n], 16, g)
    seq, pos = _tokens([n])
    k, v = torch.randn(1, 1, hd, generator=g).expand(n, -1, -1).cuda(), torch.randn(n, 1, hd, generator=g).cuda()
    c = _cache(2, 1, hd, nb, 16)
    c.store(None, k, v, seq, pos, table)
    _, vv = c.load(seq, pos, table, dtype=F32)
    q = (torch.randn(1, 2, hd, generator=g) * gain).to(BF16).cuda()
    want, mag = vv.double().mean(0, keepdim=True), vv.double().abs().mean(0, keepdim=True)
    for got in (c.attend(q, _i32([n]), table), c.attend_prompt(q, _i32([0, 1]), _i32([n]), table)):
        assert ((got.double() - want).abs() <= 2.0 ** -10 * mag + EPS[BF16] * want.abs() + 1e-6).all()
    c.check()


@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
@pytest.mark.parametrize("long", [False, True])
def test_prompt_rows_of_no_sequence_are_zero(layout, long):
    """Rows before the first and after the last sequence's, without (short) and with a split of the positions."""
    H, K, hd = layout
    lens = [2000, 1030] if long else [20, 30]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=3)
    q = torch.randn(400, H, hd, generator=g).half().cuda()
    fill = lambda: torch.full_like(q, 7.0)
    for cu in ([3, 20, 33], [0, 17, 30], [370, 387, 400], [0, 0, 400], [399, 399, 400], [0, 0, 0], [5, 5, 5], [400, 400, 400]):
        a, b = cu[0], cu[-1]
        got = c.attend_prompt(q, _i32(cu), _i32(lens), table, out=fill())
        assert not got[:a].any() and not got[b:].any()
        want, mag, top = _ref_attention(q[a:b], k, v, lens, [cu[1] - a, b - cu[1]], 1 / math.sqrt(hd), 0) if b > a else (None,) * 3
        if b > a:
            _close(got[a:b], want, mag, top, 2.0 ** -11)
    c.check()


def test_prompt_rows_of_refused_sequences_are_zero():
    """Row lists that leave the rows or go back: what they name is zero and reported, the other sequences are right."""
    from chonklm_b200 import _lib
    lens = [20, 30, 25]
    c, table, k, v, g = _filled(4, 2, 64, lens, 16, 8)
    q = torch.randn(40, 4, 64, generator=g).half().cuda()
    big = 2 ** 31 - 1
    for cu, live in [([0, 10, 30, 41], (0, 30)), ([-1, 10, 30, 40], (10, 40)), ([-big - 1, 10, 30, 40], (10, 40)), ([0, 10, 30, big], (0, 30)),
                     ([41, 42, 43, 44], (0, 0)), ([-5, -4, -3, -2], (0, 0)), ([-5, 50, 60, 70], (0, 0)), ([0, 30, 10, 40], (0, 0)),
                     ([big, 0, 0, 0], (0, 0)), ([0, big, -big, 40], (0, 0))]:
        got = c.attend_prompt(q, _i32(cu), _i32(lens), table, out=torch.full_like(q, 7.0))
        with pytest.raises(_lib.CkError, match="rows"):
            c.check()
        a, b = live
        assert not got[:a].any() and not got[b:].any(), cu
        at = a
        for i in range(3):
            if at == cu[i] and at < cu[i + 1] <= b:
                want, mag, top = _ref_attention(q[at: cu[i + 1]], k[i: i + 1], v[i: i + 1], lens[i: i + 1], [cu[i + 1] - at], 0.125, 0)
                _close(got[at: cu[i + 1]], want, mag, top, 2.0 ** -11)
                at = cu[i + 1]
        assert at == b
    c.attend_prompt(q, _i32([0, 10, 30, 40]), _i32(lens), table)
    c.check()


def test_prompt_rows_of_no_sequence_in_several_launches():
    H, K, hd, S = 4, 2, 64, 1100
    lens, news = [1 + i % 37 for i in range(S)], [1 + i % 3 for i in range(S)]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=12)
    n = sum(news)
    q = torch.randn(n, H, hd, generator=g).half().cuda()
    want = c.attend_prompt(q, _cu(news), _i32(lens), table)
    wide = torch.zeros(n + 12, H, hd, dtype=F16, device="cuda")
    wide[5: n + 5] = q
    got = c.attend_prompt(wide, _cu(news) + 5, _i32(lens), table, out=torch.full_like(wide, 7.0))
    c.check()
    assert torch.equal(got[5: n + 5], want) and not got[:5].any() and not got[n + 5:].any()


def test_refuses_to_drop_a_gradient():
    """There is no backward: a tensor that asks for one is refused while gradients are recorded, taken otherwise."""
    c, table, k, v, g = _filled(4, 2, 64, [5], 16, 8)
    seq, pos = _tokens([1])
    q, kn = torch.randn(1, 4, 64).half().cuda(), torch.randn(1, 2, 64).half().cuda()
    w = torch.ones(64, device="cuda")
    asks = lambda t: t.clone().requires_grad_()
    calls = [lambda f: c.store(f(q), kn, kn, seq, pos, table), lambda f: c.store(q, f(kn), kn, seq, pos, table),
             lambda f: c.store(q, kn, f(kn), seq, pos, table), lambda f: c.store(q, kn, kn, seq, pos, table, q_norm=f(w)),
             lambda f: c.store(q, kn, kn, seq, pos, table, k_norm=f(w)), lambda f: c.attend(f(q), _i32([5]), table),
             lambda f: c.attend_prompt(f(q), _i32([0, 1]), _i32([5]), table)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(asks)
        want = call(lambda t: t)
        with torch.no_grad():
            assert torch.equal(call(asks), want)
    c.check()


def test_read_kv_right_after_a_new_sequence(tiny_dir):
    """A running sequence's pages can be read whatever was added since the last step."""
    from chonklm_b200 import _lib
    from test_gpu_batch import _engine
    loaded, V = _engine(tiny_model(tiny_dir, "llama", "q4_k_m"))
    batch = _lib.Batch(loaded.engine.dev, max_seqs=3, kv="q8")
    first = batch.add([5, 6, 7, 8], 40)
    for _ in range(20):
        batch.step()
    want = batch.read_kv(first, 1)
    new = batch.add([9, 10], 30)
    got = batch.read_kv(first, 1)
    assert got[0].shape[0] == 20 and all(np.array_equal(a, b) for a, b in zip(got, want))
    assert batch.read_kv(new, 0)[0].shape[0] == 0
    batch.step()
    assert batch.read_kv(first, 1)[0].shape[0] == 21 and batch.read_kv(new, 0)[0].shape[0] == 1
    assert np.array_equal(batch.read_kv(first, 1)[0][:20], want[0])
    batch.close()
    loaded.engine.dispose()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
def test_blocks_before_the_window_may_be_gone(layout, block):
    """A server with a sliding window hands blocks that no query sees any more to others and clears their entries, those
    that end inside a tile which the window reaches among them."""
    H, K, hd = layout
    lens, news, window = [318, 95, 530], [1, 40, 5], 40
    c, table, k, v, g = _filled(H, K, hd, lens, block, 8, seed=8)
    q = torch.randn(sum(news), H, hd, generator=g).half().cuda()
    ln, cu, last = _i32(lens), _cu(news), q[[0, 40, 45]].contiguous()

    def gone(back, blocks):                      # entries of blocks that end before the first position seen
        t = torch.full((3, blocks), -7, dtype=torch.int32, device="cuda")
        t[:, : table.shape[1]] = table
        for i, n in enumerate(lens):
            t[i, : max(0, n - back[i] + 1 - window) // block] = -7
        return t

    want, one = c.attend_prompt(q, cu, ln, table, window=window), c.attend(last, ln, table, window=window)
    c.check()
    for blocks in (table.shape[1], 40000):       # short tables, and wide ones
        got = c.attend(last, ln, gone([1, 1, 1], blocks), window=window)
        c.check()
        assert torch.equal(got, one)
        got = c.attend_prompt(q, cu, ln, gone(news, blocks), window=window)
        c.check()
        _close(got, *_ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), window), 2.0 ** -11)
        assert blocks > 1000 or torch.equal(got, want)


def test_numbers_that_no_argument_holds_are_refused():
    """A window of more than 32 bits or of no whole number, a scale or eps of no finite one."""
    from chonklm_b200 import _lib
    c = _cache(4, 2, 64, 4)
    table, one = _i32([[0, 1]]), _i32([1])
    q, k = torch.zeros(1, 4, 64, dtype=F16, device="cuda"), torch.zeros(1, 2, 64, dtype=F16, device="cuda")
    w = torch.ones(64, device="cuda")
    for f in (lambda: c.attend(q, one, table, window=1 << 40), lambda: c.attend(q, one, table, window=0.5),
              lambda: c.attend(q, one, table, scale="1"), lambda: c.attend_prompt(q, _i32([0, 1]), one, table, window=1 << 31),
              lambda: c.attend_prompt(q, _i32([0, 1]), one, table, scale=1j), lambda: c.store(q, k, k, one, one, table, eps="1")):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: c.attend(q, one, table, scale=1e300), lambda: c.attend_prompt(q, _i32([0, 1]), one, table, scale=-1e39),
              lambda: c.store(q, k, k, one, one, table, q_norm=w, eps=1e300), lambda: c.store(q, k, k, one, one, table, k_norm=w, eps=math.inf)):
        with pytest.raises((ValueError, _lib.CkError), match="scale|eps|float"):
            f()
    c.check()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads", [128, 129, 130, 300])
def test_prompt_groups_of_many_heads(heads, hd):
    """A kv head's query heads in several units where a CTA's rows do not hold them."""
    lens, news = [70, 33], [9, 33]
    c, table, k, v, g = _filled(heads, 1, hd, lens, 16, 8, seed=heads)
    q = torch.randn(sum(news), heads, hd, generator=g).mul_(2).half().cuda()
    got = c.attend_prompt(q, _cu(news), _i32(lens), table, window=50)
    c.check()
    want, mag, top = _ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), 50)
    _close(got, want, mag, top, 2.0 ** -11)
    one = c.attend(q[:2].contiguous(), _i32(lens), table)
    c.check()
    _close(one, *_ref_attention(q[:2], k, v, lens, [1, 1], 1 / math.sqrt(hd), 0), 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
def test_prompt_split_with_4_bit_values(layout, dtype):
    H, K, hd = layout
    lens, news = [3000, 17, 0, 1500, 5], [33, 17, 2, 1, 9]
    c, table, k, v, g = _filled(H, K, hd, lens, 32, 4, seed=6)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).to(dtype).cuda()
    got = c.attend_prompt(q, _cu(news), _i32(lens), table, window=900)
    c.check()
    _close(got, *_ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), 900), 2.0 ** -11)


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("layout", [(9, 3, 64), (4, 1, 256), (24, 2, 64)])
def test_bf16_prompts(layout, v_bits):
    """Rows of very different sizes, all-zero ones among them: each is brought to its own power of two."""
    H, K, hd = layout
    lens, news = [150, 290], [150, 77]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, v_bits, seed=4)
    q = (torch.randn(sum(news), H, hd, generator=g) * torch.exp(3 * torch.randn(sum(news), H, 1, generator=g) - 4)).to(BF16).cuda()
    q[3], q[200, 1] = 0, 0
    got = c.attend_prompt(q, _cu(news), _i32(lens), table)
    c.check()
    _close(got, *_ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), 0), 2.0 ** -11)


@pytest.mark.parametrize("scale", [-0.1, 0.0, -0.0, 1e-30])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
def test_scales_of_either_sign_and_zero(layout, dtype, scale):
    H, K, hd = layout
    lens, news = [150, 1, 77], [20, 1, 77]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=14)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).to(dtype).cuda()
    got = c.attend_prompt(q, _cu(news), _i32(lens), table, scale=scale, window=60)
    c.check()
    _close(got, *_ref_attention(q, k, v, lens, news, scale, 60), 2.0 ** -11)
    one = c.attend(q[:3].contiguous(), _i32(lens), table, scale=scale, window=60)
    c.check()
    _close(one, *_ref_attention(q[:3], k, v, lens, [1, 1, 1], scale, 60), 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
def test_attention_rows_off_the_vector_alignment(layout, dtype):
    """q and out at odd elements with odd strides: the same bits as aligned rows, nothing beside them written; the rows of
    q may be the output's."""
    H, K, hd = layout
    lens, news = [150, 2500], [150, 31]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, 8, seed=15)
    n, ln, cu = sum(news), _i32(lens), _cu(news)
    q = torch.randn(n, H, hd, generator=g).mul_(2).to(dtype).cuda()

    def odd(m):
        base = torch.full((m * (H * hd + 3) + 1,), 7.0, dtype=dtype, device="cuda")
        return base, base.as_strided((m, H, hd), (H * hd + 3, hd, 1), 1)

    for call, m in ((lambda x, o: c.attend_prompt(x, cu, ln, table, out=o), n), (lambda x, o: c.attend(x, ln, table, out=o), 2)):
        want = call(q[:m].contiguous(), None)
        (_, x), (base, o) = odd(m), odd(m)
        x.copy_(q[:m])
        assert call(x, o) is o and torch.equal(o, want)
        o.fill_(7.0)
        assert (base == 7).all()
        same = q[:m].clone()
        assert torch.equal(call(same, same), want)
    c.check()


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("layout", [(6, 2, 64), (16, 8, 128), (4, 1, 256)])
@pytest.mark.parametrize("bad", ["k", "v"])
def test_a_visible_nan_reaches_the_rows_that_see_it(layout, bad, v_bits):
    """Prompts: exactly the rows that see the position, all of their dims.  One token: all dims for a key, its group's for
    a value."""
    H, K, hd = layout
    n, at, window = 200, 90, 64
    c, table, k, v, g = _filled(H, K, hd, [n], 16, v_bits, seed=16)
    x = torch.randn(1, K, hd, generator=g).cuda()
    y = x.clone()
    y[0, 0, 33] = float("nan")                   # kv head 0, group 1
    c.store(None, *((y, x) if bad == "k" else (x, y)), _i32([0]), _i32([at]), table)
    q = torch.randn(n, H, hd, generator=g).half().cuda()
    got = c.attend_prompt(q, _i32([0, n]), _i32([n]), table, window=window)
    sees = torch.zeros(n, H, 1, dtype=torch.bool, device="cuda")
    sees[at: at + window, : H // K] = True
    assert torch.equal(torch.isnan(got), sees.expand_as(got))
    one = torch.isnan(c.attend(q[:1], _i32([at + 5]), table))
    assert one[0, : H // K, 32:64].all() and not one[0, H // K:].any()
    assert one[0, : H // K].all() if bad == "k" else not one[0, : H // K, :32].any() and not one[0, : H // K, 64:].any()
    assert not torch.isnan(c.attend(q[:1], _i32([at]), table)).any()
    c.check()


def test_replayed_writes_go_where_the_inputs_say():
    """A captured decode step replayed on other tokens at other positions: the pages hold them, and the outputs are those
    of a second cache that takes the same calls one by one."""
    H, K, hd, block = 4, 2, 64, 16
    c, table, _, _, g = _filled(H, K, hd, [96, 96], block, 8)
    other, table2, _, _, _ = _filled(H, K, hd, [96, 96], block, 8)
    assert torch.equal(table, table2)
    q, kn, vn = (torch.randn(2, h, hd, generator=g).half().cuda() for h in (H, K, K))
    seq, pos, length = _i32([0, 1]), _i32([4, 89]), _i32([5, 90])
    f = torch.rand(hd // 2, generator=g).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(c.store(q, kn, vn, seq, pos, table, inv_freq=f), length, table)
    torch.cuda.current_stream().wait_stream(s)
    other.store(q, kn, vn, seq, pos, table, inv_freq=f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned = c.store(q, kn, vn, seq, pos, table, inv_freq=f)
        out = c.attend(turned, length, table)
    every = _tokens([96, 96])
    for _ in range(4):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g))
        pos.add_(1)
        length.add_(1)
        graph.replay()
        want = other.store(q, kn, vn, seq, pos, table, inv_freq=f)
        assert torch.equal(turned, want) and torch.equal(out, other.attend(want, length, table))
        for a, b in zip(c.load(*every, table), other.load(*every, table)):
            assert torch.equal(a, b)
    c.check()
    other.check()


def test_batch_by_list_follows_the_plain_model(tiny_dir):
    """Contexts past 2048 and more slots than fill the device by unit: the attention's list form and its join, with the
    number of queries on the device (5 or fewer of 40)."""
    from chonklm_b200 import _lib
    from chonklm_b200.registry import ModelDef
    from chonklm_b200.runtime import loadLlamaWgslModel
    from test_gpu_batch import _run
    from test_gpu_batch_quantised import TOL, PlainModel
    path = tiny_model(tiny_dir, "llama", "q4_k_m", context_length=4096)
    V = 1000
    loaded = loadLlamaWgslModel(ModelDef(id="t", label="t", vocab=V, maxContext=4096, gguf=path, eosIds=[]))
    rng = np.random.default_rng(3)
    pending = [(rng.integers(0, V, size=n).tolist(), m, ()) for n, m in ((3, 20), (40, 12), (1, 30), (90, 5), (170, 9))]
    batch = _lib.Batch(loaded.engine.dev, max_seqs=40, kv="q8")
    got = _run(batch, pending)
    batch.close()
    for (prompt, _, _), ids in zip(pending, got):
        plain = PlainModel(path, loaded, 8)
        for t in prompt[:-1]:
            plain.step(t)
        t = prompt[-1]
        for want in ids:
            logits = plain.step(t)
            assert logits[want] >= logits.max() - 2 * TOL * np.abs(logits).max(), (len(prompt), want)
            t = want
    loaded.engine.dispose()


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("length", [2, 700])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_fp16_prompts_keep_the_bits_of_keys(hd, length, v_bits):
    """Two kinds of key whose code * scale lies at the middle between two fp16 numbers, one rounded up and one down in
    every dim that the query looks at, and scores of 50: keys as single fp16 numbers move the two kinds' probabilities by
    several times what is left when the scale's upper 4 bits are a product of their own.  Its rest is below 2^-3 of the
    scale and rounded to 11 bits: 2^-14 of a key."""
    d, codes = 1406 * 2.0 ** -14, (95, 96)
    rel = [(float(np.float16(d * x)) - d * x) / (d * x) for x in codes]
    assert abs(rel[0] - rel[1]) > 2.0 ** -10.1
    g = torch.Generator().manual_seed(hd)
    table, nb = _tables([length], 16, g)
    seq, pos = _tokens([length])
    k = torch.empty(length, 1, hd)
    k[0::2], k[1::2] = codes[0] * d, codes[1] * d
    k[:, 0, 1::32] = 127 * d                     # the groups' largest values, which the query does not look at
    v = torch.ones(length, 1, hd)
    v[1::2] = -1
    c = _cache(1, 1, hd, nb, 16, v_bits)
    c.store(None, k.cuda(), v.cuda(), seq, pos, table)
    kk, vv = c.load(seq, pos, table, dtype=F32)
    assert torch.equal(kk.cpu(), k)
    q = torch.ones(1, 1, hd, dtype=F16, device="cuda")
    q[0, 0, 1::32] = 0
    scale = 50 / (hd * 31 / 32 * codes[0] * d)
    want, mag, top = _ref_attention(q, [kk], [vv], [length], [1], scale, 0)
    for rows, blocks in ((1, table.shape[1]), (1, 1000), (100, table.shape[1])):   # whole, split, on many CTAs
        wide = torch.zeros(rows, blocks, dtype=torch.int32, device="cuda")
        wide[:, : table.shape[1]] = table
        got = c.attend_prompt(q.expand(rows, -1, -1).contiguous(), _cu([1] * rows), _i32([length] * rows), wide, scale=scale)
        c.check()
        _close(got, want.expand_as(got), mag, top, 2.0 ** -14)


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("layout", [(9, 3, 64), (16, 8, 128), (4, 1, 256)])
def test_fp16_prompts_to_14_bits_of_a_key(layout, v_bits):
    """Many position tiles and CTAs, ragged, with a window and without."""
    H, K, hd = layout
    lens, news = [700, 65, 1300, 64, 129], [700, 65, 300, 1, 129]
    c, table, k, v, g = _filled(H, K, hd, lens, 16, v_bits, seed=31)
    q = torch.randn(sum(news), H, hd, generator=g).mul_(2).half().cuda()
    for window in (0, 150):
        got = c.attend_prompt(q, _cu(news), _i32(lens), table, window=window)
        c.check()
        _close(got, *_ref_attention(q, k, v, lens, news, 1 / math.sqrt(hd), window), 2.0 ** -14)
        for _ in range(50):
            assert torch.equal(got, c.attend_prompt(q, _cu(news), _i32(lens), table, window=window))


def _half_and_half(hd, length, v_bits):
    """Two kinds of value in turn, equally likely: their mean is small beside them, and code * scale of each lies near the
    middle between two fp16 numbers.  8 bits: 95 d and -96 d; 4 bits: 7 d and -6 d (and -8 d, the groups' largest)."""
    d, a, b, top = (1406 * 2.0 ** -14, 95, -96, 127) if v_bits == 8 else (1404 * 2.0 ** -14, 7, -6, -8)
    g = torch.Generator().manual_seed(hd)
    table, nb = _tables([length], 16, g)
    seq, pos = _tokens([length])
    v = torch.empty(length, 1, hd)
    v[0::2], v[1::2] = a * d, b * d
    v[:, 0, 1::32] = top * d
    c = _cache(1, 1, hd, nb, 16, v_bits)
    c.store(None, torch.ones(length, 1, hd, device="cuda"), v.cuda(), seq, pos, table)
    _, vv = c.load(seq, pos, table, dtype=F32)
    assert torch.equal(vv.cpu(), v)
    want, mag = v.double().mean(0)[0].cuda(), v.double().abs().mean(0)[0].cuda()
    # the probabilities are equal, powers of two, and exact; the scale's rest below 2^-3 of it is rounded to 11 bits, or
    # (4 bits) not at all
    tol = (2.0 ** -14 if v_bits == 8 else 2.0 ** -20) * mag + EPS[F16] * want.abs() + 1e-6
    wide = torch.zeros(1, 40000, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    return c, table, wide, want, tol


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("length", [2, 100, 2000])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_fp16_outputs_of_one_token_keep_the_bits_of_values(hd, length, v_bits):
    c, table, wide, want, tol = _half_and_half(hd, length, v_bits)
    q = torch.ones(400, 1, hd, dtype=F16, device="cuda")
    for n, t in ((1, table), (1, wide), (400, table)):       # in clusters, by list, a CTA each
        got = c.attend(q[:n], _i32([length] * n), t.expand(n, -1).contiguous())
        assert ((got.double() - want).abs() <= tol).all()
    c.check()


@pytest.mark.parametrize("v_bits", [8, 4])
@pytest.mark.parametrize("length", [2, 100, 2000])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_fp16_prompts_keep_the_bits_of_values(hd, length, v_bits):
    c, table, wide, want, tol = _half_and_half(hd, length, v_bits)
    q = torch.ones(400, 1, hd, dtype=F16, device="cuda")
    for n, t in ((1, table), (1, wide), (400, table)):       # whole, split, on many CTAs
        got = c.attend_prompt(q[:n], _cu([1] * n), _i32([length] * n), t.expand(n, -1).contiguous())
        assert ((got.double() - want).abs() <= tol).all()
    c.check()
