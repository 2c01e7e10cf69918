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
