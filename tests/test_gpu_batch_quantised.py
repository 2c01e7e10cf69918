"""Batched decode over a quantised cache (ck_batch_create_kv): a step's norms,
rotation, quantised store and attention against a plain 64-bit model whose
cache is quantised by the definition."""
import numpy as np
import pytest

from conftest import tiny_model
from oracle import oracle
from test_gpu_batch import _engine, _run

pytestmark = pytest.mark.gpu


class PlainModel:
    """The llama / qwen3 graph in 64 bits, one token at a time, its keys and values quantised per 32 values."""

    def __init__(self, path, loaded, v_bits):
        from chonklm_b200.gguf import ByteSource
        self.m, self.bits = loaded.manifest.model, v_bits
        src, self.w = ByteSource(path), {}
        for name, t in loaded.manifest.tensors.items():
            raw = np.frombuffer(src.read(t.offset, t.length), dtype=np.uint8)
            if t.ggml_type == 0:
                self.w[name] = raw.view(np.float32).astype(np.float64)
            elif t.ggml_type == 1:
                self.w[name] = raw.view(np.float16).astype(np.float64)
            else:
                n, k = t.shape[-2], t.shape[-1]
                self.w[name] = oracle.dequant(t.ggml_type, raw, k, n).astype(np.float64)
        self.kv = [([], []) for _ in range(self.m.layers)]

    def norm(self, x, w, eps):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w

    def quantise(self, x, bits):
        g = x.reshape(-1, 32)
        if bits == 8:
            d, lo, hi = np.abs(g).max(-1) / 127, -127, 127
        else:
            d, lo, hi = np.where(g.max(-1) >= -g.min(-1), g.max(-1), g.min(-1)) / -8, -8, 7
        d = d.astype(np.float16).astype(np.float64)
        inv = np.where(d == 0, 0, 1 / np.where(d == 0, 1, d))
        return (np.clip(np.rint(g * inv[:, None]), lo, hi) * d[:, None]).reshape(x.shape)

    def rotate(self, x, pos, theta):
        hd = x.shape[-1]
        a = pos * float(theta) ** (-2.0 * np.arange(hd // 2) / hd)
        c, s = np.cos(a), np.sin(a)
        if self.m.ropeLayout == "interleaved":
            y = np.empty_like(x)
            y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 0::2] * s + x[:, 1::2] * c
            return y
        h = hd // 2
        return np.concatenate((x[:, :h] * c - x[:, h:] * s, x[:, :h] * s + x[:, h:] * c), -1)

    def step(self, token):
        m, w = self.m, self.w
        x = w["token_embd.weight"][token] * m.embeddingScale
        for i in range(m.layers):
            p = f"blk.{i}."
            y = self.norm(x, w[p + "attn_norm.weight"], m.normEps)
            q, k, v = (( w[p + f"attn_{n}.weight"] @ y).reshape(-1, m.headDim) for n in "qkv")
            if m.qkNorm:
                q = self.norm(q, w[p + "attn_q_norm.weight"], m.qkNormEps)
                k = self.norm(k, w[p + "attn_k_norm.weight"], m.qkNormEps)
            ks, vs = self.kv[i]
            pos = len(ks)
            q, k = (self.rotate(t, pos, m.layerRopeTheta[i]) for t in (q, k))
            ks.append(self.quantise(k, 8))
            vs.append(self.quantise(v, self.bits))
            K, V = np.stack(ks), np.stack(vs)
            G = m.heads // m.kvHeads
            o = np.empty_like(q)
            for h in range(m.heads):
                s = K[:, h // G] @ q[h] / np.sqrt(m.headDim)
                e = np.exp(s - s.max())
                o[h] = e @ V[:, h // G] / e.sum()
            x = x + w[p + "attn_output.weight"] @ o.reshape(-1)
            y = self.norm(x, w[p + "ffn_norm.weight"], m.normEps)
            g = w[p + "ffn_gate.weight"] @ y
            x = x + w[p + "ffn_down.weight"] @ (g / (1 + np.exp(-g)) * (w[p + "ffn_up.weight"] @ y))
        head = w.get("output.weight", w["token_embd.weight"])
        return head @ self.norm(x, w["output_norm.weight"], m.normEps)


# Logits of the engine are within 1e-3 of a 64-bit restatement over the same cache values (the parity suite's bound).
# Here a stored code may also come out one off where a value lies at the middle between two (the engine's 32-bit key
# differs in its last bits), and the attention's probabilities and values are rounded to 11 bits: 2^-10 of an output in
# each of the 2 layers, on top.  An id that is not the plain model's first has to be within that of it.
TOL = 1e-3 + 2 * 2.0 ** -10


@pytest.mark.parametrize("kv", ["q8", "q8v4"])
@pytest.mark.parametrize("arch,kw", [("llama", {}), ("qwen3", {}), ("llama", {"heads": 6, "kv_heads": 2}), ("qwen3", {"head_dim": 128}),
                                     ("llama", {"heads": 8, "kv_heads": 2})])
def test_quantised_batch_follows_the_plain_model(tiny_dir, arch, kw, kv):
    from chonklm_b200 import _lib
    path = tiny_model(tiny_dir, arch, "q4_k_m", **kw)
    loaded, V = _engine(path)
    rng = np.random.default_rng(3)
    pending = [(rng.integers(0, V, size=n).tolist(), m, ()) for n, m in ((3, 20), (40, 12), (1, 30), (90, 5), (17, 9))]
    batch = _lib.Batch(loaded.engine.dev, max_seqs=3, kv=kv)     # fewer slots than sequences: slots are reused
    got = _run(batch, pending)
    for (prompt, _, _), ids in zip(pending, got):
        plain = PlainModel(path, loaded, 8 if kv == "q8" else 4)
        for t in prompt[:-1]:
            plain.step(t)
        t = prompt[-1]
        for want in ids:                                          # fed the engine's own ids
            logits = plain.step(t)
            assert logits[want] >= logits.max() - 2 * TOL * np.abs(logits).max(), (len(prompt), want)
            t = want
    # a sequence's ids do not depend on its neighbours
    alone = _lib.Batch(loaded.engine.dev, max_seqs=1, kv=kv)
    assert _run(alone, pending[:2]) == got[:2]
    batch.close()
    alone.close()
    loaded.engine.dispose()


@pytest.mark.parametrize("kv", ["q8", "q8v4"])
def test_read_kv(tiny_dir, kv):
    """Layer 0's pages (no attention before them) against the plain model's: a step of a code where the 32-bit value
    lies at the middle between two, else the value to 1e-5."""
    from chonklm_b200 import _lib
    path = tiny_model(tiny_dir, "qwen3", "q4_k_m")
    loaded, V = _engine(path)
    batch = _lib.Batch(loaded.engine.dev, max_seqs=2, kv=kv)
    prompt = np.random.default_rng(8).integers(0, V, size=37).tolist()
    other = batch.add([5, 6, 7], 60)
    sid = batch.add(prompt, 10)
    for _ in range(30):
        batch.step()
    k, v = batch.read_kv(sid, 0)
    assert k.shape[0] == 30 and batch.read_kv(other, 1)[0].shape[0] == 30
    plain = PlainModel(path, loaded, 8 if kv == "q8" else 4)
    for t in prompt[:30]:
        plain.step(t)
    for got, want, levels in ((k, np.stack(plain.kv[0][0]), 127), (v, np.stack(plain.kv[0][1]), 127 if kv == "q8" else 8)):
        top = np.abs(want).reshape(30, -1, 32).max(-1).repeat(32, -1).reshape(want.shape)
        off = np.abs(got - want)
        assert (off <= top / levels * 1.01 + 1e-5 * top).all()
        assert (off > 1e-3 * top).mean() < 0.01
    with pytest.raises(_lib.CkError, match="layer"):
        batch.read_kv(sid, 2)
    with pytest.raises(_lib.CkError, match="unknown"):
        batch.read_kv(99, 0)
    batch.close()
    plain16 = _lib.Batch(loaded.engine.dev, max_seqs=1)
    s = plain16.add([1, 2], 4)
    with pytest.raises(_lib.CkError, match="not quantised"):
        plain16.read_kv(s, 0)
    plain16.close()
    with pytest.raises(ValueError, match="unknown cache"):
        _lib.Batch(loaded.engine.dev, max_seqs=1, kv="q4")
    loaded.engine.dispose()
