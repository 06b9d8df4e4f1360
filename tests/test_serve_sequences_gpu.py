"""The paged model of examples/serve_sequences.py: packed prompts, the 4-bit
cache and its pages together, against a plain 64-bit forward pass."""
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

import holo_b200 as hb
from holo_b200 import synth

pytestmark = pytest.mark.gpu
CFG = {"dim": 512, "n_layers": 2, "n_heads": 8, "n_kv_heads": 2, "head_dim": 64, "ffn_dim": 768, "vocab": 512,
       "layer_type": hb.Q4_K, "out_type": hb.Q4_K, "emb_type": 1}
# Activations are quantised to 8 bits in blocks of 32 before each product: a
# step of max/127 leaves an error of max/127/sqrt(12), and the largest of 32
# normal values is about 2.2 of their rms, so 0.5 % of a product's rms.  A
# logit has seen at most 4 products a layer in turn and the output matrix, 9 of
# them: 1.5 % when they add up in quadrature.  (bf16 and fp16 roundings are
# 0.1 to 0.2 %.)  The bound is twice that.
BOUND = 3e-2


@pytest.fixture(scope="module")
def example(dev):
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import serve_sequences
    finally:
        sys.path.pop(0)
    return serve_sequences


@pytest.fixture
def model(example):
    m = example.PagedModel(CFG, synth.llama_weights(CFG, 5), 64, 16, 8, 32)
    yield m
    m.close()


def plain(model, example, x, pos, layer_kv):
    """Logits of rows x (64-bit residual stream) at positions pos; layer_kv(layer, k, v) gives the keys and values of each row
    as (K [rows][positions][n_kv][hd], V, a mask of the positions that it sees)."""
    cfg, hd = CFG, CFG["head_dim"]

    def weight(w, t):
        ptr, (n, k) = w
        out = torch.empty(n, k, device="cuda")
        model.dev.lib.cuda_dequantize_rows(out.data_ptr(), ptr, t, n, k)
        return out.double()

    for i, w in enumerate(model.layers):
        h = example.PagedModel.norm(x, w["attn_norm"].double())
        q, k, v = ((h @ weight(w[m], cfg["layer_type"]).T).view(len(x), -1, hd) for m in ("wq", "wk", "wv"))
        angle = pos[:, None, None].double() * 10000.0 ** (-torch.arange(0, hd, 2, device="cuda").double() / hd)

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

        K, V, seen = layer_kv(i, turn(k), v)
        g = cfg["n_heads"] // cfg["n_kv_heads"]
        s = torch.einsum("rhd,rphd->rhp", turn(q), K.repeat_interleave(g, 2)) * hd ** -0.5
        p = torch.softmax(s.masked_fill(~seen[:, None], float("-inf")), -1)
        o = torch.einsum("rhp,rphd->rhd", p, V.repeat_interleave(g, 2))
        x = x + o.reshape(len(x), -1) @ weight(w["wo"], cfg["layer_type"]).T
        h = example.PagedModel.norm(x, w["ffn_norm"].double())
        a, b = h @ weight(w["w1"], cfg["layer_type"]).T, h @ weight(w["w3"], cfg["layer_type"]).T
        x = x + (a * torch.sigmoid(a) * b) @ weight(w["w2"], cfg["layer_type"]).T
    return example.PagedModel.norm(x, model.final_norm.double()) @ weight(model.output, cfg["out_type"]).T


def near(got, want):
    err = (got.double() - want).square().mean(-1).sqrt() / want.square().mean(-1).sqrt()
    assert float(err.max()) <= BOUND


def texts(lens, seed=3):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, CFG["vocab"], n).tolist() for n in lens]


def test_prefill(example, model):
    prompts = texts([1, 70, 33])
    with model.on():
        got = model.prefill(prompts, example.seq_ids(0, 3))
        for i, p in enumerate(prompts):
            n = len(p)
            tri = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            x = model.embed[torch.tensor(p, device="cuda")].double()
            want = plain(model, example, x, torch.arange(n, device="cuda"),
                         lambda _, k, v: (k[None].expand(n, -1, -1, -1), v[None].expand(n, -1, -1, -1), tri))
            near(got[i:i + 1], want[-1:])
        model.cache.check()


def test_step(example, model):
    prompts = texts([1, 64, 45, 100])
    with model.on():
        seqs = example.seq_ids(0, 4)
        model.prefill(prompts, seqs)
        for step in range(3):
            token = torch.tensor([7, 100, 3, 250], device="cuda") + step
            got = model.step(token, seqs)
            for i, p in enumerate(prompts):
                n = len(p) + 1 + step
                cu, start, one = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, n], [0], [i]))

                def held(layer, k, v):   # what the cache holds of the sequence, its newest position included
                    kv = [torch.empty(n, CFG["n_kv_heads"], CFG["head_dim"], device="cuda") for _ in range(2)]
                    K, V = model.cache.read(layer, cu, start, *kv, seqs=one)
                    return K[None].double(), V[None].double(), torch.ones(1, n, dtype=torch.bool, device="cuda")

                want = plain(model, example, model.embed[token[i:i + 1]].double(), torch.tensor([n - 1], device="cuda"), held)
                near(got[i:i + 1], want)
        model.cache.check()


def test_forks_and_compaction_keep_the_logits(example, model):
    """A sample's logits do not depend on whose pages it shares, where they lie, or which other sequences come and go."""
    prompts = texts([50, 90, 32])
    with model.on():
        seqs = example.seq_ids(0, 3)
        model.prefill(prompts, seqs)
        kids = example.seq_ids(4, 6)
        model.cache.fork(seqs.repeat_interleave(2), kids)
        model.cache.fork(seqs, example.seq_ids(10, 3))
        token = torch.arange(6, device="cuda") // 2 + 20
        a = model.step(token, kids)
        assert torch.equal(a[::2], a[1::2])
        model.cache.release(seqs)
        model.cache.release(kids)
        model.cache.compact()
        b = model.step(token[::2], example.seq_ids(10, 3))
        assert torch.equal(a[::2], b)
        model.cache.check()


def test_the_example(example):
    said = example.serve(CFG, prompts=3, samples=2, new=12, out=lambda *_: None)
    again = example.serve(CFG, prompts=3, samples=2, new=12, out=lambda *_: None)
    assert said == again
    assert sorted(map(len, said.values())) == [6] * 3 + [12] * 3
    assert all(0 <= t < CFG["vocab"] for s in said.values() for t in s)
