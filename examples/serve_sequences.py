"""Several prompts served from one paged 4-bit KV cache.

    python examples/serve_sequences.py [--prompts 4] [--samples 3] [--new 32]

Prompts of different lengths go through a random-init Llama-shaped model
(Q4_K weights) as the packed rows of one pass: the projections are
cuda_matmul_quant_batched, the attention attention_packed, and each layer's
keys and values are appended to the cache.  Each prompt is then forked, so
that its samples share the prompt's pages, and every sample is decoded a token
a step with the cache's attention.  Half of the samples end early and are
released, the cache is compacted, and the others go on.  Norms, rotation and
the gate are torch's: they are not what is shown here.
"""
from __future__ import annotations

import argparse
import pathlib
import sys

import numpy as np
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
if str(ROOT / "google-classic_b200") not in sys.path:
    sys.path.insert(0, str(ROOT / "google-classic_b200"))

import holo_b200 as hb  # noqa: E402
from holo_b200 import synth  # noqa: E402
from holo_b200.attention import attention_packed  # noqa: E402
from holo_b200.kv4 import Kv4Cache  # noqa: E402

SMALL = {"dim": 1024, "n_layers": 4, "n_heads": 16, "n_kv_heads": 4, "head_dim": 64, "ffn_dim": 2816, "vocab": 2048,
         "layer_type": hb.Q4_K, "out_type": hb.Q4_K, "emb_type": 1}
EPS, ROPE_BASE = 1e-5, 10000.0


class PagedModel:
    """A Llama-shaped model whose sequences live in a Kv4Cache.

    The library's matmuls run on its own stream; everything here is enqueued
    under `with self.on():`, which makes that stream torch's current one."""

    def __init__(self, cfg: dict, weights: dict, n_pages: int, max_seqs: int, max_pages: int, page_tokens: int = 64):
        self.cfg, self.dev = cfg, hb.Device(0, 1)
        self.stream = torch.cuda.ExternalStream(self.dev.lib.cuda_get_stream())
        dim, hd, ffn = cfg["dim"], cfg["head_dim"], cfg["ffn_dim"]
        q, kv = cfg["n_heads"] * hd, cfg["n_kv_heads"] * hd
        shapes = {"wq": (q, dim), "wk": (kv, dim), "wv": (kv, dim), "wo": (dim, q), "w1": (ffn, dim), "w3": (ffn, dim),
                  "w2": (dim, ffn)}
        with self.on():
            self.layers = [{n: (self.dev.upload_quant(w[n], cfg["layer_type"], *s), s) for n, s in shapes.items()}
                           | {n: torch.from_numpy(w[n]).cuda() for n in ("attn_norm", "ffn_norm")} for w in weights["layers"]]
            self.output = (self.dev.upload_quant(weights["output"], cfg["out_type"], cfg["vocab"], dim), (cfg["vocab"], dim))
            self.embed = torch.from_numpy(weights["tok_emb"]).cuda()
            self.final_norm = torch.from_numpy(weights["final_norm"]).cuda()
            self.freq = ROPE_BASE ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd)
            self.cache = Kv4Cache(cfg["n_layers"], cfg["n_kv_heads"], hd, page_tokens, n_pages, max_seqs, max_pages)

    def on(self):
        return torch.cuda.stream(self.stream)

    def close(self):
        self.dev.sync()
        for w in [w for layer in self.layers for w in layer.values() if isinstance(w, tuple)] + [self.output]:
            self.dev.free(w[0])

    def matmul(self, weight, x):
        ptr, (n, k) = weight
        y = torch.empty(x.shape[0], n, device="cuda")
        if x.shape[0] and self.dev.lib.cuda_matmul_quant_batched(y.data_ptr(), ptr, x.contiguous().data_ptr(), x.shape[0], n, k):
            self.dev.check("cuda_matmul_quant_batched")
        return y

    @staticmethod
    def norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w

    def rope(self, x, pos):
        angle = pos[:, None, None].float() * self.freq
        a, b = x.chunk(2, -1)
        c, s = angle.cos(), angle.sin()
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def rows(self, tokens, pos, attend):
        """The residual stream of the rows after the last layer; attend(layer, q, k, v) is their attention."""
        n, hd = tokens.shape[0], self.cfg["head_dim"]
        x = self.embed[tokens.long()].float()
        for i, w in enumerate(self.layers):
            h = self.norm(x, w["attn_norm"])
            q, k, v = (self.matmul(w[m], h).view(n, -1, hd) for m in ("wq", "wk", "wv"))
            o = attend(i, self.rope(q, pos), self.rope(k, pos), v)
            x = x + self.matmul(w["wo"], o.reshape(n, -1).float())
            h = self.norm(x, w["ffn_norm"])
            x = x + self.matmul(w["w2"], torch.nn.functional.silu(self.matmul(w["w1"], h)) * self.matmul(w["w3"], h))
        return x

    def logits(self, x):
        return self.matmul(self.output, self.norm(x, self.final_norm))

    def prefill(self, prompts, seqs):
        """The prompts (lists of tokens) become the sequences seqs, which are
        empty; returns the logits after each one's last token."""
        lens = [len(p) for p in prompts]
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        start = self.cache.extend(cu[1:] - cu[:-1], seqs)
        pos = torch.cat([torch.arange(n, device="cuda") for n in lens])

        def attend(layer, q, k, v):
            self.cache.append(layer, k, v, cu, start, seqs)
            return attention_packed(q.bfloat16(), k.bfloat16(), v.bfloat16(), cu)

        x = self.rows(torch.tensor([t for p in prompts for t in p], device="cuda"), pos, attend)
        return self.logits(x[cu[1:].long() - 1])

    def step(self, tokens, seqs):
        """One more token of each sequence: its key and value are appended,
        and it attends to all that its sequence holds.  Returns the logits."""
        ones = torch.ones_like(seqs)
        start = self.cache.extend(ones, seqs)
        cu = torch.arange(seqs.shape[0] + 1, dtype=torch.int32, device="cuda")

        def attend(layer, q, k, v):
            self.cache.append(layer, k, v, cu, start, seqs)
            return self.cache.attention(layer, q, seqs=seqs)

        return self.logits(self.rows(tokens, start, attend))


def pick(logits, gen, temperature=0.8):
    return torch.multinomial(torch.softmax(logits / temperature, -1), 1, generator=gen)[:, 0]


def seq_ids(first, n):
    return torch.arange(first, first + n, dtype=torch.int32, device="cuda")


def serve(cfg=SMALL, prompts=4, samples=3, new=32, seed=0, page=64, out=print):
    rng = np.random.default_rng(seed)
    texts = [rng.integers(0, cfg["vocab"], n).tolist() for n in rng.integers(1, 400, prompts)]
    most = -(-(max(map(len, texts)) + new) // page)
    m = PagedModel(cfg, synth.llama_weights(cfg, seed), prompts * (samples + 1) * most, prompts * (samples + 1), most, page)
    try:
        with m.on():
            gen = torch.Generator("cuda").manual_seed(seed)
            parents, children = seq_ids(0, prompts), seq_ids(prompts, prompts * samples)
            logits = m.prefill(texts, parents)
            own = int((m.cache.refs > 0).sum())
            m.cache.fork(parents.repeat_interleave(samples), children)
            m.cache.release(parents)
            out(f"{prompts} prompts of {[len(t) for t in texts]} tokens in {own} pages; "
                f"{prompts * samples} samples in {int((m.cache.refs > 0).sum())}")
            token = pick(logits.repeat_interleave(samples, 0), gen)
            said = {int(c): [int(t)] for c, t in zip(children, token)}
            for i in range(1, new):
                if i == new // 2:   # every second sample ends here
                    m.cache.release(children[1::2].contiguous())
                    children, token = children[::2].contiguous(), token[::2]
                    m.cache.compact()
                    used = m.cache.refs > 0
                    out(f"{len(children)} samples go on in pages 0..{int(used.sum()) - 1}")
                    if not bool(used[:int(used.sum())].all()):
                        raise AssertionError("pages in use are not at the front")
                token = pick(m.step(token, children), gen)
                for c, t in zip(children.tolist(), token.tolist()):
                    said[c].append(t)
            m.cache.check()
            m.cache.release(children)
            m.cache.check()
            if int(m.cache.refs.sum()):
                raise AssertionError("pages left in use")
        for c, t in said.items():
            out(f"prompt {(c - prompts) // samples} sample {(c - prompts) % samples}: {len(t)} tokens {t[:8]}...")
        return said
    finally:
        m.close()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, d in (("prompts", 4), ("samples", 3), ("new", 32), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=d)
    a = ap.parse_args()
    serve(prompts=a.prompts, samples=a.samples, new=a.new, seed=a.seed)
