"""decode_beam_hip against a 64-bit restatement of the model over the quantised cache.

The restatement runs a hypothesis token by token: the layers of src/infer.c:311-472, K and V rows rounded to binary16 (as the model's cache
keeps them) and then to the paged cache's codes (tests/test_paged.py: Cache).  Two evaluations of one token differ by rounding, and where a row
value lies next to a border by one code; conftest's FP8KV_TOL bounds what that does to the logits of a model of two layers (its e5m2 codes
are 12.5 - 25 % apart, a code here is at most 1 / 64 of its block's largest value), so a step's log-probability is off by at most twice that share
of the largest logit, and a score by the sum over its steps.  Selections follow from the scores: a search may only differ from the
restatement's where two candidates are closer than that, so the scores are compared, sorted, and every hypothesis' score with the
restatement's of the SAME tokens."""
import copy

import numpy as np
import pytest

from calm_amd import abi
from calm_amd import calmfile as cf
from calm_amd.host import HipBackend, HostModel
from conftest import FP8KV_TOL, rel_err
from test_paged import Cache, attention


class Model:
    """the model in 64 bits; a state is (position, per layer [K cache, V cache])"""

    def __init__(self, tensors, md, spec, dtype, window=0, sinks=0):
        self.t, self.s, self.dtype, self.window, self.sinks = {}, spec, dtype, window, sinks
        self.eps, self.L = float(md["norm_eps"]), int(md["n_layers"])
        for n, a in tensors.items():
            if n.startswith("model."):
                self.t[n] = a.astype(np.float64) if a.dtype == np.float32 and "weight" in n and "norm" in n else (
                    a.astype(np.float64) if "bias" in n else cf.dequantize(a, dtype).astype(np.float64))
        d = np.arange(0, spec.head_dim, 2)
        self.freq = np.where(d >= spec.rotary_dim, 0.0, float(md["rope_theta"]) ** (-d / spec.rotary_dim))

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean() + self.eps) * w

    def rope(self, x, pos):
        c, s = np.cos(pos * self.freq), np.sin(pos * self.freq)
        y = x.copy()
        y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 0::2] * s + x[:, 1::2] * c
        return y

    def step(self, tok, pos, layers):
        """layers: per layer (append, values) of K and V; -> logits"""
        s, t = self.s, self.t
        x = t["model.embed.weight"][tok].copy()
        for l in range(self.L):
            p = f"model.layers.{l}."
            xb = self.norm(x, t[p + "attn.norm.weight"])
            q, k, v = (t[p + f"attn.w{n}.weight"] @ xb for n in "qkv")
            q, k, v = (y.reshape(-1, s.head_dim) for y in (q, k, v))
            q, k = self.rope(q, pos), self.rope(k, pos)
            kc, vc = layers[l]
            kc.append(0, k.astype(np.float16).astype(np.float64)[None]), vc.append(0, v.astype(np.float16).astype(np.float64)[None])
            att = attention(q[None], kc.values(0), vc.values(0), s.head_dim ** -0.5, self.window, self.sinks)
            x = x + t[p + "attn.wo.weight"] @ att.ravel()
            xb = self.norm(x, t[p + "mlp.norm.weight"])
            f = lambda w1, w2, w3: w2 @ ((lambda a: a / (1 + np.exp(-a)))(w1 @ xb) * (w3 @ xb))  # noqa: E731
            w1, w2, w3 = (t[p + f"mlp.w{i}.weight"] for i in (1, 2, 3))
            if s.n_experts:
                g = t[p + "moegate.weight"] @ xb
                top = np.argsort(-g, kind="stable")[: s.n_experts_active]
                w = np.exp(g[top] - g[top].max())
                x = x + sum(a * f(w1[e], w2[e], w3[e]) for a, e in zip(w / w.sum(), top))
            else:
                x = x + f(w1, w2, w3)
        out = "model.output.weight" if "model.output.weight" in t else "model.embed.weight"
        return t[out] @ self.norm(x, t["model.norm.weight"])


class Half:
    """a cache of binary16 rows, as the model's own"""

    def __init__(self):
        self.rows = []

    def append(self, s, rows):
        self.rows.extend(rows)

    def values(self, s):
        return np.array(self.rows)


def e5m2(x):
    """binary16 rounded to nearest even to its upper byte (the fp8 cache), saturating"""
    b = np.asarray(x, dtype=np.float16).view(np.uint16).astype(np.uint32)
    r = ((b + 0x7F + ((b >> 8) & 1)) >> 8) << 8
    sat = (r & 0x7FFF) >= 0x7C00
    return np.where(sat, (b & 0x8000) | 0x7B00, r).astype(np.uint16).view(np.float16).astype(np.float64)


class Fp8(Half):
    def append(self, s, rows):
        self.rows.extend(e5m2(rows))


def prompt_caches(model, prompt, fp8):
    """the model's own cache after the prompt, then the paged one that takes it over"""
    own = [[(Fp8 if fp8 else Half)() for _ in range(2)] for _ in range(model.L)]
    w, model.window = model.window, 0  # (the prompt itself runs on the model's cache)
    for pos, tok in enumerate(prompt):
        model.step(tok, pos, own)
    model.window = w
    paged = [[Cache(model.s.n_kv_heads, model.s.head_dim) for _ in range(2)] for _ in range(model.L)]
    for a, b in zip(own, paged):
        for x, y in zip(a, b):
            if prompt:
                y.append(0, x.values(0))
    return paged


def logp(x):
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


def search(model, caches, token, pos, n_steps, beams, eos):
    hyps = [(0.0, [], caches, token, False)]
    top = 0.0
    for i in range(n_steps):
        cand = []
        for w, (score, toks, c, tok, done) in enumerate(hyps):
            if done:
                cand.append((score, w, eos, c, True))
                continue
            x = model.step(tok, pos + i, c)
            top = max(top, np.abs(x).max())
            lp = score + logp(x)
            for t in np.argsort(-lp, kind="stable")[:beams]:
                cand.append((lp[t], w, int(t), c, False))
        cand.sort(key=lambda a: (-a[0], a[1], a[2]))
        hyps = [(s, hyps[w][1] + [t], copy.deepcopy(c), t, d or t == eos) for s, w, t, c, d in cand[:beams]]
    return hyps, top


def score_of(model, caches, token, pos, toks, eos):
    c, total = copy.deepcopy(caches), 0.0
    for i, t in enumerate(toks):
        total += logp(model.step(token, pos + i, c))[t]
        token = int(t)
        if token == eos:
            assert all(int(x) == eos for x in toks[i:])
            break
    return total


CASES = [
    # dtype, spec, prompt, steps, beams, eos, window, sinks, kvbits
    ("fp16", dict(head_dim=64, dim=128, hidden_dim=256), 20, 9, 4, -1, 0, 0, 16),
    ("fp8", dict(head_dim=64, dim=128, hidden_dim=256), 61, 70, 3, -1, 0, 0, 16),   # across pages, forks inside pages
    ("gf4", dict(head_dim=128, dim=256, hidden_dim=256, n_heads=4, n_kv_heads=1), 64, 6, 5, -1, 0, 0, 16),
    ("fp8", dict(head_dim=64, dim=128, hidden_dim=256), 150, 12, 4, -1, 70, 3, 16),  # a window whose pages are given up
    ("fp16", dict(head_dim=64, dim=128, hidden_dim=256), 33, 8, 4, -1, 0, 0, 8),    # out of an fp8 cache
    ("fp8", dict(head_dim=64, dim=128, hidden_dim=256, n_experts=4, n_experts_active=2), 17, 6, 4, -1, 0, 0, 16),
    ("fp16", dict(head_dim=96, dim=192, hidden_dim=256, n_heads=2, n_kv_heads=1), 0, 7, 2, -1, 0, 0, 16),  # no prompt
    ("fp16", dict(head_dim=64, dim=128, hidden_dim=256, vocab_size=40), 5, 1, 32, -1, 0, 0, 16),           # one step, the most beams
    ("fp16", dict(head_dim=64, dim=128, hidden_dim=256, vocab_size=24), 9, 40, 3, "early", 0, 0, 16),      # hypotheses that end, and a search that does
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_beam_search_of_a_model(hiplib, case):
    dtype, kw, n_prompt, n_steps, beams, eos, window, sinks, kvbits = CASES[case]
    spec = cf.tiny_spec(f"beam{case}", max_seq_len=256, **kw)
    tensors, md = cf.synth_model(spec, dtype, seed=40 + case)
    rng = np.random.default_rng(case)
    prompt = [int(t) for t in rng.integers(1, spec.vocab_size, n_prompt)]
    token = int(rng.integers(1, spec.vocab_size))
    m = Model(tensors, md, spec, dtype, window, sinks)
    caches = prompt_caches(m, prompt, kvbits == 8)
    if eos == "early":  # a token that the search takes soon
        eos = search(m, copy.deepcopy(caches), token, n_prompt, 3, beams, -1)[0][0][1][1]
    want, top = search(m, copy.deepcopy(caches), token, n_prompt, n_steps, beams, eos)
    gpu = HipBackend(HostModel(tensors, md), kvbits=kvbits)
    if prompt:
        gpu.prefill(prompt, 0)
    toks, scores = gpu.decode_beam(token, n_prompt, n_steps, beams, eos=eos, window=window, sinks=sinks)
    tol = n_steps * 2 * FP8KV_TOL * top
    np.testing.assert_allclose(scores, [h[0] for h in want], rtol=0, atol=tol)
    assert (np.diff(scores) <= 0).all()
    assert len({tuple(t) for t in toks.tolist()}) == beams
    for t, s in zip(toks, scores):
        assert abs(score_of(m, caches, token, n_prompt, t, eos) - s) <= tol
    # again: the same; and smaller, then larger, searches on the same buffers
    again = gpu.decode_beam(token, n_prompt, n_steps, beams, eos=eos, window=window, sinks=sinks)
    np.testing.assert_array_equal(again[0], toks), np.testing.assert_array_equal(again[1], scores)
    one = gpu.decode_beam(token, n_prompt, 1, 1)
    assert one[0].shape == (1, 1)
    gpu.decode_beam(token, n_prompt, n_steps + 2, beams)
    again = gpu.decode_beam(token, n_prompt, n_steps, beams, eos=eos, window=window, sinks=sinks)
    np.testing.assert_array_equal(again[0], toks), np.testing.assert_array_equal(again[1], scores)
    # the model's own cache is as it was
    if prompt:
        other = HipBackend(HostModel(tensors, md), kvbits=kvbits)
        other.prefill(prompt, 0)
        assert rel_err(gpu.forward(token, n_prompt).copy(), other.forward(token, n_prompt)) == 0.0
        other.close()
    gpu.close()


@pytest.mark.gpu
def test_beam_search_refuses(hiplib):
    spec = cf.tiny_spec("beamr", head_dim=64, dim=128, hidden_dim=256)
    tensors, md = cf.synth_model(spec, "fp16", seed=1)
    gpu = HipBackend(HostModel(tensors, md))
    n = gpu.model.config.seq_len
    for args, kw, words in [((3, n, 1, 2), {}, "context window"), ((3, n - 2, 3, 2), {}, "context window"), ((3, -1, 3, 2), {}, "context window"), ((-1, 0, 3, 2), {}, "vocabulary"),
                            ((spec.vocab_size, 0, 3, 2), {}, "vocabulary"), ((3, 0, 3, 2), dict(eos=spec.vocab_size), "vocabulary"), ((3, 0, 3, 2), dict(window=-1), "negative"),
                            ((3, 0, 3, 33), {}, "beams"), ((3, 0, 0, 3), {}, "step")]:
        with pytest.raises(ValueError, match=words):
            gpu.decode_beam(*args, **kw)
    assert gpu.decode_beam(3, n - 3, 3, 2)[0].shape == (2, 3)
    gpu.close()
    spec = cf.tiny_spec("beamd")  # head size 16
    tensors, md = cf.synth_model(spec, "fp16", seed=1)
    gpu = HipBackend(HostModel(tensors, md))
    with pytest.raises(ValueError, match="head sizes"):
        gpu.decode_beam(3, 0, 3, 2)
    gpu.close()


def test_beam_options_layout(tmp_path):
    import ctypes as C
    import os
    import subprocess

    from conftest import ROOT

    src = tmp_path / "o.c"
    names = [f for f, _ in abi.BeamOptions._fields_]
    src.write_text(f'#include <stdio.h>\n#include "{os.path.join(ROOT, "include", "calm_hip.h")}"\nint main(void) {{ printf("%zu\\n", sizeof(struct BeamOptions)); '
                   + " ".join(f'printf("%zu\\n", offsetof(struct BeamOptions, {n}));' for n in names) + " return 0; }")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "o")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "o")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(abi.BeamOptions)] + [getattr(abi.BeamOptions, n).offset for n in names]
