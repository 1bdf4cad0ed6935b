"""decode_beam_hip step by step: what each step keeps are the best continuations of what the step before kept.

A search of i steps returns the hypotheses that step i keeps, and the steps of a longer search are the same steps, so searches of 1, 2, .. n steps show every
selection.  Each is held against the 64-bit restatement of tests/test_beam_decode.py along the search's own hypotheses, from the search's own scores of
the step before, so that a step answers for its own error alone and nothing adds up.

Tolerance: a step's logits are off by conftest's logit_tol (1e-3 of the largest; 4e-3 where the prompt comes out of an e5m2 cache), a log-probability by twice that
(the logit and the sum), and so is a total: EPS = 2 * logit_tol * max|logit|.  Of two candidates whose restated totals are further apart than
2 * EPS the larger must be kept before the smaller."""
import copy

import numpy as np
import pytest

from calm_amd import calmfile as cf
from calm_amd.host import HipBackend, HostModel
from conftest import logit_tol
from test_beam_decode import CASES, Model, logp, prompt_caches, search


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_step_keeps_the_best(hiplib, case):
    dtype, kw, n_prompt, n_steps, beams, eos, window, sinks, kvbits = CASES[case]
    spec = cf.tiny_spec(f"beam{case}", max_seq_len=256, **kw)
    tensors, md = cf.synth_model(spec, dtype, seed=40 + case)
    rng = np.random.default_rng(case)
    prompt = [int(t) for t in rng.integers(1, spec.vocab_size, n_prompt)]
    token = int(rng.integers(1, spec.vocab_size))
    m = Model(tensors, md, spec, dtype, window, sinks)
    caches = prompt_caches(m, prompt, kvbits == 8)
    if eos == "early":
        eos = search(m, copy.deepcopy(caches), token, n_prompt, 3, beams, -1)[0][0][1][1]
    gpu = HipBackend(HostModel(tensors, md), kvbits=kvbits)
    if prompt:
        gpu.prefill(prompt, 0)
    # what the step before kept: tokens -> (score, the restatement's caches behind them)
    kept = {(): (0.0, caches)}
    checked = 0
    for i in range(1, n_steps + 1):
        toks, scores = gpu.decode_beam(token, n_prompt, i, beams, eos=eos, window=window, sinks=sinks)
        rows = [tuple(int(t) for t in r) for r in toks]
        assert len(set(rows)) == beams and (np.diff(scores) <= 0).all()
        assert all(r[:-1] in kept for r in rows), "a hypothesis that the step before did not keep"
        total, after, top = {}, {}, 0.0  # restated totals of every continuation
        for h, (s, c) in kept.items():
            if s == -np.inf:
                continue
            if h and h[-1] == eos:
                total[h + (eos,)], after[h] = s, c  # finished: its score unchanged
                continue
            c = copy.deepcopy(c)
            x = m.step(h[-1] if h else token, n_prompt + i - 1, c)
            after[h], top = c, max(top, np.abs(x).max())
            for t, v in enumerate(s + logp(x)):
                total[h + (t,)] = v
        eps = 2 * logit_tol(kvbits) * top
        for r, s in zip(rows, scores):
            if s == -np.inf:
                assert len(total) < beams  # (fewer continuations than beams)
            else:
                assert abs(s - total[r]) <= (eps if not (r[-1] == eos and r[-2:-1] == (eos,)) else 0.0), (i, r, s, total[r])
        least = min(total[r] for r in rows if r in total)
        best_left = max((v for r, v in total.items() if r not in set(rows)), default=-np.inf)
        assert best_left <= least + 2 * eps, (i, best_left, least, eps)
        checked += len(total)
        kept = {r: (float(s), after.get(r[:-1])) for r, s in zip(rows, scores)}
    assert checked >= n_steps
    gpu.close()
