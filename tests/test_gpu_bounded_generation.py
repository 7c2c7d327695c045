"""examples/bounded_generation.py against a float64 restatement of the whole
loop that follows the program's own evictions and chosen tokens.

Bar: with U = 2^-24 and values of size 1, a projection's sum of 256 products of
variance 1 / 256 is off by about 16 U (rms), a score by 16 U sqrt(2), an output,
a logit (512 products) and a log probability by 2 to 5 times that, about 5e-6.
Fifty times as much is allowed, 2^-12; a slot left out or counted twice moves a
logit by 1 / 64 at least, 60 times the bar.  A weight in the history gathers
that over its steps: 2^-12 of itself and 2^-12 more."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BAR = 2.0 ** -12


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "bounded_generation.py"
    spec = importlib.util.spec_from_file_location("bounded_generation", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("keep,slack,recent,steps,new", [(48, 16, 12, 90, 40), (17, 1, 5, 40, 20), (40, 24, 0, 30, 10)])
def test_scores_and_evictions(keep, slack, recent, steps, new):
    m = example()
    w = m.weights(3)
    text = np.random.default_rng(4).integers(0, m.VOCAB, (3, steps)).astype(np.int32)
    r = m.run(w, text, new, keep, slack, recent, dtype="f32")
    assert len(r["evictions"]) == max(0, -(-(steps + new - keep - slack) // slack))
    w = {name: x.astype(np.float64) for name, x in w.items()}
    G, D = m.N_HEAD // m.N_HEAD_KV, m.HEAD_DIM
    evictions = dict(r["evictions"])
    tokens = r["tokens"]
    assert np.array_equal(tokens[:steps], text.T)
    for b in range(text.shape[0]):
        K, V, W, P = ([[] for _ in range(m.N_HEAD_KV)] for _ in range(4))
        for t in range(steps + new):
            if t in evictions:
                for h in range(m.N_HEAD_KV):
                    kept = evictions[t][b, h]
                    assert len(set(kept.tolist())) == keep and kept.min() >= 0 and kept.max() < keep + slack
                    gone = sorted(set(range(keep + slack)) - set(kept.tolist()))
                    newest = max(P[h])
                    assert all(P[h][j] <= newest - recent for j in gone)
                    old = [W[h][j] for j in kept if P[h][j] <= newest - recent]
                    heaviest = max(W[h][j] for j in gone)
                    assert min(old) >= heaviest - 2 * BAR * (1 + heaviest)
                    for c in (K, V, W, P):
                        c[h] = [c[h][j] for j in kept]
            x = w["embed"][tokens[t, b]]
            q, kn, vn = w["q"] @ x, w["k"] @ x, w["v"] @ x
            out = np.zeros(m.N_HEAD * D)
            for h in range(m.N_HEAD_KV):
                K[h].append(kn[h * D:(h + 1) * D]), V[h].append(vn[h * D:(h + 1) * D]), W[h].append(0.0), P[h].append(t)
                total = np.zeros(len(W[h]))
                for i in range(h * G, (h + 1) * G):
                    s = np.stack(K[h]) @ q[i * D:(i + 1) * D] / np.sqrt(D)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[i * D:(i + 1) * D] = p @ np.stack(V[h])
                    total += p
                W[h] = list(np.array(W[h]) + total)
            logits = w["head"] @ out
            lse = logits.max() + np.log(np.exp(logits - logits.max()).sum())
            p = np.exp(logits - lse)
            assert abs(r["entropy"][t, b] - (lse - (p * logits).sum())) < 4 * BAR
            assert np.allclose(r["top_logprob"][t, b], logits[r["top_id"][t, b]] - lse, rtol=0, atol=BAR)
            assert np.sort(logits)[-1] - logits[r["top_id"][t, b, 0]] < 2 * BAR
            nxt = tokens[t + 1, b]
            assert abs(r["logprob"][t, b] - (logits[nxt] - lse)) < BAR
            assert np.sum(logits > logits[nxt] + 2 * BAR) <= r["rank"][t, b] <= np.sum(logits > logits[nxt] - 2 * BAR)
            if t + 1 >= steps:
                assert nxt == r["top_id"][t, b, 0]
        for h in range(m.N_HEAD_KV):
            assert r["pos"][b, h].tolist() == P[h]
            got = r["weight"][b, h]
            assert np.all(np.abs(got - np.array(W[h])) <= BAR * (1 + np.array(W[h])))


def test_bf16_cache_and_command(capsys, monkeypatch):
    m = example()
    monkeypatch.setattr("sys.argv", ["bounded_generation.py", "--seqs", "2", "--text", "40", "--new", "20", "--keep", "16", "--slack", "8"])
    m.main()
    assert "evictions to 16" in capsys.readouterr().out
